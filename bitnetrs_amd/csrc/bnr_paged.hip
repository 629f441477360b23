// bnr_paged.hip -- gfx950 kernels of the paged KV cache: rows rotated and
// quantised as they are written (append), read back as fp32 (read), and the
// attention of one new token of each sequence over its pages (decode), in the
// form that takes any head dimension, group, page size and alignment.
#include "bnr_paged.h"

namespace bnr {
namespace {

constexpr int kWaves = 4;  // waves of a workgroup, all kernels of this file
constexpr long long kMaxRowGrid = 1 << 20;  // workgroups of the row kernels at most

// ---------------------------------------------------------------------------
// Append, any even head dimension.  One wave per row: lane l holds the pairs
// (i, i + d/2) for i = l, l + 64, ..., so that a rotation needs no other
// lane, and the row's maximum is one wave reduction.
// ---------------------------------------------------------------------------
constexpr int kPairs = kPagedMaxDim / 2 / 64;

template <int F>
__global__ __launch_bounds__(64 * kWaves) void paged_append_kernel(PagedAppendArgs a) {
  const int lane = threadIdx.x & 63;
  const int half = a.pool.d / 2;
  for (long long row = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6); row < append_rows(a);
       row += (long long)gridDim.x * kWaves) {
    AppendRow r;
    if (!append_row(a, row, r)) continue;
    float lo[kPairs], hi[kPairs];
    float mx = 0.f;
    bool finite = true;
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int i = lane + 64 * j;
      lo[j] = hi[j] = 0.f;
      if (i < half) {
        lo[j] = r.in[i];
        hi[j] = r.in[half + i];
        if (r.cos) {
          float l, h;
          rot_pair(lo[j], hi[j], r.cos[i], r.sin[i], l, h);
          lo[j] = l;
          hi[j] = h;
        }
        mx = fmaxf(mx, fmaxf(fabsf(lo[j]), fabsf(hi[j])));
        finite = finite && is_finite(lo[j]) && is_finite(hi[j]);
      }
    }
    if (r.out) {
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const int i = lane + 64 * j;
        if (i < half) {
          r.out[i] = lo[j];
          r.out[half + i] = hi[j];
        }
      }
      continue;
    }
    float inv = 1.f;
    if (kPagedScaled<F>) {
      const RowScale s = row_scale<F>(wave_max(mx), __all(finite));
      inv = s.inv;
      if (lane == 0) *r.scale = s.scale;
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j) {
      const int i = lane + 64 * j;
      if (i < half) {
        store_code<F>(r.codes, r.at + i, lo[j], inv);
        store_code<F>(r.codes, r.at + half + i, hi[j], inv);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Read, any head dimension: one wave per (sequence, kv head, row), k then v.
// ---------------------------------------------------------------------------
template <int F>
__global__ __launch_bounds__(64 * kWaves) void paged_read_kernel(PagedReadArgs a) {
  const int lane = threadIdx.x & 63;
  const long long per = a.cap * a.pool.n_kv;
  for (long long n = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6); n < per * a.batch;
       n += (long long)gridDim.x * kWaves) {
    const long long b = n / per;
    const int h = (int)((n - b * per) / a.cap);
    const long long i = n - b * per - h * a.cap;
    const int start = a.starts ? a.starts[b] : 0;
    const int len = paged_len(a.lens[b], a.pool);
    const long long t = start + i;
    if (start < 0 || t >= len) continue;
    const long long at = paged_row(a.pool, b, h, (int)t);
    const int d = a.pool.d;
    float *ko = a.k_out + n * d, *vo = a.v_out + n * d;
    float ks = 1.f, vs = 1.f;
    if (kPagedScaled<F> && at >= 0) {
      ks = a.pool.k_scales[at];
      vs = a.pool.v_scales[at];
    }
    for (int x = lane; x < d; x += 64) {
      ko[x] = at < 0 ? 0.f : load_code<F>(a.pool.k, at * d + x) * ks;
      vo[x] = at < 0 ? 0.f : load_code<F>(a.pool.v, at * d + x) * vs;
    }
  }
}

// ---------------------------------------------------------------------------
// Decode attention, any shape.  An item is one (sequence, query head); a wave
// takes every fourth row of its piece, one row at a time: the 64 lanes hold
// the row's elements l, l + 64, ..., a dot product is one wave reduction, and
// the softmax's running maximum and sum move row by row.
// ---------------------------------------------------------------------------
constexpr int kElems = kPagedMaxDim / 64;

template <int F>
__global__ __launch_bounds__(64 * kWaves) void paged_decode_generic_kernel(PagedDecodeArgs a) {
  __shared__ float s_o[kWaves][kPagedMaxDim];
  __shared__ float s_m[kWaves], s_l[kWaves];
  __shared__ JoinShared<kWaves, 1> s_join;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = a.pool.d;
  const int first_len = paged_first_len(a);
  PagedShare sh = paged_share(a, a.n_heads);
  for (PagedPiece p; sh.next(a.lens, a.pool, p);) {
    const int h = p.h / a.group;
    const float *q = a.q + ((long long)p.b * a.n_heads + p.h) * d;
    float qr[kElems], o[kElems];
#pragma unroll
    for (int j = 0; j < kElems; ++j) {
      qr[j] = lane + 64 * j < d ? q[lane + 64 * j] : 0.f;
      o[j] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    for (int t = p.row0 + wave; t < p.row1; t += kWaves) {
      const long long at = paged_row(a.pool, p.b, h, t);
      if (at < 0) continue;
      float x = 0.f;
#pragma unroll
      for (int j = 0; j < kElems; ++j)
        if (lane + 64 * j < d) x = fmaf(qr[j], load_code<F>(a.pool.k, at * d + lane + 64 * j), x);
      x = wave_sum(x) * a.scale_log2;
      float vs = 1.f;
      if (kPagedScaled<F>) {
        x *= a.pool.k_scales[at];
        vs = a.pool.v_scales[at];
      }
      const float mn = fmaxf(m, x), mu = mn == -INFINITY ? 0.f : mn;
      const float keep = fast_exp2(m - mu), w = fast_exp2(x - mu);
      m = mn;
      l = fmaf(l, keep, w);
#pragma unroll
      for (int j = 0; j < kElems; ++j)
        if (lane + 64 * j < d)
          o[j] = fmaf(o[j], keep, w * (load_code<F>(a.pool.v, at * d + lane + 64 * j) * vs));
    }
    __syncthreads();  // the piece before this one has been read
#pragma unroll
    for (int j = 0; j < kElems; ++j)
      if (lane + 64 * j < d) s_o[wave][lane + 64 * j] = o[j];
    if (lane == 0) {
      s_m[wave] = m;
      s_l[wave] = l;
    }
    __syncthreads();
    const auto get = [&](int w, int, int x, float(&to)[1]) { to[0] = s_o[w][x]; };
    paged_finish<kWaves, 1, kPagedMaxDim>(a, p, sh.wg, sh.wg_of(p.item0), sh.wg_of(p.item1 - 1), get, s_m,
                                          s_l, 1, s_join);
  }
  paged_empty(a, first_len);
}

}  // namespace

#define BNR_BY_FORMAT(F, CALL)                         \
  switch (F) {                                         \
    case kPagedF32: CALL(kPagedF32); break;            \
    case kPagedBf16: CALL(kPagedBf16); break;          \
    case kPagedFp8: CALL(kPagedFp8); break;            \
    case kPagedInt8: CALL(kPagedInt8); break;          \
    default: return hipErrorInvalidValue;              \
  }

// Workgroups for `rows` rows, one a wave; past the limit a wave takes several.
static dim3 row_grid(long long rows) {
  const long long wgs = (rows + kWaves - 1) / kWaves;
  return dim3((unsigned)(wgs < kMaxRowGrid ? wgs : kMaxRowGrid));
}

hipError_t launch_paged_append(const PagedAppendArgs &a, int format, hipStream_t s) {
  const dim3 grid = row_grid(append_rows(a));
#define CALL(F) paged_append_kernel<F><<<grid, 64 * kWaves, 0, s>>>(a)
  BNR_BY_FORMAT(format, CALL)
#undef CALL
  return hipGetLastError();
}

hipError_t launch_paged_read(const PagedReadArgs &a, int format, hipStream_t s) {
  const dim3 grid = row_grid(a.batch * a.cap * a.pool.n_kv);
#define CALL(F) paged_read_kernel<F><<<grid, 64 * kWaves, 0, s>>>(a)
  BNR_BY_FORMAT(format, CALL)
#undef CALL
  return hipGetLastError();
}

hipError_t launch_paged_decode_generic(const PagedDecodeArgs &a, int format, hipStream_t s) {
  const dim3 grid((unsigned)a.wgs);
#define CALL(F) paged_decode_generic_kernel<F><<<grid, 64 * kWaves, 0, s>>>(a)
  BNR_BY_FORMAT(format, CALL)
#undef CALL
  return hipGetLastError();
}

}  // namespace bnr

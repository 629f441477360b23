// bnr_paged.hip -- gfx950 kernels of the paged KV cache: rows rotated and
// quantised as they are written (append), read back as fp32 (read), and the
// attention of one new token of each sequence over its pages (decode), in the
// form that takes any head dimension, group, page size and alignment.
#include "bnr_paged.h"

#include <algorithm>

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

// Maximum over the N lanes (a power of two) that share a row.
template <int N>
__device__ __forceinline__ unsigned row_largest(unsigned v) {
  auto step = [&](unsigned u) { v = v > u ? v : u; };
#define BNR_DPP(CTRL) (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false)
  if (N >= 2) step(BNR_DPP(0xB1));    // quad_perm [1,0,3,2]
  if (N >= 4) step(BNR_DPP(0x4E));    // quad_perm [2,3,0,1]
  if (N >= 8) step(BNR_DPP(0x141));   // row_half_mirror
  if (N >= 16) step(BNR_DPP(0x140));  // row_mirror
#undef BNR_DPP
  if (N >= 32) step(__shfl_xor(v, 16));
  if (N >= 64) step(__shfl_xor(v, 32));
  return v;
}

// What a wave wrote to LDS is there for its other lanes: LDS works in order, so
// only the compiler has to keep the order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Eight neighbouring elements (n of them in the row) as codes, and their
// group's exponent: the lane's neighbours have the group's others.
__device__ __forceinline__ void store_group4(const AppendRow &r, bool in, int x, int n, float4 lo, float4 hi) {
  unsigned largest = max(max(max(magnitude(lo.x), magnitude(lo.y)), max(magnitude(lo.z), magnitude(lo.w))),
                         max(max(magnitude(hi.x), magnitude(hi.y)), max(magnitude(hi.z), magnitude(hi.w))));
  largest = row_largest<kPagedGroup4 / 8>(largest);
  const unsigned e = exponent4(largest), w = codes4(lo, hi, e);
  if (!in || n <= 0) return;
  if (x % kPagedGroup4 == 0) r.exps[x / kPagedGroup4] = (unsigned char)e;
  unsigned char *to = static_cast<unsigned char *>(r.codes) + (r.at + x) / 2;
  if (n >= 8 && reinterpret_cast<uintptr_t>(to) % 4 == 0) {
    *reinterpret_cast<unsigned *>(to) = w;
  } else {
    for (int i = 0; 2 * i < n && i < 4; ++i) to[i] = (unsigned char)(w >> (8 * i));
  }
}

template <int F>
__global__ __launch_bounds__(64 * kWaves) void paged_append_kernel(PagedAppendArgs a) {
  __shared__ float s_row[F == kPagedFp4 ? kWaves : 1][F == kPagedFp4 ? kPagedMaxDim : 1];
  const int lane = threadIdx.x & 63, half = a.pool.d / 2, per = append_rows(a);
  for (long long n = (long long)blockIdx.x * kWaves + (threadIdx.x >> 6); n < a.n_tokens * per;
       n += (long long)gridDim.x * kWaves) {
    const long long token = n / per;
    const int j = (int)(n - token * per);
    AppendRow r;
    if (!append_row(a, token, j, r)) continue;
    const float *in = append_in(a, token, j);
    float lo[kPairs], hi[kPairs];
    unsigned largest = 0;
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const int i = lane + 64 * k;
      lo[k] = hi[k] = 0.f;
      if (i < half) {
        lo[k] = in[i];
        hi[k] = in[half + i];
        if (r.cos) {
          float l, h;
          rot_pair(lo[k], hi[k], r.cos[i], r.sin[i], l, h);
          lo[k] = l;
          hi[k] = h;
        }
        largest = max(largest, max(magnitude(lo[k]), magnitude(hi[k])));
      }
    }
    if constexpr (F == kPagedFp4) {
      if (!r.out) {
        // eight neighbours a lane, of which a group of four has one exponent
        float *row = s_row[threadIdx.x >> 6];
        wave_order();  // the row before this one has been read
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          const int i = lane + 64 * k;
          if (i >= half) continue;
          row[i] = lo[k];
          row[half + i] = hi[k];
        }
        wave_order();
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 8 * lane + i < a.pool.d ? row[8 * lane + i] : 0.f;
        store_group4(r, true, 8 * lane, a.pool.d - 8 * lane, make_float4(x[0], x[1], x[2], x[3]),
                     make_float4(x[4], x[5], x[6], x[7]));
        continue;
      }
    }
    float inv = 1.f;
    if (kPagedScaled<F> && !r.out) {
      const RowScale s = row_scale<F>(row_largest<64>(largest));
      inv = s.inv;
      if (lane == 0) *r.scale = s.scale;
    }
#pragma unroll
    for (int k = 0; k < kPairs; ++k) {
      const int i = lane + 64 * k;
      if (i >= half) continue;
      if (r.out) {
        r.out[i] = lo[k];
        r.out[half + i] = hi[k];
      } else if constexpr (F != kPagedFp4) {
        store_code<F>(r.codes, r.at + i, lo[k], inv);
        store_code<F>(r.codes, r.at + half + i, hi[k], inv);
      }
    }
  }
}

// ---------------------------------------------------------------------------
// Append, head dimensions that are multiples of 8, 16-byte aligned rows: L
// lanes (d / 8, rounded up to a power of two) share a row, each with 4 pairs:
// 16 bytes of either half.  A workgroup takes a run of rows, a token's rows
// being neighbours, so that most tokens' positions, table entries and
// rotations are read by one workgroup only.  Bound by the rows' bytes; with the
// loads of two or four rows in flight in a thread 8000 tokens of 32/8 heads
// took 3 and 10 us more.
// ---------------------------------------------------------------------------
template <int F>
__device__ __forceinline__ void store_codes4(void *codes, long long at, float4 x, float inv) {
  if constexpr (F == kPagedF32) {
    st4(static_cast<float *>(codes) + at, x);
  } else if constexpr (F == kPagedBf16) {
    uint2 w;
    w.x = code_of<F>(x.x, inv) | code_of<F>(x.y, inv) << 16;
    w.y = code_of<F>(x.z, inv) | code_of<F>(x.w, inv) << 16;
    *reinterpret_cast<uint2 *>(static_cast<unsigned short *>(codes) + at) = w;
  } else {
    *reinterpret_cast<unsigned *>(static_cast<unsigned char *>(codes) + at) =
        code_of<F>(x.x, inv) | code_of<F>(x.y, inv) << 8 | code_of<F>(x.z, inv) << 16 |
        code_of<F>(x.w, inv) << 24;
  }
}

__device__ __forceinline__ unsigned largest4(float4 x) {
  return max(max(magnitude(x.x), magnitude(x.y)), max(magnitude(x.z), magnitude(x.w)));
}

template <int F, int L>
__global__ __launch_bounds__(64 * kWaves) void paged_append_vec_kernel(PagedAppendArgs a, bool stream) {
  constexpr int kRows = 64 * kWaves / L;
  __shared__ float4 s_row[F == kPagedFp4 ? kRows : 1][F == kPagedFp4 ? 2 * L : 1];
  const int x = 4 * (threadIdx.x % L), half = a.pool.d / 2, per = append_rows(a);
  const unsigned long long total = (unsigned long long)a.n_tokens * per;
  for (unsigned long long n0 = (unsigned long long)blockIdx.x * kRows; n0 < total;
       n0 += (unsigned long long)gridDim.x * kRows) {
    const unsigned long long first = n0 >> 32 ? n0 / per : (unsigned)n0 / (unsigned)per;
    const int n = (int)(n0 - first * per) + threadIdx.x / L, i = n / per, j = n - i * per;
    const long long token = (long long)first + i;
    float4 lo = make_float4(0.f, 0.f, 0.f, 0.f), hi = lo;
    AppendRow r;
    bool in = token < a.n_tokens && x < half;
    if (in) {
      const float *src = append_in(a, token, j);
      lo = ld4(src + x);
      hi = ld4(src + half + x);
      in = append_row(a, token, j, r);
    }
    if (in && r.cos) {
      const float4 c = ld4(r.cos + x), s = ld4(r.sin + x);
      float4 l, h;
      rot4(lo, hi, c, s, l, h);
      lo = l;
      hi = h;
    }
    float inv = 1.f;
    if (kPagedScaled<F>) {
      // every lane takes part: those past a row's end bring zeros
      const RowScale s = row_scale<F>(row_largest<L>(max(largest4(lo), largest4(hi))));
      inv = s.inv;
      if (in && !r.out && x == 0) *r.scale = s.scale;
    }
    if constexpr (F == kPagedFp4) {
      // the row as eight neighbours a lane; a row's lanes are of one wave
      float4 *row = s_row[threadIdx.x / L];
      wave_order();  // the rows before these have been read
      if (x < half) {
        row[x / 4] = lo;
        row[(half + x) / 4] = hi;
      }
      wave_order();
      float4 l8 = make_float4(0.f, 0.f, 0.f, 0.f), h8 = l8;
      if (2 * x < a.pool.d) {
        l8 = row[x / 2];
        h8 = row[x / 2 + 1];
      }
      // every lane takes part: those past a row's end bring zeros
      store_group4(r, in && !r.out, 2 * x, a.pool.d - 2 * x, l8, h8);
    }
    if (!in) continue;
    if (r.out && stream) {
      st4_nt(r.out + x, lo);
      st4_nt(r.out + half + x, hi);
    } else if (r.out) {
      st4(r.out + x, lo);
      st4(r.out + half + x, hi);
    } else if constexpr (F != kPagedFp4) {
      store_codes4<F>(r.codes, r.at + x, lo, inv);
      store_codes4<F>(r.codes, r.at + half + x, hi, inv);
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
      ko[x] = at < 0 ? 0.f : load_element<F>(a.pool.k, a.pool.k_exps, at, d, x) * ks;
      vo[x] = at < 0 ? 0.f : load_element<F>(a.pool.v, a.pool.v_exps, at, d, x) * vs;
    }
  }
}

// ---------------------------------------------------------------------------
// Read, head dimensions that are multiples of 4, rows and outputs aligned to
// four elements: L lanes (d / 4, rounded up to a power of two) share a row,
// each with four elements, so that a wave's stores are whole lines; a
// workgroup takes equal shares of all rows that are to be read, kReadRows of
// one kv head at a time, k and v, a thread with all its loads in flight.
// Bound by the outputs' bytes: 4 of them to one or two of the rows'.
// ---------------------------------------------------------------------------
// Workgroups at most: many more than the card holds, so that what is written
// at one time lies close together.  32 int8 sequences of 100 to 4096 rows: 90
// us; 95 with 4096, 102 with 2048, 108 with a workgroup for every 32 rows that
// there is room for (half of them without a row).
constexpr int kReadWgs = 16384;
constexpr int kReadPasses = 4;  // 2: 111 us, 8: 116 us, of 107 us then
template <int L>
constexpr int kReadRows = kReadPasses * 64 * kWaves / L;

// Four codes as fp32, before the scale; `power`: FP4's.
template <int F>
__device__ __forceinline__ float4 load_codes4(const void *codes, long long at, float power) {
  if constexpr (F == kPagedF32) {
    return ld4(static_cast<const float *>(codes) + at);
  } else if constexpr (F == kPagedFp4) {
    const unsigned w = *reinterpret_cast<const unsigned short *>(static_cast<const unsigned char *>(codes) + at / 2);
    const unsigned p = pair4<0>(w, power), q = pair4<1>(w, power);
    return make_float4(low16(p), high16(p), low16(q), high16(q));
  } else if constexpr (F == kPagedBf16) {
    const uint2 w = *reinterpret_cast<const uint2 *>(static_cast<const unsigned short *>(codes) + at);
    return make_float4(__builtin_bit_cast(float, w.x << 16), __builtin_bit_cast(float, w.x & 0xffff0000u),
                       __builtin_bit_cast(float, w.y << 16), __builtin_bit_cast(float, w.y & 0xffff0000u));
  } else {
    const unsigned w = *reinterpret_cast<const unsigned *>(static_cast<const unsigned char *>(codes) + at);
    if constexpr (F == kPagedInt8)
      return make_float4((float)(signed char)w, (float)(signed char)(w >> 8),
                         (float)(signed char)(w >> 16), (float)(signed char)(w >> 24));
    return make_float4(__builtin_amdgcn_cvt_f32_fp8((int)w, 0), __builtin_amdgcn_cvt_f32_fp8((int)w, 1),
                       __builtin_amdgcn_cvt_f32_fp8((int)w, 2), __builtin_amdgcn_cvt_f32_fp8((int)w, 3));
  }
}

template <int F, int L>
__global__ __launch_bounds__(64 * kWaves) void paged_read_vec_kernel(PagedReadArgs a) {
  constexpr int kPass = 64 * kWaves / L;  // rows of a pass
  const int x = 4 * (threadIdx.x % L), d = a.pool.d;
  const auto rows = [&](int b) {
    const int start = a.starts ? a.starts[b] : 0, len = paged_len(a.lens[b], a.pool);
    if (start < 0 || start >= len) return 0;
    return len - start < a.cap ? len - start : (int)a.cap;
  };
  PagedShare sh = paged_share(rows, (int)a.batch, a.pool.n_kv, a.tile, a.wgs);
  for (PagedPiece p; sh.next(rows, p);) {
    const int start = a.starts ? a.starts[p.b] : 0;
    const long long to = ((long long)p.b * a.pool.n_kv + p.h) * a.cap;
    for (int i0 = p.row0 + (int)threadIdx.x / L; i0 < p.row1; i0 += kReadRows<L>) {
      if (x >= d) continue;
      long long at[kReadPasses];
      float4 k[kReadPasses], v[kReadPasses];
      float ks[kReadPasses], vs[kReadPasses];
#pragma unroll
      for (int n = 0; n < kReadPasses; ++n) {
        const int i = i0 + n * kPass;
        // past the last row: the first again, not written (a branch would part the loads)
        at[n] = paged_row(a.pool, p.b, p.h, start + (i < p.row1 ? i : i0));
      }
#pragma unroll
      for (int n = 0; n < kReadPasses; ++n) {
        const long long from = at[n] < 0 ? 0 : at[n];
        float kp = 1.f, vp = 1.f;
        if constexpr (F == kPagedFp4) {
          const long long group = from * paged_groups4(d) + x / kPagedGroup4;
          kp = power4(a.pool.k_exps[group]);
          vp = power4(a.pool.v_exps[group]);
        }
        k[n] = load_codes4<F>(a.pool.k, from * d + x, kp);
        v[n] = load_codes4<F>(a.pool.v, from * d + x, vp);
        ks[n] = vs[n] = 1.f;
        if (kPagedScaled<F>) {
          ks[n] = a.pool.k_scales[from];
          vs[n] = a.pool.v_scales[from];
        }
      }
#pragma unroll
      for (int n = 0; n < kReadPasses; ++n) {
        const int i = i0 + n * kPass;
        if (i >= p.row1) break;
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        st4_nt(a.k_out + (to + i) * d + x, at[n] < 0 ? zero : kPagedScaled<F> ? scale4(ks[n], k[n]) : k[n]);
        st4_nt(a.v_out + (to + i) * d + x, at[n] < 0 ? zero : kPagedScaled<F> ? scale4(vs[n], v[n]) : v[n]);
      }
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
  const auto rows = [&](int b) { return paged_len(a.lens[b], a.pool); };
  PagedShare sh = paged_share(rows, a.batch, a.n_heads, a.tile, a.wgs);
  for (PagedPiece p; sh.next(rows, p);) {
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
        if (lane + 64 * j < d)
          x = fmaf(qr[j], load_element<F>(a.pool.k, a.pool.k_exps, at, d, lane + 64 * j), x);
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
          o[j] = fmaf(o[j], keep, w * (load_element<F>(a.pool.v, a.pool.v_exps, at, d, lane + 64 * j) * vs));
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
    paged_finish<kWaves, 1, kPagedMaxDim, 16>(a, p, sh.wg, sh.wg_of(p.item0), sh.wg_of(p.item1 - 1), get, s_m,
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
    case kPagedFp4: CALL(kPagedFp4); break;            \
    default: return hipErrorInvalidValue;              \
  }

// Workgroups for n of them; past the limit a workgroup takes several turns.
static unsigned row_grid(long long n) { return (unsigned)(n < kMaxRowGrid ? n : kMaxRowGrid); }

template <int F, int L>
static void append_vec(const PagedAppendArgs &a, hipStream_t s) {
  const long long rows = a.n_tokens * append_rows(a), per = 64 * kWaves / L;
  // 4 MB of q and more go out with the non-temporal hint.  20/5 heads of 128: 2048 tokens in int8 13.1 -> 12.7
  // us, with the kernels that make the inputs and read q 38.8 -> 37.8; 4096 25.6 -> 22.1 and 67.4 -> 68.7;
  // 8192 46.9 -> 43.8 and 130.5 -> 132.0; 16384 87.8 -> 80.7 and 231.6 -> 223.4.  (40 to 80 MB of q the next
  // kernel would have found in the 256 MB cache; in 4 bits those two are 68.3 -> 68.8 and 133.8 -> 133.0, in
  // bf16 67.1 -> 67.6 and 130.1 both, and 16384 238.2 -> 231.5 and 235.8 -> 223.7.)  64 tokens, if they had
  // it: 3.7 both, 11.2 -> 11.5.
  const bool stream = a.q && a.n_tokens * a.n_heads * a.pool.d >= 1 << 20;
  paged_append_vec_kernel<F, L><<<row_grid((rows + per - 1) / per), 64 * kWaves, 0, s>>>(a, stream);
}

template <int F>
static void append_format(const PagedAppendArgs &a, bool vec, hipStream_t s) {
  const int d = a.pool.d;
  if (!vec)
    paged_append_kernel<F><<<row_grid((a.n_tokens * append_rows(a) + kWaves - 1) / kWaves), 64 * kWaves, 0, s>>>(a);
  else if (d <= 64)
    append_vec<F, 8>(a, s);
  else if (d <= 128)
    append_vec<F, 16>(a, s);
  else if (d <= 256)
    append_vec<F, 32>(a, s);
  else
    append_vec<F, 64>(a, s);
}

hipError_t launch_paged_append(const PagedAppendArgs &a, int format, bool vec, hipStream_t s) {
#define CALL(F) append_format<F>(a, vec, s)
  BNR_BY_FORMAT(format, CALL)
#undef CALL
  return hipGetLastError();
}

template <int F, int L>
static void read_vec(PagedReadArgs a, hipStream_t s) {
  // units that there is room for: under 2^31, and no fewer than workgroups
  const long long items = a.batch * a.pool.n_kv;
  a.tile = kReadRows<L>;
  while ((a.cap + a.tile - 1) / a.tile * items >= 1ll << 31) a.tile *= 2;
  a.wgs = (int)std::min<long long>(kReadWgs, (a.cap + a.tile - 1) / a.tile * items);
  paged_read_vec_kernel<F, L><<<a.wgs, 64 * kWaves, 0, s>>>(a);
}

template <int F>
static void read_format(const PagedReadArgs &a, bool vec, hipStream_t s) {
  const int d = a.pool.d;
  if (!vec)
    paged_read_kernel<F><<<row_grid((a.batch * a.cap * a.pool.n_kv + kWaves - 1) / kWaves), 64 * kWaves, 0, s>>>(a);
  else if (d <= 64)
    read_vec<F, 16>(a, s);
  else if (d <= 128)
    read_vec<F, 32>(a, s);
  else if (d <= 256)
    read_vec<F, 64>(a, s);
  else
    read_vec<F, 128>(a, s);
}

hipError_t launch_paged_read(const PagedReadArgs &a, int format, bool vec, hipStream_t s) {
#define CALL(F) read_format<F>(a, vec, s)
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

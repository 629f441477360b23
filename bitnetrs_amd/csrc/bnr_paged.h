// bnr_paged.h -- device code shared by the paged KV cache's kernels: the four
// row formats, where a row lies, and how a decode launch's work is cut into
// equal shares and joined again.  Included by the .hip sources only.
#pragma once

#include "bnr_device.h"

namespace bnr {

// ---------------------------------------------------------------------------
// Formats.  INT8 and FP8 (e4m3) keep one fp32 scale a row (one token of one
// kv head): with m = max(max|x|, 2^-100) of the row,
//   scale = m / top,  code = round(x * (top / m)),  top = 127 or 448,
// both quotients correctly rounded, the code rounded to nearest, ties to even
// (e4m3's too).  |x * (top / m)| exceeds top by at most 2^-23 of it, which
// rounds to top.  A row that holds an infinity or a NaN gets the scale NaN
// and codes 0, so it reads back as NaN and never as plausible numbers.
// ---------------------------------------------------------------------------
template <int F>
constexpr bool kPagedScaled = F == kPagedFp8 || F == kPagedInt8;
template <int F>
constexpr float kPagedTop = F == kPagedInt8 ? 127.0f : 448.0f;

__device__ __forceinline__ bool is_finite(float x) {
  return (__builtin_bit_cast(unsigned, x) & 0x7f800000u) != 0x7f800000u;
}

struct RowScale {
  float scale, inv;
};
template <int F>
__device__ __forceinline__ RowScale row_scale(float mx, bool finite) {
  const float m = fmaxf(mx, kPagedTiny);
  return finite ? RowScale{m / kPagedTop<F>, kPagedTop<F> / m}
                : RowScale{__builtin_nanf(""), 0.f};
}

// bf16 bits of x, rounded to nearest even; a NaN stays one.
__device__ __forceinline__ unsigned bf16_bits(float x) {
  unsigned u = __builtin_bit_cast(unsigned, x);
  if ((u & 0x7fffffffu) > 0x7f800000u) return (u >> 16) | 0x40u;
  return (u + 0x7fffu + ((u >> 16) & 1u)) >> 16;
}

template <int F>
__device__ __forceinline__ unsigned code_of(float x, float inv) {
  if (F == kPagedBf16) return bf16_bits(x);
  // inv is 0 for a row with a non-finite value; 0 * inf would be NaN
  const float y = inv == 0.f ? 0.f : x * inv;
  if (F == kPagedInt8) return (unsigned)(int)rintf(y) & 0xffu;
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xffu;
}

template <int F>
__device__ __forceinline__ void store_code(void *codes, long long i, float x, float inv) {
  if (F == kPagedF32)
    static_cast<float *>(codes)[i] = x;
  else if (F == kPagedBf16)
    static_cast<unsigned short *>(codes)[i] = (unsigned short)code_of<F>(x, inv);
  else
    static_cast<unsigned char *>(codes)[i] = (unsigned char)code_of<F>(x, inv);
}

// A code's value before its scale.
template <int F>
__device__ __forceinline__ float load_code(const void *codes, long long i) {
  if (F == kPagedF32) return static_cast<const float *>(codes)[i];
  if (F == kPagedBf16)
    return __builtin_bit_cast(float, (unsigned)static_cast<const unsigned short *>(codes)[i] << 16);
  if (F == kPagedInt8) return (float)static_cast<const signed char *>(codes)[i];
  return __builtin_amdgcn_cvt_f32_fp8(static_cast<const unsigned char *>(codes)[i], 0);
}

// ---------------------------------------------------------------------------
// Rows.
// ---------------------------------------------------------------------------
// A sequence's length as the table can hold it.
__device__ __forceinline__ int paged_len(int len, const PagedPool &p) {
  const long long most = p.table_stride * p.page;  // at most INT_MAX, checked by the host
  return len < 0 ? 0 : len > most ? (int)most : len;
}

// The page of row t of a sequence, or -1 where there is none.  0 <= t < stride * page.
__device__ __forceinline__ int paged_page(const PagedPool &p, long long seq, int t) {
  const int page = p.table[seq * p.table_stride + t / p.page];
  return page < 0 || page >= p.n_pages ? -1 : page;
}

// Row t of kv head h, counted in rows of the pool; -1 where its page is not there.
__device__ __forceinline__ long long paged_row(const PagedPool &p, long long seq, int h, int t) {
  const int page = paged_page(p, seq, t);
  if (page < 0) return -1;
  return ((long long)page * p.n_kv + h) * p.page + t % p.page;
}

// Rows of an append launch.
__host__ __device__ __forceinline__ long long append_rows(const PagedAppendArgs &a) {
  return a.n_tokens * ((a.q ? a.n_heads : 0) + 2 * a.pool.n_kv);
}

// Row `row` of an append launch: the q rows of a token, its k rows, its v rows.
struct AppendRow {
  const float *in;
  float *out;           // q rows: where the rotated row goes
  const float *cos, *sin;  // null: not rotated
  void *codes;          // k and v rows: the pool, the row's first element in it,
  long long at;
  float *scale;         // and where its scale goes
};
// False: nothing to do (a token whose position or sequence is outside the
// table, or outside the rotation's tables; a page that is not there).
__device__ __forceinline__ bool append_row(const PagedAppendArgs &a, long long row, AppendRow &r) {
  const PagedPool &p = a.pool;
  const int nq = a.q ? a.n_heads : 0, per = nq + 2 * p.n_kv;
  const long long i = row / per;
  const int j = (int)(row - i * per);
  const int pos = a.positions[i];
  const long long seq = a.seqs ? a.seqs[i] : i;
  if (pos < 0 || pos >= p.table_stride * p.page || seq < 0 || seq >= a.n_seqs) return false;
  if (a.cos_tab && pos >= a.n_positions) return false;
  r = AppendRow{};
  if (a.cos_tab && j < nq + p.n_kv) {
    r.cos = a.cos_tab + (long long)pos * (p.d / 2);
    r.sin = a.sin_tab + (long long)pos * (p.d / 2);
  }
  if (j < nq) {
    r.in = a.q + (i * nq + j) * p.d;
    r.out = a.q_out + (i * nq + j) * p.d;
    return true;
  }
  const bool is_v = j >= nq + p.n_kv;
  const int h = j - nq - (is_v ? p.n_kv : 0);
  const long long at = paged_row(p, seq, h, pos);
  if (at < 0) return false;
  r.in = (is_v ? a.v : a.k) + (i * p.n_kv + h) * p.d;
  r.codes = is_v ? p.v : p.k;
  r.at = at * p.d;
  float *sc = is_v ? p.v_scales : p.k_scales;
  r.scale = sc ? sc + at : nullptr;
  return true;
}

// ---------------------------------------------------------------------------
// Shares of a decode launch.  Sequence b has ceil(lens[b] / tile) units for
// each of its `items` heads; all units in order are one line, and workgroup w
// takes units w * per + min(w, rest) .. of it (total = per * wgs + rest).  A
// workgroup's share is a run of pieces, each of one item: at most its first
// and its last piece belong to items that other workgroups share.  Nothing
// about the lengths is known on the host, so a captured launch serves every
// later step, and ragged batches are balanced to one unit.
// ---------------------------------------------------------------------------
struct PagedPiece {
  int b, h;         // sequence, item
  int row0, row1;   // rows of it
  long long item0, item1;  // the whole item's units on the line
  long long unit;   // the piece's first unit
};

struct PagedShare {
  const int *lens;
  const PagedPool *pool;
  long long at, end;   // units left to this workgroup
  long long base;      // first unit of sequence b
  unsigned long long per, rest;
  int b, items, tile, len, n;  // n: units of an item of sequence b
  unsigned wg;

  // The workgroup that has unit t.
  __device__ unsigned wg_of(unsigned long long t) const {
    const unsigned long long big = rest * (per + 1);
    if (t < big) return (unsigned)div(t, per + 1);
    return (unsigned)(rest + div(t - big, per));
  }
  __device__ static unsigned long long div(unsigned long long x, unsigned long long y) {
    return (x | y) >> 32 ? x / y : (unsigned)x / (unsigned)y;
  }
  __device__ bool next(PagedPiece &p) {
    if (at >= end) return false;
    while (at >= base + (long long)items * n) {
      base += (long long)items * n;
      ++b;
      len = paged_len(lens[b], *pool);
      n = (len + tile - 1) / tile;  // len + tile is in range: the host bounds len
    }
    p.b = b;
    p.h = (int)div((unsigned long long)(at - base), (unsigned)n);
    p.item0 = base + (long long)p.h * n;
    p.item1 = p.item0 + n;
    p.unit = at;
    const long long to = p.item1 < end ? p.item1 : end;
    p.row0 = (int)(at - p.item0) * tile;
    const long long r1 = (to - p.item0) * tile;
    p.row1 = r1 < len ? (int)r1 : len;
    at = to;
    return true;
  }
};

// Sum over the wave's lanes; inclusive sums of its lanes.
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const unsigned u = __shfl_up(v, o);
    if (lane >= o) v += u;
  }
  return v;
}

__device__ __forceinline__ PagedShare paged_share(const int *lens, int batch, int items,
                                                  const PagedPool &pool, int tile, unsigned wg,
                                                  unsigned wgs) {
  const int lane = threadIdx.x & 63;
  // Units of an item of each sequence, 64 sequences at a time.  A wave's sum
  // of them fits 32 bits: a sequence has under 2^31 rows, a tile 64 or more.
  auto units = [&](int b) -> unsigned {
    return b < batch ? ((unsigned)paged_len(lens[b], pool) + tile - 1) / tile : 0u;
  };
  const unsigned first = wave_scan(units(lane));
  unsigned long long total = (unsigned)__builtin_amdgcn_readlane((int)first, 63);
  for (int b0 = 64; b0 < batch; b0 += 64)
    total += (unsigned)__builtin_amdgcn_readlane((int)wave_scan(units(b0 + lane)), 63);
  total *= (unsigned)items;
  PagedShare s;
  s.lens = lens;
  s.pool = &pool;
  s.per = PagedShare::div(total, wgs);
  s.rest = total - s.per * wgs;
  s.wg = wg;
  s.items = items;
  s.tile = tile;
  s.at = (long long)(wg * s.per + (wg < s.rest ? wg : s.rest));
  s.end = s.at + (long long)(s.per + (wg < s.rest ? 1 : 0));
  s.base = 0;
  s.b = 0;
  s.n = 0;
  s.len = 0;
  if (s.at >= s.end) return s;
  // The sequence that has unit `at`.
  const unsigned long long want = PagedShare::div((unsigned long long)s.at, (unsigned)items);
  unsigned long long before = 0;
  unsigned incl = first;
  for (int b0 = 0;; b0 += 64) {
    if (b0) incl = wave_scan(units(b0 + lane));
    const unsigned sum = (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
    if (want < before + sum) {
      const int k = __builtin_ctzll(__ballot(before + incl > want));
      s.b = b0 + k;
      before += k ? (unsigned)__builtin_amdgcn_readlane((int)incl, k - 1) : 0u;
      break;
    }
    before += sum;
  }
  s.base = (long long)(before * (unsigned)items);
  s.len = paged_len(lens[s.b], pool);
  s.n = (s.len + tile - 1) / tile;
  return s;
}

// A sequence without a row has no unit on the line; its outputs are zeros.
__device__ __forceinline__ void paged_empty(const PagedDecodeArgs &a) {
  for (int b = (int)blockIdx.x; b < a.batch; b += a.wgs) {
    if (a.lens[b] > 0) continue;
    float *out = a.out + (long long)b * a.n_heads * a.pool.d;
    for (int e = (int)threadIdx.x; e < a.n_heads * a.pool.d; e += (int)blockDim.x) out[e] = 0.f;
  }
}

// ---------------------------------------------------------------------------
// The end of a piece.  The workgroup's waves have left their states in LDS:
// for each of `heads` query heads a maximum, a sum and d unnormalised outputs
// (wave w, head g at o[(w * heads + g) * o_stride]).  A piece that is a whole
// item is normalised and written.  Otherwise it goes to the launch's
// workspace; the last workgroup to bring a piece of the item joins all of
// them, in the line's order, so the same inputs give the same bits.
// ---------------------------------------------------------------------------
constexpr int kJoin = 32;      // pieces joined at a time
constexpr int kJoinHeads = 16;  // heads of an item at most
struct JoinShared {
  float m[kJoinHeads], l[kJoinHeads];
  float w[kJoin][kJoinHeads];
  int last;
};

// exp2(m - top), 0 for a state without a row (whose m is -inf).
__device__ __forceinline__ float join_weight(float m, float top) {
  return m == -INFINITY ? 0.f : fast_exp2(m - top);
}

template <int W>
__device__ void paged_finish(const PagedDecodeArgs &a, const PagedPiece &p, const PagedShare &sh,
                             const float *o, int o_stride, const float *wm, const float *wl,
                             int heads, JoinShared &js) {
  const int tid = threadIdx.x, nt = W * 64, d = a.pool.d;
  const unsigned w0 = sh.wg_of((unsigned long long)p.item0);
  const unsigned w1 = sh.wg_of((unsigned long long)(p.item1 - 1));
  const bool whole = w0 == w1;
  float *part = a.parts + (size_t)(2 * sh.wg + (sh.wg == w0 ? 1 : 0)) * a.part_floats;
  float *out = a.out + ((long long)p.b * a.n_heads + (long long)p.h * heads) * d;
  if (tid < heads) {
    float m = -INFINITY, l = 0.f;
    for (int w = 0; w < W; ++w) m = fmaxf(m, wm[w * heads + tid]);
    for (int w = 0; w < W; ++w) {
      const float f = join_weight(wm[w * heads + tid], m);
      js.w[w][tid] = f;
      l = fmaf(f, wl[w * heads + tid], l);
    }
    js.m[tid] = m;
    js.l[tid] = l;
    if (!whole) {
      st_agent(part + heads * d + 2 * tid, m);
      st_agent(part + heads * d + 2 * tid + 1, l);
    }
  }
  __syncthreads();
  for (int e = tid; e < heads * d; e += nt) {
    const int g = e / d, x = e - g * d;
    float s = 0.f;
    for (int w = 0; w < W; ++w) s = fmaf(js.w[w][g], o[(w * heads + g) * o_stride + x], s);
    if (whole)
      out[e] = js.l[g] == 0.f ? 0.f : s / js.l[g];
    else
      st_agent(part + e, s);
  }
  if (whole) return;
  // every store of the workgroup is at the device's coherence point before its ticket
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  unsigned *ticket = a.tickets + (size_t)p.b * (a.n_heads / heads) + p.h;
  const unsigned n = w1 - w0 + 1;
  if (tid == 0)
    js.last = __hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == n - 1;
  __syncthreads();
  if (!js.last) return;
  if (tid == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // piece i of the item: the first is its workgroup's last piece, the others their workgroups' first
  auto piece = [&](unsigned i) {
    return a.parts + (size_t)(2 * (w0 + i) + (i == 0 ? 1 : 0)) * a.part_floats;
  };
  const int wave = tid >> 6, lane = tid & 63;
  for (int g = wave; g < heads; g += W) {
    float m = -INFINITY;
    for (unsigned i = lane; i < n; i += 64) m = fmaxf(m, ld_agent(piece(i) + heads * d + 2 * g));
    m = wave_max(m);
    float l = 0.f;
    for (unsigned i = lane; i < n; i += 64)
      l = fmaf(join_weight(ld_agent(piece(i) + heads * d + 2 * g), m),
               ld_agent(piece(i) + heads * d + 2 * g + 1), l);
    l = wave_sum(l);
    if (lane == 0) {
      js.m[g] = m;
      js.l[g] = l;
    }
  }
  for (int e0 = 0; e0 < heads * d; e0 += nt) {
    const int e = e0 + tid, g = e / d;
    float s = 0.f;
    for (unsigned i0 = 0; i0 < n; i0 += kJoin) {
      const int c = (int)(n - i0 < kJoin ? n - i0 : kJoin);
      __syncthreads();
      for (int k = tid; k < c * heads; k += nt) {
        const int i = k / heads, hg = k - i * heads;
        js.w[i][hg] = join_weight(ld_agent(piece(i0 + i) + heads * d + 2 * hg), js.m[hg]);
      }
      __syncthreads();
      if (e < heads * d)
#pragma unroll 4
        for (int i = 0; i < c; ++i) s = fmaf(js.w[i][g], ld_agent(piece(i0 + i) + e), s);
    }
    if (e < heads * d) out[e] = js.l[g] == 0.f ? 0.f : s / js.l[g];
  }
  __syncthreads();
}

}  // namespace bnr

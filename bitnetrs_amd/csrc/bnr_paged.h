// bnr_paged.h -- device code shared by the paged KV cache's kernels: the four
// row formats, and how a decode launch's pieces are joined.  Included by the
// .hip sources only.
#pragma once

#include "bnr_device.h"
#include "bnr_paged_index.h"

#include <type_traits>

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

// |x| as an integer: ordered as the magnitudes are, infinity and NaN on top, so
// that one maximum finds a row's largest value and whether all are finite.
__device__ __forceinline__ unsigned magnitude(float x) {
  return __builtin_bit_cast(unsigned, x) & 0x7fffffffu;
}

struct RowScale {
  float scale, inv;
};
template <int F>
__device__ __forceinline__ RowScale row_scale(unsigned largest) {
  const float m = fmaxf(__builtin_bit_cast(float, largest), kPagedTiny);
  return largest < 0x7f800000u ? RowScale{m / kPagedTop<F>, kPagedTop<F> / m}
                               : RowScale{__builtin_nanf(""), 0.f};
}

// bf16 bits of x, rounded to nearest even; a NaN stays one.
__device__ __forceinline__ unsigned bf16_bits(float x) {
  return __builtin_bit_cast(unsigned short, (__bf16)x);
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
// FP4: the codes of 32 neighbouring elements of a row (the last group of a row
// may have fewer) are e2m1, 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign, times one
// power of two, kept as its exponent + 127 in a byte.  With m = max(max|x|,
// 2^-100) of the group the power is the one that leaves 3.5 <= m / 2^e < 7, at
// most 2^125: one that leaves 4 <= m / 2^e < 8 cuts values between 7 and 8 by up
// to 2, this one leaves every error at or under half a step and 1 at the top (6
// to 7).  x / 2^e is exact, so a code is one rounding, to nearest, ties to the
// even code.  A group with an infinity or a NaN gets the exponent 255, which
// reads back as NaN, and codes 0.
// ---------------------------------------------------------------------------
constexpr unsigned kPagedNan4 = 255, kPagedTop4 = 252;

__device__ __forceinline__ unsigned exponent4(unsigned largest) {
  const unsigned tiny = __builtin_bit_cast(unsigned, kPagedTiny);
  if (largest >= 0x7f800000u) return kPagedNan4;
  const unsigned m = largest > tiny ? largest : tiny;
  // a mantissa of 1.75 and more carries into the exponent
  const unsigned e = ((m + 0x200000u) >> 23) - 2;
  return e < kPagedTop4 ? e : kPagedTop4;
}
// The power as the conversions take it: NaN for 255.
__device__ __forceinline__ float power4(unsigned e) { return __builtin_bit_cast(float, e << 23); }

// Eight elements as codes, the first in the lowest bits.
__device__ __forceinline__ unsigned codes4(float4 lo, float4 hi, unsigned e) {
  if (e == kPagedNan4) return 0u;
  const float p = power4(e);
  unsigned w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, lo.x, lo.y, p, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, lo.z, lo.w, p, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, hi.x, hi.y, p, 2);
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, hi.z, hi.w, p, 3);
}

// The two elements of byte I of w, as bf16, which holds all of them exactly.
template <int I>
__device__ __forceinline__ unsigned pair4(unsigned w, float power) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, I));
}
__device__ __forceinline__ float low16(unsigned w) { return __builtin_bit_cast(float, w << 16); }
__device__ __forceinline__ float high16(unsigned w) { return __builtin_bit_cast(float, w & 0xffff0000u); }

// Element x of row `at` of a pool, before a row's scale.
template <int F>
__device__ __forceinline__ float load_element(const void *codes, const unsigned char *exps, long long at, int d,
                                              int x) {
  if constexpr (F == kPagedFp4) {
    const unsigned w = static_cast<const unsigned char *>(codes)[at * (d / 2) + x / 2];
    const unsigned p = pair4<0>(w, power4(exps[at * paged_groups4(d) + x / kPagedGroup4]));
    return x & 1 ? high16(p) : low16(p);
  } else {
    return load_code<F>(codes, at * d + x);
  }
}

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ unsigned wave_scan(unsigned v) {
#define BNR_SCAN(CTRL, ROWS) \
  v += (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false)
  BNR_SCAN(0x111, 0xF);  // row_shr:1, 2, 4, 8: sums within each row of 16 lanes
  BNR_SCAN(0x112, 0xF);
  BNR_SCAN(0x114, 0xF);
  BNR_SCAN(0x118, 0xF);
  BNR_SCAN(0x142, 0xA);  // row_bcast:15 into rows 1 and 3
  BNR_SCAN(0x143, 0xC);  // row_bcast:31 into rows 2 and 3
#undef BNR_SCAN
  return v;
}

__device__ __forceinline__ unsigned lane_of(unsigned v, int lane) {
  return (unsigned)__builtin_amdgcn_readlane((int)v, lane);
}

template <class Rows>
__device__ __forceinline__ PagedShare paged_share(Rows rows, int batch, int items, unsigned tile,
                                                  unsigned wgs) {
  const int lane = threadIdx.x & 63;
  // Rows, and units of an item, of each sequence, 64 sequences at a time.
  auto length = [&](int b) { return b < batch ? rows(b) : 0; };
  auto units = [&](int len) { return ((unsigned)len + tile - 1) / tile; };
  const int first_len = length(lane);
  const unsigned first = wave_scan(units(first_len));
  unsigned total = lane_of(first, 63);
  for (int b0 = 64; b0 < batch; b0 += 64) total += lane_of(wave_scan(units(length(b0 + lane))), 63);
  total *= (unsigned)items;
  PagedShare s;
  s.take(total, blockIdx.x, wgs, batch, items, tile);
  if (s.at >= s.end) return s;
  // The sequence that has unit `at`, and the item of it.
  const unsigned want = s.at / (unsigned)items;
  unsigned before = 0, incl = first;
  int len = first_len;
  for (int b0 = 0;; b0 += 64) {
    if (b0) {
      len = length(b0 + lane);
      incl = wave_scan(units(len));
    }
    const unsigned sum = lane_of(incl, 63);
    if (want < before + sum) {
      const int k = __builtin_ctzll(__ballot(before + incl > want));
      const unsigned lo = k ? lane_of(incl, k - 1) : 0u;
      s.b = b0 + k;
      s.n = lane_of(incl, k) - lo;
      s.len = (int)lane_of((unsigned)len, k);
      before += lo;
      break;
    }
    before += sum;
    if (b0 + 64 >= batch) {  // not reached: `at` is less than the sum of all units
      s.end = s.at;
      return s;
    }
  }
  s.h = (int)((s.at - before * (unsigned)items) / s.n);
  s.item0 = before * (unsigned)items + (unsigned)s.h * s.n;
  return s;
}

// A sequence without a row has no unit on the line; its outputs are zeros.
// Workgroup w sees to sequences w, w + wgs, ...; first_len: lens[w], loaded at
// the kernel's start so that its end does not wait for it (1 past the batch).
__device__ __forceinline__ int paged_first_len(const PagedDecodeArgs &a) {
  return (int)blockIdx.x < a.batch ? a.lens[blockIdx.x] : 1;
}
__device__ __forceinline__ void paged_empty(const PagedDecodeArgs &a, int first_len) {
  for (int b = (int)blockIdx.x; b < a.batch; b += a.wgs) {
    if ((b == (int)blockIdx.x ? first_len : a.lens[b]) > 0) continue;
    float *out = a.out + (long long)b * a.n_heads * a.pool.d;
    for (int e = (int)threadIdx.x; e < a.n_heads * a.pool.d; e += (int)blockDim.x) out[e] = 0.f;
  }
}

// ---------------------------------------------------------------------------
// The end of a piece.  The workgroup's waves have left their states in LDS:
// for each of `heads` query heads a maximum, a sum (wm, wl: [wave][head]) and
// d unnormalised outputs (get(w, g, x, o): V of them from x on).  A piece that is a whole
// item is normalised and written.  Otherwise it goes to the launch's
// workspace; the last workgroup to bring a piece of the item joins all of
// them, in the line's order, so the same inputs give the same bits.  Many
// pieces are joined in groups first (JoinStep): the groups by several
// workgroups at a time, then their states by one.
//
// What a join costs is latency: a store, a ticket and a load, each to the
// device's coherence point and back.  So the loads of N pieces are all in
// flight before the first is used, and nothing else waits for memory.
// ---------------------------------------------------------------------------
template <int W, int V>
struct JoinShared {
  float o[W * 64][V], m[W * 64], l[W * 64];
  int last;
};

// A running maximum as something to subtract: 0 while there is no row, so that
// exp2 of what it is subtracted from (-inf) is 0.
__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.f : m; }

// A state of one head and V outputs.
template <int V>
struct JoinState {
  float m, l, o[V];
  // N more states.
  template <int N>
  __device__ __forceinline__ void add(const float (&m2)[N], const float (&l2)[N], const float (&o2)[N][V]) {
    float top = m;
#pragma unroll
    for (int k = 0; k < N; ++k) top = fmaxf(top, m2[k]);
    const float mu = above(top), f = fast_exp2(m - mu);
    m = top;
    l *= f;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] *= f;
#pragma unroll
    for (int k = 0; k < N; ++k) {
      const float w = fast_exp2(m2[k] - mu);
      l = fmaf(l2[k], w, l);
#pragma unroll
      for (int i = 0; i < V; ++i) o[i] = fmaf(o2[k][i], w, o[i]);
    }
  }
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.f;
  }
  // l is 0 only where no row has a weight, else near 1 or more
  __device__ __forceinline__ void write(float *out) const {
    const float r = l == 0.f ? 0.f : 1.0f / l;
    if constexpr (V == 4)
      st4(out, make_float4(o[0] * r, o[1] * r, o[2] * r, o[3] * r));
    else
      out[0] = o[0] * r;
  }
};

// V: outputs of a thread, 4 where d is a multiple of 4 and out is 16-byte
// aligned, or 1.  D: d rounded up to a power of two; w0, w1: the first and the
// last workgroup of the item; N: pieces in flight in a thread.
template <int W, int V, int D, int N, class Get>
__device__ __forceinline__ void paged_finish(const PagedDecodeArgs &a, const PagedPiece &p, unsigned wg,
                                             unsigned w0, unsigned w1, Get get, const float *wm,
                                             const float *wl, int heads, JoinShared<W, V> &js) {
  constexpr int nt = W * 64, per = D / V;
  const int tid = threadIdx.x, d = a.pool.d, work = heads * per;
  const bool whole = w0 == w1;
  float *out = a.out + ((long long)p.b * a.n_heads + (long long)p.h * heads) * d;
  const __amdgpu_buffer_rsrc_t parts = agent_buf(a.parts);
  const int stride = a.part_floats * 4;
  const int mine = (int)(2 * wg + (wg == w0 ? 1 : 0)) * stride;
  for (int e = tid; e < work; e += nt) {
    const int g = e / per, x = e % per * V;
    if (x >= d) continue;
    JoinState<V> s;
    s.clear();
    float m[W], l[W], ow[W][V];
#pragma unroll
    for (int w = 0; w < W; ++w) {
      m[w] = wm[w * heads + g];
      l[w] = wl[w * heads + g];
      get(w, g, x, ow[w]);
    }
    s.add(m, l, ow);
    if (whole) {
      s.write(out + g * d + x);
    } else {
      if constexpr (V == 4)
        st4_agent(parts, mine + (g * d + x) * 4, make_float4(s.o[0], s.o[1], s.o[2], s.o[3]));
      else
        st_agent(a.parts + mine / 4 + g * d + x, s.o[0]);
      if (x == 0) st2_agent(parts, mine + (heads * d + 2 * g) * 4, s.m, s.l);
    }
  }
  if (whole) return;
  // `ways` threads share the pieces of one output; thread k of them takes
  // pieces k, k + ways, ...
  const int ways = work >= nt ? 1 : nt / work;
  const int region = 2 * kPagedMaxWgs * stride;  // bytes of all pieces; the groups' states lie behind them
  JoinStep c = join_start(w0, w1, wg, N * ways, (work + nt - 1) / nt);
  for (int from = 0;; from = region) {
    // every store of the workgroup is at the device's coherence point before its ticket
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    unsigned *ticket = a.tickets + c.ticket(w0) * kCounterStride;
    if (tid == 0)
      js.last = (int)__hip_atomic_fetch_add(ticket, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == c.count - 1;
    __syncthreads();
    if (!js.last) return;
    if (tid == 0) __hip_atomic_store(ticket, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    for (int e0 = 0; e0 < work; e0 += nt) {
      const int way = work >= nt ? 0 : tid / work, e = work >= nt ? e0 + tid : tid - way * work;
      const int g = e / per, x = e % per * V;
      const bool in = way < ways && e < work && x < d;
      JoinState<V> s;
      s.clear();
      const auto take = [&](auto at_once) {
        constexpr int M = decltype(at_once)::value;
        for (int i0 = way; in && i0 < c.count; i0 += M * ways) {
          float m[M], l[M], po[M][V];
#pragma unroll
          for (int k = 0; k < M; ++k) {
            // past the last piece: the last again, without a weight (a branch would part the loads)
            const int i = i0 + k * ways < c.count ? i0 + k * ways : c.count - 1;
            const int at = c.slot(i, w0) * stride + from;
            const float2 ml = ld2_agent(parts, at + (heads * d + 2 * g) * 4);
            m[k] = ml.x;
            l[k] = ml.y;
            if constexpr (V == 4) {
              const float4 v = ld4_agent(parts, at + (g * d + x) * 4);
              po[k][0] = v.x, po[k][1] = v.y, po[k][2] = v.z, po[k][3] = v.w;
            } else {
              po[k][0] = ld_agent(a.parts + at / 4 + g * d + x);
            }
          }
#pragma unroll
          for (int k = 0; k < M; ++k) {
            const bool there = i0 + k * ways < c.count;
            m[k] = there ? m[k] : -INFINITY;
            l[k] = there ? l[k] : 0.f;
#pragma unroll
            for (int j = 0; j < V; ++j) po[k][j] = there ? po[k][j] : 0.f;
          }
          s.add(m, l, po);
        }
      };
      // few pieces: no loads for the places of more (8 sequences of 100 to 900 int8 rows 8.7 -> 7.9 us)
      if (c.count <= 4 * ways)
        take(std::integral_constant<int, 4>{});
      else
        take(std::integral_constant<int, N>{});
      if (ways > 1) {  // work < nt: one round
        js.m[tid] = s.m;
        js.l[tid] = s.l;
#pragma unroll
        for (int i = 0; i < V; ++i) js.o[tid][i] = s.o[i];
        __syncthreads();
        if (way == 0)
          for (int k = 1; k < ways; ++k) {
            const int at = tid + k * work;
            const float m[1] = {js.m[at]}, l[1] = {js.l[at]};
            float po[1][V];
#pragma unroll
            for (int i = 0; i < V; ++i) po[0][i] = js.o[at][i];
            s.add(m, l, po);
          }
      }
      if (way == 0 && in) {
        if (c.last) {
          s.write(out + g * d + x);
        } else {
          const int to = c.slot(0, w0) * stride + region;
          if constexpr (V == 4)
            st4_agent(parts, to + (g * d + x) * 4, make_float4(s.o[0], s.o[1], s.o[2], s.o[3]));
          else
            st_agent(a.parts + to / 4 + g * d + x, s.o[0]);
          if (x == 0) st2_agent(parts, to + (heads * d + 2 * g) * 4, s.m, s.l);
        }
      }
    }
    if (c.last) return;
    c = join_groups(w0, w1);
  }
}

}  // namespace bnr

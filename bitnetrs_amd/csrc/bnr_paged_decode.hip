// bnr_paged_decode.hip -- gfx950 decode attention over a paged KV cache on the
// matrix cores.
//
// An item is one (sequence, kv head): its G <= 16 query heads share one read
// of each row.  A wave takes 32 rows at a time; K, V, the scores and the weights
// stay in its registers.  The query operands, the same for the workgroup's
// waves, are read from LDS in each step.
//
//   S  = K q^T   A = 16 rows of K, B = the query heads as 16 columns
//   O += V^T P   A = 16 dims of V, B = the weights of 32 rows
//
// K's rows are operand A as they lie in memory (a lane holds 16 bytes of one
// row).  D of the first product has a lane hold 4 rows of each 16-row tile
// for one head, which is how the second product wants its B, for the row
// order (tile, lane group, 4 rows) within the step.  V's A operand then needs
// one element of 8 rows from each lane: a lane reads E neighbouring elements
// of its 8 rows, and output dim E * i + m belongs to row i of product m, so
// the transposition is inside the lane (byte permutes, or the conversion that
// the 8-bit formats need anyway).  More than 16 bytes of a row (E = u * U) are
// u units of 16, each over the 16 lanes' neighbouring bytes: dim 16 U unit +
// U i + m.
//
// Precision.  f32 rows multiply on the f32 matrix cores.  bf16, e4m3 and
// int8 codes are exact in bf16; q and the weights are cut into three bf16
// parts of 8 bits each, which together hold all 24 bits of an fp32 value, and
// every part has fp32's exponent range: the products are those of fp32, at a
// third of the bf16 rate, which is far above what the rows' bytes need.  Their
// sum within an instruction keeps 2^-24 of its largest operand and is cut
// there, not rounded to nearest (2 - 2^-69 beside a product of 4 came out as
// 2 - 2^-22); outputs end up 3e-7 to 5e-7 of their norm from 64 bits.  A row's
// scale multiplies its score and its weight in fp32.
//
// Bound by the rows' bytes once there are many: with the products taken out
// the loads alone take 96 to 97 % of the time of 64 int8 sequences of up to
// 32768 rows (231 to 238 us, 6.1 TB/s; a plain read of this card 7.1).  A short
// call is latency: lengths, table and rows one after the other (3.5 us), a step,
// then a store, a ticket and a load to join the pieces (3.5 us); 9.1 us over 4096
// bf16 rows, 5.3 where nothing is joined.  Of the vector instructions of an
// int8 step, 365 of a wave, half turn codes into bf16.
#include "bnr_paged_mfma.h"

#include <type_traits>

namespace bnr {
namespace {

constexpr int kW = 4;  // waves of a workgroup
constexpr int kStep = 32;  // rows of a wave's step

template <int F>
constexpr int kBytes = F == kPagedF32 ? 4 : F == kPagedBf16 ? 2 : 1;

// Waves of a SIMD that the registers are shared out for.  With three the join's
// loads spill: one token over 4096 bf16 rows took 12.6 us.
template <int F, int DP>
constexpr int kWavesOf = paged_waves(F, DP);

// Code i (0..3) of a dword of 8-bit codes, as a float.
template <int F, int I>
__device__ __forceinline__ float code8(unsigned w) {
  if constexpr (F == kPagedInt8) return (float)(signed char)(w >> (8 * I));
  return __builtin_amdgcn_cvt_pk_f32_fp8((int)w, I >= 2)[I & 1];
}

// 8 codes (two dwords) as bf16.
template <int F>
__device__ __forceinline__ u32x4 widen8(unsigned a, unsigned b) {
  u32x4 r;
  if constexpr (F == kPagedFp8) {  // two codes an instruction
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
    r[2] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
    r[3] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
    return r;
  }
  r[0] = pack_hi(code8<F, 0>(a), code8<F, 1>(a));
  r[1] = pack_hi(code8<F, 2>(a), code8<F, 3>(a));
  r[2] = pack_hi(code8<F, 0>(b), code8<F, 1>(b));
  r[3] = pack_hi(code8<F, 2>(b), code8<F, 3>(b));
  return r;
}

// The query heads as operands of the first product, in LDS for the whole
// workgroup: chunk c of a lane's operand is at q[c * 64 + lane].
// f32: four of the lane's floats; else eight dims as bf16, chunk (c, part).
template <int F, int DP>
constexpr int kQChunks = F == kPagedF32 ? DP / 16 : DP / 32 * 3;

// One workgroup's share of the line; waves take steps of kStep rows in turn.
// DP: head dim, rounded up to 64, 128 or 256; FULL: head dim is DP.
template <int F, int DP, bool FULL>
__global__ __launch_bounds__(64 * kW, (kWavesOf<F, DP>)) void paged_decode_kernel(PagedDecodeArgs a) {
  constexpr int B = kBytes<F>;
  constexpr int E = DP / 16;        // dims of a lane and V row
  constexpr int KW = DP * B / 64;   // 16-byte loads of a lane and K tile
  constexpr int VW = E * B / 4;     // dwords of a lane and V row
  constexpr int U = E * B > 16 ? 16 / B : E, VU = E / U;  // dims of a unit, units
  constexpr int QN = kQChunks<F, DP>;
  // outputs of the waves, four dims at a time: [kW][E][4 group + 1], lane (g, row) of quad q at
  // q * (4 group + 1) + g * group + row, which is free of bank conflicts both ways
  extern __shared__ f32x4 s_o[];
  __shared__ u32x4 s_q[QN * 64];
  __shared__ float s_m[kW * kPagedMaxGroup], s_l[kW * kPagedMaxGroup];
  __shared__ JoinShared<kW, 4> s_join;
  const int lane = threadIdx.x & 63, d = FULL ? DP : a.pool.d, G = a.group;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  const int page = a.pool.page, page_shift = page & (page - 1) ? -1 : __builtin_ctz(page);
  const unsigned row_bytes = (unsigned)d * B;
  const unsigned k_off = row * row_bytes + 16 * g;
  const unsigned v_off = 4 * g * row_bytes + row * (U * B);
  const int first_len = paged_first_len(a);
  const auto rows = [&](int b) { return paged_len(a.lens[b], a.pool); };
  PagedShare sh = paged_share(rows, a.batch, a.pool.n_kv, a.tile, a.wgs);

  for (PagedPiece p; sh.next(rows, p);) {
    const int row1 = __builtin_amdgcn_readfirstlane(p.row1);
    const int hk = __builtin_amdgcn_readfirstlane(p.h);
    const int bs = __builtin_amdgcn_readfirstlane(p.b);
    const int *table = a.pool.table + (long long)bs * a.pool.table_stride;
    int t = __builtin_amdgcn_readfirstlane(p.row0) + kStep * wave;

    // Where the 16-row tiles of the wave's next 32 steps lie, lane 2 i + h tile
    // h of step i: one load for all of them.  The page, -1 past the piece or
    // where it is not there; and the tile's row in it.
    int pages, rows_in, step = 0;
    auto load_pages = [&](int t0) {
      const int at = t0 + (lane >> 1) * (kW * kStep) + (lane & 1) * 16;
      const int i = page_shift >= 0 ? at >> page_shift : at / page;
      const int pg = at < row1 ? table[i] : -1;
      pages = (unsigned)pg < (unsigned)a.pool.n_pages ? pg : -1;
      rows_in = at - i * page;
    };
    load_pages(t);

    // The wave's chunks of the query heads: the dims that a lane's K bytes
    // hold, 16 bytes at 64 c + 16 g of the row.
    constexpr int QL = F == kPagedF32 ? QN : QN / 3, QC = (QL + kW - 1) / kW;
    float4 qx[QC][F == kPagedF32 ? 1 : 2];
#pragma unroll
    for (int i = 0; i < QC; ++i) {
      const int c = wave + i * kW;
      const float *q = a.q + ((long long)bs * a.n_heads + (long long)hk * G + row) * d;
      const int e0 = F == kPagedF32    ? 16 * c + 4 * g
                     : F == kPagedBf16 ? 32 * c + 8 * g
                                       : 64 * (c >> 1) + 16 * g + 8 * (c & 1);
      const bool in = c < QL && row < G && (FULL || e0 < d);
#pragma unroll
      for (int k = 0; k < (F == kPagedF32 ? 1 : 2); ++k)
        qx[i][k] = in ? ld4(q + e0 + 4 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
    }

    float m = -INFINITY, l = 0.f;  // of head `row`; l over this lane's rows only
    f32x4 o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    unsigned kr[2][KW * 4], vr[2][4][VW];
    f32x4 ks[2], vs[2];
    // First row in the pool of the tile at row `in` of page pg, page 0's first where there is none.
    auto tile_row = [&](int pg, int in) {
      return ((long long)(pg < 0 ? 0 : pg) * a.pool.n_kv + hk) * page + (pg < 0 ? 0 : in);
    };
    auto load_k = [&](const int (&pg)[2], const int (&in)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long at = tile_row(pg[h], in[h]);
        const char *src = static_cast<const char *>(a.pool.k) + at * row_bytes;
#pragma unroll
        for (int c = 0; c < KW; ++c) {
          unsigned w[4] = {0u, 0u, 0u, 0u};
          if (FULL || (64 * c + 16 * g) / B < d) load_bytes<false>(src + 64 * c + k_off, w);
#pragma unroll
          for (int i = 0; i < 4; ++i) kr[h][4 * c + i] = w[i];
        }
        if (kPagedScaled<F>) ks[h] = *reinterpret_cast<const f32x4 *>(a.pool.k_scales + at + 4 * g);
      }
    };
    auto load_v = [&](const int (&pg)[2], const int (&in)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long at = tile_row(pg[h], in[h]);
        const char *src = static_cast<const char *>(a.pool.v) + at * row_bytes;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
#pragma unroll
          for (int u = 0; u < VU; ++u) {
            unsigned w[VW / VU];
#pragma unroll
            for (int i = 0; i < VW / VU; ++i) w[i] = 0u;
            if (FULL || 16 * U * u + U * row < d) load_bytes<true>(src + r * row_bytes + 16 * U * B * u + v_off, w);
#pragma unroll
            for (int i = 0; i < VW / VU; ++i) vr[h][r][u * (VW / VU) + i] = w[i];
          }
        }
        if (kPagedScaled<F>) vs[h] = *reinterpret_cast<const f32x4 *>(a.pool.v_scales + at + 4 * g);
      }
    };

    // pages of this step's and the next one's tiles, and the latter's rows there
    int pg[2], pn[2], in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      pg[h] = __builtin_amdgcn_readlane(pages, h);
      in[h] = __builtin_amdgcn_readlane(rows_in, h);
      pn[h] = __builtin_amdgcn_readlane(pages, 2 + h);
    }
    if (t < row1) {
      load_k(pg, in);
      load_v(pg, in);
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) in[h] = __builtin_amdgcn_readlane(rows_in, 2 + h);
    // while they are on their way
    __syncthreads();  // the piece before this one has been read
#pragma unroll
    for (int i = 0; i < QC; ++i) {
      const int c = wave + i * kW;
      if (c >= QL) break;
      // scores come out times log2(e) / sqrt(d): their weights are powers of two
      if constexpr (F == kPagedF32) {
        s_q[c * 64 + lane] = __builtin_bit_cast(u32x4, scale4(a.scale_log2, qx[i][0]));
      } else {
        const float4 lo = scale4(a.scale_log2, qx[i][0]), hi = scale4(a.scale_log2, qx[i][1]);
        const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        const Parts s = split8<F == kPagedBf16>(x);  // 8-bit rows hold no infinity
#pragma unroll
        for (int k = 0; k < 3; ++k) s_q[(c * 3 + k) * 64 + lane] = s.p[k];
      }
    }
    const unsigned w0 = sh.wg_of(p.item0), w1 = sh.wg_of(p.item1 - 1);
    __syncthreads();  // the operands

    // One step; `more`: with another behind it, whose loads it issues.  (A
    // branch around them would make every wait one for all loads.)
    const auto one_step = [&](auto more) {
      constexpr bool kMore = decltype(more)::value;
      const int tn = t + kW * kStep;
      // Scores: lane has head `row`, rows 4 g + r of both tiles.  The operands
      // are read again in each step, a chunk ahead of their products: kept in
      // registers they would leave one wave a SIMD.
      f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      int ql = lane;
      asm volatile("" : "+v"(ql));
      constexpr int QP = F == kPagedF32 ? 1 : 3;
      u32x4 qc[QP], qn[QP];
#pragma unroll
      for (int k = 0; k < QP; ++k) qn[k] = s_q[k * 64 + ql];
#pragma unroll
      for (int c = 0; c < QL; ++c) {
#pragma unroll
        for (int k = 0; k < QP; ++k) {
          qc[k] = qn[k];
          if (c + 1 < QL) qn[k] = s_q[((c + 1) * QP + k) * 64 + ql];
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (F == kPagedF32) {
          const f32x4 qf = __builtin_bit_cast(f32x4, qc[0]);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
              s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(
                  __builtin_bit_cast(float, kr[h][4 * c + i]), qf[i], s[h], 0, 0, 0);
        } else {
          u32x4 w[2];
#pragma unroll
          for (int h = 0; h < 2; ++h)
            w[h] = F == kPagedBf16
                       ? u32x4{kr[h][4 * c], kr[h][4 * c + 1], kr[h][4 * c + 2], kr[h][4 * c + 3]}
                       : widen8<F>(kr[h][2 * c], kr[h][2 * c + 1]);
#pragma unroll
          for (int k = 0; k < 3; ++k)
#pragma unroll
            for (int h = 0; h < 2; ++h) s[h] = mfma_bf16(w[h], qc[k], s[h]);
        }
      }
      float x[8];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int r = 0; r < 4; ++r)
          x[4 * h + r] = kPagedScaled<F> ? s[h][r] * ks[h][r] : s[h][r];
      const bool all = pg[0] >= 0 && pg[1] >= 0 && t + kStep <= row1;
      if (!all)
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pg[h] < 0 || t + 16 * h + 4 * g + r >= row1) x[4 * h + r] = -INFINITY;
      // the next step's K goes out while this one's weights are made
      if constexpr (kMore) load_k(pn, in);

      float mx = m;
#pragma unroll
      for (int i = 0; i < 8; ++i) mx = fmaxf(mx, x[i]);
      if (__any(mx > m)) {
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float keep = fast_exp2(m - above(mx));
        m = mx;
        l *= keep;
#pragma unroll
        for (int i = 0; i < E; ++i) o[i] *= keep;
      }
      const float mu = above(m);
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        w[i] = fast_exp2(x[i] - mu);
        l += w[i];
        if (kPagedScaled<F>) w[i] *= vs[i >> 2][i & 3];
      }
      if (!all)  // rows that are not there: no weight, whatever lies in their place
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pg[h] < 0 || t + 16 * h + 4 * g + r >= row1) {
              w[4 * h + r] = 0.f;
#pragma unroll
              for (int i = 0; i < VW; ++i) vr[h][r][i] = 0u;
            }

      if constexpr (F == kPagedF32) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < E; ++i)
              o[i] = __builtin_amdgcn_mfma_f32_16x16x4f32(__builtin_bit_cast(float, vr[h][r][i]),
                                                          w[4 * h + r], o[i], 0, 0, 0);
      } else {
        const Parts wp = split8<false>(w);
#pragma unroll
        for (int i = 0; i < E; ++i) {
          u32x4 c;  // dim i of the lane's 8 rows
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const unsigned lo = vr[k >> 1][2 * (k & 1)][i * B / 4];
            const unsigned hi = vr[k >> 1][2 * (k & 1) + 1][i * B / 4];
            if constexpr (F == kPagedBf16)
              c[k] = __builtin_amdgcn_perm(hi, lo, i & 1 ? 0x07060302u : 0x05040100u);
            else
              c[k] = i % 4 == 0   ? pack_hi(code8<F, 0>(lo), code8<F, 0>(hi))
                     : i % 4 == 1 ? pack_hi(code8<F, 1>(lo), code8<F, 1>(hi))
                     : i % 4 == 2 ? pack_hi(code8<F, 2>(lo), code8<F, 2>(hi))
                                  : pack_hi(code8<F, 3>(lo), code8<F, 3>(hi));
          }
#pragma unroll
          for (int k = 0; k < 3; ++k) o[i] = mfma_bf16(c, wp.p[k], o[i]);
        }
      }
      if constexpr (kMore) {
        load_v(pn, in);
        if (++step == 31) {  // pages of the step after the next
          load_pages(tn + kW * kStep);
          step = -1;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          pg[h] = pn[h];
          pn[h] = __builtin_amdgcn_readlane(pages, 2 * (step + 1) + h);
          in[h] = __builtin_amdgcn_readlane(rows_in, 2 * (step + 1) + h);
        }
        t = tn;
      }
    };
    if (t < row1) {
      while (t + kW * kStep < row1) one_step(std::true_type{});
      one_step(std::false_type{});
    }

    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (row < G) {
      if (g == 0) {
        s_m[wave * G + row] = m;
        s_l[wave * G + row] = l;
      }
      f32x4 *so = s_o + wave * E * (4 * G + 1) + g * G + row;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < E; i += 4)
          so[(r * (E / 4) + i / 4) * (4 * G + 1)] = f32x4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
    }
    __syncthreads();
    const auto get = [&](int w, int hd, int x, float(&to)[4]) {
      const int i = x / (16 * U) * U + x % U, rg = x % (16 * U) / U;  // element of the lane; 4 g + r
      const f32x4 v = s_o[(w * E + (rg & 3) * (E / 4) + i / 4) * (4 * G + 1) + (rg >> 2) * G + hd];
#pragma unroll
      for (int k = 0; k < 4; ++k) to[k] = v[k];
    };
    paged_finish<kW, 4, DP, paged_in_flight(F)>(a, p, sh.wg, w0, w1, get, s_m, s_l, G, s_join);
  }
  paged_empty(a, first_len);
}

template <int F>
hipError_t launch_format(const PagedDecodeArgs &a, hipStream_t s) {
  const int d = a.pool.d;
  const int dp = paged_dim(d);
  const size_t lds = (size_t)kW * (dp / 16) * (4 * a.group + 1) * sizeof(f32x4);
  const dim3 grid((unsigned)a.wgs), block(64 * kW);
  // what a workgroup gets unasked is 64 KB, of which up to 32 are static
  constexpr size_t kUnasked = 32 * 1024;
#define BNR_LAUNCH(DP)                                          \
  {                                                             \
    const auto kernel = d == DP ? paged_decode_kernel<F, DP, true> : paged_decode_kernel<F, DP, false>; \
    if (lds > kUnasked) {                                       \
      const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), \
                                               hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds); \
      if (e != hipSuccess) return e;                            \
    }                                                           \
    kernel<<<grid, block, lds, s>>>(a);                         \
  }
  if (dp == 64) {
    BNR_LAUNCH(64)
  } else if (dp == 128) {
    BNR_LAUNCH(128)
  } else {
    BNR_LAUNCH(256)
  }
#undef BNR_LAUNCH
  return hipGetLastError();
}

}  // namespace

hipError_t launch_paged_decode(const PagedDecodeArgs &a, int format, hipStream_t s) {
  switch (format) {
    case kPagedF32: return launch_format<kPagedF32>(a, s);
    case kPagedBf16: return launch_format<kPagedBf16>(a, s);
    case kPagedFp8: return launch_format<kPagedFp8>(a, s);
    case kPagedInt8: return launch_format<kPagedInt8>(a, s);
    case kPagedFp4: return launch_paged_decode_fp4(a, s);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace bnr

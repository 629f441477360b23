// bnr_paged_fp4.hip -- gfx950 decode attention over a paged KV cache of 4-bit
// rows on the matrix cores.
//
// The products, the split of the work and the joins are those of the other
// formats (bnr_paged_decode.hip): S = K q^T and O += V^T P over 32 rows of a
// wave's step, with q and the weights as three bf16 parts.  What differs is how
// operands come from 4-bit codes:
//
//   K  A lane's 16 bytes of a row (of 128 dims) are 32 neighbouring dims: one
//      group, so one exponent a lane and row, and each of its dwords is the
//      lane's operand of one product, four conversions of two codes.
//   V  A lane has E neighbouring dims of 8 rows, E codes of one group each: the
//      rows are converted with their own exponents, and the pairs of
//      neighbouring dims of two rows become pairs of rows by byte permutes.
//
// The conversion multiplies with the group's power of two, and bf16 holds a
// code times a power exactly: no scale is left for the scores or the weights,
// and a NaN group (exponent 255) comes out as NaN.
//
// With at most four query heads a kv head the three parts of q and of the weights
// are columns 4 part + head of one product instead of three products (64
// sequences of up to 32768 rows, 20/5 heads of 128: 172 -> 150 us; short calls, which
// would pay 0.2 to 0.8 us for adding the columns at a piece's end, keep the
// products).  V's exponents come 16 bytes a
// load there (150 -> 136).
//
// Bound by the rows' bytes where there are many: those 64 sequences take 136 us,
// 5.4 TB/s, their loads alone 124.  254 vector instructions of a wave's step, 64 of
// them conversions.  Loads two steps ahead (148), steps of 64 rows (141; short
// shares lose more) and a third workgroup a CU (137) gained nothing.  A short call
// is latency as in the other formats: 8.8 us over 4096 rows.
#include "bnr_paged_mfma.h"

#include <type_traits>

namespace bnr {
namespace {

constexpr int kW = 4;      // waves of a workgroup
constexpr int kStep = 32;  // rows of a wave's step
constexpr int kOcc = 2;

// Sums over the lanes of a DPP row that hold one head's parts, four lanes apart.
__device__ __forceinline__ float sum_parts(float v) {
  v += dpp<0x128>(v);  // row_ror:8
  return v + dpp<0x124>(v);  // row_ror:4
}

// The power whose exponent is byte (turn - 9) / 8 of w: the conversion reads the
// exponent's bits of its scale only (checked for all codes and exponents with
// every other bit set), so the other bytes may stay.
__device__ __forceinline__ float power_at(unsigned w, unsigned turn) {
  return __builtin_bit_cast(float, __builtin_amdgcn_alignbit(w, w, turn));
}

// DP: head dim, rounded up to 64, 128 or 256; FULL: head dim is DP; PACK: at most
// four heads, the three parts of q and of the weights in columns 4 part + head.
template <int DP, bool FULL, bool PACK>
__global__ __launch_bounds__(64 * kW, kOcc) void paged_decode_fp4_kernel(PagedDecodeArgs a) {
  constexpr int E = DP / 16;               // dims of a lane and V row
  constexpr int KL = DP > 128 ? 2 : 1;     // loads of a lane and K tile
  constexpr int KD = DP / 32 / KL;         // dwords of each: 2 (8 bytes) or 4 (16)
  constexpr int VD = E > 8 ? E / 8 : 1;    // dwords of a lane and V row
  constexpr int QL = DP / 32;              // products of a tile's scores
  // outputs of the waves, as in the other formats' kernel
  extern __shared__ f32x4 s_o[];
  constexpr int QP = PACK ? 1 : 3;         // operands of a product's q and weights
  __shared__ u32x4 s_q[QL * QP * 64];
  __shared__ float s_m[kW * kPagedMaxGroup], s_l[kW * kPagedMaxGroup];
  __shared__ JoinShared<kW, 4> s_join;
  const int lane = threadIdx.x & 63, d = FULL ? DP : a.pool.d, G = a.group;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int row = lane & 15, g = lane >> 4;
  const int head = PACK ? row & 3 : row, part = PACK ? row >> 2 : 0;
  // V's exponents: of 128 dims the four of a row are a dword, and those of a lane's
  // four rows 16 bytes; else a byte each.  How far they turn to the exponent's place.
  constexpr bool kRowExps = FULL && DP == 128;
  const unsigned v_turn = 9 + (kRowExps ? 8 * (row * E / kPagedGroup4) : 0);
  // what a weight loses before its part is cut
  const unsigned cut1 = part >= 1 ? 0xffff0000u : 0u, cut2 = part >= 2 ? 0xffff0000u : 0u;
  const int page = a.pool.page, page_shift = page & (page - 1) ? -1 : __builtin_ctz(page);
  const int groups = paged_groups4(d);
  const unsigned row_bytes = (unsigned)d / 2;
  // the lane's dims of K: KD * 8 of them from KD * 8 * (4 j + g) on, load by load
  const auto k_dim = [&](int j) { return KD * 8 * (4 * j + g); };
  const auto k_in = [&](int j, int i) { return FULL || k_dim(j) + 8 * i < d; };  // dword i's
  // the lane's first dim of V; behind the head's end the first ones again, whose outputs go nowhere
  const int v_dim = FULL || row * E < d ? row * E : 0;
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

    // The wave's chunks of the query heads: the dims of the lane's K dwords.
    constexpr int QC = (QL + kW - 1) / kW;
    float4 qx[QC][2];
#pragma unroll
    for (int i = 0; i < QC; ++i) {
      const int c = wave + i * kW;
      const float *q = a.q + ((long long)bs * a.n_heads + (long long)hk * G + head) * d;
      const int e0 = k_dim(c / KD) + 8 * (c % KD);
      const bool in = c < QL && head < G && (FULL || e0 < d);
#pragma unroll
      for (int k = 0; k < 2; ++k) qx[i][k] = in ? ld4(q + e0 + 4 * k) : make_float4(0.f, 0.f, 0.f, 0.f);
    }

    float m = -INFINITY, l = 0.f;  // of head `row`; l over this lane's rows only
    f32x4 o[E];
#pragma unroll
    for (int i = 0; i < E; ++i) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    unsigned kr[2][QL], vr[2][4][VD];
    unsigned ke[2][KL], ve[2][4];
    // First row in the pool of the tile at row `in` of page pg, page 0's first where there is none.
    auto tile_row = [&](int pg, int in) {
      return ((long long)(pg < 0 ? 0 : pg) * a.pool.n_kv + hk) * page + (pg < 0 ? 0 : in);
    };
    auto load_k = [&](const int (&pg)[2], const int (&in)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long at = tile_row(pg[h], in[h]);
        const char *src = static_cast<const char *>(a.pool.k) + at * row_bytes;
        const unsigned char *exps = a.pool.k_exps + at * groups;
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          unsigned w[KD];
          if constexpr (FULL) {
            load_bytes<true>(src + row * row_bytes + k_dim(j) / 2, w);
          } else {
            // a head dim that is a multiple of 16 ends between two halves of 16 bytes;
            // those behind it read the row's start (a branch would part the loads)
#pragma unroll
            for (int i = 0; i < KD; i += 2) {
              unsigned x[2];
              load_bytes<true>(src + row * row_bytes + (k_in(j, i) ? k_dim(j) / 2 + 4 * i : 0), x);
              w[i] = x[0];
              w[i + 1] = x[1];
            }
          }
#pragma unroll
          for (int i = 0; i < KD; ++i) kr[h][j * KD + i] = w[i];
          ke[h][j] = exps[row * groups + (k_in(j, 0) ? k_dim(j) / kPagedGroup4 : 0)];
        }
      }
    };
    auto load_v = [&](const int (&pg)[2], const int (&in)[2]) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const long long at = tile_row(pg[h], in[h]);
        const char *src = static_cast<const char *>(a.pool.v) + at * row_bytes;
        const unsigned char *exps = a.pool.v_exps + at * groups;
        if constexpr (kRowExps) {
          const u32x4 e = *reinterpret_cast<const u32x4 *>(exps + 16 * g);
#pragma unroll
          for (int r = 0; r < 4; ++r) ve[h][r] = e[r];
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const char *from = src + (4 * g + r) * row_bytes + v_dim / 2;
          if constexpr (E == 4)
            vr[h][r][0] = *reinterpret_cast<const unsigned short *>(from);
          else
            load_bytes<true>(from, vr[h][r]);
          if constexpr (!kRowExps) ve[h][r] = exps[(4 * g + r) * groups + v_dim / kPagedGroup4];
        }
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
      // (the fourth column is added to them too: 2^-40 of q there, for an infinity as in split8)
      const float scale = PACK && part == 3 ? a.scale_log2 * 0x1p-40f : a.scale_log2;
      const float4 lo = scale4(scale, qx[i][0]), hi = scale4(scale, qx[i][1]);
      const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
      const Parts s = split8<true>(x);  // exponents of 253 and 254 make infinities
      if constexpr (PACK) {
        s_q[c * 64 + lane] = part == 1 ? s.p[1] : part == 2 ? s.p[2] : s.p[0];
      } else {
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
      // Scores: lane has one head, rows 4 g + r of both tiles.
      f32x4 s[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
      int ql = lane;
      asm volatile("" : "+v"(ql));
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
        u32x4 w[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const unsigned x = kr[h][c];
          // q is zero behind the head's end; so are these, whatever the row's start holds
          const float e = power4(k_in(c / KD, c % KD) ? ke[h][c / KD] : 0u);
          w[h] = u32x4{pair4<0>(x, e), pair4<1>(x, e), pair4<2>(x, e), pair4<3>(x, e)};
        }
#pragma unroll
        for (int k = 0; k < QP; ++k)
#pragma unroll
          for (int h = 0; h < 2; ++h) s[h] = mfma_bf16(w[h], qc[k], s[h]);
      }
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = PACK ? sum_parts(s[i >> 2][i & 3]) : s[i >> 2][i & 3];
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
      }
      if (!all)  // rows that are not there: no weight, whatever lies in their place
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (pg[h] < 0 || t + 16 * h + 4 * g + r >= row1) {
              w[4 * h + r] = 0.f;
              ve[h][r] = 0u;
#pragma unroll
              for (int i = 0; i < VD; ++i) vr[h][r][i] = 0u;
            }

      Parts wp;
      if constexpr (PACK) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          w[i] -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, w[i]) & cut1);
          w[i] -= __builtin_bit_cast(float, __builtin_bit_cast(unsigned, w[i]) & cut2);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) wp.p[0][i] = pack_hi(w[2 * i], w[2 * i + 1]);
      } else {
        wp = split8<false>(w);
      }
      // four dims of the lane's 8 rows at a time, as pairs of dims of a row first
#pragma unroll
      for (int q = 0; q < E / 4; ++q) {
        unsigned two[8][2];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const unsigned x = vr[i >> 2][i & 3][q / 2];
          const float e = power_at(ve[i >> 2][i & 3], v_turn);
          two[i][0] = q % 2 ? pair4<2>(x, e) : pair4<0>(x, e);
          two[i][1] = q % 2 ? pair4<3>(x, e) : pair4<1>(x, e);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u32x4 c;  // dim 4 q + i of the 8 rows
#pragma unroll
          for (int k = 0; k < 4; ++k)
            c[k] = __builtin_amdgcn_perm(two[2 * k + 1][i / 2], two[2 * k][i / 2],
                                         i & 1 ? 0x07060302u : 0x05040100u);
#pragma unroll
          for (int k = 0; k < QP; ++k) o[4 * q + i] = mfma_bf16(c, wp.p[k], o[4 * q + i]);
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
    if constexpr (PACK) {
#pragma unroll
      for (int i = 0; i < E; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r)  // lanes 0..3 of a row: the parts of their heads
          o[i][r] = (o[i][r] + dpp<0x104>(o[i][r])) + dpp<0x108>(o[i][r]);
    }
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
      const int i = x % E, rg = x / E;  // element of the lane; 4 g + r
      const f32x4 v = s_o[(w * E + (rg & 3) * (E / 4) + i / 4) * (4 * G + 1) + (rg >> 2) * G + hd];
#pragma unroll
      for (int k = 0; k < 4; ++k) to[k] = v[k];
    };
    paged_finish<kW, 4, DP, paged_in_flight(kPagedFp4)>(a, p, sh.wg, w0, w1, get, s_m, s_l, G, s_join);
  }
  paged_empty(a, first_len);
}

template <bool PACK>
auto kernel_of(int d) {
  const int dp = paged_dim(d);
  return dp == 64    ? (d == 64 ? paged_decode_fp4_kernel<64, true, PACK> : paged_decode_fp4_kernel<64, false, PACK>)
         : dp == 128 ? (d == 128 ? paged_decode_fp4_kernel<128, true, PACK> : paged_decode_fp4_kernel<128, false, PACK>)
                     : (d == 256 ? paged_decode_fp4_kernel<256, true, PACK> : paged_decode_fp4_kernel<256, false, PACK>);
}

}  // namespace

hipError_t launch_paged_decode_fp4(const PagedDecodeArgs &a, hipStream_t s) {
  const int d = a.pool.d, dp = paged_dim(d);
  const size_t lds = (size_t)kW * (dp / 16) * (4 * a.group + 1) * sizeof(f32x4);
  const dim3 grid((unsigned)a.wgs), block(64 * kW);
  // what a workgroup gets unasked is 64 KB, of which up to 32 are static
  constexpr size_t kUnasked = 32 * 1024;
  // Columns instead of products pay once a wave has more than two steps or so; what
  // they cost is the adding at a piece's end.  20/5 heads of 128: 4 sequences of 4096
  // rows (640 units) 11.9 us, 11.1 with products, 8 of them (1280) 14.3 and 14.2, 32 of
  // 128 to 4096 21.9 and 22.5; 16 of 2000 of 8/8 heads (2048) 14.3 and 15.0.
  const long long rows = a.pool.table_stride * a.pool.page;
  const long long units = (rows + a.tile - 1) / a.tile * a.batch * a.pool.n_kv;
  const bool pack = a.group <= 4 && units > 2 * kPagedMaxWgs;
  const auto kernel = pack ? kernel_of<true>(d) : kernel_of<false>(d);
  if (lds > kUnasked) {
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void *>(kernel),
                                             hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
    if (e != hipSuccess) return e;
  }
  kernel<<<grid, block, lds, s>>>(a);
  return hipGetLastError();
}

}  // namespace bnr

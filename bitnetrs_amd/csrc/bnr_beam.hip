// bnr_beam.hip -- gfx950 kernels of beam search: of each request's beams the k
// best continuations over the whole vocabulary.
//
//   score(b, t) = scores[b] + logit[b, t] - lse[b],   lse = log sum_t exp(logit)
//
// Within a beam the order is that of the logits, so one pass over them finds
// the sum and the k best: of a workgroup's first logits, in registers, the threads'
// maxima give a threshold that at least k of them reach, and the few that do are
// ranked by counting at the end.  A second launch joins the parts of each row and
// then the beams.
//
// Beams are compared by scores in 64 bits: lse is what the order of two beams'
// continuations hangs on, so its exponentials carry the part of log2(e) that
// fp32 leaves out, and at most 16 of them are added in fp32 before they join a
// sum in 64 bits: lse is within 2^-17 whatever the vocabulary.
//
// Read once, the logits of 16 requests of 8 beams and 128256 tokens (61 MB) take 8.6
// us at the rate of a plain read; the rows' launch takes 16.2, of which 12.0 are
// left without search, candidates and exponentials (its start, the first load and
// the stream), and the join 5.8.  Four beams: 4.8 and 4.3, all latency.
#include "bnr_device.h"

#include <algorithm>

namespace bnr {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kJoinWaves = 16;
constexpr int kJoinEntries = 4096;           // of the lists that LDS has room for
constexpr int kCap = 128;                    // candidates of a wave that LDS has room for
constexpr float kLargest = 3.402823466e38f;  // of fp32
// How far a logit may lie above what a thread's exponentials are taken from.  Each
// factor that raises it costs a sum a place of exp2, so that it does not follow every logit.
constexpr float kSlack = 2.f;

typedef unsigned long long u64;

__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.f : m; }

// exp(x - m): log2(e) in two parts, so that no term has an error of its own sign
// (with one part all terms of a row are off by 1.3e-8 of their exponent).
__device__ __forceinline__ float exp_from(float x, float m) {
  const float d = x - m;
  return fast_exp2(fmaf(d, 1.925963033500e-8f, d * 1.442695021629f));
}

// A beam's continuations as whole numbers in their order, the larger logit first,
// then the lower index; 0 is none (a NaN does not come here; -0 counts as 0).
__device__ __forceinline__ unsigned ordered(float v) {
  const unsigned b = __builtin_bit_cast(unsigned, v + 0.0f);
  return b ^ ((int)b < 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ u64 key_of(float v, int i) { return (u64)ordered(v) << 32 | ~(unsigned)i; }
__device__ __forceinline__ float logit_of(u64 key) {
  const unsigned b = (unsigned)(key >> 32);
  return __builtin_bit_cast(float, b ^ ((int)b < 0 ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int index_of(u64 key) { return (int)~(unsigned)key; }

__device__ __forceinline__ u64 wave_best(u64 x) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const u64 y = __shfl_xor(x, k);
    x = y > x ? y : x;
  }
  return x;
}

// What a wave wrote to LDS is there for its other lanes: LDS works in order, so
// only the compiler has to keep the order.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

__device__ __forceinline__ int lanes_below(u64 mask) {
  return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(mask >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)mask, 0u));
}

template <int CTRL>
__device__ __forceinline__ double dpp64(double v) {
  const u64 b = __builtin_bit_cast(u64, v);
  const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, 0xF, 0xF, false);
  const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, 0xF, 0xF, false);
  return __builtin_bit_cast(double, (u64)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum64(double v) {
  v += dpp64<0xB1>(v);   // quad_perm [1,0,3,2]
  v += dpp64<0x4E>(v);   // quad_perm [2,3,0,1]
  v += dpp64<0x141>(v);  // row_half_mirror
  v += dpp64<0x140>(v);  // row_mirror
  const auto of = [&](int lane) {
    const u64 b = __builtin_bit_cast(u64, v);
    return __builtin_bit_cast(double, (u64)(unsigned)__builtin_amdgcn_readlane((int)(b >> 32), lane) << 32 |
                                          (unsigned)__builtin_amdgcn_readlane((int)(unsigned)b, lane));
  };
  return (of(0) + of(16)) + (of(32) + of(48));
}

// How many of the n keys in LDS are larger than this one: eight at a time, 16
// bytes a load; behind them are zeros up to a multiple of eight.
__device__ __forceinline__ int larger(const u64 *keys, int n, u64 key) {
  int p = 0;
  for (int j = 0; j < n; j += 8) {
    u64 other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = keys[j + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) p += other[i] > key;
  }
  return p;
}

// A workgroup's part of a row, H logits of a thread at a time, the next ones on
// their way meanwhile.  After the first logits, whose threads' maxima give the
// threshold, the waves work by themselves until the end.
template <bool VEC, int H>
__global__ __launch_bounds__(kThreads) void beam_rows_kernel(BeamArgs a) {
  constexpr int kTile = H * kThreads;
  __shared__ __attribute__((aligned(16))) u64 s_cand[kWaves][kCap + 8];
  __shared__ float s_best[kWaves], s_top[kWaves];
  __shared__ int s_have[kWaves];
  __shared__ double s_sum[kWaves];
  const int row = blockIdx.x / (unsigned)a.chunks, part = blockIdx.x - row * a.chunks;
  const bool ended = a.done && a.done[row];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x, k = a.k;
  const float *x = a.logits + row * a.stride;
  const int v0 = part * a.chunk, v1 = min(v0 + a.chunk, a.vocab);
  float m = -INFINITY;  // what exponentials are taken from
  double sum = 0.0;
  u64 *cand = s_cand[wave];
  int have = 0;  // candidates so far, the same in all lanes
  // What a candidate must reach: at least k of the workgroup's do.  Masked tokens (-infinity) are none: the join
  // knows which of them fill up.
  float least = -kLargest;

  // Element n of the thread's logits of the tile at t0.
  const auto index = [&](int t0, int n) {
    return VEC ? t0 + 4 * (tid + kThreads * (n / 4)) + n % 4 : t0 + tid + kThreads * n;
  };
  const auto load = [&](int t0, float (&h)[H]) {
#pragma unroll
    for (int n = 0; n < H; n += VEC ? 4 : 1) {
      const int i = index(t0, n);
      if constexpr (VEC) {  // a part ends at a multiple of 4 or at the row's end
        float4 w = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i + 4 <= v1) {
          w = ld4_nt(x + i);
        } else if (i < v1) {
          w.x = x[i];
          if (i + 1 < v1) w.y = x[i + 1];
          if (i + 2 < v1) w.z = x[i + 2];
        }
        h[n] = w.x, h[n + 1] = w.y, h[n + 2] = w.z, h[n + 3] = w.w;
      } else {
        h[n] = i < v1 ? x[i] : -INFINITY;
      }
    }
  };
  float h[H], next[H];
  if (v0 < v1) load(v0, next);
  if (ended) return;  // the join knows it (asked before the loads, that it be here with them)
  for (int t0 = v0; t0 < v1; t0 += kTile) {
#pragma unroll
    for (int n = 0; n < H; ++n) h[n] = next[n];
    if (t0 + kTile < v1) load(t0 + kTile, next);
    float top = h[0];
#pragma unroll
    for (int n = 1; n < H; ++n) top = fmaxf(top, h[n]);
    if (!(top > -INFINITY)) top = -INFINITY;  // all NaN
    // places past the end hold -infinity: they add nothing
    const bool rise = top > m + kSlack;
    const float mn = rise ? top : m, mu = above(mn), keep = rise ? exp_from(m, mn) : 1.f;
    float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int n = 0; n < H; ++n) add[n % 4] += exp_from(h[n], mu);
    sum = fma(sum, (double)keep, (double)((add[0] + add[1]) + (add[2] + add[3])));
    m = mn;

    // The first tile's threshold: of each wave's lane maxima the n-th largest, n
    // a quarter of k or more, and of these the least.  (The k-th of all 256 leaves
    // half as many candidates and costs four times the rounds.)
    if (t0 == v0) {
      float v = top, nth = -INFINITY;
      for (int r = 0; r < k; r += kWaves) {
        nth = wave_max(v);
        const int first = __builtin_ctzll(__ballot(v == nth));
        if (lane == first) v = -INFINITY;
      }
      if (lane == 0) s_best[wave] = nth;
      __syncthreads();
      nth = s_best[0];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) nth = fminf(nth, s_best[w]);
      least = fmaxf(least, nth);
    }
    if (!__any(top >= least)) continue;
    const int before = have;
#pragma unroll
    for (int n = 0; n < H; ++n) {
      const u64 in = __ballot(h[n] >= least);
      if (in == 0) continue;
      const int at = have + lanes_below(in);
      if (h[n] >= least && at < kCap) cand[at] = key_of(h[n], index(t0, n));
      have += __builtin_popcountll(in);
    }
    if (have <= 64) continue;
    if (have <= kCap) {
      if (lane < 8) cand[have + lane] = 0;
      wave_order();
      const u64 mine[2] = {cand[lane], 64 + lane < have ? cand[64 + lane] : 0};
      const int place[2] = {larger(cand, have, mine[0]), larger(cand, have, mine[1])};
      wave_order();
#pragma unroll
      for (int i = 0; i < 2; ++i)
        if (place[i] < k && mine[i]) cand[place[i]] = mine[i];
      have = k;
    } else {
      // Too many (equal ones, say): the best that is left, k times.  Those of the
      // tiles before, 64 at most, are held by a lane each.
      wave_order();
      const u64 old = lane < before ? cand[lane] : 0;
      wave_order();
      u64 last = ~0ull;
      for (int r = 0; r < k; ++r) {
        u64 best = old < last ? old : 0;
#pragma unroll
        for (int n = 0; n < H; ++n) {
          const u64 key = h[n] >= least ? key_of(h[n], index(t0, n)) : 0;
          best = key < last && key > best ? key : best;
        }
        last = wave_best(best);
        if (lane == 0) cand[r] = last;
      }
      have = k;  // there were more than k
    }
    // the k best so far: later logits have higher indexes, so only the next larger float
    // is a candidate (above the largest, infinity: such a row has no continuation)
    wave_order();
    least = logit_of((cand[k - 1] | 0xffffffffull) + 1);
  }
  // The part's k best: a candidate's place is how many of all waves' are larger.
  const float wm = wave_max(m);
  const double ws = wave_sum64(sum * (double)exp_from(above(m) == m ? m : above(wm), above(wm)));
  if (lane < 8) cand[have + lane] = 0;
  if (lane == 0) {
    s_top[wave] = wm;
    s_sum[wave] = ws;
    s_have[wave] = have;
  }
  __syncthreads();
  const long long at = (long long)row * a.chunks + part;
  const u64 mine = lane < have ? cand[lane] : 0;
  int place = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const int n = s_have[w];
    place += larger(s_cand[w], n, mine);
    all += n;
  }
  if (mine && place < k) a.part_key[at * k + place] = mine;
  if (tid >= all && tid < k) a.part_key[at * k + tid] = 0;
  if (tid != 0) return;
  float top = s_top[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_top[w]);
  double total = 0.0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    total += s_sum[w] * (double)exp_from(above(s_top[w]) == s_top[w] ? s_top[w] : above(top), above(top));
  a.part_max[at] = top;
  a.part_sum[at] = total;
}

__device__ __forceinline__ unsigned wave_umax(unsigned v) {
#define BNR_MAX(CTRL) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xF, 0xF, false))
  BNR_MAX(0xB1);   // quad_perm [1,0,3,2]
  BNR_MAX(0x4E);   // quad_perm [2,3,0,1]
  BNR_MAX(0x141);  // row_half_mirror
  BNR_MAX(0x140);  // row_mirror
#undef BNR_MAX
  const auto of = [&](int lane) { return (unsigned)__builtin_amdgcn_readlane((int)v, lane); };
  return max(max(of(0), of(16)), max(of(32), of(48)));
}

// A double as a whole number of the same order (no NaN comes here; -0 is not made).
__device__ __forceinline__ u64 ordered(double v) {
  const long long b = __builtin_bit_cast(long long, v);
  return (u64)b ^ (u64)(b < 0 ? -1ll : (long long)(1ull << 63));
}

// Joins the parts of each beam's row, and then the request's beams.  Of a beam one
// wave finds the k best, lane c having part c's list and its best that is not
// taken (of equal logits the lowest lane's has the lowest index), while another
// makes lse.  Then a thread has one continuation of one beam, whose place is how
// many come before it: rounds of the wave for these too took 2 us more of 8.
__global__ __launch_bounds__(64 * kJoinWaves) void beam_join_kernel(BeamArgs a, int pairs) {
  __shared__ __attribute__((aligned(16))) u64 s_key[kMaxBeams * kMaxBeams + 8];
  __shared__ double s_base[kMaxBeams], s_lse[kMaxBeams];
  __shared__ unsigned char s_done[kMaxBeams];
  extern __shared__ u64 s_list[];  // [pairs][chunks * k]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = a.k;
  const long long b = blockIdx.x;
  if (wave < pairs) {
    u64 *list = s_list + wave * a.chunks * k;
    for (int beam = wave; beam < a.beams; beam += pairs) {
      const long long at = (b * a.beams + beam) * a.chunks;  // (of an ended beam's parts, whatever is there)
      wave_order();  // the list before this one has been read
      for (int e = lane; e < a.chunks * k; e += 64) list[e] = a.part_key[at * k + e];
      wave_order();
      const u64 *next = list + lane * k, *const end = lane < a.chunks ? next + k : next;
      u64 mine = next < end ? *next++ : 0;
      for (int r = 0; r < k; ++r) {
        const u64 then = next < end ? *next : 0;
        const unsigned v = wave_umax((unsigned)(mine >> 32));
        const int first = __builtin_ctzll(__ballot((unsigned)(mine >> 32) == v));
        if (lane == first) {
          s_key[beam * k + r] = mine;  // 0 where none is left
          mine = then;
          ++next;
        }
      }
    }
  } else if (wave < 2 * pairs) {
    for (int beam = wave - pairs; beam < a.beams; beam += pairs) {
      const long long row = b * a.beams + beam, at = row * a.chunks;
      const float m = lane < a.chunks ? a.part_max[at + lane] : -INFINITY;
      const double s = lane < a.chunks ? a.part_sum[at + lane] : 0.0;
      if (lane == 0) {
        s_done[beam] = a.done ? a.done[row] : 0;
        s_base[beam] = (double)a.scores[row] + 0.0;  // no -0
      }
      const float top = wave_max(m);
      const double sum = wave_sum64(s == 0.0 ? 0.0 : s * exp((double)m - (double)top));
      if (lane == 0) s_lse[beam] = (double)top + log(sum);
    }
  }
  __syncthreads();
  // continuation e % k of beam e / k: its token, its score and that as a key
  const int n = a.beams * k;
  int token = 0;
  double y = -INFINITY;
  u64 key = 0;
  const int e = threadIdx.x;
  if (e < n) {
    const int beam = e / k, r = e - beam * k;
    const double base = s_base[beam], lse = s_lse[beam];
    const bool ended = s_done[beam] != 0, fine = fabs(base) < INFINITY;
    const u64 best = s_key[e];
    if (ended && fine) {
      // an ended beam goes on with the end's token alone
      y = r == 0 ? base : -INFINITY;
      token = r == 0 ? a.eos : r - 1 + (r - 1 >= a.eos);
    } else if (ended || !fine || !(fabs(lse) < INFINITY)) {
      // no continuation of its own: the first tokens, behind all others
      token = r;
    } else if (best) {
      y = base + ((double)logit_of(best) - lse);
      token = index_of(best);
    } else {
      // all other tokens are masked: the lowest of them, in order
      int skip = r;
      for (int i = 0; i < k; ++i) skip -= s_key[beam * k + i] != 0;
      for (token = 0;; ++token) {  // ends: k <= vocab, and fewer than k are taken
        bool taken = false;
        for (int i = 0; i < k; ++i) {
          const u64 other = s_key[beam * k + i];
          taken = taken || (other != 0 && index_of(other) == token);
        }
        if (!taken && skip-- == 0) break;
      }
    }
    key = ordered(y);
  }
  __syncthreads();  // the beams' lists have been read
  if (e < n) s_key[e] = key;
  if (e < 8) s_key[n + e] = 0;
  __syncthreads();
  if (e >= n) return;
  // the larger score, of equal ones the lower beam's, then its larger logit's
  int place = 0;
  for (int j = 0; j < n; j += 8) {
    u64 other[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) other[i] = s_key[j + i];
#pragma unroll
    for (int i = 0; i < 8; ++i) place += other[i] > key || (other[i] == key && j + i < e);
  }
  if (place >= k) return;
  const long long to = b * k + place;
  a.tokens[to] = token;
  a.parents[to] = e / k;
  a.scores_out[to] = (float)y;
  if (a.done_out) a.done_out[to] = s_done[e / k] != 0 || token == a.eos;
}

template <bool VEC>
void launch_rows(const BeamArgs &a, hipStream_t s) {
  const unsigned grid = (unsigned)a.batch * (unsigned)a.beams * (unsigned)a.chunks;
  // registers for a part's logits, or for 16 of a thread at a time
  if (a.chunk <= 4 * kThreads)
    beam_rows_kernel<VEC, 4><<<grid, kThreads, 0, s>>>(a);
  else if (a.chunk <= 8 * kThreads)
    beam_rows_kernel<VEC, 8><<<grid, kThreads, 0, s>>>(a);
  else
    beam_rows_kernel<VEC, 16><<<grid, kThreads, 0, s>>>(a);
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs &a, bool vec, hipStream_t s) {
  if (vec)
    launch_rows<true>(a, s);
  else
    launch_rows<false>(a, s);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // two waves a beam, and a thread for each of its continuations
  const int pairs = std::min({a.beams, kJoinWaves / 2, kJoinEntries / (a.chunks * a.k)});
  const int waves = std::max(2 * pairs, (a.beams * a.k + 63) / 64);
  beam_join_kernel<<<(unsigned)a.batch, 64 * waves, (size_t)pairs * a.chunks * a.k * sizeof(u64), s>>>(a, pairs);
  return hipGetLastError();
}

}  // namespace bnr

// bnr_beam.hip -- gfx950 kernels of beam search: of each request's beams the k
// best continuations over the whole vocabulary.
//
//   score(b, t) = scores[b] + logit[b, t] - lse[b],   lse = log sum_t exp(logit)
//
// Within a beam the order is that of the logits, so one pass over them finds
// the sum and the k best: a workgroup holds 4096 logits in registers, and what
// is under the k-th largest of a wave's 64 lane maxima (at least k logits are
// no smaller) is not among the k best.  The few that are left are ranked by
// counting.  A second launch joins the parts of each row and then the beams.
//
// Beams are compared by scores in 64 bits: lse is what the order of two beams'
// continuations hangs on, so its exponentials carry the part of log2(e) that
// fp32 leaves out and their sums are joined in 64 bits.
//
// Bound by the logits' bytes, read once.
#include "bnr_device.h"

namespace bnr {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kHeld = kBeamTile / kThreads;  // logits of a thread
constexpr int kCap = 512;                    // candidates of a tile that LDS has room for
constexpr int kNone = 0x7fffffff;

__device__ __forceinline__ float above(float m) { return m == -INFINITY ? 0.f : m; }

// exp(x - m): log2(e) in two parts, so that no term has an error of its own sign
// (with one part all terms of a row are off by 1.3e-8 of their exponent).
__device__ __forceinline__ float exp_from(float x, float m) {
  const float d = x - m;
  return fast_exp2(fmaf(d, 1.925963033500e-8f, d * 1.442695021629f));
}

// Order of a beam's continuations: the larger logit, then the lower index.
__device__ __forceinline__ bool better(float v, int i, float w, int j) { return v > w || (v == w && i < j); }

struct Best {
  float v;
  int i;
};
__device__ __forceinline__ Best wave_best(Best x) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const float v = __shfl_xor(x.v, k);
    const int i = __shfl_xor(x.i, k);
    if (better(v, i, x.v, x.i)) {
      x.v = v;
      x.i = i;
    }
  }
  return x;
}

__device__ __forceinline__ double wave_sum64(double v) {
#pragma unroll
  for (int k = 1; k < 64; k *= 2) v += __shfl_xor(v, k);
  return v;
}

// A workgroup's part of a row.
template <bool VEC>
__global__ __launch_bounds__(kThreads) void beam_rows_kernel(BeamArgs a) {
  __shared__ float s_v[kCap], s_top[kWaves];
  __shared__ int s_i[kCap], s_n;
  __shared__ double s_sum[kWaves];
  __shared__ Best s_best[kWaves];
  const int row = blockIdx.x / (unsigned)a.chunks, part = blockIdx.x - row * a.chunks;
  if (a.done && a.done[row]) return;  // the joins know it
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, tid = threadIdx.x, k = a.k;
  const float *x = a.logits + row * a.stride;
  const int v0 = part * a.chunk, v1 = min(v0 + a.chunk, a.vocab);
  float m = -INFINITY, sum = 0.f;
  int have = 0;  // entries of the list so far: s_v[0..have), the best first

  // Element n of the thread's logits of the tile at t0.
  const auto index = [&](int t0, int n) {
    return VEC ? t0 + 4 * (tid + kThreads * (n / 4)) + n % 4 : t0 + tid + kThreads * n;
  };
  for (int t0 = v0; t0 < v1; t0 += kBeamTile) {
    float h[kHeld];
#pragma unroll
    for (int n = 0; n < kHeld; n += VEC ? 4 : 1) {
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
    float top = h[0];
#pragma unroll
    for (int n = 1; n < kHeld; ++n) top = fmaxf(top, h[n]);
    if (!(top > -INFINITY)) top = -INFINITY;  // all NaN
    // places past the end hold -infinity: they add nothing
    const float mn = fmaxf(m, top), mu = above(mn);
    sum *= exp_from(above(m) == m ? m : mu, mu);
#pragma unroll
    for (int n = 0; n < kHeld; ++n) sum += exp_from(h[n], mu);
    m = mn;

    // What a candidate must reach: the k-th largest lane maximum of some wave, or the list's last entry.
    float least = -INFINITY;
    if (have < k) {
      float v = top;
      for (int r = 0; r < k; ++r) {
        least = wave_max(v);
        const int first = __builtin_ctzll(__ballot(v == least));
        if (lane == first) v = -INFINITY;
      }
      __syncthreads();  // the list is complete; s_top has been read
      if (lane == 0) s_top[wave] = least;
      if (tid == 0) s_n = have;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kWaves; ++w) least = fmaxf(least, s_top[w]);
    } else {
      const float last = s_v[k - 1];
      // later logits have higher indexes: an equal one stays behind
      if (!__syncthreads_or(top > last)) continue;
      least = last;
      if (tid == 0) s_n = have;
      __syncthreads();
    }
    const bool full = have == k;
#pragma unroll
    for (int n = 0; n < kHeld; ++n) {
      const int i = index(t0, n);
      if (i < v1 && (full ? h[n] > least : h[n] >= least)) {
        const int at = atomicAdd(&s_n, 1);
        if (at < kCap) {
          s_v[at] = h[n];
          s_i[at] = i;
        }
      }
    }
    __syncthreads();
    const int n_cand = s_n;
    if (n_cand <= kCap) {
      // a candidate's place is how many are better
      int place[kCap / kThreads];
      Best mine[kCap / kThreads];
#pragma unroll
      for (int c = 0; c < kCap / kThreads; ++c) {
        const int e = tid + c * kThreads;
        place[c] = k;
        if (e >= n_cand) continue;
        mine[c] = Best{s_v[e], s_i[e]};
        int p = 0;
        for (int j = 0; j < n_cand; ++j) p += better(s_v[j], s_i[j], mine[c].v, mine[c].i);
        place[c] = p;
      }
      __syncthreads();
#pragma unroll
      for (int c = 0; c < kCap / kThreads; ++c)
        if (place[c] < k) {
          s_v[place[c]] = mine[c].v;
          s_i[place[c]] = mine[c].i;
        }
      have = n_cand < k ? n_cand : k;
    } else {
      // Too many equal ones: the best that is left, k times.  The old list is
      // held by the first threads.
      const Best old = tid < have ? Best{s_v[tid], s_i[tid]} : Best{-INFINITY, kNone};
      Best last = {INFINITY, -1};
      have = k;  // there are more than k candidates
      for (int r = 0; r < k; ++r) {
        Best b = {-INFINITY, kNone};
        if (better(last.v, last.i, old.v, old.i) && better(old.v, old.i, b.v, b.i)) b = old;
#pragma unroll
        for (int n = 0; n < kHeld; ++n) {
          const int i = index(t0, n);
          if (i < v1 && better(last.v, last.i, h[n], i) && better(h[n], i, b.v, b.i)) b = Best{h[n], i};
        }
        b = wave_best(b);
        __syncthreads();  // s_best and, the first time, the old list have been read
        if (lane == 0) s_best[wave] = b;
        __syncthreads();
        b = s_best[0];
#pragma unroll
        for (int w = 1; w < kWaves; ++w)
          if (better(s_best[w].v, s_best[w].i, b.v, b.i)) b = s_best[w];
        last = b;
        if (tid == 0) {
          s_v[r] = b.v;
          s_i[r] = b.i;
        }
      }
    }
    __syncthreads();  // the list
  }

  // the part's maximum and sum
  const float wm = wave_max(m);
  if (lane == 0) s_top[wave] = wm;
  __syncthreads();
  float top = s_top[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s_top[w]);
  const double ws = wave_sum64((double)sum * (double)exp_from(above(m) == m ? m : above(top), above(top)));
  if (lane == 0) s_sum[wave] = ws;
  __syncthreads();
  const long long at = (long long)row * a.chunks + part;
  if (tid == 0) {
    a.part_max[at] = top;
    a.part_sum[at] = (s_sum[0] + s_sum[1]) + (s_sum[2] + s_sum[3]);
  }
  if (tid < k) {
    a.part_val[at * k + tid] = tid < have ? s_v[tid] : -INFINITY;
    a.part_idx[at * k + tid] = tid < have ? s_i[tid] : kNone;
  }
}

// Joins the parts of each beam's row, a wave for each, and then the request's
// beams: lane c has part (beam) c's list and the best of them that is not taken.
__global__ __launch_bounds__(kThreads) void beam_join_kernel(BeamArgs a) {
  __shared__ double s_y[kMaxBeams * kMaxBeams];
  __shared__ int s_t[kMaxBeams * kMaxBeams];
  extern __shared__ Best s_list[];  // [kWaves][chunks * k]
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, k = a.k;
  const long long b = blockIdx.x;
  Best *list = s_list + wave * a.chunks * k;
  for (int beam = wave; beam < a.beams; beam += kWaves) {
    const long long row = b * a.beams + beam;
    const double base = (double)a.scores[row];
    double *y = s_y + beam * k;
    int *t = s_t + beam * k;
    if (a.done && a.done[row] && fabs(base) < INFINITY) {
      // an ended beam goes on with the end's token alone
      if (lane < k) {
        y[lane] = lane == 0 ? base : -INFINITY;
        t[lane] = lane == 0 ? a.eos : lane - 1 + (lane - 1 >= a.eos);
      }
      continue;
    }
    const bool ended = a.done && a.done[row];  // its parts have not been made
    const long long at = row * a.chunks;
    const int parts = ended ? 0 : a.chunks;
    const float m = lane < parts ? a.part_max[at + lane] : -INFINITY;
    const double s = lane < parts ? a.part_sum[at + lane] : 0.0;
    for (int e = lane; e < parts * k; e += 64) list[e] = Best{a.part_val[at * k + e], a.part_idx[at * k + e]};
    const float top = wave_max(m);
    const double sum = wave_sum64(s == 0.0 ? 0.0 : s * exp((double)m - (double)top));
    const double lse = (double)top + log(sum);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (!(fabs(base) < INFINITY) || !(fabs(lse) < INFINITY)) {
      // no continuation of its own: the first tokens, behind all others
      if (lane < k) {
        y[lane] = -INFINITY;
        t[lane] = lane;
      }
      continue;
    }
    int head = 0;
    Best mine = lane < parts ? list[lane * k] : Best{-INFINITY, kNone};
    for (int r = 0; r < k; ++r) {
      const Best w = wave_best(mine);
      if (lane == 0) {
        y[r] = base + ((double)w.v - lse);
        t[r] = w.i;
      }
      if (mine.i == w.i && lane < parts) {  // indexes of a row are all different
        ++head;
        mine = head < k ? list[lane * k + head] : Best{-INFINITY, kNone};
      }
    }
  }
  __syncthreads();
  if (wave != 0) return;
  int head = 0;
  const bool in = lane < a.beams;
  double y = in ? s_y[lane * k] : -INFINITY;
  for (int r = 0; r < k; ++r) {
    // the largest score, of equal ones the first beam's; one without an entry left is behind all
    double best = y;
    int who = in && head < k ? lane : 64 + lane;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const double v = __shfl_xor(best, o);
      const int w = __shfl_xor(who, o);
      const bool there = w < 64, here = who < 64;
      if (there && (!here || v > best || (v == best && w < who))) {
        best = v;
        who = w;
      }
    }
    if (lane == who) {
      const long long to = b * k + r;
      const int token = s_t[lane * k + head];
      a.tokens[to] = token;
      a.parents[to] = lane;
      a.scores_out[to] = (float)y;
      if (a.done_out) a.done_out[to] = (a.done && a.done[b * a.beams + lane]) || token == a.eos;
      ++head;
      if (head < k) y = s_y[lane * k + head];
    }
  }
}

}  // namespace

hipError_t launch_beam_select(const BeamArgs &a, bool vec, hipStream_t s) {
  const unsigned grid = (unsigned)a.batch * (unsigned)a.beams * (unsigned)a.chunks;
  if (vec)
    beam_rows_kernel<true><<<grid, kThreads, 0, s>>>(a);
  else
    beam_rows_kernel<false><<<grid, kThreads, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  beam_join_kernel<<<(unsigned)a.batch, kThreads, (size_t)kWaves * a.chunks * a.k * sizeof(Best), s>>>(a);
  return hipGetLastError();
}

}  // namespace bnr

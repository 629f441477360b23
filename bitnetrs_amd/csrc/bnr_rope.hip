// bnr_rope.hip -- gfx950 kernels of the rotary embeddings: q and k heads of any
// strides rotated at each token's position, and the rotation's tables.
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_b cos t + x_a sin t),  t = position * rate
//
// for the pairs (a, b) = (i, i + dim/2) or (2i, 2i + 1); elements from dim on
// are copied.  A position times a rate needs more places than fp32 has: the
// angle is counted in turns in fp64, whole turns and the nearest eighths are
// taken off exactly, and what is left (at most an eighth of a turn) goes to
// fp32's sine and cosine.
//
// Bound by the heads' bytes, read once and written once.  A workgroup takes one
// token, or several where there are many, and makes their angles once, in LDS,
// for all heads.
#include "bnr_device.h"

namespace bnr {
namespace {

constexpr int kThreads = 256;

// cos and sin of `turns` whole turns and fractions, times m.
__device__ __forceinline__ float2 rope_angle(double turns, float m) {
  double t = turns - rint(turns);
  const double q = rint(4.0 * t);
  t -= 0.25 * q;  // at most an eighth, exact
  float s, c;
  sincospif((float)(2.0 * t), &s, &c);
  const int k = (int)q & 3;
  const float x = k & 1 ? s : c, y = k & 1 ? c : s;
  return make_float2(m * (k == 1 || k == 2 ? -x : x), m * (k >= 2 ? -y : y));
}

template <class T>
__device__ __forceinline__ float widen(T x) {
  return (float)x;
}

// N elements (16 bytes at most) at p.
template <class T, int N>
struct Some {
  T x[N];
};
template <class T, int N>
__device__ __forceinline__ Some<T, N> load_some(const T *p) {
  Some<T, N> r;
  if constexpr (sizeof(r) == 16) {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    const u4 w = *reinterpret_cast<const u4 *>(p);
    __builtin_memcpy(&r, &w, 16);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.x[i] = p[i];
  }
  return r;
}
template <class T, int N>
__device__ __forceinline__ void store_some(T *p, const Some<T, N> &r) {
  if constexpr (sizeof(r) == 16) {
    typedef unsigned u4 __attribute__((ext_vector_type(4)));
    u4 w;
    __builtin_memcpy(&w, &r, 16);
    *reinterpret_cast<u4 *>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = r.x[i];
  }
}

// U: pairs of a thread's step, whose elements are two runs of U; 1 where
// alignment or sizes leave no more.
template <class T, int U, bool HALF>
__global__ __launch_bounds__(kThreads) void rope_kernel(RopeArgs a) {
  __shared__ float2 s_cs[kThreads > kRopeMaxPairs ? kThreads : kRopeMaxPairs];
  __shared__ int s_pos[kThreads];
  const int pairs = a.pairs, tid = threadIdx.x;
  const long long token0 = (long long)blockIdx.x * a.tokens;
  const int here = (int)(a.n_tokens - token0 < a.tokens ? a.n_tokens - token0 : a.tokens);
  if (tid < here) s_pos[tid] = a.positions[token0 + tid];
  for (int i = tid; i < here * pairs; i += kThreads) {
    const int p = a.positions[token0 + i / pairs];
    s_cs[i] = rope_angle((double)p * a.turns[i % pairs], a.magnitude);
  }
  __syncthreads();
  // A row's (a head's) steps: those of its pairs, then those of the elements behind
  // them; `lanes` threads (a power of two) share a row.
  const int rot = (pairs + U - 1) / U, steps = rot + (a.d - 2 * pairs + 2 * U - 1) / (2 * U);
  const int heads = a.q.heads + a.k.heads, rows = here * heads;
  const int u0 = tid & (a.lanes - 1), per = kThreads / a.lanes;
  for (int r = tid / a.lanes; r < rows; r += per) {
    const int t = r / heads, h = r - t * heads;
    if (s_pos[t] < 0) continue;  // left out
    const bool is_k = h >= a.q.heads;
    const RopeHeads &x = is_k ? a.k : a.q;
    const int head = is_k ? h - a.q.heads : h;
    const T *in = static_cast<const T *>(x.in) + (token0 + t) * x.in_token + head * x.in_head;
    T *out = static_cast<T *>(x.out) + (token0 + t) * x.out_token + head * x.out_head;
    for (int u = u0; u < steps; u += a.lanes) {
      if (u >= rot) {
        if (in == out) continue;
        const int e = 2 * pairs + (u - rot) * 2 * U;
        if constexpr (U == 1) {
          out[e] = in[e];
          if (e + 1 < a.d) out[e + 1] = in[e + 1];
        } else {
          const auto lo = load_some<T, U>(in + e), hi = load_some<T, U>(in + e + U);
          store_some(out + e, lo);
          store_some(out + e + U, hi);
        }
        continue;
      }
      const int i = u * U, e0 = HALF ? i : 2 * i, e1 = HALF ? i + pairs : 2 * i + U;
      Some<T, U> lo = load_some<T, U>(in + e0), hi = load_some<T, U>(in + e1);
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const float2 cs = s_cs[t * pairs + i + j];
        // pairs: the runs' elements j, or neighbours of the two runs taken as one
        T &p = HALF || U == 1 ? lo.x[j] : 2 * j < U ? lo.x[(2 * j) % U] : hi.x[(2 * j) % U];
        T &q = HALF || U == 1 ? hi.x[j] : 2 * j < U ? lo.x[(2 * j + 1) % U] : hi.x[(2 * j + 1) % U];
        float y, z;
        rot_pair((float)p, (float)q, cs.x, cs.y, y, z);
        p = (T)y;
        q = (T)z;
      }
      store_some(out + e0, lo);
      store_some(out + e1, hi);
    }
  }
}

__global__ __launch_bounds__(kThreads) void rope_table_kernel(RopeTableArgs a) {
  const unsigned long long total = (unsigned long long)a.n_positions * a.pairs;
  for (unsigned long long n = (unsigned long long)blockIdx.x * kThreads + threadIdx.x; n < total;
       n += (unsigned long long)gridDim.x * kThreads) {
    const unsigned long long p = n >> 32 ? n / a.pairs : (unsigned)n / (unsigned)a.pairs;
    const int i = (int)(n - p * a.pairs);
    const float2 cs = rope_angle((double)(a.first + (long long)p) * a.turns[i], a.magnitude);
    a.cos_out[n] = cs.x;
    a.sin_out[n] = cs.y;
  }
}

template <class T, int U>
void launch_layout(const RopeArgs &a, bool half, hipStream_t s) {
  const unsigned grid = (unsigned)((a.n_tokens + a.tokens - 1) / a.tokens);
  if (half)
    rope_kernel<T, U, true><<<grid, kThreads, 0, s>>>(a);
  else
    rope_kernel<T, U, false><<<grid, kThreads, 0, s>>>(a);
}

template <class T>
void launch_type(const RopeArgs &a, bool half, bool vec, hipStream_t s) {
  if (vec)
    launch_layout<T, 16 / sizeof(T)>(a, half, s);
  else
    launch_layout<T, 1>(a, half, s);
}

}  // namespace

hipError_t launch_rope(RopeArgs a, int type, bool half, bool vec, hipStream_t s) {
  // tokens of a workgroup: as many as its threads make the angles of, where
  // there are workgroups enough
  a.tokens = 1;
  if (a.n_tokens >= 2048 && a.pairs <= kThreads / 2) a.tokens = kThreads / a.pairs;
  if (a.tokens > 32) a.tokens = 32;
  const int unit = vec ? 16 / (type == kRopeF32 ? 4 : 2) : 1;
  const int steps = (a.pairs + unit - 1) / unit + (a.d - 2 * a.pairs + 2 * unit - 1) / (2 * unit);
  a.lanes = 1;
  while (a.lanes < steps && a.lanes < kThreads) a.lanes *= 2;
  switch (type) {
    case kRopeF32: launch_type<float>(a, half, vec, s); break;
    case kRopeBf16: launch_type<__bf16>(a, half, vec, s); break;
    case kRopeF16: launch_type<_Float16>(a, half, vec, s); break;
    default: return hipErrorInvalidValue;
  }
  return hipGetLastError();
}

hipError_t launch_rope_table(const RopeTableArgs &a, hipStream_t s) {
  const unsigned long long wgs = ((unsigned long long)a.n_positions * a.pairs + kThreads - 1) / kThreads;
  rope_table_kernel<<<(unsigned)(wgs < 65536 ? wgs : 65536), kThreads, 0, s>>>(a);
  return hipGetLastError();
}

}  // namespace bnr

// bnr_rope.hip -- gfx950 kernels of the rotary embeddings: q and k heads of any
// strides rotated at each token's position, and the rotation's tables.
//
//   y_a = m (x_a cos t - x_b sin t),  y_b = m (x_b cos t + x_a sin t),  t = position * rate
//
// for the pairs (a, b) = (i, i + dim/2) or (2i, 2i + 1); elements from dim on
// are copied.  A position times a rate needs more places than fp32 has: the
// angle is counted in turns in fp64, whole turns and the nearest quarters are
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
__device__ __forceinline__ void rotate(T &p, T &q, float2 cs) {
  float y, z;
  rot_pair((float)p, (float)q, cs.x, cs.y, y, z);
  p = (T)y;
  q = (T)z;
}

// N elements at p; WIDE: 8 or 16 aligned bytes in one access.
template <class T, int N>
struct Some {
  T x[N];
};
template <int BYTES>
struct Words {
  typedef unsigned type __attribute__((ext_vector_type(BYTES / 4)));
};
template <bool WIDE, class T, int N>
__device__ __forceinline__ Some<T, N> load_some(const T *p) {
  Some<T, N> r;
  if constexpr (WIDE) {
    typedef typename Words<sizeof(r)>::type W;
    const W w = *reinterpret_cast<const W *>(p);
    __builtin_memcpy(&r, &w, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) r.x[i] = p[i];
  }
  return r;
}
template <bool WIDE, class T, int N>
__device__ __forceinline__ void store_some(T *p, const Some<T, N> &r) {
  if constexpr (WIDE) {
    typedef typename Words<sizeof(r)>::type W;
    W w;
    __builtin_memcpy(&w, &r, sizeof(r));
    if constexpr (sizeof(r) == 16)
      __builtin_nontemporal_store(w, reinterpret_cast<W *>(p));
    else
      *reinterpret_cast<W *>(p) = w;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = r.x[i];
  }
}

// U: elements of 16 bytes, of 8, or 1 where alignment or sizes leave no more.  A step of
// a thread is U pairs of two runs (half), U / 2 pairs of one run (interleaved; one
// pair where U is 1), or U elements that are copied: neighbouring threads' steps
// are neighbours, so a wave's loads and stores are whole lines.  16384 tokens of
// 32/8 bf16 heads of 128, 32 of them rotated in pairs of neighbours: 66 us, 5.1 TB/s,
// as a copy; with 32 bytes a thread 80.  16 bytes go out with the non-temporal hint (69
// without; 512 f32 tokens of 32/8 heads of 128 6.2, 7.1 without; 64 3.7 both).  With
// kernels that make q and read it the hint changes nothing: 64 tokens 11.2, 512 of f32
// 19.5, 4096 of bf16 48.8, 16384 158 with it and without.  4096
// tokens of 32/8 bf16 heads of 80, 40 of them rotated in halves, so that runs are units
// of 8 bytes: 14 us, 44 with single elements.
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
  constexpr int W = HALF || U > 1 ? U : 2;  // elements of a run
  const int rot = HALF ? pairs / U : 2 * pairs / W, steps = rot + (a.d - 2 * pairs) / U;
  const int heads = a.q.heads + a.k.heads, rows = here * heads, per = kThreads / a.lanes;
  constexpr int N = U > 1 ? 2 : 1;  // rows of a thread on their way at a time
  for (int u = tid & (a.lanes - 1); u < steps; u += a.lanes) {
    const bool turn = u < rot;
    const int e = turn ? u * W : 2 * pairs + (u - rot) * U, e2 = HALF && turn ? e + pairs : e;
    for (int r0 = tid / a.lanes; r0 < rows; r0 += N * per) {
      Some<T, W> x[N], x2[N];
      T *out[N];
      int at[N];
      bool there[N];
#pragma unroll
      for (int n = 0; n < N; ++n) {
        // past the last row: the first again, not written (a branch would part the loads)
        const int r = r0 + n * per < rows ? r0 + n * per : r0, t = r / heads, h = r - t * heads;
        const bool is_k = h >= a.q.heads;
        const RopeHeads &o = is_k ? a.k : a.q;
        const int head = is_k ? h - a.q.heads : h;
        const T *in = static_cast<const T *>(o.in) + (token0 + t) * o.in_token + head * o.in_head;
        out[n] = static_cast<T *>(o.out) + (token0 + t) * o.out_token + head * o.out_head;
        at[n] = t;
        there[n] = r0 + n * per < rows && s_pos[t] >= 0 && (turn || in != out[n]);
        if (W == U || turn) x[n] = load_some<(U > 1), T, W>(in + e);
        else x[n].x[0] = in[e];
        if (HALF) x2[n] = load_some<(U > 1), T, W>(in + e2);
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!there[n]) continue;
        if (turn) {
          const float2 *cs = s_cs + at[n] * pairs + (HALF ? u * U : u * (W / 2));
#pragma unroll
          for (int j = 0; j < (HALF ? U : W / 2); ++j) {
            if constexpr (HALF)
              rotate(x[n].x[j], x2[n].x[j], cs[j]);
            else
              rotate(x[n].x[2 * j], x[n].x[2 * j + 1], cs[j]);
          }
          if (HALF) store_some<(U > 1)>(out[n] + e2, x2[n]);
        }
        if (W == U || turn)
          store_some<(U > 1)>(out[n] + e, x[n]);
        else
          out[n][e] = x[n].x[0];
      }
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

// A launch holds fewer than 2^32 threads: more tokens go in pieces.
constexpr long long kMaxGrid = 1 << 22;

template <class T>
void skip_tokens(RopeHeads &h, long long n) {
  h.in = static_cast<const T *>(h.in) + n * h.in_token;
  h.out = static_cast<T *>(h.out) + n * h.out_token;
}

template <class T, int U>
void launch_layout(RopeArgs &a, bool half, hipStream_t s) {
  const long long piece = kMaxGrid * a.tokens;
  for (long long left = a.n_tokens; left > 0; left -= piece) {
    a.n_tokens = left < piece ? left : piece;
    const unsigned grid = (unsigned)((a.n_tokens + a.tokens - 1) / a.tokens);
    if (half)
      rope_kernel<T, U, true><<<grid, kThreads, 0, s>>>(a);
    else
      rope_kernel<T, U, false><<<grid, kThreads, 0, s>>>(a);
    if (left <= piece) break;
    a.positions += piece;
    skip_tokens<T>(a.q, piece);
    skip_tokens<T>(a.k, piece);
  }
}

template <class T>
void launch_type(RopeArgs &a, bool half, int bytes, hipStream_t s) {
  if (bytes == 16)
    launch_layout<T, 16 / sizeof(T)>(a, half, s);
  else if (bytes == 8)
    launch_layout<T, 8 / sizeof(T)>(a, half, s);
  else
    launch_layout<T, 1>(a, half, s);
}

}  // namespace

hipError_t launch_rope(RopeArgs a, int type, bool half, int bytes, hipStream_t s) {
  // tokens of a workgroup: as many as its threads make the angles of, at most
  // four, where there are workgroups enough
  a.tokens = 1;
  if (a.n_tokens >= 2048 && a.pairs <= kThreads / 2) a.tokens = kThreads / a.pairs;
  if (a.tokens > 4) a.tokens = 4;
  const int unit = bytes ? bytes / (type == kRopeF32 ? 4 : 2) : 1;
  const int steps = (half ? a.pairs / unit : unit > 1 ? 2 * a.pairs / unit : a.pairs) + (a.d - 2 * a.pairs) / unit;
  a.lanes = 1;
  while (a.lanes < steps && a.lanes < kThreads) a.lanes *= 2;
  switch (type) {
    case kRopeF32: launch_type<float>(a, half, bytes, s); break;
    case kRopeBf16: launch_type<__bf16>(a, half, bytes, s); break;
    case kRopeF16: launch_type<_Float16>(a, half, bytes, s); break;
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

// bnr_pages.hip -- gfx950 kernels of the paged cache's bookkeeping: pages for
// new tokens and the arrays that say where each goes (extend), pages given back
// (release), the tables of reordered beams, and rows copied between sequences.
#include "bnr_paged.h"

#include <algorithm>

namespace bnr {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

typedef unsigned long long u64;

// Rows of a page as a divisor; the shift where it is a power of two.
struct PageSize {
  int rows, shift;
  __device__ __forceinline__ explicit PageSize(int page)
      : rows(page), shift(page & (page - 1) ? -1 : __builtin_ctz((unsigned)page)) {}
  __device__ __forceinline__ int of(int row) const { return shift >= 0 ? row >> shift : row / rows; }
  // pages of n rows; n + rows <= 2^31
  __device__ __forceinline__ int pages(int n) const { return of(n + rows - 1); }
};

// The sequence whose part of the line off[0..n] has place x: off[s] <= x < off[s + 1].
__device__ __forceinline__ int part_of(const int *off, int n, int x) {
  int lo = 0, hi = n;  // off[lo] <= x < off[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (off[mid] <= x)
      lo = mid;
    else
      hi = mid;
  }
  return lo;
}

// Sums that stay at 2^32 - 1: more than any limit.
__device__ __forceinline__ unsigned sat(unsigned a, unsigned b) { return __builtin_elementwise_add_sat(a, b); }

// Inclusive sums over the wave's lanes.
__device__ __forceinline__ unsigned scan_sat(unsigned v) {
#define BNR_SCAN(CTRL, ROWS) v = sat(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xF, false))
  BNR_SCAN(0x111, 0xF);  // row_shr:1, 2, 4, 8: sums within each row of 16 lanes
  BNR_SCAN(0x112, 0xF);
  BNR_SCAN(0x114, 0xF);
  BNR_SCAN(0x118, 0xF);
  BNR_SCAN(0x142, 0xA);  // row_bcast:15 into rows 1 and 3
  BNR_SCAN(0x143, 0xC);  // row_bcast:31 into rows 2 and 3
#undef BNR_SCAN
  return v;
}

// Every workgroup adds up the whole batch for itself, so that one launch does
// it all and nothing is kept between launches: two loads a sequence, from L2.
// want(s, a, b): the sequence's two amounts.  Leaves in line_a and line_b
// [n_seqs + 1] (LDS) what each sequence's parts of the two lines start at.  In order,
// up to the first sequence that goes past a limit: it and those behind it get nothing.
struct Shares {
  unsigned wave[kWaves][2], stop[2];
};
template <class Want>
__device__ __forceinline__ void share_out(int n_seqs, unsigned limit_a, unsigned limit_b, Shares &sh, int *line_a,
                                          int *line_b, Want want) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // a run of sequences a thread
  const int per = (n_seqs + kThreads - 1) / kThreads, s0 = tid * per, s1 = s0 + per < n_seqs ? s0 + per : n_seqs;
  unsigned sum[2] = {0, 0};
  for (int s = s0; s < s1; ++s) {
    unsigned a, b;
    want(s, a, b);
    line_a[s] = (int)a;
    line_b[s] = (int)b;
    sum[0] = sat(sum[0], a);
    sum[1] = sat(sum[1], b);
  }
  const unsigned in[2] = {scan_sat(sum[0]), scan_sat(sum[1])};
  if (lane == 63) {
    sh.wave[wave][0] = in[0];
    sh.wave[wave][1] = in[1];
  }
  __syncthreads();
  unsigned at[2], all[2] = {0, 0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    at[i] = (unsigned)__builtin_amdgcn_update_dpp(0, (int)in[i], 0x138, 0xF, 0xF, false);  // wave_shr:1
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) at[i] = sat(at[i], sh.wave[w][i]);
      all[i] = sat(all[i], sh.wave[w][i]);
    }
  }
  const bool whole = all[0] <= limit_a && all[1] <= limit_b;
  for (int s = s0; s < s1; ++s) {
    const unsigned to[2] = {sat(at[0], (unsigned)line_a[s]), sat(at[1], (unsigned)line_b[s])};
    // the first that does not fit (sums only grow): there is one
    if ((to[0] > limit_a || to[1] > limit_b) && at[0] <= limit_a && at[1] <= limit_b) {
      sh.stop[0] = at[0];
      sh.stop[1] = at[1];
    }
    line_a[s] = (int)at[0];
    line_b[s] = (int)at[1];
    at[0] = to[0];
    at[1] = to[1];
  }
  __syncthreads();
  const unsigned end[2] = {whole ? all[0] : sh.stop[0], whole ? all[1] : sh.stop[1]};
  if (!whole)
    for (int s = s0; s < s1; ++s)
      if ((unsigned)line_a[s] > end[0] || (unsigned)line_b[s] > end[1]) {
        line_a[s] = (int)end[0];
        line_b[s] = (int)end[1];
      }
  if (tid == 0) {
    line_a[n_seqs] = (int)end[0];
    line_b[n_seqs] = (int)end[1];
  }
  __syncthreads();
}

// ---------------------------------------------------------------------------
// Extend.  16 bytes written for each token, N tokens a thread: four where that
// leaves workgroups enough (790949 tokens of 300 sequences: 8.5 us, 11 with one),
// one for a decode step, which is latency: lengths and counts, sums, then a page
// and its entry (64 sequences: 4.6 us, 5.3 with four).
// ---------------------------------------------------------------------------
typedef int int4v __attribute__((ext_vector_type(4)));
typedef long long ll2v __attribute__((ext_vector_type(2)));

template <int N>
__global__ __launch_bounds__(kThreads) void paged_extend_kernel(ExtendArgs a) {
  extern __shared__ int s_line[];  // [3][n_seqs + 1]: places of pages, of tokens; lengths
  __shared__ Shares sh;
  int *s_page = s_line, *s_tok = s_line + a.n_seqs + 1, *s_len = s_tok + a.n_seqs + 1;
  const PageSize ps(a.page);
  const int room = (int)(a.table_stride * a.page);
  int free = *a.free_count;
  free = free < 0 ? 0 : free > a.free_cap ? a.free_cap : free;
  share_out(a.n_seqs, (unsigned)free, (unsigned)a.n_tokens, sh, s_page, s_tok, [&](int s, unsigned &p, unsigned &n) {
    const int len = max(a.lens[s], 0), more = max(a.fresh[s], 0);
    s_len[s] = len;
    n = len <= room && more <= room - len ? (unsigned)more : 0u;
    p = n ? (unsigned)(ps.pages(len + (int)n) - ps.pages(len)) : 0u;
  });
  const int pages = s_page[a.n_seqs], tokens = s_tok[a.n_seqs], tid = threadIdx.x;
  const long long first = (long long)blockIdx.x * kThreads + tid, step = (long long)gridDim.x * kThreads;
  for (long long e = first; e < pages; e += step) {
    const int s = part_of(s_page, a.n_seqs, (int)e);
    a.table[s * a.table_stride + ps.pages(s_len[s]) + ((int)e - s_page[s])] = a.free_pages[free - 1 - e];
  }
  for (long long i0 = N * first; i0 < a.n_tokens; i0 += N * step) {
    int seq[N], at[N];
    long long slot[N];
    int s = i0 < tokens ? part_of(s_tok, a.n_seqs, (int)i0) : 0;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const long long i = i0 + j;
      seq[j] = at[j] = -1;
      slot[j] = -1;
      if (i >= tokens) continue;
      while (s_tok[s + 1] <= (int)i) ++s;  // ends: i < tokens
      const int len = s_len[s], t = len + ((int)i - s_tok[s]);
      seq[j] = s;
      at[j] = t;
      if (a.slots) {
        const int p = ps.of(t), have = ps.pages(len);
        const int page = p < have ? a.table[s * a.table_stride + p] : a.free_pages[free - 1 - (s_page[s] + p - have)];
        slot[j] = page < 0 ? -1 : (long long)page * a.page + (t - p * a.page);
      }
    }
    if constexpr (N == 4)
      if (a.vec && i0 + 4 <= a.n_tokens) {
        *reinterpret_cast<int4v *>(a.seqs + i0) = int4v{seq[0], seq[1], seq[2], seq[3]};
        *reinterpret_cast<int4v *>(a.positions + i0) = int4v{at[0], at[1], at[2], at[3]};
        if (a.slots) {
          *reinterpret_cast<ll2v *>(a.slots + i0) = ll2v{slot[0], slot[1]};
          *reinterpret_cast<ll2v *>(a.slots + i0 + 2) = ll2v{slot[2], slot[3]};
        }
        continue;
      }
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (i0 + j < a.n_tokens) {
        a.seqs[i0 + j] = seq[j];
        a.positions[i0 + j] = at[j];
        if (a.slots) a.slots[i0 + j] = slot[j];
      }
  }
  for (long long s = first; s < a.n_seqs; s += step) {
    a.lens_out[s] = s_len[s] + (s_tok[s + 1] - s_tok[s]);
    a.offsets[s] = s_tok[s];
  }
  if (first == 0) {
    a.offsets[a.n_seqs] = tokens;
    *a.count_out = free - pages;
  }
}

// ---------------------------------------------------------------------------
// Release: the marked sequences' pages behind those to keep, back on the stack.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void paged_release_kernel(ReleaseArgs a) {
  extern __shared__ int s_line[];  // [2][n_seqs + 1]: places of pages; nothing
  __shared__ Shares sh;
  int *s_page = s_line;
  const PageSize ps(a.page);
  const int room = (int)(a.table_stride * a.page);
  int free = *a.free_count;
  free = free < 0 ? 0 : free > a.free_cap ? a.free_cap : free;
  const auto kept = [&](int s) { return a.keep ? max(a.keep[s], 0) : 0; };
  const auto pages_of = [&](int s) { return ps.pages(min(max(a.lens[s], 0), room)); };
  share_out(a.n_seqs, (unsigned)(a.free_cap - free), 0u, sh, s_page, s_line + a.n_seqs + 1,
            [&](int s, unsigned &p, unsigned &none) {
              const int n = a.which[s] ? pages_of(s) - kept(s) : 0;
              p = n > 0 ? (unsigned)n : 0u;
              none = 0;
            });
  const int pages = s_page[a.n_seqs], tid = threadIdx.x;
  const long long first = (long long)blockIdx.x * kThreads + tid, step = (long long)gridDim.x * kThreads;
  for (long long e = first; e < pages; e += step) {
    const int s = part_of(s_page, a.n_seqs, (int)e);
    int *entry = a.table + s * a.table_stride + kept(s) + ((int)e - s_page[s]);
    a.free_pages[free + e] = *entry;
    *entry = -1;
  }
  for (long long s = first; s < a.n_seqs; s += step) {
    const long long len = max(a.lens[s], 0), most = (long long)kept((int)s) * a.page;
    // all of its pages went (none where it does not fit), or it had none to give
    const bool gone = a.which[s] && (s_page[s + 1] > s_page[s] || pages_of((int)s) <= kept((int)s));
    a.lens_out[s] = (int)(gone && most < len ? most : len);
  }
  if (first == 0) *a.count_out = free + pages;
}

// ---------------------------------------------------------------------------
// Tables of reordered beams, a workgroup for each row.  Of the beams that go on
// from one parent the first has its pages; the others have those of the parents
// that nothing goes on from, both in order: as many of the one as of the other.
// Lane j of every wave holds beam j's parent.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void beam_reorder_kernel(BeamTableArgs a) {
  const int lane = threadIdx.x & 63, K = a.beams;
  const long long b = blockIdx.x / (unsigned)K;
  const int j = (int)(blockIdx.x - b * K);
  int parent = -1;
  if (lane < K) {
    parent = a.parents[b * K + lane];
    if (parent < 0 || parent >= K) parent = lane;
  }
  u64 heirs = 0, live = 0;  // of the beams, of the parents
  for (int i = 0; i < K; ++i) {
    const u64 children = __ballot(parent == i);
    if (children) {
      heirs |= children & -children;
      live |= 1ull << i;
    }
  }
  const int mine = __builtin_amdgcn_readlane(parent, j);
  const u64 all = K == 64 ? ~0ull : (1ull << K) - 1, before = (1ull << j) - 1;
  int row = mine, src = -1;
  if (!(heirs >> j & 1)) {
    src = (int)(b * K) + __builtin_ctzll(__ballot(parent == mine));
    u64 ended = all & ~live;
    for (int n = __builtin_popcountll(all & ~heirs & before); n > 0; --n) ended &= ended - 1;
    row = __builtin_ctzll(ended);
  }
  const int *from = a.table + (b * K + row) * a.table_stride;
  int *to = a.table_out + (b * K + j) * a.table_stride;
  for (long long i = threadIdx.x; i < a.table_stride; i += kThreads) to[i] = from[i];
  if (threadIdx.x == 0) a.src[b * K + j] = src;
}

// ---------------------------------------------------------------------------
// Copy: rows starts[s] .. lens[s]-1 of sequence src[s] to sequence s, their codes
// and scales as they are, in equal shares of all rows that are to be copied;
// `lanes` threads share a row.  Bound by the rows' bytes, read and written: 126 MB in
// 24.1 us, 5.2 TB/s (16 requests of 8 beams, 523 bf16 rows of 5 heads of 128 each;
// 27.9 before stores had the non-temporal hint, then shares of 32 rows 34, of 16 rows
// 48, two rows of a thread on their way 29).
// ---------------------------------------------------------------------------
constexpr int kCopyWgs = 4096, kCopyRows = 64;
constexpr int kCopyPasses = 4;  // rows of a thread on their way at a time

template <int U>
struct Unit;
template <>
struct Unit<16> { typedef unsigned type __attribute__((ext_vector_type(4))); };
template <>
struct Unit<8> { typedef unsigned type __attribute__((ext_vector_type(2))); };
template <>
struct Unit<4> { typedef unsigned type; };
template <>
struct Unit<2> { typedef unsigned short type; };
template <>
struct Unit<1> { typedef unsigned char type; };

// Whole lines go out with the non-temporal hint: 16 requests of 8 beams, 523 bf16 rows of 5 heads of 128 each,
// 31.5 -> 26.7 us with the tables'; eight layers copied and then attended over, as a step does, 86.3 -> 80.0 a
// layer; each layer's attention right behind its copy 74.3 -> 75.2.
template <int U, class T>
__device__ __forceinline__ void store_unit(T *p, T v) {
  if constexpr (U == 16)
    __builtin_nontemporal_store(v, p);
  else
    *p = v;
}

template <int U>
__global__ __launch_bounds__(kThreads) void paged_copy_kernel(PagedCopyArgs a) {
  typedef typename Unit<U>::type T;
  const auto start = [&](int s) { return a.starts ? max(a.starts[s], 0) : 0; };
  const auto rows = [&](int s) {
    const int from = a.src[s], len = paged_len(a.lens[s], a.pool), first = start(s);
    return from < 0 || from >= a.n_seqs || from == s || first >= len ? 0 : len - first;
  };
  const int units = a.row_bytes / U, x0 = threadIdx.x & (a.lanes - 1), pass = kThreads / a.lanes;
  const T *const k = static_cast<const T *>(a.pool.k), *const v = static_cast<const T *>(a.pool.v);
  T *const ko = static_cast<T *>(a.pool.k), *const vo = static_cast<T *>(a.pool.v);
  PagedShare sh = paged_share(rows, a.n_seqs, a.pool.n_kv, a.tile, a.wgs);
  for (PagedPiece p; sh.next(rows, p);) {
    const int first = start(p.b) + p.row0, src = a.src[p.b], n = p.row1 - p.row0;
    for (int r0 = (int)threadIdx.x / a.lanes; r0 < n; r0 += kCopyPasses * pass) {
      long long from[kCopyPasses], to[kCopyPasses];
#pragma unroll
      for (int i = 0; i < kCopyPasses; ++i) {
        // past the last row: the first again, not written (a branch would part the loads)
        const int r = r0 + i * pass < n ? r0 + i * pass : r0;
        from[i] = paged_row(a.pool, src, p.h, first + r);
        to[i] = paged_row(a.pool, p.b, p.h, first + r);
        if (r0 + i * pass >= n || from[i] < 0 || from[i] == to[i]) to[i] = -1;
        if (from[i] < 0) from[i] = 0;
      }
      for (int x = x0; x < units; x += a.lanes) {
        T ks[kCopyPasses], vs[kCopyPasses];
#pragma unroll
        for (int i = 0; i < kCopyPasses; ++i) {
          ks[i] = k[from[i] * units + x];
          vs[i] = v[from[i] * units + x];
        }
#pragma unroll
        for (int i = 0; i < kCopyPasses; ++i)
          if (to[i] >= 0) {
            store_unit<U>(ko + to[i] * units + x, ks[i]);
            store_unit<U>(vo + to[i] * units + x, vs[i]);
          }
      }
    }
    if (a.scale_bytes == 0) continue;
    for (int e = threadIdx.x; e < n * 2 * a.scale_bytes; e += kThreads) {
      const int r = e / (2 * a.scale_bytes), x = e - r * 2 * a.scale_bytes, t = first + r;
      const long long from = paged_row(a.pool, src, p.h, t), to = paged_row(a.pool, p.b, p.h, t);
      if (from < 0 || to < 0 || from == to) continue;
      const int is_v = x >= a.scale_bytes, at = x - is_v * a.scale_bytes;
      unsigned char *sc = a.pool.k_exps
                              ? (is_v ? a.pool.v_exps : a.pool.k_exps)
                              : reinterpret_cast<unsigned char *>(is_v ? a.pool.v_scales : a.pool.k_scales);
      sc[to * a.scale_bytes + at] = sc[from * a.scale_bytes + at];
    }
  }
}

}  // namespace

// Workgroups for n items, each of which adds up all sequences first.
static unsigned grid_for(long long n, long long per) {
  return (unsigned)std::max<long long>(1, std::min<long long>((n + per - 1) / per, 1024));
}

hipError_t launch_paged_extend(const ExtendArgs &a, hipStream_t s) {
  const size_t lds = 3 * (a.n_seqs + 1) * sizeof(int);
  if (a.n_tokens >= 256 * kThreads)
    paged_extend_kernel<4><<<grid_for(a.n_tokens, 4 * kThreads), kThreads, lds, s>>>(a);
  else
    paged_extend_kernel<1><<<grid_for(a.n_tokens, kThreads), kThreads, lds, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_release(const ReleaseArgs &a, hipStream_t s) {
  const long long pages = std::min<long long>(a.n_seqs * a.table_stride, a.free_cap);
  paged_release_kernel<<<grid_for(pages, kThreads), kThreads, 2 * (a.n_seqs + 1) * sizeof(int), s>>>(a);
  return hipGetLastError();
}

hipError_t launch_beam_reorder(const BeamTableArgs &a, hipStream_t s) {
  beam_reorder_kernel<<<(unsigned)a.batch * (unsigned)a.beams, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_copy(PagedCopyArgs a, int unit, hipStream_t s) {
  const long long items = (long long)a.n_seqs * a.pool.n_kv, rows = a.pool.table_stride * a.pool.page;
  a.tile = kCopyRows;
  while ((rows + a.tile - 1) / a.tile * items >= 1ll << 31) a.tile *= 2;
  a.wgs = (int)std::min<long long>(kCopyWgs, (rows + a.tile - 1) / a.tile * items);
  a.lanes = 1;
  while (a.lanes < a.row_bytes / unit && a.lanes < kThreads) a.lanes *= 2;
  switch (unit) {
    case 16: paged_copy_kernel<16><<<a.wgs, kThreads, 0, s>>>(a); break;
    case 8: paged_copy_kernel<8><<<a.wgs, kThreads, 0, s>>>(a); break;
    case 4: paged_copy_kernel<4><<<a.wgs, kThreads, 0, s>>>(a); break;
    case 2: paged_copy_kernel<2><<<a.wgs, kThreads, 0, s>>>(a); break;
    default: paged_copy_kernel<1><<<a.wgs, kThreads, 0, s>>>(a);
  }
  return hipGetLastError();
}

}  // namespace bnr

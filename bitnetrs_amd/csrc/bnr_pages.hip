// bnr_pages.hip -- gfx950 kernels of the paged cache's bookkeeping: pages for
// new tokens and the arrays that say where each goes (extend), pages given back
// (release), the tables of reordered beams, and rows copied between sequences.
#include "bnr_paged.h"

#include <algorithm>

namespace bnr {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;

typedef unsigned long long u64;

// Inclusive sums of two values over a workgroup's threads.
struct Two {
  u64 a, b;
};
__device__ __forceinline__ Two block_scan(Two v, Two *s_wave) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) {
    const u64 a = __shfl_up(v.a, k), b = __shfl_up(v.b, k);
    if (lane >= k) {
      v.a += a;
      v.b += b;
    }
  }
  __syncthreads();  // the sums before these have been read
  if (lane == 63) s_wave[wave] = v;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    v.a += s_wave[w].a;
    v.b += s_wave[w].b;
  }
  return v;
}

__device__ __forceinline__ int pages_of(long long rows, int page) { return (int)((rows + page - 1) / page); }

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

// Every workgroup adds up the whole batch for itself, so that one launch does
// it all and nothing is kept between launches: two loads a sequence, from L2.
// want(s): the sequence's two amounts; keep(s, first, taken): what precedes it on
// the two lines, and whether it has its place.  In order, up to the first
// sequence that goes past a limit: it and those behind it get nothing.
struct Shares {
  Two wave[kWaves];
  Two stop;
  int stopped;
};
template <class Want, class Keep>
__device__ __forceinline__ Two share_out(int n_seqs, u64 limit_a, u64 limit_b, Shares &sh, Want want, Keep keep) {
  const int tid = threadIdx.x;
  Two base = {0, 0};
  if (tid == 0) sh.stopped = 0;
  for (int s0 = 0; s0 < n_seqs; s0 += kThreads) {
    const int s = s0 + tid;
    Two v = {0, 0};
    if (s < n_seqs) v = want(s);
    const Two own = v;
    v = block_scan(v, sh.wave);
    v.a += base.a;
    v.b += base.b;
    const Two first = {v.a - own.a, v.b - own.b};
    const bool fits = v.a <= limit_a && v.b <= limit_b;
    if (!fits && first.a <= limit_a && first.b <= limit_b && !sh.stopped) {
      // the first that does not fit (sums only grow); there is one such thread
      sh.stop = first;
      sh.stopped = 1;
    }
    __syncthreads();
    const bool stopped = sh.stopped;
    if (s < n_seqs) keep(s, fits ? first : sh.stop, fits);
    if (stopped) {
      base = sh.stop;
      for (int r = s0 + kThreads + tid; r < n_seqs; r += kThreads) {
        want(r);
        keep(r, base, false);
      }
      break;
    }
    if (tid == kThreads - 1) sh.wave[0] = v;
    __syncthreads();
    base = sh.wave[0];
  }
  __syncthreads();
  return base;
}

// ---------------------------------------------------------------------------
// Extend.  16 bytes written for each token; a decode step's is latency: lengths
// and counts, sums, then a page and its entry.
// ---------------------------------------------------------------------------
__global__ __launch_bounds__(kThreads) void paged_extend_kernel(ExtendArgs a) {
  __shared__ int s_tok[kPagesMaxSeqs + 1], s_page[kPagesMaxSeqs + 1], s_len[kPagesMaxSeqs];
  __shared__ Shares sh;
  const long long room = a.table_stride * a.page;
  int free = *a.free_count;
  free = free < 0 ? 0 : free > a.free_cap ? a.free_cap : free;
  const auto want = [&](int s) {
    const long long len = max(a.lens[s], 0);
    long long n = max(a.fresh[s], 0);
    if (len + n > room) n = 0;
    s_len[s] = (int)len;
    return Two{n == 0 ? 0 : (u64)(pages_of(len + n, a.page) - pages_of(len, a.page)), (u64)n};
  };
  const auto keep = [&](int s, Two first, bool) {
    s_page[s] = (int)first.a;
    s_tok[s] = (int)first.b;
  };
  const Two all = share_out(a.n_seqs, (u64)free, (u64)a.n_tokens, sh, want, keep);
  const int pages = (int)all.a, tokens = (int)all.b, tid = threadIdx.x;
  if (tid == 0) {
    s_page[a.n_seqs] = pages;
    s_tok[a.n_seqs] = tokens;
  }
  __syncthreads();
  const long long first = (long long)blockIdx.x * kThreads + tid, step = (long long)gridDim.x * kThreads;
  for (long long e = first; e < pages; e += step) {
    const int s = part_of(s_page, a.n_seqs, (int)e);
    a.table[s * a.table_stride + pages_of(s_len[s], a.page) + ((int)e - s_page[s])] = a.free_pages[free - 1 - e];
  }
  for (long long i = first; i < a.n_tokens; i += step) {
    int seq = -1, at = -1;
    long long slot = -1;
    if (i < tokens) {
      seq = part_of(s_tok, a.n_seqs, (int)i);
      const int len = s_len[seq];
      at = len + ((int)i - s_tok[seq]);
      if (a.slots) {
        const int p = at / a.page, have = pages_of(len, a.page);
        const int page = p < have ? a.table[seq * a.table_stride + p]
                                  : a.free_pages[free - 1 - (s_page[seq] + p - have)];
        slot = page < 0 ? -1 : (long long)page * a.page + at % a.page;
      }
    }
    a.seqs[i] = seq;
    a.positions[i] = at;
    if (a.slots) a.slots[i] = slot;
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
  __shared__ int s_page[kPagesMaxSeqs + 1];
  __shared__ Shares sh;
  const long long room = a.table_stride * a.page;
  int free = *a.free_count;
  free = free < 0 ? 0 : free > a.free_cap ? a.free_cap : free;
  const auto kept = [&](int s) { return a.keep ? max(a.keep[s], 0) : 0; };
  const auto length = [&](int s) {
    const long long len = max(a.lens[s], 0);
    return len < room ? len : room;
  };
  const auto want = [&](int s) {
    const int n = a.which[s] ? pages_of(length(s), a.page) - kept(s) : 0;
    return Two{n > 0 ? (u64)n : 0, 0};
  };
  const auto keep = [&](int s, Two first, bool) { s_page[s] = (int)first.a; };
  const Two all = share_out(a.n_seqs, (u64)(a.free_cap - free), 0, sh, want, keep);
  const int pages = (int)all.a, tid = threadIdx.x;
  if (tid == 0) s_page[a.n_seqs] = pages;
  __syncthreads();
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
    const bool gone = a.which[s] && (s_page[s + 1] > s_page[s] || pages_of(length((int)s), a.page) <= kept((int)s));
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
// and scales as they are, in equal shares of all rows that are to be copied; L
// lanes share a row.  Bound by the rows' bytes, read and written.
// ---------------------------------------------------------------------------
constexpr int kCopyWgs = 4096, kCopyRows = 64;

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

template <int U>
__global__ __launch_bounds__(kThreads) void paged_copy_kernel(PagedCopyArgs a) {
  typedef typename Unit<U>::type T;
  const auto start = [&](int s) { return a.starts ? max(a.starts[s], 0) : 0; };
  const auto rows = [&](int s) {
    const int from = a.src[s], len = paged_len(a.lens[s], a.pool), first = start(s);
    return from < 0 || from >= a.n_seqs || from == s || first >= len ? 0 : len - first;
  };
  const int units = a.row_bytes / U, per = 2 * units;
  const char *pool[2] = {static_cast<const char *>(a.pool.k), static_cast<const char *>(a.pool.v)};
  PagedShare sh = paged_share(rows, a.n_seqs, a.pool.n_kv, a.tile, a.wgs);
  for (PagedPiece p; sh.next(rows, p);) {
    const int first = start(p.b), src = a.src[p.b], n = p.row1 - p.row0;
    for (int e = threadIdx.x; e < n * per; e += kThreads) {
      const int r = e / per, x = e - r * per, t = first + p.row0 + r;
      const long long from = paged_row(a.pool, src, p.h, t), to = paged_row(a.pool, p.b, p.h, t);
      if (from < 0 || to < 0 || from == to) continue;
      const int v = x >= units, at = x - v * units;
      char *base = const_cast<char *>(pool[v]);
      reinterpret_cast<T *>(base + to * a.row_bytes)[at] = reinterpret_cast<const T *>(base + from * a.row_bytes)[at];
    }
    if (a.scale_bytes == 0) continue;
    for (int e = threadIdx.x; e < n * 2 * a.scale_bytes; e += kThreads) {
      const int r = e / (2 * a.scale_bytes), x = e - r * 2 * a.scale_bytes, t = first + p.row0 + r;
      const long long from = paged_row(a.pool, src, p.h, t), to = paged_row(a.pool, p.b, p.h, t);
      if (from < 0 || to < 0 || from == to) continue;
      const int v = x >= a.scale_bytes, at = x - v * a.scale_bytes;
      unsigned char *sc = a.pool.k_exps ? (v ? a.pool.v_exps : a.pool.k_exps)
                                        : reinterpret_cast<unsigned char *>(v ? a.pool.v_scales : a.pool.k_scales);
      sc[to * a.scale_bytes + at] = sc[from * a.scale_bytes + at];
    }
  }
}

}  // namespace

static unsigned grid_for(long long n) {
  return (unsigned)std::max<long long>(1, std::min<long long>((n + 2 * kThreads - 1) / (2 * kThreads), 2048));
}

hipError_t launch_paged_extend(const ExtendArgs &a, hipStream_t s) {
  paged_extend_kernel<<<grid_for(a.n_tokens), kThreads, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_paged_release(const ReleaseArgs &a, hipStream_t s) {
  const long long pages = std::min<long long>(a.n_seqs * a.table_stride, a.free_cap);
  paged_release_kernel<<<grid_for(pages), kThreads, 0, s>>>(a);
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

// bnr_paged_index.h -- where the rows of the paged KV cache lie and how a
// launch's work is cut into equal shares: integer code that the kernels run and
// the tests check on the host.
#pragma once

#include "bnr_internal.h"

namespace bnr {

// ---------------------------------------------------------------------------
// Rows.
// ---------------------------------------------------------------------------
// A sequence's length as the table can hold it.
__host__ __device__ inline int paged_len(int len, const PagedPool &p) {
  const long long most = p.table_stride * p.page;  // at most 2^30, checked by the host
  return len < 0 ? 0 : len > most ? (int)most : len;
}

// The page of row t of a sequence, or -1 where there is none.  0 <= t < stride * page.
__host__ __device__ inline int paged_page(const PagedPool &p, long long seq, int t) {
  const int page = p.table[seq * p.table_stride + t / p.page];
  return page < 0 || page >= p.n_pages ? -1 : page;
}

// Row t of kv head h, counted in rows of the pool; -1 where its page is not there.
__host__ __device__ inline long long paged_row(const PagedPool &p, long long seq, int h, int t) {
  const int page = paged_page(p, seq, t);
  if (page < 0) return -1;
  return ((long long)page * p.n_kv + h) * p.page + t % p.page;
}

// Rows of a token of an append launch.
__host__ __device__ inline int append_rows(const PagedAppendArgs &a) {
  return (a.q ? a.n_heads : 0) + 2 * a.pool.n_kv;
}

// Row j of a token of an append launch: its q rows, its k rows, its v rows.
struct AppendRow {
  float *out;           // q rows: where the rotated row goes
  const float *cos, *sin;  // null: not rotated
  void *codes;          // k and v rows: the pool, the row's first element in it,
  long long at;
  float *scale;         // and where its scale goes
  unsigned char *exps;  // or its groups' exponents
};
__host__ __device__ inline const float *append_in(const PagedAppendArgs &a, long long i, int j) {
  const int nq = a.q ? a.n_heads : 0, kv = a.pool.n_kv;
  return j < nq        ? a.q + (i * nq + j) * a.pool.d
         : j < nq + kv ? a.k + (i * kv + (j - nq)) * a.pool.d
                       : a.v + (i * kv + (j - nq - kv)) * a.pool.d;
}

// False: nothing to do (a token whose position or sequence is outside the
// table, or outside the rotation's tables; a page that is not there).
__host__ __device__ inline bool append_row(const PagedAppendArgs &a, long long i, int j,
                                           AppendRow &r) {
  const PagedPool &p = a.pool;
  const int nq = a.q ? a.n_heads : 0;
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
    r.out = a.q_out + (i * nq + j) * p.d;
    return true;
  }
  const bool is_v = j >= nq + p.n_kv;
  const int h = j - nq - (is_v ? p.n_kv : 0);
  const long long at = paged_row(p, seq, h, pos);
  if (at < 0) return false;
  r.codes = is_v ? p.v : p.k;
  r.at = at * p.d;
  float *sc = is_v ? p.v_scales : p.k_scales;
  r.scale = sc ? sc + at : nullptr;
  unsigned char *ex = is_v ? p.v_exps : p.k_exps;
  r.exps = ex ? ex + at * paged_groups4(p.d) : nullptr;
  return true;
}

// ---------------------------------------------------------------------------
// Shares of a launch.  Sequence b has ceil(rows(b) / tile) units for each of
// its `items` heads; all units in order are one line, and workgroup w takes
// units w * per + min(w, rest) .. of it (total = per * wgs + rest).  A
// workgroup's share is a run of pieces, each of one item: at most its first
// and its last piece belong to items that other workgroups share.  Nothing
// about the lengths is known on the host, so a captured launch serves every
// later step, and ragged batches are balanced to one unit.  The host picks
// `tile` so that all units that the table has room for fit 31 bits.
// ---------------------------------------------------------------------------
struct PagedPiece {
  int b, h;        // sequence, item
  int row0, row1;  // rows of it
  unsigned item0, item1;  // the item's units
};

struct PagedShare {
  unsigned at, end;     // units left to this workgroup
  unsigned item0;       // first unit of the item at `at`
  unsigned per, rest, wg;
  int b, h, items, tile, len, batch;
  unsigned n;           // units of an item of sequence b

  // The part of `total` units that workgroup `id` has where `used` of the
  // launch's workgroups share them; none for the others.
  __host__ __device__ void take(unsigned total, unsigned id, unsigned used, int batch_, int items_,
                                unsigned tile_) {
    wg = id;
    batch = batch_;
    per = total / used;
    rest = total - per * used;
    items = items_;
    tile = (int)tile_;
    at = id < used ? id * per + (id < rest ? id : rest) : total;
    end = id < used ? at + per + (id < rest ? 1 : 0) : total;
  }
  // The workgroup that has unit t.
  __host__ __device__ unsigned wg_of(unsigned t) const {
    const unsigned big = rest * (per + 1);
    return t < big ? t / (per + 1) : rest + (t - big) / per;
  }
  // The next piece.
  template <class Rows>
  __host__ __device__ bool next(Rows rows, PagedPiece &p) {
    if (at >= end) return false;
    if (at == item0 + n) {  // past the item before
      item0 = at;
      if (++h == items) {
        h = 0;
        do {
          if (++b >= batch) return false;  // not reached: `end` lies in the last sequence with a row
          len = rows(b);
        } while (len == 0);
        n = (unsigned)(len + tile - 1) / (unsigned)tile;
      }
    }
    p.b = b;
    p.h = h;
    p.item0 = item0;
    p.item1 = item0 + n;
    const unsigned to = p.item1 < end ? p.item1 : end;
    p.row0 = (int)((at - item0) * (unsigned)tile);
    const unsigned r1 = (to - item0) * (unsigned)tile;
    p.row1 = r1 < (unsigned)len ? (int)r1 : len;
    at = to;
    return true;
  }
};

// ---------------------------------------------------------------------------
// Joins.  The item on workgroups w0 .. w1 has a piece of each: w0's is its
// last, in slot 2 w0 + 1, the others' their first, in slot 2 w.  A step of a
// join takes `count` states from slots 2 (base + j * stride) (one higher for
// w0's): all pieces at once, or kJoinGroup neighbours, whose joined state goes
// to the first one's slot of a second array, and then those states.  A slot is
// one piece's, so a group's ticket may go by its first slot; of the items that
// a workgroup starts only the last can go on in the next, so an item's may go
// by w0.
// ---------------------------------------------------------------------------
constexpr int kJoinGroup = 16;
struct JoinStep {
  unsigned base, stride;
  int count;
  bool last;  // the item's outputs come out, not a group's state
  __host__ __device__ int slot(int j, unsigned w0) const {
    const unsigned w = base + (unsigned)j * stride;
    return (int)(2 * w + (w == w0 ? 1 : 0));
  }
  __host__ __device__ unsigned ticket(unsigned w0) const {
    return last ? w0 : (unsigned)kPagedMaxWgs + (unsigned)slot(0, w0);
  }
};

// The step of workgroup wg's piece.  A workgroup loads `at_once` states of an
// output in one go, `rounds` times over for all outputs: past four goes the
// pieces are grouped.  One token over 30000 bf16 rows of one kv head with 16
// query heads: 45.6 us with every piece joined at once, 24.5 with shares kept
// large so that pieces are few, 16.6 with groups; over 85937 f32 rows of one
// with 12 of 80: 57.5 with large shares, 32.0 with groups.  Up to 2 % more where
// nothing is grouped (15 int8 sequences 44.2 -> 45.1, 4096 bf16 rows 8.9 -> 9.0).
__host__ __device__ inline JoinStep join_start(unsigned w0, unsigned w1, unsigned wg, int at_once, int rounds) {
  const int n = (int)(w1 - w0) + 1;
  if ((n + at_once - 1) / at_once * rounds <= 4 || n <= kJoinGroup) return JoinStep{w0, 1, n, true};
  const unsigned base = wg - (wg - w0) % kJoinGroup;
  const int left = (int)(w1 - base) + 1;
  return JoinStep{base, 1, left < kJoinGroup ? left : kJoinGroup, false};
}

// The step of the groups' states.
__host__ __device__ inline JoinStep join_groups(unsigned w0, unsigned w1) {
  return JoinStep{w0, kJoinGroup, (int)(w1 - w0) / kJoinGroup + 1, true};
}

}  // namespace bnr

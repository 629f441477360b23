// Host check of the paged KV cache's index code (bnr_paged_index.h), which the
// kernels run as it stands: every row lies inside the pool whatever the table,
// positions and sequences hold, and shares of any launch cover its line once,
// with the workgroups of an item and its ticket as the join takes them to be.
// Prints "ok" and what it covered; a failed check names itself and ends it.
#include "../../bitnetrs_amd/csrc/bnr_paged_index.h"

#include <algorithm>
#include <climits>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <set>
#include <vector>

using namespace bnr;

#define CHECK(x)                                                \
  do {                                                          \
    if (!(x)) {                                                 \
      std::printf("failed: %s (line %d)\n", #x, __LINE__);      \
      std::exit(1);                                             \
    }                                                           \
  } while (0)

// What paged_share finds with the lanes of a wave, one sequence after another.
template <class Rows>
static PagedShare share_of(Rows rows, int batch, int items, unsigned tile, unsigned wg, unsigned wgs) {
  unsigned total = 0;
  for (int b = 0; b < batch; ++b) total += ((unsigned)rows(b) + tile - 1) / tile * (unsigned)items;
  PagedShare s{};
  s.take(total, wg, wgs, batch, items, tile);
  CHECK(s.at <= s.end && s.end <= total);
  if (s.at >= s.end) return s;
  unsigned before = 0;
  for (int b = 0;; ++b) {
    CHECK(b < batch);
    s.len = rows(b);
    s.n = ((unsigned)s.len + tile - 1) / tile;
    if (s.at < before + s.n * (unsigned)items) {
      s.b = b;
      break;
    }
    before += s.n * (unsigned)items;
  }
  s.h = (int)((s.at - before) / s.n);
  s.item0 = before + (unsigned)s.h * s.n;
  return s;
}

// The steps that join an item's pieces: each piece is taken once, in order, by
// the group that all its workgroups take it to be in; each group's state once.
static void joins(unsigned w0, unsigned w1, int at_once, int turns, std::set<unsigned> &group_ticket) {
  const auto piece = [&](unsigned w) { return (int)(2 * w + (w == w0 ? 1 : 0)); };
  std::vector<int> groups;  // slots of their states
  unsigned next = w0;
  for (unsigned w = w0; w <= w1; ++w) {
    const JoinStep c = join_start(w0, w1, w, at_once, turns);
    CHECK(c.count >= 1 && c.base <= w && w < c.base + (unsigned)c.count && c.base + (unsigned)c.count <= w1 + 1);
    CHECK(c.last ? c.base == w0 && c.count == (int)(w1 - w0) + 1 && c.ticket(w0) == w0
                 : c.count <= kJoinGroup);
    if (w != next) continue;  // the same group as the piece before
    for (int j = 0; j < c.count; ++j) CHECK(c.slot(j, w0) == piece(w + (unsigned)j));
    next = w + (unsigned)c.count;
    if (c.last) return;
    CHECK(c.ticket(w0) >= (unsigned)kPagedMaxWgs && c.ticket(w0) < (unsigned)kPagedTickets);
    CHECK(group_ticket.insert(c.ticket(w0)).second);
    groups.push_back(c.slot(0, w0));
  }
  CHECK(next == w1 + 1);
  const JoinStep c = join_groups(w0, w1);
  CHECK(c.last && c.count == (int)groups.size() && c.ticket(w0) == w0);
  for (int j = 0; j < c.count; ++j) CHECK(c.slot(j, w0) == groups[(size_t)j]);
}

static long long shares(std::mt19937 &rng) {
  long long pieces = 0;
  for (int round = 0; round < 400; ++round) {
    const int batch = 1 + (int)(rng() % (round % 3 ? 7 : 130)), items = 1 + (int)(rng() % 9);
    const unsigned tile = 64u << rng() % 3;
    const int top = round % 5 == 0 ? 3 : round % 5 == 1 ? 1 << 20 : 5000;
    std::vector<int> len((size_t)batch);
    for (int &n : len) n = rng() % 4 ? (int)(rng() % (unsigned)top) : 0;
    const auto rows = [&](int b) { return len[(size_t)b]; };
    unsigned room = 0;
    for (int n : len) room += ((unsigned)n + tile - 1) / tile * (unsigned)items;
    const unsigned wgs = 1 + rng() % (round % 2 ? 512u : std::max(1u, std::min(512u, room + 5)));
    unsigned line = 0;              // units given out so far
    std::set<unsigned> first;       // first workgroups of shared items
    std::set<unsigned> group_ticket;  // of groups of pieces
    const int at_once = 8 << rng() % 4, turns = 1 + (int)(rng() % 3);
    std::vector<std::vector<long long>> next((size_t)batch, std::vector<long long>((size_t)items, 0));
    // workgroups past the `wgs` that share the line have nothing
    for (unsigned wg = 0; wg < wgs + 20; ++wg) {
      PagedShare s = share_of(rows, batch, items, tile, wg, wgs);
      CHECK(s.at == line);
      CHECK(wg < wgs || s.at == s.end);
      const unsigned end = s.end;
      unsigned unfinished = 0;
      for (PagedPiece p; s.next(rows, p); ++pieces) {
        CHECK(p.b >= 0 && p.b < batch && p.h >= 0 && p.h < items);
        // rows follow each other within an item, from 0 to its end
        CHECK(p.row0 == next[(size_t)p.b][(size_t)p.h] && p.row0 < p.row1 && p.row1 <= len[(size_t)p.b]);
        CHECK(p.row0 % (int)tile == 0);
        next[(size_t)p.b][(size_t)p.h] = p.row1;
        const unsigned units = ((unsigned)p.row1 - (unsigned)p.row0 + tile - 1) / tile;
        const unsigned unit = p.item0 + (unsigned)p.row0 / tile;
        CHECK(unit == line);
        line += units;
        CHECK(p.item1 - p.item0 == ((unsigned)len[(size_t)p.b] + tile - 1) / tile);
        const unsigned w0 = s.wg_of(p.item0), w1 = s.wg_of(p.item1 - 1);
        CHECK(w0 <= wg && wg <= w1 && w1 < wgs);
        CHECK((w0 == w1) == (p.row0 == 0 && p.row1 == len[(size_t)p.b]));
        if (w0 != w1) {
          // a piece that others share: in the workgroup's slot 2 wg + 1 if it starts the item, else 2 wg
          const unsigned slot = wg == w0 ? 2u : 1u;
          CHECK(!(unfinished & slot));
          unfinished |= slot;
          if (wg == w0) {
            CHECK(first.insert(w0).second);  // the ticket is this item's alone
            joins(w0, w1, at_once, turns, group_ticket);
          }
        }
      }
      CHECK(line == end);
    }
    CHECK(line == room);
    for (int b = 0; b < batch; ++b)
      for (int h = 0; h < items; ++h) CHECK(next[(size_t)b][(size_t)h] == len[(size_t)b]);
  }
  return pieces;
}

static long long rows(std::mt19937 &rng) {
  long long checked = 0;
  const int odd[] = {INT_MIN, INT_MIN + 1, -2, -1, 0, 1, 2, 3, 7, 8, INT_MAX - 1, INT_MAX};
  for (int round = 0; round < 200; ++round) {
    PagedAppendArgs a{};
    PagedPool &p = a.pool;
    p.n_pages = 1 + (int)(rng() % 9);
    p.page = 1 + (int)(rng() % 33);
    p.n_kv = 1 + (int)(rng() % 4);
    p.d = 2 + 2 * (int)(rng() % 8);
    p.table_stride = 1 + (long long)(rng() % 5);
    a.n_heads = p.n_kv * 3;
    a.n_tokens = 40;
    a.n_seqs = 1 + (long long)(rng() % 4);
    a.n_positions = (long long)(rng() % 200);
    const long long room = (long long)p.n_pages * p.n_kv * p.page;
    // the exact sizes, so that an access outside them is one of a vector's
    std::vector<int> table((size_t)(a.n_seqs * p.table_stride)), pos(40), seq(40);
    std::vector<float> q(40u * (size_t)(a.n_heads * p.d)), kv(40u * (size_t)(p.n_kv * p.d));
    std::vector<float> tab((size_t)(a.n_positions * p.d / 2) + 1), pool((size_t)(room * p.d)), sc((size_t)room);
    const auto any = [&](int most) {
      return rng() % 2 ? odd[rng() % (sizeof odd / sizeof *odd)] : (int)(rng() % (unsigned)most);
    };
    for (int &x : table) x = any(p.n_pages + 1);
    for (int &x : pos) x = any((int)p.table_stride * p.page + 3);
    for (int &x : seq) x = any((int)a.n_seqs + 1);
    p.table = table.data();
    p.k = p.v = pool.data();
    p.k_scales = p.v_scales = round % 2 ? sc.data() : nullptr;
    a.q = round % 3 ? q.data() : nullptr;
    a.q_out = q.data();
    a.k = a.v = kv.data();
    a.positions = pos.data();
    a.seqs = round % 5 ? seq.data() : nullptr;
    if (round % 4) a.cos_tab = a.sin_tab = tab.data();
    for (long long i = 0; i < a.n_tokens; ++i)
      for (int j = 0; j < append_rows(a); ++j) {
        const float *in = append_in(a, i, j);
        const bool is_q = a.q && j < a.n_heads;
        CHECK(is_q ? in >= q.data() && in + p.d <= q.data() + q.size()
                   : in >= kv.data() && in + p.d <= kv.data() + kv.size());
        AppendRow r;
        const long long s = a.seqs ? seq[(size_t)i] : i;
        const int t = pos[(size_t)i];
        const bool in_table = t >= 0 && t < p.table_stride * p.page && s >= 0 && s < a.n_seqs &&
                              (!a.cos_tab || t < a.n_positions);
        ++checked;
        if (!append_row(a, i, j, r)) {
          CHECK(!in_table || (!is_q && paged_page(p, s, t) < 0));
          continue;
        }
        CHECK(in_table);
        if (r.cos) CHECK(r.cos >= tab.data() && r.cos + p.d / 2 <= tab.data() + a.n_positions * (p.d / 2));
        CHECK(!r.cos == !(a.cos_tab && j < (a.q ? a.n_heads : 0) + p.n_kv));
        if (is_q) {
          CHECK(r.out >= q.data() && r.out + p.d <= q.data() + q.size());
        } else {
          CHECK(!r.out && r.codes == p.k && r.at >= 0 && r.at + p.d <= room * p.d);
          CHECK(!p.k_scales || (r.scale >= sc.data() && r.scale < sc.data() + room));
        }
      }
    for (long long s = 0; s < a.n_seqs; ++s)
      for (int len : odd) {
        const int n = paged_len(len, p);
        CHECK(n >= 0 && n <= p.table_stride * p.page && (len < 0 ? n == 0 : n <= len));
        for (int t = 0; t < n; ++t)
          for (int h = 0; h < p.n_kv; ++h, ++checked) {
            const long long at = paged_row(p, s, h, t);
            CHECK(at >= -1 && at < room);
          }
      }
  }
  return checked;
}

int main() {
  std::mt19937 rng(20240711);
  const long long pieces = shares(rng), at = rows(rng);
  std::printf("ok: %lld pieces, %lld rows\n", pieces, at);
  return 0;
}

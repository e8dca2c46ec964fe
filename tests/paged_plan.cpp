// The paged attention's plans on the host: the kernels' own code with an array of 64 in a register's place.
// Reads a call (heads, head size, page, table, lengths) and checks that the shares, or units, cover every key step of
// every tile once, and that partial sums have records of their own.
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <map>
#include <tuple>
#include <vector>

#include "paged_attend.h"

using namespace spectra;

struct Lanes {
  int v[64];
  Lanes(int x = 0) {
    for (int& e : v) e = x;
  }
};
template <typename F>
static Lanes each(const Lanes& a, const Lanes& b, F f) {
  Lanes r;
  for (int i = 0; i < 64; ++i) r.v[i] = f(a.v[i], b.v[i]);
  return r;
}
// (sums and products wrap, as a register's do)
static Lanes operator+(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return (int)((unsigned)x + (unsigned)y); }); }
static Lanes operator-(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return (int)((unsigned)x - (unsigned)y); }); }
static Lanes operator*(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return (int)((unsigned)x * (unsigned)y); }); }
static Lanes operator/(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return x / y; }); }
static Lanes operator>>(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return x >> y; }); }
static Lanes operator<(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return (int)(x < y); }); }
static Lanes operator<=(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return (int)(x <= y); }); }
static Lanes operator>(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return (int)(x > y); }); }

struct HostWave {
  typedef Lanes Int;
  static Lanes read(const int* p, const Lanes& at) {
    return each(at, at, [p](int x, int) { return p[x]; });
  }
  static int load(const int* p) { return *p; }
  static int uniform(int v) { return v; }
  static Lanes least(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return x < y ? x : y; }); }
  static Lanes most(const Lanes& a, const Lanes& b) { return each(a, b, [](int x, int y) { return x > y ? x : y; }); }
  static Lanes select(const Lanes& c, const Lanes& a, const Lanes& b) {
    Lanes r;
    for (int i = 0; i < 64; ++i) r.v[i] = c.v[i] ? a.v[i] : b.v[i];
    return r;
  }
  static Lanes quotient(const Lanes& a, const Lanes& b) {
    return each(a, b, [](int x, int y) { return (int)((unsigned)x / (unsigned)y); });
  }
  static uint64_t above(const Lanes& a, const Lanes& b) {
    uint64_t r = 0;
    for (int i = 0; i < 64; ++i) r |= (uint64_t)(a.v[i] > b.v[i]) << i;
    return r;
  }
  static int of(const Lanes& v, int lane) { return v.v[lane]; }
  static Lanes scan(const Lanes& v) {
    Lanes r = v;
    for (int i = 1; i < 64; ++i) r.v[i] = (int)((unsigned)r.v[i] + (unsigned)r.v[i - 1]);
    return r;
  }
  static float product(const Lanes& a, const Lanes& b) {  // partners 32, 16, .. apart, as the wave adds them
    float s[64], t[64];
    for (int i = 0; i < 64; ++i) s[i] = (float)a.v[i] * (float)b.v[i];
    for (int d = 32; d > 0; d /= 2) {
      for (int i = 0; i < 64; ++i) t[i] = s[i] + s[i ^ d];
      memcpy(s, t, sizeof s);
    }
    return s[0];
  }
};

#define CHECK(c, ...)                 \
  do {                                \
    if (!(c)) {                       \
      printf("%s: ", #c);             \
      printf(__VA_ARGS__);            \
      printf("\n");                   \
      return 1;                       \
    }                                 \
  } while (0)

struct Call {
  int kind, heads, hd, window, g;
  PagedKv kv;
  PagedScore sc;
  std::vector<int> n, lens, starts, prefix;
};

// The tiles that the call has, by sequence.
static int64_t tiles_of(const Call& c, int b, int rows) { return ((int64_t)c.n[b] * c.g + rows - 1) / rows; }

static int check_few(const Call& c, const PagedGrid& grid, const Lanes& lane) {
  struct Part {
    int b, kvh, tile, t0, steps, from, to, record;
  };
  std::vector<Part> parts;
  PagedLine line = {};
  const int groups = (int)grid.units;
  int64_t most = 0;
  int end = 0;
  for (int w = 0; w < groups; ++w) {
    PagedWalk<HostWave> walk(c.kv, c.g, grid.rows, grid.rows / c.g, kFewKeys, c.sc, w, groups, grid.wide, lane);
    if (w > 0) CHECK(walk.line.total == line.total && walk.line.each == line.each, "share %d has another line", w);
    line = walk.line;
    CHECK(line.begin == end || line.begin == line.end, "share %d begins at %d, not %d", w, line.begin, end);
    end = line.end > end ? line.end : end;
    most = std::max<int64_t>(most, line.end - line.begin);
    PagedPart p;
    for (int x = line.begin; x < line.end && walk.part(x, p); x = p.t0 + p.to) {
      CHECK(p.t0 + p.from == x && p.from < p.to && p.to <= p.steps, "part %d..%d of %d at %d", p.from, p.to, p.steps, x);
      CHECK(p.seq.q0 == c.starts[p.b] && p.seq.n == c.n[p.b] && p.seq.len == c.lens[p.b], "sequence %d", p.b);
      CHECK(p.prefix == (c.prefix.empty() ? 0 : c.prefix[p.b]), "prefix of %d", p.b);
      const bool whole = p.from == 0 && p.to == p.steps;
      parts.push_back({p.b, p.kvh, p.tile, p.t0, p.steps, p.from, p.to, whole ? -1 : line.record(w, x)});
    }
  }
  CHECK(end == line.total, "shares end at %d of %d", end, line.total);
  int64_t want = 0;
  for (int b = 0; b < (int)c.n.size(); ++b) want += c.kv.kv_heads * tiles_of(c, b, grid.rows);
  std::vector<char> used(2 * groups, 0);
  int64_t tiles = 0;
  int at = 0;
  int64_t last = -1;  // tiles come by sequence, KV head, tile
  for (size_t i = 0; i < parts.size();) {
    const Part& f = parts[i];
    CHECK(f.t0 == at && f.from == 0, "tile at %d, expected at %d", f.t0, at);
    const int64_t name = ((int64_t)f.b * c.kv.kv_heads + f.kvh) * ((int64_t)1 << 32) / 4 + f.tile;
    CHECK(name > last && f.tile < tiles_of(c, f.b, grid.rows), "tile %d of KV head %d of %d", f.tile, f.kvh, f.b);
    last = name;
    const PagedCut cut(line, f.t0, f.steps);
    int to = 0, n = 0;
    for (; i < parts.size() && parts[i].t0 == f.t0; ++i, ++n) {
      const Part& p = parts[i];
      CHECK(p.from == to && p.steps == f.steps, "a gap in the tile at %d", f.t0);
      to = p.to;
      if (p.record < 0) continue;
      CHECK(p.record == cut.record(n) && p.record < 2 * groups && !used[p.record], "record %d", p.record);
      used[p.record] = 1;
    }
    CHECK(to == f.steps && (n == cut.pieces || f.t0 + f.steps > line.total), "the tile at %d ends at %d of %d", f.t0, to, f.steps);
    at = f.t0 + f.steps;
    ++tiles;
  }
  CHECK(at == line.total, "tiles end at %d of %d", at, line.total);
  CHECK(tiles == want, "%lld tiles of %lld", (long long)tiles, (long long)want);
  printf("ok few: %lld tiles of %d rows, %d steps%s, at most %lld a share\n", (long long)tiles, grid.rows, line.total,
         grid.wide ? " (wide)" : "", (long long)most);
  return 0;
}

static int check_many(const Call& c, const PagedGrid& grid, const Lanes& lane) {
  std::map<std::tuple<int, int, int>, std::vector<int>> seen;  // a tile's pieces
  std::vector<char> used(kManySlots, 0);
  int64_t want = 0, units = 0;
  for (int b = 0; b < (int)c.n.size(); ++b) want += c.kv.kv_heads * tiles_of(c, b, grid.rows);
  bool past = false;
  for (int64_t u = 0; u < grid.units + 64; ++u) {
    PagedUnit un;
    if (!paged_unit<HostWave>(c.kv, c.g, grid.rows, kManyKeys, kManyMinKeys / kManyKeys, kManyTarget, kManySlots, c.sc, (int)u,
                              lane, un)) {
      past = true;
      continue;
    }
    CHECK(!past && u < grid.units, "unit %lld past the grid of %lld", (long long)u, (long long)grid.units);
    ++units;
    CHECK(un.seq.q0 == c.starts[un.b] && un.seq.n == c.n[un.b] && un.seq.len == c.lens[un.b], "sequence %d", un.b);
    CHECK(un.tile >= 0 && un.tile < tiles_of(c, un.b, grid.rows) && un.kvh < c.kv.kv_heads, "tile %d of %d", un.tile, un.b);
    auto& p = seen[{un.b, un.kvh, un.tile}];
    if (p.empty()) p.assign(un.pieces, 0);
    CHECK((int)p.size() == un.pieces && un.piece < un.pieces && !p[un.piece], "piece %d of %d", un.piece, un.pieces);
    p[un.piece] = 1;
    if (un.pieces > 1) {
      CHECK(un.slot >= 0 && un.slot < kManySlots && !used[un.slot], "slot %d", un.slot);
      used[un.slot] = 1;
    }
  }
  CHECK((int64_t)seen.size() == want, "%lld tiles of %lld", (long long)seen.size(), (long long)want);
  for (auto& t : seen)
    for (char x : t.second) CHECK(x, "a piece of sequence %d is missing", std::get<0>(t.first));
  printf("ok many: %lld tiles of %d rows, %lld units\n", (long long)want, grid.rows, (long long)units);
  return 0;
}

// Regions of random runs in a small memory, against marks of their bytes.
static int check_meet(unsigned seed) {
  auto next = [&](int n) { return (int)(((seed = seed * 1664525u + 1013904223u) >> 8) % (unsigned)n); };
  int both[2] = {0, 0};
  for (int it = 0; it < 200000; ++it) {
    PagedRegion r[2];
    const int64_t one = 1 + next(24);
    uint8_t marks[2][1024] = {};
    for (int i = 0; i < 2; ++i) {
      const int64_t step = next(3) ? one + 8 : 1 + next(40), n = 1 + next(12);
      r[i] = {"", (const void*)(uintptr_t)(64 + next(200)), 1 + next((int)step), next(8) ? step : 0, n};
      if (r[i].step == 0) r[i].n = 1;
      for (int64_t j = 0; j < r[i].n; ++j)
        for (int64_t k = 0; k < r[i].bytes; ++k) marks[i][(uintptr_t)r[i].at + j * r[i].step + k] = 1;
    }
    bool want = false;
    for (int k = 0; k < 1024; ++k) want |= marks[0][k] && marks[1][k];
    CHECK(paged_meet(r[0], r[1]) == want && paged_meet(r[1], r[0]) == want, "%zu + %lld of %lld x %lld, %zu + %lld of %lld x %lld",
          (size_t)r[0].at, (long long)r[0].bytes, (long long)r[0].step, (long long)r[0].n, (size_t)r[1].at, (long long)r[1].bytes,
          (long long)r[1].step, (long long)r[1].n);
    ++both[want];
  }
  CHECK(both[0] > 10000 && both[1] > 10000, "%d apart, %d not", both[0], both[1]);
  printf("ok\n");
  return 0;
}

int main(int argc, char** argv) {
  if (argc > 1) return check_meet((unsigned)atoi(argv[1]));
  Call c = {};
  int kvh, page, batch, width, pad;
  if (scanf("%d %d %d %d %d %d %d %d %d", &c.kind, &c.heads, &kvh, &c.hd, &page, &width, &batch, &pad, &c.window) != 9) return 2;
  c.g = c.heads / kvh;
  c.n.resize(batch);
  c.lens.resize(batch);
  c.starts.assign(batch + 1, 0);
  int most = 0;
  for (int b = 0; b < batch; ++b) {
    int pre;
    if (scanf("%d %d %d", &c.n[b], &c.lens[b], &pre) != 3) return 2;
    if (pre >= 0) c.prefix.push_back(pre);
    c.starts[b + 1] = c.starts[b] + c.n[b];
    most = std::max(most, c.lens[b]);
  }
  int shift = 0;
  while ((1 << shift) < page) ++shift;
  c.kv.q_start = c.starts.data();
  c.kv.lens = c.lens.data();
  c.kv.batch = batch;
  c.kv.kv_heads = kvh;
  c.kv.page_shift = shift;
  c.kv.table_width = width > 0 ? width : (most + page - 1) / page;
  c.kv.tokens = c.starts[batch] + pad;
  c.sc.window = c.window;
  c.sc.prefix = c.prefix.empty() ? nullptr : c.prefix.data();
  Lanes lane;
  for (int i = 0; i < 64; ++i) lane.v[i] = i;
  const PagedGrid grid = paged_grid(c.kv, c.kv.tokens, c.g, c.kind, c.hd);
  if (grid.tiles >= (1LL << 28) || (int64_t)c.kv.table_width * page >= (1LL << 30)) return 3;  // (the entry refuses it)
  return grid.rows >= 64 ? check_many(c, grid, lane) : check_few(c, grid, lane);
}

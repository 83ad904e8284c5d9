// How the tiles of several products are dealt out to the blocks of a launch: host code alone, which a test
// compiles by itself.  Every tile's K is taken once, by one unit or by parts of it in order whose sums have
// slots of their own in the workspace.
#ifndef AD_B200_SCHEDULE_H
#define AD_B200_SCHEDULE_H

#include <algorithm>
#include <cstddef>

namespace adgemm {

constexpr int BK = 64;  // elements of K a stage: 128 bytes, the swizzle's width
constexpr int MAX_GROUPS = 4;

// The three tilings: rows and columns, blocks, and measured us for 64 elements of K
// (with the clocks that large products leave; 2047 x 50001 over 1024 took 152, 250
// and 453 us).
struct Tiling {
  int m, n, ctas;
  double us;
};
constexpr Tiling TILINGS[3] = {{256, 256, 2, 0.38}, {128, 128, 1, 0.36}, {128, 64, 1, 0.33}};

// m, n, k and k0 of a product: k0 of K in its first operands (k where there is one pair), the rest in its second.
template <typename P>
int kblocks_of(const P& p) {
  return static_cast<int>((p.k0 + BK - 1) / BK + (p.k - p.k0 + BK - 1) / BK);
}

constexpr int MAX_WORKERS = 256;
constexpr int SMALL_LIST = 256, LARGE_LIST = 2048;  // units of a launch: 3 and 25 KB of parameters
// 64 elements of K that a part of a tile has at least (anything from 2 to 12 takes the same time, within the
// noise, for gradients of 600 to 8000 rows of 512 to 2048).
constexpr int LEAST = 6;

struct Listed {
  unsigned where;  // group, row and column of the tile
  unsigned short kb0, kb1;
};
inline unsigned pack_where(int group, int row, int col) {
  return static_cast<unsigned>(group) << 30 | static_cast<unsigned>(row) << 15 | static_cast<unsigned>(col);
}
// A tile that was cut: its parts' sums lie in slots one behind another, in the order of K.
struct Cut {
  unsigned where;
  short slot, parts;
};
// Elements of partial sums in 32 bits that a schedule may use, whatever its tiling: of two parts for each
// pair of blocks of 256 x 256, as there are no more parts than workers and cut tiles, and fewer of these than workers.
constexpr size_t partial_elements(int sms) { return static_cast<size_t>(2) * (sms / 2) * 256 * 256; }

struct Schedule {
  int tiling, workers, units, cuts;
  double us;
  Listed unit[LARGE_LIST];
  short slot[LARGE_LIST], first[MAX_WORKERS + 1];
  Cut cut[MAX_WORKERS];
};

// Deals the tiles of all products out to `workers`; false when there are too many.
template <typename P>
bool make_schedule(const P* p, int count, int tiling, int workers, Schedule& s) {
  const Tiling& t = TILINGS[tiling];
  workers = std::min(workers, MAX_WORKERS);
  s.tiling = tiling, s.workers = workers, s.cuts = 0;
  long long all = 0, total = 0;
  int order[MAX_GROUPS], rows[MAX_GROUPS], cols[MAX_GROUPS], kb[MAX_GROUPS];
  for (int g = 0; g < count; ++g) {
    const long long r = (p[g].m + t.m - 1) / t.m, c = (p[g].n + t.n - 1) / t.n;
    if (r > 0x7fff || c > 0x7fff || p[g].k > 64ll * 65000) return false;
    rows[g] = static_cast<int>(r), cols[g] = static_cast<int>(c), kb[g] = kblocks_of(p[g]);
    all += r * c, total += r * c * kb[g];
  }
  if (all + 3 * workers > LARGE_LIST) return false;
  // a unit's worker, besides what goes to the device
  static_assert(LARGE_LIST < 0x7fff, "");
  struct Piece {
    Listed l;
    short worker, slot;
  };
  Piece piece[LARGE_LIST];
  int pieces = 0, slots = 0, load[MAX_WORKERS] = {}, most = 0;
  // The height that all would have if work could be dealt out evenly.
  int height = static_cast<int>((total + all + workers - 1) / workers) + 1;
  // A few tiles that are longer than that, beside others: all of them in the same parts, so that
  // those under way at a time share operands in L2 (dx and dW of 2047 x 50001 over 1024, cut at
  // odd places: 342 us and 1.5 GB from memory; so 303 and 0.5).  Parts of at most 3/5 of the height: of
  // all of it, gradients of 64 x 2048 over 32000 tokens take 135 us instead of 93; of 2/5 the example is not cut in parts
  // any more, and its gradients take 540 us instead of 473.
  int parts[MAX_GROUPS], length[MAX_GROUPS];
  bool in_parts = false;
  int budget = workers;  // for parts: no more of them than workers, those of all groups together
  for (int g = 0; g < count; ++g) {
    const long long tiles = static_cast<long long>(rows[g]) * cols[g];
    const int n = (kb[g] + 1) * 5 / (height * 3) + 1;
    const bool few = count > 1 && kb[g] + 1 > height && tiles * n <= budget && kb[g] / n >= 2 * LEAST;
    length[g] = few ? (kb[g] + n - 1) / n : kb[g];
    parts[g] = (kb[g] + length[g] - 1) / length[g];  // none of them empty
    if (few) in_parts = true, budget -= static_cast<int>(tiles) * parts[g];
    order[g] = g;
    for (int i = g; i > 0 && length[order[i]] > length[order[i - 1]]; --i) std::swap(order[i], order[i - 1]);
  }
  // Tiles, the longest first, to the worker that is done first, as long as they stay
  // below that height.
  int heap[MAX_WORKERS];  // load and worker in one number
  for (int w = 0; w < workers; ++w) heap[w] = w;
  auto later = [](int a, int b) { return a > b; };
  auto give = [&](unsigned where, int kb0, int kb1, int slot) {
    std::pop_heap(heap, heap + workers, later);
    const int w = heap[workers - 1] % MAX_WORKERS;
    piece[pieces++] = {{where, static_cast<unsigned short>(kb0), static_cast<unsigned short>(kb1)}, static_cast<short>(w), static_cast<short>(slot)};
    load[w] += kb1 - kb0 + 1;
    most = std::max(most, load[w]);
    heap[workers - 1] = load[w] * MAX_WORKERS + w;
    std::push_heap(heap, heap + workers, later);
  };
  struct Rest {
    unsigned where;
    int k;
  } rest[LARGE_LIST];
  int left = 0;
  for (int i = 0; i < count; ++i) {
    const int g = order[i], first_slot = slots;
    // about as many rows as columns under way at a time (all rows that workers have where there are
    // eight columns: 1930 us instead of 1890 for the four gradients of 16384 x 2048 x 8192)
    const int band_rows = t.m == 256 ? 8 : 16;
    for (int part = 0; part < parts[g]; ++part)
      for (int b = 0; b < rows[g]; b += band_rows)
        for (int c = 0; c < cols[g]; ++c)
          for (int r = b; r < std::min(b + band_rows, rows[g]); ++r) {
            const unsigned where = pack_where(g, r, c);
            if (parts[g] > 1) {
              const int slot = first_slot + (r * cols[g] + c) * parts[g];
              if (part == 0) s.cut[s.cuts++] = {where, static_cast<short>(slot), static_cast<short>(parts[g])};
              give(where, part * length[g], std::min(kb[g], (part + 1) * length[g]), slot + part);
              ++slots;
            } else if (heap[0] / MAX_WORKERS + kb[g] + 1 <= height) {
              give(where, 0, kb[g], -1);
            } else {
              rest[left++] = {where, kb[g]};
            }
          }
  }
  const int kept = pieces;
  int before[MAX_WORKERS], by_load[MAX_WORKERS];
  for (int w = 0; w < workers; ++w) before[w] = load[w], by_load[w] = w;
  std::stable_sort(by_load, by_load + workers, [&](int a, int b) { return load[a] < load[b]; });
  for (int i = 0; i < left; ++i) give(rest[i].where, 0, rest[i].k, -1);  // uncut
  // Cut, the remaining tiles fill all workers up to one height.
  // a part's sums, there and back at 3 TB/s (at 1, too few tiles are cut: 36 us instead of 28 and 87 instead of
  // 78 for the gradients of 600 and 4095 x 512 x 2048; at 9 the same as at 3)
  const double slot_us = 2.0 * 4 * t.m * t.n / 3e6;
  s.us = most * t.us + 4.0 + (slots ? 5.0 + slot_us * slots : 0.0);
  // about one part for each worker
  bool cut = !in_parts && left > 0 && left < workers && height > LEAST && (most - height) * t.us > 5.0 + slot_us * workers;
  while (cut) {
    pieces = kept;
    s.cuts = slots = 0;
    int w = 0, filled[MAX_WORKERS];
    for (int k = 0; k < workers; ++k) filled[k] = before[k];
    bool fits = true;
    for (int i = 0; i < left && fits; ++i) {
      int kb0 = 0;
      const int from = pieces;
      while (kb0 < rest[i].k) {
        while (w < workers && height - filled[by_load[w]] - 1 < LEAST) ++w;
        if (w == workers) {
          fits = false;
          break;
        }
        int n = std::min(rest[i].k - kb0, height - filled[by_load[w]] - 1);
        if (rest[i].k - kb0 - n < LEAST) n = rest[i].k - kb0;  // no crumbs
        piece[pieces++] = {{rest[i].where, static_cast<unsigned short>(kb0), static_cast<unsigned short>(kb0 + n)},
                           static_cast<short>(by_load[w]), -1};
        filled[by_load[w]] += n + 1;
        kb0 += n;
      }
      if (fits && pieces - from > 1) {
        s.cut[s.cuts++] = {rest[i].where, static_cast<short>(slots), static_cast<short>(pieces - from)};
        for (int k = from; k < pieces; ++k) piece[k].slot = static_cast<short>(slots++);
      }
    }
    if (fits) {
      most = 0;
      for (int k = 0; k < workers; ++k) most = std::max(most, filled[k]);
      s.us = most * t.us + 4.0 + (s.cuts ? 5.0 + slot_us * slots : 0.0);
      break;
    }
    height += 1 + height / 64;
  }
  // each worker's units side by side, in order
  int counts[MAX_WORKERS + 1] = {};
  for (int i = 0; i < pieces; ++i) ++counts[piece[i].worker + 1];
  for (int w = 0; w < workers; ++w) counts[w + 1] += counts[w];
  for (int w = 0; w <= workers; ++w) s.first[w] = static_cast<short>(counts[w]);
  for (int i = 0; i < pieces; ++i) {
    const int to = counts[piece[i].worker]++;
    s.unit[to] = piece[i].l, s.slot[to] = piece[i].slot;
  }
  s.units = pieces;
  return true;
}

}  // namespace adgemm

#endif

"""How the tiles of products are dealt out to blocks (csrc/schedule.h, host code): over random sets of products
each tile's K is taken once, and what is written stays inside the lists and the workspace."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "ad_b200", "csrc")

PROGRAM = r"""
#include <cmath>
#include <cstdio>
#include <cstdlib>
#include <cstring>
#include <memory>
#include <random>
#include <vector>

#include "schedule.h"

using namespace adgemm;

struct Product {
  long long m, n, k, k0;
};

// What is wrong with a schedule, or NULL.
const char* wrong(const Product* p, int count, int tiling, int sms, const Schedule& s) {
  const Tiling& t = TILINGS[tiling];
  if (s.workers < 1 || s.workers > MAX_WORKERS || s.units < 1 || s.units > LARGE_LIST) return "workers or units";
  if (s.cuts < 0 || s.cuts > MAX_WORKERS) return "cut tiles past their list";
  if (s.first[0] != 0 || s.first[s.workers] != s.units) return "the workers' units";
  for (int w = 0; w < s.workers; ++w)
    if (s.first[w] > s.first[w + 1]) return "the workers' units";
  const long long slots = static_cast<long long>(partial_elements(sms) / (static_cast<size_t>(t.m) * t.n));
  std::vector<int> used(slots, -1);  // the unit that writes a slot
  struct Tile {
    std::vector<int> units;
    int cut = -1;
  };
  std::vector<std::vector<Tile>> tiles(count);
  std::vector<int> rows(count), cols(count);
  for (int g = 0; g < count; ++g) {
    rows[g] = static_cast<int>((p[g].m + t.m - 1) / t.m), cols[g] = static_cast<int>((p[g].n + t.n - 1) / t.n);
    tiles[g].resize(static_cast<size_t>(rows[g]) * cols[g]);
  }
  auto tile_of = [&](unsigned where) -> Tile* {
    const int g = where >> 30, r = where >> 15 & 0x7fff, c = where & 0x7fff;
    return g < count && r < rows[g] && c < cols[g] ? &tiles[g][static_cast<size_t>(r) * cols[g] + c] : nullptr;
  };
  for (int u = 0; u < s.units; ++u) {
    Tile* tile = tile_of(s.unit[u].where);
    if (!tile) return "a unit outside of the tiles";
    if (s.unit[u].kb1 <= s.unit[u].kb0) return "an empty part";
    tile->units.push_back(u);
    if (s.slot[u] < -1 || s.slot[u] >= slots) return "a slot outside of the workspace";
    if (s.slot[u] < 0) continue;
    if (used[s.slot[u]] >= 0) return "a slot that is written twice";
    used[s.slot[u]] = u;
  }
  for (int c = 0; c < s.cuts; ++c) {
    Tile* tile = tile_of(s.cut[c].where);
    if (!tile || tile->cut >= 0) return "a cut tile";
    tile->cut = c;
  }
  for (int g = 0; g < count; ++g) {
    const int kb = kblocks_of(p[g]);
    for (const Tile& tile : tiles[g]) {
      if (tile.cut < 0) {
        if (tile.units.size() != 1) return "a tile that is taken by none, or by parts that nothing joins";
        const int u = tile.units[0];
        if (s.slot[u] != -1 || s.unit[u].kb0 != 0 || s.unit[u].kb1 != kb) return "a whole tile's K";
      } else {
        const Cut& c = s.cut[tile.cut];
        if (c.parts != static_cast<int>(tile.units.size()) || c.parts < 2) return "the number of parts";
        int at = 0;
        for (int i = 0; i < c.parts; ++i) {  // in the order of their slots
          if (c.slot + i >= slots || used[c.slot + i] < 0) return "a part's slot";
          const int u = used[c.slot + i];
          if (tile_of(s.unit[u].where) != &tile || s.unit[u].kb0 != at) return "a cut tile's K";
          at = s.unit[u].kb1;
        }
        if (at != kb) return "a cut tile's K";
      }
    }
  }
  return nullptr;
}

int main(int argc, char** argv) {
  std::mt19937_64 gen(std::strtoull(argv[1], nullptr, 10));
  const long long sets = std::atoll(argv[2]);
  auto upto = [&](long long lo, long long hi) {  // spread over the logarithm
    std::uniform_real_distribution<double> d(std::log(static_cast<double>(lo)), std::log(static_cast<double>(hi) + 1.0));
    return std::min(hi, std::max(lo, static_cast<long long>(std::exp(d(gen)))));
  };
  std::unique_ptr<Schedule> s(new Schedule);
  long long made = 0, cut = 0, spoilt = 0;
  for (long long i = 0; i < sets; ++i) {
    Product p[MAX_GROUPS];
    int count;
    const long long a = upto(1, 1 << (8 + i % 16)), b = upto(1, 20000), c = upto(1, 1 << (8 + i % 11));
    if (i % 5 == 0) {  // some tens of tiles each, nearly as long as one another
      count = 2 + static_cast<int>(gen() % (MAX_GROUPS - 1));
      const long long k = upto(2000, 200000);
      for (int g = 0; g < count; ++g) {
        const long long kg = k - k * static_cast<long long>(gen() % 40) / 100;
        p[g] = {upto(1, 1800), upto(1, 1800), kg, kg};
      }
    } else if (i % 4 == 0) {  // a block's gradients: dx over two K's, three weights
      count = 4;
      p[0] = {a, c, 2 * b, b}, p[1] = p[2] = {b, c, a, a}, p[3] = {c, b, a, a};
    } else if (i % 4 == 1) {  // dx and dW of a piece
      count = 2;
      p[0] = {a, c, b, b}, p[1] = {b, c, a, a};
    } else {
      count = i % 4 == 2 ? 1 : 1 + static_cast<int>(gen() % MAX_GROUPS);
      for (int g = 0; g < count; ++g) {
        const long long k = upto(1, 1 << (4 + gen() % 19));
        p[g] = {upto(1, 1 << (4 + gen() % 14)), upto(1, 1 << (4 + gen() % 14)), k, gen() % 3 ? k : upto(1, k)};
      }
    }
    const int sms = gen() % 4 ? 148 : 2 + static_cast<int>(gen() % 200);
    for (int tiling = 0; tiling < 3; ++tiling) {
      const int most = sms / TILINGS[tiling].ctas, workers = gen() % 4 ? most : 1 + static_cast<int>(gen() % most);
      if (!make_schedule(p, count, tiling, workers, *s)) continue;
      ++made, cut += s->cuts > 0;
      if (const char* what = wrong(p, count, tiling, sms, *s)) {
        std::printf("%s: tiling %d, %d workers, %d multiprocessors", what, tiling, workers, sms);
        for (int g = 0; g < count; ++g) std::printf(", %lld x %lld over %lld (%lld)", p[g].m, p[g].n, p[g].k, p[g].k0);
        std::printf("\n");
        return 1;
      }
      // the check itself: one mistake in each of some schedules is found
      if (made % 16 == 0) {
        const int u = static_cast<int>(gen() % s->units);
        switch (gen() % 4) {
          case 0: s->unit[u].kb1 = s->unit[u].kb0; break;
          case 1: s->unit[u].kb1 += 1; break;
          case 2: s->slot[u] = static_cast<short>(s->slot[u] < 0 ? 0 : -1); break;
          default: s->unit[u].where ^= 1u << 14;
        }
        if (!wrong(p, count, tiling, sms, *s)) {
          std::printf("a mistake went unseen\n");
          return 1;
        }
        ++spoilt;
      }
    }
  }
  std::printf("%lld %lld %lld\n", made, cut, spoilt);
  return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    cxx = shutil.which("g++") or shutil.which("c++")
    assert cxx, "the library's host compiler"
    d = tmp_path_factory.mktemp("schedule")
    (d / "check.cc").write_text(PROGRAM)
    r = subprocess.run([cxx, "-std=c++17", "-O1", "-g", "-Wall", "-Werror", "-fsanitize=undefined,address", "-fno-sanitize-recover=all",
                        "-I", CSRC, str(d / "check.cc"), "-o", str(d / "check")], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr
    return str(d / "check")


@pytest.mark.parametrize("seed", range(4))
def test_each_part_of_each_tile_once_and_inside_the_workspace(program, seed):
    r = subprocess.run([program, str(seed), "4000"], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr[-3000:]
    made, cut, spoilt = map(int, r.stdout.split())
    assert made > 4000 and cut > 400 and spoilt > 200

"""How an attention call over a paged cache is dealt out (`csrc/paged_deal.h`): arithmetic on lengths, compiled here on its own and held to
counting tile by tile."""
import subprocess
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]

PROGRAM = r"""
#include <cassert>
#include <cstdio>
#include <random>
#include <vector>
#include "paged_deal.h"
using namespace hl;

struct View {
  const int32_t *first, *lengths;
  int sequences, kv_heads, tokens, max_new, max_length;
};
struct Tile { int s, head, block, tile, tiles; };

int main() {
  std::mt19937 rng(7);
  auto pick = [&](int a, int b) { return a + (int)(rng() % (unsigned)(b - a + 1)); };
  for (int round = 0; round < 3000; ++round) {  // Euclid's steps against adding up
    const unsigned n = pick(0, 60), m = pick(1, 300), a = pick(0, 500), b = pick(0, 100000);
    long long want = 0;
    for (unsigned i = 0; i < n; ++i) want += ((long long)a * i + b) / m;
    assert(floor_sum(n, m, a, b) == want);
  }
  for (int d = 1; d < 300; ++d) {  // division by multiplication
    const DealDivide by((uint32_t)d);
    for (int i = 0; i < 200; ++i) {
      const int n = i < 100 ? (int)(rng() >> 1) : pick(0, 1000) * d - (i & 1);
      assert(n < 0 || by(n) == n / d);
    }
    assert(by(0x7fffffff) == 0x7fffffff / d);
  }
  for (int round = 0; round < 4000; ++round) {
    const int groups[] = {1, 2, 3, 4, 5, 7, 8, 16, 20, 64};
    DealShape z = deal_shape(pick(0, 1) ? 4 : 7, pick(5, 7), groups[pick(0, 9)], pick(1, 40), pick(4, 12), pick(0, 3));
    View v{};
    v.sequences = pick(1, 9);
    v.kv_heads = pick(1, 4);
    std::vector<int32_t> first(1, 0), lengths;
    const bool steps = pick(0, 2) == 0;
    for (int s = 0; s < v.sequences; ++s) {
      const int n = steps ? 1 : pick(0, 3) == 0 ? 0 : pick(1, 300);
      first.push_back(first.back() + n);
      lengths.push_back(pick(0, 4) == 0 ? pick(0, n) : n + pick(0, 700));  // some stand partly, or wholly, at no position
    }
    v.first = steps && pick(0, 1) ? nullptr : first.data();
    v.lengths = lengths.data();
    v.tokens = first.back();
    v.max_new = 300;
    v.max_length = pick(0, 3) ? 1000 : 600;  // beyond it: left out
    std::vector<Tile> line;
    std::vector<long long> start;
    for (int s = 0; s < v.sequences; ++s) {
      start.push_back((long long)line.size());
      const int n = first[s + 1] - first[s];
      if (lengths[s] > v.max_length) continue;
      long long counted = (long long)line.size();
      for (int h = 0; h < v.kv_heads; ++h)
        for (int r0 = 0, b = 0; r0 < n * z.group; r0 += z.rows(), ++b) {
          const int last = std::min(n * z.group, r0 + z.rows()) - 1, sees = std::max(0, lengths[s] - n + last / z.group + 1);
          const int tiles = std::max(1, (sees + z.keys() - 1) / z.keys());
          for (int t = -z.extra; t < tiles; ++t) line.push_back(Tile{s, h, b, t, tiles});  // -extra .. -1: what the item costs besides
        }
      assert(deal_sequence(v, z, s) == (long long)line.size() - counted);
    }
    const long long total = (long long)line.size(), chunk = std::max((total + z.streams - 1) / z.streams, (long long)z.least);
    long long seen = 0;
    for (int i = 0; i < z.streams; ++i) {
      const long long from = chunk * i, until = std::min(total, from + chunk);
      DealPlace place{v.sequences, total};
      if (from < total) place = DealPlace{line[from].s, start[line[from].s]};
      int pieces[2] = {0, 0};
      for (DealItem it = deal_item(v, z, place, from, until); deal_valid(it); deal_next(v, z, it)) {
        for (int t = it.tile0; t < it.tile1; ++t, ++seen) {
          const Tile& w = line[it.at + z.extra + t];
          while (line[seen].tile < 0) ++seen;
          assert(it.at + z.extra + t == seen && it.at + z.extra + t >= from && it.at + z.extra + t < until && w.s == it.s && w.head == it.head && w.block == it.block && w.tile == t && w.tiles == it.tiles);
        }
        if (it.tile0 > 0 || it.tile1 < it.tiles) ++pieces[it.tile0 > 0 ? 0 : 1];
      }
      assert(pieces[0] <= 1 && pieces[1] <= 1);
    }
    while (seen < total && line[seen].tile < 0) ++seen;
    assert(seen == total);
  }
  // the largest sizes that a call may have
  DealShape z = deal_shape(4, 5, 64, 296, 8, 0);
  int32_t first[2] = {0, 33000000}, lengths[1] = {33000000};
  View v{first, lengths, 1, 8, 33000000, 33000000, 33000000};
  const long long blocks = 33000000ll * 64 / 16;  // block b ends with token b / 4
  long long want = 0;
  for (long long b = 0; b < blocks; ++b) want += (b / 4 + 1 + 31) / 32;
  assert(deal_sequence(v, z, 0) == 8 * want);
  puts("deal ok");
}
"""


def test_every_tile_is_dealt_once(tmp_path):
    (tmp_path / "main.cpp").write_text("#include <algorithm>\n" + PROGRAM)
    exe = tmp_path / "main"
    subprocess.run(["g++", "-std=c++17", "-O2", f"-I{ROOT / 'heirloom_b200' / 'csrc'}", "-o", str(exe), str(tmp_path / "main.cpp")], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert "deal ok" in got.stdout, got.stderr

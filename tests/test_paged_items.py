"""How the attention of a shared prefix is cut into pieces (csrc/mtl_paged_items.h), in a host program
that walks every piece of a call as the kernel's workgroups do: each block of each item is taken
once, by the pieces that the second launch reads, and in the form that it expects (CPU)."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "moss-tts-lite_amd", "csrc")

# Arguments: query heads to a kv head, kv heads, sequences, seed.  Groups come first, then the
# sequences' own parts; 64 lanes have a run of each, and a piece begins at the first run that
# reaches into it.  A third of the sequences or so has nothing of its own.
PROGRAM = r"""
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <vector>
#include "mtl_paged_items.h"
using namespace mtl;

struct Part { int columns, blocks; };                // a group's shared part, a sequence's own

template <int WIDE>
int walk(const std::vector<Part> (&parts)[2], int per_kv, int workgroups) {
  long upto[2][64], total = 0, most = per_kv < WIDE ? per_kv : WIDE;
  int run[2];
  std::vector<std::vector<Span>> want[2];            // pieces of each item, as the join reads them
  std::map<std::vector<int>, std::vector<int>> taken;    // (kind, part, item): blocks, by piece
  for (int k = 0; k < 2; ++k) {
    run[k] = ((int)parts[k].size() + 63) / 64;
    long sum = 0;
    for (int lane = 0; lane < 64; ++lane) {
      for (int i = lane * run[k]; i < (lane + 1) * run[k] && i < (int)parts[k].size(); ++i) {
        sum += cost_of(parts[k][i].columns, parts[k][i].blocks, WIDE);
        if (parts[k][i].blocks && parts[k][i].columns > most)
          most = parts[k][i].columns < WIDE ? parts[k][i].columns : WIDE;
      }
      upto[k][lane] = sum;
    }
    total += sum;
  }
  const int first_own = (int)upto[0][63], each = block_cost((int)most);
  int pieces = total / each < workgroups ? (int)(total / each) : workgroups;
  if (pieces < 1) pieces = 1;
  const Pieces cut{(int)(total / pieces), (int)(total % pieces)};
  for (int k = 0, base = 0; k < 2; ++k) {
    want[k].resize(parts[k].size());
    for (size_t i = 0; i < parts[k].size(); ++i)
      for (int c = 0; c < parts[k][i].columns; c += WIDE) {
        const int n = parts[k][i].columns - c < WIDE ? parts[k][i].columns - c : WIDE;
        want[k][i].push_back(cut.pieces_of(base, parts[k][i].blocks, n));
        base += item_cost(n, parts[k][i].blocks);
      }
  }
  for (int piece = 0; piece < pieces; ++piece) {
    const int lo = cut.start(piece), hi = cut.start(piece + 1);
    if (lo >= hi) continue;
    int k = lo >= first_own, base = k ? first_own : 0, from = 0, slots[2] = {0, 0}, bad = 0;
    while (lo - base >= upto[k][from]) ++from;
    if (from) base += (int)upto[k][from - 1];
    size_t i = (size_t)from * run[k];
    while (base < hi) {
      if (i >= parts[k].size()) {
        if (k == 1) break;
        k = 1;
        i = 0;
        base = first_own;
        continue;
      }
      const Part& p = parts[k][i];
      items_within<WIDE>(base, p.columns, p.blocks, lo, hi, [&](int c, int n, Span b) {
        const Span w = want[k][i][c / WIDE];
        const bool whole = b.x == 0 && b.y == p.blocks;
        bad |= n > WIDE || c + n > p.columns || whole != (w.x == w.y) || piece < w.x ||
               piece > w.y || (piece == w.x) != (b.x == 0);
        if (!whole && slots[b.x == 0]++) bad = 1;    // a piece has room for two cut items
        auto& t = taken[{k, (int)i, c / WIDE}];
        for (int x = b.x; x < b.y; ++x) t.push_back(x);
        if (piece == w.y && b.y != p.blocks) bad = 1;
      });
      ++i;
    }
    if (bad) return std::printf("piece %d of %d is not what the join reads\n", piece, pieces), 1;
  }
  for (int k = 0; k < 2; ++k)
    for (size_t i = 0; i < parts[k].size(); ++i)
      for (int t = 0; t * WIDE < parts[k][i].columns; ++t) {
        const auto& got = taken[{k, (int)i, t}];
        bool same = (int)got.size() == parts[k][i].blocks;
        for (size_t x = 0; same && x < got.size(); ++x) same = got[x] == (int)x;
        if (!same)
          return std::printf("part %d of kind %d, item %d: %zu blocks of %d\n", (int)i, k, t,
                             got.size(), parts[k][i].blocks), 1;
      }
  return 0;
}

int main(int, char** arg) {
  const int per_kv = std::atoi(arg[1]), kv_heads = std::atoi(arg[2]), seqs = std::atoi(arg[3]);
  for (int round = 0; round < 12; ++round) {
    std::mt19937 rng(std::atoi(arg[4]) * 100 + round);
    auto any = [&](int lo, int hi) { return lo + (int)(rng() % (unsigned)(hi - lo + 1)); };
    std::vector<Part> parts[2];
    for (int s = 0; s < seqs;) {
      const int n = round % 3 ? any(1, seqs - s) : any(1, 6), in = n < seqs - s ? n : seqs - s;
      const int shared = any(0, 2) && in > 1 ? any(0, 3) ? any(1, 3) : any(4, 60) : 0;
      if (round % 4) parts[0].push_back({in * per_kv, shared});
      for (int i = 0; i < in; ++i) parts[1].push_back({per_kv, any(0, 2) ? any(0, 3) : any(0, 16)});
      s += in;
    }
    if (round == 5) for (Part& p : parts[1]) p.blocks = 0;
    const int groups = kv_heads < 512 ? 512 / kv_heads : 1;
    if (seqs * per_kv <= 16 ? walk<16>(parts, per_kv, groups) : walk<kWide>(parts, per_kv, groups))
      return std::printf("round %d\n", round), 1;
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    if shutil.which("g++") is None:
        pytest.skip("needs a host compiler")
    at = tmp_path_factory.mktemp("items")
    src, exe = at / "walk.cpp", at / "walk"
    src.write_text(PROGRAM)
    subprocess.run(["g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-I", CSRC, str(src), "-o",
                    str(exe)], check=True)
    return str(exe)


@pytest.mark.parametrize("seqs", [1, 2, 5, 63, 64, 65, 96, 130, 192, 300, 600])
@pytest.mark.parametrize("per_kv,kv_heads", [(1, 1), (1, 8), (3, 2), (4, 8), (7, 1), (16, 1), (17, 1),
                                             (20, 2), (48, 2), (63, 1), (64, 1), (64, 8), (65, 1),
                                             (71, 1), (128, 1), (128, 2), (130, 1)])
def test_every_block_is_taken_once(program, seqs, per_kv, kv_heads):
    for seed in range(3):
        r = subprocess.run([program, str(per_kv), str(kv_heads), str(seqs), str(seed)],
                           capture_output=True, text=True, timeout=60)
        assert r.returncode == 0, (seed, r.stdout)

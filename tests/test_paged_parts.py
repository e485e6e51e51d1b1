"""The paged attention's division of work as its source has it: the functions and the prompt kernel's loop over tiles are cut
out of the kernels' files, compiled for the host and run. Positions go by starts and lengths as they stand, a block's parts
cover its tiles once, a tile is computed from where it was staged and as it was staged, and a page that is missing under
a tile taken for whole is found."""

import random
import re
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "pdum_dsl_amd" / "csrc"
LIMIT = 1 << 30


def _between(text, first, last):
    i = text.index(first)
    return text[i : text.index(last, i)]


MAIN = """
#include <cstdint>
#include <cstdio>
#include <type_traits>
#include <vector>
#define __device__
#define __forceinline__ inline
struct pdh_paged_batch {
  const int32_t *table, *starts, *lengths;
  int64_t seqs, rows, width, ld_table;
};
#include "seq.inc"
static int scalar(int x) { return x; }
struct PagedAttn {
  pdh_paged_batch b;
  int group, window, sinks, reach, zero_rest;
  static bool has(int page) { return page >= 0; }
};
#include "plan.inc"
#include "keys.inc"
static void wait_vmcnt0() {}
static void __syncthreads() {}

struct Did {
  int key0, computed_cut, staged_cut, staged_key0;
};

template <int BITS>
bool sweep(const PagedAttn& a, const BlockKeys& bk, int pos_lo, int pos_hi, int v0, int v1, int missing, std::vector<Did>& did) {
  struct Tile {
    int key0, p[2];
  };
  struct Held {
    int key0, cut;
  };
  Held held[2] = {{-1, 0}, {-1, 0}}, ahead = {-1, 0};
  bool lost = false;
  const bool busy = true;
  const int wpos_hi = 2147483647;
  auto tile_at = [&](int v) { const int k = bk.tile(v) * 32; return Tile{k, {k == missing ? -1 : 0, 0}}; };
  auto stage16 = [&](const Tile& t, int buf, bool cut) { held[buf] = Held{t.key0, cut}; };
  auto fetch4 = [&](const Tile& t, bool cut) { ahead = Held{t.key0, cut}; };
  auto commit4 = [&](int buf) { held[buf] = ahead; };
  auto tile = [&](int buf, const Tile& t, auto cutc) {
    did.push_back(Did{t.key0, decltype(cutc)::value, held[buf].cut, held[buf].key0});
  };
#include "sweep.inc"
  return lost;
}

int main() {
  // a line: rows group reach window sinks nsplit bits missing start end length
  long long rows, group, reach, window, sinks, nsplit, bits, missing, start, end, length;
  while (scanf("%lld %lld %lld %lld %lld %lld %lld %lld %lld %lld %lld", &rows, &group, &reach, &window, &sinks, &nsplit, &bits,
               &missing, &start, &end, &length) == 11) {
    const int32_t starts[2] = {(int32_t)start, (int32_t)end}, lengths[1] = {(int32_t)length};
    const PagedAttn a{{nullptr, starts, lengths, 1, rows, 0, 0}, (int)group, (int)window, (int)sinks, (int)reach, 0};
    const SeqPlan d = plan_of<16>(a, 0), p = plan_of<128>(a, 0);
    printf("plan %d %d %d %d %d %d %d %d\\n", p.row0, p.n, p.pos0, p.nb, d.nb, p.sb, p.wb, p.blocks);
    for (int rb = 0; rb < p.nb; ++rb) {
      const int f0 = rb * 128, fend = p.n * a.group - f0 < 128 ? p.n * a.group : f0 + 128;
      const int lo = p.pos0 + f0 / a.group, hi = p.pos0 + (fend - 1) / a.group;
      const BlockKeys bk = block_keys(a, lo, hi, nsplit ? (int)nsplit : 1);
      if (nsplit == 0) continue;  // the plan and a block's keys alone
      printf("block %d %d %d %d %d %d %d\\n", lo, hi, bk.sb, bk.wb, bk.tiles, bk.part, bk.parts);
      for (int split = 0; split < bk.parts; ++split) {
        const int v0 = split * bk.part, v1 = v0 + bk.part < bk.tiles ? v0 + bk.part : bk.tiles;
        std::vector<Did> did;
        const bool lost = bits == 16 ? sweep<16>(a, bk, lo, hi, v0, v1, (int)missing, did)
                                     : sweep<4>(a, bk, lo, hi, v0, v1, (int)missing, did);
        printf("part %d\\n", (int)lost);
        for (const Did& x : did) printf("tile %d %d %d %d\\n", x.key0, x.computed_cut, x.staged_cut, x.staged_key0);
      }
    }
    printf("end\\n");
  }
}
"""


@pytest.fixture(scope="module")
def run(tmp_path_factory):
    at = tmp_path_factory.mktemp("parts")
    head, attn = (CSRC / "paged.h").read_text(), (CSRC / "paged_attn.hip").read_text()
    (at / "seq.inc").write_text(_between(head, "constexpr int kMaxTokens", "// The sequence that owns a row"))
    (at / "plan.inc").write_text(_between(attn, "struct SeqPlan {", "__device__ __forceinline__ int scalar(")
                                 + _between(attn, "template <int ROWS>\n__device__ __forceinline__ SeqPlan plan_of", "// The plan of a"))
    (at / "keys.inc").write_text(_between(attn, "constexpr int kPartTiles", "// The sequence of a slot"))
    (at / "sweep.inc").write_text(_between(attn, "  // Tiles [c0, c1) are whole", "  // ---- rows out"))
    (at / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-O1", "-ftrapv", "-w", str(at / "main.cpp"), "-o", str(at / "main")], check=True)

    def go(cases):
        text = "\n".join(" ".join(map(str, c)) for c in cases)
        out = subprocess.run([str(at / "main")], input=text, check=True, capture_output=True, text=True).stdout
        return [part.strip().split("\n") for part in out.split("end\n")[:-1]]

    return go


def _cases(seed, count):
    rng = random.Random(seed)
    pick = lambda *xs: rng.choice(xs)  # noqa: E731
    for _ in range(count):
        n, group = pick(1, 1, 3, 40, 130, rng.randint(1, 700)), pick(1, 4, 7, 20)
        length = pick(n, n + rng.randint(0, 3000), rng.randint(0, 9000), max(0, n - 3))
        start = pick(0, 0, 5, 1000)
        rows = pick(start + n, start + n, start + n + 9, max(start, start + n - rng.randint(0, n)))  # the last rows may not be there
        reach = pick(16384, 16384, -(-max(length, 1) // 16) * 16, rng.randint(0, 300) * 16)
        window, sinks = pick((LIMIT + (1 << 24), 0), (LIMIT + (1 << 24), 0), (rng.randint(1, 3000), pick(0, 1, 4, 33, 100)))
        missing = 32 * rng.randint(0, max(1, length // 32))
        yield rows, group, reach, window, sinks, pick(1, 1, 2, 5, 32), pick(16, 4), missing, start, start + n, length


def test_every_tile_is_computed_once_as_it_was_staged(run):
    cases = list(_cases(1, 2500))
    singles = found = 0
    for case, lines in zip(cases, run(cases)):
        rows, group, reach, window, sinks, nsplit, bits, missing, start, end, length = case
        n = max(0, min(end, rows) - start)
        row0, got_n, pos0, nb, nb16, sb, wb, blocks = map(int, lines[0].split()[1:])
        assert (got_n, nb, nb16) == (n, -(-n * group // 128), -(-n * group // 16)), case
        if n:
            assert row0 == start
        true0 = length - (end - start)  # the first row's position, though rows behind the last one there are not
        sees = n and true0 + n > 0
        assert not sees or pos0 == true0, case
        assert sees or n == 0 or pos0 + n <= 0, case
        tiles, rb = [], -1
        pending = []
        for line in lines[1:] + ["block"]:
            kind, *nums = line.split()
            if kind == "block":
                if pending:
                    _check_block(pending, case, sees)
                    singles += sum(1 for p in pending[1:] for t in p[1] if t[1] and t[4])
                    found += any(p[0] for p in pending[1:])
                pending = [tuple(map(int, nums))]
            elif kind == "part":
                pending.append((int(nums[0]), []))
            else:
                key0, computed, staged, at = map(int, nums)
                lo, hi = pending[0][:2]
                whole = key0 + 31 <= lo and key0 + 32 <= reach and key0 > hi - window
                pending[-1][1].append((key0, computed, staged, at, whole))
    assert singles > 100 and found > 100  # whole tiles computed by themselves, and missing pages among pairs


def _check_block(pending, case, sees):
    rows, group, reach, window, sinks, nsplit, bits, missing, start, end, length = case
    (lo, hi, sb, wb, tiles, part, parts), swept = pending[0], pending[1:]
    assert len(swept) == parts and 1 <= parts <= max(1, nsplit)
    keys = [t[0] for _, did in swept for t in did]
    assert keys == [32 * (v if v < sb else v - sb + wb) for v in range(tiles)]  # each once, in order
    held = set(keys)
    for pos in (lo, hi):  # what the block's first and last rows see lies in them
        for key in {0, sinks - 1, pos - window + 1, pos, reach - 1, pos // 2, (2 * pos - window) // 2}:
            if 0 <= key <= pos and key < reach and (key < sinks or key > pos - window):
                assert key // 32 * 32 in held, (case, key)
    for lost, did in swept:
        for key0, computed, staged, at, whole in did:
            assert at == key0 and computed == staged, (case, key0)
            assert computed or whole, (case, key0)  # taken for whole only where every row sees every key
        assert lost == any(key0 == missing and not computed for key0, computed, *_ in did), case


def test_positions_of_any_starts_and_lengths(run):
    """Every row's position is what starts and lengths say, or no table's; no sum passes 32 bits (the build traps one)."""
    rng = random.Random(3)
    odd = lambda: rng.choice((rng.randint(-5, 400), rng.randint(-(2**31), 2**31 - 1), 2**31 - 1, LIMIT, LIMIT + rng.randint(-300, 300)))  # noqa: E731
    cases = []
    for _ in range(2500):
        rows, group = rng.randint(1, 300), rng.choice((1, 4, 20))
        reach, window = rng.choice((0, 64, 4096, LIMIT)), rng.choice((1, 7, 500, LIMIT + (1 << 24)))
        cases.append((rows, group, reach, window, rng.choice((0, 3)), 0, 16, -1, odd(), odd(), odd()))
    some = 0
    for case, lines in zip(cases, run(cases)):
        rows, group, reach, window, sinks, *_, start, end, length = case
        row0, n, pos0, *_ = map(int, lines[0].split()[1:])
        assert 0 <= row0 and row0 + n <= rows
        assert n == max(0, min(max(end, 0), rows) - min(max(start, 0), rows))
        for r in {row0, row0 + n // 2, row0 + n - 1} if n else ():
            true, got = length - (end - r), pos0 + r - row0
            assert got == true or (got < 0 and true < 0) or (got >= LIMIT and true >= LIMIT), case
            some += 0 <= true < LIMIT
    assert some > 200


def test_the_constants_that_other_tests_restate():
    text = (CSRC / "paged_attn.hip").read_text()
    assert re.search(r"constexpr int kHeadsRun = 3;", text)
    assert re.search(r"constexpr int kPartTiles = 8;", text)

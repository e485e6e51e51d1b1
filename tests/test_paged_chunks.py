"""The append's rule on chunks a thread, as its source has it, compiled for the host: several only where a row has more chunks
than a workgroup has threads, and the call fills the chip."""

import subprocess
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "pdum_dsl_amd" / "csrc"

MAIN = """
#include <cstdint>
#include <cstdio>
#include <type_traits>
#include "rule.inc"
int main() {
  long long rows, items;
  while (scanf("%lld %lld", &rows, &items) == 2) by_chunks(rows, items, [](auto n) { printf("%d\\n", (int)decltype(n)::value); });
}
"""


def test_several_chunks_a_thread_where_a_thread_has_several(tmp_path):
    text = (CSRC / "paged.hip").read_text()
    first = text.index("constexpr int64_t kManyItems")
    rule = text.index("template <typename F>\nvoid by_chunks")
    (tmp_path / "rule.inc").write_text(text[first : text.index("\n", first) + 1] + text[rule : text.index("}  // namespace", rule)])
    (tmp_path / "main.cpp").write_text(MAIN)
    subprocess.run(["g++", "-std=c++17", "-w", str(tmp_path / "main.cpp"), "-o", str(tmp_path / "main")], check=True)
    layouts = [(hq + 2 * hkv) * (d // 8) for hq, hkv, d in ((32, 8, 128), (12, 12, 64), (16, 4, 64), (0, 1, 64), (4, 2, 64), (16, 8, 64))]
    calls = [(rows, items) for items in layouts for rows in (1, 64, 1000, 16384, (1 << 24) - 1)]
    got = subprocess.run([str(tmp_path / "main")], input="\n".join(f"{r} {i}" for r, i in calls), check=True, capture_output=True,
                         text=True).stdout.split()
    for (rows, items), n in zip(calls, map(int, got)):
        if n > 1:
            assert items > 256 and rows * items > 1 << 18, (rows, items)
        else:
            assert items <= 256 or rows * items <= 1 << 18, (rows, items)
    assert {int(n) for n in got} == {1, 4}

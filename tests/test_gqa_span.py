"""Which pages tokens look up, restated: the kernels' own arithmetic (gqa_span.h) compiled for the host against a count of every entry.  No GPU needed."""
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "dsv4_attn_b200" / "csrc"
PROGRAM = r"""
#include "gqa_span.h"
#include <cstdio>
#include <cstdlib>
#include <vector>
using namespace dsv4;
static bool sees(int p, int j, int window, int first) { return j <= p && (window == 0 || p - j < window || j < first); }
int main(int argc, char** argv) {
    const int pages = atoi(argv[1]), room = 64 * pages, windows[] = {0, 1, 2, 63, 64, 65, 130, 1 << 30}, firsts[] = {0, 1, 64, 65, 500, 0x7FFFFFFF}, tokens[] = {1, 5, 70};
    long calls = 0;
    for (int n = 0; n <= room + 3 * 64 + 10; ++n)
        for (int window : windows) for (int first : firsts) for (int T : tokens) for (int part = 0; part < 2; ++part) {
            const int place0 = n - T, entries = n < room ? n : room, t0 = part ? T / 2 : 0, t1 = part ? T - 1 : T / 2;
            const GqaSpan s = gqa_token_span(place0, entries, t0, t1, window, first);
            std::vector<int> looked(pages, 0), wanted(pages, 0);
            if (s.count < 1) { printf("no tile: n %d window %d first %d\n", n, window, first); return 1; }
            for (int k = 0; k < s.count; ++k) {
                const int slot = s.slot(k);
                if (!s.has(slot)) { if (s.hi > 0 || k > 0) { printf("a tile without a page: n %d window %d first %d\n", n, window, first); return 1; }  continue; }
                if (slot < 0 || slot >= pages) { printf("page %d of %d looked up: n %d window %d first %d tokens %d..%d of %d\n", slot, pages, n, window, first, t0, t1, T); return 1; }
                if (looked[slot]++) { printf("a page twice: n %d window %d first %d\n", n, window, first); return 1; }
            }
            for (int j = 0; j < entries; ++j) {
                bool seen = false;
                for (int t = t0; t <= t1 && !seen; ++t) seen = sees(place0 + t, j, window, first);
                if (seen) wanted[j / 64] = 1;
                const bool inside = j < s.hi && (j >= s.lo || j < s.first);
                if (seen != inside) { printf("entry %d: n %d window %d first %d tokens %d..%d of %d\n", j, n, window, first, t0, t1, T); return 1; }
            }
            for (int i = 0; i < pages; ++i) if (wanted[i] > looked[i]) { printf("page %d is missed: n %d window %d first %d\n", i, n, window, first); return 1; }
            ++calls;
        }
    // a request as long as 32 bits hold, over the widest table
    const GqaSpan s = gqa_token_span(0x7FFFFFFF - 5, 0x7FFFFFC0, 0, 4, 7, 0);
    for (int k = 0; k < s.count; ++k) if (s.has(s.slot(k)) && s.slot(k) >= 0x1FFFFFF) { printf("widest table\n"); return 1; }
    printf("%ld\n", calls);
    return 0;
}
"""


@pytest.fixture(scope="module")
def program(tmp_path_factory):
    at = tmp_path_factory.mktemp("span")
    (at / "span.cpp").write_text(PROGRAM)
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-I", str(CSRC), str(at / "span.cpp"), "-o", str(at / "span")], check=True)
    return at / "span"


@pytest.mark.parametrize("pages", [1, 2, 5])
def test_every_entry_that_is_seen_and_no_page_outside_the_table(program, pages):
    r = subprocess.run([str(program), str(pages)], capture_output=True, text=True)
    assert r.returncode == 0, r.stdout
    assert int(r.stdout) > 10_000


def test_every_kernel_asks_whether_the_table_has_a_page():
    """Each look at the block table by a span's slot stands behind `has`."""
    found = 0
    for name in ("gqa_decode.cuh", "gqa_rows.cuh", "gqa_prefill.cuh"):
        lines = (CSRC / name).read_text().splitlines()
        for i, line in enumerate(lines):
            if "ptx::ld(a.block_table + int64_t(w.b)" in line:
                assert ".has(" in lines[i - 1], f"{name}:{i + 1}"
                found += 1
    assert found == 3

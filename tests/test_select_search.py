"""The search that a page selection's threshold comes from, built for the host from the kernel's own
header and run over counts of keys: it ends, at the largest value that enough keys are at least."""

import shutil
import subprocess

import pytest

from sgl_amd_mono_amd import build

# argv: need lo hi key ..; prints the result, how many keys were counted to be at least it, and the steps
SOURCE = """
#include <stdio.h>
#include <stdlib.h>
#include "prompt_search.h"
int main(int argc, char** argv) {
  int kept, steps = 0;
  const uint32_t top = mono::prompt::largest_kept_by(
      atoi(argv[1]), (uint32_t)strtoul(argv[2], 0, 10), (uint32_t)strtoul(argv[3], 0, 10), kept, [&](uint32_t mid) {
        if (++steps > 64) printf("does not end\\n"), exit(1);
        int n = 0;
        for (int i = 4; i < argc; ++i) n += (uint32_t)strtoul(argv[i], 0, 10) >= mid;
        return n;
      });
  printf("%u %d %d\\n", top, kept, steps);
}
"""


@pytest.fixture(scope="module")
def search(tmp_path_factory):
    cc = shutil.which("g++")
    if cc is None:
        pytest.skip("no host compiler")
    d = tmp_path_factory.mktemp("search")
    (d / "search.cpp").write_text(SOURCE)
    subprocess.run([cc, "-std=c++17", "-O1", "-Wno-unknown-pragmas", f"-I{build.CSRC}", str(d / "search.cpp"), "-o", str(d / "search")], check=True)

    def run(need, lo, hi, keys):
        r = subprocess.run([str(d / "search"), *map(str, (need, lo, hi, *keys))], capture_output=True, text=True, timeout=20)
        assert r.returncode == 0, r.stdout
        return tuple(int(v) for v in r.stdout.split())

    return run


# (keys in the order of their values: 0x7fffffff as a score has the largest key, 0xffffffff the smallest)
ODD = [0, 1, 2, 0x7F800001 | 1 << 31, 0x80000000, 0xFFC00000, 0xFFFFFFFD, 0xFFFFFFFE, 0xFFFFFFFF]


@pytest.mark.parametrize("keys", [
    [0xFFFFFFFF], [0xFFFFFFFF] * 40, [0] * 39 + [0xFFFFFFFF], [0xFFFFFFFE, 0xFFFFFFFF], [0x80000000 + 77 * i for i in range(40)] + [0xFFFFFFFF],
    [0x80000000 + 99 * i for i in range(99)] + [0xFFFFFFFF], ODD, ODD * 9, [1], [5] * 70, [0, 0, 1],
])  # fmt: skip
def test_the_search_ends_at_the_largest_value_kept(search, keys):
    ranked = sorted(keys, reverse=True)
    for need in sorted({1, 2, 3, 31, 64, 65, 70, len(keys) - 1, len(keys)}):
        if not 1 <= need <= len(keys):
            continue
        kth = ranked[need - 1]
        for lo in sorted({0, kth // 2, kth}):
            top, kept, steps = search(need, lo, ranked[0], keys)
            assert steps <= 33
            at_least = sum(k >= top for k in keys)
            assert kept in (0, at_least) and (kept == 0) <= (top == lo)
            # the k-th largest key itself, or a value between it and the next that the same keys are at least
            assert at_least == need if kept == need else top == kth

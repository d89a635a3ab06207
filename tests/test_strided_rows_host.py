"""Whether two sets of strided rows share a byte, against sets of addresses."""
import os
import subprocess

import numpy as np
import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

DRIVER = r"""
#include "it_strided.hpp"
#include <cstdio>
using itkv::StridedRows;
int main() {
  long long x[12];
  while (std::scanf("%lld%lld%lld%lld%lld%lld%lld%lld%lld%lld%lld%lld", x, x + 1, x + 2, x + 3, x + 4, x + 5, x + 6, x + 7, x + 8, x + 9,
                    x + 10, x + 11) == 12) {
    const StridedRows a{uintptr_t(x[0]), x[1], x[2], x[3], x[4], x[5]}, b{uintptr_t(x[6]), x[7], x[8], x[9], x[10], x[11]};
    if (itkv::share_memory(a, b) != itkv::share_memory(b, a)) return 1;
    std::printf("%d\n", int(itkv::share_memory(a, b)));
  }
  return 0;
}
"""


@pytest.fixture(scope="module")
def share(tmp_path_factory):
    d = tmp_path_factory.mktemp("strided")
    (d / "driver.cpp").write_text(DRIVER)
    subprocess.run(["g++", "-O1", "-std=c++17", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I",
                    os.path.join(ROOT, "infer_train_amd", "csrc"), str(d / "driver.cpp"), "-o", str(d / "driver")], check=True)

    def run(cases):
        text = "\n".join(" ".join(str(int(v)) for v in a + b) for a, b in cases)
        out = subprocess.run([str(d / "driver")], input=text, capture_output=True, text=True, check=True).stdout.split()
        return [x == "1" for x in out]

    return run


def touched(rows):
    at, token, head, size, tokens, heads = rows
    return {at + t * token + h * head + i for t in range(tokens) for h in range(heads) for i in range(size)}


@pytest.mark.parametrize("same", ["token", "both", "one token", "head-major"])
def test_against_sets_of_bytes(share, same):
    rng = np.random.default_rng(len(same))
    cases = []
    for _ in range(3000):
        n, token = int(rng.integers(1, 6)), int(rng.integers(1, 60))
        a = [int(rng.integers(100, 400)), token, int(rng.integers(1, 20)), int(rng.integers(1, 9)), n, int(rng.integers(1, 5))]
        b = [int(rng.integers(100, 400)), token, int(rng.integers(1, 20)), int(rng.integers(1, 9)), n, int(rng.integers(1, 5))]
        if same == "both":
            b[2] = a[2]
        elif same == "one token":
            a[4] = b[4] = 1
            b[1] = int(rng.integers(0, 60))
        elif same == "head-major":
            a[1] = b[1] = int(rng.integers(1, 20))
            a[2] = b[2] = int(rng.integers(20, 120))
        cases.append((a, b))
    want = [bool(touched(a) & touched(b)) for a, b in cases]
    assert share(cases) == want and 100 < sum(want) < 2900


def test_other_token_strides_are_judged_by_their_ends(share):
    """Never less than what is shared."""
    rng = np.random.default_rng(9)
    cases = []
    for _ in range(2000):
        a, b = ([int(rng.integers(100, 400)), int(rng.integers(0, 60)), int(rng.integers(0, 20)), int(rng.integers(0, 9)), int(rng.integers(0, 6)),
                 int(rng.integers(0, 5))] for _ in range(2))
        cases.append((a, b))
    got, want = share(cases), [bool(touched(a) & touched(b)) for a, b in cases]
    assert all(g or not w for g, w in zip(got, want))


def test_large_projections(share):
    """4096 tokens of 128 heads beside their rows, either way round, and one byte into them."""
    width, row, es = 128 * 192, 576, 2
    token = (width + row) * es
    q = [1 << 33, token, 192 * es, 64 * es, 4096, 128]
    kv = [(1 << 33) + (width - 128) * es, token, 0, row * es, 4096, 1]
    assert share([(q, kv)]) == [False]
    last = q[0] + 127 * 192 * es + 64 * es  # the end of the last head's rope part
    assert share([(q, [last] + kv[1:]), (q, [last - 1] + kv[1:])]) == [False, True]
    head_major = [1 << 33, 128, 4096 * 128, 64, 4096, 128]
    assert share([(head_major, [(1 << 33) + 64] + head_major[1:]), (head_major, [(1 << 33) + 63] + head_major[1:])]) == [False, True]

"""The weights by which the 4-bit cache's attention is cut into shares
(csrc/kv4_shares.hpp, compiled for the host) against what the tiles see."""

from __future__ import annotations

import ctypes
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                    "flash-kmeans-cuda_amd", "csrc")
SOURCE = """
#include "kv4_shares.hpp"
extern "C" int item() { return fkc::kItem; }
extern "C" int idle() { return fkc::kIdle; }
extern "C" int weight(int cols, int gr, int G, int causal, int nq, int end, int j) {
  return fkc::kv4_weight(cols, gr, G, causal != 0, nq, end, j);
}
extern "C" long long most(int cols, int gr, int G, long long max_seq) {
  return fkc::kv4_most_weight(cols, gr, G, max_seq);
}
"""
# (columns of a tile, tokens of a granule) of every form
FORMS = [(16, 256), (16, 128), (32, 128), (256, 64), (128, 32)]


@pytest.fixture(scope="module")
def shares(tmp_path_factory):
    d = tmp_path_factory.mktemp("shares")
    src, so = d / "shares.cpp", d / "shares.so"
    src.write_text(SOURCE)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-fPIC", "-shared", "-I", CSRC,
                    str(src), "-o", str(so)], check=True)
    lib = ctypes.CDLL(str(so))
    lib.most.restype = ctypes.c_longlong
    lib.most.argtypes = [ctypes.c_int] * 3 + [ctypes.c_longlong]
    return lib


def _tiles(cols, G, nq):
    return -(-nq * G // cols)


def _granules(cols, gr, G, causal, nq, end, tile):
    """Granules that a tile's last column sees."""
    last = min((tile + 1) * cols, nq * G) - 1
    lim = min(max(0, end - nq + 1 + last // G), end) if causal else end
    return -(-lim // gr)


@pytest.mark.parametrize("cols,gr", FORMS)
@pytest.mark.parametrize("causal", [0, 1])
def test_rows_that_see_nothing_weigh_a_constant_each(shares, cols, gr, causal):
    """Padding rows and queries in front of a request's first token: no more
    per tile than what an item costs by itself, whatever their number."""
    own = shares.idle()
    assert 1 <= own <= 1 + shares.item()
    for G in 1, 3, 4, 16, 33:
        for nq in 1, 300, 4096, 70000:
            n = _tiles(cols, G, nq)
            assert shares.weight(cols, gr, G, causal, nq, 0, n) == n * own
            if not causal:
                continue
            for end in 5, 300, 4000:
                if end >= nq:
                    continue
                seen = _tiles(cols, G, end)
                limit = shares.weight(cols, gr, G, 1, end, end, seen + 1) + (n - seen) * own
                assert shares.weight(cols, gr, G, 1, nq, end, n) <= limit


@pytest.mark.parametrize("cols,gr", FORMS)
def test_weights_follow_what_tiles_see(shares, cols, gr):
    """A tile weighs at least an idle one's cost, and within two tiles' columns
    and two granules what it sees beyond an item's own cost."""
    rng = random.Random(cols + gr)
    for _ in range(300):
        G = rng.choice([1, 2, 3, 4, 7, 16, 33])
        end, nq = (int(2 ** rng.uniform(0, 13)) for _ in range(2))
        causal = rng.random() < 0.8
        n = _tiles(cols, G, nq)
        at = [shares.weight(cols, gr, G, causal, nq, end, j) for j in range(n + 1)]
        assert at[0] == 0
        slack = 2 * cols / (G * gr) + 2
        for j in range(n):
            assert at[j + 1] - at[j] >= shares.idle()
            w = at[j + 1] - at[j] - shares.item()
            assert abs(w - _granules(cols, gr, G, causal, nq, end, j)) <= slack


@pytest.mark.parametrize("cols,gr", FORMS)
def test_the_bound_holds_for_every_request(shares, cols, gr):
    """No request weighs more than the bound per tile, so sums that the launch
    admits fit 32 bits: the weight computed in 32 is the one in any number."""
    rng = random.Random(cols * gr)
    for _ in range(2000):
        G = rng.choice([1, 2, 4, 5, 16, 33, 128])
        end = int(2 ** rng.uniform(0, 24))
        nq = int(2 ** rng.uniform(0, 30)) // G + 1
        n, most = _tiles(cols, G, nq), shares.most(cols, gr, G, end)
        if n * most >= 2 ** 31:
            continue
        last = 0
        for j in sorted({1, 2, n // 3 + 1, n // 2 + 1, n}):
            w = shares.weight(cols, gr, G, 1, nq, end, j)
            assert last <= w <= j * most or j > n
            last = w
        assert 0 < shares.weight(cols, gr, G, 0, nq, end, n) <= n * most

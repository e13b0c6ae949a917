"""Which kernel takes a product grouped by expert, and the GEMM's tiles (mlx_b200/csrc/experts_plan.h), compiled for the host."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx_b200", "csrc")
SHIM = """
#include "experts_plan.h"
using namespace luxcuda;
extern "C" int many(size_t rows, int experts, int K, int N, int bits, int gather, int sms) { return experts_have_many_rows({rows, experts, K, N, bits, gather != 0}, sms); }
extern "C" void plan(size_t rows, int experts, int K, int N, int bits, int gated, int pieces, int sms, int pair, int* out) {
    const ExpertsPlan p = plan_experts({rows, experts, K, N, bits, false}, gated != 0, pieces != 0, sms, pair);
    const int v[] = {p.bm, p.box, p.w_slots, p.n_tiles, p.pair, p.y_staged, (int)p.smem};
    for (int i = 0; i < 7; i++) out[i] = v[i];
}
"""


@pytest.fixture(scope="module")
def lib(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "shim.cpp"), "-o", str(d / "plan.so")], check=True)
    lib = C.CDLL(str(d / "plan.so"))
    lib.many.argtypes = [C.c_size_t] + [C.c_int] * 6
    lib.plan.argtypes = [C.c_size_t] + [C.c_int] * 8 + [C.c_void_p]
    return lib


def test_every_plan_can_be_launched(lib):
    """Heights that the matrix instructions take (pairs of CTAs: multiples of 32; one CTA: of 16), boxes that divide what a CTA fetches and of which a
    warp's 16 lanes a sub-block are enough, shared memory within a CTA's 227 KB, both kinds met."""
    rng = random.Random(4)
    kinds = set()
    for _ in range(20000):
        rows, experts = int(2 ** rng.uniform(0, 31)) % (2 ** 31 - 1) + 1, rng.choice([1, 2, 7, 64, 500, 1024, rng.randint(1, 1024)])
        N, bits, gated, pieces, pair = int(2 ** rng.uniform(0, 16)), rng.choice([4, 8]), rng.randint(0, 1), rng.randint(0, 1), rng.choice([-1, -1, 0, 1])
        out = (C.c_int * 7)()
        lib.plan(rows, experts, 64 * rng.randint(1, 256), N, bits, gated, pieces, 148, pair, out)
        bm, box, slots, n_tiles, is_pair, staged, smem = out
        kinds.add((is_pair, staged))
        half = bm // 2 if is_pair else bm
        assert bm % (32 if is_pair else 16) == 0 and 32 <= bm <= (256 if is_pair else 128)
        assert half % box == 0 and box % 16 == 0 and half // box <= 16
        assert smem <= 227 * 1024 and slots == (2 if bits == 8 else 1)
        tiles = -(-N // 128)
        assert n_tiles == (-(-tiles // 2) if is_pair else tiles)
        assert not staged or (is_pair and pieces)
    assert kinds == {(0, 0), (1, 0), (1, 1)}
    out = (C.c_int * 7)()
    lib.plan(10 ** 6, 8, 4096, 4096, 4, 0, 1, 147, 1, out)
    assert not out[4]  # (an odd number of SMs has no pairs of all of them)


def test_few_and_many_rows(lib):
    """One row an expert is for the decode kernel, a hundred for the GEMM, and there is one border between, but for the rounds of tiles that come in steps."""
    for experts, K, N, bits in ((8, 4096, 8192, 4), (64, 4096, 2816, 4), (64, 1408, 4096, 4), (64, 4096, 2816, 8), (128, 2048, 1024, 8), (1, 4096, 11008, 4)):
        for gather in (0, 1):
            got = [lib.many(mean * experts, experts, K, N, bits, gather, 148) for mean in range(1, 150)]
            assert not got[0] and all(got[99:]), (experts, K, N, bits, gather)
            assert sum(a != b for a, b in zip(got, got[1:])) <= 3, (experts, K, N, bits, gather, got)
    assert not lib.many(0, 8, 4096, 4096, 4, 0, 148)

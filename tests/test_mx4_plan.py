"""How mx4_matmul cuts a product with few rows of x (mlx_b200/csrc/mx4_plan.h), compiled for the host."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx_b200", "csrc")
SHIM = """
#include "mx4_plan.h"
extern "C" void plan(int M, int K, int N, int st, int sms, long long* out) {
    const luxcuda::mx4_plan::TilePlan t = luxcuda::mx4_plan::plan_tile(M, K, N, st, sms);
    const long long v[] = {t.bm, t.m_tiles, t.split, t.stages, t.stage_bytes, t.per_sm, t.tiles, t.sf_col, t.tmem_cols, t.smem};
    for (int i = 0; i < 10; i++) out[i] = v[i];
}
"""
KEYS = ("bm", "m_tiles", "split", "stages", "stage_bytes", "per_sm", "tiles", "sf_col", "tmem_cols", "smem")
SCALE_TILES = {"e8m0": 2, "e4m3": 4}  # along K per stage of 256 codes


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "shim.cpp"), "-o", str(d / "plan.so")], check=True)
    f = C.CDLL(str(d / "plan.so")).plan

    def call(M, K, N, fmt, sms=148):
        out = (C.c_longlong * 10)()
        f(M, K, N, SCALE_TILES[fmt], sms, out)
        return dict(zip(KEYS, out))
    return call


def shapes():
    rng = random.Random(11)
    for fmt in SCALE_TILES:
        for M in list(range(1, 161, 3)) + [64, 65, 80, 96, 97, 112, 113, 128, 129, 256, 300]:
            for K in (32, 256, 288, 512, 1024, 3840, 4096, 8192):
                for N in (1, 128, 384, 640, 1024, 4096, 28672):
                    yield M, K, N, fmt, 148
    for _ in range(20000):
        yield (int(4096 ** rng.random()), 32 * int(1024 ** rng.random()), int(60000 ** rng.random()), rng.choice(list(SCALE_TILES)), rng.choice([148, 148, 132, 16]))


def test_no_cta_of_a_cluster_waits_for_tensor_memory(plan):
    """CTAs of a cluster wait for one another: as many as an SM's shared memory (228 KB, one of them reserved per CTA) holds find room in its tensor
    memory (512 columns) at once.  M = 145, K = 3840, N = 384 at E4M3: clusters of eight with 256 columns each."""
    clusters = 0
    for shape in shapes():
        p = plan(*shape)
        assert p["smem"] <= 226 * 1024, shape
        if p["split"] > 1:
            clusters += 1
            assert 228 * 1024 // (p["smem"] + 1024) * p["tmem_cols"] <= 512, (shape, p)
    assert clusters > 10000
    assert plan(145, 3840, 384, "e4m3")["split"] == 8


def test_every_plan_can_be_launched(plan):
    for shape in shapes():
        M, K, N, fmt, sms = shape
        p = plan(*shape)
        st = SCALE_TILES[fmt]
        assert p["bm"] % 16 == 0 and 16 <= p["bm"] <= 128 and (p["m_tiles"] - 1) * p["bm"] < M <= p["m_tiles"] * p["bm"], (shape, p)
        assert p["tiles"] == p["m_tiles"] * ((N + 127) // 128)
        assert 1 <= p["split"] <= min(8, (K + 255) // 256)       # every part has a stage
        assert 2 <= p["stages"] <= 6
        assert p["stages"] * p["stage_bytes"] >= 128 * p["bm"] * 4  # the sums take the ring's place
        assert p["tmem_cols"] in (32, 64, 128, 256, 512) and p["sf_col"] >= p["bm"] and p["sf_col"] + p["stages"] * 2 * st * 4 <= p["tmem_cols"]
        assert p["smem"] >= p["stages"] * p["stage_bytes"] + 13 * 8 + 1024
        assert 1 <= p["per_sm"] <= 512 // p["tmem_cols"]

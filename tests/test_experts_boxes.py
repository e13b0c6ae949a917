"""Where the decode kernel's boxes of the experts' packed weights end (mlx_b200/csrc/experts_plan.h), compiled for the host: at the end of the weights or ahead of it."""
import ctypes as C
import os
import random
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mlx_b200", "csrc")
SHIM = """
#include "experts_plan.h"
using namespace luxcuda;
static long long end_of(const ExpertsMap& m, int n, unsigned long long row0, unsigned long long half0, unsigned long long kb0) {
    const unsigned long long at[4] = {0, row0, half0, kb0};
    long long last = 0;  // (a box's elements past the map's dimensions are filled in, not read)
    for (int d = 0; d < n; d++) {
        const unsigned long long hi = std::min(at[d] + m.box[d], m.dims[d]);
        if (hi <= at[d]) return 0;
        last += (hi - 1) * (d ? m.strides[d - 1] : 1);
    }
    return last + 1;
}
// the byte behind the last one that the boxes of a tile read
extern "C" long long tile_end(int experts, int K, int N, int bits, int gated, int kbc, int e, int tile) {
    const long long row = (long long)K * bits / 8;
    const int nkb = (row + 127) / 128, n_rt = (N + 15) / 16, tr = gated ? 8 : 16, half0 = gated ? 2 * e : e;
    const bool whole = experts_whole(row % 128 != 0, e, experts, tile, 1, n_rt) == 1;
    long long end = 0;
    for (int kb = 0; kb < nkb; kb += kbc)
        if (whole) end = std::max(end, end_of(experts_map(experts, K, N, bits, gated, kbc), 4, (long long)tile * tr, half0, kb));
    if (!whole) {  // single k-blocks of 128 bytes: the first dimension's coordinate
        const ExpertsMap m = experts_map_end(experts, K, N, bits, gated);
        for (int kb = 0; kb < nkb; kb++) {
            const long long hi = std::min<long long>(128LL * kb + 128, m.dims[0]);
            end = std::max(end, end_of(m, 3, (long long)tile * tr, half0, 0) - (long long)std::min<long long>(128, m.dims[0]) + hi);
        }
    }
    return end;
}
"""


@pytest.fixture(scope="module")
def tile_end(tmp_path_factory):
    d = tmp_path_factory.mktemp("boxes")
    (d / "shim.cpp").write_text(SHIM)
    subprocess.run(["g++", "-std=c++17", "-O1", "-Wall", "-Werror", "-shared", "-fPIC", "-I", CSRC, str(d / "shim.cpp"), "-o", str(d / "boxes.so")], check=True)
    f = C.CDLL(str(d / "boxes.so")).tile_end
    f.restype = C.c_longlong
    return f


def check(tile_end, E, K, N, bits, gated):
    row = K * bits // 8
    tiles, total = -(-N // 16), E * N * row
    nkb = -(-row // 128)
    kbc = -(-nkb // -(-nkb // 16))  # k-blocks a box, as the plan has them
    read = 0
    for e in range(E):
        for tile in range(tiles):
            end = tile_end(E, K, N, bits, gated, kbc, e, tile)
            assert end <= total, (E, K, N, bits, gated, e, tile, end - total)
            rows_end = (N // 2 if gated else 0) + min((tile + 1) * (8 if gated else 16), N)  # the tile's last row of the expert's
            assert end >= (e * N + rows_end) * row  # (all of the tile's own rows)
            read = max(read, end)
    assert read == total


@pytest.mark.parametrize("bits,K", [(4, 32), (4, 64), (4, 96), (4, 128), (4, 224), (4, 256), (4, 288), (4, 2912), (8, 32), (8, 64), (8, 96), (8, 128), (8, 160), (8, 2080)])
def test_no_box_ends_behind_the_weights(tile_end, bits, K):
    """Rows of 16 bytes and more, last tiles of one row and more, experts of one row: a box of whole k-blocks over them reaches up to seven rows further."""
    for E in (1, 2, 3, 17):
        for N in (1, 2, 15, 16, 17, 18, 31, 33, 129):
            check(tile_end, E, K, N, bits, False)
        for N in (16, 32, 272):
            check(tile_end, E, K, N, bits, True)


def test_any_shape(tile_end):
    rng = random.Random(8)
    for _ in range(400):
        bits, gated = rng.choice([4, 8]), rng.random() < 0.3
        check(tile_end, rng.randint(1, 40), 32 * rng.randint(1, 40), 16 * rng.randint(1, 9) if gated else rng.randint(1, 150), bits, gated)

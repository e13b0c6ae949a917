"""The microscaled format and block_norm as far as they go without a GPU: sizes, refusals, the table's layout, the oracle's own consistency."""
import ctypes as C
import os
import subprocess

import numpy as np
import pytest

import mlx_b200
from mlx_b200 import plugin as P
from oracle import mx4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def q():
    return mlx_b200.Plugin(require_gpu=False).quant


def test_scale_bytes(q):
    for rows, K, fmt in ((0, 32, 1), (1, 32, 1), (1, 32, 2), (128, 128, 1), (129, 160, 1), (300, 2880, 2), (11008, 4096, 1), (2 ** 31 - 1, 16384, 2)):
        assert q.mx4_scale_bytes(rows, K, fmt) == mx4.scale_bytes(rows, K, fmt)
    for rows, K, fmt in ((-1, 32, 1), (1, 0, 1), (1, 48, 2), (1, -32, 1), (1, 32, 0), (1, 32, 3)):
        assert q.mx4_scale_bytes(rows, K, fmt) == 0


def test_null_arguments(q):
    assert q.mx4_quantize(None, None, None, None, 1, 32, 0, 1, P.F32, 1.0) == P.ERR_INVALID
    assert q.mx4_dequantize(None, None, None, None, 1, 32, 1, P.F32, 1.0) == P.ERR_INVALID
    assert q.mx4_matmul(None, None, None, None, None, None, 1, 32, 1, 1, P.F32, 1.0) == P.ERR_INVALID
    assert q.block_norm(None, None, *[None] * 10) == P.ERR_INVALID
    prm = P.Context.block_norm_params(1, 32)
    assert q.block_norm(None, C.byref(prm), *[None] * 10) == P.ERR_INVALID


def test_header_as_a_c_host_sees_it(tmp_path):
    """The entries are found by the table's size; the parameter block has the mirror's layout."""
    src = tmp_path / "h.c"
    src.write_text("""
#include <stdio.h>
#include <stddef.h>
#include "lux_cuda_quant.h"
int main(void) {
    lux_gpu_quant_vtbl t = {0};
    t.magic = LUX_CUDA_QUANT_MAGIC;
    t.size = sizeof t;
    int now = LUX_CUDA_QUANT_HAS(&t, mx4_matmul) && LUX_CUDA_QUANT_HAS(&t, block_norm);
    t.size = offsetof(lux_gpu_quant_vtbl, mx4_scale_bytes);
    int before = LUX_CUDA_QUANT_HAS(&t, mx4_scale_bytes) || LUX_CUDA_QUANT_HAS(&t, block_norm);
    printf("%d %d %zu %zu %zu %zu", now, before, sizeof(lux_block_norm_params), offsetof(lux_block_norm_params, post_norm),
           offsetof(lux_block_norm_params, eps), offsetof(lux_block_norm_params, out_pre));
    return 0;
}
""")
    exe = tmp_path / "h"
    from mlx_b200 import build
    inc = build.reference_include() or os.path.join(ROOT, "include")
    subprocess.run(["/usr/bin/gcc", "-std=c11", "-Wall", "-Werror", "-I", inc, "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    now, before, size, post, eps, pre = map(int, subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split())
    B = P.BlockNormParams
    assert (now, before) == (1, 0)
    assert (size, post, eps, pre) == (C.sizeof(B), B.post_norm.offset, B.eps.offset, B.out_pre.offset)


@pytest.mark.parametrize("fmt", [mx4.E8M0, mx4.E4M3])
def test_oracle_round_trip(fmt):
    """What the format holds stays as it is when it is quantised again, and no value is further from its code than half a step."""
    rng = np.random.default_rng(fmt)
    w = rng.standard_normal((37, 160)).astype(np.float32)
    code, byte = mx4.quantize(w, fmt)
    v = mx4.values(code, byte, fmt)
    again = mx4.values(*mx4.quantize(v.astype(np.float32), fmt), fmt)
    top = np.abs(v).reshape(37, -1, mx4.BLOCK[fmt]).max(-1)
    same = np.repeat(top >= (4 if fmt == mx4.E8M0 else 6) * mx4.scale_values(byte, fmt), mx4.BLOCK[fmt], 1)
    np.testing.assert_array_equal(again[same], v[same])
    s = np.repeat(mx4.scale_values(byte, fmt), mx4.BLOCK[fmt], 1)
    a = np.abs(w) / s
    half = np.where(a < 2, 0.25, np.where(a < 4, 0.5, 1.0))
    assert (np.abs(v - w) / s <= np.where(a > 6, a - 6, half) + 1e-12).all()
    np.testing.assert_array_equal(mx4.unpack(mx4.pack(code)), code)
    np.testing.assert_array_equal(mx4.from_tiles(mx4.to_tiles(byte), *byte.shape), byte)


def test_extents_at_the_end_of_their_range(q):
    """Sizes whose rounding up would leave 32 bits have no scales, so no call takes them."""
    top = 2 ** 31 - 512
    for fmt in (mx4.E8M0, mx4.E4M3):
        assert q.mx4_scale_bytes(1, top, fmt) == mx4.scale_bytes(1, top, fmt)
        assert q.mx4_scale_bytes(2 ** 31 - 1, 32, fmt) == mx4.scale_bytes(2 ** 31 - 1, 32, fmt)
        for K in (top + 32, 2 ** 31 - 32):
            assert q.mx4_scale_bytes(1, K, fmt) == 0


def test_compiled_binding_checks_its_arguments():
    """The short calls reach the same entries without ctypes: same codes, and errors of Python's for what is no C argument."""
    from mlx_b200 import build
    if not os.path.exists(build.FASTCALL_PATH):
        pytest.skip("built without Python's headers: these calls go through ctypes")
    plugin = mlx_b200.Plugin(require_gpu=False)
    e = plugin.short_calls
    assert e is not plugin.quant
    prm = P.Context.block_norm_params(1, 32)
    assert e.mx4_quantize(None, None, None, None, 1, 32, 0, 1, P.F32, 1.0) == P.ERR_INVALID
    assert e.mx4_dequantize(None, None, None, None, 1, 32, 1, P.F32, 1) == P.ERR_INVALID
    assert e.mx4_matmul(None, None, None, None, None, None, 1, 32, 1, 1, P.F32, 1.0) == P.ERR_INVALID
    assert e.block_norm(None, prm, *[None] * 10) == e.block_norm(None, None, *[None] * 10) == P.ERR_INVALID
    for args, error in (((1, 32), TypeError), ((1 << 31, 32, 0, 1, P.F32, 1.0), OverflowError), ((-(1 << 31) - 1, 32, 0, 1, P.F32, 1.0), OverflowError), ((1.5, 32, 0, 1, P.F32, 1.0), TypeError),
                        ((1, 32, -1, 1, P.F32, 1.0), OverflowError), ((1, 32, 1 << 64, 1, P.F32, 1.0), OverflowError), ((1, 32, 0, 1, P.F32, "1"), TypeError), ((1, 32, 0, None, P.F32, 1.0), TypeError)):
        with pytest.raises(error):
            e.mx4_quantize(None, None, None, None, *args)
    for bad in (b"short", C.c_int(0), 7):
        with pytest.raises(TypeError):
            e.block_norm(None, bad, *[None] * 10)
    with pytest.raises(TypeError):
        e.mx4_matmul(None, "x", None, None, None, None, 1, 32, 1, 1, P.F32, 1.0)
    old = P.QuantVtbl(magic=P.QUANT_MAGIC, size=C.sizeof(P.QuantVtbl) - 8)
    with pytest.raises(ValueError):
        type(e)(C.addressof(old))
    assert P._short_calls(old) is old

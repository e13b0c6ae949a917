"""mx4_quantize with factors that are no ordinary numbers: what belongs to the format behind the last block of a row stays zero."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32
from mlx_b200 import plugin as P
from oracle import mx4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", [P.MX4_E8M0, P.MX4_E4M3])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("pre", [np.inf, -np.inf, np.nan, 3.4e38])
@pytest.mark.parametrize("rows,K", [(1, 32), (5, 96), (130, 544), (3, 1056)])
def test_bytes_of_blocks_past_the_last_are_zero(ctx, oracle, fmt, dtype, pre, rows, K):
    w = np.random.default_rng(K).choice([-2.0, -1.0, 1.0, 2.0], (rows, K)).astype(np.float32)
    src = ctx.upload(oracle.to_bf16(w) if dtype == BF16 else w)
    codes, scales = ctx.empty((rows, K // 8), np.uint32), ctx.upload(np.full(ctx.mx4_scale_bytes(rows, K, fmt), 0xA5, np.uint8))
    ctx.mx4_quantize(src, codes, scales, rows, K, fmt, dtype, pre)
    nb = K // mx4.BLOCK[fmt]
    tiles = mx4.from_tiles(scales.to_host(), (rows + 127) // 128 * 128, (nb + 3) // 4 * 4)
    assert not tiles[:rows, nb:].any()
    assert (tiles[rows:] == 0xA5).all()
    code, byte = mx4.quantize(w, fmt, pre)
    np.testing.assert_array_equal(tiles[:rows, :nb], byte)
    if not np.isnan(pre):
        np.testing.assert_array_equal(mx4.VALUES[mx4.unpack(codes.to_host())], mx4.VALUES[code])


@pytest.mark.parametrize("fmt", [P.MX4_E8M0, P.MX4_E4M3])
@pytest.mark.parametrize("K", [32, 288])
def test_a_product_behind_an_infinite_factor(ctx, fmt, K):
    """Infinities count as the largest value that a block holds: the product of such a row is a number, not NaN."""
    M, N = 3, 20
    x, w = np.ones((M, K), np.float32), np.full((N, K), 2.0 ** -20 if fmt == P.MX4_E8M0 else 1.0, np.float32)  # (sums within fp32's range)
    bx, bw = ctx.upload(x), ctx.upload(w)
    xq, xs = ctx.empty((M, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(M, K, fmt))
    wq, ws = ctx.empty((N, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(N, K, fmt))
    y = ctx.empty((M, N), np.float32)
    ctx.mx4_quantize(bx, xq, xs, M, K, fmt, F32, np.inf)
    ctx.mx4_quantize(bw, wq, ws, N, K, fmt, F32, 1.0)
    ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, N, fmt, F32, 2.0 ** -80)
    v, u = (mx4.values(*mx4.quantize(a, fmt, pre), fmt) for a, pre in ((x, np.inf), (w, 1.0)))
    want = 2.0 ** -80 * (v @ u.T)
    # fp32 sums of K products, K roundings at most, and the factor's
    assert (np.abs(y.to_host() - want) <= np.abs(want) * (K + 1) * 2.0 ** -23).all()

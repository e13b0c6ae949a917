"""Microscaled 4-bit floating point on the GPU: quantisation and expansion bit for bit, the product against 64 bits."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32, BackendError
from mlx_b200 import plugin as P
from oracle import mx4

pytestmark = pytest.mark.gpu
FORMATS = [P.MX4_E8M0, P.MX4_E4M3]


def at(ctx, a, shift=0):
    """`a` on the device, `shift` bytes past a 16-byte boundary."""
    room = ctx.upload(np.concatenate([np.zeros(shift, np.uint8), np.frombuffer(np.ascontiguousarray(a).tobytes(), np.uint8), np.zeros(16, np.uint8)]))
    return ctx.wrap(room.device_ptr + shift, a.nbytes, a.shape, a.dtype), room


def bf16(oracle, a):
    b = oracle.to_bf16(np.ascontiguousarray(a, np.float32))
    return b, oracle.from_bf16(b)


def quantize(ctx, w, rows, K, fmt, dtype, pre=1.0, ld=0, shift=0, fill=0xA5):
    src, _room = at(ctx, w, shift)
    codes = ctx.upload(np.full((rows, K // 8), 0xDEADBEEF, np.uint32))
    scales = ctx.upload(np.full(ctx.mx4_scale_bytes(rows, K, fmt), fill, np.uint8))
    ctx.mx4_quantize(src, codes, scales, rows, K, fmt, dtype, pre, ld)
    return codes, scales


def check_quantized(codes, scales, w32, rows, K, fmt, pre=1.0, fill=0xA5):
    code, byte = mx4.quantize(w32, fmt, pre)
    got, tiles = mx4.unpack(codes.to_host()), scales.to_host()
    nb, nt = byte.shape[1], (byte.shape[1] + 3) // 4
    np.testing.assert_array_equal(mx4.from_tiles(tiles, rows, nb), byte)
    every = tiles[mx4.tile_index((rows + 127) // 128 * 128, nt * 4)]
    assert not every[:rows, nb:].any()          # blocks behind the last of a row: zero
    assert (every[rows:] == fill).all()         # rows behind the last: as they were
    v, t = mx4.values(got, byte, fmt), mx4.values(code, byte, fmt)
    np.testing.assert_array_equal(v, t)         # (minus zero is zero)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("rows,K", [(1, 32), (3, 96), (1, 512), (5, 544), (127, 160), (129, 2880), (300, 64)])
def test_quantize(ctx, oracle, fmt, dtype, rows, K):
    rng = np.random.default_rng(rows * K + fmt)
    w = rng.standard_normal((rows, K)).astype(np.float32) * np.exp2(rng.integers(-6, 7, (rows, 1))).astype(np.float32)
    raw, w = bf16(oracle, w) if dtype == BF16 else (w, w)
    codes, scales = quantize(ctx, raw, rows, K, fmt, dtype)
    check_quantized(codes, scales, w, rows, K, fmt)
    codes, scales = quantize(ctx, raw, rows, K, fmt, dtype, pre=0.37, shift=4 if dtype == F32 else 2)
    check_quantized(codes, scales, w, rows, K, fmt, pre=0.37)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("ld", [128, 131, 136])
def test_quantize_column_block(ctx, oracle, fmt, dtype, ld):
    """Columns of a wider buffer, which ends with the last row's last column."""
    rows, K = 9, 96
    w = np.random.default_rng(ld).standard_normal((rows, ld)).astype(np.float32)
    raw, w = bf16(oracle, w) if dtype == BF16 else (w, w)
    raw = raw.reshape(-1)[:(rows - 1) * ld + K]
    codes, scales = quantize(ctx, raw, rows, K, fmt, dtype, ld=ld)
    check_quantized(codes, scales, w[:, :K], rows, K, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_borders(ctx, fmt):
    """Every border between two codes and its neighbours in fp32, under every scale that a block's largest value gives; and the
    borders between two scales."""
    rng = np.random.default_rng(5)
    borders = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], np.float32)
    near = np.concatenate([np.nextafter(borders, np.float32(0)), borders, np.nextafter(borders, np.float32(9)), -borders])[:28]
    bs = mx4.BLOCK[fmt]
    if fmt == P.MX4_E8M0:
        tops = np.exp2(np.arange(-126, 125, 7)).astype(np.float64) * 4
    else:
        tops = mx4.E4M3_VALUES[1:127] * 6
    rows = []
    for top in tops:
        s = top / (4 if fmt == P.MX4_E8M0 else 6)
        for part in np.array_split(near, 2):
            blk = rng.choice(part, bs).astype(np.float64)
            blk[:len(part)] = part
            blk[-1] = top / s
            rows.append((blk * s).astype(np.float32))
        for up in (0, np.inf):
            blk = (rng.standard_normal(bs) * s).clip(-top, top).astype(np.float32)
            blk[3] = np.nextafter(np.float32(top), np.float32(up))
            rows.append(blk)
    w = np.concatenate([np.stack(rows)] * (32 // bs), axis=1)
    codes, scales = quantize(ctx, w, len(w), 32, fmt, F32)
    check_quantized(codes, scales, w, len(w), 32, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
def test_quantize_extremes(ctx, fmt):
    tiny, big = np.float32(1e-45), np.finfo(np.float32).max
    rows = [np.zeros(32), np.full(32, -0.0), np.full(32, tiny), np.full(32, 1.2e-38), np.linspace(-1e-38, 1e-38, 32), np.full(32, big), np.linspace(-1.0, 1.0, 32) * np.float64(big),
            np.r_[np.inf, np.linspace(-4, 4, 31)], np.r_[np.linspace(-4, 4, 31), -np.inf], np.r_[np.inf, np.full(31, big)], np.r_[np.nan, np.linspace(-4, 4, 31)],
            np.r_[np.linspace(-4, 4, 20), np.nan, np.inf, np.zeros(10)], np.r_[np.linspace(1, 2, 16), np.zeros(16)], np.full(32, 2688.0), np.full(32, 2689.0), np.full(32, 0.0058)]
    w = np.stack(rows).astype(np.float32)
    w = np.concatenate([w, w[::-1]], axis=1)  # a block's neighbours are not touched by it
    codes, scales = quantize(ctx, w, len(w), 64, fmt, F32)
    check_quantized(codes, scales, w, len(w), 64, fmt)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("post,shift", [(1.0, 0), (0.0123, 4)])
def test_dequantize_every_code_and_scale(ctx, oracle, fmt, out, post, shift):
    K = 2 * mx4.BLOCK[fmt] if fmt == P.MX4_E4M3 else 96
    nb = K // mx4.BLOCK[fmt]
    byte = np.concatenate([np.arange(256), np.arange(256)[::-1]])[:512 // nb * nb].reshape(-1, nb).astype(np.uint8)
    rows = len(byte)
    code = np.tile(np.arange(16, dtype=np.uint8), (rows, K // 16))
    codes, scales = ctx.upload(mx4.pack(code)), ctx.upload(mx4.to_tiles(byte, 0xFF))
    dst, _room = at(ctx, np.zeros((rows, K), np.float32 if out == F32 else np.uint16), shift)
    ctx.mx4_dequantize(codes, scales, dst, rows, K, fmt, out, post)
    got = dst.to_host()
    with np.errstate(over="ignore", invalid="ignore"):
        want = mx4.values(code, byte, fmt).astype(np.float32) * np.float32(post)
    if out == BF16:
        got, want = oracle.from_bf16(got), oracle.from_bf16(oracle.to_bf16(want))
    np.testing.assert_array_equal(got, want)


@pytest.mark.parametrize("fmt", FORMATS)
def test_scales_past_32_bits_of_weights(ctx, fmt):
    """More than 2^31 values: the last rows come out as those of a small call."""
    K, rows = 16384, (1 << 31) // 16384 + 200
    rng = np.random.default_rng(fmt)
    tail = rng.standard_normal((200, K)).astype(np.float32)
    raw = (tail.view(np.uint32) >> 16).astype(np.uint16)
    src = ctx.alloc(rows * K * 2)
    part = ctx.wrap(src.device_ptr + (rows - 200) * K * 2, raw.nbytes, raw.shape, raw.dtype)
    part.from_host(raw)
    codes, scales = ctx.alloc(rows * K // 2), ctx.alloc(ctx.mx4_scale_bytes(rows, K, fmt))
    ctx.mx4_quantize(src, codes, scales, rows, K, fmt, BF16)
    got = ctx.wrap(codes.device_ptr + (rows - 200) * K // 2, 200 * K // 2, (200, K // 8), np.uint32).to_host()
    code, byte = mx4.quantize((raw.astype(np.uint32) << 16).view(np.float32), fmt)
    np.testing.assert_array_equal(VAL(mx4.unpack(got)), VAL(code))
    back = ctx.alloc(rows * K * 2)
    ctx.mx4_dequantize(codes, scales, back, rows, K, fmt, BF16)
    got = ctx.wrap(back.device_ptr + (rows - 200) * K * 2, 200 * K * 2, (200, K), np.uint16).to_host()
    want = mx4.values(code, byte, fmt)  # at most six significant bits: exact in bf16
    np.testing.assert_array_equal((got.astype(np.uint32) << 16).view(np.float32), want)
    for b in (src, codes, scales, back):
        b.free()


def VAL(code):
    return mx4.VALUES[code]


def operand(ctx, rng, rows, K, fmt, fill=0xFF):
    """Random codes and scales on the device (NaN scales behind the last row) and their values."""
    code, byte = mx4.random_operand(rng, rows, K, fmt)
    return ctx.upload(mx4.pack(code)), ctx.upload(mx4.to_tiles(byte, fill)), mx4.values(code, byte, fmt)


def matmul(ctx, x, w, M, K, N, fmt, y_dtype, alpha=1.0, shift=0):
    y, _room = at(ctx, np.full((M, N), 0x7FC1, np.uint16) if y_dtype == BF16 else np.full((M, N), np.nan, np.float32), shift)
    ctx.mx4_matmul(x[0], x[1], w[0], w[1], y, M, K, N, fmt, y_dtype, alpha)
    return y.to_host()


def check_product(oracle, y, xv, wv, alpha, y_dtype):
    """Products are exact; a sum of K of them in fp32, whatever its order and whether it rounds or truncates, is off by at most
    K * 2^-23 of the sum of magnitudes; alpha and the rounding to y's type: half a step each."""
    t = alpha * (xv @ wv.T)
    mag = abs(alpha) * (np.abs(xv) @ np.abs(wv).T)
    tol = mag * xv.shape[1] * 2.0 ** -23 + np.abs(t) * 2.0 ** -24
    got = y.astype(np.float64)
    if y_dtype == BF16:
        got = oracle.from_bf16(y).astype(np.float64)
        tol = tol + (np.abs(t) + tol) * 2.0 ** -8
    bad = ~(np.abs(got - t) <= tol)
    assert not bad.any(), (int(bad.sum()), np.argwhere(bad)[:5], got[bad][:5], t[bad][:5])


SHAPES = [(1, 32, 1), (1, 64, 16), (1, 1024, 1024), (2, 96, 130), (3, 544, 127), (5, 2880, 333), (8, 4096, 256), (16, 8192, 128), (16, 11008, 64), (17, 512, 128),
          (33, 2048, 129), (48, 4096, 300), (100, 992, 77), (128, 1024, 512), (129, 256, 128), (200, 160, 1000), (257, 2880, 515), (300, 32, 40), (520, 1056, 1030),
          (1024, 512, 2048)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", SHAPES)
def test_matmul(ctx, oracle, fmt, M, K, N):
    rng = np.random.default_rng(M * 7 + K * 3 + N)
    xq, xs, xv = operand(ctx, rng, M, K, fmt)
    wq, ws, wv = operand(ctx, rng, N, K, fmt)
    for y_dtype, alpha, shift in ((BF16, 1.0, 0), (F32, 0.3, 4)):
        y = matmul(ctx, (xq, xs), (wq, ws), M, K, N, fmt, y_dtype, alpha, shift)
        check_product(oracle, y, xv, wv, np.float64(np.float32(alpha)), y_dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(520, 32, 8192), (1300, 96, 3333), (2048, 544, 2050), (257, 4128, 9001), (700, 1024, 5004), (1100, 2880, 4096),
                                   (2048, 544, 5002), (1300, 2080, 8333), (1500, 96, 9001), (2100, 4128, 2311), (600, 2048, 5000)])
def test_matmul_pairs(ctx, oracle, fmt, M, K, N):
    """Many rows: several tiles per pair of CTAs, K inside a stage, rows of y on any boundary, halves of tiles without rows.  Four of the shapes are so near
    to where single CTAs are as fast that either may take them; the others are the pairs'."""
    either = (M, N) in ((1300, 3333), (2048, 2050), (700, 5004), (1100, 4096))
    rng = np.random.default_rng(M + K + N)
    xq, xs, xv = operand(ctx, rng, M, K, fmt)
    wq, ws, wv = operand(ctx, rng, N, K, fmt)
    for y_dtype, alpha, shift in ((BF16, 1.0, 0), (F32, 0.3, 4), (F32, 1.0, 0), (BF16, -2.0, 2)):
        y = matmul(ctx, (xq, xs), (wq, ws), M, K, N, fmt, y_dtype, alpha, shift)
        assert either or ctx.last_kernel().startswith("mx4_pairs")
        check_product(oracle, y, xv, wv, np.float64(np.float32(alpha)), y_dtype)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(3, 512, 200), (200, 544, 300), (600, 288, 4100)])
def test_matmul_places(ctx, oracle, fmt, M, K, N):
    """One value per row of x, another place each: every code, scale and row has to be read from where it lies."""
    rng = np.random.default_rng(M)
    wq, ws, wv = operand(ctx, rng, N, K, fmt)
    bs = mx4.BLOCK[fmt]
    for shift in (0, 17):
        code, byte = np.zeros((M, K), np.uint8), np.full((M, K // bs), 127 if fmt == P.MX4_E8M0 else 0x38, np.uint8)
        place = (np.arange(M) * 37 + shift) % K
        code[np.arange(M), place] = 2  # 1.0
        y = matmul(ctx, (ctx.upload(mx4.pack(code)), ctx.upload(mx4.to_tiles(byte, 0xFF))), (wq, ws), M, K, N, fmt, F32)
        np.testing.assert_array_equal(y, wv.T[place].astype(np.float32))


@pytest.mark.parametrize("fmt", FORMATS)
def test_matmul_nan_and_infinite_scales_stay_in_their_rows(ctx, oracle, fmt):
    M, K, N = 20, 256, 150
    rng = np.random.default_rng(2)
    xc, xb = mx4.random_operand(rng, M, K, fmt)
    wc, wb = mx4.random_operand(rng, N, K, fmt)
    xb[7, 3] = 255 if fmt == P.MX4_E8M0 else 127
    wb[100, 1] = 255 if fmt == P.MX4_E8M0 else 127
    y = matmul(ctx, (ctx.upload(mx4.pack(xc)), ctx.upload(mx4.to_tiles(xb, 0xFF))), (ctx.upload(mx4.pack(wc)), ctx.upload(mx4.to_tiles(wb, 0xFF))), M, K, N, fmt, F32)
    assert np.isnan(y[7]).all() and np.isnan(y[:, 100]).all()
    rows, cols = np.arange(M) != 7, np.arange(N) != 100
    check_product(oracle, y[rows][:, cols], mx4.values(xc, xb, fmt)[rows], mx4.values(wc, wb, fmt)[cols], 1.0, F32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(1, 4096, 4096), (16, 2048, 640), (300, 1024, 900), (600, 2048, 5000)])
def test_matmul_is_repeatable_and_replayable(ctx, oracle, fmt, M, K, N):
    """The same bits from call to call and from a recorded graph, which follows new activations; launches one behind the other
    without a wait between them."""
    rng = np.random.default_rng(M + N)
    wq, ws, wv = operand(ctx, rng, N, K, fmt)
    xs = [bf16(oracle, rng.standard_normal((M, K)))[0] for _ in range(3)]
    bx, xq, sc, y = ctx.upload(xs[0]), ctx.empty((M, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(M, K, fmt)), ctx.empty((M, N), np.float32)
    pre = 64.0 if fmt == P.MX4_E4M3 else 1.0

    def step():
        ctx.mx4_quantize(bx, xq, sc, M, K, fmt, BF16, pre)
        ctx.mx4_matmul(xq, sc, wq, ws, y, M, K, N, fmt, F32, 1 / pre)

    want = []
    for x in xs:
        bx.from_host(x)
        for _ in range(4):
            step()
        want.append(y.to_host())
        code, byte = mx4.quantize(oracle.from_bf16(x), fmt, pre)
        check_product(oracle, want[-1], mx4.values(code, byte, fmt), wv, 1 / pre, F32)
    ctx.graph_begin()
    step()
    g = ctx.graph_end()
    for x, t in zip(xs, want):
        bx.from_host(x)
        for _ in range(5):
            ctx.graph_launch(g)
        assert np.array_equal(y.to_host().view(np.uint32), t.view(np.uint32))
    ctx.graph_destroy(g)


@pytest.mark.parametrize("fmt", FORMATS)
def test_weights_quantized_right_before_they_are_used(ctx, oracle, fmt):
    """The product fetches weights ahead of the kernel before it, unless that kernel writes them."""
    M, K, N = 4, 1024, 700
    rng = np.random.default_rng(11)
    xq, xs, xv = operand(ctx, rng, M, K, fmt)
    wq, ws = ctx.empty((N, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(N, K, fmt))
    y = ctx.empty((M, N), np.float32)
    ws_host = [rng.standard_normal((N, K)).astype(np.float32) for _ in range(3)]
    src = [ctx.upload(w) for w in ws_host]
    for _ in range(3):
        for w, b in zip(ws_host, src):
            ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, N, fmt, F32)  # (opens the chain)
            ctx.mx4_quantize(b, wq, ws, N, K, fmt, F32)
            ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, N, fmt, F32)
            check_product(oracle, y.to_host(), xv, mx4.values(*mx4.quantize(w, fmt), fmt), 1.0, F32)


def test_two_contexts_side_by_side(plugin, oracle):
    fmt, M, K, N = P.MX4_E8M0, 8, 2048, 1500
    a, b = plugin.context(0), plugin.context(0)
    try:
        rng = np.random.default_rng(3)
        sets = []
        for c in (a, b):
            xq, xs, xv = operand(c, rng, M, K, fmt)
            wq, ws, wv = operand(c, rng, N, K, fmt)
            sets.append((c, xq, xs, wq, ws, c.empty((M, N), np.float32), xv, wv))
            c.sync()
        for _ in range(20):
            for c, xq, xs, wq, ws, y, _, _ in sets:
                c.mx4_matmul(xq, xs, wq, ws, y, M, K, N, fmt, F32)
        for c, *_, y, xv, wv in sets:
            check_product(oracle, y.to_host(), xv, wv, 1.0, F32)
    finally:
        a.close()
        b.close()


def test_refusals(ctx, plugin):
    fmt = P.MX4_E8M0
    M, K, N = 3, 64, 20
    x, xq, xs = ctx.empty((M, K), np.float32), ctx.empty((M, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(M, K, fmt))
    wq, ws, y = ctx.empty((N, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(N, K, fmt)), ctx.empty((M, N), np.float32)
    odd = ctx.wrap(xq.device_ptr + 4, xq.nbytes - 4)
    ctx.mx4_quantize(x, xq, xs, 0, K, fmt, F32)                  # no rows: nothing to do
    ctx.mx4_dequantize(xq, xs, x, 0, K, fmt, F32)
    ctx.mx4_matmul(xq, xs, wq, ws, y, 0, K, N, fmt, F32)
    ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, 0, fmt, F32)
    bad = [lambda: ctx.mx4_quantize(x, xq, xs, M, K, 3, F32), lambda: ctx.mx4_quantize(x, xq, xs, M, 48, fmt, F32), lambda: ctx.mx4_quantize(x, xq, xs, -1, K, fmt, F32),
           lambda: ctx.mx4_quantize(x, xq, xs, M, 0, fmt, F32), lambda: ctx.mx4_quantize(x, xq, xs, M, K, fmt, P.F16), lambda: ctx.mx4_quantize(x, xq, xs, M, K, fmt, F32, ld=63),
           lambda: ctx.mx4_quantize(x, xq, xs, M, K, fmt, F32, ld=65), lambda: ctx.mx4_quantize(x, xq, xs, M, K, fmt, F32, ld=1 << 62), lambda: ctx.mx4_quantize(x, xq, xs, M + 1, K, fmt, F32),
           lambda: ctx.mx4_quantize(x, xq, xs, M, K, P.MX4_E8M0, F32, ld=K + 1), lambda: ctx.mx4_quantize(x, odd, xs, 1, 32, fmt, F32), lambda: ctx.mx4_quantize(x, x, xs, M, K, fmt, F32),
           lambda: ctx.mx4_dequantize(xq, xs, x, M, K, fmt, P.F16), lambda: ctx.mx4_dequantize(xq, xs, x, 129, K, fmt, F32), lambda: ctx.mx4_dequantize(xq, xs, xq, 1, 32, fmt, F32),
           lambda: ctx.mx4_dequantize(odd, xs, x, 1, 32, fmt, F32), lambda: ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, N + 1, fmt, F32), lambda: ctx.mx4_matmul(xq, xs, wq, ws, y, M + 1, K, N, fmt, F32),
           lambda: ctx.mx4_matmul(xq, xs, wq, ws, y, M, K + 32, N, fmt, F32), lambda: ctx.mx4_matmul(xq, xs, wq, ws, y, M, 0, N, fmt, F32), lambda: ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, N, 0, F32),
           lambda: ctx.mx4_matmul(xq, xs, wq, ws, y, M, K, N, fmt, P.I32), lambda: ctx.mx4_matmul(xq, xs, wq, ws, wq, M, K, N, fmt, BF16), lambda: ctx.mx4_matmul(odd, xs, wq, ws, y, 1, 32, N, fmt, F32)]
    for call in bad:
        with pytest.raises(BackendError) as e:
            call()
        assert e.value.code == P.ERR_INVALID
    assert ctx.mx4_scale_bytes(1, 48, fmt) == 0 and ctx.mx4_scale_bytes(1, 64, 7) == 0 and ctx.mx4_scale_bytes(-1, 64, fmt) == 0
    assert plugin.last_error()


def test_refuses_lengths_past_their_range(ctx, plugin):
    """K whose last chunk would pass 2^31: refused for that, ahead of any look at the buffers' sizes."""
    K, fmt = 2 ** 31 - 32, P.MX4_E8M0
    b = [ctx.alloc(4096) for _ in range(5)]
    for call in (lambda: ctx.mx4_quantize(b[0], b[1], b[2], 1, K, fmt, BF16), lambda: ctx.mx4_dequantize(b[1], b[2], b[0], 1, K, fmt, BF16),
                 lambda: ctx.mx4_matmul(b[0], b[1], b[2], b[3], b[4], 1, K, 1, fmt, BF16),
                 lambda: ctx.block_norm(ctx.block_norm_params(1, K, pre=P.NORM_RMS, out_format=fmt), b[0], None, None, None, None, None, None, None, b[1], b[2])):
        with pytest.raises(BackendError) as e:
            call()
        assert e.value.code == P.ERR_INVALID and "2^31 - 512" in plugin.last_error()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("K,N", [(512, 200), (2080, 1300)])
def test_matmul_of_a_matrix_with_itself(ctx, oracle, fmt, K, N):
    """Both operands in the same buffers."""
    w, ws, wv = operand(ctx, np.random.default_rng(K), N, K, fmt)
    y = ctx.empty((N, N), np.float32)
    ctx.mx4_matmul(w, ws, w, ws, y, N, K, N, fmt, F32)
    check_product(oracle, y.to_host(), wv, wv, 1.0, F32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("M,K,N", [(1, 4096, 1024), (20, 2048, 2048)])
def test_products_of_one_x_and_x_written_anew(ctx, oracle, fmt, M, K, N):
    """Several layers on the same x (which no kernel still at work writes), then x from a layer's output, then layers again: without a
    wait between the calls as with one after each."""
    rng = np.random.default_rng(M)
    ws = [operand(ctx, rng, N, K, fmt)[:2] for _ in range(6)]
    start = ctx.upload(oracle.to_bf16(rng.standard_normal((M, K)).astype(np.float32)))
    xq, xs = ctx.empty((M, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(M, K, fmt))
    wide = ctx.empty((M, K), np.uint16)

    def steps(after):
        ys = [ctx.empty((M, N), np.float32) for _ in ws]
        for i, w in enumerate(ws):
            if i % 3 == 0:
                if i:  # (of the last product, where it is as wide)
                    for _ in range(2):
                        ctx.mx4_quantize(ys[i - 1] if N >= K else wide, xq, xs, M, K, fmt, F32 if N >= K else BF16, 0.01)
                        after()
                else:
                    ctx.mx4_quantize(start, xq, xs, M, K, fmt, BF16)
                    after()
            ctx.mx4_matmul(xq, xs, *w, ys[i], M, K, N, fmt, F32)
            after()
        return [y.to_host() for y in ys]

    wide.from_host(oracle.to_bf16(rng.standard_normal((M, K)).astype(np.float32)))
    want = steps(ctx.sync)
    assert any(not np.array_equal(a, b) for a, b in zip(want[:3], want[3:]))
    for _ in range(20):
        for a, b in zip(steps(lambda: None), want):
            np.testing.assert_array_equal(a, b)


@pytest.mark.parametrize("seed,M,K", [(0, 8, 1024), (1, 1, 4096), (2, 40, 512), (3, 300, 1024), (4, 16, 2048), (5, 700, 2048)])
def test_any_order_of_calls_is_as_with_a_wait_after_each(ctx, oracle, seed, M, K):
    """Random programs over a few buffers, so that calls read what the one before writes, write what it reads, or have nothing to do with
    it: quantisations of activations and of weights, products, row steps, older chain kernels.  Eagerly and as a replayed graph, against one call at a time."""
    rng = np.random.default_rng(seed)
    fmt = P.MX4_E8M0 if seed % 2 else P.MX4_E4M3
    bits = lambda shape: oracle.to_bf16(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    acts = [ctx.upload(bits((M, K))) for _ in range(4)]
    raw = [ctx.upload(bits((K, K))) for _ in range(2)]  # weights before the format
    codes = [(ctx.empty((M, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(M, K, fmt))) for _ in range(3)]
    layers = [(ctx.empty((K, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(K, K, fmt))) for _ in range(3)]
    start = [(b, b.to_host()) for b in acts]
    prm = ctx.block_norm_params(M, K, post=P.NORM_RMS, pre=P.NORM_RMS, eps=1e-5, res_scale=0.5)
    prm_mx = ctx.block_norm_params(M, K, post=P.NORM_RMS, pre=P.NORM_RMS, eps=1e-5, res_scale=0.5, out_format=fmt)
    pick = lambda a: int(rng.integers(len(a)))  # noqa: E731
    steps = [lambda q=c: ctx.mx4_quantize(acts[0], *q, M, K, fmt, BF16) for c in codes] + [lambda q=w: ctx.mx4_quantize(raw[0], *q, K, K, fmt, BF16) for w in layers]
    for _ in range(70):
        kind = rng.random()
        a, b, c, w = pick(acts), pick(acts), codes[pick(codes)], layers[pick(layers)]
        if kind < 0.35:
            steps.append(lambda a=a, c=c: ctx.mx4_quantize(acts[a], *c, M, K, fmt, BF16))
        elif kind < 0.75:
            steps.append(lambda a=a, c=c, w=w: ctx.mx4_matmul(*c, *w, acts[a], M, K, K, fmt, BF16, 1.0 / K ** 0.5))
        elif kind < 0.8:
            steps.append(lambda r=raw[pick(raw)], w=w: ctx.mx4_quantize(r, *w, K, K, fmt, BF16))
        elif kind < 0.9:
            d = (a + 1 + pick(acts[1:])) % len(acts)
            r = next(i for i in range(len(acts)) if i not in (a, d))
            steps.append(lambda a=a, d=d, r=r: ctx.block_norm(prm, acts[a], None, acts[r], None, None, None, None, acts[r], acts[d]))
        elif kind < 0.95:
            r = (a + 1) % len(acts)
            steps.append(lambda a=a, r=r, c=c: ctx.block_norm(prm_mx, acts[a], None, acts[r], None, None, None, None, acts[r], *c))
        else:
            if a != b:
                steps.append(lambda a=a, b=b: ctx.rms_norm(acts[a], acts[b], M, K, 1e-5, BF16, BF16))

    def reset():
        for b, v in start:
            b.from_host(v)

    def state():
        return [b.to_host() for b in acts] + [x.to_host() for c in codes + layers for x in c[:1]]

    reset()
    for s in steps:
        s()
        ctx.sync()
    want = state()
    for _ in range(4):
        reset()
        for s in steps:
            s()
        for got, w in zip(state(), want):
            np.testing.assert_array_equal(got, w)
    reset()
    ctx.graph_begin()
    for s in steps:
        s()
    g = ctx.graph_end()
    for _ in range(4):
        reset()
        ctx.graph_launch(g)
        for got, w in zip(state(), want):
            np.testing.assert_array_equal(got, w)
    ctx.graph_destroy(g)

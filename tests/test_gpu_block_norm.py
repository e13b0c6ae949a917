"""The row step between two blocks (block_norm) against 64 bits, and a decode step of the calls that it stands between."""
import itertools

import numpy as np
import pytest

from mlx_b200 import BF16, F32, BackendError
from mlx_b200 import plugin as P
from oracle import mx4

pytestmark = pytest.mark.gpu
EPS = 1e-5


def place(ctx, oracle, a, dtype, shift=0):
    """(buffer, values as the device sees them); shift: elements past a 16-byte boundary."""
    raw = oracle.to_bf16(np.ascontiguousarray(a, np.float32)) if dtype == BF16 else np.ascontiguousarray(a, np.float32)
    room = ctx.upload(np.concatenate([np.zeros(shift, raw.dtype), raw.reshape(-1)]))
    b = ctx.wrap(room.device_ptr + shift * raw.itemsize, raw.nbytes, raw.shape, raw.dtype)
    b.room = room
    return b, (oracle.from_bf16(raw) if dtype == BF16 else raw).astype(np.float64).reshape(a.shape)


def empty(ctx, shape, dtype, shift=0):
    item = 2 if dtype == BF16 else 4
    n = int(np.prod(shape))
    room = ctx.upload(np.full(n * item + shift * item + 64, 0xC3, np.uint8))
    b = ctx.wrap(room.device_ptr + shift * item, n * item, tuple(shape), np.uint16 if dtype == BF16 else np.float32)
    b.room = room
    return b


def host(oracle, b, dtype):
    return (oracle.from_bf16(b.to_host()) if dtype == BF16 else b.to_host()).astype(np.float64)


def norm_tolerance(v, kind, w, b, out):
    """fp32 statistics: a sum over dim elements in at most 64 levels (elements per thread, then trees) is off by 64 * 2^-24 of the sum of magnitudes,
    the mean by that of the mean magnitude; the root, the products and the bias: a few roundings of 2^-24 each."""
    if kind == 0:
        return np.zeros_like(out)
    mean = np.abs(v).mean(-1, keepdims=True)
    c = v - v.mean(-1, keepdims=True) if kind == 2 else v
    inv = 1 / np.sqrt((c * c).mean(-1, keepdims=True) + EPS)
    w = 1.0 if w is None else np.abs(w)
    shift = 64 * 2.0 ** -24 * mean if kind == 2 else 0.0
    rel = 72 * 2.0 ** -24 + (64 * 2.0 ** -24 * mean * inv) ** 2  # (of inv: half the sum's error and, through the mean, its square)
    return (shift * (1 + rel) + np.abs(c) * rel) * inv * w + 4 * 2.0 ** -24 * (np.abs(out) + (0 if b is None else np.abs(b)))


def rounding(t, dtype):
    return np.abs(t) * (2.0 ** -8 if dtype == BF16 else 2.0 ** -24)


def run(ctx, oracle, rows, dim, post, pre, gate_rows, act, xd, rd, od, seed=0, shift=0, h_ld=0, gate_ld=0, weights=True, res=1.0, branch=1.0, use_r=True, in_place=False, offset=0.0):
    rng = np.random.default_rng(seed + rows * dim)
    N = lambda shape, s=1.0, m=0.0: (rng.standard_normal(shape) * s + m).astype(np.float32)  # noqa: E731
    hw, gw = h_ld or dim, gate_ld or dim
    bh, h = place(ctx, oracle, N((rows, hw), 0.8, offset), xd, shift)
    br, r = place(ctx, oracle, N((rows, dim), 2.0), rd, shift) if use_r else (None, None)
    bg = g = None
    if gate_rows is not None:
        n = (rows + gate_rows - 1) // gate_rows if gate_rows else 1
        bg, g = place(ctx, oracle, N((n, gw)), xd, shift)
    ws = {k: place(ctx, oracle, N((dim,), 0.2, 0.0 if k.endswith("b") else 1.0), F32, shift) if weights and kind >= need else (None, None)
          for k, kind, need in (("post_w", post, 1), ("post_b", post, 2), ("pre_w", pre, 1), ("pre_b", pre, 2))}
    new = br if in_place else empty(ctx, (rows, dim), rd, shift)
    out = empty(ctx, (rows, dim), od, shift)
    prm = ctx.block_norm_params(rows, dim, post=post, pre=pre, gate_act=act, gate_rows=gate_rows or 0, x_dtype=xd, r_dtype=rd, out_dtype=od, eps=EPS, res_scale=res,
                                branch_scale=branch, h_ld=h_ld, gate_ld=gate_ld)
    ctx.block_norm(prm, bh, bg, br, ws["post_w"][0], ws["post_b"][0], ws["pre_w"][0], ws["pre_b"][0], new, out)
    w = {k: v[1] for k, v in ws.items()}
    hv = h[:, :dim]
    b = mx4.norm(hv, post, EPS, w["post_w"], w["post_b"])
    tol = norm_tolerance(hv, post, w["post_w"], w["post_b"], b)
    if g is not None:
        a = mx4.gate(np.repeat(g[:, :dim], gate_rows, 0)[:rows] if gate_rows else g[:, :dim], act)
        tol = tol * np.abs(a) + np.abs(b * a) * 8 * 2.0 ** -24  # (the functions of CUDA: two or three steps)
        b = b * a
    s32 = lambda v: np.float64(np.float32(v))  # noqa: E731
    t = s32(branch) * b + (s32(res) * r if r is not None else 0)
    tol = abs(s32(branch)) * tol + 2 * 2.0 ** -24 * (np.abs(s32(branch) * b) + np.abs(t))
    got = host(oracle, new, rd)
    assert (np.abs(got - t) <= tol + rounding(np.abs(t) + tol, rd)).all(), np.abs(got - t).max()
    # the second norm is that of the stream as it was stored
    o = mx4.norm(got, pre, EPS, w["pre_w"], w["pre_b"])
    tol = norm_tolerance(got, pre, w["pre_w"], w["pre_b"], o)
    res_out = host(oracle, out, od)
    assert (np.abs(res_out - o) <= tol + rounding(np.abs(o) + tol, od)).all(), np.abs(res_out - o).max()
    return got, res_out


KINDS = [P.NORM_NONE, P.NORM_RMS, P.NORM_LAYER]


@pytest.mark.parametrize("post,pre", list(itertools.product(KINDS, KINDS)))
@pytest.mark.parametrize("dim", [4096, 333])
def test_norms(ctx, oracle, post, pre, dim):
    run(ctx, oracle, 5, dim, post, pre, 1, P.GATE_SIGMOID, BF16, BF16, BF16, seed=post * 3 + pre)
    run(ctx, oracle, 5, dim, post, pre, None, 0, F32, F32, F32, seed=post * 3 + pre, res=0.7, branch=-0.3)


@pytest.mark.parametrize("xd,rd,od", list(itertools.product([F32, BF16], repeat=3)))
@pytest.mark.parametrize("shift", [0, 3])
def test_types_and_alignment(ctx, oracle, xd, rd, od, shift):
    run(ctx, oracle, 3, 264, 1, 2, 1, P.GATE_TANH, xd, rd, od, shift=shift)
    run(ctx, oracle, 2, 41, 2, 1, 1, P.GATE_IDENTITY, xd, rd, od, shift=shift)


@pytest.mark.parametrize("rows,dim", [(1, 1), (1, 2), (2, 8), (1, 32), (1, 8192), (7, 8200), (700, 512), (301, 1031), (2, 16384), (300, 16392), (3, 16385), (3, 32768), (2, 40000), (2, 32776)])
def test_sizes(ctx, oracle, rows, dim):
    run(ctx, oracle, rows, dim, P.NORM_RMS, P.NORM_LAYER if dim > 1 else P.NORM_RMS, 0, P.GATE_SIGMOID, BF16, F32, BF16)


@pytest.mark.parametrize("gate_rows", [0, 1, 2, 3, 100])
def test_rows_that_share_a_gate(ctx, oracle, gate_rows):
    run(ctx, oracle, 10, 96, 1, 1, gate_rows, P.GATE_IDENTITY, BF16, BF16, BF16)


@pytest.mark.parametrize("h_ld,gate_ld", [(300, 264), (264, 300), (264 + 8, 264 + 16), (601, 277)])
@pytest.mark.parametrize("xd", [F32, BF16])
def test_column_blocks(ctx, oracle, h_ld, gate_ld, xd):
    run(ctx, oracle, 4, 264, 2, 1, 1, P.GATE_TANH, xd, BF16, F32, h_ld=h_ld, gate_ld=gate_ld)


@pytest.mark.parametrize("dim", [512, 99, 40000])
def test_in_place_without_weights_and_without_stream(ctx, oracle, dim):
    run(ctx, oracle, 6, dim, 1, 2, 0, 0, BF16, F32, BF16, in_place=True)
    run(ctx, oracle, 6, dim, 2, 1, None, 0, BF16, BF16, BF16, weights=False, in_place=True)
    run(ctx, oracle, 6, dim, 1, 1, 1, 0, F32, BF16, F32, use_r=False)


def test_mean_far_from_zero(ctx, oracle):
    """The variance is that of the differences, not the difference of two large sums."""
    run(ctx, oracle, 4, 4096, P.NORM_LAYER, P.NORM_LAYER, None, 0, F32, F32, F32, offset=300.0, use_r=False)


def test_stream_alone(ctx, oracle):
    """Without a block's output: the norm before the first block; without an output: the residual sum alone."""
    rng = np.random.default_rng(1)
    rows, dim = 4, 160
    br, r = place(ctx, oracle, rng.standard_normal((rows, dim)), BF16)
    out = empty(ctx, (rows, dim), F32)
    ctx.block_norm(ctx.block_norm_params(rows, dim, pre=P.NORM_RMS, out_dtype=F32, eps=EPS), None, None, br, None, None, None, None, None, out)
    want = mx4.norm(r, 1, EPS)
    assert (np.abs(host(oracle, out, F32) - want) <= norm_tolerance(r, 1, None, None, want)).all()
    bh, h = place(ctx, oracle, rng.standard_normal((rows, dim)), BF16)
    new = empty(ctx, (rows, dim), F32)
    ctx.block_norm(ctx.block_norm_params(rows, dim, r_dtype=F32, branch_scale=0.25), bh, None, None, None, None, None, None, new, None)
    assert np.array_equal(host(oracle, new, F32), 0.25 * h)


def test_infinities_and_nan_stay_in_their_row(ctx, oracle):
    rng = np.random.default_rng(4)
    rows, dim = 5, 256
    x = rng.standard_normal((rows, dim)).astype(np.float32)
    clean = x.copy()
    x[1, 7], x[3, 200] = np.nan, np.inf
    got = []
    for a in (x, clean):
        bh, _ = place(ctx, oracle, a, BF16)
        br, _ = place(ctx, oracle, np.ones((rows, dim)), BF16)
        new, out = empty(ctx, (rows, dim), BF16), empty(ctx, (rows, dim), BF16)
        ctx.block_norm(ctx.block_norm_params(rows, dim, post=1, pre=2, eps=EPS), bh, None, br, None, None, None, None, new, out)
        got.append((host(oracle, new, BF16), host(oracle, out, BF16)))
    keep = [0, 2, 4]
    assert np.isnan(got[0][1][[1, 3]]).any()
    for a, b in zip(*got):
        assert np.array_equal(a[keep], b[keep])


@pytest.mark.parametrize("fmt", [P.MX4_E8M0, P.MX4_E4M3])
@pytest.mark.parametrize("rows,dim", [(1, 32), (3, 96), (2, 4096), (9, 288), (130, 2880), (700, 512), (4, 8224), (2, 33024)])
@pytest.mark.parametrize("shift", [0, 1])
def test_microscaled_output(ctx, oracle, fmt, rows, dim, shift):
    """The codes and scales of mx4_quantize on the bf16 output, bit for bit; rows behind the last are left alone."""
    rng = np.random.default_rng(dim)
    bh, _ = place(ctx, oracle, rng.standard_normal((rows, dim)), BF16, shift)
    br, _ = place(ctx, oracle, rng.standard_normal((rows, dim)), F32, shift)
    bw, _ = place(ctx, oracle, rng.standard_normal(dim), F32, shift)
    kw = dict(post=P.NORM_RMS, pre=P.NORM_LAYER, r_dtype=F32, eps=EPS, branch_scale=0.5)
    n = ctx.mx4_scale_bytes(rows, dim, fmt)
    new, out = empty(ctx, (rows, dim), F32), empty(ctx, (rows, dim), BF16)
    codes = [ctx.empty((rows, dim // 8), np.uint32) for _ in range(2)]
    scales = [ctx.upload(np.full(n, 0x5A, np.uint8)) for _ in range(2)]
    ctx.block_norm(ctx.block_norm_params(rows, dim, **kw), bh, None, br, bw, None, bw, bw, new, out)
    ctx.mx4_quantize(out, codes[0], scales[0], rows, dim, fmt, BF16, 3.7)
    first = new.to_host()
    ctx.block_norm(ctx.block_norm_params(rows, dim, out_format=fmt, out_pre=3.7, **kw), bh, None, br, bw, None, bw, bw, new, codes[1], scales[1])
    assert np.array_equal(new.to_host(), first)
    np.testing.assert_array_equal(scales[1].to_host(), scales[0].to_host())
    np.testing.assert_array_equal(codes[1].to_host(), codes[0].to_host())


@pytest.mark.parametrize("fmt", [P.MX4_E8M0, P.MX4_E4M3])
@pytest.mark.parametrize("M", [1, 8, 150])
def test_decode_step(ctx, oracle, fmt, M):
    """Two blocks as they would be run, eagerly and recorded: block_norm into the format, gate|up product, mul_rms_norm, mx4_quantize, down
    product; every call checked on the inputs that it saw."""
    d, f = 512, 768
    rng = np.random.default_rng(M)
    pre, wpre = (1.0, 1.0) if fmt == P.MX4_E8M0 else (64.0, 2000.0)
    alpha = np.float64(np.float32(1 / (pre * wpre)))

    def layer(N, K):
        w = (rng.standard_normal((N, K)) * 0.05).astype(np.float32)
        src, c, s = ctx.upload(w), ctx.empty((N, K // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(N, K, fmt))
        ctx.mx4_quantize(src, c, s, N, K, fmt, F32, wpre)
        return c, s, mx4.values(*mx4.quantize(w, fmt, wpre), fmt)

    blocks = []
    for _ in range(2):
        blocks.append(dict(gu=layer(2 * f, d), down=layer(d, f), w=place(ctx, oracle, 1 + 0.1 * rng.standard_normal(d), F32), gate=place(ctx, oracle, rng.standard_normal((1, d)), BF16),
                           xq=ctx.empty((M, d // 8), np.uint32), xs=ctx.upload(np.full(ctx.mx4_scale_bytes(M, d, fmt), 0xFF, np.uint8)), mq=ctx.empty((M, f // 8), np.uint32),
                           ms=ctx.upload(np.full(ctx.mx4_scale_bytes(M, f, fmt), 0xFF, np.uint8)), g=empty(ctx, (M, 2 * f), BF16), m=empty(ctx, (M, f), BF16), h=empty(ctx, (M, d), BF16),
                           r=empty(ctx, (M, d), BF16)))
    bh, bh_v = place(ctx, oracle, rng.standard_normal((M, d)), BF16)
    br, br_v = place(ctx, oracle, rng.standard_normal((M, d)), BF16)
    prm = ctx.block_norm_params(M, d, post=P.NORM_RMS, pre=P.NORM_RMS, gate_act=P.GATE_SIGMOID, eps=EPS, branch_scale=0.5, out_format=fmt, out_pre=pre)

    def step():
        h, r = bh, br
        for b in blocks:
            ctx.block_norm(prm, h, b["gate"][0], r, b["w"][0], None, b["w"][0], None, b["r"], b["xq"], b["xs"])
            ctx.mx4_matmul(b["xq"], b["xs"], b["gu"][0], b["gu"][1], b["g"], M, d, 2 * f, fmt, BF16, alpha)
            ctx.mul_rms_norm(b["g"], b["m"], M, f, 2 * f, EPS)
            ctx.mx4_quantize(b["m"], b["mq"], b["ms"], M, f, fmt, BF16, pre)
            ctx.mx4_matmul(b["mq"], b["ms"], b["down"][0], b["down"][1], b["h"], M, f, d, fmt, BF16, alpha)
            h, r = b["h"], b["r"]

    def product_ok(y, code, byte, wv):
        v = mx4.values(code, byte, fmt)
        t, mag = alpha * (v @ wv.T), alpha * (np.abs(v) @ np.abs(wv).T)
        tol = mag * v.shape[1] * 2.0 ** -23
        return (np.abs(y - t) <= tol + (np.abs(t) + tol) * 2.0 ** -8).all()

    def snapshot():
        return [{k: host(oracle, b[k], BF16) for k in ("r", "g", "m", "h")} | {k: b[k].to_host() for k in ("xq", "xs", "mq", "ms")} for b in blocks]

    step()
    eager = snapshot()
    h, r = bh_v, br_v
    for b, s in zip(blocks, eager):
        w = b["w"][1]
        t = 0.5 * mx4.norm(h, 1, EPS, w) * mx4.gate(b["gate"][1], 1) + r
        assert (np.abs(s["r"] - t) <= np.abs(t) * 2.0 ** -8 + 2.0 ** -16 * (1 + np.abs(t))).all()
        n = mx4.norm(s["r"], 1, EPS, w)
        code, byte = mx4.unpack(s["xq"]), mx4.from_tiles(s["xs"], M, d // mx4.BLOCK[fmt])
        v = mx4.values(code, byte, fmt) / pre
        # a code is at most half a step of the grid away (a quarter of the value, half a unit of the scale near zero, a quarter where the largest is cut off)
        assert (np.abs(v - n) <= 0.25 * np.abs(n) + 0.26 * np.repeat(mx4.scale_values(byte, fmt), mx4.BLOCK[fmt], 1) / pre + 0.01).all()
        assert product_ok(s["g"], code, byte, b["gu"][2])
        m = oracle.from_bf16(oracle.to_bf16((s["g"][:, :f] * s["g"][:, f:]).astype(np.float32))).astype(np.float64)
        m = mx4.norm(m, 1, EPS)
        assert (np.abs(s["m"] - m) <= np.abs(m) * (2.0 ** -8 + 2.0 ** -16)).all()
        want = mx4.quantize(s["m"].astype(np.float32), fmt, pre)
        code, byte = mx4.unpack(s["mq"]), mx4.from_tiles(s["ms"], M, f // mx4.BLOCK[fmt])
        np.testing.assert_array_equal(byte, want[1])
        np.testing.assert_array_equal(mx4.VALUES[code], mx4.VALUES[want[0]])
        assert product_ok(s["h"], code, byte, b["down"][2])
        h, r = s["h"], s["r"]
    for _ in range(5):  # without a wait between the steps
        step()
    again = snapshot()
    ctx.graph_begin()
    step()
    g = ctx.graph_end()
    for _ in range(5):
        ctx.graph_launch(g)
    replayed = snapshot()
    ctx.graph_destroy(g)
    for a, b, c in zip(eager, again, replayed):
        for k in a:
            assert np.array_equal(a[k], b[k]) and np.array_equal(a[k], c[k]), k


def test_refusals(ctx, plugin):
    rows, dim = 4, 64
    h, r, out, new = (ctx.empty((rows, dim), np.uint16) for _ in range(4))
    w = ctx.empty((dim,), np.float32)
    codes, scales = ctx.empty((rows, dim // 8), np.uint32), ctx.alloc(ctx.mx4_scale_bytes(rows, dim, 1))
    ok = dict(post=1, pre=1)

    def call(prm=None, rows=rows, dim=dim, h=h, gate=None, r=r, pw=None, pb=None, qw=None, qb=None, new=new, out=out, scales=None, **kw):
        ctx.block_norm(ctx.block_norm_params(rows, dim, **{**ok, **kw}), h, gate, r, pw, pb, qw, qb, new, out, scales)

    call()
    call(rows=0)
    call(new=r)
    small = ctx.wrap(h.device_ptr, h.nbytes - 2)
    odd = ctx.wrap(codes.device_ptr + 4, codes.nbytes - 4)
    byte = ctx.wrap(h.device_ptr + 1, h.nbytes - 1)
    bad = [dict(dim=0), dict(rows=5), dict(h=None, r=None, post=0), dict(new=None, out=None), dict(h=None), dict(h=None, post=0, gate=h), dict(post=3), dict(pre=-1), dict(gate_act=3),
           dict(x_dtype=P.F16), dict(r_dtype=P.I32), dict(out_dtype=P.U32), dict(pb=w), dict(qb=w), dict(pre=0, qw=w), dict(post=0, pw=w), dict(h_ld=63), dict(gate=h, gate_ld=32),
           dict(h=small), dict(h=byte, rows=3), dict(out_format=1, out=codes), dict(out_format=3, out=codes, scales=scales), dict(out_format=1, out=odd, scales=scales, rows=1, dim=32),
           dict(out_format=1, out=codes, scales=scales, dim=48), dict(scales=scales), dict(out=h), dict(new=h), dict(out=new), dict(r_dtype=F32), dict(gate=h, gate_rows=1, gate_ld=128),
           dict(rows=1, dim=1 << 20, h=None, post=0, new=None), dict(rows=1 << 40)]
    for kw in bad:
        with pytest.raises(BackendError) as e:
            call(**kw)
        assert e.value.code == P.ERR_INVALID, kw
    assert plugin.last_error()
    assert plugin.quant.block_norm(None, None, *[None] * 10) == P.ERR_INVALID


@pytest.mark.parametrize("post,pre", [(0, 1), (1, 1), (2, 2), (1, 0)])
@pytest.mark.parametrize("rows,dim,gate_rows", [(1200, 2048, None), (1300, 2880, 0), (1184, 4096, 1), (1500, 2056, 7), (600, 4096, 0), (650, 1536, 1), (1800, 2048, None)])
def test_many_rows(ctx, oracle, rows, dim, gate_rows, post, pre):
    """Rows that one block per SM takes in turn: with and without a gate, shared by all, by some or of each row's own; every type."""
    for xd, rd, od, act in ((BF16, BF16, BF16, P.GATE_TANH), (BF16, F32, F32, P.GATE_SIGMOID), (F32, BF16, F32, P.GATE_IDENTITY), (F32, F32, BF16, P.GATE_SIGMOID)):
        run(ctx, oracle, rows, dim, post, pre, gate_rows, act if gate_rows is not None else 0, xd, rd, od, seed=post)


@pytest.mark.parametrize("fmt", [P.MX4_E8M0, P.MX4_E4M3])
@pytest.mark.parametrize("rows,dim", [(1300, 2048), (1200, 2912)])
def test_many_rows_microscaled_in_place_and_column_blocks(ctx, oracle, fmt, rows, dim):
    rng = np.random.default_rng(dim)
    bh, _ = place(ctx, oracle, rng.standard_normal((rows, dim + 64)), BF16)
    stream = rng.standard_normal((rows, dim)).astype(np.float32)
    bw, _ = place(ctx, oracle, rng.standard_normal(dim), F32)
    kw = dict(post=P.NORM_LAYER, pre=P.NORM_RMS, r_dtype=F32, eps=EPS, branch_scale=0.5, h_ld=dim + 64)
    n = ctx.mx4_scale_bytes(rows, dim, fmt)
    out, new = empty(ctx, (rows, dim), BF16), ctx.upload(stream)
    codes = [ctx.empty((rows, dim // 8), np.uint32) for _ in range(2)]
    scales = [ctx.upload(np.full(n, 0x5A, np.uint8)) for _ in range(2)]
    ctx.block_norm(ctx.block_norm_params(rows, dim, **kw), bh, None, new, bw, bw, bw, None, new, out)
    ctx.mx4_quantize(out, codes[0], scales[0], rows, dim, fmt, BF16, 3.7)
    first = new.to_host()
    new.from_host(stream)
    for _ in range(3):  # the stream in place: every call adds the branch again; the last of three replays after a reset is compared
        new.from_host(stream)
        ctx.block_norm(ctx.block_norm_params(rows, dim, out_format=fmt, out_pre=3.7, **kw), bh, None, new, bw, bw, bw, None, new, codes[1], scales[1])
    assert np.array_equal(new.to_host(), first)
    np.testing.assert_array_equal(scales[1].to_host(), scales[0].to_host())
    np.testing.assert_array_equal(codes[1].to_host(), codes[0].to_host())
    # without a block's output: the norm of the stream alone
    ctx.block_norm(ctx.block_norm_params(rows, dim, pre=P.NORM_RMS, r_dtype=F32, eps=EPS), None, None, new, None, None, bw, None, None, out)
    want = mx4.norm(first, 1, EPS, bw.room.to_host())
    tol = norm_tolerance(first.astype(np.float64), 1, bw.room.to_host(), None, want)
    assert (np.abs(host(oracle, out, BF16) - want) <= tol + rounding(np.abs(want) + tol, BF16)).all()


@pytest.mark.parametrize("rows,dim", [(5, 96), (3, 40008), (1200, 2048)])
@pytest.mark.parametrize("gate_rows", [1 << 31, 1 << 32, (1 << 64) - 1])
def test_a_gate_shared_by_more_rows_than_there_are(ctx, rows, dim, gate_rows):
    """One row of gate serves them all, as with 0; a gate with less than a row is refused however many share it."""
    rng = np.random.default_rng(rows)
    bits = lambda shape: ctx.upload((rng.standard_normal(shape).astype(np.float32).view(np.uint32) >> 16).astype(np.uint16))  # noqa: E731
    h, r, g = bits((rows, dim)), bits((rows, dim)), bits((dim,))
    got = []
    for n in (0, gate_rows):
        new, out = empty(ctx, (rows, dim), BF16), empty(ctx, (rows, dim), BF16)
        ctx.block_norm(ctx.block_norm_params(rows, dim, post=P.NORM_RMS, pre=P.NORM_RMS, gate_act=P.GATE_SIGMOID, gate_rows=n, eps=EPS), h, g, r, None, None, None, None, new, out)
        got.append((new.to_host(), out.to_host()))
    np.testing.assert_array_equal(got[1][0], got[0][0])
    np.testing.assert_array_equal(got[1][1], got[0][1])
    for less in (dim - 1, 1):
        with pytest.raises(BackendError) as e:
            ctx.block_norm(ctx.block_norm_params(rows, dim, post=P.NORM_RMS, pre=P.NORM_RMS, gate_rows=gate_rows, eps=EPS), h, ctx.wrap(g.device_ptr, less * 2), r, None, None, None, None,
                           new, out)
        assert e.value.code == P.ERR_INVALID


@pytest.mark.parametrize("post,pre", list(itertools.product(KINDS, KINDS)))
@pytest.mark.parametrize("rows,dim", [(5, 64), (1201, 8), (1185, 64), (1299, 128), (1500, 200), (1187, 256), (2000, 136)])
def test_short_rows(ctx, oracle, rows, dim, post, pre):
    """Two rows to a warp, the last of them alone."""
    run(ctx, oracle, rows, dim, post, pre, 3, P.GATE_TANH, BF16, F32, BF16, seed=rows)
    run(ctx, oracle, rows, dim, post, pre, None, 0, F32, BF16, F32, seed=rows, in_place=True)


@pytest.mark.parametrize("fmt", [P.MX4_E8M0, P.MX4_E4M3])
@pytest.mark.parametrize("rows,dim", [(3, 128), (1201, 64), (1185, 128), (1311, 160), (1400, 256)])
def test_short_rows_microscaled(ctx, oracle, fmt, rows, dim):
    """As a bf16 output and its quantisation, bit for bit; nothing is written for a row that is not there."""
    rng = np.random.default_rng(dim)
    bh, _ = place(ctx, oracle, rng.standard_normal((rows, dim)), BF16)
    out, n = empty(ctx, (rows, dim), BF16), ctx.mx4_scale_bytes(rows, dim, fmt)
    codes = [ctx.upload(np.full((rows + 1, dim // 8), 0x5A5A5A5A, np.uint32)) for _ in range(2)]
    scales = [ctx.upload(np.full(n, 0x5A, np.uint8)) for _ in range(2)]
    kw = dict(pre=P.NORM_LAYER, eps=EPS, post=P.NORM_RMS)
    ctx.block_norm(ctx.block_norm_params(rows, dim, **kw), bh, None, None, None, None, None, None, None, out)
    ctx.mx4_quantize(out, codes[0], scales[0], rows, dim, fmt, BF16)
    ctx.block_norm(ctx.block_norm_params(rows, dim, out_format=fmt, **kw), bh, None, None, None, None, None, None, None, codes[1], scales[1])
    np.testing.assert_array_equal(scales[1].to_host(), scales[0].to_host())
    np.testing.assert_array_equal(codes[1].to_host(), codes[0].to_host())

"""Products grouped by expert against 64 bits: every form of the kernels, groups of any size, what is not to be written."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32, BackendError
from mlx_b200 import plugin as P
from oracle import moe

pytestmark = pytest.mark.gpu
GUARD = 64  # elements ahead of y and behind it


def layer(oracle, E, N, K, bits, group, seed=0):
    """Packed weights of E experts and their values."""
    wq, s, b = oracle.make_layer(E * N, K, bits, group, oracle.BF16, config_id=31, layer=K, proj=N + seed)
    return (wq, s, b), oracle.from_bf16(oracle.dequantize(wq, s, b, K, bits, group, oracle.BF16)).reshape(E, N, K)


def groups(rng, E, rows, kind):
    """Offsets of E experts over `rows` rows."""
    if kind == "even":
        cuts = np.linspace(0, rows, E + 1).astype(int)
    elif kind == "one":           # all to one expert, not the first or last where there are others
        cuts = np.where(np.arange(E + 1) > E // 2, rows, 0)
    elif kind == "tail":          # rows that belong to nobody
        cuts = np.linspace(0, max(rows - 5, 0), E + 1).astype(int)
    elif kind == "none":
        cuts = np.zeros(E + 1, int)
    else:                         # ragged, some empty
        cuts = np.concatenate([[0], np.sort(rng.integers(0, rows + 1, E - 1)), [rows]])
    return cuts.astype(np.int32)


def run(ctx, oracle, w, values, x, offsets, E, K, N, bits, group, order=None, top_k=1, act=0, gated=False, bias=None, y_dtype=BF16, rows=None):
    """One call, checked; returns the raw rows of y."""
    xv = oracle.from_bf16(x)
    rows = (len(x) if order is None else len(order)) if rows is None else rows
    n_out = N // 2 if gated else N
    kind, size = (np.uint16, 2) if y_dtype == BF16 else (np.float32, 4)
    mark = kind(0x7E7E) if y_dtype == BF16 else kind(-12345.5)
    room = ctx.upload(np.full(rows * n_out + 2 * GUARD, mark, kind))
    y = ctx.wrap(room.device_ptr + GUARD * size, max(rows * n_out * size, 1))
    prm = ctx.experts_params(rows, len(x), E, K, N, bits, group, top_k=top_k, act=act, gated=gated, y_dtype=y_dtype)
    ctx.qmatmul_experts(prm, ctx.upload(x), None if order is None else ctx.upload(order), ctx.upload(offsets), *(ctx.upload(a) for a in w),
                        None if bias is None else ctx.upload(bias), y)
    raw = room.to_host()
    ctx.sync()
    assert (raw[:GUARD] == mark).all() and (raw[GUARD + rows * n_out:] == mark).all()
    raw = raw[GUARD:GUARD + rows * n_out].reshape(rows, n_out)
    got = oracle.from_bf16(raw).astype(np.float64) if y_dtype == BF16 else raw.astype(np.float64)
    mine = np.zeros(rows, bool)
    for e in range(E):
        lo, hi = offsets[e], offsets[e + 1]
        if lo >= hi:
            continue
        mine[lo:hi] = True
        src = np.arange(lo, hi) if order is None else np.where(order[lo:hi] >= 0, order[lo:hi] // top_k, -1)
        there = (src >= 0) & (src < len(x))
        xe = np.where(there[:, None], xv[np.where(there, src, 0)], 0)
        want, tol = moe.epilogue(*moe.product(xe, values[e], None if bias is None else bias[e]), K, act, gated)
        if y_dtype == BF16:
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol) + 2.0 ** -134
        bad = ~(np.abs(got[lo:hi] - want) <= tol)
        assert not bad.any(), (e, np.argwhere(bad)[:4], got[lo:hi][bad][:4], want[bad][:4], tol[bad][:4])
    assert (raw[~mine] == mark).all()
    return raw


# experts, rows, kind of groups, top_k: a token; a few rows an expert; more than 8 and 16; many
SIZES = [(8, 4, "one", 4), (16, 40, "ragged", 4), (5, 64, "even", 2), (3, 100, "tail", 2), (4, 900, "ragged", 3), (2, 530, "one", 1)]


@pytest.mark.parametrize("bits,group", [(4, 32), (4, 64), (4, 128), (8, 32), (8, 64), (8, 128)])
@pytest.mark.parametrize("E,rows,kind,top_k", SIZES)
@pytest.mark.parametrize("gated", [False, True])
def test_experts(ctx, oracle, bits, group, E, rows, kind, top_k, gated):
    rng = np.random.default_rng(rows * 10 + group + bits)
    K, N = 384, 176 if gated else 163
    w, values = layer(oracle, E, N, K, bits, group)
    offsets = groups(rng, E, rows, kind)
    tokens = (rows + top_k - 1) // top_k
    order = rng.permutation(tokens * top_k)[:rows].astype(np.int32)
    bias = (rng.standard_normal((E, N))).astype(np.float32)
    x = oracle.make_x(tokens, K, oracle.BF16, tag=rows)
    run(ctx, oracle, w, values, x, offsets, E, K, N, bits, group, order=order, top_k=top_k, act=P.ACT_SILU if gated else P.ACT_NONE, gated=gated, bias=bias)
    run(ctx, oracle, w, values, oracle.make_x(rows, K, oracle.BF16, tag=1), offsets, E, K, N, bits, group, gated=gated, y_dtype=F32)


# K: inside a k-block, off 64, several chunks of 16 k-blocks, odd groups a row; N: below a tile, one more than a tile, several
@pytest.mark.parametrize("bits,group,K", [(4, 32, 32), (4, 32, 96), (4, 32, 2912), (8, 32, 32), (8, 32, 1440), (4, 128, 4352), (8, 64, 4160), (4, 64, 1408), (8, 128, 128)])
@pytest.mark.parametrize("N", [1, 15, 17, 129])
@pytest.mark.parametrize("rows", [9, 200])
def test_odd_sizes(ctx, oracle, bits, group, K, N, rows):
    rng = np.random.default_rng(K + N)
    E = 3
    w, values = layer(oracle, E, N, K, bits, group)
    offsets = groups(rng, E, rows, "ragged")
    x = oracle.make_x(rows, K, oracle.BF16, tag=N)
    run(ctx, oracle, w, values, x, offsets, E, K, N, bits, group, act=P.ACT_RELU, y_dtype=F32)


@pytest.mark.parametrize("bits,group,K", [(4, 32, 96), (4, 64, 4160), (8, 32, 2912), (8, 128, 1408)])
@pytest.mark.parametrize("N", [16, 48, 272])
@pytest.mark.parametrize("rows", [3, 70, 600])
def test_odd_gated_sizes(ctx, oracle, bits, group, K, N, rows):
    rng = np.random.default_rng(K + N)
    E = 3
    w, values = layer(oracle, E, N, K, bits, group)
    x = oracle.make_x(rows, K, oracle.BF16, tag=N)
    run(ctx, oracle, w, values, x, groups(rng, E, rows, "ragged"), E, K, N, bits, group, act=P.ACT_GELU, gated=True)


# one sub-block of k, an odd number of them, odd groups a row; single CTAs and pairs; tiles of W short of 128 rows, of two tiles, and an odd number of tiles
@pytest.mark.parametrize("bits,group,K", [(4, 64, 64), (8, 32, 192), (4, 32, 320), (4, 128, 1408), (8, 128, 640)])
@pytest.mark.parametrize("N,gated", [(120, False), (131, False), (400, False), (16, True), (272, True)])
@pytest.mark.parametrize("rows", [250, 1500])
@pytest.mark.parametrize("pair", ["0", "1"])
def test_many_rows(ctx, oracle, monkeypatch, bits, group, K, N, gated, rows, pair):
    monkeypatch.setenv("LUXCUDA_EXPERTS", "many")
    monkeypatch.setenv("LUXCUDA_EXPERTS_PAIR", pair)
    rng = np.random.default_rng(K + N + rows)
    E = 4
    w, values = layer(oracle, E, N, K, bits, group)
    x = oracle.make_x(rows, K, oracle.BF16, tag=N)
    offsets = groups(rng, E, rows, "ragged")
    order = rng.permutation(rows).astype(np.int32)
    run(ctx, oracle, w, values, x, offsets, E, K, N, bits, group, order=order, act=P.ACT_GELU_TANH, gated=gated)
    assert ctx.last_kernel() == f"qmm_experts<{bits}{',pairs' if pair == '1' else ''}>"
    run(ctx, oracle, w, values, x, groups(rng, E, rows, "tail"), E, K, N, bits, group, gated=gated, y_dtype=F32)


@pytest.mark.parametrize("rows", [11, 250, 1000])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("gated", [False, True])
def test_y_on_no_wide_boundary(ctx, oracle, rows, y_dtype, gated):
    """One element past a 16-byte boundary: the same bits."""
    E, K, N = 3, 256, 160
    w, values = layer(oracle, E, N, K, 4, 64)
    x = oracle.make_x(rows, K, oracle.BF16)
    offsets = groups(None, E, rows, "even")
    want = run(ctx, oracle, w, values, x, offsets, E, K, N, 4, 64, gated=gated, y_dtype=y_dtype)
    kind, size = (np.uint16, 2) if y_dtype == BF16 else (np.float32, 4)
    room = ctx.upload(np.zeros(want.size + 2, kind))
    ctx.qmatmul_experts(ctx.experts_params(rows, rows, E, K, N, 4, 64, gated=gated, y_dtype=y_dtype), ctx.upload(x), None, ctx.upload(offsets), *(ctx.upload(a) for a in w), None,
                        ctx.wrap(room.device_ptr + size, want.nbytes))
    got = room.to_host()
    np.testing.assert_array_equal(got[1:-1].reshape(want.shape), want)
    assert got[0] == 0 and got[-1] == 0


@pytest.mark.parametrize("act", [P.ACT_NONE, P.ACT_RELU, P.ACT_SILU, P.ACT_GELU, P.ACT_GELU_TANH])
@pytest.mark.parametrize("y_dtype", [BF16, F32])
@pytest.mark.parametrize("rows", [20, 400])
def test_activations(ctx, oracle, act, y_dtype, rows):
    E, K, N = 4, 256, 160
    rng = np.random.default_rng(act)
    w, values = layer(oracle, E, N, K, 4, 64)
    x = oracle.make_x(rows, K, oracle.BF16, tag=act)
    bias = (rng.standard_normal((E, N)) * 3).astype(np.float32)
    for gated in (False, True):
        run(ctx, oracle, w, values, x, groups(rng, E, rows, "ragged"), E, K, N, 4, 64, act=act, gated=gated, bias=bias, y_dtype=y_dtype)


def test_many_experts_and_empty_ones(ctx, oracle):
    E, K, N, rows = 1024, 64, 24, 90
    rng = np.random.default_rng(2)
    w, values = layer(oracle, E, N, K, 8, 64)
    x = oracle.make_x(rows, K, oracle.BF16)
    for kind in ("ragged", "none", "one", "tail"):
        run(ctx, oracle, w, values, x, groups(rng, E, rows, kind), E, K, N, 8, 64)


@pytest.mark.parametrize("rows", [12, 300])
def test_a_row_depends_on_itself_and_its_expert(ctx, oracle, rows):
    """The same bits whatever the other rows, their number and the order."""
    E, K, N = 4, 512, 96
    w, values = layer(oracle, E, N, K, 4, 64)
    x = oracle.make_x(rows, K, oracle.BF16)
    offsets = np.linspace(0, rows, E + 1).astype(np.int32)
    args = (E, K, N, 4, 64)
    whole = run(ctx, oracle, w, values, x, offsets, *args)
    again = run(ctx, oracle, w, values, x, offsets, *args)
    np.testing.assert_array_equal(whole, again)
    back = np.arange(rows)[::-1].astype(np.int32)
    gathered = run(ctx, oracle, w, values, np.ascontiguousarray(x[::-1]), offsets, *args, order=back)
    np.testing.assert_array_equal(whole, gathered)


@pytest.mark.parametrize("rows", [10, 300])
def test_offsets_and_order_that_are_wrong(ctx, oracle, rows):
    """Offsets are cut to the rows there are, an expert whose offsets fall has none; rows of x that do not exist are zero."""
    E, K, N, k = 4, 128, 64, 2
    w, values = layer(oracle, E, N, K, 4, 32)
    tokens = rows // k
    x = oracle.make_x(tokens, K, oracle.BF16)
    order = np.arange(rows, dtype=np.int32)
    order[1], order[2], order[5] = -3, 2 ** 31 - 1, rows + 1
    offsets = np.array([-7, 3, 2, 2, rows + 100], np.int32)
    seen = np.array([0, 3, 2, 2, rows], np.int32)
    bias = np.ones((E, N), np.float32)
    # what the kernels see is `seen`; the checked run is made with it, the wrong one has to give the same rows
    want = run(ctx, oracle, w, values, x, seen, E, K, N, 4, 32, order=order, top_k=k, bias=bias)
    y = ctx.upload(np.full((rows, N), 0x7E7E, np.uint16))
    prm = ctx.experts_params(rows, tokens, E, K, N, 4, 32, top_k=k)
    ctx.qmatmul_experts(prm, ctx.upload(x), ctx.upload(order), ctx.upload(offsets), *(ctx.upload(a) for a in w), ctx.upload(bias), y)
    got = y.to_host()
    np.testing.assert_array_equal(got[3:], want[3:])  # (rows 2 of expert 0 and of expert 3 are written by both)
    np.testing.assert_array_equal(got[:2], want[:2])
    ctx.sync()


def test_infinite_and_missing_weights_of_other_experts(ctx, oracle):
    """NaN in the scales and x rows of one expert stays there."""
    E, K, N = 3, 256, 40
    for rows in (9, 240):
        w, values = layer(oracle, E, N, K, 4, 64)
        x = oracle.make_x(rows, K, oracle.BF16)
        offsets = np.linspace(0, rows, E + 1).astype(np.int32)
        want = run(ctx, oracle, w, values, x, offsets, E, K, N, 4, 64)
        s = w[1].copy()
        s[N:2 * N] = 0x7FC0
        x2 = x.copy()
        x2[offsets[1]:offsets[2]] = 0x7F80
        y = ctx.upload(np.zeros((rows, N), np.uint16))
        ctx.qmatmul_experts(ctx.experts_params(rows, rows, E, K, N, 4, 64), ctx.upload(x2), None, ctx.upload(offsets), ctx.upload(w[0]), ctx.upload(s), ctx.upload(w[2]), None, y)
        got = y.to_host()
        for e in (0, 2):
            np.testing.assert_array_equal(got[offsets[e]:offsets[e + 1]], want[offsets[e]:offsets[e + 1]])
        assert np.isnan(oracle.from_bf16(got[offsets[1]:offsets[2]])).all()


@pytest.mark.parametrize("bits,group", [(4, 32), (4, 64), (4, 128), (8, 32), (8, 64), (8, 128)])
@pytest.mark.parametrize("which,pair", [("few", "0"), ("many", "0"), ("many", "1")])
def test_scales_of_any_size(ctx, oracle, monkeypatch, bits, group, which, pair):
    """Zero, negative, the smallest normal one, on both sides of 2^-5 and large: where the kernels' short dequantisation ends, alone in a row and mixed."""
    monkeypatch.setenv("LUXCUDA_EXPERTS", which)
    monkeypatch.setenv("LUXCUDA_EXPERTS_PAIR", pair)
    E, K, N, rows = 2, 640, 200, 90
    (wq, s, b), _ = layer(oracle, E, N, K, bits, group)
    rng = np.random.default_rng(group + bits)
    sizes = oracle.to_bf16(np.array([0.0, 2.0 ** -126, 1e-3, -1e-3, 0.0311, 0.03125, -0.03125, 0.7, 9.0], np.float32))
    s = s.reshape(E * N, -1).copy()
    for n in range(E * N):
        if n % 40 < 9:
            s[n] = sizes[n % 40]
        elif n % 40 < 20 or n % 80 == 47:
            s[n] = rng.choice(sizes, s.shape[1])
    values = oracle.from_bf16(oracle.dequantize(wq, s, b, K, bits, group, oracle.BF16)).reshape(E, N, K)
    run(ctx, oracle, (wq, s, b), values, oracle.make_x(rows, K, oracle.BF16), groups(None, E, rows, "even"), E, K, N, bits, group, y_dtype=F32)


@pytest.mark.parametrize("bits,group,K", [(4, 32, 32), (4, 32, 96), (4, 64, 320), (4, 128, 4224), (8, 32, 160), (8, 64, 192)])
@pytest.mark.parametrize("N,gated", [(19, False), (48, False), (32, True)])
@pytest.mark.parametrize("rows", [7, 300])
def test_an_infinite_scale_stays_in_its_row(ctx, oracle, bits, group, K, N, gated, rows):
    """K ends inside a block of the kernels': what lies behind it there is the next row's."""
    E = 2
    w, _ = layer(oracle, E, N, K, bits, group)
    x, offsets = oracle.make_x(rows, K, oracle.BF16), groups(None, E, rows, "even")
    prm = ctx.experts_params(rows, rows, E, K, N, bits, group, gated=gated, y_dtype=F32)
    xb, off, y = ctx.upload(x), ctx.upload(offsets), ctx.empty((rows, N // 2 if gated else N), np.float32)

    def call(scales, biases):
        ctx.qmatmul_experts(prm, xb, None, off, ctx.upload(w[0]), ctx.upload(scales), ctx.upload(biases), None, y)
        return y.to_host()

    want = call(w[1], w[2])
    for n in (0, 5, N - 1):
        s, b = w[1].reshape(E * N, -1).copy(), w[2].reshape(E * N, -1).copy()
        s[n], b[n] = 0x7F80, 0xFF80  # infinity, minus infinity: of expert 0
        got = call(s, b)
        cols = [c for c in range(want.shape[1]) if c != n and not (gated and c + N // 2 == n)]
        np.testing.assert_array_equal(got[:, cols], want[:, cols])
        np.testing.assert_array_equal(got[offsets[1]:], want[offsets[1]:])
        assert not np.isfinite(got[:offsets[1], n % want.shape[1]]).any()


@pytest.mark.parametrize("rows", [16, 500])
def test_recorded(ctx, oracle, rows):
    """Recorded once, replayed with other offsets in the same buffer."""
    E, K, N = 4, 256, 128
    w, values = layer(oracle, E, N, K, 4, 64)
    x = oracle.make_x(rows, K, oracle.BF16)
    bufs = [ctx.upload(a) for a in w]
    xb, off, y = ctx.upload(x), ctx.upload(groups(None, E, rows, "even")), ctx.empty((rows, N), np.uint16)
    prm = ctx.experts_params(rows, rows, E, K, N, 4, 64)
    ctx.qmatmul_experts(prm, xb, None, off, *bufs, None, y)
    ctx.sync()
    ctx.graph_begin()
    ctx.qmatmul_experts(prm, xb, None, off, *bufs, None, y)
    ctx.qmatmul_experts(prm, xb, None, off, *bufs, None, y)
    g = ctx.graph_end()
    rng = np.random.default_rng(1)
    for kind in ("ragged", "one", "even"):
        cuts = groups(rng, E, rows, kind)
        want = run(ctx, oracle, w, values, x, cuts, E, K, N, 4, 64)
        off.from_host(cuts)
        y.from_host(np.zeros((rows, N), np.uint16))
        ctx.graph_launch(g)
        np.testing.assert_array_equal(y.to_host(), want)
    ctx.graph_destroy(g)


def test_workspace_of_a_gathered_product(ctx, oracle):
    """It grows between calls and not while a graph is recorded; a graph recorded with the outgrown one still gives its bits."""
    E, K, N = 2, 128, 64
    w, values = layer(oracle, E, N, K, 4, 64)
    bufs = [ctx.upload(a) for a in w]

    def call(rows):
        x = oracle.make_x(rows, K, oracle.BF16, tag=rows)
        order = np.random.default_rng(rows).permutation(rows).astype(np.int32)
        y = ctx.empty((rows, N), np.uint16)
        keep = (ctx.upload(x), ctx.upload(order), ctx.upload(groups(None, E, rows, "even")))
        return lambda: ctx.qmatmul_experts(ctx.experts_params(rows, rows, E, K, N, 4, 64), keep[0], keep[1], keep[2], *bufs, None, y), y
    small, y_small = call(200)
    big, y_big = call(3000)
    small()
    want = y_small.to_host()
    ctx.graph_begin()
    small()
    with pytest.raises(BackendError) as e:
        big()
    assert e.value.code == P.ERR_NOT_SUPPORTED
    g = ctx.graph_end()
    big()
    want_big = y_big.to_host()
    y_small.from_host(np.zeros_like(want))
    ctx.graph_launch(g)
    big()
    np.testing.assert_array_equal(y_small.to_host(), want)
    np.testing.assert_array_equal(y_big.to_host(), want_big)
    ctx.graph_destroy(g)


def test_refusals(ctx, oracle):
    E, K, N, rows = 2, 64, 32, 6
    w, _ = layer(oracle, E, N, K, 4, 32)
    bufs = dict(zip(("wq", "scales", "biases"), (ctx.upload(a) for a in w)))
    x, y = ctx.upload(oracle.make_x(rows, K, oracle.BF16)), ctx.empty((rows, N), np.uint16)
    off, order = ctx.upload(np.array([0, 3, 6], np.int32)), ctx.upload(np.arange(rows, dtype=np.int32))
    E_ = ctx.experts_params

    def refused(prm=None, **other):
        a = dict(x=x, order=None, offsets=off, **bufs, bias=None, y=y)
        a.update(other)
        with pytest.raises(BackendError) as e:
            ctx.qmatmul_experts(prm or E_(rows, rows, E, K, N, 4, 32), *a.values())
        assert e.value.code == P.ERR_INVALID, str(e.value)
    for prm in (E_(rows, rows, 0, K, N, 4, 32), E_(rows, rows, 1025, K, N, 4, 32), E_(rows, rows, E, K, N, 3, 32), E_(rows, rows, E, K, N, 4, 48), E_(rows, rows, E, 48, N, 4, 32),
                E_(rows, rows, E, K, -1, 4, 32), E_(rows, rows, E, K, N, 4, 32, act=5), E_(rows, rows, E, K, N, 4, 32, y_dtype=P.F16), E_(rows, rows, E, K, 24, 4, 32, gated=True),
                E_(rows + 1, rows, E, K, N, 4, 32), E_(rows, rows + 1, E, K, N, 4, 32), E_(rows, rows, 3, K, N, 4, 32), E_(rows, rows, E, K, N, 8, 32),
                E_(2 ** 31, rows, E, K, N, 4, 32), E_(rows, 2 ** 31, E, K, N, 4, 32), E_(rows, rows, 1024, K, 2 ** 21, 4, 32)):
        refused(prm)
    refused(E_(rows, rows, E, K, N, 4, 32, top_k=0), order=order)
    refused(E_(rows, rows, E, K, N, 4, 32, top_k=33), order=order)
    refused(bias=ctx.upload(np.zeros(E * N - 1, np.float32)))
    refused(offsets=ctx.upload(np.zeros(E, np.int32)))
    refused(y=x)
    refused(x=ctx.wrap(x.device_ptr + 2, rows * K * 2 - 2), prm=E_(rows, rows - 1, E, K, N, 4, 32))
    refused(y=ctx.wrap(y.device_ptr + 1, rows * N * 2 - 1), prm=E_(rows - 1, rows, E, K, N, 4, 32))
    ctx.qmatmul_experts(E_(0, rows, E, K, N, 4, 32), x, None, off, *bufs.values(), None, y)  # nothing to do
    ctx.sync()

"""The router: its choice and the sort exactly, its weights against 64 bits."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32, BackendError
from mlx_b200 import plugin as P
from oracle import moe

pytestmark = pytest.mark.gpu
MARK = -77


def run(ctx, prm, logits, bias, T, k, E, ids=None):
    new = lambda n: ctx.upload(np.full(max(n, 1), MARK, np.int32))  # noqa: E731
    b = {"ids": new(T * k) if ids is None else ctx.upload(ids.astype(np.int32)), "weights": ctx.upload(np.full(max(T * k, 1), -9, np.float32)), "order": new(T * k),
         "pos": new(T * k), "offsets": new(E + 1)}
    ctx.moe_route(prm, logits, bias, b["ids"], b["weights"], b["order"], b["pos"], b["offsets"])
    return {n: v.to_host()[:E + 1 if n == "offsets" else T * k] for n, v in b.items()}


def check_sort(got, ids, E):
    order, pos, offsets = moe.sort(ids, E)
    np.testing.assert_array_equal(got["offsets"], offsets)
    np.testing.assert_array_equal(got["pos"], pos)
    np.testing.assert_array_equal(got["order"][:len(order)], order)
    assert (got["order"][len(order):] == MARK).all()  # behind the last pair: as it was


def check(got, want, T, k, E):
    ids, w = want
    np.testing.assert_array_equal(got["ids"].reshape(T, k), ids)
    # fp32: exponentials 2 units in the last place (4 U) and the rounding of their argument (|v| < 32: 32 U), a sum of E terms in 5 steps of a
    # tree behind E / 32 of a lane, a quotient, a product
    np.testing.assert_allclose(got["weights"].reshape(T, k), w, rtol=(2 * (4 + 32) + E / 32 + 5 + 3) * moe.U, atol=2.0 ** -126)
    check_sort(got, ids, E)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("score,renorm,with_bias", [(P.SCORE_SOFTMAX, True, False), (P.SCORE_SOFTMAX, False, False), (P.SCORE_SIGMOID, True, True), (P.SCORE_SIGMOID, False, False)])
@pytest.mark.parametrize("T,E,k", [(1, 1, 1), (1, 64, 8), (3, 5, 5), (16, 33, 4), (64, 32, 32), (32, 64, 8), (65, 100, 7), (777, 40, 3), (300, 513, 6), (40, 1024, 32), (5000, 256, 8)])
def test_route(ctx, oracle, dtype, score, renorm, with_bias, T, E, k):
    rng = np.random.default_rng(T * E + k)
    v = (rng.standard_normal((T, E)) * 2).astype(np.float32)
    v[rng.random(T) < 0.15] = -np.inf               # tokens of padding
    v[rng.random((T, E)) < 0.05] = -np.inf          # masked experts
    raw = oracle.to_bf16(v) if dtype == BF16 else v  # (bf16: ties by the hundred)
    if dtype == BF16:
        v = oracle.from_bf16(raw)
    bias = (rng.standard_normal(E) * 0.1).astype(np.float32) if with_bias else None
    prm = ctx.moe_route_params(T, E, k, score=score, renorm=renorm, logits_dtype=dtype, scale=1.5)
    got = run(ctx, prm, ctx.upload(raw), ctx.upload(bias) if with_bias else None, T, k, E)
    check(got, moe.route(v, k, score == P.SCORE_SOFTMAX, renorm, 1.5, bias), T, k, E)


@pytest.mark.parametrize("T", [1, 4, 70])
def test_extremes(ctx, T):
    """Infinities, NaN, both zeros, the type's lowest value, sums that vanish."""
    inf, lowest = np.inf, np.finfo(np.float32).min
    rows = np.array([[0.0, -0.0, 0.0, -0.0], [np.nan, 1, inf, inf], [lowest] * 4, [lowest, -inf, lowest, 0], [-inf, -inf, -inf, -inf], [inf, inf, -inf, 1],
                     [np.nan] * 4, [-200, -300, -200, -201]], np.float32)
    v = rows[np.arange(T) % len(rows)]
    for score in (P.SCORE_SOFTMAX, P.SCORE_SIGMOID):
        got = run(ctx, ctx.moe_route_params(T, 4, 3, score=score), ctx.upload(v), None, T, 3, 4)
        ids, w = moe.route(v, 3, score == P.SCORE_SOFTMAX)
        if score == P.SCORE_SIGMOID:  # (their fp32 sigmoids are 0: so is the sum, and so are the weights)
            w[np.arange(T) % len(rows) == 7] = 0
            w[np.arange(T) % len(rows) == 2] = 0
        check(got, (ids, w), T, 3, 4)
    bias = np.array([-inf, np.nan, 0.5, 0.25], np.float32)
    got = run(ctx, ctx.moe_route_params(T, 4, 3, score=P.SCORE_SIGMOID, renorm=False), ctx.upload(v), ctx.upload(bias), T, 3, 4)
    check(got, moe.route(v, 3, False, False, 1.0, bias), T, 3, 4)


@pytest.mark.parametrize("T,E,k", [(3, 64, 8), (100, 300, 6)])
def test_scores_next_to_a_border(ctx, T, E, k):
    """sigmoid + bias that differ in the last bits of fp32, or only beyond them: few such experts, and more than a warp has lanes."""
    rng = np.random.default_rng(E)
    v = rng.standard_normal((T, E)).astype(np.float32)
    prm = ctx.moe_route_params(T, E, k, score=P.SCORE_SIGMOID)
    for near in (4, 20, E):
        one = v.copy()
        one[:, :near] = 2.0 + np.arange(near, dtype=np.float32) % 5 * np.float32(2.0 ** -22)
        bias = np.where(np.arange(E) < near, 3.0, 0.0).astype(np.float32)   # (the sum has 22 bits behind the point)
        got = run(ctx, prm, ctx.upload(one), ctx.upload(bias), T, k, E)
        check(got, moe.route(one, k, False, True, 1.0, bias), T, k, E)
        bias = np.where(np.arange(E) < near, 1e6, 0.0).astype(np.float32)   # all alike in fp32
        got = run(ctx, prm, ctx.upload(one), ctx.upload(bias), T, k, E)
        check(got, moe.route(one, k, False, True, 1.0, bias), T, k, E)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_row_stride_and_alignment(ctx, oracle, dtype):
    """Rows of a wider buffer that ends with the last row's last logit, off any wide boundary."""
    T, E, k, ld = 100, 37, 4, 41
    v = np.random.default_rng(3).standard_normal((T, ld)).astype(np.float32)
    raw = oracle.to_bf16(v) if dtype == BF16 else v
    v = oracle.from_bf16(raw) if dtype == BF16 else v
    flat = raw.reshape(-1)[:(T - 1) * ld + E]
    room = ctx.upload(np.concatenate([flat[:1], flat]))
    src = ctx.wrap(room.device_ptr + flat.itemsize, flat.nbytes)
    got = run(ctx, ctx.moe_route_params(T, E, k, logits_dtype=dtype, ld=ld), src, None, T, k, E)
    check(got, moe.route(v[:, :E], k), T, k, E)


@pytest.mark.parametrize("T,E,k", [(1, 4, 2), (50, 16, 8), (3000, 300, 4)])
def test_experts_that_are_given(ctx, T, E, k):
    """ids is read: values of no expert go nowhere, a token may name one twice."""
    ids = np.random.default_rng(T).integers(-2, E + 2, (T, k)).astype(np.int32)
    ids[0, 1] = ids[0, 0]
    got = run(ctx, ctx.moe_route_params(T, E, k), None, None, T, k, E, ids=ids)
    np.testing.assert_array_equal(got["ids"].reshape(T, k), ids)
    assert (got["weights"] == -9).all()
    check_sort(got, np.where((ids >= 0) & (ids < E), ids, -1), E)


def test_no_tokens(ctx):
    got = run(ctx, ctx.moe_route_params(0, 9, 2), ctx.upload(np.zeros(4, np.float32)), None, 0, 2, 9)
    assert not got["offsets"].any()


def test_all_tokens_to_one_expert(ctx):
    T, E, k = 4000, 128, 1
    v = np.zeros((T, E), np.float32)
    v[:, 77] = 1
    got = run(ctx, ctx.moe_route_params(T, E, k), ctx.upload(v), None, T, k, E)
    check(got, moe.route(v, k), T, k, E)


def test_repeated_and_recorded(ctx):
    """The same bits every time, eagerly and from a graph; a graph recorded before the workspace exists is refused."""
    T, E, k = 2000, 64, 8
    v = np.random.default_rng(9).standard_normal((T, E)).astype(np.float32)
    prm, logits = ctx.moe_route_params(T, E, k), ctx.upload(v)
    bufs = [ctx.upload(np.zeros(T * k, np.int32)) for _ in range(4)] + [ctx.upload(np.zeros(E + 1, np.int32))]
    ctx.graph_begin()
    with pytest.raises(BackendError) as e:
        ctx.moe_route(prm, logits, None, *bufs)
    assert e.value.code == P.ERR_NOT_SUPPORTED
    ctx.graph_destroy(ctx.graph_end())
    ctx.moe_route(prm, logits, None, *bufs)
    want = [b.to_host() for b in bufs]
    ctx.graph_begin()
    ctx.moe_route(prm, logits, None, *bufs)
    g = ctx.graph_end()
    for _ in range(3):
        for b in bufs:
            b.from_host(np.full(b.nbytes // 4, 5, np.int32))
        ctx.graph_launch(g)
        for b, w in zip(bufs, want):
            np.testing.assert_array_equal(b.to_host(), w)
    ctx.graph_destroy(g)


def test_refusals(ctx):
    E, k, T = 8, 2, 4
    f = lambda n: ctx.upload(np.zeros(n, np.float32))  # noqa: E731
    logits, bias, ids, w, order, pos, off = f(T * E), f(E), f(T * k), f(T * k), f(T * k), f(T * k), f(E + 1)

    def refused(prm=None, **other):
        a = dict(logits=logits, bias=None, ids=ids, weights=w, order=order, pos=pos, offsets=off)
        a.update(other)
        with pytest.raises(BackendError) as e:
            ctx.moe_route(prm or ctx.moe_route_params(T, E, k), *a.values())
        assert e.value.code == P.ERR_INVALID, str(e.value)
    R = ctx.moe_route_params
    for prm in (R(T, 0, k), R(T, 1025, k), R(T, E, 0), R(T, E, 9), R(T, E, 33), R(T, E, k, score=2), R(T, E, k, logits_dtype=P.F16), R(T, E, k, ld=7), R(2 ** 31, E, k),
                R(T + 1, E, k), R(T, E + 1, k), R(T, E, 3)):
        refused(prm)
    refused(bias=bias)                                        # softmax has none
    refused(R(T, E, k, score=P.SCORE_SIGMOID), logits=None, bias=bias)
    refused(weights=None)
    refused(order=pos)
    refused(offsets=logits)
    refused(pos=ctx.wrap(pos.device_ptr + 2, T * k * 4))
    refused(logits=f(T * E - 1))
    refused(offsets=f(E))
    ctx.sync()

"""Buffers past 2^31 elements or bytes: the last rows, the last expert.  The rest of the buffers is never looked at and holds whatever it holds."""
import numpy as np
import pytest

from mlx_b200 import BF16
from oracle import moe

pytestmark = pytest.mark.gpu
ROWS, DIM, TAIL = 270000, 8192, 20  # rows x DIM: more than 2^31 elements


def tail(ctx, buf, total, a):
    """a at the end of the `total` bytes of buf; the part of buf that holds it."""
    part = ctx.wrap(buf.device_ptr + total - a.nbytes, a.nbytes, a.shape, a.dtype)
    part.from_host(a)
    return part


def close(oracle, raw, want, tol):
    got = oracle.from_bf16(raw).astype(np.float64)
    bad = ~(np.abs(got - want) <= tol + 2.0 ** -8 * (np.abs(want) + tol))
    assert not bad.any(), (np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])


@pytest.mark.parametrize("which", ["few", "many"])
@pytest.mark.parametrize("gathered", [False, True])
def test_experts(ctx, oracle, monkeypatch, which, gathered):
    monkeypatch.setenv("LUXCUDA_EXPERTS", which)
    E, K, N, bits, group = 136, DIM, DIM, 4, 128  # packed weights of 4.5 GB
    layer = oracle.make_layer(N, K, bits, group, oracle.BF16, config_id=51)
    bufs = [ctx.alloc(E * a.nbytes, None, None) for a in layer]
    for buf, a in zip(bufs, layer):
        tail(ctx, buf, E * a.nbytes, a)
    x, y = ctx.empty((ROWS, K), np.uint16), ctx.empty((ROWS, N), np.uint16)
    xs = oracle.make_x(TAIL, K, oracle.BF16)
    tail(ctx, x, ROWS * K * 2, xs)
    out = tail(ctx, y, ROWS * N * 2, np.zeros((TAIL, N), np.uint16))
    offsets = np.full(E + 1, ROWS - TAIL, np.int32)
    offsets[E] = ROWS
    order = None
    if gathered:
        rows = np.arange(ROWS, dtype=np.int32)
        rows[-TAIL:] = rows[-TAIL:][::-1]
        order, xs = ctx.upload(rows), xs[::-1]
    ctx.qmatmul_experts(ctx.experts_params(ROWS, ROWS, E, K, N, bits, group), x, order, ctx.upload(offsets), *bufs, None, y)
    got = out.to_host()
    ctx.sync()
    assert ctx.last_kernel().startswith("qmv" if which == "few" else "qmm")
    values = oracle.from_bf16(oracle.dequantize(*layer, K, bits, group, oracle.BF16))
    close(oracle, got, *moe.epilogue(*moe.product(oracle.from_bf16(xs), values), K, 0, False))


def test_epilogue(ctx, oracle):
    K, N = 128, DIM
    layer = oracle.make_layer(N, K, 4, 64, oracle.BF16, config_id=52)
    x, y, res = ctx.empty((ROWS, K), np.uint16), ctx.empty((ROWS, N), np.uint16), ctx.empty((ROWS, N), np.uint16)
    xs, rs = oracle.make_x(TAIL, K, oracle.BF16), oracle.make_x(TAIL, N, oracle.BF16, tag=1)
    tail(ctx, x, ROWS * K * 2, xs)
    tail(ctx, res, ROWS * N * 2, rs)
    out = tail(ctx, y, ROWS * N * 2, np.zeros((TAIL, N), np.uint16))
    ctx.qmatmul_epi(ctx.qmm_epi_params(ROWS, K, N, 4, 64, r_dtype=BF16), x, *(ctx.upload(a) for a in layer), None, res, y)
    got = out.to_host()
    ctx.sync()
    values = oracle.from_bf16(oracle.dequantize(*layer, K, 4, 64, oracle.BF16))
    close(oracle, got, *moe.epilogue(*moe.product(oracle.from_bf16(xs), values), K, 0, False, oracle.from_bf16(rs)))


@pytest.mark.parametrize("dim", [DIM, DIM - 1])
def test_combine(ctx, oracle, dim):
    """(8191: no wide loads, still 2.2e9 elements)"""
    T, k = 5, 4
    y = ctx.empty((ROWS, dim), np.uint16)
    ys = oracle.make_x(T * k, dim, oracle.BF16)
    tail(ctx, y, ROWS * dim * 2, ys)
    pos, w = np.arange(ROWS - T * k, ROWS, dtype=np.int32).reshape(T, k), np.random.default_rng(0).random((T, k)).astype(np.float32)
    out = ctx.empty((T, dim), np.uint16)
    ctx.moe_combine(ctx.moe_combine_params(T, dim, k, ROWS), y, ctx.upload(pos), ctx.upload(w), None, out)
    v = oracle.from_bf16(ys).astype(np.float64).reshape(T, k, dim)
    terms = np.abs(v * w[..., None]).sum(1)
    close(oracle, out.to_host(), (v * w[..., None]).sum(1), k * 2.0 ** -24 * terms)


def test_route(ctx, oracle):
    """A row stride of 4e8 elements."""
    T, E, k, ld = 8, 64, 4, 400_000_000
    rng = np.random.default_rng(3)
    v = np.stack([rng.permutation(E) for _ in range(T)]).astype(np.float32) / 8
    logits = ctx.alloc(((T - 1) * ld + E) * 2, None, None)
    for t in range(T):
        row = oracle.to_bf16(v[t])
        ctx.wrap(logits.device_ptr + t * ld * 2, row.nbytes).from_host(row)
    ids, weights = ctx.empty((T, k), np.int32), ctx.empty((T, k), np.float32)
    order, pos, offsets = ctx.empty((T * k,), np.int32), ctx.empty((T * k,), np.int32), ctx.empty((E + 1,), np.int32)
    ctx.moe_route(ctx.moe_route_params(T, E, k, logits_dtype=BF16, ld=ld), logits, None, ids, weights, order, pos, offsets)
    np.testing.assert_array_equal(ids.to_host(), np.argsort(-v, axis=1)[:, :k])

"""The weighted sum of a token's expert outputs against 64 bits."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32, BackendError
from mlx_b200 import plugin as P
from oracle import moe

pytestmark = pytest.mark.gpu


def values(ctx, oracle, rng, shape, dtype, shift=0):
    """Random values on the device, `shift` elements past a 16-byte boundary, and as fp64."""
    v = rng.standard_normal(shape).astype(np.float32)
    raw = oracle.to_bf16(v) if dtype == BF16 else v
    v = oracle.from_bf16(raw) if dtype == BF16 else v
    room = ctx.upload(np.concatenate([np.zeros(shift, raw.dtype), raw.reshape(-1)]))
    return ctx.wrap(room.device_ptr + shift * raw.itemsize, raw.nbytes, shape, raw.dtype), room, v.astype(np.float64)


@pytest.mark.parametrize("y_dtype", [F32, BF16])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("T,dim,k,shift", [(1, 8, 1, 0), (1, 4096, 8, 0), (7, 5003, 3, 0), (16, 2048, 32, 0), (300, 1, 5, 0), (33, 96, 9, 1), (2000, 264, 2, 0)])
def test_combine(ctx, oracle, y_dtype, out_dtype, T, dim, k, shift):
    rng = np.random.default_rng(T * dim + k)
    y, _r1, yv = values(ctx, oracle, rng, (T * k, dim), y_dtype, shift)
    res, _r2, rv = values(ctx, oracle, rng, (T, dim), out_dtype, shift)
    pos = rng.permutation(T * k).astype(np.int32)
    pos[rng.random(T * k) < 0.2] = -1
    pos[:k] = -1                     # a token without an expert
    if T > 2:
        pos[k] = T * k               # outside: adds nothing
    w = rng.standard_normal(T * k).astype(np.float32)
    there = (pos >= 0) & (pos < T * k)
    for weights, residual, in_place in ((w, True, False), (None, True, True), (w, False, False)):
        out = res if in_place else ctx.empty((T, dim), np.uint16 if out_dtype == BF16 else np.float32)
        prm = ctx.moe_combine_params(T, dim, k, T * k, y_dtype=y_dtype, out_dtype=out_dtype)
        ctx.moe_combine(prm, y, ctx.upload(pos), None if weights is None else ctx.upload(weights), res if residual else None, out)
        got = out.to_host((T, dim), np.uint16 if out_dtype == BF16 else np.float32)
        got = oracle.from_bf16(got).astype(np.float64) if out_dtype == BF16 else got.astype(np.float64)
        ww = np.where(there, 1.0 if weights is None else weights.astype(np.float64), 0.0).reshape(T, k)
        rows = yv[np.where(there, pos, 0)].reshape(T, k, dim)
        want = np.einsum("tk,tkd->td", ww, rows) + (rv if residual else 0)
        size = np.einsum("tk,tkd->td", np.abs(ww), np.abs(rows)) + (np.abs(rv) if residual else 0)
        tol = k * moe.U * size  # k roundings of partial sums, none larger than the sum of magnitudes
        tol = tol + (2.0 ** -8 * (np.abs(want) + tol) if out_dtype == BF16 else 0)
        assert (np.abs(got - want) <= tol).all()
        if in_place:
            res.from_host(oracle.to_bf16(rv.astype(np.float32)) if out_dtype == BF16 else rv.astype(np.float32))


@pytest.mark.parametrize("y_dtype", [F32, BF16])
@pytest.mark.parametrize("out_dtype", [F32, BF16])
@pytest.mark.parametrize("dim", [4, 12, 2, 6, 3, 5, 1028, 1030, 1031])
@pytest.mark.parametrize("T,k,shift", [(9, 5, 0), (9, 5, 2), (9, 5, 4), (9, 2, 0), (9, 1, 2), (700, 5, 0)])
def test_pieces_of_a_row(ctx, oracle, y_dtype, out_dtype, dim, T, k, shift):
    """Pieces of 4, 2 and single columns, buffers that begin so many elements past a 16-byte boundary: the bits of a row of the same values whose
    pieces are wide ones."""
    rng = np.random.default_rng(dim + shift)
    wide = (dim + 7) // 8 * 8
    v, r = rng.standard_normal((T * k, wide)).astype(np.float32), rng.standard_normal((T, wide)).astype(np.float32)
    pos, w = ctx.upload(rng.permutation(T * k).astype(np.int32)), ctx.upload(rng.standard_normal(T * k).astype(np.float32))

    def run(n, shift):
        bufs = []
        for a, dt in ((v, y_dtype), (r, out_dtype), (np.zeros_like(r), out_dtype)):
            raw = a[:, :n].reshape(-1)
            raw = oracle.to_bf16(raw) if dt == BF16 else raw
            room = ctx.upload(np.concatenate([np.full(shift, 7, raw.dtype), raw, np.full(8, 7, raw.dtype)]))
            bufs.append((room, ctx.wrap(room.device_ptr + shift * raw.itemsize, raw.nbytes)))
        ctx.moe_combine(ctx.moe_combine_params(T, n, k, T * k, y_dtype=y_dtype, out_dtype=out_dtype), bufs[0][1], pos, w, bufs[1][1], bufs[2][1])
        got = bufs[2][0].to_host()
        assert (got[:shift] == 7).all() and (got[-8:] == 7).all()
        return got[shift:-8].reshape(T, n)

    np.testing.assert_array_equal(run(dim, shift), run(wide, 0)[:, :dim])


def test_rows_of_nobody_are_not_read(ctx):
    """Infinities and NaN in rows that no pair stands for do not come through."""
    T, dim, k = 5, 64, 2
    y = np.full((T * k, dim), np.nan, np.float32)
    y[3] = 2.0
    pos = np.full(T * k, -1, np.int32)
    pos[4] = 3
    out = ctx.empty((T, dim), np.float32)
    ctx.moe_combine(ctx.moe_combine_params(T, dim, k, T * k, y_dtype=F32, out_dtype=F32), ctx.upload(y), ctx.upload(pos), ctx.upload(np.full(T * k, 0.5, np.float32)), None, out)
    want = np.zeros((T, dim), np.float32)
    want[2] = 1.0
    np.testing.assert_array_equal(out.to_host(), want)


def test_refusals(ctx):
    T, dim, k = 4, 16, 2
    f = lambda n: ctx.upload(np.zeros(n, np.float32))  # noqa: E731
    y, pos, w, res, out = f(T * k * dim), f(T * k), f(T * k), f(T * dim), f(T * dim)
    C = lambda *a, **kw: ctx.moe_combine_params(*a, **dict(dict(y_dtype=F32, out_dtype=F32), **kw))  # noqa: E731

    def refused(prm, *args):
        with pytest.raises(BackendError) as e:
            ctx.moe_combine(prm, *args)
        assert e.value.code == P.ERR_INVALID
    good = C(T, dim, k, T * k)
    for prm in (C(T, dim, 0, T * k), C(T, dim, 33, T * k), C(T + 1, dim, k, T * k), C(T, dim, k, T * k + 1), C(T, dim, k, T * k, y_dtype=P.F16), C(2 ** 31, dim, k, 1), C(T, 2 ** 31, k, 1)):
        refused(prm, y, pos, w, res, out)
    refused(good, y, pos, w, res, y)
    refused(good, y, pos, w, ctx.wrap(out.device_ptr + 4, T * dim * 4 - 4), out)
    refused(good, y, pos, w, out, ctx.wrap(out.device_ptr, T * dim * 4 - 4))
    refused(good, y, ctx.wrap(pos.device_ptr + 2, T * k * 4), w, res, out)
    ctx.moe_combine(C(0, dim, k, T * k), y, pos, w, res, out)  # nothing to do
    ctx.sync()

"""The gate functions of block_norm over their whole range, in every kernel that has them."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32
from mlx_b200 import plugin as P
from oracle import mx4

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def gates(dtype):
    """bf16: all of them (as bits); fp32: where the sigmoid's exponential leaves the range, the ends of the range, both signs of everything."""
    if dtype == BF16:
        bits = np.arange(65536, dtype=np.uint32).astype(np.uint16)
        return bits, (bits.astype(np.uint32) << 16).view(np.float32)
    rng = np.random.default_rng(7)
    top = np.finfo(np.float32).max
    a = np.concatenate([np.linspace(80, 110, 24000), np.exp(rng.uniform(np.log(1e-38), np.log(float(top)), 8000)), [0.0, 20, 87, 88.7, 89, 95, 112, 1000, 1e-45, np.inf, np.nan, top, 2.36e38, 2.4e38]])
    a = np.concatenate([a, -a]).astype(np.float32)
    return a, a


def want_and_tolerance(g, act):
    """Sigmoid: 2^t by the machine's exponential (2 units in the last place, 4 U, from its rounded value, U), its correction and 1 + 2^t (U each), the
    machine's reciprocal (2 U), results below the normal numbers flushed; tanh: two units in the last place; the product with 1 is exact."""
    with np.errstate(over="ignore", invalid="ignore"):
        want = mx4.gate(g, act)
    if act == P.GATE_IDENTITY:
        return want, np.zeros_like(want)
    return want, np.abs(want) * 10 * U + 2.0 ** -126 if act == P.GATE_SIGMOID else np.abs(want) * 4 * U + 2.0 ** -148


# rows, dim, gate_rows: registers, whole rows; registers, cut rows; two rows to a warp; off 16-byte boundaries; long rows, eight and one at a time; the
# ring with a gate of the rows' own; the ring and the registers with a gate that all rows share
FORMS = [(17, 4096, 1), (16, 4104, 1), (2100, 32, 1), (65, 1025, 1), (5, 16392, 1), (5, 16385, 1), (620, 4096, 36), (600, 8192, 0), (3, 8192, 0)]


@pytest.mark.parametrize("act", [P.GATE_IDENTITY, P.GATE_SIGMOID, P.GATE_TANH])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,dim,gate_rows", FORMS)
def test_every_gate(ctx, act, dtype, rows, dim, gate_rows):
    raw, values = gates(dtype)
    n = (rows + gate_rows - 1) // gate_rows if gate_rows else 1
    h = ctx.upload(np.full((rows, dim), 0x3F80 if dtype == BF16 else 1, np.uint16 if dtype == BF16 else np.float32))
    out = ctx.empty((rows, dim), np.float32)
    prm = ctx.block_norm_params(rows, dim, gate_act=act, gate_rows=gate_rows, x_dtype=dtype, r_dtype=F32)
    gate = ctx.empty((n, dim), raw.dtype)
    for first in range(0, len(raw), n * dim):
        at = np.arange(first, first + n * dim) % len(raw)
        gate.from_host(raw[at].reshape(n, dim))
        ctx.block_norm(prm, h, gate, None, None, None, None, None, out, None)
        want, tol = want_and_tolerance(values[at].reshape(n, dim), act)
        per_row = np.arange(rows) // gate_rows if gate_rows else np.zeros(rows, int)
        got = out.to_host().astype(np.float64)
        for r in range(rows):
            w, t, o = want[per_row[r]], tol[per_row[r]], got[r]
            nan = np.isnan(w)
            assert np.array_equal(np.isnan(o), nan), values[at].reshape(n, dim)[per_row[r]][np.isnan(o) != nan][:8]
            same = (o == w) | nan  # (infinities among them)
            with np.errstate(invalid="ignore"):
                assert (same | (np.abs(o - w) <= t)).all(), np.nanmax(np.abs(o - w))


@pytest.mark.parametrize("rows,dim", [(4, 256), (4, 99), (3, 16400), (1200, 2048)])
def test_a_closed_gate_leaves_the_stream(ctx, rows, dim):
    """A sigmoid gate of minus infinity (or the lowest value) on some channels, of infinity on the others: the stream alone there, with the whole branch here;
    the norm behind it sees neither infinities nor NaN."""
    rng = np.random.default_rng(dim)
    h, r = rng.integers(-8, 9, (2, rows, dim)).astype(np.float32)
    g = np.where(np.arange(dim) % 3 == 0, np.float32(-np.inf), np.where(np.arange(dim) % 3 == 1, np.finfo(np.float32).min, np.float32(np.inf))).astype(np.float32)
    new, out = ctx.empty((rows, dim), np.float32), ctx.empty((rows, dim), np.float32)
    prm = ctx.block_norm_params(rows, dim, pre=P.NORM_RMS, gate_act=P.GATE_SIGMOID, x_dtype=F32, r_dtype=F32, out_dtype=F32, branch_scale=0.5, eps=1e-5)
    bh, bg, br = ctx.upload(h), ctx.upload(g), ctx.upload(r)
    ctx.block_norm(prm, bh, bg, br, None, None, None, None, new, out)
    want = r + np.where(g > 0, np.float32(0.5), np.float32(0)) * h  # exact: small whole numbers and halves
    np.testing.assert_array_equal(new.to_host(), want)
    assert np.isfinite(out.to_host()).all()

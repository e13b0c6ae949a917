"""The activations of the products' epilogues, value by value: x is zero, so that a product is its bias, exactly.

Tolerances, relative to the result, in U = 2^-24 (half a unit of the 24th bit):
  silu       v / (1 + e), e = exp(-u) with u = v: the machine's exponential 4 U, the correction's rounding 1, log2(e) in 24 bits 0.23 |u|; the sum 1, the machine's
             reciprocal 2, the product 1; 1 for what is of second order
  gelu_tanh  the same with u = v (c0 + c1 v^2): four roundings and constants on the way to u, 4 |u| more
  gelu       v erfc(t) / 2, t = -v / sqrt 2: erfc 8 U (a library's; the kernels' own polynomial 5.4 U with its roundings, exponential and reciprocal 7.4 more with
             both at their worst), the product 1; t is off by 1.3 U of itself, which erfc, falling by d log erfc / d log t <= 2 t^2 + 1 = v^2 + 1, makes
             1.3 (v^2 + 1) (the kernels' exponent: 1.1 v^2); 1 for what is of second order
For v > 0 the errors in u and t count by e's share of 1 + e and by erfc's fall, 4.23 u e / (1 + e) < 1.2 and 1.3 |t erfc'(t) / erfc(t)| < 0.7: 12 U in all.
Below u = -87 (gelu: v = -13) results and errors are below |v| 2^-125, where numbers have fewer bits."""
import math

import numpy as np
import pytest

from mlx_b200 import BF16, F32
from mlx_b200 import plugin as P

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
ACTS = {"none": P.ACT_NONE, "relu": P.ACT_RELU, "silu": P.ACT_SILU, "gelu": P.ACT_GELU, "gelu_tanh": P.ACT_GELU_TANH}


def values():
    v = np.concatenate([np.linspace(-10, 10, 1201), np.linspace(-13, -4, 181), np.linspace(-0.01, 0.01, 41), 2.0 ** np.arange(-140, 128, 7), -2.0 ** np.arange(-140, 128, 7),
                        [-3.4e38, -1e30, -1e4, -700, -127, -104, -90, -89, -88.5, -88, -87.5, -87, -86, -60, -40, -20, 20, 40, 87, 88, 89, 127, 1e4, 1e30, 3.4e38],
                        [0.0, -0.0, np.inf, -np.inf, np.nan]]).astype(np.float32)
    return np.concatenate([v, np.zeros(-len(v) % 64, np.float32)])


def want(act, v):
    """(values, tolerances) in 64 bits."""
    v = v.astype(np.float64)
    if act == "none":
        return v, np.zeros_like(v)
    if act == "relu":
        return np.where(v < 0, 0.0, v), np.zeros_like(v)
    with np.errstate(all="ignore"):
        if act == "gelu":
            r = np.array([math.nan if math.isnan(a) else 0.5 * a * math.erfc(-a / math.sqrt(2)) for a in v])
            rel, few = (10 + 1.3 * (v * v + 1)) * U, v < -13
        else:
            u = v if act == "silu" else 2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3)
            r = v / (1 + np.exp(-u))
            rel, few = (10 + 0.23 * np.abs(u) + (4 * np.abs(u) if act == "gelu_tanh" else 0)) * U, u < -87
        rel = np.where(v > 0, np.minimum(rel, 12 * U), rel)
        return r, np.where(few, np.abs(v) * 2.0 ** -125, rel * np.abs(r) + 2.0 ** -149)


def check(got, act, v, times=1.0):
    r, tol = want(act, v)
    with np.errstate(invalid="ignore"):
        r, tol = r * times, tol * abs(times)
        tol = np.where(np.isinf(r) | (np.abs(v) == np.inf), 0.0, tol)
        big = np.abs(r) > np.finfo(np.float32).max
        bad = ~((np.abs(got - r) <= tol) | (got == r) | (np.isnan(got) & np.isnan(r)) | (big & np.isinf(got) & (np.sign(got) == np.sign(r))))
    assert not bad.any(), (act, [(i, float(v[i[-1]]), float(got[tuple(i)]), float(np.broadcast_to(r, got.shape)[tuple(i)])) for i in np.argwhere(bad)[:6]])


def test_what_is_asked_for():
    """The tolerances are below the values, but where these vanish, and the formulas' values at both infinities are these."""
    v = values()
    for act in ACTS:
        r, tol = want(act, v)
        some = np.isfinite(r) & (np.abs(r) > 2.0 ** -100)
        assert (tol[some] <= 1e-4 * np.abs(r[some])).all()
        at = dict(zip(v.tolist(), r.tolist()))
        assert at[math.inf] == math.inf
        assert {"none": at[-math.inf] == -math.inf, "relu": at[-math.inf] == 0}.get(act, math.isnan(at[-math.inf]))


# one row, sixteen, rows by sixteen (K off 64), single CTAs, pairs of CTAs that store by copy and directly, stream-K
@pytest.mark.parametrize("M,K,schedule,pair,direct", [(1, 128, None, None, 0), (16, 128, None, None, 0), (40, 96, None, None, 0), (40, 128, "tiles", "0", 0), (40, 128, "tiles", "1", 0),
                                                      (40, 128, "tiles", "1", 1), (40, 256, "streamk", "0", 0)])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("y_dtype", [F32, BF16])
def test_epilogue(ctx, oracle, monkeypatch, M, K, schedule, pair, direct, act, y_dtype):
    if schedule:
        monkeypatch.setenv("LUXCUDA_QMM_SCHEDULE", schedule)
        monkeypatch.setenv("LUXCUDA_QMM_PAIR", pair)
        if direct:
            monkeypatch.setenv("LUXCUDA_QMM_NO_YTMA", "1")
    v = values()
    N = len(v)
    w = [ctx.upload(a) for a in oracle.make_layer(N, K, 4, 32, oracle.BF16, config_id=46)]
    y = ctx.empty((M, N), np.float32 if y_dtype == F32 else np.uint16)
    ctx.qmatmul_epi(ctx.qmm_epi_params(M, K, N, 4, 32, act=ACTS[act], y_dtype=y_dtype), ctx.upload(np.zeros((M, K), np.uint16)), *w, ctx.upload(v), None, y)
    if schedule:
        assert ctx.last_kernel() == "qmm_tc<4" + {"0": ",stream-k>" if schedule == "streamk" else ">", "1": ",pairs>"}[pair]
    finish(ctx, oracle, y, y_dtype, act, v, 1.0)


def finish(ctx, oracle, y, y_dtype, act, v, times):
    if y_dtype == F32:
        check(y.to_host().astype(np.float64), act, v, times)
        return
    # bf16: the nearest to a value within the tolerance
    got = oracle.from_bf16(y.to_host()).astype(np.float64)
    r, tol = want(act, v)
    with np.errstate(invalid="ignore", over="ignore"):
        r, tol = r * times, np.where(np.isfinite(r), tol * abs(times), 0.0)
        tol = tol + 2.0 ** -8 * (np.abs(r) + tol) + 2.0 ** -134
        over = np.abs(r) >= 2.0 ** 128 * (1 - 2.0 ** -9)
        bad = ~((np.abs(got - r) <= tol) | (got == r) | (np.isnan(got) & np.isnan(r)) | (over & np.isinf(got)))
    assert not bad.any(), (act, [(float(v[i[-1]]), float(got[tuple(i)])) for i in np.argwhere(bad)[:6]])


@pytest.mark.parametrize("rows,which,pair", [(6, "few", "0"), (90, "many", "0"), (90, "many", "1")])
@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("y_dtype", [F32, BF16])
@pytest.mark.parametrize("up", [None, 1.0, -2.0])
def test_experts(ctx, oracle, monkeypatch, rows, which, pair, act, y_dtype, up):
    monkeypatch.setenv("LUXCUDA_EXPERTS", which)
    monkeypatch.setenv("LUXCUDA_EXPERTS_PAIR", pair)
    v = values()
    E, K, N = 2, 128, len(v) * (1 if up is None else 2)
    bias = np.stack([v if up is None else np.concatenate([v, np.full_like(v, up)])] * E)
    w = [ctx.upload(a) for a in oracle.make_layer(E * N, K, 4, 32, oracle.BF16, config_id=47)]
    y = ctx.empty((rows, len(v)), np.float32 if y_dtype == F32 else np.uint16)
    prm = ctx.experts_params(rows, rows, E, K, N, 4, 32, act=ACTS[act], gated=up is not None, y_dtype=y_dtype)
    ctx.qmatmul_experts(prm, ctx.upload(np.zeros((rows, K), np.uint16)), None, ctx.upload(np.array([0, rows // 3, rows], np.int32)), *w, ctx.upload(bias), y)
    assert ctx.last_kernel() == ("qmv_experts<4>" if which == "few" else "qmm_experts<4,pairs>" if pair == "1" else "qmm_experts<4>")
    finish(ctx, oracle, y, y_dtype, act, v, 1.0 if up is None else up)

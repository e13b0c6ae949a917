"""Every form of the prefill GEMM with an epilogue, each forced in turn: whole tiles of one CTA, of pairs of CTAs (stored by copy and directly), stream-K (whole and split
tiles); and the products' sums in the 2-norm, where a bound is far sharper than value by value."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32
from mlx_b200 import plugin as P
from oracle import moe

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
GUARD = 64
FORMS = {"tiles": ("tiles", "0", False, ">"), "pairs": ("tiles", "1", False, ",pairs>"), "pairs, direct": ("tiles", "1", True, ",pairs>"), "stream-k": ("streamk", "0", False, ",stream-k>")}


def force(monkeypatch, form):
    schedule, pair, direct, end = FORMS[form]
    monkeypatch.setenv("LUXCUDA_QMM_SCHEDULE", schedule)
    monkeypatch.setenv("LUXCUDA_QMM_PAIR", pair)
    if direct:
        monkeypatch.setenv("LUXCUDA_QMM_NO_YTMA", "1")
    return end


# two tiles of W, three (the second CTA of the last pair has none), columns that are no multiple of 8, one column more than a tile; an odd number of sub-blocks of K; more tiles
# than SMs (stream-K: CTAs that hold whole tiles between two split ones), fewer (tiles over many CTAs)
@pytest.mark.parametrize("form", list(FORMS))
@pytest.mark.parametrize("M,K,N,bits,group", [(300, 1024, 264, 4, 64), (40, 192, 1003, 8, 32), (257, 320, 129, 4, 32), (100, 256, 12800, 8, 64), (600, 256, 4104, 4, 128), (64, 4096, 512, 8, 128)])
def test_epilogue(ctx, oracle, monkeypatch, form, M, K, N, bits, group):
    end = force(monkeypatch, form)
    rng = np.random.default_rng(N)
    wq, s, b = oracle.make_layer(N, K, bits, group, oracle.BF16, config_id=48, layer=K, proj=N)
    x = oracle.make_x(M, K, oracle.BF16, tag=N)
    sums = moe.product(oracle.from_bf16(x), oracle.from_bf16(oracle.dequantize(wq, s, b, K, bits, group, oracle.BF16)))
    bias = rng.standard_normal(N).astype(np.float32)
    res = (rng.standard_normal((M, N)) * 2).astype(np.float32)
    res16 = oracle.to_bf16(res)
    bx, bw, bbias = ctx.upload(x), [ctx.upload(a) for a in (wq, s, b)], ctx.upload(bias)
    for act, with_bias, r_dtype, y_dtype, in_place in ((P.ACT_SILU, True, None, BF16, False), (P.ACT_GELU, False, BF16, BF16, True), (P.ACT_NONE, True, F32, F32, True),
                                                       (P.ACT_GELU_TANH, True, F32, BF16, False), (P.ACT_RELU, False, BF16, F32, False)):
        kind, size = (np.uint16, 2) if y_dtype == BF16 else (np.float32, 4)
        mark = kind(0x7E7E) if y_dtype == BF16 else kind(-12345.5)
        raw_res = None if r_dtype is None else res16 if r_dtype == BF16 else res
        filled = np.full(M * N + 2 * GUARD, mark, kind)
        if in_place:
            filled[GUARD:GUARD + M * N] = raw_res.reshape(-1)
        prm = ctx.qmm_epi_params(M, K, N, bits, group, act=act, r_dtype=BF16 if r_dtype is None else r_dtype, y_dtype=y_dtype)
        room, outs = ctx.upload(filled), []
        y = ctx.wrap(room.device_ptr + GUARD * size, M * N * size)
        r = None if r_dtype is None else y if in_place else ctx.upload(raw_res)
        for _ in range(3):
            room.from_host(filled)
            ctx.qmatmul_epi(prm, bx, *bw, bbias if with_bias else None, r, y)
            assert ctx.last_kernel() == f"qmm_tc<{bits}" + end
            outs.append(room.to_host())
        ctx.sync()
        assert all(np.array_equal(outs[0], o) for o in outs)
        assert (outs[0][:GUARD] == mark).all() and (outs[0][GUARD + M * N:] == mark).all()
        got = outs[0][GUARD:GUARD + M * N].reshape(M, N)
        got = oracle.from_bf16(got).astype(np.float64) if y_dtype == BF16 else got.astype(np.float64)
        v, mag = sums
        if with_bias:
            v, mag = v + bias, mag + np.abs(bias.astype(np.float64))
        want, tol = moe.epilogue(v, mag, K, act, False, None if r_dtype is None else oracle.from_bf16(res16) if r_dtype == BF16 else res)
        if y_dtype == BF16:
            tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        bad = ~(np.abs(got - want) <= tol)
        assert not bad.any(), (form, act, np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])
        for h in (room, *([] if r is None or in_place else [r])):
            h.free()


def close_in_norm(got, want, K):
    """A sum over K is K / 16 steps of the matrix instruction, each of which cuts off up to a unit of the running sum's last place (on average half of one, 2^-24 times
    0.72 of the sum).  The running sums of independent products grow as the root of the step, those of products with a mean as the step itself, so that all
    that is cut off comes to 0.72 / sqrt 3 or 0.72 / 2 of the steps: below K / 32 units U of the result's norm.  4 U for what is added behind."""
    err = np.linalg.norm(got.astype(np.float64) - want) / np.linalg.norm(want)
    assert err <= (K / 32 + 4) * U, (err, (K / 32 + 4) * U)


@pytest.mark.parametrize("M,form", [(1, None), (16, None), (96, "tiles"), (96, "pairs"), (96, "stream-k")])
@pytest.mark.parametrize("K,bits", [(4096, 4), (2880, 8), (512, 4)])
def test_sums_keep_their_bits(ctx, oracle, monkeypatch, M, form, K, bits):
    if form:
        force(monkeypatch, form)
    N = 640
    wq, s, b = oracle.make_layer(N, K, bits, 32, oracle.BF16, config_id=49, layer=K)
    x = oracle.make_x(M, K, oracle.BF16, tag=M)
    want, _ = moe.product(oracle.from_bf16(x), oracle.from_bf16(oracle.dequantize(wq, s, b, K, bits, 32, oracle.BF16)))
    y = ctx.empty((M, N), np.float32)
    ctx.qmatmul_epi(ctx.qmm_epi_params(M, K, N, bits, 32, y_dtype=F32), ctx.upload(x), *(ctx.upload(a) for a in (wq, s, b)), None, None, y)
    close_in_norm(y.to_host(), want, K)


@pytest.mark.parametrize("rows,which,pair", [(9, "few", "0"), (150, "many", "0"), (500, "many", "1")])
@pytest.mark.parametrize("K,bits", [(4096, 4), (2880, 8), (512, 4)])
def test_sums_of_experts_keep_their_bits(ctx, oracle, monkeypatch, rows, which, pair, K, bits):
    monkeypatch.setenv("LUXCUDA_EXPERTS", which)
    monkeypatch.setenv("LUXCUDA_EXPERTS_PAIR", pair)
    E, N = 2, 320
    w = oracle.make_layer(E * N, K, bits, 32, oracle.BF16, config_id=50, layer=K)
    values = oracle.from_bf16(oracle.dequantize(*w, K, bits, 32, oracle.BF16)).reshape(E, N, K)
    x, cut = oracle.make_x(rows, K, oracle.BF16, tag=rows), rows // 3
    want = np.concatenate([moe.product(oracle.from_bf16(part), values[e])[0] for e, part in enumerate((x[:cut], x[cut:]))])
    y = ctx.empty((rows, N), np.float32)
    prm = ctx.experts_params(rows, rows, E, K, N, bits, 32, y_dtype=F32)
    ctx.qmatmul_experts(prm, ctx.upload(x), None, ctx.upload(np.array([0, cut, rows], np.int32)), *(ctx.upload(a) for a in w), None, y)
    close_in_norm(y.to_host(), want, K)

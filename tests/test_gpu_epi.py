"""A product with bias, activation and residual against 64 bits, in every kernel that has the epilogue."""
import numpy as np
import pytest

from mlx_b200 import BF16, F32, BackendError
from mlx_b200 import plugin as P
from oracle import moe

pytestmark = pytest.mark.gpu
GUARD = 64


def run(ctx, oracle, M, K, N, bits, group, act=0, with_bias=True, res=None, y_dtype=BF16, in_place=False, seed=0):
    rng = np.random.default_rng(M * N + K + seed)
    wq, s, b = oracle.make_layer(N, K, bits, group, oracle.BF16, config_id=41, layer=K, proj=N)
    values = oracle.from_bf16(oracle.dequantize(wq, s, b, K, bits, group, oracle.BF16))
    x = oracle.make_x(M, K, oracle.BF16, tag=N + seed)
    bias = rng.standard_normal(N).astype(np.float32) if with_bias else None
    rb = rv = None
    if res is not None:
        rv = (rng.standard_normal((M, N)) * 2).astype(np.float32)
        raw = oracle.to_bf16(rv) if res == BF16 else rv
        rv = oracle.from_bf16(raw) if res == BF16 else rv
    kind, size = (np.uint16, 2) if y_dtype == BF16 else (np.float32, 4)
    mark = kind(0x7E7E) if y_dtype == BF16 else kind(-12345.5)
    filled = np.full(M * N + 2 * GUARD, mark, kind)
    if in_place:
        filled[GUARD:GUARD + M * N] = raw.reshape(-1)
    room = ctx.upload(filled)
    y = ctx.wrap(room.device_ptr + GUARD * size, M * N * size)
    if res is not None:
        rb = y if in_place else ctx.upload(raw)
    prm = ctx.qmm_epi_params(M, K, N, bits, group, act=act, r_dtype=BF16 if res is None else res, y_dtype=y_dtype)
    ctx.qmatmul_epi(prm, ctx.upload(x), ctx.upload(wq), ctx.upload(s), ctx.upload(b), None if bias is None else ctx.upload(bias), rb, y)
    got = room.to_host()
    ctx.sync()
    assert (got[:GUARD] == mark).all() and (got[GUARD + M * N:] == mark).all()
    raw_y = got[GUARD:GUARD + M * N].reshape(M, N)
    got = oracle.from_bf16(raw_y).astype(np.float64) if y_dtype == BF16 else raw_y.astype(np.float64)
    want, tol = moe.epilogue(*moe.product(oracle.from_bf16(x), values, bias), K, act, False, rv)
    if y_dtype == BF16:
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (ctx.last_kernel(), np.argwhere(bad)[:4], got[bad][:4], want[bad][:4], tol[bad][:4])
    return raw_y


ACTS = [P.ACT_NONE, P.ACT_RELU, P.ACT_SILU, P.ACT_GELU, P.ACT_GELU_TANH]


@pytest.mark.parametrize("M", [1, 8, 9, 16, 17, 100, 300])
@pytest.mark.parametrize("y_dtype,res", [(BF16, BF16), (BF16, F32), (F32, F32), (F32, BF16), (BF16, None)])
@pytest.mark.parametrize("bits,group", [(4, 64), (8, 32)])
def test_epilogue(ctx, oracle, M, y_dtype, res, bits, group):
    run(ctx, oracle, M, 512, 264, bits, group, act=ACTS[M % 5], res=res, y_dtype=y_dtype)


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M", [3, 48])
def test_activations(ctx, oracle, act, M):
    for with_bias in (False, True):
        run(ctx, oracle, M, 256, 130, 4, 32, act=act, with_bias=with_bias, res=F32, y_dtype=F32)


# inside a k-block, off 64, long with few columns (where qmatmul splits K), odd N, whole tiles over and over (pairs of CTAs), stream-K
@pytest.mark.parametrize("M,K,N,bits,group", [(1, 96, 7, 4, 32), (20, 96, 33, 8, 32), (4, 16384, 48, 4, 64), (16, 8192, 20, 8, 128), (5, 2912, 129, 4, 32), (40, 2880, 501, 4, 64),
                                              (129, 4096, 640, 4, 128), (512, 2048, 4096, 8, 64), (777, 1024, 1003, 4, 32), (1024, 512, 4104, 4, 64)])
def test_shapes(ctx, oracle, M, K, N, bits, group):
    run(ctx, oracle, M, K, N, bits, group, act=P.ACT_SILU, res=BF16)
    run(ctx, oracle, M, K, N, bits, group, res=F32, y_dtype=F32)


@pytest.mark.parametrize("M", [1, 16, 64, 600])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("N", [512, 515])
def test_in_place(ctx, oracle, M, dtype, N):
    apart = run(ctx, oracle, M, 1024, N, 4, 64, act=P.ACT_GELU, res=dtype, y_dtype=dtype)
    np.testing.assert_array_equal(run(ctx, oracle, M, 1024, N, 4, 64, act=P.ACT_GELU, res=dtype, y_dtype=dtype, in_place=True), apart)


@pytest.mark.parametrize("M", [5, 200])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_on_no_wide_boundary(ctx, oracle, M, dtype):
    """y and the residual one element past a 16-byte boundary (the prefill GEMM does not take that y: within a rounding of its result)."""
    K, N = 512, 264
    w = [ctx.upload(a) for a in oracle.make_layer(N, K, 4, 64, oracle.BF16, config_id=44)]
    x, kind, size = ctx.upload(oracle.make_x(M, K, oracle.BF16)), np.uint16 if dtype == BF16 else np.float32, 2 if dtype == BF16 else 4
    res = oracle.make_x(M, N, oracle.BF16 if dtype == BF16 else oracle.F32, tag=1)
    apart, y = ctx.upload(np.concatenate([res.reshape(-1)[:1], res.reshape(-1)])), ctx.empty((M, N), kind)
    prm = ctx.qmm_epi_params(M, K, N, 4, 64, act=P.ACT_SILU, r_dtype=dtype, y_dtype=dtype)
    ctx.qmatmul_epi(prm, x, *w, None, ctx.upload(res), y)
    want = y.to_host()
    ctx.qmatmul_epi(prm, x, *w, None, ctx.wrap(apart.device_ptr + size, res.nbytes), y)
    np.testing.assert_array_equal(y.to_host(), want)
    room = ctx.upload(np.zeros(M * N + 2, kind))
    ctx.qmatmul_epi(prm, x, *w, None, ctx.upload(res), ctx.wrap(room.device_ptr + size, res.nbytes))
    got = room.to_host()
    assert got[0] == 0 and got[-1] == 0
    a, b = (oracle.from_bf16(v).astype(np.float64) if dtype == BF16 else v.astype(np.float64) for v in (got[1:-1].reshape(M, N), want))
    assert (np.abs(a - b) <= (2.0 ** -7 * np.abs(b) + 1e-4 if dtype == BF16 else 1e-4)).all()


@pytest.mark.parametrize("M,K,N", [(1, 1024, 300), (16, 4096, 512), (64, 1024, 512), (600, 1024, 4096), (33, 96, 50)])
def test_nothing_but_the_product(ctx, oracle, M, K, N):
    """Without bias, activation and residual: the bits of qmatmul (the shapes are none whose K qmatmul splits over CTAs)."""
    wq, s, b = oracle.make_layer(N, K, 4, 32, oracle.BF16, config_id=42)
    x = ctx.upload(oracle.make_x(M, K, oracle.BF16))
    w = [ctx.upload(a) for a in (wq, s, b)]
    y0, y1 = ctx.empty((M, N), np.float32), ctx.empty((M, N), np.float32)
    ctx.qmatmul(x, *w, y0, M, K, N, 4, 32, BF16, BF16, F32)
    ctx.qmatmul_epi(ctx.qmm_epi_params(M, K, N, 4, 32, y_dtype=F32), x, *w, None, None, y1)
    np.testing.assert_array_equal(y0.to_host(), y1.to_host())


@pytest.mark.parametrize("M", [2, 200])
def test_recorded_in_a_chain(ctx, oracle, M):
    """Two layers, each onto the stream in place, recorded and replayed: the bits of calls that wait for each other."""
    K = 256
    layers = [[ctx.upload(a) for a in oracle.make_layer(K, K, 4, 64, oracle.BF16, config_id=43, layer=i)] for i in range(2)]
    start = oracle.make_x(M, K, oracle.BF16)
    r, h = ctx.upload(start), ctx.empty((M, K), np.uint16)
    prm = ctx.qmm_epi_params(M, K, K, 4, 64, act=P.ACT_SILU)

    def step(wait):
        for w in layers:
            ctx.qmatmul_epi(prm, r, *w, None, None, h)
            if wait:
                ctx.sync()
            ctx.qmatmul_epi(prm, h, *w, None, r, r)
            if wait:
                ctx.sync()
    step(True)
    want = r.to_host()
    r.from_host(start)
    step(False)
    np.testing.assert_array_equal(r.to_host(), want)
    ctx.graph_begin()
    step(False)
    g = ctx.graph_end()
    for _ in range(2):
        r.from_host(start)
        ctx.graph_launch(g)
        np.testing.assert_array_equal(r.to_host(), want)
    ctx.graph_destroy(g)


def test_refusals(ctx, oracle):
    M, K, N = 4, 64, 24
    w = dict(zip(("wq", "scales", "biases"), (ctx.upload(a) for a in oracle.make_layer(N, K, 4, 32, oracle.BF16))))
    x, y = ctx.upload(oracle.make_x(M, K, oracle.BF16)), ctx.empty((M, N), np.uint16)
    bias, res = ctx.empty((N,), np.float32), ctx.empty((M, N), np.float32)
    E = ctx.qmm_epi_params

    def refused(prm=None, **other):
        a = dict(x=x, **w, bias=bias, residual=res, y=y)
        a.update(other)
        with pytest.raises(BackendError) as e:
            ctx.qmatmul_epi(prm or E(M, K, N, 4, 32, r_dtype=F32), *a.values())
        assert e.value.code == P.ERR_INVALID, str(e.value)
    for prm in (E(-1, K, N, 4, 32), E(M, K, -1, 4, 32), E(M, 48, N, 4, 32), E(M, K, N, 5, 32), E(M, K, N, 4, 16), E(M, K, N, 4, 32, act=-1), E(M, K, N, 4, 32, act=5),
                E(M, K, N, 4, 32, r_dtype=P.F16), E(M, K, N, 4, 32, y_dtype=P.I32), E(M + 1, K, N, 4, 32), E(M, K, N + 1, 4, 32), E(M, 128, N, 4, 32), E(M, K, N, 8, 32),
                E(M, K, N, 4, 32, y_dtype=F32), E(2 ** 31 - 1, 2 ** 31 - 64, 2 ** 31 - 1, 8, 64)):
        refused(prm)
    refused(bias=ctx.empty((N - 1,), np.float32))
    refused(y=x)
    refused(E(M, K, N, 4, 32, r_dtype=F32), residual=ctx.wrap(y.device_ptr, M * N * 4))      # the stream in fp32, y in bf16, at one place
    refused(E(M - 1, K, N, 4, 32), residual=ctx.wrap(y.device_ptr + 2, M * N * 2 - 2))
    refused(x=ctx.wrap(x.device_ptr + 8, M * K * 2 - 8), prm=E(M - 1, K, N, 4, 32))
    for prm in (E(0, K, N, 4, 32), E(M, K, 0, 4, 32)):
        ctx.qmatmul_epi(prm, x, *w.values(), None, None, y)
    ctx.sync()

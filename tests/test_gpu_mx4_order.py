"""Orders of the chained calls, codes and scales compared; chains of two contexts at once."""
import numpy as np
import pytest

from mlx_b200 import BF16
from mlx_b200 import plugin as P

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("seed,M,K", [(0, 8, 1024), (1, 1, 4096), (2, 40, 512), (3, 130, 1056), (4, 16, 2048), (5, 90, 512)])
def test_codes_and_scales_of_any_order_of_calls(ctx, oracle, seed, M, K):
    """Random programs over a few buffers, as recorded graphs and eagerly, against one call at a time: activations, codes and every scale byte (those of
    rows past the last as they were put there)."""
    rng = np.random.default_rng(100 + seed)
    fmt = P.MX4_E8M0 if seed % 2 else P.MX4_E4M3
    bits = lambda shape: oracle.to_bf16(rng.standard_normal(shape).astype(np.float32))  # noqa: E731
    acts = [ctx.upload(bits((M, K))) for _ in range(3)]
    raw = [ctx.upload(bits((K, K))) for _ in range(2)]

    def operand(rows):
        return ctx.upload(np.zeros((rows, K // 8), np.uint32)), ctx.upload(np.full(ctx.mx4_scale_bytes(rows, K, fmt), 0x11, np.uint8))
    codes, layers = [operand(M) for _ in range(3)], [operand(K) for _ in range(2)]
    prm_mx = ctx.block_norm_params(M, K, post=P.NORM_RMS, pre=P.NORM_LAYER, eps=1e-5, res_scale=0.5, out_format=fmt)
    # half of the quantisations and row steps are written over before anything reads them; what is left at the end is compared whole
    steps = [lambda q=w, r=r: ctx.mx4_quantize(r, *q, K, K, fmt, BF16) for w, r in zip(layers, raw)]
    for _ in range(60):
        kind, a, b = rng.random(), int(rng.integers(3)), int(rng.integers(3))
        c, w = codes[rng.integers(3)], layers[rng.integers(2)]
        if kind < 0.45:
            steps.append(lambda a=a, c=c, pre=float(rng.choice([0.5, 1.0, 3.0])): ctx.mx4_quantize(acts[a], *c, M, K, fmt, BF16, pre))
        elif kind < 0.7:
            steps.append(lambda a=a, c=c, w=w: ctx.mx4_matmul(*c, *w, acts[a], M, K, K, fmt, BF16, 1.0 / K ** 0.5))
        elif kind < 0.78:
            steps.append(lambda w=w, r=raw[rng.integers(2)]: ctx.mx4_quantize(r, *w, K, K, fmt, BF16))
        elif kind < 0.86:
            steps.append(lambda a=a, c=c: ctx.mx4_dequantize(*c, acts[a], M, K, fmt, BF16, 0.5))
        else:
            r = (a + 1 + b % 2) % 3
            steps.append(lambda a=a, r=r, c=c: ctx.block_norm(prm_mx, acts[a], None, acts[r], None, None, None, None, acts[r], *c))
    held = acts + [x for q in codes + layers for x in q]
    start = [b.to_host() for b in held]

    def reset():
        for b, v in zip(held, start):
            b.from_host(v)

    def same(want):
        for b, w in zip(held, want):
            np.testing.assert_array_equal(b.to_host(), w)

    reset()
    for s in steps:
        s()
        ctx.sync()
    want = [b.to_host() for b in held]
    for _ in range(4):
        reset()
        for s in steps:
            s()
        same(want)
    reset()
    ctx.graph_begin()
    for s in steps:
        s()
    g = ctx.graph_end()
    for _ in range(4):
        reset()
        ctx.graph_launch(g)
        same(want)
    ctx.graph_destroy(g)


@pytest.mark.parametrize("shapes", [[(145, 3840, 384, P.MX4_E4M3), (96, 512, 1024, P.MX4_E8M0)], [(128, 4096, 640, P.MX4_E4M3), (16, 4096, 4096, P.MX4_E4M3)],
                                    [(70, 2048, 256, P.MX4_E8M0), (512, 2048, 4096, P.MX4_E4M3)]])
def test_products_of_two_contexts_at_once(plugin, shapes):
    """Clusters of one context's products beside those of another's, and beside pairs: each as by itself."""
    rng = np.random.default_rng(5)
    ctxs = [plugin.context(0) for _ in shapes]
    calls, outs = [], []
    for c, (M, K, N, fmt) in zip(ctxs, shapes):
        def operand(rows):
            scale = rng.integers(125, 129, c.mx4_scale_bytes(rows, K, fmt)) if fmt == P.MX4_E8M0 else rng.integers(50, 60, c.mx4_scale_bytes(rows, K, fmt))
            return c.upload(rng.integers(0, 1 << 32, (rows, K // 8), dtype=np.uint64).astype(np.uint32)), c.upload(scale.astype(np.uint8))
        x, ws, ys = operand(M), [operand(N) for _ in range(3)], [c.empty((M, N), np.float32) for _ in range(3)]
        calls.append(lambda i, c=c, x=x, ws=ws, ys=ys, s=(M, K, N, fmt): c.mx4_matmul(*x, *ws[i % 3], ys[i % 3], *s, P.F32, 0.01))
        outs.append(ys)
    want = []
    for c, call, ys in zip(ctxs, calls, outs):
        for i in range(3):
            call(i)
            c.sync()
        want.append([y.to_host() for y in ys])
    for i in range(300):
        for call in calls:
            call(i)
    for c, ys, w in zip(ctxs, outs, want):
        c.sync()
        for y, v in zip(ys, w):
            np.testing.assert_array_equal(y.to_host(), v)
    for c in ctxs:
        c.close()

"""A layer of experts as a program runs it: route, gate and up, down, sum; eagerly, recorded, in two contexts at once."""
import threading

import numpy as np
import pytest


from mlx_b200 import plugin as P
from oracle import moe

pytestmark = pytest.mark.gpu


class Layer:
    def __init__(self, ctx, oracle, T, E, k, K, F, bits=4, group=64, seed=0, pad=0):
        self.ctx, self.shape = ctx, (T, E, k, K, F, bits, group)
        rng = np.random.default_rng(seed)
        self.logits = rng.standard_normal((T, E)).astype(np.float32)
        if pad:
            self.logits[-pad:] = -np.inf
        self.x, self.res = oracle.make_x(T, K, oracle.BF16, tag=seed), oracle.make_x(T, K, oracle.BF16, tag=seed + 1)
        self.up = oracle.make_layer(E * 2 * F, K, bits, group, oracle.BF16, config_id=51, layer=seed, scale_range=(0.0005, 0.005))
        self.down = oracle.make_layer(E * K, F, bits, group, oracle.BF16, config_id=52, layer=seed, scale_range=(0.0005, 0.005))
        u = ctx.upload
        self.b = dict(logits=u(self.logits), x=u(self.x), res=u(self.res), up=[u(a) for a in self.up], down=[u(a) for a in self.down], ids=ctx.empty((T, k), np.int32),
                      weights=ctx.empty((T, k), np.float32), order=ctx.empty((T * k,), np.int32), pos=ctx.empty((T, k), np.int32), offsets=ctx.empty((E + 1,), np.int32),
                      h=ctx.empty((T * k, F), np.uint16), y=ctx.empty((T * k, K), np.uint16), out=ctx.empty((T, K), np.uint16))
        self.prm = (ctx.moe_route_params(T, E, k), ctx.experts_params(T * k, T, E, K, 2 * F, bits, group, top_k=k, act=P.ACT_SILU, gated=True),
                    ctx.experts_params(T * k, T * k, E, F, K, bits, group), ctx.moe_combine_params(T, K, k, T * k))

    def step(self, wait=False):
        c, b = self.ctx, self.b
        calls = [lambda: c.moe_route(self.prm[0], b["logits"], None, b["ids"], b["weights"], b["order"], b["pos"], b["offsets"]),
                 lambda: c.qmatmul_experts(self.prm[1], b["x"], b["order"], b["offsets"], *b["up"], None, b["h"]),
                 lambda: c.qmatmul_experts(self.prm[2], b["h"], None, b["offsets"], *b["down"], None, b["y"]),
                 lambda: c.moe_combine(self.prm[3], b["y"], b["pos"], b["weights"], b["res"], b["out"])]
        for call in calls:
            call()
            if wait:
                c.sync()

    def check(self, oracle, got):
        """Against 64 bits, with what the calls store between them rounded as they round it."""
        T, E, k, K, F, bits, group = self.shape
        values = lambda w, n, d: oracle.from_bf16(oracle.dequantize(*w, d, bits, group, oracle.BF16)).reshape(E, n, d).astype(np.float64)  # noqa: E731
        up, down, x = values(self.up, 2 * F, K), values(self.down, K, F), oracle.from_bf16(self.x).astype(np.float64)
        ids, w = moe.route(self.logits, k)
        want, tol = oracle.from_bf16(self.res).astype(np.float64), np.zeros((T, K))
        for t in range(T):
            for j in range(k):
                e = ids[t, j]
                if e < 0:
                    continue
                v, s = moe.product(x[t:t + 1], up[e])
                h, dh = moe.epilogue(v, s, K, P.ACT_SILU, True)
                dh = dh + 2.0 ** -8 * (np.abs(h) + dh)
                y, s = moe.product(h, down[e])
                dy = np.abs(down[e]) @ dh[0] + (F + 2) * moe.U * s[0]
                dy = dy + 2.0 ** -8 * (np.abs(y[0]) + dy)
                want[t] += w[t, j] * y[0]
                tol[t] += w[t, j] * (dy + 60 * moe.U * np.abs(y[0])) + moe.U * (np.abs(want[t]) + np.abs(w[t, j] * y[0]))
        tol = tol + 2.0 ** -8 * (np.abs(want) + tol)
        diff = np.abs(oracle.from_bf16(got).astype(np.float64) - want)
        assert (diff <= tol).all(), (diff - tol).max()


@pytest.mark.parametrize("T,E,k,K,F,bits,group,pad", [(1, 8, 2, 256, 128, 4, 64, 0), (5, 16, 4, 512, 192, 8, 32, 2), (40, 4, 2, 256, 256, 4, 128, 7), (150, 2, 1, 128, 64, 4, 32, 0)])
def test_layer(ctx, oracle, T, E, k, K, F, bits, group, pad):
    layer = Layer(ctx, oracle, T, E, k, K, F, bits, group, pad=pad)
    layer.step(wait=True)
    got = layer.b["out"].to_host()
    layer.check(oracle, got)
    layer.b["out"].from_host(np.zeros_like(got))
    layer.step()                       # one launch behind the other, as they overlap
    np.testing.assert_array_equal(layer.b["out"].to_host(), got)
    ctx.graph_begin()
    layer.step()
    layer.step()
    g = ctx.graph_end()
    for _ in range(3):
        layer.b["out"].from_host(np.zeros_like(got))
        ctx.graph_launch(g)
        np.testing.assert_array_equal(layer.b["out"].to_host(), got)
    ctx.graph_destroy(g)


@pytest.mark.parametrize("T", [4, 300])
def test_two_contexts_at_once(plugin, oracle, T):
    """Each with its own stream and workspaces, from two threads: the bits of either alone."""
    ctxs = [plugin.context(0) for _ in range(2)]
    layers = [Layer(c, oracle, T, 8, 4, 512, 256, seed=i) for i, c in enumerate(ctxs)]
    want = []
    for layer in layers:
        layer.step()
        want.append(layer.b["out"].to_host())
    got = [[], []]

    def work(i):
        for _ in range(20):
            for _ in range(3):
                layers[i].step()
            got[i].append(layers[i].b["out"].to_host())
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        assert len(got[i]) == 20
        for g in got[i]:
            np.testing.assert_array_equal(g, want[i])
    for c in ctxs:
        c.close()


def test_chained_with_the_rest(ctx, oracle):
    """Behind a product with its residual and ahead of the norm of the next block, one after the other without a wait: the bits of calls that wait."""
    T, K = 24, 256
    layer = Layer(ctx, oracle, T, 4, 2, K, 128)
    w = [ctx.upload(a) for a in oracle.make_layer(K, K, 4, 64, oracle.BF16, config_id=53, scale_range=(0.0005, 0.005))]
    attn, stream, normed = ctx.upload(oracle.make_x(T, K, oracle.BF16, tag=9)), ctx.upload(layer.res), ctx.empty((T, K), np.uint16)
    epi = ctx.qmm_epi_params(T, K, K, 4, 64)
    norm = ctx.block_norm_params(T, K, pre=P.NORM_RMS)
    weight = ctx.upload(np.full(K, 1.5, np.float32))

    def step(wait):
        done = ctx.sync if wait else (lambda: None)
        stream.from_host(layer.res)
        ctx.qmatmul_epi(epi, attn, *w, None, stream, stream)
        done()
        ctx.block_norm(norm, None, None, stream, None, None, weight, None, None, layer.b["x"])
        done()
        layer.b["res"], keep = stream, layer.b["res"]
        layer.step(wait)
        layer.b["res"] = keep
        ctx.block_norm(norm, None, None, layer.b["out"], None, None, weight, None, None, normed)
        return normed.to_host()
    want = step(True)
    for _ in range(5):
        np.testing.assert_array_equal(step(False), want)


def test_the_kernels_that_take_a_layer(ctx, oracle):
    """Few rows an expert: the decode kernel; many: the GEMM, pairs of CTAs where they are many more and single ones would have several tiles each."""
    for T, E, k, F, first in ((1, 4, 2, 512, "qmv_experts<4>"), (150, 4, 2, 512, "qmm_experts<4>"), (600, 4, 2, 512, "qmm_experts<4>"), (300, 16, 8, 1024, "qmm_experts<4,pairs>")):
        layer = Layer(ctx, oracle, T, E, k, 512, F)
        layer.step()
        ctx.qmatmul_experts(layer.prm[1], layer.b["x"], layer.b["order"], layer.b["offsets"], *layer.b["up"], None, layer.b["h"])
        assert ctx.last_kernel() == first

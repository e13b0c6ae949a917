"""Performance cases of the feed-forward layer of experts on affine quantized weights, and of a product with its epilogue.

Every case is a dict of plain values.  `op` says which calls a pass consists of:
  epi       a quantized product with bias, activation and residual in its epilogue (qmatmul_epi)
  route     the router: the best experts of every token, their weights, and the tokens sorted by expert (moe_route)
  experts   products grouped by expert, groups of any size (qmatmul_experts): `dir` "up" gathers the tokens' rows and multiplies
            act(gate) with up, "down" takes rows sorted by expert as they lie
  combine   the weighted sum of a token's expert outputs and the residual (moe_combine)
  layer     all of a layer of experts, recorded once and replayed: route, up, down, combine
Weights are 4 or 8 bits with bf16 scales and biases per group along K.  With `own` the passes are the calls of the framework;
without, the same operators in elementary operations on the same tensors.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPI = {"op": "epi", "bits": 4, "group": 64, "act": "none", "bias": True, "res": "bf16", "out": "bf16"}
EXPERTS = {"op": "experts", "bits": 4, "group": 64, "E": 64, "k": 8, "pad": 0.0, "bias": False, "out": "bf16"}
UP = dict(EXPERTS, dir="up", act="silu")
DOWN = dict(EXPERTS, dir="down", act="none")
ROUTE = {"op": "route", "E": 64, "k": 8, "score": "softmax", "renorm": True, "logits": "f32", "bias": False, "pad": 0.0}
COMBINE = {"op": "combine", "k": 8, "y": "bf16", "out": "bf16", "pad": 0.0}


def listed():
    return [
        # one token through a down projection, its sum with the residual stream
        dict(EPI, name="epi_m1", M=1, K=11008, N=4096, bias=False),
        # a prompt of 2048 tokens through an output projection with a bias, onto an fp32 residual stream
        dict(EPI, name="epi_m2048", M=2048, K=4096, N=4096, res="f32", out="f32"),
        # a prompt of no particular length through a layer of no particular width: 8 bit, activation, no residual
        dict(EPI, name="epi_ragged_m333", M=333, K=2880, N=5003, bits=8, group=32, act="gelu", res="none"),
        # the router for one token
        dict(ROUTE, name="route_m1", T=1),
        # the router for a long batch, one in twenty tokens padding, sigmoid scores with a bias that balances the experts
        dict(ROUTE, name="route_m8192", T=8192, E=256, score="sigmoid", bias=True, pad=0.05),
        # one token through the gate and up projections of its eight experts
        dict(UP, name="experts_m1", T=1, K=4096, F=1408),
        # 32 requests through the down projections: four rows an expert
        dict(DOWN, name="experts_m32", T=32, K=1408, N=4096),
        # the largest: a prompt of 2048 tokens through the gate and up projections, 256 rows an expert
        dict(UP, name="experts_m2048", T=2048, K=4096, F=1408),
        # few wide experts, three a token, 8 bit with a bias, odd sizes, some tokens padding
        dict(DOWN, name="experts_ragged_m777", T=777, E=40, k=3, K=2880, N=5003, bits=8, group=32, act="relu", bias=True, out="f32", pad=0.1),
        # sixteen requests' sums
        dict(COMBINE, name="combine_m16", T=16, N=4096),
        # a long prompt's sums onto an fp32 residual stream
        dict(COMBINE, name="combine_m4096", T=4096, N=4096, out="f32", pad=0.05),
        # a decode step at sixteen requests through a layer of experts
        dict(EXPERTS, op="layer", name="layer_m16", T=16, K=2048, F=1408, act="silu", score="softmax", renorm=True, logits="f32"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["epi", "epi", "route", "experts", "experts", "experts", "combine", "layer"])
    bits, group = rng.choice([4, 4, 8]), rng.choice([32, 64, 64, 128])
    if op == "epi":
        return dict(EPI, M=_log(rng, 1, 2048), K=128 * _log(rng, 4, 86), N=_log(rng, 64, 11008), bits=bits, group=group, bias=rng.random() < 0.5,
                    act=rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"]), res=rng.choice(["none", "bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
    if op == "route":
        E = _log(rng, 4, 512)
        score = rng.choice(["softmax", "sigmoid"])
        return dict(ROUTE, T=_log(rng, 1, 16384), E=E, k=rng.randint(1, min(8, E)), score=score, renorm=rng.random() < 0.5, logits=rng.choice(["f32", "bf16"]),
                    bias=score == "sigmoid" and rng.random() < 0.5, pad=rng.choice([0.0, 0.1]))
    E = _log(rng, 2, 128)
    k = rng.randint(1, min(8, E))
    if op == "combine":
        return dict(COMBINE, T=_log(rng, 1, 8192), k=k, N=_log(rng, 64, 8192), y=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]), pad=rng.choice([0.0, 0.1]))
    some = dict(E=E, k=k, bits=bits, group=group, pad=rng.choice([0.0, 0.0, 0.1]))
    if op == "layer":
        return dict(EXPERTS, op="layer", T=_log(rng, 1, 64), K=128 * _log(rng, 4, 32), F=128 * _log(rng, 4, 16), act=rng.choice(["silu", "gelu_tanh"]),
                    score=rng.choice(["softmax", "sigmoid"]), renorm=rng.random() < 0.5, logits=rng.choice(["f32", "bf16"]), **some)
    T, K = _log(rng, 1, 4096), 128 * _log(rng, 4, 32)
    if rng.random() < 0.5:
        return dict(UP, T=T, K=K, F=8 * _log(rng, 16, 256), act=rng.choice(["silu", "gelu", "gelu_tanh"]), **some)
    return dict(DOWN, T=T, K=K, N=_log(rng, 128, 8192), bias=rng.random() < 0.3, act=rng.choice(["none", "none", "relu"]), out=rng.choice(["bf16", "f32"]), **some)


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.4e12, w["flops"] / 1.6e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most and c.get("E", 1) * c.get("K", 1) * c.get("N", 2 * c.get("F", 1)) <= 1 << 30:
            return c


def _size(t):
    return {"bf16": 2, "f32": 4, "none": 0}[t]


def _weight_bytes(rows, K, c):
    return rows * (K * c["bits"] // 8 + 4 * K // c["group"])


def _active(c):
    """Experts that get a token, where all are equally likely."""
    return c["E"] * (1.0 - (1.0 - c["k"] / c["E"]) ** (c["T"] * (1.0 - c["pad"])))


def work(case):
    c = case
    if c["op"] == "epi":
        M, K, N = c["M"], c["K"], c["N"]
        return {"bytes": _weight_bytes(N, K, c) + M * K * 2 + M * N * (_size(c["res"]) + _size(c["out"])) + 4 * N * c["bias"], "flops": 2 * M * K * N}
    T, k = c["T"], c["k"]
    P = int(T * (1.0 - c["pad"])) * k
    if c["op"] == "route":
        return {"bytes": T * c["E"] * _size(c["logits"]) + T * k * 16 + 4 * c["E"], "flops": T * c["E"] * 8}
    if c["op"] == "combine":
        return {"bytes": P * c["N"] * _size(c["y"]) + 2 * T * c["N"] * _size(c["out"]) + 8 * T * k, "flops": 2 * P * c["N"]}
    K = c["K"]
    if c["op"] == "layer":
        F = c["F"]
        return {"bytes": int(_active(c) * (_weight_bytes(2 * F, K, c) + _weight_bytes(K, F, c))) + T * c["E"] * _size(c["logits"]) + T * k * 24
                + T * K * 6 + P * (F + K) * 4, "flops": 2 * P * K * 3 * F}
    N, n_out = (2 * c["F"], c["F"]) if c["dir"] == "up" else (c["N"], c["N"])
    x = T * K * 2 if c["dir"] == "up" else P * K * 2
    return {"bytes": int(_active(c) * (_weight_bytes(N, K, c) + 4 * N * c["bias"])) + x + P * (n_out * _size(c["out"]) + 4), "flops": 2 * P * K * N}


# ---- the operators in elementary operations ---------------------------------------------------------------------------
def _unpack(words, bits):
    """Codes of packed words, lowest bits first along K."""
    shift = torch.arange(0, 32, bits, device=words.device, dtype=torch.int32)
    return ((words[..., None] >> shift) & ((1 << bits) - 1)).flatten(-2)


def _weights(w, e=0):
    """What expert e's packed words stand for: scale * code + bias, rounded once to bf16."""
    q = _unpack(w["words"][e], w["bits"]).float().unflatten(-1, (-1, w["group"]))
    return (q * w["scales"][e].float()[..., None] + w["biases"][e].float()[..., None]).bfloat16().float().flatten(-2)


def _act(v, act):
    if act == "relu":
        return torch.where(v > 0, v, torch.zeros_like(v))
    if act == "silu":
        return v / (1.0 + torch.exp(-v))
    if act == "gelu":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    return v


def _expert(x, w, e, bias, act, gated):
    v = x.float() @ _weights(w, e).T
    if bias is not None:
        v = v + bias[e]
    if gated:
        f = v.shape[-1] // 2
        return _act(v[:, :f], act) * v[:, f:]
    return _act(v, act)


def _scores(logits, c):
    """What a token's experts are ordered by (minus infinity: not to be chosen), and in 32 bits what their weights come from."""
    v = logits.float()
    ok = v > -math.inf
    if c["score"] == "sigmoid":
        s = 1.0 / (1.0 + torch.exp(-v))
        return ok, s
    top = v.amax(-1, keepdim=True)
    p = torch.exp(torch.where(v == top, torch.zeros_like(v), v - top))
    return ok, torch.where(ok, p, torch.zeros_like(p))


def _choose(key, ok, k):
    """The k best of every row, the lower index first where two are alike; -1 for what must not be chosen."""
    key = torch.where(ok, key, torch.full_like(key, -math.inf))
    ids = torch.sort(key, dim=-1, descending=True, stable=True).indices[:, :k]
    return torch.where(ok.gather(1, ids), ids, torch.full_like(ids, -1))


def _route(logits, bias, c):
    ok, s = _scores(logits, c)
    key = logits if bias is None else 1.0 / (1.0 + torch.exp(-logits.double())) + bias.double()  # (next to a border the 32nd bit would decide)
    ids = _choose(key, ok, c["k"])
    got = ids >= 0
    w = torch.where(got, s.gather(1, ids.clamp(min=0)), torch.zeros_like(s[:, :1]))
    if c["renorm"]:
        total = w.sum(-1, keepdim=True)
    else:
        total = s.sum(-1, keepdim=True) if c["score"] == "softmax" else torch.ones_like(w[:, :1])
    return ids, torch.where(total > 0, w / total, torch.zeros_like(w))


def _sort(ids, E):
    """(order, pos, offsets): pairs (token, slot) by expert, where each pair went (-1: nowhere), and where each expert's begin."""
    flat = ids.flatten()
    n = torch.zeros(E + 1, dtype=torch.int64, device=ids.device).scatter_add_(0, torch.where(flat < 0, E, flat), torch.ones_like(flat, dtype=torch.int64))
    offsets = torch.cat((torch.zeros_like(n[:1]), n[:E].cumsum(0)))
    by = torch.sort(torch.where(flat < 0, E, flat), stable=True).indices
    rank = torch.arange(flat.numel(), device=ids.device)
    order = torch.where(rank < offsets[E], by, torch.zeros_like(by))
    pos = torch.empty_like(rank).scatter_(0, by, torch.where(rank < offsets[E], rank, torch.full_like(rank, -1)))
    return order.int(), pos.int().view_as(ids), offsets.int()


def _combine(y, pos, weights, res):
    v = y.float()[pos.clamp(min=0).long()] * weights[..., None]
    return torch.where(pos[..., None] >= 0, v, torch.zeros_like(v)).sum(1) + res.float()


# ---- inputs -----------------------------------------------------------------------------------------------------------
class _State:
    """Tensors, and where the framework's calls are made its handles to them."""

    def __init__(self, case, seed):
        self.case, self.handles, self.held, self.graph = case, {}, {}, None
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, dtype=torch.float32, std=1.0):
        return torch.randn(shape, generator=self.gen, device="cuda").mul_(std).to(dtype)

    def weights(self, E, N, K):
        """E experts' trained weights in the format: least squares is not needed, smallest and largest of a group are met."""
        bits, group = self.case["bits"], self.case["group"]
        w = {"bits": bits, "group": group, "E": E, "N": N, "K": K, "words": torch.empty((E, N, K * bits // 32), dtype=torch.int32, device="cuda"),
             "scales": torch.empty((E, N, K // group), dtype=torch.bfloat16, device="cuda"), "biases": torch.empty((E, N, K // group), dtype=torch.bfloat16, device="cuda")}
        shift = torch.arange(0, 32, bits, device="cuda")
        step = max(1, (1 << 25) // K)
        for e in range(E):
            for i in range(0, N, step):
                v = self.normal((min(step, N - i), K // group, group), std=1.0 / math.sqrt(K))
                lo = v.amin(-1)
                s = ((v.amax(-1) - lo) / ((1 << bits) - 1)).bfloat16()
                q = ((v - lo[..., None]) / s.float()[..., None]).round_().clamp_(0, (1 << bits) - 1).to(torch.int64).reshape(v.shape[0], -1, 32 // bits)
                w["words"][e, i:i + step] = (q << shift).sum(-1).to(torch.int32)
                w["scales"][e, i:i + step], w["biases"][e, i:i + step] = s, lo.bfloat16()
        return w

    def logits(self, dtype):
        """Some experts are liked better than others; a token of padding likes none."""
        c = self.case
        v = self.normal((c["T"], c["E"])) + self.normal((1, c["E"]), std=0.3)
        v[torch.rand(c["T"], generator=self.gen, device="cuda") < c["pad"]] = -math.inf
        return v.to(dtype)

    def routing(self):
        """A router's answer: what the products and the sums that follow it have in hand."""
        c = self.case
        ids, weights = _route(self.logits(torch.float32), None, dict(c, score="softmax", renorm=True))
        return (*_sort(ids, c["E"]), weights)

    def handle(self, t):
        if t is None:
            return None
        h = self.handles.get(t.data_ptr())
        if h is None:
            h = self.handles[t.data_ptr()] = _ctx().wrap(t.data_ptr(), t.numel() * t.element_size())
            self.held[t.data_ptr()] = t
        return h

    def __del__(self):
        if self.graph is not None:
            _ctx().graph_destroy(self.graph)
        for h in self.handles.values():
            h.free()


_context = None


def _ctx():
    """The process's one context, as a program has."""
    global _context
    if _context is None:
        import mlx_b200
        _context = mlx_b200.Plugin().context(0)
    return _context


def _empty(shape, dtype):
    return torch.zeros(shape, dtype=dtype, device="cuda")


def _inputs(case, seed):
    st = _State(case, seed)
    c = case
    if c["op"] == "epi":
        st.w = st.weights(1, c["N"], c["K"])
        st.x = st.normal((c["M"], c["K"]), torch.bfloat16)
        st.bias = st.normal((1, c["N"]), std=0.3) if c["bias"] else None
        st.res = None if c["res"] == "none" else st.normal((c["M"], c["N"]), DTYPES[c["res"]], 2.0)
        st.y = _empty((c["M"], c["N"]), DTYPES[c["out"]])
        return st
    T, k, E = c["T"], c["k"], c.get("E", 16)
    st.case = c = dict(c, E=E)
    if c["op"] in ("route", "layer"):
        st.logits_in = st.logits(DTYPES[c["logits"]])
        st.route_bias = st.normal((E,), std=0.05) if c["bias"] else None
        st.ids, st.weights_out = _empty((T, k), torch.int32), _empty((T, k), torch.float32)
        st.order, st.pos, st.offsets = _empty((T * k,), torch.int32), _empty((T, k), torch.int32), _empty((E + 1,), torch.int32)
    if c["op"] == "layer":
        K, F = c["K"], c["F"]
        st.up, st.down = st.weights(E, 2 * F, K), st.weights(E, K, F)
        st.x, st.res = st.normal((T, K), torch.bfloat16), st.normal((T, K), torch.bfloat16, 2.0)
        st.h, st.y, st.out = _empty((T * k, F), torch.bfloat16), _empty((T * k, K), torch.bfloat16), _empty((T, K), torch.bfloat16)
    if c["op"] == "experts":
        st.order, st.pos, st.offsets, _ = st.routing()
        st.ends = st.offsets.tolist()  # for the plain form, which takes one expert at a time
        up = c["dir"] == "up"
        N = 2 * c["F"] if up else c["N"]
        st.w = st.weights(E, N, c["K"])
        st.bias = st.normal((E, N), std=0.3) if c["bias"] else None
        st.x = st.normal((T if up else T * k, c["K"]), torch.bfloat16)
        st.y = _empty((T * k, c["F"] if up else N), DTYPES[c["out"]])
    if c["op"] == "combine":
        st.order, st.pos, st.offsets, st.w = st.routing()
        st.y, st.res = st.normal((T * k, c["N"]), DTYPES[c["y"]]), st.normal((T, c["N"]), DTYPES[c["out"]], 2.0)
        st.out = _empty((T, c["N"]), DTYPES[c["out"]])
    return st


def prepare(case, seed):
    st = _inputs(case, seed)
    torch.cuda.synchronize()
    if own:  # the same tensors; the handles to them, and the recorded step, that a program of the framework keeps
        st.calls = _calls(st)
        if case["op"] == "layer":
            ctx = _ctx()
            for record in (False, True):
                if record:
                    ctx.graph_begin()
                for call, args in st.calls:
                    call(*args)
                if record:
                    st.graph = ctx.graph_end()
                else:
                    ctx.sync()
    return st


# ---- a pass -----------------------------------------------------------------------------------------------------------
def run(st):
    op = st.case["op"]
    if own:
        if st.graph is not None:
            _ctx().graph_launch(st.graph)
        else:
            for call, args in st.calls:
                call(*args)
        return {"epi": lambda: [st.y], "route": lambda: [st.ids, st.weights_out, st.order, st.pos, st.offsets], "experts": lambda: [st.y],
                "combine": lambda: [st.out], "layer": lambda: [st.ids, st.weights_out, st.out]}[op]()
    return {"epi": _plain_epi, "route": _plain_route, "experts": _plain_experts, "combine": _plain_combine, "layer": _plain_layer}[op](st)


def _plain_epi(st):
    v = _expert(st.x, st.w, 0, st.bias, st.case["act"], False)
    return [(v if st.res is None else v + st.res.float()).to(st.y.dtype)]


def _plain_route(st):
    ids, w = _route(st.logits_in, st.route_bias, st.case)
    return [ids.int(), w, *_sort(ids, st.case["E"])]


def _plain_experts(st):
    c, y = st.case, torch.zeros_like(st.y)
    up = c["dir"] == "up"
    for e in range(c["E"]):
        lo, hi = st.ends[e], st.ends[e + 1]
        if lo < hi:
            x = st.x[st.order[lo:hi].long() // c["k"]] if up else st.x[lo:hi]
            y[lo:hi] = _expert(x, st.w, e, st.bias, c["act"], up).to(y.dtype)
    return [y]


def _plain_combine(st):
    return [_combine(st.y, st.pos, st.w, st.res).to(st.out.dtype)]


def _plain_layer(st):
    c = st.case
    ids, w = _route(st.logits_in, st.route_bias, c)
    total = st.res.float()
    for e in range(c["E"]):  # every expert on every token: who goes where is known on the device only
        h = _expert(st.x, st.up, e, None, c["act"], True).bfloat16()
        y = _expert(h, st.down, e, None, "none", False).bfloat16().float()
        mine = ids == e
        total = total + torch.where(mine.any(-1, keepdim=True), y, torch.zeros_like(y)) * torch.where(mine, w, torch.zeros_like(w)).sum(-1, keepdim=True)
    return [ids.int(), w, total.to(st.out.dtype)]


def _code(name):
    import mlx_b200.plugin as P
    return {"bf16": P.BF16, "f32": P.F32, "none": P.ACT_NONE, "relu": P.ACT_RELU, "silu": P.ACT_SILU, "gelu": P.ACT_GELU, "gelu_tanh": P.ACT_GELU_TANH,
            "softmax": P.SCORE_SOFTMAX, "sigmoid": P.SCORE_SIGMOID}[name]


def _calls(st):
    """A pass as (function, arguments)."""
    c, ctx, H = st.case, _ctx(), st.handle

    def packed(w):
        return H(w["words"]), H(w["scales"]), H(w["biases"])

    if c["op"] == "epi":
        prm = ctx.qmm_epi_params(c["M"], c["K"], c["N"], c["bits"], c["group"], act=_code(c["act"]), r_dtype=_code(c["res"] if st.res is not None else "bf16"),
                                 y_dtype=_code(c["out"]))
        return [(ctx.qmatmul_epi, (prm, H(st.x), *packed(st.w), H(st.bias), H(st.res), H(st.y)))]
    T, k, E = c["T"], c["k"], c["E"]
    calls = []
    if c["op"] in ("route", "layer"):
        prm = ctx.moe_route_params(T, E, k, score=_code(c["score"]), renorm=c["renorm"], logits_dtype=_code(c["logits"]))
        calls.append((ctx.moe_route, (prm, H(st.logits_in), H(st.route_bias), H(st.ids), H(st.weights_out), H(st.order), H(st.pos), H(st.offsets))))
    if c["op"] == "experts":
        up = c["dir"] == "up"
        prm = ctx.experts_params(T * k, st.x.shape[0], E, c["K"], st.w["N"], c["bits"], c["group"], top_k=k, act=_code(c["act"]), gated=up, y_dtype=_code(c["out"]))
        calls.append((ctx.qmatmul_experts, (prm, H(st.x), H(st.order) if up else None, H(st.offsets), *packed(st.w), H(st.bias), H(st.y))))
    if c["op"] == "layer":
        K, F = c["K"], c["F"]
        prm = ctx.experts_params(T * k, T, E, K, 2 * F, c["bits"], c["group"], top_k=k, act=_code(c["act"]), gated=True)
        calls.append((ctx.qmatmul_experts, (prm, H(st.x), H(st.order), H(st.offsets), *packed(st.up), None, H(st.h))))
        prm = ctx.experts_params(T * k, T * k, E, F, K, c["bits"], c["group"])
        calls.append((ctx.qmatmul_experts, (prm, H(st.h), None, H(st.offsets), *packed(st.down), None, H(st.y))))
        prm = ctx.moe_combine_params(T, K, k, T * k)
        calls.append((ctx.moe_combine, (prm, H(st.y), H(st.pos), H(st.weights_out), H(st.res), H(st.out))))
    if c["op"] == "combine":
        prm = ctx.moe_combine_params(T, c["N"], k, T * k, y_dtype=_code(c["y"]), out_dtype=_code(c["out"]))
        calls.append((ctx.moe_combine, (prm, H(st.y), H(st.pos), H(st.w), H(st.res), H(st.out))))
    return calls


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
def _exact_weights(w, e):
    """scale * code + bias of expert e, rounded to the nearest bf16 (ties to even), as 64-bit numbers."""
    n = 32 // w["bits"]
    word = w["words"][e].long() & 0xFFFFFFFF
    q = torch.stack([(word >> (w["bits"] * i)) & ((1 << w["bits"]) - 1) for i in range(n)], -1).reshape(w["N"], -1, w["group"]).double()
    v = q * w["scales"][e].double().unsqueeze(-1) + w["biases"][e].double().unsqueeze(-1)
    step = torch.exp2((torch.frexp(v)[1] - 8).double())
    return torch.where(v == 0, v, torch.round(v / step) * step).reshape(w["N"], -1)


def _exact_act(v, act):
    if act == "relu":
        return v.clamp(min=0)
    if act == "silu":
        return v * torch.special.expit(v)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "gelu_tanh":
        return v * torch.special.expit(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v ** 3))
    return v


def _exact_expert(x, w, e, bias, act, gated):
    v = x.double() @ _exact_weights(w, e).T
    if bias is not None:
        v = v + bias[e].double()
    if not gated:
        return _exact_act(v, act)
    gate, up = v.chunk(2, -1)
    return _exact_act(gate, act) * up


def _exact_route(logits, bias, c):
    """ids, weights: one best expert after the other."""
    v = logits.double()
    key = v if bias is None else torch.special.expit(v) + bias.double()
    left = v > -math.inf
    ids = []
    for _ in range(c["k"]):
        masked = torch.where(left, key, torch.full_like(key, -math.inf))
        first = (masked == masked.amax(-1, keepdim=True)).to(torch.uint8).argmax(-1, keepdim=True)
        ids.append(torch.where(left.any(-1, keepdim=True), first, torch.full_like(first, -1)))
        left = left & (torch.arange(c["E"], device=v.device) != first)
    ids = torch.cat(ids, -1)
    if c["score"] == "sigmoid":
        s = torch.special.expit(v)
    else:
        s = torch.softmax(torch.where(v.amax(-1, keepdim=True) > -math.inf, v, torch.zeros_like(v)), -1)
    w = torch.where(ids >= 0, s.gather(-1, ids.clamp(min=0)), torch.zeros_like(s[:, :1]))
    if c["renorm"]:
        w = torch.where(w.sum(-1, keepdim=True) > 0, w / w.sum(-1, keepdim=True), torch.zeros_like(w))
    return ids, w


def exact(case, seed):
    st = _inputs(case, seed)
    c = st.case
    if c["op"] == "epi":
        v = _exact_expert(st.x, st.w, 0, st.bias, c["act"], False)
        return [v if st.res is None else v + st.res.double()]
    T, k, E = c["T"], c["k"], c["E"]
    if c["op"] == "combine":
        total = st.res.double()
        for j in range(k):
            rows = st.pos[:, j].long()
            total = total + torch.where(rows[:, None] >= 0, st.w[:, j, None].double() * st.y.double()[rows.clamp(min=0)], torch.zeros_like(total))
        return [total]
    if c["op"] == "experts":
        y = torch.zeros(st.y.shape, dtype=torch.float64, device="cuda")
        for e in range(E):
            rows = slice(st.ends[e], st.ends[e + 1])
            if st.ends[e] < st.ends[e + 1]:
                x = st.x[torch.div(st.order[rows], k, rounding_mode="floor").long()] if c["dir"] == "up" else st.x[rows]
                y[rows] = _exact_expert(x, st.w, e, st.bias, c["act"], c["dir"] == "up")
        return [y]
    ids, w = _exact_route(st.logits_in, st.route_bias, c)
    if c["op"] == "route":
        expert = ids.flatten().cpu()
        lists = [torch.nonzero(expert == e).flatten() for e in range(E)]
        routed = torch.cat(lists)
        order, pos = torch.zeros(T * k, dtype=torch.int32), torch.full((T * k,), -1, dtype=torch.int32)
        order[:routed.numel()] = routed.int()
        pos[routed] = torch.arange(routed.numel(), dtype=torch.int32)
        offsets = torch.tensor([0] + [x.numel() for x in lists], dtype=torch.int64).cumsum(0).int()
        return [ids.int(), w, order.cuda(), pos.view(T, k).cuda(), offsets.cuda()]
    total = st.res.double()
    for e in range(E):  # what the calls store between them is rounded by definition
        t, j = torch.nonzero(ids == e, as_tuple=True)
        if t.numel():
            h = _exact_expert(st.x[t], st.up, e, None, c["act"], True).bfloat16()
            y = _exact_expert(h, st.down, e, None, "none", False).bfloat16().double()
            total.index_add_(0, t, w[t, j, None] * y)
    return [ids.int(), w, total]

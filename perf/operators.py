"""Performance cases of the microscaled 4-bit operators and of the norms around a block: what a program that serves a model asks of them.

Every case is a dict of plain values.  `op` says which calls a pass consists of:
  linear    per layer: the activations into the microscaled format (mx4_quantize), the product with the layer's weights (mx4_matmul)
  requant   weights into the format and back (mx4_quantize, mx4_dequantize)
  norm      the norm after a block, its gate, the residual sum and the norm before the next block (block_norm)
  chain     a decode step through several blocks: block_norm into the format, gate|up product, mul_rms_norm, mx4_quantize, down product
`fmt` is "e8m0" (blocks of 32, scales that are powers of two) or "e4m3" (blocks of 16, 8-bit floating scales and a factor per tensor).
With `own` the passes are the calls of the framework; without, the same operators in elementary operations on the same tensors.
"""
import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
BLOCK = {"e8m0": 32, "e4m3": 16}
LINEAR = {"op": "linear", "fmt": "e8m0", "out": "bf16", "layers": 1}
NORM = {"op": "norm", "post": "rms", "pre": "rms", "gate": "channel", "act": "none", "x": "bf16", "res": "bf16", "out": "bf16"}


def listed():
    return [
        # one small layer, one row: the latency of two calls
        dict(LINEAR, name="small_call", M=1, K=1024, N=1024),
        # one token through the gate projections of eight decoder layers
        dict(LINEAR, name="decode_m1", M=1, K=4096, N=11008, layers=8),
        # a large output layer at sixteen requests, fp32 logits
        dict(LINEAR, name="decode_m16", M=16, K=8192, N=28672, fmt="e4m3", out="f32"),
        # short prompts or many requests at once
        dict(LINEAR, name="short_prefill_m48", M=48, K=4096, N=11008, layers=4),
        # prefill of 2048 tokens through a square projection
        dict(LINEAR, name="prefill_m2048", M=2048, K=4096, N=4096),
        # the largest: a long prompt through a wide layer, the finer scales
        dict(LINEAR, name="prefill_m4096_wide", M=4096, K=8192, N=28672, fmt="e4m3"),
        # a prompt of no particular length on a layer of no particular width
        dict(LINEAR, name="prefill_ragged_m777", M=777, K=2880, N=5003, layers=2, fmt="e4m3"),
        # a layer's fp32 weights on their way into the format, and expanded to bf16
        dict(op="requant", name="requant_e8m0", K=4096, N=11008, fmt="e8m0", x="f32", out="bf16"),
        # bf16 weights of odd height, the finer scales, expanded to fp32
        dict(op="requant", name="requant_ragged_e4m3", K=2880, N=5003, fmt="e4m3", x="bf16", out="f32"),
        # eight decoded tokens between two blocks
        dict(NORM, name="norm_m8", M=8, K=4096),
        # a prompt of 2048 tokens: layer norms, a gate per token and channel, fp32 residual stream
        dict(NORM, name="norm_m2048", M=2048, K=4096, post="layer", pre="layer", gate="row", act="sigmoid", res="f32"),
        # one decode step at eight requests through four blocks, recorded once and replayed
        dict(op="chain", name="decode_chain_m8", M=8, K=4096, N=11008, layers=4, fmt="e8m0"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _draw(rng):
    op = rng.choice(["linear", "linear", "linear", "prefill", "prefill", "requant", "norm", "norm", "chain"])
    fmt = rng.choice(["e8m0", "e4m3"])
    if op == "linear":   # decode and short prompts
        return dict(LINEAR, M=_log(rng, 1, 128), K=32 * _log(rng, 8, 512), N=_log(rng, 64, 28672), layers=rng.randint(1, 6), fmt=fmt,
                    out=rng.choice(["bf16", "bf16", "f32"]))
    if op == "prefill":
        return dict(LINEAR, M=_log(rng, 129, 4096), K=32 * _log(rng, 16, 344), N=_log(rng, 256, 28672), layers=rng.randint(1, 2), fmt=fmt,
                    out=rng.choice(["bf16", "bf16", "f32"]))
    if op == "requant":
        return dict(op="requant", K=32 * _log(rng, 8, 344), N=_log(rng, 64, 28672), fmt=fmt, x=rng.choice(["f32", "bf16"]), out=rng.choice(["f32", "bf16"]))
    if op == "norm":
        gate = rng.choice(["none", "channel", "row"])
        return dict(NORM, M=_log(rng, 1, 8192), K=rng.choice([8, 1]) * _log(rng, 64, 1400), post=rng.choice(["none", "rms", "layer"]),
                    pre=rng.choice(["none", "rms", "layer"]), gate=gate, act="none" if gate == "none" else rng.choice(["none", "sigmoid", "tanh"]),
                    x=rng.choice(["bf16", "bf16", "f32"]), res=rng.choice(["bf16", "f32"]), out=rng.choice(["bf16", "f32"]))
    return dict(op="chain", M=_log(rng, 1, 64), K=32 * _log(rng, 32, 128), N=32 * _log(rng, 64, 344), layers=rng.randint(1, 4), fmt=fmt)


def _cost(case):
    w = work(case)
    return max(w["bytes"] / 6.4e12, w["flops"] / 1.6e15)


def draw(rng):
    most = max(_cost(c) for c in listed())
    while True:
        c = _draw(rng)
        if _cost(c) <= most:
            return c


def _size(t):
    return 2 if t == "bf16" else 4


def _operand_bytes(rows, K, fmt):
    return rows * (K // 2 + K // BLOCK[fmt])


def work(case):
    M, K, N, fmt = case.get("M"), case["K"], case.get("N"), case.get("fmt")
    if case["op"] == "requant":  # weights in, codes and scales out; and those in, weights out
        return {"bytes": N * K * (_size(case["x"]) + _size(case["out"])) + 2 * _operand_bytes(N, K, fmt), "flops": 8 * N * K}
    if case["op"] == "norm":
        gate = {"none": 0, "channel": K, "row": M * K}[case["gate"]] * _size(case["x"])
        return {"bytes": M * K * (_size(case["x"]) + 2 * _size(case["res"]) + _size(case["out"])) + gate + 4 * K * 4, "flops": 16 * M * K}
    if case["op"] == "chain":
        n = case["layers"]
        rows = M * K * 2 * 5 + M * N * 2 * 3  # r in and out, codes (a byte and a half), h; gate|up, their product's codes
        return {"bytes": n * (_operand_bytes(2 * N, K, fmt) + _operand_bytes(K, N, fmt) + rows), "flops": n * 2 * M * 3 * N * K}
    n = case["layers"]
    return {"bytes": n * (_operand_bytes(N, K, fmt) + M * K * 2 + M * N * _size(case["out"])), "flops": n * 2 * M * N * K}


# ---- the operators in elementary operations ---------------------------------------------------------------------------
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _tile_index(rows, nb, device):
    """Where the scale of (row, block) lies: tiles of 128 rows x 4 blocks, 512 bytes."""
    r = torch.arange(rows, device=device)[:, None]
    b = torch.arange(nb, device=device)[None, :]
    return ((r // 128) * ((nb + 3) // 4) + b // 4) * 512 + (r % 32) * 16 + (r // 32 % 4) * 4 + b % 4


def scale_bytes(rows, K, fmt):
    return (rows + 127) // 128 * ((K // BLOCK[fmt] + 3) // 4) * 512


def _quantize(v, fmt, pre):
    """Codes (0..15, a byte each) and scale bytes [rows, blocks] of v [rows, K]."""
    rows, K = v.shape
    u = (v.float() * pre).reshape(rows, -1, BLOCK[fmt])
    amax = u.abs().amax(-1)
    nan = torch.isnan(amax)
    if fmt == "e8m0":  # the largest power of two that the largest value is at least four times of
        field = (amax.nan_to_num(0.0, posinf=3e38).view(torch.int32) >> 23).clamp(max=254)
        byte = (field - 2).clamp(min=0)
        t = u * torch.ldexp(torch.ones_like(amax), 127 - byte)[..., None]
        byte = torch.where(nan, 255, byte).to(torch.uint8)
    else:
        s = (amax / 6.0).clamp(max=448.0).to(torch.float8_e4m3fn)
        byte = torch.where(nan, torch.full_like(s.view(torch.uint8), 0x7F), s.view(torch.uint8))
        f = s.float()[..., None]
        t = torch.where(f > 0, u / f, torch.zeros_like(u))
    a = t.abs()
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)).to(torch.uint8)
    code = code + 8 * (t < 0).to(torch.uint8)
    return code.reshape(rows, K), byte


def _scale_value(byte, fmt):
    if fmt == "e4m3":
        return byte.view(torch.float8_e4m3fn).float()
    e = byte.to(torch.int32)  # 2^(e - 127); the smallest is half of the smallest normal number
    s = torch.where(e > 0, e << 23, 1 << 22).view(torch.float32)
    return torch.where(e == 255, torch.full_like(s, float("nan")), s)


def _expand(code, byte, fmt, post):
    """The values that codes and scale bytes stand for, times post."""
    rows, K = code.shape
    table = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=code.device)
    v = table[code.to(torch.int32)].reshape(rows, -1, BLOCK[fmt]) * _scale_value(byte, fmt)[..., None]
    return v.reshape(rows, K) * post


def _unpack(words, scales, rows, K, fmt):
    """Codes and scale bytes out of packed words [rows, K/8] and scales in tiles."""
    shift = torch.arange(0, 32, 4, device=words.device, dtype=torch.int32)
    code = ((words[..., None] >> shift) & 15).reshape(rows, K).to(torch.uint8)
    return code, scales[_tile_index(rows, K // BLOCK[fmt], scales.device)]


def _pack(code, byte):
    """The reverse: packed words and tiles, zeros where a tile has no block."""
    rows, K = code.shape
    c = code.reshape(rows, K // 8, 8).to(torch.int64)
    words = (c << torch.arange(0, 32, 4, device=code.device)).sum(-1).to(torch.int32)
    nb = byte.shape[1]
    tiles = torch.zeros((rows + 127) // 128 * ((nb + 3) // 4) * 512, dtype=torch.uint8, device=code.device)
    tiles[_tile_index(rows, nb, code.device)] = byte
    return words, tiles


def _norm(v, kind, weight, bias):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(-1, keepdim=True)
    v = v * (v.square().mean(-1, keepdim=True) + EPS).rsqrt() * weight
    return v + bias if kind == "layer" else v


def _act(g, act):
    return torch.sigmoid(g) if act == "sigmoid" else torch.tanh(g) if act == "tanh" else g


def _block_norm(h, gate, r, w, case):
    """(new residual stream, input of the next block) from a block's output h and the stream r."""
    b = _norm(h.float(), case["post"], w["post"], w["post_bias"])
    if gate is not None:
        b = b * _act(gate.float(), case["act"])
    new = (case["res_scale"] * r.float() + case["branch_scale"] * b).to(r.dtype)
    return new, _norm(new.float(), case["pre"], w["pre"], w["pre_bias"])


def _product(code, byte, layer, fmt, alpha, out):
    x = _expand(code, byte, fmt, 1.0)
    w = _expand(*_unpack(layer["words"], layer["scales"], layer["N"], layer["K"], fmt), fmt, 1.0)
    return (x @ w.T * alpha).to(DTYPES[out])


# ---- inputs -----------------------------------------------------------------------------------------------------------
class _State:
    """Tensors, and where the framework's calls are made its handles to them."""

    def __init__(self, case, seed):
        self.case, self.handles, self.graph, self.held = case, {}, None, {}
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, shape, dtype=torch.float32, std=1.0, mean=0.0):
        return torch.randn(shape, generator=self.gen, device="cuda").mul_(std).add_(mean).to(dtype)

    def weights(self, N, K):
        """Trained weights' values in the format, in pieces that leave room for the other states."""
        fmt = self.case["fmt"]
        # e4m3: the tensor's factor brings the largest scale to the top of its range (the largest of a normal sample lies near 6 of its widths)
        factor = 1.0 if fmt == "e8m0" else float(torch.tensor(0.02 * 6.0 / (6.0 * 448.0)))
        words = torch.empty((N, K // 8), dtype=torch.int32, device="cuda")
        byte = torch.empty((N, K // BLOCK[fmt]), dtype=torch.uint8, device="cuda")
        step = max(1, (1 << 26) // K)
        for i in range(0, N, step):
            code, b = _quantize(self.normal((min(step, N - i), K), std=0.02), fmt, _f32(1.0 / factor))
            words[i:i + step], byte[i:i + step] = _pack(code, b)[0], b
        tiles = torch.zeros(scale_bytes(N, K, fmt), dtype=torch.uint8, device="cuda")
        tiles[_tile_index(N, K // BLOCK[fmt], "cuda")] = byte
        return {"words": words, "scales": tiles, "N": N, "K": K, "factor": factor}

    def codes(self, rows, K):
        """Room for activations in the format."""
        return {"words": torch.empty((rows, K // 8), dtype=torch.int32, device="cuda"),
                "scales": torch.empty(scale_bytes(rows, K, self.case["fmt"]), dtype=torch.uint8, device="cuda")}

    def handle(self, t):
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


X_FACTOR = float(torch.tensor(5.0 / (6.0 * 448.0)))  # e4m3 activations: the factor that a calibration leaves


def _f32(v):
    """A host factor as the 32-bit argument that it becomes."""
    return float(torch.tensor(v, dtype=torch.float32))


def _x_factor(fmt):
    return 1.0 if fmt == "e8m0" else X_FACTOR


def prepare(case, seed):
    st = _State(case, seed)
    {"linear": _prepare_linear, "requant": _prepare_requant, "norm": _prepare_norm, "chain": _prepare_chain}[case["op"]](st)
    torch.cuda.synchronize()
    if own:  # the same tensors; the handles to them, and the recorded step, that a program of the framework keeps
        if case["op"] == "chain":
            _own_chain(st)
            _ctx().sync()
            _ctx().graph_begin()
            _own_chain(st)
            st.graph = _ctx().graph_end()
        else:
            st.calls = {"linear": _calls_linear, "requant": _calls_requant, "norm": _calls_norm}[case["op"]](st)
    return st


def _prepare_linear(st):
    c = st.case
    st.x = [st.normal((c["M"], c["K"]), torch.bfloat16) for _ in range(c["layers"])]
    st.layers = [st.weights(c["N"], c["K"]) for _ in range(c["layers"])]
    st.q = [st.codes(c["M"], c["K"]) for _ in range(c["layers"])]
    st.y = [torch.empty((c["M"], c["N"]), dtype=DTYPES[c["out"]], device="cuda") for _ in range(c["layers"])]


def _prepare_requant(st):
    c = st.case
    st.src = st.normal((c["N"], c["K"]), DTYPES[c["x"]], 0.02)
    st.factor = 1.0 if c["fmt"] == "e8m0" else float(torch.tensor(0.02 / 448.0))
    st.q = st.codes(c["N"], c["K"])
    st.back = torch.empty((c["N"], c["K"]), dtype=DTYPES[c["out"]], device="cuda")


def _norm_weights(st, K):
    return {"post": st.normal((K,), std=0.1, mean=1.0), "post_bias": st.normal((K,), std=0.1), "pre": st.normal((K,), std=0.1, mean=1.0),
            "pre_bias": st.normal((K,), std=0.1)}


def _prepare_norm(st):
    c = st.case
    M, K, x, res = c["M"], c["K"], DTYPES[c["x"]], DTYPES[c["res"]]
    st.form = dict(c, res_scale=1.0, branch_scale=0.5)
    st.h, st.r = st.normal((M, K), x, 0.7, 0.1), st.normal((M, K), res, 2.0)
    st.gate = None if c["gate"] == "none" else st.normal((M if c["gate"] == "row" else 1, K), x)
    st.w = _norm_weights(st, K)
    st.new, st.out = torch.empty((M, K), dtype=res, device="cuda"), torch.empty((M, K), dtype=DTYPES[c["out"]], device="cuda")


def _prepare_chain(st):
    c = st.case
    M, d, f = c["M"], c["K"], c["N"]
    st.form = dict(post="rms", pre="rms", act="none", res_scale=1.0, branch_scale=0.5)
    st.h, st.r = st.normal((M, d), torch.bfloat16), st.normal((M, d), torch.bfloat16, 2.0)
    bf16 = lambda w: torch.empty((M, w), dtype=torch.bfloat16, device="cuda")  # noqa: E731
    st.blocks = [{"gateup": st.weights(2 * f, d), "down": st.weights(d, f), "gate": st.normal((1, d), torch.bfloat16), "w": _norm_weights(st, d), "new": bf16(d),
                  "x": st.codes(M, d), "gu": bf16(2 * f), "m": bf16(f), "mq": st.codes(M, f), "h": bf16(d)} for _ in range(c["layers"])]


# ---- a pass -----------------------------------------------------------------------------------------------------------
def run(st):
    if own:
        if st.graph is not None:
            _ctx().graph_launch(st.graph)
            return [t for b in st.blocks for t in (b["new"], b["h"])]
        for call, args in st.calls:
            call(*args)
        return {"linear": lambda: st.y, "requant": lambda: [st.back], "norm": lambda: [st.new, st.out]}[st.case["op"]]()
    return {"linear": _plain_linear, "requant": _plain_requant, "norm": _plain_norm, "chain": _plain_chain}[st.case["op"]](st)


def _plain_linear(st):
    c, fx = st.case, _x_factor(st.case["fmt"])
    return [_product(*_quantize(x, c["fmt"], _f32(1.0 / fx)), w, c["fmt"], _f32(fx * w["factor"]), c["out"])
            for x, w in zip(st.x, st.layers)]


def _plain_requant(st):
    c = st.case
    return [_expand(*_quantize(st.src, c["fmt"], _f32(1.0 / st.factor)), c["fmt"], st.factor).to(DTYPES[c["out"]])]


def _plain_norm(st):
    new, out = _block_norm(st.h, st.gate, st.r, st.w, st.form)
    return [new, out.to(st.out.dtype)]


def _plain_chain(st):
    fmt = st.case["fmt"]
    fx = _x_factor(fmt)
    pre, h, r, got = _f32(1.0 / fx), st.h, st.r, []
    for b in st.blocks:
        r, n = _block_norm(h, b["gate"], r, b["w"], st.form)
        gu = _product(*_quantize(n.bfloat16(), fmt, pre), b["gateup"], fmt, _f32(fx * b["gateup"]["factor"]), "bf16")
        f = b["down"]["K"]
        m = (gu[:, :f].float() * gu[:, f:].float()).bfloat16().float()
        m = (m * (m.square().mean(-1, keepdim=True) + EPS).rsqrt()).bfloat16()
        h = _product(*_quantize(m, fmt, pre), b["down"], fmt, _f32(fx * b["down"]["factor"]), "bf16")
        got += [r, h]
    return got


def _codes(name):
    import mlx_b200.plugin as P
    return {"e8m0": P.MX4_E8M0, "e4m3": P.MX4_E4M3, "bf16": P.BF16, "f32": P.F32, "none": 0, "rms": P.NORM_RMS, "layer": P.NORM_LAYER,
            "sigmoid": P.GATE_SIGMOID, "tanh": P.GATE_TANH}[name]


def _calls_linear(st):
    c, ctx, calls = st.case, _ctx(), []
    fmt, fx = _codes(c["fmt"]), _x_factor(c["fmt"])
    for x, w, q, y in zip(st.x, st.layers, st.q, st.y):
        hq, hs = st.handle(q["words"]), st.handle(q["scales"])
        calls.append((ctx.mx4_quantize, (st.handle(x), hq, hs, c["M"], c["K"], fmt, _codes("bf16"), 1.0 / fx)))
        calls.append((ctx.mx4_matmul, (hq, hs, st.handle(w["words"]), st.handle(w["scales"]), st.handle(y), c["M"], c["K"], c["N"], fmt, _codes(c["out"]),
                                       fx * w["factor"])))
    return calls


def _calls_requant(st):
    c, ctx = st.case, _ctx()
    hq, hs, fmt = st.handle(st.q["words"]), st.handle(st.q["scales"]), _codes(c["fmt"])
    return [(ctx.mx4_quantize, (st.handle(st.src), hq, hs, c["N"], c["K"], fmt, _codes(c["x"]), 1.0 / st.factor)),
            (ctx.mx4_dequantize, (hq, hs, st.handle(st.back), c["N"], c["K"], fmt, _codes(c["out"]), st.factor))]


def _norm_call(st, ctx, h, gate, r, w, form, new, out, out_scales=None, **more):
    """One block_norm as (function, arguments)."""
    H = st.handle
    rows, dim = h.shape
    prm = ctx.block_norm_params(rows, dim, post=_codes(form["post"]), pre=_codes(form["pre"]), gate_act=_codes(form["act"]),
                                gate_rows=0 if gate is None or gate.shape[0] == 1 else 1, eps=EPS, res_scale=form["res_scale"],
                                branch_scale=form["branch_scale"], **more)
    affine = lambda kind, name: (None if kind == "none" else H(w[name]), H(w[name + "_bias"]) if kind == "layer" else None)  # noqa: E731
    return ctx.block_norm, (prm, H(h), None if gate is None else H(gate), H(r), *affine(form["post"], "post"), *affine(form["pre"], "pre"), H(new), H(out),
                            None if out_scales is None else H(out_scales))


def _calls_norm(st):
    c = st.case
    return [_norm_call(st, _ctx(), st.h, st.gate, st.r, st.w, st.form, st.new, st.out, x_dtype=_codes(c["x"]), r_dtype=_codes(c["res"]), out_dtype=_codes(c["out"]))]


def _own_chain(st):
    c, ctx, H = st.case, _ctx(), st.handle
    M, d, f, fx = c["M"], c["K"], c["N"], _x_factor(c["fmt"])
    bf, fmt = _codes("bf16"), _codes(c["fmt"])
    h, r = st.h, st.r
    for b in st.blocks:
        call, args = _norm_call(st, ctx, h, b["gate"], r, b["w"], st.form, b["new"], b["x"]["words"], b["x"]["scales"], x_dtype=bf, r_dtype=bf, out_dtype=bf,
                                out_format=fmt, out_pre=1.0 / fx)
        call(*args)
        g, w = b["gateup"], b["down"]
        ctx.mx4_matmul(H(b["x"]["words"]), H(b["x"]["scales"]), H(g["words"]), H(g["scales"]), H(b["gu"]), M, d, 2 * f, fmt, bf, fx * g["factor"])
        ctx.mul_rms_norm(H(b["gu"]), H(b["m"]), M, f, 2 * f, EPS)
        ctx.mx4_quantize(H(b["m"]), H(b["mq"]["words"]), H(b["mq"]["scales"]), M, f, fmt, bf, 1.0 / fx)
        ctx.mx4_matmul(H(b["mq"]["words"]), H(b["mq"]["scales"]), H(w["words"]), H(w["scales"]), H(b["h"]), M, f, d, fmt, bf, fx * w["factor"])
        h, r = b["h"], b["new"]


# ---- the definition in 64 bits ----------------------------------------------------------------------------------------
GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _exact_block_values(v, fmt, pre):
    """v [rows, K] rounded into the format, as the values that its codes and scales stand for, in 64 bits: every value goes to the nearest point of the
    grid, between two of them to the one of even number."""
    rows, K = v.shape
    u = (v.float() * torch.tensor(pre, dtype=torch.float32, device=v.device)).double().reshape(rows, K // BLOCK[fmt], BLOCK[fmt])
    top = u.abs().max(-1, keepdim=True).values
    if fmt == "e8m0":
        s = torch.exp2((torch.frexp(top)[1] - 3).clamp(min=-127).double())  # top = f * 2^e, f in [1/2, 1): e - 1 is its exponent
        s = torch.where(top > 0, s, torch.full_like(s, 2.0 ** -127))
    else:
        s = _exact_e4m3((top.float() / 6).double())
    grid = torch.tensor(GRID, dtype=torch.float64, device=v.device)
    a = torch.where(s > 0, u.abs() / torch.where(s > 0, s, torch.ones_like(s)), torch.zeros_like(u))
    hi = torch.searchsorted(grid, a.contiguous()).clamp(max=7)
    lo = (hi - 1).clamp(min=0)
    below, above = a - grid[lo], grid[hi] - a
    near = torch.where((below < above) | ((below == above) & (lo % 2 == 0)), lo, hi)
    return (torch.sign(u) * grid[near] * s).reshape(rows, K)


def _exact_e4m3(v):
    """Nearest number of four significant bits, exponents from -6 on and eighths of 2^-6 below, at most 448; ties to even."""
    step = torch.exp2((torch.frexp(v)[1] - 4).clamp(min=-9).double())
    return torch.clamp(torch.round(v / step) * step, max=448.0)


def _exact_weights(layer, fmt):
    """The weights that packed words and tiles stand for, in 64 bits."""
    N, K, bs = layer["N"], layer["K"], BLOCK[fmt]
    nb = K // bs
    grid = torch.tensor(GRID, dtype=torch.float64, device="cuda")
    byte = layer["words"].view(torch.uint8).reshape(N, K // 2)
    code = torch.stack((byte & 15, byte >> 4), -1).reshape(N, K).long()
    v = torch.where(code >= 8, -grid[code & 7], grid[code & 7])
    na = (nb + 3) // 4
    t = layer["scales"].reshape((N + 127) // 128, na, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(-1, na * 4)[:N, :nb]  # [tile, quarter, row, four, block]
    s = torch.exp2(t.double() - 127) if fmt == "e8m0" else t.contiguous().view(torch.float8_e4m3fn).double()
    return (v.reshape(N, nb, bs) * s[..., None]).reshape(N, K)


def _exact_norm(v, kind, w, b):
    if kind == "none":
        return v
    if kind == "layer":
        d = v - v.sum(-1, keepdim=True) / v.shape[-1]
        return d / torch.sqrt((d * d).sum(-1, keepdim=True) / v.shape[-1] + EPS) * w.double() + b.double()
    return v / torch.sqrt((v * v).sum(-1, keepdim=True) / v.shape[-1] + EPS) * w.double()


def _exact_block_norm(h, gate, r, w, form):
    b = _exact_norm(h.double(), form["post"], w["post"], w["post_bias"])
    if gate is not None:
        g = gate.double()
        b = b * (1 / (1 + torch.exp(-g)) if form["act"] == "sigmoid" else torch.tanh(g) if form["act"] == "tanh" else g)
    new = form["res_scale"] * r.double() + form["branch_scale"] * b
    return new, _exact_norm(new.to(r.dtype).double(), form["pre"], w["pre"], w["pre_bias"])


def exact(case, seed):
    st = _State(case, seed)
    {"linear": _prepare_linear, "requant": _prepare_requant, "norm": _prepare_norm, "chain": _prepare_chain}[case["op"]](st)
    fmt = case.get("fmt")
    fx = _x_factor(fmt) if fmt else 1.0
    if case["op"] == "requant":
        return [_exact_block_values(st.src, fmt, 1.0 / st.factor) * st.factor]
    if case["op"] == "norm":
        return list(_exact_block_norm(st.h, st.gate, st.r, st.w, st.form))
    if case["op"] == "linear":
        return [_exact_block_values(x, fmt, 1.0 / fx) @ _exact_weights(w, fmt).T * _f32(fx * w["factor"]) for x, w in zip(st.x, st.layers)]
    got, h, r = [], st.h, st.r
    for b in st.blocks:  # what the calls store between them is rounded by definition
        new, n = _exact_block_norm(h, b["gate"], r, b["w"], st.form)
        gu = _exact_block_values(n.bfloat16(), fmt, 1.0 / fx) @ _exact_weights(b["gateup"], fmt).T * _f32(fx * b["gateup"]["factor"])
        gu = gu.bfloat16().double()
        f = b["down"]["K"]
        m = (gu[:, :f] * gu[:, f:]).bfloat16().double()
        m = (m / torch.sqrt((m * m).mean(-1, keepdim=True) + EPS)).bfloat16()
        out = _exact_block_values(m, fmt, 1.0 / fx) @ _exact_weights(b["down"], fmt).T * _f32(fx * b["down"]["factor"])
        got += [new, out]
        h, r = out.bfloat16(), new.bfloat16()
    return got

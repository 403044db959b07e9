"""What is measured of the microscaled 4-bit operators and of the expert layer for few tokens.

Four operators: `quantize` (a tensor to 4-bit codes with one power-of-two scale per 32 elements, and back), `product`
(row groups times their experts' weights, both in 4 bits), `ffn` (the expert FFN on 4-bit operands, the hidden
activations re-quantised between the projections) and `few` (the whole mixture-of-experts layer for a handful of
tokens: gate, top-k, the chosen experts, weighted sum), its weights in 16 bits, in 8 bits (e4m3, one fp32 scale per
128 x 128 block) or in 4 bits.

The 4-bit format: elements e2m1 (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), two to a byte, the even column in
the low half; a block of 32 consecutive columns shares the scale 2^(s - 127), s = floor(log2(largest magnitude)) + 125
clamped at 0; elements are rounded to nearest even and saturate at 6. Scales are held in tiles of 128 rows x 4 blocks:
(..., row / 128, block / 4, row % 32, row / 32 % 4, block % 4).

The sizes are those of the repository's five configurations (hidden sizes 256, 2048, 4096, 7168, intermediate sizes
512, 1024, 2048, 14336, 8 to 256 experts, one to eight experts per token) and of its tests, or plain powers of two and
ragged numbers between them.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
RELU, GELU, SWIGLU = 0, 1, 2


# ---- cases ----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # the tokens of the smallest configuration: a call that latency decides
        dict(name="quantize-tokens-small", op="quantize", mats=1, rows=128, cols=256, type="f32"),
        # one rank's tokens of the Mixtral-shaped configuration before their experts
        dict(name="quantize-tokens", op="quantize", mats=1, rows=16384, cols=4096, type="bf16"),
        # a checkpoint's expert weights, odd row count (rows of several matrices do not fill the scale tiles)
        dict(name="quantize-weights-ragged", op="quantize", mats=13, rows=2009, cols=7168, type="f16"),
        # a few rows per expert, small sizes
        dict(name="product-small", op="product", groups=8, rows=40, n=512, k=256, type="bf16"),
        # the up projection of the Mixtral-shaped configuration, ragged rows per expert
        dict(name="product-large", op="product", groups=8, rows=4096, n=14336, k=4096, type="bf16"),
        # 64 experts, some hundred rows each, GELU
        dict(name="ffn-gelu-64-experts", op="ffn", groups=64, rows=320, h=2048, i=2048, act=GELU, type="f16"),
        # one of eight ranks of the 256-expert configuration: 32 experts, ragged rows, SwiGLU
        dict(name="ffn-swiglu-32-experts", op="ffn", groups=32, rows=1111, h=7168, i=2048, act=SWIGLU, type="bf16"),
        # three tokens of a small layer with biases: launches and latency
        dict(name="few-small", op="few", n=3, e=8, topk=1, h=256, i=512, act=RELU, gate=0, renorm=0, weights="16",
             type="f16", bias=True),
        # one token of the Mixtral-shaped layer: decoding for one user
        dict(name="few-one-token", op="few", n=1, e=8, topk=2, h=4096, i=14336, act=SWIGLU, gate=0, renorm=0,
             weights="16", type="bf16", bias=False),
        # one token per sequence of a large batch, 64 experts
        dict(name="few-batch-64", op="few", n=64, e=64, topk=2, h=2048, i=2048, act=GELU, gate=0, renorm=1,
             weights="16", type="bf16", bias=True),
        # five users of the 256-expert layer, 8-bit weights
        dict(name="few-fp8", op="few", n=5, e=256, topk=8, h=7168, i=2048, act=SWIGLU, gate=1, renorm=1, weights="8",
             type="bf16", bias=False),
        # seventeen users of the same layer, 4-bit weights
        dict(name="few-fp4", op="few", n=17, e=256, topk=8, h=7168, i=2048, act=SWIGLU, gate=1, renorm=1, weights="4",
             type="bf16", bias=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["quantize", "product", "ffn", "few", "few"])
    if op == "quantize":
        mats, cols = rng.randint(1, 16), 64 * _spread(rng, 1, 112)
        rows = _spread(rng, 1, max(1, min(16384, 180_000_000 // (mats * cols))))
        return dict(op=op, mats=mats, rows=rows, cols=cols, type=rng.choice(["bf16", "f16", "f32"]))
    if op == "product":
        groups, n, k = rng.randint(1, 64), 64 * _spread(rng, 1, 112), 64 * _spread(rng, 1, 112)
        rows = _spread(rng, 1, max(1, min(2000, 150_000_000 // (groups * max(n, k)))))
        return dict(op=op, groups=groups, rows=rows, n=n, k=k, type=rng.choice(["bf16", "f16"]))
    if op == "ffn":
        groups, h, i = rng.randint(1, 32), 64 * _spread(rng, 1, 112), 64 * _spread(rng, 1, 64)
        return dict(op=op, groups=groups, rows=_spread(rng, 1, 1111), h=h, i=i, act=rng.choice([RELU, GELU, SWIGLU]),
                    type=rng.choice(["bf16", "f16"]))
    weights = rng.choice(["16", "16", "8", "4"])
    unit = 128 if weights == "8" else 64
    e = _spread(rng, 1, 256)
    h, i = unit * _spread(rng, 1, 7168 // unit), unit * _spread(rng, 1, 4096 // unit)
    while e * h * i > 256 * 7168 * 2048 // 4:
        e = (e + 1) // 2
    return dict(op=op, n=_spread(rng, 1, 64), e=e, topk=rng.randint(1, min(8, e)), h=h, i=i,
                act=rng.choice([RELU, GELU, SWIGLU]), gate=rng.randint(0, 1), renorm=rng.randint(0, 1), weights=weights,
                type="bf16" if weights == "8" else rng.choice(["bf16", "f16"]), bias=rng.random() < 0.5)


def work(case):
    c = case
    size = {"bf16": 2, "f16": 2, "f32": 4}[c["type"]]
    if c["op"] == "quantize":
        n = c["mats"] * c["rows"] * c["cols"]
        # the source read, codes and scales written, the values written that they stand for
        return {"bytes": n * (2 * size + 0.5 + 1 / 32), "flops": 4 * n}
    fp4 = 0.5 + 1 / 32
    if c["op"] == "product":
        rows = 0.75 * c["groups"] * c["rows"]              # counts are spread over the upper half of the capacity
        return {"bytes": fp4 * (c["groups"] * c["n"] + rows) * c["k"] + size * rows * c["n"],
                "flops": 2 * rows * c["n"] * c["k"]}
    if c["op"] == "ffn":
        rows = 0.75 * c["groups"] * c["rows"]
        m = 3 if c["act"] == SWIGLU else 2
        return {"bytes": fp4 * (m * c["groups"] * c["h"] * c["i"] + rows * c["h"]) + size * rows * c["h"],
                "flops": 2 * m * rows * c["h"] * c["i"]}
    m = 3 if c["act"] == SWIGLU else 2
    touched = c["e"] * (1 - (1 - c["topk"] / c["e"]) ** c["n"])     # experts that some token chose
    per = {"16": 2, "8": 1, "4": fp4}[c["weights"]]
    return {"bytes": touched * m * c["h"] * c["i"] * per + 2 * (c["e"] + 2 * c["n"]) * c["h"],
            "flops": 2 * c["n"] * (c["topk"] * m * c["h"] * c["i"] + c["e"] * c["h"])}


# ---- the 4-bit format in elementary operations ----------------------------------------------------------------------
def _scale_tiles(s):
    """(..., rows, blocks) -> (..., rows / 128, blocks / 4, 32, 4, 4), padded with zeros."""
    rows, blocks = s.shape[-2:]
    rt, bt = -(-rows // 128), -(-blocks // 4)
    full = torch.zeros((*s.shape[:-2], rt * 128, bt * 4), dtype=torch.uint8, device=s.device)
    full[..., :rows, :blocks] = s
    full = full.reshape(*s.shape[:-2], rt, 4, 32, bt, 4)
    d = full.dim() - 5
    return full.permute(*range(d), d, d + 3, d + 2, d + 1, d + 4).contiguous()


def _scale_rows(t, rows, blocks):
    """The inverse of _scale_tiles."""
    d = t.dim() - 5
    rt, bt = t.shape[d], t.shape[d + 1]
    s = t.permute(*range(d), d, d + 3, d + 2, d + 1, d + 4).reshape(*t.shape[:d], rt * 128, bt * 4)
    return s[..., :rows, :blocks]


def _power(field):
    """2^(field - 127) in 32 bits from its bits (a power or logarithm of 2 need not come out exact); field 0: 2^-127."""
    return torch.where(field > 0, field << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _quantize(x):
    """Codes and tiled scales of x (..., rows, cols)."""
    rows, cols = x.shape[-2:]
    v = x.float().reshape(*x.shape[:-1], cols // 32, 32)
    # the exponent field of the largest magnitude is floor(log2) + 127; the scale's own field is 2 less
    field = ((v.abs().amax(-1).view(torch.int32) >> 23) - 2).clamp(min=0)
    a = v.abs() * _power(254 - field)[..., None]
    # borders between neighbouring magnitudes; at a border the even code wins
    code = ((a > 0.25).to(torch.uint8) + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0))
    code = (code + 8 * torch.signbit(v)).to(torch.uint8).reshape(*x.shape[:-1], cols // 2, 2)
    return code[..., 0] + 16 * code[..., 1], _scale_tiles(field.to(torch.uint8))


_TABLE = {}


def _pairs(device):
    if device not in _TABLE:
        m = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
        m = torch.cat([m, -m])
        _TABLE[device] = torch.stack([m.repeat(16), m.repeat_interleave(16)], -1).to(device)
    return _TABLE[device]


def _dequantize(q, s):
    """The values of codes q (..., rows, cols / 2) with tiled scales, in 32 bits."""
    rows, cols = q.shape[-2], 2 * q.shape[-1]
    v = _pairs(q.device)[q.int()].reshape(*q.shape[:-1], cols // 32, 32)
    return (v * _power(_scale_rows(s, rows, cols // 32).int())[..., None]).reshape(*q.shape[:-1], cols)


def _act(g, u, act):
    if act == SWIGLU:
        return g / (1 + torch.exp(-g)) * u
    if act == GELU:
        return 0.5 * g * (1 + torch.erf(g * 0.5 ** 0.5))
    return torch.clamp(g, min=0)


# ---- inputs ---------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    c = dict(case)
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    dt = DTYPES[c["type"]]

    def normal(shape, std=1.0, dtype=dt):
        return torch.randn(shape, device=DEV, dtype=torch.float32, generator=g).mul_(std).to(dtype)

    def per_matrix(shape, make, std=0.02):
        """Weights of all experts, made one expert at a time (their 32-bit originals never exist all at once)."""
        parts = [make(normal(shape[1:], std, torch.bfloat16)) for _ in range(shape[0])]
        if isinstance(parts[0], tuple):
            return tuple(torch.stack(p) for p in zip(*parts))
        return torch.stack(parts)

    c["dt"] = dt
    if c["op"] == "quantize":
        x = normal((c["mats"], c["rows"], c["cols"]))
        x *= torch.exp2(torch.randint(-6, 3, (c["mats"], c["rows"], 1), device=DEV, generator=g).to(dt))
        c["x"] = x
        return c
    if c["op"] in ("product", "ffn"):
        groups, rows = c["groups"], c["rows"]
        # rows per expert: the upper half of the capacity, and one expert that got none
        c["count"] = torch.randint(rows // 2, rows + 1, (groups,), device=DEV, generator=g, dtype=torch.int32)
        if groups > 2:
            c["count"][groups // 2] = 0
        wide = c["k"] if c["op"] == "product" else c["h"]
        c["xq"], c["sx"] = per_matrix((groups, rows, wide), _quantize, 1.0)
        if c["op"] == "product":
            c["wq"], c["sw"] = per_matrix((groups, c["n"], c["k"]), _quantize)
            c["y"] = torch.zeros((groups, rows, c["n"]), device=DEV, dtype=dt)
        else:
            c["w1q"], c["s1"] = per_matrix((groups, c["i"], c["h"]), _quantize)
            c["w3q"], c["s3"] = per_matrix((groups, c["i"], c["h"]), _quantize) if c["act"] == SWIGLU else (None, None)
            c["w2q"], c["s2"] = per_matrix((groups, c["h"], c["i"]), _quantize)
            c["y"] = torch.zeros((groups, rows, c["h"]), device=DEV, dtype=dt)
        return c
    n, e, h, i = c["n"], c["e"], c["h"], c["i"]
    c["x"], c["wg"] = normal((n, h)), normal((e, h), 0.02)
    c["gate_bias"] = torch.randn(e, device=DEV, generator=g) * 0.1 if c["bias"] else None

    def blocks8(w):
        """e4m3 codes and one fp32 scale per 128 x 128 block."""
        r, k = w.shape
        v = w.float().reshape(r // 128, 128, k // 128, 128)
        s = v.abs().amax((1, 3)) / 448
        s = torch.where(s > 0, s, 1.0)
        return (v / s[:, None, :, None]).to(torch.float8_e4m3fn).view(torch.uint8).reshape(r, k), s

    def weights(rows, cols):
        if c["weights"] == "16":
            return per_matrix((e, rows, cols), lambda w: w.to(dt)), None
        return per_matrix((e, rows, cols), blocks8 if c["weights"] == "8" else _quantize)

    c["w1"], c["s1"] = weights(i, h)
    c["w3"], c["s3"] = weights(i, h) if c["act"] == SWIGLU else (None, None)
    c["w2"], c["s2"] = weights(h, i)
    c["b1"] = normal((e, i), 0.1) if c["bias"] else None
    c["b3"] = normal((e, i), 0.1) if c["bias"] and c["act"] == SWIGLU else None
    c["b2"] = normal((e, h), 0.1) if c["bias"] else None
    return c


# ---- one pass -------------------------------------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(c):
    import cuplayground_b200.layer as layer

    if c["op"] == "quantize":
        q, s = layer.quantize_fp4(c["x"])
        return layer.dequantize_fp4(q, s, c["dt"])
    if c["op"] == "product":
        return layer.expert_product_fp4(c["xq"], c["sx"], c["count"], c["wq"], c["sw"], y=c["y"])
    if c["op"] == "ffn":
        return layer.expert_ffn_fp4(c["xq"], c["sx"], c["count"], c["w1q"], c["s1"], c["w3q"], c["s3"], c["w2q"],
                                    c["s2"], c["act"], y=c["y"])
    scales = None if c["weights"] == "16" else (c["s1"], c["s3"], c["s2"])
    return layer.moe_few_tokens(c["x"], c["wg"], c["w1"], c["w3"], c["w2"], c["topk"], c["act"], gate_fn=c["gate"],
                                renorm=c["renorm"], gate_bias=c["gate_bias"], scales=scales, b1=c["b1"], b3=c["b3"],
                                b2=c["b2"])


def _run_plain(c):
    if c["op"] == "quantize":
        return _dequantize(*_quantize(c["x"])).to(c["dt"])
    if c["op"] in ("product", "ffn"):
        a = _dequantize(c["xq"], c["sx"])
        if c["op"] == "product":
            y = a @ _dequantize(c["wq"], c["sw"]).transpose(1, 2)
        else:
            g = a @ _dequantize(c["w1q"], c["s1"]).transpose(1, 2)
            u = a @ _dequantize(c["w3q"], c["s3"]).transpose(1, 2) if c["act"] == SWIGLU else None
            h = _dequantize(*_quantize(_act(g, u, c["act"])))
            y = h @ _dequantize(c["w2q"], c["s2"]).transpose(1, 2)
        # rows past a group's count stay as they were
        valid = torch.arange(c["rows"], device=DEV) < c["count"][:, None]
        return torch.where(valid[:, :, None], y.to(c["dt"]), c["y"], out=c["y"])
    n, e, k = c["n"], c["e"], c["topk"]
    # the routing is decided between neighbouring logits: 64 bits
    logits = c["x"].double() @ c["wg"].double().T
    if c["gate_bias"] is not None:
        logits = logits + c["gate_bias"].double()
    top, idx = torch.sort(logits, dim=-1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    if c["gate"] == 0:
        w = torch.exp(top - top[:, :1]) / torch.exp(logits - top[:, :1]).sum(-1, keepdim=True)
    else:
        w = 1 / (1 + torch.exp(-top))
    if c["renorm"]:
        w = w / w.sum(-1, keepdim=True)
    w = w.float()
    x = c["x"].float()
    # few choices: the chosen experts' weights, gathered; else all the experts on all the tokens
    gathered = n * k < e
    if gathered:
        rows = x.repeat_interleave(k, 0)[:, None, :]
        share = w.reshape(n * k, 1, 1)
    else:
        rows = x.expand(e, n, x.shape[1])
        share = torch.zeros((n, e), device=DEV).scatter_(1, idx, w).T[:, :, None]

    def project(rows, name):
        """rows (experts, m, in) through projection `name` of the experts in question."""
        v, s, b = c["w" + name], c["s" + name], c["b" + name]
        if gathered:
            v, s, b = (p if p is None else p.index_select(0, idx.reshape(-1)) for p in (v, s, b))
        if c["weights"] == "16":
            v = v.float()
        elif c["weights"] == "4":
            v = _dequantize(v, s)
        else:
            blocks = v.view(torch.float8_e4m3fn).float().reshape(len(v), v.shape[1] // 128, 128, v.shape[2] // 128, 128)
            v = (blocks * s[:, :, None, :, None]).reshape(v.shape)
        out = rows @ v.transpose(1, 2)
        return out if b is None else out + b.float()[:, None, :]

    h = _act(project(rows, "1"), project(rows, "3") if c["act"] == SWIGLU else None, c["act"])
    y = project(h, "2") * share
    y = y.reshape(n, k, -1).sum(1) if gathered else y.sum(0)
    return y.to(c["dt"]), idx.int(), w


# ---- the same in 64 bits, from the definitions ----------------------------------------------------------------------
def exact(case, seed):
    c = prepare(case, seed)
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=DEV, dtype=torch.float64)

    def scale_bytes(s, rows, blocks):
        r = torch.arange(rows, device=DEV)[:, None]
        b = torch.arange(blocks, device=DEV)[None, :]
        return s[r // 128, b // 4, r % 32, r % 128 // 32, b % 4]

    def values4(q, s):
        nib = torch.stack([q & 15, q >> 4], -1).reshape(q.shape[0], -1).long()
        powers = ((scale_bytes(s, nib.shape[0], nib.shape[1] // 32).long() - 127 + 1023) << 52).view(torch.float64)
        v = grid[nib & 7] * torch.where(nib >= 8, -1.0, 1.0).double()
        return v * powers.repeat_interleave(32, 1)

    def rounded4(v):
        """What a (rows, cols) matrix becomes in the 4-bit format, in 64 bits."""
        b = v.reshape(v.shape[0], -1, 32)
        top = b.abs().amax(-1, keepdim=True)
        # floor(log2(top)) - 2, at least -127, out of the bits of the 64-bit number
        e = torch.clamp((top.view(torch.int64) >> 52) - 1023 - 2, min=-127)
        x = ((e + 1023) << 52).view(torch.float64)
        m = b.abs() / x
        # steps of 0.5 below 2, of 1 below 4, of 2 above; round() takes ties to even multiples of the step
        step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
        m = torch.clamp(torch.round(m / step) * step, max=6.0)
        return (torch.copysign(m, b) * x).reshape(v.shape)

    def activated(g, u):
        if c["act"] == SWIGLU:
            return g * torch.sigmoid(g) * u
        return g * 0.5 * torch.erfc(-g / math.sqrt(2.0)) if c["act"] == GELU else torch.relu(g)

    if c["op"] == "quantize":
        return torch.stack([rounded4(m.double()) for m in c["x"]])
    if c["op"] in ("product", "ffn"):
        y = torch.zeros(c["y"].shape, device=DEV, dtype=torch.float64)
        for e, m in enumerate(c["count"].tolist()):
            a = values4(c["xq"][e], c["sx"][e])[:m]
            if c["op"] == "product":
                y[e, :m] = a @ values4(c["wq"][e], c["sw"][e]).T
            elif m:
                g = a @ values4(c["w1q"][e], c["s1"][e]).T
                u = a @ values4(c["w3q"][e], c["s3"][e]).T if c["act"] == SWIGLU else None
                y[e, :m] = rounded4(activated(g, u)) @ values4(c["w2q"][e], c["s2"][e]).T
        return y
    logits = (c["x"].double()[:, None, :] * c["wg"].double()[None, :, :]).sum(-1)
    if c["gate_bias"] is not None:
        logits += c["gate_bias"].double()
    table = logits.cpu().tolist()
    order = [sorted(range(c["e"]), key=lambda j: (-row[j], j))[:c["topk"]] for row in table]
    share = []
    for row, chosen in zip(table, order):
        if c["gate"] == 0:
            top = max(row)
            total = math.fsum(math.exp(v - top) for v in row)
            p = [math.exp(row[j] - top) / total for j in chosen]
        else:
            p = [1 / (1 + math.exp(-row[j])) for j in chosen]
        share.append([v / sum(p) for v in p] if c["renorm"] else p)

    def matrix(name, j):
        w = c["w" + name][j]
        if c["weights"] == "16":
            return w.double()
        if c["weights"] == "4":
            return values4(w, c["s" + name][j])
        s = c["s" + name][j].double()
        return w.view(torch.float8_e4m3fn).double() * s.repeat_interleave(128, 0).repeat_interleave(128, 1)

    y = torch.zeros(c["x"].shape, device=DEV, dtype=torch.float64)
    for j in sorted({j for chosen in order for j in chosen}):
        who = [t for t, chosen in enumerate(order) if j in chosen]
        p = torch.tensor([share[t][order[t].index(j)] for t in who], device=DEV, dtype=torch.float64)
        bias = {m: c["b" + m][j].double() if c["b" + m] is not None else 0.0 for m in ("1", "3", "2")}
        rows = c["x"][who].double()
        g = rows @ matrix("1", j).T + bias["1"]
        u = rows @ matrix("3", j).T + bias["3"] if c["act"] == SWIGLU else None
        y[who] += p[:, None] * (activated(g, u) @ matrix("2", j).T + bias["2"])
    return y, None, torch.tensor(share, dtype=torch.float64)

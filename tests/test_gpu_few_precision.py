"""How many bits of the hidden activations the down projection of the few-token layer sees, and that a token's results do not
depend on which of the ways through the down projection its expert takes."""
import pytest

from test_gpu_few_tokens import FORMATS, Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n", [1, 7, 12, 40])           # one and two token tiles, several passes over the weights
@pytest.mark.parametrize("weights,dtype", [("16", "bfloat16"), ("16", "float16"), ("8", "bfloat16")])
def test_the_down_projection_sees_hidden_activations_beyond_16_bits(weights, dtype, n):
    """W1 adds columns of x: h[r] = a + c + b for r < 64 and a + c for r >= 64, with a in [1, 2) of 8 bits, c in [2^-9, 2^-8) of
    8 bits and b an odd multiple of 2^-17, all of them exact in the operand types, h exact in fp32. W2 takes differences, so
    every output is +-b. An h of 11 bits loses b and c altogether. An h of two bf16 numbers ends at 2^-16: it is off by
    2^-17. fp32 sums may be off by a whole step (2^-22, for partial sums below 2) per addition: three for the two h, five for
    the up to six operands behind them."""
    import torch
    import cuplayground_b200.layer as layer
    dt = getattr(torch, dtype)
    H, I, m = 256, 128, 64
    g = torch.Generator(device="cuda")
    g.manual_seed(n)
    draw = lambda lo, hi: torch.randint(lo, hi, (n, m), device="cuda", generator=g).double()
    a, c, b = draw(128, 256) * 2.0 ** -7, draw(128, 256) * 2.0 ** -16, (2 * draw(0, 4) + 1) * 2.0 ** -17
    x = torch.zeros(n, H, device="cuda", dtype=torch.float64)
    x[:, :m], x[:, m:2 * m], x[:, 2 * m:3 * m] = a, c, b
    assert torch.equal(x.to(dt).double(), x)
    r = torch.arange(m, device="cuda")
    w1, w2 = torch.zeros(1, I, H, device="cuda"), torch.zeros(1, H, I, device="cuda")
    for row, parts in ((r, 3), (m + r, 2)):
        for p in range(parts):
            w1[0, row, p * m + r] = 1.0
    o = torch.arange(H, device="cuda")
    sign = torch.where(o < H // 2, 1.0, -1.0)
    w2[0, o, o % m], w2[0, o, m + o % m] = sign, -sign
    if weights == "8":                                  # 1, -1 and 0 in e4m3, scales of 1
        code = lambda w: w.to(torch.float8_e4m3fn).view(torch.uint8)
        one = lambda w: torch.ones(1, w.shape[1] // 128, w.shape[2] // 128, device="cuda")
        scales, w1, w2 = (one(w1), None, one(w2)), code(w1), code(w2)
    else:
        scales, w1, w2 = None, w1.to(dt), w2.to(dt)
    wg = torch.zeros(1, H, device="cuda", dtype=dt)
    out = layer.moe_few_tokens(x.to(dt), wg, w1, None, w2, 1, 0, scales=scales)[0].double()
    want = sign.double() * b[:, o % m]
    bound = 8 * 2.0 ** -22 + torch.finfo(dt).eps / 2 * want.abs()
    assert ((out - want).abs() <= bound).all(), (out - want).abs().max().item() * 2 ** 17


@pytest.mark.parametrize("weights,dtype", FORMATS)
def test_a_token_does_not_depend_on_who_else_chose_its_experts(weights, dtype):
    """3 experts, 2 of them per token: up to 40 tokens of an expert (several passes, two tiles), then 8 or fewer, 4 or fewer, 1."""
    import torch
    c = Case(40, 3, 2, 256, 384, 2, weights, dtype, renorm=1, seed=40)
    want = c.run()
    for lo, hi in ((0, 40), (0, 9), (9, 17), (20, 25), (30, 33), (39, 40)):
        got = c.run(c.x[lo:hi].contiguous())
        for g, w in zip(got, want):
            assert torch.equal(g, w[lo:hi]), (lo, hi)


@pytest.mark.parametrize("n", [3, 30])
@pytest.mark.parametrize("weights,dtype", [("16", "float16"), ("8", "bfloat16")])
def test_hidden_activations_of_very_different_size(weights, dtype, n):
    """The two fp16 terms are scaled per 16 columns and again per row: columns 2^60 apart (e4m3: scales of their own; fp16: 2^14),
    columns of zeros, and an expert whose hidden activations are all zero. Two fp16 terms are off by 2^-24 of the value, and by
    2^-38 of the largest of the row, which the reference adds by itself."""
    import torch
    import fp4_reference as R
    c = Case(n, 3, 2, 256, 512, 0, weights, dtype, seed=n)
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    if weights == "8":
        c.s["1"] = c.s["1"] * torch.exp2(torch.randint(-30, 31, c.s["1"].shape[:2] + (1,), device="cuda", generator=g).float())
        c.s["1"][0, 1], c.s["1"][2] = 0.0, 0.0
        c.mats["1"] = lambda e: R.decode_fp8(c.w["1"][e], c.s["1"][e])
    else:
        shift = torch.randint(-8, 7, (3, 32, 1, 1), device="cuda", generator=g).float()
        w = (c.w["1"].float().reshape(3, 32, 16, 256) * torch.exp2(shift)).reshape(3, 512, 256)
        w[0, 48:80], w[2] = 0.0, 0.0
        c.w["1"] = w.half()
        c.mats["1"] = lambda e: c.w["1"][e].double()
    out, idx, w = c.run()
    ref, bound = R.moe_few(c.x, idx, w, c.mats, c.b, 0, 2.0 ** -24)
    R.assert_within(out, ref, bound + R.half_step(c.dt) * (ref.abs() + bound) * 1.01 + 2.0 ** -25)


def test_e4m3_scales_that_are_parts_of_one_tensor():
    """3 experts of one 128 x 128 block: the scales of w3 start 12 bytes behind those of w1."""
    import torch
    c = Case(5, 3, 2, 128, 128, 2, "8", seed=12)
    want = c.run()
    packed = torch.cat([c.s[m].reshape(-1) for m in ("1", "3", "2")])
    c.s = {m: packed[3 * i:3 * i + 3].view(3, 1, 1) for i, m in enumerate(("1", "3", "2"))}
    assert all(torch.equal(a, b) for a, b in zip(c.run(), want))


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n", [3, 8, 24])
def test_an_infinite_weight_reaches_its_own_outputs_only(dtype, n):
    """An infinity in w2 meets all terms of a hidden activation, zeros among them: its column is not finite for the tokens of its
    expert, nothing else changes."""
    import math
    import torch
    c = Case(n, 4, 2, 256, 384, 2, "16", dtype, seed=n)
    clean, idx, _ = c.run()
    c.w["2"][1, 77, 5] = math.inf
    out = c.run()[0]
    mine = (idx == 1).any(1)
    rest = torch.arange(256, device="cuda") != 77
    assert mine.any() and not torch.isfinite(out[mine][:, 77]).any()
    assert torch.equal(out[:, rest], clean[:, rest]) and torch.equal(out[~mine], clean[~mine])

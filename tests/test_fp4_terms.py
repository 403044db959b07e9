"""The split of activations into 4-bit terms (few-token layer, 4-bit weights): eight terms hold what seven do not."""
import pytest

torch = pytest.importorskip("torch")

import fp4_reference as R

H = 128


def split(v, terms):
    """What `terms` e2m1 numbers of a block of 32 stand for, in float64: in units of 2^(s0 - 3 j) with the block's largest magnitude in
    [2, 4) * 2^s0, each the nearest to what the ones before left over."""
    b = v.double().reshape(*v.shape[:-1], -1, 32)
    unit = R.pow2((b.abs().amax(-1, keepdim=True).view(torch.int64) >> 52) - 1023 - 1)
    r, total = b / unit, torch.zeros_like(b)
    for _ in range(terms):
        step = torch.where(r.abs() < 2, 0.5, torch.where(r.abs() < 4, 1.0, 2.0)).double()
        d = torch.copysign((torch.round(r.abs() / step) * step).clamp(max=6.0), r)
        total += d * unit
        r, unit = (r - d) * 8, unit / 8
    return total.reshape(v.shape)


def tokens(n, device="cpu"):
    """Every block of 32 columns: one number in [1, 2) of 8 bits, and 31 odd multiples of 2^-21 (1 to 7). The units of such a block are
    2^-1, 2^-4, ..: the seventh term is a multiple of 2^-20, the eighth of 2^-23, so that seven terms are off by 2^-21 at
    least in every small number and eight are exact."""
    g = torch.Generator()
    g.manual_seed(n)
    x = (2 * torch.randint(0, 4, (n, H), generator=g) + 1).double() * 2.0 ** -21
    x[:, ::32] = 1.0 + torch.randint(0, 128, (n, H // 32), generator=g).double() / 128
    return x.to(device)


def picked(x):
    """What the weights of the test below pick: one small number per output."""
    r = torch.arange(H, device=x.device)
    return x[:, 32 * (r % 4) + 1 + r % 31]


def bound(want, dtype):
    """Products of a picked number with 1 and sums with zeros are exact: half a step of the output, and 2^-24 for its smallest one."""
    return R.half_step(dtype) * want.abs() + (2.0 ** -25 if dtype == torch.float16 else 0.0)


def test_seven_terms_are_outside_the_bound_and_eight_are_exact():
    x = tokens(5)
    assert torch.equal(split(x, 8), x)
    for dtype in (torch.bfloat16, torch.float16):
        want = picked(x)
        assert ((picked(split(x, 7)) - want).abs() > 8 * bound(want, dtype)).all()
        assert torch.equal(x.to(dtype).double(), x)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("n", [1, 4, 20])
def test_4_bit_weights_meet_the_eighth_term(n, dtype):
    """W1 is the identity and W2 picks: tokens and hidden activations (the same numbers) both need their eighth term."""
    import cuplayground_b200.layer as layer
    dt = getattr(torch, dtype)
    x = tokens(n, "cuda")
    r = torch.arange(H, device="cuda")
    w1, w2 = torch.eye(H, device="cuda")[None], torch.zeros(1, H, H, device="cuda")
    w2[0, r, 32 * (r % 4) + 1 + r % 31] = 1.0
    (q1, s1), (q2, s2) = layer.quantize_fp4(w1), layer.quantize_fp4(w2)
    wg = torch.zeros(1, H, device="cuda", dtype=dt)
    out = layer.moe_few_tokens(x.to(dt), wg, q1, None, q2, 1, 0, scales=(s1, None, s2))[0]
    want = picked(x)
    assert ((out.double() - want).abs() <= bound(want, dt)).all(), ((out.double() - want).abs() * 2 ** 21).max()

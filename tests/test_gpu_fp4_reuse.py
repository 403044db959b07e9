"""The 4-bit products where every CTA pair has more than two tiles of many stages: both accumulators, the columns that they share,
and all buffers of scales are used again and again, in each of the kernels."""
import pytest

import fp4_reference as R

pytestmark = pytest.mark.gpu

GROUPS, ROWS, COUNTS = 4, 1100, [1100, 1024, 3, 900]                  # 5 + 4 + 1 + 4 row tiles of 256


def _operand(torch, layer, shape, seed, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return layer.quantize_fp4(torch.randn(shape, device="cuda", generator=g) * std)


@pytest.mark.parametrize("name", ["float32", "bfloat16", "float16"])
def test_product(name):
    """14 x 18 tiles of 8 stages for at most 74 pairs."""
    import torch
    import cuplayground_b200.layer as layer
    dt, N, K = getattr(torch, name), 4608, 2048
    a, b = _operand(torch, layer, (GROUPS, ROWS, K), 1), _operand(torch, layer, (GROUPS, N, K), 2, 0.05)
    count = torch.tensor(COUNTS, dtype=torch.int32, device="cuda")
    run = lambda: layer.expert_product_fp4(*a, count, *b, dtype=dt)
    y = run()
    for g, m in enumerate(COUNTS):
        x, w = R.decode(a[0][g], a[1][g])[:m], R.decode(b[0][g], b[1][g])
        ref = x @ w.T
        R.assert_within(y[g, :m], ref, R.dot_bound(x, w.T) + R.half_step(dt) * ref.abs() * 1.01 + 1e-30, f"group {g}")
        assert (y[g, m:] == 0).all()
    for _ in range(5):
        assert torch.equal(run(), y)


@pytest.mark.parametrize("act", [0, 1, 2])
def test_ffn(act):
    """Up: 14 x 16 (SwiGLU 14 x 32) tiles of 18 stages; down: 14 x 18 tiles of 16."""
    import torch
    import cuplayground_b200.layer as layer
    H, I = 4608, 4096
    x = _operand(torch, layer, (GROUPS, ROWS, H), 3)
    w1, w2 = _operand(torch, layer, (GROUPS, I, H), 4, 0.02), _operand(torch, layer, (GROUPS, H, I), 6, 0.02)
    w3 = _operand(torch, layer, (GROUPS, I, H), 5, 0.02) if act == 2 else (None, None)
    count = torch.tensor(COUNTS, dtype=torch.int32, device="cuda")
    run = lambda: layer.expert_ffn_fp4(*x, count, *w1, *w3, *w2, act)
    y = run()
    for g, m in enumerate(COUNTS):
        mats = [None if q is None else R.decode(q[g], s[g]) for q, s in (w1, w3, w2)]
        ref, bound = R.ffn_fp4(R.decode(x[0][g], x[1][g])[:m], *mats, act)
        R.assert_within(y[g, :m], ref, bound + R.half_step(torch.bfloat16) * (ref.abs() + bound) * 1.01 + 1e-30, f"group {g}")
        assert (y[g, m:] == 0).all()
    for _ in range(5):
        assert torch.equal(run(), y)

"""Microscaled 4-bit operands on the GPU: quantisation and its way back (exact), the grouped product and the expert FFN
against 64-bit references."""
import math

import numpy as np
import pytest

import fp4_reference as R

pytestmark = pytest.mark.gpu


def _mods():
    import torch
    import cuplayground_b200 as cp
    import cuplayground_b200.layer as layer
    return torch, cp, layer


def _normal(torch, shape, seed, dtype, std=1.0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


# ---- quantisation -----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [(1, 64), (3, 64), (128, 128), (129, 192), (77, 320), (5, 130, 448), (2, 3, 31, 64),
                                   (1000, 2048), (1, 7168)])
@pytest.mark.parametrize("name", ["float32", "bfloat16", "float16"])
def test_quantize_is_exact(shape, name):
    torch, cp, layer = _mods()
    dt = getattr(torch, name)
    x = _normal(torch, shape, 3, dt)
    x = x * torch.exp2(torch.randint(-9, 6, (*shape[:-1], 1), device="cuda").to(dt))
    x.view(-1)[::37] = 0.0
    if x.numel() > 64:
        x.view(-1)[32:64] = 0.0                                    # a block of zeros
    q, s = layer.quantize_fp4(x)
    rows, cols = shape[-2:]
    want_s = R.block_scale(x)
    assert torch.equal(R.scale_bytes(s, rows, cols // 32).long(), want_s)
    assert torch.equal(R.decode(q, s), R.rounded(x))
    # what only fills up the scale tiles is zero
    full = s.permute(*range(s.dim() - 5), -5, -2, -3, -4, -1).reshape(*s.shape[:-5], s.shape[-5] * 128, s.shape[-4] * 4)
    assert int(full[..., rows:, :].sum()) == 0 and int(full[..., cols // 32:].sum()) == 0
    for back in (torch.float32, torch.bfloat16):
        assert torch.equal(layer.dequantize_fp4(q, s, back).double(), R.decode(q, s))
    assert torch.equal(layer.dequantize_fp4(q, s, torch.float16), R.decode(q, s).to(torch.float16))


def test_quantize_ties_saturation_and_signs():
    torch, cp, layer = _mods()
    v = torch.zeros(8, 64)
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 0.24999, 0.25001, 5.0001, 6.0, 6.5, 7.99, -0.25, -0.75, -2.5, -5.0, -7.9,
            -0.1, -0.0]
    v[0, :len(ties)] = torch.tensor(ties)
    v[0, 31] = 4.0                                                 # largest in [4, 8): scale 1
    v[1] = v[0] * 2.0 ** 100
    v[2] = v[0] * 2.0 ** -120
    v[3] = v[0] * 2.0 ** -128                                      # scale clamped at 2^-127
    v[4, 3], v[4, 40] = 1e-45, -1e-40                              # subnormal blocks
    v[5, 0] = torch.finfo(torch.float32).max
    v[5, 33] = -torch.finfo(torch.float32).max
    v[6, 0], v[6, 33] = 1.0, 2.0 - 2.0 ** -23                      # next to a power of two
    x = v.cuda()
    q, s = layer.quantize_fp4(x)
    assert torch.equal(R.scale_bytes(s, 8, 2).long(), R.block_scale(x))
    want = R.rounded(x)
    got = R.decode(q, s)
    assert torch.equal(got, want)
    assert torch.equal(torch.signbit(got), torch.signbit(want))


@pytest.mark.parametrize("name", ["float32", "bfloat16", "float16"])
def test_a_block_with_infinity_or_nan_comes_back_as_nan_and_no_other(name):
    torch, cp, layer = _mods()
    dt = getattr(torch, name)
    x = _normal(torch, (40, 192), 5, dt)
    x[3, 40], x[17, 0], x[39, 191] = math.inf, math.nan, -math.inf
    q, s = layer.quantize_fp4(x)
    back = layer.dequantize_fp4(q, s, dt)
    bad = torch.zeros(40, 6, dtype=torch.bool, device="cuda")
    bad[3, 1] = bad[17, 0] = bad[39, 5] = True
    assert torch.equal(torch.isnan(back), bad.repeat_interleave(32, 1))
    assert torch.equal(R.scale_bytes(s, 40, 6) == 255, bad)


def test_every_code_and_scale_decodes():
    torch, cp, layer = _mods()
    codes = torch.arange(256, dtype=torch.uint8, device="cuda").repeat(256, 1)[:, :, None].expand(256, 256, 16)
    q = codes.reshape(256, 4096).contiguous()                       # row r: block b holds byte b sixteen times
    s = torch.zeros((2, 64, 32, 4, 4), dtype=torch.uint8, device="cuda")
    r = torch.arange(256, device="cuda")
    s[r // 128, :, r % 32, r % 128 // 32, :] = r.to(torch.uint8)[:, None, None]    # row r: scale r everywhere
    want = R.decode(q, s)
    got = layer.dequantize_fp4(q, s, torch.float32)
    f32 = want.to(torch.float32)                                   # beyond fp32's range: infinity
    assert torch.equal(torch.isnan(got), torch.isnan(f32)) and torch.equal(got.nan_to_num(1.0), f32.nan_to_num(1.0))
    for dt in (torch.bfloat16, torch.float16):
        got, w = layer.dequantize_fp4(q, s, dt), f32.to(dt)
        assert torch.equal(got.nan_to_num(1.0), w.nan_to_num(1.0))


# ---- product ----------------------------------------------------------------------------------------------------------
def _operand(torch, layer, shape, seed, std=1.0):
    return layer.quantize_fp4(_normal(torch, shape, seed, torch.bfloat16, std))


@pytest.mark.parametrize("name", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("groups,rows,experts,N,K,counts", [
    (1, 128, 1, 256, 256, [128]),                # one tile, one stage
    (1, 1, 1, 64, 64, [1]),                      # the smallest
    (2, 200, 2, 320, 192, [200, 77]),            # ragged rows, columns and K (a stage of three steps)
    (3, 300, 3, 128, 448, [300, 0, 129]),        # an empty group, an odd number of scale tiles
    (6, 130, 3, 512, 1024, [130, 1, 128, 0, 129, 64]),   # two groups per expert
    (2, 640, 2, 1088, 2048, [640, 513]),         # several tiles per CTA order
    (1, 128, 1, 256, 7168, [128]),
])
def test_product(groups, rows, experts, N, K, counts, name):
    torch, cp, layer = _mods()
    dt = getattr(torch, name)
    aq, sa = _operand(torch, layer, (groups, rows, K), 11)
    bq, sb = _operand(torch, layer, (experts, N, K), 12, 0.05)
    count = torch.tensor(counts, dtype=torch.int32, device="cuda")
    y = torch.full((groups, rows, N), 7.0, dtype=dt, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    out = layer.expert_product_fp4(aq, sa, count, bq, sb, y=y, dev_status=status)
    assert out is y and int(status) == 0
    a, b = R.decode(aq, sa), R.decode(bq, sb)
    for g, m in enumerate(counts):
        bt = b[g % experts].T
        ref = a[g, :m] @ bt
        R.assert_within(y[g, :m], ref, R.dot_bound(a[g, :m], bt) + R.half_step(dt) * ref.abs() * 1.01 + 1e-30, f"group {g}")
        assert (y[g, m:] == 7.0).all(), "rows past the count are not touched"


def test_product_many_tiles_per_cta():
    """More tiles than two rounds of CTAs: both accumulators, their shared columns and the scale buffers are reused."""
    torch, cp, layer = _mods()
    groups, rows, N, K = 4, 1100, 2944, 576
    aq, sa = _operand(torch, layer, (groups, rows, K), 21)
    bq, sb = _operand(torch, layer, (groups, N, K), 22)
    counts = [1100, 1024, 3, 900]
    count = torch.tensor(counts, dtype=torch.int32, device="cuda")
    y = layer.expert_product_fp4(aq, sa, count, bq, sb, dtype=torch.float32)
    y2 = layer.expert_product_fp4(aq, sa, count, bq, sb, dtype=torch.float32)
    assert torch.equal(y, y2)
    for g, m in enumerate(counts):
        a, b = R.decode(aq[g], sa[g])[:m], R.decode(bq[g], sb[g])
        R.assert_within(y[g, :m], a @ b.T, R.dot_bound(a, b.T) + 1e-30, f"group {g}")


def test_product_scales_far_from_one_and_rows_of_nan():
    torch, cp, layer = _mods()
    rows, N, K = 70, 128, 256
    x = _normal(torch, (1, rows, K), 31, torch.float32)
    x *= torch.exp2(torch.randint(-40, 40, (1, rows, K // 32), device="cuda").float()).repeat_interleave(32, -1)
    w = _normal(torch, (1, N, K), 32, torch.float32)
    w *= torch.exp2(torch.randint(-30, 30, (1, N, K // 32), device="cuda").float()).repeat_interleave(32, -1)
    x[0, 5, 100] = math.nan
    w[0, 9, 3] = math.inf
    (aq, sa), (bq, sb) = layer.quantize_fp4(x), layer.quantize_fp4(w)
    # rows past the count hold NaN scales: they stay out of the valid rows
    sa_bad = sa.clone()
    keep = 60
    r = torch.arange(keep, rows, device="cuda")
    sa_bad[0, r // 128, :, r % 32, r % 128 // 32, :] = 255
    count = torch.tensor([keep], dtype=torch.int32, device="cuda")
    y = layer.expert_product_fp4(aq, sa_bad, count, bq, sb, dtype=torch.float32)[0]
    a, b = R.decode(aq, sa)[0, :keep], R.decode(bq, sb)[0]
    nan = torch.zeros(keep, N, dtype=torch.bool, device="cuda")
    nan[5], nan[:, 9] = True, True
    assert torch.equal(torch.isnan(y[:keep]), nan)
    a, b = a.nan_to_num(0.0), b.nan_to_num(0.0)
    ref = a @ b.T
    R.assert_within(y[:keep][~nan], ref[~nan], (R.dot_bound(a, b.T) + 1e-30)[~nan])
    assert (y[keep:] == 0).all()


def test_product_counts_outside_the_range_are_clamped():
    torch, cp, layer = _mods()
    aq, sa = _operand(torch, layer, (3, 40, 128), 41)
    bq, sb = _operand(torch, layer, (3, 64, 128), 42)
    want = layer.expert_product_fp4(aq, sa, torch.tensor([40, 0, 40], dtype=torch.int32, device="cuda"), bq, sb)
    got = layer.expert_product_fp4(aq, sa, torch.tensor([41, -3, 2 ** 31 - 1], dtype=torch.int32, device="cuda"), bq, sb)
    assert torch.equal(got, want)


# ---- expert FFN -------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("groups,rows,experts,H,I,act,counts", [
    (1, 128, 1, 256, 256, 0, [128]),
    (1, 1, 1, 64, 64, 2, [1]),
    (2, 200, 2, 512, 320, 1, [200, 77]),
    (3, 300, 3, 192, 448, 2, [300, 0, 129]),
    (4, 160, 2, 1024, 576, 2, [160, 1, 128, 33]),
    (4, 260, 4, 640, 1088, 0, [260, 256, 0, 5]),
])
@pytest.mark.parametrize("name", ["bfloat16", "float16", "float32"])
def test_ffn(groups, rows, experts, H, I, act, counts, name):
    torch, cp, layer = _mods()
    dt = getattr(torch, name)
    xq, sx = _operand(torch, layer, (groups, rows, H), 51)
    w1 = _operand(torch, layer, (experts, I, H), 52, 0.05)
    w3 = _operand(torch, layer, (experts, I, H), 53, 0.05) if act == 2 else (None, None)
    w2 = _operand(torch, layer, (experts, H, I), 54, 0.05)
    count = torch.tensor(counts, dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    y = torch.full((groups, rows, H), -3.0, dtype=dt, device="cuda")
    layer.expert_ffn_fp4(xq, sx, count, *w1, *w3, *w2, act, y=y, dev_status=status)
    assert int(status) == 0
    x = R.decode(xq, sx)
    for g, m in enumerate(counts):
        e = g % experts
        mats = [None if q is None else R.decode(q[e], s[e]) for q, s in (w1, w3, w2)]
        ref, bound = R.ffn_fp4(x[g, :m], *mats, act)
        R.assert_within(y[g, :m], ref, bound + R.half_step(dt) * (ref.abs() + bound) * 1.01 + 1e-30, f"group {g}")
        assert (y[g, m:] == -3.0).all()


def test_ffn_in_a_graph_and_on_another_stream():
    torch, cp, layer = _mods()
    xq, sx = _operand(torch, layer, (2, 96, 256), 61)
    w1, w2 = _operand(torch, layer, (2, 192, 256), 62, 0.1), _operand(torch, layer, (2, 256, 192), 63, 0.1)
    count = torch.tensor([96, 50], dtype=torch.int32, device="cuda")
    run = lambda: layer.expert_ffn_fp4(xq, sx, count, *w1, None, None, *w2, 1)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for c in ([96, 50], [1, 96]):
        count.copy_(torch.tensor(c, dtype=torch.int32))
        graph.replay()
        again = run()
        torch.cuda.synchronize()
        assert torch.equal(held, again)


def test_quantize_to_combine_with_the_other_stages():
    """The 4-bit FFN between the stages that a layer runs around it: gate, dispatch, gather, quantise, FFN, combine."""
    torch, cp, layer = _mods()
    S, H, I, E, k, act = 300, 256, 320, 6, 2, 2
    x = _normal(torch, (S, H), 71, torch.bfloat16)
    wg = _normal(torch, (E, H), 72, torch.bfloat16, 0.1)
    mats = [_operand(torch, layer, shape, 73 + i, 0.05) for i, shape in enumerate([(E, I, H), (E, I, H), (E, H, I)])]
    idx, w = layer.gate_topk(x, wg, k)
    cap = 96
    count, slot_of, tos = layer.dispatch(idx, E, cap)
    xg = layer.permute(x, slot_of, E * cap, zero=True).reshape(E, cap, H)
    xq, sx = layer.quantize_fp4(xg)
    y = layer.expert_ffn_fp4(xq, sx, count, *mats[0], *mats[1], *mats[2], act)
    out = layer.combine(y.reshape(E * cap, H), slot_of, w)
    xr = R.rounded(x)                                              # a row's blocks are its own: rounding commutes with the gather
    ref, bound = torch.zeros(S, H, device="cuda").double(), torch.zeros(S, H, device="cuda").double()
    for e in range(E):
        rows, j = ((idx == e) & (slot_of >= 0)).nonzero(as_tuple=True)
        r, b = R.ffn_fp4(xr[rows], *(R.decode(q[e], s[e]) for q, s in mats), act)
        p = w[rows, j].double()[:, None]
        half = R.half_step(torch.bfloat16)
        ref.index_add_(0, rows, p * r)
        bound.index_add_(0, rows, p * (b + 1.01 * half * (r.abs() + b)))
    assert int((slot_of < 0).sum()) > 0, "some assignments were dropped"
    R.assert_within(out, ref, bound * 1.01 + half * (ref.abs() + bound) * 1.01 + 1e-30)


# ---- refusals ---------------------------------------------------------------------------------------------------------
def test_tensors_that_do_not_fit_are_refused():
    torch, cp, layer = _mods()
    xq, sx = _operand(torch, layer, (2, 40, 128), 81)
    wq, sw = _operand(torch, layer, (2, 64, 128), 82)
    count = torch.tensor([40, 40], dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError):
        layer.expert_product_fp4(xq, sx[:, :, :0], count, wq, sw)
    with pytest.raises(ValueError):
        layer.expert_product_fp4(xq, sx, count.long(), wq, sw)
    with pytest.raises(ValueError):
        layer.expert_product_fp4(xq, sx, count, wq[:, :, :32].contiguous(), sw)
    with pytest.raises(ValueError):
        layer.expert_product_fp4(xq, sx, count, wq, sw, y=torch.zeros(2, 40, 63, device="cuda"))
    with pytest.raises(ValueError):
        layer.expert_product_fp4(xq.cpu(), sx, count, wq, sw)
    with pytest.raises(ValueError):
        layer.quantize_fp4(torch.zeros(64, 128, device="cuda").T)            # not contiguous
    with pytest.raises(TypeError):
        layer.quantize_fp4(torch.zeros(4, 64, device="cuda", dtype=torch.float64))
    with pytest.raises(cp.AristosError):
        layer.quantize_fp4(torch.zeros(4, 96, device="cuda"))
    with pytest.raises(ValueError):
        layer.expert_ffn_fp4(xq, sx, count, wq, sw, None, None, wq, sw, 2)
    # nothing to do is not an error
    q, s = layer.quantize_fp4(torch.zeros(0, 64, device="cuda"))
    assert q.shape == (0, 32) and layer.dequantize_fp4(q, s).shape == (0, 64)
    none = layer.expert_product_fp4(xq[:, :0].contiguous(), sx[:, :0].contiguous(), count, wq, sw)
    assert none.shape == (2, 0, 64)


@pytest.mark.parametrize("act", [0, 1, 2])
def test_ffn_keeps_a_nan_of_the_up_projection(act):
    """One weight row with a NaN scale: that column of h is NaN (ReLU does not turn it into 0), its block of h gets the NaN
    scale, and every output of the expert that reads the block is NaN; the other experts' are as before."""
    torch, cp, layer = _mods()
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    mk = lambda *s: layer.quantize_fp4(torch.randn(s, device="cuda", generator=g) * 0.1)
    x, w1, w3, w2 = mk(2, 20, 256), mk(2, 320, 256), mk(2, 320, 256), mk(2, 256, 320)
    count = torch.tensor([20, 17], dtype=torch.int32, device="cuda")
    run = lambda: layer.expert_ffn_fp4(*x, count, *w1, *(w3 if act == 2 else (None, None)), *w2, act)
    clean = run()
    assert torch.isfinite(clean).all()
    w1[1][1, 2, 1, 300 % 32, 300 // 32 % 4, 0] = 255
    out = run()
    assert torch.equal(out[0], clean[0])
    assert torch.isnan(out[1, :17]).all() and (out[1, 17:] == 0).all()

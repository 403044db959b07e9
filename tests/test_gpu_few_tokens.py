"""The layer for few tokens (moe_few_tokens): routing bit for bit as the gate's, outputs against 64 bits, at the sizes where
tiles, steps and lists end, for every weight format; graphs, streams and overlapping calls."""
import math

import pytest

import fp4_reference as R

pytestmark = pytest.mark.gpu


def _mods():
    import torch
    import cuplayground_b200 as cp
    import cuplayground_b200.layer as layer
    return torch, cp, layer


class Case:
    def __init__(self, n, E, k, H, I, act, weights="16", dtype="bfloat16", gate_fn=0, renorm=0, bias=False, seed=1, std=0.05):
        torch, cp, layer = _mods()
        self.torch, self.layer = torch, layer
        self.dt = getattr(torch, dtype)
        self.act, self.k, self.weights = act, k, weights
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        mk = lambda shape, s: (torch.randn(shape, device="cuda", generator=g) * s).to(self.dt)
        self.x, self.wg = mk((n, H), 1.0), mk((E, H), 0.1)
        names = ["1", "3", "2"] if act == 2 else ["1", "2"]
        self.w, self.s, self.mats, self.b = {}, {}, {}, {}
        for m in names:
            w = mk((E, H, I) if m == "2" else (E, I, H), std)
            if weights == "16":
                self.w[m], self.s[m], self.mats[m] = w, None, (lambda e, w=w: w[e].double())
            elif weights == "8":
                q, s = layer.quantize_fp8(w, 128)
                self.w[m], self.s[m], self.mats[m] = q, s, (lambda e, q=q, s=s: R.decode_fp8(q[e], s[e]))
            else:
                q, s = layer.quantize_fp4(w)
                self.w[m], self.s[m], self.mats[m] = q, s, (lambda e, q=q, s=s: R.decode(q[e], s[e]))
            self.b[m] = mk((E, H if m == "2" else I), 0.3) if bias else None
        self.gate_bias = torch.randn(E, device="cuda", generator=g) * 0.2 if bias else None
        self.kw = dict(gate_fn=gate_fn, renorm=renorm)

    def run(self, x=None, **more):
        s = None if self.weights == "16" else (self.s["1"], self.s.get("3"), self.s["2"])
        return self.layer.moe_few_tokens(self.x if x is None else x, self.wg, self.w["1"], self.w.get("3"), self.w["2"],
                                         self.k, self.act, gate_bias=self.gate_bias, scales=s, b1=self.b["1"],
                                         b3=self.b.get("3"), b2=self.b["2"], **self.kw, **more)

    def check(self, got, x=None):
        torch = self.torch
        x = self.x if x is None else x
        out, idx, w = got
        want_idx, want_w = self.layer.gate_topk(x, self.wg, self.k, gate_bias=self.gate_bias, **self.kw)
        assert torch.equal(idx, want_idx), "the routing is the gate's"
        assert torch.equal(w, want_w), "the combine weights are the gate's, bit for bit"
        # bf16 weights: h as value and remainder, two half steps of bf16; else one rounding to fp16
        h_step = 2.0 ** -18 if self.weights == "16" and self.dt == torch.bfloat16 else 2.0 ** -12
        ref, bound = R.moe_few(x, idx, w, self.mats, self.b, self.act, h_step)
        R.assert_within(out, ref, bound + R.half_step(self.dt) * (ref.abs() + bound) * 1.01 + 2.0 ** -25)


FORMATS = [("16", "bfloat16"), ("16", "float16"), ("8", "bfloat16"), ("4", "bfloat16"), ("4", "float16")]


@pytest.mark.parametrize("weights,dtype", FORMATS)
@pytest.mark.parametrize("n,E,k,H,I,act", [
    (1, 8, 2, 256, 512, 2),
    (1, 1, 1, 128, 128, 0),             # one expert, the smallest sizes: most warps have no step
    (3, 8, 1, 384, 256, 1),
    (8, 4, 4, 640, 384, 2),             # every expert, one full token tile
    (9, 5, 2, 256, 640, 0),             # two token tiles
    (17, 40, 8, 512, 256, 2),
    (33, 3, 2, 384, 384, 1),            # long lists, four tiles in use of eight
    (64, 2, 1, 256, 256, 2),
    (64, 300, 16, 128, 128, 1),         # more experts than one word of lanes covers, the largest k
])
def test_layer(n, E, k, H, I, act, weights, dtype):
    c = Case(n, E, k, H, I, act, weights, dtype, gate_fn=n % 2, renorm=(n + E) % 2, bias=n % 3 == 0, seed=n)
    got = c.run()
    c.check(got)
    again = c.run()
    assert all(c.torch.equal(a, b) for a, b in zip(got, again)), "the same call gives the same bits"


@pytest.mark.parametrize("weights,dtype", [f for f in FORMATS if f[0] != "8"])
@pytest.mark.parametrize("H,I", [(64, 64), (192, 320), (1088, 192)])
def test_feature_sizes_of_64(H, I, weights, dtype):
    """Sizes at which the last step of a 4-bit row is cut in the middle and units of 64 rows end inside a scale tile."""
    for n, act in ((2, 2), (11, 0)):
        c = Case(n, 6, 2, H, I, act, weights, dtype, bias=True, seed=H + I)
        c.check(c.run())


@pytest.mark.parametrize("weights", ["16", "8", "4"])
def test_wide_layer(weights):
    c = Case(2, 8, 2, 4096, 1536, 2, weights, std=0.02, renorm=1)
    c.check(c.run())


def test_every_number_of_tokens():
    c = Case(64, 7, 3, 128, 192, 2, "16")
    for n in range(1, 65):
        x = c.x[:n]
        c.check(c.run(x), x)


def test_all_tokens_on_one_expert_and_none_on_the_others():
    torch, cp, layer = _mods()
    c = Case(64, 16, 2, 256, 256, 2, "4")
    c.gate_bias = torch.full((16,), -1000.0, device="cuda")
    c.gate_bias[5], c.gate_bias[11] = 1000.0, 900.0
    got = c.run()
    assert (got[1] == torch.tensor([5, 11], device="cuda", dtype=torch.int32)).all()
    c.check(got)


def test_equal_logits_go_to_the_lower_expert():
    torch, cp, layer = _mods()
    c = Case(5, 12, 3, 128, 128, 0)
    c.wg = c.wg[:1].expand(12, -1).contiguous()
    got = c.run()
    assert (got[1] == torch.arange(3, device="cuda", dtype=torch.int32)).all()
    c.check(got)


@pytest.mark.parametrize("weights", ["16", "8", "4"])
def test_infinities_and_nan_stay_in_their_token(weights):
    torch, cp, layer = _mods()
    c = Case(6, 4, 2, 256, 256, 2, weights)
    clean = c.run()[0]
    x = c.x.clone()
    x[2, 7], x[4, 100] = math.nan, math.inf
    out = c.run(x)[0]
    keep = [0, 1, 3, 5]
    assert torch.equal(out[keep], clean[keep])
    assert not torch.isfinite(out[[2, 4]]).any()


def test_nan_in_an_expert_that_nobody_chose_does_not_show():
    torch, cp, layer = _mods()
    c = Case(4, 8, 1, 128, 128, 2)
    c.gate_bias = torch.zeros(8, device="cuda")
    c.gate_bias[3] = -1000.0
    for m in ("1", "3", "2"):
        c.w[m][3] = math.nan
    assert torch.isfinite(c.run()[0]).all()


def test_4_bit_weights_with_scales_far_from_one():
    torch, cp, layer = _mods()
    c = Case(3, 4, 2, 256, 256, 0, "4")
    for m in ("1", "2"):
        w = R.decode(c.w[m], c.s[m]).float()
        shift = torch.randint(-50, 30, (*w.shape[:2], w.shape[2] // 32), device="cuda").float()
        w = w * torch.exp2(shift).repeat_interleave(32, -1)
        q, s = layer.quantize_fp4(w)
        c.w[m], c.s[m], c.mats[m] = q, s, (lambda e, q=q, s=s: R.decode(q[e], s[e]))
    c.check(c.run())


def test_in_graphs_with_new_inputs():
    torch, cp, layer = _mods()
    a, b = Case(3, 8, 2, 256, 256, 2, "16", seed=1), Case(20, 8, 2, 256, 256, 2, "4", seed=2)
    graphs, held = [], []
    for c in (a, b):
        c.run()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            held.append(c.run())
        graphs.append(g)
    for seed in range(3):
        for c, g, h in zip((a, b), graphs, held):
            c.x.copy_(torch.randn(c.x.shape, device="cuda"))
            g.replay()
        torch.cuda.synchronize()
        for c, h in zip((a, b), held):
            c.check(h)


def test_calls_that_overlap_on_two_streams():
    torch, cp, layer = _mods()
    cases = [Case(4, 16, 2, 1024, 1024, 2, "16", seed=1), Case(9, 16, 2, 1024, 1024, 1, "4", seed=2)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    results = [[], []]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    for _ in range(20):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                results[i].append(c.run(dev_status=status))
    torch.cuda.synchronize()
    assert int(status) == 0
    for r, w in zip(results, want):
        for got in r:
            assert all(torch.equal(p, q) for p, q in zip(got, w))


def test_no_tokens():
    torch, cp, layer = _mods()
    c = Case(4, 4, 2, 128, 128, 0)
    out, idx, w = c.run(c.x[:0])
    assert out.shape == (0, 128) and idx.shape == (0, 2) and w.shape == (0, 2)


def test_refusals():
    torch, cp, layer = _mods()
    c = Case(4, 4, 2, 128, 128, 2)
    with pytest.raises(cp.AristosError) as e:
        c.run(torch.zeros(65, 128, device="cuda", dtype=torch.bfloat16))
    assert e.value.status == 2 and "64" in str(e.value)
    c.k = 5
    with pytest.raises(cp.AristosError):
        c.run()
    c.k = 2
    with pytest.raises(ValueError):
        c.run(c.x.float())
    with pytest.raises(ValueError):
        layer.moe_few_tokens(c.x, c.wg, c.w["1"], None, c.w["2"], 2, 2)
    with pytest.raises(ValueError):
        layer.moe_few_tokens(c.x, c.wg, c.w["1"], c.w["3"][:2], c.w["2"], 2, 2)
    with pytest.raises(ValueError):
        layer.moe_few_tokens(c.x, c.wg[:, :64], c.w["1"], c.w["3"], c.w["2"], 2, 2)
    with pytest.raises(ValueError):
        layer.moe_few_tokens(c.x, c.wg, c.w["1"].view(torch.uint8), c.w["3"], c.w["2"], 2, 2)
    f = Case(4, 4, 2, 128, 128, 0, "8")
    f.dt, f.x, f.wg = torch.float16, f.x.half(), f.wg.half()
    with pytest.raises(cp.AristosError) as e:                          # 8-bit weights go with bf16 tokens
        f.run()
    assert e.value.status == 6


# ---- through the layer handle -------------------------------------------------------------------------------------------
@pytest.mark.parametrize("torch_dtype,H,I,act", [(2, 256, 320, 2), (3, 192, 256, 1), (4, 512, 256, 2), (2, 128, 128, 0)])
def test_decode_of_a_layer(torch_dtype, H, I, act):
    """decode on a handle made for many tokens: the same bits as the stage, between forwards that it leaves alone."""
    torch, cp, layer = _mods()
    E, k, n = 8, 2, 5
    cfg = cp.AristosConfig(capacity_factor=1.25, drop_tokens=1, expert_top_k=k, hidden_act=act, hidden_size=H,
                           intermediate_size=I, num_experts=E, torch_dtype=torch_dtype, tokens=256, renorm_topk=1,
                           gate_bias_zipf_s=0.3)
    c = Case(n, E, k, H, I, act, "8" if torch_dtype == 4 else "16", "float16" if torch_dtype == 3 else "bfloat16", renorm=1)
    L = layer.MoELayer(cfg)
    scales = None
    if torch_dtype == 4:
        scales = torch.cat([c.s[m].reshape(-1) for m in ("1", "3", "2") if m in c.s]).contiguous()
    weights = (c.wg, c.w["1"], c.w.get("3"), c.w["2"])
    big = torch.randn(256, H, device="cuda").to(c.dt)
    full = L.forward(big, *weights, scales=scales)
    routing = L.routing()
    c.gate_bias = layer.zipf_prior(E, 0.3).cuda()
    want = c.run()
    launches = L.launch_count
    got = L.decode(c.x, *weights, scales=scales)
    assert L.launch_count - launches == 2
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    other = L.decode(c.x, *weights, scales=scales, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    for a, b, o in zip(got, want, other):
        assert torch.equal(a, b) and torch.equal(o, b)
    L.status()
    again = L.routing()
    assert all(torch.equal(routing[m], again[m]) for m in ("topk_idx", "topk_w", "slot_of", "count"))
    assert torch.equal(L.forward(big, *weights, scales=scales), full)
    if torch_dtype != 4:
        b1, b2 = (torch.randn(E, s, device="cuda").to(c.dt) for s in (I, H))
        L.set_bias(b1=b1, b2=b2)
        c.b["1"], c.b["2"] = b1, b2
        assert torch.equal(L.decode(c.x, *weights)[0], c.run()[0])
    assert L.decode(c.x[:0], *weights, scales=scales)[0].shape == (0, H)
    with pytest.raises(cp.AristosError) as e:
        L.decode(big, *weights, scales=scales)
    assert e.value.status == 1 and "64" in str(e.value)
    with pytest.raises(ValueError):
        L.decode(c.x.float(), *weights, scales=scales)
    L.close()


def test_decode_is_refused_where_the_layer_has_none():
    torch, cp, layer = _mods()
    L = layer.MoELayer(cp.AristosConfig(hidden_size=128, intermediate_size=128, num_experts=4, torch_dtype=0, tokens=128))
    x, wg = torch.zeros(2, 128, device="cuda"), torch.zeros(4, 128, device="cuda")
    w = torch.zeros(4, 128, 128, device="cuda")
    with pytest.raises(cp.AristosError) as e:
        L.decode(x, wg, w, None, w)
    assert e.value.status == 6
    L.close()


def test_module_decode():
    torch, cp, layer = _mods()
    from cuplayground_b200.torch_op import AristosMoE
    cfg = cp.AristosConfig(expert_top_k=2, hidden_act=2, hidden_size=256, intermediate_size=512, num_experts=8,
                           torch_dtype=2, tokens=512, renorm_topk=1)
    m = AristosMoE(cfg)
    x = torch.randn(2, 3, 256, device="cuda", dtype=torch.bfloat16)
    out = m.decode(x)
    want = layer.moe_few_tokens(x.reshape(6, 256), m.w_gate, m.w1, m.w3, m.w2, 2, 2, renorm=1)[0]
    assert torch.equal(out, want.reshape(2, 3, 256))
    m.close()


# ---- 4-bit weights: the split into terms, the parts of K, the order of tiles ----------------------------------------------
@pytest.mark.parametrize("n,E,k,H,I,act", [
    (5, 3, 2, 64, 1024, 0),             # more parts of K asked for than there are whole stages
    (3, 4, 2, 128, 1600, 2),            # parts of unequal length, the last stage cut
    (24, 64, 8, 512, 1024, 2),          # several rounds of up tiles, the CTAs with one tile less are dealt more
    (24, 64, 8, 2048, 512, 1),          # the same with long up and short down tiles
    (64, 3, 3, 320, 448, 2),            # four passes over every expert's weights
    (64, 512, 16, 128, 192, 0),         # the most experts and choices
])
def test_tiles_of_4_bit_weights(n, E, k, H, I, act):
    c = Case(n, E, k, H, I, act, "4", gate_fn=n % 2, bias=n % 3 == 0, seed=n + H)
    got = c.run()
    c.check(got)
    again = c.run()
    assert all(c.torch.equal(a, b) for a, b in zip(got, again)), "the same call gives the same bits"


def test_most_experts_and_choices():
    c = Case(64, 512, 16, 128, 64, 1, "16", seed=3)
    c.check(c.run())


def test_4_bit_products_scale_with_the_tokens():
    """Everything behind a split is a power of two away: without biases, with ReLU and the same routing, tokens times 2^a give
    outputs times 2^a, bit for bit, as long as all terms have a scale (2^-127 or more). Of tokens near 2^-110 the terms
    below 2^-127 are left out: some 16 bits stay, of which the tolerance asks for 8 (the output is bf16)."""
    torch, cp, layer = _mods()
    c = Case(7, 6, 2, 256, 320, 0, "4", seed=9)
    c.wg = torch.zeros_like(c.wg)
    want = c.run()[0].double()
    for a in (-60, -13, 1, 40, 60):
        got = c.run((c.x.double() * 2.0 ** a).to(c.dt))[0].double()
        assert torch.equal(got, want * 2.0 ** a), a
    got = c.run((c.x.double() * 2.0 ** -110).to(c.dt))[0].double() * 2.0 ** 110
    scale = want.abs().amax()
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -9 * scale).all()


def test_4_bit_weights_meet_all_24_bits_of_the_hidden_activations():
    """W1 picks columns, so h is known exactly: every block of 32 holds one large and 31 small numbers, and W2 cancels the
    large one. What is left are the small numbers, 2^-15 of the largest: an h rounded to 11 or 16 bits of its block would
    lose them. Terms are off by at most 2^-23 of a block's largest magnitude (half a unit of the eighth: 2^(s0 - 22), the
    largest being 2^(s0 + 1) or more), i.e. 2^-8 of the small numbers; fp32 sums of K = 128 add 128 * 2^-24 * 2^15 of them
    at most where the large ones cancel: one of each sign per two blocks, exactly equal, so nothing is rounded on the way
    but what is smaller than 2^-24 of the large ones."""
    torch, cp, layer = _mods()
    H, n = 128, 4
    c = Case(n, 1, 1, H, H, 0, "4", seed=4)
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = 1.0 + torch.randint(0, 128, (n, H), device="cuda", generator=g).float() / 128       # 8 bits, in [1, 2)
    x[:, 0::32] = 2.0 ** 15
    c.x = x.to(c.dt)
    assert torch.equal(c.x.float(), x)
    eye = torch.eye(H, device="cuda")[None]
    w2 = torch.zeros(1, H, H, device="cuda")
    for r in range(H):
        for b in range(H // 32):
            w2[0, r, 32 * b] = 1.0 if b % 2 else -1.0                                       # the large ones cancel
        w2[0, r, 32 * (r % 4) + 1 + r % 31] += 1.0
    for m, w in (("1", eye), ("2", w2)):
        q, s = layer.quantize_fp4(w)
        assert torch.equal(layer.dequantize_fp4(q, s, torch.float32), w)
        c.w[m], c.s[m], c.mats[m] = q, s, None
    out = c.run()[0].double()
    want = torch.stack([x[:, 32 * (r % 4) + 1 + r % 31] for r in range(H)], 1).double()
    # 2^-23 * 2^15 per number of the split, twice (x and h); sums within 2^-24 * 2^16 per added pair of large numbers, at most 8
    bound = 2 * 2.0 ** -8 + 8 * 2.0 ** -8 + 2.0 ** -9 * want
    assert ((out - want).abs() <= bound).all(), (out - want).abs().max()


def test_4_bit_calls_that_overlap_on_two_streams():
    torch, cp, layer = _mods()
    cases = [Case(6, 16, 2, 512, 512, 2, "4", seed=1), Case(33, 16, 3, 512, 1024, 1, "4", seed=2)]
    want = [c.run() for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    torch.cuda.synchronize()
    results = [[], []]
    for _ in range(20):
        for i, (c, st) in enumerate(zip(cases, streams)):
            with torch.cuda.stream(st):
                results[i].append(c.run(dev_status=status))
    torch.cuda.synchronize()
    assert int(status) == 0
    for r, w in zip(results, want):
        for got in r:
            assert all(torch.equal(p, q) for p, q in zip(got, w))


def test_a_nan_scale_of_a_4_bit_weight_row_reaches_its_expert_only():
    torch, cp, layer = _mods()
    c = Case(6, 4, 1, 256, 256, 0, "4", seed=6)
    clean, idx, _ = c.run()
    for m, row in (("2", 77), ("1", 200)):
        s = c.s[m].clone()
        e = int(idx[0, 0])
        s[e, row // 128, 1, row % 32, row // 32 % 4, 2] = 255
        keep, c.s[m] = c.s[m], s
        out, again, _ = c.run()
        c.s[m] = keep
        assert torch.equal(again, idx)
        mine = (idx == e).any(1)
        assert torch.equal(out[~mine], clean[~mine])
        if m == "2":
            assert torch.isnan(out[mine][:, row]).all()
            rest = torch.arange(256, device="cuda") != row
            assert torch.equal(out[mine][:, rest], clean[mine][:, rest])
        else:
            assert torch.isnan(out[mine]).all()                     # that column of h is NaN, and every output reads it


def test_4_bit_layer_beside_4_bit_products():
    """Both kernels want all of an SM's tensor memory: whoever comes second waits, nobody waits for the other's end."""
    torch, cp, layer = _mods()
    c = Case(20, 32, 4, 512, 512, 2, "4", seed=8)
    g = torch.Generator(device="cuda")
    g.manual_seed(9)
    q = [layer.quantize_fp4(torch.randn(s, device="cuda", generator=g)) for s in ((8, 300, 512), (8, 768, 512))]
    count = torch.tensor([300, 0, 1, 129, 256, 299, 64, 200], dtype=torch.int32, device="cuda")
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    product = lambda: layer.expert_product_fp4(*q[0], count, *q[1], dev_status=status)
    want, want_y = c.run(), product()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got, got_y = [], []
    for _ in range(30):
        with torch.cuda.stream(streams[0]):
            got.append(c.run(dev_status=status))
        with torch.cuda.stream(streams[1]):
            got_y.append(product())
    torch.cuda.synchronize()
    assert int(status) == 0
    assert all(torch.equal(a, b) for r in got for a, b in zip(r, want))
    assert all(torch.equal(y, want_y) for y in got_y)


def test_decode_in_a_graph():
    torch, cp, layer = _mods()
    cfg = cp.AristosConfig(expert_top_k=2, hidden_act=2, hidden_size=256, intermediate_size=320, num_experts=8, torch_dtype=2,
                           tokens=256, renorm_topk=1)
    c = Case(9, 8, 2, 256, 320, 2, renorm=1, seed=11)
    weights = (c.wg, c.w["1"], c.w["3"], c.w["2"])
    L = layer.MoELayer(cfg)
    L.decode(c.x, *weights)                                          # allocates the layer's workspace
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = L.decode(c.x, *weights)
    for seed in range(3):
        c.x.copy_(torch.randn(c.x.shape, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, c.run()))
    L.status()
    L.close()

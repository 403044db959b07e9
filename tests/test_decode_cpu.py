"""What MoELayer.decode refuses before anything reaches the library: needs no GPU, nothing is launched."""
import pytest

torch = pytest.importorskip("torch")

import cuplayground_b200 as cp
import cuplayground_b200.layer as layer


def _layer(**kw):
    """A layer object without a handle: a call that got as far as the library would end in an AttributeError."""
    cfg = cp.AristosConfig(**{**dict(hidden_size=512, intermediate_size=256, num_experts=4, expert_top_k=2, hidden_act=2,
                                     torch_dtype=2, tokens=128), **kw})
    L = object.__new__(layer.MoELayer)
    L.cfg, L._lib, L._h, L.device = cfg, None, None, 0
    L.H, L.I, L.E, L.E_local, L.k = cfg.hidden_size, cfg.intermediate_size, cfg.num_experts, cfg.num_experts, cfg.expert_top_k
    L.dtype = layer._TORCH_DTYPE[cfg.torch_dtype]
    return L


def _args(L, weights=None):
    dt = weights or L.dtype
    z = lambda *s: torch.zeros(s).to(dt)
    return dict(x=torch.zeros(3, 512, dtype=L.dtype), w_gate=torch.zeros(4, 512, dtype=L.dtype), w1=z(4, 256, 512), w3=z(4, 256, 512),
                w2=z(4, 512, 256))


def test_tensors_off_the_gpu_are_refused():
    L = _layer()
    with pytest.raises(ValueError, match="CUDA device"):
        L.decode(**_args(L))


BF = torch.bfloat16


@pytest.mark.parametrize("name,value", [
    ("x", torch.zeros(512, dtype=BF)), ("x", torch.zeros(3, 256, dtype=BF)), ("x", torch.zeros(3, 512)),
    ("w_gate", torch.zeros(2, 512, dtype=BF)), ("w_gate", torch.zeros(4, 512)),
    ("w1", torch.zeros(2, 256, 512, dtype=BF)), ("w1", torch.zeros(4, 256, 512, dtype=torch.float16)),
    ("w1", torch.zeros(4, 512, 256, dtype=BF)), ("w3", torch.zeros(4, 128, 512, dtype=BF)), ("w2", torch.zeros(4, 256, 512, dtype=BF)),
    ("gate_bias", torch.zeros(3)), ("gate_bias", torch.zeros(4, dtype=BF)),
    ("out", torch.zeros(2, 512, dtype=BF)), ("out", torch.zeros(3, 512)),
])
def test_tensors_of_another_shape_or_type_are_refused(name, value):
    L = _layer()
    with pytest.raises(ValueError, match=name):
        L.decode(**{**_args(L), name: value})


@pytest.mark.parametrize("scales", [torch.zeros(3 * 4 * 2 * 4 - 1), torch.zeros(3 * 4 * 2 * 4, dtype=BF), torch.zeros(2 * 4 * 2 * 4)])
def test_fp8_scales_that_are_too_few_or_of_another_type_are_refused(scales):
    L = _layer(torch_dtype=4)
    with pytest.raises(ValueError, match="scales"):
        L.decode(**_args(L, torch.uint8), scales=scales)


def test_fp8_weights_are_codes():
    L = _layer(torch_dtype=4)
    scales = torch.zeros(3 * 4 * 2 * 4)
    with pytest.raises(ValueError, match="w1"):
        L.decode(**_args(L), scales=scales)
    for codes in (torch.uint8, torch.float8_e4m3fn):               # as they are, or typed: as far as the device
        with pytest.raises(ValueError, match="CUDA device"):
            L.decode(**_args(L, codes), scales=scales)


def test_e4m3_scales_need_no_more_than_their_own_alignment():
    """Scales may be parts of one tensor [s1 | s3 | s2], as a layer's are: with an odd number of blocks per matrix the second and
    third start on 4 bytes. The kernels read them one at a time. (A workspace of 0 bytes is refused last: nothing is launched.)"""
    import ctypes as C
    lib = cp._lib.load()
    P = 1 << 20
    call = lambda s1, s3, s2, wdt: lib.aristos_moe_few_tokens(P, P, None, P, P, P, s1, s3, s2, None, None, None, 4, 128, 128, 3, 2, 0,
                                                              0, 2, 2, wdt, P, None, None, P, 0, None, None)
    WORKSPACE, INVALID = 7, 1
    assert call(P, P + 12, P + 24, 4) == WORKSPACE
    assert call(P + 4, P + 4, P + 4, 4) == WORKSPACE
    assert call(P + 2, P, P, 4) == INVALID and call(P, P, P + 1, 4) == INVALID and call(P, P + 2, P, 4) == INVALID
    assert call(P, P + 12, P + 24, 5) == INVALID               # scale tiles of 4-bit weights travel in pieces of 16 bytes

"""decode's workspace is its own: a layer that never decodes needs none, and a caller's buffer of the forward's size stays enough."""
import ctypes as C

import pytest

pytestmark = pytest.mark.gpu


def _mods():
    import torch
    import cuplayground_b200 as cp
    import cuplayground_b200.layer as layer
    return torch, cp, layer


def _layer(cp, layer, **kw):
    return layer.MoELayer(cp.AristosConfig(**{**dict(expert_top_k=2, hidden_act=0, hidden_size=128, intermediate_size=256, num_experts=8,
                                                     torch_dtype=2, tokens=1024), **kw}))


def _weights(torch, E=8, H=128, I=256):
    mk = lambda *s: (torch.randn(s, device="cuda") * 0.1).bfloat16()
    return mk(E, H), mk(E, I, H), None, mk(E, H, I)


def test_the_layers_workspace_does_not_hold_decodes():
    """64 more columns of h, for every expert's rows: nothing else depends on the intermediate size."""
    torch, cp, layer = _mods()
    a, b = _layer(cp, layer), _layer(cp, layer, intermediate_size=320)
    h = lambda I: -(-8 * a.cap * I * 2 // 1024) * 1024
    assert b.workspace_bytes - a.workspace_bytes == h(320) - h(256)
    lib = cp._lib.load()
    assert lib.aristos_moe_decode_workspace_bytes(b._h) > lib.aristos_moe_decode_workspace_bytes(a._h) > 0
    a.close(), b.close()


def test_create_says_nothing_about_a_decode_that_the_layer_does_not_have():
    torch, cp, layer = _mods()
    lib = cp._lib.load()
    assert lib.aristos_moe_set_workspace(None, None, 0) != 0
    assert lib.aristos_quantize_fp4(None, -1, 0, 64, 2, None, None, None) != 0
    before = lib.aristos_last_error()
    L = _layer(cp, layer, num_experts=600)
    assert lib.aristos_last_error() == before and b"quantize" in before
    assert lib.aristos_moe_decode_workspace_bytes(L._h) == 0
    ws = torch.empty(1 << 20, dtype=torch.uint8, device="cuda")
    assert lib.aristos_moe_set_decode_workspace(L._h, C.c_void_p(ws.data_ptr()), 1 << 20) == 6
    L.close()


def test_a_callers_decode_workspace():
    torch, cp, layer = _mods()
    w = _weights(torch)
    x = torch.randn(7, 128, device="cuda").bfloat16()
    L = _layer(cp, layer)
    want = L.decode(x, *w)
    lib = cp._lib.load()
    n = lib.aristos_moe_decode_workspace_bytes(L._h)
    ws = torch.full((n + 512,), 0xAB, dtype=torch.uint8, device="cuda")
    base = (ws.data_ptr() + 255) // 256 * 256
    off = base - ws.data_ptr()
    setws = lambda p, b: lib.aristos_moe_set_decode_workspace(L._h, C.c_void_p(p), b)
    assert setws(base, n - 1) == 7 and setws(base + 16, n) == 1 and setws(None, n) == 1
    assert all(torch.equal(a, b) for a, b in zip(L.decode(x, *w), want))           # still the layer's own
    assert setws(base, n) == 0
    assert all(torch.equal(a, b) for a, b in zip(L.decode(x, *w), want))
    torch.cuda.synchronize()
    assert (ws[:off] == 0xAB).all() and (ws[off + n:] == 0xAB).all() and not (ws[off:off + n] == 0xAB).all()
    L.close()


def test_the_first_decode_may_be_captured_where_torch_has_the_workspaces():
    torch, cp, layer = _mods()
    w = _weights(torch)
    x = torch.randn(7, 128, device="cuda").bfloat16()
    ref = _layer(cp, layer)
    L = _layer(cp, layer)
    L.use_torch_workspace()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = L.decode(x, *w)
    for _ in range(2):
        x.copy_(torch.randn(7, 128, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, ref.decode(x, *w)))
    L.close(), ref.close()


def test_a_torch_workspace_belongs_to_the_stream_of_the_first_decode():
    """A block that the current stream has just given back may still be in use there: the workspace of a decode on another stream
    must not be that block."""
    torch, cp, layer = _mods()
    w = _weights(torch)
    x = torch.randn(7, 128, device="cuda").bfloat16()
    L = _layer(cp, layer)
    L.use_torch_workspace()
    n = int(cp._lib.load().aristos_moe_decode_workspace_bytes(L._h))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    given_back = torch.empty(n, dtype=torch.uint8, device="cuda")
    at = given_back.data_ptr()
    del given_back
    L.decode(x, *w, stream=side)
    assert L._decode_ws.data_ptr() != at
    torch.cuda.synchronize()
    L.close()

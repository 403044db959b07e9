"""Argument checks of the 4-bit operators and of the few-token layer that need no GPU (every refusal comes before the first
CUDA call), and the reference that their GPU tests are held to."""
import ctypes as C

import numpy as np
import pytest

import fp4_reference as R


@pytest.fixture(scope="module")
def lib():
    from cuplayground_b200 import build
    build.build_library()
    import cuplayground_b200
    return cuplayground_b200._lib.load()


P = C.c_void_p(1 << 20)              # never dereferenced: 16-byte aligned, refused or returned before any use
ODD = C.c_void_p((1 << 20) + 4)


def test_scale_bytes(lib):
    assert lib.aristos_fp4_scale_bytes(1, 1, 64) == 512
    assert lib.aristos_fp4_scale_bytes(3, 129, 192) == 3 * 2 * 2 * 512
    assert lib.aristos_fp4_scale_bytes(0, 128, 128) == 0
    assert lib.aristos_fp4_scale_bytes(1, 0, 128) == 0
    assert lib.aristos_fp4_scale_bytes(-1, 128, 128) == 0


@pytest.mark.parametrize("args,status", [
    ((P, 1, 16, 96, 2, P, P), 1),                 # columns not a multiple of 64
    ((P, -1, 16, 64, 2, P, P), 1),
    ((P, 1, -1, 64, 2, P, P), 1),
    ((P, 1, 16, 0, 2, P, P), 1),
    ((None, 1, 16, 64, 2, P, P), 1),
    ((P, 1, 16, 64, 2, None, P), 1),
    ((ODD, 1, 16, 64, 2, P, P), 1),
    ((P, 1, 16, 64, 2, P, ODD), 1),
    ((P, 1, 1 << 40, 64, 2, P, P), 2),
    ((P, 1, 0, 64, 2, P, P), 0),                  # nothing to do
    ((None, 0, 16, 64, 2, None, None), 0),
])
def test_quantize_refusals(lib, args, status):
    src, mats, rows, cols, dt, q, s = args
    assert lib.aristos_quantize_fp4(src, mats, rows, cols, dt, q, s, None) == status
    assert lib.aristos_dequantize_fp4(q, s, mats, rows, cols, dt, src, None) == status


def _product(lib, **kw):
    a = dict(aq=P, sa=P, count=P, groups=2, rows=100, experts=2, bq=P, sb=P, N=128, K=128, dt=2, y=P)
    a.update(kw)
    return lib.aristos_expert_product_fp4(a["aq"], a["sa"], a["count"], a["groups"], a["rows"], a["experts"], a["bq"], a["sb"],
                                          a["N"], a["K"], a["dt"], a["y"], None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(N=100), 2), (dict(K=96), 2), (dict(N=0), 1), (dict(groups=-1), 1), (dict(experts=0), 1), (dict(rows=-5), 1),
    (dict(groups=1025), 2), (dict(dt=4), 6), (dict(dt=5), 6), (dict(aq=None), 1), (dict(count=None), 1), (dict(y=ODD), 1),
    (dict(sb=ODD), 1), (dict(groups=1024, rows=1 << 30), 2), (dict(groups=0, aq=None), 0), (dict(rows=0, y=None), 0),
])
def test_product_refusals(lib, kw, status):
    assert _product(lib, **kw) == status


def _ffn(lib, **kw):
    a = dict(xq=P, sx=P, count=P, groups=2, rows=100, experts=2, w1=P, s1=P, w3=P, s3=P, w2=P, s2=P, hq=P, sh=P, y=P, H=128,
             I=192, act=2, dt=2)
    a.update(kw)
    return lib.aristos_expert_ffn_fp4(*[a[n] for n in ("xq", "sx", "count", "groups", "rows", "experts", "w1", "s1", "w3", "s3",
                                                       "w2", "s2", "hq", "sh", "y", "H", "I", "act", "dt")], None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(act=3), 1), (dict(act=-1), 1), (dict(H=96), 2), (dict(I=100), 2), (dict(w3=None), 1), (dict(s3=None), 1),
    (dict(w3=ODD), 1), (dict(hq=None), 1), (dict(sh=ODD), 1), (dict(dt=1), 6), (dict(groups=2000), 2), (dict(groups=0), 0),
])
def test_ffn_refusals(lib, kw, status):
    assert _ffn(lib, **kw) == status


def _few(lib, **kw):
    a = dict(x=P, wg=P, gb=None, w1=P, w3=P, w2=P, s1=None, s3=None, s2=None, b1=None, b3=None, b2=None, tokens=4, H=128, I=128,
             E=8, k=2, gate=0, renorm=0, act=2, dt=2, wdt=2, out=P, idx=None, w=None, ws=P, bytes=1 << 30)
    a.update(kw)
    return lib.aristos_moe_few_tokens(*a.values(), None, None)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=65), 2), (dict(tokens=-1), 1), (dict(H=96), 2), (dict(I=32), 2), (dict(k=9), 2), (dict(k=0), 1),
    (dict(E=2000, k=2), 2), (dict(E=64, k=17), 2), (dict(dt=0, wdt=0), 6), (dict(dt=1, wdt=1), 6), (dict(dt=2, wdt=3), 6),
    (dict(dt=3, wdt=4, s1=P, s3=P, s2=P), 6), (dict(wdt=4), 1), (dict(wdt=5, s1=P, s2=P), 1),
    (dict(wdt=4, s1=P, s3=P, s2=P, H=192), 2), (dict(w3=None), 1), (dict(act=3), 1), (dict(gate=2), 1), (dict(out=None), 1),
    (dict(x=ODD), 1), (dict(w3=ODD), 1), (dict(ws=None), 1), (dict(bytes=100), 7), (dict(tokens=0, x=None, ws=None), 0),
    (dict(E=1024, H=64 * (1 << 20), I=64 * (1 << 20)), 2),
])
def test_few_tokens_refusals(lib, kw, status):
    assert _few(lib, **kw) == status


def test_few_tokens_workspace(lib):
    size = lib.aristos_moe_few_tokens_workspace_bytes
    assert size(4, 128, 128, 8, 2) > 0 and size(64, 7168, 2048, 256, 8) > size(1, 7168, 2048, 256, 8)
    assert size(65, 128, 128, 8, 2) == 0 and size(4, 100, 128, 8, 2) == 0 and size(4, 128, 128, 8, 9) == 0


def test_reference_rounds_to_nearest_even():
    import torch
    v = torch.zeros(1, 32, dtype=torch.float64)
    v[0, :12] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, -0.25, -3.5, 7.9, 0.3, 4.0])
    want = [0, 1, 1, 2, 2, 4, 4, 0, -4, 6, 0.5, 4]
    assert R.rounded(v)[0, :12].tolist() == want and R.block_scale(v).item() == 127


def test_reference_finds_a_planted_mistake():
    """A sum with one term left out, or one element of the hidden activations a step off, is outside the bounds."""
    import torch
    torch.manual_seed(0)
    x, w1, w2 = torch.randn(4, 128).double(), torch.randn(192, 128).double() * 0.1, torch.randn(64, 192).double() * 0.1
    x, w1, w2 = R.rounded(x), R.rounded(w1), R.rounded(w2)
    y, bound = R.ffn_fp4(x, w1, None, w2, 0)
    R.assert_within(y, y, bound + 1e-30)
    short = R.rounded(torch.relu(x @ w1.T))
    short[:, 100] += 1.0
    with pytest.raises(AssertionError):
        R.assert_within(short @ w2.T, y, bound + 1e-30)
    with pytest.raises(AssertionError):
        R.assert_within(x[:, :-1] @ w1[:, :-1].T, x @ w1.T, R.dot_bound(x, w1.T))


def test_a_status_word_of_another_type_is_refused():
    """The kernels OR 32 bits into it: one byte would be followed by somebody else's memory."""
    torch = pytest.importorskip("torch")
    import cuplayground_b200.layer as layer
    u8 = lambda *shape: torch.zeros(shape, dtype=torch.uint8)
    tiles = lambda *lead: u8(*lead, 1, 1, 32, 4, 4)
    count = torch.zeros(1, dtype=torch.int32)
    for status in (u8(1), torch.zeros(0, dtype=torch.int32), torch.zeros(1)):
        with pytest.raises(ValueError, match="dev_status"):
            layer.expert_product_fp4(u8(1, 4, 32), tiles(1), count, u8(1, 64, 32), tiles(1), dev_status=status)
        with pytest.raises(ValueError, match="dev_status"):
            layer.expert_ffn_fp4(u8(1, 4, 32), tiles(1), count, u8(1, 64, 32), tiles(1), None, None, u8(1, 64, 32), tiles(1), 0,
                                 dev_status=status)
        x = torch.zeros(2, 64, dtype=torch.bfloat16)
        w = torch.zeros(3, 64, 64, dtype=torch.bfloat16)
        with pytest.raises(ValueError, match="dev_status"):
            layer.moe_few_tokens(x, x.new_zeros(3, 64), w, None, w, 1, 0, dev_status=status)

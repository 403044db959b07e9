"""NaN in a token of decode: reported where a forward of the layer reports it, kept in the token's own output by every activation."""
import math

import pytest

pytestmark = pytest.mark.gpu


def _layer(E, act=0, torch_dtype=2):
    import torch
    import cuplayground_b200 as cp
    import cuplayground_b200.layer as layer
    H, I = 128, 192
    L = layer.MoELayer(cp.AristosConfig(expert_top_k=2, hidden_act=act, hidden_size=H, intermediate_size=I, num_experts=E,
                                        torch_dtype=torch_dtype, tokens=256))
    dt = L.dtype
    mk = lambda *s: (torch.randn(s, device="cuda") * 0.1).to(dt)
    return torch, cp, L, (mk(E, H), mk(E, I, H), mk(E, I, H) if act == 2 else None, mk(E, H, I)), mk(6, H)


@pytest.mark.parametrize("torch_dtype", [2, 3])
@pytest.mark.parametrize("E,reported", [(64, True), (8, False)])         # the layer's gate screens 64 to 256 experts
def test_nan_logits_of_a_decode_are_reported(E, reported, torch_dtype):
    torch, cp, L, w, x = _layer(E, torch_dtype=torch_dtype)
    L.decode(x, *w)
    L.status()                                                           # numbers only
    x[3, 7] = math.nan
    L.decode(x, *w)
    if reported:
        with pytest.raises(cp.AristosError) as e:
            L.status()
        assert e.value.status == 12 and "NaN" in str(e.value)
    L.status()                                                           # reported once
    wg = w[0].clone()
    wg[5] = math.nan                                                     # one expert's logits: every token has others
    x[3, 7] = 0.0
    L.decode(x, wg, *w[1:])
    L.status()
    L.close()


@pytest.mark.parametrize("act", [0, 1, 2])
def test_a_nan_token_stays_nan(act):
    torch, cp, L, w, x = _layer(8, act)
    clean = L.decode(x, *w)[0].clone()
    x[3, 7] = math.nan
    out = L.decode(x, *w)[0]
    assert torch.isnan(out[3]).all()
    rest = [0, 1, 2, 4, 5]
    assert torch.equal(out[rest], clean[rest])
    L.close()

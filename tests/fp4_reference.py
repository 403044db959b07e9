"""The microscaled 4-bit format, the expert FFN and the layer for few tokens in 64 bits (torch float64, any device), with
bounds on what fp32 arithmetic may add. Used by the tests of the 4-bit operators and of the few-token layer."""
from __future__ import annotations

import math

import torch

GRID = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64 from the exponent bits, e in -1022 .. 1023."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def scale_bytes(tiles: torch.Tensor, rows: int, blocks: int) -> torch.Tensor:
    """Scale tiles (..., rt, ct, 32, 4, 4) -> bytes (..., rows, blocks)."""
    r = torch.arange(rows, device=tiles.device)[:, None]
    b = torch.arange(blocks, device=tiles.device)[None, :]
    return tiles[..., r // 128, b // 4, r % 32, r % 128 // 32, b % 4]


def block_scale(v: torch.Tensor) -> torch.Tensor:
    """Scale byte of every block of 32: floor(log2 of the largest magnitude) + 125, at least 0; 255 for infinities and NaN."""
    b = v.double().reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    top = b.abs().amax(-1)
    bad = ~torch.isfinite(b).all(-1)
    e = (torch.where(bad, 1.0, top).view(torch.int64) >> 52) - 1023
    return torch.where(bad, 255, (e + 125).clamp(min=0))


def round_with(v: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """Values of v (..., cols) rounded to e2m1 times 2^(s - 127), s (..., cols / 32), in float64."""
    b = v.double().reshape(*v.shape[:-1], v.shape[-1] // 32, 32)
    x = pow2(s - 127)[..., None]
    m = torch.nan_to_num(b / x, 0.0, 0.0, 0.0).abs()
    step = torch.where(m < 2, 0.5, torch.where(m < 4, 1.0, 2.0)).double()
    m = (torch.round(m / step) * step).clamp(max=6.0)
    out = torch.copysign(m, b) * x
    return torch.where((s == 255)[..., None], math.nan, out).reshape(v.shape)


def rounded(v: torch.Tensor) -> torch.Tensor:
    return round_with(v, block_scale(v))


def decode(q: torch.Tensor, tiles: torch.Tensor) -> torch.Tensor:
    """Values of codes (..., rows, cols / 2) with scale tiles, in float64."""
    nib = torch.stack([q & 15, q >> 4], -1).reshape(*q.shape[:-1], 2 * q.shape[-1]).long()
    v = torch.tensor(GRID, dtype=torch.float64, device=q.device)[nib & 7] * torch.where(nib >= 8, -1.0, 1.0).double()
    s = scale_bytes(tiles, v.shape[-2], v.shape[-1] // 32).long()
    x = torch.where(s == 255, math.nan, pow2(s - 127))
    return v * x.repeat_interleave(32, -1)


def decode_fp8(q: torch.Tensor, s: torch.Tensor) -> torch.Tensor:
    """e4m3 codes (..., rows, cols) with one fp32 scale per 128 x 128."""
    s = s.double().repeat_interleave(128, -2).repeat_interleave(128, -1)
    return q.view(torch.float8_e4m3fn).double() * s[..., : q.shape[-2], : q.shape[-1]]


def dot_bound(a: torch.Tensor, bt: torch.Tensor) -> torch.Tensor:
    """How far an fp32 sum of the products a . bt may be off in any order: every one of the K additions is off by at most a
    whole step of 2^-23 (a tensor core may truncate) of a partial sum that the sum of magnitudes bounds."""
    return a.shape[-1] * 2.0 ** -23 * (a.abs() @ bt.abs())


def half_step(dtype: torch.dtype) -> float:
    return torch.finfo(dtype).eps / 2


def act64(g, u, act):
    if act == 2:
        return g * torch.sigmoid(g) * u
    return 0.5 * g * torch.erfc(-g / math.sqrt(2.0)) if act == 1 else torch.relu(g)


def act_bound(g, u, dg, du, act):
    """|act(g + dg, u + du) - act(g, u)| at most: the slopes of silu and gelu are below 1.13; the function itself is good
    to 2^-19 of its value plus 2^-21 of its argument (fast exponential and division, erf in fp32)."""
    if act == 2:
        s = (g * torch.sigmoid(g)).abs()
        return 1.13 * dg * (u.abs() + du) + s * du + (2.0 ** -19 * s + 2.0 ** -21 * g.abs()) * u.abs()
    own = 0.0 if act == 0 else 2.0 ** -21 * g.abs() + 2.0 ** -19 * act64(g, u, act).abs()
    return 1.13 * dg + own


def ffn_fp4(x, w1, w3, w2, act):
    """One expert on decoded float64 operands: (y, how far fp32 sums may move it, the roundings that may flip among it)."""
    g, dg = x @ w1.T, dot_bound(x, w1.T)
    u, du = (x @ w3.T, dot_bound(x, w3.T)) if act == 2 else (None, None)
    h, dh = act64(g, u, act), act_bound(g, u, dg, du, act)
    y = rounded(h) @ w2.T
    # a rounding may go either way where h +- dh straddles a border, and a block's scale where its maximum does
    lo = hi = rounded(h)
    for s in (block_scale(h), block_scale((h.abs() - dh).clamp(min=0)), block_scale(h.abs() + dh)):
        for v in (h - dh, h, h + dh):
            r = round_with(v, s)
            lo, hi = torch.minimum(lo, r), torch.maximum(hi, r)
    return y, (hi - lo) @ w2.T.abs() + dot_bound(torch.maximum(lo.abs(), hi.abs()), w2.T)


def moe_few(x, idx, w, mats, biases, act, h_step):
    """out (n, H) and its bound for given routing; mats: {"1", "3", "2"} -> (E, ...) float64 (or a function of e);
    biases the same or None; h_step: relative error of the hidden activations as an operand of the down projection.
    Operands may be scaled fp16 numbers (largest magnitude in [2^14, 2^15), smallest step 2^-24): what is far below the
    largest of its row is off by at most 2^-38 of that."""
    n, k = idx.shape
    y = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    d = torch.zeros_like(y)
    get = lambda m, e: mats[m](e) if callable(mats[m]) else mats[m][e]
    bias = lambda m, e: 0.0 if biases.get(m) is None else biases[m][e].double()
    for e in sorted(set(idx.reshape(-1).tolist())):
        who, j = (idx == e).nonzero(as_tuple=True)
        rows = x[who].double()
        w1, w2 = get("1", e), get("2", e)
        g, dg = rows @ w1.T + bias("1", e), dot_bound(rows, w1.T)
        far = 2.0 ** -38 * rows.abs().amax(1, keepdim=True)
        dg = dg + 2.0 ** -23 * g.abs() + far * w1.abs().sum(1)
        u = du = None
        if act == 2:
            w3 = get("3", e)
            u, du = rows @ w3.T + bias("3", e), dot_bound(rows, w3.T)
            du = du + 2.0 ** -23 * u.abs() + far * w3.abs().sum(1)
        h = act64(g, u, act)
        dh = act_bound(g, u, dg, du, act) + h_step * h.abs() + 2.0 ** -38 * h.abs().amax(1, keepdim=True)
        out = h @ w2.T + bias("2", e)
        do = dh @ w2.T.abs() + dot_bound(h, w2.T) + 2.0 ** -23 * out.abs()
        p = w[who, j].double()[:, None]
        y.index_add_(0, who, p * out)
        d.index_add_(0, who, p * (do + (k + 1) * 2.0 ** -23 * out.abs()))
    return y, d


def assert_within(got, ref, bound, what=""):
    err = (got.double() - ref).abs()
    bad = ~(err <= bound)
    if bad.any():
        at = bad.nonzero()[0].tolist()
        worst = (err / bound).nan_to_num(math.inf).max().item()
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound (worst {worst:.3g} times it); first at "
                             f"{at}: {got[tuple(at)].item()} against {ref[tuple(at)].item()} +- {bound[tuple(at)].item()}")

"""Host-side mirror of the C ABI: the MoE layer handle and the stage entry points on torch tensors.

torch is used for device memory, streams and (by callers) torch.distributed; every computation goes through
libaristos_moe.so. Nothing here falls back to PyTorch ops."""
from __future__ import annotations

import ctypes as C
import functools
from typing import Optional

import torch

from . import _lib
from .config import AristosConfig

_TORCH_DTYPE = {_lib.DTYPE_F32: torch.float32, _lib.DTYPE_TF32: torch.float32, _lib.DTYPE_BF16: torch.bfloat16,
                _lib.DTYPE_F16: torch.float16, _lib.DTYPE_FP8_E4M3: torch.bfloat16}   # fp8: activations are bf16
# storage type -> dtype code; fp32 tensors mean exact fp32 math unless a call asks for tf32 explicitly
_ARISTOS_DTYPE = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_F16}


def _ptr(t: Optional[torch.Tensor]):
    if t is None:
        return None
    if not t.is_contiguous():
        raise ValueError("tensors passed to the C ABI must be contiguous")
    return C.c_void_p(t.data_ptr())


def _stream_ptr(stream: Optional[torch.cuda.Stream] = None):
    s = stream if stream is not None else torch.cuda.current_stream()
    return C.c_void_p(s.cuda_stream)


def _dt(t: torch.Tensor) -> int:
    try:
        return _ARISTOS_DTYPE[t.dtype]
    except KeyError:
        raise TypeError(f"unsupported tensor dtype {t.dtype}") from None


def nccl_unique_id() -> bytes:
    buf = C.create_string_buffer(128)
    _lib.check(_lib.load().aristos_nccl_unique_id(buf))
    return buf.raw


def fill_normal(t: torch.Tensor, mean: float, std: float, seed: int, stream_id: int) -> torch.Tensor:
    _lib.check(_lib.load().aristos_fill_normal(_ptr(t), t.numel(), mean, std, seed, stream_id, _dt(t), _stream_ptr()))
    return t


def zipf_prior(num_experts: int, s: float) -> torch.Tensor:
    """The per-expert gate prior of `gate_bias_zipf_s` (-s ln(e + 1), fp32, host) as the layer builds it itself."""
    b = (C.c_float * num_experts)()
    _lib.check(_lib.load().aristos_zipf_bias_host(b, num_experts, float(s)))
    return torch.tensor(list(b), dtype=torch.float32)


def interleaved_expert_prior(prior: torch.Tensor, world: int) -> torch.Tensor:
    """Round-robin expert placement for a per-expert gate prior given in the experts' own order (entry e = expert e).

    A rank owns a contiguous block of E / world expert slots (rank r: slots [r E/world, (r + 1) E/world)). Holding
    expert e in slot (e % world) * (E / world) + e // world gives consecutive experts to different ranks, so the hot
    experts of a skewed prior do not all land on rank 0. Returns the prior indexed by slot - the gate_bias argument
    of the forward; the gate and expert weights of slot p are then those of expert (p % (E/world)) * world +
    p // (E/world). With world = 1 the prior is returned unchanged."""
    E = prior.numel()
    if world <= 1:
        return prior.clone()
    if E % world != 0:
        raise ValueError("the number of experts must be a multiple of the number of ranks")
    El = E // world
    slots = torch.arange(E)
    expert_of_slot = (slots % El) * world + slots // El
    return prior[expert_of_slot].clone()


def synthetic_tensors(cfg: AristosConfig, rank: int = 0, world: int = 1):
    """Seeded synthetic inputs of one rank, generated on the device: x ~ N(0,1) (a different stream per rank),
    gate weights and this rank's expert weights ~ N(0, 0.02). Expert e draws from its own Philox streams, so the
    shards of every world size are slices of the same global weights. Returns (x, w_gate, w1, w3, w2, scales);
    for torch_dtype 4 the expert weights are e4m3 codes (uint8) and scales holds their 128x128-block scales
    [s1 | s3 | s2], otherwise scales is None."""
    fp8 = cfg.torch_dtype == _lib.DTYPE_FP8_E4M3
    dt = _TORCH_DTYPE[cfg.torch_dtype]
    S, H, I, E = cfg.S, cfg.hidden_size, cfg.intermediate_size, cfg.num_experts
    El = E // world
    swiglu = cfg.hidden_act == _lib.ACT_SWIGLU
    new = lambda *shape: torch.empty(shape, dtype=dt, device="cuda")
    x = fill_normal(new(S, H), 0.0, 1.0, cfg.seed, 0 if rank == 0 else 0x1000 + rank)
    wg = fill_normal(new(E, H), 0.0, 0.02, cfg.seed, 1)

    def expert_tensor(rows, cols, which):
        if not fp8:
            w = new(El, rows, cols)
            for el in range(El):
                fill_normal(w[el], 0.0, 0.02, cfg.seed, 16 * (rank * El + el + 1) + which)
            return w, None
        q = torch.empty((El, rows, cols), dtype=torch.uint8, device="cuda")
        sc = torch.empty((El, (rows + 127) // 128, cols // 128), dtype=torch.float32, device="cuda")
        tmp = new(rows, cols)
        for el in range(El):          # one expert at a time: the bf16 originals never exist all at once
            fill_normal(tmp, 0.0, 0.02, cfg.seed, 16 * (rank * El + el + 1) + which)
            qe, se = quantize_fp8(tmp, 128)
            q[el].copy_(qe)
            sc[el].copy_(se)
        return q, sc

    w1, s1 = expert_tensor(I, H, 2)
    w3, s3 = expert_tensor(I, H, 3) if swiglu else (None, None)
    w2, s2 = expert_tensor(H, I, 4)
    scales = torch.cat([t.reshape(-1) for t in (s1, s3, s2) if t is not None]).contiguous() if fp8 else None
    return x, wg, w1, w3, w2, scales


# ---- stage entry points ---------------------------------------------------------------------------------------------
def gate_topk(x, w_gate, k: int, gate_fn: int = 0, renorm: int = 0, gate_bias=None, want_logits: bool = False):
    S, H = x.shape
    E = w_gate.shape[0]
    idx = torch.empty((S, k), dtype=torch.int32, device=x.device)
    w = torch.empty((S, k), dtype=torch.float32, device=x.device)
    logits = torch.empty((S, E), dtype=torch.float32, device=x.device) if want_logits else None
    _lib.check(_lib.load().aristos_gate_topk(_ptr(x), _ptr(w_gate), _ptr(gate_bias), S, H, E, k, gate_fn, renorm,
                                             _dt(x), _ptr(idx), _ptr(w), _ptr(logits), _stream_ptr()))
    return (idx, w, logits) if want_logits else (idx, w)


def gate_topk_screened(x, w_gate, k: int, gate_fn: int = 0, renorm: int = 0, gate_bias=None):
    """aristos_gate_topk_screened: tensor-core screen + exact evaluation of the experts that can still reach the
    top k (the layer's gate for 16-bit inputs and 32 <= E <= 256). Returns (topk_idx, topk_w, status word)."""
    S, H = x.shape
    E = w_gate.shape[0]
    lib = _lib.load()
    idx = torch.empty((S, k), dtype=torch.int32, device=x.device)
    w = torch.empty((S, k), dtype=torch.float32, device=x.device)
    nbytes = lib.aristos_gate_scratch_bytes(S, E)
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=x.device)
    status = torch.zeros(1, dtype=torch.int32, device=x.device)
    _lib.check(lib.aristos_gate_topk_screened(_ptr(x), _ptr(w_gate), _ptr(gate_bias), S, H, E, k, gate_fn, renorm,
                                              _dt(x), _ptr(idx), _ptr(w), _ptr(scratch), nbytes, _ptr(status),
                                              _stream_ptr()))
    return idx, w, status


def dispatch(topk_idx, E: int, cap: int):
    S, k = topk_idx.shape
    dev = topk_idx.device
    lib = _lib.load()
    nbytes = lib.aristos_dispatch_scratch_bytes(S, k, E)
    scratch = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=dev)
    count = torch.empty(E, dtype=torch.int32, device=dev)
    slot_of = torch.empty((S, k), dtype=torch.int32, device=dev)
    tos = torch.empty(E * cap, dtype=torch.int32, device=dev)
    _lib.check(lib.aristos_dispatch(_ptr(topk_idx), S, k, E, cap, _ptr(count), _ptr(slot_of), _ptr(tos),
                                    _ptr(scratch), nbytes, _stream_ptr()))
    return count, slot_of, tos


def dispatch_static(topk_idx, E: int, cap: int):
    """aristos_dispatch_static: the dispatch for callers that cannot allocate device memory (the library's built-in
    64 KiB scratch; S*k <= 131072, E <= 256). The outputs are still the caller's (here: torch) buffers."""
    S, k = topk_idx.shape
    dev = topk_idx.device
    count = torch.empty(E, dtype=torch.int32, device=dev)
    slot_of = torch.empty((S, k), dtype=torch.int32, device=dev)
    tos = torch.empty(E * cap, dtype=torch.int32, device=dev)
    _lib.check(_lib.load().aristos_dispatch_static(_ptr(topk_idx), S, k, E, cap, _ptr(count), _ptr(slot_of),
                                                   _ptr(tos), _stream_ptr()))
    return count, slot_of, tos


def permute(x, slot_of, nslots: int, zero: bool = False):
    S, H = x.shape
    k = slot_of.shape[1]
    xg = (torch.zeros if zero else torch.empty)((nslots, H), dtype=x.dtype, device=x.device)
    _lib.check(_lib.load().aristos_permute(_ptr(x), _ptr(slot_of), S, k, H, _dt(x), _ptr(xg), _stream_ptr()))
    return xg


def expert_ffn(xg, count, w1, w3, w2, hidden_act: int, *, experts: Optional[int] = None, row_begin: int = 0,
               row_end: Optional[int] = None, sm_limit: int = 0, dev_status=None, y=None, h=None, b1=None, b3=None,
               b2=None, dtype: Optional[int] = None):
    """xg (groups, rows, H); w1/w3 (experts, I, H); w2 (experts, H, I); optional biases b1/b3 (experts, I),
    b2 (experts, H) -> y (groups, rows, H)."""
    groups, rows, H = xg.shape
    I = w1.shape[1]
    experts = w1.shape[0] if experts is None else experts
    row_end = rows if row_end is None else row_end
    if h is None:
        h = torch.empty((groups, rows, I), dtype=xg.dtype, device=xg.device)
    if y is None:
        y = torch.zeros((groups, rows, H), dtype=xg.dtype, device=xg.device)
    _lib.check(_lib.load().aristos_expert_ffn_bias(_ptr(xg), _ptr(count), groups, rows, experts, _ptr(w1), _ptr(w3),
                                                   _ptr(w2), _ptr(b1), _ptr(b3), _ptr(b2), _ptr(h), _ptr(y), H, I,
                                                   hidden_act, _dt(xg) if dtype is None else dtype, row_begin, row_end,
                                                   sm_limit,
                                                   _ptr(dev_status), _stream_ptr()))
    return y


def quantize_fp8(src: torch.Tensor, block_rows: int):
    """e4m3 codes (uint8, same shape) and fp32 scales of a bf16 / fp32 tensor (..., rows, cols): block_rows 1 = per
    row and 128 columns (activations), 128 = per 128 x 128 block of every (rows, cols) matrix (weights)."""
    rows, cols = src.shape[-2], src.shape[-1]
    mats = src.numel() // (rows * cols)
    q = torch.empty(src.shape, dtype=torch.uint8, device=src.device)
    if block_rows == 1:
        scales = torch.empty((*src.shape[:-1], cols // 128), dtype=torch.float32, device=src.device)
    else:
        scales = torch.empty((*src.shape[:-2], (rows + 127) // 128, cols // 128), dtype=torch.float32,
                             device=src.device)
    _lib.check(_lib.load().aristos_quantize_fp8(_ptr(src), mats, rows, cols, block_rows, _dt(src), _ptr(q),
                                                _ptr(scales), _stream_ptr()))
    return q, scales


def expert_ffn_fp8(xq, sx, count, w1q, s1, w3q, s3, w2q, s2, hidden_act: int, dev_status=None):
    """FP8 expert FFN: xq (groups, rows, H) uint8 + sx (groups, rows, H/128); weights uint8 + block scales ->
    y (groups, rows, H) bf16."""
    groups, rows, H = xq.shape
    I = w1q.shape[1]
    dev = xq.device
    h = torch.empty((groups, rows, I), dtype=torch.bfloat16, device=dev)
    hq = torch.empty((groups, rows, I), dtype=torch.uint8, device=dev)
    sh = torch.empty((groups, rows, I // 128), dtype=torch.float32, device=dev)
    y = torch.zeros((groups, rows, H), dtype=torch.bfloat16, device=dev)
    _lib.check(_lib.load().aristos_expert_ffn_fp8(_ptr(xq), _ptr(sx), _ptr(count), groups, rows, w1q.shape[0],
                                                  _ptr(w1q), _ptr(s1), _ptr(w3q), _ptr(s3), _ptr(w2q), _ptr(s2),
                                                  _ptr(h), _ptr(hq), _ptr(sh), _ptr(y), H, I, hidden_act, 0, rows, 0,
                                                  _ptr(dev_status), _stream_ptr()))
    return y


# ---- microscaled 4-bit operands -------------------------------------------------------------------------------------
# The current stream of a device as an address, without a Stream object around it (1 us of a small call).
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


class _Device:
    """Makes the device that all the given tensors (None: not given) are on the current one for a call of the library, and
    gives the call its current stream. Only another device than the current one costs a switch."""
    __slots__ = ("index", "previous", "stream")

    def __init__(self, *tensors):
        index = None
        for t in tensors:
            if t is None:
                continue
            at = t.get_device()                  # -1: not on a GPU
            if index is None:
                index = at
            if at != index or at < 0:
                raise ValueError("tensors must all be on one CUDA device, got "
                                 f"{sorted({str(t.device) for t in tensors if t is not None})}")
        self.index = index

    def __enter__(self):
        self.previous = torch.cuda.current_device()
        if self.previous != self.index:
            torch.cuda.set_device(self.index)
        self.stream = _raw_stream(self.index)
        return self

    def __exit__(self, *_):
        if self.previous != self.index:
            torch.cuda.set_device(self.previous)


def _addr(t: Optional[torch.Tensor]):
    """The address that the C ABI takes for a tensor (ctypes makes a pointer of it)."""
    if t is None:
        return None
    if not t.is_contiguous():
        raise ValueError("tensors passed to the C ABI must be contiguous")
    return t.data_ptr()


def _fp4_scale_shape(lead, rows: int, cols: int):
    return (*lead, (rows + 127) // 128, (cols + 127) // 128, 32, 4, 4)


def _expect(name: str, t: torch.Tensor, shape, dtype: torch.dtype) -> None:
    if t.dtype != dtype or t.shape != shape:
        raise ValueError(f"{name} must be {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def quantize_fp4(src: torch.Tensor):
    """MXFP4 codes and scales of a (..., rows, cols) tensor in f32, bf16 or f16, cols a multiple of 64: codes uint8
    (..., rows, cols / 2), two e2m1 elements to a byte, the even column in the low half; scales uint8
    (..., ceil(rows / 128), ceil(cols / 128), 32, 4, 4): the byte 2^(s - 127) of row r and columns 32 b .. 32 b + 31 is
    [..., r / 128, b / 4, r % 32, r / 32 % 4, b % 4]. See aristos_quantize_fp4."""
    rows, cols = src.shape[-2], src.shape[-1]
    lead = src.shape[:-2]
    with _Device(src) as on:
        q = src.new_empty((*lead, rows, cols // 2), dtype=torch.uint8)
        scales = src.new_empty(_fp4_scale_shape(lead, rows, cols), dtype=torch.uint8)
        _lib.check(_lib.load().aristos_quantize_fp4(_addr(src), lead.numel(), rows, cols, _dt(src), _addr(q), _addr(scales),
                                                    on.stream))
    return q, scales


def dequantize_fp4(q: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values that MXFP4 codes and scales (as quantize_fp4 gives them) stand for, in f32, bf16 or f16."""
    rows, cols = q.shape[-2], 2 * q.shape[-1]
    lead = q.shape[:-2]
    _expect("q", q, q.shape, torch.uint8)
    _expect("scales", scales, _fp4_scale_shape(lead, rows, cols), torch.uint8)
    with _Device(q, scales) as on:
        out = q.new_empty((*lead, rows, cols), dtype=dtype)
        _lib.check(_lib.load().aristos_dequantize_fp4(_addr(q), _addr(scales), lead.numel(), rows, cols, _dt(out),
                                                      _addr(out), on.stream))
    return out


def _expect_status(t: Optional[torch.Tensor]) -> None:
    if t is not None and (t.dtype != torch.int32 or t.numel() < 1):
        raise ValueError(f"dev_status must hold an int32, got {t.dtype} {tuple(t.shape)}")


def _fp4_output(y, shape, dtype, device):
    if y is None:
        return torch.zeros(shape, dtype=dtype or torch.bfloat16, device=device)
    _expect("y", y, shape, dtype or y.dtype)
    return y


def expert_product_fp4(aq, sa, count, bq, sb, y=None, dtype: Optional[torch.dtype] = None, dev_status=None):
    """y[g, r] = A[g, r] . B[g % experts]^T for r < count[g], both operands in MXFP4: aq (groups, rows, K / 2) with sa,
    bq (experts, N, K / 2) with sb, count (groups) int32 -> y (groups, rows, N) in `dtype` (bf16 unless given; f32 and
    f16). Rows past count[g] keep what y holds (zeros in a y made here)."""
    groups, rows, half = aq.shape
    experts, N = bq.shape[:2]
    for name, t, shape in (("aq", aq, (groups, rows, half)), ("sa", sa, _fp4_scale_shape((groups,), rows, 2 * half)),
                           ("bq", bq, (experts, N, half)), ("sb", sb, _fp4_scale_shape((experts,), N, 2 * half))):
        _expect(name, t, shape, torch.uint8)
    _expect("count", count, (groups,), torch.int32)
    _expect_status(dev_status)
    with _Device(aq, sa, count, bq, sb, y, dev_status) as on:
        y = _fp4_output(y, (groups, rows, N), dtype, aq.device)
        _lib.check(_lib.load().aristos_expert_product_fp4(_addr(aq), _addr(sa), _addr(count), groups, rows, experts, _addr(bq),
                                                          _addr(sb), N, 2 * half, _dt(y), _addr(y), _addr(dev_status),
                                                          on.stream))
    return y


def expert_ffn_fp4(xq, sx, count, w1q, s1, w3q, s3, w2q, s2, hidden_act: int, y=None,
                   dtype: Optional[torch.dtype] = None, dev_status=None):
    """Expert FFN on MXFP4 operands: xq (groups, rows, H / 2) with sx; w1q / w3q (experts, I, H / 2) and w2q
    (experts, H, I / 2) with their scales (w3q, s3: SwiGLU only, else None) -> y (groups, rows, H) in `dtype` (bf16 unless
    given). The hidden activations are rounded to MXFP4 between the projections. Rows past count[g] keep what y holds."""
    groups, rows, half = xq.shape
    experts, I = w1q.shape[:2]
    H = 2 * half
    checks = [("xq", xq, (groups, rows, half)), ("sx", sx, _fp4_scale_shape((groups,), rows, H)),
              ("w1q", w1q, (experts, I, half)), ("s1", s1, _fp4_scale_shape((experts,), I, H)),
              ("w2q", w2q, (experts, H, I // 2)), ("s2", s2, _fp4_scale_shape((experts,), H, I))]
    if hidden_act == _lib.ACT_SWIGLU:
        if w3q is None or s3 is None:
            raise ValueError("SwiGLU needs w3q and s3")
        checks += [("w3q", w3q, (experts, I, half)), ("s3", s3, _fp4_scale_shape((experts,), I, H))]
    else:
        w3q = s3 = None
    for name, t, shape in checks:
        _expect(name, t, shape, torch.uint8)
    _expect("count", count, (groups,), torch.int32)
    _expect_status(dev_status)
    with _Device(xq, sx, count, w1q, s1, w3q, s3, w2q, s2, y, dev_status) as on:
        y = _fp4_output(y, (groups, rows, H), dtype, xq.device)
        hq = xq.new_empty((groups, rows, I // 2))
        sh = xq.new_empty(_fp4_scale_shape((groups,), rows, I))
        _lib.check(_lib.load().aristos_expert_ffn_fp4(_addr(xq), _addr(sx), _addr(count), groups, rows, experts, _addr(w1q),
                                                      _addr(s1), _addr(w3q), _addr(s3), _addr(w2q), _addr(s2), _addr(hq),
                                                      _addr(sh), _addr(y), H, I, hidden_act, _dt(y), _addr(dev_status),
                                                      on.stream))
    return y


# ---- the layer for a few tokens ---------------------------------------------------------------------------------------
@functools.lru_cache(maxsize=1024)
def _few_workspace_bytes(n: int, H: int, I: int, E: int, k: int) -> int:
    return _lib.load().aristos_moe_few_tokens_workspace_bytes(n, H, I, E, k)


def moe_few_tokens(x, w_gate, w1, w3, w2, k: int, hidden_act: int, *, gate_fn: int = 0, renorm: int = 0, gate_bias=None,
                   scales=None, b1=None, b3=None, b2=None, out=None, dev_status=None):
    """The whole layer for up to 64 tokens in two kernels: x (tokens, H) bf16 or f16; w_gate (E, H); w1 / w3 (E, I, H) and
    w2 (E, H, I) in x's dtype, or quantised (uint8) with scales = (s1, s3, s2): e4m3 codes as quantize_fp8(w, 128) gives
    them (bf16 tokens only) or MXFP4 codes (E, I, H / 2), (E, H, I / 2) as quantize_fp4 gives them. Optional biases
    b1 / b3 (E, I), b2 (E, H) in x's dtype, gate_bias (E) fp32. w3, s3 and b3 are SwiGLU's. Nothing is dropped.
    Returns (out (tokens, H), topk_idx (tokens, k) int32, topk_w (tokens, k) fp32). See aristos_moe_few_tokens."""
    n, H = x.shape
    E, I = w1.shape[:2]
    gated = hidden_act == _lib.ACT_SWIGLU
    if gated and w3 is None:
        raise ValueError("SwiGLU needs w3")
    w3, b3 = (w3, b3) if gated else (None, None)
    dt = _dt(x)
    _expect("w_gate", w_gate, (E, H), x.dtype)
    if w1.dtype == torch.uint8:
        if scales is None:
            raise ValueError("quantised weights need scales = (s1, s3, s2)")
        s1, s3, s2 = scales
        s3 = s3 if gated else None
        fp4 = w1.shape[2] * 2 == H
        wdt, per, code = (_lib.DTYPE_FP4_E2M1, 2, torch.uint8) if fp4 else (_lib.DTYPE_FP8_E4M3, 1, torch.uint8)
        shape = ((lambda r, c: _fp4_scale_shape((E,), r, c)) if fp4 else (lambda r, c: (E, (r + 127) // 128, c // 128)))
        for name, t, r, c in (("s1", s1, I, H), ("s3", s3, I, H), ("s2", s2, H, I)):
            if t is not None or name != "s3" or gated:
                if t is None:
                    raise ValueError(f"{name} is missing")
                _expect(name, t, shape(r, c), torch.uint8 if fp4 else torch.float32)
    else:
        s1 = s3 = s2 = None
        wdt, per, code = dt, 1, x.dtype
    _expect("w1", w1, (E, I, H // per), code)
    _expect("w2", w2, (E, H, I // per), code)
    if gated:
        _expect("w3", w3, (E, I, H // per), code)
    for name, t, shape, d in (("gate_bias", gate_bias, (E,), torch.float32), ("b1", b1, (E, I), x.dtype),
                              ("b3", b3, (E, I), x.dtype), ("b2", b2, (E, H), x.dtype), ("out", out, (n, H), x.dtype)):
        if t is not None:
            _expect(name, t, shape, d)
    _expect_status(dev_status)
    lib = _lib.load()
    with _Device(x, w_gate, w1, w3, w2, s1, s3, s2, gate_bias, b1, b3, b2, out, dev_status) as on:
        if out is None:
            out = torch.empty_like(x)
        idx = x.new_empty((n, k), dtype=torch.int32)
        w = x.new_empty((n, k), dtype=torch.float32)
        nbytes = _few_workspace_bytes(n, H, I, E, k)
        ws = x.new_empty(max(nbytes, 16), dtype=torch.uint8)
        _lib.check(lib.aristos_moe_few_tokens(_addr(x), _addr(w_gate), _addr(gate_bias), _addr(w1), _addr(w3), _addr(w2),
                                              _addr(s1), _addr(s3), _addr(s2), _addr(b1), _addr(b3), _addr(b2), n, H, I, E, k,
                                              gate_fn, renorm, hidden_act, dt, wdt, _addr(out), _addr(idx), _addr(w),
                                              _addr(ws), nbytes, _addr(dev_status), on.stream))
    return out, idx, w


def combine(y, slot_of, topk_w):
    S, k = slot_of.shape
    H = y.shape[-1]
    out = torch.empty((S, H), dtype=y.dtype, device=y.device)
    _lib.check(_lib.load().aristos_combine(_ptr(y), _ptr(slot_of), _ptr(topk_w), S, k, H, _dt(y), _ptr(out),
                                           _stream_ptr()))
    return out


def ffn_set_tile_mode(mode: int) -> None:
    """aristos_ffn_set_tile_mode: 0 automatic, 1 single-CTA tiles, 2 CTA pairs + single-CTA tail, 3 CTA pairs padded,
    -1 re-read ARISTOS_FFN_TILES."""
    _lib.check(_lib.load().aristos_ffn_set_tile_mode(int(mode)))


# ---- layer ----------------------------------------------------------------------------------------------------------
class MoELayer:
    """One MoE layer on the current CUDA device (aristos_moe_create ... aristos_moe_destroy)."""

    def __init__(self, cfg: AristosConfig, rank: int = 0, world: int = 1, nccl_uid: Optional[bytes] = None):
        if not torch.cuda.is_available():
            raise RuntimeError("cuplayground_b200 needs a CUDA device (sm_100a); there is no CPU fallback")
        self.cfg = cfg
        self.rank, self.world = rank, world
        self._lib = _lib.load()
        self._h = C.c_void_p()
        self.device = torch.cuda.current_device()
        s = cfg.to_struct()
        uid = C.create_string_buffer(nccl_uid, 128) if nccl_uid is not None else None
        _lib.check(self._lib.aristos_moe_create(C.byref(s), rank, world, uid, C.byref(self._h)))
        self.S, self.H, self.I = cfg.S, cfg.hidden_size, cfg.intermediate_size
        self.E, self.k, self.cap = cfg.num_experts, cfg.expert_top_k, cfg.capacity
        self.E_local = self.E // world
        self.dtype = _TORCH_DTYPE[cfg.torch_dtype]
        self._ws = self._decode_ws = None

    @property
    def workspace_bytes(self) -> int:
        return int(self._lib.aristos_moe_workspace_bytes(self._h))

    def use_torch_workspace(self) -> None:
        """Allocate the workspace (and decode's own, when it first decodes) from torch's caching allocator instead of cudaMalloc
        inside the library."""
        self._ws = torch.empty(self.workspace_bytes + 1024, dtype=torch.uint8, device="cuda")
        base = (self._ws.data_ptr() + 1023) // 1024 * 1024
        _lib.check(self._lib.aristos_moe_set_workspace(self._h, C.c_void_p(base), self.workspace_bytes))

    def set_bias(self, b1=None, b3=None, b2=None) -> None:
        """Expert biases (E_local, I) / (E_local, I) / (E_local, H) for every later forward; kept alive here."""
        self._bias = (b1, b3, b2)
        _lib.check(self._lib.aristos_moe_set_bias(self._h, _ptr(b1), _ptr(b3), _ptr(b2)))

    def forward(self, x, w_gate, w1, w3, w2, gate_bias=None, out=None, stream=None, scales=None):
        """scales: fp8 only - the weights' block scales [s1 | s3 | s2] as one contiguous fp32 tensor."""
        if out is None:
            out = torch.empty_like(x)
        _lib.check(self._lib.aristos_moe_forward(self._h, _ptr(x), _ptr(w_gate), _ptr(gate_bias), _ptr(w1), _ptr(w3),
                                                 _ptr(w2), _ptr(scales), _ptr(out), _stream_ptr(stream)))
        return out

    def forward_host(self, x_host, w_gate, w1, w3, w2, out_host, gate_bias=None, stream=None, scales=None):
        """x_host / out_host: CPU tensors (pinned for full speed); weights stay on the device. Synchronous."""
        if x_host.is_cuda or out_host.is_cuda:
            raise ValueError("forward_host takes host tensors")
        _lib.check(self._lib.aristos_moe_forward_host(self._h, _ptr(x_host), _ptr(w_gate), _ptr(gate_bias), _ptr(w1),
                                                      _ptr(w3), _ptr(w2), _ptr(scales), _ptr(out_host),
                                                      _stream_ptr(stream)))
        return out_host

    def submit_host(self, x_host, w_gate, w1, w3, w2, out_host, gate_bias=None, stream=None, scales=None):
        """Asynchronous forward_host: returns once the copies and kernels are enqueued (four calls may be in flight);
        the host tensors must stay alive and untouched until wait_host()."""
        if x_host.is_cuda or out_host.is_cuda:
            raise ValueError("submit_host takes host tensors")
        _lib.check(self._lib.aristos_moe_submit_host(self._h, _ptr(x_host), _ptr(w_gate), _ptr(gate_bias), _ptr(w1),
                                                     _ptr(w3), _ptr(w2), _ptr(scales), _ptr(out_host),
                                                     _stream_ptr(stream)))

    def wait_host(self) -> None:
        _lib.check(self._lib.aristos_moe_wait_host(self._h))

    def decode(self, x, w_gate, w1, w3, w2, gate_bias=None, out=None, stream=None, scales=None):
        """The forward for up to 64 tokens, x (tokens, H): two kernels, nothing dropped, activations not quantised. w_gate
        (E, H); w1 / w3 (E, I, H) and w2 (E, H, I) in the layer's dtype (fp8: e4m3 codes, scales as for forward); all on the
        layer's device. Returns (out, topk_idx (tokens, k), topk_w (tokens, k)). See aristos_moe_decode."""
        if x.dim() != 2 or x.shape[1] != self.H or x.dtype != self.dtype:
            raise ValueError(f"x must be {self.dtype} (tokens, {self.H}), got {x.dtype} {tuple(x.shape)}")
        n, E, H, I = x.shape[0], self.E_local, self.H, self.I
        gated = self.cfg.hidden_act == _lib.ACT_SWIGLU
        fp8 = self.cfg.torch_dtype == _lib.DTYPE_FP8_E4M3
        w3, scales = w3 if gated else None, scales if fp8 else None
        if w_gate is not None:
            _expect("w_gate", w_gate, (self.E, H), self.dtype)
        for name, t, shape in (("w1", w1, (E, I, H)), ("w3", w3, (E, I, H)), ("w2", w2, (E, H, I))):
            if t is not None:
                code = torch.float8_e4m3fn if fp8 and t.dtype == torch.float8_e4m3fn else torch.uint8 if fp8 else self.dtype
                _expect(name, t, shape, code)
        if gate_bias is not None:
            _expect("gate_bias", gate_bias, (self.E,), torch.float32)
        if scales is not None:
            blocks = E * (I // 128) * (H // 128) * (3 if gated else 2)
            if scales.dtype != torch.float32 or scales.numel() != blocks:
                raise ValueError(f"scales must be {blocks} torch.float32, got {scales.numel()} {scales.dtype}")
        if out is not None:
            _expect("out", out, (n, H), self.dtype)
        bias = getattr(self, "_bias", (None, None, None))
        for name, t, cols in zip(("b1", "b3", "b2"), bias, (I, I, H)):
            if t is not None and (t.dtype != self.dtype or t.numel() != E * cols):
                raise ValueError(f"{name} must be {E * cols} {self.dtype}, got {t.numel()} {t.dtype}")
        with _Device(x, w_gate, w1, w3, w2, gate_bias, scales, out, *bias) as on:
            if on.index != self.device or (stream is not None and stream.device.index != self.device):
                raise ValueError(f"the layer, its tensors and the stream must be on one device, the layer is on cuda:{self.device}")
            with torch.cuda.stream(stream):              # workspace and outputs belong to the stream that writes them
                if self._ws is not None and self._decode_ws is None:
                    nbytes = int(self._lib.aristos_moe_decode_workspace_bytes(self._h))
                    if nbytes:                           # 0: the library refuses
                        ws = torch.empty(nbytes, dtype=torch.uint8, device=x.device)
                        _lib.check(self._lib.aristos_moe_set_decode_workspace(self._h, _addr(ws), nbytes))
                        self._decode_ws = ws
                out = torch.empty_like(x) if out is None else out
                idx = x.new_empty((n, self.k), dtype=torch.int32)
                w = x.new_empty((n, self.k), dtype=torch.float32)
            _lib.check(self._lib.aristos_moe_decode(self._h, _addr(x), n, _addr(w_gate), _addr(gate_bias), _addr(w1), _addr(w3),
                                                    _addr(w2), _addr(scales), _addr(out), _addr(idx), _addr(w),
                                                    on.stream if stream is None else stream.cuda_stream))
        return out, idx, w

    def routing(self) -> dict:
        """Host copies (CPU torch tensors) of the routing tensors of the last forward."""
        S, k, E, cap = self.S, self.k, self.E, self.cap
        idx = torch.empty((S, k), dtype=torch.int32)
        w = torch.empty((S, k), dtype=torch.float32)
        count = torch.empty(E, dtype=torch.int32)
        slot_of = torch.empty((S, k), dtype=torch.int32)
        tos = torch.empty(E * cap, dtype=torch.int32)
        _lib.check(self._lib.aristos_moe_routing_to_host(self._h, _ptr(idx), _ptr(w), _ptr(count), _ptr(slot_of),
                                                         _ptr(tos)))
        return dict(topk_idx=idx, topk_w=w, count=count, slot_of=slot_of, token_of_slot=tos, capacity=cap)

    def set_profiling(self, enable: bool) -> None:
        _lib.check(self._lib.aristos_moe_set_profiling(self._h, int(enable)))

    def stage_ms(self) -> dict:
        """Milliseconds of the stages of the last forward (profiling must be on)."""
        ms = (C.c_float * 5)()
        _lib.check(self._lib.aristos_moe_stage_ms(self._h, ms))
        return dict(gate=ms[0], dispatch=ms[1], ffn=ms[2], combine=ms[3], total=ms[4])

    def exchange_ms(self) -> float:
        """Milliseconds of the outgoing exchange (counts + gather into the peers + flags) of the last forwards."""
        ms = C.c_float(0.0)
        _lib.check(self._lib.aristos_moe_exchange_ms(self._h, C.byref(ms)))
        return float(ms.value)

    def exchange_profile(self) -> dict:
        """The expert-FFN stage of an expert-parallel layer split at its cross-rank waits (milliseconds)."""
        ms = (C.c_float * 4)()
        _lib.check(self._lib.aristos_moe_exchange_profile(self._h, ms))
        return dict(rows_sent=ms[0], counts_arrived=ms[1], gemms=ms[2], returns_arrived=ms[3])

    def status(self) -> None:
        _lib.check(self._lib.aristos_moe_status(self._h))

    def training_state(self) -> dict:
        """is_training = 1: what the last forward saved for a backward pass - host copies of the routing and the
        load-balance statistics (frac, prob per expert; aux loss; dropped share)."""
        ts = _lib.AristosTrainingStateStruct()
        _lib.check(self._lib.aristos_moe_training_state(self._h, C.byref(ts)))
        S, k, E = ts.tokens, ts.top_k, ts.num_experts
        idx = torch.empty((S, k), dtype=torch.int32)
        w = torch.empty((S, k), dtype=torch.float32)
        slot = torch.empty((S, k), dtype=torch.int32)
        lb = torch.empty(2 * E + 2, dtype=torch.float32)
        _lib.check(self._lib.aristos_moe_training_state_to_host(self._h, _ptr(idx), _ptr(w), _ptr(slot), _ptr(lb)))
        return dict(topk_idx=idx, topk_w=w, slot_of=slot, frac=lb[:E], prob=lb[E:2 * E], aux=float(lb[2 * E]),
                    dropped=float(lb[2 * E + 1]),
                    device_ptrs=(ts.topk_idx, ts.topk_w, ts.slot_of, ts.load_balance))

    def set_training_buffer(self, buf: Optional[torch.Tensor]) -> None:
        """Point the next forwards' saved training state at a caller-owned device buffer (uint8, at least
        training_bytes, 256-byte aligned); None returns to the layer's own buffer."""
        self._train_buf = buf
        if buf is None:
            _lib.check(self._lib.aristos_moe_set_training_buffer(self._h, None, 0))
        else:
            _lib.check(self._lib.aristos_moe_set_training_buffer(self._h, C.c_void_p(buf.data_ptr()), buf.numel()))

    @property
    def training_bytes(self) -> int:
        return int(self._lib.aristos_moe_training_bytes(self._h))

    def set_timeout_ms(self, timeout_ms: int) -> None:
        """Wall-clock limit of the waits for an expert-parallel forward (status, wait_host, routing, close)."""
        _lib.check(self._lib.aristos_moe_set_timeout_ms(self._h, int(timeout_ms)))

    @property
    def ep_transport(self) -> str:
        return self._lib.aristos_moe_ep_transport(self._h).decode()

    @property
    def launch_count(self) -> int:
        return int(self._lib.aristos_moe_launch_count(self._h))

    def close(self) -> None:
        if self._h:
            self._lib.aristos_moe_destroy(self._h)
            self._h = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:
            pass

"""Torch-facing binding of the state-space operators (include/gdn_ssm.h): the short causal
convolution, the selective scan and the gated group norm of hybrid layers, for prompts (batched
or packed) and for single tokens. No counterparts in the reference; same conventions as the gated
delta rule's entries (``binding.py``): ValueError for bad arguments, GdnError for a launch that
failed, torch's current CUDA stream of the inputs' device, outputs allocated with torch, no autograd.

Inputs may be slices of a wider projection (a row stride above the row's width); other layouts
are copied to contiguous memory first.
"""
from __future__ import annotations

import torch

from ._lib import load_library
from .binding import _check, _workspace, _ws_cache

__all__ = ["causal_conv_prefill", "causal_conv_prefill_varlen", "causal_conv_decode", "selective_scan_prefill",
           "selective_scan_prefill_varlen", "selective_scan_decode", "gated_group_rmsnorm"]

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_MAX_GRID = 65535  # sequences and heads of a scan are grid dimensions
_MAX_INT = (1 << 31) - 1  # sizes cross the C ABI as int, and ctypes keeps the low bits of larger ones
_MAX_ROWS = _MAX_INT - 128  # token rows of a scan over prompts (32-bit tile coordinates, whole tiles)
# the current stream's handle without a Stream object: a single-token call is bound by its host time
_raw_stream = torch._C._cuda_getCurrentRawStream


def _on(dev, fn, *args):
    """fn(*args) with device index ``dev`` current."""
    if dev == torch.cuda.current_device():
        return fn(*args)
    with torch.cuda.device(dev):
        return fn(*args)


def _call(dev, what, fn, *args):
    """fn(*args, stream) on torch's current stream of device index ``dev``."""
    code = _on(dev, fn, *args, _raw_stream(dev))
    if code:
        _check(code, what)


def _p(t):
    return None if t is None else t.data_ptr()


def _out(x):
    """A contiguous tensor of x's shape, type and device."""
    return torch.empty_like(x) if x.is_contiguous() else x.new_empty(x.shape)


def _on_one_device(first, *others):
    """The index of the CUDA device that holds every tensor."""
    dev = first.get_device()
    for t in others:
        if t.get_device() != dev:
            if dev >= 0 and t.get_device() >= 0:
                raise ValueError("all tensors must be on the same CUDA device")
            dev = -1
    if dev < 0:
        raise ValueError("all inputs must be CUDA tensors")
    return dev


def _status(dev):
    """Address of the status word of the device's first cached workspace (one of those that ``read_status`` reads)."""
    made = _ws_cache.get(dev)
    return (made[0] if made else _workspace(torch.device("cuda", dev), 256)).data_ptr()


def _rows(t, lead, align=1):
    """(t, row stride in elements): t with its ``lead`` leading dims as evenly spaced rows and its
    other dims contiguous inside a row, t itself where that holds and pointer and stride are
    multiples of ``align`` elements, else a contiguous copy."""
    shape = t.shape
    width = 1
    for n in shape[lead:]:
        width *= n
    if not t.is_contiguous():
        strides = t.stride()
        inner = 1
        for d in range(len(shape) - 1, lead - 1, -1):
            if shape[d] != 1 and strides[d] != inner:
                return _packed_rows(t, width, align)
            inner *= shape[d]
        stride, rows = None, 1
        for d in range(lead - 1, -1, -1):
            if shape[d] == 1:
                continue
            if stride is None:
                stride = strides[d]
            elif strides[d] != stride * rows:
                return _packed_rows(t, width, align)
            rows *= shape[d]
        if stride is None:  # one row
            stride = width
        if stride < width:
            return _packed_rows(t, width, align)
    else:
        stride = width
    if align > 1 and (stride % align or t.data_ptr() % (align * t.element_size())):
        return _packed_rows(t, width, align)
    return t, stride


def _wide_rows(t, lead, width, align=1):
    """``_rows`` of a t whose rows are known to be ``width`` wide: a contiguous one takes no walk over its dims."""
    if t.is_contiguous() and (align == 1 or (width % align == 0 and t.data_ptr() % (align * t.element_size()) == 0)):
        return t, width
    return _rows(t, lead, align)


def _packed_rows(t, width, align):
    t = t.contiguous()
    if t.data_ptr() % (align * t.element_size()):
        t = t.clone()
    return t, width


def _vector(t, n, dtype, name, dev):
    if t is None:
        return None
    if t.dtype != dtype or t.dim() != 1 or t.shape[0] != n:
        raise ValueError(f"{name} must be {dtype} of shape [{n}]")
    if t.get_device() != dev:
        raise ValueError("all tensors must be on the same CUDA device")
    return t if t.is_contiguous() else t.contiguous()


def _initial(s0, shape, dtype, dev):
    """The initial state as a contiguous, 16-byte aligned tensor of ``dtype`` (or None)."""
    if s0 is None:
        return None
    if tuple(s0.shape) != shape:
        raise ValueError(f"initial state must have shape {shape}, got {tuple(s0.shape)}")
    if s0.dtype != dtype or s0.get_device() != dev:
        s0 = s0.to(device=torch.device("cuda", dev), dtype=dtype)
    s0 = s0.contiguous()
    return s0 if s0.data_ptr() % 16 == 0 else s0.clone()


def _offsets(cu_seqlens, dev):
    if cu_seqlens.dtype != torch.int32 or cu_seqlens.dim() != 1 or not cu_seqlens.is_cuda or cu_seqlens.numel() < 1:
        raise ValueError("cu_seqlens must be a 1-D int32 CUDA tensor of at least one element")
    if cu_seqlens.get_device() != dev:
        raise ValueError("all tensors must be on the same CUDA device")
    return cu_seqlens.contiguous()


# ---------------------------------------------------------------- causal convolution
def _check_conv(x, w, bias, packed=False):
    dev = _on_one_device(x, w)
    dtype = x.dtype
    if dtype not in _DTYPES or w.dtype != dtype:
        raise ValueError("x and w must share dtype fp16, bf16 or fp32")
    if x.dim() != 3 or w.dim() != 2:
        raise ValueError("bad shapes: x must be [B, T, C] and w [C, W]")
    B, _, C = x.shape
    rows, W = w.shape
    if rows != C:
        raise ValueError("bad shapes: x must be [B, T, C] and w [C, W]")
    if not 2 <= W <= 4:
        raise ValueError("only 2 to 4 taps are supported")
    if C < 1:
        raise ValueError("x needs at least one channel")
    if B > _MAX_INT or x.shape[1] > _MAX_INT or C > _MAX_INT:
        raise ValueError("sizes of x must be below 2^31")
    if packed and B != 1:
        raise ValueError("varlen inputs are packed: B must be 1")
    return dev, _vector(bias, C, dtype, "bias", dev)


def _conv_prefill(x, w, bias, s0, silu, cu):
    dev, bias = _check_conv(x, w, bias, cu is not None)
    B, T, C = x.shape
    W = w.shape[1]
    if cu is not None:
        cu = _offsets(cu, dev)
    n = B if cu is None else cu.numel() - 1
    s0 = _initial(s0, (n, W - 1, C), x.dtype, dev)
    x, stride = _wide_rows(x, 2, C)
    w = w.contiguous()
    y = _out(x)
    sf = x.new_empty((n, W - 1, C))
    _call(dev, "causal_conv_prefill", load_library().causal_conv_prefill, _p(x), stride, _p(w), _p(bias), _p(s0), _p(y),
          _p(sf), _p(cu), n, T, C, W, bool(silu), _DTYPES[x.dtype])
    return [y, sf]


def causal_conv_prefill(x, w, bias=None, s0=None, silu: bool = True):
    """Short causal depthwise convolution over prompts: [y [B,T,C], final state [B,W-1,C]].

    y[t, c] = act(bias[c] + sum_j w[c, j] x[t - W + 1 + j, c]), act = silu unless ``silu`` is false.
    x [B,T,C], w [C,W] with 2 to 4 taps, bias [C], all fp16, bf16 or fp32 (fp32 math). Inputs before
    the start are ``s0`` [B,W-1,C] (oldest first) or zeros; the final state is the last W-1 inputs.
    """
    return _conv_prefill(x, w, bias, s0, silu, None)


def causal_conv_prefill_varlen(x, w, cu_seqlens, bias=None, s0=None, silu: bool = True):
    """``causal_conv_prefill`` of packed sequences (B = 1): [y [1,T,C], final states [N,W-1,C]].

    Sequence i covers tokens [cu[i], cu[i+1]) of int32 ``cu_seqlens`` [N+1] (on the device) and starts
    from s0[i] or zeros. Tokens that no sequence covers are not computed: their rows of y hold no
    defined values.
    """
    return _conv_prefill(x, w, bias, s0, silu, cu_seqlens)


def causal_conv_decode(x, w, state, bias=None, silu: bool = True):
    """The convolution of the next token(s) x [B,T,C] (T usually 1): returns y [B,T,C]; ``state``
    [B,W-1,C] (a prefill's final state, x's dtype, contiguous) is updated in place."""
    dev, bias = _check_conv(x, w, bias)
    B, T, C = x.shape
    W = w.shape[1]
    if state.dtype != x.dtype or not state.is_contiguous() or state.shape != (B, W - 1, C):
        raise ValueError(f"state must be a contiguous tensor of x's dtype and shape {(B, W - 1, C)}")
    _on_one_device(x, state)
    x, stride = _wide_rows(x, 2, C)
    w = w.contiguous()
    y = _out(x)
    _call(dev, "causal_conv_decode", load_library().causal_conv_decode, _p(x), stride, _p(w), _p(bias), _p(state), _p(y),
          B, T, C, W, bool(silu), _DTYPES[x.dtype])
    return y


# ---------------------------------------------------------------- selective scan
def _check_scan(x, dt, A, B, C, D, dt_bias, packed=False):
    dev = _on_one_device(x, dt, A, B, C)
    if not (x.dtype == B.dtype == C.dtype == torch.bfloat16):
        raise ValueError("x/B/C must be bf16")
    if dt.dtype not in (torch.float32, torch.bfloat16):
        raise ValueError("dt must be fp32 or bf16")
    if x.dim() != 4 or B.dim() != 4 or C.dim() != 4 or dt.dim() != 3:
        raise ValueError("bad ranks: x must be 4-D [B,T,H,P], B/C 4-D [B,T,G,N], dt 3-D [B,T,H]")
    b, T, H, P = x.shape
    bshape = B.shape
    bb, bt, G, N = bshape
    if bb != b or bt != T or C.shape != bshape or dt.shape != (b, T, H):
        raise ValueError("shape mismatch between x/dt/B/C")
    if G < 1 or H < 1 or H % G != 0:
        raise ValueError("H must be a multiple of G")
    if not (8 <= P <= 128 and P % 8 == 0 and 8 <= N <= 128 and N % 8 == 0):
        raise ValueError("P and N must be multiples of 8 up to 128")
    if packed and b != 1:
        raise ValueError("varlen inputs are packed: B must be 1")
    if b > _MAX_GRID or H > _MAX_GRID:
        raise ValueError(f"at most {_MAX_GRID} sequences and heads are supported")
    if T > _MAX_INT:
        raise ValueError("sizes must be below 2^31")
    A = _vector(A, H, torch.float32, "A", dev)
    D = _vector(D, H, torch.float32, "D", dev)
    dt_bias = _vector(dt_bias, H, torch.float32, "dt_bias", dev)
    return dev, (b, T, H, P, G, N), A, D, dt_bias


def _scan_prefill(x, dt, A, B, C, D, dt_bias, s0, dt_softplus, cu):
    dev, (b, T, H, P, G, N), A, D, dt_bias = _check_scan(x, dt, A, B, C, D, dt_bias, cu is not None)
    if cu is not None:
        cu = _offsets(cu, dev)
    n = b if cu is None else cu.numel() - 1
    if b * T > _MAX_ROWS:
        raise ValueError(f"at most {_MAX_ROWS} token rows are supported")
    if n > _MAX_GRID:
        raise ValueError(f"at most {_MAX_GRID} sequences and heads are supported")
    s0 = _initial(s0, (n, H, P, N), torch.float32, dev)
    (x, xs), (dt, dts) = _wide_rows(x, 2, H * P, 8), _wide_rows(dt, 2, H)
    (B, bs), (C, cs) = _wide_rows(B, 2, G * N, 8), _wide_rows(C, 2, G * N, 8)
    y = _out(x)
    sf = A.new_empty((n, H, P, N))
    lib = load_library()
    nbytes = _on(dev, lib.selective_scan_scratch_size, n, T, cu is not None, H, P, G, N)  # (plans for the current device)
    scratch = A.new_empty(nbytes // 4) if nbytes else None
    _call(dev, "selective_scan_prefill", lib.selective_scan_prefill, _p(x), xs, _p(dt), dts, dt.dtype == torch.bfloat16,
          _p(A), _p(B), bs, _p(C), cs, _p(D), _p(dt_bias), bool(dt_softplus), _p(s0), _p(y), _p(sf), _p(cu), n, T, H, P,
          G, N, _status(dev), 256, _p(scratch), nbytes)
    return [y, sf]


def selective_scan_prefill(x, dt, A, B, C, D=None, dt_bias=None, s0=None, dt_softplus: bool = False):
    """Selective state space scan over prompts: [y (bf16 [B,T,H,P]), final state (fp32 [B,H,P,N])].

    Per head h of group g = h // (H // G), with d = dt + dt_bias (softplus'ed if ``dt_softplus``):
        S <- exp(d A) S + d x B^T;   y = S C + D x.
    x bf16 [B,T,H,P], dt fp32 or bf16 [B,T,H], B/C bf16 [B,T,G,N], A, D, dt_bias fp32 [H], initial
    state s0 fp32 [B,H,P,N] or zeros. P and N are multiples of 8 up to 128, B and H at most 65535, B T at
    most 2^31 - 129, and d A <= 0. A token with d = 0 (dt of minus infinity under the softplus) leaves the state as it is, so
    padding in front of or between tokens (of finite x and B) is possible. An x that is not finite
    makes its channel's outputs NaN from the start of its 128 tokens (of its sequence) on.

    Calls of 16 tokens and more run in chunks of 128 on the tensor cores: sums and the state are fp32, but two operands
    of y, the weights of a chunk's tokens and the state at its start, are rounded to bf16 (as y is); the state is not
    affected. Shorter calls are fp32 throughout.
    """
    return _scan_prefill(x, dt, A, B, C, D, dt_bias, s0, dt_softplus, None)


def selective_scan_prefill_varlen(x, dt, A, B, C, cu_seqlens, D=None, dt_bias=None, s0=None, dt_softplus: bool = False):
    """``selective_scan_prefill`` of packed sequences (B = 1): [y [1,T,H,P], final states [N,H,P,N]].

    ``cu_seqlens`` as in ``chunk_prefill_varlen``; sequence i starts from s0[i] or zeros. Tokens that
    no sequence covers are not computed: their rows of y hold no defined values. Every sequence takes at least the
    time of 128 tokens: the single tokens of many requests are faster through ``selective_scan_decode``.
    """
    return _scan_prefill(x, dt, A, B, C, D, dt_bias, s0, dt_softplus, cu_seqlens)


def selective_scan_decode(x, dt, A, B, C, state, D=None, dt_bias=None, dt_softplus: bool = False):
    """The scan of the next token(s) x [B,T,H,P] (T usually 1), shapes as in ``selective_scan_prefill``:
    returns y; the fp32 ``state`` [B,H,P,N] (e.g. a prefill's final state) is updated in place."""
    dev, (b, T, H, P, G, N), A, D, dt_bias = _check_scan(x, dt, A, B, C, D, dt_bias)
    if state.dtype != torch.float32 or not state.is_contiguous() or state.shape != (b, H, P, N):
        raise ValueError("state must be a contiguous fp32 [B, H, P, N] tensor")
    _on_one_device(x, state)
    if state.data_ptr() % 16:
        raise ValueError("state must be 16-byte aligned")
    (x, xs), (dt, dts) = _wide_rows(x, 2, H * P, 8), _wide_rows(dt, 2, H)
    (B, bs), (C, cs) = _wide_rows(B, 2, G * N, 8), _wide_rows(C, 2, G * N, 8)
    y = _out(x)
    _call(dev, "selective_scan_decode", load_library().selective_scan_decode, _p(x), xs, _p(dt), dts,
          dt.dtype == torch.bfloat16, _p(A), _p(B), bs, _p(C), cs, _p(D), _p(dt_bias), bool(dt_softplus), _p(state),
          _p(y), b, T, H, P, G, N)
    return y


# ---------------------------------------------------------------- gated group norm
def gated_group_rmsnorm(x, z, w, groups: int = 1, eps: float = 1e-6):
    """Gated RMSNorm over channel groups with the gate before the norm, over the last dim:
    u = x silu(z); y = w u rsqrt(mean_group(u^2) + eps). x, z [..., C], w [C], all fp16, bf16 or fp32;
    ``groups`` divides C. (``gated_rmsnorm`` has the gate behind the norm.)"""
    dev = _on_one_device(x, z, w)
    if x.dtype not in _DTYPES or z.dtype != x.dtype or w.dtype != x.dtype:
        raise ValueError("x, z, w must share dtype fp16, bf16 or fp32")
    if x.dim() < 1 or z.shape != x.shape or w.dim() != 1 or w.shape[0] != x.shape[-1]:
        raise ValueError("z must match x and w must be [C]")
    C = x.shape[-1]
    if groups < 1 or C < 1 or C % groups != 0:
        raise ValueError("groups must divide the last dim")
    if C > _MAX_INT:
        raise ValueError("the last dim must be below 2^31")
    y = _out(x)
    lead = x.dim() - 1
    (x, xs), (z, zs) = _wide_rows(x, lead, C), _wide_rows(z, lead, C)
    w = w.contiguous()
    _call(dev, "gated_group_rmsnorm_forward", load_library().gated_group_rmsnorm_forward, _p(x), xs, _p(z), zs, _p(w), _p(y),
          x.numel() // C, C, int(groups), float(eps), _DTYPES[x.dtype])
    return y

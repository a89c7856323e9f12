"""Training operators around the layer's GEMMs: token order, 8-bit activation copies, router gradient.

    idx, w = layer.route(logits, bias, factor)
    order = sort_tokens(idx, E_local, offset)                     # expert-sorted tables
    x_rows = permute(x, order)                                    # token rows in expert order      -> GEMM1 per expert
    act, q, scale = swiglu_save(g_rows, order.expert_row0)        # activation, 8-bit copy of g     -> GEMM2 per expert
    out = combine(y_rows, w, order)                               # weighted sum back per token

and in the backward pass, with what GEMM2's and GEMM1's gradients give between them,

    grad_y, grad_w = combine_backward(grad_out, y_rows, w, order)
    grad_g, act = swiglu_backward(q, scale, grad_act, order.expert_row0)      # act again: it need not be kept
    x_rows = restore_1x128(xq, xscale, order)                     # or permute(x, order): GEMM1's input rows again
    grad_x = permute_backward(grad_rows, order)
    grad_logits = route_backward(logits, bias, idx, grad_w, factor, mode)

Every call runs on the current stream of its tensors' device, whichever device is current, allocates nothing but its outputs (and a table of
counts in `sort_tokens`), keeps nothing, and can be captured into a CUDA graph.  Row tensors are bf16, fp16 or fp32; tensors that are not contiguous, or do
not start at a 32-byte boundary, are copied first (`out` tensors are refused).  Row tensors have room for `order.row_pair.numel()` rows:
`permute`, `restore_1x128` and `combine_backward` write the rows in use, padding of the segments included (as zeros).  The SwiGLU pair takes padding for
rows like any other: zeros give zeros, but what a GEMM leaves unset there comes out as whatever it makes, so GEMMs have to write zeros into it (from the
zeros that they read).  All of them leave rows behind `expert_row0[-1]` as they were (unset where the call makes the tensor).  The gradients are plain
functions: autograd does not record these calls.  A call that writes an `out` tensor counts as a change of it in place: a backward pass that had saved
it raises, as after any change in place.
"""
from __future__ import annotations

import ctypes as C
import functools
from typing import NamedTuple, Optional

import torch

from . import _lib
from .inputs import ROUTING_DS
from .main import _raw_stream

_TYPES = {torch.bfloat16: 0, torch.float16: 1, torch.float32: 2}
_BYTES = (2, 2, 4)              # by the codes above
_ALIGN = 32
_I32, _F32, _E4M3 = torch.int32, torch.float32, torch.float8_e4m3fn
_current_device = torch._C._cuda_getDevice if hasattr(torch._C, "_cuda_getDevice") else torch.cuda.current_device
_written = torch.autograd.graph.increment_version      # the caller's tensors changed: autograd refuses a backward pass that had saved them


@functools.lru_cache(maxsize=1024)
def _sort_bytes(T, K, El, device):
    """Workspace of b200moe_sort_tokens over these sizes (and smaller ones) on that device."""
    n = C.c_size_t()
    with torch.cuda.device(device):
        _lib.check(_lib.lib.b200moe_sort_workspace_bytes(T, K, El, C.byref(n)), "b200moe_sort_workspace_bytes")
    return n.value


class TokenOrder(NamedTuple):
    """Tables of `sort_tokens`, int32: first row of each local expert [E_local + 1], pair of each row [max_rows] and row of
    each pair [T, top_k]; -1 where there is none."""
    expert_row0: torch.Tensor
    row_pair: torch.Tensor
    pair_row: torch.Tensor


def _call(fn, device, *args):
    """fn(*args) with `device` current; the last argument is the device's current stream."""
    if _current_device() == device:
        rc = fn(*args)
    else:
        with torch.cuda.device(device):
            rc = fn(*args)
    if rc:
        _lib.check(rc, fn.__name__)


def _device(t, name):
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    return device


def _off(t, name, dtype, shape):
    raise ValueError(f"{name}: expected {dtype} {tuple(shape)}, got {t.dtype} {tuple(t.shape)}")


def _in(t, name, device, dtype, shape, align=1):
    """An input of a known form: (the tensor, its address); copied if it is not contiguous or not aligned."""
    if t.dtype is not dtype or t.shape != shape:
        _off(t, name, dtype, shape)
    if t.get_device() != device:
        raise ValueError(f"{name} is not on cuda:{device}")
    at = t.data_ptr()
    if at % align or not t.is_contiguous():
        t = t.clone(memory_format=torch.contiguous_format)
        at = t.data_ptr()
    return t, at


def _rows(t, name, columns=128):
    """A row tensor that tells the call's type, device and sizes: (the tensor, its address, type, device, rows, columns)."""
    kind, shape = _TYPES.get(t.dtype), t.shape
    if kind is None or len(shape) != 2:
        raise ValueError(f"{name} must be a 2-D bf16, fp16 or fp32 tensor, got {t.dtype} {tuple(shape)}")
    device = t.get_device()
    if device < 0:
        raise ValueError(f"{name} must be a CUDA tensor")
    n, H = shape
    if H <= 0 or H % columns or H > columns << 13:
        raise ValueError(f"{name}: columns must be a multiple of {columns} up to {columns << 13}, got {H}")
    at = t.data_ptr()
    if at % _ALIGN or not t.is_contiguous():
        t = t.clone(memory_format=torch.contiguous_format)
        at = t.data_ptr()
    return t, at, kind, device, n, H


def _given(t, name, device, dtype, shape, size, align, *taken):
    """The address of the caller's output of `size` bytes, which has to be of the form that is written in place and share no memory with the call's
    inputs and other outputs (their addresses and ends)."""
    at = t.data_ptr()
    if t.dtype is not dtype or t.shape != shape or t.get_device() != device or at % align or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} {tuple(shape)} tensor on cuda:{device} that starts at a multiple of {align} bytes")
    end = at + size
    for start, stop in taken:
        if start < end and at < stop:
            raise ValueError(f"{name} must not share memory with an input or another output")
    return at


def _order(order, device):
    """An order's tables (kept by the caller until the call is made), their addresses, T, top_k, E_local, rows."""
    row0, row_pair, pair_row = order
    try:
        (El,), (R,), (T, K) = row0.shape, row_pair.shape, pair_row.shape
    except ValueError:                       # another number of dimensions
        El = None
    if not (El is not None and row0.dtype is _I32 and row_pair.dtype is _I32 and pair_row.dtype is _I32 and row0.get_device() == device
            and row_pair.get_device() == device and pair_row.get_device() == device):
        raise ValueError(f"an order is int32 expert_row0 [E_local + 1], row_pair [max_rows] and pair_row [T, top_k] on cuda:{device}")
    if not (row0.is_contiguous() and row_pair.is_contiguous() and pair_row.is_contiguous()):
        order = row0, row_pair, pair_row = row0.contiguous(), row_pair.contiguous(), pair_row.contiguous()
    El -= 1
    if not (1 <= El <= 512 and 1 <= K <= 8):
        raise ValueError("an order has 1 to 512 local experts and 1 to 8 picks per token")
    return order, row0.data_ptr(), row_pair.data_ptr(), pair_row.data_ptr(), T, K, El, R


def sort_tokens(topk_idx: torch.Tensor, num_local_experts: int, local_expert_offset: int = 0, align: int = 16,
                max_rows: Optional[int] = None) -> TokenOrder:
    """Expert-sorted tables of the picks `topk_idx` (int32 [T, top_k], as `MoELayer.route` gives them): every pick of an expert in
    [local_expert_offset, local_expert_offset + num_local_experts) gets a row, in ascending (token, pick) order inside an expert, experts' segments
    padded to multiples of `align` rows (a power of two up to 128).  Other picks get none.  `max_rows`: room of the row tensors, by default
    enough for every case; pairs whose row would lie behind it get none."""
    if topk_idx.dim() != 2 or topk_idx.dtype != torch.int32:
        raise ValueError(f"topk_idx must be int32 [T, top_k], got {topk_idx.dtype} {tuple(topk_idx.shape)}")
    device = _device(topk_idx, "topk_idx")
    T, K = topk_idx.shape
    El, align, local_expert_offset = int(num_local_experts), int(align), int(local_expert_offset)
    if not 1 <= K <= 8 or not 1 <= El <= 512 or T * K > 1 << 30:
        raise ValueError("1 to 8 picks per token, 1 to 512 local experts, at most 2^30 pairs")
    if align not in (1, 2, 4, 8, 16, 32, 64, 128):
        raise ValueError("align must be a power of two up to 128")
    rows = T * K + (align - 1) * El if max_rows is None else int(max_rows)
    if not 0 <= rows <= 1 << 30 or not -(1 << 31) <= local_expert_offset < (1 << 31):
        raise ValueError("max_rows or local_expert_offset out of range")
    topk_idx, idx_at = _in(topk_idx, "topk_idx", device, _I32, (T, K))
    n = _sort_bytes(T, K, El, device)
    dev = topk_idx.device
    row0 = torch.empty(El + 1, dtype=_I32, device=dev)
    row_pair = torch.empty(rows, dtype=_I32, device=dev)
    pair_row = torch.empty_like(topk_idx)
    counts = torch.empty(n, dtype=torch.uint8, device=dev) if n else None
    _call(_lib.lib.b200moe_sort_tokens, device, idx_at, T, K, El, local_expert_offset, align, rows, row0.data_ptr(), row_pair.data_ptr(),
          pair_row.data_ptr(), None if counts is None else counts.data_ptr(), n, _raw_stream(device))
    return TokenOrder(row0, row_pair, pair_row)


def permute(x: torch.Tensor, order: TokenOrder, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[T, H] -> [max_rows, H]: row r is the row of its pair's token, zeros in the padding of a segment."""
    x, x_at, kind, device, n, H = _rows(x, "x")
    order, row0, row_pair, pair_row, T, K, El, R = _order(order, device)
    if n != T:
        _off(x, "x", x.dtype, (T, H))
    made = out is None
    if made:
        out = x.new_empty((R, H))
        at = out.data_ptr()
    else:
        row = H * _BYTES[kind]
        at = _given(out, "out", device, x.dtype, (R, H), R * row, _ALIGN, (x_at, x_at + T * row), (row0, row0 + 4 * El + 4),
                    (row_pair, row_pair + 4 * R), (pair_row, pair_row + 4 * T * K))
    _call(_lib.lib.b200moe_permute, device, x_at, kind, row0, row_pair, pair_row, T, K, El, H, R, at, _raw_stream(device))
    if not made:
        _written(out)
    return out


def _combine(rows, w, order, out):
    rows, rows_at, kind, device, n, H = _rows(rows, "rows")
    order, _, _, pair_row, T, K, _, R = _order(order, device)
    if n != R:
        _off(rows, "rows", rows.dtype, (R, H))
    w, w_at = (None, None) if w is None else _in(w, "topk_w", device, _F32, (T, K))
    made = out is None
    if made:
        out = rows.new_empty((T, H))
        at = out.data_ptr()
    else:
        row = H * _BYTES[kind]
        at = _given(out, "out", device, rows.dtype, (T, H), T * row, _ALIGN, (rows_at, rows_at + R * row), (pair_row, pair_row + 4 * T * K),
                    (0, 0) if w is None else (w_at, w_at + 4 * T * K))
    _call(_lib.lib.b200moe_combine, device, rows_at, kind, w_at, pair_row, T, K, H, R, at, _raw_stream(device))
    if not made:
        _written(out)
    return out


def permute_backward(grad_rows: torch.Tensor, order: TokenOrder, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of `permute` (and of `restore_1x128`, as far as the activations go): [max_rows, H] -> [T, H], the sum over a
    token's rows in fp32, rounded once."""
    return _combine(grad_rows, None, order, out)


def combine(rows: torch.Tensor, topk_w: torch.Tensor, order: TokenOrder, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """[max_rows, H] and routing weights fp32 [T, top_k] -> [T, H]: the weighted sum over a token's rows in fp32, rounded once;
    zeros for a token without rows."""
    return _combine(rows, topk_w, order, out)


def combine_backward(grad_out: torch.Tensor, rows: torch.Tensor, topk_w: torch.Tensor, order: TokenOrder, out: Optional[torch.Tensor] = None):
    """Gradients of `combine`: (grad_rows [max_rows, H], grad_w fp32 [T, top_k]); `out` takes the first."""
    rows, rows_at, kind, device, n, H = _rows(rows, "rows")
    order, row0, row_pair, pair_row, T, K, El, R = _order(order, device)
    if n != R:
        _off(rows, "rows", rows.dtype, (R, H))
    grad_out, grad_at = _in(grad_out, "grad_out", device, rows.dtype, (T, H), _ALIGN)
    topk_w, w_at = _in(topk_w, "topk_w", device, _F32, (T, K))
    made = out is None
    if made:
        out = torch.empty_like(rows)
        at = out.data_ptr()
    else:
        row = H * _BYTES[kind]
        at = _given(out, "out", device, rows.dtype, (R, H), R * row, _ALIGN, (rows_at, rows_at + R * row), (grad_at, grad_at + T * row),
                    (w_at, w_at + 4 * T * K), (row0, row0 + 4 * El + 4), (row_pair, row_pair + 4 * R), (pair_row, pair_row + 4 * T * K))
    grad_w = torch.empty_like(topk_w)
    _call(_lib.lib.b200moe_combine_backward, device, grad_at, rows_at, kind, w_at, row0, row_pair, pair_row, T, K, El, H, R, at, grad_w.data_ptr(),
          _raw_stream(device))
    if not made:
        _written(out)
    return out, grad_w


def restore_1x128(q: torch.Tensor, scale: torch.Tensor, order: Optional[TokenOrder] = None, dtype=torch.bfloat16,
                  out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Activations kept in 8 bits (e4m3 [T, H] and scales [H/128, T], as `quantize_1x128` makes them) read back as `dtype` (that of `out`, where it is
    given): [T, H], or, with an order, rows in expert order like `permute`'s."""
    if q.dim() != 2:
        raise ValueError("q must be e4m3 [T, H]")
    device = _device(q, "q")
    T, H = q.shape
    if H <= 0 or H % 128 or H > 1 << 20:
        raise ValueError(f"q: columns must be a multiple of 128 up to 2^20, got {H}")
    if out is not None:
        dtype = out.dtype
    kind = _TYPES.get(dtype)
    if kind is None:
        raise ValueError(f"rows are bf16, fp16 or fp32, not {dtype}")
    q, q_at = _in(q, "q", device, _E4M3, (T, H), 16)
    scale, scale_at = _in(scale, "scale", device, _F32, (H // 128, T))
    if order is None:
        row0 = row_pair = pair_row = None
        K, El, R = 1, 1, T
    else:
        order, row0, row_pair, pair_row, tokens, K, El, R = _order(order, device)
        if tokens != T:
            raise ValueError(f"q has {T} tokens, the order {tokens}")
    made = out is None
    if made:
        out = q.new_empty((R, H), dtype=dtype)
        at = out.data_ptr()
    else:
        tables = () if order is None else ((row0, row0 + 4 * El + 4), (row_pair, row_pair + 4 * R), (pair_row, pair_row + 4 * T * K))
        at = _given(out, "out", device, dtype, (R, H), R * H * _BYTES[kind], _ALIGN, (q_at, q_at + T * H), (scale_at, scale_at + T * H // 32), *tables)
    _call(_lib.lib.b200moe_restore_1x128, device, q_at, scale_at, kind, row0, row_pair, pair_row, T, K, El, H, R, at, _raw_stream(device))
    if not made:
        _written(out)
    return out


def _used(expert_row0, device):
    """(the table, kept by the caller until the call is made; its address and end; the address of its last entry: the number of rows in use)"""
    if expert_row0 is None:
        return None, (0, 0), None
    shape = expert_row0.shape
    if len(shape) != 1 or shape[0] < 1:
        raise ValueError("expert_row0 must be int32 [E_local + 1]")
    t, at = _in(expert_row0, "expert_row0", device, _I32, shape)
    end = at + 4 * shape[0]
    return t, (at, end), end - 4


def swiglu_save(gemm1_rows: torch.Tensor, expert_row0: Optional[torch.Tensor] = None, out=None):
    """[R, 2I] -> (act [R, I] = rows[:, :I] * silu(rows[:, I:]), q e4m3 [R, 2I], scale fp32 [2I/128, R]): the activation, and the 8-bit copy
    of its inputs for `swiglu_backward`.  A group of 128 columns is scaled by the smallest power of two not below its largest
    magnitude / 448; one that holds an infinity or a NaN gets the scale NaN.  `expert_row0`: only its last entry's number of rows is in use (None:
    all).  `out`: the three tensors to write."""
    x, x_at, kind, device, R, I2 = _rows(gemm1_rows, "gemm1_rows", 256)
    keep, table, used = _used(expert_row0, device)
    if out is None:
        act, q = x.new_empty((R, I2 // 2)), x.new_empty((R, I2), dtype=_E4M3)
        scale = x.new_empty((I2 // 128, R), dtype=_F32)
        act_at, q_at, scale_at = act.data_ptr(), q.data_ptr(), scale.data_ptr()
    else:
        act, q, scale = out
        act_bytes, n = R * I2 // 2 * _BYTES[kind], R * I2
        ins = (x_at, x_at + 2 * act_bytes)
        act_at = _given(act, "act", device, x.dtype, (R, I2 // 2), act_bytes, _ALIGN, ins, table)
        acts = (act_at, act_at + act_bytes)
        q_at = _given(q, "q", device, _E4M3, (R, I2), n, 16, ins, table, acts)
        scale_at = _given(scale, "scale", device, _F32, (I2 // 128, R), n // 32, 4, ins, table, acts, (q_at, q_at + n))
    _call(_lib.lib.b200moe_swiglu_save, device, x_at, kind, used, R, I2 // 2, act_at, q_at, scale_at, _raw_stream(device))
    if out is not None:
        _written((act, q, scale))
    return act, q, scale


def swiglu_backward(q: torch.Tensor, scale: torch.Tensor, grad_act: torch.Tensor, expert_row0: Optional[torch.Tensor] = None,
                    with_act: bool = True, out=None):
    """Gradient of `swiglu_save`'s activation from its 8-bit copy: (grad of gemm1_rows [R, 2I], act [R, I] again or None), both of
    grad_act's type.  `out`: the two tensors to write (the second None without `with_act`)."""
    d, d_at, kind, device, R, I = _rows(grad_act, "grad_act")
    keep, table, used = _used(expert_row0, device)
    q, q_at = _in(q, "q", device, _E4M3, (R, 2 * I), 16)
    scale, scale_at = _in(scale, "scale", device, _F32, (2 * I // 128, R))
    if out is None:
        grad_x, act = d.new_empty((R, 2 * I)), torch.empty_like(d) if with_act else None
        grad_at, act_at = grad_x.data_ptr(), act.data_ptr() if with_act else None
    else:
        grad_x, act = out
        if (act is not None) != with_act:
            raise ValueError("out has a tensor for act if and only if with_act asks for it")
        n = R * I * _BYTES[kind]
        ins = (q_at, q_at + 2 * R * I), (scale_at, scale_at + R * I // 16), (d_at, d_at + n), table
        grad_at = _given(grad_x, "grad_gemm1_rows", device, d.dtype, (R, 2 * I), 2 * n, _ALIGN, *ins)
        act_at = _given(act, "act", device, d.dtype, (R, I), n, _ALIGN, *ins, (grad_at, grad_at + 2 * n)) if with_act else None
    _call(_lib.lib.b200moe_swiglu_backward, device, q_at, scale_at, d_at, kind, used, R, I, grad_at, act_at, _raw_stream(device))
    if out is not None:
        _written((grad_x, act) if with_act else grad_x)
    return grad_x, act


def route_backward(routing_logits: torch.Tensor, routing_bias: Optional[torch.Tensor], topk_idx: torch.Tensor, grad_w: torch.Tensor,
                   routed_scaling_factor, routing_mode: int = ROUTING_DS, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Gradient of the routing weights (`MoELayer.route` with the same logits, bias, factor and mode, which gave the picks
    `topk_idx`) down to the logits: fp32 [T, E].  In modes 1 to 5 the bias's gradient is its column sum; in mode 0 the bias only selects."""
    if routing_logits.dim() != 2 or topk_idx.dim() != 2:
        raise ValueError("routing_logits must be [T, E] and topk_idx [T, top_k]")
    device = _device(routing_logits, "routing_logits")
    (T, E), K = routing_logits.shape, topk_idx.shape[1]
    if E < 32 or E > 512 or E % 32 or not 1 <= K <= 8:
        raise ValueError("E must be a multiple of 32 up to 512, top_k 1 to 8")
    routing_mode = int(routing_mode)
    if not 0 <= routing_mode <= 5 or (routing_mode == 4 and K != 1):
        raise ValueError("routing_mode must be one of ROUTING_* (0 to 5; mode 4 picks one expert)")
    logits, logits_at = _in(routing_logits, "routing_logits", device, _F32, (T, E), 16)
    bias, bias_at = (None, None) if routing_bias is None else _in(routing_bias, "routing_bias", device, torch.bfloat16, (E,))
    topk_idx, idx_at = _in(topk_idx, "topk_idx", device, _I32, (T, K))
    grad_w, grad_at = _in(grad_w, "grad_w", device, _F32, (T, K))
    made = out is None
    if made:
        out = torch.empty_like(logits)
        at = out.data_ptr()
    else:
        at = _given(out, "out", device, _F32, (T, E), 4 * T * E, 16, (logits_at, logits_at + 4 * T * E), (idx_at, idx_at + 4 * T * K),
                    (grad_at, grad_at + 4 * T * K), (0, 0) if bias is None else (bias_at, bias_at + 2 * E))
    _call(_lib.lib.b200moe_route_backward, device, logits_at, bias_at, idx_at, grad_at, T, E, K, float(routed_scaling_factor), routing_mode, at,
          _raw_stream(device))
    if not made:
        _written(out)
    return out

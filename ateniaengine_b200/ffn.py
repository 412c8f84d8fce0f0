"""The dense gated feed-forward block, its backward pass, and low-rank adapters of many requests beside shared projections.

The dense counterpart of an MoE layer's expert (gate, up, SwiGLU, down) for the layers of a model that have no router, for training
it, and for serving it with one adapter per request.  Every computation runs in the CUDA library; torch owns the memory (the
calls take their workspace from its allocator, on the current stream) and nothing is recorded for torch's autograd: a training
step calls `gated_ffn_backward` itself, or wraps the two calls in a torch.autograd.Function of its own.  An x that requires a gradient is
refused while torch records.
"""
import ctypes as C
import functools
import struct
from typing import NamedTuple

import torch

from . import _lib
from .moe import _launching

BF16 = torch.bfloat16
_PARTS = {"gate", "up", "down"}
_MAX_ROWS, _MAX_WIDTH = 1 << 24, 1 << 20  # (the library's sizes are 32 bits: larger ones would come to it as others)


class LowRankAdapters(NamedTuple):
    """n adapters of one projection [out, in]: token t of adapter i adds scale[i] * (x_t A_i^T) B_i^T.

    a: CUDA bf16 [n, rank, in]; b: CUDA bf16 [n, out, rank]; scale: CUDA f32 [n].  rank: a multiple of 8 up to 128 (zero-pad a's rows
    and b's columns otherwise)."""
    a: torch.Tensor
    b: torch.Tensor
    scale: torch.Tensor


def _operand(t, name, shape, dtype, device):
    """`t`, contiguous, where it is a tensor of this shape and type on this device; else the refusal.  (One test where all is well: the
    checks of a call cost as much host time as a launch.)"""
    if isinstance(t, torch.Tensor) and t.dtype is dtype and t.shape == shape and t.device == device:
        return t if t.is_contiguous() else t.contiguous()
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a tensor")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} must have shape {shape}, got {tuple(t.shape)}")
    raise ValueError(f"{name} is on {t.device}, x on {device}")


def _rows(x, recorded=False):
    """x, contiguous.  `recorded` False: the result has no history, so that an x that has one would lose its gradient without a word.
    (Parameters are ordinary arguments: a program that calls gated_ffn_backward itself passes them.)"""
    if not isinstance(x, torch.Tensor) or x.dtype is not BF16:
        raise TypeError("x must be a bf16 tensor")
    shape = x.shape
    if len(shape) != 2:
        raise ValueError(f"x must be [tokens, width], got {tuple(shape)}")
    if shape[0] > _MAX_ROWS:
        raise ValueError(f"x: at most 2^24 tokens, got {shape[0]}")
    if not recorded and x.requires_grad and torch.is_grad_enabled():
        raise ValueError("x requires a gradient, which this call does not record: detach it, call under torch.no_grad(), or from a "
                         "torch.autograd.Function")
    if not x.is_cuda:
        raise ValueError("x must be a CUDA tensor")
    return x if x.is_contiguous() else x.contiguous()


def _output(out, shape, x):
    if out is None:
        return torch.empty_like(x) if shape == x.shape else x.new_empty(shape)
    if not isinstance(out, torch.Tensor) or out.dtype is not BF16 or out.shape != shape or out.device != x.device:
        raise ValueError(f"out must be a bf16 tensor of shape {shape} on {x.device}")
    if not out.is_contiguous():
        raise ValueError("out must be contiguous")
    return out


# AteniaLowRank and AteniaFfnAdapters as their bytes: a fifth of the time that filling in ctypes structures takes
_LOW_RANK = struct.Struct("@PPPii")
_FFN_ADAPTERS = struct.Struct("@" + 3 * "PPPii" + "Pii")
_NONE = (0, 0, 0, 0, 0)
assert _LOW_RANK.size == C.sizeof(_lib.LowRank) and _FFN_ADAPTERS.size == C.sizeof(_lib.FfnAdapters)


def _low_rank(set_, name, n_in, n_out, device):
    """The fields of AteniaLowRank of one projection's adapters, how many there are, and the tensors they point to."""
    a, b, scale = set_
    if not isinstance(a, torch.Tensor) or a.dim() != 3:
        raise ValueError(f"{name}.a must be [n, rank, {n_in}]")
    n, rank, _ = a.shape
    if n < 1 or rank < 8 or rank > 128 or rank % 8:
        raise ValueError(f"{name}: at least one adapter, of a rank that is a multiple of 8 up to 128, got {tuple(a.shape)}")
    a = _operand(a, name + ".a", (n, rank, n_in), BF16, device)
    b = _operand(b, name + ".b", (n, n_out, rank), BF16, device)
    scale = _operand(scale, name + ".scale", (n,), torch.float32, device)
    return (a.data_ptr(), b.data_ptr(), scale.data_ptr(), rank, 0), n, (a, b, scale)


# Bytes of a call's workspace: functions of the sizes alone.
@functools.lru_cache(maxsize=256)
def _ffn_bytes(T, d, F, r_gate, r_up, r_down, backward):
    ranks = _FFN_ADAPTERS.pack(0, 0, 0, r_gate, 0, 0, 0, 0, r_up, 0, 0, 0, 0, r_down, 0, 0, 0, 0)
    return _lib.lib().atenia_gated_ffn_workspace_bytes(T, d, F, ranks, backward)


@functools.lru_cache(maxsize=256)
def _linear_bytes(T, rank):
    return _lib.lib().atenia_adapter_linear_workspace_bytes(T, rank)


def _workspace(nbytes, x):
    return x.new_empty(nbytes // 2 or 1)  # (bf16 elements; the sizes are multiples of 256)


def _check_widths(a, b, what):
    if a < 16 or b < 16 or a % 16 or b % 16 or a > _MAX_WIDTH or b > _MAX_WIDTH:
        raise ValueError(f"{what} must be multiples of 16, at most 2^20, got {a} and {b}")


def _projection(x, weight):
    """tokens, in, out and the checked weight [out, in] of adapter_linear."""
    if not isinstance(weight, torch.Tensor) or weight.dim() != 2:
        raise ValueError("weight must be [out, in]")
    T, n_in = x.shape
    n_out = weight.shape[0]
    _check_widths(n_in, n_out, "the projection's sizes")
    return T, n_in, n_out, _operand(weight, "weight", (n_out, n_in), BF16, x.device)


def _block(x, gate, up, down):
    if not isinstance(gate, torch.Tensor) or gate.dim() != 2:
        raise ValueError("gate must be [d_ff, d_model]")
    T, d = x.shape
    F = gate.shape[0]
    _check_widths(d, F, "d_model and d_ff")
    device = x.device
    return (T, d, F, _operand(gate, "gate", (F, d), BF16, device), _operand(up, "up", (F, d), BF16, device),
            _operand(down, "down", (d, F), BF16, device))


def _block_adapters(adapters, adapter_ids, T, d, F, save, device):
    """AteniaFfnAdapters, the three ranks, and the tensors it points to."""
    if save:
        raise ValueError("the backward pass is that of the block without adapters: save=True takes none")
    if not adapters.keys() <= _PARTS:
        raise ValueError(f"adapters of {sorted(set(adapters) - _PARTS)}: the block has gate, up and down")
    ids = _operand(adapter_ids, "adapter_ids", (T,), torch.int32, device)
    fields, n, ranks, keep = (), 0, [], [ids]
    for name in ("gate", "up", "down"):
        set_ = adapters.get(name)
        if set_ is None:
            fields += _NONE
            ranks.append(0)
            continue
        low, here, tensors = _low_rank(set_, name, F if name == "down" else d, d if name == "down" else F, device)
        if n not in (0, here):
            raise ValueError("the projections have different numbers of adapters")
        n = here
        fields += low
        ranks.append(low[3])
        keep.append(tensors)
    if n == 0:
        raise ValueError("adapter_ids without adapters")
    return _FFN_ADAPTERS.pack(*fields, ids.data_ptr(), n, 0), ranks, keep


def gated_ffn(x, gate, up, down, adapters=None, adapter_ids=None, save=False, out=None, sync=False):
    """y = (silu(x gate^T) * (x up^T)) down^T, not recorded for autograd.  x: CUDA bf16 [T, d], T up to 2^24; gate, up: bf16 [F, d];
    down: bf16 [d, F].

    `adapters`: a dict of LowRankAdapters for any of "gate", "up", "down" (the same number in each), with `adapter_ids` int32 [T]:
    the adapter of each token, outside [0, n) for none.  `save=True` returns (y, saved) for gated_ffn_backward; saved is f32
    [2, F / 4, T, 4], the two projections before the activation.  `out` may be x, and overlaps nothing else that is read.
    `sync=True` waits and raises what the kernels recorded."""
    x = _rows(x)
    T, d, F, gate, up, down = _block(x, gate, up, down)
    ad, ranks = None, (0, 0, 0)
    if adapters:
        ad, ranks, keep = _block_adapters(adapters, adapter_ids, T, d, F, save, x.device)
    elif adapter_ids is not None:
        raise ValueError("adapter_ids without adapters")
    y = _output(out, (T, d), x)
    saved, at_gate, at_up = None, None, None
    if save:
        saved = x.new_empty((2, F // 4, T, 4), dtype=torch.float32)
        at_gate = saved.data_ptr()
        at_up = at_gate + 4 * T * F
    nbytes = _ffn_bytes(T, d, F, *ranks, 0)
    ws = _workspace(nbytes, x)
    lib = _lib.lib()
    with _launching(x.device) as st:
        rc = lib.atenia_gated_ffn_forward(x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), T, d, F,
                                          ad, y.data_ptr(), at_gate, at_up, ws.data_ptr(), nbytes, st)
        if rc or sync:
            _lib.check(rc or lib.atenia_ffn_check(st), "gated_ffn")
    return (y, saved) if save else y


def gated_ffn_backward(dy, x, gate, up, down, saved, sync=False):
    """Gradients of gated_ffn(x, gate, up, down) for the gradient dy [T, d] of its output, from what save=True returned:
    (dx [T, d], dgate [F, d], dup [F, d], ddown [d, F]), bf16.  `saved` is left as it is."""
    x = _rows(x, recorded=True)  # (nothing is asked of autograd here)
    T, d, F, gate, up, down = _block(x, gate, up, down)
    dy = _operand(dy, "dy", (T, d), BF16, x.device)
    saved = _operand(saved, "saved", (2, F // 4, T, 4), torch.float32, x.device)
    dx = torch.empty_like(x)
    dgate, dup, ddown = torch.empty_like(gate), torch.empty_like(up), torch.empty_like(down)
    nbytes = _ffn_bytes(T, d, F, 0, 0, 0, 1)
    ws = _workspace(nbytes, x)
    at_gate = saved.data_ptr()
    lib = _lib.lib()
    with _launching(x.device) as st:
        rc = lib.atenia_gated_ffn_backward(dy.data_ptr(), x.data_ptr(), gate.data_ptr(), up.data_ptr(), down.data_ptr(), at_gate,
                                           at_gate + 4 * T * F, T, d, F, dx.data_ptr(), dgate.data_ptr(), dup.data_ptr(),
                                           ddown.data_ptr(), ws.data_ptr(), nbytes, st)
        if rc or sync:
            _lib.check(rc or lib.atenia_ffn_check(st), "gated_ffn_backward")
    return dx, dgate, dup, ddown


def adapter_linear(x, weight, adapters, adapter_ids, out=None, sync=False):
    """y = x weight^T + scale[i] * (x A_i^T) B_i^T with i = adapter_ids[t], outside [0, n) for none: one shared projection with the
    adapters of many requests.  x: CUDA bf16 [T, in]; weight: bf16 [out, in]; adapters: LowRankAdapters; adapter_ids: int32 [T].
    `out` must not overlap what is read."""
    x = _rows(x)
    T, n_in, n_out, weight = _projection(x, weight)
    device = x.device
    ids = _operand(adapter_ids, "adapter_ids", (T,), torch.int32, device)
    low, n, keep = _low_rank(adapters, "adapters", n_in, n_out, device)
    y = _output(out, (T, n_out), x)
    nbytes = _linear_bytes(T, low[3])
    ws = _workspace(nbytes, x)
    lib = _lib.lib()
    with _launching(device) as st:
        rc = lib.atenia_adapter_linear(x.data_ptr(), weight.data_ptr(), T, n_in, n_out, _LOW_RANK.pack(*low), ids.data_ptr(), n, y.data_ptr(),
                                       ws.data_ptr(), nbytes, st)
        if rc or sync:
            _lib.check(rc or lib.atenia_ffn_check(st), "adapter_linear")
    return y

"""Operators of [B, T, C] sequences: the causal depthwise convolution, the gated linear recurrence
and the layer norm, forward and backward, and the one-row steps that serve token by token.

They have no counterpart in the reference, whose maps are two-dimensional; names, argument checks,
streams and errors follow ``depthwise_conv2d``.  Kernels: ``csrc/seq_*.cu`` through the C entry
points of ``include/dwconv_b200.h``.  fp32, fp16 and bf16 tensors; arithmetic and the recurrence's state in
fp32 (the convolution's state holds input rows, in their type).

Packed sequences: ``offsets`` is an int32 tensor of S + 1 ascending row numbers on the input's device
(``offsets[0] == 0``); the input is [1, T, C] and sequence j is its rows ``offsets[j]`` to
``offsets[j + 1] - 1``, none where the two are equal.  Rows behind ``offsets[S]`` belong to no
sequence: zeros in every output, and what they hold is not looked at.  The list stays on the device;
a list that is not ascending gives unspecified values (never an access out of bounds).

Every function runs on the current stream of the input's device, never synchronises, and may be
captured into a CUDA graph.  Gradients are first-order and reverse-mode only: with ``create_graph`` they carry
an error for whoever differentiates them.  A backward pass is not to be captured while an eager graph of the same
leaves is alive on the default stream: PyTorch's engine would break the capture, which can end the process.  The
compiled module refuses it where its own nodes lead to such a leaf; without the module nothing notices.
"""
import functools

import torch
from torch import nn
from torch.autograd import Function

from . import _C, _lib
from .dwconv import _ACTIVATIONS, _native

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


# ---- over ctypes: the same functions as csrc/torch_binding.cpp ---------------------------------

def _ptr(t):
    return t.data_ptr() if t is not None else None


def _sequence_dtype(t):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise RuntimeError(f"dwconv_b200: unsupported dtype {_dtype_name(t.dtype)} (float32, float16, bfloat16)")
    return code


def _dtype_name(dtype):
    # the names C++ uses in messages
    return {torch.float32: "float", torch.float64: "double", torch.float16: "c10::Half",
            torch.bfloat16: "c10::BFloat16", torch.int32: "int", torch.int64: "long"}.get(dtype, str(dtype))


def _rows_of(t):
    """Channels side by side; any other strides are read as they are."""
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


def _rows_arg(t):
    return _lib.Rows(t.data_ptr(), t.stride(0), t.stride(1))


def _contiguous(t):
    return t.contiguous() if t is not None else None


def _check_operand(fn, name, t, shape, dtype, input):
    if t.device != input.device or t.dtype != dtype:
        raise RuntimeError(f"dwconv_b200.{fn}: {name} must be {_dtype_name(dtype)} on {input.device}, "
                           f"got {_dtype_name(t.dtype)} on {t.device}")
    if tuple(t.shape) != tuple(shape):
        raise RuntimeError(f"dwconv_b200.{fn}: {name} must be {tuple(shape)}, got {tuple(t.shape)}")


def _check_kept(fn, name, t, shape, input):
    # what the forward call left, and hooks on saved tensors may have had in hand since
    _check_operand(fn, name, t, shape, torch.float32, input)
    if not t.is_contiguous():
        raise RuntimeError(f"dwconv_b200.{fn}: {name} must be contiguous")


def _check_sequences(fn, input, offsets):
    _C._check_cuda(input, "input")
    _sequence_dtype(input)
    if input.dim() != 3:
        raise RuntimeError(f"dwconv_b200.{fn}: expected input [B, T, C], got {tuple(input.shape)}")
    if max(input.shape) > 1 << 30:
        raise RuntimeError(f"dwconv_b200.{fn}: input is too large: {tuple(input.shape)}")
    s = _lib.Sequence(*input.shape, None, 0)
    if offsets is not None:
        if not (offsets.device == input.device and offsets.dtype == torch.int32 and offsets.dim() == 1
                and offsets.is_contiguous() and offsets.shape[0] >= 2):
            raise RuntimeError(f"dwconv_b200.{fn}: offsets must be a contiguous 1-d int32 tensor of at least "
                               f"2 row numbers on {input.device}")
        if s.B != 1:
            raise RuntimeError(f"dwconv_b200.{fn}: packed sequences (offsets) need a batch of 1, got {s.B}")
        s.offsets = offsets.data_ptr()
        s.S = offsets.shape[0] - 1
    return s


def _state_or_zeros(state, shape, dtype, device):
    if state is not None:
        return state.clone(memory_format=torch.contiguous_format)
    return torch.zeros(shape, dtype=dtype, device=device)


def _check_weight(fn, weight, C, input):
    if not (weight.dim() == 3 and weight.shape[0] == C and weight.shape[1] == 1
            and 1 <= weight.shape[2] <= _lib.MAX_TAPS):
        raise RuntimeError(f"dwconv_b200.{fn}: weight must be [C, 1, taps] with C = {C} and 1 to "
                           f"{_lib.MAX_TAPS} taps, got {tuple(weight.shape)}")
    _check_operand(fn, "weight", weight, weight.shape, input.dtype, input)
    return weight.shape[2]


def _check_conv1d(fn, input, weight, bias, initial, offsets):
    s = _check_sequences(fn, input, offsets)
    taps = _check_weight(fn, weight, s.C, input)
    if bias is not None:
        _check_operand(fn, "bias", bias, (s.C,), input.dtype, input)
    state = (s.S if s.offsets else s.B, taps - 1, s.C)
    if initial is not None:
        _check_operand(fn, "initial_state", initial, state, input.dtype, input)
    return s, taps, state


def _conv1d_causal(input, weight, bias, act, initial, offsets, want_state):
    fn = "depthwise_conv1d_causal"
    s, taps, state_shape = _check_conv1d(fn, input, weight, bias, initial, offsets)
    y = torch.empty(input.shape, dtype=input.dtype, device=input.device)
    state = None
    if input.numel() == 0:
        if want_state:
            state = _state_or_zeros(initial, state_shape, input.dtype, input.device)
        return y, state
    if want_state:
        state = torch.empty(state_shape, dtype=input.dtype, device=input.device)
    x, w, b, init = _rows_of(input), weight.contiguous(), _contiguous(bias), _contiguous(initial)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_conv1d_causal(
            _rows_arg(x), w.data_ptr(), _ptr(b), _ptr(init), y.data_ptr(), _ptr(state), _DTYPES[x.dtype],
            s, taps, act, _C._stream(input))
    _lib.check(st, fn)
    return y, state


def _conv1d_causal_backward(input, weight, bias, act, initial, offsets, grad, grad_state, want_initial):
    fn = "depthwise_conv1d_causal backward"
    s, taps, state_shape = _check_conv1d(fn, input, weight, bias, initial, offsets)
    if grad is not None:
        _check_operand(fn, "grad_output", grad, input.shape, input.dtype, input)
    if grad_state is not None:
        _check_operand(fn, "grad_state", grad_state, state_shape, input.dtype, input)
    like = dict(dtype=input.dtype, device=input.device)
    db = dinit = None
    if input.numel() == 0:
        if bias is not None:
            db = torch.zeros(bias.shape, **like)
        if want_initial:
            dinit = _state_or_zeros(grad_state, state_shape, input.dtype, input.device)
        return torch.empty(input.shape, **like), torch.zeros(weight.shape, **like), db, dinit
    dx, dw = torch.empty(input.shape, **like), torch.empty(weight.shape, **like)
    if bias is not None:
        db = torch.empty(bias.shape, **like)
    if want_initial:
        dinit = torch.empty(state_shape, **like)
    x, w, b, init = _rows_of(input), weight.contiguous(), _contiguous(bias), _contiguous(initial)
    g = _rows_of(grad) if grad is not None else torch.zeros(input.shape, **like)
    gs = _contiguous(grad_state)
    code = _DTYPES[x.dtype]
    nbytes = int(_lib.lib.dwconv_b200_conv1d_causal_workspace_bytes(code, s, taps))
    if nbytes == 0:
        raise RuntimeError(f"dwconv_b200.{fn}: invalid geometry")
    ws = torch.empty(nbytes, dtype=torch.uint8, device=input.device)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_conv1d_causal_backward(
            _rows_arg(x), w.data_ptr(), _ptr(b), _ptr(init), _rows_arg(g), _ptr(gs), dx.data_ptr(),
            dw.data_ptr(), _ptr(db), _ptr(dinit), ws.data_ptr(), nbytes, code, s, taps, act,
            _C._stream(input))
    _lib.check(st, fn)
    return dx, dw, db, dinit


def _check_step_input(fn, input):
    _C._check_cuda(input, "input")
    _sequence_dtype(input)
    if input.dim() != 2:
        raise RuntimeError(f"dwconv_b200.{fn}: expected input [B, C], got {tuple(input.shape)}")
    if max(input.shape) > 1 << 30:
        raise RuntimeError(f"dwconv_b200.{fn}: input is too large: {tuple(input.shape)}")


def _check_state(fn, state, shape, dtype, input):
    _check_operand(fn, "state", state, shape, dtype, input)
    if not state.is_contiguous():
        raise RuntimeError(f"dwconv_b200.{fn}: state is updated in place and must be contiguous")


def _note_written(t):
    # the kernels write through raw pointers: a graph that saved this state must learn of it
    if not t.is_inference():
        torch.autograd.graph.increment_version(t)


def _conv1d_causal_step(input, weight, state, bias, act):
    fn = "depthwise_conv1d_causal_step"
    _check_step_input(fn, input)
    B, C = input.shape
    taps = _check_weight(fn, weight, C, input)
    if bias is not None:
        _check_operand(fn, "bias", bias, (C,), input.dtype, input)
    _check_state(fn, state, (B, taps - 1, C), input.dtype, input)
    y = torch.empty((B, C), dtype=input.dtype, device=input.device)
    if input.numel() == 0:
        return y
    _note_written(state)
    x, w, b = _rows_of(input), weight.contiguous(), _contiguous(bias)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_conv1d_causal_step(
            x.data_ptr(), x.stride(0), w.data_ptr(), _ptr(b), state.data_ptr(), y.data_ptr(),
            _DTYPES[x.dtype], B, C, taps, act, _C._stream(input))
    _lib.check(st, fn)
    return y


def _check_recurrence(fn, input, u, v, decay, initial, offsets, scale):
    s = _check_sequences(fn, input, offsets)
    _check_operand(fn, "recurrence_gate", u, input.shape, input.dtype, input)
    _check_operand(fn, "input_gate", v, input.shape, input.dtype, input)
    _check_operand(fn, "decay", decay, (s.C,), torch.float32, input)
    state = (s.S if s.offsets else s.B, s.C)
    if initial is not None:
        _check_operand(fn, "initial_state", initial, state, torch.float32, input)
    if not scale > 0:
        raise RuntimeError(f"dwconv_b200.{fn}: scale must be positive")
    return s, state


def _recurrence(input, u, v, decay, initial, offsets, scale, want_state, want_backward):
    fn = "gated_linear_recurrence"
    s, state_shape = _check_recurrence(fn, input, u, v, decay, initial, offsets, scale)
    y = torch.empty(input.shape, dtype=input.dtype, device=input.device)
    wide = dict(dtype=torch.float32, device=input.device)
    state = ckpt = None
    if input.numel() == 0:
        if want_state:
            state = _state_or_zeros(initial, state_shape, torch.float32, input.device)
        return y, state, torch.empty(0, **wide) if want_backward else None
    if want_state:
        state = torch.empty(state_shape, **wide)
    if want_backward:
        ckpt = torch.empty(int(_lib.lib.dwconv_b200_recurrence_checkpoint_bytes(s)) // 4, **wide)
    x, u, v, d, init = _rows_of(input), _rows_of(u), _rows_of(v), decay.contiguous(), _contiguous(initial)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_recurrence(
            _rows_arg(x), _rows_arg(u), _rows_arg(v), d.data_ptr(), _ptr(init), y.data_ptr(), _ptr(state),
            _ptr(ckpt), _DTYPES[x.dtype], s, scale, _C._stream(input))
    _lib.check(st, fn)
    return y, state, ckpt


def _recurrence_backward(input, u, v, decay, initial, offsets, scale, ckpt, grad, grad_state, want_initial):
    fn = "gated_linear_recurrence backward"
    s, state_shape = _check_recurrence(fn, input, u, v, decay, initial, offsets, scale)
    if grad is not None:
        _check_operand(fn, "grad_output", grad, input.shape, input.dtype, input)
    if grad_state is not None:
        _check_operand(fn, "grad_state", grad_state, state_shape, torch.float32, input)
    like = dict(dtype=input.dtype, device=input.device)
    wide = dict(dtype=torch.float32, device=input.device)
    dx, du, dv = (torch.empty(input.shape, **like) for _ in range(3))
    dinit = None
    if input.numel() == 0:
        if want_initial:
            dinit = _state_or_zeros(grad_state, state_shape, torch.float32, input.device)
        return dx, du, dv, torch.zeros(decay.shape, **wide), dinit
    _check_kept(fn, "checkpoints", ckpt, (int(_lib.lib.dwconv_b200_recurrence_checkpoint_bytes(s)) // 4,), input)
    dd = torch.empty(decay.shape, **wide)
    if want_initial:
        dinit = torch.empty(state_shape, **wide)
    x, u, v, d, init = _rows_of(input), _rows_of(u), _rows_of(v), decay.contiguous(), _contiguous(initial)
    g = _rows_of(grad) if grad is not None else torch.zeros(input.shape, **like)
    gs = _contiguous(grad_state)
    nbytes = int(_lib.lib.dwconv_b200_recurrence_workspace_bytes(s))
    ws = torch.empty(nbytes, dtype=torch.uint8, device=input.device)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_recurrence_backward(
            _rows_arg(x), _rows_arg(u), _rows_arg(v), d.data_ptr(), _ptr(init), ckpt.data_ptr(), _rows_arg(g),
            _ptr(gs), dx.data_ptr(), du.data_ptr(), dv.data_ptr(), dd.data_ptr(), _ptr(dinit), ws.data_ptr(),
            nbytes, _DTYPES[x.dtype], s, scale, _C._stream(input))
    _lib.check(st, fn)
    return dx, du, dv, dd, dinit


def _recurrence_step(input, u, v, decay, state, scale):
    fn = "gated_linear_recurrence_step"
    _check_step_input(fn, input)
    B, C = input.shape
    _check_operand(fn, "recurrence_gate", u, input.shape, input.dtype, input)
    _check_operand(fn, "input_gate", v, input.shape, input.dtype, input)
    _check_operand(fn, "decay", decay, (C,), torch.float32, input)
    _check_state(fn, state, (B, C), torch.float32, input)
    if not scale > 0:
        raise RuntimeError(f"dwconv_b200.{fn}: scale must be positive")
    y = torch.empty((B, C), dtype=input.dtype, device=input.device)
    if input.numel() == 0:
        return y
    _note_written(state)
    x, u, v, d = _rows_of(input), _rows_of(u), _rows_of(v), decay.contiguous()
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_recurrence_step(
            x.data_ptr(), x.stride(0), u.data_ptr(), u.stride(0), v.data_ptr(), v.stride(0), d.data_ptr(),
            state.data_ptr(), y.data_ptr(), _DTYPES[x.dtype], B, C, scale, _C._stream(input))
    _lib.check(st, fn)
    return y


def _norm_rows(t):
    """A tensor of any rank as rows over its last dimension, as they lie where one stride steps
    through them, else as a contiguous copy."""
    C = t.shape[-1]
    a = _rows_of(t)
    stride, span = None, 1
    for n, st in zip(reversed(a.shape[:-1]), reversed(a.stride()[:-1])):
        if n == 1:
            continue
        if stride is None:
            stride = st
        elif st != stride * span:
            return a.contiguous().view(-1, C)
        span *= n
    return a.as_strided((span, C), (C if stride is None else stride, 1), a.storage_offset())


def _check_norm(fn, input, weight, bias, eps):
    _C._check_cuda(input, "input")
    _sequence_dtype(input)
    if input.dim() < 1 or not 1 <= input.shape[-1] <= 1 << 26:
        raise RuntimeError(f"dwconv_b200.{fn}: expected input [..., C], got {tuple(input.shape)}")
    C = input.shape[-1]
    for name, t in (("weight", weight), ("bias", bias)):
        if t is not None:
            _check_operand(fn, name, t, (C,), input.dtype, input)
    if not eps >= 0:
        raise RuntimeError(f"dwconv_b200.{fn}: eps must not be negative")
    return C


def _layer_norm(input, weight, bias, eps, want_backward):
    fn = "layer_norm"
    C = _check_norm(fn, input, weight, bias, eps)
    rows = input.numel() // C
    y = torch.empty(input.shape, dtype=input.dtype, device=input.device)
    stats = torch.empty((rows, 2), dtype=torch.float32, device=input.device) if want_backward else None
    if rows == 0:
        return y, stats
    x, w, b = _norm_rows(input), _contiguous(weight), _contiguous(bias)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_layer_norm(x.data_ptr(), x.stride(0), _ptr(w), _ptr(b), y.data_ptr(),
                                             _ptr(stats), _DTYPES[x.dtype], rows, C, eps, _C._stream(input))
    _lib.check(st, fn)
    return y, stats


def _layer_norm_backward(input, weight, stats, grad, want_weight, want_bias):
    fn = "layer_norm backward"
    C = _check_norm(fn, input, weight, None, 0.)
    rows = input.numel() // C
    _check_operand(fn, "grad_output", grad, input.shape, input.dtype, input)
    like = dict(dtype=input.dtype, device=input.device)
    dx = torch.empty(input.shape, **like)
    if rows == 0:
        return (dx, torch.zeros(C, **like) if want_weight else None,
                torch.zeros(C, **like) if want_bias else None)
    _check_kept(fn, "stats", stats, (rows, 2), input)
    dw = torch.empty(C, **like) if want_weight else None
    db = torch.empty(C, **like) if want_bias else None
    x, g, w = _norm_rows(input), _norm_rows(grad), _contiguous(weight)
    code, ws, nbytes = _DTYPES[x.dtype], None, 0
    if want_weight or want_bias:
        nbytes = int(_lib.lib.dwconv_b200_layer_norm_workspace_bytes(code, rows, C))
        ws = torch.empty(nbytes, dtype=torch.uint8, device=input.device)
    with _C._on_device(input):
        st = _lib.lib.dwconv_b200_layer_norm_backward(
            x.data_ptr(), x.stride(0), _ptr(w), stats.data_ptr(), g.data_ptr(), g.stride(0), dx.data_ptr(),
            _ptr(dw), _ptr(db), _ptr(ws), nbytes, code, rows, C, _C._stream(input))
    _lib.check(st, fn)
    return dx, dw, db


CTYPES_FORMS = {
    "conv1d_causal": _conv1d_causal, "conv1d_causal_backward": _conv1d_causal_backward,
    "conv1d_causal_step": _conv1d_causal_step, "recurrence": _recurrence,
    "recurrence_backward": _recurrence_backward, "recurrence_step": _recurrence_step,
    "layer_norm": _layer_norm, "layer_norm_backward": _layer_norm_backward,
}


class _Forms:
    """The compiled functions, or the ones above where the module has not been built."""

    def __init__(self, native):
        for name, fn in CTYPES_FORMS.items():
            setattr(self, name, getattr(native, name) if native is not None else fn)


_forms = _Forms(_native)


# ---- autograd ----------------------------------------------------------------------------------
# The compiled module has nodes of its own (no interpreter in the backward pass); these functions are
# what runs without it, and where the device flags are checked after every call (that is not captured).

_nodes = _native if not _lib.CHECK_STATUS else None


def _check_flags(what):
    if _lib.CHECK_STATUS and not torch.cuda.is_current_stream_capturing():
        _lib.check_device_status(what)


def _wants_grad(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _refuse_tangents(fn, *tensors):
    # there are no forward-mode derivatives: a tangent that an operand carries would be lost
    if any(t is not None and torch.autograd.forward_ad.unpack_dual(t, level=0).tangent is not None for t in tensors):
        raise RuntimeError(f"dwconv_b200.{fn}: forward-mode differentiation is not supported")


def _activation(activation):
    if activation not in _ACTIVATIONS:
        raise ValueError(f"unknown activation {activation!r}; expected one of "
                         f"{sorted(k for k in _ACTIVATIONS if k)}")
    return _ACTIVATIONS[activation]


def _first_order(backward):
    """A backward pass whose results cannot be differentiated: with ``create_graph`` they carry an error.
    (``once_differentiable`` lets them pass as constants where the incoming gradients are constants, although
    they depend on the inputs.)"""
    @functools.wraps(backward)
    def wrapped(ctx, *grads):
        with torch.no_grad():
            out = backward(ctx, *grads)
        if not torch.is_grad_enabled() or all(t is None for t in out):
            return out
        error = torch._C._functions.DelayedError(
            "trying to differentiate twice a function that was marked with @once_differentiable", len(out))
        return error(*[t if t is None else t.detach().requires_grad_() for t in out])
    return wrapped


class CausalConv1dFunction(Function):
    @staticmethod
    def forward(ctx, input, weight, bias, initial, offsets, act, want_state):
        y, state = _forms.conv1d_causal(input, weight, bias, act, initial, offsets, want_state)
        _check_flags("depthwise_conv1d_causal")
        ctx.save_for_backward(input, weight, bias, initial, offsets)
        ctx.act, ctx.want_state = act, want_state
        ctx.set_materialize_grads(False)
        return (y, state) if want_state else y

    @staticmethod
    @_first_order
    def backward(ctx, grad, grad_state=None):
        input, weight, bias, initial, offsets = ctx.saved_tensors
        if grad is None and grad_state is None:
            return (None,) * 7
        dx, dw, db, dinit = _forms.conv1d_causal_backward(
            input, weight, bias, ctx.act, initial, offsets, grad, grad_state, ctx.needs_input_grad[3])
        _check_flags("depthwise_conv1d_causal backward")
        return dx, dw, db, dinit, None, None, None


class GatedLinearRecurrenceFunction(Function):
    @staticmethod
    def forward(ctx, input, recurrence_gate, input_gate, decay, initial, offsets, scale, want_state):
        y, state, ckpt = _forms.recurrence(input, recurrence_gate, input_gate, decay, initial, offsets,
                                           scale, want_state, True)
        _check_flags("gated_linear_recurrence")
        ctx.save_for_backward(input, recurrence_gate, input_gate, decay, initial, offsets, ckpt)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return (y, state) if want_state else y

    @staticmethod
    @_first_order
    def backward(ctx, grad, grad_state=None):
        input, u, v, decay, initial, offsets, ckpt = ctx.saved_tensors
        if grad is None and grad_state is None:
            return (None,) * 8
        dx, du, dv, dd, dinit = _forms.recurrence_backward(
            input, u, v, decay, initial, offsets, ctx.scale, ckpt, grad, grad_state,
            ctx.needs_input_grad[4])
        _check_flags("gated_linear_recurrence backward")
        return dx, du, dv, dd, dinit, None, None, None


class LayerNormFunction(Function):
    @staticmethod
    def forward(ctx, input, weight, bias, eps):
        y, stats = _forms.layer_norm(input, weight, bias, eps, True)
        _check_flags("layer_norm")
        ctx.save_for_backward(input, weight, stats)
        return y

    @staticmethod
    @_first_order
    def backward(ctx, grad):
        input, weight, stats = ctx.saved_tensors
        dx, dw, db = _forms.layer_norm_backward(input, weight, stats, grad, ctx.needs_input_grad[1],
                                                ctx.needs_input_grad[2])
        _check_flags("layer_norm backward")
        return dx, dw, db, None


# ---- public functions --------------------------------------------------------------------------

def depthwise_conv1d_causal(input, weight, bias=None, activation=None, initial_state=None, offsets=None,
                            return_state=False):
    """Causal depthwise convolution of a sequence [B, T, C], with bias and activation:
    ``act(bias[c] + sum_k weight[c, 0, k] * input[b, t - (taps - 1) + k, c])``.

    ``weight``: [C, 1, taps] (the layout of ``nn.Conv1d(groups=C)``), 1 to 8 taps; ``bias``: [C] or
    ``None``; both of the input's dtype.  ``activation`` as in ``depthwise_conv2d_epilogue``; every one
    of them has its gradient here.  ``initial_state``: [B, taps - 1, C] (packed: [S, taps - 1, C]), the
    rows in front of each sequence, oldest first; ``None`` stands for zeros.  ``offsets``: packed
    sequences (see the module's text).  With ``return_state`` the result is ``(output, state)``, the
    state being what the sequence's next piece takes as ``initial_state``.

    Gradients flow to input, weight, bias and initial state, and from output and returned state.
    """
    act = _activation(activation)
    if _nodes is not None:
        return _nodes.conv1d_causal_autograd(input, weight, bias, act, initial_state, offsets, bool(return_state))
    _refuse_tangents("depthwise_conv1d_causal", input, weight, bias, initial_state)
    if _wants_grad(input, weight, bias, initial_state):
        return CausalConv1dFunction.apply(input, weight, bias, initial_state, offsets, act, bool(return_state))
    y, state = _forms.conv1d_causal(input, weight, bias, act, initial_state, offsets, bool(return_state))
    _check_flags("depthwise_conv1d_causal")
    return (y, state) if return_state else y


def depthwise_conv1d_causal_step(input, weight, state, bias=None, activation=None):
    """One row of each of B sequences: input [B, C], ``state`` [B, taps - 1, C] of the input's dtype,
    contiguous, updated in place.  The values of ``depthwise_conv1d_causal`` with T = 1.
    Inference only."""
    act = _activation(activation)
    if _nodes is not None:
        return _nodes.conv1d_causal_step_checked(input, weight, state, bias, act)
    _refuse_tangents("depthwise_conv1d_causal_step", input, weight, state, bias)
    if _wants_grad(input, weight, state, bias):
        raise RuntimeError("dwconv_b200.depthwise_conv1d_causal_step: the state is updated in place and "
                           "has no gradient; use depthwise_conv1d_causal or torch.no_grad()")
    y = _forms.conv1d_causal_step(input, weight, state, bias, act)
    _check_flags("depthwise_conv1d_causal_step")
    return y


def gated_linear_recurrence(input, recurrence_gate, input_gate, decay, initial_state=None, offsets=None,
                            return_state=False, scale=8.0):
    """Gated linear recurrence over a sequence [B, T, C], channel by channel::

        a[t] = exp(-scale * softplus(decay) * sigmoid(recurrence_gate[t]))
        h[t] = a[t] * h[t - 1] + sqrt(1 - a[t] ** 2) * sigmoid(input_gate[t]) * input[t]

    Returns h, in the input's dtype.  The gates are given before their sigmoid, shaped and typed like
    the input; any row strides are read in place (slices of one projection need no copy).  ``decay``:
    fp32 [C]; ``scale`` > 0.  ``initial_state``: fp32 [B, C] (packed: [S, C]), the state each sequence
    starts from; ``None`` stands for zeros.  With ``return_state`` the result is ``(h, state)``, the
    state (fp32, not rounded) being what the sequence's next piece starts from.

    Gradients flow to input, both gates, decay and initial state, and from h and returned state.
    """
    scale = float(scale)
    if _nodes is not None:
        return _nodes.recurrence_autograd(input, recurrence_gate, input_gate, decay, initial_state, offsets, scale,
                                          bool(return_state))
    _refuse_tangents("gated_linear_recurrence", input, recurrence_gate, input_gate, decay, initial_state)
    if _wants_grad(input, recurrence_gate, input_gate, decay, initial_state):
        return GatedLinearRecurrenceFunction.apply(input, recurrence_gate, input_gate, decay, initial_state,
                                                   offsets, scale, bool(return_state))
    y, state, _ = _forms.recurrence(input, recurrence_gate, input_gate, decay, initial_state, offsets, scale,
                                    bool(return_state), False)
    _check_flags("gated_linear_recurrence")
    return (y, state) if return_state else y


def gated_linear_recurrence_step(input, recurrence_gate, input_gate, decay, state, scale=8.0):
    """One row of each of B sequences: input and gates [B, C], ``state`` fp32 [B, C], contiguous,
    updated in place.  Inference only."""
    if _nodes is not None:
        return _nodes.recurrence_step_checked(input, recurrence_gate, input_gate, decay, state, float(scale))
    _refuse_tangents("gated_linear_recurrence_step", input, recurrence_gate, input_gate, decay, state)
    if _wants_grad(input, recurrence_gate, input_gate, decay, state):
        raise RuntimeError("dwconv_b200.gated_linear_recurrence_step: the state is updated in place and "
                           "has no gradient; use gated_linear_recurrence or torch.no_grad()")
    y = _forms.recurrence_step(input, recurrence_gate, input_gate, decay, state, float(scale))
    _check_flags("gated_linear_recurrence_step")
    return y


def layer_norm(input, weight=None, bias=None, eps=1e-5):
    """``(input - mean) / sqrt(var + eps) * weight + bias`` over the last dimension, of any rank.

    ``weight`` and ``bias``: [C] of the input's dtype, or ``None``.  Rows that lie at one stride are
    read in place: the map that a channels-last ``depthwise_conv2d`` leaves is normalised over its
    channels as ``layer_norm(y.permute(0, 2, 3, 1), ...)`` without a copy.
    """
    eps = float(eps)
    if _nodes is not None:
        return _nodes.layer_norm_autograd(input, weight, bias, eps)
    _refuse_tangents("layer_norm", input, weight, bias)
    if _wants_grad(input, weight, bias):
        return LayerNormFunction.apply(input, weight, bias, eps)
    y = _forms.layer_norm(input, weight, bias, eps, False)[0]
    _check_flags("layer_norm")
    return y


# ---- modules -----------------------------------------------------------------------------------
# The functions take filter, bias and norm weights in the input's type.  Under torch.autocast, where activations
# come in 16 bits and parameters stay in fp32, the modules convert, each as torch converts for the layer whose
# state_dict it shares: the convolution runs in the activations' type, the norm in the parameters'.

def _mixed(input, parameter):
    return input.dtype != parameter.dtype and torch.is_autocast_enabled("cuda")


class CausalDepthwiseConv1d(nn.Module):
    """Module form of ``depthwise_conv1d_causal``; ``state_dict`` interchangeable with
    ``nn.Conv1d(channels, channels, kernel_size, groups=channels)``."""

    def __init__(self, channels, kernel_size, bias=True, activation=None):
        super().__init__()
        if not 1 <= kernel_size <= _lib.MAX_TAPS:
            raise ValueError(f"CausalDepthwiseConv1d supports 1 to {_lib.MAX_TAPS} taps")
        _activation(activation)
        self.channels, self.kernel_size, self.activation = channels, kernel_size, activation
        self.weight = nn.Parameter(torch.randn(channels, 1, kernel_size) / kernel_size ** 0.5)
        self.bias = nn.Parameter(torch.zeros(channels)) if bias else None

    def _filter(self, input):
        w, b = self.weight, self.bias
        if _mixed(input, w):    # rounded to the activations' type, and so are their gradients
            w, b = w.to(input.dtype), b.to(input.dtype) if b is not None else None
        return w, b

    def forward(self, input, initial_state=None, offsets=None, return_state=False):
        w, b = self._filter(input)
        return depthwise_conv1d_causal(input, w, b, self.activation, initial_state, offsets, return_state)

    def step(self, input, state):
        w, b = self._filter(input)
        return depthwise_conv1d_causal_step(input, w, state, b, self.activation)


class GatedLinearRecurrence(nn.Module):
    """Module form of ``gated_linear_recurrence``: holds ``decay``, drawn so that a fully open gate
    decays by a factor between ``low`` and ``high`` per row.  The parameter stays fp32, unrounded, when
    the module or a model around it is converted (``.half()``, ``.bfloat16()``, ``.to(dtype)``)."""

    def __init__(self, channels, scale=8.0, low=0.9, high=0.999):
        super().__init__()
        if not 0 < low <= high < 1:
            raise ValueError("expected 0 < low <= high < 1")
        self.channels, self.scale = channels, float(scale)
        a = low + (high - low) * torch.rand(channels, dtype=torch.float64)
        self.decay = nn.Parameter(torch.log(torch.expm1(-torch.log(a) / scale)).float())

    def _apply(self, fn, recurse=True):
        kept, grad = self.decay.data, self.decay.grad
        grad = None if grad is None else grad.data
        out = super()._apply(fn, recurse)
        if self.decay.dtype != torch.float32:
            self.decay.data = kept.to(self.decay.device)
            self.decay.grad = None if grad is None else grad.to(self.decay.device)
        return out

    def forward(self, input, recurrence_gate, input_gate, initial_state=None, offsets=None, return_state=False):
        return gated_linear_recurrence(input, recurrence_gate, input_gate, self.decay, initial_state, offsets,
                                       return_state, self.scale)

    def step(self, input, recurrence_gate, input_gate, state):
        return gated_linear_recurrence_step(input, recurrence_gate, input_gate, self.decay, state, self.scale)


class LayerNorm(nn.Module):
    """Module form of ``layer_norm``; ``state_dict`` interchangeable with ``nn.LayerNorm(channels)``."""

    def __init__(self, channels, eps=1e-5, bias=True):
        super().__init__()
        self.channels, self.eps = channels, eps
        self.weight = nn.Parameter(torch.ones(channels))
        self.bias = nn.Parameter(torch.zeros(channels)) if bias else None

    def forward(self, input):
        if _mixed(input, self.weight):
            input = input.to(self.weight.dtype)
        return layer_norm(input, self.weight, self.bias, self.eps)


class RecurrentMixer(nn.Module):
    """The token-mixing half of a recurrent block, built from the operators above::

        n = norm(x);  gate, z = split(project_in(n));  z = conv(z);  u, v = split(project_gates(z))
        x + project_out(recurrence(z, u, v) * gelu(gate))

    ``forward`` runs whole sequences ([B, T, C], or packed) from an optional state and returns the
    state that ``step`` carries on from, one row at a time: ``(conv state, recurrence state)``.
    """

    def __init__(self, channels, width=None, taps=4, scale=8.0):
        super().__init__()
        width = channels if width is None else width
        self.channels, self.width, self.taps = channels, width, taps
        self.norm = LayerNorm(channels)
        self.project_in = nn.Linear(channels, 2 * width)
        self.conv = CausalDepthwiseConv1d(width, taps)
        self.project_gates = nn.Linear(width, 2 * width)
        self.recurrence = GatedLinearRecurrence(width, scale)
        self.project_out = nn.Linear(width, channels)

    def initial_state(self, count, dtype=None, device=None):
        """Zeros for ``count`` sequences; ``dtype``: of the convolution's rows, the type that ``project_in`` gives
        (under autocast that of autocast)."""
        w = self.conv.weight
        if dtype is None:
            dtype = torch.get_autocast_dtype("cuda") if torch.is_autocast_enabled("cuda") else w.dtype
        device = device or w.device
        return (torch.zeros(count, self.taps - 1, self.width, dtype=dtype, device=device),
                torch.zeros(count, self.width, dtype=torch.float32, device=device))

    def forward(self, x, state=None, offsets=None):
        conv_state, rec_state = state if state is not None else (None, None)
        gate, z = self.project_in(self.norm(x)).chunk(2, dim=-1)
        z, conv_state = self.conv(z, conv_state, offsets, return_state=True)
        u, v = self.project_gates(z).chunk(2, dim=-1)
        h, rec_state = self.recurrence(z, u, v, rec_state, offsets, return_state=True)
        return x + self.project_out(h * nn.functional.gelu(gate)), (conv_state, rec_state)

    @torch.no_grad()
    def step(self, x, state):
        """x [B, C]; ``state`` as from ``forward`` or ``initial_state``, updated in place."""
        gate, z = self.project_in(self.norm(x)).chunk(2, dim=-1)
        z = self.conv.step(z, state[0])
        u, v = self.project_gates(z).chunk(2, dim=-1)
        h = self.recurrence.step(z, u, v, state[1])
        return x + self.project_out(h * nn.functional.gelu(gate))

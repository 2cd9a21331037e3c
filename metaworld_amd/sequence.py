"""The operators of a policy with memory, on the device: layer norm, the short causal convolution and the selective state space scan.

For a learner whose policy lives on the same GPU as its environments (torch_env.MetaWorldTorchVectorEnv): one token of every
environment at a time while it acts (`*_step`, the state updated in place), whole segments of a rollout while it trains, with the
environments' episode ends as `reset` flags.  recurrent_policy.RecurrentPolicy is made of them.

Every function takes CUDA tensors of one device (float32, bfloat16 or float16 activations), works on the current stream of that
device, does not wait for the host and keeps nothing between calls; outputs and scratch memory come from torch's allocator, so that
calls may be captured into graphs.  Sums, statistics and scan states are float32 whatever the activations' type.  The last dimension
should be contiguous (it is copied otherwise), all other strides are free.  The kernels are in libmwseq.so (csrc_seq/, C ABI:
include/mwseq.h); without it, or on CPU tensors, the functions raise: there is no fallback.

Tokens are [batch, time].  `reset` (bool or uint8, [batch, time]) is true at an episode's first token, from which on neither the
state nor earlier tokens are seen.  `lengths` (int32 [batch]) says how many tokens of a padded row count, taken into 0 .. time: the
others' inputs are not looked at, their outputs and gradients are zero, and the returned state is that after the last token that
counts.  Gradients are deterministic (no atomic additions) and once differentiable.
"""
from __future__ import annotations

import ctypes as C
import os
import struct

import torch
from torch.autograd.function import once_differentiable

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmwseq.so")
MAX_WIDTH, MAX_TAPS, MAX_STATES = 16384, 4, 32           # MWS_NORM_MAX_WIDTH, MWS_CONV_MAX_TAPS (at least 2), MWS_SCAN_MAX_STATES
EXPORTED_SYMBOLS = ["mws_" + s for s in ("last_error", "sizeof", "norm_forward", "norm_workspace", "norm_backward", "conv_forward", "conv_workspace", "conv_backward", "conv_step",
                                         "scan_kept", "scan_workspace", "scan_forward", "scan_backward", "scan_step")]

_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
# the argument structs of include/mwseq.h, field by field
_NORM = struct.Struct("@9Q4q3if")
_CONV = struct.Struct("@15Q9q4i")
_SCAN = struct.Struct("@26Q17q4i")

_lib = None


def load():
    """libmwseq.so with its argument and result types (opened once)"""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} not found: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
                               "(hipcc --offload-arch=gfx950); there is no CPU fallback")
        lib = C.CDLL(LIB_PATH)
        for name in EXPORTED_SYMBOLS:
            f = getattr(lib, name)
            f.restype, f.argtypes = C.c_int32, [C.c_char_p, C.c_void_p]
        lib.mws_last_error.restype, lib.mws_last_error.argtypes = C.c_char_p, []
        lib.mws_sizeof.restype, lib.mws_sizeof.argtypes = C.c_int64, [C.c_int32]
        for name in ("norm_workspace", "conv_workspace", "scan_kept"):
            f = getattr(lib, "mws_" + name)
            f.restype, f.argtypes = C.c_int64, [C.c_char_p]
        lib.mws_scan_workspace.restype, lib.mws_scan_workspace.argtypes = C.c_int64, [C.c_char_p, C.c_int32]
        for k, s in enumerate((_NORM, _CONV, _SCAN)):
            if lib.mws_sizeof(k) != s.size:
                raise RuntimeError(f"{LIB_PATH} does not match include/mwseq.h: build it again")
        _lib = lib
    return _lib


def _check(code):
    if code < 0:
        raise RuntimeError("mwseq: " + load().mws_last_error().decode())
    return code


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _launch(fn, args, device):
    """one call of the library on the current stream of `device`"""
    if torch.cuda.current_device() == device.index:
        _check(fn(args, torch.cuda.current_stream().cuda_stream))
    else:
        with torch.cuda.device(device):
            _check(fn(args, torch.cuda.current_stream().cuda_stream))


def _tensor(what, t, shape=None, dtype=None, device=None, optional=False):
    if t is None and optional:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{what} has to be a tensor, not {type(t).__name__}")
    if shape is not None and tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} has shape {tuple(t.shape)}, {tuple(shape)} is wanted")
    if dtype is not None and t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise TypeError(f"{what} is {t.dtype}, {dtype} is wanted")
    if device is not None and t.device != device:
        raise ValueError(f"{what} is on {t.device}, {device} is wanted")


def _activations(what, t, dims=None):
    _tensor(what, t)
    if t.dtype not in _TYPES:
        raise TypeError(f"{what} is {t.dtype}: float32, bfloat16 and float16 are supported")
    if dims is not None and t.dim() != dims:
        raise ValueError(f"{what} has {t.dim()} dimensions, {dims} are wanted")
    if t.dim() and t.shape[-1] < 1:
        raise ValueError(f"{what} has no channels")


def _on_gpu(what, t):
    if t.device.type != "cuda":
        raise ValueError(f"{what} is on {t.device}: the kernels run on a GPU and there is no CPU fallback")


def _rows(t):
    """`t` with its last dimension contiguous"""
    return t if t is None or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _records(*tensors):
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


def _acting(what, *tensors):
    if _records(*tensors):
        raise RuntimeError(f"{what} has no gradient and updates the state in place: call it under torch.no_grad()")


def _updated(state):
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)


# ---- layer norm ----
def _norm_args(x, weight, bias, eps, dy=None, y=None, dx=None, dweight=None, dbias=None, workspace=None, space=0):
    p = weight if weight is not None else bias
    return _NORM.pack(_ptr(x), _ptr(weight), _ptr(bias), _ptr(dy), _ptr(y), _ptr(dx), _ptr(dweight), _ptr(dbias), _ptr(workspace), x.shape[0], x.stride(0),
                      dy.stride(0) if dy is not None else 0, space, x.shape[1], _TYPES[x.dtype], _TYPES[p.dtype] if p is not None else 0, eps)


def _norm_forward(x, weight, bias, eps):
    flat = _rows(x.reshape(-1, x.shape[-1]))
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    _launch(load().mws_norm_forward, _norm_args(flat, weight, bias, eps, y=y), x.device)
    return y


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        ctx.save_for_backward(x, weight, bias)
        ctx.eps = eps
        return _norm_forward(x, weight, bias, eps)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, bias = ctx.saved_tensors
        lib, need = load(), ctx.needs_input_grad
        flat, dflat = (_rows(t.reshape(-1, x.shape[-1])) for t in (x, dy))
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dweight = torch.empty_like(weight, memory_format=torch.contiguous_format) if need[1] else None
        dbias = torch.empty_like(bias, memory_format=torch.contiguous_format) if need[2] else None
        args = (flat, weight, bias, ctx.eps, dflat, None, dx, dweight, dbias)
        space = _check(lib.mws_norm_workspace(_norm_args(*args)))
        workspace = torch.empty(space, dtype=torch.uint8, device=x.device) if space else None
        _launch(lib.mws_norm_backward, _norm_args(*args, workspace, space), x.device)
        return dx, dweight, dbias, None


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (1 .. 16384 wide; var: the mean squared deviation).

    x [..., width]; weight and bias [width], each float32 or of x's type (both alike) or None.  Returns a tensor of x's type and shape."""
    _activations("x", x)
    if x.dim() < 1:
        raise ValueError("x has no dimension to normalise over")
    width = x.shape[-1]
    if width > MAX_WIDTH:
        raise ValueError(f"x is {width} wide: {MAX_WIDTH} is the most")
    for what, p in (("weight", weight), ("bias", bias)):
        _tensor(what, p, (width,), (torch.float32, x.dtype), x.device, optional=True)
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise TypeError(f"weight is {weight.dtype} and bias {bias.dtype}: one type is wanted")
    if not eps >= 0:
        raise ValueError(f"eps is {eps}: it must not be negative")
    _on_gpu("x", x)
    weight, bias = _rows(weight), _rows(bias)
    return _LayerNorm.apply(x, weight, bias, eps) if _records(x, weight, bias) else _norm_forward(x, weight, bias, eps)


# ---- what convolution and scan share ----
def _tokens(batch, time, device, reset, lengths):
    _tensor("reset", reset, (batch, time) if time is not None else (batch,), (torch.bool, torch.uint8), device, optional=True)
    _tensor("lengths", lengths, (batch,), torch.int32, device, optional=True)


def _two(t):
    return (t.stride(0), t.stride(1)) if t is not None else (0, 0)


def _first(t):
    return t.stride(0) if t is not None else 0


# ---- the short causal convolution ----
def _conv_args(x, weight, bias, state, reset, lengths, shape, strides, dy=None, dlast=None, y=None, last=None, dx=None, dweight=None, dbias=None, dstate=None, workspace=None, space=0):
    return _CONV.pack(_ptr(x), _ptr(weight), _ptr(bias), _ptr(state), _ptr(dy), _ptr(dlast), _ptr(reset), _ptr(lengths), _ptr(y), _ptr(last), _ptr(dx), _ptr(dweight), _ptr(dbias),
                      _ptr(dstate), _ptr(workspace), *shape, *strides, space, weight.shape[0], weight.shape[1], _TYPES[x.dtype], _TYPES[weight.dtype])


def _conv_forward(x, weight, bias, state, reset, lengths):
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    last = torch.empty((x.shape[0], weight.shape[1] - 1, x.shape[2]), dtype=x.dtype, device=x.device)
    args = _conv_args(x, weight, bias, state, reset, lengths, x.shape[:2], (*_two(x), 0, 0, *_two(reset)), y=y, last=last)
    _launch(load().mws_conv_forward, args, x.device)
    return y, last


class _CausalConv(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, state, reset, lengths):
        ctx.save_for_backward(x, weight, bias, state, reset, lengths)
        ctx.set_materialize_grads(False)
        return _conv_forward(x, weight, bias, state, reset, lengths)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        x, weight, bias, state, reset, lengths = ctx.saved_tensors
        lib, need = load(), ctx.needs_input_grad
        dy = _rows(dy) if dy is not None else torch.zeros_like(x, memory_format=torch.contiguous_format)
        dlast = dlast.contiguous() if dlast is not None else None
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if need[0] else None
        dweight = torch.empty(weight.shape, dtype=weight.dtype, device=x.device) if need[1] else None
        dbias = torch.empty(bias.shape, dtype=bias.dtype, device=x.device) if need[2] else None
        dstate = torch.empty(state.shape, dtype=state.dtype, device=x.device) if need[3] else None
        args = (x, weight, bias, state, reset, lengths, x.shape[:2], (*_two(x), *_two(dy), *_two(reset)), dy, dlast, None, None, dx, dweight, dbias, dstate)
        space = _check(lib.mws_conv_workspace(_conv_args(*args)))
        workspace = torch.empty(space, dtype=torch.uint8, device=x.device) if space else None
        _launch(lib.mws_conv_backward, _conv_args(*args, workspace, space), x.device)
        return dx, dweight, dbias, dstate, None, None


def _conv_check(x, weight, bias, state, dims):
    _activations("x", x, dims)
    _tensor("weight", weight, None, (torch.float32, x.dtype), x.device)
    width = x.shape[-1]
    if weight.dim() != 2 or weight.shape[0] != width or not 2 <= weight.shape[1] <= MAX_TAPS:
        raise ValueError(f"weight has shape {tuple(weight.shape)}, ({width}, 2 .. {MAX_TAPS} taps) is wanted")
    _tensor("bias", bias, (width,), weight.dtype, x.device, optional=True)
    _tensor("state", state, (x.shape[0], weight.shape[1] - 1, width), x.dtype, x.device, optional=dims == 3)


def causal_conv(x, weight, bias=None, *, state=None, reset=None, lengths=None):
    """silu(bias + sum_j weight[:, j] * x[t - taps + 1 + j]), channel by channel, over the tokens up to and including t.

    x [batch, time, width]; weight [width, taps] (2 .. 4 taps), bias [width] or None, both float32 or of x's type; `state`
    [batch, taps - 1, width] of x's type holds the inputs before the first token, oldest first (None: zeros).
    Returns (y, state after the last token)."""
    _conv_check(x, weight, bias, state, 3)
    _tokens(x.shape[0], x.shape[1], x.device, reset, lengths)
    _on_gpu("x", x)
    x, weight, bias = _rows(x), weight.contiguous(), _rows(bias)
    state = state.contiguous() if state is not None else None
    lengths = lengths.contiguous() if lengths is not None else None
    args = (x, weight, bias, state, reset, lengths)
    return _CausalConv.apply(*args) if _records(x, weight, bias, state) else _conv_forward(*args)


def causal_conv_step(x, weight, bias=None, *, state, reset=None):
    """One token of causal_conv: x [batch, width]; `state` [batch, taps - 1, width] (contiguous) is updated in place;
    reset [batch].  Returns y.  Without gradient."""
    _conv_check(x, weight, bias, state, 2)
    _tokens(x.shape[0], None, x.device, reset, None)
    if not state.is_contiguous():
        raise ValueError("state has to be contiguous: it is updated in place")
    _on_gpu("x", x)
    _acting("causal_conv_step", x, weight, bias, state)
    x, weight, bias = _rows(x), weight.contiguous(), _rows(bias)
    y = torch.empty(x.shape, dtype=x.dtype, device=x.device)
    args = _conv_args(x, weight, bias, state, reset, None, (x.shape[0], 1), (x.stride(0), 0, 0, 0, _first(reset), 0), y=y, last=state)
    _launch(load().mws_conv_step, args, x.device)
    _updated(state)
    return y


# ---- the selective state space scan ----
def _scan_args(u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths, shape, strides, dy=None, dlast=None, y=None, last=None, kept=None, du=None, ddt=None, dz=None, dB=None, dC=None,
               dA=None, dD=None, ddt_bias=None, dstate=None, workspace=None, space=0):
    return _SCAN.pack(_ptr(u), _ptr(dt), _ptr(z), _ptr(B), _ptr(C_), _ptr(dy), _ptr(A), _ptr(D), _ptr(dt_bias), _ptr(state), _ptr(dlast), _ptr(reset), _ptr(lengths), _ptr(y),
                      _ptr(last), _ptr(kept), _ptr(du), _ptr(ddt), _ptr(dz), _ptr(dB), _ptr(dC), _ptr(dA), _ptr(dD), _ptr(ddt_bias), _ptr(dstate), _ptr(workspace), *shape, *strides,
                      space, A.shape[0], A.shape[1], _TYPES[u.dtype], 0)


def _scan_forward(u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths, keep):
    lib = load()
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    last = torch.empty((u.shape[0], *A.shape), dtype=torch.float32, device=u.device)
    strides = (*_two(u), *_two(dt), *_two(z), *_two(B), *_two(C_), 0, 0, *_two(reset))
    args = (u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths, u.shape[:2], strides, None, None, y, last)
    plain = _scan_args(*args)
    kept = torch.empty(_check(lib.mws_scan_kept(plain)), dtype=torch.float32, device=u.device) if keep else None
    space = _check(lib.mws_scan_workspace(plain, 0))
    workspace = torch.empty(space, dtype=torch.uint8, device=u.device)
    _launch(lib.mws_scan_forward, _scan_args(*args, kept=kept, workspace=workspace, space=space), u.device)
    return y, last, kept


class _SelectiveScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths):
        y, last, kept = _scan_forward(u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths, True)
        ctx.save_for_backward(u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths)
        ctx.kept = kept
        ctx.set_materialize_grads(False)
        return y, last

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dlast):
        u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths = ctx.saved_tensors
        lib, device = load(), u.device
        dy = _rows(dy) if dy is not None else torch.zeros_like(u, memory_format=torch.contiguous_format)
        dlast = dlast.contiguous() if dlast is not None else None

        def like(t):
            return torch.empty(t.shape, dtype=t.dtype, device=device) if t is not None else None

        du, ddt, dz, dB, dC, dA, dD, ddt_bias, dstate = (like(t) for t in (u, dt, z, B, C_, A, D, dt_bias, state))
        strides = (*_two(u), *_two(dt), *_two(z), *_two(B), *_two(C_), *_two(dy), *_two(reset))
        args = (u, dt, A, B, C_, D, z, dt_bias, state, reset, lengths, u.shape[:2], strides, dy, dlast, None, None, ctx.kept, du, ddt, dz, dB, dC, dA, dD, ddt_bias, dstate)
        space = _check(lib.mws_scan_workspace(_scan_args(*args), 1))
        workspace = torch.empty(space, dtype=torch.uint8, device=device)
        _launch(lib.mws_scan_backward, _scan_args(*args, workspace, space), device)
        return du, ddt, dA, dB, dC, dD, dz, ddt_bias, dstate, None, None


def _scan_check(u, dt, A, B, C_, D, z, dt_bias, state, dims):
    _activations("u", u, dims)
    width, device = u.shape[-1], u.device
    _tensor("A", A, None, torch.float32, device)
    if A.dim() != 2 or A.shape[0] != width or not 1 <= A.shape[1] <= MAX_STATES:
        raise ValueError(f"A has shape {tuple(A.shape)}, ({width}, 1 .. {MAX_STATES} states) is wanted")
    _tensor("dt", dt, u.shape, u.dtype, device)
    _tensor("z", z, u.shape, u.dtype, device, optional=True)
    for what, t in (("B", B), ("C", C_)):
        _tensor(what, t, (*u.shape[:-1], A.shape[1]), u.dtype, device)
    for what, t in (("D", D), ("dt_bias", dt_bias)):
        _tensor(what, t, (width,), torch.float32, device, optional=True)
    _tensor("state", state, (u.shape[0], *A.shape), torch.float32, device, optional=dims == 3)


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, *, state=None, reset=None, lengths=None):
    """The selective state space scan over time, channel by channel with `states` states each:

        d_t = softplus(dt_t + dt_bias);  h_t = exp(d_t A) h_{t-1} + d_t u_t B_t;  y_t = (C_t . h_t + D u_t) silu(z_t)

    u, dt and z [batch, time, width] (z None: no gate) and B and C [batch, time, states] of one type; A [width, states] (1 .. 32
    states), D and dt_bias [width] (None: zeros) float32; `state` [batch, width, states] float32 is h before the first token (None:
    zeros).  Returns (y, h after the last token)."""
    _scan_check(u, dt, A, B, C, D, z, dt_bias, state, 3)
    _tokens(u.shape[0], u.shape[1], u.device, reset, lengths)
    _on_gpu("u", u)
    u, dt, B, C, D, z, dt_bias = (_rows(t) for t in (u, dt, B, C, D, z, dt_bias))
    A = A.contiguous()
    state = state.contiguous() if state is not None else None
    lengths = lengths.contiguous() if lengths is not None else None
    args = (u, dt, A, B, C, D, z, dt_bias, state, reset, lengths)
    return _SelectiveScan.apply(*args) if _records(u, dt, A, B, C, D, z, dt_bias, state) else _scan_forward(*args, False)[:2]


def selective_scan_step(u, dt, A, B, C, D=None, z=None, dt_bias=None, *, state, reset=None):
    """One token of selective_scan: u, dt and z [batch, width], B and C [batch, states]; `state` [batch, width, states] (float32,
    contiguous) is updated in place; reset [batch].  Returns y.  Without gradient."""
    _scan_check(u, dt, A, B, C, D, z, dt_bias, state, 2)
    _tokens(u.shape[0], None, u.device, reset, None)
    if not state.is_contiguous():
        raise ValueError("state has to be contiguous: it is updated in place")
    _on_gpu("u", u)
    _acting("selective_scan_step", u, dt, A, B, C, D, z, dt_bias, state)
    u, dt, B, C, D, z, dt_bias = (_rows(t) for t in (u, dt, B, C, D, z, dt_bias))
    A = A.contiguous()
    y = torch.empty(u.shape, dtype=u.dtype, device=u.device)
    strides = (u.stride(0), 0, dt.stride(0), 0, _first(z), 0, B.stride(0), 0, C.stride(0), 0, 0, 0, _first(reset), 0)
    args = _scan_args(u, dt, A, B, C, D, z, dt_bias, state, reset, None, (u.shape[0], 1), strides, y=y, last=state)
    _launch(load().mws_scan_step, args, u.device)
    _updated(state)
    return y

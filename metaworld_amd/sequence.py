"""The operators of a policy with memory, on the device: layer norm, the short causal convolution and the selective state space scan.

For a learner whose policy lives on the same GPU as its environments (torch_env.MetaWorldTorchVectorEnv): one token of every
environment at a time while it acts (`*_step`, the state updated in place), whole segments of a rollout while it trains, with the
environments' episode ends as `reset` flags.  recurrent_policy.RecurrentPolicy is made of them.

Every function takes CUDA tensors of one device (float32, bfloat16 or float16 activations), works on the current stream of that
device, does not wait for the host and keeps nothing between calls; outputs and scratch memory come from torch's allocator, so that
calls may be captured into graphs.  Sums, statistics and scan states are float32 whatever the activations' type.  The last dimension
should be contiguous (it is copied otherwise), all other strides are free.  The kernels are in libmwseq.so (csrc_seq/, C ABI:
include/mwseq.h), their torch side in _sequence.so; without them, or on CPU tensors, the functions raise: there is no fallback.

Tokens are [batch, time].  `reset` (bool or uint8, [batch, time]) is true at an episode's first token, from which on neither the
state nor earlier tokens are seen.  `lengths` (int32 [batch]) says how many tokens of a padded row count, taken into 0 .. time: the
others' inputs are not looked at, their outputs and gradients are zero, and the returned state is that after the last token that
counts.  Gradients are deterministic (no atomic additions) and not differentiable again (create_graph is refused, as are forward
derivatives).  A call gives the same values to the last bit whether it is recorded for them or not.

Infinities and NaN in inputs that count give what the formulas give token by token; no padding of a width, of a number of states or of a
row adds a NaN to an output.  Of the gradients that holds for those that are numbers by the formulas; another may be NaN where the
formula has an infinity.  Rates A above zero let states grow: they pass the range of a number where they do token by token.

Calls are no operations that torch knows: they run inside torch.compile's programs between its graphs, and raise where torch records
its operations (torch.jit.trace, torch.fx), which would hold their outputs' memory and not the kernels that fill it.
"""
from __future__ import annotations

import ctypes as C
import os

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libmwseq.so")
MAX_WIDTH, MAX_TAPS, MAX_STATES = 16384, 4, 32           # MWS_NORM_MAX_WIDTH, MWS_CONV_MAX_TAPS (at least 2), MWS_SCAN_MAX_STATES
EXPORTED_SYMBOLS = ["mws_" + s for s in ("last_error", "sizeof", "norm_forward", "norm_workspace", "norm_backward", "conv_forward", "conv_workspace", "conv_backward", "conv_step",
                                         "scan_kept", "scan_workspace", "scan_forward", "scan_backward", "scan_step")]
_HOW = "build it with `python -c 'import __graft_entry__ as g; g.build()'` (hipcc --offload-arch=gfx950); there is no CPU fallback"

_binding = None


def library():
    """ctypes handle on libmwseq.so, the C ABI of include/mwseq.h"""
    if not os.path.exists(LIB_PATH):
        raise RuntimeError(f"{LIB_PATH} not found: {_HOW}")
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
    return lib


def binding():
    """the torch side of the library (_sequence.so), loaded at the first call"""
    global _binding
    if _binding is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(f"{LIB_PATH} not found: {_HOW}")
        try:
            from . import _sequence
        except ImportError as e:
            raise RuntimeError(f"{os.path.join(_HERE, '_sequence.so')} cannot be loaded ({e}): {_HOW}") from e
        _binding = _sequence
    return _binding


def layer_norm(x, weight=None, bias=None, eps=1e-5):
    """(x - mean) / sqrt(var + eps) * weight + bias over the last dimension (1 .. 16384 wide; var: the mean squared deviation).

    x [..., width]; weight and bias [width], each float32 or of x's type (both alike) or None.  Returns a tensor of x's type and shape."""
    return (_binding or binding()).layer_norm(x, weight, bias, eps)


def causal_conv(x, weight, bias=None, *, state=None, reset=None, lengths=None):
    """silu(bias + sum_j weight[:, j] * x[t - taps + 1 + j]), channel by channel, over the tokens up to and including t.

    x [batch, time, width]; weight [width, taps] (2 .. 4 taps), bias [width] or None, both float32 or of x's type; `state`
    [batch, taps - 1, width] of x's type holds the inputs before the first token, oldest first (None: zeros).
    Returns (y, state after the last token)."""
    return (_binding or binding()).causal_conv(x, weight, bias, state, reset, lengths)


def causal_conv_step(x, weight, bias=None, *, state, reset=None):
    """One token of causal_conv: x [batch, width]; `state` [batch, taps - 1, width] (contiguous) is updated in place;
    reset [batch].  Returns y.  Without gradient."""
    return (_binding or binding()).causal_conv_step(x, weight, bias, state, reset)


def selective_scan(u, dt, A, B, C, D=None, z=None, dt_bias=None, *, state=None, reset=None, lengths=None):
    """The selective state space scan over time, channel by channel with `states` states each:

        d_t = softplus(dt_t + dt_bias);  h_t = exp(d_t A) h_{t-1} + d_t u_t B_t;  y_t = (C_t . h_t + D u_t) silu(z_t)

    u, dt and z [batch, time, width] (z None: no gate) and B and C [batch, time, states] of one type; A [width, states] (1 .. 32
    states), D and dt_bias [width] (None: zeros) float32; `state` [batch, width, states] float32 is h before the first token (None:
    zeros).  Returns (y, h after the last token)."""
    return (_binding or binding()).selective_scan(u, dt, A, B, C, D, z, dt_bias, state, reset, lengths)


def selective_scan_step(u, dt, A, B, C, D=None, z=None, dt_bias=None, *, state, reset=None):
    """One token of selective_scan: u, dt and z [batch, width], B and C [batch, states]; `state` [batch, width, states] (float32,
    contiguous) is updated in place; reset [batch].  Returns y.  Without gradient."""
    return (_binding or binding()).selective_scan_step(u, dt, A, B, C, D, z, dt_bias, state, reset)

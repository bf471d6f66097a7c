"""Selective state space mixer: the short causal convolution and the selective scan, for prompts, training and single tokens.

The other recurrent token mixer of models that use the delta rule, with the same conventions: channels lie next to each other
(``[B, T, D]``), a call may carry states in and out, sequences of different lengths are packed along the time axis with
``cu_seqlens``, and everything runs in hand-written kernels behind the C ABI of ``include/hdla.h``.

``short_convolution`` / ``selective_scan`` take whole sequences and are differentiable; ``short_convolution_step`` /
``selective_scan_step`` take one token of each of B sequences and move the states on in place.  A prompt's final states are what
the steps go on with:

    x, conv_state = short_convolution(x, w_conv, b_conv, output_final_state=True)
    y, state = selective_scan(x, dt, A, B, C, D=skip, z=z, dt_bias=bias, output_final_state=True)
    ...                                                     # each further token
    x_t = short_convolution_step(x_t, conv_state, w_conv, b_conv)
    y_t = selective_scan_step(x_t, dt_t, A, B_t, C_t, state, D=skip, z=z_t, dt_bias=bias)

Inputs that are slices of a wider projection (dense along their last dimension) are read where they are.  Under CUDA graph
capture give ``cu_seqlens`` as an int64 tensor on the GPU; then nothing is copied or waited for, and a replay goes by what the
tensor then holds.  Offsets on the host are checked; those on the GPU are not looked at before the kernels, which take the first one
as 0 and cut the others to 0..T: they must not fall (nothing outside the tensors is touched if they do, but what comes out means
nothing).  Rows behind the last offset may hold anything.  The gradients have no graph of their own (no double backward).
``torch.jit.trace`` records the operators for whole sequences as calls; the steps refuse to be traced.  ``torch.compile`` leaves all
of them out of its graphs.
"""
from __future__ import annotations

import operator
from typing import Optional, Tuple

import torch

from . import _lib
from .hrdplr import _plain, autocast_custom_bwd, autocast_custom_fwd, save_workspace_default

MAX_TAPS, MAX_STATES, MAX_TOKENS = 8, 128, 1 << 30
# torch.compile leaves the operators out of its graphs: while it looks at one, that one calls itself as torch.compiler.disable
# gives it.  (As a decorator that would cost a single-token call a tenth of its time.)
_compiling = torch.compiler.is_dynamo_compiling


# ------------------------------------------------------------------------------------------ arguments
def _offsets(cu_seqlens, x) -> Optional[torch.Tensor]:
    """Offsets of a packed batch as an int64 tensor on x's device.  Those that are on the host are checked there; a tensor on the
    GPU is not looked at (that would wait for it): offsets outside 0..T are cut to that range by the kernels."""
    if cu_seqlens is None:
        return None
    if isinstance(cu_seqlens, torch.Tensor) and cu_seqlens.is_cuda:
        if cu_seqlens.dtype == torch.int64 and cu_seqlens.is_contiguous():
            return cu_seqlens
        if cu_seqlens.is_floating_point() or cu_seqlens.dim() != 1:
            raise ValueError("cu_seqlens must be a vector of integers")
        return cu_seqlens.to(torch.int64).contiguous()
    try:
        host = [operator.index(c) for c in (cu_seqlens.tolist() if isinstance(cu_seqlens, torch.Tensor) else cu_seqlens)]
    except TypeError:
        raise ValueError("cu_seqlens must be a vector of integers") from None
    _need(x.dim() == 3, f"x must have 3 dimensions [B, T, D], got {x.dim()}")
    T = x.shape[1]
    if len(host) < 2 or host[0] != 0 or host[-1] > T or any(b < a for a, b in zip(host, host[1:])):
        raise ValueError(f"cu_seqlens {host} must rise from 0 to at most T={T}")
    return torch.tensor(host, dtype=torch.int64, device=x.device)


def _need(ok: bool, text: str) -> None:
    if not ok:
        raise ValueError(text)


def _need_type(ok: bool, text: str) -> None:
    if not ok:
        raise TypeError(text)


def _check_packed(x, cu) -> int:
    """Number of states of the batch."""
    if cu is None:
        return x.shape[0]
    _need(x.shape[0] == 1, f"The batch size is expected to be 1 rather than {x.shape[0]} when using `cu_seqlens`.")
    _need(cu.dim() == 1 and cu.shape[0] >= 2, "cu_seqlens must be a vector of at least two offsets")
    _lib.require_cuda(x, cu)
    return cu.shape[0] - 1


def _check_conv(x, weight, bias, activation, state, n, rows) -> None:
    _lib.require_cuda(x, weight, bias, state)
    D = x.shape[-1]
    _need(weight.dim() == 2 and weight.shape[0] == D, f"weight {tuple(weight.shape)} must be [D, W] with D={D}")
    W = weight.shape[1]
    _need(1 <= W <= MAX_TAPS, f"{W} taps: 1 to {MAX_TAPS} are supported")
    _need(x.numel() > 0, f"x {tuple(x.shape)} is empty")
    _need(rows == 2 or x.shape[1] <= MAX_TOKENS, f"T={x.shape[-2]}: at most {MAX_TOKENS} tokens are supported")
    _need(bias is None or tuple(bias.shape) == (D,), "bias must be [D]")
    _lib.dtype_code(x.dtype)
    _lib.dtype_code(weight.dtype)
    _need_type(bias is None or bias.is_floating_point(), "bias must be a floating-point tensor")
    if state is not None:
        _need(tuple(state.shape) == (n, W - 1, D), f"the state {tuple(state.shape)} must be [{n}, W-1, D] = {(n, W - 1, D)}")
        _need_type(state.dtype == x.dtype, f"the state holds rows of x: it must be {x.dtype}, not {state.dtype}")


def _check_scan(x, dt, A, B, C, D, z, dt_bias, state, n) -> None:
    _lib.require_cuda(x, dt, A, B, C, D, z, dt_bias, state)
    lead, ch = tuple(x.shape[:-1]), x.shape[-1]
    _need(x.numel() > 0, f"x {tuple(x.shape)} is empty")
    _need(len(lead) == 1 or x.shape[1] <= MAX_TOKENS, f"T={x.shape[-2]}: at most {MAX_TOKENS} tokens are supported")
    _need(A.dim() == 2 and A.shape[0] == ch, f"A {tuple(A.shape)} must be [D, N] with D={ch}")
    N = A.shape[1]
    _need(1 <= N <= MAX_STATES, f"N={N}: 1 to {MAX_STATES} states are supported")
    _need(dt.shape == x.shape, f"dt {tuple(dt.shape)} must match x {tuple(x.shape)}")
    _need(z is None or z.shape == x.shape, f"z must match x {tuple(x.shape)}")
    for name, t in (("B", B), ("C", C)):
        _need(t.dim() in (len(lead) + 1, len(lead) + 2) and tuple(t.shape[:len(lead)]) == lead and t.shape[-1] == N,
              f"{name} {tuple(t.shape)} must be {list(lead)} + [G, N] or + [N] with N={N}")
    _need(B.shape == C.shape, f"B {tuple(B.shape)} and C {tuple(C.shape)} must have one shape")
    G = B.shape[-2] if B.dim() == len(lead) + 2 else 1
    _need(G >= 1 and ch % G == 0, f"{G} groups do not divide {ch} channels")
    for name, t in (("D", D), ("dt_bias", dt_bias)):
        _need(t is None or tuple(t.shape) == (ch,), f"{name} must be [D] with D={ch}")
    _need(state is None or tuple(state.shape) == (n, ch, N), f"the state must be [{n}, D, N] = {(n, ch, N)}")
    _lib.dtype_code(x.dtype)
    _need_type(all(t is None or t.dtype == x.dtype for t in (dt, B, C, z)), "x, dt, B, C, z must share one dtype")
    _need_type(all(t is None or t.is_floating_point() for t in (A, D, dt_bias, state)), "A, D, dt_bias and states must be floating-point tensors")


def _a_step_can_be_taken(*tensors) -> None:
    if torch.jit.is_tracing():
        raise RuntimeError("single-token steps update their state in place, which a trace would not record: they cannot be traced "
                           "with torch.jit.trace")
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors):
        raise RuntimeError("single-token steps update their state in place and have no backward; use the operator for whole "
                           "sequences, or torch.no_grad()")


# ------------------------------------------------------------------------------------------ tensor subclasses, tracing
class _ShortConv(torch.autograd.Function):
    """The operator for arguments that need a Python autograd function."""

    @staticmethod
    @autocast_custom_fwd
    def forward(ctx, x, weight, bias, silu, h0, cu, want):
        ctx.silu = silu
        ctx.save_for_backward(x, weight, bias, h0, cu)
        r = _lib.native().short_conv(*[_plain(t) for t in (x, weight, bias)], silu, _plain(h0), _plain(cu), want, True)
        if r is NotImplemented:
            raise TypeError("short_convolution: unsupported arguments")
        return r

    @staticmethod
    @autocast_custom_bwd
    def backward(ctx, dy, dht):
        x, weight, bias, h0, cu = [_plain(t) for t in ctx.saved_tensors]
        dx, dw, db, dh0 = _lib.native().short_conv_backward(x, weight, bias, ctx.silu, h0, cu, _plain(dy), _plain(dht))
        return dx, dw, db, None, dh0, None, None


class _SelectiveScan(torch.autograd.Function):
    """The operator for arguments that need a Python autograd function."""

    @staticmethod
    @autocast_custom_fwd
    def forward(ctx, x, dt, A, B, C, D, z, dt_bias, softplus, h0, cu, want):
        keep = save_workspace_default() and any(
            isinstance(t, torch.Tensor) and t.requires_grad for t in (x, dt, A, B, C, D, z, dt_bias, h0))
        r = _lib.native().selective_scan(*[_plain(t) for t in (x, dt, A, B, C, D, z, dt_bias)], softplus, _plain(h0), _plain(cu),
                                         want, keep)
        if r is NotImplemented:
            raise TypeError("selective_scan: unsupported arguments")
        y, ht, checkpoints = r
        ctx.softplus = softplus
        ctx.save_for_backward(x, dt, A, B, C, D, z, dt_bias, h0, cu, checkpoints)
        return y, ht

    @staticmethod
    @autocast_custom_bwd
    def backward(ctx, dy, dht):
        x, dt, A, B, C, D, z, dt_bias, h0, cu, checkpoints = [_plain(t) for t in ctx.saved_tensors]
        g = _lib.native().selective_scan_backward(x, dt, A, B, C, D, z, dt_bias, ctx.softplus, h0, cu, checkpoints, _plain(dy), _plain(dht))
        return (*g[:8], None, g[8], None, None)


# ------------------------------------------------------------------------------------------ entry points
_ACTIVATIONS = {None: False, "silu": True}


def _silu(activation) -> bool:
    if activation not in _ACTIVATIONS:
        raise ValueError(f"activation {activation!r} must be 'silu' or None")
    return _ACTIVATIONS[activation]


def short_convolution(
    x: torch.Tensor,                               # [B, T, D]
    weight: torch.Tensor,                          # [D, W]
    bias: Optional[torch.Tensor] = None,           # [D]
    activation: Optional[str] = "silu",
    initial_state: Optional[torch.Tensor] = None,  # [n, W-1, D], of x's type
    output_final_state: bool = False,
    cu_seqlens=None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Depthwise causal convolution: ``y_t = act(bias + sum_{k<W} weight[:, W-1-k] x_{t-k})`` for W of 1 to 8 taps.  The rows
    before a sequence come from ``initial_state`` (its last row the most recent) or are zero; the final state is the last W-1 rows
    of (initial state, x).  Weight and bias may be of other types than x and than each other; all arithmetic is fp32.  With
    ``cu_seqlens`` B is 1 and n the number of sequences; rows behind the last offset give zeros."""
    if _compiling():
        return _short_convolution(x, weight, bias, activation, initial_state, output_final_state, cu_seqlens)
    silu = _silu(activation)
    cu = _offsets(cu_seqlens, x)
    r = (_lib._native or _lib.native()).short_conv(x, weight, bias, silu, initial_state, cu, output_final_state, False)
    if r is not NotImplemented:
        return r
    _need(x.dim() == 3, f"x must have 3 dimensions [B, T, D], got {x.dim()}")
    _check_conv(x, weight, bias, activation, initial_state, _check_packed(x, cu), 3)
    return _ShortConv.apply(x, weight, bias, silu, initial_state, cu, bool(output_final_state))


def short_convolution_step(
    x: torch.Tensor,                               # [B, D]
    state: torch.Tensor,                           # [B, W-1, D], updated in place
    weight: torch.Tensor,
    bias: Optional[torch.Tensor] = None,
    activation: Optional[str] = "silu",
) -> torch.Tensor:
    """One token of each of B sequences through ``short_convolution``; ``state`` (contiguous) moves on by one row in place."""
    if _compiling():
        return _short_convolution_step(x, state, weight, bias, activation)
    silu = _silu(activation)
    r = (_lib._native or _lib.native()).short_conv_step(x, state, weight, bias, silu)
    if r is not NotImplemented:
        return r
    _need(x.dim() == 2, f"x must have 2 dimensions [B, D], got {x.dim()}")
    _check_conv(x, weight, bias, activation, state, x.shape[0], 2)
    _need(state.is_contiguous(), "the state is updated in place: it must be contiguous")
    _a_step_can_be_taken(x, state, weight, bias)
    r = _lib.native().short_conv_step(*[_plain(t) for t in (x, state, weight, bias)], silu)
    if r is NotImplemented:
        raise TypeError("short_convolution_step: unsupported arguments")
    return r


def selective_scan(
    x: torch.Tensor,                               # [B, T, D]
    dt: torch.Tensor,                              # [B, T, D]
    A: torch.Tensor,                               # [D, N]  decay rates (<= 0)
    B: torch.Tensor,                               # [B, T, G, N] or [B, T, N]
    C: torch.Tensor,                               # like B
    D: Optional[torch.Tensor] = None,              # [D]  skip weight
    z: Optional[torch.Tensor] = None,              # [B, T, D]  gate
    dt_bias: Optional[torch.Tensor] = None,        # [D]
    dt_softplus: bool = True,
    initial_state: Optional[torch.Tensor] = None,  # [n, D, N] fp32
    output_final_state: bool = False,
    cu_seqlens=None,
) -> Tuple[torch.Tensor, Optional[torch.Tensor]]:
    """Selective scan over D channels of N states (1 to 128), groups of D / G channels sharing B and C:
    ``d_t = softplus(dt_t + dt_bias)``, ``h_t = exp(d_t A) h_{t-1} + d_t x_t B_t``, ``y_t = (C_t . h_t + D x_t) silu(z_t)``.
    x, dt, z, B, C are fp32 or bf16, all of one type; A, D, dt_bias and the states are used in fp32, and all arithmetic is fp32.
    The final state is fp32.  A call that needs gradients keeps its states at every eighth token for backward, in fp32: N / 2 bytes a
    token and channel (N rounded up to 8, 16, 32, 64 or 128; at 16 states four times x in bf16).  With HDLA_RECOMPUTE=1 in the
    environment nothing of them is kept, and backward runs the forward pass once more.  Rows of sequences are expected to be finite
    (an infinite input gives NaN where the formula might give an infinity).  With ``cu_seqlens`` B is 1 and n the number of
    sequences; rows behind the last offset give zeros."""
    if _compiling():
        return _selective_scan(x, dt, A, B, C, D, z, dt_bias, dt_softplus, initial_state, output_final_state, cu_seqlens)
    cu = _offsets(cu_seqlens, x)
    softplus = bool(dt_softplus)
    r = (_lib._native or _lib.native()).selective_scan(x, dt, A, B, C, D, z, dt_bias, softplus, initial_state, cu, output_final_state, None)
    if r is not NotImplemented:
        return r
    _need(x.dim() == 3, f"x must have 3 dimensions [B, T, D], got {x.dim()}")
    _check_scan(x, dt, A, B, C, D, z, dt_bias, initial_state, _check_packed(x, cu))
    return _SelectiveScan.apply(x, dt, A, B, C, D, z, dt_bias, softplus, initial_state, cu, bool(output_final_state))


def selective_scan_step(
    x: torch.Tensor,                               # [B, D]
    dt: torch.Tensor,                              # [B, D]
    A: torch.Tensor,                               # [D, N]
    B: torch.Tensor,                               # [B, G, N] or [B, N]
    C: torch.Tensor,                               # like B
    state: torch.Tensor,                           # [B, D, N] fp32, updated in place
    D: Optional[torch.Tensor] = None,
    z: Optional[torch.Tensor] = None,
    dt_bias: Optional[torch.Tensor] = None,
    dt_softplus: bool = True,
) -> torch.Tensor:
    """One token of each of B sequences through ``selective_scan``; ``state`` (contiguous, fp32) moves on in place."""
    if _compiling():
        return _selective_scan_step(x, dt, A, B, C, state, D, z, dt_bias, dt_softplus)
    softplus = bool(dt_softplus)
    r = (_lib._native or _lib.native()).selective_scan_step(x, dt, A, B, C, D, z, dt_bias, softplus, state)
    if r is not NotImplemented:
        return r
    _need(x.dim() == 2, f"x must have 2 dimensions [B, D], got {x.dim()}")
    _check_scan(x, dt, A, B, C, D, z, dt_bias, state, x.shape[0])
    _need(state.dtype == torch.float32 and state.is_contiguous(), "the state is updated in place: it must be contiguous and float32")
    _a_step_can_be_taken(x, dt, A, B, C, D, z, dt_bias, state)
    r = _lib.native().selective_scan_step(*[_plain(t) for t in (x, dt, A, B, C, D, z, dt_bias)], softplus, _plain(state))
    if r is NotImplemented:
        raise TypeError("selective_scan_step: unsupported arguments")
    return r


_short_convolution, _short_convolution_step, _selective_scan, _selective_scan_step = (
    torch.compiler.disable(f) for f in (short_convolution, short_convolution_step, selective_scan, selective_scan_step))

"""Gated delta rule on B200: the chunked operator for sequences and the one-token step for decoding.

The second recurrence of this backend, for layers that correct what their state holds under a key instead of
adding to it.  Per value head, with a state ``S (P, N)`` and ``a_t = exp(g_t)``:

    y_t = v_t - a_t S_{t-1} k_t          (what the decayed state gets wrong about v_t)
    S_t = a_t S_{t-1} + beta_t y_t k_t^T
    o_t = scale * S_t q_t

Tensors are laid out as the scan's: ``q, k (b,Hk,T,N)``, ``v, o (b,H,T,P)``, ``g, beta (b,H,T)``, states
``(b,H,P,N)``.  Value head ``h`` reads key head ``h // (H // Hk)``.
"""

from __future__ import annotations

from typing import Optional

import torch

from .. import _lib
from . import _trace


def _check(q, k, v, g, beta, initial_state, tokens: bool) -> None:
    """Raises for arguments that the kernels cannot take."""
    names = ("q", "k", "v", "g", "beta")
    for name, t in zip(names, (q, k, v, g, beta)):
        if t.device.type != "cuda":
            raise ValueError(f"slinoss_b200 gated delta rule requires CUDA tensors ({name} is on {t.device}).")
    _lib.same_device(q, k, v, g, beta, initial_state)
    t = "T, " if tokens else ""
    if q.ndim != (4 if tokens else 3) or q.shape != k.shape:
        raise ValueError(f"q and k must be (batch, key_heads, {t}N) and equal. Got {tuple(q.shape)}, {tuple(k.shape)}.")
    if v.ndim != q.ndim or v.shape[0] != q.shape[0] or (tokens and v.shape[2] != q.shape[2]):
        raise ValueError(f"v must be (batch, heads, {t}P) beside q {tuple(q.shape)}. Got {tuple(v.shape)}.")
    H, Hk = int(v.shape[1]), int(q.shape[1])
    if Hk == 0 or H % Hk != 0:
        raise ValueError(f"the heads of v ({H}) must be a multiple of those of q and k ({Hk}).")
    for name, x in (("g", g), ("beta", beta)):
        if x.shape != v.shape[:-1]:
            raise ValueError(f"{name} must be {tuple(v.shape[:-1])}. Got {tuple(x.shape)}.")
    if not (q.dtype == k.dtype == v.dtype):
        raise TypeError(f"q, k and v must share one dtype. Got {q.dtype}, {k.dtype}, {v.dtype}.")
    for x in (v, g, beta):
        _lib.dtype_code(x.dtype)
    P, N = int(v.shape[-1]), int(q.shape[-1])
    if not 1 <= N <= 128:
        raise ValueError(f"key dim N must be 1..128. Got {N}.")
    if not 1 <= P <= 256:
        raise ValueError(f"value dim P must be 1..256. Got {P}.")
    want = (int(v.shape[0]), H, P, N)
    if initial_state is not None and tuple(initial_state.shape) != want:
        raise ValueError(f"initial_state must be (batch,heads,P,N)={want}. Got {tuple(initial_state.shape)}.")
    if tokens and want[0] * H > 65535:
        raise ValueError(f"batch * heads must be at most 65535. Got {want[0] * H}.")


def _dense(t):
    return t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()


@torch.compiler.disable
def gated_delta_rule_b200(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                          scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                          return_state: bool = False, residual: str = "keep"):
    """``o`` or ``(o, final_state)``, differentiable in ``q, k, v, g, beta`` and ``initial_state``.

    ``scale`` defaults to ``N ** -0.5``.  ``q, k, v`` share one dtype (float32, bfloat16 or float16), ``g`` and ``beta``
    may each have another; any strides are read as they are where the last axis of ``q, k, v`` is dense (column slices
    of one projection, token-major or head-major).  ``N <= 128``, ``P <= 256``.  The state is carried in fp32 and
    ``final_state`` is fp32; ``o`` and the gradients have the dtypes of what they belong to.

    ``g`` is a log decay (usually negative); ``-inf`` drops the state, which separates documents packed into one
    sequence.  Tokens with ``beta = 0`` and ``g = 0`` leave the state as it is, which pads sequences.  The recurrence is
    stable for ``beta |k|^2 < 2``; keys usually come normalised.  At most 65535 heads (``batch * heads``).

    A non-finite value among the inputs (``-inf`` in ``g`` apart) makes NaN of what is scaled together with it: from its
    chunk of 64 tokens on all outputs of the heads that read it for ``k``, ``g`` and ``beta``, those of its block of 16
    value channels for ``v`` and ``initial_state``, and the outputs of its chunk alone for ``q``.  Gradients are NaN where
    they meet one of these.

    Accuracy.  fp32 and fp16 results and all states are formed from operands of 22 bits, bfloat16 ones from operands of 11:
    gradients of fp32 gates beside bfloat16 activations are right to about ``1e-3``.  Values are held relative to the
    largest of their chunk of 64 tokens: what a closing gate inside a chunk makes smaller than ``2^-31`` of it may come back
    as zero.  The carried state and the gradient of the gate itself keep their own scale; below ``2^-100`` anything may be
    taken for zero.  With ``N < 16`` keys are alike, and the initial state's and the gates' gradients are differences of sums
    over a chunk, each right to ``2^-16`` of its terms: ``2^-15`` of the result for unit keys and tokens of like size, less
    (``1e-3`` at ``N = 1``) where ``beta`` is near 2 or tokens differ in size a thousandfold.

    ``residual`` chooses what autograd keeps: ``"keep"`` (default) what the forward has made of its inputs, and none of
    them: per 64 tokens and value head the triangular matrices of the chunk, the state before it and the prediction
    errors, per key head the keys and queries as scaled fp16 tiles (93 KB at ``N = 128, P = 64`` in bfloat16, where ``q``
    and ``k`` have 32); ``"recompute"`` nothing but the inputs: the backward runs one more forward pass, with bitwise
    the same gradients.
    """
    if residual not in ("keep", "recompute"):
        raise ValueError(f"residual must be 'keep' or 'recompute'. Got {residual!r}.")
    if scale is None:
        scale = float(q.shape[-1]) ** -0.5 if q.shape[-1] else 1.0
    if _trace.tracing():
        def call(q, k, v, g, beta, init):
            o = gated_delta_rule_b200(q, k, v, g, beta, scale=scale, initial_state=init, return_state=return_state,
                                      residual=residual)
            return o if return_state else (o,)
        out = _trace.recorded(call, q, k, v, g, beta, initial_state)
        return out if return_state else out[0]
    out = _lib.host().gated_delta_rule(q, k, v, g, beta, scale, initial_state, return_state, residual == "recompute")
    if out is None:
        _check(q, k, v, g, beta, initial_state, True)
        b, H, T, P = map(int, v.shape)
        if T == 0 or b == 0 or H == 0:
            o = v.new_empty(v.shape)
            if not return_state:
                return o
            return o, (torch.zeros((b, H, P, int(q.shape[-1])), device=v.device, dtype=torch.float32)
                       if initial_state is None else initial_state.to(torch.float32, copy=True))
        if initial_state is not None and not initial_state.is_floating_point():
            raise TypeError(f"initial_state must be a floating-point tensor. Got {initial_state.dtype}.")
        init = initial_state
        if init is not None:
            init = (init if init.dtype in _lib._DTYPE_CODE else init.to(torch.float32)).contiguous()
        out = _lib.host().gated_delta_rule(_dense(q), _dense(k), _dense(v), g, beta, scale, init, return_state,
                                           residual == "recompute")
        if out is None:
            raise ValueError(f"gated delta rule: unsupported arguments q {tuple(q.shape)}, v {tuple(v.shape)}.")
    return tuple(out) if return_state else out[0]


@torch.compiler.disable
def gated_delta_step_b200(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, g: torch.Tensor, beta: torch.Tensor, *,
                          scale: Optional[float] = None, initial_state: Optional[torch.Tensor] = None,
                          final_state_out: Optional[torch.Tensor] = None):
    """One token: ``q, k (b,Hk,N)``, ``v (b,H,P)``, ``g, beta (b,H)`` -> ``(o (b,H,P), final_state (b,H,P,N) fp32)``.

    The arithmetic of ``gated_delta_rule_b200`` at ``T = 1``, in fp32 throughout.  Without ``initial_state`` the state
    is zero.  ``final_state_out`` (fp32, contiguous) receives the state; ``final_state_out=initial_state`` updates it in
    place (otherwise the two must not overlap).  Inference only (no autograd)."""
    if scale is None:
        scale = float(q.shape[-1]) ** -0.5 if q.shape[-1] else 1.0
    out = _lib.host().gated_delta_step(q, k, v, g, beta, scale, initial_state, final_state_out)
    if out is not None:
        return out
    _check(q, k, v, g, beta, initial_state, False)
    b, H, P = map(int, v.shape)
    want = (b, H, P, int(q.shape[-1]))
    if final_state_out is not None:
        if tuple(final_state_out.shape) != want:
            raise ValueError(f"final_state_out must be {want}. Got {tuple(final_state_out.shape)}.")
        if final_state_out.device != v.device:
            raise ValueError(f"final_state_out must be on {v.device}.")
        if final_state_out.dtype != torch.float32:
            raise TypeError(f"final_state_out must be float32. Got {final_state_out.dtype}.")
        if not final_state_out.is_contiguous():
            raise ValueError(f"final_state_out must be contiguous; got strides {final_state_out.stride()}.")
    if b == 0 or H == 0:
        return v.new_empty(v.shape), v.new_empty(want, dtype=torch.float32) if final_state_out is None else final_state_out
    with torch.no_grad():
        init = None if initial_state is None else initial_state.to(torch.float32).contiguous()
        out = _lib.host().gated_delta_step(_dense(q), _dense(k), _dense(v), g, beta, scale, init, final_state_out)
    if out is None:
        raise ValueError(f"gated delta step: unsupported arguments q {tuple(q.shape)}, v {tuple(v.shape)}.")
    return out


__all__ = ["gated_delta_rule_b200", "gated_delta_step_b200"]

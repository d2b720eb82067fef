"""Tokens from logits on B200: the last step of a decode loop, on the device and from given random numbers."""

from __future__ import annotations

import torch

from .. import _lib


def _setting(name, x, logits, low, high):
    """A setting as ``(tensor of one fp32 value per row or None, number)``."""
    if not isinstance(x, torch.Tensor):
        x = float(x)
        if not low <= x <= high:
            raise ValueError(f"{name} must be in [{low}, {high}]. Got {x}.")
        return None, x
    if tuple(x.shape) != (logits.shape[0],):
        raise ValueError(f"{name} must be a number or ({logits.shape[0]},). Got {tuple(x.shape)}.")
    _lib.same_device(logits, x)
    return x.to(torch.float32).contiguous(), 0.0


@torch.compiler.disable
def sample_b200(logits: torch.Tensor, u: torch.Tensor, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0) -> torch.Tensor:
    """``logits (b, V)`` and random numbers ``u (b,)`` in ``[0, 1)`` -> tokens ``(b,)`` int64.

    Tokens are ranked by logit (ties: the lower index first).  The first ``top_k`` stay (``<= 0``: all); of these the
    shortest run that holds at least ``top_p`` of their mass; of these the ones with at least ``min_p`` of the largest
    mass (the first always stays).  The draw takes, in the order of the indices, the first token at which the running
    mass exceeds ``u`` times the whole.  Masses are ``exp((logit - largest) / temperature)`` in 64 bits, rounded to
    multiples of ``2^-44``, so that a draw depends on nothing but its row: not on the batch, the device's load or the run.
    (A token more than 31 temperatures below the largest has no mass; borders and draws that lie within ``V 2^-44`` of a
    token's running mass may go either way.)

    Each setting is a number, or a tensor ``(b,)`` with one value per row (values of tensors are not checked:
    ``temperature <= 0``, ``top_p <= 0`` and ``min_p > 1`` take the first largest logit, ``top_p >= 1`` keeps all).
    ``u`` is float32 or float64.  NaN logits count as ``-inf``; where several logits are ``+inf`` they share the mass; a
    row without any logit above ``-inf`` gives ``-1``.  ``b <= 65535``, ``V <= 262144``; rows may have any stride."""
    out = None
    if logits.ndim == 2:
        numbers = [x for x in (temperature, top_p, min_p) if not isinstance(x, torch.Tensor)]
        if all(0.0 <= x for x in numbers):  # (the plain call: everything else is looked at below)
            pick = lambda x: (x, 0.0) if isinstance(x, torch.Tensor) else (None, float(x))
            k = (top_k, 0) if isinstance(top_k, torch.Tensor) else (None, int(top_k))
            if (isinstance(top_p, torch.Tensor) or top_p <= 1.0) and (isinstance(min_p, torch.Tensor) or min_p <= 1.0):
                out = _lib.host().sample(logits, u, *pick(temperature), *k, *pick(top_p), *pick(min_p))
    if out is not None:
        return out
    if logits.device.type != "cuda":
        raise ValueError("slinoss_b200 sample requires CUDA tensors.")
    if logits.ndim != 2:
        raise ValueError(f"logits must be (batch, vocabulary). Got {tuple(logits.shape)}.")
    _lib.dtype_code(logits.dtype)
    b, V = map(int, logits.shape)
    if not 1 <= V <= 262144:
        raise ValueError(f"the vocabulary must have 1..262144 tokens. Got {V}.")
    if b > 65535:
        raise ValueError(f"the batch must be at most 65535 rows. Got {b}.")
    if tuple(u.shape) != (b,):
        raise ValueError(f"u must be ({b},). Got {tuple(u.shape)}.")
    if u.dtype not in (torch.float32, torch.float64):
        raise TypeError(f"u must be float32 or float64. Got {u.dtype}.")
    _lib.same_device(logits, u)
    inf = float("inf")
    t, t0 = _setting("temperature", temperature, logits, 0.0, inf)
    p, p0 = _setting("top_p", top_p, logits, 0.0, 1.0)
    m, m0 = _setting("min_p", min_p, logits, 0.0, 1.0)
    k, k0 = None, 0
    if isinstance(top_k, torch.Tensor):
        if tuple(top_k.shape) != (b,):
            raise ValueError(f"top_k must be a number or ({b},). Got {tuple(top_k.shape)}.")
        if top_k.is_floating_point() or top_k.is_complex() or top_k.dtype == torch.bool:
            raise TypeError(f"top_k must hold integers. Got {top_k.dtype}.")
        _lib.same_device(logits, top_k)
        k = (top_k if top_k.dtype in (torch.int32, torch.int64) else top_k.to(torch.int64)).contiguous()
    else:
        k0 = int(top_k)
    if b == 0:
        return torch.empty((0,), device=logits.device, dtype=torch.int64)
    dense = logits if V == 1 or logits.stride(1) == 1 else logits.contiguous()
    out = _lib.host().sample(dense.detach(), u.contiguous(), t, t0, k, k0, p, p0, m, m0)
    if out is None:
        raise ValueError(f"sample: unsupported arguments {tuple(logits.shape)}.")
    return out


__all__ = ["sample_b200"]

"""Gradients of gates that are nearly closed: as small as what they let through, and right to that.

Tolerances (2-norm of the difference over 2-norm of the result, head by head or over one token of every head): dg is a sum of
products over what crosses a gate, each with its decay.  With bf16 activations two operands of a product hold 11 bits (2^-11
each), made from operands that hold 11 bits themselves, in two passes: 8 * 2^-11, as for the other gradients; with fp16 and
fp32 1e-5.  The gates are fp32 here, so that no rounding of the result hides what its sum is worth.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gated_delta_gpu import _np, make, reference, run

pytestmark = pytest.mark.gpu

TOL = {"bf16": 2.0 ** -8, "fp16": 1e-5, "fp32": 1e-5}


def gate_errors(inp, axes):
    got = _np(run(inp)[2]["g"])
    want = reference(inp)[2]["g"]
    norm = lambda x: np.sqrt((x ** 2).sum(axes))
    return norm(got - want) / norm(want), norm(want)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("g", [-0.5, -3.0, -5.0, -8.0, -12.0, -20.0, -40.0])
@pytest.mark.parametrize("b,h,hk,T,N,P", [(1, 3, 3, 192, 128, 64), (2, 4, 2, 130, 64, 24), (1, 2, 1, 100, 96, 130)])
def test_heads_of_one_decay(dtype, g, b, h, hk, T, N, P):
    inp = make(b, h, hk, T, N, P, dtype, seed=41, gates="fp32")
    inp["g"].fill_(g)
    err, _ = gate_errors(inp, 2)
    print(f"{err.max():.2e}")
    assert err.max() <= TOL[dtype], err


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("g", [-8.0, -20.0, -60.0])
@pytest.mark.parametrize("N,P", [(64, 32), (128, 64)])
def test_one_closed_gate_among_open_ones(dtype, g, N, P):
    """At every kind of place of a chunk, one of a head: what crosses the gate is far below what does not."""
    places = [0, 1, 15, 16, 17, 31, 32, 40, 47, 48, 62, 63, 64, 65, 100, 129]
    inp = make(16, 16, 16, 130, N, P, dtype, seed=42, gates="fp32")
    for h, t in enumerate(places):
        inp["g"][:, h, t] = g
    got, want = _np(run(inp)[2]["g"]), reference(inp)[2]["g"]
    for h, t in enumerate(places):
        err = np.linalg.norm(got[:, h, t] - want[:, h, t]) / np.linalg.norm(want[:, h, t])
        assert err <= TOL[dtype], (t, err)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_heads_of_unlike_decays(dtype):
    """Open and closing heads side by side, each judged by itself; the other gradients as ever."""
    inp = make(1, 8, 4, 257, 64, 48, dtype, seed=43, gates="fp32", speed=1.0)
    inp["g"] *= torch.tensor([1e-3, 0.1, 1.0, 3.0, 6.0, 10.0, 20.0, 30.0], device="cuda")[None, :, None]
    err, _ = gate_errors(inp, 2)
    assert err.max() <= TOL[dtype], err


@pytest.mark.parametrize("dtype", ["bf16", "fp32"])
def test_many_heads_that_close(dtype):
    """The same where heads fill the GPU and warps walk along the sequence alone."""
    inp = make(40, 8, 8, 100, 64, 16, dtype, seed=44, gates="fp32")
    inp["g"][:, ::2] = -10.0
    err, _ = gate_errors(inp, 2)
    assert err.max() <= TOL[dtype], err.max()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("b", [2, 40])
@pytest.mark.parametrize("g", [-12.0, -30.0, -60.0])
def test_states_behind_closed_gates_keep_their_scale(dtype, b, g):
    """A gate that closes and nothing written behind it: the state is e^g of what it was, rows written before it in the same
    chunk included.  The other way round, the initial state's gradient where only what lies behind the gate is read: a gate
    inside a chunk enters by the chunk's triangular matrices, whose entries are pairs of fp16 beside a largest of one (off by
    2^-39 each); over 64 tokens and the three operands made with them that is 3 * 64 * 2^-39 < 2^-31 of what an open gate
    would give."""
    from oracle import delta as odelta
    from test_gated_delta_gpu import NAMES, tolerance
    from util import rel_err
    for t, T in [(20, 64), (63, 70), (64, 130), (100, 130)]:
        inp = make(b, 4, 4, T, 64, 32, dtype, seed=45 + t, gates="fp32")
        inp["g"][:, :, t] = g
        late = {n: x.clone() for n, x in inp.items()}
        late["beta"][:, :, t:] = 0
        _, final, _ = run(late)
        _, want, _ = odelta.forward(*(_np(late[n]) for n in NAMES[:5]), 0.125, _np(late["init"]))
        assert rel_err(_np(final), want) <= tolerance(inp["q"].dtype, "final", final.dtype), t
        inp["do"][:, :, :t] = 0
        got, ref = _np(run(inp)[2]["init"]), reference(inp)[2]["init"]
        inp["g"][:, :, t] = 0
        size = np.linalg.norm(reference(inp)[2]["init"])
        assert np.linalg.norm(got - ref) <= 1e-5 * np.linalg.norm(ref) + 2.0 ** -31 * size, t

"""Ends of what the gated delta rule accepts: keys of few values, one key throughout, and how far a non-finite value reaches."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from test_gated_delta_gpu import NAMES, _np, coarse, make, reference, run, tolerance
from util import rel_err

pytestmark = pytest.mark.gpu


# Unit keys of N values are alike where N is small (N = 1: all are +-1): what a token writes, the next ones overwrite.  The
# gradient of a chunk's initial state, the gates' with it, is then the difference of two sums over the chunk's 64 tokens of which
# as little may be left as one term; fp32 sums of operands of 22 bits are off by 64 * 2^-22 each, together by 2^-15.
@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("speed", [0.01, 1.0])
@pytest.mark.parametrize("N", [1, 2, 3, 5, 8, 12, 15])
def test_narrow_keys(dtype, speed, N):
    inp = make(2, 4, 2, 200, N, 32, dtype, seed=50 + N, speed=speed)
    o, final, grads = run(inp)
    ro, rfinal, rgrads = reference(inp)
    dt = inp["q"].dtype
    assert rel_err(_np(o), ro) <= tolerance(dt, "o", dt)
    assert rel_err(_np(final), rfinal) <= tolerance(dt, "final", final.dtype)
    for n, t in grads.items():
        extra = 2.0 ** -15 if n in ("init", "g") else 0.0
        operands = tolerance(dt, "q", t.dtype) if n == "g" else tolerance(dt, n, t.dtype)  # (dg: as the other gradients)
        assert rel_err(_np(t), rgrads[n]) <= operands + extra + coarse(t, rgrads[n]), n


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_one_token_and_one_value_channel(dtype):
    for T, N, P in [(1, 1, 1), (64, 1, 1), (65, 2, 1), (3, 1, 16)]:
        inp = make(8, 8, 8, T, N, P, dtype, seed=60 + T)
        o, final, grads = run(inp)
        ro, rfinal, rgrads = reference(inp)
        dt = inp["q"].dtype
        assert rel_err(_np(o), ro) <= tolerance(dt, "o", dt) and rel_err(_np(final), rfinal) <= tolerance(dt, "final", final.dtype)
        for n, t in grads.items():
            extra = 2.0 ** -15 if n in ("init", "g") else 0.0
            assert rel_err(_np(t), rgrads[n]) <= tolerance(dt, n, t.dtype) + extra + coarse(t, rgrads[n]), (T, n)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("many", [False, True])
@pytest.mark.parametrize("name", ["q", "k", "v", "g", "beta", "init"])
def test_how_far_a_non_finite_value_reaches(dtype, many, name):
    """From its chunk of 64 tokens on the heads that read it (k, g, beta), there its block of 16 value channels (v, the initial
    state), or the outputs of its chunk (q) are NaN.  Everything else keeps its bits."""
    import slinoss_b200 as sb
    inp = make(60 if many else 2, 4, 2, 200, 64, 48, dtype, seed=70)

    def forward(x):
        o, final = sb.gated_delta_rule_b200(*(x[n] for n in NAMES[:5]), initial_state=x["init"], return_state=True)
        return o, final

    clean, clean_final = forward(inp)
    at = {"q": (1, 1, 70, 3), "k": (1, 1, 70, 3), "v": (1, 2, 70, 20), "g": (1, 2, 70), "beta": (1, 2, 70), "init": (1, 2, 20, 5)}
    for value in (torch.nan, torch.inf):
        bad = dict(inp)
        bad[name] = inp[name].clone()
        bad[name][at[name]] = value
        o, final = forward(bad)
        hit, hit_final = torch.zeros_like(o, dtype=torch.bool), torch.zeros_like(final, dtype=torch.bool)
        heads = slice(2, 4) if name in ("q", "k") else slice(2, 3)
        tokens = slice(0, None) if name == "init" else slice(64, 128) if name == "q" else slice(64, None)
        channels = slice(16, 32) if name in ("v", "init") else slice(None)
        hit[1, heads, tokens, channels] = True
        if name != "q":
            hit_final[1, heads, channels] = True
        assert torch.equal(o.isnan(), hit) and torch.equal(final.isnan(), hit_final), value
        assert torch.equal(o[~hit], clean[~hit]) and torch.equal(final[~hit_final], clean_final[~hit_final]), value


# Independent roundings add up like the root of their number.  bf16: a result's own (steps of at most 2^-7 of it: 2^-7 / sqrt 12 =
# 2.3e-3) and eight operands' of 11 bits (2^-10 / sqrt 12 each, together 8e-4): 2.4e-3, held to 3e-3.  fp16: 2^-10 / sqrt 12 =
# 2.8e-4 and operands that do not show: 3e-4.  fp32: eight operands of 22 bits (4e-7 together), left-out products of two low parts
# (2^-22 each), and sums whose instructions cut off up to 2^-24 at each of a chunk's 8 steps of 8 products, all downwards
# (64 * 2^-24 / 2 = 2e-6 at worst): 3e-6.
@pytest.mark.parametrize("dtype,bound,wide", [("bf16", 3e-3, 3e-6), ("fp16", 3e-4, 3e-6), ("fp32", 3e-6, 3e-6)])
@pytest.mark.parametrize("b,h,hk,T,N,P", [(2, 4, 2, 300, 128, 64), (20, 8, 8, 130, 64, 64), (1, 4, 4, 200, 128, 128)])
def test_errors_are_those_of_the_roundings(dtype, bound, wide, b, h, hk, T, N, P):
    inp = make(b, h, hk, T, N, P, dtype, seed=80)
    o, final, grads = run(inp)
    ro, rfinal, rgrads = reference(inp)
    errs = {"o": rel_err(_np(o), ro), **{n: rel_err(_np(t), rgrads[n]) for n, t in grads.items()}}
    assert rel_err(_np(final), rfinal) <= wide and errs.pop("init") <= wide
    assert max(errs.values()) <= bound, errs

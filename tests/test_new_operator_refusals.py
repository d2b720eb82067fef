"""Gated delta rule and sampling without a GPU: what the C entry points and the Python functions refuse, and the float64
oracles against differences and by hand."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import delta as odelta
from oracle import sample as osample


@pytest.fixture(scope="module")
def lib():
    from slinoss_b200 import _lib, build

    build.build()
    return _lib.lib()


def _shape(**kw):
    from slinoss_b200 import _lib
    a = dict(batch=1, heads=2, key_heads=1, T=8, P=16, N=16, dtype=0, g_dtype=0, beta_dtype=0, scale=1.0)
    a.update(kw)
    return _lib.GatedDeltaShape(*(a[n] for n in ("batch", "heads", "key_heads", "T", "P", "N", "dtype", "g_dtype",
                                                 "beta_dtype", "scale")))


@pytest.mark.parametrize("kw,code", [(dict(batch=0), -2), (dict(T=-1), -2), (dict(key_heads=3), -2), (dict(key_heads=0), -2),
                                     (dict(N=129), -3), (dict(P=257), -3), (dict(batch=40000), -3), (dict(dtype=3), -5),
                                     (dict(g_dtype=-1), -5), (dict(beta_dtype=7), -5)])
def test_shapes_that_no_kernel_takes(lib, kw, code):
    s = ctypes.byref(_shape(**kw))
    one = ctypes.c_void_p(256)
    assert lib.slx_gated_delta_fwd(s, *([one] * 5), None, 0, one, None, None, one, 1 << 40, None) == code
    assert lib.slx_gated_delta_bwd(s, one, one, None, 0, *([one] * 5), None, 0, one, 1 << 40, None) == code
    assert lib.slx_gated_delta_fwd_workspace_bytes(s) == 0
    assert lib.slx_gated_delta_residual_bytes(s) == 0 and lib.slx_gated_delta_bwd_workspace_bytes(s) == 0


def test_pointers_and_workspaces(lib):
    s = _shape()
    r = ctypes.byref(s)
    one, n = ctypes.c_void_p(256), lib.slx_gated_delta_fwd_workspace_bytes(ctypes.byref(s))
    fwd = lambda *a: lib.slx_gated_delta_fwd(r, *a, None)
    assert lib.slx_gated_delta_fwd(None, *([one] * 5), None, 0, one, None, None, one, n, None) == -1
    assert fwd(None, *([one] * 4), None, 0, one, None, None, one, n) == -1
    assert fwd(*([one] * 5), None, 0, one, None, None, None, n) == -1
    assert fwd(*([one] * 5), None, 0, one, None, None, one, n - 1) == -4
    assert fwd(*([one] * 5), None, 0, one, None, None, ctypes.c_void_p(264), n) == -4
    assert fwd(*([one] * 5), None, 0, one, None, ctypes.c_void_p(264), one, n) == -4
    assert fwd(*([one] * 5), one, 9, one, None, None, one, n) == -5
    m = lib.slx_gated_delta_bwd_workspace_bytes(r)
    bwd = lambda *a: lib.slx_gated_delta_bwd(r, *a, None)
    assert bwd(None, one, None, 0, *([one] * 5), None, 0, one, m) == -1
    assert bwd(one, one, None, 0, *([one] * 4), None, None, 0, one, m) == -1
    assert bwd(one, one, None, 0, *([one] * 5), None, 0, one, m - 1) == -4
    assert bwd(ctypes.c_void_p(264), one, None, 0, *([one] * 5), None, 0, one, m) == -4
    assert bwd(one, one, one, 5, *([one] * 5), None, 0, one, m) == -5
    assert bwd(one, one, None, 0, *([one] * 5), one, 5, one, m) == -5
    one_token = _shape(T=1)
    step = lambda sh, *a: lib.slx_gated_delta_step(ctypes.byref(sh), *a, None)
    assert step(s, *([one] * 5), None, one, one) == -2  # T is not 1
    assert step(one_token, *([one] * 5), None, None, one) == -1
    assert step(one_token, *([one] * 5), ctypes.c_void_p(256), one, ctypes.c_void_p(260)) == -2  # states that overlap
    # sizes past 32 bits: workspaces are counted in 64
    big = _shape(batch=1, heads=32, key_heads=32, T=1 << 30, P=64, N=128, dtype=1)
    assert lib.slx_gated_delta_fwd_workspace_bytes(ctypes.byref(big)) == 32 * (1 << 24) * (31360 + 2 * 64 * 136 * 2)


def test_sample_refusals(lib):
    from slinoss_b200 import _lib
    one = ctypes.c_void_p(256)
    call = lambda s, *a: lib.slx_sample(ctypes.byref(s), *a, None)
    make = lambda **kw: _lib.SampleShape(**{**dict(rows=2, vocab=10, dtype=0, u_bytes=4, top_k_bytes=8, temperature=1.0,
                                                   top_p=1.0, min_p=0.0, top_k=0, row_stride=10), **kw})
    assert call(make(), None, one, None, None, None, None, one) == -1
    assert call(make(rows=0), one, one, None, None, None, None, one) == -2
    assert call(make(vocab=262145), one, one, None, None, None, None, one) == -3
    assert call(make(dtype=4), one, one, None, None, None, None, one) == -5
    assert call(make(u_bytes=2), one, one, None, None, None, None, one) == -5
    assert call(make(top_k_bytes=2), one, one, None, one, None, None, one) == -5


def test_cpu_tensors_are_refused(lib):
    import slinoss_b200 as sb
    x = torch.zeros
    with pytest.raises(ValueError, match="CUDA"):
        sb.gated_delta_rule_b200(x(1, 1, 4, 8), x(1, 1, 4, 8), x(1, 1, 4, 8), x(1, 1, 4), x(1, 1, 4))
    with pytest.raises(ValueError, match="CUDA"):
        sb.gated_delta_step_b200(x(1, 1, 8), x(1, 1, 8), x(1, 1, 8), x(1, 1), x(1, 1))
    with pytest.raises(ValueError, match="CUDA"):
        sb.sample_b200(x(1, 8), x(1))


def test_oracle_gradients_against_differences():
    r = np.random.default_rng(0)
    b, h, hk, T, N, P = 1, 4, 2, 5, 4, 3
    x = dict(q=r.normal(size=(b, hk, T, N)), k=r.normal(size=(b, hk, T, N)) / 2, v=r.normal(size=(b, h, T, P)),
             g=-r.random((b, h, T)), beta=r.random((b, h, T)), init=r.normal(size=(b, h, P, N)))
    do, df = r.normal(size=(b, h, T, P)), r.normal(size=(b, h, P, N))
    args = lambda x: (x["q"], x["k"], x["v"], x["g"], x["beta"], 0.7, x["init"])

    def loss(x):
        o, final, _ = odelta.forward(*args(x))
        return (o * do).sum() + (final * df).sum()

    got = odelta.backward(*args(x), do, df)
    for n in x:
        d = r.normal(size=x[n].shape)
        want = (loss({**x, n: x[n] + 1e-6 * d}) - loss({**x, n: x[n] - 1e-6 * d})) / 2e-6
        assert abs(want - (got[n] * d).sum()) < 1e-7  # second differences of order one, times 1e-12 / 1e-6, and rounding


def test_oracle_draws_by_hand():
    row = np.log([0.1, 0.4, 0.2, 0.3])
    assert [osample.draw(row, u)[0] for u in (0.05, 0.2, 0.6, 0.9)] == [0, 1, 2, 3]
    assert np.count_nonzero(osample.kept(row, 1.0, 2, 1.0, 0.0)) == 2
    assert np.flatnonzero(osample.kept(row, 1.0, 0, 0.7, 0.0)).tolist() == [1, 3]
    assert np.flatnonzero(osample.kept(row, 1.0, 0, 0.71, 0.0)).tolist() == [1, 2, 3]
    assert np.flatnonzero(osample.kept(row, 1.0, 0, 1.0, 0.51)).tolist() == [1, 3]
    assert osample.kept(np.full(4, -np.inf), 1.0, 0, 1.0, 0.0) is None

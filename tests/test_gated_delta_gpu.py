"""The gated delta rule and its one-token step on the GPU against the float64 recurrence, through the public entry points.

Tolerances (2-norm of the difference over 2-norm of the result), by arithmetic:
* an output rounded to its dtype is off by at most eps / 2 per value;
* bf16 activations: computed operands hold 11 bits, off by 2^-11 each, at most four in a row on the way to a result and
  its gradients, which two passes (forward, backward) go through: 8 * 2^-11 = 2^-8 on top of the output's eps / 2 = 2^-8;
* fp16 and fp32 activations, and fp32 states: computed operands hold 22 bits, and sums of up to 64 + 128 products run in
  fp32 (2^-24 each, growing like their root: 14 * 2^-24); over a few chunks 1e-5 covers both, as for the scan;
* dg is a sum over the rest of its sequence of differences that cancel: its operands' share counts four times.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import delta as odelta
from util import rel_err

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NAMES = ("q", "k", "v", "g", "beta", "init")


def _np(t):
    return None if t is None else t.detach().double().cpu().numpy()


def make(b, h, hk, T, N, P, dtype, *, seed=0, init=True, gates=None, rows=False, speed=0.1, init_dtype=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    dt = DT[dtype]
    rand = lambda *s: torch.randn(*s, generator=gen, dtype=torch.float64)
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)
    q, k, v = unit(rand(b, hk, T, N)), unit(rand(b, hk, T, N)), rand(b, h, T, P)
    if rows:  # column slices of one token-major projection
        row = torch.cat([x.transpose(1, 2).flatten(2) for x in (q, k, v)], -1).to(dt).cuda()
        q = row[..., :hk * N].unflatten(-1, (hk, N)).transpose(1, 2)
        k = row[..., hk * N:2 * hk * N].unflatten(-1, (hk, N)).transpose(1, 2)
        v = row[..., 2 * hk * N:].unflatten(-1, (h, P)).transpose(1, 2)
    else:
        q, k, v = (x.to(dt).cuda() for x in (q, k, v))
    gd = DT[gates or dtype]
    g = (-speed * torch.nn.functional.softplus(rand(b, h, T))).to(gd).cuda()
    beta = torch.sigmoid(rand(b, h, T)).to(gd).cuda()
    inp = dict(q=q, k=k, v=v, g=g, beta=beta,
               init=(0.3 * rand(b, h, P, N)).to(init_dtype).cuda() if init else None)
    inp["do"] = rand(b, h, T, P).to(dt).cuda()
    inp["dfinal"] = (0.1 * rand(b, h, P, N)).float().cuda()
    return inp


def run(inp, *, scale=None, with_final=True, **kw):
    import slinoss_b200 as sb

    leaves = {n: None if inp[n] is None else inp[n].detach().requires_grad_(True) for n in NAMES}
    o, final = sb.gated_delta_rule_b200(*(leaves[n] for n in NAMES[:5]), scale=scale, initial_state=leaves["init"],
                                        return_state=True, **kw)
    outs, gs = ([o, final], [inp["do"], inp["dfinal"]]) if with_final else ([o], [inp["do"]])
    names = [n for n in NAMES if leaves[n] is not None]
    grads = dict(zip(names, torch.autograd.grad(outs, [leaves[n] for n in names], gs)))
    return o, final, grads


def reference(inp, *, scale=None, with_final=True):
    scale = inp["q"].shape[-1] ** -0.5 if scale is None else scale
    args = [_np(inp[n]) for n in NAMES[:5]]
    o, final, _ = odelta.forward(*args, scale, _np(inp["init"]))
    grads = odelta.backward(*args, scale, _np(inp["init"]), _np(inp["do"]), _np(inp["dfinal"]) if with_final else None)
    return o, final, grads


def tolerance(dtype, name, out_dtype):
    operands = 2.0 ** -8 if dtype == torch.bfloat16 and name not in ("final", "init") else 1e-5
    if name == "g":
        operands *= 4
    return operands + (0.0 if out_dtype == torch.float32 else torch.finfo(out_dtype).eps / 2)


def coarse(t, ref):
    """What rounding below the dtype's normal range adds: half of its smallest step a value, relative to the result's norm
    (fp16 values below 2^-14 are multiples of 2^-24: off by up to 2^-25 each)."""
    fi = torch.finfo(t.dtype)
    norm = np.linalg.norm(ref)
    return 0.5 * fi.smallest_normal * fi.eps * ref.size ** 0.5 / norm if norm > 0 else 0.0


def compare(inp, got, want):
    dt = inp["q"].dtype
    o, final, grads = got
    ro, rfinal, rgrads = want
    errs = {"o": (rel_err(_np(o), ro), tolerance(dt, "o", o.dtype)),
            "final": (rel_err(_np(final), rfinal), tolerance(dt, "final", final.dtype))}
    for n, t in grads.items():
        assert t.shape == inp[n].shape and t.dtype == inp[n].dtype
        errs["d" + n] = (rel_err(_np(t), rgrads[n]), tolerance(dt, n, t.dtype) + coarse(t, rgrads[n]))
    print({n: f"{e:.2e}" for n, (e, _) in errs.items()})
    for n, (e, tol) in errs.items():
        assert e <= tol, (n, e, tol)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("b,h,hk,T,N,P", [
    (1, 1, 1, 1, 16, 16),     # one token
    (2, 2, 2, 64, 64, 64),    # one whole chunk
    (1, 2, 1, 65, 128, 64),   # a chunk and one token
    (2, 3, 1, 130, 40, 24),   # widths that fill no tile
    (1, 4, 2, 200, 33, 17),   # widths that no vector access fits
    (1, 2, 2, 150, 128, 128),  # two tiles of value channels
    (1, 1, 1, 100, 96, 200),  # four, the last one ragged
    (2, 6, 2, 257, 64, 64),
    (1, 4, 2, 67, 33, 16),    # shared keys, whose gradients do not divide into fours
])
def test_forward_and_gradients(dtype, b, h, hk, T, N, P):
    inp = make(b, h, hk, T, N, P, dtype, seed=T + N + P)
    compare(inp, run(inp), reference(inp))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("b,h,hk,T,N,P", [
    (40, 4, 2, 70, 64, 32),     # 320 blocks of 16 value channels: a warp each
    (24, 4, 4, 130, 128, 64),   # 384, and the wide state
    (18, 6, 2, 100, 33, 40),    # 324: three warps a CTA, ragged widths
    (11, 2, 1, 65, 96, 130),    # 198: CTAs of four warps, of which the last ones are idle
    (32, 2, 2, 66, 40, 64),     # 256: two rounds of teams
])
def test_many_heads(dtype, b, h, hk, T, N, P):
    inp = make(b, h, hk, T, N, P, dtype, seed=b + P)
    compare(inp, run(inp), reference(inp))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_many_heads_are_as_few(dtype):
    """A head's result does not depend on which kernels the number of heads has chosen, but for roundings."""
    inp = make(40, 4, 4, 200, 64, 64, dtype, seed=31)
    few = {n: x if x is None else x[:2] for n, x in inp.items()}
    (o, final, grads), (o2, final2, grads2) = run(inp), run(few)
    dt = inp["q"].dtype
    assert rel_err(_np(o[:2]), _np(o2)) <= 2 * tolerance(dt, "o", dt)
    assert rel_err(_np(final[:2]), _np(final2)) <= 2 * tolerance(dt, "final", final.dtype)
    for n in grads2:
        assert rel_err(_np(grads[n][:2]), _np(grads2[n])) <= 2 * tolerance(dt, n, grads2[n].dtype), n


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("b", [2, 60])
def test_states_that_fade(dtype, b):
    """The state decays by 2^-100 and more while nothing is written: small values keep their scale, down to zero."""
    inp = make(b, 3, 3, 129, 128, 32, dtype, seed=33)
    inp["g"] = torch.full_like(inp["g"], -1.0)
    inp["beta"][:, :, 64:] = 0
    _, final, _ = run(inp)
    _, want, _ = odelta.forward(*(_np(inp[n]) for n in NAMES[:5]), 128 ** -0.5, _np(inp["init"]))
    assert rel_err(_np(final), want) <= tolerance(inp["q"].dtype, "final", final.dtype)
    inp["g"] = torch.full_like(inp["g"], -2.0)  # e^-130 of a state near one
    _, final, _ = run(inp)
    assert torch.isfinite(final).all() and float(final.detach().abs().max()) < 1e-37


def test_a_dropped_state_has_no_gate_gradient():
    inp = make(2, 2, 2, 150, 64, 32, "bf16", seed=34)
    for t in (0, 1, 16, 63, 64, 97, 149):
        inp["g"][:, :, t] = -torch.inf
    grads = run(inp)[2]
    assert (grads["g"][:, :, [0, 1, 16, 63, 64, 97, 149]] == 0).all() and (grads["g"][:, :, 2] != 0).all()
    one = make(1, 2, 2, 1, 64, 16, "fp32", seed=35)
    one["g"].fill_(-torch.inf)
    assert (run(one)[2]["g"] == 0).all()


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_special_rows_among_many(dtype):
    inp = make(84, 2, 2, 140, 64, 32, dtype, seed=32)
    far = 2.0 ** (10 if dtype == "fp16" else 30)
    inp["g"][0, :, [64, 70]] = -torch.inf
    inp["v"][1] *= far
    inp["init"][1] *= far
    for n in ("do", "dfinal"):
        inp[n][1] /= far
    inp["g"][2, :, 37:] = 0
    inp["beta"][2, :, 37:] = 0
    inp["v"][4, 1, 100, 5] = torch.inf
    o, final, grads = run(inp)
    for r in range(4):
        row = {n: x[r:r + 1] for n, x in inp.items()}
        compare(row, (o[r:r + 1], final[r:r + 1], {n: x[r:r + 1] for n, x in grads.items()}), reference(row))
    assert not torch.isfinite(o[4, 1, 100:, 5]).any() and not torch.isfinite(final[4, 1, 5]).any()
    assert not torch.isfinite(grads["k"][4, 1]).all()
    assert torch.isfinite(o[4, 0]).all() and all(torch.isfinite(x[5:]).all() for x in (o, final, *grads.values()))


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("rows", [False, True])
def test_strides_without_states(dtype, rows):
    inp = make(2, 4, 2, 140, 64, 32, dtype, seed=5, init=False, rows=rows)
    if rows:
        for n in ("g", "beta"):
            inp[n] = inp[n].transpose(1, 2).contiguous().transpose(1, 2)
    assert rows != inp["q"].is_contiguous()
    compare(inp, run(inp, scale=1.0, with_final=False), reference(inp, scale=1.0, with_final=False))


@pytest.mark.parametrize("gates", ["fp32", "bf16"])
@pytest.mark.parametrize("init_dtype", [torch.float32, torch.bfloat16])
def test_gates_and_states_in_other_dtypes(gates, init_dtype):
    inp = make(1, 4, 2, 100, 64, 64, "bf16", seed=7, gates=gates, init_dtype=init_dtype)
    compare(inp, run(inp), reference(inp))


def test_decays_from_open_to_closed():
    """Gates whose sums pass the range of fp32 exponentials inside a chunk, beside gates that are wide open."""
    inp = make(1, 3, 3, 192, 64, 64, "fp32", seed=8, speed=1.0)
    inp["g"][:, 0] *= 20.0
    inp["g"][:, 1] *= 1e-4
    compare(inp, run(inp), reference(inp))


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("cut", [[64], [1, 77], [10, 11, 100]])
def test_minus_infinity_separates_documents(dtype, cut):
    inp = make(1, 2, 2, 130, 64, 32, dtype, seed=9)
    whole = {n: t for n, t in inp.items()}
    whole["g"] = inp["g"].clone()
    whole["g"][:, :, cut] = -torch.inf
    o, final, grads = run(whole)
    ro, rfinal, rgrads = reference(whole)
    compare(whole, (o, final, grads), (ro, rfinal, rgrads))
    # every document by itself gives the same bits up to where chunks begin: the last one's outputs by value
    tail = {n: (t[:, :, cut[-1]:].contiguous() if n in ("q", "k", "v", "g", "beta", "do") else t) for n, t in inp.items()}
    tail["init"] = None
    to, tfinal, _ = run(tail)
    assert rel_err(_np(tfinal), _np(final)) < 1e-5
    assert rel_err(_np(to), _np(o[:, :, cut[-1]:])) < 2 * tolerance(inp["q"].dtype, "o", o.dtype)


def test_closed_and_padded_tokens_leave_the_state():
    inp = make(2, 2, 1, 90, 64, 64, "bf16", seed=10)
    for n in ("g", "beta"):
        inp[n][:, :, 37:] = 0
    _, final, grads = run(inp)
    head = {n: (t[:, :, :37].contiguous() if n in ("q", "k", "v", "g", "beta", "do") else t) for n, t in inp.items()}
    _, short, _ = run(head)
    assert rel_err(_np(final), _np(short)) < 1e-6
    assert all(torch.isfinite(t).all() for t in grads.values())
    compare(inp, run(inp), reference(inp))  # (beta = 0: its gradient is that of opening the gate)


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_equal_keys_and_full_writes(dtype):
    """beta = 1 with one key throughout: the triangular system is as far from the identity as unit keys make it."""
    inp = make(1, 2, 2, 128, 64, 32, dtype, seed=11, speed=0.01)
    inp["k"] = inp["k"][:, :, :1].expand(-1, -1, 128, -1).contiguous()
    inp["beta"] = torch.ones_like(inp["beta"])
    # each row of the inverse differs from its neighbour by an entry near -1: differences cancel up to 2 / (1 - e^g) of a value
    o, final, grads = run(inp)
    ro, rfinal, rgrads = reference(inp)
    for name, t, r in [("o", o, ro), ("final", final, rfinal), ("v", grads["v"], rgrads["v"]), ("q", grads["q"], rgrads["q"])]:
        assert rel_err(_np(t), r) < 4 * tolerance(inp["q"].dtype, name, t.dtype), name


@pytest.mark.parametrize("power", [-30, 30])
def test_magnitudes_far_from_one(power):
    """Values and output gradients of 2^+-30: operands are scaled per tile, nothing under- or overflows fp16."""
    inp = make(1, 2, 1, 140, 64, 32, "bf16", seed=12, init=False)
    inp["v"] = inp["v"] * 2.0 ** power
    inp["do"] = inp["do"] * 2.0 ** -power
    inp["dfinal"] = inp["dfinal"] * 2.0 ** -power
    compare(inp, run(inp), reference(inp))


def test_a_small_row_beside_large_ones():
    inp = make(1, 1, 1, 100, 64, 32, "bf16", seed=13, init=False)
    inp["v"][..., 3] *= 2.0 ** -20
    o, _, _ = run(inp)
    ro, _, _ = reference(inp)
    assert rel_err(_np(o)[..., 3], ro[..., 3]) < tolerance(torch.bfloat16, "o", torch.bfloat16)


def test_non_finite_values_never_come_back_finite():
    inp = make(1, 2, 2, 192, 64, 32, "bf16", seed=14)
    clean, clean_final, _ = run(inp)
    inp["v"][0, 1, 100, 5] = torch.inf
    o, final, _ = run(inp)
    assert torch.equal(o[0, 0], clean[0, 0]) and torch.equal(final[0, 0], clean_final[0, 0])
    assert torch.equal(o[0, 1, :64], clean[0, 1, :64])
    assert not torch.isfinite(o[0, 1, 100:, 5]).any() and not torch.isfinite(final[0, 1, 5]).any()


def test_gradients_against_differences():
    inp = make(1, 2, 1, 70, 16, 8, "fp32", seed=15)
    _, _, grads = run(inp)

    def loss(x):
        o, final, _ = odelta.forward(*(_np(x[n]) for n in NAMES[:5]), 16 ** -0.5, _np(x["init"]))
        return float((o * _np(inp["do"])).sum() + (final * _np(inp["dfinal"])).sum())

    gen = torch.Generator().manual_seed(1)
    for n in NAMES:
        d = torch.randn(inp[n].shape, generator=gen, dtype=torch.float64).cuda()
        h = 1e-5
        wide = {m: t if t is None else t.double() for m, t in inp.items()}
        want = (loss({**wide, n: wide[n] + h * d}) - loss({**wide, n: wide[n] - h * d})) / (2 * h)
        got = float((grads[n].double() * d).sum())
        scale = float(grads[n].double().norm() * d.norm())
        assert abs(got - want) < 1e-5 * scale, (n, got, want)


def test_broadcast_inputs_get_summed_gradients():
    inp = make(2, 4, 4, 80, 32, 16, "fp32", seed=16, init=False)
    import slinoss_b200 as sb
    leaf = {n: inp[n].detach().requires_grad_(True) for n in ("v", "g", "beta")}
    q1, k1 = (inp[n][:, :1].detach().requires_grad_(True) for n in ("q", "k"))
    o = sb.gated_delta_rule_b200(q1.expand(-1, 4, -1, -1), k1.expand(-1, 4, -1, -1), leaf["v"], leaf["g"], leaf["beta"])
    got = torch.autograd.grad(o, [q1, k1, leaf["v"]], inp["do"])
    # a shared key head says the same
    o2 = sb.gated_delta_rule_b200(q1, k1, leaf["v"], leaf["g"], leaf["beta"])
    want = torch.autograd.grad(o2, [q1, k1, leaf["v"]], inp["do"])
    assert torch.equal(o, o2)
    for x, y in zip(got, want):
        assert rel_err(_np(x), _np(y)) < 1e-6


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_recompute_gives_the_same_bits_and_runs_repeat(dtype):
    inp = make(2, 4, 2, 200, 64, 64, dtype, seed=17)
    a, b, c = run(inp), run(inp, residual="recompute"), run(inp)
    for x, y, z in zip([a[0], a[1], *a[2].values()], [b[0], b[1], *b[2].values()], [c[0], c[1], *c[2].values()]):
        assert torch.equal(x, y) and torch.equal(x, z)


def test_only_the_final_state_is_used():
    import slinoss_b200 as sb
    inp = make(1, 2, 2, 70, 32, 16, "fp32", seed=18)
    leaves = [inp[n].detach().requires_grad_(True) for n in NAMES]
    _, final = sb.gated_delta_rule_b200(*leaves[:5], initial_state=leaves[5], return_state=True)
    got = torch.autograd.grad(final, leaves, inp["dfinal"])
    want = odelta.backward(*(_np(x) for x in leaves[:5]), 32 ** -0.5, _np(leaves[5]), 0 * _np(inp["do"]), _np(inp["dfinal"]))
    for n, t in zip(NAMES, got):
        assert (rel_err(_np(t), want[n]) < 4e-5) if n != "q" else not t.any()


# ---- one token ---------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("b,h,hk,N,P", [(1, 1, 1, 1, 1), (1, 16, 16, 128, 64), (3, 6, 2, 40, 24), (2, 4, 4, 33, 17), (300, 4, 2, 64, 64),
                                        (2, 2, 1, 7, 256), (1, 2, 2, 16, 100)])
def test_step(dtype, b, h, hk, N, P):
    import slinoss_b200 as sb
    inp = make(b, h, hk, 1, N, P, dtype, seed=b + N)
    args = [inp[n][:, :, 0] for n in NAMES[:5]]
    o, final = sb.gated_delta_step_b200(*args, initial_state=inp["init"])
    ro, rfinal, _ = odelta.forward(*(_np(inp[n]) for n in NAMES[:5]), N ** -0.5, _np(inp["init"]))
    assert rel_err(_np(final), rfinal) < 1e-6  # sums of 128 fp32 products
    assert rel_err(_np(o), ro[:, :, 0]) < 1e-6 + (0 if dtype == "fp32" else torch.finfo(DT[dtype]).eps / 2)
    # in place, and from nothing
    state = inp["init"].clone()
    o2, same = sb.gated_delta_step_b200(*args, initial_state=state, final_state_out=state)
    assert same.data_ptr() == state.data_ptr() and torch.equal(state, final) and torch.equal(o2, o)
    oz, fz = sb.gated_delta_step_b200(*args)
    oy, fy = sb.gated_delta_step_b200(*args, initial_state=torch.zeros_like(state))
    assert torch.equal(oz, oy) and torch.equal(fz, fy)


def test_step_state_that_starts_off_an_aligned_address():
    import slinoss_b200 as sb
    inp = make(2, 2, 2, 1, 64, 32, "bf16", seed=3)
    args = [inp[n][:, :, 0] for n in NAMES[:5]]
    want = sb.gated_delta_step_b200(*args, initial_state=inp["init"])
    store = torch.zeros(inp["init"].numel() + 1, device="cuda")
    odd = store[1:].view(inp["init"].shape)
    odd.copy_(inp["init"])
    got = sb.gated_delta_step_b200(*args, initial_state=odd, final_state_out=odd)
    assert torch.equal(got[0], want[0]) and torch.equal(odd, want[1])


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_prefill_then_steps_are_one_sequence(dtype):
    import slinoss_b200 as sb
    inp = make(2, 4, 2, 75, 64, 32, dtype, seed=19)
    args = [inp[n] for n in NAMES[:5]]
    whole, final = sb.gated_delta_rule_b200(*args, initial_state=inp["init"], return_state=True)
    o, state = sb.gated_delta_rule_b200(*(x[:, :, :70] for x in args), initial_state=inp["init"], return_state=True)
    assert rel_err(_np(o), _np(whole[:, :, :70])) < 2 * tolerance(inp["q"].dtype, "o", o.dtype)
    for t in range(70, 75):
        o, state = sb.gated_delta_step_b200(*(x[:, :, t] for x in args), initial_state=state, final_state_out=state)
        assert rel_err(_np(o), _np(whole[:, :, t])) < 2 * tolerance(inp["q"].dtype, "o", o.dtype)
    assert rel_err(_np(state), _np(final)) < 1e-5


# ---- how programs call them ------------------------------------------------------------------------------------------

def test_other_stream_and_graph_replay():
    import slinoss_b200 as sb
    inp = make(1, 4, 2, 150, 64, 64, "bf16", seed=20, init=False)
    args = [inp[n] for n in NAMES[:5]]
    want = sb.gated_delta_rule_b200(*args)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sb.gated_delta_rule_b200(*args)
    side.synchronize()
    assert torch.equal(got, want)
    state = torch.zeros(1, 4, 64, 64, device="cuda")
    one = [x[:, :, 0].clone() for x in args]
    graphs, outs = [], []
    for _ in range(2):  # two graphs of the same calls, replayed one after the other
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append((sb.gated_delta_rule_b200(*args), sb.gated_delta_step_b200(*one, initial_state=state)))
        graphs.append(g)
    for t in args:
        t.mul_(0.5)
    for g in graphs:
        g.replay()
    torch.cuda.synchronize()
    want = sb.gated_delta_rule_b200(*args)
    step = sb.gated_delta_step_b200(*one, initial_state=state)
    for o, s in outs:
        assert torch.equal(o, want) and torch.equal(s[0], step[0]) and torch.equal(s[1], step[1])


def test_backward_inside_a_graph():
    import slinoss_b200 as sb
    inp = make(1, 2, 1, 100, 32, 32, "fp32", seed=21, init=False)
    static = [inp[n].detach().clone().requires_grad_(True) for n in NAMES[:5]]

    def once():
        return torch.autograd.grad(sb.gated_delta_rule_b200(*static), static, inp["do"])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        want = once()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = once()
    g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_traced_call():
    import slinoss_b200 as sb
    inp = make(1, 2, 2, 70, 32, 16, "fp32", seed=22, init=False)
    args = tuple(inp[n] for n in NAMES[:5])
    traced = torch.jit.trace(lambda *a: sb.gated_delta_rule_b200(*a, scale=0.5), args, check_trace=False)
    other = make(1, 2, 2, 70, 32, 16, "fp32", seed=23, init=False)
    other = tuple(other[n] for n in NAMES[:5])
    assert torch.equal(traced(*other), sb.gated_delta_rule_b200(*other, scale=0.5))


def test_nothing_is_written_past_a_ragged_end():
    """The outputs of a sequence that ends inside a chunk leave what lies behind them in memory."""
    from ctypes import byref

    from slinoss_b200 import _lib
    inp = make(1, 2, 2, 70, 24, 20, "bf16", seed=24, init=False)
    s = _lib.GatedDeltaShape(1, 2, 2, 70, 20, 24, _lib.SLX_BF16, _lib.SLX_BF16, _lib.SLX_BF16, 1.0)
    for name in ("q", "k", "v", "g", "beta"):
        st = inp[name].stride()
        for i in range(3):
            getattr(s, f"{name}_stride")[i] = st[i]
    lib = _lib.lib()
    n = lib.slx_gated_delta_fwd_workspace_bytes(byref(s))
    ws = torch.empty(n, device="cuda", dtype=torch.uint8)
    o = torch.full((2 * 70 * 20 + 4096,), 7.0, device="cuda", dtype=torch.bfloat16)
    final = torch.full((2 * 20 * 24 + 4096,), 7.0, device="cuda")
    _lib.check(lib.slx_gated_delta_fwd(byref(s), *(inp[x].data_ptr() for x in NAMES[:5]), None, 0, o.data_ptr(),
                                       final.data_ptr(), None, ws.data_ptr(), n, _lib.stream_ptr(o.device)), "forward")
    torch.cuda.synchronize()
    assert (o[2 * 70 * 20:] == 7).all() and (final[2 * 20 * 24:] == 7).all()
    import slinoss_b200 as sb
    assert torch.equal(o[:2 * 70 * 20].view(1, 2, 70, 20), sb.gated_delta_rule_b200(*(inp[x] for x in NAMES[:5]), scale=1.0))


# ---- what is refused or empty --------------------------------------------------------------------------------------------

def test_refusals():
    import slinoss_b200 as sb
    x = lambda *s, dt=torch.float32: torch.zeros(*s, device="cuda", dtype=dt)
    ok = dict(q=x(1, 2, 8, 16), k=x(1, 2, 8, 16), v=x(1, 4, 8, 16), g=x(1, 4, 8), beta=x(1, 4, 8))
    call = lambda **kw: sb.gated_delta_rule_b200(**{**ok, **kw})
    assert call().shape == (1, 4, 8, 16)
    for kw in (dict(k=x(1, 2, 8, 8)), dict(q=x(1, 3, 8, 16), k=x(1, 3, 8, 16)), dict(g=x(1, 2, 8)), dict(beta=x(1, 4, 7)),
               dict(v=x(1, 4, 9, 16)), dict(initial_state=x(1, 4, 16, 8)), dict(q=x(1, 2, 8, 130), k=x(1, 2, 8, 130)),
               dict(v=x(1, 4, 8, 257)), dict(residual="none"), dict(q=ok["q"].cpu())):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(v=x(1, 4, 8, 16, dt=torch.bfloat16)), dict(g=x(1, 4, 8, dt=torch.float64)),
               dict(q=x(1, 2, 8, 16, dt=torch.float64), k=x(1, 2, 8, 16, dt=torch.float64), v=x(1, 4, 8, 16, dt=torch.float64))):
        with pytest.raises(TypeError):
            call(**kw)
    step = dict(q=x(1, 2, 16), k=x(1, 2, 16), v=x(1, 4, 16), g=x(1, 4), beta=x(1, 4))
    run_step = lambda **kw: sb.gated_delta_step_b200(**{**step, **kw})
    store = x(4 * 16 * 16 + 4)
    for kw in (dict(v=x(1, 3, 16)), dict(final_state_out=x(1, 4, 16, 8)), dict(final_state_out=x(1, 4, 16, 32)[..., ::2]),
               dict(initial_state=store[:-4].view(1, 4, 16, 16), final_state_out=store[4:].view(1, 4, 16, 16))):
        with pytest.raises(ValueError):
            run_step(**kw)
    with pytest.raises(TypeError):
        run_step(final_state_out=x(1, 4, 16, 16, dt=torch.float16))


def test_empty_and_converted_arguments():
    import slinoss_b200 as sb
    inp = make(2, 2, 2, 9, 16, 8, "fp32", seed=25)
    empty = [inp[n][:, :, :0] for n in NAMES[:5]]
    o, final = sb.gated_delta_rule_b200(*empty, initial_state=inp["init"], return_state=True)
    assert o.shape == (2, 2, 0, 8) and torch.equal(final, inp["init"]) and final.data_ptr() != inp["init"].data_ptr()
    o, final = sb.gated_delta_rule_b200(*empty, return_state=True)
    assert final.shape == (2, 2, 8, 16) and not final.any()
    want = sb.gated_delta_rule_b200(*(inp[n] for n in NAMES[:5]))
    odd = [inp[n].transpose(-1, -2).contiguous().transpose(-1, -2) if n in "qkv" else inp[n] for n in NAMES[:5]]
    assert torch.equal(sb.gated_delta_rule_b200(*odd), want)
    init = inp["init"].double()
    a = sb.gated_delta_rule_b200(*(inp[n] for n in NAMES[:5]), initial_state=init)
    assert torch.equal(a, sb.gated_delta_rule_b200(*(inp[n] for n in NAMES[:5]), initial_state=inp["init"]))

"""top_p borders that fall between the steps by which the sampling kernel narrows them down, against float64.

The kernel's masses are integers of 2^-44 of the largest, so a sum of V of them is off by at most V halves of that, and so are
the whole that top_p refers to and the mass that the draw goes through: a token may be drawn whose place in the ranking lies
within e = V * 2^-44 of top_p's border (two such sums), and whose place in the draw within 3 e of u times the whole (the
running sum, the whole, and what the tokens within e of the border add to both).  A heavier token that ends within e of the
border stays or goes as a whole: the draw may be that of either.
"""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def far_off(row, temperature, top_p, u, got):
    """How far each drawn token lies outside of what float64 allows it, in masses of the largest (0: inside)."""
    x = row.double().cpu().numpy()
    mass = np.exp((x - x.max()) / temperature)
    order = np.argsort(-x, kind="stable")
    upto = np.cumsum(mass[order])
    rank = np.empty_like(order)
    rank[order] = np.arange(len(x))
    off, e = [], len(x) * 2.0 ** -44
    for p, v, token in zip(top_p, u, got):
        want = p * upto[-1]
        count = lambda border: min(len(x), int(np.searchsorted(upto, border)) + 1)  # the first so many reach it
        here = []
        for n in {count(want - e), count(want), count(want + e)}:
            kept = np.zeros_like(mass)
            kept[order[:n]] = mass[order[:n]]
            run = np.cumsum(kept)
            target = v * run[-1]
            here.append(max(0.0, run[token] - kept[token] - target, target - run[token]))
        off.append(max(min(here), upto[rank[token]] - mass[token] - want))  # (the latter: ranked behind the border)
    return np.array(off)


def compare(row, temperature, top_p, u):
    import slinoss_b200 as sb
    n = len(top_p)
    got = sb.sample_b200(row.expand(n, -1), torch.as_tensor(u, device="cuda", dtype=torch.float64), temperature=temperature,
                         top_p=torch.as_tensor(top_p, device="cuda", dtype=torch.float32)).cpu().numpy()
    off = far_off(row, temperature, top_p, u, got)
    wrong = off > 3 * row.numel() * 2.0 ** -44
    assert not wrong.any(), (int(wrong.sum()), n, top_p[wrong][:4], off[wrong][:4])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("V,temperature", [(131072, 2.0), (50021, 4.0), (150001, 1.0)])
def test_borders_at_the_edges_of_masses_sixteenth_powers(dtype, V, temperature):
    """Whole bins of thousands of tokens above the border: rounded sums say one bin, exact ones its neighbour."""
    gen = torch.Generator().manual_seed(0)
    row = torch.randn(V, generator=gen).to(dtype).cuda()
    x = row.double().cpu().numpy()
    mass = np.exp((x - x.max()) / temperature)
    step = -np.log2(mass) * 16
    edges = np.arange(1, 320)
    share = np.array([mass[step < e].sum() for e in edges]) / mass.sum()
    some = [s for e, s in zip(edges, share) if np.count_nonzero((step >= e - 1) & (step < e + 1)) > 4096 and 0.01 < s < 0.999]
    top_p = []
    for s in some:
        p = np.float32(s)
        top_p += [float(p + k * np.spacing(p)) for k in range(-3, 4)]
    top_p = np.array(top_p)
    assert len(top_p) >= 50
    compare(row, temperature, top_p, torch.rand(len(top_p), generator=gen, dtype=torch.float64).numpy())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("V,low,high", [(131072, 14.5, 24.0), (60000, 15.0, 19.0), (262144, 14.5, 29.0)])
def test_borders_in_the_bin_of_small_masses(dtype, V, low, high):
    """One token above tens of thousands whose masses lie below 2^-20: the bin that holds the border has them all."""
    gen = torch.Generator().manual_seed(1)
    row = -(low + (high - low) * torch.rand(V, generator=gen))
    row[V // 3] = 0.0
    row = row.to(dtype).cuda()
    rest = float(torch.exp(row.double()).sum()) - 1.0
    # borders all over what lies below the largest: evenly in mass, and in its logarithm
    part = torch.cat([torch.rand(80, generator=gen, dtype=torch.float64), 2.0 ** -(14 * torch.rand(80, generator=gen, dtype=torch.float64))])
    top_p = ((1.0 + rest * (1.0 - part)) / (1.0 + rest)).float().clamp(max=1 - 2.0 ** -24).double().numpy()
    u = 1.0 - rest * torch.rand(160, generator=gen, dtype=torch.float64).numpy()
    compare(row, 1.0, top_p, u)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_borders_among_shared_values_far_inside_a_bin(dtype):
    """Tens of thousands of tokens a value, 2^-13 below the first of their bin: the same rounding would be taken for all."""
    gen = torch.Generator().manual_seed(3)
    V = 262144
    row = -22.0 - 0.125 * torch.randint(0, 19, (V,), generator=gen)
    row[torch.randint(0, V, (50,), generator=gen)] = -14.0
    row[V - 1] = 0.0
    row = row.to(dtype).cuda()
    whole = float(torch.exp(row.double()).sum())
    far = float(torch.exp(row.double()[row < -20]).sum()) / whole
    top_p = (1.0 - far * torch.rand(100, generator=gen, dtype=torch.float64)).float().clamp(max=1 - 2.0 ** -24).double().numpy()
    # (of the tokens that share the border's value the first ones stay: draws among the low indices see how many)
    compare(row, 1.0, top_p, 0.2 * far * torch.rand(100, generator=gen, dtype=torch.float64).numpy())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_borders_among_equal_masses_in_wide_bins(dtype):
    """High temperatures put a row into few bins, each divided by the keys of its logits; many tokens share a value."""
    gen = torch.Generator().manual_seed(2)
    row = (torch.randn(100003, generator=gen) * 4).round().div(4).to(dtype).cuda()
    top_p = (0.02 + 0.97 * torch.rand(120, generator=gen)).double().numpy()
    compare(row, 30.0, top_p, torch.rand(120, generator=gen, dtype=torch.float64).numpy())
    fine = torch.randn(100003, generator=gen).to(dtype).cuda()
    compare(fine, 30.0, top_p, torch.rand(120, generator=gen, dtype=torch.float64).numpy())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("finite,k", [(5000, 6000), (9000, 9999), (300, 700), (6000, 6001)])
def test_top_k_beyond_the_tokens_that_a_mask_leaves(dtype, finite, k):
    """All of them stay, the small masses behind the first one too."""
    import slinoss_b200 as sb
    gen = torch.Generator().manual_seed(4)
    V = 10000
    row = torch.full((V,), -torch.inf)
    some = torch.randperm(V - 1, generator=gen)[:finite]
    row[some] = -18.0 - 2.0 * torch.rand(finite, generator=gen)
    row[V - 1] = 0.0
    row = row.to(dtype).cuda()
    tail = float(torch.exp(row.double()).sum()) - 1.0
    u = (tail * torch.rand(60, generator=gen, dtype=torch.float64)).numpy()
    for p in (1.0, float(np.float32(1 - 0.3 * tail))):
        got = sb.sample_b200(row.expand(60, -1), torch.as_tensor(u, device="cuda"), top_k=k, top_p=p).cpu().numpy()
        assert (far_off(row, 1.0, np.full(60, p), u, got) <= 3 * V * 2.0 ** -44).all()

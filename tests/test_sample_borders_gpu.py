"""top_p borders that fall between the steps by which the sampling kernel narrows them down, against float64.

The kernel's masses are integers of 2^-44 of the largest, so a sum of V of them is off by at most V halves of that, and so are
the whole that top_p refers to and the mass that the draw goes through: a token may be drawn whose place in the ranking lies
within e = V * 2^-44 of top_p's border (two such sums), and whose place in the draw within 3 e of u times the whole (the
running sum, the whole, and what the border's tokens add to both).
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
    off = []
    for p, v, token in zip(top_p, u, got):
        want = p * upto[-1]
        n = min(len(x), int(np.searchsorted(upto, want)) + 1)  # the first n whose mass reaches it
        kept = np.zeros_like(mass)
        kept[order[:n]] = mass[order[:n]]
        run = np.cumsum(kept)
        target = v * run[-1]
        beyond = upto[rank[token]] - mass[token] - want  # positive: ranked behind the border
        off.append(max(0.0, beyond, run[token] - kept[token] - target, target - run[token]))
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

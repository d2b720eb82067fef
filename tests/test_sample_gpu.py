"""Token sampling on the GPU against float64, token by token equal."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import sample as osample

pytestmark = pytest.mark.gpu

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def check(logits, u, temperature, top_k, top_p, min_p):
    """Equal tokens, but where the float64 running mass meets the draw's border more closely than the kernel's integers tell
    apart (V halves of 2^-44 against a mass of at least one)."""
    import slinoss_b200 as sb
    got = sb.sample_b200(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p).cpu().numpy()
    assert got.dtype == np.int64 and got.shape == (logits.shape[0],)
    at = lambda x, i: x[i].item() if isinstance(x, torch.Tensor) else x
    rows = logits.detach().double().cpu().numpy()
    f32 = lambda x: float(np.float32(x))
    for i, row in enumerate(rows):
        want, margin = osample.draw(row, at(u, i), f32(at(temperature, i)), int(at(top_k, i)), f32(at(top_p, i)), f32(at(min_p, i)))
        assert got[i] == want or margin < logits.shape[1] * 2.0 ** -44, (i, got[i], want, margin)
    return got


def rows(b, V, dtype, seed=0, spread=3.0):
    gen = torch.Generator().manual_seed(seed)
    return ((spread * torch.randn(b, V, generator=gen)).to(DT[dtype]).cuda(), torch.rand(b, generator=gen).cuda())


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
@pytest.mark.parametrize("V", [1, 2, 31, 256, 1000, 4099, 50021])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (1, 1.0, 0.0), (50, 1.0, 0.0), (0, 0.9, 0.0), (0, 1.0, 0.05), (40, 0.8, 0.02),
                                   (0, 0.999, 0.0), (300, 0.99, 0.0)])
def test_filters(dtype, V, k, p, m):
    logits, u = rows(6, V, dtype, seed=V + k)
    check(logits, u, 0.8, k, p, m)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_settings_of_each_row(dtype):
    b = 64
    logits, u = rows(b, 3001, dtype, seed=1)
    gen = torch.Generator().manual_seed(2)
    r = lambda: torch.rand(b, generator=gen)
    temperature, top_p, min_p = (0.2 + 2 * r()).cuda(), (0.3 + 0.9 * r()).cuda(), (0.2 * (r() - 0.5)).clamp(min=0).cuda()
    top_k = torch.randint(-2, 200, (b,), generator=gen).cuda()
    got = check(logits, u, temperature, top_k, top_p, min_p)
    assert np.array_equal(check(logits, u.double(), temperature, top_k.int(), top_p, min_p), got)
    # rows do not see one another, nor the stride they lie at
    wide = torch.full((b, 4000), 100.0, device="cuda", dtype=logits.dtype)
    wide[:, 7:3008] = logits
    pick = [3, 60, 17]
    assert np.array_equal(check(wide[pick][:, 7:3008], u[pick], temperature[pick], top_k[pick], top_p[pick], min_p[pick]), got[pick])


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_ties_go_by_index(dtype):
    logits = torch.zeros(8, 500, dtype=DT[dtype], device="cuda")
    logits[4:, ::3] = 1.0
    u = torch.linspace(0, 0.999, 8).cuda()
    for k, p, m in [(0, 1.0, 0.0), (7, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.99), (100, 0.31, 0.0), (0, 0.75, 0.0), (200, 0.9, 0.0)]:
        got = check(logits, u, 1.0, k, p, m)
        if k:
            assert (got[:4] < k).all()


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("b,V,spread", [(256, 20000, 1.0), (256, 9000, 2.0), (40, 131072, 3.0), (300, 3000, 0.2)])
def test_wide_nuclei_draw_exactly(dtype, b, V, spread):
    """Thousands of tokens stay: an error of 1e-6 in the whole mass would give one row in a hundred its neighbour."""
    logits, u = rows(b, V, dtype, seed=V, spread=spread)
    gen = torch.Generator().manual_seed(9)
    top_p = (0.9 + 0.099 * torch.rand(b, generator=gen)).cuda()
    check(logits, u, 1.1, 0, top_p, 0.0)
    check(logits, u, 0.9, V // 2, top_p, 0.001)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
@pytest.mark.parametrize("gap,below", [(12.0, 1e-3), (16.0, 1e-4), (25.0, 2.0 ** -23)])
def test_borders_far_below_the_largest(dtype, gap, below):
    """One token far above tens of thousands, of which a filter keeps some: steps, bins and small masses at their ends."""
    V = 50021
    logits, _ = rows(8, V, dtype, seed=7, spread=1.0)
    logits[:, 17] = gap + 4.5
    u = 1.0 - below * torch.rand(8, generator=torch.Generator().manual_seed(8), dtype=torch.float64).cuda()
    for k, p in ((0, 1.0 - below), (1000, 1.0), (1000, 1.0 - below), (30000, 1.0 - below), (50, 1.0)):
        check(logits, u, 1.0, k, p, 0.0)
        check(logits, u, 0.4, k, p, 0.0)


@pytest.mark.parametrize("k,p", [(700, 1.0), (2500, 0.9), (0, 0.3), (3900, 0.95)])
def test_few_values_shared_by_many_tokens(k, p):
    gen = torch.Generator().manual_seed(11)
    values = torch.tensor([2.0, 1.0, 0.5, -40.0])
    logits = values[torch.randint(0, 4, (16, 6000), generator=gen)].to(torch.bfloat16).cuda()
    logits[8:] += (0.01 * torch.randn(8, 6000, generator=gen)).bfloat16().cuda()
    check(logits, torch.rand(16, generator=gen).cuda(), 0.7, k, p, 0.0)


@pytest.mark.parametrize("dtype", ["fp32", "bf16"])
def test_borders_between_tokens_far_apart(dtype):
    """top_p a millionth above what some of the tokens hold: the next one counts, however far below it lies."""
    b = 400
    gen = torch.Generator().manual_seed(12)
    logits = (4.0 * torch.randn(b, 10, generator=gen)).to(DT[dtype])
    mass = torch.exp(logits.double() - logits.double().amax(-1, keepdim=True)).sort(-1, descending=True)[0]
    share = mass.cumsum(-1) / mass.sum(-1, keepdim=True)
    some = torch.randint(0, 5, (b,), generator=gen)
    top_p = share.gather(1, some[:, None])[:, 0] * torch.where(torch.arange(b) % 2 == 0, 1 + 1e-6, 1 - 1e-6)
    top_p = top_p.float().clamp(max=1 - 2.0 ** -23)
    check(logits.cuda(), (1.0 - 1e-9 * torch.rand(b, generator=gen, dtype=torch.float64)).cuda(), 1.0, 0, top_p.cuda(), 0.0)
    check(logits.cuda(), torch.rand(b, generator=gen).cuda(), 1.0, 0, top_p.cuda(), 0.0)


def test_signed_zeros_are_one_value():
    logits = torch.tensor([[-0.0, 0.0, -0.0, -1.0]], device="cuda").repeat(3, 1)
    got = check(logits, torch.tensor([0.0, 0.4, 0.9]).cuda(), 1.0, 2, 1.0, 0.0)
    assert got.tolist() == [0, 0, 1]


@pytest.mark.parametrize("dtype", ["fp32", "fp16", "bf16"])
def test_masked_infinite_and_nan_logits(dtype):
    inf = math.inf
    logits, u = rows(10, 700, dtype, seed=3)
    low = torch.finfo(DT[dtype]).min
    logits[0] = -inf
    logits[1] = torch.nan
    logits[2] = -inf
    logits[2, 123] = -3.0
    logits[3, ::2] = -inf
    logits[4, ::2] = torch.nan
    logits[5, [5, 600]] = inf
    logits[6] = low
    logits[7, 100:] = low
    logits[8] = -inf
    logits[8, 300:303] = low
    u[5] = 0.7
    for k, p, m in [(0, 1.0, 0.0), (20, 0.9, 0.01), (1, 1.0, 0.0), (0, 0.6, 0.0), (600, 1.0, 0.0)]:
        got = check(logits, u, 0.7, k, p, m)
        assert got[0] == -1 and got[1] == -1 and got[2] == 123
        assert got[3] % 2 == 1 and got[4] % 2 == 1
        assert got[5] in (5, 600) and 300 <= got[8] < 303 and got[7] < 100
    assert check(logits, u, 1.0, 0, 1.0, 0.0)[5] == 600


def test_greedy_forms_and_borders_of_u():
    logits, u = rows(4, 1000, "bf16", seed=4)
    best = logits.float().argmax(-1)
    first = torch.tensor([(row == row.max()).nonzero()[0, 0].item() for row in logits.float().cpu()])
    import slinoss_b200 as sb
    for kw in (dict(temperature=0.0), dict(top_k=1), dict(top_p=0.0), dict(min_p=1.0, top_k=1), dict(top_p=1e-30)):
        assert torch.equal(sb.sample_b200(logits, u, **kw).cpu(), first), kw
    assert (logits.float().gather(1, best[:, None]) == logits.float().gather(1, first[:, None].cuda())).all()
    flat = torch.zeros(5, 8, device="cuda")
    edge = torch.tensor([0.0, 0.125, 1.0, 2.0, -1.0]).cuda()
    assert sb.sample_b200(flat, edge).tolist() == [0, 1, 7, 7, 0]


def test_draws_follow_the_masses():
    """Even u walk through the distribution: each token comes as often as its mass says, to within one draw."""
    import slinoss_b200 as sb
    gen = torch.Generator().manual_seed(6)
    row = torch.randn(40, generator=gen)
    n = 4096
    u = ((torch.arange(n, dtype=torch.float64) + 0.5) / n).cuda()
    got = torch.bincount(sb.sample_b200(row.cuda().expand(n, -1), u, temperature=0.9).cpu(), minlength=40).double()
    want = torch.softmax(row.double() / np.float32(0.9), -1) * n
    assert (got - want).abs().max() <= 1.0


def test_large_vocabulary_and_the_same_token_whatever_the_batch():
    import slinoss_b200 as sb
    logits, u = rows(3, 262144, "fp32", seed=7)
    got = check(logits, u, 1.0, 0, 0.95, 0.0)
    many = sb.sample_b200(logits.repeat(50, 1), u.repeat(50), top_p=0.95).cpu().numpy().reshape(50, 3)
    assert (many == got).all()


def test_streams_and_graphs():
    import slinoss_b200 as sb
    logits, u = rows(5, 2000, "bf16", seed=8)
    want = sb.sample_b200(logits, u, top_k=40, top_p=0.9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = sb.sample_b200(logits, u, top_k=40, top_p=0.9)
    side.synchronize()
    assert torch.equal(got, want)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = sb.sample_b200(logits, u, top_k=40, top_p=0.9)
    logits.copy_(logits.flip(-1))
    u.mul_(0.5)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, sb.sample_b200(logits, u, top_k=40, top_p=0.9))


def test_refusals():
    import slinoss_b200 as sb
    logits, u = rows(2, 10, "fp32")
    for kw in (dict(temperature=-1.0), dict(temperature=math.nan), dict(top_p=1.5), dict(top_p=-0.1), dict(min_p=2.0),
               dict(top_k=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(temperature=torch.ones(1, device="cuda"))):
        with pytest.raises(ValueError):
            sb.sample_b200(logits, u, **kw)
    with pytest.raises(ValueError):
        sb.sample_b200(logits, u[:1])
    with pytest.raises(ValueError):
        sb.sample_b200(logits[0], u)
    with pytest.raises(ValueError):
        sb.sample_b200(logits.cpu(), u.cpu())
    with pytest.raises(ValueError):
        sb.sample_b200(torch.zeros(1, 262145, device="cuda"), u[:1])
    with pytest.raises(TypeError):
        sb.sample_b200(logits, u.half())
    with pytest.raises(TypeError):
        sb.sample_b200(logits.double(), u)
    with pytest.raises(TypeError):
        sb.sample_b200(logits, u, top_k=torch.ones(2, device="cuda"))
    assert sb.sample_b200(logits[:0], u[:0]).shape == (0,)
    # other dtypes of settings, and logits whose tokens are not dense
    t = sb.sample_b200(logits, u, temperature=torch.ones(2, device="cuda", dtype=torch.float64))
    assert torch.equal(t, sb.sample_b200(logits, u))
    assert torch.equal(sb.sample_b200(logits.t().contiguous().t(), u), t)

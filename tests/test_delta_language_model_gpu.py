"""A small language model of the gated delta rule's operators, as a program uses them together: the causal convolution, the
delta rule and the gate in training; prefill, one-token steps and sampling in generation, eager and as a captured graph.

Tolerances, in fp32: an operator is off by at most 1e-5 of its result's norm (each has tests of its own for that).  Six stand
in a row from the tokens to the logits, and six more on the way back: 6e-5 and 1.2e-4 where errors only add up, doubled for
the division by the keys' norms and the softmax between them."""

from __future__ import annotations

import numpy as np
import pytest
import torch
import torch.nn.functional as F

from oracle import sample as osample
from util import rel_err

pytestmark = pytest.mark.gpu

V, H, HK, P, N = 97, 4, 2, 16, 24
D, C = H * P, 2 * HK * N + H * P  # width; channels that the convolution takes (q, k, v)
FORWARD, BACKWARD = 1.2e-4, 2.4e-4


def weights():
    gen = torch.Generator().manual_seed(5)
    rand = lambda *s: torch.randn(*s, generator=gen)
    return dict(emb=rand(V, D), inp=rand(D, C + D + 2 * H) * D ** -0.5, conv=0.4 * rand(C, 4), bias=0.1 * rand(C),
                skip=rand(D), head=rand(D, V) * 3 * D ** -0.5)


def split(z):
    """Of the projection's output: what goes into the convolution, the gate, g and beta."""
    return (z[..., :C], z[..., C:C + D], -F.softplus(z[..., C + D:C + D + H]), torch.sigmoid(z[..., C + D + H:]))


def heads(x):
    q, k, v = x[..., :HK * N], x[..., HK * N:2 * HK * N], x[..., 2 * HK * N:]
    q, k, v = q.unflatten(-1, (HK, N)), k.unflatten(-1, (HK, N)), v.unflatten(-1, (H, P))
    return F.normalize(q, dim=-1), F.normalize(k, dim=-1), v


def whole(w, tokens, states=False):
    """Logits (b, T, V) of whole sequences by the operators, and the states behind them."""
    import slinoss_b200 as sb
    x, gate, g, beta = split(w["emb"][tokens] @ w["inp"])
    x, conv = sb.cconv1d_b200(x, w["conv"], w["bias"], activation="silu")
    q, k, v = (t.transpose(1, 2) for t in heads(x))
    o = sb.gated_delta_rule_b200(q, k, v, g.transpose(1, 2), beta.transpose(1, 2), return_state=states)
    o, state = o if states else (o, None)
    logits = sb.gate_skip_b200(o, v.contiguous(), gate, w["skip"]) @ w["head"]
    return (logits, conv, state) if states else logits


def one(w, token, conv, state):
    """Logits (b, V) of the next token; conv and state are updated in place."""
    import slinoss_b200 as sb
    x, gate, g, beta = split(w["emb"][token] @ w["inp"])
    x, _ = sb.cconv1d_update_b200(x, w["conv"], w["bias"], conv, activation="silu", inplace=True)
    q, k, v = heads(x)
    o, _ = sb.gated_delta_step_b200(q, k, v, g, beta, initial_state=state, final_state_out=state)
    return sb.gate_skip_b200(o.unsqueeze(2), v.unsqueeze(2).contiguous(), gate.unsqueeze(1), w["skip"])[:, 0] @ w["head"]


def plain(w, tokens):
    """The same logits by elementary operations, token by token."""
    x, gate, g, beta = split(w["emb"][tokens] @ w["inp"])
    T = x.shape[1]
    past = F.pad(x, (0, 0, 3, 0))
    x = F.silu(sum(past[:, i:i + T] * w["conv"][:, i] for i in range(4)) + w["bias"])
    q, k, v = heads(x)
    q, k = (t.repeat_interleave(H // HK, 2) for t in (q, k))
    S = x.new_zeros(x.shape[0], H, P, N)
    out = []
    for t in range(T):
        S = S * g[:, t, :, None, None].exp()
        y = v[:, t] - (S @ k[:, t, :, :, None])[..., 0]
        S = S + (beta[:, t, :, None] * y)[..., None] * k[:, t, :, None]
        out.append(N ** -0.5 * (S @ q[:, t, :, :, None])[..., 0])
    o = torch.stack(out, 1) + v * w["skip"].view(H, P)
    return (o.flatten(2) * F.silu(gate)) @ w["head"]


def _np(t):
    return t.detach().double().cpu().numpy()


@pytest.mark.parametrize("T", [1, 65, 150])
def test_training_step(T):
    tokens = torch.randint(0, V, (3, T + 1), generator=torch.Generator().manual_seed(T))
    want_w = {n: t.double().requires_grad_(True) for n, t in weights().items()}
    want = plain(want_w, tokens[:, :-1])
    F.cross_entropy(want.flatten(0, 1), tokens[:, 1:].flatten()).backward()
    w = {n: t.cuda().requires_grad_(True) for n, t in weights().items()}
    got = whole(w, tokens[:, :-1].cuda())
    F.cross_entropy(got.flatten(0, 1), tokens[:, 1:].flatten().cuda()).backward()
    errs = {"logits": rel_err(_np(got), _np(want))}
    errs.update((n, rel_err(_np(w[n].grad), _np(want_w[n].grad))) for n in w)
    print({n: f"{e:.2e}" for n, e in errs.items()})
    assert errs.pop("logits") <= FORWARD
    for n, e in errs.items():
        assert e <= BACKWARD, (n, e)


@pytest.mark.parametrize("length", [1, 70])
def test_generation_eager_and_captured(length):
    import slinoss_b200 as sb
    gen = torch.Generator().manual_seed(length)
    b, steps = 3, 12
    w = {n: t.cuda() for n, t in weights().items()}
    prompt = torch.randint(0, V, (b, length), generator=gen).cuda()
    u = torch.rand(steps + 1, b, generator=gen, dtype=torch.float64).cuda()
    # one setting of each row: the whole distribution, a nucleus of few, the largest
    t, k, p = (torch.tensor(x, device="cuda") for x in ([1.0, 0.8, 0.0], [0, 20, 0], [1.0, 0.9, 1.0]))
    draw = lambda logits, u: sb.sample_b200(logits, u, temperature=t, top_k=k, top_p=p)

    def begin():
        logits, conv, state = whole(w, prompt, states=True)
        return logits[:, -1], conv.contiguous(), state

    logits, conv, state = begin()
    seen, tokens = [logits], [draw(logits, u[0])]
    for i in range(steps):
        seen.append(one(w, tokens[-1], conv, state))
        tokens.append(draw(seen[-1], u[i + 1]))
    everything = torch.cat([prompt, torch.stack(tokens, 1)], 1)
    want = plain({n: x.double().cpu() for n, x in w.items()}, everything[:, :-1].cpu())[:, length - 1:]
    assert rel_err(_np(torch.stack(seen, 1)), _np(want)) <= FORWARD
    for i, (logits, token) in enumerate(zip(seen, tokens)):
        for row in range(b):
            x = _np(logits[row])
            assert int(token[row]) == osample.draw(x, float(u[i, row]), float(t[row]), int(k[row]), float(p[row]))[0]

    logits, conv, state = begin()
    token, chance = draw(logits, u[0]), u[0].clone()
    saved = [x.clone() for x in (token, conv, state)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (a first call outside of the capture, as capturing programs do)
        token.copy_(draw(one(w, token, conv, state), chance))
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip((token, conv, state), saved):
        x.copy_(y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        token.copy_(draw(one(w, token, conv, state), chance))
    got = [token.clone()]
    for i in range(steps):
        chance.copy_(u[i + 1])
        graph.replay()
        got.append(token.clone())
    assert np.array_equal(_np(torch.stack(got)), _np(torch.stack(tokens)))

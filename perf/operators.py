"""Performance cases of the gated delta rule and of token sampling, through the framework's public entry points.

Three operators, in the sizes of this repository's configurations and tests or in generic ones:

* ``delta``   the chunked gated delta rule (``gated_delta_rule_b200``): training (forward + all gradients) or prefill
              (states in and out);
* ``step``    one token of the same recurrence on carried states (``gated_delta_step_b200``);
* ``sample``  tokens from logits and given random numbers (``sample_b200``).

The recurrence of a head, with state ``S (P, N)``, ``a_t = exp(g_t)``:

    d_t = beta_t (v_t - a_t S_{t-1} k_t),   S_t = a_t S_{t-1} + d_t k_t^T,   o_t = scale S_t q_t

``own`` chooses between the plain form (elementary torch operations in 32 bits) and the framework's kernels.
"""

from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CHUNK = 64


def _delta(name, dtype, b, h, T, N, *, hk=None, P=64, train=True, state=False, rows=False):
    # rows: q, k, v are column slices of one token-major projection row, not head-major tensors
    return dict(name=name, kind="delta", dtype=dtype, b=b, h=h, hk=h if hk is None else hk, T=T, N=N, P=P, train=train,
                state=state, rows=rows)


def _step(name, dtype, b, h, N, *, hk=None, P=64):
    return dict(name=name, kind="step", dtype=dtype, b=b, h=h, hk=h if hk is None else hk, N=N, P=P)


def _sample(name, dtype, b, V, *, k=0, p=1.0, minp=0.0):
    return dict(name=name, kind="sample", dtype=dtype, b=b, V=V, k=k, p=p, minp=minp)


def listed():
    return [
        # one layer of the language-model training configuration: 16 heads, state width 128, 16 sequences of 4096 tokens
        _delta("delta_train_lm", "bf16", 16, 16, 4096, 128, rows=True),
        # one long document: few sequences, many chunks
        _delta("delta_train_long", "bf16", 1, 32, 32768, 128),
        # a training segment that carries state in and out; ragged, key heads shared by three value heads each
        _delta("delta_train_segment", "fp16", 3, 12, 1537, 64, hk=4, state=True, rows=True),
        # a small full-precision model on short sequences: the smallest configured heads
        _delta("delta_train_short_fp32", "fp32", 2, 4, 77, 16, P=32, state=True),
        # prompt of one request, odd length, continued from a carried state
        _delta("delta_prefill", "bf16", 1, 16, 4093, 128, train=False, state=True),
        # serving, the largest configured decode batch
        _step("step_batch", "bf16", 256, 32, 128),
        # serving a few requests of a model with shared key heads
        _step("step_shared", "fp16", 24, 12, 64, hk=4),
        # one request: the smallest call
        _step("step_one", "bf16", 1, 16, 128),
        # a byte vocabulary, the plain temperature draw of a text demo, many streams at once
        _sample("sample_bytes", "bf16", 256, 256),
        # one request, a word-piece vocabulary of odd size, the usual chat settings
        _sample("sample_one", "bf16", 1, 50021, k=50, p=0.9),
        # a serving batch with nucleus sampling over a large vocabulary
        _sample("sample_nucleus", "fp32", 64, 131072, p=0.95),
        # a large batch in which each request has settings of its own, all filters at once
        _sample("sample_mixed", "bf16", 192, 150001, k=1000, p=0.9, minp=0.02),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["delta", "delta", "delta", "step", "sample", "sample"])
    dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "delta":
        hk, share = rng.choice([1, 2, 4, 6, 8]), rng.choice([1, 1, 2, 3])
        T = _spread(rng, 1, 8192)
        b = max(1, min(_spread(rng, 1, 16), 131072 // (T * hk * share)))
        train = rng.random() < 0.6
        return dict(kind="delta", dtype=dtype, b=b, h=hk * share, hk=hk, T=T, N=rng.choice([16, 32, 40, 64, 96, 128, 128]),
                    P=rng.choice([24, 32, 64, 64, 96, 128]), train=train, state=not train or rng.random() < 0.4,
                    rows=rng.random() < 0.5)
    if kind == "step":
        hk, share = rng.choice([1, 2, 4, 8, 16]), rng.choice([1, 1, 2, 3])
        return dict(kind="step", dtype=dtype, b=max(1, min(_spread(rng, 1, 256), 4096 // (hk * share))), h=hk * share, hk=hk,
                    N=rng.choice([16, 40, 64, 96, 128]), P=rng.choice([24, 32, 64, 128]))
    V = _spread(rng, 100, 160000)
    return dict(kind="sample", dtype=dtype, b=max(1, min(_spread(rng, 1, 256), 16000000 // V)), V=V,
                k=rng.choice([0, 0, 1, 20, 50, 1000]), p=rng.choice([1.0, 0.5, 0.9, 0.95, 0.99]),
                minp=rng.choice([0.0, 0.0, 0.02, 0.1]))


# --------------------------------------------------------------------------------------------------------------------
# what a program has in hand before the call
# --------------------------------------------------------------------------------------------------------------------

def _inputs(case, gen):
    b, h, hk, N, P = (case[x] for x in ("b", "h", "hk", "N", "P"))
    dt, T = DTYPES[case["dtype"]], case.get("T")
    n = (T,) if T is not None else ()
    rand = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    unit = lambda x: x / x.norm(dim=-1, keepdim=True)  # queries and keys come normalised
    if case.get("rows"):
        row = torch.cat([unit(rand(b, T, 2 * hk, N)).flatten(2), rand(b, T, h * P)], -1).to(dt)
        q, k = (row[..., i * hk * N:(i + 1) * hk * N].unflatten(-1, (hk, N)).transpose(1, 2) for i in (0, 1))
        v = row[..., 2 * hk * N:].unflatten(-1, (h, P)).transpose(1, 2)
    else:
        q, k = (unit(rand(b, hk, *n, N)).to(dt) for _ in (0, 1))
        v = rand(b, h, *n, P).to(dt)
    # gates as trained layers have them: from nearly closed to nearly always open, a write strength in (0, 1)
    speed = torch.exp(torch.empty(h, device="cuda").uniform_(math.log(1e-3), math.log(0.5), generator=gen))
    g = (-speed.view(1, h, *(1 for _ in n)) * torch.nn.functional.softplus(rand(b, h, *n))).to(dt)
    beta = torch.sigmoid(rand(b, h, *n)).to(dt)
    return dict(q=q, k=k, v=v, g=g, beta=beta)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    dev = torch.device("cuda")
    state = dict(case=case)
    if case["kind"] == "sample":
        b, V = case["b"], case["V"]
        logits = 3.0 * torch.randn(b, V, generator=gen, device=dev) + 1.5 * torch.randn(V, generator=gen, device=dev)
        spread = lambda lo, hi: lo + (hi - lo) * torch.rand(b, generator=gen, device=dev)
        state.update(logits=logits.to(DTYPES[case["dtype"]]), u=torch.rand(b, generator=gen, device=dev),
                     temperature=spread(0.5, 1.2))
        # every request has settings of its own around the case's; some switch a filter off
        k = (spread(0.5, 1.5) * case["k"]).round().int().clamp(min=1 if case["k"] else 0)
        state.update(top_k=k, top_p=case["p"] ** spread(0.5, 2.0), min_p=case["minp"] * spread(0.0, 2.0))
        return state
    state.update(_inputs(case, gen))
    b, h, N, P, dt = case["b"], case["h"], case["N"], case["P"], DTYPES[case["dtype"]]
    if case["kind"] == "step" or case["state"]:
        state["init"] = 0.3 * torch.randn(b, h, P, N, generator=gen, device=dev)
    if case.get("train"):
        for x in ("q", "k", "v", "g", "beta", "init"):
            if x in state:
                state[x].requires_grad_(True)
        state["do"] = torch.randn(b, h, case["T"], P, generator=gen, device=dev).to(dt)
        if case["state"]:
            state["dfinal"] = 0.1 * torch.randn(b, h, P, N, generator=gen, device=dev)
    return state


# --------------------------------------------------------------------------------------------------------------------
# the plain forms
# --------------------------------------------------------------------------------------------------------------------

def _heads(x, h):
    """Key heads as value heads see them."""
    return x if x.shape[1] == h else x.repeat_interleave(h // x.shape[1], dim=1)


def _unit_lower_inverse(A):
    """Inverse of I + A for strictly lower triangular A (..., L, L), L a power of two, from that of its diagonal blocks."""
    L = A.shape[-1]
    inv = A.new_ones(*A.shape[:-1], 1, 1)  # one block per row
    size = 1
    while size < L:
        blocks = A.unflatten(-2, (L // (2 * size), 2 * size)).unflatten(-1, (L // (2 * size), 2 * size))
        below = blocks[..., size:, :, :size].diagonal(dim1=-4, dim2=-2).movedim(-1, -3)
        first, second = inv[..., 0::2, :, :], inv[..., 1::2, :, :]
        low = torch.cat([-(second @ below @ first), second], -1)
        inv = torch.cat([torch.cat([first, torch.zeros_like(first)], -1), low], -2)
        size *= 2
    return inv[..., 0, :, :]


def _delta_plain(q, k, v, g, beta, scale, init):
    """Chunks of 64 tokens: with G the sums of g inside a chunk, D the written rows and S0 the state before it,
    (I + tril(beta e^{G_t-G_s} k k^T, -1)) D = beta (v - e^G S0 k),  o = scale (e^G S0 q + tril(e^{G_t-G_s} q k^T) D),
    S1 = e^{G_L} S0 + sum_s e^{G_L-G_s} d_s k_s^T."""
    b, h, T, P = v.shape
    N, L, dt = q.shape[-1], CHUNK, v.dtype
    pad = -T % L
    chunks = lambda x: torch.nn.functional.pad(x, (0, 0, 0, pad)).unflatten(2, (-1, L))
    q, k = (chunks(_heads(x, h).float()) for x in (q, k))
    v, beta, g = chunks(v.float()), chunks(beta.float().unsqueeze(-1)), chunks(g.double().unsqueeze(-1))
    G = g.cumsum(3)
    # (for s > t the exponent may be large: those places are closed before the exponential)
    decay = torch.exp((G - G.transpose(-1, -2)).float().tril().masked_fill(
        torch.ones(L, L, dtype=torch.bool, device=v.device).triu(1), -math.inf))
    inv = _unit_lower_inverse((beta * decay * (k @ k.transpose(-1, -2))).tril(-1))
    scores = decay * (q @ k.transpose(-1, -2))
    opened, closing = torch.exp(G.float()), torch.exp((G[..., -1:, :] - G).float())
    S = torch.zeros(b, h, P, N, device=v.device) if init is None else init.float()
    out = []
    for c in range(v.shape[2]):  # the state's way through the sequence has no plain form without a loop
        D = inv[:, :, c] @ (beta[:, :, c] * (v[:, :, c] - opened[:, :, c] * (k[:, :, c] @ S.transpose(-1, -2))))
        out.append(opened[:, :, c] * (q[:, :, c] @ S.transpose(-1, -2)) + scores[:, :, c] @ D)
        S = opened[:, :, c, -1:] * S + (closing[:, :, c] * D).transpose(-1, -2) @ k[:, :, c]
    o = (scale * torch.stack(out, 2)).flatten(2, 3)[:, :, :T]
    return o.to(dt), S


def _step_plain(q, k, v, g, beta, scale, S):
    h, dt = v.shape[1], v.dtype
    q, k = (_heads(x, h).float() for x in (q, k))
    S = torch.exp(g.float())[..., None, None] * S
    d = beta.float().unsqueeze(-1) * (v.float() - (S * k.unsqueeze(-2)).sum(-1))
    S = S + d.unsqueeze(-1) * k.unsqueeze(-2)
    return (scale * (S * q.unsqueeze(-2)).sum(-1)).to(dt), S


def _sample_plain(logits, u, temperature, top_k, top_p, min_p):
    """Tokens in the order of their logits (ties: lower index first); the first top_k stay, of these the shortest run with
    at least top_p of their mass, of these the ones with at least min_p of the largest.  The draw goes through what is
    left in the order of the indices: the first token at which the running mass exceeds u times the whole.  In 64 bits,
    since the running mass meets its borders closely."""
    x = logits.double()
    mass = torch.exp((x - x.amax(-1, keepdim=True)) / temperature.double().unsqueeze(-1))
    x, order = x.sort(dim=-1, descending=True, stable=True)
    ranked = mass.gather(-1, order)
    rank = torch.arange(x.shape[-1], device=x.device)
    k = top_k.unsqueeze(-1)
    ranked = torch.where((rank < k) | (k <= 0), ranked, 0.0)
    total = ranked.cumsum(-1)
    before = total - ranked
    stays = (before < top_p.double().unsqueeze(-1) * total[..., -1:]) & (ranked >= min_p.double().unsqueeze(-1))
    stays[..., 0] = True
    mass = torch.zeros_like(mass).scatter_(-1, order, torch.where(stays, ranked, 0.0))
    running = mass.cumsum(-1)
    return (running > u.double().unsqueeze(-1) * running[..., -1:]).int().argmax(-1)


# --------------------------------------------------------------------------------------------------------------------

LEAVES = ("q", "k", "v", "g", "beta", "init")


def run(state):
    case = state["case"]
    if case["kind"] == "sample":
        args = [state[x] for x in ("logits", "u", "temperature", "top_k", "top_p", "min_p")]
        if own:
            import slinoss_b200 as sb
            logits, u, temperature, top_k, top_p, min_p = args
            return sb.sample_b200(logits, u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
        return _sample_plain(*args)
    args = [state[x] for x in ("q", "k", "v", "g", "beta")]
    init, scale = state.get("init"), case["N"] ** -0.5
    if case["kind"] == "step":
        if own:
            import slinoss_b200 as sb
            return sb.gated_delta_step_b200(*args, scale=scale, initial_state=init)
        return _step_plain(*args, scale, init)
    if own:
        import slinoss_b200 as sb
        o, final = sb.gated_delta_rule_b200(*args, scale=scale, initial_state=init, return_state=True)
    else:
        o, final = _delta_plain(*args, scale, init)
    outs = dict(o=o, final=final) if case["state"] else dict(o=o)
    if not case["train"]:
        return outs
    names = [x for x in LEAVES if x in state]
    ends, grads = ([o, final], [state["do"], state["dfinal"]]) if case["state"] else ([o], [state["do"]])
    got = torch.autograd.grad(ends, [state[x] for x in names], grads)
    return {**{x: t.detach() for x, t in outs.items()}, **{"d_" + x: t for x, t in zip(names, got)}}


def work(case):
    size = DTYPES[case["dtype"]].itemsize
    b = case["b"]
    if case["kind"] == "sample":
        # the logits once; an exponential and a comparison or two for each
        return dict(bytes=b * case["V"] * size + 32 * b, flops=4 * b * case["V"])
    h, hk, N, P, T = case["h"], case["hk"], case["N"], case["P"], case.get("T", 1)
    ins = b * T * (2 * hk * N + h * P + 2 * h) * size
    out, states = b * T * h * P * size, 4 * b * h * P * N
    # of a token and head: S k, d k^T, S q and the decay of S; backward: the same again and seven such products
    flops = 7 * b * h * T * P * N
    if case["kind"] == "step":
        return dict(bytes=ins + out + 2 * states, flops=flops)
    moved = ins + out + (2 * states if case["state"] else 0)
    if case["train"]:
        moved += ins + ins + out + (2 * states if case["state"] else 0)  # the inputs again, d_o, the gradients
        flops += 22 * b * h * T * P * N
    return dict(bytes=moved, flops=flops)


# --------------------------------------------------------------------------------------------------------------------
# the definition, token by token in 64 bits
# --------------------------------------------------------------------------------------------------------------------

def _walk(S, tok, lo, hi, keep):
    """The recurrence over tokens lo..hi-1 from S: states before each token (if kept) and the state after the last."""
    seen = []
    for t in range(lo, hi):
        if keep:
            seen.append(S)
        S = S * tok["a"][:, :, t, None, None]
        d = tok["beta"][:, :, t, None] * (tok["v"][:, :, t] - torch.einsum("bhpn,bhn->bhp", S, tok["k"][:, :, t]))
        S = S + torch.einsum("bhp,bhn->bhpn", d, tok["k"][:, :, t])
        if not keep:
            tok["o"][:, :, t] = tok["scale"] * torch.einsum("bhpn,bhn->bhp", S, tok["q"][:, :, t])
    return seen, S


def exact(case, seed):
    if case["kind"] == "sample":
        return None
    if case.get("T", 1) * (4 if case.get("train") else 1) * (1 + case["b"] * case["h"] * case["P"] * case["N"] / 4e6) > 60000:
        return None
    s = prepare(case, seed)
    with torch.no_grad():
        return _exact(case, s)


def _exact(case, s):
    b, h, hk, N, P, T = (case.get(x, 1) for x in ("b", "h", "hk", "N", "P", "T"))
    share, scale = h // hk, 1.0 / math.sqrt(N)
    dim = (lambda x: x.detach().double().unsqueeze(2)) if case["kind"] == "step" else (lambda x: x.detach().double())
    wide = lambda x: x.unsqueeze(2).expand(b, hk, share, T, N).reshape(b, h, T, N)
    tok = dict(q=wide(dim(s["q"])), k=wide(dim(s["k"])), v=dim(s["v"]), a=dim(s["g"]).exp(), beta=dim(s["beta"]), scale=scale)
    tok["o"] = torch.zeros_like(tok["v"])
    S = s["init"].detach().double() if "init" in s else torch.zeros(b, h, P, N, dtype=torch.float64, device="cuda")
    part, starts = 64, []
    for lo in range(0, T, part):
        starts.append(S)
        S = _walk(S, tok, lo, min(T, lo + part), False)[1]
    if case["kind"] == "step":
        return tok["o"][:, :, 0], S
    outs = dict(o=tok["o"], final=S) if case["state"] else dict(o=tok["o"])
    if not case["train"]:
        return outs
    do = s["do"].double() * scale
    R = s["dfinal"].double() if case["state"] else torch.zeros_like(S)
    dq, dk, dv, dg, dbeta = (torch.zeros_like(tok[x]) for x in ("q", "k", "v", "a", "beta"))
    for lo in reversed(range(0, T, part)):
        hi = min(T, lo + part)
        seen, after = _walk(starts.pop(), tok, lo, hi, True)
        seen.append(after)
        for t in reversed(range(lo, hi)):
            q, k, v, a, beta = (tok[x][:, :, t] for x in ("q", "k", "v", "a", "beta"))
            before = seen[t - lo] * a[..., None, None]
            rest = v - torch.einsum("bhpn,bhn->bhp", before, k)
            dq[:, :, t] = torch.einsum("bhpn,bhp->bhn", seen[t - lo + 1], do[:, :, t])
            R = R + torch.einsum("bhp,bhn->bhpn", do[:, :, t], q)
            dd = torch.einsum("bhpn,bhn->bhp", R, k)
            dbeta[:, :, t] = (dd * rest).sum(-1)
            dv[:, :, t] = beta[..., None] * dd
            dk[:, :, t] = (torch.einsum("bhpn,bhp->bhn", R, beta[..., None] * rest)
                           - torch.einsum("bhpn,bhp->bhn", before, dv[:, :, t]))
            R = R - torch.einsum("bhp,bhn->bhpn", dv[:, :, t], k)
            dg[:, :, t] = (R * before).sum((-1, -2))
            R = R * a[..., None, None]
    grads = dict(q=dq.unflatten(1, (hk, share)).sum(2), k=dk.unflatten(1, (hk, share)).sum(2), v=dv, g=dg, beta=dbeta, init=R)
    return {**outs, **{"d_" + x: grads[x] for x in LEAVES if x in s}}

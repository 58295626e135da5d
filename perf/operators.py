"""The gated delta rule (chunked and recurrent) and the clipped policy loss, as a
user's program calls them, for timing and comparison.

A case names its operator with ``op``: ``delta`` (a whole sequence, forward or
with its gradients), ``step`` (a few tokens against a carried state) or
``policy`` (the loss with the gradient of the logits).  ``run`` computes the
operators in plain torch, in 32 bits and rounded once at the end, or (``own``)
calls ``thetascan_amd``; ``exact`` is their definition in 64 bits, token by token.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64


def listed():
    return [
        # a training step of a memory layer of the benchmark's size (8 heads of 64, B8 T4096)
        dict(name="delta_train", op="delta", train=True, B=8, Hk=8, H=8, T=4096, dk=64, dv=64, dtype="bf16",
             ragged=False, carried=False),
        # a wider layer: value heads that share keys and queries, 128-wide heads, continued from a state
        dict(name="delta_train_wide", op="delta", train=True, B=2, Hk=8, H=16, T=2048, dk=128, dv=128, dtype="bf16",
             ragged=False, carried=True),
        # a small model's step on a padded batch of a length that no chunk divides
        dict(name="delta_train_small", op="delta", train=True, B=2, Hk=4, H=4, T=131, dk=64, dv=64, dtype="bf16",
             ragged=True, carried=False),
        # fp32 training with odd head widths
        dict(name="delta_train_f32", op="delta", train=True, B=2, Hk=4, H=4, T=515, dk=48, dv=80, dtype="f32",
             ragged=False, carried=True),
        # a long prompt of one sequence read into a state
        dict(name="delta_prefill_long", op="delta", train=False, B=1, Hk=8, H=8, T=32768, dk=64, dv=64, dtype="bf16",
             ragged=False, carried=False),
        # a padded batch of prompts
        dict(name="delta_prefill_ragged", op="delta", train=False, B=8, Hk=4, H=8, T=1999, dk=128, dv=128,
             dtype="bf16", ragged=True, carried=False),
        # one token for each of eight sequences, where the call's latency is what counts
        dict(name="delta_step", op="step", B=8, Hk=8, H=8, T=1, dk=64, dv=64, dtype="bf16"),
        # one token for each sequence of a large serving batch with 128-wide heads
        dict(name="delta_step_batch", op="step", B=128, Hk=8, H=16, T=1, dk=128, dv=128, dtype="bf16"),
        # the hybrid LM's rollouts: its vocabulary, batch and soft cap
        dict(name="policy_lm", op="policy", N=65536, V=1024, dtype="bf16", cap=30.0, kl=0.05),
        # a few long-vocabulary sequences, no soft cap
        dict(name="policy_vocabulary", op="policy", N=8192, V=32768, dtype="bf16", cap=0.0, kl=0.05),
        # fp32 logits of an odd vocabulary, no KL term
        dict(name="policy_odd_f32", op="policy", N=517, V=5003, dtype="f32", cap=0.0, kl=0.0),
        # one short answer
        dict(name="policy_small", op="policy", N=64, V=1024, dtype="bf16", cap=30.0, kl=0.05),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def _widths(rng):
    return rng.choice([(64, 64), (64, 64), (128, 128), (128, 64), (64, 128), (48, 80), (32, 64), (96, 40), (80, 56)])


def draw(rng):
    kind = rng.choice(["train", "train", "prefill", "prefill", "step", "policy", "policy"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "policy":
        V = _log_int(rng, 500, 32768)
        if rng.random() < 0.5:
            V = max(512, V // 512 * 512)
        most = (32768 * 8192 if dtype == "bf16" else 32768 * 2048) // V
        N = _log_int(rng, 32, min(65536, most))
        return dict(op="policy", N=N, V=V, dtype=dtype, cap=rng.choice([0.0, 30.0]), kl=rng.choice([0.0, 0.05, 0.2]))
    dk, dv = _widths(rng)
    H = rng.choice([2, 4, 6, 8, 16])
    Hk = rng.choice([h for h in (1, 2, 3, 4, 8, 16) if H % h == 0])
    if kind == "step":
        return dict(op="step", B=_log_int(rng, 1, 128), Hk=Hk, H=H, T=rng.choice([1, 1, 1, 2, 5, 8]), dk=dk, dv=dv,
                    dtype=dtype)
    # rows (tokens times heads times width) up to those of the largest listed cases
    most = 8 * 8 * 4096 * 64 // (H * max(dk, dv))
    if dtype == "f32":
        most //= 8
    if kind == "prefill":
        tokens = _log_int(rng, 32, most)
        B = rng.choice([b for b in (1, 2, 3, 5, 8) if b * 16 <= tokens])
    else:
        tokens = _log_int(rng, 96, most)
        B = rng.choice([b for b in (2, 3, 5, 8) if b * 32 <= tokens])
    T = min(32768 if kind == "prefill" else 4096, tokens // B)
    T = T | 1 if rng.random() < 0.5 else max(32, T // 32 * 32)
    return dict(op="delta", train=kind == "train", B=B, Hk=Hk, H=H, T=T, dk=dk, dv=dv, dtype=dtype,
                ragged=rng.random() < 0.3, carried=rng.random() < 0.4)


# ------------------------------------------------------------------ inputs

def _unit_rows(x):
    return x / (x * x).sum(-1, keepdim=True).sqrt()


def _delta_inputs(case, g):
    """Normalized queries and keys (neighbouring keys are alike, as those of a
    running text are), values of unit variance, write strengths from a sigmoid, a
    learned decay of which one token in two hundred is a reset.  A bf16 model
    trains on pieces of a long text, each continued from the last one's state; in
    fp32 the state and its successor have gradients too."""
    B, Hk, H, T, dk, dv = (case[n] for n in ("B", "Hk", "H", "T", "dk", "dv"))
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    # token-major memory, as projections give it
    q = _unit_rows(normal(B, T, Hk, dk))
    k = normal(B, T, Hk, dk)
    k = _unit_rows(k + 0.7 * torch.roll(k, 1, 1))
    v = normal(B, T, H, dv)
    beta = torch.sigmoid(normal(B, T, H))
    decay = -torch.nn.functional.softplus(normal(B, T, H) - 4.0)
    decay = torch.where(torch.rand(B, T, H, generator=g, device="cuda") < 0.005, decay - 12.0, decay)
    s = dict(q=q.to(dt).transpose(1, 2), k=k.to(dt).transpose(1, 2), v=v.to(dt).transpose(1, 2),
             beta=beta.to(dt).transpose(1, 2), decay=decay.to(dt).transpose(1, 2))
    if case["op"] == "step" or case["carried"]:
        s["state"] = 0.3 * normal(B, H, dk, dv)
    if case["op"] == "delta":
        if case["ragged"]:
            lengths = torch.randint(0, T + 1, (B,), generator=g, device="cuda")
            lengths[0] = T
            s["lengths"] = lengths
        if case["train"]:
            s["dout"] = normal(B, T, H, dv).to(dt).transpose(1, 2)
            if case["dtype"] == "f32":
                s["dstate"] = normal(B, H, dk, dv)
    return s


def _policy_inputs(case, g):
    """Logits with a clear first choice now and then, log-probabilities of an
    older and a reference policy near the present one, normalized advantages, and
    rows of the prompts and the padding, of weight zero, some of them never
    written.  No ratio lies within 1e-3 of a clipping border."""
    N, V = case["N"], case["V"]
    z = 2.0 * torch.randn(N, V, generator=g, device="cuda")
    tokens = torch.randint(0, V, (N,), generator=g, device="cuda")
    rows = torch.arange(N, device="cuda")
    z[rows, tokens] += 6.0 * torch.rand(N, generator=g, device="cuda")
    z = z.to(DTYPES[case["dtype"]])
    lp = torch.empty(N, dtype=torch.float64, device="cuda")
    for i in range(0, N, 2048):
        lp[i:i + 2048] = _token_logp(z[i:i + 2048].double(), tokens[i:i + 2048], case["cap"])
    change = 0.15 * torch.randn(N, generator=g, device="cuda", dtype=torch.float64)
    for border in (1.0 - LOW, 1.0 + HIGH):
        change = torch.where((change.exp() - border).abs() < 2e-3, change + 5e-3, change)
    s = dict(z=z, tokens=tokens, old=(lp - change).float(),
             ref=(lp + 0.3 * torch.randn(N, generator=g, device="cuda", dtype=torch.float64)).float(),
             advantages=torch.randn(N, generator=g, device="cuda"))
    used = torch.rand(N, generator=g, device="cuda") < 0.8
    used[0] = True
    s["weights"] = torch.where(used, 1.0 / used.sum(), 0.0).float()
    unwritten = ~used & (torch.rand(N, generator=g, device="cuda") < 0.2)
    z[unwritten] = float("nan")
    return s


LOW, HIGH = 0.2, 0.28


def _leaves(s):
    return ["q", "k", "v", "beta", "decay"] + (["state"] if "state" in s and "dstate" in s else [])


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = _policy_inputs(case, g) if case["op"] == "policy" else _delta_inputs(case, g)
    if case["op"] == "policy":
        s["z"].requires_grad_()
    elif case["op"] == "delta" and case["train"]:
        for name in _leaves(s):
            s[name].requires_grad_()
    s["case"] = case
    return s


# ------------------------------------------------------------------ plain forms

def _plain_delta(q, k, v, beta, decay, state, lengths):
    """The chunked form of the delta rule: per chunk the triangular system's
    inverse (by blocks of 1, 2, 4 .. 32 rows), then the states in order."""
    B, H, T, dv = v.shape
    dk, rep, C = q.shape[-1], H // q.shape[1], CHUNK
    n = -(-T // C)
    q, k, v, beta, decay = q.float(), k.float(), v.float(), beta.float(), decay.float()
    if lengths is not None:
        seen = (torch.arange(T, device=q.device) < lengths[:, None])[:, None]
        q, k, v = (torch.where(seen[..., None], x, 0.0) for x in (q, k, v))
        beta, decay = torch.where(seen, beta, 0.0), torch.where(seen, decay, 0.0)
    if rep > 1:
        q, k = (x[:, :, None].expand(B, H // rep, rep, T, dk).reshape(B, H, T, dk) for x in (q, k))

    def chunks(x):
        pad = n * C - T
        if pad:
            x = torch.cat([x, x.new_zeros(*x.shape[:2], pad, *x.shape[3:])], 2)
        return x.reshape(B, H, n, C, *x.shape[3:])

    q, k, v, beta, decay = (chunks(x) for x in (q, k, v, beta, decay))
    G = decay.double().cumsum(-1)  # (differences of sums: 64 bits)
    i = torch.arange(C, device=q.device)
    below, lower = i[:, None] > i, i[:, None] >= i
    D = torch.where(lower, (G[..., :, None] - G[..., None, :]).clamp(max=0.0), 0.0).float().exp()
    up = k.transpose(-1, -2).contiguous()
    L = torch.where(below, (k @ up) * D * beta[..., None], 0.0)
    P = torch.where(lower, (q @ up) * D, 0.0)
    inv = torch.eye(C, device=q.device).expand_as(L)
    size = 1
    while size < C:
        # pairs of neighbouring diagonal blocks: the lower left block of their inverse
        block = (i[:, None] // size % 2 == 1) & (i // size % 2 == 0) & (i[:, None] // (2 * size) == i // (2 * size))
        inv = inv - inv @ torch.where(block, L, 0.0) @ inv
        size *= 2
    eG, last = G.float().exp()[..., None], G[..., -1:]
    tail = (last - G).float().exp()[..., None]
    w = inv @ (beta[..., None] * eG * k)
    u = inv @ (beta[..., None] * v)
    S = q.new_zeros(B, H, dk, dv) if state is None else state
    whole = last.float().exp()[..., None]
    out = []
    for c in range(n):
        uc = u[:, :, c] - w[:, :, c] @ S
        out.append((eG[:, :, c] * q[:, :, c]) @ S + P[:, :, c] @ uc)
        S = whole[:, :, c] * S + (tail[:, :, c] * k[:, :, c]).transpose(-1, -2).contiguous() @ uc
    return torch.stack(out, 2).reshape(B, H, n * C, dv)[:, :, :T], S


def _plain_step(q, k, v, beta, decay, state):
    rep = v.shape[1] // q.shape[1]
    q, k, v = q.float().repeat_interleave(rep, 1), k.float().repeat_interleave(rep, 1), v.float()
    out, S = [], state
    for t in range(q.shape[2]):
        S = decay[:, :, t, None, None].float().exp() * S
        u = beta[:, :, t, None].float() * (v[:, :, t] - (S * k[:, :, t, :, None]).sum(2))
        S = S + k[:, :, t, :, None] * u[:, :, None]
        out.append((S * q[:, :, t, :, None]).sum(2))
    return torch.stack(out, 2), S


def _token_logp(z, tokens, cap):
    if cap:
        z = cap * torch.tanh(z / cap)
    m = z.amax(-1, keepdim=True).detach()
    chosen = z.gather(-1, tokens[:, None])[:, 0]
    return (chosen - m[:, 0]).double() - (z - m).exp().sum(-1, dtype=torch.float64).log()


def _plain_policy(s, case):
    """Per row in 32 bits, the rows' terms in 64: normalized advantages all but
    cancel in their sum."""
    w = s["weights"]
    z = torch.where((w != 0)[:, None], s["z"].float(), 0.0)
    lp = torch.where(w != 0, _token_logp(z, s["tokens"], case["cap"]), 0.0)
    ratio = torch.where(w != 0, lp - s["old"], 0.0).exp()
    clipped = ratio.clamp(1.0 - LOW, 1.0 + HIGH)
    loss = -torch.minimum(ratio * s["advantages"], clipped * s["advantages"])
    if case["kl"]:
        off = torch.where(w != 0, s["ref"] - lp, 0.0)
        loss = loss + case["kl"] * (off.exp() - off - 1.0)
    loss = (w * loss).sum()
    return loss.float(), lp.detach().float()


# ------------------------------------------------------------------ the calls

def run(state):
    case = state["case"]
    if case["op"] == "policy":
        return _run_policy(state, case)
    if case["op"] == "step":
        with torch.no_grad():
            if own:
                import thetascan_amd as ts

                out, S = ts.gated_delta_rule(state["q"], state["k"], state["v"], state["beta"], state["decay"],
                                             state=state["state"], return_state=True)
            else:
                out, S = _plain_step(*(state[n] for n in ("q", "k", "v", "beta", "decay", "state")))
                out = out.to(state["q"].dtype)
        return out, S
    with torch.set_grad_enabled(case["train"]):
        if own:
            import thetascan_amd as ts

            out, S = ts.gated_delta_rule(state["q"], state["k"], state["v"], state["beta"], state["decay"],
                                         state=state.get("state"), lengths=state.get("lengths"), return_state=True)
        else:
            out, S = _plain_delta(state["q"], state["k"], state["v"], state["beta"], state["decay"],
                                  state.get("state"), state.get("lengths"))
            out = out.to(state["q"].dtype)
    if not case["train"]:
        return out, S
    ends = [(out, state["dout"])] + ([(S, state["dstate"])] if "dstate" in state else [])
    grads = torch.autograd.grad([e for e, _ in ends], [state[n] for n in _leaves(state)], [d for _, d in ends])
    return [out.detach(), S.detach(), *grads]


def _run_policy(s, case):
    if own:
        import thetascan_amd as ts

        loss, lp = ts.policy_loss(s["z"], s["tokens"], s["old"], s["advantages"],
                                  ref_log_probs=s["ref"] if case["kl"] else None, weights=s["weights"],
                                  clip=(LOW, HIGH), kl=case["kl"], softcap=case["cap"] or None)
    else:
        loss, lp = _plain_policy(s, case)
    (dz,) = torch.autograd.grad(loss, [s["z"]])
    return loss.detach(), lp, dz


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "policy":
        N, V = case["N"], case["V"]
        return {"bytes": 2 * N * V * es + N * (8 + 5 * 4), "flops": 10 * N * V}
    B, Hk, H, T, dk, dv = (case[n] for n in ("B", "Hk", "H", "T", "dk", "dv"))
    rows = B * T
    keys, values, gates = rows * Hk * dk * es, rows * H * dv * es, rows * H * es
    S = B * H * dk * dv * 4
    if case["op"] == "step":
        return {"bytes": 2 * keys + 2 * values + 2 * gates + 2 * S, "flops": 7 * rows * H * dk * dv}
    forward = 6 * dk * dv + 2 * CHUNK * (dk + dv)
    if not case["train"]:
        return {"bytes": 2 * keys + 2 * values + 2 * gates + S * (1 + case["carried"]), "flops": rows * H * forward}
    # forward; backward: q, k, v, dout and the gates again, and their gradients
    return {"bytes": 6 * keys + 5 * values + 6 * gates + S * (1 + case["carried"]) * (1 + (es == 4)),
            "flops": int(3.5 * rows * H * forward)}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {n: x.detach() if torch.is_tensor(x) else x for n, x in s.items()}
    with torch.no_grad():
        return _exact_policy(s, case) if case["op"] == "policy" else _exact_delta(s, case)


def _exact_delta(s, case):
    """S_t = a S_(t-1) + k u^T, u = b (v - a S_(t-1)^T k), o = S_t^T q, one token
    after the other, and the adjoint of each line in reverse order."""
    B, Hk, H, T, dk, dv = (case[n] for n in ("B", "Hk", "H", "T", "dk", "dv"))
    rep = H // Hk
    train = case["op"] == "delta" and case["train"]

    def stream(x):  # token-first, one matrix of all (batch, head) rows per token
        x = x.double()
        if x.shape[1] != H:
            x = x.repeat_interleave(rep, 1)
        return x.reshape(B * H, T, -1).transpose(0, 1).contiguous()

    q, k, v, b, g = (stream(s[n]) for n in ("q", "k", "v", "beta", "decay"))
    if s.get("lengths") is not None:
        on = (torch.arange(T, device=q.device)[:, None] < s["lengths"].repeat_interleave(H))[..., None]
        q, k, v, b, g = (torch.where(on, x, 0.0) for x in (q, k, v, b, g))
    a = g.exp()[..., None]
    S = s["state"].double().reshape(B * H, dk, dv) if "state" in s else q.new_zeros(B * H, dk, dv)
    o = torch.empty_like(v)
    held, us = [S], []
    for t in range(T):
        A = a[t] * S
        u = b[t] * (v[t] - torch.bmm(k[t][:, None], A)[:, 0])
        S = A + k[t][:, :, None] * u[:, None]
        o[t] = torch.bmm(q[t][:, None], S)[:, 0]
        if train:
            held.append(S)
            us.append(u)

    def heads(x, h=H):
        return x.transpose(0, 1).reshape(B, h, T, -1)

    out = [heads(o), S.reshape(B, H, dk, dv)]
    if not train:
        return out
    do = stream(s["dout"])
    if s.get("lengths") is not None:
        do = torch.where(on, do, 0.0)
    dS = s["dstate"].double().reshape(B * H, dk, dv) if "dstate" in s else torch.zeros_like(S)
    dq, dk_, dv_, db, dg = (torch.empty_like(x) for x in (q, k, v, b, g))
    for t in range(T - 1, -1, -1):
        S1, A, u = held[t + 1], a[t] * held[t], us[t]
        dq[t] = torch.bmm(S1, do[t][:, :, None])[..., 0]
        dS = dS + q[t][:, :, None] * do[t][:, None]
        du = torch.bmm(k[t][:, None], dS)[:, 0]
        miss = v[t] - torch.bmm(k[t][:, None], A)[:, 0]
        db[t] = (du * miss).sum(-1, keepdim=True)
        dv_[t] = b[t] * du
        dk_[t] = torch.bmm(dS, u[:, :, None])[..., 0] - torch.bmm(A, dv_[t][:, :, None])[..., 0]
        dS = dS - k[t][:, :, None] * dv_[t][:, None]
        dg[t] = (dS * A).sum((1, 2))[:, None]
        dS = a[t] * dS
    if s.get("lengths") is not None:
        dg = torch.where(on, dg, 0.0)
        db = torch.where(on, db, 0.0)
    shared = [heads(x).reshape(B, Hk, rep, T, dk).sum(2) for x in (dq, dk_)]
    out += [*shared, heads(dv_), heads(db)[..., 0], heads(dg)[..., 0]]
    if "state" in _leaves(s):
        out.append(dS.reshape(B, H, dk, dv))
    return out


def _exact_policy(s, case):
    N, V, cap, kl = case["N"], case["V"], case["cap"], case["kl"]
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    lps = torch.zeros(N, dtype=torch.float64, device="cuda")
    dz = torch.zeros(N, V, dtype=torch.float64 if N * V <= 1 << 27 else torch.float32, device="cuda")
    for i in range(0, N, 2048):
        rows = torch.arange(i, min(N, i + 2048), device="cuda")
        rows = rows[s["weights"][rows] != 0]
        z, tok, A, w = s["z"][rows].double(), s["tokens"][rows], s["advantages"][rows].double(), s["weights"][rows].double()
        y = cap * torch.tanh(z / cap) if cap else z
        slope = 1.0 - (y / cap) ** 2 if cap else torch.ones_like(y)
        p = (y - y.amax(-1, keepdim=True)).exp()
        p = p / p.sum(-1, keepdim=True)
        chosen = torch.arange(V, device="cuda") == tok[:, None]
        lp = torch.where(chosen, p, 0.0).sum(-1).log()
        r = (lp - s["old"][rows].double()).exp()
        flat = ((A > 0) & (r > 1 + HIGH)) | ((A < 0) & (r < 1 - LOW))
        edge = torch.where(A > 0, 1.0 + HIGH, 1.0 - LOW)
        each, slope_lp = -torch.where(flat, edge, r) * A, torch.where(flat, 0.0, -r * A)
        if kl:
            d = s["ref"][rows].double() - lp
            each, slope_lp = each + kl * (d.exp() - d - 1.0), slope_lp + kl * (1.0 - d.exp())
        loss = loss + (w * each).sum()
        lps[rows] = lp
        dz[rows] = ((w * slope_lp)[:, None] * (chosen.double() - p) * slope).to(dz.dtype)
    return loss, lps, dz

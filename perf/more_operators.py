"""What the hybrid language model answers with and learns from a teacher by: windowed
attention with sinks (whole sequences, and single tokens against a ring cache), sampling
of tokens, and distillation from a teacher's top log-probabilities, as a user's program
calls them, for timing and comparison.

A case names its operator with ``op``: ``attention`` (a whole sequence, forward or with
its gradients), ``step`` (one token a sequence against its cache), ``sample`` or
``distill`` (the loss with the gradient of the logits).  ``run`` computes the operators
in plain torch, in 32 bits and rounded once at the end (the sampled tokens' weights in
64, as whole numbers), or (``own``) calls ``thetascan_amd``; ``exact`` is their
definition in 64 bits.
"""
from __future__ import annotations

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
UNIT = float(1 << 44)  # a sampled token's weight is a whole number of 1 / UNIT of the largest


def listed():
    return [
        # a training step of an attention layer of the benchmark's size (8 query heads on 4 key heads of 64, B8 T4096)
        dict(name="attention_train", op="attention", train=True, B=8, H=8, Hk=4, T=4096, d=64, window=1024, sinks=4,
             dtype="bf16", ragged=False),
        # a long text of one sequence with 128-wide heads
        dict(name="attention_train_long", op="attention", train=True, B=1, H=8, Hk=2, T=16384, d=128, window=2048,
             sinks=64, dtype="bf16", ragged=False),
        # fp32 training on a padded batch, odd sizes throughout
        dict(name="attention_train_f32", op="attention", train=True, B=3, H=6, Hk=2, T=515, d=80, window=100, sinks=3,
             dtype="f32", ragged=True),
        # a long prompt read at once
        dict(name="attention_prefill", op="attention", train=False, B=1, H=8, Hk=4, T=32768, d=64, window=1024, sinks=4,
             dtype="bf16", ragged=False),
        # one token of one sequence, where the call's latency is what counts
        dict(name="step_one", op="step", B=1, H=8, Hk=4, d=64, window=4096, sinks=4, dtype="bf16"),
        # a serving batch with 128-wide heads, some places of it free
        dict(name="step_batch", op="step", B=64, H=32, Hk=8, d=128, window=4096, sinks=16, dtype="bf16"),
        # the hybrid LM's rollouts: its vocabulary and soft cap, one temperature for all
        dict(name="sample_lm", op="sample", N=512, V=1024, dtype="bf16", cap=30.0, mixed=False),
        # a serving batch of a long vocabulary, every request with settings of its own
        dict(name="sample_batch", op="sample", N=256, V=131072, dtype="bf16", cap=0.0, mixed=True),
        # two requests of an odd vocabulary in fp32
        dict(name="sample_two", op="sample", N=2, V=50257, dtype="f32", cap=0.0, mixed=True),
        # the hybrid LM learns from a teacher of its kind: its vocabulary, batch and soft cap
        dict(name="distill_lm", op="distill", N=65536, V=1024, K=32, dtype="bf16", cap=30.0, temperature=1.0, tail=True),
        # a long vocabulary, the teacher's answers softened
        dict(name="distill_vocabulary", op="distill", N=8192, V=32768, K=64, dtype="bf16", cap=0.0, temperature=2.0,
             tail=True),
        # one short answer, fp32 logits of an odd vocabulary, the teacher's top alone
        dict(name="distill_small", op="distill", N=61, V=5003, K=20, dtype="f32", cap=0.0, temperature=1.0, tail=False),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1))))))


def draw(rng):
    op = rng.choice(["train", "train", "prefill", "step", "step", "sample", "sample", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if op == "sample":
        V = _log_int(rng, 500, 131072)
        if rng.random() < 0.5:
            V = max(512, V // 512 * 512)
        N = _log_int(rng, 1, min(1024, 256 * 131072 // (V * (1 if dtype == "bf16" else 2))))
        return dict(op="sample", N=N, V=V, dtype=dtype, cap=rng.choice([0.0, 0.0, 30.0]), mixed=rng.random() < 0.7)
    if op == "distill":
        V = _log_int(rng, 500, 32768)
        if rng.random() < 0.5:
            V = max(512, V // 512 * 512)
        most = (32768 * 8192 if dtype == "bf16" else 32768 * 2048) // V
        return dict(op="distill", N=_log_int(rng, 16, min(65536, most)), V=V, K=rng.choice([1, 8, 20, 32, 64, 100, 256]),
                    dtype=dtype, cap=rng.choice([0.0, 30.0]), temperature=rng.choice([1.0, 1.0, 2.0]),
                    tail=rng.random() < 0.6)
    d = rng.choice([64, 64, 128, 128, 32, 40, 80, 96])
    Hk = rng.choice([1, 2, 3, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4, 8])
    sinks = rng.choice([0, 1, 4, 4, 16, 64])
    if op == "step":
        window = _log_int(rng, 64, 8192)
        most = 64 * 8 * 4096 * 128 // (Hk * window * d * (1 if dtype == "bf16" else 2))
        return dict(op="step", B=_log_int(rng, 1, max(1, min(256, most))), H=H, Hk=Hk, d=d, window=window, sinks=sinks,
                    dtype=dtype)
    window = _log_int(rng, 16, 4096)
    # pairs of a query and a key, times the width: up to those of the largest listed case
    pairs = 8 * 8 * 4096 * 1024 * 64 // (H * max(64, d) * (1 if dtype == "bf16" else 16))
    tokens = min(32768, _log_int(rng, 48, max(64, pairs // min(window, 2048))))
    B = rng.choice([b for b in (1, 2, 3, 5, 8) if b * 16 <= tokens])
    T = tokens // B
    T = T | 1 if rng.random() < 0.5 else max(16, T // 32 * 32)
    return dict(op="attention", train=op == "train", B=B, H=H, Hk=Hk, T=T, d=d, window=window, sinks=sinks, dtype=dtype,
                ragged=rng.random() < 0.3)


# ------------------------------------------------------------------ inputs

def _lengths(case):
    """The lengths of a padded batch, from the whole width down."""
    B, T = case["B"], case["T"]
    return [T - b * T // B if case["ragged"] else T for b in range(B)]


def _positions(case):
    """Tokens that each sequence of a serving batch has had: from few to several
    times what its ring holds, every eighth place free (-1)."""
    B, W = case["B"], case["window"]
    return [-1 if b % 8 == 7 else (W * 3 * (b + 1)) // (2 * B) + (b % 5) * (b % 2) * W for b in range(B)]


def _attention_inputs(case, g):
    """Queries and keys of unit mean square per head (neighbouring keys are alike,
    as those of a running text are), the queries with a gain of 1.5."""
    B, H, Hk, d = (case[n] for n in ("B", "H", "Hk", "d"))
    T = case["T"] if case["op"] == "attention" else 1
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    def unit(x):
        return x / (x * x).mean(-1, keepdim=True).sqrt()

    def rows(x):  # token-major memory, as projections give it
        return x.to(dt).transpose(1, 2)

    k = normal(B, T, Hk, d)
    s = dict(q=rows(1.5 * unit(normal(B, T, H, d))), k=rows(unit(k + 0.7 * torch.roll(k, 1, 1))),
             v=rows(normal(B, T, Hk, d)))
    if case["op"] == "step":
        slots = case["sinks"] + case["window"]
        s["cache_k"] = unit(normal(B, Hk, slots, d)).to(dt)
        s["cache_v"] = normal(B, Hk, slots, d).to(dt)
        order = torch.randperm(B, generator=g, device="cuda")
        s["positions"] = torch.tensor(_positions(case), device="cuda")[order]
        return s
    if case["ragged"]:
        order = torch.randperm(B, generator=g, device="cuda")
        s["lengths"] = torch.tensor(_lengths(case), device="cuda")[order]
    if case["train"]:
        s["dout"] = rows(normal(B, T, H, d))
    return s


def _sample_inputs(case, g):
    """Logits of a spread of 3 with a few clear choices now and then, some tokens
    forbidden (-inf); the random numbers; and each request's settings, or one for
    all: a tempered nucleus."""
    N, V = case["N"], case["V"]

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    z = 3.0 * torch.randn(N, V, generator=g, device="cuda")
    z[:, : min(V, 64)] += 8.0 * uniform(N, 1) * uniform(N, min(V, 64))
    z[uniform(N, V) < 0.01] = -math.inf
    s = dict(z=z.to(DTYPES[case["dtype"]]), u=uniform(N), temperature=0.8, top_k=None, top_p=0.95, min_p=None)
    if case["mixed"]:
        kind = torch.randint(0, 4, (N,), generator=g, device="cuda")
        # plain sampling, top-k, a nucleus, and both with a least share
        s["temperature"] = torch.where(kind == 0, 1.0, 0.5 + uniform(N))
        s["top_k"] = torch.where(kind % 2 == 1, torch.randint(1, 101, (N,), generator=g, device="cuda"), V)
        s["top_p"] = torch.where(kind >= 2, 0.6 + 0.39 * uniform(N), 1.0)
        s["min_p"] = torch.where(kind == 3, 0.1 * uniform(N), 0.0)
    return s


def _distill_inputs(case, g):
    """A student near its teacher; the teacher's K first tokens with their
    log-probabilities; rows of prompts and padding, of weight zero, some of them
    never written."""
    N, V, K = case["N"], case["V"], case["K"]
    z = torch.empty(N, V, dtype=DTYPES[case["dtype"]], device="cuda")
    ids = torch.empty(N, K, dtype=torch.int64, device="cuda")
    lps = torch.empty(N, K, device="cuda")
    for i in range(0, N, 8192):
        n = min(N, i + 8192) - i
        y = 2.5 * torch.randn(n, V, generator=g, device="cuda")
        z[i:i + n] = y + 0.5 * torch.randn(n, V, generator=g, device="cuda")
        lp = torch.log_softmax(y / case["temperature"], -1)
        lps[i:i + n], ids[i:i + n] = lp.topk(K, -1)
    used = torch.rand(N, generator=g, device="cuda") < 0.8
    used[0] = True
    unwritten = ~used & (torch.rand(N, generator=g, device="cuda") < 0.2)
    z[unwritten] = float("nan")
    return dict(z=z, ids=ids, lps=lps, weights=torch.where(used, 1.0 / used.sum(), 0.0).float())


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "sample":
        s = _sample_inputs(case, g)
    elif case["op"] == "distill":
        s = _distill_inputs(case, g)
        s["z"].requires_grad_()
    else:
        s = _attention_inputs(case, g)
        if case["op"] == "attention" and case["train"]:
            for name in "qkv":
                s[name].requires_grad_()
    s["case"] = case
    return s


# ------------------------------------------------------------------ plain forms

def _plain_softmax(scores, seen):
    """Rows of shares over the last axis, zero where nothing is seen."""
    scores = torch.where(seen, scores, -math.inf)
    top = scores.detach().amax(-1, keepdim=True)
    e = torch.where(seen, (scores - torch.where(top > -math.inf, top, 0.0)).exp(), 0.0)
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total > 0, total, 1.0)


def _plain_attention(q, k, v, window, sinks, lengths):
    """Blocks of at least a window of queries, each against its own and the last
    block's keys and the sinks before those."""
    B, H, T, d = q.shape
    Hk = k.shape[1]
    q, k, v = q.float(), k.float(), v.float()
    on = torch.ones(B, T, dtype=torch.bool, device=q.device)
    if lengths is not None:
        on = torch.arange(T, device=q.device) < lengths[:, None]
        q, k, v = (torch.where(on[:, None, :, None], x, 0.0) for x in (q, k, v))
    C = min(T, max(window, 64))
    n = -(-T // C)

    def blocks(x):  # [B,Hk,rep,n,C,d]
        x = torch.cat([x, x.new_zeros(B, x.shape[1], n * C - T, d)], 2)
        return x.reshape(B, Hk, -1, n, C, d)

    def pairs(x):  # each block's keys, and those of the block before it
        x = blocks(x)
        return torch.cat([torch.cat([torch.zeros_like(x[:, :, :, :1]), x[:, :, :, :-1]], 3), x], 4)

    q, kk, vv = blocks(q), pairs(k), pairs(v)
    first = min(sinks, T)
    # sinks as keys of every block
    kk, vv = (torch.cat([x[:, :, None, None, :first].expand(B, Hk, 1, n, first, d), xx], 4)
              for x, xx in ((k, kk), (v, vv)))
    i = torch.arange(n * C, device=q.device).reshape(n, C)
    j = torch.arange(n, device=q.device)[:, None] * C + torch.arange(-C, C, device=q.device)
    at = torch.arange(first, device=q.device).expand(n, first)
    near = (j[:, None] >= 0) & (j[:, None] <= i[..., None]) & (i[..., None] - j[:, None] < window)
    far = i[..., None] - at[:, None] >= window
    seen = torch.cat([far, near], -1)
    scores = (q @ kk.transpose(-1, -2).contiguous()) * d ** -0.5
    out = _plain_softmax(scores, seen) @ vv
    out = out.reshape(B, H, n * C, d)[:, :, :T]
    return torch.where(on[:, None, :, None], out, 0.0)


def _slot(positions, window, sinks):
    return torch.where(positions < sinks, positions, sinks + (positions - sinks).remainder(window))


def _plain_step(s, window, sinks):
    """The new key and value into their slots, then every slot that holds a visible token."""
    q, k, v, K, V, pos = (s[n] for n in ("q", "k", "v", "cache_k", "cache_v", "positions"))
    B, H, _, d = q.shape
    Hk = k.shape[1]
    active = pos >= 0
    rows = torch.arange(B, device=q.device)
    slot = torch.where(active, _slot(pos, window, sinks), 0)
    for cache, new in ((K, k), (V, v)):
        cache[rows, :, slot] = torch.where(active[:, None, None], new[:, :, 0], cache[rows, :, slot])
    slots = torch.arange(sinks + window, device=q.device)
    # (a ring that is not full yet holds tokens up to the newest's slot)
    seen = (slots <= pos[:, None]) & active[:, None]
    scores = (q.float().reshape(B, Hk, H // Hk, d) @ K.float().transpose(-1, -2).contiguous()) * d ** -0.5
    share = _plain_softmax(scores, seen[:, None, None])
    return torch.where(active[:, None, None, None], (share @ V.float()).reshape(B, H, 1, d), 0.0).to(q.dtype)


def _capped(z, cap):
    return cap * torch.tanh(z / cap) if cap else z


def _per_row(x, z, none):
    return torch.full(z.shape[:1], none if x is None else x, device=z.device, dtype=torch.float64) if not torch.is_tensor(x) else x


def _plain_sample(s, cap):
    """Sorted weights for what the settings leave, then the first token, in the
    order of their numbers, whose running sum passes u of the sum."""
    z, V = s["z"], s["z"].shape[1]
    y = _capped(z.double(), cap)
    top = y.amax(-1, keepdim=True)
    t, p, least = (_per_row(s[n], z, none).double()[:, None] for n, none in (("temperature", 1.0), ("top_p", 1.0), ("min_p", 0.0)))
    k = _per_row(s["top_k"], z, V).long()[:, None]
    w = (((y - top) / t).exp() * UNIT).round().long()
    order = torch.sort(z, dim=-1, descending=True, stable=True).indices
    ws = w.gather(-1, order)
    ws = torch.where(torch.arange(V, device=z.device) < k, ws, 0)
    before = ws.cumsum(-1) - ws
    ws = torch.where(before.double() < p * ws.sum(-1, keepdim=True).double(), ws, 0)
    ws = torch.where(ws.double() >= least * UNIT, ws, 0)
    kept = torch.zeros_like(w).scatter(-1, order, ws)
    running = kept.cumsum(-1)
    total = running[:, -1:]
    place = torch.minimum((s["u"].double()[:, None] * total.double()).floor().long(), total - 1)
    token = (running <= place).sum(-1)
    chosen = y.gather(-1, token[:, None])[:, 0] - top[:, 0]
    return token, (chosen - (y - top).exp().sum(-1).log()).float()


def _plain_distill(s, case):
    """Per row in 32 bits, a row's terms and the rows' sum in 64."""
    w, ids, lp = s["weights"], s["ids"], s["lps"].double()
    used = w != 0
    x = _capped(torch.where(used[:, None], s["z"].float(), 0.0), case["cap"]) / case["temperature"]
    x = x - x.amax(-1, keepdim=True).detach()
    e = x.exp()
    total = e.sum(-1, dtype=torch.float64)
    lq = x.gather(-1, ids).double() - total.log()[:, None]
    if not case["tail"]:
        lp = lp - lp.exp().sum(-1, keepdim=True).log()
    p = lp.exp()
    each = (p * (lp - lq)).sum(-1)
    if case["tail"]:
        rest = e.scatter(-1, ids, 0.0).sum(-1, dtype=torch.float64)
        left = (1.0 - p.sum(-1)).clamp(min=0.0)
        some = left > 0
        some_left = torch.where(some, left, 1.0)
        each = each + torch.where(some, left * (some_left.log() - rest.log() + total.log()), 0.0)
    each = torch.where(used, each, 0.0)
    return (w * each).sum().float(), each.detach().float()


# ------------------------------------------------------------------ the calls

def run(state):
    case = state["case"]
    return {"attention": _run_attention, "step": _run_step, "sample": _run_sample, "distill": _run_distill}[case["op"]](state, case)


def _run_attention(s, case):
    q, k, v, lengths = s["q"], s["k"], s["v"], s.get("lengths")
    with torch.set_grad_enabled(case["train"]):
        if own:
            import thetascan_amd as ts

            out = ts.windowed_attention(q, k, v, window=case["window"], sinks=case["sinks"], lengths=lengths)
        else:
            out = _plain_attention(q, k, v, case["window"], case["sinks"], lengths).to(q.dtype)
    if not case["train"]:
        return out
    return [out.detach(), *torch.autograd.grad([out], [q, k, v], [s["dout"]])]


def _run_step(s, case):
    with torch.no_grad():
        if own:
            import thetascan_amd as ts

            out = ts.windowed_attention_step(s["q"], s["k"], s["v"], s["cache_k"], s["cache_v"], s["positions"],
                                             sinks=case["sinks"])
        else:
            out = _plain_step(s, case["window"], case["sinks"])
    return out, s["cache_k"], s["cache_v"]


def _run_sample(s, case):
    with torch.no_grad():
        if own:
            import thetascan_amd as ts

            return ts.sample_tokens(s["z"], s["u"], temperature=s["temperature"], top_k=s["top_k"], top_p=s["top_p"],
                                    min_p=s["min_p"], softcap=case["cap"] or None)
        return _plain_sample(s, case["cap"])


def _run_distill(s, case):
    if own:
        import thetascan_amd as ts

        loss, each = ts.distill_loss(s["z"], s["ids"], s["lps"], weights=s["weights"], temperature=case["temperature"],
                                     tail=case["tail"], softcap=case["cap"] or None)
    else:
        loss, each = _plain_distill(s, case)
    (dz,) = torch.autograd.grad(loss, [s["z"]])
    return loss.detach(), each, dz


# ------------------------------------------------------------------ what a pass cannot do without

def _pairs(T, window, sinks):
    """Pairs of a query and a key that it sees, of one sequence of T tokens."""
    near = sum(min(i + 1, window) for i in range(T)) if T <= window else window * (window + 1) // 2 + (T - window) * window
    m = max(0, T - window)  # queries i >= window see min(sinks, i - window + 1) sinks too
    s = min(sinks, m)
    return near + s * (s + 1) // 2 + (m - s) * sinks


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "sample":
        N, V = case["N"], case["V"]
        return {"bytes": N * V * es + N * (4 + 8 + 4 + 24 * case["mixed"]), "flops": 6 * N * V}
    if case["op"] == "distill":
        N, V, K = case["N"], case["V"], case["K"]
        return {"bytes": 2 * N * V * es + N * (12 * K + 8), "flops": 8 * N * V}
    H, Hk, d, window, sinks = (case[n] for n in ("H", "Hk", "d", "window", "sinks"))
    if case["op"] == "step":
        held = sum(min(p + 1, sinks + window) for p in _positions(case) if p >= 0)
        B = case["B"]
        return {"bytes": 2 * held * Hk * d * es + B * (2 * H + 4 * Hk) * d * es, "flops": 4 * held * H * d}
    rows = sum(_lengths(case))
    pairs = sum(_pairs(T, window, sinks) for T in _lengths(case))
    wide, narrow = rows * H * d * es, rows * Hk * d * es
    if not case["train"]:
        return {"bytes": 2 * wide + 2 * narrow, "flops": 4 * pairs * H * d}
    # two products forward; the scores again and four products backward
    return {"bytes": 4 * wide + 4 * narrow, "flops": 14 * pairs * H * d}


# ------------------------------------------------------------------ the definitions in 64 bits

def exact(case, seed):
    s = prepare(case, seed)
    s = {n: x.detach() if torch.is_tensor(x) else x for n, x in s.items()}
    with torch.no_grad():
        return {"attention": _exact_attention, "step": _exact_step, "sample": _exact_sample, "distill": _exact_distill}[case["op"]](s, case)


def _exact_attention(s, case):
    """Sequence by sequence, key head by key head and 512 queries at a time, against
    every key before their end."""
    B, H, Hk, T, d, window, sinks = (case[n] for n in ("B", "H", "Hk", "T", "d", "window", "sinks"))
    rep = H // Hk
    train = case["train"]
    shape = {"out": (B, H, T, d), "q": (B, H, T, d), "k": (B, Hk, T, d), "v": (B, Hk, T, d)}
    got = {n: torch.zeros(x, dtype=torch.float64, device="cuda") for n, x in shape.items() if train or n == "out"}
    lengths = s["lengths"].tolist() if "lengths" in s else [T] * B
    for b, length in enumerate(lengths):
        for h in range(Hk):
            heads = slice(h * rep, (h + 1) * rep)
            for i0 in range(0, length, 512):
                i1 = min(length, i0 + 512)
                low = max(0, i0 - window + 1)
                cols = torch.arange(low, i1, device="cuda")
                if low:
                    cols = torch.cat([torch.arange(min(sinks, low), device="cuda"), cols])
                i = torch.arange(i0, i1, device="cuda")[:, None]
                hidden = (cols > i) | ((i - cols >= window) & (cols >= sinks))
                q, k, v = s["q"][b, heads, i0:i1].double(), s["k"][b, h, cols].double(), s["v"][b, h, cols].double()
                P = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                out = P @ v
                got["out"][b, heads, i0:i1] = out
                if not train:
                    continue
                do = s["dout"][b, heads, i0:i1].double()
                dS = P * (do @ v.T - (do * out).sum(-1, keepdim=True)) / math.sqrt(d)
                got["q"][b, heads, i0:i1] = dS @ k
                got["k"][b, h].index_add_(0, cols, (dS.transpose(1, 2) @ q).sum(0))
                got["v"][b, h].index_add_(0, cols, (P.transpose(1, 2) @ do).sum(0))
    return [got[n] for n in ("out", "q", "k", "v")] if train else got["out"]


def _exact_step(s, case):
    """Each sequence's tokens gathered in the order of their positions."""
    B, H, Hk, d, window, sinks = (case[n] for n in ("B", "H", "Hk", "d", "window", "sinks"))
    out = torch.zeros(B, H, 1, d, dtype=torch.float64, device="cuda")
    for b, pos in enumerate(s["positions"].tolist()):
        if pos < 0:
            continue
        seen = list(range(min(sinks, pos + 1))) + list(range(max(sinks, pos + 1 - window), pos + 1))
        at = [p if p < sinks else sinks + (p - sinks) % window for p in seen]
        for cache, new in (("cache_k", "k"), ("cache_v", "v")):
            s[cache][b, :, at[-1]] = s[new][b, :, 0]
        k, v = (s[n][b][:, at].double() for n in ("cache_k", "cache_v"))
        q = s["q"][b].double().reshape(Hk, H // Hk, d)
        out[b] = (torch.softmax(torch.bmm(q, k.transpose(1, 2)) / math.sqrt(d), -1) @ v).reshape(H, 1, d)
    return out, s["cache_k"].double(), s["cache_v"].double()


def _exact_sample(s, case):
    """Row by row: the settings cut a list of tokens in their order, one after the other."""
    N, V = case["N"], case["V"]
    tokens, lps = [], []

    def of(name, n, none):
        x = s[name]
        return x[n].item() if torch.is_tensor(x) else none if x is None else x

    for n in range(N):
        z = s["z"][n].double()
        y = case["cap"] * torch.tanh(z / case["cap"]) if case["cap"] else z
        off = y - y.max()
        weight = torch.round(torch.exp(off / of("temperature", n, 1.0)) * UNIT).long()
        left = torch.argsort(z, descending=True, stable=True)[: of("top_k", n, V)]
        mass = torch.cumsum(weight[left], 0)
        left = left[torch.cat([mass[:1] * 0, mass[:-1]]).double() < of("top_p", n, 1.0) * mass[-1].double()]
        left = left[weight[left].double() >= of("min_p", n, 0.0) * UNIT]
        left = torch.sort(left).values
        mass = torch.cumsum(weight[left], 0)
        place = torch.clamp(torch.floor(s["u"][n].double() * mass[-1].double()).long(), max=mass[-1] - 1)
        token = left[torch.searchsorted(mass, place, right=True)]
        tokens.append(token)
        lps.append(off[token] - torch.logsumexp(off, 0))
    return torch.stack(tokens), torch.stack(lps)


def _exact_distill(s, case):
    N, V, cap, temperature = case["N"], case["V"], case["cap"], case["temperature"]
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    each = torch.zeros(N, dtype=torch.float64, device="cuda")
    dz = torch.zeros(N, V, dtype=torch.float64 if N * V <= 1 << 27 else torch.float32, device="cuda")
    for i in range(0, N, 2048):
        rows = torch.arange(i, min(N, i + 2048), device="cuda")
        rows = rows[s["weights"][rows] != 0]
        z, ids, w, lp = s["z"][rows].double(), s["ids"][rows], s["weights"][rows].double(), s["lps"][rows].double()
        y = cap * torch.tanh(z / cap) if cap else z
        slope = (1.0 - (y / cap) ** 2 if cap else torch.ones_like(y)) / temperature
        lq = torch.log_softmax(y / temperature, -1)
        if not case["tail"]:
            lp = torch.log_softmax(lp, -1)
        teacher = torch.zeros_like(lq).scatter_(-1, ids, lp.exp())
        term = (lp.exp() * (lp - lq.gather(-1, ids))).sum(-1)
        if case["tail"]:
            outside = torch.ones_like(lq).scatter_(-1, ids, 0.0)
            Q = lq.exp() * outside
            q_rest, p_rest = Q.sum(-1), torch.clamp(1.0 - teacher.sum(-1), min=0.0)
            term = term + torch.xlogy(p_rest, p_rest / q_rest)
            # the teacher's rest as the student would spread it
            teacher = teacher + Q * (p_rest / q_rest)[:, None]
        each[rows] = term
        loss = loss + (w * term).sum()
        grad = lq.exp() * teacher.sum(-1, keepdim=True) - teacher
        dz[rows] = (w[:, None] * grad * slope).to(dz.dtype)
    return loss, each, dz

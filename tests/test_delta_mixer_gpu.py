"""The gated delta mixer and the hybrid LM around it, used as a program would:
training steps, a prompt read into a state, one-token steps (eager and captured),
rollouts, their log-probabilities and a step on the policy loss."""
from __future__ import annotations

import pytest
import torch
import torch.nn.functional as F

from tests.test_delta_gpu import reference, rel

pytestmark = pytest.mark.gpu

BF, F32 = torch.bfloat16, torch.float32


def mixer(cuda, dtype, key_heads=2, d_model=256, heads=4, seed=0):
    import thetascan_amd as ts

    torch.manual_seed(seed)
    m = ts.GatedDelta(ts.GatedDeltaConfig(d_model=d_model, n_heads=heads, key_heads=key_heads))
    for p in m.parameters():
        if p.ndim == 2:
            torch.nn.init.normal_(p, std=d_model ** -0.5)
    return m.to(cuda, dtype)


def oracle(m, x, lengths=None):
    """The mixer in float64 on the CPU."""
    w = {n: p.detach().double().cpu() for n, p in m.named_parameters()}
    x = x.detach().double().cpu()
    B, T, D = x.shape
    H, d = m.cfg.n_heads, m.cfg.head_dim

    def heads(name):
        return (x @ w[name].T).view(B, T, -1, d).transpose(1, 2)

    def gate(name):
        return (x @ w[name + ".lin.weight"].T + w[name + ".lin.bias"]).view(B, T, H, -1).transpose(1, 2)

    q, k = (F.normalize(heads(n), dim=-1) for n in ("proj_q.weight", "proj_k.weight"))
    beta, decay = torch.sigmoid(gate("beta")), -F.softplus(gate("decay.g"))
    out, _ = reference(q, k, heads("proj_v.weight"), beta, decay, lengths=lengths)
    out = out / (out.square().mean(-1, keepdim=True) + torch.finfo(torch.float32).eps).sqrt()
    out = out * F.silu(gate("ogate.g"))
    return out.transpose(1, 2).reshape(B, T, D) @ w["proj_out.weight"].T


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,key_heads", [(5, None), (150, 2)])
def test_mixer_matches_float64(cuda, T, key_heads, dtype):
    m = mixer(cuda, dtype, key_heads)
    x = torch.randn(2, T, 256, device=cuda, dtype=dtype, generator=torch.Generator(cuda).manual_seed(1))
    want = oracle(m, x)
    # some eight bf16 roundings on the way (2^-8 each), fp32 products of 256 terms otherwise
    bar = 8 * 2.0 ** -8 if dtype == BF else 2048 * 2.0 ** -24
    assert rel(m(x), want) <= bar
    lengths = torch.tensor([T, T // 2], device=cuda)
    y = m(x, lengths=lengths)
    assert rel(y[0], want[0]) <= bar and rel(y[1, :T // 2], want[1, :T // 2]) <= bar
    assert not bool(y[1, T // 2:].any())


@pytest.mark.parametrize("dtype", [BF, F32])
def test_states_steps_and_captured_steps(cuda, dtype):
    import thetascan_amd as ts
    from thetascan_amd import _lib

    m = mixer(cuda, dtype)
    x = torch.randn(3, 90, 256, device=cuda, dtype=dtype, generator=torch.Generator(cuda).manual_seed(2))
    bar = 8 * 2.0 ** -8 if dtype == BF else 2048 * 2.0 ** -24
    with torch.no_grad():
        whole = m(x)
        prompt, state = m(x[:, :80], state=m.initial_state())
        assert rel(prompt, whole[:, :80]) <= bar and state.position == 80 and state.batch == 3
        s = ts.ThetaScanState.from_state_dict(state.state_dict())
        eager = []
        for t in range(80, 90):
            with _lib.record_launches() as recs:
                y, s = m(x[:, t:t + 1], state=s)
            assert "ts_delta_step" in {r[0] for r in recs}
            eager.append(y)
        assert rel(torch.cat(eager, 1), whole[:, 80:]) <= bar
        dec = ts.DecodeGraph(m, state)
        for i, t in enumerate(range(80, 90)):
            y = dec.step(x[:, t:t + 1]).clone()
            m(x[:, :7])
            torch.cuda.synchronize()
            # (a captured library product may take another solution: each of the
            # step's eight rounded rows -- queries, keys, values, both gates, the
            # memory's, the gated and the projected ones -- then falls on a
            # neighbour where it lay near the middle, up to 2^-8 apart each)
            assert rel(y, eager[i]) <= (bar if dtype == BF else 0.0)
        fin = dec.state()
    assert fin.position == 90
    # (the state is made of four of them: keys, values, write strengths, retentions)
    for a, b in zip(fin._tensors(), s._tensors()):
        assert rel(a, b) <= (4 * 2.0 ** -8 if dtype == BF else 0.0)


def test_compiled_mixer_is_the_eager_one(cuda):
    m = mixer(cuda, BF)
    x = torch.randn(2, 70, 256, device=cuda, dtype=BF)
    y = m(x)
    z = torch.compile(m, backend="aot_eager", fullgraph=True)(x)
    assert torch.equal(y, z)
    grads = [torch.autograd.grad(t, list(m.parameters()), torch.ones_like(t)) for t in (y, z)]
    for a, b in zip(*grads):
        assert torch.equal(a, b)


def test_refused_states(cuda):
    m = mixer(cuda, F32)
    x = torch.randn(2, 4, 256, device=cuda)
    with pytest.raises(RuntimeError, match="without autograd"):
        m(x, state=m.initial_state())
    with torch.no_grad():
        _, s = m(x, state=m.initial_state())
        with pytest.raises(ValueError, match="holds 2 sequences"):
            m(x[:1], state=s)
        with pytest.raises(ValueError, match="another configuration"):
            mixer(cuda, F32, key_heads=4)(x, state=s)
        with pytest.raises(ValueError, match="no lengths"):
            m(x, state=s, lengths=torch.tensor([4, 4], device=cuda))
        y, same = m(x[:, :0], state=s)
        assert y.shape == (2, 0, 256) and same is s


def test_autocast_trains_an_fp32_mixer(cuda):
    m = mixer(cuda, F32)
    x = torch.randn(2, 70, 256, device=cuda)
    with torch.autocast("cuda", torch.bfloat16):
        y = m(x)
    y.float().square().mean().backward()
    assert rel(y, oracle(m, x)) <= 12 * 2.0 ** -8
    assert all(p.grad is not None and bool(torch.isfinite(p.grad).all()) for p in m.parameters())


@pytest.mark.parametrize("memory", ["theta", "delta"])
def test_language_model_learns_from_rollouts(cuda, memory):
    """Sampling, log-probabilities, the policy loss against its definition on the
    model's own logits, and an optimizer step that raises what was rewarded."""
    from thetascan_amd import hybrid_lm as lm, _lib

    torch.manual_seed(3)
    model = lm.HybridLM(memory=memory).to(cuda, BF)
    g = torch.Generator(cuda).manual_seed(4)
    ids = torch.randint(0, lm.VOCAB, (4, 40), device=cuda, generator=g)
    for _ in range(8):  # sampled successors
        with torch.no_grad():
            p = torch.softmax(model(ids)[:, -1], -1)
        ids = torch.cat([ids, torch.multinomial(p, 1, generator=g)], 1)
    idx, tokens = ids[:, :-1], ids[:, 1:]
    old = model.log_probs(idx, tokens)
    with torch.no_grad():
        full = torch.log_softmax(model(idx).double(), -1).gather(-1, tokens[..., None])[..., 0]
    assert float((old.double() - full).abs().max()) < 1e-4
    weights = torch.zeros(4, 47, device=cuda)
    weights[:, 39:] = 1.0 / 32
    adv = torch.tensor([1.0, -1.0, 0.5, -0.5], device=cuda)[:, None].expand(4, 47)
    with _lib.record_launches() as recs:
        loss, lp = model.policy_loss(idx, tokens, old, adv, ref_log_probs=old - 0.1, weights=weights, kl=0.02)
        loss.backward()
    names = {r[0] for r in recs}
    assert {"ts_policy_loss_fwd", "ts_policy_loss_bwd"} <= names
    assert ({"ts_delta_fwd", "ts_delta_bwd"} <= names) == (memory == "delta")
    # ratio one, and the KL term of a constant distance of 0.1
    want = -float((weights * adv).sum()) + 0.02 * (float(torch.tensor(-0.1).double().exp()) + 0.1 - 1.0)
    assert abs(float(loss) - want) < 1e-4
    assert all(bool(torch.isfinite(p.grad).all()) for p in model.parameters() if p.grad is not None)
    assert float(model.blocks[4].attn.proj_out.weight.grad.abs().sum() if memory == "delta"
                 else model.blocks[4].attn._core.proj_out.weight.grad.abs().sum()) > 0.0


def test_language_model_with_delta_memories_trains(cuda):
    from thetascan_amd import hybrid_lm as lm

    torch.manual_seed(5)
    model = lm.HybridLM(memory="delta").to(cuda, BF)
    ids = torch.randint(0, lm.VOCAB, (2, 130), device=cuda, generator=torch.Generator(cuda).manual_seed(6))
    model(ids[:, :-1], ids[:, 1:]).backward()
    grads = [p.grad for p in model.parameters() if p.requires_grad]
    assert all(x is not None and bool(torch.isfinite(x).all()) for x in grads)
    with pytest.raises(ValueError, match="memory must be"):
        lm.HybridLM(memory="gn")


@pytest.mark.parametrize("dtype", [BF, F32])
def test_padding_is_not_read(cuda, dtype):
    """Whatever the padding holds: outputs, the input's and the weights' gradients as
    with zeros there."""
    m = mixer(cuda, dtype)
    x = torch.randn(3, 70, 256, device=cuda, dtype=dtype, generator=torch.Generator(cuda).manual_seed(1))
    lengths = torch.tensor([70, 33, 0], device=cuda)
    past = (torch.arange(70, device=cuda) >= lengths[:, None])[..., None]

    def run(fill):
        xi = x.masked_fill(past, fill).requires_grad_()
        y = m(xi, lengths=lengths)
        return [y, *torch.autograd.grad(y.float().square().sum(), (xi, *m.parameters()))]

    for a, b in zip(run(0.0), run(float("nan"))):
        assert torch.equal(a, b)
    assert not run(float("nan"))[0].masked_select(past).any()
    with pytest.raises(ValueError, match="lengths"):
        m(x, lengths=lengths[:2])


def test_no_tokens(cuda):
    m = mixer(cuda, F32)
    assert m(torch.zeros(2, 0, 256, device=cuda)).shape == (2, 0, 256)
    with torch.no_grad():
        y, s = m(torch.zeros(2, 0, 256, device=cuda), m.initial_state())
    assert y.shape == (2, 0, 256) and s.position == 0

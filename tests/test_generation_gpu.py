"""The hybrid LM generates, and learns from rollouts and a teacher, by the operators together.

A generated token's log-probability (prompt, then single tokens against caches and states)
and that of the whole sequence at once are the same sums in another order: in fp32, logits of
a few ones through nine layers, each off by some 2^-20 of its values, so 1e-3 is far above
what rounding gives and far below what a wrong key, position or slot does.
"""
from __future__ import annotations

import pytest
import torch

from thetascan_amd import hybrid_lm as lm

pytestmark = pytest.mark.gpu


def _model(memory, dtype, cuda, seed=0, **kw):
    torch.manual_seed(seed)
    model = lm.HybridLM(memory=memory, **kw)
    for block in model.blocks:  # (the output projections start at zero: nothing would be mixed)
        out = block.attn.proj if not block.theta else getattr(block.attn, "proj_out", None) or block.attn._core.proj_out
        torch.nn.init.normal_(out.weight, std=0.03)
        torch.nn.init.normal_(block.mlp.proj.weight, std=0.03)
    torch.nn.init.normal_(model.tok_emb.weight, std=0.05)
    return model.to(cuda, dtype)


@pytest.mark.parametrize("memory", ["theta", "delta"])
@pytest.mark.parametrize("prompt,window,sinks", [(1, 8, 2), (5, 16, 0), (40, 16, 3), (70, 1, 1)])
def test_generated_tokens_have_the_whole_sequences_probabilities(cuda, memory, prompt, window, sinks):
    model = _model(memory, torch.float32, cuda, window=window, sinks=sinks)
    g = torch.Generator().manual_seed(1)
    idx = torch.randint(0, lm.VOCAB, (3, prompt), generator=g).to(cuda)
    u = torch.rand(3, 30, generator=g).to(cuda)
    tokens, lps = model.generate(idx, u, temperature=0.9, top_p=0.95)
    whole = torch.cat([idx, tokens], 1)
    want = model.log_probs(whole[:, :-1], whole[:, 1:])[:, prompt - 1:]
    print(f"{memory} {prompt}: {float((lps - want).abs().max()):.2e}", flush=True)
    assert torch.allclose(lps, want, atol=1e-3)
    # the same numbers draw the same tokens; none of the settings left: another
    again, _ = model.generate(idx, u, temperature=0.9, top_p=0.95)
    assert torch.equal(tokens, again)
    best, _ = model.generate(idx, u, temperature=0.0)
    z = model(torch.cat([idx, best], 1))[:, prompt - 1:-1]
    assert (z.gather(-1, best[..., None])[..., 0] >= z.amax(-1) - 1e-3).all()


@pytest.mark.parametrize("memory", ["theta", "delta"])
def test_rollouts_and_a_teacher_train_a_student(cuda, memory):
    teacher = _model(memory, torch.bfloat16, cuda, seed=1)
    student = _model(memory, torch.bfloat16, cuda, seed=2, window=24, sinks=2)
    g = torch.Generator().manual_seed(3)
    idx = torch.randint(0, lm.VOCAB, (4, 33), generator=g).to(cuda)
    tokens, old = student.generate(idx, torch.rand(4, 20, generator=g).to(cuda), top_k=50)
    whole = torch.cat([idx, tokens], 1)
    x, y = whole[:, :-1], whole[:, 1:]
    answers = torch.zeros(x.shape, device=cuda)
    answers[:, 32:] = 1.0 / (4 * 20)
    full_old = torch.zeros(x.shape, device=cuda)
    full_old[:, 32:] = old
    for p in student.parameters():
        p.grad = None
    loss, lp = student.policy_loss(x, y, full_old, torch.randn(x.shape, generator=g).to(cuda), weights=answers)
    loss.backward()
    rollout = {n: p.grad.clone() for n, p in student.named_parameters() if p.grad is not None}
    ids, lps = teacher.top_log_probs(x, 16)
    student.zero_grad(set_to_none=True)
    loss, each = student.distill_loss(x, ids, lps, weights=answers)
    loss.backward()
    assert torch.isfinite(loss) and (each >= -1e-5).all() and not each[:, :32].any()
    for n, p in student.named_parameters():
        if p.grad is not None:
            assert torch.isfinite(p.grad.float()).all() and torch.isfinite(rollout[n].float()).all(), n
    assert student.blocks[0].attn.c_k.weight.grad.float().abs().max() > 0
    # the teacher's own answers against itself, with all of its tokens: no divergence beyond rounding
    ids, lps = teacher.top_log_probs(x, lm.VOCAB)
    _, own = teacher.distill_loss(x, ids, lps)
    # (log-probabilities of some 7 in fp32: 2^-21 of them at most a token)
    assert own.abs().max() < 2e-5

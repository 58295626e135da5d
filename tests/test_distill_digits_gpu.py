"""The digits of a row's distillation loss where teacher and student are near, so that the loss
is small against the terms that it is formed from (ts_distill_fwd), against float64.

What each rounding moves a loss by is the loss's slope there, and the roundings of a row are
independent of each other, so that they add up as their squares do:

* another token's exponential, off by (|x - max| + 4) 2^-24 of itself (its argument's rounding, and its
  own): q |1 - P_r / Q_r| times that;
* the others' sum by lanes, V / 256 + 32 additions on a lane's way, each off by 2^-24 of the sum at
  most: |Q_r - P_r| times that;
* a capped logit, off by 2^-22 of itself and of the cap's part in it: |dloss / dx| times that;
* the loss's own rounding: 2^-24 of it.

All else (shares, distances, logarithms, the teacher's tokens' exponentials) is fp64.  The root mean square
over the rows has to be within four times the model's.
"""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def definition(z, ids, lps, temperature, cap, tail):
    """(loss of each row, its rounding's expected size) in float64."""
    V = z.shape[1]
    z = z.double()
    y = cap * torch.tanh(z / cap) if cap else z
    x = y / temperature
    lq = torch.log_softmax(x, -1)
    q = lq.exp()
    P = lps.double().exp()
    if not tail:
        P = P / P.sum(-1, keepdim=True)
    teacher = torch.zeros_like(q).scatter_(-1, ids, P)
    outside = torch.ones_like(q).scatter_(-1, ids, 0.0)
    Q = (q * outside).sum(-1)
    left = (1.0 - P.sum(-1)).clamp(min=0.0) if tail else torch.zeros_like(Q)
    each = (P * (P.log() - lq.gather(-1, ids))).sum(-1) + torch.special.xlogy(left, left / Q)
    ratio = (left / Q)[:, None]
    far = (x - x.amax(-1, keepdim=True)).abs()
    own = (outside * q * (1.0 - ratio).abs() * (far + 4.0) * 2.0 ** -24).square().sum(-1)
    own += ((Q - left).abs() * 2.0 ** -24).square() * (V / 256 + 32)
    if cap:
        slope = q * (1.0 - outside * ratio) - teacher
        own += (slope * x * 2.0 ** -22).square().sum(-1)
    own += (each.abs() * 2.0 ** -24).square()
    return each, own


@pytest.mark.parametrize("N,V,K,temperature,cap,tail", [
    (512, 32768, 64, 2.0, None, True), (64, 32768, 64, 2.0, None, True), (512, 8192, 100, 1.0, 30.0, True),
    (64, 50257, 64, 1.0, None, False), (600, 1024, 32, 1.0, None, True), (600, 1024, 32, 1.0, 30.0, True),
    (600, 2048, 200, 2.0, None, True), (20000, 1024, 32, 2.0, None, True), (20000, 777, 8, 1.0, None, False)])
@pytest.mark.parametrize("spread", [0.5, 0.02])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_small_losses_have_their_digits(cuda, N, V, K, temperature, cap, tail, spread, dtype):
    import thetascan_amd as ts

    g = torch.Generator(device=cuda).manual_seed(V + K)
    z = (2.5 * torch.randn(N, V, generator=g, device=cuda)).to(dtype)
    y = z.double()
    y = cap * torch.tanh(y / cap) if cap else y
    y = (y + spread * torch.randn(N, V, generator=g, device=cuda)) / temperature
    lps, ids = torch.log_softmax(y, -1).topk(K, -1)
    lps = lps.float()
    _, each = ts.distill_loss(z, ids, lps, temperature=temperature, softcap=cap, tail=tail)
    want, square = definition(z, ids, lps, temperature, cap, tail)
    err, bar = float((each.double() - want).square().mean().sqrt()), 4.0 * float(square.mean().sqrt())
    print(f"losses of {float(want.mean()):.2e}: off by {err:.2e}, {err / float(want.square().mean().sqrt()):.1e} of them; "
          f"{err / bar:.3f} of the bar", flush=True)
    assert err <= bar
    # with the gradient beside it, the same
    leaf = z.requires_grad_()
    assert torch.equal(ts.distill_loss(leaf, ids, lps, temperature=temperature, softcap=cap, tail=tail)[1], each)


@pytest.mark.parametrize("N,V,K,temperature", [(600, 1024, 32, 1.0), (600, 2048, 200, 2.0), (20000, 1024, 32, 2.0),
                                               (20000, 1999, 100, 1.0), (512, 32768, 64, 2.0), (64, 50257, 64, 1.0)])
@pytest.mark.parametrize("spread", [0.5, 0.02])
def test_the_others_gradients_have_their_digits(cuda, N, V, K, temperature, spread):
    """q (1 - P_r / Q_r) of the tokens that are none of the teacher's: an exponential's own error (as above, with
    eight 2^-24 for the products and the result), and of P_r / Q_r what the others' sum is off by: a sum by 256
    lanes or more of fp32 terms, whose independent errors average out over the lanes (V / 2^16 of 2^-48), and
    eight additions of the lanes' sums; rows of up to 2048 are summed in fp64.  Four times that."""
    import thetascan_amd as ts

    g = torch.Generator(device=cuda).manual_seed(V + K)
    z = (2.5 * torch.randn(N, V, generator=g, device=cuda)).requires_grad_()
    y = (z.detach().double() + spread * torch.randn(N, V, generator=g, device=cuda)) / temperature
    lps, ids = torch.log_softmax(y, -1).topk(K, -1)
    lps = lps.float()
    (dz,) = torch.autograd.grad(ts.distill_loss(z, ids, lps, temperature=temperature)[0], z)
    x = z.detach().double() / temperature
    q = torch.softmax(x, -1).scatter_(-1, ids, 0.0)
    Q, left = q.sum(-1, keepdim=True), (1.0 - lps.double().exp().sum(-1, keepdim=True)).clamp(min=0.0)
    ratio = left / Q
    own = ((x - x.amax(-1, keepdim=True)).abs() + 8.0).square() * (1.0 - ratio).square()
    own += ratio.square() * ((V / 65536 + 8) if V > 2048 else 1.0)
    square = (q * 2.0 ** -24).square() * own
    err = torch.where(q > 0, N * temperature * dz.double() - q * (1.0 - ratio), 0.0)
    size = float((q * (1.0 - ratio)).square().sum().sqrt())
    err, bar = float(err.square().sum().sqrt()), 4.0 * float(square.sum().sqrt())
    print(f"off by {err / size:.1e} of them; {err / bar:.3f} of the bar", flush=True)
    assert err <= bar

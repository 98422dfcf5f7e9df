"""The distillation step: attention under autograd, the loss and gradients of a small stack against a float32 copy of it in
plain torch, the orthogonalised update against its formula, and a few steps of the example, whose loss falls."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def say(*a):
    print(*a, flush=True)


def plain_attention(q, k, v, scale, lens=None):
    B, H, T, _ = q.shape
    k, v = (x.repeat_interleave(H // x.shape[1], 1) for x in (k, v))
    t = torch.arange(T, device=q.device)
    n = torch.full((B,), T, device=q.device) if lens is None else lens
    live = (t[None] < n[:, None]).view(B, 1, T, 1)
    seen = (t[None, :] <= t[:, None]) & live
    s = (q @ k.transpose(-1, -2).contiguous() * scale).masked_fill(~seen & live, -math.inf)
    return torch.where(live, torch.softmax(torch.where(live, s, 0.0), -1) @ v, 0.0)


def test_attention_under_autograd():
    from lookatmyquant_amd import distill

    g = torch.Generator(device="cuda").manual_seed(1)
    x = [torch.randn(3, 90, h, 128, generator=g, device="cuda").bfloat16().transpose(1, 2).requires_grad_() for h in (6, 2, 2)]
    lens = torch.tensor([90, 0, 41], dtype=torch.int32, device="cuda")
    f = [t.detach().float().requires_grad_() for t in x]
    for weight in (None, torch.randn(3, 6, 90, 128, generator=g, device="cuda")):
        for t in x + f:
            t.grad = None
        out, want = distill.attention(*x, 0.1, lens), plain_attention(*f, 0.1, lens)
        # a sum's gradient arrives as one expanded value
        (out.float() if weight is None else out.float() * weight).sum().backward()
        (want if weight is None else want * weight).sum().backward()
        for a, b in zip([out] + [t.grad for t in x], [want] + [t.grad for t in f]):
            # bf16 results of bf16-rounded probabilities and dS: a few units of 2^-8 in the norm
            assert float((a.float() - b).norm().detach()) <= 4 * 2.0 ** -8 * float(b.norm().detach())


def small():
    from lookatmyquant_amd import stack

    sh = stack.Shape(hidden=256, heads=4, kv_heads=2, head_dim=128, inter=512, layers=1, vocab=700)
    dev = torch.device("cuda")
    w = {k: v * (6.0 if v.dim() == 2 else 1.0) for k, v in stack.layer_weights(0, sh, dev).items()}
    g = torch.Generator(device="cuda").manual_seed(2)
    emb = (torch.randn(sh.vocab, sh.hidden, generator=g, device="cuda") * 0.1).bfloat16()
    tokens = torch.randint(0, sh.vocab, (3, 70), generator=g, device="cuda")
    rope = tuple(t.to(dev) for t in stack.rope_tables(70, sh, dev))
    return sh, w, emb, tokens, rope


def test_loss_and_gradients_of_a_stack(monkeypatch):
    """Every matrix's gradient of the weighted KL against the same stack in float32 (its attention and loss plain torch):
    bf16 activations and their gradients are rounded to 2^-8 some ten times on the way."""
    from lookatmyquant_amd import distill, stack

    sh, w, emb, tokens, rope = small()
    g = torch.Generator(device="cuda").manual_seed(3)
    ref = (torch.randn(3, 70, sh.vocab, generator=g, device="cuda") * 2).bfloat16()
    lens = torch.tensor([70, 33, 1], dtype=torch.int32, device="cuda")
    t = torch.arange(70, device="cuda")
    wt = ((t < lens[:, None]) & (t >= 0)).float() * (1 + t % 3)
    mats = list(stack.matrix_shapes(sh))
    for nm in mats:
        w[nm] = w[nm].detach().requires_grad_()
    loss = distill.loss_and_grads([w], emb, tokens, ref, sh, rope, wt, lens)
    f = {k: v.detach().float().requires_grad_(k in mats) for k, v in w.items()}
    monkeypatch.setattr(distill, "attention", plain_attention)
    out = distill.logits([f], emb.float(), tokens, sh, tuple(r.float() for r in rope), lens)
    p, s = torch.log_softmax(ref.float(), -1), torch.log_softmax(out, -1)
    want = (wt * (p.exp() * (p - s)).sum(-1)).sum() / wt.sum()
    want.backward()
    say(f"loss {float(loss):.5f}, in float32 {float(want.detach()):.5f}")
    assert abs(float(loss) - float(want.detach())) <= 10 * 2.0 ** -8 * float(want.detach())
    for nm in mats:
        off = float((w[nm].grad.float() - f[nm].grad).norm() / f[nm].grad.norm())
        say(f"  {nm} {off:.4f}")
        assert off <= 10 * 2.0 ** -8, nm


def test_update_follows_its_formula():
    from lookatmyquant_amd import distill
    from lookatmyquant_amd import engine as E

    g = torch.Generator(device="cuda").manual_seed(4)
    P = [torch.randn(*s, generator=g, device="cuda").bfloat16() for s in ((64, 200), (300, 90), (64, 200))]
    opt = distill.Muon(P, lr=0.01, momentum=0.9)
    master, mom = [p.float() for p in P], [torch.zeros_like(p, dtype=torch.float32) for p in P]
    for _ in range(3):
        G = [torch.randn(p.shape, generator=g, device="cuda").bfloat16() for p in P]
        for i, (p, x) in enumerate(zip(P, G)):
            p.grad = x.clone()
            mom[i] = 0.9 * mom[i] + x.float()
            U = E.orthogonalize(x.float() + 0.9 * mom[i]).float()
            master[i] = master[i] - 0.01 * max(1.0, p.shape[0] / p.shape[1]) ** 0.5 * U
        opt.step()
        for p, m, x in zip(P, master, opt.master):
            assert p.grad is None
            # the momentum's products and sums may round differently: 2^-22 of it, carried by the orthogonalisation to
            # units of bf16 in the update here and there
            assert float((x - m).norm()) <= 2.0 ** -8 * 0.01 * 2 * math.sqrt(min(p.shape)) + 1e-6 * float(m.norm())
            assert torch.equal(p, x.bfloat16())
    with pytest.raises(ValueError):
        distill.Muon([torch.zeros(4, dtype=torch.bfloat16, device="cuda")])
    with pytest.raises(ValueError):
        distill.Muon([torch.zeros(4, 4, device="cuda")])


def test_example_lowers_the_loss():
    from lookatmyquant_amd import distill

    losses = distill.main(["--steps", "6"])
    assert all(math.isfinite(x) for x in losses) and losses[-1] < 0.8 * losses[0]

"""The distillation step of fine-tuning on the gfx950 kernels (finetune.py of the reference trains the real weights behind a
build's codes against the original model's logits; finetune_lib.rounded puts them back onto codes): a decoder stack's
forward that torch can differentiate, the KL loss with its gradient, and an orthogonalised update.

    attention(q, k, v, scale, lens=None)   causal grouped-query attention with a gradient (engine.attention_causal_lse and
                                           attention_causal_grad)
    logits(weights, emb, tokens, sh, rope, lens=None)
                                           the stack's next-token logits, bf16, through the tied embedding
    loss_and_grads(...)                    one batch: the mean KL against reference logits, gradients left in the weights
    Muon(params, lr, momentum, nesterov)   the update: a momentum of each matrix's gradient, orthogonalised
                                           (engine.orthogonalize, matrices of one shape as one batch), bf16 weights held
                                           in float32

    python -m lookatmyquant_amd.distill --layers 1 --steps 4

quantizes a small random-initialised stack as the build does, then distils the quantized weights (as real numbers) towards
the original stack, and prints the loss of every step. The layers' matrix products, norms, rotary embedding and gate are
torch's; everything else on the way is this package's kernels.
"""

from __future__ import annotations

import torch

from . import engine as E
from . import stack


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, lens):
        out, kept = E.attention_causal_lse(q, k, v, scale, lens)
        ctx.save_for_backward(q, k, v, out, *kept, lens)
        ctx.scale = scale
        return out

    @staticmethod
    def backward(ctx, dout):
        q, k, v, out, lse, rest, lens = ctx.saved_tensors
        if dout.stride(-1) != 1 or any(s % 8 for s in dout.stride()[:3]) or dout.data_ptr() % 16:
            dout = dout.contiguous()  # e.g. a sum's gradient, one value for all
        return (*E.attention_causal_grad(dout, q, k, v, out, E.AttentionKept(lse, rest), ctx.scale, lens), None, None)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: float, lens: torch.Tensor | None = None):
    """Causal grouped-query attention of [B, heads, T, 128] bf16 q and [B, kv heads, T, 128] k, v, differentiable in all
    three; lens int32 [B] or None: tokens past a sequence's length have output and gradients 0. Returns [B, heads, T, 128]."""
    return _Attention.apply(q, k, v, float(scale), lens)


def _norm(x, g, eps):
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + eps)).to(x.dtype) * g


def _rope(x, cos, sin):
    h = x.shape[-1] // 2
    return x * cos + torch.cat([-x[..., h:], x[..., :h]], -1) * sin


def _layer(h, w, sh, rope, lens):
    B, T, _ = h.shape
    lin = torch.nn.functional.linear
    x = _norm(h, w["input_layernorm"], sh.eps)
    cos, sin = (t[:T] for t in rope)
    heads = lambda name, n: lin(x, w[f"self_attn.{name}_proj"]).view(B, T, n, sh.head_dim).transpose(1, 2)
    q = _rope(_norm(heads("q", sh.heads), w["self_attn.q_norm"], sh.eps), cos, sin)
    k = _rope(_norm(heads("k", sh.kv_heads), w["self_attn.k_norm"], sh.eps), cos, sin)
    a = attention(q, k, heads("v", sh.kv_heads), sh.head_dim ** -0.5, lens)
    h = h + lin(a.transpose(1, 2).reshape(B, T, -1), w["self_attn.o_proj"])
    x = _norm(h, w["post_attention_layernorm"], sh.eps)
    m = torch.nn.functional.silu(lin(x, w["mlp.gate_proj"])) * lin(x, w["mlp.up_proj"])
    return h + lin(m, w["mlp.down_proj"])


def logits(weights: list, emb: torch.Tensor, tokens: torch.Tensor, sh: stack.Shape, rope, lens=None) -> torch.Tensor:
    """The stack's logits [B, T, vocab] (bf16) of token ids [B, T]: weights a list of the layers' weights
    (stack.layer_weights), emb [vocab, hidden] tied to the output."""
    h = emb[tokens]
    for w in weights:
        h = _layer(h, w, sh, rope, lens)
    return torch.nn.functional.linear(_norm(h, torch.ones_like(h[0, 0]), sh.eps), emb)


def loss_and_grads(weights, emb, tokens, ref_logits, sh, rope, w=None, lens=None) -> torch.Tensor:
    """One batch: the weighted mean KL of the stack's logits against ref_logits [B, T, vocab] (w [B, T] token weights, 0
    for prompts and padding; None: all 1), a float32 scalar on the device; the gradients are added to the weights'
    .grad. Nothing synchronises."""
    out = logits(weights, emb, tokens, sh, rope, lens)
    rows = lambda x: x.detach().reshape(-1, x.shape[-1])
    _, loss, grad = E.kl_rows_grad(rows(ref_logits), rows(out), None if w is None else w.reshape(-1))
    out.backward(grad.view_as(out))
    return loss


class Muon:
    """The update of weight matrices along orthogonalised momenta: with G a matrix's gradient,
        M = momentum M + G,   D = G + momentum M (nesterov) or M,   W -= lr sqrt(max(1, rows / cols)) orthogonalize(D).
    params: bf16 matrices on the GPU; each keeps a float32 copy that the updates accumulate in and a float32 momentum.
    Matrices of one shape are orthogonalised as one batch. step() takes every .grad and clears it."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, steps: int = 5):
        self.params = list(params)
        if any(p.dim() != 2 or p.dtype != torch.bfloat16 or not p.is_cuda for p in self.params):
            raise ValueError("the orthogonalised update is of bf16 matrices on the GPU")
        self.lr, self.momentum, self.nesterov, self.steps = lr, momentum, nesterov, steps
        self.master = [p.detach().float() for p in self.params]
        self.state = [torch.zeros_like(m) for m in self.master]

    @torch.no_grad()
    def step(self):
        shapes: dict = {}
        for i, p in enumerate(self.params):
            if p.grad is not None:
                shapes.setdefault(tuple(p.shape), []).append(i)
        for (rows, cols), at in shapes.items():
            D = torch.empty(len(at), rows, cols, dtype=torch.float32, device=self.params[at[0]].device)
            for d, i in zip(D, at):
                G = self.params[i].grad.float()
                M = self.state[i].mul_(self.momentum).add_(G)
                torch.add(G, M, alpha=self.momentum, out=d) if self.nesterov else d.copy_(M)
                self.params[i].grad = None
            U = E.orthogonalize(D, self.steps)
            for u, i in zip(U, at):
                self.master[i].add_(u.float(), alpha=-self.lr * max(1.0, rows / cols) ** 0.5)
                self.params[i].copy_(self.master[i])


def quantized_start(sh: stack.Shape, tokens: torch.Tensor, layers: int, weight_seed: int = 5000):
    """(the original layers' weights, the same with every matrix as the build's codes decode it, the embedding) of a
    random-initialised stack quantized on calibration tokens."""
    b = stack.StackBuild(tokens, sh, layers=layers, keep=layers, weight_seed=weight_seed)
    teacher, student = [], []
    for i in range(layers):
        b.layer()
        w = stack.layer_weights(i, sh, b.dev, weight_seed)
        teacher.append(w)
        quant = {nm: q for s in range(len(stack.STAGES)) for nm, q in b.kept[(i, s)].get("Wq", {}).items()}
        student.append({nm: quant.get(nm, x).clone() for nm, x in w.items()})
    g = torch.Generator(device=b.dev).manual_seed(weight_seed * 1000 + 999)
    emb = torch.randn(sh.vocab, sh.hidden, generator=g, device=b.dev) * sh.std
    return teacher, student, emb.to(torch.bfloat16)


def main(argv=None):
    import argparse

    ap = argparse.ArgumentParser(prog="python -m lookatmyquant_amd.distill")
    ap.add_argument("--layers", type=int, default=1)
    ap.add_argument("--steps", type=int, default=4)
    ap.add_argument("--batch", type=int, default=8)
    ap.add_argument("--length", type=int, default=256)
    ap.add_argument("--prompt", type=int, default=32, help="leading tokens of a sequence that carry no weight")
    ap.add_argument("--lr", type=float, default=2e-3)
    args = ap.parse_args(argv)
    sh = stack.Shape(hidden=512, heads=8, kv_heads=4, head_dim=128, inter=1024, layers=args.layers, vocab=4096)
    dev = E._abi.device()
    g = torch.Generator().manual_seed(1)
    calib = torch.randint(0, sh.vocab, (8, 256), generator=g)
    teacher, student, emb = quantized_start(sh, calib, args.layers)
    rope = tuple(t.to(dev) for t in stack.rope_tables(args.length, sh, dev))
    mats = [w[nm].requires_grad_() for w in student for nm in stack.matrix_shapes(sh)]
    opt = Muon(mats, args.lr)
    tokens = torch.randint(0, sh.vocab, (args.batch, args.length), generator=g).to(dev)
    lens = torch.full((args.batch,), args.length, dtype=torch.int32)
    lens[1::2] = args.length * 3 // 4  # half the batch padded
    t = torch.arange(args.length)
    w = ((t >= args.prompt) & (t < lens[:, None])).float().to(dev)
    lens = lens.to(dev)
    with torch.no_grad():
        ref = logits(teacher, emb, tokens, sh, rope, lens)
    losses = []
    for step in range(args.steps):
        losses.append(float(loss_and_grads(student, emb, tokens, ref, sh, rope, w, lens)))
        print(f"step {step}: KL {losses[-1]:.6f}", flush=True)
        opt.step()
    return losses


if __name__ == "__main__":
    main()

"""Performance cases of the distillation step's operators: the attention that training runs (forward and backward), the
KL loss with its gradient, and the orthogonalised update of a weight matrix.

    own                 False: the operators in plain torch, in 32 bits; True: the package's entry points
    listed()            the cases, dicts of plain values
    draw(rng)           one more case of the same ranges
    prepare(case, seed) what a program holds before the call: the inputs, from the seed
    run(state)          one pass, its outputs whole
    work(case)          bytes and operations one pass cannot do without
    exact(case, seed)   the same outputs from the definitions in 64 bits
"""

from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
HEAD = 128  # head dim of the forwards' attention
COEFFS = (3.4445, -4.7750, 2.0315)  # the quintic of the orthogonalisation
STEPS = 5
TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


def listed() -> list[dict]:
    return [
        # One short odd prompt of a small model's heads: a few workgroups, the launches count.
        {"name": "attention_1x45", "kind": "attention", "B": 1, "T": 45, "heads": 8, "kv": 2, "ragged": False},
        # A padded batch of odd length with sequences of every size, one empty and one of a single token among them.
        {"name": "attention_ragged_12x733", "kind": "attention", "B": 12, "T": 733, "heads": 16, "kv": 16,
         "ragged": True},
        # Four calibration sequences of the benchmark's layer (32 query, 8 key/value heads, 2,048 tokens).
        {"name": "attention_4x2048", "kind": "attention", "B": 4, "T": 2048, "heads": 32, "kv": 8, "ragged": False},
        # One long sequence of the same layer.
        {"name": "attention_1x8192", "kind": "attention", "B": 1, "T": 8192, "heads": 32, "kv": 8, "ragged": False},
        # A handful of answer tokens at the benchmark's vocabulary: few rows, each of them long.
        {"name": "kl_5", "kind": "kl", "T": 5, "V": 151936, "dtype": "bf16", "prompt": 0},
        # A window of 2,048 tokens at the same vocabulary, its first quarter a prompt that carries no weight.
        {"name": "kl_2048", "kind": "kl", "T": 2048, "V": 151936, "dtype": "bf16", "prompt": 512},
        # float32 logits of an odd vocabulary: rows that start at any alignment.
        {"name": "kl_f32_333x32003", "kind": "kl", "T": 333, "V": 32003, "dtype": "f32", "prompt": 20},
        # A small projection's accumulated gradient: latency.
        {"name": "ortho_128x320", "kind": "ortho", "batch": 1, "m": 128, "n": 320, "dtype": "f32"},
        # Odd sizes and more rows than columns.
        {"name": "ortho_1001x333", "kind": "ortho", "batch": 1, "m": 1001, "n": 333, "dtype": "f32"},
        # k_proj and v_proj of the benchmark's layer, one batch.
        {"name": "ortho_2x1024x2560", "kind": "ortho", "batch": 2, "m": 1024, "n": 2560, "dtype": "bf16"},
        # gate_proj of the same layer, the largest matrix it has.
        {"name": "ortho_9728x2560", "kind": "ortho", "batch": 1, "m": 9728, "n": 2560, "dtype": "bf16"},
    ]


def _log(rng, lo: int, hi: int) -> int:
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng) -> dict:
    kind = rng.choice(["attention", "kl", "ortho"])
    c: dict = {"kind": kind}
    if kind == "attention":
        kv = rng.choice([1, 2, 3, 8])
        c |= {"T": _log(rng, 1, 8192), "heads": kv * rng.choice([1, 2, 4]), "kv": kv, "ragged": rng.random() < 0.5}
        c["B"] = _log(rng, 1, max(1, min(64, 2 ** 31 // (c["heads"] * max(c["T"], 64) ** 2))))
    elif kind == "kl":
        c |= {"V": rng.choice([_log(rng, 2, 4096), _log(rng, 1000, 152000), 32000, 151936]),
              "dtype": rng.choice(["bf16", "bf16", "f32"])}
        c["T"] = _log(rng, 1, min(16384, 2048 * 151936 // (c["V"] * (2 if c["dtype"] == "f32" else 1))))
        c["prompt"] = rng.choice([0, c["T"] // 4])
    else:
        m, n = _log(rng, 4, 4096), _log(rng, 4, 9728)
        if rng.random() < 0.5:
            m, n = n, m
        while min(m, n) ** 2 * max(m, n) > 2560 * 2560 * 9728:
            m, n = (m + 1) // 2, (n + 1) // 2
        c |= {"m": m, "n": n, "dtype": rng.choice(["bf16", "f32"])}
        c["batch"] = rng.randint(1, 4) if m * n < 2 ** 21 else 1
    return c


def _lengths(c: dict) -> list[int]:
    """The sequences' lengths: all T, or spread over 0 .. T, the first three T, 0 and 1."""
    B, T = c["B"], c["T"]
    if not c["ragged"]:
        return [T] * B
    return ([T, 0, 1] + [1 + (b * 7919 + 13 * T) % T for b in range(3, B)])[:B]


def prepare(case: dict, seed: int) -> dict:
    g = torch.Generator(device=DEV).manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=torch.float32)
    st = dict(case)
    if case["kind"] == "attention":
        B, T, H, K = case["B"], case["T"], case["heads"], case["kv"]
        # the layers' [B, T, heads, 128] buffers seen as [B, heads, T, 128]; q and k as a per-head norm leaves them
        for nm, h, std in (("q", H, 1.5), ("k", K, 1.0), ("v", K, 0.7), ("dout", H, 0.01)):
            st[nm] = (rand(B, T, h, HEAD) * std).to(torch.bfloat16).transpose(1, 2)
        st["lens"] = torch.tensor(_lengths(case), dtype=torch.int32, device=DEV) if case["ragged"] else None
    elif case["kind"] == "kl":
        T, V, dt = case["T"], case["V"], TYPES[case["dtype"]]
        ref = rand(T, V) * 2.5
        st["q"] = (ref + 0.8 * rand(T, V)).to(dt)  # the quantized model's logits: the reference's and noise
        st["ref"] = ref.to(dt)
        w = torch.where(rand(T) > 1.0, 4.0, 1.0)  # digits weigh more
        w[: case["prompt"]] = 0.0
        st["w"] = w
    else:
        b, m, n = case["batch"], case["m"], case["n"]
        r = min(m, n, 16)
        # a gradient: a few strong directions over noise
        st["G"] = (1e-3 * (rand(b, m, r) @ rand(b, r, n) + 0.3 * rand(b, m, n))).to(TYPES[case["dtype"]])
    return st


def _attention_plain(st: dict) -> dict:
    q, k, v, do = (st[x].float() for x in ("q", "k", "v", "dout"))
    B, H, T, D = q.shape
    K = k.shape[1]
    scale = D ** -0.5
    q, do = q.reshape(B, K, H // K, T, D), do.reshape(B, K, H // K, T, D)
    k, v = k.unsqueeze(2), v.unsqueeze(2)
    t = torch.arange(T, device=q.device)
    lens = torch.full((B,), T, device=q.device) if st["lens"] is None else st["lens"]
    live = (t[None, :] < lens[:, None]).view(B, 1, 1, T, 1)
    seen = (t[None, :] <= t[:, None]) & live
    s = torch.where(seen, q @ k.transpose(-1, -2).contiguous() * scale, float("-inf"))
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(live, m, 0.0))
    del s
    p = p / torch.where(live, p.sum(-1, keepdim=True), 1.0)
    out = p @ v
    do = do * live
    dv = (p.transpose(-1, -2).contiguous() @ do).sum(2)
    ds = do @ v.transpose(-1, -2).contiguous()
    ds = p * (ds - (do * out).sum(-1, keepdim=True)) * scale
    del p
    dq = ds @ k
    dk = (ds.transpose(-1, -2).contiguous() @ q).sum(2)
    whole = lambda x: x.reshape(B, H, T, D).to(torch.bfloat16)
    return {"out": whole(out), "dq": whole(dq), "dk": dk.to(torch.bfloat16), "dv": dv.to(torch.bfloat16)}


def _kl_plain(st: dict) -> dict:
    r, q, w = st["ref"].float(), st["q"].float(), st["w"]
    er = torch.exp(r - r.amax(-1, keepdim=True))
    sr = er.sum(-1, keepdim=True)
    eq = torch.exp(q - q.amax(-1, keepdim=True))
    sq = eq.sum(-1, keepdim=True)
    lr = r - r.amax(-1, keepdim=True) - torch.log(sr)
    lq = q - q.amax(-1, keepdim=True) - torch.log(sq)
    p = er / sr
    kl = torch.where(w > 0, (p * (lr - lq)).sum(-1), 0.0)
    grad = (w / w.sum())[:, None] * (eq / sq - p)
    return {"kl": kl, "loss": (w * kl).sum() / w.sum(), "grad": grad.to(st["q"].dtype)}


def _ortho_plain(st: dict) -> torch.Tensor:
    X = st["G"].float()
    wide = X.shape[1] <= X.shape[2]
    if not wide:
        X = X.transpose(1, 2).contiguous()
    X = X / X.square().sum((1, 2), keepdim=True).sqrt()
    a, b, c = COEFFS
    for _ in range(STEPS):
        A = X @ X.transpose(1, 2).contiguous()
        X = a * X + (b * A + c * (A @ A)) @ X
    return (X if wide else X.transpose(1, 2).contiguous()).to(torch.bfloat16)


def run(st: dict):
    if not own:
        return {"attention": _attention_plain, "kl": _kl_plain, "ortho": _ortho_plain}[st["kind"]](st)
    from lookatmyquant_amd import engine

    if st["kind"] == "attention":
        scale = HEAD ** -0.5
        out, lse = engine.attention_causal_lse(st["q"], st["k"], st["v"], scale, st["lens"])
        dq, dk, dv = engine.attention_causal_grad(st["dout"], st["q"], st["k"], st["v"], out, lse, scale, st["lens"])
        return {"out": out, "dq": dq, "dk": dk, "dv": dv}
    if st["kind"] == "kl":
        kl, loss, grad = engine.kl_rows_grad(st["ref"], st["q"], st["w"])
        return {"kl": kl, "loss": loss, "grad": grad}
    return engine.orthogonalize(st["G"], STEPS, COEFFS)


def work(case: dict) -> dict:
    if case["kind"] == "attention":
        tokens, H, K = case["B"] * case["T"], case["heads"], case["kv"]
        pairs = sum(n * (n + 1) // 2 for n in _lengths(case))
        # q, dout in and out, dq out; k, v in and their gradients out; two products forward and five backward
        return {"bytes": 2.0 * HEAD * tokens * (4 * H + 4 * K), "flops": 7.0 * 2 * HEAD * pairs * H}
    if case["kind"] == "kl":
        T, V, size = case["T"], case["V"], 2 if case["dtype"] == "bf16" else 4
        live = T - case["prompt"]
        return {"bytes": float(size * V * (2 * live + T) + 8 * T), "flops": 12.0 * live * V}
    b, m, n = case["batch"], min(case["m"], case["n"]), max(case["m"], case["n"])
    size = 2 if case["dtype"] == "bf16" else 4
    # two symmetric products (half of each) and one full product a step
    return {"bytes": float(b * m * n * (size + 2)), "flops": float(b * STEPS * (m * m * n + m ** 3 + 2 * m * m * n))}


def exact(case: dict, seed: int):
    st = prepare(case, seed)
    if case["kind"] == "attention":
        got = {x: [] for x in ("out", "dq", "dk", "dv")}
        H, K, T = case["heads"], case["kv"], case["T"]
        for b, n in enumerate(_lengths(case)):
            one = {x: torch.zeros(h, T, HEAD, dtype=torch.float64, device=DEV)
                   for x, h in (("out", H), ("dq", H), ("dk", K), ("dv", K))}
            hidden = torch.ones(n, n, dtype=torch.bool, device=DEV).triu(1)
            for h in range(H if n else 0):
                q, k, v = (st[x][b, i, :n].double().requires_grad_() for x, i in
                           (("q", h), ("k", h // (H // K)), ("v", h // (H // K))))
                s = (torch.matmul(q, k.t()) / math.sqrt(HEAD)).masked_fill(hidden, -math.inf)
                out = torch.matmul(torch.softmax(s, -1), v)
                out.backward(st["dout"][b, h, :n].double())
                one["out"][h, :n], one["dq"][h, :n] = out.detach(), q.grad
                one["dk"][h // (H // K), :n] += k.grad
                one["dv"][h // (H // K), :n] += v.grad
            for x in got:
                got[x].append(one[x])
        return {x: torch.stack(v) for x, v in got.items()}
    if case["kind"] == "kl":
        w = st["w"].double()
        share = w / w.sum()
        kl = torch.zeros(case["T"], dtype=torch.float64, device=DEV)
        grad = torch.zeros(case["T"], case["V"], dtype=torch.float64, device=DEV)
        for t0 in range(0, case["T"], 256):
            rows = slice(t0, t0 + 256)
            p = torch.log_softmax(st["ref"][rows].double(), -1)
            s = torch.log_softmax(st["q"][rows].double(), -1)
            kl[rows] = (p.exp() * (p - s)).sum(-1)
            grad[rows] = share[rows, None] * (s.exp() - p.exp())
        kl[w == 0] = 0.0
        return {"kl": kl, "loss": (share * kl).sum(), "grad": grad}
    G = st["G"].double()
    U = G / torch.linalg.matrix_norm(G, keepdim=True)
    a, b, c = COEFFS
    for _ in range(STEPS):  # from the columns' side where they are fewer: the same polynomial of the singular values
        if case["m"] <= case["n"]:
            M = torch.matmul(U, U.mT)
            U = a * U + torch.matmul(b * M + c * torch.matmul(M, M), U)
        else:
            M = torch.matmul(U.mT, U)
            U = a * U + torch.matmul(U, b * M + c * torch.matmul(M, M))
    return U

"""The attention of training (engine.attention_causal_lse, attention_causal_grad) against its formulas in float64, with
bounds derived from the kernels' roundings: bf16's unit roundoff u = 2^-8 (8 significant bits) once for every probability or dS that enters a
product and once for every result, and float32's for the scores and sums."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U16 = 2.0 ** -8  # half a unit in the last place of bf16's 8 significant bits, relative
U32 = 2.0 ** -24
D = 128
SCALE = D ** -0.5


def say(*a):
    print(*a, flush=True)


def inputs(B, H, Hkv, T, seed, gain=1.0, by_token=True):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def one(h, std):
        shape = (B, T, h, D) if by_token else (B, h, T, D)
        x = (torch.randn(*shape, generator=g, device="cuda") * std).bfloat16()
        return x.transpose(1, 2) if by_token else x

    return one(H, 1.5 * gain), one(Hkv, gain), one(Hkv, 0.7), one(H, 0.01)


def reference(q, k, v, do, scale, lens=None):
    """The results and the elementwise error bounds of bf16 operands, float64 on the CPU."""
    q, k, v, do = (x.double().cpu() for x in (q, k, v, do))
    B, H, T, _ = q.shape
    Hkv = k.shape[1]
    rep = H // Hkv
    kk, vv = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
    t = torch.arange(T)
    n = torch.full((B,), T) if lens is None else lens.cpu().long().clamp(0, T)
    live = (t[None] < n[:, None]).view(B, 1, T, 1)
    q, do = torch.where(live, q, 0.0), torch.where(live, do, 0.0)  # what padding holds is not read
    kk, vv = torch.where(live, kk, 0.0), torch.where(live, vv, 0.0)
    seen = (t[None, :] <= t[:, None]) & live
    s = (q @ kk.mT * scale).masked_fill(~seen, -math.inf)
    lse = torch.logsumexp(s, -1, keepdim=True)
    p = torch.where(seen, torch.exp(s - torch.where(live, lse, 0.0)), 0.0)
    out = p @ vv
    delta = (do * out).sum(-1, keepdim=True)
    dp = do @ vv.mT
    ds = p * (dp - delta)
    group = lambda x: x.reshape(B, Hkv, rep, T, D).sum(2)
    want = {"out": out, "lse": lse[..., 0], "dq": scale * ds @ kk, "dk": group(scale * ds.mT @ q),
            "dv": group(p.mT @ do)}
    # the exponent's error: 128 float32 products and sums, the scaled score, the log-sum-exp; P's is that, relative
    es = 2 * U32 * (D * scale * (q.abs() @ kk.abs().mT) + 4 * s.abs().masked_fill(~seen, 0.0) + 4 * lse.abs().masked_fill(~live, 0.0) + 4)
    ep = p * es.masked_fill(~seen, 0.0)
    eout = (U16 * p + 2 * ep) @ vv.abs() + 2 * T * U32 * (p @ vv.abs()) + U16 * out.abs()
    # delta takes O before its rounding, to 2^-16 of it: what is left of O's error are P's roundings
    edelta = (do.abs() * (eout - (U16 - U16 ** 2) * out.abs())).sum(-1, keepdim=True) + 2 * D * U32 * (do.abs() * out.abs()).sum(-1, keepdim=True)
    edp = 2 * D * U32 * (do.abs() @ vv.abs().mT) + 2 * U32 * delta.abs()
    eds = U16 * ds.abs() + ep * (dp - delta).abs() + p * (edelta + edp)
    sums = 2 * T * rep * U32
    more = 1.01  # products of two of these
    tol = {"out": eout, "lse": (2 * es.amax(-1) + 8 * U32 * lse[..., 0].abs()).masked_fill(~live[..., 0], 0.0),
           "dq": scale * (eds + sums * ds.abs()) @ kk.abs() + U16 * want["dq"].abs(),
           "dk": group(scale * (eds + sums * ds.abs()).mT @ q.abs()) + U16 * want["dk"].abs(),
           "dv": group((U16 * p + ep + sums * p).mT @ do.abs()) + U16 * want["dv"].abs()}
    return want, {x: more * e + 1e-38 for x, e in tol.items()}


def check(got, want, tol):
    for x in want:
        g = got[x].double().cpu()
        same = g == want[x]  # zeros and the -inf of empty rows
        off = ((g - want[x]).abs() / tol[x]).masked_fill(same, 0.0)
        assert bool(torch.isfinite(g[torch.isfinite(want[x])]).all()), x
        assert float(off.max()) <= 1.0, (x, float(off.max()))


def ours(q, k, v, do, scale, lens=None):
    from lookatmyquant_amd import engine as E

    out, kept = E.attention_causal_lse(q, k, v, scale, lens)
    dq, dk, dv = E.attention_causal_grad(do, q, k, v, out, kept, scale, lens)
    torch.cuda.synchronize()
    return {"out": out, "lse": kept.lse, "dq": dq, "dk": dk, "dv": dv}


@pytest.mark.parametrize("B,H,Hkv,T", [(1, 1, 1, 1), (2, 4, 2, 2), (1, 8, 2, 31), (3, 3, 3, 32), (1, 4, 1, 33),
                                       (2, 6, 2, 63), (1, 8, 8, 64), (1, 4, 4, 65), (2, 12, 4, 127), (1, 4, 2, 128),
                                       (1, 6, 3, 129), (1, 16, 2, 191), (1, 4, 1, 257), (8, 4, 1, 320), (1, 8, 8, 600)])
def test_gradients_against_the_formulas(B, H, Hkv, T):
    say(f"attention gradients B={B} H={H} Hkv={Hkv} T={T}")
    x = inputs(B, H, Hkv, T, 1000 + T)
    check(ours(*x, SCALE), *reference(*x, SCALE))


@pytest.mark.parametrize("B,H,Hkv,T", [(2, 4, 2, 2), (3, 8, 4, 5), (1, 32, 8, 45), (2, 4, 1, 128)])
def test_short_sequences_keep_only_the_results_rounding(B, H, Hkv, T):
    """Up to 128 tokens P and dS enter their products whole: the error is the bf16 rounding of the results, spread over
    half a unit in the last place, u / sqrt(3) of the norm at most (u = 2^-8) and more than a thousand numbers."""
    say(f"attention gradients, short B={B} H={H} Hkv={Hkv} T={T}")
    for seed in range(3):
        x = inputs(B, H, Hkv, T, 50 + seed)
        got, (want, _) = ours(*x, SCALE), reference(*x, SCALE)
        for nm in ("out", "dq", "dk", "dv"):
            assert float((got[nm].double().cpu() - want[nm]).norm() / want[nm].norm()) <= U16 / math.sqrt(3), nm


@pytest.mark.parametrize("T,lens", [(200, [200, 0, 1, 2, 31, 32, 33, 63, 64, 65, 127, 128, 129, 199, -3, 500]),
                                    (1, [1, 0, 1]), (64, [0, 0]), (333, [320, 333, 150])])
def test_lengths_and_what_padding_holds(T, lens):
    """Sequences of their own lengths, none, one and past the end among them; NaN and infinities in the padding of every
    operand reach nothing."""
    H, Hkv = 4, 2
    say(f"attention gradients T={T} lens={lens}")
    x = inputs(len(lens), H, Hkv, T, 7, by_token=T != 64)
    n = torch.tensor(lens, dtype=torch.int32, device="cuda")
    want, tol = reference(*x, SCALE, n)
    for t in x:
        for b, m in enumerate(lens):
            t[b, :, max(0, m):] = float("nan")
            t[b, :, max(0, m)::3] = float("inf")
    got = ours(*x, SCALE, n)
    check(got, want, tol)
    for b, m in enumerate(lens):
        for nm in ("out", "dq", "dk", "dv"):
            assert bool((got[nm][b, :, max(0, m):] == 0).all()), nm
        assert bool((got["lse"][b, :, max(0, m):] == -math.inf).all())


def test_second_part_is_read_where_it_was_written():
    """Of O's second part only the rows of queries below the length count: what the others hold reaches nothing."""
    from lookatmyquant_amd import engine as E

    q, k, v, do = inputs(2, 2, 2, 40, 61)
    lens = torch.tensor([40, 7], dtype=torch.int32, device="cuda")
    out, kept = E.attention_causal_lse(q, k, v, SCALE, lens)
    want = E.attention_causal_grad(do, q, k, v, out, kept, SCALE, lens)
    rows = kept.rest.view(2, 2, 2, 16, 32, 8)  # [sequence, head, block of 32 queries, chunk, query, 8 head dims]
    assert bool(torch.isfinite(rows[0, :, 0]).all()) and bool(torch.isfinite(rows[0, :, 1, :, :8]).all())
    rows[0, :, 1, :, 8:], rows[1, :, 0, :, 7:], rows[1, :, 1] = float("nan"), float("nan"), float("nan")
    got = E.attention_causal_grad(do, q, k, v, out, kept, SCALE, lens)
    assert all(torch.equal(a, b) and bool(torch.isfinite(a).all()) for a, b in zip(got, want))


@pytest.mark.parametrize("gain", [0.0, 0.05, 4.0])
def test_flat_and_peaked_rows(gain):
    """Equal scores, and rows where one key holds nearly all the weight (scores in the hundreds)."""
    x = inputs(1, 4, 2, 150, 11, gain)
    check(ours(*x, SCALE), *reference(*x, SCALE))


def test_strides_and_broadcast_inputs():
    """Operands inside wider buffers, in (batch, head, token) order, and one sequence's keys shared by the batch."""
    g = torch.Generator(device="cuda").manual_seed(3)
    B, H, Hkv, T = 3, 4, 2, 77
    wide = (torch.randn(B, T, H + 2 * Hkv + 1, D + 8, generator=g, device="cuda")).bfloat16()
    q = wide[:, :, :H, :D].transpose(1, 2)
    k = wide[:1, :, H:H + Hkv, :D].transpose(1, 2).expand(B, Hkv, T, D)
    v = wide[:, :, H + Hkv:H + 2 * Hkv, :D].transpose(1, 2)
    do = (torch.randn(B, H, T, D, generator=g, device="cuda") * 0.01).bfloat16()
    check(ours(q, k, v, do, 0.2), *reference(q, k, v, do, 0.2))


def test_gradients_against_differences():
    """dq, dk and dv against central differences of sum(out . dout) of the formula, in float64: directions of unit norm,
    the difference's own error (third derivatives, h^2) far below the bf16 results' bound."""
    x = inputs(1, 2, 1, 40, 21)
    got = ours(*x, SCALE)
    q, k, v, do = (t.double().cpu() for t in x)

    def loss(q, k, v):
        s = (q @ k.repeat_interleave(2, 1).mT * SCALE).masked_fill(torch.ones(40, 40).triu(1).bool(), -math.inf)
        return float(((torch.softmax(s, -1) @ v.repeat_interleave(2, 1)) * do).sum())

    g = torch.Generator().manual_seed(5)
    _, tol = reference(*x, SCALE)
    for i, nm in enumerate(("dq", "dk", "dv")):
        for _ in range(3):
            u = torch.randn((q, k, v)[i].shape, generator=g, dtype=torch.float64)
            u /= u.norm()
            h = 1e-4
            up, dn = [q, k, v], [q, k, v]
            up[i], dn[i] = up[i] + h * u, dn[i] - h * u
            num = (loss(*up) - loss(*dn)) / (2 * h)
            have = float((got[nm].double().cpu() * u).sum())
            assert abs(have - num) <= float((tol[nm] * u.abs()).sum()) + 1e-7, (nm, have, num)


def test_forward_agrees_with_the_forwards_attention():
    """attention_causal rounds the probabilities under another maximum: both are within the formula's bound."""
    from lookatmyquant_amd import engine as E

    x = inputs(2, 8, 2, 333, 31)
    out, _ = E.attention_causal_lse(*x[:3], SCALE)
    _, tol = reference(*x, SCALE)
    assert bool(((out - E.attention_causal(*x[:3], SCALE)).double().cpu().abs() <= 2 * tol["out"]).all())


@pytest.mark.parametrize("step", [0.5, 2.0, 7.9, 8.1, 40.0])
def test_growing_maxima(step):
    """Scores that grow along the keys by `step` (in log 2) a block of 64: the running maximum lags, by less and by more
    than it may."""
    B, H, T = 1, 2, 320
    g = torch.Generator(device="cuda").manual_seed(77)
    q = torch.zeros(B, H, T, D, device="cuda")
    k = torch.zeros(B, H, T, D, device="cuda")
    q[..., 0], k[..., 0] = 8.0, step * math.log(2.0) / 64 / 8 * torch.arange(T, device="cuda")
    q, k = (x + 0.02 * torch.randn(B, H, T, D, generator=g, device="cuda") for x in (q, k))
    v, do = (torch.randn(B, H, T, D, generator=g, device="cuda") for _ in range(2))
    x = tuple(t.bfloat16() for t in (q, k, v, do))
    check(ours(*x, 1.0), *reference(*x, 1.0))


def test_repeats_bit_for_bit_on_another_stream():
    x = inputs(4, 16, 4, 700, 41)
    a = ours(*x, SCALE)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = ours(*x, SCALE)
    torch.cuda.current_stream().wait_stream(side)
    for nm in a:
        assert torch.equal(a[nm], b[nm]), nm


def test_refusals():
    from lookatmyquant_amd import engine as E

    q, k, v, do = inputs(2, 4, 2, 40, 51)
    out, kept = E.attention_causal_lse(q, k, v, SCALE)
    lse, rest = kept
    for bad in ((q.float(), k, v), (q, k[:, :, :39], v), (q, k, v[:1]), (q.cpu(), k, v), (q[:, :3], k, v)):
        with pytest.raises(ValueError):
            E.attention_causal_lse(*bad, SCALE)
    for scale in (0.0, -1.0, math.inf, math.nan):
        with pytest.raises(ValueError):
            E.attention_causal_lse(q, k, v, scale)
    with pytest.raises(NotImplementedError):
        E.attention_causal_lse(q[..., :64], k[..., :64], v[..., :64], SCALE)
    for lens in (torch.tensor([1, 2, 3], dtype=torch.int32, device="cuda"), torch.tensor([1, 2], device="cuda"),
                 torch.tensor([1, 2], dtype=torch.int32)):
        with pytest.raises(ValueError):
            E.attention_causal_lse(q, k, v, SCALE, lens)
    odd = torch.empty(2, 40, 4, D + 4, dtype=torch.bfloat16, device="cuda")[..., :D].transpose(1, 2)
    with pytest.raises(ValueError):  # rows that do not start 16-byte aligned
        E.attention_causal_lse(odd, k, v, SCALE)
    for bad in ((do[:, :, :39], q, k, v, out, kept), (do, q, k, v, out.float(), kept), (do, q, k, v, out, (lse[:, :3], rest)),
                (do, q, k, v, out, (lse.double(), rest)), (do.transpose(2, 3), q, k, v, out, kept),
                (do, q, k, v, out, (lse, rest[:-1])), (do, q, k, v, out, (lse, rest.float()))):
        with pytest.raises(ValueError):
            E.attention_causal_grad(*bad, SCALE)
    empty = E.attention_causal_lse(q[:0], k[:0], v[:0], SCALE)
    assert empty[0].shape == (0, 4, 40, D) and empty[1].lse.shape == (0, 4, 40)
    none = E.attention_causal_grad(do[:, :, :0], q[:, :, :0], k[:, :, :0], v[:, :, :0], out[:, :, :0],
                                   (lse[:, :, :0].contiguous(), rest[:0]), SCALE)
    assert none[0].shape == (2, 4, 0, D) and none[1].shape == (2, 2, 0, D)

"""The KL loss with its gradient (engine.kl_rows_grad) against its definition in float64. The bounds: an exponential's
argument is off by a few float32 units of its size (|x| log2(e) at most), so a probability by that, relative; a gradient
by the two probabilities' errors and its own rounding; kl, whose sums are float64, by its terms' errors."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
U32 = 2.0 ** -24


def say(*a):
    print(*a, flush=True)


def inputs(T, V, dt, seed, spread=2.5, noise=0.8):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = torch.randn(T, V, generator=g, device="cuda") * spread
    return r.to(dt), (r + noise * torch.randn(T, V, generator=g, device="cuda")).to(dt)


def reference(ref, q, w=None):
    dt = ref.dtype
    r, s = ref.double().cpu(), q.double().cpu()
    T = r.shape[0]
    w = torch.ones(T, dtype=torch.float64) if w is None else w.double().cpu()
    r = torch.where((w != 0)[:, None], r, 0.0)  # what a left-out row holds is not read
    s = torch.where((w != 0)[:, None], s, 0.0)
    lp, ls = torch.log_softmax(r, -1), torch.log_softmax(s, -1)
    p, t = lp.exp(), ls.exp()
    # a word finite in the reference and -inf in the student makes kl infinite, also where its probability underflows
    term = torch.where(lp == -math.inf, 0.0, torch.where(ls == -math.inf, math.inf, p * (lp - ls)))
    kl = torch.where(w != 0, term.sum(-1), 0.0)
    coef = torch.where(w != 0, w / w.sum(), 0.0)[:, None]
    grad = coef * (t - p)
    size = lambda x: x.masked_fill(x.abs() == math.inf, 0.0).abs()
    # fma(x, log2 e, -m log2 e): the product exact, the base and the difference rounded, exp2 good to one unit
    ep = 4 * U32 * (2 + 1.5 * (size(r) + size(r).amax(-1, keepdim=True)))
    et = 4 * U32 * (2 + 1.5 * (size(s) + size(s).amax(-1, keepdim=True)))
    tg = coef.abs() * (p * (ep + 4 * U32) + t * (et + 4 * U32)) + U[dt] * grad.abs() + 1e-38
    d = torch.where(p > 0, size(lp) + size(ls) + size(r) + size(s), 0.0)
    tk = (p * (ep + 20 * U32) * (1 + d)).sum(-1) * 2 + (t * et).sum(-1) + 2 * U32 * kl.abs().nan_to_num(0, 0, 0)
    tl = (coef[:, 0].abs() * tk.nan_to_num(0, 0, 0)).sum() + 2 * U32 * float((coef[:, 0] * kl).nan_to_num(0, 0, 0).abs().sum())
    return {"kl": kl, "loss": (coef[:, 0] * kl).sum(), "grad": grad}, {"kl": tk, "loss": tl, "grad": tg}


def ours(ref, q, w=None, out=None):
    from lookatmyquant_amd import engine as E

    kl, loss, grad = E.kl_rows_grad(ref, q, w, out)
    torch.cuda.synchronize()
    return {"kl": kl, "loss": loss, "grad": grad}


def check(got, want, tol):
    for x in want:
        g = got[x].double().cpu()
        same = (g == want[x]) | (torch.isnan(g) & torch.isnan(want[x]))
        off = ((g - want[x]).abs() / tol[x]).masked_fill(same, 0.0)
        assert float(off.max()) <= 1.0, (x, float(off.max()))


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,V", [(1, 1), (3, 2), (2, 7), (5, 8), (4, 9), (7, 255), (1, 2047), (2, 2049), (300, 33),
                                 (257, 1000), (255, 4099), (1, 70001), (9, 32003), (300, 32000), (260, 24577), (260, 49153), (260, 151936)])
def test_loss_and_gradient(T, V, dt):
    say(f"kl gradient T={T} V={V} {dt}")
    ref, q = inputs(T, V, dt, T + V)
    check(ours(ref, q), *reference(ref, q))
    w = torch.rand(T, generator=torch.Generator().manual_seed(1)) * 3 + 0.1
    w[::3] = 0.0 if T > 1 else 2.0
    check(ours(ref, q, w), *reference(ref, q, w))


@pytest.mark.parametrize("T", [6, 400])
def test_left_out_rows_may_hold_anything(T):
    ref, q = inputs(T, 700, torch.bfloat16, 5)
    w = torch.ones(T)
    w[1::2] = 0.0
    want = reference(ref, q, w)
    ref[1::2], q[1::4] = float("nan"), float("inf")
    got = ours(ref, q, w.cuda())
    check(got, *want)
    assert bool((got["grad"][1::2] == 0).all()) and bool((got["kl"][1::2] == 0).all())
    none = ours(ref, q, torch.zeros(T))
    assert math.isnan(float(none["loss"])) and not none["grad"].any() and not none["kl"].any()


@pytest.mark.parametrize("T,V", [(4, 5000), (300, 900), (300, 12001), (300, 70001)])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float32])
def test_masked_words_and_rows(T, V, dt):
    """Words at -inf in both, in the reference alone (probability 0) and in the student alone (kl +inf); whole leading
    spans masked; rows with one word left and with none; the type's lowest value."""
    ref, q = inputs(T, V, dt, 9)
    inf = float("inf")
    ref[:, ::7], q[:, ::7] = -inf, -inf
    ref[:, : V // 2] = -inf
    q[2, V - 1] = -inf
    ref[2, V - 1] = 0.0
    ref[1], q[1] = -inf, -inf
    ref[1, 11], q[1, 11], q[1, 12] = 3.0, 2.0, 1.0
    ref[3, V // 2:], q[3, ::5] = torch.finfo(dt).min, torch.finfo(dt).min
    ref[3, V - 2] = 1.0
    want, tol = reference(ref, q)
    got = ours(ref, q)
    assert float(got["kl"][2]) == inf and bool(torch.isfinite(got["grad"]).all())
    keep = [t for t in range(T) if t != 2]
    check({"kl": got["kl"][keep], "grad": got["grad"]}, {"kl": want["kl"][keep], "grad": want["grad"]},
          {"kl": tol["kl"][keep], "grad": tol["grad"]})
    ref[0] = -inf
    got = ours(ref, q)
    assert math.isnan(float(got["kl"][0])) and bool(torch.isnan(got["grad"][0]).all())
    assert bool(torch.isfinite(got["grad"][1:]).all())


@pytest.mark.parametrize("T", [3, 300])
def test_strides_and_alignment(T):
    """Rows inside wider buffers that start at every alignment of the type, written into a caller's buffer whose other
    columns stay as they were."""
    V = 1237
    for dt in (torch.bfloat16, torch.float32):
        a, b = inputs(T, V + 9, dt, 13)
        for i, j, k in ((0, 1, 2), (3, 0, 1), (8, 8, 8), (5, 2, 7)):
            buf = torch.full((T, V + 9), 7.0, dtype=dt, device="cuda")
            got = ours(a[:, i:i + V], b[:, j:j + V], None, buf[:, k:k + V])
            check(got, *reference(a[:, i:i + V], b[:, j:j + V]))
            assert bool((buf[:, :k] == 7).all()) and bool((buf[:, k + V:] == 7).all())


def test_gradient_against_differences():
    """Central differences of the definition's loss in float64, against the float32 gradient."""
    ref, q = inputs(3, 50, torch.float32, 17)
    w = torch.tensor([1.0, 0.0, 4.0])
    got = ours(ref, q, w)["grad"].double().cpu()
    _, tol = reference(ref, q, w)

    def loss(s):
        lp, ls = torch.log_softmax(ref.double().cpu(), -1), torch.log_softmax(s, -1)
        return float((w.double() * (lp.exp() * (lp - ls)).sum(-1)).sum() / 5.0)

    x = q.double().cpu()
    for t in range(3):
        for v in range(0, 50, 7):
            e = torch.zeros_like(x)
            e[t, v] = 1e-5
            num = (loss(x + e) - loss(x - e)) / 2e-5
            assert abs(num - float(got[t, v])) <= float(tol["grad"][t, v]) + 1e-10


def test_kl_agrees_with_the_measure_steps():
    """The kl of the measure step's kernel on the same logits, to both kernels' float32 result."""
    from lookatmyquant_amd import engine as E

    ref, q = inputs(300, 5000, torch.bfloat16, 23)
    kl, _ = E.kl_rows(ref, q)
    _, tol = reference(ref, q)
    assert bool(((ours(ref, q)["kl"] - kl).double().cpu().abs() <= 2 * tol["kl"]).all())


def test_repeats_bit_for_bit():
    for T in (20, 500):
        ref, q = inputs(T, 20011, torch.bfloat16, 29)
        a = ours(ref, q)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            b = ours(ref, q)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a[x], b[x]) for x in a)


def test_refusals():
    from lookatmyquant_amd import engine as E

    ref, q = inputs(4, 100, torch.bfloat16, 31)
    for a, b in ((ref, q[:, :99]), (ref, q.float()), (ref.half(), q.half()), (ref.cpu(), q.cpu()), (ref.t(), q.t()),
                 (ref[0], q[0]), (ref[:, :0], q[:, :0]), (ref[:1].expand(4, 100), q)):
        with pytest.raises(ValueError):
            E.kl_rows_grad(a, b)
    with pytest.raises(ValueError):
        E.kl_rows_grad(ref, q, torch.ones(3))
    with pytest.raises(ValueError):
        E.kl_rows_grad(ref, q, None, torch.empty(4, 100, device="cuda"))
    kl, loss, grad = E.kl_rows_grad(ref[:0], q[:0])
    assert kl.shape == (0,) and grad.shape == (0, 100) and math.isnan(float(loss))

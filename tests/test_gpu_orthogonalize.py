"""The Newton-Schulz orthogonalisation (engine.orthogonalize) against its definition in float64. The bound is carried
through the steps in float64: a step adds what its float16 roundings (u = 2^-11 of hi, A and B) and float32 sums can
change, worst case in the Frobenius norm, and passes on what came before by at most its derivative's norm on the
spectrum; the result is rounded to bf16 once."""

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U16, U32, UB = 2.0 ** -11, 2.0 ** -24, 2.0 ** -8
COEFFS = (3.4445, -4.7750, 2.0315)


def say(*a):
    print(*a, flush=True)


def gradient(m, n, kind, seed, dt=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
    if kind == "noise":
        G = rand(m, n)
    elif kind == "strong":  # a few strong directions over noise
        r = min(m, n, 8)
        G = rand(m, r) @ rand(r, n) + 0.3 * rand(m, n)
    else:  # decaying: singular values 1 / i
        r = min(m, n)
        u, v = torch.linalg.qr(rand(m, r).double())[0], torch.linalg.qr(rand(n, r).double())[0]
        G = (u / torch.arange(1, r + 1, device="cuda").double()) @ v.mT
    return (1e-3 * G).to(dt)


def reference(G, steps=5, coeffs=COEFFS):
    """(the result, a bound on the Frobenius norm of the error), float64."""
    X = G.double()
    tall = X.shape[0] > X.shape[1]
    X = X.mT if tall else X
    X = X / X.norm()
    a, b, c = coeffs
    m, n = X.shape
    # hi + lo leaves 2^-22 of an entry, and 2^-25 of 2^-10 where lo is below float16's normal numbers
    part = lambda X: 2 ** -22 * float(X.norm()) + 2 ** -35 * math.sqrt(m * n)
    err = part(X)
    for _ in range(steps):
        s = torch.linalg.svdvals(X)
        A = X @ X.mT
        B = b * A + c * A @ A
        f = s * (a + b * s ** 2 + c * s ** 4)
        i, j = torch.meshgrid(s, s, indexing="ij")
        fi, fj = torch.meshgrid(f, f, indexing="ij")
        df = (a + 3 * b * s ** 2 + 5 * c * s ** 4).abs().max()
        dif = torch.where((i - j).abs() > 1e-9, (fi - fj).abs() / (i - j).abs().clamp_min(1e-9), 0.0).max()
        tot = torch.where(i + j > 1e-12, (fi + fj).abs() / (i + j).clamp_min(1e-12), 0.0).max()
        off = (f / s.clamp_min(1e-30)).abs().max() if m < n else 0.0
        lip = max(float(df), float(dif), float(tot), float(off), abs(a))
        s1, x = float(s[0]), float(X.norm())
        small = 2 ** -35  # half the spacing of float16's subnormals, over the 2^10 that entries are stored times
        acc = 2 * math.sqrt(n) * U32
        e_hi = U16 * x + small * math.sqrt(m * n)
        e_A = 2 * s1 * e_hi + (U16 + acc) * float(A.norm()) + small * m
        e_B = (abs(b) + 2 * abs(c) * s1 ** 2) * e_A + (U16 + acc) * (abs(b) + abs(c) * s1 ** 2) * float(A.norm()) + small * m
        b1 = float(torch.linalg.matrix_norm(B, 2))
        X = a * X + B @ X
        err = lip * err + s1 * e_B + b1 * e_hi + acc * b1 * x + part(X)
    err = 1.05 * err + UB * float(X.norm())  # 1.05: second orders
    return (X.mT if tall else X), err


def rounded_as_the_kernels(G, steps=5, coeffs=COEFFS):
    """The iteration in float64 with the kernels' float16 roundings at their places: what is left between it and the
    result are float32 sums, which flip a float16 rounding here and there, and the bf16 rounding of the result (half a
    unit at most, 0.4 of that in the root mean square), so the result's bound from it is that half unit's norm. A's and
    B's diagonals are whole, but in matrices of 97 to 128 rows (columns of tall ones) and up to 512 columns."""
    h = lambda x: x.to(torch.float16).double()
    X = G.double()
    tall = X.shape[0] > X.shape[1]
    X = (X.mT if tall else X) / X.norm() * 1024
    a, b, c = coeffs
    hi = h(X)
    lo = h(X - hi)
    whole = not (96 < X.shape[0] <= 128 and X.shape[1] <= 512)
    diag = lambda x: whole * x.diagonal().unsqueeze(1)
    for _ in range(steps):
        A0 = hi @ hi.mT / 1024
        A, E = h(A0), diag(A0 - h(A0))
        At = A + torch.diag(E[:, 0])
        B0 = b * At + c * (A @ A + (E + E.mT) * At) / 1024
        B = h(B0)
        X = a * (hi + lo) + (B @ hi + diag(B0 - B) * hi + diag(B0) * lo) / 1024
        hi = h(X)
        lo = h(X - hi)
    return (X.mT if tall else X) / 1024


def check(out, want, bound):
    off = float((out.double() - want).norm())
    say(f"  off {off / float(want.norm()):.2e}, bound {bound / float(want.norm()):.2e}")
    assert bool(torch.isfinite(out).all()) and off <= bound


@pytest.mark.parametrize("dt", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("m,n,kind", [(1, 1, "noise"), (1, 40, "noise"), (7, 5, "noise"), (64, 64, "decaying"),
                                      (65, 130, "strong"), (128, 128, "noise"), (129, 127, "strong"), (333, 200, "decaying"),
                                      (256, 1000, "strong"), (1000, 129, "noise"), (384, 640, "decaying"),
                                      (700, 700, "strong"), (1024, 2560, "noise")])
def test_against_the_definition(m, n, kind, dt):
    from lookatmyquant_amd import engine as E

    say(f"orthogonalize {m} x {n} {kind} {dt}")
    G = gradient(m, n, kind, m * 7 + n, dt)
    out = E.orthogonalize(G)
    assert out.dtype == torch.bfloat16 and out.shape == G.shape
    check(out, *reference(G))
    near = rounded_as_the_kernels(G)
    check(out, near, UB * float(near.norm()))


@pytest.mark.parametrize("m,n", [(1, 900), (2, 480), (3, 2000), (7, 659), (659, 7), (31, 512), (96, 512), (97, 512), (96, 513),
                                 (128, 512), (128, 513), (600, 30)])
def test_few_rows(m, n):
    """Where one rounding of A or B on the diagonal would move a whole singular direction."""
    from lookatmyquant_amd import engine as E

    say(f"orthogonalize {m} x {n}, few rows")
    for kind in ("noise", "strong", "decaying"):
        G = gradient(m, n, kind, m + 3 * n)
        out = E.orthogonalize(G)
        check(out, *reference(G))
        near = rounded_as_the_kernels(G)
        check(out, near, UB * float(near.norm()))


@pytest.mark.parametrize("steps,coeffs", [(0, COEFFS), (1, COEFFS), (2, (1.5, -0.5, 0.0)), (12, (1.875, -1.25, 0.375))])
def test_steps_and_coefficients(steps, coeffs):
    from lookatmyquant_amd import engine as E

    G = gradient(150, 90, "strong", 3)
    check(E.orthogonalize(G, steps, coeffs), *reference(G, steps, coeffs))


def test_converges_to_the_polar_factor():
    """Twelve steps of (15 s - 10 s^3 + 3 s^5) / 8, whose fixed point is 1: U V^T, rows orthonormal to bf16."""
    from lookatmyquant_amd import engine as E

    G = gradient(100, 300, "noise", 5)
    out = E.orthogonalize(G, 12, (1.875, -1.25, 0.375)).double()
    u, _, v = torch.linalg.svd(G.double(), full_matrices=False)
    # the coupling of the roundings above with a contraction at 1: 2^-8 per entry of the result, and a step's own
    assert float((out - u @ v).norm() / math.sqrt(100)) <= UB + 12 * U16


def test_batches_and_strides():
    from lookatmyquant_amd import engine as E

    G = torch.stack([gradient(70, 200, k, i) for i, k in enumerate(("noise", "strong", "decaying"))])
    want = [E.orthogonalize(g) for g in G]
    assert all(torch.equal(a, b) for a, b in zip(E.orthogonalize(G), want))
    wide = torch.zeros(3, 75, 233, device="cuda")
    wide[:, 2:72, 5:205] = G
    room = torch.full((3, 80, 211), 7.0, dtype=torch.bfloat16, device="cuda")
    got = E.orthogonalize(wide[:, 2:72, 5:205], out=room[:, 3:73, 1:201])
    assert got.data_ptr() == room[:, 3:73, 1:201].data_ptr()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    room[:, 3:73, 1:201] = 7.0
    assert bool((room == 7).all())
    shared = E.orthogonalize(G[:1].expand(4, 70, 200))
    assert all(torch.equal(a, want[0]) for a in shared)
    tall = E.orthogonalize(G.transpose(1, 2).contiguous())
    assert all(torch.equal(a.mT, b) for a, b in zip(tall, want))


@pytest.mark.parametrize("scale", [1e-36, 1e-20, 1.0, 1e20, 1e36])
def test_scale_of_the_gradient_does_not_matter(scale):
    from lookatmyquant_amd import engine as E

    G = gradient(60, 100, "strong", 9).double() * 1e3 * scale
    check(E.orthogonalize(G.float()), *reference(G.float()))


def test_zero_and_non_finite():
    from lookatmyquant_amd import engine as E

    G = torch.stack([gradient(40, 130, "noise", 1), torch.zeros(40, 130, device="cuda"), gradient(40, 130, "noise", 2)])
    G[2, 3, 5] = float("nan")
    out = E.orthogonalize(G)
    assert torch.equal(out[0], E.orthogonalize(G[0])) and not out[1].any() and bool(torch.isnan(out[2]).all())
    one = torch.zeros(20, 30, device="cuda")
    one[4, 7] = -2.0  # a single entry: singular value 1
    s = 1.0
    for _ in range(5):
        s = s * (COEFFS[0] + COEFFS[1] * s ** 2 + COEFFS[2] * s ** 4)
    got = E.orthogonalize(one)
    assert abs(float(got[4, 7]) + s) <= (UB + 5 * 3.5 * 4 * U16) * s and int((got != 0).sum()) == 1


def test_repeats_bit_for_bit():
    from lookatmyquant_amd import engine as E

    G = gradient(500, 900, "strong", 4, torch.bfloat16)
    a = E.orthogonalize(G)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        b = E.orthogonalize(G)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, b)


def test_refusals():
    from lookatmyquant_amd import engine as E

    G = gradient(20, 30, "noise", 6)
    for bad in (G.double(), G.half(), G.cpu(), G.t(), G[0], G[None, None]):
        with pytest.raises(ValueError):
            E.orthogonalize(bad)
    for steps, coeffs in ((-1, COEFFS), (5, (1.0, 2.0)), (5, (30.0, 0.0, 0.0)), (5, (math.nan, 0.0, 0.0)),
                          (5, (3.4445, -4.775, 20.0)), (200, (1.1, 0.0, 0.0))):
        with pytest.raises(ValueError):
            E.orthogonalize(G, steps, coeffs)
    for out in (torch.empty(20, 30, device="cuda"), torch.empty(20, 31, dtype=torch.bfloat16, device="cuda")):
        with pytest.raises(ValueError):
            E.orthogonalize(G, out=out)
    assert E.orthogonalize(G[:0]).shape == (0, 30) and E.orthogonalize(G[None][:0]).shape == (0, 20, 30)

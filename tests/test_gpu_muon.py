"""GPU: orthogonalise, muon_step_ and adam_step_multi_ against the formulas in 64 bits.

Tolerances.  Write X_k for the iterates, p for the step's polynomial and L for the largest of |p'(s)| and p(s) / s over the singular
values that occur: L = a = 3.4445 for the default coefficients (both are largest at s = 0).  An error E made in X_k leaves at most
L^(steps - k) |E| in the result (p acts on singular values; its divided differences are bounded by L).

fp32 precision.  What a step adds to X_k is at most u |X_k| a + u |B X_k| each for rounding X's planes (2^-23 of an entry) and for
the three-product sums (2^-22: the dropped product and the planes' rounding of both factors, plus fp32 sums, which are far smaller
at these lengths): E <= 2^-21 L |X_k|.  Hence  |error| <= 2^-21 sum_k L^(steps - k) |X_k|  in the Frobenius norm, with the |X_k| of
the 64-bit iteration: `bound32` below.

fp16 precision.  Every factor of A = X X^T, A A and B X is rounded to 11 bits (2^-11 relative at most between neighbours, half of it
for a rounding), X itself is kept.  The six rounded factors of a step change the result of a step by at most 6 * 2^-12 (|b| s^2 +
2 |c| s^4) s <= 6 * 2^-12 * 9 * s where s <= 1, in directions in which X is strong (a product B X with a rounded B or a rounded X has
the left or the right directions of the unrounded one), where later steps have |p'| <= 1.7 and mostly contract.  Roundings of different
entries and steps are independent, so that five steps add up as their root: sqrt(5) * 6 * 2^-12 * 9 = 0.03 is the most that a
relative Frobenius error can be; the entries of a product average over rows, which brings a typical one below a tenth of it.
HALF = 0.01 is asked for, and 2^-8 (bf16) or 2^-11 (fp16) of the result's type on top."""
import importlib

import pytest
import torch

pytestmark = pytest.mark.gpu

NS = (3.4445, -4.7750, 2.0315)
CUBIC = (1.5, -0.5, 0.0)
HALF = 0.01
EPS_OF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


@pytest.fixture(scope="module")
def S():
    import spin_nerf_amd as S
    return S


def oracle(x, steps=5, coefficients=NS, eps=1e-7, want_norms=False):
    """the formula in 64 bits on the CPU; also the Frobenius norms of the iterates"""
    a, b, c = coefficients
    x = x.detach().double().cpu()
    n = x.square().sum((-2, -1), keepdim=True).sqrt()
    X = x / torch.where(n < eps, torch.full_like(n, eps), n)
    norms = []
    for _ in range(steps):
        norms.append(X.flatten(-2).norm(dim=-1))
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return (X, norms) if want_norms else X


def bound32(norms, steps, L):
    return 2.0 ** -21 * sum(L ** (steps - k) * n for k, n in enumerate(norms))


def gradient_like(gen, *shape):
    m, n = shape[-2:]
    r = max(1, min(m, n) // 2)
    d = torch.arange(1, r + 1, dtype=torch.float32) ** -0.7
    x = (torch.randn(*shape[:-1], r, generator=gen) * d) @ torch.randn(*shape[:-2], r, n, generator=gen)
    return 1e-3 * (x + 0.05 * torch.randn(*shape, generator=gen))


def check(got, x, precision, steps=5, coefficients=NS, eps=1e-7):
    ref, norms = oracle(x, steps, coefficients, eps, want_norms=True)
    L = coefficients[0]
    off = (got.detach().double().cpu() - ref).flatten(-2).norm(dim=-1)
    size = ref.flatten(-2).norm(dim=-1)
    tol = EPS_OF[x.dtype] * size + (HALF * size if precision == "fp16" else bound32(norms, steps, L)) + 1e-10
    assert bool((off <= tol).all()), (float((off / size.clamp(min=1e-30)).max()), float((tol / size.clamp(min=1e-30)).max()))


SHAPES = [(1, 1), (64, 448), (449, 64), (33, 129), (257, 60), (1, 7), (5, 1), (2, 3), (31, 33), (64, 64), (63, 65), (65, 64), (16, 200), (200, 16), (128, 283), (256, 256), (256, 319),
          (319, 256), (130, 129), (1000, 333), (40, 1500)]


@pytest.mark.parametrize("m,n", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_orthogonalise_matches_the_formula(S, m, n, dtype):
    gen = torch.Generator().manual_seed(1000 * m + n)
    x = gradient_like(gen, 3, m, n).to(dtype)
    if dtype == torch.float16:
        x = (x.float() * 100).to(dtype)
    for precision in ("fp32", "fp16"):
        got = S.orthogonalise(x.cuda(), precision=precision)
        assert got.shape == x.shape and got.dtype == dtype
        check(got, x, precision)


@pytest.mark.parametrize("m,n", [(512, 512), (700, 1100), (1100, 700)])
def test_orthogonalise_of_larger_matrices(S, m, n):
    x = gradient_like(torch.Generator().manual_seed(3), 1, m, n)
    for precision in ("fp32", "fp16"):
        check(S.orthogonalise(x.cuda(), precision=precision), x, precision)


@pytest.mark.parametrize("steps,coefficients", [(1, NS), (2, NS), (8, CUBIC), (12, CUBIC), (3, (2.0, -1.5, 0.5))])
def test_other_step_counts_and_polynomials(S, steps, coefficients):
    x = gradient_like(torch.Generator().manual_seed(steps), 2, 96, 140)
    got = S.orthogonalise(x.cuda(), steps=steps, coefficients=coefficients)
    check(got, x, "fp32", steps, coefficients)


def test_default_precision_goes_by_type(S):
    x = gradient_like(torch.Generator().manual_seed(0), 100, 120).cuda()
    assert torch.equal(S.orthogonalise(x), S.orthogonalise(x, precision="fp32"))
    b = x.bfloat16()
    assert torch.equal(S.orthogonalise(b), S.orthogonalise(b, precision="fp16"))


def test_strides_orders_and_stacks(S):
    gen = torch.Generator().manual_seed(5)
    x = gradient_like(gen, 4, 70, 90).cuda()
    plain = S.orthogonalise(x)
    wide = torch.full((4, 70, 130), float("nan"), device="cuda")
    wide[..., 17:107] = x
    assert torch.equal(S.orthogonalise(wide[..., 17:107]), plain)                 # row stride, off the 16-byte grid
    assert torch.equal(S.orthogonalise(x.reshape(2, 2, 70, 90)), plain.reshape(2, 2, 70, 90))
    turned = x.mT.contiguous().mT                                                  # columns first in memory
    got = S.orthogonalise(turned)
    assert got.shape == x.shape
    check(got, x.cpu(), "fp32")
    every = torch.empty(8, 70, 90, device="cuda")
    every[::2] = x
    assert torch.equal(S.orthogonalise(every[::2]), plain)
    one = x[1].expand(3, 70, 90)                                                   # the same matrix three times
    assert torch.equal(S.orthogonalise(one), plain[1].expand(3, 70, 90))
    assert torch.equal(S.orthogonalise(x[2]), plain[2])                            # a matrix alone: the same bits
    third = x.permute(1, 2, 0).contiguous().permute(2, 0, 1)                       # no unit stride in a matrix
    assert torch.equal(S.orthogonalise(third), plain)


def test_result_into_out_and_in_place(S):
    x = gradient_like(torch.Generator().manual_seed(6), 2, 60, 50).cuda()
    plain = S.orthogonalise(x)
    buf = torch.empty_like(x)
    assert S.orthogonalise(x, out=buf) is buf and torch.equal(buf, plain)
    y = x.clone()
    S.orthogonalise(y, out=y)
    assert torch.equal(y, plain)
    z = torch.zeros(3, 60, 50, device="cuda")
    z[:2] = x
    S.orthogonalise(z[:2], out=z[1:])                                              # overlapping by one matrix
    assert torch.equal(z[1:], plain) and torch.equal(z[0], x[0])
    sq = gradient_like(torch.Generator().manual_seed(7), 64, 64).cuda()
    want = S.orthogonalise(sq.mT.contiguous())
    S.orthogonalise(sq.mT, out=sq)                                                 # the input is the output, transposed
    assert torch.equal(sq, want)


def test_zero_tiny_huge_and_not_finite(S):
    gen = torch.Generator().manual_seed(8)
    x = gradient_like(gen, 8, 40, 50)
    x[1] = 0
    x[2] *= 1e-30        # below eps: x / eps, nearly nothing
    x[3] *= 1e33         # squares pass fp32
    x[4, 3, 4] = float("nan")
    x[5, 7, 8] = float("inf")
    x[6, 0, 0] = float("-inf")
    got = S.orthogonalise(x.cuda()).cpu()
    for k in (0, 3, 7):
        check(got[k], x[k], "fp32")
    assert bool((got[1] == 0).all()) and float(got[2].abs().max()) < 1e-10
    for k in (4, 5, 6):
        assert bool(torch.isnan(got[k]).all())
    small = gradient_like(gen, 40, 50) * 1e-9       # a norm below eps all the same: x / eps is what the formula says
    ref = oracle(small)
    assert float((S.orthogonalise(small.cuda()).cpu().double() - ref).abs().max()) < 1e-4 * float(ref.abs().max()) + 1e-9


def test_rank_one_and_repeated_rows(S):
    u, v = torch.randn(90, generator=torch.Generator().manual_seed(1)), torch.randn(70, generator=torch.Generator().manual_seed(2))
    x = u[:, None] * v[None]
    check(S.orthogonalise(x.cuda()), x, "fp32")
    check(S.orthogonalise(x.cuda(), precision="fp16"), x, "fp16")
    r = torch.ones(33, 34)
    check(S.orthogonalise(r.cuda()), r, "fp32")


def test_empty_inputs(S):
    for shape in [(0, 4, 5), (3, 0, 5), (3, 4, 0), (0, 0)]:
        x = torch.empty(*shape, device="cuda")
        assert S.orthogonalise(x).shape == x.shape
    S.muon_step_([], [], [], 1e-3)
    S.adam_step_multi_([], [], [], [], 1e-3, 1)
    e = torch.empty(0, 5, device="cuda")
    S.muon_step_([e], [e], [e], 1e-3)
    e = torch.empty(0, device="cuda")
    S.adam_step_multi_([e], [e], [e], [e], 1e-3, 1)


def test_repeats_bit_for_bit_on_another_stream_and_beside_other_work(S):
    x = gradient_like(torch.Generator().manual_seed(9), 6, 256, 256).cuda()
    want = S.orthogonalise(x)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        a = [S.orthogonalise(x) for _ in range(3)]
    b = [S.orthogonalise(x) for _ in range(3)]      # two streams at once, a workspace each
    torch.cuda.synchronize()
    assert all(torch.equal(t, want) for t in a + b)


# ---- muon_step_ ---------------------------------------------------------------------------------------------------------------
def muon_oracle(p, g, m, lr, mu, nesterov, wd, scale, grad_scale, **kw):
    p, g, m = p.double().cpu(), g.double().cpu() * grad_scale, m.double().cpu()
    m = mu * m + g
    u = g + mu * m if nesterov else m
    rows, cols = p.shape[-2:]
    q = max(1.0, rows / cols) ** 0.5 if scale == "spectral" else 0.2 * max(rows, cols) ** 0.5 if scale == "rms" else 1.0
    o, norms = oracle(u, want_norms=True, **kw)
    return p * (1 - lr * wd) - lr * q * o, m, lr * q, o, norms


def muon_case(gen, shapes):
    p = [torch.rand(*s, generator=gen) * 0.2 - 0.1 for s in shapes]
    g = [gradient_like(gen, *s) for s in shapes]
    m = [3 * gradient_like(gen, *s) for s in shapes]
    return p, g, m


MUON_SHAPES = [[(256, 256)], [(7, 256, 256), (256, 319), (128, 283)], [(2, 2, 33, 20), (1, 9), (9, 1), (300, 64), (64, 300)],
               [(17, 19)] * 30]                       # more than one launch sequence's table


@pytest.mark.parametrize("shapes", MUON_SHAPES)
@pytest.mark.parametrize("precision,nesterov,scale,wd,gs", [("fp32", True, "spectral", 0.1, 1.0), ("fp32", False, "rms", 0.0, 0.25),
                                                           ("fp16", True, "none", 0.01, 1.0)])
def test_muon_step_matches_the_formula(S, shapes, precision, nesterov, scale, wd, gs):
    lr, mu = 0.02, 0.95
    p, g, m = muon_case(torch.Generator().manual_seed(11), shapes)
    dp, dg, dm = ([t.cuda() for t in ts] for ts in (p, g, m))
    S.muon_step_(dp, dg, dm, lr, momentum=mu, nesterov=nesterov, weight_decay=wd, scale=scale, grad_scale=gs, precision=precision)
    for P, G, M, gp, gg, gm in zip(p, g, m, dp, dg, dm):
        rp, rm, step, o, norms = muon_oracle(P, G, M, lr, mu, nesterov, wd, scale, gs)
        assert torch.equal(gg.cpu(), G)
        assert float((gm.cpu().double() - rm).norm()) <= 3 * 2.0 ** -24 * float(rm.norm() + G.double().norm())      # two products, one sum
        off = (gp.cpu().double() - rp).flatten(-2).norm(dim=-1)
        size = o.flatten(-2).norm(dim=-1)
        # the update's own error, the momentum's three roundings (amplified by at most L^5 |X_0| = 485) and the parameters' two
        tol = step * ((HALF * size if precision == "fp16" else bound32(norms, 5, NS[0])) + 485 * 4 * 2.0 ** -24) \
            + 4 * 2.0 ** -24 * P.double().flatten(-2).norm(dim=-1)
        assert bool((off <= tol).all()), (float(off.max()), float(tol.min()))


def test_muon_steps_in_a_row_and_rate_from_device_state(S):
    import ctypes
    p, g, m = muon_case(torch.Generator().manual_seed(12), [(64, 80), (80, 64)])
    dp, dg, dm = ([t.cuda() for t in ts] for ts in (p, g, m))
    ep, em = [t.clone() for t in dp], [t.clone() for t in dm]
    st = S._lib.StepState(0, 1, 0, 0.02, 0.1, 0.03, 0.0)
    state = torch.frombuffer(bytearray(bytes(st)), dtype=torch.uint8).cuda()
    assert state.numel() == ctypes.sizeof(S._lib.StepState)
    for _ in range(3):
        S.muon_step_(dp, dg, dm, 0.02, weight_decay=0.1)
        S.muon_step_(ep, dg, em, 123.0, weight_decay=0.1, state=state)      # the rate in memory counts
    for a, b in zip(dp + dm, ep + em):
        assert torch.equal(a, b)


def test_muon_leaves_the_surroundings_alone(S):
    flat = torch.full((3 * 4000,), 7.0, device="cuda")
    p, g, m = flat[13:13 + 50 * 61].view(50, 61), torch.randn(50, 61, device="cuda"), torch.zeros(50, 61, device="cuda")
    S.muon_step_([p], [g], [m], 0.02)
    assert bool((flat[:13] == 7).all()) and bool((flat[13 + 50 * 61:] == 7).all())
    # an entry of 7 stays where its step is below half an ulp, 2.4e-7: |O| < 1.2e-5 where O has a deviation of 61 ** -0.5 = 0.13,
    # one entry in 13 000 of these 3050
    assert float((p == 7).float().mean()) < 0.01


def test_set_captured_into_a_graph_and_replayed(S):
    """orthogonalise, muon_step_ and adam_step_multi_ as a captured step, two graphs alive at once, eager work between replays"""
    def state(seed):
        p, g, m = muon_case(torch.Generator().manual_seed(seed), [(3, 96, 64), (64, 130)])
        d = dict(p=[t.cuda() for t in p], g=[t.cuda() for t in g], m=[t.cuda() for t in m])
        r = torch.Generator().manual_seed(seed)
        d["b"] = [torch.randn(n, generator=r).cuda() for n in (64, 3, 257)]
        d["bg"] = [torch.randn(n, generator=r).cuda() for n in (64, 3, 257)]
        d["bm"], d["bv"] = [torch.zeros_like(t) for t in d["b"]], [torch.zeros_like(t) for t in d["b"]]
        return d

    def step(d):
        S.muon_step_(d["p"], d["g"], d["m"], 0.01, weight_decay=0.1)
        S.adam_step_multi_(d["b"], d["bg"], d["bm"], d["bv"], 1e-3, 1)
        d["o"] = S.orthogonalise(d["p"][0])

    eager, graphed, graphs = [state(1), state(2)], [state(1), state(2)], []
    step(state(3))
    torch.cuda.synchronize()
    for d in graphed:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step(d)
        graphs.append(g)
    for _ in range(4):
        for d, e, g in zip(graphed, eager, graphs):
            g.replay()
            step(e)
        torch.cuda.synchronize()
        for d, e in zip(graphed, eager):
            for k in ("p", "m", "b", "bm", "bv"):
                assert all(torch.equal(a, b) for a, b in zip(d[k], e[k])), k
            assert torch.equal(d["o"], e["o"])


# ---- adam_step_multi_ ------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("sizes", [[1], [16384, 256, 256, 128, 257, 387], [1023, 1024, 1025, 4096, 3, 5000], [70] * 100, [1 << 20, 1]])
def test_adam_step_multi_is_adam_step_bit_for_bit(S, sizes):
    ops = importlib.import_module("spin-nerf_amd.ops")
    gen = torch.Generator().manual_seed(len(sizes))
    n = sum(sizes)
    p, g, m, v = torch.randn(n, generator=gen), torch.randn(n, generator=gen), torch.randn(n, generator=gen), torch.rand(n, generator=gen)
    a = [t.cuda() for t in (p, m, v)]
    b = [t.cuda() for t in (p, m, v)]
    G = g.cuda()
    for k in (1, 2, 3):
        S.adam_step_multi_(list(a[0].split(sizes)), list(G.split(sizes)), list(a[1].split(sizes)), list(a[2].split(sizes)), 5e-4, k,
                           grad_scale=0.5)
        for bp, bg, bm, bv in zip(*(list(t.split(sizes)) for t in (b[0], G, b[1], b[2]))):
            t = [x.clone() for x in (bp, bg, bm, bv)]       # adam_step_ wants its buffers on the 16-byte grid
            ops.adam_step_(*t, 5e-4, k, grad_scale=0.5)
            bp.copy_(t[0]); bm.copy_(t[2]); bv.copy_(t[3])
        assert all(torch.equal(x, y) for x, y in zip(a, b))
    # and the formula in 64 bits
    P, M, V = p.double(), m.double(), v.double()
    for k in (1, 2, 3):
        gk = 0.5 * g.double()
        M, V = 0.9 * M + 0.1 * gk, 0.999 * V + 0.001 * gk * gk
        P = P - 5e-4 * (M / (1 - 0.9 ** k)) / ((V / (1 - 0.999 ** k)).sqrt() + 1e-8)
    # 1 - 0.999 is off by 1.3e-5 of itself where beta2 is a 32-bit number: half of that in the rate, three steps of at most 40 lr
    assert float((a[0].cpu().double() - P).abs().max()) <= 3 * 40 * 5e-4 * 2e-5 + 4 * 2.0 ** -24 * float(P.abs().max())


def test_refusals_on_the_device(S):
    x = torch.randn(4, 8, 8, device="cuda")
    with pytest.raises(ValueError, match="out must be"):
        S.orthogonalise(x, out=torch.empty(4, 8, 8, device="cuda", dtype=torch.float16))
    with pytest.raises(RuntimeError, match="no backward"):
        S.orthogonalise(x.clone().requires_grad_())
    with torch.no_grad():
        S.orthogonalise(x.clone().requires_grad_())
    with pytest.raises(ValueError, match="shares memory"):
        S.muon_step_([x[0], x[0]], [x[1], x[1]], [x[2], x[3]], 1e-3)
    with pytest.raises(ValueError, match="shares memory"):
        S.muon_step_([x[0]], [x[1]], [x[1]], 1e-3)
    with pytest.raises(ValueError, match="contiguous"):
        S.muon_step_([x[0].mT], [x[1]], [x[2]], 1e-3)
    with pytest.raises(S.HipLibraryError, match="device"):
        S.muon_step_([x[0]], [x[1].cpu()], [x[2]], 1e-3)
    before = x.clone()
    S.muon_step_([x[0]], [x[1].mT], [x[2]], 1e-3)                     # gradients in another order are read as they are
    y = before.clone()
    S.muon_step_([y[0]], [before[1].mT.contiguous()], [y[2]], 1e-3)
    assert torch.equal(x, y)

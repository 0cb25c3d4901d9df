"""What orthogonalise does to numbers, in torch and 64 bits: the planes that its matrices are held in are rounded as the kernels round
them, sums are exact.  Also the sizes at which the tests compare every kernel with the formula."""
import torch

NS = (3.4445, -4.7750, 2.0315)
KY, KA, LO = 1024.0, 512.0, 2048.0

# one workgroup a matrix, each instantiation
ONE = [(3, 60, 50), (2, 64, 120), (130 - 9, 60), (50, 250), (250, 33), (2, 64, 400), (448, 41), (2, 120, 100), (100, 128), (100, 190), (190, 100), (128, 300), (2, 319, 90)]
# tiles: 64 in both products, 128 and 256, 192 and 256, 128, 64 and 128, 32, 32 and 64 with fp16 products; each wide and tall, and of no round size
TILED = [(10, 250, 300), (10, 300, 250), (20, 1000, 1030), (20, 1030, 1000), (4, 1700, 1900), (4, 1900, 1700), (6, 1040, 1000), (6, 1000, 1041), (12, 700, 300),
         (12, 300, 701), (500, 512), (512, 500), (1100, 700), (700, 1103)]
# an optimizer step's lists; the last one is what two rendering networks have
LISTS = [[s] for s in ((10, 250, 300), (10, 300, 250), (20, 1030, 1000), (20, 1000, 1030), (4, 1700, 1900), (4, 1901, 1700), (6, 1040, 1000), (12, 300, 701), (512, 500), (700, 1103))] + \
        [[(14, 256, 256), (2, 256, 319), (2, 128, 283)]]


def steps_for(shape):
    return 5 if max(shape[-2:]) <= 600 else 2


def gradient_like(shape, seed):
    gen = torch.Generator().manual_seed(seed)
    m, n = shape[-2:]
    r = max(1, min(m, n) // 2)
    d = torch.arange(1, r + 1, dtype=torch.float32) ** -0.7
    x = (torch.randn(*shape[:-1], r, generator=gen) * d) @ torch.randn(*shape[:-2], r, n, generator=gen)
    return 1e-3 * (x + 0.05 * torch.randn(*shape, generator=gen))


def turned(x):
    return x.transpose(-2, -1).contiguous()


def oracle(x, steps=5, coefficients=NS, eps=1e-7):
    """the formula in 64 bits, on x's device"""
    a, b, c = coefficients
    tall = x.shape[-2] > x.shape[-1]
    X = turned(x.double()) if tall else x.double()
    X = X / X.flatten(-2).norm(dim=-1).clamp(min=eps)[..., None, None]
    for _ in range(steps):
        A = torch.matmul(X, turned(X))
        X = a * X + torch.matmul(b * A + c * torch.matmul(A, A), X)
    return turned(X) if tall else X


def emulate(x, steps=5, coefficients=NS, split=False, keep_lo=True):
    """the tiles' route; split: three products of two planes each.  keep_lo False: what it would be if a X were taken from Y's hi plane alone."""
    a, b, c = coefficients
    tall = x.shape[-2] > x.shape[-1]
    X = turned(x.double()) if tall else x.double()
    X = X / X.flatten(-2).norm(dim=-1).clamp(min=1e-7)[..., None, None]

    def planes(v, scale):
        hi = (v * scale).float().half()
        lo = ((v * scale - hi.double()) * LO).float().half()
        return hi.double() / scale, lo.double() / (LO * scale)

    def times(p, q):
        out = torch.matmul(p[0], q[0])
        return out + torch.matmul(p[0], q[1]) + torch.matmul(p[1], q[0]) if split else out
    for _ in range(steps):
        Y = planes(X, KY)
        A = planes(times(Y, [turned(t) for t in Y]), KA)
        B = planes(b * (A[0] + A[1] if split else A[0]) + c * times(A, A), KA)
        X = a * (Y[0] + Y[1] if keep_lo else Y[0]) + times(B, Y)
    return turned(X) if tall else X


def bound(x, ref, steps, precision, coefficients=NS):
    """how far a result may be from the formula's, matrix by matrix: the kernels' error is the planes' rounding, which emulate() knows but for
    the order of sums (some 1e-7 a product).  Halfway, by ratio, between that and the error of a kernel that loses something: at fp32's
    accuracy the products of the lo planes, with fp16 products Y's lo plane in a X."""
    def off(split, keep_lo):
        return (emulate(x, steps, coefficients, split, keep_lo) - ref).flatten(-2).norm(dim=-1)
    return ((off(True, True) * off(False, True)) if precision == "fp32" else (off(False, True) * off(False, False))).sqrt()

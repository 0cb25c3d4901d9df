"""The optimizer operators' cases: what a pass is, its inputs, its plain form, and its result in 64 bits.

    orthogonalise      X <- a X + (b A + c A A) X with A = X X^T, a few times, from X = x / |x|: the singular values of x driven
                       towards 1, its singular vectors kept
    muon_step_         momentum, the above, a decayed update of the parameters, for a list of matrices or stacks of matrices
    adam_step_multi_   Adam on a list of tensors (what of a network is no hidden matrix)

``own`` False: elementary torch operations in 32 bits.  ``own`` True: the framework's calls.
"""
import math

import torch

own = False

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
STEPS, EPS = 5, 1e-7
MOMENTUM, WEIGHT_DECAY, LR = 0.95, 0.01, 5e-4
BETA1, BETA2, ADAM_EPS, ADAM_STEP = 0.9, 0.999, 1e-8, 7
TYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16}

# hidden matrices of one rendering network: 6 of 256 x 256 and the feature layer, the skip layer (256 + 63 inputs), the view layer
# (256 + 27 inputs); and what of it is no hidden matrix: the input layer with its bias, the biases, the heads
HIDDEN = "7x256x256,1x256x319,1x128x283"
BOTH = "14x256x256,2x256x319,2x128x283"
REST = "16384,256,256,256,256,256,256,256,256,128,256,257,387"


def listed():
    return [
        # the one hidden 64 x 64 layer of a hash-grid network's colour head: latency
        {"name": "orth 64x64 fp32", "op": "orthogonalise", "batch": 1, "rows": 64, "cols": 64, "dtype": "fp32"},
        # view layers of the coarse and the fine network: ragged columns
        {"name": "orth 2x128x283 bf16", "op": "orthogonalise", "batch": 2, "rows": 128, "cols": 283, "dtype": "bf16"},
        # all 256 x 256 layers of both networks
        {"name": "orth 14x256x256 fp32", "op": "orthogonalise", "batch": 14, "rows": 256, "cols": 256, "dtype": "fp32"},
        # a few tall layers of no round size
        {"name": "orth 4x1000x333 fp16", "op": "orthogonalise", "batch": 4, "rows": 1000, "cols": 333, "dtype": "fp16"},
        # a square layer in full precision
        {"name": "orth 2048x2048 fp32", "op": "orthogonalise", "batch": 1, "rows": 2048, "cols": 2048, "dtype": "fp32"},
        # a wide layer, and the largest square one
        {"name": "orth 2048x8192 bf16", "op": "orthogonalise", "batch": 1, "rows": 2048, "cols": 8192, "dtype": "bf16"},
        {"name": "orth 4096x4096 bf16", "op": "orthogonalise", "batch": 1, "rows": 4096, "cols": 4096, "dtype": "bf16"},
        # one network's and both networks' hidden matrices, once a training step
        {"name": "muon one network fp32", "op": "muon", "shapes": HIDDEN, "precision": "fp32", "nesterov": True, "scale": "spectral"},
        {"name": "muon both networks fp16", "op": "muon", "shapes": BOTH, "precision": "fp16", "nesterov": True, "scale": "spectral"},
        # matrices of a larger generic model: square ones, up and down
        {"name": "muon 1024 block fp16", "op": "muon", "shapes": "4x1024x1024,1x4096x1024,1x1024x4096", "precision": "fp16",
         "nesterov": True, "scale": "rms"},
        # the rest of both networks; and one large table
        {"name": "adam rest of both networks", "op": "adam", "sizes": REST + "," + REST},
        {"name": "adam 16M and small ones", "op": "adam", "sizes": "16777216,4099,1,65537"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _shapes(text):
    return [tuple(int(v) for v in s.split("x")) for s in text.split(",")]


def _flops(b, m, n):
    r, c = min(m, n), max(m, n)
    return b * STEPS * (3.0 * r * r * c + 1.0 * r * r * r)


def draw(rng):
    op = rng.choice(["orthogonalise", "orthogonalise", "orthogonalise", "muon", "muon", "adam"])
    most = _flops(1, 2048, 4096)
    if op == "orthogonalise":
        m, n = _log(rng, 1, 3000), _log(rng, 1, 3000)
        b = _log(rng, 1, 32)
        b = max(1, min(b, int(most / _flops(1, m, n)), (1 << 24) // (m * n)))
        return {"op": op, "batch": b, "rows": m, "cols": n, "dtype": rng.choice(sorted(TYPES))}
    if op == "muon":
        shapes = []
        for _ in range(rng.randint(1, 6)):
            m, n = _log(rng, 16, 1400), _log(rng, 16, 1400)
            shapes.append("%dx%dx%d" % (min(rng.randint(1, 8), max(1, (1 << 22) // (m * n))), m, n))
        return {"op": op, "shapes": ",".join(shapes), "precision": rng.choice(["fp32", "fp16"]), "nesterov": rng.random() < 0.7,
                "scale": rng.choice(["none", "spectral", "rms"])}
    return {"op": op, "sizes": ",".join(str(_log(rng, 1, 1 << 19)) for _ in range(rng.randint(1, 24)))}


def work(case):
    if case["op"] == "orthogonalise":
        b, m, n = case["batch"], case["rows"], case["cols"]
        return {"bytes": 2.0 * b * m * n * (4 if case["dtype"] == "fp32" else 2), "flops": _flops(b, m, n)}
    if case["op"] == "muon":
        shapes = _shapes(case["shapes"])
        return {"bytes": sum(20.0 * b * m * n for b, m, n in shapes), "flops": sum(_flops(b, m, n) for b, m, n in shapes)}
    count = sum(int(s) for s in case["sizes"].split(","))
    return {"bytes": 28.0 * count, "flops": 16.0 * count}


def _gradient(gen, b, m, n):
    """A weight gradient as training makes them: a few strong directions, a decaying tail, a floor of noise."""
    r = max(1, min(m, n) // 2)
    g = dict(generator=gen, device="cuda")
    decay = torch.arange(1, r + 1, device="cuda", dtype=torch.float32) ** -0.7
    x = torch.matmul(torch.randn(b, m, r, **g) * decay, torch.randn(b, r, n, **g))
    return 1e-3 * (x + 0.05 * torch.randn(b, m, n, **g))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(int(seed))
    state = {"case": dict(case)}
    g = dict(generator=gen, device="cuda")
    if case["op"] == "orthogonalise":
        state["x"] = _gradient(gen, case["batch"], case["rows"], case["cols"]).to(TYPES[case["dtype"]])
    elif case["op"] == "muon":
        shapes = _shapes(case["shapes"])
        state["params"] = [(torch.rand(s, **g) * 2 - 1) / math.sqrt(s[2]) for s in shapes]
        state["grads"] = [_gradient(gen, *s) for s in shapes]
        state["buffers"] = [5 * _gradient(gen, *s) for s in shapes]
    else:
        sizes = [int(s) for s in case["sizes"].split(",")]
        n = sum(sizes)                 # ranges of flat buffers, as a network's parameters are here
        flat = {"params": 0.1 * torch.randn(n, **g), "grads": 1e-3 * torch.randn(n, **g), "m": 3e-4 * torch.randn(n, **g),
                "v": 1e-6 * torch.rand(n, **g)}
        state.update({k: list(t.split(sizes)) for k, t in flat.items()}, flat=flat)
    return state


def _plain_orthogonalise(x):
    a, b, c = COEFFICIENTS
    tall = x.shape[-2] > x.shape[-1]
    X = x.float()
    if tall:
        X = X.mT.contiguous()
    norm = X.double().square().sum((-2, -1), keepdim=True).sqrt().float()
    X = X / norm.clamp(min=EPS)
    for _ in range(STEPS):
        A = X @ X.mT
        X = a * X + (b * A + c * (A @ A)) @ X
    return X.mT.contiguous() if tall else X


def _scale(how, m, n):
    return math.sqrt(max(1.0, m / n)) if how == "spectral" else 0.2 * math.sqrt(max(m, n)) if how == "rms" else 1.0


def run(state):
    case = state["case"]
    if case["op"] == "orthogonalise":
        if own:
            import spin_nerf_amd as S
            return S.orthogonalise(state["x"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS)
        return _plain_orthogonalise(state["x"]).to(state["x"].dtype)
    if case["op"] == "muon":
        if own:
            import spin_nerf_amd as S
            S.muon_step_(state["params"], state["grads"], state["buffers"], LR, momentum=MOMENTUM, nesterov=case["nesterov"],
                         weight_decay=WEIGHT_DECAY, scale=case["scale"], steps=STEPS, coefficients=COEFFICIENTS, eps=EPS,
                         precision=case["precision"])
        else:
            for p, g, m in zip(state["params"], state["grads"], state["buffers"]):
                m.mul_(MOMENTUM).add_(g)
                o = _plain_orthogonalise(g + MOMENTUM * m if case["nesterov"] else m)
                p.mul_(1 - LR * WEIGHT_DECAY).sub_(o, alpha=LR * _scale(case["scale"], p.shape[1], p.shape[2]))
        return {"params": state["params"], "buffers": state["buffers"]}
    if own:
        import spin_nerf_amd as S
        S.adam_step_multi_(state["params"], state["grads"], state["m"], state["v"], LR, ADAM_STEP, BETA1, BETA2, ADAM_EPS)
    else:
        for p, g, m, v in zip(state["params"], state["grads"], state["m"], state["v"]):
            m.mul_(BETA1).add_(g, alpha=1 - BETA1)
            v.mul_(BETA2).addcmul_(g, g, value=1 - BETA2)
            p.addcdiv_(m, v.sqrt().div_(math.sqrt(1 - BETA2 ** ADAM_STEP)).add_(ADAM_EPS), value=-LR / (1 - BETA1 ** ADAM_STEP))
    return {k: state["flat"][k] for k in ("params", "m", "v")}


def _exact_orthogonalise(x):
    """The same map in 64 bits, on the shorter side's Gram matrix alone: with G = X X^T and P = a + b G + c G G, a step takes X to
    P X and G to P G P; the result is the product of the P, times X."""
    a, b, c = COEFFICIENTS
    X = x.double()
    tall = X.shape[-2] > X.shape[-1]
    X = X.transpose(-2, -1).contiguous() if tall else X
    X = X / torch.linalg.vector_norm(X, dim=(-2, -1), keepdim=True).clamp(min=EPS)
    G = torch.matmul(X, X.transpose(-2, -1).contiguous())
    one = torch.eye(G.shape[-1], dtype=torch.float64, device=x.device).expand_as(G)
    Q = one
    for _ in range(STEPS):
        P = a * one + torch.matmul(G, b * one + c * G)
        Q = torch.matmul(P, Q)
        G = torch.matmul(torch.matmul(P, G), P)
    O = torch.matmul(Q, X)
    return O.transpose(-2, -1).contiguous() if tall else O


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orthogonalise":
        return _exact_orthogonalise(state["x"])
    if case["op"] == "muon":
        P, M = [], []
        for p, g, m in zip(state["params"], state["grads"], state["buffers"]):
            p, g, m = p.double(), g.double(), m.double()
            m = MOMENTUM * m + g
            o = _exact_orthogonalise(g + MOMENTUM * m if case["nesterov"] else m)
            P.append((1 - LR * WEIGHT_DECAY) * p - LR * _scale(case["scale"], p.shape[1], p.shape[2]) * o)
            M.append(m)
        return {"params": P, "buffers": M}
    p, g, m, v = (state["flat"][k].double() for k in ("params", "grads", "m", "v"))
    m = BETA1 * m + (1 - BETA1) * g
    v = BETA2 * v + (1 - BETA2) * g * g
    p = p - LR * (m / (1 - BETA1 ** ADAM_STEP)) / ((v / (1 - BETA2 ** ADAM_STEP)).sqrt() + ADAM_EPS)
    return {"params": p, "m": m, "v": v}

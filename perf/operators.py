"""What the operators of the training step's two ends cost, and what they compute: the log likelihood of the joint's pixel under a heat map
(with the map's entropy and its most likely pixels) and its gradient, the orthogonalised update of a weight matrix, and the optimizer step
built on it.

``own`` False: the plain forms below, elementary torch operations in 32 bits.  ``own`` True: the calls of this package.
"""
import math

import torch

own = False
DEV = "cuda"
COEFFICIENTS = (3.4445, -4.7750, 2.0315)     # of the quintic iteration x -> a x + (b A + c A^2) x, A = x x^T
EPS = 1e-7
LARGEST_FLOPS = 1.4e12                       # of the largest listed case of orthogonalize
LARGEST_VALUES = 2.1e8                       # of the largest listed case of log_likelihood


def listed():
    return [
        # one bottleneck weight (1x1, 128 -> 64) alone: latency
        dict(name="orth-1x64x128-fp32", op="orth", batch=1, rows=64, cols=128, dtype="fp32"),
        # the 3x3 weights of the heads and the stem of the default network, as a batch of bf16 gradients
        dict(name="orth-13x128x1152-bf16", op="orth", batch=13, rows=128, cols=1152, dtype="bf16"),
        # odd sizes, more rows than columns
        dict(name="orth-5x1031x517-fp32", op="orth", batch=5, rows=1031, cols=517, dtype="fp32"),
        # a wide layer, the largest in 32 bits
        dict(name="orth-1x2048x8192-fp32", op="orth", batch=1, rows=2048, cols=8192, dtype="fp32"),
        # a square one, the largest in 16 bits
        dict(name="orth-1x4096x4096-bf16", op="orth", batch=1, rows=4096, cols=4096, dtype="bf16"),
        # the optimizer step of the 14-joint network with 128 features, and of the 42-joint one with 256
        dict(name="muon-J14-F128", op="muon", joints=14, stage=2, features=128, level=4, kernel=3),
        dict(name="muon-J42-F256", op="muon", joints=42, stage=2, features=256, level=4, kernel=3),
        # the confidence read-out of ONE frame, as it is served: 14 heat maps of 64 x 64
        dict(name="like-1x14x4096-fp32-top5", op="like", batch=1, joints=14, size=4096, dtype="fp32", scale=True, mask="sample", top=5, train=False),
        # the same of a validation batch
        dict(name="like-32x14x4096-fp32-top5", op="like", batch=32, joints=14, size=4096, dtype="fp32", scale=True, mask="sample", top=5, train=False),
        # one row of a long categorical axis, odd, 16 bits
        dict(name="like-1x1x100003-bf16-top8", op="like", batch=1, joints=1, size=100003, dtype="bf16", scale=False, mask="none", top=8, train=False),
        # a training step's loss: 128 samples of 42 maps of 128 x 128, and rows of a long axis in 16 bits
        dict(name="like-128x42x16384-fp32-train", op="like", batch=128, joints=42, size=16384, dtype="fp32", scale=True, mask="sample", top=0, train=True),
        dict(name="like-4096x1x50001-bf16-train", op="like", batch=4096, joints=1, size=50001, dtype="bf16", scale=False, mask="none", top=0, train=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("orth", "orth", "muon", "like", "like"))
    if op == "orth":
        while True:
            case = dict(op="orth", batch=rng.choice((1, 1, _log_int(rng, 1, 32))), rows=_log_int(rng, 1, 4096), cols=_log_int(rng, 1, 8192),
                        dtype=rng.choice(("fp32", "bf16")))
            if work(case)["flops"] <= LARGEST_FLOPS:
                return case
    if op == "muon":
        return dict(op="muon", joints=rng.randint(1, 42), stage=rng.randint(1, 3), features=8 * rng.randint(4, 32), level=rng.randint(1, 5),
                    kernel=rng.choice((1, 3, 3, 5)))
    train = rng.random() < 0.5
    while True:
        heat = rng.random() < 0.5
        case = dict(op="like", batch=_log_int(rng, 1, 4096), joints=rng.randint(1, 42) if heat else 1, size=_log_int(rng, 1, 16384 if heat else 131072),
                    dtype="fp32" if heat else rng.choice(("fp32", "bf16")), scale=heat, mask=rng.choice(("none", "sample")) if heat else "none",
                    top=0 if train else rng.randint(0, 16), train=train)
        if case["batch"] * case["joints"] * case["size"] <= LARGEST_VALUES:
            return case


# ---------------------------------------------------------------------------------------------------------------------- the cases' inputs

def _shapes(joints, stage, features, level, kernel):
    """The parameter shapes of the stacked hourglass, in their order in the flat buffer."""
    def conv(o, i, k):
        return [(o, i, k, k), (o,)]

    def norm(c):
        return [(c,), (c,)]

    def block(f):
        h = f // 2
        return norm(f) + conv(h, f, 1) + norm(h) + conv(h, h, 3) + norm(h) + conv(f, h, 1)

    def head(f):
        return (conv(f, f, kernel) + norm(f)) * 3 + conv(joints, f, kernel)

    widths = [1, 32]
    widths += [min(32 << i, features) for i in range(1, 5) if (32 << (i - 1)) < features] + [features]
    shapes = [s for i, o in zip(widths, widths[1:]) for s in conv(o, i, kernel) + norm(o)]
    for s in range(stage):
        shapes += conv(features, features if s == 0 else 2 * joints + 1, 1)
        shapes += block(features) * (2 * (level + 1) + 1)
        shapes += [(joints, 1)] + head(features) + head(features)
    return shapes


def _matrices(shapes):
    """(offset, rows, cols) of every parameter that is a matrix (an OIHW kernel is one row per output channel), and the mask of the rest."""
    sizes = [math.prod(s) for s in shapes]
    offsets = [sum(sizes[:i]) for i in range(len(sizes))]
    found = [(o, s[0], n // s[0]) for o, s, n in zip(offsets, shapes, sizes) if len(s) > 1 and min(s[0], n // s[0]) > 1]
    return found, sum(sizes)


def _gradient(gen, batch, rows, cols):
    """What a weight gradient looks like: a few strong directions over a floor of noise."""
    r = min(rows, cols, 16)
    strong = torch.randn(batch, rows, r, device=DEV, generator=gen) / torch.arange(1, r + 1, device=DEV)
    right = torch.randn(batch, r, cols, device=DEV, generator=gen)
    return 1e-3 * (strong @ right + torch.randn(batch, rows, cols, device=DEV, generator=gen))


def prepare(case, seed):
    gen = torch.Generator(device=DEV).manual_seed(int(seed))
    state = {"case": case}
    if case["op"] == "orth":
        x = _gradient(gen, case["batch"], case["rows"], case["cols"])
        state["x"] = x.to(torch.bfloat16) if case["dtype"] == "bf16" else x
    elif case["op"] == "muon":
        shapes = _shapes(case["joints"], case["stage"], case["features"], case["level"], case["kernel"])
        matrices, total = _matrices(shapes)
        state["shapes"], state["matrices"] = shapes, matrices
        state["p"] = 0.05 * torch.randn(total, device=DEV, generator=gen)
        state["buf"] = 1e-3 * torch.randn(total, device=DEV, generator=gen)
        state["v"] = (1e-3 * torch.randn(total, device=DEV, generator=gen)) ** 2
        state["g"] = 1e-3 * torch.randn(total, device=DEV, generator=gen)
        inside = torch.zeros(total, dtype=torch.bool, device=DEV)
        groups = {}
        for o, r, c in matrices:
            state["g"][o:o + r * c] = _gradient(gen, 1, r, c).reshape(-1)
            inside[o:o + r * c] = True
            groups.setdefault((r, c), []).append(o)
        # where the elements of the matrices of one shape are, and those of everything else
        state["groups"] = [(r, c, (torch.tensor(o, device=DEV)[:, None] + torch.arange(r * c, device=DEV))) for (r, c), o in groups.items()]
        state["rest"] = (~inside).nonzero().reshape(-1)
    else:
        n, j, v = case["batch"], case["joints"], case["size"]
        z = 2.0 * torch.randn(n, j, v, device=DEV, generator=gen)
        index = torch.randint(0, v, (n, j), device=DEV, generator=gen)
        z.scatter_add_(2, index[..., None], torch.full((n, j, 1), 4.0, device=DEV))      # (a trained map: the joint's pixel stands out)
        state["z"] = z.to(torch.bfloat16) if case["dtype"] == "bf16" else z
        state["index"] = torch.where(torch.rand(n, j, device=DEV, generator=gen) < 0.05, -torch.ones_like(index), index)   # some joints are not annotated
        state["w"] = 0.5 + torch.rand(j, device=DEV, generator=gen) if case["scale"] else None
        state["mask"] = None
        if case["mask"] == "sample":                                                      # the hand's pixels; one sample in 64 has none
            mask = torch.rand(n, 1, v, device=DEV, generator=gen) < 0.6
            state["mask"] = (mask & (torch.rand(n, 1, 1, device=DEV, generator=gen) < 63 / 64)).float()
        if case["train"]:
            state["glogp"] = -torch.rand(n, j, device=DEV, generator=gen) / (n * j)
            state["gentropy"] = 0.1 * torch.randn(n, j, device=DEV, generator=gen) / (n * j)
    return state


# ---------------------------------------------------------------------------------------------------------------------- plain forms

def _orthogonalize(x):
    a, b, c = COEFFICIENTS
    y = x.float()
    tall = y.shape[-2] > y.shape[-1]
    y = y.mT.contiguous() if tall else y
    y = y / (torch.linalg.vector_norm(y, dim=(-2, -1), keepdim=True) + EPS)

    def step(y):
        g = y @ y.mT
        return a * y + (b * g + c * (g @ g)) @ y

    y = step(step(step(step(step(y)))))
    return (y.mT if tall else y).contiguous().to(x.dtype)


LR, MOMENTUM, DECAY, BETA1, BETA2, ADAM_EPS, AT_STEP = 2e-3, 0.95, 0.01, 0.9, 0.999, 1e-8, 100


def _muon_group(state, rows, cols, at):
    p, g, buf = state["p"], state["g"], state["buf"]
    m = MOMENTUM * buf[at] + g[at]
    o = _orthogonalize((g[at] + MOMENTUM * m).view(-1, rows, cols)).view_as(m)
    buf[at] = m
    p[at] = p[at] * (1 - LR * DECAY) - LR * 0.2 * math.sqrt(max(rows, cols)) * o


def _muon(state):
    for group in state["groups"]:
        _muon_group(state, *group)
    at, p, g = state["rest"], state["p"], state["g"]
    m = BETA1 * state["buf"][at] + (1 - BETA1) * g[at]
    v = BETA2 * state["v"][at] + (1 - BETA2) * g[at] ** 2
    state["buf"][at], state["v"][at] = m, v
    p[at] = p[at] * (1 - LR * DECAY) - LR / (1 - BETA1 ** AT_STEP) * m / ((v / (1 - BETA2 ** AT_STEP)).sqrt() + ADAM_EPS)
    return {"p": p, "buf": state["buf"], "v": state["v"]}


def _likelihood(state):
    case, z, index, w, mask = state["case"], state["z"], state["index"], state["w"], state["mask"]
    s = z.float()
    if w is not None:
        s = s * w[:, None]
    if mask is not None:
        s = torch.where(mask != 0, s, -math.inf)
    top = s.amax(-1, keepdim=True)
    shifted = s - torch.where(torch.isfinite(top), top, 0.0)
    e = torch.exp(shifted)
    # (the sums in 64 bits: where one pixel has nearly everything, what the others add to its 1 is the whole answer)
    total = e.sum(-1, keepdim=True, dtype=torch.float64)
    some = total > 0                                              # (a row without a pixel: every log probability is -inf)
    log_total = torch.where(some, total, 1.0).log()
    p = torch.where(some, e / total.float(), 0.0)
    logs = shifted - log_total.float()
    plogp = torch.where(p > 0, p * logs, 0.0)
    entropy = -plogp.sum(-1, dtype=torch.float64).float()
    given = index >= 0
    logp = torch.where(given, logs.gather(-1, index.clamp(min=0)[..., None])[..., 0], 0.0)
    out = {"logp": logp, "entropy": entropy}
    if case["top"]:
        k = min(case["top"], case["size"])
        # one whole number orders by value, then by the lowest index
        bits = s.view(torch.int32).to(torch.int64)
        order = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits)
        key = order * (1 << 20) + ((1 << 20) - 1 - torch.arange(case["size"], device=z.device))
        at = torch.topk(key, k, dim=-1).indices
        at_log = logs.gather(-1, at)
        at = torch.where(at_log > -math.inf, at, -1)
        pad = case["top"] - k
        out["top_logp"] = torch.nn.functional.pad(at_log, (0, pad), value=-math.inf)
        out["top_index"] = torch.nn.functional.pad(at, (0, pad), value=-1)
    if case["train"]:
        glogp = torch.where(given, state["glogp"], 0.0)[..., None]
        hit = (torch.arange(case["size"], device=z.device) == index[..., None]) & (s > -math.inf)
        ds = glogp * torch.where(hit, -torch.expm1(logs), -p) - state["gentropy"][..., None] * (plogp + p * entropy[..., None])
        if w is not None:
            out["gw"] = (ds * z.float()).sum(dim=(0, 2), dtype=torch.float64).float()
            ds = ds * w[:, None]
        out["gz"] = ds.to(z.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------- the package's calls

def _own_muon(state):
    from pixelwiseregression_amd import optim
    if "optimizer" not in state:                                  # a program keeps it, with its momentum, from step to step
        state["optimizer"] = optim.Muon(state["p"], state["shapes"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY, beta1=BETA1, beta2=BETA2,
                                        adam_eps=ADAM_EPS, coefficients=COEFFICIENTS, eps=EPS, buf=state["buf"], v=state["v"])
    state["optimizer"].steps = AT_STEP - 1
    state["optimizer"].step(state["g"])
    return {"p": state["p"], "buf": state["buf"], "v": state["v"]}


def _own_likelihood(state):
    from pixelwiseregression_amd import ops
    case, z, w = state["case"], state["z"], state["w"]
    if not case["train"]:
        r = ops.log_likelihood(z, state["index"], w, state["mask"], topk=case["top"])
        out = {"logp": r.logp, "entropy": r.entropy}
        if case["top"]:
            out.update(top_logp=r.top_logp, top_index=r.top_index)
        return out
    leaves = [z.detach().requires_grad_()] + ([w.detach().requires_grad_()] if w is not None else [])
    r = ops.log_likelihood(leaves[0], state["index"], leaves[1] if w is not None else None, state["mask"])
    grads = torch.autograd.grad([r.logp, r.entropy], leaves, [state["glogp"], state["gentropy"]])
    out = {"logp": r.logp, "entropy": r.entropy, "gz": grads[0]}
    if w is not None:
        out["gw"] = grads[1]
    return out


def run(state):
    op = state["case"]["op"]
    if own:
        if op == "orth":
            from pixelwiseregression_amd import ops
            return ops.orthogonalize(state["x"], coefficients=COEFFICIENTS, eps=EPS)
        return _own_muon(state) if op == "muon" else _own_likelihood(state)
    return _orthogonalize(state["x"]) if op == "orth" else _muon(state) if op == "muon" else _likelihood(state)


# ---------------------------------------------------------------------------------------------------------------------- what they cost

def _iteration_flops(rows, cols):
    """Five steps: x x^T and A A are symmetric (half of the products), (b A + c A^2) x is not."""
    m, n = min(rows, cols), max(rows, cols)
    return 5 * (m * (m + 1) * n + m * m * (m + 1) + 2 * m * m * n)


def work(case):
    if case["op"] == "orth":
        n = case["batch"] * case["rows"] * case["cols"]
        return {"bytes": 2 * n * (2 if case["dtype"] == "bf16" else 4), "flops": case["batch"] * _iteration_flops(case["rows"], case["cols"])}
    if case["op"] == "muon":
        matrices, total = _matrices(_shapes(case["joints"], case["stage"], case["features"], case["level"], case["kernel"]))
        inside = sum(r * c for _, r, c in matrices)
        return {"bytes": 4 * (5 * inside + 7 * (total - inside)), "flops": sum(_iteration_flops(r, c) for _, r, c in matrices)}
    rows, v = case["batch"] * case["joints"], case["size"]
    item = 2 if case["dtype"] == "bf16" else 4
    b = rows * v * item * (2 if case["train"] else 1) + rows * (8 + 8 + 12 * case["top"] + (8 if case["train"] else 0))
    return {"bytes": b + (case["batch"] * v * 4 if case["mask"] == "sample" else 0), "flops": rows * v * (10 if case["train"] else 5)}


# ---------------------------------------------------------------------------------------------------------------------- 64 bits

def _polar(x):
    """The iteration in 64 bits as a polynomial of the Gram matrix alone: x5 = P x0, with P and A kept commuting."""
    a, b, c = COEFFICIENTS
    x = x.double()
    if x.shape[-2] > x.shape[-1]:
        return _polar(x.mT.contiguous()).mT
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    gram = torch.matmul(x, x.mT.contiguous())
    eye = torch.eye(x.shape[-2], dtype=torch.float64, device=x.device)
    p = eye.expand_as(gram)
    for _ in range(5):
        q = a * eye + torch.matmul(b * eye + c * gram, gram)
        p = torch.matmul(q, p)
        gram = torch.matmul(torch.matmul(q, gram), q)
    return torch.matmul(p, x)


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "orth":
        return _polar(state["x"])
    if case["op"] == "muon":
        p, g, m, v = (state[k].double() for k in ("p", "g", "buf", "v"))
        new_m, new_v = BETA1 * m + (1 - BETA1) * g, BETA2 * v + (1 - BETA2) * g * g
        den = torch.sqrt(new_v / (1 - BETA2 ** AT_STEP)) + ADAM_EPS
        new_p = p - LR * DECAY * p - LR * (new_m / (1 - BETA1 ** AT_STEP)) / den
        for o, r, c in state["matrices"]:
            at = slice(o, o + r * c)
            new_m[at] = MOMENTUM * m[at] + g[at]
            u = (g[at] + MOMENTUM * new_m[at]).view(r, c)
            new_p[at] = p[at] - LR * DECAY * p[at] - LR * 0.2 * max(r, c) ** 0.5 * _polar(u).reshape(-1)
            new_v[at] = v[at]
        return {"p": new_p, "buf": new_m, "v": new_v}
    z, index, w, mask = state["z"].double(), state["index"], state["w"], state["mask"]
    s = z if w is None else z * w.double()[:, None]
    allowed = torch.ones_like(s, dtype=torch.bool) if mask is None else (mask != 0).expand_as(s)
    s = s.masked_fill(~allowed, -math.inf)
    some = allowed.any(-1)
    logs = torch.log_softmax(s, -1).masked_fill(~allowed, -math.inf)
    p = torch.exp(logs)
    finite = logs.masked_fill(~allowed, 0.0)
    entropy = -(p * finite).sum(-1)
    t = index.clamp(min=0)[..., None]
    logp = logs.gather(-1, t)[..., 0].masked_fill(index < 0, 0.0)
    out = {"logp": logp, "entropy": entropy}
    if case["top"]:
        out.update(top_logp=None, top_index=None)
        if case["top"] <= case["size"]:
            out["top_logp"] = torch.topk(logs, case["top"], dim=-1).values
    if case["train"]:
        gl, ge = state["glogp"].double().masked_fill(index < 0, 0.0)[..., None], state["gentropy"].double()[..., None]
        one = torch.zeros_like(p).scatter_(-1, t, 1.0) * allowed
        ds = (gl * (one - p) - ge * p * (finite + entropy[..., None])) * some[..., None]
        if w is not None:
            out["gw"] = (ds * z).sum(-1).sum(0)
            ds = ds * w.double()[:, None]
        out["gz"] = ds
    return out

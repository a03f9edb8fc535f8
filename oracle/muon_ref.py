"""float64 restatement of the Newton-Schulz orthogonalisation and of the optimizer step built on it, and the same iteration with operands rounded
where the kernels round theirs (the yardstick of the tests: how far such an evaluation is from float64 on a given matrix)."""
import numpy as np

COEFFICIENTS = (3.4445, -4.7750, 2.0315)
SCALE = 4096.0


def newton_schulz(x, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    a, b, c = coefficients
    x = np.asarray(x, np.float64)
    if x.shape[0] > x.shape[1]:
        return newton_schulz(x.T, steps, coefficients, eps).T
    x = x / (np.sqrt((x * x).sum()) + eps)
    for _ in range(steps):
        g = x @ x.T
        x = a * x + (b * g + c * (g @ g)) @ x
    return x


def _pair(v):
    with np.errstate(over="ignore", invalid="ignore"):
        s = (np.asarray(v, np.float32) * np.float32(SCALE)).astype(np.float32)
        hi = s.astype(np.float16).astype(np.float32)
        lo = (s - hi).astype(np.float16).astype(np.float32)
    return hi, lo


def newton_schulz_rounded(x, terms, steps=5, coefficients=COEFFICIENTS, eps=1e-7):
    """Everything stored as a pair of fp16 (22 bits); products of `terms` = 3 (hi hi + hi lo + lo hi) or 1 (hi hi, the diagonals of the symmetric
    matrices apart in fp32), sums in fp32."""
    a, b, c = (np.float32(v) for v in coefficients)
    x = np.asarray(x, np.float64)
    if x.shape[0] > x.shape[1]:
        return newton_schulz_rounded(x.T, terms, steps, coefficients, eps).T
    x = (x / (np.sqrt((x * x).sum()) + eps)).astype(np.float32)
    inv = np.float32(1.0 / SCALE)

    def value(p):
        return (p[0] + p[1]) * inv

    def product(p, q):
        r = p[0] @ q[0].T
        if terms == 3:
            r = r + (p[0] @ q[1].T + p[1] @ q[0].T)
        return r * inv * inv

    def bare(m):
        return m - np.diag(np.diag(m))

    for _ in range(steps):
        px = _pair(x)
        g = product(px, px)
        if terms == 3:
            pg = _pair(g)
            pb = _pair(b * value(pg) + c * product(pg, pg))
            x = a * value(px) + product(pb, (px[0].T, px[1].T))
        else:
            d = np.diag(g).copy()
            pg = _pair(bare(g))
            off = value(pg)
            gg = product(pg, pg) + (d[:, None] + d[None]) * off + np.diag(d * d)
            bb = b * (off + np.diag(d)) + c * gg
            pb = _pair(bare(bb))
            x = a * value(px) + np.diag(bb)[:, None] * (px[0] * inv) + product(pb, (px[0].T, px[1].T))
    return x.astype(np.float64)


def step(p, g, buf, v, params, lr=1e-3, momentum=0.95, nesterov=True, weight_decay=0.0, update_rms=0.2, ns_steps=5, coefficients=COEFFICIENTS, eps=1e-7,
         beta1=0.9, beta2=0.999, adam_eps=1e-8, t=1, grad_scale=1.0):
    """One step on flat arrays; params: (offset, rows, cols).  Returns (p, buf, v, the matrices' directions by offset)."""
    p, g, buf, v = (np.asarray(q, np.float64).copy() for q in (p, g, buf, v))
    g *= grad_scale
    dirs = {}
    for off, rows, cols in params:
        at = slice(off, off + rows * cols)
        if min(rows, cols) == 1:
            buf[at] = beta1 * buf[at] + (1 - beta1) * g[at]
            v[at] = beta2 * v[at] + (1 - beta2) * g[at] ** 2
            den = np.sqrt(v[at] / (1 - beta2 ** t)) + adam_eps
            p[at] = p[at] * (1 - lr * weight_decay) - lr * buf[at] / (1 - beta1 ** t) / den
            continue
        buf[at] = momentum * buf[at] + g[at]
        u = g[at] + momentum * buf[at] if nesterov else buf[at]
        dirs[off] = u.reshape(rows, cols)
        o = newton_schulz(dirs[off], ns_steps, coefficients, eps)
        p[at] = p[at] * (1 - lr * weight_decay) - lr * update_rms * np.sqrt(max(rows, cols)) * o.reshape(-1)
    return p, buf, v, dirs

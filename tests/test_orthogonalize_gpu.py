"""GPU: orthogonalize and the Muon step against the float64 oracle.

Tolerances.  How far an evaluation with the kernels' roundings is from float64 depends on the matrix (small singular values are amplified), so it is
measured on the matrix at hand: the oracle runs the iteration once more with every operand rounded where the kernels round it (pairs of fp16,
22 bits; products of the high halves only for bf16).  The kernel has to be within 3 times that distance (its sums run in another order) plus the
rounding of the result: 2^-24 of an entry, 2^-8 for bf16."""
import math

import numpy as np
import pytest
import torch

from oracle import muon_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def matrix(rows, cols, kind, seed):
    r = np.random.default_rng(seed)
    if kind == "gauss":
        return r.standard_normal((rows, cols))
    if kind == "gradient":                                   # a few strong directions over noise
        k = min(rows, cols, 8)
        return 1e-3 * ((r.standard_normal((rows, k)) / np.arange(1, k + 1)) @ r.standard_normal((k, cols)) + r.standard_normal((rows, cols)))
    if kind == "lowrank":
        k = max(1, min(rows, cols) // 8)
        return r.standard_normal((rows, k)) @ r.standard_normal((k, cols))
    m = min(rows, cols)                                       # "decay": singular values over four decades
    u, _ = np.linalg.qr(r.standard_normal((rows, m)))
    v, _ = np.linalg.qr(r.standard_normal((cols, m)))
    return (u * np.exp(-9.2 * np.arange(m) / m)) @ v.T


def bound(x, bf16, **kw):
    ref = muon_ref.newton_schulz(x, **kw)
    off = np.linalg.norm(muon_ref.newton_schulz_rounded(x, 1 if bf16 else 3, **kw) - ref)
    return ref, 3 * off + (2.0 ** -8 if bf16 else 2.0 ** -22) * np.linalg.norm(ref)


def check(x, dtype=torch.float32, **kw):
    from pixelwiseregression_amd import ops
    xt = torch.from_numpy(np.asarray(x)).to(dtype)
    got = ops.orthogonalize(xt.to(DEV), **kw).cpu().double().numpy().reshape((-1,) + xt.shape[-2:])
    for g, q in zip(got, xt.double().numpy().reshape((-1,) + xt.shape[-2:])):
        ref, tol = bound(q, dtype == torch.bfloat16, **kw)
        assert np.isfinite(g).all()
        assert np.linalg.norm(g - ref) <= tol, (np.linalg.norm(g - ref), tol, np.linalg.norm(ref))
    return got


SIZES = [(1, 1), (1, 9), (9, 1), (2, 3), (14, 1152), (32, 9), (63, 65), (64, 64), (64, 576), (65, 64), (128, 29), (128, 1152), (200, 131), (257, 300)]


@pytest.mark.parametrize("rows,cols", SIZES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_sizes(rows, cols, dtype):
    check(matrix(rows, cols, "gauss", rows + cols), dtype)


@pytest.mark.parametrize("kind", ["gradient", "lowrank", "decay"])
@pytest.mark.parametrize("rows,cols", [(64, 128), (300, 100), (96, 96)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_spectra(rows, cols, kind, dtype):
    check(matrix(rows, cols, kind, 7), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,rows,cols", [(3, 40, 70), (64, 130, 260), (96, 129, 140), (70, 260, 130), (300, 20, 30)])
def test_batches(batch, rows, cols, dtype):
    check(np.stack([matrix(rows, cols, "gradient", k) for k in range(batch)]), dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,rows,cols", [(1, 1100, 4400), (4, 500, 2100), (30, 400, 450), (52, 390, 400), (1, 20, 8000), (3, 2300, 70), (4, 300, 2000),
                                             (2, 6, 70000), (28, 760, 768), (2, 2100, 1100)])
def test_products_split_along_k(batch, rows, cols, dtype):
    """Symmetric products whose tiles do not fill the chip: few of them, a last round of few, small ones with long sums."""
    x = np.random.default_rng(5).standard_normal((batch, rows, cols)).astype(np.float32)
    x[batch // 2:] = x[:batch - batch // 2]                   # (float64 checks two of them; the others have to be the same bits)
    from pixelwiseregression_amd import ops
    xt = torch.from_numpy(x).to(dtype)
    got = ops.orthogonalize(xt.to(DEV)).cpu()
    for k in {0, (batch - 1) // 2}:
        ref, tol = bound(xt[k].double().numpy(), dtype == torch.bfloat16)
        assert np.linalg.norm(got[k].double().numpy() - ref) <= tol
    one = torch.stack([ops.orthogonalize(xt[k:k + 1].to(DEV))[0].cpu() for k in (0, batch - 1)])
    for a, b in zip(one, (got[0], got[-1])):                  # (alone, a matrix's sums are split elsewhere: the same up to their rounding)
        assert (a.double() - b.double()).norm() <= tol


@pytest.mark.parametrize("steps", [1, 2, 3, 6])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_steps_and_coefficients(steps, dtype):
    x = matrix(70, 90, "gauss", 3)
    check(x, dtype, steps=steps)
    check(x, dtype, steps=steps, coefficients=(1.5, -0.5, 0.0))
    check(x, dtype, steps=steps, coefficients=(15 / 8, -10 / 8, 3 / 8), eps=0.0)


@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e-7, 1.0, 1e30])
def test_any_norm(scale):
    """A norm far below eps gives nearly nothing (eps is what divides), a huge one is divided away."""
    x = (matrix(60, 50, "gauss", 1) * scale).astype(np.float32).astype(np.float64)
    from pixelwiseregression_amd import ops
    got = ops.orthogonalize(torch.from_numpy(x).float().to(DEV)).cpu().double().numpy()
    ref = muon_ref.newton_schulz(x)
    # entries below 2^-24 / 4096 are not kept by the pairs: 480 x that per entry after five steps
    floor = 480 * 2.0 ** -36 * math.sqrt(x.size)
    off = np.linalg.norm(muon_ref.newton_schulz_rounded(x, 3) - ref)
    assert np.linalg.norm(got - ref) <= 3 * off + 2.0 ** -22 * np.linalg.norm(ref) + floor


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_zero_and_not_finite(dtype):
    from pixelwiseregression_amd import ops
    x = torch.zeros(3, 40, 50, device=DEV, dtype=dtype)
    x[1] = torch.randn(40, 50).to(dtype)
    x[2] = x[1]
    x[2, 3, 4] = math.nan
    y = ops.orthogonalize(x)
    assert (y[0] == 0).all() and torch.isfinite(y[1]).all() and torch.isnan(y[2]).any()
    assert torch.equal(y[1], ops.orthogonalize(x[1]))                       # a neighbour's NaN stays there
    x[2, 3, 4] = math.inf
    assert not torch.isfinite(ops.orthogonalize(x)[2]).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_results_and_in_place(dtype):
    from pixelwiseregression_amd import ops
    base = torch.randn(5, 60, 90, device=DEV).to(dtype)
    for x in (base[:, 3:40, 5:78], base[1:4, ::2, 1:], base.mT, base.permute(1, 0, 2), base[::2], base[2, 7:, 3:64], base[:1].expand(4, 60, 90)):
        assert torch.equal(ops.orthogonalize(x), ops.orthogonalize(x.contiguous()))
    four = base[:4].reshape(2, 2, 60, 90)
    assert torch.equal(ops.orthogonalize(four).reshape(4, 60, 90), ops.orthogonalize(base[:4]))
    want = ops.orthogonalize(base)
    out = torch.empty_like(base)
    assert ops.orthogonalize(base, out=out) is out and torch.equal(out, want)
    z = base.clone()
    assert ops.orthogonalize(z, out=z) is z and torch.equal(z, want)
    assert ops.orthogonalize(base[:0]).shape == (0, 60, 90) and ops.orthogonalize(base[:, :0]).shape == (5, 0, 90)


def test_offsets_beyond_32_bits():
    """2.2e9 entries: the last matrices are the first ones again"""
    from pixelwiseregression_amd import ops
    x = torch.zeros(33000, 256, 256, device=DEV, dtype=torch.bfloat16)
    assert x.numel() > 2 ** 31
    part = torch.randn(4, 256, 256, device=DEV).to(torch.bfloat16)
    x[:4] = part
    x[-4:] = part
    y = ops.orthogonalize(x)
    assert torch.equal(y[:4], y[-4:]) and (y[4:-4].amax() == 0) and (y[4:-4].amin() == 0)
    ref, tol = bound(part[0].double().cpu().numpy(), True)
    assert np.linalg.norm(y[-4].double().cpu().numpy() - ref) <= tol


def test_calls_on_two_streams_at_once():
    from pixelwiseregression_amd import ops
    shapes = [(64, 128), (5, 130, 260), (20, 8000), (1100, 1500)]
    xs = [torch.randn(s, device=DEV) for s in shapes]
    z, index = torch.randn(32, 14, 4096, device=DEV), torch.zeros(32, 14, dtype=torch.long, device=DEV)
    want = [ops.orthogonalize(x) for x in xs]
    like = ops.log_likelihood(z, index, topk=5)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append([ops.orthogonalize(x) for x in xs] + list(ops.log_likelihood(z, index, topk=5)))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want + list(like)))


def test_a_result_that_overlaps_is_refused():
    from pixelwiseregression_amd import ops
    store = torch.randn(4, 5, 6, device=DEV)
    for x, out in ((store[:3], store[1:]), (store[:1].expand(3, 5, 6), store[:3]), (store[0, :, :5].T, store[0, :, :5].T)):
        with pytest.raises(ValueError):
            ops.orthogonalize(x, out=out)
    square = torch.randn(6, 6, device=DEV)
    with pytest.raises(ValueError):
        ops.orthogonalize(square.T, out=square)
    want = ops.orthogonalize(store[1])
    ops.orthogonalize(store[1], out=store[2])                 # neighbours
    assert torch.equal(store[2], want)


def test_a_strided_batch_in_both_tiles():
    """The source's batch and row strides are the caller's, the result's are not (also with enough matrices for the wide tile)."""
    from pixelwiseregression_amd import ops
    for batch in (3, 80):
        base = torch.randn(batch, 140, 300, device=DEV)
        x = base[:, 2:132, 1:262]
        assert torch.equal(ops.orthogonalize(x), ops.orthogonalize(x.contiguous()))


def test_strides_of_wide_matrices():
    from pixelwiseregression_amd import ops
    for dtype in (torch.float32, torch.bfloat16):
        x = torch.randn(2, 1104, 2603, device=DEV).to(dtype)[:, 3:1103, 2:2602]
        want = ops.orthogonalize(x.contiguous())
        assert torch.equal(ops.orthogonalize(x), want) and torch.equal(ops.orthogonalize(x), want)
        y = x.contiguous()
        assert ops.orthogonalize(y, out=y) is y and torch.equal(y, want)


@pytest.mark.parametrize("shape", [(64, 128), (20, 130, 260), (64, 140, 300), (1100, 4400)])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_repeats_streams_and_graphs(shape, dtype):
    from pixelwiseregression_amd import ops
    x = torch.randn(*shape, device=DEV).to(dtype)
    want = ops.orthogonalize(x)
    assert torch.equal(want, ops.orthogonalize(x))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        other = ops.orthogonalize(x)
    s.synchronize()
    assert torch.equal(want, other)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.orthogonalize(x)
    for k in range(3):
        x.copy_(torch.randn(*shape, generator=torch.Generator().manual_seed(k)).to(dtype))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ops.orthogonalize(x)), k


# ---------------------------------------------------------------------------------------------------------------------- the optimizer step

def params_of(shapes):
    out, at = [], 0
    for s in shapes:
        n = math.prod(s)
        rows = s[0] if len(s) > 1 else 1
        out.append((at, rows, n // rows))
        at += n
    return out, at


MIXED = [(64, 32, 3, 3), (64,), (14, 1), (1, 200), (5, 7), (33, 70), (70,), (130, 64, 1, 1), (2, 2), (3,)]


def muon_case(shapes, seed=0, **kw):
    from pixelwiseregression_amd import optim
    params, n = params_of(shapes)
    r = np.random.default_rng(seed)
    p, g = 0.05 * r.standard_normal(n), 1e-3 * r.standard_normal(n)
    buf, v = 1e-3 * r.standard_normal(n), (1e-3 * r.standard_normal(n)) ** 2
    p, g, buf, v = (q.astype(np.float32) for q in (p, g, buf, v))
    t, scale = kw.pop("t", 3), kw.pop("grad_scale", 1.0)
    d = [torch.from_numpy(q.copy()).to(DEV) for q in (p, g, buf, v)]
    opt = optim.Muon(d[0], shapes, buf=d[2], v=d[3], **kw)
    opt.steps = t - 1
    opt.step(d[1], grad_scale=scale)
    assert opt.steps == t
    f32 = {k: float(np.float32(q)) for k, q in {"beta1": 0.9, "beta2": 0.999, "momentum": 0.95, **kw}.items() if isinstance(q, float)}    # as they cross the C ABI
    rp, rb, rv, dirs = muon_ref.step(p, g, buf, v, params, t=t, grad_scale=scale, **{**kw, **f32})
    got = [q.cpu().double().numpy() for q in (d[0], d[2], d[3])]
    u = 2.0 ** -24
    g64 = np.abs(g.astype(np.float64)) * scale
    assert (np.abs(got[1] - rb) <= 4 * u * (np.abs(buf) + g64)).all()          # two products and a sum
    for off, rows, cols in params:
        at = slice(off, off + rows * cols)
        if off in dirs:
            assert np.array_equal(got[2][at], v[at])                            # a matrix has no second moment
            _, tol = bound(dirs[off], False, **{k: kw[q] for k, q in (("steps", "ns_steps"), ("coefficients", "coefficients"), ("eps", "eps")) if q in kw})
            # the direction u itself is fp32: g + mu (mu buf + g), 4 roundings of its largest term, amplified like any noise in X0: within the
            # same bound once more
            step = kw.get("lr", 1e-3) * kw.get("update_rms", 0.2) * math.sqrt(max(rows, cols))
            err = np.linalg.norm(got[0][at] - rp[at])
            assert err <= step * 4 * tol + 4 * u * np.linalg.norm(p[at]), (off, rows, cols, err, step * tol)
        else:
            assert (np.abs(got[2][at] - rv[at]) <= 6 * u * (np.abs(v[at]) + g64[at] ** 2)).all()
            # m / (sqrt(v) / c + eps): a dozen roundings of the update (powf's bias corrections among them)
            assert (np.abs(got[0][at] - rp[at]) <= 4 * u * np.abs(p[at]) + 32 * u * np.abs(rp[at] - p[at]) + 32 * u * kw.get("lr", 1e-3)).all()
    return opt, d


@pytest.mark.parametrize("kw", [dict(), dict(nesterov=False), dict(weight_decay=0.1, lr=0.01), dict(momentum=0.0), dict(ns_steps=2, eps=1e-3),
                                dict(grad_scale=0.125), dict(t=1), dict(update_rms=1.0, coefficients=(1.5, -0.5, 0.0))])
def test_muon_step(kw):
    muon_case(MIXED, **kw)


@pytest.mark.parametrize("shapes", [[(40, 50)], [(7,)], [(1, 1)], [(3000, 2)], [(128, 128, 3, 3)] * 30 + [(128,)] * 30, [(9,), (0,), (4, 0), (4, 4)], [(400, 1200), (500, 2000), (64, 64), (30,), (1000, 1000), (390, 4000)],
                                    [(300, 500), (20000,)], [(64, 64), (20, 8000), (9,), (128, 3200), (2100, 60), (3, 100)],
                                    [(1000, 2100), (64, 64), (2500, 900), (30,), (20, 400), (1000, 1000)]])
def test_muon_lists(shapes):
    muon_case(shapes, seed=4)


def test_muon_keeps_everything_else():
    """The step writes the parameters it has and nothing behind them; a state goes on where it was saved."""
    from pixelwiseregression_amd import optim
    n = sum(math.prod(s) for s in MIXED)
    store = torch.full((4, n + 64), 7.0, device=DEV)
    p, g, b, v = (store[k, :n] for k in range(4))
    torch.manual_seed(0)
    for t in (p, g, b):
        t.copy_(torch.randn(n) * 0.05)
    v.copy_(torch.rand(n) * 1e-4)
    g0 = g.clone()
    opt = optim.Muon(p, MIXED, buf=b, v=v)
    for _ in range(2):
        opt.step(g)
    torch.cuda.synchronize()
    assert (store[:, n:] == 7.0).all() and torch.equal(g, g0)
    state, q = opt.state_dict(), p.clone()
    twin = optim.Muon(q, MIXED)
    twin.load_state_dict(state)
    opt.step(g)
    twin.step(g)
    assert torch.equal(q, p) and torch.equal(twin.buf, opt.buf) and twin.steps == opt.steps == 3


def test_muon_step_in_a_graph_and_on_a_stream():
    from pixelwiseregression_amd import optim
    n = sum(math.prod(s) for s in MIXED)
    torch.manual_seed(2)
    p0, g = 0.05 * torch.randn(n, device=DEV), 1e-3 * torch.randn(n, device=DEV)
    a, b = p0.clone(), p0.clone()
    eager, captured = optim.Muon(a, MIXED), optim.Muon(b, MIXED)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        captured.step(g)
    torch.cuda.current_stream().wait_stream(s)
    eager.step(g)
    assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured.step(g)                                      # (a captured step keeps the learning rate and the step number it was captured with)
    for k in range(3):
        g.copy_(1e-3 * torch.randn(n, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        eager.steps = 1
        eager.step(g)
        assert torch.equal(a, b) and torch.equal(eager.buf, captured.buf), k


def test_train_step_with_muon():
    """TrainStep(opt='muon') = its gradients (those of opt='sgd' on the same parameters) put through the step, and the loss it returns is the same."""
    from pixelwiseregression_amd import PixelwiseRegression, optim
    from pixelwiseregression_amd.synthetic import make_batch
    from pixelwiseregression_amd.train import TrainStep
    torch.manual_seed(0)
    m = PixelwiseRegression(4, stage=2, label_size=16, features=32, level=2, norm_method="instance").to(DEV).train()
    batch = {k: v.to(DEV) for k, v in make_batch(2, 4, S=32, seed=2).items()}
    p0 = m.flat_parameters().clone()
    args = (batch["img"], batch["label_img"], batch["mask"], batch["uvd"])
    loss = TrainStep(m, opt="muon", lr=2e-3, weight_decay=0.01)(*args)
    grad, p1 = m.flat_grad().clone(), m.flat_parameters().clone()
    with torch.no_grad():
        m.flat_parameters().copy_(p0)
    ref = TrainStep(m, opt="sgd", lr=0.0)(*args)
    assert torch.equal(loss, ref) and torch.equal(grad, m.flat_grad())
    q = p0.clone()
    optim.Muon(q, [s for (_, s) in m._offsets.values()], lr=2e-3, weight_decay=0.01).step(grad)
    assert torch.equal(q, p1) and not torch.equal(p0, p1)


def test_a_loss_on_the_maps_and_the_step_together():
    """As a program uses them: logits of a linear head, the joints' negative log likelihood with an entropy term, its gradient, the step.  One
    iteration against float64."""
    from pixelwiseregression_amd import ops, optim
    from oracle import likelihood_ref
    r = np.random.default_rng(0)
    B, J, C, V = 6, 4, 40, 256
    feat = r.standard_normal((B * V, C)).astype(np.float32)
    wt = (0.2 * r.standard_normal((J, C))).astype(np.float32)
    temp = np.ones((J, 1), np.float32)
    index = r.integers(0, V, (B, J))
    flat = torch.from_numpy(np.concatenate([wt.ravel(), temp.ravel()])).to(DEV)
    head, w = flat[:J * C].view(J, C).requires_grad_(), flat[J * C:].view(J, 1).requires_grad_()
    z = (torch.from_numpy(feat).to(DEV) @ head.t()).view(B, V, J).permute(0, 2, 1)
    out = ops.log_likelihood(z, torch.from_numpy(index).to(DEV), w)
    (-out.logp.mean() + 0.1 * out.entropy.mean()).backward()
    grad = torch.cat([head.grad.reshape(-1), w.grad.reshape(-1)])
    z64 = (feat.astype(np.float64) @ wt.astype(np.float64).T).reshape(B, V, J).transpose(0, 2, 1)
    n = B * J
    ref = likelihood_ref.rows(z64, index, temp[:, 0], glogp=np.full((B, J), -1.0 / n), gentropy=np.full((B, J), 0.1 / n))
    gh = ref["gz"].transpose(0, 2, 1).reshape(B * V, J).T @ feat.astype(np.float64)
    want = np.concatenate([gh.ravel(), ref["gw"]])
    # logits are sums of 40 products (40 2^-24 |z|, |z| <= 6): 1.5e-5 of a probability; 1536 of them times |feat| <= 4.5 add up to the gradient
    assert np.abs(grad.cpu().double().numpy() - want).max() <= 2e-5 * np.abs(feat).max()
    opt = optim.Muon(flat.detach(), [(J, C), (J, 1)], lr=0.01)
    before = flat.detach().clone()
    opt.step(grad)
    g64 = grad.cpu().double().numpy()
    p, _, _, dirs = muon_ref.step(before.cpu().numpy(), g64, np.zeros_like(g64), np.zeros_like(g64), [(0, J, C), (J * C, 1, J)], lr=0.01, beta1=float(np.float32(0.9)), beta2=float(np.float32(0.999)))
    _, tol = bound(dirs[0], False)
    err = np.abs(flat.detach().cpu().double().numpy() - p)
    assert np.linalg.norm(err[:J * C]) <= 0.01 * 0.2 * math.sqrt(C) * 4 * tol + 4 * 2.0 ** -24 * np.linalg.norm(p)
    assert err[J * C:].max() <= 64 * 2.0 ** -24

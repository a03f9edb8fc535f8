"""GPU: log_likelihood (log probability of a heat map's pixel, entropy, alternatives, gradients) against the float64 oracle.

Tolerances.  With S the largest |w z| of a row, fp32 evaluation rounds s = w z and s - M to 2^-24 of S each and the exponent's argument once
more, and sums at most 64 terms in a row before the reductions: a log probability is off by at most (4 S + 128) 2^-24, a probability by that much of
itself.  A gradient is a sum of such probabilities times (log p + entropy); a bf16 gradient is rounded once more, 2^-8 of itself."""
import math

import numpy as np
import pytest
import torch

from oracle import likelihood_ref

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def inputs(B, J, V, dtype=torch.float32, w=True, mask="none", seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    z = (spread * torch.randn(B, J, V, generator=g)).to(dtype)
    index = torch.randint(0, V, (B, J), generator=g)
    index[torch.rand(B, J, generator=g) < 0.15] = -1
    wv = 0.5 + torch.rand(J, generator=g) if w else None
    m = None
    if mask == "sample":
        m = (torch.rand(B, 1, V, generator=g) < 0.5).float()
        m[0] = 0                                                # one sample without an allowed pixel
    elif mask == "row":
        m = (torch.rand(B, J, V, generator=g) < 0.5).float()
        m[-1, 0] = 0
    return z, index, wv, m


def check(z, index, wv, m, topk=0, grads=True):
    from pixelwiseregression_amd import ops
    B, J, V = z.shape
    zd = z.to(DEV).requires_grad_(grads)
    wd = wv.to(DEV).requires_grad_(grads) if wv is not None else None
    r = ops.log_likelihood(zd, index.to(DEV) if index is not None else None, wd, m.to(DEV) if m is not None else None, topk=topk)
    g = torch.Generator().manual_seed(99)
    gl, ge = torch.randn(B, J, generator=g), torch.randn(B, J, generator=g)
    mm = None if m is None else np.broadcast_to(m.numpy(), (B, J, V))
    ref = likelihood_ref.rows(z.float().numpy(), None if index is None else index.numpy(), None if wv is None else wv.numpy(), mm, topk, gl.numpy(), ge.numpy())
    s = np.abs(z.float().numpy().astype(np.float64) * (1.0 if wv is None else wv.numpy()[:, None]))
    S = np.where(np.isfinite(s) & (True if mm is None else mm != 0), s, 0.0).max(-1)
    tol = (4 * S + 128) * U

    def near(got, want, bound, what):
        got = got.detach().cpu().double().numpy()
        assert got.shape == want.shape, what
        same = np.isnan(got) == np.isnan(want)
        assert same.all(), (what, "NaN", np.argwhere(~same)[:4])
        inf = np.isinf(want)
        assert (got[inf] == want[inf]).all() and not np.isinf(got[~inf]).any(), (what, "inf")
        fin = np.isfinite(want)
        err = np.abs(got - want, where=fin, out=np.zeros_like(want))
        bound = np.broadcast_to(bound, want.shape)
        assert (err[fin] <= bound[fin]).all(), (what, float((err[fin] / bound[fin]).max()), float(err[fin].max()))

    if index is not None:
        near(r.logp, ref["logp"], tol, "logp")
    near(r.entropy, ref["entropy"], (1 + np.nan_to_num(ref["entropy"])) * tol, "entropy")
    if topk:
        assert np.array_equal(r.top_index.cpu().numpy(), ref["top_index"])
        near(r.top_logp, ref["top_logp"], tol[..., None], "top_logp")
    if not grads:
        return r, ref
    outs, ups = ([r.logp, r.entropy], [gl.to(DEV), ge.to(DEV)]) if index is not None else ([r.entropy], [ge.to(DEV)])
    got = torch.autograd.grad(outs, [zd] + ([wd] if wd is not None else []), ups)
    p, lp, H = ref["p"], np.where(ref["p"] > 0, ref["logs"], 0.0), np.nan_to_num(ref["entropy"])[..., None]
    aw = np.ones((J, 1)) if wv is None else np.abs(wv.numpy().astype(np.float64))[:, None]
    size = np.abs(gl.numpy())[..., None] * p + np.abs(ge.numpy())[..., None] * p * (np.abs(lp) + H + 1)
    # (a probability below the smallest normal number, 2^-126 = e^-87.3, is 0 in fp32: its term, p times g + h (log p + entropy), is off by all of itself)
    tiny = 2.0 ** -126 * (np.abs(gl.numpy()) + 100 * np.abs(ge.numpy()))[..., None]
    ds_tol = size * 2 * tol[..., None] + tiny
    gz_tol = ds_tol * aw + np.abs(np.nan_to_num(ref["gz"])) * (4 * U + (2.0 ** -8 if z.dtype == torch.bfloat16 else 0))
    near(got[0], ref["gz"], gz_tol, "gz")
    if wd is not None:
        az = np.where(np.isfinite(s), np.abs(z.float().numpy().astype(np.float64)), 0.0)
        total = ((ds_tol + (np.abs(np.nan_to_num(ref["gz"])) / aw) * 160 * U) * az).sum((0, 2))
        near(got[1], ref["gw"], total + 1e-30, "gw")
    return r, ref


# lengths around every change of form: one wave per row (<= 64, <= 512), one workgroup (<= 4096, 8192, 16384), several; odd ones in each
@pytest.mark.parametrize("V", [1, 2, 3, 63, 64, 65, 511, 512, 513, 1000, 4095, 4096, 4097, 8193, 16383, 16384, 16385, 40001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_lengths(V, dtype):
    check(*inputs(2, 3, V, dtype, w=True, mask="none", seed=V), topk=5)


@pytest.mark.parametrize("V", [4099, 8192, 16500, 20481])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("mask", ["none", "sample"])
def test_many_long_rows(V, dtype, mask):
    """Enough rows for a workgroup to walk each: the maximum in the first part, in the last, rising from part to part; equal maxima in several parts."""
    z, index, w, m = inputs(130, 4, V, dtype, mask=mask, seed=V)
    z[1, 0, 5] = 40.0
    z[1, 1, V - 1] = 40.0
    z[1, 2] = torch.linspace(-30, 30, V).to(dtype)
    z[1, 3, ::4096] = 25.0
    check(z, index, w, m)


@pytest.mark.parametrize("V", [5, 200, 4096, 5000, 20000])
@pytest.mark.parametrize("mask", ["sample", "row"])
def test_masks_and_rows_without_a_pixel(V, mask):
    r, _ = check(*inputs(3, 4, V, w=True, mask=mask, seed=V + 1), topk=7)
    b, j = (0, 0) if mask == "sample" else (2, 0)
    assert r.entropy[b, j] == 0 and (r.top_index[b, j] == -1).all()


@pytest.mark.parametrize("K", [1, 2, 16, 31, 32])
@pytest.mark.parametrize("V", [7, 40, 300, 4096, 9001, 33000])
def test_alternatives(K, V):
    check(*inputs(2, 2, V, w=False, seed=K), topk=K, grads=False)


@pytest.mark.parametrize("K,V", [(17, 2 ** 20), (32, 2 ** 21), (32, 600001)])
def test_alternatives_of_one_long_row(K, V):
    check(*inputs(1, 1, V, w=False, seed=K), topk=K, grads=False)


def test_a_changed_input_is_noticed():
    from pixelwiseregression_amd import ops
    for changed in range(4):
        z, index, w, m = (t.to(DEV) for t in inputs(4, 3, 100, mask="sample", seed=1))
        q, v = z.clone().requires_grad_(), w.clone().requires_grad_()
        r = ops.log_likelihood(q, index, v, m)
        with torch.no_grad():
            (q, v, index, m)[changed].zero_()
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            torch.autograd.grad(r.entropy.sum(), [q, v])


@pytest.mark.parametrize("V", [50, 512, 3000, 16384, 30000])
def test_ties_go_to_the_lowest_index(V):
    # every value equal; two values only; bf16 values of a coarse grid: more candidates than the selection sorts at once
    z = torch.zeros(1, 3, V)
    z[0, 1, ::3] = 1.0
    z[0, 2] = torch.randint(0, 4, (V,), generator=torch.Generator().manual_seed(1)).float()
    for dtype in (torch.float32, torch.bfloat16):
        r, _ = check(z.to(dtype), torch.zeros(1, 3, dtype=torch.long), None, None, topk=32, grads=False)
        n = min(V, 32)
        assert r.top_index[0, 0, :n].tolist() == list(range(n))
        k = min(32, (V + 2) // 3)
        assert r.top_index[0, 1, :k].tolist() == list(range(0, 3 * k, 3))


@pytest.mark.parametrize("V", [33, 1024, 5000, 17000])
def test_extreme_values(V):
    """Lowest finite values, -inf, one pixel with everything, values far apart; NaN and inf where the mask excludes them."""
    lowest = torch.finfo(torch.float32).min
    z, index, w, m = inputs(6, 2, V, w=True, mask="none", seed=5)
    z[0, 0] = lowest; z[0, 0, V // 2] = 0.0           # masked by value
    z[1, 0] = lowest                                     # ... entirely: uniform
    z[2, 0, : V // 2] = -math.inf
    z[2, 1] = -math.inf                                  # no pixel at all
    z[3, 0] = -50.0; z[3, 0, V - 1] = 50.0            # one pixel has it all
    z[4, 0] = torch.linspace(-80, 80, V)
    m = torch.ones(6, 2, V)
    m[5, 0, ::2] = 0
    z[5, 0, ::2] = math.nan
    m[5, 1, 1::2] = 0
    z[5, 1, 1::2] = math.inf
    w = torch.ones(2)
    check(z, index, w, m, topk=4)
    check(z[:5], index[:5], None, None, topk=4)


def test_a_map_that_is_almost_one_pixel_keeps_its_small_numbers():
    """entropy and 1 - p of a map with p = 1 - 1e-6: relative to THEIR size, not to the 1 they are added to"""
    from pixelwiseregression_amd import ops
    for V in (2, 300, 4096, 20000):
        z = torch.full((1, V), -14.0 - math.log(V))
        z[0, V // 2] = 0.0
        zd = z.to(DEV).requires_grad_()
        index = torch.tensor([V // 2], device=DEV)
        r = ops.log_likelihood(zd, index)
        (gz,) = torch.autograd.grad(r.logp.sum(), zd)
        ref = likelihood_ref.rows(z[:, None].numpy(), np.array([[V // 2]]), glogp=np.ones((1, 1)))
        for got, want in ((r.logp.item(), ref["logp"][0, 0]), (r.entropy.item(), ref["entropy"][0, 0]), (gz[0, V // 2].item(), ref["gz"][0, 0, V // 2])):
            assert abs(got - want) <= (4 * 24 + 128) * U * abs(want), (V, got, want)


@pytest.mark.parametrize("V", [40, 2000, 20000])
def test_nan_and_plus_infinity_are_loud(V):
    from pixelwiseregression_amd import ops
    z = torch.randn(3, V)
    z[0, 1] = math.nan
    z[1, 2] = math.inf
    r = ops.log_likelihood(z.to(DEV), torch.zeros(3, dtype=torch.long, device=DEV))
    assert torch.isnan(r.logp).tolist() == [True, True, False] and torch.isnan(r.entropy).tolist() == [True, True, False]
    r = ops.log_likelihood(torch.randn(2, V, device=DEV), torch.tensor([V, 2 ** 40], device=DEV))     # no such pixel
    assert torch.isnan(r.logp).all() and torch.isfinite(r.entropy).all()


@pytest.mark.parametrize("V", [60, 700, 4097, 17001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_strides_and_alignment(V, dtype):
    """A slice of a wider tensor (rows a stride apart, starting at an odd element), a permuted one, an expanded one, shapes [N, V] and [B, J, H, W]."""
    from pixelwiseregression_amd import ops
    g = torch.Generator().manual_seed(3)
    wide = torch.randn(4, V + 9, generator=g).to(dtype).to(DEV)
    index = torch.randint(0, V, (4,), generator=g).to(DEV)
    for z in (wide[:, 1:V + 1], wide[:, 3:V + 3], wide[::2, 2:V + 2].repeat(2, 1), wide[:1, 5:V + 5].expand(4, V), wide[:, 1:V + 1].t().contiguous().t()):
        plain = z.contiguous().clone()
        for a, b in zip(ops.log_likelihood(z, index, topk=3), ops.log_likelihood(plain, index, topk=3)):
            assert torch.equal(a, b)
        za, zb = z.detach().requires_grad_(), plain.requires_grad_()
        ga, gb = (torch.autograd.grad(ops.log_likelihood(q, index).logp.sum(), q)[0] for q in (za, zb))
        assert torch.equal(ga, gb)
    z = torch.randn(2, 3, 5, 7, device=DEV)
    ix = torch.randint(0, 35, (2, 3), device=DEV)
    w = torch.rand(3, 1, device=DEV)
    m = (torch.rand(2, 1, 5, 7, device=DEV) < 0.7).float()
    a, b = ops.log_likelihood(z, ix, w, m, topk=2), ops.log_likelihood(z.flatten(2), ix.int(), w.view(-1), m.flatten(2) != 0, topk=2)
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and a.top_index.shape == (2, 3, 2)
    zs = torch.randn(3, 2, 5, 7, device=DEV).transpose(0, 1)                # [B, J, H, W] with J the outer axis
    assert torch.equal(ops.log_likelihood(zs, ix).logp, ops.log_likelihood(zs.contiguous(), ix).logp)


def test_gradients_against_differences():
    """Central differences of the float64 oracle, on fp32 gradients."""
    from pixelwiseregression_amd import ops
    z, index, w, m = inputs(2, 2, 9, mask="row", seed=11, spread=1.0)
    index[0] = torch.tensor([1, 4])
    m[0] = 1
    zd, wd = z.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    r = ops.log_likelihood(zd, index.to(DEV), wd, m.to(DEV))
    finite = torch.isfinite(r.logp).float()
    gz, gw = torch.autograd.grad([r.logp, r.entropy], [zd, wd], [1.5 * finite, torch.full_like(r.entropy, -0.7)])

    def f(zz, ww):
        o = likelihood_ref.rows(zz, index.numpy(), ww, np.broadcast_to(m.numpy(), z.shape))
        return 1.5 * np.where(np.isfinite(o["logp"]), o["logp"], 0.0).sum() - 0.7 * o["entropy"].sum()

    z64, w64, h = z.double().numpy(), w.double().numpy(), 1e-5
    for at in np.ndindex(*z64.shape):
        up, dn = z64.copy(), z64.copy()
        up[at] += h; dn[at] -= h
        assert abs((f(up, w64) - f(dn, w64)) / (2 * h) - gz[at].item()) < 1e-6      # (third derivative ~1: h^2; fp32 gradient: 1e-7)
    for j in range(2):
        up, dn = w64.copy(), w64.copy()
        up[j] += h; dn[j] -= h
        assert abs((f(z64, up) - f(z64, dn)) / (2 * h) - gw[j].item()) < 5e-6


def test_only_what_is_asked_for():
    from pixelwiseregression_amd import ops
    z = torch.randn(3, 2, 100, device=DEV, requires_grad=True)
    r = ops.log_likelihood(z, None, topk=3)
    assert r.logp is None and not r.top_logp.requires_grad and r.entropy.requires_grad
    (g,) = torch.autograd.grad(r.entropy.sum(), z)
    assert torch.isfinite(g).all() and g.abs().sum() > 0
    w = torch.rand(2, device=DEV, requires_grad=True)
    (gw,) = torch.autograd.grad(ops.log_likelihood(z.detach(), torch.zeros(3, 2, dtype=torch.long, device=DEV), w).logp.sum(), w)
    assert torch.isfinite(gw).all()
    with torch.no_grad():
        assert not ops.log_likelihood(z, None).entropy.requires_grad
    e = ops.log_likelihood(torch.empty(0, 2, 10, device=DEV), torch.empty(0, 2, dtype=torch.long, device=DEV), topk=2)
    assert e.logp.shape == (0, 2) and e.top_index.shape == (0, 2, 2)
    z0 = torch.empty(0, 2, 10, device=DEV, requires_grad=True)
    gz, gw = torch.autograd.grad(ops.log_likelihood(z0, None, w).entropy.sum(), [z0, w])
    assert gz.shape == (0, 2, 10) and (gw == 0).all()


@pytest.mark.parametrize("V", [100, 4096, 20000])
def test_repeats_are_bit_identical_and_streams_and_graphs_agree(V):
    from pixelwiseregression_amd import ops
    z, index, w, m = (t.to(DEV) for t in inputs(8, 3, V, mask="sample", seed=2))

    def once():
        q, v = z.detach().requires_grad_(), w.detach().requires_grad_()
        r = ops.log_likelihood(q, index, v, m, topk=4)
        g = torch.autograd.grad([r.logp[1:].sum() + r.entropy.sum()], [q, v])
        return [t.detach() for t in r] + list(g)

    a, b = once(), once()
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        c = once()
    s.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a, c))
    del b, c
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        d = once()
    for k in range(3):
        z.copy_(torch.randn(z.shape, generator=torch.Generator().manual_seed(k)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(d, once())), k


def test_offsets_beyond_32_bits():
    """2.2e9 logits: the last rows are the first ones again"""
    from pixelwiseregression_amd import ops
    V, n = 65537, 33000
    z = torch.empty(n, V, device=DEV, dtype=torch.bfloat16)
    part = torch.randn(4, V, device=DEV).to(torch.bfloat16)
    z[:4] = part
    z[4:-4] = 0
    z[-4:] = part
    assert z.numel() > 2 ** 31
    index = torch.arange(n, device=DEV) % 4 * 1000
    index[-4:] = index[:4]
    q = z.requires_grad_()
    r = ops.log_likelihood(q, index)
    (g,) = torch.autograd.grad(r.logp.sum(), q)
    assert torch.equal(r.logp[:4], r.logp[-4:]) and torch.equal(r.entropy[:4], r.entropy[-4:])
    assert torch.equal(g[:4], g[-4:])
    assert abs(r.entropy[5].item() - math.log(V)) < (128 * U) * 12


def test_train_step_likelihood_terms_match_autograd_through_the_maps():
    """TrainStep(lambda_nll, lambda_entropy) hands the engine gradients of its LOGITS; the same terms written on the maps it returns (p, log p) and
    differentiated by autograd give the same loss and parameter gradients.  The backward pass is linear in those gradients; they agree to
    (4 S + 128) 2^-24 ~ 1e-5, and the mean subtractions of the norms' backward may cancel two digits of it."""
    from pixelwiseregression_amd import PixelwiseRegression, ops
    from pixelwiseregression_amd.synthetic import make_batch
    from pixelwiseregression_amd.train import TrainStep
    torch.manual_seed(0)
    B, J, P = 3, 4, 16
    m = PixelwiseRegression(J, stage=2, label_size=P, features=32, level=2, norm_method="instance").to(DEV).train()
    b = {k: v.to(DEV) for k, v in make_batch(B, J, S=2 * P, seed=2).items()}
    b["uvd"][0, 0, 0] = 3.0                                   # a joint outside the map
    args = (b["img"], b["label_img"], b["mask"], b["uvd"])
    p0 = m.flat_parameters().clone()
    plain = TrainStep(m, opt="sgd", lr=0.0)(*args).item()
    base = m.flat_grad().clone()
    assert torch.equal(p0, m.flat_parameters())
    loss = TrainStep(m, opt="sgd", lr=0.0, lambda_nll=0.3, lambda_entropy=0.05)(*args)
    grad = m.flat_grad().clone()
    TrainStep(m, opt="sgd", lr=0.0)(*args)
    assert torch.equal(base, m.flat_grad())                   # nothing of the terms stays behind for the next step
    for p in m.parameters():
        p.grad = None
    index = ops.heatmap_pixels(b["uvd"], P)
    assert index[0, 0] == -1 and (index.view(-1)[1:] >= 0).all()
    want = 0.0
    for heat, _, uvd in m(*args[:3]):
        want = want + torch.mean(torch.sum((uvd - b["uvd"]) ** 2, dim=2))
        logs = heat.flatten(2).log()
        logp = logs.gather(2, index.clamp(min=0)[..., None])[..., 0] * (index >= 0)
        want = want - 0.3 * logp.mean() + 0.05 * -(heat.flatten(2) * logs).sum(-1).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * abs(want.item()) and abs(loss.item() - plain) > 0.1
    auto = m.flat_grad()
    assert (grad - auto).norm() <= 1e-3 * auto.norm() and (grad - base).norm() > 0.01 * base.norm()
    ws = [o for n, (o, _) in m._offsets.items() if n.endswith(".w")]
    for o in ws:                                              # the softmax temperature's gradient, in both parts
        assert (grad[o:o + J] - auto[o:o + J]).norm() <= 1e-3 * auto[o:o + J].norm()

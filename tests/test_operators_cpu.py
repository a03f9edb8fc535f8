"""CPU: what log_likelihood, orthogonalize, Muon and their C entry points refuse, the optimizer's plan, the oracles against plain definitions, and
the pixel of a joint."""
import ctypes
import math

import numpy as np
import pytest
import torch

from oracle import likelihood_ref, muon_ref
from pixelwiseregression_amd import _lib, ops, optim
from pixelwiseregression_amd.optim import _Param

EINVAL, EUNSUPPORTED, ENOSPACE = -1, -2, -3
SOME = 4096        # an address that is never read: every call below is refused on the host


def test_there_is_no_cpu_path():
    z = torch.randn(2, 3, 8)
    with pytest.raises(_lib.PwrError):
        ops.log_likelihood(z, torch.zeros(2, 3, dtype=torch.long))
    with pytest.raises(_lib.PwrError):
        ops.orthogonalize(torch.randn(4, 5))
    with pytest.raises(_lib.PwrError):
        optim.Muon(torch.zeros(20), [(4, 5)])
    with pytest.raises(_lib.PwrError):
        ops.likelihood_gradients(z, None, None, None, None)


def likelihood(**kw):
    a = dict(z=SOME, ldz=8, w=None, J=1, mask=None, mask_rows=1, index=None, logp=None, entropy=None, stats=None, top_logp=None, top_index=None, rows=4, V=8,
             K=0, dtype=0, ws=None, wsb=0)
    a.update(kw)
    return _lib.lib().pwr_likelihood_fwd(*a.values(), None)


def test_likelihood_entry_points_refuse_on_the_host():
    l = _lib.lib()
    assert likelihood(z=None) == EINVAL and likelihood(V=0) == EINVAL and likelihood(rows=-1) == EINVAL and likelihood(K=-1) == EINVAL
    assert likelihood(J=0) == EINVAL and likelihood(mask_rows=0) == EINVAL and likelihood(ldz=-1) == EINVAL and likelihood(dtype=2) == EINVAL
    assert likelihood(K=3) == EINVAL                                                       # no place for the alternatives
    assert likelihood(K=33, top_logp=SOME, top_index=SOME) == EUNSUPPORTED
    assert likelihood(K=32, top_logp=SOME, top_index=SOME, V=16384 * 129) == EUNSUPPORTED  # 129 pieces x 32
    assert likelihood(rows=2 ** 30, V=16384 * 4) == EUNSUPPORTED                           # 2^32 workgroups
    assert likelihood(V=100000) == ENOSPACE and likelihood(V=100000, ws=SOME, wsb=15) == ENOSPACE
    assert likelihood(rows=0, V=0) == 0
    assert l.pwr_likelihood_workspace_bytes(4, 4096, 32) == 0 and l.pwr_likelihood_workspace_bytes(0, 10, 0) == 0
    n = -(-100000 // 4096)                                                                 # a lone row: pieces of 4096
    assert l.pwr_likelihood_workspace_bytes(1, 100000, 5) == n * (16 + 40)
    bwd = lambda **kw: l.pwr_likelihood_bwd(*{**dict(z=SOME, ldz=8, w=None, J=1, mask=None, mr=1, index=None, stats=SOME, entropy=SOME, gl=None, ge=None,  # noqa: E731
                                                    gz=SOME, gw=None, rows=4, V=8, dtype=0, ws=None, wsb=0), **kw}.values(), None)
    assert bwd(z=None) == EINVAL and bwd(stats=None) == EINVAL and bwd(gz=None) == EINVAL and bwd(dtype=7) == EINVAL and bwd(V=0) == EINVAL
    assert bwd(gw=SOME) == EINVAL                                                          # a gradient of a w that is not there
    assert bwd(gw=SOME, w=SOME, J=3) == EINVAL                                             # rows are no multiple of the joints
    assert bwd(gw=SOME, w=SOME, J=2) == ENOSPACE and bwd(rows=0) == 0


def test_orthogonalize_entry_points_refuse_on_the_host():
    l = _lib.lib()
    orth = lambda **kw: l.pwr_orthogonalize(*{**dict(x=SOME, bs=12, rs=4, out=SOME, rows=3, cols=4, batch=1, dtype=0, steps=5, a=1.5, b=-.5, c=0.0, eps=1e-7,  # noqa: E731
                                                     ws=SOME, wsb=10 ** 9), **kw}.values(), None)
    assert orth(x=None) == EINVAL and orth(out=None) == EINVAL and orth(batch=-1) == EINVAL and orth(rows=0) == EINVAL and orth(dtype=5) == EINVAL
    assert orth(steps=0) == EINVAL and orth(steps=65) == EINVAL and orth(eps=-1.0) == EINVAL and orth(eps=math.nan) == EINVAL and orth(rs=-1) == EINVAL
    assert orth(rows=2 ** 21) == EUNSUPPORTED and orth(rows=2 ** 16, cols=2 ** 15) == EUNSUPPORTED
    assert orth(ws=None) == ENOSPACE and orth(wsb=100) == ENOSPACE and orth(batch=0) == 0
    assert l.pwr_orthogonalize_workspace_bytes(3, 4, 0) == 0 and l.pwr_orthogonalize_workspace_bytes(2 ** 21, 4, 1) == 0
    # X twice and A, B as pairs of 16 bits, in tiles of 64; small matrices live in one workgroup
    assert l.pwr_orthogonalize_workspace_bytes(70, 130, 1) >= (2 * 128 * 192 + 2 * 128 * 128) * 4 and 0 < l.pwr_orthogonalize_workspace_bytes(3, 65, 1) < 4096


def plan(params):
    l = _lib.lib()
    arr = (_Param * len(params))(*params)
    n = l.pwr_muon_plan_bytes(arr, len(params))
    if n == 0:
        buf = ctypes.create_string_buffer(64)
        assert l.pwr_muon_plan(arr, len(params), buf) == EINVAL
        return None
    buf = ctypes.create_string_buffer(n)
    assert l.pwr_muon_plan(arr, len(params), buf) == 0
    return buf


def test_muon_plan_and_step_refuse_on_the_host():
    l = _lib.lib()
    assert plan([(0, 4, 5), (19, 2, 2)]) is None                       # overlap
    assert plan([(4, 4, 5), (0, 1, 5)]) is None                        # ... in any order
    assert plan([(-1, 4, 5)]) is None and plan([(0, 0, 5)]) is None and plan([(0, 2 ** 21, 2)]) is None
    assert l.pwr_muon_plan_bytes(None, 1) == 0 and l.pwr_muon_workspace_bytes(None) == 0
    b = plan([(0, 4, 5), (30, 1, 9000), (20, 2, 2)])                   # gaps are fine
    ws = l.pwr_muon_workspace_bytes(b)
    assert ws > 0 and l.pwr_muon_workspace_bytes(ctypes.create_string_buffer(512)) == 0
    step = lambda **kw: l.pwr_muon_step(*{**dict(ph=b, pd=SOME, p=SOME, g=SOME, buf=SOME, v=SOME, lr=1e-3, mom=.95, nes=1, wd=0., rms=.2, ns=5, a=1.5, b=-.5,  # noqa: E731
                                                c=0., eps=1e-7, b1=.9, b2=.999, ae=1e-8, t=1, gs=1., ws=SOME, wsb=ws), **kw}.values(), None)
    for k in ("ph", "pd", "p", "g", "buf", "v"):
        assert step(**{k: None}) == EINVAL, k
    assert step(ph=ctypes.create_string_buffer(512)) == EINVAL and step(ns=0) == EINVAL and step(ns=65) == EINVAL and step(t=0) == EINVAL and step(eps=-1.) == EINVAL
    assert step(ws=None) == ENOSPACE and step(wsb=ws - 1) == ENOSPACE


def test_plan_of_a_network_covers_every_parameter_once():
    from pixelwiseregression_amd import PixelwiseRegression
    m = PixelwiseRegression(5, stage=2, label_size=16, features=32, level=2, norm_method="batch")
    params = [(o, s[0] if len(s) > 1 else 1, int(torch.Size(s).numel()) // (s[0] if len(s) > 1 else 1)) for o, s in m._offsets.values()]
    assert plan(params) is not None
    assert sum(r * c for _, r, c in params) == m.flat_parameters().numel()


def test_the_oracles_say_what_the_definitions_say():
    r = np.random.default_rng(0)
    x = r.standard_normal((20, 31))
    u, s, vt = np.linalg.svd(x, full_matrices=False)
    s = s / (np.linalg.norm(x) + 1e-7)
    a, b, c = muon_ref.COEFFICIENTS
    for _ in range(5):
        s = a * s + b * s ** 3 + c * s ** 5
    assert np.abs(muon_ref.newton_schulz(x) - (u * s) @ vt).max() < 1e-12
    assert np.abs(muon_ref.newton_schulz(x.T) - ((u * s) @ vt).T).max() < 1e-12
    z = torch.from_numpy(r.standard_normal((2, 3, 11))).requires_grad_()
    w = torch.from_numpy(r.random(3) + 0.5).requires_grad_()
    mask = torch.from_numpy((r.random((2, 3, 11)) < 0.7).astype(np.float64))
    mask[0, 0] = 1
    index = torch.tensor([[1, -1, 10], [0, 5, 3]])
    mask[0, 2, 10] = mask[1, 0, 0] = mask[1, 1, 5] = mask[1, 2, 3] = 1
    gl, ge = torch.from_numpy(r.standard_normal((2, 3))), torch.from_numpy(r.standard_normal((2, 3)))
    d = torch.distributions.Categorical(logits=(z * w[:, None]).masked_fill(mask == 0, -1e30))
    lp = torch.where(index >= 0, d.log_prob(index.clamp(min=0)), torch.zeros(()).double())
    gz, gw = torch.autograd.grad((lp * gl + d.entropy() * ge).sum(), [z, w])
    o = likelihood_ref.rows(z.detach().numpy(), index.numpy(), w.detach().numpy(), mask.numpy(), 0, gl.numpy(), ge.numpy())
    for got, want in ((o["logp"], lp), (o["entropy"], d.entropy()), (o["gz"], gz), (o["gw"], gw)):
        assert np.abs(got - want.detach().numpy()).max() < 1e-12


def test_the_pixel_of_a_joint_is_the_inverse_of_the_decoder_grid():
    for P in (2, 16, 64, 128):
        ax = (np.arange(P) - P // 2) / (P - 1)
        u, v = np.meshgrid(ax, ax)
        uvd = torch.from_numpy(np.stack([u, v, 0 * u], -1)).float().view(1, P * P, 3)
        assert torch.equal(ops.heatmap_pixels(uvd, P)[0], torch.arange(P * P))
    out = torch.tensor([[[0.6, 0.0, 0.0], [0.0, -0.6, 0.0], [math.nan, 0.0, 0.0], [math.inf, 0.0, 0.0], [0.0, 0.0, 9.0]]])
    assert ops.heatmap_pixels(out, 64)[0].tolist() == [-1, -1, -1, -1, 32 * 64 + 32]


def test_train_step_refuses():
    from pixelwiseregression_amd import PixelwiseRegression
    from pixelwiseregression_amd.train import TrainStep
    m = PixelwiseRegression(3, stage=1, label_size=16, features=32, level=1, heatmap_method="sum", norm_method="instance")
    with pytest.raises(ValueError, match="opt must"):
        TrainStep(m, opt="lion")
    with pytest.raises(ValueError, match="softmax"):
        TrainStep(m, lambda_nll=0.1)


def test_launches_beyond_what_the_card_takes_are_refused():
    l = _lib.lib()
    assert likelihood(rows=2 ** 26, V=10) == EUNSUPPORTED                                  # 2^32 threads: a wave per row
    assert likelihood(rows=2 ** 24, V=600) == EUNSUPPORTED and likelihood(rows=2 ** 22, V=3000) == EUNSUPPORTED
    assert likelihood(rows=2 ** 24, V=20000, ws=SOME, wsb=2 ** 62) == EUNSUPPORTED
    assert likelihood(rows=2 ** 21, V=20000, K=1, top_logp=SOME, top_index=SOME, ws=SOME, wsb=2 ** 62) == EUNSUPPORTED
    bwd = lambda rows, V: l.pwr_likelihood_bwd(SOME, 8, None, 1, None, 1, None, SOME, SOME, None, None, SOME, None, rows, V, 0, None, 0, None)  # noqa: E731
    assert bwd(2 ** 26, 10) == EUNSUPPORTED and bwd(2 ** 24, 600) == EUNSUPPORTED and bwd(2 ** 20, 16 * 4096) == EUNSUPPORTED
    orth = lambda rows, cols, batch: l.pwr_orthogonalize(SOME, 0, cols, SOME, rows, cols, batch, 0, 5, 1.5, -.5, 0., 1e-7, SOME, 2 ** 62, None)  # noqa: E731
    assert orth(3, 4, 2 ** 22) == EUNSUPPORTED and orth(128, 128, 2 ** 21) == EUNSUPPORTED and orth(65, 70, 2 ** 40) == EUNSUPPORTED


def test_a_lone_long_row_keeps_its_alternatives():
    """A row is split no further than its alternatives can be joined."""
    l = _lib.lib()
    for V in (2 ** 19, 2 ** 20, 2 ** 21):
        for K in (1, 16, 17, 32):
            need = l.pwr_likelihood_workspace_bytes(1, V, K)
            pieces = need // (16 + 8 * K)
            assert need % (16 + 8 * K) == 0 and pieces * K <= 4096 and V // 16384 <= pieces <= V // 4096
            assert likelihood(rows=1, V=V, K=K, top_logp=SOME, top_index=SOME, ws=SOME, wsb=need - 1) == ENOSPACE      # (as far as the last check)

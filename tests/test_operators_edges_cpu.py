"""CPU: calls at the edge of what log_likelihood, orthogonalize and Muon take."""
import ctypes
import math

import numpy as np
import pytest
import torch

from pixelwiseregression_amd import _lib, ops, optim
from pixelwiseregression_amd.optim import _Param

EUNSUPPORTED = -2
SOME = 4096        # an address that is never read: every call below is refused on the host


@pytest.fixture
def anywhere(monkeypatch):
    """The calls' own checks on tensors without memory."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 100), (1, 2 ** 31), (2, 1, 2 ** 32 + 1), (1, 1, 2 ** 16, 2 ** 16), (1, 2 ** 32 + 1, 1), (0, 2 ** 31, 4)])
def test_rows_beyond_an_int_are_refused(anywhere, shape):
    with pytest.raises(ValueError, match=r"2\^31"):
        ops.log_likelihood(empty(*shape), None)
    with pytest.raises(ValueError, match=r"2\^31"):
        ops.likelihood_gradients(empty(*shape), None, None, None, None)
    with pytest.raises(ValueError, match=r"2\^31"):
        ops.log_likelihood(torch.empty(1, dtype=torch.bfloat16).expand(shape), None)          # (no copy of it is tried first)


@pytest.mark.parametrize("shape", [(2 ** 32 + 2, 1), (1, 2 ** 32 + 3), (3, 4, 2 ** 32 + 3), (2 ** 20 + 1, 1), (2, 2 ** 16, 2 ** 15)])
def test_matrices_beyond_the_limit_are_refused(anywhere, shape):
    with pytest.raises(ValueError, match="larger than"):
        ops.orthogonalize(empty(*shape))


def forward(rows, V, ldz, K=0, dtype=1):
    top = SOME if K else None
    return _lib.lib().pwr_likelihood_fwd(SOME, ldz, None, 1, None, 1, None, None, SOME, None, top, top, rows, V, K, dtype, SOME, 2 ** 62, None)


def backward(rows, V, ldz, dtype=1):
    return _lib.lib().pwr_likelihood_bwd(SOME, ldz, None, 1, None, 1, None, SOME, SOME, None, None, SOME, None, rows, V, dtype, None, 0, None)


def test_rows_whose_last_piece_ends_beyond_an_int_are_refused(anywhere):
    """600 rows that are one row in memory (4 GiB): the walk over them counts in ints."""
    l = _lib.lib()
    for V in (2 ** 31 - 1, 2 ** 31 - 2 ** 14 + 1):
        for K in (0, 1):
            assert forward(600, V, 0, K) == EUNSUPPORTED and forward(1, V, 0, K) == EUNSUPPORTED
        assert backward(600, V, 0) == EUNSUPPORTED and backward(1, V, 0) == EUNSUPPORTED
        assert l.pwr_likelihood_workspace_bytes(600, V, 0) == 0 and l.pwr_likelihood_bwd_workspace_bytes(600, V) == 0
        with pytest.raises(ValueError, match=r"2\^31"):
            ops.log_likelihood(empty(600, V), None)
    assert l.pwr_likelihood_workspace_bytes(1, 2 ** 31 - 2 ** 14, 0) == 16 * (2 ** 17 - 1)


def test_numbers_of_rows_whose_launch_leaves_64_bits_are_refused():
    for rows in (2 ** 32, 2 ** 58, 2 ** 62):
        for V in (4, 600, 40000):
            assert forward(rows, V, 0) == EUNSUPPORTED and forward(rows, V, 0, 1) == EUNSUPPORTED and backward(rows, V, 0) == EUNSUPPORTED


def largest(steps, a, b, c, n=20001):
    """The largest entry that could be stored: max of s, s^2, |b s^2 + c s^4| and |a + b s^2 + c s^4| over the iterates of [0, 1] that go into a step."""
    s, m = np.linspace(0, 1, n), 0.0
    with np.errstate(over="ignore", invalid="ignore"):
        for _ in range(steps):
            u = s * s
            q = b * u + c * u * u
            m = max(m, u.max(), np.abs(q).max(), np.abs(a + q).max())
            if not m < 1e3:
                return math.inf
            s = np.linspace(0, np.abs(s * (a + q)).max(), n)
    return m


def test_coefficients_that_leave_the_pairs_are_refused(anywhere):
    l = _lib.lib()
    r = np.random.default_rng(0)
    taken = refused = 0
    for _ in range(400):
        steps = int(r.integers(1, 9))
        co = [float(np.float32(v)) for v in (r.uniform(-4, 4), r.uniform(-8, 8) * r.choice([0, 1]), r.uniform(-4, 4) * r.choice([0, 1]))]
        m, got = largest(steps, *co), l.pwr_orthogonalize_range(steps, *co)
        if m > 16.0:
            assert got == EUNSUPPORTED, (steps, co, m)
            refused += 1
        elif m < 15.9 / 1.002 ** (4 * steps) / 1.1:               # (away from the border, where an unstable map makes much of the room for roundings)
            taken += got == 0
            assert got == 0 or largest(steps, *[1.01 * v for v in co]) > 15.9, (steps, co, m)
    assert taken > 50 and refused > 50
    for steps in (1, 2, 5, 64):
        for co in (ops.NS_COEFFICIENTS, (1.5, -0.5, 0.0), (15 / 8, -10 / 8, 3 / 8), (2.0, -1.5, 0.5)):
            assert l.pwr_orthogonalize_range(steps, *co) == 0
    # linear maps and single steps: both sides of each limit
    for steps, co, ok in ((3, (1.98, 0.0, 0.0), 1), (3, (2.0, 0.0, 0.0), 0), (1, (1.0, -15.8, 0.0), 1), (1, (1.0, -16.0, 0.0), 0), (1, (15.8, -15.8, 0.0), 1),
                          (1, (16.0, -15.0, 0.0), 0), (2, (2.5, -0.06, 0.0), 1), (4, (2.5, -0.06, 0.0), 0), (5, (3.0, -0.065, 0.0), 0),
                          (1, (math.nan, 0.0, 0.0), 0), (1, (0.0, math.inf, 0.0), 0),
                          # the largest s between 0 and 1, whatever c is next to b, or b next to a c
                          (2, (6.9, -6.9, 0.0), 0), (2, (6.9, -6.9, 1e-17), 0), (2, (6.9, -6.9, -1e-30), 0), (2, (9.0, 0.0, -9.0), 0), (2, (9.0, 1e-20, -9.0), 0),
                          (2, (3.0, 1e-20, -3.0), 0), (2, (2.0, 1e-20, -2.0), 1), (64, (0.0, 0.0, 0.0), 1)):
        assert (l.pwr_orthogonalize_range(steps, *co) == 0) == bool(ok), (steps, co)
        if not ok:
            assert l.pwr_orthogonalize(SOME, 12, 4, SOME, 3, 4, 1, 0, steps, *co, 1e-7, SOME, 2 ** 40, None) == EUNSUPPORTED
            with pytest.raises(ValueError, match="coefficients"):
                ops.orthogonalize(empty(3, 4), steps=steps, coefficients=co)
    assert l.pwr_orthogonalize_range(0, 1.5, -0.5, 0.0) == -1 and l.pwr_orthogonalize_range(65, 1.5, -0.5, 0.0) == -1


def test_the_optimizer_refuses_such_coefficients(monkeypatch):
    l = _lib.lib()
    monkeypatch.setattr(optim.Muon, "_check", lambda self, t, what: t)
    with pytest.raises(ValueError, match="coefficients"):
        optim.Muon(torch.zeros(20), [(4, 5)], coefficients=(3.0, -0.065, 0.0))
    arr = (_Param * 1)((0, 4, 5))
    n = l.pwr_muon_plan_bytes(arr, 1)
    plan = ctypes.create_string_buffer(n)
    assert l.pwr_muon_plan(arr, 1, plan) == 0
    step = lambda ns, *co: l.pwr_muon_step(plan, SOME, SOME, SOME, SOME, SOME, 1e-3, .95, 1, 0., .2, ns, *co, 1e-7, .9, .999, 1e-8, 1, 1., SOME, 2 ** 40, None)  # noqa: E731
    assert step(5, 3.0, -0.065, 0.0) == EUNSUPPORTED and step(1, 1.0, -16.0, 0.0) == EUNSUPPORTED


def test_forward_mode_tangents_are_refused(anywhere):
    """(no requires_grad on a dual tensor: its derivative would be dropped without a word)"""
    import torch.autograd.forward_ad as fw
    with fw.dual_level():
        z, w = (fw.make_dual(t, torch.ones_like(t)) for t in (torch.zeros(2, 3, 8), torch.ones(3)))
        assert not z.requires_grad and not w.requires_grad
        for call in (lambda: ops.log_likelihood(z, None), lambda: ops.log_likelihood(torch.zeros(2, 3, 8), None, w),
                     lambda: ops.likelihood_gradients(z, None, None, None, None), lambda: ops.likelihood_gradients(torch.zeros(2, 3, 8), None, w, None, None),
                     lambda: ops.orthogonalize(z)):
            with pytest.raises(NotImplementedError):
                call()
            with torch.no_grad(), pytest.raises(NotImplementedError):
                call()
        assert not ops._tangents(torch.zeros(3), None)
    assert not ops._tangents(z, w)


def test_a_mask_is_of_the_maps_own_shape():
    z = torch.zeros(2, 3, 4, 6)
    with pytest.raises(ValueError, match="mask"):
        ops._Rows(z, None, None, torch.ones(2, 1, 6, 4))
    with pytest.raises(ValueError, match="mask"):
        ops._Rows(z, None, None, torch.ones(2, 3, 2, 12))
    for m in (torch.ones(2, 1, 4, 6), torch.ones(2, 3, 4, 6), torch.ones(2, 1, 24), torch.ones(2, 3, 24)):
        r = ops._Rows(z, None, None, m)
        assert r.mask.shape == m.flatten(2).shape and r.mask_rows == (3 if m.shape[1] == 1 else 1)


def test_a_mask_of_any_type_keeps_what_is_not_zero():
    values = [0.0, 1.0, 1e-300, -0.0, 5e-324, math.nan, 1e300]
    want = [False, True, True, False, True, True, True]
    r = ops._Rows(torch.zeros(1, 7), None, None, torch.tensor([values], dtype=torch.float64))
    assert r.mask.dtype is torch.float32 and (r.mask[0] != 0).tolist() == want
    for dtype in (torch.bool, torch.uint8, torch.int64, torch.float16, torch.bfloat16, torch.float32):
        m = torch.tensor([[0, 1, 1, 0, 1, 1, 1]]).to(dtype)
        assert (ops._Rows(torch.zeros(1, 7), None, None, m).mask[0] != 0).tolist() == want


def test_the_barriers_of_one_workgroup_are_every_waves():
    """In the kernel of small matrices the waves of a pair take different branches: none of its barriers stands inside one, or inside a function that is
    called from one."""
    import os
    import re
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    text = re.sub(r"//[^\n]*", "", open(os.path.join(root, "pixelwiseregression_amd", "csrc", "orth.hip")).read())
    text = text[text.index("void orth_small_kernel("):]
    stack, head, barriers = [], "", 0
    for token in re.split(r"([{};])", text):
        if token == "{":
            stack.append(head)
        elif token == "}":
            stack.pop()
            if not stack:
                break
        elif token != ";":
            if "__syncthreads" in token:
                barriers += 1
                assert "if (" not in token and not any("[&]" in h or "if (" in h for h in stack[1:]), stack[1:]
        if token in "{};":
            head = ""
        else:
            head = token
    assert barriers >= 7


def test_a_gradient_of_more_joints_than_a_launch_has_workgroups_is_refused():
    bwd = lambda rows, J: _lib.lib().pwr_likelihood_bwd(SOME, 1, SOME, J, None, 1, None, SOME, SOME, None, None, SOME, SOME, rows, 1, 0, SOME, 2 ** 62, None)  # noqa: E731
    assert bwd(2 ** 25, 2 ** 25) == EUNSUPPORTED and bwd(0, 2 ** 24) == EUNSUPPORTED


def test_rows_that_are_walked_need_no_workspace():
    """512 long rows and more without alternatives go to a workgroup each; fewer are split, and joined from a workspace."""
    l = _lib.lib()
    assert l.pwr_likelihood_workspace_bytes(512, 100000, 0) == 0 and l.pwr_likelihood_workspace_bytes(4096, 50001, 0) == 0
    assert l.pwr_likelihood_workspace_bytes(511, 100000, 0) == 511 * 7 * 16 and l.pwr_likelihood_workspace_bytes(512, 100000, 1) == 512 * 7 * (16 + 8)
    assert l.pwr_likelihood_fwd(SOME, 0, None, 1, None, 1, None, None, SOME, None, None, None, 511, 100000, 0, 0, None, 0, None) == -3
    # (refused by the number of its threads, a workgroup of 256 a row: the last check)
    assert l.pwr_likelihood_fwd(SOME, 0, None, 1, None, 1, None, None, SOME, None, None, None, 2 ** 24, 100000, 0, 0, None, 0, None) == EUNSUPPORTED

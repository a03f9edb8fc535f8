"""CPU: calls at the edge of what log_likelihood, orthogonalize and Muon take."""
import pytest
import torch

from pixelwiseregression_amd import _lib, ops

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

"""CPU: calls at the edge of what log_likelihood, orthogonalize and Muon take."""
import pytest
import torch

from pixelwiseregression_amd import ops


@pytest.fixture
def anywhere(monkeypatch):
    """The calls' own checks on tensors without memory."""
    monkeypatch.setattr(ops, "_require_cuda", lambda *ts: None)


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(*shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("shape", [(1, 2 ** 32 + 100), (1, 2 ** 31), (2, 1, 2 ** 32 + 1), (1, 1, 2 ** 16, 2 ** 16), (1, 2 ** 32 + 1, 1), (0, 2 ** 31, 4)])
def test_rows_beyond_an_int_are_refused(anywhere, shape):
    with pytest.raises(ValueError, match="2\\^31"):
        ops.log_likelihood(empty(*shape), None)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.likelihood_gradients(empty(*shape), None, None, None, None)
    with pytest.raises(ValueError, match="2\\^31"):
        ops.log_likelihood(torch.empty(1, dtype=torch.bfloat16).expand(shape), None)          # (no copy of it is tried first)


@pytest.mark.parametrize("shape", [(2 ** 32 + 2, 1), (1, 2 ** 32 + 3), (3, 4, 2 ** 32 + 3), (2 ** 20 + 1, 1), (2, 2 ** 16, 2 ** 15)])
def test_matrices_beyond_the_limit_are_refused(anywhere, shape):
    with pytest.raises(ValueError, match="larger than"):
        ops.orthogonalize(empty(*shape))

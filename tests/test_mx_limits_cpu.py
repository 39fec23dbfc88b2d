"""Refusals of the microscaled calls' settings and streams that need no GPU."""
import pytest

torch = pytest.importorskip("torch")


def test_wait_limit_refusals(b200):
    limit = b200.lib().b200_mx_wait_limit
    assert limit(0, 3) == b200.ERR_INVALID_ARG
    assert limit(0, -1) == b200.ERR_INVALID_ARG
    assert limit(5_000_000, 0) == 0
    assert limit(0, 0) == 0


class _Stream:
    """Stands in for a torch.cuda.Stream, which needs a GPU."""

    def __init__(self, device):
        self.device, self.cuda_stream = torch.device(device), 0x1000


def test_stream_of_another_device_is_refused(b200):
    """It was dropped without a word: the call ran on the current stream of the tensors' device."""
    with pytest.raises(ValueError, match="cuda:1"):
        b200._On(torch.device("cuda:0"), _Stream("cuda:1"))

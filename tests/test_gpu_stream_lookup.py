"""The stream that kernels are launched on is torch's current one of the current device."""
import pytest
import torch

from rexl3_b200.ops import lib


@pytest.mark.gpu
def test_the_current_stream_wherever_it_is_set():
    same = lambda: lib.stream_ptr() == torch.cuda.current_stream().cuda_stream  # noqa: E731
    assert same()
    side, other = torch.cuda.Stream(), torch.cuda.Stream(priority=-1)
    with torch.cuda.stream(side):
        assert lib.stream_ptr() == side.cuda_stream and same()
        with torch.cuda.stream(other):
            assert lib.stream_ptr() == other.cuda_stream and same()
        assert lib.stream_ptr() == side.cuda_stream
    torch.cuda.set_stream(other)
    assert lib.stream_ptr() == other.cuda_stream
    torch.cuda.set_stream(torch.cuda.default_stream())
    assert same()
    for device in range(torch.cuda.device_count()):
        with torch.cuda.device(device):
            assert same()
            with torch.cuda.stream(torch.cuda.Stream()):
                assert same()

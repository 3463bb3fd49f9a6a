"""Page ids far outside the cache read as zeros, also where id * KV heads * 64 passes 32 bits."""
import pytest

from test_gpu_attn_shared import Window


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("page", [2 ** 24, 2 ** 25, 2 ** 26 + 1, 2 ** 31 - 1, -2 ** 25, -2 ** 26 + 1, -2 ** 31])
def test_far_pages_read_as_zeros(page, fp8):
    w = Window([(-1, 130, 1)], 0, 10, 2, 128, fp8=fp8, seed=14)
    w.table[:] = page
    assert bool((w.run() == 0).all())

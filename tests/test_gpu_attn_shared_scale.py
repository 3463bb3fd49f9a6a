"""Scales of the scores at the ends of float32's range: the kernel takes scale * log2(e) in float32, where 0 or infinity would make NaN of a masked score."""
import pytest
import torch

from rexl3_b200.ops import kernels as K
from test_gpu_attn_shared import Window


def call(w, scale):
    out, st = torch.full_like(w.q, float("nan")), K.new_status()
    K.attn_shared(*w.maps, w.q, w.table, w.row_seq, w.ctx, w.common, K.attn_shared_scratch(w.q.shape[0], w.n_q, w.n_kv, w.hd), w.n_q, w.n_kv, w.hd, scale, out, st)
    K.check_status(st)
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-50, 1e-39, 3e38, 1e39, 1e300, 5e-324])
def test_scales_that_float32_cannot_hold_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        call(Window([(0, 100, 1), (0, 120, 1)], 1, 10, 2, 128, seed=1), scale)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-37, 1e-30])
def test_the_smallest_scales_give_the_mean_of_the_values(scale):
    """Every probability is exp of next to nothing: 1 / n.  Only the outputs are rounded (bf16, 2^-8) and the products with V summed in fp32."""
    w = Window([(0, 100, 1), (0, 120, 1)], 1, 10, 2, 128, seed=1)
    out = call(w, scale).double()
    for r in range(2):
        n = int(w.ctx[r])
        v = w.v[w.table[int(w.row_seq[r]), :2].long()].double().transpose(1, 2).reshape(-1, 2, 128)[:n]
        want, mean = (x.mean(0).repeat_interleave(5, 0).reshape(-1) for x in (v, v.abs()))
        assert bool(((out[r] - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5 * mean).all())

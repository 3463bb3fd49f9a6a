"""Attention over shared pages where each CTA's piece of the work is a few pages only, over and over: what one warp hands to another too early, or a last page that goes
unseen, shows itself in some of many calls.  (The tolerance is that of test_gpu_attn_shared.)"""
import pytest
import torch

from test_gpu_attn_shared import Window


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("seqs,shared,heads", [
    ([(-1, 9 * 64 + 1, 1)], 0, (10, 2, 128)),                            # hardly a page for each
    ([(-1, 290 * 64 - 5, 1)], 0, (10, 2, 128)),                          # two pages, in one unit or two
    ([(-1, 430 * 64 - 5, 2)], 0, (10, 2, 128)),                          # three
    ([(0, 4200 + 11 * i, 1) for i in range(12)], 60, (16, 4, 64)),
    ([(i // 8, 1300 + 11 * i, 5) for i in range(16)], 18, (32, 4, 128)),
])
def test_short_pieces(seqs, shared, heads, fp8):
    w = Window(seqs, shared, *heads, fp8=fp8, seed=len(seqs))
    first = w.check() and w.run()
    for _ in range(100):
        assert torch.equal(w.run(), first)

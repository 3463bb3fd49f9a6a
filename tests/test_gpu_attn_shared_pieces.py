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


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [True, False])
@pytest.mark.parametrize("seqs,shared,heads", [
    ([(-1, 64 * (3 + i) + 1 + 7 * i, 13 + i) for i in range(7)], 0, (10, 2, 128)),      # 65 to 95 pairs a block
    ([(-1, 64 * 9 + 40, 17 + i) for i in range(8)], 0, (16, 4, 64)),                    # 68 to 96
    ([(0, 150 + i % 20, 1) for i in range(64)], 2, (40, 8, 128)),                       # 125, 125 and 70
    ([(-1, 70 + 5 * i, 14) for i in range(40)], 0, (40, 8, 128)),
])
def test_a_warp_without_pairs_clears_its_share_of_the_last_page(seqs, shared, heads, fp8):
    """Blocks of 65 to 96 pairs, the last page of each in parts unseen and full of infinities."""
    w = Window(seqs, shared, *heads, fp8=fp8, seed=20 + len(seqs))
    first = w.check() and w.run()
    for _ in range(100):
        assert torch.equal(w.run(), first)

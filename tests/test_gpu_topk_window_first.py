"""The first row of a row's window, where it names no row before it: the row has no drafts, and its biases stay."""
import pytest
import torch

from test_gpu_topk_adjusted import rules, same, t

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("nb", [7, 1024])                                # a chunk's biases in the list, and more than it holds
@pytest.mark.parametrize("ahead", [0, 1, 2, 300])
@pytest.mark.parametrize("V", [2048, 9000])
def test_a_first_row_at_or_behind_the_row(V, ahead, nb):
    rows = 6
    kw = rules(rows, V, 2, V + nb, nb=nb)
    kw["bias"][0].copy_(torch.arange(nb, dtype=torch.int32, device="cuda") % 1500)
    kw["bias"][1][:, -200:] += 50.0                                      # the last places weigh most
    kw["window"] = (torch.arange(rows, dtype=torch.int32, device="cuda") + ahead, kw["window"][1])
    kw["row_slot"] = t([0, 1, 0, 1, 0, 1])
    same(torch.randn(rows, V, device="cuda"), 28, kw.pop("row_slot"), **kw)


@pytest.mark.parametrize("nb", [7, 1024])
@pytest.mark.parametrize("first", [2147483647, 2147483646, -1, -2147483648])
def test_a_first_row_far_outside(first, nb):
    rows, V = 6, 2048
    kw = rules(rows, V, 2, nb, nb=nb)
    kw["window"] = (t([first] * rows), kw["window"][1])
    same(torch.randn(rows, V, device="cuda"), 28, kw.pop("row_slot"), **kw)

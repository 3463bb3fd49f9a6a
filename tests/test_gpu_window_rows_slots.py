"""Page ids whose slots are past int32: as a page that is missing."""
import pytest
import torch

from rexl3_b200.ops import kernels as K


def t(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.gpu
@pytest.mark.parametrize("page", [2 ** 25, 2 ** 25 + 3, 2 ** 26, 2 ** 31 - 1])
@pytest.mark.parametrize("alloc", [False, True])
def test_a_page_past_int32_gives_rows_that_are_not_cached(page, alloc):
    last = 2 ** 25 - 1
    table, rows, starts, st, at = t([[4, -1 if alloc else page, last]]), torch.zeros(5, 66, dtype=torch.int32, device="cuda"), t([0, 0]), K.new_status(), t([0])
    kw = dict(free=t([page, last]), free_at=at, free_next=at) if alloc else {}
    K.window_rows(t([0]), t([63]), t([66]), table, rows, starts, st, **kw)
    assert st[0].item() == K.ST_BAD_ARG
    assert rows[1].tolist() == [4 * 64 + 63] + [-1] * 64 + [last * 64]
    assert table.tolist() == [[4, page, last]]

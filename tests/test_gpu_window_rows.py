"""Row maps and block tables made on the device, against the requests walked one by one on the host; refusals."""
import pytest
import torch

from rexl3_b200.ops import kernels as K


def walk(seq, have, new, table, free, at):
    """-> rows [5][total], starts, table, free position after; the table is changed only where free is given."""
    table = [list(r) for r in table]
    rows, starts, prev = [[] for _ in range(5)], [0], None
    before = [list(r) for r in table]
    for s, h, k in zip(seq, have, new):
        if free is not None:
            for b in range(-(-h // 64), -(-(h + k) // 64)):
                table[s][b] = free[at]
                at += 1
        common = 0
        if prev is not None and k:
            most = -(-min(h, prev[1]) // 64)
            while common < most and before[s][common] == before[prev[0]][common]:
                common += 1
        for p in range(h, h + k):
            for column, v in zip(rows, (p, table[s][p // 64] * 64 + p % 64, s, p + 1, common)):
                column.append(v)
        starts.append(starts[-1] + k)
        if k:
            prev = (s, h)
    return rows, starts, table, at


def t(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


CASES = {
    "one token": dict(have=[0], new=[1]),
    "one request that feeds nothing": dict(have=[5], new=[0]),
    "page borders": dict(have=[0, 63, 64, 65, 127, 128, 1], new=[64, 1, 1, 63, 2, 0, 128]),
    "requests that feed nothing between others": dict(have=[100, 100, 100, 100, 100], new=[0, 3, 0, 0, 2]),
    "one long prompt": dict(have=[7], new=[5000]),
    "64 decode rows": dict(have=[500 + 13 * i for i in range(64)], new=[1] * 64),
    "1024 requests": dict(have=[(37 * i) % 300 for i in range(1024)], new=[(i * 7) % 5 for i in range(1024)]),
    "513 requests, ragged": dict(have=[(91 * i) % 700 for i in range(513)], new=[(i * i) % 97 for i in range(513)]),
}


@pytest.mark.gpu
@pytest.mark.parametrize("shared", [0, 3])
@pytest.mark.parametrize("alloc", [True, False])
@pytest.mark.parametrize("name", list(CASES))
def test_rows_as_the_host_walks_them(name, alloc, shared):
    have, new = CASES[name]["have"], CASES[name]["new"]
    n = len(have)
    g = torch.Generator().manual_seed(n + shared)
    seq = torch.randperm(n + 5, generator=g)[:n].tolist()
    width = max(-(-(h + k) // 64) for h, k in zip(have, new)) + 2
    table = torch.randint(5000, 10000, (n + 5, width), generator=g)
    table[:, :shared] = torch.arange(shared) + 7
    need = sum(-(-(h + k) // 64) - -(-h // 64) for h, k in zip(have, new))
    free = torch.randperm(need + 9, generator=g).tolist() if alloc else None
    want_rows, want_starts, want_table, at = walk(seq, have, new, table.tolist(), free, 4)
    cap = want_starts[-1] + 6
    rows, starts, dt, st = torch.full((5, cap), -77, dtype=torch.int32, device="cuda"), t([-5] * (n + 1)), t(table.tolist()), K.new_status()
    at_dev = t([4])
    kw = dict(free=t(free), free_at=at_dev, free_next=at_dev) if alloc else {}
    K.window_rows(t(seq), t(have), t(new), dt, rows, starts, st, **kw)
    K.check_status(st)
    assert starts.tolist() == want_starts
    assert rows[:, :want_starts[-1]].tolist() == want_rows
    assert (rows[:, want_starts[-1]:] == -77).all()                  # behind the last row: as it was
    assert dt.tolist() == want_table
    if alloc:
        assert at_dev.item() == at


BAD = {
    "length below 0": dict(have=[3, -1]), "fed below 0": dict(new=[1, -1]), "beyond the table": dict(have=[3, 512]), "far beyond the table": dict(have=[3, 2147483647], new=[1, 2147483647]),
    "table row outside": dict(seq=[0, 9]), "table row below 0": dict(seq=[-1, 1]), "table row twice": dict(seq=[1, 1]), "more rows than there is room for": dict(new=[1, 12]),
    "more pages than are free": dict(have=[64, 64], free=[5], at=0), "free list used up": dict(have=[64, 64], at=3), "free position below 0": dict(have=[64, 64], at=-1),
    "no free pages at all": dict(have=[64, 64], free=[], at=0),
}


@pytest.mark.gpu
@pytest.mark.parametrize("name", list(BAD))
def test_impossible_requests_change_nothing(name):
    c = {**dict(seq=[0, 1], have=[3, 4], new=[1, 1], free=[5, 6, 7, 8], at=0), **BAD[name]}
    rows, starts, table, st = torch.full((5, 10), -77, dtype=torch.int32, device="cuda"), t([-5] * 3), torch.arange(24, dtype=torch.int32, device="cuda").view(3, 8), K.new_status()
    want, at = table.clone(), t([c["at"]])
    K.window_rows(t(c["seq"]), t(c["have"]), t(c["new"]), table, rows, starts, st, free=t(c["free"]), free_at=at, free_next=at)
    assert st[0].item() == K.ST_BAD_ARG
    assert torch.equal(table, want) and (rows == -77).all() and (starts == -5).all() and at.item() == c["at"]


@pytest.mark.gpu
def test_a_missing_page_gives_a_row_that_is_not_cached():
    table, rows, starts, st = t([[4, -1, 6]]), torch.zeros(5, 66, dtype=torch.int32, device="cuda"), t([0, 0]), K.new_status()
    K.window_rows(t([0]), t([63]), t([66]), table, rows, starts, st)
    assert st[0].item() == K.ST_BAD_ARG
    assert rows[1].tolist() == [4 * 64 + 63] + [-1] * 64 + [6 * 64]


@pytest.mark.gpu
def test_in_a_graph_step_after_step():
    """A captured call with free_next = free_at takes further pages at every replay."""
    n = 3
    have, one, table = t([63, 64, 10]), t([1] * n), t([[1, 0, 0, 0, 0], [2, 0, 0, 0, 0], [3, 0, 0, 0, 0]])
    free, at, rows, starts, st = t(list(range(10, 30))), t([0]), torch.zeros(5, n, dtype=torch.int32, device="cuda"), t([0] * (n + 1)), K.new_status()
    want_table, want_at, host = table.tolist(), 0, [63, 64, 10]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        K.window_rows(t_seq := torch.arange(n, dtype=torch.int32, device="cuda"), have, one, table, rows, starts, st, free=free, free_at=at, free_next=at)
        have += one
    assert t_seq is not None
    for _ in range(130):
        want, _, want_table, want_at = walk(list(range(n)), host, [1] * n, want_table, list(range(10, 30)), want_at)
        graph.replay()
        assert rows.tolist() == want
        host = [h + 1 for h in host]
    K.check_status(st)
    assert table.tolist() == want_table and at.item() == want_at


def test_refusals():
    x = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        K.window_rows(x, x, x, torch.zeros(2, 2, dtype=torch.int32), torch.zeros(5, 2, dtype=torch.int32), torch.zeros(3, dtype=torch.int32), torch.zeros(8, dtype=torch.int32))


@pytest.mark.gpu
def test_refusals_of_arguments():
    def call(**kw):
        a = {**dict(seq=t([0, 1]), have=t([0, 0]), new=t([1, 1]), block_table=t([[0], [1]]), rows=torch.zeros(5, 2, dtype=torch.int32, device="cuda"), starts=t([0, 0, 0]), status=K.new_status()), **kw}
        K.window_rows(**a)
    for kw in (dict(seq=t([0, 1]).long()), dict(have=t([0])), dict(new=t([0, 0, 0])[::2][:1]), dict(block_table=t([0])), dict(rows=torch.zeros(4, 2, dtype=torch.int32, device="cuda")),
               dict(starts=t([0, 0])), dict(status=t([0])), dict(free=t([3])), dict(free=t([3]), free_at=t([0])), dict(free=t([3]), free_at=t([0]), free_next=t([0, 0])),
               dict(block_table=t([[0, 1], [1, 2]]).t()), dict(seq=t([]), have=t([]), new=t([]), starts=t([0])), dict(have=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(ValueError):
            call(**kw)
    call()

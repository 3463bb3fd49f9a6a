"""Attention over pages that sequences share, against softmax attention in float64 over every row's own keys; refusals.

Tolerance.  A probability is rounded once to the operand type (bf16 2^-8 of its value at most, fp16 2^-11) and an output once to bf16 (2^-8); the sums are
fp32.  So |error| <= (2^-8 + 2^-8 (1 + 2^-8)) * sum_j p_j |v_j| / sum_j p_j plus what fp32 scores and ex2.approx (2^-21 or so, relative) give: scores of
magnitude |s| <= 64 log2 units are off by at most 64 * 2^-22 or so.  Every element is checked against 2^-7 * 1.02 * (the mean of |v| under p) + 1e-5.
The rotated output is a sum of 128 unrounded outputs times their signs / sqrt(128): at most 2^-8 * 1.02 times the same sum of the means of |v|, plus its fp16 rounding 2^-11.
"""
import math

import pytest
import torch

from rexl3_b200.ops import kernels as K


def t(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Window:
    """Sequences as (group, length, rows); group -1: shares nothing.  Groups share `shared` pages; page ids in no order, poison in every key that nobody holds."""

    def __init__(self, seqs, shared, n_q, n_kv, hd, fp8=False, seed=0, poison=True, spread=1.0, width=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        cpu = torch.Generator().manual_seed(seed)
        self.n_q, self.n_kv, self.hd, self.fp8 = n_q, n_kv, hd, fp8
        n, groups = len(seqs), {s[0] for s in seqs if s[0] >= 0}
        need = len(groups) * shared + sum(max(0, -(-s[1] // 64) - (shared if s[0] >= 0 else 0)) for s in seqs)
        ids = torch.randperm(need + 4, generator=cpu).tolist()
        self.width = width or max([shared] + [-(-s[1] // 64) for s in seqs]) + 3
        table = torch.randint(0, need + 4, (n + 2, self.width), generator=cpu).int()
        common = {c: [ids.pop() for _ in range(shared)] for c in groups}
        order = torch.randperm(n + 2, generator=cpu)[:n].tolist()
        row_seq, ctx, com, held = [], [], [], torch.zeros(need + 4, 64, dtype=torch.bool)
        for i, (c, length, rows) in enumerate(seqs):
            mine = (common[c] if c >= 0 else []) + [ids.pop() for _ in range(max(0, -(-length // 64) - (shared if c >= 0 else 0)))]
            table[order[i], :len(mine)] = torch.tensor(mine, dtype=torch.int32)
            for p in range(length):
                held[mine[p // 64], p % 64] = True
            row_seq += [order[i]] * rows
            ctx += [max(0, length - rows + 1 + j) for j in range(rows)]
            com += [shared if i and c >= 0 and seqs[i - 1][0] == c else 0] * rows
        self.k, self.v = (spread * torch.randn(need + 4, n_kv, 64, hd, device="cuda", generator=g) for _ in range(2))
        self.v += 0.5
        self.scale_kv = None
        free = ~held.cuda()[:, None, :, None].expand_as(self.k)
        if fp8:
            self.scale_kv = 0.02 + 0.01 * torch.rand(2, n_kv, device="cuda", generator=g)
            self.k, self.v = ((x / self.scale_kv[i][None, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for i, x in enumerate((self.k, self.v)))
            if poison:
                self.k[free], self.v[free] = 0x7F, 0xFF                  # NaN
        else:
            self.k, self.v = self.k.bfloat16(), self.v.bfloat16()
            if poison:
                self.k[free], self.v[free] = float("nan"), float("inf")
        self.table, self.row_seq, self.ctx, self.common = table.cuda(), t(row_seq), t(ctx), t(com)
        self.q = torch.randn(len(ctx), n_q * hd, device="cuda", generator=g).bfloat16()
        self.maps = K.KvTensorMap(self.k), K.KvTensorMap(self.v)

    def run(self, **kw):
        rows, st = self.q.shape[0], K.new_status()
        out = torch.full((rows, self.n_q * self.hd), float("nan"), dtype=torch.bfloat16, device="cuda")
        scratch = kw.pop("scratch", None)
        if scratch is None:
            scratch = torch.full_like(K.attn_shared_scratch(rows, self.n_q, self.n_kv, self.hd), float("nan"))
        K.attn_shared(*self.maps, self.q, self.table, self.row_seq, self.ctx, kw.pop("common", self.common), scratch, self.n_q, self.n_kv, self.hd,
                      1 / math.sqrt(self.hd), kw.pop("out", out), st, kv_scale=self.scale_kv, **kw)
        K.check_status(st)
        return out

    def exact(self):
        """-> (attention, the mean of |v| under the probabilities), float64 [rows, n_q * hd]"""
        G, out, mean = self.n_q // self.n_kv, [], []
        for r in range(self.q.shape[0]):
            n, width = int(self.ctx[r]), self.n_q * self.hd
            if n == 0:
                out.append(torch.zeros(width, device="cuda", dtype=torch.float64)), mean.append(out[-1])
                continue
            pages = self.table[int(self.row_seq[r]), :-(-n // 64)].long()
            k, v = ((x[pages].double() if not self.fp8 else x[pages].view(torch.float8_e4m3fn).double() * self.scale_kv[i].double()[None, :, None, None])
                    .transpose(1, 2).reshape(-1, self.n_kv, self.hd)[:n] for i, x in enumerate((self.k, self.v)))
            s = torch.einsum("gqd,ngd->gqn", self.q[r].double().view(self.n_kv, G, self.hd), k) / math.sqrt(self.hd)
            p = torch.exp(s - s.amax(-1, keepdim=True))
            p /= p.sum(-1, keepdim=True)
            out.append(torch.einsum("gqn,ngd->gqd", p, v).reshape(-1)), mean.append(torch.einsum("gqn,ngd->gqd", p, v.abs()).reshape(-1))
        return torch.stack(out), torch.stack(mean)

    def check(self, **kw):
        want, mean = self.exact()
        got = self.run(**kw).double()
        off = (got - want).abs() - (1.02 * 2.0 ** -7 * mean + 1e-5)
        assert not bool(got.isnan().any()) and float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than the bound at {divmod(int(off.argmax()), off.shape[1])}"
        return want, mean


HEADS = [(40, 8, 128), (4, 2, 64), (16, 16, 64), (5, 1, 128), (32, 2, 128), (128, 1, 64), (2, 2, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("heads", HEADS)
def test_one_group(heads, fp8):
    Window([(0, 200 + 17 * i, 1) for i in range(7)], 3, *heads, fp8=fp8, seed=1).check()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("shared", [0, 1, 5])
@pytest.mark.parametrize("lengths", [(1,), (0,), (63, 64, 65), (320, 320, 321), (0, 1, 500), (385, 0, 2, 384), (1000, 20, 64, 640)])
def test_lengths(lengths, shared, fp8):
    """Lengths of zero and one, at page borders, and sequences shorter than what their group shares."""
    Window([(0, n, 1) for n in lengths], shared, 10, 2, 128, fp8=fp8, seed=sum(lengths) + shared).check()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("seqs,shared", [
    ([(0, 300 + 5 * i, 1 + i % 6) for i in range(40)], 4),                              # verify windows of 1 to 6 rows
    ([(0, 130, 64), (0, 150, 3)], 2),                                                   # more rows of one sequence than a block holds
    ([(i // 5, 260 + i, 2) for i in range(15)], 4),                                     # three groups side by side
    ([(-1, 100, 1), (0, 400, 1), (0, 401, 1), (-1, 700, 2), (0, 500, 1)], 6),           # strangers between them
    ([(0, 70, 1)] * 130, 1),
])
@pytest.mark.parametrize("heads", [(10, 2, 128), (8, 4, 64)])
def test_windows(seqs, shared, heads, fp8):
    Window(seqs, shared, *heads, fp8=fp8, seed=len(seqs)).check()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_long_prefix_and_many_rows(fp8):
    Window([(0, 8192 + 11 * i, 1) for i in range(64)], 128, 40, 8, 128, fp8=fp8, seed=3).check()


@pytest.mark.gpu
def test_as_many_rows_as_there_may_be():
    Window([(i // 40, 100 + i % 50, 1 + i % 3) for i in range(512)], 1, 4, 2, 64, seed=4).check()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_one_long_row(fp8):
    """One row over a long cache: its pages are split over all CTAs, whose parts are joined."""
    Window([(-1, 50001, 1)], 0, 10, 2, 128, fp8=fp8, seed=5).check()


@pytest.mark.gpu
def test_large_scores():
    """Running maxima that move often, probabilities that are nearly one-hot."""
    Window([(0, 300 + i, 1) for i in range(9)], 4, 10, 2, 128, seed=6, spread=6.0).check()


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_whatever_common_says(fp8):
    """Fewer pages in common than there are, or none: the same attention; and sequences of one group that stand apart."""
    w = Window([(0, 400 + i, 1) for i in range(12)], 6, 10, 2, 128, fp8=fp8, seed=7)
    w.check(common=torch.zeros_like(w.common))
    w.check(common=(w.common - t([i % 4 for i in range(12)])).clamp_min(0))
    w.check(common=-w.common)


@pytest.mark.gpu
def test_links_of_every_kind():
    """A chain of sequences that share ever fewer pages, a stranger with one page in common between two groups: grouped or not, never wrong."""
    w = Window([(0, 700 + i, 1) for i in range(20)], 10, 10, 2, 128, seed=8)
    for links in ([0] + [10, 9, 8, 7, 6, 5, 4, 3, 2, 1] + [10] * 9, [0] + [10] * 9 + [1] + [10] * 9, [0] + [1, 10] * 9 + [1], [10] * 20):
        w.check(common=t(links))


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
def test_plan_given_and_rotated_output(fp8):
    w = Window([(0, 300 + 9 * i, 1) for i in range(6)], 4, 10, 2, 128, fp8=fp8, seed=9)
    want, mean = w.check()
    plan, st, rows = K.attn_shared_plan_buffer(), K.new_status(), w.q.shape[0]
    K.attn_shared_plan(w.table, w.row_seq, w.ctx, w.common, w.n_q, w.n_kv, plan, st)
    assert torch.equal(w.run(plan=plan), w.run())
    suh, xr = torch.randn(10 * 128, device="cuda").half(), torch.empty(rows, 10 * 128, dtype=torch.float16, device="cuda")
    both = w.run(suh=suh, xr=xr)
    assert torch.equal(both, w.run())
    alone = torch.empty_like(xr)
    w.run(out=None, suh=suh, xr=alone)
    assert torch.equal(alone, xr)
    had = torch.ones(1, 1, dtype=torch.float64, device="cuda")
    for _ in range(7):
        had = torch.cat([torch.cat([had, had], 1), torch.cat([had, -had], 1)], 0)
    ref = ((want * suh.double()).view(rows, 10, 128) @ had / math.sqrt(128)).view(rows, -1)
    room = ((mean * suh.double().abs()).view(rows, 10, 128).sum(-1, keepdim=True) / math.sqrt(128)).expand(rows, 10, 128).reshape(rows, -1)
    assert bool(((xr.double() - ref).abs() <= 1.02 * 2.0 ** -8 * room + 2.0 ** -11 * ref.abs() + 1e-4).all())


@pytest.mark.gpu
def test_again_and_again_the_same_bits():
    w = Window([(0, 500 + 31 * i, 1) for i in range(16)], 7, 40, 8, 128, seed=10)
    first = w.run()
    for _ in range(5):
        assert torch.equal(w.run(), first)


@pytest.mark.gpu
@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("seqs,shared,heads", [
    ([(0, 8200 + 9 * i, 1) for i in range(64)], 128, (40, 8, 128)),
    ([(0, 600 + 67 * i, 1) for i in range(48)], 2, (40, 8, 128)),
    ([(i // 8, 4100 + 11 * i, 5) for i in range(16)], 62, (32, 4, 128)),
    ([(i // 8, 4100 + 11 * i, 5) for i in range(16)], 62, (16, 4, 64)),
])
def test_a_full_device_gives_the_same_bits(seqs, shared, heads, fp8):
    """What one warp hands to another too early shows itself in some of many calls."""
    w = Window(seqs, shared, *heads, fp8=fp8, seed=17)
    first = w.check() and w.run()
    for _ in range(60):
        assert torch.equal(w.run(), first)


@pytest.mark.gpu
def test_a_plan_of_another_window_sets_the_status_and_gives_zeros():
    w = Window([(0, 500 + 31 * i, 2) for i in range(6)], 7, 10, 2, 128, seed=18)
    other = Window([(0, 500 + 31 * i, 1) for i in range(5)], 7, 10, 2, 128, seed=18)
    plans = [K.attn_shared_plan_buffer()]                     # none at all, of fewer rows, of other heads, of a wider table
    for a in ((other.table, other.row_seq, other.ctx, other.common, 10, 2), (w.table, w.row_seq, w.ctx, w.common, 20, 2),
              (torch.cat([w.table, w.table], 1).contiguous(), w.row_seq, w.ctx, w.common, 10, 2)):
        plans.append(K.attn_shared_plan_buffer())
        K.attn_shared_plan(*a, plans[-1], K.new_status())
    for plan in plans:
        out, st = torch.ones_like(w.q), K.new_status()
        K.attn_shared(*w.maps, w.q, w.table, w.row_seq, w.ctx, w.common, K.attn_shared_scratch(12, 10, 2, 128), 10, 2, 128, 0.1, out, st, plan=plan)
        assert int(out.abs().sum()) == 0
        with pytest.raises(RuntimeError):
            K.check_status(st)
    w.check()


@pytest.mark.gpu
def test_two_graphs_with_one_workspace_and_another_stream():
    """Two captured windows over one scratch, replayed in turn; the lengths change between replays."""
    a, b = Window([(0, 300 + i, 1) for i in range(8)], 4, 10, 2, 128, seed=11, width=40), Window([(-1, 900, 3), (0, 500, 1), (0, 600, 1)], 2, 10, 2, 128, seed=12, width=40)
    scratch = K.attn_shared_scratch(8, 10, 2, 128)
    graphs, outs = [], []
    side = torch.cuda.Stream()
    for w in (a, b):
        out, st = torch.empty(w.q.shape[0], 1280, dtype=torch.bfloat16, device="cuda"), K.new_status()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            K.attn_shared(*w.maps, w.q, w.table, w.row_seq, w.ctx, w.common, scratch, 10, 2, 128, 1 / math.sqrt(128), out, st)
        graphs.append(g), outs.append((out, st))
    for step in range(3):
        for w, g, (out, st) in zip((a, b), graphs, outs):
            with torch.cuda.stream(side):
                g.replay()
            side.synchronize()
            K.check_status(st)
            want, mean = w.exact()
            assert bool(((out.double() - want).abs() <= 1.02 * 2.0 ** -7 * mean + 1e-5).all())
            w.ctx.sub_(37)
            torch.cuda.synchronize()


@pytest.mark.gpu
def test_bad_rows_set_the_status_and_give_zero():
    w = Window([(0, 300 + i, 1) for i in range(4)], 4, 10, 2, 128, seed=13)
    (want, mean), scratch = w.exact(), K.attn_shared_scratch(4, 10, 2, 128)
    for row in range(4):
        for change in (dict(row_seq=-1), dict(row_seq=99), dict(ctx=-5), dict(ctx=w.width * 64 + 1), dict(ctx=2147483647)):
            seq, ctx, st, out = w.row_seq.clone(), w.ctx.clone(), K.new_status(), torch.empty_like(w.q)
            seq[row], ctx[row] = change.get("row_seq", seq[row]), change.get("ctx", ctx[row])
            K.attn_shared(*w.maps, w.q, w.table, seq, ctx, w.common, scratch, 10, 2, 128, 1 / math.sqrt(128), out, st)
            assert st[0].item() == K.ST_BAD_ARG
            assert bool((out[row] == 0).all())
            others = [r for r in range(4) if r != row]
            assert bool(((out[others].double() - want[others]).abs() <= 1.02 * 2.0 ** -7 * mean[others] + 1e-5).all())


@pytest.mark.gpu
def test_pages_outside_the_cache_read_as_zeros():
    w = Window([(-1, 130, 1)], 0, 10, 2, 128, seed=14)
    w.table[:] = 10 ** 5
    assert bool((w.run() == 0).all())
    w.table[:] = -1
    assert bool((w.run() == 0).all())


@pytest.mark.gpu
def test_rows_then_attention_then_candidates():
    """One decode step as a server makes it: rows and pages from the lengths, keys written at the slots, attention over the shared prompt, candidates under rules."""
    n_q, n_kv, hd, n, prompt = 10, 2, 128, 6, 320
    g = torch.Generator(device="cuda").manual_seed(15)
    table = torch.full((n, 12), -1, dtype=torch.int32, device="cuda")
    table[:, :5] = torch.arange(5, dtype=torch.int32, device="cuda")
    k, v = (torch.randn(40, n_kv, 64, hd, device="cuda", generator=g).bfloat16() for _ in range(2))
    maps, have, one = (K.KvTensorMap(k), K.KvTensorMap(v)), t([prompt] * n), t([1] * n)
    free, at, st = t(list(range(5, 40))), t([0]), K.new_status()
    rows, starts = torch.zeros(5, n, dtype=torch.int32, device="cuda"), torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    head = torch.randn(n_q * hd, 500, device="cuda", generator=g)
    counts, pen = torch.zeros(n, 500, dtype=torch.int16, device="cuda"), torch.tensor([[1.2, 0.5, 0.5]] * n, device="cuda")
    ids, vals, out = torch.empty(n, 8, dtype=torch.int32, device="cuda"), torch.empty(n, 8, device="cuda"), torch.empty(n, n_q * hd, dtype=torch.bfloat16, device="cuda")
    keys = [[torch.cat([x[:5, h].reshape(-1, hd) for x in ()] or [c[:5].transpose(1, 2).reshape(-1, n_kv, hd)]) for h in range(1)][0] for c in (k, v)]
    hist = [[c.clone() for c in keys] for _ in range(n)]
    for step in range(70):
        K.window_rows(t(list(range(n))), have, one, table, rows, starts, st, free=free, free_at=at, free_next=at)
        fresh = [torch.randn(n, n_kv, hd, device="cuda", generator=g).bfloat16() for _ in range(2)]
        slot = rows[1].long()
        for cache, x, which in zip((k, v), fresh, (0, 1)):
            cache[slot // 64, :, slot % 64] = x
            for i in range(n):
                hist[i][which] = torch.cat([hist[i][which], x[i:i + 1]])
        q = torch.randn(n, n_q * hd, device="cuda", generator=g).bfloat16()
        K.attn_shared(*maps, q, table, rows[2], rows[3], rows[4], K.attn_shared_scratch(n, n_q, n_kv, hd), n_q, n_kv, hd, 1 / math.sqrt(hd), out, st)
        logits = out.float() @ head
        K.topk_adjusted(logits, 8, K.topk_scratch(n, 500, 8), ids, vals, t(list(range(n))), counts=counts, penalties=pen)
        K.token_counts_add(counts, t(list(range(n))), ids[:, 0].contiguous(), st)
        have += 1
        if step % 23 == 0 or step == 69:
            K.check_status(st)
            for i in range(n):
                kk, vv = (c.double() for c in hist[i])
                p = torch.softmax(torch.einsum("gqd,ngd->gqn", q[i].double().view(n_kv, -1, hd), kk) / math.sqrt(hd), -1)
                want, mean = (torch.einsum("gqn,ngd->gqd", p, x).reshape(-1) for x in (vv, vv.abs()))
                assert bool(((out[i].double() - want).abs() <= 1.02 * 2.0 ** -7 * mean + 1e-5).all())
    assert int((counts & 32767).sum()) == 70 * n and rows[4].tolist() == [0] + [5] * (n - 1)


def test_refusals_without_a_device():
    x = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA tensor"):
        K.attn_shared_plan(torch.zeros(2, 2, dtype=torch.int32), x, x, x, 4, 2, x, x)
    for rows, n_q, n_kv in ((0, 4, 2), (4, 5, 2), (4, 129, 1), (4, 0, 0)):
        with pytest.raises(ValueError):
            K.attn_shared_scratch(rows, n_q, n_kv, 128, device="cpu")


@pytest.mark.gpu
def test_refusals():
    w = Window([(0, 100, 1), (0, 120, 1)], 1, 10, 2, 128, seed=16)
    ok = dict(tk=w.maps[0], tv=w.maps[1], q=w.q, block_table=w.table, row_seq=w.row_seq, ctx_len=w.ctx, common=w.common, scratch=K.attn_shared_scratch(2, 10, 2, 128), n_q=10, n_kv=2, hd=128,
              scale=0.1, out=torch.empty_like(w.q), status=K.new_status())
    f8, i8 = (K.KvTensorMap(torch.zeros(4, 2, 64, 128, dtype=d, device="cuda")) for d in (torch.uint8, torch.int8))
    half = K.KvTensorMap(torch.zeros(4, 2, 64, 64, dtype=torch.uint8, device="cuda"))
    scales, suh, xr = torch.ones(2, 2, device="cuda"), torch.ones(1280, dtype=torch.float16, device="cuda"), torch.empty(2, 1280, dtype=torch.float16, device="cuda")
    for kw in (dict(q=w.q.float()), dict(q=w.q[:1]), dict(q=w.q[:, ::2]), dict(q=w.q.cpu()), dict(block_table=w.table.long()), dict(block_table=w.table.t()), dict(row_seq=w.row_seq[:1]),
               dict(ctx_len=w.ctx.long()), dict(common=None), dict(n_q=11), dict(n_kv=3), dict(hd=96), dict(hd=64), dict(scratch=torch.empty(100, device="cuda")), dict(out=None),
               dict(out=torch.empty(2, 1280, device="cuda")), dict(status=t([0])), dict(tk=f8, tv=f8), dict(tk=i8, tv=i8), dict(kv_scale=scales), dict(tk=half, tv=half, kv_scale=scales),
               dict(tk=f8, tv=f8, kv_scale=scales[:1]), dict(suh=suh), dict(xr=xr), dict(plan=t([0])), dict(block_table=w.table[:, :0]),
               dict(scratch=torch.empty(ok["scratch"].numel() + 1, device="cuda")[1:]), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))):
        with pytest.raises(ValueError):
            K.attn_shared(**{**ok, **kw})
    big = t([1]).expand(1025).contiguous()
    with pytest.raises(ValueError):
        K.attn_shared_plan(w.table, big, big, big, 10, 2, K.attn_shared_plan_buffer(), K.new_status())
    n = K.attn_shared_plan_buffer().numel()
    with pytest.raises(ValueError):
        K.attn_shared_plan(w.table, w.row_seq, w.ctx, w.common, 10, 2, torch.zeros(n + 1, dtype=torch.int32, device="cuda")[1:], K.new_status())
    K.attn_shared(**ok)
    K.check_status(ok["status"])

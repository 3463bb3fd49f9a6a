"""Sampling rules fused with the top candidates, and the token counts that they read, against plain implementations on the host."""
import numpy as np
import pytest
import torch

from rexl3_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
NEG = float("-inf")


def t(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def plain(logits, count, row_slot=None, counts=None, penalties=None, bias=None, mask=None, window=None):
    """Row by row in numpy's float32, whose steps round as the definition's do; then sorted by (value descending, id ascending), NaN first."""
    f = np.float32
    x_all, ids, vals = logits.cpu().numpy(), [], []
    V = x_all.shape[1]
    h = lambda v: v.cpu().numpy()  # noqa: E731
    with np.errstate(all="ignore"):
        for r in range(x_all.shape[0]):
            x = x_all[r].copy()
            s = int(row_slot[r]) if row_slot is not None else -1
            if counts is not None and 0 <= s < counts.shape[0]:
                word = h(counts)[s].astype(np.int64)
                gen, prompt = word & 32767, word < 0
                if window is not None:
                    for q in range(max(0, int(window[0][r])) + 1, r + 1):
                        tok = int(window[1][q])
                        if 0 <= tok < V:
                            gen[tok] += 1
                rep, freq, pres = h(penalties)[s].astype(f)
                seen = prompt | (gen > 0)
                x = np.where(seen, np.where(x > 0, x / rep, x * rep), x)
                x = np.where(seen, x - freq * gen.astype(f), x)
                x = np.where(gen > 0, x - pres, x)
            if bias is not None and 0 <= s < bias[0].shape[0]:
                b = np.zeros(V, dtype=f)
                for i, v in zip(h(bias[0])[s], h(bias[1])[s]):
                    if 0 <= i < V:
                        b[i] += v
                x = x + b
            assert x.dtype == f
            if mask is not None and 0 <= int(mask[1][r]) < mask[0].shape[0]:
                words = h(mask[0])[int(mask[1][r])].view(np.uint32)
                x = np.where(words[np.arange(V) // 32] >> (np.arange(V) % 32).astype(np.uint32) & 1, x, f(NEG))
            order = np.lexsort((np.arange(V), -x, ~np.isnan(x)))[:count]
            ids.append(order)
            vals.append(x[order])
    return np.array(ids), np.array(vals)


def same(logits, count, row_slot=None, **kw):
    rows, V = logits.shape
    ids, vals = torch.full((rows, count), -9, dtype=torch.int32, device="cuda"), torch.zeros(rows, count, device="cuda")
    K.topk_adjusted(logits, count, K.topk_scratch(rows, V, count), ids, vals, row_slot, **kw)
    wi, wv = plain(logits, count, row_slot, **kw)
    assert np.array_equal(ids.cpu().numpy(), wi)
    assert np.array_equal(vals.cpu().numpy(), wv, equal_nan=True)        # every step rounds as the plain one does: the same bits


def rules(rows, V, slots, seed, hist=300, nb=7, bits=0.5):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=g)  # noqa: E731
    counts = torch.zeros(slots, V, dtype=torch.int32, device="cuda")
    counts.scatter_add_(1, (rand(slots, hist) * V).long(), torch.ones(slots, hist, dtype=torch.int32, device="cuda"))
    prompt = rand(slots, V) < 0.05
    words = (rand(max(1, rows // 2), (V + 31) // 32, 32) < bits).long()
    words = (words << torch.arange(32, device="cuda")).sum(2)
    return dict(row_slot=(rand(rows) * (slots + 1)).int() - 1, counts=(counts - 32768 * prompt.int()).to(torch.int16),
                penalties=torch.stack([0.7 + 0.6 * rand(slots), rand(slots) - 0.3, rand(slots) - 0.3], 1).contiguous(),
                bias=((rand(slots, nb) * V * 1.1).int(), 5 * rand(slots, nb) - 2.5),
                mask=((words - (words >> 31 << 32)).int(), (rand(rows) * rows).int() - 1),
                window=(torch.arange(rows, dtype=torch.int32, device="cuda") // 4 * 4, (rand(rows) * V).int()))


@pytest.mark.parametrize("rows,V,count", [(1, 1, 1), (1, 7, 7), (3, 64, 64), (2, 4095, 5), (2, 4096, 28), (5, 4097, 28), (4, 2048, 1), (6, 32003, 64), (9, 20000, 2), (3, 151936, 28), (13, 5001, 3)])
@pytest.mark.parametrize("which", ["all", "counts", "bias", "mask", "none"])
def test_rules(rows, V, count, which):
    g = torch.Generator(device="cuda").manual_seed(rows * V)
    kw = rules(rows, V, 5, rows + V)
    row_slot = kw.pop("row_slot")
    if which != "all":
        kw = {k: v for k, v in kw.items() if k in {"counts": ("counts", "penalties", "window"), "bias": ("bias",), "mask": ("mask",), "none": ()}[which]}
    same(4 * torch.randn(rows, V, device="cuda", generator=g), count, row_slot, **kw)


def test_without_rules_as_topk():
    x = torch.randn(17, 32003, device="cuda")
    a, b = [(torch.empty(17, 28, dtype=torch.int32, device="cuda"), torch.empty(17, 28, device="cuda")) for _ in range(2)]
    K.topk(x, 28, K.topk_scratch(17, 32003, 28), *a)
    K.topk_adjusted(x, 28, K.topk_scratch(17, 32003, 28), *b)
    assert all(torch.equal(p, q) for p, q in zip(a, b))


@pytest.mark.parametrize("pad,offset", [(1, 0), (4, 0), (64, 3), (0, 1)])
@pytest.mark.parametrize("V", [4100, 8191])
def test_rows_apart_and_unaligned(V, pad, offset):
    base = torch.randn(6 * (V + pad) + 8, device="cuda")
    x = base[offset:offset + 6 * (V + pad)].view(6, V + pad)[:, :V]
    kw = rules(6, V, 3, V)
    same(x, 28, kw.pop("row_slot"), **kw)


@pytest.mark.parametrize("allowed", [0, 1, 5, 27, 28, 29, 700])
def test_few_ids_left(allowed):
    """Fewer ids above -inf than places: the lowest others, at -inf."""
    V = 9001
    x = torch.randn(3, V, device="cuda")
    x[1, :40] = NEG
    x[2, 100:] = NEG
    keep = torch.zeros(3, (V + 31) // 32 * 32, dtype=torch.bool, device="cuda")
    keep[:, torch.randperm(V, device="cuda")[:allowed]] = True
    words = (keep.view(3, -1, 32).long() << torch.arange(32, device="cuda")).sum(2)
    same(x, 28, mask=((words - (words >> 31 << 32)).int().contiguous(), t([0, 1, 2])))


@pytest.mark.parametrize("allowed", [[], [0], list(range(63)), list(range(64)), list(range(0, 126, 2)), list(range(63, 127)), [0, 500] + list(range(64, 125)), [8999]])
def test_places_without_a_candidate_take_the_lowest_ids(allowed):
    V = 9001
    x = torch.full((1, V), NEG, device="cuda")
    x[0, allowed] = torch.randn(len(allowed), device="cuda")
    same(x, 64)


def test_infinities_nan_and_masked_nan():
    V = 5000
    x = torch.randn(4, V, device="cuda")
    x[0, [3, 4500]] = float("inf")
    x[1, [17, 4999]] = float("nan")
    x[1, 20] = -torch.tensor(float("nan"))
    x[2, 10:4000] = float("nan")                         # all of these are masked
    x[3] = torch.finfo(torch.float32).min
    x[3, 7] = NEG
    keep = torch.ones(1, 5024, dtype=torch.bool, device="cuda")
    keep[0, 10:4000] = False
    words = (keep.view(1, -1, 32).long() << torch.arange(32, device="cuda")).sum(2)
    kw = rules(4, V, 2, 1)
    kw["mask"] = ((words - (words >> 31 << 32)).int(), t([-1, -1, 0, 9]))
    kw["row_slot"] = t([0, 1, 1, 0])
    same(x, 28, **kw)


@pytest.mark.parametrize("value", [0.0, -0.0, 1.5, -3.0])
def test_equal_values_go_by_id(value):
    x = torch.full((2, 12345), value, device="cuda")
    x[1, ::2] = -value
    same(x, 64)
    same(x, 1)


def test_a_bias_given_more_than_once_adds_up_in_order():
    V, nb = 6000, 300
    ids = (torch.arange(nb, device="cuda") % 3 * 5 + 4090).int()[None]
    vals = (10.0 ** torch.linspace(-6, 6, nb, device="cuda") * torch.where(torch.arange(nb, device="cuda") % 2 == 0, 1.0, -0.999))[None].contiguous()
    same(torch.randn(1, V, device="cuda"), 28, t([0]), bias=(ids, vals))
    same(torch.randn(1, V, device="cuda"), 28, t([0]), bias=(torch.full((1, 1024), 5, dtype=torch.int32, device="cuda"), torch.randn(1, 1024, device="cuda")))


@pytest.mark.parametrize("rows,V", [(740, 100), (741, 100), (741, 5000), (371, 8192), (150, 20000)])
def test_more_rows_than_run_at_once(rows, V):
    kw = rules(rows, V, 9, rows + V, hist=50)
    same(torch.randn(rows, V, device="cuda"), 5, kw.pop("row_slot"), **kw)


@pytest.mark.parametrize("V,nb", [(2048, 200), (2048, 1024), (9000, 1024), (40, 1000)])
def test_many_biases_and_drafts(V, nb):
    kw = rules(12, V, 2, V + nb, nb=nb)
    kw["bias"][0].remainder_(max(V // 4, 30))                            # most ids more than once, some of them among the drafts
    kw["window"] = (kw["window"][0], kw["window"][1].remainder(max(V // 4, 30)))
    same(torch.randn(12, V, device="cuda"), 28, kw.pop("row_slot"), **kw)


def test_drafts_of_a_window_count_for_the_rows_behind_them():
    V = 300
    x = torch.zeros(6, V, device="cuda")
    x[:, 10], x[:, 11], x[:, 12] = 5.0, 4.0, 3.0
    counts = torch.zeros(2, V, dtype=torch.int16, device="cuda")
    counts[1, 12] = -32768
    kw = dict(counts=counts, penalties=torch.tensor([[1.0, 1.5, 0.25], [2.0, 1.0, 0.0]], device="cuda"), window=(t([0, 0, 0, 0, 4, 4]), t([10, 10, 10, 11, 10, 12])))
    row_slot = t([0, 0, 0, 0, 1, 1])
    same(x, 4, row_slot, **kw)
    ids, vals = torch.empty(6, 4, dtype=torch.int32, device="cuda"), torch.empty(6, 4, device="cuda")
    K.topk_adjusted(x, 4, K.topk_scratch(6, V, 4), ids, vals, row_slot, **kw)
    assert ids[0].tolist()[:3] == [10, 11, 12] and ids[1].tolist()[:3] == [11, 10, 12] and ids[2].tolist()[:3] == [11, 12, 10]
    assert vals[2].tolist()[:3] == [4.0, 3.0, 1.75]


@pytest.mark.parametrize("n,V,lens", [(1, 1, [3]), (1, 5, [0]), (3, 151936, [900, 0, 5000]), (5, 32003, [1, 2, 40000, 7, 7]), (70, 2049, [(i * 37) % 500 for i in range(70)])])
def test_counts_of_histories(n, V, lens):
    g = torch.Generator().manual_seed(V)
    slots = torch.randperm(n + 3, generator=g)[:n].tolist()
    hist = [((V * torch.rand(k, generator=g) ** 4).long().clamp_max(V - 1)).tolist() for k in lens]
    cut = [k * 2 // 3 for k in lens]
    before = torch.randint(-30000, 30000, (n + 3, V), generator=g).to(torch.int16)
    want = before.numpy().astype(np.int64)
    for s, hs, c in zip(slots, hist, cut):
        w = np.zeros(V, dtype=np.int64)
        np.add.at(w, hs[c:], 1)
        w = np.minimum(w, 32767)
        w[hs[:c]] -= 32768
        want[s] = w
    starts = np.concatenate([[0], np.cumsum(lens)]).tolist()
    counts, st = before.cuda(), K.new_status()
    K.token_counts(counts, t(slots), t(starts), t(cut), t([x for hs in hist for x in hs] + [1]), st)
    K.check_status(st)
    assert np.array_equal(counts.cpu().numpy(), want)


def test_counts_stop_at_their_limit():
    V = 10
    counts, st = torch.zeros(2, V, dtype=torch.int16, device="cuda"), K.new_status()
    K.token_counts(counts, t([1]), t([0, 40002]), t([1]), t([3] + [3] * 40000 + [4]), st)
    assert counts[1].tolist() == [0, 0, 0, -1, 1, 0, 0, 0, 0, 0] and (counts[0] == 0).all()
    counts[0, 2] = 32766
    K.token_counts_add(counts, t([0] * 5), t([2] * 5), st)
    K.token_counts_add(counts, t([0] * 3000 + [1]), t([7] * 3000 + [4]), st)
    K.token_counts_add(counts, t([0, 0, 1]), t([2, 9, 0]), st, prompt=True)
    K.check_status(st)
    assert counts[0].tolist() == [0, 0, -1, 0, 0, 0, 0, 3000, 0, -32768] and counts[1].tolist() == [-32768, 0, 0, -1, 2, 0, 0, 0, 0, 0]


def test_counts_pass_over_what_is_wrong():
    V, before = 50, torch.full((3, 50), 5, dtype=torch.int16, device="cuda")
    for slots, starts, tokens, want in (([0, 3], [0, 2, 4], [1, 1, 2, 2], {0: {1: 2}}), ([-1, 1], [0, 2, 4], [1, 1, 2, 2], {1: {2: 2}}), ([2, 2], [0, 2, 4], [1, 1, 2, 2], {2: {1: 2}}),
                                        ([0, 1], [0, 2, 9], [1, 1, 2, 2], {0: {1: 2}}), ([0, 1], [0, 3, 2], [1, 1, 1, 2], {0: {1: 3}}), ([0], [0, 4], [1, -1, 50, 49], {0: {1: 1, 49: 1}})):
        counts, st = before.clone(), K.new_status()
        K.token_counts(counts, t(slots), t(starts), t([0] * len(slots)), t(tokens), st)
        assert st[0].item() == K.ST_BAD_ARG
        for s in range(3):
            assert counts[s].tolist() == ([want[s].get(i, 0) for i in range(V)] if s in want else [5] * V)
    counts, st = before.clone(), K.new_status()
    K.token_counts_add(counts, t([0, -1, 3, 1, 1]), t([1, 1, 1, 50, -1]), st)
    assert st[0].item() == K.ST_BAD_ARG
    before[0, 1] += 1
    assert torch.equal(counts, before)


def test_counts_feed_the_rules():
    """Admission, two steps and a resumption: the table that the steps kept is the one that the whole history gives, and the picks follow it."""
    V, prompt = 1000, [5, 6, 7, 7]
    st, counts, again = K.new_status(), torch.zeros(2, V, dtype=torch.int16, device="cuda"), torch.zeros(2, V, dtype=torch.int16, device="cuda")
    K.token_counts(counts, t([1]), t([0, 4]), t([4]), t(prompt), st)
    x, pen = torch.randn(1, V, device="cuda"), torch.tensor([[1.0, 0.0, 0.0], [1.3, 0.7, 0.4]], device="cuda")
    made = []
    ids, vals = torch.empty(1, 8, dtype=torch.int32, device="cuda"), torch.empty(1, 8, device="cuda")
    for _ in range(20):
        K.topk_adjusted(x, 8, K.topk_scratch(1, V, 8), ids, vals, t([1]), counts=counts, penalties=pen)
        made.append(int(ids[0, 0]))
        K.token_counts_add(counts, t([1]), ids[0, :1].contiguous(), st)
    K.token_counts(again, t([1]), t([0, 24]), t([4]), t(prompt + made), st)
    K.check_status(st)
    assert torch.equal(counts, again) and len(set(made)) > 3
    same(x, 8, t([1]), counts=counts, penalties=pen)


def test_refusals():
    x, V = torch.randn(2, 100, device="cuda"), 100
    sc, ids, vals, st = K.topk_scratch(2, V, 8), torch.zeros(2, 8, dtype=torch.int32, device="cuda"), torch.zeros(2, 8, device="cuda"), K.new_status()
    counts, pen, slot = torch.zeros(3, V, dtype=torch.int16, device="cuda"), torch.ones(3, 3, device="cuda"), t([0, 1])
    bad = [dict(logits=x.half()), dict(logits=x.t()), dict(logits=x[0]), dict(logits=x.cpu()), dict(logits=x[:1].expand(2, V)), dict(count=0), dict(count=65), dict(ids=ids.long()), dict(ids=ids[:1]),
           dict(vals=vals[:, :4]), dict(scratch=sc[:1]), dict(counts=counts), dict(penalties=pen), dict(counts=counts, penalties=pen, row_slot=None), dict(counts=counts[:, :50], penalties=pen),
           dict(counts=counts.int(), penalties=pen), dict(counts=counts, penalties=pen[:2]), dict(counts=counts, penalties=pen.t()), dict(row_slot=slot[:1], counts=counts, penalties=pen),
           dict(bias=(t([[0], [1]]), torch.zeros(3, 1, device="cuda"))), dict(bias=(t([[0], [1], [2]]).repeat(1, 1025), torch.zeros(3, 1025, device="cuda"))), dict(mask=(t([[0, 0, 0]]), slot)),
           dict(mask=(t([[0, 0, 0, 0]]), slot[:1])), dict(window=(slot, slot[:1])), dict(window=(slot.long(), slot)), dict(counts=counts, penalties=pen, bias=(t([[0]]), torch.zeros(1, 1, device="cuda")))]
    for kw in bad:
        a = {**dict(logits=x, count=8, scratch=sc, ids=ids, vals=vals, row_slot=slot), **kw}
        with pytest.raises(ValueError):
            K.topk_adjusted(**a)
    with pytest.raises(ValueError):
        K.topk_adjusted(torch.randn(1, 5, device="cuda"), 8, sc, ids[:1], vals[:1])
    many, zero = torch.zeros(4097, 8, device="cuda"), torch.zeros(4097, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="4096"):
        K.topk_adjusted(many, 1, K.topk_scratch(4097, 8, 1), zero[:, None], many[:, :1].contiguous(), window=(zero, zero))
    with pytest.raises(ValueError, match="boundary"):
        K.topk_adjusted(x, 8, torch.empty(4096, dtype=torch.uint8, device="cuda")[4:], ids, vals)
    K.topk_adjusted(torch.empty(0, V, device="cuda"), 8, sc, ids[:0], vals[:0])
    for a in ((counts.int(), slot, t([0, 1, 2]), slot, slot, st), (counts, slot, slot, slot, slot, st), (counts, slot, t([0, 1, 2]), slot[:1], slot, st), (counts, slot.long(), t([0, 1, 2]), slot, slot, st),
              (counts[:, ::2], slot, t([0, 1, 2]), slot, slot, st), (counts, slot, t([0, 1, 2]), slot, slot.cpu(), st)):
        with pytest.raises(ValueError):
            K.token_counts(*a)
    with pytest.raises(ValueError):
        K.token_counts_add(counts, slot, slot[:1], st)
    K.token_counts(counts, slot[:0], t([0]), slot[:0], slot, st)
    K.token_counts_add(counts, slot[:0], slot[:0], st)
    K.check_status(st)

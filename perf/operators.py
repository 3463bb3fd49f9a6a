"""What is timed: the operators of one decode step of a batch whose streams share a prompt and run under sampling rules.

    rows     block tables and per-row slot maps, made on the device from the requests' lengths
    attn     paged attention of a decode / verify window, pages that neighbouring sequences share read once for all of them
    pick     repetition / frequency / presence penalties, biases and grammar masks on logits, then the exact top candidates
    counts   the token counts that the penalties read, rebuilt from the histories of requests that are admitted or resumed

A case is a dict of plain values; its "op" says which operator it runs.  Head counts, page size, vocabularies and candidate counts are those of the
repository's own configurations.  `own` selects the framework's kernels; without it `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

PAGE = 64
DEV = "cuda"


# ---------------------------------------------------------------------------------------------------------------- cases
def _rows(name, reqs, have_lo, have_hi, new_lo, new_hi, prefix):
    c = {"op": "rows", "reqs": reqs, "have_lo": have_lo, "have_hi": have_hi, "new_lo": new_lo, "new_hi": new_hi, "prefix": prefix}
    return c if name is None else {"name": name, **c}


def _attn(name, n_q, n_kv, hd, groups, seqs, rows, prefix, own_lo, own_hi, kv="bf16"):
    c = {"op": "attn", "n_q": n_q, "n_kv": n_kv, "hd": hd, "groups": groups, "seqs": seqs, "rows": rows, "prefix": prefix, "own_lo": own_lo, "own_hi": own_hi, "kv": kv}
    return c if name is None else {"name": name, **c}


def _pick(name, seqs, rows, vocab, count, hist, bias, masked, pad):
    c = {"op": "pick", "seqs": seqs, "rows": rows, "vocab": vocab, "count": count, "hist": hist, "bias": bias, "masked": masked, "pad": pad}
    return c if name is None else {"name": name, **c}


def _counts(name, reqs, vocab, len_lo, len_hi):
    c = {"op": "counts", "reqs": reqs, "vocab": vocab, "len_lo": len_lo, "len_hi": len_hi}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # a loaded server's plain decode step: 64 streams behind one 8K system prompt, one new token each
        _rows("rows_step_64", 64, 8200, 9000, 1, 1, 8192),
        # one slice of ragged prompts over a cached system prompt
        _rows("rows_prompts_ragged", 23, 333, 333, 61, 650, 333),
        # two streams of a small model behind a short prompt: nothing but latency
        _attn("attn_pair_small", 4, 2, 64, 1, 2, 1, 200, 3, 40),
        # the throughput point: 64 streams that share an 8K prompt, some hundred own tokens each
        _attn("attn_64_8k", 40, 8, 128, 1, 64, 1, 8192, 60, 700),
        # speculative verify windows: 16 streams with 4 drafts each, two prompts of odd length
        _attn("attn_verify_16x5", 32, 4, 128, 2, 16, 5, 4001, 20, 300),
        # a long shared document on the byte-wide cache
        _attn("attn_fp8_32k", 40, 8, 128, 1, 32, 1, 32700, 100, 900, kv="fp8"),
        # many streams, hardly anything shared: a short common instruction, long own contexts
        _attn("attn_own_48", 40, 8, 128, 1, 48, 1, 150, 500, 4000),
        # one stream under a grammar
        _pick("pick_1", 1, 1, 151936, 28, 1500, 8, 1, 0),
        # a full batch: penalties everywhere, every other stream under a grammar
        _pick("pick_64", 64, 1, 151936, 28, 4000, 16, 2, 0),
        # verify windows over an odd vocabulary in padded rows
        _pick("pick_verify_16x5", 16, 5, 32003, 64, 800, 3, 2, 61),
        # one request admitted with a short prompt
        _counts("counts_1", 1, 151936, 900, 900),
        # a batch resumed with its whole histories
        _counts("counts_64", 64, 151936, 2000, 9000),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    op = rng.choice(["rows", "attn", "attn", "attn", "pick", "pick", "counts"])
    if op == "rows":
        reqs = log(1, 256)
        prefix = rng.choice([0, log(10, 8000)])
        lo = prefix + rng.choice([0, log(1, 500)])
        new_hi = rng.choice([1, log(1, 8), log(8, max(9, 8192 // reqs))])
        return _rows(None, reqs, lo, lo + log(1, 2000), rng.choice([0, 1]) if new_hi > 1 and reqs > 1 else 1, new_hi, prefix)
    if op == "attn":
        n_q, n_kv, hd = rng.choice([(40, 8, 128), (40, 8, 128), (32, 4, 128), (20, 4, 128), (5, 1, 128), (4, 2, 64), (16, 16, 64), (32, 2, 128)])
        rows = rng.choice([1, 1, 1, log(2, 8)])
        seqs = log(1, min(96, 320 // rows))
        groups = min(seqs, rng.choice([1, 1, 2, 5]))
        budget = 24_000_000 // (n_q * rows * seqs)                   # (query head, key) pairs a row may have: 64 x 9000 keys of 40 heads
        prefix = log(1, max(2, min(32768, budget * 2 // 3)))
        hi = log(rows + 1, max(rows + 2, min(4000, budget // 3, 100_000_000 // (seqs * n_kv * hd))))
        return _attn(None, n_q, n_kv, hd, groups, seqs, rows, prefix, rng.randint(rows, hi), hi, rng.choice(["bf16", "bf16", "fp8"]) if hd == 128 else "bf16")
    if op == "pick":
        rows = rng.choice([1, 1, log(2, 8)])
        seqs = log(1, 64 // rows)
        return _pick(None, seqs, rows, rng.choice([2048, 32768, 151936, log(300, 151936)]), rng.choice([1, 2, 4, 28, 64, rng.randint(1, 64)]), log(1, 8000),
                     rng.choice([0, log(1, 300)]), rng.choice([0, 1, 2, 3]), rng.choice([0, 0, rng.randint(1, 64)]))
    reqs = log(1, 64)
    lo = log(1, 8000)
    return _counts(None, reqs, rng.choice([2048, 151936, log(300, 151936)]), rng.choice([0, lo]), lo)


def work(case):
    if case["op"] == "rows":
        have, new = _spread(case["reqs"], case["have_lo"], case["have_hi"]), _spread(case["reqs"], case["new_lo"], case["new_hi"])
        fed = sum(1 for n in new if n)
        pages = sum((h + n + PAGE - 1) // PAGE - (h + PAGE - 1) // PAGE for h, n in zip(have, new))
        return {"bytes": 12 * case["reqs"] + 20 * sum(new) + 8 * pages + 4 * fed * (case["prefix"] // PAGE) + 4 * sum((n + PAGE - 1) // PAGE for n in new), "flops": 0}
    if case["op"] == "attn":
        base, lens = case["prefix"] // PAGE * PAGE, [case["prefix"] + n for n in _spread(case["seqs"], case["own_lo"], case["own_hi"])]
        keys = case["groups"] * base + sum(n - base for n in lens)
        fed = case["seqs"] * case["rows"]
        pairs = sum(n * case["rows"] - case["rows"] * (case["rows"] - 1) // 2 for n in lens)
        return {"bytes": 2 * keys * case["n_kv"] * case["hd"] * (1 if case["kv"] == "fp8" else 2) + 4 * fed * case["n_q"] * case["hd"],
                "flops": 4 * pairs * case["n_q"] * case["hd"]}
    if case["op"] == "pick":
        fed, V = case["seqs"] * case["rows"], case["vocab"]
        masks = 0 if not case["masked"] else (case["seqs"] + case["masked"] - 1) // case["masked"] * case["rows"]
        return {"bytes": 4 * fed * V + 2 * case["seqs"] * V + masks * V // 8 + 8 * fed * case["count"], "flops": 4 * fed * V}
    lens = _spread(case["reqs"], case["len_lo"], case["len_hi"])
    return {"bytes": 2 * case["reqs"] * case["vocab"] + 4 * sum(lens), "flops": 0}


def _spread(n, lo, hi):
    """n lengths from lo to hi, ends included."""
    return [lo + (hi - lo) * i // max(1, n - 1) for i in range(n)]


# ---------------------------------------------------------------------------------------------------------------- inputs
class _Seeded:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)
        self.cpu = torch.Generator().manual_seed(seed)

    def randn(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=self.g, dtype=dtype)

    def rand(self, *shape):
        return torch.rand(*shape, device=DEV, generator=self.g)

    def shuffled(self, values):
        return [values[i] for i in torch.randperm(len(values), generator=self.cpu).tolist()]


def _i32(v):
    return torch.as_tensor(v, dtype=torch.int32).to(DEV)


def prepare(case, seed):
    r = _Seeded(seed)
    s = {"case": case, **{"rows": _prepare_rows, "attn": _prepare_attn, "pick": _prepare_pick, "counts": _prepare_counts}[case["op"]](case, r)}
    return s


def _tables(r, group_of, shared, lens, slots, width, spare):
    """Page tables [slots, width] of sequences of `lens` tokens, whose first `shared` pages are their group's, and pages left over.  Pages are in no order."""
    groups = max(group_of) + 1
    total = groups * shared + sum(max(0, (n + PAGE - 1) // PAGE - shared) for n in lens) + spare
    ids = r.shuffled(list(range(total)))
    table = torch.full((slots, width), -1, dtype=torch.int32)
    seqs = r.shuffled(list(range(slots)))[:len(lens)]
    common = [torch.tensor([ids.pop() for _ in range(shared)], dtype=torch.int32) for _ in range(groups)]
    for s, g, n in zip(seqs, group_of, lens):
        k = (n + PAGE - 1) // PAGE
        table[s, :shared] = common[g]
        if k > shared:
            table[s, shared:k] = torch.tensor([ids.pop() for _ in range(k - shared)], dtype=torch.int32)
    return table, seqs, ids, total


def _prepare_rows(case, r):
    n = case["reqs"]
    have, new = r.shuffled(_spread(n, case["have_lo"], case["have_hi"])), r.shuffled(_spread(n, case["new_lo"], case["new_hi"]))
    need = sum((h + k + PAGE - 1) // PAGE - (h + PAGE - 1) // PAGE for h, k in zip(have, new))
    width = max((h + k + PAGE - 1) // PAGE for h, k in zip(have, new)) + 1
    table, seqs, left, total = _tables(r, [0] * n, case["prefix"] // PAGE, have, n + 3, width, need + 5)
    return {"seq": _i32(seqs), "have": _i32(have), "new": _i32(new), "table": table.to(DEV), "free": _i32(left), "free_at": _i32([2]), "free_next": _i32([0]),
            "rows": torch.zeros(5, sum(new), dtype=torch.int32, device=DEV), "starts": torch.zeros(n + 1, dtype=torch.int32, device=DEV),
            "status": torch.zeros(8, dtype=torch.int32, device=DEV), "need": need}


def _prepare_attn(case, r):
    n, R, n_kv, hd = case["seqs"], case["rows"], case["n_kv"], case["hd"]
    shared = case["prefix"] // PAGE
    lens = r.shuffled([case["prefix"] + k for k in _spread(n, case["own_lo"], case["own_hi"])])
    group_of = [i * case["groups"] // n for i in range(n)]
    width = max(shared, max((k + PAGE - 1) // PAGE for k in lens)) + 2
    table, seqs, _, total = _tables(r, group_of, shared, lens, n + 2, width, 3)
    k, v = (r.randn(total, n_kv, PAGE, hd, dtype=torch.bfloat16) for _ in range(2))
    scale = None
    if case["kv"] == "fp8":                                          # stored as value / scale of the head
        scale = 0.012 + 0.01 * r.rand(2, n_kv)
        k, v = ((x.float() / scale[i][None, :, None, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8) for i, x in enumerate((k, v)))
    ctx = [m - R + 1 + j for m in lens for j in range(R)]            # the window's rows are the last R positions of their sequence
    common = [shared if i > 0 and group_of[i] == group_of[i - 1] else 0 for i in range(n) for _ in range(R)]
    return {"k": k, "v": v, "kv_scale": scale, "q": r.randn(n * R, case["n_q"] * hd, dtype=torch.bfloat16), "table": table.to(DEV),
            "row_seq": _i32([s for s in seqs for _ in range(R)]), "ctx": _i32(ctx), "common": _i32(common), "longest": max(lens),
            "out": torch.zeros(n * R, case["n_q"] * hd, dtype=torch.bfloat16, device=DEV), "status": torch.zeros(8, dtype=torch.int32, device=DEV), "kept": {}}


def _prepare_pick(case, r):
    n, R, V = case["seqs"], case["rows"], case["vocab"]
    slots, fed = n + 2, n * R
    which = r.shuffled(list(range(slots)))[:n]
    logits = (3.0 * r.randn(fed, V + case["pad"]))[:, :V]
    # histories: some tokens often, most once; the first half is the prompt
    hist = (V * r.rand(slots, case["hist"]) ** 3).long().clamp_max(V - 1)
    half = case["hist"] // 2
    counts = torch.zeros(slots, V, dtype=torch.int32, device=DEV)
    counts.scatter_add_(1, hist[:, half:], torch.ones_like(hist[:, half:], dtype=torch.int32))
    prompt = torch.zeros(slots, V, dtype=torch.bool, device=DEV)
    prompt.scatter_(1, hist[:, :half], True)
    rules = torch.stack([1.0 + 0.3 * r.rand(slots), 0.5 * r.rand(slots), 0.6 * r.rand(slots)], 1).contiguous()
    s = {"logits": logits, "row_slot": _i32([w for w in which for _ in range(R)]), "counts": (counts - 32768 * prompt.int()).to(torch.int16), "rules": rules,
         "first": _i32([i * R for i in range(n) for _ in range(R)]), "fed": (V * r.rand(fed) ** 3).int().clamp_max(V - 1), "bias": None, "mask": None,
         "ids": torch.zeros(fed, case["count"], dtype=torch.int32, device=DEV), "vals": torch.zeros(fed, case["count"], device=DEV), "kept": {}}
    if case["bias"]:
        nb = min(case["bias"], V)
        ids = torch.argsort(r.rand(slots, V), dim=1)[:, :nb].int()   # every id once, some places unused
        ids[:, nb // 2::5] = -1
        s["bias"] = (ids.contiguous(), 4.0 * r.randn(slots, nb))
    if case["masked"]:
        # every masked-th stream is under a grammar: rows in turn allow a handful of ids, or nearly all
        rows = [i * R + j for i in range(0, n, case["masked"]) for j in range(R)]
        keep = r.rand(len(rows), (V + 31) // 32 * 32) < torch.where(torch.arange(len(rows), device=DEV) % 2 == 0, 0.002, 0.98)[:, None]
        bits = (keep.view(len(rows), -1, 32).long() << torch.arange(32, device=DEV)).sum(2)
        mask_row = torch.full((fed,), -1, dtype=torch.int32)
        mask_row[rows] = torch.arange(len(rows), dtype=torch.int32)
        s["mask"] = ((bits - (bits >> 31 << 32)).int(), mask_row.to(DEV))
    return s


def _prepare_counts(case, r):
    n, V = case["reqs"], case["vocab"]
    lens = r.shuffled(_spread(n, case["len_lo"], case["len_hi"]))
    starts = [0]
    for k in lens:
        starts.append(starts[-1] + k)
    slots = n + 1
    return {"counts": torch.full((slots, V), 77, dtype=torch.int16, device=DEV), "slots": _i32(r.shuffled(list(range(slots)))[:n]), "starts": _i32(starts),
            "prompt": _i32([k * 3 // 4 for k in lens]), "tokens": (V * r.rand(starts[-1]) ** 3).int().clamp_max(V - 1), "lens": lens,
            "status": torch.zeros(8, dtype=torch.int32, device=DEV)}


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"rows": _own_rows, "attn": _own_attn, "pick": _own_pick, "counts": _own_counts}[op](s)
    return {"rows": _plain_rows, "attn": _plain_attn, "pick": _plain_pick, "counts": _plain_counts}[op](s)


def _own_rows(s):
    from rexl3_b200.ops import kernels as K
    K.window_rows(s["seq"], s["have"], s["new"], s["table"], s["rows"], s["starts"], s["status"], free=s["free"], free_at=s["free_at"], free_next=s["free_next"])
    return {"rows": s["rows"], "starts": s["starts"], "table": s["table"], "free_next": s["free_next"]}


def _plain_rows(s):
    seq, have, new = s["seq"].long(), s["have"].long(), s["new"].long()
    n, M, end = seq.numel(), s["rows"].shape[1], have + new
    held, pages = (have + PAGE - 1) // PAGE, (end + PAGE - 1) // PAGE
    need = pages - held
    table = s["table"]
    # pages of request i, in order, behind the ones of the requests before
    who = torch.repeat_interleave(torch.arange(n, device=DEV), need, output_size=s["need"])
    at = torch.arange(s["need"], device=DEV)
    table[seq[who], held[who] + at - (need.cumsum(0) - need)[who]] = s["free"][s["free_at"].long() + at]
    # pages in common with the request before that has rows
    ids = torch.arange(n, device=DEV)
    before = torch.where(new > 0, ids, -1).cummax(0).values
    before = torch.cat([before.new_full((1,), -1), before[:-1]])
    both = torch.minimum(held, held[before.clamp_min(0)])[:, None] > torch.arange(table.shape[1], device=DEV)
    same = (table[seq] == table[seq[before.clamp_min(0)]]) & both
    common = torch.where(before >= 0, same.int().cumprod(1).sum(1), 0)
    starts = torch.cat([new.new_zeros(1), new.cumsum(0)])
    row = torch.repeat_interleave(ids, new, output_size=M)
    pos = have[row] + torch.arange(M, device=DEV) - starts[row]
    slot = table[seq[row], pos // PAGE].long() * PAGE + pos % PAGE
    return {"rows": torch.stack([pos, slot, seq[row], pos + 1, common[row]]).int(), "starts": starts.int(), "table": table, "free_next": (s["free_at"] + need.sum()).int()}


def _own_attn(s):
    from rexl3_b200.ops import kernels as K
    c, kept = s["case"], s["kept"]
    if not kept:                                                     # tensor maps and scratch, as a model keeps them
        kept["maps"] = K.KvTensorMap(s["k"]), K.KvTensorMap(s["v"])
        kept["scratch"] = K.attn_shared_scratch(s["q"].shape[0], c["n_q"], c["n_kv"], c["hd"])
    K.attn_shared(*kept["maps"], s["q"], s["table"], s["row_seq"], s["ctx"], s["common"], kept["scratch"], c["n_q"], c["n_kv"], c["hd"], c["hd"] ** -0.5,
                  s["out"], s["status"], kv_scale=s["kv_scale"])
    return s["out"]


def _plain_attn(s):
    c = s["case"]
    n_kv, hd, R = c["n_kv"], c["hd"], s["q"].shape[0]
    G, pages = c["n_q"] // n_kv, (s["longest"] + PAGE - 1) // PAGE

    def cache(x, i):                                                 # every sequence's own view of its keys: [seq, n_kv, keys, hd]
        x = x if s["kv_scale"] is None else x.view(torch.float8_e4m3fn)
        x = x.view(torch.uint8 if s["kv_scale"] is not None else x.dtype)[s["table"][s["row_seq"][::c["rows"]].long(), :pages].clamp_min(0).long()]
        x = (x if s["kv_scale"] is None else x.view(torch.float8_e4m3fn)).float()
        x = x.transpose(1, 2).reshape(x.shape[0], n_kv, pages * PAGE, hd)
        return x if s["kv_scale"] is None else x * s["kv_scale"][i][None, :, None, None]

    q = s["q"].float().view(-1, c["rows"], n_kv, G, hd).permute(0, 2, 1, 3, 4).reshape(-1, n_kv, c["rows"] * G, hd)
    x = torch.matmul(q, cache(s["k"], 0).transpose(2, 3)).mul_(hd ** -0.5).view(-1, n_kv, c["rows"], G, pages * PAGE)
    x.masked_fill_(torch.arange(pages * PAGE, device=DEV) >= s["ctx"].view(-1, 1, c["rows"], 1, 1), float("-inf"))
    x = (x - x.amax(-1, keepdim=True)).exp_()
    x /= x.sum(-1, keepdim=True)
    out = torch.matmul(x.view(-1, n_kv, c["rows"] * G, pages * PAGE), cache(s["v"], 1))
    return out.view(-1, n_kv, c["rows"], G, hd).transpose(1, 2).reshape(R, c["n_q"] * hd).bfloat16()


def _own_pick(s):
    from rexl3_b200.ops import kernels as K
    kept = s["kept"]
    if not kept:
        kept["scratch"] = K.topk_scratch(s["logits"].shape[0], s["logits"].shape[1], s["case"]["count"])
    K.topk_adjusted(s["logits"], s["case"]["count"], kept["scratch"], s["ids"], s["vals"], s["row_slot"], counts=s["counts"], penalties=s["rules"], bias=s["bias"],
                    mask=s["mask"], window=(s["first"], s["fed"]))
    return {"ids": s["ids"], "vals": s["vals"]}


def _plain_pick(s):
    x, slot = s["logits"], s["row_slot"].long()
    R, V = x.shape
    c = s["counts"][slot].int()
    prompt, c = c < 0, c & 32767
    # the drafts of a row's window up to the row itself
    j = torch.arange(R, device=DEV)
    c.scatter_add_(1, s["fed"].long().expand(R, R), ((j > s["first"].view(-1, 1)) & (j <= j.view(-1, 1))).int())
    rep, freq, pres = (t.unsqueeze(1) for t in s["rules"][slot].unbind(1))
    x = torch.where(prompt | (c > 0), torch.where(x > 0, x / rep, x * rep), x)
    x = x - freq * c.float()
    x = x - torch.where(c > 0, pres, 0.0)
    if s["bias"] is not None:
        ids, vals = s["bias"][0][slot].long(), s["bias"][1][slot]
        x = x + torch.zeros(R, V + 1, device=DEV).scatter_add_(1, torch.where(ids < 0, V, ids), vals)[:, :V]
    if s["mask"] is not None:
        bits, row = s["mask"]
        v = torch.arange(V, device=DEV)
        ok = (bits[row.clamp_min(0).long()][:, v // 32] >> (v % 32)) & 1
        x = torch.where((ok != 0) | (row < 0).unsqueeze(1), x, float("-inf"))
    vals, ids = torch.sort(x, dim=1, descending=True, stable=True)
    k = s["case"]["count"]
    return {"ids": ids[:, :k].int().contiguous(), "vals": vals[:, :k].contiguous()}


def _own_counts(s):
    from rexl3_b200.ops import kernels as K
    K.token_counts(s["counts"], s["slots"], s["starts"], s["prompt"], s["tokens"], s["status"])
    return s["counts"]


def _plain_counts(s):
    counts, n, V = s["counts"], s["slots"].numel(), s["case"]["vocab"]
    at = torch.arange(s["tokens"].numel(), device=DEV)
    who = torch.searchsorted(s["starts"].long(), at, right=True) - 1
    in_prompt = at - s["starts"].long()[who] < s["prompt"].long()[who]
    flat = who * V + s["tokens"].long()
    c = torch.zeros(n * V, dtype=torch.int32, device=DEV).scatter_add_(0, flat, (~in_prompt).int())
    p = torch.zeros(n * V, dtype=torch.int32, device=DEV).scatter_add_(0, flat, in_prompt.int())
    counts[s["slots"].long()] = (c.clamp_max(32767) - 32768 * (p > 0).int()).to(torch.int16).view(n, V)
    return counts


# ---------------------------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    if case["op"] == "pick":
        return {"ids": None, "vals": _exact_pick(case, s)}
    return None                                                      # whole numbers only


def _exact_attn(case, s):
    hd, G = case["hd"], case["n_q"] // case["n_kv"]
    table, out = s["table"].tolist(), []
    for r, (seq, n) in enumerate(zip(s["row_seq"].tolist(), s["ctx"].tolist())):
        pages = torch.tensor(table[seq][:-(-n // PAGE)], device=DEV)
        heads = []
        for name, i in (("k", 0), ("v", 1)):
            x = s[name][pages]
            x = x.double() if s["kv_scale"] is None else x.view(torch.float8_e4m3fn).double() * s["kv_scale"][i].double().view(1, -1, 1, 1)
            heads.append(x.permute(1, 0, 2, 3).flatten(1, 2)[:, :n])
        q = s["q"][r].double().view(case["n_kv"], G, hd)
        w = torch.softmax(torch.einsum("hgd,hnd->hgn", q, heads[0]) / math.sqrt(hd), dim=-1)
        out.append(torch.einsum("hgn,hnd->hgd", w, heads[1]).reshape(-1))
    return torch.stack(out)


def _exact_pick(case, s):
    out, slots, fed, first = [], s["row_slot"].tolist(), s["fed"].tolist(), s["first"].tolist()
    for r, slot in enumerate(slots):
        x = s["logits"][r].double().clone()
        word = s["counts"][slot].long()
        n = torch.where(word < 0, word + 32768, word)
        for t in fed[first[r] + 1:r + 1]:
            n[t] += 1
        rep, freq, pres = (float(v) for v in s["rules"][slot])
        hit = (n > 0) | (word < 0)
        x[hit] = x[hit].clamp_min(0) / rep + x[hit].clamp_max(0) * rep
        x -= n.double() * freq + (n > 0).double() * pres
        if s["bias"] is not None:
            ids, vals = s["bias"][0][slot], s["bias"][1][slot]
            x.index_add_(0, ids[ids >= 0].long(), vals[ids >= 0].double())
        if s["mask"] is not None and int(s["mask"][1][r]) >= 0:
            words = s["mask"][0][int(s["mask"][1][r])].long() & 0xFFFFFFFF
            keep = ((words[:, None] >> torch.arange(32, device=DEV)) & 1).flatten()[:case["vocab"]].bool()
            x[~keep] = -math.inf
        out.append(torch.topk(x, case["count"]).values)
    return torch.stack(out)

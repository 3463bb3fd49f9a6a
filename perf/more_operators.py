"""What is timed: the operators of a feed-forward block whose weights and activations are 8-bit floating point (E4M3) with a scale for each block of 128.

    norm      the residual's addition and the root-mean-square norm, written as E4M3 rows with a float32 scale for each 128 columns
    act       SwiGLU of the gate | up rows, written the same way
    linear    the matrix product of such rows with a weight that has a float32 scale for each 128 x 128 block
    experts   the same product for routed experts: every row of a sorted list goes through its own expert's matrix

A case is a dict of plain values; its "op" says which operator it runs.  Widths, expert counts and top-k are those of the repository's own configurations.
`own` selects the framework's kernels; without it `run` computes the same in elementary torch operations.
"""
import math

import torch

own = False

BLOCK = 128
TINY = 2.0 ** -100                                                    # the least that a block's largest magnitude counts as
DEV = "cuda"
TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3 = torch.float8_e4m3fn


# ---------------------------------------------------------------------------------------------------------------- cases
def _norm(name, rows, d, terms, x, h, xn):
    """terms: 0 no addition (a model's first norm), 1 a sublayer's output, above that as many routed experts' outputs with their weights."""
    c = {"op": "norm", "rows": rows, "d": d, "terms": terms, "x": x, "h": h, "xn": xn}
    return c if name is None else {"name": name, **c}


def _act(name, rows, ffn, x):
    c = {"op": "act", "rows": rows, "ffn": ffn, "x": x}
    return c if name is None else {"name": name, **c}


def _linear(name, rows, k, n, out, bias):
    c = {"op": "linear", "rows": rows, "k": k, "n": n, "out": out, "bias": bias}
    return c if name is None else {"name": name, **c}


def _experts(name, rows, picks, experts, owned, k, n, form, out):
    """owned: the first so many of the experts are held here.  form: "up" reads the picking rows and writes sorted rows, "down" reads sorted rows and writes
    them where their (row, pick) pair stands."""
    c = {"op": "experts", "rows": rows, "picks": picks, "experts": experts, "owned": owned, "k": k, "n": n, "form": form, "out": out}
    return c if name is None else {"name": name, **c}


def listed():
    return [
        # one stream's decode step: nothing but latency
        _norm("norm_1", 1, 5120, 1, "bf16", "bf16", False),
        # a slice of a long prompt
        _norm("norm_8192", 8192, 5120, 1, "bf16", "bf16", False),
        # after routed experts: eight weighted outputs join the residual, and the router reads the plain norm too
        _norm("norm_experts_2100", 2100, 2048, 8, "bf16", "bf16", True),
        # a loaded server's decode step
        _act("act_64", 64, 17408, "bf16"),
        # a ragged slice of prompts
        _act("act_4097", 4097, 14336, "bf16"),
        # one stream's gate | up product: the weights' way from memory
        _linear("linear_1", 1, 5120, 34816, "bf16", False),
        # a loaded server's down product
        _linear("linear_64", 64, 17408, 5120, "bf16", False),
        # a short prompt through the latent projections: a half block of columns, rows kept in 32 bits
        _linear("linear_333", 333, 7168, 2112, "fp32", True),
        # a slice of a long prompt
        _linear("linear_8192", 8192, 5120, 34816, "bf16", False),
        # routed experts of a decode step: many experts, a row or two each
        _experts("experts_16", 16, 8, 128, 128, 2048, 1536, "up", "bf16"),
        # an eighth of a large model's experts, the rows of a loaded server
        _experts("experts_down_64", 64, 8, 256, 32, 2048, 7168, "down", "bf16"),
        # routed experts of a slice of prompts
        _experts("experts_2100", 2100, 8, 128, 128, 2048, 1536, "up", "bf16"),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))

    def width(lo, hi):                                               # a row of bytes that a copy can begin on: 16 of them
        return min(hi, max(lo, 16 * ((log(lo, hi) + 8) // 16)))
    op = rng.choice(["norm", "act", "linear", "linear", "linear", "experts", "experts"])
    if op == "norm":
        d = rng.choice([256, 2048, 4096, 5120, 7168, width(64, 16384)])
        terms = rng.choice([0, 1, 1, 1, 2, 8])
        return _norm(None, log(1, min(16384, 40_000_000 // (d * max(1, terms)))), d, terms, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.choice(["bf16", "bf16", "fp32"]),
                     rng.random() < 0.3)
    if op == "act":
        ffn = rng.choice([688, 768, 2048, 17408, width(64, 18432)])
        return _act(None, log(1, min(16384, 58_000_000 // ffn)), ffn, rng.choice(["bf16", "bf16", "fp16", "fp32"]))
    if op == "linear":
        k, n = rng.choice([(5120, 7168), (5120, 5120), (17408, 5120), (7168, 2112), (688, 256), (256, 1376), (4096, 28672), (width(64, 18432), log(1, 20000))])
        return _linear(None, log(1, min(8192, 200_000_000_000 // (k * n))), k, n, rng.choice(["bf16", "bf16", "fp16", "fp32"]), rng.random() < 0.3)
    experts, picks, k, n = rng.choice([(128, 8, 2048, 1536), (128, 8, 768, 2048), (256, 8, 2048, 7168), (256, 8, 7168, 4096), (8, 2, 256, 256), (rng.randint(4, 200), rng.randint(1, 4), width(64, 2048), log(16, 2000))])
    owned = max(1, min(experts, 470_000_000 // (k * n)))
    owned = rng.choice([owned, owned, rng.randint(1, owned)])
    least = -(-4 * experts // (picks * owned))                       # some pairs for the experts that are held
    return _experts(None, max(least, log(1, min(4096, 100_000_000_000 // (k * n * picks)))), picks, experts, owned, k, n, rng.choice(["up", "down"]), rng.choice(["bf16", "bf16", "fp16", "fp32"]))


def _size(t):
    return 4 if t == "fp32" else 2


def _blocks(n):
    return (n + BLOCK - 1) // BLOCK


def work(case):
    c = case
    if c["op"] == "norm":
        M, d = c["rows"], c["d"]
        b = M * d * (c["terms"] * _size(c["x"]) + (2 if c["terms"] else 1) * _size(c["h"]) + 1 + (2 if c["xn"] else 0)) + 4 * M * _blocks(d) + 2 * d + (4 * M * c["terms"] if c["terms"] > 1 else 0)
        return {"bytes": b, "flops": M * d * (2 * c["terms"] + 5)}
    if c["op"] == "act":
        return {"bytes": c["rows"] * (c["ffn"] * (2 * _size(c["x"]) + 1) + 4 * _blocks(c["ffn"])), "flops": 8 * c["rows"] * c["ffn"]}
    k, n = c["k"], c["n"]
    if c["op"] == "linear":
        return {"bytes": c["rows"] * (k + 4 * _blocks(k) + n * _size(c["out"])) + n * k + 4 * _blocks(n) * _blocks(k), "flops": 2 * c["rows"] * n * k}
    # rows pick experts evenly: what is held here gets its share of the pairs, and the experts that nobody picks are not read
    pairs = c["rows"] * c["picks"] * c["owned"] / c["experts"]
    hit = c["owned"] * (1 - (1 - c["picks"] / c["experts"]) ** c["rows"])
    read = (c["rows"] if c["form"] == "up" else pairs) * (k + 4 * _blocks(k))
    return {"bytes": read + pairs * n * _size(c["out"]) + hit * (n * k + 4 * _blocks(n) * _blocks(k)), "flops": 2 * pairs * n * k}


# ---------------------------------------------------------------------------------------------------------------- inputs
class _Seeded:
    def __init__(self, seed):
        self.g = torch.Generator(device=DEV).manual_seed(seed)

    def randn(self, *shape, dtype=torch.float32):
        return torch.randn(*shape, device=DEV, generator=self.g, dtype=dtype)

    def rand(self, *shape):
        return torch.rand(*shape, device=DEV, generator=self.g)

    def bytes(self, *shape):
        """E4M3 values as blocks scaled to their largest magnitude have them: some tens, up to 448."""
        return (110.0 * self.randn(*shape, dtype=torch.bfloat16)).clamp_(-448, 448).to(E4M3)


def prepare(case, seed):
    r = _Seeded(seed)
    return {"case": case, "kept": {}, **{"norm": _prepare_norm, "act": _prepare_act, "linear": _prepare_linear, "experts": _prepare_experts}[case["op"]](case, r)}


def _row_buffers(rows, d):
    return torch.zeros(rows, d, device=DEV, dtype=E4M3), torch.zeros(_blocks(d), rows, device=DEV)


def _prepare_norm(c, r):
    M, d, n = c["rows"], c["d"], c["terms"]
    # a residual stream has columns that stand far above the others
    h = r.randn(M, d) * (1.0 + 30.0 * (r.rand(d) > 0.998))
    s = {"h": h.to(TYPES[c["h"]]), "norm_w": (1.0 + 0.1 * r.randn(d)).bfloat16(), "x": None, "weights": None, "xn": torch.zeros(M, d, device=DEV, dtype=torch.bfloat16) if c["xn"] else None}
    if n:
        s["x"] = (0.3 * r.randn(M, n, d, dtype=torch.bfloat16)).to(TYPES[c["x"]])
        if n == 1:
            s["x"] = s["x"][:, 0]
        else:
            w = r.rand(M, n)
            s["weights"] = 2.5 * w / w.sum(1, keepdim=True)
    s["q"], s["s"] = _row_buffers(M, d)
    return s


def _prepare_act(c, r):
    x = (1.5 * r.randn(c["rows"], 2 * c["ffn"], dtype=torch.bfloat16)).to(TYPES[c["x"]])
    q, s = _row_buffers(c["rows"], c["ffn"])
    return {"x": x, "q": q, "s": s}


def _prepare_linear(c, r):
    M, k, n = c["rows"], c["k"], c["n"]
    return {"q": r.bytes(M, k), "s": (0.5 + 2.0 * r.rand(_blocks(k), M)) / 448, "w": r.bytes(n, k), "ws": (0.5 + r.rand(_blocks(n), _blocks(k))) * (4.0 / 448 / math.sqrt(k)),
            "bias": r.randn(n) if c["bias"] else None, "out": torch.zeros(M, n, device=DEV, dtype=TYPES[c["out"]]), "status": torch.zeros(8, dtype=torch.int32, device=DEV)}


def _prepare_experts(c, r):
    M, k, n, E = c["rows"], c["k"], c["n"], c["owned"]
    # every row picks different experts, some experts more often than others
    ids = torch.topk(r.rand(M, c["experts"]) + 0.3 * r.rand(c["experts"]), c["picks"], dim=1).indices
    pairs = ids.flatten()
    # as the framework's plan sorts them: held pairs by (expert, row, pick), positions of expert e are offs[e] .. offs[e + 1]
    key = torch.where(pairs < E, pairs, E)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=E + 1)[:E]
    offs = torch.cat([counts.new_zeros(1), counts.cumsum(0)])
    held = int(offs[-1])
    pair_of_pos = torch.where(torch.arange(M * c["picks"], device=DEV) < held, order, -1).int()
    s = {"w": r.bytes(E, n, k), "ws": (0.5 + r.rand(E, _blocks(n), _blocks(k))) * (4.0 / 448 / math.sqrt(k)), "offs": offs.int(), "pair_of_pos": pair_of_pos,
         "held": held, "most": int(counts.max()), "out": torch.zeros(M * c["picks"], n, device=DEV, dtype=TYPES[c["out"]]), "status": torch.zeros(8, dtype=torch.int32, device=DEV)}
    rows = M if c["form"] == "up" else M * c["picks"]
    s["q"], s["s"] = r.bytes(rows, k), (0.5 + 2.0 * r.rand(_blocks(k), rows)) / 448
    return s


# ---------------------------------------------------------------------------------------------------------------- one pass
def run(s):
    op = s["case"]["op"]
    if own:
        return {"norm": _own_norm, "act": _own_act, "linear": _own_linear, "experts": _own_experts}[op](s)
    return {"norm": _plain_norm, "act": _plain_act, "linear": _plain_linear, "experts": _plain_experts}[op](s)


def _norm_out(s, q, sc, xn):
    out = {"q": q, "s": sc}
    if s["x"] is not None:
        out["h"] = s["h"]
    if s["xn"] is not None:
        out["xn"] = xn
    return out


def _own_norm(s):
    from rexl3_b200.ops import kernels as K
    K.add_norm_fp8(s["x"], s["h"], s["norm_w"], 1e-6, s["q"], s["s"], weights=s["weights"], xn=s["xn"])
    return _norm_out(s, s["q"], s["s"], s["xn"])


def _to_blocks(y):
    """float32 rows as E4M3 with a scale for each 128 columns: [rows, d], [blocks, rows]"""
    M, d = y.shape
    nb = _blocks(d)
    b = torch.nn.functional.pad(y, (0, nb * BLOCK - d)).view(M, nb, BLOCK)
    sc = b.abs().amax(2).clamp_min(TINY) / 448.0
    q = (b / sc[:, :, None]).clamp_(-448, 448).to(E4M3)
    return q.view(M, nb * BLOCK)[:, :d].contiguous(), sc.t().contiguous()


def _plain_norm(s):
    y = s["h"].float()
    if s["weights"] is not None:
        y = y + (s["x"].float() * s["weights"][:, :, None]).sum(1)
    elif s["x"] is not None:
        y = y + s["x"].float()
    if s["x"] is not None:
        s["h"].copy_(y)
    y = y * torch.rsqrt((y * y).mean(1, keepdim=True) + 1e-6) * s["norm_w"].float()
    return _norm_out(s, *_to_blocks(y), y.bfloat16() if s["xn"] is not None else None)


def _own_act(s):
    from rexl3_b200.ops import kernels as K
    K.swiglu_fp8(s["x"], s["q"], s["s"])
    return {"q": s["q"], "s": s["s"]}


def _plain_act(s):
    F = s["case"]["ffn"]
    g, u = s["x"][:, :F].float(), s["x"][:, F:].float()
    q, sc = _to_blocks(g / (1.0 + torch.exp(-g)) * u)
    return {"q": q, "s": sc}


def _own_linear(s):
    from rexl3_b200.ops import kernels as K
    if not s["kept"]:                                                # the weight, as a model keeps it
        s["kept"]["w"] = K.Fp8BlockWeight(s["w"], s["ws"], s["bias"])
    K.fp8_block_linear(s["q"], s["s"], s["kept"]["w"], s["out"], s["status"])
    return s["out"]


def _wide(w, sc):
    """the float32 values of E4M3 [..., rows, k] under scales [..., rows or blocks of rows, blocks of k]"""
    n, k = w.shape[-2:]
    if sc.shape[-2] != n:
        sc = sc.repeat_interleave(BLOCK, -2)[..., :n, :]
    return w.float() * sc.repeat_interleave(BLOCK, -1)[..., :k]


def _plain_linear(s):
    y = torch.matmul(_wide(s["q"], s["s"].t()), _wide(s["w"], s["ws"]).t())
    return (y if s["bias"] is None else y + s["bias"]).to(s["out"].dtype)


def _own_experts(s):
    from rexl3_b200.ops import kernels as K
    if not s["kept"]:
        s["kept"]["w"] = K.Fp8BlockWeight(s["w"], s["ws"])
    if s["case"]["form"] == "up":
        K.fp8_block_experts(s["q"], s["s"], s["kept"]["w"], s["offs"], s["out"], s["status"], src=s["pair_of_pos"], src_div=s["case"]["picks"])
    else:
        K.fp8_block_experts(s["q"], s["s"], s["kept"]["w"], s["offs"], s["out"], s["status"], dst=s["pair_of_pos"])
    return s["out"]


def _plain_experts(s):
    c = s["case"]
    pos = torch.arange(s["held"], device=DEV)
    pair = s["pair_of_pos"][:s["held"]].long()
    e = torch.searchsorted(s["offs"].long(), pos, right=True) - 1
    at = pos - s["offs"].long()[e]
    rows = _wide(s["q"], s["s"].t())
    x = torch.zeros(c["owned"], s["most"], c["k"], device=DEV)       # an expert's rows side by side
    x[e, at] = rows[pair // c["picks"] if c["form"] == "up" else pos]
    y = torch.bmm(x, _wide(s["w"], s["ws"]).transpose(1, 2))[e, at]
    s["out"][pos if c["form"] == "up" else pair] = y.to(s["out"].dtype)
    return s["out"]


# ---------------------------------------------------------------------------------------------------------------- from the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] in ("norm", "act"):
        return (_exact_norm if case["op"] == "norm" else _exact_act)(case, s)
    return (_exact_linear if case["op"] == "linear" else _exact_experts)(case, s)


def _exact_blocks(y):
    """What stands in the bytes before they are rounded, and the scales."""
    q, scales = [], []
    for b in torch.split(y, BLOCK, dim=1):
        sc = torch.clamp(torch.amax(torch.abs(b), dim=1), min=TINY) / 448.0
        scales.append(sc)
        q.append(b / sc.unsqueeze(1))
    return torch.cat(q, dim=1), torch.stack(scales)


def _exact_norm(case, s):
    h = s["h"].double()
    for t in range(case["terms"]):
        if case["terms"] == 1:
            h = h + s["x"].double()
        else:
            h = h + s["x"][:, t].double() * s["weights"][:, t:t + 1].double()
    y = h / torch.sqrt(torch.mean(h ** 2, dim=1, keepdim=True) + 1e-6) * s["norm_w"].double()
    q, sc = _exact_blocks(y)
    out = {"q": q, "s": sc}
    if case["terms"]:
        out["h"] = h
    if case["xn"]:
        out["xn"] = y
    return out


def _exact_act(case, s):
    gate, up = torch.split(s["x"].double(), case["ffn"], dim=1)
    q, sc = _exact_blocks(gate * torch.sigmoid(gate) * up)
    return {"q": q, "s": sc}


def _exact_product(q, sc, w, ws):
    """sum over blocks of k of (the block's product) * (its row's scale) * (its columns' scales)"""
    out = torch.zeros(q.shape[0], w.shape[0], dtype=torch.float64, device=DEV)
    for b in range(sc.shape[0]):
        k = slice(b * BLOCK, (b + 1) * BLOCK)
        cols = ws[:, b].double()[torch.arange(w.shape[0], device=DEV) // BLOCK]
        out.addcmul_(q[:, k].double() @ w[:, k].double().T, torch.outer(sc[b].double(), cols))
    return out


def _exact_linear(case, s):
    y = _exact_product(s["q"], s["s"], s["w"], s["ws"])
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_experts(case, s):
    out, offs, pairs = torch.zeros(case["rows"] * case["picks"], case["n"], dtype=torch.float64, device=DEV), s["offs"].tolist(), s["pair_of_pos"].long()
    for e in range(case["owned"]):
        at = torch.arange(offs[e], offs[e + 1], device=DEV)
        if at.numel():
            src = pairs[at] // case["picks"] if case["form"] == "up" else at
            out[at if case["form"] == "up" else pairs[at]] = _exact_product(s["q"][src], s["s"][:, src], s["w"][e], s["ws"][e])
    return out

"""E4M3 caches: one key that outweighs each of thousands of others by 2^25, which together still count.  Probabilities are fp16 operands there; the row's sum has them all.

Tolerance.  An output is off by 2^-8 of itself (bf16), a probability by 2^-11 of itself or, where fp16 runs out of exponents, by half its last place: operands are the
probabilities times 2^7, so 2^-25 / 2^7 = 2^-32 of the row's largest, n of them at most n 2^-32 max |v|; the sum over n keys in fp32 adds at most n / 64 roundings of 2^-24,
the scores (25 log2 units) and ex2 2^-19 relative: together 1.05 * (2^-8 + 2^-11) mean |v| + n 2^-32 max |v|."""
import math

import pytest
import torch

from rexl3_b200.ops import kernels as K


def one_key_and_a_tail(rows, pages, below, hd, n_q):
    """-> q, k, v (E4M3 bytes), scales, table, exact row: key 0 has the score `below` log2 units above every other; half of the outputs are of the tail alone."""
    k = torch.zeros(pages, 1, 64, hd, dtype=torch.float8_e4m3fn, device="cuda")
    k[0, 0, 0] = 1.5
    v = torch.ones(pages, 1, 64, hd, device="cuda")
    v[0, 0, 0, : hd // 2] = 0.0
    v[0, 0, 0, hd // 2:] = -0.5
    scales = torch.tensor([[below * math.log(2) / (1.5 * math.sqrt(hd))], [1.0]], device="cuda")
    q = torch.ones(rows, n_q * hd, dtype=torch.bfloat16, device="cuda")
    s = (q[0, :hd].double() * (k.double() * scales[0].double()).transpose(1, 2).reshape(-1, hd)).sum(1) / math.sqrt(hd)
    p = torch.softmax(s, 0)
    vv = v.double().transpose(1, 2).reshape(-1, hd)
    table = torch.arange(pages, dtype=torch.int32, device="cuda").expand(rows, pages).contiguous()
    return q, k.view(torch.uint8), v.to(torch.float8_e4m3fn).view(torch.uint8), scales, table, p @ vv, p @ vv.abs()


@pytest.mark.gpu
@pytest.mark.parametrize("hd,n_q", [(128, 1), (64, 2)])
@pytest.mark.parametrize("below", [20.0, 23.9, 25.3, 26.5, 28.0])
def test_a_long_flat_tail_counts(below, hd, n_q):
    rows, pages = 296, 511                                               # a row's pages are one CTA's or two's: they share its running maximum
    q, k, v, scales, table, want, mean = one_key_and_a_tail(rows, pages, below, hd, n_q)
    out, st, n = torch.empty_like(q), K.new_status(), pages * 64
    seq, ctx, none = (torch.arange(rows, dtype=torch.int32, device="cuda"), torch.full((rows,), n, dtype=torch.int32, device="cuda"),
                      torch.zeros(rows, dtype=torch.int32, device="cuda"))
    K.attn_shared(K.KvTensorMap(k), K.KvTensorMap(v), q, table, seq, ctx, none, K.attn_shared_scratch(rows, n_q, 1, hd), n_q, 1, hd, 1 / math.sqrt(hd), out, st,
                  kv_scale=scales)
    K.check_status(st)
    off = (out.double().view(rows, n_q, hd) - want).abs() - (1.05 * (2.0 ** -8 + 2.0 ** -11) * mean + n * 2.0 ** -32)
    assert float(off.max()) <= 0, f"off by {float(off.max()):.3g} more than the bound, of outputs of {float(want[0]):.3g}"

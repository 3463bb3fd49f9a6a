"""Calls on several streams at once, each with a workspace of its own: the bits of the same calls one after the other."""
import math

import pytest
import torch

from rexl3_b200.ops import kernels as K
from test_gpu_attn_shared import Window
from test_gpu_topk_adjusted import rules


@pytest.mark.gpu
def test_attention_on_three_streams():
    windows = [Window([(0, 900 + 31 * i, 1) for i in range(24)], 10, 16, 4, 64, seed=1), Window([(0, 900 + 31 * i, 1) for i in range(24)], 10, 40, 8, 128, fp8=True, seed=2),
               Window([(i // 8, 1500 + 13 * i, 5) for i in range(16)], 20, 32, 4, 128, seed=3)]
    want = [w.run() for w in windows]
    streams = [torch.cuda.Stream() for _ in windows]
    scratch = [K.attn_shared_scratch(w.q.shape[0], w.n_q, w.n_kv, w.hd) for w in windows]
    outs, status = [[torch.empty_like(x) for _ in range(40)] for x in want], [K.new_status() for _ in windows]
    torch.cuda.synchronize()
    for turn in range(40):
        for w, s, sc, out, st in zip(windows, streams, scratch, outs, status):
            with torch.cuda.stream(s):
                K.attn_shared(*w.maps, w.q, w.table, w.row_seq, w.ctx, w.common, sc, w.n_q, w.n_kv, w.hd, 1 / math.sqrt(w.hd), out[turn], st, kv_scale=w.scale_kv)
    torch.cuda.synchronize()
    for x, out, st in zip(want, outs, status):
        K.check_status(st)
        assert all(torch.equal(o, x) for o in out)


@pytest.mark.gpu
def test_candidates_on_three_streams():
    calls = []
    for rows, V, count in ((1, 151936, 28), (20, 32003, 64), (40, 2048, 5)):
        kw = rules(rows, V, 4, rows + V)
        x, sc = torch.randn(rows, V, device="cuda"), K.topk_scratch(rows, V, count)
        made = [(torch.empty(rows, count, dtype=torch.int32, device="cuda"), torch.empty(rows, count, device="cuda")) for _ in range(41)]
        calls.append((x, count, sc, made, kw, torch.cuda.Stream()))
        K.topk_adjusted(x, count, sc, *made[40], **kw)
    torch.cuda.synchronize()
    for turn in range(40):
        for x, count, sc, made, kw, s in calls:
            with torch.cuda.stream(s):
                K.topk_adjusted(x, count, sc, *made[turn], **kw)
    torch.cuda.synchronize()
    for *_, made, _, _ in calls:
        assert all(torch.equal(a, made[40][0]) and torch.equal(b, made[40][1]) for a, b in made)

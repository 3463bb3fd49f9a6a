"""Products of E4M3 rows and weights under scales for blocks of 128, dense and through routed experts, against the formula in 64 bits."""
import gc
import os
import subprocess
import sys

import pytest
import torch

from rexl3_b200.engine.gpu_backend import capturing
from rexl3_b200.ops import kernels as K
from rexl3_b200.ops import lib as L

pytestmark = pytest.mark.gpu
E4M3, BF16, F16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def rows_of(M, Kd, g):
    q = (110 * torch.randn(M, Kd, device="cuda", generator=g)).clamp(-448, 448).to(E4M3)
    return q, (0.5 + torch.rand((Kd + 127) // 128, M, device="cuda", generator=g)) / 448


def weight_of(Kd, N, g, experts=None, bias=False):
    lead = () if experts is None else (experts,)
    w = (110 * torch.randn(*lead, N, Kd, device="cuda", generator=g)).clamp(-448, 448).to(E4M3)
    s = (0.5 + torch.rand(*lead, (N + 127) // 128, (Kd + 127) // 128, device="cuda", generator=g)) * 2.0 ** -6
    return K.Fp8BlockWeight(w, s, torch.randn(N, device="cuda", generator=g) if bias else None)


def values(q, s):
    return q.view(E4M3).double() * s.t().double().repeat_interleave(128, 1)[:, :q.shape[1]]


def dense64(w):
    s = w.scales.double().repeat_interleave(128, -2)[..., :w.N, :].repeat_interleave(128, -1)[..., :w.K]
    return w.w.view(E4M3).double() * s


def near(out, want, size, K_, dtype):
    """Each addition in float32 is off by at most a step (the tensor cores need not round to nearest) of a partial sum, which is at most `size`, the sum of the
    magnitudes: 128 in a block, one a block, eight parts of k, the bias; the product of the two scales and its use.  Then out is rounded."""
    steps = 128 + (K_ + 127) // 128 + 8 + 4
    off = (out.double() - want).abs()
    assert bool((off <= size * steps * 2.0 ** -23 + want.abs() * torch.finfo(dtype).eps / 2 + (2.0 ** -25 if dtype == F16 else 0)).all()), float((off / size).max())


def check_linear(M, Kd, N, dtype=F32, bias=False, seed=0, spare=0):
    g = gen(seed + M + Kd + N)
    q, s = rows_of(M, Kd, g)
    w = weight_of(Kd, N, g, bias=bias)
    if spare:                                                         # rows and blocks further apart, with NaN between
        qq, ss = torch.full((M, Kd + 16 * spare), 0x7F, dtype=torch.uint8, device="cuda"), torch.full((s.shape[0], M + spare), float("nan"), device="cuda")
        qq[:, :Kd], ss[:, :M] = q.view(torch.uint8), s
        q, s = qq[:, :Kd], ss[:, :M]
    room, status = torch.full((M + 1, N + spare), 7.0, device="cuda", dtype=dtype), K.new_status()
    out = room[:M, :N]
    K.fp8_block_linear(q, s, w, out, status)
    torch.cuda.synchronize()
    K.check_status(status)
    assert bool((room[M] == 7).all()) and bool((room[:, N:] == 7).all())
    x, m = values(q.contiguous(), s.contiguous()), dense64(w)
    b = 0 if w.bias is None else w.bias.double()
    near(out, x @ m.T + b, x.abs() @ m.abs().T + abs(b), Kd, dtype)
    return q, s, w, out


@pytest.mark.parametrize("M", [1, 2, 15, 16, 17, 32, 33, 64, 65, 128, 129, 300, 513])
@pytest.mark.parametrize("Kd,N", [(16, 1), (128, 128), (144, 130), (688, 256), (1024, 385)])
def test_linear(M, Kd, N):
    check_linear(M, Kd, N, bias=M % 2 == 1, spare=M % 3)


@pytest.mark.parametrize("M,Kd,N", [(1, 5120, 7168), (3, 17408, 640), (16, 18432, 256), (80, 5120, 5120), (333, 7168, 2112), (1000, 2048, 1000), (2048, 512, 2304), (700, 1376, 4000)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_linear_of_models_sizes(M, Kd, N, dtype):
    check_linear(M, Kd, N, dtype, bias=True)


@pytest.mark.parametrize("M,Kd,N", [(300, 1024, 517), (2000, 256, 1031), (700, 2048, 255), (1500, 128, 300)])
@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_rows_of_out_that_begin_anywhere(M, Kd, N, dtype):
    """Columns of a larger tensor from any of 9 on, of odd and even row lengths: what stands beside them stays."""
    g = gen(M)
    q, s = rows_of(M, Kd, g)
    w, status = weight_of(Kd, N, g, bias=True), K.new_status()
    x, m = values(q, s), dense64(w)
    want, size = x @ m.T + w.bias.double(), x.abs() @ m.abs().T + w.bias.double().abs()
    for at, spare in ((0, 0), (1, 0), (2, 1), (3, 0), (4, 3), (5, 2), (6, 0), (7, 1), (8, 5)):
        room = torch.full((M, N + at + spare), 7.0, device="cuda", dtype=dtype)
        K.fp8_block_linear(q, s, w, room[:, at:at + N], status)
        K.check_status(status)
        assert bool((room[:, :at] == 7).all()) and bool((room[:, at + N:] == 7).all())
        near(room[:, at:at + N], want, size, Kd, dtype)


@pytest.mark.parametrize("M,Kd,N", [(1, 2048, 256), (40, 688, 300), (200, 4096, 256), (900, 1024, 1024)])
def test_calls_repeat_to_the_bit(M, Kd, N):
    q, s, w, out = check_linear(M, Kd, N)
    status = K.new_status()
    for _ in range(20):
        again = torch.zeros(M, N, device="cuda")
        K.fp8_block_linear(q, s, w, again, status)
        assert torch.equal(again, out)
    K.check_status(status)


@pytest.mark.parametrize("M", [1, 20, 100, 300, 600])
def test_whole_numbers_are_exact(M):
    """Small whole numbers under scales of 1: every sum is exact in float32, so a wrong byte anywhere shows, on every one of many launches."""
    g = gen(M)
    Kd, N = 4096, 384
    q = torch.randint(-3, 4, (M, Kd), device="cuda", generator=g).to(BF16).to(E4M3)
    w = K.Fp8BlockWeight(torch.randint(-3, 4, (N, Kd), device="cuda", generator=g).to(BF16).to(E4M3), torch.ones(3, 32, device="cuda"))
    s, status, out = torch.ones(32, M, device="cuda"), K.new_status(), torch.zeros(30, M, N, device="cuda")
    for i in range(30):
        K.fp8_block_linear(q, s, w, out[i], status)
    K.check_status(status)
    assert torch.equal(out, (q.double() @ w.w.double().T).float().expand_as(out))


@pytest.mark.parametrize("M", [3, 70, 400])
def test_bad_values_stay_in_their_row_and_column(M):
    g = gen(5)
    q, s = rows_of(M, 400, g)
    w = weight_of(400, 300, g)
    clean, status = torch.zeros(M, 300, device="cuda"), K.new_status()
    K.fp8_block_linear(q, s, w, clean, status)
    q.view(torch.uint8)[1, 250], w.w.view(torch.uint8)[200, 3] = 0x7F, 0xFF                  # the two NaN bytes
    s[0, 2], w.scales[0, 1] = float("inf"), 0.0
    out = torch.zeros(M, 300, device="cuda")
    K.fp8_block_linear(q, s, w, out, status)
    torch.cuda.synchronize()
    K.check_status(status)
    assert bool(torch.isnan(out[1]).all()) and bool(torch.isnan(out[:, 200]).all()) and not bool(torch.isfinite(out[2]).any())
    keep = torch.ones(M, dtype=torch.bool, device="cuda")
    keep[1:3] = False
    cols = torch.arange(128, 300, device="cuda")
    cols = cols[cols != 200]                                          # (the first strip's second block is scaled by 0)
    assert torch.equal(out[keep][:, cols], clean[keep][:, cols]) and bool(torch.isfinite(out[keep][:, :128]).all())


def test_no_rows():
    w, status = weight_of(128, 128, gen(0)), K.new_status()
    K.fp8_block_linear(*K.fp8_rows(0, 128), w, torch.zeros(0, 128, device="cuda"), status)
    we = weight_of(128, 128, gen(0), experts=2)
    offs = torch.zeros(3, dtype=torch.int32, device="cuda")
    K.fp8_block_experts(*K.fp8_rows(0, 128), we, offs, torch.zeros(4, 128, device="cuda"), status)
    K.fp8_block_experts(*K.fp8_rows(4, 128), we, offs, torch.zeros(0, 128, device="cuda"), status, src=offs[:0])
    torch.cuda.synchronize()
    K.check_status(status)


# ------------------------------------------------------------------------------------------------ routed experts
def plan(rows, picks, experts, held, g, skew=0.3):
    """As the framework's plan sorts them: held pairs by (expert, row, pick)."""
    ids = torch.topk(torch.rand(rows, experts, device="cuda", generator=g) + skew * torch.rand(experts, device="cuda", generator=g), picks, dim=1).indices
    key = torch.where(ids.flatten() < held, ids.flatten(), held)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=held + 1)[:held]
    offs = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).int()
    pairs = torch.where(torch.arange(rows * picks, device="cuda") < offs[-1], order, -1).int()
    return ids.int(), offs, pairs


def check_experts(q, s, w, offs, out, before, src=None, div=1, dst=None):
    """Every position's row against its expert's matrix; the other rows of out as they were."""
    x, want, size = values(q, s), before.double().clone(), torch.zeros_like(before, dtype=torch.float64)
    o = offs.tolist()
    for e in range(w.experts):
        p = torch.arange(o[e], o[e + 1], device="cuda")
        if p.numel():
            m = (w.w[e].view(E4M3).double() * w.scales[e].double().repeat_interleave(128, 0)[:w.N].repeat_interleave(128, 1)[:, :w.K]).T
            xr = x[p if src is None else src[p].long() // div]
            to = p if dst is None else dst[p].long()
            want[to], size[to] = xr @ m, xr.abs() @ m.abs()
    written = size.sum(1) > 0
    assert torch.equal(out[~written], before[~written])
    near(out[written], want[written], size[written], w.K, out.dtype)


@pytest.mark.parametrize("rows,picks,experts,held", [(1, 1, 1, 1), (2000, 2, 600, 600), (90, 8, 20, 20), (1, 2, 8, 8), (16, 8, 128, 128), (5, 3, 300, 300), (40, 2, 6, 4), (130, 4, 16, 3), (333, 2, 5, 5), (700, 2, 3, 2), (64, 8, 40, 1)])
@pytest.mark.parametrize("Kd,N", [(128, 128), (688, 300), (272, 17), (1024, 256)])
def test_experts_up_and_down(rows, picks, experts, held, Kd, N):
    g = gen(rows + experts + Kd)
    _, offs, pairs = plan(rows, picks, experts, held, g)
    w, status = weight_of(Kd, N, g, experts=held), K.new_status()
    for dtype in (F32, BF16):
        q, s = rows_of(rows, Kd, g)
        before = torch.full((rows * picks, N), 7.0, device="cuda", dtype=dtype)
        out = before.clone()
        K.fp8_block_experts(q, s, w, offs, out, status, src=pairs, src_div=picks)
        check_experts(q, s, w, offs, out, before, src=pairs, div=picks)
        q, s = rows_of(rows * picks, Kd, g)
        out = before.clone()
        K.fp8_block_experts(q, s, w, offs, out, status, dst=pairs)
        check_experts(q, s, w, offs, out, before, dst=pairs)
        out = before.clone()
        K.fp8_block_experts(q, s, w, offs, out, status)
        check_experts(q, s, w, offs, out, before)
    torch.cuda.synchronize()
    K.check_status(status)


def test_experts_with_offsets_from_the_middle_and_none():
    g = gen(3)
    w, status = weight_of(256, 200, g, experts=4), K.new_status()
    q, s = rows_of(60, 256, g)
    for o in ([0, 0, 0, 0, 0], [7, 7, 30, 30, 59], [0, 0, 0, 0, 60], [60, 60, 60, 60, 60], [0, 1, 2, 3, 4]):
        offs = torch.tensor(o, dtype=torch.int32, device="cuda")
        before = torch.full((60, 200), 7.0, device="cuda")
        out = before.clone()
        K.fp8_block_experts(q, s, w, offs, out, status)
        check_experts(q, s, w, offs, out, before)
    K.check_status(status)


@pytest.mark.parametrize("o", [[0, 5, 3, 8, 8], [-1, 2, 4, 6, 8], [0, 2, 4, 6, 61], [0, 2, 4, 6, 2147483647], [0, -2147483648, 4, 6, 8]])
def test_bad_offsets_set_the_status(o):
    g = gen(4)
    w, status = weight_of(128, 130, g, experts=4), K.new_status()
    q, s = rows_of(60, 128, g)
    room = torch.full((62, 130), 7.0, device="cuda")
    K.fp8_block_experts(q, s, w, torch.tensor(o, dtype=torch.int32, device="cuda"), room[1:61], status)
    torch.cuda.synchronize()
    assert int(status[0]) == K.ST_BAD_ARG and bool((room[[0, 61]] == 7).all())


def test_rows_outside_set_the_status():
    g = gen(5)
    w, status = weight_of(128, 130, g, experts=2), K.new_status()
    q, s = rows_of(6, 128, g)
    offs = torch.tensor([0, 3, 6], dtype=torch.int32, device="cuda")
    good = torch.zeros(6, 130, device="cuda")
    K.fp8_block_experts(q, s, w, offs, good, status)
    K.check_status(status)
    out = torch.full((6, 130), 7.0, device="cuda")
    K.fp8_block_experts(q, s, w, offs, out, status, src=torch.tensor([0, -1, 2, 3, 6, 5], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert int(status[0]) == K.ST_BAD_ARG and bool((out[[1, 4]] == 0).all()) and torch.equal(out[[0, 2, 3, 5]], good[[0, 2, 3, 5]])
    status.zero_()
    out = torch.full((6, 130), 7.0, device="cuda")
    K.fp8_block_experts(q, s, w, offs, out, status, dst=torch.tensor([0, -1, 2, 3, 6, 5], dtype=torch.int32, device="cuda"))
    torch.cuda.synchronize()
    assert int(status[0]) == K.ST_BAD_ARG and bool((out[[1, 4]] == 7).all()) and torch.equal(out[[0, 2, 3, 5]], good[[0, 2, 3, 5]])


# ------------------------------------------------------------------------------------------------ together
def test_a_feed_forward_block():
    """norm -> gate | up -> SwiGLU -> down -> the next norm, each stage against its formula on what the stage before has written."""
    g = gen(7)
    M, d, F = 37, 512, 688
    h, x = torch.randn(M, d, device="cuda", generator=g).to(BF16), torch.randn(M, d, device="cuda", generator=g).to(BF16)
    nw = torch.ones(d, device="cuda", dtype=BF16)
    gu, dn, status = weight_of(d, 2 * F, g), weight_of(F, d, g), K.new_status()
    h0 = h.clone()
    (q, s), (q2, s2), (q3, s3) = K.fp8_rows(M, d), K.fp8_rows(M, F), K.fp8_rows(M, d)
    y, z = torch.zeros(M, 2 * F, device="cuda", dtype=BF16), torch.zeros(M, d, device="cuda", dtype=BF16)

    def block():
        K.add_norm_fp8(x, h, nw, 1e-6, q, s)
        K.fp8_block_linear(q, s, gu, y, status)
        K.swiglu_fp8(y, q2, s2)
        K.fp8_block_linear(q2, s2, dn, z, status)
        K.add_norm_fp8(z, h, nw, 1e-6, q3, s3)
    block()
    torch.cuda.synchronize()
    K.check_status(status)
    h1 = (h0.float() + x.float()).to(BF16)
    v = h0.double() + x.double()
    n = v / torch.sqrt((v * v).mean(1, keepdim=True) + 1e-6)
    # half a step of a byte, 2^-4 of the value or 2^-10 of the scale, and float32's roundings
    assert bool(((values(q, s) - n).abs() <= torch.maximum(n.abs() * 2.0 ** -4, s.t().double().repeat_interleave(128, 1) * 2.0 ** -10) * (1 + 2.0 ** -10)).all())
    near(y, values(q, s) @ dense64(gu).T, values(q, s).abs() @ dense64(gu).abs().T, d, BF16)
    a = y.double()[:, :F] * torch.sigmoid(y.double()[:, :F]) * y.double()[:, F:]
    assert bool(((values(q2, s2) - a).abs() <= torch.maximum(a.abs() * 2.0 ** -4, s2.t().double().repeat_interleave(128, 1)[:, :F] * 2.0 ** -10) * (1 + 2.0 ** -10)).all())
    near(z, values(q2, s2) @ dense64(dn).T, values(q2, s2).abs() @ dense64(dn).abs().T, F, BF16)
    assert torch.equal(h, (h1.float() + z.float()).to(BF16))
    # captured and replayed, beside eager calls on another stream with buffers of their own
    want = [t.clone() for t in (h, z, q3.view(torch.uint8), s3)]
    graph = torch.cuda.CUDAGraph()
    with capturing(graph):
        block()
    other, so = torch.zeros_like(z), K.new_status()
    stream = torch.cuda.Stream()
    for _ in range(3):
        h.copy_(h0)
        z.zero_()
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(stream):
            K.fp8_block_linear(q2, s2, dn, other, so)
        torch.cuda.synchronize()
        for t, u in zip((h, z, q3.view(torch.uint8), s3), want):
            assert torch.equal(t, u)
    K.check_status(status)
    K.check_status(so)


@pytest.mark.parametrize("rows,e_lo,e_hi", [(1, 0, 16), (21, 0, 16), (200, 4, 9)])
def test_a_routed_feed_forward_block(rows, e_lo, e_hi):
    """The framework's plan -> gate | up of the picking rows -> SwiGLU of the planned pairs -> down back to the pairs -> their weighted sum in the next norm."""
    g = gen(rows)
    d, F, E, picks, held = 256, 384, 16, 4, e_hi - e_lo
    ids = torch.topk(torch.rand(rows, E, device="cuda", generator=g), picks, dim=1).indices.int().contiguous()
    pw = torch.rand(rows, picks, device="cuda", generator=g)
    P = rows * picks
    i32 = lambda n: torch.full((n,), -5, dtype=torch.int32, device="cuda")  # noqa: E731
    offs, pos, pair, exp_of, tab, total = i32(E + 1), i32(P), i32(P), i32(P), i32(3 * 64), i32(1)
    L.check(L.load().rx_moe_plan(ids.data_ptr(), P, E, e_lo, e_hi, 16, 64, offs.data_ptr(), pos.data_ptr(), pair.data_ptr(), exp_of.data_ptr(), tab.data_ptr(), total.data_ptr(),
                                 L.stream_ptr()), "rx_moe_plan")
    gu, dn, status = weight_of(d, 2 * F, g, experts=held), weight_of(F, d, g, experts=held), K.new_status()
    h, nw = torch.randn(rows, d, device="cuda", generator=g), torch.ones(d, device="cuda", dtype=BF16)
    h0 = h.clone()
    (q, s), (q2, s2), (q3, s3) = K.fp8_rows(rows, d), K.fp8_rows(P, F), K.fp8_rows(rows, d)
    y, z = torch.zeros(P, 2 * F, device="cuda", dtype=BF16), torch.full((P, d), float("nan"), device="cuda")
    K.add_norm_fp8(None, h, nw, 1e-6, q, s)
    own = offs[e_lo:e_hi + 1]
    K.fp8_block_experts(q, s, gu, own, y, status, src=pair, src_div=picks)
    K.swiglu_fp8(y, q2, s2, total=total)
    K.fp8_block_experts(q2, s2, dn, own, z, status, dst=pair)
    here = (ids >= e_lo) & (ids < e_hi)
    weights = torch.where(here, pw, 0.0).contiguous()                 # what is computed elsewhere has the weight 0 here
    K.add_norm_fp8(z.view(rows, picks, d), h, nw, 1e-6, q3, s3, weights=weights)
    torch.cuda.synchronize()
    K.check_status(status)
    m = int(total[0])
    assert m == int(here.sum()) and bool(torch.isnan(z[~here.flatten()]).all())
    src = pair[:m].long()
    near(y[:m], torch.stack([values(q, s)[p // picks] @ dense64(gu)[e].T for p, e in zip(src.tolist(), (ids.flatten()[src] - e_lo).tolist())]),
         torch.stack([values(q, s)[p // picks].abs() @ dense64(gu)[e].abs().T for p, e in zip(src.tolist(), (ids.flatten()[src] - e_lo).tolist())]), d, BF16)
    x2 = values(q2[:m].contiguous(), s2[:, :m].contiguous())
    near(z[src], torch.stack([x2[i] @ dense64(dn)[e].T for i, e in enumerate((ids.flatten()[src] - e_lo).tolist())]),
         torch.stack([x2[i].abs() @ dense64(dn)[e].abs().T for i, e in enumerate((ids.flatten()[src] - e_lo).tolist())]), F, F32)
    terms = torch.where(weights[:, :, None] == 0, 0.0, z.view(rows, picks, d).double()) * weights.double()[:, :, None]
    assert bool(((h.double() - h0.double() - terms.sum(1)).abs() <= (h0.double().abs() + terms.abs().sum(1)) * (picks + 1) * 2.0 ** -24).all())


def test_calls_on_several_streams_at_once():
    g = gen(11)
    jobs = []
    for i, (M, Kd, N) in enumerate([(1, 4096, 1024), (64, 4096, 512), (300, 1024, 1024)]):
        q, s = rows_of(M, Kd, g)
        w, st = weight_of(Kd, N, g), K.new_status()
        want = torch.zeros(M, N, device="cuda")
        K.fp8_block_linear(q, s, w, want, st)
        jobs.append((q, s, w, st, want, torch.zeros(M, N, device="cuda"), torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for q, s, w, st, want, out, stream in jobs:
            with torch.cuda.stream(stream):
                K.fp8_block_linear(q, s, w, out, st)
    torch.cuda.synchronize()
    for q, s, w, st, want, out, stream in jobs:
        K.check_status(st)
        assert torch.equal(out, want)


def test_refusals():
    g = gen(1)
    q, s = rows_of(4, 256, g)
    w, we, out, st = weight_of(256, 128, g), weight_of(256, 128, g, experts=2), torch.zeros(4, 128, device="cuda"), K.new_status()
    ok = dict(q=q, s=s, w=w, out=out, status=st)
    K.fp8_block_linear(**ok)
    K.fp8_block_linear(**{**ok, "q": q.view(torch.uint8)})
    wide = torch.zeros(4, 512, device="cuda", dtype=E4M3)
    bad = (dict(q=q.float()), dict(q=q[:, :128]), dict(q=q.t()), dict(q=wide[:, 8:264]), dict(q=torch.zeros(4, 264, device="cuda", dtype=E4M3)[:, :256]), dict(s=s[:1]), dict(s=s.t()), dict(s=s[:, :3]),
           dict(s=s.half()), dict(out=out.double()), dict(out=out[:, :64]), dict(out=out.t()), dict(status=st[:4]), dict(status=st.float()), dict(w=w.w), dict(q=q[0]),
           dict(out=torch.zeros(512, device="cuda").as_strided((4, 128), (64, 1))))
    for b in (*bad, dict(w=we), dict(out=out[:3]), dict(s=s.cpu()), dict(out=out.cpu())):
        with pytest.raises(ValueError):
            K.fp8_block_linear(**{**ok, **b})
    offs, idx = torch.tensor([0, 2, 4], dtype=torch.int32, device="cuda"), torch.arange(4, dtype=torch.int32, device="cuda")
    ok = dict(q=q, s=s, w=we, offs=offs, out=out, status=st)
    K.fp8_block_experts(**ok)
    five = torch.zeros(5, dtype=torch.int32, device="cuda")
    for b in (*bad, dict(w=w), dict(offs=offs[:2]), dict(offs=offs.long()), dict(src=idx.long()), dict(src=idx, src_div=0), dict(src_div=2), dict(dst=five), dict(src=five), dict(src=five[:4], dst=five),
              dict(out=out[:3]), dict(src=idx[None]), dict(dst=idx.cpu())):
        with pytest.raises(ValueError):
            K.fp8_block_experts(**{**ok, **b})


# ------------------------------------------------------------------------------------------------ what else a call may meet
@pytest.mark.parametrize("first", [1, 2])
@pytest.mark.parametrize("rows,picks", [(8, 2), (5000, 2), (13000, 2)])
def test_as_many_experts_as_there_may_be(rows, picks, first):
    g = gen(rows)
    w, status = weight_of(16 * first, 16, g, experts=4096), K.new_status()
    q, s = rows_of(rows, 16 * first, g)
    ids = torch.randint(0, 4096, (rows * picks,), device="cuda", generator=g)
    pairs = torch.sort(ids, stable=True).indices.int()
    offs = torch.cat([ids.new_zeros(1), torch.bincount(ids, minlength=4096).cumsum(0)]).int()
    before = torch.full((rows * picks, 16), 7.0, device="cuda")
    out = before.clone()
    K.fp8_block_experts(q, s, w, offs, out, status, src=pairs, src_div=picks)
    K.check_status(status)
    check_experts(q, s, w, offs, out, before, src=pairs, div=picks)


@pytest.mark.parametrize("rows,picks", [(9, 2), (70, 3)])
def test_experts_with_rows_and_places_of_their_own(rows, picks):
    """src and dst in one call, rows of q and out and blocks of s further apart than they need be."""
    g = gen(rows)
    _, offs, pairs = plan(rows, picks, 4, 3, g)
    P = rows * picks
    w, status = weight_of(400, 264, g, experts=3), K.new_status()
    q, s = rows_of(rows, 400, g)
    qq, ss = torch.full((rows, 448), 0x7F, dtype=torch.uint8, device="cuda"), torch.full((4, rows + 5), float("nan"), device="cuda")
    qq[:, :400], ss[:, :rows] = q.view(torch.uint8), s
    dst = torch.randperm(P + 4, device="cuda", generator=g)[:P].int()
    for dtype in (BF16, F16, F32):
        room = torch.full((P + 4, 264 + 8), 7.0, device="cuda", dtype=dtype)
        K.fp8_block_experts(qq[:, :400], ss[:, :rows], w, offs, room[:, :264], status, src=pairs, src_div=picks, dst=dst)
        K.check_status(status)
        assert bool((room[:, 264:] == 7).all())
        check_experts(q, s, w, offs, room[:, :264], torch.full_like(room[:, :264], 7.0), src=pairs, div=picks, dst=dst)


@pytest.mark.parametrize("o", [[0, 1, 0], [0] * 300 + [1, 0], [0] * 200 + [1] * 200 + [0]])
def test_bad_offsets_behind_the_last_tile_set_the_status(o):
    """One position: as many tiles as a call of that size is cut for, and the fault stands behind them."""
    g = gen(6)
    w, status = weight_of(128, 128, g, experts=len(o) - 1), K.new_status()
    q, s = rows_of(1, 128, g)
    out = torch.zeros(1, 128, device="cuda")
    K.fp8_block_experts(q, s, w, torch.tensor(o, dtype=torch.int32, device="cuda"), out, status)
    torch.cuda.synchronize()
    assert int(status[0]) == K.ST_BAD_ARG


@pytest.mark.parametrize("rows", [4, 150])
def test_a_captured_call_follows_the_routing(rows):
    """The offsets and pairs are read when the graph runs: two graphs side by side, with new routing before every replay."""
    g = gen(rows)
    w, jobs = weight_of(256, 136, g, experts=8), []
    for _ in range(2):
        q, s = rows_of(rows, 256, g)
        _, offs, pairs = plan(rows, 3, 8, 8, g)
        out, status, graph, stream = torch.zeros(rows * 3, 136, device="cuda"), K.new_status(), torch.cuda.CUDAGraph(), torch.cuda.Stream()
        K.fp8_block_experts(q, s, w, offs, out, status, src=pairs, src_div=3)
        torch.cuda.synchronize()
        gc.collect()
        with torch.cuda.graph(graph, stream=stream):
            K.fp8_block_experts(q, s, w, offs, out, status, src=pairs, src_div=3)
        jobs.append((q, s, offs, pairs, out, status, graph, stream))
    for held in (8, 2, 5):
        for q, s, offs, pairs, out, status, graph, stream in jobs:
            _, o, p = plan(rows, 3, 8, held, g)
            offs.fill_(int(o[-1])), pairs.copy_(p), out.fill_(7.0)
            offs[:held + 1] = o
        torch.cuda.synchronize()
        for *_, graph, stream in jobs:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for q, s, offs, pairs, out, status, graph, stream in jobs:
            K.check_status(status)
            check_experts(q, s, w, offs, out, torch.full_like(out, 7.0), src=pairs, div=3)


def test_the_first_call_of_a_process_may_be_captured():
    code = """
import torch
from rexl3_b200.ops import kernels as K
q = torch.ones(M, 256, device="cuda").to(torch.float8_e4m3fn)
s, st, out = torch.ones(2, M, device="cuda"), K.new_status(), torch.zeros(M, 384, device="cuda")
w = K.Fp8BlockWeight(torch.ones(384, 256, device="cuda").to(torch.float8_e4m3fn), torch.ones(3, 2, device="cuda"))
we = K.Fp8BlockWeight(w.w[None], w.scales[None])
offs, oe = torch.tensor([0, M], dtype=torch.int32, device="cuda"), torch.zeros(M, 384, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    K.fp8_block_linear(q, s, w, out, st)
    K.fp8_block_experts(q, s, we, offs, oe, st)
g.replay()
torch.cuda.synchronize()
K.check_status(st)
assert bool((out == 256).all()) and bool((oe == 256).all())
"""
    for M in (3, 300):
        subprocess.run([sys.executable, "-c", f"M = {M}\n" + code], check=True, timeout=300, cwd=os.path.dirname(os.path.dirname(os.path.abspath(__file__))))


def gives_up(call, like):
    """`call(out, status)` under short limits and the abort word, with plain calls after each: it returns, says so if a wait gave up, and the next call is right."""
    want, st = torch.full_like(like, float("nan")), K.new_status()
    call(want, st)
    K.check_status(st)
    for us in ("abort", 1, 2, 5, 10, 20, 40, 100, "abort"):
        st = K.new_status()
        K.set_abort(st) if us == "abort" else K.set_wait_limit(st, us)
        got = torch.full_like(like, float("nan"))
        call(got, st)
        code = st.tolist()[0]
        assert code in (0, K.ST_ABORTED if us == "abort" else K.ST_TIMEOUT)
        assert code != 0 or torch.equal(got, want)
        for _ in range(2):
            st, got = K.new_status(), torch.full_like(like, float("nan"))
            call(got, st)
            K.check_status(st)
            assert torch.equal(got, want)


@pytest.mark.parametrize("M,Kd,N", [(1, 16384, 256), (24, 8192, 512), (64, 8192, 4096), (40, 2048, 20000), (333, 7168, 2112), (1000, 2048, 1000), (2404, 8192, 4096), (4000, 512, 8192)])
def test_waits_that_give_up(M, Kd, N):
    g = gen(M)
    q, s = rows_of(M, Kd, g)
    w = weight_of(Kd, N, g)
    gives_up(lambda out, st: K.fp8_block_linear(q, s, w, out, st), torch.zeros(M, N, device="cuda"))


@pytest.mark.parametrize("rows,picks,experts", [(16, 2, 32), (700, 4, 32)])
def test_experts_waits_that_give_up(rows, picks, experts):
    g = gen(rows)
    _, offs, pairs = plan(rows, picks, experts, experts, g)
    w = weight_of(2048, 512, g, experts=experts)
    q, s = rows_of(rows, 2048, g)
    gives_up(lambda out, st: K.fp8_block_experts(q, s, w, offs, out, st, src=pairs, src_div=picks), torch.zeros(rows * picks, 512, device="cuda"))
    q, s = rows_of(rows * picks, 2048, g)
    gives_up(lambda out, st: K.fp8_block_experts(q, s, w, offs, out, st, dst=pairs), torch.zeros(rows * picks, 512, device="cuda"))

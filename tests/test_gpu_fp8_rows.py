"""Residual norm and SwiGLU written as E4M3 rows with a scale for each 128 columns, against the formulas in 64 bits."""
import pytest
import torch

from rexl3_b200.engine.gpu_backend import capturing
from rexl3_b200.ops import kernels as K

pytestmark = pytest.mark.gpu
E4M3, BF16, F16, F32 = torch.float8_e4m3fn, torch.bfloat16, torch.float16, torch.float32
U = 2.0 ** -24                                                        # half a step of float32


def rand(*shape, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed))


def wide(t):
    return t.repeat_interleave(128, 1)


def check_rows(q, s, y, off):
    """q, s stand for y (float64 [rows, d]), which the kernel has with an error of up to `off` (float64 [rows, d])."""
    rows, d = y.shape
    pad = torch.nn.functional.pad
    nb = (d + 127) // 128
    amax, err = (pad(t, (0, nb * 128 - d)).view(rows, nb, 128).amax(2) for t in (y.abs(), off))
    want = amax.clamp_min(2.0 ** -100) / 448
    assert bool(((s.t().double() - want).abs() <= err / 448 + want * 2 * U).all())           # a division's rounding, and amax's
    v = y / wide(s.t().double())[:, :d]                                # what is rounded: half a step of E4M3 is 2^-4 of it, 2^-10 where the byte is subnormal
    step = torch.maximum(v.abs() * 2.0 ** -4, torch.full_like(v, 2.0 ** -10))
    got = q.view(E4M3).double()
    # the division 448 / amax, the product with it and the value's own error before the rounding; 448 is the largest byte, and the largest value may be above by them
    assert bool(((got - v).abs() <= step * (1 + 2.0 ** -20) + off / wide(s.t().double())[:, :d] + v.abs() * 4 * U).all())
    return got * wide(s.t().double())[:, :d]


def run_norm(x, h, norm_w, eps=1e-5, weights=None, xn=False, spare=0):
    """One call on rows that are `spare` values further apart than they are long; what stands between and behind is not touched."""
    rows, d = h.shape
    room = lambda t: None if t is None else torch.cat([t, torch.full((rows, spare), 7.0, device="cuda", dtype=t.dtype)], 1)  # noqa: E731
    hh = room(h)
    xx = x if weights is not None or x is None else room(x)[:, :d]
    q, s = torch.full((rows + 1, d + spare), 0x55, dtype=torch.uint8, device="cuda"), torch.full(((d + 127) // 128, rows + 3), 7.0, device="cuda")
    n = torch.full((rows, d + spare), 7.0, device="cuda", dtype=BF16) if xn else None
    K.add_norm_fp8(xx, hh[:, :d], norm_w, eps, q[:rows, :d], s[:, :rows], weights=weights, xn=None if n is None else n[:, :d])
    torch.cuda.synchronize()
    assert bool((q[rows] == 0x55).all()) and bool((q[:, d:] == 0x55).all()) and bool((s[:, rows:] == 7).all()) and bool((hh[:, d:] == 7).all())
    assert n is None or bool((n[:, d:] == 7).all())
    return q[:rows, :d].contiguous(), s[:, :rows].contiguous(), hh[:, :d].contiguous(), None if n is None else n[:, :d]


def check_norm(x, h, norm_w, eps=1e-5, weights=None, xn=False, spare=0):
    q, s, h2, n = run_norm(x, h, norm_w, eps, weights, xn, spare)
    d = h.shape[1]
    v, size, terms = h.double(), h.double().abs(), 0
    if weights is not None:
        read = torch.where((weights == 0)[:, :, None], 0.0, x.double())
        v, size, terms = v + (read * weights.double()[:, :, None]).sum(1), size + (read.abs() * weights.double().abs()[:, :, None]).sum(1), weights.shape[1]
    elif x is not None:
        v, size, terms = v + x.double(), size + x.double().abs(), 1
    off = size * terms * U                                             # a rounding an addition
    if x is None:
        assert torch.equal(h2, h)
    else:
        assert bool(((h2.double() - v).abs() <= v.abs() * torch.finfo(h.dtype).eps / 2 * (1 + 2.0 ** -10) + off).all())
        if weights is None:
            assert torch.equal(h2, (h.float() + x.float()).to(h.dtype))
    y = v
    if norm_w is not None:
        r = 1 / torch.sqrt((v ** 2).mean(1, keepdim=True) + eps)
        y = v * r * norm_w.double()
        # the sum of squares: up to 32 in a thread, then 5 + 5 halvings, each of a square or a sum of squares, half of it in the root; rsqrtf 2 steps, the mean, two products
        rel = (32 + 10 + 2) * U / 2 + 4 * U + 4 * U
        carried = (2 * off * v.abs()).mean(1, keepdim=True) / ((v ** 2).mean(1, keepdim=True) + eps) / 2
        off = (off * r + v.abs() * r * (rel + carried)) * norm_w.double().abs()
    check_rows(q, s, y, off)
    if xn:
        assert bool(((n.double() - y).abs() <= y.abs() * 2.0 ** -8 + off * 1.01 + 1e-38).all())


@pytest.mark.parametrize("rows,d", [(1, 16), (2, 128), (3, 144), (5, 688), (1, 5120), (33, 2048), (300, 256), (7, 7168), (2, 8192), (2, 8208), (3, 16384), (1, 32768)])
@pytest.mark.parametrize("xt,ht", [(BF16, BF16), (F16, F32), (F32, BF16), (BF16, F32)])
def test_add_norm(rows, d, xt, ht):
    x, h = (0.5 * rand(rows, d, seed=1)).to(xt), rand(rows, d, seed=2) * (1 + 40 * (rand(d, seed=3) > 2.5))
    w = (1 + 0.2 * rand(d, seed=4)).to(BF16)
    check_norm(x, h.to(ht), w, xn=rows % 2 == 1, spare=16 * (rows % 3))


@pytest.mark.parametrize("rows,d,terms", [(1, 128, 1), (4, 2048, 8), (9, 688, 3), (2, 7168, 8), (3, 10000, 2), (2, 144, 17)])
@pytest.mark.parametrize("xt,ht", [(BF16, BF16), (F32, F32), (F16, BF16)])
def test_add_norm_of_weighted_experts(rows, d, terms, xt, ht):
    x = rand(rows, terms, d, seed=1).to(xt)
    weights = rand(rows, terms, seed=5).abs()
    weights[0, terms // 2] = 0.0
    x[0, terms // 2] = float("nan")                                   # an output of weight 0 is not read
    check_norm(x, rand(rows, d, seed=2).to(ht), (1 + 0.2 * rand(d, seed=4)).to(BF16), weights=weights, xn=True)


@pytest.mark.parametrize("ht", [BF16, F32])
@pytest.mark.parametrize("d", [16, 144, 5120, 20000])
def test_first_norm_and_no_norm(d, ht):
    h = rand(6, d, seed=2).to(ht)
    check_norm(None, h, (1 + 0.2 * rand(d, seed=4)).to(BF16), xn=True)
    check_norm(None, h, None)
    check_norm((0.1 * rand(6, d, seed=3)).to(BF16), h, None, xn=True)


def test_values_that_eight_bits_hold_come_back():
    """Powers of two under a largest magnitude of 448 * 2^k: the scale is 2^k to the bit, and nothing is rounded."""
    h = torch.zeros(2, 256, device="cuda")
    h[:, :128] = torch.exp2(torch.arange(128, device="cuda") % 15 - 6.0)
    h[:, 0] = 448.0
    h[:, 128:] = -h[:, :128] * 2.0 ** -20
    q, s, _, _ = run_norm(None, h, None)
    assert torch.equal(s, torch.tensor([[1.0, 1.0], [2.0 ** -20, 2.0 ** -20]], device="cuda"))
    assert torch.equal(q.view(E4M3).float() * wide(s.t()), h)


def test_zeros_tiny_and_huge_values():
    h = torch.zeros(4, 384, device="cuda")
    h[1] = 1e-38
    h[2, :128], h[2, 128:] = 3e38, 2.0 ** -100
    q, s, _, _ = run_norm(None, h, None)
    assert bool(torch.isfinite(s).all()) and bool((s > 0).all())
    got = q.view(E4M3).float() * wide(s.t())
    assert bool((got[0] == 0).all()) and bool((got[3] == 0).all())
    assert torch.allclose(got[2], h[2], rtol=2.0 ** -20, atol=0)
    zero, sz, _, n = run_norm(None, torch.zeros(3, 128, device="cuda"), torch.ones(128, device="cuda", dtype=BF16), xn=True)
    assert bool((zero.view(E4M3).float() == 0).all()) and bool(torch.isfinite(sz).all()) and bool((n == 0).all())


@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_a_bad_value_reads_as_nan_in_its_block_alone(bad):
    h = rand(3, 400, seed=1)
    h[1, 130] = bad
    q, s, _, _ = run_norm(None, h, None)
    got = q.view(E4M3).float() * wide(s.t())[:, :400]
    assert bool(torch.isnan(got[1, 128:256]).all())
    got[1, 128:256] = 0
    assert bool(torch.isfinite(got).all())
    q, s, _, _ = run_norm(None, h, torch.ones(400, device="cuda", dtype=BF16))      # the norm: the row's
    got = q.view(E4M3).float() * wide(s.t())[:, :400]
    assert bool(torch.isnan(got[1, 128:256]).all()) and bool(torch.isfinite(got[[0, 2]]).all())


@pytest.mark.parametrize("rows,ffn", [(1, 16), (3, 128), (2, 144), (17, 688), (64, 17408), (5, 2048), (300, 256)])
@pytest.mark.parametrize("xt", [BF16, F16, F32])
@pytest.mark.parametrize("spare", [0, 32])
def test_swiglu(rows, ffn, xt, spare):
    x = torch.full((rows, 2 * ffn + spare), 7.0, device="cuda", dtype=xt)
    x[:, :2 * ffn] = (3.0 * rand(rows, 2 * ffn, seed=rows)).to(xt)
    x[0, :8] = torch.tensor([-90.0, -60.0, -20.0, 0.0, 20.0, 60.0, 90.0, -100.0]).to(xt)
    q, s = torch.full((rows, ffn + spare), 0x55, dtype=torch.uint8, device="cuda"), torch.full(((ffn + 127) // 128, rows + spare), 7.0, device="cuda")
    K.swiglu_fp8(x[:, :2 * ffn], q[:, :ffn], s[:, :rows])
    torch.cuda.synchronize()
    assert bool((q[:, ffn:] == 0x55).all()) and bool((s[:, rows:] == 7).all())
    g, u = x[:, :2 * ffn].double().split(ffn, 1)
    y = g * torch.sigmoid(g) * u
    # exp: 2 steps and |g| roundings of its argument; a sum, a quotient of 2 steps, a product; below 2^-126 it may be 0
    check_rows(q[:, :ffn].contiguous(), s[:, :rows].contiguous(), y, y.abs() * (12 + 2 * g.abs()) * 2 * U + 2.0 ** -120)


def test_swiglu_leaves_the_rows_behind_the_total():
    x = rand(40, 2 * 272, seed=1).to(BF16)
    full, sf = K.fp8_rows(40, 272)
    K.swiglu_fp8(x, full, sf)
    for total in (0, 1, 17, 40, 99, -3):
        q, s = torch.full((40, 272), 0x55, dtype=torch.uint8, device="cuda"), torch.full((3, 40), 7.0, device="cuda")
        K.swiglu_fp8(x, q, s, total=torch.tensor([total], dtype=torch.int32, device="cuda"))
        n = max(0, min(40, total))
        assert torch.equal(q[:n], full.view(torch.uint8)[:n]) and torch.equal(s[:, :n], sf[:, :n]) and bool((q[n:] == 0x55).all()) and bool((s[:, n:] == 7).all())


def test_bad_gates_read_as_nan():
    x = rand(2, 256, seed=1)
    x[1, 3] = float("nan")
    q, s = K.fp8_rows(2, 128)
    K.swiglu_fp8(x, q, s)
    got = q.float() * wide(s.t())
    assert bool(torch.isnan(got[1]).all()) and bool(torch.isfinite(got[0]).all())


def test_small_gates_of_large_values():
    """1 / (1 + e^90) is below the normal numbers of float32 (there in steps of 2^-149, 2^-19 of it), but a value of 2^120 brings it back."""
    x = torch.zeros(2, 256, device="cuda")
    x[0, :3], x[0, 128:] = torch.tensor([-88.0, -87.5, -80.0]), 2.0 ** 120
    x[1, 0], x[1, 128:] = -90.0, 2.0 ** 120
    q, s = K.fp8_rows(2, 128)
    K.swiglu_fp8(x, q, s)
    g = x[:, :128].double()
    y = g * torch.sigmoid(g) * x[:, 128:].double()
    check_rows(q.view(torch.uint8), s, y, y.abs() * ((12 + 2 * 90) * 2 * U + 2.0 ** -19))


def test_no_rows_and_captured_calls():
    K.add_norm_fp8(None, torch.zeros(0, 128, device="cuda"), None, 1e-6, *K.fp8_rows(0, 128))
    K.swiglu_fp8(torch.zeros(0, 256, device="cuda"), *K.fp8_rows(0, 128))
    x, h, w = rand(9, 1024, seed=1).to(BF16), rand(9, 1024, seed=2).to(BF16), torch.ones(1024, device="cuda", dtype=BF16)
    h0 = h.clone()
    q, s = K.fp8_rows(9, 1024)
    q2, s2 = K.fp8_rows(9, 512)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        K.add_norm_fp8(x, h, w, 1e-6, q, s)                           # (loads the kernels)
        K.swiglu_fp8(h, q2, s2)
    torch.cuda.synchronize()
    want = [t.clone() for t in (q.view(torch.uint8), s, q2.view(torch.uint8), s2)]
    graph = torch.cuda.CUDAGraph()
    with capturing(graph):
        K.add_norm_fp8(x, h, w, 1e-6, q, s)
        K.swiglu_fp8(h, q2, s2)
    for _ in range(3):
        h.copy_(h0)
        for t in (q, s, q2, s2):
            t.view(torch.uint8).zero_()
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip((q.view(torch.uint8), s, q2.view(torch.uint8), s2), want):
            assert torch.equal(a, b)


def test_refusals():
    h, w = torch.zeros(4, 256, device="cuda", dtype=BF16), torch.ones(256, device="cuda", dtype=BF16)
    q, s = K.fp8_rows(4, 256)
    ok = dict(x=h.clone(), h=h, norm_w=w, eps=1e-6, q=q, s=s)
    K.add_norm_fp8(**ok)
    K.add_norm_fp8(**{**ok, "q": q.view(torch.uint8)})
    long = torch.zeros(4, 512, device="cuda", dtype=BF16)
    for bad in (dict(h=h.half()), dict(h=h[0]), dict(h=h[:, :250]), dict(h=h.t()), dict(x=h.double()), dict(x=h[:3]), dict(x=h.cpu()), dict(norm_w=w.float()), dict(norm_w=w[:128]), dict(q=q[:3]),
                dict(q=q.float()), dict(q=q.t()), dict(s=s[:1]), dict(s=s.t()), dict(s=s.half()), dict(s=s[:, :3]), dict(xn=h.float()), dict(xn=h[:, :128]), dict(xn=h.cpu()),
                dict(weights=torch.ones(4, 2, device="cuda")), dict(x=None, weights=torch.ones(4, 1, device="cuda")), dict(weights=torch.ones(3, 1, device="cuda"), x=h[:, None]),
                dict(weights=torch.ones(4, 1, device="cuda").half(), x=h[:, None]), dict(weights=torch.ones(4, 0, device="cuda"), x=long[:, :0, None].expand(4, 0, 256)),
                dict(weights=torch.ones(4, 2, device="cuda"), x=long.view(4, 2, 256)[:, :, ::1].transpose(0, 1).contiguous().transpose(0, 1)),
                dict(h=long[:, 4:260]), dict(x=long[:, 1:257]), dict(q=torch.zeros(4, 264, device="cuda", dtype=E4M3)[:, :256]), dict(xn=torch.zeros(4, 260, device="cuda", dtype=BF16)[:, :256]),
                dict(norm_w=torch.ones(260, device="cuda", dtype=BF16)[4:])):
        with pytest.raises(ValueError):
            K.add_norm_fp8(**{**ok, **bad})
    x = torch.zeros(4, 512, device="cuda", dtype=BF16)
    K.swiglu_fp8(x, q, s)
    for bad in (dict(x=x.double()), dict(x=x[0]), dict(x=x[:, :500]), dict(x=x.t()), dict(x=x[:3]), dict(q=q[:, :128]), dict(s=s[:1]), dict(total=torch.zeros(1, device="cuda")),
                dict(total=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(x=torch.zeros(4, 516, device="cuda", dtype=BF16)[:, :512]), dict(q=torch.zeros(4, 264, device="cuda", dtype=E4M3)[:, 8:])):
        with pytest.raises(ValueError):
            K.swiglu_fp8(**{**dict(x=x, q=q, s=s), **bad})

"""Block-scaled E4M3 weights on the host, and what the operators refuse before anything reaches a device."""
import pytest
import torch

from rexl3_b200.ops import kernels as K
from rexl3_b200.ops import lib as L

E4M3 = torch.float8_e4m3fn


@pytest.mark.parametrize("shape", [(1, 16), (128, 128), (130, 144), (3, 200, 272)])
def test_quantize_is_off_by_half_a_step(shape):
    g = torch.Generator().manual_seed(sum(shape))
    dense = torch.randn(*shape, generator=g) * torch.exp2(torch.randint(-8, 8, (*shape[:-1], 1), generator=g).float())
    w = K.Fp8BlockWeight.quantize(dense)
    assert w.w.shape == dense.shape and (w.N, w.K) == shape[-2:] and w.experts == (shape[0] if len(shape) == 3 else None)
    s = w.scales.repeat_interleave(128, -2)[..., :w.N, :].repeat_interleave(128, -1)[..., :w.K].double()
    # half a step: 2^-4 of the value, 2^-10 of the scale where the byte is subnormal; the float32 division before it adds 2^-24
    assert bool(((w.dense().double() - dense.double()).abs() <= torch.maximum(dense.double().abs() * (2.0 ** -4 + 2.0 ** -22), s * 2.0 ** -10)).all())


def test_quantize_takes_blocks_of_zeros_and_the_largest_value():
    dense = torch.zeros(256, 256)
    dense[0, 0], dense[200, 3] = 3.0e38, -1e-30
    w = K.Fp8BlockWeight.quantize(dense)
    assert bool(torch.isfinite(w.dense()).all()) and bool((w.dense()[128:, 128:] == 0).all())
    assert abs(float(w.dense()[0, 0]) / 3.0e38 - 1) < 2.0 ** -22 and abs(float(w.dense()[200, 3]) / -1e-30 - 1) < 2.0 ** -4


def test_weights_are_refused():
    w, s = torch.zeros(256, 144, dtype=torch.uint8), torch.ones(2, 2)
    assert K.Fp8BlockWeight(w, s).bias is None
    assert K.Fp8BlockWeight(w.view(E4M3), s, torch.zeros(256)).bias is not None
    for bad in (w.float(), w[:, :136], w[None, None], w[:0]):
        with pytest.raises(ValueError, match="w:"):
            K.Fp8BlockWeight(bad, s)
    for bad in (s.double(), s[:1], torch.ones(3, 2), s[0]):
        with pytest.raises(ValueError, match="scales"):
            K.Fp8BlockWeight(w, bad)
    for bad in (torch.zeros(255), torch.zeros(256).double()):
        with pytest.raises(ValueError, match="bias"):
            K.Fp8BlockWeight(w, s, bad)
    with pytest.raises(ValueError, match="bias"):
        K.Fp8BlockWeight(w[None], s[None], torch.zeros(256))
    with pytest.raises(ValueError, match="16-byte"):
        K.Fp8BlockWeight(torch.zeros(16 * 16 + 1, dtype=torch.uint8)[1:].view(16, 16), torch.ones(1, 1))


def test_tensors_off_the_gpu_are_refused():
    h, q, s, st = torch.zeros(2, 128, dtype=torch.bfloat16), torch.zeros(2, 128, dtype=E4M3), torch.zeros(1, 2), torch.zeros(8, dtype=torch.int32)
    w = K.Fp8BlockWeight(torch.zeros(128, 128, dtype=E4M3), torch.ones(1, 1))
    for call in (lambda: K.add_norm_fp8(None, h, None, 1e-6, q, s), lambda: K.swiglu_fp8(torch.zeros(2, 256), q, s), lambda: K.fp8_block_linear(q, s, w, h, st),
                 lambda: K.fp8_block_experts(q, s, w, st, h, st)):
        with pytest.raises(ValueError, match="CUDA tensor"):
            call()


def test_entry_points_refuse_what_does_not_fit():
    """A C caller's mistakes come back as an error code, before anything is launched: pointers that are never followed."""
    lib, p = L.load(), 4096
    norm = dict(x=p, x_type=0, ldx=256, weights=None, terms=1, h=p, h_type=0, ldh=256, norm_w=p, eps=1e-6, q=p, ldq=256, s=p, lds=4, xn=None, ldn=0, rows=4, d=256, stream=None)
    for bad in (dict(rows=0), dict(d=250), dict(d=0), dict(d=65536, ldx=65536, ldh=65536, ldq=65536), dict(terms=2), dict(terms=0), dict(x_type=3), dict(h_type=1), dict(h=None), dict(q=None),
                dict(s=None), dict(ldx=240), dict(ldh=240), dict(ldq=240), dict(lds=3), dict(xn=p, ldn=128), dict(x=p + 2), dict(h=p + 8), dict(q=p + 1), dict(norm_w=p + 2), dict(ldh=260),
                dict(ldq=264), dict(xn=p, ldn=260), dict(x=p, ldx=257)):
        assert lib.rx_add_norm_fp8(*{**norm, **bad}.values()) != 0, bad
    act = dict(x=p, x_type=0, ldx=512, q=p, ldq=256, s=p, lds=4, total=None, rows=4, F=256, stream=None)
    for bad in (dict(rows=0), dict(F=8), dict(F=250), dict(F=1 << 21), dict(x_type=-1), dict(x=None), dict(q=None), dict(s=None), dict(ldx=511), dict(ldq=255), dict(lds=3), dict(x=p + 4), dict(q=p + 8),
                dict(ldx=516), dict(ldq=260)):
        assert lib.rx_swiglu_fp8(*{**act, **bad}.values()) != 0, bad
    lin = dict(q=p, ldq=256, s=p, lds=4, rows=4, K=256, w=p, ws=p, bias=None, N=128, out=p, out_type=0, ldo=128, status=p, stream=None)
    common = (dict(rows=0), dict(K=0), dict(K=250), dict(N=0), dict(ldq=240), dict(lds=3), dict(ldo=127), dict(q=None), dict(s=None), dict(w=None), dict(ws=None), dict(out=None), dict(out_type=3),
              dict(out_type=-1), dict(q=p + 8), dict(w=p + 8), dict(ldq=264), dict(s=p + 2), dict(ws=p + 1), dict(out=p + 1), dict(out=p + 2, out_type=2))
    for bad in (*common, dict(bias=p + 2)):
        assert lib.rx_fp8_block_linear(*{**lin, **bad}.values()) != 0, bad
    exp = dict(q=p, ldq=256, s=p, lds=4, rows=4, K=256, w=p, ws=p, experts=2, N=128, offs=p, src=None, src_div=1, dst=None, cap=4, out=p, out_type=0, ldo=128, out_rows=4, status=p, stream=None)
    for bad in (*common, dict(experts=0), dict(experts=5000), dict(offs=None), dict(cap=0), dict(cap=5), dict(cap=5, src=p), dict(cap=5, dst=p), dict(src_div=0), dict(out_rows=0), dict(out_rows=3)):
        assert lib.rx_fp8_block_experts(*{**exp, **bad}.values()) != 0, bad


def test_entry_points_refuse_what_their_numbers_cannot_hold():
    lib, p, many = L.load(), 4096, (1 << 30) + 1
    assert lib.rx_add_norm_fp8(p, 0, 16, None, 1, p, 0, 16, p, 1e-6, p, 16, p, many, None, 0, many, 16, None) != 0
    assert lib.rx_swiglu_fp8(p, 0, 1 << 21, p, 1 << 20, p, 1 << 18, None, 1 << 18, 1 << 20, None) != 0        # 2^31 blocks
    assert lib.rx_fp8_block_linear(p, 16, p, many, many, 16, p, p, None, 16, p, 0, 16, p, None) != 0
    for rows, cap, experts, N, ldq in ((many, 4, 1, 16, 16), (4, many, 1, 16, 16), (4, 4, 4096, 1 << 20, 16), (1 << 20, 4, 1, 16, 1 << 17)):
        assert lib.rx_fp8_block_experts(p, ldq, p, rows, rows, 16, p, p, experts, N, p, p, 1, p, cap, p, 0, N, 4, p, None) != 0, (rows, cap, experts, N, ldq)

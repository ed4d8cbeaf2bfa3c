"""Products with 4-bit weights against the dequantised weight in 64 bits.

Bound (set before the first run).  Codes and activations enter the products
exactly (a code may be carried as code + offset with the offset's share of
the sum taken off again, which multiplies the magnitudes by at most 1032);
sums and scaling are in fp32.  With S = sum_k |x_k| * scale_k an output is off by at
most 1032 * 2 * 2^-23 * S plus one rounding, u * |y|.  The gated form has a
slope of at most 1.1 in the gate: the same bound with S_gate * 1.1 * |up| +
S_up * |silu(gate)|, and 8 * 2^-23 of the result for the exponential.
"""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

U = {dt: torch.finfo(dt).eps / 2 for dt in (torch.float16, torch.bfloat16)}  # unit roundoff
EPS = 1032 * 2 * 2.0 ** -23


def _weight(K_, dev, N, K, group, zeros, dtype, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    codes = torch.randint(0, 256, (N, K // 2), generator=g, device=dev, dtype=torch.uint8)
    scales = ((0.5 + torch.rand((N, K // group), generator=g, device=dev)) / K ** 0.5).to(dtype)
    z = None
    if zeros:
        z = torch.randint(0, 16, (N, K // group), generator=g, device=dev, dtype=torch.uint8)
    return K_.W4Weight(codes, scales, z)


def _parts(w, x):
    """(y, S) in 64 bits, codes unpacked one by one."""
    c = w.codes.cpu().to(torch.int64)
    q = torch.empty((w.N, w.K), dtype=torch.float64)
    q[:, 0::2] = (c & 15).double()
    q[:, 1::2] = (c >> 4).double()
    s = w.scales.double().cpu().repeat_interleave(w.group_size, 1)
    z = 8.0 if w.zeros is None else w.zeros.double().cpu().repeat_interleave(w.group_size, 1)
    xd = x.double().cpu()
    return xd @ ((q - z) * s).t(), xd.abs() @ s.t()


def _check(got, w, x, silu=False):
    u = U[x.dtype]
    y, mag = _parts(w, x)
    tol = EPS * mag
    if silu:
        n = w.N // 2
        a, b, ta, tb = y[:, :n], y[:, n:], tol[:, :n], tol[:, n:]
        act = a * torch.sigmoid(a)
        y = act * b
        tol = 1.1 * ta * b.abs() + tb * act.abs() + 8 * 2.0 ** -23 * y.abs() + 1.1 * ta * tb
    tol = tol + u * y.abs() + 1e-7
    diff = (got.double().cpu() - y).abs()
    assert (diff / tol).max().item() <= 1.0


SHAPES = [(2560, 2048, 128), (1, 32, 32), (17, 128, 128), (130, 576, 64), (257, 1056, 32),
          (64, 8192, 128), (4096, 14336, 64), (100, 16384, 128), (1000, 4096, 32)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("N,K,group", SHAPES)
def test_matches_dequantised_weight(cuda_device, N, K, group, zeros, dtype):
    from vllm_mps_b200 import kernels as K_

    w = _weight(K_, cuda_device, N, K, group, zeros, dtype, seed=N + K)
    g = torch.Generator(device=cuda_device).manual_seed(K)
    for M in (1, 2, 8, 9, 16, 17, 32) if N * K < 10 ** 6 else (1, 5, 16, 31):
        x = torch.randn((M, K), generator=g, device=cuda_device).to(dtype)
        got = K_.w4_gemm(x, w)
        torch.cuda.synchronize()
        assert K_.error_word(cuda_device) == 0
        _check(got, w, x)
        assert torch.equal(got, K_.w4_gemm(x, w))  # the order of sums is fixed


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M,inter,K,group", [(1, 5632, 2048, 128), (3, 37, 1024, 64), (16, 64, 96, 32),
                                             (20, 300, 4096, 128), (32, 129, 640, 128)])
def test_gated_form(cuda_device, dtype, M, inter, K, group):
    from vllm_mps_b200 import kernels as K_

    w = _weight(K_, cuda_device, 2 * inter, K, group, True, dtype, seed=inter)
    g = torch.Generator(device=cuda_device).manual_seed(K)
    x = torch.randn((M, K), generator=g, device=cuda_device).to(dtype)
    _check(K_.w4_gemm(x, w, silu_mul=True), w, x, silu=True)


def test_offsets_do_not_hide_small_sums(cuda_device):
    """All codes at the zero point: the result is exactly zero.  Activations that share a
    large mean: the offset's share of the sum is taken off to fp32 accuracy."""
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    codes = torch.full((48, 256), 0x88, dtype=torch.uint8, device=dev)
    scales = torch.ones((48, 4), dtype=torch.float16, device=dev)
    x = torch.randint(-8, 9, (4, 512), device=dev).half()
    assert (K_.w4_gemm(x, K_.W4Weight(codes, scales)) == 0).all()
    w = _weight(K_, dev, 200, 1024, 128, True, torch.bfloat16, seed=3)
    g = torch.Generator(device=dev).manual_seed(1)
    x = (torch.randn((6, 1024), generator=g, device=dev) + 30).bfloat16()
    _check(K_.w4_gemm(x, w), w, x)


def test_strides_and_out(cuda_device):
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, 75, 256, 64, True, torch.float16, seed=5)
    g = torch.Generator(device=dev).manual_seed(2)
    xb = torch.randn((10, 256 + 40), generator=g, device=dev).half()
    x = xb[:, 8:264]
    want = K_.w4_gemm(x.contiguous(), w)
    buf = torch.full((10, 81), 9.0, dtype=torch.float16, device=dev)
    got = K_.w4_gemm(x, w, out=buf[:, 3:78])  # odd row stride, odd start
    assert torch.equal(got, want)
    assert (buf[:, :3] == 9.0).all() and (buf[:, 78:] == 9.0).all()
    assert K_.w4_gemm(x[:0], w).shape == (0, 75)


def test_infinite_activation_stays_in_its_row(cuda_device):
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, 64, 512, 128, True, torch.float16, seed=6)
    x = torch.ones((3, 512), device=dev).half()
    x[1, 100] = float("inf")
    got = K_.w4_gemm(x, w)
    assert torch.isfinite(got[0]).all() and torch.isfinite(got[2]).all()
    assert not torch.isfinite(got[1]).all()


def test_quantize_round_trip(cuda_device):
    """Every weight within half a step of its code's value (the scale rounds to 16 bits, so
    the extreme codes of a group may be one rounding of the scale further off)."""
    from vllm_mps_b200 import kernels as K_

    g = torch.Generator(device=cuda_device).manual_seed(9)
    for dtype in (torch.float16, torch.bfloat16):
        w = torch.randn((33, 512), generator=g, device=cuda_device).to(dtype)
        w[5] = 0
        w[6] = 0.25
        for zp in (False, True):
            for group in (32, 64, 128):
                q = K_.quantize_w4(w, group, zero_points=zp)
                step = q.scales.float().repeat_interleave(group, 1)
                err = (q.dequantize() - w.float()).abs()
                # half a step, half a step more where the zero point's rounding moves a
                # group's end past the last code, and 15 roundings of the scale
                slack = (1.0 if zp else 0.5) + 15 * U[dtype] * 2
                assert (err <= step * slack + 1e-6).all()
        x = torch.randn((2, 512), generator=g, device=cuda_device).to(dtype)
        _check(K_.w4_gemm(x, q), q, x)


def test_graph_replay(cuda_device):
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, 512, 2048, 128, True, torch.bfloat16, seed=7)
    x = torch.randn((4, 2048), device=dev).bfloat16()
    K_.w4_gemm(x, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        a = K_.w4_gemm(x, w)
        b = K_.w4_gemm(x, w)
    x.copy_(torch.randn((4, 2048), device=dev).bfloat16())
    g.replay()
    torch.cuda.synchronize()
    want = K_.w4_gemm(x, w)
    assert torch.equal(a, want) and torch.equal(b, want)


def test_refusals(cuda_device):
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, 64, 256, 64, True, torch.float16, seed=8)
    x = torch.randn((2, 256), device=dev).half()
    with pytest.raises(TypeError):
        K_.w4_gemm(x.bfloat16(), w)
    with pytest.raises(ValueError):
        K_.w4_gemm(x[:, :128], w)
    with pytest.raises(ValueError):
        K_.w4_gemm(x.t().contiguous().t(), w)
    with pytest.raises(NotImplementedError):
        K_.w4_gemm(torch.zeros((33, 256), device=dev).half(), w)
    with pytest.raises(ValueError, match="aligned"):
        K_.w4_gemm(torch.zeros((2, 264), device=dev).half()[:, 4:260], w)
    with pytest.raises(ValueError):
        K_.w4_gemm(x, _weight(K_, dev, 63, 256, 64, True, torch.float16, seed=8), silu_mul=True)
    with pytest.raises(RuntimeError, match="CUDA"):
        K_.w4_gemm(x.cpu(), w)
    with pytest.raises(ValueError):
        K_.W4Weight(w.codes, w.scales[:10], w.zeros)
    with pytest.raises(ValueError):
        K_.W4Weight(w.codes.int(), w.scales)
    with pytest.raises(NotImplementedError):  # group 256
        K_.w4_gemm(x, K_.W4Weight(w.codes, w.scales[:, :1].contiguous()))
    with pytest.raises(ValueError):
        K_.quantize_w4(torch.zeros((4, 100), device=dev).half())


def test_rows_whose_bytes_pass_31_bits(cuda_device):
    """32 rows of 2^26 columns (4 GB), zero but for a few columns all along them."""
    from vllm_mps_b200 import kernels as K_

    dev, K, M = cuda_device, 2 ** 26, 32
    w = _weight(K_, dev, 2, K, 128, False, torch.float16, seed=4)
    g = torch.Generator(device=dev).manual_seed(5)
    at = torch.unique(torch.randint(0, K, (3000,), generator=g, device=dev))
    at = torch.unique(torch.cat([at, torch.tensor([0, K - 1], device=dev)]))
    x = torch.zeros((M, K), dtype=torch.float16, device=dev)
    x[:, at] = torch.randn((M, len(at)), generator=g, device=dev).half() * 100
    got = K_.w4_gemm(x, w).double()
    assert K_.error_word(dev) == 0
    code = w.codes[:, at // 2]
    code = torch.where(at % 2 == 1, code >> 4, code & 15).double() - 8
    s = w.scales[:, at // 128].double()
    xd = x[:, at].double()
    y, mag = xd @ (code * s).t(), xd.abs() @ s.t()
    assert ((got - y).abs() <= EPS * mag + U[torch.float16] * y.abs() + 1e-7).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("silu", [False, True])
@pytest.mark.parametrize("M,N,K,group", [(2, 100, 640, 64), (5, 130, 576, 64), (12, 70, 640, 128),
                                         (20, 36, 96, 32), (32, 40, 8192, 128)])
def test_non_finite_activations_follow_the_formula(cuda_device, M, N, K, group, silu, zeros, dtype):
    """One infinity is an infinity of the code's sign (NaN where the code is the zero point),
    two may cancel to NaN, and the rows without any are untouched."""
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, N, K, group, zeros, dtype, seed=M)
    g = torch.Generator(device=dev).manual_seed(M + 1)
    x = torch.randn((M, K), generator=g, device=dev).to(dtype)
    clean = K_.w4_gemm(x, w, silu_mul=silu)
    x[1, 41] = float("inf")
    x[M - 1, 5] = float("-inf")
    x[M - 1, K - 1] = float("inf")
    if M > 2:
        x[M // 2, K // 2] = float("nan")
    y, _ = _parts(w, x)
    if silu:
        y = y[:, :N // 2] / (1.0 + torch.exp(-y[:, :N // 2])) * y[:, N // 2:]
    got = K_.w4_gemm(x, w, silu_mul=silu)
    touched = {1, M - 1} | ({M // 2} if M > 2 else set())
    for r in range(M):
        if r in touched:
            want = y[r]
            assert torch.equal(torch.isnan(got[r].cpu()), torch.isnan(want))
            sure = ~torch.isnan(want)
            assert torch.equal(got[r].cpu().double()[sure], want[sure])
        else:
            assert torch.equal(got[r], clean[r])
    if M > 2:  # (of two rows the second has all three: NaN throughout)
        assert torch.isinf(y[1]).any()


@pytest.mark.parametrize("size", [1e-4, 1e-6])
def test_subnormal_scales(cuda_device, size):
    """Weights so small that their fp16 scales are subnormal: their codes are used in full."""
    from vllm_mps_b200 import kernels as K_

    g = torch.Generator(device=cuda_device).manual_seed(3)
    full = (torch.randn((40, 512), generator=g, device=cuda_device) * size).half()
    w = K_.quantize_w4(full, 64)
    assert (w.scales < torch.finfo(torch.float16).smallest_normal).all() and (w.scales > 0).all()
    assert len(torch.unique(w.codes & 15)) > 4
    x = torch.randn((3, 512), generator=g, device=cuda_device).half() * 1000
    _check(K_.w4_gemm(x, w), w, x)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("M", [1, 10, 25])
def test_zero_points_of_all_eight_bits(cuda_device, M, dtype):
    """A zero point above 15 adds up to 255 to the magnitudes that the bound's 1032 stands for."""
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, 90, 1024, 64, True, dtype, seed=11)
    w.zeros.copy_(torch.arange(90 * 16, device=dev).view(90, 16) % 256)
    g = torch.Generator(device=dev).manual_seed(M)
    x = torch.randn((M, 1024), generator=g, device=dev).to(dtype)
    y, mag = _parts(w, x)
    diff = (K_.w4_gemm(x, w).double().cpu() - y).abs()
    assert (diff <= EPS * (1032 + 255) / 1032 * mag + U[dtype] * y.abs() + 1e-7).all()


@pytest.mark.parametrize("M", [1, 7, 16, 32])
def test_bf16_activations_of_any_size(cuda_device, M):
    """bf16 groups enter the fp16 products scaled by a power of two of their own: a power of
    two in x is the same one in y, bit for bit, and within a group small and large values,
    zeros and the smallest numbers stand side by side."""
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    w = _weight(K_, dev, 100, 1024, 64, True, torch.bfloat16, seed=12)
    g = torch.Generator(device=dev).manual_seed(M)
    x = torch.randn((M, 1024), generator=g, device=dev).bfloat16()
    want = K_.w4_gemm(x, w).double()
    for power in (-100, -40, 40, 100):
        got = K_.w4_gemm((x.double() * 2.0 ** power).bfloat16(), w).double()
        assert torch.equal(got * 2.0 ** -power, want)
    wide = (x.double() * torch.exp2(torch.randint(-40, 41, x.shape, generator=g, device=dev))).bfloat16()
    wide[:, :64] = 0                      # a group of zeros
    wide[:, 64:128] = 2.0 ** -133         # a group of bf16's smallest numbers
    wide[:, 200] = 2.0 ** -133            # one beside ordinary ones
    wide[0] = 0
    _check(K_.w4_gemm(wide, w), w, wide)
    assert (K_.w4_gemm(wide, w)[0] == 0).all()


def test_fp16_outliers_and_large_means(cuda_device):
    from vllm_mps_b200 import kernels as K_

    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(13)
    w = _weight(K_, dev, 150, 2048, 128, False, torch.float16, seed=13)
    for M in (2, 12, 30):
        x = torch.randn((M, 2048), generator=g, device=dev)
        x[:, 700] = 4000.0
        _check(K_.w4_gemm(x.half(), w), w, x.half())
        x = torch.randn((M, 2048), generator=g, device=dev) + 30
        _check(K_.w4_gemm(x.half(), w), w, x.half())

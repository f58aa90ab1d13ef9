"""int4_linear on the GPU against 64-bit products of the same codes."""
import numpy as np
import pytest
import torch

from paged_case import HALF_STEP

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(ca, M, N, K, g, zeros, dtype, seed=0):
    gen = torch.Generator().manual_seed(seed)
    codes = torch.randint(0, 16, (N, K), generator=gen, dtype=torch.uint8)
    groups = -(-K // g)
    scales = (0.01 * (0.5 + torch.rand(N, groups, generator=gen))).to(dtype)
    z = torch.randint(0, 16, (N, groups), generator=gen) if zeros else None
    x = torch.randn(M, K, generator=gen).to(dtype)
    w = ca.Int4Weight.from_codes(codes.cuda(), scales.cuda(), None if z is None else z.cuda(), g)
    return codes, scales, z, x, w


def exact(codes, scales, z, x, g):
    """Result and tolerance: each group's sums of up to g fp32 terms as large as
    31 |x| and (16 + z) |x|, twice 24 bits each over them (products are exact, fp32
    x in limbs to 2^-24); then a sum over groups and waves, and the output's rounding."""
    K = codes.shape[1]
    group = np.arange(K) // g
    s = scales.double().numpy()[:, group]
    c = codes.double().numpy()
    zero = 8.0 if z is None else z.double().numpy()[:, group]
    xd = x.double().numpy()
    y = xd @ (s * (c - zero)).T
    mag = np.abs(xd) @ (s * (16 + c + 16 + zero)).T
    groups = -(-K // g)
    tol = mag * (8 + groups) * 2.0 ** -24 * (2 if min(g, K) <= 512 else 4) + HALF_STEP[x.dtype] * np.abs(y) + 1e-30
    if x.dtype == torch.float16:
        tol += 2.0 ** -25
    return y, tol


def check(ca, M, N, K, g, zeros, dtype, seed=0):
    print(f"[case] {M} {N} {K} {g} {zeros} {dtype}", flush=True)
    codes, scales, z, x, w = make(ca, M, N, K, g, zeros, dtype, seed)
    y = ca.int4_linear(x.cuda(), w)
    assert y.shape == (M, N) and y.dtype == dtype
    want, tol = exact(codes, scales, z, x, g)
    err = np.abs(y.double().cpu().numpy() - want)
    assert (err <= tol).all(), f"{np.max(err / tol):.3g} of the tolerance"
    return x, w, y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("g", [32, 64, 128, 256, 1024])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 16, 128), (1, 100, 1000), (3, 33, 257), (17, 64, 384), (1, 48, 2048)])
def test_shapes(gpu_ca, dtype, g, zeros, M, N, K):
    check(gpu_ca, M, N, K, g, zeros, dtype, seed=M + N + K)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [2, 15, 16, 31, 32, 33, 64, 100])
def test_rows(gpu_ca, dtype, M):
    check(gpu_ca, M, 80, 520, 64, True, dtype, seed=M)


@pytest.mark.parametrize("dtype", TYPES)
def test_wide_matrices(gpu_ca, dtype):
    for M in (1, 16, 40):
        check(gpu_ca, M, 4096, 1024, 128, False, dtype, seed=1)
        check(gpu_ca, M, 1000, 5000, 32, True, dtype, seed=2)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(gpu_ca, dtype):
    x, w, y = check(gpu_ca, 6, 70, 200, 64, True, dtype, seed=3)
    x = x.cuda()
    assert torch.equal(gpu_ca.int4_linear(x.view(2, 3, 200), w), y.view(2, 3, 70))
    assert torch.equal(gpu_ca.int4_linear(x[0], w), y[0])
    wide = torch.full((6, 333), float("nan"), device="cuda", dtype=dtype)
    wide[:, 5:205] = x
    assert torch.equal(gpu_ca.int4_linear(wide[:, 5:205], w), y)
    assert torch.equal(gpu_ca.int4_linear(x.t().contiguous().t(), w), y)
    assert torch.equal(gpu_ca.int4_linear(torch._neg_view(x), w), gpu_ca.int4_linear(-x, w))
    assert gpu_ca.int4_linear(x[:0], w).shape == (0, 70)
    one = x[:1].expand(4, 200)  # the same row four times
    assert torch.equal(gpu_ca.int4_linear(one, w), y[:1].expand(4, 70))


def test_rows_do_not_touch_each_other(gpu_ca):
    """A NaN or an infinity in a row gives NaN there and nothing elsewhere."""
    x, w, y = check(gpu_ca, 5, 40, 300, 32, True, torch.bfloat16, seed=4)
    for bad in (float("nan"), float("inf"), -float("inf")):
        z = x.cuda()
        z[2, 299] = bad
        got = gpu_ca.int4_linear(z, w)
        assert torch.isnan(got[2]).all()
        assert torch.equal(got[:2], y[:2]) and torch.equal(got[3:], y[3:])


def test_captured(gpu_ca):
    _, _, _, x, w = make(gpu_ca, 4, 512, 640, 128, False, torch.bfloat16)
    x = x.cuda()
    gpu_ca.int4_linear(x, w)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = gpu_ca.int4_linear(x, w)
    for _ in range(3):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, gpu_ca.int4_linear(x, w))


@pytest.mark.parametrize("zero_points", [False, True])
def test_quantize_and_module(gpu_ca, zero_points):
    """A weight is off by at most half a step; the module is the product with it."""
    lin = torch.nn.Linear(200, 96, bias=False, device="cuda")
    w = gpu_ca.Int4Weight.quantize(lin.weight, 64, zero_points)
    d = w.dequantize()
    step = w.scales.t()[:, torch.arange(200, device="cuda") // 64]
    # symmetric: the largest value may lie half a rounding of the scale past code 15 or 1; with zero
    # points the rounded zero moves the range by up to half a step
    assert ((d - lin.weight).abs() <= step * (1.001 if zero_points else 0.501)).all()
    mod = gpu_ca.Int4Linear.from_linear(lin, 64, zero_points)
    x = torch.randn(3, 200, device="cuda")
    with torch.no_grad():
        assert torch.equal(mod(x), gpu_ca.int4_linear(x, w))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("g", [32, 64, 128])
@pytest.mark.parametrize("M,N", [(1, 5000), (9, 5000), (1, 8200), (5, 8208), (20, 100), (40, 3001), (33, 8200)])
def test_grids_past_the_compute_units(gpu_ca, dtype, g, M, N):
    """Work groups of either size: up to one for each compute unit, and more."""
    check(gpu_ca, M, N, 2500, g, True, dtype)

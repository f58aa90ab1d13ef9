"""rotary_embedding and rotary_append on the GPU against complex products in 64
bits: layouts, parts of the head, scalings, far positions, strides, gradients."""
import math

import numpy as np
import pytest
import torch

from paged_case import HALF_STEP

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def rotate64(x, positions, rotary, inverse=False):
    """[N, H, D] in numpy, as complex products; and the tolerance."""
    R = rotary.rotary_dim
    f = rotary.turns.double().cpu().numpy() * 2 * math.pi
    xs = x.detach().double().cpu().numpy()
    z = rotary.magnitude * np.exp(1j * (-1 if inverse else 1) * positions.double().cpu().numpy()[:, None, None] * f)
    y = xs.copy()
    if rotary.layout == "interleaved":
        a, b = xs[..., 0:R:2], xs[..., 1:R:2]
    else:
        a, b = xs[..., :R // 2], xs[..., R // 2:R]
    c = (a + 1j * b) * z
    tol = np.zeros_like(xs)
    size = rotary.magnitude * np.abs(a + 1j * b)
    # the fraction of a turn in 32 bits and its sine: 4 steps; two products, a sum; for
    # positions past 2^20 also 2^-53 turns per turn in the oracle itself
    part = size * (8 * 2.0 ** -24 + 2 * np.pi * 2.0 ** -52 * np.abs(positions.double().cpu().numpy()[:, None, None] * f))
    if rotary.layout == "interleaved":
        y[..., 0:R:2], y[..., 1:R:2] = c.real, c.imag
        tol[..., 0:R:2], tol[..., 1:R:2] = part, part
    else:
        y[..., :R // 2], y[..., R // 2:R] = c.real, c.imag
        tol[..., :R // 2], tol[..., R // 2:R] = part, part
    half = HALF_STEP[x.dtype]
    tol[..., :R] += half * np.abs(y[..., :R]) + (2.0 ** -25 if x.dtype == torch.float16 else 0) + 1e-37
    return y, tol


def close(got, want):
    y, tol = want
    err = np.abs(got.detach().double().cpu().numpy() - y)
    assert (err <= tol).all(), f"{np.max(err / np.maximum(tol, 1e-40)):.3g} of the tolerance"


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("D,R", [(64, 64), (128, 96), (8, 2), (48, 36), (80, 80), (64, 10)])
def test_forward_and_backward(gpu_ca, dtype, layout, D, R):
    print(f"[case] {D} {R} {layout} {dtype}", flush=True)
    rotary = gpu_ca.Rotary(D, rotary_dim=R, layout=layout, device="cuda")
    for N, Hq, Hk in ((1, 1, 1), (37, 4, 2), (700, 3, 5)):
        q = torch.randn(N, Hq, D, device="cuda").to(dtype).requires_grad_()
        k = torch.randn(N, Hk, D, device="cuda").to(dtype).requires_grad_()
        pos = torch.randint(0, 5000, (N,), device="cuda")
        yq, yk = gpu_ca.rotary_embedding(q, k, pos, rotary)
        close(yq, rotate64(q, pos, rotary))
        close(yk, rotate64(k, pos, rotary))
        gq, gk = torch.randn_like(yq), torch.randn_like(yk)
        dq, dk = torch.autograd.grad([yq, yk], [q, k], [gq, gk])
        assert dq.dtype == dtype and dk.dtype == dtype
        close(dq, rotate64(gq, pos, rotary, inverse=True))
        close(dk, rotate64(gk, pos, rotary, inverse=True))


def test_gradient_against_differences(gpu_ca):
    """The function is linear: a difference quotient of any step is its product
    with the gradient, up to rounding (2^-22 of the values' size)."""
    rotary = gpu_ca.Rotary(32, rotary_dim=24, layout="half", scaling="yarn", factor=4.0, original_length=64, device="cuda")
    q = torch.randn(9, 2, 32, device="cuda", requires_grad=True)
    pos = torch.arange(9, device="cuda") * 11
    g = torch.randn(9, 2, 32, device="cuda")
    y, none = gpu_ca.rotary_embedding(q, None, pos, rotary)
    assert none is None
    (dq,) = torch.autograd.grad(y, q, g)
    step = torch.randn_like(q)
    with torch.no_grad():
        diff = gpu_ca.rotary_embedding(q + step, None, pos, rotary)[0] - y
    a, b = (diff.double() * g.double()).sum(), (dq.double() * step.double()).sum()
    assert abs(a - b) <= 2.0 ** -21 * (step.abs().double() + q.abs()).sum() * rotary.magnitude * g.abs().max()
    # second order: the gradient's own gradient is the rotation
    y2, _ = gpu_ca.rotary_embedding(q, None, pos, rotary)
    g2 = g.clone().requires_grad_()
    (dq2,) = torch.autograd.grad(y2, q, g2, create_graph=True)
    (back,) = torch.autograd.grad(dq2, g2, step)
    assert torch.equal(back, gpu_ca.rotary_embedding(step, None, pos, rotary)[0])


def test_one_of_two_gradients(gpu_ca):
    rotary = gpu_ca.Rotary(16, device="cuda")
    q = torch.randn(5, 2, 16, device="cuda", requires_grad=True)
    k = torch.randn(5, 1, 16, device="cuda", requires_grad=True)
    pos = torch.arange(5, device="cuda", dtype=torch.int32)
    yq, yk = gpu_ca.rotary_embedding(q, k, pos, rotary)
    g = torch.ones_like(yk)
    dq, dk = torch.autograd.grad(yk, [q, k], g, allow_unused=True)
    assert dq is None or (dq == 0).all()
    close(dk, rotate64(g, pos, rotary, inverse=True))


@pytest.mark.parametrize("scaling", [None, "linear", "ntk", "yarn"])
@pytest.mark.parametrize("far", [1 << 17, 1 << 24, (1 << 31) - 1, 1 << 40])
def test_far_positions(gpu_ca, scaling, far):
    rotary = gpu_ca.Rotary(64, scaling=scaling, factor=8.0, original_length=4096, device="cuda")
    pos = far - torch.arange(50, device="cuda") * 3
    q = torch.randn(50, 2, 64, device="cuda")
    close(gpu_ca.rotary_embedding(q, None, pos, rotary)[0], rotate64(q, pos, rotary))
    if far < 1 << 31:
        assert torch.equal(gpu_ca.rotary_embedding(q, None, pos, rotary)[0],
                           gpu_ca.rotary_embedding(q, None, pos.int(), rotary)[0])
    neg = gpu_ca.rotary_embedding(q, None, -pos, rotary)[0]
    close(neg, rotate64(q, -pos, rotary))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_shapes(gpu_ca, dtype):
    """Views of a projection's output, batches, positions of one row for all,
    misaligned and spread rows, views of negated values."""
    rotary = gpu_ca.Rotary(32, device="cuda")
    qkv = torch.randn(3, 50, 3, 4, 32, device="cuda").to(dtype)
    q, k = qkv[:, :, 0], qkv[:, :, 1]
    pos = torch.arange(50, device="cuda")
    yq, yk = gpu_ca.rotary_embedding(q, k, pos, rotary)
    assert yq.shape == q.shape and yq.is_contiguous()
    close(yq.view(150, 4, 32), rotate64(q.reshape(150, 4, 32), pos.repeat(3), rotary))
    close(yk.view(150, 4, 32), rotate64(k.reshape(150, 4, 32), pos.repeat(3), rotary))
    odd = torch.empty(50 * 4 * 32 + 1, device="cuda", dtype=dtype)[1:].view(50, 4, 32).copy_(q[0])
    assert torch.equal(gpu_ca.rotary_embedding(odd, None, pos, rotary)[0], yq[0])
    spread = torch.empty(50, 4, 32, 2, device="cuda", dtype=dtype)[..., 1].copy_(q[0])
    assert torch.equal(gpu_ca.rotary_embedding(spread, None, pos, rotary)[0], yq[0])
    neg = torch._neg_view(q[0].contiguous())
    assert torch.equal(gpu_ca.rotary_embedding(neg, None, pos, rotary)[0], -yq[0])
    empty, _ = gpu_ca.rotary_embedding(q[0, :0], None, pos[:0], rotary)
    assert empty.shape == (0, 4, 32)


def test_agrees_with_the_training_rotation(gpu_ca):
    """The decoder's apply_rope in fp32, whose angles are 32-bit: 2^-24 of 300
    radians each way, and of its roundings."""
    q, k = (torch.randn(2, 3, 300, 64, device="cuda") for _ in range(2))
    want = gpu_ca.decoder.apply_rope(q, k, 10000.0)
    rotary = gpu_ca.Rotary(64, device="cuda")
    got = gpu_ca.rotary_embedding(*(x.transpose(1, 2) for x in (q, k)), torch.arange(300, device="cuda"), rotary)
    for a, b in zip(got, want):
        assert (a.transpose(1, 2) - b).abs().max() <= 8 * 300 * 2.0 ** -24 * q.abs().max()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("layout,D,R", [("interleaved", 64, 64), ("half", 64, 64), ("half", 40, 20), ("interleaved", 128, 96)])
@pytest.mark.parametrize("page", [1, 16, 20])
def test_append(gpu_ca, dtype, layout, D, R, page):
    print(f"[case] {D} {R} {layout} page {page} {dtype}", flush=True)
    rotary = gpu_ca.Rotary(D, rotary_dim=R, layout=layout, device="cuda")
    lengths, new, H, G = [33, 5, 16, 40], [2, 0, 16, 5], 2, 3
    N, rows = sum(new), 3
    needs = [-(-l // page) for l in lengths]
    pages = sum(needs) + 2
    order = torch.randperm(pages)
    table = torch.zeros(4, max(needs), dtype=torch.int32)
    at = 0
    for b, m in enumerate(needs):
        table[b, :m] = order[at:at + m]
        at += m
    kp, vp = (torch.randn(pages, H, page, D, device="cuda").to(dtype) for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    qkv = torch.randn(N + rows, (G + 2) * H * D, device="cuda").to(dtype)
    q = qkv[:, :G * H * D].view(-1, G * H, D)
    k = qkv[:, G * H * D:(G + 1) * H * D].view(-1, H, D)
    v = qkv[:, (G + 1) * H * D:].view(-1, H, D)
    pos = torch.randint(0, 9000, (N + rows,), device="cuda")
    starts = torch.tensor([0, 2, 2, 18, 23], dtype=torch.int32, device="cuda")
    lens = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    out = torch.full((N + rows, G * H, D), 9.0, device="cuda", dtype=dtype)
    y = gpu_ca.rotary_append(q, k, v, pos, rotary, kp, vp, table.cuda(), lens, starts, out=out)
    assert y is out and (out[N:] == 9).all()
    close(out[:N], rotate64(q[:N], pos[:N], rotary))
    yk, tol = rotate64(k, pos, rotary)
    t = 0
    for b, (l, n) in enumerate(zip(lengths, new)):
        for s in range(l - n, l):
            p = table[b, s // page].item()
            err = np.abs(kp[p, :, s % page].double().cpu().numpy() - yk[t])
            assert (err <= tol[t]).all()
            assert torch.equal(vp[p, :, s % page], v[t])
            kp[p, :, s % page], vp[p, :, s % page] = k0[p, :, s % page], v0[p, :, s % page]
            t += 1
    # nothing else was written
    assert torch.equal(kp, k0) and torch.equal(vp, v0)


def test_append_leaves_out_what_has_no_page(gpu_ca):
    """Slots before 0, table entries outside the cache, counts beyond the table."""
    rotary = gpu_ca.Rotary(16, device="cuda")
    kp, vp = (torch.zeros(4, 1, 8, 16, device="cuda") for _ in range(2))
    q = k = v = torch.randn(12, 1, 16, device="cuda")
    pos = torch.arange(12, device="cuda")
    table = torch.tensor([[0, -1], [99, 1], [2, 3]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([2, 10, 1000], dtype=torch.int32, device="cuda")  # the third is held to 16
    starts = torch.tensor([0, 4, 8, 12], dtype=torch.int32, device="cuda")
    y = gpu_ca.rotary_append(q, k, v, pos, rotary, kp, vp, table, lens, starts)
    close(y, rotate64(q, pos, rotary))
    want = torch.zeros_like(vp)
    want[0, 0, :2] = v[2:4, 0]    # slots -2 and -1 are left out
    want[1, 0, :2] = v[6:8, 0]    # slots 6 and 7 lie in page 99
    want[3, 0, 4:] = v[8:12, 0]
    assert torch.equal(vp, want)


def test_append_captured(gpu_ca):
    rotary = gpu_ca.Rotary(32, device="cuda")
    kp, vp = (torch.zeros(8, 2, 4, 32, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    q, k, v = (torch.randn(3, 2, 32, device="cuda").bfloat16() for _ in range(3))
    table = torch.arange(8, dtype=torch.int32, device="cuda").view(2, 4)
    lens = torch.tensor([5, 9], dtype=torch.int32, device="cuda")
    starts = torch.tensor([0, 1, 3], dtype=torch.int32, device="cuda")
    pos = torch.arange(3, device="cuda")
    out = torch.empty_like(q)
    args = (q, k, v, pos, rotary, kp, vp, table, lens, starts)
    gpu_ca.rotary_append(*args, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gpu_ca.rotary_append(*args, out=out)
    for step in range(3):
        lens.add_(1)
        pos.add_(7)
        q.mul_(-1)
        kp.zero_(), vp.zero_()
        graph.replay()
        torch.cuda.synchronize()
        ke, ve = torch.zeros_like(kp), torch.zeros_like(vp)
        assert torch.equal(out, gpu_ca.rotary_append(q, k, v, pos, rotary, ke, ve, table, lens, starts))
        assert torch.equal(kp, ke) and torch.equal(vp, ve)


def test_saved_positions_moved_away(gpu_ca):
    """A saved-tensor hook that leaves the positions on the host: the backward
    reports it, from the native function and the Python one."""
    rotary = gpu_ca.Rotary(16, device="cuda")
    pos = torch.arange(5, device="cuda")
    for q in (torch.randn(5, 2, 16, device="cuda", requires_grad=True),
              torch.randn(5, 2, 16, 2, device="cuda")[..., 0].requires_grad_()):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: t):
            y, _ = gpu_ca.rotary_embedding(q, None, pos, rotary)
        with pytest.raises(RuntimeError, match="same GPU"):
            y.sum().backward()
        with torch.autograd.graph.save_on_cpu():
            y, _ = gpu_ca.rotary_embedding(q, None, pos, rotary)
        y.sum().backward()
        close(q.grad, rotate64(torch.ones_like(q), pos, rotary, inverse=True))


def test_positions_changed_before_the_backward(gpu_ca):
    rotary = gpu_ca.Rotary(16, device="cuda")
    pos = torch.arange(5, device="cuda")
    q = torch.randn(5, 2, 16, device="cuda", requires_grad=True)
    y, _ = gpu_ca.rotary_embedding(q, None, pos, rotary)
    pos.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_training_pass_captured(gpu_ca):
    """Forward and backward in one graph, replayed with other values."""
    rotary = gpu_ca.Rotary(32, layout="half", device="cuda")
    q, k = (torch.randn(20, h, 32, device="cuda").bfloat16().requires_grad_() for h in (4, 2))
    pos = torch.arange(20, device="cuda")
    gq, gk = torch.randn_like(q), torch.randn_like(k)

    def step():
        yq, yk = gpu_ca.rotary_embedding(q, k, pos, rotary)
        return [yq.detach(), yk.detach(), *torch.autograd.grad([yq, yk], [q, k], [gq, gk])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for _ in range(3):
        with torch.no_grad():
            q.mul_(-1.5)
            k.add_(1.0)
        pos.add_(1000)
        gq.neg_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))

"""The generation operators without a GPU: argument errors of the Python entry
points and of the C ABI (before any launch), the CPU path against 64 bits, the
cache's bookkeeping, the page division."""
import ctypes
import math

import numpy as np
import pytest
import torch

from paged_case import attend, attention64, make_cache, rows_of


def test_paged_attention_on_the_cpu(ca):
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        for lengths, new, group in (([1], [1], 1), ([40, 7, 100], [3, 0, 20], 2), ([3, 9], [5, 1], 1)):
            case = make_cache(lengths, new, group=group, D=16, page=7, dtype=dtype, seed=1)
            y, want, tol = attention64(case, with_sums=True)
            sums = torch.zeros(len(lengths), 2, max(lengths))
            out = attend(ca, case, weight_sums=sums)
            assert (np.abs(out.double().numpy() - y) <= tol).all()
            for (b, h), w in want.items():
                assert np.allclose(sums[b, h, :len(w)].numpy(), w, rtol=1e-4, atol=1e-6)
    case = make_cache([40], [2], D=16, page=8, dtype=torch.float32, seed=2)
    case["table"][0, 2] = -1
    assert torch.isnan(attend(ca, case)).all()


def test_paged_attention_refusals(ca):
    base = make_cache([40, 9], [2, 1], heads=2, group=2, D=16, page=8, dtype=torch.float32)

    def refused(match, error=ValueError, **change):
        kw = {n: change.pop(n) for n in ("max_new", "max_length", "weight_sums", "out") if n in change}
        with pytest.raises(error, match=match):
            attend(ca, {**base, **change}, **kw)

    refused("q must be", q=base["q"][0])
    refused("q is", q=base["q"].bfloat16())
    refused("head dim", q=torch.randn(3, 4, 8))
    refused("query heads", q=base["q"][:, :3])
    refused("unsupported cache dtype", q=base["q"].double(), k=base["k"].double(), v=base["v"].double())
    refused("share shape", v=base["v"][:, :1])
    refused("share shape", v=base["v"].transpose(2, 3).contiguous().transpose(2, 3))
    refused("32-bit", table=base["table"].long())
    refused("32-bit", lengths=base["lengths"].long())
    refused("lengths has shape", lengths=base["lengths"][:1])
    refused("starts has shape", starts=base["starts"][:2])
    refused("log_gain", gain=base["gain"][:1])
    refused("contiguous", table=base["table"].t().contiguous().t())
    refused("contiguous", k=base["k"].transpose(2, 3), v=base["v"].transpose(2, 3))
    refused("must not be negative", max_new=-1)
    refused("must not be negative", max_length=-1)
    refused("weight_sums must be fp32", weight_sums=torch.zeros(2, 2, 40, dtype=torch.float64))
    refused("weight_sums must be fp32", weight_sums=torch.zeros(2, 3, 40))
    refused("out must have", out=torch.empty(3, 4, 16, dtype=torch.bfloat16))
    refused("share memory", out=base["q"])
    refused("apart", out=torch.empty(1, 4, 16).expand(3, 4, 16))
    refused("apart", weight_sums=torch.zeros(1, 2, 40).expand(2, 2, 40))
    refused("no backward pass", RuntimeError, q=base["q"].clone().requires_grad_())
    refused("no backward pass", RuntimeError, gain=base["gain"].clone().requires_grad_())
    with torch.no_grad():
        attend(ca, {**base, "gain": base["gain"].clone().requires_grad_()})
    wide = make_cache([9], [1], D=136, dtype=torch.float32)
    with pytest.raises(ValueError, match="head dim 136"):
        attend(ca, wide)
    narrow = make_cache([9], [1], D=12, dtype=torch.float32)
    with pytest.raises(ValueError, match="head dim 12"):
        attend(ca, narrow)
    meta = {n: t.to("meta") if isinstance(t, torch.Tensor) else t for n, t in base.items()}
    with pytest.raises(RuntimeError, match="ROCm GPU and CPU"):
        attend(ca, meta)
    none = make_cache([9], [0], D=16, dtype=torch.float32)
    assert attend(ca, none).shape == (0, 2, 16)


def rotate(x, pos, rotary):
    R = rotary.rotary_dim
    f = (rotary.turns * 2 * math.pi).numpy()
    z = rotary.magnitude * np.exp(1j * pos.double().numpy()[:, None, None] * f)
    y = x.double().numpy().copy()
    if rotary.layout == "interleaved":
        c = (y[..., 0:R:2] + 1j * y[..., 1:R:2]) * z
        y[..., 0:R:2], y[..., 1:R:2] = c.real, c.imag
    else:
        c = (y[..., :R // 2] + 1j * y[..., R // 2:R]) * z
        y[..., :R // 2], y[..., R // 2:R] = c.real, c.imag
    return y


@pytest.mark.parametrize("layout", ["interleaved", "half"])
@pytest.mark.parametrize("kw", [{}, {"scaling": "linear", "factor": 4.0}, {"scaling": "ntk", "factor": 4.0},
                                {"scaling": "yarn", "factor": 4.0, "original_length": 128}])
def test_rotary_on_the_cpu(ca, layout, kw):
    rotary = ca.Rotary(24, rotary_dim=16, layout=layout, **kw)
    q = torch.randn(7, 3, 24, requires_grad=True)
    k = torch.randn(7, 1, 24, requires_grad=True)
    pos = torch.arange(7) * 100000
    yq, yk = ca.rotary_embedding(q, k, pos, rotary)
    # cos, sin to 2^-24, two products and a sum
    for y, x in ((yq, q), (yk, k)):
        assert np.abs(y.detach().numpy() - rotate(x.detach(), pos, rotary)).max() <= 8 * 2.0 ** -24 * rotary.magnitude * 6
    g = torch.randn_like(yq)
    (dq,) = torch.autograd.grad(yq, q, g)
    assert np.abs(dq.numpy() - rotate(g, -pos, rotary)).max() <= 8 * 2.0 ** -24 * rotary.magnitude * 6


def test_rotary_frequencies(ca):
    """The scalings at their ends: what is kept, what is divided."""
    plain = ca.Rotary(64).turns
    assert torch.equal(ca.Rotary(64, scaling="linear", factor=4.0).turns, plain / 4)
    ntk = ca.Rotary(64, scaling="ntk", factor=4.0).turns
    assert ntk[0] == plain[0] and abs(ntk[-1] * 4 / plain[-1] - 1) < 1e-12
    yarn = ca.Rotary(64, scaling="yarn", factor=4.0, original_length=4096)
    turns = plain * 4096
    assert torch.equal(yarn.turns[turns >= 32], plain[turns >= 32])
    assert torch.allclose(yarn.turns[turns <= 1], plain[turns <= 1] / 4, rtol=1e-15)
    assert ((yarn.turns <= plain) & (yarn.turns >= plain / 4)).all()
    assert yarn.magnitude == 0.1 * math.log(4.0) + 1.0
    own = ca.Rotary(8, frequencies=[1.0, 0.5, 0.25, 0.0], magnitude=2.0)
    assert own.magnitude == 2.0 and torch.equal(own.turns, torch.tensor([1, 0.5, 0.25, 0], dtype=torch.float64) / (2 * math.pi))


def test_rotary_refusals(ca):
    for kw, match in (({"head_dim": 7}, "even"), ({"head_dim": 8, "rotary_dim": 10}, "even"),
                      ({"head_dim": 8, "rotary_dim": 3}, "even"), ({"head_dim": 8, "layout": "x"}, "layout"),
                      ({"head_dim": 8, "scaling": "x"}, "scaling"), ({"head_dim": 8, "theta": 0}, "theta"),
                      ({"head_dim": 8, "factor": 0.5}, "factor"), ({"head_dim": 2, "scaling": "ntk"}, "ntk"),
                      ({"head_dim": 8, "scaling": "yarn"}, "original_length"),
                      ({"head_dim": 8, "frequencies": [1.0]}, "frequencies")):
        with pytest.raises(ValueError, match=match):
            ca.Rotary(**kw)
    rotary = ca.Rotary(8)
    q, pos = torch.randn(3, 2, 8), torch.arange(3)
    for args, match in (((q[0], None, pos, rotary), "heads, head_dim"), ((q[..., :6], None, pos, rotary), "head dim 6"),
                        ((q.double(), None, pos, rotary), "unsupported dtype"),
                        ((q, q.bfloat16(), pos, rotary), "share dtype"), ((q, q[:2], pos, rotary), "share dtype"),
                        ((q, None, pos.float(), rotary), "integers"), ((q, None, torch.arange(4), rotary), "do not fit"),
                        ((q, None, [0, 1, 2], rotary), "integers")):
        with pytest.raises(ValueError, match=match):
            ca.rotary_embedding(*args)
    case = make_cache([5, 4], [2, 1], D=8, page=4, dtype=torch.float32)
    tail = (case["k"], case["v"], case["table"], case["lengths"], case["starts"])
    k = torch.randn(3, 2, 8)
    for args, match in (((q, k, k[:, :1], pos, rotary) + tail, "share their shape"),
                        ((q.bfloat16(), k.bfloat16(), k.bfloat16(), pos, rotary) + tail, "the cache"),
                        ((q, k[:, :1], k[:, :1], pos, rotary) + tail, "heads and head dim"),
                        ((q, k, k, pos, rotary) + (case["k"], case["k"]) + tail[2:], "must be apart"),
                        ((q, k, k, pos, rotary) + tail[:-1] + (None,), "starts must be given")):
        with pytest.raises(ValueError, match=match):
            ca.rotary_append(*args)
    with pytest.raises(RuntimeError, match="no backward pass"):
        ca.rotary_append(q.requires_grad_(), k, k, pos, rotary, *tail)


def test_append_on_the_cpu(ca):
    rotary = ca.Rotary(8, layout="half")
    case = make_cache([5, 4], [2, 3], D=8, page=3, dtype=torch.float32)
    q, k, v = (torch.randn(6, 2, 8) for _ in range(3))
    pos = torch.arange(6) + 50
    out = torch.full((6, 2, 8), 3.0)
    ca.rotary_append(q, k, v, pos, rotary, case["k"], case["v"], case["table"], case["lengths"], case["starts"], out=out)
    yq, yk = ca.rotary_embedding(q, k, pos, rotary)
    assert torch.equal(out[:5], yq[:5]) and (out[5] == 3).all()
    for h in range(2):
        assert (rows_of(case, case["k"], 0, h, 5)[3:] == yk[:2, h].double().numpy()).all()
        assert (rows_of(case, case["v"], 1, h, 4)[1:] == v[2:5, h].double().numpy()).all()


def test_evict_on_the_cpu_and_refusals(ca):
    case = make_cache([9, 3], [0, 0], D=8, page=4, dtype=torch.float32, spare=4)
    sums = torch.tensor([[[0, 5, 1, 5, 2, float("nan"), 0, 1, 0]] * 2, [[1.0] * 9] * 2])
    new = case["spare"].view(2, 2)
    kept, lens, s = ca.evict(case["k"], case["v"], case["table"], case["lengths"], sums, new, 5, sinks=1, recent=1)
    assert kept.tolist() == [[[0, 1, 3, 5, 8]] * 2, [[0, 1, 2, -1, -1]] * 2] and lens.tolist() == [5, 3]
    assert torch.equal(s[0, 0].isnan(), torch.tensor([False, False, False, True, False])) and s[1, 0].tolist() == [1, 1, 1, 0, 0]
    now = {**case, "table": new}
    assert (rows_of(now, case["v"], 0, 1, 5) == rows_of(case, case["v"], 0, 1, 9)[[0, 1, 3, 5, 8]]).all()
    base = dict(k_pages=case["k"], v_pages=case["v"], page_table=case["table"], lengths=case["lengths"], weight_sums=sums,
                new_table=new, budget=5)
    for change, match in (({"budget": 0}, "budget"), ({"sinks": -1}, "budget"), ({"sinks": 3, "recent": 3}, "budget"),
                          ({"budget": 9}, "do not hold"), ({"new_table": new.long()}, "32-bit"),
                          ({"new_table": new[:1]}, "new_table has shape"), ({"weight_sums": sums.double()}, "weight_sums"),
                          ({"weight_sums": sums[:, :1]}, "weight_sums"), ({"lengths": case["lengths"].long()}, "32-bit")):
        with pytest.raises(ValueError, match=match):
            ca.evict(**{**base, **change})


def test_int4_on_the_cpu_and_refusals(ca):
    codes = torch.randint(0, 16, (10, 77), dtype=torch.uint8)
    scales, zeros = torch.rand(10, 3), torch.randint(0, 16, (10, 3))
    w = ca.Int4Weight.from_codes(codes, scales, zeros, 32)
    group = torch.arange(77) // 32
    d = (codes.double() - zeros.double()[:, group]) * scales.double()[:, group]
    assert torch.equal(w.dequantize().double(), ((codes.float() - zeros.float()[:, group]) * scales[:, group]).double())
    x = torch.randn(4, 77)
    assert ((ca.int4_linear(x, w).double() - x.double() @ d.t()).abs() <= 100 * 2.0 ** -24 * (x.double().abs() @ d.abs().t())).all()
    for fn, match in ((lambda: ca.Int4Weight.from_codes(codes, scales, zeros, 48), "groups"),
                      (lambda: ca.Int4Weight.from_codes(codes.float(), scales, zeros, 32), "integers"),
                      (lambda: ca.Int4Weight.from_codes(codes, scales[:, :2], None, 32), "scales"),
                      (lambda: ca.Int4Weight(w.codes[:, :, :3], w.scales, None, 10, 77, 32), "codes"),
                      (lambda: ca.Int4Weight(w.codes, w.scales.double(), None, 10, 77, 32), "scales"),
                      (lambda: ca.int4_linear(x[:, :70], w), "columns"),
                      (lambda: ca.int4_linear(x.bfloat16(), w), "scales are")):
        with pytest.raises(ValueError, match=match):
            fn()
    with pytest.raises(RuntimeError, match="no backward pass"):
        ca.int4_linear(x.requires_grad_(), w)
    with pytest.raises(ValueError, match="no bias"):
        ca.Int4Linear.from_linear(torch.nn.Linear(4, 4))


def test_c_abi_refusals(ca):
    """Errors before any HIP call; the pointers are never followed."""
    lib = ca.native.load()
    p = 4096

    def cache(**kw):
        c = ca.native.PagedCache()
        for n in ("k", "v", "table", "lengths", "starts"):
            setattr(c, n, p)
        c.page_stride, c.head_stride, c.row_stride, c.table_stride = 4096, 1024, 64, 8
        c.dtype, c.heads, c.head_dim, c.page_size, c.num_pages, c.pages_per_seq, c.batch, c.tokens = 1, 4, 64, 16, 9, 8, 2, 3
        for n, x in kw.items():
            setattr(c, n, x)
        return c

    def attn(c, q=p, qs=(256, 64), heads=4, out=p, ws=None, nb=0, max_new=1, max_length=128, gain=p):
        return lib.ca_paged_attention(ctypes.byref(c) if c else None, q, *qs, heads, gain, out, 256, 64, None, 0, 0, 0,
                                      max_new, max_length, ws, nb, None)

    bad = [dict(k=None), dict(table=None), dict(starts=None), dict(batch=0), dict(heads=0), dict(page_size=0),
           dict(num_pages=0), dict(pages_per_seq=0), dict(tokens=-1), dict(dtype=9), dict(k=p + 4), dict(row_stride=60),
           dict(table_stride=7), dict(lengths=p + 2)]
    for kw in bad:
        assert attn(cache(**kw)) == 1, kw
        assert lib.ca_last_error()
    assert attn(None) == 1
    for kw in (dict(head_dim=12), dict(head_dim=136), dict(pages_per_seq=1 << 30, table_stride=1 << 30)):
        assert attn(cache(**kw)) == 2, kw
    assert attn(cache(), heads=3) == 1
    assert attn(cache(), q=p + 2) == 1 and attn(cache(), qs=(255, 64)) == 1 and attn(cache(), q=None) == 1
    assert attn(cache(), max_new=-1) == 1 and attn(cache(), gain=p + 1) == 1
    need = lib.ca_paged_attention_workspace_bytes(1, 2, 4, 4, 64, 3, 1, 100000, 0)
    assert need > 0
    c = cache(pages_per_seq=10000, table_stride=10000)
    assert attn(c, max_length=100000) == 3
    assert attn(c, max_length=100000, ws=p, nb=need - 1) == 3
    assert attn(cache(tokens=0)) == 0  # nothing to do

    def ev(c, budget=16, sinks=0, recent=0, table=p, stride=1):
        return lib.ca_evict(ctypes.byref(c), p, 0, 0, 128, budget, sinks, recent, table, stride, p, p, p, None)

    assert ev(cache(), budget=0) == 1 and ev(cache(), sinks=9, recent=9) == 1 and ev(cache(), table=None) == 1
    assert ev(cache(), budget=17) == 1 and ev(cache(), stride=0) == 1 and ev(cache(heads=0)) == 1

    def rot(**kw):
        r = ca.native.Rotary()
        for n in ("q", "k", "q_out", "k_out", "positions", "turns"):
            setattr(r, n, p)
        r.dtype, r.tokens, r.q_heads, r.k_heads, r.head_dim, r.rotary_dim = 1, 3, 4, 4, 64, 64
        for n, x in kw.items():
            setattr(r, n, x)
        return r

    for kw in (dict(q=None), dict(k=None), dict(turns=None), dict(turns=p + 4), dict(rotary_dim=3), dict(rotary_dim=66),
               dict(rotary_dim=0), dict(dtype=7), dict(tokens=-1), dict(q_heads=0, k_heads=0), dict(positions=p + 1),
               dict(q=p + 1)):
        assert lib.ca_rotary_embedding(ctypes.byref(rot(**kw)), None) == 1, kw
    assert lib.ca_rotary_embedding(None, None) == 1
    assert lib.ca_rotary_append(ctypes.byref(rot(k_heads=2)), p, 256, 64, ctypes.byref(cache()), None) == 1
    assert lib.ca_rotary_append(ctypes.byref(rot(inverse=1)), p, 256, 64, ctypes.byref(cache()), None) == 1
    assert lib.ca_rotary_append(ctypes.byref(rot()), None, 256, 64, ctypes.byref(cache()), None) == 1

    def i4(x=p, codes=p, dtype=1, M=1, N=16, K=128, group=128, xs=128, ys=16):
        return lib.ca_int4_linear(x, xs, codes, p, None, p, ys, dtype, M, N, K, group, None)

    assert i4(x=None) == 1 and i4(codes=p + 4) == 1 and i4(dtype=5) == 1 and i4(N=0) == 1 and i4(K=0) == 1
    assert i4(M=-1) == 1 and i4(xs=127) == 1 and i4(ys=15) == 1 and i4(x=p + 1) == 1
    assert i4(group=48) == 2 and i4(group=0) == 2 and i4(M=1 << 20) == 2
    assert i4(M=0) == 0


def test_page_division():
    """Slot / page size by a product and a shift is exact below 2^31."""
    rng = np.random.default_rng(0)
    for d in [1, 2, 3, 5, 7, 16, 24, 100, 127, 128, 129, 1000, 4097, 65535, 2 ** 20 - 1, 2 ** 30] + list(rng.integers(1, 2 ** 30, 50)):
        d = int(d)
        l = (d - 1).bit_length()
        mul = -(-(1 << (31 + l)) // d)
        assert mul < 1 << 32
        n = {0, 1, d - 1, d, d + 1, 2 ** 31 - 1, 2 ** 31 - 2} | {int(x) for x in rng.integers(0, 2 ** 31, 200)}
        n |= {k * d + e for k in (1, 2, 2 ** 31 // d - 1) for e in (-1, 0, 1)}
        for x in n:
            if 0 <= x < 2 ** 31:
                assert x * mul >> (31 + l) == x // d, (x, d)


def test_paged_cache_bookkeeping(ca):
    c = ca.PagedCache(1, 2, 1, 8, 20, pages=7, page_size=4, dtype=torch.float32, device="cpu", weight_sums=True)
    assert c.max_length == 20 and c.k(0).shape == (7, 1, 4, 8)
    c.extend([5, 0])
    assert c.lengths.tolist() == [5, 0] and c.starts.tolist() == [0, 5, 5] and c.positions.tolist() == [0, 1, 2, 3, 4]
    c.extend([3, 6])
    assert c.lengths.tolist() == [8, 6] and c.positions.tolist() == [5, 6, 7, 0, 1, 2, 3, 4, 5] and c.max_new == 6
    assert len(c.free) == 3 and len(set(c.owned[0] + c.owned[1])) == 4
    with pytest.raises(ValueError, match="exceed"):
        c.extend([13, 0])
    with pytest.raises(RuntimeError, match="out of pages"):
        c.extend([12, 6])
    assert c.counts == [8, 6] and len(c.free) == 3
    with pytest.raises(ValueError, match="counts"):
        c.extend([1])
    c.weight_sums.uniform_()
    c.evict(4)
    assert c.counts == [4, 4] and c.next == [8, 6] and len(c.free) == 5 and c.lengths.tolist() == [4, 4]
    assert (c.weight_sums[..., 4:] == 0).all() and len(set(c.owned[0] + c.owned[1] + c.free)) == 7
    c.extend([1, 1])
    assert c.positions.tolist() == [8, 6]
    c.release(0)
    assert c.counts[0] == 0 and c.next[0] == 0 and len(c.free) == 5
    tight = ca.PagedCache(1, 1, 1, 8, 12, pages=3, page_size=4, dtype=torch.float32, device="cpu", weight_sums=True)
    tight.extend([12])
    with pytest.raises(RuntimeError, match="no free pages"):
        tight.evict(4)
    assert tight.counts == [12] and len(tight.owned[0]) == 3 and not tight.free
    with pytest.raises(ValueError, match="without weight_sums"):
        ca.PagedCache(1, 1, 1, 8, 12, device="cpu").evict(4)


def test_tables_and_strides_that_would_be_read_past_their_ends(ca):
    case = make_cache([9, 3], [1, 1], D=8, page=4, dtype=torch.float32, spare=4)
    sums = torch.ones(2, 2, 9)
    with pytest.raises(ValueError, match="new_table rows must not overlap"):
        ca.evict(case["k"], case["v"], case["table"], case["lengths"], sums, case["spare"][:2].view(1, 2).expand(2, -1), 5)
    one = case["table"][:1].expand(2, -1)
    with pytest.raises(ValueError, match="page_table rows must not overlap"):
        ca.evict(case["k"], case["v"], one, case["lengths"], sums, case["spare"].view(2, 2), 5)
    with pytest.raises(ValueError, match="page_table rows must not overlap"):
        attend(ca, {**case, "table": one})
    lib = ca.native.load()
    c = ca.native.PagedCache()
    for n in ("k", "v", "table", "lengths", "starts"):
        setattr(c, n, 4096)
    c.dtype, c.heads, c.head_dim, c.page_size, c.num_pages, c.pages_per_seq, c.batch, c.tokens = 1, 4, 64, 16, 9, 8, 2, 3
    for n in ("page_stride", "head_stride", "row_stride"):
        c.page_stride, c.head_stride, c.row_stride, c.table_stride = 4096, 1024, 64, 8
        setattr(c, n, -64)
        assert lib.ca_paged_attention(ctypes.byref(c), 4096, 256, 64, 4, 4096, 4096, 256, 64, None, 0, 0, 0, 1, 128,
                                      None, 0, None) == 1
        assert b"negative strides" in lib.ca_last_error()
    c.row_stride, c.batch = 64, 1 << 20  # 2^22 (sequence, head)s
    assert lib.ca_paged_attention(ctypes.byref(c), 4096, 256, 64, 4, 4096, 4096, 256, 64, None, 0, 0, 0, 1, 128,
                                  None, 0, None) == 2
    assert lib.ca_evict(ctypes.byref(c), 4096, 0, 0, 128, 16, 0, 0, 4096, 1, 4096, 4096, 4096, None) == 2


def test_plans_of_any_size(ca):
    """Workspace sizes, which follow the plan of the grid, up to the limits."""
    lib = ca.native.load()
    for dtype in (0, 1, 2):
        for batch, tokens, new in ((1, 1, 1), (1, 1 << 20, 1 << 20), (1 << 18, 1 << 18, 1), (4096, 1 << 20, 64),
                                   (1, 1 << 20, 64), (3, 1 << 30, 1 << 30)):
            for length in (0, 1, 33, 1 << 17, 1 << 24, 1 << 30):
                n = lib.ca_paged_attention_workspace_bytes(dtype, batch, 8, 8, 64, tokens, new, length, 0)
                assert 0 <= n <= max(1 << 30, lib.ca_workspace_cap())

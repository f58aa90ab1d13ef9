"""paged_attention on the GPU against the oracle in 64 bits: types, widths,
ragged lengths from one slot up, groups, pages that end inside a tile, strides,
masks, bad page numbers, streams, captures."""
import numpy as np
import pytest
import torch

from paged_case import attend, attention64, make_cache, on_gpu

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def check(ca, case, **kw):
    y, _, tol = attention64(case)
    g = on_gpu(case)
    out = attend(ca, g, **kw)
    assert out.dtype == case["q"].dtype and out.shape == case["q"].shape
    err = np.abs(out.double().cpu().numpy() - y)
    assert (err <= tol).all(), f"error {err.max():.3g}, {np.max(err / tol):.3g} of the tolerance"
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,new", [([1], [1]), ([2], [2]), ([29], [1]), ([30], [1]), ([31], [3]),
                                         ([61], [61]), ([300], [1]), ([1, 64, 200], [1, 0, 7]),
                                         ([513, 3, 90], [40, 2, 90]), ([1000], [130])])
def test_lengths(gpu_ca, dtype, lengths, new):
    print(f"[case] {lengths} {new} {dtype}", flush=True)
    check(gpu_ca, make_cache(lengths, new, dtype=dtype, seed=len(lengths) + lengths[0]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("D", [8, 24, 32, 40, 80, 96, 128])
@pytest.mark.parametrize("new", [1, 35])
def test_head_dims(gpu_ca, dtype, D, new):
    print(f"[case] {D} {new} {dtype}", flush=True)
    check(gpu_ca, make_cache([150, 77], [new, 1], D=D, dtype=dtype, seed=D))


@pytest.mark.parametrize("page", [1, 7, 16, 33, 256])
@pytest.mark.parametrize("group,new", [(1, 1), (4, 1), (3, 9), (16, 1), (17, 1), (5, 30)])
def test_pages_and_groups(gpu_ca, page, group, new):
    print(f"[case] page {page} group {group} new {new}", flush=True)
    check(gpu_ca, make_cache([130, 45], [new, 1], group=group, page=page, seed=page + group))


@pytest.mark.parametrize("dtype", TYPES)
def test_hints_size_the_grid_and_nothing_else(gpu_ca, dtype):
    """Too small, exact and too large expectations give the same values up to
    the order of sums, in one split or many."""
    case = make_cache([2000, 700, 5], [20, 1, 5], dtype=dtype, seed=3)
    for kw in ({}, {"max_new": 20, "max_length": 2000}, {"max_new": 1, "max_length": 1},
               {"max_new": 0, "max_length": 0}, {"max_new": 1, "max_length": 100000}):
        print(f"[case] {kw}", flush=True)
        check(gpu_ca, case, **kw)


def test_large_scores_and_equal_keys(gpu_ca):
    """Scores far apart (weights of one key, segments by their closed form) and
    all alike (series at zero)."""
    check(gpu_ca, make_cache([400], [33], dtype=torch.float32, scale=4.0, seed=5))
    case = make_cache([200], [3], dtype=torch.bfloat16, seed=6)
    case["k"].copy_(case["k"][:1, :, :1].expand_as(case["k"]).clone())
    check(gpu_ca, case)


def test_scores_all_far_below_zero(gpu_ca):
    """The running maximum starts from the first tile, not from zero."""
    case = make_cache([100], [2], dtype=torch.float32, seed=7)
    case["q"].fill_(30.0)
    case["k"].fill_(-30.0).add_(0.01 * torch.randn(case["k"].shape))
    check(gpu_ca, case)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(gpu_ca, dtype):
    """Token-major pages, q out of a wider projection, out into a wider row."""
    case = make_cache([75, 20], [3, 20], heads=4, dtype=dtype, seed=8, layout="token")
    y, _, tol = attention64(case)
    g = on_gpu(case)
    k = torch.empty(g["k"].shape[0], g["page"], 4, 64, device="cuda", dtype=dtype).transpose(1, 2)
    v = torch.empty(g["v"].shape[0], g["page"], 4, 64, device="cuda", dtype=dtype).transpose(1, 2)
    g["k"], g["v"] = k.copy_(g["k"]), v.copy_(g["v"])
    wide = torch.randn(23, 3, 4, 64, device="cuda").to(dtype)
    wide[:, 1] = g["q"]
    rows = torch.full((23, 4, 128), 7.0, device="cuda", dtype=dtype)
    g["q"] = wide[:, 1]
    out = attend(gpu_ca, g, out=rows[:, :, 64:])
    assert out.data_ptr() == rows[:, :, 64:].data_ptr()
    assert (np.abs(out.double().cpu().numpy() - y) <= tol).all()
    assert (rows[:, :, :64] == 7).all()
    # rows that do not start on 16 bytes, elements apart
    odd = torch.empty(23 * 4 * 64 + 1, device="cuda", dtype=dtype)[1:].view(23, 4, 64).copy_(wide[:, 1])
    g["q"] = odd
    assert torch.equal(attend(gpu_ca, g), out)
    spread = torch.empty(23, 4, 64, 2, device="cuda", dtype=dtype)[..., 0].copy_(odd)
    g["q"] = spread
    assert torch.equal(attend(gpu_ca, g), out)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("new", [1, 3, 40])
def test_nothing_leaks_from_behind(gpu_ca, dtype, new):
    """NaN and infinities behind the last slot, in other sequences' pages and in
    later new tokens do not reach a row that must not see them."""
    case = make_cache([100, 50], [new, 1], dtype=dtype, seed=9, spare=1)
    clean = on_gpu(case)
    want = attend(gpu_ca, clean)
    ids = case["table"][0].long()
    for bad in (float("nan"), float("inf"), -float("inf")):
        g = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in clean.items()}
        for p in (g["k"], g["v"]):
            p[ids[100 // 16], :, 100 % 16:] = bad   # behind the last slot of sequence 0
            p[case["spare"].long()] = bad
        assert torch.equal(attend(gpu_ca, g), want)
        if new > 1:
            # the last token's value, then its key: only its own row changes
            for name in ("v", "k"):
                h = {n: t.clone() if isinstance(t, torch.Tensor) else t for n, t in g.items()}
                h[name][ids[99 // 16], :, 99 % 16, 0] = bad
                got = attend(gpu_ca, h)
                assert torch.equal(got[:new - 1], want[:new - 1]) and torch.equal(got[new:], want[new:])
                # (a key whose score is minus infinity has weight e^-inf = 0: its row stays finite)
                if name == "v" or bad != bad:
                    assert not torch.isfinite(got[new - 1].float()).all(-1).any()
                if name == "v":  # one column
                    assert torch.equal(got[new - 1, :, 1:], want[new - 1, :, 1:])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [16, 48, 7])
@pytest.mark.parametrize("new,group", [(1, 1), (1, 2), (3, 1), (2, 4), (1, 16)])
def test_tiles_that_share_a_wave(gpu_ca, dtype, page, new, group):
    """A table wide enough that several tiles of keys share a wave's columns: the
    results, and keys behind the last slot that are not finite, which must not
    reach other tiles' columns."""
    print(f"[case] page {page} new {new} group {group} {dtype}", flush=True)
    case = make_cache([301, 70, 559], [new, 1, new], group=group, page=page, dtype=dtype, seed=page + new)
    wide = torch.zeros(3, -(-200000 // page), dtype=torch.int32)
    wide[:, :case["table"].shape[1]] = case["table"]
    want = check(gpu_ca, {**case, "table": wide})
    g = on_gpu({**case, "table": wide})
    for bad in (float("nan"), float("inf"), -float("inf")):
        for b, length in enumerate((301, 70, 559)):
            if length % page == 0:
                continue  # no slots behind the last one
            g["k"][case["table"][b, length // page].long(), :, length % page:] = bad
            g["v"][case["table"][b, length // page].long(), :, length % page:] = bad
        assert torch.equal(attend(gpu_ca, g), want)
    if new > 1:  # the last key of a sequence: only its own row may change
        page_id, slot = case["table"][0, 300 // page].long(), 300 % page
        for bad in (float("nan"), float("inf"), -float("inf")):
            for name in ("k", "v"):
                h = {**g, name: g[name].clone()}
                h[name][page_id, :, slot] = bad
                got = attend(gpu_ca, h)
                assert torch.equal(got[:new - 1], want[:new - 1]) and torch.equal(got[new:], want[new:])


def test_many_slots_for_each_sequence(gpu_ca):
    """The plan for a table whose pages may hold 2^30 slots, many rows each."""
    case = make_cache([100, 50], [40, 33], group=4, page=16, seed=3)
    for width in (1 << 16, 1 << 20):
        wide = torch.zeros(2, width, dtype=torch.int32)
        wide[:, :case["table"].shape[1]] = case["table"]
        check(gpu_ca, {**case, "table": wide})


@pytest.mark.parametrize("lengths,new", [([3, 40], [5, 2]), ([0, 40], [4, 1]), ([0, 0], [1, 1])])
def test_rows_that_see_nothing_are_zero(gpu_ca, lengths, new):
    """More new tokens than cached slots: the first see nothing."""
    case = make_cache(lengths, new, dtype=torch.bfloat16, seed=10)
    out = check(gpu_ca, case)
    for b, (l, n) in enumerate(zip(lengths, new)):
        t0 = case["starts"][b].item()
        assert (out[t0:t0 + max(0, n - l)] == 0).all()


def test_rows_behind_the_last_sequence_stay(gpu_ca):
    case = make_cache([40, 70], [2, 3], dtype=torch.float32, seed=11)
    g = on_gpu(case)
    want = attend(gpu_ca, g)
    g["q"] = torch.cat((g["q"], torch.full((4, 2, 64), float("nan"), device="cuda")))
    out = torch.full_like(g["q"], 5.0)
    attend(gpu_ca, g, out=out)
    assert torch.equal(out[:5], want) and (out[5:] == 5).all()


def test_bad_pages_and_counts_are_not_followed(gpu_ca):
    """Page numbers outside the cache: NaN for the rows that read them, the other
    sequences as they were.  Lengths and starts beyond the tensors are held to them."""
    for lengths, new in (([40, 600, 70], [2, 1, 3]), ([40, 600, 70], [2, 100, 3])):
        case = make_cache(lengths, new, dtype=torch.bfloat16, seed=12)
        g = on_gpu(case)
        sums = torch.zeros(3, 2, 640, device="cuda")
        want = attend(gpu_ca, g)
        for bad in (-1, 10 ** 6, 2 ** 31 - 1, -2 ** 31):
            g["table"] = case["table"].cuda()
            g["table"][1, 20] = bad  # slots 320..335
            out = attend(gpu_ca, g, weight_sums=sums)
            a, b = case["starts"][1].item(), case["starts"][2].item()
            assert torch.isnan(out[a:b]).all()
            assert torch.equal(out[:a], want[:a]) and torch.equal(out[b:], want[b:])
    g = on_gpu(make_cache([40, 70], [2, 3], dtype=torch.bfloat16, seed=13))
    g["lengths"] = torch.tensor([2 ** 31 - 1, -5], dtype=torch.int32, device="cuda")
    g["starts"] = torch.tensor([-7, 2, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    out = attend(gpu_ca, g)
    assert torch.isfinite(out[:2].float()).all() and (out[2:] == 0).all()


def test_shared_pages(gpu_ca):
    """Two sequences with a common prefix in the same pages, a page named twice,
    and their weight sums apart."""
    case = make_cache([100, 90], [2, 3], page=32, dtype=torch.bfloat16, seed=21)
    case["table"][1, :2] = case["table"][0, :2]
    case["table"][0, 2] = case["table"][0, 1]
    y, want, tol = attention64(case, with_sums=True)
    g = on_gpu(case)
    sums = torch.zeros(2, 2, 100, device="cuda")
    out = attend(gpu_ca, g, weight_sums=sums)
    assert (np.abs(out.double().cpu().numpy() - y) <= tol).all()
    for (b, h), w in want.items():
        # (weights add up to one per row: 2^-16 of them as in test_weight_sums)
        assert np.abs(sums[b, h, :len(w)].double().cpu().numpy() - w).max() <= 2.0 ** -16


def test_refusals_on_the_gpu(gpu_ca):
    """Calls that the native entries hand back are reported as on the CPU."""
    g = on_gpu(make_cache([40, 9], [2, 1], heads=2, group=2, D=16, page=8, dtype=torch.float32, seed=22))
    for change, kw, error, match in (
            ({"q": g["q"].clone().requires_grad_()}, {}, RuntimeError, "no backward pass"),
            ({"q": g["q"].bfloat16()}, {}, ValueError, "q is"),
            ({"table": g["table"].long()}, {}, ValueError, "32-bit"),
            ({"lengths": g["lengths"].cpu()}, {}, RuntimeError, "device"),
            ({"gain": g["gain"].cpu()}, {}, RuntimeError, "one device"),
            ({}, {"out": g["q"]}, ValueError, "share memory"),
            ({}, {"out": g["q"].clone()[:1].expand(3, 4, 16)}, ValueError, "apart"),
            ({}, {"max_new": -2}, ValueError, "negative"),
            ({}, {"weight_sums": torch.zeros(1, 2, 40, device="cuda").expand(2, 2, 40)}, ValueError, "apart")):
        with pytest.raises(error, match=match):
            attend(gpu_ca, {**g, **change}, **kw)
    # doubles in log_gain are taken, as are parameters without grad mode
    want = attend(gpu_ca, g)
    assert torch.equal(attend(gpu_ca, {**g, "gain": g["gain"].double()}), want)
    with torch.no_grad():
        assert torch.equal(attend(gpu_ca, {**g, "gain": torch.nn.Parameter(g["gain"])}), want)


def test_far_offsets(gpu_ca):
    """A cache of more than 2^32 bytes: pages at both its ends."""
    pages, page = 5000, 64
    k = torch.zeros(pages, 16, page, 64, device="cuda", dtype=torch.bfloat16)  # 655 MB each at 16 heads
    big = torch.empty(8, *k.shape, device="cuda", dtype=torch.bfloat16).view(8 * pages, 16, page, 64)
    assert big.numel() * 2 > 2 ** 32
    del k
    case = make_cache([150], [2], heads=16, page=64, dtype=torch.bfloat16, seed=14)
    far = torch.tensor([8 * pages - 1, 0, 8 * pages - 2], dtype=torch.int32)
    y, _, tol = attention64(case)
    g = on_gpu(case)
    big[far.long().cuda()] = g["k"][case["table"][0].long()]
    g["k"] = big
    vbig = torch.empty_like(big)
    vbig[far.long().cuda()] = g["v"][case["table"][0].long()]
    g["v"], g["table"] = vbig, far.cuda()[None]
    out = attend(gpu_ca, g)
    assert (np.abs(out.double().cpu().numpy() - y) <= tol).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("lengths,new,group", [([200, 31], [1, 1], 1), ([100, 64], [64, 9], 1), ([70, 1], [3, 1], 4),
                                               ([400], [100], 2), ([3], [5], 1)])
def test_weight_sums(gpu_ca, dtype, lengths, new, group):
    print(f"[case] {lengths} {new} {group} {dtype}", flush=True)
    case = make_cache(lengths, new, group=group, dtype=dtype, seed=15)
    y, want, tol = attention64(case, with_sums=True)
    g = on_gpu(case)
    base = torch.rand(len(lengths), 2, max(lengths) + 5, device="cuda")
    sums = base.clone()
    out = attend(gpu_ca, g, weight_sums=sums)
    assert (np.abs(out.double().cpu().numpy() - y) <= tol).all()
    assert torch.equal(out, attend(gpu_ca, g))
    rows = group * max(new)
    for (b, h), w in want.items():
        n = len(w)
        got = (sums - base)[b, h].double().cpu().numpy()
        # a weight's relative error as in attention64 with scores below 8 in size, 72 * 2^-24 of
        # their terms' sum (below 32) four times over, and a rounding of the sum for each row
        limit = w * (4 * 72 * 32 * 2.0 ** -24 + 64 * 2.0 ** -24 + rows * 2.0 ** -24) + 2.0 ** -22 * (1 + w)
        assert (np.abs(got[:n] - w) <= limit).all()
        assert (got[n:] == 0).all()
    # a narrower tensor takes the slots it has
    narrow = base[..., :10].contiguous()
    attend(gpu_ca, g, weight_sums=narrow)
    assert torch.equal(narrow, sums[..., :10])


def test_two_calls_at_once(gpu_ca):
    """Two streams, each with its own outputs and workspaces."""
    cases = [on_gpu(make_cache([3000, 100], [1, 30], dtype=torch.bfloat16, seed=s)) for s in (16, 17)]
    want = [attend(gpu_ca, c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for _ in range(5):
        for c, s in zip(cases, streams):
            with torch.cuda.stream(s):
                got.append(attend(gpu_ca, c))
    torch.cuda.synchronize()
    for i, y in enumerate(got):
        assert torch.equal(y, want[i % 2])


def test_captured(gpu_ca):
    """One graph, replayed with other lengths, tables and tokens than captured."""
    a = on_gpu(make_cache([900, 40], [1, 1], dtype=torch.bfloat16, seed=18))
    sums = torch.zeros(2, 2, 1000, device="cuda")
    out = torch.zeros_like(a["q"])
    attend(gpu_ca, a, out=out, weight_sums=sums)  # sizes and library loaded
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        attend(gpu_ca, a, out=out, weight_sums=sums)
    for lengths in ([900, 40], [13, 600], [1, 1], [880, 640]):
        a["lengths"].copy_(torch.tensor(lengths, dtype=torch.int32))
        a["q"].mul_(-0.5)
        a["table"].random_(0, a["k"].shape[0])
        sums.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = torch.zeros_like(sums)
        assert torch.equal(out, attend(gpu_ca, a, weight_sums=eager))
        assert torch.equal(sums, eager)


def test_agrees_with_the_training_operator(gpu_ca):
    """Prompts of a batch through the cache, in chunks, are the causal operator."""
    B, H, T, D, page = 2, 3, 150, 64, 16
    q, k, v = (torch.randn(B, H, T, D, device="cuda") for _ in range(3))
    gain = 0.1 * torch.randn(H, device="cuda")
    want = gpu_ca.continuum_attention(q, k, v, gain)
    per = -(-T // page)
    pad = torch.nn.functional.pad
    pages = lambda x: pad(x, (0, 0, 0, per * page - T)).view(B, H, per, page, D).transpose(1, 2).reshape(B * per, H, page, D).contiguous()
    table = torch.arange(B * per, device="cuda", dtype=torch.int32).view(B, per)
    done = 0
    for n in (1, 16, 100, 33):
        done += n
        got = gpu_ca.paged_attention(q[:, :, done - n:done].transpose(1, 2).reshape(B * n, H, D), pages(k), pages(v), table,
                                     torch.full((B,), done, dtype=torch.int32, device="cuda"),
                                     torch.arange(0, B * n + 1, n, dtype=torch.int32, device="cuda"), gain)
        ref = want[:, :, done - n:done].transpose(1, 2).reshape(B * n, H, D)
        # two fp32 results, each within 2e-5 (scores below 32 in their terms' sum) of the exact one
        assert (got - ref).abs().max() <= 1e-4

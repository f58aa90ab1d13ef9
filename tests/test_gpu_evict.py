"""evict on the GPU against a selection by sorting: ties, NaN, infinities, signs,
sinks and recent slots, lengths around the budget, long rows."""
import numpy as np
import pytest
import torch

from paged_case import make_cache, rows_of

pytestmark = pytest.mark.gpu


def select(sums, n, budget, sinks, recent):
    """Kept slots of one row by the definition (numpy)."""
    if n <= budget:
        return np.arange(n)
    slot = np.arange(n)
    s = sums[:n].astype(np.float64)
    nan = np.isnan(s)
    s = np.where(nan, 0.0, s)
    always = (slot < sinks) | (slot >= n - recent)
    return np.sort(np.lexsort((slot, -s, ~nan, ~always))[:budget])


def check(ca, lengths, budget, sinks=0, recent=0, heads=2, D=32, page=16, dtype=torch.bfloat16, sums=None, seed=0):
    per = -(-budget // page)
    case = make_cache(lengths, [0] * len(lengths), heads=heads, D=D, page=page, dtype=dtype, seed=seed,
                      spare=per * len(lengths))
    if sums is None:
        g = torch.Generator().manual_seed(seed)
        sums = torch.exp(2 * torch.randn(len(lengths), heads, max(max(lengths), 1), generator=g))
    new_table = case["spare"].view(len(lengths), per)
    k, v = case["k"].cuda(), case["v"].cuda()
    s = sums.cuda()
    kept, lens, new_sums = ca.evict(k, v, case["table"].cuda(), case["lengths"].cuda(), s, new_table.cuda(), budget,
                                    sinks=sinks, recent=recent)
    assert kept.dtype == lens.dtype == torch.int32 and kept.shape == (len(lengths), heads, budget)
    assert lens.tolist() == [min(l, budget) for l in lengths]
    kept, new_sums = kept.cpu().numpy(), new_sums.cpu()
    old = {"table": case["table"], "page": page}
    new = {"table": new_table, "page": page}
    used = [p for b, n in enumerate(lengths) for p in case["table"][b, :-(-n // page)].tolist()]
    for b, n in enumerate(lengths):
        m = min(n, budget)
        for h in range(heads):
            want = select(sums[b, h].numpy(), n, budget, sinks, recent)
            assert (kept[b, h, :m] == want).all(), (b, h)
            assert (kept[b, h, m:] == -1).all() and (new_sums[b, h, m:] == 0).all()
            assert torch.equal(new_sums[b, h, :m].view(torch.int32), sums[b, h][torch.from_numpy(want)].view(torch.int32))
            if m:
                for pages, now in ((case["k"], k.cpu()), (case["v"], v.cpu())):
                    assert (rows_of(new, now, b, h, m) == rows_of(old, pages, b, h, n)[want]).all()
    # the old pages stay
    for p in used:
        assert torch.equal(k[p].cpu(), case["k"][p]) and torch.equal(v[p].cpu(), case["v"][p])
    # rows behind the kept ones of the last new page, too
    return k, case


@pytest.mark.parametrize("dtype,D", [(torch.float32, 8), (torch.bfloat16, 64), (torch.float16, 128), (torch.bfloat16, 40)])
@pytest.mark.parametrize("lengths,budget", [([1], 1), ([2], 1), ([10, 3, 7], 7), ([64, 65, 66], 65), ([500, 0, 90], 100),
                                            ([1025, 1024], 1024), ([3000], 17)])
def test_lengths(gpu_ca, dtype, D, lengths, budget):
    print(f"[case] {lengths} {budget} {dtype} {D}", flush=True)
    check(gpu_ca, lengths, budget, dtype=dtype, D=D, seed=budget)


@pytest.mark.parametrize("sinks,recent", [(0, 0), (4, 0), (0, 30), (4, 96), (50, 50), (100, 0), (0, 100), (1, 98)])
@pytest.mark.parametrize("page", [1, 16, 100])
def test_sinks_and_recent(gpu_ca, sinks, recent, page):
    check(gpu_ca, [101, 350, 99, 2000], 100, sinks, recent, page=page, seed=sinks)


def test_ties_signs_and_specials(gpu_ca):
    """Equal sums keep the first; NaN is the largest; infinities, negative
    values, both zeros and denormals are in order."""
    n = 1500
    g = torch.Generator().manual_seed(1)
    few = torch.tensor([0.0, -0.0, 1.0, -1.0, float("inf"), -float("inf"), 1e-42, -1e-42, 3e38, 0.5])
    rows = [torch.zeros(n), torch.full((n,), 2.5), few[torch.randint(0, len(few), (n,), generator=g)],
            torch.where(torch.rand(n, generator=g) < 0.02, float("nan"), torch.rand(n, generator=g)),
            torch.full((n,), float("nan")), 1.0 + 2.0 ** -23 * torch.randint(0, 3, (n,), generator=g)]
    sums = torch.stack(rows).view(3, 2, n)
    for budget, sinks, recent in ((1, 0, 0), (700, 0, 0), (1499, 3, 5), (700, 10, 90), (40, 0, 0)):
        print(f"[case] {budget} {sinks} {recent}", flush=True)
        check(gpu_ca, [n, n - 1, n], budget, sinks, recent, sums=sums, seed=2)


@pytest.mark.parametrize("n,budget", [(24576, 5000), (24577, 24576), (70001, 60000)])
def test_long_rows(gpu_ca, n, budget):
    """Past what the selection holds in shared memory."""
    check(gpu_ca, [n], budget, 4, 100, heads=1, D=8, page=64, seed=n)


def test_bad_pages_and_lengths(gpu_ca):
    """Sources outside the cache become NaN, such targets are not written; lengths
    are held to the table and the sums."""
    k = torch.randn(8, 1, 4, 8, device="cuda")
    v = torch.randn_like(k)
    k0 = k.clone()
    table = torch.tensor([[0, 77], [1, 2]], dtype=torch.int32, device="cuda")
    new = torch.tensor([[3, 4], [-9, 6]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([2 ** 31 - 1, 8], dtype=torch.int32, device="cuda")
    sums = torch.ones(2, 1, 8, device="cuda")
    kept, n, _ = gpu_ca.evict(k, v, table, lens, sums, new, 6)
    assert n.tolist() == [6, 6] and kept[0, 0].tolist() == list(range(6))
    assert torch.equal(k[3, 0], k0[0, 0]) and torch.isnan(k[4, 0, :2]).all() and torch.equal(k[4, 0, 2:], k0[4, 0, 2:])
    assert torch.equal(k[6, 0, :2], k0[2, 0, :2])
    for p in (0, 1, 2, 5, 7):
        assert torch.equal(k[p], k0[p])
    kept, n, _ = gpu_ca.evict(k, v, table, torch.full_like(lens, -3), sums, new, 6)
    assert n.tolist() == [0, 0] and (kept == -1).all()
    kept, n, _ = gpu_ca.evict(k, v, table, lens, sums[:, :, :3], new, 6)
    assert n.tolist() == [3, 3]


def test_captured(gpu_ca):
    case = make_cache([400, 90], [0, 0], D=32, seed=4, spare=8)
    k, v, table = case["k"].cuda(), case["v"].cuda(), case["table"].cuda()
    new = case["spare"].view(2, 4).cuda()
    lens = case["lengths"].cuda()
    sums = torch.rand(2, 2, 400, device="cuda")
    gpu_ca.evict(k, v, table, lens, sums, new, 64, 2, 8)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = gpu_ca.evict(k, v, table, lens, sums, new, 64, 2, 8)
    for n in ([400, 90], [70, 10], [300, 64]):
        lens.copy_(torch.tensor(n, dtype=torch.int32))
        sums.uniform_()
        graph.replay()
        torch.cuda.synchronize()
        kk = k.clone()
        want = gpu_ca.evict(k, v, table, lens, sums, new, 64, 2, 8)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(kk, k)

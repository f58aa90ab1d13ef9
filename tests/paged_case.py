"""Paged caches for tests and their results in 64 bits (numpy, the oracle's
weights), with the tolerances the kernels' arithmetic allows."""
import numpy as np
import torch

from oracle import ca_oracle as O

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_cache(lengths, new, heads=2, group=1, D=64, page=16, dtype=torch.bfloat16, seed=0, scale=1.0,
               spare=0, layout="head"):
    """CPU tensors of a cache whose sequences' pages are scattered over the pool.
    layout "token": pages stored [page_size, heads] with the heads inside."""
    g = torch.Generator().manual_seed(seed)
    needs = [max(1, -(-l // page)) for l in lengths]
    total = sum(needs) + spare
    order = torch.randperm(total, generator=g).to(torch.int32)
    table = torch.zeros(len(lengths), max(needs), dtype=torch.int32)
    at = 0
    for b, m in enumerate(needs):
        table[b, :m] = order[at:at + m]
        at += m
    shape = (total, heads, page, D) if layout == "head" else (total, page, heads, D)
    k, v = ((scale * torch.randn(shape, generator=g)).to(dtype) for _ in range(2))
    if layout == "token":
        k, v = k.transpose(1, 2), v.transpose(1, 2)
    tokens = sum(new)
    q = (scale * torch.randn(tokens, heads * group, D, generator=g)).to(dtype)
    starts = torch.tensor([0] + list(np.cumsum(new)), dtype=torch.int32)
    gain = 0.2 * torch.randn(heads * group, generator=g)
    return {"q": q, "k": k, "v": v, "table": table, "lengths": torch.tensor(lengths, dtype=torch.int32),
            "starts": starts, "gain": gain, "page": page, "group": group, "spare": order[at:]}


def rows_of(case, pages, b, h, length):
    slot = torch.arange(length)
    ids = case["table"][b].long()[slot // case["page"]]
    return pages[ids, h, slot % case["page"]].double().numpy()


def attention64(case, with_sums=False):
    """(y [tokens, heads, D], sums of the new tokens' weights per (b, key head) or
    None, tolerance like y)."""
    q, G = case["q"], case["group"]
    N, H, D = q.shape
    kv = case["k"].shape[1]
    y, tol = np.zeros((N, H, D)), np.zeros((N, H, D))
    sums = {}
    half = HALF_STEP[q.dtype]
    for b, length in enumerate(case["lengths"].tolist()):
        t0, t1 = case["starts"][b].item(), case["starts"][b + 1].item()
        for h in range(kv):
            k, v = rows_of(case, case["k"], b, h, length), rows_of(case, case["v"], b, h, length)
            total = np.zeros(length)
            for g in range(G):
                head = h * G + g
                c = np.exp(float(case["gain"][head])) / np.sqrt(D)
                for t in range(t0, t1):
                    pos = length - (t1 - t)
                    if pos < 0:
                        continue
                    qr = q[t, head].double().numpy()
                    s = c * (k[:pos + 1] @ qr)
                    w = O.ca_weights(s[None], qidx=np.array([pos]))[0][0]
                    y[t, head] = w @ v[:pos + 1]
                    total[:pos + 1] += w
                    # a score of D fp32 products, scaled: (D + 4) roundings of its terms'
                    # sum; a weight follows its own and its neighbours' errors, the
                    # normalised one twice as far; the segment formulas and the sums of
                    # weights add some 64 roundings; 16-bit weights are two limbs
                    ds = (D + 4) * 2.0 ** -24 * c * np.max(np.abs(k[:pos + 1]) @ np.abs(qr))
                    mag = w @ np.abs(v[:pos + 1])
                    limbs = 0.0 if q.dtype == torch.float32 else 2.0 ** -16
                    tol[t, head] = mag * (4 * ds + 64 * 2.0 ** -24 + limbs) + half * np.abs(y[t, head]) + 1e-30
            sums[b, h] = total
    # 16-bit outputs below the normal range round to the type's least step
    if q.dtype == torch.float16:
        tol += 2.0 ** -25
    return y, sums if with_sums else None, tol


def on_gpu(case):
    return {n: t.cuda() if isinstance(t, torch.Tensor) else t for n, t in case.items()}


def attend(ca, case, **kw):
    return ca.paged_attention(case["q"], case["k"], case["v"], case["table"], case["lengths"], case["starts"],
                              case["gain"], **kw)

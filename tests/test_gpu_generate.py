"""The generation operators together, as a program uses them: a decoder's prompt
and tokens through the cache against its whole forward pass, eviction in the
middle, 4-bit weights, two caches on two streams."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def make_model(ca, d=64, heads=4, layers=2, vocab=50, device="cuda"):
    torch.manual_seed(0)
    cfg = ca.decoder.ContinuumDecoderConfig(vocab_size=vocab, block_size=256, d_model=d, n_heads=heads, n_layers=layers)
    model = ca.decoder.ContinuumDecoderLM(cfg).to(device)
    with torch.no_grad():
        for p in model.parameters():
            p.mul_(2.0)  # so that attention matters
    return model


# fp32 logits of two layers in two orders of sums; scores of a few units, values and logits of
# about one: hidden values agree to some 2^-20 after each of six products, logits to 1e-4
LOGIT_TOL = 1e-4


@pytest.mark.parametrize("chunks", [[40], [1] * 12, [17, 1, 1, 1, 20], [30, 64, 1]])
def test_chunks_are_the_forward_pass(gpu_ca, chunks):
    model = make_model(gpu_ca)
    T = sum(chunks)
    ids = torch.randint(0, 50, (3, T), device="cuda")
    with torch.no_grad():
        want = model(ids)["logits"]
    cache = model.make_cache(3, T, page_size=16)
    done = 0
    for n in chunks:
        got = model.forward_cached(ids[:, done:done + n], cache).view(3, n, -1)
        assert (got - want[:, done:done + n]).abs().max() <= LOGIT_TOL
        done += n


def test_ragged_batch(gpu_ca):
    """Sequences that come and go at their own pace."""
    model = make_model(gpu_ca, d=96, heads=2)
    lens = [50, 3, 21]
    seqs = [torch.randint(0, 50, (1, n), device="cuda") for n in lens]
    with torch.no_grad():
        want = [model(s)["logits"][0] for s in seqs]
    cache = model.make_cache(3, 64, page_size=8)
    at = [0, 0, 0]
    for new in ([20, 1, 0], [0, 2, 1], [29, 0, 20], [1, 0, 0]):
        flat = torch.cat([s[0, a:a + n] for s, a, n in zip(seqs, at, new)])
        got = model.forward_cached(flat, cache, new)
        t = 0
        for b, n in enumerate(new):
            assert n == 0 or (got[t:t + n] - want[b][at[b]:at[b] + n]).abs().max() <= LOGIT_TOL
            at[b] += n
            t += n
    assert at == lens
    cache.release(1)
    got = model.forward_cached(seqs[1][0], cache, [0, 3, 0])
    assert (got - want[1]).abs().max() <= LOGIT_TOL
    with pytest.raises(ValueError, match="counts"):
        model.forward_cached(seqs[1][0], cache, [0, 1])
    with pytest.raises(ValueError, match="new"):
        model.forward_cached(seqs[1][0], cache)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_half_types(gpu_ca, dtype):
    """Autocast, as the decoder trains: logits within the type's roundings of the
    whole pass (six products, each off by half a step of values of about one,
    through two layers)."""
    model = make_model(gpu_ca)
    ids = torch.randint(0, 50, (2, 60), device="cuda")
    cache = model.make_cache(2, 60, dtype=dtype)
    with torch.autocast("cuda", dtype=dtype), torch.no_grad():
        want = model(ids)["logits"].float()
        got = torch.cat([model.forward_cached(ids[:, :33], cache).view(2, 33, -1),
                         *(model.forward_cached(ids[:, t:t + 1], cache).view(2, 1, -1) for t in range(33, 60))], 1)
    scale = want.abs().max()
    assert (got.float() - want).abs().max() <= 16 * torch.finfo(dtype).eps / 2 * scale


def test_generate_and_cpu(gpu_ca):
    """Greedy tokens are those of repeated whole passes, and the CPU path's."""
    model = make_model(gpu_ca)
    ids = torch.randint(0, 50, (2, 9), device="cuda")
    got = model.generate(ids, 6)
    whole = ids
    with torch.no_grad():
        for t in range(6):
            logits = model(whole)["logits"][:, -1]
            top = logits.topk(2).values
            nxt = logits.argmax(-1, keepdim=True)
            # equal up to rounding would be no test
            assert ((got[:, t:t + 1] == nxt) | (top[:, :1] - top[:, 1:] < 2 * LOGIT_TOL)).all()
            whole = torch.cat((whole, got[:, t:t + 1]), 1)
    cpu = make_model(gpu_ca, device="cpu")
    cache, host = model.make_cache(2, 20, page_size=4), cpu.make_cache(2, 20, page_size=4)
    for part in (ids[:, :5], ids[:, 5:6], ids[:, 6:]):
        a, b = model.forward_cached(part, cache), cpu.forward_cached(part.cpu(), host)
        assert (a.cpu() - b).abs().max() <= LOGIT_TOL


def test_eviction_in_the_middle(gpu_ca):
    """The cache after an eviction is the kept rows, positions go on, and the
    CPU path takes the same course."""
    model, cpu = make_model(gpu_ca), make_model(gpu_ca, device="cpu")
    ids = torch.randint(0, 50, (2, 90), device="cuda")
    caches = [m.make_cache(2, 96, page_size=8, weight_sums=True, pages=40) for m in (model, cpu)]
    for m, c, i in ((model, caches[0], ids), (cpu, caches[1], ids.cpu())):
        m.forward_cached(i[:, :64], c)
    a, b = caches
    assert (a.weight_sums.cpu() - b.weight_sums).abs().max() <= 1e-4 * 64
    # every token gives its heads a weight of one
    assert torch.allclose(a.weight_sums.sum(-1), torch.full_like(a.weight_sums.sum(-1), 64.0), rtol=1e-5)
    b.weight_sums.copy_(a.weight_sums)  # the same ranking in both
    for m, c, i in ((model, a, ids), (cpu, b, ids.cpu())):
        c.evict(24, sinks=2, recent=8)
        assert c.counts == [24, 24] and c.next == [64, 64]
    la = [model.forward_cached(ids[:, 64:80], a), model.forward_cached(ids[:, 80:81], a)]
    lb = [cpu.forward_cached(ids[:, 64:80].cpu(), b), cpu.forward_cached(ids[:, 80:81].cpu(), b)]
    for x, y in zip(la, lb):
        assert (x.cpu() - y).abs().max() <= 2 * LOGIT_TOL
    assert a.counts == [41, 41] and a.positions.tolist() == [80, 80]


def test_int4_weights(gpu_ca):
    """The quantized decoder's cached pass is its whole pass."""
    model = make_model(gpu_ca)
    gpu_ca.quantize_linears(model.blocks, 32, zero_points=True)
    assert all(isinstance(b.mlp.fc1, gpu_ca.Int4Linear) for b in model.blocks)
    ids = torch.randint(0, 50, (2, 30), device="cuda")
    with torch.no_grad():
        want = model(ids)["logits"]
        cache = model.make_cache(2, 30)
        got = torch.cat([model.forward_cached(ids[:, :29], cache).view(2, 29, -1),
                         model.forward_cached(ids[:, 29:], cache).view(2, 1, -1)], 1)
    assert (got - want).abs().max() <= LOGIT_TOL


def test_two_caches_on_two_streams(gpu_ca):
    model = make_model(gpu_ca)
    ids = [torch.randint(0, 50, (1, 40), device="cuda") for _ in range(2)]
    with torch.no_grad():
        want = [model(i)["logits"][0] for i in ids]
    model.forward_cached(ids[0][:, :1], model.make_cache(1, 4))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ids]
    caches, got = [], [[], []]
    for s in streams:
        with torch.cuda.stream(s):
            caches.append(model.make_cache(1, 40, page_size=16))
    for a, b in ((0, 30), (30, 31), (31, 40)):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(model.forward_cached(ids[i][:, a:b], caches[i]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert (torch.cat(g) - w).abs().max() <= LOGIT_TOL

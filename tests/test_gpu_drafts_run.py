"""Steps of drafted tokens as they are used together: trees through a layer's attention, verification, kept rows, and the next step behind them; an image in a prompt and
tokens behind it; the same step captured and replayed."""
import numpy as np
import pytest
import torch

from qserve_b200 import backend
from tests.drafts_util import attention_seen64, random_parents, tree64, verify64
from tests.paged_util import BASE, D, F64, PAGE, Cache, check_attention
from tests.test_gpu_paged_attention import SCALE, starts
from tests.test_gpu_paged_cache import rows
from tests.test_gpu_paged_tree import axis_of, check_rotation_at

pytestmark = pytest.mark.gpu


def empty_cache(B, hkv, bits, blocks, dev):
    c = Cache([0] * B, hkv, bits, dev, seed=1, extra_blocks=blocks - 1)
    for p in c.pools:
        p.fill_(255)  # every scale and zero that is not written is no number
    return c


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,most", [(8, 2, 4), (8, 2, 20), (4, 4, 16)])
def test_steps_of_trees(dev, bits, hq, hkv, most):
    """Three sequences, five steps of trees of unequal sizes.  The cache after each step is that of the accepted tokens alone: the accepted rows' keys and values, at
    their own depths, are found side by side, and the next step attends over them."""
    B, V = 3, 500
    rng = np.random.default_rng(bits + most)
    c = empty_cache(B, hkv, bits, 8, dev)
    cache = (PAGE, c.size, bits == 4, True)
    prompt = [70, 1, 33]
    q, k, v = rows(sum(prompt), hq, hkv, dev, seed=1)
    c.lengths.copy_(torch.tensor(prompt, dtype=torch.int32))
    backend.append_kv_cache(q, k, v, c.table, starts(prompt, dev), c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
    length = list(prompt)
    for step in range(5):
        new = [int(x) for x in rng.integers(1, most + 1, B)]
        new[0] = most
        T, cu = sum(new), starts(new, dev)
        parents = random_parents(rng, new, padded=False)
        up = torch.tensor(parents, dtype=torch.int32, device=dev)
        lengths = torch.tensor([a + n for a, n in zip(length, new)], dtype=torch.int32, device=dev)
        positions, visible = backend.draft_tree(up, cu, lengths, most)
        seen, at = tree64(parents, new, length)
        assert positions.tolist() == at
        q, k, v = rows(T, hq, hkv, dev, seed=10 + step)
        turned = backend.append_kv_cache_at(q, k, v, c.table, cu, lengths, positions, None, PAGE, c.size, D, BASE, bits == 4, True)
        check_rotation_at(turned, q, positions[None], torch.zeros(64, dtype=torch.long, device=dev))
        out = backend.paged_tree_attention(turned, c.table, cu, lengths, visible, most, 512, *cache)
        row = 0
        for b, n in enumerate(new):
            m = length[b] + n
            mask = torch.ones(n, m, dtype=torch.bool, device=dev)
            for i in range(n):
                for j in range(n):
                    mask[i, length[b] + j] = bool(seen[row + i] >> j & 1)
            check_attention(out[row:row + n], attention_seen64(turned[row:row + n], c.values(0, b, m), c.values(1, b, m), mask, SCALE), SCALE)
            row += n
        # the target's logits: of a random projection of the result, so that some drafts are its best ones
        g = torch.Generator().manual_seed(step)
        logits = (out.reshape(T, -1).float().cpu() @ torch.randn(hq * D, V, generator=g)).half().to(dev) * 2
        tokens = torch.randint(0, V, (T,), generator=g).to(dev)
        best = logits.float().argmax(-1)
        row = 0
        for n in new:
            for i in range(1, n):
                if rng.random() < 0.7:
                    tokens[row + i] = best[row + parents[row + i]]
            row += n
        coins, draws = torch.rand(T, generator=g).to(dev), torch.rand(B, generator=g).to(dev)
        heats = torch.tensor([0.0, 1.0, 0.5], device=dev)
        got = backend.verify_drafts(logits, tokens, cu, most, coins, draws, parents=up, temperatures=heats)
        want = verify64(logits.double().cpu().numpy(), tokens.cpu().numpy(), new, coins.double().cpu().numpy(), draws.double().cpu().numpy(), parents, None, heats.tolist(), most)
        assert np.array_equal(got[0].cpu().numpy(), want[0]) and np.array_equal(got[1].cpu().numpy(), want[1]) and got[2].tolist() == want[2].tolist()
        before = [[c.values(which, b, length[b] + n) for b, n in enumerate(new)] for which in (0, 1)]
        kept = backend.keep_kv_cache(c.table, cu, lengths, got[1], got[2], *cache)
        for b in range(B):
            count = int(want[2][b])
            order = list(range(length[b])) + [length[b] + int(r) for r in want[1][b][:count]]
            length[b] += count
            for which in (0, 1):
                assert torch.equal(c.values(which, b, length[b]), before[which][b][order])
        assert kept.tolist() == length
    # one token a sequence behind them, through the operator of plain steps
    q, k, v = rows(B, hq, hkv, dev, seed=99)
    lengths = kept + 1
    turned = backend.append_kv_cache(q, k, v, c.table, None, lengths, PAGE, c.size, D, BASE, bits == 4, True)
    out = backend.shared_prefix_attention(turned, c.table, lengths, 0, 512, *cache)
    for b in range(B):
        m = length[b] + 1
        check_attention(out[b:b + 1], attention_seen64(turned[b:b + 1], c.values(0, b, m), c.values(1, b, m), torch.ones(1, m, dtype=torch.bool, device=dev), SCALE), SCALE)


def test_a_chain_without_a_tree(dev):
    """Drafted chains with the operators of portions: append, prompt attention, verification with the draft's probabilities; what was not accepted is written over."""
    hq, hkv, B, n, V = 8, 2, 2, 5, 300
    c = empty_cache(B, hkv, 4, 4, dev)
    cache = (PAGE, c.size, True, True)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    cu = starts([n] * B, dev)
    g = torch.Generator().manual_seed(3)
    for step in range(6):
        q, k, v = rows(B * n, hq, hkv, dev, seed=step)
        held = lengths + n
        turned = backend.append_kv_cache(q, k, v, c.table, cu, held, PAGE, c.size, D, BASE, True, True)
        out = backend.paged_prompt_attention(turned, c.table, cu, held, n, 256, *cache)
        for b in range(B):
            m = int(held[b])
            seen = torch.arange(m, device=dev)[None] <= torch.arange(m - n, m, device=dev)[:, None]
            check_attention(out[b * n:(b + 1) * n], attention_seen64(turned[b * n:(b + 1) * n], c.values(0, b, m), c.values(1, b, m), seen, SCALE), SCALE)
        logits = (out.reshape(B * n, -1).float().cpu() @ torch.randn(hq * D, V, generator=g)).to(dev)
        probs = torch.softmax(logits + torch.randn(B * n, V, generator=g).to(dev), -1)
        tokens = torch.multinomial(probs.cpu(), 1, generator=g)[:, 0].roll(1).to(dev)
        tokens_out, rows_out, counts = backend.verify_drafts(logits, tokens, cu, n, torch.rand(B * n, generator=g).to(dev), torch.rand(B, generator=g).to(dev), draft_probs=probs)
        kept = backend.keep_kv_cache(c.table, cu, held, rows_out, counts, *cache)
        assert torch.equal(kept, lengths + counts) and ((counts >= 1) & (counts <= n)).all()
        for b in range(B):  # rows of a chain are kept where they are
            assert rows_out[b].tolist() == list(range(int(counts[b]))) + [-1] * (n - int(counts[b]))
        lengths = kept


def test_a_captured_step(dev):
    """The whole step in one graph: its lengths, tokens and random numbers change on the device, and each replay goes on from what the one before it kept."""
    hq, hkv, B, n, V = 8, 2, 2, 6, 700
    parents = [-1, 0, 0, 1, 1, 2] * B
    c, e = empty_cache(B, hkv, 4, 4, dev), empty_cache(B, hkv, 4, 4, dev)
    up, cu = torch.tensor(parents, dtype=torch.int32, device=dev), starts([n] * B, dev)
    x = [t.clone() for t in rows(B * n, hq, hkv, dev, seed=0)]
    head = torch.randn(hq * D, V, generator=torch.Generator().manual_seed(1)).half().to(dev)
    tokens, coins, draws = torch.zeros(B * n, dtype=torch.int64, device=dev), torch.zeros(B * n, device=dev), torch.zeros(B, device=dev)

    def step(cache, lengths):
        held = lengths + n
        positions, visible = backend.draft_tree(up, cu, held, n)
        turned = backend.append_kv_cache_at(*x, cache.table, cu, held, positions, None, PAGE, cache.size, D, BASE, True, True)
        out = backend.paged_tree_attention(turned, cache.table, cu, held, visible, n, 256, PAGE, cache.size, True, True)
        logits = out.view(B * n, -1) @ head
        result = backend.verify_drafts(logits, tokens, cu, n, coins, draws, parents=up)
        lengths.copy_(backend.keep_kv_cache(cache.table, cu, held, result[1], result[2], PAGE, cache.size, True, True))
        return (out, logits, *result)

    a, b = (torch.full((B,), 3, dtype=torch.int32, device=dev) for _ in range(2))
    for cache in (c, e):  # three positions to begin with
        q, k, v = rows(B * 3, hq, hkv, dev, seed=7)
        backend.append_kv_cache(q, k, v, cache.table, starts([3] * B, dev), a, PAGE, cache.size, D, BASE, True, True)
    warm = torch.full((B,), 3, dtype=torch.int32, device=dev)
    step(e, warm)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(c, a)
    a.fill_(3)
    g = torch.Generator().manual_seed(5)
    for i in range(12):
        for t, s in zip(x, rows(B * n, hq, hkv, dev, seed=20 + i)):
            t.copy_(s)
        tokens.copy_(torch.randint(0, V, (B * n,), generator=g))
        coins.copy_(torch.rand(B * n, generator=g) * 0.01)  # drafts are often taken
        draws.copy_(torch.rand(B, generator=g))
        graph.replay()
        eager = step(e, b)
        assert torch.equal(a, b)
        for s, t in zip(captured, eager):
            assert torch.equal(s, t)
    assert (a > 3 + 12).any()


def test_an_image_in_a_prompt(dev):
    """Text, an image of 6 x 8 that sees itself as a whole, text; then single tokens at the places that text goes on from, which lie behind the cache's."""
    hq, hkv = 8, 2
    c = empty_cache(1, hkv, 8, 4, dev)
    cache = (PAGE, c.size, False, True)
    text, h, w, rest = 10, 6, 8, 7
    n = text + h * w + rest
    places = [[i] * 3 for i in range(text)] + [[text, text + r, text + s] for r in range(h) for s in range(w)] + [[text + max(h, w) + i] * 3 for i in range(rest)]
    positions = torch.tensor(places, dtype=torch.int32, device=dev).t().contiguous()
    image = ((1 << (h * w)) - 1) << text
    seen = [(1 << (i + 1)) - 1 | (image if text <= i < text + h * w else 0) for i in range(n)]
    words = torch.tensor([[(s >> (64 * k)) & (2 ** 64 - 1) for k in range(2)] for s in seen], dtype=torch.uint64).view(torch.int64).to(dev)
    q, k, v = rows(n, hq, hkv, dev, seed=4)
    cu, lengths = starts([n], dev), torch.tensor([n], dtype=torch.int32, device=dev)
    axes = torch.tensor(axis_of((16, 24, 24), False), device=dev)
    turned = backend.append_kv_cache_at(q, k, v, c.table, cu, lengths, positions, (16, 24, 24), PAGE, c.size, D, BASE, False, True)
    check_rotation_at(turned, q, positions, axes)
    out = backend.paged_tree_attention(turned, c.table, cu, lengths, words, n, n, *cache)
    mask = torch.tensor([[bool(s >> j & 1) for j in range(n)] for s in seen], device=dev)
    check_attention(out, attention_seen64(turned, c.values(0, 0, n), c.values(1, 0, n), mask, SCALE), SCALE)
    for i in range(3):
        lengths += 1
        at = torch.full((3, 1), text + max(h, w) + rest + i, dtype=torch.int32, device=dev)
        q, k, v = rows(1, hq, hkv, dev, seed=50 + i)
        turned = backend.append_kv_cache_at(q, k, v, c.table, None, lengths, at, (16, 24, 24), PAGE, c.size, D, BASE, False, True)
        check_rotation_at(turned, q, at, axes)
        out = backend.shared_prefix_attention(turned, c.table, lengths, 0, 256, *cache)
        m = n + i + 1
        check_attention(out, attention_seen64(turned, c.values(0, 0, m), c.values(1, 0, m), torch.ones(1, m, dtype=torch.bool, device=dev), SCALE), SCALE)

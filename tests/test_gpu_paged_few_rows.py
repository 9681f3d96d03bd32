"""Attention with a mask among the new rows for portions of few rows, whose codes go into the products as they lie: layouts, clusters over long caches, keys that are no
numbers, ends of types, batches of unequal portions, graphs."""
import numpy as np
import pytest
import torch

from qserve_b200 import backend
from tests.drafts_util import attention_seen64, words_of
from tests.paged_util import D, F64, HALF, PAGE, Cache, check_attention
from tests.test_gpu_paged_attention import SCALE, queries, starts
from tests.test_gpu_paged_tree import attend, attend64, masks

pytestmark = pytest.mark.gpu

FEW = [  # query heads, key/value heads, new rows, positions held ahead of them: 16 rows a key/value head at most
    (16, 1, [1], [0]),
    (16, 1, [1, 1], [31, 32]),
    (32, 8, [4, 1, 0, 3], [0, 31, 12, 33]),
    (8, 8, [16, 9], [63, 64]),
    (10, 2, [3, 2, 1], [500, 0, 65]),            # five heads
    (14, 2, [2, 2], [100, 1]),                   # seven heads
    (4, 4, [16], [5000]),                        # a cluster over the keys
    (8, 2, [4, 4], [20000, 3]),                  # clusters of sixteen, one of them with next to nothing
    (32, 8, [4] * 40, list(range(0, 4000, 100))),
    (64, 64, [2, 5], [300, 250]),
    (12, 4, [5], [1]),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kind", ["tree", "any", "all"])
@pytest.mark.parametrize("hq,hkv,new,ahead", FEW, ids=lambda x: str(x)[:20])
def test_few_rows(dev, bits, kind, hq, hkv, new, ahead):
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=sum(lens) + hq)
    q, seen = queries(sum(new), hq, dev), masks(kind, new, sum(lens))
    out = attend(c, q, seen, new)
    check_attention(out, attend64(c, q, seen, new, lens), SCALE)
    ahead_of = [m for n, m in zip(new, ahead) for _ in range(n)]
    assert all(bool((out[t] == 0).all()) for t, (s, m) in enumerate(zip(seen, ahead_of)) if s == 0 and m == 0)


@pytest.mark.parametrize("bits", [4, 8])
def test_sharp_scores(dev, bits):
    """Queries ten times as large: maxima grow along the walk, in one warp's half pages and not in another's."""
    new, lens = [4, 3], [1500, 333]
    c = Cache(lens, 2, bits, dev, seed=5)
    q, seen = queries(7, 8, dev) * 10, masks("tree", new, 2)
    check_attention(attend(c, q, seen, new, softmax_scale=0.05), attend64(c, q, seen, new, lens, 0.05), 0.05)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("value", [float("nan"), float("inf")])
@pytest.mark.parametrize("new,lens", [([4, 4], [340, 84]), ([4], [4]), ([3], [35]), ([4], [3000])])
def test_keys_that_are_no_numbers_reach_the_rows_that_see_them(dev, bits, value, new, lens):
    """One new row a portion with scales and zeros that are none: the rows with its bit give NaN, the others what they give where it has numbers, within the roundings."""
    c = Cache(lens, 2, bits, dev, seed=9)
    q = queries(sum(new), 8, dev)
    seen = [[1, 3, 5, 15][i] for n in new for i in range(n)]  # the second row sees row 1, the fourth too; the others not
    want = attend64(c, q, seen, new, lens)
    for b, n in enumerate(new):
        pos = lens[b] - n + 1
        for which in (0, 1):
            c.meta(which)[c.pages[b, pos // PAGE], :, :, pos % PAGE] = value
    got = attend(c, q, seen, new)
    for t, s in enumerate(seen):
        if s >> 1 & 1:
            assert torch.isnan(got[t]).all()
        else:
            check_attention(got[t:t + 1], [x[t:t + 1] for x in want], SCALE)
    # one of the cache reaches all
    c.meta(0)[c.pages[0, 0], :, :, 0] = float("nan")
    if lens[0] > new[0]:
        assert torch.isnan(attend(c, q, seen, new)[:new[0]]).all()


@pytest.mark.parametrize("bits", [4, 8])
def test_scales_of_every_size(dev, bits):
    """Values of 2^-14 to 65504 side by side: weights go with the largest scale, and a row that sees only the small ones loses nothing that fp16 holds."""
    new, lens = [4], [260]
    c = Cache(lens, 1, bits, dev, seed=3)
    g = torch.Generator().manual_seed(1)
    size = (2.0 ** torch.randint(-14, 12, (c.pools[1].shape[0], 1, PAGE), generator=g).float()).to(dev)
    held = torch.isfinite(c.meta(1)[:, 0])
    c.meta(1)[:, 0] = torch.where(held, (c.meta(1)[:, 0].float() * size / 8).half(), c.meta(1)[:, 0])
    q = queries(4, 4, dev)
    seen = [1, 3, 7, 15]
    out = attend(c, q, seen, new)
    o, absolute, spread, mass = attend64(c, q, seen, new, lens)
    # the weights' roundings go with the largest value of a row's, as check_attention's absolute bound counts them; the results are fp16
    check_attention(out, (o, absolute, spread, mass), SCALE)


def test_what_stays_as_it_was(dev):
    """Rows behind the last sequence and behind max_seqlen, results in place, queries inside wider rows, words beyond a portion's rows, a table that ends early."""
    new, lens = [3, 4, 2], [100, 2, 200]  # the second sequence holds fewer positions than its portion has rows
    c = Cache(lens, 2, 4, dev, seed=7)
    wide = torch.randn(12, 12, D, generator=torch.Generator().manual_seed(1)).half().to(dev)
    q = wide[:, 2:10]
    seen = masks("all", new, 1) + [0, 0, 0]
    words = words_of(seen, 2, dev)
    words[:, 1] = -1
    cu = starts(new, dev)
    out = torch.full((12, 8, D), 7.0, dtype=HALF, device=dev)
    backend.paged_tree_attention(q, c.table, cu, c.lengths, words, 4, 200, *c.args, out=out)
    assert (out[9:] == 7.0).all()
    want = attend64(c, q[:9], seen, new, lens)
    check_attention(out[:9], want, SCALE)
    out = torch.full((12, 8, D), 7.0, dtype=HALF, device=dev)
    backend.paged_tree_attention(q, c.table, cu, c.lengths, words, 2, 200, *c.args, out=out)
    assert (out[2] == 7.0).all() and (out[5:7] == 7.0).all()
    short = [s & 3 for s in seen]
    check_attention(out[:2], [x[:2] for x in attend64(c, q[:9], short, new, lens)], SCALE)
    narrow = c.table[:, :, :1].contiguous()
    got = backend.paged_tree_attention(q, narrow, cu, c.lengths, words, 4, 200, *c.args)
    check_attention(got[:3], attention_seen64(q[:3], c.values(0, 0, 64), c.values(1, 0, 64), torch.ones(3, 64, dtype=torch.bool, device=dev), SCALE), SCALE)
    kept = q.clone()
    got = backend.paged_tree_attention(q, c.table, cu, c.lengths, words, 4, 200, *c.args, out=q)
    assert got.data_ptr() == q.data_ptr() and torch.equal(got[9:], kept[9:])
    check_attention(got[:9], want, SCALE)
    # lengths at the ends of their type
    c.lengths.copy_(torch.tensor([-2 ** 31, 2, 200], dtype=torch.int32))
    got = backend.paged_tree_attention(kept, c.table, cu, c.lengths, words, 4, 200, *c.args)
    assert (got[:3] == 0).all()
    check_attention(got[3:9], [x[3:9] for x in want], SCALE)


def test_graphs_and_streams(dev):
    """Two captured calls of different clusters, replayed on two streams with other lengths and masks."""
    cases = []
    for bits, hq, hkv, new, lens in ((4, 8, 2, [4, 3], [4000, 700]), (8, 4, 4, [9, 16], [120, 300])):
        c = Cache(lens, hkv, bits, dev, seed=hq)
        q = queries(sum(new), hq, dev)
        words = words_of(masks("tree", new, 1), 1, dev)
        cu = starts(new, dev)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        call = lambda c=c, q=q, cu=cu, words=words, new=new, lens=lens: backend.paged_tree_attention(q, c.table, cu, c.lengths, words, max(new), max(lens), *c.args)
        call()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        cases.append((c, q, words, new, lens, stream, graph, out, call))
    for step, kind in enumerate(("tree", "any", "all")):
        for c, q, words, new, lens, *_ in cases:
            words.copy_(words_of(masks(kind, new, step), 1, dev))
            c.lengths.copy_(torch.tensor([m - 5 * step for m in lens], dtype=torch.int32))
        torch.cuda.synchronize()
        for _ in range(3):
            for *_, stream, graph, out, call in cases:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for c, q, words, new, lens, stream, graph, out, call in cases:
            assert torch.equal(out, call())
            check_attention(out, attend64(c, q, masks(kind, new, step), new, [m - 5 * step for m in lens]), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch", [1, 2, 3, 5, 6, 7, 9, 10, 11, 13, 15, 17])
def test_batches(dev, bits, batch):
    """Sequences share the device: each batch has blocks of its own number a sequence, some of which have a half page more than others or none."""
    new, ahead = [1 + (i + batch) % 4 for i in range(batch)], [(1000 + 397 * i) % 2500 for i in range(batch)]
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, 4, bits, dev, seed=batch)
    q, seen = queries(sum(new), 16, dev), masks("tree", new, batch)
    check_attention(attend(c, q, seen, new), attend64(c, q, seen, new, lens), SCALE)


MORE = [  # in small calls up to 64 tokens, 16 rows a block
    (32, 8, [13], [500]),
    (8, 2, [5, 0, 64, 33], [0, 12, 31, 200]),
    (14, 2, [9, 3], [63, 64]),                   # seven heads: tokens across blocks' borders
    (16, 1, [26, 1, 2], [700, 0, 65]),
    (40, 8, [5, 5, 4], [130, 1, 700]),
    (4, 4, [17], [2000]),
    (32, 8, [8] * 4, [900, 500, 100, 1]),
    (64, 64, [17], [1]),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kind", ["tree", "any", "all"])
@pytest.mark.parametrize("hq,hkv,new,ahead", MORE, ids=lambda x: str(x)[:20])
def test_more_rows_in_small_calls(dev, bits, kind, hq, hkv, new, ahead):
    test_few_rows(dev, bits, kind, hq, hkv, new, ahead)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,new,ahead", [(8, 2, [2, 4, 1], [13000, 12, 14001]), (4, 1, [3, 1, 4, 2, 4, 1, 4, 2, 3, 1], [13000] + [700 * i for i in range(9)])], ids=lambda x: str(x)[:20])
def test_few_long_sequences(dev, bits, hq, hkv, new, ahead):
    """Those are cut into more parts than a cluster has blocks, every sequence's alike."""
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=3)
    q, seen = queries(sum(new), hq, dev), masks("tree", new, 7)
    check_attention(attend(c, q, seen, new), attend64(c, q, seen, new, lens), SCALE)


def test_no_work_space_is_needed(dev):
    from qserve_b200._lib import lib
    need = lib.qs_paged_tree_attention_workspace_bytes
    assert need(1, 4, 4, 10000, 32, 8) == 0 and need(2, 8, 4, 60000, 32, 8) == 0 and need(8, 32, 4, 60000, 32, 8) == 0 and need(0, 4, 4, 100, 32, 8) == 0 and need(2, 4, 0, 100, 32, 8) == 0
    # more rows, and few rows of few long sequences: the prompt operator's
    for a in ((1, 24, 24, 60000, 32, 8), (1, 4, 4, 60000, 32, 8)):
        assert need(*a) == lib.qs_paged_prompt_attention_workspace_bytes(*a) > 0

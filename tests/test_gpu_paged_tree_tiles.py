"""Masked tiles of paged_tree_attention at their edges: portions of more than 64 rows, which no other kernel takes.  Keys and values that are no numbers behind the mask, rows
that are left, portions longer than their lengths, short tables, bits of rows that are not there, masks of nothing, captured steps, results over the queries."""
import pytest
import torch

from qserve_b200 import backend
from tests.drafts_util import attention_seen64, words_of
from tests.paged_util import D, PAGE, Cache, check_attention
from tests.test_gpu_paged_attention import SCALE, queries, starts
from tests.test_gpu_paged_tree import attend, attend64, masks

pytestmark = pytest.mark.gpu
HEADS = [(2, 2), (8, 2)]  # a row a token: one tile a block; four: two tiles


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("kind", ["tree", "any"])
@pytest.mark.parametrize("new,ahead", [([100, 20], [300, 64]), ([65, 128], [0, 63]), ([257], [1]), ([90, 70, 66], [2000, 5, 700])])
def test_keys_that_no_row_names_say_nothing(dev, bits, hq, hkv, kind, new, ahead):
    """New rows whose keys and values are no numbers reach those rows alone that have their bits; others are the same to the last bit."""
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=sum(lens))
    q, seen = queries(sum(new), hq, dev), masks(kind, new, sum(lens))
    clean = attend(c, q, seen, new)
    check_attention(clean, attend64(c, q, seen, new, lens), SCALE)
    for share in (2, 3):  # of the portion: inside it, and at its end
        bad = [n - 1 if share == 3 else n // share for n in new]
        for which in (0, 1):
            pools = [p.clone() for p in c.pools]
            for b, row in enumerate(bad):
                pos = lens[b] - new[b] + row
                c.meta(which)[c.pages[b, pos // PAGE], :, :, pos % PAGE] = float("nan")
            got, at = attend(c, q, seen, new), 0
            for b, (n, row) in enumerate(zip(new, bad)):
                names = torch.tensor([bool(s >> row & 1) for s in seen[at:at + n]], device=dev)
                assert torch.isnan(got[at:at + n][names]).all()
                assert torch.equal(got[at:at + n][~names], clean[at:at + n][~names])
                at += n
            for p, was in zip(c.pools, pools):
                p.copy_(was)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_pages_behind_the_last_row_that_is_seen(dev, bits, hq, hkv):
    """Rows that see little of a long portion: what lies behind it is not read as numbers; bits past the portion, and whole words of them, name nothing."""
    new, lens = [200, 130], [203, 700]
    c = Cache(lens, hkv, bits, dev, seed=3)
    q = queries(330, hq, dev)
    for last in (0, 62, 63, 64, 65, 127, 128, 129):
        seen = [(1 << min(i + 1, last + 1)) - 1 if i % 3 else 1 << min(i, last) for n in new for i in range(n)]
        pools = [p.clone() for p in c.pools]
        for b in range(2):
            for pos in range(lens[b] - new[b] + last + 1, lens[b]):
                for which in (0, 1):
                    c.meta(which)[c.pages[b, pos // PAGE], :, :, pos % PAGE] = float("nan")
        for stray in (False, True):
            words = words_of([s | (3 << 200 if stray and t < 200 else 5 << 130 if stray else 0) for t, s in enumerate(seen)], 6, dev)
            if stray:
                words[:, 4:] = -1
            out = backend.paged_tree_attention(q, c.table, starts(new, dev), c.lengths, words, 200, 700, *c.args)
            parts, at = [], 0
            for b, n in enumerate(new):
                first, held = lens[b] - n, lens[b] - n + last + 1
                mask = torch.ones(n, held, dtype=torch.bool, device=dev)
                mask[:, first:] = torch.tensor([[bool(s >> j & 1) for j in range(last + 1)] for s in seen[at:at + n]], device=dev)
                parts.append(attention_seen64(q[at:at + n], c.values(0, b, held), c.values(1, b, held), mask, SCALE))
                at += n
            check_attention(out, [torch.cat(x) for x in zip(*parts)], SCALE)
        for p, was in zip(c.pools, pools):
            p.copy_(was)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_masks_of_nothing(dev, bits, hq, hkv):
    """Rows without a bit see what lies ahead of their portion; where that is nothing, they get zeros."""
    new, lens = [80, 200, 0, 65], [80, 200, 0, 265]
    c = Cache(lens, hkv, bits, dev, seed=4)
    q = queries(345, hq, dev)
    seen = [0] * 345
    out = attend(c, q, seen, new)
    assert (out[:280] == 0).all()
    check_attention(out, attend64(c, q, seen, new, lens), SCALE)
    seen[100] = 1 << 150  # one row of a tile, and no other
    out = attend(c, q, seen, new)
    assert (out[:100] == 0).all() and (out[101:280] == 0).all()
    check_attention(out, attend64(c, q, seen, new, lens), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_rows_that_are_left_and_portions_longer_than_their_lengths(dev, bits, hq, hkv):
    new, lens = [80, 90, 70], [300, 66, 200]  # the second sequence holds fewer positions than its portion has rows
    c = Cache(lens, hkv, bits, dev, seed=7)
    total = sum(new)
    q, seen = queries(total + 3, hq, dev), masks("all", new, 1) + [0, 0, 0]
    words = words_of(seen, 2, dev)
    out = torch.full_like(q, 7.0)
    got = backend.paged_tree_attention(q, c.table, starts(new, dev), c.lengths, words, 90, 300, *c.args, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[total:] == 7.0).all()
    check_attention(out[:total], attend64(c, q[:total], seen, new, lens), SCALE)
    # rows behind max_seqlen are left, and are no keys of the others
    top = 67
    out = torch.full_like(q, 7.0)
    backend.paged_tree_attention(q, c.table, starts(new, dev), c.lengths, words, top, 300, *c.args, out=out)
    want = attend64(c, q[:total], [s & (1 << top) - 1 for s in seen], new, lens)
    at = 0
    for n in new:
        check_attention(out[at:at + top], [x[at:at + top] for x in want], SCALE)
        assert (out[at + top:at + n] == 7.0).all()
        at += n
    # fewer pages in the table than lengths speak of: the first and third portion lie behind it, and all that it holds lies ahead of them
    narrow = c.table[:, :, :2].contiguous()
    out = backend.paged_tree_attention(q[:total], narrow, starts(new, dev), c.lengths, words[:total], 90, 300, *c.args)
    for b, at, n in ((0, 0, 80), (2, 170, 70)):
        held = torch.ones(n, 2 * PAGE, dtype=torch.bool, device=dev)
        check_attention(out[at:at + n], attention_seen64(q[at:at + n], c.values(0, b, 2 * PAGE), c.values(1, b, 2 * PAGE), held, SCALE), SCALE)
    want = attend64(c, q[:total], seen, new, lens)
    check_attention(out[80:170], [x[80:170] for x in want], SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", HEADS)
def test_strides_words_and_graphs(dev, bits, hq, hkv):
    """Queries inside wider rows, more words than the portions need, results in place of the queries; captured and replayed with other masks."""
    new, lens = [133, 70], [700, 140]
    c = Cache(lens, hkv, bits, dev, seed=11)
    wide = torch.randn(203, hq + 4, D, generator=torch.Generator().manual_seed(1)).half().to(dev)
    q = wide[:, 2:2 + hq]
    seen = masks("any", new, 5)
    words = words_of(seen, 5, dev)
    words[:, 3:] = -1  # bits of rows that are not there
    cu = starts(new, dev)
    call = lambda **more: backend.paged_tree_attention(q, c.table, cu, c.lengths, words, 133, 700, *c.args, **more)
    want = attend64(c, q, seen, new, lens)
    check_attention(call(), want, SCALE)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    check_attention(out, want, SCALE)
    other = masks("tree", new, 6)
    words.copy_(words_of(other, 5, dev))
    graph.replay()
    want = attend64(c, q, other, new, lens)
    check_attention(out, want, SCALE)
    got = call(out=q)
    assert got.data_ptr() == q.data_ptr()
    assert torch.equal(got, out)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("new,ahead", [([300], [77]), ([70], [1500]), ([90, 70], [1500, 300]), ([129, 65, 200], [0, 63, 640])])
def test_a_causal_mask_is_the_prompt_operator_to_the_last_bit(dev, bits, new, ahead):
    """Both cut the keys alike where portions fill several blocks, or are one: what the masked rows weigh is nothing either way."""
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, 2, bits, dev, seed=4)
    q = queries(sum(new), 8, dev)
    out = attend(c, q, [(1 << (i + 1)) - 1 for n in new for i in range(n)], new)
    want = backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, max(new), max(lens), *c.args)
    assert torch.equal(out, want)

"""Tokens with places of their own in the paged cache against the definition in 64 bits: append at positions of one to four axes, attention with a mask among the new
rows, rows that are kept."""
import numpy as np
import pytest
import torch

from qserve_b200 import backend
from tests.drafts_util import attention_seen64, random_parents, tree64, words_of
from tests.paged_util import BASE, D, F64, H, PAGE, Cache, check_attention
from tests.test_gpu_paged_attention import SCALE, queries, starts
from tests.test_gpu_paged_cache import check_pages, rows

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------------------
# append at positions
# ------------------------------------------------------------------------------------------------------------------------
def axis_of(sections, interleaved):
    """The axis of each of a head's 64 pairs."""
    if not interleaved:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    return [i % len(sections) if i // len(sections) < sections[i % len(sections)] else 0 for i in range(64)]


def rotated_at(x, positions, axes):
    """x [T, heads, D], positions [A, T], the axis of each pair: in 64 bits."""
    angle = positions.to(F64)[axes].t() * BASE ** (-2.0 * torch.arange(D // 2, device=x.device, dtype=F64) / D)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.to(F64).chunk(2, -1)
    return torch.cat([c * a - s * b, c * b + s * a], -1)


def check_rotation_at(got, x, positions, axes):
    want = rotated_at(x, positions, axes)
    a, b = x.to(F64).abs().chunk(2, -1)
    room = H * want.abs() + (a + b).repeat(1, 1, 2) * 4 * 2.0 ** -24 + 2.0 ** -25
    assert ((got.to(F64) - want).abs() <= room * (1 + 1e-9)).all()


def append_at(c, q, k, v, new, positions, sections, interleaved=False, **more):
    cu = None if new is None else starts(new, c.dev)
    return backend.append_kv_cache_at(q, k, v, c.table, cu, c.lengths, positions, sections, PAGE, c.size, D, BASE, c.bits == 4, True, interleaved, **more)


SECTIONS = [((64,), False), ((16, 24, 24), False), ((24, 20, 20), True), ((1, 63), False), ((32, 32), True), ((16, 16, 16, 16), True), ((40, 0, 24), False), ((64, 0), True), ((10, 20, 4, 30), False)]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("sections,interleaved", SECTIONS)
@pytest.mark.parametrize("h,new,ahead", [(2, [5, 0, 130, 64], [60, 10, 1, 128]), (8, [1], [0]), (32, [33, 200], [500, 7])])
def test_append_at(dev, bits, sections, interleaved, h, new, ahead):
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, h, bits, dev, seed=sum(lens))
    T = sum(new)
    q, k, v = rows(T, h, h, dev, seed=T)
    g = torch.Generator().manual_seed(T)
    positions = torch.randint(-50, 300000, (len(sections), T), generator=g, dtype=torch.int32).to(dev)
    axes = torch.tensor(axis_of(sections, interleaved), device=dev)
    assert all(axis_of(sections, interleaved).count(a) == n for a, n in enumerate(sections))
    check_rotation_at(append_at(c, q, k, v, new, positions, sections, interleaved), q, positions, axes)
    turned = append_at(c, k, k, v, new, positions, sections, interleaved)  # the keys as queries: what is quantised, as it is rounded
    check_rotation_at(turned, k, positions, axes)
    check_pages(c, 0, turned, new, lens)
    check_pages(c, 1, v, new, lens)


@pytest.mark.parametrize("bits", [4, 8])
def test_append_at_the_rows_own_positions_is_append(dev, bits):
    new, lens = [70, 3, 9], [3000, 3, 64]
    q, k, v = rows(82, 8, 2, dev, seed=3)
    own = torch.cat([torch.arange(m - n, m, dtype=torch.int32) for n, m in zip(new, lens)]).to(dev)
    results = []
    for how in range(3):
        c = Cache(lens, 2, bits, dev, seed=1)
        if how == 0:
            out = backend.append_kv_cache(q, k, v, c.table, starts(new, dev), c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
        elif how == 1:
            out = append_at(c, q, k, v, new, own, None)
        else:
            out = append_at(c, q, k, v, new, own.expand(3, 82).contiguous(), (16, 24, 24))
        results.append((out, c.pools))
    for out, pools in results[1:]:
        assert torch.equal(out, results[0][0]) and all(torch.equal(a, b) for a, b in zip(pools, results[0][1]))


def test_append_at_single_tokens_strides_and_padded_batches(dev):
    """One row a sequence at places that lag behind the cache (an image takes fewer positions than rows); results in place; rows behind the last sequence."""
    c = Cache([500, 64, 1], 2, 4, dev, seed=2)
    q, k, v = rows(3, 8, 2, dev, seed=5)
    positions = torch.tensor([[300, 5, 0], [310, 9, 0], [320, 7, 0]], dtype=torch.int32, device=dev)
    axes = torch.tensor(axis_of((16, 24, 24), False), device=dev)
    before = q.clone()
    out = append_at(c, q, k, v, None, positions, (16, 24, 24), out=q)
    assert out.data_ptr() == q.data_ptr()
    check_rotation_at(out, before, positions, axes)
    check_pages(c, 1, v, [1, 1, 1], c.lens)
    c = Cache([70, 12], 2, 8, dev, seed=2)
    q, k, v = rows(9, 4, 2, dev, seed=6)
    positions = torch.arange(9, dtype=torch.int32, device=dev)
    out = torch.full((9, 4, D), 7.0, dtype=torch.half, device=dev)
    pools = [p.clone() for p in c.pools]
    append_at(c, q, k, v, [4, 2], positions, (64,), out=out)
    assert (out[6:] == 7.0).all()
    check_rotation_at(out[:6], q[:6], positions[None, :6], torch.zeros(64, dtype=torch.long, device=dev))
    check_pages(c, 1, v[:6], [4, 2], c.lens)
    held = torch.zeros(c.pools[0].shape[0], PAGE, dtype=torch.bool, device=dev)
    for b, (n, m) in enumerate(((4, 70), (2, 12))):
        for pos in range(m - n, m):
            held[c.pages[b, pos // PAGE], pos % PAGE] = True
    was = pools[0][:, :c.cut].view(-1, 2, PAGE, D)
    now = c.pools[0][:, :c.cut].view(-1, 2, PAGE, D)
    assert torch.equal(was.transpose(1, 2)[~held], now.transpose(1, 2)[~held])


# ------------------------------------------------------------------------------------------------------------------------
# attention with a mask among the new rows
# ------------------------------------------------------------------------------------------------------------------------
def attend(c, q, seen, new, **more):
    words = (max(max(new), 1) + 63) // 64
    return backend.paged_tree_attention(q, c.table, starts(new, c.dev), c.lengths, words_of(seen, words, c.dev), max(new), max(c.lens), *c.args, **more)


def attend64(c, q, seen, new, lens, scale=SCALE):
    parts, at = [], 0
    for b, (n, m) in enumerate(zip(new, lens)):
        m = max(m, 0)
        mask = torch.ones(n, m, dtype=torch.bool, device=c.dev)
        for i in range(n):
            for j in range(n):
                if lens[b] - n + j >= 0:
                    mask[i, lens[b] - n + j] = bool(seen[at + i] >> j & 1)
        parts.append(attention_seen64(q[at:at + n], c.values(0, b, m), c.values(1, b, m), mask, scale))
        at += n
    return [torch.cat(x) for x in zip(*parts)]


def masks(kind, new, seed):
    rng = np.random.default_rng(seed)
    if kind == "tree":
        return tree64(random_parents(rng, new), new, [0] * len(new))[0]
    if kind == "any":  # each row sees each with a probability of its own, no matter which lies ahead; some see nothing
        return [sum(1 << j for j in range(n) if rng.random() < p) for n in new for p in [0.0 if rng.random() < 0.2 else rng.random() for _ in range(n)]]
    return [(1 << n) - 1 for n in new for _ in range(n)]  # all


TREES = [  # query heads, key/value heads, new rows, positions held ahead of them
    (4, 1, [1], [0]),
    (8, 2, [1, 3, 2], [0, 63, 64]),
    (32, 8, [5, 0, 17], [300, 12, 0]),
    (8, 8, [64, 65, 127], [0, 1, 63]),
    (10, 2, [31, 40], [100, 0]),
    (16, 1, [9, 20], [511, 77]),
    (14, 2, [33], [129]),
    (32, 8, [100, 129, 3], [70, 0, 640]),        # two tiles a block
    (4, 4, [257], [30]),
    (32, 8, [13], [5000]),                       # few rows: the keys are split
    (8, 2, [40, 7], [4000, 3001]),
    (8, 2, [200], [2000]),                       # two tiles a block, split
    (64, 64, [16] * 6, [250, 200, 180, 64, 63, 1]),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kind", ["tree", "any", "all"])
@pytest.mark.parametrize("hq,hkv,new,ahead", TREES)
def test_attend(dev, bits, kind, hq, hkv, new, ahead):
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=sum(lens) + hq)
    q, seen = queries(sum(new), hq, dev), masks(kind, new, sum(lens))
    out = attend(c, q, seen, new)
    check_attention(out, attend64(c, q, seen, new, lens), SCALE)
    ahead_of = [m for n, m in zip(new, ahead) for _ in range(n)]
    for t, (bits_of, m) in enumerate(zip(seen, ahead_of)):
        if m == 0 and bits_of == 0:
            assert (out[t] == 0).all()


LARGE = [  # tiles in any case, of one for up to 128 rows a key/value head, of two
    (32, 8, [13, 16, 1, 9, 0, 12, 16, 7], [3000, 2500, 3100, 0, 5, 63, 900, 2900]),
    (8, 2, [31] * 24, [100 * i for i in range(24)]),
    (16, 4, [65, 70], [300, 1]),
    (32, 32, [20] * 12, [100 * i for i in range(12)]),
    (14, 2, [16, 40], [7000, 6500]),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("kind", ["tree", "any", "all"])
@pytest.mark.parametrize("hq,hkv,new,ahead", LARGE, ids=lambda x: str(x)[:20])
def test_attend_large(dev, bits, kind, hq, hkv, new, ahead):
    test_attend(dev, bits, kind, hq, hkv, new, ahead)


@pytest.mark.parametrize("bits", [4, 8])
def test_a_causal_mask_is_the_prompt_operator(dev, bits):
    """The same numbers to the last bit where both cut the keys alike: what the masked rows weigh is nothing either way."""
    for new, ahead in (([70, 9], [1500, 300]), ([13], [4000]), ([300], [77]), ([1, 1], [640, 64])):
        lens = [n + m for n, m in zip(new, ahead)]
        c = Cache(lens, 2, bits, dev, seed=4)
        q = queries(sum(new), 8, dev)
        seen = [(1 << (i + 1)) - 1 for n in new for i in range(n)]
        out = attend(c, q, seen, new)
        check_attention(out, attend64(c, q, seen, new, lens), SCALE)
        want = backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, max(new), max(lens), *c.args)
        assert (out.float() - want.float()).abs().max() <= 4e-3 * want.float().abs().max()


@pytest.mark.parametrize("bits", [4, 8])
def test_keys_that_no_row_names_say_nothing(dev, bits):
    """New rows whose keys and values are no numbers, or at the ends of fp16, reach those rows alone that have their bits."""
    new, lens = [40, 20], [340, 84]
    c = Cache(lens, 2, bits, dev, seed=9)
    q = queries(60, 8, dev)
    seen = masks("tree", new, 3)
    clean = attend(c, q, seen, new)
    for row, b in ((30, 0), (11, 1)):
        pos = lens[b] - new[b] + row
        for which in (0, 1):
            c.meta(which)[c.pages[b, pos // PAGE], :, :, pos % PAGE] = float("nan")
    got = attend(c, q, seen, new)
    at = 0
    for b, (n, row) in enumerate(zip(new, (30, 11))):
        for i in range(n):
            if seen[at + i] >> row & 1:
                assert torch.isnan(got[at + i]).all()
            else:
                assert torch.equal(got[at + i], clean[at + i])
        at += n


def test_rows_that_are_left_and_portions_longer_than_their_lengths(dev):
    new, lens = [5, 9, 4], [100, 6, 200]  # the second sequence holds fewer positions than its portion has rows
    c = Cache(lens, 2, 4, dev, seed=7)
    q, seen = queries(21, 8, dev), masks("all", new, 1)
    seen += [0, 0, 0]
    out = torch.full_like(q, 7.0)
    got = backend.paged_tree_attention(q, c.table, starts(new, dev), c.lengths, words_of(seen, 1, dev), 9, 200, *c.args, out=out)
    assert got.data_ptr() == out.data_ptr() and (out[18:] == 7.0).all()
    check_attention(out[:18], attend64(c, q[:18], seen, new, lens), SCALE)
    # rows behind max_seqlen are left, and are no keys of the others
    out = torch.full_like(q, 7.0)
    backend.paged_tree_attention(q, c.table, starts(new, dev), c.lengths, words_of(seen, 1, dev), 4, 200, *c.args, out=out)
    assert (out[4] == 7.0).all() and (out[9:14] == 7.0).all()
    short = [s & 15 for s in seen]
    check_attention(out[:4], [x[:4] for x in attend64(c, q[:18], short, new, lens)], SCALE)
    # fewer pages in the table than lengths speak of
    narrow = c.table[:, :, :1].contiguous()
    out = backend.paged_tree_attention(q[:18], narrow, starts(new, dev), c.lengths, words_of(seen[:18], 1, dev), 9, 200, *c.args)
    want = attend64(c, q[:18], [0] * 5 + seen[5:14] + [0] * 4, new, lens)
    first = attention_seen64(q[:5], c.values(0, 0, 64), c.values(1, 0, 64), torch.ones(5, 64, dtype=torch.bool, device=dev), SCALE)
    check_attention(out[:5], first, SCALE)
    check_attention(out[5:14], [x[5:14] for x in want], SCALE)


def test_strides_words_and_graphs(dev):
    """Queries inside wider rows, more words than the portions need, results in place of the queries; captured and replayed with other masks."""
    new, lens = [33, 12], [700, 140]
    c = Cache(lens, 2, 8, dev, seed=11)
    wide = torch.randn(45, 12, D, generator=torch.Generator().manual_seed(1)).half().to(dev)
    q = wide[:, 2:10]
    seen = masks("any", new, 5)
    words = words_of(seen, 3, dev)
    words[:, 1:] = -1  # bits of rows that are not there
    cu = starts(new, dev)
    call = lambda **more: backend.paged_tree_attention(q, c.table, cu, c.lengths, words, 33, 700, *c.args, **more)
    want = attend64(c, q, seen, new, lens)
    check_attention(call(), want, SCALE)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    graph.replay()
    check_attention(out, want, SCALE)
    other = masks("tree", new, 6)
    words.copy_(words_of(other, 3, dev))
    graph.replay()
    check_attention(out, attend64(c, q, other, new, lens), SCALE)
    want = attend64(c, q, other, new, lens)
    got = call(out=q)
    assert got.data_ptr() == q.data_ptr()
    check_attention(got, want, SCALE)


def test_sharp_scores_and_scales(dev):
    new, ahead = [60, 20], [1440, 313]
    lens = [n + m for n, m in zip(new, ahead)]
    for bits in (4, 8):
        c = Cache(lens, 2, bits, dev, seed=5)
        q, seen = queries(80, 8, dev) * 10, masks("tree", new, 2)
        check_attention(attend(c, q, seen, new, softmax_scale=0.05), attend64(c, q, seen, new, lens, 0.05), 0.05)


# ------------------------------------------------------------------------------------------------------------------------
# rows that are kept
# ------------------------------------------------------------------------------------------------------------------------
def keep(c, new, kept, top=None):
    top = max([len(k) for k in kept] + [1]) if top is None else top
    table = torch.full((len(kept), top), -1, dtype=torch.int32)
    for b, k in enumerate(kept):
        table[b, :len(k)] = torch.tensor(k, dtype=torch.int32)
    counts = torch.tensor([len(k) for k in kept], dtype=torch.int32, device=c.dev)
    return backend.keep_kv_cache(c.table, None if new is None else starts(new, c.dev), c.lengths, table.to(c.dev), counts, *c.args)


def kept_pools(c, new, kept):
    """The pools as they should be: cell by cell, all read before the first is written."""
    want = [p.clone() for p in c.pools]
    cells = []
    for p in want:
        codes = p[:, :c.cut].view(-1, c.hkv, PAGE, D * c.bits // 8)
        cells.append((codes, p[:, c.cut:].view(torch.float16).view(-1, 2, c.hkv, PAGE)))
    for b, (n, k) in enumerate(zip(new, kept)):
        first, moves = c.lens[b] - n, []
        for j, row in enumerate(k[:n]):
            src, dst = first + row, first + j
            if 0 <= row < n and src >= 0 and dst >= 0 and max(src, dst) // PAGE < c.blocks:
                moves.append((src, dst))
        for codes, meta in cells:
            got = [(codes[c.pages[b, s // PAGE], :, s % PAGE].clone(), meta[c.pages[b, s // PAGE], :, :, s % PAGE].clone()) for s, _ in moves]
            for (_, d), (x, m) in zip(moves, got):
                codes[c.pages[b, d // PAGE], :, d % PAGE] = x
                meta[c.pages[b, d // PAGE], :, :, d % PAGE] = m
    return want


KEPT = [
    ([1], [70], [[0]]),
    ([5, 0, 9], [64, 12, 300], [[0, 2, 4], [], [0, 1, 2, 3, 8]]),
    ([26, 30], [100, 30], [[0, 3, 9, 10, 25], [0]]),
    ([64], [130], [[0] + list(range(2, 64, 3))]),                   # across a page's end
    ([256, 10], [700, 10], [list(range(0, 256, 2)), list(range(10))]),
    ([200], [200], [list(range(1, 200))]),                          # every place is the next one's source
    ([20], [90], [[19, 18, 17, 3, 2, 1, 0]]),                       # an order that is none
    ([12], [40], [[0, -1, 5, 12, 7, 7, 100]]),                      # rows that are none; one of them twice
    ([3, 4], [2, 100], [[0, 2], [0, 3]]),                           # fewer positions than rows
    ([4], [50], [[0, 1, 2, 3, 3, 3]]),                              # more than the portion has
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hkv", [1, 8])
@pytest.mark.parametrize("new,lens,kept", KEPT)
def test_keep(dev, bits, hkv, new, lens, kept):
    c = Cache(lens, hkv, bits, dev, seed=sum(lens), extra_blocks=1)
    for p in c.pools:  # also what no sequence holds has numbers, to be found unchanged
        p.copy_(torch.randint(0, 256, p.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(3)))
    want = kept_pools(c, new, kept)
    lengths = keep(c, new, kept)
    assert lengths.tolist() == [max(m - n + min(len(k), n), 0) for n, m, k in zip(new, lens, kept)]
    assert c.lengths.tolist() == lens
    for a, b in zip(c.pools, want):
        assert torch.equal(a, b)


def test_keep_counts_rows_and_tables(dev):
    c = Cache([100, 90, 80], 2, 4, dev, seed=1)
    before = [p.clone() for p in c.pools]
    rows_ = torch.full((3, 4), -1, dtype=torch.int32, device=dev)
    rows_[:, 0] = 0
    # counts below zero and past the rows; one row a sequence; a row at its own place moves nothing
    lengths = backend.keep_kv_cache(c.table, starts([6, 6, 6], dev), c.lengths, rows_, torch.tensor([-5, 4, 2 ** 31 - 1], dtype=torch.int32, device=dev), *c.args)
    assert lengths.tolist() == [94, 88, 78]
    lengths = backend.keep_kv_cache(c.table, None, c.lengths, rows_, torch.tensor([0, 1, 1], dtype=torch.int32, device=dev), *c.args)
    assert lengths.tolist() == [99, 90, 80]
    lengths = backend.keep_kv_cache(c.table, starts([6, 6, 6], dev), c.lengths, rows_[:, :0].contiguous(), torch.ones(3, dtype=torch.int32, device=dev), *c.args)
    assert lengths.tolist() == [94, 84, 74]
    assert all(torch.equal(a, b) for a, b in zip(before, c.pools))
    # a table that ends ahead of the rows
    rows_ = torch.tensor([[0, 5]] * 3, dtype=torch.int32, device=dev)
    lengths = backend.keep_kv_cache(c.table[:, :, :1].contiguous(), starts([6, 6, 6], dev), c.lengths, rows_, torch.full((3,), 2, dtype=torch.int32, device=dev), *c.args)
    assert lengths.tolist() == [96, 86, 76] and all(torch.equal(a, b) for a, b in zip(before, c.pools))
    empty = backend.keep_kv_cache(c.table[:0], None, c.lengths[:0], rows_[:0], rows_[:0, 0].contiguous(), *c.args)
    assert empty.shape == (0,)


def test_refusals(dev):
    c = Cache([70, 80], 2, 4, dev)
    q, k = queries(5, 8, dev), queries(5, 2, dev)
    cu, at = starts([2, 3], dev), torch.zeros(3, 5, dtype=torch.int32, device=dev)
    seen = torch.zeros(5, 1, dtype=torch.int64, device=dev)
    at_args = lambda **x: {**dict(q=q, k=k, v=k, kv=c.table, cu=cu, lens=c.lengths, at=at, sections=(16, 24, 24), out=None), **x}

    def append(**x):
        a = at_args(**x)
        return backend.append_kv_cache_at(a["q"], a["k"], a["v"], a["kv"], a["cu"], a["lens"], a["at"], a["sections"], 64, c.size, 128, 1e4, True, True, out=a["out"])

    append()
    for x in (dict(at=at.long()), dict(at=at[:2]), dict(at=at[:, :4].contiguous()), dict(at=at.t().contiguous().t()), dict(at=at.cpu()), dict(at=None), dict(sections=None), dict(sections=(16, 24)),
              dict(sections=(16, 24, 25)), dict(sections=(-8, 48, 24)), dict(sections=(16, 24.5, 24)), dict(sections=64), dict(at=at[0], sections=(16, 24, 24)), dict(at=at[None]),
              dict(at=torch.zeros(5, 5, dtype=torch.int32, device=dev), sections=(16, 12, 12, 12, 12)), dict(k=q), dict(q=q.float()), dict(lens=c.lengths[:1]), dict(kv=c.table.int()),
              dict(out=q[:, :4]), dict(q=q.cpu())):
        with pytest.raises((RuntimeError, TypeError)):
            append(**x)

    def tree(**x):
        a = {**dict(q=q, kv=c.table, cu=cu, lens=c.lengths, seen=seen, top=3, out=None), **x}
        return backend.paged_tree_attention(a["q"], a["kv"], a["cu"], a["lens"], a["seen"], a["top"], 80, *c.args, out=a["out"])

    tree()
    for x in (dict(seen=seen.int()), dict(seen=seen[:4]), dict(seen=seen[:, 0]), dict(seen=seen[:, :0]), dict(seen=seen.cpu()), dict(seen=None), dict(seen=torch.zeros(5, 2, dtype=torch.int64, device=dev)[:, ::2]),
              dict(top=-1), dict(q=q.float()), dict(out=q[:4]), dict(cu=cu[:2]), dict(lens=c.lengths.long())):
        with pytest.raises((RuntimeError, TypeError)):
            tree(**x)
    with pytest.raises(RuntimeError, match="words"):
        backend.paged_tree_attention(queries(70, 8, dev), c.table, starts([0, 70], dev), c.lengths, torch.zeros(70, 1, dtype=torch.int64, device=dev), 70, 80, *c.args)

    def keep_(**x):
        a = {**dict(kv=c.table, cu=cu, lens=c.lengths, rows=torch.zeros(2, 2, dtype=torch.int32, device=dev), counts=torch.zeros(2, dtype=torch.int32, device=dev)), **x}
        return backend.keep_kv_cache(a["kv"], a["cu"], a["lens"], a["rows"], a["counts"], *c.args)

    keep_()
    for x in (dict(rows=seen), dict(rows=torch.zeros(3, 2, dtype=torch.int32, device=dev)), dict(rows=torch.zeros(2, dtype=torch.int32, device=dev)), dict(counts=c.lengths.long()), dict(counts=c.lengths[:1]),
              dict(counts=c.lengths.cpu()), dict(rows=torch.zeros(2, 257, dtype=torch.int32, device=dev)), dict(rows=torch.zeros(2, 4, dtype=torch.int32, device=dev)[:, ::2]), dict(kv=c.table[:, 0]),
              dict(lens=None)):
        with pytest.raises((RuntimeError, TypeError)):
            keep_(**x)

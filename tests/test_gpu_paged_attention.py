"""Prompt attention over the paged cache and attention behind a shared prefix against the definition in 64 bits."""
import pytest
import torch

from qserve_b200 import backend
from qserve_b200._lib import lib
from tests.paged_util import D, F64, HALF, PAGE, Cache, attention64, check_attention

pytestmark = pytest.mark.gpu
SCALE = D ** -0.5


def starts(counts, dev):
    return torch.tensor([sum(counts[:i]) for i in range(len(counts) + 1)], dtype=torch.int32, device=dev)


def queries(T, hq, dev, seed=1):
    return torch.randn(T, hq, D, generator=torch.Generator().manual_seed(seed)).half().to(dev)


def prompt64(c, q, new, lens, scale=SCALE):
    parts, at = [], 0
    for b, (n, m) in enumerate(zip(new, lens)):
        limit = torch.arange(m - n, m, device=c.dev)
        parts.append(attention64(q[at:at + n], c.values(0, b, max(m, 0)), c.values(1, b, max(m, 0)), limit, scale))
        at += n
    return [torch.cat(x) for x in zip(*parts)]


def run_prompt(c, q, new, **more):
    return backend.paged_prompt_attention(q, c.table, starts(new, c.dev), c.lengths, max(new), max(c.lens), *c.args, **more)


PROMPTS = [  # query heads, key/value heads, new tokens, positions held ahead of them
    (4, 1, [1], [0]),
    (8, 2, [1, 1, 1], [0, 63, 64]),
    (32, 8, [5, 0, 17], [300, 12, 0]),           # a sequence that brings nothing
    (8, 8, [64, 65, 127], [0, 1, 63]),           # one query head a key/value head
    (10, 2, [31, 40], [100, 0]),                 # five heads: tiles that end inside a token
    (16, 1, [9, 20], [511, 77]),
    (14, 2, [33], [129]),                        # seven heads
    (32, 8, [200, 129, 3], [70, 0, 640]),        # two tiles a block
    (4, 4, [257], [0]),
    (32, 8, [3], [5000]),                        # few rows: the keys are split
    (8, 2, [40, 7], [4000, 3001]),
    (8, 2, [300], [2000]),                       # two tiles a block, split
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,new,ahead", PROMPTS)
def test_prompt(dev, bits, hq, hkv, new, ahead):
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=sum(lens) + hq)
    q = queries(sum(new), hq, dev)
    check_attention(run_prompt(c, q, new), prompt64(c, q, new, lens), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
def test_prompt_sharp_scores(dev, bits):
    """Queries ten times as large: a few keys take all the weight, maxima grow along the walk."""
    new, lens = [70, 20], [1500, 333]
    c = Cache(lens, 2, bits, dev, seed=5)
    q = queries(90, 8, dev) * 10
    check_attention(run_prompt(c, q, new, softmax_scale=0.05), prompt64(c, q, new, lens, 0.05), 0.05)


def shared64(c, q, lens, scale=SCALE):
    parts = [attention64(q[b:b + 1], c.values(0, b, m), c.values(1, b, m), torch.tensor([m - 1], device=c.dev), scale) for b, m in enumerate(lens)]
    return [torch.cat(x) for x in zip(*parts)]


SHARED = [  # query heads, key/value heads, shared pages, positions of the sequences
    (4, 1, 1, [65]),
    (8, 2, 0, [1, 64, 65, 200]),                 # nothing shared
    (32, 8, 4, [300, 257, 256, 700]),            # one sequence that ends with the prefix
    (8, 8, 16, [1025, 1100, 1024 + 640]),
    (10, 2, 7, [449, 500, 460, 451, 470]),
    (40, 2, 3, [200, 300]),                      # twenty heads a key/value head: three groups of the tail kernel
    (32, 8, 10, [700] * 20 + [641] * 20),        # two tiles a block
    (64, 64, 2, [130, 5000]),                    # long pages of one's own: clusters
    (4, 1, 33, [2113, 9000]),
    (32, 8, 5, [0, 100, 320, 321, 7, 400]),      # empty, and shorter than the prefix
    (16, 1, 300, [19201, 19300]),                # many splits
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,shared,lens", SHARED)
def test_shared(dev, bits, hq, hkv, shared, lens):
    c = Cache(lens, hkv, bits, dev, shared=shared, seed=sum(lens) + hq)
    q = queries(len(lens), hq, dev)
    out = backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args)
    check_attention(out, shared64(c, q, lens), SCALE)
    assert all(bool((out[b] == 0).all()) for b, n in enumerate(lens) if n == 0)


@pytest.mark.parametrize("bits", [4, 8])
def test_shared_is_the_prompt_operator_of_single_tokens(dev, bits):
    """The same batch through both operators; where the whole prefix lies in a sequence's table nothing has to be said about it."""
    lens = [900, 1030, 961, 1500]
    c = Cache(lens, 2, bits, dev, shared=14, seed=3)
    q = queries(4, 8, dev)
    want = shared64(c, q, lens)
    for out in (backend.shared_prefix_attention(q, c.table, c.lengths, 14, max(lens), *c.args),
                backend.shared_prefix_attention(q, c.table, c.lengths, 3, max(lens), *c.args),
                backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, max(lens), *c.args)):
        check_attention(out, want, SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("new,ahead", [([70], [10]), ([6], [2600])])
def test_a_key_that_is_no_number_reaches_the_rows_that_see_it(dev, bits, new, ahead):
    """The keys of three positions of the portion get a scale that is no number, or a value's: rows ahead of them are as they were, the others are no numbers."""
    lens = [n + m for n, m in zip(new, ahead)]
    for which, at in ((0, 4), (1, 3), (1, 5)):
        c = Cache(lens, 2, bits, dev, seed=8)
        q = queries(new[0], 8, dev)
        want = prompt64(c, q, new, lens)
        pos = ahead[0] + at
        c.meta(which)[c.pages[0, pos // PAGE], which ^ 1, :, pos % PAGE] = float("inf") if at == 3 else float("nan")
        out = run_prompt(c, q, new)
        check_attention(out[:at], [x[:at] for x in want], SCALE)
        assert bool(torch.isnan(out[at:]).all())


def test_rows_behind_the_batch_and_rows_without_a_position(dev):
    c = Cache([40, 90], 2, 4, dev, seed=2)
    new = [10, 20]
    q = queries(50, 8, dev)
    out = torch.full((50, 8, D), 7.0, dtype=HALF, device=dev)
    got = backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, 20, 90, *c.args, out=out)
    assert got.data_ptr() == out.data_ptr() and bool((out[30:] == 7).all())
    check_attention(out[:30], prompt64(c, q[:30], new, [40, 90]), SCALE)
    # split keys: the same
    out.fill_(7.0)
    backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, 20, 9000, *c.args, out=out)
    assert bool((out[30:] == 7).all())
    check_attention(out[:30], prompt64(c, q[:30], new, [40, 90]), SCALE)
    # a length smaller than the portion: its first rows have no position
    c.lengths[0] = 4
    out = backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, 20, 90, *c.args)
    assert bool((out[:6] == 0).all())
    check_attention(out[6:10], prompt64(c, q[6:10], [4], [4]), SCALE)


def test_lengths_past_the_tables_stay_inside(dev):
    """A length that says more than a sequence has pages: the pages are the limit."""
    c = Cache([128, 128], 2, 8, dev, shared=1, seed=2)
    q = queries(2, 8, dev)
    want = shared64(c, q, [128, 128])
    c.lengths.fill_(100000)
    check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, 1, 100000, *c.args), want, SCALE)
    check_attention(backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 100000, *c.args), want, SCALE)


def test_strides_and_results_in_place(dev):
    lens = [300, 180, 700]
    c = Cache(lens, 2, 4, dev, shared=2, seed=11)
    rows = torch.randn(3, 5 + 8 + 3, D, generator=torch.Generator().manual_seed(2)).half().to(dev)
    q = rows[:, 5:13]
    want = shared64(c, q, lens)
    wide = torch.zeros(3, 11, D, dtype=HALF, device=dev)
    backend.shared_prefix_attention(q, c.table, c.lengths, 2, 700, *c.args, out=wide[:, 2:10])
    check_attention(wide[:, 2:10], want, SCALE)
    assert bool((wide[:, :2] == 0).all()) and bool((wide[:, 10:] == 0).all())
    wide.zero_()
    backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 700, *c.args, out=wide[:, 2:10])
    check_attention(wide[:, 2:10], want, SCALE)
    keep = rows.clone()
    backend.shared_prefix_attention(q, c.table, c.lengths, 2, 700, *c.args, out=q)
    check_attention(rows[:, 5:13], want, SCALE)
    rows.copy_(keep)
    backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 700, *c.args, out=q)
    check_attention(rows[:, 5:13], want, SCALE)


def test_two_graphs_at_once_and_again(dev):
    """Two captured calls, replayed on two streams at a time, and the same bits every time."""
    cases = []
    for seed, lens in ((1, [3000, 2900, 3100]), (2, [2800, 3300])):
        c = Cache(lens, 2, 4, dev, shared=30, seed=seed)
        q = queries(len(lens), 8, dev, seed)
        call = lambda c=c, q=q, lens=lens: (backend.shared_prefix_attention(q, c.table, c.lengths, 30, max(lens), *c.args),  # noqa: E731
                                            backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, max(lens), *c.args))
        eager = call()
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            out = call()
        cases.append((graph, stream, out, eager, call))  # with the call its inputs: a graph does not keep them
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, stream, *_ in cases:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for _, _, out, eager, _ in cases:
        assert all(torch.equal(a, b) for a, b in zip(out, eager))


def test_lengths_change_between_replays(dev):
    """A captured step whose lengths grow: what the tables say at the time of the replay counts."""
    lens = [640, 700]
    c = Cache([1000, 1000], 2, 8, dev, shared=9, seed=4)
    c.lengths.copy_(torch.tensor(lens, dtype=torch.int32))
    q = queries(2, 8, dev)
    backend.shared_prefix_attention(q, c.table, c.lengths, 9, 1000, *c.args)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.lengths.add_(1)
        out = backend.shared_prefix_attention(q, c.table, c.lengths, 9, 1000, *c.args)
    for step in range(1, 4):
        graph.replay()
        check_attention(out, shared64(c, q, [n + step for n in lens]), SCALE)


def test_empty_calls(dev):
    c = Cache([64, 64], 2, 4, dev)
    q = queries(0, 8, dev)
    none = torch.zeros(0, 2, 1, dtype=torch.int64, device=dev)
    zero = torch.zeros(0, dtype=torch.int32, device=dev)
    assert backend.paged_prompt_attention(q, c.table, starts([0, 0], dev), c.lengths, 0, 64, *c.args).shape == (0, 8, D)
    assert backend.shared_prefix_attention(q, none, zero, 0, 0, *c.args).shape == (0, 8, D)
    assert backend.paged_prompt_attention(q, none, torch.zeros(1, dtype=torch.int32, device=dev), zero, 0, 0, *c.args).shape == (0, 8, D)


def test_estimates_decide_nothing_else(dev):
    """max_length below and far above the truth; a portion longer than max_seqlen: its rows behind that stay as they are."""
    new, lens = [20, 33], [900, 1200]
    c = Cache(lens, 2, 4, dev, seed=12)
    q = queries(53, 8, dev)
    want = prompt64(c, q, new, lens)
    for top in (0, 1, 70, 100000):
        check_attention(backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, 33, top, *c.args), want, SCALE)
    for top in (1, 1200, 100000):  # one block for all keys; a cluster or join_kernel
        out = torch.full((53, 8, D), 7.0, dtype=HALF, device=dev)
        backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, 25, top, *c.args, out=out)
        assert bool((out[45:] == 7).all())
        check_attention(out[:45], [x[:45] for x in want], SCALE)


@pytest.mark.parametrize("shared", [0, 2])
def test_lengths_at_the_ends_of_their_type(dev, shared):
    c = Cache([128, 128, 128], 2, 4, dev, shared=2 if shared else 0, seed=2)
    q = queries(3, 8, dev)
    want = shared64(c, q, [128, 128, 128])
    c.lengths.copy_(torch.tensor([2 ** 31 - 1, -2 ** 31, 128], dtype=torch.int32))
    for out in (backend.shared_prefix_attention(q, c.table, c.lengths, shared, 128, *c.args), backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 128, *c.args)):
        assert bool((out[1] == 0).all())
        check_attention(out[::2], [x[::2] for x in want], SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lens,shared", [([300, 700, 290], 4), ([5000, 4300], 64), ([640] * 200, 9)])
def test_a_shared_key_that_is_no_number(dev, bits, lens, shared):
    """Every sequence that reaches it has no number then, in the prefix and behind it; one that ends ahead of it is as it was."""
    lens = lens + [shared * PAGE - 60]
    for at in (shared * PAGE - 50, lens[0] - 1):
        c = Cache(lens, 2, bits, dev, shared=shared, seed=8)
        q = queries(len(lens), 8, dev)
        want = shared_row(c, q, lens, len(lens) - 1)  # the last sequence ends ahead of both
        c.meta(1)[c.pages[0, at // PAGE], 0, :, at % PAGE] = float("nan")
        out = backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args)
        hit = [b for b, n in enumerate(lens) if n > at and (at < shared * PAGE or b == 0)]
        rest = [b for b in range(len(lens)) if b not in hit]
        assert bool(torch.isnan(out[hit]).all()) and bool(torch.isfinite(out[rest]).all())
        check_attention(out[-1:], want, SCALE)


def shared_row(c, q, lens, b):
    return attention64(q[b:b + 1], c.values(0, b, lens[b]), c.values(1, b, lens[b]), torch.tensor([lens[b] - 1], device=c.dev), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
def test_many_sequences(dev, bits):
    """Enough runs of heads for a warp each, their number no multiple of a block's warps; ragged, some empty."""
    g = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(0, 400, (231,), generator=g)]
    for hq, hkv in ((32, 8), (9, 9)):
        c = Cache(lens, hkv, bits, dev, shared=2, seed=7)
        q = queries(len(lens), hq, dev)
        check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, 2, max(lens), *c.args), shared64(c, q, lens), SCALE)
        check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, 0, max(lens), *c.args), shared64(c, q, lens), SCALE)


def test_large_values_stay_finite(dev):
    """Values up to 60000: weights times scales and partial results stay in fp16's range."""
    lens = [700, 900]
    for bits in (4, 8):
        c = Cache(lens, 1, bits, dev, shared=3, seed=3)
        c.meta(1)[:, 0] *= 8000.0 if bits == 4 else 1000.0
        q = queries(2, 4, dev)
        for shared in (0, 3):
            check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, shared, 900, *c.args), shared64(c, q, lens), SCALE)
        check_attention(backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 900, *c.args), shared64(c, q, lens), SCALE)


def test_calls_on_two_streams_at_once(dev):
    """Eager calls of both operators on two streams, inputs of their own: what each gives alone."""
    cases = []
    for seed, lens in ((1, [3000, 2900, 3100, 2950] * 4), (2, [2800, 3300, 5000] * 5)):
        c = Cache(lens, 2, 4, dev, shared=30, seed=seed)
        q = queries(len(lens), 8, dev, seed)
        cases.append((c, q, lens, torch.cuda.Stream()))

    def both(c, q, lens):
        return (backend.shared_prefix_attention(q, c.table, c.lengths, 30, max(lens), *c.args),
                backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, max(lens), *c.args))
    want = [both(*x[:3]) for x in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (c, q, lens, stream) in enumerate(cases):
            with torch.cuda.stream(stream):
                got[i].append(both(c, q, lens))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(a, b) for x in g for a, b in zip(x, w))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,new,ahead", [(152, 152, [130], [400]), (32, 8, [1300], [500]), (32, 8, [20] * 30 + [0, 3] + [20] * 6, [2500, 2400] * 19)])
def test_the_last_round_is_split(dev, bits, hq, hkv, new, ahead):
    """More blocks than the device holds, so few of them in the last round that they are split (152 and 168 blocks of two tiles, 304 of one; a work space shows it)."""
    lens = [n + m for n, m in zip(new, ahead)]
    T, most = sum(new), max(new)
    c = Cache(lens, hkv, bits, dev, seed=hq + len(new))
    size = lib.qs_paged_prompt_attention_workspace_bytes(len(new), T, most, max(lens), hq, hkv)
    assert 0 < size < 2 * T * hq * (2 * D + 8)
    q = queries(T + 3, hq, dev)
    out = torch.full((T + 3, hq, D), 7.0, dtype=HALF, device=dev)
    backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, most, max(lens), *c.args, out=out)
    assert bool((out[T:] == 7).all())
    check_attention(out[:T], prompt64(c, q[:T], new, lens), SCALE)
    # the last portion shorter than it says: its first rows have no position
    c.lengths[-1] = 4
    backend.paged_prompt_attention(q, c.table, starts(new, dev), c.lengths, most, max(lens), *c.args, out=out)
    n = new[-1]
    assert bool((out[T:] == 7).all()) and bool((out[T - n:T - 4] == 0).all())
    check_attention(out[T - 4:T], attention64(q[T - 4:T], c.values(0, len(new) - 1, 4), c.values(1, len(new) - 1, 4), torch.arange(4, device=dev), SCALE), SCALE)


@pytest.mark.parametrize("new,top", [([1300], 1800), ([1300], 64), ([20], 4000)])
def test_blocks_without_a_key_write_zeros(dev, new, top):
    """A portion whose length leaves only its last four rows a position: blocks (and splits) that see no key.  The queries come late, out of DRAM."""
    c = Cache([4], 8, 4, dev, seed=1, extra_blocks=1)
    q, cu = queries(new[0], 32, dev), starts(new, dev)
    flush = torch.empty(64 << 20, dtype=torch.int32, device=dev)
    want = attention64(q[-4:], c.values(0, 0, 4), c.values(1, 0, 4), torch.arange(4, device=dev), SCALE)
    for i in range(10):
        out = torch.full((new[0], 32, D), 7.0, dtype=HALF, device=dev)
        flush.fill_(i)
        backend.paged_prompt_attention(q, c.table, cu, c.lengths, new[0], top, *c.args, out=out)
        assert bool((out[:-4] == 0).all())
        check_attention(out[-4:], want, SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shared,lens", [(0, [700]), (1, [65, 130, 333] * 5), (3, [200, 1500] * 9), (1, [150] * 300)])
@pytest.mark.parametrize("how", ["small queries", "small values", "growing values", "falling values"])
def test_small_numbers(dev, bits, shared, lens, how):
    """Queries of 2^-13 (as products of nibbles 16 u they would be halved four times) and values' scales down to 2^-8 of the others' (subnormal numbers of INT8): as exact
    as any others."""
    c = Cache(lens, 2, bits, dev, shared=shared, seed=sum(lens))
    q, scale = queries(len(lens), 8, dev), SCALE
    if how == "small queries":
        q, scale = q * 2.0 ** -13, SCALE * 2.0 ** 13
    else:
        at = torch.arange(c.blocks, device=dev) * 8.0 / max(c.blocks - 1, 1)  # by page
        power = {"small values": at * 0 - 8, "growing values": at - 8, "falling values": -at}[how]
        for b in range(len(lens)):
            for j in range(c.blocks):
                if b == 0 or j >= shared:
                    c.meta(1)[c.pages[b, j], 0] *= float(2.0 ** power[j])
    out = backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args, softmax_scale=scale)
    check_attention(out, shared64(c, q, lens, scale), scale)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,n", [(8, 2, 20), (32, 8, 150)])
def test_values_at_the_ends_of_their_type(dev, bits, hq, hkv, n):
    """A token in the middle of the portion whose key and value reach +- 65504: with the rounded scale some of their codes stand for more.  Rows ahead of it do not
    see it and are as they were; rows behind it are numbers (or too large for one)."""
    c = Cache([100 + n], hkv, bits, dev, seed=n)
    q, at = queries(n, hq, dev), 100 + n // 2
    want = prompt64(c, q, [n], c.lens)
    top = 2 ** bits - 1
    for which in (0, 1):
        meta, page, slot = c.meta(which), c.pages[0, at // PAGE], at % PAGE
        meta[page, 0, :, slot] = 131008.0 / top * 1.01  # a hundredth too much
        meta[page, 1, :, slot] = top // 2
    assert float(c.values(1, 0, at + 1)[at].abs().max()) > 65520
    out = run_prompt(c, q, [n])
    check_attention(out[:n // 2], [x[:n // 2] for x in want], SCALE)
    assert not bool(torch.isnan(out).any())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("hq,hkv,new,ahead", [(8, 2, [20, 3], [100, 700]), (32, 8, [150], [60])])
def test_values_near_one_end_of_their_type(dev, bits, sign, hq, hkv, new, ahead):
    """Values from -57000 to 5000, or the other way round: a scale times the largest code is past fp16, what it stands for is not."""
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=4)
    top = 2 ** bits - 1
    scale, zero = c.meta(1)[:, 0], c.meta(1)[:, 1]
    scale.copy_(torch.where(scale.isnan(), scale, 62000.0 / top))
    zero.copy_(torch.where(zero.isnan(), zero, top * (57 / 62 if sign > 0 else 5 / 62)))
    q = queries(sum(new), hq, dev)
    check_attention(run_prompt(c, q, new), prompt64(c, q, new, lens), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lens,shared", [([300, 700], 2), ([200] * 700, 1)])
@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
def test_scales_and_zeros_that_are_no_numbers(dev, bits, lens, shared, value):
    """Scale or zero of a key or a value, in the shared page or behind it: NaN, never an infinity or a key that has gone."""
    for which in (0, 1):
        for field in (0, 1):
            for at in (10, 190):
                c = Cache(lens, 2, bits, dev, shared=shared, seed=8)
                q = queries(len(lens), 8, dev)
                c.meta(which)[c.pages[0, at // PAGE], field, :, at % PAGE] = value
                out = backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args)
                hit = slice(0, 1) if at >= shared * PAGE else slice(None)
                assert bool(torch.isnan(out[hit]).all())
                assert at < shared * PAGE or bool(torch.isfinite(out[1:]).all())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("lens,shared", [([1, 2, 2, 3] * 5, 0), ([2] * 700, 0)])
def test_values_near_their_zero(dev, bits, lens, shared):
    """Few positions, values that are differences of much larger products of codes and zeros: off by the roundings of the values, not by those of the products."""
    c = Cache(lens, 2, bits, dev, shared=shared, seed=12)
    top = 2 ** bits - 1
    for b in range(len(lens)):
        meta = c.meta(1)[c.pages[b, 0]]
        meta[1, :, :lens[b]] = top / 2 + 0.0625
        raw = c.pools[1][c.pages[b, 0], :c.cut]
        raw.fill_(0x78 if bits == 4 else 0x80)  # half the top and the code behind it
    q = queries(len(lens), 8, dev)
    check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args), shared64(c, q, lens), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("batch,shared,own", [(38, 16, 500), (40, 32, 900), (64, 16, 400)])
def test_prefix_and_own_pages_side_by_side(dev, bits, batch, shared, own):
    """Batches whose own pages are read while the prefix is: fewer splits of it than the work space has room for, whatever max_length says."""
    lens = [shared * PAGE + (own * (7 + 5 * b % 9)) // 16 for b in range(batch)]
    lens[3] = shared * PAGE - 5
    c = Cache(lens, 8, bits, dev, shared=shared, seed=batch)
    q = queries(batch, 32, dev)
    want = shared64(c, q, lens)
    for top in (max(lens), 1, 100000):
        for _ in range(3):
            check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, shared, top, *c.args), want, SCALE)

"""Drafted trees and their verification against the definition in 64 bits: vocabularies and rows of every alignment, chains with and without probabilities, trees,
temperatures from greedy on, logits that are no tokens, batches with empty portions, graphs, streams, the distribution of what comes out."""
import math

import numpy as np
import pytest
import torch

from qserve_b200 import backend
from tests.drafts_util import random_parents, tree64, verify64, words_of
from tests.test_gpu_paged_attention import starts

pytestmark = pytest.mark.gpu
TYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.mark.parametrize("new", [[1], [2, 0, 5], [64, 65, 1, 31], [256, 200, 3], [13] * 300, [0, 0]])
def test_tree(dev, new):
    rng = np.random.default_rng(sum(new))
    parents = random_parents(rng, new)
    first = [int(x) for x in rng.integers(0, 5000, len(new))]
    lens = [f + n for f, n in zip(first, new)]
    top = max(max(new), 1)
    positions, visible = backend.draft_tree(torch.tensor(parents, dtype=torch.int32, device=dev), starts(new, dev), torch.tensor(lens, dtype=torch.int32, device=dev), top)
    seen, at = tree64(parents, new, first)
    assert visible.shape == (sum(new), (top + 63) // 64) and positions.dtype == torch.int32 and visible.dtype == torch.int64
    assert positions.tolist() == at
    assert torch.equal(visible, words_of(seen, (top + 63) // 64, dev))


def test_tree_of_a_chain_is_causal(dev):
    n = 256
    parents = torch.arange(-1, n - 1, dtype=torch.int32, device=dev)
    positions, visible = backend.draft_tree(parents, None if n == 1 else starts([n], dev), torch.tensor([n + 7], dtype=torch.int32, device=dev), n)
    assert torch.equal(positions, torch.arange(7, 7 + n, dtype=torch.int32, device=dev))
    assert torch.equal(visible, words_of([(1 << (i + 1)) - 1 for i in range(n)], 4, dev))
    # one row a sequence without starts
    positions, visible = backend.draft_tree(parents[:5], None, torch.arange(1, 6, dtype=torch.int32, device=dev), 1)
    assert positions.tolist() == [0, 1, 2, 3, 4] and visible.tolist() == [[1]] * 5


def inputs(dev, dtype, V, new, kind, seed, spread=2.5):
    """Logits with a few strong tokens a row, drafts that are often right, random numbers."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    T = sum(new)
    logits = spread * torch.randn(T, V, generator=g)
    if V > 8:
        logits.scatter_(1, torch.randint(0, V, (T, 4), generator=g), 8 + 5 * torch.rand(T, 4, generator=g))
    draft = logits + torch.randn(T, V, generator=g)
    logits = logits.to(dtype)
    parents = random_parents(rng, new) if kind == "tree" else None
    probs = torch.softmax(draft, -1) if kind == "probs" else None
    tokens, row = torch.zeros(T, dtype=torch.int64), 0
    best = draft.topk(min(V, 4), -1).indices
    for n in new:
        kids = {}
        for i in range(n):
            up = parents[row + i] if parents else i - 1
            if i == 0 or not 0 <= up < i:
                tokens[row + i] = int(rng.integers(-3, V + 3))
            elif probs is not None:
                tokens[row + i] = int(torch.multinomial(probs[row + up], 1, generator=g))
            else:
                kids[up] = kids.get(up, -1) + 1
                tokens[row + i] = best[row + up, kids[up] % best.shape[1]] if rng.random() > 0.05 else [-1, V, 2 ** 40][int(rng.integers(3))]
        row += n
    coins, draws = torch.rand(T, generator=g), torch.rand(len(new), generator=g)
    return {"logits": logits.to(dev), "tokens": tokens.to(dev), "parents": None if parents is None else torch.tensor(parents, dtype=torch.int32, device=dev),
            "probs": None if probs is None else probs.to(dev), "coins": coins.to(dev), "draws": draws.to(dev), "new": new, "heats": None}


def call(x, top=None, cu="starts", **more):
    a = {**x, **more}
    cu = starts(a["new"], a["logits"].device) if isinstance(cu, str) else cu
    return backend.verify_drafts(a["logits"], a["tokens"], cu, max(a["new"]) if top is None else top, a["coins"], a["draws"], a["parents"], a["probs"], a["heats"])


def definition(x, top=None):
    d = lambda t: None if t is None else t.double().cpu().numpy()
    # (an inverse temperature of 32 bits would be another one: the temperature itself is)
    return verify64(d(x["logits"]), x["tokens"].cpu().numpy(), x["new"], d(x["coins"]), d(x["draws"]), None if x["parents"] is None else x["parents"].tolist(), d(x["probs"]),
                    None if x["heats"] is None else x["heats"].double().tolist(), top)


def check(x, top=None, **more):
    got = call(x, top, **more)
    want = definition(x, top)
    # no input is so near to a border that the definition's own roundings of 2^-53 could decide
    assert want[3] > 1e-12
    assert got[2].tolist() == want[2].tolist()
    assert np.array_equal(got[1].cpu().numpy(), want[1])
    assert np.array_equal(got[0].cpu().numpy(), want[0])


SHAPES = [  # vocabulary, rows of the sequences
    (1, [1, 3, 2]),
    (7, [4, 1, 0, 6]),
    (8, [2]),
    (1000, [5, 6, 1, 9]),
    (1024, [33, 64, 2, 40]),
    (4099, [256, 3]),
    (32003, [6, 5]),
    (128256, [5, 5, 4]),
    (152064, [26]),
    (50, [3] * 200),
]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["probs", "tree", "none"])
@pytest.mark.parametrize("V,new", SHAPES, ids=lambda x: str(x)[:20])
def test_verify(dev, dtype, kind, V, new):
    check(inputs(dev, dtype, V, new, kind, seed=V + len(new)))


@pytest.mark.parametrize("kind", ["probs", "tree", "none"])
@pytest.mark.parametrize("V", [17, 2051, 20011])
@pytest.mark.parametrize("batch", [1, 7, 8, 9, 11, 14, 16, 19, 22, 25, 31, 38, 50, 75, 150])
def test_batches(dev, kind, V, batch):
    """Sequences share the device: each batch has blocks of its own number a sequence, and warps at the end of a row have few words or none."""
    check(inputs(dev, TYPES[batch % 3], V, [2 + (i + batch) % 3 for i in range(batch)], kind, seed=V + batch))


@pytest.mark.parametrize("kind", ["probs", "tree", "none"])
@pytest.mark.parametrize("V", [9, 5003, 65536])
def test_temperatures(dev, kind, V):
    new = [6, 7, 1, 12, 5, 6, 6, 3]
    x = inputs(dev, torch.float16, V, new, kind, seed=V)
    x["heats"] = torch.tensor([0.0, 0.3, 1.0, 1.7, -1.0, 0.05, 30.0, float("nan")], device=dev)
    check(x)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", ["tree", "none", "probs"])
def test_greedy_takes_the_lowest_of_equal_logits(dev, dtype, kind):
    V, new = 3333, [5, 17, 2]
    x = inputs(dev, dtype, V, new, kind, seed=3)
    x["logits"] = x["logits"].float().round().clamp(max=6).to(dtype)  # many largest ones
    x["heats"] = torch.zeros(3, device=dev)
    best = (x["logits"] == x["logits"].amax(-1, keepdim=True)).int().argmax(-1)
    x["tokens"][1:] = best[:-1]
    check(x)
    assert (call(x)[2] > 1).any()


@pytest.mark.parametrize("kind", ["probs", "tree", "none"])
@pytest.mark.parametrize("offset,stride", [(0, 1000), (1, 1001), (3, 1003), (5, 1024)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_of_every_alignment(dev, kind, dtype, offset, stride):
    x = inputs(dev, dtype, 1000, [4, 9, 3], kind, seed=offset + stride)
    wide = torch.full((16 * stride + 16,), float("inf"), dtype=dtype, device=dev)  # what lies between the rows would take all
    y = wide[offset:offset + 16 * stride].view(16, stride)[:, :1000]
    y.copy_(x["logits"])
    x["logits"] = y
    if kind == "probs":
        z = torch.full((16, stride + 1), float("nan"), device=dev)[:, 1:1001]
        z.copy_(x["probs"])
        x["probs"] = z
    check(x)


def test_logits_that_are_no_tokens(dev):
    """-inf, the type's lowest number and NaN; a row with nothing else; rows with infinities."""
    for kind in ("tree", "none", "probs"):
        for heat in (None, torch.tensor([0.0, 1.3, 0.7, 0.0], device=dev)):
            x = inputs(dev, torch.float16, 700, [5, 6, 4, 5], kind, seed=11)
            x["heats"] = heat
            x["logits"][:, 100:300] = -math.inf
            x["logits"][:, 300:350] = -65504.0
            x["logits"][:, 5] = float("nan")
            check(x)
            x["logits"][7] = -math.inf
            x["logits"][13] = float("nan")
            x["logits"][16, 40:44] = math.inf
            x["logits"][2, 690] = math.inf
            check(x)
    x = inputs(dev, torch.float32, 9, [1, 1], "none", seed=1)
    x["logits"].fill_(-math.inf)
    tokens, rows, counts = call(x)
    assert tokens.tolist() == [[-1], [-1]] and rows.tolist() == [[0], [0]] and counts.tolist() == [1, 1]


def test_numbers_at_the_ends(dev):
    """Coins and draws of 0 and just below 1, 1 itself; temperatures without end and next to zero; logits of fp32's and fp16's ends."""
    for dtype, end in ((torch.float16, 65504.0), (torch.float32, 3.0e38), (torch.bfloat16, 3.0e38)):
        for kind in ("tree", "none", "probs"):
            x = inputs(dev, dtype, 300, [4, 5, 4, 6], kind, seed=5)
            x["draws"] = torch.tensor([0.0, 1.0, 1.0 - 2.0 ** -24, 2.0 ** -30], device=dev)
            check(x)
            x["heats"] = torch.tensor([1e-30, 1e30, 3.0, 1e-3], device=dev)
            check(x)
            x["logits"][:, ::3] = end
            x["logits"][:, 1::3] = -end
            check(x)
            x["heats"] = None
            for coin in (0.0, 1.0 - 2.0 ** -24):
                y = {**x, "coins": torch.full_like(x["coins"], coin)}
                got, want = call(y), definition(y)
                assert got[2].tolist() == want[2].tolist() and np.array_equal(got[0].cpu().numpy(), want[0])


def test_a_draft_that_is_the_target(dev):
    """q = p to the last bit that fp32 holds: whatever the coin, the drafts are taken; where the last is refused by roundings, the token comes from p."""
    new = [4] * 40
    x = inputs(dev, torch.float32, 513, new, "none", seed=2)
    x["probs"] = torch.softmax(x["logits"].double(), -1).float()
    x["tokens"] = torch.multinomial(x["probs"], 1)[:, 0].roll(1)
    x["coins"] = x["coins"] * 0.9999
    tokens, rows, counts = call(x)
    assert counts.tolist() == [4] * 40
    # a draft that knows one token only, and a target that knows another: nothing is taken, and the target's own follows
    x["probs"].zero_()
    x["probs"][:, 7] = 1.0
    x["tokens"].fill_(7)
    x["logits"].fill_(-math.inf)
    x["logits"][:, 9] = 1.0
    tokens, rows, counts = call(x)
    assert counts.tolist() == [1] * 40 and tokens[:, 0].tolist() == [9] * 40
    # q covers all of p though the token is none of p's: nothing is left of p - q, so the token is drawn from p
    x["probs"].fill_(1.0)
    x["tokens"].fill_(8)
    tokens, rows, counts = call(x)
    assert counts.tolist() == [1] * 40 and tokens[:, 0].tolist() == [9] * 40


def test_children_that_cover_everything(dev):
    """A tree whose children are the whole vocabulary ends nowhere else; the same token twice counts once."""
    V, B = 3, 500
    new = [5] * B
    x = inputs(dev, torch.float32, V, new, "none", seed=4)
    x["parents"] = torch.tensor([-1, 0, 0, 0, 0] * B, dtype=torch.int32, device=dev)
    x["tokens"] = torch.tensor([0, 2, 2, 0, 1] * B, device=dev)
    check(x)
    assert set(call(x)[1][:, 1].tolist()) <= {1, 3, 4}


def test_longer_portions_and_padded_batches(dev):
    """Rows behind max_seqlen are not looked at; rows behind the last sequence belong to none; starts that run past the rows stay inside."""
    x = inputs(dev, torch.float16, 777, [6, 9, 4], "tree", seed=8)
    check(x, top=5)
    padded = {**x, "logits": torch.cat([x["logits"], torch.full((3, 777), float("nan"), dtype=torch.float16, device=dev)]), "tokens": torch.cat([x["tokens"], x["tokens"][:3]]),
              "coins": torch.cat([x["coins"], x["coins"][:3]]), "parents": torch.cat([x["parents"], x["parents"][:3]])}
    for a, b in zip(call(padded), call(x)):
        assert torch.equal(a, b)
    got = call(x, top=9, cu=torch.tensor([0, 6, 15, 400], dtype=torch.int32, device=dev))
    for a, b in zip(got, call(x, top=9)):
        assert torch.equal(a, b)


def test_plain_sampling_of_one_row_a_sequence(dev):
    """No drafts, no starts: a token for every row, as a sampler draws it."""
    x = inputs(dev, torch.bfloat16, 5001, [1] * 37, "none", seed=6)
    check(x, cu=None)
    tokens, rows, counts = call(x, top=3, cu=None)
    assert rows.tolist() == [[0, -1, -1]] * 37 and (tokens[:, 1:] == -1).all() and counts.tolist() == [1] * 37


def test_empty_calls(dev):
    none = torch.zeros(0, device=dev)
    for T, B in ((0, 0), (0, 3)):
        tokens, rows, counts = backend.verify_drafts(torch.zeros(T, 64, device=dev), torch.zeros(T, dtype=torch.int64, device=dev), torch.zeros(B + 1, dtype=torch.int32, device=dev), 2, none,
                                                     torch.zeros(B, device=dev))
        assert tokens.tolist() == [[-1, -1]] * B and rows.tolist() == [[-1, -1]] * B and counts.tolist() == [0] * B
    x = inputs(dev, torch.float16, 64, [3, 2], "none", seed=1)
    tokens, rows, counts = call(x, top=0)  # no row is looked at
    assert tokens.shape == (2, 0) and rows.shape == (2, 0) and counts.tolist() == [0, 0]
    positions, visible = backend.draft_tree(torch.zeros(0, dtype=torch.int32, device=dev), torch.zeros(1, dtype=torch.int32, device=dev), torch.zeros(0, dtype=torch.int32, device=dev), 0)
    assert positions.shape == (0,) and visible.shape == (0, 0)


@pytest.mark.parametrize("kind", ["probs", "tree"])
def test_what_comes_out_is_distributed_as_the_target(dev, kind):
    """60000 sequences of the same logits, random numbers and (with probabilities) drafts of their own: each first token as often as its probability says, within five
    standard deviations, whether it was drafted or drawn."""
    B, V, n = 60000, 6, 3
    g = torch.Generator().manual_seed(1)
    row = torch.randn(V, generator=g).to(dev)
    p = torch.softmax(row.double(), -1)
    q = torch.softmax(torch.randn(V, generator=g).to(dev), -1)
    gd = torch.Generator(device=dev).manual_seed(2)
    tokens = torch.zeros(B, n, dtype=torch.int64, device=dev)
    parents = None
    if kind == "probs":
        tokens[:, 1:] = torch.multinomial(q.expand(B, V), n - 1, replacement=True, generator=gd)
    else:
        parents = torch.tensor([-1, 0, 0], dtype=torch.int32, device=dev).repeat(B)
        tokens[:, 1], tokens[:, 2] = 4, 1
    x = {"logits": row.expand(B * n, V).contiguous(), "tokens": tokens.view(-1), "parents": parents, "probs": q.expand(B * n, V).contiguous() if kind == "probs" else None,
         "coins": torch.rand(B * n, device=dev, generator=gd), "draws": torch.rand(B, device=dev, generator=gd), "new": [n] * B, "heats": None}
    out, rows, counts = call(x)
    share = torch.bincount(out[:, 0], minlength=V).double() / B
    assert ((share - p).abs() <= 5 * (p * (1 - p) / B).sqrt()).all(), (share, p)
    assert (counts > 1).any() and (counts == 1).any()


def test_graphs_and_streams(dev):
    """Two captured calls replayed on two streams with their inputs changed in between, each what it is eagerly."""
    cases = []
    for kind, V, new in (("probs", 32000, [5, 6]), ("tree", 4097, [20, 1, 33])):
        x = inputs(dev, torch.float16, V, new, kind, seed=V)
        cu = starts(new, dev)
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        call(x, cu=cu)
        with torch.cuda.graph(graph, stream=stream):
            out = call(x, cu=cu)
        cases.append((x, cu, stream, graph, out))
    for seed in (1, 2, 3):
        for x, cu, *_ in cases:
            x["draws"].copy_(torch.rand(x["draws"].shape, generator=torch.Generator().manual_seed(seed)))
            x["coins"].copy_(torch.rand(x["coins"].shape, generator=torch.Generator().manual_seed(seed)))
        torch.cuda.synchronize()
        for _ in range(3):
            for x, cu, stream, graph, out in cases:
                with torch.cuda.stream(stream):
                    graph.replay()
        torch.cuda.synchronize()
        for x, cu, stream, graph, out in cases:
            for a, b in zip(out, call(x, cu=cu)):
                assert torch.equal(a, b)
            check(x, cu=cu)


def test_refusals(dev):
    x = inputs(dev, torch.float16, 64, [3, 2], "none", seed=1)
    bad = [dict(logits=x["logits"].double()), dict(logits=x["logits"][0]), dict(logits=x["logits"].cpu()), dict(logits=x["logits"].t().contiguous().t()), dict(tokens=x["tokens"].int()),
           dict(tokens=x["tokens"][:4]), dict(tokens=None), dict(coins=None), dict(coins=x["coins"].double()), dict(coins=x["coins"].cpu()), dict(draws=x["draws"][:, None]),
           dict(draws=x["draws"].half()), dict(parents=torch.zeros(5, dtype=torch.int64, device=dev)), dict(parents=torch.zeros(4, dtype=torch.int32, device=dev)),
           dict(probs=x["logits"]), dict(probs=x["logits"].float()[:, :63]), dict(heats=torch.ones(3, device=dev)), dict(heats=torch.ones(2, dtype=torch.half, device=dev)),
           dict(parents=torch.zeros(5, dtype=torch.int32, device=dev), probs=x["logits"].float())]
    for change in bad:
        with pytest.raises((RuntimeError, TypeError)):
            call(x, **change)
    for top in (-1, 257):
        with pytest.raises(RuntimeError):
            call(x, top=top)
    with pytest.raises(RuntimeError):
        call(x, cu=torch.zeros(2, dtype=torch.int32, device=dev))
    parents, lens = torch.zeros(5, dtype=torch.int32, device=dev), torch.zeros(2, dtype=torch.int32, device=dev)
    for a in ((parents.long(), None, lens, 2), (parents, None, lens.long(), 2), (parents, lens, lens, 2), (parents, None, lens, 257), (parents, None, lens, -1), (parents.cpu(), None, lens, 2),
              (parents[None], None, lens, 2), (parents, None, lens.cpu(), 2)):
        with pytest.raises((RuntimeError, TypeError)):
            backend.draft_tree(*a)

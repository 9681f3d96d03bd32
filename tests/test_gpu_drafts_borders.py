"""Verification of drafts where 32 bits do not tell one side from the other: drafts next to their target, of which max(p - q, 0) leaves next to nothing."""
import math

import numpy as np
import pytest
import torch

from tests.drafts_util import verify64, weights64
from tests.test_gpu_drafts import TYPES, call, definition

pytestmark = pytest.mark.gpu
ROOM = 4e-12  # a weight of 64 bits is off by 1.2e-12 of itself, so are a running sum and the whole: of a row's sum of 1, with what the definition's own roundings take


def drawn_within(rest, r, room):
    """The tokens that a draw at r may give if running sums are off by `room`."""
    sums = np.cumsum(rest)
    lo, hi = (int(np.searchsorted(sums, r * sums[-1] + e, side="right")) for e in (-room, room))
    some = np.flatnonzero(rest > 0)
    return set(some[(some >= lo) & (some <= hi)].tolist()) or {int(some[-1])}


def check_ends(x):
    """Rows and counts of the definition; the token that a sequence ends with within ROOM of its draw."""
    got, want = call(x), definition(x)
    assert want[3] > ROOM
    tokens, rows, counts = (t.cpu().numpy() for t in got)
    assert np.array_equal(counts, want[2]) and np.array_equal(rows, want[1])
    logits, probs = x["logits"].double().cpu().numpy(), x["probs"].double().cpu().numpy()
    start, other = 0, 0
    for b, n in enumerate(x["new"]):
        c = int(counts[b])
        assert tokens[b, :c - 1].tolist() == want[0][b, :c - 1].tolist()
        at = start + int(rows[b, c - 1])
        w = weights64(logits[at], 1.0)
        p = w / math.fsum(w)
        rest = np.where(p > 0, np.maximum(p - probs[at], 0.0), 0.0) if rows[b, c - 1] + 1 < n else p
        rest = rest if rest.any() else p
        if tokens[b, c - 1] != want[0][b, c - 1]:
            assert tokens[b, c - 1] in drawn_within(rest, float(x["draws"][b]), ROOM), b
            other += 1
        start += n
    return tokens, counts, other


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("refused", ["outside", "masked"])
@pytest.mark.parametrize("depth", [20, 24, 28])
@pytest.mark.parametrize("V,batch", [(40, 3), (1000, 3), (1000, 200), (4099, 20), (32003, 60), (128256, 4)])
def test_a_draft_of_the_targets_best_token_alone(dev, dtype, refused, depth, V, batch):
    """q is all on a token that has all but some 1e-12 to 1e-4 of p: a refused draft is followed by one of the others, each by its share, however little that is."""
    g = torch.Generator().manual_seed(V + depth)
    logits = (-4 + torch.randn(batch * 2, V, generator=g)).to(dtype)
    best = torch.randint(0, V, (batch * 2,), generator=g)
    logits[torch.arange(batch * 2), best] = float(depth - 4)
    child = (best + 1) % V
    tokens = torch.full((batch * 2,), -1, dtype=torch.int64)
    if refused == "masked":
        tokens[1::2] = child[::2]
        logits[torch.arange(0, batch * 2, 2), child[::2]] = -math.inf
    probs = torch.zeros(batch * 2, V)
    probs[torch.arange(batch * 2), best] = 1.0
    # (a coin above 0: at 0 times a share of 0 the decision's distance from its border is 0 as well; both sides refuse)
    x = {"logits": logits.to(dev), "tokens": tokens.to(dev), "parents": None, "probs": probs.to(dev), "coins": torch.rand(batch * 2, generator=g).to(dev),
         "draws": torch.rand(batch, generator=g).to(dev), "new": [2] * batch, "heats": None}
    if refused == "masked":  # 0 < 0 is as near to its border as can be, and refused
        x["probs"][torch.arange(0, batch * 2, 2), child[::2]] = 1e-3
        x["coins"] = x["coins"] * 0.5 + 0.25
    tokens, counts, other = check_ends(x)
    assert counts.tolist() == [1] * batch and (tokens[:, 0] != best[::2].numpy()).all()
    assert other <= 1  # (draws as near to a border as ROOM are rare)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("V,batch", [(31, 40), (513, 40), (513, 200), (5003, 12), (32003, 5)])
def test_a_draft_that_is_the_target_is_refused(dev, dtype, V, batch):
    """q is p as 32 bits round it: what is left of p - q are roundings, and the token that follows a refused draft is one of those that q has too little of."""
    g = torch.Generator().manual_seed(V)
    logits = (2.5 * torch.randn(batch * 2, V, generator=g)).to(dtype)
    probs = torch.softmax(logits.double(), -1).float()
    tokens = torch.full((batch * 2,), -1, dtype=torch.int64)
    tokens[1::2] = V + torch.arange(batch) % 3
    x = {"logits": logits.to(dev), "tokens": tokens.to(dev), "parents": None, "probs": probs.to(dev), "coins": torch.rand(batch * 2, generator=g).to(dev),
         "draws": torch.rand(batch, generator=g).to(dev), "new": [2] * batch, "heats": None}
    tokens, counts, _ = check_ends(x)
    p = torch.softmax(logits.double(), -1)
    assert counts.tolist() == [1] * batch
    some = p[::2][torch.arange(batch), torch.from_numpy(tokens[:, 0].copy())] - probs.double()[::2][torch.arange(batch), torch.from_numpy(tokens[:, 0].copy())]
    assert (some > -1e-12).all()


@pytest.mark.parametrize("batch", [3, 60, 200])
def test_coins_next_to_one_and_a_draft_that_is_the_target(dev, batch):
    """Coins of 1 - 2^-24 with q = p rounded by 32-bit operations: some drafts are refused by those roundings, and decided as the definition does."""
    V, new = 257, [4] * batch
    g = torch.Generator().manual_seed(batch)
    logits = 2.5 * torch.randn(batch * 4, V, generator=g)
    probs = torch.softmax(logits, -1) * (1 + 2.0 ** -23 * torch.randint(-1, 2, (batch * 4, V), generator=g))
    tokens = torch.multinomial(probs, 1, generator=g)[:, 0].roll(1)
    x = {"logits": logits.to(dev), "tokens": tokens.to(dev), "parents": None, "probs": probs.to(dev), "coins": torch.full((batch * 4,), 1 - 2.0 ** -24, device=dev),
         "draws": torch.rand(batch, generator=g).to(dev), "new": new, "heats": None}
    # (a decision nearer to its border than ROOM would be either's: those sequences get another coin)
    d = lambda t: t.double().cpu().numpy()
    start = 0
    for b in range(batch):
        rows = slice(start, start + 4)
        near = verify64(d(x["logits"][rows]), tokens[rows].numpy(), [4], d(x["coins"][rows]), d(x["draws"][b:b + 1]), None, d(x["probs"][rows]))[3]
        if near <= 2 * ROOM:
            x["coins"][rows] = 0.5
        start += 4
    tokens, counts, _ = check_ends(x)
    assert (counts < 4).any() and (counts == 4).any()


def test_sums_of_long_rows(dev):
    """2^20 equal weights beside a larger one, whose 32-bit sums are off one way, by up to 4.8e-5: decisions 1e-5 from their border are those of the sum itself."""
    V, B, n = 1 << 20, 150, 8
    down = (12 + torch.arange(B // 2, dtype=torch.float64) / 128).repeat(2)  # (fp16 numbers)
    p = 1 / (1 + (V - 1) * torch.exp(-down))
    side = torch.tensor([-1.0, 1.0]).repeat_interleave(B // 2)
    logits = torch.empty(B * n, V, dtype=torch.float16, device=dev)
    logits.view(B, n, V).copy_(-down.half().to(dev)[:, None, None].expand(B, n, V))
    logits[:, 5] = 0.0
    coins = (p * (1 + 1e-5 * side)).float().repeat_interleave(n)
    x = {"logits": logits, "tokens": torch.full((B * n,), 5, dtype=torch.int64, device=dev), "parents": None, "probs": None, "coins": coins.to(dev),
         "draws": torch.full((B,), 0.5, device=dev), "new": [n] * B, "heats": None}
    tokens, rows, counts = call(x)
    assert counts.tolist() == [n if s < 0 else 1 for s in side.tolist()]
    assert (tokens[B // 2:, 0] != 5).all()


@pytest.mark.parametrize("batch", [2, 200])
def test_weights_at_the_end_of_32_bits(dev, batch):
    """Children whose weights and q lie about 2^-126, or below what 32 bits hold: decided by their numbers."""
    for down in (60.0, 87.0, 87.25, 87.5, 88.0, 90.0, 95.0, 101.0, 103.5, 120.0):
        for ratio in (0.25, 0.999, 1.001, 4.0):
            q = torch.tensor(math.exp(-down) * ratio * 2, dtype=torch.float64).float()
            V, new = 33, [2] * batch
            logits = torch.full((2 * batch, V), -math.inf, device=dev)
            logits[:, 3], logits[:, 9] = 0.0, -down
            probs = torch.zeros(2 * batch, V, device=dev)
            probs[:, 9], probs[:, 3] = q.to(dev), 1.0
            x = {"logits": logits, "tokens": torch.full((2 * batch,), 9, dtype=torch.int64, device=dev), "parents": None, "probs": probs, "coins": torch.full((2 * batch,), 0.5, device=dev),
                 "draws": torch.full((batch,), 0.5, device=dev), "new": new, "heats": None}
            p, left = math.exp(-down) / (1 + math.exp(-down)), 0.5 * float(q)
            if abs(left - p) <= 1e-9 * p:  # (q has few bits here: it may have been rounded to the border itself)
                continue
            assert call(x)[2].tolist() == [2 if left < p else 1] * batch, (down, ratio)

"""Operators for steps of several drafted tokens, and of tokens with places of their own, over the quantised paged key/value cache: what they compute, in plain
torch and through `qserve_b200.backend`, and the cases they are measured on.

* tree: what each row of a portion sees of its portion and the position that it is rotated at, from the rows' parents;
* append: keys and queries rotated at given positions of one to four axes, keys and values quantised into the pages; here they are read back;
* attend: attention of portions over the cache, each row over all that lies ahead of its portion and those rows of it that its bits name;
* verify: drafted tokens, a chain or a tree, against the target's probabilities from given random numbers, and the token that follows the accepted ones;
* keep: the accepted rows' keys and values moved to the front of their portion.

A page holds 64 positions: codes [kv heads][64][128 * bits / 8], then scales and zeros [kv heads][64] in fp16; INT4 codes lie two to a byte, the even element
low.  A code u of a row with scale s and zero z stands for s u + half(-s z) (INT4) or s (u - z) (INT8).  Head sizes are 128; the numbers of heads and the sizes of
vocabularies are those of `qserve_b200.modelcfg.MODELS` and of the tests.  All inputs are random and made from the seed alone.
"""
import math

import numpy as np
import torch

own = False

PAGE, D = 64, 128
HALF, F32, F64, I32, I64 = torch.float16, torch.float32, torch.float64, torch.int32, torch.int64
BASE = 500000.0  # rotary base
HEADS = [(32, 8), (32, 32), (64, 64), (8, 2), (16, 1), (40, 8)]  # query heads, key/value heads
VOCABS = [1024, 32000, 32003, 128256, 152064]
SECTIONS = {1: (64,), 2: (20, 44), 3: (16, 24, 24), 4: (16, 16, 16, 16)}  # pairs of each axis


def listed():
    return [
        # the tree of one sequence's step: the smallest call
        {"name": "tree_b1_26", "kind": "tree", "batch": 1, "rows": 26},
        # a wide batch of large trees
        {"name": "tree_b128_64", "kind": "tree", "batch": 128, "rows": 64},
        # the rows of four small trees, rotated at their depths
        {"name": "append_int4_trees_4x13", "kind": "append", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 4, "rows": 13, "context": 1000, "axes": 1},
        # prompts with an image among the text: time, height and width, as many key/value heads as query heads
        {"name": "append_int8_images_2x4097", "kind": "append", "bits": 8, "heads": 32, "kv_heads": 32, "batch": 2, "rows": 4097, "context": 3001, "axes": 3},
        # a small tree behind a short context
        {"name": "attend_int4_tree_13", "kind": "attend", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 1, "rows": 13, "context": 500, "mask": "tree"},
        # the usual batch of a server that drafts
        {"name": "attend_int4_trees_32x16", "kind": "attend", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 32, "rows": 16, "context": 3000, "mask": "tree"},
        # prompts whose image sees itself as a whole, behind a long context, INT8: the largest case
        {"name": "attend_int8_images_2x1500", "kind": "attend", "bits": 8, "heads": 32, "kv_heads": 8, "batch": 2, "rows": 1500, "context": 12001, "mask": "image"},
        # one sequence, four drafted tokens with their probabilities, a small vocabulary
        {"name": "verify_chain_1x5", "kind": "verify", "type": "float16", "vocab": 32000, "batch": 1, "rows": 5, "draft": "probs", "heat": "none"},
        # the usual batch, a large vocabulary, temperatures of all kinds
        {"name": "verify_chains_64x6", "kind": "verify", "type": "float16", "vocab": 128256, "batch": 64, "rows": 6, "draft": "probs", "heat": "mixed"},
        # trees of the draft's best tokens, bfloat16
        {"name": "verify_trees_16x26", "kind": "verify", "type": "bfloat16", "vocab": 152064, "batch": 16, "rows": 26, "draft": "tree", "heat": "mixed"},
        # what a few sequences keep of their trees
        {"name": "keep_int4_4x26", "kind": "keep", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 4, "rows": 26, "context": 2000},
        # a wide batch of large trees, INT8, as many key/value heads as query heads
        {"name": "keep_int8_128x64", "kind": "keep", "bits": 8, "heads": 32, "kv_heads": 32, "batch": 128, "rows": 64, "context": 300},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, int(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["tree", "append", "append", "attend", "attend", "attend", "verify", "verify", "verify", "keep"])
    if kind == "tree":
        return {"kind": kind, "batch": log(1, 128), "rows": log(1, 256)}
    if kind == "verify":
        vocab, rows = rng.choice(VOCABS), log(1, 64)
        draft = rng.choice(["probs", "tree", "none"])
        batch = log(1, max(1, min(128, 45000000 // (vocab * rows))))
        return {"kind": kind, "type": rng.choice(["float16", "bfloat16", "float32"] if vocab * rows * batch < 20000000 else ["float16", "bfloat16"]), "vocab": vocab, "batch": batch,
                "rows": rows, "draft": draft, "heat": rng.choice(["none", "mixed", "greedy"])}
    heads, kv_heads = rng.choice(HEADS)
    case = {"kind": kind, "bits": rng.choice([4, 8]), "heads": heads, "kv_heads": kv_heads}
    most = 27000 * 8 // kv_heads  # positions of all sequences together
    if kind == "append":
        batch = log(1, 128)
        return {**case, "batch": batch, "rows": log(1, max(1, 8192 // batch)), "context": log(1, most // batch), "axes": rng.choice([1, 1, 2, 3, 3, 4])}
    if kind == "keep":
        batch = log(1, 128)
        return {**case, "batch": batch, "rows": log(1, 64), "context": log(1, most // batch)}
    mask = rng.choice(["tree", "tree", "image"])
    batch = log(1, 64 if mask == "tree" else 8)
    rows = log(1, 64 if mask == "tree" else max(1, 2048 // batch))
    return {**case, "batch": batch, "rows": rows, "mask": mask,
            "context": rng.choice([0, log(1, max(1, min(16000, most // batch, 40000 * 32 * 1024 // (rows * batch * heads))))])}


# ------------------------------------------------------------------------------------------------------------------------
# sizes and inputs
# ------------------------------------------------------------------------------------------------------------------------
def _ragged(count, top, step):
    """From about half of `top` up to `top`, the same for every seed."""
    return [top - (i * step) % (top // 2 + 1) for i in range(count)]


def _sizes(case):
    """New rows of every sequence, and how many positions its pages hold with them."""
    new = _ragged(case["batch"], case["rows"], 6151)
    return new, [n + c for n, c in zip(new, _ragged(case["batch"], case.get("context", 0), 7919))]


def _quantise(x, bits):
    """fp16 rows x [..., 128] -> codes, scales, zeros as the cache holds them."""
    top = float(2 ** bits - 1)
    x = x.float()
    hi, lo = x.amax(-1), x.amin(-1)
    span = hi - lo
    scale, zero = (span / top).half(), (-top * lo / span).half()
    # a row of one value, or of values too near to one another for a zero in fp16: the middle of the row, held as 1 x scale or as 0 - 1 x scale
    mid = ((hi + lo) / 2).half()
    one = (scale == 0) | ~torch.isfinite(zero)
    code = torch.round(x * (1.0 / scale.float())[..., None] + zero.float()[..., None])
    code = torch.where(one[..., None], (mid > 0).float()[..., None], code.clamp(0.0, top))
    return code.to(torch.uint8), torch.where(one, mid.abs(), scale), torch.where(one, (mid < 0).to(HALF), zero)


def _pool(g, pages, hkv, bits, keys):
    """A pool with the contents that a model leaves: normal rows, some channels of the keys several times as large as the others."""
    p = torch.empty((pages, hkv * PAGE * (D * bits // 8 + 4)), dtype=torch.uint8, device="cuda")
    wide = torch.ones(hkv, 1, D, device="cuda")
    if keys:
        wide += 2.0 * (torch.rand(hkv, 1, D, device="cuda", generator=g) < 0.06)
    for at in range(0, pages, 512):  # a few hundred MB at a time
        part = p[at:at + 512]
        n = part.shape[0]
        code, scale, zero = _quantise((torch.randn(n, hkv, PAGE, D, device="cuda", generator=g) * wide).half(), bits)
        if bits == 4:
            code = code[..., 0::2] | (code[..., 1::2] << 4)
        part[:, :hkv * PAGE * D * bits // 8] = code.reshape(n, -1)
        part[:, hkv * PAGE * D * bits // 8:] = torch.stack([scale, zero], 1).reshape(n, -1).contiguous().view(torch.uint8).view(n, -1)
    return p


def _parents(rng, new):
    """Trees: a row's parent is one of the eight rows before it; the last row of every other sequence is padding and has none."""
    out = []
    for b, n in enumerate(new):
        out += [-1] + [int(rng.integers(max(0, i - 8), i)) for i in range(1, n)]
        if b % 2 and n > 4:
            out[-1] = -1
    return out


def _bits(new, seen):
    """int64 [rows of all, words] from Python's whole numbers, one for each row."""
    words = (max(new) + 63) // 64
    flat = np.array([[(x >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for x in seen], dtype=np.uint64)
    return torch.from_numpy(flat.view(np.int64).reshape(len(seen), words)).cuda()


def _mask(case, new, parents):
    seen = []
    for n in new:
        base = len(seen)
        for i in range(n):
            if case["mask"] == "tree":
                up = parents[base + i]
                seen.append(1 << i | (seen[base + up] if up >= 0 else 0) if i == 0 or up >= 0 else 0)
            else:  # causal, but for an image that sees itself as a whole
                seen.append((1 << (n // 2 if n // 4 <= i < n // 2 else i + 1)) - 1)
    return _bits(new, seen)


def _positions(case, new, held, parents):
    """int32 [axes, rows]: depths of a tree, or places of text around an image."""
    out = []
    for n, m in zip(new, held):
        if case["axes"] == 1:
            base, depth = len(out), []
            for i in range(n):
                up = parents[base + i]
                depth.append(depth[up] + 1 if up >= 0 else 0)
            out += [[m - n + d] for d in depth]
            continue
        side = max(1, math.isqrt(3 * n // 4))
        lo, hi = n // 8, n // 8 + 3 * n // 4
        for i in range(n):
            r, c = divmod(i - lo, side)
            first = m - n
            out.append(([first + lo, first + lo + r, first + lo + c, first + i][:case["axes"]] if lo <= i < hi else [first + (i if i < lo else lo + side + i - hi)] * case["axes"]))
    return torch.tensor(out, dtype=I32).t().contiguous().cuda()


def _verify_inputs(case, g, rng, new, parents, starts):
    T, V, B = sum(new), case["vocab"], case["batch"]
    logits = 2.5 * torch.randn(T, V, device="cuda", generator=g)
    strong = torch.randint(0, V, (T, 6), device="cuda", generator=g)
    logits.scatter_(1, strong, torch.rand(T, 6, device="cuda", generator=g) * 6 + 9)
    if case["heat"] == "mixed":
        logits[:, V - V // 100:] = -math.inf  # rows of the table that are no tokens
    drafted = logits + torch.randn(T, V, device="cuda", generator=g)
    probs = None
    if case["draft"] == "probs":
        probs = torch.softmax(drafted, -1)
        chosen = (drafted - torch.log(-torch.log(torch.rand(T, V, device="cuda", generator=g).clamp(1e-20, 1 - 1e-7)))).argmax(-1)[:, None]
    else:
        chosen = drafted.topk(8 if case["draft"] == "tree" else 1, -1).indices
    tokens = torch.zeros(T, dtype=I64)
    chosen, row = chosen.cpu(), 0
    for n in new:
        children = {}
        for i in range(n):
            up = parents[row + i] if case["draft"] == "tree" else i - 1
            k = children[up] = children.get(up, -1) + 1  # (a ninth child has the first one's token again)
            tokens[row + i] = chosen[row + up, k % chosen.shape[1]] if up >= 0 else int(rng.integers(0, V))
        row += n
    heat = {"none": None, "greedy": torch.zeros(B), "mixed": torch.tensor([0.0 if b % 4 == 3 else float(rng.uniform(0.6, 1.3)) for b in range(B)])}[case["heat"]]
    return {"logits": logits.to(getattr(torch, case["type"])), "tokens": tokens.cuda(), "probs": probs, "coins": torch.rand(T, device="cuda", generator=g),
            "draws": torch.rand(B, device="cuda", generator=g), "heat": None if heat is None else heat.float().cuda()}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    rng = np.random.default_rng(seed)
    B = case["batch"]
    new, held = _sizes(case)
    T = sum(new)
    i32 = lambda x: torch.tensor(x, dtype=I32, device="cuda")
    starts = [sum(new[:i]) for i in range(B + 1)]
    parents = _parents(rng, new)
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(new, device="cuda"))
    at = torch.arange(T, device="cuda") - i32(starts).long()[seq]  # of its portion
    s = {"case": case, "cu": i32(starts), "lens": i32(held), "parents": i32(parents), "new": max(new), "top": max(held), "T": T, "seq": seq, "at": at}
    if case["kind"] == "tree":
        return {**s, "lens": i32([n + int(rng.integers(0, 20000)) for n in new])}
    if case["kind"] == "verify":
        return {**s, **_verify_inputs(case, g, rng, new, parents, starts)}
    bits, hq, hkv = case["bits"], case["heads"], case["kv_heads"]
    blocks = (max(held) + PAGE - 1) // PAGE
    s["pages"] = torch.randperm(B * blocks, device="cuda", generator=g).view(B, blocks)
    s["pools"] = [_pool(g, B * blocks, hkv, bits, keys) for keys in (True, False)]
    s["table"] = torch.stack([p.data_ptr() + s["pages"] * p.shape[1] for p in s["pools"]], 1).contiguous()
    s["first"] = i32(held).long() - i32(new).long()
    s["pos"] = s["first"][seq] + at
    if case["kind"] == "keep":
        # half of a portion's rows at most, from its second half but for the root, in order
        rows, counts = torch.full((B, max(new)), -1, dtype=I32), []
        for b, n in enumerate(new):
            k = 1 + int(rng.integers(0, (n + 1) // 2))
            rows[b, :k] = torch.tensor([0] + sorted(int(x) for x in rng.choice(np.arange(k, n), k - 1, replace=False)), dtype=I32)
            counts.append(k)
        return {**s, "rows": rows.cuda(), "counts": i32(counts)}
    qkv = torch.randn(T, (hq + 2 * hkv) * D, device="cuda", generator=g).half()
    s["q"], s["k"], s["v"] = (t.unflatten(1, (-1, D)) for t in qkv.split([hq * D, hkv * D, hkv * D], 1))
    if case["kind"] == "append":
        return {**s, "positions": _positions(case, new, held, parents)}
    return {**s, "q": s["q"].contiguous(), "visible": _mask(case, new, parents)}


# ------------------------------------------------------------------------------------------------------------------------
# plain form
# ------------------------------------------------------------------------------------------------------------------------
def _values(pool, pages, hkv, bits):
    """What whole pages stand for: [..., positions, kv heads, 128] in fp32."""
    raw = pool[pages]
    lead, cut = raw.shape[:-2], hkv * PAGE * D * bits // 8
    code = raw[..., :cut].unflatten(-1, (hkv, PAGE, D * bits // 8))
    if bits == 4:
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2)
    meta = raw[..., cut:].contiguous().view(HALF).unflatten(-1, (2, hkv, PAGE)).float()
    scale, zero = meta[..., 0, :, :, None], meta[..., 1, :, :, None]
    x = scale * code + (-scale * zero).half() if bits == 4 else scale * (code - zero)
    return x.transpose(-3, -2).reshape(*lead, -1, hkv, D)


def _cell_views(pool, s):
    c = s["case"]
    hkv, cut = c["kv_heads"], c["kv_heads"] * PAGE * D * c["bits"] // 8
    return pool[:, :cut].view(-1, hkv, PAGE, D * c["bits"] // 8), pool.view(HALF)[:, cut // 2:].view(-1, 2, hkv, PAGE)


def _rows(pool, s):
    """What the portions' places stand for: [T, kv heads, 128] in fp16."""
    page, slot = s["pages"][s["seq"], s["pos"] // PAGE], s["pos"] % PAGE
    codes, metas = _cell_views(pool, s)
    code, meta = codes[page, :, slot], metas[page, :, :, slot].float()
    if s["case"]["bits"] == 4:
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2)
    scale, zero = meta[:, 0, :, None], meta[:, 1, :, None]
    return (scale * code + (-scale * zero).half() if s["case"]["bits"] == 4 else scale * (code - zero)).half()


def _place(pool, s, x):
    page, slot = s["pages"][s["seq"], s["pos"] // PAGE], s["pos"] % PAGE
    code, scale, zero = _quantise(x, s["case"]["bits"])
    if s["case"]["bits"] == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    codes, metas = _cell_views(pool, s)
    codes[page, :, slot] = code
    metas[page, :, :, slot] = torch.stack([scale, zero], 1)


def _rotate(x, s):
    axis = torch.repeat_interleave(torch.arange(s["case"]["axes"], device="cuda"), torch.tensor(SECTIONS[s["case"]["axes"]], device="cuda"))
    angle = s["positions"][axis].t().to(F64) / BASE ** (torch.arange(D // 2, device="cuda", dtype=F64) * 2 / D)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat([cos * a - sin * b, cos * b + sin * a], -1).half()


def _plain_tree(s):
    B, n, T = s["case"]["batch"], s["new"], s["T"]
    up = torch.full((B, n), -1, device="cuda")
    up[s["seq"], s["at"]] = s["parents"].long()
    words = (n + 63) // 64
    seen, depth = torch.zeros(B, n, words, dtype=I64, device="cuda"), torch.zeros(B, n, dtype=I64, device="cuda")
    every = torch.arange(B, device="cuda")
    for i in range(n):
        inside = (up[:, i] >= 0) & (up[:, i] < i)
        above = up[:, i].clamp(0, max(i - 1, 0))
        bit = torch.tensor(1, dtype=I64, device="cuda") << (i % 64)
        row = seen[every, above] if i else seen[:, 0].clone()
        row[:, i // 64] |= bit
        seen[:, i] = torch.where(inside[:, None] | (i == 0), row, 0)
        depth[:, i] = torch.where(inside, depth[every, above] + 1, 0) if i else 0
    first = s["lens"].long() - (s["cu"][1:] - s["cu"][:-1]).long()
    return {"positions": (first[:, None] + depth)[s["seq"], s["at"]].to(I32), "visible": seen[s["seq"], s["at"]]}


def _plain_attend(s):
    c = s["case"]
    hq, hkv, bits, B = c["heads"], c["kv_heads"], c["bits"], c["batch"]
    G, n, L = hq // hkv, s["new"], s["pages"].shape[1] * PAGE
    q = torch.zeros(B, n, hq, D, device="cuda")
    q[s["seq"], s["at"]] = s["q"].float()
    q = q.view(B, n, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * n, D)
    scores = q @ _values(s["pools"][0], s["pages"], hkv, bits).permute(0, 2, 3, 1) * D ** -0.5
    # which new row a position holds: below zero ahead of the portion
    which = torch.arange(L, device="cuda")[None] - s["first"][:, None]
    word = torch.zeros(B, n, s["visible"].shape[1], dtype=I64, device="cuda")
    word[s["seq"], s["at"]] = s["visible"]
    among = which.clamp(0, n - 1)
    bit = (torch.gather(word, 2, (among // 64)[:, None].expand(B, n, L)) >> (among % 64)[:, None]) & 1
    count = (s["cu"][1:] - s["cu"][:-1]).long()
    seen = (which < 0)[:, None] | ((bit == 1) & (which < count[:, None])[:, None])
    scores = scores.view(B, hkv, G, n, L).masked_fill(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    e = torch.exp(scores - torch.where(top == -math.inf, 0.0, top))
    w = e / e.sum(-1, keepdim=True).clamp_min(1e-30)  # a row that sees nothing: zeros
    out = (w.view(B, hkv, G * n, L) @ _values(s["pools"][1], s["pages"], hkv, bits).transpose(1, 2)).view(B, hq, n, D)
    return out.transpose(1, 2)[s["seq"], s["at"]].half()


def _plain_verify(s):
    c = s["case"]
    B, n, V = c["batch"], s["new"], c["vocab"]
    heat = torch.ones(B, device="cuda") if s["heat"] is None else s["heat"]
    warm = torch.where(heat > 0, heat, 1.0).to(F64)[s["seq"]][:, None]
    x = s["logits"].to(F64) / warm
    top = x.amax(-1, keepdim=True)
    best = torch.where(x == top, torch.arange(V, device="cuda"), V).amin(-1)
    e = torch.exp(x - top)
    z = e.sum(-1)
    start, count = s["cu"][:-1].long(), (s["cu"][1:] - s["cu"][:-1]).long()
    tok, up = torch.full((B, n), -1, device="cuda"), torch.full((B, n), -2, device="cuda")
    tok[s["seq"], s["at"]] = s["tokens"]
    up[s["seq"], s["at"]] = s["parents"].long() if c["draft"] == "tree" else s["at"] - 1
    every, last = torch.arange(B, device="cuda"), s["T"] - 1
    node, mass = torch.zeros(B, dtype=I64, device="cuda"), torch.zeros(B, dtype=F64, device="cuda")
    rows, tokens = torch.full((B, n), -1, dtype=I64, device="cuda"), torch.full((B, n), -1, dtype=I64, device="cuda")
    rows[:, 0], accepted = 0, torch.zeros(B, dtype=I64, device="cuda")
    for i in range(1, n):
        row, t = (start + node).clamp(max=last), tok[:, i].clamp(0, V - 1)
        child = (up[:, i] == node) & (i < count) & (tok[:, i] == t)
        p, u = e[row, t] / z[row], s["coins"][row].to(F64)
        if c["draft"] == "probs":
            take = u * s["probs"][row, t].to(F64) < p
        else:
            again = ((up[:, :i] == node[:, None]) & (tok[:, :i] == tok[:, i:i + 1]))[:, 1:].any(1)
            mass = mass + torch.where(child & ~again, p, 0.0)
            take = (u < mass) & ~again
        take = child & torch.where(heat > 0, take, best[row] == t)
        tokens[every, accepted] = torch.where(take, tok[:, i], tokens[every, accepted])
        accepted = accepted + take
        rows[every, accepted] = torch.where(take, torch.full_like(node, i), rows[every, accepted])
        node, mass = torch.where(take, i, node), torch.where(take, 0.0, mass)
    row = start + node
    full = e[row]
    if c["draft"] == "probs":
        w = torch.where((node < count - 1)[:, None], (full / z[row][:, None] - s["probs"][row].to(F64)).clamp_min(0.0), full)
    else:
        w = full.clone()
        for i in range(1, n):
            child = (up[:, i] == node) & (i < count)
            t = tok[:, i].clamp(0, V - 1)
            w[every, t] = torch.where(child & (tok[:, i] == t), 0.0, w[every, t])
    w = torch.where(w.sum(-1, keepdim=True) > 0, w, full)
    run_up = w.cumsum(-1)
    end = torch.where(w > 0, torch.arange(V, device="cuda"), -1).amax(-1)
    drawn = torch.searchsorted(run_up, (s["draws"].to(F64) * run_up[:, -1])[:, None], right=True)[:, 0]
    tokens[every, accepted] = torch.where(heat > 0, torch.minimum(drawn, end), best[row])
    return {"tokens": tokens, "rows": rows.to(I32), "counts": (accepted + 1).to(I32)}


def _plain_keep(s):
    B, K = s["rows"].shape
    kept = torch.arange(K, device="cuda")[None] < s["counts"][:, None]
    b, j = torch.nonzero(kept, as_tuple=True)
    src, dst = s["first"][b] + s["rows"].long()[b, j], s["first"][b] + j
    for pool in s["pools"]:
        for view, axes in zip(_cell_views(pool, s), (1, 2)):
            here = (s["pages"][b, src // PAGE], *[slice(None)] * axes, src % PAGE)
            there = (s["pages"][b, dst // PAGE], *[slice(None)] * axes, dst % PAGE)
            view[there] = view[here]
    return {"lengths": (s["first"] + s["counts"]).to(I32), "k": _rows(s["pools"][0], s), "v": _rows(s["pools"][1], s)}


def _plain_append(s):
    q, k = _rotate(s["q"], s), _rotate(s["k"], s)
    _place(s["pools"][0], s, k)
    _place(s["pools"][1], s, s["v"])
    return {"q": q, "k": _rows(s["pools"][0], s), "v": _rows(s["pools"][1], s)}


# ------------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------------
def _own(s):
    from qserve_b200 import backend
    c = s["case"]
    if c["kind"] == "tree":
        positions, visible = backend.draft_tree(s["parents"], s["cu"], s["lens"], s["new"])
        return {"positions": positions, "visible": visible}
    if c["kind"] == "verify":
        tokens, rows, counts = backend.verify_drafts(s["logits"], s["tokens"], s["cu"], s["new"], s["coins"], s["draws"],
                                                     parents=s["parents"] if c["draft"] == "tree" else None, draft_probs=s["probs"], temperatures=s["heat"])
        return {"tokens": tokens, "rows": rows, "counts": counts}
    int4, size = c["bits"] == 4, c["kv_heads"] * D * c["bits"] // 8
    if c["kind"] == "attend":
        return backend.paged_tree_attention(s["q"], s["table"], s["cu"], s["lens"], s["visible"], s["new"], s["top"], PAGE, size, int4, True)
    if c["kind"] == "append":
        first = {"q": backend.append_kv_cache_at(s["q"], s["k"], s["v"], s["table"], s["cu"], s["lens"], s["positions"], SECTIONS[c["axes"]], PAGE, size, D, BASE, int4, True)}
    else:
        first = {"lengths": backend.keep_kv_cache(s["table"], s["cu"], s["lens"], s["rows"], s["counts"], PAGE, size, int4, True)}
    k, v = backend.read_kv_cache(s["table"], s["cu"], s["lens"], s["T"], PAGE, size, int4, True)
    return {**first, "k": k, "v": v}


def run(state):
    if own:
        return _own(state)
    return {"tree": _plain_tree, "append": _plain_append, "attend": _plain_attend, "verify": _plain_verify, "keep": _plain_keep}[state["case"]["kind"]](state)


def work(case):
    new, held = _sizes(case)
    T, B = sum(new), case["batch"]
    if case["kind"] == "tree":
        words = (max(new) + 63) // 64
        return {"bytes": T * (4 + 4 + 8 * words) + 8 * B, "flops": T * (words + 1)}
    if case["kind"] == "verify":
        # of a tree the rows that are walked: about three a sequence
        rows = T if case["draft"] != "tree" else sum(min(n, 3) for n in new)
        size = {"float16": 2, "bfloat16": 2, "float32": 4}[case["type"]]
        probs = 4 * B * case["vocab"] if case["draft"] == "probs" else 0
        return {"bytes": rows * case["vocab"] * size + probs + T * 16 + B * max(new) * 12, "flops": 4 * rows * case["vocab"]}
    hq, hkv, cell = case["heads"], case["kv_heads"], case["kv_heads"] * (D * case["bits"] // 8 + 4) * 2
    if case["kind"] == "append":  # q, k, v in; q, cells, and what they stand for out
        return {"bytes": T * ((hq + 2 * hkv) * D * 2 + hq * D * 2 + cell + 2 * hkv * D * 2 + 4 * case["axes"]), "flops": T * ((hq + hkv) * D * 3 + 2 * hkv * D * 6)}
    if case["kind"] == "keep":  # about a quarter of the rows move; all are read
        return {"bytes": T * (cell // 2 + cell + 2 * hkv * D * 2), "flops": T * 2 * hkv * D * 2}
    if case["mask"] == "tree":  # about five of its portion
        pairs = sum(n * (m - n) + n * min(n, 5) for n, m in zip(new, held))
    else:
        pairs = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, held))
    return {"bytes": 2 * T * hq * D * 2 + sum(held) * cell + T * 8 * ((max(new) + 63) // 64), "flops": 4 * D * hq * pairs}


# ------------------------------------------------------------------------------------------------------------------------
# the definition in 64 bits
# ------------------------------------------------------------------------------------------------------------------------
def _cells(pool, row, lo, hi, hkv, bits):
    """Positions lo .. hi - 1 of a sequence with page numbers `row`: [hi - lo, kv heads, 128] in 64 bits."""
    t = torch.arange(lo, hi, device="cuda")
    page = pool[row[torch.div(t, PAGE, rounding_mode="floor")]]
    per = D * bits // 8
    got = []
    for h in range(hkv):
        place = (h * PAGE + t % PAGE)[:, None]
        byte = torch.gather(page, 1, place * per + torch.arange(per, device="cuda")).to(torch.int64)
        u = torch.stack((byte % 16, byte // 16), 2).reshape(len(t), D) if bits == 4 else byte
        words = page[:, hkv * PAGE * per:].contiguous().view(HALF)
        sc, ze = (torch.gather(words, 1, place + kind * hkv * PAGE).to(F64) for kind in (0, 1))
        got.append(u.to(F64) * sc + (-(sc * ze)).to(HALF).to(F64) if bits == 4 else (u.to(F64) - ze) * sc)
    return torch.stack(got, 1)


def _turned(x, s):
    out = torch.empty(x.shape, dtype=F64, device="cuda")
    ends = np.cumsum(SECTIONS[s["case"]["axes"]])
    for i in range(D // 2):
        w = s["positions"][int(np.searchsorted(ends, i, side="right"))].to(F64) * BASE ** (-2.0 * i / D)
        c, sn = torch.cos(w)[:, None], torch.sin(w)[:, None]
        lo, hi = x[..., i].to(F64), x[..., i + D // 2].to(F64)
        out[..., i], out[..., i + D // 2] = lo * c - hi * sn, hi * c + lo * sn
    return out


def _held(x, bits):
    """What the cache makes of rows of fp16 values: scale and zero are stored in fp16, codes are the nearest."""
    top = 2 ** bits - 1
    x = x.to(F64)
    big, small = x.max(-1, keepdim=True).values, x.min(-1, keepdim=True).values
    sc = ((big - small) / top).to(HALF).to(F64)
    ze = (-top * small / (big - small)).to(HALF).to(F64)
    u = torch.clamp(torch.round(x / sc + ze), 0, top)
    return u * sc + (-(sc * ze)).to(HALF).to(F64) if bits == 4 else (u - ze) * sc


def _exact_tree(s):
    new, held = _sizes(s["case"])[0], s["lens"].tolist()
    parents, positions, seen, row = s["parents"].tolist(), [], [], 0
    for n, m in zip(new, held):
        for i in range(n):
            path, at = [], i
            while at > 0 and 0 <= parents[row + at] < at:
                path.append(at)
                at = parents[row + at]
            rooted = at == 0
            stray = not rooted and not path  # padding sees nothing, not itself either
            # what hangs below padding sees its own way up to there
            positions.append(m - n + len(path))
            seen.append(0 if stray else sum(1 << k for k in path) + (1 if rooted else 0))
        row += n
    return {"positions": torch.tensor(positions, dtype=I32, device="cuda"), "visible": _bits(new, seen)}


def _exact_verify(s):
    c = s["case"]
    new, _ = _sizes(c)
    n, V = max(new), c["vocab"]
    toks, parents, coins, draws = s["tokens"].tolist(), s["parents"].tolist(), s["coins"].tolist(), s["draws"].tolist()
    heats = [1.0] * c["batch"] if s["heat"] is None else s["heat"].tolist()
    out = {"tokens": np.full((c["batch"], n), -1, dtype=np.int64), "rows": np.full((c["batch"], n), -1, dtype=np.int32), "counts": np.zeros(c["batch"], dtype=np.int32)}
    start = 0
    for b, m in enumerate(new):
        chain, node, path = c["draft"] != "tree", 0, [0]
        while True:
            x = s["logits"][start + node].double().cpu().numpy()
            children = [i for i in range(node + 1, m) if (i - 1 if chain else parents[start + i]) == node]
            follow = None
            if heats[b] == 0.0:
                final = int(np.argmax(x))
                follow = next((i for i in children if toks[start + i] == final), None)
            else:
                p = np.exp(x / heats[b] - np.max(x / heats[b]))
                p /= math.fsum(p)
                if c["draft"] == "probs":
                    q = s["probs"][start + node].double().cpu().numpy()
                    rest = np.maximum(p - q, 0.0) if children else p
                    follow = next((i for i in children if coins[start + node] * q[toks[start + i]] < p[toks[start + i]]), None)
                else:
                    rest, mass = p.copy(), 0.0
                    for i in children:
                        mass += rest[toks[start + i]]
                        if follow is None and rest[toks[start + i]] > 0 and coins[start + node] < mass:
                            follow = i
                        rest[toks[start + i]] = 0.0
                if not rest.any():
                    rest = p
                sums = np.cumsum(rest)
                final = min(int(np.searchsorted(sums, draws[b] * sums[-1], side="right")), int(np.flatnonzero(rest)[-1]))
            if follow is None:
                break
            path.append(follow)
            node = follow
        out["counts"][b] = len(path)
        out["rows"][b, :len(path)] = path
        out["tokens"][b, :len(path)] = [toks[start + i] for i in path[1:]] + [final]
        start += m
    return {k: torch.from_numpy(v).cuda() for k, v in out.items()}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "tree":
        return _exact_tree(s)
    if case["kind"] == "verify":
        return _exact_verify(s)
    hq, hkv, bits = case["heads"], case["kv_heads"], case["bits"]
    new, held = _sizes(case)
    kp, vp = s["pools"]
    if case["kind"] == "append":
        return {"q": _turned(s["q"], s), "k": _held(_turned(s["k"], s).to(HALF), bits), "v": _held(s["v"], bits)}
    if case["kind"] == "keep":
        out = {"lengths": [], "k": [], "v": []}
        for b, (n, m) in enumerate(zip(new, held)):
            k = int(s["counts"][b])
            order = s["rows"][b, :k].long().cpu().tolist() + list(range(k, n))
            out["lengths"].append(m - n + k)
            for name, pool in (("k", kp), ("v", vp)):
                out[name].append(_cells(pool, s["pages"][b], m - n, m, hkv, bits)[order])
        return {"lengths": torch.tensor(out["lengths"], dtype=I32, device="cuda"), "k": torch.cat(out["k"]), "v": torch.cat(out["v"])}
    out, at = torch.zeros(s["T"], hq, D, dtype=F64, device="cuda"), 0
    for b, (n, m) in enumerate(zip(new, held)):
        k, v = (_cells(p, s["pages"][b], 0, m, hkv, bits) for p in (kp, vp))
        words = s["visible"][at:at + n].cpu().numpy()
        own_rows = np.stack([words[:, j // 64] >> np.int64(j % 64) & 1 for j in range(n)], 1) == 1
        seen = torch.ones(n, m, dtype=torch.bool, device="cuda")
        seen[:, m - n:] = torch.from_numpy(own_rows).cuda()
        some = seen.any(1)
        for h in range(hq):
            g = h * hkv // hq
            scores = (s["q"][at:at + n, h].to(F64) @ k[:, g].T) / math.sqrt(D)
            w = torch.softmax(scores.masked_fill(~seen, -math.inf)[some], 1)
            out[at:at + n, h][some] = w @ v[:, g]
        at += n
    return out

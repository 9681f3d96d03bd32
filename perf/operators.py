"""Operators over the quantised paged key/value cache for prompts that come in portions and for batches that share a long prefix: what they compute, in
plain torch and through `qserve_b200.backend`, and the cases they are measured on.

* append: a portion of each sequence (a single token or thousands) is rotated at its positions behind what the cache holds, its keys and values are
  quantised and put into the pages; here they are read back, so that what the pages stand for can be compared;
* read: positions of sequences out of their pages, as fp16;
* prompt: causal attention of portions of prompts over everything the cache holds of their sequences;
* shared: attention of one token per sequence where the sequences' first pages are the same pages.

A page holds 64 positions: codes [kv heads][64][128 * bits / 8], then scales and zeros [kv heads][64] in fp16; INT4 codes lie two to a byte, the even element
low.  A code u of a row with scale s and zero z stands for s u + half(-s z) (INT4) or s (u - z) (INT8).  Head sizes are 128; the numbers of heads are those of
`qserve_b200.modelcfg.MODELS` and of the tests.  All inputs are random and made from the seed alone.
"""
import math

import torch

own = False

PAGE, D = 64, 128
HALF, F32, F64 = torch.float16, torch.float32, torch.float64
BASE = 500000.0  # rotary base
HEADS = [(32, 8), (32, 32), (64, 64), (8, 2), (16, 1), (40, 8)]  # query heads, key/value heads


def listed():
    return [
        # decoded tokens of a batch of 16 take their places in the cache: the smallest call of a step
        {"name": "append_int4_b16", "kind": "append", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 16, "tokens": 1, "context": 1000},
        # a mixed step of portions of odd sizes, as many key/value heads as query heads
        {"name": "append_int8_portions", "kind": "append", "bits": 8, "heads": 32, "kv_heads": 32, "batch": 5, "tokens": 301, "context": 3001},
        # one long portion far into a sequence
        {"name": "append_int4_8192", "kind": "append", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 1, "tokens": 8192, "context": 100000},
        # the last pages of a few sequences, taken out
        {"name": "read_int8_3x200", "kind": "read", "bits": 8, "heads": 8, "kv_heads": 2, "batch": 3, "tokens": 200, "context": 0},
        # a whole long context
        {"name": "read_int4_50000", "kind": "read", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 2, "tokens": 50000, "context": 0},
        # a question of 17 tokens behind a short context
        {"name": "prompt_int4_17", "kind": "prompt", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 1, "tokens": 17, "context": 500},
        # ragged portions of six prompts
        {"name": "prompt_int8_6x250", "kind": "prompt", "bits": 8, "heads": 32, "kv_heads": 32, "batch": 6, "tokens": 250, "context": 2047},
        # a short portion behind a long document: few rows, many keys
        {"name": "prompt_int4_24_at_60000", "kind": "prompt", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 1, "tokens": 24, "context": 60000},
        # a large portion behind a long context: the largest case
        {"name": "prompt_int4_4096", "kind": "prompt", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 1, "tokens": 4096, "context": 12000},
        # a small batch behind a short system prompt
        {"name": "shared_int4_b8", "kind": "shared", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 8, "shared": 1024, "context": 100},
        # the usual batch behind a long one
        {"name": "shared_int4_b64", "kind": "shared", "bits": 4, "heads": 32, "kv_heads": 8, "batch": 64, "shared": 8192, "context": 700},
        # a wide batch behind a document, INT8, as many key/value heads as query heads
        {"name": "shared_int8_b128", "kind": "shared", "bits": 8, "heads": 32, "kv_heads": 32, "batch": 128, "shared": 16384, "context": 511},
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))

    kind = rng.choice(["append", "read", "prompt", "prompt", "shared", "shared"])
    heads, kv_heads = rng.choice(HEADS)
    case = {"kind": kind, "bits": rng.choice([4, 8]), "heads": heads, "kv_heads": kv_heads}
    most = 65536 // kv_heads * 8  # positions of all sequences together
    if kind == "append":
        batch = log(1, 128)
        return {**case, "batch": batch, "tokens": rng.choice([1, log(1, max(1, 8192 // batch))]), "context": log(1, most // batch)}
    if kind == "read":
        batch = log(1, 64)
        return {**case, "batch": batch, "tokens": log(1, most // batch), "context": rng.choice([0, log(1, 1000)])}
    if kind == "prompt":
        batch = log(1, 8)
        tokens = log(1, 4096 // batch)
        return {**case, "batch": batch, "tokens": tokens, "context": log(1, max(1, min(16000, most // batch, 12000 * 4096 * 8 // (tokens * batch * heads))))}
    batch = log(1, 128)
    return {**case, "batch": batch, "shared": PAGE * log(1, 256), "context": log(1, min(2000, most // batch))}


# ------------------------------------------------------------------------------------------------------------------------
# sizes and inputs
# ------------------------------------------------------------------------------------------------------------------------
def _ragged(count, top, step):
    """From about half of `top` up to `top`, the same for every seed."""
    return [top - (i * step) % (top // 2 + 1) for i in range(count)]


def _sizes(case):
    """New tokens of every sequence, and how many positions its pages hold with them."""
    if case["kind"] == "shared":
        return [1] * case["batch"], [case["shared"] + n for n in _ragged(case["batch"], case["context"], 7919)]
    new = _ragged(case["batch"], case["tokens"], 6151)
    if case["kind"] == "read" and not case["context"]:
        return new, new
    return new, [n + c for n, c in zip(new, _ragged(case["batch"], case["context"], 7919))]


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


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    bits, hq, hkv, B = case["bits"], case["heads"], case["kv_heads"], case["batch"]
    new, held = _sizes(case)
    blocks = (max(held) + PAGE - 1) // PAGE
    first = case["shared"] // PAGE if case["kind"] == "shared" else 0
    count = first + B * (blocks - first)
    place = torch.randperm(count, device="cuda", generator=g)
    pages = torch.cat([place[:first].expand(B, first), place[first:].view(B, blocks - first)], 1).contiguous()
    pools = [_pool(g, count, hkv, bits, keys) for keys in (True, False)]
    table = torch.stack([p.data_ptr() + pages * p.shape[1] for p in pools], 1).contiguous()
    T = sum(new)
    qkv = torch.randn(T, (hq + 2 * hkv) * D, device="cuda", generator=g).half()
    q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([hq * D, hkv * D, hkv * D], 1))
    if case["kind"] in ("prompt", "shared"):
        q = q.contiguous()  # as rotated
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    starts = [sum(new[:i]) for i in range(B + 1)]
    # plain indexing of the same layout: sequence and position of every new token
    seq = torch.repeat_interleave(torch.arange(B, device="cuda"), torch.tensor(new, device="cuda"))
    pos = (i32(held) - i32(new) - i32(starts[:-1])).long()[seq] + torch.arange(T, device="cuda")
    return {"case": case, "pools": pools, "pages": pages, "table": table, "q": q, "k": k, "v": v, "cu": i32(starts), "lens": i32(held), "seq": seq, "pos": pos,
            "new": max(new), "top": max(held), "T": T}


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


def _rows(pool, s):
    """What the new tokens' places stand for: [T, kv heads, 128] in fp32."""
    c = s["case"]
    hkv, bits = c["kv_heads"], c["bits"]
    page, slot, cut = s["pages"][s["seq"], s["pos"] // PAGE], s["pos"] % PAGE, hkv * PAGE * D * bits // 8
    code = pool[:, :cut].view(-1, hkv, PAGE, D * bits // 8)[page, :, slot]
    if bits == 4:
        code = torch.stack([code & 15, code >> 4], -1).flatten(-2)
    meta = pool.view(HALF)[:, cut // 2:].view(-1, 2, hkv, PAGE)[page, :, :, slot].float()
    scale, zero = meta[:, 0, :, None], meta[:, 1, :, None]
    return scale * code + (-scale * zero).half() if bits == 4 else scale * (code - zero)


def _place(pool, s, x):
    c = s["case"]
    hkv, bits = c["kv_heads"], c["bits"]
    page, slot, cut = s["pages"][s["seq"], s["pos"] // PAGE], s["pos"] % PAGE, hkv * PAGE * D * bits // 8
    code, scale, zero = _quantise(x, bits)
    if bits == 4:
        code = code[..., 0::2] | (code[..., 1::2] << 4)
    pool[:, :cut].view(-1, hkv, PAGE, D * bits // 8)[page, :, slot] = code
    pool.view(HALF)[:, cut // 2:].view(-1, 2, hkv, PAGE)[page, :, :, slot] = torch.stack([scale, zero], 1)


def _rotate(x, pos):
    angle = pos.to(F64)[:, None] / BASE ** (torch.arange(D // 2, device="cuda", dtype=F64) * 2 / D)
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]
    a, b = x.float().chunk(2, -1)
    return torch.cat([cos * a - sin * b, cos * b + sin * a], -1).half()


def _weights(scores):
    e = torch.exp(scores - scores.amax(-1, keepdim=True))
    return e / e.sum(-1, keepdim=True)


def _plain(s):
    c = s["case"]
    hq, hkv, bits, B = c["heads"], c["kv_heads"], c["bits"], c["batch"]
    if c["kind"] == "append":
        q, k = _rotate(s["q"], s["pos"]), _rotate(s["k"], s["pos"])
        _place(s["pools"][0], s, k)
        _place(s["pools"][1], s, s["v"])
        return {"q": q, "k": _rows(s["pools"][0], s).half(), "v": _rows(s["pools"][1], s).half()}
    if c["kind"] == "read":
        return {"k": _rows(s["pools"][0], s).half(), "v": _rows(s["pools"][1], s).half()}
    G = hq // hkv
    if c["kind"] == "prompt":
        n, L = s["new"], s["pages"].shape[1] * PAGE
        at = torch.arange(s["T"], device="cuda") - s["cu"].long()[s["seq"]]
        q = torch.zeros(B, n, hq, D, device="cuda")
        q[s["seq"], at] = s["q"].float()
        limit = torch.full((B, n), -1, device="cuda")
        limit[s["seq"], at] = s["pos"]
        q = q.view(B, n, hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, hkv, G * n, D)
        scores = q @ _values(s["pools"][0], s["pages"], hkv, bits).permute(0, 2, 3, 1) * D ** -0.5
        seen = torch.arange(L, device="cuda") <= limit[..., None]
        scores = scores.view(B, hkv, G, n, L).masked_fill(~seen[:, None, None], -1e30)
        v = _values(s["pools"][1], s["pages"], hkv, bits).transpose(1, 2)
        out = (_weights(scores).view(B, hkv, G * n, L) @ v).view(B, hq, n, D)
        return out.transpose(1, 2)[s["seq"], at].half()
    first = c["shared"] // PAGE
    mine = s["pages"][:, first:]
    q = s["q"].float().view(B, hkv, G, D)
    k = [_values(s["pools"][0], p, hkv, bits) for p in (s["pages"][0, :first], mine)]
    scores = torch.cat([torch.einsum("bhgd,nhd->bhgn", q, k[0]), torch.einsum("bhgd,bnhd->bhgn", q, k[1])], -1) * D ** -0.5
    seen = torch.arange(scores.shape[-1], device="cuda") < s["lens"][:, None]
    w = _weights(scores.masked_fill(~seen[:, None, None], -1e30))
    out = torch.einsum("bhgn,nhd->bhgd", w[..., :c["shared"]], _values(s["pools"][1], s["pages"][0, :first], hkv, bits))
    out = out + torch.einsum("bhgn,bnhd->bhgd", w[..., c["shared"]:], _values(s["pools"][1], mine, hkv, bits))
    return out.reshape(B, hq, D).half()


# ------------------------------------------------------------------------------------------------------------------------
# the framework's calls
# ------------------------------------------------------------------------------------------------------------------------
def _own(s):
    from qserve_b200 import backend
    c = s["case"]
    int4, size = c["bits"] == 4, c["kv_heads"] * D * c["bits"] // 8
    if c["kind"] == "append":
        q = backend.append_kv_cache(s["q"], s["k"], s["v"], s["table"], s["cu"], s["lens"], PAGE, size, D, BASE, int4, True)
        k, v = backend.read_kv_cache(s["table"], s["cu"], s["lens"], s["T"], PAGE, size, int4, True)
        return {"q": q, "k": k, "v": v}
    if c["kind"] == "read":
        k, v = backend.read_kv_cache(s["table"], s["cu"], s["lens"], s["T"], PAGE, size, int4, True)
        return {"k": k, "v": v}
    if c["kind"] == "prompt":
        return backend.paged_prompt_attention(s["q"], s["table"], s["cu"], s["lens"], s["new"], s["top"], PAGE, size, int4, True)
    return backend.shared_prefix_attention(s["q"], s["table"], s["lens"], c["shared"] // PAGE, s["top"], PAGE, size, int4, True)


def run(state):
    return _own(state) if own else _plain(state)


def work(case):
    hq, hkv, cell = case["heads"], case["kv_heads"], case["kv_heads"] * (D * case["bits"] // 8 + 4) * 2
    new, held = _sizes(case)
    T = sum(new)
    if case["kind"] == "append":  # q, k, v in; q, cells, and what they stand for out
        return {"bytes": T * ((hq + 2 * hkv) * D * 2 + hq * D * 2 + cell + 2 * hkv * D * 2), "flops": T * ((hq + hkv) * D * 3 + 2 * hkv * D * 6)}
    if case["kind"] == "read":
        return {"bytes": T * (cell + 2 * hkv * D * 2), "flops": T * 2 * hkv * D * 2}
    io = 2 * T * hq * D * 2
    if case["kind"] == "prompt":
        keys = sum(n * (m - n) + n * (n + 1) // 2 for n, m in zip(new, held))
        return {"bytes": io + sum(held) * cell, "flops": 4 * D * hq * keys}
    return {"bytes": io + (case["shared"] + sum(m - case["shared"] for m in held)) * cell, "flops": 4 * D * hq * sum(held)}


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


def _turned(x, pos):
    out = torch.empty(x.shape, dtype=F64, device="cuda")
    for i in range(D // 2):
        w = pos.to(F64) * BASE ** (-2.0 * i / D)
        c, s = torch.cos(w)[:, None], torch.sin(w)[:, None]
        lo, hi = x[..., i].to(F64), x[..., i + D // 2].to(F64)
        out[..., i], out[..., i + D // 2] = lo * c - hi * s, hi * c + lo * s
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


def _softmax_rows(q, k, v, seen):
    """q [n, D] over k, v [L, D] with seen [n, L]."""
    s = (q @ k.T) / math.sqrt(D)
    s = torch.where(seen, s, torch.full_like(s, -math.inf))
    return torch.softmax(s, 1) @ v


def exact(case, seed):
    s = prepare(case, seed)
    hq, hkv, bits = case["heads"], case["kv_heads"], case["bits"]
    new, held = _sizes(case)
    kp, vp = s["pools"]
    if case["kind"] == "append":
        return {"q": _turned(s["q"], s["pos"]), "k": _held(_turned(s["k"], s["pos"]).to(HALF), bits), "v": _held(s["v"], bits)}
    parts = {"k": [], "v": []}
    if case["kind"] == "read":
        for b, (n, m) in enumerate(zip(new, held)):
            parts["k"].append(_cells(kp, s["pages"][b], m - n, m, hkv, bits))
            parts["v"].append(_cells(vp, s["pages"][b], m - n, m, hkv, bits))
        return {name: torch.cat(x) for name, x in parts.items()}
    out, at = torch.empty(s["T"], hq, D, dtype=F64, device="cuda"), 0
    both = {}
    for b, (n, m) in enumerate(zip(new, held)):
        if case["kind"] == "shared":  # the common positions once
            if not both:
                both = {id(p): _cells(p, s["pages"][0], 0, case["shared"], hkv, bits) for p in (kp, vp)}
            k, v = (torch.cat([both[id(p)], _cells(p, s["pages"][b], case["shared"], m, hkv, bits)]) for p in (kp, vp))
        else:
            k, v = (_cells(p, s["pages"][b], 0, m, hkv, bits) for p in (kp, vp))
        t = torch.arange(m, device="cuda")
        for h in range(hq):
            for lo in range(0, n, 1024):
                hi = min(n, lo + 1024)
                seen = t[None] <= torch.arange(m - n + lo, m - n + hi, device="cuda")[:, None]
                out[at + lo:at + hi, h] = _softmax_rows(s["q"][at + lo:at + hi, h].to(F64), k[:, h * hkv // hq], v[:, h * hkv // hq], seen)
        at += n
    return out

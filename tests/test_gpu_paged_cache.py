"""Portions appended to and read from the paged cache: bits of the pages, rotations at far positions, rows that quantisation cannot hold, padded batches."""
import numpy as np
import pytest
import torch

from oracle import kv
from qserve_b200 import backend
from tests.paged_util import BASE, D, F64, H, HALF, PAGE, Cache, rotated
from tests.test_gpu_paged_attention import starts

pytestmark = pytest.mark.gpu


def rows(T, hq, hkv, dev, seed=0):
    x = torch.randn(T, hq + 2 * hkv, D, generator=torch.Generator().manual_seed(seed)).half().to(dev)
    return x.split([hq, hkv, hkv], 1)  # strided views of one product's rows


def append(c, q, k, v, new, **more):
    cu = None if new is None else starts(new, c.dev)
    return backend.append_kv_cache(q, k, v, c.table, cu, c.lengths, PAGE, c.size, D, BASE, c.bits == 4, True, **more)


def read(c, new, T):
    return backend.read_kv_cache(c.table, None if new is None else starts(new, c.dev), c.lengths, T, *c.args)


def positions(new, lens, dev):
    return torch.cat([torch.arange(m - n, m, device=dev) for n, m in zip(new, lens)])


def check_rotation(got, x, pos):
    """Sine, cosine, two products and their sum round in fp32 (2^-24 each of |a| + |b|), the result in fp16."""
    want = rotated(x, pos)
    a, b = x.to(F64).abs().chunk(2, -1)
    room = H * want.abs() + (a + b).repeat(1, 1, 2) * 4 * 2.0 ** -24 + 2.0 ** -25
    assert ((got.to(F64) - want).abs() <= room * (1 + 1e-9)).all()


def check_pages(c, which, x, new, lens):
    """The codes, scales and zeros of fp16 rows x [T, hkv, D] are those of the oracle's quantisation, bit for bit, and no other slot has changed."""
    pos = positions(new, lens, c.dev)
    seq = torch.repeat_interleave(torch.arange(len(new), device=c.dev), torch.tensor(new, device=c.dev))
    page, slot = c.pages[seq, pos // PAGE], pos % PAGE
    x = x.cpu().numpy()
    s, z = kv.kv_quant_params(x, c.bits)
    u = kv.kv_quant_codes(x, s, z, c.bits)
    assert np.array_equal(c.codes(which)[page, :, slot].cpu().numpy(), u)
    assert np.array_equal(c.meta(which)[page, 0, :, slot].cpu().numpy().view(np.uint16), s.view(np.uint16))
    assert np.array_equal(c.meta(which)[page, 1, :, slot].cpu().numpy().view(np.uint16), z.view(np.uint16))


CASES = [  # query heads, key/value heads, new tokens, positions held ahead of them
    (4, 1, [1], [0]),
    (32, 8, [1, 1, 1, 1], [0, 63, 64, 1000]),
    (8, 2, [5, 0, 130, 64], [60, 10, 1, 128]),
    (8, 8, [3, 1], [200000, 7]),
    (10, 2, [2000], [131]),
    (64, 64, [40, 33], [50, 500]),
]


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,new,ahead", CASES)
def test_append_and_read(dev, bits, hq, hkv, new, ahead):
    lens, T = [n + m for n, m in zip(new, ahead)], sum(new)
    c = Cache(lens, hkv, bits, dev, seed=T)
    before = [p.clone() for p in c.pools]
    q, k, v = rows(T, hq, hkv, dev)
    pos = positions(new, lens, dev)
    out = append(c, q, k, v, new)
    check_rotation(out, q, pos)
    # keys are quantised as the fp16 numbers that the same rotation gives queries
    turned = append(c, k.repeat(1, hq // hkv, 1), k, v, new)[:, :hkv] if hq > hkv else append(c, k, k, v, new)
    check_rotation(turned, k, pos)
    check_pages(c, 0, turned, new, lens)
    check_pages(c, 1, v, new, lens)
    ks, vs = read(c, new, T)
    for which, got in ((0, ks), (1, vs)):
        want = torch.cat([c.values(which, b, m)[m - n:] for b, (n, m) in enumerate(zip(new, lens))])
        assert ((got.to(F64) - want).abs() <= H * want.abs() * (1 if bits == 4 else 1 + 2.0 ** -10) + 2.0 ** -24 * (1 if bits == 4 else 2)).all()
        # everything else in the pool is as it was
        same = torch.ones(c.pools[which].shape[0], PAGE, dtype=torch.bool, device=dev)
        seq = torch.repeat_interleave(torch.arange(len(new), device=dev), torch.tensor(new, device=dev))
        same[c.pages[seq, pos // PAGE], pos % PAGE] = False
        now, then = (p[:, :c.cut].view(-1, hkv, PAGE, D * bits // 8).transpose(1, 2)[same] for p in (c.pools[which], before[which]))
        assert torch.equal(now, then)
        now, then = (p[:, c.cut:].view(torch.int16).view(-1, 2, hkv, PAGE).permute(0, 3, 1, 2)[same] for p in (c.pools[which], before[which]))
        assert torch.equal(now, then)


@pytest.mark.parametrize("bits", [4, 8])
def test_whole_prompts_as_the_reference_operator_appends_them(dev, bits):
    """From position 0 on, the values' pages are those of apply_bias_rope_update_kv_cache."""
    lens, hq, hkv = [100, 33, 64], 8, 2
    a, b = (Cache(lens, hkv, bits, dev, seed=1) for _ in range(2))
    q, k, v = rows(sum(lens), hq, hkv, dev)
    append(a, q, k, v, lens)
    qkv = torch.cat([q, k, v], 1).flatten(1).contiguous()
    cu = starts(lens, dev)
    offsets = backend.compute_padding_offsets(cu, 100, sum(lens))
    backend.apply_bias_rope_update_kv_cache(qkv, b.lengths, offsets, b.table, hq, hkv, 100, PAGE, b.size, D, BASE, 100000, True, bits == 4, True)
    assert torch.equal(a.pools[1], b.pools[1])


@pytest.mark.parametrize("bits", [4, 8])
def test_rows_that_quantisation_cannot_hold(dev, bits):
    """Equal values are held as they are; values too near to one another for a zero in fp16 as their middle; a row with no number or no end reads as NaN."""
    x = torch.randn(8, 1, D, generator=torch.Generator().manual_seed(3)).half().to(dev)
    x[0], x[1], x[2] = 0.0, 3.5, -0.125
    x[3] = 1000.0
    x[3, 0, 5:9] = 1000.5           # span 0.5: the zero would be -15 * 1000 / 0.5 = -30000 (INT4) or -510000 (INT8)
    x[4, 0, 7] = float("nan")
    x[5, 0, 100] = float("inf")
    x[6, 0, 1] = float("-inf")
    c = Cache([8], 1, bits, dev)
    k = torch.randn(8, 1, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
    append(c, k, k, x, [8])
    got = read(c, [8], 8)[1]
    assert bool((got[0] == 0).all()) and bool((got[1] == 3.5).all()) and bool((got[2] == -0.125).all())
    # half the span, and INT4's zero (30000 in steps of 16, each 1/30 wide)
    assert bool((got[3].float() - x[3].float()).abs().max() <= (0.25 + 0.5 if bits == 8 else 16 / 2 * 0.5 / 15 + 0.5 / 15 / 2 + 0.5))
    assert bool(torch.isnan(got[4:7]).all())
    room = (x[7].float().max() - x[7].float().min()) / (2 ** bits - 1) * 0.5 + x[7].float().abs().max() * 5 * H
    assert bool(((got[7].float() - x[7].float()).abs() <= room).all())


def test_padded_batches_positions_outside_and_results_in_place(dev):
    new = [3, 2]
    c = Cache([70, 5], 2, 4, dev, seed=6)
    q, k, v = rows(9, 8, 2, dev)
    out = torch.full((9, 8, D), 7.0, dtype=HALF, device=dev)
    append(c, q, k, v, new, out=out)
    assert bool((out[5:] == 7).all())
    check_rotation(out[:5], q[:5], positions(new, [70, 5], dev))
    after = [p.clone() for p in c.pools]
    # a length past the table, and one smaller than the portion: queries are rotated, what has no place goes nowhere
    c.lengths.copy_(torch.tensor([c.blocks * PAGE + 50, 0], dtype=torch.int32))
    append(c, q, k, v, new)
    assert all(torch.equal(a, b) for a, b in zip(c.pools, after))
    k2, v2 = read(c, new, 5)
    assert k2.shape == (5, 2, D)
    c.lengths.copy_(torch.tensor([70, 5], dtype=torch.int32))
    mine = q.clone()
    assert append(c, mine, k, v, new, out=mine).data_ptr() == mine.data_ptr()
    assert torch.equal(mine[:5], out[:5]) and torch.equal(mine[5:], q[5:])


def test_single_tokens_without_starts(dev):
    c, d = (Cache([64, 65, 300], 2, 8, dev, seed=9) for _ in range(2))
    q, k, v = rows(3, 8, 2, dev)
    a, b = append(c, q, k, v, None), append(d, q, k, v, [1, 1, 1])
    assert torch.equal(a, b) and all(torch.equal(x, y) for x, y in zip(c.pools, d.pools))
    assert all(torch.equal(x, y) for x, y in zip(read(c, None, 3), read(d, [1, 1, 1], 3)))


def test_captured_and_on_another_stream(dev):
    c = Cache([500, 640], 2, 4, dev, seed=9)
    q, k, v = rows(40, 8, 2, dev)
    new = [17, 23]
    cu = starts(new, dev)
    want = append(c, q, k, v, new), *read(c, new, 40)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = (backend.append_kv_cache(q, k, v, c.table, cu, c.lengths, PAGE, c.size, D, BASE, True, True), *backend.read_kv_cache(c.table, cu, c.lengths, 40, *c.args))
    for p in c.pools:
        p.zero_()
    with torch.cuda.stream(stream):
        graph.replay()
    stream.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))

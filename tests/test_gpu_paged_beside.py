"""The operators over portions beside the ones that the framework had: what append writes and what apply_bias_rope_update_kv_cache writes, the decode runner's step with a shared prefix and
without.  Tolerances are those that tests/test_gpu_attention.py states for the older operators (fp32 rotations that differ in the last bits: scales and zeros within one unit in the last place,
codes within one, 3 % of them; attention of single tokens within 3e-3 of the definition), and check_attention's for the newer."""
import numpy as np
import pytest
import torch

from qserve_b200 import backend
from tests.paged_util import BASE, D, F64, PAGE, Cache, attention64, check_attention
from tests.test_gpu_paged_attention import SCALE, starts
from tests.test_gpu_paged_cache import rows
from tests.util import np_of, ulp16_diff

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 4)])
def test_keys_and_queries_of_whole_prompts(dev, bits, hq, hkv):
    """From position 0 on, in one portion or in three, keys' pages and rotated queries are those of apply_bias_rope_update_kv_cache; values' bit for bit."""
    lens = [130, 33, 64]
    a, b = (Cache(lens, hkv, bits, dev, seed=1) for _ in range(2))
    q, k, v = rows(sum(lens), hq, hkv, dev)
    turned = torch.empty_like(q, memory_format=torch.contiguous_format)
    for lo, hi in ((0, 1), (1, 30), (30, 130)):  # every sequence's positions from lo to hi
        new = [max(0, min(n, hi) - lo) for n in lens]
        pick = torch.cat([torch.arange(sum(lens[:i]) + lo, sum(lens[:i]) + lo + n) for i, n in enumerate(new)]).to(dev)
        a.lengths.copy_(torch.tensor([min(n, hi) for n in lens], dtype=torch.int32))
        turned[pick] = backend.append_kv_cache(q[pick], k[pick], v[pick], a.table, starts(new, dev), a.lengths, PAGE, a.size, D, BASE, bits == 4, True)
    qkv = torch.cat([q, k, v], 1).flatten(1).contiguous()
    offsets = backend.compute_padding_offsets(starts(lens, dev), max(lens), sum(lens))
    backend.apply_bias_rope_update_kv_cache(qkv, b.lengths, offsets, b.table, hq, hkv, max(lens), PAGE, b.size, D, BASE, 100000, True, bits == 4, True)
    assert torch.equal(a.pools[1], b.pools[1])
    other = qkv.view(sum(lens), hq + 2 * hkv, D)[:, :hq]
    assert (turned.float() - other.float()).abs().max() <= 2.0 ** -9 * q.float().abs().max()  # rounded to fp16 on either side of a number
    for i in range(len(lens)):
        t = torch.arange(lens[i], device=dev)
        page, slot = a.pages[i, t // PAGE], t % PAGE
        for field in (0, 1):
            assert ulp16_diff(*(np_of(c.meta(0)[page, field, :, slot]) for c in (a, b))).max() <= 1
        off = np.abs(np.subtract(*(np_of(c.codes(0)[page, :, slot]).astype(np.int32) for c in (a, b))))
        assert off.max() <= 1 and (off > 0).mean() <= 0.03


def turned(x, pos, base):
    """rotated() with another base."""
    angle = pos.to(F64)[:, None] * float(base) ** (-2.0 * torch.arange(D // 2, device=x.device, dtype=F64) / D)
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x.to(F64).chunk(2, -1)
    return torch.cat([c * a - s * b, c * b + s * a], -1)


@pytest.mark.parametrize("precision", ["w4a8kv4", "w8a8kv8"])
@pytest.mark.parametrize("batch,shared", [(6, 256), (2, 128)])
def test_the_runners_step_with_and_without_the_operator_that_shares(dev, precision, batch, shared):
    """Two runners over the same pages, the same rows for both: their attention against the definition over what the pages hold behind each.  single_query_attention takes the new
    token's key and value as they come, the operators over the paged cache as the pages hold them."""
    from qserve_b200.decode import DecodeRunner
    with_it, without = (DecodeRunner("tiny", precision, batch=batch, ctx=300, device=dev, shared_prefix=n) for n in (shared, 0))
    without.block_tables = with_it.block_tables
    Hq, Hkv, last = with_it.Hq, with_it.Hkv, torch.full((batch,), 300, device=dev)
    x = torch.randn(batch, Hq + 2 * Hkv, D, generator=torch.Generator().manual_seed(3)).half().to(dev)
    q, k = (turned(t, last, with_it.cfg.rope_theta).half() for t in x[:, :Hq + Hkv].split([Hq, Hkv], 1))
    whole = torch.arange(batch + 1, dtype=torch.int32, device=dev) * 301
    for r in (with_it, without):
        r.qkv_buf.copy_(x.flatten(1))
        out = r._attention(0).view(batch, Hq, D)
        held = backend.read_kv_cache(r.block_tables[0], whole, r.context_lens, batch * 301, 64, r.size_per_token, r.kv_bits == 4, True)
        ks, vs = (t.view(batch, 301, Hkv, D).to(F64) for t in held)
        if r is without:
            ks[:, 300], vs[:, 300] = k.to(F64), x[:, Hq + Hkv:].to(F64)
        want = [attention64(q[b:b + 1], ks[b], vs[b], last[:1], SCALE) for b in range(batch)]
        if r is with_it:
            for b in range(batch):
                check_attention(out[b:b + 1], want[b], SCALE)
        else:  # of the largest number of the whole result, as stated there
            exact = torch.cat([w[0] for w in want])
            assert float((out.to(F64) - exact).abs().max()) <= 3e-3 * max(1.0, float(exact.abs().max()))

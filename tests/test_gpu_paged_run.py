"""The operators over the paged cache as they are used together: a prompt in portions, sequences that continue behind its pages, decode steps of a batch that shares
them, and the decode runner with a shared prefix."""
import pytest
import torch

from qserve_b200 import backend
from tests.paged_util import BASE, D, F64, H, PAGE, Cache, attention64, check_attention
from tests.test_gpu_paged_attention import SCALE, starts
from tests.test_gpu_paged_cache import check_rotation, rows

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv", [(8, 2), (4, 4)])
def test_a_prompt_in_portions_and_a_batch_behind_it(dev, bits, hq, hkv):
    prefix, B, steps = 5 * PAGE, 3, 70  # the steps cross a page's end
    c = Cache([0] * B, hkv, bits, dev, shared=5, seed=1, extra_blocks=2)
    for p in c.pools:
        p.fill_(255)  # every scale and zero that is not written is no number
    cache = (PAGE, c.size, bits == 4, True)
    one = c.table[:1].contiguous()
    length = torch.zeros(1, dtype=torch.int32, device=dev)
    x = rows(prefix, hq, hkv, dev, seed=2)
    at = 0
    for n in (1, 63, 100, 156):  # portions of the prompt into the first sequence's pages
        q, k, v = (t[at:at + n] for t in x)
        at += n
        length.fill_(at)
        cu = starts([n], dev)
        turned = backend.append_kv_cache(q, k, v, one, cu, length, PAGE, c.size, D, BASE, bits == 4, True)
        check_rotation(turned, q, torch.arange(at - n, at, device=dev))
        out = backend.paged_prompt_attention(turned, one, cu, length, n, at, *cache)
        check_attention(out, attention64(turned, c.values(0, 0, at), c.values(1, 0, at), torch.arange(at - n, at, device=dev), SCALE), SCALE)
    # questions of different lengths behind it, one of them a single token
    new = [1, 30, 45]
    c.lengths.copy_(torch.tensor([prefix + n for n in new], dtype=torch.int32))
    q, k, v = rows(sum(new), hq, hkv, dev, seed=3)
    cu = starts(new, dev)
    turned = backend.append_kv_cache(q, k, v, c.table, cu, c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
    out = backend.paged_prompt_attention(turned, c.table, cu, c.lengths, 45, prefix + 45, *cache)
    at = 0
    for b, n in enumerate(new):
        m = prefix + n
        check_attention(out[at:at + n], attention64(turned[at:at + n], c.values(0, b, m), c.values(1, b, m), torch.arange(prefix, m, device=dev), SCALE), SCALE)
        at += n
    # decode steps, one captured and replayed with its lengths on the device
    x = rows(B, hq, hkv, dev, seed=4)
    buffers = [t.clone() for t in x]

    def step():
        c.lengths.add_(1)
        turned = backend.append_kv_cache(*buffers, c.table, None, c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
        return turned, backend.shared_prefix_attention(turned, c.table, c.lengths, 5, prefix + 45 + steps, *cache)
    step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        turned, out = step()
    for i in range(1, steps):
        for t, s in zip(buffers, rows(B, hq, hkv, dev, seed=4 + i)):
            t.copy_(s)
        graph.replay()
        if i in (1, 30, steps - 1):
            for b, n in enumerate(new):
                m = prefix + n + i + 1
                assert int(c.lengths[b]) == m
                check_rotation(turned[b:b + 1], buffers[0][b:b + 1], torch.tensor([m - 1], device=dev))
                check_attention(out[b:b + 1], attention64(turned[b:b + 1], c.values(0, b, m), c.values(1, b, m), torch.tensor([m - 1], device=dev), SCALE), SCALE)
    # what the pages of the last sequence hold, taken out whole: rounded to fp16 (INT8: scale times difference, another rounding in fp32)
    k, v = backend.read_kv_cache(c.table, torch.tensor([0, 0, 0, m], dtype=torch.int32, device=dev), c.lengths, m, *cache)
    for which, got in ((0, k), (1, v)):
        want = c.values(which, B - 1, m)
        assert ((got.to(F64) - want).abs() <= H * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -23).all()


@pytest.mark.parametrize("precision", ["w4a8kv4", "w8a8kv8"])
def test_decode_runner_with_a_shared_prefix(dev, precision):
    """The runner's attention behind a shared prefix is the definition's over its own pages, eager and captured; the same step without the operator that shares."""
    from qserve_b200.decode import DecodeRunner
    r = DecodeRunner("tiny", precision, batch=6, ctx=300, device=dev, shared_prefix=256)
    assert torch.equal(r.block_tables[:, :1, :, :4].expand(-1, 6, -1, -1), r.block_tables[:, :, :, :4])
    r.forward(r.tokens_in)
    r.qkv_buf.normal_()
    out = r._attention(0).view(6, r.Hq, D)
    whole = torch.arange(7, dtype=torch.int32, device=dev) * 301
    ks, vs = backend.read_kv_cache(r.block_tables[0], whole, r.context_lens, 6 * 301, 64, r.size_per_token, r.kv_bits == 4, True)
    q = r.qkv_buf[:, :r.q_size].view(6, r.Hq, D)
    turned = backend.append_kv_cache(q, r.qkv_buf[:, r.q_size:r.q_size + r.kv_size].view(6, r.Hkv, D), r.qkv_buf[:, r.q_size + r.kv_size:].view(6, r.Hkv, D), r.block_tables[0], None,
                                     r.context_lens, 64, r.size_per_token, D, r.cfg.rope_theta, r.kv_bits == 4, True)
    for b in range(6):
        kb, vb = (t.view(6, 301, r.Hkv, D)[b].to(F64) for t in (ks, vs))
        check_attention(out[b:b + 1], attention64(turned[b:b + 1], kb, vb, torch.tensor([300], device=dev), SCALE), SCALE)
    want = r.forward(r.tokens_in)
    r.capture()
    r.step()
    assert torch.equal(r.tokens_out, want)
    with pytest.raises(AssertionError):
        DecodeRunner("tiny", precision, batch=2, ctx=300, device=dev, shared_prefix=100)

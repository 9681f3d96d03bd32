"""The operators over the paged cache where their numbers and tables end: what the pages stand for at the ends of fp16, results of one rounding, rows without a position, tables
whose shared columns count in one row alone.  H = 2^-11: a rounding to fp16 is off by at most H relative."""
import pytest
import torch

from qserve_b200 import backend
from tests.paged_util import BASE, D, F64, H, HALF, PAGE, Cache, attention64, check_attention
from tests.test_gpu_paged_attention import SCALE, prompt64, queries, run_prompt, shared64, starts

pytestmark = pytest.mark.gpu


def fill(c, which, b, codes, scale, zero):
    """Positions of sequence b: codes [n, hkv, D] (whole numbers), scale and zero [n, hkv]."""
    n = codes.shape[0]
    t = torch.arange(n, device=c.dev)
    page, slot = c.pages[b][t // PAGE], t % PAGE
    u = codes.to(torch.uint8)
    if c.bits == 4:
        u = u[..., 0::2] | (u[..., 1::2] << 4)
    c.pools[which][:, :c.cut].view(-1, c.hkv, PAGE, D * c.bits // 8)[page, :, slot] = u.to(c.dev)
    c.meta(which)[page, 0, :, slot] = scale.to(c.dev).half()
    c.meta(which)[page, 1, :, slot] = zero.to(c.dev).half()


def random_codes(n, hkv, bits, seed):
    return torch.randint(0, 2 ** bits, (n, hkv, D), generator=torch.Generator().manual_seed(seed))


# ---- lengths at the ends of their type, where a prefix is read by the tile kernel and the rest by the tail kernel ----
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,batch", [(8, 2, 9), (32, 8, 40), (32, 8, 300)])
def test_lengths_at_the_ends_of_their_type_behind_a_prefix(dev, bits, hq, hkv, batch):
    c = Cache([4 * PAGE] * batch, hkv, bits, dev, shared=2, seed=2)
    q = queries(batch, hq, dev)
    want = shared64(c, q, c.lens)
    said = torch.full((batch,), 4 * PAGE)
    said[:9] = torch.tensor([2 ** 31 - 1, -2 ** 31, 4 * PAGE, -1, 0, 100000, -2 ** 31 + 100, 2 ** 30, -64])
    c.lengths.copy_(said.int())
    out = backend.shared_prefix_attention(q, c.table, c.lengths, 2, 4 * PAGE, *c.args)
    assert bool((out[said <= 0] == 0).all())
    check_attention(out[said > 0], [x[said > 0] for x in want], SCALE)


# ---- rows that a cluster's half warps share out unevenly ----
@pytest.mark.parametrize("bits", [4, 8])
def test_any_number_of_rows_in_a_cluster(dev, bits):
    for n in [*range(1, 20), 31, 33, 47, 64, 65, 100, 127, 128]:
        c = Cache([n + 600], 1, bits, dev, seed=n)
        q = queries(n, 1, dev)
        check_attention(run_prompt(c, q, [n]), prompt64(c, q, [n], c.lens), SCALE)

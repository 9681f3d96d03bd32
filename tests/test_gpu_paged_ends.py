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


# ---- rows whose codes could stand for more than fp16 holds, and do not ----
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,new,ahead", [(8, 2, [20, 3], [100, 700]), (32, 8, [150], [60]), (8, 2, [6], [2600])])
def test_rows_of_one_value(dev, bits, hq, hkv, new, ahead):
    """Values that append holds as 1 x scale or 0 - 1 x scale, up to the end of fp16; and rows of few codes: the numbers that the pages stand for."""
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=14)
    for b, n in enumerate(lens):
        g = torch.Generator().manual_seed(b)
        size = torch.exp2(torch.rand(n, hkv, generator=g) * 16).clamp(max=64992)
        some = torch.rand(n, hkv, generator=g) < 0.5
        sign = (torch.rand(n, hkv, generator=g) < 0.5)
        fill(c, 1, b, (~sign & some).long()[..., None].expand(-1, -1, D), torch.where(some, size, 0.01), torch.where(some, sign.half(), 5.0))
        # codes 0 .. 3 around a zero of 1.5: +- 1.5 scales, where the largest code would stand for 13.5 of them, or 253.5
        few = torch.rand(n, hkv, generator=g) < 0.2
        u = torch.randint(0, 4, (n, hkv, D), generator=g)
        page, slot = c.pages[b][torch.arange(n, device=dev) // PAGE], torch.arange(n, device=dev) % PAGE
        old = c.codes(1)[page, :, slot].cpu()
        s, z = (c.meta(1)[page, i, :, slot].cpu().float() for i in (0, 1))
        fill(c, 1, b, torch.where(few[..., None], u, old.long()), torch.where(few, (size * 0.6).clamp(max=43000), s), torch.where(few, 1.5, z))
    q = queries(sum(new), hq, dev)
    check_attention(run_prompt(c, q, new), prompt64(c, q, new, lens), SCALE)


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("value", [300.0, -4400.0, 64992.0, -64992.0])
def test_appended_rows_of_one_value_are_attended_to(dev, bits, value):
    """Appended values that are all equal come out of both kernels of attention as they went in (a weighted mean of equal numbers: the weights' rounding, 2 H)."""
    n, hkv = 70, 2
    c = Cache([n], hkv, bits, dev, seed=3)
    k = torch.randn(n, hkv, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
    v = torch.full_like(k, value)
    backend.append_kv_cache(k, k, v, c.table, starts([n], dev), c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
    q = queries(n, 8, dev)
    for out in (backend.paged_prompt_attention(q, c.table, starts([n], dev), c.lengths, n, n, *c.args), backend.shared_prefix_attention(q[:1], c.table, c.lengths, 0, n, *c.args)):
        assert bool(((out.float() - value).abs() <= 2 * H * abs(value)).all()), float((out.float() / value - 1).abs().max())


# ---- one rounding of a value ----
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("shared", [0, 1])
def test_a_value_alone_is_rounded_once(dev, bits, shared):
    """Sequences of a single position: its weight is 1, the result what its codes stand for, rounded once.  INT8 adds the rounding of scale times the zero's part behind the point, at
    most half a scale.  Zeros of every size from fractions to 1000.  fp32 rounds scores (2^-18 of a weight) and products of scale with code and zero (2^-20)."""
    batch, hq, hkv = 40, 4, 1
    c = Cache([1] * batch, hkv, bits, dev, shared=0, seed=2)
    g = torch.Generator().manual_seed(7)
    for b in range(batch):
        z = (torch.rand(1, hkv, generator=g) * 2 - 1) * (15.0 if bits == 4 else [4.0, 200.0, 1000.0][b % 3])
        fill(c, 1, b, random_codes(1, hkv, bits, b), 0.01 + torch.rand(1, hkv, generator=g), z)
    q = queries(batch, hq, dev)
    if shared:
        out = backend.shared_prefix_attention(q, c.table, c.lengths, 0, 1, *c.args)
    else:
        out = backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 1, *c.args)
    for b in range(batch):
        want = c.values(1, b, 1)[0].repeat_interleave(hq // hkv, 0)
        s, z = (float(c.meta(1)[c.pages[b, 0], i, 0, 0]) for i in (0, 1))
        room = H * want.abs() * (1 + 2.0 ** -7) + (0 if bits == 4 else H * s / 2 * (1 + H)) + s * (abs(z) + 2 ** bits) * 2.0 ** -20
        off = (out[b].to(F64) - want).abs()
        assert (off <= room).all(), (b, float((off / room).max()))


# ---- rows at the ends of fp16 ----
@pytest.mark.parametrize("bits", [4, 8])
def test_appended_rows_at_the_ends_of_fp16(dev, bits):
    """Finite rows read back as finite numbers, off by half a code's step (a whole one at the ends), the rounding of scale and zero, and one of the result; attention takes them as they are.
    The scale is rounded down where the rounded one reaches past fp16 (2 H of it for each code), the zero moved by one of its steps (2 H of it, each a scale)."""
    top = 2 ** bits - 1
    g = torch.Generator().manual_seed(1)
    ends = [(-65504, 65504), (-65504, 65472), (-65472, 65504), (-65504, 0), (0, 65504), (-65504, 60000), (-60000, 65504), (64992, 65504), (-65504, -64992), (65472, 65504), (-65504, -65472),
            (-65504, -32768), (32768, 65504), (-65440, 65440), (-65504, 4096), (-65408, 65376)]
    n = len(ends)
    x = torch.empty(n, 1, D)
    for i, (lo, hi) in enumerate(ends):
        x[i] = lo + (hi - lo) * torch.rand(D, generator=g)
        x[i, 0, 3], x[i, 0, 90] = lo, hi
    x = x.half().to(dev)
    k = torch.randn(n, 1, D, generator=g).half().to(dev)
    c = Cache([n], 1, bits, dev)
    backend.append_kv_cache(k, k, x, c.table, starts([n], dev), c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
    got = backend.read_kv_cache(c.table, starts([n], dev), c.lengths, n, *c.args)[1]
    assert bool(torch.isfinite(got).all())
    span = (x.amax(-1) - x.amin(-1).float())[..., None]
    room = span / top + (span + 3 * x.float().abs().amax(-1, keepdim=True)) * 2 * H + 32
    assert bool(((got.float() - x.float()).abs() <= room).all())
    assert bool(torch.isfinite(c.values(1, 0, n)).all()) and float(c.values(1, 0, n).abs().max()) < 65520
    q = queries(n, 8, dev)
    want = prompt64(c, q, [n], [n])
    check_attention(run_prompt(c, q, [n]), want, SCALE)
    check_attention(backend.shared_prefix_attention(q[-1:], c.table, c.lengths, 0, n, *c.args), [w[-1:] for w in want], SCALE)


@pytest.mark.parametrize("bits", [4, 8])
def test_appended_rows_of_any_ends_are_finite(dev, bits):
    """Rows from one number to another, one of them above 65000 in size: whatever their codes, the pages stand for finite numbers, as near as a code's step, the scale rounded down
    (2 H of its codes) and the zero's step (2 H of the zero) allow."""
    top, n = 2 ** bits - 1, 6000
    g = torch.Generator().manual_seed(9)
    ends = torch.randint(0, 0x7c00, (n, 2), generator=g).to(torch.int16)
    ends[:, 0] = torch.randint(0x7bf0, 0x7c00, (n,), generator=g).to(torch.int16)
    ends[::2, 1] = torch.randint(0x7800, 0x7c00, (n // 2,), generator=g).to(torch.int16)
    ends = ends.view(HALF).float() * (torch.randint(0, 2, (n, 2), generator=g) * 2 - 1)
    lo, hi = ends.amin(1, keepdim=True), ends.amax(1, keepdim=True)
    x = lo + (hi - lo) * torch.rand(n, D, generator=g)
    x[:, :1], x[:, 70:71] = lo, hi
    x = x.half().to(dev)[:, None]
    k = torch.randn(n, 1, D, generator=g).half().to(dev)
    c = Cache([n], 1, bits, dev)
    backend.append_kv_cache(k, k, x, c.table, starts([n], dev), c.lengths, PAGE, c.size, D, BASE, bits == 4, True)
    got = backend.read_kv_cache(c.table, starts([n], dev), c.lengths, n, *c.args)[1]
    assert bool(torch.isfinite(got).all())
    least, most = x.amin(-1).float(), x.amax(-1).float()
    room = (most - least) / top + (most - least + 3 * torch.maximum(most, -least)) * 2 * H + 32
    assert bool(((got.float() - x.float()).abs() <= room[..., None]).all())
    scale, zero = (c.meta(1)[c.pages[0, torch.arange(n, device=dev) // PAGE], i, 0, torch.arange(n, device=dev) % PAGE].to(F64) for i in (0, 1))
    u = c.codes(1)[c.pages[0, torch.arange(n, device=dev) // PAGE], 0, torch.arange(n, device=dev) % PAGE]
    for u in (u.amin(-1), u.amax(-1)):  # (of a row of one value: 1 x scale, whose 15 or 255 fold is nothing that it stands for)
        stands = u * scale + (-scale * zero).half().to(F64) if bits == 4 else scale * (u - zero)
        assert float(stands.abs().max()) < 65520


# ---- one rounding of a result ----
def equal_weights(c, n):
    """All keys of a head alike, so that all weights are; values that are eighths from -1 to 7 / 8 (INT8: from -16), so that values and sums are exact, and
    weights up to 2^-18 (a score's last bit, up to 2^-18, in its exponent)."""
    for b in range(len(c.lens)):
        m = c.lens[b]
        fill(c, 0, b, random_codes(1, c.hkv, c.bits, 5).expand(m, -1, -1), torch.full((m, c.hkv), 0.125), torch.full((m, c.hkv), 8.0))
        fill(c, 1, b, random_codes(m, c.hkv, c.bits, 6), torch.full((m, c.hkv), 0.125), torch.full((m, c.hkv), 8.0 if c.bits == 4 else 128.0))


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,new,ahead", [(8, 2, [17], [500]), (32, 8, [3], [5000]), (8, 2, [24], [20000]), (8, 2, [300], [2000]), (32, 8, [1300], [500]), (32, 8, [20], [64])])
def test_the_parts_of_a_split_row_are_not_rounded(dev, bits, hq, hkv, new, ahead):
    """However a row's keys are split (cluster, join kernel, a last round): one rounding."""
    lens = [n + m for n, m in zip(new, ahead)]
    c = Cache(lens, hkv, bits, dev, seed=1)
    equal_weights(c, lens)
    q = queries(sum(new), hq, dev)
    want = prompt64(c, q, new, lens)[0]
    out = run_prompt(c, q, new)
    off, room = (out.to(F64) - want).abs(), H * want.abs() * (1 + 2.0 ** -7) + 2.0 ** -20
    assert (off <= room).all(), float((off / room).max())


@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,shared,lens", [(8, 2, 33, [2200, 9000, 2112]), (32, 8, 30, [2000] * 40), (32, 8, 20, [1400] * 300), (16, 1, 300, [19300, 19201])])
def test_the_parts_of_a_shared_row_are_not_rounded(dev, bits, hq, hkv, shared, lens):
    c = Cache(lens, hkv, bits, dev, shared=shared, seed=1)
    equal_weights(c, lens)
    q = queries(len(lens), hq, dev)
    out = backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args)
    want = shared64(c, q, lens)[0]
    off, room = (out.to(F64) - want).abs(), H * want.abs() * (1 + 2.0 ** -7) + 2.0 ** -20
    assert (off <= room).all(), float((off / room).max())


# ---- shared columns of the table ----
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("hq,hkv,shared,lens", [(8, 2, 2, [200, 150, 100]), (8, 2, 16, [1300]), (8, 2, 6, [500, 384, 100, 7]), (32, 8, 3, [250] * 40)])
def test_shared_pages_are_those_of_the_first_row(dev, bits, hq, hkv, shared, lens):
    """The other rows hold other pages (the last sequence's own, NaN where it ends) in the shared columns: nothing reads them, however few sequences there are."""
    c = Cache(lens, hkv, bits, dev, shared=shared, seed=sum(lens), extra_blocks=1)
    q = queries(len(lens), hq, dev)
    want = shared64(c, q, lens)
    c.table[1:, :, :shared] = c.table[-1:, :, -1:]
    check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, shared, max(lens), *c.args), want, SCALE)


# ---- rows without a position ----
@pytest.mark.parametrize("bits", [4, 8])
def test_rows_without_a_position_read_as_zeros(dev, bits):
    """A length smaller than the portion, none, one past the table: zeros where there is no position, whatever lay in the memory of the result."""
    c = Cache([70, 64, 128, 40], 2, bits, dev, seed=6)
    new, T = [20, 3, 10, 2], 35
    c.lengths.copy_(torch.tensor([12, 0, 2 * PAGE + 4, 40], dtype=torch.int32))
    for _ in range(3):
        old = torch.full((2, T, 2, D), 7.0, dtype=HALF, device=dev)
        del old
        k, v = backend.read_kv_cache(c.table, starts(new, dev), c.lengths, T, *c.args)
        for which, got in ((0, k), (1, v)):
            none = torch.zeros(T, dtype=torch.bool)
            none[:8] = none[20:23] = none[29:33] = True
            assert bool((got[none] == 0).all())
            want = torch.cat([c.values(which, 0, 12), c.values(which, 2, 128)[122:], c.values(which, 3, 40)[38:]])
            assert ((got[~none].to(F64) - want).abs() <= H * want.abs() * (1 + 2.0 ** -10) + 2.0 ** -23).all()


# ---- results at the ends of fp16 ----
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("value", [65504.0, -65504.0])
@pytest.mark.parametrize("n", [40, 700, 5000])
def test_a_mean_of_the_largest_values_is_one(dev, bits, value, n):
    """All values +- 65504: rounded weights over their unrounded sum may be more than 1 by H / 2 and more, the result is still no infinity.  One key a page scores higher than the others, which
    all have the same weight, so that roundings add up."""
    hkv, new = 2, min(n, 30)
    c = Cache([n], hkv, bits, dev, seed=3)
    u = random_codes(1, hkv, bits, 5).expand(n, -1, -1).clone()
    u[::PAGE] = random_codes(1, hkv, bits, 6)
    fill(c, 0, 0, u, torch.full((n, hkv), 0.2 / 2 ** (bits - 4)), torch.full((n, hkv), 2.0 ** (bits - 1)))
    fill(c, 1, 0, torch.full((n, hkv, D), int(value > 0)), torch.full((n, hkv), abs(value)), torch.full((n, hkv), float(value < 0)))
    q = queries(new, 32, dev)
    one = c.table.expand(new, -1, -1).contiguous()
    lens = torch.full((new,), n, dtype=torch.int32, device=dev)
    for out in (run_prompt(c, q, [new]), backend.shared_prefix_attention(q, one, lens, 0, n, *c.args), backend.shared_prefix_attention(q, one, lens, n // PAGE, n, *c.args)):
        assert bool(((out.float() - value).abs() <= 2 * H * abs(value)).all()), float((out.float() / value - 1).abs().max())


# ---- the decode runner ----
def kernels_of(r):
    """Kernel nodes of the runner's step, captured."""
    rt = pytest.importorskip("cuda.bindings.runtime")
    r.forward(r.tokens_in)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph(keep_graph=True)
    with torch.cuda.graph(graph):
        r.tokens_out.copy_(r.forward(r.tokens_in))
    raw = rt.cudaGraph_t(graph.raw_cuda_graph())
    err, _, n = rt.cudaGraphGetNodes(raw)
    assert int(err) == 0
    err, nodes, n = rt.cudaGraphGetNodes(raw, n)
    assert int(err) == 0
    types = [rt.cudaGraphNodeGetType(x)[1] for x in nodes[:n]]
    return sum(t == rt.cudaGraphNodeType.cudaGraphNodeTypeKernel for t in types)


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("batch,shared", [(6, 256), (2, 128), (1, 256)])
def test_the_runner_counts_its_launches(dev, fused, batch, shared):
    """A shared prefix adds as many kernels to the captured step as the runner says, with the shared pages in a kernel of their own or not."""
    from qserve_b200.decode import DecodeRunner
    a, b = (DecodeRunner("tiny", "w4a8kv4", batch=batch, ctx=300, device=dev, fused=fused, shared_prefix=n) for n in (0, shared))
    more = kernels_of(b) - kernels_of(a)
    assert more > 0 and b.launches_per_step - a.launches_per_step == more


# ---- what read_kv_cache returns ----
def test_read_keys_and_values_are_tensors_of_their_own(dev):
    """Growing one in place leaves the other alone, and one that is kept does not keep the other."""
    c = Cache([64], 2, 4, dev)
    k, v = backend.read_kv_cache(c.table, starts([64], dev), c.lengths, 64, *c.args)
    assert k.untyped_storage().data_ptr() != v.untyped_storage().data_ptr()
    assert k.untyped_storage().nbytes() == v.untyped_storage().nbytes() == 64 * 2 * D * 2
    keep = v.clone()
    k.resize_(128, 2, D).fill_(7.0)
    assert torch.equal(v, keep)


# ---- another device than the current one ----
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="one GPU")
def test_tensors_on_another_device_than_the_current_one(dev):
    """How the keys are cut goes by the tensors' device, work space and launch alike."""
    for bits in (4, 8):
        c = Cache([3000, 2900], 2, bits, torch.device("cuda:1"), shared=30, seed=1)
        q = queries(2, 8, c.dev)
        want = shared64(c, q, c.lens)
        with torch.cuda.device(0):
            check_attention(backend.shared_prefix_attention(q, c.table, c.lengths, 30, 3000, *c.args), want, SCALE)
            check_attention(backend.paged_prompt_attention(q, c.table, None, c.lengths, 1, 3000, *c.args), want, SCALE)


# ---- rows whose largest number lies about fp16's end ----
@pytest.mark.parametrize("bits", [4, 8])
@pytest.mark.parametrize("which", [0, 1])
def test_rows_about_the_end_of_fp16_reach_no_row_that_does_not_see_them(dev, bits, which):
    """Two positions a sequence, the second's largest number from 65400 to 65650 in size: an infinity in its operand would make the first row, whose weight for it is 0, no number.  What the
    second row makes of values: half of the first value and the second's share, each as exact as two roundings (of value and result) and the 0.3 % that a row past the end may be taken smaller."""
    batch, hkv, top = 3000, 1, 2 ** bits - 1
    c = Cache([2] * batch, hkv, bits, dev, seed=5)
    g = torch.Generator().manual_seed(11)
    far = 65400 + 250 * torch.rand(batch, generator=g)  # of the last code, or of the first
    kind = torch.arange(batch) % 3
    last = torch.where(kind == 2, torch.randint(1, 4, (batch,), generator=g), top).float()  # the largest code that the row has
    z = torch.where(kind == 0, (torch.rand(batch, generator=g) - 0.9) * 60, torch.rand(batch, generator=g) * top).half().float()
    z = torch.where(kind == 2, torch.rand(batch, generator=g).half().float(), z)
    s = (far / torch.maximum((last - z).abs(), z.abs())).half()
    u = (torch.rand(batch, D, generator=g) * (last[:, None] + 1)).floor().clamp(max=255)
    u[:, 0], u[:, 1] = 0, last
    page = c.pages[:, 0]
    if bits == 4:
        packed = u[:, 0::2].to(torch.uint8) | (u[:, 1::2].to(torch.uint8) << 4)
    else:
        packed = u.to(torch.uint8)
    c.pools[which][:, :c.cut].view(-1, hkv, PAGE, D * bits // 8)[page, 0, 1] = packed.to(dev)
    c.meta(which)[page, 0, 0, 1] = s.to(dev)
    c.meta(which)[page, 1, 0, 1] = z.half().to(dev)
    q = queries(2 * batch, 4, dev) * (0 if which == 0 else 1)  # (no scores: keys of 65504 would outweigh everything)
    out = run_prompt(c, q, [2] * batch).view(batch, 2, 4, D)
    for b in range(0, batch, 7):
        v = c.values(1, b, 2)
        assert ((out[b, 0].to(F64) - v[0]).abs() <= H * 2 * v[0].abs() * (1 + H) + H * 2).all(), b
    assert bool(torch.isfinite(out[:, 0]).all())
    some = torch.isfinite((s.float() * z).half()) if bits == 4 else torch.isfinite(s)  # (a scale, or in INT4 its product with the zero, that is no finite number makes a row NaN)
    assert bool(torch.isfinite(out[some, 1]).all())
    if which == 0:
        for b in some.nonzero()[::7, 0].tolist():  # equal weights
            v = c.values(1, b, 2)
            assert ((out[b, 1].to(F64) - v.mean(0)).abs() <= H * 2 * v.abs().mean(0) + H * 2).all(), b

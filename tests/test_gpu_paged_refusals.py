"""What the Python mirror of the operators over portions in the paged cache refuses: layouts, types, sizes and devices of its tensors.  Nothing is launched."""
import pytest
import torch

from qserve_b200 import backend
from tests.paged_util import Cache
from tests.test_gpu_paged_attention import queries, starts

pytestmark = pytest.mark.gpu


def test_refusals(dev):
    c = Cache([70, 80], 2, 4, dev)
    q, k = queries(5, 8, dev), queries(5, 2, dev)
    cu = starts([2, 3], dev)
    good = dict(q=q, k=k, v=k, kv=c.table, cu=cu, lens=c.lengths, out=None)

    def append(**x):
        a = {**good, **x}
        return backend.append_kv_cache(a["q"], a["k"], a["v"], a["kv"], a["cu"], a["lens"], 64, c.size, 128, 1e4, True, True, a["out"])

    def prompt(**x):
        a = {**good, **x}
        return backend.paged_prompt_attention(a["q"], a["kv"], a["cu"], a["lens"], 3, 80, *c.args, out=a["out"])

    def shared(**x):
        a = {**good, "q": q[:2], **x}
        return backend.shared_prefix_attention(a["q"], a["kv"], a["lens"], 0, 80, *c.args, out=a["out"])

    def read(**x):
        a = {**good, **x}
        return backend.read_kv_cache(a["kv"], a["cu"], a["lens"], 5, *c.args)

    tables = [dict(kv=c.table.int()), dict(kv=c.table[:, 0]), dict(kv=c.table[:, :1]), dict(kv=c.table.expand(2, 2, c.table.shape[2]).transpose(0, 1)[:, :, ::2]),
              dict(lens=c.lengths.long()), dict(lens=c.lengths[:1]), dict(lens=c.lengths.cpu()), dict(kv=c.table.cpu())]
    starts_ = [dict(cu=cu[:2]), dict(cu=cu.long()), dict(cu=cu.cpu()), dict(cu=torch.zeros(6, dtype=torch.int32, device=dev)[::2])]
    rows = [dict(q=q.float()), dict(q=q[0]), dict(q=q[..., :64]), dict(q=q.transpose(1, 2).contiguous().transpose(1, 2)), dict(q=q[:, ::2]), dict(out=q[:, :4]), dict(out=q.float()), dict(out=q[:1]),
            dict(out=q.cpu())]
    for f, changes in ((append, tables + starts_ + rows + [dict(k=k[:4]), dict(v=q), dict(k=k.cpu()), dict(v=k.bfloat16())]), (prompt, tables + starts_ + rows), (shared, tables + rows),
                       (read, tables + starts_)):
        for x in changes:
            if f is shared and "q" in x and x["q"].dim() == 3:
                x = dict(q=x["q"][:2])
            with pytest.raises((RuntimeError, TypeError)):
                f(**x)
    shifted = torch.zeros(5 * 8 * 128 + 4, dtype=torch.half, device=dev)[4:].view(5, 8, 128)  # on an 8-byte boundary
    for f in (append, prompt):
        with pytest.raises(RuntimeError, match="16-byte"):
            f(q=shifted)
        with pytest.raises(RuntimeError, match="16-byte"):
            f(out=shifted)
    with pytest.raises(RuntimeError, match="one row per sequence"):
        shared(q=q)
    with pytest.raises(RuntimeError):
        backend.shared_prefix_attention(q[:2], c.table, c.lengths, c.blocks + 1, 80, *c.args)
    with pytest.raises(RuntimeError):
        backend.read_kv_cache(c.table, cu, c.lengths, -1, *c.args)

"""Refusals of the operators over portions in the paged cache, ahead of any call of CUDA: through the C ABI with made-up addresses, and through the Python mirror with
tensors that are not on a GPU.  The work space of a cut."""
import pytest
import torch

from qserve_b200 import backend
from qserve_b200._lib import lib

A = 1 << 20  # an address that nothing reads


def append(**c):
    a = dict(q=A, k=A, v=A, qs=512, ks=128, vs=128, out=A, os=512, kv=A, cu=A, lens=A, batch=1, tokens=1, blocks=1, heads=4, kv_heads=1, dim=128, tpb=64, size=64, rot=128,
             base=1e4, int4=1, zeros=1)
    a.update(c)
    return lib.qs_append_kv_cache(*a.values(), None)


def read(**c):
    a = dict(k=A, v=A, kv=A, cu=A, lens=A, batch=1, tokens=1, blocks=1, kv_heads=1, dim=128, tpb=64, size=64, int4=1, zeros=1)
    a.update(c)
    return lib.qs_read_kv_cache(*a.values(), None)


def prompt(**c):
    a = dict(q=A, qs=512, out=A, os=512, kv=A, cu=A, lens=A, batch=1, tokens=1, seq=1, top=64, blocks=1, heads=4, kv_heads=1, dim=128, tpb=64, size=64, int4=1, zeros=1, scale=0.1,
             ws=None, bytes=0)
    a.update(c)
    return lib.qs_paged_prompt_attention(*a.values(), None)


def shared(**c):
    a = dict(q=A, qs=512, out=A, os=512, kv=A, lens=A, batch=2, shared=1, top=64, blocks=1, heads=4, kv_heads=1, dim=128, tpb=64, size=64, int4=1, zeros=1, scale=0.1, ws=None, bytes=0)
    a.update(c)
    return lib.qs_shared_prefix_attention(*a.values(), None)


GEOMETRY = [dict(dim=64), dict(tpb=32), dict(zeros=0), dict(size=128), dict(size=0, kv_heads=0), dict(kv_heads=-1), dict(blocks=-1), dict(batch=-1), dict(blocks=1 << 25), dict(kv=None),
            dict(lens=None)]
ROWS = [dict(heads=3, kv_heads=2, size=128), dict(heads=0), dict(q=None), dict(q=A + 8), dict(qs=516), dict(qs=384), dict(out=None), dict(out=A + 2), dict(os=504)]
SCALES = [dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")), dict(scale=float("inf"))]


@pytest.mark.parametrize("change", GEOMETRY + ROWS + [dict(k=None), dict(v=A + 4), dict(ks=64), dict(rot=64), dict(base=0.0), dict(base=float("nan")), dict(base=float("inf")), dict(tokens=-1)],
                         ids=str)
def test_append_refuses(change):
    assert append(**change) == -1
    assert b"append_kv_cache" in lib.qs_last_error()


@pytest.mark.parametrize("change", GEOMETRY + [dict(k=None), dict(v=A + 4), dict(tokens=-1)], ids=str)
def test_read_refuses(change):
    assert read(**change) == -1
    assert b"read_kv_cache" in lib.qs_last_error()


@pytest.mark.parametrize("change", GEOMETRY + ROWS + SCALES + [dict(seq=-1), dict(top=-1), dict(tokens=-1), dict(ws=A + 4)], ids=str)
def test_prompt_attention_refuses(change):
    assert prompt(**change) == -1
    assert b"paged_prompt_attention" in lib.qs_last_error()


@pytest.mark.parametrize("change", GEOMETRY + ROWS + SCALES + [dict(shared=-1), dict(shared=2), dict(top=-1), dict(batch=65536), dict(ws=A + 4)], ids=str)
def test_shared_prefix_attention_refuses(change):
    assert shared(**change) == -1
    assert b"shared_prefix_attention" in lib.qs_last_error()


def test_empty_calls_need_nothing():
    assert append(batch=0, q=None, k=None, v=None, out=None, kv=None, lens=None) == 0 and append(tokens=0, q=None) == 0
    assert read(tokens=0, k=None, v=None) == 0 and prompt(tokens=0, q=None, out=None) == 0 and prompt(seq=0, q=None) == 0 and shared(batch=0, q=None, kv=None) == 0


def test_a_work_space_that_is_missing():
    """Splits that are left for another kernel need one, and as many bytes as the library says."""
    need = lib.qs_shared_prefix_attention_workspace_bytes(64, 128, 32, 8)
    assert need > 0
    assert shared(batch=64, shared=128, blocks=130, heads=32, kv_heads=8, size=512, qs=4096, os=4096) == -1
    assert b"workspace" in lib.qs_last_error()
    assert shared(batch=64, shared=128, blocks=130, heads=32, kv_heads=8, size=512, qs=4096, os=4096, ws=A, bytes=need - 1) == -1
    need = lib.qs_paged_prompt_attention_workspace_bytes(1, 24, 24, 60000, 32, 8)
    assert need > 0
    assert prompt(tokens=24, seq=24, top=60000, blocks=940, heads=32, kv_heads=8, size=512, qs=4096, os=4096, ws=A, bytes=need - 1) == -1
    assert b"workspace" in lib.qs_last_error()
    # portions are no longer than the rows, whatever max_seqlen says
    assert lib.qs_paged_prompt_attention_workspace_bytes(1, 24, 24000, 60000, 32, 8) == need
    # nothing to join, or joined by a cluster; and sizes that are none
    for args in ((1, 17, 17, 517, 32, 8), (8, 4096, 512, 4000, 32, 8), (0, 1, 1, 1, 4, 1), (1, 1, 1, 1, 4, 3), (1, -1, 1, 1, 4, 1)):
        assert lib.qs_paged_prompt_attention_workspace_bytes(*args) == 0
    for args in ((1, 100, 32, 8), (8, 2, 32, 8), (8, 0, 32, 8), (0, 5, 32, 8), (8, 5, 32, 0)):
        assert lib.qs_shared_prefix_attention_workspace_bytes(*args) == 0


def test_tensors_that_are_not_on_a_gpu():
    q = torch.zeros(2, 4, 128, dtype=torch.half)
    kv = torch.zeros(2, 2, 1, dtype=torch.int64)
    i32 = torch.zeros(2, dtype=torch.int32)
    args = (64, 64)
    for call in (lambda: backend.append_kv_cache(q, q[:, :1], q[:, :1], kv, None, i32, *args, 128, 1e4, True, True), lambda: backend.read_kv_cache(kv, None, i32, 2, *args, True, True),
                 lambda: backend.paged_prompt_attention(q, kv, None, i32, 1, 64, *args, True, True), lambda: backend.shared_prefix_attention(q, kv, i32, 0, 64, *args, True, True)):
        with pytest.raises(RuntimeError, match="must be on CUDA"):
            call()
    for call in (lambda: backend.append_kv_cache(1, q, q, kv, None, i32, *args, 128, 1e4, True, True), lambda: backend.read_kv_cache(None, None, i32, 2, *args, True, True),
                 lambda: backend.paged_prompt_attention(q.numpy(), kv, None, i32, 1, 64, *args, True, True)):
        with pytest.raises(TypeError):
            call()

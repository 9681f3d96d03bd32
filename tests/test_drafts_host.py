"""Refusals of the operators for drafted tokens and tokens with places of their own, ahead of any call of CUDA: through the C ABI with made-up addresses."""
import ctypes

import pytest

from qserve_b200._lib import lib
from tests.test_paged_host import GEOMETRY, ROWS, SCALES

A = 1 << 20  # an address that nothing reads


def append_at(**c):
    a = dict(q=A, k=A, v=A, qs=512, ks=128, vs=128, out=A, os=512, kv=A, cu=A, lens=A, positions=A, sections=(16, 24, 24), axes=3, interleaved=0, batch=1, tokens=1, blocks=1, heads=4,
             kv_heads=1, dim=128, tpb=64, size=64, rot=128, base=1e4, int4=1, zeros=1)
    a.update(c)
    if a["sections"] is not None:
        a["sections"] = (ctypes.c_int32 * 4)(*a["sections"])
    return lib.qs_append_kv_cache_at(*a.values(), None)


def attend(**c):
    a = dict(q=A, qs=512, out=A, os=512, kv=A, cu=A, lens=A, visible=A, words=1, batch=1, tokens=64, seq=64, top=64, blocks=1, heads=4, kv_heads=1, dim=128, tpb=64, size=64, int4=1, zeros=1,
             scale=0.1, ws=None, bytes=0)
    a.update(c)
    return lib.qs_paged_tree_attention(*a.values(), None)


def tree(**c):
    a = dict(positions=A, visible=A, parents=A, cu=A, lens=A, batch=1, tokens=1, seq=1)
    a.update(c)
    return lib.qs_draft_tree(*a.values(), None)


def verify(**c):
    a = dict(out=A, rows=A, counts=A, logits=A, type=0, stride=64, tokens=A, parents=None, probs=None, ps=0, cu=A, coins=A, draws=A, heats=None, batch=1, T=2, vocab=64, seq=2)
    a.update(c)
    return lib.qs_verify_drafts(*a.values(), None)


def keep(**c):
    a = dict(out=A, kv=A, cu=A, lens=2 * A, rows=A, counts=A, most=4, batch=1, tokens=4, blocks=1, kv_heads=1, dim=128, tpb=64, size=64, int4=1, zeros=1)
    a.update(c)
    return lib.qs_keep_kv_cache(*a.values(), None)


@pytest.mark.parametrize("change", GEOMETRY + ROWS + [dict(k=None), dict(v=A + 4), dict(ks=64), dict(rot=64), dict(base=0.0), dict(base=float("nan")), dict(tokens=-1), dict(positions=None),
                                                      dict(sections=None), dict(axes=0), dict(axes=5), dict(sections=(16, 24, 23)), dict(sections=(80, -8, -8)), dict(sections=(65, 0, -1)),
                                                      dict(sections=(10, 30, 24), interleaved=1), dict(sections=(64, 0, 1))], ids=str)
def test_append_at_refuses(change):
    assert append_at(**change) == -1
    assert b"append_kv_cache_at" in lib.qs_last_error()


@pytest.mark.parametrize("change", GEOMETRY + ROWS + SCALES + [dict(seq=-1), dict(top=-1), dict(tokens=-1), dict(ws=A + 4), dict(visible=None), dict(visible=A + 4), dict(words=0), dict(words=-1),
                                                               dict(tokens=65, seq=65), dict(words=1 << 25)], ids=str)
def test_tree_attention_refuses(change):
    assert attend(**change) == -1
    assert b"paged_tree_attention" in lib.qs_last_error()


@pytest.mark.parametrize("change", [dict(positions=None), dict(visible=None), dict(parents=None), dict(lens=None), dict(batch=-1), dict(tokens=-1), dict(seq=-1), dict(seq=257)], ids=str)
def test_tree_refuses(change):
    assert tree(**change) == -1
    assert b"draft_tree" in lib.qs_last_error()


@pytest.mark.parametrize("change", [dict(out=None), dict(rows=None), dict(counts=None), dict(logits=None), dict(logits=A + 1), dict(logits=A + 2, type=2), dict(type=3), dict(type=-1),
                                    dict(stride=63), dict(tokens=None), dict(probs=A, ps=63), dict(probs=A + 2, ps=64), dict(probs=A, ps=64, parents=A), dict(coins=None), dict(draws=None), dict(batch=-1), dict(T=-1),
                                    dict(vocab=0), dict(vocab=-1), dict(vocab=1 << 29), dict(seq=-1), dict(seq=257), dict(batch=1 << 25)], ids=str)
def test_verify_refuses(change):
    assert verify(**change) == -1
    assert b"verify_drafts" in lib.qs_last_error()


@pytest.mark.parametrize("change", GEOMETRY + [dict(out=None), dict(rows=None), dict(counts=None), dict(most=-1), dict(most=257), dict(lens=A), dict(batch=65536), dict(tokens=-1)], ids=str)
def test_keep_refuses(change):
    assert keep(**change) == -1
    assert b"keep_kv_cache" in lib.qs_last_error()


def test_empty_calls_need_nothing():
    assert append_at(batch=0, q=None, k=None, v=None, out=None, kv=None, lens=None, positions=None) == 0 and append_at(tokens=0, q=None, positions=None) == 0
    assert attend(tokens=0, q=None, out=None, visible=None, words=0) == 0 and attend(seq=0, q=None) == 0 and attend(batch=0, visible=None) == 0
    assert tree(batch=0, parents=None) == 0 and tree(tokens=0, positions=None) == 0 and tree(seq=0) == 0
    assert verify(batch=0, out=None, logits=None) == 0 and keep(batch=0, out=None, kv=None, lens=None, rows=None, counts=None) == 0

"""Refusals of the drafted-decoding and bounded-cache entry points: argument
checks run before any HIP call, so these need no GPU."""
import ctypes

import pytest

import pyvcpp

P = 4096  # an address that is never read


def pages(dtype=pyvcpp.KV_F16, bs=16, hkv=8, d=80, nb=10, stride=None, k=P, v=P, sc=None):
    return pyvcpp.KVPages(dtype, bs, hkv, d, nb, bs * hkv * d if stride is None else stride, hkv * bs, k, v, sc, sc)


def tree(pg=None, q=P, out=P, lse=None, tables=P, blocks=4, st=P, pf=P, mask=P, words=1, seqs=2, nodes=8, prefix=100, heads=64,
         ws=None, nws=0):
    pg = pages() if pg is None else pg
    return pyvcpp.lib().vcpp_paged_tree_attention(ctypes.byref(pg), q, out, lse, tables, blocks, st, pf, mask, words, seqs,
                                                  nodes, prefix, heads, ws, nws, None)


def mass(pg=None, q=P, lse=P, scores=P, stride=200, tables=P, blocks=4, st=P, pf=P, mask=P, words=1, seqs=2, nodes=8,
         prefix=100, heads=64):
    pg = pages() if pg is None else pg
    return pyvcpp.lib().vcpp_attention_mass(ctypes.byref(pg), q, lse, scores, stride, tables, blocks, st, pf, mask, words,
                                            seqs, nodes, prefix, heads, None)


def commit(pg=None, tables=P, blocks=4, pf=P, acc=P, lens=P, seqs=2, n=4, nodes=8, layers=1, ls=0, sls=0):
    pg = pages() if pg is None else pg
    return pyvcpp.lib().vcpp_kv_commit(ctypes.byref(pg), tables, blocks, pf, acc, lens, seqs, n, nodes, layers, ls, sls, None)


def plan(scores=P, pos=None, stride=100, ctx=P, seen=None, seqs=2, hkv=8, top=100, budget=60, first=4, last=16, moves=P, n=40,
         counts=P, new=2 * P, so=P, po=None):
    return pyvcpp.lib().vcpp_kv_evict_plan(scores, pos, stride, ctx, seen, seqs, hkv, top, budget, first, last, moves, n,
                                           counts, new, so, po, None)


def apply(pg=None, tables=P, blocks=4, moves=P, n=10, counts=P, seqs=2):
    pg = pages() if pg is None else pg
    return pyvcpp.lib().vcpp_kv_evict_apply(ctypes.byref(pg), tables, blocks, moves, n, counts, seqs, None)


INV, UNS, WS = pyvcpp.VCPP_E_INVALID, pyvcpp.VCPP_E_UNSUPPORTED, pyvcpp.VCPP_E_WORKSPACE


@pytest.mark.parametrize("fn", [tree, mass])
@pytest.mark.parametrize("kw,code,frag", [
    (dict(pg=pages(dtype=pyvcpp.KV_F32)), UNS, "fp32"),
    (dict(pg=pages(d=72)), UNS, "head_dim"),
    (dict(pg=pages(bs=8)), UNS, "block_size"),
    (dict(pg=pages(k=P + 2)), INV, "aligned"),
    (dict(pg=pages(dtype=pyvcpp.KV_I8)), INV, "scale"),
    (dict(heads=60), INV, "num_heads"),
    (dict(heads=0), INV, "num_heads"),
    (dict(nodes=257, words=5), UNS, "max_nodes"),
    (dict(nodes=65, words=1), INV, "mask_words"),
    (dict(words=0), INV, "mask_words"),
    (dict(nodes=-1), INV, "max_nodes"),
    (dict(seqs=-1), INV, "num_seqs"),
    (dict(prefix=-1), INV, "max_prefix_len"),
    (dict(prefix=2**31 - 300), UNS, "max_prefix_len"),
    (dict(q=None), INV, "NULL"),
    (dict(q=P + 8), INV, "aligned"),
    (dict(st=None), INV, "NULL"),
    (dict(pf=None), INV, "NULL"),
    (dict(tables=None), INV, "block_tables"),
    (dict(blocks=0), INV, "block_tables"),
    (dict(mask=P + 4), INV, "aligned"),
])
def test_tree_and_mass_refusals(fn, kw, code, frag):
    if fn is mass and kw.get("prefix", 0) > 0:
        kw = dict(kw, stride=2**40)
    assert fn(**kw) == code
    assert frag in pyvcpp.last_error()


@pytest.mark.parametrize("kw,code,frag", [
    (dict(out=None), INV, "out"),
    (dict(out=P + 4), INV, "aligned"),
    (dict(prefix=100000), WS, "workspace"),
    (dict(prefix=100000, ws=P, nws=16), WS, "workspace"),
    (dict(prefix=100000, ws=P + 4, nws=2**40), INV, "workspace"),
    (dict(seqs=2**24, nodes=200, words=4), UNS, "too many"),
    (dict(pg=pages(hkv=40000, d=128), heads=40000), UNS, "kv heads"),
    (dict(pg=pages(hkv=1), heads=65535, nodes=256, words=4, prefix=2**24 - 256, seqs=1), UNS, "positions"),
    (dict(pg=pages(hkv=1), heads=4096, nodes=256, words=4, prefix=2**20, seqs=64), UNS, "positions"),
])
def test_tree_refusals(kw, code, frag):
    assert tree(**kw) == code
    assert frag in pyvcpp.last_error()


@pytest.mark.parametrize("kw,code,frag", [
    (dict(lse=None), INV, "lse"),
    (dict(scores=None), INV, "scores"),
    (dict(stride=107), INV, "score_stride"),
])
def test_mass_refusals(kw, code, frag):
    assert mass(**kw) == code
    assert frag in pyvcpp.last_error()


@pytest.mark.parametrize("kw,code,frag", [
    (dict(tables=None), INV, "block_tables"),
    (dict(pf=None), INV, "NULL"),
    (dict(acc=None), INV, "NULL"),
    (dict(lens=None), INV, "NULL"),
    (dict(n=257), UNS, "max_accepted"),
    (dict(nodes=257), UNS, "max_nodes"),
    (dict(n=-1), INV, "max_accepted"),
    (dict(layers=-1), INV, "num_layers"),
    (dict(layers=2, ls=100), INV, "layer_stride"),
    (dict(layers=2, ls=16 * 640 + 4), INV, "aligned"),
    (dict(pg=pages(dtype=pyvcpp.KV_I8, sc=P), layers=2, ls=16 * 640, sls=8), INV, "scale_layer_stride"),
    (dict(seqs=70000), UNS, "too many"),
    (dict(layers=70000, ls=16 * 640), UNS, "too many"),
])
def test_commit_refusals(kw, code, frag):
    assert commit(**kw) == code
    assert frag in pyvcpp.last_error()


@pytest.mark.parametrize("kw,code,frag", [
    (dict(budget=0), INV, "budget"),
    (dict(first=50, last=11), INV, "budget"),
    (dict(first=-1), INV, "keep_first"),
    (dict(stride=99), INV, "stride"),
    (dict(n=39), INV, "max_moves"),
    (dict(hkv=0), INV, "num_kv_heads"),
    (dict(seqs=-1), INV, "num_seqs"),
    (dict(top=-1), INV, "max_context_len"),
    (dict(scores=None), INV, "NULL"),
    (dict(ctx=None), INV, "NULL"),
    (dict(moves=None), INV, "NULL"),
    (dict(counts=None), INV, "NULL"),
    (dict(so=None), INV, "NULL"),
    (dict(new=P), INV, "new_lens"),
    (dict(seqs=2**20), UNS, "too many"),
    (dict(top=2**27, stride=2**27, n=60), UNS, "too long"),
])
def test_plan_refusals(kw, code, frag):
    assert plan(**kw) == code
    assert frag in pyvcpp.last_error()


@pytest.mark.parametrize("kw,code,frag", [
    (dict(tables=None), INV, "block_tables"),
    (dict(moves=None), INV, "NULL"),
    (dict(counts=None), INV, "NULL"),
    (dict(n=-1), INV, "max_moves"),
    (dict(n=2**24 + 1), UNS, "max_moves"),
    (dict(moves=P + 4), INV, "aligned"),
    (dict(seqs=9000), UNS, "too many"),
])
def test_apply_refusals(kw, code, frag):
    assert apply(**kw) == code
    assert frag in pyvcpp.last_error()


def test_empty_calls_succeed_without_buffers():
    assert tree(seqs=0, q=None, out=None, st=None, pf=None, tables=None) == pyvcpp.VCPP_OK
    assert tree(nodes=0, q=None, out=None) == pyvcpp.VCPP_OK
    assert mass(seqs=0, q=None, scores=None, lse=None) == pyvcpp.VCPP_OK
    assert commit(seqs=0, tables=None) == pyvcpp.VCPP_OK
    assert commit(n=0, acc=None) == pyvcpp.VCPP_OK
    assert plan(seqs=0, scores=None) == pyvcpp.VCPP_OK
    assert apply(n=0, moves=None) == pyvcpp.VCPP_OK


def test_workspace_size_of_bad_arguments_is_zero():
    L = pyvcpp.lib()
    pg = pages()
    for a in ((0, 8, 100, 64), (1, 0, 100, 64), (1, 8, -1, 64), (1, 8, 100, 60), (1, 300, 100, 64)):
        assert L.vcpp_tree_workspace_size(ctypes.byref(pg), *a) == 0
    assert L.vcpp_tree_workspace_size(None, 1, 8, 100, 64) == 0
    assert L.vcpp_tree_workspace_size(ctypes.byref(pg), 1, 8, 20000, 64) > 0

"""Refusals of the steps of many rows that need no GPU: the typed calls check their arguments before anything else."""
import ctypes

import pytest
import torch

from tessera_b200 import capi

BAD, NOT_SERVED = int(capi.StatusCode.InvalidArgument), int(capi.StatusCode.UnsupportedFeature)
HUGE = 1 << 62


@pytest.fixture(scope="module")
def lib():
    return capi.load_library()


@pytest.fixture(scope="module")
def mem():
    block = ctypes.create_string_buffer(1 << 16)  # (host memory: nothing may run on it)
    return [ctypes.addressof(block) + (i << 12) for i in range(16)], block


def test_tree_refusals(lib, mem):
    p = mem[0]

    def call(fmt=0, q=p[0], k=p[1], v=p[2], ks=None, vs=None, parents=p[5], out=p[6], m=4, n=16, heads=4, kv=2, d=128, base=0, window=0):
        return lib.tsr_attention_tree(fmt, q, k, v, ks, vs, parents, out, m, n, heads, kv, d, base, window, None)

    for bad in (dict(q=None), dict(k=None), dict(v=None), dict(parents=None), dict(out=None), dict(m=0), dict(heads=0), dict(kv=0), dict(heads=5), dict(d=0),
                dict(fmt=2), dict(fmt=9), dict(n=HUGE)):
        assert call(**bad) == BAD, bad
    for unserved in (dict(d=64), dict(m=257), dict(heads=36)):
        assert call(**unserved) == NOT_SERVED, unserved


def test_norm_refusals(lib, mem):
    p = mem[0]

    def call(q=p[0], k=p[1], qw=p[2], kw=p[3], pos=p[4], qo=p[5], ko=p[6], rows=2, heads=2, kv=1, d=64, rope=32, theta=1e6, sec=(6, 5, 5), eps=1e-6):
        return lib.tsr_qk_norm_rope(q, k, qw, kw, pos, qo, ko, rows, heads, kv, d, rope, theta, *sec, eps, None)

    for bad in (dict(q=None), dict(k=None), dict(qw=None), dict(kw=None), dict(pos=None), dict(qo=None), dict(ko=None), dict(rows=0), dict(heads=0), dict(kv=0),
                dict(rope=66), dict(rope=33), dict(theta=-1.0), dict(theta=float("nan")), dict(sec=(6, 6, 5)), dict(sec=(HUGE, HUGE, 0)), dict(eps=-1.0),
                dict(eps=float("nan")), dict(qo=p[1]), dict(ko=p[0])):
        assert call(**bad) == BAD, bad
    assert call(d=258) == NOT_SERVED


def test_delta_refusals(lib, mem):
    p = mem[0]

    def call(ptrs=p[:8], heads=4, kh=2, dk=64, dv=16, rows=3, sbase=0, abase=0):
        return lib.tsr_delta_chunk_heads(*ptrs, heads, kh, dk, dv, rows, sbase, abase, None)

    for i in range(8):
        assert call(ptrs=[None if j == i else x for j, x in enumerate(p[:8])]) == BAD
    for bad in (dict(heads=0), dict(kh=0), dict(kh=3), dict(rows=0), dict(rows=HUGE), dict(heads=1 << 17), dict(dv=0), dict(ptrs=[*p[:4], p[2], *p[5:8]])):
        assert call(**bad) == BAD, bad
    for unserved in (dict(dk=96), dict(dv=24)):
        assert call(**unserved) == NOT_SERVED, unserved


def test_logprob_refusals(lib, mem):
    p = mem[0]

    def call(x=p[0], targets=p[1], lp=p[2], ent=p[3], ids=p[4], tops=p[5], rows=2, vocab=10, k=3, base=0):
        return lib.tsr_logprob_rows(x, targets, lp, ent, ids, tops, rows, vocab, k, base, None)

    for bad in (dict(x=None), dict(targets=None), dict(lp=None), dict(ent=None), dict(ids=None), dict(tops=None), dict(rows=0), dict(vocab=0), dict(k=33),
                dict(vocab=HUGE), dict(rows=HUGE)):
        assert call(**bad) == BAD, bad


def test_tree_over_a_cache_off_its_elements_boundary(lib, mem):
    """A binary16 or fp32 cache has to lie on its elements' boundary (bytes may lie anywhere)."""
    p = mem[0]

    def call(fmt, k, v):
        return lib.tsr_attention_tree(fmt, p[0], k, v, p[3], p[4], p[5], p[6], 4, 16, 4, 2, 128, 0, 0, None)

    for fmt, off in ((0, 1), (0, 2), (1, 1)):
        assert call(fmt, p[1] + off, p[2]) == BAD and call(fmt, p[1], p[2] + off) == BAD


def test_queries_that_are_the_keys(lib, mem):
    """In place over queries that the keys (or the weights) are read from as well: another CTA may read them after they are written."""
    p = mem[0]

    def call(q=p[0], k=p[1], qw=p[2], kw=p[3], qo=p[5], ko=p[6]):
        return lib.tsr_qk_norm_rope(q, k, qw, kw, p[4], qo, ko, 2, 1, 1, 64, 32, 1e6, 6, 5, 5, 1e-6, None)

    def append(q=p[0], k=p[1], v=p[7], qw=p[2], qo=p[5]):
        return lib.tsr_qk_norm_rope_append(0, q, k, v, qw, p[3], p[4], qo, p[8], p[9], None, None, 2, 0, 1, 1, 64, 32, 1e6, 6, 5, 5, 1e-6, None)

    for bad in (dict(k=p[0], qo=p[0]), dict(k=p[0], ko=p[0]), dict(qw=p[0], qo=p[0]), dict(kw=p[1], ko=p[1]), dict(qw=p[1], ko=p[1])):
        assert call(**bad) == BAD, bad
    for bad in (dict(k=p[0], qo=p[0]), dict(v=p[0], qo=p[0]), dict(qw=p[0], qo=p[0])):
        assert append(**bad) == BAD, bad


@pytest.mark.skipif(torch.cuda.is_available(), reason="the call would run")
def test_logprob_without_a_top_list_overlaps_nothing_there(lib, mem):
    """With no top list its places are not written, whatever they are."""
    p = mem[0]
    call = lambda k, at: lib.tsr_logprob_rows(p[0], p[1], p[2], p[3], at, at, 2, 10, k, 0, None)
    assert call(2, p[0] + 16) == BAD
    assert call(0, p[0] + 16) not in (BAD, NOT_SERVED)  # (accepted: what fails without a GPU is the launch)

"""The paged K/V cache without a GPU: what its description and its entry points refuse, and the oracle that the GPU tests rest on
against attention written over a plain sequence."""

import ctypes as C
import random

import numpy as np
import pytest
import torch

from kiln_b200 import _cabi
from kiln_b200.cache import PagedCache
from oracle import cache_oracle
from oracle.cache_oracle import Oracle

SIZES = dict(layers=2, sequences=3, max_pages=4, pages=10, kv_heads=2, head_dim=64, page_tokens=16)


@pytest.fixture(scope="module")
def lib():
    _cabi.build()
    return _cabi.load()


def desc(**changes):
    d = dict(dtype=1, **SIZES, pool=16, pool_bytes=1 << 40, table=16, held=16, lengths=16, refs=16)
    d.update(changes)
    return _cabi.CacheDesc(**d)


def test_description_layout():
    assert C.sizeof(_cabi.CacheDesc) == 8 * 4 + 8 + 8 + 4 * 8
    assert C.sizeof(_cabi.Rows) == 8 + 4 + 4 + 3 * 8


@pytest.mark.parametrize("change, status", [
    (dict(dtype=3), -1), (dict(dtype=-1), -1), (dict(layers=0), -1), (dict(sequences=0), -1), (dict(max_pages=-1), -1), (dict(pages=0), -1), (dict(kv_heads=0), -1),
    (dict(page_tokens=0), -2), (dict(page_tokens=4), -2), (dict(page_tokens=24), -2), (dict(page_tokens=512), -2), (dict(page_tokens=-16), -2),
    (dict(head_dim=8), -2), (dict(head_dim=72), -2), (dict(head_dim=272), -2), (dict(head_dim=0), -2),
    (dict(max_pages=1 << 26), -2), (dict(sequences=(1 << 20) + 1), -2), (dict(pages=1 << 30, page_tokens=8), -2),
    (dict(pool=0), -1), (dict(pool=8), -1), (dict(table=0), -1), (dict(held=0), -1), (dict(lengths=0), -1), (dict(refs=0), -1),
    (dict(pool_bytes=2 * 2 * 10 * 2 * 16 * 64 * 2 - 1), -3)])
def test_descriptions_that_are_refused(lib, change, status):
    out = C.c_void_p(1)
    assert lib.kb200_cache_check(C.byref(desc(**change))) == status
    assert lib.kb200_cache_create(C.byref(desc(**change)), 0, C.byref(out)) == status
    assert out.value is None and lib.kb200_last_error()


def test_descriptions_that_are_taken(lib):
    for change in (dict(), dict(pool_bytes=2 * 2 * 10 * 2 * 16 * 64 * 2), dict(dtype=0, head_dim=16, page_tokens=8), dict(dtype=2, head_dim=256, page_tokens=256)):
        assert lib.kb200_cache_check(C.byref(desc(**change))) == 0
    assert lib.kb200_cache_check(None) == -1
    assert lib.kb200_cache_create(None, 0, None) == -1


def test_calls_without_a_cache(lib):
    assert lib.kb200_cache_fork(None, 16, None) == -1
    assert lib.kb200_cache_reserve(None, 16, None) == -1
    assert lib.kb200_cache_truncate(None, 16, None) == -1
    assert lib.kb200_cache_compact(None, None) == -1
    assert lib.kb200_cache_append(None, 0, None, None, 1, 1, None, None, None) == -1
    assert lib.kb200_cache_accept(None, 16, None, 0, None) == -1
    assert lib.kb200_cache_attend_workspace(None, 1, 1, 1) == 0
    assert lib.kb200_cache_attend(None, 0, None, None, 1, 1, None, None, None, None, 1.0, None, 0, None) == -1
    assert lib.kb200_cache_status(None) == -1
    lib.kb200_cache_destroy(None)


@pytest.mark.parametrize("change, error", [
    (dict(dtype=torch.float64), TypeError), (dict(layers=0), ValueError), (dict(pages=-4), ValueError), (dict(sequences=True), ValueError),
    (dict(max_pages=2.0), ValueError), (dict(page_tokens=20), NotImplementedError), (dict(head_dim=100), NotImplementedError)])
def test_caches_that_are_refused_before_a_gpu_is_asked_for(lib, change, error):
    with pytest.raises(error):
        PagedCache(**dict(SIZES, **change))


@pytest.mark.skipif(torch.cuda.is_available(), reason="without a GPU only")
def test_there_is_no_cpu_path(lib):
    with pytest.raises(RuntimeError):
        PagedCache(**SIZES)


def test_oracle_keeps_sequences_through_any_operations():
    """Whatever forks, drafts and compactions do to the pages, a sequence reads as the list of its tokens."""
    dice = random.Random(5)
    o = Oracle(1, 4, 6, 30, 1, 16, 8, torch.float32)
    said = [[] for _ in range(4)]
    for step in range(300):
        kind = dice.choice(["draft", "draft", "draft", "fork", "truncate", "compact"])
        if kind == "draft":
            counts = [dice.randint(0, min(7, 48 - len(x))) for x in said]
            before = o.faults
            o.reserve(counts)
            assert o.faults == before
            tokens = torch.randn(4, 7, 1, 16)
            o.append(0, tokens, -tokens, counts)
            kept = [sorted(dice.sample(range(c), dice.randint(0, c))) for c in counts]
            o.accept([len(x) for x in kept], [x + [0] * (7 - len(x)) for x in kept])
            for s, x in enumerate(kept):
                said[s] = said[s] + [tokens[s, i, 0].double().numpy() for i in x]
        elif kind == "fork":
            sources = [dice.choice([-1, s, s, dice.randrange(4)]) for s in range(4)]
            o.fork(sources)
            said = [list(said[x]) if x >= 0 else [] for x in sources]
        elif kind == "truncate":
            cut = [dice.choice([-1, -1, dice.randint(0, 48)]) for _ in said]
            o.truncate(cut)
            said = [x if n < 0 else x[:n] for x, n in zip(said, cut)]
        else:
            o.compact()
        assert o.lengths == [len(x) for x in said] and o.faults == 0
        assert sum(o.refs) == sum(len(r) for r in o.rows) and [r for r in o.refs] == [sum(r.count(p) for r in o.rows) for p in range(30)]
        for s, x in enumerate(said):
            for at, token in enumerate(x):
                page, row = o._place(s, at)
                assert (o.pool[0, 0, page, 0, row] == token).all() and (o.pool[0, 1, page, 0, row] == -token).all()


def test_oracle_attention_against_attention_over_a_plain_sequence():
    generator = torch.Generator().manual_seed(3)
    o = Oracle(1, 1, 4, 4, 2, 32, 8, torch.float32)
    k, v, q = (torch.randn(1, 21, h, 32, generator=generator) for h in (2, 2, 6))
    o.reserve([21])
    o.append(0, k, v)
    got, *_ = o.attend(0, q)
    kk, vv = (x.double().repeat_interleave(3, 2).transpose(1, 2) for x in (k, v))
    want = torch.nn.functional.scaled_dot_product_attention(q.double().transpose(1, 2), kk, vv, is_causal=True).transpose(1, 2)
    assert np.abs(got - want.numpy()).max() < 1e-13
    o.accept([13])
    some = np.tril(np.ones((8, 8), bool))
    o.reserve([8])
    o.append(0, k[:, 13:], v[:, 13:])
    again, *_ = o.attend(0, q[:, 13:], torch.from_numpy(some))
    assert np.abs(again - want.numpy()[:, 13:]).max() < 1e-13
    assert cache_oracle.rounded(torch.tensor([1.0 + 2**-9]), torch.bfloat16)[0] == 1.0


@pytest.mark.parametrize("name", ["cache_attention.cu", "cache_attention_tc.cu"])
def test_copies_in_flight_land_before_shared_memory_is_released(name):
    """What a CTA does when one of its bounded waits has run out, read from the source (no kernel is made to fail for it): it meets, lets copies that are
    under way land, and only then frees tensor memory and ends."""
    from kiln_b200._cabi import CSRC_DIR

    text = (CSRC_DIR / name).read_text()
    way_out = text.index("if (gave_up && threadIdx.x == 0) {")
    assert text.rindex("__syncthreads();", 0, way_out) > 0
    assert text.index("let_copies_land();", way_out) < text.index("__syncthreads();", way_out)
    if "tcgen05.alloc" in text:
        assert text.index("tcgen05.dealloc") > text.index("__syncthreads();", way_out)
    assert "mbar_wait(" not in text and "mbar_try_wait(" not in text       # only waits that end

"""The paged K/V cache on the GPU: attention to a window, released pages, weighed and evicted tokens, against the oracle."""

import ctypes as C
import random

import numpy as np
import pytest
import torch

from kiln_b200 import _cabi
from oracle.cache_oracle import BAD_INDEX, NO_ROOM, SHARED
from oracle.cache_steps_oracle import Steps
import test_paged_cache_gpu
from test_paged_cache_gpu import BF16, F16, F32, faults_of, ints, make, same, tree

pytestmark = pytest.mark.gpu


def filled(lengths, counts, group=1, **sizes):
    """A cache with that many committed and drafted tokens, and queries of `group` heads to a key head."""
    cache, q = test_paged_cache_gpu.filled(lengths, counts, **sizes)
    if group > 1:
        q = torch.randn(*q.shape[:2], group * cache.kv_heads, cache.head_dim, generator=torch.Generator("cuda").manual_seed(group), device="cuda")
    return cache, q


def places_of(sees):
    return (sees.sum(-1) - 1).astype(np.int32)


def look(cache, q, mask=None, counts=None, slots=None, scale=None, window=None, sinks=0, places=None):
    """The attention and its lse against float64: errors as in test_paged_cache_gpu.bound; lse is off by what a score and a sum of weights are, and, having been a power of two's exponent,
    by 2^-21 of its own and the scores' sizes."""
    o = Steps.of(cache)
    lse = torch.full(q.shape[:3], 7.0, device="cuda")
    given = dict(mask=None if mask is None else torch.from_numpy(mask).cuda(), counts=None if counts is None else ints(counts), slots=None if slots is None else ints(slots),
                 scale=scale, window=window, sinks=sinks, places=None if places is None else ints(places.tolist()))
    got = cache.attend(0, q, **given, lse=lse)
    assert torch.equal(got, cache.attend(0, q, **given)) or window is None
    assert faults_of(cache) == 0
    want, weight, sizes, want_lse = o.look(0, q, mask, counts, slots, scale, window, sinks, places)
    dim, dtype = q.shape[3], cache.dtype
    u = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    score = sizes * ((dim / 8 + 8) * 2.0**-23 + (2.0**-21 if dtype == F32 else 0.0) + 3 * 2.0**-24)
    keys = max(o.lengths) + q.shape[1]
    wide = 2 * score + 2.0**-21 + (keys / 8 + 64) * 2.0**-23 + (2.0**-21 if dtype == F32 else 0.0)
    allowed = weight * (u + wide * (1 + u)) + (u + 2.0**-24) * np.abs(want) + 1e-30
    assert np.isfinite(got.cpu().float().numpy()).all()
    assert (np.abs(got.cpu().double().numpy() - want) / allowed).max(initial=0.0) <= 1.0
    sees = np.isfinite(want_lse)
    got_lse = lse.cpu().double().numpy()
    assert np.array_equal(got_lse == -np.inf, ~sees)
    allowed = (wide + sizes * 2.0**-21)[..., 0][sees] + np.abs(want_lse[sees]) * 2.0**-21
    assert (np.abs(got_lse[sees] - want_lse[sees]) / allowed).max(initial=0.0) <= 1.0
    return got, lse


SHAPES = [
    # dtype, lengths, counts, kv_heads, group, head_dim, page_tokens
    (BF16, [0], [1], 1, 1, 64, 16),
    (F32, [0, 1, 15, 16, 17, 200], [1, 1, 1, 1, 1, 1], 2, 1, 64, 16),
    (F16, [63, 64, 65, 127, 128, 129, 400], [1, 2, 3, 2, 1, 3, 3], 1, 4, 128, 32),
    (BF16, [5, 300, 0, 31], [7, 0, 5, 1], 3, 2, 80, 8),
    (BF16, [700, 90], [12, 3], 2, 4, 128, 64),
    (F32, [333, 20], [9, 4], 2, 2, 128, 8),
    (F32, [150], [70], 1, 1, 256, 16),
    (F16, [500, 10], [20, 31], 2, 1, 256, 128),
    (BF16, [1000], [1], 1, 8, 64, 16),
]


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("window, sinks", [(1, 0), (1, 3), (17, 0), (64, 4), (100, 70), (129, 1), (5000, 9), (None, 0)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_to_a_window(shape, window, sinks, masked):
    dtype, lengths, counts, kv_heads, group, head_dim, page_tokens = shape
    cache, q = filled(lengths, counts, dtype=dtype, kv_heads=kv_heads, group=group, head_dim=head_dim, page_tokens=page_tokens)
    mask = places = None
    if masked:
        mask = np.stack([tree(random.Random(b), q.shape[1]) for b in range(len(lengths))])
        places = None if window is None else places_of(mask)
    look(cache, q, mask, counts, window=window, sinks=sinks, places=places)


@pytest.mark.parametrize("dtype, head_dim, group, page_tokens", [(BF16, 128, 3, 16), (F16, 64, 4, 64), (F32, 64, 2, 8), (BF16, 256, 1, 32)])
@pytest.mark.parametrize("window, sinks", [(1, 0), (40, 2), (200, 0), (333, 100)])
def test_pieces_of_prompts(dtype, head_dim, group, page_tokens, window, sinks):
    """Many row tiles, each with a window of its own, and rows that end inside one."""
    cache, q = filled([500, 0, 70], [260, 130, 1], dtype=dtype, kv_heads=1, group=group, head_dim=head_dim, page_tokens=page_tokens)
    look(cache, q, None, [260, 130, 1], window=window, sinks=sinks)


@pytest.mark.parametrize("dtype, head_dim, group, tokens", [(BF16, 128, 4, 200), (F16, 64, 4, 200), (BF16, 80, 3, 200), (F16, 112, 8, 20), (BF16, 256, 1, 40), (F32, 64, 1, 70), (BF16, 64, 2, 3)])
def test_queries_of_the_caches_type(dtype, head_dim, group, tokens):
    """As they lie, in part of another tensor, and overwritten by their results; many sequences, so that a CTA goes from one item to the next."""
    counts = [tokens, 1, tokens // 2, tokens - 1] * 6
    cache, q = filled([300, 0, 77, 1000] * 6, counts, dtype=dtype, kv_heads=2, group=group, head_dim=head_dim, page_tokens=16)
    q = q.to(dtype)
    want, lse = look(cache, q, None, counts, window=100, sinks=5)
    rounded = cache.attend(0, q.float(), counts=ints(counts), window=100, sinks=5)
    assert torch.equal(rounded, want)
    wide = torch.full((tokens, 24, 2 * group + 3, head_dim + 16), float("nan"), dtype=dtype, device="cuda")
    part = wide.transpose(0, 1)[:, :, 2:-1, 8:-8]
    part.copy_(q)
    got = torch.empty_like(lse)
    assert torch.equal(cache.attend(0, part, counts=ints(counts), window=100, sinks=5, lse=got), want) and torch.equal(got, lse)
    assert cache.attend(0, part, counts=ints(counts), window=100, sinks=5, out=part) is part and torch.equal(part, want)
    assert torch.isnan(wide[:, :, :2]).all() and torch.isnan(wide[..., :8]).all() and faults_of(cache) == 0


@pytest.mark.parametrize("dtype, tokens, head_dim", [(BF16, 1, 64), (BF16, 9, 128), (F16, 40, 64), (F32, 3, 64), (F32, 20, 128), (BF16, 3, 256), (F16, 90, 128)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_a_window_hides_does_not_reach_a_row(dtype, tokens, head_dim, bad):
    """Keys and values that no row sees, in whole tiles and at both edges of the gap."""
    cache, q = filled([777], [tokens], dtype=dtype, kv_heads=2, group=2, head_dim=head_dim, page_tokens=16)
    window, sinks = 201, 21
    clean = cache.attend(0, q, window=window, sinks=sinks)
    hidden = torch.arange(sinks, 777 - window + 1, device="cuda")
    pages = cache.table[0, hidden // 16].long()
    for i in range(2):
        cache.pool[0, i, pages, :, hidden % 16] = bad
    assert torch.equal(clean, cache.attend(0, q, window=window, sinks=sinks))
    # a key that the first token still sees and the others do not
    if tokens > 1:
        last = 777 - window + 1
        page = cache.table[0, last // 16].long()
        cache.pool[0, :, page, :, last % 16] = bad
        got = cache.attend(0, q, window=window, sinks=sinks)
        assert torch.equal(clean[:, 1:], got[:, 1:]) and not torch.isfinite(got[:, 0]).all()
    assert faults_of(cache) == 0


@pytest.mark.parametrize("dtype, tokens", [(BF16, 1), (F16, 5), (F32, 5), (BF16, 40), (BF16, 70)])
def test_rows_that_see_nothing(dtype, tokens):
    """Masks that show no drafted token, and places that leave no committed one in the window; and rows of no token, and of no sequence."""
    cache, q = filled([50, 3, 0], [tokens] * 3, dtype=dtype, kv_heads=1, group=2, head_dim=64)
    mask, places = np.zeros((tokens, tokens), bool), np.full((3, tokens), tokens - 1, np.int32)
    window = max(1, tokens - 1)
    _, lse = look(cache, q, mask, None, window=window, places=places)
    assert (lse == -float("inf")).all()
    lse.fill_(5.0)
    out = cache.attend(0, q, counts=ints([0, 1, 0]), slots=ints([0, 1, 9]), window=3, lse=lse)
    assert faults_of(cache) == BAD_INDEX
    assert (out[0] == 0).all() and (out[2] == 0).all() and (out[1, 1:] == 0).all()
    assert (lse[[0, 2]] == -float("inf")).all() and (lse[1, 1:] == -float("inf")).all() and torch.isfinite(lse[1, 0]).all()


@pytest.mark.parametrize("places", [[[0, 0, 0]], [[5, 1, -4]], [[2, 2, 2]]])
def test_places_without_a_mask_and_out_of_range(places):
    cache, q = filled([300], [3], dtype=BF16, kv_heads=1, head_dim=64)
    look(cache, q, None, [3], window=30, sinks=2, places=np.array(places, np.int32))
    look(cache, q, np.ones((3, 3), bool), [3], window=2, places=np.array(places, np.int32))


@pytest.mark.parametrize("dtype, lengths, tokens, head_dim, group", [
    (F32, [0, 20, 300], 5, 64, 1), (F32, [60], 70, 64, 2), (BF16, [3, 62, 190], 12, 64, 1), (F16, [0, 50], 40, 256, 1), (BF16, [60, 200], 40, 128, 1), (F16, [1, 58, 700], 64, 64, 4),
    (BF16, [0, 60], 90, 64, 3), (F16, [26, 1], 138, 128, 1)])
@pytest.mark.parametrize("window", [None, 2**31 - 1, 2**31 - 60])
def test_masks_that_show_later_tokens_through_windows_that_hide_nothing(dtype, lengths, tokens, head_dim, group, window):
    """What a mask shows is seen wherever it stands, and how far places are in front of a key is no matter."""
    cache, q = filled(lengths, [tokens] * len(lengths), dtype=dtype, kv_heads=2, group=group, head_dim=head_dim, page_tokens=8)
    dice = np.random.default_rng(tokens)
    mask = dice.random((len(lengths), tokens, tokens)) < 0.2
    mask[:, 0] = np.arange(tokens) == tokens - 1            # the first sees the last of them only
    places = None if window is None else np.minimum(dice.integers(0, 4, (len(lengths), tokens)), tokens - 1).astype(np.int32)
    look(cache, q, mask, None, window=window, places=places)
    look(cache, q, mask[0], None, window=window, sinks=0 if window is None else 3)
    if window is not None:
        look(cache, q, None, None, window=window, places=places)


def test_strides_and_types_of_what_a_window_asks_for():
    cache, q = filled([90, 200], [3, 5], dtype=BF16, kv_heads=2, group=2, head_dim=64)
    mask = np.stack([tree(random.Random(b), 5) for b in range(2)])
    places, counts = ints(places_of(mask).tolist()), ints([3, 5])
    given = dict(mask=torch.from_numpy(mask).cuda(), counts=counts, window=40, sinks=1)
    lse = torch.empty(2, 5, 4, device="cuda")
    want = cache.attend(0, q, places=places, lse=lse, **given)
    wide = torch.zeros(4, 5, 2, 6, device="cuda")
    strided = wide.permute(2, 1, 0, 3)[..., 3]                             # [2, 5, 4]
    apart = torch.zeros(2, 10, dtype=torch.int64, device="cuda")
    apart[:, ::2] = places
    got = cache.attend(0, q, places=apart[:, ::2], lse=strided, out=torch.zeros(2, 5, 8, 64, dtype=BF16, device="cuda")[:, :, ::2], **given)
    assert torch.equal(got, want) and torch.equal(strided, lse) and wide.count_nonzero() <= 2 * 5 * 4
    version = lse._version
    cache.attend(0, q, places=places, lse=lse, **given)
    assert lse._version > version


# ---- pages and tokens that are given up ----------------------------------------------------------

@pytest.mark.parametrize("dtype, page_tokens, head_dim, sequences, pages", [(BF16, 8, 16, 5, 60), (F32, 16, 48, 3, 24), (F16, 32, 80, 40, 120), (BF16, 8, 32, 200, 1600)])
def test_any_operations_leave_what_the_lists_say(dtype, page_tokens, head_dim, sequences, pages):
    """Forks, drafts, truncations and compactions among releases and evictions."""
    dice = random.Random(page_tokens * sequences + 1)
    generator = torch.Generator("cuda").manual_seed(1)
    max_pages = 7
    cache = make(dtype=dtype, page_tokens=page_tokens, head_dim=head_dim, sequences=sequences, pages=pages, max_pages=max_pages, kv_heads=2, layers=2)
    o = Steps.of(cache)
    seen = moved = 0
    for step in range(60 if sequences < 100 else 14):
        kind = dice.choice(["draft", "draft", "draft", "fork", "truncate", "compact", "release", "evict", "evict", "evict"])
        if kind == "draft":
            counts = [dice.choice([0, 1, dice.randint(0, 3 * page_tokens)]) for _ in range(sequences)]
            counts = [min(c, max_pages * page_tokens - n) for c, n in zip(counts, o.lengths)]
            tokens = max(max(counts), 1)
            cache.reserve(ints(counts))
            o.reserve(counts)
            k, v = (torch.randn(2, sequences, tokens, 2, head_dim, generator=generator, device="cuda") for _ in range(2))
            for layer in range(2):
                cache.append(layer, k[layer], v[layer], ints(counts))
                o.append(layer, k[layer], v[layer], counts)
            cache.accept(ints(counts))
            o.accept(counts)
        elif kind == "fork":
            sources = [dice.choice([-1, s, s, s, s, dice.randrange(sequences)]) for s in range(sequences)]
            cache.fork(ints(sources))
            o.fork(sources)
        elif kind == "truncate":
            lengths = [-1 if -1 in o.rows[s] else dice.choice([-1, -1, dice.randint(0, max_pages * page_tokens)]) for s in range(sequences)]
            cache.truncate(ints(lengths))
            o.truncate(lengths)
        elif kind == "compact":
            cache.compact()
            o.compact()
        elif kind == "release":
            window, sinks = dice.randint(1, 4 * page_tokens), dice.choice([0, 1, page_tokens, page_tokens + 1])
            if dice.random() < 0.5:
                cache.release(window, sinks)
                o.release(window, sinks)
        else:
            weights = torch.rand(sequences, max_pages * page_tokens, generator=generator, device="cuda")
            weights = (weights * dice.choice([3, 1e9])).floor()               # (many that are equal, or none)
            keep = [dice.choice([-1, 0, 1, dice.randint(0, max_pages * page_tokens), n, n // 2, n // 3]) for n in o.lengths]
            recent, sinks = dice.choice([0, 1, page_tokens, 999]), dice.choice([0, 1, 5, 999])
            before = list(o.lengths)
            want = o.evict(weights.cpu().numpy(), keep, recent, sinks)
            got = cache.evict(weights, ints(keep), recent=recent, sinks=sinks)
            assert np.array_equal(got.cpu().numpy(), want), step
            moved += before != o.lengths
        same(cache, o)
        assert faults_of(cache) == o.faults, (step, kind)
        seen |= o.faults
        o.faults = 0
    assert moved > 0


@pytest.mark.parametrize("length", [1, 31, 33, 1000, 1024, 1025, 5000, 8193, 20000])
def test_evicted_tokens(length):
    """Ties, NaN, infinities and zeros of both signs; weights in place and in rows of another tensor."""
    cache, _ = filled([length, 40], [0, 0] if length < 1 else [1, 1], dtype=BF16, kv_heads=1, head_dim=16, page_tokens=8)
    dice = np.random.default_rng(length)
    start = [t.clone() for t in (cache.pool, cache.table, cache.held, cache.lengths, cache.refs)]
    width = cache.max_pages * 8
    for name, values in dict(any=dice.random((2, width)), few=dice.integers(0, 3, (2, width)), same=np.zeros((2, width)), signs=dice.choice([0.0, -0.0, -1.0, 1.0], (2, width)),
                             odd=dice.choice([np.nan, -np.nan, np.inf, -np.inf, 1.0, -3.0, 1e-42, 2e-42], (2, width)),
                             near=1.0 + dice.integers(0, 4, (2, width)) * 2.0**-23).items():
        for keep, recent, sinks in ((length // 2, 0, 0), (length // 3 + 1, 5, 3), (length - 1, length, 0), (0, 0, 0), (1, 0, 9)):
            for t, x in zip((cache.pool, cache.table, cache.held, cache.lengths, cache.refs), start):
                t.copy_(x)
            o = Steps.of(cache)
            weights = torch.from_numpy(values.astype(np.float32)).cuda()
            want = o.evict(weights.cpu().numpy(), [keep, 20], recent, sinks)
            wide = torch.full((2, width + 5), 4.0, device="cuda")
            wide[:, 2:2 + width] = weights
            out = cache.evict(wide[:, 2:2 + width], ints([keep, 20]), recent, sinks, out=wide[:, 2:2 + width])
            assert out.data_ptr() == wide.data_ptr() + 8 and (wide[:, :2] == 4).all() and (wide[:, -3:] == 4).all()
            assert np.array_equal(out.cpu().numpy(), want, equal_nan=True), name
            same(cache, o)
            assert faults_of(cache) == 0


def test_sequences_that_cannot_be_evicted_stay():
    cache, _ = filled([100, 100, 100], [1, 1, 1], dtype=F16, kv_heads=1, head_dim=16, page_tokens=8)
    cache.truncate(ints([100, 100, 100]))
    cache.fork(ints([0, 0, 2]))                     # two share their pages
    cache.release(10, 0)                            # ... and have given most of them back
    o = Steps.of(cache)
    weights = torch.rand(3, cache.max_pages * 8, device="cuda")
    want = o.evict(weights.cpu().numpy(), [50, 8, 9], 9, 0)
    got = cache.evict(weights, ints([50, 8, 9]), recent=9)
    assert np.array_equal(got.cpu().numpy(), want)
    assert faults_of(cache) == o.faults == NO_ROOM | SHARED or faults_of(cache) == 0
    same(cache, o)
    # the pages that sequences share may stay where nothing moves into them
    cache, _ = filled([100, 100], [1, 1], dtype=F16, kv_heads=1, head_dim=16, page_tokens=8)
    cache.truncate(ints([40, 0]))
    cache.fork(ints([0, 0]))
    cache.reserve(ints([60, 30]))
    k = torch.randn(2, 60, 1, 16, device="cuda")
    cache.append(0, k, k, ints([60, 30]))
    cache.accept(ints([60, 30]))
    o = Steps.of(cache)
    weights = torch.rand(2, cache.max_pages * 8, device="cuda")
    weights[:, :40] += 1
    want = o.evict(weights.cpu().numpy(), [60, 50], 0, 0)
    assert np.array_equal(cache.evict(weights, ints([60, 50])).cpu().numpy(), want) and o.lengths == [60, 50]
    same(cache, o)
    assert faults_of(cache) == 0


def test_evictions_that_would_write_into_shared_pages_are_refused():
    """Each fault by itself, and both together: told once, with the pages, the tables and the weights as they were."""
    def three(keep, release=None):
        cache, _ = filled([100, 100, 100], [1, 1, 1], dtype=F16, kv_heads=1, head_dim=16, page_tokens=8)
        cache.fork(ints([0, 0, 2]))                 # the first two share their pages, all of which are there
        if release is not None:
            cache.release(*release)
        o = Steps.of(cache)
        weights = torch.arange(3 * cache.max_pages * 8, device="cuda").view(3, -1).float()
        want = o.evict(weights.cpu().numpy(), keep, 0, 0)
        got = cache.evict(weights, ints(keep))
        told = faults_of(cache)
        assert np.array_equal(got.cpu().numpy(), want) and told == o.faults and faults_of(cache) == 0
        same(cache, o)
        return told, cache.lengths.tolist(), weights, got

    told, lengths, weights, got = three([50, 99, 40])
    assert told == SHARED and lengths == [100, 100, 40]
    assert torch.equal(got[:2, :100], weights[:2, :100]) and got[:2, 100:].count_nonzero() == 0
    told, lengths, *_ = three([-1, -1, 50], (10, 0))                   # the third's first pages are gone, into which tokens would move
    assert told == NO_ROOM and lengths == [100, 100, 100]
    told, lengths, *_ = three([50, 40, -1], (10, 40))                  # the first pages are shared, and of the heaviest tokens some are gone
    assert told == NO_ROOM | SHARED and lengths == [100, 100, 100]
    told, lengths, *_ = three([100, -1, 0])                            # nothing moves
    assert told == 0 and lengths == [100, 100, 0]


def test_released_pages_are_not_missed_by_the_window_that_left_them():
    cache, q = filled([700, 33, 512], [3, 3, 3], dtype=BF16, kv_heads=2, group=2, head_dim=64, page_tokens=8)
    before = [cache.attend(0, q, window=w, sinks=20) for w in (100, 64, 1)]
    free = (cache.refs == 0).sum().item()
    cache.release(100, 20)
    assert (cache.refs == 0).sum().item() - free == sum(max(0, (n - 99) // 8 - 3) for n in (700, 33, 512))
    cache.pool[:, :, cache.refs == 0] = float("nan")
    o = Steps.of(cache)
    assert all(torch.equal(cache.attend(0, q, window=w, sinks=20), x) for w, x in zip((100, 64, 1), before))
    assert faults_of(cache) == 0
    out = cache.attend(0, q)                        # a call that wants them
    assert faults_of(cache) == BAD_INDEX and torch.equal(out[1], cache.attend(0, q)[1])
    assert faults_of(cache) == BAD_INDEX
    cache.attend(0, q, window=120, sinks=20)
    assert faults_of(cache) == BAD_INDEX
    cache.release(100, 20)                          # again: nothing is left to give
    same(cache, o)
    cache.truncate(ints([300, -1, -1]))             # into pages that are gone
    cache.reserve(ints([1, 0, 0]))
    assert faults_of(cache) == BAD_INDEX


# ---- weights -------------------------------------------------------------------------------------

WEIGHED = [
    # dtype, lengths, counts, kv_heads, group, head_dim, page_tokens
    (BF16, [0], [1], 1, 1, 64, 16),
    (F32, [0, 1, 15, 200, 17], [1, 1, 1, 1, 1], 2, 1, 64, 16),
    (F16, [63, 64, 65, 400], [1, 2, 3, 3], 1, 4, 128, 32),
    (BF16, [5, 300, 0, 31], [7, 0, 5, 1], 3, 2, 80, 8),
    (BF16, [700, 90], [12, 3], 8, 4, 128, 64),
    (F32, [333, 20], [9, 4], 5, 2, 128, 8),
    (F32, [50], [40], 1, 1, 256, 16),
    (F32, [70, 20], [2, 3], 12, 1, 16, 16),
    (F16, [100, 10], [20, 31], 2, 1, 256, 128),
    (BF16, [77], [1], 12, 1, 112, 16),
]


def weigh(cache, q, mask=None, counts=None, slots=None, scale=None, weights=None, **kw):
    """The weights of an attention's own lse, against float64 (what they may be off by: see the oracle)."""
    given = dict(mask=None if mask is None else torch.from_numpy(mask).cuda(), counts=None if counts is None else ints(counts), slots=None if slots is None else ints(slots), scale=scale)
    lse = torch.empty(q.shape[:3], device="cuda")
    cache.attend(0, q, lse=lse, **given)
    o = Steps.of(cache)
    start = np.zeros((cache.sequences, cache.max_pages * cache.page_tokens)) if weights is None else weights.cpu().double().numpy()
    got = cache.weigh(0, q, lse, weights, **given, **kw)
    assert faults_of(cache) == 0
    want, allowed = o.weigh(0, q, lse.cpu().numpy(), start, mask, counts, slots, scale)
    got64 = got.cpu().double().numpy()
    assert (np.abs(got64 - want) <= allowed + 1e-30).all()
    assert np.array_equal(got64[want == start], start[want == start])
    return got, lse


@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("shape", WEIGHED, ids=str)
def test_weights(shape, masked):
    dtype, lengths, counts, kv_heads, group, head_dim, page_tokens = shape
    cache, q = filled(lengths, counts, dtype=dtype, kv_heads=kv_heads, group=group, head_dim=head_dim, page_tokens=page_tokens)
    mask = np.stack([tree(random.Random(b), q.shape[1]) for b in range(len(lengths))]) if masked else None
    width = cache.max_pages * page_tokens
    start = torch.rand(len(lengths), width, device="cuda")
    got, lse = weigh(cache, q, mask, counts, weights=start)
    # a row's weights are 1 together
    total = (got - start).sum(1).cpu().double().numpy()
    assert np.allclose(total, [c * kv_heads * group for c in counts], rtol=1e-3, atol=1e-3 * width * 2.0**-12)
    again, _ = weigh(cache, q, mask, counts, weights=start)
    assert torch.equal(got, again)
    fresh, _ = weigh(cache, q, mask, counts)
    in_place = start.clone()
    given = dict(mask=None if mask is None else torch.from_numpy(mask).cuda(), counts=ints(counts))
    assert cache.weigh(0, q, lse, in_place, out=in_place, **given) is in_place and torch.equal(in_place, got)
    wide = torch.full((len(lengths), width + 3), 9.0, device="cuda")
    cache.weigh(0, q, lse, None, out=wide[:, 1:1 + width], **given)
    assert torch.equal(wide[:, 1:1 + width], fresh) and (wide[:, 0] == 9).all() and (wide[:, -2:] == 9).all()
    apart = torch.zeros(len(lengths), 2 * width, device="cuda")
    cache.weigh(0, q, lse, None, out=apart[:, ::2], **given)
    assert torch.equal(apart[:, ::2], fresh) and (apart[:, 1::2] == 0).all()


@pytest.mark.parametrize("dtype, head_dim, group, tokens, page_tokens", [(BF16, 128, 4, 200, 64), (F16, 64, 2, 130, 8), (F32, 64, 2, 90, 16), (BF16, 256, 1, 150, 32), (F32, 128, 8, 33, 16)])
@pytest.mark.parametrize("masked", [False, True])
def test_weights_of_pieces_of_prompts(dtype, head_dim, group, tokens, page_tokens, masked):
    """Hundreds of rows to a key head, and masks of more than 64 tokens; the same when they have been accepted."""
    counts = [tokens, tokens // 2, 1]
    cache, q = filled([500, 0, 70], counts, dtype=dtype, kv_heads=1, group=group, head_dim=head_dim, page_tokens=page_tokens)
    mask = np.random.default_rng(tokens).random((3, tokens, tokens)) < 0.3 if masked else None
    got, lse = weigh(cache, q, mask, counts)
    cache.accept(ints(counts))
    given = dict(mask=None if mask is None else torch.from_numpy(mask).cuda(), counts=ints(counts))
    assert torch.equal(cache.weigh(0, q, lse, committed=True, **given), got) and faults_of(cache) == 0


@pytest.mark.parametrize("dtype, group, tokens", [(BF16, 1, 2), (F16, 4, 5), (F32, 2, 1)])
def test_weights_of_hundreds_of_sequences(dtype, group, tokens):
    """More than a CTA has threads; by their own numbers, and in any order."""
    dice = random.Random(tokens)
    lengths = [dice.choice([1, dice.randint(1, 60)]) for _ in range(600)]
    counts = [dice.choice([0, tokens, tokens]) for _ in range(600)]
    cache, q = filled(lengths, counts, dtype=dtype, kv_heads=1, group=group, head_dim=64, page_tokens=8)
    start = torch.rand(600, cache.max_pages * 8, device="cuda")
    got, lse = weigh(cache, q, None, counts, weights=start)
    order = list(range(600))
    dice.shuffle(order)
    assert torch.equal(cache.weigh(0, q[order], lse[order], start, counts=ints([counts[s] for s in order]), slots=ints(order)), got) and faults_of(cache) == 0


@pytest.mark.parametrize("dtype", [BF16, F16, F32])
def test_weights_of_rows_that_name_their_sequences(dtype):
    cache, q = filled([100, 5, 300, 41], [3, 3, 3, 3], dtype=dtype, kv_heads=2, group=2, head_dim=64)
    q = q[:3]
    got, lse = weigh(cache, q, None, [3, 1, 2], [3, 0, 2], weights=torch.rand(4, cache.max_pages * 16, device="cuda"))
    start = torch.rand(4, cache.max_pages * 16, device="cuda")
    one = cache.weigh(0, q[:1], lse[:1], start, slots=ints([2]))
    assert faults_of(cache) == 0
    two = cache.weigh(0, q, lse, start, slots=ints([2, 2, 7]))             # a sequence twice, and one that there is not
    assert faults_of(cache) == BAD_INDEX and torch.equal(one, two)
    wide = q.repeat(1, 1, 1, 2)[..., :64]                                  # strides, and queries of float32
    assert torch.equal(cache.weigh(0, wide, lse.transpose(1, 2).contiguous().transpose(1, 2), start, counts=ints([3, 1, 2])),
                       cache.weigh(0, q.to(dtype), lse, start, counts=ints([3, 1, 2])))


@pytest.mark.parametrize("dtype, tokens", [(BF16, 3), (F32, 3), (F16, 20)])
def test_weights_of_committed_tokens(dtype, tokens):
    """As of the same tokens before they were accepted."""
    cache, q = filled([100, 5, 0], [tokens] * 3, dtype=dtype, kv_heads=2, group=2, head_dim=64)
    lse, counts = torch.empty(3, tokens, 4, device="cuda"), ints([tokens, 1, tokens - 1])
    cache.attend(0, q, counts=counts, lse=lse)
    want = cache.weigh(0, q, lse, counts=counts)
    cache.accept(counts)
    assert torch.equal(cache.weigh(0, q, lse, counts=counts, committed=True), want) and faults_of(cache) == 0
    cache.truncate(ints([-1, 2, 0]))
    got = cache.weigh(0, q, lse, counts=ints([tokens, 3, 1]), committed=True)              # more tokens than there are
    assert faults_of(cache) == BAD_INDEX and torch.equal(got[0], want[0]) and got[2].count_nonzero() == 0 and got[1, 2:].count_nonzero() == 0


@pytest.mark.parametrize("dtype, head_dim", [(BF16, 64), (F32, 64), (F16, 128), (F32, 256), (BF16, 256)])
def test_weights_beside_rows_and_keys_that_are_no_numbers(dtype, head_dim):
    cache, q = filled([100], [4], dtype=dtype, kv_heads=2, group=2, head_dim=head_dim)
    lse = torch.empty(1, 4, 4, device="cuda")
    cache.attend(0, q, lse=lse)
    want = cache.weigh(0, q, lse)
    lse[0, 1], q[0, 1] = -float("inf"), float("nan")                       # a row that saw nothing adds nothing
    some = cache.weigh(0, q, lse)
    assert torch.isfinite(some).all() and (some <= want).all() and (some[0, :100].sum() < want[0, :100].sum())
    cache.pool[0, 0, cache.table[0, 2].long(), :, 5] = float("nan")
    got = cache.weigh(0, q, lse)
    assert torch.isnan(got[0, 37]) and torch.equal(torch.cat([got[0, :37], got[0, 38:]]), torch.cat([some[0, :37], some[0, 38:]]))
    keep = cache.evict(got, ints([1]))                                     # (NaN is heaviest)
    assert torch.isnan(keep[0, 0]) and keep[0, 1:].count_nonzero() == 0 and cache.lengths.tolist() == [1]
    assert faults_of(cache) == 0


@pytest.mark.parametrize("dtype, head_dim, tokens, group", [(BF16, 64, 1, 1), (F16, 128, 3, 2), (BF16, 256, 4, 2), (F16, 80, 16, 1), (BF16, 128, 17, 1), (F32, 64, 1, 1), (F32, 128, 5, 3)])
@pytest.mark.parametrize("bad", [float("inf"), -float("inf")])
def test_weights_of_a_key_that_holds_an_infinity(dtype, head_dim, tokens, group, bad):
    """Which leaves real rows a score of -inf, a weight of 0 exactly, as a score of -10000 does; beside rows that are not there, and one that saw nothing."""
    cache, q = filled([100, 30], [tokens, 1], dtype=dtype, kv_heads=2, group=group, head_dim=head_dim)
    page, counts = cache.table[0, 2].long(), ints([tokens, 1])
    size = 20000.0 * head_dim**0.5
    q[0, :, :group, 3] = -1.0 if bad > 0 else 1.0
    got = []
    for value in (bad, size if bad > 0 else -size):
        cache.pool[0, 0, page, 0, 5, 3] = value                            # (key 37, of one of the two key heads)
        lse = torch.empty(2, tokens, 2 * group, device="cuda")
        assert torch.isfinite(cache.attend(0, q, counts=counts, lse=lse)).all() and torch.isfinite(lse[0]).all()
        got.append(cache.weigh(0, q, lse, counts=counts))
        lse[0, 0], lse[1, 0, 0] = -float("inf"), -float("inf")
        got.append(cache.weigh(0, q, lse, counts=counts))
    assert torch.equal(got[0], got[2]) and torch.equal(got[1], got[3])
    assert torch.isfinite(torch.stack(got)).all() and faults_of(cache) == 0


@pytest.mark.parametrize("dtype, tokens", [(BF16, 3), (F16, 16), (BF16, 20), (F32, 3)])
def test_a_row_whose_lse_is_no_number_reaches_only_what_it_sees(dtype, tokens):
    cache, q = filled([90], [tokens], dtype=dtype, kv_heads=2, head_dim=64)
    lse = torch.empty(1, tokens, 2, device="cuda")
    cache.attend(0, q, lse=lse)
    rest = lse.clone()
    lse[0, 1], rest[0, 1] = float("nan"), -float("inf")
    got, want = cache.weigh(0, q, lse), cache.weigh(0, q, rest)
    assert torch.isnan(got[0, :92]).all() and torch.equal(got[0, 92:], want[0, 92:]) and faults_of(cache) == 0


@pytest.mark.parametrize("dtype, tokens, group, page_tokens", [(BF16, 1, 1, 8), (F16, 4, 4, 16), (BF16, 12, 1, 64), (BF16, 20, 2, 8), (F16, 9, 4, 32), (F32, 1, 1, 8), (F32, 6, 2, 64)])
@pytest.mark.parametrize("in_place", [False, True])
def test_keys_without_a_page_draw_nothing(dtype, tokens, group, page_tokens, in_place):
    """Whatever the pool's pages hold, and as many rows as there are: what is left of the weights is what they would have been."""
    cache, q = filled([700, 33], [tokens, 1], dtype=dtype, kv_heads=2, group=group, head_dim=64, page_tokens=page_tokens)
    lse, counts = torch.empty(2, tokens, 2 * group, device="cuda"), ints([tokens, 1])
    cache.attend(0, q, counts=counts, lse=lse)
    start = torch.rand(2, cache.max_pages * page_tokens, device="cuda")
    want = cache.weigh(0, q, lse, start, counts=counts)
    assert faults_of(cache) == 0
    cache.release(100, 20)
    lost = torch.zeros_like(want, dtype=torch.bool)
    lost[0, :cache.table.shape[1] * page_tokens] = (cache.table[0] < 0).repeat_interleave(page_tokens) & (torch.arange(want.shape[1], device="cuda") < 700)
    assert 400 < lost.sum().item() < 600
    got = cache.weigh(0, q, lse, start, counts=counts, out=start.clone() if in_place else None)
    assert faults_of(cache) == BAD_INDEX
    assert torch.equal(got, torch.where(lost, start, want))


def test_no_rows_and_no_tokens():
    cache, q = filled([30, 20], [2, 2], dtype=BF16, kv_heads=1, head_dim=64)
    start = torch.rand(2, cache.max_pages * 16, device="cuda")
    lse = torch.zeros(2, 2, 1, device="cuda")
    assert torch.equal(cache.weigh(0, q[:0], lse[:0], start), start) and torch.equal(cache.weigh(0, q[:, :0], lse[:, :0], start), start)
    assert torch.equal(cache.weigh(0, q, lse, start, counts=ints([0, 0])), start) and cache.weigh(0, q[:0], lse[:0]).count_nonzero() == 0
    assert cache.attend(0, q[:0], window=3, lse=lse[:0]).numel() == 0
    assert faults_of(cache) == 0


# ---- large, refused, captured --------------------------------------------------------------------

def test_offsets_beyond_32_bits():
    """Pages whose elements, and whose bytes, are past 2^32 of the pool's start."""
    small, q = filled([300], [4], dtype=BF16, kv_heads=2, head_dim=128, page_tokens=64, layers=1)
    q = q.to(BF16)
    large = make(sequences=1, max_pages=small.max_pages, pages=160000, kv_heads=2, head_dim=128, page_tokens=64, layers=1, fill=0.0)       # 10 GB
    pages = small.table[0, :5].long()
    large.pool[:, :, 159990:159995] = small.pool[:, :, pages]
    large.table[0, :5] = torch.arange(159990, 159995, device="cuda")
    large.refs[159990:159995] = 1
    for c in (large, small):
        c.held.fill_(5)
        c.lengths.fill_(300)
    lse = [torch.empty(1, 4, 2, device="cuda") for _ in range(2)]
    assert torch.equal(*(c.attend(0, q, window=70, sinks=3, lse=x) for c, x in zip((small, large), lse))) and torch.equal(*lse)
    weights = [c.weigh(0, q, x) for c, x in zip((small, large), lse)]
    assert torch.equal(*weights) and weights[0].count_nonzero() > 0
    assert torch.equal(*(c.evict(w, ints([150]), recent=20) for c, w in zip((small, large), weights)))
    at = torch.arange(150, device="cuda")
    rows = [c.pool[:, :, c.table[0, at // 64].long(), :, at % 64] for c in (small, large)]
    assert torch.equal(*rows) and large.table[0, :4].tolist() == [159990, 159991, 159992, -1]
    small.release(30)
    large.release(30)
    assert large.table[0, :3].tolist() == [-1, 159991, 159992] and faults_of(small) == faults_of(large) == 0


def test_arguments_that_are_refused():
    cache = make(sequences=2, pages=8, kv_heads=2, layers=2, max_pages=3)
    q, lse, weights = torch.zeros(2, 3, 2, 64, device="cuda"), torch.zeros(2, 3, 2, device="cuda"), torch.zeros(2, 48, device="cuda")
    two, places = ints([0, 0]), ints([[0, 1, 2]] * 2)
    for call, error in [
            (lambda: cache.attend(0, q, window=0), ValueError), (lambda: cache.attend(0, q, window=-1), ValueError), (lambda: cache.attend(0, q, window=2.0), ValueError),
            (lambda: cache.attend(0, q, window=2**31), ValueError), (lambda: cache.attend(0, q, window=True), ValueError), (lambda: cache.attend(0, q, window=4, sinks=-1), ValueError),
            (lambda: cache.attend(0, q, sinks=4), ValueError), (lambda: cache.attend(0, q, places=places), ValueError), (lambda: cache.attend(0, q, window=4, sinks=None), ValueError),
            (lambda: cache.attend(0, q, window=4, places=places[:1]), ValueError), (lambda: cache.attend(0, q, window=4, places=places.float()), TypeError),
            (lambda: cache.attend(0, q, window=4, places=places.cpu()), ValueError), (lambda: cache.attend(0, q, lse=lse[:1]), ValueError),
            (lambda: cache.attend(0, q, lse=lse.double()), TypeError), (lambda: cache.attend(0, q, lse=lse.cpu()), ValueError), (lambda: cache.attend(0, q, lse=1), TypeError),
            (lambda: cache.attend(0, q, lse=lse[:, :1].expand(2, 3, 2)), ValueError), (lambda: cache.attend(0, q, lse=lse.clone().requires_grad_()), ValueError),
            (lambda: cache.attend(0, q, lse=q[..., 0]), ValueError),
            (lambda: cache.release(0), ValueError), (lambda: cache.release(4, -1), ValueError), (lambda: cache.release(two), ValueError), (lambda: cache.release(None), ValueError),
            (lambda: cache.weigh(2, q, lse), ValueError), (lambda: cache.weigh(0, q, None), TypeError), (lambda: cache.weigh(0, q, lse[..., :1]), ValueError),
            (lambda: cache.weigh(0, q.half(), lse), TypeError), (lambda: cache.weigh(0, q, lse, weights[:, :40]), ValueError), (lambda: cache.weigh(0, q, lse, weights.half()), TypeError),
            (lambda: cache.weigh(0, q, lse, weights[:1]), ValueError), (lambda: cache.weigh(0, q, lse, weights.cpu()), ValueError), (lambda: cache.weigh(0, q, lse, out=weights[:, :2]), ValueError),
            (lambda: cache.weigh(0, q, lse, out=weights[:1].expand(2, 48)), ValueError), (lambda: cache.weigh(0, q, lse, out=weights.clone().requires_grad_()), ValueError),
            (lambda: cache.weigh(0, q, lse, scale=0.0), ValueError), (lambda: cache.weigh(0, q, lse, slots=ints([0, 1, 2])), ValueError),
            (lambda: cache.weigh(0, q, lse, mask=torch.ones(2, 2, dtype=torch.bool, device="cuda")), ValueError),
            (lambda: cache.weigh(0, q, lse, torch.zeros(3, 48, device="cuda")[:2], out=torch.zeros(2, 48, dtype=torch.float64, device="cuda")), TypeError),
            (lambda: cache.evict(None, two), TypeError), (lambda: cache.evict(weights, two[:1]), ValueError), (lambda: cache.evict(weights, two.float()), TypeError),
            (lambda: cache.evict(weights, two, recent=-1), ValueError), (lambda: cache.evict(weights, two, sinks=1.5), ValueError), (lambda: cache.evict(weights[:, 1:], two), ValueError),
            (lambda: cache.evict(weights, two, out=weights[:1].expand(2, 48)), ValueError), (lambda: cache.evict(weights.double(), two), TypeError),
            (lambda: cache.evict(weights.expand(2, 48), [0, 0]), TypeError)]:
        with pytest.raises(error):
            call()
    long = torch.zeros(3, 48, device="cuda").view(-1)
    with pytest.raises(ValueError, match="part"):
        cache.evict(long[:96].view(2, 48), two, out=long[48:].view(2, 48))
    wide = torch.zeros(2, 100, device="cuda")
    with pytest.raises(ValueError, match="part"):
        cache.evict(wide[:, :48], two, out=wide[:, 40:88])
    cache.evict(wide[:, :48], two, out=wide[:, 50:98])      # (side by side)
    assert faults_of(cache) == 0 and cache.lengths.tolist() == [0, 0]
    cache.close()
    for call in (lambda: cache.release(1), lambda: cache.weigh(0, q, lse), lambda: cache.evict(weights, two)):
        with pytest.raises(ValueError):
            call()


def test_c_entries_refuse():
    cache, q = filled([3000], [2], dtype=BF16, kv_heads=2, head_dim=64)
    q = q.to(BF16)
    lib, handle = _cabi.load(), cache._cache
    rows, out = _cabi.Rows(q.data_ptr(), 1, 2, q.stride()[:3]), torch.empty_like(q)
    to = _cabi.Rows(out.data_ptr(), 1, 2, out.stride()[:3])
    lse, stride = torch.empty(1, 2, 2, device="cuda"), (C.c_int64 * 3)(4, 2, 1)
    n = lib.kb200_cache_attend_window_workspace(handle, 1, 2, 2, 1000, 4)
    space = torch.empty(max(n, lib.kb200_cache_evict_workspace(handle)) + 16, dtype=torch.uint8, device="cuda")

    def attend(window=1000, sinks=4, at=space.data_ptr(), size=n, lse_at=lse.data_ptr(), strides=stride):
        return lib.kb200_cache_attend_window(handle, 0, C.byref(rows), C.byref(to), 1, 2, None, None, None, None, 0.125, window, sinks, None, lse_at, strides, at, size, None)

    assert n > 0 and attend() == 0 and attend(lse_at=None, strides=None) == 0
    assert attend(window=-1) == attend(sinks=-1) == attend(strides=None) == attend(size=n - 1) == attend(at=None) == attend(at=space.data_ptr() + 8) == -1
    assert lib.kb200_cache_attend_window_workspace(handle, 1, 2, 2, -1, 0) == 0
    width = cache.max_pages * cache.page_tokens
    weights, keep = torch.rand(1, width, device="cuda"), ints([10])
    size = lib.kb200_cache_evict_workspace(handle)
    evict = lambda *a: lib.kb200_cache_evict(handle, *a, None)  # noqa: E731
    at = (weights.data_ptr(), width, keep.data_ptr(), 0, 0, weights.data_ptr(), width)
    for i, value in ((0, None), (2, None), (3, -1), (4, -1), (5, None)):
        assert evict(*[value if j == i else x for j, x in enumerate(at)], space.data_ptr(), size) == -1
    assert evict(*at, space.data_ptr(), size - 1) == evict(*at, None, size) == evict(*at, space.data_ptr() + 8, size) == -1
    weigh = lambda q_=rows, lse_=lse.data_ptr(), strides=stride, to_=weights.data_ptr(), layer=0, scale=0.125: lib.kb200_cache_weigh(  # noqa: E731
        handle, layer, C.byref(q_), lse_, strides, 1, 2, None, None, None, None, scale, 0, None, 0, to_, width, None)
    assert weigh() == 0 and weigh(lse_=None) == weigh(strides=None) == weigh(to_=None) == weigh(layer=1) == weigh(scale=-1.0) == -1
    assert weigh(_cabi.Rows(q.data_ptr(), 1, 3, q.stride()[:3])) == weigh(_cabi.Rows(q.data_ptr() + 2, 1, 2, q.stride()[:3])) == weigh(_cabi.Rows(q.data_ptr(), 1, 2, (256, 128, 4))) == -1
    assert lib.kb200_cache_release(handle, 0, 0, None) == lib.kb200_cache_release(handle, 1, -1, None) == -1
    torch.cuda.synchronize()
    assert faults_of(cache) == 0 and cache.lengths.tolist() == [3000]


@pytest.mark.parametrize("sequences", [3, 90])
def test_a_captured_step_follows_the_tables(sequences):
    """Attention to a window and its lse, weights, evictions and released pages in one graph; two graphs take turns."""
    sizes = dict(sequences=sequences, max_pages=12, pages=12 * sequences, kv_heads=2, head_dim=64, dtype=BF16, layers=2, fill=0.0)
    cache, eager = make(**sizes), make(**sizes)
    tokens, width = 4, 12 * 16
    x = torch.zeros(3, 2, sequences, tokens, 2, 64, device="cuda")
    counts, keep = ints([4, 3, 1] * (sequences // 3)), ints([-1, 30, -1] * (sequences // 3))
    weights = [torch.zeros(sequences, width, device="cuda") for _ in range(2)]

    def step(c, data, weights):
        c.reserve(counts)
        outs = []
        for layer in range(2):
            c.append(layer, data[1, layer], data[2, layer], counts)
            lse = torch.empty(sequences, tokens, 2, device="cuda")
            outs += [c.attend(layer, data[0, layer], counts=counts, window=24, sinks=2, lse=lse), lse]
        lse = torch.empty(sequences, tokens, 2, device="cuda")
        c.attend(1, data[0, 1], counts=counts, lse=lse)
        c.weigh(1, data[0, 1], lse, weights, counts=counts, out=weights)
        c.accept(counts)
        outs += [c.evict(weights, keep, recent=8, sinks=2, out=weights).clone()]
        return outs

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, x, weights[0])
        cache.truncate(torch.zeros_like(counts))
        weights[0].zero_()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(cache, x, weights[0]))
        graphs.append(graph)
    assert cache.lengths.tolist() == [0] * sequences
    generator = torch.Generator("cuda").manual_seed(4)
    for i in range(20):
        x.copy_(torch.randn(x.shape, generator=generator, device="cuda"))
        graphs[i % 2].replay()
        for got, w in zip(outs[i % 2], step(eager, x, weights[1])):
            assert torch.equal(got, w)
    assert cache.lengths.tolist() == eager.lengths.tolist() and cache.lengths.tolist()[:3] == [80, 30, 20]
    assert torch.equal(cache.table, eager.table) and torch.equal(cache.refs, eager.refs)
    assert faults_of(cache) == faults_of(eager) == 0


def test_two_streams_at_once():
    cache, q = filled([3000, 40, 700], [2, 2, 2], dtype=BF16, kv_heads=2, head_dim=64)
    q = q.to(BF16)

    def both(x):
        lse = torch.empty(3, 2, 2, device="cuda")
        out = cache.attend(0, x, window=500, sinks=4, lse=lse)
        return out, lse, cache.weigh(0, x, lse)

    plain = [both(q), both(-q)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(both(q if i == 0 else -q))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for i in range(2) for x in outs[i] for a, b in zip(x, plain[i]))


def test_many_calls_leave_the_allocator_as_it_was():
    cache, q = filled([300], [2], dtype=BF16, kv_heads=2, head_dim=64)
    q, lse = q.to(BF16), torch.empty(1, 2, 2, device="cuda")
    weights = torch.zeros(1, cache.max_pages * 16, device="cuda")

    def all_of_them():
        cache.attend(0, q, window=50, lse=lse, out=q)
        cache.weigh(0, q, lse, weights, out=weights)
        cache.evict(weights, ints([-1]), out=weights)
        cache.release(5000)

    all_of_them()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(50):
        all_of_them()
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before

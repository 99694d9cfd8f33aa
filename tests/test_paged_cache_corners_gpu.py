"""The paged K/V cache on the GPU: calls at the corners of what its interface allows."""

import ctypes as C

import numpy as np
import pytest
import torch

from kiln_b200 import _cabi
from oracle.cache_oracle import BAD_INDEX, NO_PAGES, NO_ROOM, SHARED, Oracle
from test_paged_cache_gpu import BF16, F16, F32, check, faults_of, filled, ints, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("length", [10, 300])                         # (items whole and cut)
@pytest.mark.parametrize("few_first", [True, False])
@pytest.mark.parametrize("dtype, tokens, rows, kv_heads", [(BF16, 20, 40, 8), (F16, 9, 80, 8), (F32, 20, 40, 8), (BF16, 48, 60, 4), (F16, 90, 60, 4)])
def test_neighbouring_rows_of_one_sequence_that_end_apart(dtype, tokens, rows, kv_heads, few_first, length):
    """More items than CTAs, so that runs go from one row to the next.  Rows of one token see nothing of the pages behind theirs, whatever those hold."""
    cache, _ = filled([length], [tokens], dtype=dtype, kv_heads=kv_heads, head_dim=64, page_tokens=8 if tokens < 16 else 16)
    q = torch.randn(rows, tokens, kv_heads, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(5)).to(dtype)
    counts = ([1, tokens] if few_first else [tokens, 1]) * (rows // 2)
    clean = check(cache, q, None, counts, [0] * rows)
    behind = cache.table[0, -(-(length + 1) // cache.page_tokens):cache.held[0].item()].long()
    cache.pool[:, :, behind] = float("nan")
    again = cache.attend(0, q, counts=ints(counts), slots=ints([0] * rows))
    few = torch.tensor(counts, device="cuda") == 1
    assert behind.numel() > 0 and torch.equal(clean[few], again[few])


@pytest.mark.parametrize("head_dim", [64, 128, 256])
@pytest.mark.parametrize("length, tokens, group", [(100, 1, 1), (100, 1, 4), (100, 9, 1), (3000, 1, 2), (3000, 12, 1), (700, 33, 1)])
def test_float32_scores_far_from_zero_that_lie_close_together(length, tokens, group, head_dim):
    """Queries of ones and keys of whole numbers: every score is exact in float32 in any order of its sum, 8000 and more after the scale, and a few apart.

    What is left: the scale times log2 e is off by three roundings at most (2^-22), and so is an exponent of at most 5 / ln 2 = 7.3 by 7.3 x 2^-22 and its own
    rounding of 2^-22, a weight by ln 2 times that, 2^-20 with the 2^-22 of the exponential; once for itself and once for their sum.  Rescaling adds as much again; the
    sums add (N / 8 + 64) 2^-23."""
    cache, _ = filled([length], [tokens], dtype=F32, kv_heads=2, head_dim=head_dim)
    generator = torch.Generator("cuda").manual_seed(6)
    keys = torch.full(cache.pool[0, 0].shape, 1000.0, device="cuda")
    keys[..., 0] += torch.randint(0, int(5 * head_dim ** 0.5), keys.shape[:-1], device="cuda", generator=generator)
    cache.pool[0, 0] = keys
    got = cache.attend(0, torch.ones(1, tokens, 2 * group, head_dim, device="cuda"))
    want, weight, _ = Oracle.of(cache).attend(0, torch.ones(1, tokens, 2 * group, head_dim))
    allowed = weight * (4 * 2.0**-20 + ((length + tokens) / 8 + 64) * 2.0**-23)
    assert (np.abs(got.cpu().double().numpy() - want) <= allowed).all()


@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("dtype, tokens, head_dim", [(BF16, 1, 64), (F16, 1, 64), (BF16, 40, 128), (F16, 40, 64), (BF16, 90, 64), (F32, 3, 64), (BF16, 3, 160)])
def test_scores_beyond_float32_steps_of_one(dtype, tokens, head_dim, sign):
    """Scores of 2^28 to 2^36, exact and far apart: every row is the value of its largest key, to the bit."""
    cache, _ = filled([500], [tokens], dtype=dtype, kv_heads=2, head_dim=head_dim)
    dice = np.random.default_rng(3)
    ones = torch.from_numpy(dice.choice([1.0, 3.0], head_dim)).cuda()
    low, high = (2.0**6, 2.0**13) if dtype == F16 else (2.0**16, 2.0**18)
    at = torch.arange(500 + tokens, device="cuda")
    pages, rows = cache.table[0, at // 16].long(), at % 16
    want = []
    for head in range(2):
        sizes, top = dice.integers(2, 60, 500 + tokens), int(dice.integers(0, 500))
        sizes[top] = 64 if sign > 0 else 1
        cache.pool[0, 0, pages, head, rows] = (torch.from_numpy(sizes).cuda()[:, None] * low * ones).to(dtype)
        want.append(cache.pool[0, 1, pages[top], head, rows[top]])
    q = (sign * high * ones).expand(1, tokens, 2, head_dim).to(dtype)
    assert torch.equal(cache.attend(0, q), torch.stack(want).expand(1, tokens, 2, head_dim))


@pytest.mark.parametrize("gap", [9, 12, 15, 17])
@pytest.mark.parametrize("dtype, tokens, head_dim", [(F16, 1, 64), (F16, 40, 128), (F16, 90, 64), (F16, 3, 160), (BF16, 1, 64)])
def test_a_first_token_that_draws_nearly_all_of_the_weight(dtype, tokens, head_dim, gap):
    """Its V is zero, so that the result is the other tokens', whose weights are e^-gap of its: off by half a step of the type as any (`check`)."""
    cache, q = filled([3000], [tokens], dtype=dtype, kv_heads=2, head_dim=head_dim)
    page = cache.table[0, 0].item()
    q = (q * 0.1).to(dtype)
    q[..., 0] = 8.0
    cache.pool[0, 0, :, :, :, 0] = 0.0
    cache.pool[0, 1] = cache.pool[0, 1].abs()
    cache.pool[0, 0, page, :, 0, 0] = gap * head_dim**0.5 / 8
    cache.pool[0, 1, page, :, 0] = 0.0
    check(cache, q)


def test_a_reservation_of_two_to_the_31_pages_is_refused():
    """Every sequence asks for all of its table: 2^31 pages where there are eight."""
    cache = make(sequences=1 << 15, max_pages=1 << 16, pages=8, head_dim=16, page_tokens=8, fill=0.0)         # 8.6 GB of table, as much of scratch
    cache.reserve(torch.full((1 << 15,), 1 << 19, dtype=torch.int32, device="cuda"))
    assert faults_of(cache) == NO_PAGES
    assert cache.refs.tolist() == [0] * 8 and cache.held.max().item() == 0 and cache.table.max().item() == -1
    few = torch.zeros(1 << 15, dtype=torch.int32, device="cuda")
    few[5], few[30000] = 20, 40
    cache.reserve(few)
    assert faults_of(cache) == 0 and cache.table[5, :4].tolist() == [0, 1, 2, -1] and cache.table[30000, :6].tolist() == [3, 4, 5, 6, 7, -1]
    cache.close()
    del cache
    torch.cuda.empty_cache()


@pytest.mark.parametrize("n, dtype, head_dim", [((1 << 20) + 40, BF16, 16), ((1 << 25) + 8, F32, 256)])
def test_accepting_millions_of_tokens(n, dtype, head_dim):
    """The last few of a prompt move; their bytes, 16 at a time, are 2^31 and more in the second case (K and V of 64 GB)."""
    cache = make(layers=1, max_pages=n // 256 + 2, pages=n // 256 + 2, head_dim=head_dim, page_tokens=256, dtype=dtype, fill=0.0)
    cache.reserve(ints([n + 3]))
    at = torch.arange(n - 10, n + 3, device="cuda")
    pages, rows = cache.table[0, at // 256].long(), at % 256
    assert faults_of(cache) == 0 and pages.min().item() >= 0
    cache.pool[0, :, pages, 0, rows] = torch.arange(1.0, 14.0, device="cuda")[None, :, None].expand(2, 13, head_dim).to(dtype)
    kept = torch.arange(n, dtype=torch.int32, device="cuda")
    kept[-4:] += 3
    cache.accept(ints([n]), kept[None])
    got = cache.pool[0, :, pages[:10], 0, rows[:10]]
    assert faults_of(cache) == 0 and cache.lengths.tolist() == [n]
    want = torch.tensor([1.0, 2, 3, 4, 5, 6, 10, 11, 12, 13], device="cuda")[None, :, None].expand(2, 10, head_dim)
    assert torch.equal(got.float(), want)
    cache.close()
    del cache, kept
    torch.cuda.empty_cache()


def test_what_calls_on_other_streams_left_out_is_told_once():
    cache = make(sequences=2, pages=4, fill=0.0)
    side, wrong, many, fine = torch.cuda.Stream(), ints([5, 0]), ints([128, 0]), ints([0, 0])
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        for _ in range(300):
            cache.fork(wrong)
            assert faults_of(cache) == BAD_INDEX
            cache.reserve(many)
            assert faults_of(cache) == NO_PAGES
            cache.reserve(fine)
            assert faults_of(cache) == 0


def test_outputs_that_share_memory_are_refused():
    cache, q = filled([20, 30], [3, 3], dtype=BF16, kv_heads=2, head_dim=64)
    one = torch.full((1, 3, 2, 64), 7.0, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="share memory"):
        cache.attend(0, q, out=one.expand(2, 3, 2, 64))
    three = torch.full((3, 3, 2, 64), 7.0, dtype=BF16, device="cuda")
    with pytest.raises(ValueError, match="part of q"):
        cache.attend(0, three[:2], out=three[1:])
    assert (one == 7).all() and (three == 7).all()
    cache.attend(0, three[:2], out=three[:2])                          # the same
    fused = torch.zeros(2, 3, 6, 64, dtype=BF16, device="cuda")
    fused[:, :, :2] = q
    cache.attend(0, fused[:, :, :2], out=fused[:, :, 4:])              # beside each other
    assert torch.equal(fused[:, :, 4:], cache.attend(0, q)) and (fused[:, :, 2:4] == 0).all() and (three[2] == 7).all()


def test_inference_mode():
    """Calls inside it are as any; a tensor from there is not written to outside of it."""
    cache, q = filled([20, 30], [3, 3], dtype=BF16, kv_heads=2, head_dim=64)
    plain = cache.attend(0, q)
    with torch.inference_mode():
        out = torch.full((2, 3, 2, 64), 7.0, dtype=BF16, device="cuda")
        assert torch.equal(cache.attend(0, q), plain) and torch.equal(cache.attend(0, q, out=out.clone()), plain)
    with pytest.raises(RuntimeError, match="InferenceMode"):
        cache.attend(0, q, out=out)
    assert (out == 7).all()
    mine = torch.zeros(2, 3, 2, 64, dtype=BF16, device="cuda")
    before = mine._version
    cache.attend(0, q, out=mine)
    assert torch.equal(mine, plain) and mine._version == before + 1


def test_attention_tells_exactly_what_it_left_out():
    cache, _ = filled([8, 8, 8], [1, 1, 1], dtype=BF16, kv_heads=1, head_dim=64)
    q = torch.randn(3, 1, 1, 64, device="cuda")
    plain = cache.attend(0, q)
    assert faults_of(cache) == 0
    for slots in ([0, 7, 2], [0, -1, 2], [0, 2**31 - 1, 2]):
        out = cache.attend(0, q, slots=ints(slots))
        assert faults_of(cache) == BAD_INDEX and (out[1] == 0).all() and torch.equal(out[::2], plain[::2])
    for counts in ([1, -1, 1], [1, 2, 1]):
        cache.attend(0, q, counts=ints(counts))
        assert faults_of(cache) == BAD_INDEX
    cache.lengths[1] = 16                                              # a page's end
    cache.attend(0, q)
    assert faults_of(cache) == NO_ROOM
    cache.lengths[1] = 8
    cache.table[0, 0] = 10**6
    cache.attend(0, q[:1])
    assert faults_of(cache) == BAD_INDEX
    cache.fork(ints([0, 0, 2]))
    cache.truncate(ints([4, 4, 4]))
    cache.compact()
    assert faults_of(cache) == 0


@pytest.mark.parametrize("dtype, head_dim, page_tokens", [(F32, 64, 256), (BF16, 64, 16), (F16, 128, 256), (F32, 256, 256), (BF16, 256, 128)])
def test_prompts_in_pieces_of_hundreds_of_tokens(dtype, head_dim, page_tokens):
    cache, q = filled([0, 33, 5], [700, 513, 1], dtype=dtype, kv_heads=1, head_dim=head_dim, page_tokens=page_tokens)
    check(cache, q.to(dtype), None, [700, 513, 1])


@pytest.mark.parametrize("sequences", [64, 256])
@pytest.mark.parametrize("first", [0, 1])
def test_tokens_in_shared_pages_stay_while_the_other_holder_leaves(sequences, first):
    """Pairs share a page of drafted tokens; one of each accepts a token that would move, the other gives the page back in the same call."""
    cache = make(sequences=sequences, pages=sequences, max_pages=2, fill=0.0)
    one = torch.arange(sequences, device="cuda", dtype=torch.int32) % 2 == first
    cache.reserve(5 * one.int())
    k = torch.randn(sequences, 5, 1, 64, device="cuda")
    cache.append(0, k, k, 5 * one.int())
    both = torch.arange(sequences, device="cuda", dtype=torch.int32) // 2 * 2 + first
    kept = torch.full((sequences, 1), 3, dtype=torch.int32, device="cuda")
    table, pool = cache.table.clone(), cache.pool.clone()
    for _ in range(20):
        cache.fork(both)
        assert faults_of(cache) == 0 and cache.refs.max().item() == 2
        cache.accept(one.int(), kept)
        assert faults_of(cache) == SHARED
        assert cache.lengths.max().item() == 0 and torch.equal(cache.table, table) and torch.equal(cache.pool, pool)
    cache.accept(one.int(), kept)                                      # now they are alone
    assert faults_of(cache) == 0 and torch.equal(cache.lengths, one.int())
    page = cache.table[one, 0].long()
    assert torch.equal(cache.pool[0, 0, page, 0, 0], k[one, 3, 0].to(BF16))


def test_calls_of_more_rows_than_are_counted_are_refused():
    """Nothing is launched for them: tensors of stride 0 would describe such rows in a few bytes."""
    cache = make(sequences=2, pages=4, fill=0.0)
    lib, x = _cabi.load(), torch.zeros(64, dtype=BF16, device="cuda")
    rows = lambda heads: C.byref(_cabi.Rows(x.data_ptr(), 1, heads, (0, 0, 0)))  # noqa: E731
    slots = ints([0, 1]).data_ptr()
    for n in ((1 << 30) + 1, (1 << 31) - 1):
        assert lib.kb200_cache_append(cache._cache, 0, rows(1), rows(1), n, 1, None, slots, None) == -1
        assert lib.kb200_cache_attend(cache._cache, 0, rows(1), rows(1), n, 1, None, None, None, slots, 1.0, None, 0, None) == -1
        assert lib.kb200_cache_attend_workspace(cache._cache, n, 1, 1) == 0
    assert lib.kb200_cache_attend(cache._cache, 0, rows(1), rows(1), 1 << 20, 1025, None, None, None, slots, 1.0, None, 0, None) == -1
    many = make(kv_heads=128, pages=1, fill=0.0)                       # 2^31 chunks to a token
    assert lib.kb200_cache_attend(many._cache, 0, rows(1 << 28), rows(1 << 28), 1, 1, None, None, None, slots, 1.0, None, 0, None) == -1
    assert faults_of(cache) == 0

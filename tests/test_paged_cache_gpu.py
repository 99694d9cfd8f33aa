"""The paged K/V cache on the GPU: its pages against the oracle's lists, bit by bit, and its attention against float64."""

import random

import numpy as np
import pytest
import torch

from kiln_b200 import _cabi
from oracle.cache_oracle import BAD_INDEX, NO_PAGES, NO_ROOM, SHARED, TOO_LONG, Oracle

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def make(fill=float("nan"), **sizes):
    """An empty cache whose pool holds what no result may show."""
    from kiln_b200.cache import PagedCache

    cache = PagedCache(**dict(dict(layers=1, sequences=1, max_pages=8, pages=8, kv_heads=1, head_dim=64, page_tokens=16, dtype=BF16), **sizes))
    cache.pool.fill_(fill)
    return cache


def ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def same(cache, o):
    """The whole state, the pool bit by bit."""
    assert cache.table.tolist() == o.table()
    assert cache.held.tolist() == [len(r) for r in o.rows]
    assert cache.lengths.tolist() == o.lengths and cache.refs.tolist() == o.refs
    assert np.array_equal(cache.pool.cpu().double().numpy(), o.pool, equal_nan=True)


def faults_of(cache):
    """The status, by its text."""
    torch.cuda.synchronize()
    try:
        cache.status()
    except (ValueError, MemoryError) as e:
        assert isinstance(e, MemoryError) == ("free pages" in str(e))
        words = {NO_PAGES: "fewer free pages", TOO_LONG: "max_pages", BAD_INDEX: "out of range", NO_ROOM: "without a page", SHARED: "shared page"}
        return sum(bit for bit, text in words.items() if text in str(e))
    return 0


def tree(dice, n):
    sees = np.zeros((n, n), bool)
    for i in range(n):
        parent = dice.randint(-1, i - 1)
        if parent >= 0:
            sees[i] = sees[parent]
        sees[i, i] = True
    return sees


# ---- pages -------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype, page_tokens, head_dim, sequences, pages", [(BF16, 8, 16, 5, 40), (F32, 16, 48, 3, 17), (F16, 32, 80, 40, 90), (BF16, 64, 128, 2, 9),
                                                                      (BF16, 8, 32, 300, 2500)])
def test_any_operations_leave_what_the_lists_say(dtype, page_tokens, head_dim, sequences, pages):
    dice = random.Random(page_tokens * sequences)
    generator = torch.Generator("cuda").manual_seed(1)
    max_pages = 7
    cache = make(dtype=dtype, page_tokens=page_tokens, head_dim=head_dim, sequences=sequences, pages=pages, max_pages=max_pages, kv_heads=2, layers=2)
    o = Oracle.of(cache)
    seen = 0
    for step in range(40 if sequences < 100 else 12):
        kind = dice.choice(["draft", "draft", "draft", "fork", "fork", "truncate", "compact"])
        if kind == "draft":
            most = min(3 * page_tokens, 100)
            counts = [dice.choice([0, 1, dice.randint(0, most)]) for _ in range(sequences)]
            tokens = max(max(counts), 1)
            cache.reserve(ints(counts))
            o.reserve(counts)
            k, v = (torch.randn(2, sequences, tokens, 2, head_dim, generator=generator, device="cuda") for _ in range(2))
            for layer in range(2):
                cache.append(layer, k[layer], v[layer], ints(counts))
                o.append(layer, k[layer], v[layer], counts)
            n = [dice.choice([0, c, dice.randint(0, c)]) for c in counts]
            kept = [sorted(dice.sample(range(c), m)) + [0] * (tokens - m) for c, m in zip(counts, n)]
            if dice.random() < 0.3:
                cache.accept(ints(n))
                o.accept(n)
            else:
                cache.accept(ints(n), ints(kept))
                o.accept(n, kept)
        elif kind == "fork":
            sources = [dice.choice([-1, s, s, dice.randrange(sequences)]) for s in range(sequences)]
            cache.fork(ints(sources))
            o.fork(sources)
        elif kind == "truncate":
            lengths = [dice.choice([-1, -1, dice.randint(0, max_pages * page_tokens)]) for _ in range(sequences)]
            cache.truncate(ints(lengths))
            o.truncate(lengths)
        else:
            cache.compact()
            o.compact()
        same(cache, o)
        assert faults_of(cache) == o.faults, (step, kind)
        seen |= o.faults
        o.faults = 0
    assert sum(o.lengths) > 0


def test_a_prompt_of_many_pages_and_pages_beyond_one_scan():
    """One sequence of hundreds of pages, a pool of tens of thousands of which every other one is taken."""
    cache = make(sequences=3, max_pages=900, pages=40000, head_dim=16, page_tokens=8, fill=0.0)
    cache.refs[::2] = 1
    o = Oracle.of(cache)
    for counts in ([5000, 0, 1], [0, 2001, 7000]):
        cache.reserve(ints(counts))
        o.reserve(counts)
        assert cache.table.tolist() == o.table() and cache.refs.tolist() == o.refs
    cache.refs[::2] -= 1
    o.refs = cache.refs.tolist()
    cache.compact()
    o.compact()
    assert cache.table.tolist() == o.table() and cache.refs.tolist() == o.refs and faults_of(cache) == 0


def test_a_shared_page_stays_with_the_lowest_holder_only_if_all_write():
    cache = make(sequences=4, pages=12, fill=1.0)
    k = torch.randn(4, 20, 1, 64, device="cuda")
    cache.reserve(ints([20, 0, 0, 0]))
    cache.append(0, k, k, ints([20, 0, 0, 0]))
    cache.accept(ints([20, 0, 0, 0]))
    cache.fork(ints([0, 0, 0, -1]))
    before = cache.table.tolist()
    cache.reserve(ints([0, 1, 1, 0]))          # sequence 0 still holds the page
    after = cache.table.tolist()
    assert after[0] == before[0] and len({after[s][1] for s in range(3)}) == 3
    assert cache.refs[before[0][1]].item() == 1
    cache.fork(ints([0, 0, 0, -1]))
    before = cache.table.tolist()
    cache.reserve(ints([1, 1, 1, 0]))
    after = cache.table.tolist()
    assert after[0] == before[0] and len({after[s][1] for s in range(3)}) == 3
    page = cache.table[:3, 1].long()
    assert torch.equal(cache.pool[0, 0, page, 0, :4], k[0, 16:20, 0].to(BF16).expand(3, 4, 64))
    assert faults_of(cache) == 0


def test_too_few_pages_change_nothing():
    cache = make(sequences=3, pages=5, max_pages=4, fill=0.0)
    cache.reserve(ints([16, 17, 0]))
    state = [t.clone() for t in (cache.table, cache.held, cache.lengths, cache.refs)]
    for counts, fault in (([0, 0, 48], NO_PAGES), ([0, 65, 0], TOO_LONG), ([0, -1, 1], BAD_INDEX), ([33, 33, 33], NO_PAGES)):
        cache.reserve(ints(counts))
        assert faults_of(cache) == fault
        assert all(torch.equal(a, b) for a, b in zip(state, (cache.table, cache.held, cache.lengths, cache.refs)))
    cache.reserve(ints([0, 0, 32]))            # exactly what is left
    assert faults_of(cache) == 0 and cache.refs.tolist() == [1] * 5
    assert faults_of(cache) == 0


def test_indexes_out_of_range_are_left_out():
    cache = make(sequences=3, pages=12, layers=2, fill=0.0)
    k = torch.randn(3, 8, 1, 64, device="cuda")
    cache.reserve(ints([8, 8, 0]))
    cache.append(0, k, k, ints([8, 9, 1]))       # nine of eight tokens; no room for the third
    assert faults_of(cache) == BAD_INDEX | NO_ROOM
    cache.append(0, k, k, slots=ints([1, 1, -3]))
    assert faults_of(cache) == BAD_INDEX
    page = cache.table[1, 0]
    assert torch.equal(cache.pool[0, 0, page, 0, :8], k[0, :, 0].to(BF16))
    cache.append(0, k[:1], k[:1], slots=ints([2**31 - 1]))
    cache.fork(ints([0, 3, -2]))
    assert faults_of(cache) == BAD_INDEX and cache.held.tolist() == [1, 1, 0]
    cache.accept(ints([2, 2, 0]), ints([[1, 1], [3, 2], [0, 0]]))
    assert faults_of(cache) == BAD_INDEX and cache.lengths.tolist() == [0, 0, 0]
    cache.accept(ints([3, -1, 0]), ints([[0, 1], [0, 1], [0, 0]]))
    assert faults_of(cache) == BAD_INDEX
    cache.accept(ints([1, 17, 0]), ints([[16], [0], [0]]))
    assert faults_of(cache) == BAD_INDEX | NO_ROOM and cache.lengths.tolist() == [0, 0, 0]
    cache.accept(ints([17, 16, 1]))
    assert faults_of(cache) == NO_ROOM and cache.lengths.tolist() == [0, 16, 0]
    cache.fork(ints([1, 1, 1]))
    cache.append(0, k, k, slots=ints([0, 1, 2]))
    assert faults_of(cache) == NO_ROOM
    cache.truncate(ints([8, 8, 8]))
    before = cache.pool.clone()
    cache.append(0, k, k)
    assert faults_of(cache) == SHARED and torch.equal(before, cache.pool)
    cache.accept(ints([1, 0, 0]), ints([[3], [0], [0]]))
    assert faults_of(cache) == SHARED and cache.lengths.tolist() == [8, 8, 8]
    q = torch.randn(2, 1, 1, 64, device="cuda", dtype=BF16)
    out = cache.attend(0, q, slots=ints([0, 7]))
    assert faults_of(cache) == BAD_INDEX | NO_ROOM or faults_of(cache) == 0
    assert (out[1] == 0).all() and torch.isfinite(out).all()
    cache.table[0, 0] = 10**6
    cache.truncate(ints([8, 0, 0]))
    cache.compact()
    cache.fork(ints([0, 0, 0]))
    cache.attend(0, q[:1])
    assert faults_of(cache) != 0


def test_arguments_that_are_refused():
    cache = make(sequences=2, pages=8, kv_heads=2, layers=2)
    good = torch.zeros(2, 3, 2, 64, device="cuda")
    three, two = ints([0, 0, 0]), ints([0, 0])
    for call, error in [
            (lambda: cache.reserve([0, 0]), TypeError), (lambda: cache.reserve(three), ValueError), (lambda: cache.reserve(two.float()), TypeError),
            (lambda: cache.reserve(two.cpu()), ValueError), (lambda: cache.fork(two[None]), ValueError), (lambda: cache.truncate(three), ValueError),
            (lambda: cache.append(2, good, good), ValueError), (lambda: cache.append(-1, good, good), ValueError), (lambda: cache.append(0, good, good[:, :2]), ValueError),
            (lambda: cache.append(0, good, good.to(BF16)), ValueError), (lambda: cache.append(0, good.half(), good.half()), TypeError),
            (lambda: cache.append(0, good[..., :32], good[..., :32]), ValueError), (lambda: cache.append(0, good[:, :, :1], good[:, :, :1]), ValueError),
            (lambda: cache.append(0, good.cpu(), good.cpu()), ValueError), (lambda: cache.append(0, good[0], good[0]), ValueError),
            (lambda: cache.append(0, good, good, counts=three), ValueError), (lambda: cache.append(0, good, good, slots=three), ValueError),
            (lambda: cache.append(0, torch.zeros(3, 1, 2, 64, device="cuda"), torch.zeros(3, 1, 2, 64, device="cuda")), ValueError),
            (lambda: cache.accept(two, two), ValueError), (lambda: cache.accept(two, ints([[0]])), ValueError), (lambda: cache.accept(three), ValueError),
            (lambda: cache.attend(0, good[:, :, :1]), ValueError), (lambda: cache.attend(2, good), ValueError), (lambda: cache.attend(0, good.double()), TypeError),
            (lambda: cache.attend(0, good, mask=torch.ones(3, 3, device="cuda")), TypeError), (lambda: cache.attend(0, good, mask=torch.ones(2, 3, dtype=torch.bool, device="cuda")), ValueError),
            (lambda: cache.attend(0, good, mask=torch.ones(3, 3, dtype=torch.bool)), ValueError), (lambda: cache.attend(0, good, scale=0.0), ValueError),
            (lambda: cache.attend(0, good, scale=float("nan")), ValueError), (lambda: cache.attend(0, good, scale=1e-40), ValueError),
            (lambda: cache.attend(0, good, scale=-1.0), ValueError), (lambda: cache.attend(0, good, scale=float("inf")), ValueError), (lambda: cache.attend(0, good, out=good), ValueError),
            (lambda: cache.attend(0, good, out=good[:1].to(BF16)), ValueError), (lambda: cache.attend(0, good, counts=three), ValueError)]:
        with pytest.raises(error):
            call()
    assert faults_of(cache) == 0
    empty = torch.zeros(0, 3, 2, 64, device="cuda")
    cache.append(0, empty, empty)
    cache.append(0, good[:, :0], good[:, :0])
    assert cache.attend(0, empty).shape == (0, 3, 2, 64) and cache.attend(0, good[:, :0]).shape == (2, 0, 2, 64)
    cache.accept(two, torch.zeros(2, 0, dtype=torch.int32, device="cuda"))
    assert faults_of(cache) == 0
    cache.close()
    with pytest.raises(ValueError):
        cache.compact()


def test_a_pool_that_no_memory_holds_is_refused():
    with pytest.raises(MemoryError, match="GPU memory"):
        make(pages=1 << 22, layers=64, kv_heads=8, head_dim=128)


# ---- attention ---------------------------------------------------------------------------------

def bound(o, q, mask, counts, slots, dtype, scale):
    """The largest error that the arithmetic allows, per element, and the float64 result.

    16-bit types round every weight and the result to half a step u each.  A score is a float32 sum of D products (each exact for 16-bit operands, within 2^-21 for
    float32 ones, whose heads and tails are multiplied), summed in runs of 8 or 16 with errors of 2^-23: it is off by at most
    (D / 8 + 8) 2^-23 of the sum of its products' sizes, the exponent's argument by three roundings of 2^-24 more; a weight by that, once for itself and once for the sum of the
    weights, and by 2 x 2^-22 for the exponential.  The result's sum over N keys, 8 or more at a time, and the joins of parts add (N / 8 + 64) 2^-23."""
    want, weight, sizes = o.attend(0, q, mask, counts, slots, scale)
    dim = q.shape[3]
    u = torch.finfo(dtype).eps / 2 if dtype != F32 else 0.0
    score = sizes * ((dim / 8 + 8) * 2.0**-23 + (2.0**-21 if dtype == F32 else 0.0) + 3 * 2.0**-24)
    keys = max(o.lengths) + q.shape[1]
    wide = 2 * score + 2.0**-21 + (keys / 8 + 64) * 2.0**-23 + (2.0**-21 if dtype == F32 else 0.0)
    return want, weight * (u + wide * (1 + u)) + u * np.abs(want) + 2.0**-24 * np.abs(want) + 1e-30


def check(cache, q, mask=None, counts=None, slots=None, scale=None, **kw):
    o = Oracle.of(cache)
    got = cache.attend(0, q, mask=None if mask is None else torch.from_numpy(mask).cuda(), counts=None if counts is None else ints(counts),
                       slots=None if slots is None else ints(slots), scale=scale, **kw)
    assert faults_of(cache) == 0
    want, allowed = bound(o, q, None if mask is None else torch.from_numpy(mask), counts, slots, cache.dtype, scale)
    got64 = got.cpu().double().numpy()
    assert got.dtype == cache.dtype and np.isfinite(got64).all()
    worst = (np.abs(got64 - want) / allowed).max(initial=0.0)
    assert worst <= 1.0, worst
    return got


def filled(lengths, counts, spare=0, seed=0, spread=1.0, **sizes):
    """A cache with that many committed tokens, and drafted ones behind them."""
    tokens = max(counts)
    page = sizes.get("page_tokens", 16)
    held = [-(-(n + c) // page) for n, c in zip(lengths, counts)]
    cache = make(sequences=len(lengths) + spare, pages=sum(held) + 3, max_pages=max(held) + 1, **sizes)
    cache.refs[1] = 1                                    # so that pages do not follow each other
    generator = torch.Generator("cuda").manual_seed(seed)
    for n in (lengths, counts):
        n = list(n) + [0] * spare
        if max(n) == 0:
            continue
        cache.reserve(ints(n))
        k, v = (torch.randn(len(n), max(n), cache.kv_heads, cache.head_dim, generator=generator, device="cuda") * spread for _ in range(2))
        for layer in range(cache.layers):
            cache.append(layer, k, v, ints(n))
        if n[:len(lengths)] == list(lengths) and cache.lengths.sum().item() == 0:
            cache.accept(ints(n))
    assert cache.lengths.tolist() == list(lengths) + [0] * spare
    q = torch.randn(len(lengths), tokens, sizes["kv_heads"] * sizes.pop("group", 1), cache.head_dim, generator=generator, device="cuda")
    return cache, q


SHAPES = [
    # dtype, lengths, counts, kv_heads, group, head_dim, page_tokens
    (BF16, [0], [1], 1, 1, 64, 16),
    (F32, [0, 1, 15, 16, 17], [1, 1, 1, 1, 1], 2, 1, 64, 16),
    (F16, [63, 64, 65, 127, 128, 129], [1, 2, 3, 2, 1, 3], 1, 4, 128, 32),
    (BF16, [5, 300, 0, 31], [7, 0, 5, 1], 3, 2, 80, 8),
    (F32, [31, 32, 33, 95, 0], [4, 9, 1, 2, 3], 2, 3, 128, 16),
    (BF16, [40, 200], [33, 17], 2, 2, 32, 64),
    (F16, [100, 3], [70, 64], 2, 3, 64, 16),               # several tiles of query rows
    (F32, [77, 12], [40, 21], 1, 2, 48, 8),
    (BF16, [130], [90], 1, 1, 128, 128),
    (BF16, [37, 64], [3, 20], 1, 1, 256, 16),
    (F32, [37, 64], [3, 20], 1, 2, 256, 16),
    (F16, [50, 1], [12, 30], 1, 1, 208, 8),
    (BF16, [1500, 20, 700], [2, 1, 2], 2, 4, 128, 64),       # parts of an item in many CTAs
    (F32, [1500, 20, 700], [2, 1, 2], 2, 1, 64, 16),
    (F16, [2049], [5], 4, 8, 16, 256),
    (BF16, [900, 33, 0, 257] * 20, [1] * 80, 1, 1, 64, 32),    # more rows than CTAs look at in one round is 128
    (BF16, [33, 5, 64] * 50, [2, 1, 3] * 50, 1, 2, 64, 16),
    (BF16, [2900, 2000, 3100, 1, 2500, 2999, 130, 3000], [1, 2, 3, 2, 1, 1, 3, 2], 16, 2, 128, 16),      # dozens of tiles to a CTA
    (F32, [1900, 1200, 1, 1777], [2, 1, 2, 3], 32, 1, 64, 32),
    (F16, [1500, 1600, 1700], [9, 9, 3], 16, 3, 128, 64),
    (BF16, [1000, 2000], [40, 33], 16, 1, 64, 16),
    (F16, [2000, 900, 0, 1900], [20, 33, 17, 1], 8, 4, 128, 16),        # 128 rows and more to a key head
    (BF16, [700, 64, 3000], [64, 65, 5], 3, 5, 80, 64),
    (BF16, [0, 1, 130], [130, 100, 17], 2, 2, 48, 8),
    (F32, [300, 45], [3, 9], 2, 1, 144, 32),
    (BF16, [300, 45, 1000], [3, 9, 1], 2, 3, 144, 16),
    (F32, [600, 2], [1, 1], 1, 5, 112, 128),
]


@pytest.mark.parametrize("masked", ["chain", "shared", "each"])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{str(s[0])[6:]}-{len(s[1])}x{max(s[2])}-{s[3]}x{s[4]}-d{s[5]}-p{s[6]}-{max(s[1])}")
def test_attention(shape, masked):
    dtype, lengths, counts, kv_heads, group, head_dim, page_tokens = shape
    cache, q = filled(lengths, counts, dtype=dtype, kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens, fill=float("nan"))
    q = torch.randn(len(lengths), max(counts), kv_heads * group, head_dim, device="cuda", generator=torch.Generator("cuda").manual_seed(7)).to(dtype)
    dice = random.Random(3)
    mask = None if masked == "chain" else tree(dice, max(counts)) if masked == "shared" else np.stack([tree(dice, max(counts)) for _ in lengths])
    first = check(cache, q, mask, counts)
    assert torch.equal(first, check(cache, q, mask, counts))          # the same bits again


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_rows_that_see_nothing_are_zero(dtype):
    cache, q = filled([0, 20, 0], [6, 6, 4], dtype=dtype, kv_heads=2, head_dim=64)
    mask = np.zeros((3, 6, 6), bool)
    mask[0, 2, 4] = mask[2, 0, 5] = True                  # (token 5 of a sequence of four: not there)
    out = check(cache, q.to(dtype), mask, [6, 6, 4])
    assert (out[0, :2] == 0).all() and (out[0, 3:] == 0).all() and (out[2] == 0).all()
    assert (out[0, 2] != 0).any() and (out[1] != 0).all()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf"), 3e38])
@pytest.mark.parametrize("dtype, head_dim, tokens", [(F32, 64, 5), (BF16, 128, 5), (F16, 80, 5), (BF16, 64, 40), (F32, 128, 40)])
def test_what_a_row_does_not_see_does_not_reach_it(dtype, head_dim, tokens, bad):
    """Keys and values of a masked drafted token are infinite, NaN or the type's largest; so are those of dropped tokens behind the sequence."""
    bad = min(bad, torch.finfo(dtype).max) if 0 < bad < float("inf") else bad
    cache, q = filled([30, 7], [tokens, tokens - 2], dtype=dtype, kv_heads=1, head_dim=head_dim, fill=bad)
    q = q.to(dtype)
    mask = np.stack([tree(random.Random(1), tokens)] * 2)
    hidden = tokens // 2
    mask[:, :, hidden] = False
    counts = [tokens, tokens - 2]
    clean = check(cache, q, mask, counts)
    for s, length in enumerate((30, 7)):
        at = length + hidden
        page = cache.table[s, at // 16].item()
        cache.pool[0, :, page, :, at % 16] = bad
    dirty = cache.attend(0, q, torch.from_numpy(mask).cuda(), ints(counts))
    assert torch.equal(clean, dirty)
    # and a row that does see them shows it, alone
    if bad != bad:
        mask[0, tokens - 1, hidden] = True
        out = cache.attend(0, q, torch.from_numpy(mask).cuda(), ints(counts))
        assert out[0, tokens - 1].isnan().all() and torch.equal(out[0, :tokens - 1], clean[0, :tokens - 1]) and torch.equal(out[1], clean[1])


def test_infinite_values_reach_the_rows_that_see_them():
    cache, q = filled([10], [4], dtype=BF16, kv_heads=1, head_dim=64)
    q = q.to(BF16)
    mask = np.tril(np.ones((4, 4), bool))
    page = cache.table[0, 0].item()
    cache.pool[0, 1, page, 0, 12, 5] = float("inf")         # V of drafted token 2, one element
    out = cache.attend(0, q, torch.from_numpy(mask).cuda())
    assert out[0, 2:, 0, 5].isposinf().all() and torch.isfinite(out[0, :2]).all()
    assert torch.isfinite(out[0, :, 0, :5]).all() and torch.isfinite(out[0, :, 0, 6:]).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_nan_query_stays_with_its_row(dtype):
    cache, q = filled([700], [3], dtype=dtype, kv_heads=2, head_dim=64)
    q = q.to(dtype)
    clean = check(cache, q)
    q[0, 1, 0, 3] = float("nan")
    out = cache.attend(0, q)
    assert out[0, 1, 0].isnan().all()
    out[0, 1, 0] = clean[0, 1, 0]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_scores_of_any_size(dtype):
    """One key far above the others, scores far below zero, a scale of its own."""
    cache, q = filled([150, 40], [3, 3], dtype=dtype, kv_heads=2, head_dim=64, spread=0.5)
    q = q.to(dtype)
    check(cache, q * 20, None, None, None, 1.0)
    check(cache, q, None, None, None, 1e-6)
    cache.pool[0, 0] = torch.where(cache.pool[0, 0].isnan(), cache.pool[0, 0], -cache.pool[0, 0].abs())
    check(cache, q.abs() * 8)


def test_strides_types_and_outputs():
    """Queries inside a fused projection's rows, float32 queries of a 16-bit cache, odd strides, an output of the caller's."""
    cache, _ = filled([60, 9], [5, 5], dtype=BF16, kv_heads=2, head_dim=64)
    generator = torch.Generator("cuda").manual_seed(2)
    fused = torch.randn(2, 5, 8 * 64, generator=generator, device="cuda")
    q = fused[..., :4 * 64].unflatten(2, (4, 64))
    plain = check(cache, q.to(BF16).contiguous())
    assert torch.equal(plain, check(cache, q.to(BF16)))
    assert torch.equal(plain, cache.attend(0, q))                                  # rounded once, as .to does
    assert torch.equal(plain, cache.attend(0, q.to(BF16).transpose(1, 2).contiguous().transpose(1, 2)))
    odd = torch.empty(2, 5, 4, 65, dtype=BF16, device="cuda")[..., 1:]
    odd.copy_(q)
    assert torch.equal(plain, cache.attend(0, odd))
    assert torch.equal(plain, cache.attend(0, q.to(BF16).requires_grad_()))
    wide = torch.full((2, 5, 6, 64), 7.0, dtype=BF16, device="cuda")
    out = cache.attend(0, q, out=wide[:, :, :4])
    assert out.data_ptr() == wide.data_ptr() and torch.equal(out, plain) and (wide[:, :, 4:] == 7).all()
    own = q.to(BF16)
    assert torch.equal(plain, cache.attend(0, own, out=own)) and torch.equal(plain, own)       # in place
    odd.zero_()
    assert cache.attend(0, q, out=odd) is odd and torch.equal(odd, plain)
    sees = torch.ones(5, 5, dtype=torch.bool, device="cuda").tril()
    assert torch.equal(plain, cache.attend(0, q, mask=sees.T.contiguous().T))        # a mask of other strides
    assert torch.equal(plain, cache.attend(0, q, mask=sees.expand(2, 5, 5)))
    assert torch.equal(plain, cache.attend(0, q, counts=torch.full((2,), 5, device="cuda")))       # int64
    k = torch.randn(2, 5, 2, 3, 64, generator=generator, device="cuda")
    before = Oracle.of(cache)
    cache.append(0, k[:, :, :, 0], k[:, :, :, 1])
    before.append(0, k[:, :, :, 0], k[:, :, :, 1])
    same(cache, before)


@pytest.mark.parametrize("dtype, heads, head_dim", [(BF16, 1, 128), (F16, 3, 64), (F32, 2, 64), (BF16, 2, 160)])
def test_masks_of_hundreds_of_tokens(dtype, heads, head_dim):
    """Their columns and rows in any order of memory, hidden tokens that hold NaN in every tile, tokens that see none of the drafted ones."""
    counts = [300, 65, 0, 129]
    cache, _ = filled([40, 0, 7, 64], counts, dtype=dtype, kv_heads=1, head_dim=head_dim)
    q = torch.randn(4, 300, heads, head_dim, device="cuda", generator=torch.Generator("cuda").manual_seed(7)).to(dtype)
    dice = np.random.default_rng(5)
    mask = np.tril(dice.random((4, 300, 300)) < 0.3)
    mask[:, ::7] = False
    mask[:, :, 3::31] = False
    clean = check(cache, q, mask, counts)
    for s, length in ((0, 40), (1, 0), (3, 64)):
        for at in range(length + 3, length + counts[s], 31):
            cache.pool[0, :, cache.table[s, at // 16].item(), :, at % 16] = float("nan")
    device = torch.from_numpy(mask).cuda()
    for same_mask in (device, device.permute(2, 0, 1).contiguous().permute(1, 2, 0), torch.stack((~device, device), 3)[..., 1]):
        assert torch.equal(clean, cache.attend(0, q, mask=same_mask, counts=ints(counts)))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_many_empty_rows_are_zero(dtype):
    """A padded batch of which most rows hold no token, in an output that held something else."""
    counts = [0, 200, 1, 0, 77, 3]
    cache, q = filled([0, 5, 300, 40, 9, 0], counts, dtype=dtype, kv_heads=2, head_dim=64)
    q = q.to(dtype)
    out = torch.full_like(q, 3.0)
    cache.attend(0, q, counts=ints(counts), out=out)
    check(cache, q, None, counts)
    for s, n in enumerate(counts):
        assert (out[s, n:] == 0).all() and (out[s, :n] != 0).any() == (n > 0)
    out.fill_(3.0)
    cache.attend(0, q[:2], counts=ints([200, 0]), slots=ints([1, 1]), out=out[:2])
    assert (out[1] == 0).all() and (out[2:] == 3).all() and faults_of(cache) == 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_that_name_their_sequences(dtype):
    lengths, counts = [70, 0, 5, 33], [3, 3, 3, 3]
    cache, q = filled(lengths, counts, spare=2, dtype=dtype, kv_heads=2, head_dim=64)
    q = q.to(dtype)
    whole = check(cache, q, None, [3, 2, 0, 1])
    order = [2, 0, 3, 1]
    some = check(cache, q[order], None, [[3, 2, 0, 1][s] for s in order], order)
    assert (some[0] == 0).all()
    for b, s in enumerate(order):
        assert torch.allclose(some[b].float(), whole[s].float(), atol=2.0**-7, rtol=2.0**-7)
    check(cache, q[[0, 0, 3]], None, None, [0, 0, 3])       # the same sequence twice
    check(cache, torch.cat([q, q]), None, [3, 1] * 4, [0, 1, 2, 3] * 2)      # more rows than sequences


def test_offsets_beyond_32_bits():
    """Pages whose elements, and whose bytes, are past 2^32 of the pool's start."""
    small, q = filled([100], [4], dtype=BF16, kv_heads=2, head_dim=128, page_tokens=64, layers=1)
    large = make(sequences=1, max_pages=4, pages=160000, kv_heads=2, head_dim=128, page_tokens=64, layers=1, fill=0.0)       # 10 GB
    q = q.to(BF16)
    large.refs[:159990] = 1
    o = Oracle.of(small)
    generator = torch.Generator("cuda").manual_seed(0)
    for n, commit in ((100, True), (4, False)):
        large.reserve(ints([n]))
        k, v = (torch.randn(1, n, 2, 128, generator=generator, device="cuda") for _ in range(2))
        large.append(0, k, v)
        if commit:
            large.accept(ints([n]))
    assert large.table[0, 0].item() >= 159990
    for at in range(104):
        page, row = o._place(0, at)
        assert np.array_equal(large.pool[0, :, large.table[0, at // 64].item(), :, at % 64].cpu().double().numpy(), o.pool[0, :, page, :, row])
    assert torch.equal(large.attend(0, q), small.attend(0, q))
    large.accept(ints([2]), ints([[1, 3]]))
    small.accept(ints([2]), ints([[1, 3]]))
    large.refs[:159990] = 0
    large.compact()
    assert large.table[0].tolist() == [0, 1, -1, -1]
    assert torch.equal(large.attend(0, q[:, :0]), small.attend(0, q[:, :0]))
    for c in (small, large):
        c.reserve(ints([1]))
        c.append(0, k[:, :1], v[:, :1])
    assert torch.equal(large.attend(0, q[:, :1]), small.attend(0, q[:, :1]))
    assert faults_of(large) == 0 and faults_of(small) == 0


# ---- streams, graphs, a run of all of them ------------------------------------------------------

def test_calls_on_other_streams_and_two_at_once():
    cache, q = filled([3000, 40, 700], [2, 2, 2], dtype=BF16, kv_heads=2, head_dim=64)
    q = q.to(BF16)
    plain = [cache.attend(0, q), cache.attend(0, -q)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = [[], []]
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(cache.attend(0, q if i == 0 else -q))
    torch.cuda.synchronize()
    assert all(torch.equal(x, plain[i]) for i in range(2) for x in outs[i])


@pytest.mark.parametrize("sequences", [3, 90])                         # (tables on one CTA, on a cluster)
def test_a_captured_step_follows_the_tables(sequences):
    """Fork, reserve, append, attend and accept as one graph: replays go on where the cache is, and two graphs do not share a workspace."""
    sizes = dict(sequences=sequences, max_pages=40, pages=40 * sequences, kv_heads=2, head_dim=64, dtype=BF16, layers=2, fill=0.0)
    cache, eager = make(**sizes), make(**sizes)
    tokens = 4
    x = torch.zeros(3, 2, sequences, tokens, 2, 64, device="cuda")      # q, k, v by layer
    counts, n = ints([4, 3, 1] * (sequences // 3)), ints([2, 3, 1] * (sequences // 3))
    kept = ints([[0, 2, 0], [0, 1, 2], [0, 0, 0]] * (sequences // 3))
    sources = torch.arange(sequences, device="cuda", dtype=torch.int32)
    mask = torch.from_numpy(tree(random.Random(2), tokens)).cuda()

    def step(c, data):
        c.fork(sources)
        c.reserve(counts)
        outs = []
        for layer in range(2):
            c.append(layer, data[1, layer], data[2, layer], counts)
            outs.append(c.attend(layer, data[0, layer], mask, counts))
        c.accept(n, kept)
        return outs

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(cache, x)                                                  # loads the kernels
    torch.cuda.current_stream().wait_stream(side)
    cache.truncate(torch.zeros_like(counts))
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(step(cache, x))
        graphs.append(graph)
    assert cache.lengths.tolist() == [0] * sequences
    generator = torch.Generator("cuda").manual_seed(4)
    for i in range(20):
        x.copy_(torch.randn(x.shape, generator=generator, device="cuda"))
        sources.copy_(torch.arange(sequences, device="cuda"))
        if i == 10:
            sources[0] = 1                                              # a beam, then writes into what it shares
        graphs[i % 2].replay()
        want = step(eager, x)
        for got, w in zip(outs[i % 2], want):
            assert torch.equal(got, w)
    assert cache.lengths.tolist() == eager.lengths.tolist() and cache.lengths.tolist()[:3] == [50, 60, 20]
    assert torch.equal(cache.table, eager.table) and torch.equal(cache.refs, eager.refs)
    assert faults_of(cache) == faults_of(eager) == 0


def test_many_calls_leave_the_allocator_as_it_was():
    cache, q = filled([300], [2], dtype=BF16, kv_heads=2, head_dim=64)
    q = q.to(BF16)
    out = cache.attend(0, q)
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(50):
        cache.attend(0, q, out=out)
    torch.cuda.synchronize()
    assert torch.cuda.memory_allocated() == before


def test_c_entry_refuses_short_workspaces():
    import ctypes as C

    cache, q = filled([3000], [2], dtype=BF16, kv_heads=2, head_dim=64)
    q = q.to(BF16)
    lib = _cabi.load()
    n = lib.kb200_cache_attend_workspace(cache._cache, 1, 2, 2)
    rows, out = _cabi.Rows(q.data_ptr(), 1, 2, q.stride()[:3]), torch.empty_like(q)
    out_rows = _cabi.Rows(out.data_ptr(), 1, 2, out.stride()[:3])
    assert n > 0
    space = torch.empty(n + 16, dtype=torch.uint8, device="cuda")
    call = lambda at, size, a=rows, b=out_rows: lib.kb200_cache_attend(cache._cache, 0, C.byref(a), C.byref(b), 1, 2, None, None, None, None, 0.125, at, size, None)  # noqa: E731
    assert call(space.data_ptr(), n - 1) == -1 and call(None, n) == -1 and call(space.data_ptr() + 8, n) == -1
    assert call(space.data_ptr(), n) == 0
    assert lib.kb200_cache_attend_workspace(cache._cache, 1, 2, 3) == 0
    bad = _cabi.Rows(q.data_ptr(), 1, 2, (256, 128, 4))
    assert call(space.data_ptr(), n, bad) == -1
    assert call(space.data_ptr(), n, rows, _cabi.Rows(out.data_ptr(), 0, 2, (256, 128, 64))) == -1
    torch.cuda.synchronize()
    assert torch.equal(out, cache.attend(0, q))

"""Verification of drafted tokens on the GPU (``PagedCache.verify``): against the rules in float64, token for token."""

import random

import numpy as np
import pytest
import torch

from kiln_b200 import _cabi
from oracle.cache_oracle import BAD_INDEX
from oracle.cache_steps_oracle import BAD_VALUE, verify as by_the_rules
from test_paged_cache_gpu import BF16, F16, F32, ints

pytestmark = pytest.mark.gpu


def cache_of(sequences):
    from kiln_b200.cache import PagedCache

    return PagedCache(layers=1, sequences=sequences, max_pages=4, pages=4 * sequences, kv_heads=1, head_dim=16, page_tokens=16)


def faults_of(cache):
    torch.cuda.synchronize()
    try:
        cache.status()
    except ValueError as e:
        return (BAD_INDEX if "out of range" in str(e) else 0) | (BAD_VALUE if "no distribution" in str(e) else 0)
    return 0


def drafts(rows, tokens, vocab, dtype, draft_dtype, seed=0, trees=False, spread=2.5, noise=0.7, temperature=None):
    """Logits, and tokens as a small model draws them that knows much of what the large one does."""
    generator = torch.Generator("cuda").manual_seed(seed)
    dice = random.Random(seed)
    logits = (torch.randn(rows, tokens, vocab, device="cuda", generator=generator) * spread).to(dtype)
    t = torch.ones(rows, device="cuda") if temperature is None else temperature.clamp_min(0.3)
    q = torch.softmax(logits.float() / t[:, None, None] + noise * torch.randn(rows, tokens, vocab, device="cuda", generator=generator), -1)
    parents = [[-1] + [dice.randint(max(0, i - 3), i - 1) if trees else i - 1 for i in range(1, tokens)] for _ in range(rows)]
    of = torch.tensor(parents, device="cuda").clamp_min(0)
    drawn = q[torch.arange(rows, device="cuda")[:, None], of].reshape(-1, vocab)
    chosen = torch.multinomial(drawn, 1, generator=generator)[:, 0] if draft_dtype is not None else drawn.argmax(-1)
    uniform = torch.rand(rows, tokens, device="cuda", generator=generator)
    return dict(logits=logits, tokens=chosen.view(rows, tokens).int(), uniform=uniform, draft=None if draft_dtype is None else q.to(draft_dtype),
                parents=torch.tensor(parents, device="cuda", dtype=torch.int32) if trees else None)


def check(cache, counts=None, slots=None, **given):
    got = cache.verify(**given, counts=None if counts is None else ints(counts), slots=None if slots is None else ints(slots))
    *want, faults = by_the_rules(cache.sequences, counts=counts, slots=slots, **given)
    assert [x.tolist() for x in got] == want
    assert faults_of(cache) == faults
    return want


@pytest.mark.parametrize("trees", [False, True])
@pytest.mark.parametrize("draft", [None, F32, "same"])
@pytest.mark.parametrize("dtype, rows, tokens, vocab", [
    (F32, 1, 1, 1), (F32, 3, 2, 5), (BF16, 2, 9, 7), (F16, 4, 5, 50257), (BF16, 20, 7, 1000), (F32, 5, 33, 2049), (F32, 1, 4, 131073), (BF16, 150, 3, 4001), (F16, 2, 200, 300)])
def test_verification(dtype, rows, tokens, vocab, draft, trees):
    cache = cache_of(rows)
    dice = random.Random(vocab)
    for seed in range(3):
        counts = [dice.randint(0, tokens) if b else tokens for b in range(rows)]
        temperature = torch.tensor([dice.choice([0.0, 0.5, 1.0, 1.7]) for _ in range(rows)], device="cuda")
        given = drafts(rows, tokens, vocab, dtype, dtype if draft == "same" else draft, seed, trees, temperature=temperature)
        check(cache, counts, temperature=temperature if seed else None, **given)


def test_tokens_that_follow_the_same_one():
    """Many drafts of one token: each refusal leaves less, down to nothing."""
    rows, tokens, vocab = 40, 12, 6
    cache = cache_of(rows)
    for draft in (None, F32):
        for seed in range(6):
            given = drafts(rows, tokens, vocab, F32, draft, seed, spread=[0.5, 4.0][seed % 2], noise=[0.0, 0.5, 3.0][seed % 3])
            given["parents"] = ints([-1] + [0] * (tokens - 2) + [1])
            given["uniform"] = 1 - (1 - given["uniform"]) * 2.0**-(4 * (seed % 3))      # close to 1: more is refused
            check(cache, **given)
    # equal tokens: what was refused once is refused again
    given["tokens"] = torch.full((rows, tokens), 2, dtype=torch.int32, device="cuda")
    given["draft"] = None
    n, _, following = check(cache, **given)
    assert any(x == 1 and v != 2 for x, v in zip(n, following))


@pytest.mark.parametrize("dtype, vocab", [(F32, 5), (BF16, 4001), (F16, 50257), (F32, 131072), (BF16, 131072)])
def test_equal_logits_at_temperature_zero(dtype, vocab):
    """The first of the largest ones counts, wherever they lie: all equal, a few values only, and two of them anywhere."""
    rows = 12
    cache = cache_of(rows)
    given = drafts(rows, 4, vocab, dtype, None, 4)
    x = given["logits"]
    x[:4] = 1.5
    x[4:8] = (x[4:8] / 4).round()
    dice = random.Random(vocab)
    for b in range(8, rows):
        for i in range(4):
            x[b, i, [0, dice.randrange(vocab)] if i < 2 else [dice.randrange(vocab), vocab - 1 - dice.randrange(min(vocab, 9))]] = 60.0
    given["tokens"] = torch.zeros_like(given["tokens"])
    n, _, following = check(cache, temperature=torch.zeros(rows, device="cuda"), **given)
    assert n[:4] == [4] * 4 and following[:4] == [0] * 4


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_numbers_next_to_a_border(dtype):
    """Random numbers one step of float32 to either side of a token's chance and of the border between two tokens that may follow: float32's sums cannot tell them."""
    rows, vocab = 64, 20011
    cache = cache_of(rows)
    given = drafts(rows, 2, vocab, dtype, None, 3, spread=1.0)
    p = torch.softmax(given["logits"].double(), -1)
    given["tokens"][:, 1] = p[:, 0].topk(40, -1).indices[:, 30].int()
    chance = p[:, 0].gather(1, given["tokens"][:, 1:].long())[:, 0].float()
    at = torch.arange(rows, device="cuda")
    steps = torch.tensor([-1.0, 0.0, 1.0, 2.0], device="cuda")[at % 4]
    given["uniform"][:, 1] = (chance.view(torch.int32) + steps.int()).view(F32)
    n, *_ = check(cache, **given)
    assert {1, 2} <= set(n)
    sums = p[:, 0].cumsum(-1)[at, at * 300]
    given["uniform"][:, 0] = (sums.float().view(torch.int32) + steps.int()).view(F32)
    check(cache, **{**given, "logits": given["logits"][:, :1], "tokens": given["tokens"][:, :1], "uniform": given["uniform"][:, :1]})
    # with a draft: the ratio of two chances
    given["draft"] = torch.softmax(given["logits"].float() * 0.9, -1)
    ratio = (p[:, 0] / given["draft"][:, 0].double()).gather(1, given["tokens"][:, 1:].long())[:, 0].float()
    given["uniform"][:, 1] = (ratio.view(torch.int32) + steps.int()).view(F32)
    n, *_ = check(cache, **given)
    assert {1, 2} <= set(n)
    given["uniform"][:, 0] = torch.where(at % 2 == 0, 0.0, 1 - 2.0**-24)              # the first token and the last one that may follow
    check(cache, **given)


@pytest.mark.parametrize("rise", [0.25, 0.5, 0.75, 1.0, 1.5, 2.5, 4.0, 7.0, 40.0])
def test_logits_that_ascend(rise):
    """By as much in every 4096 of four million, so that a running maximum grows a thousand times: a row's sum is still near enough to tell which random numbers are next to a token's
    chance (from 4 x 10^-8 of it on, to either side)."""
    vocab, rows = 1 << 22, 640
    cache = cache_of(rows)
    row = (torch.arange(vocab, device="cuda") // 4096).float() * (rise / 1024)
    p = torch.softmax(row.double(), 0)
    token = vocab - 5000
    chance = p[token].item()
    near = torch.tensor(chance, device="cuda").float().view(torch.int32) + (torch.arange(rows, device="cuda") - rows // 2).int()      # (a step is 2^-24 to 2^-23 of it)
    uniform = torch.stack([torch.full((rows,), 0.37, device="cuda"), near.view(F32)], 1)
    n, accepted, following = cache.verify(row.expand(rows, 2, vocab), ints([[0, token]] * rows), uniform)
    taken = uniform[:, 1].double() < chance
    assert n.tolist() == (1 + taken.int()).tolist() and {1, 2} == set(n.tolist())
    rest = p.clone()
    rest[token] = 0
    first = [int(torch.searchsorted(x.cumsum(0), uniform[0, 0].double() * x.sum(), right=True)) for x in (rest, p)]
    assert following.tolist() == [first[int(x)] for x in taken] and faults_of(cache) == 0


def test_little_that_a_draft_leaves():
    """Ten-millionths of the model's chances, and beside them a draft that is right to float32's last bit for tokens of a thousand times as much: of those what is left changes its sign with a
    sum that is off by as little.  Random numbers next to the borders of what may follow."""
    rows, vocab = 64, 20011
    cache = cache_of(rows)
    generator = torch.Generator("cuda").manual_seed(17)
    order = torch.rand(rows, vocab, device="cuda", generator=generator).argsort(-1)
    size = torch.ones(rows, vocab, dtype=torch.float64, device="cuda")              # most tokens: equal ones, of which a draft has too much
    size[:, 0] = torch.linspace(0.3, 4.0, rows, device="cuda").double().exp()       # the largest, by which a row's weights are scaled
    rand = lambda n: 0.5 + torch.rand(rows, n, device="cuda", generator=generator).double()  # noqa: E731
    size[:, 1:801] = rand(800) * 1e-7 * vocab                                       # a draft that is nearly right: 8e-5
    size[:, 801:841] = rand(40) * 5e-9 * vocab                                      # half of it is left: 1e-7
    logits = torch.empty(rows, 2, vocab, device="cuda")
    logits[:] = size.log().float().gather(1, order.argsort(-1))[:, None]
    p = torch.softmax(logits[:, 0].double(), -1)
    factor = torch.full((rows, vocab), 1.01, dtype=torch.float64, device="cuda")
    factor[:, 1:801], factor[:, 801:841] = 1.0, 0.5
    draft = (p * factor.gather(1, order.argsort(-1))).float()
    left = (p - draft.double()).clamp_min(0)
    assert (left.sum(-1) < 2e-7).all() and (left.sum(-1) > 5e-8).all()
    sums, at = left.cumsum(-1), torch.arange(rows, device="cuda")
    border = (sums / sums[:, -1:])[at, order[at, 801 + at % 40]].float().clamp_max(0.999)
    steps = torch.tensor([-2, -1, 1, 2], dtype=torch.int32, device="cuda")[at % 4]
    uniform = torch.stack([(border.view(torch.int32) + steps).view(F32), torch.full((rows,), 0.9999, device="cuda")], 1)
    n, *_ = check(cache, logits=logits, tokens=order[:, [0, 5000]].int(), uniform=uniform, draft=draft[:, None].expand(rows, 2, vocab))
    assert n == [1] * rows


@pytest.mark.parametrize("mask", [-float("inf"), -1e9, -30000.0])
@pytest.mark.parametrize("dtype, draft_dtype, vocab, rows, trees", [(F32, F32, 20011, 9, False), (BF16, F32, 50257, 6, False), (F16, F16, 30000, 6, True), (BF16, None, 20011, 6, True)])
def test_masked_logits(dtype, draft_dtype, vocab, rows, trees, mask):
    """All but a few logits of every row, as a grammar or the top 50 leave them, and a draft that knows nothing of it."""
    cache = cache_of(rows)
    for seed, kept in enumerate((1, 50, 999)):
        given = drafts(rows, 6, vocab, dtype, draft_dtype, 30 + seed, trees)
        x = given["logits"]
        least = x.topk(kept, -1).values[..., -1:]
        x.masked_fill_(x < least, mask if dtype != F16 else max(mask, -60000.0) if mask > -float("inf") else mask)
        check(cache, temperature=None if seed else torch.full((rows,), 0.6, device="cuda"), **given)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_token_that_every_refusal_leaves(dtype):
    """Of two hundred drafts of one token none is accepted, and each time one token is left, by as much: 1 less the draft's chance of it, of 1.  What it is divided by is what it was, bit by
    bit, or nothing is left of it in the end."""
    rows, tokens, vocab = 200, 200, 90
    cache = cache_of(rows)
    generator = torch.Generator("cuda").manual_seed(23)
    logits = torch.randn(rows, 1, vocab, device="cuda", generator=generator)
    one = torch.randint(vocab, (rows, 1, 1), device="cuda", generator=generator)
    logits.scatter_(2, one, 14.0 + torch.rand(rows, 1, 1, device="cuda", generator=generator))         # 0.999 and more
    draft = torch.rand(rows, 1, vocab, device="cuda", generator=generator) + 0.1
    draft.scatter_(2, one, 0.0)
    share = torch.linspace(0.03, 0.97, rows, device="cuda")[:, None, None]
    draft = (draft / draft.sum(-1, keepdim=True) * (1 - share)).scatter(2, one, share)
    drawn = (one[:, :, 0] + torch.randint(1, vocab, (rows, tokens), device="cuda", generator=generator)) % vocab
    uniform = 0.5 + torch.rand(rows, tokens, device="cuda", generator=generator) / 2
    n, _, following = check(cache, logits=logits.to(dtype).expand(rows, tokens, vocab), tokens=drawn.int(), uniform=uniform, draft=draft.expand(rows, tokens, vocab),
                            parents=ints([-1] + [0] * (tokens - 1)))
    assert n == [1] * rows and following == one.flatten().tolist()


def test_what_is_returned_is_distributed_as_the_models_samples():
    """The first token that a step adds, over 32768 rows each: of a chain, of several drafts of one token, with probabilities of a draft and without.  A count is off by its standard
    deviation sqrt(n p (1 - p)) five times at most (24 counts: one in 70000 would be)."""
    vocab, rows = 6, 1 << 15
    cache = cache_of(rows)
    generator = torch.Generator("cuda").manual_seed(0)
    p = torch.tensor([0.4, 0.05, 0.25, 0.02, 0.08, 0.2], dtype=torch.float64, device="cuda")
    q = torch.tensor([0.1, 0.3, 0.2, 0.2, 0.15, 0.05], device="cuda")
    for tokens, parents, with_draft in ((2, None, True), (2, None, False), (4, ints([-1, 0, 0, 0]), True), (4, ints([-1, 0, 0, 0]), False)):
        drawn = torch.multinomial(q.expand(rows, vocab), tokens, replacement=True, generator=generator).int()
        if not with_draft:
            drawn[:] = ints([0, 1, 0, 5])[:tokens]
        uniform = torch.rand(rows, tokens, device="cuda", generator=generator)
        n, accepted, following = cache.verify(p.log().float().expand(rows, tokens, vocab), drawn, uniform, draft=q.expand(rows, tokens, vocab) if with_draft else None, parents=parents)
        first = torch.where(n > 1, drawn.gather(1, accepted[:, 1:2].clamp_min(0).long())[:, 0], following)
        assert (n > 1).any() and (n == 1).any()
        counts = torch.bincount(first, minlength=vocab).double()
        assert ((counts - rows * p).abs() <= 5 * (rows * p * (1 - p)).sqrt()).all()
    assert faults_of(cache) == 0


def test_rows_that_name_their_sequences():
    cache = cache_of(7)
    given = drafts(3, 4, 500, BF16, F32, 5)
    check(cache, [4, 2, 0], [6, 0, 3], **given)
    n, accepted, following = check(cache, [4, 2, 3], [5, 5, 9], **given)              # a sequence twice, and one that there is not
    assert n[5] > 0 and sum(n) == n[5] and following[:5] == [-1] * 5
    check(cache, [9, -2, 3], [1, 2, 3], **given)
    check(cache, None, None, **given)
    check(cache, [0, 0, 0], None, **given)


def test_tokens_and_parents_out_of_range():
    cache = cache_of(4)
    given = drafts(4, 4, 50, F32, F32, 6, trees=True)
    given["tokens"][:, 0] = -7                                              # (nobody asks for the first one's)
    check(cache, **given)
    for at, token in ((1, 50), (2, -1), (3, 2**31 - 1)):
        check(cache, **{**given, "tokens": given["tokens"].index_fill(1, torch.tensor([at], device="cuda"), token)})
    for at, parent in ((1, 1), (2, 3), (3, -2), (1, -1), (2, -1)):
        check(cache, **{**given, "parents": given["parents"].index_fill(1, torch.tensor([at], device="cuda"), parent)})
    check(cache, **{**given, "parents": ints([5, 0, 0, 0])})


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("temperature", [None, 0.0, 0.7])
def test_logits_that_are_no_distribution(dtype, temperature):
    """-inf is a token of no chance; NaN, +inf and nothing but -inf end a row where it reaches them, and nowhere else."""
    rows, vocab = 8, 3001
    cache = cache_of(rows)
    given = drafts(rows, 3, vocab, dtype, F32, 7, noise=0.0)
    given["uniform"] *= 0.5                                                 # most are accepted
    x = given["logits"]
    x[0, :, 1::2] = -float("inf")
    x[1, 0, 5], x[2, 1, vocab - 1], x[3, 2, 0] = float("nan"), float("nan"), float("nan")
    x[4, 1, 7] = float("inf")
    x[5, 0] = -float("inf")
    x[6, 2] = float("nan")
    t = None if temperature is None else torch.full((rows,), temperature, device="cuda")
    n, _, following = check(cache, temperature=t, **given)
    assert n[1] == 1 and following[1] == -1 and following[5] == -1 and following[7] >= 0
    given["draft"][7] = float("nan")
    check(cache, temperature=t, **given)


def test_temperatures():
    cache = cache_of(9)
    given = drafts(9, 3, 2000, F32, F32, 8)
    t = torch.tensor([-1.0, float("nan"), float("inf"), 0.0, 1e-30, 1e-42, 1e30, 0.1, -0.0], device="cuda")
    n, _, following = check(cache, temperature=t, **given)
    assert n[:3] == [0, 0, 0] and following[:3] == [-1] * 3 and min(n[3:]) > 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_alignment(dtype):
    """Rows that begin anywhere, of any number of tokens, in tensors that hold more."""
    cache = cache_of(3)
    for vocab in (1, 7, 8, 15, 64, 1001):
        plain = drafts(3, 4, vocab, dtype, dtype, vocab, trees=True)
        want = [x.tolist() for x in cache.verify(**plain)]
        assert check(cache, **plain) == want
        for lead in (1, 3, 5):
            wide = torch.full((4, 3, vocab + 9), float("nan"), dtype=dtype, device="cuda")
            logits = wide.transpose(0, 1)[:, :, lead:lead + vocab]
            logits.copy_(plain["logits"])
            far = torch.full((3, 6, vocab + 2), float("nan"), dtype=dtype, device="cuda")[:, 1:5, 1:1 + vocab]
            far.copy_(plain["draft"])
            uniform = torch.zeros(4, 3, device="cuda").T.copy_(plain["uniform"])
            got = cache.verify(logits, plain["tokens"].long(), uniform, draft=far, parents=plain["parents"].long())
            assert [x.tolist() for x in got] == want
        turned = plain["logits"].permute(2, 0, 1).contiguous().permute(1, 2, 0)
        assert [x.tolist() for x in cache.verify(**{**plain, "logits": turned, "draft": turned.to(F32).softmax(-1)})] == \
            [x.tolist() for x in cache.verify(**{**plain, "draft": turned.contiguous().to(F32).softmax(-1).contiguous()})]
        one = plain["logits"][:, :1].expand(3, 4, vocab)                    # (rows that share memory)
        check(cache, **{**plain, "logits": one})
    assert faults_of(cache) == 0


def test_offsets_beyond_32_bits():
    rows, tokens, vocab = 18, 1000, 250007                                  # 4.5e9 elements, of which each row takes two
    cache = cache_of(rows)
    logits = torch.empty(rows, tokens, vocab, dtype=BF16, device="cuda")
    given = drafts(rows, 2, vocab, BF16, F32, 9)
    logits[:, -2:] = given["logits"]
    want = [x.tolist() for x in cache.verify(**given)]
    assert [x.tolist() for x in cache.verify(**{**given, "logits": logits[:, -2:]})] == want
    logits[:, -2:] = given["draft"].to(BF16)
    assert [x.tolist() for x in cache.verify(**{**given, "draft": logits[:, -2:]})] == [x.tolist() for x in cache.verify(**{**given, "draft": given["draft"].to(BF16)})]
    assert faults_of(cache) == 0


def test_nothing_to_verify():
    cache = cache_of(2)
    for shape in ((0, 3, 10), (2, 0, 10)):
        n, accepted, following = cache.verify(torch.zeros(shape, device="cuda"), torch.zeros(shape[:2], dtype=torch.int32, device="cuda"), torch.zeros(shape[:2], device="cuda"))
        assert n.tolist() == [0, 0] and accepted.tolist() == [[-1] * shape[1]] * 2 and following.tolist() == [-1, -1]
    assert faults_of(cache) == 0


def test_arguments_that_are_refused():
    cache = cache_of(2)
    given = drafts(2, 3, 11, F32, F32, 0)
    ok = dict(given, parents=ints([-1, 0, 1]))
    cache.verify(**ok)
    for change, error in [
            (dict(logits=given["logits"].double()), TypeError), (dict(logits=given["logits"][0]), ValueError), (dict(logits=given["logits"].cpu()), ValueError), (dict(logits=None), TypeError),
            (dict(logits=given["logits"][..., :0]), ValueError), (dict(tokens=given["tokens"][:, :2]), ValueError), (dict(tokens=given["tokens"].float()), TypeError),
            (dict(tokens=given["tokens"].cpu()), ValueError), (dict(uniform=given["uniform"].double()), TypeError), (dict(uniform=given["uniform"][:1]), ValueError), (dict(uniform=None), TypeError),
            (dict(draft=given["draft"][..., :10]), ValueError), (dict(draft=given["draft"].double()), TypeError), (dict(draft=given["draft"].cpu()), ValueError),
            (dict(parents=ints([0, 1])), ValueError), (dict(parents=ints([[0, 1, 2]])), ValueError), (dict(parents=given["uniform"]), TypeError), (dict(counts=ints([1])), ValueError),
            (dict(slots=ints([1, 0, 2])), ValueError), (dict(temperature=1.0), TypeError), (dict(temperature=torch.ones(3, device="cuda")), ValueError),
            (dict(temperature=torch.ones(2, device="cuda", dtype=torch.float64)), TypeError)]:
        with pytest.raises(error):
            cache.verify(**{**ok, **change})
    three = drafts(3, 1, 11, F32, None, 0)
    with pytest.raises(ValueError):
        cache.verify(**three)
    long = drafts(1, 513, 4, F32, None, 0)
    with pytest.raises(ValueError):
        cache.verify(**long)
    assert cache.verify(**{k: v[:, :512] if v is not None else v for k, v in long.items()})[0][0].item() > 0
    assert faults_of(cache) == 0
    cache.close()
    with pytest.raises(ValueError):
        cache.verify(**ok)


def test_the_c_entry_refuses():
    import ctypes as C

    cache, lib = cache_of(2), _cabi.load()
    given = drafts(2, 3, 1000, F32, F32, 0)
    x, d = given["logits"], given["draft"]
    n = lib.kb200_cache_verify_workspace(cache._cache, 2, 3, 1000)
    space, out = torch.empty(n + 16, dtype=torch.uint8, device="cuda"), torch.empty(2, 5, dtype=torch.int32, device="cuda")
    outs = (out[:, 0].contiguous(), out[:, 1:4].contiguous(), out[:, 4].contiguous())

    def call(logits=_cabi.Scores(x.data_ptr(), 0, 0, x.stride()[:2]), draft=_cabi.Scores(d.data_ptr(), 0, 0, d.stride()[:2]), rows=2, tokens=3, vocab=1000, drafted=given["tokens"].data_ptr(),
             uniform=given["uniform"].data_ptr(), a=outs[0].data_ptr(), b=outs[1].data_ptr(), f=outs[2].data_ptr(), at=space.data_ptr(), size=n):
        return lib.kb200_cache_verify(cache._cache, C.byref(logits) if logits else None, C.byref(draft) if draft else None, rows, tokens, vocab, drafted, None, 3, uniform, None, None, None,
                                      a, b, f, at, size, None)

    assert n > 0 and call() == 0 and call(draft=None) == 0
    assert call(logits=None) == call(logits=_cabi.Scores(None, 0, 0, (3000, 1000))) == call(logits=_cabi.Scores(x.data_ptr(), 3, 0, (3000, 1000))) == -1
    assert call(draft=_cabi.Scores(d.data_ptr() + 2, 0, 0, (3000, 1000))) == call(rows=3) == call(rows=-1) == call(tokens=513) == call(vocab=0) == call(drafted=None) == call(uniform=None) == -1
    assert call(a=None) == call(b=None) == call(f=None) == call(at=None) == call(size=n - 1) == call(at=space.data_ptr() + 8) == -1
    assert lib.kb200_cache_verify_workspace(cache._cache, 2, 513, 10) == lib.kb200_cache_verify_workspace(cache._cache, 0, 3, 10) == 0
    torch.cuda.synchronize()
    assert faults_of(cache) == 0


def test_calls_in_graphs_and_on_two_streams():
    cache = cache_of(20)
    given = drafts(20, 6, 30011, BF16, F32, 11)
    other = drafts(20, 6, 30011, BF16, F32, 12)
    want, want_other = ([x.tolist() for x in cache.verify(**g)] for g in (given, other))
    static = {k: None if v is None else v.clone() for k, v in given.items()}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache.verify(**static)
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(cache.verify(**static))
        graphs.append(graph)
    for i in range(6):
        for k, v in (given, other)[i // 2 % 2].items():
            if v is not None:
                static[k].copy_(v)
        graphs[i % 2].replay()
        assert [x.tolist() for x in outs[i % 2]] == (want, want_other)[i // 2 % 2]
    streams, got = [torch.cuda.Stream() for _ in range(2)], [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                got[i].append(cache.verify(**(given, other)[i]))
    torch.cuda.synchronize()
    assert all([x.tolist() for x in r] == (want, want_other)[i] for i in range(2) for r in got[i])
    assert faults_of(cache) == 0


def test_rows_by_row_and_all_at_once():
    """As many CTAs to a row as there are few rows: the same tokens."""
    rows = 200
    cache = cache_of(rows)
    given = drafts(rows, 4, 10007, BF16, F32, 13)
    want = [x.tolist() for x in cache.verify(**given)]
    for b in range(0, rows, 23):
        one = cache.verify(**{k: None if v is None else v[b:b + 1] for k, v in given.items()}, slots=ints([b]))
        assert [x[b].tolist() for x in one] == [x[b] for x in want]

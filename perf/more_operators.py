"""More operators of the paged K/V cache (``kiln_b200.cache.PagedCache``) as calls to be timed: what a server needs whose sequences grow
past what it wants to keep, and whose tokens are drafted.

A case is one kind of call at one size: attention to a sliding window and a few first tokens (with the logarithms of the rows' sums), freeing the pages that
such a window has left, adding up what weight the tokens of a sequence draw, evicting all but the heaviest of them, and verifying drafted tokens
against the model's logits.  ``run`` computes it with elementary torch operations, or, where ``own`` is true, with the framework's operators.
"""

import os
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def listed():
    return [
        # One token of a GPT-2-small layer over a window of its sequence, exact: the smallest call, all latency.
        dict(name="window_token_fp32", kind="window", dtype="float32", rows=1, tokens=1, ragged=False, heads=12, kv_heads=12, head_dim=64,
             page_tokens=16, length=700, window=256, sinks=4, tree="chain", released=False),
        # Ordinary decoding of a batch of long sequences whose pages behind the window were given back.
        dict(name="window_decode_bf16", kind="window", dtype="bfloat16", rows=32, tokens=1, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page_tokens=64, length=32768, window=4096, sinks=64, tree="chain", released=True),
        # Pieces of prompts, many query rows to a key: the largest attention.
        dict(name="window_prompt_bf16", kind="window", dtype="bfloat16", rows=8, tokens=512, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page_tokens=64, length=8192, window=1024, sinks=4, tree="chain", released=False),
        # A few sequences of ordinary length step past a page.
        dict(name="release_small", kind="release", sequences=8, page_tokens=64, length=4096, window=512, sinks=4),
        # A server's batch of long sequences after their prompts: most of a large table goes.
        dict(name="release_batch", kind="release", sequences=64, page_tokens=16, length=32768, window=2048, sinks=64),
        # One token's weights over a sequence of a GPT-2-small layer.
        dict(name="weigh_token_fp32", kind="weigh", dtype="float32", rows=1, tokens=1, ragged=False, heads=12, kv_heads=12, head_dim=64,
             page_tokens=16, length=900),
        # The last tokens of a batch of prompts weigh what is before them.
        dict(name="weigh_batch_bf16", kind="weigh", dtype="bfloat16", rows=32, tokens=4, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page_tokens=64, length=8192),
        # A sequence of GPT-2-small gives up half of its tokens.
        dict(name="evict_small", kind="evict", dtype="float32", rows=1, ragged=False, layers=12, kv_heads=12, head_dim=64, page_tokens=16,
             length=1000, keep=500, recent=64, sinks=4),
        # A batch of prompts is cut to a quarter.
        dict(name="evict_batch", kind="evict", dtype="bfloat16", rows=16, ragged=True, layers=8, kv_heads=8, head_dim=128, page_tokens=64,
             length=4096, keep=1024, recent=128, sinks=4),
        # One sequence's looked-up draft (no probabilities of its own) against GPT-2's vocabulary.
        dict(name="verify_small", kind="verify", dtype="float32", draft="none", rows=1, tokens=5, ragged=False, vocab=50257, tree="chain", greedy=0.0),
        # Trees of a small model's tokens, some rows without chance.
        dict(name="verify_trees", kind="verify", dtype="float16", draft="float16", rows=8, tokens=12, ragged=True, vocab=50257, tree="each", greedy=0.25),
        # A server's batch with a large vocabulary.
        dict(name="verify_batch", kind="verify", dtype="bfloat16", draft="float32", rows=64, tokens=8, ragged=True, vocab=128000, tree="chain", greedy=0.0),
    ]


def draw(rng):
    def between(lo, hi):                                   # spread over the logarithm
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["window", "window", "window", "release", "weigh", "weigh", "evict", "verify", "verify", "verify"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[dtype]
    page_tokens = rng.choice([8, 16, 32, 64, 128])
    if kind == "verify":
        rows, tokens, vocab = between(1, 64), rng.choice([1, between(2, 24), between(2, 24)]), between(1000, 200000)
        while rows > 1 and rows * tokens * vocab > 6.5e7:
            rows = (rows + 1) // 2
        return dict(kind=kind, dtype=dtype, draft=rng.choice(["none", "float32", dtype]), rows=rows, tokens=tokens, ragged=rng.random() < 0.7, vocab=vocab,
                    tree=rng.choice(["chain", "chain", "each"]), greedy=rng.choice([0.0, 0.0, 0.3]))
    if kind == "release":
        sequences, length = between(1, 64), between(100, 32768)
        return dict(kind=kind, sequences=sequences, page_tokens=page_tokens, length=length, window=between(16, 4096), sinks=rng.choice([0, 1, 4, between(1, 128)]))
    kv_heads, head_dim = rng.choice([1, 2, 4, 5, 8, 12]), rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
    if kind == "evict":
        layers = rng.choice([1, 2, 4, 8, 12])
        page = 2 * layers * kv_heads * head_dim * page_tokens * size
        rows, length = between(1, 32), between(64, 6000)
        while rows > 1 and rows * (length // page_tokens + 2) * page > 1.5e9:
            rows = (rows + 1) // 2
        while length > 64 and rows * (length // page_tokens + 2) * page > 1.5e9:
            length = length * 3 // 4
        return dict(kind=kind, dtype=dtype, rows=rows, ragged=rng.random() < 0.7, layers=layers, kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens,
                    length=length, keep=between(8, max(9, length // 2)), recent=rng.choice([0, 1, between(1, 200)]), sinks=rng.choice([0, 1, 4, between(1, 64)]))
    group = rng.choice([1, 1, 2, 3, 4, 8])
    rows, length = between(1, 64), between(1, 16384)
    if kind == "weigh":
        tokens = rng.choice([1, 1, between(2, 32)])
        while rows > 1 and rows * (length + tokens) * kv_heads * head_dim * size * max(1.0, tokens * group / 16) > 2.5e8:
            rows = (rows + 1) // 2
        while length > 64 and rows * (length + tokens) * kv_heads * head_dim * size * max(1.0, tokens * group / 16) > 2.5e8:
            length = length * 3 // 4
        return dict(kind=kind, dtype=dtype, rows=rows, tokens=tokens, ragged=rng.random() < 0.7, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                    page_tokens=page_tokens, length=length)
    tokens, window, sinks = rng.choice([1, 1, between(2, 64), between(65, 600)]), between(1, 8192), rng.choice([0, 1, 4, between(1, 200)])
    seen = min(length, window + sinks) + tokens
    while rows > 1 and rows * seen * kv_heads * head_dim * size * max(1.0, tokens * group / 128) > 3e8 * (0.25 if size == 4 and tokens > 64 else 1):
        rows = (rows + 1) // 2
    tree = rng.choice(["chain", "chain", "shared", "each"]) if tokens <= 64 else "chain"
    return dict(kind=kind, dtype=dtype, rows=rows, tokens=tokens, ragged=rng.random() < 0.7, heads=kv_heads * group, kv_heads=kv_heads, head_dim=head_dim,
                page_tokens=page_tokens, length=length, window=window, sinks=sinks, tree=tree, released=rng.random() < 0.5)


# ---- what a case's program holds: numbers that the host knows ------------------------------------

def _dice(case):
    """The case's own dice: its lengths and counts do not depend on the seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _lengths(case, n):
    dice = _dice(case)
    if not case.get("ragged", True):
        return [case["length"]] * n
    lengths = [case["length"]] + [dice.randint(case["length"] // 8, case["length"]) for _ in range(n - 1)]
    dice.shuffle(lengths)
    return lengths


def _counts(case, n):
    dice = _dice(case)
    dice.random()
    return [dice.randint(1, case["tokens"]) if case["ragged"] and i else case["tokens"] for i in range(n)]


def _parents(case, n):
    """The drafted token that each drafted token follows: the first is the sequence's next, and the others follow it."""
    T, dice = case["tokens"], _dice(case)
    if case["tree"] == "chain":
        return [list(range(-1, T - 1))] * n
    one = [dice.randint(max(0, i - 4), i - 1) if i else -1 for i in range(T)]
    return [one if case["tree"] == "shared" else [dice.randint(max(0, i - 4), i - 1) if i else -1 for i in range(T)] for _ in range(n)]


def _places(parents):
    """How far each drafted token is behind the committed ones."""
    places = []
    for p in parents:
        places.append(places[p] + 1 if p >= 0 else 0)
    return places


def _ancestors(parents):
    sees = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def _keeps(case):
    """How many tokens each sequence keeps: half at most (see the weights in _inputs), or all."""
    dice = _dice(case)
    dice.random()
    keeps = [case["keep"] if not case["ragged"] else dice.randint(max(1, case["keep"] // 2), case["keep"]) for _ in range(case["rows"])]
    return [k if k >= a else max(1, min(k, (a + case["sinks"]) // 2)) for k, a in zip(keeps, _lengths(case, case["rows"]))]


def _on(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values)).to(dtype).cuda()


def _table(rows, spare=0):
    """A table with the pages of each row; as wide as the longest, and some."""
    width = max([len(r) for r in rows]) + spare
    return np.array([r + [-1] * (width - len(r)) for r in rows], np.int32).reshape(len(rows), width)


def _normal(shape, dtype, generator, std=1.0):
    return torch.empty(shape, dtype=_TYPES[dtype], device="cuda").normal_(0.0, std, generator=generator)


def _pages_of(case, lengths, counts, numbers, released=False):
    """A table of pages in any order, and how many there are."""
    P, rows, places = case["page_tokens"], [], []
    for s, (a, c) in enumerate(zip(lengths, counts)):
        rows.append([-1] * -(-(a + c) // P))
        for k in range(len(rows[s])):
            if not released or k * P < case["sinks"] or (k + 1) * P > a - case["window"] + 1:
                places.append((s, k))
    for page, at in enumerate(numbers.permutation(len(places))):
        s, k = places[at]
        rows[s][k] = page
    return rows, len(places)


def _scores(case, s, b, head):
    """Scores of a sequence's tokens for the query rows that share a key head, in 64 bits: [tokens, group, keys]."""
    length, count, group, P = s["host_lengths"][b], s["host_counts"][b], case["heads"] // case["kv_heads"], case["page_tokens"]
    pages = s["table"][b, :-(-(length + count) // P)].long()
    keys = s["pool"][0, 0][pages, head].reshape(-1, case["head_dim"])[:length + count].double()
    scores = s["q"][b, :count, head * group:(head + 1) * group].double() @ keys.T / case["head_dim"] ** 0.5
    behind = torch.arange(length + count, device=keys.device) > length + torch.arange(count, device=keys.device)[:, None]
    return scores.masked_fill(behind[:, None, :], float("-inf"))


def _inputs(case, seed):
    """The inputs of a case: the cache's tensors and the call's."""
    generator = torch.Generator("cuda").manual_seed(seed)
    numbers = np.random.default_rng(seed)
    kind = case["kind"]
    if kind in ("window", "weigh"):
        n, T, D = case["rows"], case["tokens"], case["head_dim"]
        lengths, counts = _lengths(case, n), _counts(case, n)
        rows, pages = _pages_of(case, lengths, counts, numbers, case.get("released", False))
        state = dict(pool=_normal((1, 2, pages, case["kv_heads"], case["page_tokens"], D), case["dtype"], generator), table=_on(_table(rows)),
                     held=_on([len(r) for r in rows]), lengths=_on(lengths), refs=torch.ones(pages, dtype=torch.int32, device="cuda"), counts=_on(counts),
                     q=_normal((n, T, case["heads"], D), case["dtype"], generator, 2.0), host_lengths=lengths, host_counts=counts)
        if kind == "weigh":
            lse = torch.full((n, T, case["heads"]), float("-inf"), dtype=torch.float64, device="cuda")
            group = case["heads"] // case["kv_heads"]
            for b in range(n):
                for g in range(case["kv_heads"]):
                    lse[b, :counts[b], g * group:(g + 1) * group] = torch.logsumexp(_scores(case, state, b, g), -1)
            before = torch.empty(n, state["table"].shape[1] * case["page_tokens"], device="cuda").exponential_(generator=generator)
            return dict(state, lse=lse.float(), before=before)
        mask = places = None
        if case["tree"] != "chain":
            parents = _parents(case, n)
            trees = np.stack([_ancestors(p) for p in parents])
            mask = _on(trees[0] if case["tree"] == "shared" else trees, torch.bool)
            places = _on([_places(p) for p in parents])
        return dict(state, mask=mask, places=places)
    if kind == "release":
        n, P = case["sequences"], case["page_tokens"]
        lengths = _lengths(case, n)
        rows, pages = _pages_of(case, lengths, [0] * n, numbers)
        return dict(pool=torch.zeros(1, 2, pages, 1, P, 16, dtype=torch.bfloat16, device="cuda"), table=_on(_table(rows, 1)), held=_on([len(r) for r in rows]),
                    lengths=_on(lengths), refs=torch.ones(pages, dtype=torch.int32, device="cuda"))
    if kind == "evict":
        n, P = case["rows"], case["page_tokens"]
        lengths = _lengths(case, n)
        rows, pages = _pages_of(case, lengths, [0] * n, numbers)
        shape = (case["layers"], 2, pages, case["kv_heads"], P, case["head_dim"])
        table, keeps = _on(_table(rows, 1)), _on(_keeps(case))
        # (The tokens in the places that the kept ones go to are light, but for the first ones, which stay: all that is kept lies behind, so that a pass finds it
        # where the last pass did.)
        weights = torch.empty(n, table.shape[1] * P, device="cuda").exponential_(generator=generator)
        at = torch.arange(weights.shape[1], device="cuda")
        weights = torch.where((at < keeps[:, None]) & (at >= case["sinks"]), weights * 1e-9, weights + 1e-6)
        weights = torch.where(at < _on(lengths)[:, None], weights, 0.0)
        return dict(pool=_normal(shape, case["dtype"], generator), table=table, held=_on([len(r) for r in rows]), lengths=_on(lengths),
                    refs=torch.ones(pages, dtype=torch.int32, device="cuda"), weights=weights, keep=keeps)
    n, T, V = case["rows"], case["tokens"], case["vocab"]
    dice = _dice(case)
    temperature = [0.0 if dice.random() < case["greedy"] else dice.choice([0.6, 0.8, 1.0]) for _ in range(n)]
    parents = np.array(_parents(case, n), np.int32).reshape(n, T)
    logits = _normal((n, T, V), case["dtype"], generator, 2.5)
    tokens = torch.randint(0, V, (n, T), device="cuda", generator=generator)
    draft = None
    if case["draft"] != "none":
        draft = torch.empty((n, T, V), dtype=_TYPES[case["draft"]], device="cuda")
    for b in range(n):                                     # a small model that knows much of what the large one does
        q = torch.softmax(logits[b].float() / max(temperature[b], 0.5) + torch.empty(T, V, device="cuda").normal_(0.0, 0.7, generator=generator), -1)
        if draft is None:
            of = q.argmax(-1)[_on(parents[b]).long().clamp_min(0)]
        else:
            draft[b] = q.to(draft.dtype)
            of = torch.multinomial(q[_on(parents[b]).long().clamp_min(0)], 1, generator=generator)[:, 0]
        tokens[b, 1:] = of[1:]
    return dict(logits=logits, tokens=tokens.int(), draft=draft, parents=_on(parents) if case["tree"] != "chain" else None, counts=_on(_counts(case, n)),
                temperature=_on(temperature, torch.float32), uniform=torch.rand(n, T, device="cuda", generator=generator))


_CACHE = ("pool", "table", "held", "lengths", "refs")


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] in ("release", "evict"):
        state["start"] = {name: state[name].clone() for name in ("table", "held", "lengths", "refs")}
    if own:
        sys.path.insert(1, os.path.join(os.getcwd(), "kiln-compiler_b200"))
        from kiln_b200.cache import PagedCache

        if case["kind"] == "verify":
            state["cache"] = PagedCache(layers=1, sequences=case["rows"], max_pages=1, pages=1, kv_heads=1, head_dim=16)
            return state
        pool = state["pool"]
        cache = PagedCache(layers=pool.shape[0], sequences=state["table"].shape[0], max_pages=state["table"].shape[1], pages=pool.shape[2],
                           kv_heads=pool.shape[3], page_tokens=pool.shape[4], head_dim=pool.shape[5], dtype=pool.dtype)
        for name in _CACHE:
            getattr(cache, name).copy_(state[name])
            del state[name]
        state["cache"] = cache
    return state


def run(state):
    kind = state["case"]["kind"]
    return (_run_own if "cache" in state else _run_plain)[kind](state)


# ---- the framework's operators -----------------------------------------------------------------

def _own_window(state):
    case, q = state["case"], state["q"]
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device)
    out = state["cache"].attend(0, q, mask=state["mask"], counts=state["counts"], window=case["window"], sinks=case["sinks"], places=state["places"], lse=lse)
    return out, lse


def _own_start(state):
    for name, tensor in state["start"].items():           # (a pass begins where the last one began)
        getattr(state["cache"], name).copy_(tensor)


def _own_release(state):
    cache = state["cache"]
    _own_start(state)
    cache.release(state["case"]["window"], state["case"]["sinks"])
    return {name: getattr(cache, name) for name in _CACHE[1:]}


def _own_weigh(state):
    return state["cache"].weigh(0, state["q"], state["lse"], state["before"], counts=state["counts"])


def _own_evict(state):
    cache, case = state["cache"], state["case"]
    _own_start(state)
    weights = cache.evict(state["weights"], state["keep"], recent=case["recent"], sinks=case["sinks"])
    return dict({name: getattr(cache, name) for name in _CACHE}, weights=weights)


def _own_verify(state):
    return state["cache"].verify(state["logits"], state["tokens"], state["uniform"], draft=state["draft"], parents=state["parents"], counts=state["counts"],
                                 temperature=state["temperature"])


_run_own = dict(window=_own_window, release=_own_release, weigh=_own_weigh, evict=_own_evict, verify=_own_verify)


# ---- the plain forms -----------------------------------------------------------------------------

def _attention_rows(s, rows):
    """Queries of some batch rows by key head, [rows, kv_heads, group * tokens, head_dim]."""
    n, T, H, D = s["q"].shape
    Hk = s["pool"].shape[3]
    return s["q"][rows].float().view(-1, T, Hk, H // Hk, D).permute(0, 2, 3, 1, 4).reshape(-1, Hk, H // Hk * T, D)


def _read(s, which, rows, at, there):
    """K or V of positions at [rows, n] of some batch rows, zeros where there is none: [rows, kv_heads, n, head_dim]."""
    P, M = s["pool"].shape[4], s["table"].shape[1]
    page = s["table"][rows].gather(1, (at // P).clamp(0, M - 1)).clamp_min(0).long()
    x = s["pool"][0, which][page, :, at % P].transpose(1, 2).float()
    return torch.where(there[:, None, :, None], x, 0.0)


def _plain_window(s):
    case, q, device = s["case"], s["q"], s["q"].device
    n, T, H, D = q.shape
    Hk = s["pool"].shape[3]
    G, window, sinks = H // Hk, case["window"], case["sinks"]
    drafted = torch.arange(T, device=device)
    places = s["places"].long() if s["places"] is not None else drafted.expand(n, T)
    mask = s["mask"] if s["mask"] is not None else drafted[None, :] <= drafted[:, None]
    near = min(window - 1, max(s["host_lengths"])) + T     # keys in front of a sequence's end that may be in a window
    out, lse = torch.zeros_like(q), torch.empty(n, T, H, device=device)
    piece = max(1, int(2 ** 28 / (Hk * (sinks + near) * max(D, G * T))))
    for b in range(0, n, piece):
        rows = slice(b, b + piece)
        length, count = s["lengths"][rows].long()[:, None], s["counts"][rows].long()[:, None]
        m, end = length.shape[0], length + count
        begin = (length - (window - 1)).clamp_min(0)
        first = torch.arange(sinks, device=device).expand(m, sinks)
        last = begin + torch.arange(near, device=device)
        at = torch.cat([first, last], 1)
        there = torch.cat([first < torch.minimum(begin, end), last < end], 1)
        k, v = (_read(s, i, rows, at, there) for i in range(2))
        score = (_attention_rows(s, rows) @ k.transpose(-1, -2)) * D ** -0.5
        j = at - length                                    # which drafted token
        tree = (mask[rows] if mask.dim() == 3 else mask.expand(m, T, T)).gather(2, j.clamp(0, T - 1)[:, None, :].expand(m, T, at.shape[1]))
        inside = (at < sinks)[:, None, :] | (at[:, None, :] > (length + places[rows])[:, :, None] - window)
        sees = torch.where((j < 0)[:, None, :], inside, tree & (inside if s["mask"] is None else True)) & there[:, None, :] & (drafted < count)[:, :, None]
        sees = sees[:, None, None].expand(m, Hk, G, T, at.shape[1]).reshape(m, Hk, G * T, at.shape[1])
        score = torch.where(sees, score, float("-inf"))
        top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
        e = torch.exp(score - top)
        total = e.sum(-1, keepdim=True)
        o = torch.where(total > 0, (e @ v) / total, 0.0)
        out[rows] = o.view(m, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(m, T, H, D).to(q.dtype)
        lse[rows] = torch.where(total > 0, top + torch.log(total), float("-inf")).view(m, Hk, G, T).permute(0, 3, 1, 2).reshape(m, T, H)
    return out, lse


def _plain_weigh(s):
    q, device = s["q"], s["q"].device
    n, T, H, D = q.shape
    Hk = s["pool"].shape[3]
    G, N = H // Hk, s["before"].shape[1]
    drafted, weights = torch.arange(T, device=device), s["before"].clone()
    piece = max(1, int(2 ** 28 / (Hk * N * max(D, G * T))))
    for b in range(0, n, piece):
        rows = slice(b, b + piece)
        length, count = s["lengths"][rows].long()[:, None], s["counts"][rows].long()[:, None]
        m = length.shape[0]
        at = torch.arange(N, device=device).expand(m, N)
        k = _read(s, 0, rows, at, at < length + count)
        score = (_attention_rows(s, rows) @ k.transpose(-1, -2)) * D ** -0.5
        lse = s["lse"][rows].view(m, T, Hk, G).permute(0, 2, 3, 1).reshape(m, Hk, G * T, 1)
        sees = (at[:, None, :] <= (length + drafted)[:, :, None]) & (drafted < count)[:, :, None]
        sees = sees[:, None, None].expand(m, Hk, G, T, N).reshape(m, Hk, G * T, N)
        weights[rows] += torch.where(sees, torch.exp(score - lse), 0.0).sum((1, 2))
    return weights


def _plain_start(s):
    for name, tensor in s["start"].items():
        s[name].copy_(tensor)


def _free(s, gone):
    """Gives the pages of a table's marked entries back."""
    pages = s["refs"].numel()
    at = torch.where(gone & (s["table"] >= 0), s["table"], pages).long().reshape(-1)
    s["refs"].sub_(torch.zeros(pages + 1, dtype=torch.int32, device=at.device).scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:pages])
    s["table"].copy_(torch.where(gone, -1, s["table"]))


def _plain_release(s):
    _plain_start(s)
    P, window, sinks = s["pool"].shape[4], s["case"]["window"], s["case"]["sinks"]
    k = torch.arange(s["table"].shape[1], device=s["table"].device)
    _free(s, (k * P >= sinks) & ((k + 1) * P <= (s["lengths"] - window + 1)[:, None]))
    return {name: s[name] for name in _CACHE[1:]}


def _plain_evict(s):
    _plain_start(s)
    case, P, M = s["case"], s["pool"].shape[4], s["table"].shape[1]
    length = s["lengths"].long()[:, None]
    keep = torch.minimum(s["keep"].long()[:, None], length)
    at = torch.arange(s["weights"].shape[1], device=length.device)
    first = torch.clamp(keep, max=case["sinks"])
    last = torch.clamp(keep - first, max=case["recent"])
    rank = torch.where(at < length, s["weights"], float("-inf"))
    rank = torch.where((at >= length - last) & (at < length), float("inf"), rank)
    rank = torch.where(at < first, float("inf"), rank)
    heaviest = torch.sort(rank, dim=1, descending=True, stable=True).indices
    n = int(min(case["keep"], s["weights"].shape[1]))
    kept = torch.where(at[:n] < keep, heaviest[:, :n], s["weights"].shape[1]).sort(1).values
    there = at[:n] < keep
    source = torch.where(there, kept, 0)
    seq, i = there.nonzero(as_tuple=True)
    to_page, from_page = s["table"][seq, i // P].long(), s["table"][seq, source[seq, i] // P].long()
    for layer in s["pool"]:
        for pool in layer:
            pool[to_page, :, i % P] = pool[from_page, :, source[seq, i] % P]
    weights = torch.zeros_like(s["weights"])
    weights[:, :n] = torch.where(there, s["weights"].gather(1, source), 0.0)
    s["lengths"].copy_(keep[:, 0])
    held = torch.minimum(s["held"], (s["lengths"] + P - 1) // P)
    _free(s, torch.arange(M, device=at.device) >= held[:, None])
    s["held"].copy_(held)
    return dict({name: s[name] for name in _CACHE}, weights=weights)


def _plain_verify(s):
    logits, tokens, uniform, draft = s["logits"], s["tokens"].long(), s["uniform"].double(), s["draft"]
    n, T, V = logits.shape
    row, vocabulary = torch.arange(n, device=logits.device), torch.arange(V, device=logits.device)
    warm, temperature = s["temperature"][:, None] > 0, s["temperature"].double()[:, None]

    def of(at):                                            # what follows a token of each row
        x = logits[row, at].double()
        return torch.where(warm, torch.softmax(x / torch.where(warm, temperature, 1.0), -1), (vocabulary == x.argmax(-1, keepdim=True)).double())

    at = torch.zeros(n, dtype=torch.long, device=logits.device)
    parents = s["parents"].long() if s["parents"] is not None else (torch.arange(T, device=logits.device) - 1).expand(n, T)
    accepted, steps = torch.full((n, T), -1, dtype=torch.int32, device=logits.device), torch.ones(n, dtype=torch.long, device=logits.device)
    accepted[:, 0] = 0
    left, total = of(at), torch.ones(n, 1, dtype=torch.float64, device=logits.device)
    for c in range(1, T):
        asked, x = (parents[:, c] == at) & (c < s["counts"]), tokens[:, c:c + 1]
        chance = left.gather(1, x)
        q = draft[row, at].double() if draft is not None else torch.ones(n, 1, dtype=torch.float64, device=logits.device)
        taken = asked & (uniform[:, c:c + 1] * torch.where(warm, q.gather(1, x) if draft is not None else q, 1.0) * total < chance)[:, 0]
        without = left * (vocabulary != x)
        if draft is not None:
            without = torch.where(warm, (left / total - q).clamp_min(0.0), without)
        rest = without.sum(-1, keepdim=True)
        refused = (asked & ~taken)[:, None] & (rest > 0)
        at = torch.where(taken, c, at)
        left = torch.where(taken[:, None], of(at), torch.where(refused, without, left))
        total = torch.where(taken[:, None], 1.0, torch.where(refused, rest, total))
        accepted[row, torch.where(taken, steps, T - 1)] = torch.where(taken, c, accepted[:, T - 1].long()).int()
        steps += taken
    sums = left.cumsum(-1)
    following = torch.searchsorted(sums, uniform[:, :1] * sums[:, -1:], right=True)[:, 0].clamp_max(V - 1)
    return steps.int(), accepted, following.int()


_run_plain = dict(window=_plain_window, release=_plain_release, weigh=_plain_weigh, evict=_plain_evict, verify=_plain_verify)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    kind = case["kind"]
    size = 4 if case.get("dtype") == "float32" else 2
    if kind in ("window", "weigh"):
        n, P, row = case["rows"], case["page_tokens"], case["kv_heads"] * case["head_dim"] * size
        lengths, counts = _lengths(case, n), _counts(case, n)
        queries = sum(counts) * case["heads"] * case["head_dim"] * size
        if kind == "weigh":
            pairs = sum(a * c + c * (c + 1) // 2 for a, c in zip(lengths, counts))
            seen = sum(a + c for a, c in zip(lengths, counts))
            return {"bytes": row * seen + 8 * seen + 4 * seen // P + queries + 4 * sum(counts) * case["heads"], "flops": 2 * pairs * case["heads"] * case["head_dim"]}
        W, pairs, seen = case["window"], 0, 0
        for a, c, parents in zip(lengths, counts, _parents(case, n)):
            begin = max(0, a - W + 1)
            first = min(case["sinks"], begin)
            seen += first + a + c - begin
            for t, place in enumerate(_places(parents)[:c]):
                lo = max(0, a + place - W + 1)
                pairs += max(0, a - lo) + min(case["sinks"], lo, a) + (min(place + 1, W) if case["tree"] == "chain" else place + 1)
        masks = 0 if case["tree"] == "chain" else case["tokens"] ** 2 * (n if case["tree"] == "each" else 1)
        return {"bytes": 2 * row * seen + 4 * seen // P + masks + queries + n * case["tokens"] * case["heads"] * (case["head_dim"] * size + 4),
                "flops": 4 * pairs * case["heads"] * case["head_dim"]}
    if kind == "release":
        gone = sum(max(0, (a - case["window"] + 1) // case["page_tokens"] - -(-case["sinks"] // case["page_tokens"])) for a in _lengths(case, case["sequences"]))
        return {"bytes": 16 * gone + 4 * case["sequences"], "flops": 0}
    if kind == "evict":
        lengths, row = _lengths(case, case["rows"]), 2 * case["layers"] * case["kv_heads"] * case["head_dim"] * size
        kept = [min(a, k) for a, k in zip(lengths, _keeps(case))]
        moved = sum(k - min(k, case["sinks"]) for a, k in zip(lengths, kept) if k < a)
        width = -(-max(lengths) // case["page_tokens"]) * case["page_tokens"]
        return {"bytes": 2 * moved * row + 4 * sum(lengths) + 4 * case["rows"] * width, "flops": 0}
    counts, V = _counts(case, case["rows"]), case["vocab"]
    drafts = 0 if case["draft"] == "none" else case["rows"] * V * (4 if case["draft"] == "float32" else 2)      # (of the token that a row ends at)
    return {"bytes": sum(counts) * V * size + drafts + 8 * sum(counts), "flops": 3 * sum(counts) * V}


# ---- the definition, in 64 bits and by loops -----------------------------------------------------

def exact(case, seed):
    return {"window": _exact_window, "release": _exact_release, "weigh": _exact_weigh, "evict": _exact_evict, "verify": _exact_verify}[case["kind"]](case, _inputs(case, seed))


def _exact_window(case, s):
    n, T, P, D, W = case["rows"], case["tokens"], case["page_tokens"], case["head_dim"], case["window"]
    group, device = case["heads"] // case["kv_heads"], s["q"].device
    lengths, counts, parents = _lengths(case, n), _counts(case, n), _parents(case, n)
    out, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device=device), torch.full(s["q"].shape[:3], float("-inf"), dtype=torch.float64, device=device)
    for b in range(n):
        length, count = lengths[b], counts[b]
        keys = [j for j in range(length + count) if j < case["sinks"] or j > length - W]
        sees = np.zeros((count, len(keys)), bool)
        tree, places, j = _ancestors(parents[b]), _places(parents[b]), np.array(keys)
        for t in range(count):
            inside = (j < case["sinks"]) | (j > length + places[t] - W)
            known = tree[t][np.clip(j - length, 0, T - 1)] & (j >= length)
            sees[t] = np.where(j < length, inside, known & inside if case["tree"] == "chain" else known)
        at, sees = torch.tensor(keys, device=device), torch.from_numpy(sees).to(device)
        pages = s["table"][b][at // P].long()
        for g in range(case["kv_heads"]):
            k, v = (s["pool"][0, i][pages, g, at % P].double() for i in range(2))
            for h in range(g * group, (g + 1) * group):
                scores = (s["q"][b, :count, h].double() @ k.T / D ** 0.5).masked_fill(~sees, float("-inf"))
                lse[b, :count, h] = torch.logsumexp(scores, -1)
                out[b, :count, h] = torch.softmax(scores, -1) @ v
    return out, lse


def _exact_weigh(case, s):
    weights = s["before"].double()
    group = case["heads"] // case["kv_heads"]
    for b in range(case["rows"]):
        for g in range(case["kv_heads"]):
            scores = _scores(case, s, b, g)
            lse = s["lse"][b, :scores.shape[0], g * group:(g + 1) * group].double()
            weights[b, :scores.shape[-1]] += torch.exp(scores - lse[..., None]).sum((0, 1))
    return weights


class _Books:
    """The cache's tables as lists."""

    def __init__(self, s):
        self.rows, self.refs, self.lengths, self.width = s["table"].tolist(), s["refs"].tolist(), s["lengths"].tolist(), s["table"].shape[1]
        self.held = s["held"].tolist()

    def drop(self, slot, k):
        if self.rows[slot][k] >= 0:
            self.refs[self.rows[slot][k]] -= 1
        self.rows[slot][k] = -1

    def result(self):
        return dict(table=_on(self.rows), held=_on(self.held), lengths=_on(self.lengths), refs=_on(self.refs))


def _exact_release(case, s):
    books, P = _Books(s), case["page_tokens"]
    for slot, length in enumerate(books.lengths):
        for k in range(books.held[slot]):
            if all(j >= case["sinks"] and j <= length - case["window"] for j in (k * P, k * P + P - 1)):
                books.drop(slot, k)
    return books.result()


def _exact_evict(case, s):
    books, P = _Books(s), case["page_tokens"]
    weights, after = s["weights"].double().cpu().numpy(), np.zeros(s["weights"].shape)
    for slot, keep in enumerate(_keeps(case)):
        length = books.lengths[slot]
        keep = min(keep, length)
        chosen = set(range(min(case["sinks"], keep)))
        chosen |= set(range(length - min(case["recent"], keep - len(chosen)), length))
        for j in sorted(range(length), key=lambda j: (-weights[slot, j], j)):
            if len(chosen) >= keep:
                break
            chosen.add(j)
        kept = sorted(chosen)
        after[slot, :keep] = weights[slot, kept]
        to = [(books.rows[slot][i // P], i % P) for i in range(keep)]
        of = [(books.rows[slot][j // P], j % P) for j in kept]
        (to_page, to_row), (page, row) = (torch.tensor(x, device="cuda").T for x in (to, of))
        moved = s["pool"][:, :, page, :, row].clone()
        s["pool"][:, :, to_page, :, to_row] = moved
        books.lengths[slot], need = keep, -(-keep // P)
        for k in range(need, books.held[slot]):
            books.drop(slot, k)
        books.held[slot] = min(books.held[slot], need)
    return dict(books.result(), pool=s["pool"], weights=torch.from_numpy(after).cuda())


def _exact_verify(case, s):
    n, T, V = case["rows"], case["tokens"], case["vocab"]
    counts, parents = _counts(case, n), _parents(case, n)
    tokens, uniform, temperature = s["tokens"].tolist(), s["uniform"].double().tolist(), s["temperature"].double().tolist()
    steps, accepted, following = [], [], []
    for b in range(n):
        def after(i):
            x = s["logits"][b, i].double().cpu().numpy()
            if temperature[b] == 0.0:
                p = np.zeros(V)
                p[int(np.argmax(x))] = 1.0
                return p
            x = np.exp((x - x.max()) / temperature[b])
            return x / x.sum()

        path, p, whole = [0], after(0), 1.0
        for c in range(1, counts[b]):
            if parents[b][c] != path[-1]:
                continue
            q, x = None, tokens[b][c]
            if s["draft"] is not None and temperature[b] > 0:
                q = s["draft"][b, path[-1]].double().cpu().numpy()
            if uniform[b][c] * (1.0 if q is None else q[x]) * whole < p[x]:
                path.append(c)
                p, whole = after(c), 1.0
                continue
            if q is None:
                rest = p.copy()
                rest[x] = 0.0
            else:
                rest = np.maximum(p / whole - q, 0.0)
            if rest.sum() > 0:
                p, whole = rest, rest.sum()
        sums = np.cumsum(p)
        steps.append(len(path))
        accepted.append(path + [-1] * (T - len(path)))
        following.append(min(V - 1, int(np.searchsorted(sums, uniform[b][0] * sums[-1], side="right"))))
    return _on(steps), _on(accepted), _on(following)

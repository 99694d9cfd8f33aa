"""The operators of the paged K/V cache (``kiln_b200.cache.PagedCache``) as calls to be timed.

A case is one kind of call at one size: the attention of drafted tokens over a cache, a step of beam search (fork the
sequences, make their next page their own), a step of drafting (roll back, make room, write K and V, keep what was accepted) and the compaction
of a cache's pages.  ``run`` computes it with elementary torch operations, or, where ``own`` is true, with the framework's operators.
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
        # One token of a GPT-2-small layer in the precision its modules have by default: the smallest call, all latency.
        dict(name="attend_token_fp32", kind="attend", dtype="float32", rows=1, tokens=1, ragged=False, heads=12, kv_heads=12, head_dim=64,
             page_tokens=16, length=128, tree="chain", chosen=False),
        # A server's batch of such sequences, a few drafted tokens each, still exact.
        dict(name="attend_tree_fp32", kind="attend", dtype="float32", rows=8, tokens=9, ragged=True, heads=12, kv_heads=12, head_dim=64,
             page_tokens=16, length=2000, tree="each", chosen=False),
        # Ordinary decoding of a batch of long sequences: one token each, heads that share keys.
        dict(name="attend_decode_bf16", kind="attend", dtype="bfloat16", rows=32, tokens=1, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page_tokens=64, length=8192, tree="chain", chosen=False),
        # One sequence at a desk, a wide tree drafted by a small model.
        dict(name="attend_tree_fp16", kind="attend", dtype="float16", rows=1, tokens=63, ragged=False, heads=32, kv_heads=8, head_dim=128,
             page_tokens=32, length=4097, tree="shared", chosen=False),
        # Sizes on no tile: heads of 80, three to a key head, rows that name their sequences.
        dict(name="attend_odd_bf16", kind="attend", dtype="bfloat16", rows=5, tokens=6, ragged=True, heads=15, kv_heads=5, head_dim=80,
             page_tokens=16, length=777, tree="each", chosen=True),
        # The largest: a full batch, trees of 32 tokens over long contexts.
        dict(name="attend_batch_bf16", kind="attend", dtype="bfloat16", rows=32, tokens=32, ragged=True, heads=32, kv_heads=8, head_dim=128,
             page_tokens=128, length=16384, tree="each", chosen=False),
        # Four beams of two prompts over GPT-2-small's layers.
        dict(name="beams_small", kind="beams", dtype="float32", families=2, width=4, tokens=1, layers=12, kv_heads=12, head_dim=64,
             page_tokens=16, length=200),
        # A batch of prompts with eight beams each.
        dict(name="beams_batch", kind="beams", dtype="bfloat16", families=16, width=8, tokens=1, layers=12, kv_heads=8, head_dim=128,
             page_tokens=64, length=1000),
        # One sequence drafts five tokens; K and V come as a float32 module returns them.
        dict(name="draft_small", kind="draft", dtype="bfloat16", input="float32", rows=1, tokens=5, ragged=False, layers=12, kv_heads=12,
             head_dim=64, page_tokens=16, length=301),
        # A batch drafts trees of 16 and keeps what was accepted.
        dict(name="draft_batch", kind="draft", dtype="bfloat16", input="bfloat16", rows=64, tokens=16, ragged=True, layers=8, kv_heads=8,
             head_dim=128, page_tokens=64, length=500),
        # A small cache with holes between its pages.
        dict(name="compact_small", kind="compact", dtype="float32", sequences=6, pages=96, layers=12, kv_heads=12, head_dim=64, page_tokens=16,
             used=0.6),
        # A server's pool of which half was given back here and there.
        dict(name="compact_pool", kind="compact", dtype="bfloat16", sequences=64, pages=1024, layers=8, kv_heads=8, head_dim=128, page_tokens=64,
             used=0.5),
    ]


def draw(rng):
    def between(lo, hi):                                   # spread over the logarithm
        return int(round(lo * (hi / lo) ** rng.random()))

    kind = rng.choice(["attend", "attend", "attend", "beams", "draft", "compact"])
    dtype = rng.choice(["float32", "bfloat16", "bfloat16", "float16"])
    size = {"float32": 4, "bfloat16": 2, "float16": 2}[dtype]
    if kind == "attend":
        kv_heads = rng.choice([1, 2, 4, 5, 8, 12])
        group = rng.choice([1, 1, 2, 3, 4, 8])
        head_dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 192, 256])
        tokens = rng.choice([1, 1, between(2, 64), between(2, 64), between(65, 300)])
        rows, length = between(1, 64), between(1, 16384)
        # no more bytes and products than the largest listed case
        while rows > 1 and rows * (length + tokens) * kv_heads * head_dim * size * max(1.0, tokens * group / 128) > 5e8:
            rows = (rows + 1) // 2
        while length > 64 and rows * (length + tokens) * kv_heads * head_dim * size * max(1.0, tokens * group / 128) > 5e8:
            length = length * 3 // 4
        return dict(kind=kind, dtype=dtype, rows=rows, tokens=tokens, ragged=rng.random() < 0.7, heads=kv_heads * group, kv_heads=kv_heads,
                    head_dim=head_dim, page_tokens=rng.choice([8, 16, 32, 64, 128]), length=length,
                    tree=rng.choice(["chain", "shared", "each"]), chosen=rng.random() < 0.4)
    layers, kv_heads = rng.choice([1, 2, 4, 8, 12]), rng.choice([1, 2, 4, 8, 12])
    head_dim, page_tokens = rng.choice([32, 64, 80, 128]), rng.choice([8, 16, 32, 64, 128])
    page = 2 * layers * kv_heads * head_dim * page_tokens * size
    if kind == "beams":
        families, width, length = between(1, 16), between(2, 8), between(1, 1500)
        while families > 1 and families * (length // page_tokens + 2 * width) * page > 1.2e9:
            families = (families + 1) // 2
        return dict(kind=kind, dtype=dtype, families=families, width=width, tokens=rng.choice([1, 1, between(2, 40)]), layers=layers,
                    kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens, length=length)
    if kind == "draft":
        rows, tokens, length = between(1, 64), between(1, 64), between(1, 700)
        while rows > 1 and rows * ((length + tokens) // page_tokens + 2) * page > 1.2e9:
            rows = (rows + 1) // 2
        return dict(kind=kind, dtype=dtype, input=rng.choice([dtype, "float32"]), rows=rows, tokens=tokens, ragged=rng.random() < 0.7, layers=layers,
                    kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens, length=length)
    pages = min(between(24, 2048), max(24, int(2e9 / page)))
    return dict(kind=kind, dtype=dtype, sequences=between(1, 64), pages=pages, layers=layers, kv_heads=kv_heads, head_dim=head_dim,
                page_tokens=page_tokens, used=round(rng.uniform(0.1, 0.95), 2))


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
    """The drafted token that each drafted token follows, -1: the context."""
    dice = _dice(case)
    one = [dice.randint(max(-1, i - 9), i - 1) for i in range(case["tokens"])]
    return [one if case["tree"] == "shared" else [dice.randint(max(-1, i - 9), i - 1) for i in range(case["tokens"])] for _ in range(n)]


def _kept(case, n):
    """Drafted tokens that were accepted, ascending."""
    dice = _dice(case)
    dice.random()
    return [sorted(dice.sample(range(c), dice.randint(0 if i else 1, max(1, c // 3)))) for i, c in enumerate(_counts(case, n))]


def _ancestors(parents):
    sees = np.zeros((len(parents), len(parents)), bool)
    for i, p in enumerate(parents):
        if p >= 0:
            sees[i] = sees[p]
        sees[i, i] = True
    return sees


def _on(values, dtype=torch.int32):
    return torch.as_tensor(np.asarray(values)).to(dtype).cuda()


def _pool(case, pages, generator):
    shape = (case["layers"], 2, pages, case["kv_heads"], case["page_tokens"], case["head_dim"])
    return torch.empty(shape, dtype=_TYPES[case["dtype"]], device="cuda").normal_(generator=generator)


def _table(rows, spare=0):
    """A table with the pages of each row; as wide as the longest, and some."""
    width = max([len(r) for r in rows]) + spare
    return np.array([r + [-1] * (width - len(r)) for r in rows], np.int32).reshape(len(rows), width)


def _inputs(case, seed):
    """The inputs of a case: the cache's tensors and the call's."""
    generator = torch.Generator("cuda").manual_seed(seed)
    numbers = np.random.default_rng(seed)
    kind, P = case["kind"], case["page_tokens"]
    dtype = _TYPES[case["dtype"]]
    if kind == "attend":
        n, T = case["rows"], case["tokens"]
        lengths, counts = _lengths(case, n), _counts(case, n)
        slots = list(range(n))
        if case["chosen"]:                                # the sequences of a larger cache, in any order
            slots = [int(s) for s in numbers.permutation(2 * n)[:n]]
        S = 2 * n if case["chosen"] else n
        pages = sum(-(-(a + c) // P) for a, c in zip(lengths, counts))
        order = [int(p) for p in numbers.permutation(pages)]
        rows, held = [[] for _ in range(S)], [0] * S
        all_lengths = [0] * S
        for s, a, c in zip(slots, lengths, counts):
            held[s], all_lengths[s] = -(-(a + c) // P), a
            rows[s] = [order.pop() for _ in range(held[s])]
        mask = None
        if case["tree"] != "chain":
            trees = np.stack([_ancestors(p) for p in _parents(case, n)])
            mask = _on(trees[0] if case["tree"] == "shared" else trees, torch.bool)
        return dict(pool=_pool(dict(case, layers=1), pages, generator), table=_on(_table(rows)), held=_on(held), lengths=_on(all_lengths),
                    refs=torch.ones(pages, dtype=torch.int32, device="cuda"), mask=mask, counts=_on(counts), most=max(held),
                    slots=_on(slots) if case["chosen"] else None,
                    q=torch.empty(n, T, case["heads"], case["head_dim"], dtype=dtype, device="cuda").normal_(0.0, 2.0, generator=generator))
    if kind == "compact":
        used = max(1, int(case["pages"] * case["used"]))
        order = [int(p) for p in numbers.permutation(case["pages"])[:used]]
        rows = [order[s::case["sequences"]] for s in range(case["sequences"])]
        refs = np.zeros(case["pages"], np.int32)
        for row in rows:
            refs[row] += 1
        table, held = _table(rows, 1), [len(r) for r in rows]
        return dict(pool=_pool(case, case["pages"], generator), table=_on(table), held=_on(held), lengths=_on([h * P for h in held]), refs=_on(refs))
    if kind == "beams":
        S = case["families"] * case["width"]
        first = _lengths(case, case["families"])
        lengths = [first[s // case["width"]] if s % case["width"] == 0 else 0 for s in range(S)]
        counts = [case["tokens"]] * S
        room = sum(case["width"] * (-(-(a + case["tokens"]) // P) - a // P) for a in first)
    else:
        S = case["rows"]
        lengths, counts = _lengths(case, S), _counts(case, S)
        room = sum(-(-(a + c) // P) - -(-a // P) for a, c in zip(lengths, counts))
    held = [-(-a // P) for a in lengths]
    pages = sum(held) + room + 2                          # the last is one that the program keeps for itself
    order = [int(p) for p in numbers.permutation(pages - 1)]
    rows = [[order.pop() for _ in range(h)] for h in held]
    refs = np.zeros(pages, np.int32)
    for row in rows:
        refs[row] += 1
    refs[-1] = 1
    state = dict(pool=_pool(case, pages, generator), table=_on(_table(rows, -(-case["tokens"] // P) + 1)), held=_on(held), lengths=_on(lengths),
                 refs=_on(refs), counts=_on(counts))
    if kind == "beams":
        return dict(state, sources=_on([s - s % case["width"] for s in range(S)]))
    kept = _kept(case, S)
    shape = (case["layers"], S, case["tokens"], case["kv_heads"], case["head_dim"])
    k, v = (torch.empty(shape, dtype=_TYPES[case["input"]], device="cuda").normal_(generator=generator) for _ in range(2))
    return dict(state, k=k, v=v, start=state["lengths"].clone(), kept=_on(_table(kept)), n_kept=_on([len(x) for x in kept]))


_CACHE = ("pool", "table", "held", "lengths", "refs")


def prepare(case, seed):
    state = _inputs(case, seed)
    state["case"] = case
    if case["kind"] == "compact":
        state["holes"] = (state["table"].clone(), state["refs"].clone())
    if own:
        sys.path.insert(1, os.path.join(os.getcwd(), "kiln-compiler_b200"))
        from kiln_b200.cache import PagedCache

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

def _own_state(cache):
    return {name: getattr(cache, name) for name in _CACHE}


def _own_attend(state):
    return state["cache"].attend(0, state["q"], mask=state["mask"], counts=state["counts"], slots=state["slots"])


def _own_beams(state):
    cache = state["cache"]
    cache.fork(state["sources"])
    cache.reserve(state["counts"])
    return _own_state(cache)


def _own_draft(state):
    cache = state["cache"]
    cache.truncate(state["start"])                        # what an earlier draft left is rolled back
    cache.reserve(state["counts"])
    for layer in range(state["k"].shape[0]):
        cache.append(layer, state["k"][layer], state["v"][layer], counts=state["counts"])
    cache.accept(state["n_kept"], state["kept"])
    return _own_state(cache)


def _own_compact(state):
    cache = state["cache"]
    cache.table.copy_(state["holes"][0])                  # back to the snapshot with the holes (the pages that moved are still where they were)
    cache.refs.copy_(state["holes"][1])
    cache.compact()
    return _own_state(cache)


_run_own = dict(attend=_own_attend, beams=_own_beams, draft=_own_draft, compact=_own_compact)


# ---- the plain forms -----------------------------------------------------------------------------

def _plain_attend(s):
    pool, table, q = s["pool"], s["table"], s["q"]
    n, T, H, D = q.shape
    Hk, P = pool.shape[3], pool.shape[4]
    G, N = H // Hk, s["most"] * P
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(n, device=q.device)
    at, drafted = torch.arange(N, device=q.device), torch.arange(T, device=q.device)
    mask = s["mask"] if s["mask"] is not None else drafted[None, :] <= drafted[:, None]
    out = torch.zeros_like(q)
    piece = max(1, int(2 ** 28 / (Hk * N * max(D, G * T))))
    for b in range(0, n, piece):
        rows = slots[b:b + piece]
        m = rows.numel()
        length, count = s["lengths"][rows].long(), s["counts"][b:b + piece].long()
        pages = table[rows][:, :s["most"]].clamp_min(0).long()
        k, v = (pool[0, i][pages].transpose(1, 2).reshape(m, Hk, N, D).float() for i in range(2))
        k = torch.where((at < (length + count)[:, None])[:, None, :, None], k, 0.0)
        v = torch.where((at < (length + count)[:, None])[:, None, :, None], v, 0.0)
        x = q[b:b + piece].float().view(m, T, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(m, Hk, G * T, D)
        score = (x @ k.transpose(-1, -2)) * D ** -0.5
        j = at - length[:, None]                          # [m, N]: which drafted token
        trees = (mask[b:b + piece] if mask.dim() == 3 else mask.expand(m, T, T))
        sees = trees.gather(2, j.clamp(0, T - 1)[:, None, :].expand(m, T, N)) & (j >= 0)[:, None, :] & (j < count[:, None])[:, None, :]
        sees = (sees | (j < 0)[:, None, :]) & (drafted < count[:, None])[:, :, None]
        sees = sees[:, None, None].expand(m, Hk, G, T, N).reshape(m, Hk, G * T, N)
        score = torch.where(sees, score, float("-inf"))
        top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
        e = torch.exp(score - top)
        total = e.sum(-1, keepdim=True)
        o = torch.where(total > 0, (e @ v) / total, 0.0)
        out[b:b + piece] = o.view(m, Hk, G, T, D).permute(0, 3, 1, 2, 4).reshape(m, T, H, D).to(q.dtype)
    return out


def _holders(table, pages):
    at = torch.where(table >= 0, table, pages).long().reshape(-1)
    return torch.zeros(pages + 1, dtype=torch.int32, device=table.device).scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))[:pages]


def _set_table(s, table):
    pages = s["refs"].numel()
    s["refs"].add_(_holders(table, pages) - _holders(s["table"], pages))
    s["table"].copy_(table)


def _plain_fork(s, sources):
    gone = sources < 0
    source = sources.clamp_min(0).long()
    _set_table(s, torch.where(gone[:, None], -1, s["table"][source]))
    s["held"].copy_(torch.where(gone, 0, s["held"][source]))
    s["lengths"].copy_(torch.where(gone, 0, s["lengths"][source]))


def _plain_truncate(s, lengths):
    P, k = s["pool"].shape[4], torch.arange(s["table"].shape[1], device=lengths.device)
    s["lengths"].copy_(torch.minimum(s["lengths"], lengths))
    held = torch.minimum(s["held"], (s["lengths"] + P - 1) // P)
    _set_table(s, torch.where(k < held[:, None], s["table"], -1))
    s["held"].copy_(held)


def _plain_reserve(s, counts):
    pool, table, refs, lengths = s["pool"], s["table"].clone(), s["refs"].clone(), s["lengths"]
    S, M = table.shape
    N, P = refs.numel(), pool.shape[4]
    k, slot = torch.arange(M, device=table.device), torch.arange(S, device=table.device)[:, None].expand(S, M)
    first, need = lengths // P, (lengths + counts + P - 1) // P
    writes = (counts > 0)[:, None] & (k >= first[:, None]) & (k < need[:, None])
    here, page = writes & (table >= 0), table.clamp_min(0).long()
    at = torch.where(here, page, N).reshape(-1)
    writers = torch.zeros(N + 1, dtype=torch.int32, device=table.device).scatter_add_(0, at, torch.ones_like(at, dtype=torch.int32))
    lowest = torch.full((N + 1,), S, device=table.device).scatter_reduce_(0, at, slot.reshape(-1), "amin")
    mine = here & ((refs[page] == 1) | ((writers[page] == refs[page]) & (lowest[page] == slot)))
    new = writes & ~mine
    fits = (new.sum() <= (refs == 0).sum()) & (need <= M).all()
    new = new & fits
    free = torch.argsort((refs > 0).int(), stable=True)
    order = (new.reshape(-1).cumsum(0) - 1).clamp_min(0).view(S, M)
    _set_table(s, torch.where(new, free[order].int(), table))
    s["held"].copy_(torch.where((counts > 0) & fits, torch.maximum(s["held"], need), s["held"]))
    at = first.clamp_max(M - 1).long()[:, None]
    copied = new.gather(1, at)[:, 0] & (table.gather(1, at)[:, 0] >= 0) & (lengths % P > 0)
    source = torch.where(copied, table.gather(1, at)[:, 0], N - 1).long()
    target = torch.where(copied, s["table"].gather(1, at)[:, 0], N - 1).long()
    rows = (torch.arange(P, device=table.device) < torch.where(copied, lengths % P, 0)[:, None])[None, :, None, :, None]
    for layer in pool:
        layer[:, target] = torch.where(rows, layer[:, source], layer[:, target])


def _place(s, position, there):
    """Page and row of positions [S, n]; the page that nobody writes where a position is not there."""
    P, M = s["pool"].shape[4], s["table"].shape[1]
    page = s["table"].gather(1, (position // P).clamp(0, M - 1).long())
    return torch.where(there, page, s["refs"].numel() - 1).long(), (position % P).long()


def _plain_append(s, layer, k, v, counts):
    i = torch.arange(k.shape[1], device=k.device)
    there = i < counts[:, None]
    page, row = _place(s, s["lengths"][:, None] + i, there)
    for pool, new in zip(s["pool"][layer], (k, v)):
        pool[page, :, row] = torch.where(there[..., None, None], new.to(pool.dtype), pool[page, :, row])


def _plain_accept(s, n_kept, kept):
    i = torch.arange(kept.shape[1], device=kept.device)
    there = i < n_kept[:, None]
    source, source_row = _place(s, s["lengths"][:, None] + kept, there)
    target, target_row = _place(s, s["lengths"][:, None] + i, there)
    for layer in s["pool"]:
        for pool in layer:
            pool[target, :, target_row] = torch.where(there[..., None, None], pool[source, :, source_row], pool[target, :, target_row])
    s["lengths"].add_(n_kept)
    _plain_truncate(s, s["lengths"].clone())


def _plain_beams(s):
    _plain_fork(s, s["sources"])
    _plain_reserve(s, s["counts"])
    return {name: s[name] for name in _CACHE}


def _plain_draft(s):
    _plain_truncate(s, s["start"])
    _plain_reserve(s, s["counts"])
    for layer in range(s["k"].shape[0]):
        _plain_append(s, layer, s["k"][layer], s["v"][layer], s["counts"])
    _plain_accept(s, s["n_kept"], s["kept"])
    return {name: s[name] for name in _CACHE}


def _plain_compact(s):
    s["table"].copy_(s["holes"][0])
    s["refs"].copy_(s["holes"][1])
    refs, table = s["refs"], s["table"]
    page, used = torch.arange(refs.numel(), device=refs.device), s["refs"] > 0
    n_used = used.sum()
    moves, hole = used & (page >= n_used), ~used & (page < n_used)
    moving, holes = torch.argsort((~moves).int(), stable=True), torch.argsort((~hole).int(), stable=True)
    target = torch.where(moves, holes[(moves.cumsum(0) - 1).clamp_min(0)], page)
    source = torch.where(hole, moving[(hole.cumsum(0) - 1).clamp_min(0)], page)
    for layer in s["pool"]:
        layer.copy_(layer[:, source])
    refs.copy_(torch.where(page < n_used, refs[source], 0))
    table.copy_(torch.where(table >= 0, target[table.clamp_min(0).long()].int(), table))
    return {name: s[name] for name in _CACHE}


_run_plain = dict(attend=_plain_attend, beams=_plain_beams, draft=_plain_draft, compact=_plain_compact)


# ---- what a pass cannot do without ---------------------------------------------------------------

def work(case):
    size, P = (4 if case["dtype"] == "float32" else 2), case["page_tokens"]
    kind, row = case["kind"], 2 * case.get("layers", 1) * case["kv_heads"] * case["head_dim"] * size    # a token's K and V in all layers
    if kind == "attend":
        n = case["rows"]
        lengths, counts = _lengths(case, n), _counts(case, n)
        if case["tree"] == "chain":
            pairs = sum(c * (c + 1) // 2 for c in counts)
        else:
            pairs = sum(int(_ancestors(p)[:c, :c].sum()) for p, c in zip(_parents(case, n), counts))
        pairs += sum(a * c for a, c in zip(lengths, counts))
        tables = 4 * sum(-(-(a + c) // P) for a, c in zip(lengths, counts))
        masks = 0 if case["tree"] == "chain" else case["tokens"] ** 2 * (n if case["tree"] == "each" else 1)
        return {"bytes": row * sum(a + c for a, c in zip(lengths, counts)) + tables + masks
                + (sum(counts) + n * case["tokens"]) * case["heads"] * case["head_dim"] * size,
                "flops": 4 * pairs * case["heads"] * case["head_dim"]}
    if kind == "beams":
        first = _lengths(case, case["families"])
        copied = sum((case["width"] - 1) * (a % P) for a in first)
        tables = 2 * 4 * sum(case["width"] * -(-(a + case["tokens"]) // P) for a in first)
        return {"bytes": 2 * copied * row + tables, "flops": 0}
    if kind == "draft":
        n = case["rows"]
        counts, kept = _counts(case, n), _kept(case, n)
        moved = sum(sum(i != j for i, j in enumerate(x)) for x in kept)
        return {"bytes": sum(counts) * row * (1 if case["input"] == case["dtype"] else 4 // size) + sum(counts) * row + 2 * moved * row, "flops": 0}
    pages, used = case["pages"], max(1, int(case["pages"] * case["used"]))
    moved = int(used * (pages - used) / pages)            # (as many as expected of used pages anywhere)
    return {"bytes": 2 * moved * row * P + 8 * (used + pages), "flops": 0}


# ---- the definition, in 64 bits and by loops -----------------------------------------------------

def exact(case, seed):
    return {"attend": _exact_attend, "beams": _exact_beams, "draft": _exact_draft, "compact": _exact_compact}[case["kind"]](case, _inputs(case, seed))


def _exact_attend(case, s):
    q, pool, table = s["q"].double(), s["pool"], s["table"].cpu().numpy()
    n, T, H, D = q.shape
    group, P = H // case["kv_heads"], case["page_tokens"]
    slots = s["slots"].tolist() if s["slots"] is not None else range(n)
    lengths, counts, out = _lengths(case, n), _counts(case, n), torch.zeros_like(q)
    for b, slot in enumerate(slots):
        length, count = lengths[b], counts[b]
        sees = torch.ones(count, length + count, dtype=torch.bool, device=q.device)
        tree = np.tril(np.ones((T, T), bool)) if s["mask"] is None else (s["mask"] if s["mask"].dim() == 2 else s["mask"][b]).cpu().numpy()
        sees[:, length:] = torch.from_numpy(np.ascontiguousarray(tree[:count, :count])).cuda()
        pages = torch.from_numpy(table[slot][:-(-(length + count) // P)].astype(np.int64)).cuda()
        for g in range(case["kv_heads"]):
            keys, values = (pool[0, i, pages, g].reshape(-1, D)[:length + count].double() for i in range(2))
            for h in range(g * group, (g + 1) * group):
                weights = torch.softmax((q[b, :count, h] @ keys.T / D ** 0.5).masked_fill(~sees, float("-inf")), -1)
                out[b, :count, h] = weights @ values
    return out


class _Books:
    """The cache's tables as lists."""

    def __init__(self, s):
        self.pool, self.width, self.P = s["pool"], s["table"].shape[1], s["pool"].shape[4]
        self.rows = [[p for p in r if p >= 0] for r in s["table"].tolist()]
        self.lengths, self.refs = s["lengths"].tolist(), s["refs"].tolist()

    def drop(self, slot, n):
        for page in self.rows[slot][n:]:
            self.refs[page] -= 1
        self.rows[slot] = self.rows[slot][:n]

    def reserve(self, counts):
        spans = {s: range(self.lengths[s] // self.P, -(-(self.lengths[s] + c) // self.P)) for s, c in enumerate(counts) if c > 0}
        holders = {}
        for s, span in spans.items():
            for k in span:
                if k < len(self.rows[s]):
                    holders.setdefault(self.rows[s][k], []).append(s)
        free = iter([p for p, r in enumerate(self.refs) if r == 0])
        before = list(self.refs)
        for s, span in spans.items():
            for k in span:
                old = self.rows[s][k] if k < len(self.rows[s]) else None
                if old is not None and (before[old] == 1 or (len(holders[old]) == before[old] and min(holders[old]) == s)):
                    continue
                page = next(free)
                self.refs[page] += 1
                if old is None:
                    self.rows[s].append(page)
                    continue
                self.rows[s][k] = page
                self.refs[old] -= 1
                part = self.lengths[s] % self.P
                if k == self.lengths[s] // self.P and part:
                    self.pool[:, :, page, :, :part] = self.pool[:, :, old, :, :part]

    def result(self):
        return dict(pool=self.pool, table=_on([r + [-1] * (self.width - len(r)) for r in self.rows]), held=_on([len(r) for r in self.rows]),
                    lengths=_on(self.lengths), refs=_on(self.refs))


def _exact_beams(case, s):
    books = _Books(s)
    rows, lengths = [list(r) for r in books.rows], list(books.lengths)
    sources = s["sources"].tolist()
    for slot, source in enumerate(sources):
        for page in rows[source]:
            books.refs[page] += 1
    for slot, source in enumerate(sources):
        books.drop(slot, 0)
        books.rows[slot], books.lengths[slot] = list(rows[source]), lengths[source]
    books.reserve(s["counts"].tolist())
    return books.result()


def _exact_draft(case, s):
    books, P = _Books(s), case["page_tokens"]
    for slot, length in enumerate(s["start"].tolist()):
        books.lengths[slot] = min(length, books.lengths[slot])
        books.drop(slot, -(-books.lengths[slot] // P))
    books.reserve(s["counts"].tolist())
    for slot, (count, kept) in enumerate(zip(s["counts"].tolist(), _kept(case, case["rows"]))):
        def at(i):
            return books.rows[slot][(books.lengths[slot] + i) // P], (books.lengths[slot] + i) % P
        for i in range(count):
            page, row = at(i)
            books.pool[:, 0, page, :, row] = s["k"][:, slot, i].to(books.pool.dtype)
            books.pool[:, 1, page, :, row] = s["v"][:, slot, i].to(books.pool.dtype)
        for i, j in enumerate(kept):
            (page, row), (page_j, row_j) = at(i), at(j)
            books.pool[:, :, page, :, row] = books.pool[:, :, page_j, :, row_j].clone()
        books.lengths[slot] += len(kept)
        books.drop(slot, -(-books.lengths[slot] // P))
    return books.result()


def _exact_compact(case, s):
    books = _Books(s)
    used = [p for p, r in enumerate(books.refs) if r > 0]
    holes = [p for p, r in enumerate(books.refs[:len(used)]) if r == 0]
    to = dict(zip([p for p in used if p >= len(used)], holes))
    for page, hole in to.items():
        books.pool[:, :, hole] = books.pool[:, :, page]
        books.refs[hole], books.refs[page] = books.refs[page], 0
    books.rows = [[to.get(p, p) for p in r] for r in books.rows]
    return books.result()

"""A transformer block run token by token: compiled modules around the paged cache, against the whole block in float64."""

import random

import numpy as np
import pytest
import torch

from kiln_b200.codegen import program_from_plan
from kiln_b200.runtime import GPUExecutable
from oracle.plan_oracle import run_plan, scale_relative_error
from perf import cases

pytestmark = pytest.mark.gpu

HEADS, DIM = 4, 256


def modules(rows, precision):
    """What comes in front of the attention and behind it, for so many tokens at a time; the weights of the whole block."""
    p = cases._Plan("front", (rows, DIM), (rows, 3 * DIM))
    h = p.buffer(rows, DIM)
    p.layernorm(p.x, "ln1.", h)
    p.linear(h, "c_attn.", 3 * DIM, p.y)
    front = p.spec()
    p = cases._Plan("back", (rows, DIM), (rows, DIM))
    x = cases._View(("input", 1), (rows, DIM))
    x1, h2, f = p.buffer(rows, DIM), p.buffer(rows, DIM), p.buffer(rows, 4 * DIM)
    p.linear(p.x, "c_proj.", DIM, x1, residual=x)
    p.layernorm(x1, "ln2.", h2)
    p.linear(h2, "fc.", 4 * DIM, f, gelu=True)
    p.linear(f, "proj.", DIM, p.y, residual=x1)
    back = p.spec()
    back.input_shapes.append((rows, DIM))
    whole = cases._plan({"kind": "block", "tokens": 64, "heads": HEADS})
    consts = cases._constants(whole.const_shapes, np.random.default_rng(0))
    built = []
    for plan in (front, back):
        assert set(plan.const_shapes) <= set(consts) and all(consts[n].shape == tuple(s) for n, s in plan.const_shapes.items())
        built.append(GPUExecutable(program_from_plan(plan, precision), plan.arena_bytes, consts, plan.input_shapes, plan.output_shapes))
    return built[0], built[1], consts


def whole_block(x, consts):
    """The block over a sequence of tokens, in float64."""
    plan = cases._plan({"kind": "block", "tokens": len(x), "heads": HEADS})
    own = dict(consts, mask=cases._constants({"mask": (len(x), len(x))}, None)["mask"])
    (out,) = run_plan(plan.to_json(), [x], {n: own[n] for n in plan.const_shapes}, dtype=np.float64)
    return out


# float32 modules are within 1e-5 of exact each and the attention is float32 throughout: three in a row.  BF16 modules: 2e-2, the mode's own bound; keys, values and
# weights rounded to bfloat16 are within that.
@pytest.mark.parametrize("precision, dtype, tolerance", [("fp32", torch.float32, 5e-5), ("bf16", torch.bfloat16, 2e-2)])
def test_prompts_drafts_and_beams_give_what_the_whole_block_gives(precision, dtype, tolerance):
    from kiln_b200.cache import PagedCache

    sequences, width = 4, 8
    front, back, consts = modules(sequences * width, precision)
    cache = PagedCache(layers=1, sequences=sequences, max_pages=8, pages=24, kv_heads=HEADS, head_dim=DIM // HEADS, page_tokens=8, dtype=dtype)
    cache.pool.fill_(float("nan"))
    numbers, dice = np.random.default_rng(1), random.Random(1)
    said = [np.zeros((0, DIM), np.float32) for _ in range(sequences)]        # the tokens of every sequence, as they came in
    heard = [np.zeros((0, DIM)) for _ in range(sequences)]                   # ... and what the block said to them

    def step(counts, parents):
        """One step of drafted tokens; returns what went in and what came out."""
        x = torch.from_numpy(numbers.standard_normal((sequences, width, DIM), dtype=np.float32)).cuda()
        count = torch.tensor(counts, dtype=torch.int32, device="cuda")
        mask = np.zeros((sequences, width, width), bool)
        for s in range(sequences):
            for i, parent in enumerate(parents[s]):
                if parent >= 0:
                    mask[s, i] = mask[s, parent]
                mask[s, i, i] = True
        cache.reserve(count)
        (qkv,) = front(x.view(-1, DIM))
        q, k, v = qkv.view(sequences, width, 3, HEADS, -1).unbind(2)
        cache.append(0, k, v, count)
        out = cache.attend(0, q, torch.from_numpy(mask).cuda(), count)
        (y,) = back(out.reshape(-1, DIM).float(), x.view(-1, DIM))
        return x.cpu().numpy(), y.view(sequences, width, DIM).double().cpu().numpy()

    def accept(kept, x, y):
        table = torch.tensor([k + [0] * (width - len(k)) for k in kept], dtype=torch.int32, device="cuda")
        cache.accept(torch.tensor([len(k) for k in kept], dtype=torch.int32, device="cuda"), table)
        for s, k in enumerate(kept):
            said[s], heard[s] = np.concatenate([said[s], x[s, k]]), np.concatenate([heard[s], y[s, k]])

    chain = [list(range(-1, width - 1))] * sequences
    for counts in ([8, 5, 8, 1], [8, 8, 2, 0], [3, 8, 0, 0]):                # prompts, in pieces
        x, y = step(counts, chain)
        accept([list(range(c)) for c in counts], x, y)
    for round_ in range(4):                                                  # drafts as trees, of which a path is accepted
        parents = [[dice.randint(-1, i - 1) for i in range(width)] for _ in range(sequences)]
        counts = [dice.randint(1, width) for _ in range(sequences)]
        x, y = step(counts, parents)
        kept = []
        for s in range(sequences):
            path, at = [], dice.randrange(counts[s])
            while at >= 0:
                path, at = [at] + path, parents[s][at]
            kept.append(path)
        accept(kept, x, y)
        if round_ == 1:                                                      # two beams go on from the longest
            sources = [0, 0, 2, 0]
            cache.fork(torch.tensor(sources, device="cuda"))
            said, heard = [said[i].copy() for i in sources], [heard[i].copy() for i in sources]
        if round_ == 2:
            cache.compact()
    cache.status()
    assert cache.lengths.tolist() == [len(x) for x in said]
    for s in range(sequences):
        assert len(said[s]) > 10
        assert scale_relative_error(heard[s], whole_block(said[s], consts)) <= tolerance

"""A server's loop over the paged cache, as its calls go together: compiled modules around the attention, drafted tokens that the model's own logits verify, and sequences that
give up what they have no room for.  Every step against the oracle."""

import random

import numpy as np
import pytest
import torch

from oracle.cache_steps_oracle import Steps, verify
from test_paged_cache_gpu import faults_of, ints, same
from test_paged_cache_run_gpu import DIM, HEADS, modules

pytestmark = pytest.mark.gpu

SEQUENCES, WIDTH, VOCABULARY, PAGE, PAGES_EACH = 4, 6, 300, 8, 12


def close(cache, o, q, mask, counts, window, sinks, places, got, lse):
    """Attention and lse against float64: bfloat16 rounds weights and results by 2^-9 each, and float32's sums are within 1e-4 of what sums of weights are."""
    want, weight, _, want_lse = o.look(0, q, mask, counts, window=window, sinks=sinks, places=places)
    u = torch.finfo(cache.dtype).eps / 2
    assert (np.abs(got.cpu().double().numpy() - want) <= weight * (u + 1e-4) + u * np.abs(want) + 1e-30).all()
    if lse is not None:
        sees = np.isfinite(want_lse)
        assert np.array_equal(np.isfinite(lse.cpu().numpy()), sees) and np.abs(lse.cpu().double().numpy() - want_lse)[sees].max() <= 1e-4


@pytest.mark.parametrize("by_window", [True, False])
def test_a_server_of_drafted_tokens(by_window):
    """by_window: a sliding window, and the pages that it leaves go back; else the heaviest tokens stay."""
    from kiln_b200.cache import PagedCache

    front, back, _ = modules(SEQUENCES * WIDTH, "fp32")
    cache = PagedCache(layers=1, sequences=SEQUENCES, max_pages=PAGES_EACH, pages=SEQUENCES * PAGES_EACH, kv_heads=HEADS, head_dim=DIM // HEADS, page_tokens=PAGE, dtype=torch.bfloat16)
    cache.pool.fill_(float("nan"))
    o = Steps.of(cache)
    generator = torch.Generator("cuda").manual_seed(2)
    dice = random.Random(2)
    embedding = torch.randn(VOCABULARY, DIM, device="cuda", generator=generator)
    head = torch.randn(DIM, VOCABULARY, device="cuda", generator=generator) * DIM ** -0.5
    weights = torch.zeros(SEQUENCES, PAGES_EACH * PAGE, device="cuda")
    window, sinks, most = (24, 2, None) if by_window else (None, 0, 18)
    following = torch.randint(0, VOCABULARY, (SEQUENCES,), device="cuda", generator=generator, dtype=torch.int32)
    accepted_in_all = released = evicted = 0
    for step in range(24):
        drafting = step >= 3
        counts = [dice.randint(1, WIDTH) for _ in range(SEQUENCES)]
        parents = [[-1] + [dice.randint(max(0, i - 2), i - 1) if drafting else i - 1 for i in range(1, WIDTH)] for _ in range(SEQUENCES)]
        tokens = torch.randint(0, VOCABULARY, (SEQUENCES, WIDTH), device="cuda", generator=generator, dtype=torch.int32)
        tokens[:, 0] = following
        mask = np.zeros((SEQUENCES, WIDTH, WIDTH), bool)
        for s in range(SEQUENCES):
            for i, parent in enumerate(parents[s]):
                if parent >= 0:
                    mask[s, i] = mask[s, parent]
                mask[s, i, i] = True
        places = (mask.sum(-1) - 1).astype(np.int32) if by_window else None
        x = embedding[tokens.long()]
        # the step
        cache.reserve(ints(counts))
        (qkv,) = front(x.view(-1, DIM))
        q, k, v = qkv.view(SEQUENCES, WIDTH, 3, HEADS, -1).unbind(2)
        cache.append(0, k, v, ints(counts))
        lse = torch.empty(SEQUENCES, WIDTH, HEADS, device="cuda")
        out = cache.attend(0, q, torch.from_numpy(mask).cuda(), ints(counts), window=window, sinks=sinks, places=None if places is None else ints(places.tolist()), lse=lse)
        (y,) = back(out.reshape(-1, DIM).float(), x.view(-1, DIM))
        logits = (y @ head).view(SEQUENCES, WIDTH, VOCABULARY)
        uniform = torch.rand(SEQUENCES, WIDTH, device="cuda", generator=generator)
        # the same step by the oracle, with what the modules made of it
        o.reserve(counts)
        o.append(0, k, v, counts)
        close(cache, o, q, mask, counts, window, sinks, places, out, lse)
        if drafting:
            draft = torch.softmax(logits + 0.5 * torch.randn(logits.shape, device="cuda", generator=generator), -1)
            for s in range(SEQUENCES):                                       # what a small model would have drafted, had it run in front
                for i in range(1, WIDTH):
                    tokens[s, i] = torch.multinomial(draft[s, parents[s][i]], 1, generator=generator)[0]
            given = dict(logits=logits, tokens=tokens, uniform=uniform, draft=draft, parents=ints(parents), temperature=torch.tensor([1.0, 0.7, 0.0, 1.0], device="cuda"))
            n, kept, following = cache.verify(**given, counts=ints(counts))
            want = verify(SEQUENCES, **given, counts=counts)
            assert [n.tolist(), kept.tolist(), following.tolist()] == [*want[:3]] and want[3] == 0
        else:
            n, kept, following = ints(counts), ints([list(range(WIDTH))] * SEQUENCES), torch.randint(0, VOCABULARY, (SEQUENCES,), device="cuda", generator=generator, dtype=torch.int32)
        if not by_window:
            # only what is accepted, where it is going to stand: the rows that stay, in a chain
            rows = kept.clamp_min(0).long()[:, :, None, None].expand(-1, -1, HEADS, DIM // HEADS)
            lse = lse.gather(1, rows[..., 0])
            chosen = q.gather(1, rows)
        cache.accept(n, kept)
        o.accept(n.tolist(), kept.tolist())
        same(cache, o)
        accepted_in_all += sum(n.tolist())
        if by_window:
            before = (cache.refs == 0).sum().item()
            cache.release(window, sinks)
            o.release(window, sinks)
            released += (cache.refs == 0).sum().item() - before
            for s in range(SEQUENCES):                                       # a sequence that has no room left ends, and another one begins
                if o.lengths[s] > PAGES_EACH * PAGE - WIDTH:
                    cut = ints([0 if i == s else -1 for i in range(SEQUENCES)])
                    cache.truncate(cut)
                    o.truncate(cut.tolist())
        else:
            before = weights.cpu().numpy()
            weights = cache.weigh(0, chosen.contiguous(), lse, weights, counts=n, committed=True, out=weights)
            drafted = Steps.of(cache)                                        # (the same tokens as if they were still to be accepted)
            drafted.lengths = [a - b for a, b in zip(drafted.lengths, n.tolist())]
            want, allowed = drafted.weigh(0, chosen, lse.cpu().numpy(), before, counts=n.tolist())
            assert (np.abs(weights.cpu().double().numpy() - want) <= allowed + 1e-30).all()
            keep = [most if length > 2 * most else -1 for length in o.lengths]
            want = o.evict(weights.cpu().numpy(), keep, 8, 2)
            weights = cache.evict(weights, ints(keep), recent=8, sinks=2, out=weights)
            assert np.array_equal(weights.cpu().numpy(), want)
            evicted += sum(x >= 0 for x in keep)
        same(cache, o)
        assert faults_of(cache) == o.faults == 0
    assert accepted_in_all > 24 * SEQUENCES and (released > 0 if by_window else evicted > 0)

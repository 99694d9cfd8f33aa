"""Keys and values of many sequences in pages, and the attention that reads them.

A compiled module runs a whole sequence; serving one token by token needs K and V of the tokens before it.  ``PagedCache``
keeps them: pages of ``page_tokens`` tokens, handed out to sequences as they grow, shared by sequences that continue the same
prompt, and the attention of new tokens over them.  One step of a server that drafts tokens:

    cache.reserve(counts)                                  # room for this step's tokens
    for layer in range(layers):
        q, k, v = ...                                      # of the drafted tokens, from the compiled modules
        cache.append(layer, k, v, counts)
        out = cache.attend(layer, q, mask, counts)         # over the sequence and the drafted tokens each one follows
    n_accepted, accepted, following = cache.verify(logits, tokens, uniform, draft, parents, counts)
    cache.accept(n_accepted, accepted)                     # the accepted ones become the sequence's

Ordinary decoding drafts one token and accepts it; a prompt is a chain of tokens (no mask) that are all accepted.

A sequence need not keep all of its tokens.  With a sliding window and a few first tokens (``attend(..., window=, sinks=)``) ``release`` gives the pages behind the window
back; or ``weigh`` adds up what weight its tokens draw (from ``attend(..., lse=)``), and ``evict`` keeps the heaviest.  The two do not go together: ``weigh`` knows no window
and misses pages that were released.  After an eviction a token's index in its sequence is no longer its position in the text: ``lengths``, windows, first tokens and
places count the tokens that are left, and a model whose keys and queries carry positions takes those of new tokens from its caller's own count.

All arguments and all of the cache's state are tensors on the GPU, every call is enqueued on the current stream, and none waits for the GPU: a step can be
captured into a CUDA graph whose replays follow what the tensors hold then; the cache has to live until the last of them has run.  Calls that change the cache are
ordered by the caller (one stream, or events), like calls of one ``GPUExecutable``.  What cannot be done on the way, such as a
reservation beyond the free pages, is left out and told by ``status()``.

The reference has no counterpart: its compiled graphs keep nothing between calls.
"""

from __future__ import annotations

import ctypes as C

import torch

from kiln_b200 import _cabi
from kiln_b200.runtime import check_memory, device as current_device

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


class PagedCache:
    """K and V of up to ``sequences`` sequences in ``pages`` pages, for all layers of a model.

    ``pool`` [layers, 2, pages, kv_heads, page_tokens, head_dim], ``table`` [sequences, max_pages] (-1: none), ``held``
    [sequences] (pages), ``lengths`` [sequences] (committed tokens) and ``refs`` [pages] (holders) are its tensors, to be read
    at any time and to be written between calls by a caller that keeps them consistent (restoring a snapshot, say).
    """

    def __init__(self, layers, sequences, max_pages, pages, kv_heads, head_dim, page_tokens=64, dtype=torch.bfloat16, device=None):
        if dtype not in DTYPES:
            raise TypeError(f"a cache holds float32, bfloat16 or float16, not {dtype}")
        sizes = dict(layers=layers, sequences=sequences, max_pages=max_pages, pages=pages, kv_heads=kv_heads, head_dim=head_dim, page_tokens=page_tokens)
        for name, n in sizes.items():
            if not isinstance(n, int) or isinstance(n, bool) or not 0 < n < 2**31:
                raise ValueError(f"{name} must be a positive integer, got {n!r}")
        self._cache, self._caller = C.c_void_p(), None
        self._lib = _cabi.load()
        # what the library would refuse is refused before anything is allocated
        desc = _cabi.CacheDesc(DTYPES[dtype], layers, sequences, max_pages, pages, kv_heads, page_tokens, head_dim, 16, 2**63, 16, 16, 16, 16)
        _cabi.check(self._lib.kb200_cache_check(C.byref(desc)), self._lib)
        self.device = current_device() if device is None else torch.device(device)
        if self.device.type != "cuda":
            raise RuntimeError(f"a cache lives on a GPU, not on {self.device}")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        self.layers, self.sequences, self.max_pages, self.pages = layers, sequences, max_pages, pages
        self.kv_heads, self.head_dim, self.page_tokens, self.dtype = kv_heads, head_dim, page_tokens, dtype
        shape = (layers, 2, pages, kv_heads, page_tokens, head_dim)
        pool_bytes = dtype.itemsize * layers * 2 * pages * kv_heads * page_tokens * head_dim
        check_memory(self.device, pool_bytes + 16 * max(pages, sequences) + 8 * sequences * max_pages + 8 * pages,
                     f"a cache of {pages} pages ({pool_bytes / 2**20:.1f} MiB)")
        self.pool = torch.empty(shape, dtype=dtype, device=self.device)
        self.table = torch.full((sequences, max_pages), -1, dtype=torch.int32, device=self.device)
        self.held, self.lengths = (torch.zeros(sequences, dtype=torch.int32, device=self.device) for _ in range(2))
        self.refs = torch.zeros(pages, dtype=torch.int32, device=self.device)
        self._buffers = (self.pool, self.table, self.held, self.lengths, self.refs)      # (what the library's pointers are of)
        desc.pool, desc.pool_bytes = self.pool.data_ptr(), pool_bytes
        desc.table, desc.held, desc.lengths, desc.refs = (t.data_ptr() for t in (self.table, self.held, self.lengths, self.refs))
        self._call = _cabi.load_call()
        _cabi.check(self._lib.kb200_cache_create(C.byref(desc), self.device.index, C.byref(self._cache)), self._lib)
        self._caller = self._call.cache_caller(self._cache.value, self.device.index, sequences, kv_heads, head_dim, DTYPES[dtype], max_pages * page_tokens)

    # -- pages -----------------------------------------------------------------------------------

    def fork(self, sources):
        """Every sequence ``s`` becomes what ``sources[s]`` was before the call, sharing its pages (``s`` itself: unchanged, -1: empty)."""
        self._call.cache_fork(self._caller, sources)

    def reserve(self, counts):
        """Pages of its own for the ``counts[s]`` tokens behind every sequence; all of them or, short of free pages, none."""
        self._call.cache_reserve(self._caller, counts)

    def truncate(self, lengths):
        """Keeps the first ``lengths[s]`` tokens of every sequence (0: none, the sequence is free; negative: all as it is)."""
        self._call.cache_truncate(self._caller, lengths)

    def compact(self):
        """Moves the pages in use to the front of the pool."""
        self._call.cache_compact(self._caller)

    # -- tokens ----------------------------------------------------------------------------------

    def append(self, layer, k, v, counts=None, slots=None):
        """Writes K and V of the first ``counts[b]`` tokens of every row of ``k`` and ``v`` [rows, tokens, kv_heads, head_dim] behind
        the committed tokens of sequence ``slots[b]`` (default: ``b``; none twice, rows of no token included), in the cache's type."""
        self._call.cache_append(self._caller, layer, k, v, counts, slots)

    def accept(self, counts, kept=None):
        """Commits ``counts[s]`` tokens of those appended behind every sequence: the ones with the ascending indexes ``kept[s, :counts[s]]``,
        or the first ones; the rest is dropped and its pages are free."""
        self._call.cache_accept(self._caller, counts, kept)

    def attend(self, layer, q, mask=None, counts=None, slots=None, scale=None, out=None, window=None, sinks=0, places=None, lse=None):
        """Attention of the first ``counts[b]`` tokens of every row of ``q`` [rows, tokens, heads, head_dim] over the committed tokens of
        sequence ``slots[b]`` (default: ``b``) and, of the ``counts[b]`` tokens appended behind them, those that ``mask`` ([tokens, tokens]
        or [rows, tokens, tokens], bool; default: itself and those before it) shows.  ``heads`` is a multiple of the cache's; scale defaults to
        ``head_dim ** -0.5``.  Returns ``out``, of the cache's type, with zeros in rows of no token and in rows that see nothing; it may be ``q``
        itself, but not share part of its memory.

        ``window``: a token sees itself and the ``window - 1`` tokens before it, and the sequence's first ``sinks``.  Which of the drafted tokens a mask shows
        is the mask's matter; a token of a tree stands ``places[b, i]`` (its depth, from 0 to ``tokens - 1``; what is outside counts as the nearest of these; default: ``i``)
        behind the committed ones.
        ``lse``: a float32 tensor [rows, tokens, heads] that gets the logarithm of each row's sum of exponentials (-inf where a row sees nothing)."""
        return self._call.cache_attend(self._caller, layer, q, mask, counts, slots, scale, out, window, sinks, places, lse)

    def verify(self, logits, tokens, uniform, draft=None, parents=None, counts=None, slots=None, temperature=None):
        """Which of the drafted ``tokens`` [rows, tokens] the model accepts, by its ``logits`` [rows, tokens, vocabulary] of what follows each of them and by given
        random numbers ``uniform`` [rows, tokens] from [0, 1): ``(n_accepted, accepted, following)``, by sequence, the first two as ``accept`` takes them and the third the token
        that comes next (-1: none).  What is returned is distributed as the model's own samples.

        Token 0 of a row followed the last step and is not in question; token ``i`` was drafted behind token ``parents[i]`` or ``parents[b, i]`` (default: ``i - 1``), by the
        probabilities ``draft[b, parent]`` or, without ``draft``, without chance.  Of several that follow the same token the first one that is accepted counts.
        ``temperature`` [rows], float32 (default: 1); 0 stands for the largest logit."""
        return self._call.cache_verify(self._caller, logits, tokens, uniform, draft, parents, counts, slots, temperature)

    # -- what a sequence gives up before its end ---------------------------------------------------

    def release(self, window, sinks=0):
        """Gives back the pages of every sequence that no token to come will see through this ``window``, none of whose tokens are among the first ``sinks``.
        The sequences keep their lengths; ``attend`` with that window (or a smaller one) goes on as before."""
        self._call.cache_release(self._caller, window, sinks)

    def weigh(self, layer, q, lse, weights=None, mask=None, counts=None, slots=None, scale=None, committed=False, out=None):
        """Adds up what weight the tokens of the sequences draw: ``weights`` [sequences, max_pages * page_tokens] (float32; default: zeros) plus the sum over heads and over the first
        ``counts[b]`` rows of ``q`` of the weights that ``attend`` (without a window) gave them, whose ``lse`` this takes.  Returns ``out``, which may be ``weights``.
        The rows are the tokens drafted behind the committed ones, or, ``committed``, the last of those: what a call of ``accept`` has taken, in its order (of a
        tree that was drafted, the rows of ``q`` and ``lse`` that ``accepted`` names).  ``slots`` names no sequence twice.  Tokens whose page was released draw nothing, and ``status``
        tells of them."""
        return self._call.cache_weigh(self._caller, layer, q, lse, weights, mask, counts, slots, scale, committed, out)

    def evict(self, weights, keep, recent=0, sinks=0, out=None):
        """Keeps ``keep[s]`` committed tokens of every sequence, in all layers: the first ``sinks``, the last ``recent`` and, of the others, the heaviest (of equal ones the
        first).  They become its first tokens, in their order (their indexes are then no positions in the text), and its other pages are free.  A negative entry, or a sequence of no
        more tokens, changes nothing.
        Returns ``out`` (which may be ``weights``): the weights of the tokens that are left, zeros behind them."""
        return self._call.cache_evict(self._caller, weights, keep, recent, sinks, out)

    # -- the rest --------------------------------------------------------------------------------

    def status(self):
        """Waits for the current stream and raises if an operation since the last check left something out: MemoryError for a
        reservation beyond the free pages, ValueError for indexes or counts out of range, tokens without a page, writes into shared pages, logits that are no
        distribution."""
        torch.cuda.current_stream(self.device).synchronize()
        _cabi.check(self._lib.kb200_cache_status(self._cache), self._lib)

    def close(self):
        self._caller = None
        if getattr(self, "_cache", None) is not None and self._cache:
            self._lib.kb200_cache_destroy(self._cache)
            self._cache = C.c_void_p()

    def __del__(self):
        try:
            self.close()
        except Exception:   # noqa: BLE001  (interpreter shutdown)
            pass

"""A KV cache held in 4 bits, in pages of 64 tokens, and the attention of new tokens over it.

The serving side of flash_attention_custom_mask: its masks choose 64-token blocks of keys, a page holds the keys of one block, and
the mask of a call chooses pages.  No counterpart in the reference, whose one call takes all keys in 16 bits
(fa2_custom_mask/fa2_custom_mask.py:43-94).

All bookkeeping (which pages a sequence has, how long it is) is in GPU memory and done by kernels: no call waits for the GPU, and a
captured step can be replayed while the sequences grow.  What a call finds that it cannot do (no free page, a row that names no
sequence) it leaves undone and reports.  Each later call looks, before it does anything, whether its GPU has reported something by then:
the first one that finds something raises in place of doing its own work (call it again).  That need not be the very next one, whose look may come
before the GPU is so far, and the replay of a graph does not look: PagedCache4.check() waits for the GPU and is sure to tell.

`sequences` says which sequence of the cache a row of a call is (default: row b is sequence b); it, `at`, `counts`, `start`, `keep`,
`parents` and `children` are int32 or int64 tensors on the GPU with one number a row (int32 is taken as it is).
"""
import torch

from . import _ext

_host = _ext.host()

PAGE = 64


class PagedCache4:
    """Keys and values of up to `sequences` sequences of up to `tokens` tokens each, in `pages` pages of 64 tokens.

    32 consecutive values of a token's head share a power of two, 2^(scale - 127), the smallest of which the largest magnitude is less
    than 7 times as large; each value is kept as the nearest of {0, .5, 1, 1.5, 2, 3, 4, 6} times that, with its sign (4.25 bits a
    value).  Values that are not finite make their 32 not a number.  heads, head_dim: of k and v (head_dim 16 and 32 take the room of
    64).  dtype: of what is appended, read back and asked with.

    k_codes, v_codes    uint8 [pages, heads, 64, head_dim / 2], two values a byte, the lower four bits first: index into the
                        magnitudes, 8 added for the sign
    k_scales, v_scales  uint8 [pages, heads, head_dim / 32, 4, 4, 4], token t of a page at [t % 4, t // 4 % 4, t // 16]
    page_table          int32 [sequences, pages of one], the pages of a sequence in their order, -1 behind them
    lengths             int32 [sequences]
    refs                int32 [pages], how many sequences hold a page (0, or less: free)
    free_from           int32 [1], a note of the calls': no page below this number is free

    The tensors may be read at any time, saved, and put back all together; the calls below write to them.  Who frees pages otherwise (by
    writing to refs) sets free_from to 0, which is always right: where it is too high an append takes free pages of higher numbers than it
    need, and looks at the lower ones only before it reports that there are none."""

    def __init__(self, pages, heads, head_dim, sequences, tokens, dtype=torch.bfloat16, device="cuda"):
        if min(pages, heads, sequences, tokens) < 1:
            raise ValueError("a cache has at least one page, head, sequence and token")
        D = max(head_dim, 64)
        make = lambda *size, dtype=torch.uint8: torch.empty(size, dtype=dtype, device=device)     # noqa: E731
        codes, scales = (pages, heads, PAGE, D // 2), (pages, heads, D // 32, 4, 4, 4)
        self._of(make(*codes), make(*scales), make(*codes), make(*scales), make(sequences, -(-tokens // PAGE), dtype=torch.int32).fill_(-1),
                 make(sequences, dtype=torch.int32).zero_(), make(pages, dtype=torch.int32).zero_(), head_dim, dtype)

    @classmethod
    def of(cls, k_codes, k_scales, v_codes, v_scales, page_table, lengths, refs, dtype, head_dim=None, free_from=None):
        """A cache made of tensors that are there already (not copied; scale bytes at most 140 for float16, 252 for bfloat16, or
        255).  free_from: None for a new one that says 0, or that of another cache made of the same tensors."""
        cache = cls.__new__(cls)
        cache._of(k_codes, k_scales, v_codes, v_scales, page_table, lengths, refs, 2 * k_codes.shape[-1] if head_dim is None else head_dim, dtype, free_from)
        return cache

    def _of(self, k_codes, k_scales, v_codes, v_scales, page_table, lengths, refs, head_dim, dtype, free_from=None):
        self._handle = _host.PagedCache(k_codes, k_scales, v_codes, v_scales, page_table, lengths, refs, head_dim, torch.empty(0, dtype=dtype), free_from)
        self.k_codes, self.k_scales, self.v_codes, self.v_scales = k_codes, k_scales, v_codes, v_scales
        self.page_table, self.lengths, self.refs, self.free_from = page_table, lengths, refs, self._handle.free_from
        self.head_dim, self.dtype, self.device = head_dim, dtype, k_codes.device

    def check(self):
        """Waits for the GPU and raises what the calls and replays so far have reported."""
        torch.cuda.synchronize(self.device)
        self._handle.poll()


def cache_append(cache, k, v, at=None, counts=None, sequences=None):
    """k, v [B, heads, N, head_dim] go behind the sequences' tokens; of row b the first counts[b] (default: all N).  at: the sequences are
    first cut to that many tokens (a draft that was not taken, a new prompt in place of an old one).  Pages are taken as needed, lowest
    numbers first; a page that other sequences hold too is copied before it is written to.  At most 1024 rows."""
    _host.cache_append(cache._handle, k, v, at, counts, sequences)


def cache_read(cache, tokens, start=None, sequences=None):
    """(k, v), [B, heads, tokens, head_dim] each: the values that the cache holds for tokens start[b] (default: 0) and following of each
    row's sequence (default: all sequences), zeros where a sequence has none."""
    return _host.cache_read(cache._handle, tokens, start, sequences)


def cache_attention(q, cache, mask, sm_scale, counts=None, sequences=None):
    """Attention of each row's last tokens over its sequence, as it is in the cache (their own keys and values appended before).
    q [B, H, N, head_dim], H a multiple of the cache's heads (consecutive heads share one); the first counts[b] (default: N) queries of
    row b are the sequence's last counts[b] tokens and see the tokens up to their own.  mask: None, or bool
    [1 | B, 1 | heads | H, 1 | ceil(N / 64), pages of a sequence], the pages that are kept (for all queries, or for each 64 of
    the call).  Returns o like q; queries that see no token, and those behind counts[b], get 0.  There is no gradient."""
    return _host.cache_attention(cache._handle, q, mask, sm_scale, counts, sequences, False, False)


def cache_attention_lse(q, cache, mask, sm_scale, counts=None, sequences=None, out_fp32=False):
    """The same, also returning the natural-log logsumexp [B, H, N] fp32 of the scaled scores seen (-inf: none); out_fp32=True returns o
    in fp32, for callers that merge it with others' (of a bfloat16 cache it is computed with probabilities of 16 bits behind the point in
    place of 8)."""
    return _host.cache_attention(cache._handle, q, mask, sm_scale, counts, sequences, out_fp32, True)


def cache_fork(cache, parents, children):
    """Sequence children[i], which holds no tokens, becomes a copy of parents[i].  The two share their pages; an append to either copies
    the one page that it writes to."""
    _host.cache_fork(cache._handle, parents, children)


def cache_free(cache, sequences=None, keep=None):
    """The sequences (default: all) keep their first keep[i] (default: 0) tokens; pages that no sequence holds any longer are free."""
    _host.cache_free(cache._handle, sequences, keep)


def cache_compact(cache):
    """Moves the pages in use to the lowest page numbers (free numbers in ascending order take the used pages behind, in ascending order)
    and renames them in the page table, so that the memory behind them can be used otherwise."""
    _host.cache_compact(cache._handle)

"""The KV cache in pages of 4-bit values on the GPU against lists and 64-bit values (cache_reference.py): what it keeps, where, and the
attention over it."""
import math
import random

import numpy as np
import pytest
import torch

from cache_reference import PAGE, Reference, attention, scale_of, stands_for, within

pytestmark = pytest.mark.gpu
F16, BF16 = torch.float16, torch.bfloat16


def make(dev, pages, heads, D, sequences, tokens, dtype):
    import fa2_custom_mask as fm
    cache = fm.PagedCache4(pages, heads, D, sequences, tokens, dtype, dev)
    # memory that was somebody else's: nothing of it may show
    for x in (cache.k_codes, cache.v_codes):
        x.random_(0, 256)
    for x in (cache.k_scales, cache.v_scales):
        x.random_(250, 256)
    return cache, Reference(pages, heads, D, sequences, tokens, dtype)


def ints(x, dev, dtype=torch.int32):
    return None if x is None else torch.tensor(x, dtype=dtype, device=dev)


def tokens(B, heads, N, D, dtype, g, dev):
    return [torch.randn(B, heads, N, D, generator=g).to(dtype).to(dev) for _ in range(2)]


def append(cache, ref, k, v, at=None, counts=None, sequences=None, index=torch.int32):
    import fa2_custom_mask as fm
    dev = cache.device
    fm.cache_append(cache, k, v, at=ints(at, dev, index), counts=ints(counts, dev, index), sequences=ints(sequences, dev, index))
    return ref.append(k, v, at, counts, sequences)


def same_tables(cache, ref):
    assert cache.lengths.tolist() == ref.length
    assert cache.page_table.tolist() == ref.tables()
    assert cache.refs.tolist() == ref.refs


def same_values(cache, ref):
    import fa2_custom_mask as fm
    n = max(1, max(ref.length))
    for got, want in zip(fm.cache_read(cache, n), ref.read(n)):
        assert np.array_equal(got.double().cpu().numpy(), want, equal_nan=True)


def said(cache, words):
    """The next call raises what was reported, once."""
    if words:
        with pytest.raises(RuntimeError, match="an earlier"):
            cache.check()
    cache.check()


def attend(cache, ref, q, mask=None, scale=None, counts=None, sequences=None, out_fp32=False):
    """Through the public call and within the bounds of the reference; returns (o, lse)."""
    import fa2_custom_mask as fm
    B, H, N, D = q.shape
    scale = scale_of(D) if scale is None else scale
    dev = cache.device
    o, lse = fm.cache_attention_lse(q, cache, None if mask is None else mask.to(dev), scale, ints(counts, dev), ints(sequences, dev), out_fp32)
    plain = fm.cache_attention(q, cache, None if mask is None else mask.to(dev), scale, counts=ints(counts, dev), sequences=ints(sequences, dev))
    assert plain.dtype == q.dtype and o.dtype == (torch.float32 if out_fp32 else q.dtype)
    if not out_fp32:
        assert torch.equal(plain.view(torch.int16), o.view(torch.int16))
    cache.check()
    q = q.double().cpu().numpy()
    got_o, got_lse = o.double().cpu().numpy(), lse.double().cpu().numpy()
    for b in range(B):
        s, n = b if sequences is None else sequences[b], N if counts is None else counts[b]
        kept = None
        if mask is not None:
            m = mask[b % mask.shape[0]].numpy()
            group = H // ref.H
            heads = [0 if m.shape[0] == 1 else (h if m.shape[0] == H else h // group) for h in range(H)]
            rows = [i // PAGE if m.shape[1] > 1 else 0 for i in range(n)]
            kept = m[heads][:, rows]
        k, v = ref.values(s)
        ro, rl, mean = attention(q[b, :, :n], k, v, ref.length[s] - n, scale, kept)
        assert within(got_o[b, :, :n], ro, mean, cache.dtype, o.dtype), (b, n, ref.length[s])
        assert not got_o[b, :, n:].any() and (got_lse[b, :, n:] == -np.inf).all()
        none = rl == -np.inf
        assert np.array_equal(got_lse[b, :, :n] == -np.inf, none) and np.array_equal(np.isnan(got_lse[b, :, :n]), np.isnan(rl))
        ok = ~none & ~np.isnan(rl)
        assert (np.abs(got_lse[b, :, :n][ok] - rl[ok]) <= 2e-4 * np.maximum(1, np.abs(rl[ok]) / 16)).all()
    return o, lse


# ---- what is kept ----
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [64, 128, 256])
def test_every_value(dev, dtype, D):
    """All 2^16 values of the type, each in a group of its own size and in random ones."""
    x = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    g = torch.Generator().manual_seed(3)
    x = torch.cat((x, x[torch.randperm(65536, generator=g)], x.double().mul(0.3).to(dtype)))
    n = x.numel() // D
    cache, ref = make(dev, -(-n // PAGE) + 1, 1, D, 1, n, dtype)
    x = x.view(1, 1, n, D).to(dev)
    append(cache, ref, x, x.flip(2))
    same_tables(cache, ref)
    same_values(cache, ref)
    cache.check()


@pytest.mark.parametrize("D,dtype", [(16, BF16), (32, F16), (64, F16), (64, BF16), (128, BF16), (256, F16)])
def test_append_and_read(dev, D, dtype):
    g = torch.Generator().manual_seed(D)
    cache, ref = make(dev, 23, 3, D, 5, 300, dtype)
    assert not append(cache, ref, *tokens(4, 3, 70, D, dtype, g, dev), counts=[70, 1, 0, 64], sequences=[3, 0, 4, 1])
    same_tables(cache, ref)
    same_values(cache, ref)
    for i in range(3):                                       # one token each: into a new page, the middle of one, its last slot
        assert not append(cache, ref, *tokens(5, 3, 1, D, dtype, g, dev))
    same_tables(cache, ref)
    same_values(cache, ref)
    # cut back and written over; cut without anything behind; a cut to the very length
    assert not append(cache, ref, *tokens(3, 3, 90, D, dtype, g, dev), at=[66, 0, 3], counts=[90, 0, 2], sequences=[3, 1, 0], index=torch.int64)
    same_tables(cache, ref)
    same_values(cache, ref)
    assert not append(cache, ref, *tokens(2, 3, 0, D, dtype, g, dev), at=[65, 1], sequences=[3, 4])
    same_tables(cache, ref)
    # strided: [B, N, H, D] in memory, one of two heads' halves
    k, v = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in tokens(2, 3, 130, D, dtype, g, dev)]
    assert not append(cache, ref, k, v, sequences=[2, 4])
    k, v = [x[:, ::2] for x in tokens(1, 6, 9, D, dtype, g, dev)]
    assert not append(cache, ref, k, v)
    k, v = [x[..., 1:D + 1] for x in tokens(1, 3, 9, D + 1, dtype, g, dev)]        # rows that are not aligned
    assert not append(cache, ref, k, v)
    same_tables(cache, ref)
    same_values(cache, ref)
    import fa2_custom_mask as fm
    for got, want in zip(fm.cache_read(cache, 70, start=ints([-3, 60, 500, 0], dev), sequences=ints([3, 3, 2, 4], dev)), ref.read(70, [-3, 60, 500, 0], [3, 3, 2, 4])):
        assert got.shape == (4, 3, 70, D) and np.array_equal(got.double().cpu().numpy(), want)
    cache.check()


@pytest.mark.parametrize("seed", range(6))
def test_random_calls(dev, seed):
    """Appends, cuts, forks, frees and compactions in random order, some of which the cache has to refuse, agree with lists."""
    import fa2_custom_mask as fm
    r = random.Random(seed)
    g = torch.Generator().manual_seed(seed)
    heads, D, dtype, S = r.choice([1, 2, 3]), r.choice([64, 128, 256]), r.choice([F16, BF16]), 7
    cache, ref = make(dev, 24, heads, D, S, 400, dtype)
    for _ in range(40):
        what = r.choice(["append"] * 4 + ["step"] * 3 + ["fork", "fork", "free", "free", "compact"])
        some = r.sample(range(S), r.randint(1, S))
        if r.random() < 0.1:
            some[r.randrange(len(some))] = r.choice([-1, S, some[0], 1 << 20])
        if what == "append":
            n = r.choice([1, 5, 64, 100, 200])
            at = [r.choice([ref.length[s] if 0 <= s < S else 0, r.randint(0, 130)]) for s in some] if r.random() < 0.4 else None
            counts = [r.randint(0, n + (r.random() < 0.1)) for _ in some] if r.random() < 0.6 else None
            words = append(cache, ref, *tokens(len(some), heads, n, D, dtype, g, dev), at=at, counts=counts, sequences=some)
        elif what == "step":
            words = append(cache, ref, *tokens(S, heads, 1, D, dtype, g, dev))
        elif what == "fork":
            children = r.sample(range(S), len(some))
            fm.cache_fork(cache, ints(some, dev), ints(children, dev))
            words = ref.fork(some, children)
        elif what == "free":
            keep = [r.choice([0, 64, r.randint(-1, 300)]) for _ in some] if r.random() < 0.5 else None
            fm.cache_free(cache, ints(some, dev), ints(keep, dev))
            words = ref.free(some, keep)
        else:
            fm.cache_compact(cache)
            ref.compact()
            words = set()
        said(cache, words)
        same_tables(cache, ref)
    same_values(cache, ref)
    q = torch.randn(S, heads * 2, 3, D, generator=g).to(dtype).to(dev)
    attend(cache, ref, q)


def test_copy_on_write(dev):
    """Parent and children append in one call, one of them behind a cut inside a page that all share."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(2)
    cache, ref = make(dev, 40, 2, 128, 6, 400, BF16)
    append(cache, ref, *tokens(1, 2, 200, 128, BF16, g, dev), sequences=[2])
    fm.cache_fork(cache, ints([2, 2, 2], dev), ints([0, 5, 3], dev))
    assert not ref.fork([2, 2, 2], [0, 5, 3])
    same_tables(cache, ref)
    assert not append(cache, ref, *tokens(4, 2, 3, 128, BF16, g, dev), at=[200, 70, 199, 128], sequences=[2, 0, 5, 3])
    same_tables(cache, ref)
    same_values(cache, ref)
    fm.cache_free(cache, ints([2], dev))
    ref.free([2])
    assert not append(cache, ref, *tokens(3, 2, 60, 128, BF16, g, dev), sequences=[3, 0, 5])
    same_tables(cache, ref)
    same_values(cache, ref)
    # of a page that one sequence holds alone again nothing is copied
    fm.cache_fork(cache, ints([0], dev), ints([1], dev))
    fm.cache_free(cache, ints([0], dev))
    ref.fork([0], [1]), ref.free([0])
    before = cache.page_table[1].tolist()
    assert not append(cache, ref, *tokens(1, 2, 1, 128, BF16, g, dev), sequences=[1])
    assert cache.page_table[1].tolist() == before
    same_tables(cache, ref)
    same_values(cache, ref)


def test_no_free_page(dev):
    """Rows are served in their order; one that does not fit, and those behind it that need pages, stay as they are; nothing else is lost."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(4)
    cache, ref = make(dev, 5, 1, 64, 4, 640, F16)
    assert not append(cache, ref, *tokens(4, 1, 60, 64, F16, g, dev), counts=[60, 10, 60, 0])
    assert append(cache, ref, *tokens(4, 1, 100, 64, F16, g, dev), counts=[100, 3, 20, 1]) == {1}
    same_tables(cache, ref)
    said(cache, {1})
    assert append(cache, ref, *tokens(2, 1, 200, 64, F16, g, dev), sequences=[3, 1], counts=[200, 1]) == {1}
    with pytest.raises(RuntimeError, match="no free page"):
        torch.cuda.synchronize()
        fm.cache_read(cache, 1)
    same_tables(cache, ref)
    same_values(cache, ref)
    fm.cache_free(cache, ints([0], dev))
    ref.free([0])
    assert not append(cache, ref, *tokens(1, 1, 64, 64, F16, g, dev), sequences=[3])
    same_tables(cache, ref)
    same_values(cache, ref)
    cache.check()


def test_compact(dev):
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(5)
    cache, ref = make(dev, 70, 2, 64, 12, 500, F16)
    fm.cache_compact(cache)                                        # nothing in use
    for n in (40, 130, 3):
        append(cache, ref, *tokens(12, 2, n, 64, F16, g, dev), counts=[max(0, n - 9 * b) for b in range(12)])
    fm.cache_free(cache, ints([0, 3, 4, 9], dev), ints([0, 64, 1, 0], dev))
    ref.free([0, 3, 4, 9], [0, 64, 1, 0])
    fm.cache_fork(cache, ints([11, 2], dev), ints([0, 9], dev))
    ref.fork([11, 2], [0, 9])
    q = torch.randn(12, 4, 2, 64, generator=g).to(F16).to(dev)
    before = fm.cache_attention(q, cache, None, 0.125)
    for _ in range(2):                                             # (the second time there is nothing to move)
        fm.cache_compact(cache)
        ref.compact()
        same_tables(cache, ref)
        assert torch.equal(fm.cache_attention(q, cache, None, 0.125), before)
    assert not append(cache, ref, *tokens(12, 2, 70, 64, F16, g, dev))
    same_tables(cache, ref)
    same_values(cache, ref)
    cache.check()


def test_thousands_of_pages(dev):
    """Searches and moves that take more than one round of a workgroup."""
    import fa2_custom_mask as fm
    S, M = 64, 160
    cache, ref = make(dev, S * M, 1, 64, S, M * PAGE, F16)
    full = ints(list(range(S)), dev)
    cache.page_table.copy_(torch.arange(S * M, dtype=torch.int32).view(S, M))
    cache.lengths.fill_(M * PAGE)
    cache.refs.fill_(1)
    ref.table, ref.length, ref.refs = cache.page_table.tolist(), cache.lengths.tolist(), cache.refs.tolist()
    keep = [0 if s % 3 == 0 else (s * 97) % (M * PAGE) for s in range(S)]
    fm.cache_free(cache, full, ints(keep, dev))
    ref.free(list(range(S)), keep)
    same_tables(cache, ref)
    fm.cache_compact(cache)
    ref.k, ref.v = np.zeros((S * M, 1, 1, 1)), np.zeros((S * M, 1, 1, 1))
    ref.compact()
    same_tables(cache, ref)
    # holes again, then more than 4096 pages in one append, some behind the first round of the search
    fm.cache_free(cache, ints([1, 10], dev))
    ref.free([1, 10])
    assert [r > 0 for r in ref.refs] == [r > 0 for r in cache.refs.tolist()]
    x = torch.zeros(1, 1, 1, 64, dtype=F16, device=dev).expand(S, 1, M * PAGE, 64)
    counts = [M * PAGE - n for n in ref.length]
    ref.k, ref.v = [np.zeros((S * M, 1, PAGE, 64)) for _ in range(2)]
    fm.cache_append(cache, x, x, counts=ints(counts, dev))
    free = iter([p for p in range(S * M) if not ref.refs[p]])
    for s in range(S):
        while len(ref.table[s]) < M:
            ref.table[s].append(next(free))
            ref.refs[ref.table[s][-1]] = 1
        ref.length[s] = M * PAGE
    same_tables(cache, ref)
    cache.check()


# ---- attention ----
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("D", [16, 64, 128, 256])
@pytest.mark.parametrize("heads,group", [(1, 1), (2, 3), (3, 8), (2, 16), (1, 40)])
def test_next_token(dev, D, heads, group, dtype):
    g = torch.Generator().manual_seed(D + group)
    lengths = [1, 0, 63, 64, 65, 128, 700, 2]
    cache, ref = make(dev, 40, heads, D, 10, 1000, dtype)
    append(cache, ref, *tokens(8, heads, 700, D, dtype, g, dev), counts=lengths, sequences=[9, 1, 2, 8, 3, 4, 7, 5])
    q = torch.randn(8, heads * group, 1, D, generator=g).to(dtype).to(dev)
    attend(cache, ref, q, sequences=[9, 1, 2, 8, 3, 4, 7, 5])
    attend(cache, ref, q[:4], sequences=[7, 7, 2, 7], out_fp32=True)          # the same sequence more than once


@pytest.mark.parametrize("D,dtype", [(64, F16), (64, BF16), (128, F16), (128, BF16), (256, F16), (256, BF16)])
@pytest.mark.parametrize("N,group", [(2, 1), (5, 3), (17, 2), (33, 1), (70, 7), (130, 4)])
def test_some_tokens(dev, D, dtype, N, group):
    """Drafts and pieces of prompts: rows of fewer tokens, of none, of more than the sequence has."""
    g = torch.Generator().manual_seed(N)
    cache, ref = make(dev, 30, 2, D, 6, 600, dtype)
    append(cache, ref, *tokens(6, 2, 300, D, dtype, g, dev), counts=[300, 129, 64, N, 1, 0])
    q = torch.randn(6, 2 * group, N, D, generator=g).to(dtype).to(dev)
    attend(cache, ref, q, counts=[N, N - 1, 0, N, N, 2 if N > 2 else 1])


@pytest.mark.parametrize("D,dtype", [(64, F16), (128, BF16), (256, F16)])
@pytest.mark.parametrize("N,group,mask_rows", [(1, 1, 1), (1, 4, 1), (3, 2, 1), (64, 1, 1), (100, 2, 2), (140, 3, 3)])
@pytest.mark.parametrize("mask_heads", ["one", "cache", "q"])
def test_masks(dev, D, dtype, N, group, mask_rows, mask_heads):
    """Kept pages for all heads, for those of the cache and for each of q's; for all queries and for each 64; rows of it that leave nothing."""
    g = torch.Generator().manual_seed(N + D)
    heads = 2
    cache, ref = make(dev, 40, heads, D, 5, 700, dtype)
    append(cache, ref, *tokens(5, heads, 640, D, dtype, g, dev), counts=[640, 257, 140, 200, 0])
    q = torch.randn(5, heads * group, N, D, generator=g).to(dtype).to(dev)
    Hm = {"one": 1, "cache": heads, "q": heads * group}[mask_heads]
    mask = torch.rand(5, Hm, mask_rows, 11, generator=g) < 0.5
    mask[3] = False
    mask[1, 0, 0] = False
    attend(cache, ref, q, mask=mask)
    attend(cache, ref, q, mask=mask[:1])
    wide = torch.zeros(5, Hm, mask_rows, 22, dtype=torch.bool)
    wide[..., ::2] = mask
    attend(cache, ref, q, mask=wide[..., ::2], counts=[N, max(0, N - 2), N, 0, N])          # strides of its own


def close_in_fp32(o, ref, mean):
    """A result in fp32 of a bf16 cache: half a step of it, P in two bf16 parts (half a step of the second, which is half a step of the first at
    most: 2^-18 of P, and as much again where it is rounded up to the next power of two), and the sums and exponentials in 32 bits as in
    within()."""
    return o.dtype == torch.float32 and bool((np.abs(o.double().cpu().numpy() - ref) <= (2.0 ** -17 + 2.0 ** -12) * mean + 2.0 ** -24 * np.abs(ref) + 2.0 ** -25).all())


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("N,group,masked", [(1, 1, False), (1, 8, True), (5, 3, False), (5, 3, True), (40, 2, False), (70, 1, True)])
def test_results_in_fp32_of_bf16(dev, D, N, group, masked):
    """Are not made of probabilities in 8 bits."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(D + N)
    heads, lengths = 2, [700, 65, N, 333]
    cache, ref = make(dev, 40, heads, D, 4, 700, BF16)
    append(cache, ref, *tokens(4, heads, 700, D, BF16, g, dev), counts=lengths)
    q = torch.randn(4, heads * group, N, D, generator=g).to(BF16).to(dev)
    mask = (torch.rand(4, heads * group, -(-N // PAGE), 11, generator=g) < 0.6) if masked else None
    o, _ = attend(cache, ref, q, mask=mask, out_fp32=True)
    rounded = fm.cache_attention(q, cache, None if mask is None else mask.to(dev), scale_of(D))
    error, size, coarse = 0.0, 0.0, 0.0
    for b in range(4):
        kept = None
        if masked:
            kept = mask[b].numpy()[:, [i // PAGE for i in range(N)]]
        k, v = ref.values(b)
        ro, _, mean = attention(q[b].double().cpu().numpy(), k, v, lengths[b] - N, scale_of(D), kept)
        assert close_in_fp32(o[b], ro, mean), b
        error += ((o[b].double().cpu().numpy() - ro) ** 2).sum()
        coarse += ((rounded[b].double().cpu().numpy() - ro) ** 2).sum()
        size += (ro ** 2).sum()
    assert error <= size * 2.0 ** -28 and error * 100 < coarse            # (2^-14 where the sums of 32 bits do not add up one way)


@pytest.mark.parametrize("D,heads,group,N,lengths", [(64, 1, 16, 1, [40000]), (128, 2, 4, 3, [20000, 100, 9000]), (256, 1, 5, 9, [9000, 30])])
def test_long_results_in_fp32_of_bf16(dev, D, heads, group, N, lengths):
    """The same where parts of several workgroups are merged."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(D)
    B = len(lengths)
    cache, _ = make(dev, sum(-(-n // PAGE) for n in lengths), heads, D, B, max(lengths), BF16)
    k, v = tokens(B, heads, max(lengths), D, BF16, g, dev)
    fm.cache_append(cache, k, v, counts=ints(lengths, dev))
    rk, rv = [x.double().cpu().numpy() for x in fm.cache_read(cache, max(lengths))]
    q = torch.randn(B, heads * group, N, D, generator=g).to(BF16).to(dev)
    o, lse = fm.cache_attention_lse(q, cache, None, scale_of(D), out_fp32=True)
    for b, n in enumerate(lengths):
        ro, rl, mean = attention(q[b].double().cpu().numpy(), rk[b, :, :n], rv[b, :, :n], n - N, scale_of(D))
        assert close_in_fp32(o[b], ro, mean), b
        assert np.abs(lse[b].double().cpu().numpy() - rl).max() <= 2e-4
    for _ in range(3):
        assert torch.equal(o, fm.cache_attention_lse(q, cache, None, scale_of(D), out_fp32=True)[0])
    cache.check()


@pytest.mark.parametrize("scale", [-0.3, 0.0, 3.0])
def test_scales(dev, scale):
    g = torch.Generator().manual_seed(9)
    cache, ref = make(dev, 12, 2, 64, 2, 300, F16)
    append(cache, ref, *tokens(2, 2, 200, 64, F16, g, dev), counts=[200, 3])
    attend(cache, ref, torch.randn(2, 4, 3, 64, generator=g).to(F16).to(dev), scale=scale)


def test_strided_queries(dev):
    g = torch.Generator().manual_seed(10)
    cache, ref = make(dev, 12, 2, 128, 2, 300, BF16)
    append(cache, ref, *tokens(2, 2, 200, 128, BF16, g, dev), counts=[200, 70])
    q = torch.randn(2, 5, 6, 128, generator=g).to(BF16).to(dev).transpose(1, 2)               # [B, N, H, D] in memory
    o, _ = attend(cache, ref, q)
    assert o.stride() == q.stride()
    packed = torch.randn(2, 5, 3, 4, 128, generator=g).to(BF16).to(dev)
    attend(cache, ref, packed[:, :, 1].transpose(1, 2))
    odd = torch.randn(2, 4, 5, 129, generator=g).to(BF16).to(dev)
    attend(cache, ref, odd[..., 1:])



@pytest.mark.parametrize("D,dtype,heads,group,lengths", [(64, F16, 1, 1, [40000]), (128, BF16, 2, 4, [20000, 100, 9000]), (256, F16, 1, 20, [9000, 1]),
                                                         (128, F16, 1, 40, [12000])])
def test_long_sequences(dev, D, dtype, heads, group, lengths):
    """Pages dealt to many workgroups, whose parts meet in the workspace: the same bits in every run."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(11)
    B = len(lengths)
    pages = sum(-(-n // PAGE) for n in lengths) + 3
    cache, ref = make(dev, pages, heads, D, B, max(lengths) + 5, dtype)
    k, v = tokens(B, heads, max(lengths), D, dtype, g, dev)
    fm.cache_append(cache, k, v, counts=ints(lengths, dev))
    rk, rv = [x.double().cpu().numpy() for x in fm.cache_read(cache, max(lengths))]
    q = torch.randn(B, heads * group, 1, D, generator=g).to(dtype).to(dev)
    o, lse = fm.cache_attention_lse(q, cache, None, scale_of(D))
    for b, n in enumerate(lengths):
        ro, rl, mean = attention(q[b].double().cpu().numpy(), rk[b, :, :n], rv[b, :, :n], n - 1, scale_of(D))
        assert within(o[b], ro, mean, dtype)
        assert np.abs(lse[b].double().cpu().numpy() - rl).max() <= 2e-4
    for _ in range(4):
        o2, lse2 = fm.cache_attention_lse(q, cache, None, scale_of(D))
        assert torch.equal(o, o2) and torch.equal(lse, lse2)


@pytest.mark.parametrize("B,heads,group,D,dtype,most", [(150, 2, 2, 64, F16, 700), (70, 4, 5, 128, BF16, 2000), (520, 8, 1, 64, BF16, 200), (300, 3, 3, 256, F16, 130)])
def test_many_sequences(dev, B, heads, group, D, dtype, most):
    """More sequences than a wavefront looks at at a time, than a head has workgroups, and so many that each has a workgroup of its own."""
    g = torch.Generator().manual_seed(B)
    lengths = [int(x) for x in torch.exp(torch.rand(B, generator=g) * math.log(most)).long()]
    lengths[3], lengths[-1] = 0, most
    cache, ref = make(dev, sum(-(-n // PAGE) for n in lengths) + 2, heads, D, B, most + 4, dtype)
    k, v = tokens(B, heads, most, D, dtype, g, dev)
    import fa2_custom_mask as fm
    fm.cache_append(cache, k, v, counts=ints(lengths, dev))
    rk, rv = [x.double().cpu().numpy() for x in fm.cache_read(cache, most)]
    q = torch.randn(B, heads * group, 1, D, generator=g).to(dtype).to(dev)
    o, lse = fm.cache_attention_lse(q, cache, None, scale_of(D))
    cache.check()
    o, lse, q = o.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy()
    for b, n in enumerate(lengths):
        ro, rl, mean = attention(q[b], rk[b, :, :n], rv[b, :, :n], n - 1, scale_of(D))
        assert within(o[b], ro, mean, dtype), (b, n)
        assert np.array_equal(lse[b] == -np.inf, rl == -np.inf) and (n == 0 or np.abs(lse[b] - rl).max() <= 2e-4)


@pytest.mark.parametrize("B,heads,group,N,D,dtype,most", [(24, 8, 4, 100, 64, F16, 500), (100, 8, 6, 60, 64, BF16, 200), (70, 2, 3, 90, 128, F16, 900), (130, 3, 1, 33, 256, BF16, 300)])
def test_many_pieces(dev, B, heads, group, N, D, dtype, most):
    """Pieces of many prompts: units in ranges, more than a wavefront looks at at a time, and so many that each has a workgroup of its own."""
    g = torch.Generator().manual_seed(B + N)
    lengths = [max(1, int(x)) for x in torch.exp(torch.rand(B, generator=g) * math.log(most)).long()]
    lengths[-1] = most
    counts = [min(N, n) if b % 3 else min(n, 1 + b % N) for b, n in enumerate(lengths)]
    cache, ref = make(dev, sum(-(-n // PAGE) for n in lengths) + 2, heads, D, B, most + 4, dtype)
    k, v = tokens(B, heads, most, D, dtype, g, dev)
    import fa2_custom_mask as fm
    fm.cache_append(cache, k, v, counts=ints(lengths, dev))
    rk, rv = [x.double().cpu().numpy() for x in fm.cache_read(cache, most)]
    q = torch.randn(B, heads * group, N, D, generator=g).to(dtype).to(dev)
    o, lse = fm.cache_attention_lse(q, cache, None, scale_of(D), counts=ints(counts, dev))
    cache.check()
    o, lse, q = o.double().cpu().numpy(), lse.double().cpu().numpy(), q.double().cpu().numpy()
    for b in list(range(0, B, 7)) + [B - 1]:
        n, c = lengths[b], counts[b]
        ro, rl, mean = attention(q[b, :, :c], rk[b, :, :n], rv[b, :, :n], n - c, scale_of(D))
        assert within(o[b, :, :c], ro, mean, dtype), (b, n, c)
        assert np.abs(lse[b, :, :c] - rl).max() <= 2e-4
        assert not o[b, :, c:].any() and (lse[b, :, c:] == -np.inf).all()


@pytest.mark.parametrize("heads,group,N,n,D,dtype", [(1, 16, 2200, 2300, 64, F16), (2, 3, 1000, 5000, 128, BF16), (1, 1, 700, 700, 256, F16)])
def test_long_prompts(dev, heads, group, N, n, D, dtype):
    """Hundreds of tiles of one sequence, also more than ranges are made for; the masks' rows of 64 queries among them."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(N)
    cache, ref = make(dev, -(-n // PAGE) + 2, heads, D, 1, n, dtype)
    k, v = tokens(1, heads, n, D, dtype, g, dev)
    fm.cache_append(cache, k, v)
    rk, rv = [x.double()[0] for x in fm.cache_read(cache, n)]
    q = torch.randn(1, heads * group, N, D, generator=g).to(dtype).to(dev)
    M = cache.page_table.shape[1]
    mask = torch.rand(1, heads * group, -(-N // PAGE), M, generator=g).to(dev) < 0.3
    see = torch.arange(n, device=dev) <= (n - N + torch.arange(N, device=dev))[:, None]
    for m in (None, mask):
        o = fm.cache_attention(q, cache, m, scale_of(D))
        for h in range(heads * group):
            seen = see if m is None else see & m[0, h].repeat_interleave(PAGE, 0)[:N].repeat_interleave(PAGE, 1)[:, :n]
            s = (q[0, h].double() @ rk[h // group].T * scale_of(D)).masked_fill(~seen, -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            assert within(o[0, h], (p @ rv[h // group]).cpu().numpy(), (p @ rv[h // group].abs()).cpu().numpy(), dtype), h
    cache.check()


# Units with more positions than a wavefront looks up at a time (64 of its own, or with a mask 64 of the workgroup's), in ranges and with a
# workgroup each: what is asked for ahead, and how many kept pages there were before, go from one round to the next.
def filled(dev, lengths, heads, D, dtype):
    """A cache of sequences of these lengths with random codes, scales of 2^-7 .. 2^0, pages in random order."""
    import fa2_custom_mask as fm
    count = [-(-n // PAGE) for n in lengths]
    M = max(count) + 1
    cache = fm.PagedCache4(sum(count) + 3, heads, D, len(lengths), M * PAGE, dtype, dev)
    g = torch.Generator(device=dev).manual_seed(sum(count) + D)
    for x in (cache.k_codes, cache.v_codes):
        x.random_(0, 256, generator=g)
    for x in (cache.k_scales, cache.v_scales):
        x.random_(120, 128, generator=g)
    order = torch.randperm(sum(count) + 3, generator=g, device=dev, dtype=torch.int32)
    table, at = torch.full((len(lengths), M), -1, dtype=torch.int32), 0
    for s, c in enumerate(count):
        table[s, :c] = order[at:at + c].cpu()
        at += c
    cache.page_table.copy_(table)
    cache.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
    cache.refs[order[:at].long()] = 1
    return cache, M


def agrees(o, lse, q, cache, rows, heads, mask, counts):
    """These rows and heads of q against 64 bits."""
    import fa2_custom_mask as fm
    B, H, N, D = q.shape
    group, dev = H // cache.k_codes.shape[1], q.device
    lengths = cache.lengths.tolist()
    for b in rows:
        n, c = lengths[b], counts[b]
        k, v = [x[0] for x in fm.cache_read(cache, n, sequences=ints([b], dev))]
        behind = torch.arange(n, device=dev) > (n - c + torch.arange(c, device=dev))[:, None]
        for h in heads:
            kk, vv = k[h // group].double(), v[h // group].double()
            s = (q[b, h, :c].double() @ kk.T * scale_of(D)).masked_fill(behind, -math.inf)
            if mask is not None:
                m = mask[b % mask.shape[0], h if mask.shape[1] == H else 0]
                m = m[torch.arange(c, device=dev) // PAGE] if m.shape[0] > 1 else m.expand(c, -1)
                s = s.masked_fill(~m.repeat_interleave(PAGE, 1)[:, :n], -math.inf)
            p = torch.nan_to_num(torch.softmax(s, -1), nan=0.0)
            want = torch.logsumexp(s, -1)
            assert within(o[b, h, :c], (p @ vv).cpu().numpy(), (p @ vv.abs()).cpu().numpy(), q.dtype), (b, h, n)
            assert torch.equal(lse[b, h, :c] == -math.inf, want == -math.inf), (b, h)
            assert bool(((lse[b, h, :c].double() - want).abs() <= 2e-4).logical_or(want == -math.inf).all()), (b, h)


def masks_of(g, dev, B, H, rows, M, lengths):
    """None, one for all heads, and one for each head with heads and stretches that keep nothing."""
    one = torch.rand(B, 1, rows, M, generator=g) < 0.5
    each = torch.rand(B, H, rows, M, generator=g) < torch.rand(B, H, rows, 1, generator=g)
    each[:, 0, :, 64:128] = False
    each[-1, H - 1] = False
    thin = torch.zeros(1, 1, 1, M, dtype=torch.bool)
    thin[..., 70::67] = True
    return [None] + [m.to(dev) for m in (one, each, thin)]


@pytest.mark.parametrize("B,heads,group,D,dtype,longest", [(513, 1, 1, 64, F16, [17000]), (520, 1, 5, 128, BF16, [17100, 36000]), (600, 2, 2, 256, F16, [16500]),
                                                           (1500, 1, 3, 128, F16, [100000]), (2048, 8, 1, 64, BF16, [9000]), (2060, 1, 1, 64, F16, [17000]),
                                                           (2100, 1, 5, 128, BF16, [17100, 36000]), (24, 200, 1, 64, F16, [17000]), (24, 200, 2, 256, BF16, [16500])])
def test_long_ones_among_many_sequences(dev, B, heads, group, D, dtype, longest):
    """A few long sequences among hundreds (in ranges) and thousands, or of very many heads (a workgroup for each)."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(B)
    lengths = [1 + (37 * b) % 100 for b in range(B)]
    where = [(7 + 255 * i) % B for i in range(len(longest))]
    for b, n in zip(where, longest):
        lengths[b] = n
    cache, M = filled(dev, lengths, heads, D, dtype)
    q = torch.randn(B, heads * group, 1, D, generator=g).to(dtype).to(dev)
    for mask in masks_of(g, dev, B, heads * group, 1, M, lengths):
        o, lse = fm.cache_attention_lse(q, cache, mask, scale_of(D))
        agrees(o, lse, q, cache, where + [0, 3, B - 1], range(heads * group), mask, [1] * B)
    cache.check()


@pytest.mark.parametrize("heads,group,D,N,dtype,lengths", [(192, 1, 64, 1, F16, [40000, 33000]), (128, 2, 128, 1, BF16, [37000, 45000]), (128, 1, 256, 3, F16, [41000, 30000]),
                                                           (64, 1, 128, 40, BF16, [90000, 61000])])
def test_long_ranges(dev, heads, group, D, N, dtype, lengths):
    """Few workgroups a head: ranges of hundreds of pages, cut inside a sequence."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(heads + D)
    cache, M = filled(dev, lengths, heads, D, dtype)
    q = torch.randn(2, heads * group, N, D, generator=g).to(dtype).to(dev)
    some = [0, 1, heads * group // 2, heads * group - 2, heads * group - 1]
    for mask in masks_of(g, dev, 2, heads * group, 1, M, lengths):
        o, lse = fm.cache_attention_lse(q, cache, mask, scale_of(D))
        agrees(o, lse, q, cache, [0, 1], some, mask, [N, N])
    cache.check()


@pytest.mark.parametrize("B,group,N,D,dtype", [(130, 4, 128, 64, F16), (150, 3, 150, 128, BF16), (1030, 3, 21, 256, F16)])
def test_many_pieces_with_masks(dev, B, group, N, D, dtype):
    """More tiles than ranges are made for, with the mask's rows of 64 queries, one of the sequences long."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(B)
    lengths = [1 + (61 * b) % 500 for b in range(B)]
    lengths[5], lengths[B - 1] = 5000, 17000
    counts = [min(n, N if b % 2 else 1 + b % N) for b, n in enumerate(lengths)]
    assert B * -(-N * group // 32) > 2048
    cache, M = filled(dev, lengths, 1, D, dtype)
    q = torch.randn(B, group, N, D, generator=g).to(dtype).to(dev)
    for mask in masks_of(g, dev, B, group, -(-N // PAGE), M, lengths):
        o, lse = fm.cache_attention_lse(q, cache, mask, scale_of(D), counts=ints(counts, dev))
        agrees(o, lse, q, cache, [0, 1, 5, 6, 77, B - 1], range(group), mask, counts)
        assert not bool(o[0, :, counts[0]:].any())
    cache.check()


def test_large_scores(dev):
    """A maximum that grows from page to page, scores that 32 bits of an exponential cannot hold."""
    g = torch.Generator().manual_seed(12)
    cache, ref = make(dev, 12, 1, 64, 1, 500, F16)
    k, v = tokens(1, 1, 450, 64, F16, g, dev)
    k = (k * torch.linspace(0, 60, 450, device=dev)[:, None]).to(F16)
    append(cache, ref, k, v)
    attend(cache, ref, (8 * torch.randn(1, 2, 450, 64, generator=g)).to(F16).to(dev), scale=1.0)


@pytest.mark.parametrize("D,dtype", [(64, BF16), (128, F16), (256, BF16)])
def test_values_that_are_not_numbers(dev, D, dtype):
    """In what a query does not see (behind its position, in pages that its head does not keep) they do not show; in what it sees they do, in
    the columns that share their scale."""
    g = torch.Generator().manual_seed(13)
    cache, ref = make(dev, 12, 1, D, 3, 300, dtype)
    k, v = tokens(3, 1, 200, D, dtype, g, dev)
    v[0, 0, 150, 40] = math.nan
    v[0, 0, 199, 1] = math.inf
    k[1, 0, 130, 3] = -math.inf
    v[2, 0, 70] = math.nan
    append(cache, ref, k, v, counts=[200, 200, 200])
    q = torch.randn(3, 3, 60, D, generator=g).to(dtype).to(dev)
    o, _ = attend(cache, ref, q)                                   # (positions 140 .. 199)
    assert bool(torch.isnan(o[0]).any()) and not bool(torch.isnan(o[0]).all())
    mask = torch.ones(1, 3, 1, 5, dtype=torch.bool)
    mask[0, 1, 0, 1] = False                                       # tokens 64 .. 127: head 1 leaves them out
    mask[0, 2, 0, 2] = False
    o, _ = attend(cache, ref, q, mask=mask)
    assert bool(torch.isnan(o[2, 0]).all()) and bool(torch.isfinite(o[2, 1]).all())
    # queries that are not finite
    q[1, 0, 5, 2] = math.inf
    q[1, 2, 7] = math.nan
    import fa2_custom_mask as fm
    o = fm.cache_attention(q, cache, None, scale_of(D))
    assert bool(torch.isnan(o[1, 2, 7]).all()) and bool(torch.isnan(o[1, 0, 5]).any())


def test_pages_that_do_not_exist(dev):
    """Numbers in the page table that the cache does not have are never followed; they are reported."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(14)
    cache, ref = make(dev, 12, 1, 64, 3, 300, F16)
    append(cache, ref, *tokens(2, 1, 200, 64, F16, g, dev))
    for wrong in (12, -1, 1 << 30, -(1 << 31)):
        good = cache.page_table.clone()
        cache.page_table[0, 1] = wrong
        q = torch.randn(2, 1, 1, 64, generator=g).to(F16).to(dev)
        o = fm.cache_attention(q, cache, None, 0.125)
        said(cache, {2})
        k, v = [np.delete(x, np.s_[64:128], axis=1) for x in ref.values(0)]
        ro, _, mean = attention(q[0].double().cpu().numpy(), k, v, 200, 0.125)
        assert within(o[0], ro, mean, F16)
        fm.cache_read(cache, 200)
        said(cache, {2})
        fm.cache_fork(cache, ints([0], dev), ints([2], dev))
        said(cache, {2})
        assert cache.lengths.tolist() == ref.length
        k, v = tokens(2, 1, 5, 64, F16, g, dev)
        fm.cache_append(cache, k, v, at=ints([70, 200], dev))
        said(cache, {2})
        ref.append(k[1:], v[1:], at=[200], sequences=[1])
        assert cache.lengths.tolist() == ref.length and cache.refs.tolist() == ref.refs
        cache.page_table.copy_(good)
        same_tables(cache, ref)
    cache.lengths[1] = 1 << 30                                     # beyond the table: taken for as long as that has room
    fm.cache_attention(q, cache, None, 0.125)
    said(cache, {2})


@pytest.mark.parametrize("rows,sequences", [(3, 4200), (64, 4200), (70, 90), (256, 9000), (300, 9000), (1024, 5000)])
def test_rows_that_name_a_sequence_twice(dev, rows, sequences):
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(16)
    cache, ref = make(dev, 1200, 1, 64, sequences, 64, F16)
    for _ in range(3):                        # the first row of a sequence stands, however far the second is from it
        named = torch.randperm(sequences, generator=g)[:rows].tolist()
        if sequences > 4096:
            named[rows // 2] = (named[0] + 4096) % 8192 if (named[0] + 4096) % 8192 < sequences else named[0] % 100
        again = named[:-1] + [named[0]]
        assert append(cache, ref, *tokens(rows, 1, 2, 64, F16, g, dev), sequences=again) == {0}
        said(cache, {0})
        same_tables(cache, ref)
        words = append(cache, ref, *tokens(rows, 1, 2, 64, F16, g, dev), sequences=list(reversed(named)))
        said(cache, words)
        same_tables(cache, ref)
        fm.cache_free(cache)
        ref.free(range(sequences))


@pytest.mark.parametrize("pages", [2, 3, 9, 5000])
def test_holders_below_zero(dev, pages):
    """Pages whose number of holders is below zero are free: compact has a target for each page it moves, append takes them."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(pages)
    cache, ref = make(dev, pages, 1, 64, 2, 64 * pages, F16)
    k, v = tokens(1, 1, 100, 64, F16, g, dev)
    used = [pages - 1, (pages - 1) // 2]                             # pages of sequence 1, in this order
    cache.refs[:] = torch.tensor([-1 - p % 3 for p in range(pages)], dtype=torch.int32)
    cache.refs[used] = 0
    others = [p for p in range(pages) if p not in used]
    saved = cache.refs.clone()
    cache.refs[others] = 1
    fm.cache_append(cache, k, v, sequences=ints([1], dev))       # (the two pages that are left, lowest number first)
    assert cache.page_table[1, :2].tolist() == used[::-1]
    cache.refs.copy_(saved)
    cache.refs[used] = 1
    want = [stands_for(x[0].double().cpu().numpy(), F16) for x in (k, v)]
    fm.cache_compact(cache)
    assert cache.refs[:2].tolist() == [1, 1] and bool((cache.refs[2:] <= 0).all())
    assert sorted(cache.page_table[1, :2].tolist()) == [0, 1]
    for x, y in zip(fm.cache_read(cache, 100, sequences=ints([1], dev)), want):
        assert np.array_equal(x[0].double().cpu().numpy(), y)
    if pages > 4:
        fm.cache_append(cache, *[x[:, :, :70] for x in (k, v)], sequences=ints([0], dev))
        assert cache.page_table[0, :2].tolist() == [2, 3] and cache.refs[:4].tolist() == [1, 1, 1, 1]
    cache.check()


def test_pages_given_up_more_often_than_held(dev):
    """Tables that name a page more often than its number of holders says: it is free once, and never held by less than nobody."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(17)
    cache, _ = make(dev, 8, 1, 64, 6, 256, F16)
    cache.page_table[:, :2] = ints([[3, 3], [3, 5], [3, 5], [5, 3], [6, 3], [-1, -1]], dev)
    cache.lengths[:5] = 128
    cache.refs[:] = ints([0, 0, 0, 2, 0, 4, 0, 0], dev)
    cache = fm.PagedCache4.of(cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.page_table, cache.lengths, cache.refs, F16)

    def found(match):
        with pytest.raises(RuntimeError, match=match):
            cache.check()
        cache.check()

    # by a copy on write of three rows, of which the page has two holders
    fm.cache_append(cache, *tokens(3, 1, 64, 64, F16, g, dev), at=ints([64, 0, 0], dev))
    found("more often than refs says")
    assert cache.refs.tolist() == [1, 1, 1, 0, 0, 2, 0, 0] and cache.lengths.tolist() == [128, 64, 64, 128, 128, 0]
    assert cache.page_table[:3, :2].tolist() == [[3, 0], [1, -1], [2, -1]]
    # by an append that cuts, and by cache_free
    fm.cache_append(cache, *tokens(1, 1, 0, 64, F16, g, dev), at=ints([5], dev), sequences=ints([3], dev))
    found("more often than refs says")
    assert cache.refs.tolist() == [1, 1, 1, 0, 0, 2, 0, 0] and cache.page_table[3].tolist() == [5, -1, -1, -1]
    fm.cache_free(cache)
    found("more often than refs says")
    assert cache.refs.tolist() == [0, 0, 0, 0, 0, 1, 0, 0] and bool((cache.page_table == -1).all()) and not bool(cache.lengths.any())
    fm.cache_compact(cache)
    fm.cache_append(cache, *tokens(1, 1, 200, 64, F16, g, dev))
    assert cache.refs.tolist() == [1, 1, 1, 1, 1, 0, 0, 0]
    cache.check()


@pytest.mark.parametrize("rows", [3, 100, 300])
def test_append_by_the_cache_s_own_numbers(dev, rows):
    """counts, at and sequences that are the cache's lengths themselves: they count as they were before the call."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(rows)
    cache, ref = make(dev, 3 * rows, 2, 64, rows, 300, F16)
    first = [(s + 1) % rows for s in range(rows)] if rows < 64 else [1 + s % 60 for s in range(rows)]
    assert not append(cache, ref, *tokens(rows, 2, 60, 64, F16, g, dev), counts=first)
    k, v = tokens(rows, 2, 60, 64, F16, g, dev)
    fm.cache_append(cache, k, v, counts=cache.lengths)                            # twice as many of each
    assert not ref.append(k, v, counts=first)
    same_tables(cache, ref)
    same_values(cache, ref)
    fm.cache_append(cache, k[:, :, :7], v[:, :, :7], at=cache.lengths)
    assert not ref.append(k[:, :, :7], v[:, :, :7], at=list(ref.length))
    same_tables(cache, ref)
    same_values(cache, ref)
    if rows < 64:
        fm.cache_append(cache, k[:, :, :0], v[:, :, :0], at=ints(first, dev))       # (lengths: a permutation of the sequences)
        ref.append(k[:, :, :0], v[:, :, :0], at=first)
        fm.cache_append(cache, k[:, :, :9], v[:, :, :9], sequences=cache.lengths)
        assert not ref.append(k[:, :, :9], v[:, :, :9], sequences=first)
        same_tables(cache, ref)
        same_values(cache, ref)
    cache.check()


def test_free_and_fork_by_the_cache_s_own_numbers(dev):
    """keep, sequences, parents and children that are the cache's tables themselves: they count as they were before the call."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(18)
    S = 30000                                                               # (many times the workgroups that are on the GPU at once)
    cache = fm.PagedCache4(2 * S, 1, 64, S, 128, F16, dev)
    for _ in range(3):
        lengths = torch.randint(1, 129, (S,), generator=g, dtype=torch.int32)
        pages = torch.arange(2 * S, dtype=torch.int32).view(S, 2)
        pages[lengths <= PAGE, 1] = -1
        cache.page_table.copy_(pages), cache.lengths.copy_(lengths)
        cache.refs.zero_()[pages[pages >= 0].long().to(dev)] = 1
        order = torch.randperm(S, generator=g)
        fm.cache_free(cache, order.to(dev), keep=cache.lengths)               # sequence order[i] to the length of sequence i
        want = lengths.clone()
        want[order] = torch.minimum(lengths[order], lengths)
        pages[want <= PAGE, 1] = -1
        assert torch.equal(cache.lengths.cpu(), want) and torch.equal(cache.page_table.cpu(), pages)
        assert int(cache.refs.sum()) == int((pages >= 0).sum()) == int((cache.refs > 0).sum())
    # lengths that are numbers of sequences: parents 3, 4, 5, and their children 0, 1, 2
    cache, ref = make(dev, 20, 1, 64, 6, 128, F16)
    append(cache, ref, *tokens(6, 1, 5, 64, F16, g, dev), counts=[0, 0, 0, 3, 4, 5])
    fm.cache_fork(cache, cache.lengths[3:], ints([0, 1, 2], dev))
    assert not ref.fork([3, 4, 5], [0, 1, 2])
    same_tables(cache, ref)
    fm.cache_free(cache, cache.lengths[3:], cache.lengths[:3] - 3)
    assert not ref.free([3, 4, 5], [0, 1, 2])
    same_tables(cache, ref)
    cache.check()


def test_every_report_is_told(dev):
    """Reports of several kinds since the last look are all in the error, each kind once, and in no later one."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(20)
    texts = ("a row that it refused", "found no free page", "a page number in page_table")

    def told(words):
        torch.cuda.synchronize()
        with pytest.raises(RuntimeError) as e:
            cache.check()
        assert [str(e.value).count(x) for x in texts] == [int(w in words) for w in range(3)]
        cache.check()

    cache, ref = make(dev, 3, 1, 64, 4, 256, F16)
    k, v = tokens(3, 1, 100, 64, F16, g, dev)
    assert append(cache, ref, k, v, sequences=[0, 9, 1]) == {0, 1}         # one call: a bad row, and one without pages
    told({0, 1})
    same_tables(cache, ref)
    assert append(cache, ref, k[:1], v[:1], sequences=[2]) == {1}
    told({1})
    cache.page_table[0, 1] = 77
    for twice in range(2):
        fm.cache_attention(k[:, :, :1], cache, None, 0.1, sequences=ints([0, -1, 1], dev))
        if twice:
            told({0, 2})
        torch.cuda.synchronize()
        if not twice:
            with pytest.raises(RuntimeError, match="refused.*page_table"):
                fm.cache_read(cache, 1)                                    # (any later call tells, and is not made)
    fm.cache_attention(k[:1, :, :1], cache, None, 0.1)
    told({2})


def test_tables_put_back(dev):
    """The tensors of a cache, saved and put back behind a compaction; appends then take what they took the first time."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(21)
    cache, ref = make(dev, 40, 1, 64, 5, 640, F16)
    append(cache, ref, *tokens(5, 1, 300, 64, F16, g, dev))
    fm.cache_free(cache, ints([0, 2], dev), ints([0, 100], dev))
    ref.free([0, 2], [0, 100])
    x = tokens(5, 1, 90, 64, F16, g, dev)
    state = [cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.page_table, cache.lengths, cache.refs, cache.free_from]
    saved = [t.clone() for t in state]
    fm.cache_append(cache, *x)
    want = [t.clone() for t in state]
    for a, b in zip(state, saved):
        a.copy_(b)
    fm.cache_compact(cache)
    assert int(cache.free_from) == 5 * 5 - 5 - 3
    for a, b in zip(state, saved):
        a.copy_(b)
    assert not append(cache, ref, *x)
    same_tables(cache, ref)
    same_values(cache, ref)
    assert all(torch.equal(a, b) for a, b in zip(state[4:], want[4:]))
    cache.check()


def test_free_from_that_is_refused(dev):
    import fa2_custom_mask as fm
    a, _ = make(dev, 4, 1, 64, 2, 128, F16)
    tensors = (a.k_codes, a.k_scales, a.v_codes, a.v_scales, a.page_table, a.lengths, a.refs)
    for bad, error in ((ints([0, 0], dev), ValueError), (ints([[0]], dev), ValueError), (ints([0], dev, torch.int64), TypeError), (ints([0], "cpu"), RuntimeError)):
        with pytest.raises(error):
            fm.PagedCache4.of(*tensors, F16, free_from=bad)


@pytest.mark.parametrize("rows,pages", [(1, 7), (1, 3), (1, 6000), (80, 500), (300, 3000)])
def test_free_from_too_high(dev, rows, pages):
    """A note of free pages that is too high (refs written to, or pages freed by another handle): free pages from there on come first, then those
    below; no row is refused for it, and afterwards the note is right again."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(pages)
    D, M = 64, max(1, pages // rows - 1)
    a, _ = make(dev, pages, 1, D, rows + 1, M * PAGE, F16)
    k, v = [x.expand(rows, 1, -1, -1) for x in tokens(1, 1, M * PAGE, D, F16, g, dev)]
    tensors = (a.k_codes, a.k_scales, a.v_codes, a.v_scales, a.page_table, a.lengths, a.refs)
    other, shared = fm.PagedCache4.of(*tensors, F16), fm.PagedCache4.of(*tensors, F16, free_from=a.free_from)
    assert shared.free_from.data_ptr() == a.free_from.data_ptr() and int(other.free_from) == 0
    fm.cache_append(a, k, v)
    used = rows * M
    assert int(a.free_from) == used
    fm.cache_free(other, ints(list(range(rows)), dev))                     # `a` does not hear of it
    assert int(a.free_from) == used and int(other.free_from) == 0 and not bool(a.refs.any())
    fm.cache_append(a, k, v)                                               # (fewer than that many pages are left behind the note)
    a.check()
    assert a.page_table[:rows].flatten().tolist() == list(range(used)) and int(a.free_from) == used
    # enough of them behind the note: these are taken
    fm.cache_free(shared, ints([0], dev))
    assert int(a.free_from) == 0
    a.free_from.fill_(used)
    fm.cache_append(a, k[:1, :, :1], v[:1, :, :1])
    a.check()
    assert int(a.page_table[0, 0]) == used and int(a.free_from) == used + 1
    # a row that finds too few anywhere is refused; one that does not need more than there are is not
    some = sorted(torch.randperm(pages, generator=g)[:M - 1].tolist())
    a.refs.fill_(1)
    a.refs[some] = 0
    a.free_from.fill_(some[-1])
    fm.cache_append(a, k[:1], v[:1], sequences=ints([rows], dev))
    with pytest.raises(RuntimeError, match="no free page"):
        a.check()
    assert int(a.free_from) == 0 and int(a.lengths[rows]) == 0
    a.free_from.fill_(pages)
    fm.cache_append(a, k[:1, :, 64:], v[:1, :, 64:], sequences=ints([rows], dev))
    a.check()
    assert a.page_table[rows].tolist() == some + [-1] and int(a.free_from) == some[-1] + 1


def test_rows_that_are_refused(dev):
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(15)
    cache, ref = make(dev, 12, 1, 64, 3, 300, F16)
    append(cache, ref, *tokens(2, 1, 100, 64, F16, g, dev))
    q = torch.randn(4, 2, 3, 64, generator=g).to(F16).to(dev)
    o, lse = fm.cache_attention_lse(q, cache, None, 0.1, counts=ints([3, 4, 3, -1], dev), sequences=ints([0, 1, 3, 1], dev))
    assert bool((o[1:] == 0).all()) and bool((lse[1:] == -math.inf).all()) and bool((o[0] != 0).any())
    said(cache, {0})
    k, _ = fm.cache_read(cache, 5, sequences=ints([-1, 0], dev))
    assert not bool(k[0].any()) and bool(k[1].any())
    said(cache, {0})
    for kw in ({"at": [101, 5]}, {"at": [-1, 5]}, {"counts": [-1, 3]}, {"counts": [8, 3]}, {"sequences": [3, 1]}, {"sequences": [1, 1]}):
        assert append(cache, ref, *tokens(2, 1, 7, 64, F16, g, dev), **kw) == {0}
        said(cache, {0})
        same_tables(cache, ref)
    assert append(cache, ref, *tokens(1, 1, 260, 64, F16, g, dev)) == {0}
    said(cache, {0})
    same_tables(cache, ref)
    for parents, children in (([0], [1]), ([0], [0]), ([0, 2], [2, 2]), ([2], [0]), ([5], [2]), ([0], [-1]), ([0, 0], [2, 2])):
        fm.cache_fork(cache, ints(parents, dev), ints(children, dev))
        words = ref.fork(parents, children)
        assert words == {0}
        said(cache, words)
        same_tables(cache, ref)
        ref.free([2])
        fm.cache_free(cache, ints([2], dev))
    same_values(cache, ref)


def test_refusals(dev):
    """What is wrong with the arguments themselves raises at once and enqueues nothing."""
    import fa2_custom_mask as fm
    cache, _ = make(dev, 4, 2, 64, 3, 128, F16)
    x = lambda *s, dtype=F16: torch.zeros(*s, dtype=dtype, device=dev)     # noqa: E731
    k = x(1, 2, 5, 64)
    with pytest.raises(RuntimeError):
        fm.cache_append(cache, k.cpu(), k.cpu())
    with pytest.raises(TypeError):
        fm.cache_append(cache, k.to(BF16), k.to(BF16))
    for bad in (x(1, 3, 5, 64), x(1, 2, 5, 128), x(2, 5, 64), x(4, 2, 5, 64), x(0, 2, 5, 64), x(1, 2, 129, 64)):
        with pytest.raises(ValueError):
            fm.cache_append(cache, bad, bad)
    with pytest.raises(ValueError):
        fm.cache_append(cache, k, x(1, 2, 4, 64))
    for name in ("at", "counts", "sequences"):
        for bad, error in ((ints([0, 0], dev), ValueError), (ints([[0]], dev), ValueError), (x(1), TypeError), (torch.zeros(1, dtype=torch.int32), RuntimeError)):
            with pytest.raises(error):
                fm.cache_append(cache, k, k, **{name: bad})
    with pytest.raises(RuntimeError):
        fm.cache_append(cache, k.clone().requires_grad_(), k)
    q = x(1, 4, 5, 64)
    ok = torch.ones(1, 1, 1, 2, dtype=torch.bool, device=dev)
    fm.cache_attention(q, cache, ok, 0.1)
    for bad in (x(1, 3, 5, 64), x(1, 0, 5, 64), x(1, 4, 0, 64), x(4, 4, 1, 64), x(1, 4, 5, 32)):
        with pytest.raises(ValueError):
            fm.cache_attention(bad, cache, None, 0.1)
    with pytest.raises(TypeError):
        fm.cache_attention(q.to(BF16), cache, None, 0.1)
    with pytest.raises(RuntimeError):
        fm.cache_attention(q.clone().requires_grad_(), cache, None, 0.1)
    with torch.no_grad():
        fm.cache_attention(q.clone().requires_grad_(), cache, None, 0.1)
    for bad in (ok[0], ok.expand(2, 1, 1, 2), ok.expand(1, 3, 1, 2), ok.expand(1, 1, 2, 2), torch.ones(1, 1, 1, 3, dtype=torch.bool, device=dev)):
        with pytest.raises(ValueError):
            fm.cache_attention(q, cache, bad, 0.1)
    with pytest.raises(TypeError):
        fm.cache_attention(q, cache, ok.int(), 0.1)
    with pytest.raises(RuntimeError):
        fm.cache_attention(q, cache, ok.cpu(), 0.1)
    with pytest.raises(ValueError):
        fm.cache_read(cache, 0)
    with pytest.raises(ValueError):
        fm.cache_fork(cache, ints([0], dev), ints([1, 2], dev))
    with pytest.raises(ValueError):
        fm.cache_fork(cache, ints([], dev), ints([], dev))
    with pytest.raises(ValueError):
        fm.cache_free(cache, ints([0, 1, 2, 0], dev))
    for args in ((4, 2, 48, 3, 128), (0, 2, 64, 3, 128), (4, 2, 64, 3, 0)):
        with pytest.raises(ValueError):
            fm.PagedCache4(*args, F16, dev)
    with pytest.raises(TypeError):
        fm.PagedCache4(4, 2, 64, 3, 128, torch.float32, dev)
    t = (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales, cache.page_table, cache.lengths, cache.refs)
    fm.PagedCache4.of(*t, F16)
    for i in range(7):
        with pytest.raises(ValueError):
            fm.PagedCache4.of(*t[:i], torch.cat((t[i], t[i])), *t[i + 1:], F16)
        with pytest.raises(TypeError):
            fm.PagedCache4.of(*t[:i], t[i].short(), *t[i + 1:], F16)
    cache.check()


def test_tangents_are_refused(dev):
    """A dual tensor that requires no gradient: its tangent would be dropped without a word."""
    import torch.autograd.forward_ad as fwad
    import fa2_custom_mask as fm
    cache, _ = make(dev, 4, 2, 64, 3, 128, F16)
    x = torch.ones(1, 2, 5, 64, dtype=F16, device=dev)
    with fwad.dual_level():
        dual = fwad.make_dual(x, torch.ones_like(x))
        for call in (lambda: fm.cache_append(cache, dual, x), lambda: fm.cache_append(cache, x, dual), lambda: fm.cache_attention(dual, cache, None, 0.1),
                     lambda: fm.cache_attention_lse(dual, cache, None, 0.1)):
            with pytest.raises(RuntimeError, match="tangent"):
                call()
            with torch.no_grad(), pytest.raises(RuntimeError, match="tangent"):
                call()
        assert not bool(cache.lengths.any())
        fm.cache_append(cache, fwad.unpack_dual(dual).primal.detach(), x)
        with torch.inference_mode():
            fm.cache_attention(dual, cache, None, 0.1)                     # (nothing is differentiated in there)
    fm.cache_append(cache, dual, x)                                        # behind its level a dual tensor is none
    cache.check()


# ---- as they are used ----
def test_far_pages(dev):
    """Codes beyond 4 GB from where they begin."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(16)
    pages = 70000
    cache = fm.PagedCache4(pages, 8, 256, 2, 300, BF16, dev)
    assert cache.k_codes.numel() > 1 << 32
    cache.refs[:pages - 12] = 1
    near, ref = make(dev, 12, 8, 256, 2, 300, BF16)
    k, v = tokens(2, 8, 200, 256, BF16, g, dev)
    fm.cache_append(cache, k, v)
    append(near, ref, k, v)
    assert torch.equal(cache.page_table, torch.where(near.page_table >= 0, near.page_table + pages - 12, -1))
    q = torch.randn(2, 8, 3, 256, generator=g).to(BF16).to(dev)
    assert torch.equal(fm.cache_attention(q, cache, None, 0.1), fm.cache_attention(q, near, None, 0.1))
    assert all(torch.equal(a, b) for a, b in zip(fm.cache_read(cache, 200), fm.cache_read(near, 200)))
    cache.refs[:pages - 12] = 0
    fm.cache_compact(cache)
    assert torch.equal(cache.page_table, near.page_table)
    assert all(torch.equal(a, b) for a, b in zip(fm.cache_read(cache, 200), fm.cache_read(near, 200)))
    cache.check()


def test_prompt_and_steps(dev):
    """A prompt through flash_attention_custom_mask on the values that the cache serves, then the same queries over the cache with the block
    mask's rows: one result; then steps."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(17)
    H, D, N = 4, 128, 300
    cache, ref = make(dev, 16, H, D, 3, 400, BF16)
    k, v = tokens(1, H, N, D, BF16, g, dev)
    q = torch.randn(1, H, N, D, generator=g).to(BF16).to(dev)
    append(cache, ref, k, v, sequences=[1])
    kept, vals = fm.cache_read(cache, N, sequences=ints([1], dev))
    nb = -(-N // PAGE)
    blocks = (torch.rand(1, H, nb, nb, generator=g) < 0.6) | torch.eye(nb, dtype=torch.bool)
    dense = (blocks.repeat_interleave(PAGE, 2).repeat_interleave(PAGE, 3)[..., :N, :N] & torch.ones(N, N, dtype=torch.bool).tril()).to(dev)
    whole = fm.flash_attention_custom_mask(q, kept, vals, dense, scale_of(D))
    mask = torch.zeros(1, H, nb, cache.page_table.shape[1], dtype=torch.bool)
    mask[..., :nb] = blocks
    o, _ = attend(cache, ref, q, mask=mask, sequences=[1])
    assert float((o.float() - whole.float()).abs().max()) <= 6e-2               # (both within the bounds of bf16 numerators: |v| of up to 6)
    fm.cache_fork(cache, ints([1, 1], dev), ints([0, 2], dev))
    ref.fork([1, 1], [0, 2])
    for step in range(3):
        append(cache, ref, *tokens(3, H, 1, D, BF16, g, dev))
        attend(cache, ref, torch.randn(3, 2 * H, 1, D, generator=g).to(BF16).to(dev))
        if step == 0:
            fm.cache_free(cache, ints([2], dev), ints([250], dev))
            ref.free([2], [250])
        if step == 1:
            fm.cache_compact(cache)
            ref.compact()
    same_tables(cache, ref)
    same_values(cache, ref)


def test_captured_steps(dev):
    """A step (append, attention) captured once and replayed while the sequences grow, beside eager work on the same streams; two graphs at a
    time have workspaces of their own."""
    import fa2_custom_mask as fm
    H, D, S = 2, 128, 3
    def state(seed):
        g = torch.Generator().manual_seed(seed)
        pair = [make(dev, 400, H, D, S, 9000, F16) for _ in range(2)]
        k, v = tokens(S, H, 8000, D, F16, g, dev)
        for c, _ in pair:
            fm.cache_append(c, k, v, counts=ints([8000, 130, 63], dev))
        return pair[0][0], pair[1][0], g
    runs = []
    for seed in (1, 2):
        cache, eager, g = state(seed)
        k, v = tokens(S, H, 1, D, F16, g, dev)
        q = torch.randn(S, 2 * H, 1, D, generator=g).to(F16).to(dev)
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            fm.cache_attention_lse(q, cache, None, 0.1)
        torch.cuda.current_stream().wait_stream(stream)
        with torch.cuda.graph(graph):
            fm.cache_append(cache, k, v)
            out = fm.cache_attention_lse(q, cache, None, 0.1)
            back = fm.cache_read(cache, 5, start=cache.lengths - 5)
        runs.append((graph, cache, eager, (q, k, v), out, back, g))
    side = torch.cuda.Stream()
    for step in range(6):
        for graph, cache, eager, inputs, *_, g in runs:
            for x in inputs:
                x.copy_(torch.randn(x.shape, generator=g).to(F16))
        torch.cuda.synchronize()
        if step % 2:                                       # both at once
            side.wait_stream(torch.cuda.current_stream())
            runs[0][0].replay()
            with torch.cuda.stream(side):
                runs[1][0].replay()
            torch.cuda.current_stream().wait_stream(side)
        else:
            for r in runs:
                r[0].replay()
        for _, cache, eager, (q, k, v), out, back, _ in runs:
            fm.cache_append(eager, k, v)
            o, lse = fm.cache_attention_lse(q, eager, None, 0.1)
            read = fm.cache_read(eager, 5, start=eager.lengths - 5)
            torch.cuda.synchronize()
            assert torch.equal(out[0], o) and torch.equal(out[1], lse)
            assert all(torch.equal(a, b) for a, b in zip(back, read))
            assert torch.equal(cache.page_table, eager.page_table) and torch.equal(cache.lengths, eager.lengths)
            cache.check(), eager.check()


def test_graphs_that_share_a_pool(dev):
    """Graphs of one memory pool, whose workspaces may lie in the same place, replayed in any order, beside eager calls: bookkeeping and
    attention with parts of many workgroups, in 16 bits and in fp32."""
    import fa2_custom_mask as fm
    H, D, S, M = 2, 64, 4, 160
    g = torch.Generator().manual_seed(23)
    pair = [make(dev, 700, H, D, S, M * PAGE, BF16)[0] for _ in range(2)]
    k, v = tokens(S, H, 9000, D, BF16, g, dev)
    for c in pair:
        fm.cache_append(c, k, v, counts=ints([9000, 5000, 70, 0], dev))
    k1, v1 = tokens(S, H, 1, D, BF16, g, dev)
    q1, q3 = [torch.randn(S, 4 * H, n, D, generator=g).to(BF16).to(dev) for n in (1, 3)]
    mask = (torch.rand(1, 4 * H, 1, M, generator=g) < 0.5).to(dev)
    three = ints([0, 1, 2], dev)
    last, kept, child = ints([3], dev), ints([4000], dev, torch.int64), ints([1], dev, torch.int64)

    def step(c):
        fm.cache_append(c, k1[:3], v1[:3], sequences=three)
        return fm.cache_attention_lse(q1, c, None, 0.1, out_fp32=True) + (fm.cache_attention(q3, c, mask, 0.1),)

    def branch(c):
        fm.cache_free(c, last)
        fm.cache_fork(c, child, last)
        fm.cache_free(c, last, kept)
        fm.cache_append(c, k1[:1], v1[:1], sequences=last)
        fm.cache_compact(c)
        return fm.cache_attention_lse(q3, c, None, 0.1) + fm.cache_read(c, 70, start=c.lengths - 60)

    calls = (step, branch)
    cache, eager = pair
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        for q in (q1, q3):
            fm.cache_attention_lse(q, cache, None, 0.1, out_fp32=True)
            fm.cache_attention(q, cache, mask, 0.1)
    torch.cuda.current_stream().wait_stream(stream)
    graphs, outs = [], []
    for call in calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], pool=graphs[0].pool() if len(graphs) > 1 else None):
            outs.append(call(cache))
    for i in (0, 1, 0, 0, 1, 1, 0):
        for x in (k1, v1, q1, q3):
            x.copy_(torch.randn(x.shape, generator=g).to(BF16))
        graphs[i].replay()
        want = calls[i](eager)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs[i], want)), i
        assert torch.equal(cache.page_table, eager.page_table) and torch.equal(cache.lengths, eager.lengths) and torch.equal(cache.refs, eager.refs)
        assert torch.equal(cache.free_from, eager.free_from)
        cache.check(), eager.check()


def test_threads(dev):
    """Two threads, each with a cache and a stream of its own, and two that share both kinds of calls on one stream."""
    import threading
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(19)
    jobs = []
    for i in range(4):
        cache, _ = make(dev, 200, 2, 64, 3, 3000, F16)
        k, v = tokens(3, 2, 1500, 64, F16, g, dev)
        q = torch.randn(3, 4, 1, 64, generator=g).to(F16).to(dev)
        jobs.append((cache, k, v, q))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    streams += [streams[1]] * 2
    torch.cuda.synchronize()
    results = [None] * 4

    def work(i):
        cache, k, v, q = jobs[i]
        with torch.cuda.stream(streams[i]):
            for step in range(20):
                fm.cache_append(cache, k[:, :, step * 70:step * 70 + 70], v[:, :, step * 70:step * 70 + 70])
                out = fm.cache_attention(q, cache, None, 0.1)
            results[i] = out

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    for i, (cache, k, v, q) in enumerate(jobs):
        cache.check()
        rk, rv = [x.double().cpu().numpy() for x in fm.cache_read(cache, 1400)]
        want = stands_for(k[:, :, :1400].double().cpu().numpy(), F16)
        assert np.array_equal(rk, want)
        for b in range(3):
            ro, _, mean = attention(q[b].double().cpu().numpy(), rk[b], rv[b], 1399, 0.1)
            assert within(results[i][b], ro, mean, F16)


def test_streams(dev):
    """Calls on a stream that is not the default one, and on two at a time."""
    import fa2_custom_mask as fm
    g = torch.Generator().manual_seed(18)
    cache, ref = make(dev, 300, 1, 64, 2, 16000, BF16)
    k, v = tokens(2, 1, 9000, 64, BF16, g, dev)
    q = torch.randn(2, 3, 1, 64, generator=g).to(BF16).to(dev)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    with torch.cuda.stream(streams[0]):
        fm.cache_append(cache, k, v, counts=ints([9000, 500], dev))
        ready = streams[0].record_event()
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            s.wait_event(ready)
            results.append([fm.cache_attention(q, cache, None, 0.1) for _ in range(5)])
    torch.cuda.synchronize()
    want = fm.cache_attention(q, cache, None, 0.1)
    assert all(torch.equal(o, want) for r in results for o in r)
    rk, rv = [x.double().cpu().numpy() for x in fm.cache_read(cache, 500, sequences=ints([1], dev))]
    ro, _, mean = attention(q[1].double().cpu().numpy(), rk[0], rv[0], 499, 0.1)
    assert within(want[1], ro, mean, BF16)

"""The reference that the cache's GPU tests compare with, against the definition written out value by value, and the refusals of calls
that need no GPU."""
import ctypes
import math

import numpy as np
import pytest
import torch

from cache_reference import LARGEST, MAGNITUDES, Reference, stands_for, attention


def one_group(x, dtype):
    if not all(math.isfinite(v) for v in x):
        return [math.nan] * 32
    top = max(abs(v) for v in x)
    e = -127
    while e < LARGEST[dtype] and not top < 7 * 2.0 ** e:
        e += 1
    out = []
    for v in x:
        y = abs(v) / 2.0 ** e
        best = min(range(8), key=lambda i: (abs(MAGNITUDES[i] - y), i % 2))
        out.append(math.copysign(MAGNITUDES[best] * 2.0 ** e, v))
    return out


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_values_in_4_bits(dtype):
    g = torch.Generator().manual_seed(1)
    x = (torch.randn(40, 32, generator=g) * torch.exp(4 * torch.randn(40, 1, generator=g))).to(dtype).double()
    x[3] = 0
    x[4, 5] = math.inf
    x[5, 6] = math.nan
    x[6] = torch.tensor(MAGNITUDES * 4)
    x[7] = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0] * 4)      # ties
    x[8] = torch.finfo(dtype).max
    x[9] = torch.finfo(dtype).smallest_normal / 2
    got = stands_for(x.numpy(), dtype)
    want = np.array([one_group(r.tolist(), dtype) for r in x])
    assert np.array_equal(got, want, equal_nan=True)
    assert np.array_equal(got[6], x[6].numpy()) and list(got[7][:8]) == [0, 1, 1, 2, 2, 4, 4, 6]
    finite = torch.from_numpy(got[np.isfinite(got).all(1)])
    assert torch.equal(finite.to(dtype).double(), finite)                      # every value is one of the type


def test_reference_attention():
    g = np.random.default_rng(0)
    q, k, v = g.normal(size=(4, 3, 8)), g.normal(size=(2, 70, 8)), g.normal(size=(2, 70, 8))
    o, lse, _ = attention(q, k, v, 67, 0.3)
    s = torch.from_numpy(q[1, 2]) @ torch.from_numpy(k[0]).T * 0.3
    assert np.allclose(o[1, 2], (torch.softmax(s, -1) @ torch.from_numpy(v[0])).numpy()) and np.isclose(lse[1, 2], torch.logsumexp(s, -1))
    o, lse, _ = attention(q, k, v, -2, 0.3)
    assert not o[:, :2].any() and (lse[:, :2] == -np.inf).all() and np.allclose(o[3, 2], v[1, 0])


def test_reference_pages():
    r = Reference(6, 1, 64, 3, 256, torch.float16)
    x = lambda n: torch.ones(1, 1, n, 64)     # noqa: E731
    assert r.append(x(100), x(100), sequences=[1]) == set() and r.table[1] == [0, 1]
    assert r.fork([1], [0]) == set() and r.refs[:2] == [2, 2]
    assert r.append(x(1), x(1), sequences=[0]) == set() and r.table[0] == [0, 2] and r.refs[:3] == [2, 1, 1]
    assert r.append(x(200), x(200), sequences=[2]) == {1}                       # 3 free pages, 4 needed
    assert r.free([1]) == set() and r.refs[:3] == [1, 0, 1]
    r.compact()
    assert r.table[0] == [0, 1] and r.refs == [1, 1, 0, 0, 0, 0]


class CacheStruct(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("k_codes", "v_codes", "k_scales", "v_scales", "page_table", "lengths", "refs", "free_from", "status")] + \
               [(n, ctypes.c_int32) for n in ("pages", "heads", "head_dim", "sequences", "max_pages", "dtype")]


def struct(**kw):
    a = dict(k_codes=4096, v_codes=4096, k_scales=4096, v_scales=4096, page_table=4096, lengths=4096, refs=4096, free_from=4096, status=None,
             pages=8, heads=2, head_dim=64, sequences=3, max_pages=4, dtype=0)
    a.update(kw)
    return CacheStruct(**a)


def test_c_entry_points_refuse_bad_arguments():
    """Nothing is launched: the pointers are never followed."""
    from fa2_custom_mask import _ext
    l = _ext.lib()
    P, n = ctypes.c_void_p(4096), ctypes.c_size_t()
    ok = (ctypes.c_int64 * 4)(2 * 64 * 64, 64 * 64, 64, 1)
    inner, odd = (ctypes.c_int64 * 4)(2 * 64 * 64, 64 * 64, 64, 2), (ctypes.c_int64 * 4)(2 * 64 * 68, 64 * 68, 68, 1)
    ref = ctypes.byref
    big = 1 << 40

    def append(c=None, k=P, v=P, ks=ok, B=2, N=5, ws=P, wsb=big, seq=None):
        return l.bsattn_cache_append(ref(c or struct()), k, v, ks, ok, seq, None, None, B, N, ws, wsb, None)

    def attn(c=None, q=P, o=P, mask=None, ms=None, Bm=1, Hm=1, Nm=1, B=2, H=4, N=5, odt=0, qs=ok, os=ok, ws=P, wsb=big, seq=None):
        return l.bsattn_cache_attn(ref(c or struct()), q, o, None, mask, ms, Bm, Hm, Nm, seq, None, B, H, N, odt, 0.1, qs, os, ws, wsb, None)

    def read(c=None, k=P, v=P, ks=ok, B=2, N=5, seq=None):
        return l.bsattn_cache_read(ref(c or struct()), k, v, ks, ok, seq, None, B, N, None)

    for call in (append, attn, read):
        for field in ("k_codes", "v_codes", "k_scales", "v_scales", "page_table", "lengths", "refs", "free_from"):
            assert call(struct(**{field: None})) == -1
        for field in ("pages", "heads", "sequences", "max_pages"):
            assert call(struct(**{field: 0})) == -2
        assert call(struct(head_dim=96)) == -4 and call(struct(dtype=2)) == -3
        assert call(struct(k_codes=4100)) == -5 and call(struct(max_pages=1 << 26)) == -8 and call(struct(heads=70000)) == -8
        assert call(B=0) == -2 and call(B=4) == -2                               # (more rows than sequences, without a list of them)
        assert call(N=-1) == -2
    assert append(k=None) == -1 and append(v=None) == -1 and append(ks=None) == -1 and append(ks=inner) == -5 and append(ks=odd) == -5
    assert append(k=ctypes.c_void_p(4100)) == -5 and append(B=1025, seq=P) == -8 and append(N=257) == -8
    assert append(ws=None) == -6 and append(wsb=8) == -6 and append(ws=ctypes.c_void_p(4100)) == -5
    assert read(k=None) == -1 and read(ks=odd) == -5 and read(N=0) == -2
    assert attn(q=None) == -1 and attn(o=None) == -1 and attn(qs=inner) == -5 and attn(os=odd) == -5 and attn(H=3) == -2 and attn(N=0) == -2
    assert attn(odt=1) == -3 and attn(mask=P) == -1 and attn(mask=P, ms=ok, Bm=3) == -2 and attn(mask=P, ms=ok, Hm=3) == -2 and attn(mask=P, ms=ok, Nm=2) == -2
    assert attn(ws=None) == -6 and attn(wsb=8) == -6 and attn(N=1 << 30) == -8
    assert l.bsattn_cache_attn_workspace(ref(struct()), 2, 4, 5, None) == -1 and l.bsattn_cache_attn_workspace(ref(struct()), 2, 4, 5, ref(n)) == 0 and n.value > 0
    assert l.bsattn_cache_append_workspace(None, 2, 5, ref(n)) == -1
    assert l.bsattn_cache_fork(ref(struct()), None, P, 1, None) == -1 and l.bsattn_cache_fork(ref(struct()), P, P, 0, None) == -2
    assert l.bsattn_cache_fork(ref(struct()), P, P, 4, None) == -8
    assert l.bsattn_cache_free(ref(struct()), None, None, 0, None) == -2 and l.bsattn_cache_free(ref(struct()), None, None, 4, None) == -8
    assert l.bsattn_cache_compact(ref(struct()), None, big, None) == -6 and l.bsattn_cache_compact(ref(struct()), P, 8, None) == -6
    assert l.bsattn_cache_compact_workspace(ref(struct(refs=None)), ref(n)) == -1


def test_no_cpu_path():
    import fa2_custom_mask as fm
    with pytest.raises(RuntimeError):
        fm.PagedCache4(4, 1, 64, 1, 128, device="cpu")
    with pytest.raises(ValueError):
        fm.PagedCache4(0, 1, 64, 1, 128, device="cpu")

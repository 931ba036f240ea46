"""What stands around a step over the token cache, and attention through a window and over shared pages, without a
GPU: what the entry points refuse, and the 64-bit oracle against torch and against itself."""
import ctypes
import math

import numpy as np
import pytest
import torch

from chestnut import _lib
from chestnut import kernels as K
from oracle import token_cache as O

f16, bf16, f32, i32 = torch.float16, torch.bfloat16, torch.float32, torch.int32


def z(*shape, dtype=f16):
    return torch.zeros(*shape, dtype=dtype)


F = torch.ones(16, dtype=torch.float64)
A = torch.zeros(16, dtype=i32)


def norm(q=None, k=None, wq=None, wk=None, pos=None, f=F, **kw):
    return K.norm_rope(z(4, 2, 64) if q is None else q, z(4, 1, 64) if k is None else k, z(64) if wq is None else wq,
                       z(64) if wk is None else wk, z(4, dtype=i32) if pos is None else pos, f, **kw)


def maps(new=None, kv=None, table=None, page=16, tokens=8, **kw):
    return K.cache_maps(z(3, dtype=i32) if new is None else new, z(3, dtype=i32) if kv is None else kv,
                        z(3, 5, dtype=i32) if table is None else table, page, tokens, **kw)


def varlen(**kw):
    return K.attention_varlen(z(4, 4, 64), z(4, 2, 64), z(4, 2, 64), z(3, dtype=i32), **kw)


def paged(**kw):
    return K.attention_paged(z(4, 4, 64), z(3, 2, 16, 64), z(3, 2, 16, 64), z(2, 3, dtype=i32), z(3, dtype=i32), z(2, dtype=i32), **kw)


def groups(n=1, cu=None, lens=None):
    return (z(n + 1, dtype=i32) if cu is None else cu, z(n, dtype=i32) if lens is None else lens)


FREE = dict(free_pages=z(9, dtype=i32), taken=z(1, dtype=i32))
REFUSED = [
    ('rope axes type', lambda: K.rope(z(4, 2, 64), z(3, 4, dtype=i32), F, axes=A.long()), 'axes must be torch.int32'),
    ('rope axes length', lambda: K.rope(z(4, 2, 64), z(3, 4, dtype=i32), F, axes=A[:15]), 'axes must have shape'),
    ('rope axes with one row of positions', lambda: K.rope(z(4, 2, 64), z(4, dtype=i32), F, axes=A), 'positions must be int32 \\[axes, T\\]'),
    ('rope axes without positions', lambda: K.rope(z(4, 2, 64), z(0, 4, dtype=i32), F, axes=A), 'positions must be int32 \\[axes, T\\]'),
    ('rope rows of positions without axes', lambda: K.rope(z(4, 2, 64), z(3, 4, dtype=i32), F), 'positions must have shape'),
    ('rope positions of several axes type', lambda: K.rope(z(4, 2, 64), z(3, 4, dtype=torch.int64), F, axes=A), 'positions must be torch.int32'),
    ('rope positions of several axes length', lambda: K.rope(z(4, 2, 64), z(3, 5, dtype=i32), F, axes=A), 'positions must have shape'),
    ('rope positions transposed', lambda: K.rope(z(4, 2, 64), z(4, 3, dtype=i32).T, F, axes=A), 'positions must be contiguous'),
    ('rope axes cpu tensors', lambda: K.rope(z(4, 2, 64), z(3, 4, dtype=i32), F, axes=A), 'must be a CUDA tensor'),
    ('sections empty', lambda: K.rope_axes([]), 'sections must be'),
    ('sections without pairs', lambda: K.rope_axes([0, 0]), 'sections must be'),
    ('sections negative', lambda: K.rope_axes([4, -1]), 'sections must be'),
    ('sections fractions', lambda: K.rope_axes([4, 1.5]), 'sections must be'),
    ('norm q type', lambda: norm(z(4, 2, 64, dtype=f32)), 'q must be float16 or bfloat16'),
    ('norm q rank', lambda: norm(z(4, 64)), 'q must be'),
    ('norm k type', lambda: norm(k=z(4, 1, 64, dtype=bf16)), 'k must be torch.float16'),
    ('norm k rows', lambda: norm(k=z(5, 1, 64)), 'k must have shape'),
    ('norm k head_dim', lambda: norm(k=z(4, 1, 128)), 'k must have shape'),
    ('norm k without heads', lambda: norm(k=z(4, 0, 64)), 'norm_rope takes'),
    ('norm k missing, its weight not', lambda: K.norm_rope(z(4, 2, 64), None, None, z(64), z(4, dtype=i32), F), 'belong to k'),
    ('norm k missing, k_out not', lambda: K.norm_rope(z(4, 2, 64), None, None, None, z(4, dtype=i32), F, k_out=z(4, 1, 64)), 'belong to k'),
    ('norm weight type', lambda: norm(wq=z(64, dtype=bf16)), 'q_weight must be torch.float16'),
    ('norm weights of two types', lambda: norm(wq=z(64, dtype=f32)), 'one type'),
    ('norm weight length', lambda: norm(wk=z(63)), 'k_weight must have shape'),
    ('norm weight strided', lambda: norm(wk=z(128)[::2]), 'k_weight must be contiguous'),
    ('norm eps zero', lambda: norm(eps=0.0), 'eps must be positive'),
    ('norm eps below the normal numbers', lambda: norm(eps=1e-40), 'eps must be positive'),
    ('norm eps nan', lambda: norm(eps=math.nan), 'eps must be positive'),
    ('norm eps infinite', lambda: norm(eps=math.inf), 'eps must be positive'),
    ('norm head_dim', lambda: norm(z(4, 2, 514), z(4, 1, 514), z(514), z(514)), 'head_dim up to 512'),
    ('norm elements', lambda: norm(z(1, 100, 512), z(1, 29, 512), z(512), z(512), z(1, dtype=i32)), '65536 elements'),
    ('norm last stride', lambda: norm(z(4, 64, 2).transpose(1, 2)), 'contiguous in its last'),
    ('norm out type', lambda: norm(q_out=z(4, 2, 64, dtype=bf16)), 'q_out must be torch.float16'),
    ('norm out shape', lambda: norm(k_out=z(4, 2, 64)), 'k_out must have shape'),
    ('norm out overlaps itself', lambda: norm(k_out=z(1, 1, 64).expand(4, 1, 64)), 'k_out must not overlap itself'),
    ('norm in place on an expanded q', lambda: (lambda q: norm(q, q_out=q))(z(1, 2, 64).expand(4, 2, 64)), 'must not overlap itself'),
    ('norm positions', lambda: norm(pos=z(5, dtype=i32)), 'positions must have shape'),
    ('norm axes', lambda: norm(axes=A), 'positions must be int32 \\[axes, T\\]'),
    ('norm inv_freq', lambda: norm(f=F.float()), 'inv_freq must be torch.float64'),
    ('norm cpu tensors', norm, 'must be a CUDA tensor'),
    ('maps new_lens type', lambda: maps(z(3, dtype=torch.int64)), 'new_lens must be torch.int32'),
    ('maps new_lens rank', lambda: maps(z(3, 1, dtype=i32)), 'new_lens must be int32'),
    ('maps kv_lens', lambda: maps(kv=z(4, dtype=i32)), 'kv_lens must have shape'),
    ('maps table rows', lambda: maps(table=z(4, 5, dtype=i32)), 'block_table must have shape'),
    ('maps table rank', lambda: maps(table=z(15, dtype=i32)), 'block_table must be'),
    ('maps table strided', lambda: maps(table=z(3, 10, dtype=i32)[:, ::2]), 'block_table must be contiguous'),
    ('maps table width', lambda: maps(table=torch.empty(3, (1 << 26) + 1, dtype=i32, device='meta')), 'at most 2\\^30 places'),
    ('maps page', lambda: maps(page=24), 'power of two'),
    ('maps page too large', lambda: maps(page=2048), 'power of two'),
    ('maps page fraction', lambda: maps(page=16.0), 'power of two'),
    ('maps tokens', lambda: maps(tokens=-1), 'tokens must be'),
    ('maps tokens fraction', lambda: maps(tokens=8.0), 'tokens must be'),
    ('maps tokens past 30 bits', lambda: maps(tokens=1 << 30), 'under 2\\^30'),
    ('maps requests', lambda: maps(torch.empty(1 << 20, dtype=i32, device='meta')), 'under 2\\^20'),
    ('maps free without taken', lambda: maps(free_pages=FREE['free_pages']), 'belong together'),
    ('maps taken without free', lambda: maps(taken=FREE['taken']), 'belong together'),
    ('maps taken_out alone', lambda: maps(taken_out=FREE['taken']), 'belong together'),
    ('maps taken shape', lambda: maps(free_pages=FREE['free_pages'], taken=z(2, dtype=i32)), 'taken must have shape'),
    ('maps free rank', lambda: maps(free_pages=z(3, 3, dtype=i32), taken=FREE['taken']), 'free_pages must have shape'),
    ('maps taken_out', lambda: maps(taken_out=z(1, dtype=torch.int64), **FREE), 'taken_out must be torch.int32'),
    ('maps kv_out', lambda: maps(kv_out=z(2, dtype=i32)), 'kv_out must have shape'),
    ('maps cpu tensors', lambda: maps(**FREE), 'must be a CUDA tensor'),
    ('varlen window of none', lambda: varlen(window=0), 'window must be'),
    ('varlen window negative', lambda: varlen(window=-1), 'window must be'),
    ('varlen window fraction', lambda: varlen(window=2.0), 'window must be'),
    ('varlen window true', lambda: varlen(window=True), 'window must be'),
    ('varlen window, not causal', lambda: varlen(window=4, causal=False), 'belongs to causal'),
    ('varlen sinks negative', lambda: varlen(window=4, sinks=-1), 'sinks must be'),
    ('varlen sinks fraction', lambda: varlen(window=4, sinks=1.0), 'sinks must be'),
    ('varlen sinks without a window', lambda: varlen(sinks=3), 'sinks belong to a window'),
    ('varlen window cpu tensors', lambda: varlen(window=4), 'must be a CUDA tensor'),
    ('paged window, not causal', lambda: paged(window=4, causal=False), 'belongs to causal'),
    ('paged sinks without a window', lambda: paged(sinks=3), 'sinks belong to a window'),
    ('paged window and shared', lambda: paged(window=4, shared=groups()), 'exclude each other'),
    ('paged shared alone', lambda: paged(shared=z(2, dtype=i32)), 'shared must be'),
    ('paged shared of no group', lambda: paged(shared=groups(0)), 'shared must be'),
    ('paged shared lens type', lambda: paged(shared=groups(lens=z(1, dtype=torch.int64))), 'shared_lens must be torch.int32'),
    ('paged shared cu type', lambda: paged(shared=groups(cu=z(2, dtype=torch.int64))), 'cu_shared must be torch.int32'),
    ('paged shared cu length', lambda: paged(shared=groups(2, cu=z(2, dtype=i32))), 'cu_shared must have shape'),
    ('paged shared strided', lambda: paged(shared=groups(2, lens=z(4, dtype=i32)[::2])), 'shared_lens must be contiguous'),
    ('paged shared groups', lambda: paged(shared=groups(lens=torch.empty(1 << 20, dtype=i32, device='meta'))), 'shared must be'),
    ('paged shared on the CPU', lambda: paged(shared=groups()), 'must be a CUDA tensor'),
    ('workspace window', lambda: K.attention_workspace(1, 1, 64, 8, 8, 64, window=0), 'window must be'),
    ('workspace sinks', lambda: K.attention_workspace(1, 1, 64, 8, 8, 64, sinks=2), 'sinks belong to a window'),
    ('workspace groups', lambda: K.attention_workspace(1, 1, 64, 8, 8, 64, groups=-1), 'groups must be'),
    ('workspace window and groups', lambda: K.attention_workspace(1, 1, 64, 8, 8, 64, window=4, groups=1), 'groups must be'),
]


@pytest.mark.parametrize('name,fn,msg', REFUSED, ids=[r[0] for r in REFUSED])
def test_refused_with_value_error(name, fn, msg):
    with pytest.raises(ValueError, match=msg):
        fn()


X = ctypes.c_void_p(1 << 20)      # an aligned address that nothing reads


def native_norm(T=4, H=2, kv=1, hd=64, rot=64, dtype=1, wt=1, eps=1e-6, q=X, qo=X, axes=None, n=1, qst=128, ost=128):
    return ('ck_norm_rope', q, X, qo, X, X, X, X, n, axes, X, T, H, kv, hd, rot, qst, 64, 64, 64, ost, 64, 64, 64, dtype, wt, eps, 0, 1.0, None)


def native_maps(B=3, width=5, n_free=9, page=16, tokens=8, free=X, taken=X, out=X, ws=None, cu=X, table=X):
    return ('ck_cache_maps', X, X, table, width, free, n_free, taken, B, page, tokens, cu, X, X, X, out, ws, 0, None)


def native_window(window=8, sinks=0, scale=0.1, paged=True):
    return ('ck_attention_paged_window', X, X, X, None, None, X, X, 3, X, X, 2, 4, 4, 3, 2, 16, 64, 256, 64, 256, 64, 1, 1, window, sinks, scale,
            None, 0, None) if paged else ('ck_attention_varlen_window', X, X, X, X, X, X, 2, 4, 4, 4, 2, 64, 256, 64, 128, 64, 128, 64, 256, 64, 1,
                                          window, sinks, scale, None, 0, None)


def native_shared(n=1, cu=X, lens=X, hd=64):
    return ('ck_attention_paged_shared', X, X, X, None, None, X, X, 3, X, X, cu, lens, n, 2, 4, 4, 3, 2, 16, hd, 256, hd, 256, hd, 1, 1, 1, 0.1,
            None, 0, None)


NATIVE = [
    ('paged window', native_window(0), 'must have a key'),
    ('varlen window', native_window(-4, paged=False), 'must have a key'),
    ('paged sinks', native_window(8, -1), 'must not be negative'),
    ('varlen scale', native_window(scale=-1.0, paged=False), 'positive and finite'),
    ('shared groups', native_shared(0), 'need a group'),
    ('shared too many groups', native_shared(1 << 20), 'under 2\\^20'),
    ('shared null', native_shared(cu=None), 'null pointer'),
    ('shared head_dim', native_shared(hd=96), 'head_dim must be 64 or 128'),
    ('shared workspace', native_shared(), 'workspace too small'),
    ('range workspace', ('ck_attention_range_workspace', 1, 1, 64, 8, 8, 64, 0, 0, 1, None), 'null argument'),
    ('range workspace sizes', ('ck_attention_range_workspace', 1, 1, 64, 8, 8, 64, -1, 0, 0, ctypes.byref(ctypes.c_size_t())), 'bad sizes'),
    ('rope axes', ('ck_rope_axes', X, X, X, 3, None, X, 4, 2, 64, 64, 128, 64, 128, 64, 1, 0, 1.0, 0, None), "every pair's axis"),
    ('rope no axis', ('ck_rope_axes', X, X, X, 0, X, X, 4, 2, 64, 64, 128, 64, 128, 64, 1, 0, 1.0, 0, None), "every pair's axis"),
    ('norm rot', native_norm(rot=7), 'must be even'),
    ('norm type', native_norm(dtype=5), 'f16 or bf16'),
    ('norm weights', native_norm(wt=5), 'weights must be'),
    ('norm eps', native_norm(eps=0.0), 'eps must be'),
    ('norm heads', native_norm(H=0, kv=0), 'sizes must be'),
    ('norm null', native_norm(q=None), 'null pointer'),
    ('norm in place', native_norm(ost=256), 'in place'),
    ('norm axes', native_norm(n=2), "every pair's axis"),
    ('norm tokens', native_norm(T=1 << 30, rot=2), 'too many tokens'),
    ('maps page', native_maps(page=48), 'power of two'),
    ('maps requests', native_maps(B=1 << 20), 'bad sizes'),
    ('maps rows', native_maps(tokens=1 << 30), 'bad sizes'),
    ('maps width', native_maps(width=(1 << 26) + 1), 'at most 2\\^30 places'),
    ('maps null', native_maps(cu=None), 'null pointer'),
    ('maps null table', native_maps(table=None), 'null pointer'),
    ('maps free without taken', native_maps(taken=None, out=None), 'free pages need'),
    ('maps taken without out', native_maps(out=None), 'free pages need'),
    ('maps workspace', native_maps(tokens=5000), 'workspace too small'),     # taken_out is taken, kv_out is kv
    ('maps workspace null', ('ck_cache_maps_workspace', 1, 1, 0, None), 'null argument'),
    ('maps workspace sizes', ('ck_cache_maps_workspace', -1, 1, 0, ctypes.byref(ctypes.c_size_t())), 'bad sizes'),
]


@pytest.mark.parametrize('name,args,msg', NATIVE, ids=[r[0] for r in NATIVE])
def test_native_checks(name, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(*args)


def test_cache_maps_workspace():
    assert K.cache_maps_workspace(32, 32, True) == K.cache_maps_workspace(700, 10 ** 6, False) == K.cache_maps_workspace(0, 5000, True) == 0
    assert K.cache_maps_workspace(700, 5000, True) >= 700 * 4 and K.cache_maps_workspace(9000, 50000, False) >= 9000 * 4
    with pytest.raises(ValueError, match='under 2\\^31'):
        K.cache_maps_workspace(2 ** 32 + 4, 4, False)


def test_axes():
    assert K.rope_axes([2, 3, 1], device='cpu').tolist() == [0, 0, 1, 1, 1, 2]
    assert K.rope_axes([2, 3, 1], True, device='cpu').tolist() == [0, 1, 2, 0, 1, 1]
    assert K.rope_axes([0, 2], device='cpu').tolist() == [1, 1] and K.rope_axes([4], device='cpu').dtype is i32


def test_oracle_rope_by_axes():
    x = np.random.default_rng(2).standard_normal((4, 2, 12))
    f, pos = np.array([1.0, 0.1, 0.01]), np.array([[0, 1, 5, 1000], [3, 2, 1, 0]])
    for inter in (False, True):
        y = O.rope(x, pos, f, inter, 2.0, axes=[0, 1, 0])
        a, b = O.rope(x, pos[0], f, inter, 2.0), O.rope(x, pos[1], f, inter, 2.0)
        mid = [2, 3] if inter else [1, 4]
        rest = [i for i in range(12) if i not in mid]
        assert np.array_equal(y[..., mid], b[..., mid]) and np.array_equal(y[..., rest], a[..., rest])


def test_oracle_norm():
    x = torch.randn(5, 3, 40, dtype=torch.float64)
    w = torch.randn(40, dtype=torch.float64)
    assert np.allclose(O.rms_norm(x.numpy(), w.numpy(), 1e-3), torch.nn.functional.rms_norm(x, (40,), w, 1e-3).numpy(), rtol=1e-13)


def test_oracle_maps():
    """Slots are places: writing each row's request and place to its slot leaves, read back by the table, each request's
    places in order; a page belongs to one request."""
    r = np.random.default_rng(3)
    B, page = 9, 16
    new, kv = r.integers(0, 60, B), r.integers(0, 50, B)
    width = 8
    free = list(r.permutation(200)[:120])
    table = np.full((B, width), -1)
    have = [-(-int(m) // page) for m in kv]
    at = 100
    for b in range(B):
        table[b, :have[b]] = np.arange(200 + at, 200 + at + have[b])
        at += have[b]
    cu, out, pos, slots, got, taken = O.cache_maps(new, kv, table, page, int(new.sum()) + 3, free, 4)
    assert pos[-3:] == [0, 0, 0] and slots[-3:] == [-1, -1, -1] and cu[-1] == new.sum() and list(out) == list(new + kv)
    cache = {}
    for b in range(B):
        for i in range(cu[b], cu[b + 1]):
            assert slots[i] not in cache and pos[i] == kv[b] + i - cu[b]
            cache[slots[i]] = (b, pos[i])
    for b in range(B):
        for j in range(kv[b], out[b]):
            assert cache[got[b][j // page] * page + j % page] == (b, j)
    used = [x for row in got for x in row if x >= 0]
    assert len(set(used)) == len(used) and taken == 4 + sum(-(-int(m) // page) for m in out) - sum(have)
    assert sorted(used) == sorted([int(x) for x in free[4:taken]] + [int(x) for x in table[table >= 0]])


@pytest.mark.parametrize('n,m,window,sinks', [(5, 5, 2, 0), (3, 9, 4, 2), (6, 2, 1, 1), (4, 7, 100, 0), (2, 0, 3, 3), (4, 12, 3, 20)])
def test_oracle_window(n, m, window, sinks):
    r = np.random.default_rng(n + m)
    q, k, v = r.standard_normal((n, 4, 8)), r.standard_normal((m, 2, 8)), r.standard_normal((m, 2, 8))
    out, _, _ = O.attention(q, k, v, window=window, sinks=sinks)
    for i in range(n):
        place = i + m - n
        js = [j for j in range(m) if j <= place and (place - j < window or j < sinks)]
        for h in range(4):
            w = np.array([math.exp(q[i, h] @ k[j, h // 2] / math.sqrt(8)) for j in js])
            want = sum((x * v[j, h // 2] for x, j in zip(w / w.sum(), js)), np.zeros(8)) if js else np.zeros(8)
            assert np.allclose(out[i, h], want, atol=1e-12)


def test_range_workspace():
    whole = K.attention_workspace(1, 1, 6144, 8, 8, 64)
    assert K.attention_workspace(1, 1, 6144, 8, 8, 64, window=6144) == whole > 0
    assert K.attention_workspace(1, 1, 6144, 8, 8, 64, window=1 << 40, sinks=1 << 40) == whole
    assert K.attention_workspace(1, 1, 6144, 8, 8, 64, window=64) == 0          # few keys: not split
    assert K.attention_workspace(40, 4000, 4000, 8, 8, 64, groups=3) > 0         # what is shared is always joined
    assert K.attention_workspace(0, 0, 0, 8, 8, 64, groups=3) == 0
    t = torch.tensor(1)
    assert K.attention_workspace(t, 1, 6144, 8, 8, 64, window=6144) == whole


@pytest.mark.parametrize('listed', [False, True])
def test_oracle_maps_of_any_lengths(listed):
    """Row by row as token by token, where both can be had; at lengths past 31 bits by what they must be."""
    r = np.random.default_rng(6)
    for page, width in ((16, 7), (16, 3), (32, 40)):
        new, kv = r.integers(-3, 90, 20), r.integers(-9, 150, 20)
        table = r.permutation(20 * width).reshape(20, width)
        table[r.random(table.shape) < 0.1] = -1
        free = list(r.permutation(100) + 20 * width) if listed else None
        for tokens in (0, 9, 300, 1400):
            a, b = (f(new, kv, table, page, tokens, free, 3 * listed) for f in (O.cache_maps, O.cache_maps_of_any_lengths))
            assert all(np.array_equal(x, y) for x, y in zip(a, b))
    most = 2 ** 31 - 1
    cu, out, pos, slots, table, taken = O.cache_maps_of_any_lengths([2, most, 5], [most - 1, 100, 7], [[3] * 8] * 3, 16, 40, [9] * 50, 0)
    assert list(cu) == [0, 2, most, most] and list(out) == [most, most, 12] and taken == 2 ** 27   # ceil((2^31 + 99) / 16) - 7
    assert list(pos[:4]) == [most - 1, most, 100, 101] and list(slots[:4]) == [-1, -1, 3 * 16 + 4, 3 * 16 + 5]
    assert (table[1][:7] == 3).all() and table[1][7] == 9 and pos[14] == 112 and slots[14] == 9 * 16


def test_a_workspace_that_is_missing_is_named_by_its_function():
    """The one that knows of windows and groups: ck_attention_workspace may answer 0 for these calls."""
    few = ('ck_attention_paged_window', X, X, X, None, None, X, X, 400, X, X, 2, 4, 4, 3, 2, 16, 64, 256, 64, 256, 64, 1, 1, 4000, 0, 0.1, None, 0, None)
    rows = ('ck_attention_varlen_window', X, X, X, X, X, X, 2, 4, 9000, 4, 2, 64, 256, 64, 128, 64, 128, 64, 256, 64, 1, 4000, 0, 0.1, None, 0, None)
    for args in (native_shared(), few, rows):
        with pytest.raises(RuntimeError, match='workspace too small \\(ck_attention_range_workspace\\)'):
            _lib.call(*args)
    whole = ('ck_attention_paged', X, X, X, None, None, X, X, 400, X, X, 2, 4, 4, 3, 2, 16, 64, 256, 64, 256, 64, 1, 1, 1, 0.1, None, 0, None)
    with pytest.raises(RuntimeError, match='workspace too small \\(ck_attention_workspace\\)'):
        _lib.call(*whole)

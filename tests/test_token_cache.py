"""The token cache's operators without a GPU: what the entry points refuse, the frequencies
of rope, and the 64-bit oracle against torch and against itself."""
import ctypes
import math

import numpy as np
import pytest
import torch

from chestnut import _lib
from chestnut import kernels as K
from oracle import token_cache as O

f16, bf16, f32, i32 = torch.float16, torch.bfloat16, torch.float32, torch.int32
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def z(*shape, dtype=f16):
    return torch.zeros(*shape, dtype=torch.uint8).view(dtype) if dtype in (E4M3, E8M0) else torch.zeros(*shape, dtype=dtype)


def cache(n=3, kv=2, page=16, hd=64, dtype=f16):
    return z(n, kv, page, hd, dtype=dtype), z(n, kv, page, hd, dtype=dtype)


def paged(q=None, kp=None, vp=None, table=None, cu=None, lens=None, **kw):
    a, b = cache()
    return K.attention_paged(z(4, 4, 64) if q is None else q, a if kp is None else kp, b if vp is None else vp,
                             z(2, 3, dtype=i32) if table is None else table, z(3, dtype=i32) if cu is None else cu,
                             z(2, dtype=i32) if lens is None else lens, **kw)


def varlen(q=None, k=None, v=None, cu=None, **kw):
    return K.attention_varlen(z(4, 4, 64) if q is None else q, z(4, 2, 64) if k is None else k,
                              z(4, 2, 64) if v is None else v, z(3, dtype=i32) if cu is None else cu, **kw)


F = torch.ones(16, dtype=torch.float64)
S = dict(k_scale=z(3, 2, 16, dtype=E8M0), v_scale=z(3, 2, 16, dtype=E8M0))
REFUSED = [
    ('rope x type', lambda: K.rope(z(4, 2, 64, dtype=f32), z(4, dtype=i32), F), 'x must be float16 or bfloat16'),
    ('rope x rank', lambda: K.rope(z(4, 64), z(4, dtype=i32), F), 'x must be'),
    ('rope positions type', lambda: K.rope(z(4, 2, 64), z(4, dtype=torch.int64), F), 'positions must be torch.int32'),
    ('rope positions length', lambda: K.rope(z(4, 2, 64), z(5, dtype=i32), F), 'positions must have shape'),
    ('rope inv_freq type', lambda: K.rope(z(4, 2, 64), z(4, dtype=i32), F.float()), 'inv_freq must be torch.float64'),
    ('rope inv_freq too long', lambda: K.rope(z(4, 2, 24), z(4, dtype=i32), F), 'inv_freq must have 1 to'),
    ('rope inv_freq empty', lambda: K.rope(z(4, 2, 24), z(4, dtype=i32), F[:0]), 'inv_freq must have 1 to'),
    ('rope last stride', lambda: K.rope(z(4, 64, 2).transpose(1, 2), z(4, dtype=i32), F), 'contiguous in its last'),
    ('rope out type', lambda: K.rope(z(4, 2, 64), z(4, dtype=i32), F, out=z(4, 2, 64, dtype=bf16)), 'out must be torch.float16'),
    ('rope out overlaps itself', lambda: K.rope(z(4, 2, 64), z(4, dtype=i32), F, out=z(1, 2, 64).expand(4, 2, 64)),
     'must not overlap itself'),
    ('rope in place on an expanded x', lambda: (lambda x: K.rope(x, z(4, dtype=i32), F, out=x))(z(1, 2, 64).expand(4, 2, 64)),
     'must not overlap itself'),
    ('rope head_dim', lambda: K.rope(z(1, 1, 514), z(1, dtype=i32), F), 'head_dim up to 512'),
    ('write cache rank', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), z(3, 16, 64), z(3, 16, 64), z(4, dtype=i32)), 'k_pages must be'),
    ('write page size', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(page=24), z(4, dtype=i32)), 'power of two'),
    ('write page too small', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(page=8), z(4, dtype=i32)), 'power of two'),
    ('write rows type', lambda: K.cache_write(z(4, 2, 64, dtype=bf16), z(4, 2, 64, dtype=bf16), *cache(), z(4, dtype=i32)),
     'cache must be torch.bfloat16 or'),
    ('write v type', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64, dtype=bf16), *cache(), z(4, dtype=i32)), 'v must be torch.float16'),
    ('write heads', lambda: K.cache_write(z(4, 3, 64), z(4, 3, 64), *cache(), z(4, dtype=i32)), 'k must have shape'),
    ('write slots', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(), z(3, dtype=i32)), 'slots must have shape'),
    ('write row alignment', lambda: K.cache_write(z(4, 2, 68)[:, :, 2:66], z(4, 2, 64), *cache(), z(4, dtype=i32)), 'multiples of 16 bytes'),
    ('write e4m3 without scales', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(dtype=E4M3), z(4, dtype=i32)), 'needs k_scale'),
    ('write scales of f16', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(), z(4, dtype=i32), **S), 'belong to an e4m3'),
    ('write scale shape', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(dtype=E4M3), z(4, dtype=i32),
                                                k_scale=z(3, 2, 8, dtype=E8M0), v_scale=S['v_scale']), 'k_scale must have shape'),
    ('write scale type', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(dtype=E4M3), z(4, dtype=i32),
                                               k_scale=z(3, 2, 16, dtype=torch.uint8), v_scale=S['v_scale']), 'k_scale must be'),
    ('read dtype', lambda: K.cache_read(*cache(), z(2, 3, dtype=i32), z(3, dtype=i32), 4, dtype=bf16), 'dtype must be'),
    ('read e4m3 without a dtype', lambda: K.cache_read(*cache(dtype=E4M3), z(2, 3, dtype=i32), z(3, dtype=i32), 4, **S), 'dtype must be'),
    ('read cu', lambda: K.cache_read(*cache(), z(2, 3, dtype=i32), z(2, dtype=i32), 4), 'cu_seqlens must have shape'),
    ('read tokens', lambda: K.cache_read(*cache(), z(2, 3, dtype=i32), z(3, dtype=i32), -1), 'tokens must be'),
    ('read out', lambda: K.cache_read(*cache(), z(2, 3, dtype=i32), z(3, dtype=i32), 4, k_out=z(5, 2, 64)), 'k_out must have shape'),
    ('varlen head_dim', lambda: varlen(z(4, 4, 96), z(4, 2, 96), z(4, 2, 96)), 'head_dim must be 64 or 128'),
    ('varlen heads', lambda: varlen(z(4, 3, 64)), 'multiple of the K/V heads'),
    ('varlen types', lambda: varlen(k=z(4, 2, 64, dtype=bf16)), 'k must be torch.float16'),
    ('varlen f32', lambda: varlen(z(4, 4, 64, dtype=f32)), 'q must be float16 or bfloat16'),
    ('varlen k rows', lambda: varlen(k=z(5, 2, 64), v=z(5, 2, 64)), 'k must have the 4 rows'),
    ('varlen v rows', lambda: varlen(v=z(5, 2, 64)), 'v must have shape'),
    ('varlen cu_k', lambda: varlen(cu_k=z(4, dtype=i32)), 'cu_k must have shape'),
    ('varlen cu type', lambda: varlen(cu=z(3, dtype=torch.int64)), 'cu_q must be torch.int32'),
    ('varlen cu empty', lambda: varlen(cu=z(0, dtype=i32)), 'B \\+ 1 offsets'),
    ('varlen scale', lambda: varlen(scale=0.0), 'scale must be positive'),
    ('varlen nan scale', lambda: varlen(scale=math.nan), 'scale must be positive'),
    ('varlen out', lambda: varlen(out=z(4, 4, 65)[:, :, :64]), 'multiples of 8 bytes'),
    ('varlen q alignment', lambda: varlen(z(4, 4, 72)[:, :, 1:65]), 'multiples of 16 bytes'),
    ('varlen out overlaps itself', lambda: varlen(out=z(1, 4, 64).expand(4, 4, 64)), 'must not overlap itself'),
    ('rope out token 1 is head 1 of token 0', lambda: K.rope(z(4, 2, 64), z(4, dtype=i32), F, out=z(320).as_strided((4, 2, 64), (64, 64, 1))),
     'must not overlap itself'),
    ('varlen out heads in each other', lambda: varlen(out=z(1024).as_strided((4, 4, 64), (128, 64, 1))), 'must not overlap itself'),
    ('varlen out head by head', lambda: varlen(out=z(4, 4, 64).transpose(0, 1)), 'must be a CUDA tensor'),
    ('varlen out in wider rows', lambda: varlen(out=z(4, 6, 72)[:, 1:5, :64]), 'must be a CUDA tensor'),
    ('paged cache type', lambda: paged(z(4, 4, 64, dtype=bf16)), 'cache must be torch.bfloat16 or'),
    ('paged head_dim', lambda: paged(z(4, 4, 128)), 'head_dim must be 64 or 128 for q and the keys alike'),
    ('paged table rows', lambda: paged(table=z(3, 3, dtype=i32)), 'block_table must have shape'),
    ('paged table type', lambda: paged(table=z(2, 3, dtype=torch.int64)), 'block_table must be torch.int32'),
    ('paged lens', lambda: paged(lens=z(3, dtype=i32)), 'kv_lens must have shape'),
    ('paged table strided', lambda: paged(table=z(2, 6, dtype=i32)[:, ::2]), 'block_table must be contiguous'),
    ('varlen token stride', lambda: varlen(k=torch.empty_strided((4, 2, 64), (1 << 24, 64, 1), dtype=f16, device='meta')),
     'under 2\\^24 elements'),
    ('paged table width', lambda: paged(table=torch.empty(2, (1 << 26) + 1, dtype=i32, device='meta')), 'at most 2\\^30 places'),
    ('paged table rank', lambda: paged(table=z(6, dtype=i32)), 'block_table must be int32'),
    ('paged cpu tensors', paged, 'must be a CUDA tensor'),
    ('varlen cpu tensors', varlen, 'must be a CUDA tensor'),
    ('rope cpu tensors', lambda: K.rope(z(4, 2, 64), z(4, dtype=i32), F), 'must be a CUDA tensor'),
    ('write cpu tensors', lambda: K.cache_write(z(4, 2, 64), z(4, 2, 64), *cache(), z(4, dtype=i32)), 'must be a CUDA tensor'),
    ('read cpu tensors', lambda: K.cache_read(*cache(), z(2, 3, dtype=i32), z(3, dtype=i32), 4), 'must be a CUDA tensor'),
]


@pytest.mark.parametrize('name,fn,msg', REFUSED, ids=[r[0] for r in REFUSED])
def test_refused_with_value_error(name, fn, msg):
    with pytest.raises(ValueError, match=msg):
        fn()


# The native entry points check again what reaches them as plain numbers (no call below launches).
X = ctypes.c_void_p(1 << 20)      # an aligned address that nothing reads


def attn(T=4, H=4, n=3, kv=2, page=16, hd=64, dtype=1, cdtype=1, scale=0.1, q=X, ks=None, width=3, st=256, B=2):
    return ('ck_attention_paged', q, X, X, ks, ks, X, X, width, X, X, B, T, H, n, kv, page, hd, st, hd, st, hd, dtype, cdtype, 1,
            scale, None, 0, None)


NATIVE = [
    ('rope rot', ('ck_rope', X, X, X, X, 4, 2, 64, 7, 128, 64, 128, 64, 1, 0, 1.0, 0, None), 'must be even'),
    ('rope dtype', ('ck_rope', X, X, X, X, 4, 2, 64, 64, 128, 64, 128, 64, 0, 0, 1.0, 0, None), 'f16 or bf16'),
    ('rope null', ('ck_rope', None, X, X, X, 4, 2, 64, 64, 128, 64, 128, 64, 1, 0, 1.0, 0, None), 'null pointer'),
    ('rope in place', ('ck_rope', X, X, X, X, 4, 2, 64, 64, 128, 64, 256, 64, 1, 0, 1.0, 0, None), 'in place'),
    ('write page', ('ck_cache_write', X, X, X, X, None, None, X, 4, 3, 2, 24, 64, 128, 64, 128, 64, 1, 1, None), 'power of two'),
    ('write type', ('ck_cache_write', X, X, X, X, None, None, X, 4, 3, 2, 16, 64, 128, 64, 128, 64, 1, 4, None), "rows' type or e4m3"),
    ('write scales', ('ck_cache_write', X, X, X, X, None, None, X, 4, 3, 2, 16, 64, 128, 64, 128, 64, 1, 5, None), 'needs its scales'),
    ('write stride', ('ck_cache_write', X, X, X, X, None, None, X, 4, 3, 2, 16, 64, 130, 64, 128, 64, 1, 1, None), '16-byte aligned'),
    ('write slots', ('ck_cache_write', X, X, X, X, None, None, X, 4, 1 << 28, 2, 16, 64, 128, 64, 128, 64, 1, 1, None), '2\\^31 slots'),
    ('read null', ('ck_cache_read', X, X, None, None, None, 3, X, 2, 4, 3, 2, 16, 64, X, X, 1, 1, None), 'null pointer'),
    ('paged heads', attn(H=3), 'multiple of the K/V heads'),
    ('paged head_dim', attn(hd=96), 'head_dim must be 64 or 128'),
    ('paged dtype', attn(dtype=0), 'q must be f16 or bf16|of q'),
    ('paged cache dtype', attn(cdtype=4), "q's type or e4m3"),
    ('paged scales', attn(cdtype=5), 'needs its scales'),
    ('paged scale', attn(scale=-1.0), 'positive and finite'),
    ('paged null', attn(q=None), 'null pointer'),
    ('paged stride', attn(st=250), 'aligned'),
    # a launch has under 2^32 threads
    ('rope tokens', ('ck_rope', X, X, X, X, 1 << 28, 1, 512, 510, 513, 512, 513, 512, 1, 0, 1.0, 0, None), 'too many tokens'),
    ('write rows', ('ck_cache_write', X, X, X, X, None, None, X, 1 << 26, 3, 2, 16, 64, 0, 64, 0, 64, 1, 1, None), '2\\^27 rows'),
    ('read tokens', ('ck_cache_read', X, X, None, None, X, 3, X, 2, 1 << 28, 3, 1, 16, 8, X, X, 1, 1, None), '2\\^28 tokens'),
    ('paged sequences', attn(T=1 << 19, B=1 << 19, H=32, kv=32), 'too many sequences'),
    ('paged width', attn(width=(1 << 26) + 1), 'at most 2\\^30 places'),
]


@pytest.mark.parametrize('name,args,msg', NATIVE, ids=[r[0] for r in NATIVE])
def test_native_checks(name, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(*args)


def test_frequencies():
    f, s = K.rope_frequencies(8, base=100.0, device='cpu')
    assert s == 1.0 and f.dtype is torch.float64 and np.allclose(f, [100.0 ** (-i / 4) for i in range(4)], rtol=1e-15)
    g, s = K.rope_frequencies(8, base=100.0, method='linear', factor=4.0, device='cpu')
    assert s == 1.0 and torch.equal(g, f / 4)
    g, _ = K.rope_frequencies(8, base=100.0, method='base', factor=4.0, device='cpu')
    assert g[0] == 1.0 and math.isclose(g[-1], f[-1] / 4, rel_tol=1e-14)
    g, s = K.rope_frequencies(128, method='parts', factor=8.0, context=4096, device='cpu')
    f, _ = K.rope_frequencies(128, device='cpu')
    turns = 4096 * f / (2 * math.pi)
    assert torch.equal(g[turns >= 32], f[turns >= 32]) and torch.equal(g[turns <= 1], f[turns <= 1] / 8)
    mid = (turns > 1) & (turns < 32)
    assert mid.any() and (g[mid] < f[mid]).all() and (g[mid] > f[mid] / 8).all() and math.isclose(s, 0.1 * math.log(8) + 1)
    for bad in (dict(rot=7), dict(rot=0), dict(rot=8, method='x'), dict(rot=8, factor=0.5), dict(rot=2, method='base'),
                dict(rot=8, method='parts', factor=2.0), dict(rot=8, base=1.0)):
        with pytest.raises(ValueError):
            K.rope_frequencies(device='cpu', **bad)


def test_oracle_codes_are_the_formats():
    v = O.e4m3_values()
    t = torch.arange(256, dtype=torch.uint8).view(E4M3).double().numpy()
    assert np.array_equal(v[~np.isnan(v)], t[~np.isnan(t)]) and np.array_equal(np.isnan(v), np.isnan(t))
    x = np.concatenate([np.random.default_rng(0).standard_normal(5000) * 100, v[~np.isnan(v)], (v[:126] + v[1:127]) / 2,
                        np.arange(-40, 40) * 2.0 ** -11]).clip(-448, 448).astype(np.float32)
    assert np.array_equal(O.e4m3_codes(x.astype(np.float64)), torch.from_numpy(x).to(E4M3).view(torch.uint8).numpy())


def test_oracle_rows_hold_half_a_step():
    x = np.random.default_rng(1).standard_normal((50, 64)) * np.logspace(-4, 4, 50)[:, None]
    c, b = O.quantise(x, 61440.0)
    y, s = O.values(c, b), 2.0 ** (b.astype(float) - 127)
    assert np.all(np.abs(x) <= 448 * s[:, None]) and np.all(np.abs(x).max(-1) > 224 * s)
    assert np.all(np.abs(y - x) <= np.maximum(2.0 ** -4 * np.abs(x), 2.0 ** -10 * s[:, None]))


@pytest.mark.parametrize('n,m,causal', [(5, 5, True), (3, 9, True), (6, 2, True), (4, 7, False), (2, 0, True)])
def test_oracle_attention_is_the_masked_softmax(n, m, causal):
    r = np.random.default_rng(n + m)
    q, k, v = r.standard_normal((n, 4, 8)), r.standard_normal((m, 2, 8)), r.standard_normal((m, 2, 8))
    out, mag, _ = O.attention(q, k, v, causal)
    for i in range(n):
        for h in range(4):
            js = [j for j in range(m) if not causal or j <= i + m - n]
            w = np.array([math.exp(q[i, h] @ k[j, h // 2] / math.sqrt(8)) for j in js])
            want = sum((x * v[j, h // 2] for x, j in zip(w / w.sum(), js)), np.zeros(8)) if js else np.zeros(8)
            assert np.allclose(out[i, h], want, atol=1e-12) and np.all(mag[i, h] >= np.abs(want) - 1e-12)


def test_oracle_rope_turns_and_turns_back():
    x = np.random.default_rng(2).standard_normal((4, 2, 12))
    f = np.array([1.0, 0.1, 0.01])
    for inter in (False, True):
        y = O.rope(x, [0, 1, 5, 1000], f, inter, 2.0)
        assert np.allclose(y[0, :, :6], 2 * x[0, :, :6]) and np.array_equal(y[..., 6:], x[..., 6:])
        assert np.allclose(O.rope(y, [0, 1, 5, 1000], f, inter, 0.5, True), x)
        i, j = (0, 1) if inter else (0, 3)
        z = (x[2, 1, i] + 1j * x[2, 1, j]) * np.exp(5j) * 2
        assert np.allclose([y[2, 1, i], y[2, 1, j]], [z.real, z.imag])


def test_attention_workspace():
    assert K.attention_workspace(0, 0, 0, 8, 8, 64) == K.attention_workspace(40, 4000, 4000, 8, 8, 64) == 0
    one = K.attention_workspace(1, 1, 6144, 8, 8, 64)
    assert one % 16 == 0 and one >= 8 * 32 * (64 + 2) * 4 * 2     # two parts of a tile of 32 rows a head at least
    for bad in ((1, 1, 64, 8, 3, 64), (-1, 1, 64, 8, 8, 64), (1, 1, -64, 8, 8, 64)):
        with pytest.raises(RuntimeError, match='bad sizes'):
            K.attention_workspace(*bad)


def test_oracle_attention_of_nan_scores_is_nan():
    r = np.random.default_rng(3)
    q, k, v = r.standard_normal((3, 4, 8)), r.standard_normal((5, 2, 8)), r.standard_normal((5, 2, 8))
    want = O.attention(q, k, v)[0]
    q[1, 2, 0], k[4, 0, 3] = np.nan, np.nan              # one query row; one key, which the last query alone sees
    out = O.attention(q, k, v)[0]
    nan = np.zeros((3, 4), bool)
    nan[1, 2], nan[2, :2] = True, True
    assert np.isnan(out[nan]).all() and np.array_equal(out[~nan], want[~nan])


def test_attention_workspace_remembers_plain_integers_only():
    t = torch.tensor(1)
    assert K.attention_workspace(t, 200, 6400, 8, 8, 64) == K.attention_workspace(1, 200, 6400, 8, 8, 64) > 0
    t.fill_(200)
    assert K.attention_workspace(t, 200, 6400, 8, 8, 64) == K.attention_workspace(200, 200, 6400, 8, 8, 64) == 0
    for at in range(6):
        args = [3, 200, 6400, 8, 8, 64]
        K.attention_workspace(*args)
        args[at] = float(args[at])
        with pytest.raises(ctypes.ArgumentError):
            K.attention_workspace(*args)


def test_tiles_of_256_rows_keep_their_keys_whole():
    for B in (1, 2, 7, 40):
        for T in (1000, 4101, 8192, 100000):
            for H, kv in ((32, 8), (16, 16), (64, 1)):
                if T * H // kv > 32 * B and (T * (H // kv) // 256 + B) * kv >= 512:
                    assert K.attention_workspace(B, T, 1 << 24, H, kv, 128) == 0
    assert K.attention_workspace(2, 1000, 1 << 24, 32, 8, 128) > 0


def many(n, *shape, dtype=f16):
    """n rows that take no memory."""
    return torch.empty(1, *shape, dtype=dtype, device='meta').expand(n, *shape)


def ints(*shape):
    return torch.empty(*shape, dtype=i32, device='meta')


N = 2 ** 32 + 4                       # 4 if it is cut to 32 bits
PAST_32_BITS = [
    ('rope tokens', lambda: K.rope(many(N, 2, 64), ints(N), F)),
    ('write tokens', lambda: K.cache_write(many(N, 2, 64), many(N, 2, 64), *cache(), ints(N))),
    ('read tokens', lambda: K.cache_read(*cache(), z(2, 3, dtype=i32), z(3, dtype=i32), N)),
    ('read table width', lambda: K.cache_read(*cache(), ints(2, N), z(3, dtype=i32), 4)),
    ('read sequences', lambda: K.cache_read(*cache(), ints(N, 3), ints(N + 1), 4)),
    ('varlen queries', lambda: varlen(many(N, 4, 64), many(N, 2, 64), many(N, 2, 64))),
    ('varlen keys', lambda: varlen(k=many(N, 2, 64), v=many(N, 2, 64), cu_k=z(3, dtype=i32))),
    ('varlen sequences', lambda: varlen(cu=ints(N + 1))),
    ('paged sequences', lambda: paged(table=ints(N, 3), cu=ints(N + 1), lens=ints(N))),
    ('workspace', lambda: K.attention_workspace(N, N, 64, 8, 8, 64)),
    ('workspace keys', lambda: K.attention_workspace(1, 1, 2 ** 64 + 1, 8, 8, 64)),
]


@pytest.mark.parametrize('name,fn', PAST_32_BITS, ids=[r[0] for r in PAST_32_BITS])
def test_counts_past_32_bits_are_refused(name, fn):
    with pytest.raises(ValueError, match='under 2\\^31'):
        fn()


@pytest.mark.parametrize('scale', [1e-50, 2.5e38, 1e39, math.inf])
def test_scales_that_f32_does_not_hold_are_refused(scale):
    with pytest.raises(ValueError, match='scale must be positive and finite'):
        varlen(scale=scale)
    with pytest.raises(RuntimeError, match='positive and finite'):
        _lib.call(*attn(scale=scale))

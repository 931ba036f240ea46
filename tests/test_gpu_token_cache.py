"""Rotary positions, the paged cache and attention over packed sequences and pages on the
GPU, against oracle.token_cache in 64 bits.

Tolerances.  u = eps / 2 of the element type is the relative error of one rounding.
rope: angles are exact to 2^-45 turns, cos and sin to 2^-22 each; two products and a sum
in f32, one rounding to the type.
cache: bit-exact codes and scales; a value read back is one rounding of code * scale.
attention: the output is rounded once (u |o|) and each softmax weight once (u a weight, so
u times A = the same sum with |v|); f16 weights are kept 2^7 times as large, and those below the
smallest normal round to its subnormals (2^-32 of the strongest each, n of them at most, each
times |v| < 6, against a row sum of at least 1); a score is a chain of hd f32 sums ((hd + 4) 2^-24 of its sum
of magnitudes, twice: numerator and denominator); exp2, the rescalings and the sums add
less than 2^-17."""
import numpy as np
import pytest
import torch

from oracle import token_cache as O

pytestmark = pytest.mark.gpu
DT = {'f16': torch.float16, 'bf16': torch.bfloat16}
TOP = {'f16': 61440.0, 'bf16': 1.875 * 2.0 ** 127}


def u(dt):
    return torch.finfo(DT[dt]).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def rows(seed, T, H, hd, dt, scale=1.0):
    """Values of the type, exact in f64, on the device."""
    x = np.random.default_rng(seed).standard_normal((T, H, hd)) * scale
    return torch.from_numpy(x).to(DT[dt]).cuda()


def i32(v):
    return torch.tensor(np.asarray(v, np.int32).reshape(-1) if np.ndim(v) < 2 else np.asarray(v, np.int32)).cuda()


def cu(lens):
    return i32(np.concatenate([[0], np.cumsum(lens)]))


def near(out, ref, mag, most, n, hd, dt, what=''):
    out = f64(out)
    tiny = 6 * n * 2.0 ** -32 if dt == 'f16' else 0.0
    tol = u(dt) * (np.abs(ref) + mag) * (1 + 2.0 ** -6) + (2 * (hd + 4) * 2.0 ** -24 * most + 2.0 ** -17) * mag + tiny
    bad = ~(np.abs(out - ref) <= tol)
    assert not bad.any(), f'{what}: {bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(out - ref) - tol)}, first {np.argwhere(bad)[0]}'


# ---------------------------------------------------------------------- rope --
@pytest.mark.parametrize('T,H,hd,rot', [(1, 1, 64, 64), (3, 5, 128, 64), (17, 20, 128, 128), (700, 3, 64, 16),
                                        (9, 2, 80, 24), (5, 3, 33, 10), (2, 1, 2, 2), (33, 4, 256, 256)])
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_rope(gpu, T, H, hd, rot, inter, dt):
    from chestnut import kernels as K
    x = rows(T + hd, T, H, hd, dt)
    pos = np.random.default_rng(1).integers(0, 1 << 20, T)
    pos[0] = 0 if T > 1 else 999999
    f, s = K.rope_frequencies(rot, base=5e5, method='parts', factor=8.0, context=8192)
    ref = O.rope(f64(x), pos, f64(f), inter, s)
    mag = np.abs(f64(x)).max() * 2 * s
    out = K.rope(x, i32(pos), f, interleaved=inter, scale=s)
    assert np.all(np.abs(f64(out) - ref) <= u(dt) * np.abs(ref) * (1 + 2.0 ** -6) + 2.0 ** -20 * mag + 2.0 ** -25)
    assert torch.equal(out[..., rot:], x[..., rot:])
    back = K.rope(out, i32(pos), f, interleaved=inter, scale=1 / s, inverse=True)
    assert np.all(np.abs(f64(back) - f64(x)) <= 4 * u(dt) * mag)
    y = x.clone()
    assert K.rope(y, i32(pos), f, interleaved=inter, scale=s, out=y) is y and torch.equal(y, out)


@pytest.mark.parametrize('off', [0, 1, 8])
def test_rope_strided_views(gpu, off):
    from chestnut import kernels as K
    T, H, hd = 6, 3, 64
    qkv = rows(2, T, 9, hd + 16, 'f16')
    x = qkv[:, 2:2 + H, off:off + hd]
    buf = torch.full((T, 5, 100), 7.0, dtype=torch.float16, device='cuda')
    f, _ = K.rope_frequencies(32)
    want = K.rope(x.contiguous(), i32(np.arange(T)), f)
    got = K.rope(x, i32(np.arange(T)), f, out=buf[:, 1:1 + H, 8:8 + hd])
    assert torch.equal(got, want) and torch.equal(buf[:, 1:1 + H, 8:8 + hd], want)
    buf[:, 1:1 + H, 8:8 + hd] = 7.0
    assert (buf == 7.0).all()


# --------------------------------------------------------------------- cache --
def pages_of(n, kv, page, hd, dt, cache):
    if cache != 'e4m3':
        return [torch.full((n, kv, page, hd), 3.0, dtype=DT[dt], device='cuda') for _ in 'kv'] + [None, None]
    return ([torch.full((n, kv, page, hd), 0x5A, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn) for _ in 'kv'] +
            [torch.full((n, kv, page), 99, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu) for _ in 'kv'])


@pytest.mark.parametrize('T,kv,hd,page', [(1, 1, 128, 16), (7, 3, 64, 32), (100, 8, 128, 64), (33, 2, 40, 16), (20, 1, 256, 1024),
                                          (5, 5, 8, 16)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
def test_cache_write_and_read_back(gpu, T, kv, hd, page, dt, quant):
    from chestnut import kernels as K
    rng = np.random.default_rng(T + hd)
    k, v = rows(3, T, 2 * kv, hd, dt, 5.0)[:, :kv], rows(4, T, kv, hd, dt, 1e-3)
    v[0, 0] = 0
    v[0, 0, hd // 2] = 448 * 2.0 ** -9          # the scale's border: held, and the next value up
    if T > 1:
        v[1, 0] = v[1, 0] * 0
        v[1, 0, 0] = torch.nextafter(torch.tensor(448 * 2.0 ** -9, dtype=DT[dt]), torch.tensor(9e9, dtype=DT[dt]))
        k[1, 0] = torch.linspace(-500, 500, hd).to(DT[dt]).cuda()
    if T > 3:
        k[2, 0], k[3, 0] = 0, 0
        k[3, 0, 0], k[3, 0, 1], k[3, 0, 2] = float('inf'), float('-inf'), float('nan')
    n = -(-T // page) + 2
    slots = rng.permutation(n * page)[:T]
    keep = np.ones(T, bool)
    if T > 5:
        slots[4], keep[4] = -1, False
        slots[5], keep[5] = n * page, False     # outside the cache: not written
    kp, vp, ks, vs = pages_of(n, kv, page, hd, dt, 'e4m3' if quant else dt)
    K.cache_write(k, v, kp, vp, i32(slots), k_scale=ks, v_scale=vs)
    for x, p, s in ((k, kp, ks), (v, vp, vs)):
        if quant:
            codes, byte = O.quantise(f64(x), TOP[dt])
            wantp, wants = np.full(p.shape, 0x5A, np.uint8), np.full(s.shape, 99, np.uint8)
            for t in np.nonzero(keep)[0]:
                wantp[slots[t] // page, :, slots[t] % page] = codes[t]
                wants[slots[t] // page, :, slots[t] % page] = byte[t]
            got = p.view(torch.uint8).cpu().numpy()
            nan = (wantp & 127) == 127
            assert np.array_equal(got[~nan], wantp[~nan]) and np.all((got[nan] & 127) == 127)
            assert np.array_equal(s.view(torch.uint8).cpu().numpy(), wants)
        else:
            want = torch.full(p.shape, 3.0, dtype=DT[dt])
            for t in np.nonzero(keep)[0]:
                want[slots[t] // page, :, slots[t] % page] = x[t].cpu()
            assert torch.equal(p.cpu().view(torch.int16), want.view(torch.int16))


@pytest.mark.parametrize('lens,kv,hd,page', [([1], 1, 64, 16), ([0, 33, 0, 5, 64], 3, 128, 32), ([700, 16], 2, 72, 16),
                                             ([1] * 150, 1, 64, 16)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
def test_cache_read(gpu, lens, kv, hd, page, dt, quant):
    from chestnut import kernels as K
    table, n = tables(lens, page, 7)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if quant else dt, 9)
    T = sum(lens) + 3
    ko = torch.full((T, kv, hd), 5.0, dtype=DT[dt], device='cuda')
    k, v = K.cache_read(kp, vp, i32(table), cu(lens), T, k_scale=ks, v_scale=vs, dtype=DT[dt], k_out=ko)
    assert k is ko and (k[T - 3:] == 5.0).all()
    for got, p, s in ((k, kp, ks), (v, vp, vs)):
        want = np.concatenate([gathered(p, s, table[b], m, page) for b, m in enumerate(lens)])
        assert torch.equal(got[:T - 3].cpu(), torch.from_numpy(want).to(DT[dt]))


def tables(lens, page, seed):
    """Shuffled pages; entries behind a sequence's last page point nowhere."""
    need = [-(-m // page) for m in lens]
    perm = np.random.default_rng(seed).permutation(sum(need) + 1)
    t = np.full((len(lens), max(need + [0]) + 2), -123456, np.int64)
    t[:, -1] = 2 ** 31 - 1
    at = 0
    for b, m in enumerate(need):
        t[b, :m] = perm[at:at + m]
        at += m
    return t, sum(need) + 1


def filled(n, kv, page, hd, dt, cache, seed):
    """Pages full of normal values; every place that holds none is NaN (quantised: code 0x7F)."""
    r = np.random.default_rng(seed)
    out = []
    for _ in 'kv':
        x = r.standard_normal((n, kv, page, hd))
        if cache == 'e4m3':
            c, b = O.quantise(x, TOP[dt])
            out.append((torch.from_numpy(c).cuda().view(torch.float8_e4m3fn), torch.from_numpy(b).cuda().view(torch.float8_e8m0fnu)))
        else:
            out.append((torch.from_numpy(x).to(DT[dt]).cuda(), None))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def gathered(p, s, row, m, page):
    """The first m places of a sequence, [m, kv, hd] f64."""
    row = torch.from_numpy(np.ascontiguousarray(row[:-(-m // page)])).cuda()
    if s is None:
        x = f64(p[row])
    else:
        x = O.values(p.view(torch.uint8)[row].cpu().numpy(), s.view(torch.uint8)[row].cpu().numpy())
    return x.transpose(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:m]


# ----------------------------------------------------------------- attention --
VARLEN = [([1], None), ([64], None), ([33, 1, 0, 257], None), ([127, 129, 128], None), ([700], None), ([5, 3], [900, 65]),
          ([40, 7, 9], [8, 0, 9]), ([1] * 70, None), ([1, 1, 1], [1, 4000, 130])]


@pytest.mark.parametrize('lens,klens', VARLEN, ids=lambda x: str(x)[:20])
@pytest.mark.parametrize('H,kv,hd', [(2, 2, 64), (5, 1, 128), (8, 2, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('causal', [True, False])
def test_attention_varlen(gpu, lens, klens, H, kv, hd, dt, causal):
    from chestnut import kernels as K
    T, kl = sum(lens), klens or lens
    qkv = rows(T, T, H + 2, hd, dt)
    kvb = rows(T + 1, sum(kl), 2 * kv + 1, hd, dt)
    q, k, v = qkv[:, 1:1 + H], kvb[:, :kv], kvb[:, kv:2 * kv]
    out = torch.full((T + 2, H, hd), 9.0, dtype=DT[dt], device='cuda')
    qq = torch.cat((q, q[:1], q[:1])) if T else q
    got = K.attention_varlen(qq, k, v, cu(lens), cu(kl), causal=causal, out=out)
    assert got is out and (out[T:] == 9.0).all()
    a = b = 0
    for n, m in zip(lens, kl):
        ref, mag, most = O.attention(f64(q[a:a + n]), f64(k[b:b + m]), f64(v[b:b + m]), causal)
        near(out[a:a + n], ref, mag, most, m, hd, dt, f'{n} over {m}')
        a, b = a + n, b + m


@pytest.mark.parametrize('qlens,klens', [([1], [1]), ([1, 1, 1], [63, 64, 1025]), ([64], [64]), ([5, 0, 100], [5, 20, 333]),
                                         ([130, 1, 31], [700, 900, 17]), ([1] * 9, [100 * i for i in range(9)]), ([1], [5000])])
@pytest.mark.parametrize('H,kv,hd,page', [(4, 4, 64, 16), (8, 2, 128, 32), (7, 1, 128, 256)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('causal', [True, False])
def test_attention_paged(gpu, qlens, klens, H, kv, hd, page, dt, quant, causal):
    from chestnut import kernels as K
    table, n = tables(klens, page, 5)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if quant else dt, 6)
    q = rows(8, sum(qlens), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, causal=causal)
    a = 0
    for b, (x, m) in enumerate(zip(qlens, klens)):
        k, v = gathered(kp, ks, table[b], m, page), gathered(vp, vs, table[b], m, page)
        ref, mag, most = O.attention(f64(q[a:a + x]), k, v, causal)
        near(out[a:a + x], ref, mag, most, m, hd, dt, f'{x} over {m}')
        a += x


def attention_on_gpu(q, k, v, causal):
    """oracle.attention's three results for long sequences of finite values: f64 on the device."""
    q, k, v = q.double(), k.double(), v.double()
    (n, H, hd), (m, kv, _) = q.shape, k.shape
    out, mag, most = torch.zeros_like(q), torch.zeros_like(q), 0.0
    see = torch.arange(m, device='cuda')[None] <= torch.arange(n, device='cuda')[:, None] + (m - n if causal else m)
    for h in range(H):
        g = h // (H // kv)
        p = torch.softmax((q[:, h] @ k[:, g].T / hd ** 0.5).masked_fill(~see, -float('inf')), -1)
        out[:, h], mag[:, h] = p @ v[:, g], p @ v[:, g].abs()
        most = max(most, (q[:, h].norm(dim=-1).max() * k[:, g].norm(dim=-1).max() / hd ** 0.5).item())
    return f64(out), f64(mag), most


@pytest.mark.parametrize('lens,H,kv,hd', [([4500, 300, 1111], 8, 2, 128), ([3000], 4, 4, 64), ([2500, 2049, 64], 32, 8, 64),
                                          ([4200], 32, 8, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('causal', [True, False])
def test_long_prompts(gpu, lens, H, kv, hd, dt, causal):
    """Many tiles a row: every buffer of the pipeline many times over, and both tile heights."""
    from chestnut import kernels as K
    q, k, v = rows(1, sum(lens), H, hd, dt), rows(2, sum(lens), kv, hd, dt), rows(3, sum(lens), kv, hd, dt)
    out = K.attention_varlen(q, k, v, cu(lens), causal=causal)
    assert torch.equal(out, K.attention_varlen(q, k, v, cu(lens), causal=causal))
    a = 0
    for n in lens:
        near(out[a:a + n], *attention_on_gpu(q[a:a + n], k[a:a + n], v[a:a + n], causal), n, hd, dt, str(n))
        a += n


@pytest.mark.parametrize('qlens,klens,H,kv,hd', [([2417, 2], [2417, 2], 16, 4, 128), ([5800], [5800], 1, 1, 64), ([1300], [1300], 1, 1, 128),
                                                 ([700, 33, 1500], [4000, 20, 1500], 3, 1, 64), ([200], [9000], 2, 1, 128),
                                                 ([601] * 9 + [40, 0, 1] * 3, [601] * 5 + [1777] * 4 + [2900, 5, 63] * 3, 6, 2, 64)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_causal_prompts_with_their_keys_split(gpu, qlens, klens, H, kv, hd, dt):
    """Tiles of one sequence with different numbers of chunks; nothing behind the workspace is written."""
    from chestnut import kernels as K
    q, k, v = rows(1, sum(qlens), H, hd, dt), rows(2, sum(klens), kv, hd, dt), rows(3, sum(klens), kv, hd, dt)
    nf = K.attention_workspace(len(qlens), sum(qlens), sum(klens), H, kv, hd) // 4
    assert nf > 0
    ws = torch.full((nf + 4096,), 7.0, device='cuda')
    out = K.attention_varlen(q, k, v, cu(qlens), cu(klens), workspace=ws)
    assert (ws[nf:] == 7.0).all()
    ws[:nf] = float('nan')
    assert torch.equal(out, K.attention_varlen(q, k, v, cu(qlens), cu(klens), workspace=ws))
    a = c = 0
    for n, m in zip(qlens, klens):
        e = max(0, n - m)
        assert (out[a:a + e] == 0).all()
        if n > e:
            near(out[a + e:a + n], *attention_on_gpu(q[a + e:a + n], k[c:c + m], v[c:c + m], True), m, hd, dt, f'{n} over {m}')
        a, c = a + n, c + m


@pytest.mark.parametrize('qlens,klens,H,kv,hd,page', [([512], [5000], 2, 2, 128, 64), ([1, 300, 2, 77], [3000, 2500, 6000, 77], 8, 2, 128, 32),
                                                      ([1] * 12, [300 * i + 1 for i in range(12)], 16, 2, 64, 256),
                                                      ([1] * 130, [7 * i for i in range(130)], 4, 2, 128, 16),
                                                      ([800, 900], [3000, 900], 4, 4, 64, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('causal', [True, False])
def test_long_histories(gpu, qlens, klens, H, kv, hd, page, dt, quant, causal):
    """Keys split over workgroups: chunks, more sequences than lanes, ragged lengths."""
    from chestnut import kernels as K
    table, n = tables(klens, page, 5)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if quant else dt, 6)
    q = rows(8, sum(qlens), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, causal=causal)
    assert torch.equal(out, K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, causal=causal))
    a = 0
    for b, (x, m) in enumerate(zip(qlens, klens)):
        if m:
            k, v = (torch.from_numpy(gathered(p, s, table[b], m, page)).cuda() for p, s in ((kp, ks), (vp, vs)))
            near(out[a:a + x], *attention_on_gpu(q[a:a + x], k, v, causal), m, hd, dt, f'{x} over {m}')
        else:
            assert (out[a:a + x] == 0).all()
        a += x


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('paged', [False, True])
@pytest.mark.parametrize('n,m', [(200, 200), (40, 170), (3, 64), (1, 66)])
def test_what_a_row_does_not_see_does_not_reach_it(gpu, dt, hd, paged, n, m):
    """NaN and infinities in K and V of later tokens, and in the places behind the last key."""
    from chestnut import kernels as K
    H, kv, page = 4, 2, 64
    q, k, v = rows(1, n, H, hd, dt), rows(2, m, kv, hd, dt), rows(3, m, kv, hd, dt)
    first = m - n                     # the first query's own place
    for j, x in ((first + (n + 1) // 2, float('nan')), (first + (3 * n) // 4, float('inf')), (m - 1, float('-inf'))):
        if first < j < m:
            v[j, :, j % hd] = x
            k[j, :, 3] = x
    if paged:
        need = -(-m // page)
        kp, vp = (torch.full((need, page, kv, hd), float('nan'), dtype=DT[dt], device='cuda') for _ in 'kv')
        kp.view(-1, kv, hd)[:m], vp.view(-1, kv, hd)[:m] = k, v
        kp, vp = (t.permute(0, 2, 1, 3).contiguous() for t in (kp, vp))
        out = K.attention_paged(q, kp, vp, i32([list(range(need))]), cu([n]), i32([m]))
    else:
        big = torch.full((m + 70, 2 * kv, hd), float('nan'), dtype=DT[dt], device='cuda')
        big[:m, :kv], big[:m, kv:] = k, v
        out = K.attention_varlen(q, big[:, :kv], big[:, kv:], cu([n]), cu([m]))
    clean = min([j for j in range(first, m) if not torch.isfinite(k[j]).all()] + [m]) - first
    ref, mag, most = O.attention(f64(q[:clean]), f64(k[:first + clean]), f64(v[:first + clean]))
    near(out[:clean], ref, mag, most, m, hd, dt)
    assert clean > 0 and not torch.isfinite(out[clean:]).all(-1).any() or clean == n


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('n,m', [(200, 200), (40, 1170), (3, 64)])
def test_nan_codes_that_a_row_does_not_see_do_not_reach_it(gpu, dt, n, m):
    from chestnut import kernels as K
    H, kv, hd, page = 4, 2, 128, 32
    table, total = tables([m], page, 3)
    kp, vp, ks, vs = filled(total, kv, page, hd, dt, 'e4m3', 4)
    k, v = gathered(kp, ks, table[0], m, page), gathered(vp, vs, table[0], m, page)
    first, bad = m - n, m - n // 2          # the first query's own place, and of the first NaN
    for j in list(range(bad, m)) + list(range(m, -(-m // page) * page)):
        vp.view(torch.uint8)[table[0][j // page], :, j % page, j % hd] = 0x7F
        kp.view(torch.uint8)[table[0][j // page], :, j % page, 5] = 0xFF
    q = rows(1, n, H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu([n]), i32([m]), k_scale=ks, v_scale=vs)
    clean = bad - first
    ref, mag, most = O.attention(f64(q[:clean]), k[:bad], v[:bad])
    near(out[:clean], ref, mag, most, m, hd, dt)
    assert not torch.isfinite(out[clean:]).all(-1).any()


@pytest.mark.parametrize('G', [1, 6, 15, 16, 17, 31, 32, 33])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('cache', ['rows', 'pages', 'e4m3'])
def test_few_rows(gpu, G, hd, dt, cache):
    """Single tokens of every group size around the tiles' heights, two tokens at once among them;
    the last key of that sequence holds what its first token must not see."""
    from chestnut import kernels as K
    qlens, klens, kv, page = [2, 0, 1, 1], [777, 9, 64, 5], 2, 16
    q = rows(1, 4, G * kv, hd, dt)
    if cache == 'rows':
        k, v = rows(2, sum(klens), kv, hd, dt), rows(3, sum(klens), kv, hd, dt)
        v[776, 0, 3], v[776, 1, 5] = float('inf'), float('nan')
        out = K.attention_varlen(q, k, v, cu(qlens), cu(klens))
        ks, vs = ([x[sum(klens[:b]):sum(klens[:b + 1])] for b in range(4)] for x in (k, v))
    else:
        table, n = tables(klens, page, 5)
        kp, vp, sk, sv = filled(n, kv, page, hd, dt, 'e4m3' if cache == 'e4m3' else dt, 6)
        at = (int(table[0][776 // page]), 1, 776 % page, 5)
        vp.view(torch.uint8 if cache == 'e4m3' else torch.int16)[at] = 0x7F if cache == 'e4m3' else 0x7FC1
        out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=sk, v_scale=sv)
        ks, vs = ([torch.from_numpy(gathered(p, s, table[b], m, page)).cuda() for b, m in enumerate(klens)]
                  for p, s in ((kp, sk), (vp, sv)))
    assert torch.isnan(out[1, G:, 5]).all() and (cache != 'rows' or (out[1, :G, 3] == float('inf')).all())
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[2:]).all()
    vs[0] = torch.where(torch.isfinite(vs[0]), vs[0], torch.zeros_like(vs[0]))
    out[1, :, 3], out[1, :, 5] = 0, 0
    for a, b, n in ((0, 0, 2), (2, 2, 1), (3, 3, 1)):
        ref, mag, most = attention_on_gpu(q[a:a + n], ks[b], vs[b], True)
        if n == 2:
            ref[1, :, 3], ref[1, :, 5] = 0, 0
        near(out[a:a + n], ref, mag, most, klens[b], hd, dt, f'sequence {b}')


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_infinite_values_of_v_reach_the_rows_that_see_them(gpu, dt):
    from chestnut import kernels as K
    n, hd = 150, 64
    q, k, v = rows(1, n, 2, hd, dt), rows(2, n, 2, hd, dt), rows(3, n, 2, hd, dt)
    v[70, 0, 5], v[100, 0, 5], v[90, 1, 7] = float('inf'), float('-inf'), float('-inf')
    out = f64(K.attention_varlen(q, k, v, cu([n])))
    ref, _, _ = O.attention(f64(q), f64(k), f64(v))
    assert np.array_equal(np.isfinite(out), np.isfinite(ref))
    assert np.array_equal(out[70:100, 0, 5], np.full(30, np.inf)) and np.all(out[90:, 1, 7] == -np.inf)
    assert np.isnan(out[100:, 0, 5]).all()


@pytest.mark.parametrize('hd', [64, 128])
def test_one_key_rules_each_row(gpu, hd):
    """Row t's output is V's row (37 t + 5) mod (t + 1): the order of keys and features."""
    from chestnut import kernels as K
    n = 300
    at = (37 * np.arange(n) + 5) % (np.arange(n) + 1)
    k = rows(1, n, 1, hd, 'f16')
    k = k / k.float().norm(dim=-1, keepdim=True).half()
    q = (k[torch.from_numpy(at).cuda()].float() * 400).half()
    v = rows(2, n, 1, hd, 'f16')
    out = K.attention_varlen(q, k, v, cu([n]), scale=1.0)
    assert torch.equal(out[:, 0].cpu(), v[:, 0].cpu()[torch.from_numpy(at)])


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('T', [1, 300])
@pytest.mark.parametrize('last', [False, True])
def test_many_weak_keys_beside_a_strong_one(gpu, dt, T, last):
    """One key of score 17 and v = 0 beside 60000 of score 0 and v = 1: each of those weighs 2^-24.5
    of it, less than f16 can tell from 1 or 0.  Output 60000 e^-17 / (1 + 60000 e^-17): u of a
    weight and of the output, f16's subnormals 2^-32 each, and 2^-17 for the exponentials and sums."""
    from chestnut import kernels as K
    n = 60001
    q, k, v = (torch.zeros(m, 1, 64, dtype=DT[dt], device='cuda') for m in (T, n, n))
    q[..., 0] = 8.0
    k[n - 1 if last else 0, 0, 0] = 17.0
    v[...] = 1.0
    v[n - 1 if last else 0] = 0.0
    out = f64(K.attention_varlen(q, k, v, cu([T]), cu([n]), causal=False, scale=0.125))
    w = (n - 1) * np.exp(-17.0)
    ref = w / (1 + w)
    tol = ref * (2 * u(dt) * (1 + 2.0 ** -6) + 2.0 ** -17) + ((n - 1) * 2.0 ** -32 if dt == 'f16' else 0.0)
    assert np.abs(out - ref).max() <= tol


def test_index_values_outside_the_tensors_stay_inside(gpu):
    """Lengths, offsets and pages that point outside: the call ends, nothing outside is written,
    and well-formed sequences of the same call are right."""
    from chestnut import kernels as K
    H, kv, hd, page = 2, 1, 64, 16
    kp, vp, _, _ = filled(3, kv, page, hd, 'f16', 'f16', 1)
    q = rows(1, 4, H, hd, 'f16')
    guard = torch.full((6, H, hd), 4.0, dtype=torch.float16, device='cuda')
    K.attention_paged(q, kp, vp, i32([[0, 1], [-7, 99], [2, 0]]), i32([0, 1, 3, 900]), i32([20, 1000000, -5]), out=guard[1:5])
    assert (guard[0] == 4.0).all() and (guard[5] == 4.0).all()
    ref, mag, most = O.attention(f64(q[:1]), gathered(kp, None, np.array([0, 1]), 20, page), gathered(vp, None, np.array([0, 1]), 20, page))
    near(guard[1:2], ref, mag, most, 20, hd, 'f16')
    # offsets that do not ascend name more rows than there are
    kp2, vp2, _, _ = filled(200, kv, page, hd, 'f16', 'f16', 2)
    buf = torch.full((42, H, hd), 4.0, dtype=torch.float16, device='cuda')
    K.attention_paged(rows(2, 40, H, hd, 'f16'), kp2, vp2, i32([list(range(200))] * 5), i32([0, 40, 0, 40, 0, 40]),
                      i32([3000] * 5), out=buf[1:41])
    assert (buf[0] == 4.0).all() and (buf[41] == 4.0).all()
    k, v = K.cache_read(kp, vp, i32([[0, -1], [50, 1]]), i32([0, 17, 40]), 30)
    assert torch.equal(k[:16], kp[0].permute(1, 0, 2)) and k.shape == (30, kv, hd)
    K.cache_read(kp, vp, i32([[0, -1], [50, 1]]), i32([5, -3, 10 ** 9]), 30)


def test_empty_calls(gpu):
    from chestnut import kernels as K
    kp, vp, _, _ = filled(1, 1, 16, 64, 'f16', 'f16', 1)
    e = torch.empty(0, 2, 64, dtype=torch.float16, device='cuda')
    assert K.attention_varlen(e, e[:, :1], e[:, :1], cu([0])).shape == (0, 2, 64)
    assert K.attention_paged(e, kp, vp, torch.empty(0, 1, dtype=torch.int32, device='cuda'), i32([0]), i32([])).shape == (0, 2, 64)
    assert K.rope(e, i32([]), K.rope_frequencies(64)[0]).shape == (0, 2, 64)
    K.cache_write(e[:, :1], e[:, :1], kp, vp, i32([]))
    assert K.cache_read(kp, vp, torch.empty(0, 0, dtype=torch.int32, device='cuda'), i32([0]), 0)[0].shape == (0, 1, 64)
    out = K.attention_paged(rows(1, 2, 2, 64, 'f16'), kp, vp, torch.empty(1, 0, dtype=torch.int32, device='cuda'), i32([0, 2]), i32([7]))
    assert (out == 0).all()


# ------------------------------------------------------- a run of them together --
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
def test_prompt_then_tokens_through_the_cache(gpu, dt, quant):
    """Two streams: a prompt as one packed call, its rows kept in the cache, then a chunk and single
    tokens over the cache.  Without quantisation every step equals attention over the whole sequence."""
    from chestnut import kernels as K
    H, kv, hd, page = 4, 2, 64, 16
    prompt, steps = [37, 90], [20, 1, 1]
    total = [p + sum(steps) for p in prompt]
    f, s = K.rope_frequencies(hd, method='linear', factor=4.0)
    stream = [rows(10 + b, t, H + 2 * kv, hd, dt) for b, t in enumerate(total)]
    need = [-(-t // page) for t in total]
    table = np.zeros((2, max(need)), int)
    table[0, :need[0]] = np.arange(need[0])[::-1]
    table[1, :need[1]] = need[0] + np.arange(need[1])
    kp, vp, ks, vs = pages_of(sum(need), kv, page, hd, dt, 'e4m3' if quant else dt)
    done, outs = [0, 0], [[], []]
    for lens in [prompt] + [[x, x] for x in steps]:
        x = torch.cat([stream[b][done[b]:done[b] + lens[b]] for b in range(2)])
        pos = np.concatenate([np.arange(done[b], done[b] + lens[b]) for b in range(2)])
        slots = np.concatenate([table[b][np.arange(done[b], done[b] + lens[b]) // page] * page +
                                np.arange(done[b], done[b] + lens[b]) % page for b in range(2)])
        x[:, :H + kv] = K.rope(x[:, :H + kv], i32(pos), f, scale=s)
        K.cache_write(x[:, H:H + kv], x[:, H + kv:], kp, vp, i32(slots), k_scale=ks, v_scale=vs)
        done = [d + n for d, n in zip(done, lens)]
        if lens is prompt and not quant:
            o = K.attention_varlen(x[:, :H], x[:, H:H + kv], x[:, H + kv:], cu(lens))
        else:
            o = K.attention_paged(x[:, :H], kp, vp, i32(table), cu(lens), i32(done), k_scale=ks, v_scale=vs)
        outs[0].append(o[:lens[0]])
        outs[1].append(o[lens[0]:])
    k, v = K.cache_read(kp, vp, i32(table), cu(total), sum(total), k_scale=ks, v_scale=vs, dtype=DT[dt])
    at = 0
    for b, t in enumerate(total):
        x = stream[b]
        q = f64(K.rope(x[:, :H], i32(np.arange(t)), f, scale=s))
        ref, mag, most = O.attention(q, f64(k[at:at + t]), f64(v[at:at + t]))
        near(torch.cat(outs[b]), ref, mag, most, t, hd, dt)
        if not quant:
            assert torch.equal(k[at:at + t], K.rope(x[:, H:H + kv], i32(np.arange(t)), f, scale=s))
            assert torch.equal(v[at:at + t], x[:, H + kv:])
        at += t


def test_a_captured_step_replays(gpu):
    """One graph of a decoding step (rotate, write, attend) replayed over moving positions,
    slots and lengths, with eager work between the replays."""
    from chestnut import kernels as K
    H, kv, hd, page, B = 8, 2, 128, 32, 3
    f, _ = K.rope_frequencies(hd)
    kp, vp, ks, vs = filled(60, kv, page, hd, 'bf16', 'e4m3', 3)
    table = i32(np.random.default_rng(0).permutation(60).reshape(B, 20))
    x = rows(1, B, H + 2 * kv, hd, 'bf16')
    pos, slots, lens, cq = i32([0] * B), i32([-1] * B), i32([1] * B), cu([1] * B)

    def step(kp, vp, ks, vs):
        y = K.rope(x[:, :H + kv], pos, f)
        K.cache_write(y[:, H:], x[:, H + kv:], kp, vp, slots, k_scale=ks, v_scale=vs)
        return K.attention_paged(y[:, :H], kp, vp, table, cq, lens, k_scale=ks, v_scale=vs)

    other = [t.clone() for t in (kp, vp)] + [t.view(torch.uint8).clone().view(torch.float8_e8m0fnu) for t in (ks, vs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*other)
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(kp, vp, ks, vs)
    t = table.cpu().numpy()
    for n in (1, 31, 32, 33, 500, 640, 7):
        place = np.array([n, max(1, n // 2), max(1, n - 1)]) - 1
        pos.copy_(i32(place))
        lens.copy_(i32(place + 1))
        slots.copy_(i32(t[np.arange(B), place // page] * page + place % page))
        x.copy_(rows(n, B, H + 2 * kv, hd, 'bf16'))
        want = step(*other)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want), n
        assert torch.equal(kp.view(torch.uint8), other[0].view(torch.uint8))


def test_two_streams_at_once(gpu):
    """Split calls on two streams, each with its own workspace, and a workspace that the caller keeps."""
    from chestnut import kernels as K
    H, kv, hd, page = 8, 2, 128, 32
    sets = []
    for i in range(2):
        table, n = tables([3000, 900], page, i)
        c = filled(n, kv, page, hd, 'f16', 'e4m3', i)
        sets.append((rows(i, 60, H, hd, 'f16'), c, i32(table), cu([1, 59]), i32([3000, 900])))
    run = lambda s, ws=None: K.attention_paged(s[0], s[1][0], s[1][1], s[2], s[3], s[4], k_scale=s[1][2], v_scale=s[1][3], workspace=ws)
    want = [run(s) for s in sets]
    kept = [torch.full((1 << 22,), float('nan'), device='cuda') for _ in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = [[], []]
    for _ in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(sets[i], kept[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i]) for g in got[i])


def test_long_cache_offsets_pass_32_bits(gpu):
    """A cache of over 2^32 elements: a sequence on its last pages, written, read back and attended."""
    from chestnut import kernels as K
    kv, hd, page, n = 8, 128, 1024, 4200                 # 4.4e9 elements of one byte, K and V
    kp, vp = (torch.zeros(n, kv, page, hd, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn) for _ in 'kv')
    ks, vs = (torch.full((n, kv, page), 127, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu) for _ in 'kv')
    m = 1500
    table = np.array([[n - 1, n - 3]])
    k, v, q = rows(1, m, kv, hd, 'f16'), rows(2, m, kv, hd, 'f16'), rows(3, 70, kv, hd, 'f16')
    place = np.arange(m)
    K.cache_write(k, v, kp, vp, i32(table[0][place // page] * page + place % page), k_scale=ks, v_scale=vs)
    gk, gv = K.cache_read(kp, vp, i32(table), cu([m]), m, k_scale=ks, v_scale=vs, dtype=torch.float16)
    for x, g in ((k, gk), (v, gv)):
        assert np.array_equal(f64(g), O.values(*O.quantise(f64(x), TOP['f16'])))
    for rows_of in (q, q[:1]):                           # many rows, few rows
        x = rows_of.shape[0]
        out = K.attention_paged(rows_of, kp, vp, i32(table), cu([x]), i32([m]), k_scale=ks, v_scale=vs)
        ref, mag, most = O.attention(f64(rows_of), f64(gk), f64(gv))
        near(out, ref, mag, most, m, hd, 'f16')


def test_on_another_stream(gpu):
    from chestnut import kernels as K
    q, k, v = rows(1, 300, 4, 64, 'f16'), rows(2, 300, 2, 64, 'f16'), rows(3, 300, 2, 64, 'f16')
    want = K.attention_varlen(q, k, v, cu([100, 200]))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    c = cu([100, 200])
    torch.cuda.synchronize()
    with torch.cuda.stream(s):
        got = K.attention_varlen(q, k, v, c)
    s.synchronize()
    assert torch.equal(got, want)


# ------------------------------------------------------------- NaN that a row sees --
def cached(cache, m, kv, hd, dt, page=16):
    """m keys of a sequence as rows, pages or quantised pages: (k, v) f64 and put(which, a, b): NaN
    into feature 5 of keys a .. b of K/V head 0, and attend(q, causal)."""
    from chestnut import kernels as K
    if cache == 'rows':
        kv_ = [rows(2, m, kv, hd, dt), rows(3, m, kv, hd, dt)]

        def put(which, a, b):
            kv_[which][a:b, 0, 5] = float('nan')
        return f64(kv_[0]), f64(kv_[1]), put, lambda q, causal: K.attention_varlen(q, *kv_, cu([q.shape[0]]), cu([m]), causal=causal)
    table, n = tables([m], page, 3)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if cache == 'e4m3' else dt, 4)

    def put(which, a, b):
        p = (kp, vp)[which]
        j = np.arange(a, b)
        at = (i32(table[0][j // page]).long(), 0, i32(j % page).long(), 5)
        if cache == 'e4m3':
            p.view(torch.uint8)[at] = 0x7F
        else:
            p[at] = float('nan')
    k, v = (gathered(p, s, table[0], m, page) for p, s in ((kp, ks), (vp, vs)))
    return k, v, put, lambda q, causal: K.attention_paged(q, kp, vp, i32(table), cu([q.shape[0]]), i32([m]), k_scale=ks, v_scale=vs,
                                                          causal=causal)


# n queries over m keys of which a .. b are NaN.  Of one or 12 queries the keys are taken in blocks of 32
# over four waves, and in chunks of 128 where they pass 256; of 70 in chunks of 256 where they pass 512:
# the NaN fill a wave's share, a chunk, all the keys, or stand beside finite keys.
NAN_KEYS = [(1, 33, 32, 33), (1, 190, 64, 96), (1, 512, 128, 256), (1, 700, 0, 700), (1, 700, 3, 4), (12, 44, 32, 44), (12, 512, 128, 256),
            (70, 300, 290, 291), (70, 1024, 256, 512), (70, 1024, 0, 1024)]


@pytest.mark.parametrize('n,m,a,b', NAN_KEYS)
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('cache', ['rows', 'pages', 'e4m3'])
@pytest.mark.parametrize('causal', [True, False])
def test_nan_keys_reach_every_row_that_sees_them(gpu, n, m, a, b, hd, dt, cache, causal):
    k, v, put, attend = cached(cache, m, 2, hd, dt)
    put(0, a, b)
    q = rows(1, n, 4, hd, dt)
    out = attend(q, causal)
    clean = min(max(0, a - (m - n)), n) if causal else 0        # queries before the first that sees key a
    assert torch.isnan(out[clean:, :2]).all()
    near(out[:, 2:], *O.attention(f64(q[:, 2:]), k[:, 1:], v[:, 1:], causal), m, hd, dt, 'the other K/V head')
    if clean:
        near(out[:clean, :2], *O.attention(f64(q[:clean, :2]), k[:m - n + clean, :1], v[:m - n + clean, :1], True), m, hd, dt, 'before')


@pytest.mark.parametrize('n,m', [(1, 1), (1, 33), (1, 700), (12, 44), (12, 700), (70, 100), (70, 1024)])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('cache', ['rows', 'pages', 'e4m3'])
@pytest.mark.parametrize('causal', [True, False])
def test_a_nan_query_gives_a_nan_row(gpu, n, m, hd, dt, cache, causal):
    k, v, _, attend = cached(cache, m, 2, hd, dt)
    q = rows(1, n, 4, hd, dt)
    ref, mag, most = O.attention(f64(q), k, v, causal)
    q[n // 2, 1, 7] = float('nan')
    out = attend(q, causal)
    assert torch.isnan(out[n // 2, 1]).all()
    out[n // 2, 1] = torch.from_numpy(ref[n // 2, 1]).to(out)
    near(out, ref, mag, most, m, hd, dt)


def test_offsets_that_name_more_tiles_than_32_bits_hold(gpu):
    """66000 sequences of which every other is all of the queries, 66000 tiles of 16 rows: over 2^31 in all.  All
    compute the same rows, so that the output is that of one.  (k and v are one row repeated, of which 640 are used,
    so that the keys seem many enough to be split.)"""
    from chestnut import kernels as K
    B = T = 66000
    q = rows(1, T, 16, 64, 'f16')
    k, v = (rows(s, 1, 1, 64, 'f16').expand(300 * B, 1, 64) for s in (2, 3))
    assert K.attention_workspace(B, T, 300 * B, 16, 1, 64) > 0
    ends = np.arange(B + 1) % 2
    out = torch.full((T + 2, 16, 64), 9.0, dtype=torch.float16, device='cuda')
    K.attention_varlen(q, k, v, i32(ends * T), i32(ends * 640), causal=False, out=out[1:T + 1])
    want = v[:1].double()
    assert ((out[1:T + 1].double() - want).abs() <= 2 * u('f16') * want.abs()).all()   # equal weights: one rounding
    assert (out[0] == 9.0).all() and (out[T + 1] == 9.0).all()


# ------------------------------------------------------------------ forms by size --
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('causal', [True, False])
def test_long_chunks_over_pages(gpu, hd, dt, quant, causal):
    """Enough rows for tiles of 256 over pages: (4101 * 4 / 256 + 2) * 8 of them."""
    from chestnut import kernels as K
    qlens, klens, H, kv, page = [3001, 1100], [3078, 2001], 32, 8, 32
    assert K.attention_workspace(2, sum(qlens), 2 * 99 * page, H, kv, hd) == 0
    table, n = tables(klens, page, 5)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if quant else dt, 6)
    q = rows(8, sum(qlens), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, causal=causal)
    a = 0
    for b, (x, m) in enumerate(zip(qlens, klens)):
        k, v = (torch.from_numpy(gathered(p, s, table[b], m, page)).cuda() for p, s in ((kp, ks), (vp, vs)))
        near(out[a:a + x], *attention_on_gpu(q[a:a + x], k, v, causal), m, hd, dt, f'{x} over {m}')
        a += x


@pytest.mark.parametrize('byte', [0, 1, 127, 247, 254, 255])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('n', [1, 70])
def test_scales_at_the_ends_of_their_type(gpu, byte, dt, n):
    """A code times its scale as the two types have them (255 is NaN), read back and, being the only key's V, attended."""
    from chestnut import kernels as K
    codes = torch.arange(256, dtype=torch.uint8, device='cuda').view(4, 64)[None, :, None].expand(1, 4, 16, 64).contiguous()
    kp, vp = torch.zeros_like(codes).view(torch.float8_e4m3fn), codes.view(torch.float8_e4m3fn)
    ks, vs = (torch.full((1, 4, 16), b, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu) for b in (127, byte))
    with np.errstate(invalid='ignore', over='ignore'):
        want = torch.from_numpy(O.e4m3_values() * (np.nan if byte == 255 else 2.0 ** (byte - 127))).to(DT[dt]).view(4, 64)
    _, v = K.cache_read(kp, vp, i32([[0]]), cu([1]), 1, k_scale=ks, v_scale=vs, dtype=DT[dt])
    out = K.attention_paged(rows(1, n, 4, 64, dt), kp, vp, i32([[0]]), cu([n]), i32([1]), k_scale=ks, v_scale=vs, causal=False)
    # below the smallest normal number of bf16 a value may be a subnormal or zero
    small = 2.0 ** -126 if dt == 'bf16' else 0.0
    for got in [v[0]] + list(out):
        got = got.cpu()
        nan = torch.isnan(want)
        assert torch.equal(torch.isnan(got), nan)
        assert torch.equal(got[~nan], want[~nan]) if not small else ((got == want) | nan | (want.abs() < small) & (got.abs() < small)).all()


@pytest.mark.parametrize('n', [1, 70])
def test_rows_of_bf16_past_the_range_of_f16(gpu, n):
    """Cached as e4m3 they read and attend as they are in bf16, as infinities in f16."""
    from chestnut import kernels as K
    x = rows(1, 16, 2, 64, 'bf16').clamp(-3, 3)
    x[:, :, ::2] = 2.0 ** 20
    kp, vp, ks, vs = pages_of(1, 2, 16, 64, 'bf16', 'e4m3')
    K.cache_write(torch.zeros_like(x), x, kp, vp, i32(np.arange(16)), k_scale=ks, v_scale=vs)
    for dt in ('bf16', 'f16'):
        _, v = K.cache_read(kp, vp, i32([[0]]), cu([16]), 16, k_scale=ks, v_scale=vs, dtype=DT[dt])
        out = K.attention_paged(rows(2, n, 2, 64, dt), kp, vp, i32([[0]]), cu([n]), i32([16]), k_scale=ks, v_scale=vs, causal=False)
        want = 2.0 ** 20 if dt == 'bf16' else float('inf')
        assert (v[..., ::2] == want).all() and (out[..., ::2] == want).all()
        assert torch.isfinite(v[..., 1::2]).all() and torch.isfinite(out[..., 1::2]).all()


@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_rope_of_an_output_that_the_caches_do_not_hold(gpu, inter, dt):
    from chestnut import kernels as K
    T, H, hd, rot = 6401, 21, 128, 64
    assert T * H * hd * 2 > 32 << 20
    x = rows(1, T, H, hd, dt)
    pos = np.random.default_rng(1).integers(0, 1 << 20, T)
    f, _ = K.rope_frequencies(rot, base=5e5)
    out = K.rope(x, i32(pos), f, interleaved=inter)
    ref = O.rope(f64(x), pos, f64(f), inter)
    mag = np.abs(f64(x)).max() * 2
    assert np.all(np.abs(f64(out) - ref) <= u(dt) * np.abs(ref) * (1 + 2.0 ** -6) + 2.0 ** -20 * mag + 2.0 ** -25)
    assert torch.equal(out[..., rot:], x[..., rot:])
    assert K.rope(x, i32(pos), f, interleaved=inter, out=x) is x and torch.equal(x, out)


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
def test_cache_read_of_an_output_that_the_caches_do_not_hold(gpu, dt, quant):
    from chestnut import kernels as K
    lens, kv, hd, page = [5001, 0, 3299], 16, 128, 64
    assert sum(lens) * kv * hd * 2 > 32 << 20
    table, n = tables(lens, page, 7)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if quant else dt, 9)
    T = sum(lens) + 3
    ko, vo = (torch.full((T, kv, hd), 5.0, dtype=DT[dt], device='cuda') for _ in 'kv')
    K.cache_read(kp, vp, i32(table), cu(lens), T, k_scale=ks, v_scale=vs, k_out=ko, v_out=vo)
    for got, p, s in ((ko, kp, ks), (vo, vp, vs)):
        want = np.concatenate([gathered(p, s, table[b], m, page) for b, m in enumerate(lens)])
        assert torch.equal(got[:T - 3].cpu(), torch.from_numpy(want).to(DT[dt])) and (got[T - 3:] == 5.0).all()


@pytest.mark.parametrize('qlens,klens,H,kv,hd,page', [([1], [1], 4, 4, 64, 16), ([1, 1, 1, 1], [63, 64, 1025, 0], 8, 2, 128, 32),
                                                      ([9, 0, 5], [70, 20, 333], 4, 2, 64, 256), ([130, 1, 31], [700, 900, 17], 7, 1, 128, 16),
                                                      ([200, 100], [4000, 2501], 4, 2, 64, 16), ([200, 100], [4000, 2501], 4, 2, 128, 256),
                                                      ([3001, 1100], [3001, 1999], 32, 8, 64, 64)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('causal', [True, False])
def test_places_behind_the_last_key_do_not_count(gpu, qlens, klens, H, kv, hd, page, dt, quant, causal):
    """NaN (and scale bytes of 255) in every place that holds no key, the pages that no sequence names among them."""
    from chestnut import kernels as K
    table, n = tables(klens, page, 5)
    kp, vp, ks, vs = filled(n, kv, page, hd, dt, 'e4m3' if quant else dt, 6)
    q = rows(8, sum(qlens), H, hd, dt)

    def attend():
        return K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, causal=causal)
    want = attend()
    none = np.ones((n, page), bool)
    for b, m in enumerate(klens):
        j = np.arange(m)
        none[table[b][j // page], j % page] = False
    none = torch.from_numpy(none).cuda()[:, None].expand(n, kv, page)
    for p, s in ((kp, ks), (vp, vs)):
        if quant:
            p.view(torch.uint8)[none] = 0x7F
            s.view(torch.uint8)[none] = 255
        else:
            p[none] = float('nan')
    assert torch.isfinite(want).all() and torch.equal(attend(), want)


@pytest.mark.parametrize('n,m', [(1, 90), (12, 90), (70, 300)])
@pytest.mark.parametrize('hd', [64, 128])
def test_e4m3_rows_below_the_normal_numbers_of_f16(gpu, n, m, hd):
    """V of about 2^-17, whose values in f16 are subnormal: each is rounded to a multiple of 2^-24 (half a
    step: 2^-25), and so is the output."""
    from chestnut import kernels as K
    table, pages = tables([m], 16, 3)
    kp, vp, ks, vs = filled(pages, 2, 16, hd, 'f16', 'e4m3', 4)
    vs.view(torch.uint8).sub_(17)
    q = rows(1, n, 4, hd, 'f16')
    out = f64(K.attention_paged(q, kp, vp, i32(table), cu([n]), i32([m]), k_scale=ks, v_scale=vs))
    k, v = (gathered(p, s, table[0], m, 16) for p, s in ((kp, ks), (vp, vs)))
    assert np.abs(v).max() < 2.0 ** -14 and np.abs(v).mean() > 2.0 ** -19
    ref, mag, most = O.attention(f64(q), k, v)
    tol = u('f16') * mag * (1 + 2.0 ** -6) + (2 * (hd + 4) * 2.0 ** -24 * most + 2.0 ** -17) * mag + 2 * 2.0 ** -25 * (1 + 2.0 ** -6)
    assert np.all(np.abs(out - ref) <= tol) and np.abs(ref).max() > 2.0 ** -20


def test_out_may_be_q(gpu):
    """Whole keys and split ones, few rows and many."""
    from chestnut import kernels as K
    for n, m in ((1, 40), (1, 3000), (12, 2000), (70, 300), (70, 3000), (300, 300)):
        q, k, v = rows(1, n, 4, 64, 'f16'), rows(2, m, 2, 64, 'f16'), rows(3, m, 2, 64, 'f16')
        want = K.attention_varlen(q, k, v, cu([n]), cu([m]))
        assert K.attention_varlen(q, k, v, cu([n]), cu([m]), out=q) is q and torch.equal(q, want)

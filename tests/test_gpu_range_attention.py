"""Attention through a sliding window with first tokens that stay visible, and of sequences that
share their first pages, on the GPU against oracle.token_cache in 64 bits.

Tolerances as in the tests of attention over all keys: u = eps / 2 of the type; the output is rounded
once (u |o|) and each softmax weight once (u times A, the same sum with |v|); f16 weights below the
smallest normal are off by 2^-32 of the strongest each, n of them at most, times |v| < 6; a score is a chain of hd f32
sums ((hd + 4) 2^-24 of its sum of magnitudes, twice); exp2, rescalings and sums less than 2^-17."""
import numpy as np
import pytest
import torch

from oracle import token_cache as O

pytestmark = pytest.mark.gpu
DT = {'f16': torch.float16, 'bf16': torch.bfloat16}


def u(dt):
    return torch.finfo(DT[dt]).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def rows(seed, T, H, hd, dt, scale=1.0):
    return torch.from_numpy(np.random.default_rng(seed).standard_normal((T, H, hd)) * scale).to(DT[dt]).cuda()


def i32(v):
    return torch.tensor(np.asarray(v, np.int32)).cuda()


def cu(lens):
    return i32(np.concatenate([[0], np.cumsum(lens)]))


def near(out, ref, mag, most, n, hd, dt, what=''):
    out = f64(out)
    tiny = 6 * n * 2.0 ** -32 if dt == 'f16' else 0.0
    tol = u(dt) * (np.abs(ref) + mag) * (1 + 2.0 ** -6) + (2 * (hd + 4) * 2.0 ** -24 * most + 2.0 ** -17) * mag + tiny
    bad = ~(np.abs(out - ref) <= tol)
    assert not bad.any(), f'{what}: {bad.sum()} of {bad.size}, worst {np.nanmax(np.abs(out - ref) - tol)}, first {np.argwhere(bad)[0]}'


def pages_of(seed, n, kv, page, hd, dt, cache):
    """Filled pages: (k_pages, v_pages, k_scale, v_scale), and their values in f64."""
    r = np.random.default_rng(seed)
    p, s, vals = [], [], []
    pool = O.e4m3_codes(np.clip(r.standard_normal(4096) * 100, -448, 448))
    for _ in 'kv':
        if cache == 'e4m3':       # values of about a normal distribution's, under 4.5 of rows of three sizes
            c, b = pool[r.integers(0, 4096, (n, kv, page, hd))], r.integers(118, 121, (n, kv, page)).astype(np.uint8)
            p.append(torch.from_numpy(c).cuda().view(torch.float8_e4m3fn))
            s.append(torch.from_numpy(b).cuda().view(torch.float8_e8m0fnu))
            vals.append(O.values(c, b))
        else:
            x = torch.from_numpy(r.standard_normal((n, kv, page, hd))).to(DT[dt])
            p.append(x.cuda())
            s.append(None)
            vals.append(f64(x))
    return p + s, vals


def gathered(vals, table, m, page):
    j = np.arange(m)
    return [x[table[j // page], :, j % page] for x in vals]


def tables(lens, page, seed, spare=3):
    need = [-(-m // page) for m in lens]
    order = np.random.default_rng(seed).permutation(sum(need) + spare)
    t = np.full((len(lens), max(1, max(need, default=1))), -1)
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = order[at:at + n]
        at += n
    return t, sum(need) + spare


def attention_on_gpu(q, k, v, window=None, sinks=0, causal=True):
    """oracle.attention's result by torch in f64, for finite inputs."""
    n, H, hd = q.shape
    m, kv = k.shape[:2]
    q, k, v = q.double(), k.double(), v.double()
    far = (torch.arange(n, device='cuda') + m - n)[:, None] - torch.arange(m, device='cuda')[None]
    see = far >= 0 if causal else torch.ones_like(far, dtype=torch.bool)
    if window is not None:
        see &= (far < window) | (torch.arange(m, device='cuda') < sinks)[None]
    out, mag, most = torch.zeros_like(q), torch.zeros_like(q), 0.0
    for h in range(H):
        g = h // (H // kv)
        s = torch.where(see, q[:, h] @ k[:, g].T / hd ** 0.5, float('-inf'))
        most = max(most, float(torch.where(see, q[:, h].abs() @ k[:, g].abs().T / hd ** 0.5, 0).max()))
        p = torch.nan_to_num(torch.softmax(s, -1))
        out[:, h], mag[:, h] = p @ v[:, g], p @ v[:, g].abs()
    return f64(out), f64(mag), most


def expect(q, k, v, window=None, sinks=0, causal=True):
    """oracle.attention of a sequence of finite values (k, v f64), by torch where that is quicker."""
    if q.shape[0] * k.shape[0] < 30000:
        return O.attention(f64(q), k, v, causal, window=window, sinks=sinks)
    return attention_on_gpu(q, torch.from_numpy(k).cuda(), torch.from_numpy(v).cuda(), window, sinks, causal)


# --------------------------------------------------------------- sliding window --
WINDOWS = [(1, 0), (1, 1), (5, 2), (16, 0), (63, 1), (64, 4), (65, 64), (100, 65), (130, 200), (500, 3), (2 ** 31 + 5, 0), (70, 2 ** 40)]


@pytest.mark.parametrize('window,sinks', WINDOWS)
@pytest.mark.parametrize('lens,klens', [([1], None), ([17, 0, 130], None), ([300], None), ([1, 40, 3], [500, 40, 333]), ([200, 9], [150, 1000]),
                                        ([64], [64]), ([5, 7], [0, 3])], ids=lambda x: str(x)[:20])
@pytest.mark.parametrize('H,kv,hd', [(2, 2, 64), (5, 1, 128), (8, 2, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_window_varlen(gpu, window, sinks, lens, klens, H, kv, hd, dt):
    from chestnut import kernels as K
    ks = klens or lens
    q, k, v = rows(1, sum(lens) + 2, H, hd, dt), rows(2, sum(ks) + (0 if klens else 2), kv, hd, dt), rows(3, sum(ks) + (0 if klens else 2), kv, hd, dt)
    out = torch.full_like(q, 9.0)
    got = K.attention_varlen(q, k, v, cu(lens), None if klens is None else cu(klens), window=window, sinks=sinks, out=out)
    assert got is out and (out[sum(lens):] == 9.0).all()
    a = c = 0
    for n, m in zip(lens, ks):
        ref = expect(q[a:a + n], f64(k[c:c + m]), f64(v[c:c + m]), window, sinks)
        near(out[a:a + n], *ref, m, hd, dt, f'{n} over {m}')
        a, c = a + n, c + m


@pytest.mark.parametrize('window,sinks', [(1, 0), (33, 4), (512, 4), (130, 70), (1500, 0), (4096, 16)])
@pytest.mark.parametrize('qlens,klens', [([1], [1]), ([1], [6144]), ([1, 1, 1], [63, 64, 2025]), ([5, 0, 100], [5, 20, 3333]), ([9, 1], [1700, 4])],
                         ids=lambda x: str(x)[:20])
@pytest.mark.parametrize('H,kv,hd,page', [(4, 4, 64, 16), (8, 2, 128, 32), (7, 1, 128, 256), (32, 2, 64, 64)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
def test_window_paged(gpu, window, sinks, qlens, klens, H, kv, hd, page, dt, quant):
    from chestnut import kernels as K
    table, n = tables(klens, page, 1)
    (kp, vp, ks, vs), vals = pages_of(2, n, kv, page, hd, dt, 'e4m3' if quant else dt)
    q = rows(3, sum(qlens), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, window=window, sinks=sinks)
    a = 0
    for b, (x, m) in enumerate(zip(qlens, klens)):
        k, v = gathered(vals, table[b], m, page)
        near(out[a:a + x], *expect(q[a:a + x], k, v, window, sinks), m, hd, dt, f'{x} over {m}')
        a += x


@pytest.mark.parametrize('lens,H,kv,hd', [([3500, 300, 1111], 8, 2, 128), ([3000], 4, 4, 64), ([2500, 2049, 64], 32, 8, 64)])
@pytest.mark.parametrize('window,sinks', [(40, 4), (1000, 130), (2048, 0)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_long_prompts_through_a_window(gpu, lens, H, kv, hd, window, sinks, dt):
    from chestnut import kernels as K
    T = sum(lens)
    qkv = rows(1, T, H + 2 * kv, hd, dt)
    q, k, v = qkv[:, :H], qkv[:, H:H + kv], qkv[:, H + kv:]
    out = K.attention_varlen(q, k, v, cu(lens), window=window, sinks=sinks)
    a = 0
    for n in lens:
        near(out[a:a + n], *attention_on_gpu(q[a:a + n], k[a:a + n], v[a:a + n], window, sinks), window + sinks, hd, dt, str(n))
        a += n


@pytest.mark.parametrize('qlens,klens,H,kv,hd,page', [([300, 77, 1], [5000, 2500, 3000], 8, 2, 128, 32), ([512], [9000], 4, 4, 64, 16),
                                                      ([1] * 70, list(range(900, 4400, 50)), 8, 2, 128, 64)])
@pytest.mark.parametrize('window,sinks', [(700, 4), (3500, 300)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
def test_chunks_through_a_window(gpu, qlens, klens, H, kv, hd, page, window, sinks, dt, quant):
    from chestnut import kernels as K
    table, n = tables(klens, page, 1)
    (kp, vp, ks, vs), vals = pages_of(2, n, kv, page, hd, dt, 'e4m3' if quant else dt)
    q = rows(3, sum(qlens), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(klens), k_scale=ks, v_scale=vs, window=window, sinks=sinks)
    a = 0
    for b, (x, m) in enumerate(zip(qlens, klens)):
        k, v = (torch.from_numpy(t).cuda() for t in gathered(vals, table[b], m, page))
        near(out[a:a + x], *attention_on_gpu(q[a:a + x], k, v, window, sinks), window + sinks, hd, dt, f'{x} over {m}')
        a += x


@pytest.mark.parametrize('n,m', [(200, 200), (40, 170), (3, 700), (1, 66), (1, 1300)])
@pytest.mark.parametrize('window,sinks', [(20, 0), (50, 4), (64, 70)])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('paged', [False, True])
def test_what_the_window_hides_does_not_reach_a_row(gpu, n, m, window, sinks, hd, dt, paged):
    """Infinities and NaN of V in keys that some rows see and others do not, on both sides of the window; NaN in K is
    NaN for the rows that see it."""
    from chestnut import kernels as K
    H, kv, page = 4, 2, 16
    q, k, v = rows(1, n, H, hd, dt), rows(2, m, kv, hd, dt), rows(3, m, kv, hd, dt)
    r = np.random.default_rng(4)
    for x in (float('inf'), float('-inf'), float('nan')):
        for _ in range(6):
            v[r.integers(m), r.integers(kv), r.integers(hd)] = x
    v[m - 1 - min(window, m - 1), 0, 3], v[max(0, m - window), 1, 5], v[min(sinks, m - 1), 0, 7] = float('inf'), float('nan'), float('-inf')
    k[max(0, m - window - 3), 0, 0] = float('nan')
    if paged:
        table, pages = tables([m], page, 5)
        kp, vp = (torch.full((pages, kv, page, hd), float('nan'), dtype=DT[dt], device='cuda') for _ in 'kv')
        j = np.arange(m)
        slots = i32(table[0][j // page] * page + j % page)
        K.cache_write(k, v, kp, vp, slots)
        out = K.attention_paged(q, kp, vp, i32(table), cu([n]), i32([m]), window=window, sinks=sinks)
    else:
        out = K.attention_varlen(q, k, v, cu([n]), cu([m]), window=window, sinks=sinks)
    ref, mag, most = O.attention(f64(q), f64(k), f64(v), window=window, sinks=sinks)
    got, odd = f64(out), ~np.isfinite(ref)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    assert np.array_equal(got[odd & ~np.isnan(ref)], ref[odd & ~np.isnan(ref)])
    ref[odd], mag[odd] = 0, 0
    near(torch.from_numpy(np.where(odd, 0, got)), ref, np.nan_to_num(mag), most, m, hd, dt)


# ----------------------------------------------------------------- shared pages --
def shared_batch(groups, common, qlens, own, page, seed):
    """Tables of sequences of which those of a group begin with the same pages: (table, pages, kv_lens)."""
    r = np.random.default_rng(seed)
    lens, first = [], []
    for g, n in enumerate(groups):
        for _ in range(n):
            first.append(common[g] // page)
            lens.append(common[g] // page * page + own[len(lens)])
    width = max(1, max(-(-m // page) for m in lens))
    order = list(r.permutation(len(lens) * width + sum(c // page for c in common) + 5))
    n = len(order)
    table = np.full((len(lens), width), -1)
    b = 0
    for g, x in enumerate(groups):
        pre = [order.pop() for _ in range(common[g] // page)]
        for _ in range(x):
            need = max(0, -(-lens[b] // page))
            table[b, :need] = (pre + [order.pop() for _ in range(max(0, need - len(pre)))])[:need]
            b += 1
    return table, n, lens


SHARED = [([1], [64], [1], [1]), ([3], [256], [1, 1, 1], [1, 100, 300]), ([6], [2048], [1] * 6, [1, 64, 100, 7, 300, 129]),
          ([2, 1, 4], [96, 0, 700], [1] * 7, [5, 2000, 90, 1, 1, 33, 64]), ([4], [1024], [40, 1, 0, 200], [40, 10, 3, 500]),
          ([24, 20], [640, 320], [1] * 44, [1 + 37 * i % 200 for i in range(44)]), ([2, 2], [128, 4096], [30, 90, 3, 1], [30, 200, 3, 1000])]


@pytest.mark.parametrize('groups,common,qlens,own', SHARED, ids=lambda x: str(x)[:16])
@pytest.mark.parametrize('H,kv,hd,page', [(4, 4, 64, 16), (8, 2, 128, 32), (7, 1, 128, 64), (32, 2, 64, 32)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('causal', [True, False])
def test_shared_pages(gpu, groups, common, qlens, own, H, kv, hd, page, dt, quant, causal):
    from chestnut import kernels as K
    table, n, lens = shared_batch(groups, common, qlens, own, page, 1)
    (kp, vp, ks, vs), vals = pages_of(2, n, kv, page, hd, dt, 'e4m3' if quant else dt)
    q = rows(3, sum(qlens) + 1, H, hd, dt)
    out = torch.full_like(q, 9.0)
    got = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), k_scale=ks, v_scale=vs, causal=causal, out=out,
                            shared=(cu(groups), i32(common)))
    assert got is out and (out[sum(qlens):] == 9.0).all()
    a = 0
    for b, (x, m) in enumerate(zip(qlens, lens)):
        k, v = gathered(vals, table[b], m, page)
        near(out[a:a + x], *expect(q[a:a + x], k, v, causal=causal), m, hd, dt, f'sequence {b}: {x} over {m}')
        a += x


@pytest.mark.parametrize('H,kv,hd', [(4, 4, 64), (8, 2, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('causal', [True, False])
@pytest.mark.parametrize('many', [False, True])
def test_sequences_that_end_within_the_shared_pages(gpu, H, kv, hd, dt, causal, many):
    """Queries that see a part of the shared keys only, sequences shorter than these, more queries than keys, sequences in no
    group, a length that does not fill its last page, and one that names more than the table holds."""
    from chestnut import kernels as K
    page = 16
    r = np.random.default_rng(5)
    B = 90 if many else 9
    width = 12
    pre = [list(range(0, 12)), list(range(12, 24))]
    cu_s, s_lens = ([3, 40, 80] if many else [1, 4, 8]), [150, 16 * 40]
    table = np.zeros((B, width), int)
    at = 24
    for b in range(B):
        g = 0 if cu_s[0] <= b < cu_s[1] else 1 if cu_s[1] <= b < cu_s[2] else -1
        have = [] if g < 0 else pre[g][:(9 if g == 0 else 12)]
        table[b] = have + list(range(at, at + width - len(have)))
        at += width - len(have)
    lens = r.integers(0, width * page + 1, B)
    qlens = r.integers(0, 14, B)
    qlens[1] = lens[1] + 5
    (kp, vp, _, _), vals = pages_of(2, at, kv, page, hd, dt, dt)
    q = rows(3, int(qlens.sum()), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), causal=causal, shared=(i32(cu_s), i32(s_lens)))
    a = 0
    for b, (x, m) in enumerate(zip(qlens, lens)):
        k, v = gathered(vals, table[b], m, page)
        near(out[a:a + x], *O.attention(f64(q[a:a + x]), k, v, causal), max(1, m), hd, dt, f'sequence {b}: {x} over {m}')
        a += x

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


@pytest.mark.parametrize('sizes', [[1] * 70, [3] * 70 + [0] * 5 + [40], [100, 31]], ids=['70 of one', '76', '2 of many'])
@pytest.mark.parametrize('q', [1, 9])
@pytest.mark.parametrize('H,kv,hd', [(4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_many_groups_and_sequences(gpu, sizes, q, H, kv, hd, dt):
    """More groups and sequences than a wave has lanes; the last sequences in no group."""
    from chestnut import kernels as K
    page = 16
    r = np.random.default_rng(7)
    common = [int(x) * page for x in r.integers(0, 9, len(sizes))]
    n = sum(sizes)
    qlens = list(r.integers(0, q + 1, n + 4)) if q > 1 else [1] * (n + 4)
    own = [int(x + y) for x, y in zip(qlens, r.integers(0, 100, n + 4))]
    table, pages, lens = shared_batch(sizes + [1] * 4, common + [0] * 4, qlens, own, page, 1)
    (kp, vp, _, _), vals = pages_of(2, pages, kv, page, hd, dt, dt)
    x = rows(3, int(sum(qlens)), H, hd, dt)
    out = K.attention_paged(x, kp, vp, i32(table), cu(qlens), i32(lens), shared=(cu(sizes), i32(common)))
    a = 0
    for b, (m, l) in enumerate(zip(qlens, lens)):
        k, v = gathered(vals, table[b], l, page)
        near(out[a:a + m], *expect(x[a:a + m], k, v), max(1, l), hd, dt, f'sequence {b}')
        a += m


@pytest.mark.parametrize('quant', [False, True])
def test_many_rows_over_shared_pages(gpu, quant):
    """So many tiles that no keys are split: the two parts of every row are joined all the same."""
    from chestnut import kernels as K
    H, kv, hd, page, dt = 32, 8, 64, 64, 'bf16'
    groups, common, qlens, own = [2, 1], [640, 128], [1500, 1001, 1800], [1500, 1300, 1800]
    table, n, lens = shared_batch(groups, common, qlens, own, page, 1)
    (kp, vp, ks, vs), vals = pages_of(2, n, kv, page, hd, dt, 'e4m3' if quant else dt)
    q = rows(3, sum(qlens), H, hd, dt)
    out = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), k_scale=ks, v_scale=vs, shared=(cu(groups), i32(common)))
    a = 0
    for b, (x, m) in enumerate(zip(qlens, lens)):
        k, v = gathered(vals, table[b], m, page)
        near(out[a:a + x], *expect(q[a:a + x], k, v), m, hd, dt, f'sequence {b}')
        a += x


@pytest.mark.parametrize('n', [1, 12, 70])
@pytest.mark.parametrize('hd', [64, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_infinities_and_nan_over_shared_pages(gpu, n, hd, dt):
    """In V, in keys that some rows see and others do not, within the shared pages and behind them; NaN in a shared key's K;
    NaN in every place that holds no key."""
    from chestnut import kernels as K
    H, kv, page, common = 4, 2, 16, 128
    lens, qlens = [100 + n, 190, 128 + n, 700], [n] * 4              # the first one's queries end within the shared keys
    B, width = 4, 48
    table = np.array([list(range(8)) + list(range(8 + 40 * b, 8 + 40 * b + 40)) for b in range(B)])
    pages = 8 + 40 * B
    r = np.random.default_rng(4)
    k, v = (torch.full((pages, kv, page, hd), float('nan'), dtype=DT[dt], device='cuda') for _ in 'kv')
    kx, vx = (torch.from_numpy(r.standard_normal((B, width * page, kv, hd))).to(DT[dt]).cuda() for _ in 'kv')
    kx[1:, :common], vx[1:, :common] = kx[:1, :common], vx[:1, :common]
    for x in (float('inf'), float('-inf'), float('nan')):
        for j in r.integers(0, common, 3):
            vx[:, j, r.integers(kv), r.integers(hd)] = x
        for b in range(B):
            vx[b, r.integers(common, max(common + 1, lens[b])), r.integers(kv), r.integers(hd)] = x
    vx[:, 100 + n - 1, 1, 3] = float('inf')                          # the first sequence's last key
    kx[:, 100 + n - 1, 0, 0] = float('nan')
    for b in range(B):
        j = np.arange(max(lens[b], common))
        K.cache_write(kx[b, j], vx[b, j], k, v, i32(table[b][j // page] * page + j % page))
    q = rows(1, sum(qlens), H, hd, dt)
    out = f64(K.attention_paged(q, k, v, i32(table), cu(qlens), i32(lens), shared=(i32([0, B]), i32([common]))))
    for b in range(B):
        a = b * n
        ref, mag, most = O.attention(f64(q[a:a + n]), f64(kx[b, :lens[b]]), f64(vx[b, :lens[b]]))
        got, odd = out[a:a + n], ~np.isfinite(ref)
        assert np.array_equal(np.isnan(got), np.isnan(ref)), b
        assert np.array_equal(got[odd & ~np.isnan(ref)], ref[odd & ~np.isnan(ref)])
        ref[odd], mag[odd] = 0, 0
        near(torch.from_numpy(np.where(odd, 0, got)), ref, np.nan_to_num(mag), most, lens[b], hd, dt, f'sequence {b}')


# --------------------------------------------------------- what users do with them --
def test_index_values_outside_the_tensors_stay_inside(gpu):
    """Whatever the index tensors hold, rows outside `out` and the workspace stay as they were, and the call returns."""
    from chestnut import kernels as K
    r = np.random.default_rng(11)
    B, H, kv, hd, page, n, width, T = 50, 8, 2, 64, 16, 40, 6, 90
    (kp, vp, _, _), _ = pages_of(2, n, kv, page, hd, 'f16', 'f16')
    q = rows(3, T, H, hd, 'f16')
    wild = lambda *s: i32(np.where(r.random(s) < 0.5, r.integers(-2 ** 31, 2 ** 31, s), r.integers(-3, 100, s)))
    for trial in range(12):
        N = [1, 3, 70][trial % 3]
        out = torch.full((T + 2, H, hd), 7.0, dtype=torch.float16, device='cuda')
        nb = K.attention_workspace(B, T, B * width * page, H, kv, hd, groups=N)
        ws = torch.full((nb // 4 + 64,), float(trial), device='cuda')
        ws[:nb // 4].view(torch.int32).copy_(wild(nb // 4))              # what stands in a workspace says nothing
        table, lens, offs = wild(B, width), wild(B), wild(B + 1)
        if trial % 2:
            offs = i32(np.sort(r.integers(0, T + 1, B + 1)))
        K.attention_paged(q, kp, vp, table, offs, lens, out=out[1:T + 1], workspace=ws[:nb // 4], shared=(wild(N + 1), wild(N)))
        K.attention_paged(q, kp, vp, table, offs, lens, out=out[1:T + 1], window=int(r.integers(1, 60)), sinks=int(r.integers(0, 9)))
        K.attention_varlen(q, rows(4, 200, kv, hd, 'f16'), rows(5, 200, kv, hd, 'f16'), offs, wild(B + 1), out=out[1:T + 1], window=17, sinks=3)
        torch.cuda.synchronize()
        assert (out[0] == 7.0).all() and (out[T + 1] == 7.0).all() and (ws[nb // 4:] == float(trial)).all()


def test_what_stands_in_a_workspace_does_not_count(gpu):
    from chestnut import kernels as K
    for qlens, own, H, kv, hd in (([1] * 30, [40 * i + 1 for i in range(30)], 8, 2, 128), ([1] * 5, [9, 800, 30, 1, 64], 8, 8, 64),
                                  ([50, 1, 90, 7], [60, 1000, 90, 7], 8, 2, 64)):
        B, page = len(qlens), 32
        table, n, lens = shared_batch([B], [1600], qlens, own, page, 1)
        (kp, vp, ks, vs), _ = pages_of(2, n, kv, page, hd, 'bf16', 'e4m3')
        q = rows(3, sum(qlens), H, hd, 'bf16')
        call = lambda ws, **kw: K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), k_scale=ks, v_scale=vs, workspace=ws, **kw)
        for kw, nb in ((dict(shared=(i32([0, B]), i32([1600]))), K.attention_workspace(B, sum(qlens), table.size * page, H, kv, hd, groups=1)),
                       (dict(window=1500, sinks=4), K.attention_workspace(B, sum(qlens), table.size * page, H, kv, hd, window=1500, sinks=4))):
            want = call(None, **kw)
            for fill in (float('nan'), 0.0, 1e30):
                assert torch.equal(call(torch.full((nb // 4 + 1,), fill, device='cuda'), **kw), want)
            assert torch.equal(call(torch.full((nb // 4 + 1,), -1, dtype=torch.int32, device='cuda').view(torch.float32), **kw), want)


def test_two_streams_at_once(gpu):
    from chestnut import kernels as K
    H, kv, hd, page = 8, 2, 128, 32
    sets = []
    for i in range(2):
        qlens, own = [1] * 20, [13 * j + i + 1 for j in range(20)]
        table, n, lens = shared_batch([12, 8], [3200, 640], qlens, own, page, i)
        c, _ = pages_of(i, n, kv, page, hd, 'f16', 'e4m3')
        sets.append((rows(i, 20, H, hd, 'f16'), c, i32(table), cu(qlens), i32(lens), (i32([0, 12, 20]), i32([3200, 640]))))

    def run(s, ws, window):
        kw = dict(window=1000, sinks=4) if window else dict(shared=s[5])
        return K.attention_paged(s[0], s[1][0], s[1][1], s[2], s[3], s[4], k_scale=s[1][2], v_scale=s[1][3], workspace=ws, **kw)
    want = [[run(s, None, w) for w in (False, True)] for s in sets]
    kept = [torch.full((1 << 24,), float('nan'), device='cuda') for _ in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for j in range(20):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got[i].append(run(sets[i], kept[i], j % 2))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(g, want[i][j % 2]) for j, g in enumerate(got[i]))


def test_out_may_be_q(gpu):
    from chestnut import kernels as K
    for qlens, own in (([1] * 6, [40] * 6), ([1] * 40, [500] * 40), ([70, 3, 200], [70, 300, 900])):
        B, page, H, kv, hd = len(qlens), 16, 8, 2, 64
        table, n, lens = shared_batch([B], [1024], qlens, own, page, 1)
        (kp, vp, _, _), _ = pages_of(2, n, kv, page, hd, 'f16', 'f16')
        for kw in (dict(shared=(i32([0, B]), i32([1024]))), dict(window=700, sinks=5)):
            q = rows(3, sum(qlens), H, hd, 'f16')
            want = K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), **kw)
            assert K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), out=q, **kw) is q and torch.equal(q, want)


@pytest.mark.parametrize('H,kv,hd', [(160, 1, 64), (96, 2, 128), (66, 1, 128)])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('qlens', [[1], [1, 1, 1], [2, 0, 3, 40]], ids=str)
def test_many_heads_on_one_of_the_cache(gpu, H, kv, hd, dt, qlens):
    """A query's heads fill a tile and more; rows before the first sequence and behind the last stay as they were."""
    from chestnut import kernels as K
    B, page, front, own = len(qlens), 16, 5, [1 + 90 * b + x for b, x in enumerate(qlens)]
    table, n, lens = shared_batch([B], [448], qlens, own, page, 1)
    (kp, vp, _, _), vals = pages_of(2, n, kv, page, hd, dt, dt)
    q = rows(3, front + sum(qlens) + 2, H, hd, dt)
    starts = cu(qlens) + front
    for kw in (dict(shared=(i32([0, B]), i32([448]))), dict(window=200, sinks=5)):
        out = torch.full_like(q, 9.0)
        K.attention_paged(q, kp, vp, i32(table), starts.int(), i32(lens), out=out, **kw)
        assert (out[:front] == 9.0).all() and (out[front + sum(qlens):] == 9.0).all()
        a = front
        for b, (x, m) in enumerate(zip(qlens, lens)):
            k, v = gathered(vals, table[b], m, page)
            near(out[a:a + x], *expect(q[a:a + x], k, v, kw.get('window'), kw.get('sinks', 0)), m, hd, dt, f'sequence {b}: {x} over {m}')
            a += x


def test_strided_queries_and_outputs(gpu):
    from chestnut import kernels as K
    H, kv, hd, page, qlens, own = 6, 3, 64, 16, [1, 5, 33], [20, 5, 400]
    table, n, lens = shared_batch([3], [160], qlens, own, page, 1)
    (kp, vp, _, _), _ = pages_of(2, n, kv, page, hd, 'bf16', 'bf16')
    wide = rows(3, sum(qlens), H + 4, hd + 8, 'bf16')
    q = wide[:, 2:2 + H, :hd]
    for kw in (dict(shared=(i32([0, 3]), i32([160]))), dict(window=100, sinks=5)):
        want = K.attention_paged(q.contiguous(), kp, vp, i32(table), cu(qlens), i32(lens), **kw)
        buf = torch.full((sum(qlens), H + 2, hd + 4), 5.0, dtype=torch.bfloat16, device='cuda')
        K.attention_paged(q, kp, vp, i32(table), cu(qlens), i32(lens), out=buf[:, 1:1 + H, :hd], **kw)
        assert torch.equal(buf[:, 1:1 + H, :hd], want)
        buf[:, 1:1 + H, :hd] = 5.0
        assert (buf == 5.0).all()


def test_empty_calls(gpu):
    from chestnut import kernels as K
    (kp, vp, _, _), _ = pages_of(2, 3, 2, 16, 64, 'f16', 'f16')
    none = torch.zeros(0, 4, 64, dtype=torch.float16, device='cuda')
    for kw in (dict(shared=(i32([0, 2]), i32([16]))), dict(window=5)):
        assert K.attention_paged(none, kp, vp, i32([[0], [0]]), i32([0, 0, 0]), i32([16, 16]), **kw).shape == (0, 4, 64)
        q = rows(1, 3, 4, 64, 'f16')
        assert (K.attention_paged(q, kp, vp, i32(np.zeros((2, 0))), i32([0, 1, 3]), i32([5, 5]), **kw) == 0).all()     # no pages: no keys
        out = torch.full_like(q, 3.0)
        K.attention_paged(q, kp, vp, i32([[0], [0]]), i32([0, 0, 0]), i32([16, 16]), out=out, **kw)                    # no sequence has a row
        assert (out == 3.0).all()
    assert K.attention_varlen(none, none, none, i32([0]), window=3).shape == (0, 4, 64)


def test_long_cache_offsets_pass_32_bits(gpu):
    """A cache of over 2^32 elements: shared pages and a window on its last pages."""
    from chestnut import kernels as K
    kv, hd, page, n = 8, 128, 1024, 4200
    kp, vp = (torch.zeros(n, kv, page, hd, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn) for _ in 'kv')
    ks, vs = (torch.full((n, kv, page), 127, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu) for _ in 'kv')
    table = np.array([[n - 1, n - 3], [n - 1, n - 2]])
    lens = [1500, 1324]
    k, v = rows(1, 2048 + 1024, kv, hd, 'f16'), rows(2, 2048 + 1024, kv, hd, 'f16')
    j = np.arange(1024)
    K.cache_write(k, v, kp, vp, i32(np.concatenate([(n - 1) * page + j, (n - 3) * page + j, (n - 2) * page + j])), k_scale=ks, v_scale=vs)
    gk, gv = (O.values(*O.quantise(f64(x), 61440.0)) for x in (k, v))
    for m in (1, 60):
        q = rows(3, 2 * m, kv, hd, 'f16')
        for kw in (dict(shared=(i32([0, 2]), i32([1024]))), dict(window=700, sinks=70)):
            out = K.attention_paged(q, kp, vp, i32(table), cu([m, m]), i32(lens), k_scale=ks, v_scale=vs, **kw)
            for b in range(2):
                at = np.concatenate([j, (1 + b) * 1024 + j])[:lens[b]]
                ref = O.attention(f64(q[b * m:b * m + m]), gk[at], gv[at], window=kw.get('window'), sinks=kw.get('sinks', 0))
                near(out[b * m:b * m + m], *ref, lens[b], hd, 'f16', str(kw.keys()))


# ------------------------------------------------------------------ a run of them --
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('kind', ['window', 'shared'])
def test_a_run_of_steps(gpu, dt, quant, kind):
    """Prompts, then single tokens, a step each of cache_maps, norm_rope, cache_write and attention_paged, whose results follow
    from the whole sequence: its rows normed, turned by three axes, cached (e4m3: as cache_read reads them) and attended in
    64 bits.  The last steps are replays of a captured one, beside the same steps run eagerly on state of their own."""
    from chestnut import kernels as K
    H, kv, hd, page, B, steps = 8, 2, 64, 16, 5, 9
    r = np.random.default_rng(12)
    lens, pre = np.array([3, 40, 17, 1, 64]), (48 if kind == 'shared' else 0)
    total = lens + steps
    qkv = [rows(30 + b, int(total[b]), H + 2 * kv, hd, dt) for b in range(B)]
    first = rows(29, pre, H + 2 * kv, hd, dt)                                         # what all share
    f, s = K.rope_frequencies(48, base=1e4)
    axes = K.rope_axes([8, 8, 8], turns=True)
    wq, wk = (torch.rand(hd, device='cuda').to(DT[dt]) + 0.5 for _ in 'qk')
    width = -(-int(pre + total.max()) // page) + 1
    n_pages = B * width + 3
    free = i32(r.permutation(n_pages))

    def state():
        if quant:
            c = [torch.zeros(n_pages, kv, page, hd, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn) for _ in 'kv'] + \
                [torch.zeros(n_pages, kv, page, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu) for _ in 'kv']
        else:
            c = [torch.zeros(n_pages, kv, page, hd, dtype=DT[dt], device='cuda') for _ in 'kv'] + [None, None]
        return dict(cache=c, table=torch.full((B, width), -1, dtype=torch.int32, device='cuda'), kv=torch.zeros(B, dtype=torch.int32, device='cuda'),
                    taken=i32([0]))

    def step(st, new, x, out=None):
        cu_q, kv_lens, pos, slots = K.cache_maps(new, st['kv'], st['table'], page, x.shape[0], free_pages=free, taken=st['taken'], kv_out=st['kv'])
        at = torch.stack([pos, pos // 7, pos % 7])                                     # time, row and column of a place
        q, k = x[:, :H], x[:, H:H + kv]
        K.norm_rope(q, k, wq, wk, at, f, axes=axes, scale=s, q_out=q, k_out=k)
        kp, vp, ks, vs = st['cache']
        K.cache_write(k, x[:, H + kv:], kp, vp, slots, k_scale=ks, v_scale=vs)
        kw = dict(window=21, sinks=2) if kind == 'window' else dict(shared=(i32_dev[0], i32_dev[1]))
        return K.attention_paged(q, kp, vp, st['table'], cu_q, kv_lens, k_scale=ks, v_scale=vs, out=out, **kw)
    i32_dev = (i32([0, B]), i32([pre]))

    def begin(st):
        """The shared rows in pages that all tables begin with."""
        if not pre:
            return
        K.cache_maps(i32([pre]), i32([0]), st['table'][:1], page, pre, free_pages=free, taken=st['taken'])
        st['table'][1:] = st['table'][:1]
        j = np.arange(pre)
        slots = (st['table'][0][i32(j // page).long()] * page + i32(j % page)).int()
        x = first.clone()
        pos = i32(j)
        K.norm_rope(x[:, :H], x[:, H:H + kv], wq, wk, torch.stack([pos, pos // 7, pos % 7]), f, axes=axes, scale=s, q_out=x[:, :H],
                    k_out=x[:, H:H + kv])
        K.cache_write(x[:, H:H + kv], x[:, H + kv:], st['cache'][0], st['cache'][1], slots, k_scale=st['cache'][2], v_scale=st['cache'][3])
        st['kv'].fill_(pre)

    # the whole sequences in 64 bits
    want = []
    for b in range(B):
        x = f64(torch.cat([first, qkv[b]]))
        j = np.arange(x.shape[0])
        at = np.stack([j, j // 7, j % 7])
        y = [O.rope(O.rms_norm(x[:, a:c], f64(w)), at, f64(f), False, s, axes=axes.tolist()) for a, c, w in ((0, H, wq), (H, H + kv, wk))]
        q, k = (f64(torch.from_numpy(t).to(DT[dt])) for t in y)
        v = x[:, H + kv:]
        if quant:
            k, v = (O.values(*O.quantise(t, 61440.0 if dt == 'f16' else 1.875 * 2.0 ** 127)) for t in (k, v))
        ref, mag, most = O.attention(q, k, v, window=21 if kind == 'window' else None, sinks=2 if kind == 'window' else 0)
        want.append((ref[pre:], mag[pre:], most))

    def close(out, b, i, what):
        """q, k (and their codes) differ from the oracle's by a step here and there: a rounding of the norm's result that falls
        the other way, u of its size each, moves a score by 2 u sum |q k| (e4m3: a code by 2^-3 of its size), and the
        weights and the output by as much of A."""
        ref, mag, most = want[b]
        move = 2 * u(dt) * most + (2.0 ** -3 * most if quant else 0)
        tol = (u(dt) * 3 + 2 * move + 2.0 ** -10) * mag[i]
        assert np.all(np.abs(f64(out) - ref[i]) <= tol + u(dt) * np.abs(ref[i])), f'{what}: request {b}, row {i}'

    a, e = state(), state()                  # one stepped by replays at last, one eagerly
    outs = []
    for st in (a, e):
        begin(st)
        x = torch.cat([qkv[b][:lens[b]] for b in range(B)] + [torch.zeros(2, H + 2 * kv, hd, dtype=DT[dt], device='cuda')])     # and padded rows
        outs.append(step(st, i32(lens), x)[:int(lens.sum())])
    assert torch.equal(*outs)
    at = 0
    for b in range(B):
        for i in range(lens[b]):
            close(outs[0][at + i], b, i, 'prompt')
        at += lens[b]
    ones, x = i32([1] * B), torch.zeros(B, H + 2 * kv, hd, dtype=DT[dt], device='cuda')
    token = lambda t: torch.stack([qkv[b][lens[b] + t] for b in range(B)])
    out = torch.zeros(B, H, hd, dtype=DT[dt], device='cuda')
    x.copy_(token(0))
    step(a, ones, x, out)
    wanted = step(e, ones, token(0))
    assert torch.equal(out, wanted)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            step(a, ones, x, out)
    torch.cuda.synchronize()
    for t in range(1, steps):
        x.copy_(token(t))
        g.replay()
        wanted = step(e, ones, token(t))
        torch.cuda.synchronize()
        assert torch.equal(out, wanted) and torch.equal(a['kv'], e['kv']) and torch.equal(a['table'], e['table']), t
        assert torch.equal(a['cache'][0].view(torch.uint8), e['cache'][0].view(torch.uint8)) and torch.equal(a['taken'], e['taken'])
        for b in range(B):
            close(out[b], b, lens[b] + t, f'step {t}')
    assert np.array_equal(a['kv'].cpu().numpy(), pre + total)


# --------------------------------------------- many groups and sequences, keys split --
def splits(B, T, keys, H, kv, hd, groups):
    """Whether a call over shared pages splits its keys: the sums of chunks then have room in the workspace."""
    from chestnut import kernels as K
    return K.attention_workspace(B, T, keys, H, kv, hd, groups=groups) > K.attention_workspace(B, T, 0, H, kv, hd, groups=groups)


def long_batch(sizes, alone, q, page, seed):
    """Groups of these sizes on up to 1500 shared keys and sequences of up to 2500 of their own, most of them short;
    `alone` sequences in no group behind them: (table, pages, kv_lens, q_lens, common)."""
    r = np.random.default_rng(seed)
    common = [int(x) // page * page for x in r.choice([0, 40, 700, 1100, 1500], len(sizes), p=[0.1, 0.1, 0.3, 0.3, 0.2])]
    first = [common[g] for g, n in enumerate(sizes) for _ in range(n)] + [0] * alone
    qlens = [1] * len(first) if q == 1 else [int(x) for x in r.integers(0, q + 1, len(first))]
    own = [x + int(y) for x, y in zip(qlens, r.choice([0, 3, 90, 600, 2500], len(first), p=[0.2, 0.3, 0.3, 0.15, 0.05]))]
    own[-1] = 2500
    lens = [f + o for f, o in zip(first, own)]
    need = [-(-o // page) for o in own]
    order = list(r.permutation(sum(c // page for c in common) + sum(need) + 3))
    table = np.full((len(first), -(-max(lens) // page)), -1)
    b = 0
    for g, n in enumerate(list(sizes) + [1] * alone):
        pre = [order.pop() for _ in range(common[g] // page)] if g < len(sizes) else []
        for _ in range(n):
            mine = pre + [order.pop() for _ in range(need[b])]
            table[b, :len(mine)] = mine
            b += 1
    return table, sum(c // page for c in common) + sum(need) + 3, lens, qlens, common


@pytest.mark.parametrize('sizes,alone', [([1] * 70, 4), ([3] * 70 + [0] * 5 + [40], 4), ([100, 31], 4), ([2] * 100, 0)],
                         ids=['70 of one', '76', '2 of many', '100 of two'])
@pytest.mark.parametrize('q', [1, 9])
@pytest.mark.parametrize('H,kv,hd', [(4, 4, 64), (16, 2, 128)])
@pytest.mark.parametrize('dt,quant', [('f16', False), ('bf16', True)])
def test_many_groups_and_sequences_whose_keys_are_split(gpu, sizes, alone, q, H, kv, hd, dt, quant):
    """More groups and sequences than a wave has lanes, several chunks of shared and of own keys each: by 16 rows, by tiles
    beside 16 rows, and by tiles."""
    from chestnut import kernels as K
    page = 32
    table, pages, lens, qlens, common = long_batch(sizes, alone, q, page, 7)
    B, T = len(lens), sum(qlens)
    assert splits(B, T, table.size * page, H, kv, hd, len(sizes))
    (kp, vp, ks, vs), vals = pages_of(2, pages, kv, page, hd, dt, 'e4m3' if quant else dt)
    x = rows(3, T, H, hd, dt)
    out = K.attention_paged(x, kp, vp, i32(table), cu(qlens), i32(lens), k_scale=ks, v_scale=vs, shared=(cu(sizes), i32(common)))
    a = 0
    for b, (m, l) in enumerate(zip(qlens, lens)):
        k, v = gathered(vals, table[b], l, page)
        near(out[a:a + m], *expect(x[a:a + m], k, v), max(1, l), hd, dt, f'sequence {b}: {m} over {l}')
        a += m


@pytest.mark.parametrize('T', [90, 300, 700])
def test_index_values_outside_the_tensors_stay_inside_where_keys_are_split(gpu, T):
    """As test_index_values_outside_the_tensors_stay_inside, with tables and windows of so many keys that every form splits
    them: by few rows and by tiles, and their joining launches."""
    from chestnut import kernels as K
    r = np.random.default_rng(13)
    B, H, kv, hd, page, n, width, Tk = 50, 8, 2, 64, 16, 40, 200, 45000
    (kp, vp, _, _), _ = pages_of(2, n, kv, page, hd, 'f16', 'f16')
    q, k, v = rows(3, T, H, hd, 'f16'), rows(4, Tk, kv, hd, 'f16'), rows(5, Tk, kv, hd, 'f16')
    wild = lambda *s: i32(np.where(r.random(s) < 0.5, r.integers(-2 ** 31, 2 ** 31, s), r.integers(-3, 4000, s)))
    for trial in range(12):
        N, window, sinks = [1, 3, 70][trial % 3], int(r.integers(800, 2500)), int(r.integers(0, 90))
        assert splits(B, T, B * width * page, H, kv, hd, N)
        table, lens, offs = wild(B, width), wild(B), wild(B + 1)
        if trial % 2:
            offs = i32(np.sort(r.integers(0, T + 1, B + 1)))
        paged = lambda **kw: K.attention_paged(q, kp, vp, table, offs, lens, **kw)
        calls = [(B * width * page, dict(groups=N), lambda **kw: paged(shared=(wild(N + 1), wild(N)), **kw)),
                 (B * width * page, dict(groups=N), lambda **kw: paged(shared=(i32(np.sort(r.integers(0, B + 1, N + 1))), wild(N)), causal=False, **kw)),
                 (B * width * page, dict(window=window, sinks=sinks), lambda **kw: paged(window=window, sinks=sinks, **kw)),
                 (Tk, dict(window=window, sinks=sinks), lambda **kw: K.attention_varlen(q, k, v, offs, wild(B + 1), window=window, sinks=sinks, **kw))]
        for keys, form, call in calls:
            nb = K.attention_workspace(B, T, keys, H, kv, hd, **form)
            assert nb > 0
            ws = torch.full((nb // 4 + 64,), float(trial), device='cuda')
            ws[:nb // 4].view(torch.int32).copy_(wild(nb // 4))
            out = torch.full((T + 2, H, hd), 7.0, dtype=torch.float16, device='cuda')
            print(f'trial {trial}: {form}', flush=True)
            call(out=out[1:T + 1], workspace=ws[:nb // 4])
            torch.cuda.synchronize()
            assert (out[0] == 7.0).all() and (out[T + 1] == 7.0).all() and (ws[nb // 4:] == float(trial)).all()


@pytest.mark.parametrize('n', [1, 70])
def test_a_window_over_rows_whose_offsets_pass_32_bits(gpu, n):
    from chestnut import kernels as K
    H, kv, hd, m, Tk = 4, 1, 64, 2500, 2 ** 26 + 5000
    k, v = (torch.zeros(Tk, kv, hd, dtype=torch.float16, device='cuda') for _ in 'kv')
    k[-m:], v[-m:] = rows(2, m, kv, hd, 'f16'), rows(3, m, kv, hd, 'f16')
    assert k[-m:].storage_offset() > 2 ** 32
    q = rows(1, n, H, hd, 'f16')
    for window, sinks in ((1000, 70), (300, 0)):
        out = K.attention_varlen(q, k, v, i32([0, 0, n]), i32([0, Tk - m, Tk]), window=window, sinks=sinks)
        near(out, *expect(q, f64(k[-m:]), f64(v[-m:]), window, sinks), m, hd, 'f16', f'{window} and {sinks}')

"""What stands around a step over the token cache, on the GPU against oracle.token_cache in 64 bits:
the step's index tensors from its requests' lengths, rotary positions of several axes, and head
norms with the rotation.

Tolerances.  u = eps / 2 of the element type is the relative error of one rounding.
Index tensors: equal.
rope: as in the tests of one axis (angles exact to 2^-45 turns, cos and sin to 2^-22 each, two
products and a sum in f32, one rounding to the type).
norm_rope: the sum of hd squares is a sum of positive f32 terms, relative error (hd + 4) 2^-24, of
which the root takes half; root, reciprocal and three products add 2^-24 each; then as rope."""
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
    x = np.random.default_rng(seed).standard_normal((T, H, hd)) * scale
    return torch.from_numpy(x).to(DT[dt]).cuda()


def i32(v):
    return torch.tensor(np.asarray(v, np.int32)).cuda()


# -------------------------------------------------------------- rope by axes --
@pytest.mark.parametrize('T,H,hd,sections,turns', [(1, 1, 64, [8, 12, 12], False), (3, 5, 128, [16, 24, 24], True), (700, 3, 64, [8, 8], False),
                                                   (9, 2, 80, [5, 0, 7], True), (5, 3, 33, [1, 2, 1, 1], False), (2, 1, 2, [1], False),
                                                   (33, 4, 256, [100, 28], True), (6500, 21, 128, [16, 8, 8], False)])
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_rope_by_axes(gpu, T, H, hd, sections, turns, inter, dt):
    from chestnut import kernels as K
    half = sum(sections)
    x = rows(T + hd, T, H, hd, dt)
    pos = np.random.default_rng(1).integers(0, 1 << 20, (len(sections), T))
    f, s = K.rope_frequencies(2 * half, base=5e5, method='parts', factor=8.0, context=8192)
    axes = K.rope_axes(sections, turns)
    ref = O.rope(f64(x), pos, f64(f), inter, s, axes=axes.tolist())
    mag = np.abs(f64(x)).max() * 2 * s
    out = K.rope(x, i32(pos), f, interleaved=inter, scale=s, axes=axes)
    assert np.all(np.abs(f64(out) - ref) <= u(dt) * np.abs(ref) * (1 + 2.0 ** -6) + 2.0 ** -20 * mag + 2.0 ** -25)
    assert torch.equal(out[..., 2 * half:], x[..., 2 * half:])
    back = K.rope(out, i32(pos), f, interleaved=inter, scale=1 / s, inverse=True, axes=axes)
    assert np.all(np.abs(f64(back) - f64(x)) <= 4 * u(dt) * mag)
    y = x.clone()
    assert K.rope(y, i32(pos), f, interleaved=inter, scale=s, out=y, axes=axes) is y and torch.equal(y, out)
    # axes that say the same everywhere are one axis.  (Another form of the kernel: where one rounds the product and sum to
    # f16 at once, the other may round to f32 first.  Both are f16 neighbours of the exact value or it: one step apart.)
    one = K.rope(x, i32(pos[0]), f, interleaved=inter, scale=s)
    same = K.rope(x, i32(pos), f, interleaved=inter, scale=s, axes=torch.zeros_like(axes))
    assert torch.equal(K.rope(x, i32(pos[:1].repeat(len(sections), 0)), f, interleaved=inter, scale=s, axes=axes), same)
    step = 2 * u(dt) * torch.maximum(one.abs(), same.abs()).double() + 2.0 ** -24
    assert torch.equal(same, one) or (dt == 'f16' and ((same.double() - one.double()).abs() <= step).all())


def test_axes_outside_the_positions_are_held_to_them(gpu):
    from chestnut import kernels as K
    x, f = rows(1, 40, 3, 64, 'f16'), K.rope_frequencies(64)[0]
    pos = i32(np.random.default_rng(2).integers(0, 5000, (3, 40)))
    axes = i32(np.random.default_rng(3).integers(-2 ** 31, 2 ** 31, 32))
    axes[:6] = i32([-1, 3, 2 ** 31 - 1, -2 ** 31, 0, 2])
    want = K.rope(x, pos, f, axes=axes.clamp(0, 2))
    assert torch.equal(K.rope(x, pos, f, axes=axes), want)
    q, _ = K.norm_rope(x, None, None, None, pos, f, axes=axes)
    assert torch.equal(q, K.norm_rope(x, None, None, None, pos, f, axes=axes.clamp(0, 2))[0])


def test_rope_is_its_own_transpose_by_axes(gpu):
    """inverse is the gradient: <rope(x), g> = <x, inverse(g)>, and as differences say."""
    from chestnut import kernels as K
    T, H, hd = 11, 3, 64
    f = K.rope_frequencies(48)[0]
    axes, pos = K.rope_axes([8, 10, 6]), np.random.default_rng(4).integers(0, 3000, (3, T))
    x, g = rows(5, T, H, hd, 'f16'), rows(6, T, H, hd, 'f16')
    dx = f64(K.rope(g, i32(pos), f, scale=1.5, inverse=True, axes=axes)[..., :48])
    y = lambda v: O.rope(v, pos, f64(f), False, 1.5, axes=axes.tolist())
    for at in [(0, 0, 0), (3, 1, 7), (10, 2, 47), (5, 0, 24)]:
        d = np.zeros((T, H, hd))
        d[at] = 1.0
        want = float(((y(f64(x) + d) - y(f64(x) - d)) / 2 * f64(g)).sum())
        # one rounding to f16 of a sum of two products of up to 1.5 * |g|
        assert abs(dx[at] - want) <= u('f16') * abs(want) * (1 + 2.0 ** -6) + 2.0 ** -19 * 1.5 * 2 * np.abs(f64(g)).max() + 2.0 ** -25


# ------------------------------------------------------------------ norm_rope --
def norm_near(out, x, w, pos, f, inter, scale, axes, eps, dt, what=''):
    hd, rot = x.shape[-1], 2 * len(f)
    y = O.rms_norm(x, w, eps)
    ref = O.rope(y, pos, f, inter, scale, axes=axes)
    mag = np.abs(y).max(-1, keepdims=True) * 2 * max(scale, 1.0)
    tol = u(dt) * np.abs(ref) * (1 + 2.0 ** -6) + mag * (((hd + 4) / 2 + 5) * 2.0 ** -24 + 2.0 ** -20) + (2.0 ** -25 if dt == 'f16' else 0)
    bad = ~(np.abs(f64(out) - ref) <= tol)
    assert not bad.any(), f'{what}: {bad.sum()} of {bad.size}, first {np.argwhere(bad)[0]}'


@pytest.mark.parametrize('T,H,kv,hd,rot', [(1, 1, 1, 64, 64), (3, 5, 1, 128, 64), (17, 16, 4, 128, 128), (700, 3, 2, 64, 16), (9, 2, 2, 80, 24),
                                           (5, 3, 1, 33, 10), (2, 1, 1, 2, 2), (33, 4, 4, 256, 256), (4, 2, 1, 512, 512), (3, 2, 1, 511, 254),
                                           (20, 7, 3, 128, 48), (2, 1, 1, 96, 96), (1, 100, 28, 512, 32)])
@pytest.mark.parametrize('inter', [False, True])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('weight', ['own', 'f32', None])
def test_norm_rope(gpu, T, H, kv, hd, rot, inter, dt, weight):
    from chestnut import kernels as K
    q, k = rows(T + hd, T, H, hd, dt, 3.0), rows(T + hd + 1, T, kv, hd, dt, 0.01)
    if T > 1:
        q[1, 0], k[1, 0] = 0, 0              # no length: zeros
        q[0, 0, 0] = 30000.0                 # one that rules its head
    wt = torch.float32 if weight == 'f32' else DT[dt]
    wq, wk = ((torch.randn(hd, generator=torch.Generator().manual_seed(i)) * 0.3 + 1).to(wt).cuda() if weight else None for i in (0, 1))
    n = 3 if rot >= 8 else 1
    pos = np.random.default_rng(1).integers(0, 1 << 20, (n, T))
    f, s = K.rope_frequencies(rot, base=5e5, method='linear', factor=2.0)
    axes = K.rope_axes([rot // 2 - 2 * (rot // 6), rot // 6, rot // 6]) if n == 3 else None
    p = i32(pos) if n == 3 else i32(pos[0])
    ax = axes.tolist() if n == 3 else None
    for eps, scale in ((1e-6, 1.0), (1e-2, 1.25)):
        a, b = K.norm_rope(q, k, wq, wk, p, f, eps=eps, axes=axes, interleaved=inter, scale=scale)
        for out, x, w, what in ((a, q, wq, 'q'), (b, k, wk, 'k')):
            norm_near(out, f64(x), None if w is None else f64(w), pos if n == 3 else pos[0], f64(f), inter, scale, ax, np.float32(eps), dt, what)
    y, z = q.clone(), k.clone()              # in place, q alone
    c, d = K.norm_rope(y, z, wq, wk, p, f, eps=1e-2, axes=axes, interleaved=inter, scale=1.25, q_out=y, k_out=z)
    assert c is y and d is z and torch.equal(y, a) and torch.equal(z, b)
    c, d = K.norm_rope(q, None, wq, None, p, f, eps=1e-2, axes=axes, interleaved=inter, scale=1.25)
    assert d is None and torch.equal(c, a)


@pytest.mark.parametrize('off', [0, 1, 8])
@pytest.mark.parametrize('hd', [64, 128])
def test_norm_rope_of_a_fused_projection(gpu, off, hd):
    """Strided views in, strided views out; what stands between them is left alone."""
    from chestnut import kernels as K
    T, H, kv = 6, 3, 2
    qkv = rows(2, T, 9, hd + 16, 'f16')
    q, k = qkv[:, 1:1 + H, off:off + hd], qkv[:, 1 + H:1 + H + kv, off:off + hd]
    wq, wk = (torch.rand(hd, device='cuda').half() + 0.5 for _ in 'qk')
    f, _ = K.rope_frequencies(32)
    pos = i32(np.arange(T) * 7)
    wantq, wantk = K.norm_rope(q.contiguous(), k.contiguous(), wq, wk, pos, f)
    buf = torch.full((T, 8, hd + 40), 7.0, dtype=torch.float16, device='cuda')
    oq, ok = buf[:, 1:1 + H, 8:8 + hd], buf[:, 5:5 + kv, 8:8 + hd]
    gq, gk = K.norm_rope(q, k, wq, wk, pos, f, q_out=oq, k_out=ok)
    # (unaligned rows go by another form, whose sum of squares has another order: at most one step of f16, and
    # 2^-20 where products of up to 4.5 cancel)
    tol = 2 * u('f16') + 2.0 ** -16
    for got, view, want in ((gq, oq, wantq), (gk, ok, wantk)):
        assert torch.equal(got, view) and (torch.equal(view, want) if off != 1 else
                                           ((view - want).abs().double() <= tol * want.abs().double() + 2.0 ** -20).all())
    gq, gk = gq.clone(), gk.clone()
    buf[:, 1:1 + H, 8:8 + hd] = 7.0
    buf[:, 5:5 + kv, 8:8 + hd] = 7.0
    assert (buf == 7.0).all()
    keep = qkv.clone()
    K.norm_rope(q, k, wq, wk, pos, f, q_out=q, k_out=k)
    assert torch.equal(q, gq) and torch.equal(k, gk)
    q.copy_(keep[:, 1:1 + H, off:off + hd])
    k.copy_(keep[:, 1 + H:1 + H + kv, off:off + hd])
    assert torch.equal(qkv, keep)


@pytest.mark.parametrize('hd', [64, 80, 128])
@pytest.mark.parametrize('dt', ['f16', 'bf16'])
def test_infinities_and_nan_stay_in_their_head(gpu, hd, dt):
    from chestnut import kernels as K
    q, f = rows(1, 20, 4, hd, dt), K.rope_frequencies(16)[0]
    pos = i32(np.arange(20))
    want = K.norm_rope(q, None, None, None, pos, f)[0]
    q[3, 2, 5], q[7, 0, hd - 1], q[9, 1, 0] = float('nan'), float('inf'), float('-inf')
    got = K.norm_rope(q, None, None, None, pos, f)[0]
    hit = torch.zeros(20, 4, dtype=torch.bool, device='cuda')
    hit[3, 2] = hit[7, 0] = hit[9, 1] = True
    assert torch.equal(got[~hit], want[~hit]) and torch.isnan(got[3, 2]).all() and torch.isnan(got[7, 0, hd - 1])


# ----------------------------------------------------------------- cache_maps --
def check_maps(new, kv, table, page, tokens, free=None, taken=0, in_place=False):
    from chestnut import kernels as K
    want = O.cache_maps(new, kv, table, page, tokens, free, taken)
    t, m = i32(table), i32(kv)
    args = {}
    if free is not None:
        args = dict(free_pages=i32(free), taken=i32([taken]))
        if not in_place:
            args['taken_out'] = torch.full((1,), 77, dtype=torch.int32, device='cuda')
    cu, kv_out, positions, slots = K.cache_maps(i32(new), m, t, page, tokens, kv_out=m if in_place else None, **args)
    assert (kv_out is m) == in_place and (in_place or torch.equal(m, i32(kv)))
    for got, w, what in zip((cu, kv_out, positions, slots, t), want, 'cu kv positions slots table'.split()):
        w = np.asarray(w, np.int64).reshape(tuple(got.shape))
        g = got.cpu().numpy()
        assert np.array_equal(g, w), f'{what}: first {np.argwhere(g != w)[0]}'
    if free is not None:
        assert (args['taken'] if in_place else args['taken_out']).item() == want[5]
        assert in_place or args['taken'].item() == taken


def batch(seed, B, longest, history, page, spare_cols=0):
    r = np.random.default_rng(seed)
    new, kv = r.integers(0, longest + 1, B), r.integers(0, history + 1, B)
    width = max(1, -(-(history + longest) // page) + spare_cols)
    order = r.permutation(B * width + 50)
    table = np.full((B, width), -1)
    at = 0
    for b in range(B):
        n = -(-int(kv[b]) // page)
        table[b, :n] = order[at:at + n]
        at += n
    return new, kv, table, order[at:]


@pytest.mark.parametrize('B,longest,history,page', [(1, 1, 0, 16), (1, 1, 100, 16), (4, 1, 700, 32), (32, 1, 3000, 32), (7, 300, 900, 64), (65, 40, 50, 16),
                                                    (1025, 1, 99, 16), (1500, 9, 40, 16), (3, 5000, 1000, 1024), (200, 17, 0, 128), (5000, 3, 20, 16)])
@pytest.mark.parametrize('listed', [False, True])
@pytest.mark.parametrize('in_place', [False, True])
def test_cache_maps(gpu, B, longest, history, page, listed, in_place):
    new, kv, table, free = batch(B + page, B, longest, history, page)
    if not listed:     # the table names the new pages already, but for one request's
        table = np.random.default_rng(1).permutation(table.size).reshape(table.shape)
        table[B // 2, table.shape[1] // 2:] = -1
    for spare in (0, 1, 1300):
        check_maps(new, kv, table, page, int(new.sum()) + spare, free if listed else None, 3 if listed else 0, in_place)


@pytest.mark.parametrize('in_place', [False, True])
def test_pages_that_run_out(gpu, in_place):
    new, kv, table, free = batch(5, 40, 100, 300, 16)
    total = sum(-(-int(a + b) // 16) - -(-int(b) // 16) for a, b in zip(new, kv))
    for n in (0, 1, total - 1, total):
        check_maps(new, kv, table, 16, int(new.sum()), free[:n], 0, in_place)
    check_maps(new, kv, table, 16, int(new.sum()), free[:total], total, in_place)
    check_maps(new, kv, table, 16, int(new.sum()), free[:total], 2 ** 30, in_place)


def test_places_past_the_table_and_slots_past_31_bits(gpu):
    new, kv, table, free = batch(6, 30, 90, 200, 32)
    check_maps(new, kv, table[:, :3].copy(), 32, int(new.sum()), free, 0)
    check_maps(new, kv, table[:, :3].copy(), 32, int(new.sum()))
    check_maps(new, kv, table[:, :0].copy(), 32, int(new.sum()), free, 0)
    check_maps(new, kv, np.where(table % 3 == 0, 2 ** 26 - 1 + table % 2, table), 32, int(new.sum()))
    check_maps(new, kv, table, 32, int(new.sum()), [2 ** 31 - 1, 5, -3] * 200, 0)
    check_maps([], [], np.zeros((0, 4), np.int32), 16, 0)
    check_maps([], [], np.zeros((0, 4), np.int32), 16, 2000)
    check_maps([0] * 70, [5] * 70, np.zeros((70, 4), np.int32), 16, 10)
    check_maps([3] * 7, [0] * 7, np.full((7, 2), -1), 16, 21, list(range(7)), 0)


@pytest.mark.parametrize('in_place', [False, True])
def test_rows_fewer_than_the_new_tokens(gpu, in_place):
    new, kv, table, free = batch(7, 60, 100, 300, 16)
    for tokens in (0, 1, 900, 1025, 2000):
        check_maps(new, kv, table, 16, tokens, free, 0, in_place)


@pytest.mark.parametrize('in_place', [False, True])
def test_lengths_that_make_no_sense_stay_inside(gpu, in_place):
    """Negative ones count as none; sums are held at 2^31 - 1; nothing outside the tensors is written."""
    from chestnut import kernels as K
    r = np.random.default_rng(8)
    B, T, width = 5000, 3000, 3
    new, kv = r.integers(-2 ** 31, 2 ** 31, B), r.integers(-2 ** 31, 2 ** 31, B)
    new[:1000] = r.integers(-3, 3, 1000)
    kv[:1000] = r.integers(-3, 60, 1000)
    buf = torch.full((B + 2, width), -9, dtype=torch.int32, device='cuda')
    m = i32(kv)
    taken = i32([-5])
    cu, kv_out, positions, slots = K.cache_maps(i32(new), m, buf[1:B + 1], 16, T, free_pages=i32(np.arange(200)), taken=taken,
                                                kv_out=m if in_place else None)
    n = np.maximum(new, 0).astype(np.int64)
    assert np.array_equal(cu.cpu().numpy(), np.minimum(np.concatenate([[0], np.cumsum(n)]), 2 ** 31 - 1))
    assert np.array_equal(kv_out.cpu().numpy(), np.minimum(np.maximum(kv, 0).astype(np.int64) + n, 2 ** 31 - 1))
    assert (buf[0] == -9).all() and (buf[-1] == -9).all() and taken.item() == 2 ** 31 - 1
    assert (slots < 200 * 16).all() and (positions >= 0).all()


def test_kv_out_may_not_be_new_lens(gpu):
    from chestnut import kernels as K
    n = i32([1, 2])
    with pytest.raises(ValueError, match='kv_out must not be new_lens'):
        K.cache_maps(n, i32([0, 0]), i32([[0], [1]]), 16, 3, kv_out=n)


def test_maps_norms_and_axes_replay(gpu):
    """Captured with padded rows; lengths, positions and rows change between the replays, beside eager calls."""
    from chestnut import kernels as K
    B, T, H, kv, hd, page = 6, 1500, 4, 2, 64, 16                     # (over 1024 rows and in place: two launches)
    r = np.random.default_rng(9)
    f, axes = K.rope_frequencies(64)[0], K.rope_axes([16, 8, 8])
    free = i32(r.permutation(2000))
    new, kvl, x = i32([1] * B), i32([0] * B), rows(1, T, H + 2 * kv, hd, 'bf16')
    table, taken = torch.full((B, 200), -1, dtype=torch.int32, device='cuda'), i32([0])
    y = torch.empty(T, H + kv, hd, dtype=torch.bfloat16, device='cuda')

    def step(kvl, table, taken):
        cu, k, pos, slots = K.cache_maps(new, kvl, table, page, T, free_pages=free, taken=taken, kv_out=kvl)
        at = torch.stack([pos, pos // 5, pos % 5])
        a, b = K.norm_rope(x[:, :H], x[:, H:H + kv], None, None, at, f, axes=axes)
        return cu, pos, slots, a, b, K.rope(x[:, :H + kv], at, f, interleaved=True, axes=axes, out=y)
    mine = [t.clone() for t in (kvl, table, taken)]
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            got = step(kvl, table, taken)
    torch.cuda.synchronize()
    for lens in ([1] * 6, [250] * 6, [0, 0, 900, 1, 0, 3], [3, 1, 4, 1, 5, 9], [0] * 6):
        new.copy_(i32(lens))
        x.copy_(rows(sum(lens) + 3, T, H + 2 * kv, hd, 'bf16'))
        g.replay()
        out = [t.clone() for t in got]
        want = step(*mine)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(out, want)), lens
        assert torch.equal(kvl, mine[0]) and torch.equal(table, mine[1]) and torch.equal(taken, mine[2])


def test_cache_maps_on_two_streams_with_workspaces_of_their_own(gpu):
    from chestnut import kernels as K
    sets, want = [], []
    for i in range(2):
        new, kv, table, free = batch(20 + i, 900, 30, 300, 16)
        sets.append((new, kv, table, free))
        want.append(O.cache_maps(new, kv, table, 16, 30000, free, 0))
    ws = [torch.empty(1024, device='cuda') for _ in sets]
    dev = [(i32(n), [i32(k) for _ in range(10)], [i32(t) for _ in range(10)], i32(f), [i32([0]) for _ in range(10)]) for n, k, t, f in sets]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], [[], []]
    for j in range(10):
        for i in range(2):
            n, k, t, f, a = dev[i]
            with torch.cuda.stream(streams[i]):
                got[i].append(K.cache_maps(n, k[j], t[j], 16, 30000, free_pages=f, taken=a[j], kv_out=k[j], workspace=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for j in range(10):
            for g, w in zip(got[i][j] + (dev[i][2][j],), want[i]):
                assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1))


def held_batches():
    most = 2 ** 31 - 1
    r = np.random.default_rng(31)
    yield 'a sum that is held', [most], [100]
    yield 'between others', [5, most, 7], [3, 100, 9]
    yield 'behind a history that is held', [4, 10, 30, most], [most - 4, most, 50, 33]
    yield 'none and fewer', [-5, 0, 3, -most - 1, 1500, 20], [-1, 40, -most - 1, 9, -7, most - 10]
    new, kv = r.integers(-3, 4, 4000), r.integers(-3, 60, 4000)
    at = r.integers(0, 4000, 300)
    kv[at] = r.integers(-2 ** 31, 2 ** 31, 300)
    yield 'many', new, kv
    new = new.copy()
    new[2000:] = r.integers(-2 ** 31, 2 ** 31, 2000)
    yield 'many, past what is held', new, kv
    yield 'more than one launch takes', np.concatenate([new[:2000], new]), np.concatenate([kv[:2000], kv])


@pytest.mark.parametrize('what,new,kv', held_batches(), ids=[x[0] for x in held_batches()])
@pytest.mark.parametrize('listed', [False, True])
@pytest.mark.parametrize('taken', [-4, 2])
def test_both_forms_of_cache_maps(gpu, what, new, kv, listed, taken):
    """One launch and two answer alike, also where a sum or a place is held at 2^31 - 1."""
    from chestnut import kernels as K
    B, page, width, T = len(new), 16, 12, 2600
    r = np.random.default_rng(32)
    table = r.integers(-1, 1 << 20, (B, width))
    free = r.integers(-1, 1 << 20, 900) if listed else None
    want = O.cache_maps_of_any_lengths(new, kv, table, page, T, free, taken)
    for in_place in (False, True):
        assert (K.cache_maps_workspace(B, T, in_place) > 0) == (in_place or B > 4096)
        t, m = i32(table), i32(kv)
        args = dict(free_pages=i32(free), taken=i32([taken])) if listed else {}
        if listed and not in_place:
            args['taken_out'] = i32([77])
        got = K.cache_maps(i32(new), m, t, page, T, kv_out=m if in_place else None, **args)
        for x, w, name in zip(got + (t,), want, 'cu kv positions slots table'.split()):
            x = x.cpu().numpy()
            assert np.array_equal(x, w), f'{name}, in place {in_place}: first {np.argwhere(x != w)[0]}'
        if listed:
            assert args['taken' if in_place else 'taken_out'].item() == want[5]


def test_cache_maps_in_a_workspace_that_is_kept(gpu):
    """Of the bytes asked for and no more, whatever stands in them; two streams, one each."""
    from chestnut import kernels as K
    new, kv, table, free = batch(33, 900, 30, 300, 16)
    want = O.cache_maps(new, kv, table, 16, 30000, free, 0)
    nb = K.cache_maps_workspace(900, 30000, True)
    assert nb % 4 == 0 and nb > 0
    buf = [torch.full((nb // 4 + 2,), f, device='cuda') for f in (float('nan'), 1e30)]
    dev = [[(i32(new), i32(kv), i32(table), i32(free), i32([0])) for _ in range(5)] for _ in buf]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in buf], [[], []]
    for j in range(5):
        for i in range(2):
            n, k, t, f, a = dev[i][j]
            with torch.cuda.stream(streams[i]):
                got[i].append(K.cache_maps(n, k, t, 16, 30000, free_pages=f, taken=a, kv_out=k, workspace=buf[i][1:nb // 4 + 1]))
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.isnan(buf[i][[0, -1]]).all() if i == 0 else (buf[i][[0, -1]] == 1e30).all()
        for j in range(5):
            for g, w in zip(got[i][j] + (dev[i][j][2], dev[i][j][4]), want):
                assert np.array_equal(g.cpu().numpy().reshape(-1), np.asarray(w).reshape(-1))


@pytest.mark.parametrize('hd', [128, 96])
def test_norms_and_axes_where_offsets_pass_32_bits(gpu, hd):
    """Rows behind the first 2^32 elements: as a call on these rows alone gives them."""
    from chestnut import kernels as K
    H, kv = 40, 8
    T = 2 ** 32 // ((H + kv) * hd) + 300
    x = torch.zeros(T, H + kv, hd, dtype=torch.bfloat16, device='cuda')
    assert x[-200:].storage_offset() > 2 ** 32
    x[-200:] = rows(1, 200, H + kv, hd, 'bf16')
    last = x[-200:].clone()
    pos = torch.zeros(3, T, dtype=torch.int32, device='cuda')
    pos[:, -200:] = i32(np.random.default_rng(2).integers(0, 5000, (3, 200)))
    f, axes = K.rope_frequencies(48)[0], K.rope_axes([8, 8, 8])
    w = torch.rand(hd, device='cuda').bfloat16()
    at = pos[:, -200:].contiguous()
    want = K.norm_rope(last[:, :H], last[:, H:], w, w, at, f, axes=axes)
    turned = K.rope(last, at, f, axes=axes)
    y = K.rope(x, pos, f, axes=axes, out=torch.empty_like(x))
    assert torch.equal(y[-200:], turned) and not y[:1000].any()
    q, k = K.norm_rope(x[:, :H], x[:, H:], w, w, pos, f, axes=axes, q_out=y[:, :H], k_out=y[:, H:])
    assert torch.equal(q[-200:], want[0]) and torch.equal(k[-200:], want[1]) and not y[:1000].any()

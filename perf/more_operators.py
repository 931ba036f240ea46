"""The measured operators around a step over the token cache: the step's maps built on the device,
rotary positions of several axes, head norms with the rotation in the same pass, attention
through a sliding window, and attention of streams that share their first pages.

Kinds of case:
  maps    chestnut.kernels.cache_maps        offsets, positions, slots and new pages of a batch from its requests' lengths
  axes    chestnut.kernels.rope              rotary positions whose pairs belong to several axes (time, row, column)
  norm    chestnut.kernels.norm_rope         RMS norm of every Q and K head and the rotation, one pass
  window  chestnut.kernels.attention_paged, attention_varlen with window and sinks
  shared  chestnut.kernels.attention_paged with shared: groups of sequences whose first pages are the same

Heads, widths and lengths are those of the package's model specs (16 heads of 128 and 512
tokens a frame, 8 of 64 and 256 tokens; 24 past frames), K/V heads shared by groups of query
heads where a cache of many streams has to be small.
"""
import math
import os
import sys

import torch

own = False
_K = None


def _kernels():
    """The package's kernels, imported on first use (only the framework's side needs them)."""
    global _K
    if _K is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                        'chestnut-on-pc_amd'))
        from chestnut import kernels
        _K = kernels
    return _K


# ------------------------------------------------------------------ the cases --
def listed():
    return [
        # One new token of each of 32 streams, a page more for those whose last one is full: latency.
        dict(name='maps_step', kind='maps', B=32, longest=1, spare=0, history=32000, page=32),
        # Prompts and chunks of 700 requests at once, padded rows behind them: every page is taken here.
        dict(name='maps_prompts', kind='maps', B=700, longest=512, spare=1000, history=4096, page=64),
        # One frame of the small model: Q and K heads of 256 tokens, a pair's axis time, row or column.
        dict(name='axes_frame', kind='axes', T=256, heads=8, kv=8, hd=64, sections='8,12,12', turns=False, dtype='f16',
             interleaved=False, base=1e4, far=4096),
        # 24 frames of 512 tokens, the axes by turns along the pairs, neighbouring elements.
        dict(name='axes_frames', kind='axes', T=12288, heads=16, kv=4, hd=128, sections='16,24,24', turns=True, dtype='bf16',
             interleaved=True, base=5e5, far=1000000),
        # One new token of each of 32 streams, Q and K heads of a fused projection: latency.
        dict(name='norm_step', kind='norm', T=32, heads=16, kv=4, hd=128, rot=128, sections='', dtype='bf16', interleaved=False,
             base=5e5, far=32000),
        # 24 frames of the wide model, half of each head rotated, by three axes: bandwidth.
        dict(name='norm_frames', kind='norm', T=12288, heads=16, kv=16, hd=128, rot=64, sections='16,8,8', dtype='bf16',
             interleaved=False, base=1e4, far=100000),
        # One token of one stream of the small model, two frames of its 24 seen: latency.
        dict(name='window_one', kind='window', q='1', kv_len='6144', heads=8, kv=8, hd=64, page=64, dtype='f16',
             cache='f16', window=512, sinks=4),
        # One token of each of 32 streams, ragged histories in e4m3, grouped heads, eight frames seen.
        dict(name='window_streams', kind='window', q=','.join(['1'] * 32),
             kv_len=','.join(str(1025 + (i * 7919) % 31744) for i in range(32)), heads=16, kv=4, hd=128, page=32,
             dtype='bf16', cache='e4m3', window=4096, sinks=16),
        # The largest: long ragged prompts through a window, over their own rows.
        dict(name='window_prompts', kind='window', q='9001,5120,2263', kv_len='', heads=16, kv=4, hd=128, page=0,
             dtype='bf16', cache='', window=2048, sinks=4),
        # A few tokens of the small model over the frames that they share.
        dict(name='shared_few', kind='shared', groups='6', common='6144', q=','.join(['1'] * 6), own_len='1,64,100,7,300,129',
             heads=8, kv=8, hd=64, page=64, dtype='f16', cache='f16'),
        # 64 streams in two groups, one token each over a long common history in e4m3 and a ragged one of their own.
        dict(name='shared_streams', kind='shared', groups='40,24', common='24576,12800', q=','.join(['1'] * 64),
             own_len=','.join(str(1 + (i * 197) % 1500) for i in range(64)), heads=16, kv=4, hd=128, page=32, dtype='bf16',
             cache='e4m3'),
        # Chunks of several frames each over the frames before, which they share.
        dict(name='shared_chunks', kind='shared', groups='6', common='12800', q='512,77,1,200,333,512',
             own_len='512,600,1,200,1500,512', heads=16, kv=4, hd=128, page=64, dtype='f16', cache='f16'),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _split(rng, n, parts):
    """n pairs over `parts` axes, one at least for each."""
    cuts = sorted(rng.sample(range(1, n), parts - 1))
    return ','.join(str(b - a) for a, b in zip([0] + cuts, cuts + [n]))


def draw(rng):
    kind = rng.choice(['maps', 'axes', 'norm', 'window', 'window', 'shared', 'shared'])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8] if kv < 8 else [1, 2])
    dtype = rng.choice(['f16', 'bf16'])
    cache = rng.choice(['e4m3', dtype])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == 'maps':
        B = _log_int(rng, 1, 1000)
        return dict(kind=kind, B=B, longest=rng.choice([1, 1, _log_int(rng, 2, 512)]), spare=rng.choice([0, _log_int(rng, 1, 500)]),
                    history=_log_int(rng, 1, 4000000 // B), page=page)
    if kind == 'axes':
        rot = rng.choice([hd, hd // 2])
        return dict(kind=kind, T=_log_int(rng, 1, 12288), heads=heads, kv=kv, hd=hd, sections=_split(rng, rot // 2, rng.choice([2, 3, 3, 4])),
                    turns=rng.random() < 0.5, dtype=dtype, interleaved=rng.random() < 0.5, base=rng.choice([1e4, 5e5]),
                    far=_log_int(rng, 100, 1000000))
    if kind == 'norm':
        rot = rng.choice([hd, hd // 2])
        return dict(kind=kind, T=_log_int(rng, 1, 12288), heads=heads, kv=kv, hd=hd, rot=rot,
                    sections=rng.choice(['', _split(rng, rot // 2, 3)]), dtype=dtype, interleaved=rng.random() < 0.5,
                    base=rng.choice([1e4, 5e5]), far=_log_int(rng, 100, 1000000))
    if kind == 'window':
        window, sinks = _log_int(rng, 16, 4096), rng.choice([0, 1, 4, _log_int(rng, 2, 128)])
        form = rng.random()
        if form < 0.4:     # single tokens
            n = _log_int(rng, 1, 48)
            q = [1] * n
            k = [_log_int(rng, 1, 16384) for _ in range(n)]
        elif form < 0.7:   # chunks
            n = rng.randint(1, 6)
            q = [_log_int(rng, 1, 512) for _ in range(n)]
            k = [x + rng.choice([0, _log_int(rng, 1, 8000)]) for x in q]
        else:              # prompts over their own rows
            n = _log_int(rng, 1, 24)
            q, k = [_log_int(rng, 1, 4096 if n < 5 else 1024) for _ in range(n)], []
        return dict(kind=kind, q=','.join(map(str, q)), kv_len=','.join(map(str, k)), heads=heads, kv=kv, hd=hd,
                    page=page if k else 0, dtype=dtype, cache=cache if k else '', window=window, sinks=sinks)
    groups = [_log_int(rng, 1, 24) for _ in range(rng.choice([1, 1, 2, 3]))]
    n = sum(groups)
    most = 1 if rng.random() < 0.6 else 256
    q = [_log_int(rng, 1, most) for _ in range(n)]
    return dict(kind=kind, groups=','.join(map(str, groups)), common=','.join(str(page * _log_int(rng, 1, 16384 // page)) for _ in groups),
                q=','.join(map(str, q)), own_len=','.join(str(x + rng.choice([0, _log_int(rng, 1, 1500)])) for x in q),
                heads=heads, kv=kv, hd=hd, page=page, dtype=dtype, cache=cache)


# ------------------------------------------------------------------ the inputs --
DT = {'f16': torch.float16, 'bf16': torch.bfloat16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu
EPS = 1e-6


def _ints(text):
    return [int(x) for x in text.split(',')] if text else []


def _i32(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def _cu(lens):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).cuda()


def _rows(g, T, heads, hd, dtype):
    """Activations as a projection leaves them: normal, a few channels of a head several times larger."""
    x = torch.randn(T, heads, hd, generator=g, device='cuda')
    big = torch.rand(heads, hd, generator=g, device='cuda') < 0.03
    return (x * (1.0 + 2.0 * big)).to(DT[dtype])


def _pages(g, n, kv, page, hd, c):
    """A cache with a history in it: (k_pages, v_pages, k_scale, v_scale)."""
    if c['cache'] != 'e4m3':
        k, v = (_rows(g, n * page, kv, hd, c['dtype']).view(n, page, kv, hd).permute(0, 2, 1, 3).contiguous() for _ in 'kv')
        return k, v, None, None
    out = []
    for _ in 'kv':
        x = _rows(g, n * page, kv, hd, c['dtype']).float().view(n, page, kv, hd).permute(0, 2, 1, 3)
        # the least power of two, 2^(byte - 127), with amax <= 448 of it
        bits = x.abs().amax(-1).view(torch.int32)
        byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=1)
        inv = ((254 - byte) << 23).view(torch.float32)
        out.append(((x * inv[..., None]).contiguous().to(E4M3), byte.to(torch.uint8).contiguous().view(E8M0)))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _axes(sections, turns):
    """Every pair's axis: the axes' sections one after the other, or an axis after the other by turns."""
    if not turns:
        return [a for a, n in enumerate(sections) for _ in range(n)]
    left, out = list(sections), []
    while any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return out


def _positions(g, c, n_axes):
    """Positions of a clip's tokens: the first axis runs on, the others name places in a frame."""
    T = c['T']
    if n_axes < 2:
        return torch.randint(0, c['far'], (T,), generator=g, device='cuda', dtype=torch.int32)
    first = torch.randint(0, c['far'], (1, T), generator=g, device='cuda', dtype=torch.int32)
    rest = torch.randint(0, 64, (n_axes - 1, T), generator=g, device='cuda', dtype=torch.int32)
    return torch.cat((first, rest)).contiguous()


def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda').manual_seed(int(seed) * 1000003 + 17)
    s = dict(case=c)
    if c['kind'] == 'maps':
        B, page = c['B'], c['page']
        s['new'] = torch.randint(1, c['longest'] + 1, (B,), generator=g, device='cuda', dtype=torch.int32)
        s['kv'] = torch.randint(0, c['history'] + 1, (B,), generator=g, device='cuda', dtype=torch.int32)
        have = (s['kv'] + page - 1) // page
        width = -(-(c['history'] + c['longest']) // page)
        n = B * width
        order = torch.randperm(n, generator=g, device='cuda').to(torch.int32)
        held = order[:B * width].view(B, width)
        cols = torch.arange(width, device='cuda', dtype=torch.int32)
        s['table'] = torch.where(cols < have[:, None], held, torch.full_like(held, -1))
        free = held[cols >= have[:, None]]
        s['free'] = torch.cat((torch.full((5,), -7, dtype=torch.int32, device='cuda'), free))   # five are taken already
        s['taken'] = _i32([5])
        s['taken_out'] = torch.empty_like(s['taken'])
        s['tokens'] = B * c['longest'] + c['spare']
    elif c['kind'] in ('axes', 'norm'):
        H, hd, T, kv = c['heads'], c['hd'], c['T'], c['kv']
        sections = _ints(c['sections'])
        rot = 2 * sum(sections) if c['kind'] == 'axes' else c['rot']
        s['qkv'] = _rows(g, T, H + 2 * kv, hd, c['dtype'])
        s['positions'] = _positions(g, c, len(sections))
        s['axes'] = _i32(_axes(sections, c.get('turns', False))) if sections else None
        s['inv_freq'] = torch.pow(torch.tensor(c['base'], dtype=torch.float64),
                                  -torch.arange(0, rot, 2, dtype=torch.float64) / rot).cuda()
        if c['kind'] == 'axes':
            s['x'] = s['qkv'][:, :H + kv]             # the Q and K heads of the fused projection
            s['out'] = torch.empty(T, H + kv, hd, dtype=DT[c['dtype']], device='cuda')
        else:
            s['q'], s['k'] = s['qkv'][:, :H], s['qkv'][:, H:H + kv]
            s['q_out'], s['k_out'] = (torch.empty(T, h, hd, dtype=DT[c['dtype']], device='cuda') for h in (H, kv))
            s['wq'], s['wk'] = ((1.0 + 0.2 * torch.randn(hd, generator=g, device='cuda')).to(DT[c['dtype']]) for _ in 'qk')
    elif c['kind'] == 'window':
        q, k = _ints(c['q']), _ints(c['kv_len'])
        s['q'] = _rows(g, sum(q), c['heads'], c['hd'], c['dtype'])
        s['cu_q'], s['q_lens'], s['k_lens'] = _cu(q), q, k or q
        if k:
            need = [-(-n // c['page']) for n in k]
            perm = torch.randperm(sum(need), generator=g, device='cuda').to(torch.int32)
            s['table'] = torch.full((len(k), max(need)), -1, dtype=torch.int32, device='cuda')
            at = 0
            for b, n in enumerate(need):
                s['table'][b, :n] = perm[at:at + n]
                at += n
            s['pages'] = _pages(g, sum(need), c['kv'], c['page'], c['hd'], c)
            s['kv_lens'] = _i32(k)
        else:
            s['k'], s['v'] = (_rows(g, sum(q), c['kv'], c['hd'], c['dtype']) for _ in 'kv')
    else:
        groups, common, q, mine = (_ints(c[x]) for x in ('groups', 'common', 'q', 'own_len'))
        page = c['page']
        lens = [common[i] + m for i, m in zip((i for i, n in enumerate(groups) for _ in range(n)), mine)]
        firsts, owns = [n // page for n in common], [-(-m // page) for m in mine]
        total = sum(firsts) + sum(owns)
        perm = torch.randperm(total, generator=g, device='cuda').to(torch.int32)
        s['table'] = torch.full((len(q), max(-(-n // page) for n in lens)), -1, dtype=torch.int32, device='cuda')
        at, b = 0, 0
        for i, n in enumerate(groups):
            pages = perm[at:at + firsts[i]]
            at += firsts[i]
            for b in range(b, b + n):
                s['table'][b, :firsts[i]] = pages
                s['table'][b, firsts[i]:firsts[i] + owns[b]] = perm[at:at + owns[b]]
                at += owns[b]
            b += 1
        s['pages'] = _pages(g, total, c['kv'], page, c['hd'], c)
        s['q'] = _rows(g, sum(q), c['heads'], c['hd'], c['dtype'])
        s['cu_q'], s['kv_lens'], s['q_lens'], s['k_lens'] = _cu(q), _i32(lens), q, lens
        s['shared'] = (_cu(groups), _i32(common))
    return s


# ------------------------------------------------------------- the plain forms --
def _maps(s, c):
    new, old, page, T, width = s['new'], s['kv'], c['page'], s['tokens'], s['table'].shape[1]
    kv = old + new
    cu = torch.zeros(c['B'] + 1, dtype=torch.int32, device='cuda')
    cu[1:] = torch.cumsum(new, 0)
    have, need = (old + page - 1) // page, (kv + page - 1) // page
    ends = torch.cumsum(need - have, 0).to(torch.int32)
    first = s['taken'] + ends - (need - have)
    col = torch.arange(width, dtype=torch.int32, device='cuda')
    at = first[:, None] + col - have[:, None]
    fresh = (col >= have[:, None]) & (col < need[:, None])
    page_of = torch.where(at < s['free'].shape[0], s['free'][at.clamp(0, s['free'].shape[0] - 1).long()], torch.full_like(at, -1))
    s['table'].copy_(torch.where(fresh, page_of, s['table']))
    s['taken_out'].copy_(s['taken'] + ends[-1])
    t = torch.arange(T, dtype=torch.int32, device='cuda')
    b = torch.searchsorted(cu[1:], t, right=True).clamp(max=c['B'] - 1)
    place = old[b] + t - cu[b]
    mine = t < cu[-1]
    col = (place // page).clamp(max=width - 1).long()
    held = s['table'][b, col]
    none = torch.full_like(t, -1)
    slots = torch.where(mine & (held >= 0), held * page + place % page, none)
    positions = torch.where(mine, place, torch.zeros_like(t))
    return cu, kv, positions, slots, s['table'], s['taken_out']


def _turned(x, positions, inv_freq, axes, interleaved):
    """x in 32 bits [T, heads, hd], its first 2 * len(inv_freq) elements turned."""
    r = 2 * inv_freq.shape[0]
    p = positions.double()[:, None] if axes is None else positions.double()[axes.long()].T
    a = (p * inv_freq)[:, None]
    cos, sin = a.cos().float(), a.sin().float()
    x0, x1 = (x[..., 0:r:2], x[..., 1:r:2]) if interleaved else (x[..., :r // 2], x[..., r // 2:r])
    y0, y1 = x0 * cos - x1 * sin, x1 * cos + x0 * sin
    y = torch.stack((y0, y1), -1).flatten(-2) if interleaved else torch.cat((y0, y1), -1)
    return torch.cat((y, x[..., r:]), -1)


def _values(pages, scale):
    """What pages hold, in 32 bits."""
    if scale is None:
        return pages.float()
    return pages.float() * (scale.view(torch.uint8).int() << 23).view(torch.float32)[..., None]


def _gather(pages, scale, table):
    """The pages of every row of a table in order, [rows, Hkv, width * page, hd] in 32 bits."""
    t = table.clamp(min=0).long()
    x = _values(pages.view(torch.uint8)[t].view(E4M3) if scale is not None else pages[t],
                scale.view(torch.uint8)[t].view(E8M0) if scale is not None else None)
    B, n, H, page, hd = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, n * page, hd)


def _padded(q, cu_q, max_q, Hkv):
    """Packed queries as rows of their K/V head: [B, Hkv, G * max_q, hd] in 32 bits."""
    T, Hq, hd = q.shape
    B, G = cu_q.shape[0] - 1, Hq // Hkv
    rows = (cu_q[:-1, None] + torch.arange(max_q, device='cuda')).clamp(max=T - 1).long()
    return q[rows].float().view(B, max_q, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * max_q, hd)


def _packed(o, cu_q, T, Hq, max_q):
    """The rows of _padded as packed queries."""
    B, Hkv, _, hd = o.shape
    o = o.view(B, Hkv, Hq // Hkv, max_q, hd).permute(0, 3, 1, 2, 4).reshape(B, max_q, Hq, hd)
    t = torch.arange(T, device='cuda', dtype=torch.int32)
    b = torch.searchsorted(cu_q[1:], t, right=True)
    return o[b, (t - cu_q[b]).long()]


def _window(s, c):
    kv = c['kv']
    max_q = max(s['q_lens'])
    n = s['cu_q'][1:] - s['cu_q'][:-1]
    if c['kv_len']:
        kp, vp, ks, vs = s['pages']
        k, v = _gather(kp, ks, s['table']), _gather(vp, vs, s['table'])
        m = s['kv_lens']
    else:
        rows = (s['cu_q'][:-1, None] + torch.arange(max_q, device='cuda')).clamp(max=s['q'].shape[0] - 1).long()
        k, v = (t[rows].float().permute(0, 2, 1, 3).contiguous() for t in (s['k'], s['v']))
        m = n
    B, L = k.shape[0], k.shape[2]
    w = torch.matmul(_padded(s['q'], s['cu_q'], max_q, kv) / math.sqrt(c['hd']), k.transpose(-1, -2).contiguous())
    w = w.view(B, kv, -1, max_q, L)
    place = (m - n)[:, None] + torch.arange(max_q, device='cuda')          # of each query
    j = torch.arange(L, device='cuda')
    see = (j <= place[..., None]) & ((j > place[..., None] - c['window']) | (j < c['sinks'])) & (j < m[:, None, None])
    w.masked_fill_(~see[:, None, None], -math.inf)
    top = w.amax(-1, keepdim=True)
    w.sub_(torch.where(top == -math.inf, torch.zeros_like(top), top)).exp_()
    l = w.sum(-1, keepdim=True).view(B, kv, -1, 1)
    o = torch.matmul(w.view(B, kv, -1, L), v)
    o = torch.where(l > 0, o / l, torch.zeros_like(o))
    return _packed(o, s['cu_q'], s['q'].shape[0], c['heads'], max_q).to(s['q'].dtype)


def _shared(s, c):
    """The common keys of a group against all its queries at once, a sequence's own ones against its own."""
    kv, page, out = c['kv'], c['page'], []
    kp, vp, ks, vs = s['pages']
    b0 = at = 0
    for n, P in zip(_ints(c['groups']), _ints(c['common'])):
        ql, ml = s['q_lens'][b0:b0 + n], _ints(c['own_len'])[b0:b0 + n]
        max_q, width = max(ql), max(-(-m // page) for m in ml)
        q = s['q'][at:at + sum(ql)]
        cu = s['cu_q'][b0:b0 + n + 1] - s['cu_q'][b0]
        x = _padded(q, cu, max_q, kv) / math.sqrt(c['hd'])                  # [n, kv, rows, hd]
        rows = x.shape[2]
        table = s['table'][b0:b0 + n]
        ck, cv = (_gather(p, f, table[:1, :P // page])[0] for p, f in ((kp, ks), (vp, vs)))
        own = table[:, P // page:P // page + width]
        k, v = _gather(kp, ks, own), _gather(vp, vs, own)
        w0 = torch.matmul(x.transpose(0, 1).reshape(kv, n * rows, -1), ck.transpose(-1, -2).contiguous())
        w1 = torch.matmul(x, k.transpose(-1, -2).contiguous()).view(n, kv, -1, max_q, width * page)
        m = s['kv_lens'][b0:b0 + n] - P
        last = (m - (cu[1:] - cu[:-1]))[:, None] + torch.arange(max_q, device='cuda')
        j = torch.arange(width * page, device='cuda')
        see = (j <= last[..., None]) & (j < m[:, None, None])
        w1.masked_fill_(~see[:, None, None], -math.inf)
        w1 = w1.view(n, kv, rows, -1)
        top = torch.maximum(w0.amax(-1).view(kv, n, rows).transpose(0, 1), w1.amax(-1))[..., None]
        w1.sub_(top).exp_()
        w0.sub_(top.transpose(0, 1).reshape(kv, n * rows, 1)).exp_()
        l = w0.sum(-1).view(kv, n, rows).transpose(0, 1) + w1.sum(-1)
        o = torch.matmul(w0, cv).view(kv, n, rows, -1).transpose(0, 1) + torch.matmul(w1, v)
        out.append(_packed((o / l[..., None]).contiguous(), cu, q.shape[0], c['heads'], max_q))
        b0 += n
        at += sum(ql)
    return torch.cat(out).to(s['q'].dtype)


def run(state):
    s, c = state, state['case']
    if c['kind'] == 'maps':
        if not own:
            return _maps(s, c)
        cu, kv, positions, slots = _kernels().cache_maps(s['new'], s['kv'], s['table'], c['page'], s['tokens'], free_pages=s['free'],
                                                         taken=s['taken'], taken_out=s['taken_out'])
        return cu, kv, positions, slots, s['table'], s['taken_out']
    if c['kind'] == 'axes':
        if own:
            return _kernels().rope(s['x'], s['positions'], s['inv_freq'], interleaved=c['interleaved'], axes=s['axes'], out=s['out'])
        return _turned(s['x'].float(), s['positions'], s['inv_freq'], s['axes'], c['interleaved']).to(s['x'].dtype)
    if c['kind'] == 'norm':
        if own:
            return _kernels().norm_rope(s['q'], s['k'], s['wq'], s['wk'], s['positions'], s['inv_freq'], eps=EPS, axes=s['axes'],
                                        interleaved=c['interleaved'], q_out=s['q_out'], k_out=s['k_out'])
        out = []
        for x, w in ((s['q'].float(), s['wq']), (s['k'].float(), s['wk'])):
            y = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * w.float()
            out.append(_turned(y, s['positions'], s['inv_freq'], s['axes'], c['interleaved']).to(s['q'].dtype))
        return tuple(out)
    if c['kind'] == 'window':
        if not own:
            return _window(s, c)
        if not c['kv_len']:
            return _kernels().attention_varlen(s['q'], s['k'], s['v'], s['cu_q'], window=c['window'], sinks=c['sinks'])
        kp, vp, ks, vs = s['pages']
        return _kernels().attention_paged(s['q'], kp, vp, s['table'], s['cu_q'], s['kv_lens'], k_scale=ks, v_scale=vs,
                                          window=c['window'], sinks=c['sinks'])
    if not own:
        return _shared(s, c)
    kp, vp, ks, vs = s['pages']
    return _kernels().attention_paged(s['q'], kp, vp, s['table'], s['cu_q'], s['kv_lens'], k_scale=ks, v_scale=vs,
                                      shared=s['shared'])


# ------------------------------------------------------------------- the work --
def _seen(q, k, window, sinks):
    """(query, key) pairs seen and keys that some query sees: the last q of k places are the queries'."""
    pairs = 0
    for i in range(k - q, k):
        if i >= 0:
            lo = max(0, i + 1 - window)
            pairs += i + 1 - lo + min(lo, sinks)
    lo = max(0, k - q + 1 - window)
    return pairs, k - lo + min(lo, sinks)


def work(case):
    c, e = case, 2
    if c['kind'] == 'maps':
        # lengths in and out, offsets; a position and a slot a token; a new page in the list and in the table
        T = c['B'] * c['longest'] + c['spare']
        fresh = c['B'] * (c['longest'] + 1) // (2 * c['page'])
        return dict(bytes=4 * (4 * c['B'] + 1 + 2 * T + 2 * fresh), flops=0)
    if c['kind'] in ('axes', 'norm'):
        rot = 2 * sum(_ints(c['sections'])) if c['kind'] == 'axes' else c['rot']
        n = c['T'] * (c['heads'] + c['kv'])
        return dict(bytes=2 * e * n * c['hd'] + 4 * c['T'] * max(1, len(_ints(c['sections']))),
                    flops=n * (3 * rot + (4 * c['hd'] if c['kind'] == 'norm' else 0)))
    w = 1 if c['cache'] == 'e4m3' else 2
    row = 2 * c['kv'] * (c['hd'] * w + (w == 1))                            # a key's K and V
    q = _ints(c['q'])
    if c['kind'] == 'window':
        seen = [_seen(a, b, c['window'], c['sinks']) for a, b in zip(q, _ints(c['kv_len']) or q)]
        pairs, keys = sum(x[0] for x in seen), sum(x[1] for x in seen)
    else:
        groups, common, mine = (_ints(c[x]) for x in ('groups', 'common', 'own_len'))
        pairs, keys, b = 0, sum(common) + sum(mine), 0
        for n, P in zip(groups, common):
            pairs += sum(a * (P + m - a) + a * (a + 1) // 2 for a, m in zip(q[b:b + n], mine[b:b + n]))
            b += n
    return dict(bytes=2 * e * sum(q) * c['heads'] * c['hd'] + keys * row, flops=4 * c['hd'] * c['heads'] * pairs)


# ------------------------------------------------ the definitions, in 64 bits --
def _exact_maps(s, c):
    """Request by request, with whole numbers on the host."""
    new, old, free = (s[x].tolist() for x in ('new', 'kv', 'free'))
    table, page = s['table'].tolist(), c['page']
    taken = s['taken'].item()
    cu, kv, positions, slots = [0], [], [], []
    for b, (n, m) in enumerate(zip(new, old)):
        for col in range(-(-m // page), -(-(m + n) // page)):
            table[b][col] = free[taken] if taken < len(free) else -1
            taken += 1
        for at in range(m, m + n):
            positions.append(at)
            slots.append(table[b][at // page] * page + at % page if table[b][at // page] >= 0 else -1)
        cu.append(cu[-1] + n)
        kv.append(m + n)
    positions += [0] * (s['tokens'] - len(positions))
    slots += [-1] * (s['tokens'] - len(slots))
    return tuple(torch.tensor(x, dtype=torch.int64, device='cuda') for x in (cu, kv, positions, slots, table, [taken]))


def _exact_turn(x, s, c):
    """x f64 [T, heads, hd]: pairs as complex numbers, turned."""
    r = 2 * s['inv_freq'].shape[0]
    if s['axes'] is None:
        turn = s['positions'].double()[:, None] * s['inv_freq'][None]
    else:
        turn = torch.stack([s['positions'][a].double() * f for a, f in zip(s['axes'].tolist(), s['inv_freq'])], -1)
    turn = torch.remainder(turn, 2.0 * math.pi)
    z = torch.polar(torch.ones_like(turn), turn)[:, None]
    p = x[..., :r].unflatten(-1, (r // 2, 2) if c['interleaved'] else (2, r // 2))
    p = p if c['interleaved'] else p.transpose(-1, -2)
    y = torch.view_as_real(torch.complex(p[..., 0].contiguous(), p[..., 1].contiguous()) * z)
    x = x.clone()
    x[..., :r] = (y if c['interleaved'] else y.transpose(-1, -2)).flatten(-2)
    return x


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c['kind'] == 'maps':
        return _exact_maps(s, c)
    if c['kind'] == 'axes':
        return _exact_turn(s['x'].double(), s, c)
    if c['kind'] == 'norm':
        out = []
        for x, w in ((s['q'].double(), s['wq']), (s['k'].double(), s['wk'])):
            size = torch.sqrt(torch.linalg.vector_norm(x, dim=-1, keepdim=True) ** 2 / c['hd'] + EPS)
            out.append(_exact_turn(x / size * w.double(), s, c))
        return tuple(out)
    out, at, G = [], 0, c['heads'] // c['kv']
    if 'pages' in s:
        # a scale byte is the exponent of a power of two, 127 more than it is (in 64 bits: 1023 more)
        kx, vx = (p.double() if f is None else p.double() * ((f.view(torch.uint8).long() + 896) << 52).view(torch.float64)[..., None]
                  for p, f in zip(s['pages'][:2], s['pages'][2:]))
    for b, (n, m) in enumerate(zip(s['q_lens'], s['k_lens'])):
        q = s['q'][at:at + n].double()
        if 'pages' in s:
            t = s['table'][b, :-(-m // c['page'])].long()
            k, v = (x[t].permute(0, 2, 1, 3).flatten(0, 1)[:m] for x in (kx, vx))
        else:
            k, v = (s[x][at:at + n].double() for x in 'kv')
        far = (torch.arange(n, device='cuda') + m - n)[:, None] - torch.arange(m, device='cuda')[None]   # places back
        see = far >= 0
        if c['kind'] == 'window':
            see &= (far < c['window']) | (torch.arange(m, device='cuda') < c['sinks'])[None]
        o = torch.zeros_like(q)
        for h in range(c['heads']):
            w = (q[:, h] @ k[:, h // G].T) / math.sqrt(c['hd'])
            w = torch.where(see, w, torch.full_like(w, -math.inf))
            o[:, h] = torch.nan_to_num(torch.softmax(w, -1)) @ v[:, h // G]
        out.append(o)
        at += n
    return torch.cat(out)

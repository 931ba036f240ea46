"""The measured operators of the token cache: rotary positions, writing and reading a paged
(and quantised) cache, attention of a chunk of new tokens over it, and attention over whole
packed sequences.

Kinds of case:
  rope    chestnut.kernels.rope              rotary positions of the Q and K heads of a fused projection
  write   chestnut.kernels.cache_write       K and V rows into pages, e4m3 with a power-of-two scale a row or as they are
  read    chestnut.kernels.cache_read        the pages of packed sequences back to contiguous rows
  paged   chestnut.kernels.attention_paged   new tokens (one or a chunk) over the paged cache
  varlen  chestnut.kernels.attention_varlen  whole packed sequences

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
        # The smallest call: one new token of each of four streams, Q and K heads of the small model.
        dict(name='rope_step', kind='rope', T=4, heads=8, kv=8, hd=64, rot=64, dtype='f16', interleaved=False,
             base=1e4, factor=1.0, far=4096),
        # 24 frames of 512 tokens at once, half of each head rotated, neighbouring pairs, positions scaled.
        dict(name='rope_prompt', kind='rope', T=12288, heads=16, kv=4, hd=128, rot=64, dtype='bf16', interleaved=True,
             base=5e5, factor=8.0, far=1000000),
        # One new token of each of 32 streams into an e4m3 cache: latency.
        dict(name='write_step', kind='write', T=32, kv=4, hd=128, page=32, pages=2000, dtype='f16', cache='e4m3'),
        # 24 frames of the wide model into an e4m3 cache, quantised on the way: bandwidth.
        dict(name='write_frames', kind='write', T=12288, kv=16, hd=128, page=64, pages=256, dtype='bf16', cache='e4m3'),
        # A few short sequences of the small model from a cache that is not quantised.
        dict(name='read_short', kind='read', lens='300,1,77', kv=8, hd=64, page=16, dtype='f16', cache='f16'),
        # Many streams' histories read back from e4m3, ragged lengths.
        dict(name='read_streams', kind='read', lens='12288,6143,9000,12800,257,12031,8192,11111', kv=16, hd=128, page=64,
             dtype='f16', cache='e4m3'),
        # One token of one stream over 24 frames of 256 tokens: latency, few rows, a long axis.
        dict(name='step_one', kind='paged', q='1', kv_len='6144', heads=8, kv=8, hd=64, page=64, dtype='f16',
             cache='f16', causal=True),
        # One token of each of 32 streams, ragged long histories in e4m3, grouped heads: bandwidth.
        dict(name='step_streams', kind='paged', q=','.join(['1'] * 32),
             kv_len=','.join(str(1025 + (i * 7919) % 31744) for i in range(32)), heads=16, kv=4, hd=128, page=32,
             dtype='bf16', cache='e4m3', causal=True),
        # A frame's 512 tokens over 24 past frames and themselves, as the model's blocks attend (all of the frame).
        dict(name='frame_chunk', kind='paged', q='512', kv_len='12800', heads=16, kv=16, hd=128, page=64, dtype='f16',
             cache='f16', causal=False),
        # A serving batch in the middle of its prompts: ragged chunks and single tokens, e4m3.
        dict(name='mixed_chunks', kind='paged', q='1,200,1,333,17,64,1,511', heads=16, kv=4, hd=128, page=32,
             kv_len='900,2200,5001,333,4017,6000,77,8191', dtype='f16', cache='e4m3', causal=True),
        # Many short ragged sequences of the small model.
        dict(name='prompt_short', kind='varlen', q=','.join(str(1 + (i * 37) % 255) for i in range(40)), heads=8, kv=8,
             hd=64, dtype='f16', causal=True),
        # The largest: long ragged prompts, grouped heads, causal.
        dict(name='prompt_long', kind='varlen', q='9001,5120,2263', heads=16, kv=4, hd=128, dtype='bf16', causal=True),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(['rope', 'write', 'read', 'paged', 'paged', 'varlen', 'varlen'])
    hd = rng.choice([64, 128])
    kv = rng.choice([1, 2, 3, 4, 8])
    heads = kv * rng.choice([1, 2, 4, 5, 8] if kv < 8 else [1, 2])
    dtype = rng.choice(['f16', 'bf16'])
    cache = rng.choice(['e4m3', dtype])
    page = rng.choice([16, 32, 64, 128, 256])
    if kind == 'rope':
        return dict(kind=kind, T=_log_int(rng, 1, 12288), heads=heads, kv=kv, hd=hd, rot=rng.choice([hd, hd // 2, 16]),
                    dtype=dtype, interleaved=rng.random() < 0.5, base=rng.choice([1e4, 5e5]),
                    factor=rng.choice([1.0, 4.0, 8.0]), far=_log_int(rng, 20000, 1000000))
    if kind == 'write':
        T = _log_int(rng, 1, 12288)
        return dict(kind=kind, T=T, kv=kv, hd=hd, page=page, pages=-(-T // page) + _log_int(rng, 1, 200), dtype=dtype,
                    cache=cache)
    if kind == 'read':
        n = rng.randint(1, 8)
        return dict(kind=kind, lens=','.join(str(_log_int(rng, 1, 12800)) for _ in range(n)), kv=kv, hd=hd, page=page,
                    dtype=dtype, cache=cache)
    if kind == 'paged':
        if rng.random() < 0.5:   # single tokens
            n = _log_int(rng, 1, 48)
            q = [1] * n
            k = [_log_int(rng, 1, 16384) for _ in range(n)]
        else:                    # chunks
            n = rng.randint(1, 6)
            q = [_log_int(rng, 1, 512) for _ in range(n)]
            k = [x + rng.choice([0, _log_int(rng, 1, 8000)]) for x in q]
        return dict(kind=kind, q=','.join(map(str, q)), kv_len=','.join(map(str, k)), heads=heads, kv=kv, hd=hd,
                    page=page, dtype=dtype, cache=cache, causal=rng.random() < 0.7)
    n = _log_int(rng, 1, 24)
    return dict(kind=kind, q=','.join(str(_log_int(rng, 1, 4096 if n < 5 else 1024)) for _ in range(n)), heads=heads,
                kv=kv, hd=hd, dtype=dtype, causal=rng.random() < 0.8)


# ------------------------------------------------------------------ the inputs --
DT = {'f16': torch.float16, 'bf16': torch.bfloat16}
E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _ints(text):
    return [int(x) for x in text.split(',')]


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
        codes, byte = _quantise(_rows(g, n * page, kv, hd, c['dtype']))
        out.append((codes.view(n, page, kv, hd).permute(0, 2, 1, 3).contiguous().view(E4M3),
                    byte.view(n, page, kv).permute(0, 2, 1).contiguous().view(E8M0)))
    return out[0][0], out[1][0], out[0][1], out[1][1]


def _table(g, lens, page):
    """Every sequence's pages, in no order; entries behind a sequence's last page are -1."""
    need = [-(-n // page) for n in lens]
    total, width = sum(need), max(1, max(need))
    perm = torch.randperm(max(1, total), generator=g, device='cuda').to(torch.int32)
    t = torch.full((len(lens), width), -1, dtype=torch.int32, device='cuda')
    at = 0
    for b, n in enumerate(need):
        t[b, :n] = perm[at:at + n]
        at += n
    return t, max(1, total)


def _frequencies(c):
    """Inverse frequencies of the rotated pairs, positions scaled for a longer context by the base."""
    r = c['rot']
    base = c['base'] * c['factor'] ** (r / (r - 2.0))
    return torch.pow(torch.tensor(base, dtype=torch.float64),
                     -torch.arange(0, r, 2, dtype=torch.float64) / r).cuda(), 0.1 * math.log(c['factor']) + 1.0


def prepare(case, seed):
    c = case
    g = torch.Generator(device='cuda').manual_seed(int(seed) * 1000003 + 17)
    s = dict(case=c)
    if c['kind'] == 'rope':
        H, hd, T = c['heads'] + 2 * c['kv'], c['hd'], c['T']
        s['qkv'] = _rows(g, T, H, hd, c['dtype'])
        s['x'] = s['qkv'][:, :c['heads'] + c['kv']]     # the Q and K heads of the fused projection
        s['out'] = torch.empty(T, c['heads'] + c['kv'], hd, dtype=DT[c['dtype']], device='cuda')
        s['positions'] = torch.randint(0, c['far'], (T,), generator=g, device='cuda', dtype=torch.int32)
        s['inv_freq'], s['scale'] = _frequencies(c)
    elif c['kind'] == 'write':
        s['k'], s['v'] = (_rows(g, c['T'], c['kv'], c['hd'], c['dtype']) for _ in 'kv')
        s['pages'] = _pages(g, c['pages'], c['kv'], c['page'], c['hd'], c)
        s['slots'] = torch.randperm(c['pages'] * c['page'], generator=g, device='cuda')[:c['T']].to(torch.int32)
    elif c['kind'] == 'read':
        lens = _ints(c['lens'])
        s['table'], n = _table(g, lens, c['page'])
        s['pages'] = _pages(g, n, c['kv'], c['page'], c['hd'], c)
        s['cu'], s['tokens'] = _cu(lens), sum(lens)
    elif c['kind'] == 'paged':
        q, k = _ints(c['q']), _ints(c['kv_len'])
        s['q'] = _rows(g, sum(q), c['heads'], c['hd'], c['dtype'])
        s['table'], n = _table(g, k, c['page'])
        s['pages'] = _pages(g, n, c['kv'], c['page'], c['hd'], c)
        s['cu_q'], s['kv_lens'], s['max_q'] = _cu(q), _i32(k), max(q)
    else:
        q = _ints(c['q'])
        s['q'] = _rows(g, sum(q), c['heads'], c['hd'], c['dtype'])
        s['k'], s['v'] = (_rows(g, sum(q), c['kv'], c['hd'], c['dtype']) for _ in 'kv')
        s['cu_q'], s['max_q'] = _cu(q), max(q)
    return s


# ------------------------------------------------------------- the plain forms --
def _quantise(x):
    """Rows of x in e4m3 (as bytes) and each row's scale byte: the least power of two, 2^(byte - 127), with
    amax <= 448 of it.  Values are held to what their type still holds after a rounding to four bits."""
    top = 1.875 * 2.0 ** (15 if x.dtype == torch.float16 else 127)
    x = x.float().clamp(-top, top)
    bits = x.abs().amax(-1).view(torch.int32)
    byte = ((bits >> 23) - 8 + ((bits & 0x7FFFFF) > 0x600000)).clamp(min=1)
    inv = ((254 - byte) << 23).view(torch.float32)
    return (x * inv[..., None]).to(E4M3).view(torch.uint8), byte.to(torch.uint8)


def _values(pages, scale):
    """What pages hold, in 32 bits."""
    if scale is None:
        return pages.float()
    return pages.view(E4M3).float() * (scale.int() << 23).view(torch.float32)[..., None]


def _gather(pages, scale, table):
    """The pages of every sequence in order, [B, Hkv, width * page, hd] in 32 bits."""
    t = table.clamp(min=0).long()
    p = pages.view(torch.uint8)[t].view(E4M3) if scale is not None else pages[t]
    x = _values(p, scale.view(torch.uint8)[t] if scale is not None else None)
    B, n, H, page, hd = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(B, H, n * page, hd)


def _places(cu, T):
    """Sequence and place in it of each of T packed rows."""
    t = torch.arange(T, device='cuda', dtype=torch.int32)
    b = torch.searchsorted(cu[1:], t, right=True)
    return b, (t - cu[b]).long()


def _attention(q, k, v, cu_q, kv_lens, max_q, causal, scale):
    """q packed [T, Hq, hd]; k, v padded [B, Hkv, L, hd] in 32 bits."""
    T, Hq, hd = q.shape
    B, Hkv, L, _ = k.shape
    G = Hq // Hkv
    n = (cu_q[1:] - cu_q[:-1])[:, None]
    i = torch.arange(max_q, device='cuda')[None]
    rows = (cu_q[:-1, None] + i).clamp(max=T - 1).long()
    x = q[rows].float().view(B, max_q, Hkv, G, hd).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * max_q, hd)
    s = torch.matmul(x * scale, k.transpose(-1, -2).contiguous()).view(B, Hkv, G, max_q, L)
    last = (kv_lens[:, None] - n + i) if causal else (kv_lens[:, None] - 1).expand(B, max_q)
    last = torch.minimum(last, kv_lens[:, None] - 1)
    s.masked_fill_(torch.arange(L, device='cuda') > last[:, None, None, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    s.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)).exp_()
    l = s.sum(-1, keepdim=True)
    o = torch.matmul(s.view(B, Hkv, G * max_q, L), v).view(B, Hkv, G, max_q, hd)
    o = torch.where(l > 0, o / l, torch.zeros_like(o)).permute(0, 3, 1, 2, 4).reshape(B, max_q, Hq, hd)
    return o[_places(cu_q, T)].to(q.dtype)


def run(state):
    s, c = state, state['case']
    if c['kind'] == 'rope':
        if own:
            return _kernels().rope(s['x'], s['positions'], s['inv_freq'], interleaved=c['interleaved'], scale=s['scale'],
                                   out=s['out'])
        r = c['rot']
        a = s['positions'].double()[:, None, None] * s['inv_freq']
        cos, sin = a.cos().float(), a.sin().float()
        x = s['x'].float()
        x0, x1 = (x[..., 0:r:2], x[..., 1:r:2]) if c['interleaved'] else (x[..., :r // 2], x[..., r // 2:r])
        y0, y1 = s['scale'] * (x0 * cos - x1 * sin), s['scale'] * (x1 * cos + x0 * sin)
        y = torch.stack((y0, y1), -1).flatten(-2) if c['interleaved'] else torch.cat((y0, y1), -1)
        return torch.cat((y, x[..., r:]), -1).to(s['x'].dtype)
    if c['kind'] == 'write':
        kp, vp, ks, vs = s['pages']
        if own:
            _kernels().cache_write(s['k'], s['v'], kp, vp, s['slots'], k_scale=ks, v_scale=vs)
        else:
            page, at = (s['slots'] // c['page']).long(), (s['slots'] % c['page']).long()
            if ks is None:
                kp[page, :, at], vp[page, :, at] = s['k'], s['v']
            else:
                kp.view(torch.uint8)[page, :, at], ks.view(torch.uint8)[page, :, at] = _quantise(s['k'])
                vp.view(torch.uint8)[page, :, at], vs.view(torch.uint8)[page, :, at] = _quantise(s['v'])
        return [t for t in s['pages'] if t is not None]
    if c['kind'] == 'read':
        kp, vp, ks, vs = s['pages']
        if own:
            return _kernels().cache_read(kp, vp, s['table'], s['cu'], s['tokens'], k_scale=ks, v_scale=vs,
                                         dtype=DT[c['dtype']])
        b, i = _places(s['cu'], s['tokens'])
        page, at = s['table'][b, i // c['page']].long(), i % c['page']
        if ks is None:
            return kp[page, :, at], vp[page, :, at]
        return tuple(_values(p.view(torch.uint8)[page, :, at], f.view(torch.uint8)[page, :, at]).to(DT[c['dtype']])
                     for p, f in ((kp, ks), (vp, vs)))
    scale = 1.0 / math.sqrt(c['hd'])
    if c['kind'] == 'paged':
        kp, vp, ks, vs = s['pages']
        if own:
            return _kernels().attention_paged(s['q'], kp, vp, s['table'], s['cu_q'], s['kv_lens'], k_scale=ks, v_scale=vs,
                                              causal=c['causal'])
        return _attention(s['q'], _gather(kp, ks, s['table']), _gather(vp, vs, s['table']), s['cu_q'], s['kv_lens'],
                          s['max_q'], c['causal'], scale)
    if own:
        return _kernels().attention_varlen(s['q'], s['k'], s['v'], s['cu_q'], causal=c['causal'])
    n = s['cu_q'][1:] - s['cu_q'][:-1]
    rows = (s['cu_q'][:-1, None] + torch.arange(s['max_q'], device='cuda')).clamp(max=s['q'].shape[0] - 1).long()
    k, v = (t[rows].float().permute(0, 2, 1, 3).contiguous() for t in (s['k'], s['v']))
    return _attention(s['q'], k, v, s['cu_q'], n, s['max_q'], c['causal'], scale)


# ------------------------------------------------------------------- the work --
def _pairs(q, k, causal):
    """(query, key) pairs seen: the last q of k places are the queries'."""
    if not causal:
        return q * k
    first = k - q + 1                      # keys of the first query
    return sum(max(0, first + i) for i in range(q)) if first < 1 else q * first + q * (q - 1) // 2


def work(case):
    c, e = case, 2
    w = 1 if c.get('cache') == 'e4m3' else 2
    if c['kind'] == 'rope':
        n = c['T'] * (c['heads'] + c['kv'])
        return dict(bytes=2 * e * n * c['hd'] + 4 * c['T'], flops=3 * n * c['rot'])
    if c['kind'] in ('write', 'read'):
        n = 2 * (c['T'] if c['kind'] == 'write' else sum(_ints(c['lens']))) * c['kv']
        return dict(bytes=n * (c['hd'] * (e + w) + (w == 1)), flops=n * c['hd'] * 2 if w == 1 else 0)
    q = _ints(c['q'])
    k = _ints(c['kv_len']) if c['kind'] == 'paged' else q
    flops = 4 * c['hd'] * c['heads'] * sum(_pairs(a, b, c['causal']) for a, b in zip(q, k))
    return dict(bytes=2 * e * sum(q) * c['heads'] * c['hd'] + 2 * sum(k) * c['kv'] * (c['hd'] * w + (w == 1)),
                flops=flops)


# ------------------------------------------------ the definitions, in 64 bits --
def _two(e):
    """2^e in 64 bits, for whole e (written as its exponent field: a power function may be off by a step)."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def _exact_codes(x):
    """e4m3 code values and scales of rows of f64 values, by the format's definition."""
    amax = x.abs().amax(-1, keepdim=True)
    m, e = torch.frexp(amax / 448.0)                       # amax / 448 = m 2^e, m in [0.5, 1)
    e = (e - (m == 0.5).int()).clamp(min=-126)             # the least e with amax / 448 <= 2^e
    y = x * _two(-e)
    _, f = torch.frexp(y)
    step = _two(torch.clamp(f - 1, min=-6) - 3)
    return torch.round(y / step) * step, _two(e).squeeze(-1)


def _exact_values(pages, scale, c):
    return pages.double() if scale is None else pages.double() * _two(scale.view(torch.uint8).long() - 127)[..., None]


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c['kind'] == 'rope':
        x, r = s['x'].double(), c['rot']
        turn = torch.remainder(s['positions'].double()[:, None] * s['inv_freq'][None], 2.0 * math.pi)
        z = torch.polar(torch.full_like(turn, s['scale']), turn)[:, None]
        p = x[..., :r].unflatten(-1, (r // 2, 2) if c['interleaved'] else (2, r // 2))
        p = p if c['interleaved'] else p.transpose(-1, -2)
        y = torch.view_as_real(torch.complex(p[..., 0].contiguous(), p[..., 1].contiguous()) * z)
        x[..., :r] = (y if c['interleaved'] else y.transpose(-1, -2)).flatten(-2)
        return x
    if c['kind'] == 'write':
        kp, vp, ks, vs = s['pages']
        page, at = (s['slots'] // c['page']).long(), (s['slots'] % c['page']).long()
        out = [kp.double(), vp.double()]
        if ks is not None:
            out += [_two(t.view(torch.uint8).long() - 127) for t in (ks, vs)]
        for j, x in enumerate((s['k'], s['v'])):
            if ks is None:
                out[j][page, :, at] = x.double()
            else:
                out[j][page, :, at], out[2 + j][page, :, at] = _exact_codes(x.double())
        return out
    if c['kind'] == 'read':
        got = []
        for p, f in zip(s['pages'][:2], s['pages'][2:]):
            x, parts = _exact_values(p, f, c), []
            for b, n in enumerate(_ints(c['lens'])):
                t = s['table'][b, :-(-n // c['page'])].long()
                parts.append(x[t].permute(0, 2, 1, 3).flatten(0, 1)[:n])
            got.append(torch.cat(parts))
        return tuple(got)
    qs = _ints(c['q'])
    out, G = [], c['heads'] // c['kv']
    if c['kind'] == 'paged':
        kx, vx = (_exact_values(p, f, c) for p, f in zip(s['pages'][:2], s['pages'][2:]))
    at = 0
    for b, n in enumerate(qs):
        q = s['q'][at:at + n].double()
        if c['kind'] == 'paged':
            L = _ints(c['kv_len'])[b]
            t = s['table'][b, :-(-L // c['page'])].long()
            k, v = (x[t].permute(0, 2, 1, 3).flatten(0, 1)[:L] for x in (kx, vx))
        else:
            L = n
            k, v = (s[x][at:at + n].double() for x in 'kv')
        o = torch.zeros_like(q)
        see = torch.arange(L, device='cuda')[None] <= torch.arange(n, device='cuda')[:, None] + (L - n if c['causal'] else L)
        for h in range(c['heads']):
            w = (q[:, h] @ k[:, h // G].T) / math.sqrt(c['hd'])
            w = torch.where(see, w, torch.full_like(w, -math.inf))
            o[:, h] = torch.nan_to_num(torch.softmax(w, -1)) @ v[:, h // G]
        out.append(o)
        at += n
    return torch.cat(out)

"""A run of steps over the token cache, each link held by itself: what norm_rope wrote against 64 bits of the
rows it was given, the cache's codes against the quantisation of what norm_rope wrote, and the attention
against 64 bits over what the cache then holds.  So nothing of one link's rounding loosens the next one's check.

Tolerances as in the tests of each: norm_rope in test_gpu_step_ops.py, attention in test_gpu_range_attention.py."""
import numpy as np
import pytest
import torch

from oracle import token_cache as O

pytestmark = pytest.mark.gpu
DT = {'f16': torch.float16, 'bf16': torch.bfloat16}
TOP = {'f16': 61440.0, 'bf16': 1.875 * 2.0 ** 127}
H, KV, HD, PAGE = 8, 2, 64, 16


def u(dt):
    return torch.finfo(DT[dt]).eps / 2


def f64(t):
    return t.detach().double().cpu().numpy()


def i32(v):
    return torch.tensor(np.asarray(v, np.int32)).cuda()


def attention_tol(ref, mag, most, n, dt):
    tiny = 6 * n * 2.0 ** -32 if dt == 'f16' else 0.0
    return u(dt) * (np.abs(ref) + mag) * (1 + 2.0 ** -6) + (2 * (HD + 4) * 2.0 ** -24 * most + 2.0 ** -17) * mag + tiny


def norm_tol(ref, y, dt):
    mag = np.abs(y).max(-1, keepdims=True) * 2
    return u(dt) * np.abs(ref) * (1 + 2.0 ** -6) + mag * (((HD + 4) / 2 + 5) * 2.0 ** -24 + 2.0 ** -20) + (2.0 ** -25 if dt == 'f16' else 0)


def misses(got, ref, tol):
    """The share of elements that are further off than tol."""
    return float(np.mean(~(np.abs(got - ref) <= tol)))


class Streams:
    """A batch's cache, tables and lengths, and a step over them."""

    def __init__(self, B, width, dt, quant, kind, pre, seed):
        from chestnut import kernels as K
        self.K, self.B, self.dt, self.quant, self.kind, self.pre = K, B, dt, quant, kind, pre
        n = B * width + 3
        if quant:
            self.cache = [torch.zeros(n, KV, PAGE, HD, dtype=torch.uint8, device='cuda').view(torch.float8_e4m3fn) for _ in 'kv'] + \
                [torch.zeros(n, KV, PAGE, dtype=torch.uint8, device='cuda').view(torch.float8_e8m0fnu) for _ in 'kv']
        else:
            self.cache = [torch.zeros(n, KV, PAGE, HD, dtype=DT[dt], device='cuda') for _ in 'kv'] + [None, None]
        self.table = torch.full((B, width), -1, dtype=torch.int32, device='cuda')
        self.kv, self.taken = i32([0] * B), i32([0])
        self.free = i32(np.random.default_rng(seed).permutation(n))
        self.f, self.s = K.rope_frequencies(48, base=1e4)
        self.axes = K.rope_axes([8, 8, 8], turns=True)
        g = torch.Generator().manual_seed(seed)
        self.wq, self.wk = ((torch.rand(HD, generator=g) + 0.5).to(DT[dt]).cuda() for _ in 'qk')
        self.shared = (i32([0, B]), i32([pre]))
        self.heads = {'window': dict(window=21, sinks=2), 'shared': dict(shared=self.shared), 'all': {}}[kind]

    def normed(self, x, pos):
        at = torch.stack([pos, pos // 7, pos % 7])                      # time, row and column of a place
        q, k = x[:, :H], x[:, H:H + KV]
        self.K.norm_rope(q, k, self.wq, self.wk, at, self.f, axes=self.axes, scale=self.s, q_out=q, k_out=k)

    def write(self, x, slots):
        kp, vp, ks, vs = self.cache
        self.K.cache_write(x[:, H:H + KV], x[:, H + KV:], kp, vp, slots, k_scale=ks, v_scale=vs)

    def step(self, new, x, out=None):
        """x [rows, H + 2 KV, HD]: its Q and K heads normed and turned in place."""
        cu, kv, pos, slots = self.K.cache_maps(new, self.kv, self.table, PAGE, x.shape[0], free_pages=self.free, taken=self.taken, kv_out=self.kv)
        self.normed(x, pos)
        self.write(x, slots)
        kp, vp, ks, vs = self.cache
        return self.K.attention_paged(x[:, :H], kp, vp, self.table, cu, kv, k_scale=ks, v_scale=vs, out=out, **self.heads)

    def begin(self, x):
        """x [pre, ...]: the shared rows, in pages that all tables begin with."""
        n = x.shape[0]
        _, _, pos, slots = self.K.cache_maps(i32([n]), i32([0]), self.table[:1], PAGE, n, free_pages=self.free, taken=self.taken)
        self.normed(x, pos)
        self.write(x, slots)
        self.table[1:] = self.table[:1]
        self.kv.fill_(n)

    def held(self, b, n):
        """What the cache holds of sequence b's first n places: (k, v) f64, and with e4m3 their codes and scales."""
        table, j = self.table[b].cpu().numpy(), np.arange(n)
        assert (table[j // PAGE] >= 0).all()
        at = lambda t: t.cpu().numpy()[table[j // PAGE], :, j % PAGE]
        if not self.quant:
            return [at(t.double()) for t in self.cache[:2]], None
        codes, byte = [[at(t.view(torch.uint8)) for t in pair] for pair in (self.cache[:2], self.cache[2:])]
        return [O.values(c, s) for c, s in zip(codes, byte)], (codes, byte)

    def check(self, new, before, raw, done, out, what, last=False):
        """A step's links, request by request; last: also that what is wrong would be seen."""
        a, f, axes, seen = 0, f64(self.f), self.axes.tolist(), 0
        for b, n in enumerate(new):
            where = f'{what}: request {b}'
            if not n:
                continue
            places = before[b] + np.arange(n)
            x, y = f64(raw[a:a + n]), f64(done[a:a + n])
            at = np.stack([places, places // 7, places % 7])
            for lo, hi, w, name in ((0, H, self.wq, 'q'), (H, H + KV, self.wk, 'k')):
                normed = O.rms_norm(x[:, lo:hi], f64(w))
                ref = O.rope(normed, at, f, False, self.s, axes=axes)
                assert misses(y[:, lo:hi], ref, norm_tol(ref, normed, self.dt)) == 0, f'{where}, {name}'
                if last and (at[:, 0] > 0).all():
                    assert misses(normed, ref, norm_tol(ref, normed, self.dt)) > 0.1, f'{where}: {name} not turned would pass'
            assert np.array_equal(y[:, H + KV:], x[:, H + KV:])
            m = before[b] + n
            (k, v), codes = self.held(b, m)
            for i, rows in enumerate((y[:, H:H + KV], y[:, H + KV:])):
                if codes is None:
                    assert np.array_equal((k, v)[i][places], rows), where
                else:
                    c, s = O.quantise(rows, TOP[self.dt])
                    assert np.array_equal(codes[0][i][places], c) and np.array_equal(codes[1][i][places], s), where
            seen_by = dict(window=21, sinks=2) if self.kind == 'window' else {}
            q, got = y[:, :H], f64(out[a:a + n])
            ref, mag, most = O.attention(q, k, v, **seen_by)
            tol = attention_tol(ref, mag, most, m, self.dt)
            assert misses(got, ref, tol) == 0, f'{where}: worst {np.max(np.abs(got - ref) - tol)}'
            if last and m > 30:
                wrong = {'zeros': 0 * ref, 'negated': -ref, 'a key less': O.attention(q, k[:-1], v[:-1], **seen_by)[0],
                         'values of another': O.attention(q, k, np.roll(v, 1, 0), **seen_by)[0]}
                if self.kind == 'window':
                    wrong['a wider window'] = O.attention(q, k, v, window=29, sinks=2)[0]
                    wrong['no window'] = O.attention(q, k, v)[0]
                    wrong['no first keys'] = O.attention(q, k, v, window=21)[0]
                if self.kind == 'shared':
                    wrong['own keys alone'] = O.attention(q, k[self.pre:], v[self.pre:])[0]
                    wrong['shared keys alone'] = O.attention(q, k[:self.pre], v[:self.pre])[0]
                for name, w in wrong.items():
                    assert misses(w, ref, tol) > (0.05 if name == 'a key less' else 0.5), f'{where}: {name} would pass ({misses(w, ref, tol)})'
                seen += 1
            a += n
        assert seen >= 3 or not last


@pytest.mark.parametrize('dt', ['f16', 'bf16'])
@pytest.mark.parametrize('quant', [False, True])
@pytest.mark.parametrize('kind', ['window', 'shared', 'all'])
def test_each_link_of_a_run_of_steps(gpu, dt, quant, kind):
    """Prompts with padded rows behind them, a chunk, then single tokens; the last steps are replays of a captured one, with
    eager steps on state of their own between them."""
    B, singles = 5, 7
    r = np.random.default_rng(21)
    rows = lambda n: torch.from_numpy(r.standard_normal((n, H + 2 * KV, HD))).to(DT[dt]).cuda()
    pre = 48 if kind == 'shared' else 0
    width = -(-(pre + 64 + 30 + singles + 2) // PAGE) + 1
    first, a, e = rows(pre), *(Streams(B, width, dt, quant, kind, pre, 5) for _ in 'ae')
    before = np.full(B, pre)
    if pre:
        for st in (a, e):
            st.begin(first.clone())
    for new in ([3, 40, 17, 1, 64], [2, 0, 30, 5, 1]):
        raw = torch.cat([rows(sum(new)), torch.zeros(2, H + 2 * KV, HD, dtype=DT[dt], device='cuda')])
        done = [raw.clone() for _ in 'ae']
        outs = [st.step(i32(new), x) for st, x in zip((a, e), done)]
        n = sum(new)
        assert torch.equal(outs[0][:n], outs[1][:n]) and torch.equal(done[0][:n], done[1][:n])
        a.check(new, before, raw, done[0], outs[0], f'{new}')
        before = before + new
    ones = i32([1] * B)
    x, out = rows(B), torch.zeros(B, H, HD, dtype=DT[dt], device='cuda')
    raw = x.clone()
    a.step(ones, x, out)
    assert torch.equal(e.step(ones, raw.clone()), out)
    a.check([1] * B, before, raw, x, out, 'a token')
    before = before + 1
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.cuda.synchronize()
        with torch.cuda.graph(g, stream=side):
            a.step(ones, x, out)
    torch.cuda.synchronize()
    for t in range(1, singles):
        raw = rows(B)
        x.copy_(raw)
        g.replay()
        wanted = e.step(ones, raw.clone())
        torch.cuda.synchronize()
        assert torch.equal(out, wanted), t
        a.check([1] * B, before, raw, x, out, f'step {t}', last=t == singles - 1)
        before = before + 1
    assert np.array_equal(a.kv.cpu().numpy(), before)

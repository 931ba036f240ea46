"""Per-kernel entry points on torch device tensors (probe / bench harness).

torch provides device memory and the current stream only; every computation
is a call into libchestnut.so.  The native side receives raw pointers plus
sizes, so every tensor argument is validated here first -- dtype, shape
against the sizes derived from the operands, contiguity, and that all of
them live on the current CUDA device -- and a mismatch raises ValueError
before anything is launched.  The native entry points then check sizes and
alignment again.  Shapes are checked before the device, so the checks run
(and are tested) without a GPU.
"""
import ctypes
import functools
import math

import torch

from ._lib import check, lib

# What a call costs the host: the launch itself is about 4 us, so each wrapper
# keeps its own share small -- one pass over the arguments, the raw stream and
# device queries torch itself uses, plain integers for pointers, and the GEMM
# planner's answer remembered by sizes (LayerNorm of 64 x 128: 10.8 -> 6.7 us per
# call, of which the raw C call is 4.0 and the output's allocation 1.1).
try:
    from torch._C import _cuda_getCurrentRawStream as _raw_stream
    from torch._C import _cuda_getDevice as _device
except ImportError:   # a torch without GPU support: the argument checks still run

    def _raw_stream(dev):
        return torch.cuda.current_stream(dev).cuda_stream

    def _device():
        return torch.cuda.current_device()


def _ptr(t):
    return t.data_ptr() if t is not None else None


def _check(t, dtype, name, shape=None):
    """dtype, exact shape (None entries are free) and contiguity of one tensor."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f'{name} must be a torch tensor')
    if t.dtype != dtype:
        raise ValueError(f'{name} must be {dtype}, got {t.dtype}')
    if shape is not None:
        ok = t.dim() == len(shape) and all(s is None or int(a) == int(s) for a, s in zip(t.shape, shape))
        if not ok:
            want = tuple('*' if s is None else int(s) for s in shape)
            raise ValueError(f'{name} must have shape {want}, got {tuple(t.shape)}')
    if not t.is_contiguous():
        raise ValueError(f'{name} must be contiguous')


def _validate_each(args):
    """The checks of _validate one by one, with the message of the first that fails."""
    present = [a for a in args if a[0] is not None]
    for a in present:
        _check(*a)
    for a in present:
        t, name = a[0], a[2]
        if not t.is_cuda:
            raise ValueError(f'{name} must be a CUDA tensor')
        if t.device.index != torch.cuda.current_device():
            raise ValueError(f'{name} is on {t.device}, not the current device cuda:{torch.cuda.current_device()}')
    return torch.cuda.current_device()


def _validate(*args):
    """args: (tensor or None, dtype, name[, shape]), the first a tensor.  Every
    present tensor is checked for dtype, shape and contiguity, and all of them
    for placement on the current CUDA device, whose index is returned."""
    first = args[0][0]
    dev = first.get_device() if type(first) is torch.Tensor else -1
    if dev < 0 or dev != _device():
        return _validate_each(args)
    for a in args:
        t = a[0]
        if t is None:
            continue
        if (type(t) is not torch.Tensor or t.dtype is not a[1] or t.get_device() != dev or not t.is_contiguous() or
                (len(a) == 4 and t.shape != a[3])):
            return _validate_each(args)
    return dev


def gemv(W, x, bias=None, act=0, rows_per_wg=0, out=None):
    """y = act(W @ x + bias): W f16 [rows, K], x f32 [K] -> f32 [rows]."""
    if W.dim() != 2:
        raise ValueError('W must be 2-D [rows, K]')
    rows, K = W.shape
    if act not in (0, 1):
        raise ValueError('act must be 0 (none) or 1 (gelu)')
    dev = _validate((W, torch.float16, 'W'), (x, torch.float32, 'x', (K,)), (bias, torch.float32, 'bias', (rows,)),
                    (out, torch.float32, 'out', (rows,)))
    y = out if out is not None else torch.empty(rows, dtype=torch.float32, device=W.device)
    check(lib().ck_gemv(W.data_ptr(), x.data_ptr(), _ptr(bias), y.data_ptr(), rows, K, K, act, rows_per_wg,
                        _raw_stream(dev)))
    return y


def _plan(M, N, K, b_kn, tile, split_k):
    t, s, nb = ctypes.c_int(tile), ctypes.c_int(split_k), ctypes.c_size_t()
    check(lib().ck_gemm_workspace(M, N, K, b_kn, ctypes.byref(t), ctypes.byref(s), ctypes.byref(nb)))
    return t.value, s.value, nb.value


_cached_plan = functools.lru_cache(maxsize=256)(_plan)


def gemm_workspace(M, N, K, b_kn, tile=0, split_k=0):
    """(tile, split, workspace bytes) of the planner.  Remembered for plain
    integers only: a float equal to one is refused here as by the library, and
    an object that can change (a 0-d tensor) is asked for its value each time."""
    plan = _cached_plan if type(M) is type(N) is type(K) is type(tile) is type(split_k) is int else _plan
    return plan(M, N, K, 1 if b_kn else 0, tile, split_k)


def _workspace(ws, nb, device):
    """The caller's f32 workspace if it holds nb bytes, else a new one."""
    if not nb:
        return None
    if ws is not None:
        _validate((ws, torch.float32, 'workspace'))
        if ws.numel() * 4 >= nb:
            return ws
    return torch.empty(nb // 4, dtype=torch.float32, device=device)


def gemm(A, B, b_kn=True, bias=None, tile=0, split_k=0, out=None, workspace=None):
    """C f32 = A @ B (+ bias): A f16 [M, K]; B f16 [K, N] (b_kn) or [N, K]."""
    if A.dim() != 2 or B.dim() != 2:
        raise ValueError('A and B must be 2-D')
    M, K = A.shape
    N = B.shape[1] if b_kn else B.shape[0]
    dev = _validate((A, torch.float16, 'A'), (B, torch.float16, 'B', (K, N) if b_kn else (N, K)),
                    (bias, torch.float32, 'bias', (N,)), (out, torch.float32, 'out', (M, N)))
    plan = _cached_plan if type(tile) is type(split_k) is int else _plan   # as gemm_workspace
    tile, split_k, nb = plan(M, N, K, 1 if b_kn else 0, tile, split_k)
    C = out if out is not None else torch.empty(M, N, dtype=torch.float32, device=A.device)
    ws = _workspace(workspace, nb, A.device)
    check(lib().ck_gemm(A.data_ptr(), B.data_ptr(), C.data_ptr(), _ptr(bias), M, N, K, K, N if b_kn else K, N,
                        1 if b_kn else 0, tile, split_k, _ptr(ws), nb, _raw_stream(dev)))
    return C


_EPI_OUT = {1: torch.float16, 2: torch.float16, 3: torch.float16, 4: torch.float32}


def gemm_epi(A, W, bias, epi, out, tile=0, split_k=0):
    """Fused-epilogue GEMM: A f16 [M, K], W f16 [N, K], bias f32 [N] or None;
    epi 1 f16(acc+bias), 2 f16(relu), 3 f16(gelu) -> out f16 [M, N];
    epi 4 out f32 [M, N] += acc + bias."""
    if epi not in _EPI_OUT:
        raise ValueError('epi must be 1..4')
    if A.dim() != 2 or W.dim() != 2:
        raise ValueError('A and W must be 2-D')
    M, K = A.shape
    N = W.shape[0]
    if out is None:
        raise ValueError('out is required')
    dev = _validate((A, torch.float16, 'A'), (W, torch.float16, 'W', (N, K)), (bias, torch.float32, 'bias', (N,)),
                    (out, _EPI_OUT[epi], 'out', (M, N)))
    plan = _cached_plan if type(tile) is type(split_k) is int else _plan   # as gemm_workspace
    tile, split_k, nb = plan(M, N, K, 0, tile, split_k)
    ws = _workspace(None, nb, A.device)
    check(lib().ck_gemm_epi(A.data_ptr(), W.data_ptr(), out.data_ptr(), _ptr(bias), M, N, K, K, K, N, epi, tile,
                            split_k, _ptr(ws), nb, _raw_stream(dev)))
    return out


def wmma_rdna4(fa, fb, fc):
    """RDNA4 WMMA fragments u16 [n,32,8] x2 + f32 [n,32,8] -> f32 [n,32,8]."""
    if fa.dim() != 3:
        raise ValueError('fragA must be [n, 32, 8]')
    n = fa.shape[0]
    dev = _validate((fa, torch.int16, 'fragA', (n, 32, 8)), (fb, torch.int16, 'fragB', (n, 32, 8)),
                    (fc, torch.float32, 'fragC', (n, 32, 8)))
    fd = torch.empty_like(fc)
    check(lib().ck_wmma_rdna4(_ptr(fa), _ptr(fb), _ptr(fc), _ptr(fd), n, _raw_stream(dev)))
    return fd


def mfma_kat(variant, A, B):
    """One MFMA on row-major operands: variant 0 A [16,32] B [32,16];
    variant 1 A [32,16] B [16,32]."""
    if variant not in (0, 1):
        raise ValueError('variant must be 0 (16x16x32) or 1 (32x32x16)')
    M, N, Kk = (16, 16, 32) if variant == 0 else (32, 32, 16)
    dev = _validate((A, torch.int16, 'A', (M, Kk)), (B, torch.int16, 'B', (Kk, N)))
    D = torch.empty(M, N, dtype=torch.float32, device=A.device)
    check(lib().ck_mfma_kat(variant, _ptr(A), _ptr(B), _ptr(D), _raw_stream(dev)))
    return D


def pack_yuv(Y, U, V):
    """Full-resolution Y, U, V planes u8 [H, W] -> u8 [6, H/2, W/2]."""
    if Y.dim() != 2 or Y.shape[0] % 2 or Y.shape[1] % 2:
        raise ValueError('Y must be u8 [H, W] with H and W even')
    H, W = Y.shape
    dev = _validate((Y, torch.uint8, 'Y', (H, W)), (U, torch.uint8, 'U', (H, W)), (V, torch.uint8, 'V', (H, W)))
    out = torch.empty((6, H // 2, W // 2), dtype=torch.uint8, device=Y.device)
    check(lib().ck_pack_yuv(Y.data_ptr(), U.data_ptr(), V.data_ptr(), H, W, out.data_ptr(), _raw_stream(dev)))
    return out


def frames_to_tensor(frame):
    """I420 frame u8 [H*3/2, W] -> u8 [6, H/2, W/2]."""
    if frame.dim() != 2 or frame.shape[0] % 6 or frame.shape[1] % 2:
        raise ValueError('frame must be u8 [H*3/2, W] with H a multiple of 4 and W even')
    dev = _validate((frame, torch.uint8, 'frame'))
    H = frame.shape[0] * 2 // 3
    W = frame.shape[1]
    out = torch.empty((6, H // 2, W // 2), dtype=torch.uint8, device=frame.device)
    check(lib().ck_frames_to_tensor(frame.data_ptr(), H, W, out.data_ptr(), _raw_stream(dev)))
    return out


def img_gather(img, yx):
    """img [A, B, lanes] (any 1/2/4-byte dtype), yx int32 [n, 2] -> [n, lanes]."""
    if img.dim() != 3 or img.element_size() not in (1, 2, 4):
        raise ValueError('img must be [A, B, lanes] of a 1-, 2- or 4-byte dtype')
    if yx.dim() != 2:
        raise ValueError('yx must be int32 [n, 2]')
    dev = _validate((img, img.dtype, 'img'), (yx, torch.int32, 'yx', (yx.shape[0], 2)))
    A, B, lanes = img.shape
    n = yx.shape[0]
    out = torch.empty(n, lanes, dtype=img.dtype, device=img.device)
    check(lib().ck_img_gather(img.data_ptr(), A, B, lanes, img.element_size(), yx.data_ptr(), n, out.data_ptr(),
                              _raw_stream(dev)))
    return out


def attention(qk, vt, n_heads, head_dim):
    """qk f16 [T, 2d] (Q | K), vt f16 [d, T] -> f16 [T, d], d = n_heads * head_dim."""
    d = n_heads * head_dim
    if qk.dim() != 2:
        raise ValueError('qk must be f16 [T, 2d]')
    T = qk.shape[0]
    dev = _validate((qk, torch.float16, 'qk', (T, 2 * d)), (vt, torch.float16, 'vt', (d, T)))
    out = torch.empty((T, d), dtype=torch.float16, device=qk.device)
    check(lib().ck_attention(qk.data_ptr(), vt.data_ptr(), out.data_ptr(), T, n_heads, head_dim, _raw_stream(dev)))
    return out


def layernorm(x, g, b, eps=1e-5, out_f16=True):
    """Row LayerNorm of x f32 [rows, d] with g, b f32 [d] -> f16 or f32 [rows, d]."""
    if x.dim() != 2:
        raise ValueError('x must be f32 [rows, d]')
    rows, d = x.shape
    dev = _validate((x, torch.float32, 'x'), (g, torch.float32, 'g', (d,)), (b, torch.float32, 'b', (d,)))
    out = torch.empty((rows, d), dtype=torch.float16 if out_f16 else torch.float32, device=x.device)
    check(lib().ck_layernorm(x.data_ptr(), g.data_ptr(), b.data_ptr(), out.data_ptr(), 1 if out_f16 else 0, rows, d,
                             eps, _raw_stream(dev)))
    return out


def warp_nv12(frame, big_frame, tfm, big_tfm, cam_w, cam_h, stride, y_height, model_w=512, model_h=256, out=None,
              division='ieee'):
    """NV12 frames (u8 device buffers) + f32 [3,3] inverse transforms ->
    u8 [2, 6, model_h/2, model_w/2] (the engine's `warped`).  division:
    'ieee' (src_x / src_w) or 'rcp' (src_x * (1 / src_w)), as
    oracle.warp's `div`."""
    if division not in ('ieee', 'rcp'):
        raise ValueError("division must be 'ieee' or 'rcp'")
    nb = stride * y_height + (cam_h // 2) * stride
    for t, n in ((frame, 'frame'), (big_frame, 'big_frame')):
        if t.numel() != nb:
            raise ValueError(f'{n} must hold {nb} bytes of NV12 (stride {stride}, y_height {y_height}), '
                             f'got {t.numel()}')
    for t, n in ((tfm, 'tfm'), (big_tfm, 'big_tfm')):
        if t.numel() != 9:
            raise ValueError(f'{n} must be 3x3')
    shape = (2, 6, model_h // 2, model_w // 2)
    dev = _validate((frame, torch.uint8, 'frame'), (big_frame, torch.uint8, 'big_frame'), (tfm, torch.float32, 'tfm'),
                    (big_tfm, torch.float32, 'big_tfm'), (out, torch.uint8, 'out', shape))
    if out is None:
        out = torch.empty(shape, dtype=torch.uint8, device=frame.device)
    check(lib().ck_warp_nv12(frame.data_ptr(), big_frame.data_ptr(), nb, tfm.data_ptr(), big_tfm.data_ptr(), cam_w,
                             cam_h, stride, y_height, model_w, model_h, 1 if division == 'rcp' else 0, out.data_ptr(),
                             _raw_stream(dev)))
    return out


# ------------------------------------------------------------ the token cache --
# K and V rows of past tokens in pages k_pages, v_pages [n_pages, n_kv, page, head_dim] (page a
# power of two, 16 to 1024): f16, bf16, or float8_e4m3fn with k_scale, v_scale [n_pages, n_kv, page]
# of float8_e8m0fnu, a power of two a row (cache_write leaves 2^-126 to 2^120; a row whose scale is
# that type's NaN is NaN).
# A slot is page index * page + place.
#
# Index tensors are int32 on the device; their values are not checked here (that would wait for
# the device).  Whatever they hold, nothing outside the tensors of a call is read or written.

_F16, _BF16, _E4M3, _E8M0 = torch.float16, torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
_DTYPE = {_F16: 1, _BF16: 4, _E4M3: 5}   # the codes of include/chestnut.h
_INT = 2 ** 31 - 1   # counts reach the library as C ints, to which ctypes would cut larger ones


def _rows(t, dtype, name, shape, unit=8, write=False):
    """Strides of tokens and heads of rows [tokens, heads, head_dim]; the
    elements of a head are contiguous, and every row starts at a multiple of
    `unit` elements."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f'{name} must be a torch tensor')
    if t.dtype is not dtype:
        raise ValueError(f'{name} must be {dtype}, got {t.dtype}')
    T, H, hd = shape
    if t.shape != shape:
        raise ValueError(f'{name} must have shape {(T, H, hd)}, got {tuple(t.shape)}')
    if T > _INT:
        raise ValueError(f'{name} must have under 2^31 rows, got {T}')
    s0, s1, s2 = t.stride()
    if s2 != 1 and hd > 1:
        raise ValueError(f'{name} must be contiguous in its last dimension')
    if T <= 1:
        s0 = 0
    if H <= 1:
        s1 = 0
    if (s0 | s1) % unit or t.data_ptr() % (2 * unit):
        raise ValueError(f'{name} must have rows that start at multiples of {2 * unit} bytes')
    # written rows: token by token or head by head, each behind the end of the last
    if write and T > 0 and ((H > 1 and s1 < hd) or (T > 1 and s0 < (H - 1) * s1 + hd)) and \
            ((T > 1 and s0 < hd) or (H > 1 and s1 < (T - 1) * s0 + hd)):
        raise ValueError(f'{name} must not overlap itself')
    return s0, s1


def _is(t, dtype, name, shape):
    """_check, at a fraction of its time where all is well."""
    if type(t) is not torch.Tensor or t.dtype is not dtype or t.shape != shape or not t.is_contiguous():
        _check(t, dtype, name, shape)


def _on_device(names, *tensors):
    """The current device, on which every present tensor must be (the first one always is)."""
    dev = tensors[0].get_device()
    for t in tensors:
        if t is not None and t.get_device() != dev:
            dev = -2
            break
    if dev < 0 or dev != _device():
        present = [(t, n) for t, n in zip(tensors, names.split()) if t is not None]
        for t, n in present:
            if not t.is_cuda:
                raise ValueError(f'{n} must be a CUDA tensor')
        raise ValueError('; '.join(f'{n} is on {t.device}' for t, n in present) +
                         f', not the current device cuda:{_device()}')
    return dev


def _cache_each(k_pages, v_pages, k_scale, v_scale):
    """The checks of _cache one by one, with the message of the first that fails."""
    if not isinstance(k_pages, torch.Tensor) or k_pages.dim() != 4:
        raise ValueError('k_pages must be [n_pages, n_kv, page, head_dim]')
    dtype = k_pages.dtype
    if dtype not in _DTYPE:
        raise ValueError(f'k_pages must be float16, bfloat16 or float8_e4m3fn, got {dtype}')
    n, kv, page, hd = k_pages.shape
    if page < 16 or page > 1024 or page & (page - 1):
        raise ValueError(f'the page size must be a power of two from 16 to 1024, got {page}')
    if n < 1 or kv < 1:
        raise ValueError('k_pages must hold a page and a head')
    _check(k_pages, dtype, 'k_pages')
    _check(v_pages, dtype, 'v_pages', (n, kv, page, hd))
    if dtype is _E4M3:
        if k_scale is None or v_scale is None:
            raise ValueError('an e4m3 cache needs k_scale and v_scale')
        _check(k_scale, _E8M0, 'k_scale', (n, kv, page))
        _check(v_scale, _E8M0, 'v_scale', (n, kv, page))
    elif k_scale is not None or v_scale is not None:
        raise ValueError('k_scale and v_scale belong to an e4m3 cache')


def _cache(k_pages, v_pages, k_scale, v_scale):
    """The checks of a cache; its shape (n_pages, n_kv, page, head_dim)."""
    T = torch.Tensor
    if type(k_pages) is T and type(v_pages) is T:
        dtype, shape = k_pages.dtype, k_pages.shape
        if len(shape) == 4 and v_pages.dtype is dtype and v_pages.shape == shape:
            n, kv, page, _ = shape
            if 16 <= page <= 1024 and not page & (page - 1) and n and kv and k_pages.is_contiguous() and \
                    v_pages.is_contiguous():
                if dtype is _E4M3:
                    if type(k_scale) is T and type(v_scale) is T and k_scale.dtype is v_scale.dtype is _E8M0 and \
                            k_scale.shape == v_scale.shape == shape[:3] and k_scale.is_contiguous() and \
                            v_scale.is_contiguous():
                        return shape
                elif dtype in _DTYPE and k_scale is None and v_scale is None:
                    return shape
    _cache_each(k_pages, v_pages, k_scale, v_scale)
    return k_pages.shape


def rope_frequencies(rot, base=10000.0, method='none', factor=1.0, context=None, slow=1.0, fast=32.0, device='cuda'):
    """(inv_freq f64 [rot/2], scale) for `rope`: the inverse frequencies
    base^(-2i/rot) of the pairs of the first `rot` elements of a head, fitted
    to a context `factor` times as long as the one trained on:
      'none'    as they are;
      'linear'  positions divided by factor (Chen et al. 2023);
      'base'    base * factor^(rot/(rot-2)), which stretches the slowest pair by
                factor and leaves the fastest;
      'parts'   pairs that turn fewer than `slow` times within `context`
                positions (the trained length) divided by factor, those that turn
                more than `fast` times left, linear in the turns between, and
                scale 0.1 ln(factor) + 1 (YaRN, Peng et al. 2023)."""
    if not isinstance(rot, int) or rot < 2 or rot % 2:
        raise ValueError('rot must be an even number of elements')
    if method not in ('none', 'linear', 'base', 'parts'):
        raise ValueError("method must be 'none', 'linear', 'base' or 'parts'")
    if not base > 1.0 or not factor >= 1.0:
        raise ValueError('base must be above 1 and factor at least 1')
    if method == 'base':
        if rot < 4:
            raise ValueError("method 'base' needs rot of at least 4")
        base = base * factor ** (rot / (rot - 2.0))
    f = torch.pow(torch.tensor(float(base), dtype=torch.float64), -torch.arange(0, rot, 2, dtype=torch.float64) / rot)
    scale = 1.0
    if method == 'linear':
        f = f / factor
    elif method == 'parts':
        if not context or context < 1 or not 0 < slow < fast:
            raise ValueError("method 'parts' needs the trained context and 0 < slow < fast")
        keep = ((context * f / (2 * math.pi) - slow) / (fast - slow)).clamp(0.0, 1.0)
        f = f * keep + f / factor * (1.0 - keep)
        scale = 0.1 * math.log(factor) + 1.0
    return f.to(device), scale


def rope(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False, out=None):
    """Rotary positions: the first 2 * len(inv_freq) elements of every head of x
    [T, heads, head_dim] (f16 or bf16; token and head strides are free) turned
    by positions[t] * inv_freq[i], pairs (i, i + rot/2) or, interleaved, (2i,
    2i+1), times scale; the rest is copied.  positions int32 [T], inv_freq f64.
    out: x itself (in place) or rows that do not overlap it."""
    if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.dtype not in (_F16, _BF16):
        raise ValueError('x must be float16 or bfloat16 [T, heads, head_dim]')
    T, H, hd = x.shape
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
        raise ValueError('inv_freq must be float64 [rot/2]')
    rot = 2 * inv_freq.shape[0]
    _check(inv_freq, torch.float64, 'inv_freq')
    if rot < 2 or rot > hd:
        raise ValueError(f'inv_freq must have 1 to head_dim / 2 = {hd // 2} entries, got {rot // 2}')
    if H < 1 or hd > 512 or H > 1024 or H * hd > 65536:
        raise ValueError('rope takes head_dim up to 512, heads up to 1024 and 65536 elements a token')
    _is(positions, torch.int32, 'positions', (T,))
    st, sh = _rows(x, x.dtype, 'x', x.shape, 1, out is x)
    if out is None:
        ot, oh = H * hd, hd
    else:
        ot, oh = (st, sh) if out is x else _rows(out, x.dtype, 'out', x.shape, 1, True)
    dev = _on_device('x positions inv_freq out', x, positions, inv_freq, out)
    y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    check(lib().ck_rope(x.data_ptr(), y.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), T, H, hd, rot, st, sh,
                        ot, oh, _DTYPE[x.dtype], 1 if interleaved else 0, scale, 1 if inverse else 0, _raw_stream(dev)))
    return y


def cache_write(k, v, k_pages, v_pages, slots, k_scale=None, v_scale=None):
    """Rows k and v [T, n_kv, head_dim] (token and head strides are free) to
    slots [T] of the cache; negative slots are left out, the others must
    differ.  The cache has the rows' type, or is e4m3: every row is then scaled
    by the least power of two that fits it and rounded to nearest even."""
    n, kv, page, hd = _cache(k_pages, v_pages, k_scale, v_scale)
    if not isinstance(k, torch.Tensor) or k.dim() != 3 or k.dtype not in (_F16, _BF16):
        raise ValueError('k must be float16 or bfloat16 [T, n_kv, head_dim]')
    if k_pages.dtype not in (k.dtype, _E4M3):
        raise ValueError(f'the cache must be {k.dtype} or float8_e4m3fn, got {k_pages.dtype}')
    T = k.shape[0]
    kt, kh = _rows(k, k.dtype, 'k', (T, kv, hd))
    vt, vh = _rows(v, k.dtype, 'v', (T, kv, hd))
    _is(slots, torch.int32, 'slots', (T,))
    dev = _on_device('k v k_pages v_pages slots k_scale v_scale', k, v, k_pages, v_pages, slots, k_scale, v_scale)
    check(lib().ck_cache_write(k.data_ptr(), v.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale),
                               _ptr(v_scale), slots.data_ptr(), T, n, kv, page, hd, kt, kh, vt, vh, _DTYPE[k.dtype],
                               _DTYPE[k_pages.dtype], _raw_stream(dev)))


def cache_read(k_pages, v_pages, block_table, cu_seqlens, tokens, k_scale=None, v_scale=None, dtype=None, k_out=None,
               v_out=None):
    """(k, v) [tokens, n_kv, head_dim]: the first cu_seqlens[b+1] - cu_seqlens[b]
    places of every sequence b, whose pages are block_table[b] (int32 [B,
    width]), at rows cu_seqlens[b]...  dtype: float16 or bfloat16 for an e4m3
    cache (whose values above 65504, of rows that were bfloat16, are infinite in
    float16), else the cache's own.  Rows behind the last sequence are not written."""
    n, kv, page, hd = _cache(k_pages, v_pages, k_scale, v_scale)
    if dtype is None:
        dtype = k_out.dtype if k_out is not None else k_pages.dtype
    if dtype not in (_F16, _BF16) or k_pages.dtype not in (dtype, _E4M3):
        raise ValueError(f'dtype must be float16 or bfloat16, and that of the cache ({k_pages.dtype}) unless it is e4m3')
    if not isinstance(tokens, int) or not 0 <= tokens <= _INT:
        raise ValueError('tokens must be the number of rows, under 2^31')
    _check(block_table, torch.int32, 'block_table', (None, None))
    B, width = block_table.shape
    if B > _INT or width > _INT:
        raise ValueError(f'block_table must have under 2^31 rows and columns, got {(B, width)}')
    _is(cu_seqlens, torch.int32, 'cu_seqlens', (B + 1,))
    for t, name in ((k_out, 'k_out'), (v_out, 'v_out')):
        if t is not None:
            _check(t, dtype, name, (tokens, kv, hd))
    dev = _on_device('k_pages v_pages block_table cu_seqlens k_scale v_scale k_out v_out', k_pages, v_pages,
                     block_table, cu_seqlens, k_scale, v_scale, k_out, v_out)
    k, v = (t if t is not None else torch.empty((tokens, kv, hd), dtype=dtype, device=k_pages.device)
            for t in (k_out, v_out))
    check(lib().ck_cache_read(k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale), _ptr(v_scale),
                              block_table.data_ptr(), width, cu_seqlens.data_ptr(), B, tokens, n, kv, page, hd,
                              k.data_ptr(), v.data_ptr(), _DTYPE[dtype], _DTYPE[k_pages.dtype], _raw_stream(dev)))
    return k, v


def _queries(q, cu_q, kv, hd, out, scale):
    """The checks of packed queries [T, heads, head_dim] over kv K/V heads of hd:
    (T, heads, B, q strides, out strides, scale)."""
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in (_F16, _BF16):
        raise ValueError('q must be float16 or bfloat16 [T, heads, head_dim]')
    T, H, d = q.shape
    if d not in (64, 128) or hd != d:
        raise ValueError(f'head_dim must be 64 or 128 for q and the keys alike, got {d} and {hd}')
    if kv < 1 or H < 1 or H % kv or H > 1024:
        raise ValueError(f'the query heads ({H}, up to 1024) must be a multiple of the K/V heads ({kv})')
    if type(cu_q) is not torch.Tensor or cu_q.dtype is not torch.int32 or cu_q.dim() != 1 or not cu_q.is_contiguous():
        _check(cu_q, torch.int32, 'cu_q', (None,))
    if not 1 <= cu_q.shape[0] <= _INT:
        raise ValueError('cu_q must hold B + 1 offsets, under 2^31')
    qs = _rows(q, q.dtype, 'q', q.shape)
    os = (H * d, d) if out is None else _rows(out, q.dtype, 'out', q.shape, 4, True)
    scale = 1.0 / math.sqrt(d) if scale is None else float(scale)
    if not 2.0 ** -149 <= scale < 2e38:   # of an f32, and log2(e) times it too
        raise ValueError(f'scale must be positive and finite, from 2^-149 to 2e38, got {scale}')
    return T, H, cu_q.shape[0] - 1, qs, os, scale


def _attention_bytes(B, Tq, keys, n_heads, n_kv, head_dim):
    nb = ctypes.c_size_t()
    check(lib().ck_attention_workspace(B, Tq, keys, n_heads, n_kv, head_dim, ctypes.byref(nb)))
    return nb.value


_cached_attention_bytes = functools.lru_cache(maxsize=256)(_attention_bytes)


def attention_workspace(B, Tq, keys, n_heads, n_kv, head_dim):
    """Bytes of workspace (0: none) of attention_varlen (keys = Tk) and
    attention_paged (keys = B * table width * page) for B sequences of Tq
    queries in all.  Remembered for plain integers only, as gemm_workspace."""
    ints = type(B) is type(Tq) is type(keys) is type(n_heads) is type(n_kv) is type(head_dim) is int
    if any(abs(n) > _INT for n in (B, Tq, n_heads, n_kv, head_dim)) or abs(keys) >= 2 ** 63:
        raise ValueError('counts must be under 2^31, and keys under 2^63')
    return (_cached_attention_bytes if ints else _attention_bytes)(B, Tq, keys, n_heads, n_kv, head_dim)


def attention_varlen(q, k, v, cu_q, cu_k=None, causal=True, scale=None, out=None, workspace=None):
    """Attention of packed sequences: q [Tq, heads, head_dim] over k, v [Tk, n_kv,
    head_dim] (f16 or bf16; token and head strides are free), sequence b at rows
    cu_q[b] .. cu_q[b+1] of q and cu_k[b] .. cu_k[b+1] of k and v (int32 [B+1];
    cu_k None: the same).  causal: query i of n over m keys sees the keys
    j <= i + m - n; else all.  heads a multiple of n_kv, head_dim 64 or 128,
    scale 1/sqrt(head_dim) unless given.  A query without a key gets zeros; rows
    behind the last sequence are not written.  out may be q itself, and must not
    overlap q, k or v otherwise.
    workspace: a buffer to keep, of at least attention_workspace bytes (else a new
    one is made); one for each call that may run beside another, and for each
    captured graph."""
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError('k must be [Tk, n_kv, head_dim]')
    Tk, kv, hd = k.shape
    T, H, B, (qt, qh), (ot, oh), scale = _queries(q, cu_q, kv, hd, out, scale)
    kt, kh = _rows(k, q.dtype, 'k', k.shape)
    vt, vh = _rows(v, q.dtype, 'v', k.shape)
    if kt >= 1 << 24 or vt >= 1 << 24:
        raise ValueError('k and v must have under 2^24 elements from one token to the next')
    if cu_k is None:
        if Tk != T:
            raise ValueError(f'k must have the {T} rows of q where cu_k is not given, got {Tk}')
        cu_k = cu_q
    else:
        _is(cu_k, torch.int32, 'cu_k', (B + 1,))
    dev = _on_device('q k v cu_q cu_k out', q, k, v, cu_q, cu_k, out)
    o = out if out is not None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    nb = _cached_attention_bytes(B, T, Tk, H, kv, hd)
    ws = _workspace(workspace, nb, q.device)
    check(lib().ck_attention_varlen(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu_q.data_ptr(),
                                    cu_k.data_ptr(), B, T, Tk, H, kv, hd, qt, qh, kt, kh, vt, vh, ot, oh,
                                    _DTYPE[q.dtype], 1 if causal else 0, scale, _ptr(ws), nb, _raw_stream(dev)))
    return o


def attention_paged(q, k_pages, v_pages, block_table, cu_q, kv_lens, k_scale=None, v_scale=None, causal=True,
                    scale=None, out=None, workspace=None):
    """Attention of new tokens over a paged cache that holds their own K and V
    rows already: q [Tq, heads, head_dim], sequence b at rows cu_q[b] ..
    cu_q[b+1] (int32 [B+1]), its kv_lens[b] keys (int32 [B]) at places 0.. of the
    pages block_table[b] (int32 [B, width]); the queries are the last of them
    (causal: query i of n sees the keys j <= i + kv_lens[b] - n; else all).  The
    cache has q's type or is e4m3, whose values are rounded to q's type as cache_read
    rounds them (past float16's range: infinite).  Otherwise as attention_varlen."""
    n, kv, page, hd = _cache(k_pages, v_pages, k_scale, v_scale)
    T, H, B, (qt, qh), (ot, oh), scale = _queries(q, cu_q, kv, hd, out, scale)
    if k_pages.dtype not in (q.dtype, _E4M3):
        raise ValueError(f'the cache must be {q.dtype} or float8_e4m3fn, got {k_pages.dtype}')
    _is(kv_lens, torch.int32, 'kv_lens', (B,))
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError('block_table must be int32 [B, width]')
    width = block_table.shape[1]
    if width * page > 1 << 30:
        raise ValueError('block_table must name at most 2^30 places of a sequence')
    _is(block_table, torch.int32, 'block_table', (B, width))
    dev = _on_device('q k_pages v_pages block_table cu_q kv_lens k_scale v_scale out', q, k_pages, v_pages, block_table,
                     cu_q, kv_lens, k_scale, v_scale, out)
    o = out if out is not None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    nb = _cached_attention_bytes(B, T, B * width * page, H, kv, hd)
    ws = _workspace(workspace, nb, q.device)
    check(lib().ck_attention_paged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale), _ptr(v_scale),
                                   o.data_ptr(), block_table.data_ptr(), width, cu_q.data_ptr(), kv_lens.data_ptr(), B,
                                   T, H, n, kv, page, hd, qt, qh, ot, oh, _DTYPE[q.dtype], _DTYPE[k_pages.dtype],
                                   1 if causal else 0, scale, _ptr(ws), nb, _raw_stream(dev)))
    return o

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
    if t.is_contiguous():   # rows side by side
        s0, s1 = H * hd if T > 1 else 0, hd if H > 1 else 0
        if (s0 | s1) % unit or t.data_ptr() % (2 * unit):
            raise ValueError(f'{name} must have rows that start at multiples of {2 * unit} bytes')
        return s0, s1
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


def rope_axes(sections, turns=False, device='cuda'):
    """int32 [sum(sections)] for `rope` and `norm_rope`: every pair's axis, of which
    axis a has sections[a] pairs -- the axes' sections one after the other, or
    (turns) an axis after the other while it has pairs left.  With inv_freq =
    rope_frequencies(2 * sum(sections)) the axes share one ladder of
    frequencies; torch.cat of one rope_frequencies(2 * n) a section gives each its own."""
    left = list(sections)
    if not left or any(not isinstance(n, int) or n < 0 for n in left) or not any(left):
        raise ValueError('sections must be whole numbers of pairs, one for each axis')
    out = [] if turns else [a for a, n in enumerate(left) for _ in range(n)]
    while turns and any(left):
        for a, n in enumerate(left):
            if n:
                out.append(a)
                left[a] -= 1
    return torch.tensor(out, dtype=torch.int32, device=device)


def _angles(what, positions, inv_freq, axes, T, hd):
    """The checks of positions, frequencies and axes: (rot, number of axes)."""
    if not isinstance(inv_freq, torch.Tensor) or inv_freq.dim() != 1:
        raise ValueError('inv_freq must be float64 [rot/2]')
    half = inv_freq.shape[0]
    _check(inv_freq, torch.float64, 'inv_freq')
    if half < 1 or 2 * half > hd:
        raise ValueError(f'inv_freq must have 1 to head_dim / 2 = {hd // 2} entries, got {half}')
    if axes is None:
        _is(positions, torch.int32, 'positions', (T,))
        return 2 * half, 1
    _is(axes, torch.int32, 'axes', (half,))
    if not isinstance(positions, torch.Tensor) or positions.dim() != 2 or not 1 <= positions.shape[0] <= _INT:
        raise ValueError(f'positions must be int32 [axes, T] where {what} gets axes')
    n = positions.shape[0]
    _is(positions, torch.int32, 'positions', (n, T))
    return 2 * half, n


def rope(x, positions, inv_freq, interleaved=False, scale=1.0, inverse=False, out=None, axes=None):
    """Rotary positions: the first 2 * len(inv_freq) elements of every head of x
    [T, heads, head_dim] (f16 or bf16; token and head strides are free) turned
    by positions[t] * inv_freq[i], pairs (i, i + rot/2) or, interleaved, (2i,
    2i+1), times scale; the rest is copied.  positions int32 [T], inv_freq f64.
    out: x itself (in place) or rows that do not overlap it.
    axes (int32 [rot/2], `rope_axes`): positions are int32 [n, T], one row for
    each of n axes (time, row, column, ...), and pair i goes by positions[axes[i], t];
    an axis outside 0 .. n - 1 is held to it."""
    if not isinstance(x, torch.Tensor) or x.dim() != 3 or x.dtype not in (_F16, _BF16):
        raise ValueError('x must be float16 or bfloat16 [T, heads, head_dim]')
    T, H, hd = x.shape
    rot, n = _angles('rope', positions, inv_freq, axes, T, hd)
    if H < 1 or hd > 512 or H > 1024 or H * hd > 65536:
        raise ValueError('rope takes head_dim up to 512, heads up to 1024 and 65536 elements a token')
    st, sh = _rows(x, x.dtype, 'x', x.shape, 1, out is x)
    if out is None:
        ot, oh = H * hd, hd
    else:
        ot, oh = (st, sh) if out is x else _rows(out, x.dtype, 'out', x.shape, 1, True)
    dev = _on_device('x positions inv_freq out axes', x, positions, inv_freq, out, axes)
    y = out if out is not None else torch.empty(x.shape, dtype=x.dtype, device=x.device)
    check(lib().ck_rope_axes(x.data_ptr(), y.data_ptr(), positions.data_ptr(), n, _ptr(axes), inv_freq.data_ptr(), T, H, hd,
                             rot, st, sh, ot, oh, _DTYPE[x.dtype], 1 if interleaved else 0, scale, 1 if inverse else 0,
                             _raw_stream(dev)))
    return y


_WEIGHT = {torch.float32: 0, _F16: 1, _BF16: 4}


def norm_rope(q, k, q_weight, k_weight, positions, inv_freq, eps=1e-6, axes=None, interleaved=False, scale=1.0,
              q_out=None, k_out=None):
    """Every head of q [T, heads, head_dim] and k [T, n_kv, head_dim] (f16 or bf16
    alike; token and head strides are free) divided by sqrt(mean of its squares
    + eps), times q_weight or k_weight [head_dim] (both float32 or of q's type;
    None: ones), then turned as `rope` turns it, in one pass and with one rounding:
    (q_out, k_out).  k None: q alone (and k_out None).  q_out may be q and
    k_out k (in place); outputs overlap nothing else.  The squares are summed in
    32 bits: heads with values of 2^59 and more (bfloat16) become zeros."""
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.dtype not in (_F16, _BF16):
        raise ValueError('q must be float16 or bfloat16 [T, heads, head_dim]')
    T, H, hd = q.shape
    if k is None:
        if k_weight is not None or k_out is not None:
            raise ValueError('k_weight and k_out belong to k')
        kv = 0
    else:
        if not isinstance(k, torch.Tensor) or k.dim() != 3:
            raise ValueError('k must be [T, n_kv, head_dim]')
        kv = k.shape[1]
    rot, n = _angles('norm_rope', positions, inv_freq, axes, T, hd)
    if H < 1 or hd > 512 or H > 1024 or kv > 1024 or (H + kv) * hd > 65536 or (k is not None and kv < 1):
        raise ValueError('norm_rope takes head_dim up to 512, heads up to 1024 and 65536 elements a token')
    eps = float(eps)
    if not 2.0 ** -126 <= eps < 3e38:
        raise ValueError(f'eps must be positive and finite, from 2^-126, got {eps}')
    wt = q.dtype
    for w, name in ((q_weight, 'q_weight'), (k_weight, 'k_weight')):
        if w is not None:
            wt = w.dtype if isinstance(w, torch.Tensor) and w.dtype is torch.float32 else q.dtype
            _is(w, wt, name, (hd,))
    if q_weight is not None and k_weight is not None and q_weight.dtype is not k_weight.dtype:
        raise ValueError('q_weight and k_weight must have one type')
    strides, outs = [], []
    for x, out, name in ((q, q_out, 'q'), (k, k_out, 'k')):
        if x is None:
            strides.append((0, 0, 0, 0))
            outs.append(None)
            continue
        shape = (T, x.shape[1], hd)
        st, sh = _rows(x, q.dtype, name, shape, 1, out is x)
        ot, oh = (shape[1] * hd, hd) if out is None else (st, sh) if out is x else _rows(out, q.dtype, name + '_out', shape, 1, True)
        strides.append((st, sh, ot, oh))
        outs.append(out)
    dev = _on_device('q k q_weight k_weight positions inv_freq axes q_out k_out', q, k, q_weight, k_weight, positions, inv_freq,
                     axes, q_out, k_out)
    y, z = (o if o is not None or x is None else torch.empty(x.shape, dtype=q.dtype, device=q.device) for x, o in ((q, outs[0]), (k, outs[1])))
    (qt, qh, qot, qoh), (kt, kh, kot, koh) = strides
    check(lib().ck_norm_rope(q.data_ptr(), _ptr(k), y.data_ptr(), _ptr(z), _ptr(q_weight), _ptr(k_weight), positions.data_ptr(), n,
                             _ptr(axes), inv_freq.data_ptr(), T, H, kv, hd, rot, qt, qh, kt, kh, qot, qoh, kot, koh,
                             _DTYPE[q.dtype], _WEIGHT[wt], eps, 1 if interleaved else 0, scale, _raw_stream(dev)))
    return y, z


def _maps_bytes(B, tokens, in_place):
    nb = ctypes.c_size_t()
    check(lib().ck_cache_maps_workspace(B, tokens, 1 if in_place else 0, ctypes.byref(nb)))
    return nb.value


_cached_maps_bytes = functools.lru_cache(maxsize=256)(_maps_bytes)


def cache_maps_workspace(B, tokens, in_place):
    """Bytes of workspace (0: none) of cache_maps for B requests and `tokens` rows;
    in_place: kv_out is kv_lens or taken_out is taken."""
    if any(abs(n) > _INT for n in (B, tokens)):
        raise ValueError('counts must be under 2^31')
    return _maps_bytes(B, tokens, in_place)


def cache_maps(new_lens, kv_lens, block_table, page, tokens, free_pages=None, taken=None, kv_out=None, taken_out=None,
               workspace=None):
    """The index tensors of a step, built on the device from the lengths of its
    requests: new_lens [B] new tokens behind the kv_lens [B] places that each has
    (int32, as are all).  (cu_q [B+1], kv_out [B] = kv_lens + new_lens, positions
    [tokens], slots [tokens]): row cu_q[b] + i is place kv_lens[b] + i of request
    b, at slot block_table[b, place // page] * page + place % page -- what `rope`,
    `cache_write` and `attention_paged` take.  Rows behind the last request have
    position 0 and slot -1, which cache_write leaves out; tokens must hold the
    sum of new_lens (what passes it gets no row).

    free_pages [n] and taken [1]: new pages come from this list, request by request
    from entry taken on, and are entered in block_table; taken is advanced (in
    taken_out, if given, else in place) by all that were asked for.  Past the list's
    end entries and slots are -1, and taken above n says so.  Without them
    block_table names the new pages already.  A place without a page (a negative entry, or past the
    table) has slot -1.
    kv_out: kv_lens itself (a captured step then advances by itself), another
    tensor that overlaps no input, or None: a new one.
    workspace: a float32 buffer to keep, of at least cache_maps_workspace bytes (else
    a new one is made), one for each call that may run beside another."""
    B, width, n_free, dev = _maps(new_lens, kv_lens, block_table, page, tokens, free_pages, taken, kv_out, taken_out)
    if kv_out is not None and B and kv_out.data_ptr() == new_lens.data_ptr():
        raise ValueError('kv_out must not be new_lens')
    # one allocation for all outputs, cut up in one call
    if kv_out is None:
        cu, positions, slots, kv_out = torch.split_with_sizes(new_lens.new_empty(2 * (B + tokens) + 1), (B + 1, tokens, tokens, B))
    else:
        cu, positions, slots = torch.split_with_sizes(new_lens.new_empty(B + 1 + 2 * tokens), (B + 1, tokens, tokens))
    if taken is not None and taken_out is None:
        taken_out = taken
    nb = 0
    if tokens > 1024:   # (fewer need none)
        nb = _cached_maps_bytes(B, tokens, kv_out.data_ptr() == kv_lens.data_ptr() or
                                (taken is not None and taken_out.data_ptr() == taken.data_ptr()))
    ws = _workspace(workspace, nb, new_lens.device) if nb else None
    check(lib().ck_cache_maps(new_lens.data_ptr(), kv_lens.data_ptr(), block_table.data_ptr(), width,
                              (free_pages.data_ptr() or taken.data_ptr()) if free_pages is not None else None, n_free, _ptr(taken),
                              B, page, tokens, cu.data_ptr(), kv_out.data_ptr(), positions.data_ptr(), slots.data_ptr(),
                              _ptr(taken_out), _ptr(ws), nb, _raw_stream(dev)))
    return cu, kv_out, positions, slots


def _maps(new_lens, kv_lens, block_table, page, tokens, free_pages, taken, kv_out, taken_out):
    """The checks of cache_maps: (B, table width, pages in the list, device)."""
    T, i32 = torch.Tensor, torch.int32
    if type(new_lens) is type(kv_lens) is type(block_table) is T and type(tokens) is type(page) is int and \
            new_lens.dtype is kv_lens.dtype is block_table.dtype is i32:
        # all in one pass where all is well
        shape, at, dev = block_table.shape, new_lens.shape, new_lens.get_device()
        if len(shape) == 2 and at == shape[:1] == kv_lens.shape and shape[0] < 1 << 20 and 0 <= tokens < 1 << 30 and \
                16 <= page <= 1024 and not page & (page - 1) and shape[1] * page <= 1 << 30 and dev >= 0 and \
                kv_lens.get_device() == block_table.get_device() == dev == _device() and new_lens.is_contiguous() and \
                kv_lens.is_contiguous() and block_table.is_contiguous():
            ok = kv_out is None or (type(kv_out) is T and kv_out.dtype is i32 and kv_out.shape == at and
                                    kv_out.get_device() == dev and kv_out.is_contiguous())
            if ok and free_pages is None and taken is None and taken_out is None:
                return shape[0], shape[1], 0, dev
            if ok and type(free_pages) is type(taken) is T and free_pages.dtype is taken.dtype is i32 and free_pages.dim() == 1 and \
                    taken.shape == (1,) and free_pages.get_device() == taken.get_device() == dev and free_pages.is_contiguous() and \
                    (taken_out is None or (type(taken_out) is T and taken_out.dtype is i32 and taken_out.shape == (1,) and
                                           taken_out.get_device() == dev)):
                n_free = free_pages.shape[0]
                if n_free <= _INT:
                    return shape[0], shape[1], n_free, dev
    return _maps_each(new_lens, kv_lens, block_table, page, tokens, free_pages, taken, kv_out, taken_out)


def _maps_each(new_lens, kv_lens, block_table, page, tokens, free_pages, taken, kv_out, taken_out):
    """The checks of _maps one by one, with the message of the first that fails."""
    if not isinstance(tokens, int) or not 0 <= tokens < 1 << 30:
        raise ValueError('tokens must be the number of rows, under 2^30')
    if not isinstance(page, int) or page < 16 or page > 1024 or page & (page - 1):
        raise ValueError(f'the page size must be a power of two from 16 to 1024, got {page}')
    if type(new_lens) is not torch.Tensor or new_lens.dim() != 1:
        raise ValueError('new_lens must be int32 [B]')
    B = new_lens.shape[0]
    if B >= 1 << 20:
        raise ValueError(f'new_lens must have under 2^20 requests, got {B}')
    i32 = torch.int32
    _is(new_lens, i32, 'new_lens', (B,))
    _is(kv_lens, i32, 'kv_lens', (B,))
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError('block_table must be int32 [B, width]')
    width = block_table.shape[1]
    if width * page > 1 << 30:
        raise ValueError('block_table must name at most 2^30 places of a request')
    _is(block_table, i32, 'block_table', (B, width))
    if (free_pages is None) != (taken is None) or (taken is None and taken_out is not None):
        raise ValueError('free_pages, taken and taken_out belong together')
    n_free = 0
    if free_pages is not None:
        _check(free_pages, i32, 'free_pages', (None,))
        n_free = free_pages.shape[0]
        if n_free > _INT:
            raise ValueError(f'free_pages must have under 2^31 entries, got {n_free}')
        _is(taken, i32, 'taken', (1,))
        if taken_out is not None:
            _is(taken_out, i32, 'taken_out', (1,))
    if kv_out is not None:
        _is(kv_out, i32, 'kv_out', (B,))
    return B, width, n_free, _on_device('new_lens kv_lens block_table free_pages taken kv_out taken_out', new_lens, kv_lens,
                                        block_table, free_pages, taken, kv_out, taken_out)


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


def _range_bytes(B, Tq, keys, n_heads, n_kv, head_dim, window, sinks, groups):
    nb = ctypes.c_size_t()
    check(lib().ck_attention_range_workspace(B, Tq, keys, n_heads, n_kv, head_dim, window, sinks, groups, ctypes.byref(nb)))
    return nb.value


_cached_attention_bytes = functools.lru_cache(maxsize=256)(_attention_bytes)
_cached_range_bytes = functools.lru_cache(maxsize=256)(_range_bytes)


def attention_workspace(B, Tq, keys, n_heads, n_kv, head_dim, window=None, sinks=0, groups=0):
    """Bytes of workspace (0: none) of attention_varlen (keys = Tk) and
    attention_paged (keys = B * table width * page) for B sequences of Tq
    queries in all, through a window or with this many groups of shared pages.
    Remembered for plain integers only, as gemm_workspace."""
    ints = type(B) is type(Tq) is type(keys) is type(n_heads) is type(n_kv) is type(head_dim) is int
    if any(abs(n) > _INT for n in (B, Tq, n_heads, n_kv, head_dim)) or abs(keys) >= 2 ** 63:
        raise ValueError('counts must be under 2^31, and keys under 2^63')
    if window is None and not groups:
        _window(None, sinks, True)
        return (_cached_attention_bytes if ints else _attention_bytes)(B, Tq, keys, n_heads, n_kv, head_dim)
    window, sinks = _window(window, sinks, True)
    if not isinstance(groups, int) or not 0 <= groups < 1 << 20 or (groups and window):
        raise ValueError('groups must be a number under 2^20, and 0 with a window')
    return (_cached_range_bytes if ints else _range_bytes)(B, Tq, keys, n_heads, n_kv, head_dim, window, sinks, groups)


def _window(window, sinks, causal):
    """The checks of a window: (window or 0, sinks), held to 2^30."""
    if type(sinks) is not int or sinks < 0:
        raise ValueError('sinks must be a number of keys, 0 or more')
    if window is None:
        if sinks:
            raise ValueError('sinks belong to a window')
        return 0, 0
    if type(window) is not int or window < 1:
        raise ValueError('window must be a number of keys, 1 or more')
    if not causal:
        raise ValueError('a window belongs to causal attention')
    return min(window, 1 << 30), min(sinks, 1 << 30)


def attention_varlen(q, k, v, cu_q, cu_k=None, causal=True, scale=None, out=None, workspace=None, window=None, sinks=0):
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
    captured graph.
    window (causal only): of the keys above, query i sees the last `window` -- its own
    place and those before it -- and the first `sinks` of its sequence."""
    if not isinstance(k, torch.Tensor) or k.dim() != 3:
        raise ValueError('k must be [Tk, n_kv, head_dim]')
    Tk, kv, hd = k.shape
    T, H, B, (qt, qh), (ot, oh), scale = _queries(q, cu_q, kv, hd, out, scale)
    ranged = window is not None or sinks != 0
    if ranged:
        window, sinks = _window(window, sinks, causal)
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
    if ranged:
        nb = _cached_range_bytes(B, T, Tk, H, kv, hd, window, sinks, 0)
        ws = _workspace(workspace, nb, q.device) if workspace is not None else q.new_empty(nb >> 1) if nb else None
        check(lib().ck_attention_varlen_window(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu_q.data_ptr(),
                                               cu_k.data_ptr(), B, T, Tk, H, kv, hd, qt, qh, kt, kh, vt, vh, ot, oh,
                                               _DTYPE[q.dtype], window, sinks, scale, _ptr(ws), nb, _raw_stream(dev)))
        return o
    nb = _cached_attention_bytes(B, T, Tk, H, kv, hd)
    ws = _workspace(workspace, nb, q.device)
    check(lib().ck_attention_varlen(q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), cu_q.data_ptr(),
                                    cu_k.data_ptr(), B, T, Tk, H, kv, hd, qt, qh, kt, kh, vt, vh, ot, oh,
                                    _DTYPE[q.dtype], 1 if causal else 0, scale, _ptr(ws), nb, _raw_stream(dev)))
    return o


def attention_paged(q, k_pages, v_pages, block_table, cu_q, kv_lens, k_scale=None, v_scale=None, causal=True,
                    scale=None, out=None, workspace=None, window=None, sinks=0, shared=None):
    """Attention of new tokens over a paged cache that holds their own K and V
    rows already: q [Tq, heads, head_dim], sequence b at rows cu_q[b] ..
    cu_q[b+1] (int32 [B+1]), its kv_lens[b] keys (int32 [B]) at places 0.. of the
    pages block_table[b] (int32 [B, width]); the queries are the last of them
    (causal: query i of n sees the keys j <= i + kv_lens[b] - n; else all).  The
    cache has q's type or is e4m3, whose values are rounded to q's type as cache_read
    rounds them (past float16's range: infinite).  Otherwise as attention_varlen.
    shared: (cu_shared int32 [N+1], shared_lens int32 [N]) on the device -- the tables of the
    sequences cu_shared[g] .. cu_shared[g+1] (ascending) begin with the same pages, which hold
    their first shared_lens[g] keys (as far as these fill whole pages).  The shared keys are then
    read once for all queries of the group, from the table of its first sequence; the result
    is the same up to rounding.  Sequences may be in no group, which is the better place for one
    whose queries end within the shared keys: in a group it slows the shared keys of all of them
    (to 2 to 3 times).  Not with a window.  Its workspace: attention_workspace with groups=N."""
    n, kv, page, hd = _cache(k_pages, v_pages, k_scale, v_scale)
    T, H, B, (qt, qh), (ot, oh), scale = _queries(q, cu_q, kv, hd, out, scale)
    if k_pages.dtype not in (q.dtype, _E4M3):
        raise ValueError(f'the cache must be {q.dtype} or float8_e4m3fn, got {k_pages.dtype}')
    ranged, groups, cu_s, s_lens = window is not None or sinks != 0, 0, None, None
    if ranged:
        window, sinks = _window(window, sinks, causal)
    if shared is not None:
        if ranged:
            raise ValueError('a window and shared pages exclude each other')
        if not isinstance(shared, (tuple, list)) or len(shared) != 2 or not isinstance(shared[1], torch.Tensor) or \
                shared[1].dim() != 1 or not 1 <= shared[1].shape[0] < 1 << 20:
            raise ValueError('shared must be (cu_shared int32 [N + 1], shared_lens int32 [N]) of 1 to 2^20 - 1 groups')
        cu_s, s_lens = shared
        groups = s_lens.shape[0]
        _is(s_lens, torch.int32, 'shared_lens', (groups,))
        _is(cu_s, torch.int32, 'cu_shared', (groups + 1,))
    _is(kv_lens, torch.int32, 'kv_lens', (B,))
    if not isinstance(block_table, torch.Tensor) or block_table.dim() != 2:
        raise ValueError('block_table must be int32 [B, width]')
    width = block_table.shape[1]
    if width * page > 1 << 30:
        raise ValueError('block_table must name at most 2^30 places of a sequence')
    _is(block_table, torch.int32, 'block_table', (B, width))
    dev = _on_device('q k_pages v_pages block_table cu_q kv_lens k_scale v_scale out cu_shared shared_lens', q, k_pages,
                     v_pages, block_table, cu_q, kv_lens, k_scale, v_scale, out, cu_s, s_lens)
    o = out if out is not None else torch.empty(q.shape, dtype=q.dtype, device=q.device)
    if ranged or groups:
        nb = _cached_range_bytes(B, T, B * width * page, H, kv, hd, window if ranged else 0, sinks, groups)
        ws = _workspace(workspace, nb, q.device) if workspace is not None else q.new_empty(nb >> 1) if nb else None
        if ranged:
            check(lib().ck_attention_paged_window(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale), _ptr(v_scale),
                                                  o.data_ptr(), block_table.data_ptr(), width, cu_q.data_ptr(), kv_lens.data_ptr(), B,
                                                  T, H, n, kv, page, hd, qt, qh, ot, oh, _DTYPE[q.dtype], _DTYPE[k_pages.dtype],
                                                  window, sinks, scale, _ptr(ws), nb, _raw_stream(dev)))
        else:
            check(lib().ck_attention_paged_shared(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale), _ptr(v_scale),
                                                  o.data_ptr(), block_table.data_ptr(), width, cu_q.data_ptr(), kv_lens.data_ptr(),
                                                  cu_s.data_ptr(), s_lens.data_ptr(), groups, B, T, H, n, kv, page, hd, qt, qh, ot,
                                                  oh, _DTYPE[q.dtype], _DTYPE[k_pages.dtype], 1 if causal else 0, scale, _ptr(ws),
                                                  nb, _raw_stream(dev)))
        return o
    nb = _cached_attention_bytes(B, T, B * width * page, H, kv, hd)
    ws = _workspace(workspace, nb, q.device)
    check(lib().ck_attention_paged(q.data_ptr(), k_pages.data_ptr(), v_pages.data_ptr(), _ptr(k_scale), _ptr(v_scale),
                                   o.data_ptr(), block_table.data_ptr(), width, cu_q.data_ptr(), kv_lens.data_ptr(), B,
                                   T, H, n, kv, page, hd, qt, qh, ot, oh, _DTYPE[q.dtype], _DTYPE[k_pages.dtype],
                                   1 if causal else 0, scale, _ptr(ws), nb, _raw_stream(dev)))
    return o

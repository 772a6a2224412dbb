"""The native-operator surface of the reference, re-implemented on the B200 C ABI.

Function names and argument order follow the two extension modules the reference's
``DynamicLinear`` calls -- ``kairos_cuda_accel`` (kernels/csrc/pybind.cpp:16-24) and
``awq_backend`` (thirdparty/AWQ/kernels/csrc/pybind.cpp:17-26) -- so a call site can switch
by changing the import.  All tensors must be contiguous CUDA tensors; work is enqueued on
torch's current stream (the reference's GEMV/GEMM launch on the legacy default stream).
"""
from __future__ import annotations

import torch

from ._lib import check, lib
from .runtime import gemm_workspace

_current_device = torch._C._cuda_getDevice
_raw_stream = torch._C._cuda_getCurrentRawStream


class _AlreadyCurrent:
    def __enter__(self):
        return None

    def __exit__(self, *exc):
        return False


_ALREADY_CURRENT = _AlreadyCurrent()


def _on(device):
    """Device guard for a launch: free when `device` is the current one (one process per GPU), a real
    ``torch.cuda.device`` switch otherwise.  A call costs microseconds of host time, which is what the
    smallest kernels take on the device, so the wrappers avoid work that is not needed."""
    return _ALREADY_CURRENT if device.index == _current_device() else torch.cuda.device(device)


def stream_ptr():
    """torch's current stream on the current device, as the integer the C ABI takes."""
    return _raw_stream(_current_device())


def _chk(t, dtype, name):
    if not (t.is_cuda and t.is_contiguous() and t.dtype == dtype):
        raise ValueError(f'{name}: expected a contiguous CUDA tensor of {dtype}, got {t.dtype} on {t.device}')
    return t.data_ptr()


# ---- kairos_cuda_accel ------------------------------------------------------
def quant_fp16_to_int8(out, input, scale):
    """out[int8 ..,K], scale[fp16 tokens] <- per-token symmetric quantization of input."""
    k = input.shape[-1]
    m = input.numel() // k
    with _on(input.device):
        check(lib.kairos_act_quant_i8(_chk(input, torch.float16, 'input'), _chk(out, torch.int8, 'out'),
                                      _chk(scale, torch.float16, 'scale'), m, k, stream_ptr()), 'quant_fp16_to_int8')


def dequant_interleaved_int4_to_int8(output, input, scale, scaled_zero, group_size=128):
    assert group_size == 128
    n, k = output.shape
    with _on(output.device):
        check(lib.kairos_w4_to_w8(_chk(input, torch.int16, 'input'), _chk(scale, torch.float16, 'scale'),
                                  _chk(scaled_zero, torch.float16, 'scaled_zero'), _chk(output, torch.int8, 'output'),
                                  n, k, stream_ptr()), 'dequant_interleaved_int4_to_int8')


def dequant_interleaved_int4_to_fp16(output, input, scale, scaled_zero, group_size=128):
    assert group_size == 128
    n, k = output.shape
    with _on(output.device):
        check(lib.kairos_w4_to_f16(_chk(input, torch.int16, 'input'), _chk(scale, torch.float16, 'scale'),
                                   _chk(scaled_zero, torch.float16, 'scaled_zero'),
                                   _chk(output, torch.float16, 'output'), n, k, stream_ptr()),
              'dequant_interleaved_int4_to_fp16')


def trans_layout_c16_to_c8_awq(qweight, n, k):
    """AWQ interleaved int16 [N/4,K] -> QServe int8 [N,K/2]."""
    out = torch.empty((n, k // 2), dtype=torch.int8, device=qweight.device)
    with _on(qweight.device):
        check(lib.kairos_awq_to_qserve(_chk(qweight, torch.int16, 'qweight'), out.data_ptr(), n, k, stream_ptr()),
              'trans_layout_c16_to_c8_awq')
    return out


# ---- awq_backend ------------------------------------------------------------
def _bias_ptr(bias):
    return None if bias is None else _chk(bias, torch.float16, 'bias')


def gemv_forward_cuda_new(in_feats, kernel, scaling_factors, zeros, m, n, k, group_size=128, bias=None):
    """Kernel id 1 as the switched linear runs it (CUDA-core streamer or warp-MMA decode kernel)."""
    assert group_size == 128
    x = in_feats.reshape(-1, k)
    out = torch.empty((m, n), dtype=torch.float16, device=x.device)
    with _on(x.device):
        check(lib.kairos_w4a16_small_batch(_chk(x, torch.float16, 'in_feats'), _chk(kernel, torch.int16, 'kernel'),
                                           _chk(scaling_factors, torch.float16, 'scaling_factors'),
                                           _chk(zeros, torch.float16, 'zeros'), _bias_ptr(bias), out.data_ptr(), m,
                                           n, k, stream_ptr()), 'gemv_forward_cuda_new')
    return out


def gemv_cuda_core(in_feats, kernel, scaling_factors, zeros, m, n, k, bias=None):
    """The CUDA-core weight-streaming GEMV alone, 1 <= m <= 32."""
    x = in_feats.reshape(-1, k)
    out = torch.empty((m, n), dtype=torch.float16, device=x.device)
    with _on(x.device):
        check(lib.kairos_w4a16_gemv(_chk(x, torch.float16, 'in_feats'), _chk(kernel, torch.int16, 'kernel'),
                                    _chk(scaling_factors, torch.float16, 'scaling_factors'),
                                    _chk(zeros, torch.float16, 'zeros'), _bias_ptr(bias), out.data_ptr(), m, n, k,
                                    stream_ptr()), 'gemv_forward_cuda_new')
    return out


def decode_forward(in_feats, kernel, scaling_factors, zeros, m, n, k, bias=None):
    """W4A16 for 1 <= m <= 32 on the warp-level tensor-core decode kernel."""
    x = in_feats.reshape(-1, k)
    out = torch.empty((m, n), dtype=torch.float16, device=x.device)
    with _on(x.device):
        check(lib.kairos_w4a16_decode(_chk(x, torch.float16, 'in_feats'), _chk(kernel, torch.int16, 'kernel'),
                                      _chk(scaling_factors, torch.float16, 'scaling_factors'),
                                      _chk(zeros, torch.float16, 'zeros'), _bias_ptr(bias), out.data_ptr(), m, n, k,
                                      stream_ptr()), 'decode_forward')
    return out


def decode_silu_forward(in_feats, kernel, scaling_factors, zeros, m, n, k, bias=None):
    """Gate|up linear (n = 2 I weight rows in the blocked order) with SiLU(gate) * up applied in the decode kernel's
    epilogue, 1 <= m <= 32: returns [m, I]."""
    x = in_feats.reshape(-1, k)
    out = torch.empty((m, n // 2), dtype=torch.float16, device=x.device)
    with _on(x.device):
        check(lib.kairos_w4a16_decode_silu(_chk(x, torch.float16, 'in_feats'), _chk(kernel, torch.int16, 'kernel'),
                                           _chk(scaling_factors, torch.float16, 'scaling_factors'),
                                           _chk(zeros, torch.float16, 'zeros'), _bias_ptr(bias), out.data_ptr(), m, n, k,
                                           stream_ptr()), 'decode_silu_forward')
    return out


def gemm_forward_cuda_new(in_feats, kernel, scaling_factors, zeros, bias=None):
    k = in_feats.shape[-1]
    x = in_feats.reshape(-1, k)
    m, n = x.shape[0], kernel.shape[0] * 4
    out = torch.empty((m, n), dtype=torch.float16, device=x.device)
    with _on(x.device):
        ws = gemm_workspace(x.device, m, n, k)
        check(lib.kairos_w4a16_gemm(_chk(x, torch.float16, 'in_feats'), _chk(kernel, torch.int16, 'kernel'),
                                    _chk(scaling_factors, torch.float16, 'scaling_factors'),
                                    _chk(zeros, torch.float16, 'zeros'), _bias_ptr(bias), out.data_ptr(), m, n, k,
                                    ws.data_ptr(), ws.numel(), stream_ptr()), 'gemm_forward_cuda_new')
    return out


def w8a8_gemm_forward_cuda(in_feats, kernel, wscales, ascales, out_feats, bias=None, acc_out=None):
    m, k = in_feats.shape
    n = kernel.shape[0]
    with _on(in_feats.device):
        ws = gemm_workspace(in_feats.device, m, n, k)
        check(lib.kairos_w8a8_gemm(_chk(in_feats, torch.int8, 'in_feats'), _chk(kernel, torch.int8, 'kernel'),
                                   _chk(wscales, torch.float16, 'wscales'), _chk(ascales, torch.float16, 'ascales'),
                                   _bias_ptr(bias), _chk(out_feats, torch.float16, 'out_feats'),
                                   None if acc_out is None else _chk(acc_out, torch.int32, 'acc_out'), m, n, k,
                                   ws.data_ptr(), ws.numel(), stream_ptr()), 'w8a8_gemm_forward_cuda')
    return out_feats


# ---- kernels the reference reaches through torch / declares without a kernel ----
def f16_gemm(x, w16, bias=None):
    """``input @ weight.T`` with fp32 accumulation (kairos/dynamic_linear.py:163)."""
    m, k = x.shape
    n = w16.shape[0]
    out = torch.empty((m, n), dtype=torch.float16, device=x.device)
    with _on(x.device):
        ws = gemm_workspace(x.device, m, n, k)
        check(lib.kairos_f16_gemm(_chk(x, torch.float16, 'x'), _chk(w16, torch.float16, 'w16'), _bias_ptr(bias),
                                  out.data_ptr(), m, n, k, ws.data_ptr(), ws.numel(), stream_ptr()), 'f16_gemm')
    return out


def w8a16_gemm(x, w8, wscales, bias=None):
    """Kernel id 3: fp16 activations times the int8 weight widened to fp16 * s1."""
    m, k = x.shape
    n = w8.shape[0]
    out = torch.empty((m, n), dtype=torch.float16, device=x.device)
    with _on(x.device):
        ws = gemm_workspace(x.device, m, n, k)
        check(lib.kairos_w8a16_gemm(_chk(x, torch.float16, 'x'), _chk(w8, torch.int8, 'w8'),
                                    _chk(wscales, torch.float16, 'wscales'), _bias_ptr(bias), out.data_ptr(), m, n, k,
                                    ws.data_ptr(), ws.numel(), stream_ptr()), 'w8a16_gemm')
    return out


# ---- element-wise operators around the linears ------------------------------------------------
def rms_norm(x, weight, eps, residual_delta=None):
    """RMSNorm over the last dimension.  With `residual_delta`, x <- x + residual_delta IN PLACE first (the
    residual addition of the preceding block, carried by this pass)."""
    k = x.shape[-1]
    m = x.numel() // k
    y = torch.empty_like(x)
    with _on(x.device):
        if hasattr(residual_delta, 'peer_args'):
            # the delta is still spread over a tensor-parallel group (tp.PendingPeerSum): summed while loaded
            peer_in, peer_sig, world, rank = residual_delta.peer_args()
            check(lib.kairos_add_rms_norm_peer(_chk(x, torch.float16, 'x'), peer_in, peer_sig, world, rank,
                                               _chk(weight, torch.float16, 'weight'), y.data_ptr(), m, k, float(eps),
                                               stream_ptr()), 'add_rms_norm_peer')
        elif residual_delta is None:
            check(lib.kairos_rms_norm(_chk(x, torch.float16, 'x'), _chk(weight, torch.float16, 'weight'), y.data_ptr(),
                                      m, k, float(eps), stream_ptr()), 'rms_norm')
        else:
            check(lib.kairos_add_rms_norm(_chk(x, torch.float16, 'x'), _chk(residual_delta, torch.float16, 'delta'),
                                          _chk(weight, torch.float16, 'weight'), y.data_ptr(), m, k, float(eps),
                                          stream_ptr()), 'add_rms_norm')
    return y


def silu_mul(gate_up, blocked=False):
    """silu(gate) * up for the fused activation [..., 2I] -> [..., I]; `blocked`: gate and up channels alternate
    in blocks of 16 (see the header) instead of lying one after the other."""
    i2 = gate_up.shape[-1]
    m = gate_up.numel() // i2
    out = torch.empty(gate_up.shape[:-1] + (i2 // 2,), dtype=torch.float16, device=gate_up.device)
    fn = lib.kairos_silu_mul_blocked if blocked else lib.kairos_silu_mul
    with _on(gate_up.device):
        check(fn(_chk(gate_up, torch.float16, 'gate_up'), out.data_ptr(), m, i2 // 2, stream_ptr()), 'silu_mul')
    return out


def rope_kv(qkv, cos, sin, q_out, k_cache, v_cache, b, s, h, hkv, d, pos_dev=None, pos0=0):
    """Rotary embedding of q / k and the KV-cache write for a fused QKV activation (see the header)."""
    with _on(qkv.device):
        check(lib.kairos_rope_kv(_chk(qkv, torch.float16, 'qkv'), _chk(cos, torch.float16, 'cos'),
                                 _chk(sin, torch.float16, 'sin'), None if pos_dev is None else pos_dev.data_ptr(),
                                 int(pos0), _chk(q_out, torch.float16, 'q_out'), _chk(k_cache, torch.float16, 'k_cache'),
                                 _chk(v_cache, torch.float16, 'v_cache'), b, s, h, hkv, d, k_cache.shape[2],
                                 stream_ptr()), 'rope_kv')
    return q_out


def rms_norm_quant(x, weight, eps, want_f16=False, residual_delta=None):
    """RMSNorm emitting per-token int8 + fp16 scales (what a W8A8 linear consumes); also the fp16 result
    when `want_f16`; with `residual_delta`, x <- x + residual_delta in place first.
    Returns (xq, sx, y_or_None)."""
    k = x.shape[-1]
    m = x.numel() // k
    xq = torch.empty(x.shape, dtype=torch.int8, device=x.device)
    sx = torch.empty((m,), dtype=torch.float16, device=x.device)
    y = torch.empty_like(x) if want_f16 else None
    if hasattr(residual_delta, 'peer_args'):
        peer_in, peer_sig, world, rank = residual_delta.peer_args()
        with _on(x.device):
            check(lib.kairos_rms_norm_quant_peer(_chk(x, torch.float16, 'x'), peer_in, peer_sig, world, rank,
                                                 _chk(weight, torch.float16, 'weight'), None if y is None else y.data_ptr(),
                                                 xq.data_ptr(), sx.data_ptr(), m, k, float(eps), stream_ptr()),
                  'rms_norm_quant_peer')
        return xq, sx, y
    with _on(x.device):
        check(lib.kairos_rms_norm_quant(_chk(x, torch.float16, 'x'),
                                        None if residual_delta is None else _chk(residual_delta, torch.float16, 'delta'),
                                        _chk(weight, torch.float16, 'weight'), None if y is None else y.data_ptr(), xq.data_ptr(), sx.data_ptr(), m, k,
                                        float(eps), stream_ptr()), 'rms_norm_quant')
    return xq, sx, y


def silu_mul_quant(gate_up, want_f16=False, blocked=False):
    """silu(gate) * up emitting per-token int8 + fp16 scales.  Returns (xq, sx, y_or_None)."""
    i2 = gate_up.shape[-1]
    m = gate_up.numel() // i2
    shape = gate_up.shape[:-1] + (i2 // 2,)
    xq = torch.empty(shape, dtype=torch.int8, device=gate_up.device)
    sx = torch.empty((m,), dtype=torch.float16, device=gate_up.device)
    y = torch.empty(shape, dtype=torch.float16, device=gate_up.device) if want_f16 else None
    fn = lib.kairos_silu_mul_quant_blocked if blocked else lib.kairos_silu_mul_quant
    with _on(gate_up.device):
        check(fn(_chk(gate_up, torch.float16, 'gate_up'), None if y is None else y.data_ptr(), xq.data_ptr(),
                 sx.data_ptr(), m, i2 // 2, stream_ptr()), 'silu_mul_quant')
    return xq, sx, y


# ---- decoding over a paged key-value cache ----------------------------------------------------------
# A call costs microseconds of host time, as much as the smallest kernels take, so the checks below ask each tensor for
# as little as they can and tell what is wrong only once something is.
_FLOATS = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}
_HALVES = {torch.float16: 0, torch.bfloat16: 1}
_int32, _int64 = torch.int32, torch.int64


def _call(index, fn, *args):
    """fn(*args, stream) on torch's current stream of device `index`."""
    if index == _current_device():
        return fn(*args, _raw_stream(index))
    with torch.cuda.device(index):
        return fn(*args, _raw_stream(index))


def _one_device(index, owner, name):
    """The activations' device (-1: none) has to be the one of the cache or the plan."""
    if index < 0 or index != owner:
        raise ValueError(f'the activations are on CUDA device {index}, {name} is on {owner} (-1: not a CUDA device)')


def _bad(t, name, want, index):
    return ValueError(f'{name}: expected {want} on CUDA device {index}, got {t.dtype} {tuple(t.shape)}, strides {t.stride()}, '
                      f'on {t.device}')


def _rows(shape, strides):
    """Where the rows of a tensor with a dense last dimension begin, in elements, in ascending order."""
    at = torch.zeros(1, dtype=_int64, device='cpu')
    for n, step in zip(shape[:-1], strides[:-1]):
        at = (at[:, None] + torch.arange(n, device='cpu') * step).flatten()
    return at.sort().values


def _distinct(shape, strides):
    """Whether every element of a tensor with a dense last dimension has a place of its own.  It has if each dimension steps
    over all that the smaller ones reach; else the rows' places decide."""
    reach = 0
    for step, n in sorted((step, n) for step, n in zip(strides, shape) if n > 1):
        if step <= reach:
            return bool((_rows(shape, strides).diff() >= shape[-1]).all())
        reach += (n - 1) * step
    return True


def _disjoint(shape, a, b, offset):
    """Whether a tensor of strides `a` and one of strides `b` that begins `offset` elements behind it, both with a dense last
    dimension, have no element in common."""
    if 0 in shape:
        return True
    ends = [sum((n - 1) * step for n, step in zip(shape, strides)) for strides in (a, b)]
    if offset > ends[0] or -offset > ends[1]:
        return True
    dims = sorted((step, n) for step, n in zip(a, shape) if n > 1)
    if dims == sorted((step, n) for step, n in zip(b, shape) if n > 1):
        # slices of one activation: modulo a step that divides the larger ones both stay within a part of it
        reach = 0
        for i, (step, n) in enumerate(dims):
            if step and all(larger % step == 0 for larger, _ in dims[i:]) and reach < offset % step < step - reach:
                return True
            reach += (n - 1) * step
    first, second = _rows(shape, a), _rows(shape, b) + offset
    near = torch.searchsorted(first, second)                  # the rows of `a` on either side of each row of `b`
    behind = first[near.clamp(max=len(first) - 1)] - second
    before = second - first[(near - 1).clamp(min=0)]
    d = shape[-1]
    return not bool((((near < len(first)) & (behind < d)) | ((near > 0) & (before < d))).any())


def rotary(x, positions, rotary, transpose=False, out=None):
    """Heads [T, H, D] or [B, S, H, D] (fp16, bf16 or fp32; dense last dimension, any other strides) turned by their
    int64 positions, [T] or broadcastable to [B, S], with the plan of a :class:`Rotary`.  ``transpose`` turns back with the same
    magnitude: the gradient of x from that of the result.  ``out`` may be x, and must not overlap it otherwise.
    Like the other operators here it records no autograd graph."""
    shape, strides, code, index = x.shape, x.stride(), _FLOATS.get(x.dtype), x.get_device()
    dims = len(shape)
    if code is None or not 3 <= dims <= 4 or shape[-1] != rotary.head_dim or strides[-1] != 1:
        raise _bad(x, 'x', f'fp16, bf16 or fp32 [.., heads, {rotary.head_dim}] with a dense last dimension', index)
    if index < 0 or index != rotary.index:
        _one_device(index, rotary.index, 'rotary')
    if positions.dtype != _int64 or positions.get_device() != index:
        raise _bad(positions, 'positions', 'int64', index)
    if out is None:
        out = torch.empty_like(x)
        if out.stride(-1) != 1:                 # overlapping windows: another dimension came out as the dense one
            out = x.new_empty(shape)
    elif out.shape != shape or out.dtype != x.dtype or out.get_device() != index or out.stride(-1) != 1 or \
            not (out.is_contiguous() or _distinct(shape, out.stride())):
        raise _bad(out, 'out', f'{x.dtype} {tuple(shape)} with a dense last dimension and a place for every element', index)
    elif out is not x and not (out.data_ptr() == x.data_ptr() and
                               all(a == b or n == 1 for a, b, n in zip(out.stride(), strides, shape))) and \
            not _disjoint(shape, strides, out.stride(), (out.data_ptr() - x.data_ptr()) // x.element_size()):
        raise ValueError('out: overlaps x without being it')
    to, at = out.stride(), positions
    if dims == 3:
        b, xb, yb, pb, (s, h, d) = 1, 0, 0, 0, shape
        if at.shape != (s,):
            at = at.expand(s)
    else:
        b, s, h, d = shape
        if at.shape != (b, s):
            at = at.expand(b, s)
        xb, yb, pb = (strides[0], to[0], at.stride(0)) if b > 1 else (0, 0, 0)
    # the stride of a dimension of one element may be anything: none
    xs, ys, ps = (strides[-3], to[-3], at.stride(-1)) if s > 1 else (0, 0, 0)
    xh, yh = (strides[-2], to[-2]) if h > 1 else (0, 0)
    rc = _call(index, lib.kairos_rotary, x.data_ptr(), xb, xs, xh, out.data_ptr(), yb, ys, yh, at.data_ptr(), pb, ps,
               rotary.plan_ptr, code, 1 if transpose else 0, b, s, h, d)
    if rc < 0:
        check(rc, 'rotary')
    return out


def rope_paged_kv(qkv, positions, slots, rotary, cache, layer=0, q_out=None):
    """One pass over the fused activation qkv [T, (H + 2 kv_heads) * D] (fp16 / bf16, rows may be strided): returns the
    turned q heads [T, H, D], and stores the turned k heads and the v heads at ``slots`` [T] of the cache's `layer`, in
    the cache's type (int8 / e4m3 rows are quantized from fp32).  positions and slots are int64 [T]; a negative slot is
    padding and stores nothing; slots must be distinct, and q_out must not overlap qkv."""
    d, shape, code, index = cache.head_dim, qkv.shape, _HALVES.get(qkv.dtype), qkv.get_device()
    if code is None or len(shape) != 2 or shape[1] % d or qkv.stride(1) != 1:
        raise _bad(qkv, 'qkv', f'fp16 or bf16 [tokens, heads * {d}] with dense rows', index)
    t, h = shape[0], shape[1] // d - 2 * cache.kv_heads
    if h <= 0 or rotary.head_dim != d:
        raise ValueError(f'qkv has {shape[1] // d} heads of {d}: the cache holds {cache.kv_heads} kv heads, the rotary plan '
                         f'turns heads of {rotary.head_dim}')
    if index < 0 or index != cache.index or index != rotary.index:
        _one_device(index, cache.index, 'cache')
        _one_device(index, rotary.index, 'rotary')
    if positions.dtype != _int64 or positions.get_device() != index or positions.shape != (t,) or not positions.is_contiguous():
        raise _bad(positions, 'positions', f'contiguous int64 [{t}]', index)
    if slots.dtype != _int64 or slots.get_device() != index or slots.shape != (t,) or not slots.is_contiguous():
        raise _bad(slots, 'slots', f'contiguous int64 [{t}]', index)
    if q_out is None:
        q_out = qkv.new_empty((t, h, d))
    elif q_out.shape != (t, h, d) or q_out.dtype != qkv.dtype or q_out.get_device() != index or not q_out.is_contiguous():
        raise _bad(q_out, 'q_out', f'contiguous {qkv.dtype} [{t}, {h}, {d}]', index)
    rc = _call(index, lib.kairos_rope_paged_kv, qkv.data_ptr(), qkv.stride(0) if t > 1 else shape[1], positions.data_ptr(),
               slots.data_ptr(), rotary.plan_ptr, cache.layer_ptrs[layer], q_out.data_ptr(), t, h, code)
    if rc < 0:
        check(rc, 'rope_paged_kv')
    return q_out


def paged_kv_read(cache, slots, layer=0, dtype=torch.float16, out=None):
    """(k, v), each [T, kv_heads, D] of `dtype` (fp16, bf16 or fp32): what the cache's `layer` holds at ``slots`` (int64
    [T]), quantized rows as the values they stand for; zeros where the slot is negative.  ``out``: the two tensors to
    fill."""
    code, index = _FLOATS.get(dtype), slots.get_device()
    if code is None:
        raise ValueError(f'dtype: expected fp16, bf16 or fp32, got {dtype}')
    if index < 0 or index != cache.index:
        _one_device(index, cache.index, 'cache')
    if slots.dtype != _int64 or slots.dim() != 1 or not slots.is_contiguous():
        raise _bad(slots, 'slots', 'contiguous int64 [tokens]', index)
    t = slots.shape[0]
    shape = (t, cache.kv_heads, cache.head_dim)
    if out is None:
        k = slots.new_empty(shape, dtype=dtype)
        v = torch.empty_like(k)
    else:
        k, v = out
        for o in (k, v):
            if o.shape != shape or o.dtype != dtype or o.get_device() != index or not o.is_contiguous():
                raise _bad(o, 'out', f'two contiguous {dtype} {shape}', index)
    rc = _call(index, lib.kairos_paged_kv_read, cache.layer_ptrs[layer], slots.data_ptr(), k.data_ptr(), v.data_ptr(), t, code)
    if rc < 0:
        check(rc, 'paged_kv_read')
    return k, v


def paged_attention(q, cache, page_table, lens, layer=0, scale=None, out=None, return_lse=False):
    """Attention of one new token per sequence: q [B, H, D] (fp16 / bf16, strided batch and heads) over the first
    ``lens[b]`` positions of sequence b, whose pages are row b of ``page_table``.  page_table is int32 [B, W] (entries
    behind the end may hold anything), lens int32 [B]; scale defaults to 1 / sqrt(D).  Returns o [B, H, D], with
    ``return_lse`` also the fp32 [B, H] logarithm of the softmax's denominator.  An empty sequence gives zeros and
    -inf."""
    shape, strides, code, index = q.shape, q.stride(), _HALVES.get(q.dtype), q.get_device()
    if code is None or len(shape) != 3 or shape[2] != cache.head_dim or strides[2] != 1:
        raise _bad(q, 'q', f'fp16 or bf16 [batch, heads, {cache.head_dim}] with a dense last dimension', index)
    if index < 0 or index != cache.index:
        _one_device(index, cache.index, 'cache')
    b, h, d = shape
    pages, steps = page_table.shape, page_table.stride()
    if len(pages) != 2 or pages[0] != b or page_table.dtype != _int32 or page_table.get_device() != index or \
            (steps[1] != 1 and pages[1] > 1):
        raise _bad(page_table, 'page_table', f'int32 [{b}, pages] with dense rows', index)
    if lens.dtype != _int32 or lens.get_device() != index or lens.shape != (b,) or not lens.is_contiguous():
        raise _bad(lens, 'lens', f'contiguous int32 [{b}]', index)
    if out is None:
        out = torch.empty_like(q) if q.is_contiguous() else q.new_empty(shape)
    elif out.shape != shape or out.dtype != q.dtype or out.get_device() != index or not out.is_contiguous():
        raise _bad(out, 'out', f'contiguous {q.dtype} {tuple(shape)}', index)
    lse = q.new_empty((b, h), dtype=torch.float32) if return_lse else None
    width, kv = pages[1], cache.layer_ptrs[layer]
    key = (b, h, width)
    need = cache.workspace_bytes.get(key)
    if need is None:
        if len(cache.workspace_bytes) > 4096:
            cache.workspace_bytes.clear()
        with torch.cuda.device(index):
            need = cache.workspace_bytes[key] = lib.kairos_paged_attention_workspace_bytes(kv, b, h, width)
    # scratch of this call alone: an allocation that is cached per stream, and private to a graph under capture
    ws = page_table.new_empty(need >> 2) if need else None
    rc = _call(index, lib.kairos_paged_attention, q.data_ptr(), strides[0] if b > 1 else 0, strides[1] if h > 1 else 0, kv,
               page_table.data_ptr(), steps[0] if b > 1 else width, width, lens.data_ptr(), out.data_ptr(),
               lse.data_ptr() if return_lse else None, b, h, d ** -0.5 if scale is None else scale, code,
               ws.data_ptr() if need else None, need)
    if rc < 0:
        check(rc, 'paged_attention')
    return (out, lse) if return_lse else out

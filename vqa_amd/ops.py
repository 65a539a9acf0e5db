"""Token-level operators of libvqa_hip.so as functions of tensors.

A block in which the tokens of a question or caption read the image: ``gated_scan`` mixes the tokens,
``cross_attention`` reads the regions, ``norm_gate`` adds a block's output to the residual stream and norms it for the
next one.  (The reference reduces question and image to one vector each, seq2vec.py:16-25 and model.py:161-164, and has
no counterpart.)

Each operator comes as a differentiable function and as the explicit pair ``*_fwd`` / ``*_bwd`` it is made of, for
training loops that keep their own buffers.  Tensors live on one HIP device; the work goes to torch's current stream of
THAT device, whichever device is current.  Storage is float32 or bfloat16, arithmetic float32 (the factors that attention's
matrix products take in bfloat16 are named in include/vqa_hip.h).  An operand whose rows the kernels cannot read in 16-byte
pieces (odd strides or addresses) is copied first.  Outputs are new tensors.
"""
from __future__ import annotations

import functools
import math
from ctypes import byref

import torch

from . import _lib
from ._lib import VqaHipError


def _call(device, name, *args):
    """An entry point on torch's current stream of `device`.  The stream is asked for at every call (the module's bound
    stream belongs to the model that bound it) and the device is made current for the launch."""
    fn = _entry(name)
    stream = _raw_stream(device.index)
    if device.index == _current_device():
        rc = fn(*args, stream)
    else:
        with torch.cuda.device(device):
            rc = fn(*args, stream)
    if rc != 0:
        raise VqaHipError(f'{name} failed ({rc}): {_lib.load().vqa_last_error_string().decode()}')


# handle of torch's current stream of a device, and the current device, without the Python objects around them: a
# microsecond each on calls whose kernels take three
_raw_stream = getattr(torch._C, '_cuda_getCurrentRawStream', None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)
_current_device = getattr(torch._C, '_cuda_getDevice', None) or torch.cuda.current_device


@functools.lru_cache(None)
def _entry(name):
    return getattr(_lib.load(), name)


@functools.lru_cache(1024)
def _floats(name, *sizes):
    """What a workspace-size function says for these sizes (a foreign call costs as much as an allocation)."""
    return _entry(name)(*sizes)


def _new(t):
    """An uninitialised, contiguous tensor like `t` (None for None)."""
    return None if t is None else torch.empty_like(t, memory_format=torch.contiguous_format)


def _ptr(t):
    return None if t is None else t.data_ptr()


def _need(cond, msg, *args):
    if not cond:
        raise ValueError(msg.format(*args))


def _storage(name, t):
    if not t.is_cuda:
        raise VqaHipError(f'{name} runs on a HIP device only (inputs must be cuda tensors); there is no CPU path')
    return _lib.BF16 if t.dtype is torch.bfloat16 else _lib.dtype_code(t.dtype)


def _like(name, what, t, ref, shape, dtype=None):
    """`t` checked against the operand `ref` it goes with."""
    if t.shape != shape or t.dtype is not (dtype or ref.dtype) or t.get_device() != ref.get_device():
        raise ValueError(f'{name}: {what} must be {tuple(shape)} {dtype or ref.dtype} on {ref.device}, '
                         f'got {tuple(t.shape)} {t.dtype} on {t.device}')


def _packed(t):
    """`t`, contiguous and 16-byte aligned."""
    if t is None or (t.is_contiguous() and t.data_ptr() % 16 == 0):
        return t
    return t.clone(memory_format=torch.contiguous_format)


def _lengths(name, what, t, ref, n):
    if t is None:
        return None
    _need(t.shape == (n,) and t.device == ref.device and t.dtype in (torch.int32, torch.int64),
          '{}: {} must be ({},) int32 or int64 on {}', name, what, n, ref.device)
    if t.dtype != torch.int32:
        t = t.clamp(-1, 2 ** 31 - 1).to(torch.int32)
    return t.contiguous()


# ---- gated linear recurrence -------------------------------------------------------------------

def _scan_operands(gates, lengths, c0, name):
    dt = _storage(name, gates)
    _need(gates.dim() == 3 and gates.shape[2] % 32 == 0, '{}: gates must be (B, T, 4H) with H a multiple of 8', name)
    B, T, H = gates.shape[0], gates.shape[1], gates.shape[2] // 4
    sb, st, one = gates.stride()
    sb, st = sb if B > 1 else 0, st if T > 1 else 4 * H          # the stride of a size of 1 says nothing
    if one != 1 or sb % 8 or st % 8 or st < 4 * H or sb < 0 or gates.data_ptr() % 16:
        gates = gates.clone(memory_format=torch.contiguous_format)
        sb, st = T * 4 * H, 4 * H
    if c0 is not None:
        _like(name, 'c0', c0, gates, (B, H), torch.float32)
        c0 = _packed(c0)
    return dt, gates, sb, st, _lengths(name, 'lengths', lengths, gates, B), c0, B, T, H


def gated_scan_fwd(gates, lengths=None, c0=None, save=True):
    """c_t = s(f_t) c_{t-1} + s(i_t) tanh(g_t), h_t = s(o_t) tanh(c_t) over ``gates`` (B, T, 4H), gate order i, f, g, o.

    ``lengths`` (B,): steps of each sample (behind them h is 0 and the state stays); ``c0`` (B, H) float32 starting
    state.  Returns ``h`` (B, T, H), the last state ``c`` (B, H) float32, and what ``gated_scan_bwd`` needs (None unless
    ``save``).  With T = 1 and ``c0`` the state of the last call this is one step of a running sequence."""
    dt, gates, sb, st, lengths, c0, B, T, H = _scan_operands(gates, lengths, c0, 'gated_scan')
    dev = gates.device
    h = gates.new_empty((B, T, H))
    c = gates.new_empty((B, H), dtype=torch.float32)
    saved = gates.new_empty(((T + _SAVE - 1) // _SAVE, B, H), dtype=torch.float32) if save else None
    if B == 0 or T == 0 or H == 0:
        return h, c.zero_() if c0 is None else c.copy_(c0), saved
    ws = _workspace(_floats('vqa_gated_scan_workspace_floats', B, T, H, dt), gates)
    _call(dev, 'vqa_gated_scan_fwd', gates.data_ptr(), sb, st, _ptr(lengths), _ptr(c0), h.data_ptr(), c.data_ptr(),
          _ptr(saved), _ptr(ws), B, T, H, dt)
    return h, c, saved


def gated_scan_bwd(dh, dc, gates, saved, lengths=None, c0=None):
    """Gradients of ``gated_scan_fwd``: (dgates (B, T, 4H), dc0 (B, H) float32) from dh (B, T, H) and dc (B, H) float32,
    the gradient at the last state (either may be None: zero)."""
    dt, gates, sb, st, lengths, c0, B, T, H = _scan_operands(gates, lengths, c0, 'gated_scan')
    dev = gates.device
    dgates = _new(gates)
    dc0 = gates.new_empty((B, H), dtype=torch.float32)
    if dh is not None:
        _like('gated_scan', 'dh', dh, gates, (B, T, H))
        dh = _packed(dh)
    if dc is not None:
        _like('gated_scan', 'dc', dc, gates, (B, H), torch.float32)
        dc = _packed(dc)
    if B == 0 or T == 0 or H == 0 or (dh is None and dc is None):
        return dgates.zero_(), dc0.zero_() if dc is None else dc0.copy_(dc)
    _need(saved is not None, 'gated_scan: the backward needs what gated_scan_fwd(..., save=True) returned for these gates')
    _like('gated_scan', 'saved', saved, gates, ((T + _SAVE - 1) // _SAVE, B, H), torch.float32)
    saved = _packed(saved)
    ws = _workspace(_floats('vqa_gated_scan_workspace_floats', B, T, H, dt), gates)
    _call(dev, 'vqa_gated_scan_bwd', _ptr(dh), _ptr(dc), gates.data_ptr(), sb, st, _ptr(lengths), _ptr(c0),
          saved.data_ptr(), dgates.data_ptr(), dc0.data_ptr(), _ptr(ws), B, T, H, dt)
    return dgates, dc0


_SAVE = 8                    # VQA_GATED_SCAN_SAVE of include/vqa_hip.h


def _workspace(floats, like):
    """Scratch of one call, from torch's allocator: it belongs to the stream of the call (and, under capture, to the
    graph), so calls on two streams and two captured graphs never share it."""
    return like.new_empty(floats, dtype=torch.float32) if floats else None


class _GatedScan(torch.autograd.Function):
    @staticmethod
    def forward(ctx, gates, lengths, c0):
        h, c, saved = gated_scan_fwd(gates, lengths, c0, save=ctx.needs_input_grad[0] or ctx.needs_input_grad[2])
        ctx.save_for_backward(gates, lengths, c0, saved)
        ctx.set_materialize_grads(False)
        return h, c

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dh, dc):
        gates, lengths, c0, saved = ctx.saved_tensors
        if dh is None and dc is None:
            return None, None, None
        dgates, dc0 = gated_scan_bwd(dh, dc, gates, saved, lengths, c0)
        return dgates, None, dc0 if c0 is not None else None


def gated_scan(gates, lengths=None, c0=None):
    """Differentiable ``gated_scan_fwd``: (h, last state)."""
    return _GatedScan.apply(gates, lengths, c0)


# ---- norms with gate and residual update ---------------------------------------------------------

def _rows(t):
    """(tensor, leading dimension): `t` (..., D) as rows the kernels can read, copied if its strides do not allow it."""
    if t is None:
        return None, 0
    D, n = t.shape[-1], t.dim()
    if t.is_contiguous():
        return (t if t.data_ptr() % 16 == 0 else t.clone()), D
    ld, ok = None, t.stride(-1) == 1 or D == 1
    for i in range(n - 2, -1, -1):                              # one stride for all rows together
        if t.shape[i] == 1:
            continue
        if ld is None:
            ld, span = t.stride(i), t.stride(i) * t.shape[i]
        else:
            ok, span = ok and t.stride(i) == span, span * t.shape[i]
    ld = D if ld is None else ld
    if not ok or ld < D or ld % 8 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        ld = D
    return t, ld


def _norm_operands(name, x, f, gate, residual_scale, w_post, w_pre):
    dt, shape = _storage(name, x), x.shape
    D = shape[-1] if shape else 0
    _need(D % 8 == 0 and 8 <= D <= 8192, '{}: the width must be a multiple of 8 in [8, 8192]', name)
    rows = x.numel() // D
    if f is not None:
        _like(name, 'f', f, x, shape)
    elif gate is not None or residual_scale is not None or w_post is not None:
        raise ValueError(f'{name}: gate, residual_scale and w_post belong to the block output f')
    per = 0
    if gate is not None:
        per, gs = 1, gate.shape
        if gs != shape:
            # the gate's leading dimensions are x's up to some point, then ones: row r belongs to gate row r // per
            if len(gs) == 3 == len(shape) and gs[0] == shape[0] and gs[1] == 1 and gs[2] == D:
                per = shape[1]
            else:
                lead, full = list(gs[:-1]), list(shape[:-1])
                cut = max([i + 1 for i, s in enumerate(lead) if s != 1], default=0)
                _need(len(gs) and gs[-1] == D and len(lead) <= len(full) and lead[:cut] == full[:cut],
                      '{}: gate {} must share the leading dimensions of x {} up to some point and have size 1 behind it',
                      name, tuple(gs), tuple(shape))
                n = gate.numel() // D
                per = rows // n if n else 1
            per = max(per, 1)
        _like(name, 'gate', gate, x, gs)
    for what, w in (('residual_scale', residual_scale), ('w_post', w_post), ('w_pre', w_pre)):
        if w is not None:
            _like(name, what, w, x, (D,), torch.float32)
    return dt, D, rows, per


def norm_gate_fwd(x, f=None, gate=None, residual_scale=None, w_post=None, w_pre=None, eps=1e-6, want_y=True, want_h=True, save=True):
    """y = residual_scale x + s(gate) w_post f / rms(f) and h = w_pre y / rms(y) over the last dimension of ``x``.

    ``gate`` holds pre-activations in x's dtype, shaped as x or with size 1 in its last leading dimensions ((B, 1, D) or
    (B, D) for x (B, T, D): one gate row per sample); the weights are (D,) float32; what is None counts as 1.  With f
    None only h = w_pre x / rms(x) is made.  Returns (y, h, stats): y or h None when not made, stats for
    ``norm_gate_bwd`` (None unless ``save``)."""
    name = 'norm_gate'
    dt, D, rows, per = _norm_operands(name, x, f, gate, residual_scale, w_post, w_pre)
    want_y = want_y and f is not None
    _need(want_y or want_h, '{}: one of y, h must be wanted', name)
    _need(want_h or w_pre is None, '{}: w_pre belongs to h', name)
    y = _new(x) if want_y else None
    h = _new(x) if want_h else None
    stats = x.new_empty((rows, 2), dtype=torch.float32) if save else None
    if rows == 0:
        return y, h, stats
    (x, ldx), (f, ldf), (gate, ldg) = _rows(x), _rows(f), _rows(gate)
    rho, w_post, w_pre = _packed(residual_scale), _packed(w_post), _packed(w_pre)
    _call(x.device, 'vqa_norm_gate_fwd', x.data_ptr(), ldx, _ptr(f), ldf, _ptr(gate), ldg, per, _ptr(rho), _ptr(w_post), _ptr(w_pre),
          eps, _ptr(y), D, _ptr(h), D, _ptr(stats), rows, D, dt)
    return y, h, stats


def norm_gate_bwd(dy, dh, x, stats, f=None, gate=None, residual_scale=None, w_post=None, w_pre=None):
    """Gradients of ``norm_gate_fwd`` from dy and dh (either None: zero): (dx, df, dgate, dresidual_scale, dw_post,
    dw_pre), None for what was not given (dgate in the gate's shape, summed over the rows that share a gate row)."""
    name = 'norm_gate'
    dt, D, rows, per = _norm_operands(name, x, f, gate, residual_scale, w_post, w_pre)
    _need(dy is not None or dh is not None, '{}: one of dy, dh is needed', name)
    _need(dy is None or f is not None, '{}: without f there is no y, so no dy', name)
    for what, g in (('dy', dy), ('dh', dh)):
        if g is not None:
            _like(name, what, g, x, x.shape)
    _like(name, 'stats', stats, x, (rows, 2), torch.float32)

    dx, df, dgate = _new(x), _new(f), _new(gate)
    drho, dw_post, dw_pre = _new(residual_scale), _new(w_post), _new(w_pre)
    if rows == 0:
        for g in (drho, dw_post, dw_pre, dgate):
            if g is not None:
                g.zero_()
        return dx, df, dgate, drho, dw_post, dw_pre
    (x, ldx), (f, ldf), (gate, ldg), (dy, lddy), (dh, lddh) = _rows(x), _rows(f), _rows(gate), _rows(dy), _rows(dh)
    rho, w_post, w_pre, stats = _packed(residual_scale), _packed(w_post), _packed(w_pre), _packed(stats)
    ws = _workspace(_floats('vqa_norm_gate_workspace_floats', rows, D, per), x)
    _call(x.device, 'vqa_norm_gate_bwd', _ptr(dy), lddy, _ptr(dh), lddh, x.data_ptr(), ldx, _ptr(f), ldf, _ptr(gate), ldg, per,
          _ptr(rho), _ptr(w_post), _ptr(w_pre), stats.data_ptr(), dx.data_ptr(), D, _ptr(df), D, _ptr(dgate), D,
          _ptr(drho), _ptr(dw_post), _ptr(dw_pre), ws.data_ptr(), rows, D, dt)
    return dx, df, dgate, drho, dw_post, dw_pre


class _NormGate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, f, gate, residual_scale, w_post, w_pre, eps):
        y, h, stats = norm_gate_fwd(x, f, gate, residual_scale, w_post, w_pre, eps, save=any(ctx.needs_input_grad))
        ctx.save_for_backward(x, f, gate, residual_scale, w_post, w_pre, stats)
        ctx.set_materialize_grads(False)
        return y, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy, dh):
        x, f, gate, residual_scale, w_post, w_pre, stats = ctx.saved_tensors
        if dy is None and dh is None:
            return (None,) * 7
        return (*norm_gate_bwd(dy, dh, x, stats, f, gate, residual_scale, w_post, w_pre), None)


def norm_gate(x, f=None, gate=None, residual_scale=None, w_post=None, w_pre=None, eps=1e-6):
    """Differentiable ``norm_gate_fwd``: (y, h); y is None when f is."""
    return _NormGate.apply(x, f, gate, residual_scale, w_post, w_pre, eps)


# ---- cross attention -----------------------------------------------------------------------------

def _view(t):
    """(tensor, VqaAttnView) of a (B, T, H, D) operand, copied if the kernels cannot read its strides."""
    sb, st, sh, one = t.stride()
    nb, nt, nh, D = t.shape                                      # the stride of a size of 1 says nothing
    sb, st, sh = sb if nb > 1 else 0, st if nt > 1 else 0, sh if nh > 1 else 0
    if one != 1 or (sb | st | sh) % 8 or sb < 0 or st < 0 or sh < 0 or st >= 1 << 25 or t.data_ptr() % 16:
        t = t.clone(memory_format=torch.contiguous_format)
        sb, st, sh, one = t.stride()
    return t, _lib.AttnView(t.data_ptr(), sb, st, sh)


def _attn_operands(q, k, v, kv_len, mask, scale):
    name = 'cross_attention'
    dt = _storage(name, q)
    _need(q.dim() == 4 and k.dim() == 4, '{}: q is (B, Tq, H, D), k and v are (B, Tk, Hkv, D)', name)
    B, Tq, H, D = q.shape
    _, Tk, Hkv, _ = k.shape
    _like(name, 'k', k, q, (B, Tk, Hkv, D))
    _like(name, 'v', v, q, (B, Tk, Hkv, D))
    _need(Hkv > 0 and H > 0 and H % Hkv == 0, '{}: {} query heads cannot share {} key heads evenly', name, H, Hkv)
    _need(D % 8 == 0 and 8 <= D <= 128, '{}: the head width must be a multiple of 8 in [8, 128], got {}', name, D)
    mask_sb = 0
    if mask is not None:
        _need(mask.shape == (B, Tk) and mask.device == q.device and mask.dtype in (torch.bool, torch.uint8),
              '{}: mask must be ({}, {}) bool or uint8 on {}', name, B, Tk, q.device)
        if Tk > 1 and mask.stride(1) != 1:
            mask = mask.contiguous()
        mask_sb = mask.stride(0)
    scale = D ** -0.5 if scale is None else float(scale)
    _need(math.isfinite(scale), '{}: scale must be finite, got {}', name, scale)
    return dt, _lengths(name, 'kv_len', kv_len, q, B), mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D


def cross_attention_fwd(q, k, v, kv_len=None, mask=None, scale=None, save=True):
    """softmax(scale q k^T) v of the token rows ``q`` (B, Tq, H, D) over the regions ``k``, ``v`` (B, Tk, Hkv, D); head h
    reads key head h // (H // Hkv).

    ``kv_len`` (B,): regions of each sample; ``mask`` (B, Tk): regions that count (True); what does not count
    may hold anything.  ``scale`` (finite) defaults to D ** -0.5.  Returns o (B, Tq, H, D), a row with nothing to attend 0, and what
    ``cross_attention_bwd`` needs (None unless ``save``): the log-sum-exp of the scores (B, H, Tq) float32, -inf for such a
    row, and for bfloat16 what rounding took from o."""
    dt, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D = _attn_operands(q, k, v, kv_len, mask, scale)
    dev = q.device
    o = _new(q)
    lse = q.new_empty((B, H, Tq), dtype=torch.float32) if save else None
    rest = _new(q) if save and dt == _lib.BF16 else None
    if B == 0 or Tq == 0 or Tk == 0:
        return o.zero_(), (lse.fill_(float('-inf')), rest if rest is None else rest.zero_()) if save else None
    (q, vq), (k, vk), (v, vv) = _view(q), _view(k), _view(v)
    ws = _workspace(_floats('vqa_cross_attn_fwd_workspace_floats', B, Tq, Tk, H, Hkv, D, dt), q)
    _call(dev, 'vqa_cross_attn_fwd', byref(vq), byref(vk), byref(vv), _ptr(kv_len), _ptr(mask), mask_sb, scale, o.data_ptr(),
          _ptr(rest), _ptr(lse), _ptr(ws), B, Tq, Tk, H, Hkv, D, dt)
    return o, (lse, rest) if save else None


def cross_attention_bwd(do, q, k, v, o, saved, kv_len=None, mask=None, scale=None):
    """Gradients (dq, dk, dv) of ``cross_attention_fwd`` from do (B, Tq, H, D) and the two things it returned."""
    dt, kv_len, mask, mask_sb, scale, B, Tq, Tk, H, Hkv, D = _attn_operands(q, k, v, kv_len, mask, scale)
    dev = q.device
    _like('cross_attention', 'do', do, q, q.shape)
    _like('cross_attention', 'o', o, q, q.shape)
    _need(saved is not None, 'cross_attention: the backward needs what cross_attention_fwd(..., save=True) returned')
    lse, rest = saved
    _like('cross_attention', 'the saved log-sum-exp', lse, q, (B, H, Tq), torch.float32)
    if rest is not None:
        _like('cross_attention', "the saved rest of o", rest, q, q.shape)
    dq, dk, dv = _new(q), _new(k), _new(v)
    if B == 0 or Tq == 0 or Tk == 0:
        return dq.zero_(), dk.zero_(), dv.zero_()
    (q, vq), (k, vk), (v, vv) = _view(q), _view(k), _view(v)
    do, o, lse, rest = _packed(do), _packed(o), _packed(lse), _packed(rest)
    ws = _workspace(_floats('vqa_cross_attn_bwd_workspace_floats', B, Tq, Tk, H, Hkv, D, dt), q)
    _call(dev, 'vqa_cross_attn_bwd', do.data_ptr(), byref(vq), byref(vk), byref(vv), o.data_ptr(), _ptr(rest), lse.data_ptr(),
          _ptr(kv_len), _ptr(mask), mask_sb, scale, dq.data_ptr(), dk.data_ptr(), dv.data_ptr(), _ptr(ws), B, Tq, Tk, H, Hkv, D, dt)
    return dq, dk, dv


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, kv_len, mask, scale):
        o, saved = cross_attention_fwd(q, k, v, kv_len, mask, scale, save=any(ctx.needs_input_grad[:3]))
        ctx.save_for_backward(q, k, v, o, *(saved or (None, None)), kv_len, mask)
        ctx.scale = scale
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        q, k, v, o, lse, rest, kv_len, mask = ctx.saved_tensors
        return (*cross_attention_bwd(do, q, k, v, o, (lse, rest), kv_len, mask, ctx.scale), None, None, None)


def cross_attention(q, k, v, kv_len=None, mask=None, scale=None):
    """Differentiable ``cross_attention_fwd``: o alone."""
    return _CrossAttention.apply(q, k, v, kv_len, mask, scale)

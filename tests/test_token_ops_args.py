"""Refusals of the token-level operators.  The C entry points check their arguments before any HIP call, so they can be
tested without a GPU; the addresses below are never followed (every call is refused)."""
import ctypes as C
import os
import re

import pytest
import torch

from vqa_amd import _lib, ops

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
P = 1 << 20                       # an aligned address that nothing reads


def refused(name, *args):
    lib = _lib.load()
    rc = getattr(lib, name)(*args, None)
    assert rc == -22, (name, rc)
    text = lib.vqa_last_error_string().decode()
    assert name in text, text
    return text


def test_constants_agree_with_the_header():
    text = open(os.path.join(ROOT, 'include', 'vqa_hip.h')).read()
    assert int(re.search(r'#define VQA_GATED_SCAN_SAVE (\d+)', text).group(1)) == ops._SAVE
    assert int(re.search(r'#define VQA_CROSS_ATTN_MAX_D (\d+)', text).group(1)) == 128


SCAN = dict(gates=P, sb=64, st=32, lengths=None, c0=None, h=P, c=P, saved=None, ws=None, B=2, T=2, H=8, dtype=0)


@pytest.mark.parametrize('change', [dict(gates=None), dict(gates=P + 4), dict(st=24), dict(st=36), dict(sb=4), dict(sb=-64), dict(c0=P + 8),
                                    dict(h=None), dict(h=P + 2), dict(B=0), dict(T=0), dict(H=0), dict(H=12), dict(dtype=2), dict(T=(1 << 20) + 1),
                                    dict(B=1 << 20, H=1 << 12, st=1 << 14), dict(ws=P + 4), dict(B=1, T=4096, H=8)])
def test_scan_forward_refuses(change):
    refused('vqa_gated_scan_fwd', *{**SCAN, **change}.values())


def test_scan_backward_refuses():
    ok = dict(dh=P, dc=P, gates=P, sb=64, st=32, lengths=None, c0=None, saved=P, dgates=P, dc0=P, ws=None, B=2, T=2, H=8, dtype=0)
    for change in (dict(dh=None, dc=None), dict(dgates=None), dict(dh=P + 4), dict(saved=P + 4), dict(saved=None), dict(dtype=3), dict(gates=0)):
        refused('vqa_gated_scan_bwd', *{**ok, **change}.values())


NORM = dict(x=P, ldx=16, f=P, ldf=16, gate=P, ldg=16, per=2, rho=P, w_post=P, w_pre=P, eps=1e-6, y=P, ldy=16, h=P, ldh=16, stats=P,
            rows=4, D=16, dtype=1)


@pytest.mark.parametrize('change', [dict(D=12), dict(D=0), dict(D=8200), dict(rows=-1), dict(rows=(1 << 30) + 2), dict(per=0), dict(per=3), dict(x=None),
                                    dict(x=P + 2), dict(ldx=8), dict(ldx=20), dict(f=None), dict(y=None, h=None), dict(h=None),
                                    dict(eps=-1.0), dict(w_pre=P + 4), dict(dtype=2), dict(ldg=12)])
def test_norm_forward_refuses(change):
    refused('vqa_norm_gate_fwd', *{**NORM, **change}.values())


def test_norm_backward_refuses():
    ok = dict(dy=P, lddy=16, dh=P, lddh=16, x=P, ldx=16, f=P, ldf=16, gate=P, ldg=16, per=2, rho=P, w_post=P, w_pre=P, stats=P, dx=P, lddx=16,
              df=P, lddf=16, dgate=P, lddg=16, drho=P, dw_post=P, dw_pre=P, ws=P, rows=4, D=16, dtype=1)
    for change in (dict(dy=None, dh=None), dict(df=None), dict(dgate=None), dict(gate=None), dict(stats=None), dict(ws=None), dict(dx=None),
                   dict(rows=0), dict(D=20), dict(ws=P + 4), dict(lddf=8), dict(f=None)):
        refused('vqa_norm_gate_bwd', *{**ok, **change}.values())


def view(data=P, sb=1024, st=64, sh=16):
    return C.byref(_lib.AttnView(data, sb, st, sh))


ATTN = dict(q=view(), k=view(), v=view(), kv_len=None, mask=None, mask_sb=0, scale=0.25, o=P, rest=None, lse=P, ws=None, B=2, Tq=3, Tk=16, H=4,
            Hkv=2, D=16, dtype=1)


@pytest.mark.parametrize('change', [dict(D=12), dict(D=136), dict(D=0), dict(H=3), dict(Hkv=0), dict(B=0), dict(Tq=0), dict(Tk=0), dict(dtype=4),
                                    dict(q=None), dict(k=view(data=None)), dict(v=view(data=P + 8)), dict(k=view(st=20)), dict(q=view(sb=-64)),
                                    dict(k=view(st=1 << 25)), dict(o=None), dict(o=P + 2), dict(rest=P + 2), dict(Tk=(1 << 24) + 1),
                                    dict(Tq=1 << 27), dict(mask=P, mask_sb=-4), dict(B=1, Tk=100000), dict(scale=float('nan')), dict(scale=float('-inf')),
                                    dict(B=1 << 23, Tq=1), dict(B=1 << 17, Tq=1, Tk=3000)])
def test_attention_forward_refuses(change):
    refused('vqa_cross_attn_fwd', *{**ATTN, **change}.values())


def test_attention_backward_refuses():
    ok = dict(do=P, q=view(), k=view(), v=view(), o=P, rest=None, lse=P, kv_len=None, mask=None, mask_sb=0, scale=0.25, dq=P, dk=P, dv=P, ws=P, B=2,
              Tq=3, Tk=16, H=4, Hkv=2, D=16, dtype=1)
    for change in (dict(do=None), dict(o=None), dict(lse=None), dict(dq=None), dict(dk=P + 4), dict(dv=None), dict(D=10), dict(v=view(st=4)),
                   dict(Tq=40, Tk=64, ws=None), dict(ws=P + 4), dict(rest=P + 4), dict(scale=float('inf'))):
        refused('vqa_cross_attn_bwd', *{**ok, **change}.values())


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.vqa_gated_scan_workspace_floats(256, 14, 2400, 1) == 0 and lib.vqa_gated_scan_workspace_floats(1, 4096, 512, 1) > 0
    assert lib.vqa_gated_scan_saved_floats(2, 17, 8) == 3 * 2 * 8 and lib.vqa_gated_scan_saved_floats(2, 1, 8) == 2 * 8
    assert lib.vqa_norm_gate_workspace_floats(100, 64, 0) >= 3 * 64 and lib.vqa_norm_gate_workspace_floats(100, 64, 7) == 0
    assert lib.vqa_cross_attn_fwd_workspace_floats(256, 14, 196, 15, 15, 80, 1) == 0
    assert lib.vqa_cross_attn_fwd_workspace_floats(1, 1, 4096, 8, 2, 64, 1) > 0
    assert lib.vqa_cross_attn_bwd_workspace_floats(2, 40, 64, 4, 2, 64, 0) >= 2 * 40 * 4
    assert lib.vqa_cross_attn_fwd_workspace_floats(1, 1, 4096, 8, 3, 64, 1) == 0        # sizes that are refused


def test_cpu_tensors_are_refused():
    x, g, q = torch.zeros(2, 3, 16), torch.zeros(2, 3, 32), torch.zeros(2, 3, 2, 8)
    for call in (lambda: ops.gated_scan(g), lambda: ops.norm_gate(x), lambda: ops.cross_attention(q, q, q)):
        with pytest.raises(_lib.VqaHipError, match='cuda'):
            call()


def test_scan_backward_reads_saved_states_as_they_were_saved(monkeypatch):
    """Saved states of another type or shape are refused before any call; strided ones are packed for it."""
    monkeypatch.setattr(ops, '_storage', lambda name, t: _lib.F32)
    calls = []
    monkeypatch.setattr(ops, '_call', lambda device, name, *args: calls.append(args))
    gates, dh = torch.zeros(2, 9, 32), torch.zeros(2, 9, 8)
    saved = torch.zeros(2, 2, 8)
    for bad in (saved.bfloat16(), saved.half(), saved.double(), saved[:1], saved[..., :4], None):
        with pytest.raises(ValueError, match='gated_scan'):
            ops.gated_scan_bwd(dh, None, gates, bad)
    assert not calls
    wide = torch.arange(64.0).reshape(2, 2, 16)[..., ::2]                    # in place it would be read past its steps
    ops.gated_scan_bwd(dh, None, gates, wide)
    assert len(calls) == 1 and calls[0][7] != wide.data_ptr()
    ops.gated_scan_bwd(dh, None, gates, saved)
    assert calls[1][7] == saved.data_ptr()

"""The token-level operators as they are used: together in a block, captured in a graph, on side streams and threads, and
what they refuse."""
import threading

import pytest
import torch

from _token_ref import attention, close, norm_gate, scan

pytestmark = pytest.mark.gpu


def _block(p, tokens, regions, lengths, kv_len, f):
    """A question's tokens through one block: the recurrence mixes them, the norms join, the attention reads the image.
    `f` names the operators: the package's, or the plain 64-bit ones."""
    B, T, D = tokens.shape
    H = p['heads']
    x, n = tokens, f['norm'](tokens, w_pre=p['w0'])[1]
    h = f['scan']((n @ p['w_gates']), lengths)[0]
    x, n = f['norm'](x, f=h, gate=p['g1'], rho=p['rho1'], w_post=p['w1'], w_pre=p['w2'])
    q = (n @ p['w_q']).reshape(B, T, H, -1)
    kv = (regions @ p['w_kv']).reshape(B, regions.shape[1], 2, H // 2, -1)
    o = f['attn'](q, kv[:, :, 0], kv[:, :, 1], kv_len).reshape(B, T, -1)
    return f['norm'](x, f=o, gate=p['g2'], rho=p['rho2'], w_post=p['w3'], w_pre=p['w4'])


def _params(B, T, D, Dv, H, dtype, seed):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def r(*s, mul=1.0, dt=dtype):
        return (torch.randn(*s, device='cuda', generator=g) * mul).to(dt)

    p = dict(w_gates=r(D, 4 * D, mul=D ** -0.5), w_q=r(D, D, mul=D ** -0.5), w_kv=r(Dv, D, mul=Dv ** -0.5), g1=r(B, 1, D), g2=r(B, T, D))
    for n in ('w0', 'w1', 'w2', 'w3', 'w4', 'rho1', 'rho2'):
        p[n] = (1 + r(D, mul=0.1, dt=torch.float32))
    return p, r(B, T, D), r(B, 21, Dv)


def test_a_block_of_all_three_matches_64_bits():
    """fp32, forward and every gradient.  Seven operators and products deep, each good to 2e-5 of its largest value, with
    slopes of order one between them: 1e-3 of the largest value is generous and far below any wrong term."""
    from vqa_amd import ops
    B, T, D, Dv, H = 3, 9, 32, 48, 4
    p, tokens, regions = _params(B, T, D, Dv, H, torch.float32, 1)
    lengths = torch.tensor([9, 4, 1], device='cuda', dtype=torch.int32)
    kv_len = torch.tensor([21, 13, 5], device='cuda', dtype=torch.int32)
    ours = dict(norm=lambda x, rho=None, **k: ops.norm_gate(x, residual_scale=rho, **k), scan=ops.gated_scan, attn=ops.cross_attention)
    plain = dict(norm=norm_gate, scan=scan, attn=lambda *a: attention(*a)[0])

    def run(f, dt):
        q = {n: v.detach().to(dt).requires_grad_(True) for n, v in p.items()}
        t, r = tokens.detach().to(dt).requires_grad_(True), regions.detach().to(dt).requires_grad_(True)
        y, h = _block({**q, 'heads': H}, t, r, lengths, kv_len, f)
        g = torch.Generator(device='cuda').manual_seed(2)
        loss = (y * torch.randn(y.shape, device='cuda', generator=g).to(dt)).sum() + (h * torch.randn(h.shape, device='cuda', generator=g).to(dt)).sum()
        loss.backward()
        return {'y': y, 'h': h, 'tokens': t.grad, 'regions': r.grad, **{n: v.grad for n, v in q.items()}}

    got, ref = run(ours, torch.float32), run(plain, torch.float64)
    for n in ref:
        close(got[n], ref[n], 1e-3 * max(1.0, float(ref[n].detach().abs().max())), n)


def _calls(dtype):
    """One forward and backward of each operator, sizes that need every workspace: a list of functions of their inputs."""
    from vqa_amd import ops
    g = torch.Generator(device='cuda').manual_seed(3)

    def r(*s, dt=dtype):
        return torch.randn(*s, device='cuda', generator=g).to(dt)

    gates, c0, dh, dc = r(2, 700, 4 * 64), r(2, 64, dt=torch.float32), r(2, 700, 64), r(2, 64, dt=torch.float32)
    lengths = torch.tensor([700, 433], device='cuda', dtype=torch.int32)
    x, f, gate, dy = r(2, 600, 72), r(2, 600, 72), r(2, 1, 72), r(2, 600, 72)
    w = [r(72, dt=torch.float32) for _ in range(3)]
    q, k, v, do = r(1, 2, 4, 64), r(1, 1500, 2, 64), r(1, 1500, 2, 64), r(1, 2, 4, 64)
    q2, do2 = r(1, 90, 4, 64), r(1, 90, 4, 64)

    def scan_():
        h, c, saved = ops.gated_scan_fwd(gates, lengths, c0)
        return [h, c, *ops.gated_scan_bwd(dh, dc, gates, saved, lengths, c0)]

    def norm_():
        kw = dict(f=f, gate=gate, residual_scale=w[0], w_post=w[1], w_pre=w[2])
        y, h, st = ops.norm_gate_fwd(x, **kw)
        return [y, h, *ops.norm_gate_bwd(dy, dy, x, st, **kw)]

    def attn_(q_=q, do_=do):
        o, saved = ops.cross_attention_fwd(q_, k, v)
        return [o, saved[0], *ops.cross_attention_bwd(do_, q_, k, v, o, saved)]

    return [gates, x, q, q2], [scan_, norm_, attn_, lambda: attn_(q2, do2)]


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_captured_and_replayed(dtype):
    """Each operator's forward and backward in a graph of its own, two graphs of each, replayed in turn with eager work
    between and on changed inputs: every replay equals the eager call, bit for bit."""
    inputs, calls = _calls(dtype)
    for call in calls:
        call()
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                out = call()
            graphs.append((g, out))
        for i in range(4):
            for t in inputs:
                t.mul_(0.75).add_(0.01 * i)
            eager = [t.clone() for t in call()]
            for g, out in graphs:
                g.replay()
            torch.cuda.synchronize()
            for g, out in graphs:
                for a, b in zip(out, eager):
                    assert torch.equal(a, b), i


def test_side_streams_and_threads():
    """Work goes to the calling thread's current stream, and two threads on two streams do not disturb each other."""
    _, calls = _calls(torch.bfloat16)
    want = [[t.clone() for t in c()] for c in calls]
    torch.cuda.synchronize()
    bad = []

    def work(order):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            for _ in range(5):
                for i in order:
                    got = calls[i]()
                    for a, b in zip(got, want[i]):
                        if not torch.equal(a, b):
                            bad.append(i)
        s.synchronize()

    threads = [threading.Thread(target=work, args=(o,)) for o in ([0, 1, 2, 3], [3, 2, 1, 0])]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad, bad


def test_work_follows_the_stream_it_is_called_on():
    """The operand is written by a long chain on the side stream; the operator called there sees the finished value."""
    from vqa_amd import _lib, ops
    _lib.bind_stream()                                       # what a model bound earlier does not matter
    x = torch.zeros(64, 512, 512, device='cuda')
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        for _ in range(200):
            x.add_(1.0)
        h = ops.norm_gate(x)[1]
    s.synchronize()
    assert float((h - 1).abs().max()) < 1e-5


def test_keys_far_apart():
    """Offsets past 32 bits: rows of keys 2^24 elements apart (5 GB of them), batches beyond."""
    from vqa_amd import ops
    st, Tk = 1 << 24, 80
    big = torch.empty(2 * Tk * st + 64, device='cuda', dtype=torch.bfloat16)
    k = big.as_strided((2, Tk, 1, 64), (Tk * st, st, 64, 1))
    g = torch.Generator(device='cuda').manual_seed(1)
    k.copy_(torch.randn(2, Tk, 1, 64, device='cuda', generator=g))
    for Tq in (2, 40):
        q = torch.randn(2, Tq, 2, 64, device='cuda', generator=g).to(torch.bfloat16)
        o, saved = ops.cross_attention_fwd(q, k, k)
        o2, saved2 = ops.cross_attention_fwd(q, k.contiguous(), k.contiguous())
        assert torch.equal(o, o2)
        for a, b in zip(ops.cross_attention_bwd(q, q, k, k, o, saved), ops.cross_attention_bwd(q, q, k.contiguous(), k.contiguous(), o, saved)):
            assert torch.equal(a, b)


def test_refusals():
    from vqa_amd import _lib, ops
    c = dict(device='cuda')
    x, f = torch.zeros(2, 3, 16, **c), torch.zeros(2, 3, 16, **c)
    q, k = torch.zeros(2, 3, 4, 16, **c), torch.zeros(2, 5, 2, 16, **c)
    gates = torch.zeros(2, 3, 64, **c)
    o, saved = ops.cross_attention_fwd(q, k, k)
    for call in (lambda: ops.norm_gate(torch.zeros(2, 12, **c)), lambda: ops.norm_gate(torch.zeros(1, 8200, **c)),
                 lambda: ops.norm_gate(x, f=f[:, :2]), lambda: ops.norm_gate(x, f=f.bfloat16()), lambda: ops.norm_gate(x, gate=x),
                 lambda: ops.norm_gate(x, f=f, gate=torch.zeros(3, 1, 16, **c)), lambda: ops.norm_gate(x, f=f, gate=torch.zeros(1, 3, 16, **c)),
                 lambda: ops.norm_gate(x, w_pre=torch.zeros(16, dtype=torch.bfloat16, **c)), lambda: ops.norm_gate(x, f=f, w_post=torch.zeros(8, **c)),
                 lambda: ops.norm_gate_fwd(x, want_h=False), lambda: ops.norm_gate_bwd(None, None, x, torch.zeros(6, 2, **c)),
                 lambda: ops.norm_gate_bwd(x, None, x, torch.zeros(6, 2, **c)), lambda: ops.norm_gate_bwd(None, x, x, torch.zeros(5, 2, **c)),
                 lambda: ops.gated_scan(torch.zeros(2, 3, 48, **c)), lambda: ops.gated_scan(gates[0]),
                 lambda: ops.gated_scan(gates, torch.zeros(3, dtype=torch.int32, **c)), lambda: ops.gated_scan(gates, torch.zeros(2, **c)),
                 lambda: ops.gated_scan(gates, None, torch.zeros(2, 8, **c)), lambda: ops.gated_scan(gates, None, torch.zeros(2, 16, dtype=torch.bfloat16, **c)),
                 lambda: ops.gated_scan_bwd(torch.zeros(2, 3, 16, **c), None, gates, None),
                 lambda: ops.cross_attention(q, k, k[:, :4]), lambda: ops.cross_attention(q[:, :, :3], k, k), lambda: ops.cross_attention(q, k.bfloat16(), k),
                 lambda: ops.cross_attention(torch.zeros(2, 3, 4, 12, **c), torch.zeros(2, 5, 2, 12, **c), torch.zeros(2, 5, 2, 12, **c)),
                 lambda: ops.cross_attention(torch.zeros(2, 3, 4, 136, **c), torch.zeros(2, 5, 2, 136, **c), torch.zeros(2, 5, 2, 136, **c)),
                 lambda: ops.cross_attention(q, k, k, mask=torch.ones(2, 4, dtype=torch.bool, **c)), lambda: ops.cross_attention(q, k, k, mask=torch.ones(2, 5, **c)),
                 lambda: ops.cross_attention(q, k, k, kv_len=torch.ones(2, dtype=torch.int32)),
                 lambda: ops.cross_attention(q, k, k, scale=float('nan')), lambda: ops.cross_attention_bwd(o, q, k, k, o, None), lambda: ops.cross_attention_bwd(o[:, :2], q, k, k, o, saved)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: ops.norm_gate(x.half()), lambda: ops.gated_scan(gates.double()), lambda: ops.cross_attention(q.half(), k.half(), k.half())):
        with pytest.raises(_lib.VqaHipError, match='dtype'):
            call()
    with pytest.raises(RuntimeError):                        # a second derivative is refused, not wrong
        xr = x.clone().requires_grad_(True)
        (g,) = torch.autograd.grad(ops.norm_gate(xr)[1].sum(), xr, create_graph=True)
        g.sum().backward()

"""The gated residual norms against the formula in 64 bits on the same inputs.

Error of the fp32 arithmetic: a sum over D <= 8192 columns is taken 8 to a thread, then in at most 6 + 16 additions, so
it is good to 30 x 2^-24 = 2e-6 of the sum of its terms' sizes; a row's values pass about ten more roundings.  Outputs
are therefore good to 5e-6 of the largest value of the row's terms, the gradients (two such sums deep) to 2e-5 of the
largest term that enters them; column sums over the rows to 2e-5 of the sum of their terms' sizes."""
import pytest
import torch

from _token_ref import close, norm_gate

pytestmark = pytest.mark.gpu


def _case(B, T, D, dtype, gate, seed, weights=True):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def r(*s, dt=dtype, add=0.0, mul=1.0):
        return (torch.randn(*s, device='cuda', generator=g) * mul + add).to(dt)

    kw = dict(f=r(B, T, D, mul=0.3))
    if gate:
        kw['gate'] = r(*{'row': (B, T, D), 'sample': (B, 1, D), 'flat': (B, D), 'all': (1, 1, D)}[gate])
    if weights:
        kw.update(residual_scale=r(D, dt=torch.float32, add=1, mul=0.2), w_post=r(D, dt=torch.float32, add=1, mul=0.2),
                  w_pre=r(D, dt=torch.float32, add=1, mul=0.2))
    return r(B, T, D, mul=2.0), kw, r(B, T, D), r(B, T, D)


def _check(x, kw, dy, dh):
    from vqa_amd import ops
    y, h, stats = ops.norm_gate_fwd(x, **kw)
    got = ops.norm_gate_bwd(dy, dh, x, stats, **kw)
    names = ['x'] + [n for n in ('f', 'gate', 'residual_scale', 'w_post', 'w_pre') if n in kw]
    leaf = {n: (x if n == 'x' else kw[n]).double().requires_grad_(True) for n in names}
    ref_kw = {('rho' if n == 'residual_scale' else n): v for n, v in leaf.items() if n != 'x'}
    yr, hr = norm_gate(leaf['x'], **ref_kw)
    outs, into = [hr], [dh.double()]
    if dy is not None:
        outs, into = [yr, hr], [dy.double(), dh.double()]
    ref = dict(zip(names, torch.autograd.grad(outs, [leaf[n] for n in names], into, allow_unused=True)))
    if 'f' in kw:
        close(y, yr, 5e-6 * (float(yr.abs().max()) + 3), 'y')
    close(h, hr, 5e-6 * (float(hr.abs().max()) + 3), 'h')
    big = float(max(ref['x'].abs().max(), ref['f'].abs().max() if 'f' in kw else 0)) + 1
    x2 = leaf['x'].detach()
    rho = leaf['residual_scale'].detach() if 'residual_scale' in leaf else 1.0
    dyt = ref['x'] / rho                                     # the gradient at y
    for n, v in zip(('x', 'f', 'gate', 'residual_scale', 'w_post', 'w_pre'), got):
        if n not in ref:
            assert v is None
            continue
        lead = tuple(range(x.dim() - 1))
        if n in ('x', 'f'):
            lim = 2e-5 * big
        elif n == 'gate':
            lim = 2e-5 * big * (4 + x.numel() / x.shape[-1] / max(1, kw['gate'].numel() // x.shape[-1]))
        elif n == 'residual_scale':
            lim = 2e-5 * (dyt * x2).abs().sum(lead) + 1e-6
        elif n == 'w_post':
            u = kw['f'].double()
            u = u / torch.sqrt((u * u).mean(-1, keepdim=True) + 1e-6)
            lim = 2e-5 * (dyt * u).abs().sum(lead) + 1e-6
        else:
            lim = 2e-5 * (dh.double() * hr.detach() / leaf['w_pre'].detach()).abs().sum(lead) + 1e-6
        close(v, ref[n], lim, n)
    again = ops.norm_gate_bwd(dy, dh, x, stats, **kw)
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize('B,T,D', [(1, 1, 8), (2, 3, 16), (3, 5, 24), (2, 7, 104), (1, 14, 1200), (5, 14, 520), (3, 33, 512),
                                   (2, 9, 1024), (2, 6, 2400), (1, 5, 8192), (4, 300, 64), (300, 2, 40), (2, 700, 136)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('gate', [None, 'row', 'sample', 'flat', 'all'])
def test_norm_gate_and_gradients_match_64_bits(B, T, D, dtype, gate):
    if gate == 'flat' and B == 1:
        gate = 'sample'
    _check(*_case(B, T, D, dtype, gate, B * 1000 + T + D))


@pytest.mark.parametrize('B,T,D', [(500, 200, 64), (1, 700000, 8), (1500, 4, 1024), (50, 50, 2400), (12, 50, 8192), (3000, 3, 64), (5000, 2, 136)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('gate', [None, 'row', 'sample', 'all'])
def test_workgroups_walk_over_rows(B, T, D, dtype, gate):
    """More rows than a launch holds at once, narrow and wide; several gate groups to a workgroup and several workgroups to
    a group."""
    _check(*_case(B, T, D, dtype, gate, 5))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_parts_alone(dtype):
    """No weights; the norm alone; y alone; h alone."""
    from vqa_amd import ops
    x, kw, dy, dh = _case(3, 10, 72, dtype, 'row', 1, weights=False)
    _check(x, kw, dy, dh)
    _check(x, {}, None, dh)
    _check(x, {'w_pre': torch.rand(72, device='cuda') + 0.5}, None, dh)
    y, h, st = ops.norm_gate_fwd(x, **kw)
    y1, h1, s1 = ops.norm_gate_fwd(x, **kw, want_h=False)
    y2, h2, s2 = ops.norm_gate_fwd(x, **kw, want_y=False, save=False)
    assert h1 is None and torch.equal(y, y1) and y2 is None and torch.equal(h, h2) and s2 is None
    # a zero gradient is the same as none
    z = torch.zeros_like(x)
    for a, b in (((dy, None), (dy, z)), ((None, dh), (z, dh))):
        for p, q in zip(ops.norm_gate_bwd(*a, x, st, **kw), ops.norm_gate_bwd(*b, x, st, **kw)):
            assert (p is None and q is None) or torch.equal(p, q)
    # w_pre's gradient without dh is zero
    w = torch.ones(72, device='cuda')
    y, h, st = ops.norm_gate_fwd(x, **kw, w_pre=w)
    assert float(ops.norm_gate_bwd(dy, None, x, st, **kw, w_pre=w)[5].abs().max()) == 0.0


def test_rows_of_any_stride():
    from vqa_amd import ops
    g = torch.Generator(device='cuda').manual_seed(4)
    wide = torch.randn(4, 6, 3 * 40, device='cuda', generator=g).to(torch.bfloat16)
    x, f = wide[:, :, 40:80], wide[:, :, 80:]                # rows of 40 at a pitch of 120: read in place
    want = ops.norm_gate_fwd(x.contiguous(), f=f.contiguous())
    for a, b in ((x, f), (x.transpose(0, 1).contiguous().transpose(0, 1), f), (wide[:, :, 40:80].clone()[:, :, :], f)):
        y, h, st = ops.norm_gate_fwd(a, f=b)
        assert torch.equal(y, want[0]) and torch.equal(h, want[1]) and torch.equal(st, want[2])
    odd = torch.empty(4 * 6 * 40 + 1, device='cuda', dtype=torch.bfloat16)[1:].view(4, 6, 40).copy_(x)
    assert torch.equal(ops.norm_gate_fwd(odd, f=f)[0], want[0])
    one = x[:1, :1].expand(4, 6, 40)
    assert torch.equal(ops.norm_gate_fwd(one)[1], ops.norm_gate_fwd(one.contiguous())[1])


def test_zero_rows_and_zero_inputs():
    from vqa_amd import ops
    y, h, st = ops.norm_gate_fwd(torch.zeros(0, 5, 16, device='cuda'), f=torch.zeros(0, 5, 16, device='cuda'))
    assert y.shape == h.shape == (0, 5, 16) and st.shape == (0, 2)
    x = torch.zeros(2, 3, 16, device='cuda')
    w = torch.ones(16, device='cuda')
    y, h, st = ops.norm_gate_fwd(x, f=x, w_pre=w)
    assert float(y.abs().max()) == 0 and float(h.abs().max()) == 0       # eps keeps 0 / 0 away
    g = ops.norm_gate_bwd(torch.ones_like(x), torch.ones_like(x), x, st, f=x, w_pre=w)
    assert all(bool(torch.isfinite(v).all()) for v in g if v is not None)
    e = torch.zeros(0, 5, 16, device='cuda')
    g = ops.norm_gate_bwd(e, e, e, torch.zeros(0, 2, device='cuda'), f=e, w_pre=w)
    assert float(g[5].abs().max()) == 0 and g[0].shape == e.shape


def test_gradient_against_differences():
    """Central differences of the fp32 forward along a random direction, step 1e-3: truncation below 1e-6 of the
    gradient's norm, noise (n outputs good to 1e-6, summed at random) / (2 step) below 1e-3 of it."""
    from vqa_amd import ops
    x, kw, dy, dh = _case(3, 4, 64, torch.float32, 'sample', 8)
    names = ['x', *kw]
    leaves = [x.requires_grad_(True)] + [kw[n].requires_grad_(True) for n in kw]

    def loss(vals):
        y, h = ops.norm_gate(vals[0], **dict(zip(names[1:], vals[1:])))
        return (y.double() * dy.double()).sum() + (h.double() * dh.double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    g = torch.Generator(device='cuda').manual_seed(3)
    with torch.no_grad():
        for k, n in enumerate(names):
            v = torch.randn(leaves[k].shape, device='cuda', generator=g)
            vals = [t.detach() for t in leaves]
            up, dn = list(vals), list(vals)
            up[k], dn[k] = vals[k] + 1e-3 * v, vals[k] - 1e-3 * v
            num = float((loss(up) - loss(dn)) / 2e-3)
            ana = float((grads[k].double() * v.double()).sum())
            assert abs(num - ana) <= 1e-2 * float(grads[k].norm()), (n, num, ana)

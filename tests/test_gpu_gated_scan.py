"""The gated linear recurrence against a step-by-step loop in 64 bits on the same inputs.

Error of the fp32 arithmetic: a step computes s(f) c + s(i) tanh(g) with about ten roundings of 2^-24 relative to
|c| + 1 and three exponentials good to 2^-22 absolute: below 1e-6 (|c| + 1) per step, and what a step adds shrinks by
the next forget gates, whose product over the inputs used here (gates N(0, 1), forget gates N(1, 1), mean 0.7) sums to
well under 20 steps.  So c is good to 2e-5 (1 + max |c|); h = s(o) tanh(c) inherits that bound (slopes at most 1).  The
gradients sum over as many steps the same way with factors of at most 1 from the saturating functions, so they are good
to 2e-5 (1 + max |c|) times the largest gradient that enters (max |dc| over the run)."""
import pytest
import torch

from _token_ref import HALF, close, scan

pytestmark = pytest.mark.gpu


def _inputs(B, T, H, dtype, seed, ragged, state):
    g = torch.Generator(device='cuda').manual_seed(seed)
    gates = torch.randn(B, T, 4, H, device='cuda', generator=g)
    gates[:, :, 1] += 1.0
    gates = gates.reshape(B, T, 4 * H).to(dtype)
    lengths = torch.randint(0, T + 1, (B,), device='cuda', generator=g, dtype=torch.int32) if ragged else None
    if ragged and B > 1:
        lengths[0], lengths[-1] = 0, T
    c0 = torch.randn(B, H, device='cuda', generator=g) if state else None
    dh = torch.randn(B, T, H, device='cuda', generator=g).to(dtype)
    dc = torch.randn(B, H, device='cuda', generator=g)
    return gates, lengths, c0, dh, dc


@pytest.mark.parametrize('B,T,H', [(1, 1, 8), (3, 1, 24), (2, 2, 8), (4, 14, 40), (5, 15, 72), (3, 16, 64), (3, 17, 64),
                                   (2, 33, 16), (1, 64, 2400), (2, 65, 136), (1, 577, 96), (7, 130, 8), (1, 1201, 200)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('ragged,state', [(False, True), (True, False), (True, True)])
def test_scan_and_gradients_match_64_bits(B, T, H, dtype, ragged, state):
    from vqa_amd import ops
    gates, lengths, c0, dh, dc = _inputs(B, T, H, dtype, B * 100 + T, ragged, state)
    if lengths is not None:                                  # what lies behind a sequence is not read
        behind = torch.arange(T, device='cuda')[None, :] >= lengths[:, None]
        gates[behind] = float('nan')
        dh[behind] = float('inf')
    h, c, saved = ops.gated_scan_fwd(gates, lengths, c0)
    dgates, dc0 = ops.gated_scan_bwd(dh, dc, gates, saved, lengths, c0)

    clean = gates if lengths is None else torch.where(behind[:, :, None], torch.zeros_like(gates), gates)
    gd = clean.double().requires_grad_(True)
    cd = (c0.double() if c0 is not None else torch.zeros(B, H, device='cuda', dtype=torch.float64)).requires_grad_(True)
    hr, cr = scan(gd, lengths, cd)
    dhd = dh.double() if lengths is None else torch.where(behind[:, :, None], torch.zeros_like(dh), dh).double()
    rg, rc = torch.autograd.grad((hr, cr), (gd, cd), (dhd, dc.double()))
    top = 1 + max(float(cd.detach().abs().max()), float(cr.detach().abs().max()), 2.0)
    close(c, cr, 2e-5 * top, 'c')
    close(h, hr, 2e-5 * top, 'h')
    enter = 20 * max(1.0, float(dhd.abs().max()) if dhd.numel() else 1.0)
    close(dgates, rg, 2e-6 * top * enter, 'dgates')
    close(dc0, rc, 2e-6 * top * enter, 'dc0')
    if lengths is not None:
        assert float(h[behind].abs().sum()) == 0.0 and float(dgates[behind].abs().sum()) == 0.0
    # the same inputs give the same bits
    h2, c2, saved2 = ops.gated_scan_fwd(gates, lengths, c0)
    dg2, dc02 = ops.gated_scan_bwd(dh, dc, gates, saved2, lengths, c0)
    assert torch.equal(h, h2) and torch.equal(c, c2) and torch.equal(dgates, dg2) and torch.equal(dc0, dc02)


@pytest.mark.parametrize('T,H', [(5000, 24), (17000, 8)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_runs_of_several_chunks(T, H, dtype):
    """Time cut into 79 and 266 chunks: the chain's 32 runs hold up to 3 and 9 maps each."""
    test_scan_and_gradients_match_64_bits(1, T, H, dtype, False, True)
    test_scan_and_gradients_match_64_bits(2, T // 2, H, dtype, True, False)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_single_steps_continue_a_sequence(dtype):
    """T = 1 calls that hand the state on against one call over all steps: the same bits for the first 8 steps, which one
    wave walks from the same state; from there on the one call starts from P c + C, the first 8 steps as one map, which
    rounds 8 x 3 times where the steps round 8 x 2 times: 40 x 2^-24 of 1 + |c| apart at most.  A stored h may then fall
    on the other side of a rounding border: one step of its type."""
    from vqa_amd import ops
    gates, _, c0, _, _ = _inputs(3, 13, 48, dtype, 5, False, True)
    h, c, _ = ops.gated_scan_fwd(gates, None, c0, save=False)
    st, hs = c0, []
    for t in range(13):
        ht, st, none = ops.gated_scan_fwd(gates[:, t:t + 1], None, st, save=False)   # a strided view of the gates
        assert none is None
        hs.append(ht)
    hs = torch.cat(hs, 1)
    assert torch.equal(hs[:, :8], h[:, :8])
    apart = 40 * 2.0 ** -24 * (1 + float(c0.abs().max()) + 13)
    assert float((st - c).abs().max()) <= apart
    assert bool(((hs.double() - h.double()).abs() <= apart + 2 * HALF[dtype] * h.double().abs()).all())


def test_strided_and_unaligned_gates():
    from vqa_amd import ops
    g = torch.Generator(device='cuda').manual_seed(3)
    B, T, H = 3, 11, 24
    big = torch.randn(T, B, 4 * H + 16, device='cuda', generator=g).to(torch.bfloat16)
    view = big[:, :, 8:8 + 4 * H].transpose(0, 1)            # time-major storage, padded rows: read in place
    want = ops.gated_scan_fwd(view.contiguous())[0]
    assert torch.equal(ops.gated_scan_fwd(view)[0], want)
    odd = torch.empty(B * T * 4 * H + 1, device='cuda', dtype=torch.bfloat16)[1:].view(B, T, 4 * H)
    odd.copy_(view)                                          # address not a multiple of 16 bytes: copied
    assert torch.equal(ops.gated_scan_fwd(odd)[0], want)
    wide = torch.randn(B, T, 8 * H, device='cuda', generator=g)
    assert torch.equal(ops.gated_scan_fwd(wide[:, :, ::2])[0], ops.gated_scan_fwd(wide[:, :, ::2].contiguous())[0])


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_strides_that_say_nothing(dtype):
    """A size of 1 may have any stride: one step of one sample out of padded rows, one sample out of a padded batch."""
    from vqa_amd import ops
    H = 8
    g = torch.Generator(device='cuda').manual_seed(6)
    for base, take in ((torch.randn(1, 5, 4 * H + 4, device='cuda', generator=g), lambda x: x[:, 2:3, :4 * H]),
                       (torch.randn(3, 2 * 4 * H + 4, device='cuda', generator=g), lambda x: x[:1, :2 * 4 * H].view(1, 2, 4 * H)),
                       (torch.randn(3, 4 * H + 3, device='cuda', generator=g), lambda x: x[1:2, None, :4 * H])):
        gates = take(base.to(dtype))
        plain = torch.empty(gates.shape, device='cuda', dtype=dtype).copy_(gates)
        a, b = ops.gated_scan_fwd(gates), ops.gated_scan_fwd(plain)
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        for x, y in zip(ops.gated_scan_bwd(a[0], a[1], gates, a[2]), ops.gated_scan_bwd(b[0], b[1], plain, b[2])):
            assert torch.equal(x, y)


@pytest.mark.parametrize('B,T,H', [(3, 24, 40), (1, 300, 8)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('size', [0.03, 1e-2, 1e-4, 1e-6])
def test_small_states_keep_their_digits(B, T, H, dtype, size):
    """Candidates and states of a size far below 1.  Everything is positive and the gates lie within +-2, so nothing
    cancels and every result is good to a RELATIVE bound: a logistic or hyperbolic value to 2^-21, 1 - s(x) >= 0.12 to
    2^-18, and each of the T steps multiplies by a forget gate (2^-21) and adds (2^-24): 2^-19 T + 2^-16 covers both directions."""
    from vqa_amd import ops
    g = torch.Generator(device='cuda').manual_seed(31)
    gates = torch.randn(B, T, 4, H, device='cuda', generator=g).clamp(-2, 2)
    gates[:, :, 2] = size * (0.5 + torch.rand(B, T, H, device='cuda', generator=g))
    gates = gates.reshape(B, T, 4 * H).to(dtype)
    c0 = size * (0.5 + torch.rand(B, H, device='cuda', generator=g))
    dh = (0.5 + torch.rand(B, T, H, device='cuda', generator=g)).to(dtype)
    dc = 0.5 + torch.rand(B, H, device='cuda', generator=g)
    h, c, saved = ops.gated_scan_fwd(gates, None, c0)
    dgates, dc0 = ops.gated_scan_bwd(dh, dc, gates, saved, None, c0)
    gd, cd = gates.double().requires_grad_(True), c0.double().requires_grad_(True)
    hr, cr = scan(gd, None, cd)
    ref = torch.autograd.grad((hr, cr), (gd, cd), (dh.double(), dc.double()))
    unit = 2.0 ** -19 * T + 2.0 ** -16
    for what, x, r in (('c', c, cr), ('h', h, hr), ('dgates', dgates, ref[0]), ('dc0', dc0, ref[1])):
        close(x, r, unit * r.detach().abs(), what)


def test_gradient_against_differences():
    """Directional derivative of the fp32 forward by central differences.  Step e = 1e-2: the third derivative of the
    loss along a unit direction is of the order of the gradient's norm, so the truncation is below e^2 of it, and the
    noise of the loss (n values of size 1, 1e-6 each, random) over 2 e is below 1e-4 sqrt(n) / sqrt(n)."""
    from vqa_amd import ops
    gates, _, c0, dh, dc = _inputs(2, 40, 64, torch.float32, 11, False, True)
    lengths = torch.tensor([40, 23], device='cuda', dtype=torch.int32)
    leaves = [gates.requires_grad_(True), c0.requires_grad_(True)]

    def loss(gt, c):
        h, cl = ops.gated_scan(gt, lengths, c)
        return (h.double() * dh.double()).sum() + (cl.double() * dc.double()).sum()

    grads = torch.autograd.grad(loss(*leaves), leaves)
    g = torch.Generator(device='cuda').manual_seed(12)
    for k in range(2):
        v = torch.randn(leaves[k].shape, device='cuda', generator=g)
        e = 1e-2
        with torch.no_grad():
            a = [x.detach() for x in leaves]
            up, dn = list(a), list(a)
            up[k], dn[k] = a[k] + e * v, a[k] - e * v
            num = float((loss(*up) - loss(*dn)) / (2 * e))
        ana = float((grads[k].double() * v.double()).sum())
        assert abs(num - ana) <= 2e-3 * float(grads[k].norm()), (k, num, ana)


def test_only_some_gradients_arrive():
    from vqa_amd import ops
    gates, lengths, c0, dh, dc = _inputs(3, 37, 32, torch.float32, 9, True, True)
    h, c, saved = ops.gated_scan_fwd(gates, lengths, c0)
    both = ops.gated_scan_bwd(dh, dc, gates, saved, lengths, c0)
    zero_h, zero_c = torch.zeros_like(dh), torch.zeros_like(dc)
    for a, b in (((dh, None), (dh, zero_c)), ((None, dc), (zero_h, dc))):
        x, y = ops.gated_scan_bwd(*a, gates, saved, lengths, c0), ops.gated_scan_bwd(*b, gates, saved, lengths, c0)
        assert torch.equal(x[0], y[0]) and torch.equal(x[1], y[1])
    assert both[0].shape == gates.shape
    gl = gates.clone().requires_grad_(True)
    hh, _ = ops.gated_scan(gl, lengths)                      # no state, last state unused
    hh.float().sum().backward()
    assert bool(torch.isfinite(gl.grad).all())


def test_empty_and_oversized_lengths():
    from vqa_amd import ops
    gates = torch.randn(2, 5, 32, device='cuda')
    c0 = torch.randn(2, 8, device='cuda')
    over = torch.tensor([99, -4], device='cuda', dtype=torch.int32)         # clamped to [0, T]
    same = torch.tensor([5, 0], device='cuda', dtype=torch.int64)
    a, b = ops.gated_scan_fwd(gates, over, c0), ops.gated_scan_fwd(gates, same, c0)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and torch.equal(a[1][1], c0[1])
    h, c, _ = ops.gated_scan_fwd(gates[:, :0], None, c0)
    assert h.shape == (2, 0, 8) and torch.equal(c, c0)
    h, c, saved = ops.gated_scan_fwd(gates[:0])
    assert h.shape == (0, 5, 8) and c.shape == (0, 8)
    dg, dc0 = ops.gated_scan_bwd(h, c, gates[:0], saved)
    assert dg.shape == (0, 5, 32) and dc0.shape == (0, 8)

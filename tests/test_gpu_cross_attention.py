"""Cross attention against the definition in 64 bits on the same inputs, one sample after the other over the regions
that count.

fp32: a score is a sum of D <= 128 products (relative 128 x 2^-24 at worst, 1e-6 of |q||k| scale in practice) and enters an
exponential, p is good to about 2^-21 (1 + |z|); sums over the regions keep that.  Inputs are N(0, 1), |z| < 8: outputs
are good to 1e-5 of the largest value that is averaged (5), gradients to 1e-5 of the largest term size times the sums
they are, stated below as 2e-5 x (sum of |terms|), computed from the 64-bit form.
bf16: p and ds are rounded to bf16 for their products: 2^-8 of each TERM at most, so an output is good to 2^-8 x (sum of
|terms|) where the terms are p v, p dO, ds q, ds k; o enters delta = sum dO o rounded (2^-8 of sum |dO o|), which shifts
every ds by p times that."""
import pytest
import torch

from _token_ref import HALF, attention, close

pytestmark = pytest.mark.gpu


def _inputs(B, Tq, Tk, H, Hkv, D, dtype, seed, fused=True):
    g = torch.Generator(device='cuda').manual_seed(seed)

    def r(*s):
        return torch.randn(*s, device='cuda', generator=g).to(dtype)

    q, do = r(B, Tq, H, D), r(B, Tq, H, D)
    if fused:
        kv = r(B, Tk, 2, Hkv, D)
        return q, kv[:, :, 0], kv[:, :, 1], do
    return q, r(B, Tk, Hkv, D), r(B, Tk, Hkv, D), do


def _bounds(q, k, v, do, o, lse, live, scale):
    """Sums of the sizes of the terms of o, dq, dk, dv, in 64 bits (everything (B, Hkv, rows or Tk, D))."""
    B, Tq, H, D = q.shape
    Hkv, Tk = k.shape[2], k.shape[1]
    G = H // Hkv

    def rows(x):
        return x.reshape(B, Tq, Hkv, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Tq * G, -1)

    def back(x):
        return x.reshape(B, Hkv, Tq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Tq, H, D)

    Q, DO, O = rows(q), rows(do), rows(o)
    L = rows(lse.permute(0, 2, 1)[..., None])
    K, V = k.transpose(1, 2), v.transpose(1, 2)
    z = Q @ K.transpose(2, 3).contiguous() * scale
    p = torch.where(live[:, None, None, :] & torch.isfinite(L), torch.exp(z - L), torch.zeros_like(z))
    dp = DO @ V.transpose(2, 3).contiguous()
    delta = (DO * O).sum(-1, keepdim=True)
    dabs = (DO * O).abs().sum(-1, keepdim=True)
    ds = (p * (dp - delta)).abs() + p * (DO.abs() @ V.abs().transpose(2, 3).contiguous()) * 2.0 ** -8 + p * dabs
    pa = p
    return (back(pa @ V.abs()), back(ds @ K.abs()) * abs(scale), (ds.transpose(2, 3).contiguous() @ Q.abs()).transpose(1, 2) * abs(scale),
            (pa.transpose(2, 3).contiguous() @ DO.abs()).transpose(1, 2))


def _run(q, k, v, do, kv_len=None, mask=None, scale=None):
    from vqa_amd import ops
    o, saved = ops.cross_attention_fwd(q, k, v, kv_len, mask, scale)
    grads = ops.cross_attention_bwd(do, q, k, v, o, saved, kv_len, mask, scale)
    return (o, saved[0], *grads)


def _check(q, k, v, do, kv_len=None, mask=None, scale=None):
    got = _run(q, k, v, do, kv_len, mask, scale)
    B, Tk, D = q.shape[0], k.shape[1], q.shape[3]
    live = torch.ones(B, Tk, dtype=torch.bool, device='cuda')
    if kv_len is not None:
        live &= torch.arange(Tk, device='cuda')[None] < kv_len[:, None]
    if mask is not None:
        live &= mask.bool()
    clean = [torch.where(live[:, :, None, None], x, torch.zeros_like(x)).double() for x in (k, v)]
    leaf = [x.requires_grad_(True) for x in (q.double(), *clean)]
    o, lse = attention(*leaf, kv_len, mask, scale)
    ref = torch.autograd.grad(o, leaf, do.double())
    o, lse = o.detach(), lse.detach()
    s = D ** -0.5 if scale is None else scale
    lim = _bounds(*(x.detach() for x in leaf), do.double(), o, lse, live, s)
    unit = 2e-5 if q.dtype == torch.float32 else 1.05 * HALF[torch.bfloat16]
    fin = torch.isfinite(lse)
    assert torch.equal(torch.isfinite(got[1]), fin)
    assert not bool(fin.logical_not().any()) or float(got[1][~fin].max()) == -float('inf')
    assert not bool(fin.any()) or float((got[1].double() - lse)[fin].abs().max()) <= 2e-5 * (1 + float(lse[fin].abs().max()))
    for what, x, r, b in zip(('o', 'dq', 'dk', 'dv'), (got[0], *got[2:]), (o, *ref), lim):
        close(x, r, unit * b + 1e-6, what)
    dead = ~live
    assert float(got[3][dead].abs().sum()) == 0 and float(got[4][dead].abs().sum()) == 0
    again = _run(q, k, v, do, kv_len, mask, scale)
    assert all(torch.equal(a, b) for a, b in zip(got, again))
    return got


SHAPES = [  # B, Tq, Tk, H, Hkv, D
    (1, 1, 1, 1, 1, 8), (2, 1, 15, 2, 1, 16), (1, 3, 16, 4, 4, 24), (3, 2, 17, 8, 2, 40), (2, 14, 33, 3, 3, 80),
    (2, 5, 196, 12, 4, 64), (1, 1, 700, 16, 2, 128), (2, 16, 63, 2, 2, 96), (2, 17, 65, 2, 2, 72), (1, 20, 129, 6, 3, 32),
    (2, 33, 50, 4, 4, 56), (1, 65, 130, 8, 2, 112), (1, 130, 577, 2, 1, 128), (3, 40, 7, 4, 1, 48), (1, 8, 2000, 8, 1, 88),
    # more than 64 rows on more than 256 regions: the matrix-bound kernels, each width and both workgroup sizes
    (1, 70, 300, 1, 1, 24), (2, 100, 513, 2, 2, 64), (1, 40, 260, 8, 2, 96), (1, 150, 321, 2, 1, 80), (1, 257, 700, 1, 1, 120),
    (2, 33, 449, 6, 2, 104), (1, 20, 385, 16, 2, 8),
    # more than 32 rows on at most 32 regions: the regions stay on the chip, whole and split rows
    (3, 17, 1, 4, 2, 16), (2, 100, 5, 3, 3, 128), (1, 300, 16, 8, 2, 72), (1, 333, 17, 6, 3, 104), (2, 90, 32, 2, 1, 48), (5, 33, 23, 4, 4, 88),
    (2, 20, 20, 3, 3, 64), (3, 24, 7, 1, 1, 128), (4, 16, 1, 2, 1, 104), (2, 9, 31, 4, 2, 32)]


@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', SHAPES)
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('masked', ['none', 'len', 'mask', 'both'])
def test_attention_and_gradients_match_64_bits(B, Tq, Tk, H, Hkv, D, dtype, masked):
    q, k, v, do = _inputs(B, Tq, Tk, H, Hkv, D, dtype, 7 * Tk + Tq)
    g = torch.Generator(device='cuda').manual_seed(Tk)
    kv_len = mask = None
    if masked in ('len', 'both'):
        kv_len = torch.randint(0, Tk + 1, (B,), device='cuda', generator=g, dtype=torch.int32)
    if masked in ('mask', 'both'):
        mask = torch.rand(B, Tk, device='cuda', generator=g) < 0.6
        if B > 1:
            mask[0] = False                                  # a sample with nothing to attend
    if masked != 'none':                                     # what does not count may hold anything
        live = torch.ones(B, Tk, dtype=torch.bool, device='cuda') if mask is None else mask.clone()
        if kv_len is not None:
            live &= torch.arange(Tk, device='cuda')[None] < kv_len[:, None]
        k[~live] = float('nan')
        v[~live] = float('inf')
    _check(q, k, v, do, kv_len, mask)


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_long_and_many(dtype):
    """Key ranges split over workgroups (few rows, many regions) and many row blocks."""
    for B, Tq, Tk, H, Hkv, D in ((1, 1, 4096, 8, 2, 64), (2, 4, 3001, 4, 1, 128), (1, 300, 1111, 4, 2, 64)):
        q, k, v, do = _inputs(B, Tq, Tk, H, Hkv, D, dtype, Tk)
        _check(q, k, v, do)
        _check(q, k, v, do, kv_len=torch.full((B,), Tk // 3, device='cuda', dtype=torch.int32))


@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', [(1, 41, 1500, 8, 1, 72), (1, 35, 600, 1, 1, 64), (1, 301, 70, 3, 1, 40), (3, 37, 777, 5, 5, 128),
                                             (1, 700, 300, 2, 1, 104), (1, 19, 31, 2, 1, 24)])
def test_few_workgroups_split_keys_and_rows(B, Tq, Tk, H, Hkv, D, dtype):
    """dq summed over ranges of keys, dk and dv over ranges of rows, where the pairs alone leave the chip empty."""
    q, k, v, do = _inputs(B, Tq, Tk, H, Hkv, D, dtype, Tq)
    _check(q, k, v, do)
    mask = torch.rand(B, Tk, device='cuda', generator=torch.Generator(device='cuda').manual_seed(1)) < 0.7
    _check(q, k, v, do, kv_len=torch.full((B,), Tk // 3, device='cuda', dtype=torch.int32), mask=mask)


def test_strides_scale_and_sharp_scores():
    q, k, v, do = _inputs(2, 6, 37, 4, 2, 32, torch.bfloat16, 1, fused=False)
    want = _check(q, k, v, do, scale=0.3)
    heads_first = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]        # (B, H, T, D) storage
    for a, b in zip(want, _run(*heads_first, do.transpose(1, 2).contiguous().transpose(1, 2), scale=0.3)):
        assert torch.equal(a, b)
    odd = [torch.empty(x.numel() + 1, device='cuda', dtype=x.dtype)[1:].view(x.shape).copy_(x) for x in (q, k, v, do)]
    for a, b in zip(want, _run(*odd, scale=0.3)):
        assert torch.equal(a, b)
    one = [k[:, :, :1].expand(-1, -1, 2, -1), v[:, :1].expand(-1, 37, -1, -1)]               # stride 0: broadcast keys
    for a, b in zip(_run(q, *one, do), _run(q, *(x.contiguous() for x in one), do)):
        assert torch.equal(a, b)
    # one region far above the others, in a late tile: the running maximum jumps
    q, k, v, do = _inputs(1, 20, 300, 2, 2, 64, torch.float32, 2, fused=False)
    k[:, 271] = 6 * q[:, 3]
    _check(q, k, v, do)


@pytest.mark.parametrize('shape', [(3, 7, 90, 2, 2, 64), (3, 40, 70, 4, 2, 64), (3, 90, 400, 2, 2, 64), (3, 40, 20, 3, 1, 64), (3, 5, 1, 2, 1, 24)])
def test_masks_of_any_layout(shape):
    """One mask for all samples (stride 0), a slice of a wider one, every second byte of one, numbers other than 1; counts in
    64 bits, below zero and past the regions."""
    q, k, v, do = _inputs(*shape, torch.bfloat16, 13)
    Tk, g = shape[2], torch.Generator(device='cuda').manual_seed(8)
    wide = torch.rand(3, 2 * Tk + 3, device='cuda', generator=g) < 0.6
    kv_len = torch.tensor([2 ** 40, -5, (Tk + 1) // 2], device='cuda')
    for mask in (wide[:1, :Tk].expand(3, -1), wide[:, 3:3 + Tk], wide[:, 1:2 * Tk:2], wide[:, :Tk].to(torch.uint8) * 6):
        for n in (None, kv_len):
            plain = torch.empty(mask.shape, dtype=torch.bool, device='cuda').copy_(mask != 0)
            for a, b in zip(_run(q, k, v, do, n, mask), _run(q, k, v, do, None if n is None else n.clamp(0, Tk).int(), plain)):
                assert torch.equal(a, b)


@pytest.mark.parametrize('shape', [(2, 7, 90, 2, 2, 64), (1, 40, 70, 4, 2, 64), (2, 90, 400, 2, 2, 64), (2, 40, 20, 3, 1, 64)])
@pytest.mark.parametrize('scale', [0.6, -0.6, 0.0, -1e-3])
def test_scores_far_below_zero_and_signs_of_the_scale(shape, scale):
    """Scores near -115 (0.6), where a masked key's 0 would be exp(115) times more than any that counts; a scale that turns
    them, and none.  |z| of 115 is good to 115 x 2^-21, below a bf16 half step's thirtieth."""
    q, k, v, do = _inputs(*shape, torch.bfloat16, 9, fused=False)
    q, k = (q * 0.05 + 1).bfloat16(), (k * 0.05 - 3).bfloat16()
    B, Tk = shape[0], shape[2]
    mask = torch.rand(B, Tk, device='cuda', generator=torch.Generator(device='cuda').manual_seed(2)) < 0.6
    mask[0] = False
    _check(q, k, v, do, scale=scale)
    _check(q, k, v, do, kv_len=torch.full((B,), Tk - 5, device='cuda', dtype=torch.int32), mask=mask, scale=scale)


@pytest.mark.parametrize('shape', [(2, 7, 90, 2, 2, 64), (2, 40, 70, 4, 2, 64), (2, 90, 400, 2, 2, 64), (2, 40, 20, 3, 1, 64), (2, 20, 60, 1, 1, 24)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_an_infinite_output_gradient_stays_with_what_counts(shape, dtype):
    """dO infinite in one row of the first sample: regions that do not count keep zero gradients there, a sample with nothing
    to attend keeps its own at zero, the other sample is untouched."""
    from vqa_amd import ops
    q, k, v, do = _inputs(*shape, dtype, 12, fused=False)
    mask = torch.rand(2, shape[2], device='cuda', generator=torch.Generator(device='cuda').manual_seed(4)) < 0.5
    o, saved = ops.cross_attention_fwd(q, k, v, mask=mask)
    clean = ops.cross_attention_bwd(do, q, k, v, o, saved, mask=mask)
    do[0, 1] = float('inf')
    got = ops.cross_attention_bwd(do, q, k, v, o, saved, mask=mask)
    for a, b in zip(got, clean):
        assert torch.equal(a[1], b[1])
    for x in got[1:]:
        assert float(x[~mask].abs().sum()) == 0
    assert not bool(torch.isfinite(got[2][0][mask[0]]).any())
    none = torch.zeros_like(mask)
    o, saved = ops.cross_attention_fwd(q, k, v, mask=none)
    assert all(float(x.abs().sum()) == 0 for x in (o, *ops.cross_attention_bwd(do, q, k, v, o, saved, mask=none)))


@pytest.mark.parametrize('shape', [(2, 7, 1000, 2, 2, 8), (2, 7, 1000, 2, 2, 24), (2, 5, 1000, 4, 2, 40), (2, 20, 1000, 2, 2, 72), (2, 10, 1000, 4, 2, 120),
                                   (2, 40, 200, 2, 2, 24), (2, 90, 400, 2, 2, 40), (2, 40, 20, 2, 2, 24)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_an_output_gradient_that_is_not_a_number_stays_with_its_row(shape, dtype):
    """One NaN in dO: by the formula dq of that row, dk of its key head and the NaN's own column of dv follow, and nothing
    else changes a bit (1000 regions: every wave walks several tiles of them)."""
    from vqa_amd import ops
    q, k, v, do = _inputs(*shape, dtype, 21, fused=False)
    o, saved = ops.cross_attention_fwd(q, k, v)
    clean = ops.cross_attention_bwd(do, q, k, v, o, saved)
    do[0, 1, 0, 3] = float('nan')
    got = ops.cross_attention_bwd(do, q, k, v, o, saved)
    bad = [torch.zeros_like(x, dtype=torch.bool) for x in got]
    bad[0][0, 1, 0], bad[1][0, :, 0], bad[2][0, :, 0, 3] = True, True, True
    for what, x, y, b in zip(('dq', 'dk', 'dv'), got, clean, bad):
        assert bool(torch.isnan(x[b]).all()) and torch.equal(x[~b], y[~b]), what


def test_infinite_and_nan_operands_spread_as_in_the_formula():
    from vqa_amd import ops
    q, k, v, do = _inputs(2, 3, 40, 2, 2, 16, torch.float32, 3, fused=False)
    v[0, 5, 0, 2] = float('nan')
    k[1, 7, 1, 0] = float('nan')
    o, _ = ops.cross_attention_fwd(q, k, v)
    bad = torch.isnan(o)
    want = torch.zeros_like(bad)
    want[0, :, 0, 2] = True
    want[1, :, 1] = True
    assert torch.equal(bad, want)


def _tight(q, k, v, do, kv_len=None, mask=None, scale=None):
    """bf16 results against bounds that a factor rounded once too often breaks.

    Products of bf16 values are exact in fp32.  A matrix instruction adds 32 of them (a tree of 5 additions) to its sum, and
    a lane adds up to n / 4 numbers itself, so sums are good to F = 2^-19 of their terms' sizes over D <= 128 columns and to
    S(n) = 2^-19 + 2^-24 n over n rows or regions.  z is good to F scale |q||k| and 2^-21 of |z| and |lse|, p to R of itself.
    A factor in two parts is good to U = 2^-16.  Where the kernels for many rows on many regions round p once for its
    product (W = 2^-8 of each weight), o stays a weighted mean: it moves by W sum p |v - o|, delta by W sum |ds|."""
    B, Tq, H, D = q.shape
    Tk, Hkv = k.shape[1], k.shape[2]
    G = H // Hkv
    got = _run(q, k, v, do, kv_len, mask, scale)
    live = torch.ones(B, Tk, dtype=torch.bool, device='cuda')
    if kv_len is not None:
        live &= torch.arange(Tk, device='cuda')[None] < kv_len[:, None]
    if mask is not None:
        live &= mask
    s = D ** -0.5 if scale is None else scale
    leaf = [x.double().requires_grad_(True) for x in (q, k, v)]
    o, lse = attention(*leaf, kv_len, mask, s)
    ref = torch.autograd.grad(o, leaf, do.double())
    o, lse = o.detach(), lse.detach()

    def rows(x):
        return x.reshape(B, Tq, Hkv, G, -1).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Tq * G, -1)

    def back(x):
        return x.reshape(B, Hkv, Tq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Tq, H, D)

    def t(x):
        return x.transpose(2, 3).contiguous()

    Q, DO, O, L = rows(q.double()), rows(do.double()), rows(o), rows(lse.permute(0, 2, 1)[..., None])
    K, V = (x.double().transpose(1, 2).contiguous() for x in (k, v))
    many = Tq * G > 64 and Tk > 256
    F, U, W = 2.0 ** -19, 2.0 ** -16, 1.01 * 2.0 ** -8 if many else 0.0
    here = live[:, None, None, :] & torch.isfinite(L)

    def S(n):
        return 2.0 ** -19 + 2.0 ** -24 * n

    z = Q @ t(K) * s
    L = torch.where(torch.isfinite(L), L, torch.zeros_like(L))
    p = torch.where(here, torch.exp(z - L), torch.zeros_like(z))
    R = torch.where(here, F * abs(s) * (Q.abs() @ t(K.abs())) + 2.0 ** -21 * (2 + z.abs() + L.abs()), torch.zeros_like(z))
    R = R + R.amax(-1, keepdim=True) + S(Tk)                                    # of p in the backward: z's error and the sum's
    dp = DO @ t(V)
    ds = p * (dp - (DO * O).sum(-1, keepdim=True))
    spread = torch.cat([(p[:, :, i, :, None] * (V - O[:, :, i:i + 1]).abs()).sum(2, keepdim=True) for i in range(Tq * G)], 2)
    base = (R * p) @ V.abs() + (U + S(Tk)) * (p @ V.abs())
    oe = base + W * spread                                                      # of o before its rounding
    de = (DO.abs() * (base + (U + F) * O.abs())).sum(-1, keepdim=True) + W * ds.abs().sum(-1, keepdim=True)
    dse = p * (F * (DO.abs() @ t(V.abs())) + de) + (R + 2.0 ** -22) * ds.abs()
    two = not many or D <= 64                                                   # dq's factor
    lim = {'o': back(oe), 'dq': back((dse + (U if two else W) * ds.abs() + S(Tk) * ds.abs()) @ K.abs()) * abs(s),
           'dk': (t(dse + (W or U) * ds.abs() + S(Tq * G) * ds.abs()) @ Q.abs()).transpose(1, 2) * abs(s),
           'dv': (t(p * (R + (W or U) + S(Tq * G))) @ DO.abs()).transpose(1, 2)}
    for what, x, r in zip(('o', 'dq', 'dk', 'dv'), (got[0], *got[2:]), (o, *ref)):
        close(x, r, lim[what] + 1e-30, what)


@pytest.mark.parametrize('units', [5.0, 6.5, 7.6, 7.97])
@pytest.mark.parametrize('D', [128, 64])
def test_one_region_above_a_lagging_maximum(units, D):
    """More than 64 rows on more than 256 regions, nearly all weight on one late region whose score is `units` powers of two
    above the first tile's largest, the rest 25 powers below: dO (v - o) of that region is what little the others leave."""
    q, k, v, do = _inputs(1, 80, 300, 2, 2, D, torch.bfloat16, 41, fused=False)
    scale = 0.125
    k *= 0.02
    q[..., 0] = 1
    k[..., 0] = -25 * 0.6931 / scale
    k[:, 3, :, 0] = 0
    k[:, 290, :, 0] = units * 0.6931 / scale
    _tight(q, k, v, do, scale=scale)


TIGHT = [  # B, Tq, Tk, H, Hkv, D: one row, one pass of 16 and 32 rows, few regions, two kernels, regions and rows in ranges
    (2, 1, 300, 8, 2, 64), (1, 1, 4000, 8, 2, 128), (3, 14, 196, 4, 4, 80), (2, 20, 300, 4, 4, 40), (2, 15, 150, 6, 3, 120), (2, 40, 20, 4, 2, 72),
    (1, 60, 9, 2, 2, 128), (2, 40, 200, 4, 2, 96), (1, 33, 700, 2, 2, 24), (1, 300, 70, 3, 1, 40)]


@pytest.mark.parametrize('shape', TIGHT)
@pytest.mark.parametrize('sharp', [0.25, 1.0, 4.0])
def test_weights_and_their_gradients_keep_two_parts(shape, sharp):
    """Everything but the kernels for many rows on many regions: no factor of a product is rounded to bf16 alone, the
    backward's delta knows what rounding took from o."""
    q, k, v, do = _inputs(*shape, torch.bfloat16, 43, fused=False)
    q *= sharp
    _tight(q, k, v, do)


@pytest.mark.parametrize('B,Tq,Tk,H,Hkv,D', [(53, 1, 100, 17, 17, 24), (53, 5, 90, 34, 17, 40), (53, 20, 70, 17, 17, 72), (53, 40, 100, 17, 17, 64),
                                             (53, 1, 300, 17, 17, 128), (31, 70, 60, 17, 17, 96)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_two_waves_share_a_work_item(B, Tq, Tk, H, Hkv, D, dtype):
    """More than 512 work items, an odd number of them: two to a workgroup, the last one alone."""
    q, k, v, do = _inputs(B, Tq, Tk, H, Hkv, D, dtype, 61)
    kv_len = torch.randint(0, Tk + 1, (B,), device='cuda', generator=torch.Generator(device='cuda').manual_seed(7), dtype=torch.int32)
    _check(q, k, v, do, kv_len)


@pytest.mark.parametrize('shape', [(1, 90, 400, 4, 2, 64), (1, 70, 700, 2, 2, 128), (1, 40, 2000, 2, 1, 96)])
@pytest.mark.parametrize('sharp', [0.25, 1.0, 4.0])
def test_weights_rounded_once_leave_a_mean(shape, sharp):
    """The kernels for many rows on many regions, also with the regions split over workgroups: flat, ordinary and peaked
    weights (q scaled)."""
    q, k, v, do = _inputs(*shape, torch.bfloat16, 43, fused=False)
    q *= sharp
    _tight(q, k, v, do)


def test_few_regions_count_under_many_rows():
    """The kernels for many regions where all but a few are masked or behind the sample's count."""
    q, k, v, do = _inputs(2, 80, 500, 2, 2, 128, torch.bfloat16, 44, fused=False)
    _tight(q, k, v, do, kv_len=torch.tensor([3, 70], device='cuda', dtype=torch.int32))
    mask = torch.rand(2, 500, device='cuda', generator=torch.Generator(device='cuda').manual_seed(3)) < 0.01
    mask[:, 499] = True
    _tight(q, k, v, do, mask=mask)


@pytest.mark.parametrize('shape', [(2, 5, 90, 2, 2, 24), (1, 2, 3000, 4, 1, 64), (2, 40, 70, 4, 2, 40), (1, 95, 400, 2, 1, 64), (1, 80, 2000, 2, 1, 64),
                                   (2, 40, 20, 3, 1, 72)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_a_row_that_is_not_a_number_has_no_log_sum_exp(shape, dtype):
    """q NaN in one row: its output and log-sum-exp are NaN (-inf says that a row attends to nothing), no other changes."""
    from vqa_amd import ops
    q, k, v, _ = _inputs(*shape, dtype, 52, fused=False)
    o, (lse, _) = ops.cross_attention_fwd(q, k, v)
    q[0, 1, -1, 3] = float('nan')
    o2, (lse2, _) = ops.cross_attention_fwd(q, k, v)
    bad = torch.zeros(q.shape[:3], dtype=torch.bool, device='cuda')
    bad[0, 1, -1] = True
    assert bool(torch.isnan(o2[bad]).all()) and torch.equal(o2[~bad], o[~bad])
    bad = bad.transpose(1, 2)
    assert bool(torch.isnan(lse2[bad]).all()) and torch.equal(lse2[~bad], lse[~bad])


def _formula(q, k, v, do, mask):
    """o, dq, dk, dv product by product in 64 bits, infinities and all (regions that do not count taken out)."""
    B, Tq, H, D = q.shape
    G, s = H // k.shape[2], D ** -0.5
    o, dq, dk, dv = (torch.zeros(x.shape, dtype=torch.float64, device='cuda') for x in (q, q, k, v))
    for b in range(B):
        at = torch.nonzero(mask[b])[:, 0]
        for h in range(H):
            Q, DO, K, V = (x.double() for x in (q[b, :, h], do[b, :, h], k[b, at, h // G], v[b, at, h // G]))
            p = torch.softmax(Q @ K.t().contiguous() * s, -1)
            o[b, :, h] = p @ V
            ds = p * (DO @ V.t().contiguous() - (DO * o[b, :, h]).sum(-1, keepdim=True)) * s
            dq[b, :, h] = ds @ K
            dk[b, at, h // G] += ds.t().contiguous() @ Q
            dv[b, at, h // G] += p.t().contiguous() @ DO
    return o, dq, dk, dv


@pytest.mark.parametrize('shape', [(2, 5, 90, 2, 2, 24), (1, 1, 1500, 4, 1, 64), (2, 20, 70, 2, 2, 64), (2, 40, 70, 4, 2, 40), (1, 95, 400, 2, 1, 64),
                                   (1, 77, 300, 1, 1, 128), (2, 40, 20, 3, 1, 72)])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('where', ['v', 'do'])
def test_infinities_that_count_spread_as_in_the_formula(shape, dtype, where):
    """+inf, -inf, NaN and finite results fall where the products of the formula put them.  Scores stay small, so no weight
    is rounded to nothing."""
    from vqa_amd import ops
    q, k, v, do = _inputs(*shape, dtype, 51, fused=False)
    mask = torch.rand(shape[0], shape[2], device='cuda', generator=torch.Generator(device='cuda').manual_seed(6)) < 0.7
    mask[:, 5] = True
    if where == 'v':
        v[0, 5, 0, 2] = float('inf')
        v[-1, 5, -1, 3] = float('-inf')
    else:
        do[0, -1, 0, 2] = float('inf')
        do[-1, 0, -1, 3] = float('-inf')
    o, saved = ops.cross_attention_fwd(q, k, v, mask=mask)
    got = (o, *ops.cross_attention_bwd(do, q, k, v, o, saved, mask=mask))
    for what, x, r in zip(('o', 'dq', 'dk', 'dv'), got, _formula(q, k, v, do, mask)):
        for kind in (torch.isnan, torch.isposinf, torch.isneginf):
            assert torch.equal(kind(x), kind(r)), (what, kind.__name__, int(kind(x).sum()), int(kind(r).sum()))


def test_gradient_against_differences():
    """Central differences of the fp32 forward, step 1e-2: truncation 1e-4 of the gradient's norm, noise (o good to 1e-6,
    n random terms) / (2 step) about 1e-4 of it."""
    from vqa_amd import ops
    q, k, v, do = _inputs(2, 7, 45, 4, 2, 32, torch.float32, 4, fused=False)
    kv_len = torch.tensor([45, 30], device='cuda')
    leaves = [x.clone().requires_grad_(True) for x in (q, k, v)]

    def loss(x):
        return (ops.cross_attention(*x, kv_len=kv_len).double() * do.double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    g = torch.Generator(device='cuda').manual_seed(5)
    with torch.no_grad():
        for i in range(3):
            d = torch.randn(leaves[i].shape, device='cuda', generator=g)
            up, dn = [x.detach() for x in leaves], [x.detach() for x in leaves]
            up[i], dn[i] = up[i] + 1e-2 * d, dn[i] - 1e-2 * d
            num, ana = float((loss(up) - loss(dn)) / 2e-2), float((grads[i].double() * d.double()).sum())
            assert abs(num - ana) <= 5e-3 * float(grads[i].norm()), (i, num, ana)


def test_empty_sizes():
    from vqa_amd import ops
    for B, Tq, Tk in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        q, k = torch.randn(B, Tq, 2, 8, device='cuda'), torch.randn(B, Tk, 1, 8, device='cuda')
        o, saved = ops.cross_attention_fwd(q, k, k)
        assert o.shape == q.shape and float(o.abs().sum()) == 0 and saved[0].shape == (B, 2, Tq)
        assert ops.cross_attention_fwd(q, k, k, save=False)[1] is None
        dq, dk, dv = ops.cross_attention_bwd(o, q, k, k, o, saved)
        assert dq.shape == q.shape and dk.shape == k.shape and float(dq.abs().sum() + dk.abs().sum() + dv.abs().sum()) == 0

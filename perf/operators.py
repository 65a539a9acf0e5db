"""The token-level operators on the workloads they are meant for: a question's (or caption's) tokens read an image.

Three operators, each in every direction and storage type it has:

* ``attn``: cross attention of Tq token rows to Tk image regions (grouped heads, per-sample region counts, region masks);
  ``serve`` is the forward alone, ``train`` the forward and the gradients of q, k, v;
* ``scan``: the gated linear recurrence c_t = s(f_t) c_{t-1} + s(i_t) tanh(g_t), h_t = s(o_t) tanh(c_t) over (B, T, 4H)
  gate rows in the LSTM's order i, f, g, o; ``serve`` carries a state over T tokens, ``train`` adds the gradients;
* ``norm``: the residual update y = rho x + s(gate) w_post f / rms(f) with the next block's norm h = w_pre y / rms(y).

``own`` selects between elementary torch operations (False) and the framework's kernels (True).
"""
import math

import torch

own = False
DT = {'bf16': torch.bfloat16, 'fp32': torch.float32}
SIZE = {'bf16': 2, 'fp32': 4}
EPS = 1e-6


def listed():
    return [
        # one answer token of one image looks at its 14 x 14 regions: latency only
        dict(name='attn serve 1x1 R196', op='attn', mode='serve', dtype='bf16', B=1, Tq=1, Tk=196, Hkv=4, G=4, D=64, ragged=False, mask=False),
        # one new token for each of 64 images at the largest region count the framework takes, grouped heads
        dict(name='attn serve 64x1 R4096', op='attn', mode='serve', dtype='bf16', B=64, Tq=1, Tk=4096, Hkv=8, G=4, D=128, ragged=True, mask=False),
        # the benchmark's batch: 14 question tokens, 196 regions, width 1200 = 15 heads of 80, detected regions vary
        dict(name='attn train 256x14 R196', op='attn', mode='train', dtype='bf16', B=256, Tq=14, Tk=196, Hkv=15, G=1, D=80, ragged=True, mask=False),
        # long texts (a caption set or a dialogue) against the largest region count: matrix-bound
        dict(name='attn train 8x509 R4096', op='attn', mode='train', dtype='bf16', B=8, Tq=509, Tk=4096, Hkv=8, G=2, D=128, ragged=False, mask=False),
        # the fp32 parity mode on 24 x 24 regions with dropped regions
        dict(name='attn train fp32 32x20 R576', op='attn', mode='train', dtype='fp32', B=32, Tq=20, Tk=576, Hkv=8, G=1, D=64, ragged=False, mask=True),
        # one decoding step of 16 questions at the question vector's width, state carried
        dict(name='scan serve 16x1 H2400', op='scan', mode='serve', dtype='bf16', B=16, T=1, H=2400, ragged=False),
        # the benchmark's questions: 14 tokens, lengths 3..14, hidden width 2400
        dict(name='scan train 256x14 H2400', op='scan', mode='train', dtype='bf16', B=256, T=14, H=2400, ragged=True),
        # one very long sequence: all parallelism is along time
        dict(name='scan train 1x16001 H2048', op='scan', mode='train', dtype='bf16', B=1, T=16001, H=2048, ragged=False),
        # fp32 over a 24 x 24 region grid read in raster order, odd length
        dict(name='scan train fp32 7x577 H1200', op='scan', mode='train', dtype='fp32', B=7, T=577, H=1200, ragged=True),
        # the 14 tokens of one question at the attention width
        dict(name='norm serve 1x14 D1200', op='norm', mode='serve', dtype='bf16', B=1, T=14, D=1200, per_row=False),
        # the benchmark's question tokens in fp32 at the question vector's width, one gate row per token
        dict(name='norm train fp32 255x14 D2400', op='norm', mode='train', dtype='fp32', B=255, T=14, D=2400, per_row=True),
        # every region of the benchmark's 512-image batch, one gate row per image
        dict(name='norm train 512x196 D2048', op='norm', mode='train', dtype='bf16', B=512, T=196, D=2048, per_row=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _pairs(c):
    return c['B'] * c['Tq'] * c['Tk'] * c['Hkv'] * c['G'] * (3 if c['ragged'] else 4) // 4


def draw(rng):
    op = rng.choice(('attn', 'attn', 'scan', 'norm'))
    dtype = rng.choice(('bf16', 'bf16', 'fp32'))
    mode = rng.choice(('serve', 'train', 'train'))
    if op == 'attn':
        c = dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, 256), Tq=_log(rng, 1, 8 if mode == 'serve' else 512),
                 Tk=_log(rng, 1, 4096), Hkv=rng.randint(1, 16), G=rng.choice((1, 1, 2, 4, 8)), D=8 * rng.randint(1, 16),
                 ragged=rng.random() < 0.5, mask=rng.random() < 0.3)
        # no more (token, region) pairs than the largest listed case, in fp32 a sixteenth (the fp32 matrix rate)
        most, nbytes = _pairs(listed()[3]) // (1 if dtype == 'bf16' else 16), work(listed()[1])['bytes']
        while _pairs(c) > most or work(c)['bytes'] > nbytes:
            c['B' if c['B'] > 1 else 'Tq'] = max(1, (c['B'] if c['B'] > 1 else c['Tq']) // 2)
        return c
    if op == 'scan':
        c = dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, 256), T=_log(rng, 1, 4 if mode == 'serve' else 16001),
                 H=8 * _log(rng, 4, 300), ragged=rng.random() < 0.5)
        while work(c)['bytes'] > work(listed()[7])['bytes']:
            c['B' if c['B'] > 1 else 'T'] = max(1, (c['B'] if c['B'] > 1 else c['T']) // 2)
        return c
    c = dict(op=op, mode=mode, dtype=dtype, B=_log(rng, 1, 512), T=_log(rng, 1, 256), D=8 * _log(rng, 1, 512),
             per_row=rng.random() < 0.5)
    while work(c)['bytes'] > work(listed()[11])['bytes']:
        c['B'] = max(1, c['B'] // 2)
    return c


def work(case):
    c, s = case, SIZE[case['dtype']]
    train = c['mode'] == 'train'
    if c['op'] == 'attn':
        q = c['B'] * c['Tq'] * c['Hkv'] * c['G'] * c['D'] * s
        kv = 2 * c['B'] * c['Tk'] * c['Hkv'] * c['D'] * s
        if c['ragged']:                                        # on average three quarters of the regions are there
            kv = kv * 3 // 4
        # forward: two products; backward: five. Inputs once, outputs once: q, k, v, o, and dO, dq, dk, dv
        return {'bytes': 2 * q + kv + (2 * q + kv if train else 0), 'flops': (14 if train else 4) * _pairs(c) * c['D']}
    if c['op'] == 'scan':
        n = c['B'] * c['T'] * c['H']
        live = n * (5 if c['ragged'] else 8) // 8
        state = 2 * c['B'] * c['H'] * 4
        # gates in, h out, c0 in, c out; dh in, dgates out, dc in, dc0 out
        return {'bytes': (4 * live + n) * s + state + ((live + 4 * n) * s + state if train else 0), 'flops': (50 if train else 20) * live}
    n = c['B'] * c['T'] * c['D']
    g = n if c['per_row'] else c['B'] * c['D']
    return {'bytes': (4 * n + g) * s + 12 * c['D'] + ((4 * n + g) * s + 12 * c['D'] if train else 0), 'flops': (60 if train else 15) * n}


def prepare(case, seed):
    c, dt = case, DT[case['dtype']]
    gen = torch.Generator(device='cuda').manual_seed(seed)

    def rnd(*shape, dtype=dt, mul=1.0, add=0.0):
        return (torch.randn(*shape, device='cuda', generator=gen) * mul + add).to(dtype)

    def lengths(n, lo, hi):
        return torch.randint(lo, hi + 1, (n,), device='cuda', generator=gen, dtype=torch.int32)

    s = dict(case=c)
    if c['op'] == 'attn':
        B, Tq, Tk, Hkv, H, D = c['B'], c['Tq'], c['Tk'], c['Hkv'], c['Hkv'] * c['G'], c['D']
        s['q'] = rnd(B, Tq, H, D)
        kv = rnd(B, Tk, 2, Hkv, D)                             # k and v of a region come out of one projection
        s['k'], s['v'] = kv[:, :, 0], kv[:, :, 1]
        s['kv_len'] = lengths(B, (Tk + 1) // 2, Tk) if c['ragged'] else None
        s['mask'] = torch.rand(B, Tk, device='cuda', generator=gen) < 0.8 if c['mask'] else None
        s['do'] = rnd(B, Tq, H, D) if c['mode'] == 'train' else None
    elif c['op'] == 'scan':
        B, T, H = c['B'], c['T'], c['H']
        bias = torch.tensor([0.0, 1.0, 0.0, 0.0], device='cuda')   # forget gates start open, as LSTM encoders are initialised
        s['gates'] = (torch.randn(B, T, 4, H, device='cuda', generator=gen) + bias[:, None]).reshape(B, T, 4 * H).to(dt)
        s['lengths'] = lengths(B, max(1, T // 4), T) if c['ragged'] else None
        s['c0'] = rnd(B, H, dtype=torch.float32, mul=0.5)
        if c['mode'] == 'train':
            s['dh'], s['dc'] = rnd(B, T, H), rnd(B, H, dtype=torch.float32)
    else:
        B, T, D = c['B'], c['T'], c['D']
        s['x'], s['f'] = rnd(B, T, D, mul=2.0), rnd(B, T, D, mul=0.3)
        s['gate'] = rnd(B, T, D) if c['per_row'] else rnd(B, 1, D)
        s['rho'], s['w_post'], s['w_pre'] = (rnd(D, dtype=torch.float32, mul=0.1, add=1.0) for _ in range(3))
        if c['mode'] == 'train':
            s['dy'], s['dh'] = rnd(B, T, D), rnd(B, T, D)
    return s


# ---- plain forms ---------------------------------------------------------------------------------------------------

def _live(s, n_keys, device):
    """(B, Tk) truth values: the regions a sample has."""
    m = s['mask']
    if s['kv_len'] is not None:
        r = torch.arange(n_keys, device=device)[None, :] < s['kv_len'][:, None]
        m = r if m is None else m & r
    return m


def _plain_attn(s):
    c = s['case']
    B, Tq, Tk, Hkv, G, D = c['B'], c['Tq'], c['Tk'], c['Hkv'], c['G'], c['D']
    dt, scale = s['q'].dtype, 1.0 / math.sqrt(D)

    def heads(x):                                              # (B, Tq, H, D) -> (B, Hkv, Tq * G, D)
        return x.float().reshape(B, Tq, Hkv, G, D).permute(0, 2, 1, 3, 4).reshape(B, Hkv, Tq * G, D)

    def back(x):
        return x.reshape(B, Hkv, Tq, G, D).permute(0, 2, 1, 3, 4).reshape(B, Tq, Hkv * G, D).to(dt)

    q, k, v = heads(s['q']), s['k'].float().transpose(1, 2).contiguous(), s['v'].float().transpose(1, 2).contiguous()
    live = _live(s, Tk, q.device)
    z = torch.matmul(q, k.transpose(2, 3).contiguous()) * scale
    if live is not None:
        z = z.masked_fill(~live[:, None, None, :], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = torch.exp(z - torch.where(torch.isinf(top), torch.zeros_like(top), top))
    del z
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, torch.ones_like(total), total)
    o = torch.matmul(p, v)
    if c['mode'] == 'serve':
        return back(o)
    do = heads(s['do'])
    dv = torch.matmul(p.transpose(2, 3).contiguous(), do)
    dz = torch.matmul(do, v.transpose(2, 3).contiguous())
    dz = p * (dz - (do * o).sum(-1, keepdim=True)) * scale
    dq = torch.matmul(dz, k)
    dk = torch.matmul(dz.transpose(2, 3).contiguous(), q)
    return {'o': back(o), 'dq': back(dq), 'dk': dk.transpose(1, 2).to(dt), 'dv': dv.transpose(1, 2).to(dt)}


def _linear_scan(a, b):
    """c_t = a_t c_{t-1} + b_t along dim 1 by doubling the span each step covers: log2(T) elementwise passes, which is
    the shortest form the recurrence has in elementary operations that stays finite (a product of T decays does not)."""
    step, T = 1, a.shape[1]
    while step < T:
        tail = a[:, step:]
        b = torch.cat((b[:, :step], torch.addcmul(b[:, step:], tail, b[:, :-step])), 1)
        a = torch.cat((a[:, :step], tail * a[:, :-step]), 1)
        step *= 2
    return b


def _plain_scan(s):
    c = s['case']
    B, T, H = c['B'], c['T'], c['H']
    dt = s['gates'].dtype
    zi, zf, zg, zo = s['gates'].float().reshape(B, T, 4, H).unbind(2)
    i, f, g, o = torch.sigmoid(zi), torch.sigmoid(zf), torch.tanh(zg), torch.sigmoid(zo)
    live = None
    if s['lengths'] is not None:
        live = (torch.arange(T, device=f.device)[None, :] < s['lengths'][:, None])[:, :, None]
        i, f, o = i * live, torch.where(live, f, torch.ones_like(f)), o * live
    b = i * g
    b = torch.cat(((b[:, 0] + f[:, 0] * s['c0'])[:, None], b[:, 1:]), 1)
    st = _linear_scan(f, b)
    tc = torch.tanh(st)
    h = o * tc
    if c['mode'] == 'serve':
        return {'h': h.to(dt), 'c': st[:, -1]}
    dh = s['dh'].float()
    e = dh * o * (1 - tc * tc)
    e = torch.cat((e[:, :-1], (e[:, -1] + s['dc'])[:, None]), 1)
    nxt = torch.cat((f[:, 1:], torch.ones_like(f[:, :1])), 1)
    d = _linear_scan(nxt.flip(1), e.flip(1)).flip(1)           # gradient at c_t
    prev = torch.cat((s['c0'][:, None], st[:, :-1]), 1)
    df = d * prev * f * (1 - f)                                # a padded step has f = 1: no gradient
    dg = torch.stack((d * g * i * (1 - i), df, d * i * (1 - g * g), dh * tc * o * (1 - o)), 2)
    return {'h': h.to(dt), 'c': st[:, -1], 'dgates': dg.reshape(B, T, 4 * H).to(dt), 'dc0': d[:, 0] * f[:, 0]}


def _plain_norm(s):
    c = s['case']
    dt = s['x'].dtype
    x, f, gate = s['x'].float(), s['f'].float(), torch.sigmoid(s['gate'].float())
    r1 = torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS)
    u = f * r1
    y = s['rho'] * x + gate * (s['w_post'] * u)
    r2 = torch.rsqrt((y * y).mean(-1, keepdim=True) + EPS)
    n = y * r2
    h = s['w_pre'] * n
    if c['mode'] == 'serve':
        return {'y': y.to(dt), 'h': h.to(dt)}
    dh = s['dh'].float()
    dn = s['w_pre'] * dh
    dy = s['dy'].float() + r2 * (dn - n * (dn * n).mean(-1, keepdim=True))
    dgate = dy * (s['w_post'] * u)
    if not c['per_row']:
        dgate = dgate.sum(1, keepdim=True)
    du = dy * (gate * s['w_post'])
    return {'y': y.to(dt), 'h': h.to(dt), 'dx': (s['rho'] * dy).to(dt), 'df': (r1 * (du - u * (du * u).mean(-1, keepdim=True))).to(dt),
            'dgate': (dgate * gate * (1 - gate)).to(dt), 'drho': (dy * x).sum((0, 1)), 'dw_post': (dy * gate * u).sum((0, 1)),
            'dw_pre': (dh * n).sum((0, 1))}


# ---- the framework's kernels -----------------------------------------------------------------------------------------

def _own_attn(s):
    from vqa_amd import ops
    o, lse = ops.cross_attention_fwd(s['q'], s['k'], s['v'], kv_len=s['kv_len'], mask=s['mask'])
    if s['case']['mode'] == 'serve':
        return o
    dq, dk, dv = ops.cross_attention_bwd(s['do'], s['q'], s['k'], s['v'], o, lse, kv_len=s['kv_len'], mask=s['mask'])
    return {'o': o, 'dq': dq, 'dk': dk, 'dv': dv}


def _own_scan(s):
    from vqa_amd import ops
    if s['case']['mode'] == 'serve':
        h, c = ops.gated_scan_fwd(s['gates'], lengths=s['lengths'], c0=s['c0'], save=False)[:2]
        return {'h': h, 'c': c}
    h, c, saved = ops.gated_scan_fwd(s['gates'], lengths=s['lengths'], c0=s['c0'])
    dgates, dc0 = ops.gated_scan_bwd(s['dh'], s['dc'], s['gates'], saved, lengths=s['lengths'], c0=s['c0'])
    return {'h': h, 'c': c, 'dgates': dgates, 'dc0': dc0}


def _own_norm(s):
    from vqa_amd import ops
    kw = dict(f=s['f'], gate=s['gate'], residual_scale=s['rho'], w_post=s['w_post'], w_pre=s['w_pre'])
    y, h, stats = ops.norm_gate_fwd(s['x'], eps=EPS, **kw)
    if s['case']['mode'] == 'serve':
        return {'y': y, 'h': h}
    dx, df, dgate, drho, dw_post, dw_pre = ops.norm_gate_bwd(s['dy'], s['dh'], s['x'], stats, **kw)
    return {'y': y, 'h': h, 'dx': dx, 'df': df, 'dgate': dgate, 'drho': drho, 'dw_post': dw_post, 'dw_pre': dw_pre}


def run(state):
    op = state['case']['op']
    if own:
        return {'attn': _own_attn, 'scan': _own_scan, 'norm': _own_norm}[op](state)
    return {'attn': _plain_attn, 'scan': _plain_scan, 'norm': _plain_norm}[op](state)


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------

def _exact_attn(s):
    """Sample by sample over the regions the sample has (taken out by index, nothing is masked), autograd's gradients."""
    c = s['case']
    train = c['mode'] == 'train'
    out = {n: torch.zeros(s[m].shape, dtype=torch.float64, device='cuda') for n, m in (('o', 'q'), ('dq', 'q'), ('dk', 'k'), ('dv', 'v'))}
    for b in range(c['B']):
        q, k, v = (s[n][b].double().requires_grad_(train) for n in ('q', 'k', 'v'))
        idx = torch.arange(c['Tk'] if s['kv_len'] is None else int(s['kv_len'][b]), device='cuda')
        if s['mask'] is not None:
            idx = idx[s['mask'][b][idx]]
        if idx.numel() == 0:
            continue
        kk, vv = (x[idx].repeat_interleave(c['G'], 1).transpose(0, 1) for x in (k, v))       # (H, R, D)
        o = torch.softmax((q.transpose(0, 1) @ kk.transpose(1, 2)) / c['D'] ** 0.5, -1) @ vv
        o = o.transpose(0, 1)
        out['o'][b] = o.detach()
        if train:
            for n, g in zip(('dq', 'dk', 'dv'), torch.autograd.grad(o, (q, k, v), s['do'][b].double())):
                out[n][b] = g
    return out if train else out['o']


def _exact_scan(s):
    """Step by step, every step in 64 bits; autograd's gradients."""
    c = s['case']
    train = c['mode'] == 'train'
    B, T, H = c['B'], c['T'], c['H']
    gates, c0 = s['gates'].double().requires_grad_(train), s['c0'].double().requires_grad_(train)
    zi, zf, zg, zo = gates.reshape(B, T, 4, H).permute(2, 1, 0, 3)
    add, keep = (torch.sigmoid(zi) * torch.tanh(zg)).unbind(0), torch.sigmoid(zf).unbind(0)
    n = torch.full((B,), T, device='cuda') if s['lengths'] is None else s['lengths']
    here = (torch.arange(T, device='cuda')[:, None] < n[None, :])
    st, sts = c0, []
    for t in range(T):
        new = keep[t] * st + add[t]
        st = new if s['lengths'] is None else torch.where(here[t][:, None], new, st)
        sts.append(st)
    h = (torch.sigmoid(zo) * torch.tanh(torch.stack(sts)) * here[:, :, None]).transpose(0, 1)
    out = {'h': h.detach(), 'c': st.detach()}
    if train:
        out['dgates'], out['dc0'] = torch.autograd.grad((h, st), (gates, c0), (s['dh'].double(), s['dc'].double()))
    return out


def _exact_norm(s):
    c = s['case']
    train = c['mode'] == 'train'
    x, f, gate, rho, w_post, w_pre = (s[n].double().requires_grad_(train) for n in ('x', 'f', 'gate', 'rho', 'w_post', 'w_pre'))

    def rms(z):
        return torch.sqrt(torch.sum(z ** 2, -1, keepdim=True) / c['D'] + EPS)

    y = rho * x + torch.sigmoid(gate) * (f / rms(f) * w_post)
    h = y / rms(y) * w_pre
    out = {'y': y.detach(), 'h': h.detach()}
    if train:
        g = torch.autograd.grad((y, h), (x, f, gate, rho, w_post, w_pre), (s['dy'].double(), s['dh'].double()))
        out.update(zip(('dx', 'df', 'dgate', 'drho', 'dw_post', 'dw_pre'), g))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    return {'attn': _exact_attn, 'scan': _exact_scan, 'norm': _exact_norm}[case['op']](s)

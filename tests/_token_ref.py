"""Plain 64-bit forms of the token-level operators, and the comparison the tests use.

A stored value is off by half a step of its type at most (bf16 2^-8, fp32 2^-24 of the value) plus the error of the
fp32 arithmetic in front of it, which the caller states as an absolute bound derived beside the test."""
import torch

HALF = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


def close(got, ref, atol, what=''):
    """|got - ref| <= atol + half a step of got's type, elementwise; atol a number or a tensor."""
    ref = ref.detach().double()
    err = (got.detach().double() - ref).abs()
    lim = atol + HALF[got.dtype] * ref.abs() * (1 + 1e-6)
    if not torch.is_tensor(lim):
        lim = torch.full_like(ref, lim)
    bad = ~(err <= lim)
    assert not bool(bad.any()), (what, int(bad.sum()), float(err[bad].max()), float((err / lim.clamp_min(1e-300)).max()))


def scan(gates, lengths=None, c0=None):
    B, T, H4 = gates.shape
    H = H4 // 4
    c = torch.zeros(B, H, dtype=torch.float64, device=gates.device) if c0 is None else c0
    h = []
    for t in range(T):
        i, f, g, o = gates[:, t].reshape(B, 4, H).unbind(1)
        new = torch.sigmoid(f) * c + torch.sigmoid(i) * torch.tanh(g)
        out = torch.sigmoid(o) * torch.tanh(new)
        if lengths is not None:
            live = (t < lengths)[:, None]
            new, out = torch.where(live, new, c), torch.where(live, out, torch.zeros_like(out))
        c = new
        h.append(out)
    return torch.stack(h, 1), c


def norm_gate(x, f=None, gate=None, rho=None, w_post=None, w_pre=None, eps=1e-6):
    def one(w):
        return 1.0 if w is None else w

    def normed(z):
        return z / torch.sqrt((z * z).mean(-1, keepdim=True) + eps)

    y = x
    if f is not None:
        g = 1.0
        if gate is not None:
            g = torch.sigmoid(gate.reshape(*gate.shape[:-1], *(1,) * (x.dim() - gate.dim()), gate.shape[-1]))
        y = one(rho) * x + g * one(w_post) * normed(f)
    return y, one(w_pre) * normed(y)


def attention(q, k, v, kv_len=None, mask=None, scale=None):
    """Sample by sample over the regions that count; (o, lse)."""
    B, Tq, H, D = q.shape
    G = H // k.shape[2]
    scale = D ** -0.5 if scale is None else scale
    os, ls = [], []
    for b in range(B):
        idx = torch.arange(k.shape[1] if kv_len is None else max(0, min(int(kv_len[b]), k.shape[1])), device=q.device)
        if mask is not None:
            idx = idx[mask[b][idx].bool()]
        if idx.numel() == 0:
            os.append(q[b] * 0 + 0 * (k[b].sum() + v[b].sum()))      # zero, with zero gradients
            ls.append(torch.full((H, Tq), -float('inf'), dtype=q.dtype, device=q.device))
            continue
        kk, vv = (x[b][idx].repeat_interleave(G, 1).transpose(0, 1) for x in (k, v))
        z = (q[b].transpose(0, 1) @ kk.transpose(1, 2).contiguous()) * scale
        os.append((torch.softmax(z, -1) @ vv).transpose(0, 1))
        ls.append(torch.logsumexp(z, -1))
    return torch.stack(os), torch.stack(ls)

"""Experts in 4 bits, the layer over them and the SwiGLU that keeps 8-bit inputs, from their definitions in 64 bits on the CPU.

Results come with the sums of the magnitudes of their terms (``*_terms``), which bound what 32-bit sums in any order can be off by."""
import torch

from oracle.int8_oracle import route  # noqa: F401

LEVELS = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def quantize(w):
    """(E, K, N) -> codes (E, N, G * 16), scales (E, N, G), both uint8."""
    w = w.double().transpose(1, 2)
    E, N, K = w.shape
    G = -(-K // 32)
    v = torch.zeros(E, N, G * 32, dtype=torch.float64)
    v[..., :K] = w
    v = v.view(E, N, G, 32)
    fine = torch.isfinite(v).all(-1, keepdim=True)
    v = torch.where(fine, v, torch.zeros_like(v))
    a = v.abs().amax(-1, keepdim=True)
    p = torch.full_like(a, -127.0)
    for e in range(-127, 128):   # the least power of two that leaves a at 7 units or below
        p = torch.where((a <= 7 * 2.0 ** e) & (a > 7 * 2.0 ** (e - 1)), torch.full_like(p, float(e)), p)
    t = (v / torch.pow(2.0, p)).abs()
    d = (t.unsqueeze(-1) - LEVELS).abs()
    # the nearest level, the even code of two
    order = torch.tensor([0, 2, 4, 6, 1, 3, 5, 7])
    c = order[d[..., order].argmin(-1)]
    c = c + 8 * (v < 0)
    c = c.view(E, N, G * 16, 2)
    scale = torch.where(fine.squeeze(-1), p.squeeze(-1) + 127, torch.full_like(p.squeeze(-1), 255.0))
    return (c[..., 0] + 16 * c[..., 1]).to(torch.uint8), scale.to(torch.uint8)


def weights(codes, scales, K):
    """(E, N, K) in 64 bits."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).long()
    v = LEVELS[c & 7] * torch.where(c >= 8, -1.0, 1.0).double()
    p = torch.pow(torch.tensor(2.0, dtype=torch.float64), scales.double() - 127)
    p = torch.where(scales == 255, torch.full_like(p, float("nan")), p)
    return (v.view(*scales.shape, 32) * p.unsqueeze(-1)).flatten(-2)[..., :K]


def linear(x, w, k, sei, ssi, gates=None, dout=None, grouped_in=False, grouped_out=False):
    """x (T, K), w (E, N, K): y (and y_rows), dx, d_gates in 64 bits with their terms, rows at their flat positions (grouped ones where asked)."""
    x = x.double()
    R, N, K = ssi.numel(), w.size(1), w.size(2)
    m = torch.arange(R)
    rows_in, rows_out = m if grouped_in else ssi // k, m if grouped_out else ssi
    y, yt = torch.zeros(R, N, dtype=torch.float64), torch.zeros(R, N, dtype=torch.float64)
    for e in sei.unique().tolist():
        i = (sei == e).nonzero().squeeze(1)
        y[rows_out[i]] = x[rows_in[i]] @ w[e].t()
        yt[rows_out[i]] = x[rows_in[i]].abs() @ w[e].abs().t()
    out = dict(y_rows=y, y=y, y_terms=yt, y_sums=yt)
    if gates is not None:
        T, kk = gates.shape
        g = gates.double().unsqueeze(-1)
        out.update(y=(y.view(T, kk, N) * g).sum(1), y_terms=(yt.view(T, kk, N) * g.abs()).sum(1), y_sums=(y.view(T, kk, N) * g).abs().sum(1))
    if dout is None:
        return out
    dx, dxt = torch.zeros(R, K, dtype=torch.float64), torch.zeros(R, K, dtype=torch.float64)
    for e in sei.unique().tolist():
        i = (sei == e).nonzero().squeeze(1)
        g = dout.double()[ssi[i] // gates.size(1)] * gates.double().reshape(-1)[ssi[i]][:, None] if gates is not None else dout.double()[rows_out[i]]
        at = i if grouped_in else ssi[i]
        dx[at] = g @ w[e]
        dxt[at] = g.abs() @ w[e].abs()
    out.update(dx=dx.view(-1, k, K).sum(1), dx_sums=dx.abs().view(-1, k, K).sum(1), dx_terms=dxt.view(-1, k, K).sum(1))
    if gates is not None:
        T, kk = gates.shape
        d = dout.double().unsqueeze(1)
        out.update(d_gates=(y.view(T, kk, N) * d).sum(-1), d_gates_sums=(y.view(T, kk, N) * d).abs().sum(-1), d_gates_terms=(yt.view(T, kk, N) * d.abs()).sum(-1))
    return out


def router(x, wg, k, normalize=True):
    """Scores (T, E), weights (T, k), indices (T, k); ties to the lower expert."""
    s = (x.double() @ wg.double().t()).softmax(-1)
    top, idx = s.sort(dim=-1, descending=True, stable=True)
    top, idx = top[:, :k], idx[:, :k]
    return s, top / top.sum(-1, keepdim=True) if normalize else top, idx


def layer(x, wg, w1, w3, w2, k, normalize=True):
    """w1, w3 (E, f, d), w2 (E, d, f) in 64 bits: out, weights, indices, and what bounds the error of out: with h off by e_h in every element,
    out is off by e_h . |w2| weighted (``back``: a function of per-row errors of h)."""
    x = x.double()
    _, w, idx = router(x, wg, k, normalize)
    T, d = x.shape
    out, terms = torch.zeros(T, d, dtype=torch.float64), torch.zeros(T, d, dtype=torch.float64)
    h_all, ht_all = [], []
    for t in range(T):
        for j in range(k):
            e = int(idx[t, j])
            g, u = w1[e] @ x[t], w3[e] @ x[t]
            gt, ut = w1[e].abs() @ x[t].abs(), w3[e].abs() @ x[t].abs()
            s = torch.sigmoid(g)
            h = g * s * u
            # first-order effect of errors of gate and up in units of their terms: |silu'| <= 1.1
            ht = 1.1 * gt * u.abs() + (g * s).abs() * ut
            out[t] += w[t, j] * (w2[e] @ h)
            terms[t] += w[t, j] * (w2[e].abs() @ h.abs())
            h_all.append(w[t, j] * (w2[e].abs() @ ht))
            ht_all.append(h)
    back = torch.stack(h_all).view(T, k, d).sum(1)
    return out, w, idx, terms, back


def kept(v):
    """v (rows, cols) as its 8-bit codes give it back, and the scale of every value's block."""
    v = v.double()
    out, scale = torch.empty_like(v), torch.empty_like(v)
    for at in range(0, v.size(1), 64):
        b = v[:, at:at + 64]
        fine = torch.isfinite(b).all(1, keepdim=True)
        a = torch.where(fine, torch.nan_to_num(b, posinf=0.0, neginf=0.0).abs().amax(1, keepdim=True), torch.full_like(b[:, :1], float("nan")))
        q = torch.where(a > 0, torch.round(127 * b / a), torch.zeros_like(b))
        out[:, at:at + 64] = torch.where(torch.isnan(a), a, q * (a / 127))
        scale[:, at:at + 64] = a / 127
    return out, scale


def swiglu(gate, up, dh=None):
    g, u = gate.double(), up.double()
    h = g * torch.sigmoid(g) * u
    if dh is None:
        return h
    g, _ = kept(gate)
    u, _ = kept(up)
    s, d = torch.sigmoid(g), dh.double()
    return h, d * u * s * (1 + g * (1 - s)), d * g * s, (d * u * s).abs() * (1 + (g * (1 - s)).abs()), (d * g * s).abs()

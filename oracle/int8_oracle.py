"""The expert products over 8-bit weights, from their definition in 64 bits, expert by expert on the CPU.

``codes(v)`` gives, besides the codes and the scales of rows, which codes lie within ``near`` steps of a rounding border: an
implementation whose values differ from these in their last bits may round those the other way."""
import torch


def codes(v, near=0.0):
    v = v.double()
    finite = torch.isfinite(v).all(dim=1, keepdim=True)
    a = torch.where(finite, v.abs().amax(dim=1, keepdim=True) if v.size(1) else v.new_zeros(v.size(0), 1), torch.ones_like(v[:, :1]) if v.size(1) else v.new_ones(v.size(0), 1))
    q = torch.where(finite & (a > 0), 127 * v / torch.where(a > 0, a, torch.ones_like(a)), torch.zeros_like(v))
    c = torch.round(q)
    scale = torch.where(finite, a / 127, torch.full_like(a, float("nan")))
    edge = (q - c).abs() > 0.5 - near
    return c, scale, edge


def route(T, E, k, seed, absent=()):
    """Flat choices of k different experts for each token, none of them in ``absent``; sorted ids, positions, inclusive offsets, gates."""
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn(T, E, generator=g)
    logits[:, list(absent)] = -1e9
    w, idx = logits.softmax(-1).topk(k, dim=-1)
    sei, ssi = idx.reshape(-1).sort(stable=True)
    return sei, ssi, torch.bincount(sei, minlength=E).cumsum(0), w / w.sum(-1, keepdim=True)


def linear(x, w, ws, k, sei, ssi, gates=None, dout=None, grouped_in=False, grouped_out=False, near=0.0):
    """x (T, K), w (E, K, N) codes, ws (E, N): {y_rows, y, dx_rows, dx, dx_slack, d_gates} in 64 bits, rows at their flat positions
    (grouped ones where asked); dx_slack: what codes of the gradient next to a border can change of dx_rows."""
    cx, sx, _ = codes(x)
    w, ws = w.double(), ws.double()
    sx = sx.float().double()
    R, N = ssi.numel(), w.size(2)
    m = torch.arange(R)
    rows_in = m if grouped_in else ssi // k
    rows_out = m if grouped_out else ssi
    y = torch.zeros(R, N, dtype=torch.float64)
    for e in sei.unique().tolist():
        i = (sei == e).nonzero().squeeze(1)
        y[rows_out[i]] = (cx[rows_in[i]] @ w[e]) * sx[rows_in[i]] * ws[e]
    out = {"y_rows": y, "y": y}
    if gates is not None:
        T, kk = gates.shape
        out["y"] = (y.view(T, kk, N) * gates.double().unsqueeze(-1)).sum(1)
        out["y_terms"] = (y.view(T, kk, N) * gates.double().unsqueeze(-1)).abs().sum(1)
    if dout is None:
        return out
    dx, slack = torch.zeros(R, w.size(1), dtype=torch.float64), torch.zeros(R, w.size(1), dtype=torch.float64)
    for e in sei.unique().tolist():
        i = (sei == e).nonzero().squeeze(1)
        if gates is not None:
            g = dout.double()[ssi[i] // gates.size(1)] * gates.double().reshape(-1)[ssi[i]][:, None]
        else:
            g = dout.double()[rows_out[i]]
        cg, sg, edge = codes(g * ws[e], near)
        at = m[i] if grouped_in else ssi[i]
        dx[at] = (cg @ w[e].t()) * sg
        slack[at] = (edge.double() @ w[e].abs().t()) * sg
    out.update(dx_rows=dx, dx=dx.view(-1, k, dx.size(1)).sum(1), dx_terms=dx.abs().view(-1, k, dx.size(1)).sum(1), dx_slack=slack.view(-1, k, dx.size(1)).sum(1))
    if gates is not None:
        T, kk = gates.shape
        out["d_gates"] = (y.view(T, kk, N) * dout.double().unsqueeze(1)).sum(-1)
        out["d_gates_terms"] = (y.view(T, kk, N) * dout.double().unsqueeze(1)).abs().sum(-1)
    return out


def mlp(x, w, k, sei, ssi, gates=None, dout=None, grouped_out=False, near=0.0):
    """w: (w1, s1, w2, s2, w3, s3).  {y_rows, y, y_slack_rows, dx, d_gates}, rows at flat positions (grouped ones where asked)."""
    w1, s1, w2, s2, w3, s3 = (t.double() for t in w)
    cx, sx, _ = codes(x)
    sx = sx.float().double()
    R, d = ssi.numel(), x.size(1)
    rows_out = torch.arange(R) if grouped_out else ssi
    y, slack = torch.zeros(R, d, dtype=torch.float64), torch.zeros(R, d, dtype=torch.float64)
    dx = torch.zeros(R, d, dtype=torch.float64)
    for e in sei.unique().tolist():
        i = (sei == e).nonzero().squeeze(1)
        t = ssi[i] // k
        gate, up = (cx[t] @ w1[e].t()) * sx[t] * s1[e], (cx[t] @ w3[e].t()) * sx[t] * s3[e]
        sig = torch.sigmoid(gate)
        ch, sh, edge = codes(gate * sig * up, near)
        y[rows_out[i]] = (ch @ w2[e]) * sh * s2[e]
        slack[rows_out[i]] = (edge.double() @ w2[e].abs()) * sh * s2[e]
        if dout is None:
            continue
        g = dout.double()[ssi[i] // gates.size(1)] * gates.double().reshape(-1)[ssi[i]][:, None] if gates is not None else dout.double()[rows_out[i]]
        cg, sg, _ = codes(g * s2[e])
        dh = (cg @ w2[e].t()) * sg
        a = torch.cat([dh * up * sig * (1 + gate * (1 - sig)) * s1[e], dh * gate * sig * s3[e]], 1)
        ca, sa, _ = codes(a)
        f = gate.size(1)
        dx[ssi[i]] = (ca[:, :f] @ w1[e] + ca[:, f:] @ w3[e]) * sa
    out = {"y_rows": y, "y": y, "y_slack": slack}
    if gates is not None:
        T, kk = gates.shape
        z = gates.double().unsqueeze(-1)
        out["y"], out["y_slack"] = (y.view(T, kk, d) * z).sum(1), (slack.view(T, kk, d) * z.abs()).sum(1)
        out["y_terms"] = (y.view(T, kk, d) * z).abs().sum(1)
    if dout is not None:
        out["dx"] = dx.view(-1, k, d).sum(1)
        if gates is not None:
            out["d_gates"] = (y.view(T, kk, d) * dout.double().unsqueeze(1)).sum(-1)
    return out

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


STEP = 2.0 ** -24     # relative rounding error of fp32


def _segment_max(v):
    return v.abs().view(v.size(0), -1, 32).amax(2, keepdim=True).expand(-1, -1, 32).reshape(v.shape)


def _stored(v, err):
    """Error of values that are off by err and then kept as 24-bit multiples of a step of their 32-column segment: half a step, and the fp32 roundings of the
    factor (a reciprocal, off by its last bit), of the product and of the way back."""
    return err + 8 * STEP * v.abs() + 1.01 * STEP * _segment_max(v)


def _codes_of_approximate(v, err):
    """Codes and scales of rows whose values are off by up to err; which codes an implementation may round the other way, and the relative error of its scales."""
    c, s, _ = codes(v)
    top = s * 127
    top = torch.where(top > 0, top, torch.ones_like(top))
    worst = err.amax(1, keepdim=True) / top
    near = 127 * (err + v.abs() * (worst + 4 * STEP)) / top
    edge = (127 * v / top - c).abs() > 0.5 - near
    return c, s, edge.double(), worst + 2 * STEP


def mlp_bounds(x, w, k, sei, ssi, gates=None, dout=None):
    """As mlp(), with a bound for every element of y, dx and d_gates before their last rounding: codes that lie so near a border that the roundings of fp32
    arithmetic and of 24-bit interims may carry them over it count with a whole step, everything else with its roundings.  Codes of x and of the gradient's rows are
    exact.  The logistic function: exp2 of a rounded product (relative error 2 |g| + 2 steps), one sum, one reciprocal."""
    w1, s1, w2, s2, w3, s3 = (t.double() for t in w)
    cx, sx, _ = codes(x)
    sx = sx.float().double()
    R, d, f = ssi.numel(), x.size(1), w1.size(1)
    y, y_slack, dx, dx_slack = (torch.zeros(R, d, dtype=torch.float64) for _ in range(4))
    flat = None if gates is None else gates.double().reshape(-1)
    for e in sei.unique().tolist():
        i = (sei == e).nonzero().squeeze(1)
        at, t = ssi[i], ssi[i] // k
        g, u = (cx[t] @ w1[e].t()) * sx[t] * s1[e], (cx[t] @ w3[e].t()) * sx[t] * s3[e]
        sig = torch.sigmoid(g)
        slope = sig * torch.sigmoid(-g)
        sig_err = torch.where(g > 18, torch.exp(-g), slope * (2 * g.abs() + 2) * STEP + 4 * STEP * sig) + 2.0 ** -125
        ge, ue = 3 * STEP * g.abs(), 3 * STEP * u.abs()
        h = g * sig * u
        h_err = u.abs() * (sig + g.abs() * slope) * ge + (g * sig).abs() * ue + (g * u).abs() * sig_err + 3 * STEP * h.abs() + 2.0 ** -148
        ch, sh, edge, off = _codes_of_approximate(h, _stored(h, h_err))
        y[at] = (ch @ w2[e]) * sh * s2[e]
        y_slack[at] = (edge @ w2[e].abs()) * sh * s2[e] + y[at].abs() * (off + 6 * STEP)
        if dout is None:
            continue
        dy = dout.double()[at // gates.size(1)] * flat[at][:, None] if gates is not None else dout.double()[at]
        cg, sg, _ = codes(dy * s2[e])
        dh = (cg @ w2[e].t()) * sg
        ge, ue, de = _stored(g, ge), _stored(u, ue), _stored(dh, 4 * STEP * dh.abs())
        rest = torch.sigmoid(-g)
        a, b = dh * u * sig * (1 + g * rest) * s1[e], dh * g * sig * s3[e]
        p_err = (2 + g.abs()) * slope * ge + sig_err * (1 + g.abs() * (rest + sig)) + 4 * STEP * sig * (1 + g.abs() * rest)
        a_err = ((u * sig * (1 + g * rest)).abs() * de + (dh * sig * (1 + g * rest)).abs() * ue + (dh * u).abs() * p_err) * s1[e] + 6 * STEP * a.abs()
        b_err = ((g * sig).abs() * de + dh.abs() * (sig + g.abs() * slope) * ge + (dh * g).abs() * sig_err) * s3[e] + 6 * STEP * b.abs()
        ca, sa, edge, off = _codes_of_approximate(torch.cat([a, b], 1), torch.cat([a_err, b_err], 1) + 2.0 ** -148)
        dx[at] = (ca[:, :f] @ w1[e] + ca[:, f:] @ w3[e]) * sa
        dx_slack[at] = (edge[:, :f] @ w1[e].abs() + edge[:, f:] @ w3[e].abs()) * sa + dx[at].abs() * (off + 4 * STEP)
    out = {"y": y, "y_slack": y_slack}
    if gates is not None:
        T, kk = gates.shape
        z = gates.double().unsqueeze(-1)
        terms = (y.view(T, kk, d) * z).abs().sum(1)
        out["y"], out["y_slack"] = (y.view(T, kk, d) * z).sum(1), (y_slack.view(T, kk, d) * z.abs()).sum(1) + 2 * kk * STEP * terms
    if dout is not None:
        out["dx"] = dx.view(-1, k, d).sum(1)
        out["dx_slack"] = dx_slack.view(-1, k, d).sum(1) + (k * STEP * dx.abs().view(-1, k, d).sum(1) if k > 1 else 0)
        if gates is not None:
            dd = dout.double().unsqueeze(1)
            out["d_gates"] = (y.view(T, kk, d) * dd).sum(-1)
            out["d_gates_slack"] = (y_slack.view(T, kk, d) * dd.abs()).sum(-1) + (d + 1) * STEP * (y.view(T, kk, d) * dd).abs().sum(-1)
    return out

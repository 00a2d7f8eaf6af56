"""Plain float64 forms of the recurrent mixers' operators and their gradients, written from
the formulas token by token, and the bound their comparison uses.

Every output comes with a magnitude: the same sums over absolute values.  A kernel whose
every term passes at most ``rounds`` roundings of fp32 is within rounds * 2^-24 of that
magnitude, plus half a step of the output's type (``check``)."""
import torch


def check(got, want, magnitude, rounds, label=""):
    """|got - want| <= half a step of got's type times |want| + rounds * 2^-24 * magnitude,
    element by element; prints the largest share of that bound used."""
    assert got.dtype in (torch.bfloat16, torch.float32), (label, got.dtype)
    step = torch.finfo(got.dtype).eps / 2
    got, want, magnitude = (t.detach().double().cpu() for t in (got, want, magnitude))
    bound = step * want.abs() + (1 + step) * rounds * 2.0 ** -24 * magnitude + 1e-37
    share = ((got - want).abs() / bound).max().item() if got.numel() else 0.0
    print(f"[parity] {label}: share={share:.3f}", flush=True)
    assert got.shape == want.shape, (label, got.shape, want.shape)
    assert torch.isfinite(got).all(), label
    assert share <= 1.0, (label, share)


def wide(t):
    return None if t is None else t.detach().double().cpu()


def sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def silu(x):
    return x * sigmoid(x)


def silu_slope(x):
    s = sigmoid(x)
    return s * (1 + x * (1 - s))


# --- short convolution -----------------------------------------------------------

def conv(x, w, bias, act, dy=None, state=None, lengths=None):
    """{name: (value, magnitude)} of y, the state after, and with dy the gradients."""
    x, w, bias, dy, state = (wide(t) for t in (x, w, bias, dy, state))
    b, n, c = x.shape
    k = w.shape[1]
    rows = torch.cat([x.new_zeros(b, k - 1, c) if state is None else state, x], 1)
    pre, mag = x.new_zeros(b, n, c), x.new_zeros(b, n, c)
    for j in range(k):
        pre = pre + w[:, j] * rows[:, j:j + n]
        mag = mag + (w[:, j] * rows[:, j:j + n]).abs()
    if bias is not None:
        pre, mag = pre + bias, mag + bias.abs()
    y = silu(pre) if act else pre
    ends = [n] * b if lengths is None else [max(0, min(n, int(e))) for e in lengths]
    for i, end in enumerate(ends):
        y[i, end:] = 0
    last = torch.stack([rows[i, end:end + k - 1] for i, end in enumerate(ends)]) if b else \
        x.new_zeros(b, k - 1, c)
    # the slope of silu is at most 1.1: what pre is off moves y by that much
    out = dict(y=(y, 1.1 * mag + y.abs()), state=(last, torch.zeros_like(last)))
    if dy is None:
        return out
    slope = silu_slope(pre) if act else torch.ones_like(pre)
    g = dy * slope
    # the second derivative of silu is at most 0.5
    gm = g.abs() + dy.abs() * (1 + 0.5 * mag if act else 1)
    dx, dxm = torch.zeros_like(x), torch.zeros_like(x)
    dw, dwm = torch.zeros_like(w), torch.zeros_like(w)
    for j in range(k):
        ahead = k - 1 - j            # x_t meets tap j in token t + k - 1 - j
        dx[:, :n - ahead or None] += (w[:, j] * g[:, ahead:]) if n > ahead else 0
        dxm[:, :n - ahead or None] += (w[:, j] * gm[:, ahead:]).abs() if n > ahead else 0
        dw[:, j] = (g * rows[:, j:j + n]).sum((0, 1))
        dwm[:, j] = (gm * rows[:, j:j + n].abs()).sum((0, 1))
    out.update(dx=(dx, dxm), dweight=(dw, dwm), dbias=(g.sum((0, 1)), gm.sum((0, 1))))
    return out


# --- selective state space scan ----------------------------------------------------

def ssm(x, dt, A, B, C, D=None, z=None, dt_bias=None, softplus=True, dy=None, state=None,
        lengths=None):
    """{name: (value, magnitude)} of y, the state after, and with dy the gradients.

    Magnitudes take x, B, C, D, dy and silu(z) absolute and keep the decays (exponents'
    errors, in proportion to the exponent X, meet a factor e^-X: X e^-X < 1)."""
    x, dt, A, B, C, D, z, dt_bias, dy, state = (
        wide(t) for t in (x, dt, A, B, C, D, z, dt_bias, dy, state))
    b, n, e = x.shape
    if B.dim() == 3:
        B, C = B[:, :, None], C[:, :, None]
    each = e // B.shape[2]
    Be, Ce = B.repeat_interleave(each, 2), C.repeat_interleave(each, 2)   # [B, L, E, N]
    pre = dt if dt_bias is None else dt + dt_bias
    delta = pre.clamp_min(0) + torch.log1p(torch.exp(-pre.abs())) if softplus else pre
    inside = torch.ones(b, n, 1, dtype=torch.bool)
    if lengths is not None:
        inside = (torch.arange(n)[None] < torch.as_tensor(lengths).cpu()[:, None])[..., None]
        delta = torch.where(inside, delta, 0.0)
    u = torch.where(inside, delta * x, 0.0)
    gate = silu(z) if z is not None else torch.ones_like(x)
    skip = D if D is not None else x.new_zeros(e)
    a = torch.exp(delta[..., None] * A)

    def walk(u, Be, Ce, x, gate, skip, h):
        hs, ys = [h], []
        for t in range(n):
            h = a[:, t] * h + u[:, t, :, None] * Be[:, t]
            hs.append(h)
            ys.append((h * Ce[:, t]).sum(-1))
        mixed = torch.stack(ys, 1) + skip * x if n else torch.zeros_like(x)
        return torch.stack(hs, 1), mixed, torch.where(inside, mixed * gate, 0.0)
    h0 = x.new_zeros(b, e, A.shape[1]) if state is None else state
    hs, mixed, y = walk(u, Be, Ce, x, gate, skip, h0)
    hm, mm, ym = walk(u.abs(), Be.abs(), Ce.abs(), x.abs(), gate.abs(), skip.abs(), h0.abs())
    out = dict(y=(y, ym), state=(hs[:, -1], hm[:, -1]))
    if dy is None:
        return out

    def back(dm, h, u, Be, Ce, x, A, D, slope):
        g = x.new_zeros(b, e, A.shape[1])
        grads = {k: [] for k in ("x", "dt", "B", "C")}
        dA = torch.zeros_like(A)
        for t in reversed(range(n)):
            g = dm[:, t, :, None] * Ce[:, t] + (a[:, t + 1] * g if t + 1 < n else 0)
            v = a[:, t] * g * h[:, t]
            du = (g * Be[:, t]).sum(-1)
            grads["x"].append(delta_of[:, t] * du + D * dm[:, t])
            grads["dt"].append(((v * A).sum(-1) + x[:, t] * du) * slope[:, t])
            grads["B"].append((g * u[:, t, :, None]).unflatten(1, (-1, each)).sum(2))
            grads["C"].append((dm[:, t, :, None] * h[:, t + 1]).unflatten(1, (-1, each)).sum(2))
            dA += (v * delta_of[:, t, :, None]).sum(0)
        r = {k: torch.stack(v[::-1], 1) for k, v in grads.items()}
        r.update(A=dA, D=(dm * x).sum((0, 1)), dt_bias=r["dt"].sum((0, 1)))
        return r
    slope = sigmoid(pre) if softplus else torch.ones_like(pre)
    delta_of = delta
    want = back(dy * gate, hs, u, Be, Ce, x, A, skip, slope)
    delta_of = delta.abs()
    mag = back((dy * gate).abs(), hm, u.abs(), Be.abs(), Ce.abs(), x.abs(), A.abs(), skip.abs(),
               slope)
    if z is not None:
        want["z"] = dy * mixed * silu_slope(z)
        mag["z"] = (dy * mm).abs() * (1.1 + silu_slope(z).abs())
    out.update({"d" + k: (want[k], mag[k]) for k in want})
    return out


# --- group norm ---------------------------------------------------------------------

def norm(x, groups, w=None, bias=None, gate=None, act=True, eps=1e-5, dy=None):
    """{name: (value, magnitude)} of y and with dy the gradients; x [..., C]."""
    x, w, bias, gate, dy = (wide(t) for t in (x, w, bias, gate, dy))
    shape = x.shape
    width = shape[-1] // groups
    rows = x.reshape(-1, groups, width)
    ones = rows.new_ones(groups, width)
    wg = ones if w is None else w.view(groups, width)
    bg = 0 * ones if bias is None else bias.view(groups, width)
    mean = rows.mean(-1, keepdim=True)
    rstd = ((rows - mean).square().mean(-1, keepdim=True) + eps) ** -0.5
    unit = (rows - mean) * rstd
    # what rounding moves unit by: the difference's own terms, over the deviation
    um = (rows.abs() + rows.abs().mean(-1, keepdim=True)) * rstd + unit.abs()
    o = unit * wg + bg
    om = um * wg.abs() + bg.abs()
    z = None if gate is None else gate.reshape(-1, groups, width)
    if z is not None:
        f, fm = (silu(z), silu(z).abs()) if act else (z, z.abs())
        y, ym = o * f, om * fm + (o * f).abs()
    else:
        y, ym = (silu(o), 1.1 * om + silu(o).abs()) if act else (o, om)
    out = dict(y=(y.reshape(shape), ym.reshape(shape)))
    if dy is None:
        return out
    dy = dy.reshape(-1, groups, width)
    if z is not None:
        d, dm = dy * f, (dy * f).abs()
        slope = silu_slope(z) if act else torch.ones_like(z)
        dz, dzm = dy * o * slope, dy.abs() * om * (slope.abs() + 1.1)
        out["dgate"] = (dz.reshape(shape), dzm.reshape(shape))
    elif act:
        d, dm = dy * silu_slope(o), dy.abs() * (silu_slope(o).abs() + 1 + 0.5 * om)
    else:
        d, dm = dy, dy.abs()
    dn, dnm = d * wg, dm * wg.abs()
    dx = rstd * (dn - dn.mean(-1, keepdim=True) - unit * (dn * unit).mean(-1, keepdim=True))
    cross = (dnm * um).mean(-1, keepdim=True)
    dxm = rstd * (dnm + dnm.mean(-1, keepdim=True) + um * cross) + dx.abs()
    out.update(dx=(dx.reshape(shape), dxm.reshape(shape)),
               dweight=((d * unit).sum(0).flatten(), (dm * um).sum(0).flatten()),
               dbias=(d.sum(0).flatten(), dm.sum(0).flatten()))
    return out

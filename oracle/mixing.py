"""The sequence mixing operators (residual_norm, causal_conv, selective_scan) and their gradients from the formulas,
token after token, in the precision of the inputs (the tests: fp64).

Each function also gives ``sizes``: for every result the sum of the magnitudes of the terms that it is made of, which is
what roundings inside a computation are relative to."""

from __future__ import annotations

import torch


def _sum_to(v, like):
    """``v`` summed over the axes that ``like`` is broadcast along."""
    while v.dim() > like.dim():
        v = v.sum(0)
    for axis in range(like.dim()):
        if like.shape[axis] == 1 and v.shape[axis] != 1:
            v = v.sum(axis, keepdim=True)
    return v


def residual_norm(x, y, gate, y_weight, scale, weight, eps, dr=None, dh=None, post_norm=True, pre_norm=True):
    """(results, sizes): r, h and, with dr, the gradients of x, y, gate, y_weight, scale, weight (None where absent)."""
    one = torch.ones(x.shape[-1], dtype=x.dtype)
    yw, k, w = (one if t is None else t for t in (y_weight, scale, weight))
    s = torch.ones((), dtype=x.dtype) if gate is None else torch.sigmoid(gate)
    rho_y = (y.square().mean(-1, keepdim=True) + eps).rsqrt() if post_norm else torch.ones_like(y[..., :1])
    n = y * rho_y
    v = k * s * n * yw
    r, r_size = x + v, x.abs() + v.abs()
    results, sizes = [r], [r_size]
    rho_r = (r.square().mean(-1, keepdim=True) + eps).rsqrt()
    # an error of r of its size moves the row's norm by at most as much, relative to the row
    loss = 1 + (r_size.square().sum(-1, keepdim=True) / (r.square().sum(-1, keepdim=True) + eps)).sqrt()
    r_hat, hat_size = r * rho_r, r_size * rho_r * loss
    if pre_norm:
        results.append(r_hat * w)
        sizes.append(hat_size * w.abs())
    if dr is None:
        return results, sizes
    mean = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    dR, dR_size = dr, dr.abs()
    if pre_norm:
        e = dh * w
        dR = dR + rho_r * (e - r_hat * mean(e * r_hat))
        dR_size = dR_size + rho_r * loss * (e.abs() + hat_size * mean(e.abs() * hat_size))
    n_abs, f = n.abs(), dR * s * k * yw
    f_size = dR_size * (s * k * yw).abs()
    dy, dy_size = f, f_size
    if post_norm:
        dy, dy_size = rho_y * (f - n * mean(f * n)), rho_y * (f_size + n_abs * mean(f_size * n_abs))

    def pair(value, size, like):
        return (_sum_to(value, like), _sum_to(size, like)) if like is not None else (None, None)

    dgate = pair(dR * v * (1 - s), dR_size * v.abs(), gate)  # 1 - s is off by a rounding of s
    grads = [(dR, dR_size), (dy, dy_size), dgate, pair(dR * s * k * n, dR_size * (s * k * n).abs(), y_weight),
             pair(dR * s * n * yw, dR_size * (s * n * yw).abs(), scale),
             pair(dh * r_hat, dh.abs() * hat_size, weight) if pre_norm else (None, None)]
    return results + [g for g, _ in grads], sizes + [g for _, g in grads]


def silu_slope(p):
    s = torch.sigmoid(p)
    return s + p * s * (1 - s)


def causal_conv(x, weight, bias, state, lengths, silu, dy=None, dnext=None):
    """(results, sizes): y, the last inputs and, with dy, the gradients of x, weight, bias, state."""
    b, t, c = x.shape
    width = weight.shape[1]
    y, p_size, y_size = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(x)
    nxt = x.new_zeros(b, width - 1, c)
    drows, drows_size = x.new_zeros(b, width - 1 + t, c), x.new_zeros(b, width - 1 + t, c)
    dw, dw_size = torch.zeros_like(weight), torch.zeros_like(weight)
    db, db_size = x.new_zeros(c), x.new_zeros(c)
    for i in range(b):
        end = lengths[i]
        first = x.new_zeros(width - 1, c) if state is None else state[i]
        rows = torch.cat([first, x[i, :end]])
        nxt[i] = rows[end:]
        if dnext is not None:
            drows[i, end:end + width - 1] += dnext[i]
            drows_size[i, end:end + width - 1] += dnext[i].abs()
        for at in range(end):
            taps = rows[at:at + width]  # [W, C]
            p = (taps * weight.T).sum(0) + (0 if bias is None else bias)
            size = (taps * weight.T).abs().sum(0) + (0 if bias is None else bias.abs())
            y[i, at] = p * torch.sigmoid(p) if silu else p
            y_size[i, at] = size * 1.1 + 0 * p if silu else size  # |silu'| <= 1.1
            if dy is None:
                continue
            slope = silu_slope(p) if silu else torch.ones_like(p)
            # |silu''| <= 1/2: an error of p moves the slope by half of it; the slope's own terms are at most 1 + |p|
            slope_size = (1 + p.abs() + size) if silu else torch.ones_like(p)
            dp, dp_size = dy[i, at] * slope, dy[i, at].abs() * slope_size
            dw += (dp * taps).T
            dw_size += (dp_size * taps.abs()).T
            db += dp
            db_size += dp_size
            drows[i, at:at + width] += weight.T * dp
            drows_size[i, at:at + width] += weight.T.abs() * dp_size
    results, sizes = [y, nxt], [y_size, nxt.abs()]
    if dy is not None:
        results += [drows[:, width - 1:], dw, None if bias is None else db, None if state is None else drows[:, :width - 1]]
        sizes += [drows_size[:, width - 1:], dw_size, db_size, drows_size[:, :width - 1]]
    return results, sizes


def _scan_core(d, a, u, B, C, D, first, lengths, dy, dlast):
    """h, y and the gradients of one scan from its steps d and decays a [B, T, C(, N)]; maps B, C [B, T, C, N]; sums of
    magnitudes where everything given is one."""
    b, t, c, n = a.shape
    y, last = torch.zeros_like(u), first.clone()
    hs = [[None] * t for _ in range(b)]
    for i in range(b):
        h = first[i]
        for at in range(lengths[i]):
            hs[i][at] = h
            h = a[i, at] * h + (d[i, at] * u[i, at])[:, None] * B[i, at]
            y[i, at] = (h * C[i, at]).sum(-1) + D * u[i, at]
        last[i] = h
    if dy is None:
        return y, last
    du, dd, dA = torch.zeros_like(u), torch.zeros_like(u), torch.zeros_like(first[0])
    gB, gC, gAh = torch.zeros_like(a), torch.zeros_like(a), torch.zeros_like(a)
    dfirst, dD = torch.zeros_like(first), torch.zeros_like(D)
    for i in range(b):
        X = dlast[i]
        for at in range(lengths[i] - 1, -1, -1):
            h = hs[i][at]
            after = a[i, at] * h + (d[i, at] * u[i, at])[:, None] * B[i, at]
            gC[i, at] = dy[i, at][:, None] * after
            G = C[i, at] * dy[i, at][:, None] + X
            gB[i, at] = G * (d[i, at] * u[i, at])[:, None]
            X = a[i, at] * G
            gAh[i, at] = X * h
            dA = dA + X * h * d[i, at][:, None]
            into = (G * B[i, at]).sum(-1)
            du[i, at] = d[i, at] * into + D * dy[i, at]
            dd[i, at] = u[i, at] * into  # and sum_n A X h, added by the caller
            dD = dD + dy[i, at] * u[i, at]
        dfirst[i] = X
    return y, last, du, dd, gAh, dA, gB, gC, dD, dfirst


def selective_scan(u, dt, A, B, C, D, z, dt_bias, state, lengths, softplus=True, dout=None, dlast=None):
    """(results, sizes): out, the last state and, with dout, the gradients of u, dt, A, B, C, D, z, dt_bias, state."""
    b, t, c = u.shape
    groups, n = B.shape[2:]
    keep = (torch.arange(t)[None, :] < torch.tensor(lengths)[:, None]).to(u.dtype)[..., None]
    u, dt, B, C = (torch.where(keep.reshape(b, t, *[1] * (v.dim() - 2)) > 0, v, torch.zeros_like(v)) for v in (u, dt, B, C))
    logit = dt if dt_bias is None else dt + dt_bias
    d = torch.nn.functional.softplus(logit, threshold=1e9) if softplus else logit
    a = torch.exp(d[..., None] * A)
    wide = lambda m: m.repeat_interleave(c // groups, 2)  # noqa: E731
    skip = u.new_zeros(c) if D is None else D
    first = u.new_zeros(b, c, n) if state is None else state
    zs = None if z is None else torch.where(keep > 0, z, torch.zeros_like(z))
    gate = keep if z is None else zs * torch.sigmoid(zs) * keep
    back = None if dout is None else torch.where(keep > 0, dout, torch.zeros_like(dout))
    dlast = torch.zeros_like(first) if dlast is None else dlast
    core = _scan_core(d, a, u, wide(B), wide(C), skip, first, lengths, None if back is None else back * gate, dlast)
    # |softplus(x)| <= |x| + 1 bounds what an error of its input is relative to
    d_size = (d.abs() + (dt.abs() + (0 if dt_bias is None else dt_bias.abs())) * (torch.sigmoid(logit) if softplus else 1))
    size = _scan_core(d_size, a, u.abs(), wide(B).abs(), wide(C).abs(), skip.abs(), first.abs(), lengths,
                      None if back is None else (back * gate).abs(), dlast.abs())
    results, sizes = [core[0] * gate, core[1]], [size[0] * gate.abs(), size[1]]
    if dout is None:
        return results, sizes

    def grads(values, magnitude):
        y, _, du, dd, gAh, dA, gB, gC, dD, dfirst = values
        slope = torch.sigmoid(logit) if softplus else torch.ones_like(logit)
        ddt = (dd + (gAh * (A.abs() if magnitude else A)).sum(-1)) * slope * keep
        narrow = lambda m: m.unflatten(2, (groups, c // groups)).sum(3)  # noqa: E731
        dz = None
        if z is not None:
            zslope = silu_slope(zs)
            dz = (back.abs() * y * (zslope.abs() + 1 if magnitude else zslope) if magnitude else back * y * zslope) * keep
        return [du * keep, ddt, dA, narrow(gB), narrow(gC), None if D is None else dD, dz,
                None if dt_bias is None else ddt.sum((0, 1)), None if state is None else dfirst]

    return results + grads(core, False), sizes + grads(size, True)

"""Plain 64-bit forms of the selective state space operators and of the rotated, normed queries,
for their tests. Each returns its results with a second set: the same sums over the absolute
values of their terms, which bound what float32 roundings inside a kernel can add up to."""

import torch

F64 = torch.float64


def silu(x):
    return x * torch.sigmoid(x)


def dsilu(x):
    s = torch.sigmoid(x)
    return s * (1 + x * (1 - s))


def ranges(B, T, cu):
    """(batch row, first token, end token) of every sequence."""
    if cu is None:
        return [(b, 0, T) for b in range(B)]
    return [(0, a, b) for a, b in zip(cu, cu[1:])]


def scan(u, delta, A, B, C, D=None, z=None, delta_bias=None, softplus=False, h0=None, cu=None,
         dy=None, dht=None, mag=False):
    """selective_scan and, with dy, its gradients: {"y", "ht", "u", "delta", ...}."""
    p = torch.abs if mag else (lambda t: t)
    c = lambda t: None if t is None else t.detach().cpu().to(F64)   # noqa: E731
    u, delta, A, B, C, D, z, bias, h0, dy, dht = map(
        c, (u, delta, A, B, C, D, z, delta_bias, h0, dy, dht))
    Bt, T, Dn = u.shape
    N = A.shape[1]
    G = B.shape[2] if B.dim() == 4 else 1
    Bx, Cx = (t.reshape(Bt, T, G, 1, N).expand(Bt, T, G, Dn // G, N).reshape(Bt, T, Dn, N)
              for t in (B, C))
    pre = delta if bias is None else delta + bias
    dl = torch.logaddexp(pre, torch.zeros_like(pre)) if softplus else pre
    dsp = torch.sigmoid(pre) if softplus else torch.ones_like(pre)
    Dv = torch.zeros(Dn, dtype=F64) if D is None else D
    zv = torch.ones_like(u) if z is None else silu(z)
    # |silu'| <= 1.1, and an error of it is one of that size also where it crosses zero
    dzv = (torch.zeros_like(u) if z is None else torch.full_like(u, 1.1) if mag else dsilu(z))
    seqs = ranges(Bt, T, cu)
    S = len(seqs)
    out = {"y": torch.zeros_like(u), "ht": torch.zeros(S, Dn, N, dtype=F64)}
    g = {n: torch.zeros_like(t) for n, t in
         (("u", u), ("delta", u), ("z", u), ("A", A), ("D", Dv), ("delta_bias", Dv))}
    gB, gC = torch.zeros(Bt, T, Dn, N, dtype=F64), torch.zeros(Bt, T, Dn, N, dtype=F64)
    g["initial_state"] = torch.zeros(S, Dn, N, dtype=F64)
    for s, (b, t0, t1) in enumerate(seqs):
        h = torch.zeros(Dn, N, dtype=F64) if h0 is None else p(h0[s])
        hs = []
        for t in range(t0, t1):
            hs.append(h)
            d = dl[b, t, :, None]
            h = torch.exp(d * A) * h + p(d * u[b, t, :, None] * Bx[b, t])
            out["y"][b, t] = ((p(Cx[b, t]) * h).sum(-1) + p(Dv * u[b, t])) * p(zv[b, t])
        out["ht"][s] = h
        if dy is None:
            continue
        carry = torch.zeros(Dn, N, dtype=F64) if dht is None else p(dht[s])
        for t in reversed(range(t0, t1)):
            d, ut, prev = dl[b, t, :, None], p(u[b, t]), hs.pop()
            a = torch.exp(d * A)
            dyt = p(dy[b, t] * zv[b, t])
            h = a * prev + p(d * u[b, t, :, None] * Bx[b, t])
            yp = (p(Cx[b, t]) * h).sum(-1) + p(Dv * u[b, t])
            g["z"][b, t] = p(dy[b, t] * dzv[b, t]) * yp
            carry = carry + p(Cx[b, t]) * dyt[:, None]
            gC[b, t] = dyt[:, None] * h
            gB[b, t] = carry * p(d) * ut[:, None]
            sB = (carry * p(Bx[b, t])).sum(-1)
            gp = carry * a * prev
            g["u"][b, t] = sB * p(d[:, 0]) + p(Dv) * dyt
            g["delta"][b, t] = (sB * ut + (gp * p(A)).sum(-1)) * dsp[b, t]
            g["A"] += gp * p(d)
            g["D"] += dyt * ut
            carry = carry * a
        g["initial_state"][s] = carry
    if dy is not None:
        g["delta_bias"] = g["delta"].sum((0, 1))
        g["B"] = gB.reshape(Bt, T, G, Dn // G, N).sum(3).reshape(B.shape)
        g["C"] = gC.reshape(Bt, T, G, Dn // G, N).sum(3).reshape(C.shape)
        out.update({"d" + n: t for n, t in g.items()})
    return out


def conv(x, w, bias=None, act=False, init=None, cu=None, dy=None, dfin=None, mag=False):
    """causal_conv1d and, with dy, its gradients."""
    p = torch.abs if mag else (lambda t: t)
    c = lambda t: None if t is None else t.detach().cpu().to(F64)   # noqa: E731
    x, w, bias, init, dy, dfin = map(c, (x, w, bias, init, dy, dfin))
    B, T, D = x.shape
    w = w.reshape(D, -1)
    W = w.shape[1]
    seqs = ranges(B, T, cu)
    S = len(seqs)
    bv = torch.zeros(D, dtype=F64) if bias is None else bias
    out = {"y": torch.zeros_like(x), "ht": torch.zeros(S, W, D, dtype=F64)}
    dx, dw, db = torch.zeros_like(x), torch.zeros_like(w), torch.zeros_like(bv)
    di = torch.zeros(S, W, D, dtype=F64)
    for s, (b, t0, t1) in enumerate(seqs):
        n = t1 - t0
        e = torch.cat([torch.zeros(W, D, dtype=F64) if init is None else init[s], x[b, t0:t1]])
        out["ht"][s] = e[n:]
        ge = torch.zeros_like(e)
        for t in range(n):
            win = e[t + 1:t + 1 + W]
            z = (win * w.t()).sum(0) + bv
            zm = (p(win) * p(w).t()).sum(0) + p(bv)
            # |silu'| <= 1.1: an error of z is an error of at most that of the output
            out["y"][b, t0 + t] = (1.1 * zm if act else zm) if mag else silu(z) if act else z
            if dy is None:
                continue
            gz = dy[b, t0 + t] * (dsilu(z) if act else 1)
            if mag:   # |silu''| <= 0.5
                gz = dy[b, t0 + t].abs() * (1.1 + 0.5 * zm if act else 1)
            ge[t + 1:t + 1 + W] += gz * p(w).t()
            dw += (gz * p(win)).t()
            db += gz
        if dfin is not None:
            ge[n:] += p(dfin[s])
        dx[b, t0:t1] = ge[W:]
        di[s] = ge[:W]
    if dy is not None:
        out.update(dx=dx, dweight=dw, dbias=db, dinitial_state=di)
    return out


def rotate(t, ang, inter):
    R = 2 * ang.shape[-1]
    cos, sin = torch.cos(ang), torch.sin(ang)
    r, t = t.clone(), t
    i = slice(0, R, 2) if inter else slice(0, R // 2)
    j = slice(1, R, 2) if inter else slice(R // 2, R)
    r[..., i] = t[..., i] * cos - t[..., j] * sin
    r[..., j] = t[..., j] * cos + t[..., i] * sin
    return r


def qk(x, w, inv_freq, pos, eps, inter, dy=None):
    """One of the two halves of qk_norm_rope and, with dy, its gradients."""
    c = lambda t: None if t is None else t.detach().cpu().to(F64)   # noqa: E731
    x, w, dy = map(c, (x, w, dy))
    ang = (pos.cpu().to(F64)[..., None, None] * inv_freq.cpu() if inv_freq is not None
           else torch.zeros(1, 1, 1, 0, dtype=F64))
    x.requires_grad_(True)
    w = torch.ones(x.shape[-1], dtype=F64) if w is None else w
    w.requires_grad_(True)
    y = rotate(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w, ang, inter)
    out = {"y": y.detach()}
    if dy is not None:
        out["dx"], out["dw"] = torch.autograd.grad(y, [x, w], dy)
    return out


def close(name, got, ref, mag, terms):
    """|got - ref| <= half a step of got's type + `terms` float32 roundings of the terms' sum."""
    got = got.detach().cpu()
    half = torch.finfo(got.dtype).eps / 2
    tol = half * ref.abs() + terms * 2.0 ** -24 * (1 + half) * mag + 1e-30
    err = (got.to(F64) - ref).abs()
    bad = ~(err <= tol)
    if bad.any():
        i = torch.argmax(torch.where(bad, err / tol, torch.zeros_like(err)))
        raise AssertionError(
            f"{name}: {int(bad.sum())} of {bad.numel()} off, worst {err.flatten()[i]:.3e} against "
            f"a bound of {tol.flatten()[i]:.3e} (value {ref.flatten()[i]:.6g})")

"""The sequence operators' formulas in float64, and error bounds for them.

Every reference returns its outputs with, for each, a magnitude: the same sums
over the absolute values of their terms.  A float32 evaluation differs from the
exact value by at most (number of roundings along a term) x 2^-24 x magnitude,
and a result of a narrower type by half a step of that type more; ``close``
checks that.
"""
from __future__ import annotations

import torch

U = 2.0 ** -24


def close(got, ref, mag, roundings, what):
    """|got - ref| <= half a step of got's type + roundings x 2^-24 x mag."""
    assert got.shape == ref.shape, f"{what}: shape {tuple(got.shape)} != {tuple(ref.shape)}"
    half = 0.0 if got.dtype in (torch.float32, torch.float64) else torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal  # below it, steps are absolute
    g, r, m = got.detach().double().cpu(), ref.detach().double().cpu(), mag.detach().double().cpu()
    err = (g - r).abs()
    bound = (half * (r.abs() + roundings * U * m) + roundings * U * m) * 1.001 + tiny
    bad = ~(err <= bound)
    if bad.any():
        i = int(torch.where(bad, err / bound, torch.zeros_like(err)).flatten().argmax())
        raise AssertionError(f"{what}: {int(bad.sum())}/{bad.numel()} outside; worst at {i}: got {g.flatten()[i]:.9g}, "
                             f"want {r.flatten()[i]:.9g}, error {err.flatten()[i]:.3g}, bound {bound.flatten()[i]:.3g}")


def layer_norm(x, w, b, eps, dy=None):
    """{name: (value, magnitude)}; x (..., D) any type, w, b (D,) or None."""
    x = x.detach().double().cpu()
    D = x.shape[-1]
    w = torch.ones(D, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.detach().double().cpu()
    mean = x.mean(-1, keepdim=True)
    rstd = 1 / ((x - mean).square().mean(-1, keepdim=True) + eps).sqrt()
    xh = (x - mean) * rstd
    X = rstd * (x.abs() + x.abs().mean(-1, keepdim=True))  # bounds xh before its difference cancels
    out = {"y": (xh * w + b, X * w.abs() * (1 + xh.abs()) + b.abs())}
    if dy is not None:
        dy = dy.detach().double().cpu()
        g = dy * w
        rows = tuple(range(x.dim() - 1))
        mg, mgx = g.mean(-1, keepdim=True), (g * xh).mean(-1, keepdim=True)
        ga, gX = g.abs().mean(-1, keepdim=True), (g.abs() * X).mean(-1, keepdim=True)
        # an error of xh enters twice: directly, and through the mean of g xh
        out["dx"] = (rstd * (g - mg - xh * mgx), rstd * (1 + X) * (g.abs() + ga + X * gX))
        out["dw"] = ((dy * xh).sum(rows), (dy.abs() * X * (1 + xh.abs())).sum(rows))
        out["db"] = (dy.sum(rows), dy.abs().sum(rows))
    return out


def causal_conv(x, w, b, silu, lengths=None, past=None, dy=None, dstate=None):
    x, w = x.detach().double().cpu(), w.detach().double().cpu()
    B, N, D = x.shape
    W = w.shape[1]
    b = torch.zeros(D, dtype=torch.float64) if b is None else b.detach().double().cpu()
    n = torch.full((B,), N) if lengths is None else lengths.cpu().long().clamp(0, N)
    live = (torch.arange(N)[None] < n[:, None])[..., None]
    past = torch.zeros(B, W - 1, D, dtype=torch.float64) if past is None else past.detach().double().cpu()
    s = torch.cat([past, torch.where(live, x, torch.zeros(()).double())], 1)
    v, vm = b.expand(B, N, D).clone(), b.abs().expand(B, N, D).clone()
    for k in range(W):
        v += s[:, k:k + N] * w[:, k]
        vm += (s[:, k:k + N] * w[:, k]).abs()
    zero = torch.zeros_like(v)
    sg = torch.sigmoid(v)
    y, ym = (v * sg, vm * (1 + v.abs())) if silu else (v, vm)
    last = torch.stack([s[i, int(n[i]):int(n[i]) + W - 1] for i in range(B)])
    out = {"y": (torch.where(live, y, zero), torch.where(live, ym, zero)), "state": (last, torch.zeros_like(last))}
    if dy is not None:
        dy = torch.where(live, dy.detach().double().cpu(), zero)
        g = dy * (sg * (1 + v * (1 - sg))) if silu else dy
        gm = dy.abs() * (1 + v.abs() + vm) if silu else dy.abs()
        ds, dm = torch.zeros_like(s), torch.zeros_like(s)
        dw, dwm = torch.zeros_like(w), torch.zeros_like(w)
        for k in range(W):
            ds[:, k:k + N] += g * w[:, k]
            dm[:, k:k + N] += gm * w[:, k].abs()
            dw[:, k] = (g * s[:, k:k + N]).sum((0, 1))
            dwm[:, k] = (gm * s[:, k:k + N].abs()).sum((0, 1))
        if dstate is not None:
            for i in range(B):
                ds[i, int(n[i]):int(n[i]) + W - 1] += dstate[i].detach().double().cpu()
                dm[i, int(n[i]):int(n[i]) + W - 1] += dstate[i].detach().double().cpu().abs()
        out["dx"] = tuple(torch.where(live, t[:, W - 1:], zero) for t in (ds, dm))
        out["dpast"] = (ds[:, :W - 1], dm[:, :W - 1])
        out["dw"], out["db"] = (dw, dwm), (g.sum((0, 1)), gm.sum((0, 1)))
    return out


def selective_scan(x, delta, A, B, C, D=None, z=None, bias=None, softplus=False, lengths=None, h0=None, dy=None,
                   dstate=None):
    """B, C (Bt, N, S) or (Bt, N, G, S)."""
    d64 = lambda t: None if t is None else t.detach().double().cpu()  # noqa: E731
    x, delta, A, D, z, bias, h0, dy, dstate = (d64(t) for t in (x, delta, A, D, z, bias, h0, dy, dstate))
    Bt, N, Dm = x.shape
    S = A.shape[1]
    bshape = B.shape
    B, C = d64(B).reshape(Bt, N, -1, S), d64(C).reshape(Bt, N, -1, S)
    G = B.shape[2]
    n = torch.full((Bt,), N) if lengths is None else lengths.cpu().long().clamp(0, N)
    live = (torch.arange(N)[None] < n[:, None])[..., None]
    cut = lambda t: torch.where(live, t, torch.zeros(()).double())  # noqa: E731
    raw = delta if bias is None else delta + bias
    x, raw = cut(x), cut(raw)
    B, C = torch.where(live[..., None], B, 0.0), torch.where(live[..., None], C, 0.0)
    dt = cut(torch.nn.functional.softplus(raw, threshold=60.0) if softplus else raw)
    dtm = cut(dt.abs() + raw.abs() + (0 if bias is None else bias.abs()))  # for the rounding of delta + bias
    wide = lambda t: t.repeat_interleave(Dm // G, dim=1)  # noqa: E731  (Bt, G, S) -> (Bt, Dm, S)
    h = torch.zeros(Bt, Dm, S, dtype=torch.float64) if h0 is None else h0
    hm = h.abs()
    hs, hms, ys, yms = [h], [hm], [], []
    for t in range(N):
        a = torch.exp(dt[:, t, :, None] * A)
        h = a * h + (dt * x)[:, t, :, None] * wide(B[:, t])
        hm = a * hm + (dtm * x.abs())[:, t, :, None] * wide(B[:, t]).abs()
        hs.append(h)
        hms.append(hm)
        ys.append((h * wide(C[:, t])).sum(-1))
        yms.append((hm * wide(C[:, t]).abs()).sum(-1))
    core = torch.stack(ys, 1) if N else torch.zeros(Bt, 0, Dm, dtype=torch.float64)
    corem = torch.stack(yms, 1) if N else core
    if D is not None:
        core, corem = core + D * x, corem + (D * x).abs()
    y, ym = core, corem
    if z is not None:
        z = cut(z)
        sg = torch.sigmoid(z)
        y, ym = core * z * sg, corem * (z * sg).abs() * (1 + z.abs())
    out = {"y": (cut(y), cut(ym)), "state": (h, hm)}
    if dy is None:
        return out
    dy = cut(dy)
    gy, gm = dy, dy.abs()
    if z is not None:
        ds = sg * (1 + z * (1 - sg))
        out["dz"] = (dy * core * ds, dy.abs() * corem * sg * (1 + z.abs()))
        gy, gm = dy * z * sg, dy.abs() * (z * sg).abs() * (1 + z.abs())
    r = torch.zeros(Bt, Dm, S, dtype=torch.float64) if dstate is None else dstate
    rm = r.abs()
    dA, dAm = torch.zeros(Bt, Dm, S, dtype=torch.float64), torch.zeros(Bt, Dm, S, dtype=torch.float64)
    q, qm, s_, sm_ = (torch.zeros_like(x) for _ in range(4))
    dB, dBm, dC, dCm = (torch.zeros(Bt, N, G, S, dtype=torch.float64) for _ in range(4))
    grp = lambda t: t.reshape(Bt, G, Dm // G, S).sum(2)  # noqa: E731
    for t in range(N - 1, -1, -1):
        g4, gm4, u4, um4 = gy[:, t, :, None], gm[:, t, :, None], (dt * x)[:, t, :, None], (dtm * x.abs())[:, t, :, None]
        gh, ghm = r + g4 * wide(C[:, t]), rm + gm4 * wide(C[:, t]).abs()
        dC[:, t], dCm[:, t] = grp(g4 * hs[t + 1]), grp(gm4 * hms[t + 1])
        dB[:, t], dBm[:, t] = grp(gh * u4), grp(ghm * um4)
        q[:, t], qm[:, t] = (gh * wide(B[:, t])).sum(-1), (ghm * wide(B[:, t]).abs()).sum(-1)
        a = torch.exp(dt[:, t, :, None] * A)
        r, rm = a * gh, a * ghm
        k, km = r * hs[t], rm * hms[t]
        s_[:, t], sm_[:, t] = (k * A).sum(-1), (km * A.abs()).sum(-1)
        dA, dAm = dA + k * dt[:, t, :, None], dAm + km * dtm[:, t, :, None]
    sp = torch.sigmoid(raw) if softplus else torch.ones_like(raw)
    dd, ddm = cut((q * x + s_) * sp), cut((qm * x.abs() + sm_) * sp * (1 + raw.abs()))
    Dx = 0.0 if D is None else D
    out["dx"] = (cut(q * dt + gy * Dx), cut(qm * dtm + gm * abs(Dx)))
    out["ddelta"] = (dd, ddm)
    out["dbias"] = (dd.sum((0, 1)), ddm.sum((0, 1)))
    out["dA"] = (dA.sum(0), dAm.sum(0))
    out["dB"] = (dB.reshape(bshape), dBm.reshape(bshape))
    out["dC"] = (dC.reshape(bshape), dCm.reshape(bshape))
    out["dD"] = ((gy * x).sum((0, 1)), (gm * x.abs()).sum((0, 1)))
    out["dh0"] = (r, rm)
    return out

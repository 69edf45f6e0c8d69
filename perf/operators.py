"""Measured cases of the sequence operators: layer_norm, causal_conv and selective_scan.

These are the operators of an encoder or decoder of series whose outputs the
Soft-DTW loss compares: every tensor is a batch of series (B, N, D), time
first, features last.  Each operator is measured forward only (a prompt read
by a trained model), as a training step (outputs and all gradients), and, for
the recurrent two, as the single-token form that serves one new time step of
every series.

  layer_norm      y = (x - mean) / sqrt(var + eps) * w + b over the features
  causal_conv     y[t] = act(bias + sum_k w[:, k] x[t - W + 1 + k]) per feature
  selective_scan  dt = softplus(delta + delta_bias)
                  h[t] = exp(dt A) h[t-1] + dt B[t] x[t]      (state D x S)
                  y[t] = (C[t] . h[t] + D x[t]) * silu(z[t])

``own`` False computes each in plain torch operations in float32, True calls
softdtw_cuda.  ``exact`` is float64 and takes its gradients from autograd.
"""
from __future__ import annotations

import math
import os
import sys

import torch

own = False

_DT = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_SIZE = {"float32": 4, "float16": 2, "bfloat16": 2}
EPS = 1e-5


def _lib():
    pkg = os.path.join(os.getcwd(), "sdtw-cuda-torch_b200")
    if pkg not in sys.path:
        sys.path.insert(1, pkg)
    import softdtw_cuda

    return softdtw_cuda


# ----------------------------------------------------------------------------- cases
def _ln(name, mode, dtype, B, N, D):
    return {"name": name, "op": "layer_norm", "mode": mode, "dtype": dtype, "B": B, "N": N, "D": D}


def _conv(name, mode, dtype, B, N, D, W=4, ragged=False):
    return {"name": name, "op": "causal_conv", "mode": mode, "dtype": dtype, "B": B, "N": N, "D": D, "W": W,
            "ragged": ragged}


def _scan(name, mode, dtype, B, N, D, S=16, G=1, gate=True, ragged=False):
    return {"name": name, "op": "selective_scan", "mode": mode, "dtype": dtype, "B": B, "N": N, "D": D, "S": S,
            "G": G, "gate": gate, "ragged": ragged}


def listed():
    return [
        # One new time step of 32 series through a norm: the smallest call, all latency.
        _ln("ln_step", "prompt", "bfloat16", 32, 1, 512),
        # A training batch of 64 series of 1024 steps, 768 features.
        _ln("ln_train", "train", "bfloat16", 64, 1024, 768),
        # Odd lengths and an odd feature count in float32: rows that no vector width divides.
        _ln("ln_train_odd_f32", "train", "float32", 13, 1021, 1001),
        # One new time step of 64 series being forecast.
        _conv("conv_step", "step", "bfloat16", 64, 1, 1024),
        # A padded batch of prompts of different lengths.
        _conv("conv_prompt_ragged", "prompt", "float16", 24, 777, 640, 3, True),
        # The training pass of the largest encoder here.
        _conv("conv_train", "train", "bfloat16", 16, 2048, 1536),
        # One new time step of 64 series.
        _scan("scan_step", "step", "bfloat16", 64, 1, 1024),
        # One long recording, few features: hardly any rows, the time axis is the work.
        _scan("scan_prompt_long", "prompt", "float32", 1, 8192, 64, 16, 1, False, False),
        # A padded batch of prompts of different lengths, gated, whose states go on to single steps.
        _scan("scan_prompt_ragged", "prompt", "bfloat16", 12, 1500, 1024, 16, 1, True, True),
        # Training on 32 series of 512 steps.
        _scan("scan_train", "train", "bfloat16", 32, 512, 512),
        # Training on series with odd sizes, a small state and two groups, in float32.
        _scan("scan_train_odd_f32", "train", "float32", 5, 333, 210, 7, 2, True, True),
        # The training pass of the largest encoder here.
        _scan("scan_train_large", "train", "bfloat16", 8, 2048, 1536),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["layer_norm", "causal_conv", "selective_scan", "selective_scan"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    mode = rng.choice(["train", "prompt"] if op == "layer_norm" else ["train", "prompt", "step"])
    D = _log_int(rng, 24, 1536)
    if rng.random() < 0.5:
        D = max(32, D // 32 * 32)
    if op == "layer_norm":
        B, N = _log_int(rng, 1, 64), _log_int(rng, 1, 2048)
        return {k: v for k, v in _ln("", mode, dtype, B, N, D).items() if k != "name"}
    N = 1 if mode == "step" else _log_int(rng, 2, 8192 if mode == "prompt" else 2048)
    B = _log_int(rng, 1, 128 if mode == "step" else 32)
    while B > 1 and B * N * D > 8 * 2048 * 1536:
        B //= 2
    ragged = mode != "step" and rng.random() < 0.4
    if op == "causal_conv":
        c = _conv("", mode, dtype, B, N, D, rng.choice([2, 3, 4, 4, 4]), ragged)
    else:
        G = rng.choice([1, 1, 2])
        S = rng.choice([4, 8, 16, 16, 16, rng.randint(1, 16)])
        c = _scan("", mode, dtype, B, N, D // G * G, S, G, rng.random() < 0.7, ragged)
    return {k: v for k, v in c.items() if k != "name"}


# ----------------------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = _DT[case["dtype"]]
    B, N, D = case["B"], case["N"], case["D"]
    train = case["mode"] == "train"

    def rn(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    def ru(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    s = {"case": dict(case)}
    if case["op"] == "layer_norm":
        # Features with their own offsets and scales, as activations have.
        x = torch.randn(B, N, D, generator=g, device="cuda") * (0.5 + ru(D)) + rn(D, dtype=torch.float32)
        s["x"] = x.to(dt)
        s["w"] = 1.0 + rn(D, scale=0.2, dtype=torch.float32)
        s["b"] = rn(D, scale=0.2, dtype=torch.float32)
        leaves = ("x", "w", "b")
    elif case["op"] == "causal_conv":
        W = case["W"]
        if case["mode"] == "step":
            s["x"] = rn(B, D)
            s["state"] = rn(B, W - 1, D)
            s["state_out"] = torch.empty_like(s["state"])
        else:
            s["x"] = rn(B, N, D)
        s["w"] = (ru(D, W) * 2 - 1) / math.sqrt(W)
        s["b"] = (ru(D) * 2 - 1) / math.sqrt(W)
        leaves = ("x", "w", "b")
    else:
        S, G = case["S"], case["G"]
        seq = (B,) if case["mode"] == "step" else (B, N)
        grp = (G, S) if G > 1 else (S,)
        s["x"] = rn(*seq, D)
        s["delta"] = rn(*seq, D, scale=0.5)
        # Decay rates 1 .. S as such models start out, spread as they are after training.
        s["A"] = -torch.arange(1, S + 1, device="cuda", dtype=torch.float32) * torch.exp(
            rn(D, S, scale=0.3, dtype=torch.float32))
        s["B"] = rn(*seq, *grp)
        s["C"] = rn(*seq, *grp)
        s["D"] = 1.0 + rn(D, scale=0.2, dtype=torch.float32)
        # Biases whose softplus is a step size between 1e-3 and 1e-1.
        step = torch.exp(ru(D) * (math.log(0.1) - math.log(1e-3)) + math.log(1e-3))
        s["bias"] = step + torch.log(-torch.expm1(-step))
        s["z"] = rn(*seq, D) if case["gate"] else None
        if case["mode"] == "step":
            s["state"] = rn(B, D, S, dtype=torch.float32)
            s["state_out"] = torch.empty_like(s["state"])
        leaves = ("x", "delta", "A", "B", "C", "D", "bias") + (("z",) if case["gate"] else ())
    s["lengths"] = None
    if case.get("ragged"):
        lo = N // 3
        s["lengths"] = lo + (ru(B) * (N - lo + 1)).to(torch.int64).clamp(max=N - lo)
        s["lengths"][0] = N
    s["leaves"] = leaves if train else ()
    for k in s["leaves"]:
        s[k].requires_grad_(True)
    if train:
        s["dy"] = rn(B, N, D)
        if s["lengths"] is not None:  # a loss does not look at the padding
            s["dy"] *= (torch.arange(N, device="cuda")[None, :] < s["lengths"][:, None])[..., None]
    return s


# ----------------------------------------------------------------------------- plain forms
def _valid(s, B, N):
    if s["lengths"] is None:
        return None
    return (torch.arange(N, device="cuda")[None, :] < s["lengths"][:, None])[..., None]


def _sigmoid(v):
    return 1.0 / (1.0 + torch.exp(-v))


def _plain_layer_norm(s):
    dt = s["x"].dtype
    x, w, b = s["x"].detach().float(), s["w"].detach(), s["b"].detach()
    mean = x.mean(-1, keepdim=True)
    xc = x - mean
    rstd = torch.rsqrt((xc * xc).mean(-1, keepdim=True) + EPS)
    xh = xc * rstd
    y = xh * w + b
    if not s["leaves"]:
        return y.to(dt)
    dy = s["dy"].float()
    gw = dy * w
    dx = rstd * (gw - gw.mean(-1, keepdim=True) - xh * (gw * xh).mean(-1, keepdim=True))
    return y.to(dt), dx.to(dt), (dy * xh).sum((0, 1)), dy.sum((0, 1))


def _plain_conv(s):
    dt = s["x"].dtype
    x, w, b = s["x"].detach().float(), s["w"].detach(), s["b"].detach()
    W = w.shape[1]
    if s["case"]["mode"] == "step":
        win = torch.cat([s["state"].float(), x[:, None]], 1)
        v = (win * w.t()[None]).sum(1) + b
        s["state_out"].copy_(win[:, 1:])
        return (v * _sigmoid(v)).to(dt), s["state_out"]
    B, N, D = x.shape
    keep = _valid(s, B, N)
    if keep is not None:
        x = torch.where(keep, x, torch.zeros_like(x))
    xp = torch.cat([x.new_zeros(B, W - 1, D), x], 1)
    v = b.expand(B, N, D)
    for k in range(W):
        v = v + xp[:, k:k + N] * w[:, k]
    sg = _sigmoid(v)
    y = v * sg
    if keep is not None:
        y = torch.where(keep, y, torch.zeros_like(y))
    if not s["leaves"]:
        n = s["lengths"] if s["lengths"] is not None else torch.full((B,), N, device="cuda")
        at = n[:, None] + torch.arange(W - 1, device="cuda")[None, :]  # the last W-1 inputs, in xp's positions
        return y.to(dt), torch.gather(xp, 1, at[..., None].expand(B, W - 1, D)).to(dt)
    g = s["dy"].float() * (sg + y * (1.0 - sg))
    if keep is not None:
        g = torch.where(keep, g, torch.zeros_like(g))
    gp = torch.cat([g, g.new_zeros(B, W - 1, D)], 1)
    dx = torch.zeros_like(x)
    dw = torch.empty_like(w)
    for k in range(W):
        o = W - 1 - k
        dx = dx + gp[:, o:o + N] * w[:, k]
        dw[:, k] = (g * xp[:, k:k + N]).sum((0, 1))
    return y.to(dt), dx.to(dt), dw, g.sum((0, 1))


def _plain_scan(s):
    dt_ = s["x"].dtype
    f = {k: (None if s[k] is None else s[k].detach().float()) for k in ("x", "delta", "A", "B", "C", "D", "bias", "z")}
    if s["case"]["mode"] == "step":
        f = {k: (v[:, None] if k in ("x", "delta", "B", "C", "z") and v is not None else v) for k, v in f.items()}
    x, A = f["x"], f["A"]
    B, N, D = x.shape
    S, G = s["case"]["S"], s["case"]["G"]
    Bm, Cm = f["B"].reshape(B, N, G, 1, S), f["C"].reshape(B, N, G, 1, S)
    raw = f["delta"] + f["bias"]
    dt = torch.log1p(torch.exp(-raw.abs())) + raw.clamp(min=0)
    keep = _valid(s, B, N) if s["case"]["mode"] != "step" else None
    if keep is not None:
        dt = torch.where(keep, dt, torch.zeros_like(dt))
    u = dt * x
    train = bool(s["leaves"])
    h = s["state"].reshape(B, G, D // G, S) if s["case"]["mode"] == "step" else x.new_zeros(B, G, D // G, S)
    Ag = A.reshape(1, G, D // G, S)
    dtg, ug = dt.reshape(B, N, G, D // G, 1), u.reshape(B, N, G, D // G, 1)
    hs = x.new_empty(N, B, G, D // G, S) if train else None
    yc = x.new_empty(B, N, G, D // G)
    for t in range(N):
        h = torch.exp(dtg[:, t] * Ag) * h + ug[:, t] * Bm[:, t]
        if train:
            hs[t] = h
        yc[:, t] = (h * Cm[:, t]).sum(-1)
    yc = yc.reshape(B, N, D) + f["D"] * x
    sg = _sigmoid(f["z"]) if f["z"] is not None else None
    y = yc if sg is None else yc * f["z"] * sg
    if keep is not None:
        y = torch.where(keep, y, torch.zeros_like(y))
    if s["case"]["mode"] == "step":
        s["state_out"].copy_(h.reshape(B, D, S))
        return y[:, 0].to(dt_), s["state_out"]
    if not train:
        return y.to(dt_), h.reshape(B, D, S)
    # Reverse recurrence: gh[t] = C[t] dyc[t] + exp(dt[t+1] A) gh[t+1].
    dy = s["dy"].float()
    if keep is not None:
        dy = torch.where(keep, dy, torch.zeros_like(dy))
    dz = None
    if sg is not None:
        dz = dy * yc * (sg + f["z"] * sg * (1.0 - sg))
        dy = dy * f["z"] * sg
    dyg = dy.reshape(B, N, G, D // G, 1)
    gh = torch.zeros_like(h)
    dA = torch.zeros_like(Ag.expand(B, G, D // G, S))
    dB, dC = torch.empty_like(Bm[..., 0, :]), torch.empty_like(Cm[..., 0, :])
    du, ddt = torch.empty_like(ug[..., 0]), torch.empty_like(dtg[..., 0])
    for t in range(N - 1, -1, -1):
        gh = gh + dyg[:, t] * Cm[:, t]
        dC[:, t] = (hs[t] * dyg[:, t]).sum(-2)
        dB[:, t] = (gh * ug[:, t]).sum(-2)
        du[:, t] = (gh * Bm[:, t]).sum(-1)
        gh = gh * torch.exp(dtg[:, t] * Ag)
        if t > 0:
            q = gh * hs[t - 1]
            ddt[:, t] = (q * Ag).sum(-1)
            dA += q * dtg[:, t]
        else:
            ddt[:, t] = 0
    du, ddt = du.reshape(B, N, D), ddt.reshape(B, N, D)
    dx = du * dt + dy * f["D"]
    dd = (ddt + du * x) * _sigmoid(raw)
    if keep is not None:
        dd = torch.where(keep, dd, torch.zeros_like(dd))
    out = [y.to(dt_), dx.to(dt_), dd.to(dt_), dA.sum(0).reshape(D, S), dB.reshape(s["B"].shape).to(dt_),
           dC.reshape(s["C"].shape).to(dt_), (dy * x).sum((0, 1)), dd.sum((0, 1))]
    if dz is not None:
        out.append(dz.to(dt_))
    return tuple(out)


# ----------------------------------------------------------------------------- one pass
def _own(s):
    L = _lib()
    op, mode = s["case"]["op"], s["case"]["mode"]
    if op == "layer_norm":
        y = L.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        if not s["leaves"]:
            return y
    elif op == "causal_conv":
        if mode == "step":
            y = L.causal_conv_step(s["x"], s["w"], s["b"], state=s["state"], activation="silu",
                                   state_out=s["state_out"])
            return y, s["state_out"]
        if mode == "prompt":
            return L.causal_conv(s["x"], s["w"], s["b"], activation="silu", lengths=s["lengths"], return_state=True)
        y = L.causal_conv(s["x"], s["w"], s["b"], activation="silu", lengths=s["lengths"])
    else:
        kw = dict(D=s["D"], z=s["z"], delta_bias=s["bias"], delta_softplus=True)
        if mode == "step":
            y = L.selective_scan_step(s["x"], s["delta"], s["A"], s["B"], s["C"], state=s["state"],
                                      state_out=s["state_out"], **kw)
            return y, s["state_out"]
        if mode == "prompt":
            return L.selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], lengths=s["lengths"],
                                    return_state=True, **kw)
        y = L.selective_scan(s["x"], s["delta"], s["A"], s["B"], s["C"], lengths=s["lengths"], **kw)
    return (y.detach(), *torch.autograd.grad(y, [s[k] for k in s["leaves"]], s["dy"]))


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    return {"layer_norm": _plain_layer_norm, "causal_conv": _plain_conv, "selective_scan": _plain_scan}[op](state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    e = _SIZE[case["dtype"]]
    B, N, D, train = case["B"], case["N"], case["D"], case["mode"] == "train"
    n = B * N * D
    if case["op"] == "layer_norm":
        # forward: x in, y out; backward: x and dy in, dx out; the forward's x is the backward's.
        return {"bytes": n * e * (4 if train else 2) + D * 4 * (4 if train else 2), "flops": n * (19 if train else 8)}
    if case["op"] == "causal_conv":
        W = case["W"]
        state = B * (W - 1) * D * e * {"step": 2, "prompt": 1, "train": 0}[case["mode"]]
        par = D * (W + 1) * 4
        return {"bytes": n * e * (4 if train else 2) + state + par * (2 if train else 1),
                "flops": n * ((6 * W + 16) if train else (2 * W + 5))}
    S, G = case["S"], case["G"]
    z = 1 if case["gate"] else 0
    bc = 2 * B * N * G * S * e
    par = D * (S + 2) * 4
    state = B * D * S * 4 * {"step": 2, "prompt": 1, "train": 0}[case["mode"]]
    if train:  # x, delta, (z), dy, B, C in; y and the gradients of all but dy out
        return {"bytes": n * e * (6 + 2 * z) + 2 * bc + 2 * par, "flops": n * S * 25}
    # per state: dt A, exp, u B, a h +, C h +
    return {"bytes": n * e * (3 + z) + bc + par + state, "flops": n * S * 7}


# ----------------------------------------------------------------------------- float64
def exact(case, seed):
    """From the definitions in float64; gradients by differentiating the definition."""
    s = prepare(case, seed)
    op, mode = case["op"], case["mode"]
    with torch.enable_grad():
        p = {k: v.detach().double().requires_grad_(k in s["leaves"]) for k, v in s.items()
             if isinstance(v, torch.Tensor) and v.is_floating_point() and k not in ("dy", "state_out")}
        if op == "layer_norm":
            x = p["x"]
            y = (x - x.mean(-1, keepdim=True)) / (x.var(-1, unbiased=False, keepdim=True) + EPS).sqrt() * p["w"] + p["b"]
            outs = (y,)
        elif op == "causal_conv":
            outs = _exact_conv(p, s, case)
        else:
            outs = _exact_scan(p, s, case)
        if mode != "train":
            return outs[0] if len(outs) == 1 else outs
        grads = torch.autograd.grad(outs[0], [p[k] for k in s["leaves"]], s["dy"].double())
    return (outs[0].detach(), *grads)


def _exact_conv(p, s, case):
    W = case["W"]
    x = p["x"] if case["mode"] != "step" else p["x"][:, None]
    B, N, D = x.shape
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), N, device="cuda", dtype=torch.int64)
    live = torch.arange(N, device="cuda")[None, :, None] < n[:, None, None]
    past = p["state"] if "state" in p else x.new_zeros(B, W - 1, D)
    series = torch.cat([past, x * live], 1)
    pre = torch.einsum("bndk,dk->bnd", series.unfold(1, W, 1), p["w"]) + p["b"]
    y = torch.nn.functional.silu(pre) * live
    last = torch.stack([series[i, int(n[i]):int(n[i]) + W - 1] for i in range(B)])
    if case["mode"] == "step":
        return y[:, 0], last
    return (y,) if case["mode"] == "train" else (y, last)


def _exact_scan(p, s, case):
    step = case["mode"] == "step"
    one = (lambda v: v[:, None]) if step else (lambda v: v)
    x, delta, Bm, Cm = (one(p[k]) for k in ("x", "delta", "B", "C"))
    B, N, D = x.shape
    S, G = case["S"], case["G"]
    Bm, Cm = (v.reshape(B, N, G, S).repeat_interleave(D // G, dim=2) for v in (Bm, Cm)) if B * N * D * S < 2 ** 24 \
        else (v.reshape(B, N, G, S) for v in (Bm, Cm))
    wide = Bm.shape[2] == D
    dt = torch.nn.functional.softplus(delta + p["bias"], threshold=60.0)
    n = s["lengths"] if s["lengths"] is not None else torch.full((B,), N, device="cuda", dtype=torch.int64)
    live = torch.arange(N, device="cuda")[None, :, None] < n[:, None, None]
    dt = dt * live
    h = p["state"] if step else x.new_zeros(B, D, S)
    ys = []
    # Unbound once: a slice of a whole tensor per step would cost a whole gradient per step.
    for dt_t, x_t, B_t, C_t in zip(dt.unbind(1), x.unbind(1), Bm.unbind(1), Cm.unbind(1)):
        if not wide:
            B_t, C_t = (v[:, :, None].expand(B, G, D // G, S).reshape(B, D, S) for v in (B_t, C_t))
        h = torch.exp(dt_t[..., None] * p["A"]) * h + (dt_t * x_t)[..., None] * B_t
        ys.append((h * C_t).sum(-1))
    y = torch.stack(ys, 1) + p["D"] * x
    if case["gate"]:
        y = y * torch.nn.functional.silu(one(p["z"]))
    y = y * live
    if step:
        return y[:, 0], h
    return (y,) if case["mode"] == "train" else (y, h)

"""The sequence operators' kernels against float64 (tests/_seq_ref.py), at sizes
next to their tile edges, odd sizes, strides, ragged batches and every type.

Tolerances count roundings (a unit is 2^-24 of the sum of the absolute terms)
along the longest path of a term:
  layer norm  a row sum is 32 values in a lane and 5 to 9 exchanges deep, twice, then a few
              products: 128; a gradient chains two such sums: 256; a sum over R rows adds R
  conv        W products and sums, the logistic function's 8: 2 W + 32, gradients twice that; sums add B N
  scan        per step: dt (6), dt A log2(e) (2, relative to an exponent of up to 4 here, so 16 in the
              decay), the exponential (4), two products and a sum (3), all of it once more for the
              product of decays: 64 per step and as many again backwards; sums add the terms added
"""
import threading

import pytest
import torch

import _seq_ref as R
import softdtw_cuda as S
from softdtw_cuda import SoftDTW, _native

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _gen(seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return lambda *s, dtype=torch.float32, scale=1.0: (torch.randn(*s, device="cuda", generator=g) * scale).to(dtype)


# ----------------------------------------------------------------------------- layer norm
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 2), (5, 31), (2, 64), (7, 257), (300, 96), (65, 768), (9, 1001), (4, 1024),
                                    (5, 1025), (3, 1032), (6, 4096), (3, 4097), (2, 8192), (2, 8200), (130, 8201)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm(rows, D, dtype):
    rn = _gen(rows * 10000 + D)
    x = (rn(rows, D) + rn(D) * 2).to(dtype).requires_grad_(True)
    w, b = (1 + rn(D) * 0.3).requires_grad_(True), rn(D).requires_grad_(True)
    dy = rn(rows, D, dtype=dtype)
    ref = R.layer_norm(x, w, b, 1e-5, dy)
    y = S.layer_norm(x, w, b)
    R.close(y, *ref["y"], 128, "y")
    with torch.no_grad():
        assert torch.equal(S.layer_norm(x, w, b), y)
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy, retain_graph=True)
    R.close(dx, *ref["dx"], 256, "dx")
    R.close(dw, *ref["dw"], 256 + rows, "dweight")
    R.close(db, *ref["db"], 64 + rows, "dbias")
    (only_x,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    (only_b,) = torch.autograd.grad(y, b, dy)
    assert torch.equal(only_x, dx) and torch.equal(only_b, db)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layer_norm_views_and_no_parameters(dtype):
    rn = _gen(5)
    big = rn(4, 6, 100, dtype=dtype)
    for v in (big[..., :64], big[..., 3:67], big[:, 1:5, :40], big.transpose(0, 2), big[:, ::2], big[0, 0, :50],
              big[:1, :1].expand(3, 5, 100)):
        x = v.detach().requires_grad_(True)
        y = S.layer_norm(x)
        dy = rn(*x.shape, dtype=dtype)
        ref = R.layer_norm(x, None, None, 1e-5, dy)
        R.close(y, *ref["y"], 128, "y of a view")
        R.close(torch.autograd.grad(y, x, dy)[0], *ref["dx"], 256, "dx of a view")
    x = rn(3, 32, dtype=dtype).requires_grad_(True)
    (g,) = torch.autograd.grad(S.layer_norm(x).sum(), x)  # an expanded upstream gradient
    R.close(g, *R.layer_norm(x, None, None, 1e-5, torch.ones(3, 32))["dx"], 256, "dx of a sum")


def test_layer_norm_constant_rows_and_offsets():
    x = torch.full((3, 48), 7.0, device="cuda")
    assert torch.equal(S.layer_norm(x), torch.zeros_like(x))
    rn = _gen(6)
    x = rn(5, 300) + 1000.0  # the variance is not a difference of squares
    R.close(S.layer_norm(x), *R.layer_norm(x, None, None, 1e-5)["y"], 128, "far from zero")


# ----------------------------------------------------------------------------- causal convolution
def _conv_case(seed, B, N, D, W, dtype, ragged, state):
    rn = _gen(seed)
    x, w, b = rn(B, N, D, dtype=dtype), rn(D, W) / W, rn(D) * 0.3
    past = rn(B, W - 1, D, dtype=dtype) if state else None
    n = None
    if ragged:
        n = torch.randint(0, N + 1, (B,), generator=torch.Generator().manual_seed(seed)).cuda()
        n[0], n[-1] = N, 0
    return x, w, b, past, n, rn(B, N, D, dtype=dtype), rn(B, W - 1, D, dtype=dtype)


@pytest.mark.parametrize("B,N,D,W", [(1, 1, 1, 4), (2, 3, 5, 4), (3, 16, 8, 2), (2, 17, 33, 3), (2, 65, 64, 4), (1, 130, 260, 4),
                                     (4, 33, 12, 1), (2, 40, 24, 8), (2, 19, 30, 6), (3, 2, 520, 5), (2, 1000, 7, 4)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("act,ragged,state", [("silu", False, False), (None, True, True), ("silu", True, True)])
def test_causal_conv(B, N, D, W, dtype, act, ragged, state):
    x, w, b, past, n, dy, ds = _conv_case(N * 100 + D, B, N, D, W, dtype, ragged, state)
    leaves = [t.requires_grad_(True) for t in (x, w, b) + ((past,) if state else ())]
    ref = R.causal_conv(x, w, b, act == "silu", n, past, dy, ds if state else None)
    y, st = S.causal_conv(x, w, b, activation=act, lengths=n, initial_state=past, return_state=True)
    R.close(y, *ref["y"], 2 * W + 32, "y")
    assert torch.equal(st.double().cpu(), ref["state"][0])
    with torch.no_grad():
        assert torch.equal(S.causal_conv(x, w, b, activation=act, lengths=n, initial_state=past), y)
    outs, ups = ((y, st), (dy, ds)) if state else ((y,), (dy,))
    g = torch.autograd.grad(outs, leaves, ups, allow_unused=True)
    R.close(g[0], *ref["dx"], 4 * W + 64, "dx")
    R.close(g[1], *ref["dw"], 4 * W + 64 + B * N, "dweight")
    R.close(g[2], *ref["db"], 4 * W + 64 + B * N, "dbias")
    if state and W > 1:
        R.close(g[3], *ref["dpast"], 4 * W + 64, "dinitial_state")


@pytest.mark.parametrize("dtype", DTYPES)
def test_causal_conv_views(dtype):
    rn = _gen(7)
    big = rn(3, 20, 96, dtype=dtype)
    w = rn(32, 4)
    for v in (big[..., :32], big[..., 5:37], big[:, ::2, 32:64], big.transpose(1, 2)[:, :32].transpose(1, 2),
              big[:1, :, :32].expand(4, 20, 32), big[:, :1, :32].expand(3, 9, 32)):
        x = v.detach().requires_grad_(True)
        y = S.causal_conv(x, w)
        dy = rn(*x.shape[:2], 64, dtype=dtype)[..., 32:]
        ref = R.causal_conv(x, w, None, False, dy=dy)
        R.close(y, *ref["y"], 40, "y of a view")
        R.close(torch.autograd.grad(y, x, dy)[0], *ref["dx"], 80, "dx of a view")


# ----------------------------------------------------------------------------- selective scan
def _scan_case(seed, Bt, N, Dm, St, G, dtype, ragged, opts):
    rn = _gen(seed)
    grp = (St,) if G is None else (G, St)
    c = dict(x=rn(Bt, N, Dm, dtype=dtype), delta=rn(Bt, N, Dm, dtype=dtype, scale=0.5),
             A=-torch.exp(rn(Dm, St) * 0.5).clamp(max=2.0), B=rn(Bt, N, *grp, dtype=dtype), C=rn(Bt, N, *grp, dtype=dtype),
             D=None, z=None, bias=None)
    if opts:
        c["D"], c["z"], c["bias"] = rn(Dm), rn(Bt, N, Dm, dtype=dtype), rn(Dm) * 0.5 - 1.0
    else:
        c["delta"] = c["delta"].abs() * 0.3
    n = None
    if ragged:
        n = torch.randint(0, N + 1, (Bt,), generator=torch.Generator().manual_seed(seed)).cuda()
        n[0], n[-1] = N, 0
    return c, n, rn(Bt, Dm, St), rn(Bt, N, Dm, dtype=dtype), rn(Bt, Dm, St)


def _run(c, softplus, n=None, h0=None):
    return S.selective_scan(c["x"], c["delta"], c["A"], c["B"], c["C"], D=c["D"], z=c["z"], delta_bias=c["bias"],
                            delta_softplus=softplus, lengths=n, initial_state=h0, return_state=True)


def _ref(c, softplus, *rest):
    return R.selective_scan(c["x"], c["delta"], c["A"], c["B"], c["C"], c["D"], c["z"], c["bias"], softplus, *rest)


NAMES = dict(x="dx", delta="ddelta", A="dA", B="dB", C="dC", D="dD", z="dz", bias="dbias")


def _check_scan(c, n, h0, dy, dh, opts, state):
    Bt, N, Dm = c["x"].shape
    leaves = {k: v.requires_grad_(True) for k, v in c.items() if v is not None}
    args = list(leaves.values())
    if state:
        args.append(h0.requires_grad_(True))
    ref = _ref(c, opts, n, h0 if state else None, dy, dh if state else None)
    y, h = _run(c, opts, n, h0 if state else None)
    K = 64 * N + 128
    R.close(y, *ref["y"], K, "y")
    R.close(h, *ref["state"], K, "state")
    with torch.no_grad():
        y2, h2 = _run(c, opts, n, h0 if state else None)
        assert torch.equal(y2, y) and torch.equal(h2, h)
    outs, ups = ((y, h), (dy, dh)) if state else ((y,), (dy,))
    g = torch.autograd.grad(outs, args, ups, retain_graph=True)
    sums = {"A": Bt * N, "D": Bt * N, "bias": Bt * N, "B": Dm, "C": Dm}
    for k, got in zip(list(leaves) + ["h0"], g):
        R.close(got, *ref[NAMES.get(k, "dh0")], 2 * K + 64 + sums.get(k, 0), NAMES.get(k, "dh0"))
    for a, b in zip(torch.autograd.grad(outs, args, ups), g):  # sums in a fixed order
        assert torch.equal(a, b)


@pytest.mark.parametrize("Bt,N,Dm,St,G", [
    (1, 1, 1, 1, None), (2, 7, 3, 3, None), (1, 8, 16, 16, None), (2, 9, 17, 16, None), (3, 31, 5, 4, None), (2, 33, 70, 5, None),
    (1, 64, 64, 8, None), (2, 70, 40, 16, 2), (1, 45, 12, 17, 3), (2, 20, 9, 32, None), (1, 40, 10, 33, 2), (2, 34, 6, 64, None),
    (1, 100, 130, 2, 1), (5, 40, 66, 12, 3)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("opts,ragged,state", [(True, False, False), (False, True, True), (True, True, True)])
def test_selective_scan(Bt, N, Dm, St, G, dtype, opts, ragged, state):
    c, n, h0, dy, dh = _scan_case(N * 1000 + Dm, Bt, N, Dm, St, G, dtype, ragged, opts)
    _check_scan(c, n, h0, dy, dh, opts, state)


@pytest.mark.parametrize("Bt,N,Dm,St,G", [
    (2, 37, 64, 4, 2),      # whole tiles of 32 features
    (1, 50, 24, 32, 3),     # of 4
    (500, 18, 32, 16, 1),   # more blocks than three per SM: the variant with four
    (1, 1000, 32, 16, 1),   # few warps: segments of time, whole tiles
    (2, 900, 7, 5, 1)])     # the same with ragged ones
@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_scan_variants(Bt, N, Dm, St, G, dtype):
    c, n, h0, dy, dh = _scan_case(N + Dm, Bt, N, Dm, St, G, dtype, Bt > 1, True)
    _check_scan(c, n, h0, dy, dh, True, True)


def test_selective_scan_long():
    c, n, h0, dy, dh = _scan_case(3, 2, 700, 24, 16, None, torch.float32, True, True)
    _check_scan(c, n, h0, dy, dh, True, True)


@pytest.mark.parametrize("dtype", DTYPES)
def test_selective_scan_views(dtype):
    """Slices of one projection, as a model makes them, at offsets that are not 16-byte aligned."""
    rn = _gen(11)
    Bt, N, Dm, St = 3, 37, 32, 16
    xz = rn(Bt, N, 2 * Dm, dtype=dtype)
    dbc = rn(Bt, N, 5 + 2 * St + Dm, dtype=dtype)
    c = dict(x=xz[..., :Dm], z=xz[..., Dm:], delta=dbc[..., -Dm:], B=dbc[..., 5:5 + St], C=dbc[..., 5 + St:5 + 2 * St],
             A=-torch.exp(rn(Dm, St) * 0.5).clamp(max=2.0), D=rn(Dm), bias=rn(Dm) - 1)
    c = {k: v.detach() for k, v in c.items()}
    _check_scan(c, None, rn(Bt, Dm, St), rn(N, Bt, Dm, dtype=dtype).transpose(0, 1), rn(Bt, Dm, St), True, True)
    c["x"] = rn(1, N, Dm, dtype=dtype).expand(Bt, N, Dm)
    c["B"] = rn(Bt, 1, 1, St, dtype=dtype).expand(Bt, N, 2, St)
    c["C"] = rn(Bt, 2, N, St, dtype=dtype).transpose(1, 2)
    c = {k: v.detach() for k, v in c.items()}
    _check_scan(c, None, rn(Bt, Dm, St), rn(Bt, N, Dm, dtype=dtype), rn(Bt, Dm, St), True, True)


def test_padding_is_not_read():
    c, n, h0, dy, dh = _scan_case(21, 3, 50, 20, 16, None, torch.float32, True, True)
    w = _gen(1)(20, 4)
    clean = [*_run(c, True, n, h0), S.causal_conv(c["x"], w, lengths=n, activation="silu")]
    dead = torch.arange(50, device="cuda")[None, :] >= n[:, None]
    for k in ("x", "delta", "B", "C", "z"):
        c[k] = c[k].masked_fill(dead[..., None], float("nan")).requires_grad_(True)
    y, h = _run(c, True, n, h0)
    v = S.causal_conv(c["x"], w, lengths=n, activation="silu")
    for a, b in zip((y, h, v), clean):
        assert torch.equal(a, b)
    dy = dy.masked_fill(dead[..., None], float("nan"))
    for g in torch.autograd.grad((y, h), [c[k] for k in ("x", "delta", "B", "C", "z")], (dy, dh)):
        assert torch.isfinite(g).all() and (g[dead] == 0).all()
    (g,) = torch.autograd.grad(v, c["x"], dy)
    assert torch.isfinite(g).all() and (g[dead] == 0).all()
    big = torch.tensor([10 ** 12, -5, 50], device="cuda")  # lengths are clamped
    a = S.causal_conv(clean[0], w, lengths=big)
    assert torch.equal(a, S.causal_conv(clean[0], w, lengths=big.clamp(0, 50).int()))


def test_strong_decays_and_large_steps():
    rn = _gen(31)
    x, delta = rn(1, 40, 8), rn(1, 40, 8).abs() * 100 + 1
    bc = rn(1, 40, 16)
    A = -torch.rand(8, 16, device="cuda") * 200 - 50  # decays that are 0 in float32
    y, h = S.selective_scan(x, delta, A, bc, bc, return_state=True)
    ref = R.selective_scan(x, delta, A, bc, bc)
    R.close(y, *ref["y"], 64, "y")
    R.close(h, *ref["state"], 64, "state")
    y = S.selective_scan(x, torch.full_like(delta, -200.0), A, bc, bc, delta_softplus=True)  # steps of size 0
    assert torch.equal(y, torch.zeros_like(y))


def test_infinite_and_nan_steps_follow_the_formula():
    """delta of any size through softplus: 0 and the identity at the ends, NaN only from NaN."""
    v = torch.tensor([float("inf"), 3e38, 1e30, 200.0, 88.0, 17.0, 1e-3, -17.0, -88.0, -200.0, -3e38, float("-inf"), float("nan")],
                     device="cuda").reshape(-1, 1, 1)
    one = torch.ones_like(v)
    y = S.selective_scan(one, v, -torch.ones(1, 1, device="cuda"), one, one, delta_softplus=True)
    want = torch.nn.functional.softplus(v.double(), threshold=1e4).float()
    torch.testing.assert_close(y, want, rtol=1e-6, atol=1e-37, equal_nan=True)


def test_steps_of_size_zero_keep_the_state_exactly():
    rn = _gen(32)
    h0 = rn(2, 8, 16)
    x = rn(2, 100, 8)
    bc = rn(2, 100, 16)
    A = -torch.rand(8, 16, device="cuda") * 20
    _, h = S.selective_scan(x, torch.zeros_like(x), A, bc, bc, initial_state=h0, return_state=True)
    assert torch.equal(h, h0)
    n = torch.zeros(2, dtype=torch.int64, device="cuda")
    _, h = S.selective_scan(x, x, A, bc, bc, initial_state=h0, lengths=n, return_state=True)
    assert torch.equal(h, h0)


# ----------------------------------------------------------------------------- single steps, continued series
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("Bt,Dm,St,G,W", [(1, 1, 1, None, 1), (3, 33, 16, None, 4), (2, 30, 5, 3, 2), (5, 24, 64, 2, 8), (70, 64, 17, None, 3)])
def test_steps(dtype, Bt, Dm, St, G, W):
    c, _, h0, _, _ = _scan_case(Dm, Bt, 1, Dm, St, G, dtype, False, True)
    one = {k: (v[:, 0] if k in ("x", "delta", "B", "C", "z") else v) for k, v in c.items()}
    ref = _ref(c, True, None, h0)
    kw = dict(D=one["D"], z=one["z"], delta_bias=one["bias"], delta_softplus=True)
    pos = [one[k] for k in ("x", "delta", "A", "B", "C")]
    before, out = h0.clone(), torch.full_like(h0, float("nan"))
    y = S.selective_scan_step(*pos, state=h0, state_out=out, **kw)
    R.close(y, ref["y"][0][:, 0], ref["y"][1][:, 0], 192, "y of a step")
    R.close(out, *ref["state"], 192, "state of a step")
    assert torch.equal(h0, before)
    cache = torch.full((Bt, 2, Dm, St), 3.0, device="cuda")  # slots of a larger tensor, in place
    cache[:, 1] = h0
    assert torch.equal(S.selective_scan_step(*pos, state=cache[:, 1], **kw), y)
    assert torch.equal(cache[:, 1], out) and (cache[:, 0] == 3).all()

    x, w, b, past, _, _, _ = _conv_case(Dm, Bt, 1, Dm, W, dtype, False, True)
    ref = R.causal_conv(x, w, b, True, None, past)
    new = torch.empty_like(past)
    y = S.causal_conv_step(x[:, 0], w, b, state=past, activation="silu", state_out=new)
    R.close(y, ref["y"][0][:, 0], ref["y"][1][:, 0], 2 * W + 32, "y of a step")
    assert torch.equal(new.double().cpu(), ref["state"][0])
    version = past._version
    assert torch.equal(S.causal_conv_step(x[:, 0], w, b, state=past, activation="silu"), y)
    assert torch.equal(past, new) and past._version > version


def test_steps_in_inference_mode():
    with torch.inference_mode():
        x, st = torch.ones(2, 8, device="cuda"), torch.zeros(2, 3, 8, device="cuda")
        S.causal_conv_step(x, torch.ones(8, 4, device="cuda"), state=st)
        assert torch.equal(st[:, -1], x)
        h = torch.zeros(2, 8, 4, device="cuda")
        S.selective_scan_step(x, x, -torch.ones(8, 4, device="cuda"), x[:, :4], x[:, :4], state=h)
        assert (h == 1).all()


def test_prompt_in_pieces_then_steps_is_one_series():
    c, _, _, _, _ = _scan_case(41, 2, 90, 24, 16, None, torch.float32, False, True)
    w = _gen(2)(24, 4)
    with torch.no_grad():
        full, _ = _run(c, True)
        fconv = S.causal_conv(c["x"], w, activation="silu")
        h = st = None
        ys, vs = [], []
        for a, b in ((0, 1), (1, 50), (50, 83)):
            piece = {k: (v[:, a:b] if k in ("x", "delta", "B", "C", "z") else v) for k, v in c.items()}
            y, h = _run(piece, True, None, h)
            v, st = S.causal_conv(piece["x"], w, activation="silu", initial_state=st, return_state=True)
            ys.append(y)
            vs.append(v)
        for t in range(83, 90):
            ys.append(S.selective_scan_step(c["x"][:, t], c["delta"][:, t], c["A"], c["B"][:, t], c["C"][:, t], D=c["D"],
                                            z=c["z"][:, t], delta_bias=c["bias"], delta_softplus=True, state=h)[:, None])
            vs.append(S.causal_conv_step(c["x"][:, t], w, state=st, activation="silu")[:, None])
    ref = _ref(c, True)
    R.close(torch.cat(ys, 1), *ref["y"], 64 * 90 + 128, "pieces")
    R.close(full, *ref["y"], 64 * 90 + 128, "whole")
    R.close(torch.cat(vs, 1), *R.causal_conv(c["x"], w, None, True)["y"], 40, "convolved pieces")
    assert fconv.shape == full.shape


# ----------------------------------------------------------------------------- streams, graphs, threads
def _block(p, x, n=None):
    """The operators as a model uses them, one after the other."""
    v = S.layer_norm(x, p["ln_w"], p["ln_b"])
    xz = v @ p["w_in"]
    u = S.causal_conv(xz[..., :32], p["conv_w"], p["conv_b"], activation="silu", lengths=n)
    dbc = u @ p["w_dbc"]
    y = S.selective_scan(u, dbc[..., :32], p["A"], dbc[..., 32:40], dbc[..., 40:], D=p["D"], z=xz[..., 32:],
                         delta_bias=p["bias"], delta_softplus=True, lengths=n)
    return x + y @ p["w_out"]


def _block_params(dtype=torch.float32, grad=True):
    rn = _gen(77)
    p = dict(ln_w=1 + rn(16) * 0.1, ln_b=rn(16) * 0.1, w_in=rn(16, 64, dtype=dtype) / 4, conv_w=rn(32, 4) / 2, conv_b=rn(32) * 0.1,
             w_dbc=rn(32, 48, dtype=dtype) / 6, A=-torch.exp(rn(32, 8) * 0.3), D=rn(32), bias=rn(32) - 2,
             w_out=rn(32, 16, dtype=dtype) / 6)
    return {k: v.requires_grad_(grad) for k, v in p.items()}


def test_block_trains_under_the_loss():
    """Norm, projection, convolution, scan, projection, and the Soft-DTW loss behind them: gradients
    against central differences of the same network in float64 on the CPU."""
    p = _block_params()
    rn = _gen(78)
    x, target = rn(3, 30, 16), rn(3, 25, 16)
    n = torch.tensor([30, 30, 30], device="cuda")
    loss = SoftDTW(gamma=1.0)(_block(p, x, n), target).mean()
    grads = torch.autograd.grad(loss, list(p.values()))
    p64 = {k: v.detach().double().cpu().requires_grad_(True) for k, v in p.items()}
    l64 = SoftDTW(gamma=1.0)(_block(p64, x.double().cpu(), n.cpu()), target.double().cpu()).mean()
    g64 = torch.autograd.grad(l64, list(p64.values()))
    # The loss's own gradient is float32 to 1e-4 (the tests' bar for it); the operators and the
    # matrix products add less.
    assert abs(loss.item() - l64.item()) <= 1e-5 * abs(l64.item())
    for k, a, b in zip(p, grads, g64):
        err = (a.double().cpu() - b).abs().max()
        assert err <= 1e-3 * b.abs().max(), (k, err, b.abs().max())
    with torch.no_grad():
        for k, step in (("A", 1e-5), ("conv_w", 1e-5), ("ln_w", 1e-5), ("bias", 1e-5)):
            d = torch.randn(p64[k].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(1))
            f = lambda s: SoftDTW(gamma=1.0)(_block({**p64, k: p64[k] + s * d}, x.double().cpu(), n.cpu()),  # noqa: E731
                                             target.double().cpu()).mean().item()
            num = (f(step) - f(-step)) / (2 * step)
            ana = (g64[list(p).index(k)] * d).sum().item()
            assert abs(num - ana) <= 1e-5 * abs(ana) + 1e-6, (k, num, ana)


def test_side_stream_and_threads_give_the_same():
    p = _block_params()
    rn = _gen(79)
    x = rn(4, 100, 16)
    n = torch.tensor([100, 3, 0, 57], device="cuda")

    def step():
        return [g.clone() for g in torch.autograd.grad(_block(p, x, n).square().sum(), list(p.values()))]

    want = step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step()
    side.synchronize()
    results = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            results.append(step())
            torch.cuda.current_stream().synchronize()

    ts = [threading.Thread(target=work) for _ in range(3)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    assert len(results) == 3
    for other in [got] + results:
        for a, b in zip(want, other):
            assert torch.equal(a, b)


def test_captured_training_steps_and_running_steps():
    """Two captured training steps replayed in turn with new inputs, and a captured single step that
    advances its state in place."""
    p = _block_params()
    rn = _gen(80)
    leaves = list(p.values())

    def train(x):
        return torch.autograd.grad(_block(p, x).square().sum(), leaves)

    xs = [rn(2, 40, 16), rn(3, 70, 16)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for x in xs:
            train(x)
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for x in xs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = train(x)
        graphs.append((g, out))
    for _ in range(2):
        for x in xs:
            x.copy_(rn(*x.shape))
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for x, (_, out) in zip(xs, graphs):
            for a, b in zip(out, train(x)):
                assert torch.equal(a, b)
    with torch.no_grad():
        c, _, h0, _, _ = _scan_case(81, 2, 4, 32, 16, None, torch.float32, False, False)
        state, xt = h0.clone(), [c[k][:, 0].clone() for k in ("x", "delta", "B", "C")]
        st, w = rn(2, 3, 32), rn(32, 4)
        conv0 = st.clone()

        def one():
            u = S.causal_conv_step(xt[0], w, state=st)
            return S.selective_scan_step(u, xt[1], c["A"], xt[2], xt[3], state=state)

        with torch.cuda.stream(side):
            one()
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = one()
        state.copy_(h0)
        st.copy_(conv0)
        got = []
        for t in range(4):
            for dst, k in zip(xt, ("x", "delta", "B", "C")):
                dst.copy_(c[k][:, t])
            g.replay()
            got.append(y.clone())
        u = S.causal_conv(c["x"], w, initial_state=conv0)
        want, last = S.selective_scan(u, c["delta"], c["A"], c["B"], c["C"], initial_state=h0, return_state=True)
        torch.testing.assert_close(torch.stack(got, 1), want, rtol=1e-5, atol=1e-5)
        torch.testing.assert_close(state, last, rtol=1e-5, atol=1e-5)


@pytest.mark.parametrize("backend", ["aot_eager", "inductor"])
def test_compiled_block_matches_eager(backend):
    p = _block_params()
    x = _gen(82)(2, 33, 16).requires_grad_(True)
    n = torch.tensor([33, 12], device="cuda")
    f = lambda x: _block(p, x, n).square().sum()  # noqa: E731
    want = torch.autograd.grad(f(x), [x, *p.values()])
    got = torch.autograd.grad(torch.compile(f, fullgraph=True, backend=backend)(x), [x, *p.values()])
    for a, b in zip(got, want):
        torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))
    with torch.no_grad():
        st = _gen(3)(2, 3, 32)
        w, xt = p["conv_w"].detach(), _gen(4)(2, 32)
        st2 = st.clone()
        want = S.causal_conv_step(xt, w, state=st)
        step = torch.compile(lambda x, s: S.causal_conv_step(x, w, state=s), fullgraph=True, backend=backend)
        assert torch.equal(step(xt, st2), want) and torch.equal(st, st2)


def test_compiled_block_with_changing_lengths():
    p = _block_params()
    f = lambda x: _block(p, x).square().sum()  # noqa: E731
    compiled = torch.compile(f, fullgraph=True, backend="aot_eager")
    for N in (33, 40, 47, 5):
        x = _gen(N)(2, N, 16).requires_grad_(True)
        want = torch.autograd.grad(f(x), [x, *p.values()])
        for a, b in zip(torch.autograd.grad(compiled(x), [x, *p.values()]), want):
            torch.testing.assert_close(a, b, rtol=1e-4, atol=1e-4 * float(b.abs().max()))


def test_opcheck():
    rn = _gen(83)
    x, w, b = rn(2, 9, 6).requires_grad_(True), rn(6).requires_grad_(True), rn(6).requires_grad_(True)
    torch.library.opcheck(torch.ops.softdtw_cuda.layer_norm_forward, (x, w, b, 1e-5))
    cw = rn(6, 3).requires_grad_(True)
    torch.library.opcheck(torch.ops.softdtw_cuda.causal_conv_forward, (x, cw, b, True, None, None, True))
    A, bc = (-torch.exp(rn(6, 4))).requires_grad_(True), rn(2, 9, 1, 4).requires_grad_(True)
    torch.library.opcheck(torch.ops.softdtw_cuda.selective_scan_forward,
                          (x, x.detach().abs(), A, bc, bc.detach(), w, None, None, False, None, None, True, True))
    torch.library.opcheck(torch.ops.softdtw_cuda.selective_scan_step,
                          (rn(2, 6), rn(2, 6).abs(), A.detach(), rn(2, 1, 4), rn(2, 1, 4), None, None, None, False, rn(2, 6, 4), None))


def test_refusals_on_the_device():
    x = torch.zeros(2, 3, 4, device="cuda")
    with pytest.raises(ValueError, match="x's device"):
        S.layer_norm(x, torch.ones(4))
    with pytest.raises(ValueError, match="x's device"):
        S.causal_conv(x, torch.ones(4, 2, device="cuda"), lengths=torch.tensor([1, 2]))
    with pytest.raises(ValueError, match="x's device"):
        S.selective_scan(x, x, -torch.ones(4, 2), x[..., :2], x[..., :2])
    p = torch.ones(4, 2, device="cuda", requires_grad=True)
    with pytest.raises(ValueError, match="not differentiable"):
        S.causal_conv_step(x[:, 0], p, state=torch.zeros(2, 1, 4, device="cuda"))


def test_kernels_are_counted_and_float64_is_not_rounded():
    rn = _gen(90)
    x = rn(2, 12, 8)
    n0 = _native.launches()
    S.layer_norm(x)
    S.causal_conv(x, rn(8, 4))
    assert _native.launches() == n0 + 2
    xd = x.double()
    torch.testing.assert_close(S.layer_norm(xd).cpu(), R.layer_norm(xd, None, None, 1e-5)["y"][0], rtol=1e-12, atol=1e-12)

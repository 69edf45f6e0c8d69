"""The sequence operators without a GPU: the torch-op formulas of CPU tensors
against the float64 references, their gradients against differences, the
argument checks, the C entry points' refusals and the fake kernels."""
import ctypes

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

import _seq_ref as R
import softdtw_cuda as S
from softdtw_cuda import _native


def _scan_inputs(seed, Bt=2, N=6, Dm=4, St=3, G=None, dtype=torch.float64):
    g = torch.Generator().manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, dtype=torch.float64)  # noqa: E731
    grp = (St,) if G is None else (G, St)
    d = dict(x=rn(Bt, N, Dm), delta=rn(Bt, N, Dm) * 0.5, A=-torch.exp(rn(Dm, St) * 0.3), B=rn(Bt, N, *grp),
             C=rn(Bt, N, *grp), D=rn(Dm), z=rn(Bt, N, Dm), delta_bias=rn(Dm) * 0.5)
    return {k: v.to(dtype) if k in ("x", "delta", "B", "C", "z") else v for k, v in d.items()}


def test_layer_norm_cpu_matches_formula_and_differences():
    torch.manual_seed(0)
    x, w, b = torch.randn(3, 5, 7, dtype=torch.float64) + 3, torch.randn(7, dtype=torch.float64), torch.randn(7, dtype=torch.float64)
    dy = torch.randn(3, 5, 7, dtype=torch.float64)
    for t in (x, w, b):
        t.requires_grad_(True)
    ref = R.layer_norm(x, w, b, 1e-3, dy)
    y = S.layer_norm(x, w, b, eps=1e-3)
    torch.testing.assert_close(y, ref["y"][0], rtol=1e-12, atol=1e-12)
    for got, k in zip(torch.autograd.grad(y, (x, w, b), dy), ("dx", "dw", "db")):
        torch.testing.assert_close(got, ref[k][0], rtol=1e-11, atol=1e-11)
    assert torch.autograd.gradcheck(lambda *a: S.layer_norm(*a, eps=1e-3), (x, w, b))
    R.close(S.layer_norm(x.detach().bfloat16()), R.layer_norm(x.detach().bfloat16(), None, None, 1e-5)["y"][0],
            R.layer_norm(x.detach().bfloat16(), None, None, 1e-5)["y"][1], 64, "bf16 on the CPU")


@pytest.mark.parametrize("W", [1, 2, 4, 8])
@pytest.mark.parametrize("act", [None, "silu"])
def test_causal_conv_cpu_matches_formula_and_differences(W, act):
    torch.manual_seed(W)
    x, w, b = (torch.randn(*s, dtype=torch.float64, requires_grad=True) for s in ((3, 6, 4), (4, W), (4,)))
    past = torch.randn(3, W - 1, 4, dtype=torch.float64, requires_grad=True)
    dy, ds = torch.randn(3, 6, 4, dtype=torch.float64), torch.randn(3, W - 1, 4, dtype=torch.float64)
    n = torch.tensor([6, 0, 2])
    ref = R.causal_conv(x, w, b, act == "silu", n, past, dy, ds)
    f = lambda *a: S.causal_conv(*a[:3], activation=act, lengths=n, initial_state=a[3], return_state=True)  # noqa: E731
    y, st = f(x, w, b, past)
    torch.testing.assert_close(y, ref["y"][0], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(st, ref["state"][0], rtol=0, atol=0)
    grads = torch.autograd.grad((y, st), (x, w, b, past), (dy, ds), allow_unused=W == 1)
    for got, k in zip(grads, ("dx", "dw", "db", "dpast")):
        if got is not None:
            torch.testing.assert_close(got, ref[k][0], rtol=1e-11, atol=1e-11)
    if W > 1:
        assert torch.autograd.gradcheck(f, (x, w, b, past))


@pytest.mark.parametrize("G", [None, 2])
@pytest.mark.parametrize("gate,softplus", [(True, True), (False, False)])
def test_selective_scan_cpu_matches_formula_and_differences(G, gate, softplus):
    p = _scan_inputs(1, G=G)
    if not gate:
        p["z"] = p["D"] = p["delta_bias"] = None
    if not softplus:
        p["delta"] = p["delta"].abs()
    leaves = {k: v.requires_grad_(True) for k, v in p.items() if v is not None}
    h0 = torch.randn(2, 4, 3, dtype=torch.float64, requires_grad=True)
    n = torch.tensor([4, 6])
    dy, dh = torch.randn(2, 6, 4, dtype=torch.float64), torch.randn(2, 4, 3, dtype=torch.float64)
    ref = R.selective_scan(p["x"], p["delta"], p["A"], p["B"], p["C"], p["D"], p["z"], p["delta_bias"], softplus, n, h0, dy, dh)

    def f(*a):
        q = dict(zip(leaves, a))
        pos = [q.pop(k) for k in ("x", "delta", "A", "B", "C")]
        return S.selective_scan(*pos, **q, delta_softplus=softplus, lengths=n, initial_state=a[-1], return_state=True)

    args = (*leaves.values(), h0)
    y, h = f(*args)
    torch.testing.assert_close(y, ref["y"][0], rtol=1e-12, atol=1e-12)
    torch.testing.assert_close(h, ref["state"][0], rtol=1e-12, atol=1e-12)
    names = {"x": "dx", "delta": "ddelta", "A": "dA", "B": "dB", "C": "dC", "D": "dD", "z": "dz", "delta_bias": "dbias"}
    grads = torch.autograd.grad((y, h), args, (dy, dh))
    for got, k in zip(grads, [names[k] for k in leaves] + ["dh0"]):
        torch.testing.assert_close(got, ref[k][0], rtol=1e-10, atol=1e-10, msg=lambda m, k=k: f"{k}: {m}")
    assert torch.autograd.gradcheck(f, args)


def test_padding_is_not_read_on_the_cpu():
    p = _scan_inputs(2)
    n = torch.tensor([3, 0])
    dead = torch.arange(6)[None, :] >= n[:, None]
    clean = S.selective_scan(p["x"], p["delta"], p["A"], p["B"], p["C"], z=p["z"], delta_softplus=True, lengths=n)
    for k in ("x", "delta", "B", "C", "z"):
        p[k] = p[k].masked_fill(dead[..., None], float("nan")).requires_grad_(True)
    y = S.selective_scan(p["x"], p["delta"], p["A"], p["B"], p["C"], z=p["z"], delta_softplus=True, lengths=n)
    assert torch.equal(y, clean)
    dy = torch.ones_like(y).masked_fill(dead[..., None], float("nan"))
    for g in torch.autograd.grad(y, [p[k] for k in ("x", "delta", "B", "C", "z")], dy):
        assert torch.isfinite(g).all() and (g[dead] == 0).all()


def test_empty_series():
    x, w = torch.zeros(2, 0, 4), torch.randn(4, 3)
    past = torch.randn(2, 2, 4)
    y, st = S.causal_conv(x, w, initial_state=past, return_state=True)
    assert y.shape == (2, 0, 4) and torch.equal(st, past)
    h0 = torch.randn(2, 4, 5)
    bc = torch.zeros(2, 0, 5)
    y, h = S.selective_scan(x, x, -torch.ones(4, 5), bc, bc, initial_state=h0, return_state=True)
    assert y.shape == (2, 0, 4) and torch.equal(h, h0)
    assert S.layer_norm(torch.zeros(0, 4)).shape == (0, 4)
    assert S.selective_scan(torch.zeros(0, 3, 4), torch.zeros(0, 3, 4), -torch.ones(4, 5), torch.zeros(0, 3, 5),
                            torch.zeros(0, 3, 5)).shape == (0, 3, 4)


def test_steps_continue_a_series_on_the_cpu():
    p = _scan_inputs(3)
    kw = dict(D=p["D"], delta_bias=p["delta_bias"], delta_softplus=True)
    y, _ = S.selective_scan(p["x"], p["delta"], p["A"], p["B"], p["C"], z=p["z"], return_state=True, **kw)
    _, h = S.selective_scan(*(p[k][:, :4] for k in ("x", "delta")), p["A"], p["B"][:, :4], p["C"][:, :4], return_state=True, **kw)
    for t in (4, 5):
        h2 = torch.empty_like(h)
        got = S.selective_scan_step(p["x"][:, t], p["delta"][:, t], p["A"], p["B"][:, t], p["C"][:, t], z=p["z"][:, t],
                                    state=h, state_out=h2, **kw)
        torch.testing.assert_close(got, y[:, t], rtol=1e-12, atol=1e-12)
        h = h2
    x, w = p["x"], torch.randn(4, 4, dtype=torch.float64)
    y = S.causal_conv(x, w, activation="silu")
    _, st = S.causal_conv(x[:, :2], w, return_state=True)
    for t in range(2, 6):
        torch.testing.assert_close(S.causal_conv_step(x[:, t], w, state=st, activation="silu"), y[:, t], rtol=1e-12, atol=1e-12)


def _step_args():
    x = torch.randn(2, 4)
    return x, x, -torch.ones(4, 3), torch.randn(2, 3), torch.randn(2, 3)


@pytest.mark.parametrize("call,error,text", [
    (lambda: S.layer_norm([1.0]), TypeError, "must be a torch.Tensor"),
    (lambda: S.layer_norm(torch.zeros(3, dtype=torch.int64)), TypeError, "Unsupported dtype"),
    (lambda: S.layer_norm(torch.zeros(3, 0)), ValueError, "last dimension"),
    (lambda: S.layer_norm(torch.zeros(3, 4), torch.ones(3)), ValueError, "weight must have shape"),
    (lambda: S.layer_norm(torch.zeros(3, 4), eps=-1.0), ValueError, "eps must be >= 0"),
    (lambda: S.causal_conv(torch.zeros(3, 4), torch.zeros(4, 2)), ValueError, "x must have shape"),
    (lambda: S.causal_conv(torch.zeros(2, 3, 4), torch.zeros(3, 2)), ValueError, "weight must have shape"),
    (lambda: S.causal_conv(torch.zeros(2, 3, 4), torch.zeros(4, 9)), ValueError, "width must be between"),
    (lambda: S.causal_conv(torch.zeros(2, 3, 4), torch.zeros(4, 2), activation="relu"), ValueError, "Unknown activation"),
    (lambda: S.causal_conv(torch.zeros(2, 3, 4), torch.zeros(4, 2), lengths=torch.ones(2)), TypeError, "int32 or int64"),
    (lambda: S.causal_conv(torch.zeros(2, 3, 4), torch.zeros(4, 2), lengths=torch.ones(3, dtype=torch.int64)), ValueError, "lengths must have shape"),
    (lambda: S.causal_conv(torch.zeros(2, 3, 4), torch.zeros(4, 3), initial_state=torch.zeros(2, 3, 4)), ValueError, "initial_state must have shape"),
    (lambda: S.causal_conv_step(torch.zeros(2, 4), torch.zeros(4, 3), state=torch.zeros(2, 2, 4, dtype=torch.float64)), TypeError, "state must be"),
    (lambda: S.causal_conv_step(torch.zeros(2, 4), torch.zeros(4, 3), state=torch.zeros(2, 4, 2).transpose(1, 2)), ValueError, "contiguously"),
    (lambda: S.causal_conv_step(torch.zeros(2, 4), torch.zeros(4, 3), state=torch.zeros(1, 2, 4).expand(2, 2, 4)), ValueError, "contiguously"),
    (lambda: S.causal_conv_step(torch.zeros(2, 4), torch.zeros(4, 3, requires_grad=True), state=torch.zeros(2, 2, 4)), ValueError, "not differentiable"),
    (lambda: S.selective_scan(torch.zeros(2, 3, 4), torch.zeros(2, 3, 5), -torch.ones(4, 2), torch.zeros(2, 3, 2), torch.zeros(2, 3, 2)), ValueError, "delta must have shape"),
    (lambda: S.selective_scan(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4).half(), -torch.ones(4, 2), torch.zeros(2, 3, 2), torch.zeros(2, 3, 2)), TypeError, "x's dtype"),
    (lambda: S.selective_scan(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), -torch.ones(4, 65), torch.zeros(2, 3, 65), torch.zeros(2, 3, 65)), ValueError, "state size"),
    (lambda: S.selective_scan(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), -torch.ones(4, 2), torch.zeros(2, 3, 3, 2), torch.zeros(2, 3, 3, 2)), ValueError, "must divide"),
    (lambda: S.selective_scan(torch.zeros(2, 3, 4), torch.zeros(2, 3, 4), -torch.ones(4, 2), torch.zeros(2, 3, 2), torch.zeros(2, 3, 1, 2)), ValueError, "C must have shape"),
    (lambda: S.selective_scan_step(*_step_args(), state=torch.zeros(2, 4, 2)), ValueError, "state must have shape"),
    (lambda: S.selective_scan_step(*_step_args(), state=torch.zeros(2, 4, 3, dtype=torch.float64)), TypeError, "state must be"),
])
def test_refusals(call, error, text):
    with pytest.raises(error, match=text):
        call()


def test_overlapping_states_are_refused_and_interleaved_ones_are_not():
    args = _step_args()
    buf = torch.randn(3, 4, 3)
    with pytest.raises(ValueError, match="overlaps"):
        S.selective_scan_step(*args, state=buf[:2], state_out=buf[1:])
    cache = torch.randn(2, 2, 4, 3)  # two slots per series
    ref = cache[:, 0].clone()
    y = S.selective_scan_step(*args, state=ref)
    y2 = S.selective_scan_step(*args, state=cache[:, 0], state_out=cache[:, 1])
    assert torch.equal(y, y2) and torch.equal(cache[:, 1], ref)


def test_c_entry_points_refuse_bad_arguments():
    L = _native.lib()
    msg = lambda: L.sdtw_last_error_message()  # noqa: E731
    for fn in ("layer_norm_forward", "layer_norm_backward", "conv_forward", "conv_backward", "conv_step", "scan_forward",
               "scan_backward", "scan_step"):
        assert getattr(L, f"sdtw_{fn}")(None, None) == 1 and b"null pointer" in msg()
    buf = (ctypes.c_float * 64)()
    p = ctypes.addressof(buf)
    ln = _native.LayerNormArgs(dtype=3, dim=4, rows=1, x=p, y=p)
    assert L.sdtw_layer_norm_forward(ctypes.byref(ln), None) == 1 and b"dtype" in msg()
    ln.dtype, ln.rows = 0, 0
    assert L.sdtw_layer_norm_forward(ctypes.byref(ln), None) == 1 and b"must be > 0" in msg()
    ln.rows, ln.eps = 1, -1.0
    assert L.sdtw_layer_norm_forward(ctypes.byref(ln), None) == 1 and b"eps" in msg()
    ln.mean = ln.rstd = ln.dy = ln.dweight = p
    assert L.sdtw_layer_norm_backward(ctypes.byref(ln), None) == 1 and b"workspace" in msg()
    c = _native.ConvArgs(batch=1, length=2, dim=4, width=9, x=p, weight=p, y=p, dy=p)
    assert L.sdtw_conv_forward(ctypes.byref(c), None) == 1 and b"width" in msg()
    c.width = 3
    assert L.sdtw_conv_step(ctypes.byref(c), None) == 1 and b"length 1" in msg()
    c.dweight = p
    assert L.sdtw_conv_backward(ctypes.byref(c), None) == 1 and b"workspace" in msg()
    s = _native.ScanArgs(batch=1, length=2, dim=4, groups=3, nstate=2, x=p, delta=p, A=p, B=p, C=p, y=p, dy=p, saved=p)
    assert L.sdtw_scan_forward(ctypes.byref(s), None) == 1 and b"groups" in msg()
    s.groups, s.nstate = 1, 65
    assert L.sdtw_scan_forward(ctypes.byref(s), None) == 1 and b"nstate" in msg()
    s.nstate = 2
    assert L.sdtw_scan_backward(ctypes.byref(s), None) == 1 and b"workspace" in msg()
    assert L.sdtw_scan_step(ctypes.byref(s), None) == 1 and b"length 1" in msg()
    assert L.sdtw_scan_workspace_bytes(1, 2, 4, 3, 2) == 0 and L.sdtw_scan_workspace_bytes(1, 2, 4, 2, 65) == 0
    assert L.sdtw_scan_saved_elems(3, 33, 5, 7) % (3 * 5 * 7) == 0


def test_fake_shapes():
    with FakeTensorMode():
        x = torch.empty(2, 40, 6, device="cuda", dtype=torch.bfloat16)
        f = lambda *s: torch.empty(*s, device="cuda")  # noqa: E731
        y, stats = torch.ops.softdtw_cuda.layer_norm_forward(x, f(6), None, 1e-5)
        assert y.shape == x.shape and y.dtype == x.dtype and stats.shape == (2, 80)
        y, st = torch.ops.softdtw_cuda.causal_conv_forward(x, f(6, 4), None, True, None, None, True)
        assert y.shape == x.shape and st.shape == (2, 3, 6)
        B = torch.empty(2, 40, 2, 5, device="cuda", dtype=torch.bfloat16)
        y, h, saved = torch.ops.softdtw_cuda.selective_scan_forward(x, x, f(6, 5), B, B, None, x, None, True, None, None, True, True)
        assert y.shape == x.shape and h.shape == (2, 6, 5) and saved.shape == (_native.scan_saved_elems(2, 40, 6, 5),)
        need = [True, False, True, True, False, True, True, False, False]
        g = torch.ops.softdtw_cuda.selective_scan_backward(x, x, f(6, 5), B, B, None, x, None, True, None, saved, y, None, need)
        assert g[0].shape == x.shape and g[1].numel() == 0 and g[2].shape == (6, 5) and g[3].shape == B.shape

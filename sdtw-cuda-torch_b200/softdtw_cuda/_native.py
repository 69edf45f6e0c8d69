"""ctypes binding of libsdtw_b200.so (the C ABI declared in include/sdtw_b200.h).

Every CUDA tensor operation of the package goes through this module.  There is
no fallback: if the library is missing or a call fails, a RuntimeError is
raised.  PyTorch supplies device memory (outputs and workspaces) and the
current CUDA stream; the kernels are the library's.
"""
from __future__ import annotations

import contextlib
import ctypes
import os
import struct
import threading

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "_lib", "libsdtw_b200.so")

_lib = None
_lock = threading.Lock()

_P = ctypes.c_void_p
_I = ctypes.c_int
_F = ctypes.c_float
_Dbl = ctypes.c_double
_SZ = ctypes.c_size_t

_SIGS = {
    "sdtw_version": ([], ctypes.c_char_p),
    "sdtw_error_string": ([_I], ctypes.c_char_p),
    "sdtw_last_error_message": ([], ctypes.c_char_p),
    "sdtw_status": ([], _I),
    "sdtw_set_wait_timeout_ns": ([ctypes.c_ulonglong], None),
    "sdtw_debug_stall_stripe": ([_I], None),
    "sdtw_timing_enable": ([_I], None),
    "sdtw_timing_read": ([ctypes.c_char_p, _SZ, _P, _P, _I], _I),
    "sdtw_set_plan_override": ([_I, _I, _I], None),
    "sdtw_plan_info": ([_I, _I, _I, _P], _I),
    "sdtw_launch_count": ([], ctypes.c_ulonglong),
    "sdtw_score_elems": ([_I, _I, _I], _SZ),
    "sdtw_cost_elems": ([_I, _I, _I], _SZ),
    "sdtw_workspace_bytes": ([_I, _I, _I], _SZ),
    "sdtw_workspace_bytes_xy": ([_I, _I, _I, _I], _SZ),
    "sdtw_cost_sqeuclid_f32": ([_P, _P, _P, _I, _I, _I, _I, _I, _P], _I),
    "sdtw_forward_f32": ([_P, _P, _P, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_backward_f32": ([_P, _P, _P, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_forward_xy_f32": ([_P, _P, _P, _P, _I, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_backward_xy_f32": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_forward_noalloc_f32": ([_P, _P, _P, _I, _I, _I, _F, _F, _P], _I),
    "sdtw_forward_sqeuclid_f32": ([_P, _P, _P, _P, _P, _I, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_backward_sqeuclid_f32": ([_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_grad_sqeuclid_f32": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _I, _P], _I),
    "sdtw_workspace_bytes_norm": ([_I, _I, _I], _SZ),
    "sdtw_forward_xy_norm_f32": ([_P, _P, _P, _P, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_backward_xy_norm_f32": ([_P, _P, _P, _P, _P, _P, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_forward_sqeuclid_norm_f32": ([_P, _P, _P, _P, _P, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_backward_sqeuclid_norm_f32": ([_P, _P, _P, _P, _P, _P, _P, _I, _I, _I, _F, _F, _P, _SZ, _P], _I),
    "sdtw_score_to_R_f32": ([_P, _P, _I, _I, _I, _F, _P], _I),
    "sdtw_R_to_score_f32": ([_P, _P, _I, _I, _I, _F, _P], _I),
    "sdtw_forward_f64": ([_P, _P, _P, _I, _I, _I, _Dbl, _Dbl, _P], _I),
    "sdtw_backward_f64": ([_P, _P, _P, _P, _I, _I, _I, _Dbl, _Dbl, _P], _I),
    "sdtw_cost_sqeuclid_f64": ([_P, _P, _P, _I, _I, _I, _I, _P], _I),
    "sdtw_grad_sqeuclid_f64": ([_P, _P, _P, _P, _P, _I, _I, _I, _I, _P], _I),
    "sdtw_barycenter_workspace_bytes": ([_I, _I, _I, _I], _SZ),
    "sdtw_barycenter_grad_f32": ([_P, _P, _P, _P, _I, _I, _I, _I, _F, _P, _SZ, _P], _I),
    "sdtw_barycenter_adam_f32": ([_P, _P, _P, _P, _SZ, _P, _I, _P, _P, _P, _F, _F, _F, _F, _P], _I),
    "sdtw_barycenter_sync_bytes": ([_SZ, _I], _SZ),
    "sdtw_barycenter_sync_adam_f32": ([_P, _SZ, _P, _I, _I, _P, _P, _P, _P, _P, _I, _P, _P, _P, _F, _F, _F, _F, _P],
                                      _I),
    "sdtw_layer_norm_workspace_bytes": ([ctypes.c_longlong, _I], _SZ),
    "sdtw_layer_norm_forward": ([_P, _P], _I),
    "sdtw_layer_norm_backward": ([_P, _P], _I),
    "sdtw_conv_workspace_bytes": ([_I, _I, _I, _I], _SZ),
    "sdtw_conv_forward": ([_P, _P], _I),
    "sdtw_conv_backward": ([_P, _P], _I),
    "sdtw_conv_step": ([_P, _P], _I),
    "sdtw_scan_saved_elems": ([_I, _I, _I, _I], _SZ),
    "sdtw_scan_forward_workspace_bytes": ([_I, _I, _I, _I, _I], _SZ),
    "sdtw_scan_workspace_bytes": ([_I, _I, _I, _I, _I], _SZ),
    "sdtw_scan_forward": ([_P, _P], _I),
    "sdtw_scan_backward": ([_P, _P], _I),
    "sdtw_scan_step": ([_P, _P], _I),
    "sdtw_cpu_forward_f64": ([_P, _P, _P, _I, _I, _I, _Dbl, _Dbl], _I),
    "sdtw_cpu_backward_f64": ([_P, _P, _P, _I, _I, _I, _Dbl, _Dbl], _I),
}

# Every symbol the header declares (tests check the library exports them).
EXPORTED = tuple(_SIGS)


def lib():
    """Load the library once (RuntimeError if it has not been built)."""
    global _lib
    if _lib is not None:
        return _lib
    with _lock:
        if _lib is None:
            if not os.path.exists(LIB_PATH):
                raise RuntimeError(
                    f"softdtw_cuda: native library {LIB_PATH} is missing; build it with "
                    "`python -m softdtw_cuda._build` (or __graft_entry__.build())")
            L = ctypes.CDLL(LIB_PATH)
            for name, (args, res) in _SIGS.items():
                fn = getattr(L, name)
                fn.argtypes = args
                fn.restype = res
            _lib = L
    return _lib


class NativeError(RuntimeError):
    pass


def launches() -> int:
    """Kernels the library has launched since it was loaded (its own counter)."""
    return int(lib().sdtw_launch_count())


# When a list, every op appends (name, start_event, end_event) recorded on the
# stream it launched on (used by bench.py for per-kernel timing).
profile_events = None


def _op_begin(device):
    if profile_events is None:
        return None
    ev = torch.cuda.Event(enable_timing=True)
    ev.record(torch.cuda.current_stream(device))
    return ev


def _op_end(name, device, ev0, n_kernels=None):
    if ev0 is not None:
        ev1 = torch.cuda.Event(enable_timing=True)
        ev1.record(torch.cuda.current_stream(device))
        profile_events.append((name, ev0, ev1))


def _check(rc: int, what: str) -> None:
    if rc != 0:
        L = lib()
        msg = L.sdtw_last_error_message().decode(errors="replace")
        kind = L.sdtw_error_string(rc).decode(errors="replace")
        raise NativeError(f"softdtw_cuda: {what} failed: {kind}: {msg}")


def _ptr(t: torch.Tensor | None):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


_SAME_DEVICE = contextlib.nullcontext()


def _on(device: torch.device):
    """The device's context for a library call: a no-op when it is already current."""
    if device.index is None or device.index == torch.cuda.current_device():
        return _SAME_DEVICE
    return torch.cuda.device(device)


def _stream(device: torch.device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def status() -> int:
    """Read and clear the device wait status (0 = ok).  Synchronise first."""
    return int(lib().sdtw_status())


def check_status(device=None) -> None:
    """Synchronise ``device`` and raise if a device-side wait timed out."""
    if torch.cuda.is_available():
        torch.cuda.synchronize(device)
    s = status()
    if s != 0:
        raise NativeError(f"softdtw_cuda: device-side wait failed (status {s}): "
                          f"{lib().sdtw_last_error_message().decode(errors='replace')}")


def set_plan_override(warps_per_cta: int = 0, cluster_size: int = 0, rows_per_lane: int = 0) -> None:
    """Force the wavefront launch geometry (zeros restore the automatic plan).
    A forward and its backward must run under the same rows_per_lane."""
    lib().sdtw_set_plan_override(int(warps_per_cta), int(cluster_size), int(rows_per_lane))


def plan_info(B: int, N: int, M: int) -> dict:
    """Launch geometry the library chooses for a (B, N, M) problem on the
    current device (diagnostic)."""
    info = (ctypes.c_int * 6)()
    _check(lib().sdtw_plan_info(int(B), int(N), int(M), info), "plan_info")
    keys = ("rows_per_lane", "warps_per_cta", "cluster_size", "bands", "stripes", "clusters_fit")
    return dict(zip(keys, list(info)))


def set_wait_timeout(seconds: float) -> None:
    lib().sdtw_set_wait_timeout_ns(int(seconds * 1e9))


def debug_stall_stripe(stripe: int) -> None:
    lib().sdtw_debug_stall_stripe(int(stripe))


def timing_enable(on: bool = True) -> None:
    """Bracket every library kernel with CUDA events on its stream (clears totals)."""
    lib().sdtw_timing_enable(1 if on else 0)


def timing_read() -> dict:
    """{kernel name: (total ms, launches)} since timing_enable (synchronises the events)."""
    import numpy as np
    buf = ctypes.create_string_buffer(4096)
    ms = np.zeros(64, dtype=np.float64)
    cnt = np.zeros(64, dtype=np.int64)
    n = lib().sdtw_timing_read(buf, 4096, ms.ctypes.data_as(ctypes.c_void_p), cnt.ctypes.data_as(ctypes.c_void_p), 64)
    names = buf.value.decode().split(",") if n else []
    return {names[i]: (float(ms[i]), int(cnt[i])) for i in range(n)}


def version() -> str:
    return lib().sdtw_version().decode()


# ----------------------------------------------------------------------------- sizes
def score_elems(B: int, N: int, M: int) -> int:
    return int(lib().sdtw_score_elems(B, N, M))


def cost_elems(B: int, N: int, M: int) -> int:
    return int(lib().sdtw_cost_elems(B, N, M))


def workspace(B: int, N: int, M: int, device, dim: int | None = None) -> torch.Tensor:
    """Caller-owned scratch of the size the library asks for (torch allocations
    are 256-byte aligned, as the library requires)."""
    L = lib()
    n = L.sdtw_workspace_bytes(B, N, M) if dim is None else L.sdtw_workspace_bytes_xy(B, N, M, dim)
    return torch.empty(max(int(n), 256), dtype=torch.uint8, device=device)


def _f32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype is torch.float32 and t.is_contiguous():
        return t.detach()
    return t.detach().to(dtype=torch.float32).contiguous()


# ----------------------------------------------------------------------------- CUDA ops
def barycenter_workspace(B: int, N: int, M: int, dim: int, device) -> torch.Tensor:
    n = lib().sdtw_barycenter_workspace_bytes(B, N, M, dim)
    return torch.empty(max(int(n), 256), dtype=torch.uint8, device=device)


def barycenter_grad(bary: torch.Tensor, X: torch.Tensor, w: torch.Tensor, grad_loss: torch.Tensor, gamma: float,
                    ws: torch.Tensor) -> None:
    """grad_loss (N*D + 1,) <- [sum_b w_b dSoftDTW(bary, X_b)/dbary | sum_b w_b SoftDTW(bary, X_b)].
    All operands contiguous float32 on one device (not copied: the call can
    be captured in a CUDA graph)."""
    B, M, dim = X.shape
    N = bary.shape[0]
    for t in (bary, X, w, grad_loss):
        if t.dtype != torch.float32 or not t.is_contiguous() or t.device != X.device:
            raise ValueError("barycenter_grad: operands must be contiguous float32 tensors on one device")
    if bary.shape != (N, dim) or w.shape != (B,) or grad_loss.numel() != N * dim + 1:
        raise ValueError("barycenter_grad: shape mismatch")
    with _on(X.device):
        rc = lib().sdtw_barycenter_grad_f32(_ptr(bary), _ptr(X), _ptr(w), _ptr(grad_loss), B, N, M, dim,
                                            float(gamma), _ptr(ws), ws.numel(), _stream(X.device))
    _check(rc, "barycenter gradient")


def barycenter_adam(bary, exp_avg, exp_avg_sq, grad_loss, lr_table, step, loss_hist, bary_hist,
                    beta1=0.9, beta2=0.999, eps=1e-8, max_norm=1.0) -> None:
    """Clip grad_loss[:n] to max_norm, one Adam step on bary with lr_table[step],
    record the loss and the new bary at index step, step += 1 (all on the device)."""
    n = bary.numel()
    if step.dtype != torch.int32:
        raise ValueError("barycenter_adam: step must be an int32 tensor")
    with _on(bary.device):
        rc = lib().sdtw_barycenter_adam_f32(_ptr(bary), _ptr(exp_avg), _ptr(exp_avg_sq), _ptr(grad_loss), n,
                                            _ptr(lr_table), lr_table.numel(), _ptr(step), _ptr(loss_hist),
                                            _ptr(bary_hist), float(beta1), float(beta2), float(eps), float(max_norm),
                                            _stream(bary.device))
    _check(rc, "barycenter Adam step")


def barycenter_sync_bytes(n: int, world: int) -> int:
    return int(lib().sdtw_barycenter_sync_bytes(n, world))


def barycenter_sync_adam(grad_loss, peers, world, rank, epoch, bary, exp_avg, exp_avg_sq, lr_table, step, loss_hist,
                         bary_hist, beta1=0.9, beta2=0.999, eps=1e-8, max_norm=1.0) -> None:
    """Sum grad_loss (n + 1,) over the ranks through the exchange buffers whose
    addresses `peers` (int64 device tensor, one per rank) holds, then the Adam
    step of barycenter_adam.  `epoch`: int64 device counter (zero at first)."""
    n = bary.numel()
    if step.dtype != torch.int32 or epoch.dtype != torch.int64 or peers.dtype != torch.int64:
        raise ValueError("barycenter_sync_adam: step int32, epoch and peers int64 tensors")
    with _on(bary.device):
        rc = lib().sdtw_barycenter_sync_adam_f32(_ptr(grad_loss), n, _ptr(peers), int(world), int(rank), _ptr(epoch),
                                                 _ptr(bary), _ptr(exp_avg), _ptr(exp_avg_sq), _ptr(lr_table),
                                                 lr_table.numel(), _ptr(step), _ptr(loss_hist), _ptr(bary_hist),
                                                 float(beta1), float(beta2), float(eps), float(max_norm),
                                                 _stream(bary.device))
    _check(rc, "barycenter exchange and Adam step")


def cost_sqeuclid(x: torch.Tensor, y: torch.Tensor, direct: bool = False) -> torch.Tensor:
    x = _f32(x)
    y = _f32(y)
    B, N, dim = x.shape
    M = y.shape[1]
    D = torch.empty((B, N, M), dtype=torch.float32, device=x.device)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_cost_sqeuclid_f32(_ptr(x), _ptr(y), _ptr(D), B, N, M, dim, int(direct), _stream(x.device))
    _check(rc, "cost")
    _op_end("cost", x.device, ev)
    return D


def forward(D: torch.Tensor, gamma: float, bandwidth: float):
    """(out (B,), score) for a CUDA cost tensor D (B,N,M)."""
    D = _f32(D)
    B, N, M = D.shape
    score = torch.empty(score_elems(B, N, M), dtype=torch.float32, device=D.device)
    out = torch.empty(B, dtype=torch.float32, device=D.device)
    ws = workspace(B, N, M, D.device)
    ev = _op_begin(D.device)
    with _on(D.device):
        rc = lib().sdtw_forward_f32(_ptr(D), _ptr(score), _ptr(out), B, N, M, float(gamma), float(bandwidth),
                                    _ptr(ws), ws.numel(), _stream(D.device))
    _check(rc, "forward")
    _op_end("forward", D.device, ev)
    return out, score


def backward(score: torch.Tensor, grad_out: torch.Tensor | None, B: int, N: int, M: int, gamma: float,
             bandwidth: float) -> torch.Tensor:
    """E (B,N,M) = grad_out[b] * dR[N,M]/dD."""
    dev = score.device
    E = torch.empty((B, N, M), dtype=torch.float32, device=dev)
    g = None if grad_out is None else _f32(grad_out.reshape(-1))
    ws = workspace(B, N, M, dev)
    ev = _op_begin(dev)
    with _on(dev):
        rc = lib().sdtw_backward_f32(_ptr(score), _ptr(g), _ptr(E), B, N, M, float(gamma), float(bandwidth),
                                     _ptr(ws), ws.numel(), _stream(dev))
    _check(rc, "backward")
    _op_end("backward", dev, ev)
    return E


def forward_xy(x: torch.Tensor, y: torch.Tensor, gamma: float, bandwidth: float):
    x = _f32(x)
    y = _f32(y)
    B, N, dim = x.shape
    M = y.shape[1]
    score = torch.empty(score_elems(B, N, M), dtype=torch.float32, device=x.device)
    out = torch.empty(B, dtype=torch.float32, device=x.device)
    ws = workspace(B, N, M, x.device, dim)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_forward_xy_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(out), B, N, M, dim, float(gamma),
                                       float(bandwidth), _ptr(ws), ws.numel(), _stream(x.device))
    _check(rc, "fused forward")
    _op_end("forward_xy", x.device, ev)
    return out, score


def backward_xy(x: torch.Tensor, y: torch.Tensor, score: torch.Tensor, grad_out: torch.Tensor | None,
                gamma: float, bandwidth: float, need_x: bool = True, need_y: bool = True):
    x = _f32(x)
    y = _f32(y)
    B, N, dim = x.shape
    M = y.shape[1]
    gx = torch.empty_like(x) if need_x else None
    gy = torch.empty_like(y) if need_y else None
    g = None if grad_out is None else _f32(grad_out.reshape(-1))
    ws = workspace(B, N, M, x.device, dim)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_backward_xy_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(g), _ptr(gx), _ptr(gy), B, N, M, dim,
                                        float(gamma), float(bandwidth), _ptr(ws), ws.numel(), _stream(x.device))
    _check(rc, "fused backward")
    _op_end("backward_xy", x.device, ev, 2 + int(need_x) + int(need_y))
    return gx, gy


def forward_sqeuclid(x: torch.Tensor, y: torch.Tensor, gamma: float, bandwidth: float):
    """Unfused path: (out, score, cost) with the clamped expanded cost kept for the backward."""
    x = _f32(x)
    y = _f32(y)
    B, N, dim = x.shape
    M = y.shape[1]
    score = torch.empty(score_elems(B, N, M), dtype=torch.float32, device=x.device)
    cost = torch.empty(cost_elems(B, N, M), dtype=torch.float32, device=x.device)
    out = torch.empty(B, dtype=torch.float32, device=x.device)
    ws = workspace(B, N, M, x.device)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_forward_sqeuclid_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(cost), _ptr(out), B, N, M, dim,
                                             float(gamma), float(bandwidth), _ptr(ws), ws.numel(), _stream(x.device))
    _check(rc, "unfused forward")
    _op_end("forward_sqeuclid", x.device, ev)
    return out, score, cost


def backward_sqeuclid(x: torch.Tensor, y: torch.Tensor, score: torch.Tensor, cost: torch.Tensor,
                      grad_out: torch.Tensor | None, gamma: float, bandwidth: float, need_x: bool = True,
                      need_y: bool = True):
    x = _f32(x)
    y = _f32(y)
    B, N, dim = x.shape
    M = y.shape[1]
    gx = torch.empty_like(x) if need_x else None
    gy = torch.empty_like(y) if need_y else None
    g = None if grad_out is None else _f32(grad_out.reshape(-1))
    ws = workspace(B, N, M, x.device, dim)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_backward_sqeuclid_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(cost), _ptr(g), _ptr(gx), _ptr(gy),
                                              B, N, M, dim, float(gamma), float(bandwidth), _ptr(ws), ws.numel(),
                                              _stream(x.device))
    _check(rc, "unfused backward")
    _op_end("backward_sqeuclid", x.device, ev, 2 + int(need_x) + int(need_y))
    return gx, gy


# ----------------------------------------------------------------------------- normalize=True
# The 3B problems (x_b, y_b), (x_b, x_b), (y_b, y_b) read x and y in place
# (softdtw_cuda/module.py:99-111 of the reference concatenates copies).
def _norm_pair(x: torch.Tensor, y: torch.Tensor):
    if x.dim() != 3 or x.shape != y.shape or not (x.is_cuda and y.is_cuda) or x.device != y.device:
        raise ValueError(f"normalize: expected CUDA x, y of one shape (B,N,D); got {tuple(x.shape)}, {tuple(y.shape)}")
    return _f32(x), _f32(y)


def _norm_ws(B: int, N: int, dim: int, device) -> torch.Tensor:
    n = lib().sdtw_workspace_bytes_norm(B, N, dim)
    return torch.empty(max(int(n), 256), dtype=torch.uint8, device=device)


def forward_xy_norm(x: torch.Tensor, y: torch.Tensor, gamma: float, bandwidth: float):
    """Fused forward of the normalized triple: (out (3B,) [xy | xx | yy], score)."""
    x, y = _norm_pair(x, y)
    B, N, dim = x.shape
    score = torch.empty(score_elems(3 * B, N, N), dtype=torch.float32, device=x.device)
    out = torch.empty(3 * B, dtype=torch.float32, device=x.device)
    ws = workspace(3 * B, N, N, x.device, dim)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_forward_xy_norm_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(out), B, N, dim, float(gamma),
                                            float(bandwidth), _ptr(ws), ws.numel(), _stream(x.device))
    _check(rc, "fused normalized forward")
    _op_end("forward_xy", x.device, ev)
    return out, score


def backward_xy_norm(x: torch.Tensor, y: torch.Tensor, score: torch.Tensor, grad_out: torch.Tensor | None,
                     gamma: float, bandwidth: float):
    """grad_x, grad_y of sum_p grad_out[p] * out[p] over the normalized triple."""
    x, y = _norm_pair(x, y)
    B, N, dim = x.shape
    gx = torch.empty_like(x)
    gy = torch.empty_like(y)
    g = None if grad_out is None else _f32(grad_out.reshape(-1))
    if g is not None and g.numel() != 3 * B:
        raise ValueError(f"normalize: expected {3 * B} upstream gradients, got {g.numel()}")
    ws = _norm_ws(B, N, dim, x.device)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_backward_xy_norm_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(g), _ptr(gx), _ptr(gy), B, N, dim,
                                             float(gamma), float(bandwidth), _ptr(ws), ws.numel(), _stream(x.device))
    _check(rc, "fused normalized backward")
    _op_end("backward_xy", x.device, ev)
    return gx, gy


def forward_sqeuclid_norm(x: torch.Tensor, y: torch.Tensor, gamma: float, bandwidth: float):
    """Unfused forward of the normalized triple: (out (3B,), score, cost)."""
    x, y = _norm_pair(x, y)
    B, N, dim = x.shape
    score = torch.empty(score_elems(3 * B, N, N), dtype=torch.float32, device=x.device)
    cost = torch.empty(cost_elems(3 * B, N, N), dtype=torch.float32, device=x.device)
    out = torch.empty(3 * B, dtype=torch.float32, device=x.device)
    ws = workspace(3 * B, N, N, x.device)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_forward_sqeuclid_norm_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(cost), _ptr(out), B, N, dim,
                                                  float(gamma), float(bandwidth), _ptr(ws), ws.numel(),
                                                  _stream(x.device))
    _check(rc, "unfused normalized forward")
    _op_end("forward_sqeuclid", x.device, ev)
    return out, score, cost


def backward_sqeuclid_norm(x: torch.Tensor, y: torch.Tensor, score: torch.Tensor, cost: torch.Tensor,
                           grad_out: torch.Tensor | None, gamma: float, bandwidth: float):
    x, y = _norm_pair(x, y)
    B, N, dim = x.shape
    gx = torch.empty_like(x)
    gy = torch.empty_like(y)
    g = None if grad_out is None else _f32(grad_out.reshape(-1))
    if g is not None and g.numel() != 3 * B:
        raise ValueError(f"normalize: expected {3 * B} upstream gradients, got {g.numel()}")
    ws = _norm_ws(B, N, dim, x.device)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_backward_sqeuclid_norm_f32(_ptr(x), _ptr(y), _ptr(score), _ptr(cost), _ptr(g), _ptr(gx),
                                                   _ptr(gy), B, N, dim, float(gamma), float(bandwidth), _ptr(ws),
                                                   ws.numel(), _stream(x.device))
    _check(rc, "unfused normalized backward")
    _op_end("backward_sqeuclid", x.device, ev)
    return gx, gy


def grad_sqeuclid(G: torch.Tensor, D_mask: torch.Tensor | None, x: torch.Tensor, y: torch.Tensor,
                  need_x: bool = True, need_y: bool = True):
    G = _f32(G)
    x = _f32(x)
    y = _f32(y)
    Dm = None if D_mask is None else _f32(D_mask)
    B, N, dim = x.shape
    M = y.shape[1]
    gx = torch.empty_like(x) if need_x else None
    gy = torch.empty_like(y) if need_y else None
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_grad_sqeuclid_f32(_ptr(G), _ptr(Dm), _ptr(x), _ptr(y), _ptr(gx), _ptr(gy), B, N, M, dim,
                                          _stream(x.device))
    _check(rc, "cost gradient")
    _op_end("grad_sqeuclid", x.device, ev, int(need_x) + int(need_y))
    return gx, gy


def score_to_R(score: torch.Tensor, B: int, N: int, M: int, gamma: float) -> torch.Tensor:
    R = torch.empty((B, N + 2, M + 2), dtype=torch.float32, device=score.device)
    with _on(score.device):
        rc = lib().sdtw_score_to_R_f32(_ptr(score), _ptr(R), B, N, M, float(gamma), _stream(score.device))
    _check(rc, "score_to_R")
    _op_end("score_to_R", score.device, None)
    return R


def R_to_score(R: torch.Tensor, gamma: float) -> torch.Tensor:
    R = _f32(R)
    B, N2, M2 = R.shape
    N, M = N2 - 2, M2 - 2
    score = torch.empty(score_elems(B, N, M), dtype=torch.float32, device=R.device)
    with _on(R.device):
        rc = lib().sdtw_R_to_score_f32(_ptr(R), _ptr(score), B, N, M, float(gamma), _stream(R.device))
    _check(rc, "R_to_score")
    _op_end("R_to_score", R.device, None)
    return score


# ----------------------------------------------------------------------------- CUDA float64 ops
def _f64(t: torch.Tensor) -> torch.Tensor:
    return t.detach().to(dtype=torch.float64).contiguous()


def forward_f64(D: torch.Tensor, gamma: float, bandwidth: float):
    """(out (B,), R (B,N+2,M+2)) in float64 for a CUDA float64 cost tensor."""
    D = _f64(D)
    B, N, M = D.shape
    R = torch.empty((B, N + 2, M + 2), dtype=torch.float64, device=D.device)
    out = torch.empty(B, dtype=torch.float64, device=D.device)
    ev = _op_begin(D.device)
    with _on(D.device):
        rc = lib().sdtw_forward_f64(_ptr(D), _ptr(R), _ptr(out), B, N, M, float(gamma), float(bandwidth),
                                    _stream(D.device))
    _check(rc, "float64 forward")
    _op_end("forward_f64", D.device, ev)
    return out, R


def backward_f64(D: torch.Tensor, R: torch.Tensor, grad_out: torch.Tensor | None, gamma: float,
                 bandwidth: float) -> torch.Tensor:
    """E (B,N,M) = grad_out[b] * dR[N,M]/dD in float64 on the GPU."""
    D = _f64(D)
    B, N, M = D.shape
    E = torch.empty((B, N, M), dtype=torch.float64, device=D.device)
    g = None if grad_out is None else grad_out.detach().reshape(-1).to(device=D.device, dtype=torch.float64).contiguous()
    ev = _op_begin(D.device)
    with _on(D.device):
        rc = lib().sdtw_backward_f64(_ptr(D), _ptr(R), _ptr(g), _ptr(E), B, N, M, float(gamma), float(bandwidth),
                                     _stream(D.device))
    _check(rc, "float64 backward")
    _op_end("backward_f64", D.device, ev)
    return E


def cost_sqeuclid_f64(x: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
    """D = sum_k (x_ik - y_jk)^2 in float64 on the GPU (the fused cost's direct form)."""
    x = _f64(x)
    y = _f64(y)
    B, N, dim = x.shape
    M = y.shape[1]
    D = torch.empty((B, N, M), dtype=torch.float64, device=x.device)
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_cost_sqeuclid_f64(_ptr(x), _ptr(y), _ptr(D), B, N, M, dim, _stream(x.device))
    _check(rc, "float64 cost")
    _op_end("cost_f64", x.device, ev)
    return D


def grad_sqeuclid_f64(G: torch.Tensor, x: torch.Tensor, y: torch.Tensor, need_x: bool = True,
                      need_y: bool = True):
    """grad_x = 2 (x rowsum(G) - G y), grad_y = 2 (y colsum(G) - G^T x) in float64 on the GPU."""
    G = _f64(G)
    x = _f64(x)
    y = _f64(y)
    B, N, dim = x.shape
    M = y.shape[1]
    gx = torch.empty_like(x) if need_x else None
    gy = torch.empty_like(y) if need_y else None
    ev = _op_begin(x.device)
    with _on(x.device):
        rc = lib().sdtw_grad_sqeuclid_f64(_ptr(G), _ptr(x), _ptr(y), _ptr(gx), _ptr(gy), B, N, M, dim,
                                          _stream(x.device))
    _check(rc, "float64 chain rule")
    _op_end("grad_f64", x.device, ev)
    return gx, gy


# ----------------------------------------------------------------------------- CPU ops
def cpu_forward(D: torch.Tensor, gamma: float, bandwidth: float):
    """(out, R) in float64 for a CPU cost tensor; R uses the reference layout."""
    Dd = D.detach().to(dtype=torch.float64).contiguous()
    B, N, M = Dd.shape
    R = torch.empty((B, N + 2, M + 2), dtype=torch.float64)
    out = torch.empty(B, dtype=torch.float64)
    rc = lib().sdtw_cpu_forward_f64(_ptr(Dd), _ptr(R), _ptr(out), B, N, M, float(gamma), float(bandwidth))
    _check(rc, "cpu forward")
    return out, R


def cpu_backward(R: torch.Tensor, grad_out: torch.Tensor | None, gamma: float, bandwidth: float) -> torch.Tensor:
    Rd = R.detach().to(dtype=torch.float64).contiguous()
    B, N2, M2 = Rd.shape
    N, M = N2 - 2, M2 - 2
    E = torch.empty((B, N, M), dtype=torch.float64)
    g = None if grad_out is None else grad_out.detach().reshape(-1).to(dtype=torch.float64).contiguous()
    rc = lib().sdtw_cpu_backward_f64(_ptr(Rd), _ptr(g), _ptr(E), B, N, M, float(gamma), float(bandwidth))
    _check(rc, "cpu backward")
    return E


# ----------------------------------------------------------------------------- sequence operators
# Argument blocks of include/sdtw_b200.h, field for field: a ctypes Structure,
# and the same layout as a struct.Struct.  Calls use the latter: a single new
# time step is a call of a few microseconds, and filling a Structure field by
# field costs as much again.
_KINDS = {"i": ("i", ctypes.c_int), "l": ("q", ctypes.c_longlong), "f": ("f", ctypes.c_float),
          "p": ("P", ctypes.c_void_p), "z": ("N", ctypes.c_size_t)}


def _block(name: str, spec: str):
    fields = [(f, kind) for kind, names in (part.split(":") for part in spec.split()) for f in names.split(",")]
    cls = type(name, (ctypes.Structure,), {"_fields_": [(f, _KINDS[k][1]) for f, k in fields]})
    return cls, struct.Struct("@" + "".join(_KINDS[k][0] for _, k in fields)).pack


LayerNormArgs, _ln_pack = _block(
    "LayerNormArgs", "i:dtype,dim l:rows f:eps p:x l:x_stride p:weight,bias,y,mean,rstd,dy l:dy_stride "
                     "p:dx,dweight,dbias,workspace z:workspace_bytes")
ConvArgs, _conv_pack = _block(
    "ConvArgs", "i:dtype,batch,length,dim,width,silu p:x l:x_batch,x_time p:weight,bias,lengths,state_in "
                "l:state_in_batch p:state_out l:state_out_batch p:y,dy l:dy_batch,dy_time "
                "p:dstate_out,dx,dstate_in,dweight,dbias,workspace z:workspace_bytes")
ScanArgs, _scan_pack = _block(
    "ScanArgs", "i:dtype,batch,length,dim,groups,nstate,softplus p:x,delta,z "
                "l:x_batch,x_time,delta_batch,delta_time,z_batch,z_time p:B,C "
                "l:B_batch,B_time,B_group,C_batch,C_time,C_group p:A,D,delta_bias,lengths,state_in "
                "l:state_in_batch p:state_out l:state_out_batch p:saved,y,dy l:dy_batch,dy_time "
                "p:dstate_out,dx,ddelta,dz,dB,dC,dA,dD,ddelta_bias,dstate_in,workspace z:workspace_bytes")

_SERIES_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
_F32 = torch.float32


def _at(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def _last_contiguous(t: torch.Tensor) -> torch.Tensor:
    """t with its features side by side in memory (a copy only where they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """t (..., D) with one stride between its rows, and that stride."""
    if t.is_contiguous():
        return t, t.shape[-1]
    t = _last_contiguous(t)
    try:
        return t, t.view(-1, t.shape[-1]).stride(0)
    except RuntimeError:
        return t.contiguous(), t.shape[-1]


def _param(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None or (t.dtype is _F32 and t.is_contiguous()):
        return t
    return t.detach().to(_F32).contiguous()


def _call(fn, what: str, block: bytes, device: torch.device) -> None:
    ev = _op_begin(device)
    index = device.index
    if index == torch._C._cuda_getDevice():
        rc = fn(block, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            rc = fn(block, torch._C._cuda_getCurrentRawStream(index))
    if rc:
        _check(rc, what)
    _op_end(what, device, ev)


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    return torch.empty(nbytes, dtype=torch.uint8, device=like.device)


def _new(like: torch.Tensor, shape=None, dtype=None, when: bool = True) -> torch.Tensor | None:
    return torch.empty(like.shape if shape is None else shape, dtype=dtype or like.dtype, device=like.device) if when else None


def layer_norm_forward(x, weight, bias, eps: float, stats: bool = True):
    """(y, stats) of x (..., D); stats (2, rows) float32 holds each row's mean and 1 / deviation, or is None."""
    r, stride = _rows(x)
    dim = x.shape[-1]
    rows = x.numel() // dim
    y = _new(x)
    weight, bias = _param(weight), _param(bias)
    st, mean = None, 0
    if stats:
        st = _new(x, (2, rows), _F32)
        mean = st.data_ptr()
    _call(lib().sdtw_layer_norm_forward, "layer_norm",
          _ln_pack(_SERIES_DTYPES[x.dtype], dim, rows, eps, r.data_ptr(), stride, _at(weight), _at(bias), y.data_ptr(), mean,
                   mean + 4 * rows if stats else 0, 0, 0, 0, 0, 0, 0, 0), x.device)
    return y, st


def layer_norm_backward(x, weight, stats, dy, need_x=True, need_weight=True, need_bias=True):
    """(dx, dweight, dbias); dweight and dbias (D,) float32, None where not needed."""
    r, stride = _rows(x)
    g, gstride = _rows(dy)
    dim = x.shape[-1]
    rows = x.numel() // dim
    weight = _param(weight)
    dx, dw, db = _new(x, when=need_x), _new(x, (dim,), _F32, need_weight), _new(x, (dim,), _F32, need_bias)
    L = lib()
    nbytes = L.sdtw_layer_norm_workspace_bytes(rows, dim) if need_weight or need_bias else 0
    ws = _scratch(nbytes, x) if nbytes else None
    mean = stats.data_ptr()
    _call(L.sdtw_layer_norm_backward, "layer_norm gradient",
          _ln_pack(_SERIES_DTYPES[x.dtype], dim, rows, 0.0, r.data_ptr(), stride, _at(weight), 0, 0, mean, mean + 4 * rows,
                   g.data_ptr(), gstride, _at(dx), _at(dw), _at(db), _at(ws), nbytes), x.device)
    return dx, dw, db


def conv_forward(x, weight, bias, silu: bool, lengths, state_in, want_state: bool):
    """(y, state_out) of x (B, N, D), weight (D, W); state_out (B, W - 1, D) or None."""
    x, weight, bias = _last_contiguous(x), _param(weight), _param(bias)
    batch, length, dim = x.shape
    width = weight.shape[1]
    state_in = None if state_in is None else state_in.contiguous()
    state = _new(x, (batch, width - 1, dim), when=want_state)
    y = _new(x)
    per = (width - 1) * dim
    _call(lib().sdtw_conv_forward, "causal_conv",
          _conv_pack(_SERIES_DTYPES[x.dtype], batch, length, dim, width, silu, x.data_ptr(), x.stride(0), x.stride(1),
                     weight.data_ptr(), _at(bias), _at(lengths), _at(state_in), per, _at(state), per, y.data_ptr(),
                     0, 0, 0, 0, 0, 0, 0, 0, 0, 0), x.device)
    return y, state


def conv_backward(x, weight, bias, silu: bool, lengths, state_in, dy, dstate, need_x=True, need_weight=True,
                  need_bias=True, need_state=False):
    """(dx, dweight, dbias, dstate_in), None where not needed."""
    x, weight, bias, dy = _last_contiguous(x), _param(weight), _param(bias), _last_contiguous(dy)
    batch, length, dim = x.shape
    width = weight.shape[1]
    state_in = None if state_in is None else state_in.contiguous()
    dstate = None if dstate is None else dstate.contiguous()
    dx, dw, db = _new(x, when=need_x), _new(x, (dim, width), _F32, need_weight), _new(x, (dim,), _F32, need_bias)
    ds = _new(x, (batch, width - 1, dim), when=need_state)
    L = lib()
    nbytes = L.sdtw_conv_workspace_bytes(batch, length, dim, width) if need_weight or need_bias else 0
    ws = _scratch(nbytes, x) if nbytes else None
    per = (width - 1) * dim
    _call(L.sdtw_conv_backward, "causal_conv gradient",
          _conv_pack(_SERIES_DTYPES[x.dtype], batch, length, dim, width, silu, x.data_ptr(), x.stride(0), x.stride(1),
                     weight.data_ptr(), _at(bias), _at(lengths), _at(state_in), per, 0, 0, 0,
                     dy.data_ptr(), dy.stride(0), dy.stride(1), _at(dstate), _at(dx), _at(ds), _at(dw), _at(db), _at(ws),
                     nbytes), x.device)
    return dx, dw, db, ds


def conv_step(x, weight, bias, silu: bool, state_in, state_out):
    """y (B, D) for x (B, D); state_out <- the window moved up by x (may be state_in)."""
    x, weight, bias = _last_contiguous(x), _param(weight), _param(bias)
    y = _new(x)
    batch, dim = x.shape
    _call(lib().sdtw_conv_step, "causal_conv step",
          _conv_pack(_SERIES_DTYPES[x.dtype], batch, 1, dim, weight.shape[1], silu, x.data_ptr(), x.stride(0), 0,
                     weight.data_ptr(), _at(bias), 0, state_in.data_ptr(), state_in.stride(0), state_out.data_ptr(),
                     state_out.stride(0), y.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0), x.device)
    return y


def scan_saved_elems(batch: int, length: int, dim: int, nstate: int) -> int:
    return int(lib().sdtw_scan_saved_elems(batch, length, dim, nstate))


def _scan_block(x, delta, A, B, C, D, z, bias, softplus, lengths, state_in, state_out, tail) -> bytes:
    """x, delta, z (Bt, N, D) or, for a step, (Bt, D); B, C (Bt, N, G, S) or (Bt, G, S).  `tail`: from `saved` on."""
    step = x.dim() == 2
    dim, S = A.shape
    # Strides of the batch, the time and the groups (no time for a step).
    xb, db, zb = x.stride(0), delta.stride(0), 0 if z is None else z.stride(0)
    xt, dt, zt = (0, 0, 0) if step else (x.stride(1), delta.stride(1), 0 if z is None else z.stride(1))
    Bs, Cs = B.stride(), C.stride()
    Bt, Ct = (0, 0) if step else (Bs[1], Cs[1])
    return _scan_pack(_SERIES_DTYPES[x.dtype], x.shape[0], 1 if step else x.shape[1], dim, B.shape[-2], S, softplus,
                      x.data_ptr(), delta.data_ptr(), _at(z), xb, xt, db, dt, zb, zt, B.data_ptr(), C.data_ptr(),
                      Bs[0], Bt, Bs[-2], Cs[0], Ct, Cs[-2], A.data_ptr(), _at(D), _at(bias), _at(lengths), _at(state_in),
                      0 if state_in is None else state_in.stride(0), _at(state_out),
                      0 if state_out is None else state_out.stride(0), *tail)


def _scan_inputs(x, delta, A, B, C, D, z, bias):
    return (_last_contiguous(x), _last_contiguous(delta), _param(A), _last_contiguous(B), _last_contiguous(C), _param(D),
            None if z is None else _last_contiguous(z), _param(bias))


def scan_forward(x, delta, A, B, C, D, z, bias, softplus: bool, lengths, state_in, want_state: bool, save: bool):
    """(y, state_out, saved) of x, delta, z (Bt, N, D), A (D, S), B, C (Bt, N, G, S)."""
    ins = _scan_inputs(x, delta, A, B, C, D, z, bias)
    batch, length, dim = x.shape
    G, S = B.shape[2], A.shape[1]
    L = lib()
    state_in = _param(state_in)
    state = _new(x, (batch, dim, S), _F32, want_state)
    y = _new(x)
    saved = _new(x, (L.sdtw_scan_saved_elems(batch, length, dim, S),), _F32) if save else None
    nbytes = L.sdtw_scan_forward_workspace_bytes(batch, length, dim, G, S)
    ws = _scratch(nbytes, x) if nbytes else None
    tail = (_at(saved), y.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, _at(ws), nbytes)
    _call(L.sdtw_scan_forward, "selective_scan", _scan_block(*ins, softplus, lengths, state_in, state, tail), x.device)
    return y, state, saved


def scan_backward(x, delta, A, B, C, D, z, bias, softplus: bool, lengths, saved, dy, dstate, need):
    """Gradients of (x, delta, A, B, C, D, z, delta_bias, initial_state), None where ``need`` is false."""
    ins = _scan_inputs(x, delta, A, B, C, D, z, bias)
    dy, dstate = _last_contiguous(dy), _param(dstate)
    batch, length, dim = x.shape
    G, S = B.shape[2], A.shape[1]
    series, groups = x.shape, (batch, length, G, S)
    dx, ddelta, dz = _new(x, series, None, need[0]), _new(x, series, None, need[1]), _new(x, series, None, need[6])
    dB, dC = _new(x, groups, None, need[3]), _new(x, groups, None, need[4])
    dA, dD, db = _new(x, (dim, S), _F32, need[2]), _new(x, (dim,), _F32, need[5]), _new(x, (dim,), _F32, need[7])
    dh = _new(x, (batch, dim, S), _F32, need[8])
    L = lib()
    nbytes = L.sdtw_scan_workspace_bytes(batch, length, dim, G, S)
    ws = _scratch(nbytes, x)
    tail = (saved.data_ptr(), 0, dy.data_ptr(), dy.stride(0), dy.stride(1), _at(dstate), _at(dx), _at(ddelta), _at(dz), _at(dB),
            _at(dC), _at(dA), _at(dD), _at(db), _at(dh), ws.data_ptr(), nbytes)
    _call(L.sdtw_scan_backward, "selective_scan gradient", _scan_block(*ins, softplus, lengths, None, None, tail), x.device)
    return [dx, ddelta, dA, dB, dC, dD, dz, db, dh]


def scan_step(x, delta, A, B, C, D, z, bias, softplus: bool, state_in, state_out):
    """y (Bt, D) for x, delta, z (Bt, D), B, C (Bt, G, S); state_out <- the next state (may be state_in)."""
    ins = _scan_inputs(x, delta, A, B, C, D, z, bias)
    y = _new(x)
    tail = (0, y.data_ptr(), 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0)
    _call(lib().sdtw_scan_step, "selective_scan step", _scan_block(*ins, softplus, None, state_in, state_out, tail), x.device)
    return y

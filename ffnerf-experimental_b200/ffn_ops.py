"""The block operators of libffnerf.so on torch CUDA tensors: RMS norm with the residual's addition,
gated linear recurrence, matrix products grouped by expert -- each with its backward pass.

They are what a residual block over per-sample features needs next to the fused training step: the
norm of the residual stream (with an e4m3 output for the experts' 8-bit product), a recurrence that
mixes the samples of a ray in depth order (with a sigmoid gate it composites feature vectors), and
the products of samples with the sub-network of their region.  Every call is ordered on the current
stream (or ``stream``), launches CUDA kernels only and does not synchronise; gradients are explicit
functions.  Arguments that an operator cannot take raise ValueError; there is no fallback.  As with
torch's own operators, work that produced the inputs on another stream has to be ordered before the
call by the caller.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

import ffn_native as fn

F32, F16, BF16, E4M3 = range(4)                       # include/ffnerf.h FFN_F32 ...
SCAN_FORMS = {"linear": 0, "sigmoid": 1}
DTYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16, torch.float8_e4m3fn: E4M3}
_WIDE = (torch.float32, torch.float16, torch.bfloat16)

# What torch.cuda.current_stream().cuda_stream and torch.cuda.current_device() return, without building a
# Stream object: a call on a single row is bound by the host, about 10 us of it.
_raw_stream = torch._C._cuda_getCurrentRawStream
_device_now = torch._C._cuda_getDevice


def _bad(what: str):
    raise ValueError(what)


def _rows(t, name: str, d: int, n: int, dtype, device) -> int:
    """Checks a matrix [n, d] of contiguous columns and returns its row stride in elements."""
    if t.dtype is not dtype:
        _bad(f"{name} is {t.dtype}, expected {dtype}")
    if t.device != device:
        _bad(f"{name} is on {t.device}, expected {device}")
    if t.shape != (n, d):
        _bad(f"{name} has shape {tuple(t.shape)}, expected {(n, d)}")
    if t.is_contiguous():
        return d
    ld, sc = t.stride()
    if d > 1 and sc != 1:
        _bad(f"{name} must have contiguous columns")
    if n <= 1:
        return d
    if ld < d:
        _bad(f"{name} must not overlap itself (row stride {ld} below {d} columns)")
    return ld


def _matrix(t, name: str):
    """(rows, columns, device) of the CUDA matrix that sets a call's shape."""
    if not t.is_cuda:
        _bad(f"{name} must be a CUDA tensor")
    if t.dim() != 2:
        _bad(f"{name} must be a matrix [rows, columns], got shape {tuple(t.shape)}")
    return *t.shape, t.device


def _like(t):
    """An uninitialised contiguous tensor of t's shape and type."""
    return torch.empty_like(t) if t.is_contiguous() else torch.empty(t.shape, dtype=t.dtype, device=t.device)


def _plain(t, name: str, shape: tuple, dtype, device):
    """Checks a contiguous tensor of exactly this shape and type; None passes."""
    if t is None:
        return None
    if t.shape != shape or t.dtype is not dtype or t.device != device or not t.is_contiguous():
        _bad(f"{name} must be a contiguous {dtype} tensor of shape {shape} on {device}, got {t.dtype} "
             f"{tuple(t.shape)} on {t.device}")
    return t.data_ptr()


def _call(name: str, device, *args):
    """One native call on `device` and its current stream."""
    f = getattr(fn._lib or fn.load_library(), name)
    i = device.index
    if _device_now() == i:
        rc = f(*args, _raw_stream(i))
    else:
        with torch.cuda.device(device):
            rc = f(*args, _raw_stream(i))
    if rc != fn.FFN_OK:
        msg = fn.load_library().ffn_last_error(None).decode()
        raise (ValueError if rc in (fn.FFN_E_CONFIG, fn.FFN_E_CAPACITY) else RuntimeError)(f"{name} failed ({rc}): {msg}")


def _on(stream, f, *args):
    """f(*args) with `stream` current: outputs and workspaces are then allocated on that stream too, so
    the caching allocator cannot hand their memory to other work early."""
    if not isinstance(stream, torch.cuda.Stream):
        stream = torch.cuda.ExternalStream(int(stream))
    with torch.cuda.stream(stream):
        return f(*args)


def _workspace(device, name: str, *args):
    """(tensor or None, pointer, bytes) of the workspace that the library asks for."""
    f = getattr(fn._lib or fn.load_library(), name)
    if _device_now() == device.index:
        need = f(*args)
    else:
        with torch.cuda.device(device):
            need = f(*args)
    if not need:
        return None, None, 0
    t = torch.empty(need, dtype=torch.uint8, device=device)
    return t, t.data_ptr(), need


# ---------------------------------------------------------------------------------------- RMS norm
class NormState(NamedTuple):
    """What the backward pass of ``rmsnorm`` needs: the row factors (float32 [n]) and the inputs."""
    rstd: torch.Tensor
    x: torch.Tensor
    residual: torch.Tensor | None


def rmsnorm(x, gamma, residual=None, eps: float = 1e-6, out: str = "same", group: int = 0, stream=None):
    """RMS norm of ``x + residual`` over the columns: returns ``(y, h, state, scale)``.

    x, residual [n, d] (float32, float16 or bfloat16; rows may be strided), gamma [d] float32.  y is in
    x's type, or (``out="e4m3"``) float8_e4m3fn with float32 ``scale`` [n], or [n, d / group] for
    ``group`` 32, 64 or 128; value = y * scale (scale is None for ``out="same"``).  h is the sum in x's
    type, the residual stream that goes on (x itself without a residual); state is what
    ``rmsnorm_bwd`` takes."""
    if stream is not None:
        return _on(stream, rmsnorm, x, gamma, residual, eps, out, group)
    dt = x.dtype
    if dt not in _WIDE:
        _bad(f"x must be float32, float16 or bfloat16, got {dt}")
    n, d, dev = _matrix(x, "x")
    x_ld = _rows(x, "x", d, n, dt, dev)
    code = DTYPES[dt]
    g = _plain(gamma, "gamma", (d,), torch.float32, dev)
    if out == "same":
        if group:
            _bad("group needs out='e4m3'")
        y, scale, sp, out_code = _like(x), None, None, code
    elif out == "e4m3":
        if group not in (0, 32, 64, 128) or (group and d % group):
            _bad(f"group must be 0, 32, 64 or 128 and divide the {d} columns, got {group}")
        y, out_code = torch.empty((n, d), dtype=torch.float8_e4m3fn, device=dev), E4M3
        scale = gamma.new_empty((n, d // group) if group else (n,))
        sp = scale.data_ptr()
    else:
        _bad(f"out must be 'same' or 'e4m3', got {out!r}")
    rstd = gamma.new_empty((n,))
    if residual is None:
        h, hp, rp, res_ld = x, None, None, 0
    else:
        res_ld = _rows(residual, "residual", d, n, dt, dev)
        h = _like(x)
        hp, rp = h.data_ptr(), residual.data_ptr()
    _call("ffn_rmsnorm", dev, x.data_ptr(), x_ld, rp, res_ld, g, hp, y.data_ptr(), sp, rstd.data_ptr(), n, d, eps, code,
          out_code, group)
    return y, h, NormState(rstd, x, residual), scale


def rmsnorm_bwd(dy, h, gamma, state, dresidual=None, stream=None):
    """Backward pass of ``rmsnorm``: returns ``(dx, dgamma)``.  dx (the gradient of x and of the residual
    alike) includes ``dresidual``, the gradient that reaches h past the norm.

    state is the NormState of the forward call; the sum is then formed again from its inputs, unrounded,
    and h is not read.  A caller who kept only h and the row factors passes the float32 [n] tensor
    ``state.rstd`` instead: xhat then carries the rounding of h, one array less is read, and x and the
    residual need not be kept."""
    if stream is not None:
        return _on(stream, rmsnorm_bwd, dy, h, gamma, state, dresidual)
    dt = dy.dtype
    if dt not in _WIDE:
        _bad(f"dy must be float32, float16 or bfloat16, got {dt}")
    n, d, dev = _matrix(dy, "dy")
    dy_ld = _rows(dy, "dy", d, n, dt, dev)
    rstd, x, residual = state if isinstance(state, NormState) else (state, h, None)
    x_ld = _rows(x, "x", d, n, dt, dev)
    res_ld = 0 if residual is None else _rows(residual, "residual", d, n, dt, dev)
    dr_ld = 0 if dresidual is None else _rows(dresidual, "dresidual", d, n, dt, dev)
    g, r = _plain(gamma, "gamma", (d,), torch.float32, dev), _plain(rstd, "rstd", (n,), torch.float32, dev)
    dx, dgamma = _like(dy), _like(gamma)
    ws, p, size = _workspace(dev, "ffn_rmsnorm_bwd_workspace", n, d)
    _call("ffn_rmsnorm_bwd", dev, dy.data_ptr(), dy_ld, x.data_ptr(), x_ld,
          None if residual is None else residual.data_ptr(), res_ld, g, r,
          None if dresidual is None else dresidual.data_ptr(), dr_ld, dx.data_ptr(), dgamma.data_ptr(), p, size, n, d,
          DTYPES[dt])
    return dx, dgamma


# -------------------------------------------------------------------------- gated linear recurrence
def _scan_layout(gate, value, offsets, max_len, form, h0):
    """The packed [rows, d] view of a scan's arguments and its sequences."""
    if form not in SCAN_FORMS:
        _bad(f"form must be one of {sorted(SCAN_FORMS)}, got {form!r}")
    if gate.dtype not in _WIDE:
        _bad(f"gate must be float32, float16 or bfloat16, got {gate.dtype}")
    dev = gate.device
    if offsets is None:
        if gate.dim() != 3:
            _bad("without offsets gate must be [sequences, steps, channels]")
        seqs, max_len, d = gate.shape
        off = None
    else:
        if offsets.dim() != 1 or offsets.dtype is not torch.int32 or offsets.device != dev or offsets.numel() < 1 \
                or not offsets.is_contiguous():
            _bad(f"offsets must be a contiguous int32 vector [sequences + 1] on {dev}")
        if gate.dim() != 2:
            _bad("with offsets gate must be [rows, channels]")
        seqs, d = offsets.numel() - 1, gate.shape[1]
        max_len = gate.shape[0] if max_len is None else int(max_len)
        off = offsets.data_ptr()
    return seqs, max_len, d, off, _plain(h0, "h0", (seqs, d), torch.float32, dev)


def _packed(t, name: str, like, d: int):
    """(pointer, row stride) of a [rows, d] or [sequences, steps, d] tensor."""
    if t.shape != like.shape:
        _bad(f"{name} has shape {tuple(t.shape)}, expected {tuple(like.shape)}")
    if t.dtype is not like.dtype or t.device != like.device or not t.is_cuda:
        _bad(f"{name} must be a {like.dtype} CUDA tensor on {like.device}, got {t.dtype} on {t.device}")
    if t.is_contiguous():
        return t.data_ptr(), d
    if t.dim() == 3:
        b, s, _ = t.shape
        if s > 1 and b > 1 and t.stride(0) != s * t.stride(1):
            _bad(f"{name}: the sequences must follow one another at a constant row stride")
        t = t.as_strided((b * s, d), (t.stride(1) if s > 1 else t.stride(0), t.stride(2)))
    return t.data_ptr(), _rows(t, name, d, t.shape[0], like.dtype, like.device)


def gated_scan(gate, value, h0=None, offsets=None, max_len: int | None = None, form: str = "sigmoid",
               reverse: bool = False, stream=None):
    """The recurrence ``h_t = a_t h_{t-1} + b_t`` per channel: returns ``(h, h_last)``.

    form "sigmoid": a = sigmoid(gate), b = (1 - a) value; "linear": a = gate (magnitude at most about
    1), b = value.  gate and value (float32, float16 or bfloat16) are [sequences, steps, channels], or
    packed [rows, channels] with int32 ``offsets`` [sequences + 1] on the device (sequences may be
    empty; rows of no sequence give zeros).  ``max_len`` says how long a packed sequence is expected to
    get (it chooses the split of the work and bounds nothing).  h0 [sequences, channels] float32 is the
    state before the first step (None: zero); h_last, float32, the state after the last.  ``reverse``
    runs every sequence from its last step to its first (back-to-front compositing)."""
    if stream is not None:
        return _on(stream, gated_scan, gate, value, h0, offsets, max_len, form, reverse)
    seqs, max_len, d, off, p0 = _scan_layout(gate, value, offsets, max_len, form, h0)
    gp, g_ld = _packed(gate, "gate", gate, d)
    vp, v_ld = _packed(value, "value", gate, d)
    h = _like(gate)
    last = torch.empty((seqs, d), dtype=torch.float32, device=gate.device) if h0 is None else torch.empty_like(h0)
    rows = seqs * max_len if off is None else gate.shape[0]
    if seqs == 0:
        return h.zero_(), last
    buf, p, size = _workspace(gate.device, "ffn_gated_scan_workspace", seqs, max_len, d)
    _call("ffn_gated_scan", gate.device, gp, g_ld, vp, v_ld, p0, off, h.data_ptr(), last.data_ptr(), rows, seqs,
          max_len, d, DTYPES[gate.dtype], SCAN_FORMS[form], 1 if reverse else 0, p, size)
    return h, last


def gated_scan_bwd(dh, gate, value, h, h0=None, dh_last=None, offsets=None, max_len: int | None = None,
                   form: str = "sigmoid", reverse: bool = False, stream=None):
    """Backward pass of ``gated_scan`` from its inputs and its h: returns ``(dgate, dvalue, dh0)``.
    dh_last [sequences, channels] float32 is the gradient of h_last (None: zero); dh0 is float32."""
    if stream is not None:
        return _on(stream, gated_scan_bwd, dh, gate, value, h, h0, dh_last, offsets, max_len, form, reverse)
    seqs, max_len, d, off, p0 = _scan_layout(gate, value, offsets, max_len, form, h0)
    dev = gate.device
    gp, g_ld = _packed(gate, "gate", gate, d)
    vp, v_ld = _packed(value, "value", gate, d)
    dp, d_ld = _packed(dh, "dh", gate, d)
    hp, h_ld = _packed(h, "h", gate, d)
    pl = _plain(dh_last, "dh_last", (seqs, d), torch.float32, dev)
    dgate, dvalue = _like(gate), _like(gate)
    dh0 = torch.empty((seqs, d), dtype=torch.float32, device=dev)
    rows = seqs * max_len if off is None else gate.shape[0]
    if seqs == 0:
        return dgate.zero_(), dvalue.zero_(), dh0
    buf, p, size = _workspace(dev, "ffn_gated_scan_workspace", seqs, max_len, d)
    _call("ffn_gated_scan_bwd", dev, dp, d_ld, pl, gp, g_ld, vp, v_ld, hp, h_ld, p0, off, dgate.data_ptr(),
          dvalue.data_ptr(), dh0.data_ptr(), rows, seqs, max_len, d, DTYPES[gate.dtype], SCAN_FORMS[form],
          1 if reverse else 0, p, size)
    return dgate, dvalue, dh0


# ------------------------------------------------------------------- matrix products by expert
def _experts(x, w, offsets):
    if w.dim() != 3 or not w.is_contiguous():
        _bad(f"w must be a contiguous tensor [experts, out, in], got shape {tuple(w.shape)}")
    e, m, k = w.shape
    if e < 1 or m < 1 or k < 1:
        _bad(f"w must have at least one expert, output and input, got shape {tuple(w.shape)}")
    dev = x.device
    if w.dtype is not x.dtype or w.device != dev:
        _bad(f"w is {w.dtype} on {w.device}, expected {x.dtype} on {dev}")
    return e, m, k, _plain(offsets, "offsets", (e + 1,), torch.int32, dev)


def expert_mm(x, w, offsets, x_scale=None, w_scale=None, out_dtype=None, stream=None):
    """``y[r] = x[r] w[e]^T`` for the rows r of expert e: returns y [n, out].

    x [n, in] holds the rows sorted by expert (rows may be strided), offsets [experts + 1] int32 on the
    device where each expert's rows begin (offsets[0] = 0; experts may have none; rows from
    offsets[experts] on give zeros), w [experts, out, in].  x and w are both float16 or both bfloat16
    (y the same), or both float8_e4m3fn with float32 ``x_scale`` [n] and ``w_scale`` [experts, out]
    (y bfloat16, or float16 by ``out_dtype``).  Sums are float32."""
    if stream is not None:
        return _on(stream, expert_mm, x, w, offsets, x_scale, w_scale, out_dtype)
    n, _, dev = _matrix(x, "x")
    e, m, k, off = _experts(x, w, offsets)
    x_ld = _rows(x, "x", k, n, x.dtype, dev)
    xs = ws_ = None
    if x.dtype is torch.float8_e4m3fn:
        out_dtype = out_dtype or torch.bfloat16
        if x_scale is None or w_scale is None:
            _bad("float8_e4m3fn rows need x_scale [n] and w_scale [experts, out]")
        xs = _plain(x_scale, "x_scale", (n,), torch.float32, dev)
        ws_ = _plain(w_scale, "w_scale", (e, m), torch.float32, dev)
        if out_dtype not in (torch.float16, torch.bfloat16):
            _bad(f"out_dtype must be float16 or bfloat16, got {out_dtype}")
    elif x.dtype in (torch.float16, torch.bfloat16):
        if x_scale is not None or w_scale is not None:
            _bad("scales belong to float8_e4m3fn operands")
        if out_dtype not in (None, x.dtype):
            _bad(f"out_dtype must be {x.dtype} for {x.dtype} operands")
        out_dtype = x.dtype
    else:
        _bad(f"x must be float16, bfloat16 or float8_e4m3fn, got {x.dtype}")
    y = torch.empty((n, m), dtype=out_dtype, device=dev)
    code = DTYPES[x.dtype]
    xp, wp, unit = x.data_ptr(), w.data_ptr(), 16 if code == E4M3 else 8
    buf = p = None
    size = 0
    if (xp | wp) & 15 or x_ld % unit or k % unit:             # rows that TMA cannot read are copied
        buf, p, size = _workspace(dev, "ffn_expert_mm_workspace", xp, x_ld, wp, n, e, k, m, code)
    _call("ffn_expert_mm", dev, xp, x_ld, wp, off, xs, ws_, y.data_ptr(), n, e, k, m, code,
          DTYPES[out_dtype], p, size)
    return y


def expert_mm_bwd(dy, x, w, offsets, need_dx: bool = True, need_dw: bool = True, dw_dtype=None, stream=None):
    """Gradients of ``expert_mm`` for float16 or bfloat16 operands: returns ``(dx, dw)``, each None when
    not needed.  dx [n, in] is in x's type; dw [experts, out, in] in x's type or, by ``dw_dtype``,
    float32 (what ``ffn_native.adam`` takes).  An expert without rows gets a zero gradient."""
    if stream is not None:
        return _on(stream, expert_mm_bwd, dy, x, w, offsets, need_dx, need_dw, dw_dtype)
    if x.dtype not in (torch.float16, torch.bfloat16):
        _bad(f"x must be float16 or bfloat16, got {x.dtype}")
    n, _, dev = _matrix(x, "x")
    e, m, k, off = _experts(x, w, offsets)
    x_ld = _rows(x, "x", k, n, x.dtype, dev)
    dy_ld = _rows(dy, "dy", m, n, x.dtype, dev)
    dw_dtype = dw_dtype or x.dtype
    if dw_dtype not in (x.dtype, torch.float32):
        _bad(f"dw_dtype must be {x.dtype} or float32, got {dw_dtype}")
    dx = torch.empty((n, k), dtype=x.dtype, device=dev) if need_dx else None
    dw = torch.empty((e, m, k), dtype=dw_dtype, device=dev) if need_dw else None
    code = DTYPES[x.dtype]
    buf, p, size = _workspace(dev, "ffn_expert_mm_bwd_workspace", dy.data_ptr(), dy_ld, x.data_ptr(), x_ld, w.data_ptr(),
                              n, e, k, m, code)
    _call("ffn_expert_mm_bwd", dev, dy.data_ptr(), dy_ld, x.data_ptr(), x_ld, w.data_ptr(), off,
          None if dx is None else dx.data_ptr(), None if dw is None else dw.data_ptr(), n, e, k, m, code,
          DTYPES[dw_dtype], p, size)
    return dx, dw


def status(device=None) -> int:
    """Status word of the block operators on the current (or given) device since the last call; waits for
    the device.  0 when every kernel completed normally; ``ffn_native.STATUS_TC_TIMEOUT`` when a wait of
    an expert product ran out and its results are incomplete."""
    import ctypes
    v = ctypes.c_uint32()
    with torch.cuda.device(device):
        rc = fn.load_library().ffn_ops_status(ctypes.byref(v))
    if rc != fn.FFN_OK:
        raise RuntimeError(f"ffn_ops_status failed ({rc}): {fn.load_library().ffn_last_error(None).decode()}")
    return int(v.value)

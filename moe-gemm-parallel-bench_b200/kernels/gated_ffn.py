"""The gated feed-forward block over expert-sorted rows, forward and backward.

    y = h W2,   h = silu(x Wg) * (x Wu),   W13 = [Wg | Wu]

``launch_grouped_mm(..., swiglu=True)`` computes h for inference and keeps
nothing.  Training needs the block's gradients: the forward pass here also
writes the pre-activations ``gate_up`` = x W13 (from the same kernel that
writes h), and the backward pass returns the gradients of x, W13 and W2:

    dh = dy W2^T,   dgate = dh u s (1 + g (1 - s)),   dup = dh g s,   s = sigmoid(g)
    dx = [dgate | dup] W13^T,   dW13 = x^T [dgate | dup],   dW2 = h^T dy

Rows are sorted by expert, ``offs`` (int32 ``[E]``, on the device) holding the
cumulative row ends, as in ``launch_grouped_mm``; ``offs=None`` is the dense
block (one expert, every row).  Empty experts are fine (their weight gradients
are zeros); rows past ``offs[-1]`` have no effect and are not written.  The single
products' gradients are there as well: ``launch_grouped_mm_dgrad`` and
``launch_grouped_mm_wgrad``.

fp16 or bf16; hidden and ffn sizes are multiples of 8, bases 16-byte aligned,
columns contiguous; rows may be padded to a pitch that is a multiple of 8,
experts to a whole number of rows.
Accumulation is fp32; ``gate_up``, ``h`` and the gradient of ``gate_up`` are
rounded once to the operands' type between products, weight gradients are
overwritten and of the weights' type.  Inputs and outputs must
not overlap.  Every call is launches only (no synchronisation), on the current
stream of the tensors' device, with its scratch allocated on that stream, so it
can be captured in a CUDA graph.  The calls are explicit: autograd does not see
them, and their outputs carry no history even where an input requires a
gradient.  The reference has no counterpart (SiLU(gate) * up and all gradients stay
outside its timed path, README.md:55-60).
"""

from __future__ import annotations

try:
    import torch
except ImportError:  # pragma: no cover - the CPU tests import the host helpers only
    torch = None

from . import _native
from .matmul import dtype_name


_ready = False


def _require_runtime() -> None:
    global _ready
    if not _ready:
        if torch is None or not torch.cuda.is_available():
            raise RuntimeError("CUDA PyTorch and the native sm_100a library are required")
        _native.load()
        _ready = True


def _call(device, entry, *args):
    """entry(*args, stream) with ``device`` current and its current stream.
    These calls can be as short as their host side (a few microseconds on the
    device), so the guard is taken only where it changes something and the
    stream handle is read without building a Stream object."""
    index = device.index
    if torch._C._cuda_getDevice() == index:  # the tensors' device exists: CUDA is initialised
        return entry(*args, torch._C._cuda_getCurrentRawStream(index))
    with torch.cuda.device(index):
        return entry(*args, torch._C._cuda_getCurrentRawStream(index))


def _rows_of(like, rows: int, cols: int):
    """An empty [rows, cols] tensor of ``like``'s type and device."""
    return torch.empty_strided((rows, cols), (cols, 1), dtype=like.dtype, device=like.device)


def _scratch(like, nbytes: int):
    """(scratch, bytes) of a call on ``like``'s device; None where it needs none."""
    return (like.new_empty(nbytes // 2) if nbytes else None), nbytes


def _token(name: str, t, rows: int, cols: int, dtype, device) -> tuple[int, int]:
    """(address, pitch) of a [rows, cols] tensor of the call's type and device."""
    if t.shape != (rows, cols):
        raise ValueError(f"{name} must be [{rows}, {cols}], got {tuple(t.shape)}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    pitch, step = t.stride()
    if rows <= 1:
        pitch = cols
    address = t.data_ptr()
    if step != 1 or pitch < cols or pitch % 8 or address % 16:
        raise ValueError(f"{name} needs contiguous columns, a 16-byte aligned base and a row pitch that is a multiple of 8")
    return address, pitch


def _weight(name: str, t, experts: int, rows: int, cols: int, dtype, device) -> tuple[int, int, int]:
    """(address, pitch, expert stride) of an [experts, rows, cols] weight (or [rows, cols] for one expert)."""
    shape = t.shape
    if shape != (experts, rows, cols) and not (experts == 1 and shape == (rows, cols)):
        raise ValueError(f"{name} must be [{experts}, {rows}, {cols}], got {tuple(shape)}")
    if t.dtype != dtype or t.device != device:
        raise ValueError(f"{name} must be {dtype} on {device}, got {t.dtype} on {t.device}")
    strides = t.stride()
    pitch = strides[-2]
    stride = strides[0] if experts > 1 else rows * pitch
    address = t.data_ptr()
    if strides[-1] != 1 or pitch < cols or pitch % 8 or address % 16 or stride % pitch or stride < rows * pitch:
        raise ValueError(f"{name} needs contiguous columns, a 16-byte aligned base, a row pitch that is a multiple of 8 "
                         "and experts a whole number of rows apart")
    return address, pitch, stride


def _operand_type(name: str, t) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    code = _native.DTYPE_CODES[dtype_name(t.dtype)]
    if t.dtype == torch.float32:
        raise ValueError(f"{name} must be float16 or bfloat16")
    return code


def _offsets(offs, experts: int, device) -> int:
    """Address of the row ends (0: one segment of every row)."""
    if offs is None:
        if experts != 1:
            raise ValueError("offs (int32 cumulative row ends) is needed with more than one expert")
        return 0
    if offs.shape != (experts,) or offs.dtype != torch.int32 or not offs.is_contiguous():
        raise ValueError(f"offs must be contiguous int32 [{experts}] cumulative row ends")
    if offs.device != device:
        raise ValueError("offs must be on the tensors' device")
    return offs.data_ptr()


def _sizes(hidden: int, ffn: int) -> None:
    if hidden <= 0 or ffn <= 0 or hidden % 8 or ffn % 8:
        raise ValueError(f"matrix sizes must be positive multiples of 8, got {hidden} and {ffn}")


def _block_shape(x, w13, w2) -> tuple[int, int, int, int]:
    if x.ndim != 2 or w13.ndim not in (2, 3) or w2.ndim != w13.ndim:
        raise ValueError("expected x [T, H], w13 [E, H, 2F] and w2 [E, F, H] (or [H, 2F] and [F, H])")
    ffn, hidden = w2.shape[-2:]
    _sizes(hidden, ffn)
    return x.shape[0], (w13.shape[0] if w13.ndim == 3 else 1), hidden, ffn


def last_gated_ffn_info() -> list[dict]:
    """The product launches of the calling thread's most recent call of this
    module, in order: epilogue, pair, output tile, split of the contraction, grid."""
    return [info.as_dict() for info in _native.ffn_last_launches()]


def gated_ffn_forward(x, w13, w2, offs=None, *, out=None, h=None, gate_up=None):
    """(y, h, gate_up) of the block: ``x [T, H]``, ``w13 [E, H, 2F]`` packed
    [gate | up], ``w2 [E, F, H]``; ``[H, 2F]`` and ``[F, H]`` for one expert.
    ``y [T, H]`` is the output; ``h [T, F]`` and ``gate_up [T, 2F]`` are what
    ``gated_ffn_backward`` reads.  Tensors given for the three outputs are
    written in place."""
    _require_runtime()
    rows, experts, hidden, ffn = _block_shape(x, w13, w2)
    code = _operand_type("x", x)
    dtype, device = x.dtype, x.device
    args = _native.FfnArgs(code, experts, rows, hidden, ffn, _offsets(offs, experts, device))
    args.x, args.x_pitch = _token("x", x, rows, hidden, dtype, device)
    args.w13, args.w13_pitch, args.w13_stride = _weight("w13", w13, experts, hidden, 2 * ffn, dtype, device)
    args.w2, args.w2_pitch, args.w2_stride = _weight("w2", w2, experts, ffn, hidden, dtype, device)
    if out is None:
        out = _rows_of(x, rows, hidden)
    if h is None:
        h = _rows_of(x, rows, ffn)
    if gate_up is None:
        gate_up = _rows_of(x, rows, 2 * ffn)
    args.y, args.y_pitch = _token("out", out, rows, hidden, dtype, device)
    args.h, args.h_pitch = _token("h", h, rows, ffn, dtype, device)
    args.gate_up, args.gate_up_pitch = _token("gate_up", gate_up, rows, 2 * ffn, dtype, device)
    scratch, nbytes = _scratch(x, _native.ffn_scratch_bytes(experts, _native.FFN_FORWARD))
    _call(device, _native.gated_ffn_forward, args, scratch.data_ptr() if nbytes else 0, nbytes)
    return out, h, gate_up


def gated_ffn_backward(dy, x, w13, w2, h, gate_up, offs=None, *, dx=None, dw13=None, dw2=None):
    """(dx, dw13, dw2) from the output's gradient ``dy [T, H]``, the block's
    inputs and the ``h`` and ``gate_up`` that ``gated_ffn_forward`` returned.
    Gradients have their tensor's shape and type; tensors given for them are
    overwritten (nothing is accumulated)."""
    _require_runtime()
    rows, experts, hidden, ffn = _block_shape(x, w13, w2)
    code = _operand_type("x", x)
    dtype, device = x.dtype, x.device
    args = _native.FfnArgs(code, experts, rows, hidden, ffn, _offsets(offs, experts, device))
    args.y, args.y_pitch = _token("dy", dy, rows, hidden, dtype, device)
    args.x, args.x_pitch = _token("x", x, rows, hidden, dtype, device)
    args.w13, args.w13_pitch, args.w13_stride = _weight("w13", w13, experts, hidden, 2 * ffn, dtype, device)
    args.w2, args.w2_pitch, args.w2_stride = _weight("w2", w2, experts, ffn, hidden, dtype, device)
    args.h, args.h_pitch = _token("h", h, rows, ffn, dtype, device)
    args.gate_up, args.gate_up_pitch = _token("gate_up", gate_up, rows, 2 * ffn, dtype, device)
    if dx is None:
        dx = _rows_of(x, rows, hidden)
    if dw13 is None:
        dw13 = w13.new_empty(w13.shape)
    if dw2 is None:
        dw2 = w2.new_empty(w2.shape)
    args.dx, args.dx_pitch = _token("dx", dx, rows, hidden, dtype, device)
    args.dw13, args.dw13_pitch, args.dw13_stride = _weight("dw13", dw13, experts, hidden, 2 * ffn, dtype, device)
    args.dw2, args.dw2_pitch, args.dw2_stride = _weight("dw2", dw2, experts, ffn, hidden, dtype, device)
    # One workspace: the gradient of gate_up between the two launches, then
    # the scratch (128-byte aligned behind it).
    behind = -(-rows * 2 * ffn // 64) * 64
    nbytes = _native.ffn_scratch_bytes(experts, _native.FFN_BACKWARD)
    workspace = x.new_empty(behind + nbytes // 2)
    at = workspace.data_ptr()
    args.dgate_up, args.dgate_up_pitch = at, 2 * ffn
    _call(device, _native.gated_ffn_backward, args, at + behind * 2, nbytes)
    return dx, dw13, dw2


def launch_grouped_mm_dgrad(dc, mat_b, offs=None, out=None, *, gate_up=None):
    """Gradient of ``launch_grouped_mm(a, mat_b, offs)`` with respect to ``a``,
    for fp16 and bf16, sizes that are multiples of 8 and one segment per expert
    (not for offsets of several segments per expert):
    ``out[rows of e] = dc[rows of e] @ mat_b[e].T`` with ``dc [T, N]``,
    ``mat_b [E, K, N]`` (or ``[K, N]``), ``out [T, K]``.  With ``gate_up
    [T, 2K]`` the product is the gradient of ``h = silu(gate) * up`` and the
    kernel's epilogue goes on to the gradient of ``gate_up``, ``out [T, 2K]``
    (dh itself is never written).  Returns ``out``."""
    _require_runtime()
    if dc.ndim != 2 or mat_b.ndim not in (2, 3):
        raise ValueError("expected dc [T, N] and mat_b [E, K, N] or [K, N]")
    rows = dc.shape[0]
    experts = mat_b.shape[0] if mat_b.ndim == 3 else 1
    k, n = mat_b.shape[-2:]
    _sizes(n, k)
    code = _operand_type("dc", dc)
    device = dc.device
    ends = _offsets(offs, experts, device)
    dc_at, dc_pitch = _token("dc", dc, rows, n, dc.dtype, device)
    b_at, b_pitch, b_stride = _weight("mat_b", mat_b, experts, k, n, dc.dtype, device)
    cols = k if gate_up is None else 2 * k
    gu_at, gu_pitch = (0, 0) if gate_up is None else _token("gate_up", gate_up, rows, cols, dc.dtype, device)
    if out is None:
        out = _rows_of(dc, rows, cols)
    out_at, out_pitch = _token("out", out, rows, cols, dc.dtype, device)
    scratch, nbytes = _scratch(dc, _native.ffn_scratch_bytes(experts, _native.FFN_DGRAD))
    _call(device, _native.grouped_dgrad, dc_at, dc_pitch, b_at, b_pitch, b_stride, ends, experts, rows, n, k, gu_at,
          gu_pitch, out_at, out_pitch, code, scratch.data_ptr() if nbytes else 0, nbytes)
    return out


def launch_grouped_mm_wgrad(mat_a, dc, offs=None, out=None):
    """Gradient of ``launch_grouped_mm(mat_a, b, offs)`` with respect to ``b``,
    in the types and sizes of ``launch_grouped_mm_dgrad``, one matrix per segment
    (the sum over an expert's segments, where it has several, is the caller's):
    ``out[e] = mat_a[rows of e].T @ dc[rows of e]`` with ``mat_a [T, K]``,
    ``dc [T, N]``, ``out [E, K, N]`` (``[K, N]`` without ``offs``); zeros for an
    expert without rows.  Returns ``out``."""
    _require_runtime()
    if mat_a.ndim != 2 or dc.ndim != 2:
        raise ValueError("expected mat_a [T, K] and dc [T, N]")
    rows, k = mat_a.shape
    n = dc.shape[1]
    _sizes(k, n)
    code = _operand_type("mat_a", mat_a)
    device = mat_a.device
    experts = 1 if offs is None else int(offs.numel())
    if experts == 0:
        raise ValueError("offs is empty")
    ends = _offsets(offs, experts, device)
    a_at, a_pitch = _token("mat_a", mat_a, rows, k, mat_a.dtype, device)
    dc_at, dc_pitch = _token("dc", dc, rows, n, mat_a.dtype, device)
    if out is None:
        out = mat_a.new_empty((k, n) if offs is None else (experts, k, n))
    out_at, out_pitch, out_stride = _weight("out", out, experts, k, n, mat_a.dtype, device)
    scratch, nbytes = _scratch(mat_a, _native.ffn_scratch_bytes(experts, _native.FFN_WGRAD))
    _call(device, _native.grouped_wgrad, a_at, a_pitch, dc_at, dc_pitch, ends, experts, rows, n, k, out_at, out_pitch,
          out_stride, code, scratch.data_ptr(), nbytes)
    return out

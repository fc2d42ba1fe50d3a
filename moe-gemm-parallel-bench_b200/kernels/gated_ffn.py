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
are zeros); rows past ``offs[-1]`` are neither read nor written.  The single
products' gradients are there as well: ``launch_grouped_mm_dgrad`` and
``launch_grouped_mm_wgrad``.

fp16 or bf16; hidden and ffn sizes are multiples of 8, bases 16-byte aligned,
columns contiguous, rows may be padded to a pitch that is a multiple of 8.
Accumulation is fp32; ``gate_up``, ``h`` and the gradient of ``gate_up`` are
rounded once to the operands' type between products.  Inputs and outputs must
not overlap.  Every call is launches only (no synchronisation), on the current
stream of the tensors' device, with its scratch allocated on that stream, so it
can be captured in a CUDA graph.  The calls are explicit: autograd does not see
them.  The reference has no counterpart (SiLU(gate) * up and all gradients stay
outside its timed path, README.md:55-60).
"""

from __future__ import annotations

try:
    import torch
except ImportError:  # pragma: no cover - the CPU tests import the host helpers only
    torch = None

from . import _native
from .matmul import dtype_name


def _require_runtime() -> None:
    if torch is None or not torch.cuda.is_available():
        raise RuntimeError("CUDA PyTorch and the native sm_100a library are required")
    _native.load()


def _token(name: str, t, rows: int, cols: int, like) -> tuple[int, int]:
    """(address, pitch) of a [rows, cols] tensor of `like`'s type and device."""
    if t.ndim != 2 or t.shape[0] != rows or t.shape[1] != cols:
        raise ValueError(f"{name} must be [{rows}, {cols}], got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    pitch = t.stride(0) if rows > 1 else cols
    address = t.data_ptr()
    if t.stride(1) != 1 or pitch < cols or pitch % 8 or address % 16:
        raise ValueError(f"{name} needs contiguous columns, a 16-byte aligned base and a row pitch that is a multiple of 8")
    return address, pitch


def _weight(name: str, t, experts: int, rows: int, cols: int, like) -> tuple[int, int, int]:
    """(address, pitch, expert stride) of an [experts, rows, cols] weight (or [rows, cols] for one expert)."""
    dense = t.ndim == 2 and experts == 1
    if tuple(t.shape) != ((rows, cols) if dense else (experts, rows, cols)):
        raise ValueError(f"{name} must be [{experts}, {rows}, {cols}], got {tuple(t.shape)}")
    if t.dtype != like.dtype or t.device != like.device:
        raise ValueError(f"{name} must be {like.dtype} on {like.device}, got {t.dtype} on {t.device}")
    pitch = t.stride(-2)
    stride = t.stride(0) if experts > 1 else rows * pitch
    address = t.data_ptr()
    if t.stride(-1) != 1 or pitch < cols or pitch % 8 or stride % 8 or address % 16 or (
            experts > 1 and stride < (rows - 1) * pitch + cols):
        raise ValueError(f"{name} needs contiguous columns, a 16-byte aligned base, a row pitch and an expert stride "
                         "that are multiples of 8, and experts that do not overlap")
    return address, pitch, stride


def _operand_type(name: str, t) -> int:
    if not t.is_cuda:
        raise ValueError(f"{name} must be on a CUDA device")
    code = _native.DTYPE_CODES[dtype_name(t.dtype)]
    if t.dtype == torch.float32:
        raise ValueError(f"{name} must be float16 or bfloat16")
    return code


def _offsets(offs, experts: int, like) -> int:
    """Address of the row ends (0: one segment of every row)."""
    if offs is None:
        if experts != 1:
            raise ValueError("offs (int32 cumulative row ends) is needed with more than one expert")
        return 0
    if offs.ndim != 1 or offs.shape[0] != experts or offs.dtype != torch.int32 or not offs.is_contiguous():
        raise ValueError(f"offs must be contiguous int32 [{experts}] cumulative row ends")
    if offs.device != like.device:
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


def _scratch(experts: int, jobs: int, device):
    return torch.empty(_native.ffn_scratch_bytes(experts, jobs), dtype=torch.uint8, device=device)


def gated_ffn_forward(x, w13, w2, offs=None, *, out=None, h=None, gate_up=None):
    """(y, h, gate_up) of the block: ``x [T, H]``, ``w13 [E, H, 2F]`` packed
    [gate | up], ``w2 [E, F, H]``; ``[H, 2F]`` and ``[F, H]`` for one expert.
    ``y [T, H]`` is the output; ``h [T, F]`` and ``gate_up [T, 2F]`` are what
    ``gated_ffn_backward`` reads.  Tensors given for the three outputs are
    written in place."""
    _require_runtime()
    rows, experts, hidden, ffn = _block_shape(x, w13, w2)
    code = _operand_type("x", x)
    device = x.device
    args = _native.FfnArgs(code, experts, rows, hidden, ffn, _offsets(offs, experts, x))
    args.x, args.x_pitch = _token("x", x, rows, hidden, x)
    args.w13, args.w13_pitch, args.w13_stride = _weight("w13", w13, experts, hidden, 2 * ffn, x)
    args.w2, args.w2_pitch, args.w2_stride = _weight("w2", w2, experts, ffn, hidden, x)
    if out is None:
        out = torch.empty((rows, hidden), dtype=x.dtype, device=device)
    if h is None:
        h = torch.empty((rows, ffn), dtype=x.dtype, device=device)
    if gate_up is None:
        gate_up = torch.empty((rows, 2 * ffn), dtype=x.dtype, device=device)
    args.y, args.y_pitch = _token("out", out, rows, hidden, x)
    args.h, args.h_pitch = _token("h", h, rows, ffn, x)
    args.gate_up, args.gate_up_pitch = _token("gate_up", gate_up, rows, 2 * ffn, x)
    scratch = _scratch(experts, 2, device)
    with torch.cuda.device(device):
        _native.gated_ffn_forward(args, scratch.data_ptr(), scratch.numel(),
                                  torch.cuda.current_stream(device).cuda_stream)
    return out, h, gate_up


def gated_ffn_backward(dy, x, w13, w2, h, gate_up, offs=None, *, dx=None, dw13=None, dw2=None):
    """(dx, dw13, dw2) from the output's gradient ``dy [T, H]``, the block's
    inputs and the ``h`` and ``gate_up`` that ``gated_ffn_forward`` returned.
    Gradients have their tensor's shape and type; tensors given for them are
    overwritten (nothing is accumulated)."""
    _require_runtime()
    rows, experts, hidden, ffn = _block_shape(x, w13, w2)
    code = _operand_type("x", x)
    device = x.device
    args = _native.FfnArgs(code, experts, rows, hidden, ffn, _offsets(offs, experts, x))
    args.y, args.y_pitch = _token("dy", dy, rows, hidden, x)
    args.x, args.x_pitch = _token("x", x, rows, hidden, x)
    args.w13, args.w13_pitch, args.w13_stride = _weight("w13", w13, experts, hidden, 2 * ffn, x)
    args.w2, args.w2_pitch, args.w2_stride = _weight("w2", w2, experts, ffn, hidden, x)
    args.h, args.h_pitch = _token("h", h, rows, ffn, x)
    args.gate_up, args.gate_up_pitch = _token("gate_up", gate_up, rows, 2 * ffn, x)
    if dx is None:
        dx = torch.empty((rows, hidden), dtype=x.dtype, device=device)
    if dw13 is None:
        dw13 = torch.empty(w13.shape, dtype=x.dtype, device=device)
    if dw2 is None:
        dw2 = torch.empty(w2.shape, dtype=x.dtype, device=device)
    dgate_up = torch.empty((rows, 2 * ffn), dtype=x.dtype, device=device)
    args.dgate_up, args.dgate_up_pitch = dgate_up.data_ptr(), 2 * ffn
    args.dx, args.dx_pitch = _token("dx", dx, rows, hidden, x)
    args.dw13, args.dw13_pitch, args.dw13_stride = _weight("dw13", dw13, experts, hidden, 2 * ffn, x)
    args.dw2, args.dw2_pitch, args.dw2_stride = _weight("dw2", dw2, experts, ffn, hidden, x)
    scratch = _scratch(experts, 4, device)
    with torch.cuda.device(device):
        _native.gated_ffn_backward(args, scratch.data_ptr(), scratch.numel(),
                                   torch.cuda.current_stream(device).cuda_stream)
    return dx, dw13, dw2


def launch_grouped_mm_dgrad(dc, mat_b, offs=None, out=None, *, gate_up=None):
    """Gradient of ``launch_grouped_mm(a, mat_b, offs)`` with respect to ``a``:
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
    ends = _offsets(offs, experts, dc)
    dc_at, dc_pitch = _token("dc", dc, rows, n, dc)
    b_at, b_pitch, b_stride = _weight("mat_b", mat_b, experts, k, n, dc)
    cols = k if gate_up is None else 2 * k
    gu_at, gu_pitch = (0, 0) if gate_up is None else _token("gate_up", gate_up, rows, cols, dc)
    if out is None:
        out = torch.empty((rows, cols), dtype=dc.dtype, device=device)
    out_at, out_pitch = _token("out", out, rows, cols, dc)
    if rows == 0:
        return out
    scratch = _scratch(experts, 1, device)
    with torch.cuda.device(device):
        _native.grouped_dgrad(dc_at, dc_pitch, b_at, b_pitch, b_stride, ends, experts, rows, n, k, gu_at, gu_pitch,
                              out_at, out_pitch, code, scratch.data_ptr(), scratch.numel(),
                              torch.cuda.current_stream(device).cuda_stream)
    return out


def launch_grouped_mm_wgrad(mat_a, dc, offs=None, out=None):
    """Gradient of ``launch_grouped_mm(mat_a, b, offs)`` with respect to ``b``:
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
    ends = _offsets(offs, experts, mat_a)
    a_at, a_pitch = _token("mat_a", mat_a, rows, k, mat_a)
    dc_at, dc_pitch = _token("dc", dc, rows, n, mat_a)
    if out is None:
        out = torch.empty((k, n) if offs is None else (experts, k, n), dtype=mat_a.dtype, device=device)
    out_at, out_pitch, out_stride = _weight("out", out, experts, k, n, mat_a)
    scratch = _scratch(experts, 1, device)
    with torch.cuda.device(device):
        _native.grouped_wgrad(a_at, a_pitch, dc_at, dc_pitch, ends, experts, rows, n, k, out_at, out_pitch,
                              out_stride, code, scratch.data_ptr(), scratch.numel(),
                              torch.cuda.current_stream(device).cuda_stream)
    return out

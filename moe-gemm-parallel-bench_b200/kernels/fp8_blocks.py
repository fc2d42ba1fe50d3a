"""e4m3 products with power-of-two block scales, and the quantisation to them.

``kernels.fp8`` multiplies e4m3 experts whose 128-deep K blocks carry fp32
scales.  Checkpoints and training recipes that keep those scales as powers of
two (e8m0, one byte: 2^(byte - 127), ``torch.float8_e8m0fnu``) leave nothing
to do outside the tensor core, whose block-scaled MMA applies them itself:

    C[rows of e] (bf16) = sum_kb 2^sa[:, kb] * (A[rows of e, kb] @ B[e][:, kb].T) * 2^sb[e][n // 128, kb]

``launch_quantize_rows`` (activations: a scale per token and 128-deep block)
and ``launch_quantize_blocks`` (weights: a scale per 128 x 128 block) produce
the operands: s is the smallest power of two with max |x| <= 448 s over the
block's finite values (1 for a block of zeros), q = x / s rounded to nearest
even, infinities and NaNs become NaN; a call makes fewer than 2^31 scales.
``launch_block_scaled_mm`` multiplies
them, dense or over expert-sorted rows, from one token to whole prompts.
Every call is launches only, on the current stream of the tensors' device, and
can be captured in a CUDA graph.  The reference has no counterpart (it does not
emulate the model's FP8 quantization, README.md:298).
"""

from __future__ import annotations

try:
    import torch
except ImportError:  # pragma: no cover - the CPU tests import the host helpers only
    torch = None

from . import _native
from .fp8 import FP8_BLOCK, _blocks
from .gated_ffn import _call, _offsets, _require_runtime
from .matmul import dtype_name

_last_info = None


def last_block_scaled_info() -> dict | None:
    """Native kernel of the most recent launch_block_scaled_mm call (path, tile, grid)."""
    return None if _last_info is None else _last_info.as_dict()


def _source(x, cols: int, steps: tuple) -> int:
    if not x.is_cuda:
        raise ValueError("the tensor to quantise must be on a CUDA device")
    if steps[-1] != 1 and cols > 1:
        raise ValueError("the tensor to quantise needs contiguous columns")
    return _native.DTYPE_CODES[dtype_name(x.dtype)]


def _target(name: str, t, shape: tuple, dtype, device):
    if t is None:  # empty_strided: the shortest way to a tensor on the host side
        steps = (shape[1], 1) if len(shape) == 2 else (shape[1] * shape[2], shape[2], 1)
        return torch.empty_strided(shape, steps, dtype=dtype, device=device)
    if t.shape != shape or t.dtype != dtype or t.device != device or not t.is_contiguous():
        raise ValueError(f"{name} must be a contiguous {dtype} {shape} tensor on {device}")
    return t


def launch_quantize_rows(x, q=None, scale=None):
    """(q, scale) of activations ``x [M, K]`` (fp16, bf16 or fp32; rows may be
    padded): q float8_e4m3fn ``[M, K]``, scale float8_e8m0fnu ``[M, ceil(K / 128)]``."""
    _require_runtime()
    shape = x.shape
    if len(shape) != 2 or shape[1] == 0:
        raise ValueError(f"expected x [M, K], got {tuple(shape)}")
    rows, cols = shape
    steps = x.stride()
    code = _source(x, cols, steps)
    device = x.device
    q = _target("q", q, (rows, cols), torch.float8_e4m3fn, device)
    scale = _target("scale", scale, (rows, _blocks(cols)), torch.float8_e8m0fnu, device)
    pitch = steps[0] if rows > 1 else cols
    if pitch < cols:
        raise ValueError("rows of x must not overlap")
    _call(device, _native.quantize_rows, x.data_ptr(), rows, cols, pitch, code, q.data_ptr(), cols, scale.data_ptr())
    return q, scale


def launch_quantize_blocks(w, q=None, scale=None):
    """(q, scale) of weights ``w [N, K]`` or ``[E, N, K]`` (fp16, bf16 or
    fp32): q float8_e4m3fn of w's shape, scale float8_e8m0fnu ``[(E,)
    ceil(N / 128), ceil(K / 128)]``."""
    _require_runtime()
    if w.ndim not in (2, 3) or w.shape[-1] == 0 or w.shape[-2] == 0:
        raise ValueError(f"expected w [N, K] or [E, N, K], got {tuple(w.shape)}")
    steps = w.stride()
    *lead, n, k = w.shape
    code = _source(w, k, steps)
    matrices = lead[0] if lead else 1
    device = w.device
    q = _target("q", q, tuple(w.shape), torch.float8_e4m3fn, device)
    scale = _target("scale", scale, (*lead, _blocks(n), _blocks(k)), torch.float8_e8m0fnu, device)
    pitch = steps[-2] if n > 1 else k
    stride = steps[0] if matrices > 1 else n * pitch
    if pitch < k or (matrices > 1 and stride < (n - 1) * pitch + k):
        raise ValueError("rows and matrices of w must not overlap")
    _call(device, _native.quantize_blocks, w.data_ptr(), matrices, n, k, pitch, stride, code, q.data_ptr(),
          scale.data_ptr())
    return q, scale


def launch_block_scaled_mm(a, sa, b, sb, offs=None, out=None):
    """``out [T, N]`` (bf16) of tokens ``a [T, K]`` with scales ``sa [T,
    ceil(K / 128)]`` and weights ``b [N, K]`` or ``[E, N, K]`` with scales ``sb
    [(E,) ceil(N / 128), ceil(K / 128)]``; with experts the rows are sorted and
    ``offs`` (int32 ``[E]``) holds their cumulative row ends.  Empty experts are
    fine; rows past ``offs[-1]`` have no effect and are not written.  K is a multiple
    of 16, N of 8; rows of a, b and out may be padded to whole 16 bytes, scales
    are contiguous.  With few tokens per expert (8 on average) and few weight
    rows the weights are streamed by many small CTAs, else 64 x 128, 128 x 128 or
    CTA-pair tiles (224 x 256) run on the block-scaled tensor-core MMA."""
    global _last_info
    _require_runtime()
    a_shape, b_shape = a.shape, b.shape
    if len(a_shape) != 2 or len(b_shape) not in (2, 3):
        raise ValueError("expected a [T, K] and b [N, K] or [E, N, K]")
    device = a.device
    if not a.is_cuda or sa.device != device or b.device != device or sb.device != device:
        raise ValueError("a, sa, b and sb must be on the same CUDA device")
    if a.dtype != torch.float8_e4m3fn or b.dtype != torch.float8_e4m3fn:
        raise ValueError("a and b must be float8_e4m3fn")
    if sa.dtype != torch.float8_e8m0fnu or sb.dtype != torch.float8_e8m0fnu:
        raise ValueError("sa and sb must be float8_e8m0fnu")
    rows, k = a_shape
    *lead, n, kb = b_shape
    experts = lead[0] if lead else 1
    if kb != k or k == 0 or n == 0 or experts == 0 or k % 16 or n % 8:
        raise ValueError(f"a {tuple(a_shape)} and b {tuple(b_shape)} need one K, a multiple of 16, and N a multiple of 8")
    blocks = _blocks(k)
    if sa.shape != (rows, blocks) or sb.shape != (*lead, _blocks(n), blocks):
        raise ValueError(f"scale shapes {tuple(sa.shape)} / {tuple(sb.shape)} do not match a {tuple(a_shape)}, "
                         f"b {tuple(b_shape)} in blocks of {FP8_BLOCK}")
    if not sa.is_contiguous() or not sb.is_contiguous():
        raise ValueError("scales must be contiguous")
    ends = _offsets(offs, experts, device)
    if out is None:
        out = torch.empty_strided((rows, n), (n, 1), dtype=torch.bfloat16, device=device)
    elif out.shape != (rows, n) or out.dtype != torch.bfloat16 or out.device != device:
        raise ValueError(f"out must be [{rows}, {n}] bfloat16 on {device}")
    a_steps, b_steps, out_steps = a.stride(), b.stride(), out.stride()
    a_pitch = a_steps[0] if rows > 1 else k
    out_pitch = out_steps[0] if rows > 1 else n
    b_pitch = b_steps[-2]
    b_stride = b_steps[0] if experts > 1 else n * b_pitch
    a_at, b_at, out_at = a.data_ptr(), b.data_ptr(), out.data_ptr()
    if a_steps[1] != 1 or b_steps[-1] != 1 or out_steps[1] != 1 or a_pitch < k or a_pitch % 16 or b_pitch < k or (
            b_pitch % 16) or b_stride % b_pitch or b_stride < n * b_pitch or out_pitch < n or out_pitch % 8 or (
            (a_at | b_at | out_at) % 16):
        raise ValueError("a, b and out need contiguous columns, 16-byte aligned bases, rows a whole number of 16 bytes "
                         "apart that do not overlap, and experts a whole number of rows apart")
    nbytes = _native.block_scaled_scratch_bytes(experts) if experts > 1 else 0
    scratch = a.new_empty(nbytes) if nbytes else None
    _last_info = _call(device, _native.block_scaled_mm, a_at, a_pitch, sa.data_ptr(), b_at, b_pitch,
                       b_stride, sb.data_ptr(), out_at, out_pitch, ends, experts, rows, n, k,
                       scratch.data_ptr() if nbytes else 0, nbytes)
    return out

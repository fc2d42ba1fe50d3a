"""Tensors of more than 2^31 elements, thousands of experts, and forms of the C
calls that no Python call makes.  Rows, columns and experts are checked where
an offset of 32 bits would end: at the far end."""

from __future__ import annotations

import pytest

from kernels import _native

torch = pytest.importorskip("torch")
import kernels  # noqa: E402
from tests.test_fp8_blocks import BLOCK, HALF, check_quantized  # noqa: E402
from tests.test_gated_ffn import Block, within  # noqa: E402


@pytest.fixture(autouse=True)
def memory():
    torch.cuda.empty_cache()
    yield
    torch.cuda.empty_cache()


def normal(shape, dtype=torch.bfloat16, seed=0):
    """Rows that repeat every 65537: whole tensors would take longer to draw than to multiply."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    base = torch.randn((min(shape[0], 65537), *shape[1:]), device="cuda", generator=gen, dtype=torch.float32).to(dtype)
    out = torch.empty(shape, dtype=dtype, device="cuda")
    for at in range(0, shape[0], base.shape[0]):
        n = min(base.shape[0], shape[0] - at)
        out[at:at + n] = base[:n]
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("k", [1024, 1000])
def test_quantized_rows(k):
    m = (1 << 32) // k + 5
    x = normal((m, k))
    q, scale = kernels.launch_quantize_rows(x)
    kernels.check_device_errors()
    for part in (slice(0, 300), slice((1 << 31) // k - 150, (1 << 31) // k + 150), slice(m - 300, m)):
        check_quantized((q[part], scale[part]), x[part], 1)


@pytest.mark.gpu
def test_quantized_blocks():
    x = normal((70, 8192 * 8192)).view(70, 8192, 8192)  # 4.7e9 elements
    q, scale = kernels.launch_quantize_blocks(x)
    kernels.check_device_errors()
    for e in (0, 31, 32, 69):
        check_quantized((q[e, -512:], scale[e, -4:]), x[e, -512:], BLOCK)


@pytest.mark.gpu
def test_block_scaled_product():
    rows, n, k = 600_011, 4096, 256
    gen = torch.Generator(device="cuda").manual_seed(2)
    a, sa = kernels.launch_quantize_rows(normal((rows, k), seed=2))
    b, sb = kernels.launch_quantize_blocks(torch.randn((2, n, k), device="cuda", generator=gen))
    first = 300_000
    offs = torch.tensor([first, rows], dtype=torch.int32, device="cuda")
    out = kernels.launch_block_scaled_mm(a, sa, b, sb, offs)
    kernels.check_device_errors()
    cols = torch.arange(k, device="cuda") // BLOCK
    for part, e in ((slice(first - 300, first), 0), (slice(first, first + 300), 1), (slice(rows - 300, rows), 1),
                    (slice((1 << 31) // n - 150, (1 << 31) // n + 150), 1)):
        wide_a = a[part].double() * torch.exp2(sa[part].view(torch.uint8).double() - 127)[:, cols]
        scales = torch.exp2(sb[e].view(torch.uint8).double() - 127).repeat_interleave(BLOCK, 0)[:, cols]
        w = b[e].double() * scales
        value = wide_a @ w.t()
        bound = 1.01 * (HALF * value.abs() + k * 2.0**-23 * (wide_a.abs() @ w.abs().t()))
        assert bool(((out[part].double() - value).abs() <= bound).all())


class FarEnd(Block):
    """A block over rows that exist already; its formulas are taken over the last segments only."""

    def __init__(self, x, dy, w13, w2, lengths):
        self.x, self.dy, self.w13, self.w2, self.lengths = x, dy, w13, w2, lengths
        self.dtype, self.hidden, self.ffn = x.dtype, x.shape[1], w2.shape[1]


@pytest.mark.gpu
def test_feed_forward_block():
    rows, hidden, ffn = 300_011, 64, 4096  # gate_up: 2.46e9 elements
    gen = torch.Generator(device="cuda").manual_seed(4)
    lengths = [rows - 700, 400, 300]
    offs = torch.tensor(lengths).cumsum(0).to(torch.int32).cuda()
    x, dy = normal((rows, hidden), seed=4), normal((rows, hidden), seed=5)
    w13 = (torch.randn((3, hidden, 2 * ffn), device="cuda", generator=gen) / 8).to(torch.bfloat16)
    w2 = (torch.randn((3, ffn, hidden), device="cuda", generator=gen) / 64).to(torch.bfloat16)
    out = kernels.gated_ffn_forward(x, w13, w2, offs)
    y, h, gate_up = out
    kernels.check_device_errors()
    far = FarEnd(x[-700:], dy[-700:], w13[1:], w2[1:], lengths[1:])
    ref = far.forward()
    for what, got in zip(("y", "h", "gate_up"), out):
        within(got[-700:], ref[what], what)
    dx, dw13, dw2 = kernels.gated_ffn_backward(dy, x, w13, w2, h, gate_up, offs)
    kernels.check_device_errors()
    ref = far.backward(h[-700:], gate_up[-700:])
    within(dx[-700:], ref["dx"], "dx")
    within(dw13[1:], ref["dw13"], "dw13")
    within(dw2[1:], ref["dw2"], "dw2")


@pytest.mark.gpu
def test_thousands_of_experts():
    lengths = ([0, 1, 0, 3, 0, 0, 2, 129, 0, 1] * 300)[:2999]
    block = Block(lengths, 40, 24, torch.bfloat16, seed=6, tail=4)
    y, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    kernels.check_device_errors()
    within(y[:block.used], block.forward()["y"], "y")
    ref = block.backward(h, gate_up)
    within(grads[0][:block.used], ref["dx"], "dx")
    within(grads[1], ref["dw13"], "dw13")
    within(grads[2], ref["dw2"], "dw2")


@pytest.mark.gpu
@pytest.mark.parametrize("lengths", [[5], [70, 0, 333], [1, 2] * 120], ids=["one", "ragged", "many"])
def test_forward_without_a_down_projection(lengths):
    """The C call with a null w2: gate_up and h only, y neither read nor written."""
    block = Block(lengths, 136, 72, torch.float16, seed=7)
    _, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    experts, rows, hidden, ffn = len(lengths), block.rows, 136, 72
    only = torch.full_like(h, -1.0), torch.full_like(gate_up, -1.0)
    args = _native.FfnArgs(_native.DTYPE_CODES["fp16"], experts, rows, hidden, ffn, block.offs.data_ptr())
    for field, t, pitch in (("x", block.x, hidden), ("h", only[0], ffn), ("gate_up", only[1], 2 * ffn),
                            ("w13", block.w13, 2 * ffn)):
        setattr(args, field, t.data_ptr())
        setattr(args, field + "_pitch", pitch)
    args.w13_stride = hidden * 2 * ffn
    nbytes = _native.ffn_scratch_bytes(experts, _native.FFN_FORWARD)
    scratch = torch.empty(max(nbytes, 128), dtype=torch.uint8, device="cuda")
    _native.gated_ffn_forward(args, scratch.data_ptr(), nbytes, torch.cuda.current_stream().cuda_stream)
    kernels.check_device_errors()
    assert [i["epilogue"] for i in kernels.last_gated_ffn_info()] == ["swiglu"]
    assert torch.equal(only[0], h) and torch.equal(only[1], gate_up)

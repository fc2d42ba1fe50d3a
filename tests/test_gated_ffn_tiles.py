"""The gated feed-forward block's kernels, each shape with the launches that
must have run, so that a change of the choice cannot leave a kernel untested."""

from __future__ import annotations

import ctypes

import pytest

from kernels import _native

torch = pytest.importorskip("torch")
import kernels  # noqa: E402
from tests.test_gated_ffn import Block, saved_of, within  # noqa: E402

DTYPES = pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])


def launches():
    return [(i["epilogue"], i["pair"], i["tile_m"], i["tile_n"], i["split"]) for i in kernels.last_gated_ffn_info()]


def name(shape):
    return f"{sum(shape[0])}rows{len(shape[0])}e{shape[1]}x{shape[2]}"


SWIGLU_ONE, SWIGLU_PAIR = ("swiglu", False, 128, 64), ("swiglu", True, 256, 128)
BACK_ONE, BACK_PAIR = ("swiglu_backward", False, 128, 128), ("swiglu_backward", True, 256, 256)
ONE, PAIR, WIDE = ("plain", False, 128, 128), ("plain", True, 256, 256), ("plain", True, 256, 512)

# Shape; tiles of the two forward launches; of the two backward ones.  Pairs take
# several tiles each where a launch has more than 74.
SHAPES = [
    # 180 activation-gradient tiles; the last 512 columns of hidden hold 264
    (([1100, 0, 777, 5, 300, 1500], 2312, 2056), (SWIGLU_PAIR, WIDE), (BACK_PAIR, WIDE)),
    # the last 512 columns of hidden hold 136: a half without any
    (([900, 257, 0, 31, 500], 4232, 520), (SWIGLU_ONE, WIDE), (BACK_ONE, PAIR)),
    (([1100, 0, 777, 5, 300], 1160, 4104), (SWIGLU_PAIR, PAIR), (BACK_PAIR, PAIR)),
    (([2560], 1544, 2056), (SWIGLU_PAIR, PAIR), (BACK_PAIR, PAIR)),
    (([129, 0, 3], 136, 72), (SWIGLU_ONE, ONE), (BACK_ONE, ONE)),
]


@pytest.mark.gpu
@DTYPES
@pytest.mark.parametrize("shape,forward,backward", SHAPES, ids=lambda v: name(v) if isinstance(v[0], list) else "")
def test_tiles(shape, forward, backward, dtype):
    block = Block(*shape, dtype, seed=21, tail=7)
    out = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    kernels.check_device_errors()
    assert launches() == [(*tile, 1) for tile in forward]
    ref = block.forward()
    for what, got in zip(("y", "h", "gate_up"), out):
        within(got[:block.used], ref[what], what)
    del ref, out
    h, gate_up = saved_of(block)
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    kernels.check_device_errors()
    assert launches() == [(*tile, 1) for tile in backward]
    ref = block.backward(h, gate_up)
    within(grads[0][:block.used], ref["dx"], "dx")
    within(grads[1], ref["dw13"], "dw13")
    within(grads[2], ref["dw2"], "dw2")
    # The first backward launch alone, with what it hands to the second.
    dgate_up = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, block.offs, gate_up=gate_up)
    kernels.check_device_errors()
    assert launches() == [(*backward[0], 1)]
    within(dgate_up[:block.used], ref["dgate_up"], "dgate_up")


@pytest.mark.gpu
@DTYPES
def test_shared_contractions(dtype):
    """Launches of few tiles share a contraction among a cluster's CTAs, every epilogue."""
    block = Block([17], 4104, 136, dtype, seed=22)
    out = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    kernels.check_device_errors()
    assert launches()[0] == (*SWIGLU_ONE, 8)  # 65 blocks of 64
    ref = block.forward()
    for what, got in zip(("y", "h", "gate_up"), out):
        within(got, ref[what], what)
    h, gate_up = saved_of(block)
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    kernels.check_device_errors()
    assert launches()[0] == (*BACK_ONE, 8)
    ref = block.backward(h, gate_up)
    for what, got in zip(("dx", "dw13", "dw2"), grads):
        within(got, ref[what], what)
    # The plain epilogue: down projection and dx of a wide block.
    block = Block([33], 136, 4104, dtype, seed=23)
    y, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    assert launches()[1] == (*ONE, 8)
    within(y, block.forward()["y"], "y")
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    kernels.check_device_errors()
    assert launches()[1] == (*ONE, 8)
    within(grads[0], block.backward(h, gate_up)["dx"], "dx")


@pytest.mark.gpu
def test_grids():
    """At most a CTA per SM, at most a CTA or pair per tile, whole clusters."""
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    block = Block([700, 0, 40], 520, 264, torch.bfloat16, seed=24)
    y, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    infos = kernels.last_gated_ffn_info()
    kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    infos += kernels.last_gated_ffn_info()
    kernels.launch_grouped_mm_wgrad(h, block.dy, block.offs)
    infos += kernels.last_gated_ffn_info()
    kernels.check_device_errors()
    assert [i["epilogue"] for i in infos] == ["swiglu", "plain", "swiglu_backward", "plain", "plain"]
    for info in infos:
        ctas = info["split"] * (2 if info["pair"] else 1)
        assert 0 < info["grid"] <= sms and info["grid"] % ctas == 0, info
    none = Block([0, 0], 64, 40, torch.bfloat16)
    kernels.gated_ffn_forward(none.x, none.w13, none.w2, none.offs)
    assert kernels.last_gated_ffn_info() == []


def test_report_without_a_launch():
    lib = _native.load()
    assert lib.ffn_last_launches(None, 0) == lib.ffn_last_launches(None, 2)
    info = (_native.FfnLaunchInfo * 2)()
    info[0].grid = info[1].grid = -1
    lib.ffn_last_launches(info, 0)
    assert info[0].grid == info[1].grid == -1  # nothing written past the capacity
    assert lib.gated_ffn_forward_launch(ctypes.byref(_native.FfnArgs(2))) == _native.STATUS_INVALID


@pytest.mark.gpu
def test_no_rows_with_tensors_given():
    """A C caller may pass its buffers with zero rows: weight gradients become zeros, nothing else is touched."""
    hidden, ffn, experts = 64, 40, 3
    code = _native.DTYPE_CODES["bf16"]
    token = torch.full((16, 2 * ffn), 5.0, device="cuda", dtype=torch.bfloat16)
    w13 = torch.full((experts, hidden, 2 * ffn), 5.0, device="cuda", dtype=torch.bfloat16)
    w2 = torch.full((experts, ffn, hidden), 5.0, device="cuda", dtype=torch.bfloat16)
    dw13, dw2 = w13.clone(), w2.clone()
    offs = torch.zeros(experts, dtype=torch.int32, device="cuda")
    args = _native.FfnArgs(code, experts, 0, hidden, ffn, offs.data_ptr())
    for field, cols in (("x", hidden), ("y", hidden), ("dx", hidden), ("h", ffn), ("gate_up", 2 * ffn),
                        ("dgate_up", 2 * ffn)):
        setattr(args, field, token.data_ptr())
        setattr(args, field + "_pitch", cols)
    for field, t in (("w13", w13), ("w2", w2), ("dw13", dw13), ("dw2", dw2)):
        setattr(args, field, t.data_ptr())
        setattr(args, field + "_pitch", t.stride(1))
        setattr(args, field + "_stride", t.stride(0))
    nbytes = _native.ffn_scratch_bytes(experts, _native.FFN_BACKWARD)
    scratch = torch.empty(nbytes, dtype=torch.uint8, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    _native.gated_ffn_forward(args, 0, 0, stream)
    _native.gated_ffn_backward(args, scratch.data_ptr(), nbytes, stream)
    torch.cuda.synchronize()
    kernels.check_device_errors()
    assert launches() == [(*ONE, 1)]
    assert not dw13.any() and not dw2.any()
    assert bool((token == 5.0).all()) and bool((w13 == 5.0).all()) and bool((w2 == 5.0).all())


@pytest.mark.gpu
def test_a_long_contraction_is_not_a_lost_one():
    """A weight gradient's contraction is as long as its rows: here 15 thousand
    blocks of 64, milliseconds, under waits of a tenth of one for each block."""
    rows = 1_000_003
    gen = torch.Generator(device="cuda").manual_seed(25)
    a = torch.randint(-2, 3, (rows, 8), device="cuda", generator=gen).to(torch.bfloat16)
    dc = torch.randint(-1, 2, (rows, 16), device="cuda", generator=gen).to(torch.bfloat16)
    value = a.double().t() @ dc.double()  # whole numbers below 2^21: exact in fp32 sums
    kernels.launch_grouped_mm_wgrad(a, dc)  # loads the kernel under the usual waits
    torch.cuda.synchronize()
    try:
        _native.set_debug(200_000)
        out = kernels.launch_grouped_mm_wgrad(a, dc)
        torch.cuda.synchronize()
        kernels.check_device_errors()
    finally:
        _native.set_debug(0)
    assert torch.equal(out, value.to(torch.float32).to(torch.bfloat16))


@pytest.mark.gpu
def test_report_of_a_call_without_rows():
    """A call that launches nothing reports nothing, not the call before it."""
    block = Block([20, 30], 64, 40, torch.bfloat16, seed=26)
    kernels.launch_grouped_mm_dgrad(block.dy, block.w2, block.offs)
    assert len(launches()) == 1
    offs = torch.zeros(2, dtype=torch.int32, device="cuda")
    assert kernels.launch_grouped_mm_dgrad(block.dy[:0], block.w2, offs).shape == (0, 40)
    assert launches() == []
    many = Block([1] * 220, 64, 40, torch.bfloat16, seed=27)
    assert kernels.launch_grouped_mm_dgrad(many.dy[:0], many.w2, torch.zeros_like(many.offs)).shape == (0, 40)
    assert launches() == []
    kernels.check_device_errors()

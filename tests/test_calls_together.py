"""Calls of the feed-forward and block-scaled operators together: from threads
that never touched CUDA, and across streams that fork and join inside a graph."""

from __future__ import annotations

import threading

import pytest

torch = pytest.importorskip("torch")
import kernels  # noqa: E402
from tests.test_fp8_blocks import Product  # noqa: E402
from tests.test_gated_ffn import Block  # noqa: E402


def step(block):
    y, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    return (y, h, gate_up, *kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs))


def quantised(x, product):
    a, sa = kernels.launch_quantize_rows(x)
    return a, sa, kernels.launch_block_scaled_mm(a, sa, product.b, product.sb, product.offs)


def same(got, expected):
    return all(torch.equal(p.view(torch.uint8), q.view(torch.uint8)) for p, q in zip(got, expected))


@pytest.mark.gpu
def test_threads():
    """Each thread makes its first CUDA calls here, on a stream of its own."""
    blocks = [Block(lengths, 512, 264, torch.bfloat16, seed=41) for lengths in ([200, 0, 313], [3], [40, 60])]
    product = Product([200, 300], 264, 528, seed=42)
    x = torch.randn((500, 528), device="cuda").to(torch.bfloat16)
    expected = [step(b) for b in blocks]
    expected_mm = quantised(x, product)
    tiles = []
    for block in blocks:
        kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
        tiles.append(kernels.last_gated_ffn_info())
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            block = blocks[i % 3]
            with torch.cuda.stream(streams[i]):
                for _ in range(20):
                    got, mm = step(block), quantised(x, product)
                    kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
                    if kernels.last_gated_ffn_info() != tiles[i % 3]:
                        wrong.append((i, "report"))
                streams[i].synchronize()
                if not same(got, expected[i % 3]) or not same(mm, expected_mm):
                    wrong.append((i, "values"))
        except Exception as error:  # noqa: BLE001 - a thread's failure is the test's
            wrong.append((i, repr(error)))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    kernels.check_device_errors()
    assert not wrong, wrong


def dense(*shape, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, device="cuda", generator=gen).to(torch.bfloat16)


def first_calls():
    """Name, call returning a tuple of tensors: each entry point's launch as a thread's first CUDA work."""
    block, product = Block([70, 30], 136, 72, torch.float16, seed=43), Product([50], 136, 272, seed=43)
    few = Product([3], 136, 272, seed=43)
    a, b = dense(100, 136, seed=44), dense(2, 136, 264, seed=45)
    offs = torch.tensor([70, 100], dtype=torch.int32, device="cuda")
    return {
        "feed_forward": lambda: step(block),
        "dgrad": lambda: (kernels.launch_grouped_mm_dgrad(block.dy, block.w2, block.offs),),
        "wgrad": lambda: (kernels.launch_grouped_mm_wgrad(block.x, block.dy, block.offs),),
        "block_scaled": lambda: (product.run(),),
        "block_scaled_few": lambda: (few.run(),),
        "quantize": lambda: kernels.launch_quantize_rows(a),
        "grouped_mm": lambda: (kernels.launch_grouped_mm(a, b, offs),),
    }


@pytest.mark.gpu
@pytest.mark.parametrize("name", ["feed_forward", "dgrad", "wgrad", "block_scaled", "block_scaled_few", "quantize",
                                  "grouped_mm"])
def test_first_call_of_a_thread(name):
    """One call, on the default stream, is all that a thread does with CUDA."""
    call = first_calls()[name]
    expected = call()  # and torch keeps memory for the thread's tensors
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            got.append(call())
        except Exception as error:  # noqa: BLE001 - a thread's failure is the test's
            got.append(error)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert not isinstance(got[0], Exception), got[0]
    torch.cuda.synchronize()
    kernels.check_device_errors()
    assert same(got[0], expected)


@pytest.mark.gpu
def test_streams_that_fork_and_join_in_a_graph():
    """A launch may start under the kernel before it on its stream, but not under
    the work of another stream that it was made to wait for."""
    product = Product([700, 300], 2056, 1040, seed=44)
    block = Block([700, 300], 1040, 264, torch.bfloat16, seed=45)
    side = torch.cuda.Stream()
    x = torch.empty((1000, 1040), device="cuda", dtype=torch.bfloat16)
    source = torch.empty((1000, 1040), device="cuda", dtype=torch.bfloat16)
    slow = torch.randn((4096, 4096), device="cuda")

    def run():
        here = torch.cuda.current_stream()
        kernels.launch_quantize_rows(block.x)  # the kernel before, on this stream
        side.wait_stream(here)
        with torch.cuda.stream(side):
            for _ in range(3):
                torch.mm(slow, slow)
            x.copy_(source)
            q = kernels.launch_quantize_rows(x)
        kernels.launch_quantize_rows(block.dy)
        here.wait_stream(side)
        mm = kernels.launch_block_scaled_mm(*q, product.b, product.sb, product.offs)
        side.wait_stream(here)
        with torch.cuda.stream(side):
            for _ in range(3):
                torch.mm(slow, slow)
            x.mul_(2)
        kernels.launch_quantize_rows(block.dy)
        here.wait_stream(side)
        return (mm, *kernels.gated_ffn_forward(x, block.w13, block.w2, block.offs))

    source.normal_()
    run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run()
    for seed in range(5):
        torch.manual_seed(seed)
        source.normal_()
        x.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        q = kernels.launch_quantize_rows(source)
        mm = kernels.launch_block_scaled_mm(*q, product.b, product.sb, product.offs)
        expected = (mm, *kernels.gated_ffn_forward(source * 2, block.w13, block.w2, block.offs))
        torch.cuda.synchronize()
        kernels.check_device_errors()
        assert same(out, expected)


@pytest.mark.gpu
def test_first_call_of_a_thread_inside_a_capture():
    block, product = Block([70, 30], 136, 72, torch.float16, seed=46), Product([50], 136, 272, seed=46)
    expected = (*step(block), product.run())
    torch.cuda.synchronize()
    got = []

    def work():
        try:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = (*step(block), product.run())
            graph.replay()
            torch.cuda.synchronize()
            got.append((graph, out))
        except Exception as error:  # noqa: BLE001 - a thread's failure is the test's
            got.append(error)

    thread = threading.Thread(target=work)
    thread.start()
    thread.join()
    assert not isinstance(got[0], Exception), got[0]
    kernels.check_device_errors()
    assert same(got[0][1], expected)

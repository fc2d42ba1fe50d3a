"""The gated feed-forward block (forward, backward) and the grouped products'
gradients against their formulas in 64 bits.

Tolerances are bounds, element by element: u = eps / 2 of the type for every
rounding to it, and per product of depth K an fp32 accumulation error of at
most K 2^-23 sum |a| |b| (every add off by at most one unit in the last place,
truncating adders included).  The activation's fast exponential and divide are
within 2^-18 of their arguments' products.  fp16 results below its normal
range are off by at most 2^-25.
"""

from __future__ import annotations

import ctypes

import pytest

from kernels import _native

torch = pytest.importorskip("torch")
import kernels  # noqa: E402

ACC = 2.0**-23
FAST = 2.0**-18
TINY = 2.0**-25


def half_step(dtype) -> float:
    return torch.finfo(dtype).eps / 2


def segments(lengths):
    at = 0
    for e, n in enumerate(lengths):
        yield e, slice(at, at + n)
        at += n


class Block:
    """Inputs of one block on the GPU and its formulas in 64 bits with error bounds."""

    def __init__(self, lengths, hidden, ffn, dtype, seed=0, tail=0, pad=0, dense=False):
        gen = torch.Generator(device="cuda").manual_seed(seed)

        def normal(shape, std=1.0):
            *lead, cols = shape
            wide = torch.full((*lead, cols + pad), float("nan"), device="cuda", dtype=dtype)
            wide[..., :cols] = (torch.randn(shape, device="cuda", generator=gen) * std).to(dtype)
            return wide[..., :cols]

        self.lengths, self.hidden, self.ffn, self.dtype = lengths, hidden, ffn, dtype
        self.rows = sum(lengths) + tail
        self.used = sum(lengths)
        experts = len(lengths)
        self.x = normal((self.rows, hidden))
        self.dy = normal((self.rows, hidden))
        self.x[self.used:] = float("nan")  # rows behind the last segment
        self.dy[self.used:] = float("nan")
        self.w13 = normal((experts, hidden, 2 * ffn), hidden**-0.5)
        self.w2 = normal((experts, ffn, hidden), ffn**-0.5)
        ends = torch.tensor(lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        self.offs = None if dense else ends
        if dense:
            self.w13, self.w2 = self.w13[0], self.w2[0]

    def weights(self, e):
        w13, w2 = (self.w13, self.w2) if self.w13.ndim == 2 else (self.w13[e], self.w2[e])
        return w13.double(), w2.double()

    def forward(self):
        """{name: (value, bound)} of y, h and gate_up over the used rows."""
        u, f = half_step(self.dtype), self.ffn
        out = {"y": [], "h": [], "gate_up": []}
        for e, rows in segments(self.lengths):
            w13, w2 = self.weights(e)
            x = self.x[rows].double()
            pre = x @ w13
            e_pre = self.hidden * ACC * (x.abs() @ w13.abs())
            g, up = pre[:, :f], pre[:, f:]
            s = torch.sigmoid(g)
            h = g * s * up
            # |d silu / dg| <= 1.1
            e_h = 1.1 * e_pre[:, :f] * up.abs() + (g * s).abs() * e_pre[:, f:] + e_pre[:, :f] * e_pre[:, f:] * 1.1
            e_h = e_h + FAST * (1 + g.abs()) * h.abs() + u * h.abs() + TINY
            y = h @ w2
            e_y = e_h @ w2.abs() + f * ACC * (h.abs() @ w2.abs()) + u * y.abs() + TINY
            out["y"].append((y, 1.01 * e_y))
            out["h"].append((h, 1.01 * e_h))
            out["gate_up"].append((pre, 1.01 * (e_pre + u * pre.abs()) + TINY))
        return {k: tuple(torch.cat(p) for p in zip(*v)) for k, v in out.items()}

    def backward(self, h, gate_up):
        """{name: (value, bound)} of dx (used rows), dw13, dw2 and dgate_up."""
        u, f = half_step(self.dtype), self.ffn
        out = {"dx": [], "dgate_up": []}
        stacks = {"dw13": [], "dw2": []}
        for e, rows in segments(self.lengths):
            w13, w2 = self.weights(e)
            x, dy = self.x[rows].double(), self.dy[rows].double()
            g, up = gate_up[rows, :f].double(), gate_up[rows, f:].double()
            hh = h[rows].double()
            n = x.shape[0]
            dh = dy @ w2.t()
            e_dh = self.hidden * ACC * (dy.abs() @ w2.abs().t())
            s = torch.sigmoid(g)
            to_g, to_u = up * s * (1 + g * (1 - s)), g * s
            d = torch.cat([dh * to_g, dh * to_u], 1)
            rough = torch.cat([up.abs() * s * (1 + g.abs()), g.abs() * s], 1) * (1 + torch.cat([g, g], 1).abs())
            e_d = torch.cat([e_dh * to_g.abs(), e_dh * to_u.abs()], 1) + FAST * rough * torch.cat([dh, dh], 1).abs()
            e_d = e_d + u * d.abs() + TINY
            dx = d @ w13.t()
            e_dx = e_d @ w13.abs().t() + 2 * f * ACC * (d.abs() @ w13.abs().t()) + u * dx.abs() + TINY
            dw13 = x.t() @ d
            e_dw13 = x.abs().t() @ e_d + n * ACC * (x.abs().t() @ d.abs()) + u * dw13.abs() + TINY
            dw2 = hh.t() @ dy
            e_dw2 = n * ACC * (hh.abs().t() @ dy.abs()) + u * dw2.abs() + TINY
            out["dx"].append((dx, 1.01 * e_dx))
            out["dgate_up"].append((d, 1.01 * e_d))
            stacks["dw13"].append((dw13, 1.01 * e_dw13))
            stacks["dw2"].append((dw2, 1.01 * e_dw2))
        res = {k: tuple(torch.cat(p) for p in zip(*v)) for k, v in out.items()}
        res.update({k: tuple(torch.stack(p) for p in zip(*v)) for k, v in stacks.items()})
        return res


def within(got, expected, name):
    value, bound = expected
    got = got.double()
    if got.ndim == 2 and value.ndim == 3:
        got = got[None]
    assert got.shape == value.shape, name
    if not value.numel():
        return
    assert bool(torch.isfinite(got).all()), f"{name}: not finite"
    worst = ((got - value).abs() / bound.clamp_min(1e-300)).max().item()
    assert worst <= 1.0, f"{name}: {worst:.3f} times its bound"


def saved_of(block):
    """h and gate_up as a forward pass leaves them (the formulas, rounded once; NaN behind the last segment)."""
    ref = block.forward()
    full = {}
    for name, cols in (("h", block.ffn), ("gate_up", 2 * block.ffn)):
        t = torch.full((block.rows, cols), float("nan"), device="cuda", dtype=block.dtype)
        t[:block.used] = ref[name][0].to(block.dtype)
        full[name] = t
    return full["h"], full["gate_up"]


SHAPES = [
    ([1], 8, 8),
    ([1], 1024, 704),
    ([16], 64, 64),
    ([129], 136, 72),
    ([0], 128, 64),
    ([3, 0, 1, 64, 65], 264, 200),
    ([0, 127, 0, 129, 257], 200, 136),
    ([31] * 40, 72, 40),
    ([17], 1160, 2048),  # long contractions of few tiles, shared by a cluster's CTAs
    ([300, 0, 44], 4784, 184),
    ([5, 0, 9], 824, 1600),
    ([3, 0, 70, 1] * 55, 136, 72),  # tile lists in global memory
    ([700, 1, 0, 333], 4104, 2056),  # pairs' 256 x 256 tiles
    ([0, 2, 256, 0, 255, 257], 2048, 1032),
    ([31, 32, 33, 95, 128, 160, 223, 224, 225, 480, 481], 1048, 520),  # last row blocks of every length
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{sum(s[0])}rows{len(s[0])}e{s[1]}x{s[2]}")
def test_forward(shape, dtype):
    block = Block(*shape, dtype)
    y, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    kernels.check_device_errors()
    ref = block.forward()
    for name, got in (("gate_up", gate_up), ("h", h), ("y", y)):
        within(got, ref[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("shape", SHAPES, ids=lambda s: f"{sum(s[0])}rows{len(s[0])}e{s[1]}x{s[2]}")
def test_backward(shape, dtype):
    block = Block(*shape, dtype, seed=1)
    h, gate_up = saved_of(block)
    dx, dw13, dw2 = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    kernels.check_device_errors()
    ref = block.backward(h, gate_up)
    for name, got in (("dx", dx), ("dw13", dw13), ("dw2", dw2)):
        within(got, ref[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [SHAPES[3], SHAPES[5], SHAPES[8], SHAPES[12]], ids=["small", "ragged", "split", "wide"])
def test_single_product_gradients(shape):
    block = Block(*shape, torch.bfloat16, seed=2)
    h, gate_up = saved_of(block)
    ref = block.backward(h, gate_up)
    dgu = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, block.offs, gate_up=gate_up)
    within(dgu, ref["dgate_up"], "dgate_up")
    dw2 = kernels.launch_grouped_mm_wgrad(h, block.dy, block.offs)
    within(dw2, ref["dw2"], "dw2")
    dh = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, block.offs)
    kernels.check_device_errors()
    for e, rows in segments(block.lengths):
        w2, dy = block.w2[e].double(), block.dy[rows].double()
        value = dy @ w2.t()
        bound = half_step(torch.bfloat16) * value.abs() + block.hidden * ACC * (dy.abs() @ w2.abs().t()) + TINY
        within(dh[rows], (value, bound), f"dh of expert {e}")


@pytest.mark.gpu
def test_gradients_against_differences():
    """Directional derivatives of the kernels' own y by central differences."""
    block = Block([37, 0, 90], 64, 48, torch.float16, seed=3)
    y, h, gate_up = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gate_up, block.offs)
    gen = torch.Generator(device="cuda").manual_seed(9)
    step = 2.0**-5
    for which, grad in enumerate(grads):
        tensors = [block.x, block.w13, block.w2]
        scale = 1.0 if which == 0 else 0.125
        way = (torch.randint(0, 2, tensors[which].shape, device="cuda", generator=gen) * 2 - 1).double() * scale
        sides = []
        for sign in (1, -1):
            moved = list(tensors)
            moved[which] = (tensors[which].double() + sign * step * way).to(torch.float16)
            sides.append((kernels.gated_ffn_forward(*moved, block.offs)[0].double(), moved[which].double()))
        taken = sides[0][1] - sides[1][1]  # the step after rounding to fp16
        change = ((sides[0][0] - sides[1][0]) * block.dy.double()).sum().item()
        told = (grad.double() * taken).sum().item()
        # Roundings of y (half a step each side) and the gradient's, plus the third-order term of the difference.
        noise = (half_step(torch.float16) * 4 * (sides[0][0].abs() * block.dy.double().abs())).square().sum().sqrt().item()
        noise += half_step(torch.float16) * 8 * (grad.double() * taken).square().sum().sqrt().item()
        curve = step * step * (grad.double().square().sum().sqrt() * taken.square().sum().sqrt()).item()
        assert abs(change - told) <= 6 * noise + curve, (which, change, told)


@pytest.mark.gpu
def test_rows_behind_the_last_segment_and_padding_stay():
    block = Block([5, 130], 136, 72, torch.bfloat16, seed=4, tail=9, pad=8)
    mark = 7.25

    def out(rows, cols):
        return torch.full((rows, cols + 16), mark, device="cuda", dtype=torch.bfloat16)[:, :cols]

    y, h, gu, dx = (out(block.rows, c) for c in (136, 72, 144, 136))
    kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs, out=y, h=h, gate_up=gu)
    ref = block.forward()
    for name, got in (("y", y), ("h", h), ("gate_up", gu)):
        within(got[:block.used], ref[name], name)
    hs, gus = saved_of(block)
    dw13 = torch.full((2, 136, 160), mark, device="cuda", dtype=torch.bfloat16)[:, :, :144]
    _, _, dw2 = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, hs, gus, block.offs, dx=dx, dw13=dw13)
    kernels.check_device_errors()
    ref = block.backward(hs, gus)
    within(dx[:block.used], ref["dx"], "dx")
    within(dw13, ref["dw13"], "dw13")
    within(dw2, ref["dw2"], "dw2")
    for t in (y, h, gu, dx, dw13):
        whole = t._base if t._base is not None else t
        assert bool((whole[..., t.shape[-1]:] == mark).all()), "padding written"
    for t in (y, h, gu, dx):
        assert bool((t[block.used:] == mark).all()), "rows behind the last segment written"


@pytest.mark.gpu
def test_one_experts_nan_stays_its_own():
    block = Block([65, 63, 70], 128, 64, torch.bfloat16, seed=5)
    h, gu = saved_of(block)
    clean = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gu, block.offs)
    x, dy, bad_h = block.x.clone(), block.dy.clone(), h.clone()
    for t in (x, dy, bad_h):
        t[65:128] = float("nan")
    dirty = kernels.gated_ffn_backward(dy, x, block.w13, block.w2, bad_h, gu, block.offs)
    kernels.check_device_errors()
    assert torch.equal(clean[0][:65], dirty[0][:65]) and torch.equal(clean[0][128:], dirty[0][128:])
    for a, b in zip(clean[1:], dirty[1:]):
        assert torch.equal(a[[0, 2]], b[[0, 2]])
        assert bool(torch.isnan(b[1]).any())


@pytest.mark.gpu
@pytest.mark.parametrize("gate", [-60000.0, -104.0, -30.0, 30.0, 104.0, 60000.0])
def test_saturated_gates(gate):
    """sigmoid is 0 or 1 to fp32: finite gradients, the formula's limits."""
    rows, f = 40, 64
    block = Block([rows], 64, f, torch.bfloat16, seed=6, dense=True)
    gu = torch.empty((rows, 2 * f), device="cuda", dtype=torch.bfloat16)
    gu[:, :f], gu[:, f:] = gate, 2.0
    h = (gu[:, :f].double() * torch.sigmoid(gu[:, :f].double()) * 2).to(torch.bfloat16)
    out = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, gate_up=gu)
    within(out, block.backward(h, gu)["dgate_up"], "dgate_up")


@pytest.mark.gpu
def test_dense_forms_and_no_rows():
    block = Block([77], 64, 40, torch.float16, seed=7, dense=True)
    y, h, gu = kernels.gated_ffn_forward(block.x, block.w13, block.w2)
    ref = block.forward()
    within(y, ref["y"], "y")
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gu)
    assert [g.shape for g in grads] == [block.x.shape, block.w13.shape, block.w2.shape]
    none = Block([0, 0], 64, 40, torch.float16, seed=8)
    y, h, gu = kernels.gated_ffn_forward(none.x, none.w13, none.w2, none.offs)
    assert y.shape == (0, 64) and h.shape == (0, 40) and gu.shape == (0, 80)
    dx, dw13, dw2 = kernels.gated_ffn_backward(none.dy, none.x, none.w13, none.w2, h, gu, none.offs)
    kernels.check_device_errors()
    assert dx.shape == (0, 64) and not dw13.any() and not dw2.any()


@pytest.mark.gpu
def test_row_ends_out_of_range_are_clamped_and_reported():
    block = Block([20, 30], 64, 40, torch.bfloat16, seed=10)
    ref = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)[0]
    kernels.check_device_errors()
    ends = torch.tensor([20, 51], dtype=torch.int32, device="cuda")  # one past the rows
    got = kernels.gated_ffn_forward(block.x, block.w13, block.w2, ends)[0]
    with pytest.raises(RuntimeError, match="invalid dimensions"):
        kernels.check_device_errors()
    assert torch.equal(ref, got)
    kernels.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,hidden,ffn", [([5, 2, 9], 136, 72), ([700, 333, 48], 1160, 1032)], ids=["small", "pairs"])
def test_malformed_row_ends_stay_inside_and_are_reported(lengths, hidden, ffn):
    block = Block(lengths, hidden, ffn, torch.bfloat16, seed=13, tail=3)
    rows, mark = block.rows, 3.25

    def out(cols):
        return torch.full((rows + 300, cols), mark, device="cuda", dtype=torch.bfloat16)

    outs = y, h, gu, dx = out(hidden), out(ffn), out(2 * ffn), out(hidden)

    def run():
        kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs, out=y[:rows], h=h[:rows], gate_up=gu[:rows])
        return kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h[:rows], gu[:rows], block.offs,
                                          dx=dx[:rows])

    good = block.offs.clone()
    for ends in ([-7, rows // 2, rows], [rows, 3, rows - 1], [0, rows + 100, 2**31 - 1], [-2**31, 2**31 - 1, -1]):
        block.offs.copy_(torch.tensor(ends, dtype=torch.int32))
        run()
        with pytest.raises(RuntimeError, match="invalid dimensions"):
            kernels.check_device_errors()
        assert all(bool((t[rows:] == mark).all()) for t in outs)
    for t in outs:
        t.fill_(mark)
    block.offs.zero_()  # every row behind the last segment
    _, dw13, dw2 = run()
    assert all(bool((t == mark).all()) for t in outs) and not dw13.any() and not dw2.any()
    block.offs.copy_(good)
    run()
    kernels.check_device_errors()
    within(y[:block.used], block.forward()["y"], "y")


@pytest.mark.gpu
def test_repeats_bit_for_bit_and_on_another_stream():
    block = Block([200, 0, 313], 512, 264, torch.bfloat16, seed=11)
    y, h, gu = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gu, block.offs)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    again = []
    for stream in streams:  # two calls in flight at once
        with torch.cuda.stream(stream):
            a = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
            again.append((a, kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, a[1], a[2], block.offs)))
    torch.cuda.synchronize()
    kernels.check_device_errors()
    for forward, backward in again:
        assert all(torch.equal(p, q) for p, q in zip(forward, (y, h, gu)))
        assert all(torch.equal(p, q) for p, q in zip(backward, grads))


@pytest.mark.gpu
def test_training_step_captured_in_a_graph():
    """A step (forward, backward) captured once and replayed after re-routing."""
    block = Block([100, 28, 72], 128, 96, torch.bfloat16, seed=12)
    kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same step: no shared workspace
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y, h, gu = kernels.gated_ffn_forward(block.x, block.w13, block.w2, block.offs)
            grads = kernels.gated_ffn_backward(block.dy, block.x, block.w13, block.w2, h, gu, block.offs)
        graphs.append((graph, y, h, gu, grads))
    for lengths in ([100, 28, 72], [0, 200, 0], [1, 63, 136]):
        block.lengths = lengths
        block.offs.copy_(torch.tensor(lengths, dtype=torch.int32).cumsum(0).to(torch.int32))
        for graph, *_ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        kernels.check_device_errors()
        for _, y, h, gu, grads in graphs:
            within(y, block.forward()["y"], "y")
            ref = block.backward(h, gu)
            for name, got in zip(("dx", "dw13", "dw2"), grads):
                within(got, ref[name], name)


@pytest.mark.gpu
def test_refusals():
    block = Block([20, 30], 64, 40, torch.bfloat16, seed=13)
    x, w13, w2, offs = block.x, block.w13, block.w2, block.offs
    forward = kernels.gated_ffn_forward
    bad = [
        (lambda: forward(x.float(), w13.float(), w2.float(), offs), "float16 or bfloat16"),
        (lambda: forward(x.cpu(), w13, w2, offs), "CUDA"),
        (lambda: forward(x, w13.half(), w2, offs), "w13 must be"),
        (lambda: forward(x, w13[:, :, :72], w2, offs), "w13 must be"),
        (lambda: forward(x, w13, w2, offs.long()), "int32"),
        (lambda: forward(x, w13, w2, offs[:1]), "offs"),
        (lambda: forward(x, w13, w2), "offs"),
        (lambda: forward(x[:, :60], w13[:, :60], w2[:, :, :60], offs), "multiples of 8"),
        (lambda: forward(x.t().contiguous().t(), w13, w2, offs), "contiguous columns"),
        (lambda: forward(torch.empty(51 * 64 + 1, device="cuda", dtype=torch.bfloat16)[1:3201].view(50, 64), w13, w2,
                         offs), "aligned"),
        (lambda: forward(x, w13, w2, offs, out=torch.empty(50, 72, device="cuda", dtype=torch.bfloat16)), "out must"),
        (lambda: kernels.gated_ffn_backward(x[:49], x, w13, w2, x, x, offs), "dy must"),
        (lambda: kernels.launch_grouped_mm_dgrad(x, w13, offs), "dc must"),
        (lambda: kernels.launch_grouped_mm_wgrad(x, x[:7], offs), "dc must"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    kernels.check_device_errors()


def test_abi_refuses_bad_arguments_before_any_launch():
    """Checked on the host: every call returns an error without touching a device."""
    lib = _native.load()
    buf = ctypes.create_string_buffer(4096 + 16)
    at = (ctypes.addressof(buf) + 15) // 16 * 16

    def args(**changes):
        f = _native.FfnArgs(1, 2, 10, 64, 40, at)
        for name, pitch in (("x", 64), ("y", 64), ("dx", 64), ("h", 40), ("gate_up", 80), ("dgate_up", 80)):
            setattr(f, name, at)
            setattr(f, name + "_pitch", pitch)
        for name, pitch, stride in (("w13", 80, 64 * 80), ("w2", 64, 40 * 64), ("dw13", 80, 64 * 80),
                                    ("dw2", 64, 40 * 64)):
            setattr(f, name, at)
            setattr(f, name + "_pitch", pitch)
            setattr(f, name + "_stride", stride)
        for name, value in changes.items():
            setattr(f, name, value)
        return f

    bad = [dict(dtype=2), dict(experts=0), dict(rows=-1), dict(hidden=60), dict(ffn=0), dict(offs=None), dict(x=at + 2),
           dict(x=None), dict(x_pitch=60), dict(x_pitch=68), dict(w13=None), dict(w13_stride=64 * 80 - 8), dict(w13_stride=64 * 80 + 8), dict(rows=(1 << 31) - 1023),
           dict(w2_pitch=56), dict(rows=1 << 31), dict(h=None), dict(gate_up_pitch=40)]
    for change in bad:
        for entry in (lib.gated_ffn_forward_launch, lib.gated_ffn_backward_launch):
            assert entry(ctypes.byref(args(**change))) == _native.STATUS_INVALID, change
    for entry in (lib.gated_ffn_forward_launch, lib.gated_ffn_backward_launch):
        assert entry(None) == _native.STATUS_INVALID
        assert entry(ctypes.byref(args(experts=200))) == _native.STATUS_SCRATCH  # its tile lists are kept there
        assert entry(ctypes.byref(args(experts=200, scratch=at, scratch_bytes=1664))) == _native.STATUS_SCRATCH
    # Two operand maps per gradient and expert; tile lists from 200 (three jobs: 100) experts.
    calls = _native.FFN_FORWARD, _native.FFN_BACKWARD, _native.FFN_DGRAD, _native.FFN_WGRAD
    assert [_native.ffn_scratch_bytes(0, c) for c in calls] == [0] * 4
    assert [_native.ffn_scratch_bytes(4, c) for c in calls] == [0, 4 * 4 * 128, 0, 4 * 2 * 128]
    assert [_native.ffn_scratch_bytes(100, c) for c in calls] == [0, 100 * 4 * 128 + 1280, 0, 100 * 2 * 128]
    assert [_native.ffn_scratch_bytes(200, c) for c in calls] == [1792, 200 * 4 * 128 + 896 + 2432, 896, 200 * 2 * 128 + 896]

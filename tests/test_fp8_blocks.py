"""The e8m0 block-scaled e4m3 product and its quantisation against 64 bits.

Quantised values are exact: a power-of-two scale divides without rounding, so
q is the e4m3 value nearest to x / s and equality is required.  Products: the
e4m3 x e4m3 terms and their power-of-two scales are exact, so the bound is the
fp32 accumulation, at most K 2^-23 sum |a| |b| (every add off by at most one
unit in the last place), plus the bf16 rounding of the result, eps / 2.
"""

from __future__ import annotations

import ctypes

import pytest

from kernels import _native

torch = pytest.importorskip("torch")
import kernels  # noqa: E402

BLOCK = 128
HALF = 2.0**-8  # half a bf16 step


def scale_of(top):
    """(2^e, e + 127) with the smallest e such that top <= 448 2^e; 1 for zero."""
    e = torch.floor(torch.log2(top.clamp_min(2.0**-140) / 448.0)) + 1  # log2 rounds: only a start,
    for _ in range(2):  # the powers themselves are compared
        e = torch.where(top <= 448.0 * torch.exp2(e - 1), e - 1, e)
    e = e.clamp(-127, 127)
    e = torch.where(top == 0, torch.zeros_like(e), e)
    return torch.exp2(e), e + 127


def quantize_reference(x, block_rows):
    """(q, exponent byte) in 64 bits; non-finite elements become NaN and do not count for the scale."""
    x = x.double()
    m, k = x.shape
    mb, kb = -(-m // block_rows), -(-k // BLOCK)
    full = torch.zeros((mb * block_rows, kb * BLOCK), dtype=torch.float64, device=x.device)
    full[:m, :k] = x
    parts = full.view(mb, block_rows, kb, BLOCK)
    finite = torch.where(torch.isfinite(parts), parts.abs(), 0.0)
    scale, byte = scale_of(finite.amax(dim=(1, 3)))
    v = (parts / scale[:, None, :, None]).reshape(full.shape)[:m, :k]
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3)
    q = torch.round(v / step) * step
    return torch.where(torch.isfinite(x), q, float("nan")), byte


def check_quantized(got, x, block_rows):
    q, scale = got
    expected, byte = quantize_reference(x, block_rows)
    assert torch.equal(scale.view(torch.uint8).double(), byte)
    assert torch.equal(q.float().double().nan_to_num(nan=1e9), expected.nan_to_num(nan=1e9))


def hard_values(m, k, dtype, seed):
    """Normal values over many magnitudes per block, with blocks of zeros, of one
    value at a scale's border (448 2^e and the next value up) and of tiny values."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, k), device="cuda", generator=gen)
    x = x * torch.exp2(torch.randint(-12, 13, (m, 1), device="cuda", generator=gen).float())
    x = x.to(dtype)
    if m > 2:
        x[0] = 0
        x[1] = 0
        x[1, ::BLOCK] = 448.0
        x[2, :] = torch.finfo(dtype).tiny
        x[2, ::BLOCK] = 450.0  # bf16: 448 and 450 are neighbours
    return x


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 1), (1, 128), (3, 200), (5, 7168), (129, 264), (40, 1001), (2048, 1536)])
def test_quantize_rows(m, k, dtype):
    x = hard_values(m, k, dtype, m + k)
    check_quantized(kernels.launch_quantize_rows(x), x, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,k", [(1, 1), (128, 128), (3, 200), (129, 264), (130, 1001), (1536, 2048)])
def test_quantize_blocks(n, k, dtype):
    x = hard_values(n, k, dtype, n + k)
    check_quantized(kernels.launch_quantize_blocks(x), x, BLOCK)


@pytest.mark.gpu
def test_quantize_every_e4m3_border():
    """All bf16 values up to 448 in one block each: every rounding border and tie."""
    bits = torch.arange(0, 1 << 16, dtype=torch.int32).to(torch.int16).view(torch.bfloat16).cuda()
    values = bits[torch.isfinite(bits) & (bits.abs() <= 448)]
    rows = -(-values.numel() // 127)
    x = torch.zeros((rows, BLOCK), dtype=torch.bfloat16, device="cuda")
    flat = torch.zeros(rows * 127, dtype=torch.bfloat16, device="cuda")
    flat[:values.numel()] = values
    x[:, 1:] = flat.view(rows, 127)
    x[:, 0] = 448.0  # scale 1 in every block
    q, scale = kernels.launch_quantize_rows(x)
    assert bool((scale.view(torch.uint8) == 127).all())
    check_quantized((q, scale), x, 1)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [True, False])
def test_quantize_infinities_and_extremes(rows):
    x = torch.randn((130, 300), device="cuda")
    x[0, 5], x[0, 6], x[0, 140], x[129, 299] = float("inf"), float("-inf"), float("nan"), float("nan")
    x[3, :128] = float("inf")  # nothing finite: scale 1, all NaN
    x[4, 128:256] = torch.finfo(torch.float32).max
    x[5, 128:256] = 1e-44  # subnormal: the smallest scale
    if not rows:
        x[3:6] = x[6:9]
    got = (kernels.launch_quantize_rows if rows else kernels.launch_quantize_blocks)(x)
    check_quantized(got, x, 1 if rows else BLOCK)


@pytest.mark.gpu
def test_quantize_strides_batches_and_given_outputs():
    base = torch.randn((3, 140, 520), device="cuda").to(torch.bfloat16)
    for view in (base[1, :, :264], base[1, :, 3:267], base[1, ::2, 8:408]):  # padded, misaligned, every other row
        check_quantized(kernels.launch_quantize_rows(view), view, 1)
        check_quantized(kernels.launch_quantize_blocks(view), view, BLOCK)
    w = base[:, :136, 8:264]
    q = torch.empty((3, 136, 256), dtype=torch.float8_e4m3fn, device="cuda")
    s = torch.empty((3, 2, 2), dtype=torch.float8_e8m0fnu, device="cuda")
    out = kernels.launch_quantize_blocks(w, q, s)
    assert out[0] is q and out[1] is s
    for e in range(3):
        check_quantized((q[e], s[e]), w[e], BLOCK)
    none, scales = kernels.launch_quantize_rows(base[0, :0])
    assert none.shape == (0, 520) and scales.shape == (0, 5)


class Product:
    def __init__(self, lengths, n, k, seed=0, tail=0, pad=0, spread=6, dense=False):
        gen = torch.Generator(device="cuda").manual_seed(seed)
        self.lengths, self.rows, self.used = lengths, sum(lengths) + tail, sum(lengths)
        experts = len(lengths)

        def e4m3(*shape):
            wide = torch.randn((*shape[:-1], shape[-1] + pad), device="cuda", generator=gen)
            return (wide * 60).clamp(-448, 448).to(torch.float8_e4m3fn)[..., :shape[-1]]

        def e8m0(*shape):
            return torch.randint(127 - spread, 128 + spread, shape, device="cuda", generator=gen).to(
                torch.uint8).view(torch.float8_e8m0fnu)

        kb = -(-k // BLOCK)
        self.a, self.sa = e4m3(self.rows, k), e8m0(self.rows, kb)
        self.b, self.sb = e4m3(experts, n, k), e8m0(experts, -(-n // BLOCK), kb)
        self.offs = torch.tensor(lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
        if tail:
            self.sa.view(torch.uint8)[self.used:] = 255  # NaN behind the last segment
        if dense:
            self.b, self.sb, self.offs = self.b[0], self.sb[0], None
        self.n, self.k = n, k

    def run(self, **kw):
        return kernels.launch_block_scaled_mm(self.a, self.sa, self.b, self.sb, self.offs, **kw)

    def check(self, out):
        cols = torch.arange(self.k, device="cuda") // BLOCK
        rows = torch.arange(self.n, device="cuda") // BLOCK
        wide_a = self.a.double() * torch.exp2(self.sa.view(torch.uint8).double() - 127)[:, cols]
        at = 0
        for e, m in enumerate(self.lengths):
            if m == 0:
                continue
            b, sb = (self.b, self.sb) if self.b.ndim == 2 else (self.b[e], self.sb[e])
            w = b.double() * torch.exp2(sb.view(torch.uint8).double() - 127)[rows][:, cols]
            a = wide_a[at:at + m]
            value = a @ w.t()
            bound = 1.01 * (HALF * value.abs() + self.k * 2.0**-23 * (a.abs() @ w.abs().t()))
            got = out[at:at + m].double()
            assert bool(torch.isfinite(got).all())
            worst = ((got - value).abs() / bound.clamp_min(1e-300)).max().item()
            assert worst <= 1.0, f"expert {e}: {worst:.3f} times its bound"
            at += m


PRODUCTS = [
    # few tokens per expert
    ([1], 8, 16), ([1], 4096, 7168), ([3], 136, 2064), ([8], 264, 128), ([9], 24, 400), ([16], 128, 1024),
    ([32], 40, 656), ([1, 0, 7, 0, 23], 136, 528), ([0, 0, 20, 1], 200, 272), ([2] * 37, 72, 144),
    # one CTA's 128 x 128 tiles
    ([33], 128, 128), ([127], 136, 272), ([100, 0, 1, 129], 264, 656), ([300], 1032, 2000), ([64] * 5, 128, 512),
    # 64 x 128 tiles; a tile's K shared by the CTAs of a cluster
    ([50] * 3, 136, 1040), ([33], 264, 2064), ([100], 264, 4112), ([40, 0, 50], 136, 2064), ([128], 1024, 7168),
    ([17, 3, 40], 136, 4112), ([20], 264, 2064), ([65, 0, 2, 0, 9], 1032, 1168), ([5, 70, 45], 520, 1104), ([0, 200, 10], 136, 16384), ([64], 8, 2320),
    ([40, 0, 1, 63] * 60, 72, 144), ([0, 300, 0, 9] * 50, 1032, 272),  # tile lists in global memory
    # CTA pairs' tiles of up to 224 rows x 256
    ([2048], 4096, 512), ([1, 0, 1500, 255, 257], 4096, 1168), ([1999], 2248, 1040),
    ([63, 64, 65, 128, 129, 192, 193, 224, 225, 447], 4096, 144),
]


@pytest.mark.gpu
@pytest.mark.parametrize("shape", PRODUCTS, ids=lambda s: f"{sum(s[0])}rows{len(s[0])}e{s[1]}x{s[2]}")
def test_product(shape):
    product = Product(*shape)
    out = product.run()
    kernels.check_device_errors()
    product.check(out)


@pytest.mark.gpu
def test_every_kernel_was_reached():
    paths = set()
    for shape in (PRODUCTS[0], PRODUCTS[10], PRODUCTS[-3]):
        Product(*shape).run()
        paths.add(kernels.last_block_scaled_info()["path"])
    assert paths == {"warp_mma", "tcgen05_tma", "tcgen05_tma_pair"}


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [PRODUCTS[1], PRODUCTS[13], PRODUCTS[17], PRODUCTS[-1]], ids=["few", "one", "split", "pair"])
def test_one_scale_at_a_time(shape):
    """One scale byte differs from 1: only its row and K block may change."""
    product = Product(*shape, dense=True)
    product.sa.view(torch.uint8).fill_(127)
    product.sb.view(torch.uint8).fill_(127)
    kb = product.sa.shape[1]
    for row, block, n_block in ((0, 0, 0), (product.rows - 1, kb - 1, product.sb.shape[0] - 1), (product.rows // 2, 1, 0)):
        product.sa.view(torch.uint8)[row, block] = 130
        product.sb.view(torch.uint8)[n_block, min(block + 1, kb - 1)] = 121
        product.check(product.run())
    kernels.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [([5, 2], 136, 272), ([100, 130], 136, 272), ([1500, 900], 4096, 272)],
                         ids=["few", "one", "pair"])
def test_product_rows_behind_and_padding_stay(shape):
    product = Product(*shape, tail=6, pad=16)
    wide = torch.full((product.rows, product.n + 24), 3.25, device="cuda", dtype=torch.bfloat16)
    out = wide[:, :product.n]
    assert product.run(out=out) is out
    kernels.check_device_errors()
    product.check(out)
    assert bool((wide[:, product.n:] == 3.25).all()) and bool((wide[product.used:] == 3.25).all())


@pytest.mark.gpu
@pytest.mark.parametrize("lengths,n", [([5, 2, 9], 136), ([100, 130, 20], 136), ([1500, 900, 48], 4096)],
                         ids=["few", "one", "pair"])
def test_malformed_row_ends_stay_inside_and_are_reported(lengths, n):
    product = Product(lengths, n, 272, tail=3)
    wide = torch.full((product.rows + 300, n), 3.25, device="cuda", dtype=torch.bfloat16)
    out, good, rows = wide[:product.rows], product.offs.clone(), product.rows
    for ends in ([-7, rows // 2, rows], [rows, 3, rows - 1], [0, rows + 100, 2**31 - 1], [-2**31, 2**31 - 1, -1]):
        product.offs.copy_(torch.tensor(ends, dtype=torch.int32))
        product.run(out=out)
        with pytest.raises(RuntimeError, match="invalid dimensions"):
            kernels.check_device_errors()
        assert bool((wide[rows:] == 3.25).all())
    wide.fill_(3.25)
    product.offs.zero_()  # every row behind the last segment
    product.run(out=out)
    assert bool((wide == 3.25).all())
    product.offs.copy_(good)
    product.check(product.run(out=out))
    kernels.check_device_errors()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [([5], 136, 528), ([100], 136, 528), ([2048], 4096, 528)], ids=["few", "one", "pair"])
def test_extreme_scales_and_nan(shape):
    product = Product(*shape, dense=True)
    sa, sb = product.sa.view(torch.uint8), product.sb.view(torch.uint8)
    sa.fill_(127 + 100)
    sb.fill_(127 - 100)
    product.check(product.run())
    sa[1, 0] = 255  # a NaN scale: its row is NaN, the others are untouched
    out = product.run()
    kernels.check_device_errors()
    assert bool(torch.isnan(out[1]).all())
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isfinite(out[2:]).all())


@pytest.mark.gpu
@pytest.mark.parametrize("token,weight", [(0, 254), (254, 0), (1, 250), (253, 3), (200, 50), (10, 130)])
@pytest.mark.parametrize("shape", [([5], 136, 528), ([100], 136, 528), ([2048], 4096, 528)], ids=["few", "one", "pair"])
def test_scales_whose_product_alone_is_in_range(shape, token, weight):
    product = Product(*shape, dense=True)
    product.sa.view(torch.uint8).fill_(token)
    product.sb.view(torch.uint8).fill_(weight)
    product.check(product.run())
    kernels.check_device_errors()


@pytest.mark.gpu
def test_quantised_layer_end_to_end():
    """Weights quantised once, tokens on every call, expert-sorted: within the
    quantisation's own bound (half a step of each operand, 2^-4 relative, or of
    a block's largest value's subnormals) of the unquantised product."""
    gen = torch.Generator(device="cuda").manual_seed(3)
    lengths = [70, 0, 130, 1]
    offs = torch.tensor(lengths, dtype=torch.int32).cumsum(0).to(torch.int32).cuda()
    x = torch.randn((201, 512), device="cuda", generator=gen).to(torch.bfloat16)
    w = (torch.randn((4, 264, 512), device="cuda", generator=gen) / 22).to(torch.bfloat16)
    b, sb = kernels.launch_quantize_blocks(w)
    a, sa = kernels.launch_quantize_rows(x)
    out = kernels.launch_block_scaled_mm(a, sa, b, sb, offs)
    kernels.check_device_errors()
    at = 0
    for e, m in enumerate(lengths):
        if m == 0:
            continue
        xe, we = x[at:at + m].double(), w[e].double()
        # An element is off by 2^-4 of itself, or 2^-10 of its scale (2^-8 of 448) where it is subnormal.
        dx = xe.abs() * 2.0**-4 + xe.abs().amax() * 2.0**-17
        dw = we.abs() * 2.0**-4 + we.abs().amax() * 2.0**-17
        bound = dx @ we.abs().t() + xe.abs() @ dw.t() + dx @ dw.t()
        value = xe @ we.t()
        bound = bound + HALF * (value.abs() + bound) + 512 * 2.0**-23 * (xe.abs() + dx) @ (we.abs() + dw).t()
        assert bool(((out[at:at + m].double() - value).abs() <= bound).all())
        at += m


@pytest.mark.gpu
def test_streams_and_graph():
    products = [Product(*s, seed=5) for s in (([3, 9], 264, 528), ([200, 56], 264, 528), ([1500, 600], 4096, 528))]
    expected = [p.run() for p in products]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = [p.run() for p in products]
    streams = [torch.cuda.Stream() for _ in range(2)]
    outs = []
    for stream in streams:
        with torch.cuda.stream(stream):
            outs.append([p.run() for p in products])
    torch.cuda.synchronize()
    graph.replay()
    torch.cuda.synchronize()
    kernels.check_device_errors()
    for got in (*outs, captured):
        assert all(torch.equal(p, q) for p, q in zip(got, expected))
    for p in products:  # re-routed between replays
        p.lengths = [p.used, 0]
        p.offs.fill_(p.used)
    graph.replay()
    torch.cuda.synchronize()
    for p, got in zip(products, captured):
        p.check(got)


@pytest.mark.gpu
def test_refusals():
    p = Product([40, 30], 136, 272)
    mm = kernels.launch_block_scaled_mm
    bad = [
        (lambda: mm(p.a.float(), p.sa, p.b, p.sb, p.offs), "float8_e4m3fn"),
        (lambda: mm(p.a, p.sa.float(), p.b, p.sb, p.offs), "float8_e8m0fnu"),
        (lambda: mm(p.a, p.sa, p.b, p.sb), "offs"),
        (lambda: mm(p.a, p.sa, p.b, p.sb, p.offs.long()), "int32"),
        (lambda: mm(p.a, p.sa[:, :2], p.b, p.sb, p.offs), "scale shapes"),
        (lambda: mm(p.a, p.sa, p.b[:, :132], p.sb, p.offs), "multiple"),
        (lambda: mm(p.a[:, :264], p.sa, p.b[:, :, :264], p.sb, p.offs), "multiple"),
        (lambda: mm(p.a.cpu(), p.sa, p.b, p.sb, p.offs), "same CUDA device"),
        (lambda: mm(p.a, p.sa, p.b, p.sb, p.offs, out=torch.empty(70, 136, device="cuda")), "bfloat16"),
        (lambda: mm(p.a.view(torch.uint8)[:, 1:257].view(torch.float8_e4m3fn), p.sa[:, :2].contiguous(),
                    p.b[:, :, :256], p.sb[:, :, :2].contiguous(), p.offs), "aligned"),
        (lambda: kernels.launch_quantize_rows(torch.zeros(4, 4, device="cuda", dtype=torch.float64)), "unsupported dtype"),
        (lambda: kernels.launch_quantize_rows(torch.zeros(4, 4)), "CUDA"),
        (lambda: kernels.launch_quantize_rows(torch.zeros(4, 9, device="cuda").t()), "contiguous columns"),
        (lambda: kernels.launch_quantize_blocks(torch.zeros(4, device="cuda")), "expected w"),
        (lambda: kernels.launch_quantize_rows(torch.zeros(4, 8, device="cuda"),
                                              scale=torch.zeros(4, 1, device="cuda")), "scale must"),
    ]
    for call, message in bad:
        with pytest.raises(ValueError, match=message):
            call()
    kernels.check_device_errors()


def test_abi_refuses_bad_arguments_before_any_launch():
    lib = _native.load()
    buf = ctypes.create_string_buffer(4096 + 128)
    at = (ctypes.addressof(buf) + 127) // 128 * 128

    def product(**change):
        args = dict(a=at, a_pitch=64, sa=at, b=at, b_pitch=64, b_stride=64 * 40, sb=at, c=at, c_pitch=40, offs=at,
                    experts=2, rows=10, n=40, k=64, scratch=at, scratch_bytes=1 << 12, stream=None, info=None)
        args.update(change)
        return lib.block_scaled_mm_launch(*args.values())

    bad = [dict(experts=0), dict(rows=-1), dict(n=36), dict(k=56), dict(offs=None), dict(a=None), dict(a=at + 8),
           dict(sa=None), dict(b=None), dict(a_pitch=72), dict(b_pitch=48), dict(b_stride=64), dict(c_pitch=44),
           dict(rows=1 << 31)]
    for change in bad:
        assert product(**change) == _native.STATUS_INVALID, change
    for change in (dict(scratch=None), dict(scratch=at + 16), dict(scratch_bytes=64)):
        change["experts"] = 200  # their tile list is kept in scratch
        assert product(**change) == _native.STATUS_SCRATCH, change
    assert [lib.block_scaled_mm_scratch_bytes(e) for e in (0, 1, 199, 200)] == [0, 0, 0, 896]
    for change in ((None, 4, 8, 8, 1, at, 8, at, None), (at, 4, 0, 8, 1, at, 8, at, None),
                   (at, 4, 8, 7, 1, at, 8, at, None), (at, 4, 8, 8, 5, at, 8, at, None), (at + 1, 4, 8, 8, 1, at, 8, at, None)):
        assert lib.quantize_rows_launch(*change) == _native.STATUS_INVALID, change
    for change in ((None, 1, 4, 8, 8, 32, 1, at, at, None), (at, 1, 0, 8, 8, 32, 1, at, at, None),
                   (at, 1, 4, 8, 7, 32, 1, at, at, None), (at, 1, 4, 8, 8, 32, 9, at, at, None)):
        assert lib.quantize_blocks_launch(*change) == _native.STATUS_INVALID, change

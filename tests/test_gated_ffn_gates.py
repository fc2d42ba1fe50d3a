"""Far gates: sigmoid close to 0 or 1 while its product with the other factors is an ordinary number."""

from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import kernels  # noqa: E402
from tests.test_gated_ffn import ACC, FAST, TINY, Block, half_step, within  # noqa: E402


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(40, 512), (700, 448)], ids=["split", "tiles"])
@pytest.mark.parametrize("gate,scale", [(-87.0, 1e30), (-88.0, 1e30), (-88.5, 1e30), (-92.0, 1e33), (88.0, 1.0),
                                        (-20.0, 1e6)])
def test_gradients_where_sigmoid_is_tiny(gate, scale, rows, hidden):
    """sigmoid(-88) is 6e-39: times gradients of 1e30 it is no longer tiny."""
    f = 64
    block = Block([rows], hidden, f, torch.bfloat16, seed=31, dense=True)
    block.dy = (block.dy.double() * scale).to(torch.bfloat16)
    gu = torch.empty((rows, 2 * f), device="cuda", dtype=torch.bfloat16)
    gu[:, :f], gu[:, f:] = gate, 2.0
    h = torch.zeros((rows, f), device="cuda", dtype=torch.bfloat16)
    out = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, gate_up=gu)
    kernels.check_device_errors()
    within(out, block.backward(h, gu)["dgate_up"], "dgate_up")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(40, 512), (700, 448)], ids=["split", "tiles"])
@pytest.mark.parametrize("gate", ["lowest", "highest", -1e30, 1e20])
def test_gradients_of_gates_at_the_types_ends(gate, rows, hidden):
    """A gate of the type's lowest value has gradients of zero, not NaN."""
    f, top = 64, torch.finfo(torch.bfloat16).max
    gate = {"lowest": -top, "highest": top}.get(gate, gate)
    block = Block([rows], hidden, f, torch.bfloat16, seed=32, dense=True)
    if gate > 0:  # du = dh gate is a number only for small dh
        block.dy = (block.dy.double() * 1e-4).to(torch.bfloat16)
    gu = torch.empty((rows, 2 * f), device="cuda", dtype=torch.bfloat16)
    gu[:, :f], gu[:, f:] = gate, 2.0
    h = torch.zeros((rows, f), device="cuda", dtype=torch.bfloat16)
    out = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, gate_up=gu)
    kernels.check_device_errors()
    if gate < 0:
        assert not out.any()
        return
    # sigmoid is 1: dgate = 2 dh, dup = gate dh
    dy, w2 = block.dy.double(), block.w2.double()
    dh = dy @ w2.t()
    e_dh = hidden * ACC * (dy.abs() @ w2.abs().t())
    for got, factor in ((out[:, :f], 2.0), (out[:, f:], float(gu[0, 0]))):
        value = factor * dh
        within(got, (value, 1.01 * (factor * e_dh + (half_step(torch.bfloat16) + 2 * FAST) * value.abs() + TINY)), "gradient")


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(40, 512), (700, 448)], ids=["split", "tiles"])
def test_forward_where_sigmoid_is_tiny(rows, hidden):
    """Column j of the block has gate g_j and up 1e30 (one input column, the others zero): h is -88 sigmoid(-88) 1e30."""
    gates = [-85.0, -87.0, -87.5, -88.0, -88.5, -90.0, -3e38, 88.0]
    f = 8
    x = torch.zeros((rows, hidden), device="cuda", dtype=torch.bfloat16)
    x[:, 0] = 1.0
    w13 = torch.zeros((hidden, 2 * f), device="cuda", dtype=torch.bfloat16)
    w13[0, :f] = torch.tensor(gates, device="cuda")
    w13[0, f:] = 1e30
    w2 = torch.zeros((f, hidden), device="cuda", dtype=torch.bfloat16)
    y, h, gate_up = kernels.gated_ffn_forward(x, w13, w2)
    kernels.check_device_errors()
    assert torch.equal(gate_up, w13[:1].expand(rows, -1))
    g, u = w13[0, :f].double(), w13[0, f:].double()
    value = (g * torch.sigmoid(g) * u).expand(rows, -1)
    # Subnormal sigmoids are held to 2^-149; the product's rounding, the fast functions.
    bound = (half_step(torch.bfloat16) + FAST * (1 + g.abs().clamp_max(1e3))) * value.abs() + 2.0**-149 * (g * u).abs().clamp_max(1e38)
    within(h, (value, 1.01 * bound), "h")
    assert not y.any()


@pytest.mark.gpu
@pytest.mark.parametrize("rows,hidden", [(40, 512), (700, 448)], ids=["split", "tiles"])
@pytest.mark.parametrize("gate", [2.5, -1.25, 0.0, 88.0])
def test_gradients_of_the_largest_up_values(gate, rows, hidden):
    """silu'(2.5) is 1.1: up times it passes fp32's range, times a small dh it does not."""
    f, scale = 64, 1e-38
    block = Block([rows], hidden, f, torch.bfloat16, seed=33, dense=True)
    block.dy = (block.dy.double() * scale * 2.0**20).to(torch.bfloat16)
    block.w2 = (block.w2.double() * 2.0**-10).to(torch.bfloat16)
    gu = torch.empty((rows, 2 * f), device="cuda", dtype=torch.bfloat16)
    gu[:, :f], gu[:, f:] = gate, torch.finfo(torch.bfloat16).max
    gu[::2, f:] *= -1
    h = torch.zeros((rows, f), device="cuda", dtype=torch.bfloat16)
    out = kernels.launch_grouped_mm_dgrad(block.dy, block.w2, gate_up=gu)
    kernels.check_device_errors()
    within(out, block.backward(h, gu)["dgate_up"], "dgate_up")

"""Workloads of the expert feed-forward and FP8 block-product operators.

Three operators, each over the range that a mixture-of-experts program meets:

``ffn_forward`` / ``ffn_backward``
    The gated feed-forward block of every expert over tokens sorted by expert,
    y = (silu(x Wg) * (x Wu)) W2, with what its backward pass reads kept, and
    that backward pass: the gradients of x, W13 = [Wg | Wu] and W2.
``fp8_mm``
    The e4m3 matrix product with a power-of-two scale for each 128-deep block
    of a token's row and for each 128 x 128 block of the weight, alone or with
    the quantisation of the tokens before it (dynamic activation scales).
``fp8_quantize``
    The quantisation itself: rows (activations) or 128 x 128 blocks (weights).

``own = False`` runs the plain forms (elementary torch operations in 32 bits),
``own = True`` the package's entry points on the same state.
"""

import sys
from pathlib import Path

import torch

own = False

PACKAGE_DIR = Path(__file__).resolve().parents[1] / "moe-gemm-parallel-bench_b200"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 128


def _kernels():
    if str(PACKAGE_DIR) not in sys.path:
        sys.path.insert(0, str(PACKAGE_DIR))
    import kernels

    return kernels


# ------------------------------------------------------------------- cases
def listed():
    return [
        # The shared expert of a small layer while a few sequences decode or
        # fine-tune: latency counts.
        {"name": "ffn_forward_16_tokens", "op": "ffn_forward", "dtype": "bf16", "experts": 1, "tokens": 16,
         "hidden": 1024, "ffn": 704, "skew": 0.0},
        # One rank of a 128-expert layer (16 local experts, hidden 4096, ffn
        # 1536) with uneven routing.
        {"name": "ffn_forward_16_experts", "op": "ffn_forward", "dtype": "bf16", "experts": 16, "tokens": 8192,
         "hidden": 4096, "ffn": 1536, "skew": 0.6},
        # One rank of DeepSeek-V3 (32 local experts, hidden 7168, ffn 2048)
        # in a training step of 16384 routed rows: the largest call.
        {"name": "ffn_forward_32_experts", "op": "ffn_forward", "dtype": "bf16", "experts": 32, "tokens": 16384,
         "hidden": 7168, "ffn": 2048, "skew": 0.3},
        # The small layer's backward pass on a few odd tokens.
        {"name": "ffn_backward_51_tokens", "op": "ffn_backward", "dtype": "fp16", "experts": 1, "tokens": 51,
         "hidden": 1024, "ffn": 704, "skew": 0.0},
        # The 16 local experts' backward pass.
        {"name": "ffn_backward_16_experts", "op": "ffn_backward", "dtype": "bf16", "experts": 16, "tokens": 8192,
         "hidden": 4096, "ffn": 1536, "skew": 0.6},
        # A dense block (one expert, every token) with odd token and column
        # counts, fp16.
        {"name": "ffn_backward_dense", "op": "ffn_backward", "dtype": "fp16", "experts": 1, "tokens": 4093,
         "hidden": 4096, "ffn": 4088, "skew": 0.0},
        # The 32 local experts' backward pass of a training step.
        {"name": "ffn_backward_32_experts", "op": "ffn_backward", "dtype": "bf16", "experts": 32, "tokens": 16384,
         "hidden": 7168, "ffn": 2048, "skew": 0.3},
        # Decoding: one token through an FP8 projection, quantised on the way.
        {"name": "fp8_mm_1_token", "op": "fp8_mm", "experts": 1, "tokens": 1, "n": 4096, "k": 7168, "skew": 0.0,
         "quantize": True},
        # A dense FP8 projection over a prompt's tokens.
        {"name": "fp8_mm_8191_tokens", "op": "fp8_mm", "experts": 1, "tokens": 8191, "n": 4096, "k": 7168,
         "skew": 0.0, "quantize": False},
        # 32 local experts' packed gate and up projection over uneven routed
        # rows, quantised on the way.
        {"name": "fp8_mm_32_experts", "op": "fp8_mm", "experts": 32, "tokens": 4096, "n": 4096, "k": 7168,
         "skew": 0.6, "quantize": True},
        # A prompt's activations.
        {"name": "fp8_quantize_rows", "op": "fp8_quantize", "dtype": "bf16", "kind": "rows", "m": 8191, "k": 7168},
        # One expert's packed projection, quantised when a checkpoint loads.
        {"name": "fp8_quantize_blocks", "op": "fp8_quantize", "dtype": "bf16", "kind": "blocks", "m": 4096,
         "k": 7168},
    ]


def _log_int(rng, low, high, step=1):
    import math

    v = math.exp(rng.uniform(math.log(low), math.log(high)))
    return max(low, min(high, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["ffn_forward", "ffn_backward", "fp8_mm", "fp8_quantize"])
    skew = rng.choice([0.0, round(rng.uniform(0.1, 1.0), 2)])
    if op == "fp8_quantize":
        return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "kind": rng.choice(["rows", "blocks"]),
                "m": _log_int(rng, 1, 8192), "k": _log_int(rng, 128, 7168, 8)}
    experts = _log_int(rng, 1, 32)
    if op == "fp8_mm":
        return {"op": op, "experts": experts, "tokens": _log_int(rng, 1, 8192), "n": _log_int(rng, 128, 4096, 8),
                "k": _log_int(rng, 256, 7168, 16), "skew": skew, "quantize": rng.random() < 0.5}
    return {"op": op, "dtype": rng.choice(["bf16", "fp16"]), "experts": experts, "tokens": _log_int(rng, 1, 16384),
            "hidden": _log_int(rng, 256, 7168, 8), "ffn": _log_int(rng, 128, 2048, 8), "skew": skew}


# ------------------------------------------------------------------ inputs
def _lengths(tokens, experts, skew, seed):
    """Rows per expert: `tokens` draws from weights (rank + 1)^-skew, ranks shuffled."""
    gen = torch.Generator().manual_seed(seed * 7919 + 13)
    if experts == 1:
        return [tokens]
    weights = torch.arange(1, experts + 1, dtype=torch.float64) ** -skew
    weights = weights[torch.randperm(experts, generator=gen)]
    picks = torch.multinomial(weights, tokens, replacement=True, generator=gen)
    return torch.bincount(picks, minlength=experts).tolist()


def _bounds(lengths):
    ends, at = [], 0
    for n in lengths:
        at += n
        ends.append(at)
    return list(zip([0] + ends[:-1], ends))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=gen, dtype=dtype) * std).to(dtype)

    state = {"case": case}
    if case["op"] == "fp8_quantize":
        m, k = case["m"], case["k"]
        x = normal((m, k))
        # A few channels stand out, as in a layer's activations.
        channel = torch.rand((1, k), device="cuda", generator=gen)
        state["x"] = (x * torch.where(channel > 0.995, 30.0, 1.0)).to(DTYPES[case["dtype"]])
        return state
    experts, tokens = case["experts"], case["tokens"]
    state["bounds"] = _bounds(_lengths(tokens, experts, case["skew"], seed))
    state["offs"] = torch.tensor([end for _, end in state["bounds"]], dtype=torch.int32, device="cuda")
    if case["op"] == "fp8_mm":
        n, k = case["n"], case["k"]
        x = normal((tokens, k), dtype=torch.bfloat16)
        pairs = [_plain_blocks(normal((n, k), k**-0.5, torch.bfloat16)) for _ in range(experts)]
        state["b"] = torch.stack([q.view(torch.uint8) for q, _ in pairs]).view(torch.float8_e4m3fn)
        state["sb"] = torch.stack([s.view(torch.uint8) for _, s in pairs]).view(torch.float8_e8m0fnu)
        if case["quantize"]:
            state["x"] = x
        else:
            state["a"], state["sa"] = _plain_rows(x)
        return state
    dtype, h, f = DTYPES[case["dtype"]], case["hidden"], case["ffn"]
    state["x"] = normal((tokens, h), dtype=dtype)
    state["w13"] = normal((experts, h, 2 * f), h**-0.5, dtype)
    state["w2"] = normal((experts, f, h), f**-0.5, dtype)
    if case["op"] == "ffn_backward":
        state["dy"] = normal((tokens, h), dtype=dtype)
        _, state["h"], state["gate_up"] = _plain_forward(state)
    return state


# -------------------------------------------------------------- plain forms
def _plain_forward(state):
    """(y, h, gate_up): each in fp32 per expert, rounded once at the end."""
    x, w13, w2 = state["x"], state["w13"], state["w2"]
    dtype, f = x.dtype, w2.shape[1]
    gate_up = torch.cat([x[a:b].float() @ w13[e].float() for e, (a, b) in enumerate(state["bounds"])])
    gate, up = gate_up[:, :f], gate_up[:, f:]
    h = gate * torch.sigmoid(gate) * up
    y = torch.cat([h[a:b] @ w2[e].float() for e, (a, b) in enumerate(state["bounds"])])
    return y.to(dtype), h.to(dtype), gate_up.to(dtype)


def _plain_backward(state):
    """(dx, dw13, dw2) from dy and what the forward pass kept."""
    x, w13, w2, dy, h = state["x"], state["w13"], state["w2"], state["dy"], state["h"]
    dtype, f = x.dtype, w2.shape[1]
    parts = list(enumerate(state["bounds"]))
    dh = torch.cat([dy[a:b].float() @ w2[e].float().t() for e, (a, b) in parts])
    gate, up = state["gate_up"][:, :f].float(), state["gate_up"][:, f:].float()
    s = torch.sigmoid(gate)
    dgu = torch.cat([dh * up * s * (1.0 + gate * (1.0 - s)), dh * gate * s], dim=1)
    dx = torch.cat([dgu[a:b] @ w13[e].float().t() for e, (a, b) in parts]).to(dtype)
    dw13 = torch.stack([(x[a:b].float().t() @ dgu[a:b]).to(dtype) for _, (a, b) in parts])
    dw2 = torch.stack([(h[a:b].float().t() @ dy[a:b].float()).to(dtype) for _, (a, b) in parts])
    return dx, dw13, dw2


def _power_scale(amax):
    """Smallest power of two s with amax <= 448 s, as (s, its e8m0 value); 1 for a block of zeros."""
    mantissa, exponent = torch.frexp(amax)  # amax = mantissa * 2^exponent, mantissa in [0.5, 1); 448 = 0.875 * 2^9
    e = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    e = torch.where(amax == 0, torch.zeros_like(e), e).clamp(-127, 127)
    return torch.ldexp(torch.ones_like(amax, dtype=torch.float64), e), (e + 127).to(torch.uint8).view(torch.float8_e8m0fnu)


def _pad(x, rows, cols):
    return torch.nn.functional.pad(x.float(), (0, -x.shape[1] % cols, 0, -x.shape[0] % rows))


def _plain_rows(x):
    m, k = x.shape
    v = _pad(x, 1, BLOCK).view(m, -1, BLOCK)
    scale, e8 = _power_scale(v.abs().amax(dim=2))
    q = (v.double() / scale[:, :, None]).float().view(m, -1)[:, :k]
    return q.to(torch.float8_e4m3fn), e8


def _plain_blocks(w):
    n, k = w.shape
    p = _pad(w, BLOCK, BLOCK)
    v = p.view(p.shape[0] // BLOCK, BLOCK, -1, BLOCK)
    scale, e8 = _power_scale(v.abs().amax(dim=(1, 3)))
    q = (v.double() / scale[:, None, :, None]).float().reshape(p.shape)[:n, :k]
    return q.to(torch.float8_e4m3fn), e8


def _e8m0_value(s):
    """2^(byte - 127) of e8m0 scales as fp32 (bytes from 1 to 254)."""
    return (s.view(torch.uint8).to(torch.int32) << 23).view(torch.float32)


def _plain_mm(state):
    a, sa = _plain_rows(state["x"]) if "x" in state else (state["a"], state["sa"])
    k, n = a.shape[1], state["b"].shape[1]
    wide = a.float() * _e8m0_value(sa).repeat_interleave(BLOCK, dim=1)[:, :k]
    scales = _e8m0_value(state["sb"])

    def weight(e):
        full = scales[e].repeat_interleave(BLOCK, dim=0)[:n].repeat_interleave(BLOCK, dim=1)[:, :k]
        return state["b"][e].float() * full

    return torch.cat([wide[i:j] @ weight(e).t() for e, (i, j) in enumerate(state["bounds"])]).to(torch.bfloat16)


# --------------------------------------------------------------------- run
def run(state):
    case = state["case"]
    op = case["op"]
    if own:
        kernels = _kernels()
        if op == "ffn_forward":
            return kernels.gated_ffn_forward(state["x"], state["w13"], state["w2"], state["offs"])
        if op == "ffn_backward":
            return kernels.gated_ffn_backward(state["dy"], state["x"], state["w13"], state["w2"], state["h"],
                                              state["gate_up"], state["offs"])
        if op == "fp8_mm":
            a, sa = kernels.launch_quantize_rows(state["x"]) if "x" in state else (state["a"], state["sa"])
            return kernels.launch_block_scaled_mm(a, sa, state["b"], state["sb"], state["offs"])
        if case["kind"] == "rows":
            return kernels.launch_quantize_rows(state["x"])
        return kernels.launch_quantize_blocks(state["x"])
    if op == "ffn_forward":
        return _plain_forward(state)
    if op == "ffn_backward":
        return _plain_backward(state)
    if op == "fp8_mm":
        return _plain_mm(state)
    return _plain_rows(state["x"]) if case["kind"] == "rows" else _plain_blocks(state["x"])


def work(case):
    if case["op"] == "fp8_quantize":
        m, k = case["m"], case["k"]
        blocks = -(-k // BLOCK) * (m if case["kind"] == "rows" else -(-m // BLOCK))
        return {"bytes": 2 * m * k + m * k + blocks, "flops": 0}
    t, used = case["tokens"], min(case["experts"], case["tokens"])  # experts that can have rows
    if case["op"] == "fp8_mm":
        n, k = case["n"], case["k"]
        kb = -(-k // BLOCK)
        weights = used * (n * k + -(-n // BLOCK) * kb)
        return {"bytes": t * k * 2 + weights + 2 * t * n if case["quantize"] else t * (k + kb) + weights + 2 * t * n,
                "flops": 2 * t * n * k}
    h, f = case["hidden"], case["ffn"]
    weights = 3 * h * f
    if case["op"] == "ffn_forward":  # x, W13, W2 -> y, h, [gate | up]
        return {"bytes": 2 * (2 * t * h + 3 * t * f + used * weights), "flops": 6 * t * h * f}
    # dy, x, h, [gate | up], W13, W2 -> dx, dW13, dW2
    return {"bytes": 2 * (3 * t * h + 3 * t * f + (used + case["experts"]) * weights), "flops": 12 * t * h * f}


# ------------------------------------------------------------------- exact
def exact(case, seed):
    """The definitions in 64 bits, expert by expert."""
    state = prepare(case, seed)
    if case["op"] == "fp8_quantize":
        return _exact_quantize(state["x"].double(), 1 if case["kind"] == "rows" else BLOCK)
    wide = torch.float64
    if case["op"] == "fp8_mm":
        if "x" in state:
            qa, sa = _exact_quantize(state["x"].double(), 1)
        else:
            qa, sa = state["a"].to(wide), _exact_scale(state["sa"])
        t, k = qa.shape
        n = state["b"].shape[1]
        out = torch.empty((t, n), dtype=wide, device="cuda")
        cols = torch.arange(k, device="cuda") // BLOCK
        rows = torch.arange(n, device="cuda") // BLOCK
        a = qa * sa[:, cols]
        for e, (i, j) in enumerate(state["bounds"]):
            w = state["b"][e].to(wide) * _exact_scale(state["sb"][e])[rows][:, cols]
            out[i:j] = torch.einsum("mk,nk->mn", a[i:j], w)
        return out
    x, w13, w2 = state["x"], state["w13"], state["w2"]
    f, h = w2.shape[1], w2.shape[2]
    if case["op"] == "ffn_forward":
        y = torch.empty((x.shape[0], h), dtype=wide, device="cuda")
        act = torch.empty((x.shape[0], f), dtype=wide, device="cuda")
        pre = torch.empty((x.shape[0], 2 * f), dtype=wide, device="cuda")
        for e, (i, j) in enumerate(state["bounds"]):
            pre[i:j] = torch.einsum("th,hf->tf", x[i:j].to(wide), w13[e].to(wide))
            g = pre[i:j, :f]
            act[i:j] = g / (1.0 + torch.exp(-g)) * pre[i:j, f:]
            y[i:j] = torch.einsum("tf,fh->th", act[i:j], w2[e].to(wide))
        return y, act, pre
    dx = torch.empty(x.shape, dtype=wide, device="cuda")
    # The gradients leave in 32 bits (the values themselves are 64-bit sums):
    # 32 experts' weights in 64 bits would not fit beside a second state.
    dw13 = torch.empty(w13.shape, dtype=torch.float32, device="cuda")
    dw2 = torch.empty(w2.shape, dtype=torch.float32, device="cuda")
    for e, (i, j) in enumerate(state["bounds"]):
        dy, pre = state["dy"][i:j].to(wide), state["gate_up"][i:j].to(wide)
        g, u = pre[:, :f], pre[:, f:]
        dh = torch.einsum("th,fh->tf", dy, w2[e].to(wide))
        sig = 1.0 / (1.0 + torch.exp(-g))
        silu = g * sig
        d = torch.cat([dh * u * (sig + silu * (1.0 - sig)), dh * silu], dim=1)
        dx[i:j] = torch.einsum("tf,hf->th", d, w13[e].to(wide))
        dw13[e] = torch.einsum("th,tf->hf", x[i:j].to(wide), d)
        dw2[e] = torch.einsum("tf,th->fh", state["h"][i:j].to(wide), dy)
    return dx, dw13, dw2


def _exact_scale(s):
    return torch.exp2(s.view(torch.uint8).to(torch.float64) - 127.0)


def _exact_quantize(x, rows):
    """(q, scale) of blocks of `rows` x 128: the e4m3 values nearest to x / scale (ties to even)."""
    m, k = x.shape
    mb, kb = -(-m // rows), -(-k // BLOCK)
    full = torch.zeros((mb * rows, kb * BLOCK), dtype=torch.float64, device=x.device)
    full[:m, :k] = x
    blocks = full.view(mb, rows, kb, BLOCK)
    top = blocks.abs().amax(dim=(1, 3))
    e = torch.ceil(torch.log2(torch.where(top > 0, top, 448.0) / 448.0)).clamp(-127, 127)
    # log2 rounds: settle the border by comparing the powers themselves.
    e = torch.where(top > 448.0 * torch.exp2(e), e + 1, e)
    e = torch.where((top > 0) & (top <= 448.0 * torch.exp2(e - 1)), e - 1, e).clamp(-127, 127)
    scale = torch.exp2(e)
    v = (blocks / scale[:, None, :, None]).view(mb * rows, kb * BLOCK)[:m, :k]
    # e4m3: 3 fraction bits, exponents from -6 (subnormals below) to 8.
    step = torch.exp2(torch.floor(torch.log2(v.abs().clamp_min(2.0**-6))) - 3.0)
    return torch.round(v / step) * step, scale

"""Performance cases of the operators around the block-scaled FP8 product: the norm that makes its A operand, the product with
an epilogue, and the gated pair of products.

`listed()` gives the named cases, `draw(rng)` one more of the same ranges; `prepare` builds what a program holds before the
call; `run` is one pass: through the public entry points where `own` is true, else the same operator in elementary torch
operations in fp32; `exact` gives the results in 64 bits, `work` the bytes and operations a pass cannot do without.

Every case has an "op":
  norm    q, a_scale[, r_out] = rmsnorm_quantize(x, w[, r]): s = x + r, y = s / sqrt(mean(s^2) + eps) * w, then 1 x 128 scales and
          e4m3 bytes in the layout of the product's A.  Rows are padded with zero rows to a multiple of 16.
  epi     C = act(A . B + bias) + residual, in bf16
  gated   h = act(A . B_gate) * (A . B_up), in bf16 or as e4m3 bytes with 1 x 128 scales (the next product's A)
"""
import math

import torch

own = False

DEV = "cuda"
FP8 = torch.float8_e4m3fn
FP8_MAX = 448.0
EPS = 1e-6
# No drawn case costs more than the largest listed ones.
MAX_FLOPS = 2.0 * 6144 * 4608 * 7168
MAX_NORM = 6144 * 4608


def listed():
    return [
        # the norm in front of a layer while one sequence is decoded: one token, latency alone
        {"name": "norm_1x7168_bf16_residual", "op": "norm", "rows": 1, "K": 7168, "x": "bf16", "residual": True, "wide": 0},
        # the same norm in prefill of a few thousand tokens
        {"name": "norm_4096x7168_bf16_residual", "op": "norm", "rows": 4096, "K": 7168, "x": "bf16", "residual": True, "wide": 0},
        # norm of a low-rank projection that is a column slice of a wider output, an odd number of tokens
        {"name": "norm_1031x1536_bf16_slice", "op": "norm", "rows": 1031, "K": 1536, "x": "bf16", "residual": False, "wide": 2112},
        # a residual stream that is kept in fp32
        {"name": "norm_6144x4608_f32_residual", "op": "norm", "rows": 6144, "K": 4608, "x": "f32", "residual": True, "wide": 0},
        # projection back to the model's width while one sequence is decoded, the residual added
        {"name": "epi_1x7168x2304_residual", "op": "epi", "rows": 1, "N": 7168, "K": 2304, "bias": False, "act": "none",
         "residual": True},
        # a projection with bias and activation for a medium batch: few tiles, long K
        {"name": "epi_1024x1536x7168_bias_gelu", "op": "epi", "rows": 1024, "N": 1536, "K": 7168, "bias": True, "act": "gelu",
         "residual": False},
        # ragged: no dimension fills its last tile, the last row group is cut
        {"name": "epi_2051x1552x3200_bias_silu_residual", "op": "epi", "rows": 2051, "N": 1552, "K": 3200, "bias": True,
         "act": "silu", "residual": True},
        # the benchmark's compute-bound shape with everything the epilogue can do, and the largest case
        {"name": "epi_6144x4608x7168_bias_gelu_tanh_residual", "op": "epi", "rows": 6144, "N": 4608, "K": 7168, "bias": True,
         "act": "gelu_tanh", "residual": True},
        # gate and up projections of a feed-forward layer while a few sequences are decoded
        {"name": "gated_7x2048x7168_fp8", "op": "gated", "rows": 7, "N": 2048, "K": 7168, "act": "silu", "fp8": True},
        # a short prompt: more rows than the decoding kernel takes, too few tiles for the GPU
        {"name": "gated_192x2304x7168_fp8", "op": "gated", "rows": 192, "N": 2304, "K": 7168, "act": "silu", "fp8": True},
        # ragged, result in bf16 for a consumer that is not quantised
        {"name": "gated_1037x1552x3200_gelu_tanh_bf16", "op": "gated", "rows": 1037, "N": 1552, "K": 3200, "act": "gelu_tanh",
         "fp8": False},
        # the same layer in prefill
        {"name": "gated_4096x2048x7168_fp8", "op": "gated", "rows": 4096, "N": 2048, "K": 7168, "act": "silu", "fp8": True},
    ]


def _log_int(rng, lo, hi, step=1):
    """A multiple of `step` in [lo, hi], spread over the logarithm of its value."""
    v = math.exp(rng.uniform(math.log(lo), math.log(hi)))
    return min(hi, max(lo, int(round(v / step)) * step))


def draw(rng):
    op = rng.choice(["norm", "epi", "gated"])
    while True:
        rows = _log_int(rng, 1, 8192)
        K = _log_int(rng, 128, 7168, 128)
        if op == "norm":
            K = _log_int(rng, 128, 16384, 128)
            if rows * K > MAX_NORM:
                continue
            wide = K + 8 * rng.randrange(1, 97) if rng.random() < 0.3 else 0
            return {"op": op, "rows": rows, "K": K, "x": rng.choice(["bf16", "bf16", "f32"]), "residual": rng.random() < 0.6,
                    "wide": wide}
        if op == "epi":
            N = _log_int(rng, 16, 7168, 16)
            if 2.0 * rows * N * K > MAX_FLOPS:
                continue
            return {"op": op, "rows": rows, "N": N, "K": K, "bias": rng.random() < 0.6, "residual": rng.random() < 0.6,
                    "act": rng.choice(["none", "relu", "silu", "gelu", "gelu_tanh"])}
        fp8 = rng.random() < 0.7
        N = _log_int(rng, 128, 7168, 128 if fp8 else 16)
        if 4.0 * rows * N * K > MAX_FLOPS:
            continue
        return {"op": op, "rows": rows, "N": N, "K": K, "act": rng.choice(["silu", "silu", "gelu", "gelu_tanh", "relu"]),
                "fp8": fp8}


# ---------------------------------------------------------------- inputs -----------------------------------------
def _pad16(rows):
    return (rows + 15) // 16 * 16


def _activations(g, rows, K):
    """Activations of a layer: normal, with a spread between channels."""
    x = torch.randn(rows, K, generator=g, device=DEV)
    return x * torch.exp(0.5 * torch.randn(K, generator=g, device=DEV))


def _operand(x, rows_per_group):
    """[R, K] fp32 -> column-major e4m3 bytes and inverse scales [K / 128, ceil(R / rows_per_group)], as a program has them
    after quantising (R a multiple of 16)."""
    R, K = x.shape
    pad = -R % rows_per_group
    b = torch.nn.functional.pad(x, (0, 0, 0, pad)).view((R + pad) // rows_per_group, rows_per_group, K // 128, 128)
    scale = b.abs().amax(dim=(1, 3), keepdim=True).clamp(min=1e-12).reciprocal() * FP8_MAX
    q = (b * scale).clamp(-FP8_MAX, FP8_MAX).to(FP8).view(R + pad, K)[:R]
    inv = (1.0 / scale).view(-1, K // 128)
    return q.view(torch.uint8).t().contiguous().flatten(), inv.t().contiguous().flatten()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(int(seed))
    rows, K = case["rows"], case["K"]
    state = {"case": case}
    if case["op"] == "norm":
        dtype = torch.bfloat16 if case["x"] == "bf16" else torch.float32
        wide = case["wide"] or K
        state["x"] = _activations(g, rows, wide).to(dtype)[:, :K]
        state["r"] = (3.0 * _activations(g, rows, K)).to(dtype) if case["residual"] else None
        state["w"] = (1.0 + 0.2 * torch.randn(K, generator=g, device=DEV)).to(dtype)
        return state
    N, M = case["N"], _pad16(rows)
    x = torch.nn.functional.pad(_activations(g, rows, K), (0, 0, 0, M - rows))
    x /= x.square().mean().sqrt()
    state["A"], state["a_scale"] = _operand(x, 1)
    for name in ["B"] if case["op"] == "epi" else ["B_gate", "B_up"]:
        w = torch.randn(N, K, generator=g, device=DEV) * (K ** -0.5)
        state[name], state[name + "_scale"] = _operand(w, 128)
    if case["op"] == "epi":
        state["bias"] = torch.randn(N, generator=g, device=DEV) if case["bias"] else None
        state["residual"] = torch.randn(rows, N, generator=g, device=DEV).to(torch.bfloat16) if case["residual"] else None
    return state


# ---------------------------------------------------------------- one pass ----------------------------------------
def _act(x, name):
    if name == "relu":
        return torch.where(x < 0, torch.zeros_like(x), x)
    if name == "silu":
        return x / (1.0 + torch.exp(-x))
    if name == "gelu":
        return 0.5 * x * (1.0 + torch.erf(x * math.sqrt(0.5)))
    if name == "gelu_tanh":
        return 0.5 * x * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (x + 0.044715 * x * x * x)))
    return x


def _row_scaled(y, rows):
    """[rows, K] fp32 -> e4m3 values [K, M] and inverse scales [K / 128, M], zero rows behind the last."""
    K = y.shape[1]
    y = torch.nn.functional.pad(y, (0, 0, 0, _pad16(rows) - rows)).view(-1, K // 128, 128)
    scale = y.abs().amax(dim=2, keepdim=True).clamp(min=1e-12).reciprocal() * FP8_MAX
    q = (y * scale).clamp(-FP8_MAX, FP8_MAX).to(FP8).view(-1, K)
    return q.view(torch.uint8).t().contiguous().view(FP8), (1.0 / scale).view(-1, K // 128).t().contiguous()


def _dequantized(q, scale, R, K, rows_per_group):
    """[R, K] fp32 of column-major bytes and their inverse scales."""
    v = q.view(FP8).view(K, R).t().float()
    s = scale.view(K // 128, -1).t().repeat_interleave(rows_per_group, 0)[:R].repeat_interleave(128, 1)
    return v * s


def _plain(state):
    case = state["case"]
    rows, K = case["rows"], case["K"]
    if case["op"] == "norm":
        s = state["x"].float()
        if state["r"] is not None:
            s = s + state["r"].float()
        y = s * torch.rsqrt(s.square().mean(dim=1, keepdim=True) + EPS) * state["w"].float()
        q, scale = _row_scaled(y, rows)
        return (q, scale) if state["r"] is None else (q, scale, s.to(state["r"].dtype))
    N = case["N"]
    A = _dequantized(state["A"], state["a_scale"], _pad16(rows), K, 1)[:rows]
    if case["op"] == "epi":
        C = A @ _dequantized(state["B"], state["B_scale"], N, K, 128).t()
        if state["bias"] is not None:
            C = C + state["bias"]
        C = _act(C, case["act"])
        if state["residual"] is not None:
            C = C + state["residual"].float()
        return C.to(torch.bfloat16)
    gate = A @ _dequantized(state["B_gate"], state["B_gate_scale"], N, K, 128).t()
    up = A @ _dequantized(state["B_up"], state["B_up_scale"], N, K, 128).t()
    h = _act(gate, case["act"]) * up
    return _row_scaled(h, rows) if case["fp8"] else h.to(torch.bfloat16)


def run(state):
    if not own:
        return _plain(state)
    import fp8_quant_matmul_b200 as f
    case = state["case"]
    rows, K = case["rows"], case["K"]
    M = _pad16(rows)
    if case["op"] == "norm":
        q, scale, *r = f.rmsnorm_quantize(state["x"], state["w"], residual=state["r"], eps=EPS)
        return (q.view(FP8).view(K, M), scale.view(K // 128, M), *r)
    N = case["N"]
    if case["op"] == "epi":
        return f.gemm_bias_act(state["A"], state["B"], state["a_scale"], state["B_scale"], M=M, N=N, K=K, rows=rows,
                               bias=state["bias"], activation=case["act"], residual=state["residual"])
    h = f.gemm_gated(state["A"], state["B_gate"], state["B_up"], state["a_scale"], state["B_gate_scale"], state["B_up_scale"],
                     M=M, N=N, K=K, rows=rows, activation=case["act"], quantize=case["fp8"])
    return (h[0].view(FP8).view(N, M), h[1].view(N // 128, M)) if case["fp8"] else h


def work(case):
    rows, K = case["rows"], case["K"]
    M = _pad16(rows)
    if case["op"] == "norm":
        e = 2.0 if case["x"] == "bf16" else 4.0
        return {"bytes": rows * K * e * (3.0 if case["residual"] else 1.0) + M * K + 4.0 * M * (K // 128) + e * K, "flops": 0.0}
    N = case["N"]
    a = rows * K + 4.0 * rows * (K // 128)
    b = N * K + 4.0 * ((N + 127) // 128) * (K // 128)
    if case["op"] == "epi":
        return {"bytes": a + b + 2.0 * rows * N * (2.0 if case["residual"] else 1.0) + (4.0 * N if case["bias"] else 0.0),
                "flops": 2.0 * rows * N * K}
    out = M * N + 4.0 * M * (N // 128) if case["fp8"] else 2.0 * rows * N
    return {"bytes": a + 2.0 * b + out, "flops": 4.0 * rows * N * K}


# ------------------------------------------------------- the same results in 64 bits ------------------------------
def _values(q, scale, R, K, group):
    """Column-major bytes and inverse scales as [R, K] float64: value[r, k] = byte * scale[k / 128, r / group]."""
    r, k = torch.arange(R, device=DEV), torch.arange(K, device=DEV)
    s = scale.double().view(K // 128, -1)[(k // 128)[:, None], (r // group)[None, :]]
    return (q.view(FP8).view(K, R).double() * s).T


def _scaled_exactly(y, rows):
    """The quantised form before its rounding to 8 bits: y * fp8_max / amax, and amax / fp8_max; in the operand's layout."""
    K = y.shape[1]
    full = y.new_zeros(_pad16(rows), K)
    full[:rows] = y
    blocks = full.T.reshape(K // 128, 128, -1)
    inv = blocks.abs().amax(dim=1).clamp(min=1e-12) / FP8_MAX
    return (blocks / inv[:, None, :]).reshape(K, -1), inv


def _activated(x, name):
    if name == "relu":
        return x.clamp(min=0.0)
    if name == "silu":
        return x * torch.sigmoid(x)
    if name == "gelu":
        return x * torch.special.ndtr(x)
    if name == "gelu_tanh":      # (1 + tanh(z)) / 2 = sigmoid(2 z)
        return x * torch.sigmoid(2.0 * (2.0 / math.pi) ** 0.5 * (x + 0.044715 * x ** 3))
    return x


def exact(case, seed):
    t = prepare(case, seed)
    rows, K = case["rows"], case["K"]
    if case["op"] == "norm":
        s = t["x"].double() if t["r"] is None else t["x"].double() + t["r"].double()
        y = s / (s.pow(2).sum(1) / K + EPS).sqrt()[:, None] * t["w"].double()[None, :]
        out = _scaled_exactly(y, rows)
        return out if t["r"] is None else (*out, s)
    N, M = case["N"], _pad16(rows)
    A = _values(t["A"], t["a_scale"], M, K, 1)[:rows]
    if case["op"] == "epi":
        C = A @ _values(t["B"], t["B_scale"], N, K, 128).T
        if t["bias"] is not None:
            C += t["bias"].double()[None, :]
        C = _activated(C, case["act"])
        return C if t["residual"] is None else C + t["residual"].double()
    h = _activated(A @ _values(t["B_gate"], t["B_gate_scale"], N, K, 128).T, case["act"])
    h = h * (A @ _values(t["B_up"], t["B_up_scale"], N, K, 128).T)
    return _scaled_exactly(h, rows) if case["fp8"] else h

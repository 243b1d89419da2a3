"""Workloads of a decoder layer's feed-forward half, and their plain forms.

A case is one call, or a forward call and its gradients, that a program makes in every decoder layer:

* ``gated``  `gated_gemm_bf16_nt`: act(x Wg^T) * (x Wu^T) with Wg, Wu the halves of one weight [2 I, H],
             as a serving rank runs it between the norm and its row-parallel down projection;
* ``train``  the same with what its gradient needs kept, then `gated_gemm_bf16_nt_backward`: the
             gradients of x and of the weight;
* ``quant``  `quant_fp8_groups`: rows to e4m3 codes with one fp32 scale for 128 channels, of a norm's
             output or (gated) of act(gate) * up of a projection's two halves, taken on the way;
* ``block``  `gemm_fp8_block_nt`: the product of such rows with a weight of e4m3 codes that has one
             scale for each block of 128 x 128.

Sizes are those of the shipped weave tables' models (hidden 8192 or 6144; intermediate 28672, 29568
and 16384 over eight or four ranks: 3584, 3696, 2048, 7168) and generic ones.

Codes: scale = max(largest magnitude of the group, 1e-10) / 448 rounded to fp32, code = the e4m3 value
next to x / scale, ties to the even code.  The last group or block of an axis holds what is left.
"""
import math

import torch

own = False

DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
GROUP = 128
FP8 = torch.float8_e4m3fn
ACTS = ("silu", "silu", "silu", "gelu", "gelu_tanh")
#        hidden, intermediate of one rank
SHAPES = ((8192, 3584), (8192, 3696), (6144, 2048), (8192, 7168), (4096, 1376), (1024, 704), (768, 2048), (520, 1000))
MOST_GATED = 4096 * 8192 * 3584
MOST_QUANT = 8192 * 2 * 3584 * 2     # bytes of the largest listed quant
MOST_BLOCK = 4096 * 7168 * 8192


def listed():
    return [
        # one user's token on one of eight ranks: the weight is read once
        {"name": "gated_one", "op": "gated", "tokens": 1, "H": 8192, "I": 3584, "act": "silu"},
        # a ragged batch decoding on one of eight ranks
        {"name": "gated_decode", "op": "gated", "tokens": 61, "H": 8192, "I": 3696, "act": "silu"},
        # a prefill chunk on one of eight ranks
        {"name": "gated_prompt", "op": "gated", "tokens": 4096, "H": 8192, "I": 3584, "act": "silu"},
        # a small model trained on an odd count of tokens
        {"name": "train_small", "op": "train", "tokens": 1001, "H": 1024, "I": 704, "act": "gelu_tanh"},
        # one of eight ranks trained on 4096 tokens
        {"name": "train_rank", "op": "train", "tokens": 4096, "H": 8192, "I": 3584, "act": "silu"},
        # a decode batch's norm output in front of an 8-bit projection
        {"name": "quant_decode", "op": "quant", "tokens": 32, "K": 8192, "gated": False, "act": "silu", "dtype": "bf16"},
        # a ragged fp16 chunk whose rows end inside a group
        {"name": "quant_ragged", "op": "quant", "tokens": 1001, "K": 3696, "gated": False, "act": "silu", "dtype": "fp16"},
        # between the two projections of a prefill chunk: activation, product and codes in one pass
        {"name": "quant_gated", "op": "quant", "tokens": 8192, "K": 3584, "gated": True, "act": "silu", "dtype": "bf16"},
        # one user's token through a rank's down projection
        {"name": "block_one", "op": "block", "tokens": 1, "N": 8192, "K": 3584, "dtype": "bf16"},
        # a decode batch through a rank's gate and up projections
        {"name": "block_decode", "op": "block", "tokens": 96, "N": 7168, "K": 8192, "dtype": "bf16"},
        # a ragged fp16 chunk whose inner dimension ends inside a block
        {"name": "block_ragged", "op": "block", "tokens": 1000, "N": 8192, "K": 3696, "dtype": "fp16"},
        # a prefill chunk through a rank's gate and up projections
        {"name": "block_prompt", "op": "block", "tokens": 4096, "N": 7168, "K": 8192, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    """Spread over the logarithm; a third of the larger values are rounded to a multiple of 16."""
    n = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if n > 64 and rng.random() < 0.33:
        n = (n + 15) // 16 * 16
    return max(low, min(high, n))


def draw(rng):
    op = rng.choice(("gated", "gated", "train", "quant", "block", "block"))
    H, inner = rng.choice(SHAPES)
    if op in ("gated", "train"):
        if rng.random() < 0.3:
            H, inner = 8 * _log_int(rng, 8, 1024), 4 * _log_int(rng, 8, 1792)
        most = MOST_GATED // (H * inner)
        return {"op": op, "tokens": min(_log_int(rng, 1, 8192 if op == "gated" else 4096), most), "H": H, "I": inner,
                "act": rng.choice(ACTS)}
    if op == "quant":
        K, gated, dtype = rng.choice((H, inner, 16 * _log_int(rng, 1, 512))), rng.random() < 0.5, \
            rng.choice(("bf16", "bf16", "fp16", "fp32"))
        most = MOST_QUANT // (K * (2 if gated else 1) * DTYPES[dtype].itemsize)
        return {"op": op, "tokens": min(_log_int(rng, 1, 16384), most), "K": K, "gated": gated, "act": rng.choice(ACTS),
                "dtype": dtype}
    N, K = rng.choice(((2 * inner, H), (H, inner), (8 * _log_int(rng, 8, 1024), 16 * _log_int(rng, 2, 512))))
    K = (K + 15) // 16 * 16
    return {"op": op, "tokens": min(_log_int(rng, 1, 8192), MOST_BLOCK // (N * K)), "N": N, "K": K,
            "dtype": rng.choice(("bf16", "bf16", "fp16"))}


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------
def _normal(shape, g, std=1.0):
    return torch.randn(shape, generator=g, device=DEV, dtype=torch.float32) * std


def _activations(tokens, channels, g):
    """A norm's output: some channels are many times larger than the others."""
    gain = 1 + 19 * (torch.rand(channels, generator=g, device=DEV) < 0.005).float()
    return _normal((tokens, channels), g) * gain


def _scales(tokens, K):
    """[tokens, groups] fp32, the tokens of a group side by side."""
    return torch.empty((-(-K // GROUP), tokens), dtype=torch.float32, device=DEV).t()


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    T, op = case["tokens"], case["op"]
    state = {"case": case}
    if op in ("gated", "train"):
        H, inner = case["H"], case["I"]
        state["x"] = _activations(T, H, g).bfloat16()
        state["w"] = _normal((2 * inner, H), g, H ** -0.5).bfloat16()
        state["out"] = torch.empty((T, inner), dtype=torch.bfloat16, device=DEV)
        if op == "train":
            state["grad"] = _normal((T, inner), g, 1e-3).bfloat16()
            state["gate_up"] = torch.empty((T, 2 * inner), dtype=torch.bfloat16, device=DEV)
            state["grad_x"], state["grad_w"] = torch.empty_like(state["x"]), torch.empty_like(state["w"])
    elif op == "quant":
        dtype, K = DTYPES[case["dtype"]], case["K"]
        state["x"] = (_normal((T, 2 * K), g) if case["gated"] else _activations(T, K, g)).to(dtype)
        state["codes"] = torch.empty((T, K), dtype=FP8, device=DEV)
        state["scales"] = _scales(T, K)
    else:
        N, K = case["N"], case["K"]
        codes, scales = _codes(_activations(T, K, g))
        state["a"], state["a_scales"] = codes, _scales(T, K).copy_(scales)
        state["b"], state["b_scales"] = _weight_codes(_normal((N, K), g, K ** -0.5))
        state["out"] = torch.empty((T, N), dtype=DTYPES[case["dtype"]], device=DEV)
    return state


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------
def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from tokenweave_amd import ops
    case = state["case"]
    op = case["op"]
    if op == "gated":
        ops.gated_gemm_bf16_nt(state["out"], state["x"], state["w"], case["act"])
        return state["out"]
    if op == "train":
        ops.gated_gemm_bf16_nt(state["out"], state["x"], state["w"], case["act"], gate_up=state["gate_up"])
        ops.gated_gemm_bf16_nt_backward(state["grad_x"], state["grad_w"], state["grad"], state["x"], state["w"],
                                        state["gate_up"], case["act"])
        return state["out"], state["grad_x"], state["grad_w"]
    if op == "quant":
        ops.quant_fp8_groups(state["codes"], state["scales"], state["x"], case["act"] if case["gated"] else None)
        return state["codes"], state["scales"]
    ops.gemm_fp8_block_nt(state["out"], state["a"], state["a_scales"], state["b"], state["b_scales"])
    return state["out"]


def _run_plain(state):
    case = state["case"]
    op = case["op"]
    if op == "quant":
        x = state["x"].float()
        if case["gated"]:
            gate, up = x.chunk(2, -1)
            x = _act(gate, case["act"]) * up
        return _codes(x)
    if op == "block":
        a = state["a"].float() * _spread(state["a_scales"], state["a"].shape[1], 1)
        b = state["b"].float() * _spread(_spread(state["b_scales"], state["b"].shape[0], 0), state["b"].shape[1], 1)
        return (a @ b.t()).to(state["out"].dtype)
    x, w = state["x"].float(), state["w"].float()
    gate, up = (x @ w.t()).chunk(2, -1)
    act = _act(gate, case["act"])
    out = (act * up).bfloat16()
    if op == "gated":
        return out
    grad = state["grad"].float()
    both = torch.cat((grad * up * _slope(gate, case["act"]), grad * act), -1)
    return out, (both @ w).bfloat16(), (both.t() @ x).bfloat16()


# ---------------------------------------------------------------------------
# plain forms
# ---------------------------------------------------------------------------
TANH_A, TANH_B = math.sqrt(2 / math.pi), 0.044715


def _act(x, kind):
    if kind == "silu":
        return x / (1 + torch.exp(-x))
    if kind == "gelu":
        return 0.5 * x * (1 + torch.erf(x * 0.5 ** 0.5))
    return 0.5 * x * (1 + torch.tanh(TANH_A * (x + TANH_B * x * x * x)))


def _slope(x, kind):
    """The activation's derivative."""
    if kind == "silu":
        s = 1 / (1 + torch.exp(-x))
        return s * (1 + x * (1 - s))
    if kind == "gelu":
        return 0.5 * (1 + torch.erf(x * 0.5 ** 0.5)) + x * torch.exp(-0.5 * x * x) * (2 * math.pi) ** -0.5
    t = torch.tanh(TANH_A * (x + TANH_B * x * x * x))
    return 0.5 * (1 + t) + 0.5 * x * (1 - t * t) * TANH_A * (1 + 3 * TANH_B * x * x)


def _spread(scales, n, axis):
    """One scale for GROUP places of an axis -> one for each of its n places."""
    return scales.repeat_interleave(GROUP, axis).narrow(axis, 0, n)


def _nearest(q):
    """The e4m3 values next to q (64 bits: a quotient next to a border must not be rounded twice)."""
    exponent = torch.frexp(q.abs().clamp(min=2.0 ** -6))[1] - 1        # |q| in [2^e, 2^(e+1)), 2^-6 the least normal
    step = torch.exp2(exponent.double() - 3)
    return (torch.round(q / step) * step).clamp(-448, 448).float().to(FP8)


def _codes(x):
    """Codes and scales of rows, a scale for 128 channels."""
    T, K = x.shape
    padded = torch.nn.functional.pad(x, (0, -K % GROUP)).view(T, -1, GROUP)
    scales = (padded.abs().amax(-1).clamp(min=1e-10).double() / 448).float()
    return _nearest(x.double() / _spread(scales, K, 1).double()), scales


def _weight_codes(w):
    """Codes and scales of a weight, a scale for 128 x 128 values."""
    N, K = w.shape
    padded = torch.nn.functional.pad(w, (0, -K % GROUP, 0, -N % GROUP))
    blocks = padded.view(padded.shape[0] // GROUP, GROUP, padded.shape[1] // GROUP, GROUP)
    scales = (blocks.abs().amax((1, 3)).clamp(min=1e-10).double() / 448).float()
    return (w / _spread(_spread(scales, N, 0), K, 1)).clamp(-448, 448).to(FP8), scales


# ---------------------------------------------------------------------------
# the definitions in 64 bits
# ---------------------------------------------------------------------------
def _sigmoid_like(x, kind):
    """(f, f') with act(x) = x f(x)."""
    if kind == "silu":
        f = torch.where(x >= 0, 1 / (1 + torch.exp(-x.abs())), 1 - 1 / (1 + torch.exp(-x.abs())))
        return f, f * (1 - f)
    if kind == "gelu":
        return 0.5 * torch.special.erfc(-x / math.sqrt(2)), torch.exp(-x * x / 2) / math.sqrt(2 * math.pi)
    inner = math.sqrt(8 / math.pi) * (x + 0.044715 * x ** 3)           # (1 + tanh(z)) / 2 = sigmoid(2 z)
    f = torch.sigmoid(inner)
    return f, f * torch.sigmoid(-inner) * math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * x ** 2)


def exact(case, seed):
    state = prepare(case, seed)
    op = case["op"]
    if op == "quant":
        x = state["x"].double()
        if case["gated"]:
            K = case["K"]
            x = x[:, :K] * _sigmoid_like(x[:, :K], case["act"])[0] * x[:, K:]
        values = torch.arange(127, dtype=torch.uint8, device=DEV).view(FP8).double()
        borders = (values[1:] + values[:-1]) / 2
        codes, scales = [], []
        for part in x.split(GROUP, 1):
            largest = part.abs().max(1, keepdim=True).values
            scale = torch.maximum(largest, torch.full_like(largest, 1e-10)) / 448
            q = part / scale.float().double()
            # a border belongs to the even of its two codes
            low, high = torch.bucketize(q.abs(), borders), torch.bucketize(q.abs(), borders, right=True)
            at = torch.where((low != high) & (low % 2 == 1), high, low)
            codes.append(torch.copysign(values[at], q))
            scales.append(scale)
        return torch.cat(codes, 1), torch.cat(scales, 1)
    if op == "block":
        out = torch.zeros(state["out"].shape, dtype=torch.float64, device=DEV)
        for k in range(state["a_scales"].shape[1]):
            at = slice(k * GROUP, (k + 1) * GROUP)
            part = state["a"][:, at].double() @ state["b"][:, at].double().t()
            columns = state["b_scales"][:, k].double()[torch.arange(case["N"], device=DEV) // GROUP]
            out += part * state["a_scales"][:, k:k + 1].double() * columns
        return out
    x, w, inner = state["x"].double(), state["w"].double(), case["I"]
    gate, up = x @ w[:inner].t(), x @ w[inner:].t()
    f, df = _sigmoid_like(gate, case["act"])
    out = gate * f * up
    if op == "gated":
        return out
    grad = state["grad"].double()
    grad_up, grad_gate = grad * gate * f, grad * up * (f + gate * df)
    return out, grad_gate @ w[:inner] + grad_up @ w[inner:], torch.cat((grad_gate.t() @ x, grad_up.t() @ x))


def work(case):
    T, op = case["tokens"], case["op"]
    if op in ("gated", "train"):
        H, inner = case["H"], case["I"]
        size = 2 * (T * H + 2 * inner * H + T * inner)     # x, w -> out
        flops = 4 * T * H * inner
        if op == "gated":
            return {"bytes": size, "flops": flops}
        return {"bytes": size + 2 * (T * inner + T * H + 2 * inner * H), "flops": 3 * flops}
    K = case["K"]
    groups = -(-K // GROUP)
    if op == "quant":
        return {"bytes": T * K * (DTYPES[case["dtype"]].itemsize * (2 if case["gated"] else 1) + 1) + 4 * T * groups,
                "flops": T * K * (8 if case["gated"] else 3)}
    N = case["N"]
    return {"bytes": T * K + N * K + 4 * groups * (T + -(-N // GROUP)) + 2 * T * N, "flops": 2 * T * N * K}

"""The feed-forward half of a decoder layer: the gated projection with its gradient, 8-bit
block-scaled linear layers, and both as the layer schedules' ``mlp_fn``.

The reference leaves this half to its model files (``vllm/model_executor/models/llama.py:99-103``:
a merged gate and up projection, an activation op, a row-parallel down projection); here gate, up,
activation and product are one kernel.
"""
from __future__ import annotations

from typing import Any, Optional, Tuple

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable
from torch.nn.parameter import Parameter

from . import _custom_ops as ops
from .linear import RowParallelLinear, _apply_beside_codes, _check_loaded, _holds_codes, _rank_blocks


def _refuse_capture() -> None:
    """Autograd ends the process where a captured backward pass meets leaves that an eager one still holds."""
    if torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("gated_linear records no gradient while a graph is captured: capture "
                           "ops.gated_gemm_bf16_nt(..., gate_up=) and ops.gated_gemm_bf16_nt_backward")


class _GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x: torch.Tensor, weight: torch.Tensor, activation: str, max_cus: Optional[int]) -> torch.Tensor:
        _refuse_capture()
        out = torch.empty((x.shape[0], weight.shape[0] // 2), dtype=x.dtype, device=x.device)
        gate_up = torch.empty((x.shape[0], weight.shape[0]), dtype=x.dtype, device=x.device)
        ops.gated_gemm_bf16_nt(out, x, weight, activation, max_cus, gate_up)
        ctx.save_for_backward(x, weight, gate_up)
        ctx.activation, ctx.max_cus = activation, max_cus
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, grad: torch.Tensor):
        _refuse_capture()
        x, weight, gate_up = ctx.saved_tensors
        grad_x = torch.empty_like(x) if ctx.needs_input_grad[0] else None
        grad_w = torch.empty_like(weight) if ctx.needs_input_grad[1] else None
        ops.gated_gemm_bf16_nt_backward(grad_x, grad_w, grad.contiguous(), x, weight, gate_up, ctx.activation, ctx.max_cus)
        return grad_x, grad_w, None, None


def gated_linear(x: torch.Tensor, weight: torch.Tensor, activation: str = "silu",
                 max_cus: Optional[int] = None) -> torch.Tensor:
    """act(x @ weight[:I]^T) * (x @ weight[I:]^T), x [..., K], weight [2 I, K], both bf16, with the gradients of
    both where they are wanted (what the backward pass needs of the forward one are the two products, in
    bf16)."""
    rows = x.reshape(-1, x.shape[-1]).contiguous()
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad):
        out = _GatedLinear.apply(rows, weight, activation, max_cus)
    else:
        out = torch.empty((rows.shape[0], weight.shape[0] // 2), dtype=x.dtype, device=x.device)
        ops.gated_gemm_bf16_nt(out, rows, weight.detach(), activation, max_cus)
    return out.view(x.shape[:-1] + (out.shape[-1],))


class GatedLinear(nn.Module):
    """One rank's merged gate and up projection with its activation: the rows ``tp_rank`` of ``tp_size`` of both
    weights, gate rows first.  ``intermediate_size`` is the whole model's.  The weight takes part in autograd
    once ``requires_grad_()`` says so."""

    def __init__(self, input_size: int, intermediate_size: int, activation: str = "silu", *, tp_rank: int = 0,
                 tp_size: int = 1) -> None:
        super().__init__()
        if not 0 <= tp_rank < tp_size:
            raise ValueError(f"Invalid rank {tp_rank}, must be in [0, {tp_size - 1}]")
        if intermediate_size % tp_size != 0:
            raise ValueError(f"{intermediate_size} is not divisible by {tp_size}")
        ops._activation_code(activation)
        self.tp_rank, self.tp_size, self.activation = tp_rank, tp_size, activation
        self.input_size, self.intermediate_size = input_size, intermediate_size // tp_size
        self.weight = Parameter(torch.empty(2 * self.intermediate_size, input_size, dtype=torch.bfloat16),
                                requires_grad=False)

    def _apply(self, fn: Any, recurse: bool = True) -> "GatedLinear":
        return _apply_beside_codes(self, super()._apply, fn, recurse)

    def weight_loader(self, param: Parameter, loaded_weight: torch.Tensor, shard_id: int) -> None:
        """This rank's rows of a full gate (``shard_id`` 0) or up (1) weight; of an 8-bit one the codes and, as ``param``
        ``weight_scale``, the scales of its blocks."""
        _check_loaded(self, param, loaded_weight)
        n = self.intermediate_size
        if param is getattr(self, "weight_scale", None) and _holds_codes(self):
            n = _rank_blocks(self, n)
        if loaded_weight.shape[0] != n:
            loaded_weight = loaded_weight.narrow(0, self.tp_rank * n, n)
        param.data.narrow(0, shard_id * n, n).copy_(loaded_weight)

    def forward(self, x: torch.Tensor, max_cus: Optional[int] = None) -> torch.Tensor:
        return gated_linear(x, self.weight, self.activation, max_cus)

    def extra_repr(self) -> str:
        return (f"input_features={self.input_size}, intermediate_features={self.intermediate_size}, "
                f"activation={self.activation}, tp_size={self.tp_size}")


@torch.no_grad()
def quantize_fp8_blocks(weight: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """e4m3 codes of a [N, K] weight and the fp32 scales of its blocks of 128 x 128, [ceil(N / 128), ceil(K / 128)]:
    what `ops.gemm_fp8_block_nt` takes as its right operand.  (Plain torch: done once, when a model is loaded.)"""
    group = ops.FP8_GROUP
    N, K = weight.shape
    codes = torch.empty((N, K), dtype=ops.FP8_DTYPE, device=weight.device)
    scales = torch.empty((-(-N // group), -(-K // group)), dtype=torch.float32, device=weight.device)
    for first in range(0, N, group):
        rows = weight[first:first + group].float()
        blocks = nn.functional.pad(rows, (0, -K % group)).view(rows.shape[0], -1, group)
        scale = (blocks.abs().amax((0, 2)).clamp(min=1e-10).double() / 448).float()
        scales[first // group] = scale
        codes[first:first + group] = (rows / scale.repeat_interleave(group)[:K]).clamp(-448, 448).to(ops.FP8_DTYPE)
    return codes, scales


class Fp8BlockLinearMethod:
    """``quant_method`` of a linear layer whose weight is e4m3 codes with a scale for each block of 128 x 128
    (``layer.weight``, ``layer.weight_scale``): the input's rows are coded with a scale for 128 channels on the
    way.  ``process_weights`` makes both from a layer's bf16 weight; the layer's ``weight_loader`` then takes a
    checkpoint's codes and scales instead."""

    @staticmethod
    def check(layer: nn.Module) -> None:
        N, K = layer.weight.shape
        if K % 16 or N % 4:
            raise ValueError(f"8-bit block-scaled weights need an inner dimension that is a multiple of 16 and a multiple "
                             f"of 4 output channels; this one is {tuple(layer.weight.shape)}")

    def process_weights(self, layer: nn.Module) -> None:
        if isinstance(layer, GatedLinear):   # its activation is taken with the next projection's codes
            raise ValueError("a GatedLinear has no 8-bit form of its own: FeedForward.to_fp8_blocks() codes it with the "
                             "projection behind it")
        self.code_weight(layer)

    def code_weight(self, layer: nn.Module) -> None:
        """``process_weights`` for a layer whose owner calls the products itself."""
        self.check(layer)
        codes, scales = quantize_fp8_blocks(layer.weight.data)
        layer.weight = Parameter(codes, requires_grad=False)
        layer.weight_scale = Parameter(scales, requires_grad=False)
        layer.quant_method = self

    def apply(self, layer: nn.Module, x: torch.Tensor, bias: Optional[torch.Tensor] = None,
              max_cus: Optional[int] = None) -> torch.Tensor:
        output = torch.empty(x.shape[:-1] + (layer.weight.shape[0],), dtype=x.dtype, device=x.device)
        return self.apply_inplace(layer, x, output, bias, max_cus)

    def apply_inplace(self, layer: nn.Module, x: torch.Tensor, output: torch.Tensor,
                      bias: Optional[torch.Tensor] = None, max_cus: Optional[int] = None) -> torch.Tensor:
        """output <- x @ layer.weight.T, then output += bias (if given), both in place."""
        out2 = output if output.dim() == 2 else output.view(-1, output.shape[-1])
        codes, scales = _codes(x.reshape(-1, x.shape[-1]))
        ops.gemm_fp8_block_nt(out2, codes, scales, layer.weight.data, layer.weight_scale.data, max_cus)
        if bias is not None:
            out2.add_(bias)
        return output


def _codes(x: torch.Tensor, activation: Optional[str] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """`ops.quant_fp8_groups` into new tensors."""
    rows, channels = x.shape[0], x.shape[1] // (1 if activation is None else 2)
    codes = torch.empty((rows, channels), dtype=ops.FP8_DTYPE, device=x.device)
    scales = ops.fp8_group_scales(rows, channels, x.device)
    ops.quant_fp8_groups(codes, scales, x, activation)
    return codes, scales


class FeedForward(nn.Module):
    """One rank's feed-forward block as the layer schedules' ``mlp_fn``: reads the normalised rows in
    ``hidden_states`` and leaves the down projection's partial sum there, for the schedule to reduce.
    ``intermediate_size`` is the whole model's; ``gemm_cus`` is the compute-unit budget of the down projection.

    The result takes its input's place in memory, so no gradient can be recorded: where grad mode is on and the rows or a
    weight require one, the call raises.  `GatedLinear` is the projection with its gradient.

    ``to_fp8_blocks()`` turns both weights into e4m3 codes with a scale for each block of 128 x 128; a call is then
    codes of the rows, the merged projection, activation, product and codes in one pass, the down projection."""

    def __init__(self, hidden_size: int, intermediate_size: int, activation: str = "silu", *, tp_rank: int = 0,
                 tp_size: int = 1) -> None:
        super().__init__()
        self.gate_up = GatedLinear(hidden_size, intermediate_size, activation, tp_rank=tp_rank, tp_size=tp_size)
        self.down = RowParallelLinear(intermediate_size, hidden_size, bias=False, tp_rank=tp_rank, tp_size=tp_size)
        self.fp8 = False

    def to_fp8_blocks(self) -> "FeedForward":
        if not self.fp8:
            method = Fp8BlockLinearMethod()
            method.check(self.gate_up), method.check(self.down)
            for layer in (self.gate_up, self.down):
                method.code_weight(layer)
            self.fp8 = True
        return self

    def forward(self, hidden_states: torch.Tensor, gemm_cus: Optional[int] = None) -> torch.Tensor:
        ops._refuse_recording("FeedForward", "call it under torch.no_grad(), or train GatedLinear and a product of your own",
                              hidden_states, self.gate_up.weight, self.down.weight)
        if not self.fp8:
            inner = self.gate_up(hidden_states)
            self.down(inner, hidden_states, is_tokenweave=True, gemm_cus=gemm_cus)
            return hidden_states
        rows = hidden_states if hidden_states.dim() == 2 else hidden_states.view(-1, hidden_states.shape[-1])
        codes, scales = _codes(rows)
        both = torch.empty((rows.shape[0], self.gate_up.weight.shape[0]), dtype=rows.dtype, device=rows.device)
        ops.gemm_fp8_block_nt(both, codes, scales, self.gate_up.weight.data, self.gate_up.weight_scale.data)
        codes, scales = _codes(both, self.gate_up.activation)
        ops.gemm_fp8_block_nt(rows, codes, scales, self.down.weight.data, self.down.weight_scale.data, gemm_cus)
        return hidden_states

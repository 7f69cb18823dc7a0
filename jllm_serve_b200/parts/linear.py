"""out (+)= a @ W^T (+ bias): the matrix product every part uses, choosing the kernel by dtype and shape.

float32: always the CUDA-core kernel with true 32-bit products and sums (no tensor cores).
bfloat16: the tensor-core kernels where the shape fits them (K a multiple of 8), else the same CUDA-core kernel
reading bfloat16 and summing in float32. Weights are [out, in] row-major in the checkpoint
(src/main/java/org/robomiri/jllm/cpu/CpuMatmul.java:390-396); for the tensor-core kernels a bfloat16 weight is
PACKED once, when the part is built (`ops.pack_weight`: tiles of 128 rows x 64 k in the shared-memory image the
tensor cores read, so a tile is one contiguous bulk copy), and the row-major copy is let go.

With `Runtime.weights` "int8" the layers' products are `Int8Linear`s instead: weight and rows in 8-bit integers, a scale a weight row
and a scale a token (`ops.gemm_int8`). Half the bytes of a bfloat16 weight, on tensor cores of twice the rate. With "fp8" they are `Fp8Linear`s:
both in 8-bit floating point, with a scale for every 128 x 128 of a weight and every 128 values of a row (`ops.gemm_fp8`).
"""
from __future__ import annotations

import torch

from ..csrc import ops


class Linear:
    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, keep_plain: bool = False):
        """`keep_plain`: the row-major matrix stays beside the packed one (it is someone else's too: an embedding
        table that serves as the head is gathered row by row)."""
        assert weight.dim() == 2 and weight.is_contiguous()
        self.bias = bias
        self.out_features, self.in_features = weight.shape
        self.packed = None
        if weight.dtype == torch.bfloat16 and weight.is_cuda and self.in_features % 8 == 0 and self.in_features >= 8:
            self.packed = ops.pack_weight(weight)
        self.weight = weight if (self.packed is None or keep_plain) else None

    def rows(self, lo: int, hi: int) -> "Linear":
        """The product with rows [lo, hi) of the weight only (a view where the packed tiles allow it, else a copy)."""
        bias = self.bias[lo:hi] if self.bias is not None else None
        if self.packed is None:
            return Linear(self.weight[lo:hi].contiguous(), bias)
        out = Linear.__new__(Linear)
        out.bias, out.out_features, out.in_features, out.weight = bias, hi - lo, self.in_features, None
        if lo % 128 == 0:
            out.packed = ops.PackedWeight(self.packed.data[lo // 128: -(-hi // 128)], hi - lo, self.in_features)
        else:
            out.packed = ops.pack_weight(self.packed.unpack()[lo:hi].contiguous())
        return out

    def forward(self, a: torch.Tensor, out: torch.Tensor, accumulate: bool = False, swiglu: bool = False,
                relu2: bool = False) -> None:
        """a [rows, in] (compute dtype) -> out [rows, out]; `accumulate` adds into out (the float32 residual);
        `relu2` stores max(result, 0)^2 (behind the bias) instead of the result;
        `swiglu`: the weight's rows are interleaved gate / up blocks and out is [rows, out / 2]."""
        if a.shape[0] == 0:
            return
        if relu2:
            if accumulate or swiglu:
                raise ops.KernelError("relu squared in a product's epilogue goes with a stored result only")
            accumulate = ops.EPILOGUE_RELU2
        if self.packed is not None and ops.gemm_bf16_fits(a, self.packed, out):
            ops.gemm_bf16(a, self.packed, out, self.bias, accumulate, swiglu)
        elif swiglu:
            raise ops.KernelError("the fused SwiGLU epilogue exists in the tensor-core kernels only")
        else:
            weight = self.weight if self.weight is not None else self.packed.unpack()
            ops.gemm_plain(a, weight, out, self.bias, accumulate)


class Int8Linear:
    """`Linear` in 8-bit integers. The rows come in 8 bits from a norm that rounds them itself (`ops.Int8Rows`), or as a part's bfloat16
    result, which is rounded here. `glu`: the weight's rows are all gate rows, then all up rows, for `forward(swiglu=...)`."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, runtime, glu: bool = False):
        assert weight.dim() == 2
        self.bias, self.rt = bias, runtime
        self.out_features, self.in_features = weight.shape
        self.packed = ops.quantize_weight_int8(weight, glu)

    def rows(self, lo: int, hi: int) -> "Int8Linear":
        """The product with rows [lo, hi) of the weight only."""
        out = Int8Linear.__new__(Int8Linear)
        out.bias, out.rt = (self.bias[lo:hi] if self.bias is not None else None), self.rt
        out.out_features, out.in_features = hi - lo, self.in_features
        out.packed = ops.pack_int8(self.packed.unpack()[lo:hi].contiguous(), self.packed.scale[lo:hi].contiguous())
        return out

    def forward(self, a, out: torch.Tensor, accumulate: bool = False, swiglu=False, relu2: bool = False) -> None:
        """a [rows, in]: `ops.Int8Rows`, or float32 or bfloat16 rows; otherwise as `Linear.forward`."""
        if a.shape[0] == 0:
            return
        if not isinstance(a, ops.Int8Rows):
            rows8 = self.rt.int8_rows("product_input", self.in_features, a.shape[0])
            ops.quantize_int8(a, rows8)
            a = rows8
        ops.gemm_int8(a, self.packed, out, self.bias, ops.EPILOGUE_RELU2 if relu2 else accumulate, swiglu)


class Fp8Linear:
    """`Linear` in 8-bit floating point. The rows come as a norm's or a part's bfloat16 result and are rounded here. `glu`: the weight's rows are all
    gate rows, then all up rows, for `forward(swiglu=...)`."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None, runtime, glu: bool = False):
        assert weight.dim() == 2
        self.bias, self.rt = bias, runtime
        self.out_features, self.in_features = weight.shape
        self.packed = ops.quantize_weight_fp8(weight, glu)

    def rows(self, lo: int, hi: int) -> "Fp8Linear":
        """The product with rows [lo, hi) of the weight only (a view of its tiles)."""
        out = Fp8Linear.__new__(Fp8Linear)
        out.bias, out.rt = (self.bias[lo:hi] if self.bias is not None else None), self.rt
        out.out_features, out.in_features = hi - lo, self.in_features
        out.packed = self.packed.take_rows(lo, hi)
        return out

    def forward(self, a: torch.Tensor, out: torch.Tensor, accumulate: bool = False, swiglu=False, relu2: bool = False) -> None:
        """a [rows, in]: float32 or bfloat16 rows; otherwise as `Linear.forward`."""
        if a.shape[0] == 0:
            return
        rows8 = self.rt.fp8_rows("product_input", self.in_features, a.shape[0])
        ops.quantize_fp8(a, rows8)
        ops.gemm_fp8(rows8, self.packed, out, self.bias, ops.EPILOGUE_RELU2 if relu2 else accumulate, swiglu)


LOW_BIT = {"int8": Int8Linear, "fp8": Fp8Linear}          # what a layer's products are with `Runtime.weights`


def layer_linear(weight: torch.Tensor, bias: torch.Tensor | None, runtime):
    """The product of a layer's part with a weight [out, in], as the runtime has them."""
    return LOW_BIT[runtime.weights](weight, bias, runtime) if runtime.weights else Linear(weight, bias)

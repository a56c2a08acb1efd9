"""Blackwell (sm_100a) block-scaled GEMM: NVFP4 / MXFP8 operands, fp32 accumulation in
tensor memory, bf16 or fused-NVFP4 output; dense, batched, grouped (MoE) and
tensor-parallel forms.  The Python surface keeps the shape of the CUTLASS Python
Operator API; the work is done by hand-written CUDA behind a C ABI
(``include/bsgemm.h``, loaded by ``cutlass_b200.lib``)."""
from .activation import (ActivationCheckpoint, checkpoint_activation, checkpoint_activation_backward, checkpointed_activation)
from .arguments import (DenseTensor, EpilogueDescriptor, GemmArguments, GemmProblemSize, GroupedGemmArguments,
                        Mxfp8Quant, Nvfp4Quant, ScaledOperand, ScaleMode, ScaleSwizzleMode)
from .int8 import int8_linear, quantize_int8
from .operator import (AllocationRequirement, BlockScaledGemmOperator, CompiledArtifact,
                       GroupedBlockScaledGemmOperator, GroupedInt8GemmOperator, Int8GemmOperator, NativeProvider, Operator, OperatorMetadata, Workspace, all_operators,
                       get_operators, to_cuda_stream)
from .quantize import quantize_blockscaled
from .routing import Routing, route_tokens, route_tokens_backward
from .status import Status

__all__ = [
    "ActivationCheckpoint", "AllocationRequirement", "BlockScaledGemmOperator", "CompiledArtifact", "DenseTensor", "EpilogueDescriptor",
    "GemmArguments", "GemmProblemSize", "GroupedBlockScaledGemmOperator", "GroupedGemmArguments", "GroupedInt8GemmOperator", "Int8GemmOperator", "Mxfp8Quant", "NativeProvider", "Nvfp4Quant",
    "Operator", "OperatorMetadata", "Routing", "ScaleMode", "ScaleSwizzleMode", "ScaledOperand", "Status", "Workspace",
    "all_operators", "checkpoint_activation", "checkpoint_activation_backward", "checkpointed_activation", "get_operators", "int8_linear", "quantize_blockscaled", "quantize_int8", "route_tokens", "route_tokens_backward", "to_cuda_stream",
]
__version__ = "0.1.0"

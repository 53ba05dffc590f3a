"""megacu_b200: B200-native (sm_100a) fused GEMM + allreduce / reduce-scatter.

The product is the native library ``lib/libmegacu_b200.so`` behind the C ABI
in ``include/megacu_b200.h``; this package is its Python host mirror (ctypes)
plus the in-tree build. Importing it does not need a GPU; calling a launcher
does, and fails loudly if the native library is missing.
"""
from .api import (Fp4Gemm, Fp4Matrix, MegacuError, MlpChainProblem, MoeMlp, MoeProblem, Plan, Problem, Team, allgather_gemm, check,
                  co_resident_control_bytes, co_resident_status, env_team, local_exchange,
                  megacu_cuda_gemm_allreduce_f32_co_resident,
                  cuda_nvshmem_gemm_allreduce_phased_orchestrate, gemm_swiglu, mlp_chain,
                  mlp_chain_sizes, swiglu_events_bytes,
                  fp4_dequantize, fp4_events_bytes, fp4_gemm, fp4_gemm_swiglu, fp4_quantize,
                  fp4_sizes, moe_combine, moe_combine_grad, moe_dispatch, moe_mlp_fp4,
                  moe_mlp_workspace_bytes, moe_rows, moe_sort,
                  moe_workspace_bytes,
                  driver_view, events_bytes, events_counters, events_status, gemm_allreduce,
                  gemm_reduce_scatter, megacu_cuda_gemm_allreduce_phased_f32, plan, plan_pair, plan_tile,
                  tensor_from_pointer, torch_exchange, workspace_bytes)
from ._capi import (ALGO_AUTO, ALGO_ONE_SHOT, ALGO_TWO_SHOT, CTA_PAIRS_AUTO, CTA_PAIRS_OFF,
                    CTA_PAIRS_ON, DTYPE_BF16, DTYPE_F16, DTYPE_F32, FP4_MX, FP4_NV, MODE_ALLGATHER, MODE_ALLREDUCE, MODE_REDUCE_SCATTER, load)

__all__ = [
    "Fp4Gemm", "Fp4Matrix", "MegacuError", "MlpChainProblem", "MoeMlp", "MoeProblem", "Plan", "Problem", "Team", "allgather_gemm", "check",
    "co_resident_control_bytes", "co_resident_status", "env_team", "local_exchange",
    "megacu_cuda_gemm_allreduce_f32_co_resident",
    "cuda_nvshmem_gemm_allreduce_phased_orchestrate", "gemm_swiglu", "mlp_chain", "mlp_chain_sizes",
    "swiglu_events_bytes",
    "fp4_dequantize", "fp4_events_bytes", "fp4_gemm", "fp4_gemm_swiglu", "fp4_quantize",
    "fp4_sizes", "moe_combine", "moe_combine_grad", "moe_dispatch", "moe_mlp_fp4",
    "moe_mlp_workspace_bytes", "moe_rows", "moe_sort",
    "moe_workspace_bytes", "DTYPE_BF16", "DTYPE_F16", "DTYPE_F32", "FP4_MX", "FP4_NV",
    "driver_view", "events_bytes", "events_counters", "events_status", "gemm_allreduce",
    "gemm_reduce_scatter", "megacu_cuda_gemm_allreduce_phased_f32", "plan", "plan_pair", "plan_tile", "tensor_from_pointer",
    "torch_exchange", "workspace_bytes", "ALGO_AUTO", "ALGO_ONE_SHOT", "ALGO_TWO_SHOT",
    "CTA_PAIRS_AUTO", "CTA_PAIRS_OFF", "CTA_PAIRS_ON", "MODE_ALLGATHER", "MODE_ALLREDUCE", "MODE_REDUCE_SCATTER", "load",
]

"""lloom_amd -- MI355X (gfx950) quantized-weight matmul for lloom.

The compute lives in ``liblloom_hip.so`` (hand-written HIP kernels behind the
C ABI of ``include/lloom_hip.h``).  This package is the host-side mirror of
lloom-tensor's ``quantized`` surface (``QTensor``, ``QMatMul``,
``GgmlDType``; lloom-tensor/src/quantized/mod.rs) over that ABI, used by the
tests and the benchmark.  PyTorch only provides device memory and streams.
There is no CPU fallback: without the built library every call raises.
"""
from .lib import LloomHipError, lib, lib_path  # noqa: F401
from . import gguf_file  # noqa: F401
from .quantized import (  # noqa: F401
    GgmlDType,
    MoeArm,
    MvStore,
    QMatMul,
    QTensor,
    dequantize,
    quantize_act,
    synth_normal,
    synth_uniform,
)
from .paged import (  # noqa: F401
    PagedCache,
    PagedPlan,
    paged_append,
    paged_attention,
    paged_attention_workspace_bytes,
    paged_check,
    paged_plan,
)
from .fp8 import (  # noqa: F401
    MMA_F16,
    MMA_FP8,
    ExpertPlan,
    expert_plan,
    fp8_grouped_matmul,
    fp8_matmul,
    fp8_quantize,
    fp8_quantize_weight,
    fp8_silu_mul,
    fp8_workspace_bytes,
    set_fp8_mma,
)

"""nanoep_amd: expert-parallel dispatch / combine for one rank on one MI355X (PyTorch-ROCm).

The buffer's public names are those of the reference package `nano_ep`, so `from nanoep_amd import
CudaBuffer, EPConfig` is the only line a caller changes; `Buffer` is a shorter alias.
The expert layer around it in 8 bits (`rms_norm_fp8`, `experts_gated`, `experts_linear`, `combine_weighted`) has no
counterpart there: see `operators`.
"""

from . import buffer as _buffer
from . import handles as _handles
from .config import EPConfig
from .operators import (
    Fp8Rows,
    Fp8Weight,
    RmsNormResult,
    combine_weighted,
    combine_weighted_backward,
    dispatch_rows,
    experts_gated,
    experts_linear,
    fp8_payload_width,
    quantize_weight,
    rms_norm_fp8,
)

__version__ = "0.1.0"

CudaBuffer = _buffer.CudaBuffer
Buffer = _buffer.Buffer
CudaEvent = _handles.CudaEvent
NativeLayout = _handles.NativeLayout
NativeHandle = _handles.NativeHandle
NativeDispatchResult = _handles.NativeDispatchResult
NativeCombineResult = _handles.NativeCombineResult

__all__ = sorted(
    ["Buffer", "CudaBuffer", "CudaEvent", "EPConfig", "NativeLayout", "NativeHandle", "NativeDispatchResult", "NativeCombineResult",
     "Fp8Rows", "Fp8Weight", "RmsNormResult", "combine_weighted", "combine_weighted_backward", "dispatch_rows", "experts_gated",
     "experts_linear", "fp8_payload_width", "quantize_weight", "rms_norm_fp8"]
)

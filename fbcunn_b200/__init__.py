"""B200-native FFT spatial convolution behind the nn.SpatialConvolutionFBFFT interface.

    capi        ctypes binding of the C ABI (include/fbfftconv.h)
    module      SpatialConvolutionFBFFT (and its Gemm-variant name), FFTWrapper, CuBLASWrapper:
                host-side mirrors of the reference's Lua modules
    tiled       SpatialConvolutionFFTTiled: the same convolution on tiles of the image
    tuned       SpatialConvolution: times the candidates on first use and keeps the fastest
    adamw       AdamW: one optimizer step over many tensors, moments in 32 bits or in 8
    recurrence  GatedLinearRecurrence: a gated linear recurrence along sequences
    residual_norm  GatedResidualNorm: the norms around a residual block, its gate and the residual sum
    lua/        the LuaJIT FFI file a Torch7 installation would load
    csrc/       CUDA kernels (sm_100a) and the C ABI
"""
from . import capi  # noqa: F401
from .adamw import AdamW  # noqa: F401
from .module import CuBLASWrapper, FFTWrapper, SpatialConvolutionFBFFT, SpatialConvolutionFBFFTGemm  # noqa: F401
from .recurrence import GatedLinearRecurrence  # noqa: F401
from .residual_norm import GatedResidualNorm  # noqa: F401
from .tiled import SpatialConvolutionFFTTiled  # noqa: F401
from .tuned import SpatialConvolution  # noqa: F401

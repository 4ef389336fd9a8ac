"""B200-native mLSTM kernels behind the reference project's operator API.

    from <this package>.mlstm_matmul import Triton_mLSTM, mlstm_matmul
    from <this package>.mlstm_scan import mlstm_scan

and the operators around a mixer: ``short_convolution``, ``state_space_scan`` (a selective state space scan, a recurrent mixer
with one decay per channel and state) and ``residual_rms_norm``.

The compute lives in libmlstm_b200.so (CUDA for sm_100a, C ABI in include/mlstm_b200.h), loaded on
first use.  There is no CPU, PyTorch or Triton fallback: without the built library calls raise.
"""
from . import _lib
from .mlstm_matmul import Triton_mLSTM, fp32_math_mode, mlstm_matmul, mlstm_matmul_backward, mlstm_matmul_forward
from .mlstm_scan import mlstm_scan, output_gate_backward, output_gate_forward
from .mlstm_chunkwise import mlstm_chunkwise, mlstm_chunkwise_backward, mlstm_chunkwise_sequence_parallel
from .short_convolution import short_convolution, short_convolution_backward
from .state_space import state_space_scan, state_space_scan_backward, state_space_scan_forward
from .residual_norm import residual_rms_norm, residual_rms_norm_backward, residual_rms_norm_quantized
from .partition import shard_slices, slice_range, unshard_slices

__all__ = ["Triton_mLSTM", "mlstm_matmul", "mlstm_matmul_forward", "mlstm_matmul_backward", "fp32_math_mode", "mlstm_scan",
           "output_gate_forward", "output_gate_backward", "mlstm_chunkwise", "mlstm_chunkwise_backward",
           "mlstm_chunkwise_sequence_parallel", "short_convolution", "short_convolution_backward", "state_space_scan",
           "state_space_scan_forward", "state_space_scan_backward", "residual_rms_norm", "residual_rms_norm_backward",
           "residual_rms_norm_quantized",
           "slice_range", "shard_slices", "unshard_slices", "_lib"]

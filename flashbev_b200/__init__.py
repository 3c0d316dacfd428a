"""B200 (sm_100a) fused BEV pooling: the operator of yokosyun/FlashBEV's ``flashbevpool``
package on a hand-written CUDA library with a C ABI (include/fbev.h)."""
from .camera_attention import CameraAttention
from .flash_bevpool import (DepthSpec, DeviceStatus, FlashBEVPool, debug_indices, device_status, flash_bevpool,
                            forward_with_count)
from .query_ops import add_rms_norm, cross_attention, rotary_axes
from .sampling_vt import SamplingVT, create_projection_matrix

__all__ = ["FlashBEVPool", "flash_bevpool", "SamplingVT", "create_projection_matrix", "DepthSpec",
           "debug_indices", "forward_with_count", "cross_attention", "rotary_axes", "add_rms_norm",
           "CameraAttention", "device_status", "DeviceStatus"]

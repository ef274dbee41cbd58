"""Operators of image-transformer blocks on hand-written HIP kernels (libpixelsplat_ops.so), for fp32, bf16 and fp16
tensors on the GPU, each with its backward pass."""
from .group_norm import GroupNormAct, group_norm  # noqa: F401
from .gated_linear import gated_linear  # noqa: F401
from .relative_attention import (RelativePositionBias, relative_attention, relative_bucket_count,  # noqa: F401
                                 relative_buckets)

from .gemm_rcr_i8 import gemm_rcr_i8  # noqa: F401
from .quantize_rows import quantize_rows  # noqa: F401
from .residual_norm import residual_norm  # noqa: F401

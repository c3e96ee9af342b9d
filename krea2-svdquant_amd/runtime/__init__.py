from .linear import SVDQuantLinear, SVDQuantLoRAAdapter
from .mx_linear import MXLinear
from .fp8_linear import FP8Linear

__all__ = ["FP8Linear", "MXLinear", "SVDQuantLinear", "SVDQuantLoRAAdapter"]

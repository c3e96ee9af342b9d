from .linear import SVDQuantLinear, SVDQuantLoRAAdapter
from .mx_linear import MXLinear

__all__ = ["MXLinear", "SVDQuantLinear", "SVDQuantLoRAAdapter"]

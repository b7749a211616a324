from .layer import BCSRGraphConv, BCSRSPMMFunction  # noqa: F401
from .losses import distillation_loss, linear_cross_entropy  # noqa: F401

from .layer import BCSRSPMMFunction, BCSRGraphConv  # noqa: F401
from .head import LinearHead, linear_cross_entropy, linear_distill  # noqa: F401

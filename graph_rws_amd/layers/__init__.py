from .layer import BCSRSPMMFunction, BCSRGraphConv  # noqa: F401
from .head import linear_cross_entropy, linear_distill  # noqa: F401

from .layer import BCSRSPMMFunction, BCSRGraphConv  # noqa: F401
from .head import LinearHead, linear_cross_entropy, linear_distill  # noqa: F401
from .logp import LogProbs, linear_log_probs, log_probs  # noqa: F401

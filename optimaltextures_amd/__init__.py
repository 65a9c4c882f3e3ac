"""optimaltextures_amd — MI355X-native sliced-optimal-transport inner loop of JCBrouwer/OptimalTextures.

Same call surface as the reference's hot path (optex.py::optimal_transport, random_rotation; histmatch.py::hist_match,
cdf_match, interp), implemented as hand-written HIP kernels for gfx950 behind the C ABI in include/optex.h, and the layer
operators of a learned block on channels-last maps (group_norm_act, linear_act), with gradients."""
from .histmatch import cdf_match, hist_match, interp  # noqa: F401
from .layers import group_norm_act, linear_act  # noqa: F401
from .optex import optimal_transport, random_rotation  # noqa: F401

__all__ = ["optimal_transport", "random_rotation", "hist_match", "cdf_match", "interp", "group_norm_act", "linear_act"]

"""``ops.ttt_linear`` / ``ops.ttt_mlp`` with the reference's signatures (ops/__init__.py:1-2),
computed by the sm_100a kernels (forward and backward) instead of a Python scan, and the
selective state space scan with its short causal convolution beside them."""

from ops.ttt_linear import ttt_linear  # noqa: F401
from ops.ttt_mlp import ttt_mlp  # noqa: F401
from ops.selective_scan import selective_scan, selective_scan_step  # noqa: F401
from ops.causal_conv1d import causal_conv1d, causal_conv1d_step  # noqa: F401

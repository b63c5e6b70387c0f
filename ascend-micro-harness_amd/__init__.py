"""MI355X-native TurboQuant TQ4 quantised-KV hot path.

The package directory is not an importable identifier; load it with
``__graft_entry__.package()`` (importlib, registered as
``ascend_micro_harness_amd``). The compute lives in libtq4.so (HIP kernels
for gfx950 behind the C ABI of include/); ``tq4`` is the host mirror, ``kv8``
that of the 8-bit cache, and ``torch_ops`` registers them as the
``torch.ops.tq4`` operators.
"""
from .tq4 import *  # noqa: F401,F403
from .kv8 import *  # noqa: F401,F403
from . import kv8 as _kv8
from . import tq4 as _tq4

__all__ = _tq4.__all__ + _kv8.__all__
from . import torch_ops  # noqa: F401  (registers torch.ops.tq4.*)

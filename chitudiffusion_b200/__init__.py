"""B200-native attention hot path for ChituDiffusion-style DiT inference.

Public surface (mirrors the reference's attention-backend and parallel API):

* ``B200AttnBackend``            - per-rank backend callable (``infer.attn_type: b200``)
* ``PagedKVCache``               - paged key/value cache in 16 or 8 bits, appended to and attended over
* ``ops``                        - operator-level calls into libchitu_b200.so
"""

from .attention import B200AttnBackend, BACKEND_NAME  # noqa: F401
from .kv_cache import PagedKVCache  # noqa: F401
from . import ops  # noqa: F401

__all__ = ["B200AttnBackend", "BACKEND_NAME", "PagedKVCache", "ops"]

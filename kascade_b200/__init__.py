"""kascade_b200 — B200 (sm_100a) implementation of the Kascade sparse-attention hot path.

``EfficientKascadeStrategy`` is the drop-in for the reference's strategy of the same name; the
kernels live in ``libkascade_b200.so`` (C ABI in ``include/kascade_b200.h``), built in-tree by
``python -m kascade_b200.build``.
"""
from .strategy import (  # noqa: F401
    EfficientKascadeStrategy, Strategy, int4_kv_cache, rope_axis_map, topk_budget)

__version__ = "0.1.0"

"""pack3d_amd: the PACK3D attention layer of amilworks/Pack3D on AMD MI355X (gfx950).

Public API mirrors ``pack3d`` (``src/pack3d/__init__.py``) with the ``hip``
backend: ``PACK3DAttention``, ``Pack3DGeometry``, ``TokenLayout``,
``build_layout``, ``prepare_geometry``, and the core ``pack3d_hip``
(the contract of ``pack3d_reference`` / ``pack3d_streamed``).  Around the layer:
``block_norm`` and ``block_residual`` (with ``Norm``), ``counter_dropout``, and
``apply_rotary`` with ``rotary_frequencies`` and ``RotaryEncoding``.
"""
from .attention import PACK3DAttention
from .block import Norm, block_norm, block_residual
from .core import pack3d_hip, pack3d_hip_rope
from .dropout import counter_dropout
from .geometry import (Pack3DGeometry, TokenLayout, adopt_layout, build_layout, grid_coordinates, grid_tag,
                       prepare_geometry)
from .rope import balanced_pairs
from .rotary import RotaryEncoding, apply_rotary, rotary_frequencies

__version__ = "0.1.0"
__all__ = ["Norm", "PACK3DAttention", "Pack3DGeometry", "RotaryEncoding", "TokenLayout", "adopt_layout",
           "apply_rotary", "balanced_pairs", "block_norm", "block_residual", "build_layout", "counter_dropout",
           "grid_coordinates", "grid_tag", "pack3d_hip", "pack3d_hip_rope", "prepare_geometry", "rotary_frequencies"]

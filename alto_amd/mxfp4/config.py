"""Recipe-level configuration of the low-precision training ops (alto/kernels/dispatch/config.py:10-51)."""
from __future__ import annotations

from dataclasses import dataclass, fields
from typing import Literal

import torch


@dataclass(unsafe_hash=True, kw_only=True, slots=True)
class TrainingOpConfig:
    precision: Literal["mxfp4", "blockwise_fp8"] = "mxfp4"   # (the options below are MXFP4's; blockwise_fp8 has none and refuses any that is set)
    use_2dblock_x: bool = False
    use_2dblock_w: bool = True
    use_hadamard: bool = True
    use_sr_grad: bool = True
    use_dge: bool = False
    clip_mode: Literal["none", "static", "dynamic"] = "none"
    two_level_scaling: Literal["none", "tensorwise", "blockwise"] = "none"
    use_uos: bool = False

    def __post_init__(self):
        if self.precision not in ("mxfp4", "blockwise_fp8"):
            raise ValueError(f"this build implements precision='mxfp4' and 'blockwise_fp8', got {self.precision!r}")
        if self.clip_mode not in ("none", "static", "dynamic"):
            raise ValueError(f"Invalid clip mode: {self.clip_mode}")
        changed = [f.name for f in fields(self) if f.name != "precision" and getattr(self, f.name) != f.default]
        if self.precision == "blockwise_fp8" and changed:
            raise ValueError(f"precision='blockwise_fp8' has no options: {', '.join(changed)} would have no effect")


torch.serialization.add_safe_globals([TrainingOpConfig])   # dispatch/config.py:57

"""efgs -- MI355X-native fused-appearance differentiable Gaussian rasterizer.

Drop-in for the reference package's exports (FasterGSVDACudaBackend/__init__.py:14-23): diff_rasterize,
rasterize, update_pruning_scores, RasterizerSettings, initialize_appearance, initialize_residual_mlp,
FusedAdam, relocation_adjustment, add_noise. `efgs.tcnn` supplies the tiny-cuda-nn network class the appearance plugin
builds its residual MLP with (Appearance/Base.py:23, Appearance/Neural.py:13,40-66). Beside the reference's surface: `embedding`
(rows of a table by index, for shared appearance codes), `AdamW` (many tensors, 32-bit or 8-bit states) and `grad_norm`. The compute path is libefgs_hip.so
(hand-written HIP kernels for gfx950, hipRTC-specialised preprocess); importing without the built library raises
ImportError.
"""
from .rasterization import (diff_rasterize, rasterize, update_pruning_scores, RasterizerSettings, initialize_appearance,
                            initialize_residual_mlp)
from .adam import FusedAdam
from .adamw import AdamW, grad_norm
from .densification import relocation_adjustment, add_noise
from .embeddings import embedding
from . import tcnn

__all__ = ['diff_rasterize', 'rasterize', 'update_pruning_scores', 'RasterizerSettings', 'initialize_appearance',
           'initialize_residual_mlp', 'FusedAdam', 'relocation_adjustment', 'add_noise', 'tcnn', 'AdamW',
           'grad_norm', 'embedding']

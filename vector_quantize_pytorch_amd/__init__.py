"""vector_quantize_pytorch_amd -- MI355X-native drop-in for the VectorQuantize / ResidualVQ forward
path of lucidrains/vector-quantize-pytorch.  HIP kernels: csrc/vqhip.hip, C ABI:
include/vqhip.h."""
from .codebook import Codebook
from .vector_quantize import VectorQuantize, LossBreakdown
from .residual_vq import ResidualVQ, GroupedResidualVQ
from .sim_vq import SimVQ, ResidualSimVQ
from .callers import HierarchicalVQ, RandomProjectionQuantizer
from .beam import BeamStep, beam_reorder, beam_select
from .norms import GroupNorm, group_norm
from .grads import clip_grad_norm_, clip_grads

__all__ = ["VectorQuantize", "ResidualVQ", "GroupedResidualVQ", "SimVQ", "ResidualSimVQ", "RandomProjectionQuantizer", "HierarchicalVQ", "Codebook", "LossBreakdown",
           "BeamStep", "beam_select", "beam_reorder", "GroupNorm", "group_norm", "clip_grads", "clip_grad_norm_"]

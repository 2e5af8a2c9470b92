"""test1_b200: a Blackwell-native layer-sliding offload trainer.

Public API (same names as the SlideFSDP reference):
    SlideFSDPConfig, SlideFSDP, LayerAdam, SlidingCheckpoint
and for training on preferences or sampled answers:
    PreferenceObjective, PolicyObjective
"""
from .config import SlideFSDPConfig
from .optim.layer_adam import LayerAdam

__all__ = ["SlideFSDPConfig", "SlideFSDP", "LayerAdam", "SlidingCheckpoint", "LlamaConfig",
           "LlamaForCausalLM", "PreferenceObjective", "PolicyObjective"]
__version__ = "0.1.0"


def __getattr__(name):
    if name == "SlideFSDP":
        from .slide_fsdp import SlideFSDP

        return SlideFSDP
    if name == "SlidingCheckpoint":
        from .sliding_checkpoint import SlidingCheckpoint

        return SlidingCheckpoint
    if name in ("PreferenceObjective", "PolicyObjective"):
        from . import objectives

        return getattr(objectives, name)
    if name in ("LlamaConfig", "LlamaForCausalLM"):
        from .models import llama

        return getattr(llama, name)
    raise AttributeError(name)

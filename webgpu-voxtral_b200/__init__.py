"""B200-native Voxtral decode path: backbone decode loop + flow-matching transformer.

The compute lives in libvoxtral_b200.so (hand-written CUDA for sm_100a behind the C ABI
of include/voxtral_b200.h); this package is the host-side mirror of the reference's
VoxtralEngine API, and ops.py offers the serving operators on torch tensors.  The directory name is not a Python identifier, so import it with
importlib:

    vx = importlib.import_module("webgpu-voxtral_b200")
"""
from .engine import (TTSResult, VoxtralEngine, VoxtralError, default_config, header_symbols, library_path,
                     load_library, nccl_unique_id, tp_init)
from . import synth

__all__ = ["VoxtralEngine", "VoxtralError", "TTSResult", "default_config", "header_symbols", "library_path",
           "load_library", "nccl_unique_id", "tp_init", "synth", "rope_append_kv", "shared_prefix_attention",
           "shared_prefix_attention_workspace", "sample_logits"]


def __getattr__(name):
    # the operators on torch tensors (ops.py) import torch, which the engine does not need
    if name in ("rope_append_kv", "shared_prefix_attention", "shared_prefix_attention_workspace", "sample_logits"):
        from . import ops
        fn = globals()[name] = getattr(ops, name)
        return fn
    raise AttributeError(f"module {__name__!r} has no attribute {name!r}")

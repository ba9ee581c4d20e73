"""sdmchat_amd -- the run-time SDM mixer (RunTimeSdm) of SDMCHAT on AMD MI355X (gfx950).

``RunTimeSdm``      drop-in nn.Module (same constructor, state_dict and forward signature as the reference's)
``TrainedSdm``      drop-in for the trained product-key table layer (same constructor and state_dict)
``OneSdmLM``        the whole language model around the mixer (same constructor and state_dict; no archive)
``core``            torch-facing wrappers of the C ABI (addressing, the SDM core)
``synthetic``       seeded synthetic parameters and inputs of the layer workloads
``DecodeGraph``, ``ForwardGraph``  OneSdmLM.step and OneSdmLM.forward at fixed shapes, captured in HIP graphs
``TokenRules``      penalties for repeated tokens, a bias and a grammar mask on a decode loop's logits
``AdamW``           the optimiser of a training step: all tensors in a few launches, clipped, moments in 32 or in 8 bits
``build``           compiles ``csrc/*.hip`` into ``lib/libsdm_rt.so``
"""
from .runtime_sdm import RMSNorm, RunTimeSdm  # noqa: F401
from .trained_sdm import TrainedSdm  # noqa: F401
from .model import DecodeGraph, ForwardGraph, ModelDecodeState, OneSdmLM, TokenRules, decode_state_bytes  # noqa: F401
from .optim import AdamW  # noqa: F401

"""ppo_amd — MI355X-native experience path of flawedmatrix/ppo (rollout buffer -> GAE/returns ->
advantage standardisation -> shuffled minibatch gather) behind the reference's own interface.

Compute lives in libppo_xp.so (hand-written HIP for gfx950, C ABI in include/ppo_xp.h).  The
classes here mirror ppo/src/common/buffer.rs and ppo/src/model/data.rs.  There is no CPU path.
"""
import importlib
import importlib.util

from ._lib import GAE_ASSOC, GAE_NO_PACK, GAE_SEQUENTIAL, PpoXpError, PpoXpPanic, gae_chunk
from .buffer import ExperienceBuffer, device_tensor, pinned_empty
from .data import ExperienceBatch, ExperienceBatcher, ExperienceBatcherIterator, HostBatch
from .runner import RewardNormalizer

__all__ = ["ExperienceBuffer", "ExperienceBatch", "ExperienceBatcher", "ExperienceBatcherIterator", "HostBatch", "RewardNormalizer", "PpoXpError",
           "PpoXpPanic", "GAE_SEQUENTIAL", "GAE_ASSOC", "GAE_NO_PACK", "gae_chunk", "device_tensor", "pinned_empty"]

# the operators on torch tensors, imported with torch on first use (the rest of the package works without torch)
_ON_TENSORS = {"PolicyLoss": "policy", "action_stats": "policy", "policy_loss": "policy", "shape_logits": "policy",
               "shape_logits_backward": "policy", "QuantizedRows": "quant"}
if importlib.util.find_spec("torch"):
    __all__ += list(_ON_TENSORS)


def __getattr__(name):
    if name not in _ON_TENSORS:
        raise AttributeError(f"module {__name__!r} has no attribute {name!r}")
    value = globals()[name] = getattr(importlib.import_module("." + _ON_TENSORS[name], __name__), name)
    return value

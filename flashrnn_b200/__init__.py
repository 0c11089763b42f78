"""B200-native (sm_100a) backend for FlashRNN's fused recurrence.

Public surface = the reference's: ``flashrnn``, ``FlashRNNConfig``, ``flashrnn_torch``
(flashrnn/__init__.py:2-5 of the reference), running hand-written CUDA through a C ABI.
"""

from .functional import BACKEND, SIZES, FlashRNNConfig, flashrnn, flashrnn_torch, poll_errors
from .linear import flashrnn_linear
from .prepared import PreparedSequence
from .projection import flashrnn_projected, fused_projection, input_projection

__all__ = ["BACKEND", "SIZES", "FlashRNNConfig", "PreparedSequence", "flashrnn", "flashrnn_linear", "flashrnn_projected",
           "flashrnn_torch", "fused_projection", "input_projection", "poll_errors"]

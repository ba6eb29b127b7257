"""Token mixers that a hybrid stack sets beside its FLARE layers.

Each has the three faces of a FLARE layer: a differentiable call over whole sequences (of
packed documents, with ``document_ids``), a prefill that continues a cached state, and a
single-token decode that updates it in place.  The reference has no counterpart.  Attention's
queries and keys may be given rotary positions, and its cache may be held in 8 or 4 bits.

``document_ids`` and lengths are used as int32: their values have to fit it.  Nothing is checked
that would have to wait for the GPU; what a value out of range does is said at each call.
"""
from .attention import SoftmaxAttention, softmax_attention, softmax_attention_decode, softmax_attention_prefill
from .convolution import ShortConvolution, short_convolution, short_convolution_decode, short_convolution_prefill
from .quantized import quantized_cache, quantized_cache_read, quantized_cache_write
from .rotary import RotaryPositions, rotary_frequencies, rotary_positions
from .scan import StateSpaceScan, state_space_scan, state_space_scan_decode, state_space_scan_prefill

__all__ = [
    "RotaryPositions",
    "ShortConvolution",
    "SoftmaxAttention",
    "StateSpaceScan",
    "quantized_cache",
    "quantized_cache_read",
    "quantized_cache_write",
    "rotary_frequencies",
    "rotary_positions",
    "short_convolution",
    "short_convolution_decode",
    "short_convolution_prefill",
    "softmax_attention",
    "softmax_attention_decode",
    "softmax_attention_prefill",
    "state_space_scan",
    "state_space_scan_decode",
    "state_space_scan_prefill",
]

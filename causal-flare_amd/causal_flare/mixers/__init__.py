"""Token mixers that a hybrid stack sets beside its FLARE layers.

Each has the three faces of a FLARE layer: a differentiable call over whole sequences (of
packed documents, with ``document_ids``), a prefill that continues a cached state, and a
single-token decode that updates it in place.  The reference has no counterpart.

``document_ids`` and lengths are used as int32: their values have to fit it.  Nothing is checked
that would have to wait for the GPU; what a value out of range does is said at each call.
"""
from .attention import SoftmaxAttention, softmax_attention, softmax_attention_decode, softmax_attention_prefill
from .convolution import ShortConvolution, short_convolution, short_convolution_decode, short_convolution_prefill
from .scan import StateSpaceScan, state_space_scan, state_space_scan_decode, state_space_scan_prefill

__all__ = [
    "ShortConvolution",
    "SoftmaxAttention",
    "StateSpaceScan",
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

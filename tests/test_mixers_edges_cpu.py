"""Refusals of the token mixers where an argument leaves its range, without a GPU."""
import ctypes

import pytest
import torch

import causal_flare as cf
from causal_flare import _lib


def t(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


@pytest.mark.parametrize("cap", [1e-50, 1e-31, 1e31, 1e39, float("nan"), -1.0])
def test_caps_out_of_range_are_refused(cap):
    """Below float32's range a cap would be 0, which stands for none."""
    qkv, cache = [t(2, 5, 4, 32)] * 3, {x: t(2, 9, 4, 32) for x in "kv"}
    for call in (lambda: cf.softmax_attention(*qkv, softcap=cap),
                 lambda: cf.softmax_attention_prefill(*qkv, cache, ints(2), softcap=cap),
                 lambda: cf.softmax_attention_decode(*(x[:, 0] for x in qkv), cache, ints(2), softcap=cap)):
        with pytest.raises(ValueError, match="softcap None or positive"):
            call()
    if cap in (1e-31, 1e31, -1.0):
        lib, P, nine = _lib.lib(), ctypes.c_void_p(4096), (ctypes.c_int64 * 9)(*[8] * 9)
        rc = lib.flare_attn_forward(P, P, P, nine, 1, 1, 4, 4, 4, 4, 64, 1.0, cap, None, 1, None, None, None, None, P, None,
                                    None, None, 0, None)
        assert rc == -1 and b"cap" in lib.flare_last_error()


@pytest.mark.parametrize("lengths", [None, [3, 4], 3])
def test_lengths_that_are_no_tensor_are_refused(lengths):
    qkv, cache = [t(2, 1, 4, 32)] * 3, {x: t(2, 9, 4, 32) for x in "kv"}
    for call in (cf.softmax_attention_prefill, cf.softmax_attention_decode):
        with pytest.raises(ValueError, match="expects a tensor in lengths"):
            call(*qkv, cache, lengths)
        with pytest.raises(ValueError, match=r"expects a tensor in cache\['v'\]"):
            call(*qkv, {"k": cache["k"], "v": None}, ints(2))


def test_parts_of_a_causal_forward_come_for_a_range_of_sizes():
    """Rows of 16 heads that are a round of 512 workgroups, and up to five quarters of one, run in two
    parts: the workspace holds each part's sums."""
    lib, H, D = _lib.lib(), 16, 128
    parts = lambda N: lib.flare_attn_forward_workspace_size(1, N, N, H, D, 1) // (N * H * (D + 4) * 4)
    assert [parts(N) for N in (4096, 4097, 4500, 5120)] == [2] * 4
    assert parts(5121) == 0 and parts(20000) == 0

"""The paged KV cache without a GPU: what the entry points refuse before they
touch a device, and the reference formulas against each other."""
import ctypes

import pytest
import torch

from onnx_runtime_dart_b200 import PagedKVCache, _lib
from tests import paged_reference as ref


def test_null_and_host_arguments_are_refused():
    L = _lib.load()
    c = _lib.PagedCacheStruct()
    p = ctypes.addressof(c)
    assert L.ort_cuda_paged_attention(None, p, 0, 64, 1, 1, 1, 0.0, 0.0, -1, 0, 0, 0) == \
        _lib.ERR_INVALID_ARG
    assert L.ort_cuda_paged_kv_append(None, p, 0, 0, 0, 64, 0, 64, 1, 0, 0, 0, 0, 0, 0, 0) == \
        _lib.ERR_INVALID_ARG


def test_struct_matches_the_header():
    """Five pointers, five 64-bit sizes, two 32-bit fields."""
    assert ctypes.sizeof(_lib.PagedCacheStruct) == 88


def test_cache_needs_device_tensors():
    s = ref.make(0, torch.float16, [1], [3], 4, 2, 64, 16, device="cpu")
    with pytest.raises(ValueError, match="CUDA tensor"):
        PagedKVCache(s["key"], s["value"], s["table"], s["cu"], s["past"])


def test_reference_window_and_prefix():
    """A window of one key gives that key's value; a window as long as the
    sequence changes nothing; a shared prefix holds the same rows."""
    new, past = [2, 1], [20, 33]
    s = ref.make(0, torch.float32, new, past, 4, 2, 8, 16, shared=17, device="cpu")
    one = ref.attention(s, new, past, 4, window=1)
    page = int(s["table"][1, 33 // 16])
    assert torch.allclose(one[2].view(2, 2, 8)[:, 0], s["value"][page, 33 % 16].double())
    assert torch.equal(ref.attention(s, new, past, 4), ref.attention(s, new, past, 4, window=34))
    assert torch.equal(s["key"][int(s["table"][0, 1]), 0], s["key"][int(s["table"][1, 1]), 0])

"""Host-side refusals of the decode-step operators that need no device."""
import numpy as np
import pytest


def test_qlinear4_refusals_without_a_device(nne):
    lib = nne.load()
    assert lib.nne_qlinear4_forward_dev(None, None, 1, 1, None, None) == 1
    assert lib.nne_qlinear4_forward_host(None, None, 1, 1, None) == 1
    assert lib.nne_qlinear4_create_from_i4(None, None, None, None, 1, 1, 32, None) == 1
    assert lib.nne_quantize_rows4_dev(None, None, 1, 1, 32, None, None, None) == 1
    assert lib.nne_qlinear4_destroy(None) == 0 and lib.nne_qlinear4_memory_bytes(None) == 0
    with pytest.raises(nne.InvalidArgument):
        nne.QLinear4.from_fields(np.zeros((2, 4), np.uint8), np.ones((2, 1), np.float32), None, 8, 2, 16)
    with pytest.raises(nne.InvalidArgument):
        nne.QLinear4.from_fields(np.zeros((2, 3), np.uint8), np.ones((2, 1), np.float32), None, 8, 2, 32)


def test_cache_refusals_without_a_device(nne):
    lib = nne.load()
    assert lib.nne_kv_cache_create(None, None, None) == 1
    assert lib.nne_kv_append_dev(None, None, None) == 1
    assert lib.nne_kv_cache_info(None, None, None, None) == 1
    assert lib.nne_kv_cache_destroy(None) == 0


def test_attention_refusals_without_a_device(nne):
    assert nne.load().nne_tree_attention_dev(None, None, None) == 1


def test_sampling_refusals_without_a_device(nne):
    assert nne.load().nne_sample_dev(None, None, None) == 1

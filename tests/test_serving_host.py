"""The serving operators' host side, without a GPU: the header's struct as
ctypes sees it, workspace sizes and their refusals, calls without a device,
and the float64 restatement on cases worked by hand."""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib
from oracle import serving_ref as S
from test_host import _c_layout


def test_logit_rules_match_the_header():
    fields = [f[0] for f in _lib.LogitRules._fields_]
    assert _c_layout("fh_logit_rules", fields) == [ctypes.sizeof(_lib.LogitRules)] + [
        getattr(_lib.LogitRules, f).offset for f in fields]


def refused(status, name, *args):
    out = ctypes.c_uint64(7)
    with pytest.raises(_lib.HipError) as e:
        _lib.call(name, *args, ctypes.byref(out))
    assert e.value.status == status and name in str(e.value) and out.value == 7


def test_paged_attention_workspace():
    size = _lib.paged_attention_workspace_bytes
    assert size(1, 32, 8, 128, 16, 20) > 0
    # a longer table or a larger batch never needs less
    for a, b in (((1, 32, 8, 128, 16, 20), (1, 32, 8, 128, 16, 8000)), ((1, 8, 8, 64, 32, 9), (64, 8, 8, 64, 32, 9))):
        assert size(*a) <= size(*b)
    # the largest shapes stay within reason
    assert size(1, 32, 8, 128, 64, 2 ** 24) < 1 << 30
    name, bad = "fh_paged_attention_workspace", _lib.ERR_INVALID_ARGUMENT
    for args in ((1, 32, 5, 128, 16, 4), (1, 0, 1, 128, 16, 4), (1, 4, 0, 64, 16, 4), (1, 4, 2, 64, 24, 4),
                 (1, 4, 2, 64, 0, 4), (1, 4, 2, 64, 16, 0), (-1, 4, 2, 64, 16, 4), (1, 4, 2, 64, 1 << 40, 4)):
        refused(bad, name, *args)
    refused(_lib.ERR_UNSUPPORTED, name, 1, 4, 2, 96, 16, 4)
    refused(_lib.ERR_INDEX_TOO_LARGE, name, 65536, 4, 2, 64, 16, 4)
    refused(_lib.ERR_INDEX_TOO_LARGE, name, 1, 4, 2, 64, 16, 1 << 27)
    # more steps than 32 bits count, over pages that sequences share
    refused(_lib.ERR_INDEX_TOO_LARGE, name, 1024, 4, 2, 64, 1 << 30, 1)
    assert _lib.load().fh_paged_attention_workspace(1, 4, 2, 64, 16, 4, None) == bad


@pytest.mark.parametrize("heads,kv,hd,page,width", [(32, 8, 128, 16, 8), (32, 8, 128, 64, 128), (24, 8, 128, 16, 2048),
                                                    (8, 1, 256, 32, 33)])
def test_attention_workspace_of_the_largest_batch_serves_smaller_ones(heads, kv, hd, page, width):
    sizes = [_lib.paged_attention_workspace_bytes(b, heads, kv, hd, page, width)
             for b in (0, 1, 2, 7, 64, 65, 512, 1023, 1024, 1025, 5000, 16000)]
    assert sizes == sorted(sizes)


def test_lora_workspace():
    assert _lib.lora_workspace_bytes(1, 64, 8) > 0
    assert _lib.lora_workspace_bytes(0, 64, 8) >= 0
    for rank in (0, 4, 12, 136, -8):
        refused(_lib.ERR_INVALID_ARGUMENT if rank < 0 else _lib.ERR_UNSUPPORTED, "fh_lora_workspace", 1, 64, rank)
    for k in (0, 4, 60):
        refused(_lib.ERR_UNSUPPORTED, "fh_lora_workspace", 1, k, 8)
    refused(_lib.ERR_INVALID_ARGUMENT, "fh_lora_workspace", 1 << 31, 64, 8)
    assert _lib.load().fh_lora_workspace(1, 64, 8, None) == _lib.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("k", [64, 4096, 14336])
def test_lora_workspace_of_the_most_rows_serves_fewer(k):
    sizes = [_lib.lora_workspace_bytes(m, k, 16) for m in (0, 1, 64, 65, 1000, 1024, 1025, 1100, 2047, 2049, 4096)]
    assert sizes == sorted(sizes)


def test_calls_without_a_device():
    lib, f = _lib.load(), ctypes.c_float(1)
    rules = _lib.LogitRules()
    for name, args in (
            ("fh_paged_rope_kv", (None, None, 1, 1, 1, 64, None, None, 1, None, None, None, 1, 1, None, None, 1, 16, None)),
            ("fh_paged_attention", (None, None, 1, 1, 1, 64, None, None, 1, 16, None, 1, None, f, None, 0, None)),
            ("fh_lora_add", (None, None, 1, 64, 64, None, None, None, 1, 8, 1, None, None, 1, None, 1, 0, None, 0)),
            ("fh_logits_process", (None, None, 0, 1, 1, ctypes.byref(rules), None))):
        assert getattr(lib, name)(*args) == _lib.ERR_INVALID_ARGUMENT
        assert name in _lib.last_error() and "device is null" in _lib.last_error()


# ---- the restatement ----

def test_reference_attention_by_hand():
    keys = np.zeros((2, 1, 16, 2))
    values = np.zeros((2, 1, 16, 2))
    keys[1, 0, 0], keys[1, 0, 1] = [1, 0], [0, 1]
    values[1, 0, 0], values[1, 0, 1] = [10, 0], [0, 20]
    q = np.array([[[np.log(3.0), 0.0]], [[1.0, 1.0]]])
    out, weight, _ = S.attend(q, keys, values, np.array([[1], [S.NONE]], np.uint32), np.array([1, 5]), 1.0)
    assert np.allclose(out[0, 0], [7.5, 5.0]) and np.allclose(weight[0, 0], [7.5, 5.0])
    assert not out[1].any()  # no page: no key


def test_reference_logits_by_hand():
    u = {"history": np.array([[1, 1, 2, 9, 1]], np.uint32), "history_len": np.array([4], np.uint32),
         "prompt_len": np.array([1], np.uint32), "repetition": np.array([2.0], np.float32),
         "frequency": np.array([0.5], np.float32), "presence": np.array([0.25], np.float32),
         "bias_ids": np.array([[3, 3, 0]], np.uint32), "bias_values": np.array([[1.0, 4.0, 8.0]], np.float32),
         "bias_len": np.array([2], np.uint32), "mask": np.array([[0b011110]], np.uint32)}
    z = np.array([[5.0, 4.0, -1.0, 0.0, 7.0, 7.0]])
    # 1: said twice, once generated; 2: once, generated; 3: the last of its two biases
    assert np.array_equal(S.logits(z, u), [[-np.inf, 4 / 2 - 0.5 - 0.25, -1 * 2 - 0.5 - 0.25, 4.0, 7.0, -np.inf]])


def test_reference_lora_and_append_by_hand():
    y, mag, low = S.lora(np.array([[1.0, 2.0], [1.0, 1.0]]), np.array([[[3.0, -1.0]]]), np.array([[[2.0], [-4.0]]]),
                         np.array([0.5]), [0, S.NONE], np.array([[10.0, 10.0], [1.0, 2.0]]))
    assert np.array_equal(y, [[11.0, 8.0], [1.0, 2.0]])
    assert np.array_equal(mag[0], [5.0, 10.0]) and np.array_equal(low[0], [1.0, 2.0])
    one, bits = 0x3F80, lambda v: (np.asarray(v, np.float32).view(np.uint32) >> 16).astype(np.uint16)
    qkv = bits([[1.0, 2.0] * 3])
    cos, sin = np.full((4, 2), one, np.uint16), np.full((4, 2), one, np.uint16)
    q, k, v, mag, place = S.append(qkv, 1, 1, cos, sin, [0], [3], np.array([[2]], np.uint32), 3, 16)
    assert np.array_equal(q[0, 0], [-1.0, 3.0]) and np.array_equal(k[0, 0], [-1.0, 3.0])
    assert np.array_equal(v[0, 0], [1.0, 2.0]) and place == [(2, 3)] and np.array_equal(mag[0, 0], [3.0, 3.0])

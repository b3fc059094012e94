"""The host side of the operators for drafted tokens, without a GPU: the
header's structs as ctypes sees them, workspace sizes and their refusals, calls
without a device, and the float64 restatement on cases worked by hand."""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib
from oracle import draft_ref as D
from test_host import _c_layout
from test_serving_host import refused


@pytest.mark.parametrize("struct, cls", [("fh_paged_pool", _lib.PagedPool), ("fh_paged_cache", _lib.PagedCache)])
def test_structs_match_the_header(struct, cls):
    fields = [f[0] for f in cls._fields_]
    assert _c_layout(struct, fields) == [ctypes.sizeof(cls)] + [getattr(cls, f).offset for f in fields]


def test_tree_attention_workspace():
    size = _lib.paged_tree_attention_workspace_bytes
    assert size(1, 8, 32, 8, 128, 16, 20) > 0
    assert size(8, 64, 32, 8, 128, 16, 8000) < 1 << 30 and size(1, 1024, 32, 8, 128, 64, 2 ** 24) < 1 << 31
    name, bad = "fh_paged_tree_attention_workspace", _lib.ERR_INVALID_ARGUMENT
    for args in ((1, 0, 32, 8, 128, 16, 4), (1, 1025, 32, 8, 128, 16, 4), (1, 4, 32, 5, 128, 16, 4),
                 (1, 4, 0, 1, 128, 16, 4), (1, 4, 4, 0, 64, 16, 4), (1, 4, 4, 2, 64, 24, 4), (1, 4, 4, 2, 64, 0, 4),
                 (1, 4, 4, 2, 64, 16, 0), (-1, 4, 4, 2, 64, 16, 4), (1, 4, 4, 2, 64, 1 << 40, 4)):
        refused(bad, name, *args)
    refused(_lib.ERR_UNSUPPORTED, name, 1, 4, 4, 2, 96, 16, 4)
    refused(_lib.ERR_INDEX_TOO_LARGE, name, 65536, 4, 4, 2, 64, 16, 4)
    refused(_lib.ERR_INDEX_TOO_LARGE, name, 1, 4, 4, 2, 64, 16, 1 << 27)
    refused(_lib.ERR_INDEX_TOO_LARGE, name, 1, 1024, 65534, 2, 64, 16, 4)
    assert _lib.load().fh_paged_tree_attention_workspace(1, 4, 4, 2, 64, 16, 4, None) == bad


@pytest.mark.parametrize("heads,kv,hd,page,pages", [(32, 8, 128, 16, 8), (32, 8, 128, 64, 128), (20, 4, 64, 16, 2048),
                                                    (8, 1, 256, 32, 33)])
@pytest.mark.parametrize("width", [1, 6, 64, 200])
def test_tree_workspace_of_the_largest_batch_serves_smaller_ones(heads, kv, hd, page, pages, width):
    sizes = [_lib.paged_tree_attention_workspace_bytes(b, width, heads, kv, hd, page, pages)
             for b in (0, 1, 2, 7, 64, 65, 512, 1023, 1024, 1025, 5000)]
    assert sizes == sorted(sizes)


def test_probs_and_verify_workspaces():
    for size in (lambda r: _lib.logits_probs_workspace_bytes(r, 128256),
                 lambda r: _lib.verify_draft_workspace_bytes(r, 8, 128256)):
        sizes = [size(r) for r in (0, 1, 2, 63, 64, 65, 511, 512, 4000, 65535)]
        assert sizes == sorted(sizes) and sizes[0] >= 0 and sizes[1] > 0
    refused(_lib.ERR_INVALID_ARGUMENT, "fh_logits_probs_workspace", -1, 5)
    refused(_lib.ERR_INDEX_TOO_LARGE, "fh_logits_probs_workspace", 65536, 5)
    for args in ((1, 0, 5), (1, 1025, 5), (1, 4, 0), (-1, 4, 5), (1, 4, 1 << 31)):
        refused(_lib.ERR_INVALID_ARGUMENT, "fh_verify_draft_workspace", *args)
    refused(_lib.ERR_INDEX_TOO_LARGE, "fh_verify_draft_workspace", 65536, 4, 5)
    assert _lib.load().fh_logits_probs_workspace(1, 4, None) == _lib.ERR_INVALID_ARGUMENT
    assert _lib.load().fh_verify_draft_workspace(1, 4, 4, None) == _lib.ERR_INVALID_ARGUMENT


def test_calls_without_a_device():
    lib, f = _lib.load(), ctypes.c_float(1)
    cache = ctypes.byref(_lib.PagedCache())
    for name, args in (
            ("fh_paged_norm_rope_kv", (None, None, 1, 1, 1, 64, None, None, f, None, None, 1, None, None, None, None, 1, 1,
                                       None, None, 1, 16, None)),
            ("fh_paged_tree_attention", (None, None, 1, 1, 1, 1, 64, None, None, 1, 16, None, 1, None, None, None, f, None,
                                         0, None)),
            ("fh_logits_probs", (None, None, 0, 1, 1, None, None, 0, None)),
            ("fh_verify_draft", (None, None, None, 1, 1, 1, None, None, None, None, None, 0, None, None, None)),
            ("fh_paged_reserve", (None, cache, None, None)), ("fh_paged_fork", (None, cache, None, None, 1, None)),
            ("fh_paged_free", (None, cache, None, 1)), ("fh_paged_compact", (None, cache, None, None, 1, None))):
        assert getattr(lib, name)(*args) == _lib.ERR_INVALID_ARGUMENT
        assert name in _lib.last_error() and "device is null" in _lib.last_error()


# ---- the restatement ----

def test_reference_norm_and_probs_by_hand():
    assert np.allclose(D.norm(np.array([3.0, 4.0]), np.array([1.0, 2.0]), 0.0), [3 / 12.5 ** 0.5, 8 / 12.5 ** 0.5])
    z = np.array([[0.0, np.log(3.0), -np.inf], [1.0, 5.0, 5.0], [-np.inf] * 3, [np.inf, 0.0, np.inf], [np.nan, 2.0, 2.0]])
    want = [[0.25, 0.75, 0], [0, 1, 0], [0, 0, 0], [0.5, 0, 0.5], [0, 0.5, 0.5]]
    assert np.allclose(D.probs(z, [1.0, 0.0, 1.0, 0.7, 2.0]), want)
    assert np.allclose(D.probs(z[:1], [0.5]), [[0.1, 0.9, 0]])


def test_reference_tree_attention_by_hand():
    keys, values = np.zeros((1, 1, 16, 2)), np.zeros((1, 1, 16, 2))
    values[0, 0, :4] = [[8, 0], [0, 4], [2, 2], [0, 6]]
    q = np.zeros((1, 3, 1, 2))
    table, mask = np.zeros((1, 1), np.uint32), np.array([[[0b001], [0b010], [0b101]]], np.uint32)
    out, _, _ = D.tree_attend(q, keys, values, table, [1], None, mask, 1.0)
    assert np.allclose(out[0, :, 0], [[4, 2], [5, 1], [8 / 3, 10 / 3]])
    out, _, _ = D.tree_attend(q, keys, values, table, [1], [2], None, 1.0)  # a chain of two
    assert np.allclose(out[0, :, 0], [[4, 2], [10 / 3, 2], [0, 0]])
    out, _, _ = D.tree_attend(q, keys, values, table, [0], None, np.zeros((1, 3, 1), np.uint32), 1.0)
    assert not out.any()
    out, _, _ = D.tree_attend(q, keys, values, table, [14], None, None, 1.0)  # does not fit
    assert not out.any()


def test_reference_verify_by_hand():
    p = np.array([[[0.5, 0.3, 0.2], [0.1, 0.1, 0.8], [0.2, 0.2, 0.6]]], np.float32)
    q = np.array([[[0.25, 0.5, 0.25], [0.1, 0.8, 0.1], [1, 0, 0]]], np.float32)
    tokens = np.array([[9, 1, 1]], np.uint32)
    # 0.3 / 0.5: accepted below 0.6; then 0.1 / 0.8 below 0.125; then a token of row 2
    path, out, took = D.verify(p, q, tokens, None, None, np.array([[0.5, 0.59, 0.12]], np.float32))
    assert path[0].tolist() == [0, 1, 2] and out[0].tolist() == [1, 1, 2] and took[0] == 3
    # refused at once: what is left is [0.25, 0, 0]
    path, out, took = D.verify(p, q, tokens, None, None, np.array([[0.99, 0.61, 0.0]], np.float32))
    assert path[0].tolist() == [0, D.NONE, D.NONE] and out[0].tolist() == [0, D.NONE, D.NONE] and took[0] == 1
    # refused at node 1: [0, 0, 0.7] is left
    path, out, took = D.verify(p, q, tokens, None, None, np.array([[0.1, 0.0, 0.2]], np.float32))
    assert path[0].tolist() == [0, 1, D.NONE] and out[0].tolist() == [1, 2, D.NONE]
    # two children of the root picked without chance: 0.5, then 0.3 of the 0.5 left
    tokens, parents = np.array([[9, 0, 1]], np.uint32), np.array([[D.NONE, 0, 0]], np.uint32)
    path, out, _ = D.verify(p, None, tokens, parents, None, np.array([[0.5, 0.5, 0.59]], np.float32))
    assert path[0].tolist() == [0, 2, D.NONE] and out[0].tolist() == [1, 2, D.NONE]
    path, out, _ = D.verify(p, None, tokens, parents, None, np.array([[0.5, 0.5, 0.61]], np.float32))
    assert path[0].tolist() == [0, D.NONE, D.NONE] and out[0].tolist() == [2, D.NONE, D.NONE]
    # node 2 is not in use
    path, out, _ = D.verify(p, None, tokens, parents, [2], np.array([[0.5, 0.5, 0.0]], np.float32))
    assert out[0].tolist() == [1, D.NONE, D.NONE]


def test_reference_pages_by_hand():
    table = np.array([[1, 3, D.NONE], [D.NONE] * 3, [D.NONE] * 3], np.uint32)
    g = D.Pages(table, np.array([20, 0, 0], np.uint32), np.array([0, 1, 0, 1, 0], np.uint32), np.zeros((1, 5, 1, 16, 2)),
                np.zeros((1, 5, 1, 16, 2)))
    g.k[0, 3, 0, :4] = 7
    assert g.fork([0, 0, 0], [1, 2, 1]).tolist() == [0, 0, 1]
    assert g.table.tolist() == [[1, 3, D.NONE], [1, 0, D.NONE], [1, 2, D.NONE]] and g.refs.tolist() == [1, 3, 1, 1, 0]
    assert g.lengths.tolist() == [20, 20, 20] and (g.k[0, [0, 2], 0, :4] == 7).all() and not g.k[0, 0, 0, 4:].any()
    assert g.reserve([0, 13, 30]).tolist() == [0, 0, 2]  # page 4; none for the third, whose table ends too
    assert g.table[1, 2] == 4
    g.free([1, 1, 9])
    assert g.refs.tolist() == [0, 2, 1, 1, 0] and g.lengths[1] == 0 and (g.table[1] == D.NONE).all()
    g.k[0, 3, 0, 4:9] = np.arange(5).reshape(5, 1)
    assert g.compact(np.array([[0, 2, 3], [0] * 3, [0] * 3], np.uint32), np.array([3, 0, 0])).tolist() == [23, 0, 20]
    assert g.k[0, 3, 0, 4:9, 0].tolist() == [0, 2, 3, 3, 4]


@pytest.mark.parametrize("masked", [False, True])
def test_reference_tree_attention_whole_is_the_other(masked):
    rng = np.random.default_rng(3)
    q, k, v = (rng.standard_normal(s) for s in ((3, 5, 4, 8), (9, 2, 16, 8), (9, 2, 16, 8)))
    table = np.array([[1, 4, 9, 0], [7, 8, D.NONE, D.NONE], [2, 3, 5, 6]], np.uint32)
    masks = rng.integers(0, 32, (3, 5, 1)).astype(np.uint32) if masked else None
    v[4, :, 3], v[8, 1, 1, 2], v[3, 0, 15, 1] = np.inf, np.nan, -np.inf
    for lengths, counts in (([40, 20, 59], [5, 3, 5]), ([0, 12, 60], None), ([0, 0, 0], [1, 0, 4])):
        a, b = (f(q, k, v, table, lengths, counts, masks, 0.7) for f in (D.tree_attend, D.tree_attend_whole))
        for x, y in zip(a, b):
            assert np.allclose(x, y, rtol=1e-12, atol=1e-14, equal_nan=True)

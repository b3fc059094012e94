"""The pages of a cache of all layers on the GPU: fh_paged_reserve, fh_paged_fork,
fh_paged_free and fh_paged_compact against the restatement's lists
(oracle/draft_ref.py), every table entry, count and value the same."""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from foundry_amd.kv_layout import tile_k, untile_k
from oracle import draft_ref as D
from test_gpu_paged import down, p, refused, up

pytestmark = pytest.mark.gpu

NONE = D.NONE


class Cache:
    """A cache on the device and its restatement."""

    def __init__(self, dev, seed, lens, width, n_pages, page=16, layers=2, kv=2, hd=64, reserved=0):
        rng = np.random.default_rng(seed)
        ids = rng.permutation(n_pages)
        table = np.full((len(lens), width), NONE, np.uint32)
        refs, at = np.zeros(n_pages, np.uint32), 0
        for s, n in enumerate(lens):
            count = min(width, -(-(n + reserved) // page))
            table[s, :count] = ids[at:at + count]
            refs[table[s, :count]] = 1
            at += count
        self.dev, self.kv, self.hd, self.layers = dev, kv, hd, layers
        k, v = (synth.bf16_normal(seed + i, (layers, n_pages, kv, page, hd)) for i in (1, 2))
        self.ref = D.Pages(table, np.array(lens, np.uint32), refs, k, v, page)
        self.st = {"table": up(dev, table), "lengths": up(dev, self.ref.lengths), "refs": up(dev, refs)}
        self.k = [up(dev, tile_k(k[i])) for i in range(layers)]
        self.v = [up(dev, v[i]) for i in range(layers)]

    def struct(self, **o):
        pools = (_lib.PagedPool * self.layers)(*[(a.ptr, b.ptr) for a, b in zip(self.k, self.v)])
        a = dict(pools=pools, n_layers=self.layers, n_kv=self.kv, head_dim=self.hd, n_pages=self.ref.n_pages,
                 page_size=self.ref.page, page_table=self.st["table"].ptr, n_seqs=self.ref.table.shape[0],
                 max_pages=self.ref.table.shape[1], lengths=self.st["lengths"].ptr, refs=self.st["refs"].ptr)
        self.held = _lib.PagedCache(**(a | o))
        return ctypes.byref(self.held)

    def check(self):
        for name in ("table", "lengths", "refs"):
            want = getattr(self.ref, name)
            got = down(self.dev, self.st[name], np.uint32, want.shape)
            assert np.array_equal(got, want), (name, np.argwhere(got != want)[:5].tolist())
        shape = self.ref.k.shape[1:]
        for i in range(self.layers):
            assert np.array_equal(untile_k(down(self.dev, self.k[i], np.uint16, shape)), self.ref.k[i]), f"k of layer {i}"
            assert np.array_equal(down(self.dev, self.v[i], np.uint16, shape), self.ref.v[i]), f"v of layer {i}"

    def reserve(self, extra, report=True):
        s_extra, out = up(self.dev, np.array(extra, np.uint32)), up(self.dev, np.full(len(extra), 9, np.uint32))
        _lib.call("fh_paged_reserve", self.dev.handle, self.struct(pools=None, n_layers=0), p(s_extra),
                  p(out) if report else None)
        want = self.ref.reserve(extra)
        assert not report or np.array_equal(down(self.dev, out, np.uint32, want.shape), want)
        self.check()
        return want

    def free(self, seqs):
        s = up(self.dev, np.array(seqs, np.uint32))
        _lib.call("fh_paged_free", self.dev.handle, self.struct(pools=None, n_layers=0), p(s), len(seqs))
        self.ref.free(seqs)
        self.check()

    def fork(self, src, dst):
        a, b = (np.array(x, np.uint32) for x in (src, dst))
        s_a, s_b, out = up(self.dev, a), up(self.dev, b), up(self.dev, np.full(len(a), 9, np.uint32))
        _lib.call("fh_paged_fork", self.dev.handle, self.struct(), p(s_a), p(s_b), len(a), p(out))
        want = self.ref.fork(a, b)
        got = down(self.dev, out, np.uint32, want.shape)
        assert np.array_equal(got, want), (got, want)
        self.check()
        return want

    def compact(self, path, accepted, in_place=True):
        path, accepted = np.array(path, np.uint32), np.array(accepted, np.uint32)
        s_p, s_a = up(self.dev, path), up(self.dev, accepted)
        new = self.st["lengths"] if in_place else up(self.dev, np.zeros(len(accepted), np.uint32))
        _lib.call("fh_paged_compact", self.dev.handle, self.struct(refs=None), p(s_p), p(s_a), path.shape[1], p(new))
        want = self.ref.compact(path, accepted)
        if in_place:
            self.ref.lengths = want
        else:
            assert np.array_equal(down(self.dev, new, np.uint32, want.shape), want)
        self.check()


# ------------------------------------------------------------------ reserve

@pytest.mark.parametrize("page", [16, 48])
def test_reserve(device, page):
    c = Cache(device, 1, [0, 1, page, page + 1, 3 * page - 1, 0, 2 * page], 9, 60, page)
    assert not c.reserve([1, page, page, 2 * page, 1, 0, 5 * page]).any()
    assert not c.reserve([0] * 7).any()
    assert not c.reserve([2, 0, 1, 1, page + 2, 9 * page, page], report=False).any()


def test_reserve_past_the_table_and_the_free_pages(device):
    c = Cache(device, 2, [10, 30, 5, 100], 4, 14)
    lost = c.reserve([30, 16 * 5, 1 << 31, 40])
    assert lost[1] > 0 and lost[2] > 0 and lost[3] > 0
    c.free([1])
    c.reserve([16, 60, 16, 0])
    c.reserve([NONE, NONE, NONE, NONE])


def test_reserve_idle_lengths_past_the_table(device):
    c = Cache(device, 3, [4, 4, 4], 4, 20)
    for name, v in (("lengths", np.array([NONE, 0x80000000, 70], np.uint32)),):
        c.ref.lengths = v
        c.st[name] = up(device, v)
    c.reserve([0, 0, 0])
    assert (c.reserve([1, 20, 30]) > 0).all()


def test_reserve_many_sequences(device):
    """More sequences than threads, pages of many rounds, holes in rows and in the pool."""
    rng = np.random.default_rng(4)
    lens = rng.integers(0, 60, 3000).tolist()
    c = Cache(device, 4, lens, 6, 17000, layers=1, kv=1, hd=32)
    c.free(rng.choice(3000, 700, replace=False).tolist())
    c.reserve(rng.integers(0, 40, 3000).tolist())


def test_reserve_hands_out_at_most_16384_pages(device):
    c = Cache(device, 5, [0, 0, 0], 9000, 20000, layers=1, kv=1, hd=32)
    lost = c.reserve([16 * 9000, 16 * 8000, 16])
    assert lost.tolist() == [0, 616, 1]
    c.reserve([16 * 9000, 16 * 8000, 16])


# ------------------------------------------------------------- fork and free

@pytest.mark.parametrize("page,kv,hd,layers", [(16, 2, 64, 3), (48, 1, 128, 2), (32, 8, 32, 1), (16, 1, 256, 40)])
def test_fork(device, page, kv, hd, layers):
    lens = [0, 1, 15, page, page + 1, 2 * page + 17 % page, 3 * page] + [0] * 9
    c = Cache(device, 6, lens, 6, 40, page, layers, kv, hd, reserved=20)
    assert not c.fork(range(7), range(7, 14)).any()
    assert not c.fork([4, 4], [14, 15]).any()
    c.reserve([0] * 7 + [3, 20, 1, 1, 30, 1, page, 0, 1])
    c.fork([9, 9, 11], [7, 8, 10])  # over what they held
    c.free([4, 15, 4, 99, NONE])
    c.free(range(16))
    assert not c.ref.refs.any()


def test_fork_without_free_pages_leaves_the_sequence_empty(device):
    c = Cache(device, 7, [20, 32, 9] + [0] * 7, 4, 7)  # 5 pages held, 2 free
    lost = c.fork([0, 1, 2, 0, 1, 2], [3, 4, 5, 6, 7, 8])
    assert lost.tolist() == [0, 0, 0, 1, 0, 1]
    c.free([3, 4])
    assert c.fork([0], [9]).tolist() == [0]


def test_fork_takes_the_pages_that_it_frees(device):
    """The fork's own row holds the last pages."""
    c = Cache(device, 8, [20, 40], 4, 5)
    assert c.fork([0], [1]).tolist() == [0]


def test_forks_that_do_not_stand(device):
    c = Cache(device, 9, [20, 40, 10, 0, 0, 0], 4, 30)
    before = c.ref.table.copy()
    # to itself, past the sequences, into one that another is forked from, twice the same
    assert c.fork([0, 6, 0, 1, 2, 2], [0, 3, 7, 2, 4, 4]).tolist() == [1, 1, 1, 1, 0, 1]
    assert np.array_equal(before[[0, 1, 2, 3, 5]], c.ref.table[[0, 1, 2, 3, 5]])
    c.ref.lengths[1] = 65
    c.st["lengths"] = up(device, c.ref.lengths)
    assert c.fork([1, NONE, 0], [5, 5, NONE]).tolist() == [1, 1, 1]


def test_fork_of_entries_that_name_no_page(device):
    c = Cache(device, 10, [60, 40, 0, 0], 4, 30)
    c.ref.table[0, 1], c.ref.table[1, 2] = NONE, 30  # a hole; the page that would be copied
    c.ref.refs[:] = 0
    for pg in c.ref.table[c.ref.table < 30]:
        c.ref.refs[pg] += 1
    c.st["table"], c.st["refs"] = up(device, c.ref.table), up(device, c.ref.refs)
    assert not c.fork([0, 1], [2, 3]).any()


def test_a_thousand_forks(device):
    c = Cache(device, 11, [37, 5, 64] + [0] * 1024, 4, 1100, layers=1, kv=1, hd=32)
    c.fork([i % 3 for i in range(1024)], range(3, 1027))
    c.free(range(3, 1027))


# ------------------------------------------------------------------ compact

@pytest.mark.parametrize("page,kv,hd,layers", [(16, 2, 64, 3), (48, 1, 128, 2), (32, 8, 128, 1), (16, 3, 96, 128)])
@pytest.mark.parametrize("in_place", [True, False])
def test_compact(device, page, kv, hd, layers, in_place):
    lens = [0, 1, 15, 16, 17, 40, 63, 9]
    c = Cache(device, 12, lens, 8, 60, page, layers, kv, hd, reserved=40)
    rng = np.random.default_rng(13)
    path = np.full((8, 40), NONE, np.uint32)
    accepted = np.array([1, 2, 5, 0, 9, 20, 40, 3], np.uint32)
    for s, n in enumerate(accepted):
        path[s, :n] = ([0] + np.sort(rng.permutation(39)[:max(int(n) - 1, 0)] + 1).tolist())[:n]
    path[5, :20] = [0] + list(range(2, 21))  # each source is the next one's place
    path[6] = np.arange(40)                  # nothing moves
    c.compact(path, accepted, in_place)


def test_compact_passes_over_places_without_a_page(device):
    c = Cache(device, 14, [60, 10, 30, 5], 4, 12, reserved=3)  # a table of 64 places
    path = np.array([[0, 2, 4, 9, 11], [0, 1, 7, 8, 9], [0, 3, NONE, 5, 6], [0, 4, 5, 6, 20]], np.uint32)
    c.ref.table[3, 0] = NONE  # a table's entry can be none where its refs count
    c.st["table"] = up(device, c.ref.table)
    c.compact(path, [5, 5, 2, 9], in_place=False)


def test_a_step_after_another(device):
    """Reserve, compact, fork, over and over: the counts are those of the table's entries."""
    rng = np.random.default_rng(15)
    c = Cache(device, 16, [3, 20, 47, 0, 0, 0], 12, 50)
    for step in range(6):
        c.reserve([12] * 3 + [0] * 3)
        path = np.stack([np.concatenate([[0], np.sort(rng.permutation(11)[:5] + 1)]) for _ in range(6)])
        took = rng.integers(1, 7, 6)
        took[3:] = 0
        c.compact(path, took)
        c.fork([step % 3, (step + 1) % 3], [3, 4 + step % 2])
        c.free([3 + step % 3])
        want = np.bincount(c.ref.table[c.ref.table < 50], minlength=50)
        assert np.array_equal(want, c.ref.refs)


# ----------------------------------------------------------------- refusals

def test_refusals(device):
    c = Cache(device, 17, [20, 5, 0], 8, 20)
    lists = up(device, np.zeros(64, np.uint32))
    x, y, z = (p(lists, 64 * i) for i in range(3))
    bad, dev = _lib.ERR_INVALID_ARGUMENT, device.handle
    calls = {"fh_paged_reserve": lambda cache: (dev, cache, x, y), "fh_paged_free": lambda cache: (dev, cache, x, 1),
             "fh_paged_fork": lambda cache: (dev, cache, x, y, 1, z),
             "fh_paged_compact": lambda cache: (dev, cache, x, y, 4, z)}
    for name, args in calls.items():
        refused(bad, name, None, *args(c.struct())[1:])
        with pytest.raises(_lib.HipError) as e:
            _lib.call(name, dev, None, *args(None)[2:])
        assert e.value.status == bad
        for o in (dict(n_pages=0), dict(page_size=8), dict(max_pages=0), dict(n_seqs=-1)):
            refused(bad, name, *args(c.struct(**o)))
        refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(c.struct(n_seqs=16385)))
        refused(bad, name, *args(c.struct(lengths=c.st["table"].ptr)), match="overlap")
        refused(bad, name, *args(c.struct(lengths=c.st["lengths"].ptr + 2)), match="aligned")
        with pytest.raises(_lib.HipError):
            _lib.call(name, *args(c.struct(page_table=None)))
    for name in ("fh_paged_reserve", "fh_paged_free", "fh_paged_fork"):
        refused(bad, name, *calls[name](c.struct(refs=c.st["table"].ptr)), match="overlap")
        refused(_lib.ERR_OUT_OF_BOUNDS, name, *calls[name](c.struct(n_pages=10 ** 6)))
    for name in ("fh_paged_fork", "fh_paged_compact"):
        for o in (dict(pools=None), dict(n_layers=0), dict(n_layers=129), dict(n_kv=0)):
            refused(bad, name, *calls[name](c.struct(**o)))
        refused(_lib.ERR_UNSUPPORTED, name, *calls[name](c.struct(head_dim=48)))
        twice = (_lib.PagedPool * 2)(*[(c.k[0].ptr, c.v[0].ptr)] * 2)
        refused(bad, name, *calls[name](c.struct(pools=twice)), match="overlap")
        off = (_lib.PagedPool * 2)((c.k[0].ptr + 8, c.v[0].ptr), (c.k[1].ptr, c.v[1].ptr))
        refused(bad, name, *calls[name](c.struct(pools=off)), match="aligned")
        inside = (_lib.PagedPool * 2)((c.k[0].ptr + 16, c.v[0].ptr), (c.k[1].ptr, c.v[1].ptr))
        refused(_lib.ERR_OUT_OF_BOUNDS, name, *calls[name](c.struct(pools=inside)))
    refused(bad, "fh_paged_reserve", dev, c.struct(), None, y)
    refused(bad, "fh_paged_reserve", dev, c.struct(), x, x, match="overlap")
    refused(bad, "fh_paged_free", dev, c.struct(), x, -1)
    refused(bad, "fh_paged_free", dev, c.struct(), None, 1)
    refused(_lib.ERR_INDEX_TOO_LARGE, "fh_paged_free", dev, c.struct(), x, 65536)
    refused(_lib.ERR_INDEX_TOO_LARGE, "fh_paged_fork", dev, c.struct(), x, y, 1025, z)
    for a in ((None, y, 1, z), (x, None, 1, z), (x, y, 1, None), (x, x, 1, z), (x, y, 1, x), (x, y, -1, z)):
        refused(bad, "fh_paged_fork", dev, c.struct(), *a)
    for a in ((None, y, 4, z), (x, None, 4, z), (x, y, 4, None), (x, y, 0, z), (x, y, 65536, z), (x, x, 4, z), (x, y, 4, x)):
        refused(bad, "fh_paged_compact", dev, c.struct(), *a)
    c.check()
    for name, args in (("fh_paged_free", (x, 0)), ("fh_paged_fork", (x, y, 0, z))):
        _lib.call(name, dev, c.struct(), *args)
    _lib.call("fh_paged_reserve", dev, c.struct(n_seqs=0), x, y)
    _lib.call("fh_paged_compact", dev, c.struct(n_seqs=0), x, y, 4, z)
    c.check()

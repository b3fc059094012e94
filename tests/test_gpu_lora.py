"""fh_lora_add on the GPU against the float64 restatement (oracle/serving_ref.py).

Bounds: y is rounded once, by at most half a step of its dtype (2^-8 of the
value in bf16, 2^-24 in fp32), and base + delta once more in fp32. Behind that,
x . A^T is an fp32 sum of k exact products in some order (k * 2^-24 of sum
|x||A|), scaled once; v . B^T has v as two bf16 parts (2^-16 of it), for fp32
results as three (2^-23), and is a sum of 2 or 3 rank products.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from oracle import serving_ref as S

pytestmark = pytest.mark.gpu

NONE = S.NONE


def up(dev, arr):
    return dev.storage_from_bytes(np.ascontiguousarray(arr).tobytes())


def down(dev, st, dtype, shape):
    out = np.empty(shape, dtype=dtype)
    _lib.call("fh_download", dev.handle, out.ctypes.data_as(ctypes.c_void_p), ctypes.c_void_p(st.ptr), out.nbytes)
    return out


def p(st, offset=0):
    return ctypes.c_void_p(st.ptr + offset) if st is not None else None


class Case:
    """Inputs on the device; strides and offsets in elements."""

    def __init__(self, dev, seed, m, k, n, rank, n_adapters, ids, f32=False, x_ld=None, base_ld=None, y_ld=None,
                 shift=0):
        self.dev, self.dims, self.f32, self.shift = dev, (m, k, n, rank, n_adapters), f32, shift
        self.x_ld, self.base_ld, self.y_ld = x_ld or k, base_ld or n, y_ld or n
        self.kind = np.float32 if f32 else np.uint16
        rng = np.random.default_rng(seed)
        self.ids = np.asarray(ids, dtype=np.uint32)
        self.x = synth.bf16_normal(seed, (m, self.x_ld))
        self.a = synth.bf16_rne((rng.standard_normal((n_adapters, rank, k)) * k ** -0.5).astype(np.float32))
        self.b = synth.bf16_rne((rng.standard_normal((n_adapters, n, rank)) * 0.3).astype(np.float32))
        self.scales = rng.uniform(-2, 2, n_adapters).astype(np.float32)
        base = rng.standard_normal((m, self.base_ld)).astype(np.float32)
        self.base = base if f32 else synth.bf16_rne(base)
        self.st = [up(dev, v) for v in (self.x, self.a, self.b, self.scales, self.ids)]
        self.ws_bytes = _lib.lora_workspace_bytes(m, k, rank)
        self.ws = up(dev, np.full(self.ws_bytes, 0xFF, np.uint8))

    def run(self, in_place=False):
        m, k, n, rank, u = self.dims
        size = np.dtype(self.kind).itemsize
        sentinel = np.full((m, self.y_ld), 7, self.kind)
        pad = np.zeros(self.shift, self.kind)
        base = up(self.dev, np.concatenate([pad, self.base.ravel()]))
        y = base if in_place else up(self.dev, np.concatenate([pad, sentinel.ravel()]))
        y_ld = self.base_ld if in_place else self.y_ld
        st, off = self.st, self.shift * size
        _lib.call("fh_lora_add", self.dev.handle, p(st[0]), m, k, self.x_ld, p(st[1]), p(st[2]), p(st[3]), u, rank, n,
                  p(st[4]), p(base, off), self.base_ld, p(y, off), y_ld, _lib.F32 if self.f32 else _lib.BF16, p(self.ws),
                  self.ws_bytes)
        got = down(self.dev, y, self.kind, self.shift + m * y_ld)[self.shift:].reshape(m, y_ld)
        # what lies between the rows stays as it was
        assert np.array_equal(got[:, n:], (self.base if in_place else sentinel)[:, n:])
        return got[:, :n]

    def check(self, in_place=False):
        m, k, n, rank, _ = self.dims
        got = self.run(in_place)
        assert np.array_equal(got, self.run(in_place)), "the same call gave other bits"
        base = self.base[:, :n]
        val = (lambda t: t.astype(np.float64)) if self.f32 else S.f64
        ref, mag, low = S.lora(S.f64(self.x[:, :k]), S.f64(self.a), S.f64(self.b), self.scales.astype(np.float64),
                               self.ids, val(base))
        half = 2.0 ** -24 if self.f32 else 2.0 ** -8
        bound = half * np.abs(ref) + 2.0 ** -24 * (np.abs(ref) + np.abs(val(base))) + (k + 2) * 2.0 ** -24 * mag
        bound += ((2.0 ** -23 if self.f32 else 2.0 ** -16) + 3 * rank * 2.0 ** -24) * low
        assert (np.abs(val(got) - ref) <= bound * (1 + 2.0 ** -20)).all()
        bare = self.ids >= self.dims[4]
        assert np.array_equal(got[bare], base[bare]), "a row without an adapter is base"
        return got


@pytest.mark.parametrize("rank", [8, 16, 24, 40, 64, 96, 128])
@pytest.mark.parametrize("f32", [False, True])
def test_ranks(device, rank, f32):
    ids = [0, 2, NONE, 1, 0, 3, 2, 2, 5]  # 5: past the last adapter
    Case(device, rank, 9, 264, 100, rank, 5, ids, f32).check()


@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 63, 64, 65, 130, 200])
def test_rows_of_shared_and_own_adapters(device, m):
    ids = np.random.default_rng(m).integers(0, 7, m)
    Case(device, m, m, 512, 272, 16, 6, np.where(ids == 6, NONE, ids)).check()


@pytest.mark.parametrize("ids", [[4] * 70, list(range(70)), [NONE] * 70, [i // 23 for i in range(70)],
                                 [i % 2 for i in range(70)]], ids=["one", "all_own", "none", "packed", "alternating"])
def test_groupings(device, ids):
    Case(device, 5, 70, 256, 130, 32, 70, ids).check()


@pytest.mark.parametrize("k", [8, 16, 40, 56, 520, 2056, 8200])
def test_inner_sizes(device, k):
    Case(device, k, 20, k, 64, 16, 3, [i % 4 if i % 4 < 3 else NONE for i in range(20)]).check()


@pytest.mark.parametrize("rank,f32", [(16, False), (40, True), (128, True), (128, False)])
@pytest.mark.parametrize("m,k", [(3, 5120), (9, 6664), (40, 14336), (70, 10248)])
def test_long_inner_sizes(device, m, k, rank, f32):
    """k in more ranges than a short one's."""
    Case(device, m + k, m, k, 144, rank, 4, [i % 5 for i in range(m)], f32).check()
    Case(device, m + k + 1, m, k, 33, rank, 2, [0] * m, f32).check()


@pytest.mark.parametrize("m", [1024, 1025])
def test_long_inner_sizes_where_windows_change(device, m):
    Case(device, m, m, 8200, 48, 16, 3, [i // 200 % 4 for i in range(m)]).check()


@pytest.mark.parametrize("n", [1, 3, 63, 64, 65, 255, 257, 1001])
@pytest.mark.parametrize("f32", [False, True])
def test_odd_widths(device, n, f32):
    Case(device, n, 21, 128, n, 8, 4, [i % 5 for i in range(21)], f32).check()


@pytest.mark.parametrize("f32", [False, True])
def test_strides(device, f32):
    ids = [i % 4 for i in range(37)]
    Case(device, 1, 37, 192, 96, 16, 4, ids, f32, x_ld=256, base_ld=160, y_ld=104).check()
    Case(device, 2, 37, 192, 96, 16, 4, ids, f32, base_ld=97, y_ld=99).check()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("shift", [0, 1, 4])
def test_in_base_s_place_and_off_alignment(device, f32, shift):
    c = Case(device, 3, 33, 256, 200, 16, 3, [i % 4 for i in range(33)], f32, base_ld=201 if shift == 1 else 200,
             shift=shift)
    assert np.array_equal(c.check(), c.check(in_place=True))


def test_a_prompt_batch(device):
    ids = np.repeat([2, 0, NONE, 1, 2], [300, 65, 40, 1, 120])
    Case(device, 9, len(ids), 1024, 384, 32, 3, ids).check()


@pytest.mark.parametrize("n", [96, 101])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rank", [16, 40, 128])
def test_more_rows_than_a_wide_window_holds(device, rank, f32, n):
    """Past 1024 rows: packed requests from one row to hundreds, rows with no adapter among them."""
    ids = np.repeat([1, NONE, 0, 3, 2, NONE, 4, 0, 1], [500, 70, 1, 15, 64, 3, 33, 400, 130])
    c = Case(device, rank + n, len(ids), 136, n, rank, 5, ids, f32)
    assert np.array_equal(c.check(), c.run(in_place=True))


def test_many_rows_in_no_order(device):
    ids = np.random.default_rng(3).integers(0, 40, 1500)
    Case(device, 11, len(ids), 200, 80, 16, 39, np.where(ids == 39, NONE, ids)).check()


def test_special_values_stay_in_their_rows(device):
    """An inf or NaN of one row's x or base does not reach rows beside it,
    nor an adapter's NaN the rows of others."""
    c = Case(device, 4, 40, 128, 96, 16, 3, [i % 3 for i in range(40)])
    clean = c.run()
    x, a, base = c.x.copy(), c.a.copy(), c.base.copy()
    x[5, 3], x[17, 100], a[1, 2, 9], base[8, 7] = 0x7FC0, 0x7F80, 0x7FC0, 0xFF80
    c.st[0], c.st[1], c.base = up(device, x), up(device, a), base
    got = c.run()
    hit = (c.ids == 1) | np.isin(np.arange(40), [5, 17])
    hit[8] = True
    assert np.array_equal(got[~hit], clean[~hit])
    assert np.isnan(S.f64(got[5])).all() and np.isnan(S.f64(got[4])).all()


def test_infinite_down_products(device):
    """x . A^T = inf: the row is inf or NaN where the formula says so."""
    c = Case(device, 6, 3, 64, 32, 8, 1, [0, 0, NONE])
    x = np.zeros_like(c.x)
    x[0, 0] = 0x7F80
    a = np.zeros_like(c.a)
    a[0, 0, 0] = 0x3F80                     # v = [inf, 0, ...]
    a[0, 1:, 1] = 0x3F80
    b = np.zeros_like(c.b)
    b[0, :, 0] = np.where(np.arange(32) % 2, 0x3F80, 0xBF80).astype(np.uint16)
    a[0, 1:, 0] = 0x3F80                    # every v of row 0 is inf; b is 0 there: NaN by the formula
    c.st[0], c.st[1], c.st[2] = up(device, x), up(device, a), up(device, b)
    got = S.f64(c.run())
    assert np.isnan(got[0]).all() and np.isfinite(got[1:]).all()
    b[0, :, 1:] = b[0, :, :1]               # b nonzero: +inf and -inf by its sign
    c.st[2] = up(device, b)
    got = S.f64(c.run())
    sign = np.sign(c.scales[0]) * np.where(np.arange(32) % 2, 1, -1)
    assert np.array_equal(got[0], np.where(sign > 0, np.inf, -np.inf)) and np.isfinite(got[1:]).all()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("m,k,n,rank", [(1, 64, 33, 8), (3, 64, 32, 16), (12, 72, 100, 40), (40, 128, 100, 16),
                                        (40, 64, 64, 24), (200, 64, 144, 40), (90, 64, 48, 128), (1100, 136, 96, 32),
                                        (1100, 136, 101, 128), (1100, 64, 64, 16)])
def test_infinities_and_nans_of_b(device, m, k, n, rank, f32):
    """An infinite entry of B makes its column infinite, by the signs of v and
    of the entry (NaN where two of them disagree), and no other column; a NaN
    makes its column NaN. Rows of the other adapter stay as they are."""
    c = Case(device, m + rank, m, k, n, rank, 2, [i * 7 // m % 2 for i in range(m)], f32)
    clean = c.run()
    b = c.b.copy()
    b[0, 2, 3], b[0, 9, 0], b[0, n - 1, rank - 1] = 0x7F80, 0xFF80, 0x7F80
    b[0, 17, 1], b[0, 17, 6] = 0x7F80, 0xFF80
    b[0, 30, 5] = 0x7FC0
    c.st[2] = up(device, b)
    got = c.run().astype(np.float64) if f32 else S.f64(c.run())
    val = clean.astype(np.float64) if f32 else S.f64(clean)
    hit = np.isin(np.arange(n), [2, 9, 17, 30, n - 1])
    mine = c.ids == 0
    assert np.array_equal(got[~mine], val[~mine]) and np.array_equal(got[:, ~hit], val[:, ~hit])
    x, a = S.f64(c.x[mine]), S.f64(c.a[0])
    v = x @ a.T * c.scales[0]
    # rows whose v at these entries are not so near 0 that the kernel's sums may have another sign
    sure = np.abs(v) > (k + 2) * 2.0 ** -24 * (np.abs(x) @ np.abs(a).T) * abs(c.scales[0])
    sure = sure[:, [0, 1, 3, 5, 6, rank - 1]].all(1)
    assert sure.mean() > 0.9
    for col in np.flatnonzero(hit):
        with np.errstate(invalid="ignore"):
            want = (v * S.f64(b[0, col])).sum(-1)
        assert not np.isfinite(got[mine, col]).any() and not np.isfinite(want).any()
        assert np.array_equal(got[mine, col][sure], want[sure], equal_nan=True)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("m", [3, 40])
def test_v_between_the_largest_bf16_and_the_largest_f32(device, m, f32):
    """A finite v that bf16 would round to inf, times small entries of B."""
    c = Case(device, m, m, 64, 48, 8, 1, [0] * m, f32)
    x, a = np.zeros_like(c.x), np.zeros_like(c.a)
    x[:, 0] = np.where(np.arange(m) % 2, 0xFF7F, 0x7F7F)  # the largest bf16, 3.3895e38
    a[0, [0, 5], 0] = 0x3F80
    b = synth.bf16_rne((S.f64(c.b) * 2.0 ** -100).astype(np.float32))
    c.scales[:] = 1.0035  # v = 3.4014e38, past where bf16 rounds to inf (3.3962e38)
    c.x, c.a, c.b = x, a, b
    c.st[:4] = [up(device, v) for v in (x, a, b, c.scales)]
    assert np.isfinite(c.check().astype(np.float64) if f32 else S.f64(c.check())).all()


@pytest.mark.parametrize("rank", [8, 40, 128])
@pytest.mark.parametrize("m,n", [(3, 100), (40, 64), (200, 144), (1100, 96), (1100, 101)])
def test_f32_results_take_24_bits_of_v(device, m, n, rank):
    """v = scale * (power of two), so with 24 bits, times one power of two per
    column: nothing is off but three roundings. v: the product of x . A^T (one
    exact product) and scale, 2^-24. Its parts: each half a bf16 step, 2^-8, of
    what the part before lost: 2^-24. Their products are exact, the two sums of
    them within 2^-23 each (whole steps, however the matrix cores round)."""
    k, u = 8, 7
    c = Case(device, m + rank, m, k, n, rank, u, [i * u // m for i in range(m)], f32=True)
    rng = np.random.default_rng(rank + n)
    x, a, b = np.zeros((m, k)), np.zeros((u, rank, k)), np.zeros((u, n, rank))
    x[:, 3] = 2.0 ** rng.integers(-3, 4, m)
    a[:, :, 3] = 2.0 ** rng.integers(-3, 4, (u, rank))
    b[:, np.arange(n), rng.integers(0, rank, n)] = 2.0 ** rng.integers(-3, 4, n)
    c.base[:] = 0
    bits = [synth.bf16_rne(t.astype(np.float32)) for t in (x, a, b)]
    c.st[:3] = [up(device, t) for t in bits]
    got = c.run().astype(np.float64)
    ref, _, _ = S.lora(x, a, b, c.scales.astype(np.float64), c.ids, np.zeros((m, n)))
    bound = (1 + 1 + 4) * 2.0 ** -24 * np.abs(ref)
    assert (np.abs(got - ref) <= bound).all()
    # two parts (16 bits) would not do: v is its scale times a power of two
    v = c.scales
    hi = S.f64(synth.bf16_rne(v))
    two = hi + S.f64(synth.bf16_rne((v - hi).astype(np.float32)))
    assert (np.abs(two - v) > 2 * 6 * 2.0 ** -24 * np.abs(v)).any()


@pytest.mark.parametrize("rank", [24, 40, 128])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("n,y_ld", [(144, None), (96, 112), (100, None)])
def test_chunks_of_many_rows_in_windows_of_256(device, rank, f32, n, y_ld):
    """65 to 1024 rows that share two adapters: chunks of 64 and their rests,
    in whole pieces of 16 columns or not, in base's place or not."""
    ids = [NONE if i % 41 == 7 else i // 3 % 2 for i in range(300)]
    c = Case(device, rank + n, 300, 136, n, rank, 2, ids, f32, y_ld=y_ld)
    assert np.array_equal(c.check(), c.run(in_place=True))


def test_refusals(device):
    m, k, n, rank, u = 4, 64, 48, 16, 2
    nbytes = _lib.lora_workspace_bytes(m, k, rank)
    st = {key: device.zeros(size) for key, size in dict(x=m * k * 2, a=u * rank * k * 2, b=u * n * rank * 2, s=u * 4,
                                                        ids=m * 4, base=m * n * 4, y=m * n * 4,
                                                        ws=nbytes).items()}

    def args(**o):
        d = dict(dev=device.handle, x=p(st["x"]), m=m, k=k, x_ld=k, a=p(st["a"]), b=p(st["b"]), s=p(st["s"]), u=u,
                 rank=rank, n=n, ids=p(st["ids"]), base=p(st["base"]), base_ld=n, y=p(st["y"]), y_ld=n, dtype=_lib.F32,
                 ws=p(st["ws"]), nbytes=nbytes)
        assert set(o) <= set(d)
        return list((d | o).values())

    def refused(status, match="", **o):
        with pytest.raises(_lib.HipError) as e:
            _lib.call("fh_lora_add", *args(**o))
        assert e.value.status == status and match in str(e.value), str(e.value)

    bad = _lib.ERR_INVALID_ARGUMENT
    _lib.call("fh_lora_add", *args())
    _lib.call("fh_lora_add", *args(m=0))
    _lib.call("fh_lora_add", *args(n=0))
    refused(bad, dev=None)
    refused(bad, m=-1)
    refused(bad, x_ld=k - 8)
    refused(bad, x_ld=k + 4)
    refused(bad, base_ld=n - 1)
    refused(bad, y_ld=n - 1)
    refused(bad, u=0)
    refused(bad, "needed", nbytes=nbytes - 1)
    refused(bad, "aligned", x=p(st["x"], 2))
    refused(bad, "aligned", a=p(st["a"], 8))
    refused(bad, "aligned", y=p(st["y"], 2))
    refused(bad, "stride", y=p(st["base"]), y_ld=n + 1, m=2)
    refused(bad, "overlap", y=p(st["base"], 4), m=2)
    refused(bad, "overlap", y=p(st["a"]), m=2)
    refused(bad, "null", ids=None)
    refused(bad, "64 bits", u=0x7FFFFFFF, rank=128, k=0x7FFFFFF8, x_ld=0x7FFFFFF8, nbytes=1 << 62)
    for rank_ in (0, 4, 12, 136):
        refused(_lib.ERR_UNSUPPORTED, "rank", rank=rank_)
    for k_ in (0, 4, 60):
        refused(_lib.ERR_UNSUPPORTED, "k ", k=k_)
    refused(_lib.ERR_DTYPE, dtype=_lib.U32)
    refused(_lib.ERR_OUT_OF_BOUNDS, u=3)
    refused(_lib.ERR_OUT_OF_BOUNDS, n=n + 8, base_ld=n + 8, y_ld=n + 8)
    refused(_lib.ERR_FOREIGN_STORAGE, b=ctypes.c_void_p(4096))


def test_refuses_outputs_over_every_operand(device):
    m, k, n, rank, u = 4, 64, 48, 16, 2
    nbytes = _lib.lora_workspace_bytes(m, k, rank)
    st = {key: device.zeros(1 << 15) for key in ("x", "a", "b", "s", "ids", "base", "y", "ws")}
    assert nbytes <= 1 << 15

    def run(y, ws):
        _lib.call("fh_lora_add", device.handle, p(st["x"]), m, k, k, p(st["a"]), p(st["b"]), p(st["s"]), u, rank, n,
                  p(st["ids"]), p(st["base"]), n, p(st[y]), n, _lib.BF16, p(st[ws]), nbytes)

    run("y", "ws")
    run("base", "ws")
    for y, ws in [(o, "ws") for o in ("x", "a", "b", "s", "ids")] + \
                 [("y", o) for o in ("x", "a", "b", "s", "ids", "base", "y")]:
        with pytest.raises(_lib.HipError, match="overlap") as e:
            run(y, ws)
        assert e.value.status == _lib.ERR_INVALID_ARGUMENT

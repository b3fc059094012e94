"""fh_logits_probs and fh_verify_draft on the GPU against the float64
restatement (oracle/draft_ref.py).

Bounds: a probability is off by the difference to the maximum (one rounding),
its factor log2 e / t and the product (one rounding each), so 3 * 2^-24 of that
exponent in the exponent, twice (the sum has the same), by the two exponentials'
2^-22, by one rounding per addition of at most 2^12 partial sums in a row and
the division's; an exponent past -126 loses fp32's range, which leaves at most
2^-126 of the largest probability. Tokens and paths are the same numbers: sums and
comparisons are fp64 there as here.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from oracle import draft_ref as D
from oracle import serving_ref as S
from test_gpu_paged import down, p, refused, up

pytestmark = pytest.mark.gpu

NONE = D.NONE


# ------------------------------------------------------------ probabilities

def run_probs(dev, z, temperatures, offset=0):
    """z: bf16 bits or f32; offset: elements that logits and probs begin behind their storages' starts."""
    rows, n = z.shape
    s_z = up(dev, np.concatenate([np.zeros(offset, z.dtype), z.ravel()]))
    out = up(dev, np.full(offset + rows * n + 8, np.nan, np.float32))
    s_t = up(dev, temperatures) if temperatures is not None else None
    nbytes = _lib.logits_probs_workspace_bytes(rows, n)
    ws = up(dev, np.full(nbytes, 0xFF, np.uint8))
    _lib.call("fh_logits_probs", dev.handle, p(s_z, offset * z.itemsize), _lib.F32 if z.dtype == np.float32 else _lib.BF16,
              rows, n, p(s_t), p(ws), nbytes, p(out, offset * 4))
    got = down(dev, out, np.float32, (offset + rows * n + 8,))
    assert np.isnan(got[:offset]).all() and np.isnan(got[-8:]).all()  # what lies around stays
    return got[offset:-8].reshape(rows, n)


def check_probs(dev, z, temperatures=None, offset=0):
    got = run_probs(dev, z, temperatures, offset).astype(np.float64)
    z64 = z.astype(np.float64) if z.dtype == np.float32 else S.f64(z)
    ref = D.probs(z64, temperatures)
    t = np.ones(len(z)) if temperatures is None else temperatures.astype(np.float64)
    top = np.where(np.isfinite(z64), z64, -np.inf).max(-1, keepdims=True, initial=-np.inf)
    with np.errstate(all="ignore"):
        e = np.where(np.isfinite(z64) & (t > 0).reshape(-1, 1), (top - z64) / np.clip(t, 1e-30, 1e30).reshape(-1, 1), 0)
    e = np.minimum(np.nan_to_num(e * 1.4427), 200.0)
    rel = 2 * 3 * 2.0 ** -24 * e + 2 * 2.0 ** -22 + (2 ** 12 + 2) * 2.0 ** -24
    assert (np.abs(got - ref) <= rel * ref + 2.0 ** -126 * ref.max(-1, keepdims=True)).all()
    return got


@pytest.mark.parametrize("n", [1, 2, 3, 7, 8, 63, 64, 65, 511, 1000, 1024, 4097, 8192, 12345, 32003, 128256, 131073])
@pytest.mark.parametrize("f32", [False, True])
def test_probs_of_every_size(device, n, f32):
    rng = np.random.default_rng(n)
    z = (3 * rng.standard_normal((5, n))).astype(np.float32)
    z = z if f32 else synth.bf16_rne(z)
    check_probs(device, z, np.array([1.0, 0.0, 0.3, 7.0, -2.0], np.float32))
    check_probs(device, z)


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("offset", [1, 2, 3, 5, 7])
@pytest.mark.parametrize("n", [9, 1001, 20005])
def test_probs_of_rows_that_are_not_aligned(device, f32, offset, n):
    z = (2 * np.random.default_rng(offset).standard_normal((4, n))).astype(np.float32)
    check_probs(device, z if f32 else synth.bf16_rne(z), np.array([0.7, 1.0, 0.0, 1.5], np.float32), offset)


def test_probs_many_rows(device):
    z = synth.bf16_rne((3 * np.random.default_rng(4).standard_normal((700, 5003))).astype(np.float32))
    t = np.linspace(-0.2, 2.0, 700).astype(np.float32)
    got = check_probs(device, z, t)
    assert (np.abs(got.sum(-1) - 1) < 1e-5).all()
    check_probs(device, synth.bf16_rne(np.random.default_rng(5).standard_normal((65535, 3)).astype(np.float32)))


@pytest.mark.parametrize("n", [40, 3000, 40000])
@pytest.mark.parametrize("f32", [False, True])
def test_probs_infinities_nans_and_masks(device, n, f32):
    rng = np.random.default_rng(n)
    z = rng.standard_normal((12, n)).astype(np.float32)
    z[0] = -np.inf                                  # nothing is left: zeros
    z[1, rng.permutation(n)[:n - 1]] = -np.inf      # one token
    z[2, n // 2:] = -np.inf
    z[3, [1, n - 1]] = np.inf                       # two share the row
    z[4] = np.nan
    z[5, ::3] = np.nan
    z[6] = -3.3e38                                  # the lowest, all alike
    z[7], z[7, 5] = -3.3e38, 3.3e38
    z[8, 7] = np.inf                                # greedy rows
    z[9, ::2] = np.nan
    z[10] = -np.inf
    z[11] = 2.0                                     # all equal: the first
    t = np.array([1, 0.5, 1, 2, 1, 0.8, 1, 1, 0, 0, 0, 0], np.float32)
    got = check_probs(device, z if f32 else synth.bf16_rne(z), t)
    assert not got[[0, 4, 10]].any() and got[1].max() == 1 and got[3, 1] == got[3, n - 1] == 0.5
    assert got[8, 7] == 1 and got[11, 0] == 1 and got[11].sum() == 1


def test_probs_extreme_temperatures(device):
    z = np.random.default_rng(1).standard_normal((6, 2000)).astype(np.float32)
    z[:, 50:60] = -np.inf
    t = np.array([1e-38, 1e-45, 1e-5, 1e38, np.inf, np.nan], np.float32)
    got = check_probs(device, z, t)
    assert (got[:3].max(-1) == 1).all() and np.allclose(got[3:5].max(-1), 1 / 1990, rtol=1e-5)
    assert got[5, z[5].argmax()] == 1


@pytest.mark.parametrize("n", [100, 9000, 128256])
def test_probs_greedy_rows_take_the_first_of_equals(device, n):
    z = synth.bf16_rne(np.random.default_rng(2).standard_normal((40, n)).astype(np.float32))
    got = run_probs(device, z, np.zeros(40, np.float32))
    assert np.array_equal(got.argmax(-1), S.f64(z).argmax(-1)) and (got.sum(-1) == 1).all() and (got.max(-1) == 1).all()


# ------------------------------------------------------------- verification

def run_verify(dev, pr, q, tokens, parents, counts, u):
    b, width, n = pr.shape
    st = [up(dev, a) if a is not None else None for a in (pr, q, tokens, parents, counts, u)]
    out = [up(dev, np.full(b * width, 7, np.uint32)) for _ in range(2)] + [up(dev, np.full(b, 7, np.uint32))]
    nbytes = _lib.verify_draft_workspace_bytes(b, width, n)
    ws = up(dev, np.full(nbytes, 0xFF, np.uint8))
    _lib.call("fh_verify_draft", dev.handle, p(st[0]), p(st[1]), b, width, n, *[p(s) for s in st[2:]], p(ws), nbytes,
              *[p(s) for s in out])
    return [down(dev, s, np.uint32, shape) for s, shape in zip(out, ((b, width), (b, width), (b,)))]


def check_verify(dev, pr, q, tokens, parents, counts, u):
    got = run_verify(dev, pr, q, tokens, parents, counts, u)
    want = D.verify(pr, q, tokens, parents, counts, u)
    for name, a, b in zip(("path", "out_tokens", "accepted"), got, want):
        assert np.array_equal(a, b), (name, np.argwhere(a != b)[:5].tolist())
    return got


def softmax(z):
    e = np.exp(z - z.max(-1, keepdims=True))
    return (e / e.sum(-1, keepdims=True)).astype(np.float32)


def drafted(seed, b, width, n, tree, drafts, noise=0.5, spread=2.0):
    """Distributions, drafted tokens, parents, counts and uniforms as a draft model gives them."""
    rng = np.random.default_rng(seed)
    z = (spread * rng.standard_normal((b, width, n))).astype(np.float32)
    pr, q = softmax(z), softmax(z + noise * rng.standard_normal(z.shape).astype(np.float32))
    parents = np.tile(np.arange(-1, width - 1), (b, 1))
    if tree:
        parents[:, 1:] = [[rng.integers(max(0, i - 4), i) for i in range(1, width)] for _ in range(b)]
    tokens = np.zeros((b, width), np.uint32)
    for s in range(b):
        for i in range(1, width):
            row = q[s, parents[s, i]].astype(np.float64)
            if drafts:
                tokens[s, i] = min(n - 1, np.searchsorted(row.cumsum(), rng.random() * row.sum(), side="right"))
            else:
                rank = int((parents[s, :i] == parents[s, i]).sum())
                tokens[s, i] = np.argsort(-row, kind="stable")[min(rank, n - 1)]
    counts = rng.integers(0, width + 2, b).astype(np.uint32)
    counts[0] = width
    return (pr, q if drafts else None, tokens, parents.astype(np.uint32) if tree else None, counts,
            rng.random((b, width)).astype(np.float32))


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("b,width,n", [(40, 6, 5), (30, 12, 3), (300, 4, 17), (7, 33, 300), (3, 70, 1000), (9, 5, 4096),
                                       (9, 5, 4097), (4, 9, 8191), (5, 1, 2000), (3, 2, 1), (2, 200, 40), (3, 8, 33001)])
def test_verify(device, b, width, n, tree, drafts):
    got = check_verify(device, *drafted(b * width + n, b, width, n, tree, drafts))
    assert (got[2] > 0).any()


@pytest.mark.parametrize("drafts", [False, True])
def test_verify_a_full_vocabulary(device, drafts):
    check_verify(device, *drafted(5, 3, 4, 128256, drafts, drafts, spread=2.5))


@pytest.mark.parametrize("n", [50, 9001, 30004])
@pytest.mark.parametrize("at,q_at", [(0, 1), (3, 0), (2, 2), (1, 3)])
def test_verify_rows_of_any_alignment(device, n, at, q_at):
    """probs and draft_probs that begin `at` and `q_at` elements behind their storages' starts."""
    b, width = 3, 10
    pr, q, tokens, parents, counts, u = drafted(n + at, b, width, n, True, True, noise=1.5)
    behind = lambda a, skip: up(device, np.concatenate([np.full(skip, np.nan, np.float32), a.ravel()]))
    st = [behind(pr, at), behind(q, q_at)] + [up(device, a) for a in (tokens, parents, counts, u)]
    out = [up(device, np.full(b * width, 7, np.uint32)) for _ in range(2)] + [up(device, np.full(b, 7, np.uint32))]
    nbytes = _lib.verify_draft_workspace_bytes(b, width, n)
    ws = up(device, np.full(nbytes, 0xFF, np.uint8))
    _lib.call("fh_verify_draft", device.handle, p(st[0], 4 * at), p(st[1], 4 * q_at), b, width, n, *[p(s) for s in st[2:]],
              p(ws), nbytes, *[p(s) for s in out])
    want = D.verify(pr, q, tokens, parents, counts, u)
    for s, w in zip(out, want):
        assert np.array_equal(down(device, s, np.uint32, w.shape), w)


@pytest.mark.parametrize("drafts", [False, True])
def test_verify_refuses_every_child_of_wide_trees(device, drafts):
    """Many children of the root, of unlike and of the same tokens, none accepted: u is as large as it gets."""
    rng = np.random.default_rng(8)
    b, width, n = 6, 400, 900
    pr, q, _, _, _, u = drafted(9, b, width, n, False, drafts)
    tokens, parents = rng.integers(0, n, (b, width)).astype(np.uint32), np.zeros((b, width), np.uint32)
    tokens[1], tokens[2, ::2] = 3, 11
    u[:, 1:] = 1 - 2.0 ** -24
    counts = np.array([400, 400, 400, 30, 2, 1], np.uint32)
    got = check_verify(device, pr, q, tokens, parents, counts, u)
    assert got[2].min() >= 1


def test_verify_accepts_all_at_zero_draws(device):
    pr, q, tokens, _, _, u = drafted(11, 4, 9, 200, False, True)
    u[:] = 0
    got = check_verify(device, pr, q, tokens, None, None, u)
    assert (got[2] == 9).all() and np.array_equal(got[0], np.tile(np.arange(9), (4, 1)))


def test_verify_greedy_distributions(device):
    """One token has everything: drafts are accepted as far as they are the greedy ones."""
    b, width, n = 5, 6, 5000
    rng = np.random.default_rng(3)
    best = rng.integers(0, n, (b, width))
    pr = np.zeros((b, width, n), np.float32)
    np.put_along_axis(pr, best[..., None], 1.0, -1)
    tokens = np.zeros((b, width), np.uint32)
    tokens[:, 1:] = best[:, :-1]
    for s in range(1, b):
        tokens[s, s + 1 if s + 1 < width else 1] = (best[s, s if s + 1 < width else 0] + 1) % n  # wrong there
    u = rng.random((b, width)).astype(np.float32)
    for q in (None, softmax(rng.standard_normal((b, width, n)).astype(np.float32))):
        path, out, took = check_verify(device, pr, q, tokens, None, None, u)
        assert took.tolist() == [6, 2, 3, 4, 5]
        for s in range(b):
            assert out[s, :took[s]].tolist() == best[s, :took[s]].tolist()


def test_verify_where_nothing_is_left(device):
    """p = q where the draft is refused nevertheless, a row of zeros, one whose refused
    token had it all, and entries that are negative or NaN."""
    n, width = 50, 3
    rng = np.random.default_rng(6)
    pr = softmax(rng.standard_normal((5, width, n)).astype(np.float32))
    q = pr.copy()
    tokens = np.full((5, width), 4, np.uint32)
    u = np.full((5, width), 1 - 2.0 ** -24, np.float32)
    pr[1] = 0
    pr[2, 0], pr[2, 0, 4], q[2, 0, 4] = 0, 0.25, 0.5
    pr[3, 0, ::2], pr[3, 0, 1] = -1.0, np.nan
    parents = np.zeros((5, width), np.uint32)
    got = check_verify(device, pr, q, tokens, parents, None, u)
    assert got[1][1, 0] == NONE and got[1][2, 0] == 4
    # both children name the token that has everything, drawn without chance: refused at u * 1 * 1 < 0.25, then p again
    got = check_verify(device, pr, None, tokens, parents, None, u)
    assert got[1][2, 0] == 4 and got[1][1, 0] == NONE


def test_verify_passes_over_what_is_no_child(device):
    """Tokens past the vocabulary, parents that do not come before, sequences of no nodes."""
    pr, q, tokens, parents, counts, u = drafted(13, 6, 8, 60, True, True)
    tokens[0, 1:], u[:, 1:] = NONE, 0
    parents[1, 1], parents[2, 3], parents[3, 1:] = 1, 7, NONE
    tokens[4, 2] = 60
    counts[:] = [8, 8, 8, 8, 8, 0]
    got = check_verify(device, pr, q, tokens, parents, counts, u)
    assert got[2][0] == 1 and got[2][3] == 1 and got[2][5] == 0 and (got[0][5] == NONE).all() and (got[1][5] == NONE).all()


@pytest.mark.parametrize("drafts", [False, True])
def test_verify_emits_the_target_s_distribution(device, drafts):
    """The first emitted token of 60000 sequences with one distribution: each
    token's count within 5 standard deviations of a binomial's."""
    b, width, n = 60000, 4, 6
    rng = np.random.default_rng(21)
    pr = np.broadcast_to(softmax(rng.standard_normal((1, width, n)).astype(np.float32)), (b, width, n)).copy()
    q = np.broadcast_to(softmax(rng.standard_normal((1, width, n)).astype(np.float32)), (b, width, n)).copy()
    parents = np.zeros((b, width), np.uint32)  # three children of the root
    tokens = (rng.random((b, width, 1)) > q[:, :1].cumsum(-1)).sum(-1).clip(max=n - 1).astype(np.uint32)
    if not drafts:
        tokens[:] = [0, 2, 5, 1]
    u = rng.random((b, width)).astype(np.float32)
    _, out, took = run_verify(device, pr, q if drafts else None, tokens, parents, None, u)
    assert 1 <= took.min() and took.max() == 2
    have = np.bincount(out[:, 0], minlength=n)
    want = pr[0, 0].astype(np.float64)
    assert (np.abs(have - b * want) <= 5 * np.sqrt(b * want * (1 - want))).all()


# ----------------------------------------------------------------- refusals

def test_probs_refusals(device):
    rows, n = 3, 100
    nbytes = _lib.logits_probs_workspace_bytes(rows, n)
    st = {k: device.zeros(s) for k, s in dict(z=rows * n * 4, t=rows * 4, ws=nbytes, out=rows * n * 4).items()}

    def args(**o):
        a = dict(dev=device.handle, z=p(st["z"]), dtype=_lib.F32, rows=rows, n=n, t=p(st["t"]), ws=p(st["ws"]),
                 nbytes=nbytes, out=p(st["out"]))
        assert set(o) <= set(a)
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_logits_probs"
    _lib.call(name, *args())
    for o in (dict(rows=0), dict(n=0), dict(t=None), dict(dtype=_lib.BF16)):
        _lib.call(name, *args(**o))
    for o in (dict(dev=None), dict(rows=-1), dict(n=-1), dict(nbytes=nbytes - 1), dict(ws=p(st["ws"], 4)),
              dict(z=p(st["z"], 2)), dict(out=p(st["out"], 2)), dict(out=p(st["z"])), dict(out=p(st["t"])),
              dict(out=p(st["ws"]), rows=1, n=1), dict(ws=p(st["z"])), dict(ws=p(st["out"]))):
        with pytest.raises(_lib.HipError) as e:
            _lib.call(name, *args(**o))
        assert e.value.status in (bad, _lib.ERR_OUT_OF_BOUNDS) and name in str(e.value), o
    refused(_lib.ERR_DTYPE, name, *args(dtype=_lib.U32))
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(rows=65536))
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(t=p(st["t"], 4)), match="temperatures")
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(n=101))


def test_verify_refusals(device):
    b, width, n = 2, 4, 30
    nbytes = _lib.verify_draft_workspace_bytes(b, width, n)
    st = {k: device.zeros(s) for k, s in dict(pr=b * width * n * 4, q=b * width * n * 4, tok=b * width * 4,
                                              par=b * width * 4, count=b * 4, u=b * width * 4, ws=nbytes,
                                              path=b * width * 4, out=b * width * 4, took=b * 4).items()}

    def args(**o):
        a = dict(dev=device.handle, pr=p(st["pr"]), q=p(st["q"]), b=b, width=width, n=n, tok=p(st["tok"]), par=p(st["par"]),
                 count=p(st["count"]), u=p(st["u"]), ws=p(st["ws"]), nbytes=nbytes, path=p(st["path"]), out=p(st["out"]),
                 took=p(st["took"]))
        assert set(o) <= set(a)
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_verify_draft"
    _lib.call(name, *args())
    _lib.call(name, *args(b=0))
    _lib.call(name, *args(q=None, par=None, count=None))
    for o in (dict(dev=None), dict(b=-1), dict(width=0), dict(width=1025), dict(n=0), dict(nbytes=nbytes - 1),
              dict(ws=p(st["ws"], 8)), dict(pr=p(st["pr"], 2)), dict(u=p(st["u"], 2)), dict(path=p(st["out"])),
              dict(path=p(st["tok"])), dict(took=p(st["u"])), dict(out=p(st["pr"])), dict(ws=p(st["path"])),
              dict(out=p(st["path"], 1)), dict(pr=None), dict(tok=None), dict(u=None), dict(path=None), dict(out=None),
              dict(took=None)):
        with pytest.raises(_lib.HipError) as e:
            _lib.call(name, *args(**o))
        assert e.value.status in (bad, _lib.ERR_OUT_OF_BOUNDS, _lib.ERR_FOREIGN_STORAGE) and name in str(e.value), o
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(b=65536))
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(n=31))
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(par=p(st["par"], 4)), match="parents")


# ------------------------------------------------ bounds of the sums as they are

@pytest.mark.parametrize("n", [1, 7, 64, 1000, 2049, 4097, 8192, 32003, 128256, 131073, 600001])
@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows", [1, 40])
def test_probs_and_their_sums_are_as_near_as_the_additions_allow(device, n, f32, rows):
    """A thread adds at most 12 partial sums one after another (8 tokens of 4 pieces, or 4 of 8), a wavefront's
    lanes 6, a block's wavefronts 4; a lane joins J = ceil(runs / 64) runs (a product and a sum each), then one
    product and 6 sums more; a division and a product make the probability. A term of the sum has its own
    exponential and those of at most J + 1 joins, 2^-22 each, whose exponents add up to the term's own, e; the
    difference, log2 e, its division by t and the product are four roundings of that, 4 ln 2 < 3 times 2^-24 e."""
    rng = np.random.default_rng(n + rows)
    z = (3 * rng.standard_normal((rows, n))).astype(np.float32)
    z = z if f32 else synth.bf16_rne(z)
    t = np.resize(np.array([1.0, 0.3, 7.0, 0.05, 0.8], np.float32), rows)
    got = run_probs(device, z, t).astype(np.float64)
    z64 = z.astype(np.float64) if f32 else S.f64(z)
    ref = D.probs(z64, t)
    e = (z64.max(-1, keepdims=True) - z64) / t.astype(np.float64).reshape(-1, 1) * 1.4427
    runs = (n + 7) // 2048 + 1
    joins = -(-runs // 64)
    rel = 3 * 2.0 ** -24 * (e + (ref * e).sum(-1, keepdims=True)) + (joins + 3) * 2.0 ** -22 \
        + (12 + 6 + 4 + 2 * joins + 1 + 6 + 2) * 2.0 ** -24
    ok = rel * ref + 2.0 ** -126 * ref.max(-1, keepdims=True)
    assert (np.abs(got - ref) <= ok).all()
    assert (np.abs(got.sum(-1) - 1) <= ok.sum(-1)).all()


@pytest.mark.parametrize("drafts", [False, True])
@pytest.mark.parametrize("n", [300001, 4300003])
@pytest.mark.parametrize("u", [0.0, 0.5, 0.97, 0.99999])
def test_verify_rows_of_many_or_long_pieces(device, n, drafts, u):
    """More pieces than a block has threads, and pieces longer than a block takes at a time; the first sequence's
    drafted token is accepted, the second's refused, the third's row has its whole weight at the end."""
    rng = np.random.default_rng(n)
    pr, q = (softmax(rng.standard_normal((3, 2, n)).astype(np.float32)) for _ in range(2))
    pr[2, 0], pr[2, 0, n - 3:] = 0, (0.25, 0.5, 0.25)
    tokens = np.array([[0, n // 2], [0, 5], [0, 9]], np.uint32)
    draws = np.array([[u, 0], [u, 1 - 2.0 ** -24], [u, 0.5]], np.float32)
    pr[1, 0, 5] = 0
    for b in range(3):  # one sequence, whose pieces are the shortest, and all of them
        check_verify(device, pr[b:b + 1], q[b:b + 1] if drafts else None, tokens[b:b + 1], None, None, draws[b:b + 1])
    got = check_verify(device, pr, q if drafts else None, tokens, None, None, draws)
    assert got[2].tolist() == [2, 1, 1] and got[1][2, 0] >= n - 3

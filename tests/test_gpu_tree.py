"""Drafted tokens in a paged cache on the GPU: fh_paged_norm_rope_kv and
fh_paged_tree_attention against the float64 restatement (oracle/draft_ref.py).

Bounds: a bf16 output is off by at most half a step, 2^-8 of the value, from
the fp32 result behind it. The normed rotation: a head's sum of squares is off
by head_dim + 2 roundings of itself, so its root by half as many relative to each
value, and the division, the root, two products, and the rotation's three
roundings come on top, all relative to the magnitudes |n cos| + |n sin|. The
attention: the score by head_dim roundings of sum |q||k|, the difference to the
maximum, its factor (twice: constant and product) and the exponent by 2 * 2^-24
of that reach each, all in the exponent (so relative to each p, and twice, for
p's sum too); the exponential's 2^-22, p held as two bf16 parts (2^-16), and one
rounding per key in each of the two sums, relative to sum p |v|.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from foundry_amd.kv_layout import tile_k, untile_k
from oracle import draft_ref as D
from oracle import serving_ref as S
from test_gpu_paged import down, p, page_table, refused, tables, up

pytestmark = pytest.mark.gpu

NONE = S.NONE


# ------------------------------------------------------------------- append

def run_append(dev, qkv, heads, kv, hd, wq, wk, eps, cos, sin, seqs, pos, slots, table, n_pages, page, k0, v0, q0):
    st = [up(dev, a) for a in (qkv, cos, sin, pos, table, k0, v0, q0)]
    opt = [up(dev, a) if a is not None else None for a in (wq, wk, seqs, slots)]
    _lib.call("fh_paged_norm_rope_kv", dev.handle, p(st[0]), len(pos), heads, kv, hd, p(opt[0]), p(opt[1]),
              ctypes.c_float(eps), p(st[1]), p(st[2]), cos.shape[0], p(opt[2]), p(st[3]), p(opt[3]), p(st[4]),
              table.shape[0], table.shape[1], p(st[5]), p(st[6]), n_pages, page, p(st[7]))
    return [down(dev, s, np.uint16, a.shape) for s, a in ((st[5], k0), (st[6], v0), (st[7], q0))]


def check_append(dev, seed, heads, kv, hd, page, counts, tokens, table_len, norm=(True, True), placed=True, eps=1e-5,
                 named=True):
    """tokens: (sequence, position, slot) of each row; slot is left out where not placed."""
    table, n_pages = page_table(seed, counts, max(counts) + 2)
    seqs, pos, slots = (np.array(x, dtype=np.uint32) for x in zip(*tokens))
    cos, sin = tables(hd, table_len)
    x = synth.bf16_to_f32(synth.bf16_normal(seed + 1, (len(tokens), heads + 2 * kv, hd)))
    qkv = synth.bf16_rne((x * np.linspace(0.1, 9, heads + 2 * kv).reshape(-1, 1)).astype(np.float32))
    wq, wk = (synth.bf16_rne((1 + 0.5 * synth.bf16_to_f32(synth.bf16_normal(seed + i, (hd,)))).astype(np.float32))
              if on else None for i, on in zip((7, 8), norm))
    k0, v0 = (synth.bf16_normal(seed + i, (n_pages, kv, page, hd)) for i in (2, 3))
    q0 = synth.bf16_normal(seed + 4, (len(tokens), heads, hd))
    k, v, q = run_append(dev, qkv.reshape(len(tokens), -1), heads, kv, hd, wq, wk, eps, cos, sin,
                         seqs if named else None, pos, slots if placed else None, table, n_pages, page, k0, v0, q0)
    k, want_k, want_v = untile_k(k), untile_k(k0), v0.copy()
    for i, (s, j, place) in enumerate(tokens):
        place = place if placed else j
        ok = j < table_len and s < len(counts) and place < table.shape[1] * page
        at = table[s, place // page] if ok else NONE
        if at >= n_pages:
            assert np.array_equal(q[i], q0[i])
            continue
        n = S.f64(qkv[i, :heads + kv])
        for part, w in ((slice(0, heads), wq), (slice(heads, None), wk)):
            if w is not None:
                n[part] = D.norm(n[part], S.f64(w), eps)
        half = np.concatenate([-n[:, hd // 2:], n[:, :hd // 2]], -1)
        ref, mag = n * S.f64(cos[j]) + half * S.f64(sin[j]), np.abs(n * S.f64(cos[j])) + np.abs(half * S.f64(sin[j]))
        got = np.concatenate([S.f64(q[i]), S.f64(k[at, :, place % page])])
        assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + ((hd + 2) / 2 + 9) * 2.0 ** -24 * mag).all()
        want_k[at, :, place % page] = k[at, :, place % page]
        want_v[at, :, place % page] = qkv[i, heads + kv:]
    # everything else in the pools stays as it was
    assert np.array_equal(k, want_k) and np.array_equal(v, want_v)


# position = depth, slot = index behind each sequence's tokens
TREE = [(0, 20 + d, 20 + i) for i, d in enumerate([0, 1, 1, 1, 2, 2, 3])] + [(1, d, i) for i, d in enumerate([0, 1, 1, 2])]


@pytest.mark.parametrize("heads,kv,hd,page", [(4, 2, 64, 16), (6, 2, 128, 32), (5, 1, 256, 48), (3, 3, 32, 16),
                                              (2, 1, 96, 64), (3, 1, 224, 16)])
@pytest.mark.parametrize("norm", [(True, True), (False, False), (True, False), (False, True)])
def test_append_tree_nodes(device, heads, kv, hd, page, norm):
    check_append(device, hd + page, heads, kv, hd, page, [2, 1], TREE, 64, norm)


def test_append_without_slots_is_by_position(device):
    tokens = [(s, j, 0) for s, n in ((0, 37), (1, 5)) for j in range(n)]
    check_append(device, 3, 4, 2, 128, 16, [3, 1], tokens, 40, placed=False)
    check_append(device, 4, 4, 2, 128, 16, [3, 1, 1], [(i, j, 0) for i, j in enumerate([40, 0, 15])], 48, placed=False,
                 named=False)


def test_append_passes_over_what_names_no_place(device):
    # a position past the angles, a slot past the pages or of no page, no sequence, an idle row
    tokens = [(0, 3, 3), (0, 64, 4), (1, 63, 31), (1, 2, 32), (1, 2, 5 * 16), (7, 2, 2), (NONE, 2, 2), (0, NONE, 7),
              (0, 5, NONE), (0, 60, 2)]
    check_append(device, 31, 4, 2, 64, 16, [2, 2], tokens, 64)


def test_append_large_packed_batch(device):
    """Past the bytes whose stores go around the caches."""
    tokens = [(0, j, j) for j in range(3000)]
    check_append(device, 41, 8, 8, 256, 64, [47], tokens, 3000)


def test_append_norms_of_zero_and_huge_heads(device):
    heads, kv, hd = 2, 1, 64
    cos, sin = tables(hd, 4)
    qkv = np.zeros((2, 4, hd), np.uint16)
    qkv[1, :3] = 0x7F00  # 1.7e38: the squares pass fp32
    w = np.full(hd, 0x3F80, np.uint16)
    zeros, q0 = np.zeros((1, kv, 16, hd), np.uint16), np.full((2, heads, hd), 0x4000, np.uint16)
    k, v, q = run_append(device, qkv.reshape(2, -1), heads, kv, hd, w, w, 1e-6, cos, sin, np.zeros(2, np.uint32),
                         np.array([0, 1], np.uint32), None, np.zeros((1, 1), np.uint32), 1, 16, zeros, zeros, q0)
    assert not (q & 0x7FFF).any() and not (k & 0x7FFF).any()


def test_append_is_the_plain_append_without_norms(device):
    heads, kv, hd, page = 6, 2, 128, 32
    cos, sin = tables(hd, 64)
    tokens = [(s, j) for s, n in ((0, 50), (1, 9)) for j in range(n)]
    seqs, pos = (np.array(x, np.uint32) for x in zip(*tokens))
    table, n_pages = page_table(3, [2, 1], 4)
    qkv = synth.bf16_normal(1, (len(tokens), (heads + 2 * kv) * hd))
    k0, v0 = (synth.bf16_normal(i, (n_pages, kv, page, hd)) for i in (2, 3))
    q0 = synth.bf16_normal(4, (len(tokens), heads, hd))
    got = run_append(device, qkv, heads, kv, hd, None, None, 0.0, cos, sin, seqs, pos, pos, table, n_pages, page, k0, v0, q0)
    st = [up(device, a) for a in (qkv, cos, sin, seqs, pos, table, k0, v0, q0)]
    _lib.call("fh_paged_rope_kv", device.handle, p(st[0]), len(pos), heads, kv, hd, p(st[1]), p(st[2]), 64, p(st[3]),
              p(st[4]), p(st[5]), 2, 4, p(st[6]), p(st[7]), n_pages, page, p(st[8]))
    for a, s, like in zip(got, st[6:], (k0, v0, q0)):
        assert np.array_equal(a, down(device, s, np.uint16, like.shape))


# ---------------------------------------------------------------- attention

def words(seen):
    """[.., n, n] truth values as [.., n, ceil(n / 32)] u32 words."""
    n = seen.shape[-1]
    bits = np.zeros(seen.shape[:-1] + (-(-n // 32) * 32,), np.uint64)
    bits[..., :n] = seen
    return (bits.reshape(seen.shape[:-1] + (-1, 32)) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def random_masks(seed, batch, width, kind):
    rng = np.random.default_rng(seed)
    if kind == "tree":
        seen = np.zeros((batch, width, width), bool)
        for b in range(batch):
            for i in range(width):
                if i:
                    seen[b, i] = seen[b, rng.integers(max(0, i - 6), i)]
                seen[b, i, i] = True
    else:  # any bits, those of nodes behind the row's own among them
        seen = rng.random((batch, width, width)) < 0.3
    out = words(seen)
    if width % 32:  # bits past the width mean nothing
        out[..., -1] |= np.uint32(0xFFFFFFFF << (width % 32) & 0xFFFFFFFF)
    return out


def cache(seed, lens, counts, width, heads, kv, hd, page, masks="tree", pages=None, sharp=2.0):
    need = [-(-(n + c) // page) for n, c in zip(lens, counts)]
    table, n_pages = page_table(seed, need, pages or max(need) + 2)
    b = len(lens)
    q = synth.bf16_rne((synth.bf16_to_f32(synth.bf16_normal(seed + 1, (b, width, heads, hd))) * sharp).astype(np.float32))
    k, v = (synth.bf16_normal(seed + i, (n_pages, kv, page, hd)) for i in (2, 3))
    m = random_masks(seed + 5, b, width, masks) if masks else None
    return q, k, v, table, np.array(lens, np.uint32), np.array(counts, np.uint32), m


def attention(dev, q, k, v, table, lens, counts, masks, scale):
    n, kv, page, hd = k.shape
    b, width, heads, _ = q.shape
    st = [up(dev, a) for a in (q, tile_k(k), v, table, lens)]
    s_count, s_mask = (up(dev, a) if a is not None else None for a in (counts, masks))
    nbytes = _lib.paged_tree_attention_workspace_bytes(b, width, heads, kv, hd, page, table.shape[1])
    # whatever the workspace held before
    ws, out = up(dev, np.full(nbytes, 0xFF, np.uint8)), up(dev, np.full(q.shape, 0x7FC1, np.uint16))
    call = lambda: _lib.call("fh_paged_tree_attention", dev.handle, p(st[0]), b, width, heads, kv, hd, p(st[1]), p(st[2]),
                             n, page, p(st[3]), table.shape[1], p(st[4]), p(s_count), p(s_mask), ctypes.c_float(scale),
                             p(ws), nbytes, p(out))
    call()
    first = down(dev, out, np.uint16, q.shape)
    call()
    assert np.array_equal(first, down(dev, out, np.uint16, q.shape)), "the same call gave other bits"
    return first


def bound(hd, keys, ref, weight, reach):
    rel = 2 * (hd + 6) * 2.0 ** -24 * reach + 2.0 ** -22 + 2.0 ** -16 + 2 * keys * 2.0 ** -24
    return 2.0 ** -8 * np.abs(ref) + rel * weight


def check_attention(dev, q, k, v, table, lens, counts, masks, scale):
    got = S.f64(attention(dev, q, k, v, table, lens, counts, masks, scale))
    ref, weight, reach = D.tree_attend(S.f64(q), S.f64(k), S.f64(v), table, lens, counts, masks, scale)
    keys = (lens.astype(np.int64) + q.shape[1]).reshape(-1, 1, 1, 1)
    assert (np.abs(got - ref) <= bound(k.shape[3], keys, ref, weight, reach)).all()
    return got, ref


SHAPES = [(4, 2, 64), (3, 1, 128), (8, 8, 64), (8, 1, 128), (12, 1, 64), (2, 2, 256), (20, 1, 128), (16, 2, 256)]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("masks", [None, "tree", "any"])
def test_attention_short_contexts(device, heads, kv, hd, masks):
    lens = [0, 1, 15, 16, 17, 31, 33, 60, 64, 127, 128, 129, 5]
    counts = [7, 1, 2, 7, 3, 7, 5, 4, 7, 1, 7, 6, 0]
    check_attention(device, *cache(heads * hd, lens, counts, 7, heads, kv, hd, 16, masks), hd ** -0.5)


@pytest.mark.parametrize("width", [1, 2, 8, 16, 17, 31, 32, 33, 64, 65, 100, 200])
@pytest.mark.parametrize("heads,kv,hd", [(4, 1, 64), (2, 2, 128), (3, 1, 256)])
def test_attention_of_every_width(device, width, heads, kv, hd):
    lens, counts = [40, 0, 77], [width, width - width // 3, max(1, width // 2)]
    check_attention(device, *cache(width * hd, lens, counts, width, heads, kv, hd, 32), hd ** -0.5)


@pytest.mark.parametrize("masks", [None, "tree"])
def test_attention_the_widest_tree(device, masks):
    check_attention(device, *cache(91, [33], [1024], 1024, 2, 1, 64, 16, masks), 0.125)


@pytest.mark.parametrize("heads,kv,hd,page,lens,width", [
    (8, 2, 128, 16, [3000], 5), (8, 2, 128, 64, [1, 2500, 700], 9), (4, 4, 64, 32, [4097, 0, 1], 3),
    (4, 1, 256, 128, [2049], 20), (9, 3, 128, 48, [513] * 5, 12), (2, 1, 64, 16, [9000], 40), (24, 8, 128, 16, [300], 6),
    (4, 1, 128, 16, [1500, 90], 70),
])
def test_attention_split_over_the_context(device, heads, kv, hd, page, lens, width):
    counts = [width - i % 3 for i in range(len(lens))]
    check_attention(device, *cache(sum(lens) + hd, lens, counts, width, heads, kv, hd, page), hd ** -0.5)


@pytest.mark.parametrize("pages", [48, 90])
def test_attention_many_ragged_sequences(device, pages):
    lens = [(i * 7919) % 700 if i % 9 else 0 for i in range(300)]
    counts = [(i * 5) % 6 for i in range(300)]
    check_attention(device, *cache(77, lens, counts, 5, 4, 1, 64, 16, pages=pages), 64 ** -0.5)


def test_attention_idle_runs_of_a_large_batch(device):
    """Whole groups of 64 sequences without a node, at the start, between and at the end."""
    lens = [9] * 70 + [40, 900] + [3] * 130 + [5] * 3 + [0] * 80
    counts = [0] * 70 + [3, 2] + [0] * 130 + [3] * 3 + [0] * 80
    check_attention(device, *cache(80, lens, counts, 3, 4, 2, 64, 16, pages=80), 64 ** -0.5)


@pytest.mark.parametrize("pages", [8, 400])
def test_attention_more_than_1024_sequences(device, pages):
    lens = [(i * 31) % 70 if i % 13 else 0 for i in range(1100)]
    if pages > 8:
        lens[0], lens[600] = 5000, 3001
    counts = [i % 3 for i in range(1100)]
    check_attention(device, *cache(79, lens, counts, 2, 2, 1, 64, 16, pages=pages), 64 ** -0.5)


def test_attention_a_wide_table_of_short_sequences(device):
    check_attention(device, *cache(78, [40, 1, 90], [4, 3, 4], 4, 4, 2, 128, 16, pages=5000), 128 ** -0.5)


def test_attention_without_counts_takes_the_width(device):
    q, k, v, table, lens, counts, masks = cache(7, [20, 33], [6, 6], 6, 4, 2, 64, 16)
    a = attention(device, q, k, v, table, lens, counts, masks, 0.125)
    assert np.array_equal(a, attention(device, q, k, v, table, lens, None, masks, 0.125))
    assert np.array_equal(a, attention(device, q, k, v, table, lens, np.array([9, NONE], np.uint32), masks, 0.125))


def test_attention_rows_and_sequences_that_are_idle_are_zero(device):
    q, k, v, table, lens, counts, masks = cache(5, [30, 30, 30, 30, 30], [4, 2, 4, 4, 4], 4, 4, 2, 64, 16)
    capacity = table.shape[1] * 16
    lens[2], lens[3], lens[4] = capacity - 3, NONE, 0x80000000  # one place short; past any table
    got, _ = check_attention(device, q, k, v, table, lens, counts, masks, 0.125)
    assert got[0].all(-1).all() and got[1, :2].any() and not got[1, 2:].any() and not got[2:].any()
    lens[2] = capacity - 4  # fits to the last place
    got, _ = check_attention(device, q, k, v, table, lens, counts, masks, 0.125)
    assert got[2].any()


def test_attention_masks_that_leave_rows_nothing(device):
    q, k, v, table, lens, counts, masks = cache(6, [0, 0, 12], [5, 5, 5], 5, 4, 2, 128, 16)
    masks[:] = 0
    masks[0, 3] = 0b00010  # one row sees one node
    masks[1, :] = 0xFFFFFFE0  # bits past the width alone
    got, _ = check_attention(device, q, k, v, table, lens, counts, masks, 0.09)
    assert not got[0, [0, 1, 2, 4]].any() and got[0, 3].any() and not got[1].any() and got[2].any()


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("width", [6, 40])
@pytest.mark.parametrize("pages", [None, 700])
def test_attention_what_a_row_does_not_see_is_not_used(device, hd, width, pages):
    """NaN and infinities behind the nodes, in pages of no sequence, and in nodes
    that some rows see: rows that see none of them are those of a clean pool, bit for bit."""
    lens, counts = [5, 16, 37, 90], [width, width - 2, 3, width]
    q, k, v, table, lens, counts, masks = cache(9, lens, counts, width, 4, 2, hd, 16, pages=pages)
    clean = attention(device, q, k, v, table, lens, counts, masks, 0.09)
    used = np.zeros((k.shape[0], 16), bool)
    for s in range(4):
        for j in range(int(lens[s] + counts[s])):
            used[table[s, j // 16], j % 16] = True
    dirty = np.resize(np.array([0x7FC0, 0x7F80, 0xFF80, 0xFFFF, 0xFF7F], np.uint16), k.shape)
    keep = used[:, None, :, None]
    kd, vd = np.where(keep, k, dirty), np.where(keep, v, dirty)
    assert np.array_equal(clean, attention(device, q, kd, vd, table, lens, counts, masks, 0.09))
    # node 2 of every sequence, in V and K
    for s in range(4):
        j = int(lens[s]) + 2
        vd[table[s, j // 16], :, j % 16] = dirty[0, 0, 0]
        kd[table[s, j // 16], :, j % 16, 3] = 0x7FC0
    got = attention(device, q, kd, vd, table, lens, counts, masks, 0.09)
    for s in range(4):
        seen = D.visible(width, int(counts[s]), masks[s])[:, 2]
        assert seen.any() and not seen.all()
        assert np.array_equal(got[s][~seen], clean[s][~seen])
        assert np.isnan(S.f64(got[s][seen])).all()


def test_attention_infinite_values_of_nodes_and_tokens(device):
    """+inf, -inf and NaN in V of a token (every row) and of nodes (rows that see them)."""
    q, k, v, table, lens, counts, masks = cache(19, [50, 50], [9, 9], 9, 4, 1, 128, 16)
    masks[:] = words(np.tril(np.ones((2, 9, 9), bool)))
    at = lambda s, j: (table[s, j // 16], 0, j % 16)
    v[at(0, 20)][5], v[at(0, 30)][77], v[at(0, 9)][126], v[at(0, 18)][9], v[at(0, 22)][9] = (
        0x7F80, 0xFF80, 0x7FC0, 0x7F80, 0xFF80)
    v[at(0, 53)][40], v[at(0, 55)][40], v[at(0, 54)][41] = 0x7F80, 0xFF80, 0x7FC0
    got = S.f64(attention(device, q, k, v, table, lens, counts, masks, 0.05))
    assert (got[0, :, :, 5] == np.inf).all() and (got[0, :, :, 77] == -np.inf).all()
    assert np.isnan(got[0][:, :, [126, 9]]).all()
    assert np.isfinite(got[0, :3, :, 40]).all() and (got[0, 3:5, :, 40] == np.inf).all() and np.isnan(got[0, 5:, :, 40]).all()
    assert np.isfinite(got[0, :4, :, 41]).all() and np.isnan(got[0, 4:, :, 41]).all()
    rest = np.setdiff1d(np.arange(128), [5, 77, 126, 9, 40, 41])
    assert np.isfinite(got[0][:, :, rest]).all() and np.isfinite(got[1]).all()


@pytest.mark.parametrize("heads,kv,hd", [(4, 1, 64), (8, 2, 128), (4, 1, 256)])
@pytest.mark.parametrize("n,width,pages", [(250, 5, 16), (250, 5, 700), (3000, 5, None), (700, 40, 300)])
def test_attention_finite_values_of_any_size(device, heads, kv, hd, n, width, pages):
    """Values up to the type's largest: their sums pass fp32 (weights of equal keys, of keys far below a
    later one, of keys above the first ones) where what they come to does not. One sequence of each kind,
    one of ordinary values, and one with an infinity that some nodes see."""
    lens, counts = [n] * 7, [width] * 7
    q, k, v, table, lens, counts, masks = cache(hd + n, lens, counts, width, heads, kv, hd, 16, pages=pages)
    q[:], k[:] = 0, 0
    q[..., 0] = 0x3F80  # 1.0: the score is the key's dim 0
    top = synth.bf16_to_f32(np.array([0x7F7F], np.uint16))[0]
    sign = np.where(np.random.default_rng(n).random((n + width, hd)) < 0.5, -1.0, 1.0)
    ordinary = np.random.default_rng(n + 1).standard_normal((n + width, hd))
    j = np.arange(n + width)
    one = np.ones((n + width, hd))
    # (scores in powers of two, values)
    rows = [(0 * j, top * one), (0 * j, top * sign), (np.where(j % 97 == 60, 7, 0), top * sign),
            (np.where(j == n // 2, 0, -60), np.where(j == n // 2, 1.0, top)[:, None] * one),
            (0 * j, np.where(j < 30, top, 1.0)[:, None] * one), (0 * j, ordinary), (j % 5, top * one)]
    for s, (score, value) in enumerate(rows):
        score, value = synth.bf16_rne(score.astype(np.float32)), synth.bf16_rne(value.astype(np.float32))
        for i in j:
            k[table[s, i // 16], :, i % 16, 0], v[table[s, i // 16], :, i % 16] = score[i], value[i]
    at = table[6, (n + 1) // 16], slice(None), (n + 1) % 16, 5
    v[at] = 0x7F80
    got = S.f64(attention(device, q, k, v, table, lens, counts, masks, np.log(2.0)))
    ref, weight, reach = D.tree_attend(S.f64(q), S.f64(k), S.f64(v), table, lens, counts, masks, float(np.float32(np.log(2.0))))
    finite = np.isfinite(ref)
    seen = D.visible(width, width, masks[6])[:, 1]
    assert np.array_equal(~finite[6, :, :, 5], np.broadcast_to(seen[:, None], (width, heads))) and finite[:6].all()
    assert np.array_equal(got[~finite], ref[~finite])
    ok = bound(hd, n + width, ref, weight, reach)
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - ref) <= ok)[finite].all()
    # the ordinary sequence is what it is without the others, bit for bit
    alone = attention(device, q[5:6], k, v, table[5:6], lens[5:6], counts[5:6], masks[5:6], np.log(2.0)) if pages == 16 else None
    assert alone is None or np.array_equal(S.f64(alone)[0], got[5])


@pytest.mark.parametrize("hd,pages", [(64, 16), (128, None), (256, 700)])
@pytest.mark.parametrize("width", [5, 40])
def test_attention_small_values_beside_infinite_ones(device, hd, pages, width):
    """Values of 2^-90 stay what they are in rows that do not see an infinite or NaN node, and in those that do
    in the other dims; a large finite value beside the infinite one is used as well."""
    n = 190
    q, k, v, table, lens, counts, masks = cache(hd, [n, n], [width, width], width, 4, 2, hd, 16, pages=pages)
    v = synth.bf16_rne((synth.bf16_to_f32(v) * 2.0 ** -90).astype(np.float32))
    clean = attention(device, q, k, v, table, lens, counts, masks, hd ** -0.5)
    at = [(table[s, (n + 2) // 16], slice(None), (n + 2) % 16) for s in range(2)]
    v[at[0]][:, 5], v[at[0]][:, 9] = 0x7F80, 0x7FC0
    v[at[1]][:, 5], v[at[1]][:, 9] = 0x7F80, 0x7F7F  # infinite, the type's largest
    got = attention(device, q, k, v, table, lens, counts, masks, hd ** -0.5)
    ref, weight, reach = D.tree_attend(S.f64(q), S.f64(k), S.f64(v), table, lens, counts, masks, hd ** -0.5)
    ok = bound(hd, n + width, ref, weight, reach)
    rest = np.setdiff1d(np.arange(hd), [5, 9])
    for s in range(2):
        seen = D.visible(width, width, masks[s])[:, 2]
        assert seen.any() and not seen.all()
        assert (S.f64(got[s][seen])[..., 5] == np.inf).all()
        if s == 0:
            assert np.array_equal(got[s][~seen], clean[s][~seen])
            # (there the node is added to the sum apart from the others: other roundings, as many)
            assert (np.abs(S.f64(got[s, seen][..., rest]) - ref[s, seen][..., rest]) <= ok[s, seen][..., rest]).all()
            assert np.isnan(S.f64(got[s][seen])[..., 9]).all()
        else:
            assert (np.abs(S.f64(got[s, seen, :, 9]) - ref[s, seen, :, 9]) <= ok[s, seen, :, 9]).all()


@pytest.mark.parametrize("heads,kv,hd", [(2, 1, 64), (8, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("pages", [18, 600])
def test_attention_extreme_scores(device, heads, kv, hd, pages):
    """Rows whose scores are the type's lowest, its largest, -inf alone (NaN), and mixtures."""
    lens, counts = [250] * 5, [5] * 5
    q, k, v, table, lens, counts, masks = cache(hd + pages, lens, counts, 5, heads, kv, hd, 16, pages=pages)
    q[:], k[:] = 0, 0
    q[..., 0] = 0x3F80                       # 1.0: the score is the key's dim 0
    low, high = 0xFF7F, 0x7F7F               # -3.3895e38, 3.3895e38
    rows = [lambda j: low, lambda j: high if j == 201 else 0x3F80, lambda j: high if j % 100 == 3 else low,
            lambda j: 0xFF80 if j % 3 else low, lambda j: 0xFF80]
    for s, of in enumerate(rows):
        for j in range(255):
            k[table[s, j // 16], :, j % 16, 0] = of(j)
    got = S.f64(attention(device, q, k, v, table, lens, counts, masks, 1.0))
    ref, weight, _ = D.tree_attend(S.f64(q), S.f64(k), S.f64(v), table, lens, counts, masks, 1.0)
    # equal scores or none that counts: what is left is p's parts, the exponentials' and the sums' roundings
    ok = 2.0 ** -8 * np.abs(ref) + (2.0 ** -16 + 2.0 ** -22 + 2 * 255 * 2.0 ** -24) * weight
    assert np.isfinite(ref[:4]).all() and (np.abs(got - ref)[:4] <= ok[:4]).all()
    assert np.isnan(got[4]).all()


@pytest.mark.parametrize("scale,size", [(2.0 ** -126, 63), (1e-30, 49), (2e38, -60), (2e36, -60)])
@pytest.mark.parametrize("pages", [18, 600])
def test_attention_extreme_scales(device, scale, size, pages):
    """Factors at fp32's ends, with scores that they bring to a few units (hundreds for the largest)."""
    lens, counts = [250, 3], [5, 5]
    q, k, v, table, lens, counts, masks = cache(pages, lens, counts, 5, 4, 2, 64, 16, pages=pages)
    big = lambda a: synth.bf16_rne((synth.bf16_to_f32(a) * 2.0 ** size).astype(np.float32))
    q[..., 0], k[..., 0] = big(q[..., 0] * 0 + 0x3F80), big(k[..., 0])
    q[..., 1:] = 0
    check_attention(device, q, k, v, table, lens, counts, masks, scale)


def test_attention_leaves_out_entries_that_name_no_page(device):
    q, k, v, table, lens, counts, masks = cache(13, [100, 300, 40, 20], [6] * 4, 6, 4, 2, 64, 16)
    table[0, 2] = k.shape[0]          # a page in the middle
    table[1, 0] = NONE                # the first
    table[1, 19] = 0x80000001         # the nodes' last
    table[2, :] = NONE                # all of a sequence
    got, _ = check_attention(device, q, k, v, table, lens, counts, masks, 0.125)
    assert not got[2].any()


def test_attention_large_scores_do_not_overflow(device):
    check_attention(device, *cache(23, [260, 33], [8, 8], 8, 4, 2, 64, 16, sharp=40.0), 1.0)


def test_attention_sequences_share_pages(device):
    q, k, v, table, lens, counts, masks = cache(29, [70, 90], [5, 5], 5, 4, 2, 128, 16)
    table[1, :4] = table[0, :4]
    check_attention(device, q, k, v, table, lens, counts, masks, 0.09)


def test_attention_of_one_node_is_the_decode_step_s(device):
    """Width 1 against fh_paged_attention over the same keys."""
    lens = [1, 30, 700, 64]
    q, k, v, table, lens, counts, _ = cache(31, lens, [1] * 4, 1, 8, 2, 128, 16, None)
    got = S.f64(attention(device, q, k, v, table, lens, counts, None, 0.09))
    from test_gpu_paged import attention as decode
    one = S.f64(decode(device, q[:, 0], k, v, table, lens, 0.09))
    _, weight, reach = D.tree_attend(S.f64(q), S.f64(k), S.f64(v), table, lens, counts, None, 0.09)
    # each is off by its bound
    both = 2 * bound(128, 701, got, weight, reach)[:, 0]
    assert (np.abs(got[:, 0] - one) <= both).all()


def test_attention_a_pool_past_4_gib(device):
    """Pages at the far end of a pool whose offsets pass 2^32 bytes and 2^31 elements."""
    kv, hd, page, heads, width = 8, 128, 64, 8, 5
    n_pages = (5 << 30) // (kv * hd * page * 2)
    region = kv * page * hd
    pool = [device.empty(n_pages * region * 2) for _ in range(2)]
    ids = np.array([[n_pages - 1, 0, n_pages // 2 + 1]], np.uint32)
    k, v = (synth.bf16_normal(i, (3, kv, page, hd)) for i in (1, 2))
    for st, a in zip(pool, (tile_k(k), v)):
        for i, page_id in enumerate(ids[0]):
            part = np.ascontiguousarray(a[i])
            _lib.call("fh_upload", device.handle, p(st, int(page_id) * region * 2), part.ctypes.data_as(ctypes.c_void_p),
                      part.nbytes)
    q, lens = synth.bf16_normal(3, (1, width, heads, hd)), np.array([150], np.uint32)
    s_q, s_t, s_n, out = up(device, q), up(device, ids), up(device, lens), device.empty(q.nbytes)
    nbytes = _lib.paged_tree_attention_workspace_bytes(1, width, heads, kv, hd, page, 3)
    ws = device.empty(nbytes)
    _lib.call("fh_paged_tree_attention", device.handle, p(s_q), 1, width, heads, kv, hd, p(pool[0]), p(pool[1]), n_pages,
              page, p(s_t), 3, p(s_n), None, None, ctypes.c_float(0.09), p(ws), nbytes, p(out))
    got = S.f64(down(device, out, np.uint16, q.shape))
    ref, weight, reach = D.tree_attend(S.f64(q), S.f64(k), S.f64(v), np.array([[0, 1, 2]], np.uint32), lens, None, None, 0.09)
    assert (np.abs(got - ref) <= bound(hd, 155, ref, weight, reach)).all()


# ----------------------------------------------------------------- refusals

def test_append_refusals(device):
    heads, kv, hd, page, n_pages, t = 4, 2, 64, 16, 4, 3
    st = {k: device.zeros(n) for k, n in dict(qkv=t * 8 * hd * 2, wq=hd * 2, wk=hd * 2, cos=32 * hd * 2, sin=32 * hd * 2,
                                              seq=t * 4, pos=t * 4, slot=t * 4, table=2 * 2 * 4,
                                              k=n_pages * kv * page * hd * 2, v=n_pages * kv * page * hd * 2,
                                              q=t * heads * hd * 2).items()}

    def args(**o):
        a = dict(dev=device.handle, qkv=p(st["qkv"]), tokens=t, heads=heads, kv=kv, hd=hd, wq=p(st["wq"]), wk=p(st["wk"]),
                 eps=ctypes.c_float(1e-5), cos=p(st["cos"]), sin=p(st["sin"]), table_len=32, seq=p(st["seq"]),
                 pos=p(st["pos"]), slot=p(st["slot"]), table=p(st["table"]), n_seqs=2, max_pages=2, k=p(st["k"]),
                 v=p(st["v"]), n_pages=n_pages, page=page, q=p(st["q"]))
        assert set(o) <= set(a)
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_paged_norm_rope_kv"
    _lib.call(name, *args())
    _lib.call(name, *args(tokens=0))
    _lib.call(name, *args(wq=None, wk=None, slot=None))
    for o in (dict(dev=None), dict(tokens=-1), dict(page=24), dict(n_pages=0), dict(max_pages=0), dict(n_seqs=0),
              dict(table_len=0), dict(kv=0), dict(heads=0), dict(seq=None), dict(qkv=p(st["qkv"], 2)),
              dict(wq=p(st["wq"], 2)), dict(wk=p(st["wk"], 8)), dict(k=p(st["k"], 8)), dict(q=p(st["qkv"])),
              dict(q=p(st["k"])), dict(v=p(st["k"])), dict(q=p(st["slot"])), dict(q=p(st["wk"])), dict(pos=None),
              dict(eps=ctypes.c_float(-1e-5)), dict(eps=ctypes.c_float(np.nan)), dict(eps=ctypes.c_float(np.inf))):
        with pytest.raises(_lib.HipError) as e:
            _lib.call(name, *args(**o))
        assert e.value.status in (bad, _lib.ERR_FOREIGN_STORAGE, _lib.ERR_OUT_OF_BOUNDS) and name in str(e.value), o
    refused(_lib.ERR_UNSUPPORTED, name, *args(hd=48))
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(tokens=1 << 24))
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(slot=p(st["slot"], 4)), match="slots")
    other = ctypes.c_void_p(st["q"].ptr + (1 << 40))
    refused(_lib.ERR_FOREIGN_STORAGE, name, *args(wq=other), match="q_norm")


def test_attention_refusals(device):
    b, width, heads, kv, hd, page, n_pages, pages = 2, 5, 4, 2, 64, 16, 6, 3
    nbytes = _lib.paged_tree_attention_workspace_bytes(b, width, heads, kv, hd, page, pages)
    st = {k: device.zeros(n) for k, n in dict(q=b * width * heads * hd * 2, k=n_pages * kv * page * hd * 2,
                                              v=n_pages * kv * page * hd * 2, table=b * pages * 4, len=b * 4, count=b * 4,
                                              mask=b * width * 4, ws=nbytes + 8192, out=b * width * heads * hd * 2).items()}

    def args(**o):
        a = dict(dev=device.handle, q=p(st["q"]), batch=b, width=width, heads=heads, kv=kv, hd=hd, k=p(st["k"]),
                 v=p(st["v"]), n_pages=n_pages, page=page, table=p(st["table"]), pages=pages, len=p(st["len"]),
                 count=p(st["count"]), mask=p(st["mask"]), scale=ctypes.c_float(1.0), ws=p(st["ws"]), nbytes=nbytes,
                 out=p(st["out"]))
        assert set(o) <= set(a)
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_paged_tree_attention"
    _lib.call(name, *args())
    _lib.call(name, *args(batch=0))
    _lib.call(name, *args(count=None, mask=None))
    refused(bad, name, *args(dev=None))
    for o in (dict(batch=-1), dict(width=0), dict(width=1025), dict(kv=3), dict(kv=0), dict(heads=0), dict(page=8),
              dict(pages=0), dict(n_pages=0), dict(nbytes=nbytes - 1), dict(ws=p(st["ws"], 8)), dict(q=p(st["q"], 2)),
              dict(out=p(st["q"])), dict(out=p(st["v"])), dict(out=p(st["ws"])), dict(ws=p(st["k"])),
              dict(scale=ctypes.c_float(0)), dict(scale=ctypes.c_float(-1)), dict(scale=ctypes.c_float(np.nan)),
              dict(scale=ctypes.c_float(np.inf)), dict(scale=ctypes.c_float(3e38))):
        refused(bad, name, *args(**o))
    refused(_lib.ERR_UNSUPPORTED, name, *args(hd=32))
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(batch=70000))
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(len=p(st["len"], 4)), match="lengths")
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(mask=p(st["mask"], 4)), match="masks")
    with pytest.raises(_lib.HipError):
        _lib.call(name, *args(len=None))


@pytest.mark.parametrize("off", [1, 2, 3])
def test_lists_that_are_not_aligned_are_refused(device, off):
    """4-byte entries at other addresses than multiples of 4, all within their storages."""
    heads, kv, hd, page, n_pages, t = 4, 2, 64, 16, 4, 2
    big = lambda: device.zeros(n_pages * kv * page * hd * 2)
    qkv, k, v, q, cos, sin, ws = (big() for _ in range(7))
    even, odd = device.zeros(4096), device.zeros(4096)
    bad, good, at = _lib.ERR_INVALID_ARGUMENT, p(even), p(odd, off)
    for i, what in enumerate(("sequences", "positions", "slots", "page_table")):
        seq, pos, slot, table = (at if i == x else good for x in range(4))
        refused(bad, "fh_paged_norm_rope_kv", device.handle, p(qkv), t, heads, kv, hd, None, None, ctypes.c_float(0), p(cos),
                p(sin), 16, seq, pos, slot, table, 2, 2, p(k), p(v), n_pages, page, p(q), match=f"{what} must be 4-byte")
        if what != "slots":
            refused(bad, "fh_paged_rope_kv", device.handle, p(qkv), t, heads, kv, hd, p(cos), p(sin), 16, seq, pos, table, 2,
                    2, p(k), p(v), n_pages, page, p(q), match=f"{what} must be 4-byte")
    nbytes = _lib.paged_tree_attention_workspace_bytes(2, 3, heads, kv, hd, page, 2)
    assert nbytes <= n_pages * kv * page * hd * 2
    for i, what in enumerate(("page_table", "lengths", "counts", "masks")):
        table, lens, counts, masks = (at if i == x else good for x in range(4))
        refused(bad, "fh_paged_tree_attention", device.handle, p(qkv), 2, 3, heads, kv, hd, p(k), p(v), n_pages, page, table, 2,
                lens, counts, masks, ctypes.c_float(1), p(ws), nbytes, p(q), match=f"{what} must be 4-byte")
    nbytes = _lib.logits_probs_workspace_bytes(2, 30)
    assert nbytes <= n_pages * kv * page * hd * 2
    refused(bad, "fh_logits_probs", device.handle, p(qkv), _lib.F32, 2, 30, at, p(ws), nbytes, p(q),
            match="temperatures must be 4-byte")


# ------------------------------------------------------------ long contexts

def marked(seed, lens, counts, width, heads, kv, hd, page, pages):
    """A cache whose keys weigh much alike, and whose values name their key's 128: a run of keys that is
    left out or taken twice moves the dims of that run by as much as they have."""
    q, k, v, table, lens, counts, masks = cache(seed, lens, counts, width, heads, kv, hd, page, pages=pages, sharp=0.5)
    v = synth.bf16_rne((synth.bf16_to_f32(v) * 0.1).astype(np.float32))
    for s, n in enumerate(lens.astype(np.int64) + counts):
        j = np.arange(n)
        for h in range(kv):
            v[table[s, j // page], h, j % page, j // 128 % hd] = 0x4080
    return q, k, v, table, lens, counts, masks


def check_long(dev, q, k, v, table, lens, counts, masks, scale):
    got = S.f64(attention(dev, q, k, v, table, lens, counts, masks, scale))
    ref, weight, reach = D.tree_attend_whole(S.f64(q), S.f64(k), S.f64(v), table, lens, counts, masks, scale)
    keys = (lens.astype(np.int64) + q.shape[1]).reshape(-1, 1, 1, 1)
    finite = np.isfinite(ref)
    assert np.array_equal(got[~finite], ref[~finite])
    with np.errstate(invalid="ignore"):
        assert (np.abs(got - ref) <= bound(k.shape[3], keys, ref, weight, reach))[finite].all()
    return got, finite


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("infinite", [False, True])
def test_attention_of_one_long_sequence_in_an_unsplit_batch(device, hd, infinite):
    """Past 1024 sequences a block takes a whole one: 137 tiles for each of its wavefronts, so that the pages'
    places are read again four times; with infinities in tile 101 of a wavefront and in a node, in the second pass too."""
    lens, counts = [i % 4 for i in range(1026)], [1 + i % 2 for i in range(1026)]
    lens[700], counts[700] = 17500, 2
    q, k, v, table, lens, counts, masks = marked(hd, lens, counts, 2, 2, 1, hd, 16, 1200)
    if infinite:
        for j, d in ((12000, 5), (17501, 7)):
            v[table[700, j // 16], 0, j % 16, d] = 0x7F80
    got, finite = check_long(device, q, k, v, table, lens, counts, masks, hd ** -0.5)
    assert finite.all() != infinite and got[700].any(-1).all()


@pytest.mark.parametrize("hd,width,lens,page,pages", [
    (64, 600, [9000, 333, 70], 16, 700),  # 304 tiles in all: one part, every block goes over the whole batch
    (256, 600, [2500, 0, 40], 48, 70),
    (64, 256, [17500], 16, 1200),         # 128 tiles in all: four parts, 35 tiles for a wavefront
])
def test_attention_of_many_tiles(device, hd, width, lens, page, pages):
    counts = [width, width - 50, 3][:len(lens)]
    check_long(device, *marked(sum(lens) + hd, lens, counts, width, 16, 16, hd, page, pages), hd ** -0.5)

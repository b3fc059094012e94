"""The paged cache on the GPU: fh_paged_rope_kv and fh_paged_attention against
the float64 restatement (oracle/serving_ref.py).

Bounds: a bf16 output is off by at most half a step, 2^-8 of the value, from
the fp32 result behind it. The fp32 result of the rotation is off by three
roundings of its two products (3 * 2^-24 of their magnitudes). That of the
attention is off by the scores' error (head_dim roundings of sum |q||k|, and
one for the scale, in the exponent, so relative to each p; twice, for the sum
of p too), the exponential's (2^-22), p held as two bf16 parts (2^-16) and one
rounding per key in the two sums, all of them relative to sum p |v|.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from foundry_amd.kv_layout import tile_k, untile_k
from foundry_amd.llama import LlamaConfig, rope_tables
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


def tables(hd, length):
    return rope_tables(LlamaConfig(1, 64, 1, 1, hd, 64, 64), length)


def page_table(seed, counts, width, spare=3):
    """A table over a shuffled pool; entries behind a sequence's last page name no page."""
    n_pages = sum(counts) + spare
    ids = np.random.default_rng(seed).permutation(n_pages).astype(np.uint32)
    table = np.full((len(counts), width), NONE, dtype=np.uint32)
    at = 0
    for s, n in enumerate(counts):
        table[s, :n] = ids[at:at + n]
        at += n
    return table, n_pages


# ------------------------------------------------------------------- append

def run_append(dev, qkv, heads, kv, hd, cos, sin, seqs, pos, table, n_pages, page, k0, v0, q0):
    st = [up(dev, a) for a in (qkv, cos, sin, pos, table, k0, v0, q0)]
    s_seq = up(dev, seqs) if seqs is not None else None
    _lib.call("fh_paged_rope_kv", dev.handle, p(st[0]), len(pos), heads, kv, hd, p(st[1]), p(st[2]), cos.shape[0],
              p(s_seq), p(st[3]), p(st[4]), table.shape[0], table.shape[1], p(st[5]), p(st[6]), n_pages, page, p(st[7]))
    return [down(dev, s, np.uint16, a.shape) for s, a in ((st[5], k0), (st[6], v0), (st[7], q0))]


def check_append(dev, seed, heads, kv, hd, page, counts, tokens, table_len, spare=3, named=True):
    """tokens: (sequence, position) of each row."""
    width = max(counts) + 2
    table, n_pages = page_table(seed, counts, width, spare)
    seqs = np.array([s for s, _ in tokens], dtype=np.uint32)
    pos = np.array([j for _, j in tokens], dtype=np.uint32)
    cos, sin = tables(hd, table_len)
    qkv = synth.bf16_normal(seed + 1, (len(tokens), (heads + 2 * kv) * hd))
    k0, v0 = (synth.bf16_normal(seed + i, (n_pages, kv, page, hd)) for i in (2, 3))
    q0 = synth.bf16_normal(seed + 4, (len(tokens), heads, hd))
    k, v, q = run_append(dev, qkv, heads, kv, hd, cos, sin, seqs if named else None, pos, table, n_pages, page, k0, v0,
                         q0)
    rq, rk, rv, mag, place = S.append(qkv, heads, kv, cos, sin, seqs, pos, table, n_pages, page)
    k, want_k, want_v = untile_k(k), untile_k(k0), v0.copy()
    for i, at in enumerate(place):
        if at is None:
            assert np.array_equal(q[i], q0[i])
            continue
        got = np.concatenate([S.f64(q[i]), S.f64(k[at[0], :, at[1]])])
        ref = np.concatenate([rq[i], rk[i]])
        assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 3 * 2.0 ** -24 * mag[i]).all()
        want_k[at[0], :, at[1]] = k[at[0], :, at[1]]
        want_v[at[0], :, at[1]] = qkv[i].reshape(-1, hd)[heads + kv:]
    # everything else in the pools stays as it was
    assert np.array_equal(k, want_k) and np.array_equal(v, want_v)


@pytest.mark.parametrize("heads,kv,hd,page", [(4, 2, 64, 16), (6, 2, 128, 32), (5, 1, 256, 48), (3, 3, 32, 16),
                                              (2, 1, 96, 64)])
def test_append_one_token_each(device, heads, kv, hd, page):
    lens = [0, 1, page - 1, page, 2 * page + 5, 3 * page - 1, 40]
    counts = [n // page + 1 for n in lens]
    check_append(device, 11, heads, kv, hd, page, counts, list(enumerate(lens)), 200, named=False)


@pytest.mark.parametrize("page", [16, 32, 80])
def test_append_packed_prompts(device, page):
    tokens = [(0, j) for j in range(70, 173)] + [(2, j) for j in range(0, 1)] + [(1, j) for j in range(15, 34)]
    check_append(device, 21, 3, 2, 128, page, [-(-173 // page), -(-34 // page), 1], tokens, 180)


def test_append_passes_over_what_names_no_place(device):
    # idle rows, a position past the table, past the pages, a sequence that is none, an entry that names no page
    tokens = [(0, 3), (0, NONE), (1, 60), (1, 47), (7, 2), (NONE, 2), (0, 70), (1, 16 * 5), (0, 0x7FFFFFFF)]
    check_append(device, 31, 4, 2, 64, 16, [2, 3], tokens, 48)


def test_append_no_page_is_named_by_an_id_past_the_pool(device):
    heads, kv, hd, page = 2, 1, 64, 16
    cos, sin = tables(hd, 32)
    table = np.array([[1, 3], [2, 0x80000000]], dtype=np.uint32)  # 3 pages: ids 3 and 2^31 name none
    qkv = synth.bf16_normal(1, (3, 4 * hd))
    k0, v0 = (synth.bf16_normal(i, (3, kv, page, hd)) for i in (2, 3))
    q0 = synth.bf16_normal(4, (3, heads, hd))
    seqs, pos = np.array([0, 1, 1], np.uint32), np.array([17, 16, 31], np.uint32)
    k, v, q = run_append(device, qkv, heads, kv, hd, cos, sin, seqs, pos, table, 3, page, k0, v0, q0)
    assert np.array_equal(k, k0) and np.array_equal(v, v0) and np.array_equal(q, q0)


def test_append_writes_what_the_attention_layout_holds(device):
    """One page per sequence is a cache of max_len = page_size: fh_rope_kv's
    values at the same places, within the two roundings that it adds."""
    heads, kv, hd, page, t = 4, 2, 128, 64, 50
    cos, sin = tables(hd, page)
    qkv = synth.bf16_normal(5, (t, (heads + 2 * kv) * hd))
    pos = np.arange(t, dtype=np.uint32)
    zeros, q0 = np.zeros((1, kv, page, hd), np.uint16), np.zeros((t, heads, hd), np.uint16)
    k, v, q = run_append(device, qkv, heads, kv, hd, cos, sin, np.zeros(t, np.uint32), pos,
                         np.zeros((1, 1), np.uint32), 1, page, zeros, zeros, q0)
    st = [up(device, a) for a in (qkv, cos, sin, pos, zeros, zeros, q0)]
    _lib.call("fh_rope_kv", device.handle, p(st[0]), t, heads, kv, hd, p(st[1]), p(st[2]), page, p(st[3]), p(st[4]),
              p(st[5]), page, p(st[6]))
    assert np.array_equal(v, down(device, st[5], np.uint16, zeros.shape))
    _, _, _, mag, _ = S.append(qkv, heads, kv, cos, sin, np.zeros(t, np.uint32), pos, np.zeros((1, 1), np.uint32), 1,
                               page)
    other = S.f64(untile_k(down(device, st[4], np.uint16, zeros.shape)))[0, :, :t].transpose(1, 0, 2)
    mine = S.f64(untile_k(k))[0, :, :t].transpose(1, 0, 2)
    # each side rounds its result once (2^-8 each), fh_rope_kv its two products too (2^-8 of their magnitudes)
    assert (np.abs(other - mine) <= 2.0 ** -8 * 3.1 * mag[:, heads:]).all()


# ---------------------------------------------------------------- attention

def attention(dev, q, k, v, table, pos, scale, n_pages=None, page=None, q_rows=None):
    """k, v: [pages, kv, page, hd] bf16 bits, k not yet grouped."""
    n, kv, page, hd = k.shape
    b, heads = len(pos), q.shape[1]
    st = [up(dev, a) for a in (q, tile_k(k), v, table, pos)]
    nbytes = _lib.paged_attention_workspace_bytes(b, heads, kv, hd, page, table.shape[1])
    # whatever the workspace held before
    ws, out = up(dev, np.full(nbytes, 0xFF, np.uint8)), up(dev, np.full((b, heads, hd), 0x7FC1, np.uint16))
    call = lambda: _lib.call("fh_paged_attention", dev.handle, p(st[0]), b, heads, kv, hd, p(st[1]), p(st[2]), n, page,
                             p(st[3]), table.shape[1], p(st[4]), ctypes.c_float(scale), p(ws), nbytes, p(out))
    call()
    first = down(dev, out, np.uint16, q.shape)
    call()
    assert np.array_equal(first, down(dev, out, np.uint16, q.shape)), "the same call gave other bits"
    return first


def check_attention(dev, q, k, v, table, pos, scale):
    got = S.f64(attention(dev, q, k, v, table, pos, scale))
    ref, weight, reach = S.attend(S.f64(q), S.f64(k), S.f64(v), table, pos, scale)
    page, hd = k.shape[2], k.shape[3]
    n = np.array([int(j) + 1 if j < table.shape[1] * page else 1 for j in pos]).reshape(-1, 1, 1)
    rel = 2 * (hd + 1) * 2.0 ** -24 * reach + 2.0 ** -22 + 2.0 ** -16 + 2 * n * 2.0 ** -24
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + rel * weight).all()
    return got, ref


def cache(seed, lens, heads, kv, hd, page, width=None, sharp=2.0):
    counts = [-(-n // page) for n in lens]
    table, n_pages = page_table(seed, counts, width or max(counts) + 2)
    q = synth.bf16_rne((synth.bf16_to_f32(synth.bf16_normal(seed + 1, (len(lens), heads, hd))) * sharp).astype(np.float32))
    k, v = (synth.bf16_normal(seed + i, (n_pages, kv, page, hd)) for i in (2, 3))
    return q, k, v, table, np.array([n - 1 if n else NONE for n in lens], dtype=np.uint32)


SHAPES = [(4, 2, 64), (3, 1, 128), (8, 8, 64), (8, 1, 128), (12, 1, 64), (2, 2, 256), (20, 1, 128), (16, 2, 256)]


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
@pytest.mark.parametrize("page", [16, 48])
def test_attention_short_contexts(device, heads, kv, hd, page):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 0, 47, 49, 64, 65, 127, 128, 129, 200]
    check_attention(device, *cache(heads * hd + page, lens, heads, kv, hd, page), hd ** -0.5)


@pytest.mark.parametrize("heads,kv,hd,page,lens", [
    (8, 2, 128, 16, [3000]), (8, 2, 128, 64, [1, 2500, 700]), (4, 4, 64, 32, [4097, 0, 1]), (4, 1, 256, 128, [2049]),
    (9, 3, 128, 16, [513] * 5), (2, 1, 64, 16, [9000]), (24, 8, 128, 16, [300]),
])
def test_attention_split_over_the_context(device, heads, kv, hd, page, lens):
    check_attention(device, *cache(sum(lens) + hd, lens, heads, kv, hd, page), hd ** -0.5)


@pytest.mark.parametrize("width", [46, 80])
def test_attention_many_ragged_sequences(device, width):
    """A block per sequence, and (past the positions that this is for) parts
    laid out over more than 64 sequences."""
    lens = [(i * 7919) % 700 if i % 9 else 0 for i in range(300)]
    check_attention(device, *cache(77, lens, 4, 1, 64, 16, width=width), 64 ** -0.5)


@pytest.mark.parametrize("heads,kv,hd", SHAPES)
def test_attention_short_contexts_of_wide_tables(device, heads, kv, hd):
    """The parts' layout where every sequence is shorter than a step or ends near one."""
    lens = [1, 0, 17, 127, 128, 129, 255, 256, 257, 0, 0, 31, 300]
    check_attention(device, *cache(heads + hd, lens, heads, kv, hd, 16, width=100), hd ** -0.5)


def test_attention_idle_runs_of_a_large_batch(device):
    """Whole groups of 64 sequences idle, at the start, between and at the end."""
    lens = [0] * 70 + [40, 900] + [0] * 130 + [5] * 3 + [0] * 80
    check_attention(device, *cache(80, lens, 4, 2, 64, 16, width=80), 64 ** -0.5)


@pytest.mark.parametrize("width", [8, 80])
def test_attention_more_sequences_than_one_layout_holds(device, width):
    """Past 1024 sequences each is a part of its own."""
    lens = [(i * 31) % 70 if i % 13 else 0 for i in range(1100)]
    check_attention(device, *cache(79, lens, 2, 1, 64, 16, width=width), 64 ** -0.5)


@pytest.mark.parametrize("heads,kv,hd", [(2, 1, 64), (3, 3, 128)])
def test_attention_a_long_context_among_more_sequences_than_one_layout_holds(device, heads, kv, hd):
    """Past 1024 sequences, where none is split: a long one at the start, in the middle, and an idle last one."""
    lens = [(i * 31) % 40 if i % 13 else 0 for i in range(1030)]
    lens[0], lens[500], lens[1029] = 5000, 3001, 0
    check_attention(device, *cache(81, lens, heads, kv, hd, 16), hd ** -0.5)


def test_attention_a_wide_table_of_short_sequences(device):
    """A capacity far past what the sequences use."""
    check_attention(device, *cache(78, [40, 1, 90], 4, 2, 128, 16, width=5000), 128 ** -0.5)


def test_attention_idle_rows_are_zero(device):
    q, k, v, table, pos = cache(5, [30, 30, 30, 30], 4, 2, 64, 16)
    pos[1], pos[2] = table.shape[1] * 16, NONE
    got, _ = check_attention(device, q, k, v, table, pos, 0.125)
    assert not got[1].any() and not got[2].any() and got[0].any() and got[3].any()


def test_attention_all_rows_idle(device):
    q, k, v, table, pos = cache(6, [30, 30], 4, 2, 64, 16)
    pos[:] = NONE
    assert not attention(device, q, k, v, table, pos, 0.125).any()


def test_attention_what_lies_behind_the_position_is_not_used(device):
    """NaN and infinities in the slots behind each position and in pages of no
    sequence: the result is that of a clean pool, bit for bit."""
    lens = [5, 16, 37, 150, 1]
    q, k, v, table, pos = cache(9, lens, 4, 2, 128, 16)
    clean = attention(device, q, k, v, table, pos, 0.09)
    used = np.zeros((k.shape[0], 16), bool)
    for s, n in enumerate(lens):
        for j in range(n):
            used[table[s, j // 16], j % 16] = True
    dirty = np.resize(np.array([0x7FC0, 0x7F80, 0xFF80, 0xFFFF, 0xFF7F], np.uint16), k.shape)
    keep = used[:, None, :, None]
    assert np.array_equal(clean, attention(device, q, np.where(keep, k, dirty), np.where(keep, v, dirty), table, pos, 0.09))


def test_attention_leaves_out_entries_that_name_no_page(device):
    lens = [100, 300, 40, 20]
    q, k, v, table, pos = cache(13, lens, 4, 2, 64, 16)
    table[0, 2] = k.shape[0]          # a page in the middle
    table[1, 0] = NONE                # the first
    table[1, 18] = 0x80000001         # the last
    table[2, :] = NONE                # all of a sequence
    got, _ = check_attention(device, q, k, v, table, pos, 0.125)
    assert not got[2].any()


def test_attention_lowest_and_infinite_scores(device):
    """Scores of the type's lowest and -inf beside ordinary ones, a row whose
    every score is -inf, and one that holds +inf."""
    q, k, v, table, pos = cache(17, [90, 200, 70, 40], 2, 1, 64, 16)
    q[:], k[:] = 0, 0
    q[:, :, 0] = 0x3F80                      # 1.0: the score is the key's dim 0
    kk = k.reshape(-1, 16, 64)
    def put(s, j, bits):
        kk[table[s, j // 16], j % 16, 0] = bits
    for j in range(90):
        put(0, j, 0xFF7F if j != 33 else 0x3F80)   # lowest everywhere but one
    for j in range(200):
        put(1, j, 0xFF80 if j % 50 else 0x3F80)    # -inf but for four
    for j in range(70):
        put(2, j, 0xFF80)                          # -inf alone
    put(3, 7, 0x7F80)                              # +inf
    got = S.f64(attention(device, q, kk.reshape(k.shape), v, table, pos, 1.0))
    ref, weight, _ = S.attend(S.f64(q), S.f64(kk.reshape(k.shape)), S.f64(v), table, pos, 1.0)
    assert np.isnan(got[2]).all() and np.isnan(got[3]).all()
    assert (np.abs(got - ref)[:2] <= 2.0 ** -8 * np.abs(ref[:2]) + 2.0 ** -15 * weight[:2]).all()


@pytest.mark.parametrize("heads,kv,hd", [(2, 1, 64), (8, 1, 128), (4, 1, 256)])
@pytest.mark.parametrize("width", [17, 600])
def test_attention_finite_scores_up_to_the_largest_f32(device, heads, kv, hd, width):
    """Finite scores whose multiples by log2 e are not: rows whose every score
    is the type's lowest, the largest for one key or for a few, and both; at
    once for a block of its own and (the wide table) split and joined."""
    lens = [250, 250, 250, 250, 40]
    q, k, v, table, pos = cache(hd + width, lens, heads, kv, hd, 16, width=width)
    q[:], k[:] = 0, 0
    q[:, :, 0] = 0x3F80                      # 1.0: the score is the key's dim 0
    kk = k.reshape(-1, 16, hd)
    low, high = 0xFF7F, 0x7F7F               # -3.3895e38, 3.3895e38
    rows = [lambda j: low, lambda j: high if j == 201 else 0x3F80, lambda j: high if j % 100 == 3 else low,
            lambda j: 0xFF80 if j % 3 else low, lambda j: high]
    for s, of in enumerate(rows):
        for j in range(lens[s]):
            kk[table[s, j // 16], j % 16, 0] = of(j)
    kk = kk.reshape(k.shape)
    got = S.f64(attention(device, q, kk, v, table, pos, 1.0))
    ref, weight, _ = S.attend(S.f64(q), S.f64(kk), S.f64(v), table, pos, 1.0)
    # equal scores or none that counts: what is left is 2^-16 of p's parts, the exponentials' and the sums' roundings
    bound = 2.0 ** -8 * np.abs(ref) + (2.0 ** -16 + 2.0 ** -22 + 2 * 250 * 2.0 ** -24) * weight
    assert np.isfinite(ref).all() and (np.abs(got - ref) <= bound).all()


def test_attention_infinite_and_nan_values_of_used_keys(device):
    q, k, v, table, pos = cache(19, [50, 50], 4, 1, 128, 16)
    vv = v.reshape(-1, 16, 128)
    vv[table[0, 1], 3, 5] = 0x7F80
    vv[table[0, 2], 4, 77] = 0xFF80
    vv[table[0, 0], 9, 126] = 0x7FC0
    vv[table[0, 1], 2, 9] = 0x7F80
    vv[table[0, 1], 6, 9] = 0xFF80
    got = S.f64(attention(device, q, k, vv.reshape(v.shape), table, pos, 0.05))
    assert (got[0, :, 5] == np.inf).all() and (got[0, :, 77] == -np.inf).all()
    assert np.isnan(got[0, :, [126, 9]]).all()
    rest = np.setdiff1d(np.arange(128), [5, 77, 126, 9])
    assert np.isfinite(got[0][:, rest]).all() and np.isfinite(got[1]).all()


def test_attention_large_scores_do_not_overflow(device):
    q, k, v, table, pos = cache(23, [260, 33], 4, 2, 64, 16, sharp=40.0)
    check_attention(device, q, k, v, table, pos, 1.0)


def test_attention_sequences_share_pages(device):
    """Two sequences whose first pages are the same ones (a shared prefix)."""
    q, k, v, table, pos = cache(29, [70, 90], 4, 2, 128, 16)
    table[1, :4] = table[0, :4]
    check_attention(device, q, k, v, table, pos, 0.09)


def test_attention_a_pool_past_4_gib(device):
    """Pages at the far end of a pool whose offsets pass 2^32 bytes and 2^31
    elements."""
    kv, hd, page, heads = 8, 128, 64, 8
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
    q, pos = synth.bf16_normal(3, (1, heads, hd)), np.array([150], np.uint32)
    s_q, s_t, s_p, out = up(device, q), up(device, ids), up(device, pos), device.empty(q.nbytes)
    nbytes = _lib.paged_attention_workspace_bytes(1, heads, kv, hd, page, 3)
    ws = device.empty(nbytes)
    _lib.call("fh_paged_attention", device.handle, p(s_q), 1, heads, kv, hd, p(pool[0]), p(pool[1]), n_pages, page,
              p(s_t), 3, p(s_p), ctypes.c_float(0.09), p(ws), nbytes, p(out))
    got = S.f64(down(device, out, np.uint16, q.shape))
    ref, weight, _ = S.attend(S.f64(q), S.f64(k), S.f64(v), np.array([[0, 1, 2]], np.uint32), pos, 0.09)
    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 2.0 ** -14 * weight).all()
    # the append reaches the same page
    cos, sin = tables(hd, 64)
    qkv = synth.bf16_normal(7, (1, (heads + 2 * kv) * hd))
    s_qkv, s_cos, s_sin, s_pos = up(device, qkv), up(device, cos), up(device, sin), up(device, np.array([63], np.uint32))
    _lib.call("fh_paged_rope_kv", device.handle, p(s_qkv), 1, heads, kv, hd, p(s_cos), p(s_sin), 64, None, p(s_pos),
              p(s_t), 1, 3, p(pool[0]), p(pool[1]), n_pages, page, p(out))
    tail = np.empty((kv, page, hd), np.uint16)
    _lib.call("fh_download", device.handle, tail.ctypes.data_as(ctypes.c_void_p), p(pool[1], (n_pages - 1) * region * 2),
              tail.nbytes)
    assert np.array_equal(tail[:, 63], qkv.reshape(-1, hd)[heads + kv:])
    assert np.array_equal(tail[:, :63], v[0][:, :63])


def test_append_into_a_page_past_2_32_elements(device):
    """One long page (a cache that is not cut): the row of its last position
    begins past 2^32 elements, and the rows that the low 32 bits would name stay."""
    heads, kv, hd, page = 1, 1, 256, (1 << 24) + 16
    pool = [device.zeros(page * hd * 2) for _ in range(2)]
    table = device.zeros(page * hd * 2)  # cos and sin: both zero but for the last position's cos
    ones = np.full(hd, 0x3F80, np.uint16)
    last = page - 1
    _lib.call("fh_upload", device.handle, p(table, last * hd * 2), ones.ctypes.data_as(ctypes.c_void_p), ones.nbytes)
    sin = device.zeros(page * hd * 2)
    qkv = synth.bf16_normal(5, (1, 3 * hd))
    s_qkv, s_pos, s_t, out = up(device, qkv), up(device, np.array([last], np.uint32)), device.zeros(4), device.empty(hd * 2)
    _lib.call("fh_paged_rope_kv", device.handle, p(s_qkv), 1, heads, kv, hd, p(table), p(sin), page, None, p(s_pos),
              p(s_t), 1, 1, p(pool[0]), p(pool[1]), 1, page, p(out))
    q, k, v = qkv.reshape(3, hd)
    assert np.array_equal(down(device, out, np.uint16, (hd,)), q)  # cos 1, sin 0
    for st, row, is_k in ((pool[0], k, True), (pool[1], v, False)):
        group, head = np.empty((2, 16, hd), np.uint16)
        _lib.call("fh_download", device.handle, group.ctypes.data_as(ctypes.c_void_p), p(st, (page - 16) * hd * 2),
                  group.nbytes)
        _lib.call("fh_download", device.handle, head.ctypes.data_as(ctypes.c_void_p), p(st), head.nbytes)
        want = np.zeros((16, hd), np.uint16)
        want[15] = row
        assert np.array_equal(group, tile_k(want[None, None])[0, 0].reshape(16, hd) if is_k else want)
        assert not head.any()


# ----------------------------------------------------------------- refusals

def refused(status, name, *args, match=""):
    with pytest.raises(_lib.HipError) as e:
        _lib.call(name, *args)
    assert e.value.status == status and match in str(e.value), str(e.value)


def test_append_refusals(device):
    heads, kv, hd, page, n_pages, t = 4, 2, 64, 16, 4, 3
    st = {k: device.zeros(n) for k, n in dict(qkv=t * 8 * hd * 2, cos=32 * hd * 2, sin=32 * hd * 2, seq=t * 4, pos=t * 4,
                                              table=2 * 2 * 4, k=n_pages * kv * page * hd * 2,
                                              v=n_pages * kv * page * hd * 2, q=t * heads * hd * 2).items()}

    def args(**o):
        a = dict(dev=device.handle, qkv=p(st["qkv"]), tokens=t, heads=heads, kv=kv, hd=hd, cos=p(st["cos"]),
                 sin=p(st["sin"]), table_len=32, seq=p(st["seq"]), pos=p(st["pos"]), table=p(st["table"]), n_seqs=2,
                 max_pages=2, k=p(st["k"]), v=p(st["v"]), n_pages=n_pages, page=page, q=p(st["q"]))
        assert set(o) <= set(a)
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_paged_rope_kv"
    _lib.call(name, *args())
    _lib.call(name, *args(tokens=0))
    refused(bad, name, *args(dev=None))
    refused(bad, name, *args(tokens=-1))
    refused(bad, name, *args(page=24), match="multiple of 16")
    refused(bad, name, *args(page=0))
    refused(bad, name, *args(n_pages=0))
    refused(bad, name, *args(max_pages=0))
    refused(bad, name, *args(n_seqs=0))
    refused(bad, name, *args(table_len=0))
    refused(bad, name, *args(kv=0))
    refused(bad, name, *args(heads=0))
    refused(bad, name, *args(seq=None), match="sequences named")
    refused(bad, name, *args(qkv=p(st["qkv"], 2)), match="aligned")
    refused(bad, name, *args(k=p(st["k"], 8)), match="aligned")
    refused(bad, name, *args(q=p(st["qkv"])), match="overlap")
    refused(bad, name, *args(q=p(st["k"])), match="overlap")
    refused(bad, name, *args(v=p(st["k"])), match="overlap")
    refused(bad, name, *args(pos=None))
    refused(_lib.ERR_UNSUPPORTED, name, *args(hd=48))
    refused(_lib.ERR_UNSUPPORTED, name, *args(hd=288))
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(max_pages=1 << 28))
    refused(bad, name, *args(n_pages=0x7FFFFFFF, kv=0xFFFFFF, page=0x7FFFFFF0, max_pages=1, hd=32), match="64 bits")
    for key, more in (("n_pages", 5), ("n_seqs", 3), ("tokens", 4), ("table_len", 33)):
        refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(**{key: more}))
    refused(_lib.ERR_FOREIGN_STORAGE, name, *args(table=ctypes.c_void_p(64)))


def test_attention_refusals(device):
    b, heads, kv, hd, page, n_pages, width = 2, 4, 2, 64, 16, 4, 2
    nbytes = _lib.paged_attention_workspace_bytes(b, heads, kv, hd, page, width)
    st = {k: device.zeros(n) for k, n in dict(q=b * heads * hd * 2, k=max(nbytes, n_pages * kv * page * hd * 2),
                                              v=n_pages * kv * page * hd * 2, table=b * width * 4, pos=b * 4,
                                              ws=nbytes, out=b * heads * hd * 2).items()}

    def args(**o):
        a = dict(dev=device.handle, q=p(st["q"]), batch=b, heads=heads, kv=kv, hd=hd, k=p(st["k"]), v=p(st["v"]),
                 n_pages=n_pages, page=page, table=p(st["table"]), max_pages=width, pos=p(st["pos"]),
                 scale=ctypes.c_float(1.0), ws=p(st["ws"]), nbytes=nbytes, out=p(st["out"]))
        assert set(o) <= set(a)
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_paged_attention"
    _lib.call(name, *args())
    _lib.call(name, *args(batch=0))
    refused(bad, name, *args(dev=None))
    refused(bad, name, *args(kv=3), match="share")
    refused(bad, name, *args(kv=0))
    refused(bad, name, *args(page=8))
    refused(bad, name, *args(n_pages=0))
    refused(bad, name, *args(nbytes=nbytes - 1), match="needed")
    refused(bad, name, *args(q=p(st["q"], 2)), match="aligned")
    refused(bad, name, *args(ws=p(st["ws"], 4)), match="aligned")
    refused(bad, name, *args(out=p(st["q"])), match="overlap")
    refused(bad, name, *args(ws=p(st["k"])), match="overlap")
    refused(bad, name, *args(table=None))
    refused(_lib.ERR_UNSUPPORTED, name, *args(hd=96))
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(batch=65536))
    refused(_lib.ERR_OUT_OF_BOUNDS, name, *args(n_pages=1 << 20))
    refused(_lib.ERR_FOREIGN_STORAGE, name, *args(k=ctypes.c_void_p(4096)))


def test_append_refuses_outputs_over_its_device_lists(device):
    """The lists steer addresses: no output may change them under way."""
    heads, kv, hd, page, t = 4, 2, 64, 16, 3
    big = {k: device.zeros(1 << 16) for k in ("qkv", "cos", "sin", "seq", "pos", "table", "k", "v", "q")}

    def args(**o):
        a = dict(dev=device.handle, qkv=p(big["qkv"]), tokens=t, heads=heads, kv=kv, hd=hd, cos=p(big["cos"]),
                 sin=p(big["sin"]), table_len=32, seq=p(big["seq"]), pos=p(big["pos"]), table=p(big["table"]), n_seqs=2,
                 max_pages=2, k=p(big["k"]), v=p(big["v"]), n_pages=4, page=page, q=p(big["q"]))
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_paged_rope_kv"
    _lib.call(name, *args())
    for of in ("q", "k", "v"):
        for over in ("qkv", "cos", "sin", "seq", "pos", "table"):
            refused(bad, name, *args(**{of: p(big[over])}), match="overlap")
    refused(_lib.ERR_INDEX_TOO_LARGE, name, *args(tokens=1 << 24), match="tokens")


def test_attention_refuses_outputs_over_its_device_lists(device):
    b, heads, kv, hd, page, width = 2, 4, 2, 64, 16, 2
    nbytes = _lib.paged_attention_workspace_bytes(b, heads, kv, hd, page, width)
    assert nbytes <= 1 << 16
    big = {k: device.zeros(1 << 16) for k in ("q", "k", "v", "table", "pos", "ws", "out")}

    def args(**o):
        a = dict(dev=device.handle, q=p(big["q"]), batch=b, heads=heads, kv=kv, hd=hd, k=p(big["k"]), v=p(big["v"]),
                 n_pages=4, page=page, table=p(big["table"]), max_pages=width, pos=p(big["pos"]),
                 scale=ctypes.c_float(1.0), ws=p(big["ws"]), nbytes=nbytes, out=p(big["out"]))
        return list((a | o).values())

    bad, name = _lib.ERR_INVALID_ARGUMENT, "fh_paged_attention"
    _lib.call(name, *args())
    for of in ("ws", "out"):
        for over in ("q", "k", "v", "table", "pos"):
            refused(bad, name, *args(**{of: p(big[over])}), match="overlap")

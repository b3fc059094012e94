"""fh_logits_process on the GPU: bit for bit the rules taken step by step in
fp32 (oracle/serving_ref.py, each step one IEEE rounding, the result rounded
once to the logits' type), and near the same rules in float64: four steps of
half an fp32 step each, relative to the largest value on the way, and half a
step of the type.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from oracle import serving_ref as S

pytestmark = pytest.mark.gpu


def up(dev, arr):
    return dev.storage_from_bytes(np.ascontiguousarray(arr).tobytes())


def p(st, offset=0):
    return ctypes.c_void_p(st.ptr + offset) if st is not None else None


def process(dev, z, rules, in_place=False, shift=0):
    """z: float32 or bf16 bits [rows, n]; rules: numpy arrays by name. shift: elements before the rows."""
    rows, n = z.shape
    st = {k: up(dev, v) for k, v in rules.items()}
    pad = np.zeros(shift, z.dtype)
    s_z, s_out = up(dev, np.concatenate([pad, z.ravel()])), up(dev, np.full(z.size + shift, 3, z.dtype))
    fields = {k: s.ptr for k, s in st.items()}
    for key in ("history", "bias"):
        name = "history" if key == "history" else "bias_ids"
        if name in rules:
            fields[f"{key}_ld"] = rules[name].shape[1]
    u = _lib.LogitRules(**fields)
    out = s_z if in_place else s_out
    off = shift * z.dtype.itemsize
    _lib.call("fh_logits_process", dev.handle, p(s_z, off), _lib.F32 if z.dtype == np.float32 else _lib.BF16, rows, n,
              ctypes.byref(u), p(out, off))
    got = np.empty(z.size + shift, z.dtype)
    _lib.call("fh_download", dev.handle, got.ctypes.data_as(ctypes.c_void_p), p(out), got.nbytes)
    return got[shift:].reshape(z.shape)


def values(z):
    return z.astype(np.float64) if z.dtype == np.float32 else S.f64(z)


def check(dev, z, rules, **kw):
    got = process(dev, z, rules, **kw)
    assert got.tobytes() == process(dev, z, rules, **kw).tobytes(), "the same call gave other bits"
    f32 = z if z.dtype == np.float32 else synth.bf16_to_f32(z)
    with np.errstate(all="ignore"):
        want = S.logits(f32.copy(), rules, np.float32)
        exact = S.logits(values(z), rules)
    bits = want if z.dtype == np.float32 else synth.bf16_rne(want)
    nan = np.isnan(want)
    assert np.array_equal(np.isnan(values(got)), nan)
    assert np.array_equal(got[~nan].view(np.uint8), bits[~nan].view(np.uint8))
    fine = np.isfinite(exact) & np.isfinite(values(got))
    reach = np.abs(values(z)) + np.abs(exact)
    for name in ("frequency", "presence"):
        if name in rules:
            reach = reach + np.abs(rules[name].astype(np.float64))[:, None] * rules["history"].shape[1]
    if "bias_values" in rules:
        reach = reach + np.abs(rules["bias_values"].astype(np.float64)).max()
    half = 2.0 ** -24 if z.dtype == np.float32 else 2.0 ** -8
    off = np.abs(values(got)[fine] - exact[fine])
    assert (off <= half * np.abs(exact[fine]) + 5 * 2.0 ** -24 * 2 * reach[fine]).all()
    return got


def logits_of(seed, rows, n, f32):
    z = (3 * np.random.default_rng(seed).standard_normal((rows, n))).astype(np.float32)
    return z if f32 else synth.bf16_rne(z)


def rules_of(seed, rows, n, history, bias, mask, ids_max=None):
    rng = np.random.default_rng(seed)
    u = {}
    if history:
        u["history"] = rng.integers(0, ids_max or n, (rows, history)).astype(np.uint32)
        u["history_len"] = rng.integers(0, history + 1, rows).astype(np.uint32)
        u["history_len"][0] = history
        u["prompt_len"] = (u["history_len"] * rng.random(rows)).astype(np.uint32)
        u["repetition"] = rng.uniform(0.8, 1.6, rows).astype(np.float32)
        u["frequency"] = rng.uniform(-0.5, 1, rows).astype(np.float32)
        u["presence"] = rng.uniform(-0.5, 1, rows).astype(np.float32)
    if bias:
        u["bias_ids"] = rng.integers(0, n, (rows, bias)).astype(np.uint32)
        u["bias_values"] = (5 * rng.standard_normal((rows, bias))).astype(np.float32)
        u["bias_len"] = rng.integers(0, bias + 1, rows).astype(np.uint32)
    if mask:
        u["mask"] = rng.integers(0, 2 ** 32, (rows, -(-n // 32)), dtype=np.uint64).astype(np.uint32)
    return u


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("rows,n", [(1, 1), (2, 31), (3, 32), (1, 33), (5, 1000), (2, 4095), (2, 4097), (4, 32003),
                                    (1, 128256), (300, 515)])
def test_every_rule(device, rows, n, f32):
    check(device, logits_of(n, rows, n, f32), rules_of(n + 1, rows, n, 150, min(n, 40), True))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("only", ["repetition", "frequency", "presence", "bias", "mask", "none"])
def test_rules_alone(device, only, f32):
    full = rules_of(3, 4, 5003, 300, 50, True, ids_max=900)
    keep = {"bias": ["bias_ids", "bias_values", "bias_len"], "mask": ["mask"], "none": []}.get(
        only, ["history", "history_len", "prompt_len", only])
    z = logits_of(4, 4, 5003, f32)
    got = check(device, z, {k: v for k, v in full.items() if k in keep})
    if only == "none":
        assert np.array_equal(got, z)


def test_optional_lengths(device):
    """Without prompt_len every id counts as generated, without bias_len every entry is in use."""
    u = rules_of(6, 3, 700, 64, 20, False)
    del u["prompt_len"], u["bias_len"]
    check(device, logits_of(7, 3, 700, False), u)


@pytest.mark.parametrize("history", [1, 255, 257, 5000, 40000])
def test_history_lengths(device, history):
    check(device, logits_of(8, 2, 3001, False), rules_of(history, 2, 3001, history, 0, False, ids_max=60))


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("history,bias", [(40, 3000), ((1 << 20) + 5, 20), (70, 2046), (70, 2047), (70, 2048)])
def test_lists_that_need_a_table_each(device, history, bias, f32):
    """Counts and bias entries share a word up to certain lengths of the lists."""
    u = rules_of(bias, 2, 9001, history, bias, True, ids_max=50 if history > 1000 else None)
    u["bias_len"][:] = [bias, bias // 2]
    check(device, logits_of(24, 2, 9001, f32), u)


def test_lengths_past_the_lists_and_prompts_past_the_history(device):
    u = rules_of(9, 4, 900, 30, 10, False)
    u["history_len"][:] = [0, 31, 0xFFFFFFFF, 30]
    u["prompt_len"][:] = [5, 0xFFFFFFFF, 3, 30]
    u["bias_len"][:] = [0, 11, 0xFFFFFFFF, 1]
    check(device, logits_of(10, 4, 900, True), u)


def test_ids_that_are_no_token_are_passed_over(device):
    u = rules_of(11, 2, 500, 40, 12, False)
    u["history"][:, ::3] = [[500], [0xFFFFFFFF]]
    u["bias_ids"][:, ::2] = [[501], [0x80000000]]
    check(device, logits_of(12, 2, 500, False), u)


def test_an_id_listed_twice(device):
    """History ids count as often as they come; of a bias id's entries the last counts."""
    u = rules_of(13, 3, 100, 400, 64, False, ids_max=5)
    u["bias_ids"] %= 7
    check(device, logits_of(14, 3, 100, False), u)


def test_masks_that_leave_one_token_and_none(device):
    z, n = logits_of(15, 3, 1000, False), 1000
    mask = np.zeros((3, 32), np.uint32)
    mask[0, 17] = 1 << 9
    mask[2] = 0xFFFFFFFF
    got = values(check(device, z, {"mask": mask}))
    assert np.isfinite(got[0]).sum() == 1 and np.isfinite(got[0, 17 * 32 + 9])
    assert (got[1] == -np.inf).all() and np.array_equal(got[2], values(z)[2])


def test_special_logits(device):
    """Infinities, NaN, zeros of both signs and the type's lowest go through the rules; a mask covers any of them."""
    for f32 in (False, True):
        z = logits_of(16, 2, 64, f32)
        special = np.array([np.inf, -np.inf, np.nan, 0.0, -0.0, -3.38e38, 3.38e38, 1e-40], np.float32)
        z[:, :8] = special if f32 else synth.bf16_rne(special)
        u = rules_of(17, 2, 64, 200, 30, False)
        check(device, z, u)
        u["mask"] = np.array([[0, 0xFFFFFFFF], [0xFFFFFF00, 0]], np.uint32)
        got = values(check(device, z, u))
        assert (got[0, :32] == -np.inf).all() and (got[1, :8] == -np.inf).all()


@pytest.mark.parametrize("f32", [False, True])
@pytest.mark.parametrize("n,shift", [(1000, 0), (1003, 0), (1000, 1), (1000, 2)])
def test_in_place_and_off_alignment(device, n, shift, f32):
    z, u = logits_of(18, 5, n, f32), rules_of(19, 5, n, 90, 10, True)
    assert np.array_equal(check(device, z, u, shift=shift), process(device, z, u, in_place=True, shift=shift))


def test_more_rows_than_one_grid_of_blocks_holds(device):
    check(device, logits_of(20, 3000, 40, False), rules_of(21, 3000, 40, 5, 2, True))


def test_then_argmax(device):
    """The processed row's greedy token is an allowed one."""
    z, n = logits_of(22, 6, 20000, False), 20000
    u = rules_of(23, 6, n, 100, 20, True)
    got = process(device, z, u)
    s, out = up(device, got), device.empty(24)
    _lib.call("fh_argmax", device.handle, p(s), 6, n, p(out))
    ids = np.empty(6, np.uint32)
    _lib.call("fh_download", device.handle, ids.ctypes.data_as(ctypes.c_void_p), p(out), 24)
    assert np.array_equal(ids, values(got).argmax(1))
    assert ((u["mask"][np.arange(6), ids // 32] >> (ids % 32)) & 1).all()


def test_refusals(device):
    rows, n = 2, 64
    st = {k: device.zeros(size) for k, size in dict(z=rows * n * 4, out=rows * n * 4, ids=rows * 8 * 4, len=rows * 4,
                                                    f=rows * 8 * 4, mask=rows * 2 * 4).items()}

    def call(rules=None, dev=device.handle, dtype=_lib.F32, rows=rows, n=n, z=p(st["z"]), out=p(st["out"])):
        u = _lib.LogitRules(**(rules or {}))
        _lib.call("fh_logits_process", dev, z, dtype, rows, n, ctypes.byref(u), out)

    def refused(status, match="", **kw):
        with pytest.raises(_lib.HipError) as e:
            call(**kw)
        assert e.value.status == status and match in str(e.value), str(e.value)

    a = {k: s.ptr for k, s in st.items()}
    bad = _lib.ERR_INVALID_ARGUMENT
    call()
    call(rows=0)
    call(n=0)
    call(rules=dict(history=a["ids"], history_ld=8, history_len=a["len"], repetition=a["f"], bias_ids=a["ids"],
                    bias_values=a["f"], bias_ld=8, mask=a["mask"]))
    call(rules=dict(history=a["ids"], history_ld=0, history_len=a["len"], bias_ids=a["ids"], bias_values=a["f"]))
    with pytest.raises(_lib.HipError):
        _lib.call("fh_logits_process", device.handle, p(st["z"]), _lib.F32, rows, n, None, p(st["out"]))
    refused(bad, dev=None)
    refused(bad, rows=-1)
    refused(bad, "together", rules=dict(history=a["ids"], history_ld=8))
    refused(bad, "together", rules=dict(history_len=a["len"]))
    refused(bad, "history", rules=dict(frequency=a["f"]))
    refused(bad, "together", rules=dict(bias_ids=a["ids"], bias_ld=8))
    refused(bad, rules=dict(bias_ids=a["ids"], bias_values=a["f"], bias_ld=-1))
    refused(bad, "aligned", z=p(st["z"], 2), n=32)
    refused(bad, "overlap", out=p(st["z"], 4), n=32)
    refused(bad, "null", z=None)
    refused(_lib.ERR_DTYPE, dtype=_lib.U32)
    refused(_lib.ERR_INDEX_TOO_LARGE, rows=65536)
    refused(_lib.ERR_OUT_OF_BOUNDS, n=n + 1)
    refused(_lib.ERR_OUT_OF_BOUNDS, rules=dict(history=a["ids"], history_ld=9, history_len=a["len"]))
    refused(_lib.ERR_OUT_OF_BOUNDS, rules=dict(mask=a["mask"] + 8))
    refused(_lib.ERR_FOREIGN_STORAGE, rules=dict(mask=4096))


def test_refuses_out_over_a_rule(device):
    rows, n, ld = 2, 64, 8
    st = {k: device.zeros(4096) for k in ("z", "history", "history_len", "prompt_len", "repetition", "frequency",
                                          "presence", "bias_ids", "bias_values", "bias_len", "mask")}
    rules = {k: s.ptr for k, s in st.items() if k != "z"} | dict(history_ld=ld, bias_ld=ld)
    u = _lib.LogitRules(**rules)
    for dtype in (_lib.F32, _lib.BF16):
        _lib.call("fh_logits_process", device.handle, p(st["z"]), dtype, rows, n, ctypes.byref(u), p(st["z"]))
        for k in rules:
            if k.endswith("_ld"):
                continue
            with pytest.raises(_lib.HipError, match="overlap") as e:
                _lib.call("fh_logits_process", device.handle, p(st["z"]), dtype, rows, n, ctypes.byref(u), p(st[k]))
            assert e.value.status == _lib.ERR_INVALID_ARGUMENT

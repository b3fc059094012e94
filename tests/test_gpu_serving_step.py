"""The serving operators together, as a server's decode step runs them: the
embedding of each slot's token, a q4 q/k/v projection with its requests'
adapters, the append to the paged cache, attention over it, the q4 output
projection with adapters, the LM head, the logit rules over what each slot has
said, the greedy pick, and the records that move on by one. Four slots: three
requests of unlike prompt lengths and adapters, one idle.

Each stage of an eager step is held to the float64 restatement of that stage
on the inputs it had; a captured step replayed several times gives the eager
steps' tokens and caches bit for bit.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from foundry_amd.device import HipDevice
from foundry_amd.kv_layout import untile_k
from foundry_amd.llama import LlamaConfig, rope_tables
from oracle import serving_ref as S

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, HD, VOCAB, PAGE, WIDTH, RANK, STEPS = 256, 4, 2, 64, 1000, 16, 8, 8, 6
QKV = (HEADS + 2 * KV) * HD
PROMPTS = [5, 40, 31]
IDLE = 0x80000000


class Server:
    def __init__(self, dev):
        self.dev = dev
        rng = np.random.default_rng(1)
        host = {}
        for name, (n, k) in {"embed": (VOCAB, HIDDEN), "qkv": (QKV, HIDDEN), "o": (HIDDEN, HEADS * HD)}.items():
            host[name] = synth.q4_weights(len(name), n, k, 64, 7.5)
        for name, (n, k) in {"qkv": (QKV, HIDDEN), "o": (HIDDEN, HEADS * HD)}.items():
            host[name + "_lora"] = tuple(
                synth.bf16_rne((rng.standard_normal(s) * 0.1).astype(np.float32)) for s in ((3, RANK, k), (3, n, RANK)))
        cos, sin = rope_tables(LlamaConfig(1, HIDDEN, HEADS, KV, HD, 64, 64), WIDTH * PAGE)
        n_pages = 4 * WIDTH
        table = np.full((4, WIDTH), S.NONE, np.uint32)
        ids = rng.permutation(n_pages).astype(np.uint32)
        for s, n in enumerate(PROMPTS):
            count = -(-(n + STEPS + 1) // PAGE)
            table[s, :count] = ids[s * WIDTH:s * WIDTH + count]
        self.n_pages = n_pages
        history = np.zeros((4, 64), np.uint32)
        for s, n in enumerate(PROMPTS):
            history[s, :n] = rng.integers(0, VOCAB, n)
        mask = rng.integers(0, 2 ** 32, (4, -(-VOCAB // 32)), dtype=np.uint64).astype(np.uint32)
        self.host = dict(host, cos=cos, sin=sin, table=table, scales=np.array([1.0, -0.5, 2.0], np.float32),
                         adapters=np.array([2, S.NONE, 0, 1], np.uint32), history=history, mask=mask,
                         prompt_len=np.array(PROMPTS + [0], np.uint32), repetition=np.full(4, 1.3, np.float32),
                         frequency=np.full(4, 0.2, np.float32), presence=np.full(4, 0.1, np.float32),
                         bias_ids=rng.integers(0, VOCAB, (4, 5)).astype(np.uint32),
                         bias_values=np.full((4, 5), 3.0, np.float32))
        self.st = {}
        for name, v in self.host.items():
            vs = v if isinstance(v, tuple) else (v,)
            self.st[name] = tuple(dev.storage_from_bytes(np.ascontiguousarray(a).tobytes()) for a in vs)
        rows = max(sum(PROMPTS), 4)
        for name, count, size in (("x", HIDDEN, 2), ("qkv_out", QKV, 2), ("q", HEADS * HD, 2), ("attn", HEADS * HD, 2),
                                  ("o_out", HIDDEN, 2), ("logits", VOCAB, 2), ("ruled", VOCAB, 2)):
            self.st[name] = (dev.zeros(rows * count * size),)
        for name in ("k", "v"):
            self.st[name] = (dev.zeros(n_pages * KV * PAGE * HD * 2),)
        for name in ("token", "pos", "said"):
            self.st[name] = (dev.zeros(16),)
        self.ws = {"attn": _lib.paged_attention_workspace_bytes(4, HEADS, KV, HD, PAGE, WIDTH),
                   "lora": max(_lib.lora_workspace_bytes(m, k, RANK) for m in (4, rows) for k in (HIDDEN, HEADS * HD))}
        self.st["attn_ws"], self.st["lora_ws"] = ((dev.empty(n),) for n in (self.ws["attn"], self.ws["lora"]))
        self.prompt()

    def p(self, name, i=0):
        return ctypes.c_void_p(self.st[name][i].ptr)

    def put(self, name, arr):
        arr = np.ascontiguousarray(arr)
        _lib.call("fh_upload", self.dev.handle, self.p(name), arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes)

    def get(self, name, dtype, shape):
        out = np.empty(shape, dtype)
        _lib.call("fh_download", self.dev.handle, out.ctypes.data_as(ctypes.c_void_p), self.p(name), out.nbytes)
        return out

    def linear(self, x, name, rows, n, k, out, adapters):
        h = self.dev.handle
        _lib.call("fh_q4_matmul", h, self.p(x), rows, k, k, *[self.p(name, i) for i in range(3)], n, 64, self.p(out),
                  _lib.BF16)
        if adapters is not None:
            _lib.call("fh_lora_add", h, self.p(x), rows, k, k, self.p(name + "_lora", 0), self.p(name + "_lora", 1),
                      self.p("scales"), 3, RANK, n, adapters, self.p(out), n, self.p(out), n, _lib.BF16,
                      self.p("lora_ws"), self.ws["lora"])

    def append(self, rows, sequences, positions):
        _lib.call("fh_paged_rope_kv", self.dev.handle, self.p("qkv_out"), rows, HEADS, KV, HD, self.p("cos"),
                  self.p("sin"), WIDTH * PAGE, sequences, positions, self.p("table"), 4, WIDTH, self.p("k"),
                  self.p("v"), self.n_pages, PAGE, self.p("q"))

    def prompt(self):
        """The prompts' keys and values, as one packed batch; the last token of each is the first step's."""
        dev, rows = self.dev, sum(n - 1 for n in PROMPTS)
        seqs = np.repeat(np.arange(3, dtype=np.uint32), [n - 1 for n in PROMPTS])
        pos = np.concatenate([np.arange(n - 1, dtype=np.uint32) for n in PROMPTS])
        st = [dev.storage_from_bytes(np.ascontiguousarray(a).tobytes()) for a in
              (self.host["history"][seqs, pos], seqs, pos, self.host["adapters"][seqs])]
        ids, s_seq, s_pos, s_ad = (ctypes.c_void_p(s.ptr) for s in st)
        _lib.call("fh_q4_embed", dev.handle, *[self.p("embed", i) for i in range(3)], VOCAB, HIDDEN, 64, ids, rows,
                  self.p("x"))
        self.linear("x", "qkv", rows, QKV, HIDDEN, "qkv_out", s_ad)
        self.append(rows, s_seq, s_pos)
        dev.synchronize()
        self.put("token", np.array([self.host["history"][s, n - 1] for s, n in enumerate(PROMPTS)] + [0], np.uint32))
        self.put("pos", np.array([n - 1 for n in PROMPTS] + [IDLE], np.uint32))
        self.put("said", np.array(PROMPTS + [0], np.uint32))

    def step(self):
        h = self.dev.handle
        _lib.call("fh_q4_embed", h, *[self.p("embed", i) for i in range(3)], VOCAB, HIDDEN, 64, self.p("token"), 4,
                  self.p("x"))
        self.linear("x", "qkv", 4, QKV, HIDDEN, "qkv_out", self.p("adapters"))
        self.append(4, None, self.p("pos"))
        _lib.call("fh_paged_attention", h, self.p("q"), 4, HEADS, KV, HD, self.p("k"), self.p("v"), self.n_pages, PAGE,
                  self.p("table"), WIDTH, self.p("pos"), ctypes.c_float(HD ** -0.5), self.p("attn_ws"),
                  self.ws["attn"], self.p("attn"))
        self.linear("attn", "o", 4, HIDDEN, HEADS * HD, "o_out", self.p("adapters"))
        self.linear("o_out", "embed", 4, VOCAB, HIDDEN, "logits", None)
        rules = _lib.LogitRules(
            history=self.st["history"][0].ptr, history_ld=64, history_len=self.st["said"][0].ptr,
            prompt_len=self.st["prompt_len"][0].ptr, repetition=self.st["repetition"][0].ptr,
            frequency=self.st["frequency"][0].ptr, presence=self.st["presence"][0].ptr,
            bias_ids=self.st["bias_ids"][0].ptr, bias_values=self.st["bias_values"][0].ptr, bias_ld=5,
            mask=self.st["mask"][0].ptr)
        _lib.call("fh_logits_process", h, self.p("logits"), _lib.BF16, 4, VOCAB, ctypes.byref(rules), self.p("ruled"))
        _lib.call("fh_argmax", h, self.p("ruled"), 4, VOCAB, self.p("token"))
        # the token goes to its place in the history, behind the prompt
        _lib.call("fh_append_token_advance", h, self.p("token"), 4, self.p("history"), self.p("said"), 0, 64, 1)
        _lib.call("fh_advance_positions", h, self.p("pos"), 4, 1)

    def snapshot(self):
        pool = (self.n_pages, KV, PAGE, HD)
        return {"k": self.get("k", np.uint16, pool), "v": self.get("v", np.uint16, pool),
                "history": self.get("history", np.uint32, (4, 64)), "logits": self.get("ruled", np.uint16, (4, VOCAB))}


def lora_close(got, x, ab, scales, adapters, base):
    ref, mag, low = S.lora(S.f64(x), S.f64(ab[0]), S.f64(ab[1]), scales.astype(np.float64), adapters, S.f64(base))
    bound = 2.0 ** -8 * np.abs(ref) + 2.0 ** -23 * (np.abs(ref) + np.abs(S.f64(base)))
    assert (np.abs(S.f64(got) - ref) <= bound + (x.shape[1] + 2) * 2.0 ** -24 * mag + 2.0 ** -15 * low).all()


def test_each_stage_of_a_step(device):
    s = Server(device)
    pos, h = s.get("pos", np.uint32, 4), s.host
    k0, v0 = s.get("k", np.uint16, (s.n_pages, KV, PAGE, HD)), s.get("v", np.uint16, (s.n_pages, KV, PAGE, HD))
    token, said = s.get("token", np.uint32, 4), s.get("history", np.uint32, (4, 64))
    s.step()
    # q/k/v: the projection alone, then with the adapters
    x = s.get("x", np.uint16, (4, HIDDEN))
    qkv = s.get("qkv_out", np.uint16, (4, QKV))
    s.put("token", token)
    s.linear("x", "qkv", 4, QKV, HIDDEN, "logits", None)
    lora_close(qkv, x, h["qkv_lora"], h["scales"], h["adapters"], s.get("logits", np.uint16, (4, QKV)))
    # the append: every slot that is not the step's own stays
    rq, rk, rv, mag, place = S.append(qkv, HEADS, KV, h["cos"], h["sin"], np.arange(4), pos, h["table"], s.n_pages, PAGE)
    assert place[3] is None and None not in place[:3]
    q = s.get("q", np.uint16, (4, HEADS, HD))
    k, v = untile_k(s.get("k", np.uint16, k0.shape)), s.get("v", np.uint16, v0.shape)
    want_k, want_v = untile_k(k0), v0.copy()
    for i in range(3):
        page, slot = place[i]
        for got, ref, m in ((S.f64(q[i]), rq[i], mag[i, :HEADS]), (S.f64(k[page, :, slot]), rk[i], mag[i, HEADS:])):
            assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + 3 * 2.0 ** -24 * m).all()
        want_k[page, :, slot], want_v[page, :, slot] = k[page, :, slot], qkv[i].reshape(-1, HD)[HEADS + KV:]
    assert np.array_equal(k, want_k) and np.array_equal(v, want_v)
    # attention over the cache that the step has left
    attn = s.get("attn", np.uint16, (4, HEADS, HD))
    ref, weight, reach = S.attend(S.f64(q), S.f64(k), S.f64(v), h["table"], pos, HD ** -0.5)
    assert not attn[3].any()
    rel = 2 * (HD + 1) * 2.0 ** -24 * reach + 2.0 ** -15
    assert (np.abs(S.f64(attn) - ref) <= 2.0 ** -8 * np.abs(ref) + rel * weight).all()
    o = s.get("o_out", np.uint16, (4, HIDDEN))
    s.linear("attn", "o", 4, HIDDEN, HEADS * HD, "x", None)
    lora_close(o, attn.reshape(4, -1), h["o_lora"], h["scales"], h["adapters"], s.get("x", np.uint16, (4, HIDDEN)))
    # the rules, bit for bit, and the greedy token in the history
    s.linear("o_out", "embed", 4, VOCAB, HIDDEN, "logits", None)
    z = synth.bf16_to_f32(s.get("logits", np.uint16, (4, VOCAB)))
    u = {key: h[key] for key in ("prompt_len", "repetition", "frequency", "presence", "bias_ids", "bias_values", "mask")}
    want = S.logits(z, dict(u, history=said, history_len=np.array(PROMPTS + [0], np.uint32)), np.float32)
    ruled = s.get("ruled", np.uint16, (4, VOCAB))
    assert np.array_equal(ruled, synth.bf16_rne(want))
    now = s.get("history", np.uint32, (4, 64))
    for i, n in enumerate(PROMPTS):
        assert now[i, n] == S.f64(ruled[i]).argmax()
    assert np.array_equal(s.get("pos", np.uint32, 4), pos + 1)


def test_a_captured_step_replays_the_eager_ones(device):
    eager, replayed = Server(device), Server(device)
    device.capture_begin()
    replayed.step()
    graph = device.capture_end()
    for i in range(STEPS):
        eager.step()
        graph.launch()
        if i % 2:
            device.synchronize()
        a, b = eager.snapshot(), replayed.snapshot()
        for name in a:
            assert np.array_equal(a[name], b[name]), (i, name)
    lens = eager.get("said", np.uint32, 4)
    assert np.array_equal(lens[:3], np.array(PROMPTS) + STEPS)


def test_two_graphs_and_eager_calls_share_workspaces(device):
    """Two servers' captured steps over one pair of workspaces, launched in
    turn on the device's stream, beside an eager one."""
    servers = [Server(device) for _ in range(3)]
    for s in servers[1:]:
        s.st["attn_ws"], s.st["lora_ws"] = servers[0].st["attn_ws"], servers[0].st["lora_ws"]
    graphs = []
    for s in servers[:2]:
        device.capture_begin()
        s.step()
        graphs.append(device.capture_end())
    for i in range(4):
        for g in graphs:
            g.launch()
        servers[2].step()
    a, b, c = (s.snapshot() for s in servers)
    for name in a:
        assert np.array_equal(a[name], b[name]) and np.array_equal(a[name], c[name]), name


def test_another_device_s_storage_is_refused_and_its_own_stream_serves(device):
    other = HipDevice(0)
    s = Server(other)
    s.step()
    t = Server(device)
    t.step()
    assert np.array_equal(s.snapshot()["logits"], t.snapshot()["logits"])
    with pytest.raises(_lib.HipError) as e:
        s.dev, s_dev = device, s.dev
        s.append(4, None, s.p("pos"))
    assert e.value.status == _lib.ERR_FOREIGN_STORAGE
    s.dev = s_dev
    del s
    other.close()

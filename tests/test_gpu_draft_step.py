"""A serving step with drafted tokens, as a server runs it: pages for the trees'
nodes, the nodes' embeddings, per layer a q4 q/k/v projection, the normed append
at the nodes' places, tree attention and a q4 output projection, then the LM
head, the distributions, the verification and the compaction of the cache. Four
slots: three requests of unlike prompts and trees, one idle, which later becomes
a copy of another request; one request ends.

Each stage of an eager step is held to the float64 restatement of that stage on
the inputs it had; a captured step, replayed with new trees, gives the eager
steps' tokens, tables and caches bit for bit.
"""
import ctypes

import numpy as np
import pytest

from foundry_amd import _lib, synth
from foundry_amd.device import HipDevice
from foundry_amd.kv_layout import untile_k
from foundry_amd.llama import LlamaConfig, rope_tables
from oracle import draft_ref as D
from oracle import serving_ref as S
from test_gpu_tree import bound, words

pytestmark = pytest.mark.gpu

HIDDEN, HEADS, KV, HD, VOCAB, PAGE, MAX_PAGES, LAYERS, SLOTS, WIDTH, STEPS = 256, 4, 2, 64, 96, 16, 6, 2, 4, 6, 6
QKV, NODES, N_PAGES, EPS = (HEADS + 2 * KV) * HD, SLOTS * WIDTH, 20, 1e-5
PROMPTS = [5, 40, 32]
POOL = (N_PAGES, KV, PAGE, HD)
NONE = D.NONE


class Server:
    def __init__(self, dev):
        self.dev, rng = dev, np.random.default_rng(2)
        self.st, self.host = {}, {}
        shapes = {"embed": (VOCAB, HIDDEN)}
        for l in range(LAYERS):
            shapes |= {f"qkv{l}": (QKV, HIDDEN), f"o{l}": (HIDDEN, HEADS * HD)}
        for i, (name, (n, k)) in enumerate(shapes.items()):
            parts = synth.q4_weights(i, n, k, 64, 7.5)
            self.st[name] = tuple(dev.storage_from_bytes(np.ascontiguousarray(a).tobytes()) for a in parts)
        near_one = lambda: synth.bf16_rne((1 + 0.3 * rng.standard_normal(HD)).astype(np.float32))
        for l in range(LAYERS):
            self.add(f"wq{l}", near_one()), self.add(f"wk{l}", near_one())
        cos, sin = rope_tables(LlamaConfig(1, HIDDEN, HEADS, KV, HD, 64, 64), MAX_PAGES * PAGE)
        self.add("cos", cos), self.add("sin", sin)
        self.add("table", np.full((SLOTS, MAX_PAGES), NONE, np.uint32))
        self.add("lengths", np.zeros(SLOTS, np.uint32))
        self.add("refs", np.zeros(N_PAGES, np.uint32))
        self.add("temperatures", np.repeat(np.array([1.0, 0.7, 0.0, 1.3], np.float32), WIDTH))
        self.add("node_seqs", np.repeat(np.arange(SLOTS, dtype=np.uint32), WIDTH))
        # the draft model draws evenly
        self.add("draft", np.full((SLOTS, WIDTH, VOCAB), 1 / VOCAB, np.float32))
        rows = max(NODES, sum(PROMPTS))
        for name, size in (("x", HIDDEN), ("logits", VOCAB)):
            self.st[name] = (dev.zeros(rows * size * 2),)
        for l in range(LAYERS):
            for name, size in (("qkv_out", QKV), ("q", HEADS * HD), ("attn", HEADS * HD)):
                self.st[f"{name}{l}"] = (dev.zeros(rows * size * 2),)
            for name in "kv":
                self.st[f"{name}{l}"] = (dev.zeros(int(np.prod(POOL)) * 2),)
        self.st["probs"] = (dev.zeros(NODES * VOCAB * 4),)
        for name in ("tokens", "parents", "positions", "slots", "masks", "uniforms", "path", "out"):
            self.st[name] = (dev.zeros(NODES * 4),)
        for name in ("counts", "accepted", "missing"):
            self.st[name] = (dev.zeros(SLOTS * 4),)
        self.ws = {"attn_ws": _lib.paged_tree_attention_workspace_bytes(SLOTS, WIDTH, HEADS, KV, HD, PAGE, MAX_PAGES),
                   "probs_ws": _lib.logits_probs_workspace_bytes(NODES, VOCAB),
                   "verify_ws": _lib.verify_draft_workspace_bytes(SLOTS, WIDTH, VOCAB)}
        for name, n in self.ws.items():
            self.st[name] = (dev.empty(n),)
        self.pools = (_lib.PagedPool * LAYERS)(*[(self.st[f"k{l}"][0].ptr, self.st[f"v{l}"][0].ptr) for l in range(LAYERS)])
        self.cache = _lib.PagedCache(pools=self.pools, n_layers=LAYERS, n_kv=KV, head_dim=HD, n_pages=N_PAGES,
                                     page_size=PAGE, page_table=self.st["table"][0].ptr, n_seqs=SLOTS,
                                     max_pages=MAX_PAGES, lengths=self.st["lengths"][0].ptr, refs=self.st["refs"][0].ptr)
        self.prompt()

    def add(self, name, arr):
        self.host[name] = arr
        self.st[name] = (self.dev.storage_from_bytes(np.ascontiguousarray(arr).tobytes()),)

    def p(self, name, i=0):
        return ctypes.c_void_p(self.st[name][i].ptr)

    def put(self, name, arr):
        arr = np.ascontiguousarray(arr)
        _lib.call("fh_upload", self.dev.handle, self.p(name), arr.ctypes.data_as(ctypes.c_void_p), arr.nbytes)

    def get(self, name, dtype=np.uint32, shape=(SLOTS,)):
        out = np.empty(shape, dtype)
        _lib.call("fh_download", self.dev.handle, out.ctypes.data_as(ctypes.c_void_p), self.p(name), out.nbytes)
        return out

    def upload(self, arr):
        return self.dev.storage_from_bytes(np.ascontiguousarray(arr).tobytes())

    def linear(self, x, name, rows, n, k, out):
        _lib.call("fh_q4_matmul", self.dev.handle, self.p(x), rows, k, k, *[self.p(name, i) for i in range(3)], n, 64,
                  self.p(out), _lib.BF16)

    def embed(self, ids, rows):
        _lib.call("fh_q4_embed", self.dev.handle, *[self.p("embed", i) for i in range(3)], VOCAB, HIDDEN, 64, ids, rows,
                  self.p("x"))

    def append(self, l, rows, sequences, positions, slots):
        _lib.call("fh_paged_norm_rope_kv", self.dev.handle, self.p(f"qkv_out{l}"), rows, HEADS, KV, HD, self.p(f"wq{l}"),
                  self.p(f"wk{l}"), ctypes.c_float(EPS), self.p("cos"), self.p("sin"), MAX_PAGES * PAGE, sequences,
                  positions, slots, self.p("table"), SLOTS, MAX_PAGES, self.p(f"k{l}"), self.p(f"v{l}"), N_PAGES, PAGE,
                  self.p(f"q{l}"))

    def reserve(self, extra):
        _lib.call("fh_paged_reserve", self.dev.handle, ctypes.byref(self.cache), extra, self.p("missing"))

    def prompt(self):
        """Keys and values of the prompts without their last tokens, which are the first roots."""
        rng, sizes = np.random.default_rng(3), [n - 1 for n in PROMPTS] + [0]
        self.put("counts", np.array(sizes, np.uint32))
        self.reserve(self.p("counts"))
        assert not self.get("missing").any()
        seqs = np.repeat(np.arange(SLOTS, dtype=np.uint32), sizes)
        pos = np.concatenate([np.arange(n, dtype=np.uint32) for n in sizes])
        ids, s_seq, s_pos = (self.upload(a) for a in (rng.integers(0, VOCAB, len(pos)).astype(np.uint32), seqs, pos))
        self.embed(ctypes.c_void_p(ids.ptr), len(pos))
        for l in range(LAYERS):
            self.linear("x", f"qkv{l}", len(pos), QKV, HIDDEN, f"qkv_out{l}")
            self.append(l, len(pos), ctypes.c_void_p(s_seq.ptr), ctypes.c_void_p(s_pos.ptr), None)
        self.dev.synchronize()
        self.put("lengths", np.array(sizes, np.uint32))
        self.roots = rng.integers(0, VOCAB, SLOTS).astype(np.uint32)
        self.counts = np.array([WIDTH, 4, WIDTH, 0], np.uint32)

    def trees(self, seed):
        """The step's trees, drawn by the draft model from what the cache and the last step left."""
        rng, lens = np.random.default_rng(seed), self.get("lengths").astype(np.int64)
        parents = np.zeros((SLOTS, WIDTH), np.int64)
        seen = np.zeros((SLOTS, WIDTH, WIDTH), bool)
        depth = np.zeros((SLOTS, WIDTH), np.int64)
        seen[:, 0, 0] = True
        for s in range(SLOTS):
            for i in range(1, WIDTH):
                parents[s, i] = rng.integers(max(0, i - 3), i)
                seen[s, i], depth[s, i] = seen[s, parents[s, i]], depth[s, parents[s, i]] + 1
                seen[s, i, i] = True
        tokens = rng.integers(0, VOCAB, (SLOTS, WIDTH))
        tokens[:, 0] = self.roots
        used = np.arange(WIDTH) < self.counts[:, None]
        self.put("tokens", tokens.astype(np.uint32))
        self.put("parents", parents.astype(np.uint32))
        self.put("positions", np.where(used, lens[:, None] + depth, NONE).astype(np.uint32))
        self.put("slots", (lens[:, None] + np.arange(WIDTH)).astype(np.uint32))
        self.put("masks", words(seen))
        self.put("uniforms", rng.random((SLOTS, WIDTH), np.float32))
        self.put("counts", self.counts)

    def step(self, compact=True):
        h = self.dev.handle
        self.reserve(self.p("counts"))
        self.embed(self.p("tokens"), NODES)
        for l in range(LAYERS):
            self.linear("x", f"qkv{l}", NODES, QKV, HIDDEN, f"qkv_out{l}")
            self.append(l, NODES, self.p("node_seqs"), self.p("positions"), self.p("slots"))
            _lib.call("fh_paged_tree_attention", h, self.p(f"q{l}"), SLOTS, WIDTH, HEADS, KV, HD, self.p(f"k{l}"),
                      self.p(f"v{l}"), N_PAGES, PAGE, self.p("table"), MAX_PAGES, self.p("lengths"), self.p("counts"),
                      self.p("masks"), ctypes.c_float(HD ** -0.5), self.p("attn_ws"), self.ws["attn_ws"],
                      self.p(f"attn{l}"))
            self.linear(f"attn{l}", f"o{l}", NODES, HIDDEN, HEADS * HD, "x")
        self.linear("x", "embed", NODES, VOCAB, HIDDEN, "logits")
        _lib.call("fh_logits_probs", h, self.p("logits"), _lib.BF16, NODES, VOCAB, self.p("temperatures"),
                  self.p("probs_ws"), self.ws["probs_ws"], self.p("probs"))
        _lib.call("fh_verify_draft", h, self.p("probs"), self.p("draft"), SLOTS, WIDTH, VOCAB, self.p("tokens"),
                  self.p("parents"), self.p("counts"), self.p("uniforms"), self.p("verify_ws"), self.ws["verify_ws"],
                  self.p("path"), self.p("out"), self.p("accepted"))
        if compact:
            self.compact()

    def compact(self):
        _lib.call("fh_paged_compact", self.dev.handle, ctypes.byref(self.cache), self.p("path"), self.p("accepted"), WIDTH,
                  self.p("lengths"))

    def emitted(self):
        """What the step emitted; its last tokens are the next roots."""
        out, accepted = self.get("out", shape=(SLOTS, WIDTH)), self.get("accepted")
        for s in range(SLOTS):
            assert (out[s, accepted[s]:] == NONE).all() and (out[s, :accepted[s]] < VOCAB).all()
            if accepted[s]:
                self.roots[s] = out[s, accepted[s] - 1]
        return out

    def fork(self, src, dst):
        st = [self.upload(np.array([x], np.uint32)) for x in (src, dst)]
        _lib.call("fh_paged_fork", self.dev.handle, ctypes.byref(self.cache), ctypes.c_void_p(st[0].ptr),
                  ctypes.c_void_p(st[1].ptr), 1, self.p("missing"))
        assert self.get("missing")[0] == 0
        self.roots[dst] = self.roots[src]

    def free(self, seq):
        st = self.upload(np.array([seq], np.uint32))
        _lib.call("fh_paged_free", self.dev.handle, ctypes.byref(self.cache), ctypes.c_void_p(st.ptr), 1)
        self.dev.synchronize()

    def between(self, i):
        """What a server does between steps: a request is copied into the idle slot, another ends."""
        if i == 1:
            self.fork(1, 3)
            self.counts = np.array([WIDTH, 4, WIDTH, 5], np.uint32)
        if i == 3:
            self.free(0)
            self.counts = np.array([0, 4, WIDTH, 5], np.uint32)

    def pages(self):
        k, v = (np.stack([self.get(f"{n}{l}", np.uint16, POOL) for l in range(LAYERS)]) for n in "kv")
        return D.Pages(self.get("table", shape=(SLOTS, MAX_PAGES)), self.get("lengths"), self.get("refs", shape=(N_PAGES,)),
                       untile_k(k), v, PAGE)

    def snapshot(self):
        a = self.pages()
        return {"k": a.k, "v": a.v, "table": a.table, "lengths": a.lengths, "refs": a.refs,
                "probs": self.get("probs", np.float32, (NODES, VOCAB)), "path": self.get("path", shape=(SLOTS, WIDTH)),
                "out": self.get("out", shape=(SLOTS, WIDTH))}


def same(a, b, what):
    for name in a:
        assert np.array_equal(a[name], b[name]), (what, name)


def test_each_stage_of_a_step(device):
    s = Server(device)
    for i in range(3):
        s.between(i)
        s.trees(10 + i)
        was = s.pages()
        s.step(compact=False)
        # pages
        was.reserve(s.counts)
        now = s.pages()
        for name in ("table", "lengths", "refs"):
            assert np.array_equal(getattr(now, name), getattr(was, name)), name
        assert not s.get("missing").any()
        # the nodes' keys and values, and nothing else
        pos, slots = s.get("positions", shape=(SLOTS, WIDTH)), s.get("slots", shape=(SLOTS, WIDTH))
        masks = s.get("masks", shape=(SLOTS, WIDTH, 1))
        for l in range(LAYERS):
            qkv = S.f64(s.get(f"qkv_out{l}", np.uint16, (SLOTS, WIDTH, HEADS + 2 * KV, HD)))
            q = s.get(f"q{l}", np.uint16, (SLOTS, WIDTH, HEADS, HD))
            for b in range(SLOTS):
                for j in range(s.counts[b]):
                    n = qkv[b, j, :HEADS + KV].copy()
                    n[:HEADS] = D.norm(n[:HEADS], S.f64(s.host[f"wq{l}"]), EPS)
                    n[HEADS:] = D.norm(n[HEADS:], S.f64(s.host[f"wk{l}"]), EPS)
                    half = np.concatenate([-n[:, HD // 2:], n[:, :HD // 2]], -1)
                    c, d = (S.f64(s.host[t][pos[b, j]]) for t in ("cos", "sin"))
                    page, slot = now.table[b, slots[b, j] // PAGE], slots[b, j] % PAGE
                    got = np.concatenate([S.f64(q[b, j]), S.f64(now.k[l, page, :, slot])])
                    ref, mag = n * c + half * d, np.abs(n * c) + np.abs(half * d)
                    assert (np.abs(got - ref) <= 2.0 ** -8 * np.abs(ref) + ((HD + 2) / 2 + 9) * 2.0 ** -24 * mag).all()
                    assert np.array_equal(S.f64(now.v[l, page, :, slot]), qkv[b, j, HEADS + KV:])
                    was.k[l, page, :, slot], was.v[l, page, :, slot] = now.k[l, page, :, slot], now.v[l, page, :, slot]
            assert np.array_equal(now.k[l], was.k[l]) and np.array_equal(now.v[l], was.v[l])
            # attention of the nodes over that
            ref, weight, reach = D.tree_attend(S.f64(q), S.f64(now.k[l]), S.f64(now.v[l]), now.table, now.lengths, s.counts,
                                               masks, HD ** -0.5)
            got = S.f64(s.get(f"attn{l}", np.uint16, (SLOTS, WIDTH, HEADS, HD)))
            keys = (now.lengths.astype(np.int64) + WIDTH).reshape(-1, 1, 1, 1)
            assert (np.abs(got - ref) <= bound(HD, keys, ref, weight, reach)).all()
            assert not got[np.arange(WIDTH) >= s.counts[:, None]].any()
        # distributions: exponents of 3 roundings, twice, two exponentials, a sum of VOCAB and a division
        z, t = S.f64(s.get("logits", np.uint16, (NODES, VOCAB))), s.host["temperatures"]
        pr = s.get("probs", np.float32, (NODES, VOCAB))
        ref = D.probs(z, t)
        e = np.where(t[:, None] > 0, (z.max(-1, keepdims=True) - z) / np.where(t > 0, t, 1)[:, None], 0) * 1.4427
        rel = 6 * 2.0 ** -24 * e + 2.0 ** -21 + (VOCAB + 2) * 2.0 ** -24
        assert (np.abs(pr - ref) <= rel * ref + 2.0 ** -126).all()
        # the accepted paths, and the cache behind them
        tokens, parents, uniforms = (s.get(n, d, (SLOTS, WIDTH)) for n, d in
                                     (("tokens", np.uint32), ("parents", np.uint32), ("uniforms", np.float32)))
        path, out, accepted = D.verify(pr.reshape(SLOTS, WIDTH, VOCAB), s.host["draft"], tokens, parents, s.counts, uniforms)
        assert np.array_equal(s.get("path", shape=(SLOTS, WIDTH)), path)
        assert np.array_equal(s.get("out", shape=(SLOTS, WIDTH)), out) and np.array_equal(s.get("accepted"), accepted)
        want = now.compact(path, accepted)
        s.compact()
        last = s.pages()
        assert np.array_equal(last.lengths, want) and np.array_equal(last.k, now.k) and np.array_equal(last.v, now.v)
        s.emitted()


def test_a_captured_step_replays_the_eager_ones(device):
    eager, replayed = Server(device), Server(device)
    replayed.trees(0)
    device.capture_begin()
    replayed.step()
    graph = device.capture_end()
    longest = 0
    for i in range(STEPS):
        for s in (eager, replayed):
            s.between(i)
            s.trees(20 + i)
        eager.step()
        graph.launch()
        if i % 2:
            device.synchronize()
        same(eager.snapshot(), replayed.snapshot(), i)
        longest = max(longest, eager.get("accepted").max())
        assert np.array_equal(eager.emitted(), replayed.emitted())
    assert longest > 1  # some drafted token was taken


def test_two_graphs_and_eager_calls_share_workspaces(device):
    servers = [Server(device) for _ in range(3)]
    for s in servers:
        for name in s.ws:
            s.st[name] = servers[0].st[name]
        s.trees(0)
    graphs = []
    for s in servers[:2]:
        device.capture_begin()
        s.step()
        graphs.append(device.capture_end())
    for i in range(4):
        for s in servers:
            s.between(i)
            s.trees(30 + i)
        for g in graphs:
            g.launch()
        servers[2].step()
        a, b, c = (s.snapshot() for s in servers)
        same(a, b, i), same(a, c, i)
        for s in servers:
            s.emitted()


def test_another_device_s_storage_is_refused_and_its_own_stream_serves(device):
    other = HipDevice(0)
    s, t = Server(other), Server(device)
    for a in (s, t):
        a.trees(40)
        a.step()
    same(s.snapshot(), t.snapshot(), "its own stream")
    s.dev, s_dev = device, s.dev
    for call in (lambda: s.append(0, NODES, s.p("node_seqs"), s.p("positions"), s.p("slots")), s.compact,
                 lambda: s.reserve(s.p("counts")), lambda: s.step()):
        with pytest.raises(_lib.HipError) as e:
            call()
        assert e.value.status == _lib.ERR_FOREIGN_STORAGE
    s.dev = s_dev
    del s, a
    other.close()

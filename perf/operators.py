"""The operators of a serving step over many requests, as cases that can be
timed and checked: the rotated append of new keys and values to a paged cache,
one new token's attention over that cache, low-rank adapters beside a shared
projection, and penalties, biases and grammar masks on the logits.

`prepare` makes what a user's program holds before the call, `run` makes one
pass: with `own` through the library's entry points, else in plain torch (32
bits inside, each output rounded once). `exact` restates the result in 64 bits.

With `own` the work is queued on the library's stream, which torch's streams do
not wait for: synchronise the device before a result is read. Results are the
state's own buffers, which its next pass writes again.

Shapes are those of the decoders the library is configured for (8 KV heads of
128 or of 64) and generic ones.
"""
import ctypes
import math

import torch

own = False

# query heads, KV heads, head size
HEADS = {
    "h24": (24, 8, 128),
    "h32": (32, 8, 128),
    "h32s": (32, 8, 64),
    "mha": (12, 12, 64),
    "mqa": (8, 1, 256),
}
VOCAB = 128256
NONE = -1  # as u32: no sequence position, no page, no adapter


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one chat early in its context: the smallest decode call, latency counts
        {"name": "attn_short_1", "kind": "attn", "heads": "h24", "batch": 1, "lo": 300, "hi": 300, "page": 16,
         "spare": 13, "idle": 0},
        # 8 sequences a few thousand tokens deep: ordinary decode
        {"name": "attn_batch_8", "kind": "attn", "heads": "h32", "batch": 8, "lo": 1900, "hi": 4111, "page": 16,
         "spare": 4, "idle": 0},
        # a full server: 96 slots, five of them idle, contexts from a greeting to a document
        {"name": "attn_ragged_96", "kind": "attn", "heads": "h32", "batch": 96, "lo": 17, "hi": 16384, "page": 32,
         "spare": 0, "idle": 5},
        # one request over a very long context
        {"name": "attn_long_1", "kind": "attn", "heads": "h32", "batch": 1, "lo": 131077, "hi": 131077, "page": 64,
         "spare": 2, "idle": 0},
        # the new token of each of 61 sequences
        {"name": "append_decode_61", "kind": "append", "heads": "h32", "seqs": 61, "tokens": 61, "past": 2900,
         "page": 16, "idle": 3},
        # a packed batch of five prompts' chunks
        {"name": "append_prompt_8192", "kind": "append", "heads": "h32", "seqs": 5, "tokens": 8192, "past": 700,
         "page": 32, "idle": 0},
        # decode of 8 requests, each with its own adapter, at the fused q/k/v projection
        {"name": "lora_rows_8", "kind": "lora", "rows": 8, "k": 4096, "n": 6144, "rank": 16, "adapters": 8, "bare": 0,
         "packed": False, "f32": False},
        # decode of 200 requests that share 48 adapters, some with none, on the fp32 gate/up sums
        {"name": "lora_rows_200", "kind": "lora", "rows": 200, "k": 4096, "n": 28672, "rank": 16, "adapters": 48,
         "bare": 9, "packed": False, "f32": True},
        # a packed prompt batch of five requests, each with its adapter, at the output projection
        {"name": "lora_prompt_4096", "kind": "lora", "rows": 4096, "k": 4096, "n": 4096, "rank": 32, "adapters": 5,
         "bare": 1, "packed": True, "f32": False},
        # one chat's next token: penalties over what it has said
        {"name": "logits_1", "kind": "logits", "rows": 1, "n": VOCAB, "history": 700, "prompt": 400, "bias": 0,
         "mask": False, "f32": False},
        # 64 requests with every rule: long histories, biases, a grammar's mask
        {"name": "logits_64", "kind": "logits", "rows": 64, "n": VOCAB, "history": 8192, "prompt": 3000, "bias": 300,
         "mask": True, "f32": False},
        # fp32 logits of a small odd vocabulary under a grammar
        {"name": "logits_33_odd", "kind": "logits", "rows": 33, "n": 32003, "history": 60, "prompt": 0, "bias": 7,
         "mask": True, "f32": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "append", "lora", "lora", "logits"])
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 48, 64, 128])
    if kind == "attn":
        batch = _log(rng, 1, 128)
        hi = _log(rng, 1, min(131072, 217000 // batch))
        lo = _log(rng, 1, hi)
        return {"kind": kind, "heads": heads, "batch": batch, "lo": lo, "hi": hi, "page": page,
                "spare": rng.randrange(0, 9), "idle": rng.randrange(0, batch) if rng.random() < 0.3 else 0}
    if kind == "append":
        tokens = _log(rng, 1, 8192)
        seqs = _log(rng, 1, min(tokens, 128))
        return {"kind": kind, "heads": heads, "seqs": seqs, "tokens": tokens, "past": rng.randrange(0, 3000),
                "page": page, "idle": rng.randrange(0, 1 + tokens // 8)}
    if kind == "lora":
        rows, rank = _log(rng, 1, 4096), rng.choice([8, 16, 24, 32, 64, 128])
        k, n = rng.choice([(2048, 2048), (2048, 16384), (4096, 6144), (4096, 4096), (14336, 4096),
                           (8 * _log(rng, 16, 1024), _log(rng, 100, 8192))])
        rows = max(1, min(rows, 4096 * 8192 // (k + n)))
        return {"kind": kind, "rows": rows, "k": k, "n": n, "rank": rank,
                "adapters": _log(rng, 1, max(1, min(rows, 2048 // rank))), "bare": rng.choice([0, rng.randrange(1, 12)]),
                "packed": rows > 256 or rng.random() < 0.3, "f32": rng.random() < 0.4}
    history = _log(rng, 1, 8192)
    return {"kind": "logits", "rows": _log(rng, 1, 64), "n": rng.choice([VOCAB, _log(rng, 300, VOCAB)]),
            "history": history, "prompt": rng.randrange(0, history), "bias": rng.choice([0, _log(rng, 1, 300)]),
            "mask": rng.random() < 0.5, "f32": rng.random() < 0.4}


# -------------------------------------------------- sizes that a case fixes

def _spread(lo, hi, count):
    """`count` whole numbers from lo to hi, even over their logarithm, in a scattered order."""
    return [round(lo * (hi / lo) ** ((i * 0.6180339887498949 + 1.0) % 1.0 if i else 1.0)) for i in range(count)]


def _idle(count, idle):
    """Which of `count` slots are idle: `idle` of them, evenly placed."""
    return {(2 * j + 1) * count // (2 * idle) for j in range(idle)} if idle else set()


def _contexts(c):
    """Keys of each sequence of an attention case; 0 for an idle slot."""
    off = _idle(c["batch"], c["idle"])
    return [0 if i in off else n for i, n in enumerate(_spread(c["lo"], c["hi"], c["batch"]))]


def _segments(total, parts):
    """`total` cut into `parts` pieces of unlike sizes, none empty."""
    cuts = [total * (i * i + i) // (parts * parts + parts) for i in range(parts + 1)]
    cuts = [max(v, i) for i, v in enumerate(cuts)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _appended(c):
    """(sequence, position) of each token of an append case, sequence by sequence."""
    past = [c["past"] * (i + 1) // c["seqs"] for i in range(c["seqs"])]
    return [(s, past[s] + j) for s, n in enumerate(_segments(c["tokens"], c["seqs"])) for j in range(n)]


# ------------------------------------------------------------------ prepare

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, *shape):
    return torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(torch.bfloat16)


def _ints(values):
    return torch.tensor(values, device="cuda", dtype=torch.int64).to(torch.int32)


def _pages(g, counts, width):
    """A page table [sequences, width] over a shuffled pool with a few pages to
    spare; entries behind a sequence's last page name no page."""
    pool = sum(counts) + 3
    ids = torch.randperm(pool, generator=g, device="cuda")
    count = torch.tensor(counts, device="cuda")
    start = count.cumsum(0) - count
    at = torch.arange(width, device="cuda")
    table = ids[(start.unsqueeze(1) + at).clamp(max=pool - 1)]
    return torch.where(at < count.unsqueeze(1), table, NONE).to(torch.int32), pool


def _rotation(length, hd):
    """cos and sin [length, hd] in bf16, theta 500000, the angles in 64 bits."""
    f = 500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(length, device="cuda", dtype=torch.float64).unsqueeze(1) * torch.cat([f, f])
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _prepare_attn(c, g):
    heads, kv, hd = HEADS[c["heads"]]
    keys = _contexts(c)
    counts = [-(-n // c["page"]) for n in keys]
    table, pool = _pages(g, counts, max(counts) + c["spare"])
    # heads differ in how sharply they attend
    sharp = torch.linspace(0.5, 3.0, heads, device="cuda").unsqueeze(1)
    q = (torch.randn((c["batch"], heads, hd), generator=g, device="cuda") * sharp).to(torch.bfloat16)
    return {"q": q, "k": _normal(g, pool, kv, c["page"] * hd), "v": _normal(g, pool, kv, c["page"], hd),
            "table": table, "pos": _ints([n - 1 for n in keys])}


def _prepare_append(c, g):
    heads, kv, hd = HEADS[c["heads"]]
    seq, pos = zip(*_appended(c))
    last = [i for i in range(c["tokens"]) if i + 1 == c["tokens"] or seq[i + 1] != seq[i]]
    # pages of the earlier tokens that no new token touches stay out of the pool: their entries name page 0
    counts = [pos[i] // c["page"] + 1 for i in last]
    firsts = [pos[i] // c["page"] for i in range(c["tokens"]) if i == 0 or seq[i - 1] != seq[i]]
    new = [n - f for n, f in zip(counts, firsts)]
    live, pool = _pages(g, new, max(new))
    at = torch.arange(max(counts) + 2, device="cuda") - torch.tensor(firsts, device="cuda").unsqueeze(1)
    table = live.gather(1, at.clamp(0, live.shape[1] - 1))
    table = torch.where(at < 0, 0, torch.where(at < live.shape[1], table, NONE)).to(torch.int32)
    off = _idle(c["tokens"], c["idle"])
    cos, sin = _rotation(max(pos) + 1, hd)
    return {"qkv": _normal(g, c["tokens"], (heads + 2 * kv) * hd), "cos": cos, "sin": sin, "seq": _ints(seq),
            "pos": _ints([NONE if i in off else p for i, p in enumerate(pos)]), "table": table,
            "k": _normal(g, pool, kv, c["page"] * hd), "v": _normal(g, pool, kv, c["page"], hd),
            "q": torch.zeros(c["tokens"], heads, hd, device="cuda", dtype=torch.bfloat16)}


def _prepare_lora(c, g):
    m, k, n, r, u = c["rows"], c["k"], c["n"], c["rank"], c["adapters"]
    if c["packed"]:  # a segment of rows per request
        segments = torch.tensor(_segments(m, u), device="cuda")
        ids = torch.repeat_interleave(torch.randperm(u, generator=g, device="cuda"), segments)
    else:
        ids = torch.cat([torch.arange(u, device="cuda"), torch.randint(0, u, (m - u,), generator=g, device="cuda")])
        ids = ids[torch.randperm(m, generator=g, device="cuda")]
    bare = torch.tensor(sorted(_idle(m, min(c["bare"], m // 2))), device="cuda", dtype=torch.int64)
    ids[bare] = NONE
    base = torch.randn((m, n), generator=g, device="cuda")
    return {"x": _normal(g, m, k), "a": (torch.randn((u, r, k), generator=g, device="cuda") * k ** -0.5).bfloat16(),
            "b": (torch.randn((u, n, r), generator=g, device="cuda") * 0.2).bfloat16(),
            "scale": 0.5 + 1.5 * torch.rand(u, generator=g, device="cuda"), "ids": ids.to(torch.int32),
            "base": base if c["f32"] else base.bfloat16()}


def _prepare_logits(c, g):
    rows, n, h = c["rows"], c["n"], c["history"]
    z = 2.5 * torch.randn((rows, n), generator=g, device="cuda")
    # what was said repeats itself: ids cluster near the low end, as frequent tokens' ids do
    u = torch.rand((rows, h), generator=g, device="cuda", dtype=torch.float64)
    said = (n * u ** 4).long().clamp(max=n - 1)
    t = {"z": z if c["f32"] else z.bfloat16(), "said": said.to(torch.int32), "len": _ints(_spread(1, h, rows)),
         "prompt": _ints([min(c["prompt"], n_) for n_ in _spread(1, h, rows)]),
         "rep": 1.0 + 0.5 * torch.rand(rows, generator=g, device="cuda"),
         "freq": 0.6 * torch.rand(rows, generator=g, device="cuda"),
         "pres": 0.8 * torch.rand(rows, generator=g, device="cuda")}
    if c["bias"]:
        count = min(c["bias"], n)
        t["bias_id"] = torch.rand((rows, n), generator=g, device="cuda").topk(count, 1).indices.to(torch.int32)
        t["bias"] = 4.0 * torch.randn((rows, count), generator=g, device="cuda")
        t["bias_len"] = _ints([count - i % (count // 2 + 1) for i in range(rows)])
    if c["mask"]:
        # one word in two allows nothing but a bit, as a grammar's state does
        w = torch.randint(0, 2 ** 32, (rows, -(-n // 32)), generator=g, device="cuda", dtype=torch.int64)
        bit = 1 << torch.randint(0, 32, w.shape, generator=g, device="cuda", dtype=torch.int64)
        few = torch.rand(w.shape, generator=g, device="cuda") < 0.5
        w = torch.where(few, w & bit, w)
        t["mask"] = torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)
    return t


_PREPARE = {"attn": _prepare_attn, "append": _prepare_append, "lora": _prepare_lora, "logits": _prepare_logits}


def prepare(case, seed):
    state = {"case": dict(case), "t": _PREPARE[case["kind"]](case, _gen(seed))}
    if own:  # the library's operators work on memory of its device alone
        _bind(state)
    return state


# -------------------------------------------------------- the library's calls

_device = None


class _Span:
    """A storage's memory as torch sees it; keeps the storage alive."""

    def __init__(self, storage, nbytes):
        self.storage = storage
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1", "data": (storage.ptr, False),
                                         "version": 2}


def _storage(shape, dtype):
    """Memory of the library's device as a torch tensor."""
    global _device
    if _device is None:
        from foundry_amd.device import HipDevice
        _device = HipDevice(0)
    nbytes = math.prod(shape) * torch.empty((), dtype=dtype).element_size()
    span = _Span(_device.empty(max(nbytes, 16)), nbytes)
    return torch.as_tensor(span, device="cuda").view(dtype).view(shape)


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None else None


def _bind(state):
    """Moves the inputs to the library's memory, adds what a program keeps
    between calls (outputs, workspaces) and the arguments of its calls."""
    c, t = state["case"], state["t"]
    for name, x in t.items():
        held = _storage(tuple(x.shape), x.dtype)
        held.copy_(x)
        t[name] = held
    torch.cuda.synchronize()
    state["args"] = _BIND[c["kind"]](c, t)


def _bind_attn(c, t):
    from foundry_amd import _lib
    heads, kv, hd = HEADS[c["heads"]]
    t["out"] = _storage((c["batch"], heads, hd), torch.bfloat16)
    pool, width = t["k"].shape[0], t["table"].shape[1]
    nbytes = _lib.paged_attention_workspace_bytes(c["batch"], heads, kv, hd, c["page"], width)
    t["ws"] = _storage((nbytes,), torch.uint8)
    return ("fh_paged_attention", _device.handle, _ptr(t["q"]), c["batch"], heads, kv, hd, _ptr(t["k"]), _ptr(t["v"]),
            pool, c["page"], _ptr(t["table"]), width, _ptr(t["pos"]), ctypes.c_float(hd ** -0.5), _ptr(t["ws"]),
            nbytes, _ptr(t["out"]))


def _bind_append(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    seqs, width = t["table"].shape
    return ("fh_paged_rope_kv", _device.handle, _ptr(t["qkv"]), c["tokens"], heads, kv, hd, _ptr(t["cos"]),
            _ptr(t["sin"]), t["cos"].shape[0], _ptr(t["seq"]), _ptr(t["pos"]), _ptr(t["table"]), seqs, width,
            _ptr(t["k"]), _ptr(t["v"]), t["k"].shape[0], c["page"], _ptr(t["q"]))


def _bind_lora(c, t):
    from foundry_amd import _lib
    m, k, n, r, u = c["rows"], c["k"], c["n"], c["rank"], c["adapters"]
    t["y"] = _storage((m, n), t["base"].dtype)
    nbytes = _lib.lora_workspace_bytes(m, k, r)
    t["ws"] = _storage((nbytes,), torch.uint8)
    return ("fh_lora_add", _device.handle, _ptr(t["x"]), m, k, k, _ptr(t["a"]), _ptr(t["b"]), _ptr(t["scale"]), u, r, n,
            _ptr(t["ids"]), _ptr(t["base"]), n, _ptr(t["y"]), n, _lib.F32 if c["f32"] else _lib.BF16, _ptr(t["ws"]),
            nbytes)


def _bind_logits(c, t):
    from foundry_amd import _lib
    t["out"] = _storage((c["rows"], c["n"]), t["z"].dtype)
    t["rules"] = rules = _lib.LogitRules(
        history=_ptr(t["said"]), history_ld=c["history"], history_len=_ptr(t["len"]), prompt_len=_ptr(t["prompt"]),
        repetition=_ptr(t["rep"]), frequency=_ptr(t["freq"]), presence=_ptr(t["pres"]), bias_ids=_ptr(t.get("bias_id")),
        bias_values=_ptr(t.get("bias")), bias_ld=t["bias"].shape[1] if c["bias"] else 0,
        bias_len=_ptr(t.get("bias_len")), mask=_ptr(t.get("mask")))
    return ("fh_logits_process", _device.handle, _ptr(t["z"]), _lib.F32 if c["f32"] else _lib.BF16, c["rows"], c["n"],
            ctypes.byref(rules), _ptr(t["out"]))


_BIND = {"attn": _bind_attn, "append": _bind_append, "lora": _bind_lora, "logits": _bind_logits}
_RESULT = {"attn": "out", "lora": "y", "logits": "out"}


# ---------------------------------------------------------------------- run

def run(state):
    c, t = state["case"], state["t"]
    if own:
        from foundry_amd import _lib
        _lib.call(*state["args"])
        return t[_RESULT[c["kind"]]] if c["kind"] != "append" else {"q": t["q"], "k": t["k"], "v": t["v"]}
    return _PLAIN[c["kind"]](c, t)


def _key_offset(slot, page, hd):
    """Where key `slot` of a page's region holds its dims [..., hd]: groups of
    16 keys, each laid out [hd / 32][16][32]."""
    d = torch.arange(hd, device="cuda")
    return (slot // 16 * 16 * hd + slot % 16 * 32).unsqueeze(-1) + d // 32 * 512 + d % 32


def _plain_attn(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    batch, width = t["table"].shape
    ids = t["table"].clamp(min=0).long()
    at = _key_offset(torch.arange(c["page"], device="cuda"), c["page"], hd)
    k = t["k"][:, :, at.flatten()].view(t["v"].shape)[ids].float()  # [batch, pages, kv, page, hd]
    v = t["v"][ids].float()
    k = k.permute(0, 2, 4, 1, 3).reshape(batch, kv, hd, width * c["page"])
    v = v.permute(0, 2, 1, 3, 4).reshape(batch, kv, width * c["page"], hd)
    s = t["q"].float().view(batch, kv, heads // kv, hd) @ k * hd ** -0.5
    seen = (torch.arange(width * c["page"], device="cuda") <= t["pos"].unsqueeze(1)).view(batch, 1, 1, -1)
    top = s.masked_fill(~seen, -math.inf).amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = torch.where(seen, (s - top).exp(), 0.0)
    out = e @ v / e.sum(-1, keepdim=True)
    return torch.where(seen.any(-1, keepdim=True), out, 0.0).view(batch, heads, hd).bfloat16()


def _plain_append(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    live = t["pos"] >= 0
    pos, seq = t["pos"].clamp(min=0).long(), t["seq"].long()
    x = t["qkv"].float().view(c["tokens"], heads + 2 * kv, hd)
    cos, sin = t["cos"][pos].float().unsqueeze(1), t["sin"][pos].float().unsqueeze(1)
    half = torch.cat([-x[:, :heads + kv, hd // 2:], x[:, :heads + kv, :hd // 2]], -1)
    rot = (x[:, :heads + kv] * cos + half * sin).bfloat16()
    page = t["table"][seq, pos // c["page"]].long()
    page, slot, rot, value = page[live], (pos % c["page"])[live], rot[live], t["qkv"].view(x.shape)[live, heads + kv:]
    t["q"][live] = rot[:, :heads]
    row = torch.arange(kv, device="cuda")
    at = _key_offset(slot, c["page"], hd).unsqueeze(1)
    t["k"][page.view(-1, 1, 1), row.view(1, -1, 1), at] = rot[:, heads:]
    t["v"][page.view(-1, 1), row, slot.view(-1, 1)] = value
    return {"q": t["q"], "k": t["k"], "v": t["v"]}


def _plain_lora(c, t):
    m, n, r, u = c["rows"], c["n"], c["rank"], c["adapters"]
    # every row through every adapter, and its own kept
    mine = torch.arange(u, device="cuda") == t["ids"].unsqueeze(1)
    down = (t["x"].float() @ t["a"].float().view(u * r, -1).T).view(m, u, r) * t["scale"].unsqueeze(1)
    down = torch.where(mine.unsqueeze(-1), down, 0.0).view(m, u * r)
    up = t["b"].float().permute(0, 2, 1).reshape(u * r, n)
    return (t["base"].float() + down @ up).to(t["base"].dtype)


def _plain_logits(c, t):
    rows, n, h = c["rows"], c["n"], c["history"]
    at = torch.arange(h, device="cuda")
    used, new = at < t["len"].unsqueeze(1), at >= t["prompt"].unsqueeze(1)
    said = t["said"].long()
    seen = torch.zeros((rows, n), device="cuda", dtype=torch.int32).scatter_add_(1, said, used.int()) > 0
    count = torch.zeros((rows, n), device="cuda", dtype=torch.int32).scatter_add_(1, said, (used & new).int())
    z = t["z"].float()
    rep = t["rep"].unsqueeze(1)
    z = torch.where(seen, torch.where(z > 0, z / rep, z * rep), z)
    z = z - t["freq"].unsqueeze(1) * count - t["pres"].unsqueeze(1) * (count > 0)
    if c["bias"]:
        k = t["bias"].shape[1]
        use = torch.arange(k, device="cuda") < t["bias_len"].unsqueeze(1)
        z = z.scatter_add(1, t["bias_id"].long(), torch.where(use, t["bias"], 0.0))
    if c["mask"]:
        j = torch.arange(n, device="cuda")
        z = z.masked_fill((t["mask"][:, j // 32] >> (j % 32).int()) & 1 == 0, -math.inf)
    return z.to(t["z"].dtype)


_PLAIN = {"attn": _plain_attn, "append": _plain_append, "lora": _plain_lora, "logits": _plain_logits}


# --------------------------------------------------------------------- work

def work(case):
    c = case
    if c["kind"] in ("attn", "append"):
        heads, kv, hd = HEADS[c["heads"]]
    if c["kind"] == "attn":
        keys = _contexts(c)
        nbytes = 4 * sum(keys) * kv * hd + 4 * c["batch"] * heads * hd
        nbytes += 4 * sum(-(-n // c["page"]) for n in keys) + 4 * c["batch"]
        return {"bytes": nbytes, "flops": 4 * sum(keys) * heads * hd}
    if c["kind"] == "append":
        live = c["tokens"] - len(_idle(c["tokens"], c["idle"]))
        places = len({p for _, p in _appended(c)})  # rows of the two tables
        nbytes = 4 * live * (heads + 2 * kv) * hd + 4 * places * hd + 12 * c["tokens"]
        return {"bytes": nbytes, "flops": 3 * live * (heads + kv) * hd}
    if c["kind"] == "lora":
        m, k, n, r = c["rows"], c["k"], c["n"], c["rank"]
        live = m - len(_idle(m, min(c["bare"], m // 2)))
        used = min(c["adapters"], live)
        nbytes = 2 * live * k + 2 * used * r * (k + n) + 2 * m * n * (4 if c["f32"] else 2) + 8 * m
        return {"bytes": nbytes, "flops": 2 * live * r * (k + n)}
    rows, n = c["rows"], c["n"]
    nbytes = 2 * rows * n * (4 if c["f32"] else 2) + 4 * sum(_spread(1, c["history"], rows)) + 20 * rows
    nbytes += 8 * rows * min(c["bias"], n) + (rows * (-(-n // 32)) * 4 if c["mask"] else 0)
    return {"bytes": nbytes, "flops": 6 * rows * n}


# -------------------------------------------------------------------- exact

def exact(case, seed):
    t = _PREPARE[case["kind"]](case, _gen(seed))
    return _EXACT[case["kind"]](case, t)


def _exact_attn(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    out = torch.zeros(c["batch"], heads, hd, device="cuda", dtype=torch.float64)
    for b in range(c["batch"]):
        n = int(t["pos"][b]) + 1
        if n == 0:
            continue
        pages = t["table"][b, :-(-n // c["page"])].long()
        groups = t["k"][pages].view(len(pages), kv, c["page"] // 16, hd // 32, 16, 32)
        k = groups.permute(1, 0, 2, 4, 3, 5).reshape(kv, -1, hd)[:, :n]
        v = t["v"][pages].transpose(0, 1).reshape(kv, -1, hd)[:, :n]
        for h in range(heads):
            s = k[h * kv // heads].double() @ t["q"][b, h].double() / math.sqrt(hd)
            out[b, h] = torch.softmax(s, 0) @ v[h * kv // heads].double()
    return out


def _exact_append(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    pool = t["k"].shape[0]
    q = t["q"].double()
    k = t["k"].double().view(pool, kv, c["page"] // 16, hd // 32, 16, 32)
    v = t["v"].double()
    live = t["pos"] >= 0
    pos, seq = t["pos"][live].long(), t["seq"][live].long()
    x = t["qkv"][live].double().view(len(pos), heads + 2 * kv, hd)
    # the rotation as a product of complex numbers, dims d and d + hd / 2 together
    a, b = x[:, :heads + kv].chunk(2, -1)
    (ca, cb), (sa, sb) = [w[pos].double().unsqueeze(1).chunk(2, -1) for w in (t["cos"], t["sin"])]
    rot = torch.cat([a * ca - b * sa, b * cb + a * sb], -1)
    q[live] = rot[:, :heads]
    page, slot = t["table"][seq, pos // c["page"]].long(), pos % c["page"]
    k[page, :, slot // 16, :, slot % 16] = rot[:, heads:].view(len(pos), kv, hd // 32, 32)
    v[page, :, slot] = x[:, heads + kv:]
    return {"q": q, "k": k.view(t["k"].shape), "v": v}


def _exact_lora(c, t):
    y = t["base"].double()
    for u in range(c["adapters"]):
        rows = (t["ids"] == u).nonzero().flatten()
        down = t["x"][rows].double() @ t["a"][u].double().T
        y[rows] += t["scale"][u].double() * (down @ t["b"][u].double().T)
    return y


def _exact_logits(c, t):
    out = t["z"].double()
    for r in range(c["rows"]):
        z, said = out[r], t["said"][r, :int(t["len"][r])].long()
        ids = said.unique()
        rep = t["rep"][r].double()
        z[ids] = torch.where(z[ids] > 0, z[ids] / rep, z[ids] * rep)
        ids, times = said[int(t["prompt"][r]):].unique(return_counts=True)
        z[ids] -= t["freq"][r].double() * times + t["pres"][r].double()
        if c["bias"]:
            n = int(t["bias_len"][r])
            z[t["bias_id"][r, :n].long()] += t["bias"][r, :n].double()
        if c["mask"]:
            words = t["mask"][r].long() & 0xFFFFFFFF
            allowed = (words.unsqueeze(1) >> torch.arange(32, device="cuda")) & 1
            z[allowed.flatten()[:c["n"]] == 0] = -math.inf
    return out


_EXACT = {"attn": _exact_attn, "append": _exact_append, "lora": _exact_lora, "logits": _exact_logits}

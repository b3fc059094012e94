"""The operators of a serving step that drafts several tokens ahead, as cases
that can be timed and checked: normed and rotated q and k appended to places of
their own in a paged cache, attention of a tree of drafted tokens over that
cache, probabilities of logits, the verification of the drafted tokens, and the
cache's pages: the accepted tokens moved together, sequences forked and freed.

`prepare` makes what a user's program holds before the call, `run` makes one
pass: with `own` through the library's entry points, else in plain torch (32
bits inside, 64 for the sums that decide on a token; each output rounded once).
`exact` restates the result in 64 bits.

With `own` the work is queued on the library's stream, which torch's streams do
not wait for: synchronise the device before a result is read. Results are the
state's own buffers, which its next pass writes again.
"""
import ctypes
import math

import torch

own = False

# query heads, KV heads, head size
HEADS = {
    "h32": (32, 8, 128),
    "h32s": (32, 8, 64),
    "h20": (20, 4, 128),
    "mha": (12, 12, 64),
    "mqa": (8, 1, 256),
}
VOCAB = 128256
EPS = 1e-5
NONE = -1  # as u32: no position, no page, no token


# ---------------------------------------------------------------- the cases

def listed():
    return [
        # one chat with five drafted tokens in a row: the smallest attention call, latency counts
        {"name": "tree_chain_1", "kind": "tree", "heads": "h32", "batch": 1, "nodes": 6, "masked": False, "lo": 700,
         "hi": 700, "page": 16, "spare": 9, "idle": 0},
        # eight requests a few thousand tokens deep, a full tree for each
        {"name": "tree_batch_8", "kind": "tree", "heads": "h32", "batch": 8, "nodes": 64, "masked": True, "lo": 1900,
         "hi": 4111, "page": 16, "spare": 4, "idle": 0},
        # a busy server: 64 slots, three idle, small trees, contexts from a greeting to a document
        {"name": "tree_ragged_64", "kind": "tree", "heads": "h20", "batch": 64, "nodes": 12, "masked": True, "lo": 17,
         "hi": 16384, "page": 32, "spare": 0, "idle": 3},
        # one request over a very long context
        {"name": "tree_long_1", "kind": "tree", "heads": "h32", "batch": 1, "nodes": 32, "masked": True, "lo": 131077,
         "hi": 131077, "page": 64, "spare": 2, "idle": 0},
        # the trees' nodes of eight requests, q and k normed
        {"name": "append_nodes_8", "kind": "append", "heads": "h32", "seqs": 8, "tokens": 512, "past": 2900, "page": 16,
         "idle": 5, "tree": True, "norm": True},
        # a packed batch of five prompts' chunks
        {"name": "append_prompt_8192", "kind": "append", "heads": "h32", "seqs": 5, "tokens": 8192, "past": 700,
         "page": 32, "idle": 0, "tree": False, "norm": True},
        # one chat's next distribution
        {"name": "probs_1", "kind": "probs", "rows": 1, "n": VOCAB, "masked": False, "f32": False},
        # the distributions behind every node of eight trees, a grammar's mask on them
        {"name": "probs_512", "kind": "probs", "rows": 512, "n": VOCAB, "masked": True, "f32": False},
        # one chat's five drafted tokens against the target's and the draft's distributions
        {"name": "verify_chain_1", "kind": "verify", "batch": 1, "nodes": 6, "n": VOCAB, "drafts": True, "tree": False},
        # 64 requests' chains
        {"name": "verify_chain_64", "kind": "verify", "batch": 64, "nodes": 6, "n": VOCAB, "drafts": True,
         "tree": False},
        # the accepted nodes of 24 requests moved together in a deep model's caches
        {"name": "pages_compact_24", "kind": "compact", "heads": "h32", "layers": 28, "batch": 24, "nodes": 64,
         "most": 9, "lo": 300, "hi": 4000, "page": 16},
        # four prompts sampled from 4 times each: the old samples freed, the prompts forked, room for the next tokens
        {"name": "pages_fork_16", "kind": "fork", "heads": "h32", "layers": 28, "parents": 4, "forks": 16, "lo": 200,
         "hi": 900, "page": 64, "extra": 40},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    kind = rng.choice(["tree", "tree", "tree", "append", "probs", "verify", "verify", "compact", "fork"])
    heads = rng.choice(sorted(HEADS))
    page = rng.choice([16, 32, 48, 64, 128])
    if kind == "tree":
        batch = _log(rng, 1, 96)
        nodes = _log(rng, 1, min(256, max(1, 1024 // batch)))
        hi = _log(rng, 1, min(131072, 160000 // batch, 4194304 // (batch * nodes)))
        return {"kind": kind, "heads": heads, "batch": batch, "nodes": nodes, "masked": rng.random() < 0.7,
                "lo": _log(rng, 1, hi), "hi": hi, "page": page, "spare": rng.randrange(0, 9),
                "idle": rng.randrange(0, batch) if rng.random() < 0.3 else 0}
    if kind == "append":
        tokens = _log(rng, 1, 8192)
        return {"kind": kind, "heads": heads, "seqs": _log(rng, 1, min(tokens, 128)), "tokens": tokens,
                "past": rng.randrange(0, 3000), "page": page, "idle": rng.randrange(0, 1 + tokens // 8),
                "tree": rng.random() < 0.6, "norm": rng.random() < 0.7}
    if kind == "probs":
        f32 = rng.random() < 0.3
        return {"kind": kind, "rows": _log(rng, 1, 384 if f32 else 512),
                "n": rng.choice([VOCAB, _log(rng, 300, VOCAB)]), "masked": rng.random() < 0.5, "f32": f32}
    if kind == "verify":
        batch, drafts = _log(rng, 1, 64), rng.random() < 0.5
        nodes = _log(rng, 1, max(1, min(64, 384 // batch)))
        return {"kind": kind, "batch": batch, "nodes": nodes, "n": rng.choice([VOCAB, _log(rng, 300, VOCAB)]),
                "drafts": drafts, "tree": rng.random() < (0.4 if drafts else 0.8)}
    if kind == "compact":
        nodes = _log(rng, 4, 128)
        return {"kind": kind, "heads": heads, "layers": rng.randrange(1, 29), "batch": _log(rng, 2, 24), "nodes": nodes,
                "most": _log(rng, 2, min(9, nodes // 2)), "lo": 1, "hi": _log(rng, 1, 8000), "page": page}
    parents = _log(rng, 1, 4)
    hi = _log(rng, 1, 900)
    return {"kind": kind, "heads": heads, "layers": rng.randrange(1, 29), "parents": parents,
            "forks": parents * rng.randrange(1, 5), "lo": _log(rng, 1, hi), "hi": hi, "page": page,
            "extra": rng.randrange(0, 100)}


# -------------------------------------------------- sizes that a case fixes

def _spread(lo, hi, count):
    """`count` whole numbers from lo to hi, even over their logarithm, in a scattered order."""
    return [round(lo * (hi / lo) ** ((i * 0.6180339887498949 + 1.0) % 1.0 if i else 1.0)) for i in range(count)]


def _idle(count, idle):
    """Which of `count` slots are idle: `idle` of them, evenly placed."""
    return {(2 * j + 1) * count // (2 * idle) for j in range(idle)} if idle else set()


def _trees(c):
    """Keys before each sequence's tree and the tree's nodes; (0, 0) for an idle slot."""
    off = _idle(c["batch"], c["idle"])
    sizes = [max(1, c["nodes"] - (i * 5) % (c["nodes"] // 3 + 1)) for i in range(c["batch"])]
    return [(0, 0) if i in off else (n, t) for i, (n, t) in enumerate(zip(_spread(c["lo"], c["hi"], c["batch"]), sizes))]


def _segments(total, parts):
    """`total` cut into `parts` pieces of unlike sizes, none empty."""
    cuts = [total * (i * i + i) // (parts * parts + parts) for i in range(parts + 1)]
    cuts = [max(v, i) for i, v in enumerate(cuts)]
    return [b - a for a, b in zip(cuts, cuts[1:])]


def _depths(n):
    """The depth of each of a tree's n nodes, level by level, levels of 1, 2, 4, 8, 8, .. nodes."""
    sizes = [1 << min(d, 3) for d in range(n)]
    return [d for d, s in enumerate(sizes) for _ in range(s)][:n]


def _appended(c):
    """(sequence, position, slot) of each token of an append case, sequence by sequence."""
    past = [c["past"] * (i + 1) // c["seqs"] for i in range(c["seqs"])]
    at = [list(enumerate(_depths(n) if c["tree"] else range(n))) for n in _segments(c["tokens"], c["seqs"])]
    return [(s, past[s] + d, past[s] + j) for s, row in enumerate(at) for j, d in row]


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


def _late_pages(g, firsts, counts, spare):
    """A table whose entries before each sequence's first one in use name page 0
    (pages that a case does not touch stay out of its pool)."""
    live, pool = _pages(g, [n - f for n, f in zip(counts, firsts)], max(n - f for n, f in zip(counts, firsts)))
    at = torch.arange(max(counts) + spare, device="cuda") - torch.tensor(firsts, device="cuda").unsqueeze(1)
    table = live.gather(1, at.clamp(0, live.shape[1] - 1))
    return torch.where(at < 0, 0, torch.where(at < live.shape[1], table, NONE)).to(torch.int32), pool


def _rotation(length, hd):
    """cos and sin [length, hd] in bf16, theta 500000, the angles in 64 bits."""
    f = 500000.0 ** (-torch.arange(0, hd, 2, device="cuda", dtype=torch.float64) / hd)
    angle = torch.arange(length, device="cuda", dtype=torch.float64).unsqueeze(1) * torch.cat([f, f])
    return angle.cos().to(torch.bfloat16), angle.sin().to(torch.bfloat16)


def _parents(g, batch, nodes):
    """A random tree for each sequence: every node's parent comes before it (the root's is no node)."""
    at = torch.arange(nodes, device="cuda")
    # late nodes more often, so that branches get long
    u = torch.rand((batch, nodes), generator=g, device="cuda").sqrt()
    return torch.where(at > 0, (u * at).long().clamp(max=nodes - 1), NONE)


def _ancestors(parents):
    """seen[b, i, j]: whether node j is i or before it on the way to the root."""
    batch, nodes = parents.shape
    at = torch.arange(nodes, device="cuda")
    seen = (at == at.unsqueeze(1)) | (parents.unsqueeze(-1) == at)
    for _ in range(nodes.bit_length()):  # twice as many generations each time
        seen = (seen.float() @ seen.float()) > 0
    return seen


def _words(bits):
    """[.., n] truth values as [.., ceil(n / 32)] words of 32 bits."""
    n = bits.shape[-1]
    bits = torch.nn.functional.pad(bits.long(), (0, -n % 32)).view(*bits.shape[:-1], -1, 32)
    w = (bits << torch.arange(32, device="cuda")).sum(-1)
    return torch.where(w >= 2 ** 31, w - 2 ** 32, w).to(torch.int32)


def _prepare_tree(c, g):
    heads, kv, hd = HEADS[c["heads"]]
    lens, sizes = zip(*_trees(c))
    counts = [-(-(n + t) // c["page"]) for n, t in zip(lens, sizes)]
    table, pool = _pages(g, counts, max(counts) + c["spare"])
    # heads differ in how sharply they attend
    sharp = torch.linspace(0.5, 3.0, heads, device="cuda").unsqueeze(1)
    q = (torch.randn((c["batch"], c["nodes"], heads, hd), generator=g, device="cuda") * sharp).to(torch.bfloat16)
    t = {"q": q, "k": _normal(g, pool, kv, c["page"] * hd), "v": _normal(g, pool, kv, c["page"], hd), "table": table,
         "len": _ints(lens), "count": _ints(sizes)}
    if c["masked"]:
        t["mask"] = _words(_ancestors(_parents(g, c["batch"], c["nodes"])))
    return t


def _prepare_append(c, g):
    heads, kv, hd = HEADS[c["heads"]]
    seq, pos, slot = zip(*_appended(c))
    first, last = {}, {}
    for s, j in zip(seq, slot):
        first.setdefault(s, j // c["page"])
        last[s] = j // c["page"] + 1
    table, pool = _late_pages(g, list(first.values()), list(last.values()), 2)
    off = _idle(c["tokens"], c["idle"])
    cos, sin = _rotation(max(pos) + 1, hd)
    t = {"qkv": _normal(g, c["tokens"], (heads + 2 * kv) * hd), "cos": cos, "sin": sin, "seq": _ints(seq),
         "pos": _ints([NONE if i in off else p for i, p in enumerate(pos)]), "table": table,
         "k": _normal(g, pool, kv, c["page"] * hd), "v": _normal(g, pool, kv, c["page"], hd),
         "q": torch.zeros(c["tokens"], heads, hd, device="cuda", dtype=torch.bfloat16)}
    if c["tree"]:
        t["slot"] = _ints(slot)
    if c["norm"]:
        # projections' heads differ in size; a norm's weights lie about 1
        t["qkv"] = (t["qkv"].float().view(c["tokens"], -1, hd) *
                    torch.linspace(0.2, 4.0, heads + 2 * kv, device="cuda").unsqueeze(1)).flatten(1).to(torch.bfloat16)
        t["wq"], t["wk"] = ((1 + 0.3 * torch.randn(hd, generator=g, device="cuda")).to(torch.bfloat16) for _ in "qk")
    return t


def _prepare_probs(c, g):
    rows, n = c["rows"], c["n"]
    z = 2.5 * torch.randn((rows, n), generator=g, device="cuda")
    if c["masked"]:  # a grammar allows a few tokens of some rows, most of others
        share = 0.9 * torch.rand((rows, 1), generator=g, device="cuda") ** 2
        z = z.masked_fill(torch.rand((rows, n), generator=g, device="cuda") < share, -math.inf)
    heat = 0.3 + 1.2 * torch.rand(rows, generator=g, device="cuda")
    heat[torch.arange(rows, device="cuda") % 7 == 3] = 0.0  # greedy requests among them
    return {"z": z if c["f32"] else z.bfloat16(), "heat": heat}


def _prepare_verify(c, g):
    batch, nodes, n = c["batch"], c["nodes"], c["n"]
    z = 2.5 * torch.randn((batch, nodes, n), generator=g, device="cuda")
    p = torch.softmax(z, -1)
    # the draft model knows the target's distributions roughly
    q = torch.softmax(z.add_(torch.randn((batch, nodes, n), generator=g, device="cuda"), alpha=0.7), -1)
    del z
    parents = _parents(g, batch, nodes) if c["tree"] else (torch.arange(nodes, device="cuda") - 1).repeat(batch, 1)
    row = torch.arange(batch, device="cuda")
    u = torch.rand((batch, nodes), generator=g, device="cuda")
    tokens = torch.zeros((batch, nodes), device="cuda", dtype=torch.int64)
    for i in range(1, nodes):
        at = parents[:, i]
        if c["drafts"]:  # drawn from the draft's distribution at the parent
            sums = q[row, at].double().cumsum(-1)
            tokens[:, i] = torch.searchsorted(sums, u[:, i:i + 1].double() * sums[:, -1:], right=True).view(-1)
        else:  # the parent's likeliest, then its next likeliest, ..
            rank = (parents[:, :i] == at.unsqueeze(1)).sum(1).clamp(max=7)
            tokens[:, i] = q[row, at].topk(8).indices[row, rank]
    t = {"p": p, "tokens": tokens.clamp(max=n - 1).to(torch.int32),
         "count": _ints([max(1, nodes - (i * 3) % (nodes // 3 + 1)) for i in range(batch)]),
         "u": torch.rand((batch, nodes), generator=g, device="cuda")}
    if c["drafts"]:
        t["q"] = q
    if c["tree"]:
        t["parents"] = parents.to(torch.int32)
    return t


def _pools(g, c, pool):
    heads, kv, hd = HEADS[c["heads"]]
    return {"k": _normal(g, c["layers"], pool, kv, c["page"] * hd), "v": _normal(g, c["layers"], pool, kv, c["page"], hd)}


def _prepare_compact(c, g):
    lens = _spread(c["lo"], c["hi"], c["batch"])
    firsts = [n // c["page"] for n in lens]
    table, pool = _late_pages(g, firsts, [-(-(n + c["nodes"]) // c["page"]) for n in lens], 1)
    took = torch.randint(1, c["most"] + 1, (c["batch"],), generator=g, device="cuda")
    # the root, then nodes of later and later levels
    rest = torch.rand((c["batch"], c["nodes"]), generator=g, device="cuda")
    at = torch.arange(c["nodes"], device="cuda")
    rest = torch.where(at >= c["most"], rest, -1.0).topk(c["most"], 1).indices.sort(1).values
    rank = torch.arange(c["most"], device="cuda")
    path = torch.where(rank == 0, 0, rest)
    path = torch.where(rank < took.unsqueeze(1), path, NONE)
    path = torch.nn.functional.pad(path, (0, c["nodes"] - c["most"]), value=NONE)
    return _pools(g, c, pool) | {"table": table, "len": _ints(lens), "path": path.to(torch.int32),
                                 "count": took.to(torch.int32), "new": torch.zeros_like(_ints(lens))}


def _fork_sizes(c):
    lens = _spread(c["lo"], c["hi"], c["parents"])
    counts = [-(-(n + c["extra"]) // c["page"]) for n in lens]
    return lens, counts


def _prepare_fork(c, g):
    lens, counts = _fork_sizes(c)
    parents, forks = c["parents"], c["forks"]
    room = max(counts)
    spare = forks * (1 + -(-(c["page"] + c["extra"]) // c["page"])) + 2
    pool = sum(counts) + spare
    ids = torch.randperm(pool, generator=g, device="cuda")
    count = torch.tensor(counts, device="cuda")
    at = torch.arange(room + 1, device="cuda")
    table = torch.full((parents + forks, room + 1), NONE, device="cuda", dtype=torch.int64)
    table[:parents] = torch.where(at < count.unsqueeze(1),
                                  ids[((count.cumsum(0) - count).unsqueeze(1) + at).clamp(max=pool - 1)], NONE)
    refs = torch.zeros(pool, device="cuda", dtype=torch.int32)
    refs[ids[:sum(counts)]] = 1
    which = torch.arange(forks, device="cuda")
    return _pools(g, c, pool) | {"table": table.to(torch.int32), "refs": refs, "len": _ints(lens + [0] * forks),
                                 "from": (which % parents).to(torch.int32), "to": (parents + which).to(torch.int32),
                                 "extra": _ints([c["extra"]] * (parents + forks)),
                                 "lost": torch.zeros(forks, device="cuda", dtype=torch.int32),
                                 "missing": torch.zeros(parents + forks, device="cuda", dtype=torch.int32)}


_PREPARE = {"tree": _prepare_tree, "append": _prepare_append, "probs": _prepare_probs, "verify": _prepare_verify,
            "compact": _prepare_compact, "fork": _prepare_fork}


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
    for name in list(t):
        held = _storage(tuple(t[name].shape), t[name].dtype)
        held.copy_(t.pop(name))
        t[name] = held
    torch.cuda.synchronize()
    state["calls"] = _BIND[c["kind"]](c, t)


def _bind_tree(c, t):
    from foundry_amd import _lib
    heads, kv, hd = HEADS[c["heads"]]
    t["out"] = _storage(tuple(t["q"].shape), torch.bfloat16)
    pool, width = t["k"].shape[0], t["table"].shape[1]
    nbytes = _lib.paged_tree_attention_workspace_bytes(c["batch"], c["nodes"], heads, kv, hd, c["page"], width)
    t["ws"] = _storage((nbytes,), torch.uint8)
    return [("fh_paged_tree_attention", _device.handle, _ptr(t["q"]), c["batch"], c["nodes"], heads, kv, hd,
             _ptr(t["k"]), _ptr(t["v"]), pool, c["page"], _ptr(t["table"]), width, _ptr(t["len"]), _ptr(t["count"]),
             _ptr(t.get("mask")), ctypes.c_float(hd ** -0.5), _ptr(t["ws"]), nbytes, _ptr(t["out"]))]


def _bind_append(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    seqs, width = t["table"].shape
    return [("fh_paged_norm_rope_kv", _device.handle, _ptr(t["qkv"]), c["tokens"], heads, kv, hd, _ptr(t.get("wq")),
             _ptr(t.get("wk")), ctypes.c_float(EPS), _ptr(t["cos"]), _ptr(t["sin"]), t["cos"].shape[0], _ptr(t["seq"]),
             _ptr(t["pos"]), _ptr(t.get("slot")), _ptr(t["table"]), seqs, width, _ptr(t["k"]), _ptr(t["v"]),
             t["k"].shape[0], c["page"], _ptr(t["q"]))]


def _bind_probs(c, t):
    from foundry_amd import _lib
    t["out"] = _storage((c["rows"], c["n"]), torch.float32)
    nbytes = _lib.logits_probs_workspace_bytes(c["rows"], c["n"])
    t["ws"] = _storage((nbytes,), torch.uint8)
    return [("fh_logits_probs", _device.handle, _ptr(t["z"]), _lib.F32 if c["f32"] else _lib.BF16, c["rows"], c["n"],
             _ptr(t["heat"]), _ptr(t["ws"]), nbytes, _ptr(t["out"]))]


def _bind_verify(c, t):
    from foundry_amd import _lib
    batch, nodes, n = c["batch"], c["nodes"], c["n"]
    t["path"], t["said"] = (_storage((batch, nodes), torch.int32) for _ in range(2))
    t["took"] = _storage((batch,), torch.int32)
    nbytes = _lib.verify_draft_workspace_bytes(batch, nodes, n)
    t["ws"] = _storage((nbytes,), torch.uint8)
    return [("fh_verify_draft", _device.handle, _ptr(t["p"]), _ptr(t.get("q")), batch, nodes, n, _ptr(t["tokens"]),
             _ptr(t.get("parents")), _ptr(t["count"]), _ptr(t["u"]), _ptr(t["ws"]), nbytes, _ptr(t["path"]),
             _ptr(t["said"]), _ptr(t["took"]))]


def _cache(c, t):
    from foundry_amd import _lib
    heads, kv, hd = HEADS[c["heads"]]
    pools = (_lib.PagedPool * c["layers"])(*[(t["k"][i].data_ptr(), t["v"][i].data_ptr()) for i in range(c["layers"])])
    cache = _lib.PagedCache(pools=pools, n_layers=c["layers"], n_kv=kv, head_dim=hd, n_pages=t["k"].shape[1],
                            page_size=c["page"], page_table=t["table"].data_ptr(), n_seqs=t["table"].shape[0],
                            max_pages=t["table"].shape[1], lengths=t["len"].data_ptr(),
                            refs=t["refs"].data_ptr() if "refs" in t else None)
    t["cache"] = cache
    return ctypes.byref(cache)


def _bind_compact(c, t):
    return [("fh_paged_compact", _device.handle, _cache(c, t), _ptr(t["path"]), _ptr(t["count"]), c["nodes"],
             _ptr(t["new"]))]


def _bind_fork(c, t):
    cache = _cache(c, t)
    return [("fh_paged_free", _device.handle, cache, _ptr(t["to"]), c["forks"]),
            ("fh_paged_fork", _device.handle, cache, _ptr(t["from"]), _ptr(t["to"]), c["forks"], _ptr(t["lost"])),
            ("fh_paged_reserve", _device.handle, cache, _ptr(t["extra"]), _ptr(t["missing"]))]


_BIND = {"tree": _bind_tree, "append": _bind_append, "probs": _bind_probs, "verify": _bind_verify,
         "compact": _bind_compact, "fork": _bind_fork}
_RESULT = {"tree": ["out"], "append": ["q", "k", "v"], "probs": ["out"], "verify": ["path", "said", "took"],
           "compact": ["k", "v", "new"], "fork": ["k", "v", "table", "refs", "len", "lost", "missing"]}


# ---------------------------------------------------------------------- run

def run(state):
    c, t = state["case"], state["t"]
    if own:
        from foundry_amd import _lib
        for call in state["calls"]:
            _lib.call(*call)
        return {name: t[name] for name in _RESULT[c["kind"]]}
    return dict(zip(_RESULT[c["kind"]], _PLAIN[c["kind"]](c, t)))


def _key_offset(slot, hd):
    """Where key `slot` of a page's region holds its dims [..., hd]: groups of
    16 keys, each laid out [hd / 32][16][32]."""
    d = torch.arange(hd, device="cuda")
    return (slot // 16 * 16 * hd + slot % 16 * 32).unsqueeze(-1) + d // 32 * 512 + d % 32


def _plain_tree(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    batch, nodes = c["batch"], c["nodes"]
    keys = t["table"].shape[1] * c["page"]
    ids = t["table"].clamp(min=0).long()
    at = _key_offset(torch.arange(c["page"], device="cuda"), hd)
    k = t["k"][:, :, at.flatten()].view(t["v"].shape)[ids].float()  # [batch, pages, kv, page, hd]
    k = k.permute(0, 2, 4, 1, 3).reshape(batch, kv, hd, keys)
    v = t["v"][ids].float().permute(0, 2, 1, 3, 4).reshape(batch, kv, keys, hd)
    j = torch.arange(keys, device="cuda")
    length, count = t["len"].view(-1, 1, 1), t["count"].view(-1, 1, 1)
    node = torch.arange(nodes, device="cuda").view(-1, 1)
    rel = j - length  # the key's node
    if c["masked"]:
        word = t["mask"].gather(2, (rel // 32).clamp(0, t["mask"].shape[2] - 1).expand(-1, nodes, -1))
        own_branch = (word >> (rel % 32).int()) & 1 == 1
    else:
        own_branch = rel <= node
    seen = ((rel < 0) | ((rel < count) & own_branch)) & (node < count)
    seen = seen.view(batch, 1, 1, nodes, keys)
    group = heads // kv
    q = t["q"].float().view(batch, nodes, kv, group, hd).permute(0, 2, 3, 1, 4).reshape(batch, kv, group * nodes, hd)
    s = (q @ k * hd ** -0.5).view(batch, kv, group, nodes, keys)
    top = s.masked_fill(~seen, -math.inf).amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    e = torch.where(seen, (s - top).exp(), 0.0)
    del s
    out = (e.view(batch, kv, group * nodes, keys) @ v).view(batch, kv, group, nodes, hd) / e.sum(-1, keepdim=True)
    out = torch.where(seen.any(-1, keepdim=True), out, 0.0)
    return [out.permute(0, 3, 1, 2, 4).reshape(batch, nodes, heads, hd).bfloat16()]


def _plain_append(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    live = t["pos"] >= 0
    pos, seq = t["pos"].clamp(min=0).long(), t["seq"].long()
    place = t["slot"].long() if c["tree"] else pos
    x = t["qkv"].float().view(c["tokens"], heads + 2 * kv, hd)[:, :heads + kv]
    if c["norm"]:
        w = torch.cat([t["wq"].float().expand(heads, hd), t["wk"].float().expand(kv, hd)])
        x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt() * w
    cos, sin = t["cos"][pos].float().unsqueeze(1), t["sin"][pos].float().unsqueeze(1)
    half = torch.cat([-x[..., hd // 2:], x[..., :hd // 2]], -1)
    rot = (x * cos + half * sin).bfloat16()
    page = t["table"][seq, place // c["page"]].long()
    page, slot, rot = page[live], (place % c["page"])[live], rot[live]
    value = t["qkv"].view(c["tokens"], -1, hd)[live, heads + kv:]
    t["q"][live] = rot[:, :heads]
    row = torch.arange(kv, device="cuda")
    at = _key_offset(slot, hd).unsqueeze(1)
    t["k"][page.view(-1, 1, 1), row.view(1, -1, 1), at] = rot[:, heads:]
    t["v"][page.view(-1, 1), row, slot.view(-1, 1)] = value
    return [t["q"], t["k"], t["v"]]


def _plain_probs(c, t):
    z, heat = t["z"].float(), t["heat"].unsqueeze(1)
    ids = torch.arange(c["n"], device="cuda")
    best = ids == torch.where(z == z.amax(-1, keepdim=True), ids, c["n"]).amin(-1, keepdim=True)
    s = z / heat.clamp(min=1e-30)
    e = (s - s.amax(-1, keepdim=True)).exp()
    return [torch.where(heat > 0, e / e.sum(-1, keepdim=True), best.float())]


def _plain_verify(c, t):
    batch, nodes, n = c["batch"], c["nodes"], c["n"]
    row, ids = torch.arange(batch, device="cuda"), torch.arange(n, device="cuda")
    tokens, u = t["tokens"].long(), t["u"].double()
    if c["tree"]:
        parents = t["parents"].long()
    else:
        parents = (torch.arange(nodes, device="cuda") - 1).expand(batch, nodes)
    at = torch.zeros(batch, device="cuda", dtype=torch.int64)  # the last accepted node
    took = torch.ones_like(at)
    path = torch.full((batch, nodes), NONE, device="cuda", dtype=torch.int64)
    said = path.clone()
    path[:, 0] = 0
    # what is left of the target's distribution at that node: p - cut * q where positive
    cut = torch.zeros(batch, device="cuda", dtype=torch.float64)
    mass = torch.ones_like(cut)
    gone = torch.zeros((batch, n), device="cuda", dtype=torch.bool)  # tokens refused there, without the draft's distribution
    for i in range(1, nodes):
        x = tokens[:, i]
        asked = (parents[:, i] == at) & (i < t["count"])
        p_x = t["p"][row, at, x].double()
        q_x = t["q"][row, at, x].double() if c["drafts"] else torch.ones_like(p_x)
        left = (p_x - cut * q_x).clamp(min=0) if c["drafts"] else torch.where(gone[row, x], 0.0, p_x)
        yes = asked & (u[:, i] * q_x * mass < left)
        no = asked & ~yes
        if c["drafts"]:
            cut = torch.where(yes, 0.0, torch.where(no, cut + mass, cut))
            rest = (t["p"][row, at].double() - cut.unsqueeze(1) * t["q"][row, at]).clamp(min=0).sum(-1)
            mass = torch.where(yes, 1.0, torch.where(no, rest, mass))
        else:
            mass = torch.where(yes, 1.0, torch.where(no, mass - left, mass))
            gone[row, x] = gone[row, x] | no
            gone = gone & ~yes.unsqueeze(1)
        path[row, took.clamp(max=nodes - 1)] = torch.where(yes, i, path[row, took.clamp(max=nodes - 1)])
        said[row, took - 1] = torch.where(yes, x, said[row, took - 1])
        took = took + yes
        at = torch.where(yes, i, at)
    p = t["p"][row, at].double()
    if c["drafts"]:
        left = (p - cut.unsqueeze(1) * t["q"][row, at]).clamp(min=0)
    else:
        left = torch.where(gone, 0.0, p)
    left = torch.where(left.sum(-1, keepdim=True) > 0, left, p)
    sums = left.cumsum(-1)
    past = sums > u[:, :1] * sums[:, -1:]
    said[row, took - 1] = torch.where(past, ids, n).amin(-1).clamp(max=n - 1)
    return [path.to(torch.int32), said.to(torch.int32), took.to(torch.int32)]


def _plain_compact(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    at = torch.arange(c["nodes"], device="cuda")
    seq, rank = (at < t["count"].unsqueeze(1)).nonzero(as_tuple=True)
    place = lambda j: (t["table"][seq, j // c["page"]].long(), j % c["page"])  # noqa: E731
    start = t["len"].long()[seq]
    (page, slot), (page2, slot2) = place(start + t["path"].long()[seq, rank]), place(start + rank)
    t["v"][:, page2, :, slot2] = t["v"][:, page, :, slot]
    row = torch.arange(kv, device="cuda").view(1, -1, 1)
    k = t["k"][:, page.view(-1, 1, 1), row, _key_offset(slot, hd).unsqueeze(1)]
    t["k"][:, page2.view(-1, 1, 1), row, _key_offset(slot2, hd).unsqueeze(1)] = k
    t["new"].copy_(t["len"] + t["count"])
    return [t["k"], t["v"], t["new"]]


def _take(t, want):
    """The lowest free pages for the places of the table that `want` marks, in order; where they end, none."""
    free = t["refs"] == 0
    ids = torch.where(free, torch.arange(len(free), device="cuda"), len(free)).sort().values
    ids = torch.cat([torch.where(ids == len(free), NONE, ids), torch.full_like(want.flatten(), NONE, dtype=torch.int64)])
    got = ids[(want.flatten().long().cumsum(0) - 1).clamp(min=0)].view(want.shape)
    got = torch.where(want, got, NONE)
    t["refs"].scatter_add_(0, got.clamp(min=0).flatten(), (got >= 0).flatten().int())
    return got


def _plain_fork(c, t):
    page, table, refs, width = c["page"], t["table"], t["refs"], t["table"].shape[1]
    src, dst = t["from"].long(), t["to"].long()
    entry = torch.arange(width, device="cuda")
    # the old ones go
    old = table[dst].long()
    refs.scatter_add_(0, old.clamp(min=0).flatten(), -(old >= 0).flatten().int())
    table[dst], t["len"][dst] = NONE, 0
    # whole pages are shared, the last one is copied
    length = t["len"][src].long()
    whole, part = (length // page).unsqueeze(1), length % page
    shared = torch.where(entry < whole, table[src].long(), NONE)
    refs.scatter_add_(0, shared.clamp(min=0).flatten(), (shared >= 0).flatten().int())
    want = (entry == whole) & (part > 0).unsqueeze(1)
    got = _take(t, want)
    # a fork that gets no page for its copy stays empty
    lost = (want & (got < 0)).any(1)
    back = (shared >= 0) & lost.unsqueeze(1)
    refs.scatter_add_(0, shared.clamp(min=0).flatten(), -back.flatten().int())
    table[dst] = torch.where(lost.unsqueeze(1), NONE, torch.where(got >= 0, got, shared)).int()
    t["lost"].copy_(lost)
    t["len"][dst] = torch.where(lost, 0, length).int()
    slot = torch.arange(page, device="cuda")
    used = (slot < part.unsqueeze(1)) & ~lost.unsqueeze(1)
    to = got.amax(1)
    at = table[src, whole.view(-1).clamp(max=width - 1)].long()
    which, slot = used.nonzero(as_tuple=True)
    t["v"][:, to[which], :, slot] = t["v"][:, at[which], :, slot]
    heads, kv, hd = HEADS[c["heads"]]
    row, key = torch.arange(kv, device="cuda").view(1, -1, 1), _key_offset(slot, hd).unsqueeze(1)
    t["k"][:, to[which].view(-1, 1, 1), row, key] = t["k"][:, at[which].view(-1, 1, 1), row, key]
    # room for the next tokens
    first, end = t["len"].long() // page, (t["len"].long() + t["extra"] + page - 1) // page
    want = (entry >= first.unsqueeze(1)) & (entry < end.unsqueeze(1)) & (table < 0)
    got = _take(t, want)
    t["missing"].copy_((want & (got < 0)).sum(1))
    table.copy_(torch.where(got >= 0, got, table.long()))
    return [t[name] for name in _RESULT["fork"]]


_PLAIN = {"tree": _plain_tree, "append": _plain_append, "probs": _plain_probs, "verify": _plain_verify,
          "compact": _plain_compact, "fork": _plain_fork}


# --------------------------------------------------------------------- work

def work(case):
    c = case
    if "heads" in c:
        heads, kv, hd = HEADS[c["heads"]]
    if c["kind"] == "tree":
        trees = _trees(c)
        keys, nodes = sum(n + t for n, t in trees), sum(t for _, t in trees)
        nbytes = 4 * keys * kv * hd + 4 * c["batch"] * c["nodes"] * heads * hd + 8 * c["batch"]
        nbytes += 4 * sum(-(-(n + t) // c["page"]) for n, t in trees)
        nbytes += 4 * nodes * -(-c["nodes"] // 32) if c["masked"] else 0
        return {"bytes": nbytes, "flops": 4 * sum((n + t / 2) * t for n, t in trees) * heads * hd}
    if c["kind"] == "append":
        live = c["tokens"] - len(_idle(c["tokens"], c["idle"]))
        places = len({p for _, p, _ in _appended(c)})  # rows of the two tables
        nbytes = 4 * live * (heads + 2 * kv) * hd + 4 * places * hd + (16 if c["tree"] else 12) * c["tokens"]
        return {"bytes": nbytes, "flops": (8 if c["norm"] else 3) * live * (heads + kv) * hd}
    if c["kind"] == "probs":
        return {"bytes": c["rows"] * (c["n"] * (8 if c["f32"] else 6) + 4), "flops": 4 * c["rows"] * c["n"]}
    if c["kind"] == "verify":
        # the last accepted node's distributions, once each; the others matter at single tokens alone
        nbytes = c["batch"] * ((8 if c["drafts"] else 4) * c["n"] + 32 * c["nodes"])
        return {"bytes": nbytes, "flops": 3 * c["batch"] * c["n"]}
    if c["kind"] == "compact":
        moved = c["batch"] * (c["most"] - 1) / 2  # the root stays where it is
        return {"bytes": 8 * moved * c["layers"] * kv * hd + 4 * c["batch"] * c["most"], "flops": 0}
    lens, _ = _fork_sizes(c)
    each = c["forks"] // c["parents"]
    copied = each * sum(n % c["page"] for n in lens)
    entries = each * sum(-(-(n + c["extra"]) // c["page"]) for n in lens)
    return {"bytes": 8 * copied * c["layers"] * kv * hd + 16 * entries, "flops": 0}


# -------------------------------------------------------------------- exact

def exact(case, seed):
    if case["kind"] == "verify" and case["batch"] * case["nodes"] > 2000:
        return None
    t = _PREPARE[case["kind"]](case, _gen(seed))
    return dict(zip(_RESULT[case["kind"]], _EXACT[case["kind"]](case, t)))


def _grouped(k, kv, page, hd):
    """[pages, kv, page * hd] as keys [pages, kv, page, hd]."""
    return k.view(-1, kv, page // 16, hd // 32, 16, 32).transpose(3, 4).reshape(-1, kv, page, hd)


def _exact_tree(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    out = torch.zeros(t["q"].shape, device="cuda", dtype=torch.float64)
    for b in range(c["batch"]):
        n, size = int(t["len"][b]), int(t["count"][b])
        if size == 0:
            continue
        pages = t["table"][b, :-(-(n + size) // c["page"])].long()
        k = _grouped(t["k"][pages], kv, c["page"], hd).transpose(0, 1).reshape(kv, -1, hd)[:, :n + size]
        v = t["v"][pages].transpose(0, 1).reshape(kv, -1, hd)[:, :n + size]
        hidden = torch.ones(size, size, device="cuda", dtype=torch.bool).triu(1)
        if c["masked"]:
            bits = (t["mask"][b, :size].long().unsqueeze(-1) >> torch.arange(32, device="cuda")) & 1
            hidden = bits.flatten(1)[:, :size] == 0
        hidden = torch.nn.functional.pad(hidden, (n, 0))
        for h in range(heads):
            s = t["q"][b, :size, h].double() @ k[h * kv // heads].double().T / math.sqrt(hd)
            out[b, :size, h] = torch.softmax(s.masked_fill(hidden, -math.inf), -1) @ v[h * kv // heads].double()
    return [out]


def _exact_append(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    q, v = t["q"].double(), t["v"].double()
    k = _grouped(t["k"].double(), kv, c["page"], hd)
    live = t["pos"] >= 0
    pos, seq = t["pos"][live].long(), t["seq"][live].long()
    place = t["slot"][live].long() if c["tree"] else pos
    x = t["qkv"][live].double().view(len(pos), heads + 2 * kv, hd)
    y = x[:, :heads + kv]
    if c["norm"]:
        w = torch.cat([t["wq"].double().repeat(heads, 1), t["wk"].double().repeat(kv, 1)])
        y = y * torch.rsqrt((y * y).sum(-1, keepdim=True) / hd + EPS) * w
    # the rotation as a product of complex numbers, dims d and d + hd / 2 together
    a, b = y.chunk(2, -1)
    (ca, cb), (sa, sb) = [w[pos].double().unsqueeze(1).chunk(2, -1) for w in (t["cos"], t["sin"])]
    rot = torch.cat([a * ca - b * sa, b * cb + a * sb], -1)
    q[live] = rot[:, :heads]
    page, slot = t["table"][seq, place // c["page"]].long(), place % c["page"]
    k[page, :, slot] = rot[:, heads:]
    v[page, :, slot] = x[:, heads + kv:]
    k = k.view(-1, kv, c["page"] // 16, 16, hd // 32, 32).transpose(3, 4).reshape(t["k"].shape)
    return [q, k, v]


def _exact_probs(c, t):
    out = torch.zeros((c["rows"], c["n"]), device="cuda", dtype=torch.float64)
    for r in range(c["rows"]):
        heat = float(t["heat"][r])
        if heat > 0:
            out[r] = torch.softmax(t["z"][r].double() / heat, -1)
        else:
            out[r, (t["z"][r] == t["z"][r].max()).nonzero()[0]] = 1.0
    return [out]


def _exact_verify(c, t):
    path, said, took = [], [], []
    for b in range(c["batch"]):
        size, u = int(t["count"][b]), t["u"][b].tolist()
        tokens = t["tokens"][b].tolist()
        parents = t["parents"][b].tolist() if c["tree"] else list(range(-1, c["nodes"] - 1))
        nodes, words, at = [0], [], 0
        while True:
            # what may follow node `at`, as weights; nothing yet is refused
            left, total, go = t["p"][b, at].double(), 1.0, None
            for i in range(1, size):
                if parents[i] != at:
                    continue
                x = tokens[i]
                drawn = float(t["q"][b, at, x]) if c["drafts"] else 1.0
                if u[i] * drawn * total < float(left[x]):
                    go = i
                    break
                # the rest is in proportion to max(left / total - draft, 0)
                if c["drafts"]:
                    left = torch.clamp(left - total * t["q"][b, at].double(), min=0)
                    total = float(left.sum())
                else:
                    total -= float(left[x])
                    left = left.clone()
                    left[x] = 0
            if go is None:
                break
            at = go
            nodes.append(go)
            words.append(tokens[go])
        if float(left.sum()) <= 0:
            left = t["p"][b, at].double()
        sums = torch.cumsum(left, 0)
        words.append(min(c["n"] - 1, int((sums <= u[0] * float(sums[-1])).sum())))
        fill = [NONE] * (c["nodes"] - len(nodes))
        path.append(nodes + fill)
        said.append(words + fill)
        took.append(len(nodes))
    return [_ints(path), _ints(said), _ints(took)]


def _exact_compact(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    k = t["k"].view(c["layers"], -1, kv, c["page"] // 16, hd // 32, 16, 32).clone()
    v = t["v"].clone()
    for b in range(c["batch"]):
        n, row = int(t["len"][b]), t["table"][b].tolist()
        for i, node in enumerate(t["path"][b, :int(t["count"][b])].tolist()):
            (p, s), (p2, s2) = ((row[j // c["page"]], j % c["page"]) for j in (n + node, n + i))
            v[:, p2, :, s2] = v[:, p, :, s]
            k[:, p2, :, s2 // 16, :, s2 % 16] = k[:, p, :, s // 16, :, s % 16]
    return [k.view(t["k"].shape), v, t["len"] + t["count"]]


def _exact_fork(c, t):
    heads, kv, hd = HEADS[c["heads"]]
    page = c["page"]
    k = t["k"].view(c["layers"], -1, kv, page // 16, hd // 32, 16, 32).clone()
    v = t["v"].clone()
    table, refs, lens = (t[name].tolist() for name in ("table", "refs", "len"))

    def take():
        for i, r in enumerate(refs):
            if r == 0:
                refs[i] = 1
                return i
        return NONE

    for d in t["to"].tolist():
        for p in table[d]:
            if p >= 0:
                refs[p] -= 1
        table[d], lens[d] = [NONE] * len(table[d]), 0
    pairs = list(zip(t["from"].tolist(), t["to"].tolist()))
    for s, d in pairs:
        for e in range(lens[s] // page):
            table[d][e] = table[s][e]
            refs[table[s][e]] += 1
    lost = []
    for s, d in pairs:
        e, part = lens[s] // page, lens[s] % page
        lost.append(0)
        if part:
            p = table[d][e] = take()
            lost[-1] = int(p < 0)
            v[:, p, :, :part] = v[:, table[s][e], :, :part]
            for j in range(part):
                k[:, p, :, j // 16, :, j % 16] = k[:, table[s][e], :, j // 16, :, j % 16]
        lens[d] = lens[s]
    missing = []
    for s, n in enumerate(lens):
        missing.append(0)
        for e in range(n // page, -(-(n + c["extra"]) // page)):
            if table[s][e] < 0:
                table[s][e] = take()
                missing[-1] += table[s][e] < 0
    return [k.view(t["k"].shape), v, _ints(table), _ints(refs), _ints(lens), _ints(lost), _ints(missing)]


_EXACT = {"tree": _exact_tree, "append": _exact_append, "probs": _exact_probs, "verify": _exact_verify,
          "compact": _exact_compact, "fork": _exact_fork}

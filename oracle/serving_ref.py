"""The serving operators restated in float64 numpy, from their definitions in
include/foundry_hip.h: the paged append, paged attention, low-rank adapters
and logit rules. Each returns the exact result and, where sums are involved,
the magnitudes that a bound on an fp32 computation's error needs.
"""
import numpy as np

NONE = 0xFFFFFFFF


def f64(bits):
    """bf16 bits as float64."""
    return (np.asarray(bits, dtype=np.uint32) << 16).view(np.float32).astype(np.float64)


def append(qkv, n_heads, n_kv, cos, sin, sequences, positions, table, n_pages, page):
    """Rotated q [t, heads, hd] and k, plain v [t, kv, hd] (float64), the bound's
    magnitudes of q and k, and each token's (page, slot) or None."""
    t, hd = len(positions), cos.shape[1]
    x = f64(qkv).reshape(t, n_heads + 2 * n_kv, hd)
    place = []
    for i in range(t):
        p, s = int(positions[i]), int(sequences[i])
        ok = p < table.shape[1] * page and p < cos.shape[0] and s < table.shape[0]
        pid = int(table[s, p // page]) if ok else NONE
        place.append((pid, p % page) if pid < n_pages else None)
    rot = np.zeros((t, n_heads + n_kv, hd))
    mag = np.zeros_like(rot)
    for i, at in enumerate(place):
        if at is None:
            continue
        a = x[i, :n_heads + n_kv]
        half = np.concatenate([-a[:, hd // 2:], a[:, :hd // 2]], -1)
        c, s = f64(cos[int(positions[i])]), f64(sin[int(positions[i])])
        rot[i], mag[i] = a * c + half * s, np.abs(a * c) + np.abs(half * s)
    return rot[:, :n_heads], rot[:, n_heads:], x[:, n_heads + n_kv:], mag, place


def attend(q, keys, values, table, positions, scale):
    """q [b, heads, hd]; keys, values [pages, kv, page, hd], all float64.
    Returns out, sum p |v|, and the largest sum |q||k| * scale of a row."""
    b, heads, hd = q.shape
    n_pages, kv, page, _ = keys.shape
    out, weight, reach = np.zeros(q.shape), np.zeros(q.shape), np.zeros((b, heads, 1))
    for i in range(b):
        n = int(positions[i]) + 1
        if n > table.shape[1] * page:
            continue
        at = [(int(table[i, j // page]), j % page) for j in range(n)]
        at = [(p, s) for p, s in at if p < n_pages]
        if not at:
            continue
        pages, slots = np.array(at).T
        for h in range(heads):
            k, v = keys[pages, h * kv // heads, slots], values[pages, h * kv // heads, slots]
            s = k @ q[i, h] * scale
            with np.errstate(invalid="ignore"):
                e = np.exp(s - s.max())
                p = e / e.sum()
                out[i, h], weight[i, h] = p @ v, p @ np.abs(v)
                reach[i, h] = (np.abs(k) @ np.abs(q[i, h])).max() * scale
    return out, weight, reach


def lora(x, a, b, scales, adapters, base):
    """y, and the magnitude sum |x||A| pushed through |B|, plus |v| through |B|."""
    y, mag, low = base.copy(), np.zeros(base.shape), np.zeros(base.shape)
    for i, u in enumerate(adapters):
        if u < a.shape[0]:
            v = a[u] @ x[i] * scales[u]
            y[i] += b[u] @ v
            mag[i] = np.abs(b[u]) @ (np.abs(a[u]) @ np.abs(x[i])) * abs(scales[u])
            low[i] = np.abs(b[u]) @ np.abs(v)
    return y, mag, low


def logits(z, rules, dtype=np.float64):
    """The rules step by step in `dtype` (float32: the steps the library rounds
    at). rules: a dict of numpy arrays under fh_logit_rules' names."""
    rows, n = z.shape
    z = z.astype(dtype)
    for r in range(rows):
        row = z[r]
        if "history" in rules:
            ids = rules["history"][r, :min(int(rules["history_len"][r]), rules["history"].shape[1])].astype(np.int64)
            prompt = int(rules["prompt_len"][r]) if "prompt_len" in rules else 0
            seen = np.unique(ids[ids < n])
            made = ids[prompt:]
            made, times = np.unique(made[made < n], return_counts=True)
            if "repetition" in rules:
                rep = dtype(rules["repetition"][r])
                row[seen] = np.where(row[seen] > 0, row[seen] / rep, row[seen] * rep)
            if "frequency" in rules:
                row[made] = row[made] - dtype(rules["frequency"][r]) * times.astype(dtype)
            if "presence" in rules:
                row[made] = row[made] - dtype(rules["presence"][r])
        if "bias_ids" in rules:
            used = rules["bias_ids"].shape[1]
            if "bias_len" in rules:
                used = min(used, int(rules["bias_len"][r]))
            last = {int(j): dtype(v) for j, v in zip(rules["bias_ids"][r, :used], rules["bias_values"][r, :used])}
            for j, v in last.items():
                if j < n:
                    row[j] = row[j] + v
        if "mask" in rules:
            j = np.arange(n)
            row[(rules["mask"][r, j // 32] >> (j % 32).astype(np.uint32)) & 1 == 0] = -np.inf
    return z

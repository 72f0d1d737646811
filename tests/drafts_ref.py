"""Plain restatements of the operators for drafted tokens (CPU, 64 bits where
values are computed), for the tests."""
import math

import numpy as np

import serving_ref as R


def ancestors(parents, most=256):
    """(sets of rows seen or None, depths) of one request's rows."""
    sets = []
    for i, p in enumerate(parents):
        if i >= most or p < -1 or p >= i or (p >= 0 and sets[p] is None):
            sets.append(None)
        else:
            sets.append((sets[p] if p >= 0 else []) + [i])
    return sets


def draft_tree(parents, starts, lens, tokens, words, window):
    masks, positions = np.zeros((tokens, words), np.uint64), np.full(tokens, -1)
    for r in range(len(lens)):
        s0 = min(max(int(starts[r]), 0), tokens)
        past = int(starts[r + 1])
        s1 = min(max(past, s0), tokens)
        for i, up in enumerate(ancestors(parents[s0:s1], 64 * words)):
            if up is None:
                continue
            positions[s0 + i] = int(lens[r]) - (past - s0) + len(up) - 1
            for j in up[-window:] if window else up:
                masks[s0 + i, j // 64] |= np.uint64(1 << (j % 64))
    return masks.view(np.int64), positions


def bits_of(masks):
    """bool [rows, 64 * words]"""
    m = masks.view(np.uint64)
    return ((m[..., None] >> np.arange(64, dtype=np.uint64)) & np.uint64(1)).astype(bool).reshape(len(m), -1)


def tree_attention(q, codes, scales, table, lens, starts, masks, scale, window):
    """As serving_ref.attention, of rows that see what their masks say."""
    q = q.double().cpu().numpy()
    t, h, d = q.shape
    n_pages, _, hk, page, _ = codes.shape
    codes, scales, table = codes.cpu().numpy(), scales.cpu().numpy(), table.cpu().numpy()
    bits = bits_of(masks.cpu().numpy())
    out, lse = np.zeros((t, h, d)), np.full((t, h), -np.inf)
    spread, size, total = np.zeros((t, h, d)), np.zeros((t, h)), np.zeros((t, h, d))
    for r in range(len(lens)):
        n = int(starts[r + 1]) - int(starts[r])
        base, length = int(lens[r]) - n, min(int(lens[r]), table.shape[1] * page)
        if length <= 0:
            continue
        pages = table[r, :-(-length // page)]
        there = (pages >= 0) & (pages < n_pages)
        pg = np.where(there, pages, 0)
        seen_page = np.repeat(there, page)[:length]
        key = np.arange(length)
        own = key - base
        visible = []
        for row in range(int(starts[r]), min(int(starts[r + 1]), t)):
            some = int(bits[row].sum())
            committed = (some > 0) & (key < base) & ((key >= base + some - window) if window else True)
            drafted = (own >= 0) & (own < bits.shape[1]) & bits[row][np.clip(own, 0, bits.shape[1] - 1)]
            visible.append(seen_page & (committed | drafted))
        for g in range(hk):
            k = R.values(codes[pg, 0, g], scales[pg, 0, g]).reshape(-1, d)[:length]
            v = R.values(codes[pg, 1, g], scales[pg, 1, g]).reshape(-1, d)[:length]
            for i, seen in enumerate(visible):
                row = int(starts[r]) + i
                if not seen.any():
                    continue
                for j in range(g * (h // hk), (g + 1) * (h // hk)):
                    x = k[seen] @ q[row, j] * scale
                    top = x.max()
                    p = np.exp(x - top)
                    lse[row, j] = top + math.log(p.sum())
                    out[row, j] = p @ v[seen] / p.sum()
                    spread[row, j] = p @ np.abs(v[seen]) / p.sum()
                    total[row, j] = np.abs(v[seen]).sum(0)
                    size[row, j] = (np.abs(k[seen]) @ np.abs(q[row, j])).max() * abs(scale)
    return out, lse, spread, size, total


def adjust(x, starts, rules):
    """fp32 rows by the rules, each operation rounded, as numpy does it."""
    y = x.astype(np.float32).copy()
    rows, vocab = y.shape
    of = np.full(rows, -1)
    n = rows if starts is None else len(starts) - 1
    for r in range(n):
        a, b = (r, r + 1) if starts is None else (max(int(starts[r]), 0), int(starts[r + 1]))
        of[a:min(b, rows)] = r
    inside = lambda t: t[(t >= 0) & (t < vocab)]  # noqa: E731
    for row in range(rows):
        r = of[row]
        if r < 0:
            continue
        seen, count = np.zeros(vocab, bool), np.zeros(vocab, np.int64)
        if "history" in rules:
            length = min(max(int(rules["history_lens"][r]), 0), rules["history"].shape[1])
            prompt = max(int(rules["prompt_lens"][r]), 0) if "prompt_lens" in rules else 0
            h = rules["history"][r, :length]
            seen[inside(h)] = True
            np.add.at(count, inside(h[prompt:]), 1)
        if "drafted" in rules:
            a, b = max(int(starts[r]), 0), min(int(starts[r + 1]), rows)
            bits = bits_of(rules["masks"][row:row + 1])[0][:b - a]
            path = inside(rules["drafted"][a:b][np.flatnonzero(bits)])
            seen[path] = True
            np.add.at(count, path, 1)
        v = y[row]
        with np.errstate(all="ignore"):
            if "repetition" in rules:
                rep = np.float32(rules["repetition"][r])
                v = np.where(seen, np.where(v > 0, v / rep, v * rep), v)
            some = count > 0
            if "frequency" in rules:
                v = np.where(some, v - np.float32(rules["frequency"][r]) * count.astype(np.float32), v)
            if "presence" in rules:
                v = np.where(some, v - np.float32(rules["presence"][r]), v)
            if "bias_tokens" in rules:
                add, has = np.zeros(vocab, np.float32), np.zeros(vocab, bool)
                for t, b in zip(rules["bias_tokens"][r], rules["bias_values"][r]):
                    if 0 <= t < vocab:
                        add[t] = add[t] + np.float32(b) if has[t] else np.float32(b)
                        has[t] = True
                v = np.where(has, v + add, v)
            if "temperature" in rules and rules["temperature"][r] > 0:
                v = v / np.float32(rules["temperature"][r])
        if "allowed" in rules:
            bit = (rules["allowed"][row].view(np.uint32)[:, None] >> np.arange(32, dtype=np.uint32)) & 1
            v = np.where(bit.reshape(-1)[:vocab] == 1, v, np.float32(-np.inf))
        y[row] = v
    return y, of


def pick(y, of):
    out = []
    for v, r in zip(y, of):
        nan = np.flatnonzero(np.isnan(v))
        out.append(-1 if r < 0 else nan[0] if len(nan) else int(v.argmax()) if v.max() > -np.inf else -1)
    return np.array(out)


def accept(drafted, parents, picked, starts, lens, tokens):
    """(path, kept, token, lens)"""
    path, kept, token, out = np.full(tokens, -1), [], [], []
    for r in range(len(lens)):
        s0 = min(max(int(starts[r]), 0), tokens)
        past = int(starts[r + 1])
        n = min(max(past, s0), tokens) - s0
        way, last = [], -1
        if n and parents[s0] == -1:
            way = [0]
            while True:
                last = int(picked[s0 + way[-1]])
                to = [i for i in range(way[-1] + 1, n) if parents[s0 + i] == way[-1] and last >= 0 and drafted[s0 + i] == last]
                if not to:
                    break
                way.append(to[0])
        path[s0:s0 + len(way)] = way
        kept.append(len(way))
        token.append(last)
        out.append(int(lens[r]) - (past - s0) + len(way))
    return path, np.array(kept, int), np.array(token, int), np.array(out, int)


def move(arrays, table, starts, lens, path, kept, page):
    """The accepted rows of [pages, 2, kv heads, page, bytes] arrays moved up, in place."""
    n_pages = arrays[0].shape[0]
    for r in range(len(lens)):
        base = int(lens[r]) - (int(starts[r + 1]) - int(starts[r]))

        def place(p):
            pg = table[r, p // page] if 0 <= p and p // page < table.shape[1] else -1
            return (pg, p % page) if 0 <= pg < n_pages else None
        for j in range(kept[r]):
            a, b = place(base + int(path[int(starts[r]) + j])), place(base + j)
            if a and b:
                for x in arrays:
                    x[b[0], :, :, b[1]] = x[a[0], :, :, a[1]]


def trim(before, lens, table, ring, pool, page):
    ring, given = ring.copy(), int(pool[1])
    for r in range(len(lens)):
        for c in range(-(-int(lens[r]) // page), min(-(-int(before[r]) // page), table.shape[1])):
            if table[r, c] >= 0:
                ring[given % len(ring)] = table[r, c]
                given += 1
    return ring, [int(pool[0]), given]


def random_tree(n, rng, chain=False):
    return [-1] + [i - 1 if chain else int(i * rng.random() ** 1.5) for i in range(1, n)]

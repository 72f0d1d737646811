"""Plain restatements of the serving operators (CPU, 64 bits where values are
computed), for the tests."""
import math

import numpy as np
import torch

MAG = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6])


def page_tables(cached, fresh, table, ring, pool, page, most):
    table = table.copy()
    width = table.shape[1]
    starts, lens, slots, positions = [0], [], [], []
    taken, given = int(pool[0]), int(pool[1])
    lack = beyond = 0
    for r in range(len(cached)):
        c, f = max(int(cached[r]), 0), max(int(fresh[r]), 0)
        have, need = -(-c // page), -(-(c + f) // page)
        beyond += max(need - width, 0)
        for col in range(min(have, width), min(need, width)):
            if taken < given:
                table[r, col] = ring[taken % len(ring)]
                taken += 1
            else:
                table[r, col] = -1
                lack += 1
        for i in range(f):
            x = c + i
            pg = table[r, x // page] if x // page < width else -1
            slots.append(int(pg) * page + x % page if pg >= 0 else -1)
            positions.append(x)
        starts.append(starts[-1] + f)
        lens.append(c + f)
    over = max(len(slots) - most, 0)
    slots = (slots + [-1] * most)[:most]
    positions = (positions + [-1] * most)[:most]
    return dict(table=table, starts=np.array(starts), lens=np.array(lens), slots=np.array(slots),
                positions=np.array(positions), pool=np.array([taken, given]), status=np.array([lack, over, beyond]))


def turn(x, cos, sin, positions, layout, sign=1.0):
    """x [T, H, D] (numpy float64 or float32: products and sums in that type)."""
    x = np.array(x)
    half = cos.shape[1]
    i = np.arange(half)
    a, b = (i, i + half) if layout == "half" else (2 * i, 2 * i + 1)
    c = cos[positions][:, None, :].astype(x.dtype)
    s = (sign * sin[positions][:, None, :]).astype(x.dtype)
    out = x.copy()
    out[..., a] = x[..., a] * c - x[..., b] * s
    out[..., b] = x[..., b] * c + x[..., a] * s
    return out


def scale_of(byte):
    e, m = byte >> 3, byte & 7
    return m * 2.0 ** -17 if e == 0 else 2.0 ** (e - 15) * (1 + m / 8)


SCALES = np.array([scale_of(b) for b in range(0xF8)])


def quantise(x):
    """x float32 [..., D] -> (codes uint8 [..., D/2], scale bytes [..., D/32]); every decision exact."""
    g = np.asarray(x, np.float32).reshape(*x.shape[:-1], -1, 32)
    amax = np.abs(g).max(-1)
    fine = np.isfinite(g).all(-1)
    want = np.minimum(np.where(fine, amax, 0).astype(np.float32) / np.float32(6), np.float32(10240)).astype(np.float16)
    want = want.astype(np.float64)
    # nearest on the byte's grid, ties to the even byte
    up = np.searchsorted(SCALES, want)
    lo = np.maximum(up - 1, 0)
    d_up, d_lo = SCALES[up] - want, want - SCALES[lo]
    byte = np.where((d_up < d_lo) | ((d_up == d_lo) & (up % 2 == 0)), up, lo)
    byte = np.where(want == 0, 0, byte)
    sc = SCALES[byte][..., None]
    with np.errstate(invalid="ignore"):
        a = np.abs(g.astype(np.float64))
        mids = (MAG[1:] + MAG[:-1]) / 2
        mag = sum((a >= m * sc).astype(int) for m in mids)
    mag = np.where((sc > 0) & fine[..., None], mag, 0)
    code = np.where((g < 0) & (mag > 0), mag + 8, mag).reshape(x.shape)
    byte = np.where(fine, byte, 0xFF)
    return (code[..., 0::2] | (code[..., 1::2] << 4)).astype(np.uint8), byte.astype(np.uint8)


def values(codes, scales):
    """float64 [..., D] of codes [..., D/2] and scale bytes [..., D/32]."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1).astype(int)
    v = MAG[c & 7] * np.where(c & 8, -1.0, 1.0)
    sc = np.array([scale_of(b) if b < 0xF8 else np.nan for b in range(256)])[scales]
    return v * np.repeat(sc, 32, -1)


def attention(q, codes, scales, table, lens, starts, scale, window, tokens):
    """(out, lse, spread, logit size, total) in float64; spread = sum p |v| /
    sum p, total = sum |v| over the keys seen, logit size = the largest scale * sum |q k| a row sees (for error bounds)."""
    q = q.double().cpu().numpy()
    t, h, d = q.shape
    n_pages, _, hk, page, _ = codes.shape
    codes, scales, table = codes.cpu().numpy(), scales.cpu().numpy(), table.cpu().numpy()
    out, lse = np.zeros((t, h, d)), np.full((t, h), -np.inf)
    spread, size, total = np.zeros((t, h, d)), np.zeros((t, h)), np.zeros((t, h, d))
    for r in range(len(lens)):
        n = starts[r + 1] - starts[r]
        length = min(int(lens[r]), table.shape[1] * page)
        if length <= 0:
            continue
        cols = -(-length // page)
        pages = table[r, :cols]
        there = (pages >= 0) & (pages < n_pages)
        pg = np.where(there, pages, 0)
        seen_page = np.repeat(there, page)[:length]
        for g in range(hk):
            k = values(codes[pg, 0, g], scales[pg, 0, g]).reshape(-1, d)[:length]
            v = values(codes[pg, 1, g], scales[pg, 1, g]).reshape(-1, d)[:length]
            for i in range(n):
                pos = int(lens[r]) - n + i
                row = starts[r] + i
                seen = seen_page & (np.arange(length) <= pos)
                if window:
                    seen &= np.arange(length) > pos - window
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


def random_cache(n_pages, hk, page, d, gen, device="cuda"):
    """Codes as the append writes them (no code 8) and scales around 1/3."""
    nib = torch.randint(0, 15, (n_pages, 2, hk, page, d), generator=gen, device=device, dtype=torch.int32)
    nib = torch.where(nib >= 8, nib + 1, nib)
    codes = (nib[..., 0::2] | (nib[..., 1::2] << 4)).to(torch.uint8)
    scales = torch.randint(95, 120, (n_pages, 2, hk, page, d // 32), generator=gen, device=device,
                           dtype=torch.int32).to(torch.uint8)
    return codes, scales

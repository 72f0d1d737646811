"""The serving operators' measured cases: page tables, rotary positions, the
4-bit key/value cache's append and the attention that reads that cache.

Every case runs either in a plain form (elementary torch operations in 32
bits, rounded once at the end) or, with ``own``, through
``sili__new_b200.serving``.  ``exact`` restates the operators in 64 bits.

The cache format both forms share: a head vector is cut into groups of 32
along the head; a group holds 4-bit e2m1 codes (element 2i in the low nibble
of byte i) and one scale byte, the upper eight bits below the sign of an IEEE
half (5 exponent, 3 mantissa bits).  codes [pages, 2, kv heads, page, dim/2],
scales [pages, 2, kv heads, page, dim/32]; index 0 of the second axis is K.
"""
import math

import torch

own = False

GROUP = 32
SCALE_MOST = 10240.0        # largest scale: 6 * 10240 still fits a half
GOLDEN = 0.6180339887498949
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# (query heads, kv heads, head dimension) of drawn cases: grouped, one kv head a query head, one kv head in all
HEADS = ((32, 8, 128), (32, 8, 128), (40, 8, 128), (14, 14, 64), (28, 4, 128), (8, 1, 256), (16, 1, 128), (6, 2, 256),
         (32, 4, 64), (4, 4, 128))
# e2m1 magnitudes and the points from which the next one is taken (midpoints go up)
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
THRESHOLDS = (0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0)


def listed():
    return [
        # one decode step of a modest batch: pages and slots for one token per request
        dict(name="tables_decode", op="tables", requests=64, most=4096, chunk=1, one_in=1, page=16),
        # a large mixed step: most requests decode, some bring a prompt chunk, some idle
        dict(name="tables_mixed", op="tables", requests=1531, most=32768, chunk=700, one_in=16, page=64),
        # queries and keys of one decode step, half layout
        dict(name="rotary_decode", op="rotary", tokens=64, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             dtype="bfloat16", train=False, positions=32768, factor=1.0),
        # a training step's forward and gradient, the stack's own fp32, part of the head rotated, pairs interleaved
        dict(name="rotary_train", op="rotary", tokens=8191, heads=32, kv_heads=8, dim=128, rot=64,
             layout="interleaved", dtype="float32", train=True, positions=8192, factor=1.0),
        # one decode step's keys and values into the cache, fp32 activations
        dict(name="append_decode", op="append", tokens=33, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             dtype="float32", page=16, positions=32768, factor=1.0),
        # a long prompt's chunk, positions stretched past the trained context
        dict(name="append_prompt", op="append", tokens=16384, heads=32, kv_heads=8, dim=128, rot=128, layout="half",
             dtype="bfloat16", page=64, positions=131072, factor=4.0),
        # a few short conversations: latency
        dict(name="attend_few", op="attend", requests=4, new=1, least=33, most=700, heads=32, kv_heads=8, dim=128,
             page=16, dtype="bfloat16", window=0),
        # an ordinary decode batch of the folded stack (fp32 activations), ragged lengths
        dict(name="attend_batch_fp32", op="attend", requests=64, new=1, least=1, most=8192, heads=32, kv_heads=8,
             dim=128, page=16, dtype="float32", window=0),
        # a large decode batch in 16 bits
        dict(name="attend_batch", op="attend", requests=96, new=1, least=2048, most=16384, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bfloat16", window=0),
        # one very long document: one request fills the card
        dict(name="attend_long", op="attend", requests=1, new=1, least=262143, most=262143, heads=32, kv_heads=8,
             dim=128, page=64, dtype="float16", window=0),
        # prompt chunks over what is already cached
        dict(name="attend_prompt", op="attend", requests=3, new=2048, least=4000, most=7000, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bfloat16", window=0),
        # short chunks with a sliding window, fp32 activations
        dict(name="attend_window", op="attend", requests=5, new=250, least=600, most=5000, heads=32, kv_heads=8,
             dim=128, page=32, dtype="float32", window=1024),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["tables", "rotary", "append", "attend", "attend"])
        heads, kv_heads, dim = rng.choice(HEADS)
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        page = rng.choice([16, 32, 48, 64, 128])
        layout = rng.choice(["half", "interleaved"])
        rot = rng.choice([dim, dim // 2, dim // 4])
        factor = rng.choice([1.0, 1.0, 8.0])
        if op == "tables":
            case = dict(op=op, requests=_log_int(rng, 1, 3000), most=_log_int(rng, 64, 40000),
                        chunk=_log_int(rng, 1, 1000), one_in=rng.choice([1, 3, 16]), page=page)
        elif op == "rotary":
            case = dict(op=op, tokens=_log_int(rng, 1, 8000), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                        layout=layout, dtype=dtype, train=rng.random() < 0.5, positions=_log_int(rng, 512, 131072),
                        factor=factor)
        elif op == "append":
            case = dict(op=op, tokens=_log_int(rng, 1, 16000), heads=heads, kv_heads=kv_heads, dim=dim, rot=rot,
                        layout=layout, dtype=dtype, page=page, positions=_log_int(rng, 512, 131072), factor=factor)
        else:
            new = 1 if rng.random() < 0.6 else _log_int(rng, 2, 2000)
            most = max(new, _log_int(rng, 64, 200000 if new == 1 else 12000))
            case = dict(op=op, requests=_log_int(rng, 1, 128 if new == 1 else 8), new=new,
                        least=max(1, int(most * rng.choice([0.05, 0.5, 1.0]))), most=most, heads=heads,
                        kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                        window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]))
        if _padded_cost(case) <= 1.0:
            return case


def _padded_cost(case):
    """A case's size against the largest listed ones of its kind (the plain form pads ragged batches)."""
    if case["op"] == "tables":
        total, width = _table_totals(case)
        return max(total / 80000.0, case["requests"] * width / 1000000.0)
    if case["op"] in ("rotary", "append"):
        values = case["tokens"] * (case["heads"] + 2 * case["kv_heads"]) * case["dim"]
        return values / (16384 * 48 * 128)
    r, n, most = case["requests"], case["new"], case["most"]
    cache = r * most * case["kv_heads"] * case["dim"] / (96 * 16384 * 8 * 128)
    scores = r * n * case["heads"] * most / (3 * 2048 * 32 * 7000)
    return max(cache, scores * case["dim"] / 128)


# ── lengths: fixed by the case, handed out in an order that the seed shuffles ──
def _spread(n, lo, hi):
    return [lo + int((hi - lo) * ((i + 1) * GOLDEN % 1.0) + 0.5) if n > 1 else hi for i in range(n)]


def _table_lens(case):
    """(cached, new) per request; one in seven of the decoding requests idles this step."""
    r, most = case["requests"], case["most"]
    cached = _spread(r, 0, most)
    new = [case["chunk"] if i % case["one_in"] == 0 else (0 if i % 7 == 3 else 1) for i in range(r)]
    return cached, new


def _table_totals(case):
    cached, new = _table_lens(case)
    total = sum(new)
    width = max((c + n + case["page"] - 1) // case["page"] for c, n in zip(cached, new)) + 3
    return -(-(total + 5) // 64) * 64, width


def _attend_lens(case):
    """(length with the new tokens, new tokens) per request."""
    lens = _spread(case["requests"], case["least"], case["most"])
    n = case["new"]
    new = [max(1, n - (i * 37) % max(1, n // 2)) if n > 1 else 1 for i in range(case["requests"])]
    return [max(l, q) for l, q in zip(lens, new)], new


def _table(case, device):
    """cos, sin [positions, rot/2]: angles in 64 bits; stretched by `factor` where it is over 1."""
    half = case["rot"] // 2
    inv = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=device) * 2.0 / case["rot"])
    if case["factor"] > 1.0:
        # slow pairs interpolated, fast ones kept, a ramp between (by wavelength against an 8192 context)
        turns = 8192.0 * inv / (2.0 * math.pi)
        keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
        inv = inv * keep + inv / case["factor"] * (1.0 - keep)
    ang = torch.arange(case["positions"], dtype=torch.float64, device=device)[:, None] * inv[None, :]
    return ang.cos().float(), ang.sin().float()


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    s = {"case": case}

    def shuffled(values, dtype=torch.int32):
        return torch.tensor(values, dtype=dtype)

    if case["op"] == "tables":
        cached, new = _table_lens(case)
        total, width = _table_totals(case)
        order = torch.randperm(len(cached), generator=host)
        cached, new = shuffled(cached)[order], shuffled(new)[order]
        have = (cached.long() + case["page"] - 1) // case["page"]
        need = int(((cached.long() + new + case["page"] - 1) // case["page"] - have).sum())
        n_have = int(have.sum())
        n_pages = n_have + need + 11
        perm = torch.randperm(n_pages, generator=gen, device=dev).int()
        table = torch.full((len(cached), width), -1, dtype=torch.int32, device=dev)
        filled = torch.arange(width, device=dev)[None, :] < have.to(dev)[:, None]
        table[filled] = perm[:n_have]
        # the ring of free pages, somewhere in its life: `taken` pages have left it, `given` have come in
        ring = torch.full((n_pages,), -1, dtype=torch.int32, device=dev)
        taken = n_pages * 3 + int(torch.randint(0, n_pages, (1,), generator=host))
        at = (taken + torch.arange(n_pages - n_have, device=dev)) % n_pages
        ring[at] = perm[n_have:]
        s.update(cached=cached.to(dev), new=new.to(dev), table=table, ring=ring, page=case["page"],
                 pool=torch.tensor([taken, taken + n_pages - n_have], dtype=torch.int64, device=dev), most=total)
        return s

    dt = DTYPES[case["dtype"]]
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rotary", "append"):
        t = case["tokens"]
        # q, k, v as they leave one projection: slices of one row
        qkv = torch.randn(t, (h + 2 * hk) * d, generator=gen, device=dev)
        # a few channels of K are much larger than the others, as in trained models
        loud = torch.randint(0, d, (3,), generator=gen, device=dev)
        qkv.view(t, h + 2 * hk, d)[:, h:h + hk, loud] *= 8.0
        qkv = qkv.to(dt)
        s["q"] = qkv[:, : h * d].view(t, h, d)
        s["k"] = qkv[:, h * d:(h + hk) * d].view(t, hk, d)
        s["v"] = qkv[:, (h + hk) * d:].view(t, hk, d)
        s["positions"] = torch.randint(0, case["positions"], (t,), generator=gen, device=dev, dtype=torch.int32)
        s["cos"], s["sin"] = _table(case, dev)
        if case["op"] == "rotary" and case["train"]:
            s["dq"] = torch.randn(t, h, d, generator=gen, device=dev).to(dt)
            s["dk"] = torch.randn(t, hk, d, generator=gen, device=dev).to(dt)
        if case["op"] == "append":
            n_pages = -(-t * 3 // (2 * case["page"])) + 1
            slots = torch.randperm(n_pages * case["page"], generator=gen, device=dev)[:t]
            slots[torch.rand(t, generator=gen, device=dev) < 0.02] = -1      # padding of a fixed-size batch
            s["slots"] = slots
            s["codes"] = torch.zeros(n_pages, 2, hk, case["page"], d // 2, dtype=torch.uint8, device=dev)
            s["scales"] = torch.zeros(n_pages, 2, hk, case["page"], d // GROUP, dtype=torch.uint8, device=dev)
        return s

    lens, new = _attend_lens(case)
    order = torch.randperm(len(lens), generator=host)
    lens, new = shuffled(lens)[order], shuffled(new)[order]
    page = case["page"]
    used = (lens.long() + page - 1) // page
    width, n_used = int(used.max()), int(used.sum())
    n_pages = n_used + 2
    table = torch.zeros(len(lens), width, dtype=torch.int32, device=dev)
    filled = torch.arange(width, device=dev)[None, :] < used.to(dev)[:, None]
    table[filled] = torch.randperm(n_pages, generator=gen, device=dev).int()[:n_used]
    # codes distributed as quantised normal groups: 256 quantiles of the nibble, two draws a byte
    quant = torch.special.ndtri((torch.arange(256, dtype=torch.float64, device=dev) + 0.5) / 256).float() * (6.0 / 2.2)
    nib = _codes_of(quant, torch.ones_like(quant))
    both = (nib[None, :] | (nib[:, None] << 4)).to(torch.uint8).reshape(-1)
    codes = torch.empty(n_pages, 2, case["kv_heads"], page, d // 2, dtype=torch.uint8, device=dev)
    flat = codes.view(-1)
    for a in range(0, flat.numel(), 1 << 27):
        part = flat[a:a + (1 << 27)]
        part.copy_(both[torch.randint(0, 65536, part.shape, generator=gen, device=dev, dtype=torch.int32)])
    spread = torch.randn(n_pages, 2, case["kv_heads"], page, d // GROUP, generator=gen, device=dev)
    scales = _scale_bytes((spread * 0.3).exp() * 2.2)
    total = int(new.sum())
    s.update(codes=codes, scales=scales, table=table, lens=lens.to(dev), most_new=int(new.max()),
             q=(torch.randn(total, h, d, generator=gen, device=dev) * 1.5).to(dt), window=case["window"])
    starts = torch.zeros(len(lens) + 1, dtype=torch.int32)
    starts[1:] = torch.cumsum(new, 0)
    s["starts"] = None if case["new"] == 1 else starts.to(dev)
    return s


# ── the format, in elementary operations ─────────────────────────────────────
def _codes_of(x, scale):
    """e2m1 codes of x against its groups' scales: nearest, midpoints up in magnitude, at most 6, no negative zero.
    A threshold times a scale is exact in 32 bits (3 and 4 bits long), so no quotient decides; 0 under no scale."""
    a = x.abs()
    mag = sum((a >= t * scale).int() for t in THRESHOLDS)
    mag = torch.where(scale > 0, mag, torch.zeros_like(mag))
    return torch.where((x < 0) & (mag > 0), mag + 8, mag)


def _scale_bytes(amax):
    """Scale bytes of group maxima: amax / 6 as a half, its mantissa rounded to three bits (ties to even)."""
    six = torch.full_like(amax, 6.0)
    h = torch.clamp(amax / six, max=SCALE_MOST).to(torch.float16).view(torch.int16).int()
    b = (h + 0x3F + ((h >> 7) & 1)) >> 7
    return torch.where(torch.isfinite(amax), b, torch.full_like(b, 0xFF)).to(torch.uint8)


def _scales_of(b):
    return (b.int() << 7).to(torch.int16).view(torch.float16).float()


def _quantise(x):
    """x [..., dim] in 32 bits -> codes [..., dim/2], scale bytes [..., dim/32]."""
    g = x.view(*x.shape[:-1], -1, GROUP)
    b = _scale_bytes(g.abs().amax(-1))
    c = _codes_of(g, _scales_of(b)[..., None]).view(x.shape)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), b


def _values(codes, scale_bytes):
    """The values in 32 bits that codes [..., dim/2] and scale bytes [..., dim/32] stand for."""
    signed = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    byte = torch.arange(256, device=codes.device)
    pairs = torch.stack([signed[byte & 15], signed[byte >> 4]], -1)
    v = pairs[codes.int()].view(*codes.shape[:-1], -1, GROUP)
    return (v * _scales_of(scale_bytes)[..., None]).view(*codes.shape[:-1], -1)


# ── plain forms ──────────────────────────────────────────────────────────────
def _plain_tables(s):
    cached, new, ps = s["cached"].clamp(min=0).long(), s["new"].clamp(min=0).long(), s["page"]
    table, ring, pool = s["table"], s["ring"], s["pool"]
    width, cap = table.shape[1], ring.shape[0]
    lens = cached + new
    have = ((cached + ps - 1) // ps).clamp(max=width)
    need = ((lens + ps - 1) // ps).clamp(max=width)
    want = need - have
    first = torch.cumsum(want, 0) - want
    left = pool[1] - pool[0]
    col = torch.arange(width, device=table.device)
    j = first[:, None] + col[None, :] - have[:, None]
    fresh = (col[None, :] >= have[:, None]) & (col[None, :] < need[:, None])
    page = torch.where(j < left, ring[((pool[0] + j) % cap)], torch.full_like(table, -1))
    table = torch.where(fresh, page, table)
    starts = torch.zeros(len(new) + 1, dtype=torch.int64, device=table.device)
    starts[1:] = torch.cumsum(new, 0)
    i = torch.arange(s["most"], device=table.device)
    req = torch.searchsorted(starts[1:], i, right=True)
    real = req < len(new)
    rc = req.clamp(max=len(new) - 1)
    pos = cached[rc] + i - starts[rc]
    c = pos // ps
    pg = table[rc, c.clamp(max=width - 1)].long()
    ok = real & (c < width) & (pg >= 0)
    slots = torch.where(ok, pg * ps + pos % ps, torch.full_like(pos, -1))
    positions = torch.where(real, pos, torch.full_like(pos, -1)).int()
    asked = want.sum()
    got = torch.minimum(asked, left)
    status = torch.stack([asked - got, (starts[-1] - s["most"]).clamp(min=0),
                          ((lens + ps - 1) // ps - need).sum()])
    return {"table": table, "starts": starts.int(), "lens": lens.int(), "slots": slots, "positions": positions,
            "pool": torch.stack([pool[0] + got, pool[1]]), "status": status}


def _turned(x, cos, sin, layout, sign):
    """x [T, heads, dim] in 32 bits, its first 2 * cos.shape[-1] elements rotated by the tokens' angles."""
    half = cos.shape[-1]
    rot, rest = x[..., : 2 * half], x[..., 2 * half:]
    a, b = (rot[..., :half], rot[..., half:]) if layout == "half" else (rot[..., 0::2], rot[..., 1::2])
    c, n = cos[:, None, :], sin[:, None, :] * sign
    ra, rb = a * c - b * n, b * c + a * n
    if layout == "half":
        return torch.cat([ra, rb, rest], -1)
    return torch.cat([torch.stack([ra, rb], -1).flatten(-2), rest], -1)


def _plain_rotary(s):
    layout = s["case"]["layout"]
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    out = {n: _turned(s[n].float(), cos, sin, layout, 1.0).to(s[n].dtype) for n in ("q", "k")}
    if s["case"]["train"]:
        out.update({n: _turned(s[n].float(), cos, sin, layout, -1.0).to(s[n].dtype) for n in ("dq", "dk")})
    return out


def _plain_append(s):
    layout = s["case"]["layout"]
    cos, sin = s["cos"][s["positions"].long()], s["sin"][s["positions"].long()]
    k = _turned(s["k"].float(), cos, sin, layout, 1.0)
    codes, scales = s["codes"], s["scales"]
    n_pages, _, _, page, _ = codes.shape
    real = s["slots"] >= 0
    # a padding token's row goes to a spare page's worth of scratch behind the cache
    at = torch.where(real, s["slots"], torch.full_like(s["slots"], n_pages * page))
    spare = torch.cat([codes, codes.new_zeros(1, *codes.shape[1:])]), torch.cat([scales, scales.new_zeros(1, *scales.shape[1:])])
    pg, off = at // page, at % page
    for w, x in ((0, k), (1, s["v"].float())):
        c, b = _quantise(x)
        spare[0][pg, w, :, off] = c
        spare[1][pg, w, :, off] = b
    codes.copy_(spare[0][:n_pages])
    scales.copy_(spare[1][:n_pages])
    kv = [_values(codes[(at // page).clamp(max=n_pages - 1), w, :, off],
                  scales[(at // page).clamp(max=n_pages - 1), w, :, off]) for w in (0, 1)]
    kv = [torch.where(real[:, None, None], x, torch.zeros_like(x)).to(s["k"].dtype) for x in kv]
    return {"q": _turned(s["q"].float(), cos, sin, layout, 1.0).to(s["q"].dtype), "k": kv[0], "v": kv[1]}


def _plain_attend(s):
    q, table, lens, window = s["q"], s["table"].long(), s["lens"].long(), s["window"]
    t, h, d = q.shape
    r, hk = table.shape[0], s["codes"].shape[2]
    n = s["most_new"]
    starts = s["starts"].long() if s["starts"] is not None else torch.arange(r + 1, device=q.device)
    cnt = starts[1:] - starts[:-1]
    # [r, n] padded queries, [r, hk, group * n, d]
    i = torch.arange(n, device=q.device)[None, :]
    real = i < cnt[:, None]
    row = (starts[:-1, None] + i).clamp(max=t - 1)
    qp = q[row].float().view(r, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(r, hk, -1, d)
    kk = _values(s["codes"][table, 0], s["scales"][table, 0]).permute(0, 2, 1, 3, 4).reshape(r, hk, -1, d)
    x = (qp @ kk.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del kk
    pos = (lens - cnt)[:, None] + i
    key = torch.arange(x.shape[-1], device=q.device)
    seen = (key[None, None, :] <= pos[..., None]) & (key[None, None, :] < lens[:, None, None]) & real[..., None]
    if window:
        seen &= key[None, None, :] > pos[..., None] - window
    x = x.view(r, hk, h // hk, n, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    x = x.sub_(top).exp_()
    total = x.sum(-1, keepdim=True)
    vv = _values(s["codes"][table, 1], s["scales"][table, 1]).permute(0, 2, 1, 3, 4).reshape(r, hk, -1, d)
    o = (x.view(r, hk, -1, x.shape[-1]) @ vv).view(r, hk, h // hk, n, d)
    o = torch.where(total > 0, o / total, torch.zeros_like(o))
    lse = (top + total.log()).squeeze(-1)
    back = torch.arange(t, device=q.device)
    req = torch.searchsorted(starts[1:].contiguous(), back, right=True)
    at = back - starts[req]
    o = o.permute(0, 3, 1, 2, 4).reshape(r, n, h, d)[req, at].to(q.dtype)
    return {"out": o, "lse": lse.permute(0, 3, 1, 2).reshape(r, n, h)[req, at]}


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"tables": _plain_tables, "rotary": _plain_rotary, "append": _plain_append,
                "attend": _plain_attend}[op](s)
    from sili__new_b200 import serving
    if op == "tables":
        p = serving.page_tables(s["cached"], s["new"], s["table"], s["ring"], s["pool"], s["page"], s["most"])
        return {"table": s["table"], "starts": p.starts, "lens": p.lens, "slots": p.slots, "positions": p.positions,
                "pool": p.pool, "status": p.status}
    layout = s["case"].get("layout")
    if op == "rotary":
        q, k = serving.rotary(s["q"], s["k"], s["cos"], s["sin"], s["positions"], layout=layout)
        if not s["case"]["train"]:
            return {"q": q, "k": k}
        dq, dk = serving.rotary_backward(s["dq"], s["dk"], s["cos"], s["sin"], s["positions"], layout=layout)
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if op == "append":
        q = serving.cache_append(s["k"], s["v"], s["codes"], s["scales"], s["slots"], cos=s["cos"], sin=s["sin"],
                                 positions=s["positions"], layout=layout, q=s["q"])
        k, v = serving.cache_read(s["codes"], s["scales"], s["slots"], dtype=s["k"].dtype)
        return {"q": q, "k": k, "v": v}
    out, lse = serving.cache_attention(s["q"], s["codes"], s["scales"], s["table"], s["lens"], starts=s["starts"],
                                       most_new=s["most_new"], window=s["window"], return_lse=True)
    return {"out": out, "lse": lse}


def work(case):
    if case["op"] == "tables":
        cached, new = _table_lens(case)
        total, _ = _table_totals(case)
        r, page = case["requests"], case["page"]
        fresh = sum((c + n + page - 1) // page - (c + page - 1) // page for c, n in zip(cached, new))
        last = sum(1 for c, n in zip(cached, new) if n and c % page)
        # lengths in, starts and lengths out, a slot and a position a token, ring entry in and table entry out a page
        return {"bytes": 16 * r + 12 * total + 8 * fresh + 4 * last, "flops": 0}
    item = 4 if case["dtype"] == "float32" else 2
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] in ("rotary", "append"):
        t = case["tokens"]
        angles = t * (case["rot"] * 4 + 4)
        turns = 3 * t * case["rot"]
        if case["op"] == "rotary":
            times = 2 if case["train"] else 1
            return {"bytes": times * 2 * t * (h + hk) * d * item + angles, "flops": times * turns * (h + hk)}
        packed = 2 * t * hk * (d // 2 + d // GROUP)
        # q in and out, k and v in, the cache's bytes written, then read, and the values out
        return {"bytes": t * (2 * h + 2 * hk) * d * item + angles + 8 * t + 2 * packed + 2 * t * hk * d * item,
                "flops": turns * (h + hk) + 4 * t * hk * d}
    lens, new = _attend_lens(case)
    window, byts, flops = case["window"], 0, 0
    for l, n in zip(lens, new):
        seen = l if not window else min(l, n - 1 + window)
        byts += seen * hk * 2 * (d // 2 + d // GROUP) + 4 * (-(-seen // case["page"])) + 4
        if window:
            pairs = sum(min(p + 1, window) for p in range(l - n, l))
        else:
            pairs = n * (l - n) + n * (n + 1) // 2
        flops += 4 * pairs * h * d
    byts += sum(new) * h * (2 * d * item + 4)
    return {"bytes": byts, "flops": flops}


# ── the operators' definitions in 64 bits ────────────────────────────────────
def _exact_values(codes, scale_bytes):
    """Bytes -> doubles by the fields' meaning: sign, exponent (bias 1), one mantissa bit; scale bias 15, three bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).double()
    neg, m = (c >= 8).double(), c % 8
    e, f = torch.floor(m / 2), m % 2
    v = torch.where(e == 0, f * 0.5, torch.pow(2.0, e - 1) * (1 + f / 2)) * (1 - 2 * neg)
    b = scale_bytes.double()
    e, f = torch.floor(b / 8), b % 8
    sc = torch.where(e == 0, f * 2.0 ** -17, torch.pow(2.0, e - 15) * (1 + f / 8))
    return v * sc.repeat_interleave(GROUP, -1)


def _exact_rounded(x):
    """The nearest values that the cache can hold, decided in 64 bits."""
    g = x.reshape(*x.shape[:-1], -1, GROUP)
    want = (g.abs().amax(-1) / 6.0).clamp(max=SCALE_MOST)
    want = want.to(torch.float16).double()
    normal = want.clamp(min=2.0 ** -14)
    quantum = normal / torch.frexp(normal).mantissa / 16     # an exact power of two: four bits are kept
    sc = (torch.round(want / quantum) * quantum)[..., None]
    grid = torch.tensor(MAGNITUDES, dtype=torch.float64, device=x.device)
    y = torch.where(sc > 0, g / sc.clamp(min=2.0 ** -17), torch.zeros_like(g))
    mid = (grid[1:] + grid[:-1]) / 2
    near = grid[torch.bucketize(y.abs(), mid, right=True)]
    return (torch.sign(y) * near * sc).reshape(x.shape)


def _exact_turn(x, case, cos, sin, positions, sign):
    """Each pair as a complex number times e^(i angle); cos and sin are the operator's inputs."""
    half = case["rot"] // 2
    x = x.double()
    w = torch.complex(cos.double()[positions.long()], sign * sin.double()[positions.long()])[:, None, :]
    z = x.clone()
    first = torch.arange(half, device=x.device) * (1 if case["layout"] == "half" else 2)
    second = first + (half if case["layout"] == "half" else 1)
    turned = torch.complex(x[..., first], x[..., second]) * w
    z[..., first], z[..., second] = turned.real, turned.imag
    return z


def exact(case, seed):
    if case["op"] == "tables":
        return None
    s = prepare(case, seed)
    if case["op"] in ("rotary", "append"):
        turn = lambda n, sign: _exact_turn(s[n], case, s["cos"], s["sin"], s["positions"], sign)  # noqa: E731
        if case["op"] == "rotary":
            out = {"q": turn("q", 1.0), "k": turn("k", 1.0)}
            if case["train"]:
                out.update(dq=turn("dq", -1.0), dk=turn("dk", -1.0))
            return out
        real = (s["slots"] >= 0)[:, None, None].double()
        return {"q": turn("q", 1.0), "k": _exact_rounded(turn("k", 1.0)) * real,
                "v": _exact_rounded(s["v"].double()) * real}
    if work(case)["flops"] > 4e12:
        return None
    q = s["q"].double()
    t, h, d = q.shape
    hk, page = s["codes"].shape[2], s["codes"].shape[3]
    out = torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, h), float("-inf"), dtype=torch.float64, device=q.device)
    lens = s["lens"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(len(lens) + 1))
    for r, length in enumerate(lens):
        n = starts[r + 1] - starts[r]
        pages = s["table"][r, : -(-length // page)].long()
        key = torch.arange(length, device=q.device)[None, :]
        pos = torch.arange(length - n, length, device=q.device)[:, None]
        hidden = (key > pos) if not s["window"] else (key > pos) | (key <= pos - s["window"])
        for g in range(hk):
            k, v = (_exact_values(s["codes"][pages, w, g], s["scales"][pages, w, g]).reshape(-1, d)[:length] for w in (0, 1))
            for j in range(g * (h // hk), (g + 1) * (h // hk)):
                x = (q[starts[r]:starts[r + 1], j] @ k.T) / math.sqrt(d)
                x = x.masked_fill(hidden, float("-inf"))
                lse[starts[r]:starts[r + 1], j] = torch.logsumexp(x, -1)
                out[starts[r]:starts[r + 1], j] = torch.softmax(x, -1) @ v
    return {"out": out, "lse": lse}

"""The measured cases of decoding with drafted tokens: the tree of a step's
drafts, the attention of a tree over the 4-bit cache, penalties, biases and
grammar masks on the logits, the pick that follows them, and what becomes of
the accepted tokens (their way through the tree, their place in the caches,
the pages that the others held).

Every case runs either in a plain form (elementary torch operations in 32
bits, rounded once at the end) or, with ``own``, through
``sili__new_b200.serving``.  ``exact`` restates the computed values in 64 bits.

A request's drafted tokens are rows of one step, a row's parent before it:
``parents`` holds the parent's place among the request's rows, -1 for one that
follows the cached tokens.  Bit j of a row's mask (int64 words of 64) says that
it sees the request's row j: its ancestors and itself.  A row without a bit is
none: it sees nothing.  The rows' keys and values lie in the cache behind the
request's committed tokens, in the rows' order.

The cache's format: a head vector is cut into groups of 32 along the head; a
group holds 4-bit e2m1 codes (element 2i in the low nibble of byte i) and one
scale byte, the upper eight bits below the sign of an IEEE half.  codes [pages,
2, kv heads, page, dim/2], scales [pages, 2, kv heads, page, dim/32]; index 0 of
the second axis is K.
"""
import math
import random

import torch

own = False

GROUP = 32
GOLDEN = 0.6180339887498949
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
# (query heads, kv heads, head dimension) of drawn cases: grouped, one kv head a query head, one kv head in all
HEADS = ((32, 8, 128), (32, 8, 128), (40, 8, 128), (14, 14, 64), (28, 4, 128), (8, 1, 256), (16, 1, 128), (6, 2, 256),
         (32, 4, 64), (4, 4, 128))
VOCABS = (1000, 8191, 32000, 50021, 65536, 100003, 131072, 150001)
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
SPARE = 5            # rows behind the last request's: a step's fixed number of rows is seldom full


def listed():
    return [
        # the trees of one step of a few requests, one mask word
        dict(name="plan_few", op="plan", requests=4, drafts=8),
        # a large batch with wide trees, four mask words
        dict(name="plan_wide", op="plan", requests=192, drafts=250),
        # a few short conversations with small trees and a sliding window: latency
        dict(name="attend_few", op="attend", requests=4, drafts=8, least=33, most=700, heads=32, kv_heads=8, dim=128,
             page=16, dtype="bfloat16", window=256),
        # an ordinary batch of the folded stack (fp32 activations), ragged lengths, modest trees
        dict(name="attend_batch_fp32", op="attend", requests=24, drafts=16, least=1, most=8192, heads=32, kv_heads=8,
             dim=128, page=16, dtype="float32", window=0),
        # a large batch in 16 bits with full trees
        dict(name="attend_batch", op="attend", requests=40, drafts=64, least=2048, most=12288, heads=32, kv_heads=8,
             dim=128, page=64, dtype="bfloat16", window=0),
        # one long document: one request fills the card
        dict(name="attend_long", op="attend", requests=1, drafts=24, least=131071, most=131071, heads=32, kv_heads=8,
             dim=128, page=64, dtype="float16", window=0),
        # one decode step's logits of a few requests, to be sampled from
        dict(name="adjust_decode", op="adjust", requests=16, drafts=1, vocab=32000, dtype="float32", history=700,
             biases=16, masked=True),
        # the logits of a batch of trees: each row has its own path of drafted tokens behind the request's history
        dict(name="adjust_tree", op="adjust", requests=24, drafts=24, vocab=131072, dtype="bfloat16", history=4096,
             biases=300, masked=True),
        # a greedy decode step without a grammar, an odd vocabulary
        dict(name="pick_decode", op="pick", requests=64, drafts=1, vocab=50021, dtype="bfloat16", history=2000, biases=0,
             masked=False),
        # the greedy picks that decide over a batch of trees
        dict(name="pick_tree", op="pick", requests=32, drafts=32, vocab=131072, dtype="float32", history=8000, biases=64,
             masked=True),
        # the end of a small step: one layer's cache
        dict(name="settle_few", op="settle", requests=4, drafts=8, layers=1, least=33, most=700, kv_heads=8, dim=128,
             page=16),
        # the end of a large step: the accepted tokens move in the caches of several layers
        dict(name="settle_layers", op="settle", requests=96, drafts=64, layers=12, least=100, most=1500, kv_heads=8,
             dim=128, page=16),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["plan", "attend", "attend", "adjust", "pick", "settle"])
        heads, kv_heads, dim = rng.choice(HEADS)
        dtype = rng.choice(["float32", "bfloat16", "float16"])
        page = rng.choice([16, 32, 48, 64, 128])
        if op == "plan":
            case = dict(op=op, requests=_log_int(rng, 1, 256), drafts=_log_int(rng, 1, 256))
        elif op == "attend":
            drafts = _log_int(rng, 1, 130)
            most = _log_int(rng, 64, 130000)
            case = dict(op=op, requests=_log_int(rng, 1, 64), drafts=drafts, least=max(1, int(most * rng.choice([0.05, 0.5, 1.0]))),
                        most=most, heads=heads, kv_heads=kv_heads, dim=dim, page=page, dtype=dtype,
                        window=rng.choice([0, 0, 0, _log_int(rng, 16, 4096)]))
        elif op in ("adjust", "pick"):
            case = dict(op=op, requests=_log_int(rng, 1, 128), drafts=rng.choice([1, _log_int(rng, 2, 100)]),
                        vocab=rng.choice(VOCABS), dtype=dtype, history=_log_int(rng, 1, 16000),
                        biases=rng.choice([0, _log_int(rng, 1, 300)]), masked=rng.random() < 0.5)
        else:
            most = _log_int(rng, 40, 2000)
            case = dict(op=op, requests=_log_int(rng, 1, 128), drafts=_log_int(rng, 1, 250), layers=_log_int(rng, 1, 16),
                        least=max(1, most // 10), most=most, kv_heads=kv_heads, dim=dim, page=page)
        if _cost(case) <= 1.0:
            return case


def _cost(case):
    """A case's size against the largest listed ones of its kind (the plain forms pad ragged batches)."""
    op, r, n = case["op"], case["requests"], case["drafts"]
    if op == "plan":
        return r * n * n / (192 * 250 * 250)
    if op == "attend":
        cache = r * case["most"] * case["kv_heads"] * case["dim"] / (40 * 12288 * 8 * 128)
        scores = r * n * case["heads"] * case["most"] * case["dim"] / (40 * 64 * 32 * 12288 * 128)
        return max(cache, scores)
    if op in ("adjust", "pick"):
        return r * n * case["vocab"] / (32 * 32 * 131072)
    held = r * (case["most"] + n) * case["layers"] * case["kv_heads"] * case["dim"]
    return held / (96 * 1564 * 12 * 8 * 128)


# ── sizes and trees: fixed by the case, handed out in an order that the seed shuffles ──
def _spread(n, lo, hi):
    return [lo + int((hi - lo) * ((i + 1) * GOLDEN % 1.0) + 0.5) if n > 1 else hi for i in range(n)]


def _counts(case):
    """Drafted rows of each request: up to a half fewer than the case's."""
    n = case["drafts"]
    return [max(1, n - (i * 5) % max(1, n // 2)) for i in range(case["requests"])]


def _trees(case):
    """(parents of each request's rows, the way that is accepted in each, as rows)."""
    trees, ways = [], []
    for i, n in enumerate(_counts(case)):
        rng = random.Random(1000 * n + i)
        parents = [-1] + [int(k * rng.random() ** 1.5) for k in range(1, n)]
        way = [rng.randrange(n)]
        while parents[way[0]] >= 0:
            way.insert(0, parents[way[0]])
        trees.append(parents)
        ways.append(way)
    return trees, ways


def _ancestors(parents):
    seen = []
    for i, p in enumerate(parents):
        seen.append((seen[p] if p >= 0 else 0) | 1 << i)
    return seen


def _words(case):
    return -(-case["drafts"] // 64)


def _mask_tensor(seen, words, rows, device):
    flat = [(m >> 64 * w) & (1 << 64) - 1 for m in seen for w in range(words)]
    flat = [v - (1 << 64) if v >> 63 else v for v in flat] + [0] * ((rows - len(seen)) * words)
    return torch.tensor(flat, dtype=torch.int64).view(rows, words).to(device)


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    op, r = case["op"], case["requests"]
    s = {"case": case}
    trees, ways = _trees(case)
    order = torch.randperm(r, generator=host).tolist()
    trees, ways = [trees[i] for i in order], [ways[i] for i in order]
    new = torch.tensor([len(t) for t in trees])
    total = int(new.sum())
    single = op in ("adjust", "pick") and case["drafts"] == 1
    rows = total if single else total + SPARE
    starts = torch.zeros(r + 1, dtype=torch.int32)
    starts[1:] = torch.cumsum(new, 0)
    parents = torch.full((rows,), -1, dtype=torch.int32)
    parents[:total] = torch.tensor([p for t in trees for p in t], dtype=torch.int32)
    s.update(starts=None if single else starts.to(dev), parents=parents.to(dev), most_new=int(new.max()))
    if op in ("attend", "adjust", "pick"):
        s["masks"] = _mask_tensor([m for t in trees for m in _ancestors(t)], _words(case), rows, dev)

    if op in ("adjust", "pick"):
        vocab = case["vocab"]
        logits = torch.randn(rows, vocab, generator=gen, device=dev) * 2.5
        # tokens are not alike: a few are likely everywhere, and those are the ones that the history repeats
        logits += torch.randn(vocab, generator=gen, device=dev) * 1.5
        s["logits"] = logits.to(DTYPES[case["dtype"]])
        often = (torch.rand(r, case["history"], generator=gen, device=dev) ** 4 * vocab).int()
        s["history"] = often
        lens = torch.tensor(_spread(r, 0, case["history"]), dtype=torch.int32)[order].to(dev)
        s["history_lens"] = lens
        s["prompt_lens"] = (lens * torch.rand(r, generator=gen, device=dev)).int()
        s["drafted"] = (torch.rand(rows, generator=gen, device=dev) ** 4 * vocab).int()
        s["repetition"] = 1.0 + 0.5 * torch.rand(r, generator=gen, device=dev)
        s["frequency"] = 0.4 * torch.rand(r, generator=gen, device=dev)
        s["presence"] = 0.8 * torch.rand(r, generator=gen, device=dev) - 0.2
        s["temperature"] = 0.3 + torch.rand(r, generator=gen, device=dev)
        s["temperature"][0] = 0.0           # greedy: left as it is
        if case["biases"]:
            # different tokens in a list, a few places of it unused
            step = max(1, vocab // case["biases"])
            at = torch.arange(case["biases"], device=dev) * step % vocab
            s["bias_tokens"] = ((at + torch.randint(0, step, (r, 1), generator=gen, device=dev)) % vocab).int()
            s["bias_tokens"][torch.rand(r, case["biases"], generator=gen, device=dev) < 0.1] = -1
            s["bias_values"] = torch.randn(r, case["biases"], generator=gen, device=dev) * 4.0
        if case["masked"]:
            words = torch.randint(-2 ** 31, 2 ** 31, (rows, -(-vocab // 32)), generator=gen, device=dev, dtype=torch.int32)
            kind = torch.arange(rows, device=dev) % 4
            words[kind == 0] = -1                                            # no grammar: everything
            few = torch.rand(words.shape, generator=gen, device=dev) < 0.995
            words[(kind == 1)[:, None] & few] = 0                            # a narrow place of the grammar
            words[(torch.arange(rows, device=dev) % 16 == 7)] = 0            # a dead end: nothing
            s["allowed"] = words
        return s

    if op == "plan":
        s["lens"] = (torch.randint(0, 30000, (r,), generator=host) + new).int().to(dev)
        return s

    committed = torch.tensor(_spread(r, case["least"], case["most"]))[order]
    lens = committed + new
    page, hk, d = case["page"], case["kv_heads"], case["dim"]
    used = (lens + page - 1) // page
    width, n_used = int(used.max()) + 1, int(used.sum())
    n_pages = n_used + 3
    perm = torch.randperm(n_pages, generator=gen, device=dev).int()
    table = torch.full((r, width), -1, dtype=torch.int32, device=dev)
    filled = torch.arange(width, device=dev)[None, :] < used.to(dev)[:, None]
    table[filled] = perm[:n_used]
    s.update(table=table, lens=lens.int().to(dev), page=page)
    # codes distributed as quantised normal groups: 256 quantiles of the nibble, two draws a byte
    quant = torch.special.ndtri((torch.arange(256, dtype=torch.float64, device=dev) + 0.5) / 256).float() * (6.0 / 2.2)
    mag = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], device=dev)
    nib = torch.bucketize(quant.abs(), mag, right=True)
    nib = torch.where((quant < 0) & (nib > 0), nib + 8, nib)
    both = (nib[None, :] | (nib[:, None] << 4)).to(torch.uint8).reshape(-1)
    s["caches"] = []
    for _ in range(case.get("layers", 1)):
        codes = torch.empty(n_pages, 2, hk, page, d // 2, dtype=torch.uint8, device=dev)
        flat = codes.view(-1)
        for a in range(0, flat.numel(), 1 << 27):
            part = flat[a:a + (1 << 27)]
            part.copy_(both[torch.randint(0, 65536, part.shape, generator=gen, device=dev, dtype=torch.int32)])
        amax = (torch.randn(n_pages, 2, hk, page, d // GROUP, generator=gen, device=dev) * 0.3).exp() * 2.2
        half = (amax / 6.0).to(torch.float16).view(torch.int16).int()
        s["caches"].append((codes, ((half + 0x3F + ((half >> 7) & 1)) >> 7).to(torch.uint8)))
    if op == "attend":
        s["q"] = (torch.randn(rows, case["heads"], d, generator=gen, device=dev) * 1.5).to(DTYPES[case["dtype"]])
        s["window"] = case["window"]
        return s
    # settle: siblings hold different tokens; along the accepted way each pick is the next row's token
    drafted = torch.randint(0, 30000, (rows,), generator=host) * 512 + torch.arange(rows) % 512
    picked = torch.randint(0, 30000, (rows,), generator=host) * 512 + 511
    for k, way in enumerate(ways):
        for a, b in zip(way, way[1:]):
            picked[int(starts[k]) + a] = drafted[int(starts[k]) + b]
    s.update(drafted=drafted.int().to(dev), picked=picked.int().to(dev))
    ring = torch.full((n_pages,), -1, dtype=torch.int32, device=dev)
    taken = 3 * n_pages + int(torch.randint(0, n_pages, (1,), generator=host))
    ring[(taken + torch.arange(n_pages - n_used, device=dev)) % n_pages] = perm[n_used:]
    s.update(ring=ring, pool=torch.tensor([taken, taken + n_pages - n_used], dtype=torch.int64, device=dev))
    return s


# ── plain forms ──────────────────────────────────────────────────────────────
def _values(codes, scale_bytes):
    """The values in 32 bits that codes [..., dim/2] and scale bytes [..., dim/32] stand for."""
    signed = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=codes.device)
    byte = torch.arange(256, device=codes.device)
    pairs = torch.stack([signed[byte & 15], signed[byte >> 4]], -1)
    v = pairs[codes.int()].view(*codes.shape[:-1], -1, GROUP)
    scale = (scale_bytes.int() << 7).to(torch.int16).view(torch.float16).float()
    return (v * scale[..., None]).view(*codes.shape[:-1], -1)


def _rows_of(s, rows):
    """Of each row its request, its place in it and whether there is one."""
    if s["starts"] is None:
        i = torch.arange(rows, device=s["parents"].device)
        return i, torch.zeros_like(i), i >= 0
    starts = s["starts"].long()
    i = torch.arange(rows, device=starts.device)
    req = torch.searchsorted(starts[1:].contiguous(), i, right=True)
    real = req < len(starts) - 1
    req = req.clamp(max=len(starts) - 2)
    return req, i - starts[req], real


def _padded(s, x, n, fill):
    """x [rows] by request and place, [requests, n]."""
    starts = s["starts"].long()
    at = torch.arange(n, device=x.device)[None, :]
    real = at < (starts[1:] - starts[:-1])[:, None]
    return torch.where(real, x[(starts[:-1, None] + at).clamp(max=len(x) - 1)], torch.full_like(real, fill, dtype=x.dtype)), real


def _closure(parents, real):
    """[requests, n, n]: row i sees row j, from parents [requests, n]: powers of the parents' matrix by squaring."""
    n = parents.shape[1]
    step = ((parents[..., None] == torch.arange(n, device=parents.device)) & real[..., None]).float()
    seen = torch.eye(n, device=parents.device) * real[..., None] + step
    for _ in range(max(1, (n - 1).bit_length())):
        seen = (seen @ seen > 0).float()
    return seen > 0


def _packed(seen, words):
    """Bits [..., 64 * words or fewer] -> int64 [..., words]."""
    seen = torch.nn.functional.pad(seen.long(), (0, 64 * words - seen.shape[-1])).view(*seen.shape[:-1], words, 64)
    return (seen << torch.arange(64, device=seen.device)).sum(-1)


def _plain_plan(s):
    rows, n = len(s["parents"]), s["most_new"]
    parents, real = _padded(s, s["parents"], n, -1)
    seen = _closure(parents, real)
    req, at, there = _rows_of(s, rows)
    masks = _packed(seen, -(-n // 64))[req, at.clamp(max=n - 1)] * there[:, None]
    starts = s["starts"].long()
    base = s["lens"].long() - (starts[1:] - starts[:-1])
    place = base[req] + seen.sum(-1)[req, at.clamp(max=n - 1)] - 1
    return {"masks": masks, "positions": torch.where(there, place, torch.full_like(place, -1)).int()}


def _plain_attend(s):
    q, table, lens, window = s["q"], s["table"].long(), s["lens"].long(), s["window"]
    codes, scales = s["caches"][0]
    t, h, d = q.shape
    r, hk, n = table.shape[0], codes.shape[2], s["most_new"]
    starts = s["starts"].long()
    cnt = starts[1:] - starts[:-1]
    i = torch.arange(n, device=q.device)[None, :]
    row = (starts[:-1, None] + i).clamp(max=t - 1)
    qp = q[row].float().view(r, n, hk, h // hk, d).permute(0, 2, 3, 1, 4).reshape(r, hk, -1, d)
    pages = table.clamp(min=0)
    kk = _values(codes[pages, 0], scales[pages, 0]).permute(0, 2, 1, 3, 4).reshape(r, hk, -1, d)
    x = (qp @ kk.transpose(-1, -2)) * (1.0 / math.sqrt(d))
    del kk
    # the rows' own keys by their masks, [r, n, n], laid behind the committed ones
    bits = (s["masks"][..., None] >> torch.arange(64, device=q.device) & 1).flatten(-2)[row] * (i < cnt[:, None])[..., None]
    base = (lens - cnt)[:, None, None]
    key = torch.arange(x.shape[-1], device=q.device)[None, None, :]
    own_key = (key - base).clamp(0, bits.shape[-1] - 1).expand(-1, n, -1)
    some = bits.sum(-1, keepdim=True)
    before = (some > 0) & (key >= base + some - window) if window else some > 0
    seen = torch.where(key < base, before, (bits.gather(-1, own_key) > 0) & (key < base + cnt[:, None, None]))
    x = x.view(r, hk, h // hk, n, -1).masked_fill_(~seen[:, None, None], float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    x = x.sub_(top).exp_()
    whole = x.sum(-1, keepdim=True)
    vv = _values(codes[pages, 1], scales[pages, 1]).permute(0, 2, 1, 3, 4).reshape(r, hk, -1, d)
    o = (x.view(r, hk, -1, x.shape[-1]) @ vv).view(r, hk, h // hk, n, d)
    o = torch.where(whole > 0, o / whole, torch.zeros_like(o))
    lse = (top + whole.log()).squeeze(-1)
    req, at, real = _rows_of(s, t)
    at = at.clamp(max=n - 1)
    o = torch.where(real[:, None, None], o.permute(0, 3, 1, 2, 4).reshape(r, n, h, d)[req, at], torch.zeros((), device=q.device))
    lse = lse.permute(0, 3, 1, 2).reshape(r, n, h)[req, at]
    return {"out": o.to(q.dtype), "lse": torch.where(real[:, None], lse, torch.full_like(lse, float("-inf")))}


def _counted(s, vocab):
    """How often each row's own tokens (its request's output and its path), and all that it follows, hold each token."""
    history, dev = s["history"].long(), s["history"].device
    r, width = history.shape
    rows = len(s["logits"])
    at = torch.arange(width, device=dev)[None, :]
    there, fresh = at < s["history_lens"][:, None], at >= s["prompt_lens"][:, None]
    req, place, real = _rows_of(s, rows)
    one = torch.zeros(r, vocab, device=dev)
    output = one.scatter_add(1, history, (there & fresh).float())[req]
    seen = one.scatter_add(1, history, there.float())[req]
    if s["starts"] is not None:
        bits = (s["masks"][..., None] >> torch.arange(64, device=dev) & 1).flatten(-2)
        first = torch.arange(rows, device=dev) - place
        token = s["drafted"].long()[(first[:, None] + torch.arange(bits.shape[1], device=dev)).clamp(max=rows - 1)]
        output.scatter_add_(1, token, bits.float())
        seen.scatter_add_(1, token, bits.float())
    return output, seen, req, real


def _adjusted(s):
    """The rows in 32 bits: each operation rounded, in the operator's order."""
    x = s["logits"].float()
    rows, vocab = x.shape
    output, seen, req, real = _counted(s, vocab)
    a = {k: s[k][req][:, None] for k in ("repetition", "frequency", "presence", "temperature")}
    y = torch.where(seen > 0, torch.where(x > 0, x / a["repetition"], x * a["repetition"]), x)
    y = torch.where(output > 0, y - a["frequency"] * output - a["presence"], y)
    del output, seen
    if "bias_tokens" in s:
        tokens = s["bias_tokens"].long()
        bias = torch.zeros(tokens.shape[0], vocab, device=x.device)
        bias.scatter_add_(1, tokens.clamp(min=0), torch.where(tokens >= 0, s["bias_values"], torch.zeros_like(s["bias_values"])))
        y = y + bias[req]
    y = torch.where(a["temperature"] > 0, y / a["temperature"], y)
    if "allowed" in s:
        bit = s["allowed"][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32) & 1
        y = y.masked_fill(bit.flatten(-2)[:, :vocab] == 0, float("-inf"))
    return torch.where(real[:, None], y, x), real


def _plain_adjust(s):
    return {"logits": _adjusted(s)[0].to(s["logits"].dtype)}


def _plain_pick(s):
    y, real = _adjusted(s)
    top = y.amax(-1, keepdim=True)
    at = torch.where(y == top, torch.arange(y.shape[1], device=y.device), y.shape[1]).amin(-1)
    return {"token": torch.where(real & (top.squeeze(-1) > float("-inf")), at, torch.full_like(at, -1)).int()}


def _plain_settle(s):
    n, rows = s["most_new"], len(s["parents"])
    parents, real = _padded(s, s["parents"], n, -1)
    drafted, _ = _padded(s, s["drafted"], n, -1)
    picked, _ = _padded(s, s["picked"], n, -1)
    row = torch.arange(n, device=parents.device)
    # a row stands where its parent's pick is its token, the first of such siblings; it is accepted where its ancestors stand
    right = real & (parents >= 0) & (drafted == picked.gather(1, parents.clamp(min=0).long()))
    same = (parents[:, :, None] == parents[:, None, :]) & right[:, None, :] & (row[None, :] < row[:, None])
    stands = (right & ~same.any(-1)) | ((row == 0) & real)
    chosen = real & (~_closure(parents, real) | stands[:, None, :]).all(-1)
    kept = chosen.sum(1)
    path = torch.where(chosen, row, row + n).sort(1).values
    path = torch.where(path < n, path, torch.full_like(path, -1))
    token = picked.gather(1, path.amax(1, keepdim=True).clamp(min=0)).squeeze(1)
    starts, table, page = s["starts"].long(), s["table"].long(), s["page"]
    before = s["lens"].long()
    base = before - (starts[1:] - starts[:-1])
    lens = base + kept
    # the accepted rows move up behind the committed tokens
    req, j = (path >= 0).nonzero(as_tuple=True)
    source, target = base[req] + path[req, j], base[req] + j
    page_of = lambda p: table[req, p // page]  # noqa: E731
    for codes, scales in s["caches"]:
        for x in (codes, scales):
            x[page_of(target), :, :, target % page] = x[page_of(source), :, :, source % page]
    # pages that hold none of a request's tokens any more go back to the ring, in request order
    col = torch.arange(table.shape[1], device=table.device)[None, :]
    free = (col >= ((lens + page - 1) // page)[:, None]) & (col < ((before + page - 1) // page)[:, None]) & (table >= 0)
    given = s["table"][free]
    at = (s["pool"][1] + torch.arange(len(given), device=table.device)) % len(s["ring"])
    s["ring"][at] = given
    q, place, there = _rows_of(s, rows)
    path = torch.where(there, path[q, place.clamp(max=n - 1)], torch.full_like(q, -1))
    return {"path": path.int(), "kept": kept.int(), "token": token.int(), "lens": lens.int(), "ring": s["ring"],
            "pool": torch.stack([s["pool"][0], s["pool"][1] + len(given)]), "codes": [c for c, _ in s["caches"]],
            "scales": [b for _, b in s["caches"]]}


def run(state):
    s = state
    op = s["case"]["op"]
    if not own:
        return {"plan": _plain_plan, "attend": _plain_attend, "adjust": _plain_adjust, "pick": _plain_pick,
                "settle": _plain_settle}[op](s)
    from sili__new_b200 import serving
    if op == "plan":
        tree = serving.draft_tree(s["parents"], s["starts"], s["lens"], s["most_new"])
        return {"masks": tree.masks, "positions": tree.positions}
    if op == "attend":
        codes, scales = s["caches"][0]
        out, lse = serving.tree_attention(s["q"], codes, scales, s["table"], s["lens"], s["starts"], s["masks"],
                                          most_new=s["most_new"], window=s["window"], return_lse=True)
        return {"out": out, "lse": lse}
    if op in ("adjust", "pick"):
        rules = dict(history=s["history"], history_lens=s["history_lens"], prompt_lens=s["prompt_lens"],
                     repetition=s["repetition"], frequency=s["frequency"], presence=s["presence"],
                     temperature=s["temperature"], bias_tokens=s.get("bias_tokens"), bias_values=s.get("bias_values"),
                     allowed=s.get("allowed"))
        if s["starts"] is not None:
            rules.update(starts=s["starts"], drafted=s["drafted"], masks=s["masks"])
        if op == "adjust":
            return {"logits": serving.adjust_logits(s["logits"], **rules)}
        return {"token": serving.pick_tokens(s["logits"], **rules)}
    a = serving.settle_drafts(s["drafted"], s["parents"], s["picked"], s["starts"], s["lens"], s["table"], s["caches"],
                              s["ring"], s["pool"])
    return {"path": a.path, "kept": a.kept, "token": a.token, "lens": a.lens, "ring": s["ring"], "pool": a.pool,
            "codes": [c for c, _ in s["caches"]], "scales": [b for _, b in s["caches"]]}


def work(case):
    op, r = case["op"], case["requests"]
    counts = _counts(case)
    total = sum(counts)
    if op == "plan":
        # parents, starts and lengths in, a mask and a position a row out
        return {"bytes": total * (4 + 8 * _words(case) + 4) + 8 * r, "flops": 0}
    if op in ("adjust", "pick"):
        vocab, item = case["vocab"], 4 if case["dtype"] == "float32" else 2
        byts = total * vocab * item * (2 if op == "adjust" else 1) + 4 * sum(_spread(r, 0, case["history"]))
        byts += (total * -(-vocab // 32) * 4 if case["masked"] else 0) + r * (8 * case["biases"] + 24)
        return {"bytes": byts + (0 if op == "adjust" else 4 * total), "flops": total * vocab}
    trees, ways = _trees(case)
    if op == "settle":
        row = case["kv_heads"] * 2 * (case["dim"] // 2 + case["dim"] // GROUP)
        moved = sum(sum(1 for j, i in enumerate(w) if i != j) for w in ways)
        return {"bytes": 2 * moved * row * case["layers"] + 16 * total + 20 * r, "flops": 0}
    item = 4 if case["dtype"] == "float32" else 2
    h, hk, d, window = case["heads"], case["kv_heads"], case["dim"], case["window"]
    byts, flops = 0, 0
    for committed, tree in zip(_spread(r, case["least"], case["most"]), trees):
        sees = [bin(m).count("1") for m in _ancestors(tree)]
        pairs = sum(k + (min(committed, max(window - k, 0)) if window else committed) for k in sees)
        keys = len(tree) + (committed if not window else min(committed, max(window - 1, 0)))
        byts += keys * hk * 2 * (d // 2 + d // GROUP) + 4 * (-(-keys // case["page"])) + 8
        flops += 4 * pairs * h * d
    return {"bytes": byts + total * (h * (2 * d * item + 4) + 8 * _words(case)), "flops": flops}


# ── the computed values in 64 bits, from the definitions ─────────────────────
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


def _exact_attend(case, s):
    q, page = s["q"].double(), case["page"]
    t, h, d = q.shape
    codes, scales = s["caches"][0]
    hk = codes.shape[2]
    out = torch.zeros(t, h, d, dtype=torch.float64, device=q.device)
    lse = torch.full((t, h), float("-inf"), dtype=torch.float64, device=q.device)
    starts, first = s["starts"].tolist(), s["parents"].tolist()
    for r, length in enumerate(s["lens"].tolist()):
        a, b = starts[r], starts[r + 1]
        n = b - a
        base = length - n
        visible = torch.zeros(n, length, dtype=torch.bool)
        for i in range(n):
            up, depth = i, 0
            while up >= 0:
                visible[i, base + up] = True
                up, depth = first[a + up], depth + 1
            visible[i, max(0, base + depth - case["window"]) if case["window"] else 0:base] = True
        hidden = ~visible.to(q.device)
        pages = s["table"][r, : -(-length // page)].long()
        for g in range(hk):
            k, v = (_exact_values(codes[pages, w, g], scales[pages, w, g]).reshape(-1, d)[:length] for w in (0, 1))
            x = torch.einsum("nhd,ld->hnl", q[a:b, g * (h // hk):(g + 1) * (h // hk)], k) / math.sqrt(d)
            x = x.masked_fill(hidden, float("-inf"))
            lse[a:b, g * (h // hk):(g + 1) * (h // hk)] = torch.logsumexp(x, -1).T
            out[a:b, g * (h // hk):(g + 1) * (h // hk)] = torch.einsum("hnl,ld->nhd", torch.softmax(x, -1), v)
    return {"out": out, "lse": lse}


def _exact_adjust(case, s):
    x = s["logits"].double()
    starts = s["starts"].tolist() if s["starts"] is not None else list(range(case["requests"] + 1))
    parents, drafted, history = s["parents"].tolist(), s["drafted"].long(), s["history"].long()
    for r in range(case["requests"]):
        length, prompt = int(s["history_lens"][r]), int(s["prompt_lens"][r])
        past = torch.bincount(history[r, :length], minlength=case["vocab"])
        told = torch.bincount(history[r, min(prompt, length):length], minlength=case["vocab"])
        bias = torch.zeros(case["vocab"], dtype=torch.float64, device=x.device)
        if case["biases"]:
            used = s["bias_tokens"][r] >= 0
            bias.index_add_(0, s["bias_tokens"][r][used].long(), s["bias_values"][r][used].double())
        for i in range(starts[r], starts[r + 1]):
            way, up = [], i - starts[r] if s["starts"] is not None else -1
            while up >= 0:
                way.append(starts[r] + up)
                up = parents[starts[r] + up]
            path = torch.bincount(drafted[way], minlength=case["vocab"]) if way else torch.zeros_like(past)
            count, some = (told + path).double(), past + path > 0
            rep = s["repetition"][r].double()
            y = torch.where(some, x[i] * torch.where(x[i] > 0, 1.0 / rep, rep), x[i])
            y = y - count * s["frequency"][r].double() - (count > 0) * s["presence"][r].double() + bias
            heat = float(s["temperature"][r])
            y = y / heat if heat > 0 else y
            if case["masked"]:
                token = torch.arange(case["vocab"], device=x.device)
                y[(s["allowed"][i][token // 32].long() >> (token % 32)) & 1 == 0] = float("-inf")
            x[i] = y
    return {"logits": x}


def exact(case, seed):
    if case["op"] not in ("attend", "adjust") or work(case)["flops"] > 4e12:
        return None
    s = prepare(case, seed)
    return (_exact_attend if case["op"] == "attend" else _exact_adjust)(case, s)

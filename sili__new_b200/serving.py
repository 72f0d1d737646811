"""Serving a folded stack: page tables, rotary positions and attention over a
key/value cache held in 4 bits.

A step (decode, prompt chunk, or both in one batch) of a stack whose
projections are this library's sparse layers goes::

    t = page_tables(cached, fresh, table, ring, pool, cache.page, max_tokens)
    q = cache_append(k, v, cache.codes, cache.scales, t.slots, cos=cos, sin=sin,
                     positions=t.positions, q=q)
    y = cache_attention(q, cache.codes, cache.scales, table, t.lens, starts=t.starts)

Everything stays on the device: no call reads a length back to the host, so a
step can be captured in a CUDA graph.  All work is enqueued on torch's current
stream of the arrays' device; arrays made on another stream are ordered by the
caller, as for any torch operation.  fp32, fp16 and bf16 activations.  Rotary
is differentiable; the cache's calls are not, and refuse inputs that ask for a
gradient.

The cache's format (``KVCache4``): groups of 32 values along the head share
one scale byte (the upper byte below the sign of a half, amax / 6 rounded to
three mantissa bits), values are FP4 codes with the layers' codec; 4.25 bits a
value.
"""
from __future__ import annotations

import math
from typing import NamedTuple

import numpy as np
import torch
from torch.autograd import forward_ad

from . import _cuda

_DTYPES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}
HEAD_DIMS = (64, 128, 256)
GROUP = 32


def _dtype_code(t, who):
    code = _DTYPES.get(t.dtype)
    if code is None:
        raise ValueError(f"{who}: activations must be float32, float16 or bfloat16, got {t.dtype}")
    return code


_raw_stream = torch._C._cuda_getCurrentRawStream     # torch.cuda.current_stream(dev).cuda_stream, without the objects
_I32, _I64, _U8, _F32 = torch.int32, torch.int64, torch.uint8, torch.float32


def _on_device(who, dev, *arrays):
    """The current stream's handle of the CUDA device that every array is on."""
    at = dev.index
    for a in arrays:
        if a is not None and (a.get_device() != at or not a.is_cuda):
            if not a.is_cuda or dev.type != "cuda":
                raise ValueError(f"{who}: arrays must be CUDA tensors")
            raise ValueError(f"{who}: arrays are on different devices")
    if dev.type != "cuda":
        raise ValueError(f"{who}: arrays must be CUDA tensors")
    return _raw_stream(at)


class _Here:
    def __enter__(self):
        return self

    def __exit__(self, *a):
        return False


_HERE = _Here()


def _on(dev):
    """Context that makes `dev` the current device (nothing to do where it is already)."""
    return _HERE if torch._C._cuda_getDevice() == dev.index else torch.cuda.device(dev)


def _contiguous(who, name, t, dtype, shape=None):
    if t.dtype is dtype and (shape is None or t.shape == shape) and t.is_contiguous():
        return
    if t.dtype != dtype:
        raise ValueError(f"{who}: {name} must be {dtype}, got {t.dtype}")
    if not t.is_contiguous():
        raise ValueError(f"{who}: {name} must be contiguous")
    raise ValueError(f"{who}: {name} must be {list(shape)}, got {list(t.shape)}")


def _heads(who, name, t, tokens=None, dim=None, dtype=None):
    """[tokens, heads, dim] with the last axis contiguous; any other strides."""
    if t.dim() == 3 and t.stride(2) == 1 and (tokens is None or t.shape[0] == tokens) and \
            (dim is None or t.shape[2] == dim) and (dtype is None or t.dtype is dtype):
        return
    if t.dim() != 3:
        raise ValueError(f"{who}: {name} must be [tokens, heads, dim], got {list(t.shape)}")
    if t.stride(2) != 1 and t.shape[2] > 1:
        raise ValueError(f"{who}: {name}'s last axis must be contiguous")
    if tokens is not None and t.shape[0] != tokens:
        raise ValueError(f"{who}: {name} has {t.shape[0]} tokens, expected {tokens}")
    if dim is not None and t.shape[2] != dim:
        raise ValueError(f"{who}: {name} has head dimension {t.shape[2]}, expected {dim}")
    if dtype is not None and t.dtype != dtype:
        raise ValueError(f"{who}: {name} is {t.dtype}, expected {dtype}")


def _apart(who, name, t):
    """Refuses an output [tokens, heads, dim] whose rows may share elements."""
    (tokens, heads, dim), (st, sh, _) = t.shape, t.stride()
    if (heads < 2 or sh >= dim) and (tokens < 2 or st >= (sh * (heads - 1) if heads > 1 else 0) + dim):
        return
    if (tokens < 2 or st >= dim) and (heads < 2 or sh >= (st * (tokens - 1) if tokens > 1 else 0) + dim):
        return
    if t.numel():
        raise ValueError(f"{who}: {name}'s rows may share elements (strides {list(t.stride())})")


def _is_dual(t):
    return t is not None and forward_ad.unpack_dual(t).tangent is not None


def _no_gradient(who, *arrays):
    """Refuses inputs whose gradient or tangent the call would drop."""
    if torch.is_grad_enabled():
        for a in arrays:
            if a is not None and a.requires_grad:
                raise ValueError(f"{who}: has no gradient: call it under torch.no_grad() or with detached inputs")
    if forward_ad._current_level >= 0 and any(_is_dual(a) for a in arrays):
        raise ValueError(f"{who}: has no gradient: its inputs must not carry a tangent")


# ── page tables ──────────────────────────────────────────────────────────────
class PageTables(NamedTuple):
    """One step's maps (``page_tables``)."""
    starts: torch.Tensor      # int32 [requests + 1]: the new tokens' offsets
    lens: torch.Tensor        # int32 [requests]: cached + fresh
    slots: torch.Tensor       # int64 [max_tokens]: page * page size + offset, -1: none
    positions: torch.Tensor   # int32 [max_tokens], -1: no token
    pool: torch.Tensor        # int64 [2]: pages taken from and given to the ring, after this step
    status: torch.Tensor      # int64 [3]: pages that lacked, tokens beyond max_tokens, pages beyond the table


def page_pool(n_pages: int, device="cuda"):
    """(ring, pool) of a cache whose pages are all free."""
    ring = torch.arange(n_pages, dtype=torch.int32, device=device)
    return ring, torch.tensor([0, n_pages], dtype=torch.int64, device=device)


def _check_block_table(who, table, requests):
    if table.dtype != torch.int32 or table.dim() != 2 or table.shape[0] != requests:
        raise ValueError(f"{who}: table must be int32 [{requests}, width], got {table.dtype} {list(table.shape)}")
    if table.numel() and (table.shape[1] > 1 and table.stride(1) != 1 or
                          requests > 1 and table.stride(0) < table.shape[1]):
        raise ValueError(f"{who}: table's rows must be contiguous and not overlap")


def _row_stride(table):
    # a single row's stride may be anything
    return table.stride(0) if table.shape[0] > 1 else table.shape[1]


def _check_tables(who, table, ring, pool, page, requests):
    _check_block_table(who, table, requests)
    _contiguous(who, "ring", ring, torch.int32, (ring.numel(),))
    _contiguous(who, "pool", pool, torch.int64, (2,))
    if page < 1:
        raise ValueError(f"{who}: page size must be positive")


def page_tables(cached, fresh, table, ring, pool, page: int, max_tokens: int) -> PageTables:
    """Block tables and slot map of one step, from request lengths.

    Request r holds ``cached[r]`` tokens and brings ``fresh[r]`` (int32 both).
    ``table`` [requests, width] gets the pages that the new tokens open, taken
    from ``ring`` in request order (``pool`` = pages taken, given); -1 where
    the ring runs out, and the tokens of such a page have slot -1.  Nothing is
    read back: look at ``status`` when it suits.  The same inputs again write
    the same values, so pass the returned ``pool`` on to the next step.  A step
    that lacked pages is asked for again with the lengths and the ``pool`` of
    before it, after ``release_pages`` with those (its returned pool counts the
    pages that it did get as held)."""
    who = "page_tables"
    n = cached.numel()
    dev = cached.device
    _contiguous(who, "cached", cached, torch.int32, (n,))
    _contiguous(who, "fresh", fresh, torch.int32, (n,))
    _check_tables(who, table, ring, pool, page, n)
    if not 0 <= max_tokens <= 0x7FFFFFFF:
        raise ValueError(f"{who}: max_tokens out of range")
    s = _on_device(who, dev, fresh, table, ring, pool)
    with _on(dev):
        # one allocation a type: int64 slots, pool, status; int32 positions, starts, lens (and the scan of large batches)
        extra = n + 1 if n > 4096 else 0
        wide = torch.empty(max_tokens + 5, dtype=_I64, device=dev)
        small = torch.empty(max_tokens + 2 * n + 1 + extra, dtype=_I32, device=dev)
        at8, at4 = wide.data_ptr(), small.data_ptr()
        at_starts = at4 + 4 * max_tokens
        at_lens = at_starts + 4 * (n + 1)
        _cuda.page_tables_ptr(cached.data_ptr(), fresh.data_ptr(), n, table.data_ptr(), _row_stride(table), table.shape[1],
                              ring.data_ptr(), ring.numel(), pool.data_ptr(), page, max_tokens, at_starts, at_lens, at8,
                              at4, at8 + 8 * max_tokens, at8 + 8 * (max_tokens + 2), at_lens + 4 * n if extra else 0, s)
        slots, pool_out, status = wide.split_with_sizes((max_tokens, 2, 3))
        positions, starts, lens, *_ = small.split_with_sizes((max_tokens, n + 1, n, extra) if extra else
                                                             (max_tokens, n + 1, n))
    return PageTables(starts, lens, slots, positions, pool_out, status)


def release_pages(finished, lens, table, ring, pool, page: int):
    """Gives the pages of finished requests (bool [requests]) back to the
    ring: their table entries become -1 and their ``lens`` 0, in place.
    Returns the new pool."""
    who = "release_pages"
    n = lens.numel()
    dev = lens.device
    _contiguous(who, "finished", finished, torch.bool, (n,))
    _contiguous(who, "lens", lens, torch.int32, (n,))
    _check_tables(who, table, ring, pool, page, n)
    if ring.numel() < 1:
        raise ValueError(f"{who}: an empty ring")
    s = _on_device(who, dev, finished, table, ring, pool)
    with _on(dev):
        out = torch.empty(2, dtype=torch.int64, device=dev)
        scratch = torch.empty(max(n, 1), dtype=torch.int32, device=dev)
        _cuda.release_pages_ptr(finished.data_ptr(), n, lens.data_ptr(), table.data_ptr(), _row_stride(table),
                                table.shape[1], ring.data_ptr(), ring.numel(), pool.data_ptr(), page, out.data_ptr(),
                                scratch.data_ptr(), s)
    return out


# ── rotary positions ─────────────────────────────────────────────────────────
def rotary_frequencies(rotary_dim: int, base: float = 10000.0, scaling: dict | None = None):
    """(inverse frequencies float64 [rotary_dim / 2], gain) of the pairs.

    ``scaling`` stretches the positions for contexts past the trained one:

    * None -- base ** (-2 i / rotary_dim)
    * ``{"type": "linear", "factor": f}`` -- every frequency over f
    * ``{"type": "base", "factor": f}`` -- the base raised by f ** (d / (d - 2)), so
      that the slowest pair is stretched by f and the fastest kept
    * ``{"type": "yarn", "factor": f, "original": n, "fast": 32, "slow": 1}`` -- pairs
      that turn over ``fast`` times within n positions kept, under ``slow``
      times over f, a linear ramp over the pair index between; the table is
      multiplied by 0.1 ln f + 1 (or ``"gain"``)
    * ``{"type": "wavelength", "factor": f, "original": n, "fast": 4, "slow": 1}`` --
      as above with the ramp linear in the number of turns, no gain
    """
    if rotary_dim < 2 or rotary_dim % 2:
        raise ValueError(f"rotary_frequencies: rotary_dim must be even and positive, got {rotary_dim}")
    if base <= 0:
        raise ValueError("rotary_frequencies: base must be positive")
    i = np.arange(rotary_dim // 2, dtype=np.float64)
    inv = base ** (-2.0 * i / rotary_dim)
    if scaling is None:
        return inv, 1.0
    kind = scaling.get("type")
    f = float(scaling.get("factor", 1.0))
    if f <= 0:
        raise ValueError("rotary_frequencies: factor must be positive")
    if kind == "linear":
        return inv / f, 1.0
    if kind == "base":
        if rotary_dim < 4:
            raise ValueError("rotary_frequencies: 'base' needs a rotary_dim above 2")
        return (base * f ** (rotary_dim / (rotary_dim - 2.0))) ** (-2.0 * i / rotary_dim), 1.0
    if kind not in ("yarn", "wavelength"):
        raise ValueError(f"rotary_frequencies: unknown scaling type {kind!r}")
    n = float(scaling["original"])
    slow = float(scaling.get("slow", 1.0))
    fast = float(scaling.get("fast", 32.0 if kind == "yarn" else 4.0))
    if not 0 < slow < fast or n <= 0:
        raise ValueError("rotary_frequencies: needs 0 < slow < fast and a positive original length")
    if kind == "wavelength":
        keep = np.clip((n * inv / (2.0 * math.pi) - slow) / (fast - slow), 0.0, 1.0)
        return inv * keep + inv / f * (1.0 - keep), 1.0

    def pair_of(turns):   # the (fractional) pair that turns so many times within the original length
        return rotary_dim * math.log(n / (turns * 2.0 * math.pi)) / (2.0 * math.log(base))

    low = max(math.floor(pair_of(fast)), 0)
    high = min(math.ceil(pair_of(slow)), rotary_dim - 1)
    keep = 1.0 - np.clip((i - low) / max(high - low, 0.001), 0.0, 1.0)
    gain = float(scaling.get("gain", 0.1 * math.log(f) + 1.0 if f > 1.0 else 1.0))
    return inv * keep + inv / f * (1.0 - keep), gain


def rotary_table(n_positions: int, rotary_dim: int, base: float = 10000.0, scaling: dict | None = None, device="cuda"):
    """(cos, sin) float32 [n_positions, rotary_dim / 2]; the angles are taken
    in 64 bits, so the table is right at every position."""
    inv, gain = rotary_frequencies(rotary_dim, base, scaling)
    if n_positions < 1:
        raise ValueError("rotary_table: n_positions must be positive")
    dev = torch.device(device)
    if dev.type != "cuda":
        raise ValueError("rotary_table: needs a CUDA device")
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    with _on(dev):
        cos = torch.empty(n_positions, rotary_dim // 2, dtype=torch.float32, device=dev)
        sin = torch.empty_like(cos)
        _cuda.rotary_table_ptr(inv, n_positions, gain, cos.data_ptr(), sin.data_ptr(),
                               _raw_stream(dev.index))
    return cos, sin


def _check_table(who, cos, sin, positions, tokens, dim):
    shape = cos.shape
    if len(shape) == 2 and shape[0] >= 1 and 2 <= 2 * shape[1] <= dim and cos.dtype is _F32 and sin.dtype is _F32 and \
            sin.shape == shape and cos.is_contiguous() and sin.is_contiguous() and \
            positions.dtype in (_I32, _I64) and positions.shape == (tokens,) and positions.is_contiguous():
        return
    if len(shape) != 2 or shape[0] < 1 or shape[1] < 1:
        raise ValueError(f"{who}: cos must be [positions, rotary_dim / 2], got {list(shape)}")
    _contiguous(who, "cos", cos, _F32)
    _contiguous(who, "sin", sin, _F32, tuple(shape))
    if 2 * shape[1] > dim:
        raise ValueError(f"{who}: the table turns {2 * shape[1]} elements, the head has {dim}")
    if positions.dtype not in (_I32, _I64):
        raise ValueError(f"{who}: positions must be int32 or int64, got {positions.dtype}")
    raise ValueError(f"{who}: positions must be a contiguous [{tokens}], got {list(positions.shape)}")


def _interleaved(who, layout):
    if layout not in ("half", "interleaved"):
        raise ValueError(f"{who}: layout must be 'half' or 'interleaved', got {layout!r}")
    return layout == "interleaved"


def _turn(who, q, k, cos, sin, positions, layout, inverse, q_out, k_out):
    _heads(who, "q", q)
    tokens, _, dim = q.shape
    code = _dtype_code(q, who)
    if k is not None:
        _heads(who, "k", k, tokens, dim, q.dtype)
    _check_table(who, cos, sin, positions, tokens, dim)
    inter = _interleaved(who, layout)
    dev = q.device
    for name, x, o in (("q_out", q, q_out), ("k_out", k, k_out)):
        if o is not None:
            _heads(who, name, o, tokens, dim, q.dtype)
            if x is None or o.shape != x.shape:
                raise ValueError(f"{who}: {name} must have its input's shape")
            _apart(who, name, o)
    s = _on_device(who, dev, k, cos, sin, positions, q_out, k_out)
    with _on(dev):
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        if k is None:
            _cuda.rotary_ptr(code, q.data_ptr(), q.stride(0), q.stride(1), q_out.data_ptr(), q_out.stride(0),
                             q_out.stride(1), q.shape[1], 0, 0, 0, 0, 0, 0, 0, tokens, dim, 2 * cos.shape[1],
                             cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
                             positions.dtype == torch.int64, inter, inverse, s)
            return q_out, None
        if k_out is None:
            k_out = torch.empty(k.shape, dtype=k.dtype, device=dev)
        _cuda.rotary_ptr(code, q.data_ptr(), q.stride(0), q.stride(1), q_out.data_ptr(), q_out.stride(0),
                         q_out.stride(1), q.shape[1], k.data_ptr(), k.stride(0), k.stride(1), k_out.data_ptr(),
                         k_out.stride(0), k_out.stride(1), k.shape[1], tokens, dim, 2 * cos.shape[1], cos.data_ptr(),
                         sin.data_ptr(), cos.shape[0], positions.data_ptr(), positions.dtype == torch.int64, inter,
                         inverse, s)
    return q_out, k_out


class _Rotary(torch.autograd.Function):
    """The turn is linear: its gradient is the turn back, its tangent the same turn, each differentiable in its turn."""

    @staticmethod
    def forward(q, k, cos, sin, positions, layout, inverse):
        return _turn("rotary", q, k, cos, sin, positions, layout, inverse, None, None)

    @staticmethod
    def setup_context(ctx, inputs, output):
        _, _, cos, sin, positions, ctx.layout, ctx.inverse = inputs
        ctx.save_for_backward(cos, sin, positions)
        ctx.save_for_forward(cos, sin, positions)

    @staticmethod
    def _of_both(ctx, inverse, dq, dk):
        """(dq, dk) turned; either may be None."""
        cos, sin, positions = ctx.saved_tensors
        grads = [None, None]
        parts = [(i, g if g.stride(-1) == 1 else g.contiguous()) for i, g in enumerate((dq, dk)) if g is not None]
        if parts:
            out = _Rotary.apply(parts[0][1], parts[1][1] if len(parts) > 1 else None, cos, sin, positions, ctx.layout,
                                inverse)
            for (i, _), g in zip(parts, out):
                grads[i] = g
        return grads

    @staticmethod
    def backward(ctx, dq, dk):
        return (*_Rotary._of_both(ctx, not ctx.inverse, dq, dk), None, None, None, None, None)

    @staticmethod
    def jvp(ctx, tq, tk, *_):
        return tuple(_Rotary._of_both(ctx, ctx.inverse, tq, tk))


def _rotary(who, q, k, cos, sin, positions, layout, inverse, q_out, k_out):
    _no_gradient(f"{who}'s table", cos, sin)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)) or \
            forward_ad._current_level >= 0 and (_is_dual(q) or _is_dual(k)):
        if q_out is not None or k_out is not None:
            raise ValueError(f"{who}: an output array and a gradient exclude each other")
        return _Rotary.apply(q, k, cos, sin, positions, layout, inverse)
    return _turn(who, q, k, cos, sin, positions, layout, inverse, q_out, k_out)


def rotary(q, k, cos, sin, positions, layout: str = "half", q_out=None, k_out=None):
    """Rotary positions of q [tokens, heads, dim] and k [tokens, kv heads,
    dim] (or None): the first 2 * cos.shape[1] elements of each head are
    turned by the token's angles, the rest passes through.  ``layout``: pairs
    (i, i + half) or adjacent ones.  ``cos`` / ``sin`` from ``rotary_table``;
    ``positions`` int32 or int64 [tokens]: a negative one (padding) gives
    zeros, one past the table NaN.  ``q_out`` / ``k_out`` may be the inputs
    (in place), and share no elements otherwise.  Differentiable in q and k to
    any order, in reverse and forward mode, when no output is given; not in
    the table, which must not ask for a gradient.  Returns (q', k')."""
    return _rotary("rotary", q, k, cos, sin, positions, layout, False, q_out, k_out)


def rotary_backward(dq, dk, cos, sin, positions, layout: str = "half", q_out=None, k_out=None):
    """The gradient of ``rotary``: (dq, dk) of its outputs -> of its inputs
    (the turn back by the same angles); differentiable as ``rotary`` is."""
    return _rotary("rotary_backward", dq, dk, cos, sin, positions, layout, True, q_out, k_out)


# ── the 4-bit cache ──────────────────────────────────────────────────────────
class KVCache4:
    """The pages of a 4-bit key/value cache: ``codes`` uint8 [n_pages, 2,
    kv_heads, page, dim / 2] and ``scales`` uint8 [n_pages, 2, kv_heads, page,
    dim / 32] (K, then V)."""

    def __init__(self, n_pages: int, page: int, kv_heads: int, dim: int, device="cuda"):
        if dim not in HEAD_DIMS:
            raise ValueError(f"KVCache4: head dimension must be one of {HEAD_DIMS}, got {dim}")
        if page < 16 or page % 16:
            raise ValueError(f"KVCache4: page size must be a multiple of 16, got {page}")
        if n_pages < 1 or kv_heads < 1:
            raise ValueError("KVCache4: needs at least one page and one kv head")
        self.n_pages, self.page, self.kv_heads, self.dim = n_pages, page, kv_heads, dim
        self.codes = torch.zeros(n_pages, 2, kv_heads, page, dim // 2, dtype=torch.uint8, device=device)
        self.scales = torch.zeros(n_pages, 2, kv_heads, page, dim // GROUP, dtype=torch.uint8, device=device)

    @property
    def bytes_per_token(self) -> int:
        return 2 * self.kv_heads * (self.dim // 2 + self.dim // GROUP)


def _check_cache(who, codes, scales):
    shape = codes.shape
    if len(shape) == 5:
        n_pages, two, hk, page, half = shape
        if two == 2 and 2 * half in HEAD_DIMS and codes.dtype is _U8 and scales.dtype is _U8 and \
                scales.shape == (n_pages, 2, hk, page, half // (GROUP // 2)) and codes.is_contiguous() and \
                scales.is_contiguous():
            return n_pages, hk, page, 2 * half
    if len(shape) != 5 or shape[1] != 2 or 2 * shape[4] not in HEAD_DIMS:
        raise ValueError(f"{who}: codes must be [pages, 2, kv heads, page, dim / 2] with dim in {HEAD_DIMS}, "
                         f"got {list(shape)}")
    _contiguous(who, "codes", codes, _U8)
    _contiguous(who, "scales", scales, _U8, (*shape[:4], shape[4] // (GROUP // 2)))
    return shape[0], shape[2], shape[3], 2 * shape[4]


def _check_slots(who, slots, tokens):
    if slots.dim() != 1 or (tokens is not None and slots.shape[0] != tokens):
        raise ValueError(f"{who}: slots must be [{'tokens' if tokens is None else tokens}], got {list(slots.shape)}")
    _contiguous(who, "slots", slots, torch.int64)


def cache_append(k, v, codes, scales, slots, cos=None, sin=None, positions=None, layout: str = "half", q=None,
                 q_out=None):
    """Writes k, v [tokens, kv heads, dim] into the cache at ``slots`` (int64;
    a slot outside the cache, such as a padding token's -1, is passed over;
    no two tokens may share one), in one launch with the rotation of k, and of
    ``q`` when given, by ``positions`` (see ``rotary``; the rotated part a
    multiple of 16).  Head rows start on 16 bytes (any strides otherwise).
    Returns the rotated q (None without q; ``q_out`` may be q itself)."""
    who = "cache_append"
    n_pages, hk, page, dim = _check_cache(who, codes, scales)
    code = _dtype_code(k, who)
    _heads(who, "k", k, None, dim)
    tokens = k.shape[0]
    _heads(who, "v", v, tokens, dim, k.dtype)
    if k.shape[1] != hk or v.shape[1] != hk:
        raise ValueError(f"{who}: the cache has {hk} kv heads, k {k.shape[1]}, v {v.shape[1]}")
    _check_slots(who, slots, tokens)
    rot = 0
    if (cos is None) != (sin is None) or (cos is None) != (positions is None):
        raise ValueError(f"{who}: cos, sin and positions come together")
    if cos is not None:
        _check_table(who, cos, sin, positions, tokens, dim)
        rot = 2 * cos.shape[1]
    if q is None and q_out is not None:
        raise ValueError(f"{who}: q_out without q")
    if q is not None:
        if not rot:
            raise ValueError(f"{who}: q is only taken along to be rotated: give cos, sin and positions")
        _heads(who, "q", q, tokens, dim, k.dtype)
        if q_out is not None:
            _heads(who, "q_out", q_out, tokens, dim, k.dtype)
            if q_out.shape != q.shape:
                raise ValueError(f"{who}: q_out must have q's shape")
            _apart(who, "q_out", q_out)
    inter = _interleaved(who, layout)
    _no_gradient(who, k, v, q, cos, sin)
    dev = k.device
    s = _on_device(who, dev, v, codes, scales, slots, cos, sin, positions, q, q_out)
    with _on(dev):
        if q is not None and q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=dev)
        qa = (q.data_ptr(), q.stride(0), q.stride(1), q_out.data_ptr(), q_out.stride(0), q_out.stride(1), q.shape[1]) \
            if q is not None else (0, 0, 0, 0, 0, 0, 0)
        ra = (rot, cos.data_ptr(), sin.data_ptr(), cos.shape[0], positions.data_ptr(),
              positions.dtype == torch.int64) if rot else (0, 0, 0, 0, 0, False)
        _cuda.kv4_append_ptr(code, *qa, k.data_ptr(), k.stride(0), k.stride(1), v.data_ptr(), v.stride(0), v.stride(1),
                             hk, tokens, dim, *ra, inter, codes.data_ptr(), scales.data_ptr(), n_pages, page,
                             slots.data_ptr(), s)
    return q_out


def cache_read(codes, scales, slots, dtype=torch.float32):
    """(k, v) [tokens, kv heads, dim]: the values that the cache holds at
    ``slots`` (zeros for a slot outside it).  Exact in every ``dtype``."""
    who = "cache_read"
    n_pages, hk, page, dim = _check_cache(who, codes, scales)
    _check_slots(who, slots, None)
    if dtype not in _DTYPES:
        raise ValueError(f"{who}: dtype must be float32, float16 or bfloat16, got {dtype}")
    dev = codes.device
    s = _on_device(who, dev, scales, slots)
    tokens = slots.shape[0]
    with _on(dev):
        k = torch.empty(tokens, hk, dim, dtype=dtype, device=dev)
        v = torch.empty_like(k)
        _cuda.kv4_read_ptr(_DTYPES[dtype], codes.data_ptr(), scales.data_ptr(), n_pages, page, hk, dim, slots.data_ptr(),
                           tokens, k.data_ptr(), v.data_ptr(), s)
    return k, v


# a zeroed workspace per (device, stream): calls on one stream are ordered, so they may share one
_workspaces: dict = {}


def _workspace(dev, stream):
    if torch._C._cuda_isCurrentStreamCapturing():
        # a graph owns its workspace: it may be replayed on any stream, beside eager calls
        return _new_workspace(dev)
    w = _workspaces.get((dev.index, stream))
    if w is None:
        w = _workspaces[(dev.index, stream)] = _new_workspace(dev)
    return w


def _new_workspace(dev):
    w = torch.empty(_cuda.kv4_attention_workspace(), dtype=torch.uint8, device=dev)
    w[:4096].zero_()      # the counters; the rest is written before it is read
    return w


def check_attention(device=None):
    """Raises RuntimeError if a device-side wait of an eager ``cache_attention``
    on the current stream gave up since the last check (its rows are NaN).
    Waits for the stream; a captured call's rows tell by themselves."""
    dev = torch.device("cuda" if device is None else device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    w = _workspaces.get((dev.index, _raw_stream(dev.index)))
    if w is not None:
        with _on(dev):
            _cuda.kv4_attention_status_ptr(w.data_ptr(), _raw_stream(dev.index))


def cache_attention(q, codes, scales, table, lens, starts=None, most_new=None, scale=None, window: int = 0, out=None,
                    return_lse: bool = False):
    """Causal attention of q [tokens, heads, dim] (rows start on 8 bytes, any
    strides otherwise) over the 4-bit cache.

    ``table`` int32 [requests, width] and ``lens`` int32 [requests] (cached
    plus new tokens) from ``page_tables``.  ``starts`` int32 [requests + 1]:
    request r's queries are rows starts[r] .. starts[r + 1), at its last
    positions (rows that q does not have, beyond ``max_tokens``, are left out);
    without it row r is request r's one query.  ``most_new``: the
    largest number of queries of a request, if the host knows it (it picks the
    kernel, not the result; without it the mean is taken).  ``window`` > 0: only the last so many keys.
    ``scale``: 1 / sqrt(dim) by default.  Grouped queries: query head h reads
    kv head h // (heads / kv heads).  Rows that see nothing (no keys, or past
    the last request's) are zeros, their lse -inf.  Returns ``out`` [tokens,
    heads, dim] in q's type, with ``return_lse`` (out, lse float32 [tokens,
    heads], natural log)."""
    who = "cache_attention"
    n_pages, hk, page, dim = _check_cache(who, codes, scales)
    if page < 16 or page % 16:
        raise ValueError(f"{who}: page size must be a multiple of 16, got {page}")
    code = _dtype_code(q, who)
    _heads(who, "q", q, None, dim)
    tokens, heads, _ = q.shape
    if heads < 1 or heads % hk:
        raise ValueError(f"{who}: {hk} kv heads do not divide {heads} query heads")
    requests = lens.numel()
    _contiguous(who, "lens", lens, torch.int32, (requests,))
    _check_block_table(who, table, requests)
    if starts is None:
        if tokens != requests:
            raise ValueError(f"{who}: without starts q has one row a request: {tokens} rows, {requests} requests")
        most_new = 1
    else:
        _contiguous(who, "starts", starts, torch.int32, (requests + 1,))
        if most_new is None:
            most_new = -(-tokens // max(requests, 1))
    if window < 0:
        raise ValueError(f"{who}: window must not be negative")
    window, most_new = min(window, 0x7FFFFFFF), min(most_new, 0x7FFFFFFF)
    _no_gradient(who, q)
    dev = q.device
    s = _on_device(who, dev, codes, scales, table, lens, starts, out)
    with _on(dev):
        if out is None:
            out = torch.empty(tokens, heads, dim, dtype=q.dtype, device=dev)
        else:
            _contiguous(who, "out", out, q.dtype, (tokens, heads, dim))
        lse = torch.empty(tokens, heads, dtype=torch.float32, device=dev) if return_lse else None
        _cuda.kv4_attention_ptr(code, q.data_ptr(), q.stride(0), q.stride(1), tokens, heads, dim, codes.data_ptr(),
                                scales.data_ptr(), n_pages, page, hk, table.data_ptr(), _row_stride(table), table.shape[1],
                                lens.data_ptr(), requests, 0 if starts is None else starts.data_ptr(), most_new,
                                1.0 / math.sqrt(dim) if scale is None else float(scale), window, out.data_ptr(),
                                0 if lse is None else lse.data_ptr(), _workspace(dev, s).data_ptr(), s)
    return (out, lse) if return_lse else out

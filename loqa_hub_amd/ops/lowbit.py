"""Ops of a serving step in low bits: a paged key / value cache of 8 bits with a scale for each page and
kv head, the rotation and append that write it, attention off it for tokens and prompts, the pages and
slots of a step handed out on the GPU, and products with 4-bit weights and group scales.

They stand beside their bf16 counterparts in ``ops`` (:func:`ops.rope_kv_append`, :func:`ops.attention`,
:func:`ops.linear`) and the engine's host block pool. A step of one token is bound by the bytes of weights
and cache that it reads: half of them here for the cache, a quarter for the weights.

As everywhere in ``ops``: GPU tensors run the HIP kernels (``csrc/kernels/cache8.hip``,
``attn_cache8.hip``, ``linear4.hip``), CPU tensors the PyTorch references. Rows are bfloat16; scales,
softmax and sums are f32.

Sequences are given as everywhere: ``cu_q`` [B + 1] int32 bounds each sequence's rows, ``ctx_lens`` [B]
int32 its tokens with this step's, ``block_tables`` [B, max_blocks] int32 its pages; row i of a sequence
of n rows stands at position ctx - n + i. Rows behind the last sequence are neither read nor written.
Page numbers outside of the cache are never followed: nothing is appended there, and attention takes its
keys as masked. Appends and token steps take up to 65535 sequences a call. A page that gets rows belongs to one sequence; full pages may be shared.
"""
from __future__ import annotations

import contextlib
import functools
import math
from typing import NamedTuple

import torch

from . import reference as ref
from . import _sk_workspace
from ._lib import check, kernels, ptr, stream_ptr

CACHE_TYPES = {torch.int8: 0, torch.float8_e4m3fn: 1}
HEAD_DIMS = (64, 128)
PROMPT_ROWS = 128                     # rows of a workgroup (csrc/kernels/attn_cache8.hip)
SLOTS = 512                           # workgroups at once, two a compute unit


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _typed(t: torch.Tensor, dtype: torch.dtype, name: str) -> None:
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype}, got {t.dtype}")


def _i32(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    _typed(t, torch.int32, name)
    _need(t.is_contiguous(), f"{name} must be contiguous")
    _need(t.device == like.device, f"{name} must be on {like.device}")


def _there(index: int):
    """Launches go to the tensors' own device, whichever is the current one."""
    return _HERE if index == torch._C._cuda_getDevice() else torch.cuda.device(index)


def _elsewhere(cache, fn, *args, **kw):
    """The call once more with the cache's device as the current one; its checks have passed."""
    index = cache.k.get_device()
    if index == torch._C._cuda_getDevice():
        raise RuntimeError(f"{fn.__name__} does not take this call")
    with torch.cuda.device(index):
        return fn(*args, **kw)


_HERE = contextlib.nullcontext()
_stream = torch._C._cuda_getCurrentRawStream if hasattr(torch._C, "_cuda_getCurrentRawStream") else None


class Cache8:
    """A layer's paged cache in 8 bits: ``k``, ``v`` [n_blocks, n_kv, block_size, head_dim] int8 or
    float8_e4m3fn codes and ``k_scale``, ``v_scale`` [n_blocks, n_kv] f32: an entry stands for code * scale.
    A page's scale starts anew with the row at its first place and only grows until the next such row; its
    older rows are rounded again where it grows, so a page filled row by row is off by up to a step where one filled at
    once is off by half a step. e4m3 scales are powers of two, whose growth rounds nothing again but the smallest
    entries. Codes are numbers: e4m3's NaN, which no append writes, may reach every row of a feed
    that it is cached for. Scales below 2^-100, negative ones among them, count as 2^-100 everywhere. Page sizes are
    powers of two from 16 on."""

    __slots__ = ("k", "v", "k_scale", "v_scale", "kind", "n_blocks", "n_kv", "block_size", "head_dim", "cuda")

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor):
        if k.dtype not in CACHE_TYPES:
            raise TypeError(f"a cache of int8 or float8_e4m3fn, got {k.dtype}")
        _typed(v, k.dtype, "v")
        _typed(k_scale, torch.float32, "k_scale")
        _typed(v_scale, torch.float32, "v_scale")
        _need(k.dim() == 4 and v.shape == k.shape, "k and v are [n_blocks, n_kv, block_size, head_dim]")
        _need(k_scale.shape == k.shape[:2] and v_scale.shape == k.shape[:2], "scales are [n_blocks, n_kv]")
        _need(all(t.is_contiguous() and t.device == k.device for t in (k, v, k_scale, v_scale)), "contiguous tensors of one device")
        _need((k.data_ptr() | v.data_ptr()) % 16 == 0, "k and v must start at 16 bytes")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.kind, self.cuda = CACHE_TYPES[k.dtype], k.is_cuda
        self.n_blocks, self.n_kv, self.block_size, self.head_dim = k.shape
        _need(self.n_blocks > 0 and self.n_kv > 0, "a cache without pages")
        _need(self.head_dim in HEAD_DIMS, f"head_dim is one of {HEAD_DIMS}, got {self.head_dim}")
        _need(self.block_size >= 16 and self.block_size & (self.block_size - 1) == 0, "block_size is a power of two from 16 on")
        _need(self.n_blocks * self.block_size < 1 << 31 and self.n_kv * self.block_size * self.head_dim < 1 << 31,
              "slots and places within a page have 32 bits")

    @classmethod
    def empty(cls, n_blocks: int, n_kv: int, block_size: int, head_dim: int, dtype=torch.int8, device=None) -> "Cache8":
        if dtype not in CACHE_TYPES:
            raise TypeError(f"a cache of int8 or float8_e4m3fn, got {dtype}")
        shape = (n_blocks, n_kv, block_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8, device=device).view(dtype) for _ in range(2))
        return cls(k, v, torch.zeros(shape[:2], device=device), torch.zeros(shape[:2], device=device))

    @property
    def device(self) -> torch.device:
        return self.k.device

    @staticmethod
    def bytes_per_block(n_kv: int, head_dim: int, block_size: int) -> int:
        return 2 * n_kv * (block_size * head_dim + 4)


def _sequences(cu_q, ctx_lens, block_tables, like) -> tuple[int, int]:
    for t, name in ((cu_q, "cu_q"), (ctx_lens, "ctx_lens"), (block_tables, "block_tables")):
        _i32(t, name, like)
    B = ctx_lens.numel()
    _need(cu_q.numel() == B + 1 and block_tables.dim() == 2 and block_tables.shape[0] == B, "cu_q [B + 1], ctx_lens [B], block_tables [B, max_blocks]")
    _need(B == 0 or block_tables.shape[1] > 0, "a block table without columns")
    return B, block_tables.shape[1]


def _rows(t: torch.Tensor, cols: int, name: str, like) -> None:
    _typed(t, torch.bfloat16, name)
    _need(t.dim() == 2 and t.shape[1] >= cols and (t.stride(1) == 1 or t.shape[1] == 1), f"{name} must be rows of at least {cols} columns")
    _need(t.shape[0] <= 1 or t.stride(0) >= cols, f"rows of {name} must not overlap")
    _need(t.device == like.device, f"{name} must be on {like.device}")


def _rows8(x, y, cu_q, ctx_lens, block_tables, cache, cols: int, cols_y: int):
    """All of a GPU call's checks of its rows and sequences at once (csrc/launch); None: anything is otherwise."""
    return kernels().cache8_rows(x, y, cu_q, ctx_lens, block_tables, cache.k, cols, cols_y) if cache.cuda else None


def rope_append8(qkv: torch.Tensor, cos_sin: torch.Tensor | None, cache: Cache8, cu_q: torch.Tensor, ctx_lens: torch.Tensor,
                 block_tables: torch.Tensor, *, n_heads: int, max_q: int, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """Rotate q and k of a step and append k / v to the cache; returns the rotated queries [T, H * D] bf16 (``q_out``
    where given).

    qkv: [T, >= (H + 2 Hkv) * D] bf16, q | k | v; cos_sin: [max_pos, D/2, 2] f32 or None (no rotation), which covers every
    position (rows past its end are turned by its last entry). ``max_q`` bounds the rows of a sequence. Rotated keys
    go to their codes without a rounding in between (qkv whose rows do not start at 8 bytes is copied first). Rows at positions below zero or past the block table are not
    appended. No two sequences of a call append to the same page (a shared one ends before the first row that is not shared). An infinite or NaN entry makes its page's scale so, and with it
    what attention gives to rows that see a key of the page; rows ahead of the page and other sequences are as without it."""
    if cache.cuda:
        dev = torch._C._cuda_getDevice()
        q = kernels().rope_append8(qkv, q_out, cu_q, ctx_lens, block_tables, cos_sin, cache.k, cache.v, cache.k_scale, cache.v_scale, n_heads,
                                   cache.n_kv, cache.head_dim, cache.block_size, cache.n_blocks, max_q, cache.kind, dev, _stream(dev))
        if q is not None:
            return q
    H, G, D = n_heads, cache.n_kv, cache.head_dim
    _need(H > 0 and max_q >= 0, "n_heads and max_q")
    if cos_sin is not None:
        _typed(cos_sin, torch.float32, "cos_sin")
        _need(cos_sin.dim() == 3 and cos_sin.shape[1:] == (D // 2, 2) and cos_sin.shape[0] > 0 and cos_sin.is_contiguous()
              and cos_sin.device == cache.device and cos_sin.data_ptr() % 16 == 0, "cos_sin is [max_pos, head_dim / 2, 2], contiguous, at 16 bytes")
    _rows(qkv, (H + 2 * G) * D, "qkv", cache)
    T = qkv.shape[0]
    B, _ = _sequences(cu_q, ctx_lens, block_tables, cache)
    if q_out is None:
        q_out = torch.empty(T, H * D, dtype=torch.bfloat16, device=qkv.device)
    _rows(q_out, H * D, "q_out", cache)
    _need(q_out.shape[0] == T, "q_out has the rows of qkv")
    if T == 0 or B == 0 or max_q == 0:
        return q_out
    if not cache.cuda:
        return ref.rope_append8(qkv, cos_sin, cache, cu_q, ctx_lens, block_tables, n_heads=H, max_q=max_q, q_out=q_out)
    _need(q_out.data_ptr() % 8 == 0 and (T == 1 or q_out.stride(0) % 4 == 0), "rows of q_out must start at 8 bytes")
    if qkv.data_ptr() % 8 or (T > 1 and qkv.stride(0) % 4):
        qkv = qkv.clone(memory_format=torch.contiguous_format)
        if qkv.stride(0) % 4:
            qkv = torch.nn.functional.pad(qkv, (0, -qkv.shape[1] % 4))
        return rope_append8(qkv, cos_sin, cache, cu_q, ctx_lens, block_tables, n_heads=H, max_q=max_q, q_out=q_out)
    return _elsewhere(cache, rope_append8, qkv, cos_sin, cache, cu_q, ctx_lens, block_tables, n_heads=H, max_q=max_q, q_out=q_out)


def read8(cache: Cache8, cu_k: torch.Tensor, first: torch.Tensor, block_tables: torch.Tensor, *, total: int) -> tuple[torch.Tensor, torch.Tensor]:
    """Cached rows as what they stand for: row cu_k[b] + i of the results, k and v [total, Hkv, D] bf16, is position
    first[b] + i of sequence b (a prefix that moves to a bf16 cache, or is looked at). Zeros from pages that do not exist;
    rows of no sequence are zeros too."""
    if cache.cuda:
        dev = torch._C._cuda_getDevice()
        kv = kernels().read8(cu_k, first, block_tables, cache.k, cache.v, cache.k_scale, cache.v_scale, cache.n_kv, cache.head_dim, cache.block_size,
                             cache.n_blocks, total, cache.kind, dev, _stream(dev))
        if kv is not None:
            return kv
    B, _ = _sequences(cu_k, first, block_tables, cache)
    _need(0 <= total < 1 << 31, "total")
    if cache.cuda and total > 0 and B > 0:
        return _elsewhere(cache, read8, cache, cu_k, first, block_tables, total=total)
    k, v = (torch.zeros(total, cache.n_kv, cache.head_dim, dtype=torch.bfloat16, device=cache.device) for _ in range(2))
    return (k, v) if cache.cuda else ref.read8(cache, cu_k, first, block_tables, k, v)


@functools.lru_cache(maxsize=4096)
def attn8_plan(max_q: int, group: int, units: int, keys: int, D: int) -> tuple[int, int, int, int, int]:
    """(form: 0 prompts, else tiles of 16 rows of a token step; parts of a sequence's keys at most; tiles of 64 keys of a prompt's part or
    stages of a token's ring; floats of workspace; tickets) for ``units`` (sequence, kv head) pairs of up to ``max_q`` rows, ``group`` heads
    and ``keys`` keys."""
    rows = max_q * group
    if rows <= 16:
        return _token_plan(1, rows, units, keys, D)
    if rows <= 32:
        return _token_plan(2, rows, units, keys, D)
    return _prompt_plan(rows, units, keys, D)


def _token_plan(form: int, rows: int, units: int, keys: int, D: int) -> tuple[int, int, int, int, int]:
    # Two workgroups for each compute unit, no part of less than a tile for each wave, and, since a unit's parts are joined by one of
    # them, about the square root of its keys. us by parts, heads of 128 (contexts x keys x kv heads): 16 x 4000 x 8 39.4 (1), 31.7
    # (2), 33.7 (3), 31.2 (4), 35.7 (6); 12 x 4000 x 8 37.9 (1), 26.4 (2), 30.6 (3), 26.7 (4), 30.1 (6); 24 x 4000 x 8 45.9 (1), 46.7
    # (2), 32 of them 56.1 (1), 56.8 (2); 1 x 2000 x 8 of 8 rows 20.5 (1), 11.5 (4), 9.9 (8), 9.4 (16), of 32 rows 26.7, 17.8, 16.1,
    # 19.2; 1 x 30000 x 8 of 8 rows 25.4 (16), 22.8 (24), 23.0 (32), 25.1 (48), of 32 rows 37.1, 35.8, 37.1, 45.2; 64 columns: 1 x
    # 20000 x 1 of 5 rows 15.4 (16), 12.9 (24), 12.7 (32), 11.6 (48); 32 x 4000 x 8 34.8 (1), 30.4 (2), 31.1 (4). Many rows of few keys: 1
    # x 300 x 8 of 32 rows 10.1 (1), 12.8 (3), 8 x 700 14.7 (1), 16.0 (4), 8 x 1500 22.4 (1), 20.3 (2), 20.5 (6)
    parts, few = SLOTS // units, rows * D <= 1024
    if D == 128 and parts < 3:
        parts = 1
    parts = max(1, min(parts, -(-keys // 128), max(math.isqrt(keys // 8), 16) if few else math.isqrt(keys // 32) if keys > 768 else 1,
                       48 if D == 64 else 32))
    return (form, parts, 1 if keys <= 128 * parts else 2, *((units * parts * 16 * form * (D + 2), units) if parts > 1 else (0, 0)))


def _prompt_plan(rows: int, units: int, keys: int, D: int) -> tuple[int, int, int, int, int]:
    blocks, most = -(-rows // PROMPT_ROWS), max(1, -(-keys // 64))
    # parts of four tiles at least, about the square root of the keys as above. us by parts: 1 x 30000 keys x 8 kv heads of 128 columns, 48
    # rows 657 (1), 97 (8), 62 (16), 53 (24), 51.3 (30 and 32); 1 x 4000 85 (1), 24.0 (8), 23.4 (12), 23.9 (16), 31 (32); 1 x 700 21 (1),
    # 14.8 (4), 17.1 (12); 3 x 113 rows x 4 behind 5000 x 8 of 64 82 (1), 42 (4), 36 (5), 41 (6), 35 (8); 1024 x 4 causal rows x 8 of 64
    # 21.5 (1), 19.6 (2), 22.3 (3), of 128 29.0, 28.0, 29.8
    parts = max(1, min(SLOTS // (units * blocks), most // 4, math.isqrt(keys // 32), 32))
    return (0, parts, -(-most // parts), units * blocks * parts * PROMPT_ROWS * (D + 4), units * blocks) if parts > 1 else (0, 1, most, 0, 0)


def attention8(q: torch.Tensor, cache: Cache8, cu_q: torch.Tensor, ctx_lens: torch.Tensor, block_tables: torch.Tensor, *, n_heads: int,
               max_q: int, max_k: int | None = None, causal: bool = True, scale: float | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """Varlen attention off the 8-bit cache: token steps, prompts and prompt chunks behind cached tokens.

    q: [T, >= H * D] bf16 (row stride may exceed H * D). Query i of a sequence of n rows sees the keys up to position
    ctx - n + i (all ctx of them where not ``causal``). ``max_q`` bounds the rows of a sequence, ``max_k``
    its context where the host knows a smaller bound than the block table's (it only chooses the split of the keys: in
    how many parts they are summed up follows from the whole call). ``scale`` is 1 / sqrt(D) by default. Rows that see no
    key give zeros. The longest feed chooses one form and one split for all of a call: replies of a token beside a chunk of a prompt run as
    prompts, each walking its keys alone (us: eight replies of 4000 keys beside 512 rows 113, in two calls 38; one of 100000 keys beside
    them 1080, in two 62), so a program that knows its lengths calls once for each. Returns [T, H * D] bf16 (``out`` where given)."""
    H, G, D = n_heads, cache.n_kv, cache.head_dim
    _need(H > 0 and H % G == 0, "n_heads must be a multiple of the cache's heads")
    _need(max_q >= 0 and (max_k is None or max_k >= 0), "max_q and max_k")
    scale = D ** -0.5 if scale is None else float(scale)
    fast = _rows8(q, out, cu_q, ctx_lens, block_tables, cache, H * D, H * D)
    if fast is None:
        _rows(q, H * D, "q", cache)
        T = q.shape[0]
        B, _ = _sequences(cu_q, ctx_lens, block_tables, cache)
        if out is None:
            out = torch.empty(T, H * D, dtype=torch.bfloat16, device=q.device)
        _rows(out, H * D, "out", cache)
        _need(out.shape[0] == T, "out has the rows of q")
        return out if T == 0 or B == 0 or max_q == 0 else \
            ref.attention8(q, cache, cu_q, ctx_lens, block_tables, n_heads=H, max_q=max_q, causal=causal, scale=scale, out=out)
    T, B, max_blocks, ldq, ldo, out, dev = fast
    if max_q == 0:
        return out
    keys = max_blocks * cache.block_size if max_k is None else min(max_k, max_blocks * cache.block_size)
    max_q = min(max_q, T)
    form, parts, each, floats, tiles = attn8_plan(max_q, H // G, B * G, max(keys, 1), D)
    st = _stream(dev)
    with _there(dev):
        ws, tickets = _sk_workspace(q.device, st, floats, tiles) if parts > 1 else (None, None)
        check(kernels().loqa_attention8(
            q, ldq, cache.k, cache.v, cache.k_scale, cache.v_scale, cu_q, ctx_lens, block_tables, out, ldo, T, B, H, G, D, cache.block_size,
            cache.n_blocks, max_blocks, max_q, scale, int(causal), cache.kind, form, parts, each, ws, 0 if ws is None else ws.numel(), tickets,
            0 if tickets is None else tickets.numel(), st), "attention8")
    return out


# ------------------------------------------------------------------ pages of a step
PAGE_STEP_SEQS, PAGE_STEP_FEW = 4096, 512


class PageStep(NamedTuple):
    """What a step's launches want of its sequences (int32 but for ``last_rows``): ``positions`` and ``slots`` [max_tokens]
    (0 and -1 behind the last token), ``cu_q`` [B + 1], ``last_rows`` [B] int64 (the row of a sequence's last token, 0
    where it has none), ``ctx_lens`` [B] with this step's tokens, ``ring`` [2], and ``status`` [1]: 0, or the sum of
    1 (not enough free pages), 2 (more tokens than max_tokens), 4 (a sequence outgrows its table), 8 (numbers that no pool has)."""
    cu_q: torch.Tensor
    positions: torch.Tensor
    slots: torch.Tensor
    last_rows: torch.Tensor
    ctx_lens: torch.Tensor
    ring: torch.Tensor
    status: torch.Tensor


def page_step(new_lens: torch.Tensor, ctx_lens: torch.Tensor, block_tables: torch.Tensor, free_pages: torch.Tensor, ring: torch.Tensor, *,
              block_size: int, max_tokens: int, ctx_out: torch.Tensor | None = None, ring_out: torch.Tensor | None = None) -> PageStep:
    """The pages and slots of a step, on the GPU: what the host pool's ``step_meta`` does, for loops that never
    come back to the host (a captured step whose lengths live on the GPU).

    new_lens [B]: tokens of each sequence in this step (0: none; -1: the sequence has ended, and its pages go back);
    ctx_lens [B]: its tokens before; block_tables [B, max_blocks]: its pages, to which new ones are added in place;
    free_pages [N]: a ring of free pages, ``ring`` [2] = (place of the first, how many). Pages are taken in the order of the
    sequences and given back behind the last free one. ``ctx_out`` / ``ring_out`` may be ``ctx_lens`` / ``ring`` themselves.
    All or nothing: where the status is not 0, nothing changes and no token has a slot. At most 4096 sequences. A page that
    several sequences share must not be given back here."""
    if block_tables.is_cuda:
        dev = torch._C._cuda_getDevice()
        st = _stream(dev)
        # what several workgroups share; the few tokens of a decoding step take one
        tickets = _sk_workspace(block_tables.device, st, 1, 1)[1] if max_tokens > PAGE_STEP_FEW and block_tables.get_device() == dev else None
        step = kernels().page_step(new_lens, ctx_lens, block_tables, free_pages, ring, ctx_out, ring_out, tickets, block_size, max_tokens,
                                   PAGE_STEP_SEQS, dev, st)
        if step is not None:
            return PageStep._make(step)
    _typed(block_tables, torch.int32, "block_tables")
    for t, name in ((new_lens, "new_lens"), (ctx_lens, "ctx_lens"), (block_tables, "block_tables"), (free_pages, "free_pages"), (ring, "ring"),
                    (ctx_out, "ctx_out"), (ring_out, "ring_out")):
        if t is not None:
            _i32(t, name, block_tables)
    B, pool = new_lens.numel(), free_pages.numel()
    _need(0 < B <= PAGE_STEP_SEQS, f"1 to {PAGE_STEP_SEQS} sequences")
    _need(ctx_lens.numel() == B and block_tables.dim() == 2 and block_tables.shape[0] == B and block_tables.shape[1] > 0, "ctx_lens [B], block_tables [B, max_blocks]")
    _need(ring.numel() == 2 and pool > 0, "ring [2], free_pages [N]")
    _need(block_size > 0 and block_size & (block_size - 1) == 0 and pool * block_size < 1 << 31, "block_size is a power of two, slots have 32 bits")
    _need(0 <= max_tokens <= 1 << 30, "max_tokens")
    for t, n, name in ((ctx_out, B, "ctx_out"), (ring_out, 2, "ring_out")):
        _need(t is None or t.numel() == n, f"{name} has {n} entries")
    if block_tables.is_cuda:
        with torch.cuda.device(block_tables.device):
            _need(block_tables.get_device() != dev, "page_step does not take this call")
            return page_step(new_lens, ctx_lens, block_tables, free_pages, ring, block_size=block_size, max_tokens=max_tokens, ctx_out=ctx_out, ring_out=ring_out)
    ints = functools.partial(torch.empty, dtype=torch.int32)
    step = PageStep(ints(B + 1), ints(max_tokens), ints(max_tokens), torch.empty(B, dtype=torch.int64), ints(B) if ctx_out is None else ctx_out,
                    ints(2) if ring_out is None else ring_out, ints(1))
    return ref.page_step(new_lens, ctx_lens, block_tables, free_pages, ring, block_size, step)


# ------------------------------------------------------------------ 4-bit weights
GROUPS = (32, 64, 128)


def quantize4(w: torch.Tensor, group: int = 128, zeros: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """A matrix [N, K] in 4 bits, to nearest: (codes [N, K / 2] uint8, two a byte with the lower column in the lower half;
    scales [N, K / group] bf16; zeros [N, K / group] uint8 or None: 8) with w ~ (code - zero) * scale."""
    _need(w.dim() == 2 and group in GROUPS and w.shape[1] % group == 0, f"[N, K] with K a multiple of the group, one of {GROUPS}")
    x = w.float().reshape(w.shape[0], -1, group)
    z = None
    if zeros:
        lo, hi = x.amin(-1).clamp_max(0), x.amax(-1).clamp_min(0)
        s = ((hi - lo) / 15).to(torch.bfloat16)
        sf = torch.where(s > 0, s, torch.ones_like(s)).float()
        z = (-lo / sf).round().clamp(0, 15).to(torch.uint8)
        c = (x / sf[..., None]).round() + z[..., None]
    else:
        s = (x.abs().amax(-1) / 7).to(torch.bfloat16)
        sf = torch.where(s > 0, s, torch.ones_like(s)).float()
        c = (x / sf[..., None]).round() + 8
    c = c.clamp(0, 15).to(torch.uint8).reshape(w.shape)
    return c[:, 0::2] | c[:, 1::2] << 4, s, z


class Weight4:
    """A weight matrix [N, K] in 4 bits for :func:`linear4`: codes, scales and zeros as :func:`quantize4` returns them
    (zeros up to 15; group 32, 64 or 128 by their shapes), laid out once for the kernel. The tensors given are not kept on the GPU."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, zeros: torch.Tensor | None = None):
        _typed(codes, torch.uint8, "codes")
        _typed(scales, torch.bfloat16, "scales")
        _need(codes.dim() == 2 and scales.dim() == 2 and scales.shape[0] == codes.shape[0], "codes [N, K / 2], scales [N, K / group]")
        self.n, self.k = codes.shape[0], codes.shape[1] * 2
        groups = scales.shape[1]
        _need(self.n > 0 and groups > 0 and self.k % groups == 0 and self.k // groups in GROUPS, f"groups of {GROUPS}")
        self.group = self.k // groups
        if zeros is not None:
            _typed(zeros, torch.uint8, "zeros")
            _need(zeros.shape == scales.shape, "zeros have the shape of scales")
        _need(all(t is None or t.device == codes.device for t in (scales, zeros)), "tensors of one device")
        self.cuda = codes.is_cuda
        codes, scales = codes.contiguous(), scales.contiguous()
        zeros = None if zeros is None else zeros.contiguous()
        if not codes.is_cuda:
            self.codes, self.scales, self.zeros = codes, scales, zeros
            return
        tiles, blocks = -(-self.n // 16), -(-self.k // 128)
        self.codes = torch.empty(tiles * blocks * 256, dtype=torch.int32, device=codes.device)
        padded = tiles * blocks * (128 // self.group) * 16
        self.scales = torch.empty(padded, dtype=torch.bfloat16, device=codes.device)
        self.zeros = None if zeros is None else torch.empty(padded, dtype=torch.uint8, device=codes.device)
        with _there(codes.get_device()):
            check(kernels().loqa_shuffle4(ptr(codes), ptr(scales), ptr(zeros), ptr(self.codes), ptr(self.scales), ptr(self.zeros), self.n, self.k,
                                          self.group, stream_ptr(codes)), "shuffle4")

    @classmethod
    def quantize(cls, w: torch.Tensor, group: int = 128, zeros: bool = False) -> "Weight4":
        return cls(*quantize4(w, group, zeros))

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.codes, self.scales, self.zeros) if t is not None)


@functools.lru_cache(maxsize=4096)
def linear4_plan(M: int, N: int, K: int) -> tuple[int, int, int, int]:
    """(tiles of 16 features a wave of the kernel for more rows, or 0: the one for few rows; parts of K; floats of workspace,
    tickets) of a product of M rows with an [N, K] weight."""
    # us, few rows' kernel and the other, cold weights: 32 x 512 x 8192 17.3, 7.3; 32 x 4096 x 14336 30.8, 14; 32 x 28672 x 4096
    # 29.7, 24; 24 x 10240 x 2048 9.7, 8.6; 18 x 4096 x 4096 9.0, 8.0; 24 x 2048 x 2048 6.2, 5.9; 20 x 4096 x 2048 5.9, 6.5; 32 x 256 x
    # 512 3.4, 5.0
    if M <= 16 or (M <= 32 and K <= 2048 and N <= 4096):
        return 0, 1, 0, 0
    # one and two tiles a wave: 64 x 28672 x 4096 42, 37, 32 rows 25.2, 24; 64 x 24368 x 2144 20.6, 20.6; 40 x 16384 x 2048 13.1, 15.2; 17 x
    # 8192 x 4096 10.4, 11.5; 64 x 4096 x 4096 10.6, 13
    features = 2 if N >= 24576 else 1
    # two workgroups for each compute unit, and no part of less than two blocks of 128 columns: 64 x 4096 x 4096 22.4 (1), 11.1
    # (4), 10.6 (8), 15.4 (16); 20 x 3584 x 13696 47 (1), 17 (4), 13.5 (9), 14.8 (16); 64 x 14336 x 4096 24.5 (1), 20.0 (2), 23 (4)
    rows, blocks = 32 if M <= 32 else 64, -(-K // 128)
    units = -(-N // (64 * features)) * -(-M // rows)
    parts = max(1, min(512 // units, blocks // 2, 16))
    parts = -(-blocks // -(-blocks // parts))
    return (features, parts, units * parts * 64 * features * rows, units) if parts > 1 else (features, 1, 0, 0)


def linear4(x: torch.Tensor, w: Weight4, b: torch.Tensor | None = None) -> torch.Tensor:
    """x [..., K] bf16 times the transpose of a 4-bit weight (+ bias [N] bf16): [..., N] bf16, summed up in f32. Made for
    the few rows of token steps; more than 64 read the weight again for every 64. Rows that do not start at 16 bytes, and x of
    other than two dimensions, are copied first. An infinite or NaN entry of x makes its row NaN, and so may
    one past 2^112 (sums of 143 times a group's entries stay within f32 up to there)."""
    fast = None
    if w.cuda:
        dev = torch._C._cuda_getDevice()
        fast = kernels().linear4_rows(x, w.codes, w.scales, w.zeros, b, w.n, w.k, w.group, dev, _stream(dev))
        if type(fast) is torch.Tensor:
            return fast
    if fast is None:
        _typed(x, torch.bfloat16, "x")
        _need(x.dim() >= 1 and x.shape[-1] == w.k, f"x has {w.k} columns")
        _need(x.device == w.codes.device, f"x must be on {w.codes.device}")
        if b is not None:
            _typed(b, torch.bfloat16, "b")
            _need(b.shape == (w.n,) and b.is_contiguous() and b.device == x.device, f"b is [{w.n}], contiguous")
        if not w.cuda:
            return ref.linear4(x, w, b)
        if x.numel() == 0:
            return x.new_empty(*x.shape[:-1], w.n)
        rows = x.reshape(-1, w.k).clone(memory_format=torch.contiguous_format)     # whole rows at 16 bytes
        return linear4(rows, w, b).view(*x.shape[:-1], w.n)
    M, ld, y, dev = fast
    features, parts, floats, tiles = linear4_plan(M, w.n, w.k)
    st = _stream(dev)
    with _there(dev):
        ws, tickets = _sk_workspace(x.device, st, floats, tiles) if parts > 1 else (None, None)
        check(kernels().loqa_linear4(x, ld, w.codes, w.scales, w.zeros, b, y, w.n, M, w.n, w.k, w.group, features, parts, ws,
                                     0 if ws is None else ws.numel(), tickets, 0 if tickets is None else tickets.numel(), st), "linear4")
    return y

"""Plain 64-bit forms of ``ops.lowbit`` from its definitions, on the CPU, and what its kernels may be off by."""
import math

import torch

F64 = torch.float64


def entries(codes, scale):
    """Codes [n, G, P, D] and scales [n, G] as values."""
    return codes.cpu().to(torch.float32).to(F64) * scale.cpu().to(F64).clamp_min(2.0 ** -100)[..., None, None]


def attention(q, cache, cu_q, ctx_lens, block_tables, n_heads, scale=None, causal=True):
    """(o, sum of |weight * value|) [T, H * D]; rows of no sequence are zeros."""
    H, G, D, P = n_heads, cache.n_kv, cache.head_dim, cache.block_size
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    q, cu, ctx, bt = q.cpu(), cu_q.tolist(), ctx_lens.tolist(), block_tables.cpu().long()
    k8, v8 = (t.cpu() for t in (cache.k, cache.v))
    ks, vs = (t.cpu().to(F64).clamp_min(2.0 ** -100) for t in (cache.k_scale, cache.v_scale))
    o, mag = (torch.zeros(q.shape[0], H * D, dtype=F64) for _ in range(2))
    for b in range(len(ctx)):
        q0, n = cu[b], cu[b + 1] - cu[b]
        L = min(max(ctx[b], 0), P * bt.shape[1])
        pos = torch.arange(L)
        pages = bt[b, pos // P]
        ok = (pages >= 0) & (pages < cache.n_blocks)
        pages = pages.clamp(0, cache.n_blocks - 1)
        hide = ~ok[None] | (pos[None] > ctx[b] - n + torch.arange(n)[:, None] if causal else torch.zeros(n, 1, dtype=torch.bool))
        for h in range(H):
            g = h // (H // G)
            k = k8[pages, g, pos % P].float().to(F64) * ks[pages, g, None]
            v = torch.where(ok[:, None], v8[pages, g, pos % P].float().to(F64) * vs[pages, g, None], 0.0)
            w = (q[q0:q0 + n, h * D:(h + 1) * D].to(F64) @ k.t() * scale).masked_fill(hide, -math.inf)
            seen = (~hide).any(1, keepdim=True).expand(n, 1) if L else torch.zeros(n, 1, dtype=torch.bool)
            p = torch.softmax(torch.where(seen, w, 0.0), -1) * seen if L else torch.zeros(n, 0, dtype=F64)
            o[q0:q0 + n, h * D:(h + 1) * D] = p @ v
            mag[q0:q0 + n, h * D:(h + 1) * D] = p @ v.abs()
    return o, mag


def attention_bound(o, mag):
    """The result's rounding to bf16 (2^-8 of it); weights rounded to f16 (2^-11 of each) and all that f32 does - scores up
    to 2^6 off by 2^-21 of that, exponentials and sums by 2^-20 - within another 2^-14 of the magnitudes; a weight under
    2^-14 of the largest one is off by 2^-25, less than 2^-11 of the magnitudes for up to 2^14 keys of like scales."""
    return 2.0 ** -8 * o.abs() + (2.0 ** -11 + 2.0 ** -14) * mag + 1e-30


def linear4_bound(y, x, w, scales):
    """The result's rounding, and the f32 sums of 143 |x| s: some ten roundings an MFMA of 32 columns, one a
    group, one a wave."""
    K, group = x.shape[1], x.shape[1] // scales.shape[1]
    terms = x.abs().to(F64) @ scales.abs().to(F64).repeat_interleave(group, 1).t() * 143
    return 2.0 ** -8 * y.abs() + 2.0 ** -24 * (group / 32 * 10 + K / group + 16) * terms

"""``ops.lowbit``: the paged 8-bit cache and what writes and reads it, pages handed out on the GPU, 4-bit products."""
import math
import threading

import pytest
import torch

import lowbit_oracle as oracle
from loqa_hub_amd import ops
from loqa_hub_amd.ops import lowbit
from loqa_hub_amd.ops import reference as ref

BF16, I32, F64 = torch.bfloat16, torch.int32, torch.float64
INT8, E4M3 = torch.int8, torch.float8_e4m3fn
DEVICES = [pytest.param("cpu"), pytest.param("cuda", marks=pytest.mark.gpu)]
KINDS = pytest.mark.parametrize("dtype", [INT8, E4M3], ids=["int8", "e4m3"])


def _i(x, dev="cpu"):
    return torch.tensor(x, dtype=I32, device=dev)


def _cu(feeds, dev="cpu"):
    return _i([sum(feeds[:i]) for i in range(len(feeds) + 1)], dev)


def _tables(ctx, page, extra=3, seed=0, width=None):
    """Scattered pages for contexts of these lengths: (how many pages there are, the table)."""
    needs = [-(-c // page) for c in ctx]
    pool = sum(needs) + extra
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(I32)
    bt = torch.zeros(len(ctx), max(1, max(needs)) if width is None else width, dtype=I32)
    at = 0
    for b, n in enumerate(needs):
        bt[b, :n] = order[at:at + n]
        at += n
    return pool, bt


def _filled(pool, G, page, D, dtype, seed=0):
    """A CPU cache with pages of unlike scales."""
    g = torch.Generator().manual_seed(seed + 99)
    parts = []
    for _ in range(2):
        x = torch.randn(pool, G, page, D, generator=g) * (0.2 + 3 * torch.rand(pool, G, 1, 1, generator=g) ** 3) * (0.3 + torch.rand(1, G, 1, D, generator=g))
        s = ref.page_scale8(x.abs().amax((2, 3)), dtype)
        parts += [ref.codes8(x / s[..., None, None], dtype), s]
    return lowbit.Cache8(parts[0], parts[2], parts[1], parts[3])


def _to(cache, dev):
    """A copy on a device (8-bit floats by their bytes)."""
    return lowbit.Cache8(*(t.view(torch.uint8).to(dev, copy=True).view(cache.k.dtype) for t in (cache.k, cache.v)),
                         *(t.to(dev, copy=True) for t in (cache.k_scale, cache.v_scale)))


def _same(a, b):
    for n in ("k", "v"):
        assert torch.equal(getattr(a, n).cpu().view(torch.uint8), getattr(b, n).cpu().view(torch.uint8)), n
    for n in ("k_scale", "v_scale"):
        assert torch.equal(getattr(a, n).cpu(), getattr(b, n).cpu()), n


# ------------------------------------------------------------------ append
def _append_case(feeds, pasts, H, G, D, page, dtype, rope=True, seed=0, pad=0, spare=0):
    g = torch.Generator().manual_seed(seed)
    ctx = [a + b for a, b in zip(feeds, pasts)]
    pool, bt = _tables(ctx, page, seed=seed)
    cache = _filled(pool, G, page, D, dtype, seed)
    T = sum(feeds) + pad
    qkv = torch.randn(T, (H + 2 * G) * D + spare, generator=g)
    qkv[:, (H + G) * D:] *= (0.1 + 4 * torch.rand(T, 1, generator=g) ** 4)
    if pad:
        qkv[-pad:] = math.nan
    cs = ref.rope_cos_sin(D, max(max(ctx), 1), 10000.0) if rope else None
    return qkv.to(BF16), cs, cache, _cu(feeds), _i(ctx), bt


APPENDS = [((1,) * 5, (0, 15, 16, 17, 40), 8, 2, 128, 16), ((7,), (0,), 4, 4, 64, 16), ((33, 1, 0, 18), (3, 31, 9, 0), 4, 1, 128, 32),
           ((130,), (5,), 2, 2, 64, 64), ((16, 32), (16, 0), 5, 1, 64, 16), ((3,), (200,), 6, 2, 128, 128)]


@KINDS
@pytest.mark.parametrize("feeds,pasts,H,G,D,page", APPENDS)
@pytest.mark.parametrize("rope", [True, False])
def test_append_by_definition(feeds, pasts, H, G, D, page, dtype, rope):
    """The codes of the reference against 64 bits: every row within half a step of its page's scale, scales by their formula."""
    qkv, cs, cache, cu, ctx, bt = _append_case(feeds, pasts, H, G, D, page, dtype, rope)
    before = _to(cache, "cpu")
    q = lowbit.rope_append8(qkv, cs, cache, cu, ctx, bt, n_heads=H, max_q=max(feeds))
    x = qkv.to(F64).view(-1, H + 2 * G, D)
    most, eps = (127, 2.0 ** -21) if dtype is INT8 else (448, 2.0 ** -21)
    touched = torch.zeros(cache.n_blocks, dtype=torch.bool)
    for b, (n, past) in enumerate(zip(feeds, pasts)):
        if n == 0:
            continue
        rows = x[int(cu[b]):int(cu[b]) + n].clone()
        if rope:
            c, s = cs[past:past + n].to(F64)[:, None].unbind(-1)
            lo, hi = rows[:, :H + G, :D // 2].clone(), rows[:, :H + G, D // 2:].clone()
            rows[:, :H + G, :D // 2], rows[:, :H + G, D // 2:] = lo * c - hi * s, hi * c + lo * s
        err = (q[int(cu[b]):int(cu[b]) + n].to(F64).view(n, H, D) - rows[:, :H]).abs()
        assert (err <= 2.0 ** -8 * rows[:, :H].abs() + 2.0 ** -20).all()
        for p in range(past // page * page, past + n, page):
            id_ = int(bt[b, p // page])
            touched[id_] = True
            first, last = max(past, p), min(past + n, p + page)
            for codes, scale, old_codes, old_scale, new in ((cache.k, cache.k_scale, before.k, before.k_scale, rows[:, H:H + G]),
                                                            (cache.v, cache.v_scale, before.v, before.v_scale, rows[:, H + G:])):
                new = new[first - past:last - past].transpose(0, 1)
                need = new.abs().amax((1, 2)) / most
                if dtype is E4M3:
                    need = torch.exp2(torch.ceil(torch.log2(need)))
                had = old_scale[id_].to(F64)
                want = torch.maximum(need, had) if first > p else need
                now = scale[id_].to(F64)
                assert ((now - want).abs() <= 2.0 ** -22 * want).all()
                kept = old_codes[id_, :, :first - p].float().to(F64) * had[:, None, None]
                body = torch.cat([kept, new], 1)
                got = codes[id_, :, :last - p].float().to(F64) * now[:, None, None]
                step = now[:, None, None] * (0.5 if dtype is INT8 else 2.0 ** -10)
                half = step if dtype is INT8 else torch.maximum(step.expand_as(body), 2.0 ** -4 * body.abs())
                assert ((got - body).abs() <= half + now[:, None, None] * most * eps).all()
                untouched = codes.view(torch.uint8)[id_, :, last - p:]
                assert torch.equal(untouched, old_codes.view(torch.uint8)[id_, :, last - p:])
    for a, b in ((cache.k, before.k), (cache.v, before.v)):
        assert torch.equal(a.view(torch.uint8)[~touched], b.view(torch.uint8)[~touched])


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("feeds,pasts,H,G,D,page", APPENDS + [((700, 3, 90), (0, 4000, 77), 32, 8, 128, 16), ((1,) * 33, tuple(range(33)), 16, 4, 64, 16)])
@pytest.mark.parametrize("rope", [True, False])
def test_append_kernel_is_the_reference(feeds, pasts, H, G, D, page, dtype, rope):
    """Codes, scales and queries bit for bit; padding rows (NaN) touch nothing."""
    case = _append_case(feeds, pasts, H, G, D, page, dtype, rope, pad=3, spare=8)
    qkv, cs, cache, cu, ctx, bt = case
    there = [None if t is None else t.cuda() for t in (qkv, cs, cu, ctx, bt)]
    dev = _to(cache, "cuda")
    q_out = torch.full((qkv.shape[0], H * D + 4), 7.0, dtype=BF16)
    q_dev = q_out.cuda()
    a = lowbit.rope_append8(there[0], there[1], dev, *there[2:], n_heads=H, max_q=max(feeds), q_out=q_dev)
    b = lowbit.rope_append8(qkv, cs, cache, cu, ctx, bt, n_heads=H, max_q=max(feeds), q_out=q_out)
    assert a is q_dev and torch.equal(a.cpu(), b) and (b[-3:] == 7).all() and (b[:, H * D:] == 7).all()
    _same(dev, cache)
    lowbit.rope_append8(there[0], there[1], dev, *there[2:], n_heads=H, max_q=max(feeds))        # the same rows again change nothing
    _same(dev, cache)
    # rows at odd places, of an odd width
    odd = torch.empty(qkv.shape[0], qkv.shape[1] + 1, dtype=BF16, device="cuda")[:, 1:]
    odd.copy_(qkv)
    again = lowbit.rope_append8(odd, there[1], dev, *there[2:], n_heads=H, max_q=max(feeds))
    rows = sum(feeds)
    assert torch.equal(again[:rows].cpu(), b[:rows, :H * D])
    _same(dev, cache)


@KINDS
@pytest.mark.parametrize("dev", DEVICES)
def test_pages_filled_row_by_row(dtype, dev):
    """Every growth of a scale rounds older rows once more: up to sixteen half steps of scales up to the final one for int8, one
    rounding for e4m3 but at its smallest entries; and read8's own rounding."""
    G, D, P = 2, 64, 16
    cache = lowbit.Cache8.empty(3, G, P, D, dtype, dev)
    x = torch.randn(20, (1 + 2) * G * D, generator=torch.Generator().manual_seed(5)) * torch.linspace(0.05, 2, 20)[:, None]
    x = x.to(BF16)
    bt = _i([[2, 0]], dev)
    for i in range(20):
        lowbit.rope_append8(x[i:i + 1].to(dev), None, cache, _i([0, 1], dev), _i([i + 1], dev), bt, n_heads=G, max_q=1)
    k, v = lowbit.read8(cache, _i([0, 20], dev), _i([0], dev), bt, total=20)
    s = torch.stack([cache.k_scale.cpu()[[2, 0]], cache.v_scale.cpu()[[2, 0]]])            # [2, page, G]
    for got, want, sc in ((k, x[:, G * D:2 * G * D], s[0]), (v, x[:, 2 * G * D:], s[1])):
        got, want = got.cpu().to(F64), want.to(F64).view(20, G, D)
        step = sc.to(F64).repeat_interleave(16, 0)[:20, :, None]
        if dtype is INT8:
            bound = 8 * step + 2.0 ** -8 * (want.abs() + 8 * step)
        else:
            bound = torch.maximum((2.0 ** -4 + 2.0 ** -8 * 1.0625) * want.abs(), 16 * step * 2.0 ** -10 * (1 + 2.0 ** -8))
        assert ((got - want).abs() <= bound).all()


@KINDS
@pytest.mark.parametrize("dev", DEVICES)
def test_append_at_the_edges(dtype, dev):
    """Zeros, tiny rows, pages that do not exist, rows without a place, feeds past max_q, values that are no numbers."""
    G, D, P = 1, 64, 16
    cache = _to(_filled(4, G, P, D, dtype), dev)
    before = _to(cache, "cpu")
    rows = torch.ones(6, 3 * D, dtype=BF16, device=dev)
    cu = _i([0, 2, 4, 6], dev)
    # a page past the cache, a negative one, a context shorter than the feed (one row has a place)
    lowbit.rope_append8(rows, None, cache, cu, _i([2, 2, 1], dev), _i([[4], [-1], [3]], dev), n_heads=1, max_q=2)
    for name in ("k", "v"):
        now, was = getattr(cache, name).cpu().float(), getattr(before, name).float()
        assert torch.equal(now[:3], was[:3]) and torch.equal(now[3, :, 1:], was[3, :, 1:])
    k, _ = lowbit.read8(cache, _i([0, 1], dev), _i([0], dev), _i([[3]], dev), total=1)
    assert (k.cpu().float() == 1).all()
    # contexts of zero and past the table, a table column short
    lowbit.rope_append8(rows, None, cache, _i([0, 0, 6], dev), _i([0, 18], dev), _i([[0], [3]], dev), n_heads=1, max_q=6)
    assert torch.equal(cache.k[:3].cpu().float(), before.k[:3].float()) and (lowbit.read8(cache, _i([0, 16], dev), _i([0], dev), _i([[3]], dev), total=16)[0][12:] == 1).all()
    # all zeros, and rows below any scale
    for x in (0.0, 2.0 ** -120):
        lowbit.rope_append8(torch.full((2, 3 * D), x, dtype=BF16, device=dev), None, cache, _i([0, 2], dev), _i([2], dev), _i([[1]], dev), n_heads=1, max_q=2)
        assert cache.k_scale[1].item() == 2.0 ** -100 and (cache.k[1, :, :2].cpu().float() == 0).all()
    # max_q cuts a feed: its first row only
    was = cache.v[2].cpu().float()
    lowbit.rope_append8(rows, None, cache, _i([0, 6], dev), _i([6], dev), _i([[2]], dev), n_heads=1, max_q=1)
    assert torch.equal(cache.v[2, :, 1:].cpu().float(), was[:, 1:])
    assert cache.v_scale[2].item() == (torch.tensor(1.0) / 127 if dtype is INT8 else torch.tensor(2.0 ** -8)).item()
    # no numbers: the scale says so
    for x in (math.inf, math.nan):
        bad = torch.ones(2, 3 * D, device=dev)
        bad[1, D + 3] = x
        lowbit.rope_append8(bad.to(BF16), None, cache, _i([0, 2], dev), _i([2], dev), _i([[0]], dev), n_heads=1, max_q=2)
        assert not math.isfinite(cache.k_scale[0].item()) and math.isfinite(cache.v_scale[0].item())
        q = torch.ones(1, D, dtype=BF16, device=dev)
        assert lowbit.attention8(q, cache, _i([0, 1], dev), _i([2], dev), _i([[0]], dev), n_heads=1, max_q=1).isnan().all()
    # a new row at the page's first place starts it anew
    lowbit.rope_append8(torch.ones(1, 3 * D, dtype=BF16, device=dev), None, cache, _i([0, 1], dev), _i([1], dev), _i([[0]], dev), n_heads=1, max_q=1)
    assert math.isfinite(cache.k_scale[0].item())


@KINDS
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("D,P", [(64, 16), (128, 64)])
def test_read(dtype, dev, D, P):
    G = 3
    ctx = [70, 1, 0, 33]
    pool, bt = _tables(ctx, P)
    cpu = _filled(pool, G, P, D, dtype)
    bt[3, -1] = pool                                  # a page that does not exist (where that context has as many)
    first, ns = [5, 0, 0, 1], [60, 1, 0, 32]
    want = torch.zeros(sum(ns), 2, G, D, dtype=F64)
    at = 0
    for b, n in enumerate(ns):
        for i in range(n):
            pos = first[b] + i
            p = int(bt[b, pos // P])
            if p < pool:
                want[at + i, 0] = cpu.k[p, :, pos % P].float().to(F64) * cpu.k_scale[p].to(F64)[:, None]
                want[at + i, 1] = cpu.v[p, :, pos % P].float().to(F64) * cpu.v_scale[p].to(F64)[:, None]
        at += n
    k, v = lowbit.read8(_to(cpu, dev), _cu(ns, dev), _i(first, dev), bt.to(dev), total=sum(ns) + 3)
    for got, w in ((k, want[:, 0]), (v, want[:, 1])):
        assert ((got[:-3].cpu().to(F64) - w).abs() <= (2.0 ** -8 + 2.0 ** -23) * w.abs()).all() and (got[-3:] == 0).all()
    for total in (0, 5):
        none = lowbit.read8(_to(cpu, dev), _i([0], dev), _i([], dev), torch.zeros(0, 4, dtype=I32, device=dev), total=total)
        assert all(t.shape == (total, G, D) and (t == 0).all() for t in none)


@KINDS
@pytest.mark.parametrize("had", [0.0, -0.0, 2.0 ** -120, -0.5, 2.0 ** -101])
@pytest.mark.parametrize("dev", DEVICES)
def test_scales_below_the_least(dtype, had, dev):
    """They count as 2^-100 to whatever reads them: rows back, attention, and older rows that are rounded again."""
    G, D, P, least = 2, 64, 16, 2.0 ** -100
    base = _filled(3, G, P, D, dtype)
    base.k_scale[1], base.v_scale[1] = had, had
    bt = _i([[1]], dev)
    codes = {n: getattr(base, n)[1].float() for n in ("k", "v")}
    k, v = lowbit.read8(_to(base, dev), _i([0, 9], dev), _i([0], dev), bt, total=9)
    for got, n in ((k, "k"), (v, "v")):
        assert torch.equal(got.cpu(), (codes[n][:, :9].transpose(0, 1) * least).to(BF16))
    q = torch.randn(1, 2 * D, generator=torch.Generator().manual_seed(1)).to(BF16)
    _check(lowbit.attention8(q.to(dev), _to(base, dev), _i([0, 1], dev), _i([9], dev), bt, n_heads=2, max_q=1), q, base, _i([0, 1]), _i([9]), bt.cpu(), 2)
    # a row that asks for less than the least scale changes no older one; one that asks for 2^-99 halves them; a large one leaves zeros
    top = 127.0 if dtype is INT8 else 448.0
    for row, now, keep in ((2.0 ** -115, least, lambda c: c), (top * 2.0 ** -99, 2.0 ** -99, lambda c: ref.codes8(c / 2, dtype).float()),
                           (top, 1.0, lambda c: torch.zeros_like(c))):
        cache = _to(base, dev)
        x = torch.zeros(1, 3 * 2 * D, dtype=BF16)
        x[0, 2 * D:] = row
        lowbit.rope_append8(x.to(dev), None, cache, _i([0, 1], dev), _i([10], dev), bt, n_heads=2, max_q=1)
        for n in ("k", "v"):
            s, c = getattr(cache, n + "_scale")[1].cpu(), getattr(cache, n)[1].cpu().float()
            assert (s == now).all() and torch.equal(c[:, :9], keep(codes[n][:, :9])) and torch.equal(c[:, 10:], codes[n][:, 10:])
            assert (c[:, 9] == (0 if row < least else top)).all()


# ------------------------------------------------------------------ attention
def _attend_case(feeds, pasts, H, G, D, page, dtype, seed=0, std=1.5, pad=0, spare=0):
    g = torch.Generator().manual_seed(seed + 1)
    ctx = [a + b for a, b in zip(feeds, pasts)]
    pool, bt = _tables(ctx, page, seed=seed)
    cache = _filled(pool, G, page, D, dtype, seed)
    T = sum(feeds) + pad
    q = (torch.randn(T, H * D + spare, generator=g) * std).to(BF16)
    if pad:
        q[-pad:] = math.nan
    return q, cache, _cu(feeds), _i(ctx), bt


def _check(got, q, cache, cu, ctx, bt, H, **kw):
    o, mag = oracle.attention(q, cache, cu, ctx, bt, H, **kw)
    rows = int(cu[-1])
    err, bound = (got.cpu().to(F64)[:, :o.shape[1]] - o).abs()[:rows], oracle.attention_bound(o, mag)[:rows]
    assert bool((err <= bound).all()), float((err / bound).max())


ATTENDS = [  # tokens: a page, ends inside pages and tiles, one key, none, groups that fill and pass 16 rows
    ((1,) * 6, (0, 15, 31, 32, 127, 300), 8, 2, 128, 16), ((1, 1), (999, 4), 4, 4, 64, 32), ((1,), (2500,), 16, 1, 64, 16), ((2, 1, 0, 2), (17, 40, 9, 0), 8, 1, 128, 16),
    ((1, 1), (700, 1), 5, 1, 128, 128), ((3,), (3000,), 10, 2, 64, 16), ((16,), (5,), 2, 2, 128, 16),
    # prompts and chunks
    ((17,), (0,), 2, 2, 64, 16), ((130, 1, 64), (0, 77, 300), 8, 2, 128, 16), ((100,), (33,), 4, 4, 64, 64), ((33, 5), (1500, 2), 8, 1, 64, 16),
    ((9,), (4000,), 16, 4, 128, 16), ((300,), (0,), 5, 1, 128, 32), ((1,), (100,), 32, 1, 128, 16)]


@KINDS
@pytest.mark.parametrize("feeds,pasts,H,G,D,page", ATTENDS)
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dev", DEVICES)
def test_attention(feeds, pasts, H, G, D, page, dtype, causal, dev):
    q, cpu, cu, ctx, bt = _attend_case(feeds, pasts, H, G, D, page, dtype, pad=2, spare=8)
    out = torch.full((q.shape[0], H * D + 8), 3.0, dtype=BF16, device=dev)
    got = lowbit.attention8(q.to(dev), _to(cpu, dev), cu.to(dev), ctx.to(dev), bt.to(dev), n_heads=H, max_q=max(feeds), causal=causal, out=out)
    assert got is out and (out[-2:] == 3).all() and (out[:, H * D:] == 3).all()
    _check(got, q, cpu, cu, ctx, bt, H, causal=causal)


@KINDS
@pytest.mark.parametrize("max_q", [1, 40])
@pytest.mark.parametrize("dev", DEVICES)
def test_attention_without_keys(dtype, max_q, dev):
    """Contexts of zero, shorter than the feed, on pages that do not exist, wholly or in part: zeros where nothing is seen."""
    H, G, D, P = 4, 2, 64, 16
    feeds = [max_q, 1, max_q, max_q, max_q]
    ctx = [0, 1, max_q // 2, max_q + 50, max_q + 30]
    pool, bt = _tables([max(c, 1) for c in ctx], P)
    cpu = _filled(pool, G, P, D, dtype)
    free = sorted(set(range(pool)) - {int(bt[b, j]) for b, c in enumerate(ctx) for j in range(-(-max(c, 1) // P))})
    if dtype is E4M3:                                  # bytes that are NaN where nothing may be read
        cpu.k.view(torch.uint8)[free], cpu.v.view(torch.uint8)[free] = 0x7f, 0x7f
        used = bt[4, (ctx[4] - 1) // P]
        cpu.v.view(torch.uint8)[used, :, (ctx[4] - 1) % P + 1:] = 0xff
        cpu.k.view(torch.uint8)[used, :, (ctx[4] - 1) % P + 1:] = 0xff
    cpu.k_scale[free], cpu.v_scale[free] = math.nan, math.inf
    bt[3, 0], bt[3, 1] = pool, -7
    for b, c in enumerate(ctx):                        # entries behind a context name such pages
        bt[b, -(-max(c, 1) // P):] = free[b % len(free)]
    q = torch.randn(sum(feeds), H * D, generator=torch.Generator().manual_seed(3)).to(BF16)
    got = lowbit.attention8(q.to(dev), _to(cpu, dev), _cu(feeds, dev), _i(ctx, dev), bt.to(dev), n_heads=H, max_q=max_q)
    assert (got[:max_q] == 0).all() and got.isfinite().all()
    if max_q > 1:
        assert (got[max_q + 1:max_q + 1 + max_q - ctx[2]] == 0).all()
    _check(got, q, cpu, _cu(feeds), _i(ctx), bt, H)


@KINDS
@pytest.mark.parametrize("feeds,pasts,D", [((1, 1), (200, 30), 128), ((50,), (90,), 64)])
@pytest.mark.parametrize("dev", DEVICES)
def test_attention_of_unlike_sizes(feeds, pasts, D, dtype, dev):
    """Queries of 2^-120 and 2^100, pages whose value scales lie 2^40 apart, scales of zero, a scale argument, rows that no
    16-byte load takes."""
    H, G, P = 4, 2, 16
    q, cpu, cu, ctx, bt = _attend_case(feeds, pasts, H, G, D, P, dtype, spare=3)
    q[:, :D] *= 2.0 ** -120
    q[:, D:2 * D] *= 2.0 ** 100
    q[:, D + 5:2 * D:7] *= 2.0 ** -90
    cpu.k_scale *= 2.0 ** -50
    cpu.k_scale[:, 1] *= 2.0 ** 50
    cpu.v_scale[::2] *= 2.0 ** -40
    cpu.v_scale[1] = 0.0
    cpu.k_scale[1] = 0.0
    q[:, D:2 * D] *= 2.0 ** -50
    for scale in (None, 0.05, -0.1):
        got = lowbit.attention8(q.to(dev)[:, :H * D + 1], _to(cpu, dev), cu.to(dev), ctx.to(dev), bt.to(dev), n_heads=H, max_q=max(feeds), scale=scale)
        _check(got, q, cpu, cu, ctx, bt, H, scale=scale)


@pytest.mark.gpu
@KINDS
def test_attention_far_into_the_cache(dtype):
    """Pages whose bytes start past 2^32."""
    G, D, P, H = 8, 128, 16, 16
    far = (1 << 32) // (G * D * P) + 5
    cache = lowbit.Cache8.empty(far + 8, G, P, D, dtype, "cuda")
    small = _filled(8, G, P, D, dtype)
    for a, b in ((cache.k, small.k), (cache.v, small.v)):
        a.view(torch.uint8)[far:] = b.view(torch.uint8).cuda()
    cache.k_scale[far:], cache.v_scale[far:] = small.k_scale.cuda(), small.v_scale.cuda()
    for n, past in ((1, 100), (50, 60)):
        q = torch.randn(n, H * D, generator=torch.Generator().manual_seed(n)).to(BF16)
        near = torch.arange(8, dtype=I32)[None]
        got = lowbit.attention8(q.cuda(), cache, _i([0, n], "cuda"), _i([n + past], "cuda"), (near + far).cuda(), n_heads=H, max_q=n)
        _check(got, q, small, _i([0, n]), _i([n + past]), near, H)
    rows = torch.randn(20, (H + 2 * G) * D, generator=torch.Generator().manual_seed(9)).to(BF16)
    lowbit.rope_append8(rows.cuda(), None, cache, _i([0, 20], "cuda"), _i([31], "cuda"), (near + far).cuda(), n_heads=H, max_q=20)
    lowbit.rope_append8(rows, None, small, _i([0, 20]), _i([31]), near, n_heads=H, max_q=20)
    for a, b in ((cache.k, small.k), (cache.v, small.v)):
        assert torch.equal(a.view(torch.uint8)[far:].cpu(), b.view(torch.uint8)) and not a.view(torch.uint8)[:8].any()
    k, _ = lowbit.read8(cache, _i([0, 31], "cuda"), _i([0], "cuda"), (near + far).cuda(), total=31)
    assert torch.equal(k.cpu(), lowbit.read8(small, _i([0, 31]), _i([0]), near, total=31)[0])


@pytest.mark.gpu
@KINDS
@pytest.mark.parametrize("feeds,pasts", [((1,), (20000,)), ((1, 1, 1), (5000, 3, 800)), ((20,), (6000,))])
def test_attention_in_parts(dtype, feeds, pasts):
    """Many keys in as many parts as the bound on them asks for: right with any bound, and the same again."""
    H, G, D, P = 8, 2, 128, 16
    q, cpu, cu, ctx, bt = _attend_case(feeds, pasts, H, G, D, P, dtype)
    dev, there = _to(cpu, "cuda"), [t.cuda() for t in (q, cu, ctx, bt)]
    o, mag = oracle.attention(q, cpu, cu, ctx, bt, H)
    for max_k in (None, 64, 700, max(pasts) + max(feeds)):
        got = [lowbit.attention8(there[0], dev, *there[1:], n_heads=H, max_q=max(feeds), max_k=max_k) for _ in range(3)]
        assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])
        assert ((got[0].cpu().to(F64) - o).abs() <= oracle.attention_bound(o, mag)).all()


@KINDS
@pytest.mark.parametrize("feeds,pasts,H,G,D,page", [((3, 1, 2), (5, 900, 0), 8, 1, 128, 16), ((5, 5), (1300, 31), 8, 2, 64, 16), ((20, 0, 7), (0, 3, 2000), 4, 4, 64, 32), ((32,), (3000,), 2, 2, 128, 16),
                                                    ((6, 4, 1), (40, 4100, 2500), 5, 1, 128, 64), ((17, 3), (1, 40000), 1, 1, 64, 16), ((11,), (9000,), 8, 2, 128, 16)])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("dev", DEVICES)
def test_attention_of_some_tokens(feeds, pasts, H, G, D, page, dtype, causal, dev):
    """17 to 48 rows a kv head, contexts that end inside tiles and pages beside ones in many parts, any bound on the keys."""
    q, cpu, cu, ctx, bt = _attend_case(feeds, pasts, H, G, D, page, dtype, pad=3, spare=8)
    there = [q.to(dev), _to(cpu, dev), cu.to(dev), ctx.to(dev), bt.to(dev)]
    o, mag = oracle.attention(q, cpu, cu, ctx, bt, H, causal=causal)
    rows = int(cu[-1])
    for max_k in (None, 40, 1000):
        out = torch.full((q.shape[0], H * D), 3.0, dtype=BF16, device=dev)
        lowbit.attention8(*there, n_heads=H, max_q=max(feeds), max_k=max_k, causal=causal, out=out)
        assert (out[rows:] == 3).all()
        assert ((out.cpu().to(F64) - o).abs()[:rows] <= oracle.attention_bound(o, mag)[:rows]).all()


@KINDS
@pytest.mark.parametrize("dev", DEVICES)
def test_some_tokens_of_pages_that_are_none(dtype, dev):
    """24 rows a kv head: contexts of zero, shorter than the feed, on pages that do not exist, codes that are NaN behind the ends."""
    H, G, D, P, n = 8, 2, 64, 16, 6
    feeds, ctx = [n] * 5, [0, 1, n // 2, 90, 70]
    pool, bt = _tables([max(c, 1) for c in ctx], P)
    cpu = _filled(pool, G, P, D, dtype)
    free = sorted(set(range(pool)) - {int(bt[b, j]) for b, c in enumerate(ctx) for j in range(-(-max(c, 1) // P))})
    if dtype is E4M3:
        cpu.k.view(torch.uint8)[free], cpu.v.view(torch.uint8)[free] = 0x7f, 0x7f
        used = bt[4, (ctx[4] - 1) // P]
        cpu.v.view(torch.uint8)[used, :, (ctx[4] - 1) % P + 1:] = 0xff
        cpu.k.view(torch.uint8)[used, :, (ctx[4] - 1) % P + 1:] = 0xff
    cpu.k_scale[free], cpu.v_scale[free] = math.nan, math.inf
    bt[3, 0], bt[3, 1] = pool, -7
    for b, c in enumerate(ctx):
        bt[b, -(-max(c, 1) // P):] = free[b % len(free)]
    q = torch.randn(sum(feeds), H * D, generator=torch.Generator().manual_seed(3)).to(BF16)
    got = lowbit.attention8(q.to(dev), _to(cpu, dev), _cu(feeds, dev), _i(ctx, dev), bt.to(dev), n_heads=H, max_q=n)
    assert (got[:2 * n - 1] == 0).all() and got.isfinite().all()
    _check(got, q, cpu, _cu(feeds), _i(ctx), bt, H)


@KINDS
@pytest.mark.parametrize("n,H,G,D", [(1, 8, 2, 128), (3, 4, 1, 64), (6, 4, 1, 128), (20, 4, 2, 64)])
@pytest.mark.parametrize("dev", DEVICES)
def test_pages_behind_a_context_are_no_part_of_it(dtype, n, H, G, D, dev):
    """Contexts that end in either half of a tile, with table entries behind them that name pages whose scales are NaN: the
    padding of a table, or what an ended sequence left."""
    P = 16
    ctx = [20, 33, 48, 64, 300, 321, 37]
    feeds = [n] * len(ctx)
    pool, bt = _tables(ctx, P, width=24)
    cpu = _filled(pool, G, P, D, dtype)
    used = {int(bt[b, j]) for b, c in enumerate(ctx) for j in range(-(-c // P))}
    free = sorted(set(range(pool)) - used)
    cpu.k_scale[free], cpu.v_scale[free] = math.nan, math.nan
    for b, c in enumerate(ctx):
        bt[b, -(-c // P):] = free[b % len(free)]
    q = torch.randn(sum(feeds), H * D, generator=torch.Generator().manual_seed(3)).to(BF16)
    got = lowbit.attention8(q.to(dev), _to(cpu, dev), _cu(feeds, dev), _i(ctx, dev), bt.to(dev), n_heads=H, max_q=n)
    assert got.isfinite().all()
    _check(got, q, cpu, _cu(feeds), _i(ctx), bt, H)


@KINDS
@pytest.mark.parametrize("which", ["k_scale", "v_scale"])
@pytest.mark.parametrize("x", [math.nan, math.inf])
@pytest.mark.parametrize("n,past,H,D,P", [(12, 40, 1, 64, 16), (12, 25, 2, 128, 32), (40, 10, 1, 64, 16), (70, 100, 2, 128, 64), (150, 0, 4, 64, 16)])
@pytest.mark.parametrize("dev", DEVICES)
def test_rows_ahead_of_a_page_that_is_no_number(n, past, H, D, P, x, which, dtype, dev):
    """A page whose scale is no number is that to rows that see one of its keys, and nothing to those ahead of it."""
    q, cpu, cu, ctx, bt = _attend_case((n,), (past,), H, 1, D, P, dtype)
    page = (past + n // 2) // P + 1 if (past + n // 2) // P + 1 < bt.shape[1] else (past + n // 2) // P
    ahead = max(page * P - past, 0)                      # rows that see none of it
    assert 0 < ahead < n
    spoilt = _to(cpu, dev)
    getattr(spoilt, which)[int(bt[0, page])] = x
    got = lowbit.attention8(q.to(dev), spoilt, cu.to(dev), ctx.to(dev), bt.to(dev), n_heads=H, max_q=n).cpu()
    o, mag = oracle.attention(q, cpu, cu, ctx, bt, H)
    assert ((got.to(F64) - o).abs()[:ahead] <= oracle.attention_bound(o, mag)[:ahead]).all()
    if math.isnan(x):
        assert got[ahead:].isnan().all()


@KINDS
@pytest.mark.parametrize("H", [1, 20, 40])
@pytest.mark.parametrize("dev", DEVICES)
def test_many_keys_behind_a_dominant_one(dtype, H, dev):
    """2^18 keys of like weight, 2^-26.5 of the first one's, whose values are zero: what they sum up to is the result. A weight
    is f16 over a reference 2^7 below the row's largest one: off by 2^-11, or by 2^-25 of 2^7 under 2^-14 of it; in one part, so that
    all of them follow the first key."""
    D, P, L, code = 64, 16, 1 << 18, 64
    pages = L // P
    cache = lowbit.Cache8.empty(pages, 1, P, D, dtype)
    cache.k_scale.fill_(1 / code)
    cache.v_scale.fill_(1 / code)
    for t in (cache.k, cache.v):
        t[0, 0, 0] = 0
    cache.k[0, 0, 0, 0] = code
    ones = torch.full((D,), code, dtype=torch.float32).to(dtype)
    cache.v.view(torch.uint8)[:] = ones.view(torch.uint8)
    cache.v.view(torch.uint8)[0, 0, 0] = 0
    q = torch.zeros(1, H * D, dtype=BF16)
    q[0, ::D] = 26.5 * math.log(2)
    w = math.exp(-float(q[0, 0]))
    total = (L - 1) * w
    o = total / (1 + total)
    bt = torch.arange(pages, dtype=I32, device=dev)[None]
    got = lowbit.attention8(q.to(dev), _to(cache, dev), _i([0, 1], dev), _i([L], dev), bt, n_heads=H, max_q=1, max_k=1, scale=1.0).cpu().to(F64)
    assert ((got - o).abs() <= (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -14) * o + L * 2.0 ** -32).all(), (float(got.min()), float(got.max()), o)


@KINDS
@pytest.mark.parametrize("H", [4, 20, 40, 130])
@pytest.mark.parametrize("most", [20, 23, 24.5, 25.5])
@pytest.mark.parametrize("dev", DEVICES)
def test_scores_as_large_as_their_steps(dtype, H, most, dev):
    """Scores of 2^20 to 2^25 (base two) that f32 holds in steps of up to four: whatever these make of them, results stay between the
    smallest and the largest value."""
    D, P, L = 64, 16, 1500
    g = torch.Generator().manual_seed(int(most * 2) + H)
    cache = lowbit.Cache8.empty(-(-L // P), 1, P, D, dtype)
    code = 127 if dtype is INT8 else 128
    k = torch.zeros(cache.k.shape)
    k[..., 0] = code
    k[..., 1] = (torch.arange(k.shape[0]) * 127 / k.shape[0]).round()[:, None, None]        # scores that rise with the keys
    k[..., 2] = torch.randint(-1, 2, k.shape[:3], generator=g).float()
    cache.k.view(torch.uint8)[:] = k.to(dtype).view(torch.uint8)
    cache.v.view(torch.uint8)[:] = (torch.randint(32, 97, k.shape, generator=g).float()).to(dtype).view(torch.uint8)
    cache.k_scale.fill_(1.0)
    cache.v_scale.copy_(0.6 + torch.rand(cache.v_scale.shape, generator=g))
    q = torch.zeros(1, H * D)
    base = 2.0 ** most / code
    q[0, 0::D] = base * torch.where(torch.arange(H) % 5 == 4, -1.0, 1.0)
    q[0, 1::D] = 2.0 ** (3 + 6 * torch.rand(H, generator=g)) / 127                          # by 8 to 512
    q[0, 2::D] = 1.0
    bt = torch.arange(cache.n_blocks, dtype=I32, device=dev)[None]
    got = lowbit.attention8(q.to(BF16).to(dev), _to(cache, dev), _i([0, 1], dev), _i([L], dev), bt, n_heads=H, max_q=1, scale=math.log(2), max_k=1).cpu().float()
    v = cache.v.float() * cache.v_scale[..., None, None]
    # rounded to bf16, weights to f16 while their sum is not
    assert got.isfinite().all() and (got <= v.max() * (1 + 2.0 ** -7)).all() and (got >= v.min() * (1 - 2.0 ** -7)).all()


# ------------------------------------------------------------------ pages
def _pages_case(new, ctx, P, width, free, head=0, spare=2, seed=0):
    held = [-(-c // P) for c in ctx]
    pool = sum(held) + free + spare
    order = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(I32)
    bt, at = torch.full((len(new), width), -5, dtype=I32), 0
    for b, n in enumerate(held):
        bt[b, :min(n, width)] = order[at:at + min(n, width)]
        at += n
    ring = torch.full((pool,), -9, dtype=I32)
    for j in range(free):
        ring[(head + j) % pool] = order[at + j]
    return _i(new), _i(ctx), bt, ring, _i([head, free])


PAGES = [([1] * 8, [0, 1, 15, 16, 17, 31, 32, 600], 16, 50, 20, 0), ([5, 0, -1, 40, -1, 0], [3, 9, 100, 0, 0, 0], 16, 9, 30, 25), ([1], [0], 16, 1, 1, 0), ([-1], [33], 32, 4, 0, 2),
         ([300, -1, 2], [0, 64, 64], 64, 8, 9, 0), ([2] * 1500, list(range(1500)), 16, 120, 1500, 70000 // 7), ([0, 0], [0, 5], 16, 2, 0, 0)]


@pytest.mark.parametrize("new,ctx,P,width,free,head", PAGES)
@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("in_place", [False, True])
def test_page_step(new, ctx, P, width, free, head, dev, in_place):
    n, c, bt, ring_pages, ring = _pages_case(new, ctx, P, width, free, head)
    most = sum(max(x, 0) for x in new) + 5
    d = [t.clone().to(dev) for t in (n, c, bt, ring_pages, ring)]
    kw = dict(ctx_out=d[1], ring_out=d[4]) if in_place else {}
    r = lowbit.page_step(*d, block_size=P, max_tokens=most, **kw)
    assert r.status.item() == 0
    # by hand: a queue of free pages, sequences one after the other
    pool = ring_pages.numel()
    queue = [int(ring_pages[(head + j) % pool]) for j in range(free)]
    tables, after, at, gone = [row.tolist() for row in bt], [], 0, []
    pos, slots, cu, last = [], [], [0], []
    for i, (x, y) in enumerate(zip(new, ctx)):
        if x == -1:
            gone += tables[i][:-(-y // P)]
            after.append(0)
        else:
            for j in range(-(-y // P), -(-(x + y) // P)):
                tables[i][j] = queue.pop(0)
            pos += range(y, x + y)
            slots += [tables[i][t // P] * P + t % P for t in range(y, x + y)]
            after.append(x + y)
        cu.append(len(pos))
        last.append(len(pos) - 1 if x > 0 else 0)
    queue += gone
    assert r.positions.tolist() == pos + [0] * 5 and r.slots.tolist() == slots + [-1] * 5 and r.cu_q.tolist() == cu and r.last_rows.tolist() == last
    assert r.ctx_lens.tolist() == after and d[2].tolist() == tables
    h, count = r.ring.tolist()
    assert [int(d[3][(h + j) % pool]) for j in range(count)] == queue
    assert not in_place or (r.ctx_lens is d[1] and r.ring is d[4])


@pytest.mark.parametrize("dev", DEVICES)
@pytest.mark.parametrize("change,status", [(dict(free=1), 1), (dict(most=6), 2), (dict(width=3), 4), (dict(new=[1, -2, 4]), 8), (dict(ctx=[16, -1, 40]), 8),
                                           (dict(ring=[-1, 5]), 8), (dict(ring=[0, 1000]), 8), (dict(ring=[1000, 5]), 8), (dict(free=1, most=2), 3),
                                           (dict(new=[(1 << 31) - 1] * 3), 7)])
def test_page_step_all_or_nothing(dev, change, status):
    new, ctx = change.get("new", [1, 2, 30]), change.get("ctx", [16, 5, 40])
    n, c, bt, pages, ring = _pages_case([max(x, 0) for x in new], [max(x, 0) for x in ctx], 16, change.get("width", 6), change.get("free", 5), 1)
    ring = _i(change["ring"]) if "ring" in change else ring
    d = [t.to(dev) for t in (_i(new), _i(ctx), bt.clone(), pages.clone(), ring)]
    most = change.get("most", 40)
    r = lowbit.page_step(*d, block_size=16, max_tokens=most)
    assert r.status.item() == status
    assert torch.equal(d[2].cpu(), bt) and torch.equal(d[3].cpu(), pages) and r.ctx_lens.tolist() == ctx and r.ring.tolist() == ring.tolist()
    assert (r.slots == -1).all() and (r.positions == 0).all() and (r.cu_q == 0).all() and (r.last_rows == 0).all()


# ------------------------------------------------------------------ 4 bits
LINEARS = [(1, 16, 32, 32, False), (1, 4096, 4096, 128, False), (3, 50, 96, 32, True), (16, 128, 256, 64, True), (17, 33, 384, 128, True), (33, 257, 1056, 32, False),
           (64, 64, 640, 64, False), (65, 48, 128, 128, True), (8, 1000, 2112, 64, True), (130, 20, 160, 32, True)]


@pytest.mark.parametrize("M,N,K,group,zeros", LINEARS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("dev", DEVICES)
def test_linear4(M, N, K, group, zeros, bias, dev):
    g = torch.Generator().manual_seed(M * 7 + N)
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g)
    scales = (0.02 * torch.randn(N, K // group, generator=g)).to(BF16)
    z = torch.randint(0, 16, (N, K // group), dtype=torch.uint8, generator=g) if zeros else None
    x = torch.randn(M, K, generator=g).to(BF16)
    b = torch.randn(N, generator=g).to(BF16) if bias else None
    c = torch.stack([codes & 15, codes >> 4], -1).view(N, K).to(F64)
    w = (c - (z.to(F64).repeat_interleave(group, 1) if zeros else 8)) * scales.to(F64).repeat_interleave(group, 1)
    y = x.to(F64) @ w.t() + (b.to(F64) if bias else 0)
    w4 = lowbit.Weight4(codes.to(dev), scales.to(dev), z.to(dev) if zeros else None)
    got = lowbit.linear4(x.to(dev), w4, b.to(dev) if bias else None)
    assert got.shape == (M, N) and ((got.cpu().to(F64) - y).abs() <= oracle.linear4_bound(y, x, w, scales)).all()
    # rows with a stride, at odd places, and more dimensions
    wide = torch.full((M, K + 9), math.nan, dtype=BF16)
    for off in (0, 1, 8):
        v = wide.clone().to(dev)[:, off:off + K]
        v.copy_(x)
        assert torch.equal(lowbit.linear4(v, w4, b.to(dev) if bias else None), got)
    assert torch.equal(lowbit.linear4(x.to(dev)[:, None], w4, b.to(dev) if bias else None)[:, 0], got)
    assert lowbit.linear4(x.to(dev)[:0], w4).shape == (0, N)


@pytest.mark.parametrize("M,N,K,group,zeros", [(17, 200, 4224, 32, True), (32, 4104, 96, 32, False), (24, 40, 2176, 128, True), (33, 24600, 160, 32, True), (64, 24576, 512, 128, False),
                                               (40, 70, 5184, 64, True), (100, 333, 1152, 64, False), (20, 24592, 288, 32, True), (32, 64, 2112, 64, False)])
@pytest.mark.parametrize("dev", DEVICES)
def test_linear4_more_rows(M, N, K, group, zeros, dev):
    """Rows that share x in LDS: parts of K, ends inside a block, a tile and a workgroup's tiles, and what lies around y stays."""
    g = torch.Generator().manual_seed(M + N + K)
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g)
    scales = (0.02 * torch.randn(N, K // group, generator=g)).to(BF16)
    z = torch.randint(0, 16, (N, K // group), dtype=torch.uint8, generator=g) if zeros else None
    x, b = torch.randn(M, K, generator=g).to(BF16), torch.randn(N, generator=g).to(BF16)
    w = ref.dense4(codes, scales, z).to(F64)
    w4 = lowbit.Weight4(codes.to(dev), scales.to(dev), z.to(dev) if zeros else None)
    y = x.to(F64) @ w.t() + b.to(F64)
    got = lowbit.linear4(x.to(dev), w4, b.to(dev))
    assert got.shape == (M, N) and ((got.cpu().to(F64) - y).abs() <= oracle.linear4_bound(y, x, w, scales)).all()
    for _ in range(3):
        assert torch.equal(lowbit.linear4(x.to(dev), w4, b.to(dev)), got)
    # a row that is no number stays the only one
    x[M // 2, K - 1] = math.inf
    odd = lowbit.linear4(x.to(dev), w4, b.to(dev))
    rows = torch.arange(M, device=dev) != M // 2
    assert torch.equal(odd[rows], got[rows]) and not odd[~rows].isfinite().any()


@pytest.mark.parametrize("M", [1, 20, 40])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dev", DEVICES)
def test_linear4_large_entries(M, zeros, dev):
    """Entries up to 2^112, whose sums with the codes' offset stay finite."""
    g, N, K, group = torch.Generator().manual_seed(M), 48, 2304, 128
    codes = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g)
    scales = (2.0 ** -20 * (1 + torch.rand(N, K // group, generator=g))).to(BF16)
    z = torch.randint(0, 16, (N, K // group), dtype=torch.uint8, generator=g) if zeros else None
    x = torch.full((M, K), 2.0 ** 112, dtype=BF16)
    x[:, ::3] *= -0.5
    w = ref.dense4(codes, scales, z).to(F64)
    y = x.to(F64) @ w.t()
    got = lowbit.linear4(x.to(dev), lowbit.Weight4(codes.to(dev), scales.to(dev), z.to(dev) if zeros else None))
    assert ((got.cpu().to(F64) - y).abs() <= oracle.linear4_bound(y, x, w, scales)).all()


@pytest.mark.gpu
@KINDS
def test_append_in_place(dtype):
    """Rotated queries may go where the queries were."""
    H, G, D, P, n = 6, 2, 64, 16, 50
    rows = torch.randn(n, (H + 2 * G) * D, generator=torch.Generator().manual_seed(1)).to(BF16).cuda()
    cs, bt = ref.rope_cos_sin(D, 64, 10000.0).cuda(), torch.arange(4, dtype=I32, device="cuda")[None]
    a, b = (lowbit.Cache8.empty(4, G, P, D, dtype, "cuda") for _ in range(2))
    cu, ctx = _i([0, n], "cuda"), _i([n + 3], "cuda")
    want = lowbit.rope_append8(rows, cs, a, cu, ctx, bt, n_heads=H, max_q=n)
    out = rows[:, :H * D]
    assert lowbit.rope_append8(rows, cs, b, cu, ctx, bt, n_heads=H, max_q=n, q_out=out) is out
    assert torch.equal(out, want)
    _same(a, b)


@pytest.mark.gpu
def test_linear4_parts_in_graphs_and_streams():
    """Products in parts of K: a captured one replayed between eager ones, and two streams at once."""
    g = torch.Generator("cuda").manual_seed(3)
    ws = [lowbit.Weight4(*(t.cuda() for t in lowbit.quantize4(torch.randn(n, k, generator=torch.Generator().manual_seed(n)), 64, True))) for n, k in
          ((320, 4096), (700, 2304))]
    x = [torch.randn(48, w.k, device="cuda", generator=g).to(BF16) for w in ws]
    graph = torch.cuda.CUDAGraph()
    for a, w in zip(x, ws):
        lowbit.linear4(a, w)
    with ops.graph_capture(graph):
        out = [lowbit.linear4(a, w) for a, w in zip(x, ws)]
    streams = [torch.cuda.Stream() for _ in ws]
    for i in range(5):
        for a in x:
            a.normal_(generator=g)
        want = [lowbit.linear4(a, w) for a, w in zip(x, ws)]
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        torch.cuda.synchronize()
        got = []
        for st, a, w in zip(streams, x, ws):
            with torch.cuda.stream(st):
                got.append([lowbit.linear4(a, w) for _ in range(4)])
        torch.cuda.synchronize()
        assert all(torch.equal(y, b) for ys, b in zip(got, want) for y in ys), i


@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantize4(zeros, group):
    """To nearest: within half a step (of a scale that bf16 holds, 2^-8 off: seven steps of it more), and what ends are cut off."""
    w = torch.randn(24, 256, generator=torch.Generator().manual_seed(1)) + (0.5 if zeros else 0)
    w[3] = 0
    codes, s, z = lowbit.quantize4(w, group, zeros)
    back = ref.dense4(codes, s, z)
    step = s.float().repeat_interleave(group, 1)
    ends = 7 * 2.0 ** -8 if not zeros else 15 * 2.0 ** -8 + 0.5
    assert ((back - w).abs() <= (0.5 + ends + 1e-5) * step).all() and (back[3] == 0).all()
    assert codes.shape == (24, 128) and s.shape == (24, 256 // group) and (z is None) != zeros


# ------------------------------------------------------------------ together
@KINDS
@pytest.mark.parametrize("dev", DEVICES)
def test_a_decoder_step_by_step(dtype, dev):
    """Prompts of unlike length, then tokens, as a serving loop runs them: pages, projections in 4 bits, append, attention;
    a sequence ends, its pages serve a new one. The queries, keys and values of each step against 64 bits of the whole history."""
    H, G, D, P, width = 4, 2, 64, 16, 6
    gen = torch.Generator().manual_seed(11)
    w = lowbit.quantize4(torch.randn((H + 2 * G) * D, 128, generator=gen) / 11, 32, True)
    w4 = lowbit.Weight4(*(t.to(dev) for t in w))
    dense = ref.dense4(*w).to(F64)
    cs = ref.rope_cos_sin(D, 96, 10000.0)
    cache = lowbit.Cache8.empty(14, G, P, D, dtype, dev)
    bt, ctx = torch.zeros(3, width, dtype=I32, device=dev), _i([0, 0, 0], dev)
    pages, ring = torch.arange(14, dtype=I32, device=dev), _i([0, 14], dev)
    history = [[], [], []]
    for new in ([20, 0, 37], [1, 5, 1], [1, 1, 1], [1, -1, 1], [1, 60, 1], [2, 1, -1], [1, 1, 9]):
        step = lowbit.page_step(_i(new, dev), ctx, bt, pages, ring, block_size=P, max_tokens=64, ctx_out=ctx, ring_out=ring)
        assert step.status.item() == 0
        T = sum(max(n, 0) for n in new)
        x = torch.randn(64, 128, generator=gen).to(BF16)
        qkv = lowbit.linear4(x.to(dev), w4)
        q = lowbit.rope_append8(qkv, cs.to(dev), cache, step.cu_q, step.ctx_lens, bt, n_heads=H, max_q=64)
        o = lowbit.attention8(q, cache, step.cu_q, step.ctx_lens, bt, n_heads=H, max_q=64).cpu().to(F64)
        y = (x.to(F64) @ dense.t()).view(64, H + 2 * G, D)
        at = 0
        for b, n in enumerate(new):
            if n == -1:
                history[b] = []
                continue
            for i in range(n):
                r, p = y[at + i].clone(), len(history[b])
                c, s = cs[p].to(F64).unbind(-1)
                lo, hi = r[:H + G, :D // 2].clone(), r[:H + G, D // 2:].clone()
                r[:H + G, :D // 2], r[:H + G, D // 2:] = lo * c - hi * s, hi * c + lo * s
                history[b].append(r)
                kv = torch.stack(history[b])
                k, v = kv[:, H:H + G].repeat_interleave(H // G, 1), kv[:, H + G:].repeat_interleave(H // G, 1)
                pr = torch.softmax(torch.einsum("hd,jhd->hj", r[:H], k) / math.sqrt(D), -1)
                want = torch.einsum("hj,jhd->hd", pr, v).reshape(-1)
                # 8 bits of keys and values: 2^-4 of an entry in e4m3, a step of 2^-7 of a page's largest (about 4) in int8;
                # over 64 columns the scores are off by their root mean square, and with weights and values by as much again
                assert (o[at + i] - want).norm() <= 0.1 * want.norm() + 0.02 * math.sqrt(H * D), (new, b, i)
            at += n
        assert (step.positions[:T].cpu() >= 0).all() and (step.slots[T:] == -1).all()


@pytest.mark.gpu
@KINDS
def test_steps_in_a_graph(dtype):
    """A captured step with its lengths on the GPU, replayed between other work, against the same steps run eagerly."""
    H, G, D, P, B, width = 8, 2, 128, 16, 5, 40
    gen = torch.Generator().manual_seed(2)
    w4 = lowbit.Weight4(*(t.cuda() for t in lowbit.quantize4(torch.randn((H + 2 * G) * D, 256, generator=gen) / 16, 64, True)))
    cs = ref.rope_cos_sin(D, 640, 10000.0).cuda()

    def state():
        pool = B * width
        return dict(cache=lowbit.Cache8.empty(pool, G, P, D, dtype, "cuda"), bt=torch.zeros(B, width, dtype=I32, device="cuda"), ctx=_i([0] * B, "cuda"),
                    pages=torch.arange(pool, dtype=I32, device="cuda"), ring=_i([0, pool], "cuda"), new=_i([1] * B, "cuda"))

    def step(s, x, most, max_q):
        r = lowbit.page_step(s["new"], s["ctx"], s["bt"], s["pages"], s["ring"], block_size=P, max_tokens=most, ctx_out=s["ctx"], ring_out=s["ring"])
        q = lowbit.rope_append8(lowbit.linear4(x, w4), cs, s["cache"], r.cu_q, r.ctx_lens, s["bt"], n_heads=H, max_q=max_q)
        return lowbit.attention8(q, s["cache"], r.cu_q, r.ctx_lens, s["bt"], n_heads=H, max_q=max_q, out=torch.zeros_like(q)), r.slots
    a, b = state(), state()
    first = torch.randn(600, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(BF16)
    for s in (a, b):
        s["new"].copy_(_i([300, 1, 17, 0, 200]))
        step(s, first, 600, 300)
        s["new"].fill_(1)
    assert torch.equal(a["bt"], b["bt"])
    x = torch.zeros(B, 256, dtype=BF16, device="cuda")
    kept = {k: v.clone() for k, v in b.items() if k != "cache"}
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    keep = _to(b["cache"], "cuda")
    with torch.cuda.stream(side):
        step(b, x, B, 1)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with ops.graph_capture(graph):
        o, slots = step(b, x, B, 1)
    for k, v in kept.items():
        b[k].copy_(v)
    for n in ("k", "v"):
        getattr(b["cache"], n).view(torch.uint8).copy_(getattr(keep, n).view(torch.uint8))
        getattr(b["cache"], n + "_scale").copy_(getattr(keep, n + "_scale"))
    for i in range(6):
        new = torch.randn(B, 256, device="cuda", generator=torch.Generator("cuda").manual_seed(50 + i)).to(BF16)
        x.copy_(new)
        graph.replay()
        want, want_slots = step(a, new, B, 1)
        assert torch.equal(o, want) and torch.equal(slots, want_slots), i
        _same(a["cache"], b["cache"])
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_two_streams():
    """Calls in parts on two streams at once use workspaces of their own."""
    H, G, D, P = 8, 2, 128, 16
    cases = [_attend_case((1,), (30000,), H, G, D, P, INT8, seed=s) for s in (1, 2)]
    there = [[q.cuda(), _to(c, "cuda"), *(t.cuda() for t in rest)] for q, c, *rest in cases]
    want = [lowbit.attention8(*t, n_heads=H, max_q=1) for t in there]
    streams = [torch.cuda.Stream() for _ in there]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(lowbit.attention8(*there[i], n_heads=H, max_q=1))
    torch.cuda.synchronize()
    for i in (0, 1):
        assert all(torch.equal(g, want[i]) for g in got[i])


@pytest.mark.gpu
def test_calls_from_threads():
    """Threads on streams of their own and on one stream together: each gets what it gets alone."""
    H, G, D, P, n = 8, 2, 128, 16, 4
    w = lowbit.Weight4(*(t.cuda() for t in lowbit.quantize4(torch.randn(320, 4096, generator=torch.Generator().manual_seed(1)), 64, True)))
    work = []
    for i in range(n):
        q, c, *rest = _attend_case((1,) if i % 2 else (9,), (9000,), H, G, D, P, INT8, seed=i)
        x = torch.randn(33 + i, 4096, device="cuda", generator=torch.Generator("cuda").manual_seed(i)).to(BF16)
        work.append((x, q.cuda(), _to(c, "cuda"), *(t.cuda() for t in rest)))

    def both(x, q, cache, cu, ctx, bt):
        return lowbit.linear4(x, w), lowbit.attention8(q, cache, cu, ctx, bt, n_heads=H, max_q=q.shape[0])
    want = [both(*a) for a in work]
    torch.cuda.synchronize()
    for streams in ([torch.cuda.Stream() for _ in range(n)], [torch.cuda.current_stream()] * n):
        got = [None] * n

        def loop(i):
            with torch.cuda.stream(streams[i]):
                got[i] = [both(*work[i]) for _ in range(20)]
                streams[i].synchronize()
        threads = [threading.Thread(target=loop, args=(i,)) for i in range(n)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        for i in range(n):
            assert got[i] is not None and all(torch.equal(a, b) for y in got[i] for a, b in zip(y, want[i])), i


# ------------------------------------------------------------------ refusals
def _good(dev="cpu"):
    cache = lowbit.Cache8.empty(4, 2, 16, 64, device=dev)
    return dict(cache=cache, cu_q=_i([0, 2], dev), ctx_lens=_i([2], dev), block_tables=_i([[0, 1]], dev), n_heads=4, max_q=2)


@pytest.mark.parametrize("change,error", [
    (dict(cu_q=torch.tensor([0, 2])), TypeError), (dict(ctx_lens=torch.tensor([2.0])), TypeError), (dict(block_tables=_i([0, 1])), ValueError),
    (dict(block_tables=_i([[0], [1]])), ValueError), (dict(cu_q=_i([0, 1, 2])), ValueError), (dict(block_tables=torch.zeros(1, 0, dtype=I32)), ValueError),
    (dict(block_tables=_i([[0, 1, 2, 3]])[:, ::2]), ValueError), (dict(n_heads=0), ValueError), (dict(max_q=-1), ValueError)])
def test_refusals_of_sequences(change, error):
    a = {**_good(), **change}
    with pytest.raises(error):
        lowbit.attention8(torch.zeros(2, 256, dtype=BF16), **a)
    with pytest.raises(error):
        lowbit.rope_append8(torch.zeros(2, 512, dtype=BF16), None, **a)


@pytest.mark.parametrize("kw", [dict(q=torch.zeros(2, 256)), dict(q=torch.zeros(2, 255, dtype=BF16)), dict(q=torch.zeros(2, 512, dtype=BF16)[:, ::2]),
                                dict(out=torch.zeros(1, 256, dtype=BF16)), dict(out=torch.zeros(2, 256)), dict(out=torch.zeros(1, 256, dtype=BF16).expand(2, 256)),
                                dict(n_heads=3), dict(max_k=-1), dict(q=torch.zeros(2, 4, 64, dtype=BF16))])
def test_refusals_of_attention(kw):
    a = {**_good(), "q": torch.zeros(2, 256, dtype=BF16), **kw}
    with pytest.raises((TypeError, ValueError)):
        lowbit.attention8(a.pop("q"), **a)


@pytest.mark.parametrize("kw", [dict(qkv=torch.zeros(2, 511, dtype=BF16)), dict(qkv=torch.zeros(2, 512)), dict(cos_sin=torch.zeros(9, 64, 2)), dict(cos_sin=torch.zeros(0, 32, 2)),
                                dict(cos_sin=torch.zeros(9, 32, 2, dtype=F64)), dict(q_out=torch.zeros(3, 256, dtype=BF16)), dict(q_out=torch.zeros(2, 200, dtype=BF16))])
def test_refusals_of_append(kw):
    a = {**_good(), "qkv": torch.zeros(2, 512, dtype=BF16), "cos_sin": None, **kw}
    with pytest.raises((TypeError, ValueError)):
        lowbit.rope_append8(a.pop("qkv"), a.pop("cos_sin"), **a)


def test_refusals_of_caches():
    def make(shape=(4, 2, 16, 64), dtype=INT8, scales=(4, 2), sdtype=torch.float32, v=None):
        k = torch.zeros(shape, dtype=torch.uint8).view(dtype)
        return lowbit.Cache8(k, k.clone() if v is None else v, torch.zeros(scales, dtype=sdtype), torch.zeros(scales, dtype=sdtype))
    make()
    for kw in (dict(shape=(4, 2, 16, 96)), dict(shape=(4, 2, 8, 64)), dict(shape=(4, 2, 24, 64)), dict(scales=(4, 1)), dict(sdtype=BF16), dict(dtype=torch.uint8),
               dict(v=torch.zeros(4, 2, 16, 64)), dict(v=torch.zeros(4, 2, 16, 128, dtype=INT8)), dict(v=torch.zeros(4, 2, 16, 128, dtype=INT8)[..., ::2]),
               dict(shape=(0, 2, 16, 64), scales=(0, 2)), dict(dtype=torch.float8_e5m2)):
        with pytest.raises((TypeError, ValueError)):
            make(**kw)
    with pytest.raises(TypeError):
        lowbit.Cache8.empty(4, 2, 16, 64, BF16)
    assert lowbit.Cache8.bytes_per_block(8, 128, 16) == 2 * 8 * (16 * 128 + 4)


def test_refusals_of_pages_and_products():
    base = dict(new_lens=_i([1]), ctx_lens=_i([0]), block_tables=_i([[0]]), free_pages=_i([0, 1]), ring=_i([0, 2]), block_size=16, max_tokens=4)
    lowbit.page_step(**base)
    for kw in (dict(new_lens=_i([])), dict(ctx_lens=_i([0, 1])), dict(ring=_i([0])), dict(free_pages=_i([])), dict(block_size=12), dict(max_tokens=-1),
               dict(ctx_out=_i([0, 0])), dict(ring_out=torch.zeros(2)), dict(new_lens=torch.tensor([1])), dict(block_size=1 << 30),
               dict(new_lens=torch.zeros(5000, dtype=I32), ctx_lens=torch.zeros(5000, dtype=I32), block_tables=torch.zeros(5000, 1, dtype=I32))):
        with pytest.raises((TypeError, ValueError)):
            lowbit.page_step(**{**base, **kw})
    codes, s = torch.zeros(16, 64, dtype=torch.uint8), torch.ones(16, 1, dtype=BF16)
    w = lowbit.Weight4(codes, s)
    assert (w.n, w.k, w.group) == (16, 128, 128) and w.nbytes() == 16 * 64 + 32
    for args in ((codes.int(), s), (codes, s.float()), (codes, torch.ones(16, 3, dtype=BF16)), (codes, torch.ones(16, 8, dtype=BF16)), (codes, torch.ones(15, 1, dtype=BF16)),
                 (codes, s, torch.ones(16, 2, dtype=torch.uint8)), (codes, s, s)):
        with pytest.raises((TypeError, ValueError)):
            lowbit.Weight4(*args)
    x = torch.zeros(2, 128, dtype=BF16)
    for args in ((x.float(), w), (x[:, :64], w), (x, w, torch.zeros(16)), (x, w, torch.zeros(15, dtype=BF16))):
        with pytest.raises((TypeError, ValueError)):
            lowbit.linear4(*args)
    for args in ((torch.zeros(4, 100), 64), (torch.zeros(4, 128), 16), (torch.zeros(128), 64)):
        with pytest.raises(ValueError):
            lowbit.quantize4(*args)


def _there(x):
    """On the GPU, with a stride where it had one."""
    if not isinstance(x, torch.Tensor):
        return x
    return x.cuda() if x.is_contiguous() else x.cuda().repeat_interleave(2, 1)[:, ::2]


@pytest.mark.gpu
@pytest.mark.parametrize("change,error", [
    (dict(cu_q=torch.tensor([0, 2])), TypeError), (dict(ctx_lens=torch.tensor([2.0])), TypeError), (dict(block_tables=_i([0, 1])), ValueError),
    (dict(block_tables=_i([[0], [1]])), ValueError), (dict(cu_q=_i([0, 1, 2])), ValueError), (dict(block_tables=torch.zeros(1, 0, dtype=I32)), ValueError),
    (dict(block_tables=_i([[0, 1, 2, 3]])[:, ::2]), ValueError), (dict(n_heads=0), ValueError), (dict(n_heads=-1), ValueError), (dict(max_q=-1), ValueError)])
def test_refusals_of_sequences_on_the_gpu(change, error):
    """The same calls are refused, in the same way, where the checks are the launch module's."""
    a = {**_good("cuda"), **{k: _there(v) for k, v in change.items()}}
    with pytest.raises(error):
        lowbit.attention8(torch.zeros(2, 256, dtype=BF16, device="cuda"), **a)
    with pytest.raises(error):
        lowbit.rope_append8(torch.zeros(2, 512, dtype=BF16, device="cuda"), None, **a)


@pytest.mark.gpu
def test_refusals_on_the_gpu():
    rows, there = lambda *s: torch.zeros(*s, dtype=BF16, device="cuda"), dict(device="cuda")
    good = _good("cuda")
    cache = good["cache"]
    for name in ("cu_q", "ctx_lens", "block_tables"):            # one tensor on the CPU
        for fn, args in ((lowbit.attention8, (rows(2, 256),)), (lowbit.rope_append8, (rows(2, 512), None))):
            with pytest.raises(ValueError):
                fn(*args, **{**good, name: good[name].cpu()})
    for kw in (dict(q=torch.zeros(2, 256, **there)), dict(q=rows(2, 255)), dict(q=rows(2, 512)[:, ::2]), dict(q=rows(2, 256).cpu()), dict(q=rows(2, 4, 64)),
               dict(out=rows(1, 256)), dict(out=torch.zeros(2, 256, **there)), dict(out=rows(1, 256).expand(2, 256)), dict(n_heads=3), dict(max_k=-1)):
        a = {**good, "q": rows(2, 256), **kw}
        with pytest.raises((TypeError, ValueError)):
            lowbit.attention8(a.pop("q"), **a)
    for kw in (dict(qkv=rows(2, 511)), dict(qkv=torch.zeros(2, 512, **there)), dict(qkv=rows(2, 512).cpu()), dict(cos_sin=torch.zeros(9, 64, 2, **there)),
               dict(cos_sin=torch.zeros(0, 32, 2, **there)), dict(cos_sin=torch.zeros(9, 32, 2, dtype=F64, **there)), dict(cos_sin=torch.zeros(9, 32, 2)),
               dict(q_out=rows(3, 256)), dict(q_out=rows(2, 200)), dict(q_out=rows(2, 257)[:, 1:])):
        a = {**good, "qkv": rows(2, 512), "cos_sin": None, **kw}
        with pytest.raises((TypeError, ValueError)):
            lowbit.rope_append8(a.pop("qkv"), a.pop("cos_sin"), **a)
    one = (_i([0, 2], "cuda"), _i([0], "cuda"), _i([[0, 1]], "cuda"))
    for args, total in (((one[0].cpu(), *one[1:]), 2), ((one[0].long(), *one[1:]), 2), (one, -1), (one, 1 << 31), ((one[0], one[1], one[2][0]), 2), ((one[0][:1], *one[1:]), 2)):
        with pytest.raises((TypeError, ValueError)):
            lowbit.read8(cache, *args, total=total)
    base = dict(new_lens=_i([1], "cuda"), ctx_lens=_i([0], "cuda"), block_tables=_i([[0]], "cuda"), free_pages=_i([0, 1], "cuda"), ring=_i([0, 2], "cuda"),
                block_size=16, max_tokens=4)
    for kw in (dict(new_lens=_i([], "cuda")), dict(ctx_lens=_i([0, 1], "cuda")), dict(ctx_lens=_i([0])), dict(ring=_i([0], "cuda")), dict(free_pages=_i([], "cuda")),
               dict(block_size=12), dict(max_tokens=-1), dict(max_tokens=1 << 31), dict(ctx_out=_i([0, 0], "cuda")), dict(ctx_out=_i([0])),
               dict(ring_out=torch.zeros(2, **there)), dict(new_lens=torch.tensor([1], **there)), dict(block_size=1 << 30), dict(block_size=1 << 62),
               dict(new_lens=torch.zeros(5000, dtype=I32, **there), ctx_lens=torch.zeros(5000, dtype=I32, **there), block_tables=torch.zeros(5000, 1, dtype=I32, **there))):
        with pytest.raises((TypeError, ValueError)):
            lowbit.page_step(**{**base, **kw})
    codes, s = torch.zeros(16, 64, dtype=torch.uint8, **there), torch.ones(16, 1, dtype=BF16, **there)
    w = lowbit.Weight4(codes, s)
    for args in ((codes.int(), s), (codes, s.float()), (codes, s.cpu()), (codes, torch.ones(16, 3, dtype=BF16, **there)), (codes, s, s)):
        with pytest.raises((TypeError, ValueError)):
            lowbit.Weight4(*args)
    for n in (2, 20, 70):
        x = rows(n, 128)
        for args in ((x.float(), w), (x.cpu(), w), (x[:, :64], w), (x, w, torch.zeros(16, **there)), (x, w, rows(15)), (x, w, rows(16).cpu()), (x, w, rows(32)[::2])):
            with pytest.raises((TypeError, ValueError)):
                lowbit.linear4(*args)

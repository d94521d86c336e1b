"""Rotary positions, page tables, the paged 4-bit cache with its attention, and the verification of drafted tokens against plain
implementations in 64 bits.

Tolerances. A bf16 result is off by half a step, 2^-8 of its value, from the fp32 value behind it. The terms of the fp32 value:
  rotary: cos and sin of an angle that is exact to 2^-40 turns before its rounding to fp32 (2^-25 turns = 2^-22.3 radians at most) and carry 2 ulp
    of their own, each product and sum half an ulp: |err| <= (|a| + |b|) mscale 2^-21 together.
  attention: codes and q are exact, so a score is off by the roundings of its sum: n = hd + 8 of them, each at most 2^-24 of a partial sum that
    |alpha| sum|q| (31 s + |m|) bounds (the kernel may add 16 to every code and take it off again). Roundings to nearest are independent and
    have no mean, so n of them stay under 4 sqrt(n) halves of a step (7 standard deviations of sqrt(n / 3)):
    d = 4 sqrt(hd + 8) 2^-24 |alpha| sum|q| max(31 s + |m|). A weight is then off by 2 d + 2^-15 (exp2 and the sum of the weights: 2^-20; a weight
    handed to the matrix unit as two bf16 parts: 2^-16), which moves the result by that part of max|v|; the sum over L weighted values, with 16
    added to every code, is off by 4 sqrt(L + 64) 2^-24 of at most max(31 s + |m|).
  verification, page tables, codes and read values: equal.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

bf16, f32, f64, i32 = torch.bfloat16, torch.float32, torch.float64, torch.int32
HALF = 2.0 ** -8


def gen(seed):
    return torch.Generator().manual_seed(seed)


def within(out, ref, tol, what=""):
    out, ref = out.detach().cpu().to(f64), ref.cpu().to(f64)
    assert out.shape == ref.shape, (what, out.shape, ref.shape)
    bad = ~((out - ref).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((out - ref).abs().max()):.3g}, first at {bad.nonzero()[0].tolist()}"


# ----------------------------------------------------------------------------- rotary
def rotary_ref(x, pos, freq, interleaved, mscale, backward=False):
    x, rot = x.to(f64), 2 * freq.numel()
    a = pos.to(f64)[:, None, None] * freq.to(f64)
    c, s = torch.cos(a) * mscale, torch.sin(a) * (-mscale if backward else mscale)
    y = x.clone()
    ia = torch.arange(0, rot, 2) if interleaved else torch.arange(rot // 2)
    ib = ia + 1 if interleaved else ia + rot // 2
    y[..., ia], y[..., ib] = x[..., ia] * c - x[..., ib] * s, x[..., ib] * c + x[..., ia] * s
    size = torch.zeros_like(x)
    size[..., ia] = size[..., ib] = (x[..., ia].abs() + x[..., ib].abs()) * mscale
    return y, size


@pytest.mark.parametrize("dtype", [bf16, f32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,hd,rot,scaling", [
    (1, 1, 2, 2, "none"), (3, 5, 8, 6, "linear"), (8, 64, 128, 128, "none"), (37, 4, 80, 80, "yarn"), (5, 3, 96, 48, "ntk"), (259, 40, 128, 64, "yarn"),
    (2, 2, 34, 18, "none"), (1, 7, 256, 256, "linear"), (1030, 2, 64, 32, "none"), (300, 33, 72, 40, "none")])
def test_rotary(dev, dtype, interleaved, rows, heads, hd, rot, scaling):
    from grove_amd import ops
    plan = ops.rotary_plan(rot, interleaved=interleaved, scaling=scaling, factor=1.0 if scaling == "none" else 8.0, device=dev)
    g = gen(rows + hd)
    x = torch.randn(rows, heads, hd, generator=g).to(dtype)
    pos = torch.randint(0, 1 << 20, (rows,), generator=g, dtype=i32)
    pos[0] = 0
    for backward in (False, True):
        ref, size = rotary_ref(x, pos, plan.freq.cpu(), interleaved, plan.mscale, backward)
        tol = size * 2.0 ** -21 + (ref.abs() * HALF if dtype == bf16 else 0)
        d = x.to(dev)
        y = ops.rotary(d, pos.to(dev), plan, backward=backward)
        within(y, ref, tol, f"rotary backward={backward}")
        assert torch.equal(y[..., rot:].cpu(), x[..., rot:]) and torch.equal(d.cpu(), x)
        assert ops.rotary(d, pos.to(dev), plan, backward=backward, out=d) is d and torch.equal(d, y), "in place"


@pytest.mark.parametrize("shift", [0, 1, 3, 8])
def test_rotary_packed_and_unaligned(dev, shift):
    """q and k heads of a packed q | k | v row in one call, at odd starts of the row and odd row strides; v and the gaps stay."""
    from grove_amd import ops
    rows, H, K, hd = 9, 6, 2, 64
    base = torch.randn(rows, (H + 2 * K) * hd + 11 + shift, generator=gen(3)).to(bf16)
    pos = torch.randint(-3, 70000, (rows,), generator=gen(4), dtype=i32)
    plan = ops.rotary_plan(hd, device=dev)
    d = base.to(dev)
    view = lambda t: t[:, shift:shift + (H + K) * hd].unflatten(1, (H + K, hd))  # noqa: E731
    ref, size = rotary_ref(view(base), pos, plan.freq.cpu(), False, 1.0)
    ops.rotary(view(d), pos.to(dev), plan, out=view(d))
    within(view(d), ref, size * 2.0 ** -21 + ref.abs() * HALF)
    assert torch.equal(d[:, :shift].cpu(), base[:, :shift]) and torch.equal(d[:, shift + (H + K) * hd:].cpu(), base[:, shift + (H + K) * hd:])
    out = torch.full((rows, H + K + 1, hd + 6), 7.0, dtype=bf16, device=dev)
    ops.rotary(view(base.to(dev)), pos.to(dev), plan, out=out[:, 1:, 3:3 + hd])
    assert torch.equal(out[:, 1:, 3:3 + hd], view(d))
    assert (out[:, 0] == 7).all() and (out[..., :3] == 7).all() and (out[..., 3 + hd:] == 7).all()


def test_rotary_backward_is_the_gradient(dev):
    """<backward(g), x> = <g, forward(x)>, and a difference quotient of a loss in fp32."""
    from grove_amd import ops
    plan = ops.rotary_plan(24, interleaved=True, scaling="yarn", factor=4.0, device=dev)
    x, gr = (torch.randn(5, 3, 40, generator=gen(s)).to(dev) for s in (1, 2))
    pos = torch.tensor([0, 1, 77, 4095, 100000], dtype=i32, device=dev)
    back = ops.rotary(gr, pos, plan, backward=True)
    a, b = (back.double() * x).sum().item(), (gr.double() * ops.rotary(x, pos, plan)).sum().item()
    size = float((gr.abs().double().sum() * x.abs().max())) * plan.mscale * 2
    assert abs(a - b) <= size * 2.0 ** -21
    loss = lambda t: (ops.rotary(t, pos, plan).double() * gr).sum().item()  # noqa: E731
    for at in [(0, 0, 0), (2, 1, 5), (4, 2, 23), (3, 0, 39)]:
        up, dn = x.clone(), x.clone()
        up[at] += 1
        dn[at] -= 1
        step = float(up[at] - dn[at])
        assert abs((loss(up) - loss(dn)) / step - float(back[at])) <= size * 2.0 ** -21


def test_rotary_nothing(dev):
    from grove_amd import ops
    plan = ops.rotary_plan(8, device=dev)
    assert ops.rotary(torch.zeros(0, 2, 8, device=dev), torch.zeros(0, dtype=i32, device=dev), plan).shape == (0, 2, 8)


# ----------------------------------------------------------------------------- page tables
def pages_ref(ctx, new, table, held, free, P, rows):
    table, held, taken, at = [list(r) for r in table], list(held), 0, 0
    most = len(table[0])
    kv_len, cu, slots, pos = [], [0], [], []
    for b in range(len(ctx)):
        c, n, h = max(ctx[b], 0), max(new[b], 0), max(held[b], 0)
        need = max(0, min(-(-(c + n) // P), most) - h)
        got = 0
        for i in range(need):
            table[b][h + i] = free[taken] if taken < len(free) else -1
            got += taken < len(free)
            taken += 1
        held[b] = h + got
        for t in range(c, c + n):
            page = table[b][t // P] if t // P < most and t // P < h + need else -1
            slots.append(page * P + t % P if page >= 0 else -1)
            pos.append(t)
        kv_len.append(c + n)
        cu.append(cu[-1] + n)
    pad = max(0, rows - len(slots))
    return table, kv_len, cu, (slots + [-1] * pad)[:rows], (pos + [0] * pad)[:rows], held, [taken]


def check_pages(dev, ctx, new, table, held, free, P, rows):
    from grove_amd import ops
    t = lambda v: torch.tensor(v, dtype=i32, device=dev)  # noqa: E731
    wide = torch.full((len(table), len(table[0]) + 3), 99, dtype=i32, device=dev)
    wide[:, :-3] = t(table)
    step = ops.page_tables(t(ctx), t(new), wide[:, :-3], t(held), t(free), P, rows)
    ref = pages_ref(ctx, new, table, held, free, P, rows)
    assert wide[:, :-3].tolist() == ref[0] and (wide[:, -3:] == 99).all()
    for name, a, b in zip(step._fields, step, ref[1:]):
        assert a.tolist() == b, name
    return step


@pytest.mark.parametrize("requests,P,longest,most", [(1, 16, 5, 4), (8, 16, 100, 5), (63, 32, 300, 70), (257, 64, 1000, 9), (700, 1, 9, 6), (4096, 128, 3000, 3)])
def test_page_tables(dev, requests, P, longest, most):
    g = gen(requests)
    ctx = torch.randint(0, longest, (requests,), generator=g).tolist()
    new = [0 if v < 3 else most if v == 9 else 1 for v in torch.randint(0, 10, (requests,), generator=g).tolist()]
    held = [-(-c // P) + v for c, v in zip(ctx, torch.randint(0, 2, (requests,), generator=g).tolist())]  # some hold a page more than they need
    width = max(-(-(c + n) // P) for c, n in zip(ctx, new)) + 2
    ids = torch.randperm(requests * width * 2, generator=g).tolist()
    table, at = [], 0
    for h in held:
        table.append(ids[at:at + h] + [-1] * (width - h))
        at += h
    check_pages(dev, ctx, new, table, held, ids[at:], P, sum(new))
    check_pages(dev, ctx, new, table, held, ids[at:], P, sum(new) + 37)


def test_page_tables_edges(dev):
    empty = [[-1] * 4 for _ in range(3)]
    check_pages(dev, [0, 0, 0], [0, 0, 0], empty, [0, 0, 0], [5, 6], 16, 0)               # nothing at all
    check_pages(dev, [0, 0, 0], [0, 0, 0], empty, [0, 0, 0], [], 16, 4)                   # only padding rows, no free page
    check_pages(dev, [0, 0, 0], [16, 17, 0], empty, [0, 0, 0], [5, 6, 7, 8], 16, 33)      # a page exactly, one token more
    check_pages(dev, [0, 0, 0], [40, 40, 5], empty, [0, 0, 0], [9, 4], 16, 85)            # the pages run out in the first request
    check_pages(dev, [60, 0, 0], [10, 3, 3], [[1, 2, 3, 4]] + empty[1:], [4, 0, 0], [8, 9], 16, 16)  # a row of the table is full
    check_pages(dev, [-5, 3, -1], [2, -7, 1], empty, [-2, 1, 0], [8, 9], 16, 5)           # negative lengths count as none
    check_pages(dev, [5, 5, 5], [3, 3, 3], [[7, -1, -1, -1]] * 3, [1, 1, 1], [], 16, 9)   # nothing new needed
    check_pages(dev, [0, 0, 0], [30, 30, 30], empty, [0, 0, 0], list(range(20)), 16, 50)  # fewer rows asked for than there are


def test_page_tables_again(dev):
    """What ran out is handed out by the next call, and the same call twice gives the same."""
    from grove_amd import ops
    t = lambda v: torch.tensor(v, dtype=i32, device=dev)  # noqa: E731
    table = torch.full((2, 4), -1, dtype=i32, device=dev)
    a = ops.page_tables(t([0, 0]), t([20, 20]), table, t([0, 0]), t([3, 1, 2]), 16, 40)
    assert a.taken.item() == 4 and a.held.tolist() == [2, 1] and table.tolist() == [[3, 1, -1, -1], [2, -1, -1, -1]]
    b = ops.page_tables(t([20, 16]), t([1, 4]), table, a.held, t([8]), 16, 5)
    assert b.taken.item() == 1 and table.tolist() == [[3, 1, -1, -1], [2, 8, -1, -1]] and b.slots.tolist() == [20, 128, 129, 130, 131]
    c = ops.page_tables(t([20, 16]), t([1, 4]), table, a.held, t([8]), 16, 5)
    assert all(torch.equal(x, y) for x, y in zip(b, c))


# ----------------------------------------------------------------------------- the 4-bit cache
def quant_ref(x):
    """codes, scale and minimum of bf16 rows by the formula in 64 bits (finite rows)."""
    x = x.to(f64)
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    span = hi - lo
    mant, ex = torch.frexp(span / 15)
    s = torch.where(span < 2.0 ** -100, torch.zeros_like(span), torch.ldexp(torch.round(mant * 256), ex - 8))
    c = torch.where(s > 0, torch.round((x - lo) / torch.where(s > 0, s, torch.ones_like(s))), torch.zeros_like(x)).clamp(0, 15)
    return c, s, lo


def layout_ref(codes, which, P, hd):
    """The bytes of one (page, head) plane from codes [P, hd], channel by channel as the layout is written down."""
    out = [0] * (P * hd // 2)
    for r in range(P):
        for c in range(hd):
            if which == 0:
                t, h, i = c // 32, (c % 32) // 8, c % 8
                nib = [0, 2, 4, 6, 1, 3, 5, 7].index(i)
                at = r * hd + (h * (hd // 32) + t) * 8 + nib
            else:
                m, j, quad, tok = c % 16, c // 16, r // 4, r % 4
                if hd == 32:
                    at = quad * 4 * hd + m * 8 + [0, 2, 1, 3].index(tok) * 2 + j
                else:
                    at = quad * 4 * hd + m * hd // 4 + (j // 4) * 16 + tok * 4 + j % 4
            out[at // 2] |= int(codes[r, c]) << (4 * (at % 2))
    return torch.tensor(out, dtype=torch.uint8)


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
def test_cache_layout_and_codes(dev, hd):
    from grove_amd import ops
    P, kv, pages = 16, 2, 3
    k, v = (torch.randn(P, kv, hd, generator=gen(hd + s)).to(bf16) for s in (0, 1))
    cache = ops.kv4_cache(pages, P, kv, hd, dev)
    ops.kv4_append(k.to(dev), v.to(dev), cache, torch.arange(P, 2 * P, dtype=i32, device=dev))
    for which, x in enumerate((k, v)):
        c, s, m = quant_ref(x)
        for h in range(kv):
            assert torch.equal(cache.codes[1, which, h].cpu(), layout_ref(c[:, h], which, P, hd)), (which, h)
        assert torch.equal(cache.scales[1, which].cpu().to(f64), torch.cat([s, m], -1).transpose(0, 1))
    assert (cache.codes[0] == 0).all() and (cache.codes[2] == 0).all() and (cache.scales[0] == 0).all() and (cache.scales[2] == 0).all()


@pytest.mark.parametrize("rows,kv,hd,P", [(1, 1, 32, 16), (5, 32, 128, 64), (40, 3, 64, 32), (203, 8, 128, 16), (77, 2, 256, 128), (1000, 4, 64, 256), (64, 5, 32, 16)])
def test_cache_round_trip(dev, rows, kv, hd, P):
    """Scattered slots in shuffled order, k and v as columns of a packed row at an odd start; the other rows of the cache keep their bytes."""
    from grove_amd import ops
    pages = -(-rows // P) + 2
    g = gen(rows + hd)
    packed = (torch.randn(rows, 2 * kv * hd + 5, generator=g) * torch.rand(1, 2 * kv * hd + 5, generator=g) * 4).to(bf16)
    view = lambda t, i: t[:, 1 + i * kv * hd:1 + (i + 1) * kv * hd].unflatten(1, (kv, hd))  # noqa: E731
    slots = torch.randperm(pages * P, generator=g)[:rows].to(i32)
    cache = ops.kv4_cache(pages, P, kv, hd, dev)
    old = torch.randn(pages * P, kv, hd, generator=g).to(bf16).to(dev)
    every = torch.arange(pages * P, dtype=i32, device=dev)
    ops.kv4_append(old, old, cache, every)
    before = [t.cpu() for t in ops.kv4_read(cache, every, f32)]
    d = packed.to(dev)
    ops.kv4_append(view(d, 0), view(d, 1), cache, slots.to(dev))
    after = [t.cpu() for t in ops.kv4_read(cache, every, f32)]
    got = ops.kv4_read(cache, slots.to(dev), f32)
    got16 = ops.kv4_read(cache, slots.to(dev))
    for i in range(2):
        c, s, m = quant_ref(view(packed, i))
        ref = (m + c * s).to(f32)
        assert torch.equal(got[i].cpu(), ref) and torch.equal(got16[i].cpu(), ref.to(bf16))
        before[i][slots.long()] = ref
        assert torch.equal(before[i], after[i])


def test_cache_odd_rows(dev):
    """Constant rows, tiny and huge ranges, ties of the rounding, infinities and NaN, slots outside."""
    from grove_amd import ops
    hd, P = 64, 16
    x = torch.zeros(9, 1, hd)
    x[0] = 3.5                                                     # constant: scale 0
    x[1, 0, 5] = 1e-38                                             # a range below 2^-100
    x[2, 0, :2] = torch.tensor([2.0 ** 126, -2.0 ** 126])          # a huge one
    x[3, 0] = torch.arange(hd) % 31 / 2 - 7.5                      # steps of 1/2 at scale 1: every second value is a tie
    x[4, 0, 9] = math.inf
    x[5, 0, 9] = math.nan
    x[6, 0, 9], x[6, 0, 10] = 3e38, -3e38                          # finite values, a range beyond fp32
    x[7, 0, 63] = -1.0
    x[8, 0] = torch.linspace(-1, 2, hd)
    x = x.to(bf16)
    cache = ops.kv4_cache(2, P, 1, hd, dev)
    slots = torch.arange(9, dtype=i32, device=dev)
    ops.kv4_append(x.to(dev), x.to(dev), cache, slots)
    for got in ops.kv4_read(cache, slots, f32):
        got = got.cpu()
        good = [0, 1, 2, 3, 7, 8]
        c, s, m = quant_ref(x[good])
        assert torch.equal(got[good], (m + c * s).to(f32))
        assert got[[4, 5, 6]].isnan().all()
    codes = cache.codes.clone()
    out = torch.tensor([-1, 32, 2 ** 31 - 1, -2 ** 31, 100, 33, -7, 999, 32], dtype=i32, device=dev)
    ops.kv4_append(x.to(dev), x.to(dev), cache, out)
    assert torch.equal(codes, cache.codes) and all((t == 0).all() for t in ops.kv4_read(cache, out))
    none = torch.zeros(0, dtype=i32, device=dev)
    ops.kv4_append(x[:0].to(dev), x[:0].to(dev), cache, none)
    assert ops.kv4_read(cache, none)[0].shape == (0, 1, hd)


# ----------------------------------------------------------------------------- attention
class Paged:
    """A cache filled through kv4_append at shuffled pages, its rows in fp64, and every row that no request owns poisoned."""

    def __init__(self, dev, lens, kv, hd, P, seed=0, extra=2, spread=1.0, held_more=0):
        from grove_amd import ops
        g = gen(seed)
        self.dev, self.lens, self.P, self.kv, self.hd = dev, lens, P, kv, hd
        need = [-(-n // P) for n in lens]
        pages = max(1, sum(need) + extra)
        self.cache = ops.kv4_cache(pages, P, kv, hd, dev)
        self.cache.codes.fill_(0xFF)
        self.cache.scales.fill_(math.nan)
        ids = torch.randperm(pages, generator=g).tolist()
        width = max(1, max(need)) + held_more
        self.table = torch.full((len(lens), width), -1, dtype=i32)
        slots = []
        for b, n in enumerate(lens):
            mine, ids = ids[:need[b]], ids[need[b]:]
            self.table[b, :need[b]] = torch.tensor(mine, dtype=i32)
            self.table[b, need[b]:] = torch.tensor([2 ** 30, -5, pages][b % 3], dtype=i32)
            slots += [mine[t // P] * P + t % P for t in range(n)]
        self.slots = torch.tensor(slots, dtype=i32, device=dev)
        self.table = self.table.to(dev)
        k, v = (torch.randn(len(slots), kv, hd, generator=g) * spread for _ in range(2))
        k *= 0.3 + torch.rand(kv, hd, generator=g)
        ops.kv4_append(k.to(bf16).to(dev), v.to(bf16).to(dev), self.cache, self.slots)
        self.k, self.v = (t.cpu().to(f64).split(lens) for t in ops.kv4_read(self.cache, self.slots, f32))
        s = [(t.amax(-1) - t.amin(-1)) / 15 for t in (torch.cat(self.k), torch.cat(self.v))] if slots else [torch.zeros(1)] * 2
        top = [t.abs().max() if t.numel() else torch.zeros(()) for t in (torch.cat(self.k), torch.cat(self.v))]
        self.size = [float(31 * a.max() + b) for a, b in zip(s, top)]

    def ref(self, q, new, alpha):
        """(attention in 64 bits, tolerance) of packed rows q."""
        H, hd = q.shape[1:]
        out, tol, at = [], [], 0
        for b, n in enumerate(new):
            x, L = q[at:at + n].to(f64), self.lens[b]
            at += n
            k, v = (t[b].repeat_interleave(H // self.kv, 1) for t in (self.k, self.v))
            z = torch.einsum("nhd,lhd->hnl", x, k) * alpha
            dead = torch.arange(L)[None] >= torch.arange(L - n + 1, L + 1)[:, None]
            z = z.masked_fill(dead, -math.inf)
            w = torch.softmax(z, -1).nan_to_num(0.0) if L else z
            o = torch.einsum("hnl,lhd->nhd", w, v)
            d = 4 * math.sqrt(hd + 8) * 2.0 ** -24 * abs(alpha) * x.abs().sum(-1) * self.size[0]
            out.append(o)
            top = float(v.abs().max()) if L else 0.0
            tol.append(o.abs() * HALF + ((2 * d + 2.0 ** -15) * top + 4 * math.sqrt(L + 64) * 2.0 ** -24 * self.size[1])[..., None])
        return torch.cat(out).flatten(1), torch.cat(tol).flatten(1)


def check_attn(dev, lens, new, H, kv, hd, P, seed=0, max_q=None, max_len="known", q_scale=1.5, alpha=None, **kw):
    from grove_amd import ops
    c = Paged(dev, lens, kv, hd, P, seed, **kw)
    T = sum(new)
    q = (torch.randn(T, H, hd, generator=gen(seed + 1)) * q_scale).to(bf16)
    alpha = hd ** -0.5 if alpha is None else alpha
    cu = torch.tensor([0] + torch.tensor(new).cumsum(0).tolist(), dtype=i32, device=dev)
    kv_len = torch.tensor(lens, dtype=i32, device=dev)
    out = ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, max(new) if max_q is None else max_q, alpha,
                       max_len=max(lens) if max_len == "known" else max_len)
    ref, tol = c.ref(q, new, alpha)
    within(out, ref, tol, f"attention {lens[:4]} {new[:4]} H={H}/{kv} hd={hd} P={P}")
    return c, q, cu, kv_len, out


@pytest.mark.parametrize("hd", [32, 64, 128, 256])
@pytest.mark.parametrize("H,kv", [(1, 1), (4, 4), (8, 2), (7, 1), (16, 2), (14, 2)])
def test_attn_heads(dev, hd, H, kv):
    check_attn(dev, [1, 17, 100, 131], [1, 1, 1, 1], H, kv, hd, 16, seed=hd + H)
    check_attn(dev, [33, 5, 260], [5, 5, 5], H, kv, hd, 32, seed=hd + H + 1)


@pytest.mark.parametrize("P", [16, 32, 64, 128, 256])
@pytest.mark.parametrize("new", [1, 2, 8, 9, 17])
def test_attn_pages_and_queries(dev, P, new):
    """Lengths around tile and page borders."""
    lens = [new + d for d in (0, 1, 14, 15, 16, 31, 32, 33, 63, 64, 65, 127, 128, 255, 256, 257, 300)]
    check_attn(dev, lens, [new] * len(lens), 4, 2, 64, P, seed=P + new)


def test_attn_empty_rows(dev):
    """Requests without rows, without keys, with fewer keys than new tokens (their first rows see nothing and come back as zeros)."""
    c, q, cu, kv_len, out = check_attn(dev, [0, 3, 40, 0, 2, 70], [0, 5, 0, 2, 2, 3], 4, 2, 128, 16)
    assert (out[:2] == 0).all() and (out[5:7] == 0).all() and not (out[2:5] == 0).all(1).any()


@pytest.mark.parametrize("lens,new,H,kv,hd,P", [
    ([5000], [1], 8, 8, 128, 64), ([5000], [5], 16, 2, 128, 16), ([9001, 3], [2, 1], 4, 1, 64, 128), ([2500] * 3, [1] * 3, 8, 1, 256, 32),
    ([4097, 1, 64, 700], [8, 1, 3, 4], 16, 2, 128, 256), ([1500] * 40, [1] * 40, 4, 4, 64, 64), ([3000], [40], 8, 2, 32, 32)])
def test_attn_long(dev, lens, new, H, kv, hd, P):
    """Long enough that a request's keys go to several blocks."""
    check_attn(dev, lens, new, H, kv, hd, P, seed=11)


def test_attn_length_hints(dev):
    """max_len and a table wider than the lengths need change the split only; a max_len that is too short loses no key."""
    args = ([900, 30, 2000], [3, 1, 2], 8, 2, 128, 32)
    for max_len in (None, 2000, 100000, 100, 1):
        check_attn(dev, *args, seed=5, max_len=max_len, max_q=7, held_more=40)


def test_attn_peaked_and_large_scores(dev):
    """One key takes all the weight; scores of some thousands; a weightless softmax; a negative alpha."""
    check_attn(dev, [300, 64], [2, 1], 4, 2, 128, 16, q_scale=40.0)
    check_attn(dev, [300, 64], [2, 1], 4, 2, 128, 16, alpha=0.0)
    check_attn(dev, [300, 64], [2, 1], 4, 2, 128, 16, alpha=-0.05)
    check_attn(dev, [200], [1], 4, 4, 64, 16, spread=1e-3)


@pytest.mark.parametrize("H,kv,new,hd", [(4, 2, 1, 64), (8, 1, 4, 128), (16, 2, 8, 64), (4, 4, 3, 256)])
def test_attn_climbing_scores(dev, H, kv, new, hd):
    """Keys that outgrow everything before them again and again: the references of the running softmax have to follow."""
    from grove_amd import ops
    L, P = 700, 16
    c = Paged(dev, [L, 40], kv, hd, P, seed=71)
    g = gen(72)
    q = (torch.randn(2 * new, H, hd, generator=g) + 1.0).to(bf16)
    k = torch.randn(L, kv, hd, generator=g) * 0.05 + (torch.arange(L) ** 2 / 2000.0)[:, None, None] * (1 + torch.rand(kv, hd, generator=g)) / hd ** 0.5
    v = torch.randn(L, kv, hd, generator=g)
    ops.kv4_append(k.to(bf16).to(dev), v.to(bf16).to(dev), c.cache, c.slots[:L])
    kk, vv = (t.cpu().to(f64) for t in ops.kv4_read(c.cache, c.slots, f32))
    c.k, c.v = kk.split([L, 40]), vv.split([L, 40])
    step = [(t.amax(-1) - t.amin(-1)) / 15 for t in (kk, vv)]
    c.size = [float(31 * s.max() + t.abs().max()) for s, t in zip(step, (kk, vv))]
    cu = torch.tensor([0, new, 2 * new], dtype=i32, device=dev)
    out = ops.kv4_attn(q.to(dev), c.cache, c.table, torch.tensor([L, 40], dtype=i32, device=dev), cu, new, 1.0)
    ref, tol = c.ref(q, [new, new], 1.0)
    within(out, ref, tol)


@pytest.mark.parametrize("H,kv,new,hd", [(4, 4, 1, 32), (2, 1, 1, 64), (8, 2, 2, 128), (8, 1, 4, 128), (8, 1, 8, 128), (16, 1, 4, 64), (4, 4, 1, 256), (8, 2, 5, 256)])
@pytest.mark.parametrize("max_len", [1, None])
def test_attn_scores_that_climb_all_along(dev, H, kv, new, hd, max_len):
    """Every 128 keys pass the references of those before them (by some 40 in units of log2), one and many blocks per pair."""
    from grove_amd import ops
    L, P = 3000, 64
    c = Paged(dev, [L, 40], kv, hd, P, seed=73)
    g = gen(74)
    q = (1.0 + 0.1 * torch.randn(new + 1, H, hd, generator=g)).to(bf16)
    k = (torch.arange(L) * 0.22 / hd)[:, None, None] * (1 + 0.1 * torch.rand(1, kv, hd, generator=g))
    v = torch.randn(L, kv, hd, generator=g)
    ops.kv4_append(k.to(bf16).to(dev), v.to(bf16).to(dev), c.cache, c.slots[:L])
    kk, vv = (t.cpu().to(f64) for t in ops.kv4_read(c.cache, c.slots, f32))
    c.k, c.v = kk.split([L, 40]), vv.split([L, 40])
    step = [(t.amax(-1) - t.amin(-1)) / 15 for t in (kk, vv)]
    c.size = [float(31 * s.max() + t.abs().max()) for s, t in zip(step, (kk, vv))]
    cu = torch.tensor([0, new, new + 1], dtype=i32, device=dev)
    out = ops.kv4_attn(q.to(dev), c.cache, c.table, torch.tensor([L, 40], dtype=i32, device=dev), cu, new, 1.0, max_len=max_len)
    ref, tol = c.ref(q, [new, 1], 1.0)
    within(out, ref, tol)


@pytest.mark.parametrize("max_len", [1, 4000])
@pytest.mark.parametrize("H,kv,hd", [(4, 2, 64), (24, 2, 128)])
def test_attn_more_new_tokens_than_said(dev, H, kv, hd, max_len):
    """Rows past max_q are NaN, whatever the memory held, and the others right."""
    from grove_amd import ops
    c = Paged(dev, [300, 50, 7], kv, hd, 16, seed=75)
    new = [4, 2, 3]
    q = torch.randn(10, H, hd, generator=gen(76)).to(bf16)
    cu = torch.tensor([0, 4, 6, 9], dtype=i32, device=dev)
    kv_len = torch.tensor(c.lens, dtype=i32, device=dev)
    ref, tol = c.ref(q[:9], new, 0.1)
    for given in (False, True):
        out = torch.full((10, H * hd), 5.0, dtype=bf16, device=dev) if given else None
        got = ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, 2, 0.1, max_len=max_len, out=out).cpu()
        past = torch.tensor([0, 0, 1, 1, 0, 0, 0, 0, 1, 0], dtype=torch.bool)
        assert got[past].isnan().all()
        within(got[:9][~past[:9]], ref[~past[:9]], tol[~past[:9]])
        assert (got[9] == (5.0 if given else 0.0)).all()


def test_attn_single_key_is_its_value(dev):
    c, q, cu, kv_len, out = check_attn(dev, [1, 1], [1, 1], 4, 2, 128, 16)
    v = torch.stack([c.v[b][0].repeat_interleave(2, 0) for b in range(2)]).flatten(1)
    assert torch.equal(out.cpu(), v.to(f32).to(bf16))


def test_attn_strides_padding_and_out(dev):
    """q as columns of a packed row, out with a row stride, rows behind the last request: kept in `out`, zeros in a new tensor."""
    from grove_amd import ops
    lens, new, H, kv, hd = [50, 9, 200], [2, 1, 3], 8, 2, 64
    c, q, cu, kv_len, first = check_attn(dev, lens, new, H, kv, hd, 16, seed=8)
    packed = torch.full((9, 3 + (H + 2) * hd), math.nan, dtype=bf16, device=dev)
    packed[:6, 3 + hd:3 + (H + 1) * hd] = q.to(dev).flatten(1)
    view = packed[:, 3 + hd:3 + (H + 1) * hd].unflatten(1, (H, hd))
    out = torch.full((9, H * hd + 24), 5.0, dtype=bf16, device=dev)
    r = ops.kv4_attn(view, c.cache, c.table, kv_len, cu, 3, hd ** -0.5, out=out[:, 8:8 + H * hd])
    assert torch.equal(r[:6], first)
    assert (out[6:] == 5).all() and (out[:, :8] == 5).all() and (out[:, 8 + H * hd:] == 5).all()
    r = ops.kv4_attn(view, c.cache, c.table, kv_len, cu, 3, hd ** -0.5)
    assert torch.equal(r[:6], first) and (r[6:] == 0).all()


def test_attn_unseen_rows_hold_anything(dev):
    """A NaN row that later queries see and earlier ones do not; infinite scales behind the end."""
    from grove_amd import ops
    lens, new, H, kv, hd, P = [45, 80], [4, 4], 4, 2, 64, 16
    c, q, cu, kv_len, out = check_attn(dev, lens, new, H, kv, hd, P, seed=21)
    k = torch.randn(1, kv, hd, device=dev).to(bf16)
    k[0, 1, 3] = math.inf
    last = c.slots[44:45]  # token 44 of request 0: its queries 0..2 do not see it, query 3 does
    good = torch.randn(1, kv, hd, device=dev).to(bf16)
    ops.kv4_append(k, good, c.cache, last)
    r = ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, 4, hd ** -0.5).view(8, H, hd)
    o = out.view(8, H, hd)
    assert torch.equal(r[:3], o[:3]) and torch.equal(r[4:], o[4:])
    assert r[3, 2:].isnan().all() and r[3, :2].isfinite().all(), "head 1's key row is NaN for the query that sees it"
    ops.kv4_append(good, k, c.cache, last)
    r = ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, 4, hd ** -0.5).view(8, H, hd)
    assert torch.equal(r[:3], o[:3]) and r[3, 2:].isnan().all() and r[3, :2].isfinite().all()


def test_attn_bad_pages_are_not_seen(dev):
    """Table entries outside the cache within a request's length: their keys drop out, nothing is read there."""
    from grove_amd import ops
    lens, H, kv, hd, P = [100, 100, 100], 4, 2, 64, 16
    c, q, cu, kv_len, _ = check_attn(dev, lens, [1, 1, 1], H, kv, hd, P, seed=31)
    table = c.table.clone()
    table[0, 2], table[1, 6], table[2, :] = -1, 2 ** 31 - 1, -2 ** 31
    c.lens, keep = [84, 96, 0], [list(range(32)) + list(range(48, 100)), list(range(96)), []]
    c.k, c.v = ([t[b][keep[b]] for b in range(3)] for t in (c.k, c.v))
    c.lens = [len(x) for x in keep]
    out = ops.kv4_attn(q.to(dev), c.cache, table, kv_len, cu, 1, hd ** -0.5)
    ref, tol = c.ref(q, [1, 1, 1], hd ** -0.5)
    within(out, ref, tol)
    assert (out[2] == 0).all()


def test_attn_lengths_past_the_table(dev):
    """kv_len beyond what the table holds is cut; cu_q beyond the rows of q reads and writes nothing outside."""
    from grove_amd import ops
    c, q, cu, kv_len, out = check_attn(dev, [64, 64], [1, 1], 4, 2, 64, 16, seed=41)
    r = ops.kv4_attn(q.to(dev), c.cache, c.table[:, :4], kv_len + 1000, cu, 1, 0.125)
    assert torch.equal(r, out)
    wild = torch.tensor([0, 1, 900], dtype=i32, device=dev)
    r = ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, wild, 1, 0.125)
    assert torch.equal(r[0], out[0])


@pytest.mark.parametrize("lens,H,kv,hd,P", [([300, 33], 8, 2, 64, 16), ([500], 4, 4, 128, 32), ([130, 1, 0], 16, 2, 128, 64), ([90], 4, 1, 256, 16)])
def test_attn_whole_prompts(dev, lens, H, kv, hd, P):
    """Every token of the cache is new: the causal triangle from its first row, many column chunks."""
    check_attn(dev, lens, lens, H, kv, hd, P, seed=81)


def test_attn_nothing(dev):
    """No rows; rows of nobody with max_q 0; lengths below zero."""
    from grove_amd import ops
    c, q, cu, kv_len, out = check_attn(dev, [20, 30], [2, 1], 4, 2, 64, 16, seed=91)
    none = torch.zeros(3, dtype=i32, device=dev)
    assert ops.kv4_attn(q[:0].to(dev), c.cache, c.table, kv_len, none, 0, 1.0).shape == (0, 256)
    assert (ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, none, 0, 1.0) == 0).all()
    assert (ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, none, 3, 1.0) == 0).all()
    assert (ops.kv4_attn(q.to(dev), c.cache, c.table, torch.full_like(kv_len, -2 ** 31), cu, 2, 1.0) == 0).all()
    assert torch.equal(ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, 2, 0.125), out)


def test_attn_offsets_past_32_bits(dev):
    """The last pages of a cache of more than 4 GiB of codes."""
    from grove_amd import ops
    kv, hd, P, pages, L = 8, 128, 64, 70000, 150
    cache = ops.KV4Cache(torch.empty(pages, 2, kv, P * hd // 2, dtype=torch.uint8, device=dev), torch.empty(pages, 2, kv, P, 2, dtype=bf16, device=dev))
    table = torch.tensor([[69999, 3, 69997]], dtype=i32, device=dev)
    slots = (table[0, torch.arange(L, device=dev) // P] * P + torch.arange(L, device=dev) % P).to(i32)
    k, v = (torch.randn(L, kv, hd, generator=gen(s)).to(bf16) for s in (1, 2))
    ops.kv4_append(k.to(dev), v.to(dev), cache, slots)
    c = Paged.__new__(Paged)
    c.kv, c.lens, c.k, c.v, c.size = kv, [L], [], [], []
    for x, got, store in zip((k, v), ops.kv4_read(cache, slots, f32), (c.k, c.v)):
        codes, s, m = quant_ref(x)
        assert torch.equal(got.cpu(), (m + codes * s).to(f32))
        store.append(got.cpu().to(f64))
        c.size.append(float((31 * s).max() + got.abs().max()))
    q = torch.randn(2, 32, hd, generator=gen(3)).to(bf16)
    out = ops.kv4_attn(q.to(dev), cache, table, torch.tensor([L], dtype=i32, device=dev), torch.tensor([0, 2], dtype=i32, device=dev), 2, hd ** -0.5)
    ref, tol = c.ref(q, [2], hd ** -0.5)
    within(out, ref, tol)


def test_attn_same_bits_every_time(dev):
    from grove_amd import ops
    c, q, cu, kv_len, out = check_attn(dev, [7000, 30], [2, 1], 8, 2, 128, 64, seed=51)
    for _ in range(5):
        assert torch.equal(out, ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, 2, 128 ** -0.5, max_len=7000))


# ----------------------------------------------------------------------------- verification
def verify_ref(draft, q, p, u, pick, count):
    B, K = draft.shape
    V = p.shape[2]
    tokens, accepted = torch.full((B, K + 1), -1, dtype=i32), torch.zeros(B, dtype=i32)
    for b in range(B):
        n = K if count is None else max(0, min(K, int(count[b])))
        a = 0
        while a < n:
            x = int(draft[b, a])
            if not (0 <= x < V and float(u[b, a]) * (float(q[b, a, x]) if q is not None else 1.0) < float(p[b, a, x])):
                break
            tokens[b, a] = x
            a += 1
        row = p[b, a].to(f64)
        rest = row
        if a < n:
            off = torch.zeros(V, dtype=f64)
            if q is not None:
                off = q[b, a].to(f64)
            elif 0 <= int(draft[b, a]) < V:
                off[int(draft[b, a])] = 1.0
            left = (row - off).clamp(min=0)
            rest = left if left.sum() > 0 else row
        cdf = rest.cumsum(0)
        over = (cdf > float(pick[b]) * cdf[-1]).nonzero()
        tokens[b, a] = int(over[0]) if len(over) else int(rest.nonzero()[-1]) if (rest > 0).any() else -1
        accepted[b] = a
    return tokens, accepted


def drafts(B, K, V, seed, dtype=f32, agree=0.4):
    g = gen(seed)
    z = torch.randn(B, K + 1, V, generator=g) * 2
    p = torch.softmax(z, -1)
    q = torch.softmax(z[:, :K] + agree * torch.randn(B, K, V, generator=g), -1)
    d = torch.multinomial(q.flatten(0, 1), 1, generator=g).view(B, K).to(i32) if K else torch.zeros(B, 0, dtype=i32)
    return d, q.to(dtype), p.to(dtype), torch.rand(B, K, generator=g), torch.rand(B, generator=g)


def check_verify(dev, d, q, p, u, pick, count=None):
    from grove_amd import ops
    up = lambda t: None if t is None else t.to(dev)  # noqa: E731
    tokens, accepted = ops.verify_drafts(up(d), up(q), up(p), up(u), up(pick), count=up(count))
    ref = verify_ref(d, q, p, u, pick, count)
    assert torch.equal(accepted.cpu(), ref[1]), (accepted.tolist(), ref[1].tolist())
    assert torch.equal(tokens.cpu(), ref[0]), (tokens.tolist(), ref[0].tolist())
    return tokens


@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (3, 2, 5), (40, 4, 320), (8, 4, 32008), (5, 7, 1023), (6, 1, 1025), (2, 3, 128001), (300, 3, 64), (1, 70, 40),
                                   (2, 1, 1100003), (600, 1, 9001)])
def test_verify(dev, dtype, B, K, V):
    d, q, p, u, pick = drafts(B, K, V, B + V, dtype)
    check_verify(dev, d, q, p, u, pick)
    count = torch.randint(-1, K + 2, (B,), generator=gen(V), dtype=i32)
    check_verify(dev, d, q, p, u, pick, count)
    check_verify(dev, d, None, p, u, pick, count)


def test_verify_edges(dev):
    B, K, V = 6, 3, 50
    d, q, p, u, pick = drafts(B, K, V, 9)
    check_verify(dev, d, q, p, torch.zeros_like(u), torch.zeros_like(pick))                     # u = 0 takes every draft that the target can say
    check_verify(dev, d, q, p, torch.full_like(u, 1 - 2.0 ** -24), torch.full_like(pick, 1 - 2.0 ** -24))
    check_verify(dev, d, p[:, :K].clone(), p, u, pick)                                          # drafter = target: all accepted
    same = p[:, :K].clone()
    none = same.clone()
    none.scatter_(2, d.long()[..., None], 0.0)                                                  # q = 0 at the draft: u * 0 < p
    check_verify(dev, d, none, p, u, pick)
    gone = p.clone()
    gone[:, :K].scatter_(2, d.long()[..., None], 0.0)                                           # p = 0 at the draft: refused at once
    t = check_verify(dev, d, q, gone, u, pick)
    assert (t[:, 1:] == -1).all() and (t[:, 0].cpu() != d[:, 0]).all()
    bad = d.clone()
    bad[0, 0], bad[1, 1], bad[2, 2] = -1, V, 2 ** 31 - 1                                        # tokens that do not exist
    check_verify(dev, bad, q, p, u, pick)
    check_verify(dev, bad, None, p, u, pick)
    zero = p.clone()
    zero[0] = 0
    assert check_verify(dev, d, q, zero, u, pick)[0, 0] == -1                                   # no mass at all
    sure = torch.zeros_like(p)
    sure[..., 7] = 1.0
    assert (check_verify(dev, torch.full_like(d, 7), None, sure, u, pick) == 7).all()
    d, q, p, u, pick = drafts(4, 0, 33, 2)
    check_verify(dev, d, None, p, u, pick)                                                      # no drafts: a draw from the target


def test_verify_strides(dev):
    """Rows of packed logits: vocab padded behind, requests as slices of one tensor."""
    from grove_amd import ops
    d, q, p, u, pick = drafts(5, 2, 77, 3)
    P, Q = (torch.full((7, s, 90), 9.0, device=dev) for s in (4, 3))
    P[1:6, 1:, 3:80], Q[1:6, :2, 5:82] = p.to(dev), q.to(dev)
    got = ops.verify_drafts(d.to(dev), Q[1:6, :2, 5:82], P[1:6, 1:, 3:80], u.to(dev), pick.to(dev))
    ref = verify_ref(d, q, p, u, pick, None)
    assert torch.equal(got[0].cpu(), ref[0]) and torch.equal(got[1].cpu(), ref[1])


def test_verify_keeps_the_distribution(dev):
    """Token frequencies of one drafted position are the target's: 200000 draws against p by a bound on binomial deviations (6 sigma)."""
    from grove_amd import ops
    N, V = 200000, 8
    g = torch.Generator(device=dev).manual_seed(4)
    p, q = (torch.softmax(torch.randn(V, generator=gen(s)) * 1.5, 0) for s in (1, 2))
    d = torch.multinomial(q.to(dev), N, True, generator=g).to(i32).view(N, 1)
    P, Q = p.to(dev).expand(N, 2, V), q.to(dev).expand(N, 1, V)
    tokens, _ = ops.verify_drafts(d, Q, P, torch.rand(N, 1, device=dev, generator=g), torch.rand(N, device=dev, generator=g))
    freq = torch.bincount(tokens[:, 0].long(), minlength=V).cpu().double() / N
    assert ((freq - p).abs() <= 6 * torch.sqrt(p.double() * (1 - p.double()) / N)).all(), (freq, p)


# ----------------------------------------------------------------------------- together
def test_serving_steps_together(dev):
    """Some steps of three requests with drafts: tables, rotary, append, attention, verification, each against its 64-bit form; refused drafts'
    rows are written again by the next step."""
    from grove_amd import ops
    H, kv, hd, P, K, V = 8, 2, 64, 16, 3, 50
    g = gen(77)
    plan = ops.rotary_plan(hd // 2, interleaved=True, scaling="yarn", factor=4.0, device=dev)
    cache = ops.kv4_cache(40, P, kv, hd, dev)
    free = torch.randperm(40, generator=g).to(i32).to(dev)
    table = torch.full((3, 12), -1, dtype=i32, device=dev)
    ctx, held = torch.zeros(3, dtype=i32, device=dev), torch.zeros(3, dtype=i32, device=dev)
    keys, values = [torch.zeros(0, kv, hd, dtype=f64) for _ in range(3)], [torch.zeros(0, kv, hd, dtype=f64) for _ in range(3)]
    for step in range(6):
        new = [29, 1, 17] if step == 0 else [K + 1] * 3
        T = sum(new)
        s = ops.page_tables(ctx, torch.tensor(new, dtype=i32, device=dev), table, held, free, P, T)
        free, held = free[int(s.taken):], s.held
        qkv = torch.randn(T, H + 2 * kv, hd, generator=g).to(bf16)
        d = qkv.to(dev)
        ops.rotary(d[:, :H + kv], s.pos, plan, out=d[:, :H + kv])
        rot, size = rotary_ref(qkv[:, :H + kv], s.pos.cpu(), plan.freq.cpu(), True, plan.mscale)
        within(d[:, :H + kv], rot, size * 2.0 ** -21 + rot.abs() * HALF)
        ops.kv4_append(d[:, H:H + kv], d[:, H + kv:], cache, s.slots)
        out = ops.kv4_attn(d[:, :H], cache, table, s.kv_len, s.cu_q, max(new), hd ** -0.5)
        host, at = d.cpu(), 0
        view = Paged.__new__(Paged)
        view.kv, view.lens, view.k, view.v = kv, s.kv_len.tolist(), [], []
        for b, n in enumerate(new):
            c0 = int(ctx[b])
            for store, lo in ((keys, H), (values, H + kv)):
                c, sc, m = quant_ref(host[at:at + n, lo:lo + kv])
                store[b] = torch.cat([store[b][:c0], m + c * sc])
            at += n
        view.k, view.v = [t.to(f32).to(f64) for t in keys], [t.to(f32).to(f64) for t in values]
        view.size = [float(31 * 2 * max(float(t.abs().max()) for t in x) / 15 + max(float(t.abs().max()) for t in x)) for x in (keys, values)]
        ref, tol = view.ref(host[:, :H], new, hd ** -0.5)
        within(out, ref, tol, f"step {step}")
        if step == 0:
            ctx = s.kv_len.clone()
            continue
        dr, q, p, u, pick = drafts(3, K, V, step, agree=0.2)
        tokens, accepted = ops.verify_drafts(*(t.to(dev) for t in (dr, q, p, u, pick)))
        r = verify_ref(dr, q, p, u, pick, None)
        assert torch.equal(tokens.cpu(), r[0]) and torch.equal(accepted.cpu(), r[1])
        ctx = ctx + accepted + 1


def test_serving_step_in_a_graph(dev):
    """A captured step replayed with other lengths, keys and numbers, with eager work between the replays, against the eager step."""
    from grove_amd import ops
    B, H, kv, hd, P, K, V = 2, 8, 2, 128, 32, 2, 1000
    T = B * (K + 1) + 2  # two rows of padding
    plan = ops.rotary_plan(hd, device=dev)
    cache = ops.kv4_cache(300, P, kv, hd, dev)
    every = torch.arange(300 * P, dtype=i32, device=dev)
    old = torch.randn(300 * P, kv, hd, generator=gen(1)).to(bf16).to(dev)
    ops.kv4_append(old, old.flip(0), cache, every)
    start = torch.randperm(300, generator=gen(2)).to(i32).to(dev)
    ctx, new, held = (torch.zeros(B, dtype=i32, device=dev) for _ in range(3))
    table, free = torch.zeros(B, 140, dtype=i32, device=dev), start[:20].clone()
    qkv = torch.zeros(T, H + 2 * kv, hd, dtype=bf16, device=dev)
    d, q, p, u, pick = (t.to(dev) for t in drafts(B, K, V, 3))

    def body():
        s = ops.page_tables(ctx, new, table, held, free, P, T)
        x = ops.rotary(qkv[:, :H + kv], s.pos, plan)
        ops.kv4_append(x[:, H:], qkv[:, H + kv:], cache, s.slots)
        o = ops.kv4_attn(x[:, :H], cache, table, s.kv_len, s.cu_q, K + 1, hd ** -0.5)
        return (*s, x, o, *ops.verify_drafts(d, q, p, u, pick))

    def load(i):
        g = gen(100 + i)
        c = [[4000, 33], [1, 4100], [640, 639], [31, 32]][i]
        ctx.copy_(torch.tensor(c, dtype=i32))
        new.copy_(torch.tensor([K + 1, K + 1 - i % 2], dtype=i32))
        held.copy_(torch.tensor([-(-v // P) for v in c], dtype=i32))
        table.copy_(start[20:].view(2, 140))
        qkv.copy_(torch.randn(T, H + 2 * kv, hd, generator=g).to(bf16))
        for t, v in zip((d, q, p, u, pick), drafts(B, K, V, 50 + i)):
            t.copy_(v)
    load(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        body()
    torch.cuda.current_stream().wait_stream(side)
    graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = body()
    with torch.cuda.graph(other):
        res2 = body()
    for i in (1, 0, 2, 3, 1):
        load(i)
        graph.replay()
        first = [t.clone() for t in res]
        other.replay()
        torch.cuda.synchronize()
        load(i)
        ref = body()
        for a, b, c in zip(first, ref, res2):
            assert torch.equal(a, b) and torch.equal(c, b), i


def test_serving_on_another_stream(dev):
    """Calls on a stream of their own, beside the same calls on the current one."""
    from grove_amd import ops
    c, q, cu, kv_len, out = check_attn(dev, [6000, 90], [2, 1], 8, 2, 128, 64, seed=61)
    d, qq, p, u, pick = (t.to(dev) for t in drafts(4, 3, 5000, 6))
    ref = ops.verify_drafts(d, qq, p, u, pick)
    x = q.to(dev)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):
        with torch.cuda.stream(side):
            a = ops.kv4_attn(x, c.cache, c.table, kv_len, cu, 2, 128 ** -0.5, max_len=6000)
            va = ops.verify_drafts(d, qq, p, u, pick)
        b = ops.kv4_attn(x, c.cache, c.table, kv_len, cu, 2, 128 ** -0.5, max_len=6000)
        vb = ops.verify_drafts(d, qq, p, u, pick)
        torch.cuda.synchronize()
        assert torch.equal(a, out) and torch.equal(b, out)
        assert all(torch.equal(s, r) and torch.equal(t, r) for s, t, r in zip(va, vb, ref))


# ----------------------------------------------------------------------------- the decoder stack over the paged cache
@pytest.mark.parametrize("stream", [f32, bf16])
def test_decoder_stack_over_pages(dev, stream):
    """LlamaStack.paged_step: a prompt in one step, another in two pieces, then drafts, against the same stack with fp64 attention over the values
    that the cache stands for. The two differ by bf16 roundings: some eight of a layer's values, 2^-9 of each at most in the root mean square, in two
    layers, so 2^-9 sqrt(16) = 2^-7 of the hidden rows, doubled for what the norms and the residual sums pass on."""
    from grove_amd import ops
    from grove_amd.model.llama import LlamaStack
    from grove_amd.synthetic import TINY, synthetic_state_dict
    d = TINY
    sd = {k: v.to(dev).to(bf16) for k, v in synthetic_state_dict(d).items() if k.startswith(("model.layers", "model.norm"))}
    stack = LlamaStack(sd, d, dev, fp32_stream=stream == f32)
    nh, hd, H, P = d.n_heads, d.head_dim, d.hidden, 16
    cache = stack.new_kv4_cache(12, P)
    table = torch.full((2, 5), -1, dtype=i32, device=dev)
    free = torch.randperm(12, generator=gen(1)).to(i32).to(dev)
    ctx, held = torch.zeros(2, dtype=i32, device=dev), torch.zeros(2, dtype=i32, device=dev)
    plan = ops.rotary_plan(hd, d.rope_theta, device=dev)

    def by_hand(x, step, new):
        """The same with torch in fp64 between the matrix products; the cache holds this step's rows already."""
        w = lambda t: t.double().cpu()  # noqa: E731
        norm = lambda t, g: t * torch.rsqrt((t * t).mean(-1, keepdim=True) + d.rms_eps) * w(g)  # noqa: E731
        x, pos = w(x), step.pos.cpu()
        for L, kv in zip(stack.layers, cache):
            qkv = (norm(x, L["ln1"]) @ w(L["wqkv"]).T).view(-1, 3 * nh, hd)
            q = rotary_ref(qkv[:, :nh], pos, plan.freq.cpu(), False, 1.0)[0]
            o, at = [], 0
            for b, n in enumerate(new):
                L_ = int(step.kv_len[b])
                idx = torch.arange(L_, device=dev)
                k, v = (t.cpu().double() for t in ops.kv4_read(kv, (table[b, idx // P] * P + idx % P).to(i32), f32))
                z = torch.einsum("nhd,lhd->hnl", q[at:at + n], k) * hd ** -0.5
                z = z.masked_fill(torch.arange(L_)[None] >= torch.arange(L_ - n + 1, L_ + 1)[:, None], -math.inf)
                o.append(torch.einsum("hnl,lhd->nhd", torch.softmax(z, -1), v).flatten(1))
                at += n
            x = x + torch.cat(o) @ w(L["wo"]).T
            g, u = (norm(x, L["ln2"]) @ w(L["wgu"]).T).split(d.mlp, -1)
            x = x + (torch.nn.functional.silu(g) * u) @ w(L["wd"]).T
        return norm(x, stack.norm)

    for i, new in enumerate([[29, 10], [0, 21], [4, 4], [1, 1]]):
        T = sum(new)
        step = ops.page_tables(ctx, torch.tensor(new, dtype=i32, device=dev), table, held, free, P, T)
        free, held = free[int(step.taken):], step.held
        x = (torch.randn(T, H, generator=gen(20 + i)) * 0.5).to(bf16).to(dev)
        out = stack.paged_step(x, step, table, cache, max(new)).double().cpu()
        ref = by_hand(x, step, new)
        err = ((out - ref).pow(2).mean() / ref.pow(2).mean()).sqrt().item()
        assert err <= 2.0 ** -6, (i, err)
        ctx = step.kv_len.clone()
        if i == 2:
            ctx = ctx - 2  # two drafts of each refused: their rows are written again

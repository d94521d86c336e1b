"""Calls of the serving operators beside those of test_serving_gpu.py, whose references and tolerances they use."""
import math

import pytest
import torch

from test_serving_gpu import HALF, Paged, check_attn, check_verify, drafts, gen, verify_ref, within  # noqa: F401

pytestmark = pytest.mark.gpu

bf16, f32, f64, i32 = torch.bfloat16, torch.float32, torch.float64, torch.int32


# ----------------------------------------------------------------------------- tables
@pytest.mark.parametrize("max_len", [1, 100000])
def test_attn_shared_table_row(dev, max_len):
    """Requests that share one page list: an expanded row, and rows that overlap, against the same rows laid out."""
    from grove_amd import ops
    c = Paged(dev, [200], 2, 64, 16, seed=11)
    q = torch.randn(7, 4, 64, generator=gen(12)).to(bf16).to(dev)
    cu, kv_len = torch.tensor([0, 2, 3, 7], dtype=i32, device=dev), torch.tensor([200, 64, 131], dtype=i32, device=dev)
    wide = torch.cat([c.table[0], c.table[0, :4]])
    for table in (c.table.expand(3, -1), wide.as_strided((3, c.table.shape[1]), (2, 1))):
        a, b = (ops.kv4_attn(q, c.cache, t, kv_len, cu, 4, 0.125, max_len=max_len) for t in (table, table.contiguous()))
        assert torch.equal(a, b) and a.isfinite().all() and not (a == 0).all(1).any()


# ----------------------------------------------------------------------------- what rows may hold
SHAPES = [(4, 4, 1, 32), (4, 2, 4, 64), (2, 2, 1, 128), (8, 1, 4, 128), (16, 1, 4, 128), (4, 4, 1, 256), (8, 1, 4, 256), (16, 1, 4, 64)]  # every form of the kernel
POISON = [0x7f00, 0xff00, 0x7d80, 0x7f7f, 0xfd81, 0x7f80, 0x7fc0, 0x8001]  # scales and minima: finite ones from 2^124, infinity, NaN, a denormal


def poisoned(c, bits_s, bits_m):
    """Every cache row of `c` that no request owns holds (bits_s, bits_m) as its scale and minimum."""
    word = torch.tensor([bits_s, bits_m], dtype=i32).to(torch.int16).to(c.dev)
    flat = c.cache.scales.view(torch.int16)
    keep = torch.zeros(flat.shape[0] * c.P, dtype=torch.bool, device=c.dev)
    keep[c.slots.long()] = True
    keep = keep.view(-1, 1, 1, c.P, 1).expand_as(flat)
    flat.copy_(torch.where(keep, flat, word.expand_as(flat)))


@pytest.mark.parametrize("max_len", [1, 100000])
@pytest.mark.parametrize("H,kv,new,hd", SHAPES)
def test_attn_unseen_rows_hold_any_bits(dev, H, kv, new, hd, max_len):
    """Rows behind the lengths and those of other pages (page 0 stands in for a page outside the cache), whatever finite or other numbers they hold."""
    from grove_amd import ops
    lens, P, alpha = [45, 83, 16 + new], 16, hd ** -0.5
    c, q, cu, kv_len, _ = check_attn(dev, lens, [new] * 3, H, kv, hd, P, seed=hd + H, max_len=max_len)
    table = c.table.clone()
    table[1, 1] = -1  # its keys drop out
    qd = q.to(dev)
    first = [ops.kv4_attn(qd, c.cache, t, kv_len, cu, new, alpha, max_len=max_len) for t in (c.table, table)]
    assert first[0].isfinite().all() and first[1].isfinite().all()
    for s in POISON:
        for m in (POISON[0], POISON[1], 0x3f80):
            poisoned(c, s, m)
            for t, ref in zip((c.table, table), first):
                assert torch.equal(ops.kv4_attn(qd, c.cache, t, kv_len, cu, new, alpha, max_len=max_len), ref), (hex(s), hex(m))


@pytest.mark.parametrize("H,kv,new,hd", [s for s in SHAPES if s[2] > 1])
def test_attn_a_huge_row_stays_with_those_who_see_it(dev, H, kv, new, hd):
    """The last token's value row with a range just below the end of fp32 (scale 2^124): the last query of the request is no number or infinite, the
    others and the other request as they were."""
    from grove_amd import ops
    lens, P, alpha = [45, 80], 16, hd ** -0.5
    c, q, cu, kv_len, out = check_attn(dev, lens, [new] * 2, H, kv, hd, P, seed=hd + H + 3)
    k, v = (torch.zeros(1, kv, hd) for _ in range(2))
    v[0, 0, 1], v[0, 0, 2] = 1.65e38, -1.65e38
    ops.kv4_append(k.to(bf16).to(dev), v.to(bf16).to(dev), c.cache, c.slots[44:45])
    assert ops.kv4_read(c.cache, c.slots[44:45], f32)[1].isfinite().all()
    r = ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, new, alpha)
    keep = torch.ones(2 * new, dtype=torch.bool)
    keep[new - 1] = False
    assert torch.equal(r[keep], out[keep]) and not r[new - 1].view(H, hd)[:H // kv].isfinite().any()


@pytest.mark.parametrize("max_len", [1, 100000])
@pytest.mark.parametrize("H,kv,new,hd", SHAPES)
def test_attn_values_to_two_to_the_64(dev, H, kv, new, hd, max_len):
    """The largest values that are promised: powers of two pass through every sum exactly, keys' and queries' against each other too, also where the
    weights are as large as they get (scores that climb by 23 in units of log2 behind a wave's first keys)."""
    from grove_amd import ops
    L, P = 1500, 32
    c = Paged(dev, [L, 40], kv, hd, P, seed=7)
    g = gen(8)
    q = (1.0 + 0.1 * torch.randn(2 * new, H, hd, generator=g)).to(bf16)
    k = torch.where(torch.arange(L) < 128, 0.0, 15.0)[:, None, None] / hd * (1 + 0.05 * torch.rand(L, kv, hd, generator=g))
    v = torch.randn(L, kv, hd, generator=g).clamp(-1, 1)
    cu = torch.tensor([0, new, 2 * new], dtype=i32, device=dev)
    kv_len = torch.tensor([L, 40], dtype=i32, device=dev)
    res = []
    for ks, vs in ((1.0, 1.0), (2.0 ** 40, 2.0 ** 64), (2.0 ** -40, 2.0 ** -60)):
        ops.kv4_append((k * ks).to(bf16).to(dev), (v * vs).to(bf16).to(dev), c.cache, c.slots[:L])
        o = ops.kv4_attn((q / ks).to(bf16).to(dev), c.cache, c.table, kv_len, cu, new, 1.0, max_len=max_len)
        res.append(o[:new].double() / vs)
    assert res[0].isfinite().all() and torch.equal(res[0], res[1]) and torch.equal(res[0], res[2])


# ----------------------------------------------------------------------------- fewer rows than cu_q says
@pytest.mark.parametrize("max_len", [1, 100000])
@pytest.mark.parametrize("H,kv,new,hd", [s for s in SHAPES if s[2] > 1])
def test_attn_rows_cut_short(dev, H, kv, new, hd, max_len):
    """A step of fixed size that the last request's tokens pass (page_tables writes the rows that there are): those that are there keep their limits."""
    from grove_amd import ops
    lens = [20, 70, 9]
    c, q, cu, kv_len, out = check_attn(dev, lens, [new, new, new], H, kv, hd, 16, seed=hd + 5, max_len=max_len)
    qd = q.to(dev)
    for rows in (2 * new, 2 * new - 1, new + 1, 1):
        r = ops.kv4_attn(qd[:rows], c.cache, c.table, kv_len, cu, new, hd ** -0.5, max_len=max_len)
        assert torch.equal(r, out[:rows]), rows


# ----------------------------------------------------------------------------- where q lies
@pytest.mark.parametrize("rows", [1, 2, 5])
@pytest.mark.parametrize("start", [0, 1, 4, 8])
def test_attn_q_at_any_start(dev, rows, start):
    """One row or several, contiguous or columns of a wider activation, at any start; and an output row with an odd stride."""
    from grove_amd import ops
    H, kv, hd = 4, 2, 64
    c, q, cu, kv_len, ref = check_attn(dev, [70], [rows], H, kv, hd, 16, seed=rows)
    flat = torch.full((start + rows * H * hd,), math.nan, dtype=bf16, device=dev)
    flat[start:] = q.to(dev).flatten()
    wide = torch.full((rows, H * hd + 3 + start), math.nan, dtype=bf16, device=dev)
    wide[:, start:start + H * hd] = q.to(dev).flatten(1)
    odd = wide[:, start:].as_strided((rows, H, hd), (wide.stride(0), hd, 1), start)
    for x in (flat[start:].view(rows, H, hd), wide[:, start:start + H * hd].unflatten(1, (H, hd)), odd):
        assert torch.equal(ops.kv4_attn(x, c.cache, c.table, kv_len, cu, rows, hd ** -0.5), ref)
    if rows == 1:
        out = torch.full((1, H * hd + 3), 5.0, dtype=bf16, device=dev)
        ops.kv4_attn(q.to(dev), c.cache, c.table, kv_len, cu, 1, hd ** -0.5, out=out[:, :H * hd])
        assert torch.equal(out[:, :H * hd], ref) and (out[:, H * hd:] == 5).all()


# ----------------------------------------------------------------------------- the decoder stack, captured
@pytest.mark.parametrize("stream", [f32, bf16])
def test_paged_step_captured(dev, stream):
    """Tables and the decoder stack in one captured step with rows of padding, the stack's own plan used there first: replayed over several steps,
    with eager work between, against the eager step on a cache of its own."""
    from grove_amd import ops
    from grove_amd.model.llama import LlamaStack
    from grove_amd.synthetic import TINY, synthetic_state_dict
    d, P, T, B = TINY, 16, 9, 3
    sd = {k: v.to(dev).to(bf16) for k, v in synthetic_state_dict(d).items() if k.startswith(("model.layers", "model.norm"))}
    stack = LlamaStack(sd, d, dev, fp32_stream=stream == f32)
    caches = [stack.new_kv4_cache(20, P) for _ in range(2)]
    free = torch.randperm(20, generator=gen(1)).to(i32).to(dev)
    state = [dict(table=torch.full((B, 5), -1, dtype=i32, device=dev), held=torch.zeros(B, dtype=i32, device=dev), free=free.clone()) for _ in range(2)]
    x, ctx, new = torch.zeros(T, d.hidden, dtype=bf16, device=dev), torch.zeros(B, dtype=i32, device=dev), torch.zeros(B, dtype=i32, device=dev)

    def body(i, plan=None):
        s = state[i]
        step = ops.page_tables(ctx, new, s["table"], s["held"], s["free"], P, T)
        return step, stack.paged_step(x.clone(), step, s["table"], caches[i], 4, plan=plan)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # (nothing to be written: no request has a token; another plan, so that the stack's own is first used in the graph)
        body(0, ops.rotary_plan(d.head_dim, device=dev))
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        res = body(0)
    have = [0] * B
    for i, n in enumerate([[4, 4, 1], [4, 0, 3], [1, 1, 1], [2, 3, 4], [1, 4, 4], [0, 1, 0]]):
        x.copy_((torch.randn(T, d.hidden, generator=gen(30 + i)) * 0.5).to(bf16))
        ctx.copy_(torch.tensor(have, dtype=i32))
        new.copy_(torch.tensor(n, dtype=i32))
        graph.replay()
        got = [t.clone() for t in (*res[0], res[1])]
        ref = body(1)
        torch.cuda.synchronize()
        for a, b in zip(got[:-1], ref[0]):
            assert torch.equal(a, b), i
        assert torch.equal(got[-1], ref[1]) and got[-1][:sum(n)].isfinite().all(), i
        for s, step in zip(state, (res[0], ref[0])):
            taken = int(step.taken)
            s["free"].copy_(torch.roll(s["free"], -taken))
            s["held"].copy_(step.held)
        have = [a + b for a, b in zip(have, n)]


# ----------------------------------------------------------------------------- verification, one launch and two
@pytest.mark.parametrize("dtype", [f32, bf16])
@pytest.mark.parametrize("V", [50, 9001, 32008, 1100003])  # one block, several per request, chunks of more than 1024
def test_verify_edges_at_every_vocabulary(dev, dtype, V):
    B, K = 5, 3
    d, q, p, u, pick = drafts(B, K, V, V, dtype)
    bad = d.clone()
    bad[0, 0], bad[1, 1], bad[2, 2], bad[4, 0] = -1, V, 2 ** 31 - 1, V + 7       # tokens that do not exist: refused
    same = p[:, :K].clone()
    t = check_verify(dev, bad, same, p, u, pick)                                # ... where p - q leaves nothing: drawn from p itself
    assert (t[:3] >= -1).all() and (t[[0, 4], 0] >= 0).all() and (t[1, 1] >= 0) and (t[2, 2] >= 0)
    less = same.clone()
    less[4, 0, V // 3] = 0                                                      # ... and where it leaves one token
    assert check_verify(dev, bad, less, p, u, pick)[4, 0] == V // 3
    check_verify(dev, bad, q, p, u, pick)
    check_verify(dev, bad, None, p, u, pick)
    for a in (0.0, 1 - 2.0 ** -24):
        for b in (0.0, 1 - 2.0 ** -24):
            check_verify(dev, bad, q, p, torch.full_like(u, a), torch.full_like(pick, b))
    zero = p.clone()
    zero[1], zero[2, 1:] = 0, 0
    t = check_verify(dev, bad, q, zero, u, pick)                                # no mass at all: no token
    assert t[1, 0] == -1
    one = torch.zeros_like(p)
    one[..., V - 1] = 1
    assert (check_verify(dev, bad, None, one, u, pick)[:, 0] == V - 1).all()     # certain of the last token


# ----------------------------------------------------------------------------- the loop around a step
def test_serving_loop_keeps_every_context(dev):
    """Prompts in pieces, next tokens and drafts in the same steps, lengths carried on as ctx = kv_len - (count - accepted): after every step the
    cache holds exactly the rows of each request's accepted tokens, at their positions, and the step's attention saw them."""
    from grove_amd import ops
    B, H, kv, hd, P, K, V = 4, 4, 2, 64, 16, 3, 40
    g = gen(91)
    emb = torch.randn(V, H + 2 * kv, hd, generator=g).to(bf16).to(dev)
    plan = ops.rotary_plan(hd, device=dev)
    cache = ops.kv4_cache(60, P, kv, hd, dev)
    free, table = torch.randperm(60, generator=g).to(i32).to(dev), torch.full((B, 14), -1, dtype=i32, device=dev)
    ctx, held = torch.zeros(B, dtype=i32, device=dev), torch.zeros(B, dtype=i32, device=dev)
    prompts = [torch.randint(0, V, (n,), generator=g).tolist() for n in (37, 1, 50, 5)]
    seqs, todo = [[] for _ in range(B)], [[p[:20], p[20:]] if len(p) > 20 else [p] for p in prompts]
    nxt = [None] * B
    for it in range(9):
        new, count, draft = [], [], torch.zeros(B, K, dtype=i32)
        for b in range(B):
            if todo[b] and it >= b:  # (the requests come one after the other)
                new.append(todo[b].pop(0))
                count.append(0)
            elif nxt[b] is None:
                new.append([])
                count.append(0)
            else:
                n = (it + b) % (K + 1)
                draft[b, :n] = torch.randint(0, V, (n,), generator=g).to(i32)
                new.append([nxt[b]] + draft[b, :n].tolist())
                count.append(n)
        T = sum(len(t) for t in new)
        ids = torch.tensor(sum(new, []), device=dev)
        cnt = torch.tensor(count, dtype=i32, device=dev)
        step = ops.page_tables(ctx, torch.tensor([len(t) for t in new], dtype=i32, device=dev), table, held, free, P, T)
        free, held = free[int(step.taken):], step.held
        x = emb[ids]
        ops.rotary(x[:, :H + kv], step.pos, plan, out=x[:, :H + kv])
        ops.kv4_append(x[:, H:H + kv], x[:, H + kv:], cache, step.slots)
        out = ops.kv4_attn(x[:, :H], cache, table, step.kv_len, step.cu_q, max(len(t) for t in new), hd ** -0.5)
        rows = (step.cu_q[1:] - 1 - cnt)[:, None] + torch.arange(K + 1, device=dev)
        z = torch.randn(T, V, generator=g).to(dev)
        z[:, :12] += 2
        p = torch.softmax(z, -1)[rows.clamp(0, T - 1)]
        u, pick = torch.rand(B, K, generator=g).to(dev) * 0.05, torch.rand(B, generator=g).to(dev)
        tokens, accepted = ops.verify_drafts(draft.to(dev), None, p, u, pick, cnt)
        ctx = step.kv_len - (cnt - accepted)
        ref = verify_ref(draft, None, p.cpu(), u.cpu(), pick.cpu(), cnt.cpu())
        assert torch.equal(tokens.cpu(), ref[0]) and torch.equal(accepted.cpu(), ref[1])
        want, whole = [], ops.kv4_cache(B * 14, P, kv, hd, dev)
        for b in range(B):
            full = seqs[b] + new[b]
            a = int(accepted[b])
            if new[b]:
                seqs[b] = seqs[b] + new[b][:len(new[b]) - count[b] + a]
                nxt[b] = int(tokens[b, a]) if not todo[b] else None
            assert int(ctx[b]) == len(seqs[b]), (it, b)
            want.append(full)
        # the same contexts written at once into a cache of their own, pages in order
        own = torch.arange(B * 14, dtype=i32, device=dev).view(B, 14)
        for b, full in enumerate(want):
            if full:
                y, pos = emb[torch.tensor(full, device=dev)], torch.arange(len(full), dtype=i32, device=dev)
                ops.rotary(y[:, :H + kv], pos, plan, out=y[:, :H + kv])
                ops.kv4_append(y[:, H:H + kv], y[:, H + kv:], whole, b * 14 * P + pos)
        assert torch.equal(out, ops.kv4_attn(x[:, :H], whole, own, step.kv_len, step.cu_q, max(len(t) for t in new), hd ** -0.5)), it
        for b in range(B):
            t = torch.arange(len(seqs[b]), device=dev)
            at = (table[b, t // P] * P + t % P).to(i32)
            for s, w in zip(ops.kv4_read(cache, at, f32), ops.kv4_read(whole, (b * 14 * P + t).to(i32), f32)):
                assert torch.equal(s, w), (it, b)
    assert sum(len(s) for s in seqs) > 100 and any(len(s) > len(p) + 4 for s, p in zip(seqs, prompts))


# ----------------------------------------------------------------------------- queries that are no numbers
@pytest.mark.parametrize("max_len", [1, 100000])
@pytest.mark.parametrize("H,kv,new,hd", SHAPES)
def test_attn_a_query_that_is_no_number(dev, H, kv, new, hd, max_len):
    """NaN, infinities and values at the end of bf16 in one query head's row: the other rows and heads keep their bits."""
    from grove_amd import ops
    lens = [300, 80, 40]
    c, q, cu, kv_len, ref = check_attn(dev, lens, [new] * 3, H, kv, hd, 16, seed=hd + H + 9, max_len=max_len)
    keep = torch.ones(3 * new, H, dtype=torch.bool)
    keep[new, H - 1] = False
    for bad in (math.nan, math.inf, -math.inf, 3e38):
        x = q.clone()
        x[new, H - 1, 5] = bad
        r = ops.kv4_attn(x.to(dev), c.cache, c.table, kv_len, cu, new, hd ** -0.5, max_len=max_len)
        assert torch.equal(r.view(3 * new, H, hd)[keep], ref.view(3 * new, H, hd)[keep]), bad
        if bad != 3e38:
            assert r.view(3 * new, H, hd)[new, H - 1].isnan().all(), bad

"""Cases for the operators of serving from a paged 4-bit key / value cache with drafted tokens.

Five operators, in the order in which one serving step calls them:

  rotary   rotary positions of q and k: half or interleaved pairs, a part of the head, stretched for long contexts; and the gradient
  pages    block tables, slot map and positions of a step from the requests' lengths
  store    keys and values into the 4-bit pages of their slots, and back
  attn     attention of one to a few new tokens per request over the 4-bit pages
  verify   drafted tokens against the target's probabilities, from given random numbers

`own = False`: `run` computes them in elementary torch operations; `own = True`: with grove_amd.ops.

The 4-bit cache.  A row (one token, one key / value head, hd channels) is held as hd codes c in 0..15, a scale s and a minimum m, both bf16:
  m = min(row),  s = bf16((max(row) - min(row)) / 15),  c = clamp(rint((x - m) / s), 0, 15),  and stands for m + c s.
`codes` is uint8 [pages, 2, heads, page * hd / 2] (keys, values), `scales` bf16 [pages, 2, heads, page, 2] (scale, minimum). The order of the
codes within a page is the one that the matrix instructions read (pack_keys / pack_values).
"""
import math

import torch

own = False

DEV = "cuda"
bf16 = torch.bfloat16


# ------------------------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of the clip-batched captioning: 8 sequences, 32 query and 32 key heads of 128, positions of a 703-token prompt
        dict(name="rotary_step", op="rotary", rows=8, heads=64, hd=128, rot=128, pairs="half", scaling="none", factor=1.0, dtype="bf16", far=768,
             backward=False),
        # a long prompt, grouped heads (32 + 8), half of the head rotated, interleaved pairs, a context stretched 8 times
        dict(name="rotary_prompt", op="rotary", rows=16384, heads=40, hd=128, rot=64, pairs="interleaved", scaling="yarn", factor=8.0, dtype="bf16",
             far=131072, backward=False),
        # the gradient in fp32, a head of 80, an odd number of rows, positions divided by 4
        dict(name="rotary_grad", op="rotary", rows=4099, heads=32, hd=80, rot=80, pairs="half", scaling="linear", factor=4.0, dtype="f32",
             far=16384, backward=True),
        # page bookkeeping of one decode step of 8 sequences
        dict(name="pages_step", op="pages", requests=8, page=16, longest=768, drafts=0, prompts=0, prompt=0),
        # a server's step: 512 requests with drafts, 16 of them with a fresh piece of prompt
        dict(name="pages_mixed", op="pages", requests=512, page=64, longest=32768, drafts=4, prompts=16, prompt=2048),
        # the rows of one step of 8 requests with 4 drafts each, all 32 heads
        dict(name="store_step", op="store", rows=40, kv=32, hd=128, page=64),
        # a long prompt's rows, 8 heads
        dict(name="store_prompt", op="store", rows=16387, kv=8, hd=128, page=32),
        # one caption's next token: 32 heads, 703 tokens in the cache
        dict(name="attn_caption", op="attn", requests=1, heads=32, kv=32, hd=128, page=64, longest=703, even=True, queries=1),
        # 8 requests of ragged lengths, 4 drafts and the token before them, grouped heads, small pages
        dict(name="attn_drafts", op="attn", requests=8, heads=32, kv=8, hd=128, page=16, longest=4099, even=False, queries=5),
        # 32 long ragged contexts, one token each
        dict(name="attn_long", op="attn", requests=32, heads=32, kv=8, hd=128, page=128, longest=32768, even=False, queries=1),
        # 8 requests with 4 drafts each over the vocabulary of 32008
        dict(name="verify_step", op="verify", requests=8, drafts=4, vocab=32008, dtype="f32"),
        # 128 requests with up to 7 drafts over a wide vocabulary
        dict(name="verify_wide", op="verify", requests=128, drafts=7, vocab=128000, dtype="f32"),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.999)))))))


def draw(rng):
    op = rng.choice(["rotary", "pages", "store", "attn", "attn", "verify"])
    if op == "rotary":
        hd = rng.choice([32, 64, 80, 96, 128, 256])
        scaling = rng.choice(["none", "linear", "ntk", "yarn"])
        heads = _log(rng, 1, 64)
        return dict(op=op, rows=_log(rng, 1, max(1, min(16384, 40 * 128 * 16384 // (heads * hd)))), heads=heads, hd=hd,
                    rot=hd // rng.choice([1, 1, 2]), pairs=rng.choice(["half", "interleaved"]), scaling=scaling,
                    factor=1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0, 16.0]), dtype=rng.choice(["bf16", "bf16", "f32"]),
                    far=_log(rng, 1000, 131072), backward=rng.random() < 0.4)
    if op == "pages":
        requests = _log(rng, 1, 512)
        return dict(op=op, requests=requests, page=rng.choice([16, 32, 64, 128]), longest=_log(rng, 100, 32768), drafts=rng.randint(0, 7),
                    prompts=rng.randint(0, min(requests, 16)), prompt=_log(rng, 10, 2048))
    if op == "store":
        kv = rng.choice([1, 2, 4, 8, 32])
        return dict(op=op, rows=_log(rng, 1, 16384 * 8 // max(kv, 8)), kv=kv, hd=rng.choice([32, 64, 128, 128, 256]), page=rng.choice([16, 32, 64, 128]))
    if op == "attn":
        kv, group = rng.choice([(32, 1), (8, 4), (4, 8), (8, 8), (2, 7), (16, 1)])
        requests = _log(rng, 1, 64)
        hd = rng.choice([64, 128, 128, 256])
        most = 32 * 16384 * 8 * 128 // 2 // (requests * kv * hd)
        return dict(op=op, requests=requests, heads=kv * group, kv=kv, hd=hd, page=rng.choice([16, 32, 64, 128]),
                    longest=_log(rng, 30, max(30, min(65536, most))), even=rng.random() < 0.3, queries=rng.choice([1, 1, 2, 4, 5, 8]))
    return dict(op=op, requests=_log(rng, 1, 128), drafts=rng.randint(1, 7), vocab=_log(rng, 1000, 128000), dtype=rng.choice(["f32", "f32", "bf16"]))


def _dt(case):
    return torch.float32 if case["dtype"] == "f32" else bf16


def _lengths(case, seed):
    """Host lists of a `pages` or `attn` case: tokens already held and new tokens per request, made from the seed alone."""
    g = torch.Generator().manual_seed(seed * 7919 + 13)
    n = case["requests"]
    if case["op"] == "attn":
        new = [case["queries"]] * n
        if case["even"]:
            total = [max(case["longest"], case["queries"])] * n
        else:  # from a sixteenth of the longest up, one of them the longest
            lo = max(case["queries"], case["longest"] // 16)
            total = torch.randint(lo, max(lo, case["longest"]) + 1, (n,), generator=g).tolist()
            total[int(torch.randint(0, n, (1,), generator=g))] = max(lo, case["longest"])
        return [t - q for t, q in zip(total, new)], new
    ctx = torch.randint(1, case["longest"] + 1, (n,), generator=g).tolist()
    new = _new_tokens(case)
    return ctx, [new[i] for i in torch.randperm(n, generator=g).tolist()]


def _new_tokens(case):
    """New tokens of a `pages` step in some order: a piece of prompt for the first `prompts` requests, the drafts and one more for the others."""
    g = torch.Generator().manual_seed(5)
    pieces = (1 + torch.randint(0, max(1, case["prompt"]), (case["prompts"],), generator=g)).tolist()
    return pieces + [1 + case["drafts"]] * (case["requests"] - case["prompts"])


# ------------------------------------------------------------------------------------------------------------------ the page layout
def pack_keys(c):
    """codes [..., page, hd] -> uint8 [..., page * hd / 2]. A row is 4 pieces of hd / 32 words: word t of piece h holds the channels
    32 t + 8 h + (0, 2, 4, 6, 1, 3, 5, 7), lowest nibble first."""
    *b, P, hd = c.shape
    c = c.view(*b, P, hd // 32, 4, 8)[..., [0, 2, 4, 6, 1, 3, 5, 7]].transpose(-3, -2)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(*b, P * hd // 2)


def unpack_keys(u, hd):
    *b, n = u.shape
    P = n * 2 // hd
    u = u.view(*b, P, 4, hd // 32, 4)
    c = torch.stack([u & 15, u >> 4], -1).flatten(-2)[..., [0, 4, 1, 5, 2, 6, 3, 7]]
    return c.transpose(-3, -2).reshape(*b, P, hd)


def pack_values(c):
    """codes [..., page, hd] -> uint8 [..., page * hd / 2]. Four tokens together: for each m in 0..15 the channels 16 j + m of the four, four
    j at a time, the tokens in the order 0, 1, 2, 3 (a head of 32, with two j: in the order 0, 2, 1, 3), lowest nibble first."""
    *b, P, hd = c.shape
    if hd == 32:
        c = c.view(*b, P // 4, 4, 2, 16)[..., [0, 2, 1, 3], :, :]
        c = c.permute(*range(len(b)), -4, -1, -3, -2)
    else:
        c = c.view(*b, P // 4, 4, hd // 64, 4, 16).unflatten(-4, (2, 2))
        c = c.permute(*range(len(b)), -6, -1, -3, -5, -4, -2)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).reshape(*b, P * hd // 2)


def unpack_values(u, hd):
    *b, n = u.shape
    P = n * 2 // hd
    if hd == 32:
        c = torch.stack([u & 15, u >> 4], -1).view(*b, P // 4, 16, 4, 2)
        c = c.permute(*range(len(b)), -4, -2, -1, -3)[..., [0, 2, 1, 3], :, :]
    else:
        c = torch.stack([u & 15, u >> 4], -1).view(*b, P // 4, 16, hd // 64, 2, 2, 4)
        c = c.permute(*range(len(b)), -6, -3, -2, -4, -1, -5)
    return c.reshape(*b, P, hd)


def quantise(x):
    """bf16 rows [..., hd] -> codes uint8 [..., hd], scales bf16 [..., 2]."""
    x = x.float()
    lo, hi = x.amin(-1, keepdim=True), x.amax(-1, keepdim=True)
    s = ((hi.double() - lo.double()) / 15).to(bf16).float()
    c = torch.where(s > 0, torch.round((x - lo) / s), torch.zeros_like(x)).clamp(0, 15).to(torch.uint8)
    return c, torch.cat([s, lo], -1).to(bf16)


# ------------------------------------------------------------------------------------------------------------------ inputs
def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(seed * 1000003 + 17)


def _freq(case):
    """Radians per position of each pair (fp64, on the host), and the factor on the rotated values."""
    rot, theta, f = case["rot"], 10000.0, case["factor"]
    i = torch.arange(0, rot, 2, dtype=torch.float64) / rot
    if case["scaling"] == "ntk":
        theta *= f ** (rot / (rot - 2))
    w = theta ** -i
    if case["scaling"] == "linear":
        w = w / f
    if case["scaling"] == "yarn":
        dim = lambda turns: rot * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(theta))  # noqa: E731
        low, high = max(math.floor(dim(32.0)), 0), min(math.ceil(dim(1.0)), rot - 1)
        ramp = ((torch.arange(rot // 2, dtype=torch.float64) - low) / max(high - low, 0.001)).clamp(0, 1)
        w = w / f * ramp + w * (1 - ramp)
        return w, 0.1 * math.log(f) + 1.0
    return w, 1.0


def prepare(case, seed):
    g = _gen(seed)
    st = {"case": case}
    op = case["op"]
    if op == "rotary":
        st["x"] = torch.randn(case["rows"], case["heads"], case["hd"], device=DEV, generator=g).to(_dt(case))
        st["pos"] = torch.randint(0, case["far"], (case["rows"],), device=DEV, generator=g, dtype=torch.int32)
        w, st["mscale"] = _freq(case)
        st["freq"] = w.to(DEV)
    elif op == "pages":
        ctx, new = _lengths(case, seed)
        P = case["page"]
        most = -(-(case["longest"] + max(new)) // P) + 1
        held = [-(-c // P) for c in ctx]
        need = sum(max(0, -(-(c + n) // P) - h) for c, n, h in zip(ctx, new, held))
        pages = torch.randperm(sum(held) + need + 8, device=DEV, generator=g).to(torch.int32)
        table = torch.full((case["requests"], most), -1, dtype=torch.int32)
        at = 0
        host = pages.cpu()
        for b, h in enumerate(held):
            table[b, :h] = host[at:at + h]
            at += h
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        st.update(ctx=i32(ctx), new=i32(new), held=i32(held), table=table.to(DEV), free=pages[at:].clone(), tokens=sum(new))
    elif op == "store":
        R, kv, hd, P = case["rows"], case["kv"], case["hd"], case["page"]
        qkv = torch.randn(R, 2 * kv, hd, device=DEV, generator=g)
        qkv *= 0.5 + torch.rand(2 * kv, hd, device=DEV, generator=g) * 2  # channels of unequal width, as keys have them
        qkv = qkv.to(bf16)
        st["k"], st["v"] = qkv[:, :kv], qkv[:, kv:]
        n = -(-R // P) + 3
        pages = torch.randperm(n, device=DEV, generator=g)
        at = torch.arange(R, device=DEV) + P // 3  # the first page already holds some rows
        st["slots"] = (pages[at // P] * P + at % P).to(torch.int32)
        st["codes"] = torch.zeros(n, 2, kv, P * hd // 2, dtype=torch.uint8, device=DEV)
        st["scales"] = torch.zeros(n, 2, kv, P, 2, dtype=bf16, device=DEV)
    elif op == "attn":
        ctx, new = _lengths(case, seed)
        kv, hd, P = case["kv"], case["hd"], case["page"]
        held = [-(-(c + n) // P) for c, n in zip(ctx, new)]
        n = sum(held) + 3
        st["codes"] = torch.empty(n, 2, kv, P * hd // 2, dtype=torch.uint8, device=DEV)
        st["scales"] = torch.empty(n, 2, kv, P, 2, dtype=bf16, device=DEV)
        width = 0.5 + torch.rand(2, kv, 1, hd, device=DEV, generator=g)
        step = max(1, (1 << 27) // (2 * kv * P * hd))
        for lo in range(0, n, step):
            m = min(step, n - lo)
            c, s = quantise((torch.randn(m, 2, kv, P, hd, device=DEV, generator=g) * width).to(bf16))
            st["codes"][lo:lo + m, 0], st["codes"][lo:lo + m, 1] = pack_keys(c[:, 0]), pack_values(c[:, 1])
            st["scales"][lo:lo + m] = s
        pages = torch.randperm(n, device=DEV, generator=g).to(torch.int32)
        table = torch.full((case["requests"], max(held)), -1, dtype=torch.int64)
        at = 0
        for b, h in enumerate(held):
            table[b, :h] = torch.arange(at, at + h)
            at += h
        st["table"] = torch.where(table.to(DEV) < 0, -1, pages[table.to(DEV).clamp(min=0)]).to(torch.int32)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=DEV)  # noqa: E731
        st["kv_len"] = i32([c + q for c, q in zip(ctx, new)])
        st["cu_q"] = i32([0] + torch.tensor(new).cumsum(0).tolist())
        st["longest"] = max(c + q for c, q in zip(ctx, new))
        st["q"] = (torch.randn(sum(new), case["heads"], hd, device=DEV, generator=g) * 1.5).to(bf16)
        st["alpha"] = hd ** -0.5
    else:
        B, K, V = case["requests"], case["drafts"], case["vocab"]
        logits = torch.randn(B, K + 1, V, device=DEV, generator=g) * 3
        st["p"] = torch.softmax(logits, -1).to(_dt(case))
        logits = logits[:, :K] + torch.randn(B, K, V, device=DEV, generator=g) * 0.4  # a drafter that is right most of the time
        q = torch.softmax(logits, -1)
        st["q"] = q.to(_dt(case))
        cdf = q.flatten(0, 1).double().cumsum(-1)
        u = torch.rand(B * K, 1, device=DEV, generator=g, dtype=torch.float64) * cdf[:, -1:]
        st["draft"] = torch.searchsorted(cdf, u, right=True).clamp(max=V - 1).view(B, K).to(torch.int32)
        del cdf, logits, q
        st["count"] = torch.randint(max(0, K - 2), K + 1, (B,), device=DEV, generator=g, dtype=torch.int32)
        st["u"] = torch.rand(B, K, device=DEV, generator=g)
        st["pick"] = torch.rand(B, device=DEV, generator=g)
    return st


# ------------------------------------------------------------------------------------------------------------------ one pass
def run(st):
    return (_run_own if own else _run_plain)(st)


def _run_own(st):
    from grove_amd import ops
    case = st["case"]
    op = case["op"]
    if op == "rotary":
        plan = ops.RotaryPlan(st["freq"], case["pairs"] == "interleaved", st["mscale"])
        return ops.rotary(st["x"], st["pos"], plan, backward=case["backward"])
    if op == "pages":
        step = ops.page_tables(st["ctx"], st["new"], st["table"], st["held"], st["free"], case["page"], st["tokens"])
        return [st["table"], step.kv_len, step.cu_q, step.slots, step.pos, step.held, step.taken]
    cache = ops.KV4Cache(st["codes"], st["scales"]) if op in ("store", "attn") else None
    if op == "store":
        ops.kv4_append(st["k"], st["v"], cache, st["slots"])
        return list(ops.kv4_read(cache, st["slots"]))
    if op == "attn":
        return ops.kv4_attn(st["q"], cache, st["table"], st["kv_len"], st["cu_q"], case["queries"], st["alpha"], max_len=st["longest"])
    return list(ops.verify_drafts(st["draft"], st["q"], st["p"], st["u"], st["pick"], count=st["count"]))


def _run_plain(st):
    return {"rotary": _plain_rotary, "pages": _plain_pages, "store": _plain_store, "attn": _plain_attn, "verify": _plain_verify}[st["case"]["op"]](st)


def _plain_rotary(st):
    case, x = st["case"], st["x"]
    rot = case["rot"]
    a = st["pos"].double()[:, None] * st["freq"]
    sign = -1.0 if case["backward"] else 1.0
    cos, sin = ((torch.cos(a) * st["mscale"]).float()[:, None], (torch.sin(a) * (st["mscale"] * sign)).float()[:, None])
    y = x.float()
    if case["pairs"] == "interleaved":
        e, o = y[..., 0:rot:2], y[..., 1:rot:2]
        r = torch.stack([e * cos - o * sin, o * cos + e * sin], -1).flatten(-2)
    else:
        e, o = y[..., :rot // 2], y[..., rot // 2:rot]
        r = torch.cat([e * cos - o * sin, o * cos + e * sin], -1)
    return torch.cat([r, y[..., rot:]], -1).to(x.dtype)


def _plain_pages(st):
    P, ctx, new, held, table, free, T = st["case"]["page"], st["ctx"].long(), st["new"].long(), st["held"].long(), st["table"], st["free"], st["tokens"]
    B, most = table.shape
    total = ctx + new
    need = ((total + P - 1) // P - held).clamp(min=0)
    start = need.cumsum(0) - need
    j = torch.arange(most, device=table.device)[None]
    i = j - held[:, None]
    fresh = (i >= 0) & (i < need[:, None])
    at = start[:, None] + i
    page = torch.where(at < free.numel(), free[at.clamp(0, free.numel() - 1)], -1)
    table.copy_(torch.where(fresh, page, table))
    cu = torch.cat([torch.zeros_like(total[:1]), new.cumsum(0)])
    t = torch.arange(T, device=table.device)
    b = (torch.searchsorted(cu, t, right=True) - 1).clamp(0, B - 1)
    pos = ctx[b] + t - cu[b]
    pg = table[b, (pos // P).clamp(max=most - 1)].long()
    slots = torch.where((pg >= 0) & (pos // P < most), pg * P + pos % P, -1)
    i32 = torch.int32
    return [table, total.to(i32), cu.to(i32), slots.to(i32), pos.to(i32), (held + need).to(i32), need.sum().view(1).to(i32)]


def _plain_store(st):
    hd, P, kv = st["case"]["hd"], st["case"]["page"], st["case"]["kv"]
    codes, scales, slots = st["codes"], st["scales"], st["slots"].long()
    n = codes.shape[0]
    every = torch.stack([unpack_keys(codes[:, 0], hd), unpack_values(codes[:, 1], hd)], 1)
    pg, at = slots // P, slots % P
    for i, x in enumerate((st["k"], st["v"])):
        c, s = quantise(x)
        every[:, i].transpose(1, 2)[pg, at] = c
        scales[:, i].transpose(1, 2)[pg, at] = s
    codes[:, 0], codes[:, 1] = pack_keys(every[:, 0]), pack_values(every[:, 1])
    out = []
    for i, u in enumerate((unpack_keys(codes[:, 0], hd), unpack_values(codes[:, 1], hd))):
        c, s = u.transpose(1, 2)[pg, at].float(), scales[:, i].transpose(1, 2)[pg, at].float()
        out.append((s[..., 1:] + c * s[..., :1]).to(bf16))
    return out


def _plain_attn(st):
    case, q, cu = st["case"], st["q"], st["cu_q"].long()
    H, kv, hd, P, n = case["heads"], case["kv"], case["hd"], case["page"], case["queries"]
    B = case["requests"]
    pages = st["table"].clamp(min=0).long()
    L = pages.shape[1] * P
    s = st["scales"][pages].float().permute(2, 0, 3, 1, 4, 5).reshape(2, B, kv, L, 2)
    c = st["codes"][pages]
    k = unpack_keys(c[:, :, 0], hd).transpose(1, 2).reshape(B, kv, L, hd).float().mul_(s[0, ..., :1]).add_(s[0, ..., 1:])
    v = unpack_values(c[:, :, 1], hd).transpose(1, 2).reshape(B, kv, L, hd).float().mul_(s[1, ..., :1]).add_(s[1, ..., 1:])
    i = torch.arange(n, device=q.device)
    rows = (cu[:-1, None] + i).clamp(max=q.shape[0] - 1)
    new = cu[1:] - cu[:-1]
    x = q[rows].float().view(B, n, kv, H // kv, hd).permute(0, 2, 3, 1, 4).reshape(B * kv, (H // kv) * n, hd)
    z = torch.bmm(x, k.view(B * kv, L, hd).transpose(1, 2)).view(B, kv, H // kv, n, L) * st["alpha"]
    seen = st["kv_len"].long()[:, None] - new[:, None] + i + 1
    dead = torch.arange(L, device=q.device) >= seen[..., None]
    z = z.masked_fill(dead[:, None, None], -math.inf)
    z = torch.exp(z - z.amax(-1, keepdim=True))
    z = z / z.sum(-1, keepdim=True)
    o = torch.bmm(z.view(B * kv, -1, L), v.view(B * kv, L, hd)).view(B, kv, H // kv, n, hd).permute(0, 3, 1, 2, 4).reshape(B * n, H * hd)
    return o.to(bf16)


def _plain_verify(st):
    draft, p, q, count = st["draft"].long(), st["p"], st["q"], st["count"].long()
    B, K = draft.shape
    V = p.shape[-1]
    px = p[:, :K].gather(-1, draft[..., None])[..., 0].double()
    qx = q.gather(-1, draft[..., None])[..., 0].double()
    i = torch.arange(K, device=p.device)
    ok = (st["u"].double() * qx < px) & (i < count[:, None])
    taken = ok.long().cumprod(-1).sum(-1)
    b = torch.arange(B, device=p.device)
    row = p[b, taken].double()
    rest = (row - torch.where((taken < count)[:, None], q[b, taken.clamp(max=K - 1)].double(), 0.0)).clamp(min=0)
    rest = torch.where((rest.sum(-1) > 0)[:, None], rest, row)
    cdf = rest.cumsum(-1)
    token = torch.searchsorted(cdf, (st["pick"].double() * cdf[:, -1])[:, None], right=True)[:, 0].clamp(max=V - 1)
    at = torch.arange(K + 1, device=p.device)
    out = torch.where(at < taken[:, None], torch.cat([draft, draft[:, :1]], 1), -1)
    out = torch.where(at == taken[:, None], token[:, None], out)
    return [out.to(torch.int32), taken.to(torch.int32)]


# ------------------------------------------------------------------------------------------------------------------ work
def work(case):
    op = case["op"]
    if op == "rotary":
        n, e = case["rows"] * case["heads"], 4 if case["dtype"] == "f32" else 2
        return {"bytes": 2 * n * case["hd"] * e + case["rows"] * 4, "flops": 3 * n * case["rot"]}
    if op == "pages":  # lengths and held pages in, the step's tables out (two words a token)
        t = sum(_new_tokens(case))
        return {"bytes": case["requests"] * 24 + t * 8, "flops": t}
    if op == "store":  # rows in, codes and scales out and in again, rows out
        n = 2 * case["rows"] * case["kv"]
        return {"bytes": n * (2 * case["hd"] * 2 + 2 * (case["hd"] // 2 + 4)) + 8 * case["rows"], "flops": 6 * n * case["hd"]}
    if op == "attn":
        L = case["longest"] if case["even"] else case["longest"] * 17 // 32
        L = max(L, case["queries"])
        n = case["requests"] * L * case["kv"]
        return {"bytes": 2 * n * (case["hd"] // 2 + 4) + 4 * case["requests"] * case["queries"] * case["heads"] * case["hd"],
                "flops": 4 * case["requests"] * L * case["queries"] * case["heads"] * case["hd"]}
    # the row at which the drafts end, of the target and (where a draft was refused, about three in four) of the drafter
    e = 4 if case["dtype"] == "f32" else 2
    return {"bytes": case["requests"] * case["vocab"] * e * 7 // 4, "flops": 3 * case["requests"] * case["vocab"]}


# ------------------------------------------------------------------------------------------------------------------ 64 bits
def exact(case, seed):
    """The operators' definitions in 64 bits, on the inputs of prepare(case, seed)."""
    st = prepare(case, seed)
    f64 = torch.float64
    op = case["op"]
    if op == "rotary":  # a pair is a complex number, turned by e^(i angle)
        w, mscale = _freq(case)
        angle = torch.outer(st["pos"].to(f64), w.to(DEV)) * (-1 if case["backward"] else 1)
        z = torch.polar(torch.full_like(angle, mscale), angle)[:, None, :]
        x = st["x"].to(f64)
        y = x.clone()
        if case["pairs"] == "interleaved":
            c = torch.view_as_complex(x[..., :case["rot"]].unflatten(-1, (-1, 2)).contiguous()) * z
            y[..., :case["rot"]] = torch.view_as_real(c).flatten(-2)
        else:
            h = case["rot"] // 2
            c = torch.complex(x[..., :h].contiguous(), x[..., h:2 * h].contiguous()) * z
            y[..., :h], y[..., h:2 * h] = c.real, c.imag
        return y
    if op == "pages":
        ctx, new = _lengths(case, seed)
        P, held, free, table = case["page"], st["held"].tolist(), st["free"].tolist(), st["table"].tolist()
        cu, slots, pos, taken = [0], [], [], 0
        for b, (c, n) in enumerate(zip(ctx, new)):
            while held[b] * P < c + n:
                table[b][held[b]] = free[taken]
                held[b], taken = held[b] + 1, taken + 1
            for t in range(c, c + n):
                pos.append(t)
                slots.append(table[b][t // P] * P + t % P)
            cu.append(cu[-1] + n)
        return [torch.tensor(v, dtype=torch.int32) for v in (table, [c + n for c, n in zip(ctx, new)], cu, slots, pos, held, [taken])]
    if op == "store":
        out = []
        for x in (st["k"], st["v"]):
            x = x.to(f64)
            lo, span = x.min(-1, keepdim=True).values, x.max(-1, keepdim=True).values - x.min(-1, keepdim=True).values
            mant, ex = torch.frexp(span / 15)  # to the 8 bits of a bf16
            s = torch.ldexp(torch.round(mant * 256), ex - 8)
            c = torch.where(s > 0, torch.round((x - lo) / torch.where(s > 0, s, 1.0)), 0.0).clamp(0, 15)
            out.append(lo + c * s)
        return out
    if op == "attn":
        H, kv, hd, P = case["heads"], case["kv"], case["hd"], case["page"]
        out = torch.empty(st["q"].shape, dtype=f64, device=DEV)
        cu, length = st["cu_q"].tolist(), st["kv_len"].tolist()
        for b, L in enumerate(length):
            pages = st["table"][b, :-(-L // P)].long()
            sc = st["scales"][pages].to(f64)
            n = cu[b + 1] - cu[b]
            q = st["q"][cu[b]:cu[b + 1]].to(f64)
            hide = torch.ones(n, L, dtype=torch.bool, device=DEV).triu(L - n + 1)
            for h in range(kv):
                k = (sc[:, 0, h, :, 1:] + unpack_keys(st["codes"][pages, 0, h], hd) * sc[:, 0, h, :, :1]).reshape(-1, hd)[:L]
                v = (sc[:, 1, h, :, 1:] + unpack_values(st["codes"][pages, 1, h], hd) * sc[:, 1, h, :, :1]).reshape(-1, hd)[:L]
                for j in range(h * H // kv, (h + 1) * H // kv):
                    z = (q[:, j] @ k.T * st["alpha"]).masked_fill(hide, -math.inf)
                    out[cu[b]:cu[b + 1], j] = torch.softmax(z, -1) @ v
        return out.flatten(1)
    B, K = st["draft"].shape
    tokens, taken = torch.full((B, K + 1), -1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
    draft, count, u, pick = (st[k].tolist() for k in ("draft", "count", "u", "pick"))
    for b in range(B):
        n = 0
        while n < count[b] and u[b][n] * float(st["q"][b, n, draft[b][n]]) < float(st["p"][b, n, draft[b][n]]):
            tokens[b, n] = draft[b][n]
            n += 1
        r = st["p"][b, n].to(f64)
        if n < count[b]:
            left = torch.relu(r - st["q"][b, n].to(f64))
            r = left if float(left.sum()) > 0 else r
        cdf = torch.cumsum(r, 0)
        over = torch.nonzero(cdf > pick[b] * cdf[-1])
        tokens[b, n] = int(over[0]) if len(over) else case["vocab"] - 1
        taken[b] = n
    return [tokens, taken]

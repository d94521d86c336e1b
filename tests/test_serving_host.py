"""What the serving operators refuse, and the frequencies of a rotary plan: no GPU needed (the checks come before any launch)."""
import ctypes
import math

import pytest
import torch

from grove_amd import _lib, ops

bf16, f32, i32 = torch.bfloat16, torch.float32, torch.int32


def ints(*v):
    return torch.tensor(v, dtype=i32)


def cache(pages=4, P=16, kv=2, hd=64):
    return ops.kv4_cache(pages, P, kv, hd, "cpu")


# ----------------------------------------------------------------------------- rotary plan
def test_plan_plain_frequencies():
    w = ops.rotary_plan(8, 10000.0, device="cpu").freq
    assert w.dtype == torch.float64
    assert torch.allclose(w, torch.tensor([1.0, 0.1, 0.01, 0.001], dtype=torch.float64), rtol=1e-14, atol=0)


def test_plan_scalings():
    base = ops.rotary_plan(64, device="cpu")
    lin = ops.rotary_plan(64, scaling="linear", factor=4.0, device="cpu")
    assert torch.allclose(lin.freq, base.freq / 4, rtol=1e-14, atol=0) and lin.mscale == 1.0
    ntk = ops.rotary_plan(64, scaling="ntk", factor=4.0, device="cpu")
    assert ntk.freq[0] == 1.0 and math.isclose(float(ntk.freq[-1]), float(base.freq[-1]) / 4, rel_tol=1e-12)
    yarn = ops.rotary_plan(64, scaling="yarn", factor=4.0, trained_len=4096, device="cpu")
    turns = base.freq * 4096 / (2 * math.pi)
    assert torch.equal(yarn.freq[turns > 40], base.freq[turns > 40]) and torch.allclose(yarn.freq[turns < 0.7], base.freq[turns < 0.7] / 4, rtol=1e-12, atol=0)
    assert ((yarn.freq <= base.freq) & (yarn.freq >= base.freq / 4 * (1 - 1e-12))).all()
    assert math.isclose(yarn.mscale, 0.1 * math.log(4) + 1)


@pytest.mark.parametrize("kw", [dict(rot=0), dict(rot=7), dict(rot=8, scaling="cubic"), dict(rot=8, factor=2.0), dict(rot=2, scaling="ntk", factor=2.0),
                                dict(rot=8, theta=1.0), dict(rot=8, scaling="linear", factor=0.5), dict(rot=8, scaling="yarn", factor=2.0, trained_len=0)])
def test_plan_refusals(kw):
    with pytest.raises(RuntimeError):
        ops.rotary_plan(device="cpu", **kw)


# ----------------------------------------------------------------------------- refusals of the front end
def refused(text, fn, *a, **kw):
    with pytest.raises(RuntimeError, match=text):
        fn(*a, **kw)


def test_rotary_refusals():
    plan = ops.rotary_plan(16, device="cpu")
    x, pos = torch.zeros(3, 2, 16, dtype=bf16), ints(0, 1, 2)
    refused("bf16 or f32", ops.rotary, x.half(), pos, plan)
    refused("bf16 or f32", ops.rotary, x[0], pos, plan)
    refused("contiguous", ops.rotary, x.transpose(1, 2), pos, plan)
    refused("frequencies", ops.rotary, x[..., :8], pos, plan)
    refused("pos", ops.rotary, x, pos.long(), plan)
    refused("pos", ops.rotary, x, pos[:2], plan)
    refused("match x", ops.rotary, x, pos, plan, out=x.float())
    refused("share memory", ops.rotary, x, pos, plan, out=torch.zeros(1, 2, 16, dtype=bf16).expand(3, 2, 16))
    refused("overlaps", ops.rotary, x[:2], pos[:2], plan, out=x[1:])
    refused("device", ops.rotary, x, pos, plan)


def test_page_tables_refusals():
    t, n = torch.zeros(2, 4, dtype=i32), ints(1, 1)
    refused("table", ops.page_tables, n, n, t.long(), n, n, 16, 2)
    refused("table", ops.page_tables, n, n, t[:1].expand(2, 4), n, n, 16, 2)
    refused("held", ops.page_tables, n, n, t, ints(1), n, 16, 2)
    refused("free", ops.page_tables, n, n, t, n, n.long(), 16, 2)
    refused("power of two", ops.page_tables, n, n, t, n, n, 24, 2)
    refused("rows", ops.page_tables, n, n, t, n, n, 16, -1)
    refused("overlaps", ops.page_tables, n, n, t, n, t[0], 16, 2)
    refused("at most 4096", ops.page_tables, *(torch.zeros(4097, dtype=i32),) * 2, torch.zeros(4097, 1, dtype=i32), torch.zeros(4097, dtype=i32), n, 16, 2)
    refused("device", ops.page_tables, n, n, t, n, n, 16, 2)


def test_cache_refusals():
    refused("page", ops.kv4_cache, 4, 8, 2, 64, "cpu")
    refused("page", ops.kv4_cache, 4, 16, 2, 80, "cpu")
    c, k, s = cache(), torch.zeros(3, 2, 64, dtype=bf16), ints(0, 1, 2)
    refused("k and v", ops.kv4_append, k.float(), k, c, s)
    refused("k and v", ops.kv4_append, k, k[:, :1], c, s)
    refused("contiguous", ops.kv4_append, k.transpose(1, 2).contiguous().transpose(1, 2), k, c, s)
    refused("rows", ops.kv4_append, k, k[:2], c, s)
    refused("slots", ops.kv4_append, k, k, c, s.long())
    refused("fit", ops.kv4_append, k, k, ops.KV4Cache(c.codes, c.scales[:3]), s)
    refused("contiguous", ops.kv4_append, k, k, ops.KV4Cache(c.codes.transpose(0, 2), c.scales), s)
    inside = c.scales.view(-1)[:1].expand(3 * 2 * 64).as_strided((3, 2, 64), (0, 0, 1))
    refused("lies in the cache", ops.kv4_append, k, inside, c, s)
    refused("out_dtype", ops.kv4_read, c, s, torch.float16)
    refused("device", ops.kv4_append, k, k, c, s)
    refused("device", ops.kv4_read, c, s)


def test_attn_refusals():
    c, q, t = cache(), torch.zeros(3, 4, 64, dtype=bf16), torch.zeros(2, 2, dtype=i32)
    n, cu = ints(1, 2), ints(0, 1, 3)
    refused("q must", ops.kv4_attn, q.float(), c, t, n, cu, 2, 1.0)
    refused("q must", ops.kv4_attn, q[:, :3], c, t, n, cu, 2, 1.0)
    refused("q must", ops.kv4_attn, q[..., :32], c, t, n, cu, 2, 1.0)
    refused("table", ops.kv4_attn, q, c, t.long(), n, cu, 2, 1.0)
    refused("kv_len", ops.kv4_attn, q, c, t, n[:1], cu, 2, 1.0)
    refused("cu_q", ops.kv4_attn, q, c, t, n, cu[:2], 2, 1.0)
    refused("out must", ops.kv4_attn, q, c, t, n, cu, 2, 1.0, out=torch.zeros(3, 256))
    refused("out must", ops.kv4_attn, q, c, t, n, cu, 2, 1.0, out=torch.zeros(1, 256, dtype=bf16).expand(3, 256))
    refused("overlaps", ops.kv4_attn, q, c, t, n, cu, 2, 1.0, out=q.view(3, 256))
    refused("max_q", ops.kv4_attn, q, c, t, n, cu, -1, 1.0)
    refused("aligned to 4 bytes", ops.kv4_attn, q, c, t, n, cu, 2, 1.0, out=torch.zeros(3, 257, dtype=bf16)[:, 1:])
    refused("device", ops.kv4_attn, q, c, t, n, cu, 2, 1.0)


def test_verify_refusals():
    d, p, q = torch.zeros(2, 3, dtype=i32), torch.zeros(2, 4, 9), torch.zeros(2, 3, 9)
    u, k = torch.zeros(2, 3), torch.zeros(2)
    refused("draft", ops.verify_drafts, d.long(), q, p, u, k)
    refused("p must", ops.verify_drafts, d, q, p[:, :3], u, k)
    refused("p must", ops.verify_drafts, d, q, p.double(), u, k)
    refused("q must", ops.verify_drafts, d, q.bfloat16(), p, u, k)
    refused("q must", ops.verify_drafts, d, q[..., :8], p, u, k)
    refused("u must", ops.verify_drafts, d, q, p, u.double(), k)
    refused("pick", ops.verify_drafts, d, q, p, u, k[:1])
    refused("count", ops.verify_drafts, d, q, p, u, k, count=torch.zeros(2))
    refused("device", ops.verify_drafts, d, q, p, u, k)


# ----------------------------------------------------------------------------- refusals of the C entries
def entry(name, struct, **fields):
    p = struct()
    for k, v in fields.items():
        setattr(p, k, v)
    rc = getattr(_lib.lib(), name)(ctypes.byref(p), None)
    return rc, _lib.last_error() if rc else ""


@pytest.mark.parametrize("name,struct,fields,code,text", [
    ("grove_rotary", _lib.RotaryParams, dict(rows=1, heads=1, hd=8, rot=10), -1, "rotary"),
    ("grove_rotary", _lib.RotaryParams, dict(rows=1, heads=1, hd=8, rot=8), -1, "null"),
    ("grove_rotary", _lib.RotaryParams, dict(rows=1, heads=1, hd=8, rot=8, x=64, y=64, pos=64, freq=64, sx_row=8, sy_row=16), -1, "in place"),
    ("grove_page_tables", _lib.PageTablesParams, dict(requests=0, max_pages=1, page=16, ld_table=1), -1, "bad shape"),
    ("grove_page_tables", _lib.PageTablesParams, dict(requests=1, max_pages=1, page=24, ld_table=1), -1, "power of two"),
    ("grove_page_tables", _lib.PageTablesParams, dict(requests=1, max_pages=1, page=16, ld_table=1), -1, "null"),
    ("grove_kv4_append", _lib.Kv4AppendParams, dict(rows=1, kv=1, hd=80, page=16, pages=1), -1, "head size"),
    ("grove_kv4_append", _lib.Kv4AppendParams, dict(rows=1, kv=1, hd=64, page=16, pages=1 << 28), -1, "pages"),
    ("grove_kv4_append", _lib.Kv4AppendParams, dict(rows=1, kv=1, hd=64, page=16, pages=1), -1, "null"),
    ("grove_kv4_append", _lib.Kv4AppendParams, dict(rows=1, kv=1, hd=64, page=16, pages=1, k=64, v=64, codes=72, scales=64, slots=64), -3, "aligned"),
    ("grove_kv4_read", _lib.Kv4ReadParams, dict(rows=1, kv=1, hd=64, page=8, pages=1), -1, "page"),
    ("grove_kv4_read", _lib.Kv4ReadParams, dict(rows=1, kv=1, hd=64, page=16, pages=1), -1, "null"),
    ("grove_kv4_attn", _lib.Kv4AttnParams, dict(requests=1, rows=1, heads=3, kv=2, hd=64, page=16, pages=1, max_pages=1, ld_table=1, max_q=1), -1, "multiple"),
    ("grove_kv4_attn", _lib.Kv4AttnParams, dict(requests=1, rows=1, heads=2, kv=2, hd=64, page=16, pages=1, max_pages=1, ld_table=1, max_q=1), -1, "null"),
    ("grove_kv4_attn", _lib.Kv4AttnParams, dict(requests=1, rows=1, heads=2, kv=2, hd=64, page=16, pages=1, max_pages=1 << 27, ld_table=1 << 27, max_q=1, q=64,
                                                codes=64, scales=64, table=64, kv_len=64, cu_q=64, out=64, n_split=1), -1, "2^30"),
    ("grove_kv4_attn", _lib.Kv4AttnParams, dict(requests=1, rows=1, heads=2, kv=2, hd=64, page=16, pages=1, max_pages=1, ld_table=1, max_q=1, q=72,
                                                codes=64, scales=64, table=64, kv_len=64, cu_q=64, out=64, n_split=1), -3, "aligned"),
    ("grove_kv4_attn", _lib.Kv4AttnParams, dict(requests=1, rows=1, heads=2, kv=2, hd=64, page=16, pages=1, max_pages=1, ld_table=1, max_q=1, q=64,
                                                codes=64, scales=64, table=64, kv_len=64, cu_q=64, out=64, n_split=2), -4, "workspace"),
    ("grove_verify_drafts", _lib.VerifyDraftsParams, dict(requests=1, drafts=-1, vocab=5), -1, "bad shape"),
    ("grove_verify_drafts", _lib.VerifyDraftsParams, dict(requests=1, drafts=1, vocab=5), -1, "null"),
])
def test_entries_refuse(name, struct, fields, code, text):
    rc, msg = entry(name, struct, **fields)
    assert rc == code and text in msg, (rc, msg)


def test_entries_take_nothing():
    assert entry("grove_rotary", _lib.RotaryParams, rows=0, heads=2, hd=8, rot=8)[0] == 0
    assert entry("grove_kv4_append", _lib.Kv4AppendParams, rows=0, kv=1, hd=64, page=16, pages=1)[0] == 0
    assert entry("grove_kv4_attn", _lib.Kv4AttnParams, requests=1, rows=0, heads=2, kv=2, hd=64, page=16, pages=1, max_pages=1, ld_table=1, max_q=1)[0] == 0
    assert entry("grove_verify_drafts", _lib.VerifyDraftsParams, requests=0, drafts=1, vocab=5)[0] == 0

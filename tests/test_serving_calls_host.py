"""What the serving operators hand to their C entries, with the launch replaced: no GPU needed."""
import ctypes
import math

import pytest
import torch

from grove_amd import _lib, ops

bf16, i32 = torch.bfloat16, torch.int32


def ints(*v):
    return torch.tensor(v, dtype=i32)


@pytest.fixture
def launched(monkeypatch):
    """The params and tensors of every launch, in order, as (name, params struct, tensors)."""
    calls = []
    structs = {"kv4_attn": _lib.Kv4AttnParams}

    def launch(name, params, *ts):
        calls.append((name, structs[name].from_buffer_copy(params), ts))
    monkeypatch.setattr(ops, "_launch", launch)
    monkeypatch.setattr(ops, "_need_device", lambda what, t: None)
    return calls


def attn(q, table, out=None, rows_of=(1, 1, 1)):
    c = ops.kv4_cache(4, 16, 2, 64, "cpu")
    B = table.shape[0]
    cu = ints(0, *torch.tensor(rows_of).cumsum(0).tolist())
    return ops.kv4_attn(q, c, table, torch.full((B,), 9, dtype=i32), cu, max(rows_of), 1.0, out=out)


# ----------------------------------------------------------------------------- tables
@pytest.mark.parametrize("make,stride", [
    (lambda t: t[:1].expand(3, 5), 0),                       # one page list for requests that share a context
    (lambda t: t.view(-1).as_strided((3, 5), (2, 1)), 2),    # rows that overlap: the kernel only reads them
    (lambda t: t, 5),
    (lambda t: torch.zeros(3, 9, dtype=i32)[:, :5], 9)])
def test_attn_table_rows_keep_their_stride(launched, make, stride):
    """No request's row is looked for behind the tensor."""
    table = make(torch.arange(15, dtype=i32).view(3, 5))
    attn(torch.zeros(3, 4, 64, dtype=bf16), table)
    (_, p, _), = launched
    assert p.ld_table == stride and p.max_pages == 5
    last = p.table + 4 * (2 * p.ld_table + p.max_pages)
    assert last <= table.untyped_storage().data_ptr() + table.untyped_storage().nbytes()


def test_attn_entry_takes_shared_table_rows():
    """ld_table below max_pages passes the shape check (the next one, null pointers, refuses); a negative one does not."""
    fields = dict(requests=2, rows=1, heads=2, kv=2, hd=64, page=16, pages=1, max_pages=4, max_q=1)
    for ld, text in ((0, "null"), (1, "null"), (-4, "bad shape")):
        p = _lib.Kv4AttnParams(**fields, ld_table=ld)
        assert _lib.lib().grove_kv4_attn(ctypes.byref(p), None) == -1 and text in _lib.last_error(), ld


# ----------------------------------------------------------------------------- q
def packed(rows, width, start):
    """[rows, 4, 64] as columns of a wider activation."""
    return torch.randn(rows, width).to(bf16)[:, start:start + 256].unflatten(1, (4, 64))


def flat(rows, start):
    """A contiguous q that starts `start` elements behind an aligned address."""
    return torch.randn(start + rows * 256).to(bf16)[start:].view(rows, 4, 64)


@pytest.mark.parametrize("q,in_place", [
    (flat(3, 0), True), (flat(3, 1), False), (flat(1, 3), False), (flat(3, 8), True), (packed(3, 512, 8), True), (packed(3, 259, 0), False), (packed(3, 512, 1), False),
    (packed(1, 259, 0), True), (packed(1, 259, 3), False), (packed(1, 512, 8), True),
    (torch.randn(3, 4, 67).to(bf16)[..., :64], False), (torch.randn(1, 1, 4, 67).to(bf16)[0, ..., :64], False),
    (torch.randn(1, 256).to(bf16).as_strided((1, 4, 64), (3, 64, 1)), True), (torch.randn(1, 4, 64).to(bf16).expand(3, 4, 64), True)])
def test_attn_q_reaches_the_entry_aligned(launched, q, in_place):
    """Any start and any strides: read in place where the entry can, laid out anew elsewhere; what arrives are q's values."""
    rows = q.shape[0]
    attn(q, torch.zeros(3, 5, dtype=i32), rows_of=(1,) * rows + (0,) * (3 - rows))
    (_, p, (got, *_)), = launched
    assert p.q == got.data_ptr() and p.q % 16 == 0 and p.sq_row % 8 == 0 and p.sq_head % 8 == 0
    assert (got.data_ptr() == q.data_ptr()) == in_place
    assert torch.equal(got, q) and (rows == 1 or got.stride(0) == p.sq_row) and got.stride(1) == p.sq_head


def test_attn_one_head_and_odd_head_stride(launched):
    c = ops.kv4_cache(4, 16, 1, 64, "cpu")
    q = torch.randn(2, 64).to(bf16).as_strided((2, 1, 64), (64, 3, 1))
    ops.kv4_attn(q, c, torch.zeros(2, 5, dtype=i32), ints(3, 3), ints(0, 1, 2), 1, 1.0)
    (_, p, (got, *_)), = launched
    assert p.sq_head % 8 == 0 and torch.equal(got, q)


def test_attn_out_of_one_row(launched):
    """The stride of a single row is never used: any is taken."""
    c = ops.kv4_cache(4, 16, 2, 64, "cpu")
    out = torch.zeros(1, 259, dtype=bf16)[:, :256]
    assert ops.kv4_attn(flat(1, 0), c, torch.zeros(1, 5, dtype=i32), ints(3), ints(0, 1), 1, 1.0, out=out) is out
    (_, p, _), = launched
    assert p.out == out.data_ptr() and p.so_row % 2 == 0


# ----------------------------------------------------------------------------- the decoder stack
def test_stack_has_its_plan_before_the_first_step(monkeypatch):
    """The plain plan is copied from the host; the first paged_step may be a captured one, in which such a copy is an error."""
    from grove_amd.model.llama import LlamaStack
    from grove_amd.synthetic import TINY
    stack = LlamaStack.__new__(LlamaStack)
    stack.d, stack.dev, stack.layers, stack.norm, stack.fp32_stream = TINY, "cpu", [], None, False
    cache = stack.new_kv4_cache(2, 16)
    monkeypatch.setattr(ops, "rotary_plan", lambda *a, **kw: pytest.fail("a plan is made within the step"))
    monkeypatch.setattr(ops, "rmsnorm", lambda x, *a, **kw: x)
    x = torch.zeros(1, TINY.hidden, dtype=bf16)
    assert stack.paged_step(x, None, None, cache, 1) is x


# ----------------------------------------------------------------------------- stretched frequencies
@pytest.mark.parametrize("rot,theta,factor,trained", [(64, 10000.0, 4.0, 4096), (128, 10000.0, 8.0, 2048), (128, 500000.0, 16.0, 8192), (32, 10000.0, 2.0, 512)])
def test_plan_between_the_ends(rot, theta, factor, trained):
    """Every frequency of the three scalings, pair by pair; yarn's blend between its ends too."""
    base = [theta ** (-2 * i / rot) for i in range(rot // 2)]

    def plan(kind):
        return ops.rotary_plan(rot, theta, scaling=kind, factor=factor, trained_len=trained, device="cpu").freq.tolist()
    for got, w in zip(plan("linear"), base):
        assert math.isclose(got, w / factor, rel_tol=1e-12)
    for i, (got, w) in enumerate(zip(plan("ntk"), base)):
        assert math.isclose(got, w / factor ** (2 * i / (rot - 2)), rel_tol=1e-12)
    # pair p turns trained * theta^(-2 p / rot) / (2 pi) times: the real p at which that is 32, and 1
    fast, slow = (rot / 2 * math.log(trained / (2 * math.pi * t), theta) for t in (32.0, 1.0))
    low, high = max(math.floor(fast), 0), math.ceil(slow)
    assert 0 < high < rot - 1 and low < high
    inside = 0
    for i, (got, w) in enumerate(zip(plan("yarn"), base)):
        part = min(max((i - low) / (high - low), 0.0), 1.0)
        inside += 0 < part < 1
        assert math.isclose(got, w * (1 - part) + w / factor * part, rel_tol=1e-12), i
    assert inside >= 3


# ----------------------------------------------------------------------------- inputs that reach into the cache
def test_append_input_that_ends_in_the_cache():
    """A cache in one buffer with the rows before it: rows that run on into the codes are refused, rows that end where they begin are not."""
    pages, kv, P, hd = 2, 1, 16, 32
    codes, scales = pages * 2 * kv * P * hd // 2, pages * 2 * kv * P * 2
    buf = torch.zeros(256 + codes + 2 * scales, dtype=torch.uint8)
    c = ops.KV4Cache(buf[256:256 + codes].view(pages, 2, kv, P * hd // 2), buf[256 + codes:].view(bf16).view(pages, 2, kv, P, 2))
    rows, slots = buf.view(bf16)[:128].view(4, 1, 32), torch.arange(4, dtype=i32)
    over = buf.view(bf16)[32:160].view(4, 1, 32)
    other = torch.zeros(4, 1, 32, dtype=bf16)
    with pytest.raises(RuntimeError, match="need device tensors"):
        ops.kv4_append(rows, other, c, slots)
    for k, v in ((over, other), (other, over)):
        with pytest.raises(RuntimeError, match="lies in the cache"):
            ops.kv4_append(k, v, c, slots)
    with pytest.raises(RuntimeError, match="lies in the cache"):
        ops.kv4_append(other, other, c, buf[250:].view(torch.uint8)[2:18].view(i32))

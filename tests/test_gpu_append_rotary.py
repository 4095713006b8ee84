"""New tokens join a cache: keys and queries against float64, values and everything that is not written bit by bit."""
import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def make(dtype, batch, tokens, hq, hk, dim, page, lengths, seed=0, extra=3, joint=False, pool="plain"):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    if joint:
        x = rand(batch, tokens, hq + 2 * hk, dim)
        q, k, v = x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]
    else:
        q, k, v = rand(batch, tokens, hq, dim), rand(batch, tokens, hk, dim), rand(batch, tokens, hk, dim)
    width = (max(lengths) + tokens + page - 1) // page
    n = batch * width + extra
    if pool == "joint":      # keys and values of a page side by side
        x = rand(n, 2, page, hk, dim)
        kp, vp = x[:, 0], x[:, 1]
    elif pool == "heads":    # heads outside, rows inside
        kp, vp = (rand(n, hk, page, dim).transpose(1, 2) for _ in range(2))
    else:
        kp, vp = rand(n, page, hk, dim), rand(n, page, hk, dim)
    table = torch.randperm(n, generator=gen, device="cuda")[:batch * width].view(batch, width).to(torch.int32)
    return q, k, v, kp, vp, table, torch.tensor(lengths, device="cuda")


def expected(k, v, kp, vp, table, lengths, counts, turned):
    """Copies of the pools with the new tokens in them, token by token; which key rows are new."""
    page = kp.shape[1]
    kw, vw = kp.double().clone(), vp.clone()
    bounds = torch.zeros_like(kw)
    for b in range(k.shape[0]):
        fresh = k.shape[1] if counts is None else min(max(0, int(counts[b])), k.shape[1])
        for i in range(fresh):
            s = max(0, int(lengths[b])) + i
            if s // page >= table.shape[1]:
                continue
            at = int(table[b, s // page])
            if 0 <= at < kp.shape[0]:
                kw[at, s % page], vw[at, s % page] = turned[0][b, i], v[b, i]
                bounds[at, s % page] = turned[1][b, i]
    return kw, vw, bounds


CASES = [
    # dtype, batch, tokens, q heads, kv heads, dim, page, lengths, sections, adjacent, interleaved
    (BF16, 1, 1, 32, 8, 128, 16, [1601], (16, 24, 24), False, False),
    (BF16, 1, 1, 1, 1, 2, 8, [0], (1,), False, False),
    (F16, 3, 7, 4, 2, 64, 8, [0, 5, 31], (32,), True, False),
    (F32, 2, 33, 3, 3, 80, 32, [31, 1], (20, 20), False, True),
    (BF16, 2, 65, 7, 1, 72, 64, [63, 64], (10, 8), True, False),
    (F16, 1, 300, 2, 2, 34, 16, [15], (5, 4, 3, 2), False, True),
    (F32, 4, 3, 5, 5, 256, 8, [7, 8, 9, 1000], (128,), True, False),
    (BF16, 2, 129, 28, 4, 96, 128, [0, 127], (12, 12, 24), False, False),
    (BF16, 40, 1, 16, 4, 64, 256, list(range(250, 290)), (16, 16), False, False),
    (F32, 1, 17, 6, 2, 30, 8, [3], (7,), False, False),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("layout", ["plain", "joint", "heads"])
@pytest.mark.parametrize("positions", [None, torch.int32, torch.int64, F32])
def test_against_float64(pkg, case, layout, positions):
    dtype, batch, tokens, hq, hk, dim, page, lengths, sections, adjacent, interleaved = case
    q, k, v, kp, vp, table, held = make(dtype, batch, tokens, hq, hk, dim, page, lengths, joint=layout == "joint", pool=layout)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(3)
    f = torch.rand(sum(sections), generator=gen, device="cuda")
    places = (held[:, None] + torch.arange(tokens, device="cuda")).expand(len(sections), -1, -1)
    at = None if positions is None else torch.randint(0, 5000, places.shape, generator=gen, device="cuda").to(positions)
    counts = None
    if layout != "plain":
        counts = torch.randint(0, tokens + 1, (batch,), generator=gen, device="cuda", dtype=torch.int32)
    how = dict(adjacent=adjacent, interleaved=interleaved)
    kp0, vp0 = kp.clone(), vp.clone()

    def turned(x):
        want = ao.rotary(x.double(), places if at is None else at, f, sections, **how)
        return want, ao.rotary_bound(want, x.double(), sum(sections), adjacent, dtype)

    got = pkg.attention.append_rotary(q, k, v, at, f, sections, kp, vp, table, held, counts=counts, **how)
    ao.within(got, *turned(q))
    kw, vw, bounds = expected(k, v, kp0, vp0, table, held, counts, turned(k))
    ao.within(kp, kw, bounds)          # 0 where nothing is written
    assert torch.equal(vp, vw)
    # the same bits as the rotation alone
    alone = pkg.attention.rotary(q, k, (places if at is None else at).contiguous(), f, sections, **how)
    assert torch.equal(got, alone[0])


def test_without_queries_and_empty(pkg):
    q, k, v, kp, vp, table, held = make(BF16, 2, 5, 4, 2, 64, 8, [3, 9])
    f = torch.rand(32, device="cuda")
    a, b = kp.clone(), vp.clone()
    assert pkg.attention.append_rotary(None, k, v, None, f, (32,), a, b, table, held) is None
    pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table, held)
    assert torch.equal(a, kp) and torch.equal(b, vp)
    before = kp.clone()
    for tokens, batch in ((0, 2), (5, 0)):
        out = pkg.attention.append_rotary(q[:batch, :tokens], k[:batch, :tokens], v[:batch, :tokens], None, f, (32,), kp, vp, table[:batch], held[:batch])
        assert out.shape == (batch, tokens, 4, 64) and torch.equal(kp, before)
    none = kp[:0]
    out = pkg.attention.append_rotary(q, k, v, None, f, (32,), none, none.clone(), table, held)   # a pool of no pages: only queries are turned
    assert out.shape == q.shape
    pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table[:, :0], held)              # a table of no pages
    assert torch.equal(kp, before)


@pytest.mark.parametrize("integer", [torch.int32, torch.int64])
def test_pages_that_are_none(pkg, integer):
    """Entries below 0, behind the pool, places behind the table, counts and lengths outside what they count: nothing is written."""
    q, k, v, kp, vp, table, held = make(F16, 4, 20, 2, 2, 64, 8, [4, 4, 4, 4])
    f = torch.rand(32, device="cuda")
    table = table.to(integer)
    big = 2 ** 31 - 1 if integer == torch.int32 else 2 ** 40
    table[0, 1], table[1, 0], table[2, 2] = -1, kp.shape[0], big
    held = torch.tensor([4, 4, 4, 2 ** 31 - 1 if integer == torch.int32 else 2 ** 50], dtype=integer, device="cuda")
    counts = torch.tensor([20, 99, 13, 20], dtype=integer, device="cuda")
    kp0, vp0 = kp.clone(), vp.clone()
    places = (held.clamp(max=2 ** 30)[:, None] + torch.arange(20, device="cuda"))[None]
    want = ao.rotary(k.double(), places, f, (32,))
    kw, vw, bounds = expected(k, v, kp0, vp0, table, held, counts, (want, ao.rotary_bound(want, k.double(), 32, False, F16)))
    pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table, held, counts=counts)
    ao.within(kp, kw, bounds)
    assert torch.equal(vp, vw)
    held[:] = -7                       # taken as 0
    counts[:] = torch.tensor([-1, 0, -2 ** 31, 0], device="cuda")
    kp0, vp0 = kp.clone(), vp.clone()
    pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table, held, counts=counts)
    assert torch.equal(kp, kp0) and torch.equal(vp, vp0)
    places = torch.arange(20, device="cuda").expand(1, 4, -1)
    want = ao.rotary(k.double(), places, f, (32,))
    kw, vw, bounds = expected(k, v, kp0, vp0, table, held, None, (want, ao.rotary_bound(want, k.double(), 32, False, F16)))
    pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table, held)
    ao.within(kp, kw, bounds)
    assert torch.equal(vp, vw)


def test_bits_that_are_no_numbers(pkg):
    """Values keep their bits; keys that pass through the rotation too; tokens that are not written do not matter."""
    q, k, v, kp, vp, table, held = make(BF16, 1, 6, 2, 2, 64, 8, [5])
    f = torch.rand(16, device="cuda")
    v[0, 1], v[0, 2] = float("nan"), float("-inf")
    k[0, 3, :, 40:] = float("inf")
    k[0, 5], v[0, 5] = float("nan"), float("nan")
    counts = torch.tensor([5], device="cuda")
    before = kp.clone()
    pkg.attention.append_rotary(q, k, v, None, f, (16,), kp, vp, table, held, counts=counts)
    slots = [(int(table[0, s // 8]), s % 8) for s in range(5, 10)]
    for i, at in enumerate(slots):
        assert torch.equal(vp[at].view(torch.int16), v[0, i].view(torch.int16))
        assert torch.equal(kp[at][:, 32:], k[0, i, :, 32:])
    assert torch.isfinite(kp[slots[3]][:, :32]).all()
    last = (int(table[0, 10 // 8]), 10 % 8)
    assert torch.equal(kp[last], before[last])


def test_pool_beyond_32_bits(pkg):
    """More than 2^32 bytes and 2^31 elements into a pool."""
    page, hk, dim = 64, 8, 128
    pages = 2 ** 31 // (page * hk * dim) + 40
    kp, vp = (torch.empty((pages, page, hk, dim), dtype=BF16, device="cuda") for _ in range(2))
    q, k, v, *_ = make(BF16, 2, 3, 8, hk, dim, page, [0, 0])
    table = torch.tensor([[pages - 1, 5], [pages - 2, pages - 3]], device="cuda")
    held = torch.tensor([62, 0], device="cuda")
    kp[table.flatten()] = 0
    vp[table.flatten()] = 0
    f = torch.rand(64, device="cuda")
    pkg.attention.append_rotary(q, k, v, None, f, (64,), kp, vp, table, held)
    assert torch.equal(vp[pages - 1, 62:], v[0, :2]) and torch.equal(vp[5, 0], v[0, 2]) and torch.equal(vp[pages - 2, :3], v[1])
    assert not vp[pages - 1, :62].any() and not vp[5, 1:].any() and not vp[pages - 3].any() and not kp[pages - 3].any()
    want = pkg.attention.rotary(k, None, (held[:, None] + torch.arange(3, device="cuda"))[None], f, (64,))[0]
    assert torch.equal(kp[pages - 1, 62:], want[0, :2]) and torch.equal(kp[5, 0], want[0, 2]) and torch.equal(kp[pages - 2, :3], want[1])


def test_captured_and_on_another_stream(pkg):
    q, k, v, kp, vp, table, held = make(BF16, 3, 1, 8, 2, 64, 16, [0, 15, 30])
    f = torch.rand(32, device="cuda")
    a, b, n = kp.clone(), vp.clone(), held.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = pkg.attention.append_rotary(q, k, v, None, f, (32,), a, b, table, n)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table, held)
    graph.replay()
    assert torch.equal(out, eager) and torch.equal(kp, a) and torch.equal(vp, b)
    held += 1                      # the next token, with other values
    q.mul_(2), k.mul_(-1), v.add_(1)
    graph.replay()
    n += 1
    eager = pkg.attention.append_rotary(q, k, v, None, f, (32,), a, b, table, n)
    assert torch.equal(out, eager) and torch.equal(kp, a) and torch.equal(vp, b)


def test_pools_know_that_they_were_written(pkg):
    q, k, v, kp, vp, table, held = make(F32, 1, 2, 2, 2, 64, 8, [0])
    f = torch.rand(32, device="cuda")
    w = torch.ones_like(kp, requires_grad=True)
    y = (w * kp).sum()
    pkg.attention.append_rotary(q, k, v, None, f, (32,), kp, vp, table, held)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_refusals(pkg):
    A = pkg.attention
    q, k, v, kp, vp, table, held = make(BF16, 2, 3, 4, 2, 64, 8, [0, 5])
    f = torch.rand(32, device="cuda")

    def call(text, **change):
        a = dict(q=q, k=k, v=v, positions=None, frequencies=f, sections=(32,), k_pages=kp, v_pages=vp, page_table=table, lengths=held)
        a.update(change)
        with pytest.raises(ValueError, match=text):
            A.append_rotary(**a)

    call("k must be a torch tensor", k=None)
    call("v must have the shape of k", v=v[:, :2])
    call("v must have the type", v=v.float())
    call("agree in all but the number of heads", q=q[:, :2])
    call("must be .pages, page_size", k_pages=kp[:, :, :1])
    call("must be .pages, page_size", v_pages=vp[0])
    call("one shape", v_pages=vp[:-1])
    call("type and device", k_pages=kp.float())
    call("contiguous heads", k_pages=torch.empty(kp.shape[0], 8, 64, 2, dtype=BF16, device="cuda").transpose(2, 3))
    call("power of two", k_pages=kp[:, :6], v_pages=vp[:, :6])
    call("overlap", v_pages=kp)
    call("overlap", k_pages=kp[:1].expand(kp.shape))
    call("overlap", v_pages=vp.as_strided(vp.shape, (vp.stride(0), 64, 64, 1)))
    call("overlap", k_pages=kp[:-1], v_pages=kp[1:])
    call("page_table must be", page_table=table[0])
    call("page_table must be", page_table=table.float())
    call("page_table must be", page_table=table[:1])
    call("lengths must be", lengths=held[:1])
    call("lengths must be", lengths=held.float())
    call("counts must be", counts=held[None])
    call("no CPU path", lengths=held.cpu())
    call("one frequency for each pair", sections=(31,))
    call("one section for each axis", positions=torch.zeros(2, 2, 3, device="cuda"))
    call("sections", sections=(0,), frequencies=f[:0])
    call("axes", sections=(1,) * 5, frequencies=f[:5])
    call("axes", sections=(), frequencies=f[:0])
    call("must be .batch, tokens", k=k[0], v=v[0], q=q[0])
    for name, x in (("q", q), ("k", k), ("v", v), ("k_pages", kp), ("v_pages", vp)):
        call(name + " has no gradient here", **{name: x.clone().requires_grad_()})
    call("frequencies has no gradient here", frequencies=f.clone().requires_grad_())
    with torch.no_grad():
        A.append_rotary(q.clone().requires_grad_(), k, v, None, f, (32,), kp, vp, table, held)

"""New tokens read a paged cache, against float64."""
import math

import pytest

torch = pytest.importorskip("torch")
import attention_oracle as ao   # noqa: E402
import causal_oracle as co      # noqa: E402

pytestmark = pytest.mark.gpu

BF16, F16 = torch.bfloat16, torch.float16


def make(dtype, batch, tokens, hq, hk, dim, page, lengths, counts=None, seed=0, pool="plain", width=None):
    """A cache with pages in any order; NaN in every row of the pool that holds no token of a sample."""
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    width = width or (max(lengths) + tokens + page - 1) // page
    n = batch * width + 2

    def rand(*shape):
        return torch.randn(shape, generator=gen, device="cuda").to(dtype)

    q = rand(batch, tokens, hq, dim)
    if pool == "joint":
        x = rand(n, page, hk, 2, dim)
        kp, vp = x[:, :, :, 0], x[:, :, :, 1]
    elif pool == "heads":
        kp, vp = (rand(n, hk, page, dim).transpose(1, 2) for _ in range(2))
    else:
        kp, vp = rand(n, page, hk, dim), rand(n, page, hk, dim)
    table = torch.randperm(n, generator=gen, device="cuda")[:batch * width].view(batch, width).to(torch.int32)
    held = torch.zeros((n, page), dtype=torch.bool, device="cuda")
    for b in range(batch):
        fresh = tokens if counts is None else min(max(0, int(counts[b])), tokens)
        for s in range(min(width, (lengths[b] + fresh + page - 1) // page)):
            held[table[b, s], :max(0, min(page, lengths[b] + fresh - s * page))] = True
    kp.masked_fill_(~held[:, :, None, None], math.nan)
    vp.masked_fill_(~held[:, :, None, None], math.nan)
    return q, kp, vp, table, torch.tensor(lengths, device="cuda")


def check(pkg, q, kp, vp, table, held, scale=None, **how):
    out, lse = pkg.attention.cached_attention(q, kp, vp, table, held, scale=scale, return_lse=True, **how)
    scale = scale or float(torch.tensor(1 / math.sqrt(q.shape[-1])))
    read = co.cached_read(q.shape[1], table, kp.shape[0], kp.shape[1], held, **how)
    k, v = co.gathered(kp, table), co.gathered(vp, table)
    want, want_lse, p = co.attention(q, k, v, read, scale)
    ao.within(out, want, co.bound(q, k, v, want, p, read, scale))
    ao.within(lse, want_lse, co.lse_bound(q, k, read, want_lse, scale))
    assert torch.equal(pkg.attention.cached_attention(q, kp, vp, table, held, scale=scale, **how), out)
    return out, lse


def random_tree(tokens, seed, batch=None):
    gen = torch.Generator().manual_seed(seed)

    def one():
        tree = torch.zeros((tokens, tokens), dtype=torch.bool)
        for i in range(tokens):
            parent = int(torch.randint(-1, max(1, i), (), generator=gen)) if i else -1
            if parent >= 0:
                tree[i] = tree[parent]
            tree[i, i] = True
        return tree

    return (one() if batch is None else torch.stack([one() for _ in range(batch)])).cuda()


CASES = [
    # dtype, batch, tokens, q heads, kv heads, dim, page, lengths
    (BF16, 1, 1, 1, 1, 8, 8, [0]),
    (F16, 2, 1, 2, 2, 64, 8, [0, 7]),
    (BF16, 3, 1, 32, 8, 128, 16, [1601, 15, 16]),
    (F16, 5, 1, 7, 1, 72, 32, [1, 31, 32, 33, 500]),
    (BF16, 2, 1, 16, 4, 96, 256, [255, 3000]),
    (BF16, 2, 2, 40, 2, 64, 16, [100, 130]),
    (F16, 2, 5, 4, 4, 80, 64, [0, 200]),
    (BF16, 1, 13, 8, 2, 128, 32, [900]),
    (F16, 3, 16, 12, 4, 40, 8, [3, 77, 128]),
    (BF16, 2, 25, 14, 2, 128, 64, [700, 64]),
    (BF16, 1, 64, 4, 1, 64, 128, [1000]),
    (F16, 2, 100, 3, 3, 128, 16, [127, 1]),
    (BF16, 1, 129, 8, 8, 128, 512, [383]),
    (BF16, 2, 300, 4, 2, 64, 32, [0, 500]),
    (F16, 1, 257, 7, 1, 128, 16, [640]),
    (BF16, 1, 40, 130, 1, 64, 16, [50]),
    (F16, 1, 1, 200, 1, 128, 16, [500]),
]
WINDOWS = [dict(), dict(window=1), dict(window=60, sinks=4), dict(window=300, sinks=150)]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("how", WINDOWS)
@pytest.mark.parametrize("pool", ["plain", "joint"])
def test_against_float64(pkg, case, how, pool):
    dtype, batch, tokens, hq, hk, dim, page, lengths = case
    check(pkg, *make(dtype, batch, tokens, hq, hk, dim, page, lengths, seed=tokens, pool=pool), **how)


@pytest.mark.parametrize("case", [c for c in CASES if 1 < c[2] <= 129])
@pytest.mark.parametrize("how", WINDOWS)
def test_trees(pkg, case, how):
    dtype, batch, tokens, hq, hk, dim, page, lengths = case
    made = make(dtype, batch, tokens, hq, hk, dim, page, lengths, seed=tokens, pool="heads")
    check(pkg, *made, tree=random_tree(tokens, 1, batch), **how)
    # one for all; rows that read nothing of it, or what comes behind them
    tree = random_tree(tokens, 2)
    tree[0] = False
    tree[tokens // 2] = True
    check(pkg, *made, tree=tree, **how)


@pytest.mark.parametrize("case", [c for c in CASES if c[2] > 1])
@pytest.mark.parametrize("how", WINDOWS)
def test_padded_batches(pkg, case, how):
    dtype, batch, tokens, hq, hk, dim, page, lengths = case
    counts = torch.tensor([tokens // 3, tokens + 9, 0][:batch], dtype=torch.int32, device="cuda")
    q, *rest = make(dtype, batch, tokens, hq, hk, dim, page, lengths, counts=counts)
    for b in range(batch):
        q[b, int(counts[b]):] = math.nan
    out, lse = check(pkg, q, *rest, counts=counts, **how)
    assert not out[0, tokens // 3:].any() and (lse[0, :, tokens // 3:] == -math.inf).all()
    if tokens <= 129:
        check(pkg, q, *rest, counts=counts, tree=random_tree(tokens, 3, batch), **how)


@pytest.mark.parametrize("tokens", [1, 9, 200])
@pytest.mark.parametrize("integer", [torch.int32, torch.int64])
def test_pages_that_are_none(pkg, tokens, integer):
    """Keys without a page are not read, in the middle of a tile, in a whole tile, for a whole sample; queries may have no page."""
    q, kp, vp, table, held = make(BF16, 4, tokens, 8, 2, 64, 16, [300, 300, 300, 300])
    table, held = table.to(integer), held.to(integer)
    table[0, 3], table[0, 9], table[0, -1] = -1, kp.shape[0], -5
    table[1, :18] = 2 ** 31 - 1 if integer == torch.int32 else 2 ** 40
    table[2] = -1
    for how in (dict(), dict(window=100, sinks=20), dict(tree=random_tree(tokens, 5))):
        out, lse = check(pkg, q, kp, vp, table, held, **how)
        assert not out[2].any() and (lse[2] == -math.inf).all()


@pytest.mark.parametrize("tokens", [1, 20, 150])
def test_places_behind_the_table(pkg, tokens):
    q, kp, vp, table, held = make(F16, 3, tokens, 4, 2, 128, 32, [40, 63, 64], width=2)
    check(pkg, q, kp, vp, table, held)
    big = torch.tensor([2 ** 31 - 1, 2 ** 40, 63], device="cuda")
    out, _ = pkg.attention.cached_attention(q, kp, vp, table, big, window=50, return_lse=True)
    assert not out[:2].any()                                  # far behind the table, with nothing in the window
    full = torch.tensor([64, 64, 64], device="cuda")
    a = pkg.attention.cached_attention(q, kp.nan_to_num(), vp.nan_to_num(), table, big)
    b = pkg.attention.cached_attention(q, kp.nan_to_num(), vp.nan_to_num(), table, full, counts=torch.full((3,), tokens, device="cuda"))
    assert torch.equal(a[0], b[0])                            # every place of the table is before them
    held[:] = -9
    check(pkg, q, kp.nan_to_num(), vp.nan_to_num(), table, held)


def test_shapes_without_work(pkg):
    A = pkg.attention
    q, kp, vp, table, held = make(BF16, 2, 3, 4, 2, 64, 8, [9, 3])
    assert A.cached_attention(q[:0], kp, vp, table[:0], held[:0]).shape == (0, 3, 4, 64)
    out, lse = A.cached_attention(q[:, :0], kp, vp, table, held, return_lse=True)
    assert out.shape == (2, 0, 4, 64) and lse.shape == (2, 4, 0)
    for pools, rows in (((kp[:0], vp[:0]), table), ((kp, vp), table[:, :0])):
        out, lse = A.cached_attention(q, *pools, rows, held, return_lse=True)
        assert not out.any() and (lse == -math.inf).all()


def test_long_cache(pkg):
    """More than 2^31 elements into the pool, and 70000 keys."""
    page, hk, dim, n = 64, 8, 128, 70001
    pages = 2 ** 31 // (page * hk * dim) + 1200
    kp, vp = (torch.empty((pages, page, hk, dim), dtype=BF16, device="cuda") for _ in range(2))
    kp.normal_(), vp.normal_()
    width = (n + page) // page + 1
    table = (pages - 1 - torch.randperm(width, device="cuda"))[None].to(torch.int32)
    held = torch.tensor([n], device="cuda")
    for tokens, hq in ((1, 32), (7, 16), (40, 16)):
        q = torch.randn(1, tokens, hq, dim, device="cuda").to(BF16)
        for how in (dict(), dict(window=5000, sinks=10)):
            check(pkg, q, kp, vp, table, held, **how)


def test_infinite_scores(pkg):
    q, kp, vp, table, held = make(F16, 1, 3, 2, 2, 64, 8, [150])
    kp[table[0, 2], 3, 0] = math.nan
    out, lse = pkg.attention.cached_attention(q, kp, vp, table, held, window=20, return_lse=True)
    assert torch.isfinite(out).all()                          # not in the window
    out, lse = pkg.attention.cached_attention(q, kp, vp, table, held, return_lse=True)
    assert out[0, :, 0].isnan().all() and lse[0, 0].isnan().all() and torch.isfinite(out[0, :, 1]).all()
    kp[...] = 0
    kp[..., 0] = -math.inf
    q[...] = 0
    q[..., 0] = 1
    for tokens in (1, 3):
        out, lse = pkg.attention.cached_attention(q[:, :tokens], kp, vp, table, held, return_lse=True)
        assert not out.any() and (lse == -math.inf).all()


def test_captured_and_on_another_stream(pkg):
    A = pkg.attention
    for tokens in (1, 6, 140):
        q, kp, vp, table, held = make(BF16, 2, tokens, 8, 2, 128, 16, [900, 333])
        want = A.cached_attention(q, kp, vp, table, held)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = A.cached_attention(q, kp, vp, table, held)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = A.cached_attention(q, kp, vp, table, held)
        held -= 100                                           # what a replay reads is there when it runs
        q.mul_(2)
        graph.replay()
        assert torch.equal(got, A.cached_attention(q, kp, vp, table, held))
        # two graphs, replayed in turns
        other = torch.cuda.CUDAGraph()
        with torch.cuda.graph(other, pool=graph.pool()):
            got2 = A.cached_attention(q, kp, vp, table, held, window=100)
        graph.replay(), other.replay()
        assert torch.equal(got2, A.cached_attention(q, kp, vp, table, held, window=100))
        graph.replay()
        assert torch.equal(got, A.cached_attention(q, kp, vp, table, held))


def test_refusals(pkg):
    q, kp, vp, table, held = make(BF16, 2, 3, 4, 2, 64, 8, [9, 3])

    def call(text, **change):
        a = dict(q=q, k_pages=kp, v_pages=vp, page_table=table, lengths=held)
        a.update(change)
        with pytest.raises(ValueError, match=text):
            pkg.attention.cached_attention(**a)

    tree = torch.ones(3, 3, dtype=torch.bool, device="cuda")
    call("bfloat16 or float16", q=q.float())
    call("type and device", q=q.half())
    call("must be .batch, tokens", q=q[0])
    call("multiple of kv_heads", q=q[:, :, :3])
    call("must be .pages", v_pages=vp[..., :1, :])
    call("kv_heads", k_pages=kp[0])
    call("one shape", v_pages=vp[1:])
    call("power of two", k_pages=kp[:, :7], v_pages=vp[:, :7])
    call("16 bytes", k_pages=torch.empty(kp.numel() + 8, dtype=BF16, device="cuda")[1:-7].view(kp.shape))
    call("multiples of 8", k_pages=torch.empty((*kp.shape[:3], 68), dtype=BF16, device="cuda")[..., :64])
    call("page_table must be", page_table=table[0])
    call("lengths must be", lengths=held[:1])
    call("lengths has 0 dimensions", lengths=held[0])
    call("counts must be", counts=held[:1])
    call("tree must be", tree=tree[:2])
    call("tree must be", tree=tree.float())
    call("tree must be", tree=tree.expand(3, 3, 3))
    call("no CPU path", tree=tree.cpu())
    call("window must be", window=0)
    call("window must be", window="all")
    call("sinks must not", sinks=-4)
    call("scale", scale=-1.0)
    call("q has no gradient here", q=q.clone().requires_grad_())
    call("k_pages has no gradient here", k_pages=kp.clone().requires_grad_())

"""The text's own attention, as programs that use this package run it: over a paged cache in generation, over a window in training.

Three operators: ``append`` (new keys are turned by their positions and written, with the values, into the pages of a cache;
the queries are turned on the way), ``cached`` (new tokens read the cache: single tokens, chunks of a prompt, trees of drafted
tokens, a sliding window with a few first tokens that stay visible) and ``window`` (causal attention of a sequence to itself with
such a window, forward, or forward and backward).  A case names the operator ("op"), the type of the tensors and the sizes.
What decides the amount of work (how full a cache is, how long a sequence, which tokens a drafted one follows) comes from
the case's own ``shapes`` number; values and the order of pages come from the seed.

``run`` computes the plain form: products, sums and exponentials in float32, rounded once at the end; or, where ``own`` is
true, calls the package.  ``exact`` has the same from the definitions in float64.
"""
import importlib.util
import math
import os
import random
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
POSITIONS = {"i32": torch.int32, "i64": torch.int64, "f32": torch.float32}
BLOCK = 1024   # queries that the plain form of `window` takes at once


def _attention():
    """The package directory has a hyphen in its name, so it is loaded by path."""
    if "mlx_data_b200" not in sys.modules:
        root = os.path.join(os.getcwd(), "mlx-data_b200")
        spec = importlib.util.spec_from_file_location(
            "mlx_data_b200", os.path.join(root, "__init__.py"), submodule_search_locations=[root])
        mod = importlib.util.module_from_spec(spec)
        sys.modules["mlx_data_b200"] = mod
        spec.loader.exec_module(mod)
    return sys.modules["mlx_data_b200"].attention


# ------------------------------------------------------------------ cases
def _append(dtype, batch, tokens, hq, hk, dim, page, held, sections, pos="cache", ragged=False, adjacent=False, interleaved=False, shapes=0,
            **more):
    """``held``: most tokens that a sample's cache holds already.  ``pos``: the type of the positions, or "cache": a token's place in the
    cache.  ``ragged``: samples bring different numbers of tokens.  q, k and v are views of one joint projection."""
    return dict(more, op="append", dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk, dim=dim, page=page, held=held,
                sections=sections, pos=pos, ragged=ragged, adjacent=adjacent, interleaved=interleaved, shapes=shapes)


def _cached(dtype, batch, tokens, hq, hk, dim, page, held, window=0, sinks=0, tree=False, ragged=False, shapes=0, **more):
    """``window`` 0: every token before.  ``tree``: the new tokens are drafted ones, each behind one that came earlier."""
    return dict(more, op="cached", dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk, dim=dim, page=page, held=held, window=window,
                sinks=sinks, tree=tree, ragged=ragged, shapes=shapes)


def _window(do, dtype, batch, tokens, hq, hk, dim, window=0, sinks=0, ragged=False, packed=False, shapes=0, **more):
    """``ragged``: sequences of different lengths in one padded batch.  ``packed``: q, k and v are views of one joint projection."""
    return dict(more, op="window", **{"pass": do}, dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk, dim=dim, window=window,
                sinks=sinks, ragged=ragged, packed=packed, shapes=shapes)


def listed():
    return [
        # generation, one token of one sequence joins its cache: the smallest call, latency is all
        _append("bf16", 1, 1, 32, 8, 128, 16, 1601, "16,24,24", name="append_step"),
        # drafted tokens of 24 sequences, with the positions of their tree
        _append("bf16", 24, 13, 16, 4, 128, 32, 6404, "64", pos="i64", adjacent=True, shapes=1, name="append_drafts"),
        # prompts of different lengths, text and images, float16
        _append("f16", 3, 4099, 28, 4, 128, 64, 333, "16,24,24", pos="i32", ragged=True, shapes=2, name="append_prompt"),
        # generation, one token reads its sequence
        _cached("bf16", 1, 1, 32, 8, 128, 16, 1601, name="cached_step"),
        # generation of sixteen sequences, each of another length
        _cached("bf16", 16, 1, 32, 8, 128, 16, 24000, shapes=3, name="cached_step_16"),
        # the same with a window and first tokens that stay visible, heads of 64, float16
        _cached("f16", 40, 1, 16, 4, 64, 32, 12000, window=1024, sinks=4, shapes=4, name="cached_step_window"),
        # eight sequences check a tree of drafted tokens each
        _cached("bf16", 8, 25, 32, 8, 128, 64, 8192, tree=True, shapes=5, name="cached_tree"),
        # a chunk of a prompt behind what the cache holds, grouped heads
        _cached("bf16", 1, 2048, 32, 8, 128, 64, 6404, name="cached_chunk"),
        # training, forward alone: two long texts, window and first tokens
        _window("forward", "bf16", 2, 4099, 32, 8, 128, window=1024, sinks=4, packed=True, name="window_forward"),
        # training on short captions in a padded batch, heads of 80, every token before
        _window("train", "f16", 8, 255, 12, 12, 80, ragged=True, shapes=7, name="window_train"),
        # training on one long text
        _window("train", "bf16", 1, 16384, 32, 8, 128, window=2048, sinks=4, name="window_train_long"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Any operator, type and head layout; tokens, cache, window and batch spread over the logarithm of their ranges."""
    while True:
        shapes = rng.randrange(1 << 20)
        group = rng.choice([1, 1, 2, 4, 4, 7, 8])
        hk = rng.choice([1, 2, 4, 8, 12, 16])
        hq, dim = hk * group, rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128])
        if hq > 64:
            continue
        page = rng.choice([8, 16, 16, 32, 64, 128, 256])
        window = 0 if rng.random() < 0.4 else _log_int(rng, 16, 2048)
        sinks = rng.choice([0, 1, 4, 4, 16, 130]) if window else 0
        op = rng.choice(["append", "cached", "cached", "window", "window"])
        if op == "append":
            batch = _log_int(rng, 1, 40)
            tokens = 1 if rng.random() < 0.3 else _log_int(rng, 1, 4099)
            axes = rng.choice([1, 2, 3, 4])
            pairs = dim // 2 if rng.random() < 0.7 else max(axes, dim // 4)
            cuts = sorted(rng.sample(range(1, pairs), axes - 1))
            sections = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
            case = _append(rng.choice(["bf16", "bf16", "f16", "f32"]), batch, tokens, hq, hk, dim, page, _log_int(rng, 1, 6404), sections,
                           rng.choice(["cache", "i32", "i64", "f32"]), tokens > 1 and rng.random() < 0.4, rng.random() < 0.4,
                           rng.random() < 0.3, shapes)
            if _capacity(case) * batch * hk * dim > 2 ** 29 or work(case)["bytes"] > 2.5e8:
                continue
            return case
        if op == "cached":
            batch = _log_int(rng, 1, 40)
            kind = rng.choice(["step", "step", "tree", "tree", "chunk"])
            tokens = 1 if kind == "step" else _log_int(rng, 2, 64) if kind == "tree" else _log_int(rng, 2, 2048)
            case = _cached(rng.choice(["bf16", "bf16", "f16"]), batch, tokens, hq, hk, dim, page, _log_int(rng, 1, 24000), window, sinks,
                           kind == "tree", tokens > 1 and rng.random() < 0.3, shapes)
            n = _capacity(case)
            w = work(case)
            if batch * tokens * hq * n > 6e8 or n * batch * hk * dim > 4.5e8 or w["flops"] > 2.5e11:
                continue
            return case
        batch = _log_int(rng, 1, 16)
        tokens = 1 if rng.random() < 0.05 else _log_int(rng, 2, 16384)
        case = _window(rng.choice(["forward", "train", "train"]), rng.choice(["bf16", "bf16", "f16"]), batch, tokens, hq, hk, dim, window,
                       sinks, batch > 1 and rng.random() < 0.4, rng.random() < 0.4, shapes)
        if work(case)["flops"] > 8e11 or batch * hq * tokens * tokens > 9e9 or work(case)["bytes"] < 1e3:
            continue
        return case


def _capacity(case):
    """Tokens that a row of the page table has room for."""
    return (case["held"] + case["tokens"] + case["page"] - 1) // case["page"] * case["page"]


def _lengths(case):
    """Tokens that each sample's cache holds before the call, the first sample's the most."""
    rng = random.Random(case["shapes"])
    return [case["held"]] + [rng.randint((case["held"] + 2) // 3, case["held"]) for _ in range(case["batch"] - 1)]


def _counts(case):
    """New tokens of each sample, or the length of each sequence."""
    rng = random.Random(case["shapes"] + 1)
    if not case["ragged"]:
        return [case["tokens"]] * case["batch"]
    return [rng.randint((case["tokens"] + 2) // 3, case["tokens"]) for _ in range(case["batch"])]


def _trees(case):
    """tree[b][i][j]: token i reads token j, one that it follows or itself.  A token follows one of the eight before it, or the cache."""
    rng = random.Random(case["shapes"] + 2)
    trees = []
    for _ in range(case["batch"]):
        rows = []
        for i in range(case["tokens"]):
            parent = rng.randint(max(-1, i - 8), i - 1)
            row = list(rows[parent]) if parent >= 0 else [False] * case["tokens"]
            row[i] = True
            rows.append(row)
        trees.append(rows)
    return trees


def _read(case):
    """(pairs of a query and a key that it reads, keys that some query of their sample reads), for one head, over the batch."""
    window, sinks, pairs, keys = case["window"] or 1 << 40, case["sinks"], 0, 0
    held = _lengths(case) if case["op"] == "cached" else [0] * case["batch"]
    trees = _trees(case) if case["op"] == "cached" and case["tree"] else None
    for b, (n, c) in enumerate(zip(held, _counts(case))):
        if trees:
            places = [n + sum(trees[b][i][:c]) - 1 for i in range(c)]
            near = [min(n, window - 1 - (s - n)) if window > s - n else 0 for s in places]   # of the cache, behind the window's start
            pairs += sum(max(0, x) + min(sinks, n - max(0, x)) for x in near) + sum(sum(trees[b][i][:c]) for i in range(c))
            most = max([0] + near)
            keys += most + min(sinks, n - most) + c
            continue
        # places n to n + c - 1 read min(window, place + 1) keys and the first ones that lie before these
        full = max(0, min(c, window - 1 - n))                        # queries that the window does not cut
        pairs += full * n + full * (full + 1) // 2 + (c - full) * min(window, 1 << 40)
        for i in range(full, min(c, full + sinks + 1)):
            pairs += min(sinks, n + i + 1 - window)
        pairs += max(0, c - full - sinks - 1) * sinks
        first = max(0, n + 1 - window)
        keys += (n + c - first) + min(sinks, first) if c else 0
    return pairs, keys


def work(case):
    """Every input read once, every output written once; the products of the definition."""
    item = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    hq, hk, d = case["hq"], case["hk"], case["dim"]
    new = sum(_counts(case))
    if case["op"] == "append":
        axes = len(case["sections"].split(","))
        positions = 0 if case["pos"] == "cache" else axes * case["batch"] * case["tokens"] * (8 if case["pos"] == "i64" else 4)
        turned = case["batch"] * case["tokens"] * hq * d
        return {"bytes": 2 * turned * item + 4 * new * hk * d * item + positions, "flops": 3 * (turned + new * hk * d)}
    pairs, keys = _read(case)
    if case["op"] == "cached":
        return {"bytes": 2 * new * hq * d * item + 2 * keys * hk * d * item, "flops": 4 * pairs * hq * d}
    q, kv = new * hq * d * item, new * hk * d * item
    if case["pass"] == "train":   # q, k, v, dout in; out, dq, dk, dv out
        return {"bytes": 4 * q + 4 * kv, "flops": 14 * pairs * hq * d}
    return {"bytes": 2 * q + 2 * kv, "flops": 4 * pairs * hq * d}


# ------------------------------------------------------------------ inputs
def _rand(gen, dtype, *shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _joint(gen, dtype, b, t, hq, hk, d):
    """q, k and v as a joint projection leaves them: views of [batch, tokens, hq + 2 hk, dim]."""
    x = _rand(gen, dtype, b, t, hq + 2 * hk, d)
    return x[:, :, :hq], x[:, :, hq:hq + hk], x[:, :, hq + hk:]


def _axis_of_pair(case):
    """Pairs of each axis in order, or dealt to the axes in turn as long as they have some left."""
    sections = [int(x) for x in case["sections"].split(",")]
    if not case["interleaved"]:
        return sum(([a] * n for a, n in enumerate(sections)), [])
    return [a for turn in range(max(sections)) for a, n in enumerate(sections) if turn < n]


def _positions(case, gen, lengths):
    """Of new tokens on each axis: text runs on from the cache, what is drafted for one place shares it, images have rows and columns."""
    if case["pos"] == "cache":
        return None
    axes, b, t = len(case["sections"].split(",")), case["batch"], case["tokens"]
    at = torch.arange(t, device="cuda")
    steps = torch.stack((at if axes > 1 or t > 64 else at // 3, at // 40, at % 40, at // 7))[:axes]
    start = torch.randint(0, 50, (1, b, 1), generator=gen, device="cuda") + lengths[None, :, None]
    return (start + steps[:, None]).to(POSITIONS[case["pos"]]).contiguous()


def _cache(case, gen, dtype):
    """A pool with some pages more than the samples have, theirs in any order; table entries behind a sample's last page are -1."""
    b, page, hk, d = case["batch"], case["page"], case["hk"], case["dim"]
    width = _capacity(case) // page
    pool = torch.randperm(b * width + 3, generator=gen, device="cuda")
    table = pool[:b * width].view(b, width).to(torch.int32)
    lengths = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
    counts = torch.tensor(_counts(case), dtype=torch.int32, device="cuda")
    at = torch.arange(width, device="cuda") * page
    table = torch.where(at < (lengths + counts)[:, None], table, -1).contiguous()
    k, v = (_rand(gen, dtype, len(pool), page, hk, d) for _ in range(2))
    return dict(k_pages=k, v_pages=v, page_table=table, lengths=lengths, counts=counts if case["ragged"] else None)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["dim"]
    s = dict(case=dict(case))
    if case["op"] == "window":
        if case["packed"]:
            s["q"], s["k"], s["v"] = _joint(gen, dtype, b, t, hq, hk, d)
        else:
            s["q"] = _rand(gen, dtype, b, t, hq, d, scale=2.0)
            s["k"], s["v"] = _rand(gen, dtype, b, t, hk, d), _rand(gen, dtype, b, t, hk, d)
        s["lengths"] = torch.tensor(_counts(case), dtype=torch.int32, device="cuda") if case["ragged"] else None
        if case["pass"] == "train":
            s["dout"] = _rand(gen, dtype, b, t, hq, d)
        return s
    s.update(_cache(case, gen, dtype))
    if case["op"] == "append":
        s["q"], s["k"], s["v"] = _joint(gen, dtype, b, t, hq, hk, d)
        s["positions"] = _positions(case, gen, s["lengths"])
        s["axis_of_pair"] = torch.tensor(_axis_of_pair(case), device="cuda")
        pairs = len(s["axis_of_pair"])
        s["frequencies"] = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float32) / pairs)
        s["sections"] = tuple(int(x) for x in case["sections"].split(","))
        return s
    s["q"] = _rand(gen, dtype, b, t, hq, d, scale=2.0)
    s["tree"] = torch.tensor(_trees(case), device="cuda") if case["tree"] else None
    return s


# ------------------------------------------------------------------ the passes
def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "append":
        return _plain_append(s, case)
    if case["op"] == "cached":
        return _plain_cached(s, case)
    return _plain_window(s, case)


def _run_own(s, case):
    A = _attention()
    window = case.get("window") or None
    if case["op"] == "append":
        q = A.append_rotary(s["q"], s["k"], s["v"], s["positions"], s["frequencies"], s["sections"], s["k_pages"], s["v_pages"],
                            s["page_table"], s["lengths"], counts=s["counts"], adjacent=case["adjacent"], interleaved=case["interleaved"])
        return [q, s["k_pages"], s["v_pages"]]
    if case["op"] == "cached":
        return A.cached_attention(s["q"], s["k_pages"], s["v_pages"], s["page_table"], s["lengths"], counts=s["counts"], tree=s["tree"],
                                  window=window, sinks=case["sinks"])
    how = dict(window=window, sinks=case["sinks"], lengths=s["lengths"])
    if case["pass"] == "forward":
        return A.window_attention(s["q"], s["k"], s["v"], **how)
    out, lse = A.window_attention(s["q"], s["k"], s["v"], return_lse=True, **how)
    return [out, *A.window_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **how)]


def _turn(x, cos, sin, adjacent):
    p = cos.shape[-1]
    if adjacent:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., 2 * p:]), -1)


def _places(s, case):
    """The place in its sequence of each new token [batch, tokens]."""
    return s["lengths"].long()[:, None] + torch.arange(case["tokens"], device="cuda")


def _plain_append(s, case):
    places = _places(s, case)
    positions = s["positions"] if s["positions"] is not None else places.expand(len(s["sections"]), -1, -1)
    angle = (positions.float()[s["axis_of_pair"]].movedim(0, -1) * s["frequencies"])[:, :, None]
    cos, sin = angle.cos(), angle.sin()
    q, k = (_turn(s[x].float(), cos, sin, case["adjacent"]).to(s[x].dtype) for x in ("q", "k"))
    page, row, v = s["page_table"].long().gather(1, places // case["page"]), places % case["page"], s["v"]
    if s["counts"] is not None:
        new = torch.arange(case["tokens"], device="cuda") < s["counts"][:, None]
        page, row, k, v = page[new], row[new], k[new], v[new]
    s["k_pages"][page, row] = k
    s["v_pages"][page, row] = v
    return [q, s["k_pages"], s["v_pages"]]


def _plain_cached(s, case):
    q, t, hq, hk, d = s["q"], case["tokens"], case["hq"], case["hk"], case["dim"]
    b, n, device = case["batch"], _capacity(case), s["q"].device
    held = s["lengths"].long()
    new = s["counts"].long() if s["counts"] is not None else torch.full_like(held, t)
    at = torch.arange(n, device=device)
    token = torch.arange(t, device=device)
    there = at < (held + new)[:, None]                                          # [b, n]
    places = held[:, None] + token
    if s["tree"] is not None:
        tree = s["tree"] & (token < new[:, None])[:, None, :]
        places = held[:, None] + (tree & (token[:, None] != token)).sum(-1)
        drafted = (at - held[:, None])                                          # [b, n]
        read = tree.gather(2, drafted.clamp(0, t - 1)[:, None].expand(b, t, n)) & (drafted >= 0)[:, None]
        before = (at < held[:, None])[:, None].expand(b, t, n)
    else:
        read = torch.zeros((b, t, n), dtype=torch.bool, device=device)
        before = at <= places[:, :, None]
    if case["window"]:
        before = before & ((places[:, :, None] - at < case["window"]) | (at < case["sinks"]))
    read = (read | before) & there[:, None] & (token < new[:, None])[:, :, None]   # [b, t, n]
    page = s["page_table"].long().clamp(min=0)

    def gathered(x):   # [b, hk, n, d], zeros where nothing lies
        x = x[page].flatten(1, 2).float().transpose(1, 2)
        return torch.where(there[:, None, :, None], x, 0.0)

    q32 = q.float().view(b, t, hk, hq // hk, d).permute(0, 2, 3, 1, 4).reshape(b, hk, -1, d)
    x = torch.matmul(q32, gathered(s["k_pages"]).transpose(-1, -2)).view(b, hq, t, n) * (1 / math.sqrt(d))
    x = x.masked_fill(~read[:, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total > 0, total, 1.0)
    out = torch.matmul(x.view(b, hk, -1, n), gathered(s["v_pages"]))
    return out.view(b, hq, t, d).transpose(1, 2).to(q.dtype).contiguous()


def _plain_window(s, case):
    """Some queries at a time, with the keys that their windows reach."""
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["dim"]
    group, window, sinks, train = hq // hk, case["window"] or t, case["sinks"], case["pass"] == "train"
    scale, device = 1 / math.sqrt(d), s["q"].device

    def heads(x):   # [b, hk, rows of a head by head, d]
        return x.float().view(b, -1, hk, group, d).permute(0, 2, 3, 1, 4).flatten(2, 3)

    def tokens(x):
        return x.view(b, hq, -1, d).transpose(1, 2)

    k32, v32 = s["k"].float().transpose(1, 2), s["v"].float().transpose(1, 2)
    out = torch.empty((b, t, hq, d), dtype=s["q"].dtype, device=device)
    if train:
        dq, dk, dv = torch.empty_like(out), torch.zeros_like(k32), torch.zeros_like(v32)
    for first in range(0, t, BLOCK):
        end = min(t, first + BLOCK)
        start = max(0, first + 1 - window)
        at = torch.arange(start, end, device=device)
        if start and sinks:
            at = torch.cat((torch.arange(min(sinks, start), device=device), at))
        places = torch.arange(first, end, device=device)[:, None]
        read = ((at <= places) & ((places - at < window) | (at < sinks)))[None]
        if s["lengths"] is not None:
            read = read & (places < s["lengths"][:, None, None])
        read = read[:, None, None]
        q, k, v = heads(s["q"][:, first:end].contiguous()), k32[:, :, at], v32[:, :, at]
        x = torch.matmul(q, k.transpose(-1, -2)) * scale
        x = x.view(b, hk, group, end - first, len(at)).masked_fill(~read, -math.inf)
        top = x.amax(-1, keepdim=True)
        x = (x - torch.where(top == -math.inf, 0.0, top)).exp()
        total = x.sum(-1, keepdim=True)
        x = (x / torch.where(total > 0, total, 1.0)).flatten(2, 3)
        out[:, first:end] = tokens(torch.matmul(x, v))
        if train:
            do = heads(s["dout"][:, first:end])
            dv.index_add_(2, at, torch.matmul(x.transpose(-1, -2), do))
            dp = torch.matmul(do, v.transpose(-1, -2))
            ds = x * (dp - (x * dp).sum(-1, keepdim=True))
            dq[:, first:end] = tokens(torch.matmul(ds, k) * scale)
            dk.index_add_(2, at, torch.matmul(ds.transpose(-1, -2), q) * scale)
    if not train:
        return out
    return [out, dq, dk.transpose(1, 2).to(out.dtype).contiguous(), dv.transpose(1, 2).to(out.dtype).contiguous()]


# ------------------------------------------------------------------ the definitions in float64
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(s, case)
    if case["op"] == "cached":
        return _exact_cached(s, case)
    return _exact_window(s, case)


def _exact_append(s, case):
    held = s["lengths"].tolist()
    new = s["counts"].tolist() if s["counts"] is not None else [case["tokens"]] * case["batch"]
    # the angle is the float32 product of position and frequency, by definition; a pair is a complex number that it turns
    p, page = s["frequencies"].numel(), case["page"]
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    k_pages, v_pages = s["k_pages"].double(), s["v_pages"].double()
    for b in range(case["batch"]):
        places = torch.arange(held[b], held[b] + case["tokens"], device="cuda")
        where = s["positions"][:, b] if s["positions"] is not None else torch.stack([places] * len(s["sections"]))
        angle = (where.to(torch.float32)[s["axis_of_pair"]] * s["frequencies"][:, None]).double()
        unit = torch.polar(torch.ones_like(angle), angle).T[:, None]

        def turned(x):
            head = x[..., :2 * p]
            z = torch.complex(head[..., 0::2], head[..., 1::2]) if case["adjacent"] else torch.complex(head[..., :p], head[..., p:])
            z = z * unit
            y = torch.view_as_real(z).flatten(-2) if case["adjacent"] else torch.cat((z.real, z.imag), -1)
            return torch.cat((y, x[..., 2 * p:]), -1)

        q[b] = turned(s["q"][b].double())
        if new[b]:
            slots = s["page_table"][b].long()[places[:new[b]] // page] * page + places[:new[b]] % page
            k_pages.view(-1, case["hk"], case["dim"])[slots] = turned(s["k"][b].double())[:new[b]]
            v_pages.view(-1, case["hk"], case["dim"])[slots] = s["v"][b, :new[b]].double()
    return [q, k_pages, v_pages]


def _exact_cached(s, case):
    """Sample by sample: its pages put together, what each token reads from the definition."""
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["dim"]
    held = s["lengths"].tolist()
    new = s["counts"].tolist() if s["counts"] is not None else [t] * b
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    for i in range(b):
        n, c = held[i] + new[i], new[i]
        pages = s["page_table"][i, :(n + case["page"] - 1) // case["page"]].long()
        k, v = (s[x][pages].flatten(0, 1)[:n] for x in ("k_pages", "v_pages"))
        read = torch.ones((c, n), dtype=torch.bool, device="cuda").tril(held[i])
        place = torch.arange(held[i], n, device="cuda")[:, None]
        if s["tree"] is not None:
            tree = s["tree"][i, :c, :c]
            read[:, held[i]:] = tree
            place = held[i] + (tree.sum(-1) - tree.diagonal().long())[:, None]
        if case["window"]:
            at = torch.arange(n, device="cuda")
            kept = (at > place - case["window"]) | (at < case["sinks"])
            if s["tree"] is not None:
                kept[:, held[i]:] = True
            read = read & kept
        for h in range(hk):
            heads = slice(h * (hq // hk), (h + 1) * (hq // hk))
            x = torch.einsum("tgd,nd->gtn", s["q"][i, :c, heads].double(), k[:, h].double()) / math.sqrt(d)
            x = torch.softmax(torch.where(read, x, -math.inf), -1).nan_to_num(0.0)   # a row of nothing but -infinity reads nothing
            out[i, :c, heads] = torch.einsum("gtn,nd->tgd", x, v[:, h].double())
    return out


def _exact_window(s, case):
    """Sequence by sequence and head by head, a stretch of queries with the keys that it reaches."""
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["dim"]
    window, sinks, train, step = case["window"] or t, case["sinks"], case["pass"] == "train", 2048
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk = torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    for i, n in enumerate(_counts(case)):
        for first in range(0, n, step):
            rows = torch.arange(first, min(n, first + step), device="cuda")
            keys = torch.arange(int(rows[-1]) + 1, device="cuda")
            keys = keys[(keys < sinks) | (keys > first - window)]
            hidden = (keys > rows[:, None]) | ((keys <= rows[:, None] - window) & (keys >= sinks))
            for h in range(hq):
                g = h // (hq // hk)
                q, k, v = s["q"][i, rows, h].double(), s["k"][i, keys, g].double(), s["v"][i, keys, g].double()
                w = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill(hidden, -math.inf), -1)
                o = w @ v
                out[i, rows, h] = o
                if train:
                    do = s["dout"][i, rows, h].double()
                    dv[i, keys, g] += w.T @ do
                    dx = w * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(d)
                    dq[i, rows, h] = dx @ k
                    dk[i, keys, g] += dx.T @ q
    return [out, dq, dk, dv] if train else out

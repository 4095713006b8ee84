"""Attention over the batches this package makes, as programs that use it run it.

Three operators: ``rotary`` (positions on several axes turn queries and keys), ``norm_rotary`` (RMS norm of every head of
queries and keys with the rotation in the same pass) and ``cross`` (queries read the states of images or clips, whose number
differs from theirs, and whose padding is masked).  A case names the operator ("op"), what is computed of it ("pass":
"forward", "inverse", "train" for forward and backward), the type of the tensors and the sizes.  What decides the amount of
work (lengths, sizes of grids) comes from the case's own ``shapes`` number; values come from the seed.

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
EPS = 1e-6


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
def _turned(op, do, dtype, batch, tokens, hq, hk, dim, sections, adjacent=False, interleaved=False, pos="i64", packed=False,
            weights="f32", shapes=0, **more):
    """``sections``: pairs of each axis, as text ("16,24,24"); their sum may be less than dim / 2.  ``packed``: q and k are
    views of one tensor [batch, tokens, hq + 2 hk, dim], as a joint projection leaves them."""
    return dict(more, op=op, **{"pass": do}, dtype=dtype, batch=batch, tokens=tokens, hq=hq, hk=hk, dim=dim, sections=sections,
                adjacent=adjacent, interleaved=interleaved, pos=pos, packed=packed, weights=weights, shapes=shapes)


def _cross(do, dtype, batch, tokens, keys, hq, hk, dim, fill="full", rows=0, empty=False, packed=False, shapes=0, **more):
    """``fill``: "full" (every key is read), "lengths" (a number of keys per sample; what lies behind it is whatever was in
    memory), "grid" (patches of images of different sizes in one padded batch of ``rows`` rows: a mask of keys).
    ``empty``: the last sample has no image at all."""
    return dict(more, op="cross", **{"pass": do}, dtype=dtype, batch=batch, tokens=tokens, keys=keys, hq=hq, hk=hk, dim=dim,
                fill=fill, rows=rows, empty=empty, packed=packed, shapes=shapes)


def listed():
    return [
        # generation, one token of one sequence: the smallest call, latency is all
        _turned("rotary", "forward", "bf16", 1, 1, 32, 8, 128, "16,24,24", name="rotary_step"),
        # the vision tower on a batch of 448x448 images in patches of 14, rows and columns, q and k out of a joint projection
        _turned("rotary", "forward", "bf16", 16, 1024, 16, 16, 80, "20,20", pos="i32", packed=True, name="rotary_images"),
        # the gradient of a video model in float32: 16 frames of 35x35 patches, neighbours form the pairs, part of the head turned
        _turned("rotary", "inverse", "f32", 1, 19600, 24, 24, 64, "8,10,10", adjacent=True, pos="f32", name="rotary_video_grad"),
        # generation of nine sequences at once, norm and rotation
        _turned("norm_rotary", "forward", "bf16", 9, 1, 32, 8, 128, "24,20,20", interleaved=True, name="norm_rotary_step"),
        # a prompt of text and images, grouped heads, float16
        _turned("norm_rotary", "forward", "f16", 3, 4099, 28, 4, 128, "16,24,24", weights="f16", name="norm_rotary_prompt"),
        # training: forward and backward with the gradients of both weights
        _turned("norm_rotary", "train", "bf16", 8, 2048, 16, 16, 128, "24,20,20", packed=True, name="norm_rotary_train"),
        # generation, one token reads one image of 40x40 patches and a class token
        _cross("forward", "bf16", 1, 1, 1601, 32, 8, 128, name="cross_step"),
        # generation for sixteen sequences that read up to four such images each, one of them none
        _cross("forward", "bf16", 16, 1, 6404, 32, 8, 128, fill="lengths", empty=True, shapes=3, name="cross_step_16"),
        # a prompt reads a padded batch of small images, float16, heads of 64
        _cross("forward", "f16", 6, 333, 1024, 16, 16, 64, fill="grid", rows=32, shapes=5, name="cross_prompt"),
        # a long prompt reads four large images, grouped heads
        _cross("forward", "bf16", 2, 2048, 6404, 32, 8, 128, name="cross_prompt_long"),
        # training of a caption decoder on a padded batch of 224 to 448 pixel images, heads of 80, one sample without image
        _cross("train", "f16", 8, 255, 1024, 12, 12, 80, fill="grid", rows=32, empty=True, shapes=7, name="cross_train"),
        # training on long texts and clips, grouped heads, ragged lengths
        _cross("train", "bf16", 2, 2048, 4100, 32, 8, 128, fill="lengths", shapes=9, name="cross_train_long"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """Any operator, pass, type and head layout; tokens, keys and batch spread over the logarithm of their ranges."""
    while True:
        shapes = rng.randrange(1 << 20)
        group = rng.choice([1, 1, 2, 4, 7, 8])
        hk = rng.choice([1, 2, 4, 8, 12, 16])
        hq, dim = hk * group, rng.choice([32, 64, 64, 72, 80, 96, 128, 128, 128])
        if hq > 64:
            continue
        packed = rng.random() < 0.3
        if rng.random() < 0.5:
            batch = _log_int(rng, 1, 16)
            one = rng.random() < 0.25
            tokens = 1 if one else _log_int(rng, 2, 2048)
            do = rng.choice(["forward", "forward", "train"]) if not one else "forward"
            dtype = rng.choice(["bf16", "bf16", "f16"])
            fill = rng.choice(["full", "lengths", "grid"])
            rows = rng.randint(1, 48)
            keys = _log_int(rng, 1, 6404)
            if fill == "grid":
                keys = rows * max(1, keys // rows)
            case = _cross(do, dtype, batch, tokens, keys, hq, hk, dim, fill, rows if fill == "grid" else 0,
                          fill != "full" and batch > 1 and rng.random() < 0.3, packed, shapes)
            w = work(case)
            if w["flops"] > 8.3e11 or batch * tokens * keys * hq > 8.4e8 or w["bytes"] < 1e3:
                continue
            return case
        op = rng.choice(["rotary", "norm_rotary"])
        do = rng.choice(["forward", "inverse" if op == "rotary" else "train"])
        axes = rng.choice([1, 2, 3, 3, 4])
        pairs = dim // 2 if rng.random() < 0.7 else max(axes, dim // 4)
        cuts = sorted(rng.sample(range(1, pairs), axes - 1))
        sections = ",".join(str(b - a) for a, b in zip([0] + cuts, cuts + [pairs]))
        batch = _log_int(rng, 1, 16)
        tokens = 1 if rng.random() < 0.2 else _log_int(rng, 1, 20000)
        case = _turned(op, do, rng.choice(["bf16", "bf16", "f16", "f32"]), batch, tokens, hq, hk, dim, sections, rng.random() < 0.4,
                       rng.random() < 0.3, rng.choice(["i32", "i64", "i64", "f32"]), packed,
                       rng.choice(["f32", "f32", "same"]), shapes)
        if case["weights"] == "same":
            case["weights"] = case["dtype"]
        if work(case)["bytes"] > 6.7e8:
            continue
        return case


def _lengths(case):
    """Keys that each sample reads (fill "lengths")."""
    rng = random.Random(case["shapes"])
    n = [rng.randint((case["keys"] + 2) // 3, case["keys"]) for _ in range(case["batch"])]
    return n[:-1] + [0] if case["empty"] else n


def _grids(case):
    """Rows and columns of patches that each sample's image has (fill "grid")."""
    rng = random.Random(case["shapes"])
    rows, cols = case["rows"], case["keys"] // case["rows"]
    g = [(rng.randint((rows + 1) // 2, rows), rng.randint((cols + 1) // 2, cols)) for _ in range(case["batch"])]
    return g[:-1] + [(0, 0)] if case["empty"] else g


def _read_keys(case):
    if case["fill"] == "lengths":
        return _lengths(case)
    if case["fill"] == "grid":
        return [r * c for r, c in _grids(case)]
    return [case["keys"]] * case["batch"]


def work(case):
    """Every input read once, every output written once; the products of the definition."""
    item = {"bf16": 2, "f16": 2, "f32": 4}[case["dtype"]]
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["dim"]
    if case["op"] == "cross":
        n = sum(_read_keys(case))
        q, kv = b * t * hq * d * item, 2 * n * hk * d * item
        written_kv = 2 * b * case["keys"] * hk * d * item
        if case["pass"] == "train":   # q, k, v, dout in; out, dq, dk, dv out
            return {"bytes": 4 * q + kv + written_kv, "flops": 14 * t * n * hq * d}
        return {"bytes": 2 * q + kv, "flops": 4 * t * n * hq * d}
    axes = len(case["sections"].split(","))
    values = b * t * (hq + hk) * d
    positions = axes * b * t * (8 if case["pos"] == "i64" else 4)
    if case["pass"] == "train":   # q, k in, q', k' out; q, k, their gradients in, gradients out
        return {"bytes": 5 * values * item + positions, "flops": 20 * values}
    return {"bytes": 2 * values * item + positions, "flops": (3 if case["op"] == "rotary" else 7) * values}


# ------------------------------------------------------------------ inputs
def _rand(gen, dtype, *shape, scale=1.0):
    return (torch.randn(shape, generator=gen, device="cuda") * scale).to(dtype)


def _positions(case, gen):
    """Patches of images or clips behind one another: time, row, column (and sample); a single token is far into its text."""
    axes = len(case["sections"].split(","))
    b, t = case["batch"], case["tokens"]
    start = torch.randint(0, 4000, (1, b, 1), generator=gen, device="cuda")
    if t == 1:
        p = start.expand(axes, b, 1)
    else:
        cols = max(1, int(math.sqrt(min(t, 1225))))
        at = torch.arange(t, device="cuda")
        grid = torch.stack((at // (cols * cols), at // cols % cols, at % cols, at // 7))[:axes]
        p = start + grid[:, None, :]
    return p.to(POSITIONS[case["pos"]]).contiguous()


def _axis_of_pair(case):
    """Pairs of each axis in order, or dealt to the axes in turn as long as they have some left."""
    sections = [int(x) for x in case["sections"].split(",")]
    if not case["interleaved"]:
        return sum(([a] * n for a, n in enumerate(sections)), [])
    return [a for turn in range(max(sections)) for a, n in enumerate(sections) if turn < n]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    b, t, hq, hk, d = case["batch"], case["tokens"], case["hq"], case["hk"], case["dim"]
    s = dict(case=dict(case))
    if case["op"] == "cross":
        n = case["keys"]
        s["q"] = _rand(gen, dtype, b, t, hq, d, scale=2.0)
        if case["packed"]:   # a joint projection of the encoder's states
            kv = _rand(gen, dtype, b, n, 2, hk, d)
            s["k"], s["v"] = kv[:, :, 0], kv[:, :, 1]
        else:
            s["k"], s["v"] = _rand(gen, dtype, b, n, hk, d), _rand(gen, dtype, b, n, hk, d)
        s["lengths"] = s["key_mask"] = None
        if case["fill"] == "lengths":
            s["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32, device="cuda")
            behind = torch.arange(n, device="cuda") >= s["lengths"][:, None]
            s["k"].masked_fill_(behind[:, :, None, None], math.nan)
            s["v"].masked_fill_(behind[:, :, None, None], math.nan)
        elif case["fill"] == "grid":
            grid = torch.tensor(_grids(case), device="cuda")
            at, cols = torch.arange(n, device="cuda"), n // case["rows"]
            s["key_mask"] = (at // cols < grid[:, :1]) & (at % cols < grid[:, 1:])
        if case["pass"] == "train":
            s["dout"] = _rand(gen, dtype, b, t, hq, d)
        return s
    if case["packed"]:
        qkv = _rand(gen, dtype, b, t, hq + 2 * hk, d)
        s["q"], s["k"] = qkv[:, :, :hq], qkv[:, :, hq:hq + hk]
    else:
        s["q"], s["k"] = _rand(gen, dtype, b, t, hq, d), _rand(gen, dtype, b, t, hk, d)
    s["positions"] = _positions(case, gen)
    s["axis_of_pair"] = torch.tensor(_axis_of_pair(case), device="cuda")
    pairs = len(s["axis_of_pair"])
    s["frequencies"] = 10000.0 ** (-torch.arange(pairs, device="cuda", dtype=torch.float32) / pairs)
    s["sections"] = tuple(int(x) for x in case["sections"].split(","))
    if case["op"] == "norm_rotary":
        s["q_weight"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(DTYPES[case["weights"]])
        s["k_weight"] = (1 + 0.2 * torch.randn(d, generator=gen, device="cuda")).to(DTYPES[case["weights"]])
        if case["pass"] == "train":
            s["dq"], s["dk"] = _rand(gen, dtype, b, t, hq, d), _rand(gen, dtype, b, t, hk, d)
    return s


# ------------------------------------------------------------------ the passes
def run(s):
    case = s["case"]
    if own:
        return _run_own(s, case)
    if case["op"] == "cross":
        return _plain_cross(s, case["pass"] == "train")
    if case["op"] == "rotary":
        cos, sin = _cos_sin(s)
        sin = -sin if case["pass"] == "inverse" else sin
        return [_turn(s[x].float(), cos, sin, case["adjacent"]).to(s[x].dtype) for x in ("q", "k")]
    return _plain_norm_rotary(s, case["pass"] == "train")


def _run_own(s, case):
    A = _attention()
    if case["op"] == "cross":
        masks = dict(lengths=s["lengths"], key_mask=s["key_mask"])
        if case["pass"] == "forward":
            return A.cross_attention(s["q"], s["k"], s["v"], **masks)
        out, lse = A.cross_attention(s["q"], s["k"], s["v"], return_lse=True, **masks)
        return [out, *A.cross_attention_backward(s["dout"], s["q"], s["k"], s["v"], out, lse, **masks)]
    how = dict(adjacent=case["adjacent"], interleaved=case["interleaved"])
    if case["op"] == "rotary":
        return A.rotary(s["q"], s["k"], s["positions"], s["frequencies"], s["sections"], inverse=case["pass"] == "inverse", **how)
    same = (s["positions"], s["frequencies"], s["sections"], s["q_weight"], s["k_weight"], EPS)
    out = A.qk_norm_rotary(s["q"], s["k"], *same, **how)
    if case["pass"] == "train":
        out = [*out, *A.qk_norm_rotary_backward(s["dq"], s["dk"], s["q"], s["k"], *same, **how)]
    return out


def _cos_sin(s):
    angle = (s["positions"].float()[s["axis_of_pair"]].movedim(0, -1) * s["frequencies"])[:, :, None]
    return angle.cos(), angle.sin()


def _turn(x, cos, sin, adjacent):
    p = cos.shape[-1]
    if adjacent:
        a, b = x[..., 0:2 * p:2], x[..., 1:2 * p:2]
        y = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., :p], x[..., p:2 * p]
        y = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((y, x[..., 2 * p:]), -1)


def _plain_norm_rotary(s, train):
    adjacent = s["case"]["adjacent"]
    cos, sin = _cos_sin(s)

    def forward(x, w):
        n = x.float()
        n = n * (n.square().mean(-1, keepdim=True) + EPS).rsqrt()
        return _turn(n * w.float(), cos, sin, adjacent).to(x.dtype)

    def backward(dy, x, w):
        x32 = x.float()
        r = (x32.square().mean(-1, keepdim=True) + EPS).rsqrt()
        n, g = x32 * r, _turn(dy.float(), cos, -sin, adjacent)
        gw = g * w.float()
        dx = r * (gw - n * (gw * n).mean(-1, keepdim=True))
        return dx.to(x.dtype), (g * n).sum((0, 1, 2)).to(w.dtype)

    out = [forward(s["q"], s["q_weight"]), forward(s["k"], s["k_weight"])]
    if train:
        dq, dwq = backward(s["dq"], s["q"], s["q_weight"])
        dk, dwk = backward(s["dk"], s["k"], s["k_weight"])
        out += [dq, dk, dwq, dwk]
    return out


def _plain_cross(s, train):
    q, k, v, case = s["q"], s["k"], s["v"], s["case"]
    b, t, hq, d = q.shape
    n, hk = k.shape[1:3]
    scale = 1 / math.sqrt(d)
    read = s["key_mask"]
    if s["lengths"] is not None:
        read = torch.arange(n, device=q.device) < s["lengths"][:, None]

    def by_kv_head(x):   # [b, t, hq, d] -> [b, hk, t * group, d]
        return x.float().view(b, t, hk, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, hk, -1, d)

    def by_query(x):
        return x.view(b, hk, t, hq // hk, d).permute(0, 2, 1, 3, 4).reshape(b, t, hq, d).to(q.dtype)

    q32, k32, v32 = by_kv_head(q), k.float().transpose(1, 2), v.float().transpose(1, 2)
    if read is not None:
        k32 = torch.where(read[:, None, :, None], k32, 0.0)
        v32 = torch.where(read[:, None, :, None], v32, 0.0)
    x = torch.matmul(q32, k32.transpose(-1, -2)) * scale
    if read is not None:
        x = x.masked_fill(~read[:, None, None, :], -math.inf)
    top = x.amax(-1, keepdim=True)
    x = (x - torch.where(top == -math.inf, 0.0, top)).exp()
    total = x.sum(-1, keepdim=True)
    x = x / torch.where(total > 0, total, 1.0)
    out = by_query(torch.matmul(x, v32))
    if not train:
        return out
    do = by_kv_head(s["dout"])
    dv = torch.matmul(x.transpose(-1, -2), do)
    dp = torch.matmul(do, v32.transpose(-1, -2))
    ds = x * (dp - (x * dp).sum(-1, keepdim=True))
    dq = by_query(torch.matmul(ds, k32) * scale)
    dk = torch.matmul(ds.transpose(-1, -2), q32) * scale
    return [out, dq, dk.transpose(1, 2).to(k.dtype).contiguous(), dv.transpose(1, 2).to(v.dtype).contiguous()]


# ------------------------------------------------------------------ the definitions in float64
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "cross":
        return _exact_cross(s, case)
    # the angle is the float32 product of position and frequency, by definition; a pair is a complex number that it turns
    p = s["frequencies"].numel()
    angle = (s["positions"].to(torch.float32)[s["axis_of_pair"]] * s["frequencies"][:, None, None]).double()
    unit = torch.polar(torch.ones_like(angle), angle).permute(1, 2, 0).unsqueeze(2)

    def turned(x, unit):
        head = x[..., :2 * p]
        z = torch.complex(head[..., 0::2], head[..., 1::2]) if case["adjacent"] else torch.complex(head[..., :p], head[..., p:])
        z = z * unit
        y = torch.view_as_real(z).flatten(-2) if case["adjacent"] else torch.cat((z.real, z.imag), -1)
        return torch.cat((y, x[..., 2 * p:]), -1)

    if case["op"] == "rotary":
        unit = unit.conj().resolve_conj() if case["pass"] == "inverse" else unit
        return [turned(s["q"].double(), unit), turned(s["k"].double(), unit)]
    out, grads, weights = [], [], []
    for x, w, dy in (("q", "q_weight", "dq"), ("k", "k_weight", "dk")):
        x, w = s[x].double(), s[w].double()
        rms = torch.sqrt((x * x).sum(-1, keepdim=True) / x.shape[-1] + EPS)
        out.append(turned(x / rms * w, unit))
        if case["pass"] == "train":
            g = turned(s[dy].double(), unit.conj().resolve_conj())
            weights.append((g * x / rms).flatten(0, 2).sum(0))
            along = (g * w * x).sum(-1, keepdim=True)
            grads.append(g * w / rms - x * along / (x.shape[-1] * rms ** 3))
    return out + grads + weights


def _exact_cross(s, case):
    """Sample by sample and head by head, over the keys that are read alone."""
    b, t, hq, d = s["q"].shape
    hk, train = case["hk"], case["pass"] == "train"
    out = torch.zeros((b, t, hq, d), dtype=torch.float64, device="cuda")
    dq = torch.zeros_like(out)
    dk = torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda")
    dv = torch.zeros_like(dk)
    for i in range(b):
        keys = torch.arange(case["keys"], device="cuda")
        if s["lengths"] is not None:
            keys = keys[:int(s["lengths"][i])]
        if s["key_mask"] is not None:
            keys = keys[s["key_mask"][i]]
        if not len(keys):
            continue
        for h in range(hq):
            g = h // (hq // hk)
            q, k, v = s["q"][i, :, h].double(), s["k"][i, keys, g].double(), s["v"][i, keys, g].double()
            w = torch.softmax(q @ k.T / math.sqrt(d), -1)
            o = w @ v
            out[i, :, h] = o
            if train:
                do = s["dout"][i, :, h].double()
                dv[i, keys, g] += w.T @ do
                dx = w * (do @ v.T - (do * o).sum(-1, keepdim=True)) / math.sqrt(d)
                dq[i, :, h] = dx @ k
                dk[i, keys, g] += dx.T @ q
    return [out, dq, dk, dv] if train else out

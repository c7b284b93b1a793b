"""Microscaled 4-bit linears, and per-head norms with rotary positions on
several axes: the operators, and the work their speed is judged by.

They are the steps of a block whose projections are held in 4 bits, up to its
attention:

  quant    activations or weights coded in 4-bit floating point (e2m1: 0, 0.5,
           1, 1.5, 2, 3, 4, 6 and their negatives), 32 neighbours of a row under
           one power of two, and the values that the codes stand for read back.
  product  the product of two tensors that are held so, bias added.
  linear   the linear of a weight that is held so: activations coded on the
           way, then the product.
  rope     the projection's queries and keys normed per head (root of the mean
           square, a gain per channel), turned by their positions on one axis or
           on several (time, height and width of images and video), converted,
           and appended with the values to a paged cache.

Sizes are the 768-wide block of the benchmark and generic ones: from one token
to 16384, rows of 64 to 16384 elements, heads from 64 to 256.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}

# (query heads, key / value heads, head size)
HEADS = ((12, 12, 64), (16, 16, 64), (32, 8, 128), (16, 4, 128), (28, 4, 128), (64, 8, 64),
         (20, 4, 96), (16, 8, 80), (8, 1, 256), (8, 2, 192))

PRODUCT = 8192 * 8192 * 8192  # most multiplications of a drawn case


def listed():
    return [
        # one token's activations before a projection: latency
        {"name": "quant-1x4096", "kind": "quant", "type": "bf16", "rows": 1, "cols": 4096, "pad": 0},
        # rows of a slice of a wider tensor, the last block of each not whole
        {"name": "quant-f32-3001x2000", "kind": "quant", "type": "f32", "rows": 3001, "cols": 2000, "pad": 48},
        # a large prompt's activations, or a large weight
        {"name": "quant-16384x8192", "kind": "quant", "type": "bf16", "rows": 16384, "cols": 8192, "pad": 0},
        # two tensors held in 4 bits, odd sizes
        {"name": "product-333x1000x2000", "kind": "product", "m": 333, "n": 1000, "k": 2000, "out": "f32",
         "bias": False},
        # a large product: the largest
        {"name": "product-8192", "kind": "product", "m": 8192, "n": 8192, "k": 8192, "out": "bf16", "bias": False},
        # one user's next token: the weight is read once
        {"name": "linear-1x4096x4096", "kind": "linear", "m": 1, "n": 4096, "k": 4096, "in": "bf16", "out": "bf16",
         "bias": False},
        # a decode batch over a wide layer
        {"name": "linear-32x16384x4096", "kind": "linear", "m": 32, "n": 16384, "k": 4096, "in": "bf16",
         "out": "bf16", "bias": False},
        # the benchmark's 8 x 1024 tokens through the fused projection of its 768-wide block
        {"name": "linear-8192x2304x768", "kind": "linear", "m": 8192, "n": 2304, "k": 768, "in": "f32", "out": "f32",
         "bias": True},
        # a chunk of a prompt
        {"name": "linear-2048x8192x8192", "kind": "linear", "m": 2048, "n": 8192, "k": 8192, "in": "f16",
         "out": "f16", "bias": False},
        # one decode step's tokens, normed and turned: latency
        {"name": "rope-decode-64", "kind": "rope", "in": "bf16", "out": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "rot": 128, "layout": "half", "norm": True, "sections": "64", "mixed": False, "tokens": 64, "page": 16,
         "positions": 32768},
        # the tokens of a prefill batch
        {"name": "rope-prompt-8192", "kind": "rope", "in": "bf16", "out": "bf16", "hq": 32, "hkv": 8, "d": 128,
         "rot": 128, "layout": "half", "norm": True, "sections": "64", "mixed": False, "tokens": 8192, "page": 64,
         "positions": 131072},
        # an odd number of f32 tokens of images among text: three axes, their pairs taken in turn
        {"name": "rope-axes-5001", "kind": "rope", "in": "f32", "out": "f16", "hq": 28, "hkv": 4, "d": 128,
         "rot": 128, "layout": "half", "norm": True, "sections": "24,20,20", "mixed": True, "tokens": 5001,
         "page": 48, "positions": 16384},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(("quant", "product", "linear", "linear", "linear", "rope", "rope"))
    typ = rng.choice(("bf16", "bf16", "f16", "f32"))
    if kind == "quant":
        cols = _log(rng, 64, 16384)
        rows = _log(rng, 1, min(16384, 16384 * 8192 // cols // (2 if typ == "f32" else 1)))
        return {"kind": kind, "type": typ, "rows": rows, "cols": cols, "pad": rng.choice((0, 0, 8, 33))}
    if kind in ("product", "linear"):
        n, k = _log(rng, 64, 16384), _log(rng, 64, 16384)
        if rng.random() < 0.6:  # most layers' widths are multiples of 64
            n, k = -(-n // 64) * 64, -(-k // 64) * 64
        most = max(1, min(16384, PRODUCT // (n * k)))
        m = _log(rng, 1, min(64, most)) if rng.random() < 0.5 else _log(rng, 1, most)
        case = {"kind": kind, "m": m, "n": n, "k": k, "out": typ, "bias": rng.random() < 0.3}
        if kind == "linear":
            case["in"] = rng.choice((typ, typ, "f32"))
        return case
    hq, hkv, d = rng.choice(HEADS)
    rot = rng.choice((d, d, d // 2))
    half = rot // 2
    axes = rng.choice((1, 1, 2, 3))
    cut = [half] if axes == 1 else [half - half // 2, half // 2] if axes == 2 else [half - 2 * (half // 3)] + [half // 3] * 2
    return {"kind": "rope", "in": typ, "out": rng.choice((typ, "bf16", "f16")), "hq": hq, "hkv": hkv, "d": d,
            "rot": rot, "layout": rng.choice(("half", "half", "pairs")), "norm": axes == 1 or rng.random() < 0.7,
            "sections": ",".join(map(str, cut)), "mixed": axes > 1 and rng.random() < 0.5,
            "tokens": _log(rng, 1, 16384), "page": rng.choice((16, 32, 48, 64, 128, 256)),
            "positions": _log(rng, 16384, 131072)}


def _size(name):
    return {"f32": 4, "f16": 2, "bf16": 2}[name]


def _held(rows, cols):
    """Bytes of codes and scales, as whole blocks."""
    return rows * -(-cols // 32) * 17


def work(case):
    if case["kind"] == "quant":
        rows, cols = case["rows"], case["cols"]
        return {"bytes": float(rows * cols * 2 * _size(case["type"]) + 2 * _held(rows, cols)),
                "flops": float(3 * rows * cols)}
    if case["kind"] != "rope":
        m, n, k = case["m"], case["n"], case["k"]
        a = m * k * _size(case["in"]) if case["kind"] == "linear" else _held(m, k)
        return {"bytes": float(a + _held(n, k) + m * n * _size(case["out"]) + (4 * n if case["bias"] else 0)),
                "flops": 2.0 * m * n * k}
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    axes = len(case["sections"].split(","))
    row = (hq + 2 * hkv) * d * (_size(case["in"]) + _size(case["out"])) + 4 * case["rot"] + 4 * axes + 8
    per = (4 * d if case["norm"] else 0) + 3 * case["rot"]
    return {"bytes": float(case["tokens"] * row), "flops": float(case["tokens"] * (hq + hkv) * per)}


# ---- inputs ------------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed))


def _activations(g, rows, cols, dtype):
    """Gaussian, channels of different gains, a few of them much larger than the rest."""
    gain = torch.exp(0.4 * torch.randn(cols, generator=g, device="cuda"))
    big = torch.rand(cols, generator=g, device="cuda") < 0.005
    gain = torch.where(big, gain * 12.0, gain)
    return torch.randn(rows, cols, generator=g, device="cuda").mul_(gain).to(dtype)


def _weight(g, n, k):
    """A trained layer's weight in 4 bits: codes and scales."""
    codes = torch.empty(n, -(-k // 32) * 16, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, -(-k // 32), dtype=torch.uint8, device="cuda")
    for lo in range(0, n, 4096):
        hi = min(n, lo + 4096)
        w = torch.randn(hi - lo, k, generator=g, device="cuda") * 0.02
        codes[lo:hi], scales[lo:hi] = _code(w)
    return codes, scales


def _table(positions, rot):
    """cos and sin of every position and frequency, [positions, rot / 2, 2]."""
    inv = 1000000.0 ** (-torch.arange(rot // 2, device="cuda", dtype=torch.float64) * 2.0 / rot)
    a = torch.arange(positions, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.stack([a.cos(), a.sin()], -1).float().contiguous()


def _pair_axes(case):
    """The axis of each rotated pair: the sections behind each other, or in turn
    as long as they last."""
    left = [int(x) for x in case["sections"].split(",")]
    if not case["mixed"]:
        return [a for a, n in enumerate(left) for _ in range(n)]
    out = []
    while any(left):
        for a in range(len(left)):
            if left[a]:
                out.append(a)
                left[a] -= 1
    return out


def _positions(case):
    """[axes, tokens]: text, where all axes agree, with images of 24 x 24 patches between."""
    t, axes = case["tokens"], len(case["sections"].split(","))
    at = np.arange(t)
    if axes == 1:
        first = max(0, case["positions"] - t - 1)
        return ((at + first) % case["positions"])[None].astype(np.int32)
    block, inside = at // 700, at % 700
    patch = inside - 124
    start = block * 148 + np.minimum(inside, 124)
    p = np.stack([start + np.where(patch >= 0, x, 0) for x in (0 * patch, patch // 24, patch % 24)][-axes:])
    return (p % case["positions"]).astype(np.int32)


def prepare(case, seed):
    g = _gen(seed)
    s = dict(case)
    if case["kind"] == "quant":
        rows, cols = case["rows"], case["cols"]
        s["whole"] = _activations(g, rows, cols + case["pad"], TYPES[case["type"]])
        s["x"] = s["whole"][:, :cols]
        s["codes"] = torch.empty(rows, -(-cols // 32) * 16, dtype=torch.uint8, device="cuda")
        s["scales"] = torch.empty(rows, -(-cols // 32), dtype=torch.uint8, device="cuda")
        s["values"] = torch.empty(rows, cols, dtype=TYPES[case["type"]], device="cuda")
    elif case["kind"] == "rope":
        hq, hkv, d, t, page = case["hq"], case["hkv"], case["d"], case["tokens"], case["page"]
        gain = torch.exp(0.3 * torch.randn(hq + 2 * hkv, d, generator=g, device="cuda"))
        s["x"] = torch.randn(t, hq + 2 * hkv, d, generator=g, device="cuda").mul_(gain).to(TYPES[case["in"]])
        s["q"], s["k"], s["v"] = s["x"][:, :hq], s["x"][:, hq:hq + hkv], s["x"][:, hq + hkv:]
        s["q_gain"], s["k_gain"] = (torch.exp(0.3 * torch.randn(d, generator=g, device="cuda")) for _ in range(2))
        s["eps"] = 1e-6
        pages = -(-t // page) + 3
        order = torch.randperm(pages, generator=g, device="cuda")
        at = torch.arange(t, device="cuda")
        s["slots"] = (order[at // page] * page + at % page).contiguous()
        s["axes"] = _pair_axes(case)
        s["pos"] = torch.from_numpy(_positions(case)).cuda()
        s["table"] = _table(case["positions"], case["rot"])
        for name in ("k_pool", "v_pool"):
            s[name] = torch.randn(pages, hkv, page, d, generator=g, device="cuda").to(TYPES[case["out"]])
        s["q_out"] = torch.empty(t, hq, d, dtype=TYPES[case["out"]], device="cuda")
    else:
        m, n, k = case["m"], case["n"], case["k"]
        s["w"], s["w_scales"] = _weight(g, n, k)
        s["b"] = torch.randn(n, generator=g, device="cuda") if case["bias"] else None
        s["y"] = torch.empty(m, n, dtype=TYPES[case["out"]], device="cuda")
        if case["kind"] == "linear":
            s["x"] = _activations(g, m, k, TYPES[case["in"]])
        else:
            s["a"], s["a_scales"] = _code(_activations(g, m, k, torch.float32))
    if own:
        _bind(s)
    return s


# ---- the framework's operators ------------------------------------------------

_CTX = None


def _ctx():
    """One context for the program, as its stream and workspaces are meant."""
    global _CTX
    if _CTX is None:
        from tokenvector.inference_amd import device
        _CTX = device.Context(0)
    return _CTX


def _bind(s):
    """The weight's or cache's handle, and the call that a program's loop repeats."""
    from tokenvector.inference_amd import attention as A
    from tokenvector.inference_amd import device as D
    from tokenvector.inference_amd import mxfp4 as X

    names = {"f32": A.F32, "f16": A.F16, "bf16": A.BF16}
    ctx = _ctx()
    torch.cuda.synchronize()
    if s["kind"] == "quant":
        x, v, t = s["x"], s["values"], names[s["type"]]
        s["calls"] = (X.Quantize(ctx, t, x.data_ptr(), x.stride(0), s["rows"], s["cols"], s["codes"].data_ptr(),
                                 s["scales"].data_ptr()),
                      X.Dequantize(ctx, s["codes"].data_ptr(), s["scales"].data_ptr(), s["rows"], s["cols"], t,
                                   v.data_ptr(), v.stride(0)))
    elif s["kind"] == "product":
        s["calls"] = (X.Matmul(ctx, s["a"].data_ptr(), s["a_scales"].data_ptr(), s["w"].data_ptr(),
                               s["w_scales"].data_ptr(), s["m"], s["n"], s["k"], names[s["out"]], s["y"].data_ptr(),
                               s["n"], bias=s["b"].data_ptr() if s["bias"] else None),)
    elif s["kind"] == "linear":
        s["layer"] = D.QuantizedLinear.from_mxfp4(ctx, s["w"].data_ptr(), s["w_scales"].data_ptr(), s["n"], s["k"],
                                                  s["b"].data_ptr() if s["bias"] else None)
        s["calls"] = (X.Linear(ctx, s["layer"], names[s["in"]], s["x"].data_ptr(), s["k"], s["m"], names[s["out"]],
                               s["y"].data_ptr(), s["n"]),)
    else:
        def rows(x):
            return A.Rows(x.data_ptr(), x.stride(0), x.stride(1))

        hkv, d = s["hkv"], s["d"]
        s["cache"] = A.KVCache(ctx, names[s["out"]], s["k_pool"].shape[0], s["page"], hkv, d,
                               s["k_pool"].data_ptr(), s["v_pool"].data_ptr())
        norm = A.HeadNorm(s["eps"], s["q_gain"].data_ptr(), s["k_gain"].data_ptr()) if s["norm"] else None
        rope = A.Rope(s["table"].data_ptr(), s["table"].shape[0], s["rot"],
                      A.ROPE_HALF if s["layout"] == "half" else A.ROPE_PAIRS, s["pos"].data_ptr(),
                      axes=s["pos"].shape[0], stride_axis=s["pos"].stride(0), pair_axis=s["axes"])
        s["calls"] = (A.NormRopeAppend(ctx, names[s["in"]], s["tokens"], s["hq"], hkv, d, rows(s["q"]), rows(s["k"]),
                                       rows(s["v"]), norm=norm, rope=rope, q_out=rows(s["q_out"]),
                                       type_out=names[s["out"]], cache=s["cache"], slots=s["slots"].data_ptr()),)


def _out(s):
    if s["kind"] == "quant":
        return s["values"]
    return {"q": s["q_out"], "k": s["k_pool"], "v": s["v_pool"]} if s["kind"] == "rope" else s["y"]


# ---- the plain forms -------------------------------------------------------------

def _code(x):
    """Codes, two a byte and the even column's low, and scales: the exponent of a
    block's largest magnitude less 2, biased by 127."""
    x = x.float()
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % 32)).view(rows, -1, 32)
    top = torch.frexp(x.abs().amax(-1))[1] - 3
    top = top.clamp_(-127, 127)
    y = torch.ldexp(x, -top[..., None])
    a = y.abs()
    c = (a > 0.25).to(torch.uint8)
    for edge, whole in ((0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True), (5.0, False)):
        c += (a >= edge) if whole else (a > edge)
    c |= (y < 0).to(torch.uint8) << 3
    c = c.view(rows, -1, 2)
    return c[..., 0] | c[..., 1] << 4, (top + 127).to(torch.uint8)


def _values(codes, scales, cols):
    """What they stand for, f32 [rows, cols]."""
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    grid = torch.cat([grid, -grid])
    v = grid[torch.stack([codes & 15, codes >> 4], -1).long()].view(codes.shape[0], -1, 32)
    v *= torch.exp2(scales.float() - 127.0)[..., None]
    return v.view(codes.shape[0], -1)[:, :cols]


def _product(a, w, s):
    y = torch.matmul(a, w.t())
    if s["b"] is not None:
        y += s["b"]
    return s["y"].copy_(y)


def _turned(x, gain, s):
    x = x.float()
    if s["norm"]:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * gain
    rot = s["rot"]
    pair = torch.arange(rot // 2, device=x.device)
    axis = torch.tensor(s["axes"], device=x.device)
    cs = s["table"][s["pos"].long()[axis].t(), pair][:, None]
    c, n = cs[..., 0], cs[..., 1]
    if s["layout"] == "half":
        a, b = x[..., :rot // 2], x[..., rot // 2:rot]
        y = torch.cat([a * c - b * n, b * c + a * n], -1)
    else:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2)
    return torch.cat([y, x[..., rot:]], -1)


def run(state):
    s = state
    if own:
        for call in s["calls"]:
            call()
        return _out(s)
    if s["kind"] == "quant":
        s["values"].copy_(_values(*_code(s["x"]), s["cols"]))
    elif s["kind"] == "product":
        _product(_values(s["a"], s["a_scales"], s["k"]), _values(s["w"], s["w_scales"], s["k"]), s)
    elif s["kind"] == "linear":
        _product(_values(*_code(s["x"]), s["k"]), _values(s["w"], s["w_scales"], s["k"]), s)
    else:
        at, slot = s["slots"] // s["page"], s["slots"] % s["page"]
        s["q_out"].copy_(_turned(s["q"], s["q_gain"], s))
        s["k_pool"][at, :, slot] = _turned(s["k"], s["k_gain"], s).to(s["k_pool"].dtype)
        s["v_pool"][at, :, slot] = s["v"].float().to(s["v_pool"].dtype)
    return _out(s)


# ---- the definitions in 64 bits -----------------------------------------------------

def _nearest(x):
    """The values that x's codes stand for: each to the nearest multiple of its
    binade's step, ties to the even one, the largest magnitude 6."""
    x = x.double()
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, -cols % 32)).view(rows, -1, 32)
    top = x.abs().amax(-1, keepdim=True)
    unit = torch.pow(2.0, torch.floor(torch.log2(top.clamp_min(2.0 ** -125))) - 2.0)
    y = x / unit
    step = torch.pow(2.0, torch.floor(torch.log2(y.abs().clamp(1.0, 4.0))) - 1.0)
    y = (torch.round(y / step) * step).clamp_(-6.0, 6.0)
    return (y * unit).view(rows, -1)[:, :cols]


def _stood_for(codes, scales, cols):
    """Sign, exponent and mantissa bits of each code, taken apart."""
    c = torch.stack([codes & 15, codes >> 4], -1).view(codes.shape[0], -1).double()
    sign = 1.0 - 2.0 * torch.floor(c / 8.0)
    c = c - 8.0 * torch.floor(c / 8.0)
    e, man = torch.floor(c / 2.0), c - 2.0 * torch.floor(c / 2.0)
    v = torch.where(e > 0, (1.0 + man / 2.0) * torch.pow(2.0, e - 1.0), man / 2.0)
    unit = torch.pow(2.0, scales.double() - 127.0).repeat_interleave(32, 1)
    return (sign * v * unit)[:, :cols]


def _exact_turned(x, gain, s):
    x = x.double()
    if s["norm"]:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + s["eps"]) * gain.double()
    else:
        x = x.clone()
    r = s["rot"]
    first = slice(0, r // 2) if s["layout"] == "half" else slice(0, r, 2)
    second = slice(r // 2, r) if s["layout"] == "half" else slice(1, r, 2)
    table = torch.view_as_complex(s["table"].double())
    turn = torch.stack([table[s["pos"][a].long(), i] for i, a in enumerate(s["axes"])], -1)
    z = torch.complex(x[..., first], x[..., second]) * turn[:, None]
    x[..., first], x[..., second] = z.real, z.imag
    return x


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if s["kind"] == "quant":
        return _nearest(s["x"])
    if s["kind"] == "rope":
        out = {"q": _exact_turned(s["q"], s["q_gain"], s)}
        rows = {"k": _exact_turned(s["k"], s["k_gain"], s), "v": s["v"].double()}
        for name, x in rows.items():
            pool = s[name + "_pool"].double()
            flat = pool.transpose(1, 2).reshape(-1, s["hkv"], s["d"])
            flat[s["slots"]] = x
            out[name] = flat.view(-1, s["page"], s["hkv"], s["d"]).transpose(1, 2).contiguous()
        return out
    a = _nearest(s["x"]) if s["kind"] == "linear" else _stood_for(s["a"], s["a_scales"], s["k"])
    out = torch.empty(s["m"], s["n"], dtype=torch.float64, device="cuda")
    for lo in range(0, s["n"], 4096):
        hi = min(s["n"], lo + 4096)
        out[:, lo:hi] = a @ _stood_for(s["w"][lo:hi], s["w_scales"][lo:hi], s["k"]).t().contiguous()
    return out if s["b"] is None else out + s["b"].double()

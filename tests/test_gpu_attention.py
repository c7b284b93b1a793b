"""GPU tests of the attention operators (tokenvector.inference_amd.attention)
against plain numpy forms.

Rotation, conversion and append: bit for bit against the same f32 operations.
Attention: against the formula in 64 bits, within a bound per output element
derived from the roundings of the computation (see _bound): the logits' f32
dot product, exp2 and its argument, the f32 sums, for 16-bit types the weights'
rounding to the type, and the output's rounding.  What a row does not see is
filled with NaN and infinities, rows that see nothing have to be zeros, and rows
that no sequence covers have to stay as they were.
"""
import sys

import numpy as np
import pytest
import torch

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D

pytestmark = pytest.mark.gpu

TORCH = {A.F32: torch.float32, A.F16: torch.float16, A.BF16: torch.bfloat16}
ROUND = {A.F32: 2.0 ** -24, A.F16: 2.0 ** -11, A.BF16: 2.0 ** -8}
NAME = {A.F32: "f32", A.F16: "f16", A.BF16: "bf16", A.I8: "i8"}
POISON = np.array([np.nan, np.inf, -np.inf], np.float32)


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


def _bytes(x, typ):
    """f32 values rounded to the type, as raw integers of its width."""
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[typ])
    return t.view(torch.int32 if typ == A.F32 else torch.int16).numpy()


def _values(raw, typ):
    return torch.from_numpy(np.ascontiguousarray(raw)).view(TORCH[typ]).float().numpy()


def _round(x, typ):
    return _values(_bytes(x, typ), typ)


def _dev(ctx, a):
    return D.DeviceBuffer.from_host(ctx, a)


def _i32(ctx, a):
    return _dev(ctx, np.asarray(a, np.int32))


def _seen(n, t, causal, window):
    pos = np.arange(t - n, t)[:, None]
    j = np.arange(t)[None, :]
    m = np.ones((n, t), bool)
    if causal:
        m &= j <= pos
    if window:
        m &= j > pos - window
    return m


def _exact(q, k, v, mask, scale):
    """One head in 64 bits: out, and per row max |logit| (of absolute products)
    and the weighted |v| that the error bound scales with."""
    q, k, v = (x.astype(np.float64) for x in (q, k, v))
    some = mask.any(1)
    k0 = np.where(mask.any(0)[:, None], k, 0.0)
    v0 = np.where(mask.any(0)[:, None], v, 0.0)
    a = np.where(mask, scale * (q @ k0.T), -np.inf)
    top = np.where(some, a.max(1, initial=-np.inf), 0.0)
    w = np.where(mask, np.exp(a - top[:, None]), 0.0)
    total = np.where(some, w.sum(1), 1.0)[:, None]
    size = np.where(mask, scale * (np.abs(q) @ np.abs(k0).T), 0.0).max(1, initial=0.0)[:, None]
    return w @ v0 / total, size, w @ np.abs(v0) / total, np.abs(v0).max(initial=0.0) / total


def _bound(typ, typ_out, d, t, ref, size, spread, vmax):
    e = 2.0 ** -24
    # logit: d products and sums, the scale and the int8 scale; the weight's
    # argument is rounded twice more, exp2 is good to 2 ulp; sums of t terms,
    # rescaled with every running maximum (at most one per 16 keys)
    rel = 2.0 * (d + 8) * e * size + (t + t / 4 + 32) * e
    out = rel * spread
    if typ != A.F32:
        out = out + ROUND[typ] * spread * (1 + rel)        # the weights' rounding
    if typ == A.F16:
        out = out + t * 2.0 ** -25 * vmax                  # weights below f16's normal range
    out = out + ROUND[typ_out] * np.abs(ref) * (1 + rel)
    if typ_out == A.F16:
        out = out + 2.0 ** -25
    return 1.05 * out + 1e-30


def _check(got, q, k, v, mask, scale, typ, typ_out, what):
    """q, k, v, got [n or t, heads, d] of one sequence."""
    n, hq, d = q.shape
    g = hq // max(1, k.shape[1])
    for h in range(hq):
        ref, size, spread, vmax = _exact(q[:, h], k[:, h // g], v[:, h // g], mask, scale)
        bound = _bound(typ, typ_out, d, k.shape[0], ref, size, spread, vmax)
        err = np.abs(got[:, h] - ref)
        assert np.all(np.isfinite(got[:, h])), f"{what}: head {h} has values that are not finite"
        worst = np.max(err / bound, initial=0.0)
        assert worst <= 1.0, f"{what}: head {h} off by {worst:.3g} of its bound"
        assert not got[~mask.any(1), h].any(), f"{what}: a row that sees nothing is not zero"


def _fused(r, tokens, hq, hkv, d, typ, pad=0):
    """A fused projection's rows, `pad` elements between them."""
    x = r.standard_normal((tokens, (hq + 2 * hkv) * d + pad)).astype(np.float32)
    return _round(x, typ)


class Prompt:
    """Packed sequences of lens_q queries and lens_k keys; rows before, between
    and after belong to nobody."""

    def __init__(self, ctx, typ, hq, hkv, d, lens_q, lens_k=None, causal=True, window=0, typ_out=None,
                 shift=0, seed=1, spare=3, scale=None):
        r = np.random.default_rng(seed)
        self.same = lens_k is None
        lens_k = lens_q if self.same else lens_k
        self.typ, self.typ_out = typ, typ if typ_out is None else typ_out
        self.hq, self.hkv, self.d, self.causal, self.window = hq, hkv, d, causal, window
        self.scale = 1.0 / np.sqrt(d) if scale is None else scale
        self.cu_q = np.concatenate([[0], np.cumsum(lens_q)]) + (0 if self.same else spare)
        self.cu_k = self.cu_q if self.same else np.concatenate([[0], np.cumsum(lens_k)])
        tq, tk = int(self.cu_q[-1]) + spare, int(self.cu_k[-1]) + spare
        row = (hq + 2 * hkv) * d
        rows = max(tq, tk)
        self.x = _fused(r, rows, hq, hkv, d, typ)
        if self.same:
            # rows past the last sequence are nobody's: they may hold anything
            self.x[int(self.cu_k[-1]):] = POISON[0]
        # rows stay 16-byte aligned for shift 0
        flat = np.zeros(rows * row + shift, np.float32)
        flat[shift:] = self.x.reshape(-1)
        self.xd = _dev(ctx, _bytes(flat, typ))
        w = 4 if typ == A.F32 else 2
        base = self.xd.ptr + shift * w
        self.out0 = np.full((tq, hq, d), 7.25, np.float32)
        self.od = _dev(ctx, _bytes(self.out0, self.typ_out))
        self.cq, self.ck = _i32(ctx, self.cu_q), None if self.same else _i32(ctx, self.cu_k)
        self.call = A.AttentionPrompt(
            ctx, typ, tq, hq, hkv, d, len(lens_q), A.Rows(base, row, d),
            A.Rows(base + hq * d * w, row, d), A.Rows(base + (hq + hkv) * d * w, row, d),
            A.Rows(self.od, hq * d, d), self.cq, self.ck, tk, self.scale, causal, window, self.typ_out)

    def result(self):
        return _values(self.od.download(), self.typ_out).reshape(self.out0.shape)

    def check(self, what):
        got = self.result()
        hq, hkv, d = self.hq, self.hkv, self.d
        x = self.x.reshape(self.x.shape[0], hq + 2 * hkv, d)
        covered = np.zeros(got.shape[0], bool)
        for s in range(len(self.cu_q) - 1):
            q0, q1, k0, k1 = self.cu_q[s], self.cu_q[s + 1], self.cu_k[s], self.cu_k[s + 1]
            covered[q0:q1] = True
            mask = _seen(q1 - q0, k1 - k0, self.causal, self.window)
            _check(got[q0:q1], x[q0:q1, :hq], x[k0:k1, hq:hq + hkv], x[k0:k1, hq + hkv:], mask,
                   self.scale, self.typ, self.typ_out, f"{what}, sequence {s}")
        assert np.array_equal(got[~covered], self.out0[~covered]), f"{what}: wrote uncovered rows"


PROMPTS = [
    # heads, head size, lengths
    (2, 2, 64, [1]),
    (4, 1, 128, [0, 1, 2, 0, 3]),
    (3, 3, 64, [64, 65, 63]),
    (8, 2, 128, [130, 1, 257, 31]),
    (2, 1, 80, [200, 33]),
    (4, 4, 96, [97, 95]),
    (4, 2, 256, [129, 66]),
    (5, 1, 192, [70, 150]),
    (25, 25, 64, [40]),
    (2, 2, 8, [100, 3]),
    (6, 2, 40, [90, 17]),
]


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("hq,hkv,d,lens", PROMPTS)
def test_prompt(ctx, typ, hq, hkv, d, lens):
    say(f"prompt {NAME[typ]} heads {hq}/{hkv} of {d}, lengths {lens}")
    p = Prompt(ctx, typ, hq, hkv, d, lens)
    p.call()
    p.check("prompt")


@pytest.mark.parametrize("typ", [A.BF16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("causal,window", [(False, 0), (True, 1), (True, 33), (True, 100), (False, 50)])
def test_prompt_masks(ctx, typ, causal, window):
    say(f"prompt masks {NAME[typ]} causal {causal} window {window}")
    p = Prompt(ctx, typ, 4, 2, 64, [150, 7, 300], causal=causal, window=window)
    p.call()
    p.check("prompt masks")


@pytest.mark.parametrize("typ", [A.BF16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("causal", [True, False])
def test_prompt_more_queries_than_keys(ctx, typ, causal):
    """Positions count from the keys' end: early rows see nothing; a sequence
    without keys gives zeros."""
    p = Prompt(ctx, typ, 4, 2, 64, [100, 5, 40, 70], [40, 0, 300, 70], causal=causal)
    p.call()
    p.check("more queries than keys")


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("d,shift", [(33, 0), (20, 0), (1, 0), (64, 1), (128, 4)])
def test_prompt_any_layout(ctx, typ, d, shift):
    """Head sizes and addresses that are not multiples of 16 bytes."""
    p = Prompt(ctx, typ, 4, 2, d, [50, 3, 70], shift=shift)
    p.call()
    p.check(f"head size {d}, {shift} elements off")


@pytest.mark.parametrize("typ", [A.BF16, A.F16], ids=lambda t: NAME[t])
def test_prompt_f32_output(ctx, typ):
    p = Prompt(ctx, typ, 4, 2, 128, [150, 9], typ_out=A.F32)
    p.call()
    p.check("f32 output")


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
def test_prompt_long(ctx, typ):
    p = Prompt(ctx, typ, 2, 1, 64, [1500, 700], scale=0.4)
    p.call()
    p.check("long")
    first = p.od.download()
    p.call()
    assert np.array_equal(first, p.od.download()), "two runs differ"


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("at", [0, 70, 128, 199])
def test_prompt_poisoned_key_touches_only_rows_that_see_it(ctx, typ, at):
    """A key and value of NaN and infinities: rows before it are finite and right,
    rows from it on are not finite, as the formula has it."""
    d, n = 64, 200
    p = Prompt(ctx, typ, 2, 2, d, [n])
    x = p.x.reshape(-1, 6, d)
    x[at, 2:] = np.resize(POISON, (4, d))
    p.xd.upload(_bytes(p.x.reshape(-1), typ))
    p.call()
    got = p.result()
    mask = _seen(n, n, True, 0)[:at]
    _check(got[:at], x[:at, :2], np.where(np.isfinite(x[:n, 2:4]), x[:n, 2:4], 0), np.where(
        np.isfinite(x[:n, 4:]), x[:n, 4:], 0), mask, p.scale, typ, typ, "before the poisoned key")
    assert not np.isfinite(got[at:n]).any()


@pytest.mark.parametrize("typ", [A.BF16, A.F32], ids=lambda t: NAME[t])
def test_prompt_infinite_value_behind_a_finite_key(ctx, typ):
    """An infinity in one value element reaches that element of the rows that see
    it, as an infinity, and nothing else."""
    d, n, at = 64, 300, 100
    p = Prompt(ctx, typ, 1, 1, d, [n])
    x = p.x.reshape(-1, 3, d)
    x[at, 2, 5] = np.inf
    p.xd.upload(_bytes(p.x.reshape(-1), typ))
    p.call()
    got = p.result()
    assert np.all(got[at:n, 0, 5] == np.inf)
    v = x[:n, 2:].copy()
    v[at, 0, 5] = 0.0
    got[at:n, 0, 5] = 0.0
    ref = np.delete(np.arange(d), 5)
    mask = _seen(n, n, True, 0)
    whole = _exact(x[:n, 0], x[:n, 1], v[:, 0], mask, p.scale)
    bound = _bound(typ, typ, d, n, *whole)
    assert np.all(np.abs(got[:n, 0] - whole[0])[:, ref] <= bound[:, ref])
    assert np.all(np.abs(got[:at, 0] - whole[0][:at]) <= bound[:at])


@pytest.mark.parametrize("typ", [A.BF16, A.F16], ids=lambda t: NAME[t])
@pytest.mark.parametrize("d", [104, 128])
def test_prompt_many_short_sequences(ctx, typ, d):
    """Hundreds of tiles: the kernel with 32 keys a tile."""
    r = np.random.default_rng(8)
    lens = r.integers(0, 12, 200).tolist() + [70, 33, 200]
    p = Prompt(ctx, typ, 8, 4, d, lens)
    p.call()
    p.check("many short sequences")


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
def test_prompt_scale_zero_and_infinite_logits(ctx, typ):
    """Equal weights at scale 0; a key whose logits are -inf has no weight; rows that
    see nothing else are zeros."""
    p = Prompt(ctx, typ, 2, 2, 64, [90], scale=0.0)
    p.call()
    p.check("scale zero")
    p = Prompt(ctx, typ, 1, 1, 64, [90])
    x = p.x.reshape(-1, 3, 64)
    x[:90, 0] = np.abs(x[:90, 0]) + 0.5              # queries all positive
    x[0, 1] = -np.inf
    x[5, 1] = -np.inf
    p.xd.upload(_bytes(p.x.reshape(-1), typ))
    p.call()
    got = p.result()[:90]
    assert not got[0].any(), "the first row's only logit is -inf"
    mask = _seen(90, 90, True, 0)
    mask[:, [0, 5]] = False
    k = np.where(np.isfinite(x[:90, 1:2]), x[:90, 1:2], 0)
    _check(got[1:], x[1:90, :1], k, x[:90, 2:], mask[1:], p.scale, typ, typ, "keys of -inf logits")


# ---- the paged cache --------------------------------------------------------------

class Paged:
    """Sequences of `new` tokens over caches of `total` (the new ones among them).
    Unused slots of the pool hold NaN and infinities."""

    def __init__(self, ctx, typ, cache, hq, hkv, d, new, total, page=16, causal=True, window=0,
                 typ_out=None, seed=2, bounds=True, width=None, decode=None, scale=None):
        r = np.random.default_rng(seed)
        self.typ, self.typ_out, self.cache = typ, typ if typ_out is None else typ_out, cache
        self.hq, self.hkv, self.d, self.causal, self.window = hq, hkv, d, causal, window
        self.new, self.total, self.page = list(new), list(total), page
        self.scale = 1.0 / np.sqrt(d) if scale is None else scale
        seqs = len(new)
        need = [-(-t // page) for t in total]
        pages = sum(need) + 2
        order = r.permutation(pages)
        width = max(max(need), 1) if width is None else width
        table = np.full((seqs, width), -1, np.int64)  # unused entries are no page at all
        shape = (pages, hkv, page, d)
        if cache == A.I8:
            kp = r.integers(-127, 128, shape).astype(np.int8)
            vp = r.integers(-127, 128, shape).astype(np.int8)
            self.ks = np.resize(POISON, shape[:3]).copy()
            self.vs = np.resize(POISON, shape[:3]).copy()
        else:
            kp, vp = np.resize(POISON, shape).copy(), np.resize(POISON, shape).copy()
        self.kv, at = [], 0
        for s in range(seqs):
            table[s, :need[s]] = order[at:at + need[s]]
            at += need[s]
            k = np.empty((total[s], hkv, d), np.float32)
            v = np.empty_like(k)
            for j in range(total[s]):
                pg, slot = table[s, j // page], j % page
                if cache == A.I8:
                    self.ks[pg, :, slot] = r.uniform(0.005, 0.02, hkv)
                    self.vs[pg, :, slot] = r.uniform(0.005, 0.02, hkv)
                    k[j] = kp[pg, :, slot] * self.ks[pg, :, slot][:, None].astype(np.float64)
                    v[j] = vp[pg, :, slot] * self.vs[pg, :, slot][:, None].astype(np.float64)
                else:
                    k[j] = _round(r.standard_normal((hkv, d)), typ)
                    v[j] = _round(r.standard_normal((hkv, d)), typ)
                    kp[pg, :, slot], vp[pg, :, slot] = k[j], v[j]
            self.kv.append((k, v))
        tokens = sum(new)
        self.q = _round(r.standard_normal((tokens, hq, d)), typ)
        self.out0 = np.full((tokens, hq, d), 7.25, np.float32)
        raw = (lambda x: x) if cache == A.I8 else (lambda x: _bytes(x, typ))
        self.bufs = [_dev(ctx, raw(kp)), _dev(ctx, raw(vp))]
        sc = [None, None]
        if cache == A.I8:
            sc = [_dev(ctx, self.ks), _dev(ctx, self.vs)]
        self.pool = A.KVCache(ctx, cache, pages, page, hkv, d, *self.bufs, *sc)
        self.qd, self.od = _dev(ctx, _bytes(self.q, typ)), _dev(ctx, _bytes(self.out0, self.typ_out))
        self.lens, self.tab = _i32(ctx, total), _i32(ctx, table)
        decode = all(n == 1 for n in new) if decode is None else decode
        self.cu = None if decode else _i32(ctx, np.concatenate([[0], np.cumsum(new)]))
        self.call = A.AttentionPaged(
            ctx, typ, tokens, hq, self.pool, seqs, A.Rows(self.qd, hq * d, d), A.Rows(self.od, hq * d, d),
            self.tab, width, self.lens, self.cu, max(new) if bounds else 0, max(total) if bounds else 0,
            self.scale, causal, window, self.typ_out)

    def result(self):
        return _values(self.od.download(), self.typ_out).reshape(self.out0.shape)

    def check(self, what):
        got, at = self.result(), 0
        for s, (n, t) in enumerate(zip(self.new, self.total)):
            k, v = self.kv[s]
            _check(got[at:at + n], self.q[at:at + n], k, v, _seen(n, t, self.causal, self.window),
                   self.scale, self.typ, self.typ_out, f"{what}, sequence {s}")
            at += n


LAYOUTS = [(2, 2, 64), (8, 2, 128), (4, 1, 128), (3, 3, 80), (5, 1, 96), (16, 2, 64), (4, 2, 192),
           (8, 1, 256), (2, 2, 16), (20, 1, 64), (4, 2, 72), (33, 1, 64), (40, 1, 128)]
TYPES = [(A.BF16, A.BF16), (A.F16, A.F16), (A.F32, A.F32), (A.BF16, A.I8), (A.F16, A.I8), (A.F32, A.I8)]
TYPE_IDS = [f"{NAME[a]}-{NAME[b]}" for a, b in TYPES]


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hq,hkv,d", LAYOUTS)
def test_decode(ctx, typ, cache, hq, hkv, d):
    total = [1, 2, 15, 16, 17, 63, 64, 65, 130, 300]
    say(f"decode {NAME[typ]} over {NAME[cache]} heads {hq}/{hkv} of {d}")
    p = Paged(ctx, typ, cache, hq, hkv, d, [1] * len(total), total)
    p.call()
    p.check("decode")


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("page", [1, 7, 48, 256])
def test_decode_pages(ctx, typ, cache, page):
    p = Paged(ctx, typ, cache, 4, 2, 64, [1, 1, 1], [1000, 129, 777], page=page, window=0)
    p.call()
    p.check(f"pages of {page}")


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("window", [1, 40, 513])
def test_decode_window(ctx, typ, cache, window):
    p = Paged(ctx, typ, cache, 8, 2, 128, [1, 1, 1], [1200, 20, 513], window=window)
    p.call()
    p.check(f"window {window}")


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
def test_decode_long(ctx, typ, cache):
    """One sequence: its keys are split over many workgroups, and joined in the same
    order in every run."""
    p = Paged(ctx, typ, cache, 8, 2, 128, [1], [6007], page=64, scale=0.3)
    p.call()
    p.check("long decode")
    first = p.od.download()
    for _ in range(3):
        p.call()
        assert np.array_equal(first, p.od.download()), "two runs differ"


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("hq,hkv,d", [(4, 2, 64), (8, 2, 128), (3, 3, 80), (8, 1, 256)])
def test_chunks(ctx, typ, cache, hq, hkv, d):
    new, total = [3, 0, 1, 17, 64, 130, 5], [3, 10, 40, 17, 200, 331, 600]
    say(f"chunks {NAME[typ]} over {NAME[cache]} heads {hq}/{hkv} of {d}")
    p = Paged(ctx, typ, cache, hq, hkv, d, new, total, page=32)
    p.call()
    p.check("chunks")


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,total", [([300], [2500]), ([9, 2], [1500, 3000]), ([33], [4000])])
def test_chunk_long(ctx, typ, cache, new, total):
    p = Paged(ctx, typ, cache, 4, 1, 64, new, total, page=48, window=0)
    p.call()
    p.check("long chunk")
    first = p.od.download()
    p.call()
    assert np.array_equal(first, p.od.download()), "two runs differ"


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,total", [([5], [20000]), ([17, 6], [20000, 9000])])
def test_chunk_over_many_splits(ctx, typ, cache, new, total):
    """Over 16 (and over 64) splits of the keys, joined in two levels."""
    p = Paged(ctx, typ, cache, 8, 1, 64, new, total, page=256)
    p.call()
    p.check("chunk of many splits")
    first = p.od.download()
    p.call()
    assert np.array_equal(first, p.od.download()), "two runs differ"


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F32, A.F32), (A.F16, A.I8)])
@pytest.mark.parametrize("causal,window", [(True, 64), (False, 0)])
def test_chunk_masks(ctx, typ, cache, causal, window):
    p = Paged(ctx, typ, cache, 4, 2, 64, [40, 100, 2], [400, 100, 90], causal=causal, window=window)
    p.call()
    p.check("chunk masks")


class Poisoned(Paged):
    """A windowed cache whose tokens before the earliest query's window hold NaN and
    infinities (int8: such scales)."""

    def __init__(self, ctx, typ, cache, hq, hkv, d, new, total, page, window):
        super().__init__(ctx, typ, cache, hq, hkv, d, new, total, page=page, window=window)
        kp, vp = (b.download() for b in self.bufs)
        raw = _bytes(POISON, typ) if cache != A.I8 else None
        tab = self.tab.download()
        for s, (n, t) in enumerate(zip(new, total)):
            for j in range(max(0, t - n + 1 - window)):
                pg, slot = tab[s, j // page], j % page
                if cache == A.I8:
                    self.ks[pg, :, slot] = self.vs[pg, :, slot] = POISON[j % 3]
                else:
                    kp[pg, :, slot] = vp[pg, :, slot] = raw[j % 3]
        if cache == A.I8:
            self.pool._kept[2].upload(self.ks)
            self.pool._kept[3].upload(self.vs)
        else:
            self.bufs[0].upload(kp)
            self.bufs[1].upload(vp)


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("new,total,window", [([1, 1], [700, 90], 37), ([1], [6000], 3000), ([40, 3], [300, 500], 21),
                                              ([150], [5000], 2900)])
def test_window_hides_what_is_not_finite(ctx, typ, cache, new, total, window):
    p = Poisoned(ctx, typ, cache, 4, 2, 64, new, total, 16, window)
    p.call()
    p.check("poison before the window")


@pytest.mark.parametrize("typ,cache", TYPES, ids=TYPE_IDS)
@pytest.mark.parametrize("total", [60, 5000])
def test_chunk_hides_later_keys_that_are_not_finite(ctx, typ, cache, total):
    """The last new token's key and value are poison: the rows before it do not see it."""
    for new in (2, 50):
        p = Paged(ctx, typ, cache, 4, 2, 64, [new], [total], page=16)
        tab, j = p.tab.download(), total - 1
        pg, slot = tab[0, j // 16], j % 16
        if cache == A.I8:
            p.ks[pg, :, slot] = p.vs[pg, :, slot] = np.inf
            p.pool._kept[2].upload(p.ks)
            p.pool._kept[3].upload(p.vs)
        else:
            for b in p.bufs:
                x = b.download()
                x[pg, :, slot] = _bytes(POISON[1:2], typ)[0]
                b.upload(x)
        p.call()
        got = p.result()
        k, v = p.kv[0]
        mask = _seen(new, total, True, 0)[:-1]
        _check(got[:-1], p.q[:-1], k, v, mask, p.scale, typ, typ, "rows before the poisoned key")
        assert not np.isfinite(got[-1]).any()


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("lo,hi", [(1e-7, 1e-5), (1e-6, 4.0), (0.0, 0.01)])
@pytest.mark.parametrize("new", [1, 60])
def test_int8_scales_of_any_size(ctx, typ, lo, hi, new):
    p = Paged(ctx, typ, A.I8, 4, 2, 64, [new], [400], page=16)
    r = np.random.default_rng(4)
    tab = p.tab.download()
    k, v = p.kv[0]
    codes = p.bufs[1].download()
    for j in range(400):
        pg, slot = tab[0, j // 16], j % 16
        s = (np.exp(r.uniform(np.log(max(lo, 1e-7)), np.log(hi), 2)) * (lo > 0 or j % 3 > 0)).astype(np.float32)
        p.vs[pg, :, slot] = s
        v[j] = codes[pg, :, slot] * s[:, None].astype(np.float64)
    p.pool._kept[3].upload(p.vs)
    p.call()
    p.check(f"scales {lo} to {hi}")


def test_paged_uncovered_rows_stay(ctx):
    """Query rows before the first sequence and after the last are nobody's."""
    p = Paged(ctx, A.BF16, A.BF16, 4, 2, 64, [5, 40, 6], [100, 200, 30])
    p.cu.upload(np.array([5, 45, 45, 45], np.int32))
    p.lens.upload(np.array([200, 0, 0], np.int32))
    tab = p.tab.download()
    tab[0] = tab[1]
    p.tab.upload(tab)
    p.call()
    got = p.result()
    assert np.array_equal(got[:5], p.out0[:5]) and np.array_equal(got[45:], p.out0[45:])
    k, v = p.kv[1]
    _check(got[5:45], p.q[5:45], k, v, _seen(40, 200, True, 0), p.scale, A.BF16, A.BF16, "covered rows")


def test_paged_many_chunks(ctx):
    """Hundreds of tiles over a cache."""
    r = np.random.default_rng(9)
    new = r.integers(9, 30, 160).tolist()
    total = [n + int(x) for n, x in zip(new, r.integers(0, 60, 160))]
    p = Paged(ctx, A.BF16, A.BF16, 16, 4, 128, new, total, page=8)
    p.call()
    p.check("many chunks")


def test_on_another_stream(ctx):
    """A context on the caller's stream: inputs written there just before the call."""
    p = Paged(ctx, A.BF16, A.BF16, 4, 2, 64, [1, 1], [900, 50])
    p.call()
    want = p.od.download()
    q = torch.from_numpy(p.qd.download().copy()).cuda()
    out = torch.empty_like(q)
    stream = torch.cuda.Stream()
    torch.cuda.synchronize()
    _lib.check(_lib.lib().tkv_hip_ctx_set_stream(ctx.handle, stream.cuda_stream))
    try:
        call = A.AttentionPaged(ctx, A.BF16, 2, 4, p.pool, 2, A.Rows(out.data_ptr() , 256, 64),
                                A.Rows(out.data_ptr(), 256, 64), p.tab, p.tab.shape[1], p.lens, None, 1, 900,
                                p.scale)
        with torch.cuda.stream(stream):
            for _ in range(3):
                out.copy_(q)
                call()                               # in place: each row is read before it is written
        stream.synchronize()
        assert np.array_equal(out.cpu().numpy().reshape(want.shape), want)
    finally:
        _lib.check(_lib.lib().tkv_hip_ctx_set_stream(ctx.handle, None))


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F32, A.F32), (A.BF16, A.I8)])
def test_paged_rows_that_see_nothing(ctx, typ, cache):
    """An empty cache, and more new tokens than the cache holds."""
    p = Paged(ctx, typ, cache, 4, 2, 64, [1, 1], [0, 5])
    p.call()
    p.check("empty cache, one token")
    p = Paged(ctx, typ, cache, 4, 2, 64, [8, 50, 3], [0, 20, 3])
    p.call()
    p.check("more new tokens than keys")


@pytest.mark.parametrize("bounds", [True, False])
@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F32, A.I8)])
def test_paged_without_bounds(ctx, typ, cache, bounds):
    """max_q and max_kv choose the launch alone."""
    p = Paged(ctx, typ, cache, 4, 1, 128, [1, 70, 2], [900, 100, 3], bounds=bounds, decode=False)
    p.call()
    p.check("bounds" if bounds else "no bounds")


def test_paged_bounds_that_are_too_small(ctx):
    """Longer sequences than max_q and max_kv say are still right."""
    p = Paged(ctx, A.BF16, A.BF16, 4, 1, 128, [1, 70, 2], [900, 100, 3])
    call = A.AttentionPaged(ctx, A.BF16, 73, 4, p.pool, 3, A.Rows(p.qd, 512, 128), A.Rows(p.od, 512, 128),
                            p.tab, p.tab.shape[1], p.lens, p.cu, 1, 1, p.scale)
    call()
    p.check("small bounds")


@pytest.mark.parametrize("d", [20, 33])
@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F32, A.F32), (A.F16, A.I8)])
def test_paged_any_layout(ctx, typ, cache, d):
    p = Paged(ctx, typ, cache, 4, 2, d, [1, 5], [100, 30])
    p.call()
    p.check(f"head size {d}")


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F16, A.I8)])
def test_paged_f32_output(ctx, typ, cache):
    for new in ([1, 1], [1, 40]):
        p = Paged(ctx, typ, cache, 4, 2, 128, new, [3000, 77], typ_out=A.F32)
        p.call()
        p.check("f32 output")


def test_paged_clamps_lengths_and_pages(ctx):
    """Lengths beyond the table end with it; page ids outside the pool read page 0."""
    p = Paged(ctx, A.F32, A.F32, 2, 2, 64, [1, 1], [32, 32], page=16)
    kp = np.zeros((6, 2, 16, 64), np.float32) + 1.0
    p.bufs[0].upload(kp[:p.pool.num_pages])
    p.bufs[1].upload(kp[:p.pool.num_pages])
    p.lens.upload(np.array([10 ** 6, 2 ** 31 - 1], np.int32))
    p.tab.upload(np.array([[0, 1 << 30], [-5, 1]], np.int32))
    p.call()
    # equal keys, values of one: the weights sum to one within their roundings
    assert np.all(np.abs(p.result() - 1.0) <= 64 * 2.0 ** -24)


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.BF16, A.I8)])
@pytest.mark.parametrize("new,total", [([1, 1], [3000, 50]), ([100, 3], [800, 2000])])
def test_paged_graph(ctx, typ, cache, new, total):
    """Captured once, replayed on lengths that change, checked against eager calls."""
    p = Paged(ctx, typ, cache, 8, 2, 64, new, total, page=32)
    p.call()
    want = {}
    for k, lens in enumerate((total, [total[0] - 7, total[1]], [total[0], total[1] - 3])):
        p.lens.upload(np.array(lens, np.int32))
        p.call()
        want[k] = (lens, p.od.download())
    with D.Graph(ctx) as g:
        p.call()
    for _ in range(2):
        for lens, out in want.values():
            p.lens.upload(np.array(lens, np.int32))
            p.od.upload(_bytes(p.out0, p.typ_out))
            g.launch()
            assert np.array_equal(p.od.download(), out)
    g.close()


def test_offsets_beyond_32_bits(ctx):
    """A pool whose last pages begin past 2^32 elements and bytes."""
    heads, page, d = 8, 256, 128
    pages = (1 << 32) // (heads * page * d) + 3
    pool = A.KVCache(ctx, A.BF16, pages, page, heads, d)
    r = np.random.default_rng(5)
    total = 2 * page
    k = _round(r.standard_normal((total, heads, d)), A.BF16)
    v = _round(r.standard_normal((total, heads, d)), A.BF16)
    x = np.concatenate([k, v], 1)
    xd = _dev(ctx, _bytes(x, A.BF16))
    table = np.array([[pages - 1, pages - 2]], np.int32)
    slots = (table[0][:, None].astype(np.int64) * page + np.arange(page)).reshape(-1)
    sd, td, ld = _dev(ctx, slots), _i32(ctx, table), _i32(ctx, [total])
    A.RopeAppend(ctx, A.BF16, total, 0, heads, d, None, A.Rows(xd, 2 * heads * d, d),
                 A.Rows(xd.ptr + heads * d * 2, 2 * heads * d, d), cache=pool, slots=sd)()
    for n in (1, 200):
        q = _round(r.standard_normal((n, heads, d)), A.BF16)
        qd, od = _dev(ctx, _bytes(q, A.BF16)), _dev(ctx, _bytes(np.zeros_like(q), A.BF16))
        cu = _i32(ctx, [0, n])
        A.AttentionPaged(ctx, A.BF16, n, heads, pool, 1, A.Rows(qd, heads * d, d),
                         A.Rows(od, heads * d, d), td, 2, ld, cu, n, total)()
        got = _values(od.download(), A.BF16).reshape(q.shape)
        _check(got, q, k, v, _seen(n, total, True, 0), 1 / np.sqrt(d), A.BF16, A.BF16, "far pages")
    pool.close()


# ---- rotation and append -------------------------------------------------------------

def _rotated(x, table, positions, rot, layout):
    """The same f32 operations, one rounding each."""
    y = x.copy()
    if rot:
        cs = table[positions][:, None]
        c, s = cs[..., 0], cs[..., 1]
        a = slice(0, rot // 2) if layout == A.ROPE_HALF else slice(0, rot, 2)
        b = slice(rot // 2, rot) if layout == A.ROPE_HALF else slice(1, rot, 2)
        y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


ROPES = [
    # heads, head size, rotated elements, tokens
    (12, 12, 64, 0, 5),
    (12, 12, 64, 64, 1),
    (8, 2, 128, 128, 33),
    (4, 1, 96, 48, 7),
    (4, 2, 80, 80, 9),
    (3, 1, 80, 20, 9),
    (2, 1, 256, 256, 3),
    (5, 5, 33, 10, 4),
    (1, 1, 2, 2, 300),
]


@pytest.mark.parametrize("layout", [A.ROPE_HALF, A.ROPE_PAIRS], ids=["half", "pairs"])
@pytest.mark.parametrize("tin,tout,cache", [(A.F32, A.BF16, A.BF16), (A.F32, A.F32, A.F32), (A.BF16, A.BF16, A.I8),
                                            (A.F32, A.F16, A.I8), (A.F16, A.F16, A.F16), (A.BF16, A.F32, A.F32)],
                         ids=lambda t: NAME[t])
@pytest.mark.parametrize("hq,hkv,d,rot,tokens", ROPES)
def test_rope_append(ctx, tin, tout, cache, layout, hq, hkv, d, rot, tokens):
    r = np.random.default_rng(d + rot)
    positions_held, page = 5000, 12
    x = _round(r.standard_normal((tokens, hq + 2 * hkv, d)) * 2, tin)
    x[0, -1] = 0.0                                  # a row of zeros has the least scale
    inv = A.rope_inv_freq(rot, 10000.0) if rot else None
    table = A.rope_table(ctx, positions_held, inv) if rot else None
    pos = r.integers(0, positions_held, tokens).astype(np.int32)
    pages = -(-tokens // page) + 2
    slots = r.permutation(pages * page)[:tokens].astype(np.int64)
    if tokens > 3:
        pos[2] = -1                                  # padding: zeros, nothing appended
        slots[1] = -1                                # no slot
        slots[3] = pages * page                      # outside the pool
    xd, pd, sd = _dev(ctx, _bytes(x, tin)), _i32(ctx, pos), _dev(ctx, slots)
    w, row = (4 if tin == A.F32 else 2), (hq + 2 * hkv) * d
    rows = [A.Rows(xd.ptr + o * d * w, row, d) for o in (0, hq, hq + hkv)]
    old = np.full((pages, hkv, page, d), 3, np.int8 if cache == A.I8 else np.float32)
    raw = (lambda v: v) if cache == A.I8 else (lambda v: _bytes(v, cache))
    kb, vb = _dev(ctx, raw(old)), _dev(ctx, raw(old))
    sc = [_dev(ctx, np.full((pages, hkv, page), 9.0, np.float32)) for _ in range(2)] if cache == A.I8 else [None] * 2
    pool = A.KVCache(ctx, cache, pages, page, hkv, d, kb, vb, *sc)
    qo = _dev(ctx, _bytes(np.full((tokens, hq, d), 5.0), tout))
    ko = _dev(ctx, _bytes(np.full((tokens, hkv, d), 5.0), tout))
    A.RopeAppend(ctx, tin, tokens, hq, hkv, d, *rows, pd, table, positions_held, rot, layout,
                 A.Rows(qo, hq * d, d), A.Rows(ko, hkv * d, d), tout, pool, sd)()
    tab = table.download() if rot else None
    real = (pos >= 0) if rot else np.ones(tokens, bool)
    turned = _rotated(x[:, :hq + hkv], tab, np.where(real, pos, 0), rot, layout)
    turned[~real] = 0.0
    assert np.array_equal(qo.download().reshape(tokens, hq, d), _bytes(turned[:, :hq], tout))
    assert np.array_equal(ko.download().reshape(tokens, hkv, d), _bytes(turned[:, hq:], tout))
    put = real & (slots >= 0) & (slots < pages * page)
    at, slot = slots[put] // page, slots[put] % page
    for buf, scales, y in ((kb, sc[0], turned[put, hq:]), (vb, sc[1], x[put, hq + hkv:])):
        want = old.copy()
        if cache == A.I8:
            scale = np.maximum(np.abs(y).max(-1), np.float32(1e-8)) * (np.float32(1) / np.float32(127))
            inv_s = np.float32(1) / scale
            want[at, :, slot] = np.clip(np.rint(y * inv_s[..., None]), -127, 127).astype(np.int8)
            ws = np.full((pages, hkv, page), 9.0, np.float32)
            ws[at, :, slot] = scale
            assert np.array_equal(scales.download(), ws)
            assert np.array_equal(buf.download().reshape(want.shape), want)
        else:
            want[at, :, slot] = y
            assert np.array_equal(buf.download().reshape(want.shape), raw(want))


def test_rope_in_place_and_without_a_cache(ctx):
    r = np.random.default_rng(3)
    x = _round(r.standard_normal((50, 6, 64)), A.BF16)
    xd, pos = _dev(ctx, _bytes(x, A.BF16)), np.arange(50, dtype=np.int32) * 7
    table, pd = A.rope_table(ctx, 400, A.rope_inv_freq(64)), _i32(ctx, pos)
    q, k = A.Rows(xd, 6 * 64, 64), A.Rows(xd.ptr + 4 * 64 * 2, 6 * 64, 64)
    A.RopeAppend(ctx, A.BF16, 50, 4, 1, 64, q, k, None, pd, table, 400, 64, A.ROPE_HALF, q, k)()
    want = x.copy()
    want[:, :5] = _rotated(x[:, :5], table.download(), pos, 64, A.ROPE_HALF)
    assert np.array_equal(xd.download().reshape(50, 6, 64), _bytes(want, A.BF16))


@pytest.mark.parametrize("kw", [{}, {"factor": 4.0}, {"base": 500000.0}, {"factor": 8.0, "by_parts": True,
                                                                         "original_positions": 4096}])
def test_rope_table(ctx, kw):
    """f64 angles: within an f32 rounding (and f64 differences) at far positions."""
    inv = A.rope_inv_freq(64, **kw)
    n, amplitude = 140000, 1.25
    got = A.rope_table(ctx, n, inv, amplitude).download()
    p = np.r_[0:40, n - 40:n]
    a = p[:, None].astype(np.float64) * inv
    want = np.stack([np.cos(a), np.sin(a)], -1) * amplitude
    assert np.all(np.abs(got[p] - want) <= amplitude * (2.0 ** -24 + 1e-9))


def test_zero_sizes(ctx):
    z, cu = _dev(ctx, np.zeros(64, np.float32)), _i32(ctx, [0, 0])
    rows = A.Rows(z, 64, 64)
    A.AttentionPrompt(ctx, A.F32, 0, 1, 1, 64, 1, rows, rows, rows, rows, cu)()
    pool = A.KVCache(ctx, A.F32, 1, 16, 1, 64)
    A.AttentionPaged(ctx, A.F32, 0, 1, pool, 0, rows, rows, cu, 1, cu)()
    A.RopeAppend(ctx, A.F32, 0, 1, 1, 64, rows, rows, rows, cache=pool, slots=cu)()
    out = _dev(ctx, np.full(64, 3.0, np.float32))
    # no pages at all: the row sees nothing
    A.AttentionPaged(ctx, A.F32, 1, 1, pool, 1, rows, A.Rows(out, 64, 64), None, 0, _i32(ctx, [9]))()
    assert not out.download().any()


def test_refusals(ctx):
    z, cu = _dev(ctx, np.zeros(256, np.float32)), _i32(ctx, [0, 1])
    rows = A.Rows(z, 64, 64)
    pool = A.KVCache(ctx, A.BF16, 1, 16, 1, 64)

    def refused(call, *a, **k):
        with pytest.raises(ValueError):
            call(*a, **k)()

    refused(A.AttentionPrompt, ctx, A.I8, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 3, 2, 64, 1, rows, rows, rows, rows, cu)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 1, 1, 257, 1, rows, rows, rows, rows, cu)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 1, 1, 64, 1, rows, rows, rows, rows, None)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu, window=-1)
    refused(A.AttentionPrompt, ctx, A.F16, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu, type_out=A.BF16)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu, scale=-1.0)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 1, 1, 64, 1, rows, rows, rows, rows, cu, scale=float("nan"))
    refused(A.AttentionPrompt, ctx, A.F32, -1, 1, 1, 64, 1, rows, rows, rows, rows, cu)
    refused(A.AttentionPrompt, ctx, A.F32, 1, 1, 1, 64, 1, A.Rows(None, 64, 64), rows, rows, rows, cu)
    refused(A.AttentionPaged, ctx, A.F16, 1, 1, pool, 1, rows, rows, cu, 1, cu)      # the cache is bf16
    refused(A.AttentionPaged, ctx, A.BF16, 2, 1, pool, 1, rows, rows, cu, 1, cu)     # two rows, no cu_q
    refused(A.AttentionPaged, ctx, A.BF16, 1, 1, pool, 1, rows, rows, None, 1, cu)
    refused(A.AttentionPaged, ctx, A.BF16, 1, 1, pool, 1, rows, rows, cu, 1, None)
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 2, 64, rows, rows, rows, cache=pool, slots=cu)  # other heads
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 1, 64, rows, rows, rows, cache=pool)            # no slots
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 1, 64, rows, rows, None, cache=pool, slots=cu)  # no values
    refused(A.RopeAppend, ctx, A.F16, 1, 1, 1, 64, rows, rows, rows, cache=pool, slots=cu)   # type
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 1, 64, rows, rows, rows, cu, z, 2, 63)          # odd rot_dim
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 1, 64, rows, rows, rows, cu, z, 2, 128)
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 1, 64, rows, rows, rows, None, z, 2, 64)        # no positions
    refused(A.RopeAppend, ctx, A.BF16, 1, 1, 1, 64, rows, rows, rows, cu, z, 2, 64, 7)       # layout
    for bad in ((A.F32, 0, 16, 1, 64), (A.F32, 1, 0, 1, 64), (A.F32, 1, 16, 1, 300), (9, 1, 16, 1, 64),
                (A.F32, 1 << 20, 1 << 12, 1, 64)):
        with pytest.raises(ValueError):
            A.KVCache(ctx, *bad)
    with pytest.raises(ValueError):
        A.KVCache(ctx, A.I8, 1, 16, 1, 64, z, z)      # int8 pools without scales
    with pytest.raises(ValueError):
        A.rope_table(ctx, 4, np.ones(200))
    with pytest.raises(ValueError):
        _lib.check(_lib.lib().tkv_hip_dev_attention_paged(ctx.handle, A.BF16, 1, 1, 0, 1, None, None,
                                                          A.BF16, None, 0, None, None, 0, 0, 1.0, 1, 0))


def test_paged_refuses_tables_without_bound(ctx):
    """A row of 2^31 page ids: its keys would pass the kernels' 32-bit key numbers."""
    z, cu = _dev(ctx, np.zeros(256, np.float32)), _i32(ctx, [0, 1])
    rows = A.Rows(z, 64, 64)
    pool = A.KVCache(ctx, A.F32, 1, 16, 1, 64)
    for stride in (-1, 1 << 31, 1 << 62):
        with pytest.raises(ValueError):
            A.AttentionPaged(ctx, A.F32, 1, 1, pool, 1, rows, rows, cu, stride, cu)()


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F32, A.I8)])
def test_paged_bounds_beyond_every_size(ctx, typ, cache):
    """max_q and max_kv of 2^62 are bounds as well."""
    p = Paged(ctx, typ, cache, 4, 1, 128, [1, 30, 2], [300, 100, 3])
    call = A.AttentionPaged(ctx, typ, 33, 4, p.pool, 3, A.Rows(p.qd, 512, 128), A.Rows(p.od, 512, 128),
                            p.tab, p.tab.shape[1], p.lens, p.cu, 1 << 62, 1 << 62, p.scale)
    call()
    p.check("bounds beyond every size")


@pytest.mark.parametrize("typ", [A.BF16, A.F32], ids=lambda t: NAME[t])
def test_prompt_largest_scale(ctx, typ):
    """Keys of zero have logits of zero at any finite scale: equal weights."""
    p = Prompt(ctx, typ, 2, 2, 64, [70], scale=float(np.finfo(np.float32).max))
    x = p.x.reshape(-1, 6, 64)
    x[:, 2:4] = 0
    p.xd.upload(_bytes(p.x.reshape(-1), typ))
    p.call()
    got = p.result()[:70]
    _check(got, x[:70, :2], x[:70, 2:4], x[:70, 4:], _seen(70, 70, True, 0), 0.0, typ, typ, "largest scale")

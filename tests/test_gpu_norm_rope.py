"""GPU tests of norms per head with the rotation on one axis or several and the
append to a cache (attention.NormRopeAppend), against numpy.

Without norms: bit for bit the f32 operations of the rotation.  With norms:
against the formula in 64 bits.  The sum of d squares, the mean, eps, root and
quotient are off by at most (d / 2 + 4) 2^-24 of the inverse norm, the two
products with it and the gain by 2 2^-24 more, the rotation's products and sum by
2 2^-24 of the magnitudes added; then one rounding to the type.  int8 codes are
half a step off at most, of a scale that follows the row's largest value.
"""
import ctypes as C
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


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


def _bytes(x, typ):
    t = torch.from_numpy(np.ascontiguousarray(x, np.float32)).to(TORCH[typ])
    return t.view(torch.int32 if typ == A.F32 else torch.int16).numpy()


def _values(raw, typ):
    return torch.from_numpy(np.ascontiguousarray(raw)).view(TORCH[typ]).float().numpy()


def _round(x, typ):
    return _values(_bytes(x, typ), typ)


def _dev(ctx, a):
    return D.DeviceBuffer.from_host(ctx, a)


class Setting:
    """Rows of a fused projection, positions, a pool whose slots keep what they
    held, outputs; and the call."""

    def __init__(self, ctx, tin, tout, cache, layout, hq, hkv, d, rot, tokens, sections=None, mixed=False, eps=1e-6,
                 gains=True, norm=True, pad=0, seed=0, amplitude=2.0):
        r = np.random.default_rng(seed + d + rot + tokens)
        self.__dict__.update(locals())
        self.page, self.held = 12, 3000
        width = (hq + 2 * hkv) * d + pad
        host = _round(r.standard_normal((tokens, width)) * amplitude, tin)
        self.x = host[:, :width - pad].reshape(tokens, hq + 2 * hkv, d)
        self.x[0, 0] = 0.0  # a head of zeros: its norm is sqrt(eps)
        self.axes = 1 if not sections else len(sections)
        self.pairs = np.array(A.rope_pair_axes(sections, mixed) if sections else [0] * (rot // 2))
        self.pos = r.integers(0, self.held, (self.axes, tokens)).astype(np.int32)
        self.pages = -(-tokens // self.page) + 2
        self.slots = r.permutation(self.pages * self.page)[:tokens].astype(np.int64)
        if tokens > 6:
            if rot:
                self.pos[0, 2] = -1                           # padding
                self.pos[self.axes - 1, 4] = self.held        # on the last axis
            self.slots[1], self.slots[3] = -1, self.pages * self.page
        full = host.copy()
        full[:, :width - pad] = self.x.reshape(tokens, -1)
        self.xd = _dev(ctx, _bytes(full, tin))
        w = 4 if tin == A.F32 else 2
        rows = [A.Rows(self.xd.ptr + o * d * w, width, d) for o in (0, hq, hq + hkv)]
        self.table = A.rope_table(ctx, self.held, A.rope_inv_freq(rot)) if rot else None
        # positions of each axis with others between them
        self.pd = _dev(ctx, np.concatenate([self.pos, np.full((self.axes, 5), -7, np.int32)], 1))
        self.old = np.full((self.pages, hkv, self.page, d), 3, np.int8 if cache == A.I8 else np.float32)
        raw = (lambda v: v) if cache == A.I8 else (lambda v: _bytes(v, cache))
        self.kb, self.vb = _dev(ctx, raw(self.old)), _dev(ctx, raw(self.old))
        self.sc = [_dev(ctx, np.full((self.pages, hkv, self.page), 9.0, np.float32)) if cache == A.I8 else None
                   for _ in range(2)]
        self.pool = A.KVCache(ctx, cache, self.pages, self.page, hkv, d, self.kb, self.vb, *self.sc)
        self.qo = _dev(ctx, _bytes(np.full((tokens, hq, d), 5.0), tout))
        self.ko = _dev(ctx, _bytes(np.full((tokens, hkv, d), 5.0), tout))
        self.g = [r.uniform(0.5, 1.5, d).astype(np.float32) if gains else np.ones(d, np.float32) for _ in range(2)]
        self.gd = [_dev(ctx, g) if gains else None for g in self.g]
        self.call = A.NormRopeAppend(
            ctx, tin, tokens, hq, hkv, d, *rows, norm=A.HeadNorm(eps, *self.gd) if norm else None,
            rope=A.Rope(self.table, self.held, rot, layout, self.pd, self.axes, tokens + 5,
                        self.pairs.tolist() if self.axes > 1 else None) if rot else None,
            q_out=A.Rows(self.qo, hq * d, d), k_out=A.Rows(self.ko, hkv * d, d), type_out=tout, cache=self.pool,
            slots=_dev(ctx, self.slots))

    def expected(self, dtype):
        """The rows of q and k turned, and the magnitudes that their errors go by."""
        x, d, hq = self.x[:, :self.hq + self.hkv].astype(dtype), self.d, self.hq
        if self.norm:
            x = x / np.sqrt((x * x).mean(-1, keepdims=True) + dtype(np.float32(self.eps)))
            x = np.concatenate([x[:, :hq] * self.g[0].astype(dtype), x[:, hq:] * self.g[1].astype(dtype)], 1)
        size = np.abs(x)
        real = np.ones(self.tokens, bool)
        if self.rot:
            real = ((self.pos >= 0) & (self.pos < self.held)).all(0)
            tab = self.table.download().astype(dtype)
            at = np.where(real, self.pos, 0)[self.pairs]                     # [pairs, tokens]
            cs = tab[at, np.arange(self.rot // 2)[:, None]].transpose(1, 0, 2)[:, None]
            c, s = cs[..., 0], cs[..., 1]
            if self.layout == A.ROPE_HALF:
                first, second = slice(0, self.rot // 2), slice(self.rot // 2, self.rot)
            else:
                first, second = slice(0, self.rot, 2), slice(1, self.rot, 2)
            a, b = x[..., first].copy(), x[..., second].copy()
            x[..., first], x[..., second] = a * c - b * s, b * c + a * s
            size = np.abs(x)
            size[..., first] = np.abs(a * c) + np.abs(b * s)
            size[..., second] = np.abs(b * c) + np.abs(a * s)
        x[~real] = 0.0
        size[~real] = 0.0
        return x, size, real

    def put(self, real):
        put = real & (self.slots >= 0) & (self.slots < self.pages * self.page)
        return put, self.slots[put] // self.page, self.slots[put] % self.page


def _near(got, want, size, d, typ, what):
    e = 2.0 ** -24
    bound = (d / 2 + 10) * e * size
    bound = bound + ROUND[typ] * (np.abs(want) + bound) + (2.0 ** -25 if typ == A.F16 else 0.0) + 1e-37
    assert np.all(np.isfinite(got)), what
    worst = np.max(np.abs(got - want) / bound, initial=0.0)
    assert worst <= 1.0, f"{what}: off by {worst:.3g} of its bound"


CASES = [
    (A.BF16, A.BF16, A.BF16, A.ROPE_HALF, 32, 8, 128, 128, 70, None, False, 0),
    (A.BF16, A.BF16, A.BF16, A.ROPE_HALF, 12, 12, 64, 0, 33, None, False, 0),         # norms alone
    (A.F32, A.F32, A.F32, A.ROPE_PAIRS, 8, 2, 64, 64, 51, (16, 8, 8), False, 0),
    (A.F32, A.F16, A.I8, A.ROPE_HALF, 20, 4, 96, 48, 40, (8, 8, 8), True, 0),         # 12 lanes of a row's 16
    (A.F16, A.F16, A.I8, A.ROPE_PAIRS, 16, 8, 80, 80, 9, (14, 13, 13), True, 0),
    (A.F16, A.BF16, A.BF16, A.ROPE_HALF, 8, 1, 256, 256, 17, (64, 64), False, 0),
    (A.BF16, A.F32, A.F32, A.ROPE_HALF, 4, 2, 192, 192, 13, (24, 24, 24, 24), True, 0),
    (A.F32, A.BF16, A.BF16, A.ROPE_HALF, 3, 1, 20, 20, 30, (4, 3, 3), True, 0),       # no multiple of 8
    (A.BF16, A.BF16, A.I8, A.ROPE_PAIRS, 5, 5, 36, 14, 11, (3, 4), False, 0),
    (A.BF16, A.BF16, A.BF16, A.ROPE_HALF, 4, 2, 64, 64, 20, (12, 10, 10), True, 3),   # rows not aligned
    (A.F32, A.F32, A.F32, A.ROPE_HALF, 2, 1, 8, 2, 1, None, False, 0),
    (A.F16, A.F16, A.F16, A.ROPE_HALF, 2, 1, 1, 0, 5, None, False, 0),
    (A.BF16, A.BF16, A.BF16, A.ROPE_HALF, 7, 3, 64, 64, 9000, (12, 12, 8), False, 0), # four heads a lane
]


def _id(c):
    return "-".join(str(x) for x in (NAME[c[0]], NAME[c[1]], NAME[c[2]], *c[4:9], c[9] and len(c[9]), c[11]))


@pytest.mark.parametrize("gains", [True, False], ids=["gains", "ones"])
@pytest.mark.parametrize("case", CASES, ids=_id)
def test_norm_rotate_append(ctx, case, gains):
    say("norm", _id(case), gains)
    s = Setting(ctx, *case[:11], pad=case[11], gains=gains)
    s.call()
    want, size, real = s.expected(np.float64)
    hq, d = s.hq, s.d
    _near(_values(s.qo.download(), s.tout).reshape(s.tokens, hq, d), want[:, :hq], size[:, :hq], d, s.tout, "q")
    _near(_values(s.ko.download(), s.tout).reshape(s.tokens, s.hkv, d), want[:, hq:], size[:, hq:], d, s.tout, "k")
    put, at, slot = s.put(real)
    left = np.ones((s.pages, s.page), bool)
    left[at, slot] = False
    for buf, scales, y, m in ((s.kb, s.sc[0], want[put, hq:], size[put, hq:]),
                              (s.vb, s.sc[1], s.x[put, hq + s.hkv:].astype(np.float64), None)):
        got = buf.download().reshape(s.old.shape)
        if s.cache == A.I8:
            sc = scales.download().reshape(s.pages, s.hkv, s.page)
            assert (sc.transpose(0, 2, 1)[left] == 9.0).all()
            sc = sc[at, :, slot].astype(np.float64)
            off = (d / 2 + 10) * 2.0 ** -24 * (np.abs(y) if m is None else m)
            most = np.abs(y).max(-1)
            assert np.all(np.abs(sc * 127 - np.maximum(most, 1e-8)) <= off.max(-1) + most * 2.0 ** -22 + 1e-14)
            err = np.abs(got[at, :, slot] * sc[..., None] - y)
            assert np.all(err <= 0.5 * sc[..., None] * (1 + 2.0 ** -14) + off)
            assert (got.transpose(0, 2, 1, 3)[left] == 3).all()
            continue
        vals = _values(got, s.cache)
        assert (vals.transpose(0, 2, 1, 3)[left] == 3.0).all()
        if m is None:
            assert np.array_equal(vals[at, :, slot], _round(y, s.cache))
        else:
            _near(vals[at, :, slot], y, m, d, s.cache, "cached k")


@pytest.mark.parametrize("case", [c for c in CASES if c[7]], ids=_id)
def test_axes_without_norms(ctx, case):
    """Bit for bit: each product and sum rounded to f32 by itself."""
    s = Setting(ctx, *case[:11], pad=case[11], norm=False)
    s.call()
    want, _, real = s.expected(np.float32)
    assert np.array_equal(s.qo.download().reshape(s.tokens, s.hq, s.d), _bytes(want[:, :s.hq], s.tout))
    assert np.array_equal(s.ko.download().reshape(s.tokens, s.hkv, s.d), _bytes(want[:, s.hq:], s.tout))
    put, at, slot = s.put(real)
    if s.cache != A.I8:
        for buf, y in ((s.kb, want[put, s.hq:]), (s.vb, s.x[put, s.hq + s.hkv:])):
            held = s.old.copy()
            held[at, :, slot] = y
            assert np.array_equal(buf.download().reshape(held.shape), _bytes(held, s.cache))


def test_one_axis_without_norms_is_rope_append(ctx):
    s = Setting(ctx, A.F32, A.BF16, A.I8, A.ROPE_HALF, 12, 4, 64, 64, 300, norm=False)
    s.call()
    got = [b.download() for b in (s.qo, s.ko, s.kb, s.vb, *s.sc)]
    t = Setting(ctx, A.F32, A.BF16, A.I8, A.ROPE_HALF, 12, 4, 64, 64, 300, norm=False)
    rows = [A.Rows(t.xd.ptr + o * 64 * 4, 20 * 64, 64) for o in (0, 12, 16)]
    A.RopeAppend(ctx, A.F32, 300, 12, 4, 64, *rows, t.pd, t.table, t.held, 64, A.ROPE_HALF, A.Rows(t.qo, 12 * 64, 64),
                 A.Rows(t.ko, 4 * 64, 64), A.BF16, t.pool, _dev(ctx, t.slots))()
    for a, b in zip(got, (t.qo, t.ko, t.kb, t.vb, *t.sc)):
        assert np.array_equal(a, b.download())


@pytest.mark.parametrize("d", [64, 36])
def test_in_place_and_without_a_cache(ctx, d):
    r = np.random.default_rng(3)
    x = _round(r.standard_normal((50, 6, d)), A.BF16)
    xd, pos = _dev(ctx, _bytes(x, A.BF16)), (np.arange(50) * 7).astype(np.int32)
    rot = d // 4 * 2
    table, pd = A.rope_table(ctx, 400, A.rope_inv_freq(rot)), _dev(ctx, pos)
    q, k = A.Rows(xd, 6 * d, d), A.Rows(xd.ptr + 4 * d * 2, 6 * d, d)
    A.NormRopeAppend(ctx, A.BF16, 50, 4, 1, d, q, k, norm=A.HeadNorm(1e-5),
                     rope=A.Rope(table, 400, rot, A.ROPE_HALF, pd), q_out=q, k_out=k)()
    got = _values(xd.download(), A.BF16).reshape(50, 6, d)
    assert np.array_equal(got[:, 5], x[:, 5])
    y = x[:, :5].astype(np.float64)
    y = y / np.sqrt((y * y).mean(-1, keepdims=True) + np.float32(1e-5).astype(np.float64))
    cs = table.download().astype(np.float64)[pos][:, None]
    a, b = y[..., :rot // 2].copy(), y[..., rot // 2:rot].copy()
    y[..., :rot // 2], y[..., rot // 2:rot] = a * cs[..., 0] - b * cs[..., 1], b * cs[..., 0] + a * cs[..., 1]
    size = np.abs(y)
    size[..., :rot // 2] = np.abs(a * cs[..., 0]) + np.abs(b * cs[..., 1])
    size[..., rot // 2:rot] = np.abs(b * cs[..., 0]) + np.abs(a * cs[..., 1])
    _near(got[:, :5], y, size, d, A.BF16, "in place")


@pytest.mark.parametrize("amplitude,eps", [(1e-30, 1e-6), (1e-30, 1e-38), (1e12, 1e-6), (1e-3, 1e-45)])
def test_sizes_of_values_and_eps(ctx, amplitude, eps):
    """eps decides where the values are small, and matters nothing where they are
    large; squares stay inside f32's range."""
    s = Setting(ctx, A.F32, A.F32, A.F32, A.ROPE_HALF, 4, 2, 64, 64, 20, amplitude=amplitude, eps=eps)
    s.call()
    want, size, _ = s.expected(np.float64)
    got = s.qo.download().view(np.float32).reshape(20, 4, 64)
    # squares of values near 1e-30 are subnormal or zero: what they lose is below
    # 2^-149 a term beside eps
    e = 2.0 ** -24
    lost = 64 * 2.0 ** -149 / eps if amplitude < 1e-20 else 0.0
    bound = ((64 / 2 + 10) * e + lost) * size[:, :4] + 2 * e * np.abs(want[:, :4]) + 1e-37
    assert np.all(np.abs(got - want[:, :4]) <= bound)


def test_nan_and_infinity_stay_in_their_head(ctx):
    s = Setting(ctx, A.F32, A.F32, A.F32, A.ROPE_HALF, 4, 2, 64, 64, 40)
    raw = s.xd.download().view(np.float32).reshape(40, 8, 64)
    raw[7, 1, 5], raw[9, 4, 60], raw[11, 6, 3] = np.nan, np.inf, np.nan
    s.xd.upload(raw.view(np.int32))
    s.call()
    got_q = s.qo.download().view(np.float32).reshape(40, 4, 64)
    got_k = s.ko.download().view(np.float32).reshape(40, 2, 64)
    want, size, _ = s.expected(np.float64)
    assert np.isnan(got_q[7, 1]).all() and np.isnan(got_k[9, 0, [28, 60]]).all()
    clean = np.ones((40, 4), bool)
    clean[7, 1] = False
    _near(got_q[clean], want[:, :4][clean], size[:, :4][clean], 64, A.F32, "other heads")
    clean = np.ones((40, 2), bool)
    clean[9, 0] = False
    _near(got_k[clean], want[:, 4:][clean], size[:, 4:][clean], 64, A.F32, "other keys")


@pytest.mark.parametrize("layout", [A.ROPE_HALF, A.ROPE_PAIRS], ids=["half", "pairs"])
@pytest.mark.parametrize("d,rot,pad", [(64, 0, 0), (64, 32, 0), (128, 64, 0), (64, 32, 3), (36, 0, 0), (36, 16, 0)])
def test_infinity_in_elements_that_are_not_rotated(ctx, layout, d, rot, pad):
    """One in a head makes the head's finite elements zeros and is NaN itself, with
    its partner in the rotation if it has one; one in a gain is its own element's."""
    say(f"infinity d {d} rot {rot} pad {pad}")
    s = Setting(ctx, A.F32, A.F32, A.F32, layout, 4, 2, d, rot, 40, pad=pad)
    width = 8 * d + pad
    raw = s.xd.download().view(np.float32).reshape(40, width)
    rows = {(7, 1): rot, (9, 4): d - 1, (11, 5): rot + (d - rot) // 2, (20, 0): 0, (21, 2): max(rot - 1, 0)}
    for (t, h), e in rows.items():
        raw[t, h * d + e] = s.x[t, h, e] = np.inf
    s.xd.upload(raw.view(np.int32))
    for g, gd in zip(s.g, s.gd):
        g[d - 2] = np.inf
        gd.upload(g)
    s.call()
    with np.errstate(invalid="ignore"):
        want, size, real = s.expected(np.float64)
    got = np.concatenate([s.qo.download().view(np.float32).reshape(40, 4, d),
                          s.ko.download().view(np.float32).reshape(40, 2, d)], 1)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    assert np.isnan(want[7, 1]).sum() == 2 and all(real[t] for t, _ in rows)  # its own, and 0 times the gain's
    far = np.isinf(want)
    assert far.any() and np.array_equal(got[far], want[far])
    seen = np.isfinite(want)
    _near(got[seen], want[seen], size[seen], d, A.F32, "finite elements")


def test_captured_and_replayed(ctx):
    s = Setting(ctx, A.BF16, A.BF16, A.BF16, A.ROPE_HALF, 8, 2, 64, 64, 64, (12, 10, 10), True)
    s.call()
    first = [b.download() for b in (s.qo, s.kb, s.vb)]
    with D.Graph(ctx) as g:
        s.call()
    for turn in range(3):
        for b in (s.qo, s.kb, s.vb):
            D.memset(ctx, b, turn, b.nbytes)
        g.launch()
        assert np.array_equal(s.qo.download(), first[0])
        put, at, slot = s.put(s.expected(np.float64)[2])
        for b, want in ((s.kb, first[1]), (s.vb, first[2])):
            shape = s.old.shape
            assert np.array_equal(b.download().reshape(shape)[at, :, slot], want.reshape(shape)[at, :, slot])
    g.close()


def test_head_of_zeros(ctx):
    s = Setting(ctx, A.F32, A.F32, A.F32, A.ROPE_HALF, 4, 2, 64, 64, 1)
    s.call()
    assert not s.qo.download().view(np.float32).reshape(4, 64)[0].any()


def test_another_device_refuses_its_cache(ctx):
    """The handle's device is checked before anything is launched (where there is
    one device alone, a handle that says another stands for it)."""
    pool = A.KVCache(ctx, A.F32, 1, 16, 1, 64)
    z = _dev(ctx, np.zeros(64, np.float32))
    device = C.cast(pool.handle, C.POINTER(C.c_int))
    was = device[0]
    device[0] = was + 1
    rows = A.Rows(z, 64, 64)
    try:
        with pytest.raises(ValueError, match="device"):
            A.NormRopeAppend(ctx, A.F32, 1, 1, 1, 64, rows, rows, rows, A.HeadNorm(1e-6), cache=pool, slots=z)()
    finally:
        device[0] = was

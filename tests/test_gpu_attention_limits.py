"""Attention where a call stands at an edge of what the entry points take: rows
that no sequence covers before the first one, outputs over the queries, the
largest sizes, scales and lengths, values that are not finite.
"""
import numpy as np
import pytest

from tokenvector.inference_amd import _lib
from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D

from test_gpu_attention import NAME, Paged, _bytes, _check, _dev, _i32, _round, _seen, _values, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


# ---- rows before the first sequence ----------------------------------------------

# query rows, and key rows (the same, or over 256 each, which are split), of the
# sequences behind 200 rows that are nobody's: over 128 rows of two heads
LEADING = [([120, 90], [120, 90]), ([40], [3000]), ([70, 130], [2000, 600])]


@pytest.mark.parametrize("typ", [A.BF16, A.F16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("lens_q,lens_k", LEADING)
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
def test_prompt_behind_uncovered_rows(ctx, typ, lens_q, lens_k, in_place):
    lead, hq, hkv, d = 200, 4, 2, 64
    say(f"prompt {NAME[typ]} {lens_q} over {lens_k} behind {lead} rows, in place {in_place}")
    r = np.random.default_rng(sum(lens_q))
    cu_q, cu_k = lead + np.r_[0, np.cumsum(lens_q)], np.r_[0, np.cumsum(lens_k)]
    tq, tk = int(cu_q[-1]) + 9, int(cu_k[-1])
    q = _round(r.standard_normal((tq, hq, d)), typ)
    kv = _round(r.standard_normal((tk, 2 * hkv, d)), typ)
    qd, kvd = _dev(ctx, _bytes(q, typ)), _dev(ctx, _bytes(kv, typ))
    out0 = q if in_place else np.full_like(q, 7.25)
    od = qd if in_place else _dev(ctx, _bytes(out0, typ))
    w = 4 if typ == A.F32 else 2
    A.AttentionPrompt(ctx, typ, tq, hq, hkv, d, len(lens_q), A.Rows(qd, hq * d, d),
                      A.Rows(kvd, 2 * hkv * d, d), A.Rows(kvd.ptr + hkv * d * w, 2 * hkv * d, d),
                      A.Rows(od, hq * d, d), _i32(ctx, cu_q), _i32(ctx, cu_k), tk)()
    got = _values(od.download(), typ).reshape(q.shape)
    for s, (n, t) in enumerate(zip(lens_q, lens_k)):
        rows, keys = slice(cu_q[s], cu_q[s + 1]), slice(cu_k[s], cu_k[s + 1])
        _check(got[rows], q[rows], kv[keys, :hkv], kv[keys, hkv:], _seen(n, t, True, 0), d ** -0.5, typ, typ,
               f"sequence {s} behind uncovered rows")
    assert np.array_equal(got[:lead], out0[:lead]) and np.array_equal(got[cu_q[-1]:], out0[cu_q[-1]:])


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F32, A.F32), (A.F16, A.I8)],
                         ids=lambda t: NAME[t])
@pytest.mark.parametrize("total", [100, 5000])
@pytest.mark.parametrize("in_place", [False, True], ids=["apart", "in place"])
def test_chunk_behind_uncovered_rows(ctx, typ, cache, total, in_place):
    """200 of the call's rows come before the only sequence, which has 40."""
    lead, n = 200, 40
    say(f"chunk {NAME[typ]} over {NAME[cache]}, {total} keys, behind {lead} rows, in place {in_place}")
    p = Paged(ctx, typ, cache, 4, 2, 64, [lead, n], [0, total])
    out = p.qd if in_place else p.od
    call = A.AttentionPaged(ctx, typ, lead + n, 4, p.pool, 1, A.Rows(p.qd, 256, 64), A.Rows(out, 256, 64),
                            _i32(ctx, p.tab.download()[1:]), p.tab.shape[1], _i32(ctx, [total]),
                            _i32(ctx, [lead, lead + n]), n, total, p.scale)
    call()
    got = _values(out.download(), typ).reshape(p.q.shape)
    k, v = p.kv[1]
    _check(got[lead:], p.q[lead:], k, v, _seen(n, total, True, 0), p.scale, typ, typ, "the covered chunk")
    assert np.array_equal(got[:lead], (p.q if in_place else p.out0)[:lead])


# ---- the longest caches ------------------------------------------------------------

@pytest.fixture(scope="module")
def long_table(ctx):
    """Page ids of 2^31 keys, all of them page 0."""
    t = _dev(ctx, np.zeros(1 << 27, np.int32))
    yield t
    t.close()


@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F16, A.I8), (A.F32, A.F32)], ids=lambda t: NAME[t])
@pytest.mark.parametrize("d", [64, 20])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("held", [(1 << 31) - 1, (1 << 31) - 256, (1 << 31) - 300])
def test_cache_of_the_most_keys(ctx, long_table, typ, cache, d, new, held):
    """Lengths up to 2^31 - 1 count as 2^31 - 256 at most; a window keeps it short."""
    window, hkv, page = 100, 2, 16
    say(f"{new} new of {held} keys, {NAME[typ]} over {NAME[cache]}, heads of {d}")
    p = Paged(ctx, typ, cache, 2, hkv, d, [new], [page], page=page)
    total = min(held, (1 << 31) - 256)
    first = total - new - window
    slot = np.arange(first, total) % page
    # page 0 of the pool as the only one: the sequence's page by a pool of its own
    pg = int(p.tab.download()[0, 0])
    at = [b.download()[pg:pg + 1] for b in p.bufs]
    pools = [_dev(ctx, x) for x in at]
    scales = [_dev(ctx, s[pg:pg + 1]) for s in (p.ks, p.vs)] if cache == A.I8 else [None, None]
    pool = A.KVCache(ctx, cache, 1, page, hkv, d, *pools, *scales)
    call = A.AttentionPaged(ctx, typ, new, 2, pool, 1, A.Rows(p.qd, 2 * d, d), A.Rows(p.od, 2 * d, d), long_table,
                            1 << 27, _i32(ctx, [held]), _i32(ctx, [0, new]), new, 0, p.scale, True, window)
    call()
    k, v = p.kv[0]
    mask = _seen(new, new + window, True, window)
    _check(p.result(), p.q, k[slot], v[slot], mask, p.scale, typ, typ, "the most keys")


def test_refuses_rows_beyond_the_kernels_numbers(ctx):
    """Refused on the host: nothing of this size is read."""
    z = _dev(ctx, np.zeros(256, np.float32))
    rows, cu = A.Rows(z, 64, 64), _i32(ctx, [0, 1])
    with pytest.raises(_lib.TkvHipError):
        A.AttentionPrompt(ctx, A.F32, (1 << 30) - 4096, 2, 1, 64, 1, rows, rows, rows, rows, cu)()


# ---- calls of more than 2^24 workgroups -----------------------------------------------

def _single_keys(ctx, tokens, hq, hkv, d):
    """As many sequences of one token: every output row is its value, to the bit."""
    r = np.random.default_rng(d)
    q = r.integers(0x3e00, 0x4000, (tokens, hq, d), dtype=np.uint16)       # bf16 of 1 / 8 to 2
    kv = r.integers(0x3e00, 0x4000, (tokens, 2 * hkv, d), dtype=np.uint16)
    qd, kvd = _dev(ctx, q), _dev(ctx, kv)
    A.AttentionPrompt(ctx, A.BF16, tokens, hq, hkv, d, tokens, A.Rows(qd, hq * d, d),
                      A.Rows(kvd, 2 * hkv * d, d), A.Rows(kvd.ptr + 2 * hkv * d, 2 * hkv * d, d),
                      A.Rows(qd, hq * d, d), _i32(ctx, np.arange(tokens + 1)))()
    got = qd.download()
    assert np.array_equal(got, np.repeat(kv[:, hkv:], hq // hkv, axis=1))


def test_any_layout_of_2_26_rows(ctx):
    """A row per wave, four waves a workgroup."""
    _single_keys(ctx, (1 << 20) + 5, 64, 1, 2)


def test_tiles_of_2_24_units(ctx):
    """A unit per sequence and key / value head, and more."""
    _single_keys(ctx, (1 << 20) + 3, 16, 16, 8)


def test_table_of_2_32_entries(ctx):
    positions, inv = (1 << 30) + 7, A.rope_inv_freq(8)
    table = A.rope_table(ctx, positions, inv)
    p = np.arange(positions - 5, positions)
    got = np.empty((5, 4, 2), np.float32)
    _lib.check(_lib.lib().tkv_hip_memcpy_d2h(ctx.handle, got.ctypes.data, table.ptr + (positions - 5) * 32,
                                             got.nbytes))
    table.close()
    a = p[:, None].astype(np.float64) * inv
    # the product's rounding in f64 (2^-24 at 2^30), and f32's
    assert np.all(np.abs(got - np.stack([np.cos(a), np.sin(a)], -1)) <= 2.0 ** -24 + 2.0 ** -23)


# ---- a cache between contexts ----------------------------------------------------------

def test_new_cache_belongs_to_every_context(ctx):
    """Tokens appended from a second context right after the cache was made stay: the
    zeros are there before the handle is."""
    heads, page, d = 8, 256, 128
    pages = 8192                                     # 4 GiB each of keys and values
    slots = np.linspace(0, pages * page - 1, 4096).astype(np.int64)
    x = _round(np.random.default_rng(6).uniform(1.0, 2.0, (slots.size, heads, d)), A.BF16)
    other = D.Context(0)
    try:
        xd, sd = _dev(other, _bytes(x, A.BF16)), _dev(other, slots)
        rows = A.Rows(xd, heads * d, d)
        other.synchronize()
        cache = A.KVCache(ctx, A.BF16, pages, page, heads, d)
        A.RopeAppend(other, A.BF16, slots.size, 0, heads, d, None, rows, rows, cache=cache, slots=sd)()
        other.synchronize()
        ctx.synchronize()
        got = np.empty((heads, d), np.int16)
        row = np.empty(d, np.int16)
        for i in (0, 1, 2047, 4094, 4095):
            for pool in (cache.k, cache.v):
                for h in range(heads):
                    at = ((slots[i] // page * heads + h) * page + slots[i] % page) * d * 2
                    _lib.check(_lib.lib().tkv_hip_memcpy_d2h(other.handle, row.ctypes.data, int(pool + at), row.nbytes))
                    got[h] = row
                assert np.array_equal(got, _bytes(x[i], A.BF16))
        cache.close()
    finally:
        other.close()


# ---- the least scales --------------------------------------------------------------------

@pytest.mark.parametrize("typ", [A.BF16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("scale,size", [(1e-35, 1e17), (3e-38, 3e18), (0.0, 1e17), (0.0, 1e18)])
@pytest.mark.parametrize("d", [64, 33])
@pytest.mark.parametrize("new", [1, 60])
def test_least_scales(ctx, typ, scale, size, d, new):
    """Products as large as the scale is small have ordinary logits; at scale 0 all
    weights are equal whatever the products.  Products are f32: rows with one past
    its range are not compared."""
    say(f"{NAME[typ]} scale {scale} of products of {size * size}, {new} new, heads of {d}")
    p = Paged(ctx, typ, typ, 4, 2, d, [new], [300], scale=scale)
    k, v = p.kv[0]
    tab, raw = p.tab.download(), p.bufs[0].download()
    p.q = _round(p.q * np.float32(size), typ)
    k[:] = _round(k * np.float32(size), typ)
    for j in range(300):
        raw[tab[0, j // 16], :, j % 16] = _bytes(k[j], typ)
    p.qd.upload(_bytes(p.q, typ))
    p.bufs[0].upload(raw)
    p.call()
    got, mask = p.result(), _seen(new, 300, True, 0)
    for h in range(4):
        products = p.q[:, h].astype(np.float64) @ k[:, h // 2].T.astype(np.float64)
        rows = np.abs(products).max(1) <= np.finfo(np.float32).max
        _check(got[rows, h:h + 1], p.q[rows, h:h + 1], k[:, h // 2:h // 2 + 1], v[:, h // 2:h // 2 + 1], mask[rows],
               p.scale, typ, typ, f"least scale, head {h}")


# ---- values that are not finite in an int8 cache -----------------------------------------

@pytest.mark.parametrize("typ", [A.BF16, A.F32], ids=lambda t: NAME[t])
@pytest.mark.parametrize("d", [64, 96, 33])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_int8_rows_that_are_not_finite(ctx, typ, d, bad):
    """One element that is not a number, or infinite, makes its row's values NaN, as
    code times scale; the rows beside it are coded as ever, and tokens that attend
    to it are not finite."""
    tokens, heads, page = 40, 3, 16
    r = np.random.default_rng(d)
    x = _round(r.standard_normal((tokens, 2 * heads, d)), typ)
    rows = [(3, 0, 0), (17, 2, d - 1), (17, 4, 5), (30, 5, d // 2)]     # keys of heads 0, 2; values of 1, 2
    for t, h, e in rows:
        x[t, h, e] = bad
    xd = _dev(ctx, _bytes(x, typ))
    w, pages = (4 if typ == A.F32 else 2), 3
    bufs = [_dev(ctx, np.zeros((pages, heads, page, d), np.int8)) for _ in range(2)]
    scales = [_dev(ctx, np.zeros((pages, heads, page), np.float32)) for _ in range(2)]
    pool = A.KVCache(ctx, A.I8, pages, page, heads, d, *bufs, *scales)
    A.RopeAppend(ctx, typ, tokens, 0, heads, d, None, A.Rows(xd, 2 * heads * d, d),
                 A.Rows(xd.ptr + heads * d * w, 2 * heads * d, d), cache=pool,
                 slots=_dev(ctx, np.arange(tokens, dtype=np.int64)))()
    hit = np.zeros((tokens, 2 * heads), bool)
    for t, h, _ in rows:
        hit[t, h] = True
    for i in range(2):
        codes, sc = bufs[i].download(), scales[i].download()
        at, slot = np.arange(tokens) // page, np.arange(tokens) % page
        with np.errstate(invalid="ignore"):
            value = codes[at, :, slot] * sc[at, :, slot][..., None]
        part, sick = x[:, i * heads:(i + 1) * heads], hit[:, i * heads:(i + 1) * heads]
        assert np.isnan(value[sick]).all()
        y = part[~sick]
        scale = np.maximum(np.abs(y).max(-1), np.float32(1e-8)) * (np.float32(1) / np.float32(127))
        want = np.clip(np.rint(y * (np.float32(1) / scale)[:, None]), -127, 127)
        assert np.array_equal(sc[at, :, slot][~sick], scale) and np.array_equal(codes[at, :, slot][~sick], want)
    q = _round(r.standard_normal((tokens, heads, d)), typ)
    qd = _dev(ctx, _bytes(q, typ))
    A.AttentionPaged(ctx, typ, tokens, heads, pool, 1, A.Rows(qd, heads * d, d), A.Rows(qd, heads * d, d),
                     _i32(ctx, np.arange(pages)), pages, _i32(ctx, [tokens]), _i32(ctx, [0, tokens]), tokens, tokens)()
    got = _values(qd.download(), typ).reshape(q.shape)
    for h, first in ((0, 3), (1, 17), (2, 17)):
        assert np.isfinite(got[:first, h]).all() and not np.isfinite(got[first:, h]).any()


# ---- more units than there are arrival counters ---------------------------------------------

@pytest.mark.parametrize("typ,cache", [(A.BF16, A.BF16), (A.F16, A.I8)], ids=lambda t: NAME[t])
@pytest.mark.parametrize("new", [1, 9], ids=["token", "chunk"])
def test_more_than_1024_units(ctx, typ, cache, new):
    """130 sequences of 8 key / value heads, one of them long: no splits."""
    say(f"1040 units, {new} new, {NAME[typ]} over {NAME[cache]}")
    r = np.random.default_rng(3)
    total = (new + r.integers(0, 40, 130)).tolist()
    total[77] = 3000
    p = Paged(ctx, typ, cache, 32, 8, 64, [new] * 130, total)
    p.call()
    p.check("more than 1024 units")

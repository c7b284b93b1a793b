"""f16 attention where the weights, or their products with an int8 cache's value
scales, reach over more octaves than f16 has: one key far above a long tail, and
scales that differ by powers of two.

The bound of an element, from the formula in 64 bits, is that of the other
attention tests with the part of f16's range that the kernels promise:

  weights (f16 caches)        off by 2^-11 of themselves or 2^-32 of the largest
  products with scales (int8) off by 2^-11 of themselves or 2^-31 of the largest
"""
import numpy as np
import pytest

from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D

from test_gpu_attention import Paged, Prompt, _bytes, _round, _seen, say

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


def _check_f16(got, q, k, v, mask, scale, typ_out, step, vmax, what):
    """q, k, v, got [n or t, heads, d]; vmax [t, heads_kv]: the largest |v| that a
    rounded weight may stand before (127 scales of an int8 cache); step: what the
    smallest products are off by, in the largest one."""
    n, hq, d = q.shape
    g, t, e = hq // k.shape[1], k.shape[0], 2.0 ** -24
    for h in range(hq):
        qh, kh, vh = (x.astype(np.float64) for x in (q[:, h], k[:, h // g], v[:, h // g]))
        a = np.where(mask, scale * (qh @ kh.T), -np.inf)
        w = np.exp(a - a.max(1, keepdims=True))
        total = w.sum(1)[:, None]
        ref, spread = w @ vh / total, w @ np.abs(vh) / total
        size = np.where(mask, scale * (np.abs(qh) @ np.abs(kh).T), 0.0).max(1)[:, None]
        largest = (w * vmax[:, h // g]).max(1)[:, None] / total
        rel = 2.0 * (d + 8) * e * size + (t + t / 4 + 32) * e
        bound = rel * spread + 2.0 ** -11 * spread * (1 + rel) + t * step * largest * (1 + rel)
        rounding = 2.0 ** -11 if typ_out == A.F16 else e
        bound = 1.05 * (bound + rounding * np.abs(ref) * (1 + rel) + (2.0 ** -25 if typ_out == A.F16 else 0.0))
        err = np.abs(got[:, h] - ref)
        assert np.all(np.isfinite(got[:, h])), f"{what}: head {h} has values that are not finite"
        worst = np.max(err / (bound + 1e-30))
        assert worst <= 1.0, f"{what}: head {h} off by {worst:.3g} of its bound"


class Scales(Paged):
    """An int8 cache whose logits follow the keys' codes: q > 0, a key's codes all
    the same.  far: {key: (log2 of its weight, log2 of its value scale)} beside
    ordinary ones of weight about 1 and scale about 2^-6."""

    def __init__(self, ctx, new, total, far, typ_out):
        super().__init__(ctx, A.F16, A.I8, 4, 2, 64, [new], [total], page=16, typ_out=typ_out)
        r = np.random.default_rng(total + new)
        self.q = _round(r.uniform(0.5, 1.0, self.q.shape), A.F16)
        self.qd.upload(_bytes(self.q, A.F16))
        tab, codes = self.tab.download(), self.bufs[0].download()
        value_codes = self.bufs[1].download()
        k, v = self.kv[0]
        self.vmax = np.empty(k.shape[:2])
        for j in range(total):
            pg, slot = tab[0, j // 16], j % 16
            weight, octave = far.get(j, (0.0, 0.0))
            # a logit of about ks * code * 48 / 8
            code = 3 if weight == 0 else int(np.sign(weight)) * 100
            ks = r.uniform(0.01, 0.02, 2) if weight == 0 else np.full(2, abs(weight) * np.log(2.0) / 600.0)
            vs = r.uniform(0.005, 0.02, 2) * 2.0 ** octave
            codes[pg, :, slot] = code
            self.ks[pg, :, slot], self.vs[pg, :, slot] = ks, vs
            ks, vs = self.ks[pg, :, slot].astype(np.float64), self.vs[pg, :, slot].astype(np.float64)
            k[j] = code * ks[:, None]
            v[j] = value_codes[pg, :, slot] * vs[:, None]
            self.vmax[j] = 127.0 * vs
        self.bufs[0].upload(codes)
        self.pool._kept[2].upload(self.ks)
        self.pool._kept[3].upload(self.vs)

    def check(self, what):
        k, v = self.kv[0]
        _check_f16(self.result(), self.q, k, v, _seen(self.new[0], self.total[0], True, 0), self.scale,
                   self.typ_out, 2.0 ** -31, self.vmax, what)


@pytest.mark.parametrize("new", [1, 60], ids=["token", "chunk"])
@pytest.mark.parametrize("total", [400, 3000])
@pytest.mark.parametrize("octaves", [16, 20, 26, 40, 60])
@pytest.mark.parametrize("at", [10, 300])
def test_int8_scale_of_a_key_without_weight(ctx, new, total, octaves, at):
    """A key of weight 2^-40 whose value's scale is far above the others."""
    say(f"f16 over int8: {new} new of {total}, key {at} of weight 2^-40, scale 2^{octaves}")
    p = Scales(ctx, new, total, {at: (-40.0, octaves)}, A.F32)
    p.call()
    p.check("a key without weight")


@pytest.mark.parametrize("new", [1, 60], ids=["token", "chunk"])
@pytest.mark.parametrize("total", [400, 3000])
@pytest.mark.parametrize("octaves", [16, 26, 38])
@pytest.mark.parametrize("typ_out", [A.F16, A.F32], ids=["f16", "f32"])
def test_int8_scale_left_behind_by_the_maximum(ctx, new, total, octaves, typ_out):
    """A key whose product leads until a later key takes nearly all of the weight."""
    say(f"f16 over int8: {new} new of {total}, key 5 of scale 2^{octaves}, key 330 of weight 2^40")
    p = Scales(ctx, new, total, {5: (0.0, octaves), 330: (40.0, 0.0)}, typ_out)
    p.call()
    p.check("a scale left behind")


@pytest.mark.parametrize("new", [1, 60], ids=["token", "chunk"])
def test_int8_scales_far_apart_in_weight_and_size(ctx, new):
    """Products of every size, up and down, key after key."""
    r = np.random.default_rng(7)
    far = {int(j): (float(r.integers(1, 25)) * (1 if i % 2 else -1), float(r.integers(-40, 40)))
           for i, j in enumerate(range(3, 330, 6))}
    p = Scales(ctx, new, 400, far, A.F32)
    p.call()
    p.check("products of every size")


def _tail(r, tokens, heads, d, sink, at):
    """Queries of 0.5 to 1 and keys that they see as a sink `sink` octaves (at scale
    1 / 8) above a long tail; values of the tail about 1, the sink's about 2^-10."""
    q = _round(r.uniform(0.5, 1.0, (tokens, heads, d)), A.F16)
    k = _round(r.uniform(-0.02, 0.02, (tokens, heads, d)), A.F16)
    v = _round(r.uniform(0.5, 1.5, (tokens, heads, d)), A.F16)
    k[at] = _round(np.full((heads, d), sink * np.log(2.0) / 6.0 * 64 / d), A.F16)
    v[at] = _round(v[at] * 2.0 ** -10, A.F16)
    return q, k, v


@pytest.mark.parametrize("typ_out", [A.F16, A.F32], ids=["f16", "f32"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("at", [0, 700])
@pytest.mark.parametrize("sink", [26.0, 30.0])
def test_prompt_tail_below_a_sink(ctx, typ_out, d, at, sink):
    """Keys of 2^-26 and 2^-30 of the largest weight, and the larger values, have their part."""
    n = 1500
    say(f"f16 prompt of {n}, sink {sink} octaves up at {at}, heads of {d}")
    p = Prompt(ctx, A.F16, 2, 2, d, [n], typ_out=typ_out, scale=0.125)
    q, k, v = _tail(np.random.default_rng(11), n, 2, d, sink, at)
    x = p.x.reshape(-1, 6, d)
    x[:n] = np.concatenate([q, k, v], 1)
    p.xd.upload(_bytes(p.x.reshape(-1), A.F16))
    p.call()
    _check_f16(p.result()[:n], q, k, v, _seen(n, n, True, 0), 0.125, typ_out, 2.0 ** -32,
               np.abs(v).max(2).astype(np.float64), "a prompt's tail below a sink")


@pytest.mark.parametrize("typ_out", [A.F16, A.F32], ids=["f16", "f32"])
@pytest.mark.parametrize("new", [1, 60], ids=["token", "chunk"])
@pytest.mark.parametrize("at", [0, 15000])
@pytest.mark.parametrize("sink", [26.0, 30.0])
def test_cache_tail_below_a_sink(ctx, typ_out, new, at, sink):
    """The same over a long cache, in splits of which one has the sink."""
    t, d, page = 20000, 64, 256
    say(f"f16 {new} new over {t}, sink {sink} octaves up at {at}")
    q, k, v = _tail(np.random.default_rng(12), t, 2, d, sink, at)
    q, pages = q[:new], -(-t // page)
    pools = []
    for x in (k, v):
        pool = np.zeros((pages * page, 2, d), np.float32)
        pool[:t] = x
        pools.append(D.DeviceBuffer.from_host(ctx, _bytes(
            pool.reshape(pages, page, 2, d).transpose(0, 2, 1, 3), A.F16)))
    cache = A.KVCache(ctx, A.F16, pages, page, 2, d, *pools)
    put = lambda a: D.DeviceBuffer.from_host(ctx, np.asarray(a, np.int32))  # noqa: E731
    qd = D.DeviceBuffer.from_host(ctx, _bytes(q, A.F16))
    od = D.DeviceBuffer.empty(ctx, q.shape, np.uint16 if typ_out == A.F16 else np.float32)
    A.AttentionPaged(ctx, A.F16, new, 2, cache, 1, A.Rows(qd, 2 * d, d), A.Rows(od, 2 * d, d),
                     put(np.arange(pages)), pages, put([t]), put([0, new]), new, t, 0.125, type_out=typ_out)()
    got = od.download()
    got = got.view(np.float16).astype(np.float32) if typ_out == A.F16 else got
    _check_f16(got, q, k, v, _seen(new, t, True, 0), 0.125, typ_out, 2.0 ** -32,
               np.abs(v).max(2).astype(np.float64), "a cache's tail below a sink")

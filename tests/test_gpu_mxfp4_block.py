"""The served attention half of a block in 4 bits, its operators in turn: the fused
projection as an MXFP4 linear, norms per head with positions on three axes and the
append, attention over the paged cache, the output linear; prompts in chunks, then
single tokens, eager and as a captured decode step.

Every operator's output is compared with its formula in 64 bits on what the operator
before it left on the device, within the roundings of that operator alone.
"""
import sys

import numpy as np
import pytest
import torch

from tokenvector.inference_amd import attention as A
from tokenvector.inference_amd import device as D
from tokenvector.inference_amd import mxfp4 as X
from test_gpu_mxfp4 import code_of, value_of

pytestmark = pytest.mark.gpu

HQ, HKV, HD, WIDTH = 12, 4, 64, 768
ROW = (HQ + 2 * HKV) * HD
PAGE, PAGES, POSITIONS = 16, 40, 2000
E = 2.0 ** -24


def say(*a):
    print(*a, flush=True)
    sys.stdout.flush()


@pytest.fixture(scope="module")
def ctx(hip):
    c = D.Context(0)
    yield c
    c.close()


def _bf16(raw):
    return (raw.astype(np.uint32) << 16).view(np.float32)


class Layer:
    """Weights, gains, table and cache, and device buffers for up to `most` tokens."""

    def __init__(self, ctx, most):
        r = np.random.default_rng(7)
        self.ctx, self.most = ctx, most
        self.w_qkv = (r.standard_normal((ROW, WIDTH)) * 0.05).astype(np.float32)
        self.w_out = (r.standard_normal((WIDTH, HQ * HD)) * 0.05).astype(np.float32)
        self.b_out = r.standard_normal(WIDTH).astype(np.float32)
        put = self.put
        self.qkv = D.QuantizedLinear.from_float(ctx, put(self.w_qkv), ROW, WIDTH, None, D.WEIGHT_MXFP4)
        self.out = D.QuantizedLinear.from_float(ctx, put(self.w_out), WIDTH, HQ * HD, put(self.b_out), D.WEIGHT_MXFP4)
        self.gains = [r.uniform(0.5, 1.5, HD).astype(np.float32) for _ in range(2)]
        self.dg = [put(g) for g in self.gains]
        self.pairs = A.rope_pair_axes([12, 10, 10], interleaved=True)
        self.table = A.rope_table(ctx, POSITIONS, A.rope_inv_freq(HD))
        self.cache = A.KVCache(ctx, A.BF16, PAGES, PAGE, HKV, HD)
        self.free, self.tables, self.lengths = list(range(PAGES)), {}, {}
        empty = D.DeviceBuffer.empty
        self.x = empty(ctx, (most, WIDTH), np.float32)
        self.h = empty(ctx, (most, ROW), np.float32)
        self.q, self.att = (empty(ctx, (most, HQ, HD), np.uint16) for _ in range(2))
        self.y = empty(ctx, (most, WIDTH), np.float32)
        self.pos, self.slots = empty(ctx, (3, most), np.int32), empty(ctx, most, np.int64)
        self.cu, self.lens = empty(ctx, 9, np.int32), empty(ctx, 8, np.int32)
        self.pages = empty(ctx, (8, PAGES), np.int32)

    def put(self, a):
        return D.DeviceBuffer.from_host(self.ctx, a)

    def place(self, chunks):
        """Inputs, positions, slots and tables of {sequence: x} on the device."""
        pos, slots, cu, lens = [], [], [0], []
        table = np.zeros((8, PAGES), np.int32)
        for i, (name, x) in enumerate(chunks.items()):
            start = self.lengths.get(name, 0)
            pages = self.tables.setdefault(name, [])
            while len(pages) * PAGE < start + len(x):
                pages.append(self.free.pop())
            at = np.arange(start, start + len(x))
            pos.append(np.stack([at, at // 7, at % 7]))
            slots.append(np.array(pages)[at // PAGE] * PAGE + at % PAGE)
            self.lengths[name] = start + len(x)
            cu.append(cu[-1] + len(x))
            lens.append(start + len(x))
            table[i, :len(pages)] = pages
        n = cu[-1]
        host = np.full((3, self.most), -1, np.int32)
        host[:, :n] = np.concatenate(pos, 1)
        self.x.upload(np.concatenate(list(chunks.values())).astype(np.float32))
        self.pos.upload(host)
        self.slots.upload(np.concatenate(slots).astype(np.int64))
        self.cu.upload(np.array(cu, np.int32))
        self.lens.upload(np.array(lens, np.int32))
        self.pages.upload(table)
        return n, cu, lens, host

    def calls(self, n, sequences, max_q, max_kv):
        rows = [A.Rows(self.h.ptr + 4 * o * HD, ROW, HD) for o in (0, HQ, HQ + HKV)]
        q = A.Rows(self.q, HQ * HD, HD)
        return [X.Linear(self.ctx, self.qkv, A.F32, self.x, WIDTH, n, A.F32, self.h),
                A.NormRopeAppend(self.ctx, A.F32, n, HQ, HKV, HD, *rows, norm=A.HeadNorm(1e-6, *self.dg),
                                 rope=A.Rope(self.table, POSITIONS, HD, A.ROPE_HALF, self.pos, 3, self.most, self.pairs),
                                 q_out=q, type_out=A.BF16, cache=self.cache, slots=self.slots),
                A.AttentionPaged(self.ctx, A.BF16, n, HQ, self.cache, sequences, q, A.Rows(self.att, HQ * HD, HD),
                                 self.pages, PAGES, self.lens, self.cu, max_q, max_kv),
                X.Linear(self.ctx, self.out, A.BF16, self.att, HQ * HD, n, A.F32, self.y)]

    def pools(self):
        size = PAGES * HKV * PAGE * HD
        out = []
        for p in (self.cache.k, self.cache.v):
            host = np.empty(size, np.uint16)
            from tokenvector.inference_amd import _lib
            import ctypes as C
            _lib.check(_lib.lib().tkv_hip_memcpy_d2h(self.ctx.handle, host.ctypes.data_as(C.c_void_p), C.c_void_p(p),
                                                     host.nbytes))
            out.append(_bf16(host).reshape(PAGES, HKV, PAGE, HD).astype(np.float64))
        return out

    def check(self, n, cu, lens, pos, names, what):
        x = self.x.download()[:n]
        h = self.h.download()[:n]
        self.linear(h, x, self.w_qkv, None, what + " projection")
        h = h.reshape(n, HQ + 2 * HKV, HD).astype(np.float64)
        qk = h[:, :HQ + HKV] / np.sqrt((h[:, :HQ + HKV] ** 2).mean(-1, keepdims=True) + np.float64(np.float32(1e-6)))
        qk[:, :HQ] *= self.gains[0]
        qk[:, HQ:] *= self.gains[1]
        tab = self.table.download().astype(np.float64)
        cs = tab[pos[:, :n][self.pairs], np.arange(HD // 2)[:, None]].transpose(1, 0, 2)[:, None]
        c, s = cs[..., 0], cs[..., 1]
        a, b = qk[..., :HD // 2].copy(), qk[..., HD // 2:].copy()
        qk = np.concatenate([a * c - b * s, b * c + a * s], -1)
        size = np.concatenate([np.abs(a * c) + np.abs(b * s), np.abs(b * c) + np.abs(a * s)], -1)
        bound = (HD / 2 + 10) * E * size + 2.0 ** -8 * np.abs(qk) * 1.001
        q = _bf16(self.q.download()[:n]).astype(np.float64)
        assert np.all(np.abs(q - qk[:, :HQ]) <= bound[:, :HQ]), what + " queries"
        kp, vp = self.pools()
        att = _bf16(self.att.download()[:n]).astype(np.float64)
        for i, name in enumerate(names):
            lo, hi, t = cu[i], cu[i + 1], lens[i]
            at = np.arange(t)
            page = np.array(self.tables[name])[at // PAGE]
            k, v = kp[page, :, at % PAGE], vp[page, :, at % PAGE]  # [t, HKV, HD]
            new = k[t - (hi - lo):]
            assert np.all(np.abs(new - qk[lo:hi, HQ:]) <= bound[lo:hi, HQ:]), what + " cached keys"
            want_v = torch.from_numpy(h[lo:hi, HQ + HKV:].astype(np.float32)).to(torch.bfloat16).double().numpy()
            assert np.array_equal(v[t - (hi - lo):], want_v), what + " cached values"
            hidden = at[None, :] > (t - (hi - lo) + np.arange(hi - lo))[:, None]
            for head in range(HQ):
                kk, vv = k[:, head // (HQ // HKV)], v[:, head // (HQ // HKV)]
                l = q[lo:hi, head] @ kk.T / 8.0
                size_l = np.where(hidden, 0.0, np.abs(q[lo:hi, head]) @ np.abs(kk).T / 8.0).max(1)[:, None]
                l[hidden] = -np.inf
                w = np.exp(l - l.max(1, keepdims=True))
                total = w.sum(1, keepdims=True)
                ref, spread = w @ vv / total, w @ np.abs(vv) / total
                rel = 2.0 * (HD + 8) * E * size_l + (1.25 * t + 32) * E
                off = rel * spread + 2.0 ** -8 * spread * (1 + rel) + 2.0 ** -8 * np.abs(ref) * (1 + rel)
                assert np.all(np.abs(att[lo:hi, head] - ref) <= 1.05 * off + 1e-30), f"{what} attention, head {head}"
        self.linear(self.y.download()[:n], att.reshape(n, HQ * HD).astype(np.float32), self.w_out, self.b_out,
                    what + " output")

    @staticmethod
    def linear(got, x, w, bias, what):
        k = x.shape[1]
        va, vw = value_of(*code_of(x), k), value_of(*code_of(w), k)
        ref = va @ vw.T
        bound = (k / 64 + 2) * 2.0 ** -20 * (np.abs(va) @ np.abs(vw).T)
        if bias is not None:
            ref = ref + bias.astype(np.float64)
            bound = bound * (1 + E) + E * np.abs(ref)
        assert np.all(np.abs(got - ref) <= bound + E * np.abs(ref)), what


def test_prompts_in_chunks_then_single_tokens(ctx):
    layer = Layer(ctx, 300)
    r = np.random.default_rng(3)

    def tokens(n):
        return r.standard_normal((n, WIDTH)).astype(np.float32)

    steps = [{"a": tokens(130)}, {"a": tokens(65), "b": tokens(33)}, {"b": tokens(7), "c": tokens(200)}]
    steps += [{"a": tokens(1), "b": tokens(1), "c": tokens(1)} for _ in range(3)]
    for i, chunks in enumerate(steps):
        say("step", i, {k: len(v) for k, v in chunks.items()})
        n, cu, lens, pos = layer.place(chunks)
        for call in layer.calls(n, len(chunks), int(max(np.diff(cu))), int(max(lens))):
            call()
        layer.check(n, cu, lens, pos, list(chunks), f"step {i}")

    # the decode step as a graph, replayed on new tokens: bit for bit the eager call's
    names = ["a", "b", "c"]
    calls = layer.calls(3, 3, 1, 400)
    n, cu, lens, pos = layer.place({k: tokens(1) for k in names})
    for call in calls:
        call()
    eager = layer.y.download()[:3]
    with D.Graph(ctx) as g:
        for call in calls:
            call()
    D.memset(ctx, layer.y, 0, layer.y.nbytes)
    g.launch()
    assert np.array_equal(layer.y.download()[:3], eager)
    for i in range(3):
        n, cu, lens, pos = layer.place({k: tokens(1) for k in names})
        g.launch()
        layer.check(n, cu, lens, pos, names, f"replay {i}")
        got = layer.y.download()[:3]
        for call in calls:
            call()
        assert np.array_equal(layer.y.download()[:3], got)
    g.close()
    layer.qkv.close()
    layer.out.close()
    layer.cache.close()

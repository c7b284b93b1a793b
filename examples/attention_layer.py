"""The attention half of a transformer block, served: quantized projections,
rotary positions, a paged int8 cache, prompts in chunks, then token by token.

    python examples/attention_layer.py

Two sequences are prefilled (one in two chunks, as a long prompt would be),
then decoded together for a few steps.  Every buffer is a device buffer and
nothing waits for the device in between.  At the end the layer's outputs are
compared with one pass over the whole sequences: the projections are quantized
per token, so both see the same rows, and the difference is the rounding of the
attention's bfloat16 weights and outputs.
"""
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from tokenvector.inference_amd import attention as A  # noqa: E402
from tokenvector.inference_amd import device as D  # noqa: E402


class AttentionLayer:
    """Weights, rotation table and cache of one layer, and its forward pass over
    any mix of chunks and single tokens."""

    def __init__(self, ctx, w_qkv, w_out, heads, heads_kv, head_dim, positions=4096, pages=64, page_size=16):
        self.ctx, self.hq, self.hkv, self.d = ctx, heads, heads_kv, head_dim
        self.width = heads * head_dim
        n = (heads + 2 * heads_kv) * head_dim
        self.qkv = D.QuantizedLinear.from_float(ctx, D.DeviceBuffer.from_host(ctx, w_qkv), n, w_qkv.shape[1])
        self.out = D.QuantizedLinear.from_float(ctx, D.DeviceBuffer.from_host(ctx, w_out), w_out.shape[0],
                                                self.width)
        # long contexts: the low frequencies slowed by two
        self.table = A.rope_table(ctx, positions, A.rope_inv_freq(
            head_dim, factor=2.0, by_parts=True, original_positions=positions // 2))
        self.positions = positions
        self.cache = A.KVCache(ctx, A.I8, pages, page_size, heads_kv, head_dim)
        self.pages, self.page_size = pages, page_size
        self.tables, self.lengths, self.free = {}, {}, list(range(pages))

    def forward(self, chunks):
        """chunks: {sequence: x [tokens, width] f32}.  Returns {sequence: y} after
        appending the tokens to the sequences' caches."""
        ctx, hq, hkv, d = self.ctx, self.hq, self.hkv, self.d
        positions, slots, cu, lens = [], [], [0], []
        for name, x in chunks.items():
            start = self.lengths.get(name, 0)
            pages = self.tables.setdefault(name, [])
            while len(pages) * self.page_size < start + len(x):
                pages.append(self.free.pop())
            at = np.arange(start, start + len(x))
            positions.append(at)
            slots.append(np.array(pages)[at // self.page_size] * self.page_size + at % self.page_size)
            self.lengths[name] = start + len(x)
            cu.append(cu[-1] + len(x))
            lens.append(start + len(x))
        width = max(len(self.tables[name]) for name in chunks)
        table = np.zeros((len(chunks), width), np.int32)
        for i, name in enumerate(chunks):
            table[i, :len(self.tables[name])] = self.tables[name]
        tokens, row = cu[-1], (hq + 2 * hkv) * d

        def put(a, dtype):
            return D.DeviceBuffer.from_host(ctx, np.ascontiguousarray(a, dtype))

        x = put(np.concatenate(list(chunks.values())), np.float32)
        qkv = D.DeviceBuffer.empty(ctx, (tokens, row), np.float32)
        self.qkv.forward(x, tokens, qkv, D.ACT_PER_TOKEN)
        q = D.DeviceBuffer.empty(ctx, (tokens, hq, d), np.uint16)  # bfloat16
        rows = [A.Rows(qkv.ptr + 4 * o * d, row, d) for o in (0, hq, hq + hkv)]
        A.RopeAppend(ctx, A.F32, tokens, hq, hkv, d, *rows, positions=put(np.concatenate(positions), np.int32),
                     table=self.table, table_len=self.positions, rot_dim=d, q_out=A.Rows(q, hq * d, d),
                     type_out=A.BF16, cache=self.cache, slots=put(np.concatenate(slots), np.int64))()
        att = D.DeviceBuffer.empty(ctx, (tokens, hq, d), np.float32)
        A.AttentionPaged(ctx, A.BF16, tokens, hq, self.cache, len(chunks), A.Rows(q, hq * d, d),
                         A.Rows(att, hq * d, d), put(table, np.int32), width, put(lens, np.int32),
                         put(cu, np.int32), max(np.diff(cu)), max(lens), type_out=A.F32)()
        y = D.DeviceBuffer.empty(ctx, (tokens, self.out.n), np.float32)
        self.out.forward(att, tokens, y, D.ACT_PER_TOKEN)
        host = y.download()
        return {name: host[cu[i]:cu[i + 1]] for i, name in enumerate(chunks)}


def main():
    rng = np.random.default_rng(1)
    heads, heads_kv, d = 12, 4, 64
    width = heads * d
    ctx = D.Context(0)
    w_qkv = rng.standard_normal(((heads + 2 * heads_kv) * d, width)).astype(np.float32) * 0.05
    w_out = rng.standard_normal((width, width)).astype(np.float32) * 0.05

    def layer():
        return AttentionLayer(ctx, w_qkv, w_out, heads, heads_kv, d)

    a = rng.standard_normal((205, width)).astype(np.float32)
    b = rng.standard_normal((43, width)).astype(np.float32)
    served, steps = layer(), 5
    got = {"a": [], "b": []}
    chunks = [{"a": a[:128]}, {"a": a[128:200], "b": b[:38]}]
    chunks += [{"a": a[200 + i:201 + i], "b": b[38 + i:39 + i]} for i in range(steps)]
    for chunk in chunks:
        for name, y in served.forward(chunk).items():
            got[name].append(y)
    whole = layer().forward({"a": a, "b": b})
    worst = 0.0
    for name, ys in got.items():
        y = np.concatenate(ys)
        worst = max(worst, float(np.linalg.norm(y - whole[name]) / np.linalg.norm(whole[name])))
        print(f"sequence {name}: {len(y)} tokens in {len(ys)} calls")
    print(f"chunks and single tokens against whole sequences: relative difference {worst:.2e}")
    return worst


if __name__ == "__main__":
    main()

"""A layer of a serving step in which requests share a prompt and adapters,
as the operators are used together: the projection and its adapters, the
rotation and append of a ragged chunk, prefill attention, then decode steps whose
attention reads the shared pages once; run as they come and replayed from a
graph.

Each stage is checked against fp64 from the values that the stage before it left
on the device, so a tolerance covers one stage.  Projection with adapters: the
base is read back, v = x A^T is off by (K + 8) 2^-24 of V = sum |x||a|, taken to
2^-16 of |v|, and (2 rank + 8) 2^-24 of V |b| follow; 2^-8 for the store.
Rotation: 2^-20 of |x1| + |x2|, 2^-8 for the store.  Attention: 2^-8 |o| + 2 2^-8 A
with A = sum_t w_t |V_t|, weights to 2 ((D + 2) 2^-24 of scale sum |q||k| + 2^-18) and
(L + 64) 2^-24."""
import numpy as np
import pytest

from lattice_amd.bindings import KV_BF16, make_config, memcpy_dtoh, memcpy_htod
from lattice_amd.workload import SB, rope_inv_freq

pytestmark = pytest.mark.gpu

U = 2.0 ** -8
HIDDEN, HQ, HKV, D, BS, RANK = 512, 8, 2, 128, 16, 16
QKV = (HQ + 2 * HKV) * D
ENDS = [HQ * D, (HQ + HKV) * D, QKV]
GROUPS, PROMPTS, STEPS = [3, 2, 4], [203, 64, 37], 6      # sequences and tokens of each prompt
ADAPTER = [1, -1, 0]                                      # of the groups' requests


def f64(t):
    return t.double().cpu().numpy()


class Layer:
    def __init__(self, torch, lib):
        self.torch, self.lib = torch, lib
        g = torch.Generator().manual_seed(11)
        rnd = lambda *s: torch.randn(*s, generator=g).bfloat16().cuda()  # noqa: E731
        self.batch = sum(GROUPS)
        cfg = make_config(num_layers=1, kv_heads=HKV, head_dim=D, max_batch=self.batch, max_seq_len=512,
                          block_size=BS)
        self.pool = lib.create_pool(cfg, KV_BF16)
        self.w, self.a, self.b = rnd(QKV, HIDDEN), rnd(2, 3 * RANK, HIDDEN) / 16, rnd(2, QKV, RANK)
        self.wo, self.oa, self.ob = rnd(HIDDEN, HQ * D), rnd(2, RANK, HQ * D) / 16, rnd(2, HIDDEN, RANK)
        self.s = torch.tensor([0.5, 0.25], device="cuda")
        self.inv = rope_inv_freq(10000.0, D)
        self.inv_dev = torch.from_numpy(self.inv).cuda()
        self.mbps = 16
        ids = list(np.random.default_rng(2).permutation(self.pool.alloc_blocks(18 + 9 * 2)))
        self.offs = np.asarray(self.pool.all_block_offsets_f16(), np.int64)
        self.offs_dev = torch.from_numpy(self.offs).cuda()
        self.nbytes = self.pool.stats()["superblock_count"] * SB
        for base in (self.pool.va_k(0), self.pool.va_v(0)):
            memcpy_htod(base, np.full(self.nbytes, 0xFF, np.uint8))
        self.bt = np.zeros((self.batch, self.mbps), np.int32)
        self.lead, self.adapter, self.shared = [], [], []
        row = 0
        for n, t, a in zip(GROUPS, PROMPTS, ADAPTER):
            whole, lead = t // BS, row
            blocks = [ids.pop() for _ in range(whole)]
            for _ in range(n):
                # the prompt's whole blocks are the group's, the block that it ends in is
                # each sequence's own
                self.bt[row, :whole] = blocks
                for i in range(whole, whole + 2):
                    self.bt[row, i] = ids.pop()
                self.lead.append(lead)
                self.adapter.append(a)
                self.shared.append(t)
                row += 1
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        self.bt_dev, self.ids_dev, self.sh_dev = i32(self.bt), i32(self.adapter), i32(self.shared)
        self.gs_dev = i32(np.concatenate([[0], np.cumsum(GROUPS)]))
        self.lens = i32(self.shared)
        self.one_each = i32(np.arange(self.batch + 1))
        self.scratch = torch.empty(self.pool.shared_scratch_bytes(self.batch, HQ, self.mbps), dtype=torch.uint8,
                                   device="cuda")
        self.new = lambda *s: torch.full(s, 7.0, dtype=torch.bfloat16, device="cuda")
        self.x = rnd(self.batch, HIDDEN) / 32
        self.step_out = [self.new(self.batch, n) for n in (QKV, QKV, HQ * D, HQ * D, HIDDEN, HIDDEN)]
        self.low = torch.empty(1000, 3 * RANK, device="cuda")
        self.rnd, self.i32 = rnd, i32
        torch.cuda.synchronize()

    def add(self, x, base, y, ids, a, b, ends, m, n, k, stream):
        self.lib.lora_add_bf16(x.data_ptr(), a.data_ptr(), b.data_ptr(), ids.data_ptr(), self.low.data_ptr(),
                               base.data_ptr(), y.data_ptr(), m, n, k, adapters=2, rank=RANK, slice_ends=ends,
                               scales_ptr=self.s.data_ptr(), stream_ptr=stream)

    def append(self, qkv, q, bt, lens, qsl, batch, total, stream):
        self.pool.rope_append_chunk(
            layer_idx=0, qkv_ptr=qkv.data_ptr(), q_out_ptr=q.data_ptr(), block_tables_ptr=bt.data_ptr(),
            seq_lens_ptr=lens.data_ptr(), query_start_loc_ptr=qsl.data_ptr(),
            block_offsets_f16_ptr=self.offs_dev.data_ptr(), inv_freq_ptr=self.inv_dev.data_ptr(), batch=batch,
            total_query_tokens=total, num_q_heads=HQ, max_blocks_per_seq=self.mbps, stream_ptr=stream)

    def step(self):
        """A token of every sequence."""
        st = self.torch.cuda.current_stream().cuda_stream
        base, qkv, q, att, obase, out = self.step_out
        m = self.batch
        self.lens.add_(1)
        self.lib.gemm_bf16(self.x.data_ptr(), self.w.data_ptr(), base.data_ptr(), m, QKV, HIDDEN, st)
        self.add(self.x, base, qkv, self.ids_dev, self.a, self.b, ENDS, m, QKV, HIDDEN, st)
        self.append(qkv, q, self.bt_dev, self.lens, self.one_each, m, m, st)
        self.pool.paged_attn_decode_shared(
            layer_idx=0, query_ptr=q.data_ptr(), out_ptr=att.data_ptr(), block_tables_ptr=self.bt_dev.data_ptr(),
            seq_lens_ptr=self.lens.data_ptr(), shared_lens_ptr=self.sh_dev.data_ptr(),
            group_starts_ptr=self.gs_dev.data_ptr(), block_offsets_f16_ptr=self.offs_dev.data_ptr(),
            scratch_ptr=self.scratch.data_ptr(), scratch_bytes=self.scratch.numel(), batch=m,
            num_groups=len(GROUPS), num_q_heads=HQ, kv_heads=HKV, head_dim=D, block_size=BS,
            max_blocks_per_seq=self.mbps, scale=D ** -0.5, stream_ptr=st)
        self.lib.gemm_bf16(att.data_ptr(), self.wo.data_ptr(), obase.data_ptr(), m, HIDDEN, HQ * D, st)
        self.add(att, obase, out, self.ids_dev, self.oa, self.ob, [HIDDEN], m, HIDDEN, HQ * D, st)
        self.x.copy_(out / 512)       # the next token's input

    # -- fp64 of a stage ----------------------------------------------------------------------------
    def check_add(self, x, base, y, ids, a, b, ends):
        x, base, y, a, b, s = f64(x), f64(base), f64(y), f64(a), f64(b), f64(self.s)
        for t, i in enumerate(ids):
            if i < 0:
                assert np.array_equal(y[t], base[t])
                continue
            v, size, start = a[i] @ x[t], np.abs(a[i]) @ np.abs(x[t]), 0
            for j, end in enumerate(ends):
                r, w = slice(j * RANK, (j + 1) * RANK), b[i, start:end]
                exact = base[t, start:end] + s[i] * (w @ v[r])
                err = s[i] * ((x.shape[1] + 2 * RANK + 16) * 2.0 ** -24 * (np.abs(w) @ size[r]) +
                              2.0 ** -16 * (np.abs(w) @ np.abs(v[r]))) + 2.0 ** -23 * np.abs(exact)
                assert np.all(np.abs(y[t, start:end] - exact) <= U * np.abs(exact) + (1 + U) * err), (t, j)
                start = end

    def pages(self):
        """K and V as stored, fp64 [block id][BS][HKV][D]."""
        out = []
        for base in (self.pool.va_k(0), self.pool.va_v(0)):
            raw = memcpy_dtoh(base, self.nbytes).view(np.uint16)
            blocks = np.stack([raw[o:o + BS * HKV * D] for o in self.offs])
            out.append((blocks.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
                       .reshape(-1, BS, HKV, D))
        return out

    def check_append(self, qkv, q, rows):
        """rows: (row of qkv, sequence, place)."""
        qkv, q = f64(qkv).reshape(-1, HQ + 2 * HKV, D), f64(q).reshape(-1, HQ, D)
        k, v = self.pages()
        for t, b, place in rows:
            at = self.bt[b, place // BS], place % BS
            assert np.array_equal(v[at], qkv[t, HQ + HKV:])
            ang = place * self.inv.astype(np.float64)
            x, h = qkv[t, :HQ + HKV], D // 2
            exact = np.concatenate([x[:, :h] * np.cos(ang) - x[:, h:] * np.sin(ang),
                                    x[:, h:] * np.cos(ang) + x[:, :h] * np.sin(ang)], 1)
            size = np.tile(np.abs(x[:, :h]) + np.abs(x[:, h:]), 2)
            got = np.concatenate([q[t], k[at]])
            assert np.all(np.abs(got - exact) <= U * np.abs(exact) + (1 + U) * 2.0 ** -20 * size), (t, b, place)

    def check_attention(self, q, out, rows):
        """rows: (row of q, sequence, tokens that it sees)."""
        q, out = f64(q).reshape(-1, HQ, D), f64(out).reshape(-1, HQ, D)
        k, v = self.pages()
        for t, b, n in rows:
            kb, vb = (x[self.bt[b]].reshape(-1, HKV, D)[:n] for x in (k, v))
            for h in range(HQ):
                kh, vh = kb[:, h * HKV // HQ], vb[:, h * HKV // HQ]
                z, size = kh @ q[t, h] * D ** -0.5, np.abs(kh) @ np.abs(q[t, h]) * D ** -0.5
                w = np.exp(z - z.max())
                w /= w.sum()
                o, a = w @ vh, w @ np.abs(vh)
                delta = 2 * ((D + 2) * 2.0 ** -24 * size.max() + 2.0 ** -18)
                assert np.all(np.abs(out[t, h] - o) <= U * np.abs(o) + (2 * U + delta + (n + 64) * 2.0 ** -24) * a), \
                    (t, b, h)

    def prompts(self):
        """The groups' prompts in one ragged chunk, through the first sequence of each; then
        the others' copies of the blocks in which they end."""
        torch, total = self.torch, sum(PROMPTS)
        first = np.concatenate([[0], np.cumsum(GROUPS)])[:-1]
        qsl = np.concatenate([[0], np.cumsum(PROMPTS)])
        ids = np.repeat(ADAPTER, PROMPTS)
        x, base = self.rnd(total, HIDDEN) / 32, self.new(total, QKV)
        qkv, q, att = self.new(total, QKV), self.new(total, HQ * D), self.new(total, HQ * D)
        bt, lens, qsl_dev = self.i32(self.bt[first]), self.i32(PROMPTS), self.i32(qsl)
        ids_dev = self.i32(ids)
        torch.cuda.synchronize()
        self.lib.gemm_bf16(x.data_ptr(), self.w.data_ptr(), base.data_ptr(), total, QKV, HIDDEN, 0)
        self.add(x, base, qkv, ids_dev, self.a, self.b, ENDS, total, QKV, HIDDEN, 0)
        self.append(qkv, q, bt, lens, qsl_dev, len(PROMPTS), total, 0)
        self.pool.paged_attn_prefill(
            layer_idx=0, query_ptr=q.data_ptr(), out_ptr=att.data_ptr(), block_tables_ptr=bt.data_ptr(),
            seq_lens_ptr=lens.data_ptr(), query_start_loc_ptr=qsl_dev.data_ptr(),
            block_offsets_f16_ptr=self.offs_dev.data_ptr(), batch=len(PROMPTS), total_query_tokens=total,
            num_q_heads=HQ, kv_heads=HKV, head_dim=D, block_size=BS, max_blocks_per_seq=self.mbps,
            scale=D ** -0.5, stream_ptr=0)
        torch.cuda.synchronize()
        self.check_add(x, base, qkv, ids, self.a, self.b, ENDS)
        rows = [(qsl[i] + t, first[i], t) for i, n in enumerate(PROMPTS) for t in range(n)]
        self.check_append(qkv, q, rows)
        self.check_attention(q, att, [(t, b, place + 1) for t, b, place in rows[::7]])
        for base in (self.pool.va_k(0), self.pool.va_v(0)):
            raw, size = memcpy_dtoh(base, self.nbytes), BS * HKV * D * 2
            for b in range(self.batch):
                if b != self.lead[b]:
                    src, dst = (int(self.offs[self.bt[s, self.shared[b] // BS]]) * 2 for s in (self.lead[b], b))
                    raw[dst:dst + size] = raw[src:src + size]
            memcpy_htod(base, raw)

    def check_step(self, x, place):
        base, qkv, q, att, obase, out = self.step_out
        self.check_add(x, base, qkv, self.adapter, self.a, self.b, ENDS)
        self.check_append(qkv, q, [(b, b, self.shared[b] + place) for b in range(self.batch)])
        self.check_attention(q, att, [(b, b, self.shared[b] + place + 1) for b in range(self.batch)])
        self.check_add(att, obase, out, self.adapter, self.oa, self.ob, [HIDDEN])


def test_prompts_then_steps(gpu_lib):
    import torch
    layer = Layer(torch, gpu_lib)
    try:
        layer.prompts()
        start = [memcpy_dtoh(base, layer.nbytes) for base in (layer.pool.va_k(0), layer.pool.va_v(0))]
        x0, lens0, seen = layer.x.clone(), layer.lens.clone(), []
        for i in range(STEPS):
            x = layer.x.clone()
            layer.step()
            torch.cuda.synchronize()
            layer.check_step(x, i)
            seen.append([t.clone() for t in layer.step_out])
        # the same steps from a graph, on another stream, with eager work between replays
        graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):   # the projection's workspace is allocated by a first call
            layer.step()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            layer.step()
        for _ in range(2):
            layer.x.copy_(x0)
            layer.lens.copy_(lens0)
            for base, raw in zip((layer.pool.va_k(0), layer.pool.va_v(0)), start):
                memcpy_htod(base, raw)
            torch.cuda.synchronize()
            for i in range(STEPS):
                for t in layer.step_out:
                    t.fill_(7.0)
                layer.scratch.fill_(0xFF)
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(a, b) for a, b in zip(layer.step_out, seen[i])), i
    finally:
        layer.pool.destroy()

"""Decode attention of groups that share a prefix
(kcmm_paged_attn_decode_shared) on the GPU against fp64.

What a sequence may not read is poisoned: the entries of its own table for
blocks wholly below its shared length name a page of NaN, and so is every slot
behind a sequence's end.

Tolerance of an output o = sum_t w_t V_t with A = sum_t w_t |V_t| (weights that
add up to 1): the store rounds by u |o| (u: half a step, eps / 2 of the type);
the weights are rounded to the 16-bit type before the product, u A, and their
sum may be that of the unrounded ones, u A again; a score is off by at most
(D + 2) roundings of 2^-24 of scale sum |q||k|, and its exponent's argument and
the instruction by 2^-18 (|argument| <= 64 here), which change a weight by that
factor, twice (numerator and sum): delta; and sums of L terms and of the parts
by (L + 64) 2^-24."""
import math

import numpy as np
import pytest

import oracle as O
from lattice_amd.bindings import KV_BF16, KV_F16, KV_F32, KV_FP8, make_config, memcpy_htod
from lattice_amd.workload import SB, io_dtype, torch_io_dtype

pytestmark = pytest.mark.gpu

HALF_STEP = {KV_BF16: 2.0 ** -8, KV_FP8: 2.0 ** -8, KV_F16: 2.0 ** -11, KV_F32: 2.0 ** -24}


class Case:
    """`groups`: a list of lists of (shared, total) per sequence; `before` and
    `behind`: totals of sequences that lie in no group."""

    def __init__(self, torch, lib, dtype, hq, hkv, d, bs, groups, before=(), behind=(), seed=0,
                 scale=None, q_scale=1.0, lie=False):
        rng = np.random.default_rng(seed)
        self.torch, self.dtype = torch, dtype
        self.hq, self.hkv, self.d, self.bs = hq, hkv, d, bs
        self.scale = 1.0 / math.sqrt(d) if scale is None else scale
        seqs = [(7, t, None) for t in before]          # a shared length that means nothing
        starts = [len(seqs)]
        for g in groups:
            lead = len(seqs)
            seqs += [(s, t, lead) for s, t in g]
            starts.append(len(seqs))
        seqs += [(7, t, None) for t in behind]
        self.batch, self.starts = len(seqs), starts
        self.totals = [t for _, t, _ in seqs]
        self.shared = [s for s, _, _ in seqs]
        # tokens that each table has to hold: its own, and of a group's first
        # sequence what the others read there
        need = [max(t, 0) for t in self.totals]
        for s, t, lead in seqs:
            if lead is not None:
                need[lead] = max(need[lead], min(s, max(t, 0)) // bs * bs)
        self.mbps = max(1, max(-(-n // bs) for n in need))
        blocks = [-(-n // bs) for n in need]
        cfg = make_config(num_layers=1, kv_heads=hkv, head_dim=d, max_batch=self.batch,
                          max_seq_len=max(self.mbps * bs, (sum(blocks) + 2) * bs // self.batch + bs),
                          block_size=bs)
        self.pool = lib.create_pool(cfg, dtype)
        ids = []
        while len(ids) < sum(blocks) + 1:
            ids += self.pool.alloc_blocks(min(1024, sum(blocks) + 1 - len(ids)))
        poison, ids = ids[0], list(rng.permutation(ids[1:]))
        st = self.pool.stats()
        offs = np.asarray(self.pool.all_block_offsets_f16(), np.uint64)
        esize = {KV_FP8: 1, KV_F32: 4}.get(dtype, 2)
        row = hkv * d * esize
        regions = [np.full(st["superblock_count"] * SB, 0xFF, np.uint8) for _ in range(2)]   # NaN of any type
        table = np.full((self.batch, self.mbps), poison, np.int32)
        dense = []
        for b, (s, t, lead) in enumerate(seqs):
            first = 0 if lead in (None, b) else max(0, min(s, t)) // bs * bs     # own tokens from here on
            n = need[b]
            kv = []
            for _ in range(2):
                x = rng.standard_normal((blocks[b] * bs, hkv, d)).astype(np.float32)
                kv.append(x)
            stored = [np.zeros((n, hkv, d)) for _ in range(2)]
            for lb in range(first // bs, blocks[b]):
                table[b, lb] = ids.pop()
                page = int(offs[table[b, lb]]) * 2
                lo, hi = max(first - lb * bs, 0), min(n - lb * bs, bs)
                for reg, x, out in zip(regions, kv, stored):
                    blk = x[lb * bs:(lb + 1) * bs]
                    if dtype == KV_FP8:
                        sc = (np.abs(blk).max(axis=(0, 2)) / np.float32(448)).astype(np.float32)
                        enc = O.encode(O.FP8, blk / sc[None, :, None])
                        val = O.decode(O.FP8, enc).astype(np.float64) * sc[None, :, None]
                        reg[page + row * bs:page + row * bs + 4 * hkv] = sc.view(np.uint8)
                    else:
                        code = {KV_BF16: O.BF16, KV_F16: O.F16, KV_F32: O.F32}[dtype]
                        enc = O.encode(code, blk)
                        val = O.decode(code, enc)
                    raw = np.ascontiguousarray(enc).view(np.uint8).reshape(bs, row)
                    reg[page + lo * row:page + hi * row] = raw[lo:hi].reshape(-1)
                    out[lb * bs + lo:lb * bs + hi] = val[lo:hi]
            if first:
                for mine, theirs in zip(stored, dense[lead]):
                    mine[:first] = theirs[:first]
            dense.append(stored)
        self.dense = dense
        for reg, base in zip(regions, (self.pool.va_k(0), self.pool.va_v(0))):
            memcpy_htod(base, reg)
        q = (q_scale * rng.standard_normal((self.batch, hq, d))).astype(np.float32)
        qdt = {KV_BF16: O.BF16, KV_FP8: O.BF16, KV_F16: O.F16, KV_F32: O.F32}[dtype]
        qe = O.encode(qdt, q)
        self.q = O.decode(qdt, qe).astype(np.float64)
        tdt = torch_io_dtype(dtype)
        qt = torch.from_numpy(qe.copy()) if dtype == KV_F32 else \
            torch.from_numpy(qe.view(np.int16).copy()).view(tdt)
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        self.dev = dict(q=qt.cuda(), bt=i32(table), sl=i32(self.totals), sh=i32(self.shared),
                        gs=i32(starts), offs=torch.from_numpy(offs.view(np.int64)).cuda())
        self.out = torch.full((self.batch, hq, d), float("nan"), dtype=tdt, device="cuda")
        self.scratch = self.new_scratch()

    def new_scratch(self):
        n = self.pool.shared_scratch_bytes(self.batch, self.hq, self.mbps)
        return self.torch.full((n,), 0xFF, dtype=self.torch.uint8, device="cuda")

    def run(self, stream=None, out=None, scratch=None, batch=None):
        d, out = self.dev, self.out if out is None else out
        scratch = self.scratch if scratch is None else scratch
        self.pool.paged_attn_decode_shared(
            layer_idx=0, query_ptr=d["q"].data_ptr(), out_ptr=out.data_ptr(),
            block_tables_ptr=d["bt"].data_ptr(), seq_lens_ptr=d["sl"].data_ptr(),
            shared_lens_ptr=d["sh"].data_ptr(), group_starts_ptr=d["gs"].data_ptr(),
            block_offsets_f16_ptr=d["offs"].data_ptr(), scratch_ptr=scratch.data_ptr(),
            scratch_bytes=scratch.numel(), batch=self.batch, num_groups=len(self.starts) - 1,
            num_q_heads=self.hq, kv_heads=self.hkv, head_dim=self.d, block_size=self.bs,
            max_blocks_per_seq=self.mbps, scale=self.scale,
            stream_ptr=self.torch.cuda.current_stream().cuda_stream if stream is None else stream)

    def check(self, out=None):
        got = (self.out if out is None else out).double().cpu().numpy()
        u = HALF_STEP[self.dtype]
        u16 = 0.0 if self.dtype == KV_F32 else u
        for b, n in enumerate(self.totals):
            if n <= 0:
                assert not got[b].any(), b
                continue
            k, v = (x[:n] for x in self.dense[b])
            for h in range(self.hq):
                g = h * self.hkv // self.hq
                z = k[:, g] @ self.q[b, h] * self.scale
                size = np.abs(k[:, g]) @ np.abs(self.q[b, h]) * abs(self.scale)
                w = np.exp(z - z.max())
                w /= w.sum()
                o, a = w @ v[:, g], w @ np.abs(v[:, g])
                assert np.abs(z - z.max())[w > 2.0 ** -60].max() <= 64
                delta = 2 * ((self.d + 2) * 2.0 ** -24 * size.max() + 2.0 ** -18)
                tol = u * np.abs(o) + (2 * u16 + delta + (n + 64) * 2.0 ** -24) * a
                off = np.abs(got[b, h] - o)
                assert np.all(off <= tol), (b, h, n, float(np.max(off / tol)))

    def close(self):
        self.pool.destroy()


def check(torch, lib, *args, **kw):
    c = Case(torch, lib, *args, **kw)
    try:
        c.run()
        torch.cuda.synchronize()
        c.check()
    finally:
        c.close()


ALL = [KV_BF16, KV_F16, KV_FP8, KV_F32]
HEADS = [(32, 8, 128, 16), (8, 8, 64, 16), (16, 4, 64, 32), (4, 4, 128, 8), (16, 1, 128, 16),
         (12, 4, 128, 24), (10, 2, 64, 16)]
OTHER = [(6, 3, 80, 16), (7, 3, 64, 16), (4, 2, 256, 16), (8, 2, 128, 5), (40, 2, 64, 8), (4, 4, 36, 4)]
GROUP = [(100, 133), (100, 101), (100, 164), (100, 100)]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hq,hkv,d,bs", HEADS + OTHER)
def test_head_layouts(gpu_lib, dtype, hq, hkv, d, bs):
    import torch
    check(torch, gpu_lib, dtype, hq, hkv, d, bs, [GROUP, [(37, 70)]], seed=d + hq)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("groups", [
    [[(0, 1)]], [[(1, 1)]], [[(1, 2), (1, 1)]], [[(0, 33), (0, 40)]],   # one token; nothing shared
    [[(64, 64), (64, 64), (64, 64)]],                                     # everything shared
    [[(90, 50), (90, 120), (90, 20), (90, 90)]],                          # shorter than the prefix
    [[(48, 0), (48, 60), (48, -3), (48, 49)], [(0, 0)], [(5, 0), (5, 9)]],  # sequences without tokens
    [[(17, 50), (3, 60), (0, 5), (33, 33), (16, 80), (-4, 12)]],          # each another length
    [[(200, 200), (199, 231), (7, 300), (193, 194)]],
    [[(31, 32), (31, 47)], [(8, 9), (8, 8)], [(15, 16), (15, 17)], [(40, 41), (40, 72)]],
])
def test_lengths(gpu_lib, dtype, groups):
    import torch
    check(torch, gpu_lib, dtype, 8, 2, 128, 16, groups, seed=len(groups))


@pytest.mark.parametrize("dtype", [KV_BF16, KV_FP8])
def test_groups(gpu_lib, dtype):
    """Empty groups, sequences in front of and behind them all, more groups and
    sequences than a wave has lanes."""
    import torch
    rng = np.random.default_rng(5)
    pairs = [[(int(s), int(s + rng.integers(0, 40))) for _ in range(2)] for s in rng.integers(1, 90, 70)]
    check(torch, gpu_lib, dtype, 8, 2, 128, 16, [[], [(20, 30), (20, 45)], [], [(64, 70)], []],
          before=(19, 0), behind=(40, 3))
    check(torch, gpu_lib, dtype, 8, 2, 128, 16, pairs, behind=(11,))
    many = [(120, int(t)) for t in rng.integers(110, 180, 150)]
    check(torch, gpu_lib, dtype, 8, 2, 128, 16, [many])
    check(torch, gpu_lib, dtype, 8, 2, 128, 16, [many[:67], many[67:70], [], many[70:]], before=(1,))


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (4, 4, 128), (8, 1, 64), (16, 2, 64)])
def test_long_prefix(gpu_lib, dtype, hq, hkv, d):
    """Prefixes that are split over workgroups, rests that are too, and both of
    one token."""
    import torch
    if dtype == KV_FP8 and d == 64:
        d = 128
    check(torch, gpu_lib, dtype, hq, hkv, d, 16,
          [[(3001, 3002), (3001, 3100), (3001, 3001), (2500, 5000)], [(1, 2600)], [(1999, 2000)] * 3])
    check(torch, gpu_lib, dtype, hq, hkv, d, 16, [[(4100, 4100 + 9 * i) for i in range(33)]])


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (6, 3, 80)])
def test_scales(gpu_lib, dtype, hq, hkv, d):
    """A negative scale, none at all, and scores far from zero."""
    import torch
    for scale, qs in ((-0.1, 1.0), (0.0, 1.0), (0.3, 1.2)):
        check(torch, gpu_lib, dtype, hq, hkv, d, 16, [GROUP, [(300, 340), (300, 301)]], scale=scale, q_scale=qs)


@pytest.mark.parametrize("dtype", [KV_BF16, KV_FP8])
def test_scores_of_one_sign(gpu_lib, dtype):
    """Every score far below zero, or far above: the parts' maxima are no 0."""
    import torch
    for sign in (1.0, -1.0):
        c = Case(torch, gpu_lib, dtype, 8, 2, 128, 16, [[(500, 520), (500, 500)], [(40, 90)]], scale=0.0)
        try:
            # K of one value, q of one value: all scores equal, 2^7 * sign apart from 0
            kreg = torch.zeros(c.pool.stats()["superblock_count"] * SB, dtype=torch.uint8, device="cuda")
            if dtype == KV_FP8:
                kreg.fill_(0x38)                       # 1.0; the scales are 1.0 too
                flat = kreg.cpu().numpy()
                for off in np.asarray(c.pool.all_block_offsets_f16(), np.int64) * 2:
                    at = int(off) + 16 * 2 * 128
                    flat[at:at + 8] = np.ones(2, np.float32).view(np.uint8)
            else:
                flat = np.tile(np.array([0x80, 0x3F], np.uint8), kreg.numel() // 2)
            memcpy_htod(c.pool.va_k(0), flat)
            c.dev["q"].fill_(sign)
            c.scale = 1.0
            c.run()
            torch.cuda.synchronize()
            c.scale = 0.0                               # equal weights
            c.check()
        finally:
            c.close()


def test_forked_beams(gpu_lib):
    """Groups as kcmm_fork_beams makes them, against the decode attention that
    reads every sequence by itself: same weights, other parts."""
    import torch
    hq, hkv, d, bs, ctx, width = 32, 8, 128, 16, [700, 333, 48], 4
    cfg = make_config(num_layers=1, kv_heads=hkv, head_dim=d, max_batch=12, max_seq_len=1024, block_size=bs)
    pool = gpu_lib.create_pool(cfg, KV_BF16)
    try:
        n = pool.alloc_blocks(len(ctx) * 45)
        parents = []
        for i, t in enumerate(ctx):
            blocks = n[i * 45:i * 45 + -(-(t + 1) // bs)]
            parents.append(pool.register_sequence(blocks))
            pool.update_seq_len(parents[-1], t)
        nbytes = pool.stats()["superblock_count"] * SB
        g = torch.Generator().manual_seed(3)
        for base in (pool.va_k(0), pool.va_v(0)):
            memcpy_htod(base, torch.randn(nbytes // 2, generator=g).bfloat16().view(torch.int16).numpy())
        kids, _ = pool.fork_beams(parents, width)
        rows = [s for i, p in enumerate(parents) for s in [p] + kids[i * (width - 1):(i + 1) * (width - 1)]]
        # a token of its own for every beam, in the page made private for it
        mbps = 45
        bt = np.zeros((len(rows), mbps), np.int32)
        for r, s in enumerate(rows):
            t = pool.block_table(s)
            bt[r, :len(t)] = t
        slots = [int(bt[r, ctx[r // width] // bs]) * bs + ctx[r // width] % bs for r in range(len(rows))]
        kv = [torch.randn(len(rows), hkv * d, generator=g).bfloat16().cuda() for _ in range(2)]
        pool.append_kv_slots(0, slots, kv[0].data_ptr(), kv[1].data_ptr())
        torch.cuda.synchronize()
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        total = [ctx[r // width] + 1 for r in range(len(rows))]
        dev = dict(bt=i32(bt), sl=i32(total), sh=i32([t - 1 for t in total]), gs=i32([0, 4, 8, 12]),
                   offs=torch.tensor(pool.all_block_offsets_f16(), dtype=torch.int64, device="cuda"))
        q = torch.randn(len(rows), hq, d, generator=g).bfloat16().cuda()
        one, two = torch.empty_like(q), torch.empty_like(q)
        scratch = torch.empty(pool.shared_scratch_bytes(12, hq, mbps), dtype=torch.uint8, device="cuda")
        common = dict(layer_idx=0, query_ptr=q.data_ptr(), block_tables_ptr=dev["bt"].data_ptr(),
                      seq_lens_ptr=dev["sl"].data_ptr(), block_offsets_f16_ptr=dev["offs"].data_ptr(),
                      batch=12, num_q_heads=hq, kv_heads=hkv, head_dim=d, block_size=bs,
                      max_blocks_per_seq=mbps, scale=d ** -0.5, stream_ptr=0)
        torch.cuda.synchronize()
        pool.paged_attn_decode(out_ptr=one.data_ptr(), **common)
        pool.paged_attn_decode_shared(out_ptr=two.data_ptr(), shared_lens_ptr=dev["sh"].data_ptr(),
                                      group_starts_ptr=dev["gs"].data_ptr(), num_groups=3,
                                      scratch_ptr=scratch.data_ptr(), scratch_bytes=scratch.numel(), **common)
        torch.cuda.synchronize()
        # each is within 2^-8 |o| + 2 * 2^-8 A of the same value, A <= max |V| < 6
        assert float((one.float() - two.float()).abs().max()) <= 2 * 3 * 2.0 ** -8 * 6
        assert float((one.float() - two.float()).norm() / one.float().norm()) < 2 * 2.0 ** -8
    finally:
        pool.destroy()


@pytest.mark.parametrize("dtype", [KV_BF16, KV_FP8, KV_F32])
def test_graph_replays(gpu_lib, dtype):
    """Captured at once, with no warm-up; every replay and the eager calls
    between them give the same bits."""
    import torch
    c = Case(torch, gpu_lib, dtype, 8, 2, 128, 16, [[(600, 600 + 37 * i) for i in range(9)], [(50, 51)]])
    try:
        st = torch.cuda.Stream()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            c.run()
        first = None
        for _ in range(4):
            c.out.fill_(float("nan"))
            c.scratch.fill_(0xFF)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            c.check()
            first = c.out.clone() if first is None else first
            assert torch.equal(c.out, first)
            c.out.fill_(float("nan"))
            c.run()
            torch.cuda.synchronize()
            assert torch.equal(c.out, first)
    finally:
        c.close()


def test_two_graphs_and_two_streams_at_once(gpu_lib):
    """Calls with scratch of their own, captured from one stream, replayed on
    two, beside an eager call on a third."""
    import torch
    cs = [Case(torch, gpu_lib, KV_BF16, 8, 2, 128, 16, [[(900, 900 + 11 * i) for i in range(n)]], seed=n)
          for n in (12, 20, 7)]
    try:
        st, graphs = torch.cuda.Stream(), []
        torch.cuda.synchronize()
        for c in cs[:2]:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=st):
                c.run()
            graphs.append(g)
        sides = [torch.cuda.Stream() for _ in cs]
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s in zip(graphs, sides):
                with torch.cuda.stream(s):
                    g.replay()
            cs[2].run(stream=sides[2].cuda_stream)
        torch.cuda.synchronize()
        for c in cs:
            c.check()
    finally:
        for c in cs:
            c.close()


def test_scratch_is_enough(gpu_lib):
    """Nothing is written behind the bytes that the size call names."""
    import torch
    for groups in ([[(2000, 2000 + i) for i in range(40)]], [[(300, 400)] * 2] * 30, [[(0, 4000)]]):
        c = Case(torch, gpu_lib, KV_BF16, 8, 2, 128, 16, groups)
        try:
            n = c.scratch.numel()
            whole = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
            c.run(scratch=whole[:n])
            torch.cuda.synchronize()
            assert bool((whole[n:] == 0x5A).all())
            c.check()
        finally:
            c.close()


@pytest.mark.parametrize("dtype,hq,hkv,d", [(KV_BF16, 8, 2, 128), (KV_FP8, 4, 4, 128), (KV_F16, 4, 2, 64),
                                            (KV_BF16, 2, 2, 80)])
def test_large_batches(gpu_lib, dtype, hq, hkv, d):
    """More sequences than one launch takes: groups that go on into the next,
    or over more than one, with sequences of no group around them."""
    import torch
    rng = np.random.default_rng(9)

    def some(n, s):
        return [(s, int(s + t)) for t in rng.integers(-s // 2, 40, n)]

    check(torch, gpu_lib, dtype, hq, hkv, d, 16, [some(120, 100), some(250, 170), [], some(180, 33)],
          before=(5, 0, 40), behind=(17,) * 20)
    check(torch, gpu_lib, dtype, hq, hkv, d, 16, [some(600, 130)])
    check(torch, gpu_lib, dtype, hq, hkv, d, 16, [some(256, 64), some(1, 90), some(255, 64), some(2, 64)])


def test_scratch_of_large_batches(gpu_lib):
    """As many bytes as the size call names are enough, for any number of
    sequences."""
    import torch
    c = Case(torch, gpu_lib, KV_BF16, 16, 1, 128, 16, [[(64, 64 + i % 50) for i in range(520)]])
    try:
        n = c.scratch.numel()
        whole = torch.full((n + 4096,), 0x5A, dtype=torch.uint8, device="cuda")
        c.run(scratch=whole[:n])
        torch.cuda.synchronize()
        assert bool((whole[n:] == 0x5A).all())
        c.check()
    finally:
        c.close()

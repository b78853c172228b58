"""Rotation and append of chunks (kcmm_rope_append_chunk) on the GPU against
fp64.

A rotated value y = x1 cos - x2 sin has cos and sin off by 2^-21 each (the angle
2^-22, the functions and their rounding below that; positions past 2^27: 2^-20)
and two fp32 operations: TRIG = 2^-20 of |x1| + |x2| covers all, then one
rounding to the type, half a step.  v is copied: bit for bit.  On fp8 pages the
scale is amax / 448 of such values, and a code is the nearest to the value over
the stored scale, half an e4m3 step (2^-4 of it, 2^-10 of the scale among the
subnormals)."""
import numpy as np
import pytest

import oracle as O
from lattice_amd.bindings import (KV_BF16, KV_F16, KV_F32, KV_FP8, make_config, memcpy_dtoh,
                                  memcpy_htod)
from lattice_amd.workload import SB, rope_inv_freq, torch_io_dtype
from tests import e4m3 as E

pytestmark = pytest.mark.gpu

TRIG = 2.0 ** -20
HALF_STEP = {KV_BF16: 2.0 ** -8, KV_FP8: 2.0 ** -8, KV_F16: 2.0 ** -11, KV_F32: 2.0 ** -24}
TINY = {KV_BF16: 2.0 ** -134, KV_FP8: 2.0 ** -134, KV_F16: 2.0 ** -25, KV_F32: 2.0 ** -150}
CODE = {KV_BF16: O.BF16, KV_FP8: O.BF16, KV_F16: O.F16, KV_F32: O.F32}


class Case:
    """`chunks`: (tokens, length with them) per sequence.  Pages hold a pattern
    (fp8: codes and scales) before the call."""

    def __init__(self, torch, lib, dtype, hq, hkv, d, bs, chunks, positions=None, axes=None, pad=0,
                 mbps=None, seed=0, x=None, theta=10000.0):
        rng = np.random.default_rng(seed)
        self.torch, self.dtype = torch, dtype
        self.hq, self.hkv, self.d, self.bs, self.chunks = hq, hkv, d, bs, chunks
        self.positions, self.axes = positions, axes
        self.mbps = mbps or max(1, max(-(-L // bs) for _, L in chunks))
        need = [min(max(0, -(-L // bs)), self.mbps) for _, L in chunks]
        cfg = make_config(num_layers=2, kv_heads=hkv, head_dim=d, max_batch=len(chunks),
                          max_seq_len=max(self.mbps, sum(need) // len(chunks) + 2) * bs, block_size=bs)
        self.pool = lib.create_pool(cfg, dtype)
        ids = list(rng.permutation(self.pool.alloc_blocks(sum(need) + 2)))
        self.bt = np.full((len(chunks), self.mbps), ids.pop(), np.int32)   # of no sequence
        for b, n in enumerate(need):
            for i in range(n):
                self.bt[b, i] = ids.pop()
        self.offs = np.asarray(self.pool.all_block_offsets_f16(), np.uint64)
        st = self.pool.stats()
        self.bb = st["block_bytes"]
        self.row = hkv * d * {KV_FP8: 1, KV_F32: 4}.get(dtype, 2)
        self.bases = [self.pool.va_k(1), self.pool.va_v(1)]
        self.before = []
        for base in self.bases:
            reg = rng.integers(0, 256, st["superblock_count"] * SB).astype(np.uint8)
            if dtype == KV_FP8:
                reg[(reg & 0x7F) == 0x7F] = 0x11            # no NaN codes
                for off in self.offs.astype(np.int64) * 2:
                    at = off + self.row * bs
                    reg[at:at + 4 * hkv] = rng.uniform(1e-3, 2e-2, hkv).astype(np.float32).view(np.uint8)
            memcpy_htod(base, reg)
            self.before.append(reg)
        self.qsl = np.concatenate([[0], np.cumsum([n for n, _ in chunks])]).astype(np.int32)
        self.total = int(self.qsl[-1]) + pad
        heads = hq + 2 * hkv
        if x is None:
            x = rng.standard_normal((self.total, heads, d)) * np.exp(0.5 * rng.standard_normal((self.total, heads, 1)))
        enc = O.encode(CODE[dtype], x.astype(np.float32))
        self.x = O.decode(CODE[dtype], enc).astype(np.float64).reshape(self.total, heads, d)
        self.inv = rope_inv_freq(theta, d)
        tdt = torch_io_dtype(dtype)
        to = (lambda a: torch.from_numpy(a.copy())) if dtype == KV_F32 else \
            (lambda a: torch.from_numpy(a.view(np.int16).copy()).view(tdt))
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        self.dev = dict(qkv=to(enc).cuda(), bt=i32(self.bt), sl=i32([L for _, L in chunks]), qsl=i32(self.qsl),
                        offs=torch.from_numpy(self.offs.view(np.int64)).cuda(),
                        inv=torch.from_numpy(self.inv).cuda(),
                        pos=None if positions is None else i32(positions))
        self.q = torch.full((self.total + 2, hq, d), 7.0, dtype=tdt, device="cuda")
        torch.cuda.synchronize()

    def run(self, stream=0):
        d = self.dev
        p = d["pos"]
        self.pool.rope_append_chunk(
            layer_idx=1, qkv_ptr=d["qkv"].data_ptr(), q_out_ptr=self.q.data_ptr(),
            block_tables_ptr=d["bt"].data_ptr(), seq_lens_ptr=d["sl"].data_ptr(),
            query_start_loc_ptr=d["qsl"].data_ptr(), block_offsets_f16_ptr=d["offs"].data_ptr(),
            inv_freq_ptr=d["inv"].data_ptr(), batch=len(self.chunks), total_query_tokens=self.total,
            num_q_heads=self.hq, max_blocks_per_seq=self.mbps, positions_ptr=0 if p is None else p.data_ptr(),
            num_axes=0 if p is None else p.shape[0], pair_axes=self.axes, stream_ptr=stream)

    def rotated(self, t, place):
        """Exact q and k heads of row t, and the size |x1| + |x2| of each value."""
        half = self.d // 2
        at = np.full(half, float(place))
        if self.positions is not None:
            axes = self.axes or [0] * half
            at = np.array([float(self.positions[a][t]) for a in axes])
        ang = at.astype(np.longdouble) * self.inv.astype(np.longdouble)
        c, s = np.cos(ang).astype(np.float64), np.sin(ang).astype(np.float64)
        x = self.x[t, :self.hq + self.hkv]
        a, b = x[:, :half], x[:, half:]
        size = np.abs(a) + np.abs(b)
        return np.concatenate([a * c - b * s, b * c + a * s], 1), np.concatenate([size, size], 1)

    def check(self):
        u, tiny = HALF_STEP[self.dtype], TINY[self.dtype]
        q = self.q.double().cpu().numpy()
        after = [memcpy_dtoh(base, len(reg)) for base, reg in zip(self.bases, self.before)]
        want = [reg.copy() for reg in self.before]          # bytes that may not change stay
        seen = np.zeros(self.total + 2, bool)
        cap = self.mbps * self.bs
        for b, (n, L) in enumerate(self.chunks):
            first = L - n
            pages = {}
            for i in range(n):
                t, place = int(self.qsl[b]) + i, first + i
                if not 0 <= place < cap:
                    continue
                seen[t] = True
                y, size = self.rotated(t, place)
                off = np.abs(q[t] - y[:self.hq])
                tol = u * np.abs(y[:self.hq]) + (1 + u) * TRIG * size[:self.hq] + tiny
                assert np.all(off <= tol), (b, i, float(np.max(off / tol)))
                entry = int(self.bt[b, place // self.bs])
                if 0 <= entry < len(self.offs):
                    pages.setdefault(entry, []).append((place % self.bs, t, y[self.hq:], size[self.hq:]))
            for entry, rows in pages.items():
                page = int(self.offs[entry]) * 2
                v = [(s, self.x[t, self.hq + self.hkv:], np.zeros_like(y)) for s, t, y, _ in rows]
                k = [(s, y, TRIG * size) for s, _, y, size in rows]
                for got, exp, vals in zip(after, want, (k, v)):
                    self.check_page(got, exp, page, vals)
        assert np.all(q[~seen] == 7.0)
        for got, exp in zip(after, want):
            assert np.array_equal(got, exp)

    def check_page(self, got, exp, page, vals):
        """Checks the written slots and copies them over; what is left must be
        equal to the bytes."""
        hkv, d, bs, row = self.hkv, self.d, self.bs, self.row
        if self.dtype != KV_FP8:
            u, tiny = HALF_STEP[self.dtype], TINY[self.dtype]
            for s, y, slack in vals:
                at = page + s * row
                raw = got[at:at + row]
                val = O.decode(CODE[self.dtype], raw.view(np.float32 if self.dtype == KV_F32 else np.uint16))
                off = np.abs(val.astype(np.float64).reshape(hkv, d) - y)
                assert np.all(off <= np.where(slack > 0, u * np.abs(y) + (1 + u) * slack + tiny, 0)), s
                exp[at:at + row] = raw
            return
        foot = page + row * bs
        old = exp[foot:foot + 4 * hkv].view(np.float32).astype(np.float64)
        new = got[foot:foot + 4 * hkv].view(np.float32)
        y = np.stack([v for _, v, _ in vals])
        slack = np.stack([s for _, _, s in vals])
        amax = np.abs(y).max(axis=(0, 2))
        started = any(s == 0 for s, _, _ in vals) | ~(np.isfinite(old) & (old > 0))
        fresh = np.where(amax > 0, amax / 448, 1.0)
        scale = np.where(started, fresh, np.where(amax > 448 * old, fresh, old))
        # below 2^-126 fp32 has a fixed grid of 2^-149: the scale's own rounding is off by
        # half of it, 2^-150, and its amax by three such (two operations of the value and
        # the functions' product), of which 448 parts reach it: less than 2^-149 together
        assert np.all(np.abs(new - scale) <= 2.0 ** -23 * scale + slack.max(axis=(0, 2)) / 448 + 2.0 ** -149)
        s64 = new.astype(np.float64)[:, None]
        tab = E.e4m3_values()
        written = [s for s, _, _ in vals]
        for i, s in enumerate(written):
            at = page + s * row
            c = got[at:at + row].reshape(hkv, d)
            off = np.abs(tab[c] * s64 - y[i])
            half = np.maximum(2.0 ** -4 * np.abs(y[i]), 2.0 ** -10 * s64)
            assert np.all(off <= half * (1 + 2.0 ** -20) + 2 * slack[i] + 2.0 ** -148), s   # (as above)
            if not slack.any():
                assert np.array_equal(c, E.e4m3_codes((y[i].astype(np.float32) / new[:, None]))), s
            exp[at:at + row] = got[at:at + row]
        grown = ~started & (new != old.astype(np.float32))
        for s in range(bs):
            if s in written:
                continue
            at = page + s * row
            c = exp[at:at + row].reshape(hkv, d)
            again = E.e4m3_codes(tab[c].astype(np.float32) * old.astype(np.float32)[:, None] / new[:, None])
            exp[at:at + row] = np.where(grown[:, None], again, c).reshape(-1)
        exp[foot:foot + 4 * hkv] = got[foot:foot + 4 * hkv]

    def close(self):
        self.pool.destroy()


def check(*args, **kw):
    c = Case(*args, **kw)
    try:
        c.run()
        c.torch.cuda.synchronize()
        c.check()
    finally:
        c.close()


ALL = [KV_BF16, KV_F16, KV_FP8, KV_F32]


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("hq,hkv,d,bs", [(32, 8, 128, 16), (8, 8, 64, 16), (4, 2, 80, 32), (3, 1, 24, 8),
                                         (2, 1, 256, 16), (6, 2, 40, 5), (2, 2, 8, 1), (2, 1, 128, 300)])
def test_shapes(gpu_lib, dtype, hq, hkv, d, bs):
    import torch
    check(torch, gpu_lib, dtype, hq, hkv, d, bs, [(37, 37), (1, 90), (19, 50), (3, 3)], seed=d + bs)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("chunks,pad,mbps", [
    ([(1, 1)], 0, None), ([(1, 40)], 0, None), ([(2, 17)], 0, None), ([(16, 16)], 0, None),
    ([(0, 5), (4, 4), (0, 0), (7, 30), (0, 9)], 0, None),          # sequences without tokens
    ([(33, 48), (5, 5)], 9, None),                                  # rows of no sequence
    ([(20, 12), (6, 0), (5, -3), (9, 30)], 0, None),                # more tokens than the cache has
    ([(40, 60), (10, 20)], 0, 2),                                   # past the table's end
    ([(3, 1000 + i) for i in range(130)], 0, None),                 # more sequences than lanes
    ([(1, 1 + i % 40) for i in range(70)], 3, None),
    ([(700, 711), (5, 300)], 0, None),
])
def test_lengths(gpu_lib, dtype, chunks, pad, mbps):
    import torch
    check(torch, gpu_lib, dtype, 4, 2, 64, 16, chunks, pad=pad, mbps=mbps)


@pytest.mark.parametrize("hkv,d,bs", [(1, 128, 32), (3, 128, 64), (2, 128, 128), (2, 64, 48), (1, 256, 33), (3, 72, 100)])
def test_fp8_pages_of_several_waves(gpu_lib, hkv, d, bs):
    """Chunks that begin and end inside large pages, whose rows several waves
    share; whole pages, single rows, and growth of a page that has rows already."""
    import torch
    check(torch, gpu_lib, KV_FP8, 2 * hkv, hkv, d, bs, [(2 * bs + 5, 3 * bs), (1, bs + 1), (bs, bs), (3, 2 * bs + 2),
                                                       (bs - 1, 2 * bs - 1), (0, 7), (bs // 2, bs // 2 + 9)], seed=bs)
    check(torch, gpu_lib, KV_FP8, 2 * hkv, hkv, d, bs, [(5 * bs + 1, 6 * bs - 3), (9, 9)], mbps=4, seed=d)


@pytest.mark.parametrize("dtype", ALL)
@pytest.mark.parametrize("n_axes,deal", [(1, None), (2, "turn"), (3, "sections"), (4, "turn")])
def test_axes(gpu_lib, dtype, n_axes, deal):
    """Positions of their own: any order, equal ones, negative ones."""
    import torch
    rng = np.random.default_rng(n_axes)
    d, chunks = 128, [(50, 50), (21, 100)]
    pos = rng.integers(-50, 5000, (n_axes, 71 + 4))
    axes = None if deal is None else [i % n_axes for i in range(d // 2)] if deal == "turn" else \
        [0] * 16 + [1] * 24 + [2] * 24
    check(torch, gpu_lib, dtype, 8, 2, d, 16, chunks, positions=pos, axes=axes, pad=4)


def test_far_positions(gpu_lib):
    """Angles that fp32 does not hold: the values stay as near as at 0."""
    import torch
    pos = np.array([[131071, 1 << 20, (1 << 24) + 1, (1 << 27) - 1, -(1 << 27) + 1, 12345678, 0, 1]])
    check(torch, gpu_lib, KV_F32, 4, 2, 128, 16, [(8, 20)], positions=pos, theta=500000.0)
    check(torch, gpu_lib, KV_BF16, 4, 2, 128, 16, [(8, 20)], positions=pos, theta=500000.0)
    pos = np.array([[2147483647, -2147483648, 2147483646, 1 << 30]])
    check(torch, gpu_lib, KV_F32, 4, 2, 64, 16, [(4, 20)], positions=pos, theta=500000.0)


def test_decode_token_as_the_decode_form(gpu_lib):
    """A chunk of one token a sequence near position 0: what
    kcmm_rope_append_bf16 gives, but for the angle's rounding there."""
    import torch
    c = Case(torch, gpu_lib, KV_BF16, 8, 2, 128, 16, [(1, 1 + i) for i in range(40)])
    try:
        c.run()
        torch.cuda.synchronize()
        mine, pages = c.q[:40].clone(), [memcpy_dtoh(b, len(r)) for b, r in zip(c.bases, c.before)]
        c.pool.rope_append(layer_idx=1, qkv_ptr=c.dev["qkv"].data_ptr(), q_out_ptr=c.q.data_ptr(),
                           block_tables_ptr=c.dev["bt"].data_ptr(), seq_lens_ptr=c.dev["sl"].data_ptr(),
                           block_offsets_f16_ptr=c.dev["offs"].data_ptr(), inv_freq_ptr=c.dev["inv"].data_ptr(),
                           batch=40, num_q_heads=8, max_blocks_per_seq=c.mbps)
        torch.cuda.synchronize()
        # two bf16 roundings of values 2^-17 apart (|x1| + |x2| < 32, angles < 40)
        assert torch.allclose(mine.float(), c.q[:40].float(), rtol=2.0 ** -7, atol=2.0 ** -12)
        assert np.array_equal(pages[1], memcpy_dtoh(c.bases[1], len(pages[1])))
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ALL)
def test_foreign_blocks(gpu_lib, dtype):
    """Table entries that are no block of the pool: nothing is written for them,
    the tokens' q is."""
    import torch
    c = Case(torch, gpu_lib, dtype, 4, 2, 64, 16, [(50, 60), (20, 20)])
    try:
        c.bt[0, 1], c.bt[1, 0], c.bt[0, 3] = -1, len(c.offs), 2147483647
        c.dev["bt"].copy_(torch.from_numpy(c.bt))
        torch.cuda.synchronize()
        c.run()
        torch.cuda.synchronize()
        c.check()
    finally:
        c.close()


@pytest.mark.parametrize("bs", [32, 64, 128])
def test_fp8_foreign_blocks_of_several_waves(gpu_lib, bs):
    """The same where waves of a workgroup meet for a page's maximum."""
    import torch
    c = Case(torch, gpu_lib, KV_FP8, 3, 1, 128, bs, [(3 * bs, 4 * bs - 5), (20, 20), (0, 4), (bs, bs)])
    try:
        c.bt[0, 1], c.bt[1, 0], c.bt[0, 3] = -1, len(c.offs), 2147483647
        c.dev["bt"].copy_(torch.from_numpy(c.bt))
        torch.cuda.synchronize()
        c.run()
        torch.cuda.synchronize()
        c.check()
    finally:
        c.close()


@pytest.mark.parametrize("value", [0.0, 3e38, 1e-38, 1e-30])
def test_fp8_ends_of_the_range(gpu_lib, value):
    """Rows of zeros, and of values at the ends of bf16's range."""
    import torch
    rng = np.random.default_rng(1)
    x = value * rng.uniform(-0.7, 0.7, (24, 8, 64))      # (|x1| + |x2| stays in range)
    check(torch, gpu_lib, KV_FP8, 4, 2, 64, 16, [(24, 24)], x=x)
    check(torch, gpu_lib, KV_FP8, 4, 2, 64, 16, [(24, 29)], x=x)


def test_fp8_pages_never_started(gpu_lib):
    """A scale that is no finite positive number: the write starts the page."""
    import torch
    c = Case(torch, gpu_lib, KV_FP8, 4, 4, 64, 16, [(20, 25)])
    try:
        for base, reg in zip(c.bases, c.before):
            for off in c.offs.astype(np.int64) * 2:
                at = off + c.row * c.bs
                reg[at:at + 16] = np.array([0, -1, np.inf, np.nan], np.float32).view(np.uint8)
            memcpy_htod(base, reg)
        c.run()
        torch.cuda.synchronize()
        c.check()
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ALL)
def test_infinities_and_nan(gpu_lib, dtype):
    """They stay in their token and head (an fp8 page's scale is its page's)."""
    import torch
    rng = np.random.default_rng(2)
    x = rng.standard_normal((40, 8, 64)).astype(np.float32)
    bad = x.copy()
    bad[5, 0, 3], bad[6, 5, 40], bad[7, 7, 2], bad[20, 4, 1] = np.nan, np.inf, -np.inf, np.nan
    outs = []
    for v in (x, bad):
        c = Case(torch, gpu_lib, dtype, 4, 2, 64, 16, [(40, 40)], x=v)
        try:
            c.run()
            torch.cuda.synchronize()
            rows = []
            for base, reg in zip(c.bases, c.before):
                raw = memcpy_dtoh(base, len(reg))
                for lb in range(3):
                    page = int(c.offs[c.bt[0, lb]]) * 2
                    n = 16 if lb < 2 else 8
                    if dtype == KV_FP8:
                        sc = raw[page + c.row * 16:][:8].view(np.float32)
                        val = E.e4m3_values()[raw[page:page + n * c.row]].reshape(n, 2, 64) * sc[:, None]
                    else:
                        val = O.decode(CODE[dtype], raw[page:page + n * c.row].view(
                            np.float32 if dtype == KV_F32 else np.uint16)).reshape(n, 2, 64)
                    rows.append(val)
            outs.append((c.q[:40].float().cpu().numpy(), np.concatenate(rows[:3]), np.concatenate(rows[3:])))
        finally:
            c.close()
    (q0, k0, v0), (q1, k1, v1) = outs
    hit = np.zeros((40, 4), bool)
    hit[5, 0] = True
    assert np.array_equal(q0[~hit], q1[~hit]) and np.isnan(q1[5, 0, [3, 35]]).all()
    hk, hv = np.zeros((40, 2), bool), np.zeros((40, 2), bool)
    if dtype == KV_FP8:
        hk[:16, 1] = hv[:16, 1] = True                  # the scales of these pages' heads are infinite
        hk[20, 0] = True
    else:
        hk[6, 1] = hk[20, 0] = hv[7, 1] = True
        assert not np.isfinite(k1[6, 1, [8, 40]]).any() and v1[7, 1, 2] == -np.inf
    assert np.isnan(k1[20, 0, [1, 33]]).all()
    assert np.array_equal(k0[~hk], k1[~hk]) and np.array_equal(v0[~hv], v1[~hv])


@pytest.mark.parametrize("dtype", ALL)
def test_graph_replays(gpu_lib, dtype):
    """Captured at once; lengths and positions are read at every replay."""
    import torch
    c = Case(torch, gpu_lib, dtype, 8, 2, 128, 16, [(30, 30), (9, 77)])
    try:
        st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=st):
            c.run(torch.cuda.current_stream().cuda_stream)
        for n in range(3):
            c.chunks = [(30, 30 + n), (9, 77 - n)]
            c.dev["sl"].copy_(torch.tensor([30 + n, 77 - n], dtype=torch.int32))
            got = []
            for run in (graph.replay, c.run):
                for base, reg in zip(c.bases, c.before):
                    memcpy_htod(base, reg)
                c.q.fill_(7.0)
                torch.cuda.synchronize()
                run()
                torch.cuda.synchronize()
                c.check()
                got.append([c.q.clone()] + [memcpy_dtoh(b, len(r)) for b, r in zip(c.bases, c.before)])
            assert torch.equal(got[0][0], got[1][0])
            assert all(np.array_equal(x, y) for x, y in zip(got[0][1:], got[1][1:]))
    finally:
        c.close()


@pytest.mark.parametrize("dtype", ALL)
def test_blocks_issued_after_a_capture(gpu_lib, dtype):
    """A graph whose tables, updated in place, name a block that the pool issued
    after the capture writes its rows; ids that it has not issued are no blocks."""
    import torch
    hq, hkv, d, bs = 4, 2, 64, 16
    cfg = make_config(num_layers=1, kv_heads=hkv, head_dim=d, max_batch=2, max_seq_len=512, block_size=bs)
    pool = gpu_lib.create_pool(cfg, dtype)
    try:
        most = 12
        mine = pool.alloc_blocks(2)
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device="cuda")  # noqa: E731
        bt, sl, qsl = i32([[mine[0], 0, 0], [mine[1], 0, 0]]), i32([5, 9]), i32([0, 1, 2])
        offs = torch.zeros(most, dtype=torch.int64, device="cuda")
        offs[:pool.total_blocks()] = torch.tensor(pool.all_block_offsets_f16(), device="cuda")
        qkv = torch.ones(2, (hq + 2 * hkv) * d, dtype=torch_io_dtype(dtype), device="cuda")
        q = torch.zeros(2, hq, d, dtype=qkv.dtype, device="cuda")
        inv = torch.from_numpy(rope_inv_freq(10000.0, d)).cuda()
        nbytes = pool.stats()["superblock_count"] * SB
        memcpy_htod(pool.va_v(0), np.zeros(nbytes, np.uint8))

        def call():
            pool.rope_append_chunk(
                layer_idx=0, qkv_ptr=qkv.data_ptr(), q_out_ptr=q.data_ptr(), block_tables_ptr=bt.data_ptr(),
                seq_lens_ptr=sl.data_ptr(), query_start_loc_ptr=qsl.data_ptr(),
                block_offsets_f16_ptr=offs.data_ptr(), inv_freq_ptr=inv.data_ptr(), batch=2,
                total_query_tokens=2, num_q_heads=hq, max_blocks_per_seq=3,
                stream_ptr=torch.cuda.current_stream().cuda_stream)

        def capture():
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
                call()
            return graph

        def written(graph, block, row):
            q.zero_()
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            assert bool((q[:, 0, 0] != 0).all())
            at = int(pool.all_block_offsets_f16()[block]) * 2 + row * hkv * d * {KV_FP8: 1, KV_F32: 4}.get(dtype, 2)
            return bool(memcpy_dtoh(pool.va_v(0), nbytes)[at:at + 64].any())

        torch.cuda.synchronize()
        graph = capture()
        assert written(graph, mine[0], 4) and written(graph, mine[1], 8)
        for n in range(3):
            # the next block of the first sequence, in the place of the table that the graph reads
            new = pool.alloc_blocks(1)[0]
            assert pool.total_blocks() == new + 1 == 3 + n
            offs[:new + 1] = torch.tensor(pool.all_block_offsets_f16(), device="cuda")
            bt[0, 1], bt[1, 0] = new, new + 1
            sl[0] = 18
            before = memcpy_dtoh(pool.va_v(0), nbytes)
            assert written(graph, new, 1)
            after = memcpy_dtoh(pool.va_v(0), nbytes)
            page = int(offs[new]) * 2
            assert np.array_equal(before[:page], after[:page])          # (nothing else: id new + 1 is none)
            rest = page + pool.stats()["block_bytes"]
            assert np.array_equal(before[rest:], after[rest:])
    finally:
        pool.destroy()

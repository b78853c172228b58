"""Decode attention of groups that share a prefix (kcmm_paged_attn_decode_shared):
the parts of a long prefix and their join, for every number of query heads a kv
head, against fp64 under the tolerance of test_gpu_attn_shared."""
import numpy as np
import pytest

import oracle as O
from lattice_amd.bindings import KV_BF16, KV_F16, KV_F32, KV_FP8, memcpy_dtoh, memcpy_htod
from lattice_amd.workload import SB
from tests.test_gpu_attn_shared import HALF_STEP, Case, check

pytestmark = pytest.mark.gpu


def tight(c):
    got = c.out.double().cpu().numpy()
    f16, u = c.dtype == KV_F16, HALF_STEP[c.dtype]
    for b, n in enumerate(c.totals):
        k, v = (x[:n] for x in c.dense[b])
        for h in range(c.hq):
            g = h * c.hkv // c.hq
            z = k[:, g] @ c.q[b, h] * c.scale
            size = np.abs(k[:, g]) @ np.abs(c.q[b, h]) * abs(c.scale)
            w = np.exp(z - z.max())
            w /= w.sum()
            o, a = w @ v[:, g], w @ np.abs(v[:, g])
            assert np.abs(z - z.max())[w > 2.0 ** -60].max() <= 64
            delta = 2 * ((c.d + 2) * 2.0 ** -24 * size.max() + 2.0 ** -18)
            tol = u * np.abs(o) + (u * u + delta + (n + 64) * 2.0 ** -24) * a
            if f16:
                tol += 2.0 ** -32 * np.abs(v[:, g]).sum(0) + 2.0 ** -25
            off = np.abs(got[b, h] - o)
            assert np.all(off <= tol), (b, h, n, float(np.max(off / tol)))


# the page types and head widths whose parts are joined
SPLIT = [(KV_BF16, 128), (KV_F16, 128), (KV_FP8, 128), (KV_BF16, 64), (KV_F16, 64)]


@pytest.mark.parametrize("dtype,d", SPLIT)
@pytest.mark.parametrize("group", range(1, 17))
def test_heads_of_a_kv_head(gpu_lib, dtype, group, d):
    """Every width of the join's rows (group * d / 4 of its 256 threads): a few
    parts, and more than it takes at a time."""
    import torch
    check(torch, gpu_lib, dtype, 2 * group, 2, d, 16, [[(100, 133), (100, 101), (100, 164)], [(37, 70)]],
          seed=group)
    check(torch, gpu_lib, dtype, group, 1, d, 16, [[(2100, 2100 + 40 * i) for i in range(3)], [(0, 5)]], seed=group)


@pytest.mark.parametrize("dtype,hq,hkv,d,bs", [
    (KV_BF16, 8, 2, 128, 16), (KV_F16, 16, 4, 64, 16), (KV_BF16, 6, 3, 80, 16), (KV_F16, 40, 2, 64, 8),
    (KV_F32, 8, 2, 128, 16), (KV_F32, 4, 4, 36, 4)])
@pytest.mark.parametrize("rows", [[0], [0, 1, 2, 3], list(range(200)), list(range(1, 700)), [299], [5, 640]])
def test_scores_of_minus_infinity(gpu_lib, dtype, hq, hkv, d, bs, rows):
    """Tokens whose K holds an infinity that makes their scores -inf weigh
    nothing, wherever they stand: the others' softmax is left."""
    import torch
    c = Case(torch, gpu_lib, dtype, hq, hkv, d, bs,
             [[(640, 700), (640, 641), (640, 900)], [(0, 5), (0, 1024)]], seed=d)
    try:
        c.dev["q"][:, :, 0] = 1.0
        c.q[:, :, 0] = 1.0
        code = np.frombuffer({KV_BF16: b"\x80\xff", KV_F16: b"\x00\xfc", KV_F32: b"\x00\x00\x80\xff"}[dtype], np.uint8)
        keys = memcpy_dtoh(c.pool.va_k(0), c.pool.stats()["superblock_count"] * SB)
        offs, bt = np.asarray(c.pool.all_block_offsets_f16(), np.int64) * 2, c.dev["bt"].cpu().numpy()
        lead = np.repeat(c.starts[:-1], np.diff(c.starts))
        for b in range(c.batch):
            hit = [t for t in rows if t < c.totals[b]]
            if len(hit) == c.totals[b]:
                hit = hit[:-1]       # (one token is left)
            for t in hit:
                r = lead[b] if t < c.shared[b] // bs * bs else b
                at = int(offs[bt[r, t // bs]]) + t % bs * hkv * d * len(code)
                for h in range(hkv):
                    keys[at + h * d * len(code):][:len(code)] = code
            gone = np.isin(np.arange(c.totals[b]), hit)
            c.dense[b] = [x[:c.totals[b]][~gone] for x in c.dense[b]]
            c.totals[b] = int((~gone).sum())
        memcpy_htod(c.pool.va_k(0), keys)
        c.run()
        torch.cuda.synchronize()
        c.check()
    finally:
        c.close()


@pytest.mark.parametrize("dtype,hq,hkv,d", [(KV_BF16, 8, 2, 128), (KV_F16, 8, 2, 128), (KV_F16, 8, 2, 64),
                                            (KV_F16, 16, 1, 64)])
@pytest.mark.parametrize("heavy", [0, 9, 15, 90])
@pytest.mark.parametrize("nats", [12, 18, 20])
def test_small_weights_beside_a_large_one(gpu_lib, dtype, hq, hkv, d, heavy, nats):
    """One token of nearly all the weight, whose V is 0, beside tokens of e^-nats
    each: their values are the output."""
    import torch
    c = Case(torch, gpu_lib, dtype, hq, hkv, d, 16, [[(90, 100), (90, 99)], [(0, 16)]], scale=1.0, seed=nats)
    try:
        c.dev["q"].fill_(1.0)
        c.q[:] = 1.0
        offs, bt = np.asarray(c.pool.all_block_offsets_f16(), np.int64) * 2, c.dev["bt"].cpu().numpy()
        nbytes = c.pool.stats()["superblock_count"] * SB
        code = {KV_BF16: O.BF16, KV_F16: O.F16}[dtype]
        k, v = np.zeros(nbytes // 2, np.uint16), np.zeros(nbytes // 2, np.uint16)
        big = O.encode(code, np.full(hkv * d, nats / d, np.float32))
        some = O.encode(code, np.random.default_rng(nats).uniform(800, 1000, hkv * d).astype(np.float32))
        assert np.all(O.decode(code, big) * d == nats)
        for b, n in enumerate(c.totals):
            heavy_b = min(heavy, n - 1)
            for t in range(n):
                at = int(offs[bt[0 if b == 1 and t < 80 else b, t // 16]]) // 2 + t % 16 * hkv * d
                k[at:at + hkv * d] = big if t == heavy_b else 0
                v[at:at + hkv * d] = 0 if t == heavy_b else some
            c.dense[b][0][:] = 0
            c.dense[b][0][heavy_b] = nats / d
            c.dense[b][1][:] = O.decode(code, some).reshape(hkv, d)
            c.dense[b][1][heavy_b] = 0
        memcpy_htod(c.pool.va_k(0), k)
        memcpy_htod(c.pool.va_v(0), v)
        c.run()
        torch.cuda.synchronize()
        tight(c)
    finally:
        c.close()


def reads(shared, totals, bs):
    """The fewest tokens that sequences read with one common length: c + what each
    has behind it, all of it for who shares less."""
    blocks = [max(0, min(s, t)) // bs * bs for s, t in zip(shared, totals)]
    return min(c + sum(t - (c if s >= c else 0) for s, t in zip(blocks, totals)) for c in {0, *blocks})


@pytest.mark.parametrize("dtype,d", SPLIT)
@pytest.mark.parametrize("lengths", [
    [4200] + [2048] * 7,                       # the first sequence states all that is its own
    [2048] * 7 + [1040],                       # one shares half of it
    [2048] * 7 + [16], [2048] * 7 + [0],
    [3000] * 4 + [1500] * 4, [3000] * 2 + [1000] * 6,
    [500, 1000, 1500, 2000, 2500, 3000, 3500, 4000], [64] * 7 + [2000],
])
@pytest.mark.parametrize("order", [1, -1])
def test_lengths_that_differ(gpu_lib, dtype, d, lengths, order):
    """However the lengths of a group differ, its common tokens are read once, as
    few tokens in all as one common length allows.  (The second word of the
    scratch: tiles of all kv heads.)"""
    import torch
    lengths = lengths[::order]
    group = [(s, max(s + 30, 2100) + 7 * i) for i, s in enumerate(lengths)]
    c = Case(torch, gpu_lib, dtype, 8, 2, d, 16, [group], seed=len(set(lengths)))
    try:
        c.run()
        torch.cuda.synchronize()
        c.check()
        tile = 16 if d == 128 and dtype != KV_FP8 else 32
        tiles = int(c.scratch[:12].view(torch.int32)[1]) // 2
        assert tiles <= reads(lengths, c.totals, 16) // tile + 1 + len(lengths)
    finally:
        c.close()


@pytest.mark.parametrize("dtype,d", SPLIT)
@pytest.mark.parametrize("hq,hkv,bs", [(8, 2, 16), (4, 4, 8), (16, 1, 32), (14, 2, 16), (20, 2, 16)])
def test_weights_of_two_parts(gpu_lib, dtype, d, hq, hkv, bs):
    """As near as weights of two 16-bit parts are, not of one."""
    import torch
    for groups in ([[(100, 133), (100, 101), (100, 164), (100, 100)], [(37, 70)], [(0, 1)]],
                   [[(1500, 1500 + 33 * i) for i in range(5)]]):
        for q_scale in (1.0, 3.0):
            c = Case(torch, gpu_lib, dtype, hq, hkv, d, bs, groups, seed=hq + d, q_scale=q_scale)
            try:
                c.run()
                torch.cuda.synchronize()
                tight(c)
            finally:
                c.close()


@pytest.mark.parametrize("dtype,d", SPLIT)
def test_a_page_that_counts(gpu_lib, dtype, d):
    """One page's values are 64 times the others', each in turn: taken twice or not
    at all it would change outputs by several times their size.  4 items of two
    tiles or more a wave."""
    import torch
    c = Case(torch, gpu_lib, dtype, 8, 4, d, 16, [[(4100, 4100 + 21 * i) for i in range(17)]], seed=d)
    try:
        offs, bt = np.asarray(c.pool.all_block_offsets_f16(), np.int64) * 2, c.dev["bt"].cpu().numpy()
        row, nbytes = 4 * d * (1 if dtype == KV_FP8 else 2), c.pool.stats()["superblock_count"] * SB
        plain, dense = memcpy_dtoh(c.pool.va_v(0), nbytes), c.dense
        for seq, block in [(0, 0), (0, 1), (0, 131), (0, 255), (16, 256), (16, 275), (5, 261)]:
            last = min((block + 1) * 16, c.totals[seq])
            values = plain.copy()
            page = int(offs[bt[seq, block]])
            if dtype == KV_FP8:
                values[page + 16 * row:page + 16 * row + 16].view(np.float32)[:] *= 64
            else:
                n = (last - block * 16) * row
                code = {KV_BF16: O.BF16, KV_F16: O.F16}[dtype]
                raw = values[page:page + n].view(np.uint16)
                raw[:] = O.encode(code, (O.decode(code, raw) * 64).astype(np.float32))
            memcpy_htod(c.pool.va_v(0), values)
            c.dense = []
            for b, (k, v) in enumerate(dense):
                if b == seq or block < 256:
                    v = v.copy()
                    v[block * 16:last] *= 64
                c.dense.append([k, v])
            c.out.fill_(float("nan"))
            c.run()
            torch.cuda.synchronize()
            tight(c)
    finally:
        c.close()

"""Low-rank adapters beside a shared projection (kcmm_lora_add_bf16) on the GPU
against fp64, and bit for bit where every sum is a whole number that fp32 holds.

Tolerance of y = bf16(base + s sum_r v_r b_r), v_r = sum_k x_k a_rk: v is a sum of
K products in fp32, off by at most (K + 8) 2^-24 of V_r = sum |x||a|; the
product with B takes v as two bf16 parts, 2^-16 of it, and at most 2 rank + 8
roundings of 2^-24 of V_r |b_r| follow; then s and the addition, and one
rounding to bf16, 2^-8."""
import numpy as np
import pytest

from tests import e4m3 as E

pytestmark = pytest.mark.gpu


def dev16(torch, values):
    return torch.from_numpy(E.bf16_bits(values).view(np.int16)).view(torch.bfloat16).cuda()


class Case:
    def __init__(self, torch, m, widths, k, rank, adapters, ids=None, seed=0, scales=True, in_place=False,
                 whole=False, poison=False):
        rng = np.random.default_rng([seed, m, k, rank])
        self.torch, self.m, self.k, self.rank, self.adapters = torch, m, k, rank, adapters
        self.widths, self.n, self.rows = widths, sum(widths), rank * len(widths)
        ids = rng.integers(-1, adapters, m) if ids is None else np.asarray(ids)
        self.ids = ids.astype(np.int32)
        n = self.n
        if whole:
            # |v| <= 2 K <= 2^9 and v b sums below 2^15: exact in fp32, and in bf16 after
            # rounding once
            draw = lambda *s: rng.integers(-1, 2, s).astype(np.float32)  # noqa: E731
        else:
            draw = lambda *s: rng.standard_normal(s).astype(np.float32)  # noqa: E731
        scale_a = 1.0 if whole else 1 / np.sqrt(k)
        self.x, self.a = E.bf16(draw(m, k)), E.bf16(draw(adapters, self.rows, k) * np.float32(scale_a))
        self.b, self.base = E.bf16(draw(adapters, n, rank)), E.bf16(draw(m, n) * 4)
        self.s = (rng.integers(1, 3, adapters) if whole else rng.uniform(0.2, 2, adapters)).astype(np.float32)
        if not scales:
            self.s = np.ones(adapters, np.float32)
        if poison:   # adapters that no token has
            used = np.isin(np.arange(adapters), ids)
            assert not used.all()
            self.a[~used], self.b[~used], self.s[~used] = np.nan, np.nan, np.nan
        self.in_place = in_place
        full = lambda r: torch.full((r * n + 64,), 7.0, dtype=torch.bfloat16, device="cuda")  # noqa: E731
        self.dev = dict(x=dev16(torch, self.x), a=self.nan16(self.a), b=self.nan16(self.b),
                        base=dev16(torch, self.base), s=torch.from_numpy(self.s).cuda() if scales else None,
                        ids=torch.from_numpy(self.ids).cuda())
        self.y = full(m)
        if in_place:
            self.y[:m * n] = self.dev["base"].reshape(-1)
        self.low = torch.full((m * self.rows + 64,), -5.0, device="cuda")
        torch.cuda.synchronize()

    def nan16(self, v):
        bits = E.bf16_bits(np.nan_to_num(v)).reshape(v.shape)
        bits[np.isnan(v)] = 0x7FC0
        return self.torch.from_numpy(bits.view(np.int16)).view(self.torch.bfloat16).cuda()

    def run(self, lib, stream=0):
        d = self.dev
        lib.lora_add_bf16(d["x"].data_ptr(), d["a"].data_ptr(), d["b"].data_ptr(), d["ids"].data_ptr(),
                          self.low.data_ptr(), (self.y if self.in_place else d["base"]).data_ptr(),
                          self.y.data_ptr(), self.m, self.n, self.k, adapters=self.adapters, rank=self.rank,
                          slice_ends=np.cumsum(self.widths).tolist(),
                          scales_ptr=0 if d["s"] is None else d["s"].data_ptr(), stream_ptr=stream)

    def exact(self):
        """y in fp64, and its tolerance but for the store."""
        y, slack = self.base.astype(np.float64), np.zeros((self.m, self.n))
        for a in range(self.adapters):
            t = np.nonzero(self.ids == a)[0]
            if not len(t):
                continue
            x, w = self.x[t].astype(np.float64), self.a[a].astype(np.float64)
            v, V = x @ w.T, np.abs(x) @ np.abs(w).T
            at = 0
            for i, width in enumerate(self.widths):
                r = slice(i * self.rank, (i + 1) * self.rank)
                b = self.b[a, at:at + width].astype(np.float64)
                s = float(self.s[a])
                y[t, at:at + width] += s * (v[:, r] @ b.T)
                err = (self.k + 8 + 2 * self.rank + 8) * 2.0 ** -24 * (V[:, r] @ np.abs(b).T) + \
                    2.0 ** -16 * (np.abs(v[:, r]) @ np.abs(b).T)
                slack[t, at:at + width] = abs(s) * err + 2.0 ** -23 * np.abs(y[t, at:at + width])
                at += width
        return y, slack

    def get(self):
        y = E.bf16_values(self.y.cpu().view(self.torch.int16).numpy().view(np.uint16))
        assert np.all(y[self.m * self.n:] == 7.0)
        low = self.low.cpu().numpy()
        assert np.all(low[self.m * self.rows:] == -5.0)
        return y[:self.m * self.n].reshape(self.m, self.n)

    def check(self, bits=False):
        got = self.get()
        y, slack = self.exact()
        none = (self.ids < 0) | (self.ids >= self.adapters)
        assert np.array_equal(got[none], self.base[none])
        if bits:
            assert np.array_equal(got, E.bf16(y.astype(np.float32)))
            return
        off, tol = np.abs(got - y), E.BF16_HALF * np.abs(y) + slack * (1 + E.BF16_HALF)
        assert np.all(off <= tol), float(np.max(off / tol))


def check(torch, lib, *args, bits=False, **kw):
    c = Case(torch, *args, **kw)
    c.run(lib)
    torch.cuda.synchronize()
    c.check(bits)


@pytest.mark.parametrize("m", [1, 2, 7, 16, 17, 33, 64, 65, 130, 300])
@pytest.mark.parametrize("widths,k,rank", [([64], 256, 16), ([48, 16], 40, 8), ([128, 32, 32], 520, 24),
                                           ([16], 8, 128), ([272, 16, 80, 144], 1000, 64)])
def test_shapes(gpu_lib, m, widths, k, rank):
    import torch
    check(torch, gpu_lib, m, widths, k, rank, 5)


@pytest.mark.parametrize("mixed", [True, False])
@pytest.mark.parametrize("m,widths,k,rank", [(1100, [7680, 16, 528], 72, 16), (2049, [4112], 40, 8),
                                             (523, [16384, 144], 136, 32), (700, [12800], 64, 64),
                                             (1001, [8192, 272, 16], 64, 128)])
def test_many_tokens_and_columns(gpu_lib, m, widths, k, rank, mixed):
    import torch
    ids = np.random.default_rng(m).integers(-1, 5, m)
    check(torch, gpu_lib, m, widths, k, rank, 5, ids=ids if mixed else np.sort(ids), in_place=mixed)


@pytest.mark.parametrize("adapters", [2, 5, 70])
@pytest.mark.parametrize("m,widths,k,rank", [(600, [4096, 16], 72, 16), (257, [8192], 40, 8), (1000, [2064], 136, 32),
                                             (449, [4608], 64, 64), (385, [5008, 48], 64, 128)])
def test_hundreds_of_mixed_tokens(gpu_lib, m, widths, k, rank, adapters):
    import torch
    ids = np.random.default_rng(m + adapters).integers(-2, adapters + 1, m)
    check(torch, gpu_lib, m, widths, k, rank, adapters, ids=ids, in_place=adapters == 5)


@pytest.mark.parametrize("m,widths,k,rank", [(1, [4096], 4096, 16), (64, [4096, 1024, 1024], 4096, 16),
                                             (5, [1024], 14336, 64), (700, [2048], 2048, 32),
                                             (1100, [512, 512], 1024, 128), (2500, [160], 264, 8)])
def test_larger(gpu_lib, m, widths, k, rank):
    import torch
    check(torch, gpu_lib, m, widths, k, rank, 8, in_place=True)


@pytest.mark.parametrize("m", [1, 5, 40, 200, 600])
@pytest.mark.parametrize("order", ["mixed", "sorted", "one", "none", "distinct", "outside"])
def test_who_has_which(gpu_lib, m, order):
    """Adapters in any order, all the same, none, one a token, ids that are no
    adapter; adapters that no token has hold NaN."""
    import torch
    rng = np.random.default_rng(m)
    adapters = m + 2 if order == "distinct" else 6
    ids = {"mixed": rng.integers(-1, 5, m), "sorted": np.sort(rng.integers(-1, 5, m)), "one": np.full(m, 3),
           "none": np.full(m, -1), "distinct": rng.permutation(m + 1)[:m],
           "outside": rng.choice([-1, 6, 7, 2, 2147483647, -2147483648], m)}[order]
    check(torch, gpu_lib, m, [96, 32], 264, 16, adapters, ids=ids, poison=True, seed=3)
    check(torch, gpu_lib, m, [96, 32], 264, 16, adapters, ids=ids, scales=False, in_place=True)


@pytest.mark.parametrize("m", [1, 16, 63, 520])
@pytest.mark.parametrize("rank", [8, 16, 40, 64])
def test_whole_numbers(gpu_lib, m, rank):
    import torch
    check(torch, gpu_lib, m, [80, 64], 248, rank, 4, whole=True, bits=True)


@pytest.mark.parametrize("m", [3, 40, 300])
def test_infinities_and_nan(gpu_lib, m):
    """What a token or an adapter holds reaches no other."""
    import torch
    c = Case(torch, m, [64, 32], 264, 16, 3, ids=np.arange(m) % 4 - 1)
    c.run(gpu_lib)
    torch.cuda.synchronize()
    good = c.get().copy()
    bad_tokens = [0, 1]                      # without an adapter, and of adapter 0
    c.dev["x"][0, 5] = float("nan")
    c.dev["x"][1, 7] = float("inf")
    c.dev["b"][2, 3, 1] = float("inf")       # column 3 of adapter 2
    c.dev["a"][2, 17, 0] = float("nan")      # second slice of adapter 2
    c.y[:m * c.n] = 0
    c.low.fill_(-5.0)
    torch.cuda.synchronize()
    c.run(gpu_lib)
    torch.cuda.synchronize()
    got = c.get()
    same = np.ones((m, c.n), bool)
    same[1] = False
    two = c.ids == 2
    same[np.ix_(two, np.r_[3, 64:96])] = False
    assert np.array_equal(got[same], good[same])
    assert not np.isfinite(got[1]).any() and bad_tokens
    if two.any():
        assert np.isnan(got[two][:, 64:]).all() and not np.isfinite(got[two][:, 3]).any()


@pytest.mark.parametrize("m", [1, 64, 400])
def test_graph_replays(gpu_lib, m):
    import torch
    c = Case(torch, m, [128, 64], 512, 16, 4)
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        c.run(gpu_lib, torch.cuda.current_stream().cuda_stream)
    for n in range(3):
        c.ids = np.roll(c.ids, 1)
        c.dev["ids"].copy_(torch.from_numpy(c.ids))
        c.y.fill_(7.0)
        c.low.fill_(-5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check()
        first = c.y.clone()
        c.y.fill_(7.0)
        c.low.fill_(-5.0)
        torch.cuda.synchronize()
        c.run(gpu_lib)
        torch.cuda.synchronize()
        assert torch.equal(first, c.y)


def test_two_streams_at_once(gpu_lib):
    import torch
    cs = [Case(torch, m, [256], 1024, 16, 4, seed=m) for m in (40, 90)]
    sides = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(30):
        for c, s in zip(cs, sides):
            c.run(gpu_lib, s.cuda_stream)
    torch.cuda.synchronize()
    for c in cs:
        c.check()


def test_graph_of_many_tokens_and_columns(gpu_lib):
    """The form for many tokens, in place, captured without a call before and
    replayed with another order of adapters than it was captured with."""
    import torch
    c = Case(torch, 1030, [8192, 64], 136, 24, 5)
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        c.run(gpu_lib, stream=torch.cuda.current_stream().cuda_stream)
    for turn in range(3):
        c.ids = np.roll(c.ids, 7 * turn)
        c.dev["ids"].copy_(torch.from_numpy(c.ids))
        c.y[:c.m * c.n].fill_(7.0)
        c.low.fill_(-5.0)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        c.check()
        first = c.y.clone()
        c.run(gpu_lib)
        torch.cuda.synchronize()
        assert torch.equal(c.y, first)


# a shape for each form of the expand, the last three with 32 rows a workgroup of the shrink
FORMS = [(40, [4096, 16], 264, 16), (600, [4096, 16], 72, 16), (449, [4592, 16], 64, 64), (1100, [8192, 32], 72, 16),
         (1100, [4112, 16, 16, 4096], 40, 32), (2049, [4096, 16], 72, 64), (700, [32, 12800], 64, 128)]


@pytest.mark.parametrize("m,widths,k,rank", FORMS)
@pytest.mark.parametrize("order", ["mixed", "runs"])
@pytest.mark.parametrize("in_place", [False, True])
def test_infinities_and_nan_in_every_form(gpu_lib, m, widths, k, rank, order, in_place):
    """What a token or an adapter holds reaches no other, tokens side by side or in
    runs; adapters that no token has hold NaN."""
    import torch
    ids = np.arange(m) % 4 - 1
    ids = ids if order == "mixed" else np.sort(ids)
    c = Case(torch, m, widths, k, rank, 5, ids=ids, in_place=in_place, poison=True)
    base = c.dev["base"].clone()

    def run():
        c.y[:m * c.n] = base.reshape(-1) if in_place else 0
        c.low.fill_(-5.0)
        torch.cuda.synchronize()
        c.run(gpu_lib)
        torch.cuda.synchronize()
        return c.get().copy()

    run()
    c.check()
    good = c.get().copy()
    none, first, two = (np.nonzero(ids == a)[0] for a in (-1, 0, 2))
    bad = first[[0, len(first) // 2, -1]]
    c.dev["x"][int(none[0]), 5] = float("nan")
    c.dev["x"][int(none[-1])] = float("inf")
    c.dev["x"][torch.from_numpy(bad).cuda(), 7] = float("inf")
    c.dev["b"][2, 3, 1] = float("inf")                    # column 3 of adapter 2
    c.dev["a"][2, rank + 1, 0] = float("nan")             # its second slice
    got = run()
    cut = slice(widths[0], widths[0] + widths[1])
    same = np.ones((m, c.n), bool)
    same[bad] = False
    same[np.ix_(two, [3])] = same[two, cut] = False
    assert np.array_equal(got[same], good[same])
    assert not np.isfinite(got[bad]).any() and np.isnan(got[two, cut]).all()
    assert not np.isfinite(got[two, 3]).any()


@pytest.mark.parametrize("m,n", [(5, 16), (600, 4112), (1100, 8224)])
@pytest.mark.parametrize("scale,b", [(1.7e38, 2.0 ** -10), (1.7075e38, 2.0 ** -10), (-1.7075e38, 2.0 ** -10),
                                     (2.0 ** -100, 1.0), (2.0 ** -126, 2.0 ** 30), (2.0 ** -133, 2.0 ** 30)])
def test_values_at_the_ends_of_the_range(gpu_lib, m, n, scale, b):
    """Low-rank values up to the last that fp32 holds, where bf16 has none left, and
    down to its least: two parts keep 2^-16 of each, or 2^-134 (half of bf16's
    smallest step)."""
    import torch
    k = rank = 8
    rng = np.random.default_rng(m)
    x, a, w = np.zeros((m, k), np.float32), np.zeros((1, rank, k), np.float32), np.zeros((1, n, rank), np.float32)
    x[:, 0], a[0, 0, 0] = E.bf16(rng.uniform(1.0, 1.9922, m).astype(np.float32)), 1.0
    x[0, 0] = 1.9921875                     # 255 / 128: times 1.7075e38 above the largest bf16
    w[0, :, 0] = b
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    base, low = torch.zeros_like(y), torch.empty(m * rank, device="cuda")
    dev = [dev16(torch, v) for v in (x, a, w)]
    ids, s = torch.zeros(m, dtype=torch.int32, device="cuda"), torch.tensor([scale], dtype=torch.float32, device="cuda")
    torch.cuda.synchronize()
    gpu_lib.lora_add_bf16(dev[0].data_ptr(), dev[1].data_ptr(), dev[2].data_ptr(), ids.data_ptr(), low.data_ptr(),
                          base.data_ptr(), y.data_ptr(), m, n, k, adapters=1, rank=rank, scales_ptr=s.data_ptr())
    torch.cuda.synchronize()
    v = x[:, 0].astype(np.float64) * float(s[0])
    assert np.abs(v).max() < 2.0 ** 128
    want = (v * b)[:, None]
    # the parts, the product's fp32 result, the store (its own smallest step with it)
    tol = (2.0 ** -16 * np.abs(v) + 2.0 ** -134)[:, None] * b + (2.0 ** -23 + E.BF16_HALF) * np.abs(want) * (1 + 2.0 ** -8) + \
        2.0 ** -134
    off = np.abs(y.double().cpu().numpy() - want)
    assert np.all(off <= tol), float(np.max(off / tol))

"""Products with bias, activation and residual (kcmm_gemm_fp8,
kcmm_gemm_bf16_epi) on the GPU against fp64 (tests/e4m3.py has the
tolerance's derivation), and bit for bit where every sum is a whole number
that fp32 holds."""
import numpy as np
import pytest

from lattice_amd.bindings import ACT_GELU, ACT_GELU_TANH, ACT_NONE, ACT_RELU, ACT_SILU
from tests import e4m3 as E

pytestmark = pytest.mark.gpu

GUARD = 64


def dev16(torch, values):
    return torch.from_numpy(E.bf16_bits(values).view(np.int16)).view(torch.bfloat16).cuda()


def host16(t):
    import torch
    return E.bf16_values(t.cpu().view(torch.int16).numpy().view(np.uint16))


def codes_of(values):
    """Values that are e4m3 values, as codes."""
    c = E.e4m3_codes(values)
    assert np.array_equal(E.e4m3_values()[c], values)
    return c


def call(torch, lib, x, w, xs=None, ws=None, bias=None, residual=None, act=ACT_NONE,
         in_place=False, stream=None):
    """y (fp32 values) of the operands' values; checks the guard behind y."""
    m, k = x.shape
    n = w.shape[0]
    y = torch.full((m * n + GUARD,), 7.0, dtype=torch.bfloat16, device="cuda")
    bd = dev16(torch, bias) if bias is not None else None
    rd = dev16(torch, residual) if residual is not None else None
    if in_place:
        y[:m * n] = rd.reshape(-1)
    st = (stream or torch.cuda.current_stream()).cuda_stream
    kw = dict(bias_ptr=bd.data_ptr() if bd is not None else 0,
              residual_ptr=(y if in_place else rd).data_ptr() if rd is not None else 0,
              activation=act, stream_ptr=st)
    if xs is None:
        xd, wd = dev16(torch, x), dev16(torch, w)
        torch.cuda.synchronize()
        lib.gemm_bf16_epi(xd.data_ptr(), wd.data_ptr(), y.data_ptr(), m, n, k, **kw)
    else:
        xd, wd = (torch.from_numpy(codes_of(v)).cuda() for v in (x, w))
        xsd, wsd = (torch.from_numpy(E.f32(v)).cuda() for v in (xs, ws))
        torch.cuda.synchronize()
        lib.gemm_fp8(xd.data_ptr(), xsd.data_ptr(), wd.data_ptr(), wsd.data_ptr(), y.data_ptr(), m,
                     n, k, **kw)
    torch.cuda.synchronize()
    assert bool((y[m * n:] == 7.0).all())
    return host16(y[:m * n]).reshape(m, n)


def inputs(rng, m, n, k, fp8, bias, residual):
    x, w = rng.standard_normal((m, k)), rng.standard_normal((n, k)) / np.sqrt(k)
    if fp8:
        xs, ws = E.row_scale(x), E.row_scale(w)
        vals = E.e4m3_values()
        x = vals[E.e4m3_codes(E.f32(x) / xs[:, None])]
        w = vals[E.e4m3_codes(E.f32(w) / ws[:, None])]
    else:
        x, w, xs, ws = E.bf16(x), E.bf16(w), None, None
    b = E.bf16(rng.standard_normal(n)) if bias else None
    r = E.bf16(rng.standard_normal((m, n))) if residual else None
    return dict(x=x, w=w, xs=xs, ws=ws, bias=b, residual=r)


def check_product(got, x, w, xs, ws, bias, residual, act):
    """Every output within the worst case, and the outputs together within what
    rounding to bf16 alone may do (an fp8 product's cut terms, 2^-13 of a
    term each and of either sign, add up to far less than that)."""
    y, s = E.product(x, w, xs, ws, bias, residual, act)
    cut = 0.0 if xs is None else E.fp8_cut(x, w, xs, ws)
    assert np.all(np.abs(got - y) <= E.product_tolerance(y, s, x.shape[1], cut))
    if y.size >= 64:
        assert np.linalg.norm(got - y) <= E.BF16_HALF * np.linalg.norm(y)


# token counts around every tile height, weight rows odd and even, rows of
# part of a 128-byte line, of whole lines, and of a line and a bit
SHAPES = [(1, 1, 16), (1, 17, 48), (2, 64, 128), (3, 130, 272), (16, 33, 1024), (17, 100, 2064),
          (31, 255, 512), (33, 64, 4096), (63, 777, 144), (64, 512, 1040), (65, 300, 2816),
          (100, 1000, 16), (128, 256, 640), (129, 257, 128), (200, 2050, 1408), (256, 512, 64),
          (257, 31, 4112), (500, 1111, 896), (777, 640, 2048), (1025, 129, 272)]


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_against_fp64(gpu_lib, m, n, k, fp8):
    import torch
    rng = np.random.default_rng([m, n, k])
    act = [ACT_NONE, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU][(m + n) % 5]
    a = inputs(rng, m, n, k, fp8, bias=n % 2 == 0 or m % 2 == 0, residual=m % 3 != 0)
    got = call(torch, gpu_lib, act=act, **a)
    check_product(got, act=act, **a)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 4096, 4096), (5, 1003, 2816), (16, 6144, 1024),
                                   (48, 2816, 1024), (64, 4096, 2048), (96, 1024, 2816),
                                   (130, 515, 1360), (256, 1024, 4096), (333, 1000, 1024),
                                   (640, 2048, 1024), (1300, 1024, 512), (2048, 1100, 144),
                                   (2300, 2304, 256)])
def test_whole_numbers_bit_for_bit(gpu_lib, m, n, k, fp8):
    """Operands of -3..3 and scales that are powers of two: every partial sum is
    a whole number below 2^24 (times a power of two), so fp32 has it exactly
    in any order, and y is the rounding of the exact result."""
    import torch
    rng = np.random.default_rng([7, m, n, k])
    x = rng.integers(-3, 4, (m, k)).astype(np.float64)
    w = rng.integers(-3, 4, (n, k)).astype(np.float64)
    bias = E.bf16(rng.integers(-100, 101, n))
    res = E.bf16(rng.integers(-100, 101, (m, n)))
    xs = ws = None
    if fp8:
        xs, ws = np.exp2(rng.integers(-1, 2, m)), np.exp2(rng.integers(-1, 2, n))
    y, s = E.product(x, w, xs, ws, bias, res, ACT_RELU)
    assert s.max() < 2 ** 20
    got = call(torch, gpu_lib, x, w, xs, ws, bias, res, ACT_RELU)
    assert np.array_equal(got, E.bf16(y))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("tile", [*range(1, 13), 100])
def test_every_tile_whole_numbers(gpu_lib, tunables, tile, fp8):
    """Each tile of the tile kernel, and the 256-row tiles (100), with the sizes
    they are not chosen for too: one token, tiles that M and N end inside, rows
    of less than a line, of one share's lines, of more; with K splits."""
    import torch
    rng = np.random.default_rng([tile, fp8])
    tunables.setenv("KCMM_EPI_TILE", str(tile))
    for splits in (1, 2, 3):
        tunables.setenv("KCMM_GEMM_SPLITS", str(splits))
        for m, n, k in [(1, 5, 16), (9, 137, 112), (33, 64, 1168), (70, 203, 2320), (130, 264, 4112),
                        (301, 520, 1024)]:
            x = rng.integers(-3, 4, (m, k)).astype(np.float64)
            w = rng.integers(-3, 4, (n, k)).astype(np.float64)
            bias = E.bf16(rng.integers(-100, 101, n))
            res = E.bf16(rng.integers(-100, 101, (m, n)))
            xs = ws = None
            if fp8:
                xs, ws = np.exp2(rng.integers(-1, 2, m)), np.exp2(rng.integers(-1, 2, n))
            y, s = E.product(x, w, xs, ws, bias, res, ACT_NONE)
            assert s.max() < 2 ** 20
            got = call(torch, gpu_lib, x, w, xs, ws, bias, res)
            assert np.array_equal(got, E.bf16(y)), (splits, m, n, k)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("act", [ACT_NONE, ACT_RELU, ACT_GELU, ACT_GELU_TANH, ACT_SILU])
def test_activations_over_their_range(gpu_lib, act, fp8):
    """x = 1 column of ones, so z is the bias: -40 .. 40, fine near zero."""
    import torch
    k = 16
    x, w = np.zeros((3, k)), np.zeros((4096, k))
    z = E.bf16(np.concatenate([np.linspace(-40, 40, 2048), np.linspace(-6, 6, 1024),
                               np.linspace(-0.01, 0.01, 1024)]))
    one = np.ones(3), np.ones(4096)
    got = call(torch, gpu_lib, x, w, *(one if fp8 else (None, None)), bias=z, act=act)
    y = E.activation(z, act)
    assert np.all(np.abs(got - y) <= E.BF16_HALF * np.abs(y) + 2.0 ** -20 * np.abs(z))


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(3, 200, 512), (70, 130, 640), (300, 1000, 512)])
def test_residual_in_place(gpu_lib, m, n, k, fp8):
    import torch
    a = inputs(np.random.default_rng(m), m, n, k, fp8, True, True)
    apart = call(torch, gpu_lib, act=ACT_SILU, **a)
    assert np.array_equal(call(torch, gpu_lib, act=ACT_SILU, in_place=True, **a), apart)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(3, 200, 512), (70, 131, 640), (300, 1000, 512), (140, 96, 4096)])
def test_slices_of_larger_buffers(gpu_lib, m, n, k, fp8):
    """Some tokens and some weight rows of larger buffers: y, residual, bias and
    scales then start at an element, not at 16 bytes; nothing else is written."""
    import torch
    t0, n0 = 5, 3                                   # what lies before them
    a = inputs(np.random.default_rng(m + n), m + t0, n + n0, k, fp8, True, True)
    bd, rd = dev16(torch, a["bias"]), dev16(torch, a["residual"][:, n0:])
    y = torch.full(((m + t0) * n + GUARD,), 7.0, dtype=torch.bfloat16, device="cuda")
    kw = dict(bias_ptr=bd.data_ptr() + 2 * n0, residual_ptr=rd.data_ptr() + 2 * t0 * n,
              activation=ACT_SILU, stream_ptr=torch.cuda.current_stream().cuda_stream)
    eb = 1 if fp8 else 2
    if fp8:
        xd, wd = (torch.from_numpy(codes_of(a[v])).cuda() for v in ("x", "w"))
        xs, ws = (torch.from_numpy(E.f32(a[v])).cuda() for v in ("xs", "ws"))
        gpu_lib.gemm_fp8(xd.data_ptr() + t0 * k, xs.data_ptr() + 4 * t0, wd.data_ptr() + n0 * k,
                         ws.data_ptr() + 4 * n0, y.data_ptr() + 2 * t0 * n, m, n, k, **kw)
    else:
        xd, wd = dev16(torch, a["x"]), dev16(torch, a["w"])
        gpu_lib.gemm_bf16_epi(xd.data_ptr() + eb * t0 * k, wd.data_ptr() + eb * n0 * k,
                              y.data_ptr() + 2 * t0 * n, m, n, k, **kw)
    torch.cuda.synchronize()
    assert bool((y[:t0 * n] == 7.0).all()) and bool((y[(m + t0) * n:] == 7.0).all())
    got = host16(y[t0 * n:(m + t0) * n]).reshape(m, n)
    xs, ws = (a["xs"][t0:], a["ws"][n0:]) if fp8 else (None, None)
    check_product(got, a["x"][t0:], a["w"][n0:], xs, ws, a["bias"][n0:], a["residual"][t0:, n0:],
                  ACT_SILU)


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(2, 100, 272), (50, 100, 272), (300, 300, 272)])
def test_not_finite_stays_in_its_row_and_column(gpu_lib, m, n, k, fp8):
    """A NaN in one token reaches that token's outputs only, one in a weight
    row that column only (k ends inside a 128-byte line; rows are padded in
    the kernels by their neighbours)."""
    import torch
    a = inputs(np.random.default_rng(m), m, n, k, fp8, False, False)
    clean = call(torch, gpu_lib, **a)
    if fp8:
        xd, wd = codes_of(a["x"]), codes_of(a["w"])
        xd[m - 1, k - 1] = 0x7f
        wd[0, 0] = 0xff
        xt, wt = torch.from_numpy(xd).cuda(), torch.from_numpy(wd).cuda()
        xs, ws = torch.from_numpy(a["xs"]).cuda(), torch.from_numpy(a["ws"]).cuda()
    else:
        x, w = a["x"].copy(), a["w"].copy()
        x[m - 1, k - 1] = np.nan
        w[0, 0] = np.inf
        xt, wt = (torch.from_numpy((v.view(np.uint32) >> 16).astype(np.uint16).view(np.int16)).cuda()
                  for v in (x, w))
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    if fp8:
        gpu_lib.gemm_fp8(xt.data_ptr(), xs.data_ptr(), wt.data_ptr(), ws.data_ptr(), y.data_ptr(),
                         m, n, k, stream_ptr=st)
    else:
        gpu_lib.gemm_bf16_epi(xt.data_ptr(), wt.data_ptr(), y.data_ptr(), m, n, k, stream_ptr=st)
    torch.cuda.synchronize()
    got = host16(y)
    assert np.all(np.isnan(got[m - 1])) and not np.any(np.isfinite(got[:, 0]))
    assert np.array_equal(got[:-1, 1:], clean[:-1, 1:])


@pytest.mark.parametrize("fp8", [False, True])
@pytest.mark.parametrize("m,n,k", [(1, 512, 4096), (64, 1024, 2048), (200, 512, 4096),
                                   (512, 2048, 1024)])
def test_same_bits_every_time_and_on_another_stream(gpu_lib, m, n, k, fp8):
    import torch
    a = inputs(np.random.default_rng(k), m, n, k, fp8, True, True)
    first = call(torch, gpu_lib, act=ACT_GELU, **a)
    side = torch.cuda.Stream()
    for st in (None, side, side):
        assert np.array_equal(call(torch, gpu_lib, act=ACT_GELU, stream=st, **a), first)


@pytest.mark.parametrize("m", [1, 200])
def test_weights_of_almost_four_gib(gpu_lib, m):
    """Byte offsets past 2^31 in the weights."""
    import torch
    n, k = 130_000, 32_768
    rng = np.random.default_rng(9)
    w = torch.zeros(n, k, dtype=torch.uint8, device="cuda")
    at = [0, 1, 70_000, n - 1]
    rows = rng.integers(-3, 4, (4, k)).astype(np.float64)
    w[torch.tensor(at, device="cuda")] = torch.from_numpy(codes_of(rows)).cuda()
    x = rng.integers(-3, 4, (m, k)).astype(np.float64)
    xd = torch.from_numpy(codes_of(x)).cuda()
    one = torch.ones(n, dtype=torch.float32, device="cuda")
    y = torch.full((m, n), 7.0, dtype=torch.bfloat16, device="cuda")
    gpu_lib.gemm_fp8(xd.data_ptr(), one.data_ptr(), w.data_ptr(), one.data_ptr(), y.data_ptr(), m,
                     n, k, stream_ptr=torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    assert np.array_equal(host16(y[:, torch.tensor(at, device="cuda")]), E.bf16(x @ rows.T))
    y[:, torch.tensor(at, device="cuda")] = 0
    assert not bool(y.any())


class Layer:
    """A plain (H, I) MLP block on 8-bit activations, as a program chains the
    calls: norm -> gate/up -> SwiGLU -> down with the residual."""

    def __init__(self, torch, lib, m, h, i, seed=1):
        g = torch.Generator(device="cuda")
        g.manual_seed(seed)
        self.torch, self.lib, self.m, self.h, self.i = torch, lib, m, h, i
        rand = lambda *s: torch.randn(*s, generator=g, device="cuda")
        self.x, self.r = rand(m, h).bfloat16(), rand(m, h).bfloat16()
        self.nw = (1 + 0.1 * rand(h)).bfloat16()
        self.w1, self.s1 = self.quant(rand(2 * i, h) / h ** 0.5)
        self.w2, self.s2 = self.quant(rand(h, i) / i ** 0.5)
        self.b1 = (0.1 * rand(2 * i)).bfloat16()
        e = lambda *s, dt: torch.empty(*s, dtype=dt, device="cuda")
        self.hid = e(m, h, dt=torch.bfloat16)
        self.c1, self.cs1 = e(m, h, dt=torch.uint8), e(m, dt=torch.float32)
        self.gu = e(m, 2 * i, dt=torch.bfloat16)
        self.c2, self.cs2 = e(m, i, dt=torch.uint8), e(m, dt=torch.float32)
        self.y = e(m, h, dt=torch.bfloat16)

    def quant(self, w):
        s = w.abs().amax(1) / 448
        return (w / s[:, None]).clamp(-448, 448).to(self.torch.float8_e4m3fn), s

    def run(self, st):
        p = lambda t: t.data_ptr()
        L, m, h, i = self.lib, self.m, self.h, self.i
        L.add_rmsnorm_fp8(p(self.x), p(self.r), p(self.nw), p(self.hid), p(self.c1), p(self.cs1),
                          m, h, 1e-5, st)
        L.gemm_fp8(p(self.c1), p(self.cs1), p(self.w1), p(self.s1), p(self.gu), m, 2 * i, h,
                   bias_ptr=p(self.b1), stream_ptr=st)
        L.silu_mul_fp8(p(self.gu), p(self.c2), p(self.cs2), m, i, st)
        L.gemm_fp8(p(self.c2), p(self.cs2), p(self.w2), p(self.s2), p(self.y), m, h, i,
                   residual_ptr=p(self.hid), stream_ptr=st)

    def reference(self):
        """fp64 of each step on what the step before it left; tolerances as in
        this file and tests/test_gpu_quant_rows.py."""
        vals = E.e4m3_values()
        n = lambda t: t.cpu().numpy()
        f = lambda c: vals[n(c.view(self.torch.uint8))]
        h, v = E.add_rmsnorm(host16(self.x), host16(self.r), host16(self.nw), 1e-5)
        assert np.array_equal(host16(self.hid), h)
        from tests.test_gpu_quant_rows import check_rows
        check_rows(n(self.c1), n(self.cs1), v, 2.0 ** -18)
        check_product(host16(self.gu), f(self.c1), f(self.w1), n(self.cs1), n(self.s1),
                      host16(self.b1), None, ACT_NONE)
        gu = host16(self.gu).astype(np.float64)
        g = gu[:, :self.i]
        check_rows(n(self.c2), n(self.cs2), g / (1 + np.exp(-g)) * gu[:, self.i:], 2.0 ** -17)
        check_product(host16(self.y), f(self.c2), f(self.w2), n(self.cs2), n(self.s2), None, h,
                      ACT_NONE)


@pytest.mark.parametrize("m,h,i", [(1, 1024, 2816), (13, 1024, 2816), (64, 2048, 1024),
                                   (150, 1024, 2816), (520, 1024, 1408)])
def test_mlp_block(gpu_lib, m, h, i):
    import torch
    b = Layer(torch, gpu_lib, m, h, i)
    b.run(torch.cuda.current_stream().cuda_stream)
    torch.cuda.synchronize()
    b.reference()


@pytest.mark.parametrize("m", [1, 40, 150, 520])
def test_mlp_block_in_a_graph(gpu_lib, m):
    """Captured on a cold stream and replayed with other inputs, eager work
    between the replays: the bits of the eager run."""
    import torch
    b = Layer(torch, gpu_lib, m, 1024, 2816)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        b.run(torch.cuda.current_stream().cuda_stream)
    for k in range(4):
        b.x.copy_(torch.randn_like(b.x))
        b.y.zero_()
        g.replay()
        torch.cuda.synchronize()
        got = b.y.clone()
        b.reference()
        b.run(torch.cuda.current_stream().cuda_stream)
        torch.cuda.synchronize()
        b.reference()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got.view(torch.int16), b.y.view(torch.int16))


@pytest.mark.parametrize("act", [ACT_SILU, ACT_GELU_TANH])
def test_activation_at_the_exponent_s_end(gpu_lib, act):
    """z sigmoid(t) where 1 / (1 + e^-t) is below the normal numbers and y is not:
    off by the store's half step and by t's roundings, at most five of 89 * 2^-24
    with log2(e)'s, and eight more of 2^-24: less than 500 * 2^-24 < 2^-15."""
    import torch
    rng = np.random.default_rng(act)
    z = E.bf16(rng.uniform(-88.5, -85, 64) if act == ACT_SILU else rng.uniform(-10.06, -9.75, 64)).astype(np.float64)
    t = z if act == ACT_SILU else np.sqrt(8 / np.pi) * (z + 0.044715 * z ** 3)
    assert t.min() > -89 and t.max() < -80
    want = z / (1 + np.exp(-t))
    assert np.abs(want).min() > 2.0 ** -126
    x, w = np.zeros((64, 16)), np.zeros((24, 16))
    x[:, 3], w[:, 3] = z, 1
    got = call(torch, gpu_lib, x, w, None, None, None, None, act)
    assert np.all(np.abs(got - want[:, None]) <= (E.BF16_HALF + 2.0 ** -15) * np.abs(want[:, None]))


@pytest.mark.parametrize("tile", [9, 100])
def test_captures_split_nothing(gpu_lib, tunables, tile):
    """A product that an eager call splits over K (with partials and a second
    kernel) is one kernel in a graph, also on a stream whose buffer is there."""
    import torch
    from tests.test_gpu_graph import _captured_kernels
    tunables.setenv("KCMM_EPI_TILE", str(tile))
    if tile == 9:
        tunables.setenv("KCMM_GEMM_SPLITS", "4")
    m, n, k = 130, 512, 4096
    x, w = (torch.randn(r, k, device="cuda").bfloat16() for r in (m, n))
    y = torch.empty(m, n, dtype=torch.bfloat16, device="cuda")

    def run(st):
        gpu_lib.gemm_bf16_epi(x.data_ptr(), w.data_ptr(), y.data_ptr(), m, n, k, stream_ptr=st)

    torch.cuda.synchronize()
    assert len(_captured_kernels(run)) == 1
    assert len(_captured_kernels(run, warm=run)) == 1


def test_calls_from_two_threads(gpu_lib, tunables):
    """Split products from two threads at once, on streams of their own and on
    one stream: each has its own partials."""
    import concurrent.futures
    import torch
    tunables.setenv("KCMM_EPI_TILE", "9")
    tunables.setenv("KCMM_GEMM_SPLITS", "4")
    m, n, k = 64, 1024, 4096
    data = []
    for i in range(2):
        x, w = (torch.randn(r, k, device="cuda").bfloat16() for r in (m, n))
        data.append((x, w, torch.empty(m, n, dtype=torch.bfloat16, device="cuda")))
    want = []
    for x, w, y in data:
        gpu_lib.gemm_bf16_epi(x.data_ptr(), w.data_ptr(), y.data_ptr(), m, n, k)
        torch.cuda.synchronize()
        want.append(y.clone())
        y.zero_()
    own = [torch.cuda.Stream() for _ in range(2)]

    def work(i, stream):
        x, w, y = data[i]
        for _ in range(50):
            gpu_lib.gemm_bf16_epi(x.data_ptr(), w.data_ptr(), y.data_ptr(), m, n, k,
                                  stream_ptr=stream.cuda_stream)

    for streams in (own, [own[0], own[0]]):
        torch.cuda.synchronize()
        with concurrent.futures.ThreadPoolExecutor(2) as ex:
            for f in [ex.submit(work, i, streams[i]) for i in range(2)]:
                f.result()
        torch.cuda.synchronize()
        for (x, w, y), v in zip(data, want):
            assert torch.equal(y.view(torch.int16), v.view(torch.int16))
            y.zero_()


def test_two_graphs_of_one_stream_at_once(gpu_lib):
    """Two captures from the same stream, replayed on two streams at the same
    time: nothing that they share."""
    import torch
    blocks = [Layer(torch, gpu_lib, m, 1024, 2816, seed=m) for m in (150, 170)]
    st = torch.cuda.Stream()
    graphs = []
    for b in blocks:
        b.run(st.cuda_stream)          # whatever an eager call keeps is there
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=st):
            b.run(torch.cuda.current_stream().cuda_stream)
        graphs.append(g)
    sides = [torch.cuda.Stream() for _ in graphs]
    for _ in range(20):
        for g, s in zip(graphs, sides):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for b in blocks:
        b.reference()

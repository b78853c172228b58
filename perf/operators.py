"""The operators of a decoder layer whose products read 8-bit activations, as
measurable cases: their plain forms in elementary torch operations, and the
calls that a program makes of this package's kernels.

  norm   residual add + RMSNorm, e4m3 codes with an fp32 scale per row
         (KcmmLibrary.add_rmsnorm_fp8): before the QKV and gate/up products;
  quant  a row's e4m3 codes and scale (quant_rows_fp8): the attention's
         output before the O product;
  silu   SwiGLU of the [gate | up] row, as codes and scale (silu_mul_fp8):
         before the down product;
  gemm8  codes times codes with both scales, bias, activation and residual in
         the epilogue (gemm_fp8);
  gemm16 the same epilogue on bf16 operands (gemm_bf16_epi).

Sizes are those of this repository's configurations and benchmark (hidden
4096, intermediate 14336, 32/8 heads of 128; the smaller 2048/8192 and
1024/2816 models of perf/cases.py), from one token to whole prompts.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-5
E4M3_MAX = 448.0
ACTS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # one sequence's decode step: the shortest call, a launch and its latency
        dict(name="norm_one", kind="norm", rows=1, cols=4096, residual=True),
        # the benchmark's decode batch
        dict(name="norm_batch64", kind="norm", rows=64, cols=4096, residual=True),
        # a long prompt's tokens
        dict(name="norm_prompt8192", kind="norm", rows=8192, cols=4096, residual=True),
        # the attention output of ragged prompts, small model
        dict(name="quant_prompt1111", kind="quant", rows=1111, cols=2048),
        # the MLP's inner row of the decode batch
        dict(name="silu_batch64", kind="silu", rows=64, cols=14336),
        # ... and of a prompt chunk
        dict(name="silu_prompt2048", kind="silu", rows=2048, cols=14336),
        # biased QKV projection of one token: the weights' way from memory
        dict(name="gemm8_one_qkv", kind="gemm8", m=1, n=6144, k=4096, bias=True, act="none",
             residual=False),
        # gate/up of the decode batch
        dict(name="gemm8_batch64_up", kind="gemm8", m=64, n=28672, k=4096, bias=False, act="none",
             residual=False),
        # down projection of a prompt chunk with its residual
        dict(name="gemm8_prompt2048_down", kind="gemm8", m=2048, n=4096, k=14336, bias=False,
             act="none", residual=True),
        # a small model's plain MLP for a handful of tokens
        dict(name="gemm16_few_mlp", kind="gemm16", m=13, n=2816, k=1024, bias=True, act="gelu",
             residual=False),
        # O projection with bias and residual of a ragged few hundred tokens
        dict(name="gemm16_777_o", kind="gemm16", m=777, n=4096, k=4096, bias=True, act="none",
             residual=True),
        # a plain MLP's inner product for a prompt chunk
        dict(name="gemm16_prompt2048_mlp", kind="gemm16", m=2048, n=14336, k=4096, bias=True,
             act="gelu_tanh", residual=False),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """One more case, the kind as often as it is listed, sizes over the log
    of their ranges; the weights' rows (n) odd as often as not."""
    kind = rng.choice(["norm"] * 3 + ["quant"] + ["silu"] * 2 + ["gemm8"] * 3 + ["gemm16"] * 3)
    if kind in ("norm", "quant", "silu"):
        cols = 8 * _log_int(rng, 8, {"norm": 1024, "quant": 2048, "silu": 3584}[kind])
        rows = _log_int(rng, 1, min(8192, (1 << 25) // cols))
        c = dict(kind=kind, rows=rows, cols=cols)
        if kind == "norm":
            c["residual"] = rng.random() < 0.75
        return c
    m = _log_int(rng, 1, 4096)
    k = 16 * _log_int(rng, 4, 896)
    n = _log_int(rng, 64, min(65536, 28672 * 4096 // k, 30_000_000 // m,
                              (2048 * 4096 * 14336) // (m * k)))
    if rng.random() < 0.5 and n > 64:
        n = n // 64 * 64
    return dict(kind=kind, m=m, n=n, k=k, bias=rng.random() < 0.6,
                act=rng.choice(["none", "none", "relu", "gelu", "gelu_tanh", "silu"]),
                residual=rng.random() < 0.5)


# ---- what a program holds before the call ----------------------------------------------------------

def _codes(v):
    """Rows as e4m3 codes and fp32 scales (how a checkpoint's weights are made)."""
    s = v.abs().amax(1).clamp_min(1e-30) / E4M3_MAX
    return (v / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def _activations(g, rows, cols):
    """Unit-variance rows whose channels differ in size, some by a lot."""
    d = "cuda"
    ch = torch.exp(0.7 * torch.randn(cols, generator=g, device=d))
    tok = torch.exp(0.3 * torch.randn(rows, 1, generator=g, device=d))
    return torch.randn(rows, cols, generator=g, device=d) * ch * tok


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    d, bf = "cuda", torch.bfloat16
    s = dict(case)
    if case["kind"] in ("norm", "quant", "silu"):
        rows, cols = case["rows"], case["cols"]
        s["x"] = _activations(g, rows, 2 * cols if case["kind"] == "silu" else cols).to(bf)
        if case["kind"] == "norm":
            s["w"] = (1.0 + 0.2 * torch.randn(cols, generator=g, device=d)).to(bf)
            s["r"] = (3.0 * torch.randn(rows, cols, generator=g, device=d)).to(bf) \
                if case["residual"] else None
            s["hidden"] = torch.empty(rows, cols, dtype=bf, device=d)
        s["codes"] = torch.empty(rows, cols, dtype=torch.float8_e4m3fn, device=d)
        s["scales"] = torch.empty(rows, dtype=torch.float32, device=d)
        return s
    m, n, k = case["m"], case["n"], case["k"]
    x = _activations(g, m, k)
    w = torch.randn(n, k, generator=g, device=d) * (1.0 / math.sqrt(k))
    if case["kind"] == "gemm8":
        s["x"], s["xs"] = _codes(x.to(bf).float())
        s["w"], s["ws"] = _codes(w)
    else:
        s["x"], s["w"] = x.to(bf), w.to(bf)
    s["b"] = (0.5 * torch.randn(n, generator=g, device=d)).to(bf) if case["bias"] else None
    s["r"] = torch.randn(m, n, generator=g, device=d).to(bf) if case["residual"] else None
    s["y"] = torch.empty(m, n, dtype=bf, device=d)
    return s


# ---- plain forms -----------------------------------------------------------------------------------

def _plain_rows(v):
    """fp32 rows -> (codes, scales)."""
    a = torch.where(torch.isfinite(v), v.abs(), torch.zeros_like(v)).amax(1)
    s = torch.where(a > 0, (a / E4M3_MAX).clamp_min(2.0 ** -126), torch.ones_like(a))
    return (v / s[:, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), s


def _plain_act(z, act):
    if act == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if act == "gelu":
        return 0.5 * z * torch.erfc(z * -math.sqrt(0.5))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        h = s["x"] if s["r"] is None else (s["x"].float() + s["r"].float()).to(torch.bfloat16)
        f = h.float()
        v = f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * s["w"].float()
        codes, scales = _plain_rows(v)
        return {"codes": codes, "scales": scales, **({} if s["r"] is None else {"hidden": h})}
    if kind == "quant":
        codes, scales = _plain_rows(s["x"].float())
        return {"codes": codes, "scales": scales}
    if kind == "silu":
        gate, up = s["x"].float().split(s["cols"], 1)
        codes, scales = _plain_rows(gate / (1.0 + torch.exp(-gate)) * up)
        return {"codes": codes, "scales": scales}
    z = s["x"].float() @ s["w"].float().t()
    if kind == "gemm8":
        z = z * s["xs"][:, None] * s["ws"][None, :]
    if s["b"] is not None:
        z = z + s["b"].float()
    z = _plain_act(z, s["act"])
    if s["r"] is not None:
        z = z + s["r"].float()
    return {"y": z.to(torch.bfloat16)}


# ---- the package's calls ---------------------------------------------------------------------------

_lib = None


def _own(s):
    global _lib
    if _lib is None:
        from lattice_amd.bindings import KcmmLibrary
        _lib = KcmmLibrary()
    st = torch.cuda.current_stream().cuda_stream
    kind, ptr = s["kind"], lambda t: 0 if t is None else t.data_ptr()
    if kind == "norm":
        has = s["r"] is not None
        _lib.add_rmsnorm_fp8(ptr(s["x"]), ptr(s["r"]), ptr(s["w"]),
                             ptr(s["hidden"]) if has else 0, ptr(s["codes"]), ptr(s["scales"]),
                             s["rows"], s["cols"], EPS, st)
        return {"codes": s["codes"], "scales": s["scales"],
                **({"hidden": s["hidden"]} if has else {})}
    if kind == "quant":
        _lib.quant_rows_fp8(ptr(s["x"]), ptr(s["codes"]), ptr(s["scales"]), s["rows"], s["cols"],
                            st)
        return {"codes": s["codes"], "scales": s["scales"]}
    if kind == "silu":
        _lib.silu_mul_fp8(ptr(s["x"]), ptr(s["codes"]), ptr(s["scales"]), s["rows"], s["cols"], st)
        return {"codes": s["codes"], "scales": s["scales"]}
    epi = dict(bias_ptr=ptr(s["b"]), residual_ptr=ptr(s["r"]), activation=ACTS[s["act"]],
               stream_ptr=st)
    if kind == "gemm8":
        _lib.gemm_fp8(ptr(s["x"]), ptr(s["xs"]), ptr(s["w"]), ptr(s["ws"]), ptr(s["y"]), s["m"],
                      s["n"], s["k"], **epi)
    else:
        _lib.gemm_bf16_epi(ptr(s["x"]), ptr(s["w"]), ptr(s["y"]), s["m"], s["n"], s["k"], **epi)
    return {"y": s["y"]}


def run(state):
    if own:
        return _own(state)
    return _plain(state)


# ---- sizes and the definition in 64 bits --------------------------------------------------------------

def work(case):
    if case["kind"] in ("norm", "quant", "silu"):
        e = case["rows"] * case["cols"]
        per = {"norm": 7 if case.get("residual") else 3, "quant": 3, "silu": 5}[case["kind"]]
        b = e * per + 4 * case["rows"] + (2 * case["cols"] if case["kind"] == "norm" else 0)
        return {"bytes": b, "flops": e * {"norm": 8, "quant": 3, "silu": 9}[case["kind"]]}
    m, n, k = case["m"], case["n"], case["k"]
    e = 1 if case["kind"] == "gemm8" else 2
    b = e * (m * k + n * k) + 2 * m * n
    b += 4 * (m + n) if e == 1 else 0
    b += 2 * n if case["bias"] else 0
    b += 2 * m * n if case["residual"] else 0
    return {"bytes": b, "flops": 2 * m * n * k}


def _grid(v, bits, least):
    """v (fp64) to the nearest value of `bits` significant bits, ties to even,
    on the fixed grid of the exponent `least` below it."""
    e = torch.frexp(v.abs())[1].to(torch.float64) - 1.0      # |v| = m 2^e, 1 <= m < 2
    step = torch.exp2(e.clamp_min(float(least)) - (bits - 1))
    return torch.round(v / step) * step


def exact(case, seed):
    s = prepare(case, seed)
    kind = s["kind"]
    if kind in ("norm", "quant", "silu"):
        out = {}
        v = s["x"].double()
        if kind == "norm":
            if s["r"] is not None:
                out["hidden"] = v + s["r"].double()
                v = _grid(out["hidden"], 8, -126)
            v = v / (v.square().sum(1, keepdim=True) / s["cols"] + EPS).sqrt() * s["w"].double()
        elif kind == "silu":
            up = v[:, s["cols"]:]
            v = v[:, :s["cols"]]
            v = v * torch.sigmoid(v) * up
        a = v.abs().max(1).values
        scale = a / 448
        scale[a == 0] = 1
        # the codes stand for multiples of the scale that is stored, an fp32
        out["codes"] = _grid(v / scale.float().double()[:, None], 4, -6)
        out["scales"] = scale
        return out
    z = s["x"].double() @ s["w"].double().t()
    if kind == "gemm8":
        z *= s["xs"].double()[:, None]
        z *= s["ws"].double()
    if s["b"] is not None:
        z += s["b"].double()
    act = s["act"]
    if act == "relu":
        z = z.clamp_min(0)
    elif act == "gelu":
        z = z * torch.special.ndtr(z)
    elif act == "gelu_tanh":
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    elif act == "silu":
        z = z * torch.sigmoid(z)
    if s["r"] is not None:
        z += s["r"].double()
    return {"y": z}

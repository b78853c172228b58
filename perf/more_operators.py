"""Operators around the paged cache when many requests share a prompt, come as
whole chunks, or bring their own adapters, as measurable cases: their plain
forms in elementary torch operations, and the calls that a program makes of
this package's kernels.

  attn    decode attention of a batch whose sequences share long prefixes in
          groups: the prefix read and multiplied once for a group, the rest
          of each sequence by itself (KcmmPool.paged_attn_decode_shared);
  append  a prompt chunk's q and k rotated by their positions (one axis, or
          time / height / width for images) and k, v written into the pages,
          packed sequences of different lengths
          (KcmmPool.rope_append_chunk);
  lora    low-rank adapters of many requests at once, added to what the
          shared projection gave (KcmmLibrary.lora_add_bf16).

Sizes are those of this repository's configurations and benchmark (32/8 heads
of 128, hidden 4096, intermediate 14336; the smaller 16/4 and 8/8 heads of
64), pages of 16 or 32 tokens.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

SB = 2 << 20            # a pool lays its pages into superblocks of this size
E4M3_MAX = 448.0
TORCH = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.bfloat16, "f32": torch.float32}


# ---- the cases ---------------------------------------------------------------------------------

def listed():
    return [
        # two chats behind one system prompt: the shortest call, launches and latency
        dict(name="attn_two_chats", kind="attn", dtype="bf16", batch=2, groups=1, plo=700, phi=700,
             slo=20, shi=200, hq=32, hkv=8, d=128, bs=16, lens=1),
        # the benchmark's decode batch, all behind one 2048-token prompt
        dict(name="attn_batch64_prompt2048", kind="attn", dtype="bf16", batch=64, groups=1,
             plo=2048, phi=2048, slo=64, shi=512, hq=32, hkv=8, d=128, bs=16, lens=2),
        # 32 requests of four beams each on fp8 pages, contexts that end inside a page
        dict(name="attn_beams128_fp8", kind="attn", dtype="fp8", batch=128, groups=32, plo=1024,
             phi=8192, slo=1, shi=64, hq=32, hkv=8, d=128, bs=16, lens=3),
        # three long documents, sixteen questions to each, 64-wide heads
        dict(name="attn_documents_f16", kind="attn", dtype="f16", batch=48, groups=3, plo=12000,
             phi=16384, slo=100, shi=1000, hq=16, hkv=4, d=64, bs=16, lens=4),
        # a few drafted tokens of eight sequences, to be verified: latency
        dict(name="append_drafts", kind="append", dtype="bf16", batch=8, first=1000, lo=1, hi=6,
             axes=0, interleave=False, hq=32, hkv=8, d=128, bs=16, lens=5),
        # ragged prompts from their first token
        dict(name="append_prompts", kind="append", dtype="bf16", batch=4, first=0, lo=300, hi=1900,
             axes=0, interleave=False, hq=32, hkv=8, d=128, bs=16, lens=6),
        # the later chunk of ragged prompts, from inside a page, into fp8 pages
        dict(name="append_prompts_fp8", kind="append", dtype="fp8", batch=3, first=1111, lo=300,
             hi=1900, axes=0, interleave=False, hq=32, hkv=8, d=128, bs=16, lens=7),
        # images and text of two long requests, three axes, an f16 pool
        dict(name="append_images_f16", kind="append", dtype="f16", batch=2, first=0, lo=3900,
             hi=4096, axes=3, interleave=False, hq=32, hkv=8, d=128, bs=16, lens=8),
        # one request's decode step, O projection: latency
        dict(name="lora_one", kind="lora", m=1, requests=1, adapters=4, rank=16, k=4096,
             widths="4096", none=0.0, lens=9),
        # the decode batch's QKV projection, requests of sixteen adapters mixed, some without
        dict(name="lora_batch64_qkv", kind="lora", m=64, requests=64, adapters=16, rank=16, k=4096,
             widths="4096,1024,1024", none=0.2, lens=10),
        # ... its down projection, higher rank
        dict(name="lora_batch64_down", kind="lora", m=64, requests=64, adapters=8, rank=64, k=14336,
             widths="4096", none=0.1, lens=11),
        # gate and up of six ragged prompts
        dict(name="lora_prompts_up", kind="lora", m=3001, requests=6, adapters=4, rank=32, k=4096,
             widths="14336,14336", none=0.2, lens=12),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


HEADS = [(32, 8, 128), (32, 8, 64), (16, 4, 64), (8, 8, 64), (32, 4, 128), (16, 8, 128)]


def draw(rng):
    """One more case, the kind as often as it is listed, sizes over the log of
    their ranges."""
    kind = rng.choice(["attn", "append", "lora"])
    lens = rng.randrange(1 << 30)
    if kind == "lora":
        slices = rng.choice([1, 1, 2, 3])
        m = _log_int(rng, 1, 3000)
        rank = 8 * rng.choice([1, 2, 2, 3, 4, 8])
        # (no more work than the largest listed case)
        k = 8 * _log_int(rng, 32, min(14336, 3000 * 64 * 4096 // (m * slices * rank)) // 8)
        most = min(14336, 2400 * 28672 // (slices * m), 2800 * 28672 * 32 // (slices * m * rank)) // 16
        widths = [16 * _log_int(rng, 16, most) for _ in range(slices)]
        return dict(kind=kind, m=m, requests=rng.choice([m, max(1, m // 500)]),
                    adapters=_log_int(rng, 1, 16), rank=rank, k=k,
                    widths=",".join(map(str, widths)), none=rng.choice([0.0, 0.2]), lens=lens)
    dtype = rng.choice(["bf16", "bf16", "f16", "fp8"])
    hq, hkv, d = rng.choice(HEADS)
    if dtype == "fp8":
        d = 128
    c = dict(kind=kind, dtype=dtype, hq=hq, hkv=hkv, d=d, bs=rng.choice([16, 16, 32]), lens=lens)
    if kind == "attn":
        batch = _log_int(rng, 1, 128)
        phi = _log_int(rng, 32, min(16384, 500_000 // batch))
        shi = _log_int(rng, 1, min(1024, 20_000 // batch))
        groups = _log_int(rng, 1, max(1, min(batch, 48_000 // phi)))
        return dict(c, batch=batch, groups=groups, plo=max(1, phi // rng.choice([1, 3])), phi=phi,
                    slo=max(1, shi // 8), shi=shi)
    batch = _log_int(rng, 1, 32)
    hi = _log_int(rng, 1, 8000 // batch)
    return dict(c, batch=batch, first=rng.choice([0, 0, _log_int(rng, 1, 4096)]),
                lo=max(1, hi // 4), hi=hi, axes=rng.choice([0, 0, 1, 3]),
                interleave=rng.random() < 0.5)


# ---- what a program holds before the call ----------------------------------------------------------

def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _page_bytes(case):
    """Bytes of a page, and of its elements (fp8 pages: a footer of one fp32
    scale per kv head, padded to 256 bytes)."""
    data = case["bs"] * case["hkv"] * case["d"] * {"fp8": 1, "f32": 4}.get(case["dtype"], 2)
    return (-(-(data + 4 * case["hkv"]) // 256) * 256 if case["dtype"] == "fp8" else data), data


def _pages(case, g, count):
    """At least `count` pages of K or V as a pool lays them, [superblocks][pages
    of one][bs][hkv][d], and for fp8 pages their scales."""
    per = SB // _page_bytes(case)[0]
    shape = (-(-count // per), per, case["bs"], case["hkv"], case["d"])
    x = torch.randn(shape, generator=g, device="cuda")
    if case["dtype"] != "fp8":
        return x.to(TORCH[case["dtype"]]), None
    s = x.abs().amax((2, 4)) / E4M3_MAX
    return (x / s[:, :, None, :, None]).to(torch.float8_e4m3fn), s


def _layout(case):
    """Lengths and tables of page numbers: of attn with the pages of whole
    shared blocks in every table of the group, of append a page each."""
    r = np.random.default_rng(case["lens"])
    batch, bs = case["batch"], case["bs"]
    if case["kind"] == "attn":
        starts = np.sort(r.choice(np.arange(1, batch), size=case["groups"] - 1, replace=False)) \
            if case["groups"] > 1 else np.zeros(0, np.int64)
        starts = np.concatenate([[0], starts, [batch]]).astype(np.int32)
        group = np.repeat(np.arange(case["groups"]), np.diff(starts))
        shared = r.integers(case["plo"], case["phi"] + 1, size=case["groups"])[group]
        total = shared + r.integers(case["slo"], case["shi"] + 1, size=batch)
        leader = starts[group]
    else:
        starts = np.concatenate([[0], np.cumsum(r.integers(case["lo"], case["hi"] + 1, size=batch))])
        total = case["first"] + np.diff(starts)
        shared, leader = np.zeros(batch, np.int64), np.arange(batch)
    blocks = -(-total // bs)
    full = np.where(leader == np.arange(batch), 0, shared // bs)   # blocks taken from the leader
    need = blocks - full
    numbers = r.permutation(int(need.sum()) + 3)    # and some pages of no sequence
    at = np.concatenate([[0], np.cumsum(need)])
    table = np.zeros((batch, int(blocks.max())), np.int64)
    for b in range(batch):
        table[b, full[b]:blocks[b]] = numbers[at[b]:at[b + 1]]
        table[b, :full[b]] = table[leader[b], :full[b]]
    return dict(starts=starts.astype(np.int32), shared=shared.astype(np.int32),
                total=total.astype(np.int32), leader=leader, table=table, pages=len(numbers))


def _pair_axes(case):
    """The axis of each rotated pair: a quarter time, the rest height and width,
    in sections or dealt in turn."""
    half = case["d"] // 2
    if case["axes"] != 3:
        return [0] * half
    t = half // 4
    h = (half - t) // 2
    if case["interleave"]:
        return [i % 3 if i < 3 * t else 1 + i % 2 for i in range(half)]
    return [0] * t + [1] * h + [2] * (half - t - h)


def _positions(case, lay):
    """Three axes: a request's text, then images of 24 x 32 patches, then text."""
    if not case["axes"]:
        return None
    n = np.diff(lay["starts"])
    i = np.concatenate([np.arange(x) for x in n]) + case["first"]
    if case["axes"] == 1:
        return i[None].astype(np.int32)
    image = (i // 768) % 4 == 1
    p, at = i % 768, i - i % 768
    return np.stack([np.where(image, at, i), np.where(image, at + p // 32, i),
                     np.where(image, at + p % 32, i)]).astype(np.int32)


def prepare(case, seed):
    g = _generator(seed)
    d, s = "cuda", dict(case)
    if case["kind"] == "lora":
        bf = torch.bfloat16
        m, k, rank = case["m"], case["k"], case["rank"]
        widths = [int(w) for w in case["widths"].split(",")]
        n, rows = sum(widths), len(widths) * rank
        r = np.random.default_rng(case["lens"])
        cuts = np.sort(r.choice(np.arange(1, m), size=case["requests"] - 1, replace=False)) \
            if case["requests"] > 1 else np.zeros(0, np.int64)
        each = np.where(r.random(case["requests"]) < case["none"], -1,
                        r.integers(0, case["adapters"], size=case["requests"]))
        ids = np.repeat(each, np.diff(np.concatenate([[0], cuts, [m]])))
        s["ids"] = torch.from_numpy(ids.astype(np.int32)).to(d)
        s["x"] = torch.randn(m, k, generator=g, device=d).to(bf)
        s["a"] = (torch.randn(case["adapters"], rows, k, generator=g, device=d) / math.sqrt(k)).to(bf)
        s["b"] = (torch.randn(case["adapters"], n, rank, generator=g, device=d) / math.sqrt(rank)).to(bf)
        s["scales"] = 0.5 + torch.rand(case["adapters"], generator=g, device=d)
        s["base"] = torch.randn(m, n, generator=g, device=d).to(bf)
        s["low"] = torch.empty(m, rows, device=d)
        s["y"] = torch.empty(m, n, dtype=bf, device=d)
        s["slice"] = torch.from_numpy(np.repeat(np.arange(len(widths)), widths)).to(d)
        s["ends"] = np.cumsum(widths).tolist()
        return s
    lay = _layout(case)
    s["k"], s["ks"] = _pages(case, g, lay["pages"])
    s["v"], s["vs"] = _pages(case, g, lay["pages"])
    s["table"] = torch.from_numpy(lay["table"]).to(d)
    s["total"] = torch.from_numpy(lay["total"]).to(d)
    s["starts"] = torch.from_numpy(lay["starts"]).to(d)
    hq, hkv, dim = case["hq"], case["hkv"], case["d"]
    if case["kind"] == "attn":
        # the block that a prefix ends in is each sequence's own copy
        cut, at = lay["shared"] % case["bs"], lay["shared"] // case["bs"]
        for b in np.nonzero((cut > 0) & (lay["leader"] != np.arange(case["batch"])))[0]:
            here, there = int(lay["table"][b, at[b]]), int(lay["table"][lay["leader"][b], at[b]])
            for pages, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
                pages.flatten(0, 1)[here, :cut[b]] = pages.flatten(0, 1)[there, :cut[b]]
                if scales is not None:
                    scales.flatten(0, 1)[here] = scales.flatten(0, 1)[there]
        s["shared"] = torch.from_numpy(lay["shared"]).to(d)
        s["q"] = (2.0 * torch.randn(case["batch"], hq, dim, generator=g, device=d)).to(TORCH[case["dtype"]])
        s["out"] = torch.empty_like(s["q"])
    else:
        t = s["tokens"] = int(lay["starts"][-1])
        s["qkv"] = torch.randn(t, (hq + 2 * hkv) * dim, generator=g, device=d).to(TORCH[case["dtype"]])
        s["q_out"] = torch.empty(t, hq, dim, dtype=s["qkv"].dtype, device=d)
        s["inv_freq"] = (500000.0 ** (-torch.arange(0, dim, 2, dtype=torch.float64, device=d) / dim)).float()
        s["pair_axes"] = _pair_axes(case)
        s["axis"] = torch.tensor(s["pair_axes"], device=d)
        p = _positions(case, lay)
        s["positions"] = None if p is None else torch.from_numpy(p).to(d)
    if own:
        _handle(s, lay)    # the pool, and its own memory in the place of the pages
    return s


# ---- plain forms -----------------------------------------------------------------------------------

def _rows(pages, scales, index):
    """Rows `index` of the pages' tokens, in 32 bits."""
    x = pages.flatten(0, 2)[index].float()
    if scales is not None:
        x = x * scales.flatten(0, 1)[index // pages.shape[2]][..., None]
    return x


def _plain_attn(s):
    batch, hkv, dim, bs = s["batch"], s["hkv"], s["d"], s["bs"]
    at = torch.arange(s["table"].shape[1] * bs, device="cuda")
    index = s["table"][:, at // bs] * bs + at % bs
    k = _rows(s["k"], s["ks"], index)                                  # [B][L][hkv][d]
    q = s["q"].float().view(batch, hkv, -1, dim) / math.sqrt(dim)
    score = q @ k.permute(0, 2, 3, 1)
    del k
    score = score.masked_fill(at >= s["total"][:, None, None, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    o = p @ _rows(s["v"], s["vs"], index).transpose(1, 2) / p.sum(-1, keepdim=True)
    return {"out": o.reshape(batch, -1, dim).to(s["q"].dtype)}


def _write_fp8(pages, scales, page, slot, x):
    """x [T][hkv][d] into (page, slot): the rows of a page as one set."""
    codes, sc = pages.flatten(0, 1), scales.flatten(0, 1)
    n, hkv = sc.shape
    amax = torch.zeros_like(sc).scatter_reduce(0, page[:, None].expand(-1, hkv), x.abs().amax(2), "amax")
    touched = torch.zeros(n, dtype=torch.bool, device="cuda").index_fill(0, page, True)
    first = torch.zeros(n, dtype=torch.int32, device="cuda").scatter_reduce(
        0, page, (slot == 0).int(), "amax").bool()
    fresh = first[:, None] | ~(torch.isfinite(sc) & (sc > 0))
    own_scale = torch.where(amax > 0, amax / E4M3_MAX, torch.ones_like(amax))
    grown = ~fresh & (amax > E4M3_MAX * sc)
    new = torch.where(touched[:, None] & (fresh | grown), own_scale, sc)
    again = ((codes.float() * sc[:, None, :, None]) / new[:, None, :, None]).clamp(-E4M3_MAX, E4M3_MAX)
    again = again.to(torch.float8_e4m3fn).view(torch.uint8)
    bits = codes.view(torch.uint8)
    bits.copy_(torch.where((touched[:, None] & grown)[:, None, :, None], again, bits))
    bits[page, slot] = (x / new[page][..., None]).clamp(-E4M3_MAX, E4M3_MAX) \
        .to(torch.float8_e4m3fn).view(torch.uint8)
    sc.copy_(new)


def _plain_append(s):
    t, hq, hkv, dim, bs = s["tokens"], s["hq"], s["hkv"], s["d"], s["bs"]
    token = torch.arange(t, device="cuda")
    b = torch.searchsorted(s["starts"], token.int(), right=True) - 1
    place = s["total"][b] - s["starts"][b + 1] + token            # in the cache
    page, slot = s["table"][b, place // bs], place % bs
    at = place[:, None] if s["positions"] is None else s["positions"][s["axis"]].t()
    angle = at.double() * s["inv_freq"].double()
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]
    rows = s["qkv"].view(t, hq + 2 * hkv, dim)
    x1, x2 = rows[:, :hq + hkv].float().chunk(2, -1)
    y = torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1)
    k, v = y[:, hq:], rows[:, hq + hkv:].float()
    out = {"q": y[:, :hq].to(rows.dtype), "k": s["k"], "v": s["v"]}
    if s["ks"] is not None:
        _write_fp8(s["k"], s["ks"], page, slot, k)
        _write_fp8(s["v"], s["vs"], page, slot, v)
        return dict(out, ks=s["ks"], vs=s["vs"])
    s["k"].flatten(0, 1)[page, slot] = k.to(rows.dtype)
    s["v"].flatten(0, 1)[page, slot] = v.to(rows.dtype)
    return out


def _plain_lora(s):
    n_a, rank = s["adapters"], s["rank"]
    mine = s["ids"][:, None] == torch.arange(n_a, device="cuda")             # [m][adapters]
    low = s["x"].float() @ s["a"].float().flatten(0, 1).t()                  # [m][adapters * rows]
    low = low.view(s["m"], n_a, -1, rank)
    low = torch.where(mine[:, :, None, None], low * s["scales"][:, None, None], torch.zeros_like(low))
    # each slice's weights on its own rows of the low-rank values, zeros elsewhere
    which = s["slice"][:, None] == torch.arange(low.shape[2], device="cuda")   # [n][slices]
    b = (s["b"].float()[:, :, None, :] * which[:, :, None]).permute(1, 0, 2, 3).flatten(1)
    return {"y": (s["base"].float() + low.flatten(1) @ b.t()).to(torch.bfloat16)}


# ---- the package's calls ---------------------------------------------------------------------------

_lib = None


def _library():
    global _lib
    if _lib is None:
        from lattice_amd.bindings import KcmmLibrary
        _lib = KcmmLibrary()
    return _lib


class _Pool:
    """Frees the pool's memory with the state that holds it."""

    def __init__(self, pool):
        self.pool = pool

    def __del__(self):
        self.pool.destroy()


class _Region:
    """Device memory of the pool, for torch to see it in place; keeps the pool."""

    def __init__(self, owner, ptr, nbytes):
        self.owner = owner
        self.__cuda_array_interface__ = {"shape": (nbytes,), "typestr": "|u1",
                                         "data": (ptr, False), "version": 3}


def _handle(s, lay):
    from lattice_amd.bindings import KV_BF16, KV_F16, KV_F32, KV_FP8, make_config
    bb, data = _page_bytes(s)
    blocks, per = s["k"].shape[:2]
    cfg = make_config(num_layers=1, kv_heads=s["hkv"], head_dim=s["d"], max_batch=s["batch"],
                      max_seq_len=blocks * per * s["bs"], block_size=s["bs"], max_blocks=blocks * per)
    pool = _library().create_pool(cfg, {"bf16": KV_BF16, "f16": KV_F16, "fp8": KV_FP8,
                                        "f32": KV_F32}[s["dtype"]])
    s["pool"], s["keep"] = pool, _Pool(pool)
    ids = np.asarray(pool.alloc_blocks(blocks * per))
    offs = np.asarray(pool.all_block_offsets_f16(), np.uint64)
    at = offs[ids].astype(np.int64) * 2
    id_of = np.empty(blocks * per, np.int64)
    id_of[at // SB * per + at % SB // bb] = ids
    s["ids_table"] = torch.from_numpy(id_of[lay["table"]].astype(np.int32)).cuda()
    s["offs"] = torch.from_numpy(offs.view(np.int64)).cuda()
    for name, base in (("k", pool.va_k(0)), ("v", pool.va_v(0))):
        raw = torch.as_tensor(_Region(s["keep"], base, blocks * SB), device="cuda")
        pages = raw.view(blocks, SB)[:, :per * bb].view(blocks, per, bb)
        mine = pages[:, :, :data].view(s[name].dtype).unflatten(2, tuple(s[name].shape[2:]))
        mine.view(torch.uint8).copy_(s[name].view(torch.uint8))
        s[name] = mine
        if s[name + "s"] is not None:
            foot = pages[:, :, data:data + 4 * s["hkv"]].view(torch.float32)
            foot.copy_(s[name + "s"])
            s[name + "s"] = foot
    if s["kind"] == "attn":
        s["scratch"] = torch.empty(pool.shared_scratch_bytes(s["batch"], s["hq"], s["table"].shape[1]),
                                   dtype=torch.uint8, device="cuda")


def _own(s):
    st = torch.cuda.current_stream().cuda_stream
    if s["kind"] == "lora":
        _library().lora_add_bf16(
            s["x"].data_ptr(), s["a"].data_ptr(), s["b"].data_ptr(), s["ids"].data_ptr(),
            s["low"].data_ptr(), s["base"].data_ptr(), s["y"].data_ptr(), s["m"], s["ends"][-1],
            s["k"], adapters=s["adapters"], rank=s["rank"], slice_ends=s["ends"],
            scales_ptr=s["scales"].data_ptr(), stream_ptr=st)
        return {"y": s["y"]}
    if s["kind"] == "attn":
        s["pool"].paged_attn_decode_shared(
            layer_idx=0, query_ptr=s["q"].data_ptr(), out_ptr=s["out"].data_ptr(),
            block_tables_ptr=s["ids_table"].data_ptr(), seq_lens_ptr=s["total"].data_ptr(),
            shared_lens_ptr=s["shared"].data_ptr(), group_starts_ptr=s["starts"].data_ptr(),
            block_offsets_f16_ptr=s["offs"].data_ptr(), scratch_ptr=s["scratch"].data_ptr(),
            scratch_bytes=s["scratch"].numel(), batch=s["batch"], num_groups=s["groups"],
            num_q_heads=s["hq"], kv_heads=s["hkv"], head_dim=s["d"], block_size=s["bs"],
            max_blocks_per_seq=s["table"].shape[1], scale=1.0 / math.sqrt(s["d"]), stream_ptr=st)
        return {"out": s["out"]}
    p = s["positions"]
    s["pool"].rope_append_chunk(
        layer_idx=0, qkv_ptr=s["qkv"].data_ptr(), q_out_ptr=s["q_out"].data_ptr(),
        block_tables_ptr=s["ids_table"].data_ptr(), seq_lens_ptr=s["total"].data_ptr(),
        query_start_loc_ptr=s["starts"].data_ptr(), block_offsets_f16_ptr=s["offs"].data_ptr(),
        inv_freq_ptr=s["inv_freq"].data_ptr(), batch=s["batch"], total_query_tokens=s["tokens"],
        num_q_heads=s["hq"], max_blocks_per_seq=s["table"].shape[1],
        positions_ptr=0 if p is None else p.data_ptr(), num_axes=0 if p is None else p.shape[0],
        pair_axes=s["pair_axes"], stream_ptr=st)
    out = {"q": s["q_out"], "k": s["k"], "v": s["v"]}
    return out if s["ks"] is None else dict(out, ks=s["ks"], vs=s["vs"])


def run(state):
    if own:
        return _own(state)
    return {"attn": _plain_attn, "append": _plain_append, "lora": _plain_lora}[state["kind"]](state)


# ---- sizes and the definition in 64 bits --------------------------------------------------------------

def work(case):
    if case["kind"] == "lora":
        widths = [int(w) for w in case["widths"].split(",")]
        m, k, n, rank, rows = case["m"], case["k"], sum(widths), case["rank"], len(widths) * case["rank"]
        used = min(case["adapters"], case["requests"])
        return {"bytes": 2 * m * k + 2 * used * (rows * k + n * rank) + 4 * m * n + 4 * m,
                "flops": 2 * m * (rows * k + n * rank)}
    lay = _layout(case)
    eb = {"fp8": 1, "f32": 4}.get(case["dtype"], 2)
    io = 4 if case["dtype"] == "f32" else 2
    token = 2 * case["hkv"] * case["d"] * eb
    if case["kind"] == "attn":
        total, shared = lay["total"].astype(np.int64), lay["shared"].astype(np.int64)
        once = int(shared[lay["starts"][:-1]].sum()) + int((total - shared).sum())
        return {"bytes": once * token + 2 * case["batch"] * case["hq"] * case["d"] * io,
                "flops": 4 * case["hq"] * case["d"] * int(total.sum())}
    t = int(lay["starts"][-1])
    heads = 2 * case["hq"] + 2 * case["hkv"]
    return {"bytes": t * (heads * case["d"] * io + token),
            "flops": 6 * t * (case["hq"] + case["hkv"]) * case["d"]}


def _grid(v, bits, least):
    """v (fp64) to the nearest value of `bits` significant bits, ties to even,
    on the fixed grid of the exponent `least` below it."""
    e = torch.frexp(v.abs())[1].to(torch.float64) - 1.0
    step = torch.exp2(e.clamp_min(float(least)) - (bits - 1))
    return torch.round(v / step) * step


def _exact_attn(s):
    """A sequence at a time: the softmax by log-sum-exp."""
    out = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    bs, group = s["bs"], s["hq"] // s["hkv"]
    for b, n in enumerate(s["total"].tolist()):
        pages = s["table"][b, :-(-n // bs)]
        kv = []
        for x, sc in ((s["k"], s["ks"]), (s["v"], s["vs"])):
            x = x.flatten(0, 1)[pages].double()
            if sc is not None:
                x = x * sc.flatten(0, 1)[pages].double()[:, None, :, None]
            kv.append(x.flatten(0, 1)[:n].transpose(0, 1))                 # [hkv][n][d]
        for h in range(s["hkv"]):
            z = s["q"][b, h * group:(h + 1) * group].double() @ kv[0][h].t() * s["d"] ** -0.5
            out[b, h * group:(h + 1) * group] = torch.exp(z - torch.logsumexp(z, 1, keepdim=True)) @ kv[1][h]
    return {"out": out}


def _exact_pages(pages, scales, table, bs, first, x):
    """Pages of one sequence after rows x [n][hkv][d] from place `first` on, a
    page at a time; pages and scales are changed."""
    n, done = x.shape[0], 0
    while done < n:
        block, slot = divmod(first + done, bs)
        take = min(bs - slot, n - done)
        p, part = int(table[block]), x[done:done + take]
        done += take
        if scales is None:
            pages[p, slot:slot + take] = part
            continue
        old, amax = scales[p].clone(), part.abs().amax((0, 2))
        mine = torch.where(amax > 0, amax / 448, torch.ones_like(amax))
        new = mine if slot == 0 else torch.where(amax > 448 * old, mine, old)
        if slot:
            grown = (new > old)[None, :, None]
            # what is stored is a multiple of an fp32 scale
            pages[p] = torch.where(grown, _grid(pages[p] * (old / new.float().double())[None, :, None], 4, -6),
                                   pages[p])
        pages[p, slot:slot + take] = _grid(part / new.float().double()[None, :, None], 4, -6)
        scales[p] = new


def _exact_append(s):
    t, hq, hkv, dim = s["tokens"], s["hq"], s["hkv"], s["d"]
    k, v = s["k"].flatten(0, 1).double(), s["v"].flatten(0, 1).double()
    ks, vs = (None if s[n] is None else s[n].flatten(0, 1).double() for n in ("ks", "vs"))
    q = torch.empty(t, hq, dim, dtype=torch.float64, device="cuda")
    starts, total = s["starts"].tolist(), s["total"].tolist()
    rows = s["qkv"].view(t, hq + 2 * hkv, dim)
    for b in range(s["batch"]):
        lo, hi = starts[b], starts[b + 1]
        first = total[b] - (hi - lo)
        x = rows[lo:hi].double()
        if s["positions"] is None:
            at = torch.arange(first, total[b], device="cuda", dtype=torch.float64)[:, None]
        else:
            at = torch.stack([s["positions"][a, lo:hi].double() for a in s["pair_axes"]], 1)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           at * s["inv_freq"].double())[:, None]          # [n][1][d/2]
        z = torch.complex(x[:, :hq + hkv, :dim // 2], x[:, :hq + hkv, dim // 2:]) * turn
        y = torch.cat([z.real, z.imag], -1)
        q[lo:hi] = y[:, :hq]
        _exact_pages(k, ks, s["table"][b].tolist(), s["bs"], first, y[:, hq:])
        _exact_pages(v, vs, s["table"][b].tolist(), s["bs"], first, x[:, hq + hkv:])
    out = {"q": q, "k": k.view(s["k"].shape), "v": v.view(s["v"].shape)}
    return out if ks is None else dict(out, ks=ks.view(s["ks"].shape), vs=vs.view(s["vs"].shape))


def _exact_lora(s):
    y = s["base"].double()
    for a in range(s["adapters"]):
        rows = (s["ids"] == a).nonzero().flatten()
        low = s["x"][rows].double() @ s["a"][a].double().t()
        for i, end in enumerate(s["ends"]):
            start = s["ends"][i - 1] if i else 0
            part = low[:, i * s["rank"]:(i + 1) * s["rank"]] @ s["b"][a, start:end].double().t()
            y[rows, start:end] += s["scales"][a].double() * part
    return {"y": y}


def exact(case, seed):
    return {"attn": _exact_attn, "append": _exact_append, "lora": _exact_lora}[case["kind"]](prepare(case, seed))

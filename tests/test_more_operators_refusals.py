"""What the shared-prefix attention, the chunk's rotation and append and the
adapters refuse, on the host-check build: -1 with the reason, before any device
work (a call that passes the checks ends at "no device" there)."""
import ctypes as C

import pytest

from lattice_amd.bindings import (KcmmError, KcmmLora, KcmmRopePositions, KV_BF16, KV_F32, KV_FP8,
                                  make_config)

P = 1 << 20     # an aligned address; nothing is read from it
STEP = 1 << 33  # buffers this far apart overlap nothing


def at(i):
    return P + i * STEP


def pool_of(lib, dtype=KV_BF16, head_dim=64, block_size=16):
    return lib.create_pool(make_config(num_layers=2, kv_heads=2, head_dim=head_dim, max_batch=4,
                                       max_seq_len=512, block_size=block_size), dtype)


SHARED = dict(layer_idx=0, query_ptr=at(0), out_ptr=at(1), block_tables_ptr=at(2), seq_lens_ptr=at(3),
              shared_lens_ptr=at(4), group_starts_ptr=at(5), block_offsets_f16_ptr=at(6),
              scratch_ptr=at(7), scratch_bytes=1 << 40, batch=4, num_groups=2, num_q_heads=8,
              kv_heads=2, head_dim=64, block_size=16, max_blocks_per_seq=8, scale=0.125)


@pytest.mark.parametrize("dtype", [KV_BF16, KV_FP8, KV_F32])
@pytest.mark.parametrize("change,why", [
    ({}, "no device"), (dict(layer_idx=1), "no device"), (dict(num_groups=4), "no device"),
    (dict(num_q_heads=7), "no device"), (dict(scale=-1.0), "no device"),
    *[({n: 0}, "null") for n in SHARED if n.endswith("_ptr")],
    (dict(layer_idx=2), "layer_idx"), (dict(batch=0), "positive"), (dict(num_q_heads=0), "positive"),
    (dict(max_blocks_per_seq=0), "positive"), (dict(num_groups=0), "groups"),
    (dict(num_groups=5), "groups"), (dict(kv_heads=4), "geometry"), (dict(head_dim=128), "geometry"),
    (dict(block_size=8), "geometry"), (dict(num_q_heads=65536), "65535"),
    (dict(max_blocks_per_seq=65536), "65535"), (dict(batch=1 << 30, num_groups=1), "2^31"),
    (dict(scratch_bytes=16), "scratch"), (dict(scratch_ptr=at(7) + 128), "scratch"),
    (dict(query_ptr=at(0) + 8), "aligned"), (dict(out_ptr=at(1) + 2), "aligned"),
])
def test_shared_attention(hostcheck_lib, dtype, change, why):
    with pool_of(hostcheck_lib, dtype) as pool:
        with pytest.raises(KcmmError, match=why.replace("^", r"\^")):
            pool.paged_attn_decode_shared(**{**SHARED, **change})


def test_shared_scratch(hostcheck_lib):
    with pool_of(hostcheck_lib) as pool:
        assert pool.shared_scratch_bytes(4, 8, 8) > 0
        for args in ((0, 8, 8), (4, 0, 8), (4, 8, 0), (4, 65536, 8), (4, 8, 65536), (1 << 30, 8, 8)):
            with pytest.raises(KcmmError, match="positive|65535|2\\^31"):
                pool.shared_scratch_bytes(*args)
        assert hostcheck_lib.lib.kcmm_paged_attn_shared_scratch_bytes(None, 4, 8, 8) == 0


CHUNK = dict(layer_idx=0, qkv_ptr=at(0), q_out_ptr=at(1), block_tables_ptr=at(2), seq_lens_ptr=at(3),
             query_start_loc_ptr=at(4), block_offsets_f16_ptr=at(5), inv_freq_ptr=at(6), batch=4,
             total_query_tokens=20, num_q_heads=8, max_blocks_per_seq=8)


@pytest.mark.parametrize("dtype", [KV_BF16, KV_FP8, KV_F32])
@pytest.mark.parametrize("change,why", [
    ({}, "no device"), (dict(total_query_tokens=0), "no device"),
    (dict(positions_ptr=at(8), num_axes=3, pair_axes=[0] * 8 + [1] * 12 + [2] * 12), "no device"),
    (dict(positions_ptr=at(8) + 4), "no device"),
    *[({n: 0}, "null") for n in CHUNK if n.endswith("_ptr")],
    (dict(layer_idx=2), "layer_idx"), (dict(batch=0), "positive"), (dict(num_q_heads=7), "multiple"),
    (dict(num_q_heads=0), "positive"), (dict(max_blocks_per_seq=0), "positive"),
    (dict(max_blocks_per_seq=65536), "65535"), (dict(num_q_heads=65536), "65535"),
    (dict(total_query_tokens=1 << 31), "too many"),
    (dict(total_query_tokens=(1 << 31) - 1), "too many"),
    (dict(qkv_ptr=at(0) + 8), "aligned"), (dict(q_out_ptr=at(1) + 8), "aligned"),
    (dict(seq_lens_ptr=at(3) + 2), "aligned"), (dict(block_offsets_f16_ptr=at(5) + 4), "aligned"),
    (dict(q_out_ptr=at(0)), "overlaps"), (dict(q_out_ptr=at(0) + 20 * 12 * 64 * 2 - 16), "overlaps"),
    (dict(positions_ptr=at(8), num_axes=0), "axes"), (dict(positions_ptr=at(8), num_axes=5), "axes"),
    (dict(positions_ptr=at(8), num_axes=2, pair_axes=[0] * 31 + [2]), "pair 31 takes axis 2 of 2"),
    (dict(positions_ptr=at(8) + 2), "aligned"),
])
def test_chunk(hostcheck_lib, dtype, change, why):
    with pool_of(hostcheck_lib, dtype) as pool:
        with pytest.raises(KcmmError, match=why):
            pool.rope_append_chunk(**{**CHUNK, **change})


@pytest.mark.parametrize("head_dim", [12, 264])
def test_chunk_head_dim(hostcheck_lib, head_dim):
    with pool_of(hostcheck_lib, KV_F32, head_dim) as pool:
        with pytest.raises(KcmmError, match="head_dim"):
            pool.rope_append_chunk(**CHUNK)


LORA = dict(x_ptr=at(0), a_ptr=at(1), b_ptr=at(2), adapter_ids_ptr=at(3), low_ptr=at(4),
            base_ptr=at(5), y_ptr=at(6), m=4, n=96, k=64, adapters=3, rank=16, slice_ends=[32, 64, 96],
            scales_ptr=at(7))


@pytest.mark.parametrize("change,why", [
    ({}, "no device"), (dict(y_ptr=at(5)), "no device"), (dict(scales_ptr=0), "no device"),
    (dict(slice_ends=None), "no device"), (dict(m=1 << 20, y_ptr=at(5)), "no device"),
    (dict(rank=128), "no device"), (dict(k=8), "no device"),
    (dict(scales_ptr=at(7) + 4, adapter_ids_ptr=at(3) + 4), "no device"),
    *[({n: 0}, "null") for n in LORA if n.endswith("_ptr") and n != "scales_ptr"],
    (dict(m=0), "m <="), (dict(m=(1 << 20) + 1), "m <="), (dict(n=0), "m <="), (dict(n=100), "m <="),
    (dict(n=(1 << 22) + 16), "m <="), (dict(k=0), "m <="), (dict(k=12), "m <="),
    (dict(k=(1 << 20) + 8), "m <="), (dict(rank=0), "rank"), (dict(rank=12), "rank"),
    (dict(rank=136), "rank"), (dict(adapters=0), "adapters"), (dict(adapters=65536), "adapters"),
    (dict(slice_ends=[]), "slices"), (dict(slice_ends=[32, 32, 96]), "ascending"),
    (dict(slice_ends=[8, 96]), "ascending"), (dict(slice_ends=[32, 64]), "end at n"),
    (dict(slice_ends=[0, 96]), "ascending"), (dict(slice_ends=[32, 112]), "end at n"),
    (dict(x_ptr=at(0) + 8), "aligned"), (dict(low_ptr=at(4) + 4), "aligned"),
    (dict(y_ptr=at(6) + 2), "aligned"), (dict(scales_ptr=at(7) + 2), "aligned"),
    (dict(y_ptr=at(0)), "overlaps"), (dict(y_ptr=at(5) + 16), "overlaps"), (dict(y_ptr=at(2)), "overlaps"),
    (dict(low_ptr=at(5)), "overlaps"), (dict(low_ptr=at(0) + 496), "overlaps"),
    (dict(low_ptr=at(6)), "overlaps"), (dict(low_ptr=at(3)), "overlaps"), (dict(y_ptr=at(7)), "overlaps"),
])
def test_lora(hostcheck_lib, capfd, change, why):
    capfd.readouterr()
    with pytest.raises(KcmmError):
        hostcheck_lib.lora_add_bf16(**{**LORA, **change})
    said = capfd.readouterr().err
    assert why in said and said.startswith("kcmm_lora"), said


def test_null_structs(hostcheck_lib, capfd):
    assert hostcheck_lib.lib.kcmm_lora_add_bf16_on_stream(at(0), None, at(1), at(2), at(3), at(4), 1, 16,
                                                          8, 0) == -1
    assert hostcheck_lib.lib.kcmm_rope_append_chunk_on_stream(
        None, 0, *[at(i) for i in range(7)], None, 1, 1, 1, 1, 0) == -1
    assert hostcheck_lib.lib.kcmm_paged_attn_decode_shared_on_stream(
        None, 0, *[at(i) for i in range(9)], 1, 1, 1, 1, 64, 16, 1, C.c_float(1), 0) == -1
    assert C.sizeof(KcmmLora) == 56 and KcmmLora.slice_ends.offset == 36
    assert C.sizeof(KcmmRopePositions) == 144 and KcmmRopePositions.axis_of_pair.offset == 12


def test_shared_attention_of_tables_near_2_to_31(hostcheck_lib):
    """Token numbers are 32 bits, and a kernel's loop steps past the last one."""
    with hostcheck_lib.create_pool(make_config(num_layers=1, kv_heads=1, head_dim=8, max_batch=1,
                                               max_seq_len=42966, block_size=42966), KV_FP8) as pool:
        call = dict(SHARED, batch=1, num_groups=1, num_q_heads=1, kv_heads=1, head_dim=8, block_size=42966)
        for blocks, why in ((49981, "2\\^31"), (49980, "no device"), (1, "no device")):   # 2^31 - 2, and 42966 less
            with pytest.raises(KcmmError, match=why):
                pool.paged_attn_decode_shared(**{**call, "max_blocks_per_seq": blocks})
        with pytest.raises(KcmmError, match="2\\^31"):
            pool.shared_scratch_bytes(1, 1, 49981)
        assert pool.shared_scratch_bytes(1, 1, 49980) > 0


@pytest.mark.parametrize("change,why", [
    (dict(out_ptr=at(0)), "no device"), (dict(out_ptr=at(0) + 2048), "overlaps"),
    (dict(scratch_ptr=at(0)), "overlaps"), (dict(scratch_ptr=at(1)), "overlaps"),
    (dict(out_ptr=at(7) + 2048), "overlaps"), (dict(query_ptr=at(7) - 16), "overlaps"),
    (dict(query_ptr=at(7) - 4096), "no device"), (dict(block_tables_ptr=at(7) - 64), "overlaps"),
    (dict(block_tables_ptr=at(7) - 128), "no device"), (dict(seq_lens_ptr=at(7) + 4), "overlaps"),
    (dict(shared_lens_ptr=at(7) - 12), "overlaps"), (dict(group_starts_ptr=at(7) - 8), "overlaps"),
    (dict(group_starts_ptr=at(7) - 12), "no device"),
])
def test_shared_attention_buffers(hostcheck_lib, change, why):
    with pool_of(hostcheck_lib) as pool:
        with pytest.raises(KcmmError, match=why):
            pool.paged_attn_decode_shared(**{**SHARED, **change})


@pytest.mark.parametrize("axes", [[256] * 32, [0] * 31 + [-256], [0] * 129, [1 << 32]])
def test_axes_that_are_no_bytes(hostcheck_lib, axes):
    """They would wrap round to an axis that is there."""
    with pool_of(hostcheck_lib) as pool:
        with pytest.raises(KcmmError, match="pair_axes"):
            pool.rope_append_chunk(**CHUNK, positions_ptr=at(8), num_axes=2, pair_axes=axes)

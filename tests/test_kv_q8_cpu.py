"""The 8-bit pool and the rotary by position without a GPU: the oracle's own invariants, the frequencies, and every
refusal of the Python and C entry points (checked on the host before any launch)."""
import ctypes as C
import math
import types

import numpy as np
import pytest
import torch

from oracle import kv_q8_oracle as O


@pytest.fixture(scope="module")
def mk():
    import __graft_entry__
    __graft_entry__.build()
    import morphserve_b200
    return morphserve_b200


# ------------------------------------------------------------------------------------------------- number format
@pytest.mark.parametrize("code", ["int8", "e4m3"])
def test_oracle_quantisation_error_is_half_a_step(code):
    rs = np.random.RandomState(0)
    for _ in range(50):
        x = (rs.randn(16, 8) * 10.0 ** rs.uniform(-30, 30)).astype(np.float32).astype(np.float64)
        s = O.scale_of(np.abs(x).max(), code)
        y = O.values(O.encode(x, O.inverse_of(s), code), code) * np.float64(s)
        # int8: half a code, and 127 * 2^-23 codes for the two roundings of the scale.  e4m3: half a step of 2^-3
        # relative, at least half of the smallest code 2^-9
        bound = 0.5001 * s if code == "int8" else np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** -10 * s)
        assert (np.abs(y - x) <= bound).all()


def test_oracle_e4m3_agrees_with_torch():
    x = torch.randn(4096, dtype=torch.float32) * 100
    x = torch.cat([x.clamp(-448, 448), torch.from_numpy(O.E4M3[:127]).float(), torch.linspace(-0.02, 0.02, 999)])
    want = x.to(torch.float8_e4m3fn).view(torch.uint8).numpy()
    assert (O.encode(x.double().numpy(), 1.0, "e4m3") == want).all()
    assert np.array_equal(O.values(want, "e4m3"), x.to(torch.float8_e4m3fn).double().numpy())


def test_oracle_e4m3_scale_is_the_smallest_power_of_two():
    for amax in [448.0, 448.5, 224.0, 1.0, 1.75, 1.7500001, 3e38, 2.0 ** -100, 5e-39]:
        s = float(O.scale_of(amax, "e4m3"))
        if s:
            assert amax <= 448 * s and amax > 448 * s / 2 and math.frexp(s)[0] == 0.5
        else:
            assert amax < 448 * 2.0 ** -126


# --------------------------------------------------------------------------------------------------- frequencies
def cfg(**kw):
    return types.SimpleNamespace(**{"head_dim": 128, "rope_theta": 10000.0, "max_position_embeddings": 4096, **kw})


def test_frequencies_plain_and_linear(mk):
    inv, scale = mk.rotary_inv_freq(cfg(), device="cpu")
    want = 10000.0 ** (-np.arange(0, 128, 2) / 128)
    assert inv.dtype == torch.float64 and np.allclose(inv.numpy(), want, rtol=1e-15) and scale == 1.0
    inv, _ = mk.rotary_inv_freq(cfg(rope_scaling=4, partial_rotary_factor=0.25), device="cpu")
    assert np.allclose(inv.numpy(), 10000.0 ** (-np.arange(0, 32, 2) / 32) / 4, rtol=1e-15)


def test_frequencies_ntk_keep_the_first_and_stretch_the_last(mk):
    inv, _ = mk.rotary_inv_freq(cfg(rope_scaling={"rope_type": "ntk", "factor": 8.0}), device="cpu")
    plain, _ = mk.rotary_inv_freq(cfg(), device="cpu")
    assert inv[0] == plain[0] and abs(float(plain[-1] / inv[-1]) - 8.0) < 1e-12


def test_frequencies_llama3_bands(mk):
    sc = {"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
          "original_max_position_embeddings": 8192}
    inv, scale = mk.rotary_inv_freq(cfg(rope_theta=500000.0, rope_scaling=sc), device="cpu")
    base = 500000.0 ** (-np.arange(0, 128, 2) / 128)
    for f, b in zip(inv.tolist(), base):
        wavelen = 2 * math.pi / b
        if wavelen < 8192 / 4:
            want = b
        elif wavelen > 8192 / 1:
            want = b / 8
        else:
            smooth = (8192 / wavelen - 1) / 3
            want = (1 - smooth) * b / 8 + smooth * b
        assert abs(f / want - 1) < 1e-12
    assert scale == 1.0


def test_frequencies_yarn_ramp(mk):
    sc = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    inv, scale = mk.rotary_inv_freq(cfg(rope_scaling=sc), device="cpu")
    base = 10000.0 ** (-np.arange(0, 128, 2) / 128)
    ratio = inv.numpy() / base
    assert ratio[0] == 1 and abs(ratio[-1] - 0.25) < 1e-15 and (np.diff(ratio) <= 1e-15).all()
    assert abs(scale - (0.1 * math.log(4.0) + 1)) < 1e-15
    assert mk.rotary_inv_freq(cfg(rope_scaling={**sc, "attention_factor": 2.0}), device="cpu")[1] == 2.0


def test_frequencies_refusals(mk):
    for sc in ({"rope_type": "other", "factor": 2.0}, {"rope_type": "linear", "factor": 0.0},
               {"rope_type": "llama3", "factor": 2.0, "low_freq_factor": 4.0, "high_freq_factor": 4.0}):
        with pytest.raises(ValueError):
            mk.rotary_inv_freq(cfg(rope_scaling=sc), device="cpu")
    with pytest.raises(ValueError):
        mk.rotary_inv_freq(cfg(max_position_embeddings=None, rope_scaling={"rope_type": "yarn", "factor": 2.0}), device="cpu")
    with pytest.raises(ValueError):
        mk.rotary_inv_freq(cfg(head_dim=1), device="cpu")


# ------------------------------------------------------------------------------------------------------ refusals
def test_python_entry_points_refuse_cpu_tensors(mk):
    mc, ec = types.SimpleNamespace(num_layers=1, num_q_heads=2, num_kv_heads=2, head_dim=8), types.SimpleNamespace(block_size=4, max_blocks_per_seq=2)
    pool = mk.alloc_kvcache_q8(3, mc, ec, torch.int8, device="cpu")
    z = torch.zeros(1, dtype=torch.int32)
    st = types.SimpleNamespace(num_decoding_seqs=1, num_prefill_seqs=0, num_prefill_tokens=0, decoding_seq_lens=z + 1, seq_ids=z,
                               softmax_scale=1.0, num_blocks_org=3, kv_cache_new_block_size=0, max_decoding_len=1)
    rows, table = torch.zeros(1, 2, 8, dtype=torch.float16), torch.zeros(1, 2, dtype=torch.int32)
    for call in (lambda: mk.store_kvcache_q8(rows, rows, *pool, [], [], [], [], table, mc, ec, st, 0),
                 lambda: mk.paged_attention_q8(rows, *pool, [], [], [], [], table, mc, ec, st, 0, rows),
                 lambda: mk.load_kvcache_q8(rows, rows, *pool, [], [], [], [], table, mc, ec, z, z, z, z, 1, 0),
                 lambda: mk.rotary_embedding_positions(rows, rows, z, torch.zeros(4, dtype=torch.float64))):
        with pytest.raises(RuntimeError, match="no CPU path"):
            call()
    with pytest.raises(RuntimeError, match="unsupported"):
        mk.alloc_kvcache_q8(3, mc, ec, torch.float16, device="cpu")


def _pool_q8(L, **kw):
    p = L.MkvPoolQ8()
    for name, x in {**dict(num_segments=1, code=1, num_layers=2, num_kv_heads=2, block_size=16, head_dim=64, num_blocks_org=4,
                           chunk_blocks=0), **kw}.items():
        setattr(p, name, x)
    for i in range(2):
        p.k_base[i] = p.v_base[i] = p.k_scale[i] = p.v_scale[i] = 4096
    return p


def test_c_entry_points_check_their_arguments_on_the_host(mk):
    from morphserve_b200 import _lib as L
    lib, ok = L.lib, 4096       # an address that is never read: every call below is refused or has nothing to do

    def decode(pool, k=ok, stride=128, dtype=0, batch=1, layer=0, cols=4, rows=4, ids=ok):
        return lib.mkv_store_kv_q8_decode(0, None, k, ok, stride, stride, dtype, pool, ok, cols, rows, ids, ok, batch, layer)

    def prefill(pool, k=ok, stride=128, dtype=0, n=1, max_len=1, layer=0, tokens=1):
        return lib.mkv_store_kv_q8_prefill(0, None, k, ok, stride, stride, dtype, tokens, pool, ok, 4, 4, ok, ok, ok, n, max_len, layer)

    def load(pool, k=ok, stride=128, dtype=0, n=1, max_len=1, layer=0, rows=1):
        return lib.mkv_load_kv_q8(0, None, k, ok, stride, stride, dtype, rows, pool, ok, 4, 4, ok, ok, ok, ok, n, max_len, layer)

    def attn(pool, q=ok, stride=256, dtype=0, batch=1, hq=4, layer=0, ws=ok, nbytes=1 << 30, cols=4):
        return lib.mkv_paged_attention_q8(0, None, q, stride, ok, dtype, pool, ok, cols, 4, ok, ok, batch, hq, layer, 1.0, 16, ws, nbytes)

    for call in (decode, prefill, load, attn):
        assert call(None) == -1
        assert call(_pool_q8(L, code=0)) == -3 and call(_pool_q8(L, code=3)) == -3
        for bad in (dict(num_segments=0), dict(num_segments=66), dict(num_layers=0), dict(num_kv_heads=0), dict(block_size=0),
                    dict(head_dim=0), dict(num_blocks_org=-1), dict(num_segments=2, chunk_blocks=0)):
            assert call(_pool_q8(L, **bad)) == -2, bad
        null = _pool_q8(L)
        null.v_scale[0] = None
        assert call(null) == -1
        odd = _pool_q8(L)
        odd.k_scale[0] = 4098
        assert call(odd) == -8
        assert call(_pool_q8(L), dtype=3) == -3
        assert call(_pool_q8(L), layer=2) == -5 and call(_pool_q8(L), layer=-1) == -5
        assert call(_pool_q8(L), stride=127) == -2
        assert call(_pool_q8(L), None) == -1
    assert decode(_pool_q8(L), batch=-1) == -2 and decode(_pool_q8(L), batch=0) == 0
    assert decode(_pool_q8(L), cols=0) == -2 and decode(_pool_q8(L), rows=-1) == -2 and decode(_pool_q8(L), ids=None) == -1
    assert prefill(_pool_q8(L), n=0) == 0 and prefill(_pool_q8(L), max_len=0) == 0 and prefill(_pool_q8(L), tokens=-1) == -2
    assert load(_pool_q8(L), n=0) == 0 and load(_pool_q8(L), rows=0) == 0 and load(_pool_q8(L), max_len=-1) == -2
    assert attn(_pool_q8(L), batch=0) == 0 and attn(_pool_q8(L), batch=-1) == -2
    assert attn(_pool_q8(L), hq=3) == -2 and attn(_pool_q8(L), hq=0) == -2
    assert attn(_pool_q8(L, head_dim=513), stride=4 * 513) == -2
    assert attn(_pool_q8(L), ws=4097) == -4


def test_rotary_c_entry_point_checks_its_arguments_on_the_host(mk):
    from morphserve_b200 import _lib as L
    strides = (C.c_int64 * 8)(*[128] * 8)

    def call(q=4096, strides=strides, pos=4096, pos_bytes=4, inv=4096, pairs=32, n=1, hq=2, hkv=2, d=64, dtype=0):
        return L.lib.mkv_rotary_positions(0, None, q, 4096, 4096, 4096, strides, pos, pos_bytes, inv, pairs, 0, 1.0, n, hq, hkv, d, dtype)

    assert call(n=0) == 0
    assert call(dtype=3) == -3 and call(pos_bytes=2) == -3
    for bad in (dict(pairs=0), dict(pairs=33), dict(d=1), dict(n=-1), dict(hq=0, hkv=0), dict(hq=-1)):
        assert call(**bad) == -2, bad
    assert call(q=None) == -1 and call(pos=None) == -1 and call(inv=None) == -1 and call(strides=None) == -1


def test_sizes_that_32_bits_do_not_count_are_refused(mk):
    from morphserve_b200 import _lib as L
    wide = _pool_q8(L, block_size=1 << 12, head_dim=1 << 12, num_kv_heads=65)     # 65 * 2^24 elements a page
    assert L.lib.mkv_store_kv_q8_decode(0, None, 4096, 4096, 65 << 12, 65 << 12, 0, wide, 4096, 4, 4, 4096, 4096, 1, 0) == -2
    strides = (C.c_int64 * 8)(*[2] * 8)
    assert L.lib.mkv_rotary_positions(0, None, 4096, 4096, 4096, 4096, strides, 4096, 4, 4096, 1, 0, 1.0, 1, 65535, 1, 2, 0) == -2


def test_rows_that_overlap_are_refused():
    from morphserve_b200.worker.kernels.rotary_pos import _strides
    base = torch.zeros(128)
    for shape, stride in (((4, 3, 8), (8, 8, 1)), ((4, 3, 8), (16, 8, 1)), ((4, 3, 8), (8, 16, 1)), ((2, 2, 8), (15, 8, 1)),
                          ((2, 1, 8), (7, 8, 1)), ((1, 2, 8), (8, 7, 1)), ((2, 2, 8), (16, 8, 2))):
        with pytest.raises(AssertionError):
            _strides(base.as_strided(shape, stride), shape[0], shape[1], shape[2])
    for shape, stride in (((2, 3, 8), (24, 8, 1)), ((2, 3, 8), (8, 16, 1)), ((2, 2, 8), (17, 9, 1)), ((1, 3, 8), (0, 8, 1)),
                          ((2, 1, 8), (8, 0, 1))):
        assert _strides(base.as_strided(shape, stride), shape[0], shape[1], shape[2]) == stride


def test_yarn_variants_are_refused(mk):
    sc = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 4096}
    for more in ({"mscale": 1.0}, {"mscale_all_dim": 0.5}, {"truncate": False}):
        with pytest.raises(ValueError):
            mk.rotary_inv_freq(cfg(rope_scaling={**sc, **more}), device="cpu")
    assert mk.rotary_inv_freq(cfg(rope_scaling={**sc, "truncate": True, "mscale": None}), device="cpu")[1] > 1


# ------------------------------------------------------------------------------------------- the model state's tables
def test_rotary_tables_take_the_scaling_mappings(mk):
    from morphserve_b200.worker.kv_model import make_rotary_tables
    plain = make_rotary_tables(cfg(), "cpu")
    assert all(torch.equal(a, b) for a, b in zip(plain, make_rotary_tables(cfg(rope_scaling={"rope_type": "default"}), "cpu")))
    assert plain[0].shape == (4096 + 128, 64) and plain[0].dtype == torch.float16
    number = make_rotary_tables(cfg(rope_scaling=4.0), "cpu")
    assert number[0].shape[0] == 4 * 4096 + 128
    assert all(torch.equal(a, b) for a, b in zip(number, make_rotary_tables(cfg(rope_scaling={"type": "linear", "factor": 4.0}), "cpu")))
    for sc, rows in (({"rope_type": "ntk", "factor": 2.5}, 10240),
                     ({"rope_type": "llama3", "factor": 8.0, "low_freq_factor": 1.0, "high_freq_factor": 4.0,
                       "original_max_position_embeddings": 512}, 4096),
                     ({"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048}, 8192)):
        inv, att = mk.rotary_inv_freq(cfg(rope_scaling=sc), device="cpu")
        angles = np.outer(np.arange(rows + 128, dtype=np.float64), inv.numpy())
        got = make_rotary_tables(cfg(rope_scaling=sc), "cpu")
        for f, t in zip((np.cos, np.sin), got):
            assert t.shape == angles.shape and t.dtype == torch.float16 and t.is_contiguous()
            # one rounding to fp16; angles up to 10^4 in 64 bits
            assert (np.abs(t.double().numpy() - f(angles) * att) <= 2.0 ** -11 * np.abs(f(angles) * att) + 2.0 ** -25 + 1e-11).all()
    with pytest.raises(ValueError):
        make_rotary_tables(cfg(rope_scaling={"rope_type": "other", "factor": 2.0}), "cpu")

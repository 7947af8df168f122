"""GPU: calls of the 8-bit pool's operators at the far ends of what they accept."""
import types

import numpy as np
import pytest
import torch

from oracle import kv_q8_oracle as O

from .test_gpu_kv_q8 import CODES, DTYPES, HALF, Case, mk  # noqa: F401  (mk: the fixture)
from .test_gpu_kv_q8_precision import check_32

pytestmark = pytest.mark.gpu


def i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("apart", [2 ** 27 - 16, 2 ** 28, 2 ** 31 + 64])     # the last two: more than 32 bits count in a page
def test_rows_further_apart_than_32_bits_count(mk, code, apart):  # noqa: F811
    """Tokens may lie any distance apart, in elements: prompts, appended tokens and rows that are read back."""
    c = Case(code, [3, 2], hkv=2, d=32, seed=40)
    room = torch.empty((2 * apart + 256,), dtype=torch.float16, device="cuda")
    k, v = (room.as_strided((3, 2, 32), (apart, 32, 1), at) for at in (0, 128))
    kn, vn = c.rs.randn(3, 2, 32).astype(np.float16), c.rs.randn(3, 2, 32).astype(np.float16)
    k.copy_(torch.from_numpy(kn)), v.copy_(torch.from_numpy(vn))
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=[3], decode=[], ids=c.ids[:1]), c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, c.ids[:1], [0], [3], c.layer, c.bs)
    c.same()
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(decode=[3, 2]), c.layer)
    O.store_append(c.segs, code, kn, vn, c.table, c.ids, [3, 2], c.layer, c.bs)
    c.same()
    k.zero_(), v.zero_()
    mk.load_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, i32(c.ids[:1]), i32([0]), i32([3]), i32([0]), 3, c.layer)
    for got, want in zip((k, v), O.cached(c.segs, code, c.table, c.ids[0], 3, c.layer, c.bs)):
        assert (np.abs(got.double().cpu().numpy() - want) <= (2.0 ** -11 + 2.0 ** -23) * np.abs(want) + 2.0 ** -25).all()


@pytest.mark.parametrize("bs", [1, 16])
def test_a_length_hint_far_above_the_lengths(mk, bs):  # noqa: F811
    """max_prefill_len and max_len size a launch only: the largest 32-bit number does no more than the lengths themselves."""
    c = Case("int8", [7, 20], hkv=2, d=32, bs=bs, seed=41)
    k, kn = c.rows(27, 2, torch.float16)
    v, vn = c.rows(27, 2, torch.float16)
    st = c.state(prefill=[7, 20], decode=[])
    st.max_prefill_len = 2 ** 31 - 1
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, st, c.layer)
    O.store_prefill(c.segs, "int8", kn, vn, c.table, c.ids, [0, 7], [7, 20], c.layer, bs)
    c.same()
    mk.load_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, i32(c.ids), i32([0, 3]), i32([7, 20]), i32([0, 7]), 2 ** 31 - 1, c.layer)
    want = [np.concatenate([a, b[3:]]) for a, b in zip(*(O.cached(c.segs, "int8", c.table, i, n, c.layer, bs)[:2] for i, n in zip(c.ids, (7, 20))))]
    for got, w in zip((k, v), want):
        assert (np.abs(got[:24].double().cpu().numpy() - w) <= (2.0 ** -11 + 2.0 ** -23) * np.abs(w) + 2.0 ** -25).all()


@pytest.mark.parametrize("scaling", [None, 2.0, {"type": "linear", "factor": 2.0}, {"rope_type": "ntk", "factor": 2.0},
                                     {"rope_type": "llama3", "factor": 8.0, "original_max_position_embeddings": 64},
                                     {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 64}],
                         ids=["none", "number", "linear", "ntk", "llama3", "yarn"])
def test_a_step_with_scaled_frequencies(mk, scaling):  # noqa: F811
    """One model configuration for rotary_inv_freq and the model state's steps: positions and tables say the same."""
    mc = types.SimpleNamespace(num_layers=1, num_q_heads=4, num_kv_heads=2, head_dim=64, max_position_embeddings=256, rope_scaling=scaling)
    ec = types.SimpleNamespace(block_size=16, max_blocks_per_seq=16, max_seqs_in_block_table=6, num_cpu_blocks=2)
    state = mk.KVCacheModelState(mc, ec)
    state.gpu_block_manager = mk.BlockManager("GPU", 40, 6, 16, 16)
    inv, att = mk.rotary_inv_freq(mc)
    st = state.prepare_step([[0] * 100, [0]], [2, 4], [200])
    assert st.positions.tolist() == list(range(100)) + [199]
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k = (torch.randn((101, h, 64), device="cuda", generator=gen, dtype=torch.float16) for h in (4, 2))
    q2, k2 = q.clone(), k.clone()
    mk.rotary_embedding_inplace(q2, k2, st)
    size = (q.float().abs() + q.float().abs().roll(32, -1), k.float().abs() + k.float().abs().roll(32, -1))
    mk.rotary_embedding_positions(q, k, st.positions, inv, attention_scale=att)
    for a, b, s in zip((q, k), (q2, k2), size):
        # tables: fp16 cosines of fp32 angles (2^-11, and 199 * 2^-24 twice); fp16 arithmetic on one side, one rounding on the other
        assert ((a.float() - b.float()).abs() <= att * s * 4 * 2.0 ** -11).all()
    st = state.prepare_step([[0], [0]], [2, 4], [101, 201], rotary_tables=False)
    assert st.position_cos is None and st.position_sin is None and st.positions.tolist() == [100, 200]


def test_a_step_beyond_the_rotary_tables_is_refused_on_the_host(mk):  # noqa: F811
    mc = types.SimpleNamespace(num_layers=1, num_q_heads=4, num_kv_heads=2, head_dim=64, max_position_embeddings=16, rope_scaling=None)
    ec = types.SimpleNamespace(block_size=16, max_blocks_per_seq=16, max_seqs_in_block_table=6, num_cpu_blocks=2)
    state = mk.KVCacheModelState(mc, ec)
    state.gpu_block_manager = mk.BlockManager("GPU", 40, 6, 16, 16)
    free = state.gpu_block_manager.num_free_blocks
    with pytest.raises(RuntimeError, match="rotary tables"):
        state.prepare_step([[0]], [1], [145])
    assert state.gpu_block_manager.num_free_blocks == free
    assert state.prepare_step([[0]], [1], [144]).position_cos.shape == (1, 32)
    assert state.prepare_step([[0]], [1], [200], rotary_tables=False).positions.tolist() == [199]


@pytest.mark.parametrize("code", CODES)
def test_a_length_hint_of_zero(mk, code):  # noqa: F811
    """... stores and loads what the lengths say all the same."""
    c = Case(code, [7, 40], hkv=2, d=32, seed=42)
    k, kn = c.rows(47, 2, torch.float16)
    v, vn = c.rows(47, 2, torch.float16)
    st = c.state(prefill=[7, 40], decode=[])
    st.max_prefill_len = 0
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, st, c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, c.ids, [0, 7], [7, 40], c.layer, c.bs)
    c.same()
    k.zero_(), v.zero_()
    mk.load_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, i32(c.ids[1:]), i32([0]), i32([40]), i32([7]), 0, c.layer)
    for got, want in zip((k, v), O.cached(c.segs, code, c.table, c.ids[1], 40, c.layer, c.bs)):
        assert (np.abs(got[7:].double().cpu().numpy() - want) <= (2.0 ** -11 + 2.0 ** -23) * np.abs(want) + 2.0 ** -25).all()


# ------------------------------------------------------------------------------------------------- wide batches, many heads
def wide_lens(rs, n):
    """Mostly short sequences, a few long ones, runs of empty ones longer than a warp - one of them at the front, one at the
    end, one across a multiple of 384 - and single empty ones."""
    lens = rs.randint(1, 40, n)
    lens[rs.choice(n, 5, replace=False)] = rs.randint(300, 900, 5)
    lens[rs.rand(n) < 0.1] = 0
    lens[:35] = 0
    lens[n - 40:] = 0
    at = 384 if n > 500 else n // 2
    lens[at - 30:at + 37] = 0
    lens[n // 3] = 1200
    return lens.tolist()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("n,hq,hkv", [(385, 1, 1), (385, 8, 1), (700, 8, 2), (700, 2, 2), (1000, 8, 1), (1000, 4, 1), (257, 16, 1), (600, 16, 1),
                                      (600, 40, 2), (1537, 2, 1), (4000, 4, 1)])
def test_attention_over_more_sequences_than_threads(mk, code, n, hq, hkv):  # noqa: F811
    """A block's threads then count several sequences each, and a warp's range starts inside one of their shares."""
    c = Case(code, wide_lens(np.random.RandomState(n + hq), n), hq=hq, hkv=hkv, d=64, seed=n + hq)
    q, qn = c.rows(n, hq, torch.float16)
    st = c.state()
    o = c.attend(mk, q, st)
    # With thousands of rows some have nearly all weight on a token whose value is 0: what is left is below the steps of a
    # sum that held 128 s of that weight, s the block's scale, on the way (int8 codes are held as q + 128).  Such a row is
    # off by 2 * 128 s 2^-23, 7e-7 at s = 0.024, where check_attention's bound, which leaves this out, has 2e-7; check_32's has it.
    check_32(c, o, qn)
    assert torch.equal(c.attend(mk, q, st), o)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("hkv,d,bs", [(9, 128, 16), (16, 32, 16), (17, 64, 16), (33, 40, 8), (40, 128, 32), (130, 32, 4)])
def test_store_and_load_with_many_heads(mk, code, dtype, hkv, d, bs):  # noqa: F811
    """More heads than a thread block has warps: prompts, appends (twice as many pieces) and the way back."""
    t, pre, dec = DTYPES[dtype], [bs + 3, 1, 2 * bs], [7, bs + 1]
    c = Case(code, pre + dec, hkv=hkv, d=d, bs=bs, seed=hkv + d)
    n = sum(pre)
    k, kn = c.rows(n + 2, hkv, t, strided=True)
    v, vn = c.rows(n + 2, hkv, t)
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=pre, decode=dec), c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, c.ids[:3], np.cumsum([0] + pre[:-1]), pre, c.layer, bs)
    O.store_append(c.segs, code, kn[n:], vn[n:], c.table, c.ids[3:], dec, c.layer, bs)
    c.same()
    half, least = HALF[t]
    mk.load_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, i32(c.ids[:3]), i32([0] * 3), i32(pre), i32(np.cumsum([0] + pre[:-1])), 2 * bs, c.layer)
    for i, (start, m) in enumerate(zip(np.cumsum([0] + pre[:-1]), pre)):
        for got, want in zip((k, v), O.cached(c.segs, code, c.table, c.ids[i], m, c.layer, bs)):
            got = got[start:start + m].double().cpu().numpy()
            assert (np.abs(got - want) <= (half + 2.0 ** -23) * np.abs(want) + least).all()

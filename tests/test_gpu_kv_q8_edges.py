"""GPU: calls of the 8-bit pool's operators at the far ends of what they accept."""
import numpy as np
import pytest
import torch

from oracle import kv_q8_oracle as O

from .test_gpu_kv_q8 import CODES, Case, mk  # noqa: F401  (mk: the fixture)

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

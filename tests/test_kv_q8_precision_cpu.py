"""The bound that the attention's precision is judged by notices weights that were rounded to fp16 (planted in the oracle)."""
import numpy as np
import pytest

from oracle import kv_q8_oracle as O

from . import test_gpu_kv_q8_precision as G


@pytest.mark.parametrize("code", G.CODES)
def test_fp16_weights_without_their_remainder_are_outside_the_bound(code, monkeypatch):
    monkeypatch.setattr(G, "Case", lambda *a, **kw: G_CASE(*a, device="cpu", **kw))
    lens, hq, hkv, d, bs = [2, 2, 17, 40], 8, 1, 64, 16
    c, q = G.cancelling(code, lens, hq, hkv, d, bs, seed=1)
    want, slack = O.attention(c.segs, code, q, c.table, c.ids, lens, c.layer, bs, c.scale, weights=32)
    for remainder in (False, True):
        off = 0.0
        for i, n in enumerate(lens):
            k, v, _ = O.cached(c.segs, code, c.table, c.ids[i], n, c.layer, bs)
            for h in range(hq):
                s = k[:, 0] @ q[i, h] * c.scale
                w = np.exp(s - s.max()) * 100
                held = w.astype(np.float16).astype(np.float64)
                if remainder:
                    held += (w - held).astype(np.float16).astype(np.float64)
                got = held @ v[:, 0] / w.sum()
                off = max(off, (np.abs(got - want[i, h]) / (2.0 ** -11 * np.abs(want[i, h]) + slack[i, h])).max())
        assert off < 0.5 if remainder else off > 5


G_CASE = G.Case

"""GPU: how many bits the attention over the 8-bit pool keeps.  Outputs that nearly cancel are small beside the weighted
values they are the sum of, so that the output's own rounding does not hide what the weights lost."""
import numpy as np
import pytest
import torch

from oracle import kv_q8_oracle as O

from .test_gpu_kv_q8 import CODES, DTYPES, HALF, Case, mk  # noqa: F401  (mk: the fixture)

pytestmark = pytest.mark.gpu


def cancelling(code, lens, hq, hkv, d, bs, seed):
    """A case and its queries: head h of a group asks for one element of K alone, and in the dims d = h (mod group) V has two
    tokens, whose codes are chosen so that their weighted sum is close to 0 there; the other tokens' values are 0."""
    c = Case(code, lens, hq=hq, hkv=hkv, d=d, bs=bs, seed=seed)
    group = hq // hkv
    table = O.INT8 if code == "int8" else O.E4M3
    q = np.zeros((len(lens), hq, d))
    for h in range(hq):
        q[:, h, h % group] = 2.0 ** c.rs.randint(1, 4, len(lens))
    big = np.array([x for x in range(256) if np.isfinite(table[x]) and 30 <= abs(table[x]) <= 127])
    for i, n in enumerate(lens):
        k, _, _ = O.cached(c.segs, code, c.table, c.ids[i], n, c.layer, bs)
        at = [O.page(c.segs, c.table, c.ids[i], t // bs) for t in range(n)]
        for t in range(n):
            at[t][0]["v"][at[t][1], c.layer, :, t % bs] = 0
        for hk in range(hkv):
            for e in range(d):
                h = hk * group + e % group
                s = k[:, hk] @ q[i, h] * c.scale
                a, b = 0, n - 1
                w = [np.exp(s[t] - s[b]) * at[t][0]["vs"][at[t][1], c.layer, hk] for t in (a, b)]
                one = c.rs.choice(big, 24)
                want = -table[one] * w[0] / w[1]
                best = np.abs(table[big][None] - want[:, None])
                pick = np.unravel_index(np.argmin(best / np.abs(want)[:, None]), best.shape)
                at[a][0]["v"][at[a][1], c.layer, hk, a % bs, e] = one[pick[0]]
                at[b][0]["v"][at[b][1], c.layer, hk, b % bs, e] = big[pick[1]]
    for g, s in zip(c.gpu, c.segs):
        g["v"].copy_(c._codes(s["v"]))
    return c, q


# groups of 1 ... 20 query heads (units of 4, 8 and 16), both dims of the tensor-core kernel, and shapes of the plain one
SHAPES = [(2, 2, 128, 16), (8, 2, 128, 16), (8, 2, 64, 16), (5, 1, 128, 16), (16, 2, 128, 16), (8, 1, 64, 32), (16, 1, 128, 16),
          (20, 1, 128, 16), (24, 2, 64, 16), (8, 1, 80, 16), (4, 1, 128, 8)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hkv,d,bs", SHAPES)
def test_attention_keeps_its_weights_to_32_bits(mk, code, dtype, hq, hkv, d, bs):  # noqa: F811
    lens = [2, 2, 2, 17, 33, 40]
    c, qn = cancelling(code, lens, hq, hkv, d, bs, seed=hq * 100 + d)
    t = DTYPES[dtype]
    q = torch.from_numpy(qn).to(t).cuda()
    got = c.attend(mk, q, c.state()).double().cpu().numpy().reshape(qn.shape)
    want, slack = O.attention(c.segs, code, qn, c.table, c.ids, lens, c.layer, bs, c.scale, weights=32)
    half, least = HALF[t]
    room = half * np.abs(want) * (1 + 2.0 ** -6) + slack + least
    off = np.abs(got - want)
    assert (off <= room).all(), f"{(off / room).max():.3g} of the room"


def check_32(c, o, qn):
    want, slack = O.attention(c.segs, c.code, qn, c.table, c.ids, c.lens, c.layer, c.bs, c.scale, weights=32)
    half, least = HALF[o.dtype]
    got = o.double().cpu().numpy().reshape(want.shape)
    assert np.array_equal(np.isnan(got), np.isnan(want)), f"NaN in {np.argwhere(np.isnan(got) != np.isnan(want))[:4].tolist()}"
    room = half * np.abs(want) * (1 + 2.0 ** -6) + slack + least
    off = np.abs(got - want)
    assert (off <= room).all(), f"{np.nanmax(off / room):.3g} of the room at {np.argwhere(off > room)[:4].tolist()}"


def scales(c, name, exponents):
    """Scales 2^exponent (int8: up to twice that) in place of the case's, one for each block and head."""
    for g, s in zip(c.gpu, c.segs):
        x = 2.0 ** c.rs.choice(exponents, s[name].shape)
        s[name][:] = (x * c.rs.uniform(1, 2, x.shape) if c.code == "int8" else x).astype(np.float32)
        g[name].copy_(c._dev(s[name]))


# groups of 2, 8 and 16 on the tensor cores in both dims, and the plain kernel
EXTREME = [(4, 2, 128), (4, 2, 64), (8, 1, 128), (16, 1, 128), (16, 1, 64), (4, 2, 80)]
PLAIN = EXTREME[-1:]
EXTREME_LENS = [1, 16, 17, 40, 100, 333, 64]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", PLAIN)
@pytest.mark.parametrize("exponents", [range(-126, -109), range(108, 119), range(-40, 11), range(-126, 119), [-126, 118]],
                         ids=["tiny", "huge", "spread", "all", "both ends"])
def test_attention_takes_every_scale_of_v(mk, code, hq, hkv, d, exponents):  # noqa: F811
    """Scales that a cache of bf16 rows can have, down to the smallest normal number and up to the largest."""
    c = Case(code, EXTREME_LENS, hq=hq, hkv=hkv, d=d, seed=d + hq)
    scales(c, "vs", list(exponents))
    q, qn = c.rows(len(c.lens), hq, torch.bfloat16)
    check_32(c, c.attend(mk, q, c.state()), qn)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", EXTREME)
@pytest.mark.parametrize("exponent", [-126, -100, 100, 106, 118])
def test_attention_takes_every_scale_of_k(mk, code, hq, hkv, d, exponent):  # noqa: F811
    """... with queries that bring the scores back to ordinary sizes, or are 0."""
    c = Case(code, EXTREME_LENS, hq=hq, hkv=hkv, d=d, seed=d + hq + 1)
    scales(c, "ks", [exponent, exponent - 1 if exponent > 0 else exponent + 1])
    q, _ = c.rows(len(c.lens), hq, torch.float32)
    q = (q * 2.0 ** (-exponent // 2) * 2.0 ** (-7 - exponent - (-exponent // 2))).to(torch.bfloat16)
    q[1], q[4, 1], q[5, -1] = 0, 0, 0
    check_32(c, c.attend(mk, q, c.state()), q.double().cpu().numpy())

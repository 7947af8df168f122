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
    empty = np.asarray(c.lens) <= 0
    assert (got[empty] == 7.0).all(), "a row of length 0 was written"
    got, want, slack = got[~empty], want[~empty], slack[~empty]
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
EXTREME_LENS = [1, 16, 17, 40, 100, 333, 64]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", EXTREME)
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


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", EXTREME)
def test_attention_over_all_zero_blocks(mk, code, hq, hkv, d):  # noqa: F811
    """Blocks of zeros have the scale 0: among others, a whole sequence of them, and with what a recycled page holds."""
    c = Case(code, EXTREME_LENS + [50, 48], hq=hq, hkv=hkv, d=d, seed=d + hq + 2)
    for g, s in zip(c.gpu, c.segs):
        for name, codes in (("ks", "k"), ("vs", "v")):
            zero = c.rs.rand(*s[name].shape) < 0.4
            for i in (1, 7, 8):
                for lb in range(-(-c.lens[i] // c.bs)):
                    zero[c.table[c.ids[i], lb]] = name == "vs" or i == 8
            s[name][zero] = 0
            stale = c.rs.rand(*s[name].shape) < 0.3         # (not what store leaves, but 0 times it is 0 as well)
            s[codes][zero & ~stale] = 0
            g[name].copy_(c._dev(s[name])), g[codes].copy_(c._codes(s[codes]))
    q, qn = c.rows(len(c.lens), hq, torch.bfloat16)
    o = c.attend(mk, q, c.state())
    check_32(c, o, qn)
    assert (o[[1, 7, 8]] == 0).all()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", EXTREME)
@pytest.mark.parametrize("nats", [5, 20, 31, 35, 42])
def test_attention_where_the_heaviest_tokens_have_the_smallest_values(mk, code, hq, hkv, d, nats):  # noqa: F811
    """A few blocks hold scores 2 * nats above all others', and values that are next to nothing or 0."""
    c = Case(code, [333, 100, 64, 48, 200, 33], hq=hq, hkv=hkv, d=d, seed=d + hq + nats)
    q = np.zeros((len(c.lens), hq, d))
    q[:, :, 0] = 16
    unit = nats / (127 * 16 * c.scale)
    code_of = (lambda x: np.int8(x).view(np.uint8)) if code == "int8" else (lambda x: O.encode(np.float64(x), 1.0, "e4m3"))
    for s in c.segs:
        s["ks"][:] = np.float32(unit) if code == "int8" else np.float32(2.0 ** np.floor(np.log2(unit)))
        s["k"][..., 0] = code_of(-127)
    for i, n in enumerate(c.lens):
        blocks = -(-n // c.bs)
        for lb, exponent in zip(c.rs.permutation(blocks)[:3], [(-120, -100, -95), (-60,), (None, None, None), (None, -110), (-126, -120), (None,)][i]):
            seg, r = O.page(c.segs, c.table, c.ids[i], lb)
            seg["k"][r, c.layer, ..., 0] = c.rs.choice([code_of(127), code_of(120), code_of(104)], seg["k"][r, c.layer, ..., 0].shape)
            seg["vs"][r, c.layer] = 0 if exponent is None else 2.0 ** exponent
            if exponent is None:
                seg["v"][r, c.layer] = 0
    for g, s in zip(c.gpu, c.segs):
        for name in ("k", "v"):
            g[name].copy_(c._codes(s[name]))
        for name in ("ks", "vs"):
            g[name].copy_(c._dev(s[name]))
    qt = torch.from_numpy(q).to(torch.bfloat16).cuda()
    check_32(c, c.attend(mk, qt, c.state()), q)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,d", EXTREME)
def test_attention_keeps_what_is_not_finite_among_zero_blocks(mk, code, hq, hkv, d):  # noqa: F811
    """A key block that was not finite makes its row NaN although its values are 0: alone, as the first and as the last block."""
    c = Case(code, [16, 40, 40, 40], hq=hq, hkv=hkv, d=d, seed=d + hq + 3)
    s, g = c.segs[0], c.gpu[0]
    for i, lb in ((0, 0), (1, 0), (2, 2)):
        r = c.table[c.ids[i], lb]
        s["ks"][r, c.layer], s["vs"][r, c.layer], s["v"][r, c.layer] = np.nan, 0, 0
    s["vs"][c.table[c.ids[3], :2], c.layer] = 0
    s["v"][c.table[c.ids[3], :2], c.layer] = 0
    for name in ("ks", "vs"):
        g[name].copy_(c._dev(s[name]))
    g["v"].copy_(c._codes(s["v"]))
    q, qn = c.rows(4, hq, torch.bfloat16)
    o = c.attend(mk, q, c.state()).double().cpu().numpy().reshape(4, -1)
    assert np.isnan(o[:3]).all() and not np.isnan(o[3]).any()

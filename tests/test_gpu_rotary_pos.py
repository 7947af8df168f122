"""GPU parity of the rotary embedding by position against the 64-bit oracle."""
from fractions import Fraction

import numpy as np
import pytest
import torch

from oracle import kv_q8_oracle as O

pytestmark = pytest.mark.gpu
HALF = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float32: (2.0 ** -24, 2.0 ** -150)}


@pytest.fixture(scope="module")
def mk():
    import morphserve_b200
    return morphserve_b200


def inv_freq(dim, base=10000.0):
    return base ** (-np.arange(0, dim, 2) / dim)


def check(got, x, positions, inv, interleaved, scale):
    """cos and sin are off by 2^-23 at most (angle: 2^-24 of half a turn, function: 2^-23 together with its rounding),
    times the factor another 2^-24; a product and the fused sum round three times more: 2^-20 of |a| + |b| covers them."""
    want = O.rotary(x, positions, inv, interleaved, scale)
    half, least = HALF[got.dtype]
    n = len(inv)
    size = np.zeros(x.shape)
    a, b = (np.abs(x[..., 0:2 * n:2]), np.abs(x[..., 1:2 * n:2])) if interleaved else (np.abs(x[..., :n]), np.abs(x[..., n:2 * n]))
    if interleaved:
        size[..., 0:2 * n:2] = size[..., 1:2 * n:2] = a + b
    else:
        size[..., :n] = size[..., n:2 * n] = a + b
    g = got.double().cpu().numpy()
    room = half * np.abs(want) * (1 + 2.0 ** -10) + size * abs(scale) * 2.0 ** -20 + least
    assert (np.abs(g - want) <= room).all(), float((np.abs(g - want) / room).max())
    assert np.array_equal(g[..., 2 * n:], x[..., 2 * n:]), "what is behind the rotated part has changed"


def rows(rs, n, heads, d, dtype, layout):
    x = torch.from_numpy(rs.randn(n, heads, d)).to(dtype).cuda()
    if layout == "heads first":
        return x.transpose(0, 1).contiguous().transpose(0, 1)
    if layout == "padded":              # odd distances and an odd first element: single elements only
        wide = torch.zeros((n, heads, d + 3), dtype=dtype, device="cuda")
        wide[..., 1:1 + d] = x
        return wide[..., 1:1 + d]
    return x


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,d,rd,layout", [
    (1, 1, 1, 2, 2, "rows"), (3, 4, 2, 128, 128, "rows"), (65, 32, 8, 128, 64, "rows"), (7, 5, 1, 80, 60, "rows"),
    (33, 3, 3, 64, 16, "heads first"), (9, 2, 1, 96, 96, "padded"), (130, 1, 1, 18, 6, "rows"), (5, 2, 2, 112, 112, "padded"),
    (1000, 2, 1, 256, 256, "rows"), (4, 70, 70, 256, 128, "rows")])
def test_rotary_positions(mk, dtype, interleaved, n, hq, hkv, d, rd, layout):
    rs = np.random.RandomState(n + d)
    q, k = rows(rs, n, hq, d, dtype, layout), rows(rs, n, hkv, d, dtype, layout)
    qn, kn = q.double().cpu().numpy(), k.double().cpu().numpy()
    pos = rs.randint(0, 100000, n)
    inv = inv_freq(rd)
    inv_t = torch.from_numpy(inv).cuda()
    for ints, scale in ((torch.int32, 1.0), (torch.int64, 1.3)):
        p = torch.from_numpy(pos).to(ints).cuda()
        qo, ko = torch.empty((n, hq, d), dtype=dtype, device="cuda"), torch.empty((n, hkv, d), dtype=dtype, device="cuda")
        mk.rotary_embedding_positions(q, k, p, inv_t, interleaved=interleaved, attention_scale=scale, q_out=qo, k_out=ko)
        check(qo, qn, pos, inv, interleaved, scale)
        check(ko, kn, pos, inv, interleaved, scale)
        assert np.array_equal(q.double().cpu().numpy(), qn), "the input has changed"
    mk.rotary_embedding_positions(q, k, p, inv_t, interleaved=interleaved, attention_scale=scale)
    assert torch.equal(q, qo) and torch.equal(k, ko), "in place differs"


def test_far_and_negative_positions(mk):
    """The angle of position 10^9 is as good as that of position 1."""
    rs = np.random.RandomState(1)
    pos = np.array([0, 1, -1, 10 ** 5, 10 ** 6 + 1, -10 ** 6, 10 ** 9, 2 ** 31 - 1, -2 ** 31, 2 ** 40 + 1])
    q = torch.from_numpy(rs.randn(10, 2, 64)).float().cuda()
    k = torch.from_numpy(rs.randn(10, 1, 64)).float().cuda()
    qn, kn = q.double().cpu().numpy(), k.double().cpu().numpy()
    # frequencies with few bits: position * frequency is exact in 64 bits on both sides
    inv = 2.0 ** -np.arange(32.0)
    mk.rotary_embedding_positions(q, k, torch.from_numpy(pos).cuda(), torch.from_numpy(inv).cuda())
    # 2^40 * 2^-53 of the angle's own rounding is left: 2^-13 of a radian for the last one, 2^-22 up to 2^31
    check(q[:9], qn[:9], pos[:9], inv, False, 1.0)
    want = O.rotary(qn[9:], pos[9:], inv, False, 1.0)
    assert np.abs(q[9:].double().cpu().numpy() - want).max() < 2.0 ** -11 * np.abs(qn[9]).max()


def test_empty_and_refusals(mk):
    z = lambda *s, dtype=torch.float16: torch.zeros(s, dtype=dtype, device="cuda")  # noqa: E731
    inv, pos = torch.ones(8, dtype=torch.float64, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    mk.rotary_embedding_positions(z(0, 2, 16), z(0, 1, 16), pos[:0], inv)
    for q, k, p, f in ((z(2, 2, 16), z(2, 1, 16), pos[:1], inv), (z(2, 2, 16), z(3, 1, 16), pos, inv), (z(2, 2, 14), z(2, 1, 14), pos, inv),
                       (z(2, 2, 16), z(2, 1, 18), pos, inv), (z(2, 2, 16), z(2, 1, 16), pos.float(), inv), (z(2, 2, 16), z(2, 1, 16), pos, inv.float()),
                       (z(2, 2, 16), z(2, 1, 16, dtype=torch.bfloat16), pos, inv), (z(2, 1, 16).expand(2, 2, 16), z(2, 1, 16), pos, inv),
                       (z(1, 2, 16).expand(2, 2, 16), z(2, 1, 16), pos, inv), (z(2, 2, 16), z(2, 1, 16), pos.cpu(), inv)):
        with pytest.raises(AssertionError):
            mk.rotary_embedding_positions(q, k, p, f)
    with pytest.raises(RuntimeError):
        mk.rotary_embedding_positions(z(2, 2, 16, dtype=torch.float64), z(2, 1, 16, dtype=torch.float64), pos, inv)


def test_in_a_graph(mk):
    rs = np.random.RandomState(2)
    q, k = rows(rs, 12, 4, 64, torch.float16, "rows"), rows(rs, 12, 2, 64, torch.float16, "rows")
    qn = q.double().cpu().numpy()
    qo, ko = torch.empty_like(q), torch.empty_like(k)
    inv, pos = inv_freq(64), torch.zeros(12, dtype=torch.int32, device="cuda")
    inv_t = torch.from_numpy(inv).cuda()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        mk.rotary_embedding_positions(q, k, pos, inv_t, q_out=qo, k_out=ko)
    for first in (5, 70000):
        pos.copy_(torch.arange(first, first + 12))
        g.replay()
        torch.cuda.synchronize()
        check(qo, qn, np.arange(first, first + 12), inv, False, 1.0)


def test_positions_up_to_what_64_bits_count(mk):
    """Frequencies with all their digits: the angle is the exact product's, however many turns it has."""
    rs = np.random.RandomState(3)
    pos = np.concatenate([rs.randint(2 ** b, 2 ** (b + 1), 6) for b in (20, 31, 36, 40, 44, 48, 52)] + [[2 ** 53, -2 ** 53, 2 ** 53 - 1]])
    inv = np.sort(rs.uniform(0.001, 1, 32))[::-1].copy()
    n = len(pos)
    q, k = (torch.from_numpy(rs.randn(n, h, 64)).float().cuda() for h in (2, 1))
    qn = q.double().cpu().numpy()
    mk.rotary_embedding_positions(q, k, torch.from_numpy(pos).cuda(), torch.from_numpy(inv).cuda())
    # the product as a fraction, its remainder of a turn with 70 digits of pi
    turn = 2 * Fraction("3.1415926535897932384626433832795028841971693993751058209749445923078164")
    angle = np.array([[float(Fraction(int(p)) * Fraction(float(f)) % turn) for f in inv] for p in pos])
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    a, b = qn[..., :32], qn[..., 32:]
    want = np.concatenate([a * c - b * s, a * s + b * c], -1)
    size = np.concatenate([np.abs(a) + np.abs(b)] * 2, -1)
    assert (np.abs(q.double().cpu().numpy() - want) <= (2.0 ** -20 + 2.0 ** -24) * size).all()     # (as in check())


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("n,hq,hkv,d,rd", [(7109, 2, 1, 128, 128), (10657, 3, 2, 32, 16), (14211, 1, 1, 80, 64), (30000, 1, 1, 8, 2)])
def test_several_tokens_a_thread_block(mk, dtype, interleaved, n, hq, hkv, d, rd):
    """Enough tokens for blocks of two and more of them, the last one cut."""
    rs = np.random.RandomState(n)
    qkv = torch.from_numpy(rs.randn(n, hq + hkv, d)).to(dtype).cuda()
    q, k = qkv[:, :hq], qkv[:, hq:]
    qn, kn = q.double().cpu().numpy(), k.double().cpu().numpy()
    pos, inv = rs.randint(0, 100000, n), inv_freq(rd)
    mk.rotary_embedding_positions(q, k, torch.from_numpy(pos).cuda(), torch.from_numpy(inv).cuda(), interleaved=interleaved)
    check(q, qn, pos, inv, interleaved, 1.0)
    check(k, kn, pos, inv, interleaved, 1.0)

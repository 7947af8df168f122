"""GPU parity of the 8-bit pool's operators against the 64-bit oracle: store (codes and scales byte for byte), load (one
rounding), decode attention (bounds derived from the roundings that the kernels make), and a run of them together."""
import types

import numpy as np
import pytest
import torch

from oracle import kv_q8_oracle as O

pytestmark = pytest.mark.gpu

CODE_DTYPE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# half a step of a rounding, relative, and half of the type's smallest step
HALF = {torch.float16: (2.0 ** -11, 2.0 ** -25), torch.bfloat16: (2.0 ** -8, 2.0 ** -134), torch.float32: (2.0 ** -24, 2.0 ** -150)}


class Case:
    """A pool in use with a batch of sequences on it, on the CPU (oracle) and on the GPU."""

    def __init__(self, code, lens, *, hq=4, hkv=2, d=32, bs=16, layers=2, layer=1, chunks=0, chunk_blocks=3, seed=0,
                 tail="codes", device="cuda"):
        self.rs = np.random.RandomState(seed)
        self.code, self.lens, self.hq, self.hkv, self.d, self.bs, self.layer = code, list(lens), hq, hkv, d, bs, layer
        need = [max(0, -(-n // bs)) for n in lens]
        total = sum(need) + 5
        n0 = max(1, total - chunks * chunk_blocks)
        self.segs = []
        for n in [n0] + [chunk_blocks] * chunks:
            shape = (n, layers, hkv, bs, d)
            if code == "int8":
                c = [self.rs.randint(-127, 128, shape).astype(np.int8).view(np.uint8) for _ in range(2)]
                s = [self.rs.uniform(0.005, 0.03, shape[:3]).astype(np.float32) for _ in range(2)]
            else:       # any finite code; NaN codes (0x7f, 0xff) only where nothing may read them
                c = [self.rs.randint(0, 127, shape).astype(np.uint8) + (self.rs.randint(0, 2, shape) * 128).astype(np.uint8) for _ in range(2)]
                s = [(2.0 ** self.rs.randint(-9, -6, shape[:3])).astype(np.float32) for _ in range(2)]
            self.segs.append(dict(k=c[0], v=c[1], ks=s[0], vs=s[1]))
        blocks = n0 + chunks * chunk_blocks
        rows = len(lens) + 2
        self.table = np.full((rows, max(need + [1]) + 1), -1, np.int32)
        ids = self.rs.permutation(blocks)
        self.ids = self.rs.permutation(rows)[:len(lens)].astype(np.int32)
        at = 0
        for i, n in enumerate(need):
            self.table[self.ids[i], :n] = ids[at:at + n]
            at += n
        if tail == "nan" and code == "e4m3":     # slots behind the sequences' ends hold NaN codes
            for i, n in enumerate(lens):
                if n > 0 and n % bs:
                    seg, r = O.page(self.segs, self.table, self.ids[i], n // bs)
                    for c in "kv":
                        seg[c][r, layer, :, n % bs:] = 0x7f
        self.device = device
        self.gpu = [dict(k=self._codes(s["k"]), v=self._codes(s["v"]), ks=self._dev(s["ks"]), vs=self._dev(s["vs"])) for s in self.segs]
        self.mc = types.SimpleNamespace(num_layers=layers, num_q_heads=hq, num_kv_heads=hkv, head_dim=d)
        self.ec = types.SimpleNamespace(block_size=bs, max_blocks_per_seq=self.table.shape[1])
        self.table_t = self._dev(self.table)
        self.scale = d ** -0.5

    def _dev(self, a):
        return torch.from_numpy(np.ascontiguousarray(a).copy()).to(self.device)

    def _codes(self, a):
        return self._dev(a).view(CODE_DTYPE[self.code])

    def pool(self):
        g = self.gpu
        return (g[0]["k"], g[0]["v"], g[0]["ks"], g[0]["vs"], [s["k"] for s in g[1:]], [s["v"] for s in g[1:]],
                [s["ks"] for s in g[1:]], [s["vs"] for s in g[1:]])

    def state(self, prefill=(), decode=None, ids=None, starts=None, max_len=None):
        pre, dec = list(prefill), list(self.lens if decode is None else decode)
        ids = self.ids if ids is None else np.asarray(ids, np.int32)
        starts = np.concatenate([[0], np.cumsum(pre)[:-1]]) if starts is None and pre else starts if pre else []
        i32 = lambda a: self._dev(np.asarray(a, np.int32))  # noqa: E731
        return types.SimpleNamespace(
            seq_ids=i32(ids), softmax_scale=self.scale, num_prefill_seqs=len(pre), num_prefill_tokens=sum(max(0, n) for n in pre),
            prefill_seq_start_locs=i32(starts), prefill_seq_lens=i32(pre), max_prefill_len=max(pre + [0]),
            num_decoding_seqs=len(dec), decoding_seq_lens=i32(dec), max_decoding_len=max_len or max(dec + [0]),
            num_blocks_org=self.segs[0]["k"].shape[0], kv_cache_new_block_size=self.segs[1]["k"].shape[0] if len(self.segs) > 1 else 0)

    def rows(self, n, heads, dtype, size=1.0, strided=False):
        """[n, heads, d] on the GPU and as float64; `strided`: a view of wider rows."""
        x = torch.from_numpy(self.rs.randn(n, heads + (3 if strided else 0), self.d) * np.exp(self.rs.randn(n, 1, 1) * 0.5) * size)
        x = x.to(dtype).to(self.device)
        if strided:
            x = x[:, 2:2 + heads]
        return x, x.double().cpu().numpy()

    def same(self):
        """The GPU's pool equals the oracle's, byte for byte."""
        for i, (g, s) in enumerate(zip(self.gpu, self.segs)):
            for c in ("k", "v"):
                got = g[c].view(torch.uint8).cpu().numpy()
                assert np.array_equal(got, s[c]), f"segment {i} {c}: {np.argwhere(got != s[c])[:4].tolist()}"
            for c in ("ks", "vs"):
                got = g[c].cpu().numpy()
                assert np.array_equal(got, s[c], equal_nan=True), f"segment {i} {c}"

    def attend(self, mk, q, st, o=None):
        o = torch.full((q.shape[0], self.hq * self.d), 7.0, dtype=q.dtype, device=self.device) if o is None else o
        mk.paged_attention_q8(q, *self.pool(), self.table_t, self.mc, self.ec, st, self.layer, o)
        return o

    def check_attention(self, o, qn, lens=None, ids=None, untouched=7.0):
        lens = self.lens if lens is None else lens
        want, slack = O.attention(self.segs, self.code, qn, self.table, self.ids if ids is None else ids, lens, self.layer, self.bs, self.scale)
        half, least = HALF[o.dtype]
        got = o.double().cpu().numpy().reshape(want.shape)
        for i, n in enumerate(lens):
            if n <= 0:
                assert (got[i] == untouched).all(), f"row {i} of length {n} was written"
                continue
            assert np.array_equal(np.isnan(got[i]), np.isnan(want[i])), f"row {i}: NaN"
            fine = ~np.isnan(want[i])
            off = np.abs(got[i] - want[i])[fine]
            room = (half * np.abs(want[i]) * (1 + 2.0 ** -6) + slack[i] + least)[fine]
            assert (off <= room).all(), f"row {i} len {n}: {off.max():.3g}, {(off / room).max():.3g} of the room"


@pytest.fixture(scope="module")
def mk():
    import morphserve_b200
    return morphserve_b200


CODES = ["int8", "e4m3"]


# ---------------------------------------------------------------------------------------------------------- store
# dims: 16-byte vectors (128, 64, 32, 40), single elements (20, 7); odd head counts; block sizes 1 ... 32
STORE = [(2, 128, 16), (1, 64, 16), (3, 40, 8), (5, 20, 16), (1, 7, 1), (2, 256, 32), (8, 128, 16)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hkv,d,bs", STORE)
def test_store_prefill(mk, code, dtype, hkv, d, bs):
    lens = [1, bs, bs + 1, 3 * bs - 1, 2 * bs, 0, 5]
    c = Case(code, lens, hkv=hkv, d=d, bs=bs, seed=hkv * 1000 + d)
    k, kn = c.rows(sum(lens), hkv, DTYPES[dtype], strided=True)
    v, vn = c.rows(sum(lens), hkv, DTYPES[dtype])
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=lens, decode=[]), c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, c.ids, np.cumsum([0] + lens[:-1]), lens, c.layer, bs)
    c.same()


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hkv,d,bs", STORE)
def test_store_append_many_steps(mk, code, dtype, hkv, d, bs):
    """Tokens of growing and shrinking size enter one after the other: fresh blocks, kept scales, raised scales."""
    c = Case(code, [4 * bs + 3] * 5, hkv=hkv, d=d, bs=bs, seed=d)
    first = np.array([1, bs, bs + 1, 2 * bs - 1, 2])
    for step in range(bs + 2):
        lens = (first + step).tolist()
        size = 10.0 ** c.rs.uniform(-3, 3)
        k, kn = c.rows(5, hkv, DTYPES[dtype], size if dtype != "f16" else min(size, 50.0), strided=step % 2 == 0)
        v, vn = c.rows(5, hkv, DTYPES[dtype])
        mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(decode=lens), c.layer)
        O.store_append(c.segs, code, kn, vn, c.table, c.ids, lens, c.layer, bs)
    c.same()


@pytest.mark.parametrize("code", CODES)
def test_store_mixed_batch_over_elastic_chunks(mk, code):
    pre, dec = [33, 1, 16], [17, 40, 0, 5]
    c = Case(code, pre + dec, d=64, chunks=3, seed=5)
    n = sum(pre)
    k, kn = c.rows(n + len(dec), c.hkv, torch.float16)
    v, vn = c.rows(n + len(dec), c.hkv, torch.float16, strided=True)
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=pre, decode=dec), c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, c.ids[:3], np.cumsum([0] + pre[:-1]), pre, c.layer, c.bs)
    O.store_append(c.segs, code, kn[n:], vn[n:], c.table, c.ids[3:], dec, c.layer, c.bs)
    c.same()


@pytest.mark.parametrize("code", CODES)
def test_store_extremes(mk, code):
    """Zeros, the type's largest and smallest values, infinities and NaN: a bad token spoils its own block and head only,
    and only from then on; the first slot of a block starts anew."""
    c = Case(code, [20] * 6, d=32, seed=3)
    lens = [16, 17, 18, 5, 1, 20]
    x = torch.randn(6, c.hkv, c.d)
    x[0, 0], x[1, 1, 3], x[2, 0, 5], x[3, 1, 0] = 0, float("inf"), float("nan"), -float("inf")
    x[4], x[5, 0] = 65504.0, 2.0 ** -24
    for dtype in (torch.float16, torch.float32):
        y = x.to(dtype).clone()
        if dtype == torch.float32:
            y[4, 0], y[4, 1], y[5, 1] = 3.4e38, 1e-44, -1.1754944e-38
        mk.store_kvcache_q8(y.cuda(), y.cuda(), *c.pool(), c.table_t, c.mc, c.ec, c.state(decode=lens), c.layer)
        O.store_append(c.segs, code, y.double().numpy(), y.double().numpy(), c.table, c.ids, lens, c.layer, c.bs)
        c.same()
        z = torch.cat([y, y, y]).cuda()
        mk.store_kvcache_q8(z, z, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=[18], decode=[], ids=c.ids[:1]), c.layer)
        zn = z.double().cpu().numpy()
        O.store_prefill(c.segs, code, zn, zn, c.table, c.ids[:1], [0], [18], c.layer, c.bs)
        c.same()


@pytest.mark.parametrize("code", CODES)
def test_store_skips_what_has_no_page_and_takes_the_last_of_two(mk, code):
    c = Case(code, [16, 32, 7, 20], d=32, seed=8)
    a, b = int(c.ids[0]), int(c.ids[1])
    c.table[c.ids[2], 0] = 10 ** 6                  # outside the pool
    c.table_t.copy_(torch.from_numpy(c.table))
    ids = [a, b, a, 99, -1, int(c.ids[2]), a, int(c.ids[3])]
    lens = [3, 32, 5, 4, 4, 7, 0, 10 ** 6]          # the last one lies behind the table's last column
    k, kn = c.rows(8, c.hkv, torch.float16)
    v, vn = c.rows(8, c.hkv, torch.float16)
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(decode=lens, ids=ids, max_len=32), c.layer)
    O.store_append(c.segs, code, kn, vn, c.table, ids, lens, c.layer, c.bs)
    c.same()
    pre = [16, 20, 3, 4, 7]
    ids = [a, b, a, 99, int(c.ids[2])]
    k, kn = c.rows(sum(pre), c.hkv, torch.float16)
    v, vn = c.rows(sum(pre), c.hkv, torch.float16)
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=pre, decode=[], ids=ids), c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, ids, np.cumsum([0] + pre[:-1]), pre, c.layer, c.bs)
    c.same()


# ----------------------------------------------------------------------------------------------------------- load
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hkv,d,bs", STORE)
def test_load(mk, code, dtype, hkv, d, bs):
    lens = [1, bs, 2 * bs + 1, 40, 7, 9]
    c = Case(code, lens, hkv=hkv, d=d, bs=bs, chunks=1, seed=d + bs)
    begins = [0, 0, bs - 1, 13, 7, -3]
    ends = [1, bs, 2 * bs + 1, 40, 7, 4]
    starts = [50, 0, 60, 70, 3, 180]        # row 180 would be token -3; its token 0 is row 183
    k = torch.full((200, hkv + 2, d), 3.0, dtype=DTYPES[dtype], device="cuda")[:, 1:1 + hkv]
    v = torch.full((200, hkv, d), 3.0, dtype=DTYPES[dtype], device="cuda")
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    for max_len in (40, 1):     # the second sizes the launch too small: still everything
        k.fill_(3.0), v.fill_(3.0)
        mk.load_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, i32(c.ids), i32(begins), i32(ends), i32(starts), max_len, c.layer)
        # what two ranges reach holds either's, element by element (nothing orders them)
        first = [np.full((200, hkv, d), 3.0) for _ in range(2)]
        for i in range(len(lens)):
            b = max(begins[i], 0)
            if ends[i] > b:
                got = O.cached(c.segs, code, c.table, c.ids[i], ends[i], c.layer, bs)
                for w, x in zip(first, got):
                    w[starts[i] + b - begins[i]:starts[i] + ends[i] - begins[i]] = x[b:]
        last = [w.copy() for w in first]
        for i in reversed(range(len(lens))):
            b = max(begins[i], 0)
            if ends[i] > b:
                got = O.cached(c.segs, code, c.table, c.ids[i], ends[i], c.layer, bs)
                for w, x in zip(last, got):
                    w[starts[i] + b - begins[i]:starts[i] + ends[i] - begins[i]] = x[b:]
        half, least = HALF[DTYPES[dtype]]
        for x, *both in zip((k, v), first, last):
            # the product in fp32 (2^-24), then the rounding to the type
            y = x.double().cpu().numpy()
            fits = [(np.abs(y - w) <= (half + 2.0 ** -23) * np.abs(w) + least) for w in both]
            ok = fits[0] | fits[1]
            assert ok.all(), f"rows {np.argwhere(~ok)[:4].tolist()}"


@pytest.mark.parametrize("code", CODES)
def test_load_leaves_alone_what_it_cannot_reach(mk, code):
    c = Case(code, [40, 40], d=32, seed=2)
    c.table[c.ids[0], 1] = -5
    c.table_t.copy_(torch.from_numpy(c.table))
    k = torch.full((50, c.hkv, c.d), 3.0, dtype=torch.float16, device="cuda")
    v = k.clone()
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    # a page that is not there; an id outside the table; rows behind the output; rows in front of it; no range at all
    mk.load_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, i32([c.ids[0], 77, c.ids[1], c.ids[1], c.ids[1]]), i32([0, 0, 0, 0, 9]),
                       i32([40, 5, 40, 6, 9]), i32([0, 0, 45, -2, 0]), 40, c.layer)
    got = k.double().cpu().numpy()
    a = O.cached(c.segs, code, c.table, c.ids[0], 40, c.layer, c.bs)[0]
    b = O.cached(c.segs, code, c.table, c.ids[1], 40, c.layer, c.bs)[0]
    # rows 0-3 are written by the first range (tokens 0-3) and by the fourth (tokens 2-5), in either order
    assert np.allclose(got[4:16], a[4:16], rtol=2.0 ** -10) and (got[16:32] == 3.0).all() and np.allclose(got[32:40], a[16:24], rtol=2.0 ** -10)
    assert (got[40:45] == 3.0).all() and np.allclose(got[45:], b[:5], rtol=2.0 ** -10)
    for r in range(4):
        assert np.allclose(got[r], a[r], rtol=2.0 ** -10) or np.allclose(got[r], b[r + 2], rtol=2.0 ** -10)


# ------------------------------------------------------------------------------------------------------ attention
ATTN_LENS = [1, 2, 15, 16, 17, 0, 33, 100, 300, 64, 5, 31]
# (q heads, kv heads, dim, block size): groups of 1 ... 40, both fast dims, block sizes with several tiles a page, and
# shapes that only the plain kernel has
ATTN = [(4, 4, 128, 16), (8, 2, 128, 16), (10, 2, 128, 16), (8, 1, 128, 16), (9, 1, 128, 16), (32, 2, 128, 16), (20, 1, 128, 16),
        (40, 1, 128, 16), (4, 1, 64, 16), (16, 2, 64, 16), (24, 2, 64, 32), (6, 2, 128, 32), (3, 3, 64, 64), (4, 2, 80, 16),
        (2, 1, 7, 1), (4, 2, 128, 8), (4, 2, 128, 48), (2, 2, 256, 16), (5, 1, 32, 16)]


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("hq,hkv,d,bs", ATTN)
def test_attention(mk, code, dtype, hq, hkv, d, bs):
    c = Case(code, ATTN_LENS, hq=hq, hkv=hkv, d=d, bs=bs, seed=hq * 7 + d, tail="nan")
    q, qn = c.rows(len(c.lens), hq, DTYPES[dtype], strided=hq % 2 == 0)
    c.check_attention(c.attend(mk, q, c.state()), qn)
    from morphserve_b200.worker.kernels._common import read_attn_error_flags
    assert read_attn_error_flags(0) == 0


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("hq,hkv,lens", [(4, 1, [5000]), (8, 2, [3000, 1]), (1, 1, [4097]), (16, 1, [2500, 2600]), (32, 8, [1] * 40),
                                         (8, 8, list(range(1, 200, 3))), (24, 3, [16] * 300)])
def test_attention_splits_and_merges(mk, code, hq, hkv, lens):
    c = Case(code, lens, hq=hq, hkv=hkv, d=128, seed=len(lens), chunks=2)
    q, qn = c.rows(len(lens), hq, torch.float16)
    st = c.state()
    o = c.attend(mk, q, st)
    c.check_attention(o, qn)
    for _ in range(3):      # whatever warp or block comes first: the same bits
        assert torch.equal(c.attend(mk, q, st), o)


@pytest.mark.parametrize("code", CODES)
def test_attention_long_context(mk, code):
    """One long sequence among short ones; the oracle on its last queries' heads only would not see a wrong page, so all."""
    c = Case(code, [20000, 3, 700], hq=2, hkv=1, d=64, layers=1, layer=0, seed=4)
    q, qn = c.rows(3, 2, torch.bfloat16)
    c.check_attention(c.attend(mk, q, c.state()), qn)


@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("d", [128, 80])
def test_attention_scores_far_apart(mk, code, d):
    """Scores that rise, fall and overflow the exponential's range: the running maximum has to follow."""
    c = Case(code, [400, 90, 33], hq=4, hkv=2, d=d, seed=9)
    q, qn = c.rows(3, 4, torch.float16, size=30.0)
    c.check_attention(c.attend(mk, q, c.state()), qn)


@pytest.mark.parametrize("d", [128, 80])
def test_attention_not_finite(mk, d):
    """A block whose scale is NaN makes its own sequence and head NaN; an infinite query element does so for its row."""
    c = Case("int8", [40, 40, 40], hq=4, hkv=2, d=d, seed=10)
    seg, r = O.page(c.segs, c.table, c.ids[1], 1)
    seg["ks"][r, c.layer, 1] = np.nan
    c.gpu[0]["ks"].copy_(torch.from_numpy(c.segs[0]["ks"]))
    q, qn = c.rows(3, 4, torch.float16)
    o = c.attend(mk, q, c.state()).double().cpu().numpy().reshape(3, 4, d)
    assert np.isnan(o[1, 2:]).all() and not np.isnan(o[1, :2]).any() and not np.isnan(o[[0, 2]]).any()
    q[2, 0, 5] = float("inf")
    o = c.attend(mk, q, c.state()).double().cpu().numpy().reshape(3, 4, d)
    assert np.isnan(o[2, 0]).all() and not np.isnan(o[2, 1:]).any()


@pytest.mark.parametrize("d", [128, 80])
def test_attention_leaves_out_pages_that_are_not_there(mk, d):
    from morphserve_b200.worker.kernels._common import _workspaces_q8, read_attn_error_flags
    c = Case("e4m3", [100, 40, 16, 50, 64], hq=4, hkv=2, d=d, seed=11)
    c.table[c.ids[0], 2] = 10 ** 7
    c.table[c.ids[1], 0] = -1
    c.table[c.ids[2], 0] = -1           # nothing is left of this one
    c.table_t.copy_(torch.from_numpy(c.table))
    ids, lens = c.ids.copy(), list(c.lens)
    ids[3] = 1000                       # not a row of the table
    lens[4] = 16 * (c.table.shape[1] + 3)     # longer than its row
    q, qn = c.rows(5, 4, torch.float16)
    o = c.attend(mk, q, c.state(decode=lens, ids=ids))
    c.check_attention(o, qn, lens=lens, ids=ids)
    assert torch.isnan(o[2]).all() and torch.isnan(o[3]).all()
    assert read_attn_error_flags(0) & 1
    for ws, _ in _workspaces_q8.values():
        ws[:4].zero_()


def test_attention_rows_behind_the_batch_and_zero_lengths_stay(mk):
    c = Case("int8", [0, -4, 20, 0], hq=8, hkv=2, d=128, seed=12)
    q, qn = c.rows(6, 8, torch.float16)
    o = torch.full((6, 8 * 128), 7.0, dtype=torch.float16, device="cuda")
    c.attend(mk, q, c.state(), o)
    c.check_attention(o[:4], qn[:4])
    assert (o[4:] == 7.0).all()
    c.attend(mk, q[:1], c.state(decode=[0], ids=c.ids[:1]), o)
    assert (o[:2] == 7.0).all()


def test_attention_in_graphs_follows_lengths_and_shares_no_scratch(mk):
    """Two captured launches, replayed at once on two streams while an ordinary one runs on a third; then the lengths
    grow far beyond those of the capture."""
    c = Case("int8", [900, 2000, 40, 1, 700], hq=8, hkv=2, d=128, seed=13)
    small = [3, 5, 1, 1, 2]
    jobs = []
    side = [torch.cuda.Stream() for _ in range(2)]
    for s in side:
        q, qn = c.rows(5, 8, torch.float16)
        st = c.state(decode=small)
        o = torch.zeros((5, 8 * 128), dtype=torch.float16, device="cuda")
        c.attend(mk, q, st, o)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.attend(mk, q, st, o)
        jobs.append((g, s, q, qn, st, o))
    q, qn = c.rows(5, 8, torch.float16)
    st = c.state()
    for lens in (small, c.lens, [1, 1, 0, 1, 1], c.lens):
        for g, s, _, _, s_t, o in jobs:
            s_t.decoding_seq_lens.copy_(torch.tensor(lens, dtype=torch.int32))
            o.fill_(7.0)
        torch.cuda.synchronize()
        for _ in range(5):
            for g, s, *_ in jobs:
                with torch.cuda.stream(s):
                    g.replay()
            o0 = c.attend(mk, q, st)
        torch.cuda.synchronize()
        for _, _, _, n, _, o in jobs:
            c.check_attention(o, n, lens=lens)
        c.check_attention(o0, qn)


def test_attention_on_two_streams_at_once(mk):
    c = Case("e4m3", [1500, 30, 800], hq=4, hkv=1, d=128, seed=14)
    streams = [torch.cuda.Stream() for _ in range(3)]
    jobs = [(s, *c.rows(3, 4, torch.float16), torch.zeros((3, 512), dtype=torch.float16, device="cuda")) for s in streams]
    st = c.state()
    torch.cuda.synchronize()
    for _ in range(20):
        for s, q, _, o in jobs:
            with torch.cuda.stream(s):
                c.attend(mk, q, st, o)
    torch.cuda.synchronize()
    for _, _, qn, o in jobs:
        c.check_attention(o, qn)


def test_offsets_beyond_32_bits(mk):
    """Pages at the far end of a pool of more than 4 GiB of codes for K."""
    c = Case("int8", [40, 17], hq=8, hkv=8, d=128, layers=2, layer=1, seed=15)
    blocks = (1 << 32) // (2 * 8 * 16 * 128) + 64
    small = c.gpu[0]
    shape = (blocks,) + tuple(small["k"].shape[1:])
    n = small["k"].shape[0]
    big = dict(k=torch.empty(shape, dtype=torch.int8, device="cuda"), v=torch.empty(shape, dtype=torch.int8, device="cuda"),
               ks=torch.empty(shape[:3], device="cuda"), vs=torch.empty(shape[:3], device="cuda"))
    for name, x in big.items():
        x[blocks - n:] = small[name]
    c.gpu = [big]
    c.table_t = torch.where(c.table_t >= 0, c.table_t + blocks - n, c.table_t)
    k, kn = c.rows(2, 8, torch.float16)
    st = c.state()
    st.num_blocks_org = blocks
    mk.store_kvcache_q8(k, k, *c.pool(), c.table_t, c.mc, c.ec, st, c.layer)
    O.store_append(c.segs, "int8", kn, kn, c.table, c.ids, c.lens, c.layer, c.bs)
    q, qn = c.rows(2, 8, torch.float16)
    c.check_attention(c.attend(mk, q, st), qn)
    for name in big:
        got = big[name][blocks - n:].view(torch.uint8 if name in "kv" else torch.float32).cpu().numpy()
        assert np.array_equal(got, c.segs[0][name])


# ------------------------------------------------------------------------------------------------- all of them
@pytest.mark.parametrize("code", CODES)
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_prefill_and_decode_steps_together(mk, code, dtype):
    """rotary -> store -> attention for a prompt batch and twenty steps, then the cache read back."""
    t = DTYPES[dtype]
    prompts = [31, 1, 16]
    c = Case(code, [n + 20 for n in prompts], hq=8, hkv=2, d=64, chunks=1, seed=21)
    inv, att = mk.rotary_inv_freq(types.SimpleNamespace(head_dim=64, rope_scaling={"rope_type": "yarn", "factor": 2.0},
                                                        max_position_embeddings=64))
    def step(n, positions):
        qkv, _ = c.rows(n, c.hq + 2 * c.hkv, t)
        q, k, v = qkv[:, :c.hq], qkv[:, c.hq:c.hq + c.hkv], qkv[:, c.hq + c.hkv:]
        want = O.rotary(k.double().cpu().numpy(), positions, inv.cpu().numpy(), True, att)
        mk.rotary_embedding_positions(q, k, torch.tensor(positions, device="cuda"), inv, interleaved=True, attention_scale=att)
        got = k.double().cpu().numpy()
        assert (np.abs(got - want) <= HALF[t][0] * np.abs(want) + 2.0 ** -19 * np.abs(want).max()).all()
        return q, k, v, got, v.double().cpu().numpy()       # the kernels' own rotated rows go on: the pool is exact in them

    q, k, v, kn, vn = step(sum(prompts), [i for n in prompts for i in range(n)])
    mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, c.state(prefill=prompts, decode=[]), c.layer)
    O.store_prefill(c.segs, code, kn, vn, c.table, c.ids, np.cumsum([0] + prompts[:-1]), prompts, c.layer, c.bs)
    for i in range(20):
        lens = [n + i + 1 for n in prompts]
        q, k, v, kn, vn = step(3, [n - 1 for n in lens])
        st = c.state(decode=lens)
        mk.store_kvcache_q8(k, v, *c.pool(), c.table_t, c.mc, c.ec, st, c.layer)
        O.store_append(c.segs, code, kn, vn, c.table, c.ids, lens, c.layer, c.bs)
        o = c.attend(mk, q, st)
        if i % 6 == 0 or i == 19:
            c.check_attention(o, q.double().cpu().numpy(), lens=lens)
    c.same()


def test_python_refusals_on_the_gpu(mk):
    c = Case("int8", [5, 6], d=32, seed=1)
    k, _ = c.rows(2, c.hkv, torch.float16)
    q, _ = c.rows(2, c.hq, torch.float16)
    pool, st = c.pool(), c.state()
    store = lambda k=k, pool=pool, table=c.table_t, st=st: mk.store_kvcache_q8(k, k, *pool, table, c.mc, c.ec, st, c.layer)  # noqa: E731
    store()
    for bad in (dict(k=k.transpose(1, 2).contiguous().transpose(1, 2)), dict(k=k[:1]), dict(k=k.cpu()), dict(table=c.table_t.long()),
                dict(table=c.table_t[:, ::2]), dict(pool=pool[:2] + (pool[2].half(),) + pool[3:]),
                dict(pool=pool[:3] + (pool[3][:1],) + pool[4:]), dict(pool=pool[:4] + ([pool[0]],) + pool[5:])):
        with pytest.raises(AssertionError):
            store(**bad)
    with pytest.raises(RuntimeError):
        store(k=k.double())
    with pytest.raises(RuntimeError):
        store(pool=(pool[0].half(), pool[1].half()) + pool[2:])
    with pytest.raises(AssertionError):
        c.attend(mk, q, st, torch.zeros((2, c.hq * c.d), dtype=torch.bfloat16, device="cuda"))
    with pytest.raises(AssertionError):
        c.attend(mk, q[:1], st)
    with pytest.raises(RuntimeError):
        mk.paged_attention_q8(q, *pool, c.table_t, c.mc, c.ec, st, 2, torch.zeros((2, c.hq * c.d), dtype=torch.float16, device="cuda"))


def test_steps_of_the_model_state_on_an_8_bit_pool(mk):
    """The framework's own step - block manager, lengths and positions from prepare_step - over an 8-bit pool, with a chunk
    added to it half way."""
    mc = types.SimpleNamespace(num_layers=2, num_q_heads=8, num_kv_heads=2, head_dim=64, max_position_embeddings=256)
    ec = types.SimpleNamespace(block_size=16, max_blocks_per_seq=8, max_seqs_in_block_table=6, num_cpu_blocks=2)
    state = mk.KVCacheModelState(mc, ec)
    state.gpu_block_manager = mk.BlockManager("GPU", 12, 6, 8, 16)
    pool = [mk.alloc_kvcache_q8(12, mc, ec, torch.int8)]
    c = Case("int8", [1], hq=8, hkv=2, d=64, layers=2, layer=1, seed=30)
    as_numpy = lambda p: dict(k=p[0].view(torch.uint8).cpu().numpy(), v=p[1].view(torch.uint8).cpu().numpy(),  # noqa: E731
                              ks=p[2].cpu().numpy(), vs=p[3].cpu().numpy())
    c.segs = [as_numpy(pool[0])]
    inv, att = mk.rotary_inv_freq(mc)
    lens = {3: 17, 0: 5}
    for i in range(30):
        order = list(lens)
        if i == 0:
            st = state.prepare_step([[0] * n for n in lens.values()], order, [])
        else:
            for s in lens:
                lens[s] += 1
            st = state.prepare_step([[0]] * len(lens), order, list(lens.values()))
        if i == 20:     # the pool grows, as an elastic expansion does it
            pool.append(mk.alloc_kvcache_q8(4, mc, ec, torch.int8))
            c.segs.append(as_numpy(pool[1]))
        st.kv_cache_new_block_size = 4
        n = st.num_tokens
        want = [p for s in order for p in range(lens[s])] if i == 0 else [lens[s] - 1 for s in order]
        assert st.positions.tolist() == want
        qkv, _ = c.rows(n, 12, torch.float16)
        q, k, v = qkv[:, :8], qkv[:, 8:10], qkv[:, 10:]
        mk.rotary_embedding_positions(q, k, st.positions, inv, attention_scale=att)
        table = state.gpu_block_manager.block_table
        args = (*pool[0], [p[0] for p in pool[1:]], [p[1] for p in pool[1:]], [p[2] for p in pool[1:]], [p[3] for p in pool[1:]],
                table, mc, ec, st, 1)
        mk.store_kvcache_q8(k, v, *args)
        kn, vn, c.table = k.double().cpu().numpy(), v.double().cpu().numpy(), table.cpu().numpy()
        if i == 0:
            O.store_prefill(c.segs, "int8", kn, vn, c.table, order, [0, 17], [17, 5], 1, 16)
        else:
            O.store_append(c.segs, "int8", kn, vn, c.table, order, list(lens.values()), 1, 16)
            o = torch.zeros((2, 512), dtype=torch.float16, device="cuda")
            mk.paged_attention_q8(q, *args, o)
            c.check_attention(o, q.double().cpu().numpy(), lens=list(lens.values()), ids=order)
    for p, s in zip(pool, c.segs):
        assert np.array_equal(p[0].view(torch.uint8).cpu().numpy(), s["k"]) and np.array_equal(p[3].cpu().numpy(), s["vs"])


def test_block_swap_of_an_8_bit_pool_as_views(mk):
    """Codes as an fp16 pool of half the head dim, scales as an fp32 pool: out to the host and back, byte for byte."""
    from morphserve_b200 import swiftllm_c
    mc = types.SimpleNamespace(num_layers=2, num_kv_heads=4, head_dim=64)
    pool = mk.alloc_kvcache_q8(10, mc, types.SimpleNamespace(block_size=16), torch.float8_e4m3fn)
    for t in pool:
        t.view(torch.uint8).random_(0, 256)
    codes = [t.view(torch.float16) for t in pool[:2]]
    scales = [t.view(10, 2, 4, 1, 1) for t in pool[2:]]
    before = [t.view(torch.uint8).clone() for t in pool]
    out = torch.tensor([7, 2, 9], dtype=torch.int64, device="cuda")
    host = torch.tensor([0, 3, 1], dtype=torch.int64, device="cuda")
    back = torch.tensor([1, 4, 0], dtype=torch.int64, device="cuda")
    for pair in (codes, scales):
        swap = [torch.zeros((4,) + tuple(t.shape[1:]), dtype=t.dtype).pin_memory() for t in pair]
        swiftllm_c.swap_blocks(out, host, False, *pair, *swap)
        torch.cuda.synchronize()
        swiftllm_c.swap_blocks(host, back, True, *pair, *swap)
    torch.cuda.synchronize()
    for t, was in zip(pool, before):
        now = t.view(torch.uint8)
        assert torch.equal(now[back], was[out]) and torch.equal(now[[2, 3, 5, 6, 7, 8, 9]], was[[2, 3, 5, 6, 7, 8, 9]])

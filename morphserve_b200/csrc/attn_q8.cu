// Decode attention over the 8-bit pool.
//
// HBM bound: every code is read once for the query heads that share its kv head; what a token costs beyond its bytes is
// the conversion of its codes to fp16, which is why the tensor-core tile is laid out for as few instructions as it is.
//
// One launch.  The launch's tiles (16 tokens of one kv head: 16 x D codes of K and of V) stand in one order - sequence by
// sequence, kv head by kv head, tile by tile, with a few phantom tiles in front of every (sequence, head) for what
// starting one costs - and are dealt out in equal ranges: to thread blocks, and inside a block to its warps.  Every block
// finds its range itself from a prefix sum over the lengths, so there is no plan to keep from one call to the next and
// a captured launch follows the lengths as they are when it runs.
//
// A warp streams its range through a private ring in shared memory (16-byte cp.async, XOR swizzle) and computes
//   S^T = K Q^T     tokens are the 16 rows, up to 8 query heads the 8 columns of mma.m16n8k16
//   O^T = V^T P^T   dims are the rows, heads the columns: half the instructions and accumulators that heads as rows
//                   would take
// Codes go from shared memory to A fragments with plain 16-byte loads: the order of dims inside the k axis of the first
// product and of rows in the second is free, so each thread takes whole 16-byte pieces.
// Pieces of a (sequence, head) that is cut meet in their thread block through shared memory, across blocks through fp32
// rows in the workspace, merged by the block that arrives last.  Nothing waits for another block.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kv_q8.cuh"

namespace mkv {

constexpr float kLog2e = 1.4426950408889634f;

// ------------------------------------------------------------------ plain kernel
// One warp per (sequence, query head); lane l holds dims l, l + 32, ...  fp32 throughout.
constexpr int kPlainDims = 16;  // head_dim <= 512

template <typename T, int CODE>
__global__ void attn_q8_plain_kernel(const T *__restrict__ q, int64_t q_stride, T *__restrict__ o,
                                     const __grid_constant__ PoolViewQ8 pool, const int32_t *__restrict__ block_table,
                                     int64_t table_stride, int num_rows, const int32_t *__restrict__ seq_ids,
                                     const int32_t *__restrict__ seq_lens, int batch, int num_q_heads, int cur_layer,
                                     float scale_log2, int *error_flags) {
    const int lane = threadIdx.x & 31;
    const int64_t wid = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (wid >= (int64_t)batch * num_q_heads) return;
    const int b = (int)(wid / num_q_heads), hq = (int)(wid - (int64_t)b * num_q_heads);
    const int h = hq / (num_q_heads / pool.num_kv_heads);
    const int D = pool.head_dim, bs = pool.block_size;
    const int len = seq_lens[b], row = seq_ids[b];
    if (len <= 0) return;
    float qr[kPlainDims], acc[kPlainDims];
#pragma unroll
    for (int i = 0; i < kPlainDims; ++i) {
        const int d = lane + 32 * i;
        qr[i] = d < D ? value_of<T>(q[b * q_stride + (int64_t)hq * D + d]) : 0.f;
        acc[i] = 0.f;
    }
    float m = -INFINITY, l = 0.f;
    bool bad = row < 0 || row >= num_rows;
    const int nblk = bad ? 0 : (int)min(((int64_t)len + bs - 1) / bs, table_stride);
    bad |= (int64_t)nblk * bs < len;
    for (int jb = 0; jb < nblk; ++jb) {
        const int64_t blk = __ldg(block_table + (int64_t)row * table_stride + jb);
        if (blk < 0 || blk >= pool.total_blocks) {
            bad = true;
            continue;
        }
        int seg;
        int64_t brow;
        locate_block(pool, blk, seg, brow);
        const int64_t tile = tile_index(pool, brow, cur_layer, h);
        const uint8_t *kt = pool.k_base[seg] + tile * pool.tile_bytes, *vt = pool.v_base[seg] + tile * pool.tile_bytes;
        const float ks = pool.k_scale[seg][tile] * scale_log2, vs = pool.v_scale[seg][tile];
        const int ntok = (int)min((int64_t)bs, len - (int64_t)jb * bs);
        for (int tk = 0; tk < ntok; ++tk) {
            float dot = 0.f;
#pragma unroll
            for (int i = 0; i < kPlainDims; ++i) {
                const int d = lane + 32 * i;
                if (d < D) dot += qr[i] * decode1<CODE>(kt[(int64_t)tk * D + d]);
            }
#pragma unroll
            for (int s = 16; s > 0; s >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, s);
            const float sc = dot * ks;
            const float mn = fmaxf(m, sc), base = mn == -INFINITY ? 0.f : mn;  // no finite score yet: all weights are 0
            const float a = exp2f(m - base), w = exp2f(sc - base);
            l = l * a + w;
#pragma unroll
            for (int i = 0; i < kPlainDims; ++i) {
                const int d = lane + 32 * i;
                if (d < D) acc[i] = acc[i] * a + w * (decode1<CODE>(vt[(int64_t)tk * D + d]) * vs);
            }
            m = mn;
        }
    }
    if (bad && lane == 0 && error_flags) atomicOr(error_flags, 1);
#pragma unroll
    for (int i = 0; i < kPlainDims; ++i) {
        const int d = lane + 32 * i;
        if (d < D) o[((int64_t)b * num_q_heads + hq) * D + d] = rounded<T>(acc[i] / l);
    }
}

// ------------------------------------------------------------------ fast kernel
constexpr int kTileTokens = 16;
constexpr int kUnitCost = 2;      // phantom tiles in front of a (sequence, head)
constexpr int kMinTiles = 8;      // ... least number of tiles a thread block is started for
constexpr float kBoost = 6.f;     // weights are held as 2^(score - max + 6): fp16 then reaches 2^-20 of the largest in full
constexpr float kLag = 4.f;       // the running maximum follows only when a score is above it by 2^4
constexpr float kScaleRange = 16.f;  // block scales within this factor of the piece's first go into the weights

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp4(uint32_t dst, const void *src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t addr) {
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds8(uint32_t addr) {
    uint2 v;
    asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];\n" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void mma(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }

// Four codes (one word) as two half2, exact.  int8: the byte with its sign bit flipped is q + 128; set behind the byte 0x64 it
// is the fp16 number 1024 + 128 + q.
template <int CODE>
__device__ __forceinline__ void widen(uint32_t w, uint32_t &lo, uint32_t &hi) {
    if (CODE == MKV_Q8_INT8) {
        const uint32_t x = w ^ 0x80808080u;
        const __half2 off = __float2half2_rn(-1152.f);
        lo = half2_bits(__hadd2(bits_half2(__byte_perm(x, 0x64646464u, 0x4140)), off));
        hi = half2_bits(__hadd2(bits_half2(__byte_perm(x, 0x64646464u, 0x4342)), off));
    } else {
        lo = e4m3x2_to_half2(w & 0xffffu);
        hi = e4m3x2_to_half2(w >> 16);
    }
}

template <typename T>
__device__ __forceinline__ void store4(T *dst, float a, float b, float c, float d) {
    struct alignas(8) Four { T x[4]; } v;
    v.x[0] = rounded<T>(a); v.x[1] = rounded<T>(b); v.x[2] = rounded<T>(c); v.x[3] = rounded<T>(d);
    *reinterpret_cast<Four *>(dst) = v;
}

struct AttnQ8Params {
    PoolViewQ8 pool;
    const void *q;
    void *o;
    int64_t q_stride;
    const int32_t *block_table;
    int64_t table_cols;
    int num_rows;
    const int32_t *seq_ids, *seq_lens;
    int batch, num_q_heads, group, groups;  // groups: units of up to 8 * NT query heads for each kv head
    int cur_layer, tile_shift;              // tiles of a block: 1 << tile_shift
    float scale_log2;
    int *error_flags, *arrive;
    float *head_rows, *block_rows;          // [worker] and [2 * block] rows of HC * D values + HC log-sums
};

struct Piece {      // a (sequence, head) that a warp has some tiles of
    int b, hp;      // batch index; kv head * groups + head group
    int flags;      // 1 valid, 2 has the first tile, 4 has the last tile, 8 parked in the ring (else in the warp's row)
    int nt;         // tiles of the whole (sequence, head)
    long long p0;   // where it starts in the launch's order
};

// First position of thread block c's range.
__device__ __forceinline__ long long range_start(int c, long long T, int R) { return (long long)c * T / R; }
// Thread block whose range holds position x.
__device__ __forceinline__ int range_owner(long long x, long long T, int R) { return (int)(((x + 1) * R - 1) / T); }

template <typename T, int CODE, int D, int NT, bool DUP, int WARPS, int STAGES, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) attn_q8_kernel(const __grid_constant__ AttnQ8Params p) {
    constexpr int HC = DUP ? 4 : 8 * NT;        // query heads of a unit
    constexpr int TILE = kTileTokens * D;       // bytes of K (or V)
    constexpr int STAGE = 2 * TILE + 48;        // K, V, and: K scale, V scale, b, hp, flags, tokens, tile, tiles, start
    constexpr int KW = D / 16;                  // words of K a thread takes from a token's row = k-steps
    constexpr int VW = D / 32;                  // words of V a thread takes from a token's row
    constexpr int MT = D / 16;                  // row tiles of O^T
    constexpr int ROW = HC * D + HC;            // floats of a partial row
    static_assert(STAGES * STAGE >= ROW * 4, "a piece is parked in its warp's ring");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Piece first_piece[WARPS], last_piece[WARPS];
    __shared__ long long scan_w[WARPS], start_pos[WARPS];
    __shared__ int start_b[WARPS];
    __shared__ int cross_valid[2], cross_f[2], cross_n[2], cross_b[2], cross_hp[2], cross_last[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int P = p.pool.num_kv_heads * p.groups;
    uint8_t *ring_ptr = smem + warp * (STAGES * STAGE);
    const uint32_t ring = smem_addr(ring_ptr);

    // ---- this block's range ---------------------------------------------------------------------------------
    const long long most_tiles = p.table_cols << p.tile_shift;  // what a row of the table can hold
    auto tiles_of = [&](int len) { return len <= 0 ? 0 : (int)min(((long long)len + kTileTokens - 1) / kTileTokens, most_tiles); };
    const int per = (p.batch + WARPS * 32 - 1) / (WARPS * 32);
    long long mine = 0;
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        if (b < p.batch) {
            const int nt = tiles_of(p.seq_lens[b]);
            if (nt > 0) mine += nt + kUnitCost;
        }
    }
    mine *= P;
    long long incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long n = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += n;
    }
    if (lane == 31) scan_w[warp] = incl;
    if (lane == 0) first_piece[warp].flags = last_piece[warp].flags = 0;
    if (tid < 2) cross_valid[tid] = cross_last[tid] = 0;
    __syncthreads();
    long long total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += scan_w[w];
        total += scan_w[w];
    }
    const int R = (int)max(1ll, min((long long)gridDim.x, total / kMinTiles));
    const int cta = blockIdx.x;
    if (total == 0 || cta >= R) return;
    const long long lo = range_start(cta, total, R), hi = range_start(cta + 1, total, R);
    {
        const long long from = before + incl - mine;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const long long x = lo + (hi - lo) * w / WARPS;
            if (x >= from && x < from + mine) {
                start_b[w] = tid * per;
                start_pos[w] = from;
            }
        }
    }
    __syncthreads();
    const long long wlo = lo + (hi - lo) * warp / WARPS, whi = lo + (hi - lo) * (warp + 1) / WARPS;

    // ---- where the warp reads next (all of this is the same in every lane, the windows apart) ---------------------
    bool bad = false;
    int cb = 0, chp = 0, ch = 0, chg = 0, cnt = 0, cj = 0, cjend = 0, clen = 0, crow = 0, cbase = 0;
    long long cp0 = 0;
    bool more = false, cfirst = true;
    int wb = 0, wlen = 0, wrow = 0;         // lane l: length and table row of sequence wb + l
    int ids = 0, ids_next = 0, ids0 = 0, ids0_next = 0;  // block ids of 32 tiles: at cbase, behind it, at tile 0 of this
                                                         // sequence and of the next
    auto load_window = [&](int b) {
        wb = b;
        wlen = b + lane < p.batch ? __ldg(p.seq_lens + b + lane) : 0;
        wrow = b + lane < p.batch ? __ldg(p.seq_ids + b + lane) : 0;
    };
    auto load_ids = [&](int row, int first, int nt) {
        const int tile = first + lane;
        if (row < 0 || row >= p.num_rows || tile >= nt) return -1;
        return __ldg(p.block_table + (int64_t)row * p.table_cols + (tile >> p.tile_shift));
    };
    // first sequence behind cb that has tokens: its window lane is found by a vote; -1: none
    auto next_sequence = [&]() {
        int at = cb + 1;
        while (at < p.batch) {
            if (at >= wb + 32) load_window(at);
            const unsigned some = __ballot_sync(0xffffffffu, wlen > 0) & (0xffffffffu << (at - wb));
            if (some) return wb + __ffs(some) - 1;
            at = wb + 32;
        }
        return -1;
    };
    int nb = -1, nrow = 0, nlen = 0;        // the next sequence
    auto look_ahead = [&]() {
        nb = next_sequence();
        if (nb >= 0) {
            nrow = __shfl_sync(0xffffffffu, wrow, nb - wb);
            nlen = __shfl_sync(0xffffffffu, wlen, nb - wb);
            ids0_next = load_ids(nrow, 0, tiles_of(nlen));
        }
    };
    if (wlo < whi) {
        // the sequence that holds position wlo
        long long at = start_pos[warp];
        int b = start_b[warp];
        while (b < p.batch) {
            load_window(b);
            const int nt = tiles_of(wlen);
            const long long w = nt > 0 ? (long long)(nt + kUnitCost) * P : 0;
            long long sum = w;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const long long n = __shfl_up_sync(0xffffffffu, sum, d);
                if (lane >= d) sum += n;
            }
            const unsigned here = __ballot_sync(0xffffffffu, wlo < at + sum);
            if (here) {
                const int src = __ffs(here) - 1;
                cb = b + src;
                at += __shfl_sync(0xffffffffu, sum - w, src);
                clen = __shfl_sync(0xffffffffu, wlen, src);
                crow = __shfl_sync(0xffffffffu, wrow, src);
                break;
            }
            at += __shfl_sync(0xffffffffu, sum, 31);
            b += 32;
        }
        cnt = tiles_of(clen);
        const int w = cnt + kUnitCost;
        const long long rem = wlo - at;
        chp = (int)min(rem / w, (long long)P - 1);
        cp0 = at + (long long)chp * w;
        cj = max((int)(wlo - cp0) - kUnitCost, 0);
        ch = chp / p.groups;
        chg = chp - ch * p.groups;
        cjend = (int)min((long long)cnt, whi - cp0 - kUnitCost);
        more = cj < cjend;
        if (more) {
            cbase = cj;
            ids = load_ids(crow, cj, cnt);
            ids_next = load_ids(crow, cj + 32, cnt);
            ids0 = load_ids(crow, 0, cnt);
            look_ahead();
            bad |= crow < 0 || crow >= p.num_rows || (long long)cnt * kTileTokens < clen;
        }
    }
    // One tile into ring stage `slot`, and the cursor moves on.
    int issued = 0;
    auto issue = [&](int slot) {
        if (!more) return;
        if (cj - cbase == 32) {
            ids = ids_next;
            cbase += 32;
            ids_next = load_ids(crow, cbase + 32, cnt);
        }
        const int blk = __shfl_sync(0xffffffffu, ids, cj - cbase);
        const uint32_t st = ring + slot * STAGE;
        int tokens = min(kTileTokens, clen - cj * kTileTokens);
        if (blk >= 0 && blk < p.pool.total_blocks) {
            int seg = 0;
            int64_t row = blk;
            if (p.pool.num_segments > 1) locate_block(p.pool, blk, seg, row);
            const int64_t tile = tile_index(p.pool, row, p.cur_layer, ch);
            const int64_t off = ((tile << p.tile_shift) + (cj & ((1 << p.tile_shift) - 1))) * TILE;
            const uint8_t *kt = p.pool.k_base[seg] + off, *vt = p.pool.v_base[seg] + off;
#pragma unroll
            for (int i = 0; i < TILE / 512; ++i) {
                // 16-byte piece `id` of the tile; D = 128: piece c of token r goes to c ^ (r & 7); D = 64: two tokens share a
                // 128-byte line, whose pieces go to c ^ (line & 3) * 2.  Either way the reads below meet no conflict.
                const int id = i * 32 + lane, line = id >> 3, c = id & 7;
                const uint32_t to = line * 128 + ((c ^ (D == 128 ? line & 7 : (line & 3) * 2)) << 4);
                cp16(st + to, kt + id * 16);
                cp16(st + TILE + to, vt + id * 16);
            }
            if (lane < 2) cp4(st + 2 * TILE + lane * 4, (lane ? p.pool.v_scale[seg] : p.pool.k_scale[seg]) + tile);
        } else {
            tokens = 0;
            bad = true;
        }
        const bool last = cj + 1 == cjend;
        if (lane == 0) {
            const int flags = (cfirst ? 1 : 0) | (last ? 2 : 0);
            asm volatile("st.shared.v2.b32 [%0], {%1,%2};\n" ::"r"(st + 2 * TILE + 8), "r"(cb), "r"(chp) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(st + 2 * TILE + 16), "r"(flags), "r"(tokens), "r"(cj), "r"(cnt) : "memory");
            asm volatile("st.shared.b64 [%0], %1;\n" ::"r"(st + 2 * TILE + 32), "l"(cp0) : "memory");
        }
        ++issued;
        cfirst = false;
        ++cj;
        if (last) {     // the next (sequence, head)
            cfirst = true;
            cp0 += cnt + kUnitCost;
            if (++chp == P) {
                if (nb < 0) {
                    more = false;
                    return;
                }
                cb = nb;
                crow = nrow;
                clen = nlen;
                cnt = tiles_of(clen);
                chp = ch = chg = 0;
                ids0 = ids0_next;
                look_ahead();
                bad |= crow < 0 || crow >= p.num_rows || (long long)cnt * kTileTokens < clen;
            } else if (++chg == p.groups) {
                chg = 0;
                ++ch;
            }
            cj = cbase = 0;
            cjend = (int)min((long long)cnt, whi - cp0 - kUnitCost);
            more = cjend > 0;
            ids = ids0;
            if (more) ids_next = load_ids(crow, 32, cnt);
        }
    };

    float o[NT][MT][4];
    uint32_t qf[NT][KW][2];
    float qfac[NT][2];       // scale_log2 and what undoes the normalisation of q, for heads 2t and 2t + 1
    float thr[NT][2], base[NT][2], l[NT][2];
    float vref = 0.f, vinv = 0.f;
    int piece_starts = 0;

#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) {
        issue(s);
        cp_commit();
    }
    int slot = 0, done = 0;
    while (done < issued) {
        cp_wait<STAGES - 2>();
        __syncwarp();       // every lane's part of the tile has landed, and the stage before it is read
        issue(slot == 0 ? STAGES - 1 : slot - 1);
        cp_commit();
        const uint32_t st = ring + slot * STAGE;
        ++done;
        slot = slot + 1 == STAGES ? 0 : slot + 1;
        const uint4 ma = lds16(st + 2 * TILE), mb = lds16(st + 2 * TILE + 16);
        const float ks = __uint_as_float(ma.x), vs = __uint_as_float(ma.y);
        const int b = (int)ma.z, hp = (int)ma.w, flags = (int)mb.x, tokens = (int)mb.y;
        int hq0 = 0, heads = 0;     // query heads of the unit
        if (flags & 3) {
            const int kvh = hp / p.groups;
            hq0 = kvh * p.group + (hp - kvh * p.groups) * HC;
            heads = min(HC, (kvh + 1) * p.group - hq0);
        }

        if (flags & 1) {    // first tile of a piece
            piece_starts = mb.z == 0;
            const T *qb = (const T *)p.q + b * p.q_stride + (int64_t)hq0 * D + t * (D / 4);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                // column g of the tile is query head g (DUP: g & 3, so that columns 4-7 repeat 0-3); this thread holds its
                // dims [t D / 4, (t + 1) D / 4)
                const int head = DUP ? (g & 3) : n * 8 + g;
                uint32_t raw[KW * 2];
#pragma unroll
                for (int i = 0; i < KW / 2; ++i) {
                    uint4 x = make_uint4(0u, 0u, 0u, 0u);
                    if (head < heads) x = __ldg(reinterpret_cast<const uint4 *>(qb + (int64_t)head * D) + i);
                    raw[4 * i] = x.x; raw[4 * i + 1] = x.y; raw[4 * i + 2] = x.z; raw[4 * i + 3] = x.w;
                }
                float fac = p.scale_log2;
                if constexpr (sizeof(T) == 2 && !std::is_same<T, __half>::value) {
                    // bf16: a power of two brings the head's largest element to [2^14, 2^15); then fp16 holds every element
                    // down to 2^-28 of it exactly
                    uint32_t peak = 0;
#pragma unroll
                    for (int i = 0; i < KW * 2; ++i) peak = max(peak, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
                    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
                    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
                    const int e = peak == 0 ? 0 : min(max(14 + 127 - (int)(peak >> 7), -120), 120);
                    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                    fac *= __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                    for (int i = 0; i < KW * 2; ++i)
                        raw[i] = half2_bits(__floats2half2_rn(__uint_as_float(raw[i] << 16) * up, __uint_as_float(raw[i] & 0xffff0000u) * up));
                }
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    qf[n][i][0] = raw[2 * i];
                    qf[n][i][1] = raw[2 * i + 1];
                }
                // columns 2t and 2t + 1 belong to the lanes with g = 2t and 2t + 1
                qfac[n][0] = __shfl_sync(0xffffffffu, fac, 8 * t);
                qfac[n][1] = __shfl_sync(0xffffffffu, fac, 8 * t + 4);
#pragma unroll
                for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
                thr[n][0] = thr[n][1] = -INFINITY;
                base[n][0] = base[n][1] = l[n][0] = l[n][1] = 0.f;
            }
            vref = 0.f;
        }

        if (tokens > 0) {
            // ---- S^T = K Q^T
            float sc[NT][2][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][0][e] = sc[n][1][e] = 0.f;
            {
                uint32_t lo8[KW], hi8[KW];      // words of tokens g and g + 8
                if constexpr (D == 128) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t at = st + g * 128 + (((2 * t + i) ^ g) << 4);
                        const uint4 x = lds16(at), y = lds16(at + 1024);
                        lo8[4 * i] = x.x; lo8[4 * i + 1] = x.y; lo8[4 * i + 2] = x.z; lo8[4 * i + 3] = x.w;
                        hi8[4 * i] = y.x; hi8[4 * i + 1] = y.y; hi8[4 * i + 2] = y.z; hi8[4 * i + 3] = y.w;
                    }
                } else {
                    const int line = g >> 1;
                    const uint32_t at = st + line * 128 + (((((g & 1) << 2) + t) ^ (line * 2)) << 4);
                    const uint4 x = lds16(at), y = lds16(at + 512);
                    lo8[0] = x.x; lo8[1] = x.y; lo8[2] = x.z; lo8[3] = x.w;
                    hi8[0] = y.x; hi8[1] = y.y; hi8[2] = y.z; hi8[3] = y.w;
                }
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    uint32_t a0, a1, a2, a3;
                    widen<CODE>(lo8[i], a0, a2);
                    widen<CODE>(hi8[i], a1, a3);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma(sc[n][i & 1], a0, a1, a2, a3, qf[n][i][0], qf[n][i][1]);
                }
            }
            // ---- softmax: token g (elements 0, 1) and g + 8 (2, 3) of heads 2t, 2t + 1
            const bool on0 = g < tokens, on1 = g + 8 < tokens;
            float s0[NT][4];
            bool above = false;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float f0 = qfac[n][0] * ks, f1 = qfac[n][1] * ks;
                s0[n][0] = on0 ? (sc[n][0][0] + sc[n][1][0]) * f0 : -INFINITY;
                s0[n][1] = on0 ? (sc[n][0][1] + sc[n][1][1]) * f1 : -INFINITY;
                s0[n][2] = on1 ? (sc[n][0][2] + sc[n][1][2]) * f0 : -INFINITY;
                s0[n][3] = on1 ? (sc[n][0][3] + sc[n][1][3]) * f1 : -INFINITY;
                above |= fmaxf(s0[n][0], s0[n][2]) > thr[n][0] || fmaxf(s0[n][1], s0[n][3]) > thr[n][1];
            }
            if (__any_sync(0xffffffffu, above)) {   // the maxima settle after the first tiles of a piece
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float m = fmaxf(s0[n][e], s0[n][e + 2]);
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                        m = fmaxf(m, thr[n][e] - kLag);
                        const float nb = m == -INFINITY ? 0.f : m - kBoost;
                        const float a = thr[n][e] == -INFINITY ? 1.f : ex2(base[n][e] - nb);   // before: all weights were 0
                        thr[n][e] = m + kLag;
                        base[n][e] = nb;
                        l[n][e] *= a;
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            o[n][i][e] *= a;
                            o[n][i][e + 2] *= a;
                        }
                    }
            }
            // The block's V scale goes into the weights while it is near the piece's first one, otherwise the block's
            // product is scaled on its own.
            if (vref == 0.f) {
                vref = vs > 0.f ? vs : 1.f;
                vinv = 1.f / vref;
            }
            const float ratio = vs * vinv;
            const bool near_ref = ratio <= kScaleRange && ratio >= 1.f / kScaleRange;
            const float wr = near_ref ? ratio : 1.f;
            uint32_t pb[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float w0 = ex2(s0[n][0] - base[n][0]), w1 = ex2(s0[n][1] - base[n][1]);
                const float w2 = ex2(s0[n][2] - base[n][0]), w3 = ex2(s0[n][3] - base[n][1]);
                l[n][0] += w0 + w2;
                l[n][1] += w1 + w3;
                __half2 x = __floats2half2_rn(w0 * wr, w1 * wr), y = __floats2half2_rn(w2 * wr, w3 * wr);
                if (DUP) {  // columns 4-7: what the rounding of columns 0-3 left over
                    const float2 fx = __half22float2(x), fy = __half22float2(y);
                    const __half2 rx = __floats2half2_rn(w0 * wr - fx.x, w1 * wr - fx.y);
                    const __half2 ry = __floats2half2_rn(w2 * wr - fy.x, w3 * wr - fy.y);
                    if (t >= 2) {
                        x = rx;
                        y = ry;
                    }
                }
                pb[n][0] = transpose8x8(half2_bits(x));
                pb[n][1] = transpose8x8(half2_bits(y));
            }
            // ---- O^T += V^T P^T: row tile i has dim (D / 8) g + i in its row g and dim (D / 8) g + MT + i in its row g + 8
            uint32_t vw[4][VW];     // tokens 2t, 2t + 1, 2t + 8, 2t + 9
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int tok = 2 * t + (k & 1) + (k >> 1) * 8;
                if constexpr (D == 128) {
                    const uint4 x = lds16(st + TILE + tok * 128 + ((g ^ (tok & 7)) << 4));
                    vw[k][0] = x.x; vw[k][1] = x.y; vw[k][2] = x.z; vw[k][3] = x.w;
                } else {
                    const int line = tok >> 1;
                    const uint2 x = lds8(st + TILE + line * 128 + (((((tok & 1) << 2) + (g >> 1)) ^ ((line & 3) * 2)) << 4) + (g & 1) * 8);
                    vw[k][0] = x.x; vw[k][1] = x.y;
                }
                if (CODE == MKV_Q8_E4M3 && tokens < kTileTokens && tok >= tokens) {
                    // behind the sequence's end any byte may stand, NaN among them, and 0 x NaN is NaN
#pragma unroll
                    for (int i = 0; i < VW; ++i) vw[k][i] = 0u;
                }
            }
            auto fragments = [&](int i, uint32_t (&x)[4], uint32_t (&y)[4]) {
                // words i: dims 4i ... 4i + 3 of this thread's; x[d]: (token 2t, token 2t + 1), y[d]: tokens 2t + 8, 2t + 9
                widen<CODE>(__byte_perm(vw[0][i], vw[1][i], 0x5140), x[0], x[1]);
                widen<CODE>(__byte_perm(vw[0][i], vw[1][i], 0x7362), x[2], x[3]);
                widen<CODE>(__byte_perm(vw[2][i], vw[3][i], 0x5140), y[0], y[1]);
                widen<CODE>(__byte_perm(vw[2][i], vw[3][i], 0x7362), y[2], y[3]);
            };
#pragma unroll
            for (int i = 0; i < VW / 2; ++i) {
                uint32_t xa[4], ya[4], xb[4], yb[4];
                fragments(i, xa, ya);               // dims 4i + d
                fragments(i + VW / 2, xb, yb);      // dims MT + 4i + d
                if (near_ref) {
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma(o[n][4 * i + d], xa[d], xb[d], ya[d], yb[d], pb[n][0], pb[n][1]);
                } else {
#pragma unroll
                    for (int d = 0; d < 4; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            float part[4] = {0.f, 0.f, 0.f, 0.f};
                            mma(part, xa[d], xb[d], ya[d], yb[d], pb[n][0], pb[n][1]);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[n][4 * i + d][e] = fmaf(part[e], ratio, o[n][4 * i + d][e]);
                        }
                }
            }
        }

        if (flags & 2) {    // last tile of the piece
            const bool ends = (int)mb.z + 1 == (int)mb.w, whole = piece_starts && ends, final_piece = done == issued;
            const float vr = vref == 0.f ? 1.f : vref;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 4);
                    l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 8);
                    l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], 16);
                }
                if (DUP) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][i][e] += __shfl_xor_sync(0xffffffffu, o[n][i][e], 2);
                }
            }
            float *row = nullptr;
            if (!whole) {
                Piece &pc = final_piece && first_piece[warp].flags ? last_piece[warp] : first_piece[warp];
                // (a piece that is neither first nor last of its warp is whole)
                row = final_piece ? reinterpret_cast<float *>(ring_ptr)
                                  : p.head_rows + ((int64_t)cta * WARPS + warp) * ROW;
                __syncwarp();
                if (lane == 0) {
                    pc.b = b;
                    pc.hp = hp;
                    pc.nt = (int)mb.w;
                    pc.flags = 1 | (piece_starts ? 2 : 0) | (ends ? 4 : 0) | (final_piece ? 8 : 0);
                    asm volatile("ld.shared.b64 %0, [%1];\n" : "=l"(pc.p0) : "r"(st + 2 * TILE + 32) : "memory");
                }
                __syncwarp();
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int head = n * 8 + 2 * t + e;
                    if (head >= heads || head >= HC) continue;
                    if (whole) {
                        const float f = vr / l[n][e];
                        T *dst = (T *)p.o + ((int64_t)b * p.num_q_heads + hq0 + head) * D + g * (D / 8);
#pragma unroll
                        for (int i = 0; i < MT; i += 4) {
                            store4<T>(dst + i, o[n][i][e] * f, o[n][i + 1][e] * f, o[n][i + 2][e] * f, o[n][i + 3][e] * f);
                            store4<T>(dst + MT + i, o[n][i][e + 2] * f, o[n][i + 1][e + 2] * f, o[n][i + 2][e + 2] * f, o[n][i + 3][e + 2] * f);
                        }
                    } else {
                        const float f = l[n][e] == 0.f ? 0.f : vr / l[n][e];
                        float *dst = row + head * D + g * (D / 8);
#pragma unroll
                        for (int i = 0; i < MT; i += 4) {
                            *reinterpret_cast<float4 *>(dst + i) = make_float4(o[n][i][e] * f, o[n][i + 1][e] * f, o[n][i + 2][e] * f, o[n][i + 3][e] * f);
                            *reinterpret_cast<float4 *>(dst + MT + i) =
                                make_float4(o[n][i][e + 2] * f, o[n][i + 1][e + 2] * f, o[n][i + 2][e + 2] * f, o[n][i + 3][e + 2] * f);
                        }
                        if (g == 0) row[HC * D + head] = log2f(l[n][e]) + base[n][e];
                    }
                }
        }
    }
    cp_wait<0>();
    if (bad && lane == 0 && p.error_flags) atomicOr(p.error_flags, 1);

    // ---- pieces of cut (sequence, head)s: those of this block's warps are folded, one warp for each query head -----------
    __syncthreads();
    bool leads = false;     // lane c: the first or last piece of warp c / 2 is the block's first piece of its (sequence, head)
    if (lane < 2 * WARPS) {
        const int fl = ((lane & 1) ? last_piece[lane >> 1] : first_piece[lane >> 1]).flags;
        leads = fl != 0 && ((fl & 2) != 0 || lane == 0);
    }
    unsigned leaders = __ballot_sync(0xffffffffu, leads);
    int item = 0;
    while (leaders) {
        const int c = __ffs(leaders) - 1;
        leaders &= leaders - 1;
        const Piece lead = (c & 1) ? last_piece[c >> 1] : first_piece[c >> 1];
        const int kvh = lead.hp / p.groups, hq0 = kvh * p.group + (lead.hp - kvh * p.groups) * HC;
        const int heads = min(HC, (kvh + 1) * p.group - hq0);
        for (int r = 0; r < heads; ++r) {
            if (item++ % WARPS != warp) continue;
            float m = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            int x = c >> 1, fl = lead.flags;
            for (;;) {
                const float *row = (fl & 8) ? reinterpret_cast<const float *>(smem + x * (STAGES * STAGE))
                                            : p.head_rows + ((int64_t)cta * WARPS + x) * ROW;
                const float ls = row[HC * D + r];
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (lane * 4 < D) v = *reinterpret_cast<const float4 *>(row + r * D + lane * 4);
                const float nm = fmaxf(m, ls), off = nm == -INFINITY ? 0.f : nm;
                const float a = exp2f(m - off), e = exp2f(ls - off);
                acc.x = acc.x * a + v.x * e; acc.y = acc.y * a + v.y * e; acc.z = acc.z * a + v.z * e; acc.w = acc.w * a + v.w * e;
                sum = sum * a + e;
                m = nm;
                if (fl & 4) break;
                do ++x; while (x < WARPS && first_piece[x].flags == 0);
                if (x == WARPS) break;
                fl = first_piece[x].flags;
            }
            if ((lead.flags & 2) && (fl & 4)) {     // all of it lies in this block
                const float f = 1.f / sum;
                if (lane * 4 < D)
                    store4<T>((T *)p.o + ((int64_t)lead.b * p.num_q_heads + hq0 + r) * D + lane * 4, acc.x * f, acc.y * f, acc.z * f, acc.w * f);
            } else {
                // row 0 of the block: of a (sequence, head) that comes from the block before it; row 1: of one that starts here
                const int s = (lead.flags & 2) ? 1 : 0;
                float *row = p.block_rows + ((int64_t)cta * 2 + s) * ROW;
                const float f = sum == 0.f ? 0.f : 1.f / sum;
                if (lane * 4 < D) __stcg(reinterpret_cast<float4 *>(row + r * D + lane * 4), make_float4(acc.x * f, acc.y * f, acc.z * f, acc.w * f));
                if (lane == 0) {
                    __stcg(row + HC * D + r, log2f(sum) + (m == -INFINITY ? 0.f : m));
                    if (r == 0) {
                        const long long at = lead.p0 + kUnitCost;
                        cross_f[s] = range_owner(at, total, R);
                        cross_n[s] = range_owner(at + lead.nt - 1, total, R) - cross_f[s] + 1;
                        cross_b[s] = lead.b;
                        cross_hp[s] = lead.hp;
                        cross_valid[s] = 1;
                    }
                }
            }
        }
    }
    __threadfence();
    __syncthreads();
    if (tid < 2 && cross_valid[tid]) {
        int *at = p.arrive + cross_f[tid];      // no two (sequence, head)s that leave a block start in the same one
        if (atomicAdd(at, 1) == cross_n[tid] - 1) {
            *at = 0;
            cross_last[tid] = 1;
            __threadfence();
        }
    }
    __syncthreads();
#pragma unroll 1
    for (int s = 0; s < 2; ++s) {
        if (!cross_last[s]) continue;
        const int f = cross_f[s], n = cross_n[s], kvh = cross_hp[s] / p.groups;
        const int hq0 = kvh * p.group + (cross_hp[s] - kvh * p.groups) * HC, heads = min(HC, (kvh + 1) * p.group - hq0);
        for (int r = warp; r < heads; r += WARPS) {
            constexpr int U = 8;    // rows in flight
            float m = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int i0 = 0; i0 < n; i0 += U) {
                float ls[U];
                float4 v[U];
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    const int k = min(i0 + i, n - 1);
                    const float *row = p.block_rows + ((int64_t)(f + k) * 2 + (k == 0 ? 1 : 0)) * ROW;
                    ls[i] = __ldcg(row + HC * D + r);
                    v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (lane * 4 < D) v[i] = __ldcg(reinterpret_cast<const float4 *>(row + r * D + lane * 4));
                }
                float nm = m;
#pragma unroll
                for (int i = 0; i < U; ++i) nm = fmaxf(nm, ls[i]);
                const float off = nm == -INFINITY ? 0.f : nm, a = exp2f(m - off);
                acc.x *= a; acc.y *= a; acc.z *= a; acc.w *= a;
                sum *= a;
#pragma unroll
                for (int i = 0; i < U; ++i) {
                    if (i0 + i >= n) break;
                    const float e = exp2f(ls[i] - off);
                    acc.x += v[i].x * e; acc.y += v[i].y * e; acc.z += v[i].z * e; acc.w += v[i].w * e;
                    sum += e;
                }
                m = nm;
            }
            const float f1 = 1.f / sum;
            if (lane * 4 < D)
                store4<T>((T *)p.o + ((int64_t)cross_b[s] * p.num_q_heads + hq0 + r) * D + lane * 4, acc.x * f1, acc.y * f1, acc.z * f1, acc.w * f1);
        }
    }
}

// ------------------------------------------------------------------ host side
constexpr int kWarps = 8;
constexpr int kMaxBlocksPerSm = 2;
constexpr size_t kErrorBytes = 256;     // error word, then the arrival counters

static size_t zero_bytes(int sms) { return kErrorBytes + (((size_t)sms * kMaxBlocksPerSm * sizeof(int) + 255) & ~(size_t)255); }
// Query heads of a unit: 4 (columns 4-7 of the tile then carry what fp16 loses of the weights), 8 or 16.
static int unit_heads(int group) { return group <= 4 ? 4 : group <= 8 ? 8 : 16; }
static int blocks_per_sm(int heads) { return heads == 16 ? 1 : 2; }

static bool fast_shape(int group, int head_dim, int block_size) {
    (void)group;
    return (head_dim == 64 || head_dim == 128) && block_size >= 16 && (block_size & (block_size - 1)) == 0;
}

// 16-byte loads of q and of the pool, 8-byte stores of o.
static bool fast_aligned(const PoolViewQ8 &pv, const void *q, int64_t q_stride, const void *o) {
    uintptr_t bits = (uintptr_t)q | (uintptr_t)(q_stride * 2) | ((uintptr_t)o << 1);
    for (int i = 0; i < pv.num_segments; ++i) bits |= (uintptr_t)pv.k_base[i] | (uintptr_t)pv.v_base[i];
    return (bits & 15) == 0;
}

template <typename T, int CODE, int D, int NT, bool DUP, int STAGES, int BLOCKS>
static cudaError_t launch_fast(const AttnQ8Params &p, unsigned grid, cudaStream_t s) {
    constexpr int smem = kWarps * STAGES * (2 * kTileTokens * D + 48);
    auto kernel = attn_q8_kernel<T, CODE, D, NT, DUP, kWarps, STAGES, BLOCKS>;
    static std::atomic<bool> configured[64];    // per device; setting the attribute twice is harmless
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    kernel<<<grid, kWarps * 32, smem, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int CODE>
static cudaError_t launch_fast_shape(const AttnQ8Params &p, int head_dim, unsigned grid, cudaStream_t s) {
    const int heads = unit_heads(p.group);
    if (head_dim == 128)
        return heads == 4   ? launch_fast<T, CODE, 128, 1, true, 3, 2>(p, grid, s)
               : heads == 8 ? launch_fast<T, CODE, 128, 1, false, 3, 2>(p, grid, s)
                            : launch_fast<T, CODE, 128, 2, false, 6, 1>(p, grid, s);
    return heads == 4   ? launch_fast<T, CODE, 64, 1, true, 6, 2>(p, grid, s)
           : heads == 8 ? launch_fast<T, CODE, 64, 1, false, 6, 2>(p, grid, s)
                        : launch_fast<T, CODE, 64, 2, false, 8, 1>(p, grid, s);
}

}  // namespace mkv

using namespace mkv;

extern "C" {

size_t mkv_attn_q8_zero_bytes(int device) {
    int sms = 0;
    return mkv_sm_count(device, &sms) == MKV_OK ? zero_bytes(sms) : 0;
}

size_t mkv_attn_q8_workspace_bytes(int device, int batch, int num_q_heads, int num_kv_heads, int head_dim) {
    int sms = 0;
    if (batch < 0 || num_q_heads < 1 || num_kv_heads < 1 || head_dim < 1 || mkv_sm_count(device, &sms) != MKV_OK) return 0;
    const int heads = unit_heads(num_q_heads / num_kv_heads);
    const size_t rows = (size_t)sms * blocks_per_sm(heads) * (kWarps + 2);
    return zero_bytes(sms) + rows * heads * (head_dim + 1) * sizeof(float);
}

int mkv_paged_attention_q8(int device, void *stream, const void *q, int64_t q_stride, void *o, int dtype,
                           const mkv_pool_q8 *pool, const int32_t *block_table, int64_t table_stride, int num_rows,
                           const int32_t *seq_ids, const int32_t *seq_lens, int batch, int num_q_heads, int cur_layer,
                           float softmax_scale, int max_seq_len, void *workspace, size_t workspace_bytes) {
    PoolViewQ8 pv;
    int st = validate_pool_q8(pool, &pv);
    if (st) return st;
    if (!dtype_ok(dtype)) return MKV_ERR_DTYPE;
    if (batch < 0 || num_q_heads < 1 || table_stride < 1 || num_rows < 0 || max_seq_len < 0) return MKV_ERR_SHAPE;
    if (num_q_heads % pv.num_kv_heads != 0 || pv.head_dim > 32 * kPlainDims) return MKV_ERR_SHAPE;
    if (q_stride < (int64_t)num_q_heads * pv.head_dim) return MKV_ERR_SHAPE;
    if (cur_layer < 0 || cur_layer >= pv.num_layers) return MKV_ERR_RANGE;
    if (batch == 0) return MKV_OK;
    if (!q || !o || !block_table || !seq_ids || !seq_lens) return MKV_ERR_NULL;
    if (workspace && ((uintptr_t)workspace & 255) != 0) return MKV_ERR_WORKSPACE;
    const int64_t blocks = ceil_div64((int64_t)batch * num_q_heads, 4);
    if (blocks > 0x7fffffff) return MKV_ERR_SHAPE;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    int *flags = workspace && workspace_bytes >= kErrorBytes ? (int *)workspace : nullptr;
    const float scale_log2 = softmax_scale * kLog2e;
    const int group = num_q_heads / pv.num_kv_heads;
    if (dtype != MKV_F32 && fast_shape(group, pv.head_dim, pv.block_size) && fast_aligned(pv, q, q_stride, o)) {
        int sms = 0;
        if ((st = mkv_sm_count(device, &sms))) return st;
        if (!workspace || workspace_bytes < mkv_attn_q8_workspace_bytes(device, batch, num_q_heads, pv.num_kv_heads, pv.head_dim))
            return MKV_ERR_WORKSPACE;
        const int heads = unit_heads(group);
        AttnQ8Params p;
        p.pool = pv;
        p.q = q;
        p.o = o;
        p.q_stride = q_stride;
        p.block_table = block_table;
        p.table_cols = table_stride;
        p.num_rows = num_rows;
        p.seq_ids = seq_ids;
        p.seq_lens = seq_lens;
        p.batch = batch;
        p.num_q_heads = num_q_heads;
        p.group = group;
        p.groups = (group + heads - 1) / heads;
        p.cur_layer = cur_layer;
        p.tile_shift = 0;
        while ((kTileTokens << p.tile_shift) < pv.block_size) ++p.tile_shift;
        p.scale_log2 = scale_log2;
        const int most = sms * blocks_per_sm(heads);
        const int64_t positions = (int64_t)batch * (ceil_div64(max_seq_len, kTileTokens) + kUnitCost) * pv.num_kv_heads * p.groups;
        const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, positions / kMinTiles));
        p.error_flags = (int *)workspace;
        p.arrive = (int *)((char *)workspace + kErrorBytes);
        p.head_rows = (float *)((char *)workspace + zero_bytes(sms));
        p.block_rows = p.head_rows + (int64_t)most * kWarps * heads * (pv.head_dim + 1);
        cudaStream_t s = (cudaStream_t)stream;
        const cudaError_t e =
            pv.code == MKV_Q8_INT8
                ? (dtype == MKV_F16 ? launch_fast_shape<__half, MKV_Q8_INT8>(p, pv.head_dim, grid, s)
                                    : launch_fast_shape<__nv_bfloat16, MKV_Q8_INT8>(p, pv.head_dim, grid, s))
                : (dtype == MKV_F16 ? launch_fast_shape<__half, MKV_Q8_E4M3>(p, pv.head_dim, grid, s)
                                    : launch_fast_shape<__nv_bfloat16, MKV_Q8_E4M3>(p, pv.head_dim, grid, s));
        return e == cudaSuccess ? MKV_OK : set_cuda_error(e);
    }
#define PLAIN(T, CODE)                                                                                                  \
    attn_q8_plain_kernel<T, CODE><<<(unsigned)blocks, 128, 0, (cudaStream_t)stream>>>(                                  \
        (const T *)q, q_stride, (T *)o, pv, block_table, table_stride, num_rows, seq_ids, seq_lens, batch, num_q_heads, \
        cur_layer, scale_log2, flags)
    if (pv.code == MKV_Q8_INT8) {
        if (dtype == MKV_F16) PLAIN(__half, MKV_Q8_INT8);
        else if (dtype == MKV_BF16) PLAIN(__nv_bfloat16, MKV_Q8_INT8);
        else PLAIN(float, MKV_Q8_INT8);
    } else {
        if (dtype == MKV_F16) PLAIN(__half, MKV_Q8_E4M3);
        else if (dtype == MKV_BF16) PLAIN(__nv_bfloat16, MKV_Q8_E4M3);
        else PLAIN(float, MKV_Q8_E4M3);
    }
#undef PLAIN
    MKV_LAUNCH_CHECK();
    return MKV_OK;
}

}  // extern "C"

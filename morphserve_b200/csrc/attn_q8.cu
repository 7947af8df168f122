// Decode attention over the 8-bit pool.
//
// HBM bound: every code is read once for the query heads that share its kv head; what a token costs beyond its bytes is
// the conversion of its codes to fp16, which is why the tensor-core tile is laid out for as few instructions as it is.
//
// Measured (B200, copy peak 6.55 TB/s; several GPUs): 256 sequences of up to 1536, 32 / 8 heads, int8: 402 MB in 83-88 us; 64
// sequences of up to 768, 32 heads, e4m3: 217 MB in 50-51 us; 8 sequences of 8 k to 32 k, 64 / 8 heads, e4m3: 324 MB in 69-74 us
// (0.7 of the peak over all).  While it streams the kernel runs at the peak; the rest is the start (four dependent reads before
// the first tile: 5 us), warps that end 8 to 10 % after the median (SMs differ so much in speed, and equal shares do not even it
// out), and the fold and merge of cut sequences (6 us).  8 sequences of up to 2048: 16.4 us, all of it such latencies.
//
// One launch.  The launch's tiles (32 tokens of one kv head: 32 x D codes of K and of V) stand in one order - sequence by
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
constexpr float kLargest = 3.402823466e38f;     // of fp32

// The smaller one; NaN if either is NaN.
__device__ __forceinline__ float min_nan(float x, float y) {
    float z;
    asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(z) : "f"(x), "f"(y));
    return z;
}

// ------------------------------------------------------------------ plain kernel
// One warp per (sequence, query head); lane l holds dims l, l + 32, ...  fp32 throughout.  Weights are held as unit * 2^(score -
// max), whose sum l stays below 5/8: so the weighted sum of values is no larger than the largest of them.  Likewise a power of two
// takes the query's largest element to [1, 2), so that its products with codes are ordinary numbers whatever the score is made of.
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
    uint32_t peak = 0;
#pragma unroll
    for (int i = 0; i < kPlainDims; ++i) peak = max(peak, __float_as_uint(qr[i]) & 0x7fffffffu);
    const int e = min(max((int)(__reduce_max_sync(0xffffffffu, peak) >> 23), 1), 253);
    const float up = __uint_as_float((uint32_t)e << 23), down = __uint_as_float((uint32_t)(254 - e) << 23);
#pragma unroll
    for (int i = 0; i < kPlainDims; ++i) qr[i] *= down;
    float m = -INFINITY, l = 0.f, unit = 0.125f;
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
        // (a factor too large for 32 bits: 0 times it is 0 all the same)
        const float ks = min_nan(pool.k_scale[seg][tile] * up * scale_log2, kLargest), vs = pool.v_scale[seg][tile];
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
            float a = exp2f(m - base);
            if (l * a > 0.5f) {
                a *= 0.5f;
                unit *= 0.5f;
            }
            const float w = exp2f(sc - base) * unit;
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
constexpr int kHalf = 16;         // tokens of a tensor-core tile
constexpr int kTile = 32;         // tokens of a tile: two of those, so that a loop pass has enough to do
constexpr int kUnitCost = 2;      // phantom tiles in front of a (sequence, head): 1, 2, 3 took the 256-sequence batch 85.5, 87.3, 88.2
                                  // us, the 64-sequence one 53.3, 52.2, 54.0, the long contexts 69.0, 69.2, 70.5
constexpr float kBoost = 6.f;     // weights are held as 2^(score - max + 6): fp16 then reaches 2^-20 of the largest in full
constexpr float kLag = 4.f;       // the running maximum follows only when a score is above it by 2^4
constexpr float kFaint = 90.f;    // how far log2 of a V scale may lie below the reference before its weights are summed apart
constexpr float kAhead = 64.f;    // ... whose scores may then be above theirs by as much

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp16(uint32_t dst, const void *src, uint64_t policy) {
    asm volatile("cp.async.cg.shared.global.L2::cache_hint [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(src), "l"(policy) : "memory");
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
__device__ __forceinline__ void sts16(uint32_t addr, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(addr), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// Four 8 x 8 matrices of 16-bit elements, transposed: thread (g, t) gets elements (2t, g) and (2t + 1, g) of each.
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
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
// Over the lanes of a column of S^T.
__device__ __forceinline__ float column_max(float m) {
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
    return fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
__device__ __forceinline__ __half2 bits_half2(uint32_t x) { return *reinterpret_cast<__half2 *>(&x); }

// int8 codes as fp16: the byte with its sign bit flipped is u = q + 128, and as the low byte of an fp16 number it IS u 2^-24,
// a subnormal number, which the tensor core takes as it stands - no arithmetic at all.  The 128 leaves inside the products:
// the score's accumulator starts at -128 sum(q_i) instead of 0, and -128 times the weights are added to O by a product with a
// constant tile, half by half, so that sums over a long context are not buried under it (128 sum|x| 2^-23 at most, less than
// summing as many products in 32 bits may cost anyway).  2^24 goes into the scale of the scores and the last division.
// (As 1024 + u with the offset taken off by 32 additions a half instead, the 256-sequence batch took 82.9 us instead of 81.7.)
constexpr float kCodeUnit = 16777216.f;             // 2^24
constexpr float kCodeOffset = 128.f / 16777216.f;
constexpr uint32_t kMinusOffset2 = 0x80808080u;     // two fp16 numbers -128 2^-24

// Codes (0, 2) and (1, 3) of a word: for K two dims each, whose order inside the k axis is the query's too; for V two tokens
// of one dim, then of the next.  `c`: 0x00ff00ff and 0x00800080 in registers, so that (w & c.x) ^ c.y is one instruction (an
// instruction has room for one constant, and the compiler makes two of it).
template <int CODE>
__device__ __forceinline__ void widen_k(uint32_t w, uint2 c, uint32_t &even, uint32_t &odd) {
    if (CODE == MKV_Q8_INT8) {
        asm("lop3.b32 %0, %1, %2, %3, 0x6a;\n" : "=r"(even) : "r"(w), "r"(c.x), "r"(c.y));
        odd = __byte_perm(w, 0u, 0x4341) ^ c.y;
    } else {
        e4m3x4_to_half2(w, even, odd);      // (0, 1) and (2, 3): K's dims as they stand
    }
}
template <int CODE>
__device__ __forceinline__ void widen_v(uint32_t w, uint2 c, uint32_t &even, uint32_t &odd) {
    if (CODE == MKV_Q8_INT8) widen_k<CODE>(w, c, even, odd);
    else e4m3x4_to_half2(__byte_perm(w, 0u, 0x3120), even, odd);
}

template <typename T>
__device__ __forceinline__ void store2(T *dst, float a, float b) {
    struct alignas(2 * sizeof(T)) Two { T x[2]; } v;
    v.x[0] = rounded<T>(a); v.x[1] = rounded<T>(b);
    *reinterpret_cast<Two *>(dst) = v;
}
template <typename T>
__device__ __forceinline__ void store4(T *dst, float a, float b, float c, float d) {
    struct alignas(8) Four { T x[4]; } v;
    v.x[0] = rounded<T>(a); v.x[1] = rounded<T>(b); v.x[2] = rounded<T>(c); v.x[3] = rounded<T>(d);
    *reinterpret_cast<Four *>(dst) = v;
}

struct AttnQ8Params {       // what every launch reads stands together in front: constant memory is cold at a launch's start
    const int32_t *seq_ids, *seq_lens, *block_table;
    int64_t table_cols;
    int batch, num_rows, max_len;           // max_len: tokens that a row of the table can hold
    int num_q_heads, num_kv_heads, group, groups;  // groups: units of up to HC query heads for each kv head
    int cur_layer, half_shift;              // halves (16 tokens) of a block: 1 << half_shift
    int num_segments;
    uint32_t total_blocks, tile_bytes, block_tiles;  // block_tiles: layers * kv heads
    float scale_log2;
    const uint8_t *k0, *v0;                 // segment 0
    const float *ks0, *vs0;
    const void *q;
    int64_t q_stride;
    void *o;
    float *head_rows, *block_rows;          // [worker] and [2 * block] rows of HC * D values + HC log-sums
    int *error_flags, *arrive;
    PoolViewQ8 pool;                        // (the elastic segments)
};

struct Piece {      // a (sequence, head) that a warp has some tiles of
    int b, hp;      // batch index; kv head * groups + head group
    int flags;      // 1 valid, 2 has the first tile, 4 has the last tile, 8 parked in the ring (else in the warp's row)
    int nt;         // tiles of the whole (sequence, head)
    int p0;         // where its first real tile stands in the launch's order
};

// `total` positions in n contiguous shares, whose sizes differ by one at most.
struct Shares {
    int n, size, more;      // the first `more` shares have size + 1
    __device__ __forceinline__ Shares(int total, int n_) : n(n_), size(total / n_), more(total - size * n_) {}
    __device__ __forceinline__ int start(int i) const { return i * size + min(i, more); }
    __device__ __forceinline__ int owner(int x) const {
        const int big = more * (size + 1);
        return x < big ? x / (size + 1) : more + (x - big) / max(size, 1);
    }
};

template <typename T, int CODE, int D, int NT, bool DUP, int WARPS, int STAGES, int BLOCKS>
__global__ void __launch_bounds__(WARPS * 32, BLOCKS) attn_q8_kernel(const __grid_constant__ AttnQ8Params p) {
    constexpr int HC = DUP ? 4 : 8 * NT;        // query heads of a unit
    constexpr int HB = kHalf * D;               // bytes of K (or V) of a half
    constexpr int META = 4 * HB;                // scales (K, K, V, V) | flags and tokens, tile, -, - | b, hp, tiles, positions left
    constexpr int STAGE = META + 48;            // K, K, V, V, and those
    constexpr int KW = D / 16;                  // words of K a thread takes from a token's row = k-steps
    constexpr int MT = D / 16;                  // row tiles of O^T
    constexpr int ROW = HC * D + HC;            // floats of a partial row
    constexpr bool kScaledQ = !std::is_same<T, __half>::value;
    static_assert(STAGES * STAGE >= ROW * 4, "a piece is parked in its warp's ring");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ Piece first_piece[WARPS], last_piece[WARPS];
    __shared__ int scan_w[WARPS];
    __shared__ int seq_from[WARPS * 32], seq_len[WARPS * 32], seq_row[WARPS * 32];
    __shared__ int cross_valid[2], cross_f[2], cross_n[2], cross_b[2], cross_hp[2], cross_last[2];

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int P = p.num_kv_heads * p.groups;
    uint8_t *ring_ptr = smem + warp * (STAGES * STAGE);
    const uint32_t ring = smem_addr(ring_ptr);

    // ---- this block's range ---------------------------------------------------------------------------------
    auto tiles_of = [&](int len) { return len <= 0 ? 0 : (int)(((unsigned)min(len, p.max_len) + kTile - 1) / kTile); };
    // Thread i counts the positions of sequences [i per, (i + 1) per).
    const int per = (p.batch + WARPS * 32 - 1) / (WARPS * 32);
    int mine = 0, my_len = 0, my_row = 0;
    for (int i = 0; i < per; ++i) {
        const int b = tid * per + i;
        if (b < p.batch) {
            my_len = __ldg(p.seq_lens + b);
            my_row = __ldg(p.seq_ids + b);      // (used if there is one sequence a thread: fetched along with the length)
            const int nt = tiles_of(my_len);
            if (nt > 0) mine += nt + kUnitCost;
        }
    }
    mine *= P;
    int incl = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int n = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += n;
    }
    if (lane == 31) scan_w[warp] = incl;
    if (lane == 0) first_piece[warp].flags = last_piece[warp].flags = 0;
    if (tid < 2) cross_valid[tid] = cross_last[tid] = 0;
    __syncthreads();
    int total = 0, before = 0;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
        if (w < warp) before += scan_w[w];
        total += scan_w[w];
    }
    seq_from[tid] = before + incl - mine;
    seq_len[tid] = my_len;
    seq_row[tid] = my_row;
    __syncthreads();
    // A position at least for each warp of a block, so that a piece that enters a block is its first warp's.
    const Shares blocks(total, max(min((int)gridDim.x, total / WARPS), 1));
    const int cta = blockIdx.x;
    if (total == 0 || cta >= blocks.n) return;
    const int lo = blocks.start(cta), hi = blocks.start(cta + 1);
    const Shares warps(hi - lo, WARPS);
    const int wlo = lo + warps.start(warp), whi = lo + warps.start(warp + 1);

    // ---- where the warp reads next: the same in every lane, the id windows apart -----------------------------------
    // crem: positions from the current (sequence, head)'s first real tile to the end of the warp's range, whose part of it
    // therefore ends at min(cnt, crem).
    const int half_mask = (1 << p.half_shift) - 1;
    bool bad = false, more = false;
    int cb = 0, chp = 0, ch = 0, chg = 0, cnt = 0, cj = 0, cjend = 0, clen = 0, crow = 0, cbase = 0, crem = 0;
    int first_flag = 1;
    uint32_t uhead = 0;             // the unit's (layer, head) inside a block ...
    uint64_t ubase = 0;             // ... and where this lane's first piece of it stands in the block's codes
    int2 ids, ids_next;             // lane l: block ids of tile cbase + l's halves, and of the 32 tiles behind those
    int2 ids0_next = make_int2(-1, -1);  // ... of the first 32 tiles of the next sequence (nb; its row and length)
    int nb = -2, nrow = 0, nlen = 0;    // -1: there is none, -2: not looked for yet
    auto load_ids = [&](int row, int first, int nt) {
        const int tile = first + lane;
        int2 x = make_int2(-1, -1);
        if (row >= 0 && row < p.num_rows && tile < nt) {
            const int32_t *at = p.block_table + (int64_t)row * p.table_cols;
            const int a = (2 * tile) >> p.half_shift, b = (2 * tile + 1) >> p.half_shift;
            x.x = __ldg(at + a);
            if (b < p.table_cols) x.y = __ldg(at + b);
        }
        return x;
    };
    auto look_ahead = [&]() {   // the first sequence behind cb that has tokens
        nb = -1;
        for (int at = cb + 1; at < p.batch; at += 32) {
            const int len = at + lane < p.batch ? __ldg(p.seq_lens + at + lane) : 0;
            const unsigned some = __ballot_sync(0xffffffffu, len > 0);
            if (some) {
                nb = at + __ffs(some) - 1;
                nlen = __shfl_sync(0xffffffffu, len, __ffs(some) - 1);
                nrow = __ldg(p.seq_ids + nb);
                ids0_next = load_ids(nrow, 0, tiles_of(nlen));
                return;
            }
        }
    };
    auto enter_sequence = [&]() {
        cnt = tiles_of(clen);
        bad |= crow < 0 || crow >= p.num_rows || clen > p.max_len;
        clen = min(clen, p.max_len);
    };
    auto enter_head = [&]() {
        uhead = (uint32_t)(p.cur_layer * p.num_kv_heads + ch);
        ubase = (uint64_t)uhead * p.tile_bytes + (uint32_t)lane * 16;
        cjend = min(cnt, crem);
        more = cj < cjend;
        cbase = cj;
        first_flag = 1;
        if (more) ids_next = load_ids(crow, cj + 32, cnt);
    };
    if (wlo < whi) {
        // the last thread whose first position is not behind wlo holds it (one without positions shares its successor's)
        int seg = 0;
#pragma unroll
        for (int w = 1; w < WARPS; ++w)
            if (seq_from[w * 32] <= wlo) seg = w;
        const int i = seg * 32 + 31 - __clz(__ballot_sync(0xffffffffu, seq_from[seg * 32 + lane] <= wlo));
        int at = seq_from[i];
        cb = i * per;
        clen = seq_len[i];
        crow = seq_row[i];
        if (per > 1) {      // ... in one of its sequences
            for (;; ++cb) {
                clen = __ldg(p.seq_lens + cb);
                const int nt = tiles_of(clen), c = nt > 0 ? (nt + kUnitCost) * P : 0;
                if (wlo < at + c || cb + 1 >= min((i + 1) * per, p.batch)) break;
                at += c;
            }
            crow = __ldg(p.seq_ids + cb);
        }
        enter_sequence();
        const unsigned w = cnt + kUnitCost, rem = wlo - at;
        chp = min((int)(rem / w), P - 1);
        const int inside = (int)(rem - chp * w);
        cj = max(inside - kUnitCost, 0);
        crem = whi - wlo + inside - kUnitCost;
        ch = chp / p.groups;
        chg = chp - ch * p.groups;
        ids = load_ids(crow, cj, cnt);
        enter_head();
    }
    const uint32_t block_bytes = p.tile_bytes * p.block_tiles;
    // The codes are read once: they are not to push anything else out of L2 (64 sequences of up to 768, 32 heads: 52.2 -> 49.5 us;
    // long contexts 70 -> 68).  (volatile: made once, not at every copy, which cost the 256-sequence batch 2 us.)
    uint64_t policy;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;\n" : "=l"(policy));
    // 16-byte piece i * 32 + lane of a half.  D = 128: piece c of token r goes to c ^ (r & 7); D = 64: two tokens share a
    // 128-byte line, whose pieces go to c ^ (line & 3).  Either way the reads below meet no conflict.
    const uint32_t put = (uint32_t)((lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4));
    auto issue_half = [&](uint32_t st, int h, uint32_t blk, int &tokens) {
        if (tokens > 0 && blk < p.total_blocks) {
            uint32_t row = blk;
            const uint8_t *k0 = p.k0, *v0 = p.v0;
            const float *s0 = lane ? p.vs0 : p.ks0;
            if (p.num_segments > 1) {
                int seg;
                int64_t r;
                locate_block(p.pool, blk, seg, r);
                row = (uint32_t)r;
                k0 = p.pool.k_base[seg];
                v0 = p.pool.v_base[seg];
                s0 = lane ? p.pool.v_scale[seg] : p.pool.k_scale[seg];
            }
            const uint64_t off = (uint64_t)row * block_bytes + ubase + (uint32_t)(((2 * cj + h) & half_mask) * HB);
            const uint8_t *kt = k0 + off, *vt = v0 + off;
#pragma unroll
            for (int i = 0; i < HB / 512; ++i) {
                const uint32_t to = st + h * HB + i * 512 + (D == 128 && (i & 1) ? put ^ 64 : put);
                cp16(to, kt + i * 512, policy);
                cp16(to + 2 * HB, vt + i * 512, policy);
            }
            if (lane < 2)
                cp4(st + META + (lane * 2 + h) * 4, s0 + ((uint64_t)row * p.block_tiles + uhead));
        } else {
            bad |= tokens > 0;
            tokens = 0;
            if (lane < 2) asm volatile("st.shared.b32 [%0], %1;\n" ::"r"(st + META + (lane * 2 + h) * 4), "r"(0x3f800000) : "memory");
        }
    };
    // One tile into ring stage `st`, and the cursor moves on.
    auto issue = [&](uint32_t st) {
        if (!more) return;
        if (cj - cbase == 32) {
            ids = ids_next;
            cbase = cj;
            ids_next = load_ids(crow, cbase + 32, cnt);
        }
        const uint32_t blk0 = (uint32_t)__shfl_sync(0xffffffffu, ids.x, cj - cbase);
        const uint32_t blk1 = (uint32_t)__shfl_sync(0xffffffffu, ids.y, cj - cbase);
        const int left = clen - cj * kTile;
        int n0 = min(left, kHalf), n1 = min(max(left - kHalf, 0), kHalf);
        if (n1 > 0 && max(blk0, blk1) < p.total_blocks && p.num_segments == 1) {    // both halves, as nearly always
            const uint32_t sub0 = (uint32_t)((2 * cj & half_mask) * HB), sub1 = (uint32_t)(((2 * cj + 1) & half_mask) * HB);
            const uint64_t off0 = (uint64_t)blk0 * block_bytes + sub0 + ubase, off1 = (uint64_t)blk1 * block_bytes + sub1 + ubase;
            const uint8_t *k0 = p.k0 + off0, *v0 = p.v0 + off0, *k1 = p.k0 + off1, *v1 = p.v0 + off1;
#pragma unroll
            for (int i = 0; i < HB / 512; ++i) {
                const uint32_t to = st + i * 512 + (D == 128 && (i & 1) ? put ^ 64 : put);
                cp16(to, k0 + i * 512, policy);
                cp16(to + HB, k1 + i * 512, policy);
                cp16(to + 2 * HB, v0 + i * 512, policy);
                cp16(to + 3 * HB, v1 + i * 512, policy);
            }
            if (lane < 4)
                cp4(st + META + lane * 4, (lane & 2 ? p.vs0 : p.ks0) + ((uint64_t)(lane & 1 ? blk1 : blk0) * p.block_tiles + uhead));
        } else {
            issue_half(st, 0, blk0, n0);
            issue_half(st, 1, blk1, n1);
        }
        if (first_flag) {       // the unit's query rows on their way into the cache
            const int hq0 = ch * p.group + chg * HC, bytes = min(HC, p.group - chg * HC) * D * 2;
            if (lane * 128 < bytes)
                asm volatile("prefetch.global.L1 [%0];\n" ::"l"((const char *)((const T *)p.q + cb * p.q_stride + (int64_t)hq0 * D) + lane * 128));
        }
        int flags = first_flag;
        first_flag = 0;
        const int tile = cj++;
        const int b = cb, hp = chp, nt = cnt, end = crem;
        if (cj == cjend) {      // the next (sequence, head)
            flags |= 2;
            crem -= cnt + kUnitCost;
            if (crem <= 0) {
                more = false;
            } else if (++chp == P) {
                more = false;
                if (nb == -2) look_ahead();
                if (nb >= 0) {
                    cb = nb;
                    crow = nrow;
                    clen = nlen;
                    ids = ids0_next;
                    chp = ch = chg = cj = 0;
                    nb = -2;
                    enter_sequence();
                    enter_head();
                }
            } else {
                if (++chg == p.groups) {
                    chg = 0;
                    ++ch;
                }
                cj = 0;
                ids = load_ids(crow, 0, cnt);   // the row was read for the head before: an L1 hit
                enter_head();
            }
            if (!more) flags |= 4;
        }
        if (lane == 0) {
            sts16(st + META + 16, flags | (n0 << 8) | (n1 << 16), tile, 0, 0);
            if (flags & 3) sts16(st + META + 32, b, hp, nt, end);
        }
    };

    float o[NT][MT][4];
    uint32_t qf[NT][KW][2];
    float qfac[NT][2];      // scale_log2 and what undoes the normalisation of a bf16 q, for heads 2t and 2t + 1
    float kinit[NT][2];     // what takes the offset of int8 codes out of the scores
    float thr[NT][2], base[NT][2], l[NT][2], ref[NT][2];
    constexpr bool kRest = !DUP;    // what fp16 leaves over of the weights goes through products of its own
    float rest_off[NT][4];          // int8: -128 times the sum of those, which all dims share, until the piece ends
    bool piece_starts = false;
    // byte offsets inside a half: K pieces of tokens g and g + 8; V rows and pieces for ldmatrix
    const uint32_t k_at = D == 128 ? g * 128 + (((2 * t) ^ g) << 4) : (g >> 1) * 128 + ((((g & 1) * 4 + t) ^ (g >> 1)) << 4);
    const int vr = (lane & 7) + ((lane >> 3) & 1) * 8, vh = lane >> 4;
    const uint32_t v_at = 2 * HB + (D == 128 ? vr * 128 + ((vh ^ (vr & 7)) << 4)
                                             : (vr >> 1) * 128 + ((((vr & 1) * 4 + vh) ^ ((vr >> 1) & 3)) << 4));

    uint2 masks;
    asm volatile("mov.b32 %0, 0x00ff00ff;\nmov.b32 %1, 0x00800080;\n" : "=r"(masks.x), "=r"(masks.y));

    bool busy = more;
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) {
        issue(ring + i * STAGE);
        cp_commit();
    }
    uint32_t st = ring, refill = ring + (STAGES - 1) * STAGE;
    while (busy) {
        cp_wait<STAGES - 2>();
        __syncwarp();       // every lane's part of the tile has landed, and the stage before it is read
        issue(refill);
        cp_commit();
        if (more && nb == -2) look_ahead();     // early, so that the next sequence's ids are there when it comes
        const uint4 scales = lds16(st + META), ma = lds16(st + META + 16);
        const int flags = (int)(ma.x & 0xffu);
        busy = !(flags & 4);

        if (flags & 1) {    // first tile of a piece
            piece_starts = ma.y == 0;
            const uint4 mb = lds16(st + META + 32);
            const int kvh = (int)mb.y / p.groups, hq0 = kvh * p.group + ((int)mb.y - kvh * p.groups) * HC;
            const int heads = min(HC, (kvh + 1) * p.group - hq0);
            const T *qb = (const T *)p.q + (int)mb.x * p.q_stride + (int64_t)hq0 * D + t * (D / 4);
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
                if (kScaledQ) {
                    // bf16: a power of two brings the head's largest element to [2^14, 2^15); then fp16 holds every element
                    // down to 2^-28 of it exactly
                    uint32_t peak = 0;
#pragma unroll
                    for (int i = 0; i < KW * 2; ++i) peak = max(peak, max(raw[i] & 0x7fffu, (raw[i] >> 16) & 0x7fffu));
                    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 1));
                    peak = max(peak, __shfl_xor_sync(0xffffffffu, peak, 2));
                    const int e = peak == 0 ? 0 : min(max(14 + 127 - (int)(peak >> 7), -120), 120);
                    const float up = __uint_as_float((uint32_t)(127 + e) << 23);
                    const float fac = p.scale_log2 * __uint_as_float((uint32_t)(127 - e) << 23);
#pragma unroll
                    for (int i = 0; i < KW * 2; ++i)
                        raw[i] = half2_bits(__floats2half2_rn(__uint_as_float(raw[i] << 16) * up, __uint_as_float(raw[i] & 0xffff0000u) * up));
                    // columns 2t and 2t + 1 belong to the lanes with g = 2t and 2t + 1
                    qfac[n][0] = __shfl_sync(0xffffffffu, fac, 8 * t);
                    qfac[n][1] = __shfl_sync(0xffffffffu, fac, 8 * t + 4);
                }
                if (CODE == MKV_Q8_INT8) {
                    float sum = 0.f;
#pragma unroll
                    for (int i = 0; i < KW * 2; ++i) {
                        const float2 f = __half22float2(bits_half2(raw[i]));
                        sum += f.x + f.y;
                    }
                    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
                    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
                    kinit[n][0] = -kCodeOffset * __shfl_sync(0xffffffffu, sum, 8 * t);
                    kinit[n][1] = -kCodeOffset * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
                }
#pragma unroll
                for (int i = 0; i < KW; ++i) {
                    // dims 4 i ... 4 i + 3 in the order in which widen_k() has them
                    qf[n][i][0] = CODE == MKV_Q8_INT8 ? __byte_perm(raw[2 * i], raw[2 * i + 1], 0x5410) : raw[2 * i];
                    qf[n][i][1] = CODE == MKV_Q8_INT8 ? __byte_perm(raw[2 * i], raw[2 * i + 1], 0x7632) : raw[2 * i + 1];
                }
#pragma unroll
                for (int i = 0; i < MT; ++i) o[n][i][0] = o[n][i][1] = o[n][i][2] = o[n][i][3] = 0.f;
                rest_off[n][0] = rest_off[n][1] = rest_off[n][2] = rest_off[n][3] = 0.f;
                thr[n][0] = thr[n][1] = -INFINITY;
                base[n][0] = base[n][1] = l[n][0] = l[n][1] = 0.f;
                ref[n][0] = ref[n][1] = INFINITY;
            }
        }

        // One half after the other in one body: unrolled, the two would overlap, but the code a block has to fetch before its
        // first result would be twice as long.
#pragma unroll 1
        for (int h = 0; h < 2; ++h) {
            const uint32_t at = st + h * HB;
            const int tokens = (int)((ma.x >> (8 + 8 * h)) & 0xffu);
            const float ks = __uint_as_float(h ? scales.y : scales.x), vs = __uint_as_float(h ? scales.w : scales.z);
            // ---- S^T = K Q^T
            float sc[NT][4];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[n][e] = CODE == MKV_Q8_INT8 ? kinit[n][e & 1] : 0.f;
#pragma unroll
            for (int i = 0; i < KW / 4; ++i) {
                const uint4 x = lds16(at + (k_at ^ (i << 4))), y = lds16(at + (k_at ^ (i << 4)) + HB / 2);  // tokens g and g + 8
                const uint32_t xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t a0, a1, a2, a3;
                    widen_k<CODE>(xs[j], masks, a0, a2);
                    widen_k<CODE>(ys[j], masks, a1, a3);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma(sc[n], a0, a1, a2, a3, qf[n][4 * i + j][0], qf[n][4 * i + j][1]);
                }
            }
            // ---- softmax: token g (elements 0, 1) and g + 8 (2, 3), heads 2t, 2t + 1
            // The block's V scale joins the exponent: weights are w = 2^(score + log2 s_v - base), so that O accumulates across
            // blocks as the tensor core leaves it.  The denominator l takes 2^ref / s_v of them, that is 2^(score - (base - ref)):
            // ref is log2 s_v of the half that moved base last, or less, so that base - ref, about that half's largest score, never
            // falls and l never grows when base moves.  So all scales that fp32 holds are equally good.  Where s_v is below 2^ref
            // by more than 2^90 (an all-zero block's, above all) w may be nothing although l needs it: then l takes the scores.
            float lv;
            asm("lg2.approx.f32 %0, %1;\n" : "=f"(lv) : "f"(vs));
            const bool on0 = g < tokens, on1 = g + 8 < tokens;
            bool above = false, apart[NT][2];      // apart: l has this half's weights already
            float x[NT][4], fs[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                apart[n][0] = apart[n][1] = false;
                // (a factor too large for 32 bits: 0 times it is 0 all the same)
                constexpr float kUnit = CODE == MKV_Q8_INT8 ? kCodeUnit : 1.f;
                fs[n][0] = min_nan((kScaledQ ? qfac[n][0] : p.scale_log2) * ks * kUnit, kLargest);
                fs[n][1] = kScaledQ ? min_nan(qfac[n][1] * ks * kUnit, kLargest) : fs[n][0];
                x[n][0] = on0 ? fmaf(sc[n][0], fs[n][0], lv) : -INFINITY;
                x[n][1] = on0 ? fmaf(sc[n][1], fs[n][1], lv) : -INFINITY;
                x[n][2] = on1 ? fmaf(sc[n][2], fs[n][0], lv) : -INFINITY;
                x[n][3] = on1 ? fmaf(sc[n][3], fs[n][1], lv) : -INFINITY;
                above |= fmaxf(x[n][0], x[n][2]) > thr[n][0] || fmaxf(x[n][1], x[n][3]) > thr[n][1];
                above |= lv + kFaint < ref[n][0] || lv + kFaint < ref[n][1];
            }
            if (__any_sync(0xffffffffu, above)) {   // the maxima settle after the first tiles of a piece
                bool faint = vs == 0.f;
                if (!faint) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            // a head moves by 2^4 at least, so that what its factors are off counts for tokens of small weight only
                            const float m = column_max(fmaxf(x[n][e], x[n][e + 2]));
                            const bool moves = m > thr[n][e];
                            const float by = moves ? base[n][e] - (m - kBoost) : 0.f;
                            const float a = thr[n][e] == -INFINITY ? 1.f : ex2(by);     // before: all weights were 0
                            if (moves) {
                                const float r = fminf(lv, ref[n][e] - by);
                                l[n][e] *= ex2(by + (r - ref[n][e]));
                                thr[n][e] = m + kLag;
                                base[n][e] = m - kBoost;
                                ref[n][e] = r;
                            }
#pragma unroll
                            for (int i = 0; i < MT; ++i) {
                                o[n][i][e] *= a;
                                o[n][i][e + 2] *= a;
                            }
                            rest_off[n][e] *= a;
                            rest_off[n][e + 2] *= a;
                            apart[n][e] = lv + kFaint < ref[n][e];
                            faint |= apart[n][e];
                        }
                }
                if (__any_sync(0xffffffffu, faint)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            const float s0 = on0 ? sc[n][e] * fs[n][e] : -INFINITY, s1 = on1 ? sc[n][e + 2] * fs[n][e] : -INFINITY;
                            const float m = column_max(fmaxf(s0, s1)), held = base[n][e] - ref[n][e];
                            const float to = m > held + kAhead ? m : held;
                            if ((apart[n][e] || vs == 0.f) && to > -INFINITY) {
                                l[n][e] = l[n][e] * ex2(held - to) + (ex2(s0 - to) + ex2(s1 - to));
                                ref[n][e] = base[n][e] - to;
                            }
                            if (isnan(s0 + s1)) l[n][e] = s0 + s1;
                        }
                    if (vs == 0.f) continue;    // (the same for the whole warp)
                }
            }
            uint32_t pb[NT][2], pr[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const float w0 = ex2(x[n][0] - base[n][0]), w1 = ex2(x[n][1] - base[n][1]);
                const float w2 = ex2(x[n][2] - base[n][0]), w3 = ex2(x[n][3] - base[n][1]);
                l[n][0] = fmaf(w0 + w2, apart[n][0] ? 0.f : ex2(ref[n][0] - lv), l[n][0]);
                l[n][1] = fmaf(w1 + w3, apart[n][1] ? 0.f : ex2(ref[n][1] - lv), l[n][1]);
                __half2 p0 = __floats2half2_rn(w0, w1), p1 = __floats2half2_rn(w2, w3);
                const float2 fx = __half22float2(p0), fy = __half22float2(p1);
                const __half2 rx = __floats2half2_rn(w0 - fx.x, w1 - fx.y), ry = __floats2half2_rn(w2 - fy.x, w3 - fy.y);
                if (DUP) {  // columns 4-7: what the rounding of columns 0-3 left over
                    p0 = t >= 2 ? rx : p0;
                    p1 = t >= 2 ? ry : p1;
                } else {    // ... of all columns: a second B operand
                    pr[n][0] = transpose8x8(half2_bits(rx));
                    pr[n][1] = transpose8x8(half2_bits(ry));
                }
                pb[n][0] = transpose8x8(half2_bits(p0));
                pb[n][1] = transpose8x8(half2_bits(p1));
            }
            // ---- O^T += V^T P^T: row tile c has dim 16 c + 2 g in its row g and dim 16 c + 2 g + 1 in its row g + 8
            // Behind the sequence's end any byte may stand, an e4m3 NaN among them, and 0 x NaN is NaN.
            const bool cut = CODE == MKV_Q8_E4M3 && tokens < kHalf;
            if (CODE == MKV_Q8_INT8) {
#pragma unroll
                for (int c = 0; c < MT; ++c)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma(o[n][c], kMinusOffset2, kMinusOffset2, kMinusOffset2, kMinusOffset2, pb[n][0], pb[n][1]);
                if (kRest) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
                        mma(rest_off[n], kMinusOffset2, kMinusOffset2, kMinusOffset2, kMinusOffset2, pr[n][0], pr[n][1]);
                }
            }
#pragma unroll
            for (int c = 0; c < MT; c += 2) {
                uint32_t w[4];      // (16-dim piece c: tokens 0-7, 8-15; piece c + 1: the same)
                ldsm4_trans(w, at + (v_at ^ (c << 4)));
                if (cut) {
                    const int n = tokens - 2 * t;
                    const uint32_t lo = n >= 2 ? 0xffffffffu : n == 1 ? 0xffffu : 0u, hi = n >= 10 ? 0xffffffffu : n == 9 ? 0xffffu : 0u;
                    w[0] &= lo; w[1] &= hi; w[2] &= lo; w[3] &= hi;
                }
                uint32_t a[2][4];
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    widen_v<CODE>(w[2 * d], masks, a[d][0], a[d][1]);
                    widen_v<CODE>(w[2 * d + 1], masks, a[d][2], a[d][3]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma(o[n][c + d], a[d][0], a[d][1], a[d][2], a[d][3], pb[n][0], pb[n][1]);
                }
                if (kRest) {
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int n = 0; n < NT; ++n) mma(o[n][c + d], a[d][0], a[d][1], a[d][2], a[d][3], pr[n][0], pr[n][1]);
                }
            }
        }

        if (flags & 2) {    // last tile of the piece
            const uint4 mb = lds16(st + META + 32);
            const int b = (int)mb.x, kvh = (int)mb.y / p.groups, hq0 = kvh * p.group + ((int)mb.y - kvh * p.groups) * HC;
            const int heads = min(HC, (kvh + 1) * p.group - hq0);
            const bool ends = ma.y + 1 == mb.z, whole = piece_starts && ends;
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
                if (kRest && CODE == MKV_Q8_INT8) {
#pragma unroll
                    for (int i = 0; i < MT; ++i)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[n][i][e] += rest_off[n][e];
                }
            }
            float *row = nullptr;
            if (!whole) {
                // (a piece that is neither the first nor the last of its warp is whole)
                Piece &pc = !busy && first_piece[warp].flags ? last_piece[warp] : first_piece[warp];
                row = busy ? p.head_rows + ((int64_t)cta * WARPS + warp) * ROW : reinterpret_cast<float *>(ring_ptr);
                __syncwarp();
                if (lane == 0) {
                    pc.b = b;
                    pc.hp = (int)mb.y;
                    pc.nt = (int)mb.z;
                    pc.flags = 1 | (piece_starts ? 2 : 0) | (ends ? 4 : 0) | (busy ? 0 : 8);
                    pc.p0 = whi - (int)mb.w;
                }
                __syncwarp();
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int head = n * 8 + 2 * t + e;
                    if (head >= heads || head >= HC) continue;
                    // 2^ref in two factors: as one it may be too small for fp32 where the output is not.  (Where no value has had
                    // a weight ref is no scale's, and the output 0: it has to be finite.)
                    const float up = ex2(0.5f * fminf(ref[n][e], 126.f)), unit = (CODE == MKV_Q8_INT8 ? kCodeUnit : 1.f) * up;
                    if (whole) {
                        const float f = unit / l[n][e];
                        T *dst = (T *)p.o + ((int64_t)b * p.num_q_heads + hq0 + head) * D + 2 * g;
#pragma unroll
                        for (int i = 0; i < MT; ++i) store2<T>(dst + 16 * i, o[n][i][e] * f * up, o[n][i][e + 2] * f * up);
                    } else {
                        const float f = l[n][e] == 0.f ? 0.f : unit / l[n][e];
                        float *dst = row + head * D + 2 * g;
#pragma unroll
                        for (int i = 0; i < MT; ++i)
                            *reinterpret_cast<float2 *>(dst + 16 * i) = make_float2(o[n][i][e] * f * up, o[n][i][e + 2] * f * up);
                        if (g == 0) row[HC * D + head] = l[n][e] == 0.f ? -INFINITY : log2f(l[n][e]) + (base[n][e] - ref[n][e]);
                    }
                }
        }
        refill = st;
        st = st == ring + (STAGES - 1) * STAGE ? ring : st + STAGE;
    }
    cp_wait<0>();
    if (bad && lane == 0 && p.error_flags) atomicOr(p.error_flags, 1);

    // ---- pieces of cut (sequence, head)s: those of this block's warps are folded, four query heads by one warp -----------
    __syncthreads();
    // Lane c: is the first (c even) or last (odd) piece of warp c / 2 the block's first one of its (sequence, head)?  Its
    // others are the first pieces of the warps behind it, up to the one that ends.
    unsigned leaders, held, ending;
    {
        const int fl = lane < 2 * WARPS ? ((lane & 1) ? last_piece[lane >> 1] : first_piece[lane >> 1]).flags : 0;
        leaders = __ballot_sync(0xffffffffu, fl != 0 && ((fl & 2) != 0 || lane == 0));
        const int ff = lane < WARPS ? first_piece[lane].flags : 0;
        held = __ballot_sync(0xffffffffu, ff != 0);
        ending = __ballot_sync(0xffffffffu, (ff & 4) != 0);
    }
    constexpr int QUADS = (HC + 3) / 4;
    const unsigned all_leaders = leaders;
    int item = 0;
#pragma unroll 1
    for (; leaders; leaders &= leaders - 1) {
        const int c = __ffs(leaders) - 1, x0 = c >> 1;
#pragma unroll 1
        for (int quad = 0; quad < QUADS; ++quad) {
            if (item++ % WARPS != warp) continue;
            const Piece lead = (c & 1) ? last_piece[x0] : first_piece[x0];
            const int kvh = lead.hp / p.groups, hq0 = kvh * p.group + (lead.hp - kvh * p.groups) * HC;
            const int heads = min(HC, (kvh + 1) * p.group - hq0) - quad * 4;
            if (heads <= 0) continue;
            unsigned behind = 0;        // warps that hold the further pieces
            bool ends = lead.flags & 4;
            if (!ends) {
                behind = held & ~((2u << x0) - 1);
                const unsigned e = behind & ending;
                ends = e != 0;
                if (ends) behind &= (e & (0u - e)) * 2 - 1;
            }
            float m[4], sum[4];
            float4 acc[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                m[r] = -INFINITY;
                sum[r] = 0.f;
                acc[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            int x[2] = {x0, 0}, fl[2] = {lead.flags, 0};
            int n = 1;
            for (;;) {
                if (n == 1 && behind) {     // two pieces at a time: all loads before the first use
                    x[1] = __ffs(behind) - 1;
                    behind &= behind - 1;
                    fl[1] = first_piece[x[1]].flags;
                    n = 2;
                }
                float ls[2][4];
                float4 v[2][4];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float *row = (fl[i] & 8) ? reinterpret_cast<const float *>(smem + x[i] * (STAGES * STAGE))
                                                   : p.head_rows + ((int64_t)cta * WARPS + x[i]) * ROW;
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int head = quad * 4 + min(r, heads - 1);
                        ls[i][r] = -INFINITY;
                        v[i][r] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (i < n) {
                            ls[i][r] = row[HC * D + head];
                            if (lane * 4 < D) v[i][r] = *reinterpret_cast<const float4 *>(row + head * D + lane * 4);
                        }
                    }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float nm = fmaxf(m[r], fmaxf(ls[0][r], ls[1][r])), off = nm == -INFINITY ? 0.f : nm;
                    const float a = exp2f(m[r] - off), e0 = exp2f(ls[0][r] - off), e1 = exp2f(ls[1][r] - off);
                    acc[r].x = acc[r].x * a + v[0][r].x * e0 + v[1][r].x * e1;
                    acc[r].y = acc[r].y * a + v[0][r].y * e0 + v[1][r].y * e1;
                    acc[r].z = acc[r].z * a + v[0][r].z * e0 + v[1][r].z * e1;
                    acc[r].w = acc[r].w * a + v[0][r].w * e0 + v[1][r].w * e1;
                    sum[r] = sum[r] * a + e0 + e1;
                    m[r] = nm;
                }
                if (!behind) break;
                x[0] = __ffs(behind) - 1;
                behind &= behind - 1;
                fl[0] = first_piece[x[0]].flags;
                n = 1;
            }
            const bool whole = (lead.flags & 2) && ends;    // all of it lies in this block
            // row 0 of the block: of a (sequence, head) that comes from the block before it; row 1: of one that starts here
            const int s = (lead.flags & 2) ? 1 : 0;
            float *row = p.block_rows + ((int64_t)cta * 2 + s) * ROW;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (r >= heads) break;
                const int head = quad * 4 + r;
                const float f = !whole && sum[r] == 0.f ? 0.f : 1.f / sum[r];
                if (whole) {
                    if (lane * 4 < D)
                        store4<T>((T *)p.o + ((int64_t)lead.b * p.num_q_heads + hq0 + head) * D + lane * 4, acc[r].x * f, acc[r].y * f,
                                  acc[r].z * f, acc[r].w * f);
                } else {
                    if (lane * 4 < D)
                        __stcg(reinterpret_cast<float4 *>(row + head * D + lane * 4),
                               make_float4(acc[r].x * f, acc[r].y * f, acc[r].z * f, acc[r].w * f));
                    if (lane == 0) __stcg(row + HC * D + head, log2f(sum[r]) + (m[r] == -INFINITY ? 0.f : m[r]));
                }
            }
            if (!whole && quad == 0 && lane == 0) {
                cross_f[s] = blocks.owner(lead.p0);
                cross_n[s] = blocks.owner(lead.p0 + lead.nt - 1) - cross_f[s] + 1;
                cross_b[s] = lead.b;
                cross_hp[s] = lead.hp;
                cross_valid[s] = 1;
            }
        }
    }
    if (!all_leaders) return;       // (the same for every thread of the block)
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
// Warps of a block; the second with 16 query heads a unit, whose accumulators take more registers.  12 warps with two stages each
// against 8 with three (the same 192 KiB in flight): 87 and 93 us for 256 sequences, where more warps hide the conversion's
// latency; the other batches are within 1 %.
constexpr int kWarps = 12, kWarpsWide = 8;
constexpr int kBlocksPerSm = 1;
constexpr size_t kErrorBytes = 256;     // error word, then the arrival counters

static size_t zero_bytes(int sms) { return kErrorBytes + (((size_t)sms * kBlocksPerSm * sizeof(int) + 255) & ~(size_t)255); }
// Query heads of a unit: 4, 8 or 16.  The weights enter the second product as an fp16 number and what that leaves over, also
// fp16 (2^-22 of the weight together).  With 4 heads the remainders are columns 4-7 of the tile and cost nothing; with 8 and 16
// they are a second B operand, twice the products of V: without and with them (and what every scale of V takes), long contexts in
// groups of 8 take 68-71 and 69-74 us (e4m3), 66 and 76 us (int8), 256 sequences in groups of 8 48 and 54 us, of 16 65 and 72 us.
// Without them an output is off by 1.4e-4 of the weighted values' size, which shows beside fp16's own rounding and is far above
// it where values cancel.
static int unit_heads(int group) { return group <= 4 ? 4 : group <= 8 ? 8 : 16; }

static bool fast_shape(const PoolViewQ8 &pv) {
    const int bs = pv.block_size;
    return (pv.head_dim == 64 || pv.head_dim == 128) && bs >= kHalf && (bs & (bs - 1)) == 0 &&
           pv.tile_bytes * pv.num_layers * pv.num_kv_heads < (1ll << 32) && pv.total_blocks < (1ll << 31);
}
// Positions of a launch whose sequences fill the table's rows stay below 2^30 (they are counted in 32 bits).
static bool fast_positions(const PoolViewQ8 &pv, int batch, int group, int64_t cols) {
    const int64_t tokens = std::min<int64_t>(cols * pv.block_size, 0x7fffffff);
    const double per = (double)(ceil_div64(tokens, kTile) + kUnitCost) * pv.num_kv_heads * ((group + 3) / 4);
    return per * batch < (double)(1 << 30);
}
// 16-byte loads of q and of the pool, 8-byte stores of o.
static bool fast_aligned(const PoolViewQ8 &pv, const void *q, int64_t q_stride, const void *o) {
    uintptr_t bits = (uintptr_t)q | (uintptr_t)(q_stride * 2) | ((uintptr_t)o << 1);
    for (int i = 0; i < pv.num_segments; ++i) bits |= (uintptr_t)pv.k_base[i] | (uintptr_t)pv.v_base[i];
    return (bits & 15) == 0;
}

template <typename T, int CODE, int D, int NT, bool DUP, int STAGES>
static cudaError_t launch_fast(const AttnQ8Params &p, unsigned grid, cudaStream_t s) {
    constexpr int warps = NT == 2 ? kWarpsWide : kWarps;
    constexpr int smem = warps * STAGES * (4 * kHalf * D + 48);
    auto kernel = attn_q8_kernel<T, CODE, D, NT, DUP, warps, STAGES, kBlocksPerSm>;
    static std::atomic<bool> configured[64];    // per device; setting the attribute twice is harmless
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !configured[dev].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
        if (dev >= 0 && dev < 64) configured[dev].store(true, std::memory_order_release);
    }
    kernel<<<grid, warps * 32, smem, s>>>(p);
    return cudaGetLastError();
}

template <typename T, int CODE>
static cudaError_t launch_fast_shape(const AttnQ8Params &p, int head_dim, unsigned grid, cudaStream_t s) {
    const int heads = unit_heads(p.group);
    if (head_dim == 128)
        return heads == 4   ? launch_fast<T, CODE, 128, 1, true, 2>(p, grid, s)
               : heads == 8 ? launch_fast<T, CODE, 128, 1, false, 2>(p, grid, s)
                            : launch_fast<T, CODE, 128, 2, false, 3>(p, grid, s);
    return heads == 4   ? launch_fast<T, CODE, 64, 1, true, 4>(p, grid, s)
           : heads == 8 ? launch_fast<T, CODE, 64, 1, false, 4>(p, grid, s)
                        : launch_fast<T, CODE, 64, 2, false, 5>(p, grid, s);
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
    const size_t rows = (size_t)sms * kBlocksPerSm * (kWarps + 2);
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
    if (dtype != MKV_F32 && fast_shape(pv) && fast_aligned(pv, q, q_stride, o) &&
        fast_positions(pv, batch, group, table_stride)) {
        int sms = 0;
        if ((st = mkv_sm_count(device, &sms))) return st;
        if (!workspace || workspace_bytes < mkv_attn_q8_workspace_bytes(device, batch, num_q_heads, pv.num_kv_heads, pv.head_dim))
            return MKV_ERR_WORKSPACE;
        const int heads = unit_heads(group);
        AttnQ8Params p;
        p.pool = pv;
        p.num_kv_heads = pv.num_kv_heads;
        p.num_segments = pv.num_segments;
        p.total_blocks = (uint32_t)pv.total_blocks;
        p.tile_bytes = (uint32_t)pv.tile_bytes;
        p.block_tiles = (uint32_t)(pv.num_layers * pv.num_kv_heads);
        p.k0 = pv.k_base[0];
        p.v0 = pv.v_base[0];
        p.ks0 = pv.k_scale[0];
        p.vs0 = pv.v_scale[0];
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
        p.half_shift = 0;
        while ((kHalf << p.half_shift) < pv.block_size) ++p.half_shift;
        p.max_len = (int)std::min<int64_t>(table_stride * pv.block_size, 0x7fffffff);
        p.scale_log2 = scale_log2;
        const int most = sms * kBlocksPerSm;
        const int64_t positions = (int64_t)batch * (ceil_div64(max_seq_len, kTile) + kUnitCost) * pv.num_kv_heads * p.groups;
        const unsigned grid = (unsigned)std::max<int64_t>(1, std::min<int64_t>(most, positions / (heads == 16 ? kWarpsWide : kWarps)));
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

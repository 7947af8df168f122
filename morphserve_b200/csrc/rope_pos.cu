// Rotary embedding by position: no tables.  Pair j of token t turns by positions[t] * inv_freq[j].
//
// The angle is formed in 64 bits and reduced to a fraction of a turn there: a position of 10^5..10^6 leaves a 32-bit
// product without correct digits behind the point, while here the reduced angle is good to 2^-24 of half a turn for positions of
// up to 2^53 and frequencies of up to 1 (in 64 bits to 2^-53 of a turn: the product keeps what its rounding leaves over).  One
// thread block computes the sines and cosines of its tokens once, in shared memory, for all heads of q and k; its first
// row loads are in flight meanwhile.  HBM bound: every element is read and written once.
#include <algorithm>
#include <type_traits>

#include "kv_q8.cuh"

namespace mkv {

struct RopePosArgs {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_tok, q_head, k_tok, k_head, qo_tok, qo_head, ko_tok, ko_head;  // strides, elements
    const void *positions;
    const double *inv_freq;
    float scale;
    int pos64;
    int64_t num_tokens;
    int num_pairs, q_heads, heads;
    int pair_tasks;         // tasks of V pairs in a head
    int tasks;              // ... and those that copy 2 V (copy_both) or V elements behind the rotated part
    int copy_both;
    int tokens_per_block;
    uint32_t heads_magic;   // ceil(2^32 / heads): a row's token by a multiplication
};

template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
    if constexpr (std::is_same<T, __half>::value) return __half22float2(*reinterpret_cast<const __half2 *>(&w));
    else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    struct alignas(4) Two { T x, y; } t{rounded<T>(x), rounded<T>(y)};
    return *reinterpret_cast<const uint32_t *>(&t);
}

template <typename T, int V>
struct alignas(sizeof(T) * V) RopeVec {
    T x[V];
};

// One task: V pairs of one head (two vectors, read and written once), or one or two vectors that pass through.
template <typename T, int V, bool INTER>
struct RopeTask {
    T *dst;
    int tok;
    RopeVec<T, V> a, b;

    // `first`: element of the task's first vector in its head; `second`: distance of the second one, 0 if there is none
    __device__ __forceinline__ void load(const RopePosArgs &p, int64_t tok0, int row, int first, int second) {
        tok = (int)__umulhi((uint32_t)row, p.heads_magic);
        const int head = row - tok * p.heads;
        const T *src;
        if (head < p.q_heads) {
            src = (const T *)p.q + (tok0 + tok) * p.q_tok + head * p.q_head + first;
            dst = (T *)p.q_out + (tok0 + tok) * p.qo_tok + head * p.qo_head + first;
        } else {
            src = (const T *)p.k + (tok0 + tok) * p.k_tok + (head - p.q_heads) * p.k_head + first;
            dst = (T *)p.k_out + (tok0 + tok) * p.ko_tok + (head - p.q_heads) * p.ko_head + first;
        }
        a = *reinterpret_cast<const RopeVec<T, V> *>(src);
        if (second) b = *reinterpret_cast<const RopeVec<T, V> *>(src + second);
    }
    // `turns`: (cos, sin) of the task's first pair for the block's first token, the next pair's `step` behind it; null: pass
    // through
    __device__ __forceinline__ void finish(const float2 *turns, int num_pairs, int step, int second) {
        if (turns) {
            const float2 *turn = turns + tok * num_pairs;
            if constexpr (sizeof(T) == 2 && V >= 2) {   // two elements a word
                uint32_t *aw = reinterpret_cast<uint32_t *>(&a), *bw = reinterpret_cast<uint32_t *>(&b);
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    const float2 u = unpack2<T>(aw[i]), w = unpack2<T>(bw[i]);
                    if (INTER) {    // a word is a pair: pair i of the first vector, V / 2 + i of the second
                        const float2 c = turn[i * step], d = turn[(V / 2 + i) * step];
                        aw[i] = pack2<T>(u.x * c.x - u.y * c.y, u.x * c.y + u.y * c.x);
                        bw[i] = pack2<T>(w.x * d.x - w.y * d.y, w.x * d.y + w.y * d.x);
                    } else {        // pairs 2 i and 2 i + 1
                        const float2 c = turn[2 * i * step], d = turn[(2 * i + 1) * step];
                        aw[i] = pack2<T>(u.x * c.x - w.x * c.y, u.y * d.x - w.y * d.y);
                        bw[i] = pack2<T>(u.x * c.y + w.x * c.x, u.y * d.y + w.y * d.x);
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    T &m = INTER ? (2 * i < V ? a.x[2 * i % V] : b.x[2 * i % V]) : a.x[i];
                    T &n = INTER ? (2 * i + 1 < V ? a.x[(2 * i + 1) % V] : b.x[(2 * i + 1) % V]) : b.x[i];
                    const float u = value_of<T>(m), w = value_of<T>(n);
                    const float2 cs = turn[i * step];
                    m = rounded<T>(u * cs.x - w * cs.y);
                    n = rounded<T>(u * cs.y + w * cs.x);
                }
            }
        }
        *reinterpret_cast<RopeVec<T, V> *>(dst) = a;
        if (second) *reinterpret_cast<RopeVec<T, V> *>(dst + second) = b;
    }
};

// A thread keeps its place in a head and goes through the block's rows (token, head) in steps of as many rows as the
// block holds side by side.  Its first loads wait for nothing; the angles are formed while they are on their way.  One task
// in flight a thread and every thread slot of the SM filled: 64 KiB in flight, which measured better than two or four tasks
// in fewer threads (49600 tokens of 32 + 8 heads of 128 fp16: 164 us against 180 and 206 us; 154 us = 6.6 TB/s once the
// arithmetic went by words).  Full occupancy leaves 32 registers a thread: the widest variants spill about 50 bytes of what
// the loop keeps, which at the copy peak costs nothing.
constexpr int kRopeThreads = 256, kRopeBlocks = 8;

template <typename T, int V, bool INTER>
__global__ void __launch_bounds__(kRopeThreads, kRopeBlocks) rope_pos_kernel(const __grid_constant__ RopePosArgs p) {
    // (cos, sin) * scale of [token of the block][pair's place in its task][task]: the threads of a row read neighbours
    extern __shared__ float2 turns[];
    const int64_t tok0 = (int64_t)blockIdx.x * p.tokens_per_block;
    const int ntok = (int)min((int64_t)p.tokens_per_block, p.num_tokens - tok0);
    const int wide = min(p.tasks, kRopeThreads), step = kRopeThreads / wide;   // threads of a row, rows side by side
    // (few tokens: gridDim.y blocks share a token's heads)
    const int all = ntok * p.heads, rows = (int)((int64_t)all * (blockIdx.y + 1) / gridDim.y);
    const int row0 = (int)((int64_t)all * blockIdx.y / gridDim.y) + threadIdx.x / wide;
    int j = threadIdx.x % wide, first = 0, second = 0, row = row0;
    auto place = [&]() {    // of task j in its head
        if (j < p.pair_tasks) {
            first = INTER ? 2 * V * j : V * j;
            second = INTER ? V : p.num_pairs;
        } else {
            first = 2 * p.num_pairs + (j - p.pair_tasks) * (p.copy_both ? 2 * V : V);
            second = p.copy_both ? V : 0;
        }
    };
    RopeTask<T, V, INTER> t;
    const bool on = threadIdx.x / wide < step && row0 < rows;   // (the last threads, where a row's do not divide the block)
    place();
    if (on) t.load(p, tok0, row, first, second);
    for (int i = threadIdx.x; i < ntok * p.num_pairs; i += kRopeThreads) {
        const int tk = i / p.num_pairs;
        const double pos = p.pos64 ? (double)((const int64_t *)p.positions)[tok0 + tk]
                                   : (double)((const int32_t *)p.positions)[tok0 + tk];
        // a + e radians, e what the product's rounding leaves over, are (a + e) / 2 pi turns; 1 / 2 pi in two parts, so that the
        // fraction keeps its digits however many whole turns go away
        const int pair = i - tk * p.num_pairs;
        const double f = p.inv_freq[pair], a = pos * f, e = fma(pos, f, -a);
        const double x = fma(a, 0.15915494309189535, -rint(a * 0.15915494309189535)) + fma(a, -9.839338337591243e-18, e * 0.15915494309189535);
        float sn, cs;
        sincospif((float)(2.0 * x), &sn, &cs);
        turns[tk * p.num_pairs + (pair % V) * p.pair_tasks + pair / V] = make_float2(cs * p.scale, sn * p.scale);
    }
    __syncthreads();
    if (!on) return;
    for (;;) {
        t.finish(j < p.pair_tasks ? turns + j : nullptr, p.num_pairs, p.pair_tasks, second);
        row += step;
        if (row >= rows) {      // the next place, where a head has more of them than the block has threads
            j += wide;
            if (j >= p.tasks) break;
            row = row0;
            place();
        }
        t.load(p, tok0, row, first, second);
    }
}

template <typename T, int V>
static cudaError_t launch_rope_pos(RopePosArgs p, bool interleaved, int copied, int sms, cudaStream_t s) {
    p.pair_tasks = p.num_pairs / V;
    p.copy_both = copied % (2 * V) == 0;
    p.tasks = p.pair_tasks + copied / (p.copy_both ? 2 * V : V);
    // Whole tokens for each block: up to a sine and cosine of each thread, as long as three rounds of blocks are left for
    // the SMs to even out (4097 tokens, 72 heads: 30 us with one or two tokens a block, 35-55 with eight or sixteen).
    int n = (int)std::max<int64_t>(1, std::min<int64_t>(kRopeThreads / p.num_pairs, p.num_tokens / (3ll * kRopeBlocks * sms)));
    while (n > 1 && (int64_t)n * p.heads * p.heads >= (1ll << 31)) --n;
    if (p.heads == 1) n = 1;    // (the magic below is exact for rows up to 2^32 / heads, and for row 0 alone with one head)
    p.tokens_per_block = n;
    p.heads_magic = p.heads == 1 ? 0xffffffffu : (uint32_t)(((1ull << 32) + p.heads - 1) / p.heads);
    const int64_t blocks = ceil_div64(p.num_tokens, n);
    const size_t smem = (size_t)n * p.num_pairs * sizeof(float2);
    // few tokens: a token's heads go to several blocks, until every SM has one or a thread has one task
    const int64_t rounds = ceil_div64((int64_t)p.heads * p.tasks, kRopeThreads);
    const dim3 grid((unsigned)blocks, (unsigned)(n > 1 ? 1 : std::max<int64_t>(1, std::min<int64_t>(rounds, 2 * sms / blocks))));
    if (interleaved)
        rope_pos_kernel<T, V, true><<<grid, kRopeThreads, smem, s>>>(p);
    else
        rope_pos_kernel<T, V, false><<<grid, kRopeThreads, smem, s>>>(p);
    return cudaGetLastError();
}

}  // namespace mkv

using namespace mkv;

extern "C" int mkv_rotary_positions(int device, void *stream, const void *q, const void *k, void *q_out, void *k_out,
                                    const int64_t *strides, const void *positions, int positions_bytes,
                                    const double *inv_freq, int num_pairs, int interleaved, float attention_scale,
                                    int64_t num_tokens, int num_q_heads, int num_kv_heads, int head_dim, int dtype) {
    if (!dtype_ok(dtype) || (positions_bytes != 4 && positions_bytes != 8)) return MKV_ERR_DTYPE;
    if (num_tokens < 0 || num_tokens > 0x7fffffff || num_q_heads < 0 || num_kv_heads < 0 || num_q_heads + num_kv_heads < 1 ||
        head_dim < 2 || num_pairs < 1 || 2 * num_pairs > head_dim || num_pairs > 2048)
        return MKV_ERR_SHAPE;
    const int64_t all_heads = (int64_t)num_q_heads + num_kv_heads;
    if (all_heads > 65535 || all_heads * head_dim > (1 << 26)) return MKV_ERR_SHAPE;     // (heads_magic is exact up to there)
    if (num_tokens == 0) return MKV_OK;
    if (!strides || !positions || !inv_freq) return MKV_ERR_NULL;
    if ((num_q_heads && (!q || !q_out)) || (num_kv_heads && (!k || !k_out))) return MKV_ERR_NULL;
    RopePosArgs p;
    p.q = q; p.k = k; p.q_out = q_out; p.k_out = k_out;
    p.q_tok = strides[0]; p.q_head = strides[1]; p.k_tok = strides[2]; p.k_head = strides[3];
    p.qo_tok = strides[4]; p.qo_head = strides[5]; p.ko_tok = strides[6]; p.ko_head = strides[7];
    p.positions = positions;
    p.inv_freq = inv_freq;
    p.scale = attention_scale;
    p.num_tokens = num_tokens;
    p.num_pairs = num_pairs;
    p.q_heads = num_q_heads;
    p.heads = num_q_heads + num_kv_heads;
    p.pos64 = positions_bytes == 8;
    DeviceGuard guard(device);
    if (guard.err != cudaSuccess) return set_cuda_error(guard.err);
    // the widest vector that bases, strides and the split of the head allow (16 bytes at most)
    const int copied = q == q_out && k == k_out ? 0 : head_dim - 2 * num_pairs;
    uint64_t elems = (uint64_t)num_pairs | (uint64_t)copied;
    uint64_t bytes = 0;
    for (int i = 0; i < 8; ++i)
        if ((i < 2 || i == 4 || i == 5) ? num_q_heads : num_kv_heads) elems |= (uint64_t)strides[i];
    if (num_q_heads) bytes |= (uint64_t)q | (uint64_t)q_out;
    if (num_kv_heads) bytes |= (uint64_t)k | (uint64_t)k_out;
    const int size = dtype_bytes(dtype);
    int vec = 16 / size;
    while (vec > 1 && ((elems & (vec - 1)) || (bytes & ((uint64_t)vec * size - 1)))) vec >>= 1;
    int sms = 0;
    const int st = mkv_sm_count(device, &sms);
    if (st) return st;
    const bool in = interleaved != 0;
    cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
#define ROPE_V(T)                                                              \
    (vec == 8   ? launch_rope_pos<T, 8>(p, in, copied, sms, s)                      \
     : vec == 4 ? launch_rope_pos<T, 4>(p, in, copied, sms, s)                      \
     : vec == 2 ? launch_rope_pos<T, 2>(p, in, copied, sms, s) : launch_rope_pos<T, 1>(p, in, copied, sms, s))
    if (dtype == MKV_F16) e = ROPE_V(__half);
    else if (dtype == MKV_BF16) e = ROPE_V(__nv_bfloat16);
    else e = vec == 4 ? launch_rope_pos<float, 4>(p, in, copied, sms, s)
             : vec == 2 ? launch_rope_pos<float, 2>(p, in, copied, sms, s) : launch_rope_pos<float, 1>(p, in, copied, sms, s);
#undef ROPE_V
    if (e != cudaSuccess) return set_cuda_error(e);
    return MKV_OK;
}

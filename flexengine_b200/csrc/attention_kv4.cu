// Paged causal grouped-query attention over keys and values held in 4 bits (kv4.cuh has their form), for single tokens and for short
// portions of prompts, and for all of them where the queries are 32-bit.
//
// With x = c + s n (n the code less 8, s and c of the key's or the value's group g of 32 numbers) the score of a key is
//     q . k = sum_g s_g (q_g . n_g) + sum_g c_g (sum of q_g)
// and the output, with weights p_t = 2^(score_t - m),
//     o_g = sum_t (p_t s_tg) n_tg + sum_t p_t c_tg ,
// so the codes themselves go through the tensor cores, as whole numbers that half precision holds exactly, and scales and centres are
// applied in 32 bits: the scales to the groups' partial scores and to the weights, the centres as one more product of (c_g) with the
// sums of q_g, and as sums of p_t c_tg.  What is rounded is the query to half precision (exact for bfloat16 but for numbers 2^-24 of the
// row's largest) and the weights p s; 32-bit queries take both in two parts, high and low, which leaves 22 bits.
//
// Which keys a query sees, the online softmax and its sink are those of the attention over 16-bit caches: key t is visible to the query at
// position p iff t <= p (and t > p - window, or t < keep, when window > 0).
//
// Keys are the rows of the products and the (query, head of the group) pairs their columns, eight a tile: S^T = K Q^T is m16n8k16 with 16 keys
// by 8 columns, O^T = V^T P^T has 16 numbers of the head by 8 columns.  A group of 5 or 7 heads then fills a tile (with the heads
// as the rows more than half of it were padding), and the codes, which lie in the order of the A operand, are decoded once for all columns.
// The weights change from result to operand by a transposing 8 x 8 move.  Row r of a tile is its token 2 (r / 2) + (r & 1 ^ r / 2 & 1): neighbouring
// rows then lie in different halves of the shared-memory banks both for keys and for values.
//
// A warp walks tiles of its own with a ring of bulk copies of its own (a tile of one head is one piece, 640 bytes a group, 2,560 at head size
// 128): no barrier between warps until the end, several tiles on their way.  The four warps of a block, and the blocks that share
// a row's keys, are merged at the end by their maxima and sums, in a fixed order.
//
// A weight p s has to keep its place in half precision whatever the scale of the values, so the reference point m is a maximum of score +
// exponent of the token's largest value scale: 2^(score - m) s is then at most 2, and the sum of 2^(score - m) is kept in 32 bits, where
// small scales may make it large.  The reference moves only when it has grown by more than 2^8.
#define FE_PDL_CLASS 2      // FE_PDL_DECODE_ATTENTION
#include "kv4.cuh"
#include "tcgen05.cuh"

using namespace fe;

namespace {

constexpr int WARPS = 4;
constexpr int STAGES = 4;
constexpr long long WAIT_LIMIT = 1000000000LL;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float MOVE_STEP = 8.f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma(float* c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the same with nothing added to
__device__ __forceinline__ void mma_fresh(float* c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ unsigned transposed(unsigned a) {
    unsigned d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(d) : "r"(a));
    return d;
}
__device__ __forceinline__ unsigned pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const unsigned*>(&h);
}
// what ``pack`` left over of the two
__device__ __forceinline__ unsigned pack_rest(float lo, float hi, unsigned packed) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&packed));
    return pack(lo - f.x, hi - f.y);
}
__device__ __forceinline__ float low_half(unsigned w) { return __low2float(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float high_half(unsigned w) { return __high2float(*reinterpret_cast<const __half2*>(&w)); }

// N words side by side in shared memory, in the widest loads that their place allows.
template <int N> __device__ __forceinline__ void words(const unsigned char* p, unsigned* w) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 v = *reinterpret_cast<const uint4*>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y; w[i + 2] = v.z; w[i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 v = *reinterpret_cast<const uint2*>(p + 4 * i);
            w[i] = v.x; w[i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = *reinterpret_cast<const unsigned*>(p + 4 * i);
    }
}
// NG pieces of 16 bits side by side, two a word.
template <int NG> __device__ __forceinline__ void pieces(const unsigned char* p, unsigned* w) {
    if constexpr (NG % 2 == 0) words<NG / 2>(p, w);
    else {
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const unsigned v = *reinterpret_cast<const unsigned short*>(p + 2 * i);
            if (i & 1) w[i / 2] |= v << 16;
            else w[i / 2] = v;
        }
    }
}

// false when the wait ran out
__device__ __forceinline__ bool wait_for(unsigned long long* bar, unsigned parity) { return mbar_wait(bar, parity, WAIT_LIMIT); }

__device__ __forceinline__ void copy_tile(void* dst, const unsigned char* src, int bytes, unsigned long long* bar) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}

template <typename T> __device__ __forceinline__ void put(T* p, float v);
template <> __device__ __forceinline__ void put<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void put<bf16>(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

struct Problem {
    const void* q;
    long long q_stride;
    void* out;
    long long out_stride;
    const unsigned char* cache;
    const int* block_table;
    int bt_stride;
    const int* cu_q;
    const int* q_start;
    int nq, nkv, d, ps, num_pages;
    float scale_log2;
    int window, keep, sink, splits;
    float* part;            // [token, head, split, d] float32, then [token, head, split] maxima and sums
    long long tokens;       // rows of q
    int* status;
};

// dynamic shared memory: every warp's ring, and later the warps' results
template <int NG, int NT> __host__ __device__ constexpr int ring_bytes() { return WARPS * STAGES * kv4_tile_bytes(NG); }
template <int NG, int NT> __host__ __device__ constexpr int result_bytes() { return WARPS * 8 * NT * (32 * NG + 4) * 4; }
template <int NG, int NT> __host__ __device__ constexpr int smem_bytes() {
    return ring_bytes<NG, NT>() > result_bytes<NG, NT>() ? ring_bytes<NG, NT>() : result_bytes<NG, NT>();
}

// grid (splits x column tiles, key/value heads, requests).  TQ: queries and output; 32-bit ones in two parts.  NG: groups of a row.
// NT: tiles of eight columns that a block takes.
template <typename TQ, int NG, int NT>
__global__ void __launch_bounds__(WARPS * 32)
kv4_attention_kernel(const Problem a) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int PARTS = sizeof(TQ) == 4 ? 2 : 1;
    constexpr int COLS = 8 * NT, TILE = kv4_tile_bytes(NG);
    constexpr unsigned FULL = 0xffffffffu;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) unsigned long long bars[WARPS][STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int split = blockIdx.x % a.splits, r = blockIdx.z, kvh = blockIdx.y, G = a.nq / a.nkv;
    const int tok0 = a.cu_q[r], n_q = (int)min((long long)a.cu_q[r + 1], a.tokens) - tok0, columns = n_q * G;
    // the last columns walk the most keys: first
    const int tiles_of_columns = (columns + COLS - 1) / COLS, m0 = (tiles_of_columns - 1 - (int)(blockIdx.x / a.splits)) * COLS;
    if (m0 < 0 || columns <= 0) return;
    const int start = a.q_start[r];
    const int first_q = m0 / G, last_q = min(n_q - 1, (m0 + COLS - 1) / G);
    const int hi = start + last_q, lo = first_visible(start + first_q, a.window);
    const int kept = kept_tiles<KV4_TILE>(lo, a.keep), all_tiles = kept + hi / KV4_TILE - lo / KV4_TILE + 1;
    const int per = (all_tiles + a.splits - 1) / a.splits, t_begin = split * per, t_end = min(all_tiles, t_begin + per);
    const int mine = max(0, (t_end - t_begin - warp + WARPS - 1) / WARPS);       // tiles t_begin + warp, + WARPS, ...

    if (lane < STAGES) mbar_init(&bars[warp][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    __syncwarp();

    // ---- where the tiles lie: a lane each for 32 of the warp's tiles at a time
    const int* table = a.block_table + (long long)r * a.bt_stride;
    const int per_page = a.ps / KV4_TILE;
    const unsigned char* at = nullptr;                   // of this lane's tile of the batch whose copies are being started
    unsigned here_now = 0, here_before = 0;              // which of that batch's and of the one before are in the cache
    auto look_up = [&](int batch) {
        const int k = 32 * batch + lane;
        at = nullptr;
        if (k < mine) {
            const int tile = listed_tile<KV4_TILE>(t_begin + warp + WARPS * k, kept, lo);
            const int page = tile / per_page < a.bt_stride ? table[tile / per_page] : -1;
            if (page < 0 || page >= a.num_pages) {
                if (a.status) atomicOr(a.status, FE_STATUS_BAD_PAGE);
            } else
                at = a.cache + (((long long)page * a.nkv + kvh) * per_page + tile % per_page) * TILE;
        }
        here_before = here_now;
        here_now = __ballot_sync(FULL, at != nullptr);
    };
    unsigned char* ring = smem + warp * STAGES * TILE;
    auto begin_copy = [&](int k) {
        if ((k & 31) == 0) look_up(k >> 5);
        const unsigned long long from = __shfl_sync(FULL, (unsigned long long)at, k & 31);
        if (lane == 0) {
            if (from) copy_tile(ring + (k % STAGES) * TILE, reinterpret_cast<const unsigned char*>(from), TILE, &bars[warp][k % STAGES]);
            else mbar_arrive(&bars[warp][k % STAGES]);       // nothing to bring: the stage's turn passes all the same
        }
    };
    for (int k = 0; k < STAGES - 1 && k < mine; ++k) begin_copy(k);

    // ---- the queries: column n of tile j as B operands; thread (g, t) holds numbers 32 i + 8 t .. + 7 of column g
    unsigned qf[NT][NG][4][PARTS], qsum[NT][2];          // qsum: (high, low) of the sums over group t, and over group t + 4
    float factor[NT][2];                                 // takes a score of columns 2t, 2t + 1 to log2 units
    int last_key[NT][2], first_key[NT][2];
    float m[NT][2], l[NT][2];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
        const int c = m0 + 8 * j + g;
        const bool real = c < columns;
        const TQ* row = static_cast<const TQ*>(a.q) + (long long)(tok0 + (real ? c / G : 0)) * a.q_stride + (long long)(kvh * G + (real ? c % G : 0)) * a.d;
        float v[NG][8], largest = 0.f;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const int from = 32 * i + 8 * t;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[i][e] = 0.f;
            if (real && from < a.d) load8<TQ>(row + from, v[i]);
#pragma unroll
            for (int e = 0; e < 8; ++e) largest = fmaxf(largest, fabsf(v[i][e]));
        }
        largest = fmaxf(largest, __shfl_xor_sync(FULL, largest, 1));
        largest = fmaxf(largest, __shfl_xor_sync(FULL, largest, 2));
        // a power of two brings the row's largest number to [1, 2): half precision then holds bfloat16 numbers as they are
        const int e2 = min(max((int)(__float_as_uint(largest) >> 23) - 127, -126), 126);
        const float down = __uint_as_float((unsigned)(127 - e2) << 23);
        float sums[NG];
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            sums[i] = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[i][e] *= down; sums[i] += v[i][e]; }
            sums[i] += __shfl_xor_sync(FULL, sums[i], 1);
            sums[i] += __shfl_xor_sync(FULL, sums[i], 2);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                qf[j][i][e][0] = pack(v[i][e], v[i][e + 4]);
                if (PARTS == 2) qf[j][i][e][PARTS - 1] = pack_rest(v[i][e], v[i][e + 4], qf[j][i][e][0]);
            }
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float s = 0.f;
#pragma unroll
            for (int i = 0; i < NG; ++i)
                if (i == t + 4 * h) s = sums[i];
            const float high = __half2float(__float2half_rn(s));
            qsum[j][h] = pack(high, s - high);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int mc = m0 + 8 * j + 2 * t + h;
            factor[j][h] = a.scale_log2 * __uint_as_float((unsigned)(127 + __shfl_sync(FULL, e2, (2 * t + h) * 4)) << 23);
            // a padding column sees what the last query sees: it is computed and never written, and must not make a tile a masked one
            const int pos = mc < columns ? start + mc / G : hi;
            last_key[j][h] = pos;
            first_key[j][h] = mc < columns ? first_visible(pos, a.window) : lo;
            m[j][h] = -CUDART_INF_F;
            l[j][h] = 0.f;
            if (a.sink && split == 0 && warp == 0) {
                m[j][h] = 0.f;
                l[j][h] = g == 0 ? 1.f : 0.f;            // the lanes of a column add their sums up at the end
            }
        }
    }
    int last_least = last_key[0][0], first_most = first_key[0][0];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) { last_least = min(last_least, last_key[j][h]); first_most = max(first_most, first_key[j][h]); }
    last_least = __reduce_min_sync(FULL, last_least);
    first_most = __reduce_max_sync(FULL, first_most);

    float o[NT][NG][2][4], oc[NT][NG][2];                // sums over codes, 16 numbers a tile, and over centres (this thread's tokens)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            oc[j][i][0] = oc[j][i][1] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][i][0][e] = o[j][i][1][e] = 0.f;
        }

    const int even = 2 * t + (t & 1), odd = 2 * t + 1 - (t & 1);      // tokens of rows 2t and 2t + 1 (and of 2t + 8, 2t + 9: 8 on)
    const int key_row = (g & ~1) + ((g & 1) ^ (g >> 1 & 1));          // token of row g
    bool gone = false;
    for (int k = 0; k < mine; ++k) {
        if (k + STAGES - 1 < mine) begin_copy(k + STAGES - 1);
        if (__any_sync(FULL, !wait_for(&bars[warp][k % STAGES], (k / STAGES) & 1))) {
            gone = true;
            for (int later = k + 1; later < min(mine, k + STAGES); ++later) wait_for(&bars[warp][later % STAGES], (later / STAGES) & 1);
            break;
        }
        // the batch of tile k: that of the newest copy or the one before
        const int newest = min(mine - 1, k + STAGES - 1) >> 5;
        if (!(((k >> 5) == newest ? here_now : here_before) >> (k & 31) & 1u)) continue;        // a page that is not there: nothing seen
        const unsigned char* tile = ring + (k % STAGES) * TILE;
        const int key0 = listed_tile<KV4_TILE>(t_begin + warp + WARPS * k, kept, lo) * KV4_TILE;
        const bool masked = key0 + KV4_TILE - 1 > last_least || (key0 < first_most && key0 + KV4_TILE > a.keep);

        // ---- scores of tokens key_row and key_row + 8 by columns 2t, 2t + 1
        float s[NT][4];
        {
            unsigned c0 = 0, c1 = 0, c2 = 0, c3 = 0;                  // (centre, centre) of group t, and of group t + 4
            const unsigned char* pairs = tile + kv4_key_pairs(NG);
            if (t < NG) {
                const unsigned w0 = *reinterpret_cast<const unsigned*>(pairs + (key_row * NG + t) * 4);
                const unsigned w1 = *reinterpret_cast<const unsigned*>(pairs + ((key_row + 8) * NG + t) * 4);
                c0 = __byte_perm(w0, w0, 0x3232); c1 = __byte_perm(w1, w1, 0x3232);
            }
            if (NG > 4 && t + 4 < NG) {
                const unsigned w0 = *reinterpret_cast<const unsigned*>(pairs + (key_row * NG + t + 4) * 4);
                const unsigned w1 = *reinterpret_cast<const unsigned*>(pairs + ((key_row + 8) * NG + t + 4) * 4);
                c2 = __byte_perm(w0, w0, 0x3232); c3 = __byte_perm(w1, w1, 0x3232);
            }
#pragma unroll
            for (int j = 0; j < NT; ++j) mma_fresh(s[j], c0, c1, c2, c3, qsum[j][0], NG > 4 ? qsum[j][1] : 0u);
            unsigned k0[NG], k1[NG], p0[NG], p1[NG];
            words<NG>(tile + key_row * 16 * NG + t * 4 * NG, k0);
            words<NG>(tile + (key_row + 8) * 16 * NG + t * 4 * NG, k1);
            words<NG>(pairs + key_row * 4 * NG, p0);
            words<NG>(pairs + (key_row + 8) * 4 * NG, p1);
#pragma unroll
            for (int i = 0; i < NG; ++i) {
                unsigned n0[4], n1[4];
                kv4_decode(k0[i], n0);
                kv4_decode(k1[i], n1);
                const float s0 = low_half(p0[i]), s1 = low_half(p1[i]);
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    float part[4];
                    mma_fresh(part, n0[0], n1[0], n0[1], n1[1], qf[j][i][0][0], qf[j][i][1][0]);
                    mma(part, n0[2], n1[2], n0[3], n1[3], qf[j][i][2][0], qf[j][i][3][0]);
                    if (PARTS == 2) {
                        mma(part, n0[0], n1[0], n0[1], n1[1], qf[j][i][0][PARTS - 1], qf[j][i][1][PARTS - 1]);
                        mma(part, n0[2], n1[2], n0[3], n1[3], qf[j][i][2][PARTS - 1], qf[j][i][3][PARTS - 1]);
                    }
                    s[j][0] = fmaf(s0, part[0], s[j][0]);
                    s[j][1] = fmaf(s0, part[1], s[j][1]);
                    s[j][2] = fmaf(s1, part[2], s[j][2]);
                    s[j][3] = fmaf(s1, part[3], s[j][3]);
                }
            }
        }
        // ---- weights
        unsigned v0[NG], v1[NG];                                      // (scale, centre) of the two tokens' value groups
        words<NG>(tile + kv4_value_pairs(NG) + key_row * 4 * NG, v0);
        words<NG>(tile + kv4_value_pairs(NG) + (key_row + 8) * 4 * NG, v1);
        float big0 = low_half(v0[0]), big1 = low_half(v1[0]);
#pragma unroll
        for (int i = 1; i < NG; ++i) { big0 = fmaxf(big0, low_half(v0[i])); big1 = fmaxf(big1, low_half(v1[i])); }
        // their exponents; zeros and subnormal numbers count as 2^-24, the least scale there is
        const float up0 = fmaxf((float)((int)(__float_as_uint(big0) >> 23) - 127), -24.f), up1 = fmaxf((float)((int)(__float_as_uint(big1) >> 23) - 127), -24.f);
        bool grows = false;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[j][e] *= factor[j][e & 1];
                if (masked) {
                    const int key = key0 + key_row + (e & 2) * 4;
                    if (!(key <= last_key[j][e & 1] && (key >= first_key[j][e & 1] || key < a.keep))) s[j][e] = -CUDART_INF_F;
                }
                grows |= s[j][e] + (e < 2 ? up0 : up1) > m[j][e & 1] + MOVE_STEP;
            }
        }
        if (__any_sync(FULL, grows)) {
#pragma unroll
            for (int j = 0; j < NT; ++j)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float mx = fmaxf(s[j][h] + up0, s[j][h + 2] + up1);
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, off));
                    const float to = fmaxf(m[j][h], mx);
                    const float by = to == -CUDART_INF_F ? 1.f : ex2(m[j][h] - to);      // 2^-inf = 0 at the start
                    m[j][h] = to;
                    l[j][h] *= by;
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        oc[j][i][h] *= by;
                        o[j][i][0][h] *= by; o[j][i][0][h + 2] *= by;
                        o[j][i][1][h] *= by; o[j][i][1][h + 2] *= by;
                    }
                }
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float ref = m[j][e & 1];
                s[j][e] = ex2(s[j][e] - (ref == -CUDART_INF_F ? 0.f : ref));
            }
            l[j][0] += s[j][0] + s[j][2];
            l[j][1] += s[j][1] + s[j][3];
        }
        // ---- values: tokens even, odd (+ 8) in pairs; numbers 32 i + 4 g .. + 3
        constexpr int VW = (NG + 1) / 2;
        unsigned ve[VW], vo[VW], ve8[VW], vo8[VW];
        const unsigned char* codes = tile + kv4_value_codes(NG) + g * 2 * NG;
        pieces<NG>(codes + even * 16 * NG, ve);
        pieces<NG>(codes + odd * 16 * NG, vo);
        pieces<NG>(codes + (even + 8) * 16 * NG, ve8);
        pieces<NG>(codes + (odd + 8) * 16 * NG, vo8);
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            unsigned na[4], nb[4];
            kv4_decode(__byte_perm(ve[i / 2], vo[i / 2], (i & 1) ? 0x7632 : 0x5410), na);
            kv4_decode(__byte_perm(ve8[i / 2], vo8[i / 2], (i & 1) ? 0x7632 : 0x5410), nb);
            const float s0 = low_half(v0[i]), s1 = low_half(v1[i]), c0 = high_half(v0[i]), c1 = high_half(v1[i]);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                float w[4] = {s[j][0] * s0, s[j][1] * s0, s[j][2] * s1, s[j][3] * s1};
                float z[4] = {s[j][0] * c0, s[j][1] * c0, s[j][2] * c1, s[j][3] * c1};
                if (masked) {                                         // what lies behind a mask may be anything, NaN too
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (s[j][e] == 0.f) w[e] = z[e] = 0.f;
                }
                oc[j][i][0] += z[0] + z[2];
                oc[j][i][1] += z[1] + z[3];
                const unsigned w0 = pack(w[0], w[1]), w1 = pack(w[2], w[3]);
                const unsigned b0 = transposed(w0), b1 = transposed(w1);
                mma(o[j][i][0], na[0], na[1], nb[0], nb[1], b0, b1);
                mma(o[j][i][1], na[2], na[3], nb[2], nb[3], b0, b1);
                if (PARTS == 2) {
                    const unsigned r0 = transposed(pack_rest(w[0], w[1], w0)), r1 = transposed(pack_rest(w[2], w[3], w1));
                    mma(o[j][i][0], na[0], na[1], nb[0], nb[1], r0, r1);
                    mma(o[j][i][1], na[2], na[3], nb[2], nb[3], r0, r1);
                }
            }
        }
        __syncwarp();                                                 // the stage is free: the next turn's copy goes there
    }
    if (gone && lane == 0 && a.status) atomicOr(a.status, FE_STATUS_WAIT_EXPIRED);

    // ---- the warp's sums over its lanes, then the four warps' results side by side: [warp][column][32 NG numbers, maximum, sum]
    constexpr int ROW = 32 * NG + 4;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l[j][h] += __shfl_xor_sync(FULL, l[j][h], off);
#pragma unroll
                for (int i = 0; i < NG; ++i) oc[j][i][h] += __shfl_xor_sync(FULL, oc[j][i][h], off);
            }
        }
    __syncthreads();                                                  // every warp has read its last tile
    float* results = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* to = results + (warp * COLS + 8 * j + 2 * t + h) * ROW;
#pragma unroll
            for (int i = 0; i < NG; ++i)
                *reinterpret_cast<float4*>(to + 32 * i + 4 * g) =
                    make_float4(o[j][i][0][h] + oc[j][i][h], o[j][i][0][h + 2] + oc[j][i][h], o[j][i][1][h] + oc[j][i][h], o[j][i][1][h + 2] + oc[j][i][h]);
            if (g == 0) { to[32 * NG] = m[j][h]; to[32 * NG + 1] = l[j][h]; }
        }
    __syncthreads();
    for (int c = warp; c < COLS && m0 + c < columns; c += WARPS) {
        const int mc = m0 + c, token = tok0 + mc / G, head = kvh * G + mc % G;
        float top = -CUDART_INF_F;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) top = fmaxf(top, results[(w * COLS + c) * ROW + 32 * NG]);
        float by[WARPS], sum = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) {
            const float mw = results[(w * COLS + c) * ROW + 32 * NG];
            by[w] = mw == -CUDART_INF_F ? 0.f : ex2(mw - top);
            sum += by[w] * results[(w * COLS + c) * ROW + 32 * NG + 1];
        }
        const long long line = (long long)token * a.nq + head;
        const float inv = a.splits > 1 ? 1.f : sum > 0.f ? 1.f / sum : 0.f;
        for (int i = lane; i < a.d; i += 32) {
            float v = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) v += by[w] != 0.f ? by[w] * results[(w * COLS + c) * ROW + i] : 0.f;
            if (a.splits > 1) a.part[(line * a.splits + split) * a.d + i] = v;
            else put<TQ>(static_cast<TQ*>(a.out) + (long long)token * a.out_stride + (long long)head * a.d + i, v * inv);
        }
        if (a.splits > 1 && lane == 0)
            reinterpret_cast<float2*>(a.part + a.tokens * a.nq * a.splits * a.d)[line * a.splits + split] = make_float2(top, sum);
    }
}

constexpr int MAX_SPLITS = 64;

// A block per (token, head): the splits' sums, weighted by their maxima, in the splits' order.
template <typename TQ>
__global__ void __launch_bounds__(128)
kv4_merge_kernel(const float* __restrict__ part, TQ* __restrict__ out, long long out_stride, int nq, int d, int splits, long long rows) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ float by[MAX_SPLITS];
    const long long line = blockIdx.x;
    const float2* heads = reinterpret_cast<const float2*>(part + rows * splits * d) + line * splits;
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x;
        float2 h[MAX_SPLITS / 32];
        float top = -CUDART_INF_F, sum = 0.f;
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 32; ++i) {
            h[i] = lane + 32 * i < splits ? heads[lane + 32 * i] : make_float2(-CUDART_INF_F, 0.f);
            top = fmaxf(top, h[i].x);
        }
        top = warp_max(top);
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 32; ++i) {
            h[i].x = h[i].x == -CUDART_INF_F ? 0.f : ex2(h[i].x - top);
            sum += h[i].x * h[i].y;
        }
        sum = warp_sum(sum);
        const float inv = sum > 0.f ? 1.f / sum : 0.f;
#pragma unroll
        for (int i = 0; i < MAX_SPLITS / 32; ++i) by[lane + 32 * i] = h[i].x * inv;
    }
    __syncthreads();
    const float* from = part + line * splits * d;
    TQ* to = out + line / nq * out_stride + line % nq * d;
    for (int i = threadIdx.x; i < d; i += blockDim.x) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s)
            if (by[s] != 0.f) v += by[s] * from[(long long)s * d + i];
        put<TQ>(to + i, v);
    }
}

template <typename TQ, int NG, int NT>
int launch_as(const Problem& a, int requests, int column_tiles, cudaStream_t stream) {
    constexpr int smem = smem_bytes<NG, NT>();
    if (smem > 48 * 1024) {
        const cudaError_t err = cudaFuncSetAttribute(kv4_attention_kernel<TQ, NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        FE_REQUIRE(err == cudaSuccess, "paged_attention_kv4: %s", cudaGetErrorString(err));
    }
    fe::launch(kv4_attention_kernel<TQ, NG, NT>, dim3((unsigned)(a.splits * column_tiles), (unsigned)a.nkv, (unsigned)requests), WARPS * 32, smem, stream, a);
    return fe_check_launch("paged_attention_kv4");
}

template <typename TQ, int NT>
int launch_groups(const Problem& a, int requests, int column_tiles, cudaStream_t stream) {
    switch (kv4_groups(a.d)) {
        case 1: return launch_as<TQ, 1, NT>(a, requests, column_tiles, stream);
        case 2: return launch_as<TQ, 2, NT>(a, requests, column_tiles, stream);
        case 3: return launch_as<TQ, 3, NT>(a, requests, column_tiles, stream);
        case 4: return launch_as<TQ, 4, NT>(a, requests, column_tiles, stream);
        case 5: return launch_as<TQ, 5, NT>(a, requests, column_tiles, stream);
        case 6: return launch_as<TQ, 6, NT>(a, requests, column_tiles, stream);
        case 7: return launch_as<TQ, 7, NT>(a, requests, column_tiles, stream);
        default: return launch_as<TQ, 8, NT>(a, requests, column_tiles, stream);
    }
}

template <typename TQ>
int attend(const Problem& a, int requests, int max_q_len, cudaStream_t stream) {
    const int column_tiles = (int)(((long long)max_q_len * (a.nq / a.nkv) + 7) / 8);
    return launch_groups<TQ, 1>(a, requests, column_tiles, stream);
}

}  // namespace

extern "C" int fe_kv4_attention_max_splits() { return MAX_SPLITS; }

// Bytes of ``scratch`` for ``tokens`` rows of queries.
extern "C" long long fe_kv4_attention_scratch_bytes(long long tokens, int nq, int d, int splits) {
    return splits > 1 ? tokens * nq * splits * (4LL * d + 8) : 0;
}

// q [tokens, >= nq d], rows ``q_stride`` elements apart; out likewise; dtype of both.  ``splits``: blocks that share a row's keys.
extern "C" int fe_paged_attention_kv4(const void* q, long long q_stride, void* out, long long out_stride, const void* cache, const int* block_table,
                                      int bt_stride, const int* cu_q, const int* q_start, int requests, long long tokens, int max_q_len, int nq,
                                      int nkv, int d, int ps, int num_pages, float scale, int window, int keep, int sink, int splits, void* scratch,
                                      int dtype, int* status, cudaStream_t stream) {
    FE_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0 && nkv <= 65535, "paged_attention_kv4: bad head counts %d/%d", nq, nkv);
    FE_REQUIRE(d >= 16 && d % 16 == 0 && d <= KV4_MAX_DIM, "paged_attention_kv4: head size %d; multiples of 16 up to %d", d, KV4_MAX_DIM);
    FE_REQUIRE(ps > 0 && ps % KV4_TILE == 0 && num_pages > 0, "paged_attention_kv4: page size %d (a multiple of %d) or page count", ps, KV4_TILE);
    FE_REQUIRE(q_stride % 8 == 0 && (((size_t)q | (size_t)out | (size_t)cache) & 15) == 0, "paged_attention_kv4: rows must start on 16-byte boundaries");
    FE_REQUIRE(requests >= 0 && requests <= 65535 && max_q_len >= 0 && tokens >= 0, "paged_attention_kv4: bad request count or length");
    FE_REQUIRE(window >= 0 && keep >= 0 && (keep == 0 || window > 0), "paged_attention_kv4: a window is not negative, kept keys go with one");
    FE_REQUIRE(splits >= 1 && splits <= MAX_SPLITS && (splits == 1 || (scratch && ((size_t)scratch & 15) == 0)), "paged_attention_kv4: %d splits", splits);
    FE_REQUIRE((long long)max_q_len * (nq / nkv) * splits < (1LL << 31) - 64, "paged_attention_kv4: grid too large");
    if (requests == 0 || max_q_len == 0 || tokens == 0) return 0;
    const Problem a{q, q_stride, out, out_stride, (const unsigned char*)cache, block_table, bt_stride, cu_q, q_start, nq, nkv, d, ps, num_pages,
                    scale * LOG2E, window, keep, sink, splits, (float*)scratch, tokens, status};
    FE_REQUIRE(dtype == FE_F32 || dtype == FE_BF16, "paged_attention_kv4: unknown type %d", dtype);
    const int rc = dtype == FE_F32 ? attend<float>(a, requests, max_q_len, stream) : attend<bf16>(a, requests, max_q_len, stream);
    if (rc || splits == 1) return rc;
    FE_REQUIRE(tokens * nq < (1LL << 31), "paged_attention_kv4: merge grid too large");
    if (dtype == FE_F32)
        fe::launch(kv4_merge_kernel<float>, dim3((unsigned)(tokens * nq)), 128, 0, stream, (const float*)scratch, (float*)out, out_stride, nq, d, splits, tokens * nq);
    else
        fe::launch(kv4_merge_kernel<bf16>, dim3((unsigned)(tokens * nq)), 128, 0, stream, (const float*)scratch, (bf16*)out, out_stride, nq, d, splits, tokens * nq);
    return fe_check_launch("paged_attention_kv4 merge");
}

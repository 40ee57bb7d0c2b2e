// Paged causal grouped-query attention over keys and values held in 4 bits (kv4.cuh has their form), for single tokens and for short
// portions of prompts, and for all of them where the queries are 32-bit.
//
// With x = c + s n (n the code less 8, s and c of the key's or the value's group g of 32 numbers) the score of a key is
//     q . k = sum_g s_g (q_g . n_g) + sum_g c_g (sum of q_g)
// and the output, with weights p_t = 2^(score_t - m),
//     o_g = sum_t (p_t s_tg) n_tg + sum_t p_t c_tg ,
// so the codes themselves go through the tensor cores, as whole numbers that half precision holds exactly.  Of keys, scales are applied to
// the groups' partial scores in 32 bits, centres as one more product of (c_g) with the sums of q_g.  What is rounded is the query to half precision (exact for
// bfloat16 from 2^-17 of the row's largest number on; what is smaller is off by up to 2^-25 of it).  Of values under 16-bit queries, scale and centre go into the decoded
// numbers (one multiply-add for two, rounded to half precision: 2^-11 of a number, where bfloat16 results have 2^-8) and the weights p into half
// precision; under 32-bit queries scales go to the weights in 32 bits and centres into sums of p_t c_tg, and query and weights are taken in two
// parts, high and low: 22 bits of what is near the largest, and no step below 2^-24 where that is one (a weight of 2^-11 keeps 14 bits).
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
// The reference point m is the largest score met, and moves only when it has grown by more than 2^8 (weights stay below that: in half's range).  Under 32-bit
// queries a weight p s has to keep its place in half precision whatever the scale of the values, so there m is a maximum of score +
// exponent of the token's largest value scale: 2^(score - m) s is then at most 2, and the sum of 2^(score - m) is kept in 32 bits, where
// small scales may make it large.  A NaN score never moves it: who has met no other has a NaN sum beside a maximum of -inf, and a merge passes it on.
//
// Long rows are bound by the instructions that decode: 16 requests of up to 32,768 keys, 40/8 heads of 128, 93 us for 396 MB of cache (4.3 TB/s; the copies
// alone, nothing computed, 74); 64 of up to 8,191, 28/4 heads, 63.  Short ones by latency: 8 of 2,049 13; a call of a few keys 7.6.  The kernels of head size 128 under
// 16-bit queries are held to 128 registers for four blocks an SM and spill 44 and 68 bytes a thread; 32-bit ones of head size 256 28 and 140.
#include <type_traits>

#define FE_PDL_CLASS 2      // FE_PDL_DECODE_ATTENTION
#include "kv4.cuh"
#include "tcgen05.cuh"

using namespace fe;

namespace {

constexpr int WARPS = 4;
constexpr int COLS = 8;             // columns that a block takes: (query, head of the group) pairs
constexpr int PAIR = 2;              // tiles that a warp takes at once
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
// the same, added to ``even`` and ``odd`` in every row's two columns
__device__ __forceinline__ void mma_from(float* c, unsigned a0, unsigned a1, unsigned a2, unsigned a3, unsigned b0, unsigned b1, float even, float odd) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%10,%11};\n"
                 : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(even), "f"(odd));
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
// Four pairs times a pair plus another
__device__ __forceinline__ void times_plus(unsigned* n, unsigned scale, unsigned centre) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&n[i]), *reinterpret_cast<const __half2*>(&scale), *reinterpret_cast<const __half2*>(&centre));
        n[i] = *reinterpret_cast<const unsigned*>(&x);
    }
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

// false when the wait ran out; the test itself waits a while, so the clock is asked rarely
__device__ __forceinline__ bool wait_for(unsigned long long* bar, unsigned parity, long long limit) {
    if (mbar_test(bar, parity)) return true;
    return mbar_wait(bar, parity, limit);
}

__device__ __forceinline__ void copy_tile(unsigned to, const unsigned char* from, int bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                 ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}

template <typename T> __device__ __forceinline__ void put(T* p, float v);
template <> __device__ __forceinline__ void put<float>(float* p, float v) { *p = v; }
template <> __device__ __forceinline__ void put<bf16>(bf16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
// the same variable in the shared memory of block ``rank`` of this cluster
__device__ __forceinline__ float ld_cluster(const float* own, unsigned rank) {
    unsigned remote;
    float v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"(smem_u32(own)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];\n" : "=f"(v) : "r"(remote) : "memory");
    return v;
}

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
    int requests, nq, nkv, d, ps, num_pages;
    float scale_log2;
    int window, keep, sink, splits;
    float* part;            // partial results of the blocks: see the kernel
    long long tokens;       // rows of q
    int* status;
    FeWaits waits;
};

// dynamic shared memory: every warp's ring, two places of a pair of tiles each; a warp's results go to the place that no copy is on its way to
constexpr int STAGES = 2;
template <int NG> __host__ __device__ constexpr int ring_bytes() { return WARPS * STAGES * PAIR * kv4_tile_bytes(NG); }
template <int NG> __host__ __device__ constexpr int smem_bytes() {
    static_assert(COLS * (32 * NG + 4) * 4 <= PAIR * kv4_tile_bytes(NG), "a warp's results fit a pair of tiles");
    return ring_bytes<NG>();
}

// One piece of work of a block: tiles [t_begin, t_end) of the list that the columns from m0 on of (request r, head kvh) see.
struct Segment {
    int r, kvh, m0, columns, tok0, start, hi, lo, kept, t_begin, t_end;
    int slot;               // where the partial result goes; -1: it is the whole
    bool first;             // begins with the list's first tile
};

// Columns m0 .. of a request: what they see, as a list of tiles.
__device__ __forceinline__ int fill(Segment& w, const Problem& a, int cols) {
    const int G = a.nq / a.nkv, n_q = (int)min((long long)a.cu_q[w.r + 1], a.tokens) - a.cu_q[w.r];
    w.tok0 = a.cu_q[w.r];
    w.start = a.q_start[w.r];
    w.columns = n_q * G;
    w.hi = w.start + min(n_q - 1, (w.m0 + cols - 1) / G);
    w.lo = first_visible(w.start + w.m0 / G, a.window);
    w.kept = kept_tiles<KV4_TILE>(w.lo, a.keep);
    return w.kept + w.hi / KV4_TILE - w.lo / KV4_TILE + 1;
}

// Tiles that one column of request ``r`` sees, where requests bring one token each (0 for one that brings none).
__device__ __forceinline__ int tiles_of(const Problem& a, int r) {
    if (r >= a.requests || min((long long)a.cu_q[r + 1], a.tokens) <= a.cu_q[r]) return 0;
    const int pos = a.q_start[r], lo = first_visible(pos, a.window);
    const int seen = kept_tiles<KV4_TILE>(lo, a.keep) + pos / KV4_TILE - lo / KV4_TILE + 1, held = a.bt_stride * (a.ps / KV4_TILE);
    if (seen > held && a.status) atomicOr(a.status, FE_STATUS_BAD_PAGE);
    return max(1, min(seen, held));
}

// Blocks that are resident on an SM: the registers are cut to that.  16-bit queries at head size 128: four blocks of 128 registers a thread (three of 168
// take the same time for long rows and leave fewer blocks to short ones).
template <typename TQ, int NG> __host__ __device__ constexpr int blocks_an_sm() { return sizeof(TQ) == 2 && NG <= 4 ? 4 : 2; }

// TQ: queries and output; 32-bit ones in two parts.  NG: groups of a row.
//
// SHARED = false: grid (column tiles x splits, heads, requests), the splits of a column tile a thread-block cluster, each with an equal share of its
// tiles; their results are merged through distributed shared memory: no second kernel.
// SHARED = true, where every request brings one token: the tiles of all (request, head, column tile) items, one after the other, are cut into as many
// equal shares as there are blocks, whole rounds of the block's warps each; a block then takes the pieces of items that its share holds.  So
// lengths that differ leave no block without work (a split of every item into equal parts left a seventh of the time to the last
// blocks), and nothing on the host depends on them.  A block's share ends at most one item that others began and begins at
// most one that others end: its partial results are 2 b (an item begun before) and 2 b + 1 (an item begun here).  ``part``: [blocks][2][COLS]
// [32 NG + 4] floats (numbers, maximum, sum), then for each item which blocks hold it.
struct Held { int from, to; };      // blocks from .. to - 1; one block: it wrote the result itself
template <int NG> __host__ __device__ constexpr int part_floats() { return COLS * (32 * NG + 4); }

template <typename TQ, int NG, bool SHARED>
__global__ void __launch_bounds__(WARPS * 32, blocks_an_sm<TQ, NG>())
kv4_attention_kernel(const Problem a) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int PARTS = sizeof(TQ) == 4 ? 2 : 1;
    constexpr bool EXACT = PARTS == 2;                   // scales and centres of values in 32 bits
    constexpr int GONE = 0x40000000;                     // a key that nobody sees
    constexpr int TILE = kv4_tile_bytes(NG);
    constexpr unsigned FULL = 0xffffffffu;
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(8) unsigned long long bars[WARPS][STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int G = a.nq / a.nkv;
    if (lane < STAGES) mbar_init(&bars[warp][lane], 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    __syncwarp();

    // ---- what this block does; each warp keeps the piece in hand in shared memory, for the registers' sake
    __shared__ Segment pieces_of[WARPS];
    __shared__ __align__(16) uint4 operands[PARTS][NG][32];           // of the queries; the four warps make them together and read them as they go
    __shared__ __align__(8) float2 lifts[NG][32];
    __shared__ int last_keys[COLS], first_keys[COLS];
    Segment& w = pieces_of[warp];
    Segment found{};
    constexpr int ROUND = PAIR * WARPS;
    int share_end = 0, share = 1, item_tiles = 0, item_at = 0;          // SHARED: in tiles of all items, one after the other
    const int columns_each = (G + COLS - 1) / COLS, items_each = a.nkv * columns_each;      // of a request
    if (SHARED) {
        const int mine = tiles_of(a, lane);                             // of the first 32 requests: asked for once
        int total = __reduce_add_sync(FULL, mine);
        for (int base = 32; base < a.requests; base += 32) total += __reduce_add_sync(FULL, tiles_of(a, base + lane));
        total *= items_each;                                            // fewer than 2^31: asked of the sizes before the launch
        share = ((total + (int)gridDim.x - 1) / (int)gridDim.x + ROUND - 1) / ROUND * ROUND;
        const int begin = min(total, (int)blockIdx.x * share);
        share_end = min(total, begin + share);
        if (begin >= share_end) return;
        // the request that holds tile ``begin``, from running sums
        int before = 0;
        found.r = -1;
        for (int base = 0; base < a.requests && found.r < 0; base += 32) {
            const int n = (base == 0 ? mine : tiles_of(a, base + lane)) * items_each;
            int upto = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(FULL, upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned here = __ballot_sync(FULL, begin >= before + upto - n && begin < before + upto);
            if (here) {
                const int at = __ffs(here) - 1;
                found.r = base + at;
                item_tiles = __shfl_sync(FULL, n, at) / items_each;
                before += __shfl_sync(FULL, upto - n, at);
            } else
                before += __shfl_sync(FULL, upto, 31);
        }
        const int item = (begin - before) / item_tiles;
        item_at = before + item * item_tiles;
        found.kvh = item / columns_each;
        found.m0 = item % columns_each * COLS;
        fill(found, a, COLS);
        found.t_begin = begin - item_at;
        found.t_end = min(item_tiles, share_end - item_at);
        found.slot = found.t_end - found.t_begin == item_tiles ? -1 : 2 * (int)blockIdx.x + (found.t_begin == 0);
    } else {
        found.r = blockIdx.z;
        found.kvh = blockIdx.y;
        const int n_q = (int)min((long long)a.cu_q[found.r + 1], a.tokens) - a.cu_q[found.r];
        // the last columns walk the most keys: first
        found.m0 = ((n_q * G + COLS - 1) / COLS - 1 - (int)(blockIdx.x / a.splits)) * COLS;
        if (found.m0 < 0 || n_q <= 0) return;                           // the whole cluster
        const int all = fill(found, a, COLS), split = (int)(blockIdx.x % a.splits);
        const int each = ((all + a.splits - 1) / a.splits + ROUND - 1) / ROUND * ROUND;
        found.t_begin = min(all, split * each);
        found.t_end = min(all, found.t_begin + each);
        found.slot = a.splits > 1 ? 0 : -1;
    }
    if (lane == 0) w = found;
    __syncwarp();
    // the next item of the share: its tiles may be those of another request
    auto next = [&](Segment n) {
        item_at += item_tiles;
        if (!SHARED || item_at >= share_end) return false;
        n.m0 += COLS;
        if (n.m0 >= G) {
            n.m0 = 0;
            if (++n.kvh == a.nkv) {
                n.kvh = 0;
                do item_tiles = tiles_of(a, ++n.r); while (item_tiles == 0 && n.r < a.requests);      // the share ends inside a request that has some
            }
        }
        fill(n, a, COLS);
        n.t_begin = 0;
        n.t_end = min(item_tiles, share_end - item_at);
        n.slot = n.t_end == item_tiles ? -1 : 2 * (int)blockIdx.x + 1;
        __syncwarp();
        if (lane == 0) w = n;
        __syncwarp();
        return true;
    };

    const int even = 2 * t + (t & 1), odd = 2 * t + 1 - (t & 1);      // tokens of rows 2t and 2t + 1 (and of 2t + 8, 2t + 9: 8 on)
    const int key_row = (g & ~1) + ((g & 1) ^ (g >> 1 & 1));          // token of row g
    const int key_codes = key_row * 16 * NG + t * 4 * NG, key_pairs = kv4_key_pairs(NG) + key_row * 4 * NG;
    const int even_codes = kv4_value_codes(NG) + even * 16 * NG + g * 2 * NG, odd_codes = kv4_value_codes(NG) + odd * 16 * NG + g * 2 * NG;
    const int per_page = a.ps / KV4_TILE;
    unsigned char* ring = smem + warp * STAGES * PAIR * TILE;
    __shared__ int result_place[WARPS];
    auto results_of = [&](int w) { return reinterpret_cast<float*>(smem + (w * STAGES + (SHARED ? result_place[w] : 0)) * PAIR * TILE); };
    unsigned stage = 0, parity = 0;
    bool gone = false;

    // ---- where the tiles lie: a lane each for 32 of the warp's tiles at a time.  The warp's pairs of tiles are places t_begin + 2 warp,
    // t_begin + 2 (warp + WARPS), ... of the list and the one after each
    auto pairs_of = [&](const Segment& w) { return max(0, (w.t_end - w.t_begin - PAIR * warp + PAIR * WARPS - 1) / (PAIR * WARPS)); };
    int at = -1;                                         // of this lane's tile of the batch whose copies are being started: its number in the cache
    unsigned here_now = 0, here_before = 0;              // which of that batch's and of the one before are in the cache
    auto look_up = [&](const Segment& w, int batch) {
        const int place = w.t_begin + PAIR * (warp + WARPS * (16 * batch + (lane >> 1))) + (lane & 1);
        at = -1;
        if (place < w.t_end) {
            const int tile = listed_tile<KV4_TILE>(place, w.kept, w.lo);
            const int page = tile / per_page < a.bt_stride ? a.block_table[(long long)w.r * a.bt_stride + tile / per_page] : -1;
            if (page < 0 || page >= a.num_pages) {
                if (a.status) atomicOr(a.status, FE_STATUS_BAD_PAGE);
            } else
                at = (page * a.nkv + w.kvh) * per_page + tile % per_page;
        }
        here_before = here_now;
        here_now = __ballot_sync(FULL, at >= 0);
    };
    auto begin_copy = [&](const Segment& w, unsigned k, unsigned stage) {
        if ((k & 15) == 0) look_up(w, k >> 4);
        const int first = __shfl_sync(FULL, at, 2 * (k & 15)), second = __shfl_sync(FULL, at, 2 * (k & 15) + 1);
        if (lane == 0) {
            const unsigned bar = smem_u32(&bars[warp][stage]), to = smem_u32(ring + stage * PAIR * TILE);
            // a tile that is not there brings nothing; the stage's turn passes all the same
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(bar), "r"((first >= 0 ? TILE : 0) + (second >= 0 ? TILE : 0) + a.waits.lacking) : "memory");
            if (first >= 0) copy_tile(to, a.cache + (long long)first * TILE, TILE, bar);
            if (second >= 0) copy_tile(to + TILE, a.cache + (long long)second * TILE, TILE, bar);
        }
    };
    int mine = pairs_of(w);
    if (mine > 0) begin_copy(w, 0, stage);

    for (bool more = true; more;) {
        const int m0 = w.m0, columns = w.columns, tok0 = w.tok0, start = w.start, kvh = w.kvh, lo = w.lo, kept = w.kept, t_begin = w.t_begin, t_end = w.t_end, slot = w.slot;

        // ---- the queries as B operands, a column each; thread (g, t) holds numbers 32 i + 8 t .. + 7 of column g
        // Keys' codes are multiplied raised (by 1024 or 64: kv4_raise) where queries are 16-bit; ``lift`` is what that adds to a group's partial
        // score, and eight codes' worth more, with the sign turned: the sums begin there.  That costs their last bits: with |q| in [1, 2) a sum
        // reaches some 10,000 where signs are mixed and 66,000 where 32 numbers have one sign, in steps of 2^-10 and 2^-7.  Results are then off by
        // 0.00168 of their norm where rounding them to bfloat16 is 0.00160 (one sign, scores tens apart; otherwise by less).  (Values are summed over all keys,
        // where the part of 1024 would grow: they are decoded in full, and so are keys under 32-bit queries.)
        constexpr bool RAISED = PARTS == 1;
        unsigned qsum[2];                                // (high, low) of the sums over group t, and over group t + 4
        float factor[2];                                 // takes a score of columns 2t, 2t + 1 to log2 units
        float below[2], l[2];                        // minus the reference point (infinite before the first key), the sum
        int last_least = 0x7fffffff, first_most = 0;
        const int c = m0 + g;
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
        float group_sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) { v[i][e] *= down; sum += v[i][e]; }
            sum += __shfl_xor_sync(FULL, sum, 1);
            sum += __shfl_xor_sync(FULL, sum, 2);
            if (i == t) group_sum[0] = sum;
            if (i == t + 4) group_sum[1] = sum;
            if (i % WARPS != warp) continue;                          // the other warps make the other groups' operands
            unsigned high[4], rest[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                high[e] = pack(v[i][e], v[i][e + 4]);
                if (PARTS == 2) rest[e] = pack_rest(v[i][e], v[i][e + 4], high[e]);
            }
            operands[0][i][lane] = make_uint4(high[0], high[1], high[2], high[3]);
            if (PARTS == 2) operands[PARTS - 1][i][lane] = make_uint4(rest[0], rest[1], rest[2], rest[3]);
            float raised = 0.f;
            if (RAISED) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    raised -= ((e & 1 ? KV4_RAISED_ODD : KV4_RAISED_EVEN) + 8.f) * (low_half(high[e]) + high_half(high[e]));
                raised += __shfl_xor_sync(FULL, raised, 1);
                raised += __shfl_xor_sync(FULL, raised, 2);
            }
            lifts[i][lane] = make_float2(__shfl_sync(FULL, raised, 8 * t), __shfl_sync(FULL, raised, 8 * t + 4));      // of columns 2t and 2t + 1
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const float high = __half2float(__float2half_rn(group_sum[h]));
            qsum[h] = pack(high, group_sum[h] - high);
        }
        // a padding column sees what the last query sees: it is computed and never written, and must not make a tile a masked one
        const int pos = real ? start + c / G : w.hi, from = real ? first_visible(pos, a.window) : lo;
        last_least = min(last_least, pos);
        first_most = max(first_most, from);
        if (warp == 0 && t == 0) { last_keys[g] = pos; first_keys[g] = from; }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            factor[h] = a.scale_log2 * __uint_as_float((unsigned)(127 + __shfl_sync(FULL, e2, (2 * t + h) * 4)) << 23);
            below[h] = CUDART_INF_F;
            l[h] = 0.f;
            if (a.sink && t_begin == 0 && warp == 0) {
                below[h] = 0.f;
                l[h] = g == 0 ? 1.f : 0.f;            // the lanes of a column add their sums up at the end
            }
        }
        last_least = __reduce_min_sync(FULL, last_least);
        first_most = __reduce_max_sync(FULL, first_most);
        __syncthreads();

        float o[NG][2][4], oc[NG][2];                // sums over codes (EXACT) or numbers, 16 a tile, and over centres (EXACT, this thread's tokens)
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            oc[i][0] = oc[i][1] = 0.f;
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][0][e] = o[i][1][e] = 0.f;
        }

        // places [clear_from, clear_to) of the list are seen whole by every column (kept tiles are taken with the masked)
        const int clear_from = kept + (first_most + KV4_TILE - 1) / KV4_TILE - lo / KV4_TILE;
        const int clear_to = min(t_end, kept + (last_least + 1) / KV4_TILE - lo / KV4_TILE);
        unsigned poisoned = 0;                                            // bit 2 i + h: column 2t + h has seen a NaN in group i of the values
        // a pair of tiles; ``place``: of the first in the list; ``here``: which of the two were brought
        auto take = [&](auto masked_tag, const unsigned char* pair, int place, unsigned here) {
            constexpr bool MASKED = decltype(masked_tag)::value;
            // ---- scores of tokens key_row and key_row + 8 of each tile by columns 2t, 2t + 1
            float s[PAIR][4];
#pragma unroll
            for (int u = 0; u < PAIR; ++u) {
                const unsigned char* tile = pair + u * TILE;
                const unsigned char* pairs = tile + key_pairs;
                unsigned c0 = 0, c1 = 0, c2 = 0, c3 = 0;                  // (centre, centre) of group t, and of group t + 4
                if (NG >= 4 || t < NG) {
                    const unsigned w0 = *reinterpret_cast<const unsigned*>(pairs + t * 4);
                    const unsigned w1 = *reinterpret_cast<const unsigned*>(pairs + t * 4 + 32 * NG);
                    c0 = __byte_perm(w0, w0, 0x3232); c1 = __byte_perm(w1, w1, 0x3232);
                }
                if (NG > 4 && t + 4 < NG) {
                    const unsigned w0 = *reinterpret_cast<const unsigned*>(pairs + t * 4 + 16);
                    const unsigned w1 = *reinterpret_cast<const unsigned*>(pairs + t * 4 + 16 + 32 * NG);
                    c2 = __byte_perm(w0, w0, 0x3232); c3 = __byte_perm(w1, w1, 0x3232);
                }
                mma_from(s[u], c0, c1, c2, c3, qsum[0], NG > 4 ? qsum[1] : 0u, 0.f, 0.f);
                unsigned k0[NG], k1[NG], p0[NG], p1[NG];
                words<NG>(tile + key_codes, k0);
                words<NG>(tile + key_codes + 128 * NG, k1);
                words<NG>(pairs, p0);
                words<NG>(pairs + 32 * NG, p1);
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    unsigned n0[4], n1[4];
                    if (RAISED) { kv4_raise(k0[i], n0); kv4_raise(k1[i], n1); }
                    else { kv4_decode(k0[i], n0); kv4_decode(k1[i], n1); }
                    const float s0 = low_half(p0[i]), s1 = low_half(p1[i]);
                    float part[4];
                    const uint4 q = operands[0][i][lane];
                    const float2 lift = RAISED ? lifts[i][lane] : make_float2(0.f, 0.f);
                    mma_from(part, n0[0], n1[0], n0[1], n1[1], q.x, q.y, lift.x, lift.y);
                    mma(part, n0[2], n1[2], n0[3], n1[3], q.z, q.w);
                    if (PARTS == 2) {
                        const uint4 rest = operands[PARTS - 1][i][lane];
                        mma(part, n0[0], n1[0], n0[1], n1[1], rest.x, rest.y);
                        mma(part, n0[2], n1[2], n0[3], n1[3], rest.z, rest.w);
                    }
                    s[u][0] = fmaf(s0, part[0], s[u][0]);
                    s[u][1] = fmaf(s0, part[1], s[u][1]);
                    s[u][2] = fmaf(s1, part[2], s[u][2]);
                    s[u][3] = fmaf(s1, part[3], s[u][3]);
                }
            }
            // ---- weights
            unsigned v0[PAIR][NG], v1[PAIR][NG];                          // EXACT: (scale, centre) of the two tokens' value groups
            float up0[PAIR], up1[PAIR], y[PAIR][4];
            bool grows = false;
#pragma unroll
            for (int u = 0; u < PAIR; ++u) {
                up0[u] = up1[u] = 0.f;
                if (EXACT || MASKED) {
                    words<NG>(pair + u * TILE + key_pairs + 64 * NG, v0[u]);
                    words<NG>(pair + u * TILE + key_pairs + 96 * NG, v1[u]);
                }
                if (MASKED) {
                    const int key0 = (here >> u & 1u) ? listed_tile<KV4_TILE>(place + u, kept, lo) * KV4_TILE : GONE;
                    unsigned nan0 = 0, nan1 = 0;                          // groups that read as NaN
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        if ((v0[u][i] & 0x7c00u) == 0x7c00u) { nan0 |= 1u << (2 * i); v0[u][i] = 0; }
                        if ((v1[u][i] & 0x7c00u) == 0x7c00u) { nan1 |= 1u << (2 * i); v1[u][i] = 0; }
                        if (key0 + key_row > w.hi) v0[u][i] = 0;          // behind the last token: what lies there may be anything
                        if (key0 + key_row + 8 > w.hi) v1[u][i] = 0;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = key0 + key_row + (e & 2) * 4;
                        const int column = 2 * t + (e & 1);
                        if (!(key <= last_keys[column] && (key >= first_keys[column] || key < a.keep))) s[u][e] = -CUDART_INF_F;
                        else poisoned |= (e < 2 ? nan0 : nan1) << (e & 1);
                    }
                }
                if (EXACT) {
                    float big0 = low_half(v0[u][0]), big1 = low_half(v1[u][0]);
#pragma unroll
                    for (int i = 1; i < NG; ++i) { big0 = fmaxf(big0, low_half(v0[u][i])); big1 = fmaxf(big1, low_half(v1[u][i])); }
                    // their exponents; zeros and subnormal numbers count as 2^-24, the least scale there is
                    up0[u] = fmaxf((float)(__float_as_uint(big0) >> 23) - 127.f, -24.f);
                    up1[u] = fmaxf((float)(__float_as_uint(big1) >> 23) - 127.f, -24.f);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[u][e] = fmaf(s[u][e], factor[e & 1], below[e & 1]);
                    grows |= y[u][e] > MOVE_STEP - (e < 2 ? up0[u] : up1[u]);
                }
            }
            if (__any_sync(FULL, grows)) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    float mx = -CUDART_INF_F;
#pragma unroll
                    for (int u = 0; u < PAIR; ++u)
                        mx = fmaxf(mx, fmaxf(fmaf(s[u][h], factor[h], up0[u]), fmaf(s[u][h + 2], factor[h], up1[u])));
#pragma unroll
                    for (int off = 4; off < 32; off <<= 1) mx = fmaxf(mx, __shfl_xor_sync(FULL, mx, off));
                    const float to = fmaxf(-below[h], mx);
                    const float by = to == -CUDART_INF_F ? 1.f : ex2(-below[h] - to);      // 2^-inf = 0 at the start
                    below[h] = -to;
                    l[h] *= by;
#pragma unroll
                    for (int i = 0; i < NG; ++i) {
                        if (EXACT) oc[i][h] *= by;
                        o[i][0][h] *= by; o[i][0][h + 2] *= by;
                        o[i][1][h] *= by; o[i][1][h + 2] *= by;
                    }
#pragma unroll
                    for (int u = 0; u < PAIR; ++u) {
                        y[u][h] = fmaf(s[u][h], factor[h], -to);
                        y[u][h + 2] = fmaf(s[u][h + 2], factor[h], -to);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < PAIR; ++u) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y[u][e] = ex2(y[u][e]);
                    if (MASKED && s[u][e] == -CUDART_INF_F) y[u][e] = 0.f;      // a column that has seen nothing yet has no reference point
                }
                l[0] += y[u][0] + y[u][2];
                l[1] += y[u][1] + y[u][3];
            }
            // ---- values: tokens even, odd (+ 8) in pairs; numbers 32 i + 4 g .. + 3
#pragma unroll
            for (int u = 0; u < PAIR; ++u) {
                constexpr int VW = (NG + 1) / 2;
                unsigned ve[VW], vo[VW], ve8[VW], vo8[VW];
                const unsigned char* tile = pair + u * TILE;
                pieces<NG>(tile + even_codes, ve);
                pieces<NG>(tile + odd_codes, vo);
                pieces<NG>(tile + even_codes + 128 * NG, ve8);
                pieces<NG>(tile + odd_codes + 128 * NG, vo8);
                // EXACT = false: one operand of weights for all groups, and scale and centre in the decoded numbers, which half precision rounds by 2^-12
                unsigned pe[NG], po[NG], pe8[NG], po8[NG], b0, b1;
                if (!EXACT) {
                    const unsigned char* pairs = tile + kv4_value_pairs(NG);
                    words<NG>(pairs + even * 4 * NG, pe);
                    words<NG>(pairs + odd * 4 * NG, po);
                    words<NG>(pairs + even * 4 * NG + 32 * NG, pe8);
                    words<NG>(pairs + odd * 4 * NG + 32 * NG, po8);
                    if (MASKED) {
                        const int key0 = (here >> u & 1u) ? listed_tile<KV4_TILE>(place + u, kept, lo) * KV4_TILE : GONE;
#pragma unroll
                        for (int i = 0; i < NG; ++i) {
                            if ((pe[i] & 0x7c00u) == 0x7c00u || key0 + even > w.hi) pe[i] = 0;
                            if ((po[i] & 0x7c00u) == 0x7c00u || key0 + odd > w.hi) po[i] = 0;
                            if ((pe8[i] & 0x7c00u) == 0x7c00u || key0 + even + 8 > w.hi) pe8[i] = 0;
                            if ((po8[i] & 0x7c00u) == 0x7c00u || key0 + odd + 8 > w.hi) po8[i] = 0;
                        }
                    }
                    b0 = transposed(pack(y[u][0], y[u][1]));
                    b1 = transposed(pack(y[u][2], y[u][3]));
                }
#pragma unroll
                for (int i = 0; i < NG; ++i) {
                    unsigned na[4], nb[4];
                    kv4_decode(__byte_perm(ve[i / 2], vo[i / 2], (i & 1) ? 0x7632 : 0x5410), na);
                    kv4_decode(__byte_perm(ve8[i / 2], vo8[i / 2], (i & 1) ? 0x7632 : 0x5410), nb);
                    if constexpr (!EXACT) {
                        times_plus(na, __byte_perm(pe[i], po[i], 0x5410), __byte_perm(pe[i], po[i], 0x7632));
                        times_plus(nb, __byte_perm(pe8[i], po8[i], 0x5410), __byte_perm(pe8[i], po8[i], 0x7632));
                        mma(o[i][0], na[0], na[1], nb[0], nb[1], b0, b1);
                        mma(o[i][1], na[2], na[3], nb[2], nb[3], b0, b1);
                    } else {
                        const float s0 = low_half(v0[u][i]), s1 = low_half(v1[u][i]), c0 = high_half(v0[u][i]), c1 = high_half(v1[u][i]);
                        const float* w = y[u];
                        oc[i][0] = fmaf(w[0], c0, fmaf(w[2], c1, oc[i][0]));
                        oc[i][1] = fmaf(w[1], c0, fmaf(w[3], c1, oc[i][1]));
                        const unsigned w0 = pack(w[0] * s0, w[1] * s0), w1 = pack(w[2] * s1, w[3] * s1);
                        const unsigned h0 = transposed(w0), h1 = transposed(w1);
                        const unsigned r0 = transposed(pack_rest(w[0] * s0, w[1] * s0, w0)), r1 = transposed(pack_rest(w[2] * s1, w[3] * s1, w1));
                        // A tile's products begin at zero and are added by the CUDA cores: the tensor cores' sums are cut off, not rounded,
                        // and kept there over 32,768 keys they were off by 9.8e-6 of the result's norm (so 1.8e-7; 8 x 2,048 keys take 13.3 us instead of 13.1)
                        float first[4], second[4];
                        mma_from(first, na[0], na[1], nb[0], nb[1], h0, h1, 0.f, 0.f);
                        mma_from(second, na[2], na[3], nb[2], nb[3], h0, h1, 0.f, 0.f);
                        mma(first, na[0], na[1], nb[0], nb[1], r0, r1);
                        mma(second, na[2], na[3], nb[2], nb[3], r0, r1);
#pragma unroll
                        for (int e = 0; e < 4; ++e) { o[i][0][e] += first[e]; o[i][1][e] += second[e]; }
                    }
                }
            }
        };
#pragma unroll 1
        for (unsigned k = 0; k < (unsigned)mine && !gone; ++k) {
            if (k + 1 < (unsigned)mine) begin_copy(w, k + 1, stage ^ 1);
            if (__any_sync(FULL, !wait_for(&bars[warp][stage], parity, a.waits.limit))) {
                // the row lacks these keys: said in the status word.  Copies on their way are waited for once more before results go where
                // they may still land, or the block leaves
                gone = true;
                if (lane == 0 && a.status) atomicOr(a.status, FE_STATUS_WAIT_EXPIRED);
                wait_for(&bars[warp][stage], parity, a.waits.limit);
                if (k + 1 < (unsigned)mine) wait_for(&bars[warp][stage ^ 1], parity ^ stage, a.waits.limit);
                break;
            }
            // the batch of pair k is that of the newest copy or the one before
            const unsigned newest = min((unsigned)mine - 1, k + 1) >> 4;
            const unsigned here = ((k >> 4) == newest ? here_now : here_before) >> (2 * (k & 15)) & 3u;
            const unsigned char* pair = ring + stage * PAIR * TILE;
            const int place = t_begin + PAIR * (warp + WARPS * (int)k);
            if (here == 3u && place >= clear_from && place + 1 < clear_to) take(std::false_type{}, pair, place, here);
            else take(std::true_type{}, pair, place, here);
            __syncwarp();                                                 // the stage is free: the next turn's copy goes there
            parity ^= stage;
            stage ^= 1;
        }
        // the next piece's first tiles are on their way while this one's results are put together
        const int item_last = item_at + item_tiles - 1, item = (w.r * a.nkv + kvh) * columns_each + m0 / COLS;
        more = next(w);
        if (more && !gone) {
            mine = pairs_of(w);
            if (mine > 0) begin_copy(w, 0, stage);
        }

        // ---- the warp's sums over its lanes, then the four warps' results side by side: [warp][column][32 NG numbers, maximum, sum]
        constexpr int ROW = 32 * NG + 4;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int off = 4; off < 32; off <<= 1) {
                l[h] += __shfl_xor_sync(FULL, l[h], off);
                if (!EXACT) continue;                                 // no sums over centres: it only brings NaN
#pragma unroll
                for (int i = 0; i < NG; ++i) oc[i][h] += __shfl_xor_sync(FULL, oc[i][h], off);
            }
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) poisoned |= __shfl_xor_sync(FULL, poisoned, off);
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int h = 0; h < 2; ++h)
                if (poisoned >> (2 * i + h) & 1u) oc[i][h] = CUDART_NAN_F;
        if (SHARED && lane == 0) result_place[warp] = (int)(stage ^ 1);
        __syncwarp();
        float* mine_results = results_of(warp);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float* to = mine_results + (2 * t + h) * ROW;
#pragma unroll
            for (int i = 0; i < NG; ++i)
                *reinterpret_cast<float4*>(to + 32 * i + 4 * g) =
                    make_float4(o[i][0][h] + oc[i][h], o[i][0][h + 2] + oc[i][h], o[i][1][h] + oc[i][h], o[i][1][h + 2] + oc[i][h]);
            if (g == 0) { to[32 * NG] = -below[h]; to[32 * NG + 1] = l[h]; }
        }
        __syncthreads();
        for (int c = warp; c < COLS && m0 + c < columns; c += WARPS) {
            const int mc = m0 + c, token = tok0 + mc / G, head = kvh * G + mc % G;
            const float* from[WARPS];
            float top = -CUDART_INF_F;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                from[w] = results_of(w) + c * ROW;
                top = fmaxf(top, from[w][32 * NG]);
            }
            float by[WARPS], sum = 0.f;
#pragma unroll
            for (int w = 0; w < WARPS; ++w) {
                const float mw = from[w][32 * NG];
                by[w] = mw == -CUDART_INF_F ? 0.f : ex2(mw - top);
                sum += by[w] * from[w][32 * NG + 1];
            }
            const bool whole = slot < 0;
            const float inv = !whole ? 1.f : sum > 0.f ? 1.f / sum : 0.f;
            float* part = whole ? nullptr : SHARED ? a.part + ((long long)slot * COLS + c) * ROW : results_of(0) + c * ROW;      // in place: see below
            __syncwarp();                                             // maxima and sums are read
            TQ* to = static_cast<TQ*>(a.out) + (long long)token * a.out_stride + (long long)head * a.d;
            for (int i = lane; i < a.d; i += 32) {
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) v += by[w] * from[w][i];      // 0 times NaN is NaN, as where one warp has all keys; who saw nothing left zeros
                if (whole) put<TQ>(to + i, sum != sum ? sum : v * inv);
                else part[i] = v;
            }
            if (!whole && lane == 0) { part[32 * NG] = top; part[32 * NG + 1] = sum; }
        }
        if (!SHARED && a.splits > 1) {
            // A column's sums lie where those of the first warp's were (a thread overwrote what it had read); the cluster's blocks take
            // every splits-th column, and add the splits in their order.
            const unsigned splits = a.splits, rank = blockIdx.x % a.splits;
            cluster_barrier();
            for (int c = rank + splits * warp; c < COLS && m0 + c < columns; c += splits * WARPS) {
                const int mc = m0 + c, token = tok0 + mc / G, head = kvh * G + mc % G;
                const float* own = results_of(0) + c * ROW;
                const float at = lane < (int)splits ? ld_cluster(own + 32 * NG, lane) : -CUDART_INF_F;
                const float top = warp_max(at), by = at == -CUDART_INF_F ? 0.f : ex2(at - top);
                const float sum = warp_sum(lane < (int)splits ? by * ld_cluster(own + 32 * NG + 1, lane) : 0.f);
                for (int i0 = 0; i0 < a.d; i0 += 32) {
                    const int i = i0 + lane;
                    float v = 0.f;
                    for (unsigned p = 0; p < splits; ++p) {
                        const float weight = __shfl_sync(FULL, by, p);
                        if (i < a.d) v += weight * ld_cluster(own + i, p);
                    }
                    if (i < a.d) put<TQ>(static_cast<TQ*>(a.out) + (long long)token * a.out_stride + (long long)head * a.d + i, sum != sum ? sum : sum > 0.f ? v / sum : 0.f);
                }
            }
            cluster_barrier();                                        // nobody leaves while its shared memory may still be read
        }
        if (SHARED && t_begin == 0 && threadIdx.x == 0) {
            // which blocks hold this item
            Held* held = reinterpret_cast<Held*>(a.part + (long long)gridDim.x * 2 * part_floats<NG>());
            const int b = (int)blockIdx.x;
            held[item] = Held{b, slot < 0 ? b + 1 : item_last / share + 1};
        }
        asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory");     // copies may go where results were written
        __syncthreads();                                                  // the results are read: the next piece's go there
    }
}

constexpr int MAX_SPLITS = 8;            // blocks of a cluster
constexpr int MERGE_THREADS = 256;

// A block per (head, request): what several blocks hold of an item is weighted by their maxima and added.  Sets of threads, four numbers of
// the head a thread, take every sets-th part, AHEAD parts on their way at once, with a running maximum of their own; the sets are
// added in their order.
template <typename TQ, int NG>
__global__ void __launch_bounds__(MERGE_THREADS)
kv4_merge_kernel(const Problem a, int blocks) {
    griddep_wait();
    griddep_launch_dependents();
    constexpr int ROW = 32 * NG + 4, SETS = MERGE_THREADS / (8 * NG), AHEAD = 8;
    __shared__ __align__(16) float sums[SETS][ROW];
    const int r = blockIdx.y, head = blockIdx.x, G = a.nq / a.nkv, kvh = head / G, m = head % G;
    const int token = a.cu_q[r], behind = a.cu_q[r + 1];
    const Held held = reinterpret_cast<const Held*>(a.part + (long long)blocks * 2 * part_floats<NG>())[(r * a.nkv + kvh) * ((G + COLS - 1) / COLS) + m / COLS];
    if (min((long long)behind, a.tokens) <= token) return;
    const int n = held.to - held.from;
    if (n <= 1) return;
    const int set = threadIdx.x / (8 * NG), i = threadIdx.x % (8 * NG) * 4;
    if (set < SETS) {
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        float top = -CUDART_INF_F, sum = 0.f;
        for (int s0 = set; s0 < n; s0 += AHEAD * SETS) {
            float4 x[AHEAD];
            float2 end[AHEAD];
            float most = top;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                const int s = s0 + u * SETS;
                x[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                end[u] = make_float2(-CUDART_INF_F, 0.f);
                if (s < n) {
                    // the first block's part is of the item that it began, the others' of the one they found begun
                    const float* from = a.part + ((long long)(2 * (held.from + s) + (s == 0)) * COLS + m % COLS) * ROW;
                    end[u] = *reinterpret_cast<const float2*>(from + 32 * NG);
                    x[u] = *reinterpret_cast<const float4*>(from + i);
                }
            }
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                most = fmaxf(most, end[u].x);
                // a part without a maximum has seen no key, and its sum is 0, or scores that are all NaN: then it is NaN, and so is the row
                if (end[u].x == -CUDART_INF_F) sum += end[u].y;
            }
            if (most == -CUDART_INF_F) continue;
            const float by = ex2(top - most);
            top = most;
            sum *= by;
            v.x *= by; v.y *= by; v.z *= by; v.w *= by;
#pragma unroll
            for (int u = 0; u < AHEAD; ++u) {
                if (end[u].x == -CUDART_INF_F) continue;             // its numbers are not looked at
                const float w = ex2(end[u].x - most);
                sum += w * end[u].y;
                v.x += w * x[u].x; v.y += w * x[u].y; v.z += w * x[u].z; v.w += w * x[u].w;
            }
        }
        *reinterpret_cast<float4*>(&sums[set][i]) = v;
        if (i == 0) { sums[set][32 * NG] = top; sums[set][32 * NG + 1] = sum; }
    }
    __syncthreads();
    if (threadIdx.x < a.d) {
        float top = -CUDART_INF_F, sum = 0.f, v = 0.f;
        for (int k = 0; k < SETS; ++k) top = fmaxf(top, sums[k][32 * NG]);
        for (int k = 0; k < SETS; ++k) {
            const float at = sums[k][32 * NG], by = at == -CUDART_INF_F ? 0.f : ex2(at - top);
            sum += by * sums[k][32 * NG + 1];
            v += by * sums[k][threadIdx.x];
        }
        put<TQ>(static_cast<TQ*>(a.out) + (long long)token * a.out_stride + (long long)head * a.d + threadIdx.x, sum != sum ? sum : sum > 0.f ? v / sum : 0.f);
    }
}

// Blocks of the kernel that the device holds at once (asked of the driver once per device).
template <typename TQ, int NG> int resident() {
    static int cached[64];
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
    if (cached[device] == 0) {
        int each = 0;
        constexpr int smem = smem_bytes<NG>();
        cudaFuncSetAttribute(kv4_attention_kernel<TQ, NG, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&each, kv4_attention_kernel<TQ, NG, true>, WARPS * 32, smem) != cudaSuccess || each < 1) {
            cudaGetLastError();
            each = 1;
        }
        cached[device] = each * fe_sm_count();
    }
    return cached[device];
}

struct Launch {
    const Problem* a;
    int requests, column_tiles, blocks;
    cudaStream_t stream;
};

template <typename TQ, int NG> int run(const Launch& w) {
    constexpr int smem = smem_bytes<NG>();
    const Problem& a = *w.a;
    auto kernel = w.blocks ? kv4_attention_kernel<TQ, NG, true> : kv4_attention_kernel<TQ, NG, false>;
    FE_REQUIRE(fe_allow_smem((const void*)kernel, smem), "paged_attention_kv4: no kernel with %d bytes of shared memory", smem);
    const dim3 grid = w.blocks ? dim3((unsigned)w.blocks) : dim3((unsigned)(w.column_tiles * a.splits), (unsigned)a.nkv, (unsigned)w.requests);
    if (!w.blocks && a.splits > 1) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = grid;
        cfg.blockDim = dim3(WARPS * 32);
        cfg.dynamicSmemBytes = smem;
        cfg.stream = w.stream;
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = a.splits;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        const cudaError_t launched = cudaLaunchKernelEx(&cfg, kernel, a);
        FE_REQUIRE(launched == cudaSuccess, "paged_attention_kv4 (clusters of %d): %s", a.splits, cudaGetErrorString(launched));
    } else
        fe::launch(kernel, grid, WARPS * 32, smem, w.stream, a);
    if (const int rc = fe_check_launch("paged_attention_kv4")) return rc;
    if (!w.blocks) return 0;
    fe::launch_as(FE_PDL_ELEMENTWISE, kv4_merge_kernel<TQ, NG>, dim3((unsigned)a.nq, (unsigned)w.requests), MERGE_THREADS, 0, w.stream, a, w.blocks);
    return fe_check_launch("paged_attention_kv4 merge");
}

// f(groups of a row as a constant)
template <typename F> auto with_groups(int d, F f) {
    switch (kv4_groups(d)) {
        case 1: return f(std::integral_constant<int, 1>{});
        case 2: return f(std::integral_constant<int, 2>{});
        case 3: return f(std::integral_constant<int, 3>{});
        case 4: return f(std::integral_constant<int, 4>{});
        case 5: return f(std::integral_constant<int, 5>{});
        case 6: return f(std::integral_constant<int, 6>{});
        case 7: return f(std::integral_constant<int, 7>{});
        default: return f(std::integral_constant<int, 8>{});
    }
}
bool head_size_ok(int d) { return d >= 16 && d % 16 == 0 && d <= KV4_MAX_DIM; }

}  // namespace

// How a decode step's tiles are dealt out: a positive number is that of the blocks that share the tiles of all items; a negative one, -S, a cluster of S
// blocks for each item.  ``tiles``: of the longest request.
//
// The least of what each way is expected to take.  A block takes 6.8 us and, at head size 128, 0.115 for each tile that it walks, 0.07 n where n > 1 of them
// are on its multiprocessor (and 1.7 more); a cluster 1.1 to 2 more; blocks beyond those that fit at once come after them.  Sharing out costs 15 us (running
// sums over the requests, pieces of two items in a block, a second kernel) and 0.12 for each request, and is no faster where all requests are as long as the longest, but
// lengths that differ leave no block without work: its tiles are taken as three quarters of that.  28/4 heads of 128, microseconds, one block, clusters of 2, 4
// and 8, shared: 64 requests of 512 keys 11 15 23 42 21; 64 of 1,101 19 22 32 52 34; 48 of 2,101 29 25 33 46 34; 8 of 2,049 23 17 14 14 19; 1 of
// 8,301 70 40 25 18 17; 64 of 8,192 92 84 91 106 87; 64 of 1,024 to 8,191 84 74 71 88 64.  Head sizes other than 128 are taken in proportion to their groups of 32.
// A captured step keeps the plan of the length it was captured for: at 32,768, 64 requests of 512 keys take 20 instead of 10.4.
extern "C" int fe_kv4_attention_plan(int requests, int tiles, int nq, int nkv, int d, int dtype) {
    if (!head_size_ok(d) || requests <= 0 || nq <= 0 || nkv <= 0) return -1;
    const long long items = (long long)requests * nkv * ((nq / nkv + 7) / 8), all = items * tiles;
    if (tiles <= 2 * WARPS * PAIR) return -1;
    const long long most = dtype == FE_F32 ? with_groups(d, [](auto n) { return resident<float, n.value>(); }) : with_groups(d, [](auto n) { return resident<bf16, n.value>(); });
    const int sms = fe_sm_count(), round = WARPS * PAIR;
    const double tile = kv4_groups(d) / 4.0 * (dtype == FE_F32 ? 1.1 : 1.0);
    auto walk = [&](long long blocks, long long each) {          // of so many tiles by each of the blocks on the device
        const long long beside = (blocks + sms - 1) / sms;
        return 6.8 + (beside > 1 ? 1.7 : 0.0) + (double)((each + round - 1) / round * round) * tile * (beside > 1 ? 0.07 * (double)beside : 0.115);
    };
    double least = 1e30;
    int plan = -1;
    for (int S = 1; S <= MAX_SPLITS; S *= 2) {
        if (S > 1 && S * round > tiles + round - 1) break;
        const long long at_once = most / S * S, waves = at_once > 0 ? (items * S + at_once - 1) / at_once : 1LL << 20;
        const double t = (double)waves * (walk(items * S < at_once ? items * S : at_once, (tiles + S - 1) / S) + (S == 1 ? 0.0 : S == 2 ? 1.1 : S == 4 ? 1.3 : 2.0));
        if (t < least) { least = t; plan = -S; }
    }
    if (all < (1LL << 31)) {
        const long long want = (all + 2 * round - 1) / (2 * round), blocks = want < most ? want : most;
        const double share = (double)all * (requests > 1 ? 0.75 : 1.0) / (double)blocks;
        if (walk(blocks, (long long)share) + 8.2 + 0.12 * requests < least) plan = (int)blocks;
    }
    return plan;
}

// Bytes of ``scratch`` for so many blocks.
extern "C" long long fe_kv4_attention_scratch_bytes(int blocks, int requests, int nq, int nkv, int d) {
    if (blocks <= 0 || nkv <= 0) return 0;
    return (long long)blocks * 2 * 8 * (32 * kv4_groups(d) + 4) * 4 + (long long)requests * nkv * ((nq / nkv + 7) / 8) * (long long)sizeof(Held);
}

// q [tokens, >= nq d], rows ``q_stride`` elements apart; out likewise; dtype of both.  ``blocks`` > 0 (from fe_kv4_attention_plan; every request
// brings one token at most) needs scratch.
extern "C" int fe_paged_attention_kv4(const void* q, long long q_stride, void* out, long long out_stride, const void* cache, const int* block_table,
                                      int bt_stride, const int* cu_q, const int* q_start, int requests, long long tokens, int max_q_len, int nq,
                                      int nkv, int d, int ps, int num_pages, float scale, int window, int keep, int sink, int splits, int blocks, void* scratch,
                                      int dtype, int* status, cudaStream_t stream) {
    FE_REQUIRE(nq > 0 && nkv > 0 && nq % nkv == 0 && nkv <= 65535, "paged_attention_kv4: bad head counts %d/%d", nq, nkv);
    FE_REQUIRE(head_size_ok(d), "paged_attention_kv4: head size %d; multiples of 16 up to %d", d, KV4_MAX_DIM);
    FE_REQUIRE(ps > 0 && ps % KV4_TILE == 0 && num_pages > 0 && bt_stride > 0, "paged_attention_kv4: page size %d (a multiple of %d) or page count", ps, KV4_TILE);
    FE_REQUIRE(q_stride % 8 == 0 && (((size_t)q | (size_t)out | (size_t)cache) & 15) == 0, "paged_attention_kv4: rows must start on 16-byte boundaries");
    FE_REQUIRE(requests >= 0 && requests <= 65535 && max_q_len >= 0 && tokens >= 0, "paged_attention_kv4: bad request count or length");
    FE_REQUIRE(window >= 0 && keep >= 0 && (keep == 0 || window > 0), "paged_attention_kv4: a window is not negative, kept keys go with one");
    FE_REQUIRE(blocks >= 0 && (blocks == 0 || (max_q_len <= 1 && scratch && ((size_t)scratch & 15) == 0)), "paged_attention_kv4: %d blocks", blocks);
    FE_REQUIRE((long long)num_pages * nkv * (ps / KV4_TILE) < (1LL << 31), "paged_attention_kv4: %d pages are too many", num_pages);
    FE_REQUIRE(splits >= 1 && splits <= MAX_SPLITS && (splits == 1 || blocks == 0), "paged_attention_kv4: %d splits; 1 to %d", splits, MAX_SPLITS);
    FE_REQUIRE((long long)max_q_len * (nq / nkv) * splits < (1LL << 31) - 64, "paged_attention_kv4: grid too large");
    FE_REQUIRE(blocks == 0 || (long long)requests * nkv * ((nq / nkv + 7) / 8) * bt_stride * (ps / KV4_TILE) < (1LL << 31), "paged_attention_kv4: too many tiles to share out");
    FE_REQUIRE(dtype == FE_F32 || dtype == FE_BF16, "paged_attention_kv4: unknown type %d", dtype);
    if (requests == 0 || max_q_len == 0 || tokens == 0) return 0;
    const Problem a{q, q_stride, out, out_stride, (const unsigned char*)cache, block_table, bt_stride, cu_q, q_start, requests, nq, nkv, d, ps, num_pages,
                    scale * LOG2E, window, keep, sink, splits, (float*)scratch, tokens, status, fe_waits()};
    const Launch w{&a, requests, (int)(((long long)max_q_len * (nq / nkv) + 7) / 8), blocks, stream};
    return dtype == FE_F32 ? with_groups(d, [&](auto n) { return run<float, n.value>(w); }) : with_groups(d, [&](auto n) { return run<bf16, n.value>(w); });
}

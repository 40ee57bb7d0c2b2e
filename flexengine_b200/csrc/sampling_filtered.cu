// Drawing from logits with temperature, top-k, top-p and min-p, from given uniform numbers.
//
// x = logits / T.  Of a row's tokens, largest logit first and the lower index first among equals, the first k stay (k > 0); of their masses
// e^(x - max) those stay before which less than top_p of the sum lies (top_p < 1; the first always stays); and of these the ones whose mass is at
// least min_p of the largest.  The token is the first, in index order, at which the running sum of the masses that stayed passes u times their
// sum.  T = 0: the lowest index of the maximum.  NaN counts as -inf.  Beside the token: its probability among those that stayed, and their number.
//
// Masses are whole numbers of 2^-44 of the largest (fewer bits over 2^18 tokens), so their sums are exact in any order: the result depends neither
// on the number of blocks a row has nor on what else is in the batch.
//
// A row belongs to a thread-block cluster, each block with a contiguous part of it.  Sorting is avoided.  A walk finds the maximum; a second one
// counts the tokens (for top-k) and adds up their masses to 13 bits (for top-p) by their distance to the maximum, in 4,096 steps of 1/128.  In
// the step at which the count or the mass passes its limit a few hundred tokens are left to be looked at one by one.  If that step and all
// before it hold no more than LIST tokens (small k, peaked rows), they are listed and the rest of the work is done on the list, each token
// against each other.  Else one more walk adds up exactly what lies before the step and lists the step itself; a step with more tokens than the list
// takes (equal logits, as 16-bit ones often are) is taken apart by the bits of the logits.  The masses that stay are added up by
// segments of the row, in the walk of the cut or one of their own, and the segment in which the target falls is gone through once more.
//
// Bound by the walks' integer work and, for one row, by the chain of barriers and trips between blocks; 1,024 threads have 64 registers each, and 1,344 bytes
// a thread are spilled (2,064 of loads).  64 rows of 152,064 (39 MB, read once 5.9 us), by what
// the rows ask for: the maximum alone 8 us, no limits 32, k = 50 46, top-p 0.9 75 to 88, k = 20,000 and top-p 119, a mixture 86; one row of the mixture
// 38 in a cluster of 8 blocks.
#include <math_constants.h>

#define FE_PDL_CLASS 8      // FE_PDL_SAMPLING
#include "common.cuh"
#include "cut.cuh"

using namespace fe;

namespace {

typedef unsigned long long u64;

constexpr int THREADS = 1024, WARPS = THREADS / 32;
constexpr int SEGMENTS = 256;
constexpr int MAX_CLUSTER = 8;
constexpr int STEPS = 4096;
constexpr float STEPS_A_UNIT = 128.f;
constexpr float FARTHEST = 32.f;              // STEPS / STEPS_A_UNIT: a mass beyond is below 2^-46 of the largest, and counts as nothing
constexpr int COARSE_BITS = 13;               // of a token's mass in the second walk, against that of its step
constexpr int LIST = 2048;
constexpr int BATCH = 5;                      // 16-byte loads of a lane on their way at once

__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;\n" ::: "memory");
}
__device__ __forceinline__ unsigned peer_address(const void* own, unsigned rank) {
    unsigned remote;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;\n" : "=r"(remote) : "r"((unsigned)__cvta_generic_to_shared(own)), "r"(rank));
    return remote;
}
// the same variable in the shared memory of block ``rank`` of this cluster
__device__ __forceinline__ unsigned ld_peer(const void* own, unsigned rank) {
    unsigned v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];\n" : "=r"(v) : "r"(peer_address(own, rank)) : "memory");
    return v;
}
__device__ __forceinline__ u64 ld_peer64(const void* own, unsigned rank) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];\n" : "=l"(v) : "r"(peer_address(own, rank)) : "memory");
    return v;
}
__device__ __forceinline__ uint4 ld_peer4(const void* own, unsigned rank) {
    uint4 v;
    asm volatile("ld.shared::cluster.v4.u32 {%0, %1, %2, %3}, [%4];\n" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(peer_address(own, rank)) : "memory");
    return v;
}
// order-preserving map from float to unsigned
__device__ __forceinline__ unsigned ordered_key(float v) {
    const unsigned b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float sanitize(float v) { return v != v ? -CUDART_INF_F : v + 0.f; }      // -0 and 0 are equal: one key
__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

struct Rows {
    const float* logits;
    long long ld;
    int V;
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int* tokens;
    float* probability;
    int* kept;
    int mass_bits;              // masses are whole numbers of 2^-mass_bits of the largest
};

constexpr int ROOTS = 256;                    // 2^(-i / 256) in a table

struct Shared {
    unsigned counts[STEPS], coarse[STEPS];             // tokens of a step, and their masses
    u64 fine[STEPS];                                   // exact masses where a step is taken apart
    u64 list[LIST];                                    // this block's: ordered key turned over, then the index
    u64 all[LIST];                                     // the row's; sorted: the largest logit first, the lower index first among equals
    u64 all_mass[LIST];
    u64 all_before[LIST];                              // mass of the tokens before it
    u64 segment_mass[SEGMENTS];                        // this block's segments
    int segment_ties[SEGMENTS];
    u64 row_mass[SEGMENTS + 1];
    int row_ties[SEGMENTS];
    u64 warp_mass[WARPS];
    unsigned warp_count[WARPS];
    u64 own_mass, own_mass2;
    unsigned own_count, own_low, own_high;
    float own_max;
    int own_index, listed;
    u64 found_mass;
    unsigned found_count;
    int found_at;
    long long roots[ROOTS];
    unsigned char held[THREADS];
};

// What a row's masses are made of.  A mass is a whole number, rounded down, right to 2^-32 of itself: where logits are equal, as 16-bit ones
// often are, thousands of tokens have the same one, and an error of a 32-bit exponential would come thousands of times.  It is 2^(z - z_max),
// z = log2(e) logit / T, from a table of the 256th roots of 2 and a polynomial between them (Tang's table-driven exponential): z 256 = n + r, and only the
// differences of n and of r to the maximum's count.  |r| <= 1/2 is what one rounding of a multiply-add leaves of an exact product, so it is right to 2^-25
// of itself, 2^-33 of z; the polynomial gives 2^-(difference of r) - 1, below 2^-8, as a whole number of 2^-32; the table has 62 bits.
// Logits themselves are multiplied while z_max is below 2^13; beyond, all that has a mass lies within a factor of two of the maximum, and what is
// multiplied is the difference to it, which then is exact.  (In 64-bit floating point, or with rounded differences and products kept in two parts,
// a walk over 64 rows of 152,064 took 40 us; this 20, bound by the integer pipe: two or three dozen instructions a token.)
struct Mass {
    float top, over;                         // the maximum, 1 / T
    float base;                              // 0 or the maximum
    float steps, steps_rest;                 // log2(e) / T and what it lacks
    float rest;                              // the maximum's r / 256
    float least;                             // logits below have less than one unit of mass
    float counted;                           // logits from here on count as kept: as many as have a probability at all, however small (e^-x in 64 bits is above zero up to 745)
    int whole;                               // the maximum's n + 256 (62 - bits)
    const long long* roots;                  // shared memory: 2^62 2^(-i / ROOTS)
    static constexpr float MAGIC = 49152.f;  // 1.5 2^15: adding it rounds to whole 256ths
    __device__ __forceinline__ void set(float most, float heat, int bits, const long long* table) {
        top = most;
        roots = table;
        heat = fmaxf(heat, 1e-36f);                              // so that log2(e) / T is finite
        over = 1.f / heat;
        const double exact = isinf(most) ? 0. : 1.44269504088896340736 / (double)heat;        // an infinite maximum: all of them weigh 1, the rest nothing
        steps = (float)exact;
        steps_rest = (float)(exact - (double)steps);
        base = fabsf(most) * steps < 8192.f ? 0.f : fminf(most, CUDART_MAX_NORMAL_F);
        // (an infinite temperature: all but -inf weigh the same)
        least = isinf(most) ? most : fmaxf(__double2float_ru((double)most - bits * 0.69314718055994530942 * (double)heat), -CUDART_MAX_NORMAL_F);
        counted = isinf(most) ? most : fmaxf((float)((double)most - 745. * (double)heat), -CUDART_MAX_NORMAL_F);
        whole = 0;
        rest = 0.f;
        int n;
        float r;
        split(most, n, r);
        whole = ROOTS * (62 - bits) - n;
        rest = -r;
    }
    __device__ __forceinline__ void split(float v, int& less, float& r) const {
        const float w = fminf(v, CUDART_MAX_NORMAL_F) - base, t = fmaf(w, steps, MAGIC);
        less = whole - __float_as_int(t);
        r = rest - fmaf(w, steps_rest, fmaf(w, steps, MAGIC - t));
    }
    __device__ __forceinline__ float distance(float v) const { return v == top ? 0.f : (top - v) * over; }      // infinite maxima too
    __device__ __forceinline__ u64 of(float v) const {
        int n;
        float r;                                                 // 256 y = n + 256 r, the mass 2^-y; |r| <= 2^-8
        split(v, n, r);
        constexpr float L = 0.69314718f, SCALE = 4294967296.f;                 // 2^32
        const float z = r * fmaf(r, fmaf(r, -SCALE * L * L * L / 6.f, SCALE * L * L / 2.f), -SCALE * L);       // 2^32 (2^-r - 1)
        const long long root = roots[n & (ROOTS - 1)];
        const u64 m = (u64)(root + (long long)__float2int_rn(z) * (long long)(int)(root >> 32));
        return !(v >= least) ? 0 : m >> (n / ROOTS & 63);
    }
};
__device__ __forceinline__ int step_of(float far) { return far < FARTHEST ? (int)(far * STEPS_A_UNIT) : STEPS; }

// f(logit, index) for the tokens [from, to); RAW: as they stand, for what takes NaN and -0 as it should of itself
template <bool RAW = false, typename F> __device__ __forceinline__ void over_segment(const float* x, int from, int to, bool vector, F f) {
    const int lane = threadIdx.x & 31;
    auto clean = [](float v) { return RAW ? v : sanitize(v); };
    if (vector) {
        for (int base = from; base < to; base += 128 * BATCH) {
            float4 v[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int i = base + 128 * u + 4 * lane;
                if (i < to) v[u] = *reinterpret_cast<const float4*>(x + i);
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int i = base + 128 * u + 4 * lane;
                if (i < to) { f(clean(v[u].x), i); f(clean(v[u].y), i + 1); f(clean(v[u].z), i + 2); f(clean(v[u].w), i + 3); }
            }
        }
    } else {
        for (int base = from; base < to; base += 32 * BATCH) {
            float v[BATCH];
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int i = base + 32 * u + lane;
                if (i < to) v[u] = x[i];
            }
#pragma unroll
            for (int u = 0; u < BATCH; ++u) {
                const int i = base + 32 * u + lane;
                if (i < to) f(clean(v[u]), i);
            }
        }
    }
}

// Sums over the block; every thread gets the result.
__device__ __forceinline__ u64 block_sum64(u64 v, Shared& s) {
    v = warp_sum64(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_mass[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum64(s.warp_mass[threadIdx.x & 31]);
}
__device__ __forceinline__ unsigned block_sum32(unsigned v, Shared& s) {
    v = __reduce_add_sync(0xffffffffu, v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) s.warp_count[threadIdx.x >> 5] = v;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, s.warp_count[threadIdx.x & 31]);
}
// What threads before this one hold; ``total`` what all do.
__device__ __forceinline__ u64 block_before64(u64 v, u64& total, Shared& s) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    u64 upto = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += up;
    }
    __syncthreads();
    if (lane == 31) s.warp_mass[warp] = upto;
    __syncthreads();
    const u64 w = s.warp_mass[lane];
    u64 all = w;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 up = __shfl_up_sync(0xffffffffu, all, o);
        if (lane >= o) all += up;
    }
    total = __shfl_sync(0xffffffffu, all, 31);
    return __shfl_sync(0xffffffffu, all - w, warp) + upto - v;
}

// Sorts a[0 .. n) upwards, n <= LIST (a bitonic network over the next power of two; places from n on are taken as the largest).
__device__ __forceinline__ void sort_list(u64* a, int n) {
    int size = 2;
    while (size < n) size <<= 1;
    for (int i = n + threadIdx.x; i < size; i += THREADS) a[i] = ~0ull;
    __syncthreads();
    for (int k = 2; k <= size; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            const int i = (threadIdx.x & ~(j - 1)) * 2 + (threadIdx.x & (j - 1));      // LIST / 2 threads' worth of pairs
            if (i + j < size) {
                const u64 x = a[i], y = a[i + j];
                if ((x > y) == ((i & k) == 0)) { a[i] = y; a[i + j] = x; }
            }
            // a warp's pairs are of its own 64 entries as long as they lie 32 apart at most
            if (j > 32 || (j == 1 && k > 32)) __syncthreads();
            else __syncwarp();
        }
    __syncthreads();
}
static_assert(LIST == 2 * THREADS, "a pair a thread");

__global__ void __launch_bounds__(THREADS, 1)
sample_filtered_kernel(const Rows of, const int C) {
    griddep_wait();
    griddep_launch_dependents();
    extern __shared__ __align__(16) unsigned char raw[];
    Shared& s = *reinterpret_cast<Shared*>(raw);
    const int row = blockIdx.x / C, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const unsigned rank = blockIdx.x % C;
    const float* x = of.logits + (long long)row * of.ld;
    const int V = of.V, S = ((V + SEGMENTS - 1) / SEGMENTS + 31) / 32 * 32;
    const int per_block = SEGMENTS / C, per_warp = per_block / WARPS, first_segment = (int)rank * per_block + warp * per_warp;
    const bool vector = (V & 3) == 0 && ((size_t)x & 15) == 0;
    bool by_segments = false;                              // the segments' sums are there already
    unsigned number_all = 0;                               // this thread's tokens that stay
    u64 mass_all = 0;                                      // and their mass
    // f(logit, index) over this block's part; a warp takes its segments one after the other
    auto walk = [&](auto f) {
        for (int j = 0; j < per_warp; ++j)
            over_segment<true>(x, min((long long)V, (long long)(first_segment + j) * S), min((long long)V, (long long)(first_segment + j + 1) * S), vector, f);
    };

    struct Sums { u64 mass; unsigned number; };
    // the same; f(logit, index, sums) adds up what stays, a segment at a time
    auto walk_segments = [&](auto f) {
        number_all = 0;
        mass_all = 0;
        for (int j = 0; j < per_warp; ++j) {
            Sums here{0, 0};
            over_segment<true>(x, min((long long)V, (long long)(first_segment + j) * S), min((long long)V, (long long)(first_segment + j + 1) * S), vector,
                         [&](float v, int i) { f(v, i, here); });
            mass_all += here.mass;
            here.mass = warp_sum64(here.mass);
            if (lane == 0) s.segment_mass[warp * per_warp + j] = here.mass;
            number_all += here.number;
        }
    };

    if (tid < ROOTS) s.roots[tid] = __double2ll_rn(exp2(62.0 - (double)tid / ROOTS));
    // ---- the maximum and its lowest index
    float best = -CUDART_INF_F;
    int best_at = 0x7fffffff;
    walk([&](float v, int i) { if (v > best) { best = v; best_at = i; } });        // a lane meets its indices in rising order
    auto take = [&](float v, int i) { if (v > best || (v == best && i < best_at)) { best = v; best_at = i; } };
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) take(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_at, o));
    if (lane == 0) { s.warp_mass[warp] = (u64)__float_as_uint(best) << 32 | (unsigned)best_at; }
    __syncthreads();
    if (warp == 0) {
        const u64 w = s.warp_mass[lane];
        best = __uint_as_float((unsigned)(w >> 32));
        best_at = (int)(unsigned)w;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) take(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_at, o));
        if (lane == 0) { s.own_max = best; s.own_index = best_at; s.listed = 0; }
    }
    cluster_sync();
    best = lane < C ? __uint_as_float(ld_peer(&s.own_max, lane)) : -CUDART_INF_F;      // a lane a block: one trip, not one after the other
    best_at = lane < C ? (int)ld_peer(&s.own_index, lane) : 0x7fffffff;
#pragma unroll
    for (int o = MAX_CLUSTER / 2; o > 0; o >>= 1) take(__shfl_xor_sync(0xffffffffu, best, o), __shfl_xor_sync(0xffffffffu, best_at, o));
    const float top = __shfl_sync(0xffffffffu, best, 0);
    const int top_at = __shfl_sync(0xffffffffu, best_at, 0);
    const float heat = of.temperature[row];
    if (!(heat > 0.f) || top == -CUDART_INF_F) {
        // greedy, or a row that leaves nothing: then the lowest index, with no probability
        const bool none = top == -CUDART_INF_F;
        if (rank == 0 && tid == 0) {
            of.tokens[row] = none ? 0 : top_at;
            of.probability[row] = none ? 0.f : 1.f;
            of.kept[row] = none ? 0 : 1;
        }
        cluster_sync();                                    // no block leaves while another may still read its maximum
        return;
    }
    Mass mass;
    mass.set(top, heat, of.mass_bits, s.roots);
    const int k = of.top_k[row];
    const bool use_k = k > 0 && k < V;
    const float p = fmaxf(of.top_p[row], 1e-30f), least = of.min_p[row];      // the first token always stays
    const bool use_p = p < 1.f;
    // min_p as a logit: mass >= min_p of the largest, so v >= top + T ln min_p, taken in 64 bits and rounded up
    float low_logit = -CUDART_INF_F;
    if (least > 0.f) low_logit = least >= 1.f ? top : isinf(top) ? top : __double2float_ru((double)top + (double)heat * log((double)least));

    unsigned thr = 0, need = 0;                            // what stays: keys above thr, and the first ``need`` of those equal to it
    bool all_ties = true;                                  // all that are equal to it
    // adds up two 64-bit numbers and a 32-bit one over the cluster (s.own_mass, s.own_mass2 and s.own_count are free)
    auto cluster_sum = [&](u64& m, u64& m2, unsigned& n) {
        m = block_sum64(m, s);
        m2 = block_sum64(m2, s);
        n = block_sum32(n, s);
        if (tid == 0) { s.own_mass = m; s.own_mass2 = m2; s.own_count = n; }
        cluster_sync();
        m = warp_sum64(lane < C ? ld_peer64(&s.own_mass, lane) : 0);
        m2 = warp_sum64(lane < C ? ld_peer64(&s.own_mass2, lane) : 0);
        n = __reduce_add_sync(0xffffffffu, lane < C ? ld_peer(&s.own_count, lane) : 0);
        cluster_sync();
    };

    if (use_k || use_p) {
        // ---- counts and masses by steps
        for (int i = tid; i < STEPS; i += THREADS) { s.counts[i] = 0; s.coarse[i] = 0; }
        __syncthreads();
        walk([&](float v, int) {
            const float far = mass.distance(v);
            const int step = step_of(far);
            if (step >= STEPS) return;
            if (use_k) atomicAdd(&s.counts[step], 1u);
            if (use_p) {
                // e^-(distance inside the step), the step 1/128 long: two terms of the series are good to 1e-7
                const float in = far - (float)step * (1.f / STEPS_A_UNIT);
                atomicAdd(&s.coarse[step], (unsigned)__float2int_rn((1.f - in * (1.f - 0.5f * in)) * (float)(1 << COARSE_BITS)));
            }
        });
        cluster_sync();
        // the row's steps, four a thread; the same in every block
        unsigned count[4];
        u64 coarse[4], flat[4], own_coarse = 0;           // flat: as if every token of a step weighed the same
        u64 own_count = 0;
        auto all_blocks = [&](const unsigned* own, u64* sum) {         // of four steps; all blocks' are asked for at once
            uint4 v[MAX_CLUSTER];
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c) v[c] = c < C ? ld_peer4(own, c) : make_uint4(0, 0, 0, 0);
            sum[0] = sum[1] = sum[2] = sum[3] = 0;
#pragma unroll
            for (int c = 0; c < MAX_CLUSTER; ++c) { sum[0] += v[c].x; sum[1] += v[c].y; sum[2] += v[c].z; sum[3] += v[c].w; }
        };
        // More than two blocks: each adds up its share of the steps (8 blocks: 2 x 16 KB to read instead of 8; one row 9 us less), the sums fit 32 bits
        const int share = STEPS / C;
        if (C > 2) {
            if (4 * tid < share) {
                u64 sum[4];
                const int at = (int)rank * share + 4 * tid;
                auto add_up = [&](unsigned* own) {
                    all_blocks(own, sum);
                    *reinterpret_cast<uint4*>(own) = make_uint4((unsigned)sum[0], (unsigned)sum[1], (unsigned)sum[2], (unsigned)sum[3]);
                };
                if (use_k) add_up(&s.counts[at]);
                if (use_p) add_up(&s.coarse[at]);
            }
            cluster_sync();
        }
        auto of_row = [&](const unsigned* own, u64* sum) {
            if (C <= 2) return all_blocks(own, sum);
            const uint4 v = ld_peer4(own, (unsigned)(4 * tid / share));
            sum[0] = v.x, sum[1] = v.y, sum[2] = v.z, sum[3] = v.w;
        };
        {
            u64 sum[4] = {0, 0, 0, 0};
            if (use_k) of_row(&s.counts[4 * tid], sum);
#pragma unroll
            for (int e = 0; e < 4; ++e) { count[e] = (unsigned)sum[e]; own_count += sum[e]; flat[e] = 0; }
        }
        if (use_p) of_row(&s.coarse[4 * tid], flat);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            coarse[e] = use_p ? __float2ull_rn((float)flat[e] * expf(-(float)(4 * tid + e) * (1.f / STEPS_A_UNIT)) * 65536.f) : 0;
            own_coarse += coarse[e];
        }
        // bit e: step 4 tid + e holds a token (a mass is 2^COARSE_BITS (1 - 1/128) at least); kept by its own thread, in shared memory for the registers' sake
        unsigned occupied = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) occupied |= (unsigned)(count[e] > 0 || flat[e] > 0) << e;
        s.held[tid] = (unsigned char)occupied;
        u64 all_count, all_coarse;
        const u64 count_before = block_before64(own_count, all_count, s);
        const u64 coarse_before = block_before64(own_coarse, all_coarse, s);
        // the first step at which a running sum reaches ``limit``, the last one that holds anything if none does
        auto step_at = [&](const auto* each, u64 before, u64 all, double limit) {
            if (tid == 0) s.found_at = -1;
            __syncthreads();
            u64 run = before;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const u64 upto = run + each[e];
                if (each[e] > 0 && (double)run < limit && ((double)upto >= limit || upto == all)) s.found_at = 4 * tid + e;
                run = upto;
            }
            __syncthreads();
            const int at = s.found_at;
            __syncthreads();
            return at;
        };
        auto listed_up_to = [&](int step) {                // tokens up to the step, from the counts
            if (tid == step / 4) {
                u64 run = count_before;
                for (int e = 0; e <= step % 4; ++e) run += count[e];
                s.found_mass = run;
            }
            __syncthreads();
            const u64 n = s.found_mass;
            __syncthreads();
            return n;
        };
        auto key_of = [](u64 entry) { return ~(unsigned)(entry >> 32); };
        auto logit_of = [](unsigned key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); };
        // the lowest logit of a step up to ``step``: what the steps' own arithmetic says, found among all floats, 32 at a time
        auto floor_of = [&](int step) {
            if (step >= STEPS) return -CUDART_INF_F;
            if (step < 0) return CUDART_INF_F;
            unsigned above = ordered_key(top), below = 0;              // step_of <= step at ``above``, not at ``below``
            while (above - below > 1) {
                const unsigned part = (above - below - 1) / 32 + 1, key = above - below > part * lane ? above - part * lane : below;
                const float v = logit_of(key);
                const int good = __popc(__ballot_sync(0xffffffffu, key > below && step_of(mass.distance(v)) <= step));
                above -= part * (good - 1);
                if (good < 32 && above - below > part) below = above - part;
            }
            return logit_of(above);
        };
        // Puts the tokens of steps [from, to] into the row's list, in every block; false when they do not fit.  ``above`` and ``above_count``:
        // exact sums of the steps before, ``everything`` of all steps (only where top-p is of the whole row), ``low`` and ``high`` the least and the
        // greatest key in them.
        const bool of_whole = use_p && !use_k;
        u64 above = 0, everything = 0;
        unsigned above_count = 0, low = 0, high = 0;
        int n = 0;
        auto list = [&](int from, int to) {
            if (tid == 0) s.listed = 0;
            __syncthreads();
            above = everything = 0;
            above_count = 0;
            unsigned least_key = 0xffffffffu, most_key = 0;
            const float floor_to = floor_of(to), floor_above = from > 0 ? floor_of(from - 1) : CUDART_INF_F, floor_kept = fmaxf(floor_above, low_logit);
            const bool none_above = from == 0, all_listed = to >= STEPS, min_p_bites = floor_kept > floor_above;      // min-p takes some of them away
            const bool masses = of_whole || !none_above;
            walk_segments([&](float v, int i, Sums& here) {
                const bool over = v >= floor_above && !none_above, stays = v >= floor_kept && !none_above;
                if (masses) {                              // whichever it is: one way for all lanes
                    const u64 own = mass.of(v);
                    here.mass += stays ? own : 0;
                    everything += own;
                    if (min_p_bites) above += over && !stays ? own : 0;
                }
                here.number += stays;
                if (min_p_bites) above_count += over && !stays;
                if (over || !(v >= floor_to || all_listed)) return;
                const unsigned key = ordered_key(sanitize(v));
                least_key = min(least_key, key);
                most_key = max(most_key, key);
                const int at = atomicAdd(&s.listed, 1);
                if (at < LIST) s.list[at] = (u64)~key << 32 | (unsigned)i;
            });
            least_key = __reduce_min_sync(0xffffffffu, least_key);
            most_key = __reduce_max_sync(0xffffffffu, most_key);
            if (tid == 0) { s.own_low = 0xffffffffu; s.own_high = 0; }
            __syncthreads();
            if (lane == 0) { atomicMin(&s.own_low, least_key); atomicMax(&s.own_high, most_key); }
            above += mass_all;
            above_count += number_all;
            cluster_sum(above, everything, above_count);         // barriers inside: lists and keys are there
            int here = lane < C ? (int)ld_peer(&s.listed, lane) : 0, upto = here;
            low = __reduce_min_sync(0xffffffffu, lane < C ? ld_peer(&s.own_low, lane) : 0xffffffffu);
            high = __reduce_max_sync(0xffffffffu, lane < C ? ld_peer(&s.own_high, lane) : 0u);
#pragma unroll
            for (int o = 1; o < MAX_CLUSTER; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += up;
            }
            const int total_listed = __shfl_sync(0xffffffffu, upto, C - 1);
            if (total_listed <= LIST) {
                // entry i of the row is of the block in whose share of the running sums it lies
                const int most = (total_listed + 31) & ~31;
                for (int i = tid; i < most; i += THREADS) {
                    int block = 0, first = 0;
#pragma unroll
                    for (int c = 0; c < MAX_CLUSTER - 1; ++c) {
                        const int end = __shfl_sync(0xffffffffu, upto, c);
                        if (c < C - 1 && i >= end) { block = c + 1; first = end; }
                    }
                    if (i < total_listed) s.all[i] = ld_peer64(&s.list[i - first], block);
                }
            }
            n = total_listed;
            cluster_sync();                                // the peers' lists are read
            return n <= LIST;
        };
        // The list in order, every token's mass and the mass before it.
        auto rank_list = [&]() {
            sort_list(s.all, n);
            u64 m[2], nothing64;
#pragma unroll
            for (int e = 0; e < 2; ++e) m[e] = 2 * tid + e < n ? mass.of(logit_of(key_of(s.all[2 * tid + e]))) : 0;
            const u64 before = block_before64(m[0] + m[1], nothing64, s);
#pragma unroll
            for (int e = 0; e < 2; ++e) { s.all_mass[2 * tid + e] = m[e]; s.all_before[2 * tid + e] = before + (e ? m[0] : 0); }
            __syncthreads();
        };

        const int step_k = use_k ? step_at(count, count_before, all_count, (double)k) : -1;
        const int step_p = use_p && !use_k ? step_at(coarse, coarse_before, all_coarse, (double)p * (double)all_coarse) : -1;
        // where k reaches beyond the last step, the long way takes what lies there as one step more
        const bool k_bites = use_k && all_count >= (u64)k;
        // whether everything up to the limit's step may fit the list: known from the counts, or (top-p alone) likely from the masses
        bool fits = false;
        int last = -1;
        if (k_bites) { last = step_k; fits = listed_up_to(step_k) <= LIST; }
        else if (use_p && !use_k) {
            // a step's tokens have nearly the same mass: its number of them is its coarse mass over the full one
            u64 own = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * tid + e <= step_p) own += flat[e];
            last = step_p;
            fits = (block_sum64(own, s) >> COARSE_BITS) < LIST - LIST / 16;
        }
        cluster_sync();                                    // the peers' steps are read: they may be overwritten
        if (fits && list(0, last)) {
            rank_list();
            // what stays of the list: a place below k, less than p of the sum before it
            const int reach = k_bites ? k : n;             // the list holds k tokens at least
            const u64 in_list = s.all_before[reach - 1] + s.all_mass[reach - 1], sum = k_bites ? in_list : everything;
            const double limit = (double)p * (double)sum;
            // the coarse sums may have chosen a step too early: the list then does not reach the limit, and the long way is taken
            if (k_bites || (double)in_list >= limit) {
                u64 kept_mass = 0;
                unsigned kept_count = 0;
                for (int i = tid; i < n; i += THREADS) {
                    const bool stays = i < reach && (!use_p || i == 0 || (double)s.all_before[i] < limit) && logit_of(key_of(s.all[i])) >= low_logit;
                    if (stays) { kept_mass += s.all_mass[i]; ++kept_count; }
                }
                kept_mass = block_sum64(kept_mass, s);
                kept_count = block_sum32(kept_count, s);   // a token stays with all that are ahead of it: the first so many
                if (rank == 0) {
                    // the tokens that stay by index, each with its place
                    for (int i = tid; i < (int)kept_count; i += THREADS) s.list[i] = s.all[i] << 32 | (unsigned)i;
                    __syncthreads();
                    sort_list(s.list, (int)kept_count);
                    u64 m[2], nothing64;
#pragma unroll
                    for (int e = 0; e < 2; ++e) m[e] = 2 * tid + e < (int)kept_count ? s.all_mass[(unsigned)s.list[2 * tid + e]] : 0;
                    u64 before = block_before64(m[0] + m[1], nothing64, s);
                    const float u = of.uniform[row];
                    double target = (u > 0.f ? (double)fminf(u, 1.f) : 0.0) * (double)kept_mass;
                    if (target >= (double)kept_mass) target = nextafter((double)kept_mass, 0.0);
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        if (m[e] > 0 && (double)before <= target && target < (double)(before + m[e])) {
                            of.tokens[row] = (int)(s.list[2 * tid + e] >> 32);
                            of.probability[row] = (float)((double)m[e] / (double)kept_mass);
                            of.kept[row] = (int)kept_count;
                        }
                        before += m[e];
                    }
                }
                return;                                    // no block reads another's memory any more
            }
        }
        // ---- the long way: one limit after the other, each an exact cut (thr, need)
        // ``limit`` in tokens or in mass, or (of_whole) the mass's share of the row's; ``at``: the step that is likely to hold it
        // the next step after ``at`` that holds a token, STEPS where there is none; the last one before it, -1
        auto next_held = [&](int at, bool after) {
            if (tid == 0) s.found_at = after ? STEPS : -1;
            __syncthreads();
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int step = 4 * tid + e;
                if (!(s.held[tid] >> e & 1)) continue;
                if (after && step > at) atomicMin(&s.found_at, step);
                if (!after && step < at) atomicMax(&s.found_at, step);
            }
            __syncthreads();
            const int found = s.found_at;
            __syncthreads();
            return found;
        };
        u64 last_entry = 0;                                // of the last cut: the last listed token that stays
        auto cut = [&](bool by_mass, double limit, int at) {
            const double share = limit;
            while (true) {
                const bool whole = by_segments = list(at, at);
                // what the step holds in all
                u64 here_mass = 0;
                if (whole) {
                    rank_list();
                    here_mass = n > 0 ? s.all_before[n - 1] + s.all_mass[n - 1] : 0;
                } else {
                    u64 nothing = 0;
                    unsigned none = 0;
                    const float floor_at = floor_of(at), floor_before = floor_of(at - 1);
                    walk([&](float v, int) {
                        const u64 own = mass.of(v);
                        here_mass += v >= floor_at && !(at > 0 && v >= floor_before) ? own : 0;
                    });
                    cluster_sum(here_mass, nothing, none);
                }
                if (by_mass && of_whole) limit = share * (double)everything;
                // the coarse sums may be a step off: on to the next that holds anything, however far
                const int way = by_mass ? cut_way(above, here_mass, limit) : cut_way(above_count, (unsigned)n, limit);
                if (way < 0 && at > 0 && above_count > 0) {
                    const int back = next_held(at, false);
                    if (back >= 0) { at = back; continue; }
                }
                if (way > 0 && at + 1 < STEPS) {
                    const int on = next_held(at, true);
                    if (on < STEPS) { at = on; continue; }
                }
                if (whole) {
                    // the last that stays: the one of highest place before which less than the limit lies
                    if (tid == 0) s.found_count = 0;
                    __syncthreads();
                    for (int i = tid; i < n; i += THREADS) {
                        const double ahead = by_mass ? (double)(above + s.all_before[i]) : (double)((u64)above_count + i);
                        if (ahead < limit) atomicMax(&s.found_count, (unsigned)i);
                    }
                    __syncthreads();
                    const int place = (int)s.found_count;
                    thr = key_of(s.all[place]);
                    unsigned stay = 0, ties = 0;
                    for (int i = tid; i < n; i += THREADS)
                        if (key_of(s.all[i]) == thr) { ++ties; stay += i <= place; }
                    need = block_sum32(stay, s);
                    all_ties = need == block_sum32(ties, s);
                    last_entry = s.all[place];
                    return above + s.all_before[place] + s.all_mass[place];
                }
                // too many for the list: by the bits of the keys, until one key is left
                unsigned from = low, upto = high;
                u64 run = above;
                u64 run_count = above_count;
                while (from < upto) {
                    int shift = 0;
                    while (((upto - from) >> shift) >= (unsigned)STEPS) ++shift;
                    for (int i = tid; i < STEPS; i += THREADS) { s.counts[i] = 0; s.fine[i] = 0; }
                    __syncthreads();
                    walk([&](float v, int) {
                        const unsigned key = ordered_key(sanitize(v));
                        if (key < from || key > upto) return;
                        const int bin = (int)((upto - key) >> shift);          // largest first
                        atomicAdd(&s.counts[bin], 1u);
                        atomicAdd(&s.fine[bin], mass.of(v));
                    });
                    cluster_sync();
                    u64 m[4], cnt[4], own_m = 0, own_n = 0, total_m, total_n;
                    all_blocks(&s.counts[4 * tid], cnt);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        m[e] = 0;
                        for (int c = 0; c < C; ++c) m[e] += ld_peer64(&s.fine[4 * tid + e], c);
                        own_m += m[e];
                        own_n += cnt[e];
                    }
                    u64 bm = run + block_before64(own_m, total_m, s), bn = run_count + block_before64(own_n, total_n, s);
                    if (tid == 0) s.found_at = -1;
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const double b = by_mass ? (double)bm : (double)bn, a = by_mass ? (double)(bm + m[e]) : (double)(bn + cnt[e]);
                        // the bin at which the limit is reached; the first that holds anything where nothing may come before it; the last of all
                        if (cnt[e] > 0 && (b < limit || bn == 0) && (a >= limit || bn + cnt[e] == run_count + total_n)) {
                            s.found_at = 4 * tid + e;
                            s.found_mass = bm;
                            s.found_count = (unsigned)bn;
                        }
                        bm += m[e];
                        bn += cnt[e];
                    }
                    __syncthreads();
                    const int bin = s.found_at;
                    run = s.found_mass;
                    run_count = s.found_count;
                    cluster_sync();                        // the peers' bins are read
                    const unsigned above_key = (unsigned)bin << shift;
                    const unsigned new_upto = upto - above_key, width = (1u << shift) - 1u;
                    from = new_upto - from < width ? from : new_upto - width;
                    upto = new_upto;
                }
                thr = from;
                by_segments = false;
                unsigned ties = 0;
                walk([&](float v, int) { ties += ordered_key(sanitize(v)) == thr; });
                u64 nothing64 = 0, nothing65 = 0;
                cluster_sum(nothing64, nothing65, ties);
                const u64 each = mass.of(logit_of(thr));
                if (by_mass) {
                    // the fewest with which the limit is reached, and one at least where nothing comes before
                    const double more = each > 0 ? ceil((limit - (double)run) / (double)each) : 1.0;
                    unsigned want = more < 1.0 ? 1u : more > (double)ties ? ties : (unsigned)more;
                    while (want > 1 && (double)(run + (u64)(want - 1) * each) >= limit) --want;
                    while (want < ties && (double)(run + (u64)want * each) < limit) ++want;
                    need = want;
                } else
                    need = min(ties, (unsigned)(u64)(limit - (double)run_count));
                all_ties = need == ties;
                return run + (u64)need * each;
            }
        };
        if (use_k) {
            const u64 within = cut(false, (double)k, k_bites ? step_k : STEPS);
            if (use_p) {
                // coarse sums are whole numbers of 2^-(COARSE_BITS + 16) of the largest mass
                const double limit = (double)p * (double)within;
                const int at = step_at(coarse, coarse_before, all_coarse, limit * exp2((double)(COARSE_BITS + 16 - of.mass_bits)));
                cut(true, limit, at < 0 ? 0 : at);
            }
        } else
            cut(true, (double)p, step_p < 0 ? 0 : step_p);
        if (by_segments) {
            // the segments hold what lies before the last cut's step: the tokens of the step that stay come to it, each block's own
            __syncthreads();
            for (int i = tid; i < s.listed; i += THREADS) {
                const u64 entry = s.list[i];
                const float v = logit_of(key_of(entry));
                if (entry > last_entry || v < low_logit) continue;
                atomicAdd(&s.segment_mass[(int)(unsigned)entry / S - (int)rank * per_block], mass.of(v));
                number_all += v >= mass.counted;
            }
        }
    }

    // ---- what stays, by segments of the row.  Only where ties are cut does their order count.
    if (!all_ties) {
        for (int j = 0; j < per_warp; ++j) {
            unsigned ties = 0;
            over_segment(x, min((long long)V, (long long)(first_segment + j) * S), min((long long)V, (long long)(first_segment + j + 1) * S), vector,
                         [&](float v, int) { ties += ordered_key(v) == thr; });
            ties = __reduce_add_sync(0xffffffffu, ties);
            if (lane == 0) s.segment_ties[warp * per_warp + j] = (int)ties;
        }
        cluster_sync();
        u64 before = 0, nothing;
        if (tid < SEGMENTS) before = ld_peer(&s.segment_ties[tid % per_block], tid / per_block);
        before = block_before64(before, nothing, s);
        if (tid < SEGMENTS) s.row_ties[tid] = (int)before;
        cluster_sync();
    }
    // keys above or equal to thr, and what min-p leaves, as one logit; keys 0 and of -inf: all
    const float lowest = fmaxf(thr > ordered_key(-CUDART_INF_F) ? __uint_as_float((thr & 0x80000000u) ? (thr & 0x7fffffffu) : ~thr) : -CUDART_INF_F, low_logit);
    const float lowest_counted = fmaxf(lowest, mass.counted);
    if (!by_segments) {
        if (all_ties)
            walk_segments([&](float v, int, Sums& here) {
                const u64 own = mass.of(v);
                here.mass += v >= lowest ? own : 0;
                here.number += v >= lowest_counted;
            });
        else {
            number_all = 0;
            for (int j = 0; j < per_warp; ++j) {           // 32 tokens at a time, in order
                const int segment = first_segment + j;
                const int from = (int)min((long long)V, (long long)segment * S), to = (int)min((long long)V, (long long)(segment + 1) * S);
                unsigned seen = (unsigned)s.row_ties[segment];
                u64 sum = 0;
                for (int base = from; base < to; base += 32) {
                    const int i = base + lane;
                    const float v = i < to ? sanitize(x[i]) : -CUDART_INF_F;
                    const unsigned key = ordered_key(v), tied = __ballot_sync(0xffffffffu, i < to && key == thr);
                    const unsigned place = seen + __popc(tied & ((1u << lane) - 1u));
                    seen += __popc(tied);
                    if (i < to && (key > thr || (key == thr && place < need)) && v >= low_logit) {
                        sum += mass.of(v);
                        number_all += v >= mass.counted;
                    }
                }
                sum = warp_sum64(sum);
                if (lane == 0) s.segment_mass[warp * per_warp + j] = sum;
            }
        }
    }
    number_all = block_sum32(number_all, s);
    if (tid == 0) s.own_count = number_all;
    cluster_sync();
    u64 mine = 0, total;
    if (tid < SEGMENTS) mine = ld_peer64(&s.segment_mass[tid % per_block], tid / per_block);
    const u64 before = block_before64(mine, total, s);
    if (tid < SEGMENTS) s.row_mass[tid] = before;
    if (tid == 0) s.row_mass[SEGMENTS] = total;
    number_all = __reduce_add_sync(0xffffffffu, lane < C ? ld_peer(&s.own_count, lane) : 0);
    __syncthreads();
    cluster_sync();                                        // the others' sums are read: they may leave
    const float u = of.uniform[row];
    double target = (u > 0.f ? (double)fminf(u, 1.f) : 0.0) * (double)total;
    if (target >= (double)total) target = nextafter((double)total, 0.0);
    // the segment it falls in, and the block that has it: two tokens a thread
    if (tid == 0) s.found_at = -1;
    __syncthreads();
    if (tid < per_block) {
        const int segment = (int)rank * per_block + tid;
        if ((double)s.row_mass[segment] <= target && target < (double)s.row_mass[segment + 1]) s.found_at = segment;
    }
    __syncthreads();
    const int segment = s.found_at;
    if (segment < 0) return;
    const int from = (int)min((long long)V, (long long)segment * S) + 2 * tid, to = (int)min((long long)V, (long long)(segment + 1) * S);
    float v[2];
    bool tied[2], stays[2];
    u64 m[2], nothing;
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        v[e] = from + e < to ? sanitize(x[from + e]) : -CUDART_INF_F;
        tied[e] = from + e < to && ordered_key(v[e]) == thr;
        stays[e] = from + e < to && ordered_key(v[e]) >= thr && v[e] >= low_logit;
    }
    if (!all_ties) {
        unsigned place = (unsigned)s.row_ties[segment] + (unsigned)block_before64((u64)tied[0] + (u64)tied[1], nothing, s);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            stays[e] = stays[e] && (!tied[e] || place < need);
            place += tied[e];
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) m[e] = stays[e] ? mass.of(v[e]) : 0;
    u64 run = s.row_mass[segment] + block_before64(m[0] + m[1], nothing, s);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        if (m[e] > 0 && (double)run <= target && target < (double)(run + m[e])) {
            of.tokens[row] = from + e;
            of.probability[row] = (float)((double)m[e] / (double)total);
            of.kept[row] = (int)number_all;
        }
        run += m[e];
    }
}
static_assert(((1 << 19) / SEGMENTS) <= 2 * THREADS, "a segment's tokens, two a thread");

// How many clusters of ``blocks`` blocks of the kernel the device holds at once; asked of the driver once per size and device.
int clusters_resident(int blocks) {
    static int cached[64][4];
    int device = 0, slot = blocks == 8 ? 3 : blocks == 4 ? 2 : blocks == 2 ? 1 : 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 0;
    if (cached[device][slot] == 0) {
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3((unsigned)blocks);
        cfg.blockDim = dim3(THREADS);
        cfg.dynamicSmemBytes = sizeof(Shared);
        cudaLaunchAttribute attr[1];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = blocks;
        attr[0].val.clusterDim.y = 1;
        attr[0].val.clusterDim.z = 1;
        cfg.attrs = attr;
        cfg.numAttrs = 1;
        int clusters = 0;
        if (cudaOccupancyMaxActiveClusters(&clusters, sample_filtered_kernel, &cfg) != cudaSuccess) {
            cudaGetLastError();
            clusters = 0;
        }
        cached[device][slot] = clusters > 0 ? clusters : -1;
    }
    return cached[device][slot] > 0 ? cached[device][slot] : 0;
}

}  // namespace

// ``blocks``: how many share a row (1, 2, 4 or 8); 0: the most that still lets every row's cluster be resident at once.  The results do not depend on it.
extern "C" int fe_sample_filtered(const float* logits, long long ld, int R, int V, const float* temperature, const int* top_k, const float* top_p,
                                  const float* min_p, const float* uniform, int* tokens, float* probability, int* kept, int blocks, cudaStream_t stream) {
    FE_REQUIRE(R >= 0 && V > 0 && ld >= V, "sample_filtered: bad sizes R=%d V=%d ld=%lld", R, V, ld);
    FE_REQUIRE(V < (1 << 19) && (long long)R * MAX_CLUSTER < (1LL << 31), "sample_filtered: %d rows of %d logits; fewer than 2^19 logits and 2^28 rows", R, V);      // a step's coarse mass is 32 bits
    FE_REQUIRE(blocks == 0 || blocks == 1 || blocks == 2 || blocks == 4 || blocks == 8, "sample_filtered: %d blocks a row; 1, 2, 4 or 8", blocks);
    if (R == 0) return 0;
    FE_REQUIRE(fe_allow_smem((const void*)sample_filtered_kernel, (int)sizeof(Shared)), "sample_filtered: no kernel with %d bytes of shared memory", (int)sizeof(Shared));
    if (blocks == 0)
        for (blocks = MAX_CLUSTER; blocks > 1 && R > clusters_resident(blocks);) blocks >>= 1;
    int bits = 0;
    while ((1LL << bits) < V) ++bits;
    const Rows of{logits, ld, V, temperature, top_k, top_p, min_p, uniform, tokens, probability, kept, bits <= 18 ? 44 : 62 - bits};
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(R * blocks));
    cfg.blockDim = dim3(THREADS);
    cfg.dynamicSmemBytes = sizeof(Shared);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const cudaError_t err = cudaLaunchKernelEx(&cfg, sample_filtered_kernel, of, blocks);
    FE_REQUIRE(err == cudaSuccess, "sample_filtered (clusters of %d): %s", blocks, cudaGetErrorString(err));
    return fe_check_launch("sample_filtered");
}

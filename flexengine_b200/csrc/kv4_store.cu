// New keys and values into a cache held in 4 bits (kv4.cuh has its form): bias, rotation and rounding in one pass over the projection, and
// the queries beside them; and reading rows back.
//
// Rotation of the first ``rot`` entries of every query and key head by angle = position * inv_freq[j]: entries j and j + rot / 2 (halves)
// or 2j and 2j + 1 (interleaved) turn together, a' = (a cos - b sin) gain, b' = (b cos + a sin) gain.  The angle, its sine and its
// cosine are taken in 64 bits: at position 100,000 a 32-bit product alone is off by up to 0.004, as much as bfloat16
// rounds a query by, and enough to move every twentieth 4-bit code of a fast pair.  A token has rot / 2 angles, shared by its heads.  From there on every operation is rounded by itself
// to 32 bits, up to the pair of scale and centre and the codes: next to the border of two codes the one that is taken is the formula's.
//
// A warp takes a row of d numbers (one head of one token), four neighbouring numbers a lane, so that a group of 32 is eight lanes: its
// smallest and largest number are three shuffles away, and each lane's four codes are two neighbouring bytes of the row.  What bounds
// it is reading the projection: see the figures at the launch.
#define FE_PDL_CLASS 4      // FE_PDL_ELEMENTWISE
#include "kv4.cuh"
#include "tcgen05.cuh"

using namespace fe;

namespace {

constexpr int MAX_ROT = 256;

// sine and cosine of the exact angle (31 and 24 bits make a product of 55 at most, rounded to 53), rounded to 32 bits once
__device__ __forceinline__ void angle_of(int pos, float freq, float* sn, float* cs) {
    double s, c;
    sincos((double)pos * (double)freq, &s, &c);
    *sn = (float)s;
    *cs = (float)c;
}
// a cos + b sin, each product rounded by itself: next to the border of two codes the one that is taken does not hang on which product the compiler fuses
__device__ __forceinline__ float turn_by(float a, float cs, float b, float sn) { return __fadd_rn(__fmul_rn(a, cs), __fmul_rn(b, sn)); }

// Four numbers from ``p``; VEC: from a boundary of four.
template <typename T, bool VEC> __device__ __forceinline__ void load4(const T* p, float* v);
template <> __device__ __forceinline__ void load4<float, true>(const float* p, float* v) {
    const float4 a = *reinterpret_cast<const float4*>(p);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
}
template <> __device__ __forceinline__ void load4<bf16, true>(const bf16* p, float* v) {
    const uint2 a = *reinterpret_cast<const uint2*>(p);
    v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xffff0000u);
    v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xffff0000u);
}
template <> __device__ __forceinline__ void load4<float, false>(const float* p, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = p[e];
}
template <> __device__ __forceinline__ void load4<bf16, false>(const bf16* p, float* v) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = __bfloat162float(p[e]);
}
__device__ __forceinline__ void store4(float* p, const float* v) { *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ void store4(bf16* p, const float* v) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}

struct Rotation {
    const float* inv_freq;
    int rot;
    bool interleaved;
    float gain;
};

// Where the four numbers of unit u (group u / 8) go in a tile whose token is ``at``.
struct Into {
    int codes, pair;
};
__device__ __forceinline__ Into into_of(bool is_k, int u, int groups) {
    return is_k ? Into{kv4_key_at(u >> 3, u & 7, groups), kv4_key_pairs(groups) + (u >> 3) * 4}
                : Into{kv4_value_codes(groups) + kv4_value_at(u >> 3, u & 7, groups), kv4_value_pairs(groups) + (u >> 3) * 4};
}

// Four numbers of a key or a value, a lane's share of its group of eight lanes, into their codes and (the group's first lane) its pair; ``row_codes`` and
// ``row_pairs``: bytes from the tile's first token to this one among codes and pairs.  The whole warp is here.
__device__ __forceinline__ void put_group(float* v, bool real, int u, int units, const Into& into, int row_codes, int row_pairs, unsigned char* tile) {
    const int lane = threadIdx.x & 31;
    // the group's ends over its eight lanes; a NaN is looked for by itself, since the comparisons pass it over
    float low = CUDART_INF_F, high = -CUDART_INF_F;
    bool bad = false;
    if (real) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            bad |= v[e] != v[e];
            v[e] = fminf(fmaxf(v[e], -KV4_LARGEST), KV4_LARGEST);
            low = fminf(low, v[e]);
            high = fmaxf(high, v[e]);
        }
    }
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) {
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
    }
    bad = (__ballot_sync(0xffffffffu, bad) >> (lane & 24)) & 0xffu;
    if (u >= units) return;
    // rounded to half precision, to nearest: the codes below are chosen against the rounded pair
    const __half scale = __float2half_rn(bad ? CUDART_NAN_F : (high - low) * (1.f / 15.f));
    const float s = __half2float(scale);
    const __half centre = __float2half_rn(fmaf(8.f, s, low));
    // A code is 8 + (x - centre) / scale to the nearest whole number, 8 where the scale is 0 or NaN: adding 1.5 2^23 rounds and leaves it in the lowest
    // bits.  The quotient by the hardware's reciprocal (1 ulp) is within 2^-20 of the rounded one, which is asked for next to a border only: without, one
    // code in a million was another than the formula's, a whole step away.
    const float c = bad ? 0.f : __half2float(centre);
    float each, off[4];
    asm("rcp.approx.ftz.f32 %0, %1;\n" : "=f"(each) : "f"(s));
    each = s > 0.f ? each : 0.f;
    bool close = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        off[e] = (v[e] - c) * each;
        close |= fabsf(off[e] - __fsub_rn(__fadd_rn(off[e], 12582912.f), 12582912.f)) > 0.5f - 0x1p-18f;
    }
    if (close && s > 0.f) {
#pragma unroll
        for (int e = 0; e < 4; ++e) off[e] = __fdiv_rn(v[e] - c, s);
    }
    unsigned codes = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) codes |= ((__float_as_uint(fminf(fmaxf(off[e], -8.f), 7.f) + 12582912.f) + 8u) & 15u) << (4 * e);
    *reinterpret_cast<unsigned short*>(tile + into.codes + row_codes) = (unsigned short)codes;
    if ((u & 7) == 0) *reinterpret_cast<__half2*>(tile + into.pair + row_pairs) = __halves2half2(scale, centre);
}

// Where a token's keys and values go: head 0's tile (null: nowhere) and the token's place in it.
struct Place {
    unsigned char* tile;
    int at;
};
__device__ __forceinline__ Place place_of(long long slot, long long num_slots, int ps, int nkv, int tile_bytes, unsigned char* cache, int* status, bool reports) {
    if (slot >= num_slots) {
        if (reports && status) atomicOr(status, FE_STATUS_BAD_SLOT);
        slot = -1;
    }
    if (slot < 0) return Place{nullptr, 0};
    const int page = (int)(slot / ps), within = (int)(slot - (long long)page * ps);
    return Place{cache + (long long)page * nkv * (ps / KV4_TILE * tile_bytes) + within / KV4_TILE * tile_bytes, within % KV4_TILE};
}

// A few tokens, or rows that lie anywhere: a block a token (blockIdx.y shares its heads out where tokens are few), a warp a row.  TI: the projection's type,
// TO: the queries'.  VEC: rows of the projection, the bias and half the rotated part lie on boundaries of four numbers.
template <typename TI, typename TO, bool VEC>
__global__ void __launch_bounds__(256)
kv4_store_kernel(const TI* __restrict__ src, long long ld, const float* __restrict__ bias, const int* __restrict__ positions, Rotation turn,
                 const int* __restrict__ slot_mapping, unsigned char* __restrict__ cache, TO* __restrict__ queries, int nq, int nkv, int d,
                 int ps, long long num_slots, int* __restrict__ status) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ __align__(16) float cosine[MAX_ROT / 2], sine[MAX_ROT / 2];
    const int token = blockIdx.x, half = turn.rot / 2;
    const long long slot = slot_mapping ? slot_mapping[token] : -1;
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        float sn, cs;
        angle_of(positions[token], turn.inv_freq[j], &sn, &cs);
        cosine[j] = cs * turn.gain;
        sine[j] = sn * turn.gain;
    }
    const int lane = threadIdx.x & 31, warps = (blockDim.x >> 5) * gridDim.y;
    const int groups = kv4_groups(d), units = groups * 8, tile_bytes = kv4_tile_bytes(groups);      // units: four numbers each, padding ones among them
    const Place place = place_of(slot, num_slots, ps, nkv, tile_bytes, cache, status, threadIdx.x == 0 && blockIdx.y == 0);
    __syncthreads();
    const int heads = nq + 2 * nkv;
    for (int head = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5); head < heads; head += warps) {
        const bool is_q = head < nq, is_k = !is_q && head < nq + nkv;
        if (!is_q && !place.tile) continue;
        const TI* x = src + (long long)token * ld + (long long)head * d;
        const float* b = bias ? bias + (long long)head * d : nullptr;
        for (int u0 = 0; u0 < units; u0 += 32) {                       // d > 128: two rounds
            const int u = u0 + lane, i = 4 * u;
            const bool real = i < d;                                   // d is a multiple of 16: a unit is all numbers or all padding
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (real) {
                load4<TI, VEC>(x + i, v);
                if (b) {
                    float w[4];
                    load4<float, VEC>(b + i, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += w[e];
                }
            }
            if (real && (is_q || is_k) && i < turn.rot) {
                if (turn.interleaved) {
#pragma unroll
                    for (int e = 0; e < 4; e += 2) {
                        if (i + e >= turn.rot) break;
                        const int j = (i + e) / 2;
                        const float a = v[e], c = v[e + 1];
                        v[e] = turn_by(a, cosine[j], c, -sine[j]);
                        v[e + 1] = turn_by(c, cosine[j], a, sine[j]);
                    }
                } else {
                    // the entries these four turn with, half the rotated part away
                    float o[4] = {0.f, 0.f, 0.f, 0.f};
                    if (VEC) {
                        const int partner = i < half ? i + half : i - half;
                        load4<TI, VEC>(x + partner, o);
                        if (b) {
                            float w[4];
                            load4<float, VEC>(b + partner, w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) o[e] += w[e];
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int partner = i + e < half ? i + e + half : i + e - half;
                            if (i + e < turn.rot) o[e] = to_float(x[partner]) + (b ? b[partner] : 0.f);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        if (i + e >= turn.rot) break;
                        const int j = i + e < half ? i + e : i + e - half;
                        v[e] = turn_by(v[e], cosine[j], i + e < half ? -o[e] : o[e], sine[j]);
                    }
                }
            }
            if (!is_q) put_group(v, real, u, units, into_of(is_k, u, groups), place.at * 16 * groups, place.at * 4 * groups, place.tile + (long long)(is_k ? head - nq : head - nq - nkv) * (ps / KV4_TILE * tile_bytes));
            else if (real) store4(queries + ((long long)token * nq + head) * d + i, v);
        }
    }
}

// Many tokens: blocks that stay, each with two places for tokens' rows in shared memory and the bias beside them.  A bulk copy brings a token's whole
// row (all heads) while the one before is worked on: 2,048 tokens of 40/8 heads of 128 take 21 us, of which 13 are the 85 MB's way through memory; a
// row a warp at a time waited for each load (38).  A ring of six rows and one block of 32 warps a multiprocessor took 30.
constexpr int STAY_WARPS = 16;
constexpr int BATCH = 8;        // tokens whose angles and places are worked out together, a thread an angle
__host__ __device__ inline size_t stay_bytes(int width, int item) { return (size_t)2 * width * item + (size_t)4 * width; }

template <typename TI, typename TO>
__global__ void __launch_bounds__(STAY_WARPS * 32)
kv4_store_many_kernel(const TI* __restrict__ src, long long ld, const float* __restrict__ bias, const int* __restrict__ positions, Rotation turn,
                      const int* __restrict__ slot_mapping, unsigned char* __restrict__ cache, TO* __restrict__ queries, int T, int nq, int nkv, int d,
                      int ps, long long num_slots, int* __restrict__ status, const FeWaits waits) {
    griddep_wait();
    griddep_launch_dependents();
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ __align__(16) float cosine[BATCH][MAX_ROT / 2], sine[BATCH][MAX_ROT / 2];
    __shared__ Place places[BATCH];
    __shared__ __align__(8) unsigned long long arrived[2];
    const int width = (nq + 2 * nkv) * d, half = turn.rot / 2, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const TI* rows = reinterpret_cast<const TI*>(smem);
    float* added = reinterpret_cast<float*>(smem + (size_t)2 * width * sizeof(TI));
    const int groups = kv4_groups(d), units = groups * 8, tile_bytes = kv4_tile_bytes(groups);
    const long long head_bytes = (long long)(ps / KV4_TILE) * tile_bytes;
    if (tid < 2) mbar_init(&arrived[tid], 1);
    asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    __syncthreads();
    auto bring = [&](int token, int place) {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n" ::"r"(smem_u32(&arrived[place])), "r"((int)(width * sizeof(TI)) + waits.lacking) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n"
                     ::"r"(smem_u32(rows + (size_t)place * width)), "l"(src + (long long)token * ld), "r"((int)(width * sizeof(TI))), "r"(smem_u32(&arrived[place])) : "memory");
    };
    auto prepare = [&](int token) {                                // and the BATCH - 1 tokens of this block after it
        for (int j = tid; j < half * BATCH; j += STAY_WARPS * 32) {
            const int k = j / half, at = j - k * half, t = token + k * (int)gridDim.x;
            if (t >= T) break;
            float sn, cs;
            angle_of(positions[t], turn.inv_freq[at], &sn, &cs);
            cosine[k][at] = cs * turn.gain;
            sine[k][at] = sn * turn.gain;
        }
        if (tid < BATCH) {
            const int t = token + tid * (int)gridDim.x;
            if (t < T) places[tid] = place_of(slot_mapping ? slot_mapping[t] : -1, num_slots, ps, nkv, tile_bytes, cache, status, true);
        }
    };
    int token = blockIdx.x;
    if (tid == 0) bring(token, 0);
    for (int i = tid; i < width; i += STAY_WARPS * 32) added[i] = bias ? bias[i] : 0.f;
    int place = 0, parity = 0;
    for (int turn_of = 0; token < T; token += gridDim.x, turn_of = (turn_of + 1) % BATCH) {
        if (turn_of == 0) {
            prepare(token);
            __syncthreads();
        }
        const int next = token + gridDim.x;
        if (tid == 0 && next < T) bring(next, place ^ 1);
        const Place to = places[turn_of];
        const int row_codes = to.at * 16 * groups, row_pairs = to.at * 4 * groups;
        const float *cosines = cosine[turn_of], *sines = sine[turn_of];
        const bool here = mbar_wait(&arrived[place], parity, waits.limit);
        if (!here) {
            // the copies on their way go to memory that the block is about to leave: this token's once more, and the next one's
            if (status) atomicOr(status, FE_STATUS_WAIT_EXPIRED);
            mbar_wait(&arrived[place], parity, waits.limit);
            if (next < T) mbar_wait(&arrived[place ^ 1], parity ^ place, waits.limit);
        }
        if (__syncthreads_or(!here)) return;
        for (int u0 = 0; u0 < units; u0 += 32) {
            const int u = u0 + lane, i = 4 * u;
            const bool real = i < d, turns = i < turn.rot;
            const Into into_k = into_of(true, u, groups), into_v = into_of(false, u, groups);
            // this lane's angles and the entry that its first one turns with, the same in all heads
            float cs[4] = {1.f, 1.f, 1.f, 1.f}, sn[4] = {0.f, 0.f, 0.f, 0.f};
            int partner = i;
            if (real && turns) {
                if (turn.interleaved) {
                    // entries 2j and 2j + 1: a' = a cos - b sin, b' = b cos + a sin
#pragma unroll
                    for (int e = 0; e < 4; ++e) { cs[e] = cosines[(i + e) / 2]; sn[e] = e & 1 ? sines[(i + e) / 2] : -sines[(i + e) / 2]; }
                } else {
                    partner = i < half ? i + half : i - half;
                    const int j = i < half ? i : i - half;
                    load4<float, true>(cosines + j, cs);
                    load4<float, true>(sines + j, sn);
#pragma unroll
                    for (int e = 0; e < 4; ++e) sn[e] = i < half ? -sn[e] : sn[e];
                }
            }
            const TI* x = rows + (size_t)place * width;
            auto turned = [&](int head, float* v) {
                float w[4], o[4];
                load4<TI, true>(x + head * d + i, v);
                load4<float, true>(added + head * d + i, w);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] += w[e];
                if (!turns) return;
                if (turn.interleaved) { o[0] = v[1]; o[1] = v[0]; o[2] = v[3]; o[3] = v[2]; }
                else {
                    load4<TI, true>(x + head * d + partner, o);
                    load4<float, true>(added + head * d + partner, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[e] += w[e];
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = turn_by(v[e], cs[e], o[e], sn[e]);
            };
            // keys and values first: they take the longest; then the queries
            if (to.tile)
                for (int h = warp; h < 2 * nkv; h += STAY_WARPS) {
                    const bool is_k = h < nkv;
                    float v[4] = {0.f, 0.f, 0.f, 0.f};
                    if (real) {
                        if (is_k) turned(nq + h, v);
                        else {
                            float w[4];
                            load4<TI, true>(x + (nq + h) * d + i, v);
                            load4<float, true>(added + (nq + h) * d + i, w);
#pragma unroll
                            for (int e = 0; e < 4; ++e) v[e] += w[e];
                        }
                    }
                    put_group(v, real, u, units, is_k ? into_k : into_v, row_codes, row_pairs, to.tile + (is_k ? h : h - nkv) * head_bytes);
                }
            if (real) {
                TO* q = queries + (long long)token * nq * d + i;
#pragma unroll 2
                for (int head = warp; head < nq; head += STAY_WARPS) {
                    float v[4];
                    turned(head, v);
                    store4(q + head * d, v);
                }
            }
        }
        __syncthreads();                                           // the rows and angles of this token have been read
        parity ^= place;
        place ^= 1;
    }
}

// A warp a (slot, head): its key and its value as numbers; a slot below 0 reads as zeros.
template <typename TO>
__global__ void __launch_bounds__(256)
kv4_rows_kernel(const unsigned char* __restrict__ cache, const int* __restrict__ slots, TO* __restrict__ keys, TO* __restrict__ values, long long rows,
                int nkv, int d, int ps, long long num_slots, int* __restrict__ status) {
    griddep_wait();
    griddep_launch_dependents();
    const long long row = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (row >= rows) return;
    const int lane = threadIdx.x & 31, kvh = (int)(row % nkv), groups = kv4_groups(d);
    long long slot = slots[row / nkv];
    if (slot >= num_slots) {
        if (lane == 0 && status) atomicOr(status, FE_STATUS_BAD_SLOT);
        slot = -1;
    }
    const long long page = slot < 0 ? 0 : slot / ps;
    const int within = slot < 0 ? 0 : (int)(slot - page * ps), at = within % KV4_TILE;
    const unsigned char* tile = cache + ((page * nkv + kvh) * (ps / KV4_TILE) + within / KV4_TILE) * kv4_tile_bytes(groups);
    for (int i = 4 * lane; i < d; i += 128) {
        const int g = i / KV4_GROUP, p = i % KV4_GROUP / 4;
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (slot >= 0) {
                const unsigned codes = *reinterpret_cast<const unsigned short*>(
                    tile + (side ? kv4_value_codes(groups) : 0) + at * 16 * groups + (side ? kv4_value_at(g, p, groups) : kv4_key_at(g, p, groups)));
                const float2 pair = __half22float2(*reinterpret_cast<const __half2*>(tile + (side ? kv4_value_pairs(groups) : kv4_key_pairs(groups)) + (at * groups + g) * 4));
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = fmaf((float)(int)(codes >> (4 * e) & 15u) - 8.f, pair.x, pair.y);
            }
            store4((side ? values : keys) + row * d + i, v);
        }
    }
}

template <typename TI, typename TO>
int store(const void* src, long long ld, const float* bias, const int* positions, const Rotation& turn, const int* slots, void* cache, void* queries,
          int T, int nq, int nkv, int d, int ps, long long num_slots, int* status, cudaStream_t stream) {
    const int rows = nq + 2 * nkv, width = rows * d, sms = fe_sm_count();
    const bool vec = ld % 4 == 0 && (size_t)src % (4 * sizeof(TI)) == 0 && (size_t)bias % 16 == 0 && turn.rot / 2 % 4 == 0;
    // Blocks that stay, two a multiprocessor, from where each takes two tokens and more; rows on 16-byte boundaries that fit twice beside the bias
    const size_t smem = stay_bytes(width, sizeof(TI));
    if (T >= 4 * sms && vec && turn.rot % 4 == 0 && (size_t)src % 16 == 0 && ld * sizeof(TI) % 16 == 0 && smem <= 110 * 1024) {
        auto kernel = kv4_store_many_kernel<TI, TO>;
        FE_REQUIRE(fe_allow_smem((const void*)kernel, (int)smem), "qkv_rope_kv4: no kernel with %d bytes of shared memory", (int)smem);
        // not among the overlapping launches: the split of an SM's memory that they share leaves room for one such block, not two
        fe::launch_as(0, kernel, dim3((unsigned)(2 * sms)), STAY_WARPS * 32, smem, stream, (const TI*)src, ld, bias, positions, turn, slots, (unsigned char*)cache,
                   (TO*)queries, T, nq, nkv, d, ps, num_slots, status, fe_waits());
        return fe_check_launch("qkv_rope_kv4");
    }
    // a block a token, or, where that gives multiprocessors less than one, a block for every eight rows of a token, each with its own angles
    auto kernel = vec ? kv4_store_kernel<TI, TO, true> : kv4_store_kernel<TI, TO, false>;
    fe::launch(kernel, dim3((unsigned)T, (unsigned)(T >= sms ? 1 : (rows + 7) / 8)), 256, 0, stream, (const TI*)src, ld, bias, positions, turn, slots,
               (unsigned char*)cache, (TO*)queries, nq, nkv, d, ps, num_slots, status);
    return fe_check_launch("qkv_rope_kv4");
}

}  // namespace

// ``src`` [T, >= (nq + 2 nkv) d] with rows ``ld`` elements apart; ``slots`` null: only the queries.  Slots of one call are distinct (two tokens
// of one slot would leave codes of the one beside scales of the other); a slot below 0 is not written.
extern "C" int fe_qkv_rope_kv4(const void* src, int src_dtype, long long ld, const float* bias, const int* positions, const float* inv_freq, int rot,
                               int interleaved, float gain, const int* slots, void* cache, void* queries, int out_dtype, int T, int nq, int nkv,
                               int d, int ps, long long num_slots, int* status, cudaStream_t stream) {
    FE_REQUIRE(T >= 0 && nq > 0 && nkv > 0 && nq % nkv == 0, "qkv_rope_kv4: bad sizes T=%d heads %d/%d", T, nq, nkv);
    FE_REQUIRE(d >= 16 && d % 16 == 0 && d <= KV4_MAX_DIM, "qkv_rope_kv4: head size %d; multiples of 16 up to %d", d, KV4_MAX_DIM);
    FE_REQUIRE(ps > 0 && ps % KV4_TILE == 0, "qkv_rope_kv4: page size %d; a multiple of %d", ps, KV4_TILE);
    FE_REQUIRE(rot >= 0 && rot <= d && rot % 2 == 0 && (rot == 0 || inv_freq != nullptr), "qkv_rope_kv4: rotary width %d does not fit head size %d", rot, d);
    FE_REQUIRE((long long)num_slots / ps < (1LL << 31) && (long long)ps * 40 * kv4_groups(d) < (1LL << 31), "qkv_rope_kv4: a cache of %lld slots in pages of %d is too large", num_slots, ps);
    FE_REQUIRE(ld >= (long long)(nq + 2 * nkv) * d, "qkv_rope_kv4: rows of %lld numbers are too short", ld);
    FE_REQUIRE(((size_t)cache & 15) == 0 && ((size_t)queries & 15) == 0, "qkv_rope_kv4: cache and queries must start on 16-byte boundaries");
    if (T == 0) return 0;
    const Rotation turn{inv_freq, rot, interleaved != 0, gain};
    if (src_dtype == FE_F32 && out_dtype == FE_F32)
        return store<float, float>(src, ld, bias, positions, turn, slots, cache, queries, T, nq, nkv, d, ps, num_slots, status, stream);
    if (src_dtype == FE_F32 && out_dtype == FE_BF16)
        return store<float, bf16>(src, ld, bias, positions, turn, slots, cache, queries, T, nq, nkv, d, ps, num_slots, status, stream);
    if (src_dtype == FE_BF16 && out_dtype == FE_BF16)
        return store<bf16, bf16>(src, ld, bias, positions, turn, slots, cache, queries, T, nq, nkv, d, ps, num_slots, status, stream);
    FE_REQUIRE(false, "qkv_rope_kv4: a projection of type %d for queries of type %d", src_dtype, out_dtype);
}

extern "C" int fe_kv4_rows(const void* cache, const int* slots, void* keys, void* values, int out_dtype, long long count, int nkv, int d, int ps,
                           long long num_slots, int* status, cudaStream_t stream) {
    FE_REQUIRE(count >= 0 && nkv > 0 && d >= 16 && d % 16 == 0 && d <= KV4_MAX_DIM, "kv4_rows: bad sizes");
    FE_REQUIRE(ps > 0 && ps % KV4_TILE == 0, "kv4_rows: page size %d; a multiple of %d", ps, KV4_TILE);
    const long long rows = count * nkv;
    FE_REQUIRE((rows + 7) / 8 < (1LL << 31), "kv4_rows: too many rows");
    if (rows == 0) return 0;
    if (out_dtype == FE_F32)
        fe::launch(kv4_rows_kernel<float>, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, (const unsigned char*)cache, slots, (float*)keys, (float*)values,
                   rows, nkv, d, ps, num_slots, status);
    else if (out_dtype == FE_BF16)
        fe::launch(kv4_rows_kernel<bf16>, dim3((unsigned)((rows + 7) / 8)), 256, 0, stream, (const unsigned char*)cache, slots, (bf16*)keys, (bf16*)values,
                   rows, nkv, d, ps, num_slots, status);
    else FE_REQUIRE(false, "kv4_rows: unknown type %d", out_dtype);
    return fe_check_launch("kv4_rows");
}

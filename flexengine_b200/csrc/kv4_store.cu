// New keys and values into a cache held in 4 bits (kv4.cuh has its form): bias, rotation and rounding in one pass over the projection, and
// the queries beside them; and reading rows back.
//
// Rotation of the first ``rot`` entries of every query and key head by angle = position * inv_freq[j]: entries j and j + rot / 2 (halves)
// or 2j and 2j + 1 (interleaved) turn together, a' = (a cos - b sin) gain, b' = (b cos + a sin) gain.  The angle is taken in 64 bits and
// brought to within a quarter turn there: at position 100,000 a 32-bit product alone is off by up to 0.004, as much as bfloat16
// rounds a query by, and enough to move every twentieth 4-bit code of a fast pair.  A token has rot / 2 angles, shared by its heads.
//
// A warp takes a row of d numbers (one head of one token), four neighbouring numbers a lane, so that a group of 32 is eight lanes: its
// smallest and largest number are three shuffles away, and each lane's four codes are two neighbouring bytes of the row.  What bounds
// it is reading the projection: see the figures at the launch.
#define FE_PDL_CLASS 4      // FE_PDL_ELEMENTWISE
#include "kv4.cuh"

using namespace fe;

namespace {

constexpr int MAX_ROT = 256;

__device__ __forceinline__ void angle_of(int pos, float freq, float* sn, float* cs) {
    const double a = (double)pos * (double)freq;                 // exact: 31 and 24 bits
    const double turns = rint(a * 0.63661977236758134308);       // of a quarter: a 2 / pi
    const float r = (float)fma(turns, -1.57079632679489661923, a);
    const int quarter = (int)(long long)turns & 3;
    float s, c;
    sincosf(r, &s, &c);
    *sn = quarter & 1 ? c : s;
    *cs = quarter & 1 ? s : c;
    if (quarter & 2) *sn = -*sn;
    if ((quarter + 1) & 2) *cs = -*cs;
}

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

// TI: the projection's type, TO: the queries'.  VEC: rows of the projection, the bias and half the rotated part lie on boundaries of four numbers.
template <typename TI, typename TO, bool VEC>
__global__ void __launch_bounds__(256)
kv4_store_kernel(const TI* __restrict__ src, long long ld, const float* __restrict__ bias, const int* __restrict__ positions, Rotation turn,
                 const int* __restrict__ slot_mapping, unsigned char* __restrict__ cache, TO* __restrict__ queries, int nq, int nkv, int d,
                 int ps, long long num_slots, int* __restrict__ status) {
    griddep_wait();
    griddep_launch_dependents();
    __shared__ float cosine[MAX_ROT / 2], sine[MAX_ROT / 2];
    const int token = blockIdx.x, half = turn.rot / 2;
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
        float sn, cs;
        angle_of(positions[token], turn.inv_freq[j], &sn, &cs);
        cosine[j] = cs * turn.gain;
        sine[j] = sn * turn.gain;
    }
    long long slot = slot_mapping ? slot_mapping[token] : -1;
    if (slot >= num_slots) {
        if (threadIdx.x == 0 && blockIdx.y == 0 && status) atomicOr(status, FE_STATUS_BAD_SLOT);
        slot = -1;
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warps = (blockDim.x >> 5) * gridDim.y;
    const int groups = kv4_groups(d), units = groups * 8;          // four numbers a unit, padding ones among them
    const TI* row = src + (long long)token * ld;
    for (int head = blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5); head < nq + 2 * nkv; head += warps) {
        const bool is_q = head < nq, is_k = !is_q && head < nq + nkv;
        if (!is_q && slot < 0) continue;
        const TI* x = row + (long long)head * d;
        const float* b = bias ? bias + (long long)head * d : nullptr;
        unsigned char* tile = nullptr;
        if (!is_q) {
            const long long page = slot / ps;
            const int within = (int)(slot - page * ps), kvh = is_k ? head - nq : head - nq - nkv;
            tile = cache + ((page * nkv + kvh) * (ps / KV4_TILE) + within / KV4_TILE) * kv4_tile_bytes(groups);
        }
        for (int u0 = 0; u0 < units; u0 += 32) {                   // d = 256: two rounds
            const int u = u0 + lane, i = 4 * u;
            const bool real = i < d;                               // d is a multiple of 16: a unit is all numbers or all padding
            float v[4] = {0.f, 0.f, 0.f, 0.f};
            if (real) {
                load4<TI, VEC>(x + i, v);
                if (b) {
                    float w[4];
                    load4<float, VEC>(b + i, w);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] += w[e];
                }
                if ((is_q || is_k) && i < turn.rot) {
                    if (turn.interleaved) {
#pragma unroll
                        for (int e = 0; e < 4; e += 2) {
                            const int j = (i + e) / 2;
                            if (i + e >= turn.rot) break;
                            const float a = v[e], c = v[e + 1];
                            v[e] = a * cosine[j] - c * sine[j];
                            v[e + 1] = c * cosine[j] + a * sine[j];
                        }
                    } else {
                        // the entries these four turn with, half the rotated part away: read once more (from L1)
                        float o[4];
                        if (VEC) {
                            const int at = i < half ? i + half : i - half;
                            load4<TI, VEC>(x + at, o);
                            if (b) {
                                float w[4];
                                load4<float, VEC>(b + at, w);
#pragma unroll
                                for (int e = 0; e < 4; ++e) o[e] += w[e];
                            }
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const int at = i + e < half ? i + e + half : i + e - half;
                                o[e] = i + e < turn.rot ? to_float(x[at]) + (b ? b[at] : 0.f) : 0.f;
                            }
                        }
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            if (i + e >= turn.rot) break;
                            const int j = i + e < half ? i + e : i + e - half;
                            v[e] = i + e < half ? v[e] * cosine[j] - o[e] * sine[j] : v[e] * cosine[j] + o[e] * sine[j];
                        }
                    }
                }
            }
            if (is_q) {
                if (real) store4(queries + ((long long)token * nq + head) * d + i, v);
                continue;
            }
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
            bad = __ballot_sync(0xffffffffu, bad) >> (lane & 24) & 0xffu;
            if (u >= units) continue;
            // rounded to half precision, to nearest: the codes below are chosen against the rounded pair
            const __half scale = __float2half_rn(bad ? CUDART_NAN_F : (high - low) / 15.f);
            const float s = __half2float(scale);
            const __half centre = __float2half_rn(fmaf(8.f, s, low));
            const float c = __half2float(centre);
            unsigned codes = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float n = s > 0.f ? fminf(fmaxf(rintf((v[e] - c) / s) + 8.f, 0.f), 15.f) : 8.f;
                codes |= (real ? (unsigned)n : 0u) << (4 * e);
            }
            const int g = u >> 3, p = u & 7, at = (int)(slot % KV4_TILE);         // ps is a multiple of the tile
            unsigned char* into = tile + (is_k ? 0 : kv4_value_codes(groups)) + at * 16 * groups + (is_k ? kv4_key_at(g, p, groups) : kv4_value_at(g, p, groups));
            *reinterpret_cast<unsigned short*>(into) = (unsigned short)codes;
            if (p == 0)
                *reinterpret_cast<__half2*>(tile + (is_k ? kv4_key_pairs(groups) : kv4_value_pairs(groups)) + (at * groups + g) * 4) = __halves2half2(scale, centre);
        }
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
    const int rows = nq + 2 * nkv, blocks = (rows + 7) / 8;
    // few tokens: a block for every eight rows of a token, each with its own angles, so that no warp takes two rows one after the other
    const int share = T >= fe_sm_count() ? 1 : blocks;
    const bool vec = ld % 4 == 0 && (size_t)src % (4 * sizeof(TI)) == 0 && (size_t)bias % 16 == 0 && turn.rot / 2 % 4 == 0;
    auto kernel = vec ? kv4_store_kernel<TI, TO, true> : kv4_store_kernel<TI, TO, false>;
    fe::launch(kernel, dim3((unsigned)T, (unsigned)share), 256, 0, stream, (const TI*)src, ld, bias, positions, turn, slots,
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

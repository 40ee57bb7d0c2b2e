// Keys and values held in 4 bits: the form that what writes them and what reads them share.
//
// A row (the key or the value of one token and head, d numbers) is cut into G = ceil(d / 32) groups of 32 neighbouring numbers, the last
// one padded.  A group has a scale and a centre in half precision, a number a code of 4 bits: x = centre + (code - 8) scale, with
// scale = (largest - smallest) / 15 and centre = smallest + 8 scale, each rounded before the codes are chosen, so that the codes
// make up for the roundings; both ends of the group are codes (0 and 15).  40 bytes a group for a key and a value: 5 bits a number.
//
// Cache: uint8 [pages, heads, page size / 16, 640 G].  A tile of 16 tokens lies in one piece, so that one bulk copy brings it:
//   [16][4][G][4]  key codes: word (t, g) of a token holds numbers 32 g + 8 t .. + 7, the first in the lowest bits
//   [16][8][G][2]  value codes: piece (p, g) holds numbers 32 g + 4 p .. + 3
//   [16][G]        (scale, centre) of the keys' groups, then [16][G] of the values'
// The codes of a row lie in the order in which m16n8k16 products take them: thread (g, t) of a warp finds all it needs of a token's key
// in 4 G bytes side by side, and of its value in 2 G.
#pragma once

#include <cuda_fp16.h>
#include <math_constants.h>

#include "common.cuh"

namespace fe {

constexpr int KV4_TILE = 16;             // tokens of a tile; page sizes are multiples of it
constexpr int KV4_GROUP = 32;            // numbers that share a scale
constexpr int KV4_MAX_DIM = 256;
constexpr float KV4_LARGEST = 61440.f;   // numbers beyond are stored as this: centre and scale stay finite in half precision

__host__ __device__ constexpr int kv4_groups(int d) { return (d + KV4_GROUP - 1) / KV4_GROUP; }
__host__ __device__ constexpr int kv4_tile_bytes(int groups) { return 640 * groups; }
__host__ __device__ constexpr int kv4_value_codes(int groups) { return 256 * groups; }        // where a tile's parts begin
__host__ __device__ constexpr int kv4_key_pairs(int groups) { return 512 * groups; }
__host__ __device__ constexpr int kv4_value_pairs(int groups) { return 576 * groups; }

// Bytes of the four numbers 32 g + 4 p .. + 3 (p < 8) in a row of codes.
__device__ __forceinline__ int kv4_key_at(int g, int p, int groups) { return ((p >> 1) * groups + g) * 4 + (p & 1) * 2; }
__device__ __forceinline__ int kv4_value_at(int g, int p, int groups) { return (p * groups + g) * 2; }

// Eight codes of a word as four pairs of half-precision numbers: pair i holds the codes at bits 4 i and 16 + 4 i, as KV4_RAISED_EVEN + code
// (i even: four bits under the exponent of 1024) or KV4_RAISED_ODD + code (i odd: four bits higher, under that of 64).  Integers put under an exponent
// by bit operations: Kim et al., "Who Says Elephants Can't Run", 2022.
constexpr float KV4_RAISED_EVEN = 1024.f, KV4_RAISED_ODD = 64.f;
__device__ __forceinline__ void kv4_raise(unsigned w, unsigned* out) {
    const unsigned v = w >> 8;
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(out[0]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(out[1]) : "r"(w));
    asm("lop3.b32 %0, %1, 0x000f000f, 0x64006400, 0xea;" : "=r"(out[2]) : "r"(v));
    asm("lop3.b32 %0, %1, 0x00f000f0, 0x54005400, 0xea;" : "=r"(out[3]) : "r"(v));
}
// The same as code - 8; the subtraction is exact.
__device__ __forceinline__ void kv4_decode(unsigned w, unsigned* out) {
    const __half2 even = __halves2half2(__ushort_as_half(0x6408), __ushort_as_half(0x6408));       // 1024 + 8
    const __half2 odd = __halves2half2(__ushort_as_half(0x5480), __ushort_as_half(0x5480));        // 64 + 8
    kv4_raise(w, out);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&out[i]), (i & 1) ? odd : even);
        out[i] = *reinterpret_cast<const unsigned*>(&h);
    }
}

}  // namespace fe

// Matrices in microscaled 4-bit floating point (MXFP4): how they lie in memory, and the steps between floats and codes.
//
// An element is a sign, two bits of exponent and one of mantissa (E2M1): 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives, codes
// 0 to 7 and 8 to 15.  32 neighbours of a row (a block) share a power of two, held as its exponent + 127 in a byte (E8M0; 255: not
// a number).  In memory:
//   codes   [rows, width / 2]: element 2 j of a row in the low half of byte j, element 2 j + 1 in the high half; what bulk tensor
//           copies bring into shared memory as the tensor cores read it;
//   scales  in tiles of 128 rows x 4 blocks (512 bytes), the tile of rows r / 128 and blocks b / 4 at tile index
//           (r / 128) * tiles_of_a_row + b / 4, a scale at byte (r % 32) * 16 + (r % 128 / 32) * 4 + b % 4 of its tile: what
//           one copy into tensor memory takes.  A row of tiles covers a multiple of 256 elements; scales behind the row's end are 0.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

constexpr int MX_BLOCK = 32;
constexpr int MX_TILE_BYTES = 512;

__host__ __device__ __forceinline__ long long mx_tiles_of_a_row(long long width) { return (width + 255) / 256 * 2; }

// Where the four scales of row r's blocks 4 q to 4 q + 3 lie.
__device__ __forceinline__ size_t mx_scale_offset(long long r, long long q, long long tiles_of_a_row) {
    return (size_t)((r >> 7) * tiles_of_a_row + q) * MX_TILE_BYTES + (size_t)((r & 31) * 16 + ((r >> 5) & 3) * 4);
}

// Eight floats times `inverse` to eight codes, the first in the lowest bits: to the nearest, ties to the even code, above 6 to 6.
__device__ __forceinline__ uint32_t mx_encode_8(const float (&v)[8], float inverse) {
    uint32_t r;
    asm("{\n .reg .b8 b0, b1, b2, b3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n"
        " cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n"
        " mov.b32 %0, {b0, b1, b2, b3};\n}"
        : "=r"(r)
        : "f"(v[0] * inverse), "f"(v[1] * inverse), "f"(v[2] * inverse), "f"(v[3] * inverse), "f"(v[4] * inverse),
          "f"(v[5] * inverse), "f"(v[6] * inverse), "f"(v[7] * inverse));
    return r;
}

// Eight codes to four pairs of halfs (exact).  All four have to be used: where the compiler (nvcc 12.9) finds a byte of the unpacked word
// without a use it makes zeros of the others; for four codes there is mx_decode_4.
__device__ __forceinline__ void mx_decode_8(uint32_t codes, uint32_t (&h)[4]) {
    asm("{\n .reg .b8 b0, b1, b2, b3;\n mov.b32 {b0, b1, b2, b3}, %4;\n"
        " cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n cvt.rn.f16x2.e2m1x2 %2, b2;\n cvt.rn.f16x2.e2m1x2 %3, b3;\n}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3]) : "r"(codes));
}

// The four codes of the lowest 16 bits to two pairs of halfs (exact).
__device__ __forceinline__ void mx_decode_4(uint32_t codes, uint32_t (&h)[2]) {
    asm("{\n .reg .b8 b0, b1;\n .reg .b16 low;\n cvt.u16.u32 low, %2;\n mov.b16 {b0, b1}, low;\n"
        " cvt.rn.f16x2.e2m1x2 %0, b0;\n cvt.rn.f16x2.e2m1x2 %1, b1;\n}"
        : "=r"(h[0]), "=r"(h[1]) : "r"(codes));
}

// The scale byte of a block whose largest element has the float bits `largest` (sign off): its exponent less two, so that the
// largest lies in [4, 8) times the scale; 255 for a block with an infinity or NaN in it.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t largest) {
    const int exponent = (int)(largest >> 23);
    return exponent == 255 ? 255u : (uint32_t)max(exponent - 2, 0);
}

// An infinity or NaN of x decides its row's results by itself: the products of finite elements with finite weights change nothing of an
// infinity or NaN among the others (an infinity times a weight of 0 is none either).  So halfs and parts hold the infinities and NaN of a row, or
// of a block of it, beside zeros, and what a row has of them costs nothing.  A pair of bfloat16 as such halfs (halfs' upper bytes are E5M2):
__device__ __forceinline__ uint32_t mx_not_finite_pair(uint32_t pair) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t v = (pair >> (16 * i)) & 0xFFFFu, size = v & 0x7FFFu;
        if (size >= 0x7F80u) out |= ((v & 0x8000u) | (size == 0x7F80u ? 0x7C00u : 0x7E00u)) << (16 * i);
    }
    return out;
}

// Elements of x that another form of its rows (halfs, parts) does not hold, noted by stretches of 256 elements: how many a stretch has, or
// MX_LOST_ALL if more than MX_LOST, and behind all counts MX_LOST words a stretch, place in it << 16 | bfloat16.  The product adds theirs.
constexpr int MX_LOST = 8, MX_LOST_ALL = 255;
__host__ __device__ __forceinline__ const uint32_t* mx_lost_entries(const int* counts, long long stretches) {
    return reinterpret_cast<const uint32_t*>(counts) + (stretches + 3) / 4 * 4;
}
// What a row as halfs is described by: a power of two and how many of its elements are noted (up to MX_NOTED), in one number.
constexpr int MX_NOTED_BITS = 10, MX_NOTED = (1 << MX_NOTED_BITS) - 1;
// By a whole warp, eight elements a lane, those of `mask` lost; true if they are too many.
__device__ __forceinline__ bool mx_note_lost(uint32_t mask, const uint4& raw, long long stretch, int* counts, long long stretches) {
    const int lane = threadIdx.x & 31;
    int found = 0;
    if (__any_sync(0xffffffffu, mask != 0)) {
        uint32_t* entries = const_cast<uint32_t*>(mx_lost_entries(counts, stretches)) + stretch * MX_LOST;
        const uint32_t words[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t all = __ballot_sync(0xffffffffu, (mask >> i) & 1u);
            const int index = found + __popc(all & ((1u << lane) - 1u));
            if (((mask >> i) & 1u) && index < MX_LOST) entries[index] = (uint32_t)(lane * 8 + i) << 16 | ((words[i >> 1] >> (16 * (i & 1))) & 0xFFFFu);
            found += __popc(all);
        }
    }
    if (lane == 0) counts[stretch] = found > MX_LOST ? MX_LOST_ALL : found;
    return found > MX_LOST;
}

// 2^-(byte - 127) for bytes up to 252: an ordinary number.
__device__ __forceinline__ float mx_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }
// 2^(byte - 127); byte 0 is under the ordinary numbers, byte 255 gives NaN.
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte == 255u ? 0x7FC00000u : max(byte << 23, 0x00400000u));
}

// d += a . b of bfloat16, 16 rows x 8 columns x 16
__device__ __forceinline__ void mx_mma_bf16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

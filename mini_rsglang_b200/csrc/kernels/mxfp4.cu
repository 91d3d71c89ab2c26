// Rows of bfloat16 or float32 to microscaled 4-bit floating point and back (formats: mxfp4.cuh).
//
// For a block of 32 neighbours with largest size a: e = floor(log2 a) - 2, code = the nearest E2M1 value to x 2^-e (ties to the
// even code, above 6 to 6), scale = 2^e.  The power of two makes the multiplication exact, so a code is one rounding away from x.
// Four lanes share a block (eight elements each: a 16-byte load of bfloat16), sixteen lanes the four blocks whose scales are one
// word; two exchanges find a block's largest.  Bytes bound the kernels, once their instructions are few enough.
#include <limits.h>

#include "mxfp4.cuh"

namespace {

constexpr int THREADS = 256;

// What the kernel after this one counts with, set to zero on the way.
__device__ __forceinline__ void clear(int* zeros, int count) {
    for (int i = blockIdx.x * THREADS + threadIdx.x; i < count; i += gridDim.x * THREADS) zeros[i] = 0;
}

// Two 16-bit numbers a word, both at least 0: the larger ones.
__device__ __forceinline__ uint32_t larger_pair(uint32_t a, uint32_t b) { return __viaddmax_s16x2(a, 0u, b); }

// Eight elements as they come from memory, their largest size, and they themselves.  Only exponents count for a scale, so that sizes are
// compared as the upper 16 bits of float32; `of_two` gives those of two such eights in a word.
struct Eight {
    uint4 raw;
    __device__ __forceinline__ void load(const bf16* p) { raw = *reinterpret_cast<const uint4*>(p); }
    __device__ __forceinline__ uint32_t largest() const {
        const uint32_t m = larger_pair(raw.x & 0x7FFF7FFFu, raw.y & 0x7FFF7FFFu);
        return larger_pair(raw.w & 0x7FFF7FFFu, larger_pair(raw.z & 0x7FFF7FFFu, m));
    }
    __device__ __forceinline__ uint32_t largest_of_block() const {             // the float bits, from four lanes
        uint32_t m = largest();
        m = larger_pair(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = larger_pair(m, __shfl_xor_sync(0xffffffffu, m, 2));
        return max(m << 16, m & 0xFFFF0000u);
    }
    __device__ static __forceinline__ uint32_t of_two(uint32_t a, uint32_t b) { return larger_pair(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632)); }
    __device__ __forceinline__ void values(float (&v)[8]) const {
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    }
};
struct EightFloats {
    float4 a, b;
    __device__ __forceinline__ void load(const float* p) { a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1]; }
    __device__ __forceinline__ uint32_t largest() const {
        const float v[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        return m;
    }
    __device__ static __forceinline__ uint32_t of_two(uint32_t a, uint32_t b) { return __byte_perm(a, b, 0x7632); }
    __device__ __forceinline__ void values(float (&v)[8]) const { v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w; }
};
template <typename T> struct EightOf { typedef Eight Type; };
template <> struct EightOf<float> { typedef EightFloats Type; };

struct Stretch {
    unsigned row, index;               // of its row
    __device__ __forceinline__ Stretch(unsigned stretch, unsigned of_a_row) : row(stretch / of_a_row), index(stretch - row * of_a_row) {}
    __device__ __forceinline__ void next(unsigned of_a_row) {
        if (++index == of_a_row) index = 0, ++row;
    }
};

// A warp takes four stretches of 256 elements, one after the other in a row and then in the next, all loads first.  What it does beside
// loading and storing counts: with each stretch by itself it was 122 instructions a stretch, which filled the schedulers.  So largest sizes
// are found for two stretches at a time, their scales for four, and in rows of whole stretches (WHOLE) an element's place follows from its
// stretch's number: 80.  Stretches that reach over a row's end write zero scales there.
// 2,048 x 17,408 bfloat16: 38 us with one stretch in flight, 22 with four, 17.8 with 80 instructions (90 MB: 13.7 at the bandwidth of a
// copy); 5,003 x 5,120 float32 18.9 (17.7); dequantised 15.6 and 20.9.
template <typename T, bool WHOLE>
__global__ void __launch_bounds__(THREADS) quantise_kernel(const T* __restrict__ x, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                           unsigned rows, unsigned width, unsigned of_a_row, int* __restrict__ zeros, int zero_count) {
    pdl_launch_dependents();
    pdl_wait();
    clear(zeros, zero_count);
    const unsigned lane = threadIdx.x & 31, warps = gridDim.x * (THREADS / 32);
    const unsigned block = (lane >> 2) & 3, half = lane >> 4;                   // four lanes a block; blocks of half a stretch share a word of scales
    const unsigned stretches = rows * of_a_row;
    for (unsigned first = (blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5)) * 4; first < stretches; first += warps * 4) {
        typename EightOf<T>::Type held[4];
        size_t place[4];
        bool here[4];
        Stretch at(first, of_a_row);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const unsigned column = at.index * 256 + lane * 8;
            place[u] = WHOLE ? (size_t)(first + u) * 256 + lane * 8 : (size_t)at.row * width + column;
            here[u] = first + u < stretches && (WHOLE || column < width);
            held[u] = {};
            if (here[u]) held[u].load(x + place[u]);
            if (!WHOLE) at.next(of_a_row);
        }
        uint32_t largest[2], bytes[2];                                          // stretches 0 and 1, 2 and 3
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            largest[p] = EightOf<T>::Type::of_two(held[2 * p].largest(), held[2 * p + 1].largest());
            largest[p] = larger_pair(largest[p], __shfl_xor_sync(0xffffffffu, largest[p], 1));
            largest[p] = larger_pair(largest[p], __shfl_xor_sync(0xffffffffu, largest[p], 2));
            bytes[p] = __viaddmax_s16x2((largest[p] >> 7) & 0x00FF00FFu, 0xFFFEFFFEu, 0u);      // exponents less two, at least 0
        }
        uint32_t four = __byte_perm(bytes[0], bytes[1], 0x6420);                // a byte a stretch
        const uint32_t any = larger_pair(largest[0], largest[1]);
        if ((any & 0xFFFFu) >= 0x7F80u || any >= 0x7F800000u) {                 // an infinity or NaN: no numbers, codes of zeros
#pragma unroll
            for (int u = 0; u < 4; ++u)
                if (((largest[u >> 1] >> (16 * (u & 1))) & 0xFFFFu) >= 0x7F80u) held[u] = {}, four |= 0xFFu << (8 * u);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            float v[8];
            held[u].values(v);
            const uint32_t word = mx_encode_8(v, mx_inverse((bytes[u >> 1] >> (16 * (u & 1))) & 0xFFu));
            if (here[u]) *reinterpret_cast<uint32_t*>(codes + (place[u] >> 1)) = word;
        }
        // Four lanes' words of a byte a stretch become words of a byte a block, the lane of block u with stretch u.
        uint32_t other = __shfl_xor_sync(0xffffffffu, four, 8);
        four = __byte_perm(four, other, block & 2 ? 0x3276 : 0x5410);
        other = __shfl_xor_sync(0xffffffffu, four, 4);
        four = __byte_perm(four, other, block & 1 ? 0x3715 : 0x6240);
        if ((lane & 3) == 0 && first + block < stretches) {
            const Stretch mine(first + block, of_a_row);
            *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(mine.row, mine.index * 2 + half, of_a_row * 2)) = four;
        }
    }
}

// The same stretches back.  A lane makes what one 16-byte store takes: eight bfloat16, or four floats of each half of the stretch.
template <typename T>
__global__ void __launch_bounds__(THREADS) dequantise_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, T* __restrict__ out,
                                                             unsigned rows, unsigned width, unsigned of_a_row) {
    constexpr int UNROLL = 4, EACH = sizeof(T) == 2 ? 8 : 4, PARTS = 8 / EACH;
    pdl_launch_dependents();
    pdl_wait();
    const unsigned lane = threadIdx.x & 31, warps = gridDim.x * (THREADS / 32);
    const unsigned stretches = rows * of_a_row;
    for (unsigned first = (blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5)) * UNROLL; first < stretches; first += warps * UNROLL) {
        uint32_t word[UNROLL][PARTS], byte[UNROLL][PARTS];
        Stretch at(first, of_a_row);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u, at.next(of_a_row))
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const unsigned within = p * 128 + lane * EACH, column = at.index * 256 + within;
                word[u][p] = byte[u][p] = 0;
                if (first + u < stretches && column < width) {
                    const uint8_t* from = codes + (size_t)at.row * (width >> 1) + (column >> 1);
                    word[u][p] = EACH == 8 ? *reinterpret_cast<const uint32_t*>(from) : *reinterpret_cast<const uint16_t*>(from);
                    byte[u][p] = scales[mx_scale_offset(at.row, at.index * 2 + (within >> 7), of_a_row * 2) + ((within >> 5) & 3)];
                }
            }
        at = Stretch(first, of_a_row);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u, at.next(of_a_row))
#pragma unroll
            for (int p = 0; p < PARTS; ++p) {
                const unsigned column = at.index * 256 + p * 128 + lane * EACH;
                if (first + u >= stretches || column >= width) continue;
                const float scale = mx_scale(byte[u][p]);
                uint32_t h[EACH / 2];
                if constexpr (EACH == 8) mx_decode_8(word[u][p], h);
                else mx_decode_4(word[u][p], h);
                float v[EACH];
#pragma unroll
                for (int i = 0; i < EACH / 2; ++i) {
                    const float2 pair = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
                    v[2 * i] = pair.x * scale;
                    v[2 * i + 1] = pair.y * scale;
                }
                T* to = out + (size_t)at.row * width + column;
                if constexpr (EACH == 8) {
                    uint32_t w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        __nv_bfloat162 pair = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);       // exact: one bit of mantissa
                        w[i] = *reinterpret_cast<uint32_t*>(&pair);
                    }
                    *reinterpret_cast<uint4*>(to) = make_uint4(w[0], w[1], w[2], w[3]);
                } else {
                    *reinterpret_cast<float4*>(to) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
    }
}

// Scales [rows, width / 32] of a matrix from elsewhere into tiles; the codes of blocks whose scale is not a number become 0 (a
// product that multiplies a block's sum by its scale then gives NaN however it does so).
__global__ void __launch_bounds__(THREADS) scales_to_tiles_kernel(const uint8_t* __restrict__ plain, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales,
                                                                  long long rows, long long width, long long tiles_of_a_row) {
    pdl_wait();
    const long long total = rows * tiles_of_a_row * 4, blocks = width / MX_BLOCK;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
        const long long row = i / (tiles_of_a_row * 4), block = i - row * tiles_of_a_row * 4;
        const uint8_t byte = block < blocks ? plain[row * blocks + block] : (uint8_t)0;
        if (byte == 255) *reinterpret_cast<uint4*>(codes + row * (width >> 1) + block * 16) = make_uint4(0, 0, 0, 0);
        scales[mx_scale_offset(row, block >> 2, tiles_of_a_row) + (block & 3)] = byte;
    }
}

// The smallest and the largest scale byte below 255 of the blocks that are not all zeros, into range[0] and range[1] (which begin as 256
// and -1), and whether any block is not a number, into range[2] (0).
__global__ void __launch_bounds__(THREADS) scale_range_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int* __restrict__ range,
                                                              long long rows, long long width, long long tiles_of_a_row) {
    pdl_wait();
    const long long blocks = width / MX_BLOCK, total = rows * blocks;
    int low = 256, high = -1, bad = 0;
    for (long long i = (long long)blockIdx.x * THREADS + threadIdx.x; i < total; i += (long long)gridDim.x * THREADS) {
        const long long row = i / blocks, block = i - row * blocks;
        const int byte = scales[mx_scale_offset(row, block >> 2, tiles_of_a_row) + (block & 3)];
        const uint4 c = *reinterpret_cast<const uint4*>(codes + i * 16);
        if (byte == 255) bad = 1;
        else if (((c.x | c.y | c.z | c.w) & 0x77777777u) != 0u) low = min(low, byte), high = max(high, byte);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if ((threadIdx.x & 31) == 0) {
        atomicMin(&range[0], low);
        atomicMax(&range[1], high);
    }
    if (bad) atomicOr(&range[2], 1);
}

// Rows of bfloat16 as halfs times a power of two of the row's own: row r holds x 2^-exponents[r], its largest in [2^15, 2^16).  An element's
// exponent field becomes itself less that of the largest, plus 30, its mantissa its seven bits and three zeros: exact, but for elements
// 2^30 and more below the largest, which become 0 and are noted (a few in a prompt's products of gate and up), and rows below 2^-96.  Of a row
// with infinities or NaN these are held beside zeros (mxfp4.cuh).  factors[r] is the exponent in the upper bits and the number of noted elements in the lower ones (mxfp4.cuh); HALFS_LOST if there
// are more than fit or the row is one of the others, and not to be used.
constexpr int HELD = 4;
constexpr int HALFS_LOST = INT_MIN;
__global__ void __launch_bounds__(THREADS) rows_to_halfs_kernel(const bf16* __restrict__ x, uint16_t* __restrict__ halfs, int* __restrict__ factors,
                                                                int* __restrict__ noted, long long width, int* __restrict__ zeros, int zero_count) {
    __shared__ uint32_t scratch[THREADS / 32];
    __shared__ int number;                                       // of noted elements
    if (threadIdx.x == 0) number = 0;
    pdl_launch_dependents();
    pdl_wait();
    clear(zeros, zero_count);
    const long long row = blockIdx.x;
    const uint4* from = reinterpret_cast<const uint4*>(x + row * width);
    uint4* to = reinterpret_cast<uint4*>(halfs + row * width);
    const int chunks = (int)(width >> 3);
    uint4 held[HELD];
    uint32_t largest = 0;
    auto widen = [&](const uint4& v) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int p = 0; p < 4; ++p) largest = __viaddmax_s16x2(w[p] & 0x7FFF7FFFu, 0u, largest);
    };
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int i = j * THREADS + threadIdx.x;
        held[j] = i < chunks ? from[i] : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < HELD; ++j) widen(held[j]);
    for (int i = HELD * THREADS + threadIdx.x; i < chunks; i += THREADS) widen(from[i]);
    largest = __reduce_max_sync(0xffffffffu, max(largest & 0xFFFFu, largest >> 16));
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) largest = max(largest, scratch[w]);
    const int field = (int)(largest >> 7);
    const bool empty = largest == 0, ordinary = field >= 31 && field < 255;
    const uint32_t down = empty || !ordinary ? 0u : (uint32_t)(-((field - 30) << 7)) & 0xFFFFu, both = down | down << 16;
    if (field == 255) {
        for (int i = threadIdx.x; i < chunks; i += THREADS) {
            const uint4 v = from[i];
            to[i] = make_uint4(mx_not_finite_pair(v.x), mx_not_finite_pair(v.y), mx_not_finite_pair(v.z), mx_not_finite_pair(v.w));
        }
        if (threadIdx.x == 0) factors[row] = 0;
        return;
    }
    uint32_t lost = 0;
    auto convert = [&](const uint4& v, uint32_t* gone) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
        uint32_t h[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t size = w[p] & 0x7FFF7FFFu, r = __viaddmax_s16x2(size, both, 0u);
            h[p] = (r << 3) | (w[p] & 0x80008000u);
            gone[p] = (size + 0x7FFF7FFFu) & ~(r + 0x7F807F80u);              // highest bit of each half: not 0, and below the halfs' smallest ordinary number
            lost |= gone[p];
        }
        return make_uint4(h[0], h[1], h[2], h[3]);
    };
    uint32_t gone[4];
#pragma unroll
    for (int j = 0; j < HELD; ++j) {
        const int i = j * THREADS + threadIdx.x;
        if (i < chunks) to[i] = convert(held[j], gone);
    }
    for (int i = HELD * THREADS + threadIdx.x; i < chunks; i += THREADS) to[i] = convert(from[i], gone);
    bool bad = !(empty || ordinary);
    const bool some = __syncthreads_or((lost & 0x80008000u) != 0u);
    if (some && !bad) {                                                       // once more, with zeros in their place; a warp's 32 eights are a stretch
        const long long stretches = (width + 255) >> 8;
        for (int i = threadIdx.x; (i & ~31) < chunks; i += THREADS) {
            const uint4 v = i < chunks ? from[i] : make_uint4(0, 0, 0, 0);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            uint32_t mask = 0, h[4];
            *reinterpret_cast<uint4*>(h) = convert(v, gone);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint32_t both_of = (gone[p] >> 15) & 0x00010001u;
                h[p] &= ~(both_of * 0xFFFFu);
                mask |= (both_of & 1u) << (2 * p) | (both_of >> 16) << (2 * p + 1);
                if ((both_of & 1u) && field - (int)((w[p] >> 7) & 0xFFu) > 90) bad = true;       // so small that sums of halfs could not take it up
                if ((both_of >> 16) && field - (int)((w[p] >> 23) & 0xFFu) > 90) bad = true;
            }
            if (mask) to[i] = *reinterpret_cast<uint4*>(h);
            if (mx_note_lost(mask, v, row * stretches + (i >> 5), noted, gridDim.x * stretches)) bad = true;
            if (mask) atomicAdd(&number, __popc(mask));
        }
        bad = __syncthreads_or(bad);
    }
    if (threadIdx.x == 0) factors[row] = bad ? HALFS_LOST : (ordinary ? field - 127 - 15 : 0) * (1 << MX_NOTED_BITS) + min(number, MX_NOTED);
}

// Up to `tokens` rows of bfloat16 as three parts of E5M2 (three bits of significand, exponents of -16 to 15) each, part p of row r at row
// p * tokens + r, with a power of two for 32 neighbours in scale tiles (mxfp4.cuh) of these 3 * tokens rows.  With 2^(e - 14) for a block
// whose largest size has the exponent e, x = (a + b + c 2^-8) 2^(e - 14): a is x rounded, b what is left of it rounded, c, with
// a power 2^-8 further down, the rest: of eight bits three, three signed and two are enough down to 2^-26 of the largest.  Elements of
// which that is not so are 0 in all parts and noted.  Infinities and NaN are what they are in the first part, beside zeros in their block (mxfp4.cuh).
constexpr int PART_SHIFT = 8;
__global__ void __launch_bounds__(THREADS) rows_to_parts_kernel(const bf16* __restrict__ x, uint8_t* __restrict__ parts, uint8_t* __restrict__ scales,
                                                                int* __restrict__ lost, int rows, int width, int tokens, int stretches, int* __restrict__ zeros,
                                                                int zero_count) {
    pdl_launch_dependents();
    pdl_wait();
    clear(zeros, zero_count);
    const int lane = threadIdx.x & 31, index = (int)blockIdx.x * (THREADS / 32) + (threadIdx.x >> 5);
    if (index >= rows * stretches) return;
    const int row = index / stretches, stretch = index - row * stretches, column = stretch * 256 + lane * 8;
    Eight held = {};
    if (column < width) held.load(x + (size_t)row * width + column);
    const uint32_t largest = held.largest_of_block();
    const int e = (int)(largest >> 23) - 127;                    // 128: infinity or NaN
    const bool ordinary = largest != 0 && e >= -105 && e < 128;
    const uint32_t byte = ordinary ? (uint32_t)(e - 14 + 127) : 127u;
    const float up = mx_inverse(byte), down = mx_scale(byte);
    float v[8];
    held.values(v);
    uint32_t a[2] = {0, 0}, b[2] = {0, 0}, c[2] = {0, 0}, mask = 0;
    auto part_of = [](float f) {
        uint16_t two;
        asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(two) : "f"(0.0f), "f"(f));
        return (uint32_t)two & 255u;
    };
    auto value_of = [](uint32_t part) { return __half2float(__ushort_as_half((unsigned short)(part << 8))); };      // E5M2 is a half's upper byte
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float scaled = v[i] * up;
        const uint32_t first = part_of(scaled);
        const float left = scaled - value_of(first);
        const uint32_t second = part_of(left);
        const float rest = (left - value_of(second)) * (float)(1 << PART_SHIFT);
        const uint32_t third = part_of(rest);
        if ((value_of(first) + value_of(second) + value_of(third) * (1.0f / (1 << PART_SHIFT))) * down != v[i]) {
            mask |= 1u << i;
            continue;
        }
        a[i >> 2] |= first << (8 * (i & 3));
        b[i >> 2] |= second << (8 * (i & 3));
        c[i >> 2] |= third << (8 * (i & 3));
    }
    if (e == 128) {
        const uint32_t w[4] = {held.raw.x, held.raw.y, held.raw.z, held.raw.w};
        mask = a[0] = a[1] = b[0] = b[1] = c[0] = c[1] = 0;
#pragma unroll
        for (int p = 0; p < 4; ++p) a[p >> 1] |= __byte_perm(mx_not_finite_pair(w[p]), 0, 0x4431) << (16 * (p & 1));
    }
    if (column < width) {
        *reinterpret_cast<uint2*>(parts + (size_t)row * width + column) = make_uint2(a[0], a[1]);
        *reinterpret_cast<uint2*>(parts + (size_t)(tokens + row) * width + column) = make_uint2(b[0], b[1]);
        *reinterpret_cast<uint2*>(parts + (size_t)(2 * tokens + row) * width + column) = make_uint2(c[0], c[1]);
    }
    uint32_t four = byte << (8 * ((lane >> 2) & 3));
    four |= __shfl_xor_sync(0xffffffffu, four, 4);
    four |= __shfl_xor_sync(0xffffffffu, four, 8);
    if ((lane & 15) == 0) {
        const int tiles = stretches * 2, q = stretch * 2 + (lane >> 4);
        *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(row, q, tiles)) = four;
        *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(tokens + row, q, tiles)) = four;
        *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(2 * tokens + row, q, tiles)) = four - 0x01010101u * PART_SHIFT;
    }
    mx_note_lost(mask, held.raw, index, lost, (long long)rows * stretches);
}

__global__ void __launch_bounds__(THREADS) clear_kernel(int* __restrict__ zeros, int count) {
    pdl_launch_dependents();
    pdl_wait();
    clear(zeros, count);
}

// Blocks of a launch over `items` threads of work: they loop where that is more than 64 blocks an SM.
int blocks_for(long long items) {
    const long long want = (items + THREADS - 1) / THREADS, most = (long long)mrs_sm_count() * 64;
    return (int)(want < 1 ? 1 : want < most ? want : most);
}

// (rows x stretches of 256 elements are counted in 32 bits)
bool bad_sizes(long long rows, long long width) {
    return rows < 0 || width <= 0 || width % MX_BLOCK || width > (1ll << 30) || rows > (1ll << 31) || rows * ((width + 255) / 256) > (1ll << 31);
}

}  // namespace

// Bytes of a matrix's scales.
MRS_EXPORT long long mrs_mxfp4_scale_bytes(long long rows, long long width) {
    return (rows + 127) / 128 * mx_tiles_of_a_row(width) * MX_TILE_BYTES;
}

// x [rows, width] bfloat16 (`is_bf16`) or float32 on 16-byte boundaries, width a multiple of 32.  `zeros`: `zero_count` ints that are set to 0, or null.
MRS_EXPORT int mrs_mxfp4_quantise(int is_bf16, const void* x, void* codes, void* scales, long long rows, long long width, void* zeros, int zero_count, void* stream) {
    if (rows == 0) return 0;
    if (bad_sizes(rows, width) || (zero_count && !zeros) || !x || !codes || !scales || (((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15)) return MRS_BAD_ARGUMENT;
    const unsigned of_a_row = (unsigned)((width + 255) / 256);
    const int blocks = blocks_for(rows * of_a_row * 8);
#define MRS_QUANTISE(T, WHOLE) MRS_LAUNCH((quantise_kernel<T, WHOLE>), blocks, THREADS, 0, stream, (const T*)x, (uint8_t*)codes, (uint8_t*)scales, (unsigned)rows, (unsigned)width, of_a_row, (int*)zeros, zero_count)
    if (is_bf16 && width % 256 == 0) MRS_QUANTISE(bf16, true);
    else if (is_bf16) MRS_QUANTISE(bf16, false);
    else if (width % 256 == 0) MRS_QUANTISE(float, true);
    else MRS_QUANTISE(float, false);
#undef MRS_QUANTISE
    MRS_RETURN_LAUNCH_STATUS();
}

MRS_EXPORT int mrs_mxfp4_dequantise(int is_bf16, const void* codes, const void* scales, void* out, long long rows, long long width, void* stream) {
    if (rows == 0) return 0;
    if (bad_sizes(rows, width) || !out || !codes || !scales || (((uintptr_t)out | (uintptr_t)codes | (uintptr_t)scales) & 15)) return MRS_BAD_ARGUMENT;
    const unsigned of_a_row = (unsigned)((width + 255) / 256);
    const int blocks = blocks_for(rows * of_a_row * 8);
    if (is_bf16) MRS_LAUNCH(dequantise_kernel<bf16>, blocks, THREADS, 0, stream, (const uint8_t*)codes, (const uint8_t*)scales, (bf16*)out, (unsigned)rows, (unsigned)width, of_a_row);
    else MRS_LAUNCH(dequantise_kernel<float>, blocks, THREADS, 0, stream, (const uint8_t*)codes, (const uint8_t*)scales, (float*)out, (unsigned)rows, (unsigned)width, of_a_row);
    MRS_RETURN_LAUNCH_STATUS();
}

MRS_EXPORT int mrs_mxfp4_scales_to_tiles(const void* plain, void* codes, void* scales, long long rows, long long width, void* stream) {
    if (rows == 0) return 0;
    if (bad_sizes(rows, width) || !plain || !codes || !scales || (((uintptr_t)codes | (uintptr_t)scales) & 15)) return MRS_BAD_ARGUMENT;
    const long long tiles = mx_tiles_of_a_row(width);
    MRS_LAUNCH(scales_to_tiles_kernel, blocks_for(rows * tiles * 4), THREADS, 0, stream, (const uint8_t*)plain, (uint8_t*)codes, (uint8_t*)scales, rows, width, tiles);
    MRS_RETURN_LAUNCH_STATUS();
}

// range: three ints, 256, -1 and 0 to begin with.
MRS_EXPORT int mrs_mxfp4_scale_range(const void* codes, const void* scales, void* range, long long rows, long long width, void* stream) {
    if (rows == 0) return 0;
    if (bad_sizes(rows, width) || !range || !codes || !scales || (((uintptr_t)codes | (uintptr_t)scales) & 15) || ((uintptr_t)range & 3)) return MRS_BAD_ARGUMENT;
    MRS_LAUNCH(scale_range_kernel, blocks_for(rows * (width / MX_BLOCK)), THREADS, 0, stream, (const uint8_t*)codes, (const uint8_t*)scales, (int*)range, rows, width,
               mx_tiles_of_a_row(width));
    MRS_RETURN_LAUNCH_STATUS();
}

// x [rows, width] bfloat16 to halfs [rows, width], factors [rows] int32 and lost (mxfp4.cuh; rows * ceil(width / 256) stretches).  `zeros`: `zero_count` ints that are set to 0, or null.
MRS_EXPORT int mrs_mxfp4_rows_to_halfs(const void* x, void* halfs, void* factors, void* lost, long long rows, long long width, void* zeros, int zero_count,
                                       void* stream) {
    if (rows == 0) return 0;
    if (bad_sizes(rows, width) || (zero_count && !zeros) || rows > 0x7FFFFFFF || !x || !halfs || !factors || !lost || (((uintptr_t)x | (uintptr_t)halfs) & 15) || (((uintptr_t)factors | (uintptr_t)lost) & 3)) return MRS_BAD_ARGUMENT;
    MRS_LAUNCH(rows_to_halfs_kernel, (unsigned)rows, THREADS, 0, stream, (const bf16*)x, (uint16_t*)halfs, (int*)factors, (int*)lost, width, (int*)zeros, zero_count);
    MRS_RETURN_LAUNCH_STATUS();
}

// x [rows, width] bfloat16, rows up to `tokens` (16, 32 or 64), to parts [3 tokens, width], their scales and lost (as above).
MRS_EXPORT int mrs_mxfp4_rows_to_parts(const void* x, void* parts, void* scales, void* lost, int rows, int width, int tokens, void* zeros, int zero_count,
                                       void* stream) {
    if (rows == 0) return 0;
    if (bad_sizes(rows, width) || rows > tokens || (tokens != 16 && tokens != 32 && tokens != 64) || (zero_count && !zeros) || !x || !parts || !scales || !lost ||
        (((uintptr_t)x | (uintptr_t)parts | (uintptr_t)scales) & 15) || ((uintptr_t)lost & 3))
        return MRS_BAD_ARGUMENT;
    const int stretches = (width + 255) / 256;
    MRS_LAUNCH(rows_to_parts_kernel, (rows * stretches + THREADS / 32 - 1) / (THREADS / 32), THREADS, 0, stream, (const bf16*)x, (uint8_t*)parts, (uint8_t*)scales,
               (int*)lost, rows, width, tokens, stretches, (int*)zeros, zero_count);
    MRS_RETURN_LAUNCH_STATUS();
}

// `zero_count` ints that are set to 0.
MRS_EXPORT int mrs_mxfp4_clear(void* zeros, int zero_count, void* stream) {
    if (zero_count == 0) return 0;
    if (zero_count < 0 || !zeros || ((uintptr_t)zeros & 3)) return MRS_BAD_ARGUMENT;
    MRS_LAUNCH(clear_kernel, blocks_for(zero_count), THREADS, 0, stream, (int*)zeros, zero_count);
    MRS_RETURN_LAUNCH_STATUS();
}

MRS_EXPORT const char* mrs_mxfp4_error_string(int code) {
    if (code == MRS_BAD_ARGUMENT) return "arguments outside what the kernels support (width no multiple of 32, unaligned base, a plan for other sizes)";
    if (code == -3) return "the driver refused the tensor map (address, sizes or strides)";
    return cudaGetErrorString((cudaError_t)code);
}

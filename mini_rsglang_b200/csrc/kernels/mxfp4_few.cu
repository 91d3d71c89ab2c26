// Products of few rows with a matrix in microscaled 4-bit floating point: out[m, n] = sum_k x[m, k] w[n, k], x bfloat16 (or brought
// to 4 bits here, block by block, by the rule of mxfp4.cuh), w in 4 bits, sums in float32.
//
// The bytes of w bound it: half a byte and a 32nd a weight, read once.  A warp owns 16 rows of w and a range of K, and copies
// its own 128-byte pieces of them (16 rows x 256 elements) into a ring of its own in shared memory with cp.async, so that no
// barrier stands in its loop.  A word of eight codes becomes four pairs of halfs (exact) that are A fragments of mma.m16n8k16 as
// they stand: the order of K within a block is free as long as x has the same, so lane (g, t) takes the codes 8 t to 8 t + 7
// of a block as its K indices of two MMAs and the same eight elements of x.  A block's two MMAs start from zero, and their sums are
// multiplied by the powers of two of the block and of x as they join the row's float32 sums: products of halfs are exact, every sum is
// float32.
//
// One CTA of 16 warps an SM takes an equal share of the groups of 16 rows and keeps x in shared memory for all of them.  Its
// (group, stage of 256 elements) pairs, group by group, are cut into 16 equal runs, one a warp: a warp's first and last group may
// be shared with its neighbours, whose sums meet in shared memory in the order of K.  Where x does not fit, the CTAs of a cluster
// take a range of K each and their sums meet in the ranges' order.  A result does not depend on timing.
//
// x as halfs.  A warp brings a stage of x, all tokens, into the halfs' range by one power of two, which goes into the stage's scales.
// (Where it times a scale of w may be under float32's range, it goes into the sums before the scales do: 24,576 x 4,096 times one row 13.6
// us instead of 13.0.)
// Where halfs could lose a bit of any element (2^29 and more between the sizes of two), or x has an element there that is not finite,
// or the power is beyond [2^-20, 2^15], the stage is multiplied in bfloat16 instead: x as it is, codes times their scale, which takes more
// steps to make (18.6 us).  The same products, and no sum of them before the scales, which could leave float32's range on the way.
//
// Measured from a cold L2: 24,576 x 4,096 (53 MB) 12.9 us for one token and 14.4 for eight, 6,144 x 4,096 5.9 and 7.1, 1,000 x 2,048 2.6 and
// 3.4: 4.9 us to begin and to end, then 5.7 TB/s.  tcgen05 kernels (mxfp4_tc.cu) begin with a second kernel that prepares x.
#include "mxfp4.cuh"

namespace {

constexpr int WARPS = 16, THREADS = WARPS * 32;
constexpr int STAGE_K = 256;                       // elements of K a stage: 128 bytes a row
constexpr int CODE_BYTES = 16 * 128, SCALE_BYTES = 16 * 8, STAGE_BYTES = CODE_BYTES + SCALE_BYTES;
constexpr int RING = 3;
constexpr int FACTOR_BYTES = 16 * 8 * 4;           // a stage's scales as floats
constexpr int X_PAD = 64;                          // bytes behind a row of x: two rows then fill all banks
constexpr int TOKENS = 8, GROUP_SUMS = TOKENS * 16;      // the N of the MMA
constexpr int MAX_STAGES = 512;                    // of x in shared memory
constexpr int SMEM_MOST = 227 * 1024 - 2560;
constexpr int ROUND_GROUPS = 16;                   // groups whose sums wait for the cluster's others at a time

__device__ __forceinline__ uint32_t smem_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_4(uint32_t dst, const void* src) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// d = a . b of halfs, and d += a . b
__device__ __forceinline__ void mma_first(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                 : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ void mma_more(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A half pair of codes times their scale as a pair of bfloat16 (exact: a code has two bits of significand; where the scale is not a
// number, infinity beside codes of 0, it is none).
__device__ __forceinline__ uint32_t as_bf16_pair(uint32_t halfs, __nv_bfloat162 scale) {
    const float2 v = __half22float2(*reinterpret_cast<__half2*>(&halfs));
    __nv_bfloat162 pair = __hmul2(__floats2bfloat162_rn(v.x, v.y), scale);
    return *reinterpret_cast<uint32_t*>(&pair);
}

struct Shapes {
    int M, N, K;
    int cluster;            // CTAs that share their groups, a range of K each
    int x_stages;           // the longest of these ranges, in stages
    float least_factor;     // that times any of w's scales is still a float; above 0
    int early;              // w was there before the kernel before this one: it may be fetched while that runs
    int groups_each, groups_over;      // of 16 rows a share (CTA or cluster): so many, and one more for the first `groups_over`
    int stages_each, stages_over;      // of K a CTA of a cluster, likewise
};

// Where range r begins: ranges of `each`, the first `over` of them one longer.  (Divisions in a kernel's first steps, 64-bit ones above
// all, cost it more than a stage of products.)
__device__ __forceinline__ int range_start(int each, int over, int r) { return each * r + min(r, over); }
__device__ __forceinline__ int range_of(int each, int over, int index) {
    const int longer = over * (each + 1);
    return index < longer ? (int)((unsigned)index / (unsigned)(each + 1)) : over + (int)((unsigned)(index - longer) / (unsigned)max(each, 1));
}

__device__ __forceinline__ uint32_t shared_word(uint32_t address) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(address) : "memory");
    return v;
}

// How a stage of x lies in shared memory (`factor` of bring_x): as halfs whose power goes into the scales, as halfs whose power is so small
// that it goes into the sums, as it is.
enum Form { HALFS, SMALL_HALFS, BFLOATS };

// One stage of a warp's rows joined to its sums.  `factors`: room for the stage's scales as floats.
template <Form FORM>
__device__ __forceinline__ void stage_products(uint32_t stage, float* factors, const unsigned char* x_stage, int x_pitch, float factor,
                                               int live, float (&sums)[4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    {
        // lane: row lane / 2, blocks 4 (lane % 2) to 4 (lane % 2) + 3.  Byte 0 is 2^-127; byte 255, not a number, stands beside codes of 0:
        // infinity times a sum of 0 is NaN.
        const uint32_t word = shared_word(stage + CODE_BYTES + lane * 4);
        float4 f;
        f.x = __uint_as_float(max((word << 23) & 0x7F800000u, 0x00400000u));
        f.y = __uint_as_float(max((word << 15) & 0x7F800000u, 0x00400000u));
        f.z = __uint_as_float(max((word << 7) & 0x7F800000u, 0x00400000u));
        f.w = __uint_as_float(max((word >> 1) & 0x7F800000u, 0x00400000u));
        if constexpr (FORM == HALFS) f.x *= factor, f.y *= factor, f.z *= factor, f.w *= factor;
        *reinterpret_cast<float4*>(factors + lane * 4) = f;
        __syncwarp();
    }
    const uint32_t codes = stage + g * 128 + g * 16 + t * 4;                  // stages are multiples of 128 bytes: block b lies 16 b xor-ed further
    const unsigned char* x_row = x_stage + (g < live ? g : 0) * x_pitch + t * 16;        // tokens that are not there read the first: nobody stores their sums
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const float4 f_low = *reinterpret_cast<const float4*>(factors + g * 8 + half * 4);
        const float4 f_high = *reinterpret_cast<const float4*>(factors + (g + 8) * 8 + half * 4);
        const float s_low[4] = {f_low.x, f_low.y, f_low.z, f_low.w}, s_high[4] = {f_high.x, f_high.y, f_high.z, f_high.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = half * 4 + i;
            uint32_t low[4], high[4];
            mx_decode_8(shared_word(codes ^ (b * 16)), low);
            mx_decode_8(shared_word((codes ^ (b * 16)) + 8 * 128), high);
            if constexpr (FORM == BFLOATS) {
                const __nv_bfloat162 scale_low = __float2bfloat162_rn(s_low[i]), scale_high = __float2bfloat162_rn(s_high[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) low[j] = as_bf16_pair(low[j], scale_low), high[j] = as_bf16_pair(high[j], scale_high);
            }
            const uint32_t a0[4] = {low[0], high[0], low[1], high[1]}, a1[4] = {low[2], high[2], low[3], high[3]};
            const uint4 xs = *reinterpret_cast<const uint4*>(x_row + b * 64);
            if constexpr (FORM == BFLOATS) {
                mx_mma_bf16(sums, a0, xs.x, xs.y);
                mx_mma_bf16(sums, a1, xs.z, xs.w);
                continue;
            }
            float d[4];
            mma_first(d, a0, xs.x, xs.y);
            mma_more(d, a1, xs.z, xs.w);
            if constexpr (FORM == SMALL_HALFS) d[0] *= factor, d[1] *= factor, d[2] *= factor, d[3] *= factor;         // exact
            sums[0] = fmaf(d[0], s_low[i], sums[0]);
            sums[1] = fmaf(d[1], s_low[i], sums[1]);
            sums[2] = fmaf(d[2], s_high[i], sums[2]);
            sums[3] = fmaf(d[3], s_high[i], sums[3]);
        }
    }
}

// Eight elements of x, pairs of bfloat16, as what their 4-bit codes stand for (four lanes a block).
__device__ __forceinline__ uint4 through_codes(uint4 raw) {
    uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
    float v[8];
    uint32_t largest = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(w[i] << 16);
        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        largest = max(largest, max(__float_as_uint(v[2 * i]) & 0x7FFFFFFFu, __float_as_uint(v[2 * i + 1]) & 0x7FFFFFFFu));
    }
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 1));
    largest = max(largest, __shfl_xor_sync(0xffffffffu, largest, 2));
    const uint32_t byte = mx_scale_byte(largest);
    const float scale = mx_scale(byte);
    uint32_t h[4];
    mx_decode_8(byte == 255u ? 0u : mx_encode_8(v, mx_inverse(byte)), h);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 pair = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
        __nv_bfloat162 rounded = __floats2bfloat162_rn(pair.x * scale, pair.y * scale);       // exact
        w[i] = *reinterpret_cast<uint32_t*>(&rounded);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// A stage of x, the rows first_token .. + live, into shared memory by one warp (what lies behind K as zeros).  Returns the factor 2^(e - 15)
// of elements that lie there as halfs times 2^(15 - e), or 0 where that might lose a bit and they lie there as they are.
template <bool QUANTISE>
__device__ __forceinline__ float bring_x(const bf16* __restrict__ x, unsigned char* place, int x_pitch, int live, int column, int K) {
    uint4 held[TOKENS];
    uint32_t largest = 0;                                                     // a pair
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) {
        held[j] = make_uint4(0, 0, 0, 0);
        if (j < live && column < K) held[j] = *reinterpret_cast<const uint4*>(x + (size_t)j * K + column);
    }
#pragma unroll
    for (int j = 0; j < TOKENS; ++j) {
        if (j >= live) break;
        if constexpr (QUANTISE) held[j] = through_codes(held[j]);
        const uint32_t w[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
#pragma unroll
        for (int p = 0; p < 4; ++p) largest = __viaddmax_s16x2(w[p] & 0x7FFF7FFFu, 0u, largest);
    }
    largest = __reduce_max_sync(0xffffffffu, max(largest & 0xFFFFu, largest >> 16));
    const int field = (int)(largest >> 7), e = largest == 0 ? 0 : field - 127;
    bool exact = e >= -20 && e <= 15;                                         // not with infinities or NaN
    uint32_t lost = 0;
    if (exact) {
        // a half's exponent field is the element's less that of the largest, plus 30; its mantissa the element's seven bits, then zeros
        const uint32_t down = (uint32_t)(-((e + 127 - 30) << 7)) & 0xFFFFu, both = down | down << 16;
#pragma unroll
        for (int j = 0; j < TOKENS; ++j) {
            if (j >= live) break;
            const uint32_t w[4] = {held[j].x, held[j].y, held[j].z, held[j].w};
            uint32_t h[4];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const uint32_t size = w[p] & 0x7FFF7FFFu, r = __viaddmax_s16x2(size, both, 0u);
                lost |= (size + 0x7FFF7FFFu) & ~(r + 0x7F807F80u);            // highest bit of each half: not 0, and below the halfs' smallest ordinary number
                h[p] = (r << 3) | (w[p] & 0x80008000u);
            }
            *reinterpret_cast<uint4*>(place + j * x_pitch) = make_uint4(h[0], h[1], h[2], h[3]);
        }
    }
    exact = exact && !__any_sync(0xffffffffu, (lost & 0x80008000u) != 0u);
    if (exact) return __uint_as_float((uint32_t)(127 + e - 15) << 23);
#pragma unroll
    for (int j = 0; j < TOKENS; ++j)
        if (j < live) *reinterpret_cast<uint4*>(place + j * x_pitch) = held[j];
    return 0.0f;
}

template <bool QUANTISE, typename Out>
__global__ void __launch_bounds__(THREADS, 1) few_rows_kernel(const bf16* __restrict__ x, const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, Out* __restrict__ out, const Shapes s) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ float x_factors[MAX_STAGES];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x & (s.cluster - 1), share = blockIdx.x >> (31 - __clz(s.cluster));
    const int group_from = range_start(s.groups_each, s.groups_over, share), group_to = range_start(s.groups_each, s.groups_over, share + 1);
    const int first_token = blockIdx.y * TOKENS, live = min(TOKENS, s.M - first_token);
    const int k_from = range_start(s.stages_each, s.stages_over, rank), k_to = range_start(s.stages_each, s.stages_over, rank + 1), depth = k_to - k_from;

    unsigned char* place = smem;
    const uint32_t ring = smem_address(place + warp * (RING * STAGE_BYTES));
    place += WARPS * RING * STAGE_BYTES;
    float* factors = reinterpret_cast<float*>(place + warp * FACTOR_BYTES);
    place += WARPS * FACTOR_BYTES;
    float* pieces = reinterpret_cast<float*>(place);                          // [warp][its first group, its last][token][row]
    place += WARPS * 2 * GROUP_SUMS * 4;
    float* whole = reinterpret_cast<float*>(place);                           // [group of the round][token][row], for the cluster
    if (s.cluster > 1) place += ROUND_GROUPS * GROUP_SUMS * 4;
    unsigned char* x_smem = place;
    const int x_pitch = s.x_stages * (STAGE_K * 2) + X_PAD;

    // Without a cluster one round takes all of the CTA's groups.
    const int round_groups = s.cluster > 1 ? ROUND_GROUPS : group_to - group_from;
    const long long code_pitch = s.K >> 1, tiles_of_a_row = mx_tiles_of_a_row(s.K);
    const uint32_t even = (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) << 4);                  // rows lane / 8 and + 8 of a stage
    const uint32_t odd = (4 + (lane >> 3)) * 128 + (((lane & 7) ^ (4 + (lane >> 3))) << 4);       // rows lane / 8 + 4 and + 12

    bool waited = false;
    for (int first = group_from; first < group_to; first += round_groups) {
        const int count = min(round_groups, group_to - first), units = count * depth;
        const int unit_each = units / WARPS, unit_over = units % WARPS;
        const int unit_from = range_start(unit_each, unit_over, warp), unit_to = range_start(unit_each, unit_over, warp + 1);
        const int first_index = depth ? (int)((unsigned)unit_from / (unsigned)depth) : 0, first_stage = unit_from - first_index * depth;

        // The copies' walk through this warp's units: four 16-byte copies and one of four scales a lane.  Rows behind N and columns behind K
        // are copies of the last (their sums are not stored; x is 0 there): nothing is read out of range.
        int copy_group = first + first_index, copy_stage = k_from + first_stage, left = unit_to - unit_from;
        uint32_t copy_offset = 0, used_offset = 0;
        const uint8_t *from0, *from1, *from2, *from3, *from_scales;
        auto start_group = [&]() {
            const long long row = (long long)copy_group * 16 + (lane >> 3), last = s.N - 1;
            const uint8_t* base = codes + (long long)copy_stage * 128 + (lane & 7) * 16;
            from0 = base + min(row, last) * code_pitch;
            from1 = base + min(row + 4, last) * code_pitch;
            from2 = base + min(row + 8, last) * code_pitch;
            from3 = base + min(row + 12, last) * code_pitch;
            from_scales = scales + mx_scale_offset(min((long long)copy_group * 16 + (lane >> 1), last), copy_stage * 2 + (lane & 1), tiles_of_a_row);
        };
        auto copy_next = [&]() {
            if (left > 0) {
                const uint32_t base = ring + copy_offset;
                const int behind = max(copy_stage * 128 + (lane & 7) * 16 + 16 - (int)code_pitch, 0);      // 0 but at the end of rows that end inside a stage
                copy_16(base + even, from0 - behind);
                copy_16(base + odd, from1 - behind);
                copy_16(base + even + 8 * 128, from2 - behind);
                copy_16(base + odd + 8 * 128, from3 - behind);
                copy_4(base + CODE_BYTES + lane * 4, from_scales);
                from0 += 128, from1 += 128, from2 += 128, from3 += 128;
                from_scales += 2 * MX_TILE_BYTES;
                --left;
                if (++copy_stage == k_to) {
                    ++copy_group;
                    copy_stage = k_from;
                    if (left > 0) start_group();
                }
            }
            copy_offset = copy_offset + STAGE_BYTES == RING * STAGE_BYTES ? 0 : copy_offset + STAGE_BYTES;
            copy_commit();
        };
        if (left > 0) start_group();

        if (!waited && !s.early) pdl_wait();
#pragma unroll
        for (int i = 0; i < RING - 1; ++i) copy_next();
        if (!waited) {
            pdl_launch_dependents();
            if (s.early) pdl_wait();
            waited = true;
            for (int stage = warp; stage < depth; stage += WARPS) {
                const float factor = bring_x<QUANTISE>(x + (size_t)first_token * s.K, x_smem + stage * (STAGE_K * 2) + lane * 16, x_pitch, live,
                                                       (k_from + stage) * STAGE_K + lane * 8, s.K);
                if (lane == 0) x_factors[stage] = factor;
            }
            __syncthreads();
        }

        int group = first + first_index, stage = first_stage;                   // of the CTA's range
        for (int unit = unit_from; unit < unit_to; ++group, stage = 0) {
            const int stop = min(unit + depth - stage, unit_to);               // of this warp's piece of the group
            const bool alone = stage == 0 && stop - unit == depth;
            float sums[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const int slot = unit == unit_from ? 0 : 1;
            const unsigned char* x_stage = x_smem + stage * (STAGE_K * 2);
            for (; unit < stop; ++unit, ++stage, x_stage += STAGE_K * 2) {
                const float factor = x_factors[stage];
                copy_wait<RING - 2>();
                __syncwarp();
                copy_next();
                if (factor >= s.least_factor) stage_products<HALFS>(ring + used_offset, factors, x_stage, x_pitch, factor, live, sums);
                else if (factor != 0.0f) stage_products<SMALL_HALFS>(ring + used_offset, factors, x_stage, x_pitch, factor, live, sums);
                else stage_products<BFLOATS>(ring + used_offset, factors, x_stage, x_pitch, factor, live, sums);
                used_offset = used_offset + STAGE_BYTES == RING * STAGE_BYTES ? 0 : used_offset + STAGE_BYTES;
                __syncwarp();
            }
            const int g = lane >> 2, t = lane & 3;
            if (alone && s.cluster == 1) {                                      // these sums are the results
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int token = 2 * t + (i & 1);
                    const long long row = (long long)group * 16 + g + (i >> 1) * 8;
                    if (token < live && row < s.N) out[(size_t)(first_token + token) * s.N + row] = from_float<Out>(sums[i]);
                }
            } else {
                float* mine = alone ? whole + (group - first) * GROUP_SUMS : pieces + (warp * 2 + slot) * GROUP_SUMS;
#pragma unroll
                for (int i = 0; i < 4; ++i) mine[(2 * t + (i & 1)) * 16 + g + (i >> 1) * 8] = sums[i];
            }
        }
        copy_wait<0>();
        __syncthreads();

        // groups that several warps share: their pieces in the order of K
        for (int index = warp; index < count; index += WARPS) {
            const int begin = index * depth;
            const int low = units ? range_of(unit_each, unit_over, begin) : 0, high = units ? range_of(unit_each, unit_over, begin + depth - 1) : 0;
            if (units && low == high) continue;
            float sum[GROUP_SUMS / 32];
            const float* piece = pieces + (low * 2 + (range_start(unit_each, unit_over, low) >= begin ? 0 : 1)) * GROUP_SUMS + lane;
#pragma unroll
            for (int i = 0; i < GROUP_SUMS / 32; ++i) sum[i] = units ? piece[i * 32] : 0.0f;
            for (int w = low + 1; w <= high; ++w) {
                piece = pieces + w * 2 * GROUP_SUMS + lane;
#pragma unroll
                for (int i = 0; i < GROUP_SUMS / 32; ++i) sum[i] += piece[i * 32];
            }
            const long long row = (long long)(first + index) * 16 + (lane & 15);
#pragma unroll
            for (int i = 0; i < GROUP_SUMS / 32; ++i) {
                const int token = i * 2 + (lane >> 4);
                if (s.cluster > 1) whole[index * GROUP_SUMS + i * 32 + lane] = sum[i];
                else if (token < live && row < s.N) out[(size_t)(first_token + token) * s.N + row] = from_float<Out>(sum[i]);
            }
        }
        if (s.cluster > 1) {
            asm volatile("barrier.cluster.arrive.release;" ::: "memory");
            asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
            const uint32_t base = smem_address(whole);
            for (int i = rank * THREADS + threadIdx.x; i < count * live * 16; i += s.cluster * THREADS) {
                const int index = i / (live * 16), within = i - index * (live * 16);
                float sum = 0.0f;
                for (int c = 0; c < s.cluster; ++c) {
                    uint32_t there;
                    float v;
                    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(base + (index * GROUP_SUMS + within) * 4), "r"(c));
                    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
                    sum += v;
                }
                const long long row = (long long)(first + index) * 16 + (within & 15);
                if (row < s.N) out[(size_t)(first_token + (within >> 4)) * s.N + row] = from_float<Out>(sum);
            }
            asm volatile("barrier.cluster.arrive.release;" ::: "memory");        // a CTA's sums stay until its cluster has read them
            asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
        }
    }
}

// Bytes of shared memory; 0 where x does not fit.
size_t shared_bytes(int x_stages, int live, int cluster) {
    const size_t bytes = (size_t)WARPS * (RING * STAGE_BYTES + FACTOR_BYTES) + (size_t)WARPS * 2 * GROUP_SUMS * 4 +
                         (cluster > 1 ? (size_t)ROUND_GROUPS * GROUP_SUMS * 4 : 0) + (size_t)live * ((size_t)x_stages * STAGE_K * 2 + X_PAD);
    return bytes > SMEM_MOST || x_stages > MAX_STAGES ? 0 : bytes;
}

template <bool QUANTISE, typename Out>
int launch(const void* x, const void* codes, const void* scales, void* out, Shapes s, int ctas, void* stream) {
    const int stages = (s.K + STAGE_K - 1) / STAGE_K;
    s.x_stages = (stages + s.cluster - 1) / s.cluster;
    const size_t bytes = shared_bytes(s.x_stages, s.M < TOKENS ? s.M : TOKENS, s.cluster);
    if (!bytes) return MRS_BAD_ARGUMENT;
    static PerDevice configured;
    if (!configured.get()) {
        cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<QUANTISE, Out>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM_MOST);
        if (e != cudaSuccess) return (int)e;
        configured.set(1);
    }
    const int groups = s.N / 16 + (s.N % 16 != 0), most_shares = (ctas / s.cluster) > 1 ? ctas / s.cluster : 1;
    const int shares = groups < most_shares ? groups : most_shares;
    s.groups_each = groups / shares, s.groups_over = groups % shares;
    s.stages_each = stages / s.cluster, s.stages_over = stages % s.cluster;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(shares * s.cluster), (unsigned)((s.M + TOKENS - 1) / TOKENS));
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = bytes;
    config.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = s.cluster, attributes[1].val.clusterDim.y = 1, attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = s.cluster > 1 ? 2 : 1;
    cudaError_t e = cudaLaunchKernelEx(&config, few_rows_kernel<QUANTISE, Out>, (const bf16*)x, (const uint8_t*)codes, (const uint8_t*)scales,
                                       (Out*)out, s);
    if (e != cudaSuccess) return (int)e;
    MRS_RETURN_LAUNCH_STATUS();
}

}  // namespace

// CTAs of a cluster (1, 2, 4 or 8) whose shared memory holds their ranges of up to 8 rows of K elements; 0 where none does.
MRS_EXPORT int mrs_mxfp4_few_rows_cluster(int M, int K) {
    const int stages = (K + STAGE_K - 1) / STAGE_K;
    for (int c = 1; c <= 8; c *= 2)
        if (shared_bytes((stages + c - 1) / c, M < TOKENS ? M : TOKENS, c)) return c;
    return 0;
}

// out [M, N] bfloat16 or float32 (`out_f32`); x [M, K] bfloat16; w as in mxfp4.cuh; `cluster` 1, 2, 4 or 8 ranges of K; `ctas`: the GPU's
// SMs.  `fits`: w's blocks other than zeros have scales of 2^(w_exponent - 23) or more.  `early`: nothing that still runs when this kernel
// starts writes w.
MRS_EXPORT int mrs_mxfp4_few_rows(const void* x, const void* codes, const void* scales, void* out, int out_f32, int M, int N, int K, int quantise,
                                  int cluster, int ctas, int fits, int w_exponent, int early, void* stream) {
    if (M == 0 || N == 0) return 0;
    if (M < 0 || N < 0 || K <= 0 || K % MX_BLOCK || K > (1 << 30) || M > 65535 * 8 || ctas < 1 || !x || !codes || !scales || !out) return MRS_BAD_ARGUMENT;
    if ((((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15) || ((uintptr_t)out & (out_f32 ? 3 : 1))) return MRS_BAD_ARGUMENT;
    if (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8) return MRS_BAD_ARGUMENT;
    const int least_scale = fits && w_exponent > -104 ? w_exponent - 23 : -127, least_factor = -149 - least_scale;
    Shapes s = {M, N, K, cluster, 0, ldexpf(1.0f, least_factor > -126 ? least_factor : -126), early, 0, 0, 0, 0};
    if (quantise) return out_f32 ? launch<true, float>(x, codes, scales, out, s, ctas, stream) : launch<true, bf16>(x, codes, scales, out, s, ctas, stream);
    return out_f32 ? launch<false, float>(x, codes, scales, out, s, ctas, stream) : launch<false, bf16>(x, codes, scales, out, s, ctas, stream);
}

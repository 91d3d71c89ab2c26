// Products of few rows with a matrix in microscaled 4-bit floating point: out[m, n] = sum_k x[m, k] w[n, k], x bfloat16 (or brought
// to 4 bits here, block by block, by the rule of mxfp4.cuh), w in 4 bits, sums in float32.
//
// The bytes of w bound it: half a byte and a 32nd a weight, read once.  A warp owns 16 rows of w and a range of K, and copies
// its own 128-byte pieces of them (16 rows x 256 elements) into a ring of its own in shared memory with cp.async, so that no
// barrier stands in its loop.  A word of eight codes becomes four pairs of halfs (exact) that are A fragments of mma.m16n8k16 as
// they stand: the order of K within a block is free as long as x has the same, so lane (g, t) takes the codes 8 t to 8 t + 7
// of a block as its K indices of two MMAs and the same eight elements of x.  A block's two MMAs start from zero, and their sums are
// multiplied by the block's power of two as they join the row's float32 sums: products of halfs are exact, every sum is float32.
//
// x as halfs.  A CTA brings its part of x into the halfs' range by one power of two, which goes into the scales again.
// Where that loses a bit of any element (more than 2^32 between the sizes of two), or x has an element that is not finite, or the
// power is beyond [2^-20, 2^15], the CTA multiplies in bfloat16 instead, whose codes take more steps to make: the same sums.
//
// Ranges of K: the `parts` warps that share a CTA's rows, times the CTAs of a cluster; their sums meet in shared memory, added
// in the ranges' order, so that a result does not depend on timing.
#include "mxfp4.cuh"

namespace {

constexpr int WARPS = 8, THREADS = WARPS * 32;
constexpr int STAGE_K = 256;                       // elements of K a stage: 128 bytes a row
constexpr int CODE_BYTES = 16 * 128, SCALE_BYTES = 16 * 8, STAGE_BYTES = CODE_BYTES + SCALE_BYTES;
constexpr int RING = 4;
constexpr int SEGMENT = 2048;                      // elements of K of x in shared memory at a time
constexpr int X_PAD = 64;                          // bytes behind a row of x: two rows then fill all banks

__device__ __forceinline__ uint32_t smem_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void copy_16(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_4(uint32_t dst, const void* src, bool there) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

template <bool HALFS>
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (HALFS)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// A half pair of codes as a pair of bfloat16 (exact: both have the values 0.5 to 6).
__device__ __forceinline__ uint32_t as_bf16_pair(uint32_t halfs) {
    const float2 v = __half22float2(*reinterpret_cast<__half2*>(&halfs));
    __nv_bfloat162 pair = __floats2bfloat162_rn(v.x, v.y);
    return *reinterpret_cast<uint32_t*>(&pair);
}

struct Shapes {
    int M, N, K;
    int parts;              // warps that share a CTA's rows, a range of K each: 1, 2, 4 or 8
    int cluster;            // CTAs that share them
    int segment;            // elements of K of x that shared memory holds
    int early;              // w was there before the kernel before this one: it may be fetched while that runs
};

// Ranges of K in stages: range r of `ranges`.
__device__ __forceinline__ int range_start(int stages, int ranges, int r) { return (int)((long long)stages * r / ranges); }

// Stages [from, to) of one warp's rows joined to its sums; `x_smem` holds elements of K from stage `x_from` on.
template <int NT, bool HALFS>
__device__ __forceinline__ void stage_products(const unsigned char* stage, const unsigned char* x_stage, int x_pitch, float factor,
                                               float (&sums)[NT][4]) {
    const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const unsigned char* codes = stage + g * 128 + t * 4;
    const uint2 scale_low = *reinterpret_cast<const uint2*>(stage + CODE_BYTES + g * 8);
    const uint2 scale_high = *reinterpret_cast<const uint2*>(stage + CODE_BYTES + (g + 8) * 8);
    const unsigned char* x_row = x_stage + g * x_pitch + t * 16;
#pragma unroll
    for (int b = 0; b < STAGE_K / MX_BLOCK; ++b) {
        const int place = (b ^ g) * 16;
        uint32_t low[4], high[4];
        mx_decode_8(*reinterpret_cast<const uint32_t*>(codes + place), low);
        mx_decode_8(*reinterpret_cast<const uint32_t*>(codes + place + 8 * 128), high);
        if constexpr (!HALFS) {
#pragma unroll
            for (int i = 0; i < 4; ++i) low[i] = as_bf16_pair(low[i]), high[i] = as_bf16_pair(high[i]);
        }
        const uint32_t word_low = b < 4 ? scale_low.x : scale_low.y, word_high = b < 4 ? scale_high.x : scale_high.y;
        const int shift = 23 - 8 * (b & 3);
        const uint32_t bits_low = (shift >= 0 ? word_low << (shift & 31) : word_low >> (-shift & 31)) & 0x7F800000u;
        const uint32_t bits_high = (shift >= 0 ? word_high << (shift & 31) : word_high >> (-shift & 31)) & 0x7F800000u;
        // byte 0 is 2^-127; byte 255, not a number, stands beside codes of 0: infinity times the sum of 0 is NaN
        const float s_low = __uint_as_float(max(bits_low, 0x00400000u)) * factor, s_high = __uint_as_float(max(bits_high, 0x00400000u)) * factor;
        const uint32_t a0[4] = {low[0], high[0], low[1], high[1]}, a1[4] = {low[2], high[2], low[3], high[3]};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const uint4 xs = *reinterpret_cast<const uint4*>(x_row + (size_t)n * 8 * x_pitch + b * 64);
            float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            mma<HALFS>(d, a0, xs.x, xs.y);
            mma<HALFS>(d, a1, xs.z, xs.w);
            sums[n][0] = fmaf(d[0], s_low, sums[n][0]);
            sums[n][1] = fmaf(d[1], s_low, sums[n][1]);
            sums[n][2] = fmaf(d[2], s_high, sums[n][2]);
            sums[n][3] = fmaf(d[3], s_high, sums[n][3]);
        }
    }
}

// Eight elements of x as pairs of bfloat16; with QUANTISE what their 4-bit codes stand for (four lanes a block).
template <bool QUANTISE>
__device__ __forceinline__ uint4 load_x(const bf16* x, bool there) {
    uint4 raw = make_uint4(0, 0, 0, 0);
    if (there) raw = *reinterpret_cast<const uint4*>(x);
    if constexpr (QUANTISE) {
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
        raw = make_uint4(w[0], w[1], w[2], w[3]);
    }
    return raw;
}

// x[tokens][from, from + count) into shared memory, `rows` rows (those behind M and what lies behind K as zeros).  Returns whether
// they lie there as halfs, times 2^(15 - e) (`factor` = 2^(e - 15)), or, where that would lose a bit, as they are (`factor` = 1).
template <bool QUANTISE>
__device__ bool bring_x(const bf16* __restrict__ x, unsigned char* x_smem, int x_pitch, int rows, int first_token, const Shapes& s, int from,
                        int count, uint32_t* scratch, float& factor) {
    const int chunks = count >> 3, total = rows * chunks;
    uint32_t largest = 0;
    for (int base = 0; base < total; base += THREADS) {                       // whole warps: a block's four lanes stay together
        const int i = base + threadIdx.x, row = i / chunks, column = (i - row * chunks) * 8;
        const bool there = i < total && first_token + row < s.M && from + column < s.K;
        const uint4 raw = load_x<QUANTISE>(x + (size_t)(first_token + row) * s.K + from + column, there);
        const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) largest = max(largest, max(w[j] & 0x7FFFu, (w[j] >> 16) & 0x7FFFu));
        if (i < total) *reinterpret_cast<uint4*>(x_smem + (size_t)row * x_pitch + column * 2) = raw;
    }
    largest = __reduce_max_sync(0xffffffffu, largest);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = largest;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) largest = max(largest, scratch[w]);
    const int field = (int)(largest >> 7), e = largest == 0 ? 0 : field - 127;
    bool exact = field != 255 && e >= -20 && e <= 15;
    if (exact) {
        const float up = __uint_as_float((uint32_t)(127 + 15 - e) << 23);
        for (int i = threadIdx.x; i < total; i += THREADS) {
            const int row = i / chunks, column = (i - row * chunks) * 8;
            uint4* place = reinterpret_cast<uint4*>(x_smem + (size_t)row * x_pitch + column * 2);
            const uint4 raw = *place;
            uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float a = __uint_as_float(w[j] << 16) * up, b = __uint_as_float(w[j] & 0xFFFF0000u) * up;
                __half2 pair = __floats2half2_rn(a, b);
                const float2 back = __half22float2(pair);
                exact = exact && back.x == a && back.y == b;
                w[j] = *reinterpret_cast<uint32_t*>(&pair);
            }
            *place = make_uint4(w[0], w[1], w[2], w[3]);
        }
    }
    const bool asked = field != 255 && e >= -20 && e <= 15;                   // the same for the whole CTA
    exact = !__syncthreads_or(!exact);
    factor = exact ? __uint_as_float((uint32_t)(127 + e - 15) << 23) : 1.0f;
    if (!exact && asked) {                                                     // overwritten above: read again
        for (int base = 0; base < total; base += THREADS) {
            const int i = base + threadIdx.x, row = i / chunks, column = (i - row * chunks) * 8;
            const bool there = i < total && first_token + row < s.M && from + column < s.K;
            const uint4 raw = load_x<QUANTISE>(x + (size_t)(first_token + row) * s.K + from + column, there);
            if (i < total) *reinterpret_cast<uint4*>(x_smem + (size_t)row * x_pitch + column * 2) = raw;
        }
        __syncthreads();
    }
    return exact;
}

template <int NT, bool QUANTISE, typename Out>
__global__ void __launch_bounds__(THREADS, 2) few_rows_kernel(const bf16* __restrict__ x, const uint8_t* __restrict__ codes,
                                                              const uint8_t* __restrict__ scales, Out* __restrict__ out, const Shapes s) {
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ uint32_t scratch[WARPS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int groups = WARPS / s.parts, rows_of_cta = groups * 16;
    const int rank = blockIdx.x % s.cluster, tile = blockIdx.x / s.cluster;
    const int group = warp / s.parts, part = warp - group * s.parts;
    const long long row0 = (long long)tile * rows_of_cta + group * 16;
    const int first_token = blockIdx.y * (NT * 8);
    const int stages = (s.K + STAGE_K - 1) / STAGE_K;
    const int cta_from = range_start(stages, s.cluster, rank), cta_to = range_start(stages, s.cluster, rank + 1);

    unsigned char* ring = smem + warp * (RING * STAGE_BYTES);
    unsigned char* x_smem = smem + WARPS * RING * STAGE_BYTES;
    float* partial = reinterpret_cast<float*>(x_smem);                       // x is done with when the sums meet
    const int x_pitch = s.segment * 2 + X_PAD;

    const long long code_pitch = s.K >> 1, tiles_of_a_row = mx_tiles_of_a_row(s.K);
    // A stage of this warp's rows: four 16-byte copies and one of four scales a lane.
    auto fetch = [&](int stage, int slot) {
        const uint32_t base = smem_address(ring + slot * STAGE_BYTES);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int q = j * 32 + lane, r = q >> 3, c = q & 7;
            const bool there = row0 + r < s.N && stage * 128 + c * 16 < code_pitch;
            copy_16(base + r * 128 + ((c ^ (r & 7)) << 4), there ? codes + (row0 + r) * code_pitch + stage * 128 + c * 16 : codes, there);
        }
        const long long r = row0 + (lane >> 1);
        const bool there = r < s.N;
        copy_4(base + CODE_BYTES + lane * 4, there ? scales + mx_scale_offset(r, stage * 2 + (lane & 1), tiles_of_a_row) : scales, there);
    };

    float sums[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) sums[n][0] = sums[n][1] = sums[n][2] = sums[n][3] = 0.0f;

    if (!s.early) pdl_wait();
    // this CTA's stages in segments of x; within a segment warp `part` takes stages part, part + parts, ...
    const int segment_stages = s.segment / STAGE_K;
    int next = cta_from + part, fetched = 0, used = 0;          // the next stage to fetch: this warp's walk through the CTA's range
    auto fetch_next = [&]() {
        if (next < cta_to) {
            fetch(next, fetched % RING);
            next += s.parts;
        }
        ++fetched;
        copy_commit();
    };
#pragma unroll
    for (int i = 0; i < RING - 1; ++i) fetch_next();
    pdl_launch_dependents();
    if (s.early) pdl_wait();
    // the segments are multiples of `parts` stages long, so a warp's walk through the range meets every segment in step
    for (int from = cta_from; from < cta_to; from += segment_stages) {
        const int to = min(from + segment_stages, cta_to);
        float factor;
        if (from > cta_from) __syncthreads();
        const bool halfs = bring_x<QUANTISE>(x, x_smem, x_pitch, NT * 8, first_token, s, from * STAGE_K, (to - from) * STAGE_K, scratch, factor);
        for (int stage = from + part; stage < to; stage += s.parts) {
            copy_wait<RING - 2>();
            __syncwarp();
            fetch_next();
            const unsigned char* slot = ring + (used % RING) * STAGE_BYTES;
            const unsigned char* x_stage = x_smem + (stage - from) * (STAGE_K * 2);
            if (halfs) stage_products<NT, true>(slot, x_stage, x_pitch, factor, sums);
            else stage_products<NT, false>(slot, x_stage, x_pitch, factor, sums);
            ++used;
            __syncwarp();
        }
    }
    copy_wait<0>();
    __syncthreads();

    // the ranges' sums [part][token][row of the CTA] meet
    const int tokens = NT * 8, plane = tokens * rows_of_cta;
    {
        float* mine = partial + part * plane + group * 16;
        const int g = lane >> 2, t = lane & 3;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            mine[(n * 8 + 2 * t) * rows_of_cta + g] = sums[n][0];
            mine[(n * 8 + 2 * t + 1) * rows_of_cta + g] = sums[n][1];
            mine[(n * 8 + 2 * t) * rows_of_cta + g + 8] = sums[n][2];
            mine[(n * 8 + 2 * t + 1) * rows_of_cta + g + 8] = sums[n][3];
        }
    }
    if (s.cluster > 1) {
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    } else {
        __syncthreads();
    }
    const int live = min(tokens, s.M - first_token) * rows_of_cta;
    const uint32_t base = smem_address(partial);
    for (int i = rank * THREADS + threadIdx.x; i < live; i += s.cluster * THREADS) {
        const int token = i / rows_of_cta, row = i - token * rows_of_cta;
        const long long n = (long long)tile * rows_of_cta + row;
        float sum = 0.0f;
        for (int c = 0; c < s.cluster; ++c) {
            uint32_t there;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(base + i * 4), "r"(c));
            for (int p = 0; p < s.parts; ++p) {
                float v;
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there + p * plane * 4) : "memory");
                sum += v;
            }
        }
        if (n < s.N) out[(size_t)(first_token + token) * s.N + n] = from_float<Out>(sum);
    }
    if (s.cluster > 1) {                                          // a CTA's sums stay until its cluster has read them
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");
        asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
    }
}

template <int NT, bool QUANTISE, typename Out>
int launch(const void* x, const void* codes, const void* scales, void* out, Shapes s, void* stream) {
    const int groups = WARPS / s.parts;
    const int stages = (s.K + STAGE_K - 1) / STAGE_K, of_cta = (stages + s.cluster - 1) / s.cluster;
    const int most = SEGMENT / STAGE_K;                           // a multiple of every count of parts
    s.segment = (of_cta < most ? of_cta : most) * STAGE_K;
    const size_t x_bytes = (size_t)NT * 8 * (s.segment * 2 + X_PAD), sum_bytes = (size_t)WARPS * 16 * NT * 8 * 4;
    const size_t bytes = (size_t)WARPS * RING * STAGE_BYTES + (x_bytes > sum_bytes ? x_bytes : sum_bytes);
    static PerDevice configured;
    if (!configured.get()) {
        const size_t all = (size_t)WARPS * RING * STAGE_BYTES + (size_t)NT * 8 * (SEGMENT * 2 + X_PAD);
        cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<NT, QUANTISE, Out>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)all);
        if (e != cudaSuccess) return (int)e;
        configured.set(1);
    }
    const long long rows = groups * 16, tiles = ((long long)s.N + rows - 1) / rows;
    if (tiles * s.cluster > 0x7FFFFFFFll) return MRS_BAD_ARGUMENT;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(tiles * s.cluster), (unsigned)((s.M + NT * 8 - 1) / (NT * 8)));
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = bytes;
    config.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = s.cluster, attributes[1].val.clusterDim.y = 1, attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&config, few_rows_kernel<NT, QUANTISE, Out>, (const bf16*)x, (const uint8_t*)codes, (const uint8_t*)scales,
                                       (Out*)out, s);
    if (e != cudaSuccess) return (int)e;
    MRS_RETURN_LAUNCH_STATUS();
}

template <int NT, typename Out>
int launch_x(const void* x, const void* codes, const void* scales, void* out, const Shapes& s, int quantise, void* stream) {
    return quantise ? launch<NT, true, Out>(x, codes, scales, out, s, stream) : launch<NT, false, Out>(x, codes, scales, out, s, stream);
}

}  // namespace

// out [M, N] bfloat16 or float32 (`out_f32`); x [M, K] bfloat16; w as in mxfp4.cuh; `parts` 1, 2, 4 or 8, `cluster` 1, 2, 4 or 8 ranges of K.
// `early`: nothing that still runs when this kernel starts writes w.
MRS_EXPORT int mrs_mxfp4_few_rows(const void* x, const void* codes, const void* scales, void* out, int out_f32, int M, int N, int K, int quantise,
                                  int parts, int cluster, int early, void* stream) {
    if (M == 0 || N == 0) return 0;
    if (M < 0 || N < 0 || K <= 0 || K % MX_BLOCK || K > (1 << 30) || M > 65535 * 8 || !x || !codes || !scales || !out) return MRS_BAD_ARGUMENT;
    if ((((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15) || ((uintptr_t)out & (out_f32 ? 3 : 1))) return MRS_BAD_ARGUMENT;
    if ((parts != 1 && parts != 2 && parts != 4 && parts != 8) || (cluster != 1 && cluster != 2 && cluster != 4 && cluster != 8)) return MRS_BAD_ARGUMENT;
    Shapes s = {M, N, K, parts, cluster, 0, early};
    if (M <= 8) return out_f32 ? launch_x<1, float>(x, codes, scales, out, s, quantise, stream) : launch_x<1, bf16>(x, codes, scales, out, s, quantise, stream);
    return out_f32 ? launch_x<2, float>(x, codes, scales, out, s, quantise, stream) : launch_x<2, bf16>(x, codes, scales, out, s, quantise, stream);
}

MRS_EXPORT const char* mrs_mxfp4_few_error_string(int code) {
    if (code == MRS_BAD_ARGUMENT) return "arguments outside what the kernel supports (K no multiple of 32, unaligned base, ranges)";
    return cudaGetErrorString((cudaError_t)code);
}

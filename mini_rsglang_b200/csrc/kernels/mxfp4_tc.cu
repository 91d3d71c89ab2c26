// Products of many rows with a matrix in microscaled 4-bit floating point on the tcgen05 tensor cores: out[m, n] = sum_k x[m, k] w[n, k],
// float32 sums.  A CTA takes 128 rows of w (the M of the MMA, so that a few tokens fill a narrow N) and up to 256 tokens; the CTAs
// of a cluster share a tile with a range of K each, and their sums meet in the ranges' order.
//
//   weights_kernel   x in bfloat16.  Bulk tensor copies bring 128 x 256 codes (128-byte swizzle) and their scales into a ring, x in
//                    pieces of 64 elements into another.  Eight warps make bfloat16 of the codes, a thread a row: code to half, half to
//                    float32, times the block's power of two, two floats to a pair of bfloat16 (every step exact), into tensor memory as
//                    the A operand; no shared memory is written for them.  One thread issues kind::f16 MMAs with A in tensor memory.
//   both_kernel      x in 4 bits as well: codes of both sides go from shared memory into kind::mxf4 MMAs as they are, scales are copied into
//                    tensor memory (tcgen05.cp) stage by stage.
//
// Every wait is bounded (tma.cuh).
#include "mxfp4.cuh"
#include "tcgen05.cuh"

namespace {

constexpr int BM = 128;                            // rows of w of a tile
constexpr int STAGE_K = 256;                       // elements of K of a stage of codes: 128 bytes a row
constexpr int CODE_BYTES = BM * 128, SCALE_BYTES = 2 * MX_TILE_BYTES;
constexpr int WORKERS = 8;                         // warps that make bfloat16 and store results
constexpr int THREADS = 64 + WORKERS * 32;
constexpr int TMEM_COLUMNS = 512;
constexpr int MOST_BYTES = 226 * 1024;             // of shared memory a CTA may have
constexpr size_t ALONE_BYTES = 208 * 1024;         // with so much no other CTA that uses tensor memory fits the SM

__device__ __forceinline__ int range_start(int count, int ranges, int r) { return (int)((long long)count * r / ranges); }

// Untiled copy of a multiple of 16 bytes, both sides on 16-byte boundaries.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

struct Shapes {
    int M, N, K;
    int token_tiles;
    int cluster;
    int early;              // w was there before the kernel before this one: it may be fetched while that runs
    long long w_tiles_of_a_row, x_row_tiles;
};

// The accumulator's results (lane: row of w, column: token) to memory; `sums` is shared memory for TOKENS x 128 floats, used by clusters only.
// Called by every thread of the CTA; the workers read the accumulator.
template <int TOKENS, typename Out>
__device__ __forceinline__ void store_results(uint32_t tmem, float* sums, Out* __restrict__ out, const Shapes& s, long long n0, int token0, int rank,
                                              bool empty) {
    constexpr int STEP = TOKENS < 32 ? 16 : 32;
    constexpr int GROUPS = TOKENS / STEP < 2 ? 1 : 2;                          // of four warps, that share the columns
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int live = min(TOKENS, s.M - token0);
    if (warp >= 2 && (warp - 2) >> 2 < GROUPS) {
        const int quarter = warp & 3, group = (warp - 2) >> 2, row = quarter * 32 + lane;
        const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16);
        const long long n = n0 + row;
#pragma unroll 1
        for (int c = group * STEP; c < TOKENS; c += GROUPS * STEP) {
            if (c >= live) break;
            float v[STEP];
            if (!empty) {
                if constexpr (STEP == 16) tmem_load_16_async(acc + c, v);
                else tmem_load_32_async(acc + c, v);
                tmem_load_wait();
            } else {
#pragma unroll
                for (int e = 0; e < STEP; ++e) v[e] = 0.0f;
            }
            if (s.cluster == 1) {
                if (n < s.N) {
#pragma unroll
                    for (int e = 0; e < STEP; ++e)
                        if (c + e < live) out[(size_t)(token0 + c + e) * s.N + n] = from_float<Out>(v[e]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < STEP; ++e) sums[(c + e) * BM + row] = v[e];
            }
        }
    }
    if (s.cluster > 1) {
        cluster_sync();
        const uint32_t base = smem_u32(sums);
        for (int i = rank * THREADS + threadIdx.x; i < live * BM; i += s.cluster * THREADS) {
            float sum = 0.0f;
            for (int c = 0; c < s.cluster; ++c) {
                uint32_t there;
                float v;
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(base + i * 4), "r"(c));
                asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(there) : "memory");
                sum += v;
            }
            const long long n = n0 + (i & (BM - 1));
            if (n < s.N) out[(size_t)(token0 + i / BM) * s.N + n] = from_float<Out>(sum);
        }
        cluster_sync();                            // a CTA's sums stay until its cluster has read them
    }
}

// ------------------------------------------------------------------------------------------
// x in bfloat16
// ------------------------------------------------------------------------------------------
constexpr int STEP_K = 64;                         // elements of K of a piece of x and of a buffer of A
constexpr int A_BUFFERS = 8, A_COLUMNS = STEP_K / 2, A_FIRST = 256;
constexpr int W_STAGES = 4, X_STAGES = 4;
template <int TOKENS> constexpr int x_bytes() { return TOKENS * STEP_K * 2; }
template <int TOKENS> constexpr size_t weights_smem() {
    return 1024 + (size_t)W_STAGES * (CODE_BYTES + SCALE_BYTES) + (size_t)X_STAGES * x_bytes<TOKENS>() + 512;
}

// 32 codes of a row and their scale as 16 pairs of bfloat16.
__device__ __forceinline__ void decode_block(uint4 codes, float scale, uint32_t* words) {
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[4];
        mx_decode_8(w[i], h);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const float2 v = __half22float2(*reinterpret_cast<__half2*>(&h[p]));
            __nv_bfloat162 pair = __floats2bfloat162_rn(v.x * scale, v.y * scale);
            words[i * 4 + p] = *reinterpret_cast<uint32_t*>(&pair);
        }
    }
}
__device__ __forceinline__ void tmem_store_32_words(uint32_t address, const uint32_t (&v)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
                 "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(address), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
                   "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
                   "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]),
                   "r"(v[30]), "r"(v[31]) : "memory");
}

template <int TOKENS, typename Out>
__global__ void __launch_bounds__(THREADS, 1) weights_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                             const uint8_t* __restrict__ scales, Out* __restrict__ out, const Shapes s) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* w_ring = smem;
    unsigned char* x_ring = w_ring + W_STAGES * CODE_BYTES;
    unsigned char* s_ring = x_ring + X_STAGES * x_bytes<TOKENS>();
    uint64_t* w_full = reinterpret_cast<uint64_t*>(s_ring + W_STAGES * SCALE_BYTES);
    uint64_t* w_empty = w_full + W_STAGES;
    uint64_t* x_full = w_empty + W_STAGES;
    uint64_t* x_empty = x_full + X_STAGES;
    uint64_t* a_full = x_empty + X_STAGES;
    uint64_t* a_empty = a_full + A_BUFFERS;
    uint64_t* acc_full = a_empty + A_BUFFERS;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % s.cluster, tile = blockIdx.x / s.cluster;
    const int token0 = tile % s.token_tiles * TOKENS, n_tile = tile / s.token_tiles;
    const int stages = (s.K + STAGE_K - 1) / STAGE_K, steps = (s.K + STEP_K - 1) / STEP_K;
    const int from = range_start(stages, s.cluster, rank), to = range_start(stages, s.cluster, rank + 1);
    const int step_from = from * (STAGE_K / STEP_K), step_to = min(to * (STAGE_K / STEP_K), steps);

    if (threadIdx.x == 0) {
        for (int i = 0; i < W_STAGES; ++i) {
            mbar_init(&w_full[i], 1);
            mbar_init(&w_empty[i], WORKERS);
        }
        for (int i = 0; i < X_STAGES; ++i) {
            mbar_init(&x_full[i], 1);
            mbar_init(&x_empty[i], 1);
        }
        for (int i = 0; i < A_BUFFERS; ++i) {
            mbar_init(&a_full[i], 4);
            mbar_init(&a_empty[i], 1);
        }
        mbar_init(acc_full, 1);
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLUMNS);
        tmem_relinquish_alloc_permit();
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        const bool leader = elect_one();
        if (!s.early) pdl_wait();
        bool waited = !s.early, alive = true;
        int w_next = from, x_next = step_from;
        // codes run ahead of x by as much as their ring holds
        while (alive && (w_next < to || x_next < step_to)) {
            if (w_next < to && (w_next - from < W_STAGES || x_next >= (w_next - W_STAGES + 1) * (STAGE_K / STEP_K) || x_next >= step_to)) {
                const int i = (w_next - from) % W_STAGES;
                if (!(alive = mbar_wait(&w_empty[i], (((w_next - from) / W_STAGES) & 1) ^ 1))) break;
                if (leader) {
                    mbar_arrive_expect_tx(&w_full[i], CODE_BYTES + SCALE_BYTES);
                    tma_load_2d(w_ring + i * CODE_BYTES, &w_map, &w_full[i], w_next * 128, n_tile * BM);
                    bulk_load(s_ring + i * SCALE_BYTES, scales + ((size_t)n_tile * s.w_tiles_of_a_row + 2 * w_next) * MX_TILE_BYTES, SCALE_BYTES, &w_full[i]);
                }
                __syncwarp();
                ++w_next;
                continue;
            }
            if (!waited) {
                pdl_wait();
                waited = true;
            }
            const int i = (x_next - step_from) % X_STAGES;
            if (!(alive = mbar_wait(&x_empty[i], (((x_next - step_from) / X_STAGES) & 1) ^ 1))) break;
            if (leader) {
                mbar_arrive_expect_tx(&x_full[i], x_bytes<TOKENS>());
                tma_load_2d(x_ring + i * x_bytes<TOKENS>(), &x_map, &x_full[i], x_next * STEP_K, token0);
            }
            __syncwarp();
            ++x_next;
        }
        if (!waited) pdl_wait();
    } else if (warp == 1) {
        pdl_wait();
        const bool leader = elect_one();
        constexpr uint32_t idesc = umma_idesc_bf16_f32(BM, TOKENS);
        bool alive = true;
        for (int step = step_from; step < step_to && alive; ++step) {
            const int index = step - step_from, b = index % A_BUFFERS, i = index % X_STAGES;
            if (!(alive = mbar_wait(&x_full[i], (index / X_STAGES) & 1))) break;
            if (!(alive = mbar_wait(&a_full[b], (index / A_BUFFERS) & 1))) break;
            tcgen05_fence_after_sync();
            const uint64_t b_desc = umma_smem_desc_sw128(smem_u32(x_ring + i * x_bytes<TOKENS>()));
            const uint32_t a_tmem = tmem + A_FIRST + b * A_COLUMNS;
            if (leader) {
#pragma unroll
                for (int k = 0; k < STEP_K / 16; ++k) umma_bf16_a_tmem(tmem, a_tmem + 8 * k, b_desc + 2 * k, idesc, index > 0 || k > 0);
                umma_commit(&x_empty[i]);
                umma_commit(&a_empty[b]);
            }
            __syncwarp();
        }
        if (leader) umma_commit(acc_full);
        __syncwarp();
    } else {
        pdl_wait();
        const int quarter = warp & 3, group = (warp - 2) >> 2, row = quarter * 32 + lane;
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
        bool alive = true;
        for (int stage = from; stage < to && alive; ++stage) {
            const int i = (stage - from) % W_STAGES;
            if (!(alive = mbar_wait(&w_full[i], ((stage - from) / W_STAGES) & 1))) break;
            const unsigned char* codes = w_ring + i * CODE_BYTES + row * 128;
            const unsigned char* scale_tiles = s_ring + i * SCALE_BYTES + lane * 16 + quarter * 4;
#pragma unroll
            for (int half = 0; half < 2; ++half) {                            // steps `group` and 2 + group of the stage
                const int within = half * 2 + group, step = stage * (STAGE_K / STEP_K) + within, index = step - step_from;
                if (step >= step_to) break;
                const uint32_t four = *reinterpret_cast<const uint32_t*>(scale_tiles + half * MX_TILE_BYTES) >> (group * 16);
                const uint4 first = *reinterpret_cast<const uint4*>(codes + (((within * 2) ^ (row & 7)) << 4));
                const uint4 second = *reinterpret_cast<const uint4*>(codes + (((within * 2 + 1) ^ (row & 7)) << 4));
                uint32_t words[32];
                decode_block(first, mx_scale(four & 255u), words);
                decode_block(second, mx_scale((four >> 8) & 255u), words + 16);
                const int b = index % A_BUFFERS;
                if (!(alive = mbar_wait(&a_empty[b], ((index / A_BUFFERS) & 1) ^ 1))) break;
                __syncwarp();
                tcgen05_fence_after_sync();
                tmem_store_32_words(lanes + A_FIRST + b * A_COLUMNS, words);
                tmem_store_wait();
                tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[b]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&w_empty[i]);
        }
        mbar_wait(acc_full, 0);
        __syncwarp();
        tcgen05_fence_after_sync();
    }
    __syncwarp();
    store_results<TOKENS, Out>(tmem, reinterpret_cast<float*>(smem), out, s, (long long)n_tile * BM, token0, rank, step_from >= step_to);
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc(tmem, TMEM_COLUMNS);
    }
}

// ------------------------------------------------------------------------------------------
// x in 4 bits
// ------------------------------------------------------------------------------------------
// kind::mxf4: E2M1 on both sides, one E8M0 scale for 32 elements, K 64; `id`: which pair of a word's four scales (0 or 2).
__host__ __device__ constexpr uint32_t mxf4_idesc(int m, int n, uint32_t id) {
    return (id << 4)                      // scales of B
           | (1u << 7) | (1u << 10)       // A and B: E2M1
           | ((uint32_t)(n >> 3) << 17)   // N / 8
           | (1u << 23)                   // scales: E8M0
           | ((uint32_t)(m >> 7) << 27)   // M / 128
           | (id << 29);                  // scales of A
}
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, bool accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"((uint32_t)accumulate) : "memory");
}
// 32 rows of 16 bytes (a tile of scales) into four columns of lanes 0 to 31, and the same into the other three groups of lanes.
__device__ __forceinline__ void scales_to_tmem(uint32_t columns, uint32_t smem_address) {
    uint64_t desc = (uint64_t)((smem_address & 0x3FFFF) >> 4);
    desc |= (uint64_t)(128 >> 4) << 32;                    // between groups of 8 rows; no swizzle
    desc |= (uint64_t)1 << 46;
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(columns), "l"(desc) : "memory");
}

constexpr int B_STAGES = 4;
template <int TOKENS> constexpr int token_blocks() { return TOKENS > 128 ? 2 : 1; }            // tiles of scales of the tokens
template <int TOKENS> constexpr int both_stage_bytes() { return CODE_BYTES + TOKENS * 128 + SCALE_BYTES * (1 + token_blocks<TOKENS>()); }
template <int TOKENS> constexpr size_t both_smem() { return 1024 + (size_t)B_STAGES * both_stage_bytes<TOKENS>() + 256; }
constexpr int SCALES_FIRST = 256, SCALE_COLUMNS = 32;      // tensor memory columns of a stage's scales (up to 8 + 16 used)

template <int TOKENS, typename Out>
__global__ void __launch_bounds__(THREADS, 1) both_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                          const uint8_t* __restrict__ w_scales, const uint8_t* __restrict__ x_scales, Out* __restrict__ out,
                                                          const Shapes s) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    unsigned char* w_ring = smem;
    unsigned char* x_ring = w_ring + B_STAGES * CODE_BYTES;
    unsigned char* s_ring = x_ring + B_STAGES * TOKENS * 128;
    constexpr int STAGE_SCALES = SCALE_BYTES * (1 + token_blocks<TOKENS>());
    uint64_t* full = reinterpret_cast<uint64_t*>(s_ring + B_STAGES * STAGE_SCALES);
    uint64_t* empty = full + B_STAGES;
    uint64_t* acc_full = empty + B_STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 1);

    const int warp = threadIdx.x >> 5;
    const int rank = blockIdx.x % s.cluster, tile = blockIdx.x / s.cluster;
    const int token0 = tile % s.token_tiles * TOKENS, n_tile = tile / s.token_tiles;
    const int stages = (s.K + STAGE_K - 1) / STAGE_K;
    const int from = range_start(stages, s.cluster, rank), to = range_start(stages, s.cluster, rank + 1);

    if (threadIdx.x == 0) {
        for (int i = 0; i < B_STAGES; ++i) {
            mbar_init(&full[i], 1);
            mbar_init(&empty[i], 1);
        }
        mbar_init(acc_full, 1);
        mbar_fence_init();
    }
    if (warp == 1) {
        tmem_alloc(tmem_slot, TMEM_COLUMNS);
        tmem_relinquish_alloc_permit();
    }
    tcgen05_fence_before_sync();
    __syncthreads();
    tcgen05_fence_after_sync();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();

    if (warp == 0) {
        const bool leader = elect_one();
        // w first, as far as the ring goes, then x once the kernel before has ended
        const int ahead = s.early ? min(B_STAGES, to - from) : 0;
        auto load_w = [&](int stage, int i) {
            mbar_arrive_expect_tx(&full[i], CODE_BYTES + TOKENS * 128 + STAGE_SCALES);
            tma_load_2d(w_ring + i * CODE_BYTES, &w_map, &full[i], stage * 128, n_tile * BM);
            bulk_load(s_ring + i * STAGE_SCALES, w_scales + ((size_t)n_tile * s.w_tiles_of_a_row + 2 * stage) * MX_TILE_BYTES, SCALE_BYTES, &full[i]);
        };
        if (leader)
            for (int i = 0; i < ahead; ++i) load_w(from + i, i);
        __syncwarp();
        pdl_wait();
        bool alive = true;
        for (int stage = from; stage < to && alive; ++stage) {
            const int index = stage - from, i = index % B_STAGES;
            if (!(alive = mbar_wait(&empty[i], ((index / B_STAGES) & 1) ^ 1))) break;
            if (leader) {
                if (index >= ahead) load_w(stage, i);
                tma_load_2d(x_ring + i * TOKENS * 128, &x_map, &full[i], stage * 128, token0);
#pragma unroll
                for (int t = 0; t < token_blocks<TOKENS>(); ++t) {
                    const long long row_tile = min((long long)(token0 >> 7) + t, s.x_row_tiles - 1);      // a tile behind the last token: nobody stores its sums
                    bulk_load(s_ring + i * STAGE_SCALES + SCALE_BYTES * (1 + t), x_scales + ((size_t)row_tile * s.w_tiles_of_a_row + 2 * stage) * MX_TILE_BYTES,
                              SCALE_BYTES, &full[i]);
                }
            }
            __syncwarp();
        }
    } else if (warp == 1) {
        pdl_wait();
        const bool leader = elect_one();
        bool alive = true;
        for (int stage = from; stage < to && alive; ++stage) {
            const int index = stage - from, i = index % B_STAGES;
            if (!(alive = mbar_wait(&full[i], (index / B_STAGES) & 1))) break;
            tcgen05_fence_after_sync();
            const uint64_t a_desc = umma_smem_desc_sw128(smem_u32(w_ring + i * CODE_BYTES));
            const uint64_t b_desc = umma_smem_desc_sw128(smem_u32(x_ring + i * TOKENS * 128));
            const uint32_t scales = smem_u32(s_ring + i * STAGE_SCALES);
            const uint32_t columns = tmem + SCALES_FIRST + i * SCALE_COLUMNS;
            if (leader) {
#pragma unroll
                for (int q = 0; q < 2; ++q) {                                   // 128 elements of K
                    scales_to_tmem(columns + q * 4, scales + q * MX_TILE_BYTES);
#pragma unroll
                    for (int t = 0; t < token_blocks<TOKENS>(); ++t)
                        scales_to_tmem(columns + 8 + q * 8 + t * 4, scales + SCALE_BYTES * (1 + t) + q * MX_TILE_BYTES);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    umma_mxf4(tmem, a_desc + 2 * k, b_desc + 2 * k, mxf4_idesc(BM, TOKENS, (k & 1) * 2), columns + (k >> 1) * 4, columns + 8 + (k >> 1) * 8,
                              index > 0 || k > 0);
                umma_commit(&empty[i]);
            }
            __syncwarp();
        }
        if (leader) umma_commit(acc_full);
        __syncwarp();
    } else {
        pdl_wait();
        mbar_wait(acc_full, 0);
        __syncwarp();
        tcgen05_fence_after_sync();
    }
    __syncwarp();
    store_results<TOKENS, Out>(tmem, reinterpret_cast<float*>(smem), out, s, (long long)n_tile * BM, token0, rank, from >= to);
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc(tmem, TMEM_COLUMNS);
    }
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
int make_map(CUtensorMap* map, const void* base, CUtensorMapDataType type, long long row_bytes, long long columns, long long rows, int box_columns, int box_rows) {
    mrs_encode_tiled_fn encode = mrs_tensor_map_encoder();
    if (!encode) return MRS_TENSOR_MAP_FAILED;
    const cuuint64_t dims[2] = {(cuuint64_t)columns, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)row_bytes};
    const cuuint32_t box[2] = {(cuuint32_t)box_columns, (cuuint32_t)box_rows}, ones[2] = {1, 1};
    return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : MRS_TENSOR_MAP_FAILED;
}

template <typename... KernelArgs, typename... Args>
int launch_cluster(void (*kernel)(KernelArgs...), PerDevice& configured, long long ctas, int cluster, size_t smem, void* stream, Args... args) {
    if (!configured.get()) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, MOST_BYTES);
        if (e != cudaSuccess) return (int)e;
        configured.set(1);
    }
    if (ctas > 0x7FFFFFFFll) return MRS_BAD_ARGUMENT;
    // A CTA that waits for its cluster keeps its tensor memory meanwhile: clusters that wait for one another's would wait for good, so they
    // take whole SMs.
    if (cluster > 1 && smem < ALONE_BYTES) smem = ALONE_BYTES;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)ctas);
    config.blockDim = dim3(THREADS);
    config.dynamicSmemBytes = smem;
    config.stream = (cudaStream_t)stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster, attributes[1].val.clusterDim.y = 1, attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    cudaError_t e = cudaLaunchKernelEx(&config, kernel, static_cast<KernelArgs>(args)...);
    if (e != cudaSuccess) return (int)e;
    return (int)cudaGetLastError();
}

template <int TOKENS, typename Out>
int launch_weights(const void* x, const void* codes, const void* scales, void* out, Shapes s, void* stream) {
    CUtensorMap w_map, x_map;
    int code = make_map(&w_map, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K / 2, s.K / 2, s.N, 128, BM);
    if (!code) code = make_map(&x_map, x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (long long)s.K * 2, s.K, s.M, STEP_K, TOKENS);
    if (code) return code;
    static PerDevice configured;
    s.token_tiles = (s.M + TOKENS - 1) / TOKENS;
    const long long tiles = (long long)((s.N + BM - 1) / BM) * s.token_tiles;
    return launch_cluster(weights_kernel<TOKENS, Out>, configured, tiles * s.cluster, s.cluster, weights_smem<TOKENS>(), stream, w_map, x_map,
                          (const uint8_t*)scales, (Out*)out, s);
}
template <int TOKENS, typename Out>
int launch_both(const void* x_codes, const void* x_scales, const void* codes, const void* scales, void* out, Shapes s, void* stream) {
    CUtensorMap w_map, x_map;
    int code = make_map(&w_map, codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K / 2, s.K / 2, s.N, 128, BM);
    if (!code) code = make_map(&x_map, x_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K / 2, s.K / 2, s.M, 128, TOKENS);
    if (code) return code;
    static PerDevice configured;
    s.token_tiles = (s.M + TOKENS - 1) / TOKENS;
    s.x_row_tiles = (s.M + 127) / 128;
    const long long tiles = (long long)((s.N + BM - 1) / BM) * s.token_tiles;
    return launch_cluster(both_kernel<TOKENS, Out>, configured, tiles * s.cluster, s.cluster, both_smem<TOKENS>(), stream, w_map, x_map,
                          (const uint8_t*)scales, (const uint8_t*)x_scales, (Out*)out, s);
}

bool bad(const void* x, const void* codes, const void* scales, const void* out, int out_f32, int M, int N, int K, int tokens, int cluster) {
    return M < 0 || N < 0 || K <= 0 || K % MX_BLOCK || K > (1 << 30) || !x || !codes || !scales || !out ||
           (((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales) & 15) || ((uintptr_t)out & (out_f32 ? 3 : 1)) || cluster < 1 || cluster > 8 ||
           (tokens < 128 && M > tokens);
}

}  // namespace

// out [M, N] bfloat16 or float32 (`out_f32`); x [M, K] bfloat16; w as in mxfp4.cuh.  `tokens` (16, 32, 64, 128, 256): of a tile, below 128 only
// if they are all; `cluster` 1 to 8 ranges of K.  `early`: nothing that still runs when this kernel starts writes w.
MRS_EXPORT int mrs_mxfp4_weights_rows(const void* x, const void* codes, const void* scales, void* out, int out_f32, int M, int N, int K, int tokens,
                                      int cluster, int early, void* stream) {
    if (M == 0 || N == 0) return 0;
    if (bad(x, codes, scales, out, out_f32, M, N, K, tokens, cluster)) return MRS_BAD_ARGUMENT;
    const Shapes s = {M, N, K, 0, cluster, early, mx_tiles_of_a_row(K), 0};
#define MRS_TOKENS(T) if (tokens == T) return out_f32 ? launch_weights<T, float>(x, codes, scales, out, s, stream) : launch_weights<T, bf16>(x, codes, scales, out, s, stream)
    MRS_TOKENS(16); MRS_TOKENS(32); MRS_TOKENS(64); MRS_TOKENS(128); MRS_TOKENS(256);
#undef MRS_TOKENS
    return MRS_BAD_ARGUMENT;
}

// The same with x in 4 bits.
MRS_EXPORT int mrs_mxfp4_both_rows(const void* x_codes, const void* x_scales, const void* codes, const void* scales, void* out, int out_f32, int M, int N, int K,
                                   int tokens, int cluster, int early, void* stream) {
    if (M == 0 || N == 0) return 0;
    if (bad(x_codes, codes, scales, out, out_f32, M, N, K, tokens, cluster) || !x_scales || ((uintptr_t)x_scales & 15)) return MRS_BAD_ARGUMENT;
    const Shapes s = {M, N, K, 0, cluster, early, mx_tiles_of_a_row(K), 0};
#define MRS_TOKENS(T) if (tokens == T) return out_f32 ? launch_both<T, float>(x_codes, x_scales, codes, scales, out, s, stream) : launch_both<T, bf16>(x_codes, x_scales, codes, scales, out, s, stream)
    MRS_TOKENS(16); MRS_TOKENS(32); MRS_TOKENS(64); MRS_TOKENS(128); MRS_TOKENS(256);
#undef MRS_TOKENS
    return MRS_BAD_ARGUMENT;
}

MRS_EXPORT int mrs_mxfp4_take_error(unsigned int* word) { return mrs_take_error_word(word); }
// Mirrors the error word into a word of pinned host memory from now on.
MRS_EXPORT int mrs_mxfp4_mirror_errors(unsigned int* host_word) { return mrs_set_error_mirror(host_word); }

// Products of many rows with a matrix in microscaled 4-bit floating point on the tcgen05 tensor cores: out[m, n] = sum_k x[m, k] w[n, k],
// float32 sums.  A tile is 128 rows of w (the M of the MMA, so that a few tokens fill a narrow N) and up to 192 tokens.  A CTA an SM
// takes every 148th tile, or, where that leaves SMs without work (mxfp4_tiles in kernels.py), an equal run of all tiles' stages of 256 elements
// of K, tile by tile.  It has two accumulators in tensor memory: a tile's results are stored while the next tile's MMAs run.  A
// tile at the end of a run is shared: its CTAs leave their sums in scratch memory, and the last to do so adds them in the order of K, so
// that a result does not depend on timing.
//
//   weights_kernel   x in bfloat16.  Bulk tensor copies bring 128 x 256 codes (128-byte swizzle) and their scales into a ring, x in
//                    pieces of 128 elements into another.  Eight warps make the A operand of the codes, a thread a row and 64
//                    elements, in tensor memory; no shared memory is written for it.  One thread issues kind::f16 MMAs.
//                    Making A is what a scheduler has to do for each MMA: halfs are a conversion and a multiplication for two codes (13
//                    clocks for eight codes of a warp), bfloat16 goes through float32 (21 clocks).  So x comes as halfs, times a
//                    power of two a row, from a kernel before (mxfp4.cu), and w becomes halfs times one power of two of the matrix;
//                    both powers go into the results.  All of it is exact: the few elements that lie too far below a row's largest
//                    for halfs are added one by one to the sums (lost_products), and where there are too many of them (most_lost),
//                    or the matrix's scales span more than 36 powers, the whole product is made of bfloat16 instead (4% to a quarter slower).
//                    24,576 x 4,096 times 2,048 rows: 303 us, 1.36 PFLOP/s; the tensor pipe is busy 78% of the time at the 1.43 GHz that
//                    the power cap leaves.
//   both_kernel      x in 4 bits as well: codes of both sides go from shared memory into kind::mxf4 MMAs as they are, scales are copied into
//                    tensor memory (tcgen05.cp) stage by stage.  24,576 x 4,096 times 16 rows 13.5 us (380 ns a stage, 6.8 TB/s, beyond
//                    6 us), 2,048 rows 99 us, 4,096 rows 183 (4.5 PFLOP/s): 43 KB a stage of 192 tokens come to an SM in 0.41 us, 68
//                    bytes a clock at 1.44 GHz, which bounds it; the tensor pipe is busy 65% of the time.
//
//   parts_kernel     x in bfloat16 once more, up to 64 rows: as three parts of E5M2 (mxfp4.cu), 3 x 64 columns of kind::mxf8f6f4 MMAs whose A
//                    operand is the codes, brought into bytes by the bulk tensor copies: nobody makes anything of w.  The three
//                    columns' sums are the result's.  A few elements that three parts do not hold are added one by one as well; rows with
//                    more than 8 of them in 256 elements, and all such rows where they are more than LOST_MOST, are computed from bfloat16
//                    on mma.sync (wide_products), the others as ever: what one request's row holds costs its neighbours little, infinities
//                    and NaN nothing (E5M2 has both).
//                    24,576 x 4,096 times 64 rows: none 24 us, 1 element 25, 32 in as many rows 55, one such row 64, 64 such rows 206; 4,096 x
//                    12,288: 22, 23, 43, 40, 101.  (In a decode step of 64 tokens some element of silu(gate) * up nearly always is 2^26
//                    below its neighbours.  The CUDA cores took 3.5 and 5.3 ms for all rows as soon as one row had too many.)
//                    24,576 x 4,096 times 16 rows 16.6 us, x's preparation included (430 ns a stage, 6 TB/s, beyond 6.5 us), 32 rows
//                    19.5, 64 rows 23.8 (the parts of 32 and 64 tokens, 24 and 48 KB a stage beside 17, leave room for three stages).
//
// Every wait is bounded (tma.cuh).
#include <limits.h>

#include "mxfp4.cuh"
#include "tcgen05.cuh"

// What is made of x, and counters set to zero on the way (mxfp4.cu).
extern "C" {
long long mrs_mxfp4_scale_bytes(long long rows, long long width);
int mrs_mxfp4_quantise(int is_bf16, const void* x, void* codes, void* scales, long long rows, long long width, void* zeros, int zero_count, void* stream);
int mrs_mxfp4_rows_to_halfs(const void* x, void* halfs, void* factors, void* lost, long long rows, long long width, void* zeros, int zero_count, void* stream);
int mrs_mxfp4_rows_to_parts(const void* x, void* parts, void* scales, void* lost, int rows, int width, int tokens, void* zeros, int zero_count, void* stream);
int mrs_mxfp4_clear(void* zeros, int zero_count, void* stream);
}

namespace {

constexpr int BM = 128;                            // rows of w of a tile
constexpr int STAGE_K = 256;                       // elements of K of a stage of codes: 128 bytes a row
constexpr int CODE_BYTES = BM * 128, SCALE_BYTES = 2 * MX_TILE_BYTES;
constexpr int TMEM_COLUMNS = 512;

// Untiled copy of a multiple of 16 bytes, both sides on 16-byte boundaries.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(smem_u32(dst)), "l"(src), "r"(bytes), "r"(smem_u32(bar)) : "memory");
}
// A whole warp's bounded wait, whose outcome is the same for the whole warp and whose loop the compiler does not see: what the warp walks
// through stays in uniform registers, which the MMA and copy instructions take their operands from.  (With the loop of mbar_wait and
// breaks lane by lane a step of MMAs took 510 clocks to issue, and 24,576 x 4,096 times 2,048 rows 320 us; with this one and steps of 128
// elements instead of 64 301.)
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p, q;\n .reg .u64 start, now;\n"
                 " mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n @p bra DONE;\n"
                 " mov.u64 start, %%clock64;\n"
                 "AGAIN:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %4;\n @p bra DONE;\n"
                 " mov.u64 now, %%clock64;\n sub.u64 now, now, start;\n setp.lt.u64 q, now, %3;\n @q bra AGAIN;\n"
                 "DONE:\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done) : "r"(smem_u32(bar)), "r"(parity), "n"(MRS_WAIT_CYCLES), "r"(1000000u) : "memory");       // asleep for up to a millisecond a try
    if (__all_sync(0xffffffffu, done != 0u)) return true;
    mrs_raise(MRS_ERR_BARRIER_TIMEOUT);
    return false;
}

struct Shapes {
    int M, N, K;
    int token_tiles, depth;     // stages of a tile
    int units;                  // stages of all tiles
    int early;                  // w was there before the kernel before this one: it may be fetched while that runs
    long long w_tiles_of_a_row, x_row_tiles;
    const int* x_factors;       // of x as halfs (mxfp4.cu), a row each; null: x is bfloat16
    int lost_most;              // with more elements than this to add, bfloat16 operands are faster
    int w_exponent;             // halfs are made of w times 2^-w_exponent
    const int* lost;            // elements that halfs or parts do not hold (mxfp4.cuh)
    const uint8_t *w_codes, *w_scales;
    float* scratch;             // where tiles are shared, for every CTA the sums of its first and of its last tile
    int* arrived;               // for every tile how many CTAs have left their sums; zeros to begin with
};

// A CTA's tiles; [from, to) are the stages of the tile at hand.  Shared tiles: the CTA's run of units.  Whole ones: every gridDim.x-th, so
// that CTAs at work at the same time write neighbouring columns and read neighbouring weights.
struct Walk {
    int first, begin, total, done, from, to;       // `total` stages from unit `first` on, stage `begin` of its tile (whole tiles: of this CTA's own)
    int n_tile, token_tile, n_step, token_step;    // the tile at hand, and how far to the next: no division a tile
    __device__ __forceinline__ explicit Walk(const Shapes& s) : done(0), from(0), to(0) {
        int tile = blockIdx.x, step = gridDim.x;
        first = begin = 0;
        if (s.scratch) {
            first = start(s, blockIdx.x);
            total = start(s, blockIdx.x + 1) - first;
            tile = first / s.depth, step = 1;
            begin = first - tile * s.depth;
        } else {
            total = ((s.units / s.depth - 1 - tile) / step + 1) * s.depth;
        }
        n_step = step / s.token_tiles, token_step = step - n_step * s.token_tiles;
        n_tile = tile / s.token_tiles, token_tile = tile - n_tile * s.token_tiles;
    }
    __device__ static __forceinline__ int start(const Shapes& s, int cta) { return (int)((long long)s.units * cta / gridDim.x); }
    __device__ static __forceinline__ int owner(const Shapes& s, int unit) { return (int)(((long long)(unit + 1) * gridDim.x - 1) / s.units); }
    // Rows of w and stage of this CTA's `position`-th stage.
    __device__ __forceinline__ int n_tile_of(const Shapes& s, int position) const {
        const int index = (first + position) / s.depth;
        return (s.scratch ? index : (int)blockIdx.x + index * (int)gridDim.x) / s.token_tiles;
    }
    __device__ __forceinline__ int stage_of(const Shapes& s, int position) const { return (first + position) % s.depth; }
    __device__ __forceinline__ bool step(const Shapes& s) {
        if (done >= total) return false;
        from = begin;
        if (done > 0) {
            from = 0;
            n_tile += n_step, token_tile += token_step;
            if (token_tile >= s.token_tiles) token_tile -= s.token_tiles, ++n_tile;
        }
        to = min(s.depth, from + total - done);
        done += to - from;
        return true;
    }
};

// A number a row, added to a column of sums in tensor memory, by a warp of its rows.
__device__ __forceinline__ void add_to_column(uint32_t column, float more) {
    float sum;
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n tcgen05.wait::ld.sync.aligned;" : "=f"(sum) : "r"(column) : "memory");
    sum += more;
    asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};\n tcgen05.wait::st.sync.aligned;" ::"r"(column), "f"(sum) : "memory");
}
// The sum of a token's lost elements times a row of w, for a whole warp with a row a lane (rarely called: apart, so that it takes no
// registers of others; four tokens' side by side took a stack, 2 us of every call).  `counts` and `entries`: of the token's `stretches`.
__device__ __noinline__ float lost_products(const int* counts, const uint32_t* entries, int stretches, const uint8_t* codes, const uint8_t* scales) {
    const int lane = threadIdx.x & 31;
    float sum = 0.0f;
    for (int base = 0; base < stretches; base += 32) {
        const int count = base + lane < stretches ? __ldcg(counts + base + lane) : 0;
        for (uint32_t left = __ballot_sync(0xffffffffu, count != 0); left; left &= left - 1) {
            const int at = __ffs(left) - 1, n = __shfl_sync(0xffffffffu, count, at);
            for (int i = 0; i < n; ++i) {
                const uint32_t entry = __ldcg(entries + (size_t)(base + at) * MX_LOST + i);
                const size_t k = (size_t)(base + at) * STAGE_K + (entry >> 16);
                const uint32_t code = codes[k >> 1] >> (4 * (k & 1)), size = code & 7u;
                const float w = size < 2 ? 0.5f * size : __uint_as_float((126u + (size >> 1)) << 23 | (size & 1u) << 22);
                const float scale = mx_scale(scales[(k >> 7) * MX_TILE_BYTES + ((k >> 5) & 3)]);
                sum = fmaf(__uint_as_float(entry << 16), (code & 8u ? -w : w) * scale, sum);
            }
        }
    }
    return sum;
}

// An accumulator's results (lane: row of w, column: token) to memory.  Called by WARPS warps, `index` of them 0 to WARPS - 1; a warp's lanes
// are those of its number modulo 4.  `halfs`: the rows' powers of two go into them (`factors`: 32 floats of shared memory for each warp).  A
// tile that other CTAs share goes through scratch memory; `flag` is a word of shared memory.
// `lost`: null, or elements of x are missing in the sums; with parts, a bit for each token that has some, in shared memory, and behind these
// two words two with a bit for each token whose results are computed and stored elsewhere (wide_products).
template <int TOKENS, int WARPS, typename Out, bool PARTS = false>
__device__ __forceinline__ void store_accumulator(uint32_t accumulator, Out* __restrict__ out, const Shapes& s, const Walk& walk, int index, bool halfs, int* flag, float* factors,
                                                  const uint32_t* lost = nullptr) {
    constexpr int STEP = TOKENS < 32 || WARPS <= 8 ? 16 : 32, GROUPS = WARPS / 4;       // columns at a time (32: registers spill in kernels of 19 warps); of four warps
    constexpr int TOGETHER = PARTS || (STEP == 16 && WARPS > 8) ? 4 : 2;
    const int quarter = (threadIdx.x >> 5) & 3, row = quarter * 32 + (threadIdx.x & 31);
    const int token0 = walk.token_tile * TOKENS, live = min(TOKENS, s.M - token0), tile = walk.n_tile * s.token_tiles + walk.token_tile;
    const uint32_t acc = accumulator + ((uint32_t)(quarter * 32) << 16);
    const long long n = (long long)walk.n_tile * BM + row;
    const bool whole = walk.from == 0 && walk.to == s.depth;
    auto finish = [&](int c, float (&v)[STEP]) {
        if (halfs) {                               // powers of two in the floats' range, a lane each, by way of shared memory
            const int lane = threadIdx.x & 31;
            const int factor = lane < STEP && c + lane < live ? __ldcg(s.x_factors + token0 + c + lane) : -s.w_exponent * (1 << MX_NOTED_BITS);
            __syncwarp();
            if (lane < STEP) factors[lane] = __uint_as_float((uint32_t)(127 + s.w_exponent + (factor >> MX_NOTED_BITS)) << 23);
            __syncwarp();
#pragma unroll
            for (int e = 0; e < STEP; e += 4) {
                const float4 f = *reinterpret_cast<const float4*>(factors + e);
                v[e] *= f.x, v[e + 1] *= f.y, v[e + 2] *= f.z, v[e + 3] *= f.w;
            }
        }
        if (n < s.N) {
            Out* place = out + (size_t)(token0 + c) * s.N + n;
            uint32_t left = 0;
            if constexpr (PARTS) left = lost[2 + (c >> 5)] >> (c & 31) & ((1ull << STEP) - 1);
            if (c + STEP <= live && left == 0) {
#pragma unroll
                for (int e = 0; e < STEP; ++e) place[(size_t)e * s.N] = from_float<Out>(v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < STEP; ++e)
                    if (c + e < live && !(left >> e & 1u)) place[(size_t)e * s.N] = from_float<Out>(v[e]);
            }
        }
    };
    // Lost elements go into the sums in tensor memory, where each warp takes up the columns that it reads; of a shared tile, the CTA with its beginning.
    if (lost && walk.from == 0) {
#pragma unroll 1
        for (int c = (index >> 2) * STEP; c < live; c += GROUPS * STEP) {
            const int lane = threadIdx.x & 31;
            int factor = 0;
            if constexpr (PARTS) factor = (lost[c >> 5] >> ((c + lane) & 31)) & (lane < STEP ? 1u : 0u);
            else if (lane < STEP && c + lane < live) factor = __ldcg(s.x_factors + token0 + c + lane);
            for (uint32_t some = __ballot_sync(0xffffffffu, factor & MX_NOTED); some; some &= some - 1) {
                const int at = __ffs(some) - 1;
                const long long of = n < s.N ? n : s.N - 1, token = token0 + c + at;
                float more = lost_products(s.lost + token * s.depth, mx_lost_entries(s.lost, (long long)s.M * s.depth) + token * s.depth * MX_LOST, s.depth,
                                           s.w_codes + of * (s.K >> 1), s.w_scales + mx_scale_offset(of, 0, s.w_tiles_of_a_row));
                if constexpr (!PARTS) more *= __uint_as_float((uint32_t)(127 - s.w_exponent - (__shfl_sync(0xffffffffu, factor, at) >> MX_NOTED_BITS)) << 23);
                add_to_column(acc + c + at, more);
            }
        }
    }
    // a CTA's sums of a shared tile: [column / 4][row] of four columns
    auto place_of = [&](int cta, bool head) { return reinterpret_cast<float4*>(s.scratch + ((size_t)cta * 2 + (head ? 1 : 0)) * (TOKENS * BM)) + row; };
    float4* mine = place_of(blockIdx.x, walk.from == 0);
#pragma unroll 1
    for (int c = (index >> 2) * STEP; c < live; c += GROUPS * STEP) {
        float v[STEP];
        if constexpr (STEP == 16) tmem_load_16_async(acc + c, v);
        else tmem_load_32_async(acc + c, v);
        tmem_load_wait();
        if constexpr (PARTS) {                     // the other two parts' columns, the smallest sums first
            float rest[STEP], least[STEP];
            if constexpr (STEP == 16) tmem_load_16_async(acc + TOKENS + c, rest), tmem_load_16_async(acc + 2 * TOKENS + c, least);
            else tmem_load_32_async(acc + TOKENS + c, rest), tmem_load_32_async(acc + 2 * TOKENS + c, least);
            tmem_load_wait();
#pragma unroll
            for (int e = 0; e < STEP; ++e) v[e] += rest[e] + least[e];
        }
        if (whole) {
            finish(c, v);
        } else {
#pragma unroll
            for (int e = 0; e < STEP; e += 4) __stcg(mine + ((c + e) >> 2) * BM, make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]));
        }
    }
    if (whole) return;
    const int first = Walk::owner(s, tile * s.depth), last = Walk::owner(s, (tile + 1) * s.depth - 1);
    __threadfence();
    asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
    if (index == 0 && (threadIdx.x & 31) == 0) *flag = atomicAdd(s.arrived + tile, 1) == last - first;
    asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");
    const bool finisher = *flag != 0;
    asm volatile("bar.sync 1, %0;" ::"n"(WARPS * 32) : "memory");               // the flag is read by all before it is written again
    if (!finisher) return;
    __threadfence();
#pragma unroll 1
    for (int c = (index >> 2) * STEP; c < live; c += GROUPS * STEP) {
        float v[STEP];
        // in the order of K, the first CTA's at the end of its run; TOGETHER pieces on the way at a time
#pragma unroll 1
        for (int cta = first; cta <= last; cta += TOGETHER) {
            float4 piece[TOGETHER][STEP / 4];
#pragma unroll
            for (int t = 0; t < TOGETHER; ++t) {
                const float4* from = place_of(min(cta + t, last), cta + t == first) + (c >> 2) * BM;
#pragma unroll
                for (int e = 0; e < STEP / 4; ++e) piece[t][e] = __ldcg(from + e * BM);
            }
#pragma unroll
            for (int t = 0; t < TOGETHER; ++t) {
                if (cta + t > last) break;
                const bool begin = cta + t == first;
#pragma unroll
                for (int e = 0; e < STEP / 4; ++e) {
                    v[4 * e] = begin ? piece[t][e].x : v[4 * e] + piece[t][e].x;
                    v[4 * e + 1] = begin ? piece[t][e].y : v[4 * e + 1] + piece[t][e].y;
                    v[4 * e + 2] = begin ? piece[t][e].z : v[4 * e + 2] + piece[t][e].z;
                    v[4 * e + 3] = begin ? piece[t][e].w : v[4 * e + 3] + piece[t][e].w;
                }
            }
        }
        finish(c, v);
    }
}

// ------------------------------------------------------------------------------------------
// x in bfloat16
// ------------------------------------------------------------------------------------------
constexpr int PIECE_K = 64;                        // a 128-byte row of x, and what one thread makes of its row at a time
// Elements of K of a step: a buffer of A and a slot of x.  The issuing warp's waits and commits cost some 400 clocks a step beside the
// warps that make A, as much as 40 MMAs of 16 tokens or 4 of 192; tensor memory bounds the steps of wide tiles.
template <int TOKENS> constexpr int step_k() { return TOKENS <= 64 ? 256 : 128; }
// Warps that make A, and that store results.  Sixteen and four took 757 us for 151,936 x 1,024 times 2,048 rows (four storers need 13,000
// to 22,000 clocks a tile, its MMAs 6,200), these 506; 24,576 x 4,096 took 301 and 305.
constexpr int MAKERS = 8, STORERS = 8;
constexpr int W_THREADS = (3 + MAKERS + STORERS) * 32;
// How many elements the storing warps may add one by one before bfloat16 operands are faster for all.  These cost 0.1 to 0.15 us for each of the
// `stages` of the CTA with most of them, with up to 128 tokens, where making A counts for more, 0.3.  An element takes the warps that store its
// tile of tokens 0.5 to 1 us, the first one 1 to 2 more; of several tiles a CTA only the last one's wait is not hidden behind MMAs, but for short
// tiles, whose results take as long to store as they take.
// Measured (us, without any / some in a row each, in few rows / bfloat16 operands):
//   24,576 x 4,096: 2,048 rows 305 / 64: 314, 313 / 338, 512 rows 83 / 8: 86, 88 / 92, 200 rows 55 / 8: 61, 62 / 70, 100 rows 39 / 3: 43, 43 / 49;
//   4,096 x 12,288: 2,048 rows 188 / 64: 199, 196 / 202, 512 rows 55 / 24: 66, 64 / 71, 200 rows 40 / 3: 45, 43 / 46;
//   6,145 x 4,096: 485 rows 27.0 / 1: 29.2 / 28.3; 151,936 x 1,024: 700 rows 187 / 1: 237 / 203; 24,576 x 4,128: 24 rows 31 / 3: 37, 35 / 38.
inline int most_lost(int tokens, int token_tiles, int stages, int depth) {
    const int hidden = stages > depth ? depth - 6 : depth, tile = tokens > 128 ? stages / 10 - 2 : stages / 5 - 1;
    return max(0, min(hidden, tile)) * token_tiles;
}
template <int TOKENS> constexpr int a_columns() { return step_k<TOKENS>() / 2; }
template <int TOKENS> constexpr int x_bytes() { return TOKENS * step_k<TOKENS>() * 2; }
template <int TOKENS> constexpr int x_stages() { return TOKENS > 128 ? 3 : 4; }
template <int TOKENS> constexpr int w_stages() { return TOKENS > 128 ? 4 : TOKENS > 32 ? 5 : 8; }      // as many as fit
template <int TOKENS> constexpr int a_first() { return TOKENS > 128 ? 2 * TOKENS : 256; }            // columns before it: two accumulators
template <int TOKENS> constexpr int a_buffers() { return (TMEM_COLUMNS - a_first<TOKENS>()) / a_columns<TOKENS>(); }
template <int TOKENS> constexpr size_t weights_smem() {
    return 1024 + (size_t)w_stages<TOKENS>() * (CODE_BYTES + SCALE_BYTES) + (size_t)x_stages<TOKENS>() * x_bytes<TOKENS>() + 512;
}

// 32 codes of a row as 16 pairs of halfs, times 2^(byte - 127 - w_exponent); only blocks of zeros have powers beyond [-23, 13].
__device__ __forceinline__ void decode_block_halfs(uint4 codes, uint32_t byte, int w_exponent, uint32_t* words) {
    const int d = max(min((int)byte - 127 - w_exponent, 15), -24);
    const uint32_t bits = d >= -14 ? (uint32_t)(d + 15) << 10 : 1u << (d + 24), both = bits | bits << 16;
    const __half2 scale = *reinterpret_cast<const __half2*>(&both);
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t h[4];
        mx_decode_8(w[i], h);
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const __half2 pair = __hmul2(*reinterpret_cast<const __half2*>(&h[p]), scale);
            words[i * 4 + p] = *reinterpret_cast<const uint32_t*>(&pair);
        }
    }
}
// 2^(byte - 127) as a pair of bfloat16: byte 0 under the ordinary numbers, byte 255 not a number.
__device__ __forceinline__ __nv_bfloat162 scale_pair(uint32_t byte) {
    const uint32_t bits = byte == 0u ? 0x0040u : byte == 255u ? 0x7FC0u : byte << 7, both = bits | bits << 16;
    return *reinterpret_cast<const __nv_bfloat162*>(&both);
}
// Eight codes times their scale as four pairs of bfloat16.
__device__ __forceinline__ void decode_eight(uint32_t codes, __nv_bfloat162 scale, uint32_t* words) {
    uint32_t h[4];
    mx_decode_8(codes, h);
#pragma unroll
    for (int p = 0; p < 4; ++p) {
        const float2 v = __half22float2(*reinterpret_cast<__half2*>(&h[p]));
        const __nv_bfloat162 pair = __hmul2(__floats2bfloat162_rn(v.x, v.y), scale);
        words[p] = *reinterpret_cast<const uint32_t*>(&pair);
    }
}
// 32 codes of a row and their scale byte as 16 pairs of bfloat16.
__device__ __forceinline__ void decode_block(uint4 codes, uint32_t byte, uint32_t* words) {
    const __nv_bfloat162 scale = scale_pair(byte);
    const uint32_t w[4] = {codes.x, codes.y, codes.z, codes.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) decode_eight(w[i], scale, words + 4 * i);
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
__global__ void __launch_bounds__(W_THREADS, 1) weights_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                               const __grid_constant__ CUtensorMap halfs_map, const uint8_t* __restrict__ scales,
                                                               Out* __restrict__ out, const Shapes s) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int A_FIRST = a_first<TOKENS>(), A_BUFFERS = a_buffers<TOKENS>(), ACCUMULATOR = A_FIRST / 2, X_STAGES = x_stages<TOKENS>(), W_STAGES = w_stages<TOKENS>();
    constexpr int STEP_K = step_k<TOKENS>(), STAGE_STEPS = STAGE_K / STEP_K, STEP_PIECES = STEP_K / PIECE_K, A_COLUMNS = a_columns<TOKENS>();
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
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    int* flag = reinterpret_cast<int*>(tmem_slot + 1);
    __shared__ __align__(16) float factors[STORERS * 32];
    __shared__ int lost_count;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Walk walk(s);
    // Steps of the tile at hand.  Every stage has all of its steps, also where K ends before (these are made of zeros): the warps that
    // make a step then use the buffers of A in turn, and are never more than one use of a buffer behind.
    auto steps_of = [&]() { return (walk.to - walk.from) * STAGE_STEPS; };

    if (threadIdx.x == 0) {
        lost_count = 0;
        for (int i = 0; i < W_STAGES; ++i) {
            mbar_init(&w_full[i], 1);
            mbar_init(&w_empty[i], MAKERS);
        }
        for (int i = 0; i < X_STAGES; ++i) {
            mbar_init(&x_full[i], 1);
            mbar_init(&x_empty[i], 1);
        }
        for (int i = 0; i < A_BUFFERS; ++i) {
            mbar_init(&a_full[i], 4 * STEP_PIECES);
            mbar_init(&a_empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], STORERS);
        }
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

    // The codes' first stages are on their way before anything else; then, once the kernel before has ended, whether all of x is there as
    // halfs whose powers, with the matrix's, are ordinary floats.
    const int ahead = s.early ? min(W_STAGES, walk.total) : 0;
    auto load_codes = [&](int n_tile, int stage, int slot) {
        mbar_arrive_expect_tx(&w_full[slot], CODE_BYTES + SCALE_BYTES);
        tma_load_2d(w_ring + slot * CODE_BYTES, &w_map, &w_full[slot], stage * 128, n_tile * BM);
        bulk_load(s_ring + slot * SCALE_BYTES, scales + ((size_t)n_tile * s.w_tiles_of_a_row + 2 * stage) * MX_TILE_BYTES, SCALE_BYTES, &w_full[slot]);
    };
    if (warp == 2 + MAKERS + STORERS) {
        if (elect_one())
            for (int i = 0; i < ahead; ++i) load_codes(walk.n_tile_of(s, i), walk.stage_of(s, i), i);
        __syncwarp();
    }
    pdl_wait();
    bool halfs = false, lost = false;
    if (s.x_factors) {
        bool fit = true;
        int some = 0;
        for (int i = threadIdx.x; i < s.M; i += W_THREADS) {
            const int factor = s.x_factors[i], e = factor >> MX_NOTED_BITS;
            fit = fit && factor != INT_MIN && e + s.w_exponent >= -126 && e + s.w_exponent <= 126;
            some = min(some + (factor & MX_NOTED), 1 << 20);
        }
        if (some) atomicAdd(&lost_count, some);
        halfs = __syncthreads_and(fit) && lost_count <= s.lost_most;
        lost = halfs && lost_count != 0;
    }

    // Codes and x come by the hands of two warps: a wait for the makers must not hold up x, whose pieces free up MMA by MMA.
    if (warp == 0) {
        const bool leader = elect_one();
        const CUtensorMap* map = halfs ? &halfs_map : &x_map;
        bool alive = true;
        int slot = 0;
        uint32_t phase = 1;
        while (alive && walk.step(s)) {
            const int token0 = walk.token_tile * TOKENS, steps = steps_of();
            for (int step = 0; step < steps; ++step) {
                if (!(alive = warp_wait(&x_empty[slot], phase))) break;
                if (leader) {
                    mbar_arrive_expect_tx(&x_full[slot], x_bytes<TOKENS>());
#pragma unroll
                    for (int h = 0; h < STEP_PIECES; ++h)
                        tma_load_2d(x_ring + slot * x_bytes<TOKENS>() + h * (TOKENS * 128), map, &x_full[slot],
                                    (walk.from * STAGE_STEPS + step) * STEP_K + h * PIECE_K, token0);
                }
                __syncwarp();
                if (++slot == X_STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 2 + MAKERS + STORERS) {
        const bool leader = elect_one();
        bool alive = true;
        int slot = 0;
        uint32_t phase = 1;
        int count = 0;
        while (alive && walk.step(s)) {
            const int n_tile = walk.n_tile;
            for (int stage = walk.from; stage < walk.to; ++stage, ++count) {
                if (count >= ahead) {                     // not even the wait before: the makers may be through with those stages
                    if (!(alive = warp_wait(&w_empty[slot], phase))) break;
                    if (leader) load_codes(n_tile, stage, slot);
                    __syncwarp();
                }
                if (++slot == W_STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 1) {
        const bool leader = elect_one();
        const uint32_t idesc = umma_idesc_bf16_f32(BM, TOKENS) & (halfs ? ~((1u << 7) | (1u << 10)) : ~0u);      // both operands halfs, or both bfloat16
        bool alive = true;
        int x_slot = 0, a_slot = 0, round = 0;
        uint32_t x_phase = 0, a_phase = 0;
        for (; alive && walk.step(s); ++round) {
            const int buffer = round & 1, steps = steps_of();
            if (!(alive = warp_wait(&acc_empty[buffer], ((round >> 1) & 1) ^ 1))) break;
            tcgen05_fence_after_sync();
            const uint32_t d_tmem = tmem + buffer * ACCUMULATOR;
            for (int step = 0; step < steps; ++step) {
                if (!(alive = warp_wait(&x_full[x_slot], x_phase))) break;
                if (!(alive = warp_wait(&a_full[a_slot], a_phase))) break;
                tcgen05_fence_after_sync();
                const uint64_t b_desc = umma_smem_desc_sw128(smem_u32(x_ring + x_slot * x_bytes<TOKENS>()));
                const uint32_t a_tmem = tmem + A_FIRST + a_slot * A_COLUMNS;
                if (leader) {
#pragma unroll
                    for (int k = 0; k < STEP_K / 16; ++k)
                        umma_bf16_a_tmem(d_tmem, a_tmem + 8 * k, b_desc + (k >> 2) * (TOKENS * 128 / 16) + 2 * (k & 3), idesc, step > 0 || k > 0);
                    umma_commit(&x_empty[x_slot]);
                    umma_commit(&a_empty[a_slot]);
                }
                __syncwarp();
                if (++x_slot == X_STAGES) x_slot = 0, x_phase ^= 1;
                if (++a_slot == A_BUFFERS) a_slot = 0, a_phase ^= 1;
            }
            if (leader) umma_commit(&acc_full[buffer]);
            __syncwarp();
        }
    } else if (warp < 2 + MAKERS) {
        const int quarter = warp & 3, group = (warp - 2) >> 2, row = quarter * 32 + lane;        // group: every GROUPS-th piece of a stage
        const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16) + A_FIRST;
        constexpr int GROUPS = MAKERS / 4, STAGE_PIECES = STAGE_K / PIECE_K;
        bool alive = true;
        int w_slot = 0;
        uint32_t w_phase = 0;
        for (int stage = 0; stage < walk.total && alive; ++stage) {                              // of the CTA's run
            if (!(alive = warp_wait(&w_full[w_slot], w_phase))) break;
            const unsigned char* codes = w_ring + w_slot * CODE_BYTES + row * 128;
            const unsigned char* scale_bytes = s_ring + w_slot * SCALE_BYTES + lane * 16 + quarter * 4;
#pragma unroll 1
            for (int piece = group; piece < STAGE_PIECES; piece += GROUPS) {
                const uint32_t two = *reinterpret_cast<const uint16_t*>(scale_bytes + (piece >> 1) * MX_TILE_BYTES + (piece & 1) * 2);
                const uint4 first = *reinterpret_cast<const uint4*>(codes + (((piece * 2) ^ (row & 7)) << 4));
                const uint4 second = *reinterpret_cast<const uint4*>(codes + (((piece * 2 + 1) ^ (row & 7)) << 4));
                uint32_t words[32];
                if (halfs) {
                    decode_block_halfs(first, two & 255u, s.w_exponent, words);
                    decode_block_halfs(second, two >> 8, s.w_exponent, words + 16);
                } else {
                    decode_block(first, two & 255u, words);
                    decode_block(second, two >> 8, words + 16);
                }
                const int step = stage * STAGE_STEPS + piece / STEP_PIECES, b = step % A_BUFFERS;
                if (!(alive = warp_wait(&a_empty[b], ((step / A_BUFFERS) & 1) ^ 1))) break;
                tcgen05_fence_after_sync();
                tmem_store_32_words(lanes + b * A_COLUMNS + piece % STEP_PIECES * (PIECE_K / 2), words);
                tmem_store_wait();
                tcgen05_fence_before_sync();
                __syncwarp();
                if (lane == 0) mbar_arrive(&a_full[b]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&w_empty[w_slot]);
            if (++w_slot == W_STAGES) w_slot = 0, w_phase ^= 1;
        }
    } else {
        for (int round = 0; walk.step(s); ++round) {
            const int buffer = round & 1;
            if (!warp_wait(&acc_full[buffer], (round >> 1) & 1) && !s.scratch) break;      // of shared tiles the others meet this warp at barriers
            tcgen05_fence_after_sync();
            store_accumulator<TOKENS, STORERS, Out>(tmem + buffer * ACCUMULATOR, out, s, walk, warp - 2 - MAKERS, halfs, flag, factors + (warp - 2 - MAKERS) * 32,
                                                   lost ? reinterpret_cast<const uint32_t*>(s.lost) : nullptr);
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buffer]);
        }
    }
    __syncwarp();
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

constexpr int B_STORERS = 12, B_THREADS = (3 + B_STORERS) * 32;
// as many stages as shared memory holds, and tensor memory of their scales
template <int TOKENS> constexpr int b_stages() { return TOKENS > 128 ? 5 : TOKENS > 64 ? 6 : TOKENS > 32 ? 8 : 9; }
template <int TOKENS> constexpr int token_blocks() { return TOKENS > 128 ? 2 : 1; }            // tiles of scales of the tokens
template <int TOKENS> constexpr int both_stage_bytes() { return CODE_BYTES + TOKENS * 128 + SCALE_BYTES * (1 + token_blocks<TOKENS>()); }
template <int TOKENS> constexpr size_t both_smem() { return 1024 + (size_t)b_stages<TOKENS>() * both_stage_bytes<TOKENS>() + 256; }
// Tensor memory: two accumulators, then a stage's scales in 24 columns: 2 x 4 of w, 2 x 8 of the tokens.
constexpr int SCALE_COLUMNS = 24;

template <int TOKENS, typename Out>
__global__ void __launch_bounds__(B_THREADS, 1) both_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                            const uint8_t* __restrict__ w_scales, const uint8_t* __restrict__ x_scales, Out* __restrict__ out,
                                                            const Shapes s) {
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int STAGE_SCALES = SCALE_BYTES * (1 + token_blocks<TOKENS>()), B_STAGES = b_stages<TOKENS>();
    constexpr int B_ACCUMULATOR = TOKENS > 128 ? TOKENS : 128, SCALES_FIRST = 2 * B_ACCUMULATOR;
    static_assert(SCALES_FIRST + B_STAGES * SCALE_COLUMNS <= TMEM_COLUMNS, "tensor memory");
    unsigned char* w_ring = smem;
    unsigned char* x_ring = w_ring + B_STAGES * CODE_BYTES;
    unsigned char* s_ring = x_ring + B_STAGES * TOKENS * 128;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_ring + B_STAGES * STAGE_SCALES);
    uint64_t* empty = full + B_STAGES;
    uint64_t* acc_full = empty + B_STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    int* flag = reinterpret_cast<int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Walk walk(s);

    if (threadIdx.x == 0) {
        for (int i = 0; i < B_STAGES; ++i) {
            mbar_init(&full[i], 2);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], B_STORERS);
        }
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

    // w and x come by the hands of two warps, each with its scales: four or five copies a stage took one warp some 600 clocks.
    if (warp == 0) {
        const bool leader = elect_one();
        pdl_wait();
        bool alive = true;
        int slot = 0;
        uint32_t phase = 1;
        while (alive && walk.step(s)) {
            const int token0 = walk.token_tile * TOKENS;
            const uint8_t* tile_scales = x_scales + (size_t)(token0 >> 7) * s.w_tiles_of_a_row * MX_TILE_BYTES;
            // a tile behind the last token: nobody stores its sums
            const size_t second = (token0 >> 7) + 1 < s.x_row_tiles ? (size_t)s.w_tiles_of_a_row * MX_TILE_BYTES : 0;
            for (int stage = walk.from; stage < walk.to; ++stage) {
                if (!(alive = warp_wait(&empty[slot], phase))) break;
                if (leader) {
                    mbar_arrive_expect_tx(&full[slot], TOKENS * 128 + SCALE_BYTES * token_blocks<TOKENS>());
                    tma_load_2d(x_ring + slot * TOKENS * 128, &x_map, &full[slot], stage * 128, token0);
#pragma unroll
                    for (int t = 0; t < token_blocks<TOKENS>(); ++t)
                        bulk_load(s_ring + slot * STAGE_SCALES + SCALE_BYTES * (1 + t), tile_scales + t * second + (size_t)stage * SCALE_BYTES, SCALE_BYTES, &full[slot]);
                }
                __syncwarp();
                if (++slot == B_STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 2 + B_STORERS) {
        const bool leader = elect_one();
        if (!s.early) pdl_wait();
        bool alive = true;
        int slot = 0;
        uint32_t phase = 1;
        while (alive && walk.step(s)) {
            const int n_tile = walk.n_tile;
            const uint8_t* tile_scales = w_scales + (size_t)n_tile * s.w_tiles_of_a_row * MX_TILE_BYTES;
            for (int stage = walk.from; stage < walk.to; ++stage) {
                if (!(alive = warp_wait(&empty[slot], phase))) break;
                if (leader) {
                    mbar_arrive_expect_tx(&full[slot], CODE_BYTES + SCALE_BYTES);
                    tma_load_2d(w_ring + slot * CODE_BYTES, &w_map, &full[slot], stage * 128, n_tile * BM);
                    bulk_load(s_ring + slot * STAGE_SCALES, tile_scales + (size_t)stage * SCALE_BYTES, SCALE_BYTES, &full[slot]);
                }
                __syncwarp();
                if (++slot == B_STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 1) {
        pdl_wait();
        const bool leader = elect_one();
        bool alive = true;
        int slot = 0, round = 0;
        uint32_t phase = 0;
        for (; alive && walk.step(s); ++round) {
            const int buffer = round & 1;
            if (!(alive = warp_wait(&acc_empty[buffer], ((round >> 1) & 1) ^ 1))) break;
            tcgen05_fence_after_sync();
            const uint32_t d_tmem = tmem + buffer * B_ACCUMULATOR;
            // tiles of 192 tokens begin in the middle of a tile of scales every other time: two columns, 64 tokens, further in
            const uint32_t shift = TOKENS == 192 ? (((uint32_t)walk.token_tile * TOKENS) & 127u) / 32 : 0u;
            for (int index = 0; index < walk.to - walk.from; ++index) {
                if (!(alive = warp_wait(&full[slot], phase))) break;
                tcgen05_fence_after_sync();
                const uint64_t a_desc = umma_smem_desc_sw128(smem_u32(w_ring + slot * CODE_BYTES));
                const uint64_t b_desc = umma_smem_desc_sw128(smem_u32(x_ring + slot * TOKENS * 128));
                const uint32_t scales = smem_u32(s_ring + slot * STAGE_SCALES);
                const uint32_t columns = tmem + SCALES_FIRST + slot * SCALE_COLUMNS;
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
                        umma_mxf4(d_tmem, a_desc + 2 * k, b_desc + 2 * k, mxf4_idesc(BM, TOKENS, (k & 1) * 2), columns + (k >> 1) * 4,
                                  columns + 8 + (k >> 1) * 8 + shift, index > 0 || k > 0);
                    umma_commit(&empty[slot]);
                }
                __syncwarp();
                if (++slot == B_STAGES) slot = 0, phase ^= 1;
            }
            if (leader) umma_commit(&acc_full[buffer]);
            __syncwarp();
        }
    } else {
        pdl_wait();
        for (int round = 0; walk.step(s); ++round) {
            const int buffer = round & 1;
            if (!warp_wait(&acc_full[buffer], (round >> 1) & 1) && !s.scratch) break;      // of shared tiles the others meet this warp at barriers
            tcgen05_fence_after_sync();
            store_accumulator<TOKENS, B_STORERS, Out>(tmem + buffer * B_ACCUMULATOR, out, s, walk, warp - 2, false, flag, nullptr);
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buffer]);
        }
    }
    __syncwarp();
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc(tmem, TMEM_COLUMNS);
    }
}

// ------------------------------------------------------------------------------------------
// x in three parts
// ------------------------------------------------------------------------------------------
// kind::mxf8f6f4: A E2M1 (a code a byte of shared memory, 16 codes in 8 bytes and 8 unused), B E5M2, one E8M0 scale for 32 elements, K 32;
// `id`: which of a word's four scales.
__host__ __device__ constexpr uint32_t mxf8f6f4_idesc(int m, int n, uint32_t id) {
    return (id << 4)                      // scales of B
           | (5u << 7) | (1u << 10)       // A: E2M1, B: E5M2
           | ((uint32_t)(n >> 3) << 17)   // N / 8
           | (1u << 23)                   // scales: E8M0
           | ((uint32_t)(m >> 7) << 27)   // M / 128
           | (id << 29);                  // scales of A
}
__device__ __forceinline__ void umma_mxf8f6f4(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t a_scales, uint32_t b_scales, bool accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %6, 0;\n"
                 " tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n}"
                 ::"r"(d), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(a_scales), "r"(b_scales), "r"((uint32_t)accumulate) : "memory");
}

constexpr int HALF_STAGE_K = 128;                          // elements of K of a 128-byte row of bytes
constexpr int P_A_BYTES = BM * HALF_STAGE_K;               // half a stage of w in shared memory, of which the copies count half
constexpr int P_STORERS = 8, P_THREADS = (3 + P_STORERS) * 32;
// A slot of the ring holds a stage, with 64 tokens half of one: their parts are longer than the codes, and five halves in flight fit where
// two stages would.
template <int TOKENS> constexpr int p_halves() { return TOKENS > 32 ? 1 : 2; }
template <int TOKENS> constexpr int p_stages() { return TOKENS > 32 ? 5 : TOKENS > 16 ? 3 : 4; }
template <int TOKENS> constexpr int p_x_bytes() { return 3 * TOKENS * HALF_STAGE_K; }
template <int TOKENS> constexpr int p_x_tiles() { return (3 * TOKENS + 127) / 128; }                     // of scales
template <int TOKENS> constexpr int p_slot_scale_bytes() { return p_halves<TOKENS>() * MX_TILE_BYTES * (1 + p_x_tiles<TOKENS>()); }
template <int TOKENS> constexpr size_t parts_smem() {
    return 1024 + (size_t)p_stages<TOKENS>() * (p_halves<TOKENS>() * (P_A_BYTES + p_x_bytes<TOKENS>()) + p_slot_scale_bytes<TOKENS>()) + 256;
}

// With more elements to add than this for every 16 tokens that have some, these tokens take the products below (64 rows: an element costs 0.5
// to 1 us, 16 tokens there 13 to 48).
constexpr int LOST_MOST = 32;

// The results of the tokens of a mask (bits of `low` and `high`) whose elements three parts do not hold, from x as it is and codes times their
// scale in bfloat16 (both exact, mma.sync, sums in float32).  A CTA takes 16 rows of w and 16 of the tokens at a time, its warps a range of K
// each, whose sums meet in shared memory (`pieces`: 1 KB a warp) in the order of K.  Of 128 elements of K lane (g, t) takes block t: of rows g
// and g + 8 of w and of the tokens g and g + 8.  It decodes eight codes at a time: with a whole block the kernel has 147 registers a thread
// instead of 121, the kernel that prepares the next x no longer fits beside it, and every product takes 2.3 us longer.
template <int WARPS, typename Out>
__device__ __forceinline__ void wide_products(const bf16* __restrict__ x, Out* __restrict__ out, const Shapes& s, uint32_t low, uint32_t high, float* pieces) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, count = __popc(low) + __popc(high), steps = s.K / HALF_STAGE_K;
    const int from = (int)((long long)steps * warp / WARPS), to = (int)((long long)steps * (warp + 1) / WARPS);
    auto token_of = [&](int index) {                // the index-th of them; behind the last the last
        index = min(index, count - 1);
        return index < __popc(low) ? (int)__fns(low, 0, index + 1) : 32 + (int)__fns(high, 0, index - __popc(low) + 1);
    };
    for (int group = blockIdx.x; group < (s.N + 15) / 16; group += gridDim.x) {
        const long long n = (long long)group * 16, rows[2] = {min(n + g, (long long)s.N - 1), min(n + g + 8, (long long)s.N - 1)};
        const uint8_t *codes[2], *scales[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) codes[r] = s.w_codes + rows[r] * (s.K >> 1) + t * 16, scales[r] = s.w_scales + mx_scale_offset(rows[r], 0, s.w_tiles_of_a_row) + t;
        for (int base = 0; base < count; base += 16) {
            const bf16 *first = x + (size_t)token_of(base + g) * s.K + t * MX_BLOCK, *second = x + (size_t)token_of(base + 8 + g) * s.K + t * MX_BLOCK;
            float sums[2][4] = {};
            for (int q = from; q < to; ++q) {
                const uint4 held[2] = {*reinterpret_cast<const uint4*>(codes[0] + q * 64), *reinterpret_cast<const uint4*>(codes[1] + q * 64)};
                const __nv_bfloat162 scale[2] = {scale_pair(scales[0][(size_t)q * MX_TILE_BYTES]), scale_pair(scales[1][(size_t)q * MX_TILE_BYTES])};
                const uint32_t words[2][4] = {{held[0].x, held[0].y, held[0].z, held[0].w}, {held[1].x, held[1].y, held[1].z, held[1].w}};
#pragma unroll
                for (int i = 0; i < 4; ++i) {       // eight elements of the block
                    const uint4 a = *reinterpret_cast<const uint4*>(first + q * HALF_STAGE_K + i * 8), b = *reinterpret_cast<const uint4*>(second + q * HALF_STAGE_K + i * 8);
                    uint32_t w[2][4];
                    decode_eight(words[0][i], scale[0], w[0]);
                    decode_eight(words[1][i], scale[1], w[1]);
                    const uint32_t even[4] = {w[0][0], w[1][0], w[0][1], w[1][1]}, odd[4] = {w[0][2], w[1][2], w[0][3], w[1][3]};
                    mx_mma_bf16(sums[0], even, a.x, a.y);
                    mx_mma_bf16(sums[1], even, b.x, b.y);
                    mx_mma_bf16(sums[0], odd, a.z, a.w);
                    mx_mma_bf16(sums[1], odd, b.z, b.w);
                }
            }
            // [warp][token][row]
#pragma unroll
            for (int i = 0; i < 8; ++i) pieces[warp * 256 + ((i >> 2) * 8 + 2 * t + (i & 1)) * 16 + g + (i >> 1 & 1) * 8] = sums[i >> 2][i & 3];
            __syncthreads();
            const int index = base + ((int)threadIdx.x >> 4);
            if (threadIdx.x < 256 && index < count && n + (threadIdx.x & 15) < s.N) {
                float sum = pieces[threadIdx.x];
#pragma unroll
                for (int w = 1; w < WARPS; ++w) sum += pieces[w * 256 + threadIdx.x];
                out[(size_t)token_of(index) * s.N + n + (threadIdx.x & 15)] = from_float<Out>(sum);
            }
            __syncthreads();
        }
    }
}

template <int TOKENS, typename Out>
__global__ void __launch_bounds__(P_THREADS, 1) parts_kernel(const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map,
                                                             const bf16* __restrict__ x, const uint8_t* __restrict__ x_scales, Out* __restrict__ out, const Shapes s) {
    __shared__ uint32_t lost_tokens[4];             // a bit a token with elements to add; a bit a token with too many
    __shared__ int lost_count;                      // elements to add
    static_assert(TOKENS <= 64);
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    constexpr int STAGES = p_stages<TOKENS>(), N_COLUMNS = 3 * TOKENS, ACCUMULATOR = N_COLUMNS > 128 ? 192 : 128, SCALES_FIRST = 2 * ACCUMULATOR;
    constexpr int HALVES = p_halves<TOKENS>(), PIECES = 2 / HALVES, X_TILES = p_x_tiles<TOKENS>(), X_BYTES = p_x_bytes<TOKENS>();     // pieces: slots a stage
    constexpr int W_SCALE_BYTES = HALVES * MX_TILE_BYTES, SLOT_SCALE_BYTES = p_slot_scale_bytes<TOKENS>();      // of a slot: w's scales, then the parts', tiles of 128 by tiles
    constexpr int SCALE_COLUMNS = HALVES * 4 * (1 + X_TILES);                          // in tensor memory, of a slot
    static_assert(SCALES_FIRST + STAGES * SCALE_COLUMNS <= TMEM_COLUMNS);
    unsigned char* w_ring = smem;
    unsigned char* x_ring = w_ring + STAGES * HALVES * P_A_BYTES;
    unsigned char* s_ring = x_ring + STAGES * HALVES * X_BYTES;
    uint64_t* full = reinterpret_cast<uint64_t*>(s_ring + STAGES * SLOT_SCALE_BYTES);
    uint64_t* empty = full + STAGES;
    uint64_t* acc_full = empty + STAGES;
    uint64_t* acc_empty = acc_full + 2;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
    int* flag = reinterpret_cast<int*>(tmem_slot + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    Walk walk(s);

    if (threadIdx.x < 4) lost_tokens[threadIdx.x] = 0;
    if (threadIdx.x == 0) {
        lost_count = 0;
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&full[i], 2);
            mbar_init(&empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&acc_full[i], 1);
            mbar_init(&acc_empty[i], P_STORERS);
        }
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

    // a piece of w: halves of 128 elements, and their scales
    auto load_w = [&](int n_tile, int piece, int slot) {
        mbar_arrive_expect_tx(&full[slot], HALVES * (P_A_BYTES / 2) + W_SCALE_BYTES);   // half of what the codes take in shared memory
#pragma unroll
        for (int h = 0; h < HALVES; ++h)
            tma_load_2d(w_ring + (slot * HALVES + h) * P_A_BYTES, &w_map, &full[slot], (piece * HALVES + h) * HALF_STAGE_K, n_tile * BM);
        bulk_load(s_ring + slot * SLOT_SCALE_BYTES, s.w_scales + ((size_t)n_tile * s.w_tiles_of_a_row + piece * HALVES) * MX_TILE_BYTES, W_SCALE_BYTES, &full[slot]);
    };
    const int ahead = s.early ? min(STAGES, walk.total * PIECES) : 0;
    if (warp == 2 + P_STORERS) {
        if (elect_one())
            for (int i = 0; i < ahead; ++i) load_w(walk.n_tile_of(s, i / PIECES), walk.stage_of(s, i / PIECES) * PIECES + i % PIECES, i);
        __syncwarp();
    }
    pdl_wait();
    if (warp == 0) {
        const bool leader = elect_one();
        bool alive = true;
        int slot = 0;
        uint32_t phase = 1;
        while (alive && walk.step(s)) {
            for (int piece = walk.from * PIECES; piece < walk.to * PIECES; ++piece) {
                if (!(alive = warp_wait(&empty[slot], phase))) break;
                if (leader) {
                    mbar_arrive_expect_tx(&full[slot], HALVES * X_BYTES + X_TILES * W_SCALE_BYTES);
#pragma unroll
                    for (int h = 0; h < HALVES; ++h)
                        tma_load_2d(x_ring + (slot * HALVES + h) * X_BYTES, &x_map, &full[slot], (piece * HALVES + h) * HALF_STAGE_K, 0);
#pragma unroll
                    for (int t = 0; t < X_TILES; ++t)
                        bulk_load(s_ring + slot * SLOT_SCALE_BYTES + (1 + t) * W_SCALE_BYTES,
                                  x_scales + ((size_t)t * s.w_tiles_of_a_row + piece * HALVES) * MX_TILE_BYTES, W_SCALE_BYTES, &full[slot]);
                }
                __syncwarp();
                if (++slot == STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 2 + P_STORERS) {
        const bool leader = elect_one();
        bool alive = true;
        int slot = 0, count = 0;
        uint32_t phase = 1;
        while (alive && walk.step(s)) {
            const int n_tile = walk.n_tile;
            for (int piece = walk.from * PIECES; piece < walk.to * PIECES; ++piece, ++count) {
                if (count >= ahead) {
                    if (!(alive = warp_wait(&empty[slot], phase))) break;
                    if (leader) load_w(n_tile, piece, slot);
                    __syncwarp();
                }
                if (++slot == STAGES) slot = 0, phase ^= 1;
            }
        }
    } else if (warp == 1) {
        const bool leader = elect_one();
        bool alive = true;
        int slot = 0, round = 0;
        uint32_t phase = 0;
        for (; alive && walk.step(s); ++round) {
            const int buffer = round & 1;
            if (!(alive = warp_wait(&acc_empty[buffer], ((round >> 1) & 1) ^ 1))) break;
            tcgen05_fence_after_sync();
            const uint32_t d_tmem = tmem + buffer * ACCUMULATOR;
            for (int index = 0; index < (walk.to - walk.from) * PIECES; ++index) {
                if (!(alive = warp_wait(&full[slot], phase))) break;
                tcgen05_fence_after_sync();
                const uint64_t a_desc = umma_smem_desc_sw128(smem_u32(w_ring + slot * HALVES * P_A_BYTES));
                const uint64_t b_desc = umma_smem_desc_sw128(smem_u32(x_ring + slot * HALVES * X_BYTES));
                const uint32_t scales = smem_u32(s_ring + slot * SLOT_SCALE_BYTES);
                const uint32_t columns = tmem + SCALES_FIRST + slot * SCALE_COLUMNS;
                if (leader) {
#pragma unroll
                    for (int q = 0; q < HALVES; ++q) {                              // 128 elements of K: w, then the parts' tiles side by side
                        scales_to_tmem(columns + q * 4 * (1 + X_TILES), scales + q * MX_TILE_BYTES);
#pragma unroll
                        for (int t = 0; t < X_TILES; ++t)
                            scales_to_tmem(columns + q * 4 * (1 + X_TILES) + 4 * (1 + t), scales + (1 + t) * W_SCALE_BYTES + q * MX_TILE_BYTES);
                    }
#pragma unroll
                    for (int k = 0; k < HALVES * 4; ++k)
                        umma_mxf8f6f4(d_tmem, a_desc + (k >> 2) * (P_A_BYTES / 16) + 2 * (k & 3), b_desc + (k >> 2) * (X_BYTES / 16) + 2 * (k & 3),
                                      mxf8f6f4_idesc(BM, N_COLUMNS, k & 3), columns + (k >> 2) * 4 * (1 + X_TILES), columns + (k >> 2) * 4 * (1 + X_TILES) + 4,
                                      index > 0 || k > 0);
                    umma_commit(&empty[slot]);
                }
                __syncwarp();
                if (++slot == STAGES) slot = 0, phase ^= 1;
            }
            if (leader) umma_commit(&acc_full[buffer]);
            __syncwarp();
        }
    } else {
        int some = 0;
        for (int i = threadIdx.x - 64; i < s.M * s.depth; i += P_STORERS * 32) {
            const int count = __ldcg(s.lost + i), token = i / s.depth;
            if (count == 0) continue;
            atomicOr(&lost_tokens[(count == MX_LOST_ALL ? 2 : 0) + (token >> 5)], 1u << (token & 31));
            some = min(some + count, 4 * LOST_MOST + 1);
        }
        if (some) atomicAdd(&lost_count, some);
        asm volatile("bar.sync 1, %0;" ::"n"(P_STORERS * 32) : "memory");
        if (threadIdx.x == 64) {                    // a token is in one of the two sets
            const uint32_t all[2] = {lost_tokens[0] | lost_tokens[2], lost_tokens[1] | lost_tokens[3]};
            const bool many = lost_count > LOST_MOST * ((__popc(all[0]) + __popc(all[1]) + 15) / 16);
            for (int i = 0; i < 2; ++i) {
                if (many) lost_tokens[2 + i] = all[i];
                lost_tokens[i] = all[i] & ~lost_tokens[2 + i];
            }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(P_STORERS * 32) : "memory");
        for (int round = 0; walk.step(s); ++round) {
            const int buffer = round & 1;
            if (!warp_wait(&acc_full[buffer], (round >> 1) & 1) && !s.scratch) break;      // of shared tiles the others meet this warp at barriers
            tcgen05_fence_after_sync();
            store_accumulator<TOKENS, P_STORERS, Out, true>(tmem + buffer * ACCUMULATOR, out, s, walk, warp - 2, false, flag, nullptr, lost_tokens);
            tcgen05_fence_before_sync();
            __syncwarp();
            if (lane == 0) mbar_arrive(&acc_empty[buffer]);
        }
    }
    __syncwarp();
    tcgen05_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tcgen05_fence_after_sync();
        tmem_dealloc(tmem, TMEM_COLUMNS);
    }
    if (lost_tokens[2] | lost_tokens[3]) wide_products<P_THREADS / 32>(x, out, s, lost_tokens[2], lost_tokens[3], reinterpret_cast<float*>(smem));
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

// Tiles and units of a product; false where they are too many, or more CTAs are asked for than have work.
template <int TOKENS> bool lay_out(Shapes& s, int ctas) {
    s.depth = (s.K + STAGE_K - 1) / STAGE_K;
    s.token_tiles = (s.M + TOKENS - 1) / TOKENS;
    const long long units = (long long)((s.N + BM - 1) / BM) * s.token_tiles * s.depth;
    if (units > 0x7FFFFFFF) return false;
    s.units = (int)units;
    return ctas <= (s.scratch ? s.units : s.units / s.depth);
}

template <typename... KernelArgs, typename... Args>
int launch_run(void (*kernel)(KernelArgs...), PerDevice& configured, int threads, int ctas, size_t smem, void* stream, Args... args) {
    if (!configured.get()) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        if (e != cudaSuccess) return (int)e;
        configured.set(1);
    }
    return mrs_launch(kernel, dim3(ctas), dim3(threads), smem, (cudaStream_t)stream, args...);
}

template <int TOKENS, typename Out>
int launch_weights(const void* x, const void* x_halfs, void* out, Shapes s, int ctas, void* stream) {
    CUtensorMap w_map, x_map, halfs_map;
    int code = make_map(&w_map, s.w_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K / 2, s.K / 2, s.N, 128, BM);
    if (!code) code = make_map(&x_map, x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (long long)s.K * 2, s.K, s.M, PIECE_K, TOKENS);
    halfs_map = x_map;
    if (!code && s.x_factors) code = make_map(&halfs_map, x_halfs, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, (long long)s.K * 2, s.K, s.M, PIECE_K, TOKENS);
    if (code) return code;
    static PerDevice configured;
    if (!lay_out<TOKENS>(s, ctas)) return MRS_BAD_ARGUMENT;
    const int stages = s.scratch ? (int)(((long long)s.units + ctas - 1) / ctas) : (s.units / s.depth + ctas - 1) / ctas * s.depth;
    s.lost_most = most_lost(TOKENS, s.token_tiles, stages, s.depth);
    return launch_run(weights_kernel<TOKENS, Out>, configured, W_THREADS, ctas, weights_smem<TOKENS>(), stream, w_map, x_map, halfs_map, s.w_scales, (Out*)out, s);
}
template <int TOKENS, typename Out>
int launch_both(const void* x_codes, const void* x_scales, void* out, Shapes s, int ctas, void* stream) {
    CUtensorMap w_map, x_map;
    int code = make_map(&w_map, s.w_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K / 2, s.K / 2, s.N, 128, BM);
    if (!code) code = make_map(&x_map, x_codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K / 2, s.K / 2, s.M, 128, TOKENS);
    if (code) return code;
    static PerDevice configured;
    s.x_row_tiles = (s.M + 127) / 128;
    if (!lay_out<TOKENS>(s, ctas)) return MRS_BAD_ARGUMENT;
    return launch_run(both_kernel<TOKENS, Out>, configured, B_THREADS, ctas, both_smem<TOKENS>(), stream, w_map, x_map, s.w_scales,
                      (const uint8_t*)x_scales, (Out*)out, s);
}

template <int TOKENS, typename Out>
int launch_parts(const void* x, const void* parts, const void* x_scales, void* out, Shapes s, int ctas, void* stream) {
    CUtensorMap w_map, x_map;
    int code = make_map(&w_map, s.w_codes, CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, s.K / 2, s.K, s.N, HALF_STAGE_K, BM);
    if (!code) code = make_map(&x_map, parts, CU_TENSOR_MAP_DATA_TYPE_UINT8, s.K, s.K, 3 * TOKENS, HALF_STAGE_K, 3 * TOKENS);
    if (code) return code;
    static PerDevice configured;
    if (!lay_out<TOKENS>(s, ctas)) return MRS_BAD_ARGUMENT;
    return launch_run(parts_kernel<TOKENS, Out>, configured, P_THREADS, ctas, parts_smem<TOKENS>(), stream, w_map, x_map, (const bf16*)x, (const uint8_t*)x_scales,
                      (Out*)out, s);
}

// What a product needs beside its operands, in one buffer: what x becomes and what belongs to it, elements that are lost on the way, and, where
// tiles are shared, sums and counts.  All offsets are multiples of 16 bytes.
enum Form { PARTS = 0, WEIGHTS = 1, BOTH = 2 };
struct Work {
    long long side = 0, lost = 0, scratch = 0, arrived = 0, tiles = 0, bytes = 0;
    Work(int form, long long M, long long N, long long K, int tokens, int ctas, int shared) {
        const long long depth = (K + STAGE_K - 1) / STAGE_K;
        side = form == PARTS ? 3 * tokens * K : form == WEIGHTS ? 2 * M * K : M * (K / 2);
        lost = side + (form == PARTS ? (3 * tokens + 127) / 128 * SCALE_BYTES * depth : form == WEIGHTS ? (M + 3) / 4 * 16 : mrs_mxfp4_scale_bytes(M, K));
        scratch = lost + (form == BOTH ? 0 : (M * depth + 3) / 4 * 16 + M * depth * MX_LOST * 4);
        arrived = scratch + (shared ? 2ll * ctas * tokens * BM * 4 : 0);
        tiles = shared ? (N + BM - 1) / BM * ((M + tokens - 1) / tokens) : 0;
        bytes = arrived + 4 * tiles;
    }
};

}  // namespace

// Bytes of the buffer for a product of `form` (0: x in parts, 1: as halfs or as it is, 2: in 4 bits).
MRS_EXPORT long long mrs_mxfp4_work_bytes(int form, int M, int N, int K, int tokens, int ctas, int shared) { return Work(form, M, N, K, tokens, ctas, shared).bytes; }

// out [M, N] bfloat16 or float32 (`out_f32`) = x [M, K] bfloat16 . w [N, K]^T, w as in mxfp4.cuh.  `tokens` of a tile: 16, 32, 64, 128 or 192, below
// 128 only if they are all; with parts (K a multiple of 128) at most 64.  `ctas`: at most the GPU's SMs, and the tiles or, if they are `shared`,
// cut into equal runs, the stages of 256 elements of K of all of them.  `fits`: w's blocks other than zeros have scales of 2^(w_exponent - 23) to
// 2^(w_exponent + 13), so that halfs hold them.  `early`: nothing that still runs when the product starts writes w.
MRS_EXPORT int mrs_mxfp4_rows(int form, const void* x, const void* codes, const void* scales, void* out, int out_f32, int M, int N, int K, int tokens, int ctas,
                              int shared, int fits, int w_exponent, int early, void* work, void* stream) {
    if (M == 0 || N == 0) return 0;
    if (M < 0 || N < 0 || K <= 0 || K % MX_BLOCK || K > (1 << 30) || !x || !codes || !scales || !out || !work || ctas < 1 || (tokens < 128 && M > tokens) ||
        (tokens != 16 && tokens != 32 && tokens != 64 && tokens != 128 && tokens != 192) ||
        (((uintptr_t)x | (uintptr_t)codes | (uintptr_t)scales | (uintptr_t)work) & 15) || ((uintptr_t)out & (out_f32 ? 3 : 1)) || form < PARTS || form > BOTH ||
        (form == PARTS && (K % HALF_STAGE_K || ((uintptr_t)codes & 31) || tokens > 64)))
        return MRS_BAD_ARGUMENT;
    const Work at(form, M, N, K, tokens, ctas, shared);
    if (at.tiles > 0x7FFFFFFF) return MRS_BAD_ARGUMENT;
    char* base = (char*)work;
    void *side = base + at.side, *lost = base + at.lost, *scratch = shared ? base + at.scratch : nullptr, *arrived = shared ? base + at.arrived : nullptr;
    int code;
    if (form == BOTH) code = mrs_mxfp4_quantise(1, x, base, side, M, K, arrived, (int)at.tiles, stream);
    else if (form == PARTS) code = mrs_mxfp4_rows_to_parts(x, base, side, lost, M, K, tokens, arrived, (int)at.tiles, stream);
    else if (fits) code = mrs_mxfp4_rows_to_halfs(x, base, side, lost, M, K, arrived, (int)at.tiles, stream);
    else code = mrs_mxfp4_clear(arrived, (int)at.tiles, stream);
    if (code) return code;
    Shapes s = {};
    s.M = M, s.N = N, s.K = K, s.early = early, s.w_tiles_of_a_row = mx_tiles_of_a_row(K), s.scratch = (float*)scratch, s.arrived = (int*)arrived;
    s.w_codes = (const uint8_t*)codes, s.w_scales = (const uint8_t*)scales;
    if (form != BOTH) s.lost = (const int*)lost;
    if (form == WEIGHTS && fits) s.x_factors = (const int*)side, s.w_exponent = w_exponent;
#define MRS_TOKENS(T, LAUNCH, ...) if (tokens == T) return out_f32 ? LAUNCH<T, float>(__VA_ARGS__, out, s, ctas, stream) : LAUNCH<T, bf16>(__VA_ARGS__, out, s, ctas, stream)
    if (form == PARTS) {
        MRS_TOKENS(16, launch_parts, x, base, side);
        MRS_TOKENS(32, launch_parts, x, base, side);
        MRS_TOKENS(64, launch_parts, x, base, side);
    } else if (form == WEIGHTS) {
        MRS_TOKENS(16, launch_weights, x, base);
        MRS_TOKENS(32, launch_weights, x, base);
        MRS_TOKENS(64, launch_weights, x, base);
        MRS_TOKENS(128, launch_weights, x, base);
        MRS_TOKENS(192, launch_weights, x, base);
    } else {
        MRS_TOKENS(16, launch_both, base, side);
        MRS_TOKENS(32, launch_both, base, side);
        MRS_TOKENS(64, launch_both, base, side);
        MRS_TOKENS(128, launch_both, base, side);
        MRS_TOKENS(192, launch_both, base, side);
    }
#undef MRS_TOKENS
    return MRS_BAD_ARGUMENT;
}

MRS_EXPORT int mrs_mxfp4_take_error(unsigned int* word) { return mrs_take_error_word(word); }
// Mirrors the error word into a word of pinned host memory from now on.
MRS_EXPORT int mrs_mxfp4_mirror_errors(unsigned int* host_word) { return mrs_set_error_mirror(host_word); }

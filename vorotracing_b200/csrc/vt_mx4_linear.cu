// vt_mx4_linear.cu -- y = act(q4(x) w4^T + b), both matrices in 4-bit microscaled blocks (vt_mx.cuh).
//
// The product runs on the tensor cores' block-scaled 4-bit path: 128 rows of x by TN outputs a
// tile, 256 steps of k a stage.  The weight's codes come by TMA into the 128-byte swizzle; four
// warps bring the scales of a stage into the order in which they are copied to tensor memory; one
// thread issues copies and products; four warps take finished accumulators out of tensor memory,
// add the bias, apply the activation and round once.
//
// x is rounded to 4 bits inside the same kernel while one tile spans all outputs (linear4_kernel): TMA
// brings x in as it is, deep enough ahead to keep HBM busy (112 to 128 KB), and eight warps round
// it, a lane a block of 32 columns, into the operand's place.  x is then read from HBM once and
// nothing of its 4-bit form is written.
// With more outputs the same rows would be rounded again for every tile of outputs, so a pass of
// its own writes codes and scales first, 17/32 byte a value, and pairs of CTAs multiply
// (pair4_kernel).
//
// Too few tiles to occupy the GPU (few rows, as in serving one token at a time) go the other way
// round (few_kernel): 128 outputs are the product's rows and up to 128 rows of x its columns, k is
// split over a cluster of up to 8 CTAs, each CTA rounds its part of x itself, and the parts of the
// sums meet in distributed shared memory, where they are added in the order of k.  One launch; the
// weight is spread over as many SMs as there are.
//
// Measured (bfloat16): 1088640 rows, 192 -> 64, SiLU: 115 to 123 us, 4.5 to 4.9 TB/s (floor 86 us); no unit is full (DRAM 51 %,
// issue 46 %, tensor pipe 3 % of their peaks on 500000 rows), so latency is what is left, and what of it was not
// found.  With x read by the rounding warps themselves 597 us.  One row, 4096 -> 4096: 12.5 us a call, of which
// the host takes 10; 77 rows, 1000 -> 333: 12.6 us (33 us in the large tiles).
// 4096 rows, 8192 -> 8192: 157 to 162 us, 3.4 PFLOP/s (floor 83 us), of which the pass that writes x's codes and both scales
// takes a fifth.  277867 rows, 91 -> 195: 138 us, of which copying x to whole words 24.
#include "vt_mx_rows.cuh"

namespace vt {

constexpr uint32_t L4_ROWS = 128, L4_K = 256;

template <int TN> struct L4 {
    static constexpr uint32_t A_BYTES = L4_ROWS * 128u, B_BYTES = TN * 128u;
    static constexpr uint32_t B_PARTS = TN > 128 ? 2 : 1;  // groups of 128 rows of scales
    static constexpr uint32_t SF_BYTES = (1u + B_PARTS) * 1024u;
    static constexpr uint32_t STAGE = A_BYTES + B_BYTES + SF_BYTES;
    static constexpr uint32_t STAGES = TN == 256 ? 2 : 3;
    static constexpr uint32_t X_BYTES = L4_ROWS * 128u, X_STAGES = TN == 64 ? 8 : 7;  // 64 columns of x each
    // two accumulators when they leave room for the scales
    static constexpr uint32_t ACCS = TN == 256 ? 1 : 2;
    // Scales in tensor memory have a place for every stage: nothing says that a copy waits for the products
    // before it that still read what it overwrites.
    static constexpr uint32_t SF_AT = ACCS * TN, SF_COLS = 8u + 8u * B_PARTS;
    static constexpr uint32_t TMEM_USED = SF_AT + STAGES * SF_COLS, TMEM = TMEM_USED <= 256 ? 256 : 512;
    // The warps that bring scales take stages in turn.  A parity tells a phase from the one before it only, and
    // what a warp knows of a stage is from its last turn: there may be no more turns than stages.
    static constexpr uint32_t SCALE_WARPS = 4, TURNS = STAGES < SCALE_WARPS ? STAGES : SCALE_WARPS, QUANT_WARPS = 8;
    // warps: 0 TMA, 1 products, 2 TMA of x, 3 none, 4..7 results, 8..11 scales, 12.. x to 4 bits
    static constexpr uint32_t THREADS = 32u * (8u + SCALE_WARPS + QUANT_WARPS);
    static constexpr uint32_t FULL_COUNT = 1u + 1u + QUANT_WARPS;
    struct Ctrl {
        uint64_t full[STAGES], empty[STAGES], acc_full[ACCS], acc_empty[ACCS], x_full[X_STAGES], x_empty[X_STAGES], failed;
        uint32_t tmem;
        tc::Fail fail;
        alignas(8) float bias[TN];
        uint32_t turn[4][TURN_WORDS];
    };
    static constexpr uint32_t X_AT = STAGES * STAGE, CTRL_AT = X_AT + X_STAGES * X_BYTES, SMEM = CTRL_AT + sizeof(Ctrl);
    static_assert(SMEM <= 232448 && TMEM_USED <= 512, "does not fit an SM");
};

struct L4Args {
    uint64_t rows;
    uint32_t cols, outs, blocks, chunks, last_steps, row_tiles, out_tiles;  // last_steps: of 64, in a row's last chunk
    const uint8_t *w_exps;
    const void *bias;
    void *y;
    uint32_t *err;
    bool y_wide;
};

// The scales of 8 blocks of a row, zeros (which multiply zero codes) behind its end.
__device__ __forceinline__ uint2 load_scales(const uint8_t *exps, uint64_t row, uint32_t blocks, uint32_t b0)
{
    const uint8_t *p = exps + row * blocks + b0;
    if (b0 + 8u <= blocks && (reinterpret_cast<uintptr_t>(p) & 7u) == 0) return __ldg(reinterpret_cast<const uint2 *>(p));
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i)
        if (b0 + i < blocks) w[i / 4] |= (uint32_t)__ldg(p + i) << (i % 4 * 8);
    return make_uint2(w[0], w[1]);
}
// Place of a row's scales in a stage: 16 bytes for each of 32 rows, a word a group of 32.
__device__ __forceinline__ uint32_t scale_place(uint32_t row) { return (row >> 7) * 1024u + (row & 31u) * 16u + ((row >> 5) & 3u) * 4u; }

__device__ __forceinline__ void store_scales(uint8_t *sf, uint32_t row, uint2 e)
{
    *reinterpret_cast<uint32_t *>(sf + scale_place(row)) = e.x;
    *reinterpret_cast<uint32_t *>(sf + scale_place(row) + 512u) = e.y;
}

// A block of 32 16-bit numbers to 4 bits: codes and exponent byte
template <typename T> __device__ __forceinline__ uint4 block_codes(const uint4 *w, uint32_t &E)
{
    uint32_t top = 0;
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
        top = __vmaxu2(top, w[u].x & 0x7fff7fffu);
        top = __vmaxu2(top, w[u].y & 0x7fff7fffu);
        top = __vmaxu2(top, w[u].z & 0x7fff7fffu);
        top = __vmaxu2(top, w[u].w & 0x7fff7fffu);
    }
    E = mx4_exponent(top_of_pair<T>(top));
    const f32x2 inv = both(E == 255u ? 0.0f : mx4_inverse(E));
    uint32_t codes[4];
#pragma unroll
    for (uint32_t u = 0; u < 4; ++u) {
        const uint32_t in[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
        f32x2 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 f = unpack2<T>(in[i]);
            v[i] = mul2(pair(f.x, f.y), inv);
        }
        codes[u] = mx4_word(v);
    }
    return make_uint4(codes[0], codes[1], codes[2], codes[3]);
}

// Columns col..col + 31 of a warp's 32 rows of y, a lane a row, from sums and bias.  y: the warp's first row, of which
// `rows` of the 32 exist.
template <typename T, int ACT>
__device__ __forceinline__ void store_results(T *y, uint32_t rows, uint32_t col, uint32_t cols, bool wide, const uint32_t *v, const float *bias,
                                              uint32_t *turn)
{
    uint32_t w[16];
#pragma unroll
    for (uint32_t i = 0; i < 16; ++i)
        w[i] = pack2<T>(act_value2<ACT>(add2(pair(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])),
                                             *reinterpret_cast<const f32x2 *>(bias + 2 * i))));
    const uint32_t lane = threadIdx.x & 31u;
    if (!wide) store_turned<T>(y, rows, col, cols, w, turn);
    else if (lane < rows) store_row32<T>(y + (uint64_t)lane * cols, col, cols, w);
}
// Rows of 32 from `row` on
__device__ __forceinline__ uint32_t rows_left(uint64_t row, uint64_t rows)
{
    return row >= rows ? 0u : rows - row < 32u ? (uint32_t)(rows - row) : 32u;
}

// A stage's scales to tensor memory and its products, by one lane: `steps` of 64 steps of k, 4 but
// for a row's last stage.  Descriptors of the operands at the stage's start; the scales of A
// (1 group of 128 rows) and of B (PARTS groups) at sf, going to sfa and sfb.
template <int PARTS, bool PAIR = false>
__device__ __forceinline__ void stage_products(uint32_t d, uint64_t a, uint64_t b, uint64_t sf, uint32_t sfa, uint32_t sfb, uint32_t id0,
                                               uint32_t id1, uint32_t steps, bool accumulate)
{
    const auto copy = [](uint32_t to, uint64_t from) {
        if (PAIR) tc::tmem_copy_scales_pair(to, from); else tc::tmem_copy_scales(to, from);
    };
#pragma unroll
    for (uint32_t g = 0; g < 2; ++g)
        if (2u * g < steps) {
            copy(sfa + g * 4u, sf + g * 32u);
#pragma unroll
            for (uint32_t p = 0; p < PARTS; ++p) copy(sfb + (g * PARTS + p) * 4u, sf + 64u + p * 64u + g * 32u);
        }
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k)
        if (k < steps) {
            const uint32_t id = k & 1u ? id1 : id0, ta = sfa + (k >> 1) * 4u, tb = sfb + (k >> 1) * PARTS * 4u;
            if (PAIR) tc::mma_mxf4_pair(d, a + k * 2u, b + k * 2u, id, ta, tb, accumulate || k != 0);
            else tc::mma_mxf4(d, a + k * 2u, b + k * 2u, id, ta, tb, accumulate || k != 0);
        }
}

template <typename T, int ACT, int TN>
__global__ void __launch_bounds__(L4<TN>::THREADS, 1)
    linear4_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map, const L4Args a)
{
    using P = L4<TN>;
    extern __shared__ __align__(1024) uint8_t smem[];
    typename P::Ctrl &s = *reinterpret_cast<typename P::Ctrl *>(smem + P::CTRL_AT);
    const uint32_t warp = tc::warp_number(), lane = threadIdx.x % 32u;
    const uint32_t tiles = a.row_tiles;  // one tile spans all outputs
    tc::Fail *const fail = &s.fail;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < P::STAGES; ++i) {
            tc::mbar_init(&s.full[i], P::FULL_COUNT);
            tc::mbar_init(&s.empty[i], 1);
        }
        for (uint32_t i = 0; i < P::ACCS; ++i) {
            tc::mbar_init(&s.acc_full[i], 1);
            tc::mbar_init(&s.acc_empty[i], 4);
        }
        for (uint32_t i = 0; i < P::X_STAGES; ++i) {
            tc::mbar_init(&s.x_full[i], 1);
            tc::mbar_init(&s.x_empty[i], P::QUANT_WARPS);
        }
        tc::mbar_init(&s.failed, 1);
        s.fail.failed = 0;
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&w_map);
        tc::tma_prefetch_map(&x_map);
    }
    if (warp == 1) tc::tmem_alloc<P::TMEM>(&s.tmem);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        if (lane == 0) {  // TMA
            tc::Ring r;
            bool ok = true;
            for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
                for (uint32_t c = 0; c < a.chunks; ++c) {
                    ok = tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err);
                    if (!ok) break;
                    uint8_t *st = smem + r.i * P::STAGE;
                    tc::mbar_arrive_tx(&s.full[r.i], P::B_BYTES);
                    tc::tma_load_2d(st + P::A_BYTES, &w_map, (int)(c * 128u), 0, &s.full[r.i]);
                    r.next(P::STAGES);
                }
            }
            // A stage's barrier also waits for other warps, so a failed launch cannot use it to
            // see that its copies are in: it waits for them by time, far longer than a copy takes.
            if (s.fail.failed) tc::outlast_copies();
        }
    } else if (warp == 1) {  // scales to tensor memory, products
        const uint32_t base = tc::smem_u32(smem);
        constexpr uint32_t ID0 = tc::idesc_mxf4(128, TN, 0), ID1 = tc::idesc_mxf4(128, TN, 1);
        const bool mine = tc::elect();
        tc::Ring r, acc;
        bool ok = true;
        for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            ok = __all_sync(~0u, tc::mbar_wait(&s.acc_empty[acc.i], acc.phase ^ 1u, fail, a.err));
            if (!ok) break;
            tc::fence_after();
            for (uint32_t c = 0; c < a.chunks; ++c) {
                ok = __all_sync(~0u, tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
                if (!ok) break;
                tc::fence_after();
                const uint32_t st = base + r.i * P::STAGE, sfa = tmem + P::SF_AT + r.i * P::SF_COLS, sfb = sfa + 8u;
                if (mine) {
                    stage_products<P::B_PARTS>(tmem + acc.i * TN, tc::smem_desc(st, 16, 1024), tc::smem_desc(st + P::A_BYTES, 16, 1024),
                                               tc::scale_desc(st + P::A_BYTES + P::B_BYTES), sfa, sfb, ID0, ID1,
                                               c + 1u == a.chunks ? a.last_steps : 4u, c != 0);
                    tc::commit(&s.empty[r.i]);
                    if (c + 1u == a.chunks) tc::commit(&s.acc_full[acc.i]);
                }
                __syncwarp();
                r.next(P::STAGES);
            }
            acc.next(P::ACCS);
        }
        if (!ok) {  // leave no product in flight
            if (mine) tc::commit(&s.failed);
            tc::mbar_wait_slow(&s.failed, 0, fail, a.err, true);
        }
    } else if (warp >= 4 && warp < 8) {  // results
        const uint32_t quad = warp % 4u, in_tile = quad * 32u + lane;
        for (uint32_t i = in_tile; i < TN; i += 128u) s.bias[i] = a.bias && i < a.outs ? to_f32<T>(__ldg((const T *)a.bias + i)) : 0.0f;
        asm volatile("bar.sync 1, 128;" ::: "memory");
        tc::Ring acc;
        for (uint32_t t = blockIdx.x; t < tiles; t += gridDim.x) {
            const uint64_t row = (uint64_t)t * L4_ROWS + quad * 32u;  // the warp's first
            const bool ok = tc::mbar_wait(&s.acc_full[acc.i], acc.phase, fail, a.err);
            if (!__all_sync(~0u, ok)) break;
            tc::fence_after();
#pragma unroll 1
            for (uint32_t n0 = 0; n0 < TN; n0 += 32u) {
                uint32_t v[32];
                tc::tmem_load32(tmem + acc.i * TN + (quad * 32u << 16) + n0, v);
                if (n0 + 32u == TN) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s.acc_empty[acc.i]);
                }
                store_results<T, ACT>((T *)a.y + row * a.outs, rows_left(row, a.rows), n0, a.outs, a.y_wide, v, s.bias + n0, s.turn[quad]);
            }
            acc.next(P::ACCS);
        }
    } else if (warp >= 8 && warp < 12) {  // scales: the four warps take stages in turn, which hides the loads' latency
        constexpr int ROWS = TN / 32;
        tc::Ring r;
        bool ok = warp - 8u < P::TURNS;
        uint32_t turn = warp - 8u;  // stages until this warp's
        for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            for (uint32_t c = 0; c < a.chunks; ++c, r.next(P::STAGES), turn = turn ? turn - 1u : P::TURNS - 1u) {
                if (turn != 0) continue;
                uint2 e[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; ++i)
                    e[i] = lane + i * 32u < a.outs ? load_scales(a.w_exps, lane + i * 32u, a.blocks, c * 8u) : make_uint2(0, 0);
                ok = __all_sync(~0u, tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err));
                if (!ok) break;
                uint8_t *sf = smem + r.i * P::STAGE + P::A_BYTES + P::B_BYTES + 1024u;
#pragma unroll
                for (int i = 0; i < ROWS; ++i) store_scales(sf, i * 32u + lane, e[i]);
                tc::fence_async_shared();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&s.full[r.i]);
            }
        }
    } else if (warp == 2) {
        if (lane == 0) {  // TMA of x, 64 columns at a time
            tc::Ring r;
            uint32_t issued = 0;
            bool ok = true;
            for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x)
                for (uint32_t col = 0; col < a.cols; col += 64u) {
                    ok = tc::mbar_wait(&s.x_empty[r.i], r.phase ^ 1u, fail, a.err);
                    if (!ok) break;
                    tc::mbar_arrive_tx(&s.x_full[r.i], P::X_BYTES);
                    tc::tma_load_2d(smem + P::X_AT + r.i * P::X_BYTES, &x_map, (int)col, (int)(t * L4_ROWS),
                                    &s.x_full[r.i]);
                    ++issued;
                    r.next(P::X_STAGES);
                }
            if (s.fail.failed)  // leave no copy in flight
                for (uint32_t i = 0; i < P::X_STAGES && i < issued; ++i)
                    tc::mbar_wait_slow(&s.x_full[i], ((issued - 1 - i) / P::X_STAGES) & 1u, fail, a.err, true);
        }
    } else if (warp >= 12) {  // x to 4 bits: a lane has a row, each half of the warps one of a chunk's two blocks
        const uint32_t row = warp % 4u * 32u + lane, part = (warp - 12u) / 4u;
        tc::Ring r, x;
        bool ok = true;
        for (uint32_t t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
            for (uint32_t c = 0; c < a.chunks && ok; ++c) {
                ok = __all_sync(~0u, tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err));
                if (!ok) break;
                uint8_t *st = smem + r.i * P::STAGE, *sf = st + P::A_BYTES + P::B_BYTES + scale_place(row);
                const uint32_t steps = min(4u, (a.cols - c * L4_K + 63u) / 64u);
                for (uint32_t k = 0; k < steps; ++k) {
                    ok = __all_sync(~0u, tc::mbar_wait(&s.x_full[x.i], x.phase, fail, a.err));
                    if (!ok) break;
                    const uint8_t *from = smem + P::X_AT + x.i * P::X_BYTES + row * 128u;
                    uint4 w[4];
#pragma unroll
                    for (uint32_t u = 0; u < 4; ++u) w[u] = *reinterpret_cast<const uint4 *>(from + (((part * 4u + u) ^ (row & 7u)) << 4));
                    uint32_t E;
                    const uint4 codes = block_codes<T>(w, E);
                    const uint32_t block = k * 2u + part;
                    *reinterpret_cast<uint4 *>(st + row * 128u + ((block ^ (row & 7u)) << 4)) = codes;
                    sf[(block >> 2) * 512u + (block & 3u)] = (uint8_t)E;
                    // x's place is free once its values have arrived in registers, which the stores above, made
                    // of them, have seen; an arrival right behind the loads may overtake them
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s.x_empty[x.i]);
                    x.next(P::X_STAGES);
                }
                tc::fence_async_shared();
                __syncwarp();
                if (lane == 0) tc::mbar_arrive(&s.full[r.i]);
                r.next(P::STAGES);
            }
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 1) tc::tmem_free<P::TMEM>(tmem);
}

// ---- many outputs ----
//
// Both operands come in 4 bits, their scales in the order of the stages: for 128 rows and 256 columns 1 KB as it
// is copied to tensor memory, so that TMA brings everything in.  (Warps that gathered the scales from their rows
// kept up with half the speed: each stage takes 8 bytes of 352 rows.)  stage4_kernel writes them, and x's codes.
// A pair of CTAs shares a tile of 256 rows by 224 outputs: each stages its 128 rows of x and half of the
// outputs' weights, so a byte of shared memory serves twice the products of a CTA alone.  224 outputs leave
// room in tensor memory for two accumulators and two places of scales.
// Measured: 4096 x 8192 x 8192 in 157 to 162 us, 3.4 PFLOP/s, twice what the bfloat16 library product reaches here
// (one CTA a tile: 182 us).  Under the counters stage4_kernel takes 33 us, at two thirds of its issue slots (its bytes
// would take 13), and pair4_kernel 116 us: 757 cycles a stage, of which the tensor cores are busy 59 % with its 448 cycles of
// products.  The rest is waits, of which kind was not found: more places for scales, in tiles of 192 outputs, made it
// slower (179 us).

constexpr uint32_t PAIR_N = 224, PAIR_A = 16384, PAIR_B = PAIR_N / 2 * 128, PAIR_STAGE = PAIR_A + PAIR_B + 3072, PAIR_STAGES = 6,
                   PAIR_THREADS = 256, PAIR_SF_AT = 2 * PAIR_N, PAIR_SF_COLS = 24;
struct PairCtrl {
    uint64_t full[PAIR_STAGES], empty[PAIR_STAGES], acc_full[2], acc_empty[2], failed;
    uint32_t tmem;
    tc::Fail fail;
    alignas(8) float bias[PAIR_N];
    uint32_t turn[4][TURN_WORDS];
};
constexpr uint32_t PAIR_SMEM = PAIR_STAGES * PAIR_STAGE + sizeof(PairCtrl);
static_assert(PAIR_SMEM <= 232448 && PAIR_SF_AT + 2 * PAIR_SF_COLS <= 512, "does not fit an SM");

// Workspace of a call: x's codes, x's scales in order (1 KB for 128 rows and a chunk), w's (2 KB for 224 outputs).
struct PairPlan {
    uint32_t row_tiles, out_tiles, chunks;  // tiles of 256 rows and of 224 outputs
    uint64_t x_scales_at, w_scales_at, bytes;
};
static PairPlan pair_plan(uint64_t rows, uint32_t cols, uint32_t outs)
{
    PairPlan p;
    p.row_tiles = (uint32_t)((rows + 255u) / 256u);
    p.out_tiles = (outs + PAIR_N - 1u) / PAIR_N;
    p.chunks = (cols + L4_K - 1u) / L4_K;
    p.x_scales_at = align_up(rows * mx_blocks(cols) * 16u, 1024);
    p.w_scales_at = p.x_scales_at + (uint64_t)p.row_tiles * 2u * p.chunks * 1024u;
    p.bytes = p.w_scales_at + (uint64_t)p.out_tiles * p.chunks * 2048u;
    return p;
}

// x (rows, cols) to 4 bits, four lanes a block; scales of x and of the weight in order.  Places behind the
// operands' rows and columns get zeros, which multiply zero codes.
template <typename T>
__global__ void __launch_bounds__(256) stage4_kernel(const T *__restrict__ x, uint64_t x_stride, uint64_t rows, uint32_t cols, uint32_t blocks,
                                                     bool vec, uint32_t chunks, uint64_t x_items, uint32_t *__restrict__ codes,
                                                     uint8_t *__restrict__ x_scales, const uint8_t *__restrict__ w_exps, uint32_t outs,
                                                     uint64_t w_items, uint32_t *__restrict__ w_scales)
{
    const uint64_t step = (uint64_t)gridDim.x * 256u, start = (uint64_t)blockIdx.x * 256u + threadIdx.x;
    const uint32_t per_row = chunks * 32u;  // lanes of a row, its padding included
    for (uint64_t t = start; t < x_items; t += step) {
        const uint64_t row = t >> 32 ? t / per_row : (uint32_t)t / per_row;
        const uint32_t in_row = (uint32_t)(t - row * per_row), block = in_row >> 2, col = in_row * 8u;
        Vec8<T> w;
        w.zero();
        if (row < rows && col < cols) {
            const T *p = x + row * x_stride + col;
            if (vec) w.load(p);
            else
                for (uint32_t i = 0; i < 8u && col + i < cols; ++i) reinterpret_cast<T *>(w.w)[i] = p[i];
        }
        float v[8];
        w.unpack(v);
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, __float_as_uint(v[i]) & 0x7fffffffu);
        const uint32_t lanes = 0xfu << (threadIdx.x & 28u);
        top = max(top, __shfl_xor_sync(lanes, top, 1));
        top = max(top, __shfl_xor_sync(lanes, top, 2));
        const uint32_t E = mx4_exponent(top);
        const f32x2 inv = both(mx4_inverse(E == 255u ? 1u : E));
        const bool in = row < rows && block < blocks;
        if (in) {
            f32x2 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) q[i] = mul2(pair(v[2 * i], v[2 * i + 1]), inv);
            codes[(row * blocks + block) * 4u + (in_row & 3u)] = E == 255u ? 0u : mx4_word(q);
        }
        if ((in_row & 3u) == 0)
            x_scales[((row >> 7) * chunks + (block >> 3)) * 1024u + (block >> 2 & 1u) * 512u + scale_place((uint32_t)row & 127u) + (block & 3u)] =
                in ? (uint8_t)E : 0;
    }
    for (uint64_t t = start; t < w_items; t += step) {  // a word: 4 blocks of an output
        const uint32_t slot = (uint32_t)t & 255u, half = (uint32_t)(t >> 8) & 1u;
        const uint64_t at = t >> 9;  // tile, chunk
        const uint32_t tile = (uint32_t)(at / chunks), c = (uint32_t)(at % chunks), out = tile * PAIR_N + slot, b0 = c * 8u + half * 4u;
        uint32_t w = 0;
        if (slot < PAIR_N && out < outs)
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i)
                if (b0 + i < blocks) w |= (uint32_t)__ldg(w_exps + (uint64_t)out * blocks + b0 + i) << (8u * i);
        w_scales[at * 512u + (slot >> 7) * 256u + half * 128u + (slot & 31u) * 4u + (slot >> 5 & 3u)] = w;
    }
}

template <typename T, int ACT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(PAIR_THREADS, 1)
    pair4_kernel(const __grid_constant__ CUtensorMap x_map, const __grid_constant__ CUtensorMap w_map,
                 const __grid_constant__ CUtensorMap x_scale_map, const __grid_constant__ CUtensorMap w_scale_map, const L4Args a)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    PairCtrl &s = *reinterpret_cast<PairCtrl *>(smem + PAIR_STAGES * PAIR_STAGE);
    const uint32_t warp = tc::warp_number(), lane = threadIdx.x % 32u, rank = tc::cluster_rank();
    const uint32_t tiles = a.row_tiles * a.out_tiles, first = blockIdx.x / 2u, step = gridDim.x / 2u;
    tc::Fail *const fail = &s.fail;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < PAIR_STAGES; ++i) {
            tc::mbar_init(&s.full[i], 1);  // the leader's counts the bytes of both CTAs
            tc::mbar_init(&s.empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            tc::mbar_init(&s.acc_full[i], 1);
            tc::mbar_init(&s.acc_empty[i], 8);
        }
        tc::mbar_init(&s.failed, 1);
        s.fail.failed = 0;
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&x_map);
        tc::tma_prefetch_map(&w_map);
        tc::tma_prefetch_map(&x_scale_map);
        tc::tma_prefetch_map(&w_scale_map);
    }
    if (warp == 1) tc::tmem_alloc_pair<512>(&s.tmem);
    tc::fence_before();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        if (lane == 0) {  // TMA
            tc::Ring r;
            bool ok = true;
            for (uint32_t t = first; t < tiles && ok; t += step) {
                const int row0 = (int)(t / a.out_tiles * 256u + rank * 128u), out0 = (int)(t % a.out_tiles * PAIR_N + rank * (PAIR_N / 2u));
                const uint32_t x_scales = (t / a.out_tiles * 2u + rank) * a.chunks * 8u, w_scales = t % a.out_tiles * a.chunks * 16u;
                for (uint32_t c = 0; c < a.chunks; ++c) {
                    ok = tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err);
                    if (!ok) break;
                    uint8_t *st = smem + r.i * PAIR_STAGE;
                    const uint32_t bar = tc::leader_addr(&s.full[r.i]);
                    if (rank == 0) tc::mbar_arrive_tx(&s.full[r.i], 2u * PAIR_STAGE);
                    tc::tma_load_2d_pair(st, &x_map, (int)(c * 128u), row0, bar);
                    tc::tma_load_2d_pair(st + PAIR_A, &w_map, (int)(c * 128u), out0, bar);
                    tc::tma_load_2d_pair(st + PAIR_A + PAIR_B, &x_scale_map, 0, (int)(x_scales + c * 8u), bar);
                    tc::tma_load_2d_pair(st + PAIR_A + PAIR_B + 1024, &w_scale_map, 0, (int)(w_scales + c * 16u), bar);
                    r.next(PAIR_STAGES);
                }
            }
            if (s.fail.failed) tc::outlast_copies();  // their bytes are counted in the leader alone
        }
    } else if (warp == 1) {
        if (rank == 0) {  // scales to tensor memory and products, in the leader for both
            const uint32_t base = tc::smem_u32(smem);
            constexpr uint32_t ID0 = tc::idesc_mxf4(256, PAIR_N, 0), ID1 = tc::idesc_mxf4(256, PAIR_N, 1);
            const bool mine = tc::elect();
            tc::Ring r, acc, old, sf;  // old: the stage whose scales' place comes next
            uint32_t ahead = 0;
            bool ok = true;
            for (uint32_t t = first; t < tiles && ok; t += step) {
                ok = __all_sync(~0u, tc::mbar_wait(&s.acc_empty[acc.i], acc.phase ^ 1u, fail, a.err));
                if (!ok) break;
                tc::fence_after();
                for (uint32_t c = 0; c < a.chunks; ++c) {
                    ok = __all_sync(~0u, tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
                    if (++ahead > 2u) {
                        ok = ok && __all_sync(~0u, tc::mbar_wait(&s.empty[old.i], old.phase, fail, a.err));
                        old.next(PAIR_STAGES);
                    }
                    if (!ok) break;
                    tc::fence_after();
                    const uint32_t st = base + r.i * PAIR_STAGE, sfa = tmem + PAIR_SF_AT + sf.i * PAIR_SF_COLS;
                    if (mine) {
                        stage_products<2, true>(tmem + acc.i * PAIR_N, tc::smem_desc(st, 16, 1024), tc::smem_desc(st + PAIR_A, 16, 1024),
                                                tc::scale_desc(st + PAIR_A + PAIR_B), sfa, sfa + 8u, ID0, ID1,
                                                c + 1u == a.chunks ? a.last_steps : 4u, c != 0);
                        tc::commit_pair(&s.empty[r.i]);
                        if (c + 1u == a.chunks) tc::commit_pair(&s.acc_full[acc.i]);
                    }
                    __syncwarp();
                    sf.next(2);
                    r.next(PAIR_STAGES);
                }
                acc.next(2);
            }
            if (!ok) {  // leave no product in flight
                if (mine) tc::commit_pair(&s.failed);
                tc::mbar_wait_slow(&s.failed, 0, fail, a.err, true);
            }
        }
    } else if (warp >= 4 && warp < 8) {  // results: a lane has a row of this CTA's 128
        const uint32_t quad = warp % 4u, in_tile = quad * 32u + lane;
        tc::Ring acc;
        for (uint32_t t = first; t < tiles; t += step) {
            const uint64_t row = (uint64_t)(t / a.out_tiles) * 256u + rank * 128u + quad * 32u;  // the warp's first
            const uint32_t out0 = t % a.out_tiles * PAIR_N;
            // the bias of the tile's outputs; the first barrier keeps the last tile's until it is used
            asm volatile("bar.sync 1, 128;" ::: "memory");
            for (uint32_t i = in_tile; i < PAIR_N; i += 128u)
                s.bias[i] = a.bias && out0 + i < a.outs ? to_f32<T>(__ldg((const T *)a.bias + out0 + i)) : 0.0f;
            asm volatile("bar.sync 1, 128;" ::: "memory");
            const bool ok = tc::mbar_wait(&s.acc_full[acc.i], acc.phase, fail, a.err);
            if (__all_sync(~0u, ok)) {  // else on to the next barrier with the other warps
                tc::fence_after();
#pragma unroll 1
                for (uint32_t n0 = 0; n0 < PAIR_N; n0 += 32u) {
                    uint32_t v[32];
                    tc::tmem_load32(tmem + acc.i * PAIR_N + (quad * 32u << 16) + n0, v);
                    if (n0 + 32u == PAIR_N) {
                        tc::fence_before();
                        __syncwarp();
                        if (lane == 0) tc::mbar_arrive_cluster(tc::leader_addr(&s.acc_empty[acc.i]));
                    }
                    store_results<T, ACT>((T *)a.y + row * a.outs, rows_left(row, a.rows), out0 + n0, a.outs, a.y_wide, v, s.bias + n0,
                                          s.turn[quad]);
                }
            }
            acc.next(2);
        }
    }
    __syncwarp();
    tc::fence_before();
    tc::cluster_sync();  // no CTA leaves while the other may still reach its barriers
    if (warp == 1) tc::tmem_free_pair<512>(tmem);
}

// ---- few tiles ----

constexpr uint32_t FEW_STAGES = 6, FEW_STAGE = 2u * 16384u + 2048u, FEW_THREADS = 512;
struct FewCtrl {
    uint64_t full[FEW_STAGES], empty[FEW_STAGES], acc_full;
    uint32_t tmem;
    tc::Fail fail;
};
constexpr uint32_t FEW_SMEM = FEW_STAGES * FEW_STAGE + sizeof(FewCtrl);

struct FewArgs {
    uint64_t rows, x_stride;
    uint32_t cols, outs, blocks, chunks, last_steps, chunks_a_split;
    const void *x;
    const uint8_t *w_exps;
    const void *bias;
    void *y;
    uint32_t *err;
    bool x_vec;
};

// grid: (splits of k = the cluster, tiles of 128 outputs, tiles of 128 rows)
template <typename T, int ACT>
__global__ void __launch_bounds__(FEW_THREADS, 1) few_kernel(const __grid_constant__ CUtensorMap w_map, const FewArgs a)
{
    extern __shared__ __align__(1024) uint8_t smem[];
    FewCtrl &s = *reinterpret_cast<FewCtrl *>(smem + FEW_STAGES * FEW_STAGE);
    const uint32_t warp = tc::warp_number(), lane = threadIdx.x % 32u, splits = gridDim.x, rank = blockIdx.x;
    const uint32_t out0 = blockIdx.y * 128u, c0 = rank * a.chunks_a_split, c1 = min(a.chunks, c0 + a.chunks_a_split);
    const uint64_t row0 = (uint64_t)blockIdx.z * 128u;
    const uint32_t rows = (uint32_t)(a.rows - row0 < 128u ? a.rows - row0 : 128u), n = (rows + 15u) / 16u * 16u;
    tc::Fail *const fail = &s.fail;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < FEW_STAGES; ++i) {
            tc::mbar_init(&s.full[i], 1 + 1 + 8);
            tc::mbar_init(&s.empty[i], 1);
        }
        tc::mbar_init(&s.acc_full, 1);
        s.fail.failed = 0;
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&w_map);
    }
    if (warp == 1) tc::tmem_alloc<256>(&s.tmem);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        if (lane == 0) {  // TMA of the weight's codes
            tc::Ring r;
            for (uint32_t c = c0; c < c1; ++c) {
                if (!tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err)) break;
                tc::mbar_arrive_tx(&s.full[r.i], 16384);
                tc::tma_load_2d(smem + r.i * FEW_STAGE, &w_map, (int)(c * 128u), (int)out0, &s.full[r.i]);
                r.next(FEW_STAGES);
            }
            if (s.fail.failed) tc::outlast_copies();
        }
    } else if (warp == 1) {  // scales to tensor memory, products
        const uint32_t base = tc::smem_u32(smem);
        const uint32_t id0 = tc::idesc_mxf4(128, 0, 0) | (n >> 3) << 17, id1 = tc::idesc_mxf4(128, 0, 1) | (n >> 3) << 17;
        const bool mine = tc::elect();
        tc::Ring r;
        bool ok = true;
        for (uint32_t c = c0; c < c1; ++c) {
            ok = __all_sync(~0u, tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
            if (!ok) break;
            tc::fence_after();
            const uint32_t st = base + r.i * FEW_STAGE, sfa = tmem + 128u + r.i * 16u, sfb = sfa + 8u;  // a place for every stage
            if (mine) {
                stage_products<1>(tmem, tc::smem_desc(st, 16, 1024), tc::smem_desc(st + 16384u, 16, 1024), tc::scale_desc(st + 32768u), sfa,
                                  sfb, id0, id1, c + 1u == a.chunks ? a.last_steps : 4u, c != c0);
                tc::commit(&s.empty[r.i]);
            }
            __syncwarp();
            r.next(FEW_STAGES);
        }
        if (mine) tc::commit(&s.acc_full);
        if (!ok) tc::mbar_wait_slow(&s.acc_full, 0, fail, a.err, true);  // leave no product in flight
    } else if (warp >= 4 && warp < 8) {  // the weight's scales, then this CTA's sums to its shared memory
        const uint32_t quad = warp % 4u, i = quad * 32u + lane;
        tc::Ring r;
        bool ok = true;
        for (uint32_t c = c0; c < c1; ++c, r.next(FEW_STAGES)) {
            if ((c - c0) % 4u != quad) continue;  // the warps take stages in turn
            uint2 e[4];
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                e[k] = out0 + k * 32u + lane < a.outs ? load_scales(a.w_exps, out0 + k * 32u + lane, a.blocks, c * 8u) : make_uint2(0, 0);
            ok = __all_sync(~0u, tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err));
            if (!ok) break;
            uint8_t *sf = smem + r.i * FEW_STAGE + 32768u;
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) store_scales(sf, k * 32u + lane, e[k]);
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s.full[r.i]);
        }
        if (ok && __all_sync(~0u, tc::mbar_wait(&s.acc_full, 0, fail, a.err))) {
            tc::fence_after();
            // all products are done, so the stages are free: [row][output] in binary32
            float *sum = reinterpret_cast<float *>(smem);
            for (uint32_t j = 0; j < n; j += 32u) {
                uint32_t v[32];
                tc::tmem_load32(tmem + (quad * 32u << 16) + j, v);
#pragma unroll
                for (uint32_t k = 0; k < 32; ++k)  // the last splits may have no part of k
                    if (j + k < rows) sum[(j + k) * 128u + i] = c0 < c1 ? __uint_as_float(v[k]) : 0.0f;
            }
        }
    } else if (warp >= 8) {  // x to 4 bits, a lane a block
        tc::Ring r;
        for (uint32_t c = c0; c < c1; ++c) {
            const bool ok = __all_sync(~0u, tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err));
            if (!ok) break;
            uint8_t *st = smem + r.i * FEW_STAGE + 16384u;
            // with few blocks a stage the warps' shares turn with the stages, so that all warps have loads in flight
            for (uint32_t i = (warp - c * ((rows + 3u) / 4u)) % 8u * 32u + lane; i < rows * 8u; i += 256u) {
                const uint32_t row = i / 8u, block = i % 8u, col = c * L4_K + block * 32u;
                const T *p = (const T *)a.x + (row0 + row) * a.x_stride + col;
                uint4 w[4];
                if (a.x_vec && col + 32u <= a.cols) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) w[u] = __ldg(reinterpret_cast<const uint4 *>(p) + u);
                } else {
                    uint32_t *h = reinterpret_cast<uint32_t *>(w);
#pragma unroll
                    for (uint32_t u = 0; u < 16; ++u) {
                        const uint32_t lo = col + 2 * u < a.cols ? __ldg(reinterpret_cast<const unsigned short *>(p) + 2 * u) : 0u;
                        const uint32_t hi = col + 2 * u + 1 < a.cols ? __ldg(reinterpret_cast<const unsigned short *>(p) + 2 * u + 1) : 0u;
                        h[u] = lo | hi << 16;
                    }
                }
                uint32_t E;
                const uint4 codes = block_codes<T>(w, E);
                *reinterpret_cast<uint4 *>(st + row * 128u + ((block ^ (row & 7u)) << 4)) = codes;
                st[16384u + 1024u + scale_place(row) + (block >> 2) * 512u + (block & 3u)] = (uint8_t)E;
            }
            tc::fence_async_shared();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s.full[r.i]);
            r.next(FEW_STAGES);
        }
    }
    __syncwarp();
    tc::fence_before();
    tc::cluster_sync();
    if (!s.fail.failed) {  // each CTA finishes every splits-th row: the parts in the order of k
        const uint32_t out = threadIdx.x % 128u;
        const float b = a.bias && out0 + out < a.outs ? to_f32<T>(__ldg((const T *)a.bias + out0 + out)) : 0.0f;
        for (uint32_t row = rank + splits * (threadIdx.x / 128u); row < rows; row += splits * (FEW_THREADS / 128u)) {
            float v = 0.0f;
            for (uint32_t p = 0; p < splits; ++p) v += tc::load_cluster(reinterpret_cast<float *>(smem) + row * 128u + out, p);
            if (out0 + out < a.outs)
                ((T *)a.y)[(row0 + row) * a.outs + out0 + out] = from_f32<T>(unpair(act_value2<ACT>(both(v + b))).x);
        }
    }
    __syncwarp();
    tc::cluster_sync();  // no CTA leaves while another may still read its sums
    if (warp == 1) tc::tmem_free<256>(tmem);
}

// No columns: the activation of the bias alone.
template <typename T, int ACT> __global__ void bias_rows_kernel(const T *bias, uint64_t rows, uint32_t outs, T *y)
{
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < rows * outs; i += (uint64_t)gridDim.x * 256u)
        y[i] = from_f32<T>(unpair(act_value2<ACT>(both(bias ? to_f32<T>(bias[i % outs]) : 0.0f))).x);
}
template <typename T, int ACT> static vt_status launch_bias(const L4Args &a, cudaStream_t stream)
{
    bias_rows_kernel<T, ACT><<<sm_count(), 256, 0, stream>>>((const T *)a.bias, a.rows, a.outs, (T *)a.y);
    return check_launch("bias_rows_kernel");
}

template <typename T, int ACT, int TN>
static vt_status launch_linear4(const void *x, uint64_t x_stride, const uint8_t *w_codes, L4Args a, cudaStream_t stream)
{
    static std::atomic<uint64_t> allowed{0};
    using P = L4<TN>;
    CUtensorMap x_map, w_map;
    const uint64_t pitch = (uint64_t)a.blocks * 16u;
    if (vt_status s = map_rows<T>(&x_map, x, x_stride, a.rows, a.cols, L4_ROWS)) return s;
    if (vt_status s = tc::make_map(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, w_codes, a.outs, pitch, pitch, TN, 128)) return s;
    if (vt_status s = tc::allow_smem(linear4_kernel<T, ACT, TN>, P::SMEM, allowed)) return s;
    a.row_tiles = (uint32_t)((a.rows + L4_ROWS - 1u) / L4_ROWS);
    const uint32_t sms = (uint32_t)sm_count();
    linear4_kernel<T, ACT, TN><<<a.row_tiles < sms ? a.row_tiles : sms, P::THREADS, P::SMEM, stream>>>(x_map, w_map, a);
    return check_launch("linear4_kernel");
}

template <typename T, int ACT>
static vt_status launch_pair4(const void *x, uint64_t x_stride, const uint8_t *w_codes, L4Args a, uint8_t *workspace, cudaStream_t stream)
{
    static std::atomic<uint64_t> allowed{0};
    const PairPlan p = pair_plan(a.rows, a.cols, a.outs);
    VT_REQUIRE((uint64_t)p.row_tiles * p.chunks < (1u << 26) && (uint64_t)p.out_tiles * p.chunks < (1u << 26), "vt_mx4_linear: too large");
    uint8_t *codes = workspace, *x_scales = workspace + p.x_scales_at, *w_scales = workspace + p.w_scales_at;
    const uint32_t sms = (uint32_t)sm_count(), pairs = sms / 2u;
    const uint64_t x_items = (uint64_t)p.row_tiles * 256u * p.chunks * 32u, w_items = (uint64_t)p.out_tiles * p.chunks * 512u;
    const uint64_t want = ((x_items > w_items ? x_items : w_items) + 255u) / 256u;
    const bool vec = a.cols % 8u == 0 && x_stride % 8u == 0 && aligned16(x);
    stage4_kernel<T><<<(unsigned)(want < sms * 32u ? want : sms * 32u), 256, 0, stream>>>((const T *)x, x_stride, a.rows, a.cols, a.blocks, vec,
                                                                                      p.chunks, x_items, (uint32_t *)codes, x_scales, a.w_exps,
                                                                                      a.outs, w_items, (uint32_t *)w_scales);
    if (vt_status s = check_launch("stage4_kernel")) return s;
    CUtensorMap x_map, w_map, x_scale_map, w_scale_map;
    const uint64_t pitch = (uint64_t)a.blocks * 16u;
    const CUtensorMapDataType bytes = CU_TENSOR_MAP_DATA_TYPE_UINT8;
    if (vt_status s = tc::make_map(&x_map, bytes, codes, a.rows, pitch, pitch, 128, 128)) return s;
    if (vt_status s = tc::make_map(&w_map, bytes, w_codes, a.outs, pitch, pitch, PAIR_N / 2, 128)) return s;
    if (vt_status s = tc::make_map(&x_scale_map, bytes, x_scales, (uint64_t)p.row_tiles * 2u * p.chunks * 8u, 128, 128, 8, 128, false)) return s;
    if (vt_status s = tc::make_map(&w_scale_map, bytes, w_scales, (uint64_t)p.out_tiles * p.chunks * 16u, 128, 128, 16, 128, false)) return s;
    if (vt_status s = tc::allow_smem(pair4_kernel<T, ACT>, PAIR_SMEM, allowed)) return s;
    a.row_tiles = p.row_tiles;
    a.out_tiles = p.out_tiles;
    const uint64_t tiles = (uint64_t)a.row_tiles * a.out_tiles;
    pair4_kernel<T, ACT><<<(unsigned)(tiles < pairs ? tiles : pairs) * 2u, PAIR_THREADS, PAIR_SMEM, stream>>>(x_map, w_map, x_scale_map, w_scale_map, a);
    return check_launch("pair4_kernel");
}

// Splits of k for few_kernel, a power of two up to 8; 0: there are tiles enough for linear4_kernel.
// few_kernel's tiles are 128 x 128 and every SM gets at most one CTA of it; with more of them than
// half the SMs splitting gains nothing and the larger tiles read their operands less often.
static uint32_t few_splits(uint64_t rows, uint32_t cols, uint32_t outs, uint32_t sms)
{
    const uint64_t tiles = (rows + 127u) / 128u * ((outs + 127u) / 128u);
    if (tiles > sms / 2u) return 0;
    const uint32_t chunks = (cols + L4_K - 1u) / L4_K;
    uint32_t n = 1;
    while (n < 8u && 2u * n <= chunks && tiles * 2u * n <= sms) n *= 2u;
    return n;
}

template <typename T, int ACT>
static vt_status launch_few(const uint8_t *w_codes, FewArgs a, uint32_t splits, cudaStream_t stream)
{
    static std::atomic<uint64_t> allowed{0};
    CUtensorMap w_map;
    const uint64_t pitch = (uint64_t)a.blocks * 16u;
    if (vt_status s = tc::make_map(&w_map, CU_TENSOR_MAP_DATA_TYPE_UINT8, w_codes, a.outs, pitch, pitch, 128, 128)) return s;
    if (vt_status s = tc::allow_smem(few_kernel<T, ACT>, FEW_SMEM, allowed)) return s;
    a.chunks_a_split = (a.chunks + splits - 1u) / splits;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(splits, (a.outs + 127u) / 128u, (unsigned)((a.rows + 127u) / 128u));
    config.blockDim = dim3(FEW_THREADS);
    config.dynamicSmemBytes = FEW_SMEM;
    config.stream = stream;
    cudaLaunchAttribute cluster = {};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim = {splits, 1, 1};
    config.attrs = &cluster;
    config.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, few_kernel<T, ACT>, w_map, a);
    if (e != cudaSuccess) {
        cudaGetLastError();
        return set_error(VT_ERR_CUDA, "few_kernel: %s", cudaGetErrorString(e));
    }
    return VT_OK;
}

}  // namespace vt

// copies: x's rows do not start on 16 bytes
extern "C" uint64_t vt_mx4_linear_workspace_bytes(uint64_t rows, uint32_t cols, uint32_t outs, int copies)
{
    if (vt::few_splits(rows, cols, outs, (uint32_t)vt::sm_count())) return 0;
    if (outs <= 256u) return copies ? rows * vt::align_up(cols, 8) * 2u : 0;  // x is rounded inside the kernel
    return vt::pair_plan(rows, cols, outs).bytes;
}

extern "C" vt_status vt_mx4_linear(const void *x, uint64_t x_stride, int dtype, uint64_t rows, uint32_t cols,
                                   uint32_t outs, const uint8_t *codes, const uint8_t *exps, const void *bias, int act,
                                   void *y, void *workspace, uint64_t workspace_bytes, uint32_t *err, vt_stream stream)
{
    VT_REQUIRE(rows <= (1ull << 31) - 256, "vt_mx4_linear: too many rows");
    VT_REQUIRE(cols <= (1u << 20) && outs <= (1u << 20), "vt_mx4_linear: layer too wide");
    VT_REQUIRE((rows + 127) / 128 * ((outs + 63) / 64) < (1ull << 31), "vt_mx4_linear: too many outputs");
    if (rows == 0 || outs == 0) return VT_OK;
    VT_REQUIRE(y && (cols == 0 || (x && codes && exps)), "vt_mx4_linear: null pointer");
    VT_REQUIRE(x_stride >= cols, "vt_mx4_linear: the row stride is less than a row");
    VT_REQUIRE(vt::aligned16(codes), "vt_mx4_linear: codes must be 16-byte aligned");
    cudaStream_t st = (cudaStream_t)stream;
    return vt::with_type16(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        VT_REQUIRE(vt::on_elements<T>(x, bias, y), "vt_mx4_linear: a matrix does not start on an element");
        VT_REQUIRE(workspace_bytes >= vt_mx4_linear_workspace_bytes(rows, cols, outs, !vt::whole_words<T>(x, x_stride)) &&
                       vt::aligned16(workspace),
                   "vt_mx4_linear: workspace too small or not 16-byte aligned");
        vt::L4Args a = {};
        a.rows = rows;
        a.cols = cols;
        a.outs = outs;
        a.blocks = vt::mx_blocks(cols);
        a.chunks = (cols + vt::L4_K - 1u) / vt::L4_K;
        a.last_steps = ((cols - 1u) % vt::L4_K + 64u) / 64u;
        a.w_exps = exps;
        a.bias = bias;
        a.y = y;
        a.err = err;
        a.y_wide = outs % 16u == 0 && vt::aligned32(y);
        if (cols == 0) return vt::with_act(act, [&](auto f) { return vt::launch_bias<T, decltype(f)::value>(a, st); });
        if (const uint32_t splits = vt::few_splits(rows, cols, outs, (uint32_t)vt::sm_count())) {
            vt::FewArgs f = {};
            f.rows = rows;
            f.x_stride = x_stride;
            f.cols = cols;
            f.outs = outs;
            f.blocks = a.blocks;
            f.chunks = a.chunks;
            f.last_steps = a.last_steps;
            f.x = x;
            f.w_exps = exps;
            f.bias = bias;
            f.y = y;
            f.err = err;
            f.x_vec = vt::whole_words<T>(x, x_stride);
            return vt::with_act(act, [&](auto k) { return vt::launch_few<T, decltype(k)::value>(codes, f, splits, st); });
        }
        if (outs <= 256u) {
            const void *from = x;
            uint64_t stride = x_stride;
            if (vt_status s = vt::whole_rows<T>(from, stride, rows, cols, workspace, st)) return s;
            return vt::with_act(act, [&](auto f) -> vt_status {
                constexpr int ACT = decltype(f)::value;
                if (outs <= 64u) return vt::launch_linear4<T, ACT, 64>(from, stride, codes, a, st);
                if (outs <= 128u) return vt::launch_linear4<T, ACT, 128>(from, stride, codes, a, st);
                return vt::launch_linear4<T, ACT, 256>(from, stride, codes, a, st);
            });
        }
        return vt::with_act(act, [&](auto f) -> vt_status {
            return vt::launch_pair4<T, decltype(f)::value>(x, x_stride, codes, a, (uint8_t *)workspace, st);
        });
    });
}

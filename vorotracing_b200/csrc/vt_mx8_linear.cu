// vt_mx8_linear.cu -- gradients of y = act(z) W^T + b from an 8-bit checkpoint of z (vt_mx.cuh):
//   dz = (dy W) * act'(z8),  dW = dy^T act(z8),  db = column sums of dy
//
// Layers with up to 256 outputs (narrow_kernel) make all three in one pass over the rows, so dy
// and the checkpoint are read from HBM once and act(z8) never reaches memory.  A CTA owns a slab
// of 128 columns of z and every G-th tile of 32 or 64 rows.  A tile of dy is staged once in shared
// memory (TMA, 128-byte swizzle) and used twice: as the K-major B operand of dH^T = W^T dy^T,
// whose result has z's columns in the lanes of tensor memory, and, the same bytes read the other
// way, as the MN-major B operand of dW^T += act(z8)^T dy, whose accumulator stays in tensor memory
// over all the CTA's rows.  Between the two products sixteen warps take dH out of tensor memory,
// read the 8-bit z, evaluate act and act' together (one logistic serves both), write dz, and put
// act(z8) back into the place of dH as the second product's A operand, rounded to the operands'
// 16-bit type: what the forward pass multiplied by W was rounded to it too, so dW is the gradient of the
// product that was computed.  Against 64 bits dW is off by 1.15 to 1.25 times what rounding dW itself costs.  (A second
// operand for what the rounding left would cost half as much again of the tensor cores' time in wide layers.)  The column sums of dy are one more,
// narrow product of the staged tile.  At its end a CTA writes its part of dW in binary32; a second
// kernel adds the parts in order, so results do not depend on timing.
//
// Shared memory's bandwidth is what is short between HBM and the tensor cores here, which decides
// the orientation: with z's columns in the lanes the activations need no shared memory at all, a
// warp's dz is 64 contiguous bytes a row, and the second product reads one operand instead of two.
// Up to 8 outputs (a colour) are rows of 16 bytes or less, whose TMA copies would take as long as
// eight times the bytes; one warp brings them in instead, without a copy to whole words before.
//
// Layers of up to 64 columns would leave half of the lanes empty; they get W twice instead (FOLD),
// and each half of the lanes takes half of a tile's rows: the second product of a half's rows leaves the other
// half's lanes as they are.  (Zeros in their place would make an infinity in dy a NaN of every column.)
//
// Measured (bfloat16, B200s, in a loop of calls): 1088640 rows, 256 -> 256, SiLU: 398 to 429 us by the GPU, 3.3 to 3.5 TB/s
// of what it has to read and write (floor at 6.45 TB/s: 218 us).  What bounds it: with 256 outputs dW, W and
// the column sums leave room for three buffers of dH, so one of the four sets of activation warps always
// waits; a tile of 32 rows takes 1030 cycles where its bytes would take 700.  Steps on the way: rows in the
// lanes, activations through shared memory 479 us; columns in the lanes 439; W in tensor memory instead of
// shared memory 424; column sums on the tensor cores (a warp that added took as long as all else) 404.
// 1614080 rows, 64 -> 3, ReLU: 98 us (floor 50 us), bound by the second product's warp: its wait, issue
// and commit take most of the 1000 cycles of a tile of 64 rows.  Steps: tiles of 32 rows 150 us; of 64 139;
// dy's rows loaded ahead in registers 115; parts added by blocks 98.  Two tiles a turn of that warp: no gain.
//
// Wider layers are two matrix products (wide_kernel), both on pairs of CTAs that share a 256 x 256
// tile: dz = (dy W) * act'(z8), with the slope in the epilogue, and dW = dy^T h with h = act(z8)
// written once, in the operands' type, by a pass before it: as an operand it is read once for
// every 256 outputs, and evaluating it as often would cost more than the tensor cores' time.
// Measured (binary16): 8192 rows, 4096 -> 4096, GELU: 516 to 547 us by the GPU, 1.01 to 1.07 PFLOP/s, at 1.56 GHz under
// the power limit; the tensor cores are busy 68 % of the time there, dW's 256 tiles fill 3.5 rounds of 74 pairs.
#include "vt_mx_rows.cuh"

namespace vt {

// ---- layers with up to 256 outputs ----

constexpr uint32_t NARROW_OUTS = 256, NARROW_THREADS = 640, TINY_OUTS = 8;

// Rows of a tile.  64 halve the barriers and commits a row, which bound layers of few outputs (64 -> 3:
// 150 us with 32, 139 with 64, before the steps above); more than 128 outputs leave tensor memory for buffers of 32 only.
constexpr uint32_t narrow_rows(uint32_t oc) { return oc <= 2 ? 64 : 32; }

// OC: dy's columns in chunks of 64.  A slab is 128 columns of z, or all of up to 64 (FOLD).
template <int OC, bool FOLD> struct Narrow {
    static constexpr uint32_t TILE_ROWS = narrow_rows(OC);
    static constexpr uint32_t CHUNK = TILE_ROWS * 128u, DY_BYTES = OC * CHUNK, CODE_PITCH = FOLD ? 64u : 128u;
    static constexpr uint32_t STAGE = DY_BYTES + TILE_ROWS * CODE_PITCH;
    struct Ctrl {
        float scale[16][TILE_ROWS];  // of the blocks in each activation warp's rows
        uint64_t full[12], empty[12], dh_full[narrow_ready(OC)], h_full[narrow_buffers(OC)], w_full, done, failed;
        uint32_t tmem;
        tc::Fail fail;
    };
    static constexpr uint32_t ONES = 2048u, FIT = (232448u - ONES - sizeof(Ctrl)) / STAGE, STAGES = FIT < 12u ? FIT : 12u;
    static constexpr uint32_t ONES_AT = STAGES * STAGE, CTRL_AT = ONES_AT + ONES, SMEM = CTRL_AT + sizeof(Ctrl);
    static constexpr uint32_t TMEM = 512;
    // columns of tensor memory: dW, W, db (16 for 128 outputs), and as many of dH as there is room for, up to six
    static constexpr uint32_t W_AT = OC * 64u, MT = (OC + 1) / 2, DB_AT = W_AT + OC * 32u, DH_AT = DB_AT + MT * 16u, BUFS = narrow_buffers(OC), READY = narrow_ready(OC);
    static constexpr int ROWS = FOLD ? TILE_ROWS / 2 : TILE_ROWS;  // of a tile an activation warp takes
    static_assert(NARROW_SETS == 4 && READY >= 4 && STAGES >= 4 && STAGES > BUFS && DH_AT + BUFS * TILE_ROWS <= TMEM, "does not fit an SM");
};

struct NarrowArgs {
    uint64_t rows;
    uint32_t cols, outs, blocks, tiles, groups, slabs;
    const void *weight;
    uint64_t weight_stride;
    const int8_t *codes;
    const uint8_t *exps;
    void *dz;          // null: not wanted
    // where dW and db go, null if not wanted: parts for a second kernel, [group][slab][OC * 64][128] and
    // [group][OC * 64], or with one group the results themselves
    float *dw_parts, *db_parts;
    void *dw, *db;
    uint32_t *err;
    const void *dy;    // read by a warp instead of TMA: up to TINY_OUTS outputs; else null
    uint64_t dy_stride;
    bool codes_whole;  // a tile's codes are one piece of memory
    bool dy_chunked;   // dy's columns are whole chunks of 64: one TMA copy brings all of them in
};

// 16 columns of a row: codes (4 words) and their block's scale, g = dH (binary32) in, dz out as
// packed 16-bit pairs.
template <typename T, int ACT>
__device__ __forceinline__ void slope16(const uint32_t *codes, f32x2 sc, const uint32_t *g, uint32_t *dz)
{
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const uint32_t c = codes[w] ^ 0x80808080u;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = 2 * w + i;
            const f32x2 gp = pair(__uint_as_float(g[2 * at]), __uint_as_float(g[2 * at + 1]));
            dz[at] = pack2<T>(ACT == ACT_IDENTITY ? gp : mul2(gp, act_slope2<ACT>(mul2(code_pair(c, 2 * i), sc))));
        }
    }
}

template <typename T, int ACT, int OC, bool FOLD>
__global__ void __launch_bounds__(NARROW_THREADS, 1)
    narrow_kernel(const __grid_constant__ CUtensorMap dy_map, const __grid_constant__ CUtensorMap code_map, const NarrowArgs a)
{
    using P = Narrow<OC, FOLD>;
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    constexpr uint32_t TILE_ROWS = P::TILE_ROWS;
    extern __shared__ __align__(1024) uint8_t smem[];
    typename P::Ctrl &s = *reinterpret_cast<typename P::Ctrl *>(smem + P::CTRL_AT);
    const uint32_t warp = tc::warp_number(), lane = threadIdx.x % 32u;
    const uint32_t slab = blockIdx.x % a.slabs, group = blockIdx.x / a.slabs;
    // the column sums of dy, 128 outputs at a time, are shared out among the slabs
    const uint32_t sharers = a.slabs < P::MT ? a.slabs : P::MT;
    const bool sums = (a.db_parts || a.db) && slab < sharers, tiny = OC == 1 && a.dy;
    tc::Fail *const fail = &s.fail;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < P::STAGES; ++i) {
            tc::mbar_init(&s.full[i], tiny ? 2 : 1);
            tc::mbar_init(&s.empty[i], 1);
        }
        for (uint32_t i = 0; i < P::READY; ++i) tc::mbar_init(&s.dh_full[i], 1);
        for (uint32_t i = 0; i < P::BUFS; ++i) tc::mbar_init(&s.h_full[i], 4);
        tc::mbar_init(&s.w_full, 16);
        tc::mbar_init(&s.done, 1);
        tc::mbar_init(&s.failed, 1);
        s.fail.failed = 0;
        tc::mbar_init_fence();
        if (!tiny) tc::tma_prefetch_map(&dy_map);
        if (!a.codes_whole) tc::tma_prefetch_map(&code_map);
    }
    for (uint32_t i = threadIdx.x; i < P::ONES / 4u; i += NARROW_THREADS)
        reinterpret_cast<uint32_t *>(smem + P::ONES_AT)[i] = pack2<T>(1.0f, 1.0f);
    if (tiny)  // all but the first 16 bytes of dy's rows stay zero
        for (uint32_t i = threadIdx.x; i < P::STAGES * (P::CHUNK / 16u); i += NARROW_THREADS)
            *reinterpret_cast<uint4 *>(smem + i / (P::CHUNK / 16u) * P::STAGE + i % (P::CHUNK / 16u) * 16u) = make_uint4(0, 0, 0, 0);
    tc::fence_async_shared();
    if (warp == 1) tc::tmem_alloc<P::TMEM>(&s.tmem);
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const uint32_t tmem = s.tmem, dh_at = tmem + P::DH_AT;

    if (warp == 0) {
        if (lane == 0) {  // TMA
            uint32_t issued = 0;
            tc::Ring r;
            for (uint32_t t = group; t < a.tiles; t += a.groups) {
                if (!tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err)) break;
                uint8_t *st = smem + r.i * P::STAGE;
                // a last tile's missing rows of whole codes keep those of an older tile: their dy is zero
                const uint32_t code_bytes = !a.codes_whole || t + 1u < a.tiles ? TILE_ROWS * P::CODE_PITCH
                                                                              : (uint32_t)(a.rows - (uint64_t)t * TILE_ROWS) * P::CODE_PITCH;
                tc::mbar_arrive_tx(&s.full[r.i], (tiny ? 0u : P::DY_BYTES) + code_bytes);
                if (tiny) {
                } else if (OC > 1 && a.dy_chunked) {
                    tc::tma_load_3d(st, &dy_map, 0, (int)(t * TILE_ROWS), 0, &s.full[r.i]);
                } else {
                    for (int c = 0; c < OC; ++c)
                        tc::tma_load_2d(st + c * P::CHUNK, &dy_map, c * 64, (int)(t * TILE_ROWS), &s.full[r.i]);
                }
                if (a.codes_whole)
                    tc::bulk_load(st + P::DY_BYTES, a.codes + (uint64_t)t * (TILE_ROWS * P::CODE_PITCH), code_bytes, &s.full[r.i]);
                else
                    tc::tma_load_2d(st + P::DY_BYTES, &code_map, (int)(slab * 128), (int)(t * TILE_ROWS), &s.full[r.i]);
                ++issued;
                r.next(P::STAGES);
            }
            if (s.fail.failed)  // leave no copy in flight
                for (uint32_t i = 0; i < P::STAGES && i < issued; ++i)
                    tc::mbar_wait_slow(&s.full[i], ((issued - 1 - i) / P::STAGES) & 1u, fail, a.err, true);
        }
    } else if (warp == 1) {  // dH^T = W^T dy^T
        constexpr uint32_t ID = tc::idesc_f16<BF16>(128, TILE_ROWS, false, false);
        const uint32_t st_addr = tc::smem_u32(smem);
        const bool mine = tc::elect();
        tc::Ring r, dh, ready, old;  // old: the stage of the tile that had this one's buffer of dH
        bool ok = __all_sync(~0u, tc::mbar_wait(&s.w_full, 0, fail, a.err));
        for (uint32_t t = group; t < a.tiles && ok; t += a.groups) {
            ok = __all_sync(~0u, tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
            if (t >= group + P::BUFS * a.groups) {  // its second product has left both
                ok = ok && __all_sync(~0u, tc::mbar_wait(&s.empty[old.i], old.phase, fail, a.err));
                old.next(P::STAGES);
            }
            if (!ok) break;
            tc::fence_after();
            const uint64_t b = tc::smem_desc(st_addr + r.i * P::STAGE, 16, 1024);
            if (mine) {
#pragma unroll
                for (uint32_t c = 0; c < OC; ++c)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        tc::mma_f16_tmem(dh_at + dh.i * TILE_ROWS, tmem + P::W_AT + (c * 4u + k) * 8u, b + c * (P::CHUNK >> 4) + k * 2u,
                                         ID, c + k != 0);
                tc::commit(&s.dh_full[ready.i]);
            }
            __syncwarp();
            r.next(P::STAGES);
            dh.next(P::BUFS);
            ready.next(P::READY);
        }
        if (!ok) {  // leave no product in flight
            if (mine) tc::commit(&s.failed);
            tc::mbar_wait_slow(&s.failed, 0, fail, a.err, true);
        }
    } else if (warp == 3) {  // dW^T += h^T dy, behind the activations; in a warp of its own, so that neither product waits
                              // for what the other one waits for
        constexpr uint32_t ID = tc::idesc_f16<BF16>(128, OC * 64, false, true), ID_DB = tc::idesc_f16<BF16>(128, 16, true, false);
        const uint32_t st_addr = tc::smem_u32(smem);
        const uint64_t ones = tc::smem_desc(st_addr + P::ONES_AT, 16, 1024);
        const bool mine = tc::elect();
        tc::Ring r, h;
        bool ok = true;
        for (uint32_t t = group; t < a.tiles && ok; t += a.groups) {
            ok = __all_sync(~0u, tc::mbar_wait(&s.h_full[h.i], h.phase, fail, a.err) &&
                                     tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
            if (!ok) break;
            tc::fence_after();
            const uint64_t b = tc::smem_desc(st_addr + r.i * P::STAGE, P::CHUNK, 1024);
            const uint32_t from = dh_at + h.i * TILE_ROWS;
            if (mine) {
                if (a.dw_parts || a.dw)
#pragma unroll
                    for (uint32_t k = 0; k < TILE_ROWS / 16u; ++k) {
                        if (FOLD)  // each half of the lanes adds its own half of the tile's rows
                            tc::mma_f16_tmem_half(tmem, from + k * 16u, b + k * 128u, ID, k >= TILE_ROWS / 32u,
                                                  k % (TILE_ROWS / 32u) != 0 || t != group);
                        else
                            tc::mma_f16_tmem(tmem, from + k * 16u, b + k * 128u, ID, k != 0 || t != group);
                    }
                // db += dy^T ones.  Of an odd number of chunks the last tile's upper 64 outputs are whatever
                // follows in shared memory; they are not read.
                if (sums)
#pragma unroll
                    for (uint32_t m = 0; m < P::MT; ++m)
                        if (m % sharers == slab)
#pragma unroll
                            for (uint32_t k = 0; k < TILE_ROWS / 16u; ++k)
                                tc::mma_f16(tmem + P::DB_AT + m * 16u, b + m * (2u * P::CHUNK >> 4) + k * 128u, ones, ID_DB,
                                            k != 0 || t != group);
                tc::commit(&s.empty[r.i]);
            }
            __syncwarp();
            r.next(P::STAGES);
            h.next(P::BUFS);
        }
        if (mine) tc::commit(&s.done);
        if (!ok) tc::mbar_wait_slow(&s.done, 0, fail, a.err, true);  // leave no product in flight
    } else if (warp == 2) {
        if (tiny) {  // dy of few outputs, eight rows a lane in flight
            constexpr uint32_t PARTS = TILE_ROWS / 32u, AHEAD = 8u / PARTS;
            tc::Ring r;
            bool ok = true;
            unsigned short v[8][TINY_OUTS] = {};
            // a tile; rows behind the end repeat the last one here and become zero below
            const auto load = [&](uint32_t t, unsigned short (*w)[TINY_OUTS]) {
#pragma unroll
                for (uint32_t j = 0; j < PARTS; ++j) {
                    const uint64_t row = (uint64_t)t * TILE_ROWS + j * 32u + lane;
                    const unsigned short *p = (const unsigned short *)a.dy + (row < a.rows ? row : a.rows - 1u) * a.dy_stride;
#pragma unroll
                    for (uint32_t o = 0; o < TINY_OUTS; ++o)
                        if (o < a.outs) w[j][o] = __ldg(p + o);
                }
            };
#pragma unroll
            for (uint32_t i = 0; i < AHEAD; ++i) load(group + i * a.groups, v + i * PARTS);
            for (uint32_t t0 = group; t0 < a.tiles && ok; t0 += AHEAD * a.groups)
#pragma unroll
                for (uint32_t i = 0; i < AHEAD; ++i) {
                    const uint32_t t = t0 + i * a.groups;
                    if (t >= a.tiles) break;
                    ok = ok && __all_sync(~0u, tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err));
                    if (!ok) break;
#pragma unroll
                    for (uint32_t j = 0; j < PARTS; ++j) {
                        const unsigned short *w = v[i * PARTS + j];
                        const bool in = t + 1u < a.tiles || (uint64_t)t * TILE_ROWS + j * 32u + lane < a.rows;
                        uint4 x = make_uint4(0, 0, 0, 0);
                        if (in) x = make_uint4(w[0] | (uint32_t)w[1] << 16, w[2] | (uint32_t)w[3] << 16, w[4] | (uint32_t)w[5] << 16, w[6] | (uint32_t)w[7] << 16);
                        *reinterpret_cast<uint4 *>(smem + r.i * P::STAGE + (j * 32u + lane) * 128u + ((lane & 7u) << 4)) = x;
                    }
                    tc::fence_async_shared();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s.full[r.i]);
                    r.next(P::STAGES);
                    load(t + AHEAD * a.groups, v + i * PARTS);
                }
        }
    } else if (warp >= 4) {  // activations: four sets of four warps take tiles in turn; a lane has a column of z (a
              // warp one block of 32) and ROWS rows of the tile
        constexpr int ROWS = P::ROWS;
        const uint32_t quad = warp % 4u, set = (warp - 4u) / 4u;
        const uint32_t block = FOLD ? quad & 1u : slab * 4u + quad, n = block * 32u + lane;
        const uint32_t row0 = FOLD ? (quad >> 1) * (TILE_ROWS / 2u) : 0u;  // in the tile
        const uint32_t lanes = quad * 32u << 16, code0 = row0 * P::CODE_PITCH + (FOLD ? n : quad * 32u + lane);
        float *const scale = s.scale[warp - 4u];
        const uint32_t first = group + set * a.groups, step = 4u * a.groups;
        // exponent bytes of this warp's block, a row a lane: this tile's, and the next one's on their way
        const uint64_t first_row = (uint64_t)first * TILE_ROWS + row0;
        const uint8_t *exps = a.exps + (first_row + lane) * a.blocks + block;
        const uint64_t exps_step = (uint64_t)step * TILE_ROWS * a.blocks;
        constexpr int EXPS = (ROWS + 31) / 32;  // rows a lane has the scales of
        const uint32_t last = a.tiles - 1u, last_rows = (uint32_t)(a.rows - (uint64_t)last * TILE_ROWS);  // rows of the last tile
        const uint32_t last_count = last_rows > row0 ? min(last_rows - row0, (uint32_t)ROWS) : 0u;
        auto exponent = [&](uint32_t t, uint32_t (&e)[EXPS]) {
#pragma unroll
            for (int i = 0; i < EXPS; ++i) {
                const uint32_t row = i * 32u + lane;
                const bool in = row < ROWS && block < a.blocks && (t < last || (t == last && row < last_count));
                e[i] = in ? __ldg(exps + (uint64_t)i * 32u * a.blocks) : 127u;
            }
            exps += exps_step;
        };
        uint32_t E[EXPS];
        exponent(first, E);
        unsigned short *out = (unsigned short *)a.dz + first_row * a.cols + n;
        const uint64_t out_step = ((uint64_t)step * TILE_ROWS - ROWS) * a.cols;
        const bool write = a.dz && n < a.cols;
        {  // W^T, an A operand: a lane has a column, a word two outputs; a warp a quarter of the outputs
            const T *w = (const T *)a.weight + n;
            const uint32_t o0 = set * OC * 16u;
#pragma unroll
            for (uint32_t c = 0; c < OC; ++c) {
                uint32_t v[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; ++i) {
                    const uint32_t o = o0 + c * 16u + 2u * i;
                    const unsigned short *p = (const unsigned short *)(w + o * a.weight_stride);
                    const uint32_t lo = n < a.cols && o < a.outs ? __ldg(p) : 0u;
                    const uint32_t hi = n < a.cols && o + 1u < a.outs ? __ldg(p + a.weight_stride) : 0u;
                    v[i] = lo | hi << 16;
                }
                tc::tmem_store8(tmem + P::W_AT + lanes + (o0 + c * 16u) / 2u, v);
            }
            tc::tmem_wait_store();
            tc::fence_before();
            __syncwarp();
            if (lane == 0) tc::mbar_arrive(&s.w_full);
        }
        tc::Ring r, dh, ready;
        r.skip(set, P::STAGES);
        dh.skip(set, P::BUFS);
        ready.skip(set, P::READY);
        bool ok = true;
        for (uint32_t t = first; t < a.tiles && ok; t += step) {
            uint32_t next_E[EXPS];
            exponent(t + step, next_E);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < EXPS; ++i) scale[i * 32 + lane] = mx8_scale(E[i]);
            __syncwarp();
            ok = __all_sync(~0u, tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
            ok = ok && __all_sync(~0u, tc::mbar_wait(&s.dh_full[ready.i], ready.phase, fail, a.err));
            if (!ok) break;
            tc::fence_after();
            const uint8_t *codes = smem + r.i * P::STAGE + P::DY_BYTES + code0;
            const uint32_t here = dh_at + dh.i * TILE_ROWS + lanes + row0;
            const uint32_t count = t == last ? last_count : ROWS;
#pragma unroll
            for (int p = 0; p < ROWS; p += 16) {
                uint32_t g[16], h[8], d[8];
                tc::tmem_load16(here + p, g);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const uint32_t c0 = codes[(p + 2 * i) * P::CODE_PITCH], c1 = codes[(p + 2 * i + 1) * P::CODE_PITCH];
                    // a code's byte with its sign bit turned, under the exponent of 2^23, is 2^23 + 128 + code
                    const f32x2 sc = *reinterpret_cast<const f32x2 *>(scale + p + 2 * i);
                    const f32x2 z = mul2(add2(pair(__uint_as_float(c0 ^ 0x4b000080u), __uint_as_float(c1 ^ 0x4b000080u)),
                                              both(-8388736.0f)), sc);
                    const f32x2 gp = pair(__uint_as_float(g[2 * i]), __uint_as_float(g[2 * i + 1]));
                    if constexpr (ACT == ACT_RELU) {
                        const float2 v = unpair(z), q = unpair(gp), zero = unpair(mul2(sc, both(0.0f)));  // NaN in a NaN block
                        h[i] = pack2<T>(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f));
                        d[i] = pack2<T>(v.x > 0.0f ? q.x : zero.x, v.y > 0.0f ? q.y : zero.y);
                    } else {
                        f32x2 v, slope;
                        act_pair<ACT, true, true>(z, v, slope);
                        h[i] = pack2<T>(v);
                        d[i] = pack2<T>(ACT == ACT_IDENTITY ? gp : mul2(gp, slope));
                    }
                }
                // the activations go where the dH that this warp has read was
                tc::tmem_store8(here + p, h);
                if (p + 16 == ROWS) {
                    tc::tmem_wait_store();
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive(&s.h_full[dh.i]);
                }
                if (write && count == ROWS) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        out[0] = (unsigned short)d[i];
                        out[a.cols] = (unsigned short)(d[i] >> 16);
                        out += 2 * a.cols;
                    }
                } else if (write) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (p + 2 * i < count) out[0] = (unsigned short)d[i];
                        if (p + 2 * i + 1 < count) out[a.cols] = (unsigned short)(d[i] >> 16);
                        out += 2 * a.cols;
                    }
                }
            }
            out += out_step;
            dh.skip(P::BUFS < 4u ? P::BUFS : 4u, P::BUFS);
            if (P::BUFS < 4u) dh.skip(4u - P::BUFS, P::BUFS);
            ready.skip(4, P::READY);
            r.skip(4, P::STAGES);
#pragma unroll
            for (int i = 0; i < EXPS; ++i) E[i] = next_E[i];
        }
        ok = __all_sync(~0u, ok && tc::mbar_wait(&s.done, 0, fail, a.err));
        tc::fence_after();
        // dW^T, 16 outputs at a time, to its part in memory or, of the only group, to dW
        float *const fold = reinterpret_cast<float *>(smem) + (quad & 1u) * 32u + lane;  // the upper lanes' half: [output][64]
#pragma unroll
        for (uint32_t c = 0; c < OC; ++c) {
            const uint32_t o0 = (set * OC + c) * 16u;
            uint32_t v[16];
            if (ok && (a.dw_parts || a.dw)) tc::tmem_load16(tmem + lanes + o0, v);
            if (ok && a.dw_parts) {
                float *out = a.dw_parts + (((uint64_t)group * a.slabs + slab) * (OC * 64u) + o0) * 128u + quad * 32u + lane;
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) out[i * 128u] = __uint_as_float(v[i]);
            }
            if (a.dw) {
                if (FOLD) {
                    if (ok && quad >= 2u)
#pragma unroll
                        for (uint32_t i = 0; i < 16; ++i) fold[(o0 + i) * 64u] = __uint_as_float(v[i]);
                    asm volatile("bar.sync 1, 512;" ::: "memory");  // the sixteen warps, failed or not
                }
                if (ok && n < a.cols && (!FOLD || quad < 2u))
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i)
                        if (o0 + i < a.outs)
                            ((T *)a.dw)[(uint64_t)(o0 + i) * a.cols + n] = from_f32<T>(__uint_as_float(v[i]) + (FOLD ? fold[(o0 + i) * 64u] : 0.0f));
            }
        }
        if (ok && sums && set < P::MT && set % sharers == slab) {  // a lane has an output; its 16 columns are equal
            uint32_t v[16];
            tc::tmem_load16(tmem + P::DB_AT + set * 16u + lanes, v);
            const uint32_t o = set * 128u + quad * 32u + lane;
            if (a.db_parts && o < OC * 64u) a.db_parts[(uint64_t)group * (OC * 64u) + o] = __uint_as_float(v[0]);
            if (a.db && o < a.outs) ((T *)a.db)[o] = from_f32<T>(__uint_as_float(v[0]));
        }
    }
    __syncwarp();
    tc::fence_before();
    __syncthreads();
    if (warp == 1) tc::tmem_free<P::TMEM>(tmem);
}

// Adds the groups' parts: dw (outs, cols) and db (outs).  A part has 128 columns a slab;
// with one slab of up to 64 (fold) its two halves come from different rows and are added, always in
// the same order.  The blocks after dw's take db.  With many groups (SPLIT 8) a block takes 32 numbers and each of its
// warps every eighth group of them: a thread that added all 148 groups of a number waited 20 us for its loads, now 5
// (177137 x 16 -> 16).  With few, a thread takes a number's groups (3652 x 2311 -> 197, 8 groups: 7 us, split 27).
template <typename T, uint32_t SPLIT>
__global__ void __launch_bounds__(256) narrow_reduce_kernel(const float *__restrict__ dw_parts, const float *__restrict__ db_parts,
                                                            uint32_t groups, uint32_t slabs, uint32_t part_outs, bool fold,
                                                            uint32_t cols, uint32_t outs, T *__restrict__ dw, T *__restrict__ db)
{
    static_assert(SPLIT == 1 || SPLIT == 8, "a block has eight warps");
    __shared__ float sum[8][32];
    const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u;
    const uint32_t first = SPLIT == 1u ? 0u : warp, in_block = SPLIT == 1u ? threadIdx.x : lane;
    const uint64_t per_group = (uint64_t)slabs * part_outs * 128u, at = (uint64_t)blockIdx.x * (256u / SPLIT) + in_block;
    const bool bias = at >= per_group;  // of the whole block
    const uint64_t i = bias ? at - per_group : at, step = bias ? part_outs : per_group;
    const uint32_t o = bias ? (uint32_t)i : (uint32_t)(i / 128u % part_outs);
    const uint32_t n = bias ? 0u : (uint32_t)(i / 128u / part_outs) * 128u + (uint32_t)(i % 128u);
    T *out = bias ? db : dw;
    const bool is = out && o < outs && n < cols;
    const float *p = (bias ? db_parts : dw_parts) + i;
    float v = 0.0f, u = 0.0f;
    if (is) {
#pragma unroll 8
        for (uint32_t g = first; g < groups; g += SPLIT) v += __ldg(p + g * step);
        if (fold && !bias) {
#pragma unroll 8
            for (uint32_t g = first; g < groups; g += SPLIT) u += __ldg(p + g * step + 64u);
        }
    }
    float total = v + u;
    if constexpr (SPLIT > 1u) {
        sum[warp][lane] = total;
        __syncthreads();
        if (warp) return;
        total = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < 8; ++w) total += sum[w][lane];
    }
    if (is) out[bias ? i : (uint64_t)o * cols + n] = from_f32<T>(total);
}

// ---- wider layers ----

constexpr uint32_t WIDE_STAGES = 6, WIDE_STAGE_BYTES = 32768, WIDE_THREADS = 256;
struct WideCtrl {
    uint64_t full[WIDE_STAGES], empty[WIDE_STAGES], acc_full[2], acc_empty[2], failed;
    uint32_t tmem;
    tc::Fail fail;
    uint32_t turn[4][TURN_WORDS];
};
constexpr uint32_t WIDE_SMEM = WIDE_STAGES * WIDE_STAGE_BYTES + sizeof(WideCtrl);

struct WideArgs {
    uint64_t m, n;             // sizes of the product C
    uint32_t m_tiles, n_tiles, tile_n, chunks, splits, chunks_a_split;
    uint32_t blocks;           // of a row of z
    const int8_t *codes;       // dz: the checkpoint
    const uint8_t *exps;
    void *out;                 // dz or dW
    float *parts;              // dW with splits > 1: [split][m][n]
    uint32_t *err;
    bool out_wide;
};

// C = A B on 256 x 256 tiles, 64 steps of k a stage.  DZ: A = dy (K-major), B = W, C = dz after the
// slope.  Otherwise A = dy^T (MN-major: k runs over the rows of dy), B = h, C = dW or, where k is
// split for want of tiles, parts of it.
template <typename T, int ACT, bool DZ>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(WIDE_THREADS, 1)
    wide_kernel(const __grid_constant__ CUtensorMap a_map, const __grid_constant__ CUtensorMap b_map, const WideArgs a)
{
    constexpr bool BF16 = std::is_same<T, __nv_bfloat16>::value;
    extern __shared__ __align__(1024) uint8_t smem[];
    WideCtrl &s = *reinterpret_cast<WideCtrl *>(smem + WIDE_STAGES * WIDE_STAGE_BYTES);
    const uint32_t warp = tc::warp_number(), lane = threadIdx.x % 32u, rank = tc::cluster_rank();
    const uint32_t units = a.m_tiles * a.n_tiles * a.splits, first = blockIdx.x / 2u, step = gridDim.x / 2u;
    const uint32_t half_n = a.tile_n / 2u, b_boxes = half_n > 64u ? 2u : 1u;
    tc::Fail *const fail = &s.fail;

    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < WIDE_STAGES; ++i) {
            tc::mbar_init(&s.full[i], 1);
            tc::mbar_init(&s.empty[i], 1);
        }
        for (uint32_t i = 0; i < 2; ++i) {
            tc::mbar_init(&s.acc_full[i], 1);
            tc::mbar_init(&s.acc_empty[i], 8);
        }
        tc::mbar_init(&s.failed, 1);
        s.fail.failed = 0;
        tc::mbar_init_fence();
        tc::tma_prefetch_map(&a_map);
        tc::tma_prefetch_map(&b_map);
    }
    if (warp == 1) tc::tmem_alloc_pair<512>(&s.tmem);
    tc::fence_before();
    tc::cluster_sync();
    tc::fence_after();
    const uint32_t tmem = s.tmem;

    if (warp == 0) {
        if (lane == 0) {  // TMA, in each CTA; the leader's barriers count both CTAs' bytes
            tc::Ring r;
            bool ok = true;
            for (uint32_t u = first; u < units && ok; u += step) {
                const uint32_t t = u % (a.m_tiles * a.n_tiles), c0 = u / (a.m_tiles * a.n_tiles) * a.chunks_a_split;
                const uint32_t c1 = min(a.chunks, c0 + a.chunks_a_split);
                const int m0 = (int)(t / a.n_tiles * 256u + rank * 128u), n0 = (int)(t % a.n_tiles * a.tile_n + rank * half_n);
                for (uint32_t c = c0; c < c1; ++c) {
                    ok = tc::mbar_wait(&s.empty[r.i], r.phase ^ 1u, fail, a.err);
                    if (!ok) break;
                    uint8_t *st = smem + r.i * WIDE_STAGE_BYTES;
                    const uint32_t bar = tc::leader_addr(&s.full[r.i]);
                    if (rank == 0) tc::mbar_arrive_tx(&s.full[r.i], 2u * (16384u + b_boxes * 8192u));
                    if (DZ) {
                        tc::tma_load_2d_pair(st, &a_map, (int)(c * 64u), m0, bar);
                    } else {
                        tc::tma_load_2d_pair(st, &a_map, m0, (int)(c * 64u), bar);
                        tc::tma_load_2d_pair(st + 8192, &a_map, m0 + 64, (int)(c * 64u), bar);
                    }
                    for (uint32_t b = 0; b < b_boxes; ++b)
                        tc::tma_load_2d_pair(st + 16384 + b * 8192, &b_map, n0 + (int)(b * 64u), (int)(c * 64u), bar);
                    r.next(WIDE_STAGES);
                }
            }
            // The bytes of both CTAs are counted in the leader alone, so after a failure each CTA
            // waits for its copies by time, far longer than they take.
            if (s.fail.failed) tc::outlast_copies();
        }
    } else if (warp == 1) {
        if (rank == 0) {  // products, in the leader
            const uint32_t base = tc::smem_u32(smem), id = tc::idesc_f16<BF16>(256, 0, !DZ, true) | (a.tile_n >> 3) << 17;
            const bool mine = tc::elect();
            tc::Ring r, acc;
            bool ok = true;
            for (uint32_t u = first; u < units && ok; u += step) {
                const uint32_t c0 = u / (a.m_tiles * a.n_tiles) * a.chunks_a_split, c1 = min(a.chunks, c0 + a.chunks_a_split);
                ok = __all_sync(~0u, tc::mbar_wait(&s.acc_empty[acc.i], acc.phase ^ 1u, fail, a.err));
                if (!ok) break;
                tc::fence_after();
                for (uint32_t c = c0; c < c1; ++c) {
                    ok = __all_sync(~0u, tc::mbar_wait(&s.full[r.i], r.phase, fail, a.err));
                    if (!ok) break;
                    tc::fence_after();
                    const uint32_t st = base + r.i * WIDE_STAGE_BYTES;
                    const uint64_t da = DZ ? tc::smem_desc(st, 16, 1024) : tc::smem_desc(st, 8192, 1024), db = tc::smem_desc(st + 16384u, 8192, 1024);
                    if (mine) {
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k)
                            tc::mma_f16_pair(tmem + acc.i * 256u, da + k * (DZ ? 2u : 128u), db + k * 128u, id, c != c0 || k != 0);
                        tc::commit_pair(&s.empty[r.i]);
                        if (c + 1u == c1) tc::commit_pair(&s.acc_full[acc.i]);
                    }
                    __syncwarp();
                    r.next(WIDE_STAGES);
                }
                acc.next(2);
            }
            if (!ok) {  // leave no product in flight
                if (mine) tc::commit_pair(&s.failed);
                tc::mbar_wait_slow(&s.failed, 0, fail, a.err, true);
            }
        }
    } else if (warp >= 4) {  // results: a lane has a row of this CTA's 128
        const uint32_t quad = warp % 4u, in_tile = quad * 32u + lane;
        tc::Ring acc;
        for (uint32_t u = first; u < units; u += step) {
            const uint32_t t = u % (a.m_tiles * a.n_tiles), split = u / (a.m_tiles * a.n_tiles);
            const uint64_t row = (uint64_t)(t / a.n_tiles) * 256u + rank * 128u + in_tile;
            const uint32_t n0 = t % a.n_tiles * a.tile_n;
            const bool ok = tc::mbar_wait(&s.acc_full[acc.i], acc.phase, fail, a.err);
            if (!__all_sync(~0u, ok)) break;
            tc::fence_after();
#pragma unroll 1
            for (uint32_t j = 0; j < a.tile_n; j += 32u) {
                const uint32_t col = n0 + j;
                uint32_t v[32], w[16];
                uint32_t codes[8], E = 127;
                if (DZ) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) codes[i] = 0;
                    if (row < a.m && col < a.n) {
                        const uint64_t b = row * a.blocks + col / 32u;
                        load32(a.codes + b * 32u, codes);
                        E = __ldg(a.exps + b);
                    }
                }
                tc::tmem_load32(tmem + acc.i * 256u + (quad * 32u << 16) + j, v);
                if (j + 32u >= a.tile_n) {
                    tc::fence_before();
                    __syncwarp();
                    if (lane == 0) tc::mbar_arrive_cluster(tc::leader_addr(&s.acc_empty[acc.i]));
                }
                if (!DZ && a.splits > 1) {  // parts: 8 columns at a time if the rows allow it
                    float *p = a.parts + ((uint64_t)split * a.m + row) * a.n + col;
                    if (row >= a.m) {
                    } else if (a.n % 8u == 0) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            if (col + 8u * i < a.n) store32(p + 8u * i, v + 8 * i);
                    } else {
#pragma unroll
                        for (uint32_t i = 0; i < 32; ++i)
                            if (col + i < a.n) p[i] = __uint_as_float(v[i]);
                    }
                    continue;
                }
                if (DZ) {
                    const f32x2 sc = both(mx8_scale(E));
                    slope16<T, ACT>(codes, sc, v, w);
                    slope16<T, ACT>(codes + 4, sc, v + 16, w + 8);
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 16; ++i) w[i] = pack2<T>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
                }
                const uint64_t row0 = row - lane;  // the warp's first
                if (a.out_wide) {
                    if (row < a.m) store_row32<T>((T *)a.out + row * a.n, col, (uint32_t)a.n, w);
                } else {
                    store_turned<T>((T *)a.out + row0 * a.n, row0 >= a.m ? 0u : (uint32_t)min((unsigned long long)(a.m - row0), 32ull), col,
                                    (uint32_t)a.n, w, s.turn[quad]);
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

// h = act(z8) in the operands' type, rows at a pitch of whole 16-byte words.
template <typename T, int ACT>
__global__ void __launch_bounds__(256) activate_kernel(const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps,
                                                       uint64_t rows, uint32_t blocks, uint32_t pitch, T *__restrict__ h)
{
    const uint64_t items = rows * blocks;
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < items * 4u; i += (uint64_t)gridDim.x * 256u) {
        const uint64_t b = i >> 2;
        const uint64_t row = items >> 32 ? b / blocks : (uint32_t)b / blocks;
        const uint32_t col = (uint32_t)(b - row * blocks) * 32u + (uint32_t)(i & 3u) * 8u;
        if (col >= pitch) continue;
        const uint2 c = __ldg(reinterpret_cast<const uint2 *>(codes) + i);
        const f32x2 sc = both(mx8_scale(__ldg(exps + b)));
        uint32_t w[4];
#pragma unroll
        for (int p = 0; p < 4; ++p) {
            const uint32_t x = (p < 2 ? c.x : c.y) ^ 0x80808080u;
            w[p] = pack2<T>(act_value2<ACT>(mul2(code_pair(x, p % 2 * 2), sc)));
        }
        *reinterpret_cast<uint4 *>(h + row * pitch + col) = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

// Column sums of dy in parts: a block takes 256 columns, 8 a lane, and every gridDim.y-th group of 8 rows;
// one part is the result.  Bound by HBM's latency: 31772 x 3104 takes 50 us, 3.9 TB/s, with as many blocks as fit at once
// (62 with half as many again, 89 with two an SM).  `readable` of a row's columns may be loaded: a copy's zeros make its last word whole.
template <typename T>
__global__ void __launch_bounds__(256) column_parts_kernel(const T *__restrict__ dy, uint64_t rows, uint32_t cols, uint32_t readable,
                                                           uint64_t pitch, float *__restrict__ parts, T *__restrict__ out)
{
    __shared__ float sum[8][257];
    const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, col = blockIdx.x * 256u + lane * 8u;
    float v[8] = {};
    const uint32_t step = gridDim.y * 8u, have = col >= readable ? 0u : readable - col < 8u ? readable - col : 8u;
    const auto add = [&](const Vec8<T> &x) {
        float f[8];
        x.unpack(f);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += f[i];
    };
    const auto load = [&](Vec8<T> &x, const T *p) {
        if (have == 8u) {
            x.load(p);
        } else {
            x.zero();
#pragma unroll
            for (uint32_t i = 0; i < 7; ++i)
                if (i < have) reinterpret_cast<T *>(x.w)[i] = p[i];
        }
    };
    uint64_t row = blockIdx.y * 8u + warp;
    const T *p = dy + row * pitch + col;
    if (have) {
        // four rows' loads before the first sum
        for (; row + 3ull * step < rows; row += 4ull * step, p += 4ull * step * pitch) {
            Vec8<T> x[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) load(x[i], p + (uint64_t)i * step * pitch);
#pragma unroll
            for (int i = 0; i < 4; ++i) add(x[i]);
        }
        for (; row < rows; row += step, p += (uint64_t)step * pitch) {
            Vec8<T> x;
            load(x, p);
            add(x);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) sum[warp][lane * 8u + i] = v[i];
    __syncthreads();
    const uint32_t c = blockIdx.x * 256u + threadIdx.x;
    float total = 0.0f;
    for (int w = 0; w < 8; ++w) total += sum[w][threadIdx.x];
    if (c >= cols) return;
    if (gridDim.y == 1) out[c] = from_f32<T>(total);
    else parts[(uint64_t)blockIdx.y * cols + c] = total;
}

// Column sums in one launch, for the rare matrix that no other kernel reads.
template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const T *__restrict__ p, uint64_t rows, uint32_t cols, uint64_t stride, T *__restrict__ out)
{
    __shared__ float part[256];
    float v = 0.0f;
    for (uint64_t i = threadIdx.x; i < rows; i += 256u) v += to_f32<T>(p[i * stride + blockIdx.x]);
    part[threadIdx.x] = v;
    __syncthreads();
    for (int n = 128; n; n >>= 1) {
        if (threadIdx.x < n) part[threadIdx.x] += part[threadIdx.x + n];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[blockIdx.x] = from_f32<T>(part[0]);
}

// out = the parts added in order
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float *__restrict__ parts, uint32_t count, uint64_t n, T *__restrict__ out)
{
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n; i += (uint64_t)gridDim.x * 256u) {
        float v = 0.0f;
#pragma unroll 16  // loads under way at once: few threads, many parts
        for (uint32_t p = 0; p < count; ++p) v += __ldg(parts + p * n + i);
        out[i] = from_f32<T>(v);
    }
}

// The same for few numbers of many parts: a block takes 32 numbers, a warp every eighth part of them, always in this order
template <typename T>
__global__ void __launch_bounds__(256) add_many_parts_kernel(const float *__restrict__ parts, uint32_t count, uint32_t n, T *__restrict__ out)
{
    __shared__ float sum[8][32];
    const uint32_t lane = threadIdx.x % 32u, warp = threadIdx.x / 32u, i = blockIdx.x * 32u + lane;
    float v = 0.0f;
    if (i < n) {
#pragma unroll 8
        for (uint32_t p = warp; p < count; p += 8u) v += __ldg(parts + (uint64_t)p * n + i);
    }
    sum[warp][lane] = v;
    __syncthreads();
    if (warp || i >= n) return;
    float total = 0.0f;
#pragma unroll
    for (uint32_t w = 0; w < 8; ++w) total += sum[w][lane];
    out[i] = from_f32<T>(total);
}

// Operands whose rows do not start on 16 bytes are copied
enum : int { COPY_DY = 1, COPY_WEIGHT = 2 };

// How a narrow call is cut, and where its workspace parts lie.
struct NarrowPlan {
    uint32_t oc, slabs, tiles, groups, part_outs;
    bool fold;
    uint64_t dw_at, db_at, dy_at, bytes;
};
static NarrowPlan narrow_plan(uint64_t rows, uint32_t cols, uint32_t outs, int copies, uint32_t sms)
{
    NarrowPlan p;
    p.oc = (outs + 63u) / 64u;
    p.fold = cols <= 64u;
    p.slabs = (cols + 127u) / 128u;
    const uint32_t tile_rows = narrow_rows(p.oc);
    p.tiles = (uint32_t)((rows + tile_rows - 1u) / tile_rows);
    // one CTA an SM; a slab more than there are SMs still gets its own
    // and few tiles are one group's: a CTA takes a tile every 0.4 us, less in all than a second kernel
    p.groups = p.slabs < sms && p.tiles > 16u ? sms / p.slabs : 1u;
    if (p.groups > p.tiles) p.groups = p.tiles;
    const bool parts = p.groups > 1u;
    p.part_outs = p.oc * 64u;
    p.dw_at = 0;
    p.db_at = p.dw_at + (parts ? align_up((uint64_t)p.groups * p.slabs * 128u * p.part_outs * 4u, 256) : 0);
    p.dy_at = p.db_at + (parts ? align_up((uint64_t)p.groups * p.part_outs * 4u, 256) : 0);
    p.bytes = p.dy_at + (copies & COPY_DY && outs > TINY_OUTS ? align_up(rows * align_up(outs, 8) * 2u, 256) : 0);
    return p;
}

template <typename T> static int copies_of(const void *dy, uint64_t dy_stride, const void *w, uint64_t w_stride)
{
    return (whole_words<T>(dy, dy_stride) ? 0 : COPY_DY) | (whole_words<T>(w, w_stride) ? 0 : COPY_WEIGHT);
}

template <typename T, int ACT, int OC, bool FOLD>
static vt_status launch_narrow(const CUtensorMap &dy, const NarrowArgs &a, cudaStream_t stream)
{
    static std::atomic<uint64_t> allowed{0};
    using P = Narrow<OC, FOLD>;
    CUtensorMap codes;
    const uint64_t width = (uint64_t)a.blocks * 32u;
    if (vt_status s = tc::make_map(&codes, CU_TENSOR_MAP_DATA_TYPE_UINT8, a.codes, a.rows, width, width, P::TILE_ROWS, P::CODE_PITCH, false))
        return s;
    if (vt_status s = tc::allow_smem(narrow_kernel<T, ACT, OC, FOLD>, P::SMEM, allowed)) return s;
    narrow_kernel<T, ACT, OC, FOLD><<<a.groups * a.slabs, NARROW_THREADS, P::SMEM, stream>>>(dy, codes, a);
    return check_launch("narrow_kernel");
}

template <typename T, int ACT>
static vt_status run_narrow(const void *dy, uint64_t dy_stride, const void *w, uint64_t w_stride, uint64_t rows, uint32_t cols,
                            uint32_t outs, const int8_t *codes, const uint8_t *exps, void *dz, void *dw, void *db,
                            uint8_t *workspace, uint32_t *err, cudaStream_t stream)
{
    const NarrowPlan p = narrow_plan(rows, cols, outs, copies_of<T>(dy, dy_stride, w, w_stride), (uint32_t)sm_count());
    CUtensorMap dy_map = {};
    const bool tiny = outs <= TINY_OUTS;
    if (!tiny)
        if (vt_status s = whole_rows<T>(dy, dy_stride, rows, outs, workspace + p.dy_at, stream)) return s;
    const bool chunked = outs % 64u == 0 && outs > 64u;
    if (vt_status s = tiny ? VT_OK : chunked ? tc::make_chunk_map(&dy_map, tma_type<T>(), dy, rows, p.oc, dy_stride * sizeof(T), narrow_rows(p.oc), 64, sizeof(T))
                              : map_rows<T>(&dy_map, dy, dy_stride, rows, outs, narrow_rows(p.oc)))
        return s;
    NarrowArgs a;
    a.dy = tiny ? dy : nullptr;
    a.dy_stride = dy_stride;
    a.codes_whole = mx_blocks(cols) * 32u == (p.fold ? 64u : 128u);
    a.dy_chunked = chunked;
    a.weight = w;
    a.weight_stride = w_stride;
    a.rows = rows;
    a.cols = cols;
    a.outs = outs;
    a.blocks = mx_blocks(cols);
    a.tiles = p.tiles;
    a.groups = p.groups;
    a.slabs = p.slabs;
    a.codes = codes;
    a.exps = exps;
    a.dz = dz;
    const bool parts = p.groups > 1u;
    a.dw_parts = dw && parts ? (float *)(workspace + p.dw_at) : nullptr;
    a.db_parts = db && parts ? (float *)(workspace + p.db_at) : nullptr;
    a.dw = parts ? nullptr : dw;
    a.db = parts ? nullptr : db;
    a.err = err;
    vt_status s = VT_OK;
    switch (p.oc * 2u + p.fold) {
    case 2: s = launch_narrow<T, ACT, 1, false>(dy_map, a, stream); break;
    case 3: s = launch_narrow<T, ACT, 1, true>(dy_map, a, stream); break;
    case 4: s = launch_narrow<T, ACT, 2, false>(dy_map, a, stream); break;
    case 5: s = launch_narrow<T, ACT, 2, true>(dy_map, a, stream); break;
    case 6: s = launch_narrow<T, ACT, 3, false>(dy_map, a, stream); break;
    case 7: s = launch_narrow<T, ACT, 3, true>(dy_map, a, stream); break;
    case 8: s = launch_narrow<T, ACT, 4, false>(dy_map, a, stream); break;
    default: s = launch_narrow<T, ACT, 4, true>(dy_map, a, stream); break;
    }
    if (s || !parts || !(dw || db)) return s;
    const uint64_t n = (uint64_t)p.slabs * 128u * p.part_outs + p.part_outs;
    if (p.groups >= 32u)
        narrow_reduce_kernel<T, 8><<<(unsigned)((n + 31u) / 32u), 256, 0, stream>>>(a.dw_parts, a.db_parts, p.groups, p.slabs, p.part_outs,
                                                                                   p.fold, cols, outs, (T *)dw, (T *)db);
    else
        narrow_reduce_kernel<T, 1><<<(unsigned)((n + 255u) / 256u), 256, 0, stream>>>(a.dw_parts, a.db_parts, p.groups, p.slabs,
                                                                                     p.part_outs, p.fold, cols, outs, (T *)dw, (T *)db);
    return check_launch("narrow_reduce_kernel");
}

// How a wide call is cut, and where its workspace parts lie.
struct WidePlan {
    uint32_t splits, chunks_a_split, sum_parts;
    uint64_t h_at, dw_at, db_at, dy_at, w_at, bytes;
};
static uint32_t wide_tile_n(uint32_t cols) { return cols >= 256u ? 256u : (cols + 31u) / 32u * 32u; }
static WidePlan wide_plan(uint64_t rows, uint32_t cols, uint32_t outs, int copies, uint32_t sms)
{
    WidePlan p;
    const uint32_t tn = wide_tile_n(cols), chunks = (uint32_t)((rows + 63u) / 64u);
    const uint64_t tiles = (uint64_t)((outs + 255u) / 256u) * ((cols + tn - 1u) / tn);
    // with fewer tiles than pairs of SMs the rows are split, down to 8 stages a split
    const uint64_t room = tiles < sms / 2u ? sms / 2u / tiles : 1u, most = (chunks + 7u) / 8u;
    p.splits = (uint32_t)(room < most ? room : most);
    p.chunks_a_split = (chunks + p.splits - 1u) / p.splits;
    p.splits = (chunks + p.chunks_a_split - 1u) / p.chunks_a_split;
    const uint64_t across = (outs + 255u) / 256u, most_parts = 4u * sms < across ? 1u : 4u * sms / across;  // four blocks an SM: one round
    p.sum_parts = (uint32_t)((rows + 255u) / 256u < most_parts ? (rows + 255u) / 256u : most_parts);
    p.h_at = 0;
    p.dw_at = p.h_at + align_up(rows * align_up(cols, 8) * 2u, 256);
    p.db_at = p.dw_at + (p.splits > 1 ? align_up((uint64_t)p.splits * outs * cols * 4u, 256) : 0);
    p.dy_at = p.db_at + align_up((uint64_t)p.sum_parts * outs * 4u, 256);
    p.w_at = p.dy_at + (copies & COPY_DY ? align_up(rows * align_up(outs, 8) * 2u, 256) : 0);
    p.bytes = p.w_at + (copies & COPY_WEIGHT ? align_up((uint64_t)outs * align_up(cols, 8) * 2u, 256) : 0);
    return p;
}

template <typename T, int ACT, bool DZ>
static vt_status launch_wide(const CUtensorMap &ma, const CUtensorMap &mb, const WideArgs &a, uint32_t sms, cudaStream_t stream)
{
    static std::atomic<uint64_t> allowed{0};
    if (vt_status s = tc::allow_smem(wide_kernel<T, ACT, DZ>, WIDE_SMEM, allowed)) return s;
    const uint64_t units = (uint64_t)a.m_tiles * a.n_tiles * a.splits;
    VT_REQUIRE(units < (1ull << 31), "vt_mx8_linear_bwd: too many tiles");
    const unsigned pairs = (unsigned)(units < sms / 2u ? units : sms / 2u);
    wide_kernel<T, ACT, DZ><<<pairs * 2u, WIDE_THREADS, WIDE_SMEM, stream>>>(ma, mb, a);
    return check_launch("wide_kernel");
}

template <typename T, int ACT>
static vt_status run_wide(const void *dy, uint64_t dy_stride, const void *w, uint64_t w_stride, uint64_t rows, uint32_t cols,
                          uint32_t outs, const int8_t *codes, const uint8_t *exps, void *dz, void *dw, void *db,
                          uint8_t *workspace, uint32_t *err, cudaStream_t stream)
{
    const uint32_t sms = (uint32_t)sm_count();
    const WidePlan p = wide_plan(rows, cols, outs, copies_of<T>(dy, dy_stride, w, w_stride), sms);
    if (vt_status s = whole_rows<T>(dy, dy_stride, rows, outs, workspace + p.dy_at, stream)) return s;
    WideArgs a = {};
    a.tile_n = wide_tile_n(cols);
    a.n_tiles = (cols + a.tile_n - 1u) / a.tile_n;
    a.n = cols;
    a.blocks = mx_blocks(cols);
    a.codes = codes;
    a.exps = exps;
    a.err = err;
    const uint32_t readable = dy == workspace + p.dy_at ? (uint32_t)dy_stride : outs;
    CUtensorMap ma, mb;
    if (dz) {
        if (vt_status s = whole_rows<T>(w, w_stride, outs, cols, workspace + p.w_at, stream)) return s;
        if (vt_status s = map_rows<T>(&ma, dy, dy_stride, rows, outs, 128)) return s;
        if (vt_status s = map_rows<T>(&mb, w, w_stride, outs, cols, 64)) return s;
        a.m = rows;
        a.m_tiles = (uint32_t)((rows + 255u) / 256u);
        a.chunks = a.chunks_a_split = (outs + 63u) / 64u;
        a.splits = 1;
        a.out = dz;
        a.out_wide = cols % 16u == 0 && aligned32(dz);
        if (vt_status s = launch_wide<T, ACT, true>(ma, mb, a, sms, stream)) return s;
    }
    if (dw) {
        T *h = (T *)(workspace + p.h_at);
        const uint32_t pitch = (uint32_t)align_up(cols, 8);
        const uint64_t want = (rows * a.blocks * 4u + 255u) / 256u;
        activate_kernel<T, ACT><<<(unsigned)(want < sms * 32u ? want : sms * 32u), 256, 0, stream>>>(codes, exps, rows, a.blocks, pitch, h);
        if (vt_status s = check_launch("activate_kernel")) return s;
        if (vt_status s = map_rows<T>(&ma, dy, dy_stride, rows, outs, 64)) return s;
        if (vt_status s = map_rows<T>(&mb, h, pitch, rows, cols, 64)) return s;
        a.m = outs;
        a.m_tiles = (outs + 255u) / 256u;
        a.chunks = (uint32_t)((rows + 63u) / 64u);
        a.chunks_a_split = p.chunks_a_split;
        a.splits = p.splits;
        a.out = dw;
        a.parts = (float *)(workspace + p.dw_at);
        a.out_wide = cols % 16u == 0 && aligned32(dw);
        if (vt_status s = launch_wide<T, ACT_IDENTITY, false>(ma, mb, a, sms, stream)) return s;
        if (p.splits > 1) {
            const uint64_t n = (uint64_t)outs * cols, blocks = (n + 255u) / 256u;
            add_parts_kernel<T><<<(unsigned)(blocks < sms * 8u ? blocks : sms * 8u), 256, 0, stream>>>(a.parts, p.splits, n, (T *)dw);
            if (vt_status s = check_launch("add_parts_kernel")) return s;
        }
    }
    if (db) {
        float *parts = (float *)(workspace + p.db_at);
        column_parts_kernel<T><<<dim3((outs + 255u) / 256u, p.sum_parts), 256, 0, stream>>>((const T *)dy, rows, outs, readable, dy_stride, parts,
                                                                                             (T *)db);
        if (p.sum_parts > 1) add_many_parts_kernel<T><<<(outs + 31u) / 32u, 256, 0, stream>>>(parts, p.sum_parts, outs, (T *)db);
        if (vt_status s = check_launch("column_parts_kernel")) return s;
    }
    return VT_OK;
}

template <typename T>
static vt_status zero(T *p, uint64_t n, cudaStream_t stream)
{
    if (!p || !n) return VT_OK;
    cudaError_t e = cudaMemsetAsync(p, 0, n * sizeof(T), stream);
    return e == cudaSuccess ? VT_OK : set_error(VT_ERR_CUDA, "cudaMemsetAsync: %s", cudaGetErrorString(e));
}

}  // namespace vt

extern "C" uint64_t vt_mx8_linear_bwd_workspace_bytes(uint64_t rows, uint32_t cols, uint32_t outs, int copies)
{
    if (rows == 0 || cols == 0 || outs == 0) return 0;
    const uint32_t sms = (uint32_t)vt::sm_count();
    return outs <= vt::NARROW_OUTS ? vt::narrow_plan(rows, cols, outs, copies, sms).bytes
                                   : vt::wide_plan(rows, cols, outs, copies, sms).bytes;
}

extern "C" vt_status vt_mx8_linear_bwd(const void *dy, uint64_t dy_stride, const void *weight, uint64_t weight_stride,
                                       int dtype, uint64_t rows, uint32_t cols, uint32_t outs, const int8_t *codes,
                                       const uint8_t *exps, int act, void *dz, void *dw, void *db, void *workspace,
                                       uint64_t workspace_bytes, uint32_t *err, vt_stream stream)
{
    VT_REQUIRE(rows <= (1ull << 31) - 256, "vt_mx8_linear_bwd: too many rows");
    VT_REQUIRE(cols <= (1u << 20) && outs <= (1u << 20), "vt_mx8_linear_bwd: layer too wide");
    cudaStream_t st = (cudaStream_t)stream;
    return vt::with_type16(dtype, [&](auto ty) -> vt_status {
        using T = typename decltype(ty)::type;
        if (rows == 0 || cols == 0 || outs == 0) {
            if (vt_status s = vt::zero((T *)dz, rows * cols, st)) return s;
            if (vt_status s = vt::zero((T *)dw, (uint64_t)outs * cols, st)) return s;
            if (rows == 0 || outs == 0) return vt::zero((T *)db, outs, st);
            if (!db) return VT_OK;
        }
        VT_REQUIRE(dy && (cols == 0 || (weight && codes && exps)), "vt_mx8_linear_bwd: null pointer");
        VT_REQUIRE(vt::on_elements<T>(dy, weight, dz, dw, db), "vt_mx8_linear_bwd: a matrix does not start on an element");
        VT_REQUIRE(dy_stride >= outs && weight_stride >= cols,
                   "vt_mx8_linear_bwd: a row stride is less than a row");
        VT_REQUIRE(vt::aligned32(codes), "vt_mx8_linear_bwd: codes must be 32-byte aligned");
        VT_REQUIRE(workspace_bytes >= vt_mx8_linear_bwd_workspace_bytes(rows, cols, outs, vt::copies_of<T>(dy, dy_stride, weight, weight_stride)) &&
                       vt::aligned32(workspace),
                   "vt_mx8_linear_bwd: workspace too small or not 32-byte aligned");  // parts are stored 32 bytes at a time
        if (cols == 0) {  // a layer without inputs has the bias alone
            vt::column_sum_kernel<T><<<outs, 256, 0, st>>>((const T *)dy, rows, outs, dy_stride, (T *)db);
            return vt::check_launch("column_sum_kernel");
        }
        return vt::with_act(act, [&](auto a) -> vt_status {
            constexpr int ACT = decltype(a)::value;
            if (outs <= vt::NARROW_OUTS)
                return vt::run_narrow<T, ACT>(dy, dy_stride, weight, weight_stride, rows, cols, outs, codes, exps, dz, dw, db,
                                              (uint8_t *)workspace, err, st);
            return vt::run_wide<T, ACT>(dy, dy_stride, weight, weight_stride, rows, cols, outs, codes, exps, dz, dw, db,
                                        (uint8_t *)workspace, err, st);
        });
    });
}

// Grouped product of e4m3 rows and e4m3 expert weights on the tcgen05 tensor cores:
//
//   out[m, n] = sum over blocks b of 128 columns of  sa[m, b] * sw[e, n / 128, b] * (sum over k in b of a[m, k] * w[e, n, k])
//
// plain (times a factor per row) or silu(gate) * up, to bf16 or to e4m3 with a scale for each 128 output columns.
//
// The scales are any 32-bit values, so the tensor cores sum one block of 128 columns at a time into TMEM and the epilogue warps add it, scaled,
// to sums that stay in their registers.  Rows are the M operand: a thread owns a row, its scale is one register, and a block costs it
// one multiply-add per column.  (Experts of few rows: fp8_gemm_few_sm100.cu.)
//
// A CTA computes 128 rows x 256 weight rows (tcgen05.mma, N = 256) with two block sums of 256 columns in TMEM, so that the MMAs of a block run
// under the multiply-adds of the one before.  With SwiGLU the weight rows are 64 gate rows, their 64 up rows and again 64 of each, which puts
// both factors of an output into the same thread.
//
// What bounds it.  Experts up to 128 rows: the weights' way from memory (32 experts of 7168 x 2048: 64 rows each up 174 us = 5.4 TB/s, down 99 us).  More: a
// block of 128 columns, 512 cycles of MMA, takes 0.64 to 0.70 us.  0.37 us of that are the operands' way (48 KB, 68 bytes a cycle), 0.48 us that
// and the MMAs, which read 48 KB of the same shared memory, and the rest that an epilogue warp gets through 128 columns in 0.6 us:
// under this traffic a load from shared memory or a look at a barrier takes 200 to 300 cycles.  Hence: no fence where a value read says
// enough, scales and the next block's state asked for a block ahead, the tile's description left by the warp that loads the scales.
// In a long run the power limit (1000 W, 1.6 GHz): 32 x (1024 +- 32) rows up 1340 us = 1.44 PFLOP/s of real rows, down 650 us.
//
// Tried: pairs of CTAs (cta_group::2, 256 rows, two thirds of the operand traffic): 0.69 us a block as well, with a signal between the CTAs in every
// block; at 128 rows an expert half of a pair is idle (up 257 us instead of 188).  Two columns per instruction (fma.rn.f32x2): no faster, and
// the pairs need registers.  Scales by plain loads: 0.6 us a block more.  32 columns twice in flight: registers spill.
//
// All waits are bounded; on expiry a CTA records a code in `status`, stops issuing work, waits for its own copies and frees its TMEM.
#include "fp8_gemm_sm100.hpp"

#include "fp8_prim.cuh"
#include "launch_once.hpp"
#include "row_prim.cuh"
#include "tc_prim.cuh"

namespace nep {
namespace fp8 {
namespace {

using namespace gemm::tc;
using namespace rows;

constexpr int kTileRows = 128;
constexpr int kTileCols = 256;                   // weight rows
constexpr int kRowBytes = kTileRows * 128, kWeightBytes = kTileCols * 128;
constexpr int kStageBytes = kRowBytes + kWeightBytes;
constexpr int kStages = 3;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;   // a warpgroup that loads and issues, two that add up
// A launch of 384 threads gives each 168 registers.  The sums need more: 56 + 2 * 224 = 3 * 168, what the block was launched with.
constexpr int kFewRegisters = 56, kManyRegisters = 224;
static_assert(128 * kFewRegisters + 32 * kEpiWarps * kManyRegisters <= kThreads * 168, "registers of the launch");
constexpr int kTmemCols = 512;
constexpr int kPiecePitch = 256 + 16;            // a thread's part of an output row on its way out: 8 rows hit all banks once
constexpr uint32_t kInstrDesc = instr_desc_e4m3(kTileRows, kTileCols);

struct Shared {
    alignas(16) uint8_t piece[kEpiWarps][32 * kPiecePitch];
    int4 tile[2];                                  // of the chunk's blocks: expert, first row, rows, weight tile
    float row_scales[2][kScaleBlocks][kTileRows];  // of the next blocks, by turns
    float weight_scales[2][kScaleBlocks][2];       // of the tile's two halves (of the gate and up rows)
    float most[kExchangeTurns][2][kTileRows];      // largest of each row's 64 columns, by turn and epilogue group
    uint64_t full[kStages], done[kStages], tmem_empty[2];
    uint64_t scale_full[2], scale_empty[2];
    uint64_t told[kExchangeTurns][2][4];           // by the same, and quarter: its rows' largest values are in `most`
    uint32_t tmem_base;
    int abort;
    int first_tile[kMaxExperts + 1];               // exclusive prefix of row tiles
};
constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + sizeof(Shared);
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

struct Tile {
    int expert, row0, rows, nt;
};
// The row tiles that share a weight tile are neighbours: the weights come from memory once and from L2 afterwards.
__device__ __forceinline__ Tile tile_of(const Shared& sh, const Args& args, int unit, int expert) {
    const int tiles = sh.first_tile[expert + 1] - sh.first_tile[expert], j = unit - sh.first_tile[expert] * args.n_tiles;
    int64_t first, n;
    expert_range(args, expert, first, n);
    const int start = j % tiles * kTileRows;
    return Tile{expert, int(first) + start, min(kTileRows, int(n) - start), j / tiles};
}
__device__ __forceinline__ Tile locate(const Shared& sh, const Args& args, int unit) {
    const int at = unit / args.n_tiles;
    int lo = 0, hi = args.experts;  // first_tile[lo] <= at < first_tile[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sh.first_tile[mid] <= at) lo = mid; else hi = mid;
    }
    return tile_of(sh, args, unit, lo);
}
// The same by a whole warp: 32 places at a look.
__device__ __forceinline__ Tile locate_warp(const Shared& sh, const Args& args, int unit, int lane) {
    const int at = unit / args.n_tiles;
    int lo = 0;
    for (int step = args.experts > 32 ? 32 : 1; step >= 1; step /= 32) {
        const int e = lo + lane * step;
        lo += step * (__popc(__ballot_sync(0xffffffffu, e < args.experts && sh.first_tile[e] <= at)) - 1);
    }
    return tile_of(sh, args, unit, lo);
}

// A row's piece leaves by a copy of its thread's own: whole sectors, and nothing waits for them but the piece's next use.
__device__ __forceinline__ void send_piece(void* dst, const void* piece, int bytes) {
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(smem_u32(piece)), "r"(bytes) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
__device__ __forceinline__ void pieces_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
template <int kRegisters>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters)); }
template <int kRegisters>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters)); }

template <bool kSwiGLU, bool kQuantize>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args args) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem + kStages * kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint64_t limit_ns = args.timeout_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.done[s], 1);  // one commit: the stage is free and its block sums are in TMEM
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh.tmem_empty[b], kEpiWarps);
            mbar_init(&sh.scale_full[b], 1);
            mbar_init(&sh.scale_empty[b], kEpiWarps);
        }
        for (int q = 0; q < kExchangeTurns * 8; ++q) mbar_init(&sh.told[q >> 3][q >> 2 & 1][q & 3], 1);
        sh.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    __syncthreads();  // the abort flag is clear before anyone sets it
    for (int e = threadIdx.x; e < args.experts; e += kThreads) {
        int64_t first, n;
        if (!expert_range(args, e, first, n)) {
            sh.abort = 1;
            if (atomicCAS(args.status, 0u, uint32_t(kBadOffsets)) == 0u) args.status[1] = uint32_t(e);
        }
        sh.first_tile[e] = int((n + kTileRows - 1) / kTileRows);
    }
    if (warp == 1) tmem_alloc(&sh.tmem_base, kTmemCols);
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int base = 0; base < args.experts; base += 32) {
            const int e = base + lane;
            const int tiles = e < args.experts && !sh.abort ? sh.first_tile[e] : 0;
            int incl = tiles;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int v = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= d) incl += v;
            }
            if (e < args.experts) sh.first_tile[e] = carry + incl - tiles;
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
        if (lane == 0) sh.first_tile[args.experts] = carry;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = sh.tmem_base;

    const int k_blocks = args.k_blocks;
    const int units = sh.first_tile[args.experts] * args.n_tiles;  // none after bad offsets
    volatile int* abort_flag = &sh.abort;
    auto fail = [&](uint32_t code) {
        *abort_flag = 1;
        if (atomicCAS(args.status, 0u, code) == 0u) args.status[1] = blockIdx.x;
    };

    if (warp < 4) {
    give_registers<kFewRegisters>();
    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            int64_t issued = 0;
            for (int unit = int(blockIdx.x); unit < units && !*abort_flag; unit += int(gridDim.x)) {
                const Tile t = locate(sh, args, unit);
                // rows that exist, in 16s; what the others' places hold reaches only their own sums
                const int n = (t.rows + 15) & ~15;
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!wait_block(&sh.done[stage], phase ^ 1u, limit_ns, abort_flag)) {
                        fail(kPipeTimeout);
                        break;
                    }
                    uint8_t *dst = smem + stage * kStageBytes, *w_dst = dst + kRowBytes;
                    mbar_expect_tx(&sh.full[stage], uint32_t(kWeightBytes + n * 128));
                    if (kSwiGLU) {  // 64 gate rows, their 64 up rows, and again
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            tma_load_3d(w_dst + q * 64 * 128, &maps.weights, kb * 128, t.nt * 128 + (q >> 1) * 64, 2 * t.expert + (q & 1), &sh.full[stage]);
                    } else {
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            tma_load_3d(w_dst + q * 128 * 128, &maps.weights, kb * 128, t.nt * kTileCols + q * 128, t.expert, &sh.full[stage]);
                    }
                    int at = 0;  // boxes of 128, 64, 32 and 16 rows make up any multiple of 16
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int box = 128 >> b;
                        if (n & box) {
                            tma_load_2d(dst + at * 128, &maps.rows[b], kb * 128, t.row0 + at, &sh.full[stage]);
                            at += box;
                        }
                    }
                    ++issued;
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
            if (*abort_flag)  // a kernel that gave up does not end under its own copies
                for (int64_t i = max(int64_t(0), issued - kStages); i < issued; ++i)
                    mbar_wait(&sh.full[i % kStages], uint32_t(i / kStages) & 1u, min(limit_ns, uint64_t(100000000)));
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer
        if (elect_one()) {
            int stage = 0, block = 0;
            uint32_t phase = 0;
            bool loaded = false;  // as of the block before: a look at a barrier takes 190 cycles, under the MMAs none
            for (int unit = int(blockIdx.x); unit < units && !*abort_flag; unit += int(gridDim.x)) {
                for (int kb = 0; kb < k_blocks; ++kb, ++block) {
                    const int buf = block & 1, s = stage;
                    if ((!loaded && !wait_block(&sh.full[stage], phase, limit_ns, abort_flag)) ||
                        !wait_block(&sh.tmem_empty[buf], (uint32_t(block >> 1) & 1u) ^ 1u, limit_ns, abort_flag)) {
                        fail(kPipeTimeout);
                        break;
                    }
                    tc_fence_after();
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    loaded = block_done(&sh.full[stage], phase);
                    const uint8_t* tile = smem + s * kStageBytes;
                    const uint64_t a_desc = smem_desc_sw128(tile), b_desc = smem_desc_sw128(tile + kRowBytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k)  // 32 values = 32 bytes inside the 128-byte swizzle row
                        mma_e4m3(tmem_base + uint32_t(buf * kTileCols), a_desc + uint64_t(k * 2), b_desc + uint64_t(k * 2), kInstrDesc, k != 0 ? 1u : 0u);
                    // One barrier per stage tells both the producer and the epilogue.  The epilogue has seen a block before the stage's next one can
                    // be done: that one waits for its TMEM columns.
                    tc_commit(&sh.done[s]);
                }
            }
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------------ scales
        // Eight blocks at a time and up to sixteen ahead: the epilogue warps have no registers left to wait for memory.
        constexpr int kHalves = kSwiGLU ? 2 : 1;
        int chunk = 0;
        bool ok = true;
        for (int unit = int(blockIdx.x); unit < units && ok; unit += int(gridDim.x)) {
            const Tile t = locate_warp(sh, args, unit, lane);
            // 128 weight rows share a scale: the two halves of the tile, or those of its gate and up rows
            const int half = lane & 1, block = kSwiGLU ? half * args.n_blocks + t.nt : min(2 * t.nt + half, args.n_blocks - 1);
            const float* sw = args.w_scales + (int64_t(t.expert) * kHalves * args.n_blocks + block) * k_blocks;
            for (int kb0 = 0; kb0 < k_blocks; kb0 += kScaleBlocks, ++chunk) {
                const float w = kb0 + (lane >> 1) < k_blocks && lane < 2 * kScaleBlocks ? sw[kb0 + (lane >> 1)] : 0.f;
                const int slot = chunk & 1;
                for (int i = 0; i < 4; ++i) {  // a row a lane at a time, for want of registers
                    const int r = i * 32 + lane;
                    const float* sa = args.a_scales + (int64_t(t.row0) + r) * k_blocks + kb0;
                    float v[kScaleBlocks];
#pragma unroll
                    for (int j = 0; j < kScaleBlocks; ++j) v[j] = r < t.rows && kb0 + j < k_blocks ? sa[j] : 0.f;
                    if (i == 0) ok = __all_sync(0xffffffffu, wait_block(&sh.scale_empty[slot], (uint32_t(chunk >> 1) & 1u) ^ 1u, limit_ns, abort_flag));
                    if (!ok) break;
#pragma unroll
                    for (int j = 0; j < kScaleBlocks; ++j) sh.row_scales[slot][j][r] = v[j];
                }
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
                if (lane < 2 * kScaleBlocks) sh.weight_scales[slot][lane >> 1][half] = w;
                if (lane == 0) sh.tile[slot] = make_int4(t.expert, t.row0, t.rows, t.nt);
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.scale_full[slot]);
            }
        }
    }
    } else {
        // ------------------------------------------------------------------ epilogue
        take_registers<kManyRegisters>();
        const int quarter = warp & 3;        // TMEM lanes [32 * quarter, +32) belong to this warp
        const int group = (warp - 4) >> 2;   // its 128 columns
        const int r = quarter * 32 + lane;   // row of this CTA's tile
        const uint32_t empty_addr = smem_u32(&sh.tmem_empty[0]);
        uint8_t* piece = sh.piece[warp - 4] + lane * kPiecePitch;  // this thread's row
        int block = 0, stage = 0, chunk = 0, exchanges = 0;
        uint32_t phase = 0;
        bool ok = true;
        // Under the MMAs' operand traffic an access to shared memory takes 200 to 300 cycles, a look at a barrier as well: scales and the state of
        // the next block are asked for while a block is added, the next tile's while a tile leaves, and used behind it.
        float sr = 0.f, sw0 = 0.f, sw1 = 0.f;
        auto fetch_scales = [&](int kb) {
            const int at = kb % kScaleBlocks, slot = chunk & 1;
            if (at == 0) {
                ok = __all_sync(0xffffffffu, wait_block(&sh.scale_full[slot], uint32_t(chunk >> 1) & 1u, limit_ns, abort_flag)) && ok;
                if (!ok && lane == 0) fail(kPipeTimeout);
            }
            sr = sh.row_scales[slot][at][r];
            sw0 = sh.weight_scales[slot][at][kSwiGLU ? 0 : group];
            if (kSwiGLU) sw1 = sh.weight_scales[slot][at][1];
        };
        int4 told = make_int4(0, 0, 0, 0);  // the tile: the warp that loads the scales knows it
        auto fetch_tile = [&]() {
            fetch_scales(0);
            told = sh.tile[chunk & 1];
        };
        if (!kSwiGLU && int(blockIdx.x) < units) fetch_tile();
        for (int unit = int(blockIdx.x); unit < units && ok; unit += int(gridDim.x)) {
            if (kSwiGLU) fetch_tile();  // no registers for it ahead
            const Tile t{told.x, told.y, told.z, told.w};
            const bool real = r < t.rows;
            const bool any = quarter * 32 < t.rows;  // of this warp's rows
            const int64_t row = int64_t(t.row0) + r;
            const int wb = kSwiGLU ? t.nt : t.nt * 2 + group;  // output block of this thread
            const bool inside = wb < args.n_blocks;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 128; ++j) acc[j] = 0.f;
            float f0 = 0.f, f1 = 0.f;
            auto use_scales = [&](int kb) {
                f0 = sr * sw0;
                if (kSwiGLU) f1 = sr * sw1;
                if (kb % kScaleBlocks == kScaleBlocks - 1 || kb == k_blocks - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.scale_empty[chunk & 1]);
                    ++chunk;
                }
            };
            // 64 columns at a time, two loads of 32 in flight while the two before are added; a block's first ones under the last of the block before,
            // where it is complete by then.  A wait for loads is a wait for all of them, about 130 cycles under the MMAs: two a block.
            const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(group * 128);
            uint32_t a[32], b[32];
            use_scales(0);
            float out_scale = 1.f;  // asked for ahead as well
            if (!kSwiGLU && args.row_scale != nullptr && real) out_scale = args.row_scale[row];
            bool begun = false;  // the loads of the block's first columns have been issued
            for (int kb = 0; kb < k_blocks; ++kb, ++block) {
                const int buf = block & 1;
                if (!begun) {
                    ok = __all_sync(0xffffffffu, wait_block(&sh.done[stage], phase, limit_ns, abort_flag)) && ok;
                    if (!ok) {
                        if (lane == 0) fail(kPipeTimeout);
                        break;
                    }
                    tc_fence_after();
                    if (any) {
                        tmem_ld32(taddr + uint32_t(buf * kTileCols), a);
                        tmem_ld32(taddr + uint32_t(buf * kTileCols) + 32, b);
                    }
                }
                if (++stage == kStages) {
                    stage = 0;
                    phase ^= 1u;
                }
                if (any) {
                    const uint32_t at = taddr + uint32_t(buf * kTileCols);
                    const float g0 = f0, g1 = kSwiGLU ? f1 : f0;
                    auto add = [&](const uint32_t (&v)[32], int c) {
#pragma unroll
                        for (int j = 0; j < 32; ++j) acc[c + j] = fmaf(__uint_as_float(v[j]), c < 64 ? g0 : g1, acc[c + j]);
                    };
                    tmem_ld_wait();
                    if (kb + 1 < k_blocks) fetch_scales(kb + 1);
                    add(a, 0);
                    tmem_ld32(at + 64, a);
                    add(b, 32);
                    tmem_ld32(at + 96, b);
                    const bool next_done = block_done(&sh.done[stage], phase);
                    tmem_ld_wait();
                    tc_fence_before();
                    if (lane == 0) arrive_read(empty_addr + uint32_t(buf) * 8u);
                    begun = __all_sync(0xffffffffu, kb + 1 < k_blocks && next_done);
                    if (begun) tc_fence_after();
                    const uint32_t next = taddr + uint32_t((buf ^ 1) * kTileCols);
                    add(a, 64);
                    if (begun) tmem_ld32(next, a);
                    add(b, 96);
                    if (begun) tmem_ld32(next + 32, b);
                } else {
                    tc_fence_before();
                    if (lane == 0) arrive_read(empty_addr + uint32_t(buf) * 8u);
                    if (kb + 1 < k_blocks) fetch_scales(kb + 1);
                }
                if (kb + 1 < k_blocks) use_scales(kb + 1);
            }
            if (!ok) break;
            if (!kSwiGLU && unit + int(gridDim.x) < units) fetch_tile();
            if (!any) continue;
            constexpr int kCols = kSwiGLU ? 64 : 128;  // output columns of this thread
            pieces_read();                             // the tile before, long past
            const int n0 = kSwiGLU ? t.nt * 128 + group * 64 : t.nt * kTileCols + group * 128;
            if (kSwiGLU) {
#pragma unroll
                for (int j = 0; j < 64; ++j) acc[j] = swiglu(acc[j], acc[64 + j]);
            } else if (args.row_scale != nullptr) {
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] *= out_scale;
            }
            if (kQuantize) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < kCols; ++j) m = max_nan(m, fabsf(acc[j]));  // columns behind the last are zero
                if (kSwiGLU) {
                    // The other group's warp of the same rows has the block's other 64 columns.
                    const ExchangeTurn turn = exchange_turn(exchanges);
                    sh.most[turn.at][group][r] = m;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.told[turn.at][group][quarter]);
                    ok = __all_sync(0xffffffffu, wait_block(&sh.told[turn.at][group ^ 1][quarter], turn.parity, limit_ns, abort_flag));
                    if (!ok) {
                        if (lane == 0) fail(kPipeTimeout);
                        break;
                    }
                    m = max_nan(m, sh.most[turn.at][group ^ 1][r]);
                    ++exchanges;
                }
                m = max_nan(m, kTiny);
                const WideBlock scaled(m);
                uint32_t unsure = 0;
                if (real && (kSwiGLU ? group == 0 : inside)) args.scales[row * args.n_blocks + wb] = __fdiv_rn(m, kLargest);
#pragma unroll
                for (int j = 0; j < kCols; j += 16) {
                    uint32_t q[4];
#pragma unroll
                    for (int h = 0; h < 4; ++h) q[h] = scaled.guess(acc + j + 4 * h, unsure);
                    *reinterpret_cast<uint4*>(piece + j) = make_uint4(q[0], q[1], q[2], q[3]);
                }
                if (unsure != 0) {  // quotients next to a tie (this and the second product a value: 4096 tokens, 32 experts, up 1336 -> 1346 us)
#pragma unroll
                    for (int j = 0; j < kCols; j += 4) *reinterpret_cast<uint32_t*>(piece + j) = scaled.exact(acc + j);
                }
                if (real && n0 < args.n) send_piece(args.q + row * args.n + n0, piece, min(kCols, args.n - n0));
            } else {
#pragma unroll
                for (int j = 0; j < kCols; j += 8) {
                    const float* f = acc + j;
                    *reinterpret_cast<uint4*>(piece + j * 2) = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
                }
                if (real && n0 < args.n) send_piece(args.out + row * args.n + n0, piece, 2 * min(kCols, args.n - n0));
            }
        }
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");  // the rows have left shared memory and are written
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <bool kSwiGLU, bool kQuantize>
cudaError_t launch_mode(const Maps& maps, const Args& args, int grid, cudaStream_t stream) {
    auto* fn = fp8_gemm_kernel<kSwiGLU, kQuantize>;
    static std::atomic<uint64_t> raised{0};
    const cudaError_t e = raise_shared_limit(fn, int(kSmemBytes), raised);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(grid));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmemBytes;
    config.stream = stream;
    return cudaLaunchKernelEx(&config, fn, maps, args);
}

}  // namespace

cudaError_t launch(const Maps& maps, const Args& args, int grid, cudaStream_t stream) {
    if (args.experts > kMaxExperts || grid < 1) return cudaErrorInvalidValue;
    if (args.swiglu) return args.q != nullptr ? launch_mode<true, true>(maps, args, grid, stream) : launch_mode<true, false>(maps, args, grid, stream);
    return args.q != nullptr ? launch_mode<false, true>(maps, args, grid, stream) : launch_mode<false, false>(maps, args, grid, stream);
}

}  // namespace fp8
}  // namespace nep

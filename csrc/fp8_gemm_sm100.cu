// Grouped product of e4m3 rows and e4m3 expert weights on the tcgen05 tensor cores:
//
//   out[m, n] = sum over blocks b of 128 columns of  sa[m, b] * sw[e, n / 128, b] * (sum over k in b of a[m, k] * w[e, n, k])
//
// plain (times a factor per row) or silu(gate) * up, to bf16 or to e4m3 with a scale for each 128 output columns.
//
// The scales are any 32-bit values, so the tensor cores sum one block of 128 at a time into TMEM and the epilogue warps add it, scaled,
// to sums that stay in their registers.  Rows are the M operand: a thread owns a row, its scale is one register, and a block
// costs it one multiply-add per column (with the rows as N every column would need a scale of its own from shared memory, 4 cycles a
// load for 4 columns: twice the tensor cores' time).
//
// A cluster of two CTAs computes 256 rows x 256 weight rows (tcgen05.mma.cta_group::2): each CTA loads its own 128 rows and half of the
// weight rows by TMA, the leader issues the MMAs, each CTA's TMEM holds its rows' block sums, two buffers of 256 columns, so that
// the MMAs of a block run under the multiply-adds of the one before.  With SwiGLU the 256 weight rows are 64 gate rows, their 64 up rows
// and again 64 of each, which puts both factors of an output into the same thread.
//
// All waits are bounded; on expiry a CTA records a code in `status`, stops issuing work, and both CTAs still meet at the
// final cluster barrier and free their TMEM.
#include "fp8_gemm_sm100.hpp"

#include "fp8_prim.cuh"
#include "row_prim.cuh"
#include "tc_prim.cuh"

namespace nep {
namespace fp8 {
namespace {

using namespace gemm::tc;
using namespace rows;

constexpr int kTileRows = 128;                   // of one CTA
constexpr int kTileCols = 256;                   // weight rows of a pair
constexpr int kHalfBytes = 128 * 128;            // 16 KB: this CTA's rows, or its half of the weight rows
constexpr int kStageBytes = 2 * kHalfBytes;
constexpr int kStages = 6;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;   // a warpgroup that loads and issues, two that add up
// A launch of 384 threads gives each 168 registers.  The sums need more: 80 + 2 * 208 < 3 * 168, what the block was launched with.
constexpr int kFewRegisters = 80, kManyRegisters = 208;
static_assert(128 * kFewRegisters + 32 * kEpiWarps * kManyRegisters <= kThreads * 168, "registers of the launch");
constexpr int kTmemCols = 512;
constexpr uint32_t kInstrDesc = instr_desc_e4m3(2 * kTileRows, kTileCols);

struct Shared {
    uint64_t full[kStages], empty[kStages], tmem_full[2], tmem_empty[2];
    uint64_t scale_full[2], scale_empty[2];
    uint64_t told[2][4];               // by epilogue group and quarter: its rows' largest values are in `most`
    uint32_t tmem_base;
    int abort;
    float row_scales[2][kScaleBlocks][kTileRows];  // of the next blocks, by turns
    float weight_scales[2][kScaleBlocks][2];       // of the pair's two halves (of the gate and up rows)
    float most[2][2][kTileRows];       // largest of each row's 64 columns, by parity of the tile and epilogue group
    int first_row[kMaxExperts];
    int rows[kMaxExperts];
    int first_tile[kMaxExperts + 1];   // exclusive prefix of row tiles
};
constexpr size_t kSmemBytes = size_t(kStages) * kStageBytes + sizeof(Shared);
static_assert(kSmemBytes <= 232448, "shared memory of a CTA");

struct Tile {
    int expert, row0, rows, nt;  // rows: of the pair, at most 256
};
// The row tiles that share a weight tile are neighbours: the weights come from memory once and from L2 afterwards.
__device__ __forceinline__ Tile locate(const Shared& sh, int experts, int n_tiles, int unit) {
    const int at = unit / n_tiles;
    int lo = 0, hi = experts;  // first_tile[lo] <= at < first_tile[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sh.first_tile[mid] <= at) lo = mid; else hi = mid;
    }
    const int tiles = sh.first_tile[lo + 1] - sh.first_tile[lo], j = unit - sh.first_tile[lo] * n_tiles;
    const int start = j % tiles * 2 * kTileRows;
    return Tile{lo, sh.first_row[lo] + start, min(2 * kTileRows, sh.rows[lo] - start), j / tiles};
}

__device__ __forceinline__ void tma_load_3d_pair(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar_cluster_addr) {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(
                     smem_u32(smem_dst)),
                 "l"(map), "r"(bar_cluster_addr), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void mma_pair_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem),
                 "l"(a_desc), "l"(b_desc), "r"(kInstrDesc), "r"(accumulate)
                 : "memory");
}
// 16 consecutive fp32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(taddr));
}
template <int kRegisters>
__device__ __forceinline__ void give_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegisters)); }
template <int kRegisters>
__device__ __forceinline__ void take_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegisters)); }

template <bool kSwiGLU, bool kQuantize>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args args) {
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared& sh = *reinterpret_cast<Shared*>(smem + kStages * kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t cta = cluster_ctarank();
    const bool leader = cta == 0;
    const uint64_t limit_ns = args.timeout_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.full[s], 1);   // leader: one expect_tx arrival covering both CTAs' bytes
            mbar_init(&sh.empty[s], 1);  // one commit from the leader's MMA thread
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh.tmem_full[b], 1);
            mbar_init(&sh.tmem_empty[b], 2 * kEpiWarps);  // leader: the epilogue warps of both CTAs
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh.scale_full[b], 1);
            mbar_init(&sh.scale_empty[b], kEpiWarps);
        }
        for (int q = 0; q < 8; ++q) mbar_init(&sh.told[q >> 2][q & 3], 1);
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
        sh.first_row[e] = int(first);
        sh.rows[e] = int(n);
    }
    if (warp == 1) tmem_alloc_pair(&sh.tmem_base, kTmemCols);
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int base = 0; base < args.experts; base += 32) {
            const int e = base + lane;
            const int tiles = e < args.experts && !sh.abort ? (sh.rows[e] + 2 * kTileRows - 1) / (2 * kTileRows) : 0;
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
    cluster_sync();  // both CTAs have initialised their barriers before anyone signals across
    tc_fence_after();
    const uint32_t tmem_base = sh.tmem_base;

    const int k_blocks = args.k_blocks;
    const int cluster_id = blockIdx.x >> 1, num_clusters = gridDim.x >> 1;
    const int units = sh.first_tile[args.experts] * args.n_tiles;  // none after bad offsets
    volatile int* abort_flag = &sh.abort;
    auto fail = [&](uint32_t code) {
        *abort_flag = 1;
        if (atomicCAS(args.status, 0u, code) == 0u) args.status[1] = blockIdx.x;
    };

    if (warp < 4) {
    give_registers<kFewRegisters>();
    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer (both CTAs)
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            int64_t issued = 0;
            for (int unit = cluster_id; unit < units && !*abort_flag; unit += num_clusters) {
                const Tile t = locate(sh, args.experts, args.n_tiles, unit);
                // rows that exist, in 16s; what the others' places hold reaches only their own sums
                const int both = (t.rows + 15) & ~15, mine = max(0, min(kTileRows, both - int(cta) * kTileRows));
                const uint32_t bytes = uint32_t(2 * kHalfBytes + both * 128);
                for (int kb = 0; kb < k_blocks; ++kb) {
                    if (!wait_block(&sh.empty[stage], phase ^ 1u, limit_ns, abort_flag)) {
                        fail(kPipeTimeout);
                        break;
                    }
                    uint8_t* dst = smem + stage * kStageBytes;
                    const uint32_t bar = map_to_cta(smem_u32(&sh.full[stage]), 0);
                    if (leader) mbar_expect_tx(&sh.full[stage], bytes);
                    if (kSwiGLU) {
                        const int f0 = t.nt * 128 + int(cta) * 64;
                        tma_load_3d_pair(dst + kHalfBytes, &maps.weights, kb * 128, f0, 2 * t.expert, bar);
                        tma_load_3d_pair(dst + kHalfBytes + kHalfBytes / 2, &maps.weights, kb * 128, f0, 2 * t.expert + 1, bar);
                    } else {
                        tma_load_3d_pair(dst + kHalfBytes, &maps.weights, kb * 128, t.nt * kTileCols + int(cta) * 128, t.expert, bar);
                    }
                    int at = 0;  // boxes of 128, 64, 32 and 16 rows make up any multiple of 16
#pragma unroll
                    for (int b = 0; b < 4; ++b) {
                        const int box = 128 >> b;
                        if (mine & box) {
                            tma_load_2d_pair(dst + at * 128, &maps.rows[b], kb * 128, t.row0 + int(cta) * kTileRows + at, bar);
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
            // a kernel that gave up does not end under its own copies (the leader's barriers count those of both CTAs)
            if (*abort_flag && leader)
                for (int64_t i = max(int64_t(0), issued - kStages); i < issued; ++i)
                    mbar_wait(&sh.full[i % kStages], uint32_t(i / kStages) & 1u, min(limit_ns, uint64_t(100000000)));
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issuer (leader CTA only)
        if (leader && elect_one()) {
            int stage = 0, block = 0;
            uint32_t phase = 0;
            auto commit = [&](uint64_t* bar) {  // in both CTAs, once the MMAs so far have been done
                tc_commit_pair(map_to_cta(smem_u32(bar), 0));
                tc_commit_pair(map_to_cta(smem_u32(bar), 1));
            };
            for (int unit = cluster_id; unit < units && !*abort_flag; unit += num_clusters) {
                for (int kb = 0; kb < k_blocks; ++kb, ++block) {
                    const int buf = block & 1;
                    if (!wait_block(&sh.full[stage], phase, limit_ns, abort_flag) || !wait_block(&sh.tmem_empty[buf], (uint32_t(block >> 1) & 1u) ^ 1u, limit_ns, abort_flag)) {
                        fail(kPipeTimeout);
                        break;
                    }
                    tc_fence_after();
                    const uint8_t* tile = smem + stage * kStageBytes;
                    const uint64_t a_desc = smem_desc_sw128(tile), b_desc = smem_desc_sw128(tile + kHalfBytes);
#pragma unroll
                    for (int k = 0; k < 4; ++k)  // 32 values = 32 bytes inside the 128-byte swizzle row
                        mma_pair_e4m3(tmem_base + uint32_t(buf * kTileCols), a_desc + uint64_t(k * 2), b_desc + uint64_t(k * 2), k != 0 ? 1u : 0u);
                    commit(&sh.empty[stage]);
                    commit(&sh.tmem_full[buf]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------------ scales (both CTAs)
        // Eight blocks at a time and up to sixteen ahead: the epilogue warps have no registers left to wait for memory.
        constexpr int kHalves = kSwiGLU ? 2 : 1;
        int chunk = 0;
        bool ok = true;
        for (int unit = cluster_id; unit < units && ok; unit += num_clusters) {
            const Tile t = locate(sh, args.experts, args.n_tiles, unit);
            // 128 weight rows share a scale: the two halves of the tile, or those of its gate and up rows
            const int half = lane & 1, block = kSwiGLU ? half * args.n_blocks + t.nt : min(2 * t.nt + half, args.n_blocks - 1);
            const float* sw = args.w_scales + (int64_t(t.expert) * kHalves * args.n_blocks + block) * k_blocks;
            const float* sa[4];
            bool real[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = int(cta) * kTileRows + i * 32 + lane;
                real[i] = r < t.rows;
                sa[i] = args.a_scales + (int64_t(t.row0) + r) * k_blocks;
            }
            for (int kb0 = 0; kb0 < k_blocks; kb0 += kScaleBlocks, ++chunk) {
                float v[4][kScaleBlocks];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kScaleBlocks; ++j) v[i][j] = real[i] && kb0 + j < k_blocks ? sa[i][kb0 + j] : 0.f;
                const float w = kb0 + (lane >> 1) < k_blocks && lane < 2 * kScaleBlocks ? sw[kb0 + (lane >> 1)] : 0.f;
                const int slot = chunk & 1;
                ok = __all_sync(0xffffffffu, wait_block(&sh.scale_empty[slot], (uint32_t(chunk >> 1) & 1u) ^ 1u, limit_ns, abort_flag));
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < kScaleBlocks; ++j) sh.row_scales[slot][j][i * 32 + lane] = v[i][j];
                if (lane < 2 * kScaleBlocks) sh.weight_scales[slot][lane >> 1][half] = w;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.scale_full[slot]);
            }
        }
    }
    } else {
        // ------------------------------------------------------------------ epilogue (both CTAs)
        take_registers<kManyRegisters>();
        const int quarter = warp & 3;        // TMEM lanes [32 * quarter, +32) belong to this warp
        const int group = (warp - 4) >> 2;   // its 128 columns
        const int r = quarter * 32 + lane;   // row of this CTA's tile
        int block = 0, chunk = 0, exchanges = 0;
        bool ok = true;
        for (int unit = cluster_id; unit < units && ok; unit += num_clusters) {
            const Tile t = locate(sh, args.experts, args.n_tiles, unit);
            const int in_tile = int(cta) * kTileRows + r;
            const bool real = in_tile < t.rows;
            const bool any = int(cta) * kTileRows + quarter * 32 < t.rows;  // of this warp's rows
            const int64_t row = int64_t(t.row0) + in_tile;
            const int wb = kSwiGLU ? t.nt : t.nt * 2 + group;  // output block of this thread
            const bool inside = wb < args.n_blocks;
            uint64_t sum[64];  // pairs of neighbouring columns
#pragma unroll
            for (int j = 0; j < 64; ++j) sum[j] = 0;
            for (int kb = 0; kb < k_blocks; ++kb, ++block) {
                const int buf = block & 1;
                const int at = kb % kScaleBlocks, slot = chunk & 1;
                if (at == 0) {
                    ok = __all_sync(0xffffffffu, wait_block(&sh.scale_full[slot], uint32_t(chunk >> 1) & 1u, limit_ns, abort_flag));
                    if (!ok) {
                        if (lane == 0) fail(kPipeTimeout);
                        break;
                    }
                }
                const float s = sh.row_scales[slot][at][r];
                const uint64_t f0 = pair_of(s * sh.weight_scales[slot][at][kSwiGLU ? 0 : group]);
                const uint64_t f1 = kSwiGLU ? pair_of(s * sh.weight_scales[slot][at][1]) : f0;
                if (at == kScaleBlocks - 1 || kb == k_blocks - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.scale_empty[slot]);
                    ++chunk;
                }
                ok = __all_sync(0xffffffffu, wait_block(&sh.tmem_full[buf], uint32_t(block >> 1) & 1u, limit_ns, abort_flag));
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
                tc_fence_after();
                auto drained = [&]() {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_read(map_to_cta(smem_u32(&sh.tmem_empty[buf]), 0));
                };
                if (any) {
                    // the next 16 columns are on their way while these are added
                    const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(buf * kTileCols + group * 128);
                    uint32_t v[2][16];
                    tmem_ld16(taddr, v[0]);
#pragma unroll
                    for (int c = 0; c < 8; ++c) {
                        tmem_ld_wait();
                        if (c < 7) tmem_ld16(taddr + (c + 1) * 16, v[(c + 1) & 1]);
                        else drained();
                        const uint64_t f = c < 4 ? f0 : f1;
#pragma unroll
                        for (int j = 0; j < 8; ++j) fma_pair(sum[c * 8 + j], v[c & 1][2 * j], v[c & 1][2 * j + 1], f);
                    }
                } else {
                    drained();
                }
            }
            if (!ok) break;
            if (!any) continue;
            float acc[128];
#pragma unroll
            for (int j = 0; j < 64; ++j) {
                acc[2 * j] = __uint_as_float(uint32_t(sum[j]));
                acc[2 * j + 1] = __uint_as_float(uint32_t(sum[j] >> 32));
            }
            constexpr int kCols = kSwiGLU ? 64 : 128;  // output columns of this thread
            const int n0 = kSwiGLU ? t.nt * 128 + group * 64 : t.nt * kTileCols + group * 128;
            if (kSwiGLU) {
#pragma unroll
                for (int j = 0; j < 64; ++j) acc[j] = __fdividef(acc[j], 1.f + __expf(-acc[j])) * acc[64 + j];
            } else if (args.row_scale != nullptr) {
                const float f = real ? args.row_scale[row] : 0.f;
#pragma unroll
                for (int j = 0; j < 128; ++j) acc[j] *= f;
            }
            if (kQuantize) {
                float m = 0.f;
#pragma unroll
                for (int j = 0; j < kCols; ++j) m = max_nan(m, fabsf(acc[j]));  // columns behind the last are zero
                if (kSwiGLU) {
                    // The other group's warp of the same rows has the block's other 64 columns.  What it told for a tile has been read before
                    // this warp tells for the next one, so two places by turns are enough.
                    const int turn = exchanges & 1;
                    sh.most[turn][group][r] = m;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&sh.told[group][quarter]);
                    ok = __all_sync(0xffffffffu, wait_block(&sh.told[group ^ 1][quarter], uint32_t(turn), limit_ns, abort_flag));
                    if (!ok) {
                        if (lane == 0) fail(kPipeTimeout);
                        break;
                    }
                    m = max_nan(m, sh.most[turn][group ^ 1][r]);
                    ++exchanges;
                }
                m = max_nan(m, kTiny);
                const float per = __fdiv_rn(kLargest, m);  // sums do not lie on the border of two e4m3 values: a product will do
                if (real && (kSwiGLU ? group == 0 : inside)) args.scales[row * args.n_blocks + wb] = __fdiv_rn(m, kLargest);
#pragma unroll
                for (int j = 0; j < kCols; j += 16) {
                    if (!real || n0 + j >= args.n) continue;
                    uint32_t q[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        q[i] = pack_e4m3(acc[j + 4 * i] * per, acc[j + 4 * i + 1] * per, acc[j + 4 * i + 2] * per, acc[j + 4 * i + 3] * per);
                    st_v4(args.q + row * args.n + n0 + j, q[0], q[1], q[2], q[3]);
                }
            } else {
#pragma unroll
                for (int j = 0; j < kCols; j += 8) {
                    if (!real || n0 + j >= args.n) continue;
                    st_v4(args.out + row * args.n + n0 + j, pack_bf16(acc[j], acc[j + 1]), pack_bf16(acc[j + 2], acc[j + 3]), pack_bf16(acc[j + 4], acc[j + 5]),
                          pack_bf16(acc[j + 6], acc[j + 7]));
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peer may still be reading this CTA's operands / signalling its barriers
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, kTmemCols);
    }
}

template <bool kSwiGLU, bool kQuantize>
cudaError_t launch_mode(const Maps& maps, const Args& args, int grid, cudaStream_t stream) {
    auto* fn = fp8_gemm_kernel<kSwiGLU, kQuantize>;
    cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kSmemBytes));
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(grid));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kSmemBytes;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, fn, maps, args);
}

}  // namespace

cudaError_t launch(const Maps& maps, const Args& args, int grid, cudaStream_t stream) {
    grid &= ~1;
    if (args.experts > kMaxExperts || grid < 2) return cudaErrorInvalidValue;
    if (args.swiglu) return args.q != nullptr ? launch_mode<true, true>(maps, args, grid, stream) : launch_mode<true, false>(maps, args, grid, stream);
    return args.q != nullptr ? launch_mode<false, true>(maps, args, grid, stream) : launch_mode<false, false>(maps, args, grid, stream);
}

}  // namespace fp8
}  // namespace nep

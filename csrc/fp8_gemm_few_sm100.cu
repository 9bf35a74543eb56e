// The 8-bit grouped product for experts with few rows: WEIGHTS as the tensor cores' M operand, the rows as N.
//
// Such a call is bound by the weights' way from memory.  With rows as M the tensor cores work on 256 rows whether they exist or not,
// which at 16 rows an expert costs the card its power limit and leaves two block sums in TMEM, too few to cover the way from the MMA to the
// epilogue and back.  As N a tile takes any multiple of 16 rows, and TMEM holds eight block sums of 32 rows.  The scale of a row is then
// needed per column: it comes from shared memory, four columns a load, cheap as long as there are few.
//
// A CTA computes 256 weight rows x N rows as two accumulators of 128 TMEM lanes: gate and up rows of the same 128 features with SwiGLU, so that
// a lane holds both factors of its outputs, or two neighbouring blocks of output columns; where tiles are so few that SMs stay idle, one
// block (128 weight rows).  A cluster of S CTAs splits the K axis: S times the
// SMs on one weight tile where there are few tiles, and an even share where their number is no multiple of the SMs.
// The CTAs exchange their sums through distributed shared memory, 32 rows at a time; each finishes its share of the rows, adding
// the parts in the order of K.  On the way the tile is turned: a warp finishes whole output rows.
//
// What bounds it: the weights' way from memory (32 experts of 7168 x 2048, up, us: 1 row each 150, 16 rows 154, 32 rows 159 = 5.9 TB/s, where a
// copy runs at 6.5; rows as M 171, 172, 176), and for one matrix that of few SMs, 78 GB/s each, behind about 8 us of launch, setup and
// exchange: 7168 x 4096 with one row, calls on eight such matrices by turns in a graph, 25.1 us in one CTA a tile, 16.6 in two, 13.0 in four, 12.7 in
// four on tiles of 128 weight rows.
//
// Tried: 16 columns of both accumulators per wait instead of 8: 64 rows each 193 -> 200 us; the state of the next barriers asked for under the
// MMAs: within the spread; 128 rows as N: 312 us at 128 rows each (the columns' scales), rows as M 188.
//
// All waits are bounded; on expiry a CTA records a code in `status`, stops issuing work, waits for its own copies, and the cluster's CTAs still
// meet at the final barrier and free their TMEM.
#include "fp8_gemm_sm100.hpp"

#include <algorithm>

#include "fp8_prim.cuh"
#include "launch_once.hpp"
#include "row_prim.cuh"
#include "tc_prim.cuh"

namespace nep {
namespace fp8 {
namespace {

using namespace gemm::tc;
using namespace rows;

constexpr int kLanes = 128;                    // weight rows of one accumulator
constexpr int kLanesBytes = kLanes * 128;      // an accumulator's rows of a stage, 128 columns
constexpr int kEpiWarps = 8;
constexpr int kThreads = 128 + 32 * kEpiWarps;
constexpr int kTmemCols = 512;
constexpr int kSlice = 32;                     // rows exchanged at a time, half of them from each epilogue group

// One accumulator (128 output columns a tile) or two.
template <int kAcc, int kTileRows>
struct Shape {
    static constexpr int kWeightBytes = kAcc * kLanesBytes;
    static constexpr int kStageBytes = kWeightBytes + kTileRows * 128;
    static constexpr int kStages = kAcc == 1 ? 8 : kTileRows <= 32 ? 5 : 4;
    static constexpr int kBufs = kTmemCols / (kAcc * kTileRows) < 8 ? kTmemCols / (kAcc * kTileRows) : 8;
};

template <int kAcc, int kTileRows>
struct Shared {
    using S = Shape<kAcc, kTileRows>;
    float parts[kSlice * kAcc * kLanes];  // [source CTA][row][accumulator][lane]
    float row_scales[2][kScaleBlocks][kTileRows];
    float weight_scales[2][kScaleBlocks][2];
    uint64_t full[S::kStages], empty[S::kStages], tmem_full[S::kBufs], tmem_empty[S::kBufs];
    uint64_t scale_full[2], scale_empty[2], parts_full, parts_empty;
    uint32_t tmem_base;
    int abort;
    int first_row[kMaxExperts];
    int rows[kMaxExperts];
    int first_tile[kMaxExperts + 1];
};
template <int kAcc, int kTileRows>
constexpr size_t smem_bytes() {
    return size_t(Shape<kAcc, kTileRows>::kStages) * Shape<kAcc, kTileRows>::kStageBytes + sizeof(Shared<kAcc, kTileRows>);
}
static_assert(smem_bytes<2, 32>() <= 232448 && smem_bytes<2, 64>() <= 232448 && smem_bytes<1, 32>() <= 232448 && smem_bytes<1, 64>() <= 232448, "shared memory of a CTA");

struct Tile {
    int expert, row0, rows, nt;
};
// Rows per tile of an expert with n rows: equal tiles, a multiple of 16.
__device__ __forceinline__ int tile_rows(int n, int largest) {
    const int tiles = (n + largest - 1) / largest;
    return ((n + tiles - 1) / tiles + 15) & ~15;
}
template <int kAcc, int kTileRows>
__device__ __forceinline__ Tile locate(const Shared<kAcc, kTileRows>& sh, int experts, int n_tiles, int unit) {
    const int at = unit / n_tiles;
    int lo = 0, hi = experts;  // first_tile[lo] <= at < first_tile[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sh.first_tile[mid] <= at) lo = mid; else hi = mid;
    }
    const int tiles = sh.first_tile[lo + 1] - sh.first_tile[lo], j = unit - sh.first_tile[lo] * n_tiles;
    const int n = sh.rows[lo], each = tile_rows(n, kTileRows), start = j % tiles * each;
    return Tile{lo, sh.first_row[lo] + start, min(each, n - start), j / tiles};
}

// 8 consecutive fp32 columns of this thread's TMEM lane
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
}
__device__ __forceinline__ void st_cluster_f32(uint32_t cluster_addr, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(cluster_addr), "f"(v) : "memory");
}
// Bounded wait that also orders what the other CTAs of the cluster wrote before their arrivals.
__device__ __forceinline__ bool wait_cluster(uint64_t* bar, uint32_t parity, uint64_t limit_ns, const volatile int* abort) {
    uint64_t start = 0;
    uint32_t spins = 0;
    for (;;) {
        uint32_t done;
        asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                     : "=r"(done)
                     : "r"(smem_u32(bar)), "r"(parity)
                     : "memory");
        if (done) return true;
        if ((++spins & 255u) != 0u) continue;
        if (*abort) return false;
        const uint64_t now = timer_ns();
        if (start == 0) start = now;
        if (now - start > limit_ns) return false;
    }
}

template <int kAcc, bool kSwiGLU, bool kQuantize, int kTileRows>
__global__ void __launch_bounds__(kThreads, 1) fp8_gemm_few_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args args, const int ctas) {
    static_assert(kAcc == 2 || !kSwiGLU, "gate and up rows");
    using P = Shape<kAcc, kTileRows>;
    constexpr int kStages = P::kStages, kBufs = P::kBufs;
    extern __shared__ __align__(1024) uint8_t smem[];
    Shared<kAcc, kTileRows>& sh = *reinterpret_cast<Shared<kAcc, kTileRows>*>(smem + kStages * P::kStageBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int cta = int(cluster_ctarank());
    const uint64_t limit_ns = args.timeout_ns;

    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) {
            mbar_init(&sh.full[s], 1);
            mbar_init(&sh.empty[s], 1);
        }
        for (int b = 0; b < kBufs; ++b) {
            mbar_init(&sh.tmem_full[b], 1);
            mbar_init(&sh.tmem_empty[b], kEpiWarps);
        }
        for (int b = 0; b < 2; ++b) {
            mbar_init(&sh.scale_full[b], 1);
            mbar_init(&sh.scale_empty[b], kEpiWarps);
        }
        mbar_init(&sh.parts_full, uint32_t(ctas * kEpiWarps));
        mbar_init(&sh.parts_empty, uint32_t(ctas * kEpiWarps));
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
    if (warp == 1) tmem_alloc(&sh.tmem_base, kTmemCols);
    __syncthreads();
    if (warp == 0) {
        int carry = 0;
        for (int base = 0; base < args.experts; base += 32) {
            const int e = base + lane;
            const int n = e < args.experts && !sh.abort ? sh.rows[e] : 0;
            const int tiles = n > 0 ? (n + tile_rows(n, kTileRows) - 1) / tile_rows(n, kTileRows) : 0;
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
    cluster_sync();  // every CTA has initialised its barriers before anyone signals across
    tc_fence_after();
    const uint32_t tmem_base = sh.tmem_base;

    const int cluster_id = blockIdx.x / ctas, num_clusters = gridDim.x / ctas;
    const int units = sh.first_tile[args.experts] * args.n_tiles;  // none after bad offsets
    const int k_first = args.k_blocks * cta / ctas, k_last = args.k_blocks * (cta + 1) / ctas;  // this CTA's part of the K axis
    volatile int* abort_flag = &sh.abort;
    auto fail = [&](uint32_t code) {
        *abort_flag = 1;
        if (atomicCAS(args.status, 0u, code) == 0u) args.status[1] = blockIdx.x;
    };

    if (warp == 0) {
        // ------------------------------------------------------------------ TMA producer
        if (elect_one()) {
            int stage = 0;
            uint32_t phase = 0;
            int64_t issued = 0;
            for (int unit = cluster_id; unit < units && !*abort_flag; unit += num_clusters) {
                const Tile t = locate(sh, args.experts, args.n_tiles, unit);
                const int n = (t.rows + 15) & ~15;
                for (int kb = k_first; kb < k_last; ++kb) {
                    if (!wait_block(&sh.empty[stage], phase ^ 1u, limit_ns, abort_flag)) {
                        fail(kPipeTimeout);
                        break;
                    }
                    uint8_t* dst = smem + stage * P::kStageBytes;
                    mbar_expect_tx(&sh.full[stage], uint32_t(P::kWeightBytes + n * 128));
#pragma unroll
                    for (int i = 0; i < kAcc; ++i)
                        tma_load_3d(dst + i * kLanesBytes, &maps.weights, kb * 128, kSwiGLU ? t.nt * kLanes : (kAcc * t.nt + i) * kLanes,
                                    kSwiGLU ? 2 * t.expert + i : t.expert, &sh.full[stage]);
                    int at = 0;  // boxes of 64, 32 and 16 rows make up any multiple of 16 that a tile has
#pragma unroll
                    for (int b = kTileRows <= 32 ? 2 : 1; b < 4; ++b) {
                        const int box = 128 >> b;
                        if (n & box) {
                            tma_load_2d(dst + P::kWeightBytes + at * 128, &maps.rows[b], kb * 128, t.row0 + at, &sh.full[stage]);
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
            int stage = 0, buf = 0;
            uint32_t phase = 0, buf_phase = 0;
            for (int unit = cluster_id; unit < units && !*abort_flag; unit += num_clusters) {
                const Tile t = locate(sh, args.experts, args.n_tiles, unit);
                const uint32_t idesc = instr_desc_e4m3(kLanes, (t.rows + 15) & ~15);
                for (int kb = k_first; kb < k_last; ++kb) {
                    if (!wait_block(&sh.full[stage], phase, limit_ns, abort_flag) || !wait_block(&sh.tmem_empty[buf], buf_phase ^ 1u, limit_ns, abort_flag)) {
                        fail(kPipeTimeout);
                        break;
                    }
                    tc_fence_after();
                    const uint8_t* tile = smem + stage * P::kStageBytes;
                    const uint64_t r_desc = smem_desc_sw128(tile + P::kWeightBytes);
#pragma unroll
                    for (int i = 0; i < kAcc; ++i) {
                        const uint64_t w_desc = smem_desc_sw128(tile + i * kLanesBytes);
#pragma unroll
                        for (int k = 0; k < 4; ++k)  // 32 values = 32 bytes inside the 128-byte swizzle row
                            mma_e4m3(tmem_base + uint32_t((kAcc * buf + i) * kTileRows), w_desc + uint64_t(k * 2), r_desc + uint64_t(k * 2), idesc, k != 0 ? 1u : 0u);
                    }
                    tc_commit(&sh.empty[stage]);
                    tc_commit(&sh.tmem_full[buf]);
                    if (++stage == kStages) {
                        stage = 0;
                        phase ^= 1u;
                    }
                    if (++buf == kBufs) {
                        buf = 0;
                        buf_phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 2) {
        // ------------------------------------------------------------------ scales: eight blocks at a time, up to sixteen ahead
        constexpr int kHalves = kSwiGLU ? 2 : 1;
        int chunk = 0;
        bool ok = true;
        for (int unit = cluster_id; unit < units && ok; unit += num_clusters) {
            const Tile t = locate(sh, args.experts, args.n_tiles, unit);
            const int half = lane & 1, block = kSwiGLU ? half * args.n_blocks + t.nt : min(kAcc * t.nt + half % kAcc, args.n_blocks - 1);
            const float* sw = args.w_scales + (int64_t(t.expert) * kHalves * args.n_blocks + block) * args.k_blocks;
            for (int kb0 = k_first; kb0 < k_last; kb0 += kScaleBlocks, ++chunk) {
                const int slot = chunk & 1;
                const float w = kb0 + (lane >> 1) < k_last && lane < 2 * kScaleBlocks ? sw[kb0 + (lane >> 1)] : 0.f;
                float v[kTileRows / 32][kScaleBlocks];
#pragma unroll
                for (int i = 0; i < kTileRows / 32; ++i) {
                    const int r = i * 32 + lane;
                    const float* sa = args.a_scales + (int64_t(t.row0) + r) * args.k_blocks + kb0;
#pragma unroll
                    for (int j = 0; j < kScaleBlocks; ++j) v[i][j] = r < t.rows && kb0 + j < k_last ? sa[j] : 0.f;
                }
                ok = __all_sync(0xffffffffu, wait_block(&sh.scale_empty[slot], (uint32_t(chunk >> 1) & 1u) ^ 1u, limit_ns, abort_flag));
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
#pragma unroll
                for (int i = 0; i < kTileRows / 32; ++i)
#pragma unroll
                    for (int j = 0; j < kScaleBlocks; ++j) sh.row_scales[slot][j][i * 32 + lane] = v[i][j];
                if (lane < 2 * kScaleBlocks) sh.weight_scales[slot][lane >> 1][half] = w;
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.scale_full[slot]);
            }
        }
    } else if (warp >= 4) {
        // ------------------------------------------------------------------ epilogue
        const int quarter = warp & 3;        // TMEM lanes [32 * quarter, +32) belong to this warp
        const int group = (warp - 4) >> 2;   // half of the rows
        const int feature = quarter * 32 + lane;
        constexpr int kCols = kTileRows / 2;  // rows of this thread, of both accumulators
        int buf = 0, chunk = 0, slices = 0;
        uint32_t buf_phase = 0;
        bool ok = true;
        for (int unit = cluster_id; unit < units && ok; unit += num_clusters) {
            const Tile t = locate(sh, args.experts, args.n_tiles, unit);
            const int half = ((t.rows + 15) & ~15) / 2;  // rows of a group, a multiple of 8
            uint64_t sum[kAcc][kCols / 2];
#pragma unroll
            for (int i = 0; i < kAcc; ++i)
#pragma unroll
                for (int j = 0; j < kCols / 2; ++j) sum[i][j] = 0;
            for (int kb = k_first; kb < k_last; ++kb) {
                const int at = (kb - k_first) % kScaleBlocks, slot = chunk & 1;
                if (at == 0) ok = __all_sync(0xffffffffu, wait_block(&sh.scale_full[slot], uint32_t(chunk >> 1) & 1u, limit_ns, abort_flag));
                ok = ok && __all_sync(0xffffffffu, wait_block(&sh.tmem_full[buf], buf_phase, limit_ns, abort_flag));
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
                tc_fence_after();
                uint64_t w[kAcc];
#pragma unroll
                for (int i = 0; i < kAcc; ++i) w[i] = pair_of(sh.weight_scales[slot][at][i]);
                const float* scales = &sh.row_scales[slot][at][group * half];
                const uint32_t taddr = tmem_base + (uint32_t(quarter * 32) << 16) + uint32_t(kAcc * buf * kTileRows + group * half);
#pragma unroll
                for (int c = 0; c < kCols / 8; ++c) {
                    if (c * 8 >= half) break;
                    uint32_t v[kAcc][8];
#pragma unroll
                    for (int i = 0; i < kAcc; ++i) tmem_ld8(taddr + i * kTileRows + c * 8, v[i]);
                    const ulonglong2 s0 = *reinterpret_cast<const ulonglong2*>(scales + c * 8), s1 = *reinterpret_cast<const ulonglong2*>(scales + c * 8 + 4);
                    const uint64_t s[4] = {s0.x, s0.y, s1.x, s1.y};
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int i = 0; i < kAcc; ++i) fma_pair(sum[i][c * 4 + j], v[i][2 * j], v[i][2 * j + 1], mul_pair(s[j], w[i]));
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) arrive_read(smem_u32(&sh.tmem_empty[buf]));
                if (++buf == kBufs) {
                    buf = 0;
                    buf_phase ^= 1u;
                }
                if (at == kScaleBlocks - 1 || kb == k_last - 1) {
                    if (lane == 0) mbar_arrive(&sh.scale_empty[slot]);
                    ++chunk;
                }
            }
            if (!ok) break;
            // The sums go to the CTA that finishes their row, 16 rows of each group at a time, and come back as whole output rows.
#pragma unroll
            for (int s = 0; s < (kCols + 15) / 16; ++s) {
                if (s * 16 >= half) break;
                const int each = min(16, half - s * 16);   // rows of a group in this slice
                const int share = 2 * each / ctas;         // rows that a CTA finishes
                ok = __all_sync(0xffffffffu, wait_cluster(&sh.parts_empty, (uint32_t(slices) & 1u) ^ 1u, limit_ns, abort_flag));
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    if (s * 16 + j >= kCols || j >= each) break;
                    const int q = group * each + j, to = q / share;
                    const uint32_t dst = map_to_cta(smem_u32(&sh.parts[(cta * share + q % share) * kAcc * kLanes + feature]), uint32_t(to));
#pragma unroll
                    for (int i = 0; i < kAcc; ++i) {
                        const uint64_t p = sum[i][(s * 16 + j) / 2];
                        st_cluster_f32(dst + i * kLanes * 4, __uint_as_float(j & 1 ? uint32_t(p >> 32) : uint32_t(p)));
                    }
                }
                __syncwarp();
                for (int c = lane; c < ctas; c += 32) mbar_arrive_cluster(map_to_cta(smem_u32(&sh.parts_full), uint32_t(c)));
                ok = __all_sync(0xffffffffu, wait_cluster(&sh.parts_full, uint32_t(slices) & 1u, limit_ns, abort_flag));
                if (!ok) {
                    if (lane == 0) fail(kPipeTimeout);
                    break;
                }
                // a warp per row, four neighbouring columns of each accumulator per lane
                for (int q = warp - 4; q < share; q += kEpiWarps) {
                    const int column = cta * share + q, in_tile = column / each * half + s * 16 + column % each;
                    if (in_tile >= t.rows) continue;
                    float v[kAcc][4] = {};
                    for (int c = 0; c < ctas; ++c)
#pragma unroll
                        for (int i = 0; i < kAcc; ++i) {
                            const float4 p = *reinterpret_cast<const float4*>(&sh.parts[((c * share + q) * kAcc + i) * kLanes + lane * 4]);
                            v[i][0] += p.x, v[i][1] += p.y, v[i][2] += p.z, v[i][3] += p.w;
                        }
                    const int64_t row = int64_t(t.row0) + in_tile;
                    if (kSwiGLU) {
#pragma unroll
                        for (int j = 0; j < 4; ++j) v[0][j] = swiglu(v[0][j], v[kAcc - 1][j]);
                    } else if (args.row_scale != nullptr) {
                        const float f = args.row_scale[row];
#pragma unroll
                        for (int i = 0; i < kAcc; ++i)
#pragma unroll
                            for (int j = 0; j < 4; ++j) v[i][j] *= f;
                    }
#pragma unroll
                    for (int i = 0; i < (kSwiGLU ? 1 : kAcc); ++i) {
                        const int block = kSwiGLU ? t.nt : kAcc * t.nt + i, n0 = block * 128 + lane * 4;
                        if (kQuantize) {
                            float m = 0.f;  // columns behind the last are zero
#pragma unroll
                            for (int j = 0; j < 4; ++j) m = max_nan(m, fabsf(v[i][j]));
                            m = max_nan(group_max<32>(m), kTiny);
                            if (lane == 0 && block < args.n_blocks) args.scales[row * args.n_blocks + block] = __fdiv_rn(m, kLargest);
                            if (n0 < args.n)
                                *reinterpret_cast<uint32_t*>(args.q + row * args.n + n0) = WideBlock(m).pack(v[i]);
                        } else if (n0 < args.n) {
                            *reinterpret_cast<uint2*>(args.out + row * args.n + n0) = make_uint2(pack_bf16(v[i][0], v[i][1]), pack_bf16(v[i][2], v[i][3]));
                        }
                    }
                }
                __syncwarp();
                for (int c = lane; c < ctas; c += 32) mbar_arrive_cluster(map_to_cta(smem_u32(&sh.parts_empty), uint32_t(c)));
                ++slices;
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();  // the peers may still be writing here / signalling this CTA's barriers
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc(tmem_base, kTmemCols);
    }
}

template <int kAcc, bool kSwiGLU, bool kQuantize, int kTileRows>
cudaError_t launch_tile(const Maps& maps, const Args& args, int ctas, int64_t units, int sms, cudaStream_t stream) {
    auto* fn = fp8_gemm_few_kernel<kAcc, kSwiGLU, kQuantize, kTileRows>;
    constexpr size_t kBytes = smem_bytes<kAcc, kTileRows>();
    static std::atomic<uint64_t> raised{0};
    const cudaError_t e = raise_shared_limit(fn, int(kBytes), raised);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = kBytes;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(ctas);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    config.gridDim = dim3(unsigned(ctas * std::min<int64_t>(units, few_clusters(ctas, sms))));
    return cudaLaunchKernelEx(&config, fn, maps, args, ctas);
}

template <int kAcc, bool kSwiGLU, bool kQuantize>
cudaError_t launch_mode(const Maps& maps, const Args& args, int tile, int ctas, int64_t units, int sms, cudaStream_t stream) {
    if (tile <= 32) return launch_tile<kAcc, kSwiGLU, kQuantize, 32>(maps, args, ctas, units, sms, stream);
    return launch_tile<kAcc, kSwiGLU, kQuantize, 64>(maps, args, ctas, units, sms, stream);
}

}  // namespace

// Clusters of so many CTAs that the GPU holds at a time (what the runtime's occupancy query answers): its SMs come in groups that a
// cluster does not leave.  One cluster more runs behind the others and doubles the time.
int few_clusters(int ctas, int sms) { return ctas <= 2 ? sms / ctas : ctas == 4 ? 33 * sms / 148 : 15 * sms / 148; }

cudaError_t launch_few(const Maps& maps, const Args& args, int tile, int ctas, int64_t units, int sms, cudaStream_t stream) {
    if (args.experts > kMaxExperts || units < 1 || ctas < 1 || ctas > 8) return cudaErrorInvalidValue;
    const bool q = args.q != nullptr;
    if (args.swiglu) return q ? launch_mode<2, true, true>(maps, args, tile, ctas, units, sms, stream) : launch_mode<2, true, false>(maps, args, tile, ctas, units, sms, stream);
    if (args.n_tiles == args.n_blocks)
        return q ? launch_mode<1, false, true>(maps, args, tile, ctas, units, sms, stream) : launch_mode<1, false, false>(maps, args, tile, ctas, units, sms, stream);
    return q ? launch_mode<2, false, true>(maps, args, tile, ctas, units, sms, stream) : launch_mode<2, false, false>(maps, args, tile, ctas, units, sms, stream);
}

}  // namespace fp8
}  // namespace nep

// Device helpers shared by the 8-bit grouped GEMM kernels.
#pragma once
#include "fp8_gemm_sm100.hpp"
#include "tc_prim.cuh"

namespace nep {
namespace fp8 {

constexpr int kScaleBlocks = 8;  // blocks whose scales are loaded at a time: 32 bytes of a row

// e4m3 x e4m3 -> fp32, both operands K-major, tile M x N
constexpr __host__ __device__ uint32_t instr_desc_e4m3(int m, int n) { return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24); }

// Rows of an expert; false where the offsets fall, do not start at 0 or end behind the rows (it has none then).
__device__ __forceinline__ bool expert_range(const Args& args, int e, int64_t& first, int64_t& n) {
    first = args.expert_offsets != nullptr ? args.expert_offsets[e] : 0;
    const int64_t end = args.expert_offsets != nullptr ? args.expert_offsets[e + 1] : args.rows;
    n = end - first;
    if (first < 0 || n < 0 || end > args.rows || (e == 0 && first != 0)) {
        n = 0;
        return false;
    }
    if (args.expert_counts != nullptr) n = max(int64_t(0), min(args.expert_counts[e], n));
    return true;
}

// Whether a phase is complete, without waiting: asked ahead, so that the answer's way (about 100 cycles) lies under other work.
__device__ __forceinline__ bool block_done(uint64_t* bar, uint32_t parity) {
    uint32_t done;
    asm volatile("{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
                 : "=r"(done)
                 : "r"(gemm::tc::smem_u32(bar)), "r"(parity)
                 : "memory");
    return done != 0;
}
// Bounded wait that reads the timer only once it has polled for a while: a read takes about a microsecond, and the epilogue waits for
// every block of 128 columns.
__device__ __forceinline__ bool wait_block(uint64_t* bar, uint32_t parity, uint64_t limit_ns, const volatile int* abort) {
    uint64_t start = 0;
    uint32_t spins = 0;
    while (!gemm::tc::mbar_try(bar, parity)) {
        if ((++spins & 255u) != 0u) continue;
        if (*abort) return false;
        const uint64_t now = gemm::tc::timer_ns();
        if (start == 0) start = now;
        if (now - start > limit_ns) return false;
    }
    return true;
}
// Arrival without a fence: what it stands for, TMEM columns that have been read, is complete when tcgen05.wait::ld returns.  A releasing
// arrival of cluster scope waits for the thread's loads in flight as well, the scales of the blocks ahead: 1000 cycles a block.
__device__ __forceinline__ void arrive_read(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

__device__ __forceinline__ void tma_load_2d(void* smem_dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(gemm::tc::smem_u32(smem_dst)),
                 "l"(map), "r"(gemm::tc::smem_u32(bar)), "r"(x), "r"(y)
                 : "memory");
}
__device__ __forceinline__ void tma_load_3d(void* smem_dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(gemm::tc::smem_u32(smem_dst)),
                 "l"(map), "r"(gemm::tc::smem_u32(bar)), "r"(x), "r"(y), "r"(z)
                 : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t* smem_slot, uint32_t cols) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(gemm::tc::smem_u32(smem_slot)), "r"(cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t addr, uint32_t cols) {
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(gemm::tc::smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void mma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d_tmem), "l"(a_desc),
                 "l"(b_desc), "r"(idesc), "r"(accumulate)
                 : "memory");
}

// silu(gate) * up.  The quotient is the fast one, a choice: within 2 units in the last place, and 0 for gates below -87.3 (1 + exp(-gate) is beyond 2^126 there),
// whose silu is below 2^-119 in size.  A rounded quotient, as the 16-bit kernels' epilogue has: 4096 tokens, 32 experts, up 1350 -> 1490 us.
__device__ __forceinline__ float swiglu(float gate, float up) { return __fdividef(gate, 1.f + __expf(-gate)) * up; }

__device__ __forceinline__ uint64_t pair_of(float f) {
    uint64_t p;
    asm("mov.b64 %0, {%1, %1};" : "=l"(p) : "r"(__float_as_uint(f)));
    return p;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
    uint64_t p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p) : "l"(a), "l"(b));
    return p;
}
// two columns at a time: sum += {lo, hi} * f
__device__ __forceinline__ void fma_pair(uint64_t& sum, uint32_t lo, uint32_t hi, uint64_t f) {
    asm("{\n .reg .b64 v;\n mov.b64 v, {%1, %2};\n fma.rn.f32x2 %0, v, %3, %0;\n}" : "+l"(sum) : "r"(lo), "r"(hi), "l"(f));
}

}  // namespace fp8
}  // namespace nep

// A batch sorted by expert and back, on one GPU: the counting sort of the choices, the rows' way to the experts, the weighted sum
// of what comes back, and both gradients.  No host ever waits for a count, so everything here can be captured in a graph.
//
// slot(t, k) = offset(e) + how many choices of e come in front of (t, k) in token order: the order is stable and the same on every
// run.  offset(e) = sum of the counts in front, each rounded up to `alignment`.
#include "token_order.hpp"

#include "launch_once.hpp"
#include "row_prim.cuh"

namespace nep {
namespace order {
namespace {

using namespace rows;

// ------------------------------------------------------------------------------------------------ plan
// One cluster.  Every warp owns a run of neighbouring choices and counts it by expert; prefixes over warps and CTAs turn the
// counts into each warp's first slots; the warps then walk their runs again and hand the slots out.  Equal experts within 32
// choices are found by a vote per bit of their id, so there are no atomics and the order is that of the choices.  (With the warp's match
// instruction, which takes turns with every other access to shared memory, 32768 choices took 16.7 us instead of 12.8.)
constexpr int kPlanThreads = 1024, kPlanWarps = kPlanThreads / 32, kMaxPlanCtas = 8;

struct PlanShared {
    int total[kMaxExperts];     // choices of this CTA
    int base[kMaxExperts];      // first slot of this CTA's choices
    int count[kMaxExperts];     // of the whole batch
    int64_t scan[kPlanWarps + 1];
};

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ int ld_cta(const int* p, uint32_t rank) {
    uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(p));
    int v;
    asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %1, %2;\n ld.shared::cluster.s32 %0, [a];\n}" : "=r"(v) : "r"(at), "r"(rank) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_barrier() {
    asm volatile("barrier.cluster.arrive.release;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// Lanes that hold the same expert as this one; `bits` for ids up to the number of experts (masked choices hold that).
__device__ __forceinline__ uint32_t same_expert(int e, int bits) {
    uint32_t same = 0xffffffffu;
    for (int b = 0; b < bits; ++b) {
        const bool set = (e >> b & 1) != 0;
        const uint32_t votes = __ballot_sync(0xffffffffu, set);
        same &= set ? votes : ~votes;
    }
    return same;
}

// Up to kKept * 32 choices a warp stay in registers between the two walks; longer runs are read again.
constexpr int kKept = 8;

template <bool kInRegisters>
__global__ void __launch_bounds__(kPlanThreads, 1) plan_kernel(const PlanArgs a, int ctas, int64_t per_warp) {
    extern __shared__ __align__(16) uint8_t smem[];
    PlanShared& sh = *reinterpret_cast<PlanShared*>(smem);
    int* hist = reinterpret_cast<int*>(smem + sizeof(PlanShared));  // [warps][experts]
    const int E = a.experts, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t cta = ctas > 1 ? cluster_rank() : 0;
    const int64_t first = (int64_t(cta) * kPlanWarps + warp) * per_warp;
    const int64_t last = min(a.choices, first + per_warp);
    int* mine = hist + warp * E;
    const int bits = 32 - __clz(E);
    auto read = [&](int64_t i) -> int {
        const int64_t id = i < last ? a.topk_idx[i] : -1;
        if (id >= 0 && id < E) return int(id);
        if (id != -1 && atomicCAS(a.status, 0u, uint32_t(kBadExpertId)) == 0u) a.status[1] = uint32_t(i);
        return E;
    };
    int kept[kInRegisters ? kKept : 1];
    uint32_t kept_same[kInRegisters ? kKept : 1];
    if (kInRegisters) {
#pragma unroll
        for (int j = 0; j < kKept; ++j) kept[j] = read(first + j * 32 + lane);
    }
    for (int i = tid; i < kPlanWarps * E; i += kPlanThreads) hist[i] = 0;
    __syncthreads();
    auto count_32 = [&](int e) -> uint32_t {
        const uint32_t same = same_expert(e, bits);
        if (e < E && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
        return same;
    };
    if (kInRegisters) {
#pragma unroll
        for (int j = 0; j < kKept; ++j)
            if (first + j * 32 < last) kept_same[j] = count_32(kept[j]);
    } else {
        for (int64_t at = first; at < last; at += 32) count_32(read(at + lane));
    }
    __syncthreads();
    for (int e = tid; e < E; e += kPlanThreads) {
        int run = 0;
        for (int w0 = 0; w0 < kPlanWarps; w0 += 8) {
            int n[8];
#pragma unroll
            for (int w = 0; w < 8; ++w) n[w] = hist[(w0 + w) * E + e];
#pragma unroll
            for (int w = 0; w < 8; ++w) {
                hist[(w0 + w) * E + e] = run;
                run += n[w];
            }
        }
        sh.total[e] = run;
    }
    if (ctas > 1) cluster_barrier(); else __syncthreads();

    // thread e: the expert's count, its place in the CTAs, and the scan of the padded counts
    int before = 0, count = 0;
    if (tid < E) {
        for (int c = 0; c < ctas; ++c) {
            const int n = ctas > 1 ? ld_cta(&sh.total[tid], uint32_t(c)) : sh.total[tid];
            if (c < int(cta)) before += n;
            count += n;
        }
    }
    const int64_t padded = (count + a.alignment - 1) / a.alignment * a.alignment;
    int64_t incl = padded;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t v = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= d) incl += v;
    }
    if (lane == 31) sh.scan[warp + 1] = incl;
    if (tid == 0) sh.scan[0] = 0;
    __syncthreads();
    if (warp == 0) {
        int64_t v = sh.scan[lane + 1];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, v, d);
            if (lane >= d) v += u;
        }
        sh.scan[lane + 1] = v;
    }
    __syncthreads();
    const int64_t offset = sh.scan[warp] + incl - padded;
    if (tid < E) {
        sh.base[tid] = int(offset) + before;
        sh.count[tid] = count;
        if (cta == 0) {
            a.expert_counts[tid] = count;
            a.expert_offsets[tid] = offset;
            if (tid == E - 1) a.expert_offsets[E] = offset + padded;
        }
        // rows of this expert's range that hold nothing
        for (int64_t s = offset + count + cta; s < offset + padded; s += ctas) a.slot_map[s] = -1;
    }
    __syncthreads();
    const int64_t end = sh.scan[kPlanWarps];
    for (int64_t s = end + int64_t(cta) * kPlanThreads + tid; s < a.capacity; s += int64_t(ctas) * kPlanThreads) a.slot_map[s] = -1;

    auto place_32 = [&](int64_t at, int e, uint32_t same) {
        const int64_t i = at + lane;
        int slot = -1;
        if (e < E) slot = sh.base[e] + mine[e] + __popc(same & ((1u << lane) - 1));
        __syncwarp();
        if (e < E && lane == __ffs(same) - 1) mine[e] += __popc(same);
        __syncwarp();
        if (i < last) {
            a.slots[i] = slot;
            if (slot >= 0) a.slot_map[slot] = int(i);
        }
    };
    if (kInRegisters) {
#pragma unroll
        for (int j = 0; j < kKept; ++j)
            if (first + j * 32 < last) place_32(first + j * 32, kept[j], kept_same[j]);
    } else {
        for (int64_t at = first; at < last; at += 32) {
            const int e = read(at + lane);
            place_32(at, e, same_expert(e, bits));
        }
    }
    if (ctas > 1) cluster_barrier();  // nobody's totals go away while another CTA reads them
}

// ------------------------------------------------------------------------------------------------ sort
// A warp per token and piece of its row: the piece is read once and written to every slot of the token.  Behind those, a warp per
// kZeroRows slots clears the rows that hold nothing.
constexpr int kCopyThreads = 256, kZeroRows = 4;

template <typename V>
__device__ __forceinline__ V zero_of() { return V{}; }

template <typename V, int kVecs>
__device__ __forceinline__ void copy_piece(const V* src, V* dst, int64_t vecs, int64_t first, int lane, const SortArgs& a, int my_slot) {
    V v[kVecs];
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
        const int64_t c = first + j * 32 + lane;
        if (c < vecs) v[j] = src[c];
    }
    for (int k = 0; k < a.topk; ++k) {
        const int slot = __shfl_sync(0xffffffffu, my_slot, k);
        if (uint32_t(slot) >= uint64_t(a.capacity)) continue;
        V* row = dst + int64_t(slot) * vecs;
#pragma unroll
        for (int j = 0; j < kVecs; ++j) {
            const int64_t c = first + j * 32 + lane;
            if (c < vecs) row[c] = v[j];
        }
    }
}

template <typename V, int kVecs>
__global__ void __launch_bounds__(kCopyThreads) sort_kernel(const SortArgs a, int pieces, int64_t copy_warps) {
    const int lane = threadIdx.x & 31;
    const int64_t warp = int64_t(blockIdx.x) * (kCopyThreads / 32) + (threadIdx.x >> 5);
    const int64_t vecs = a.row_bytes / int64_t(sizeof(V)), words = a.extra_bytes / 4;
    if (warp < copy_warps) {
        const int64_t t = warp / pieces;
        const int piece = int(warp % pieces);
        const int slot = lane < a.topk ? a.slots[t * a.topk + lane] : -1;
        copy_piece<V, kVecs>(static_cast<const V*>(a.x) + t * vecs, static_cast<V*>(a.rows), vecs, int64_t(piece) * 32 * kVecs, lane, a, slot);
        if (words > 0 && piece == pieces - 1)
            for (int64_t c = 0; c < words; c += 64)
                copy_piece<uint32_t, 2>(static_cast<const uint32_t*>(a.extra) + t * words, static_cast<uint32_t*>(a.extra_rows), words, c, lane, a, slot);
        return;
    }
    if (!a.zero_padding) return;
    const int64_t s0 = (warp - copy_warps) * kZeroRows;
    for (int64_t s = s0; s < min(a.capacity, s0 + kZeroRows); ++s) {
        if (a.slot_map[s] >= 0) continue;
        for (int64_t c = lane; c < vecs; c += 32) static_cast<V*>(a.rows)[s * vecs + c] = zero_of<V>();
        for (int64_t c = lane; c < words; c += 32) static_cast<uint32_t*>(a.extra_rows)[s * words + c] = 0u;
    }
}

// ------------------------------------------------------------------------------------------------ back
// A warp per token and 256 columns; the rows of a token are read eight at a time and added in ascending k, in 32 bits.
template <typename T, bool kAligned>
__device__ __forceinline__ void load8(const T* row, int c, int hidden, float* f) {
    if (kAligned) {
        Raw8<T> raw;
        raw.load(row + c);
        raw.get(f);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = c + j < hidden ? to_float(row[c + j]) : 0.f;
    }
}
template <typename T, bool kAligned>
__device__ __forceinline__ void store8(T* row, int c, int hidden, const float* f) {
    if (kAligned) {
        Raw8<T> raw;
        raw.set(f);
        raw.store(row + c);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (c + j < hidden) row[c + j] = from_float<T>(f[j]);
    }
}

// Eight columns as they lie in memory; `get` converts them.  Loads of several rows stay in flight only if none is converted in between.
template <typename T, bool kAligned>
struct Eight {
    Raw8<T> raw;
    __device__ __forceinline__ void load(const T* row, int c, int hidden) {
        if (kAligned) {
            raw.load(row + c);
        } else {
            float f[8];
            load8<T, false>(row, c, hidden, f);
            raw.set(f);
        }
    }
};

template <typename T, bool kAligned>
__global__ void __launch_bounds__(256) unsort_kernel(const UnsortArgs a, int pieces) {
    const int lane = threadIdx.x & 31;
    const int64_t warp = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5);
    const int64_t t = warp / pieces;
    if (t >= a.tokens) return;
    const int c = int(warp % pieces) * 256 + lane * 8;
    const bool inside = c < a.hidden;
    const int my_slot = lane < a.topk ? a.slots[t * a.topk + lane] : -1;
    const float my_weight = a.weights != nullptr && lane < a.topk ? a.weights[t * a.topk + lane] : 1.f;
    const T* y = static_cast<const T*>(a.y);
    float acc[8] = {};
    for (int k0 = 0; k0 < a.topk; k0 += 8) {
        Eight<T, kAligned> f[8];
        uint32_t real = 0;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int slot = k0 + k < a.topk ? __shfl_sync(0xffffffffu, my_slot, (k0 + k) & 31) : -1;
            const bool there = uint32_t(slot) < uint64_t(a.capacity);
            real |= uint32_t(there) << k;
            f[k].raw.clear();
            if (there && inside) f[k].load(y + int64_t(slot) * a.hidden, c, a.hidden);
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const float w = __shfl_sync(0xffffffffu, my_weight, (k0 + k) & 31);
            if ((real >> k & 1u) == 0) continue;  // a masked choice's weight may be anything
            float v[8];
            f[k].raw.get(v);
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] += w * v[j];
        }
    }
    if (!inside) return;
    if (a.bias != nullptr) {
        float b[8];
        load8<T, kAligned>(static_cast<const T*>(a.bias) + t * a.hidden, c, a.hidden, b);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] += b[j];
    }
    store8<T, kAligned>(static_cast<T*>(a.out) + t * a.hidden, c, a.hidden, acc);
}

// A block per token: its gradient row stays in the SM's first cache while every choice's row is read, multiplied and written.
template <typename T, bool kAligned>
__global__ void __launch_bounds__(256) unsort_grad_kernel(const UnsortGradArgs a) {
    __shared__ double part[8][kMaxTopk];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    if (int64_t(blockIdx.x) >= a.tokens) {  // rows without a choice
        const int64_t s0 = (int64_t(blockIdx.x) - a.tokens) * 8 * kZeroRows + warp * kZeroRows;
        const float zero[8] = {};
        for (int64_t s = s0; s < min(a.capacity, s0 + kZeroRows); ++s)
            if (a.slot_map[s] < 0)
                for (int c = lane * 8; c < a.hidden; c += 256) store8<T, kAligned>(static_cast<T*>(a.grad_y) + s * a.hidden, c, a.hidden, zero);
        return;
    }
    const int64_t t = blockIdx.x;
    const T* g_row = static_cast<const T*>(a.grad_out) + t * a.hidden;
    for (int k = 0; k < a.topk; ++k) {
        const int slot = a.slots[t * a.topk + k];
        double dot = 0.0;  // of eight products in 32 bits at a time: the sum may be far smaller than its terms
        if (uint32_t(slot) < uint64_t(a.capacity)) {
            const float w = a.weights != nullptr ? a.weights[t * a.topk + k] : 1.f;
            const T* y_row = static_cast<const T*>(a.y) + int64_t(slot) * a.hidden;
            for (int c = threadIdx.x * 8; c < a.hidden; c += 256 * 8) {
                float g[8], y[8];
                load8<T, kAligned>(g_row, c, a.hidden, g);
                if (a.grad_weights != nullptr) {
                    load8<T, kAligned>(y_row, c, a.hidden, y);
                    float eight = 0.f;
#pragma unroll
                    for (int j = 0; j < 8; ++j) eight += g[j] * y[j];
                    dot += double(eight);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) g[j] *= w;
                store8<T, kAligned>(static_cast<T*>(a.grad_y) + int64_t(slot) * a.hidden, c, a.hidden, g);
            }
        }
#pragma unroll
        for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        if (lane == 0) part[warp][k] = dot;
    }
    __syncthreads();
    if (a.grad_weights != nullptr && threadIdx.x < a.topk) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < 8; ++i) s += part[i][threadIdx.x];
        a.grad_weights[t * a.topk + threadIdx.x] = float(s);
    }
}

template <typename V, int kVecs>
cudaError_t sort_width(const SortArgs& a, cudaStream_t stream) {
    const int64_t vecs = a.row_bytes / int64_t(sizeof(V));
    const int pieces = int((vecs + 32 * kVecs - 1) / (32 * kVecs));
    const int64_t copy = a.tokens * pieces, zero = a.zero_padding ? (a.capacity + kZeroRows - 1) / kZeroRows : 0;
    const int64_t grid = (copy + zero + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
    if (grid == 0) return cudaSuccess;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    sort_kernel<V, kVecs><<<unsigned(grid), kCopyThreads, 0, stream>>>(a, pieces, copy);
    return cudaGetLastError();
}

template <typename T>
cudaError_t unsort_typed(const UnsortArgs& a, cudaStream_t stream) {
    const int pieces = (a.hidden + 255) / 256;
    const int64_t grid = (a.tokens * pieces + 7) / 8;
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    if (a.aligned) unsort_kernel<T, true><<<unsigned(grid), 256, 0, stream>>>(a, pieces);
    else unsort_kernel<T, false><<<unsigned(grid), 256, 0, stream>>>(a, pieces);
    return cudaGetLastError();
}

template <typename T>
cudaError_t unsort_grad_typed(const UnsortGradArgs& a, cudaStream_t stream) {
    const int64_t grid = a.tokens + (a.capacity + 8 * kZeroRows - 1) / (8 * kZeroRows);
    if (grid > 0x7fffffff) return cudaErrorInvalidValue;
    if (a.aligned) unsort_grad_kernel<T, true><<<unsigned(grid), 256, 0, stream>>>(a);
    else unsort_grad_kernel<T, false><<<unsigned(grid), 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_plan(const PlanArgs& a, cudaStream_t stream) {
    // up to 32 choices a warp one CTA is enough; more CTAs than 8 would need a non-portable cluster
    int ctas = 1;
    while (ctas < kMaxPlanCtas && a.choices > int64_t(ctas) * kPlanThreads) ctas *= 2;
    const int64_t warps = int64_t(ctas) * kPlanWarps;
    const int64_t per_warp = ((a.choices + warps - 1) / warps + 31) / 32 * 32;
    const size_t smem = sizeof(PlanShared) + size_t(kPlanWarps) * a.experts * sizeof(int);
    auto* fn = per_warp <= 32 * kKept ? plan_kernel<true> : plan_kernel<false>;
    static std::atomic<uint64_t> raised[2];
    const cudaError_t e = raise_shared_limit(fn, int(sizeof(PlanShared) + size_t(kPlanWarps) * kMaxExperts * sizeof(int)), raised[per_warp <= 32 * kKept]);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(ctas));
    config.blockDim = dim3(kPlanThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(ctas);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, fn, a, ctas, per_warp);
}

cudaError_t launch_sort(const SortArgs& a, cudaStream_t stream) {
    const uintptr_t bits = reinterpret_cast<uintptr_t>(a.x) | reinterpret_cast<uintptr_t>(a.rows) | uintptr_t(a.row_bytes);
    if (bits % 16 == 0) return sort_width<uint4, 4>(a, stream);
    if (bits % 4 == 0) return sort_width<uint32_t, 8>(a, stream);
    if (bits % 2 == 0) return sort_width<uint16_t, 8>(a, stream);
    return sort_width<uint8_t, 8>(a, stream);
}

cudaError_t launch_unsort(const UnsortArgs& a, Type type, cudaStream_t stream) {
    if (type == kBf16) return unsort_typed<__nv_bfloat16>(a, stream);
    if (type == kF16) return unsort_typed<__half>(a, stream);
    return unsort_typed<float>(a, stream);
}

cudaError_t launch_unsort_grad(const UnsortGradArgs& a, Type type, cudaStream_t stream) {
    if (type == kBf16) return unsort_grad_typed<__nv_bfloat16>(a, stream);
    if (type == kF16) return unsort_grad_typed<__half>(a, stream);
    return unsort_grad_typed<float>(a, stream);
}

}  // namespace order
}  // namespace nep

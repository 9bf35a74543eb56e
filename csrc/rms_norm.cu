// Root-mean-square norm in front of the experts, with the residual's addition and an output in 8 bits:
//
//   h = round(x + r),  rstd = 1 / sqrt(mean(h^2) + eps),  y = h * w * rstd,
//   per block of 128 columns:  m = max(max |h * w|, 1e-30),  q = e4m3(h * w * 448 / m),  scale = m * rstd / 448.
//
// rstd cancels in q: it is left out there, which keeps products on the border of two e4m3 values where they are.
#include "rms_norm.hpp"

#include <algorithm>
#include <type_traits>

#include "row_prim.cuh"

namespace nep {
namespace norm {
namespace {

using namespace rows;

constexpr int kNormThreads = 512;

// Products of two bf16 values have 16 bits.
template <typename T, typename W>
using ProductBlock = std::conditional_t<std::is_same<T, __nv_bfloat16>::value && std::is_same<W, __nv_bfloat16>::value, NarrowBlock, WideBlock>;
template <typename T>
using ValueBlock = std::conditional_t<std::is_same<T, float>::value, WideBlock, NarrowBlock>;

// Sum over the block, the same value in every thread; `scratch` holds 32 floats and is free again after the next block barrier.
__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5;
    float s = 0.f;
    for (int i = 0; i < warps; ++i) s += scratch[i];
    return s;
}

// A row per block and turn, eight columns per thread and unit, rows and weights in registers: a block of 128 columns is 16 neighbouring
// lanes.  The next row's loads are under way while a row is worked on: what bounds the kernel is memory, and a block that loads, meets and
// stores one after the other leaves it idle (4096 rows of 7168, all outputs: 62 us with a block per row).
template <typename T, typename W, int kUnits>
__global__ void __launch_bounds__(kNormThreads, sizeof(T) + sizeof(W) == 4 && kUnits <= 2 ? 2 : 1) norm_kernel(const NormArgs a) {
    __shared__ float scratch[2][32];
    const int units = a.hidden / 8, blocks = (a.hidden + kBlock - 1) / kBlock;
    Raw8<W> weight[kUnits];
    Raw8<T> raw[kUnits], add[kUnits];
    auto load = [&](int64_t row) {
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = threadIdx.x + i * blockDim.x;
            raw[i].clear();
            add[i].clear();
            if (row >= a.tokens || u >= units) continue;
            raw[i].load(static_cast<const T*>(a.x) + row * a.hidden + u * 8);
            if (a.residual != nullptr) add[i].load(static_cast<const T*>(a.residual) + row * a.hidden + u * 8);
        }
    };
    load(blockIdx.x);
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * blockDim.x;
        weight[i].clear();
        if (u < units) weight[i].load(static_cast<const W*>(a.weight) + u * 8);
    }
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x, turn ^= 1) {
        Raw8<T> h[kUnits];
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = threadIdx.x + i * blockDim.x;
            float v[8];
            h[i] = raw[i];
            h[i].get(v);
            if (a.residual != nullptr) {
                float f[8];
                add[i].get(f);
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] += f[j];
                h[i].set(v);  // the stream is held in its type, and that is what the norm sees
                if (u < units) h[i].store(static_cast<T*>(a.stream_out) + row * a.hidden + u * 8);
                h[i].get(v);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) sum += v[j] * v[j];
        }
        load(row + gridDim.x);
        const float rstd = rsqrtf(block_sum(sum, scratch[turn]) / float(a.hidden) + a.eps);
        if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = threadIdx.x + i * blockDim.x;
            float f[8], v[8], m = 0.f;
            h[i].get(v);
            weight[i].get(f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                f[j] *= v[j];
                m = max_nan(m, fabsf(f[j]));
            }
            if (a.q != nullptr) {
                m = max_nan(group_max<16>(m), kTiny);
                if (u < units) {
                    const ProductBlock<T, W> block(m);
                    *reinterpret_cast<uint2*>(a.q + row * a.hidden + u * 8) = make_uint2(block.pack(f), block.pack(f + 4));
                    if ((u & 15) == 0) a.scales[row * blocks + u / 16] = __fdiv_rn(m * rstd, kLargest);
                }
            }
            if (a.y != nullptr && u < units) {
#pragma unroll
                for (int j = 0; j < 8; ++j) f[j] *= rstd;
                Raw8<T> out;
                out.set(f);
                out.store(static_cast<T*>(a.y) + row * a.hidden + u * 8);
            }
        }
    }
}

// Any width and alignment, and rows too long for registers: a warp per block of 128 columns, the row read three times.
template <typename T, typename W>
__global__ void __launch_bounds__(512) norm_any_kernel(const NormArgs a) {
    __shared__ float scratch[32];
    const int64_t row = blockIdx.x, at = row * a.hidden;
    const T* x = static_cast<const T*>(a.x) + at;
    const T* r = a.residual != nullptr ? static_cast<const T*>(a.residual) + at : nullptr;
    const W* w = static_cast<const W*>(a.weight);
    auto value = [&](int c) { return r != nullptr ? to_float(from_float<T>(to_float(x[c]) + to_float(r[c]))) : to_float(x[c]); };
    float sum = 0.f;
    for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) {
        const float h = value(c);
        sum += h * h;
        if (r != nullptr) static_cast<T*>(a.stream_out)[at + c] = from_float<T>(h);
    }
    const float rstd = rsqrtf(block_sum(sum, scratch) / float(a.hidden) + a.eps);
    if (a.rstd != nullptr && threadIdx.x == 0) a.rstd[row] = rstd;
    const int blocks = (a.hidden + kBlock - 1) / kBlock, lane = threadIdx.x & 31;
    for (int b = threadIdx.x >> 5; b < blocks; b += blockDim.x >> 5) {
        float f[4], m = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = b * kBlock + j * 32 + lane;
            f[j] = c < a.hidden ? value(c) * to_float(w[c]) : 0.f;
            m = max_nan(m, fabsf(f[j]));
        }
        m = max_nan(group_max<32>(m), kTiny);
        const ProductBlock<T, W> block(m);
        const uint32_t q = a.q != nullptr ? block.pack(f) : 0u;
        if (a.q != nullptr && lane == 0) a.scales[row * blocks + b] = __fdiv_rn(m * rstd, kLargest);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = b * kBlock + j * 32 + lane;
            if (c >= a.hidden) continue;
            if (a.q != nullptr) a.q[at + c] = uint8_t(q >> (8 * j));
            if (a.y != nullptr) static_cast<T*>(a.y)[at + c] = from_float<T>(f[j] * rstd);
        }
    }
}

// Gradients.  With xhat = h * rstd and g = dy * w:  dx = rstd * (g - xhat * mean(g * xhat)) + dh;  dw = sum over rows of dy * xhat.
// A block takes every grid-th row and keeps its columns' part of dw in registers, so the sum has one order on every run.
template <typename T, typename W, int kUnits>
__global__ void __launch_bounds__(512) norm_grad_kernel(const NormGradArgs a) {
    __shared__ float scratch[2][32];
    const int units = a.hidden / 8;
    float dw[kUnits][8] = {};
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x, turn ^= 1) {
        const int64_t at = row * a.hidden;
        const float rstd = a.rstd[row];
        float g[kUnits][8], xhat[kUnits][8], dot = 0.f;
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = threadIdx.x + i * blockDim.x;
            Raw8<T> dy, h;
            Raw8<W> w;
            dy.clear();
            h.clear();
            w.clear();
            if (u < units) {
                dy.load(static_cast<const T*>(a.grad_y) + at + u * 8);
                h.load(static_cast<const T*>(a.h) + at + u * 8);
                w.load(static_cast<const W*>(a.weight) + u * 8);
            }
            float f[8];
            dy.get(g[i]);
            h.get(xhat[i]);
            w.get(f);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                xhat[i][j] *= rstd;
                dw[i][j] += g[i][j] * xhat[i][j];
                g[i][j] *= f[j];
                dot += g[i][j] * xhat[i][j];
            }
        }
        const float mean = block_sum(dot, scratch[turn]) / float(a.hidden);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
            const int u = threadIdx.x + i * blockDim.x;
            if (u >= units) continue;
            float f[8] = {};
            if (a.grad_stream != nullptr) {
                Raw8<T> dh;
                dh.load(static_cast<const T*>(a.grad_stream) + at + u * 8);
                dh.get(f);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] += rstd * (g[i][j] - xhat[i][j] * mean);
            Raw8<T> out;
            out.set(f);
            out.store(static_cast<T*>(a.grad_x) + at + u * 8);
        }
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int u = threadIdx.x + i * blockDim.x;
        if (u >= units) continue;
        Raw8<float> out;
        out.set(dw[i]);
        out.store(a.partial + int64_t(blockIdx.x) * a.hidden + u * 8);
    }
}

template <typename T, typename W>
__global__ void __launch_bounds__(512) norm_grad_any_kernel(const NormGradArgs a) {
    __shared__ float scratch[2][32];
    float* partial = a.partial + int64_t(blockIdx.x) * a.hidden;
    for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) partial[c] = 0.f;
    int turn = 0;
    for (int64_t row = blockIdx.x; row < a.tokens; row += gridDim.x, turn ^= 1) {
        const int64_t at = row * a.hidden;
        const float rstd = a.rstd[row];
        const T *dy = static_cast<const T*>(a.grad_y) + at, *h = static_cast<const T*>(a.h) + at;
        const T* dh = a.grad_stream != nullptr ? static_cast<const T*>(a.grad_stream) + at : nullptr;
        const W* w = static_cast<const W*>(a.weight);
        float dot = 0.f;
        for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) {
            const float xhat = to_float(h[c]) * rstd, g = to_float(dy[c]);
            partial[c] += g * xhat;  // this thread's column alone
            dot += g * to_float(w[c]) * xhat;
        }
        const float mean = block_sum(dot, scratch[turn]) / float(a.hidden);
        for (int c = threadIdx.x; c < a.hidden; c += blockDim.x) {
            const float xhat = to_float(h[c]) * rstd, g = to_float(dy[c]) * to_float(w[c]);
            static_cast<T*>(a.grad_x)[at + c] = from_float<T>((dh != nullptr ? to_float(dh[c]) : 0.f) + rstd * (g - xhat * mean));
        }
    }
}

// dw = the blocks' parts, each warp a run of the blocks, the runs in order: 32 columns per thread block.
template <typename W>
__global__ void __launch_bounds__(1024) norm_grad_weight_kernel(const float* partial, W* grad_weight, int blocks, int hidden) {
    __shared__ float part[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    const int each = (blocks + 31) / 32, first = warp * each, last = min(blocks, first + each);
    float s = 0.f;
    if (c < hidden) {
#pragma unroll 4
        for (int b = first; b < last; ++b) s += partial[int64_t(b) * hidden + c];
    }
    part[warp][lane] = s;
    __syncthreads();
    // a warp per column: the runs' sums meet in a tree
    const float t = warp_sum(part[lane][warp]);
    if (lane == 0 && blockIdx.x * 32 + warp < hidden) grad_weight[blockIdx.x * 32 + warp] = from_float<W>(t);
}

// Rows to 8 bits without a norm: 16 lanes per block of 128 columns.
template <typename T>
__global__ void __launch_bounds__(256) quantize_kernel(const QuantizeArgs a) {
    const int blocks = (a.columns + kBlock - 1) / kBlock;
    const int64_t total = a.rows * blocks, first = (int64_t(blockIdx.x) * blockDim.x + threadIdx.x) / 16;
    const int part = threadIdx.x & 15;
    // the lanes of a warp stay together for the exchange of their largest value: the bound is that of the warp's first block
    for (int64_t b = first; (b & ~int64_t(1)) < total; b += int64_t(gridDim.x) * blockDim.x / 16) {
        const int64_t row = b / blocks;
        const int block = int(b % blocks), c = block * kBlock + part * 8;
        const bool inside = b < total && c < a.columns;
        const int64_t at = row * a.columns + c;
        float f[8] = {}, m = 0.f;
        if (inside) {
            if (a.aligned) {
                Raw8<T> raw;
                raw.load(static_cast<const T*>(a.x) + at);
                raw.get(f);
            } else {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (c + j < a.columns) f[j] = to_float(static_cast<const T*>(a.x)[at + j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max_nan(m, fabsf(f[j]));
        m = max_nan(group_max<16>(m), kTiny);
        if (!inside) continue;
        if (part == 0) a.scales[b] = __fdiv_rn(m, kLargest);
        const ValueBlock<T> block_of(m);
        const uint2 q = make_uint2(block_of.pack(f), block_of.pack(f + 4));
        if (a.aligned) {
            *reinterpret_cast<uint2*>(a.q + at) = q;
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j < a.columns) a.q[at + j] = uint8_t((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
        }
    }
}

template <typename T, typename W>
cudaError_t norm_typed(const NormArgs& a, int sms, cudaStream_t stream) {
    const int units = a.hidden / 8;
    if (!a.aligned || units > 4 * kNormThreads) {
        norm_any_kernel<T, W><<<unsigned(a.tokens), 512, 0, stream>>>(a);
        return cudaGetLastError();
    }
    const int per = units <= kNormThreads ? 1 : units <= 2 * kNormThreads ? 2 : 4;
    const int threads = ((units + per - 1) / per + 31) / 32 * 32;
    // as many blocks as an SM's registers hold
    const unsigned grid = unsigned(std::min<int64_t>(a.tokens, int64_t(sms) * std::max(1, std::min(16, (per == 1 ? 1536 : 1024) / threads))));
    if (per == 1) norm_kernel<T, W, 1><<<grid, threads, 0, stream>>>(a);
    if (per == 2) norm_kernel<T, W, 2><<<grid, threads, 0, stream>>>(a);
    if (per == 4) norm_kernel<T, W, 4><<<grid, threads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T, typename W>
cudaError_t norm_grad_typed(const NormGradArgs& a, int sms, cudaStream_t stream) {
    const int blocks = grad_blocks(a.tokens, sms), units = a.hidden / 8;
    if (!a.aligned || units > 4 * 512) {
        norm_grad_any_kernel<T, W><<<blocks, 512, 0, stream>>>(a);
    } else {
        const int per = units <= 512 ? 1 : units <= 1024 ? 2 : 4;
        const int threads = ((units + per - 1) / per + 31) / 32 * 32;
        if (per == 1) norm_grad_kernel<T, W, 1><<<blocks, threads, 0, stream>>>(a);
        if (per == 2) norm_grad_kernel<T, W, 2><<<blocks, threads, 0, stream>>>(a);
        if (per == 4) norm_grad_kernel<T, W, 4><<<blocks, threads, 0, stream>>>(a);
    }
    norm_grad_weight_kernel<W><<<(a.hidden + 31) / 32, 1024, 0, stream>>>(a.partial, static_cast<W*>(a.grad_weight), blocks, a.hidden);
    return cudaGetLastError();
}

}  // namespace

cudaError_t launch_norm(const NormArgs& a, Type type, int sms, cudaStream_t stream) {
    if (type == kF32) return norm_typed<float, float>(a, sms, stream);
    if (type == kF16) return a.weight_f32 ? norm_typed<__half, float>(a, sms, stream) : norm_typed<__half, __half>(a, sms, stream);
    return a.weight_f32 ? norm_typed<__nv_bfloat16, float>(a, sms, stream) : norm_typed<__nv_bfloat16, __nv_bfloat16>(a, sms, stream);
}

int grad_blocks(int64_t tokens, int sms) { return int(tokens < 2 * sms ? tokens : 2 * sms); }

cudaError_t launch_norm_grad(const NormGradArgs& a, Type type, int sms, cudaStream_t stream) {
    if (type == kF32) return norm_grad_typed<float, float>(a, sms, stream);
    if (type == kF16) return a.weight_f32 ? norm_grad_typed<__half, float>(a, sms, stream) : norm_grad_typed<__half, __half>(a, sms, stream);
    return a.weight_f32 ? norm_grad_typed<__nv_bfloat16, float>(a, sms, stream) : norm_grad_typed<__nv_bfloat16, __nv_bfloat16>(a, sms, stream);
}

cudaError_t launch_quantize(const QuantizeArgs& a, Type type, cudaStream_t stream) {
    const int64_t blocks = a.rows * ((a.columns + kBlock - 1) / kBlock), needed = (blocks + 15) / 16;
    const unsigned grid = unsigned(needed < (1 << 20) ? needed : 1 << 20);
    if (type == kBf16) quantize_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a);
    if (type == kF16) quantize_kernel<__half><<<grid, 256, 0, stream>>>(a);
    if (type == kF32) quantize_kernel<float><<<grid, 256, 0, stream>>>(a);
    return cudaGetLastError();
}

}  // namespace norm
}  // namespace nep

// Grouped product of e4m3 rows and e4m3 expert weights:
//
//   out[m, n] = sum over blocks b of 128 columns of  sa[m, b] * sw[e, n / 128, b] * (sum over k in b of a[m, k] * w[e, n, k])
//
// plain (times a factor per row) or silu(gate) * up, to bf16 or to e4m3 with a scale for each 128 output columns.
#include "fp8_gemm_sm100.hpp"

#include "row_prim.cuh"

namespace nep {
namespace fp8 {
namespace {

using namespace rows;

// 32 rows x 128 output columns per block of 256 threads; a thread holds 16 neighbouring columns of one row.
constexpr int kRows = 32, kCols = 128, kPitch = 128 + 4;

__device__ __forceinline__ float e4m3(uint8_t v) { return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3))); }

__global__ void __launch_bounds__(256) simple_kernel(const Args p) {
    __shared__ uint8_t a_tile[kRows][kPitch], w_tile[2][kCols][kPitch];
    __shared__ float a_scale[kRows];
    __shared__ int64_t tile_first, tile_last;
    __shared__ int tile_expert;
    const int tid = threadIdx.x, r = tid / 8, c0 = tid % 8 * 16, n0 = blockIdx.x * kCols, halves = p.swiglu ? 2 : 1;
    if (tid == 0) {
        int64_t left = blockIdx.y;
        tile_expert = -1;
        for (int e = 0; e < p.experts && tile_expert < 0; ++e) {
            const int64_t lo = p.expert_offsets ? p.expert_offsets[e] : 0, hi = p.expert_offsets ? p.expert_offsets[e + 1] : p.rows;
            if (lo < 0 || hi < lo || hi > p.rows || (e == 0 && lo != 0)) {
                if (atomicCAS(p.status, 0u, uint32_t(kBadOffsets)) == 0u) p.status[1] = uint32_t(e);
                break;
            }
            const int64_t n = p.expert_counts ? max(int64_t(0), min(p.expert_counts[e], hi - lo)) : hi - lo, tiles = (n + kRows - 1) / kRows;
            if (left < tiles) {
                tile_expert = e;
                tile_first = lo + left * kRows;
                tile_last = min(lo + n, tile_first + kRows);
            }
            left -= tiles;
        }
    }
    __syncthreads();
    const int e = tile_expert;
    if (e < 0) return;
    const int64_t row = tile_first + r;
    const bool real = row < tile_last;
    float acc[2][16] = {};
    for (int b = 0; b < p.k_blocks; ++b) {
        for (int i = tid; i < kRows * 128; i += 256) {
            const int rr = i / 128, k = i % 128;
            a_tile[rr][k] = tile_first + rr < tile_last && b * 128 + k < p.k ? p.a[(tile_first + rr) * p.k + b * 128 + k] : 0;
        }
        for (int h = 0; h < halves; ++h)
            for (int i = tid; i < kCols * 128; i += 256) {
                const int n = n0 + i / 128, k = i % 128;
                w_tile[h][i / 128][k] = n < p.n && b * 128 + k < p.k ? p.w[((int64_t(e) * halves + h) * p.n + n) * p.k + b * 128 + k] : 0;
            }
        if (tid < kRows) a_scale[tid] = tile_first + tid < tile_last ? p.a_scales[(tile_first + tid) * p.k_blocks + b] : 0.f;
        __syncthreads();
        for (int h = 0; h < halves; ++h) {
            float part[16] = {};
            for (int k = 0; k < 128; ++k) {
                const float a = e4m3(a_tile[r][k]);
#pragma unroll
                for (int j = 0; j < 16; ++j) part[j] += a * e4m3(w_tile[h][c0 + j][k]);
            }
            const float s = a_scale[r] * p.w_scales[((int64_t(e) * halves + h) * p.n_blocks + blockIdx.x) * p.k_blocks + b];
#pragma unroll
            for (int j = 0; j < 16; ++j) acc[h][j] += s * part[j];
        }
        __syncthreads();
    }
    const float scale = real && p.row_scale ? p.row_scale[row] : 1.f;
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        acc[0][j] = (p.swiglu ? acc[0][j] / (1.f + expf(-acc[0][j])) * acc[1][j] : acc[0][j]) * scale;
        m = max_nan(m, n0 + c0 + j < p.n ? fabsf(acc[0][j]) : 0.f);
    }
    m = max_nan(group_max<8>(m), kTiny);
    if (!real) return;
    if (p.q && c0 == 0) p.scales[row * p.n_blocks + blockIdx.x] = __fdiv_rn(m, kLargest);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int n = n0 + c0 + j;
        if (n >= p.n) break;
        if (p.q) p.q[row * p.n + n] = __nv_cvt_float_to_fp8(quotient(acc[0][j], m), __NV_SATFINITE, __NV_E4M3);
        else p.out[row * p.n + n] = __float2bfloat16_rn(acc[0][j]);
    }
}

}  // namespace

cudaError_t launch(const Args& p, int, cudaStream_t stream) {
    const int64_t tiles = p.rows / kRows + p.experts;
    if (tiles > 65535) return cudaErrorInvalidValue;
    simple_kernel<<<dim3(unsigned(p.n_blocks), unsigned(tiles)), 256, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace fp8
}  // namespace nep

// Launch interface of the 8-bit grouped GEMM with a scale for each block of 128 (fp8_gemm_sm100.cu).
#pragma once
#include <cstdint>
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include "layout.hpp"

namespace nep {
namespace fp8 {

constexpr int kMaxExperts = 1024;
enum Fp8Status : uint32_t { kPipeTimeout = 101, kBadOffsets = 106 };

// Two warps that hold one output block's columns swap their rows' largest values, tile after tile: each writes its own, arrives on its barrier and waits
// for the other's arrival.  Nothing else holds the two together where K has one or two blocks: a warp may arrive for the next tile before the other one has
// looked at its arrival for this tile, but it waits there for what the other tells for that next tile, behind the look.  So two turns are enough, with
// a barrier each: one barrier for both could go through two phases between two looks, and the wait for the first would not end.
constexpr int kExchangeTurns = 2;
struct ExchangeTurn {
    int at;           // place of the values, and of the barrier
    uint32_t parity;  // of that barrier's phase
};
NEP_HD ExchangeTurn exchange_turn(int exchange) { return ExchangeTurn{exchange % kExchangeTurns, uint32_t(exchange / kExchangeTurns) & 1u}; }

// Tensor maps: rows in boxes of 128, 64, 32 and 16 (by 128 columns), weights [experts (* 2)][n][k].
struct Maps {
    CUtensorMap weights;
    CUtensorMap rows[4];
};

struct Args {
    const float* a_scales;          // [rows, k_blocks]
    const float* w_scales;          // [experts, (2 *) n_blocks, k_blocks]
    const int64_t* expert_offsets;  // [experts + 1], or null: one expert owns all rows
    const int64_t* expert_counts;   // [experts] rows that exist, or null: all rows of the range
    const float* row_scale;         // or null: [rows]
    __nv_bfloat16* out;             // [rows, n], or
    uint8_t* q;                     // e4m3 [rows, n] with
    float* scales;                  // [rows, n_blocks]
    int64_t rows;
    int experts, n;                 // n: output columns (with SwiGLU half of the weight's rows)
    int k_blocks, n_blocks;         // of 128
    int n_tiles;                    // of 256 output columns; of 128 with SwiGLU, or (few rows) where that many are given
    int swiglu;
    uint32_t* status;               // 2 words: first error code, detail
    uint64_t timeout_ns;
};
// Rows as M (fp8_gemm_sm100.cu).  Weight boxes of 128 rows, 64 with SwiGLU.
cudaError_t launch(const Maps& maps, const Args& args, int grid, cudaStream_t stream);

// Few rows per expert: weights as M, `tile` (32 or 64) rows at most as N, the K axis split over clusters of `ctas` (1, 2, 4 or 8) CTAs
// (fp8_gemm_few_sm100.cu).  `units`: tiles that the rows allow.  Weight boxes of 128 rows.
cudaError_t launch_few(const Maps& maps, const Args& args, int tile, int ctas, int64_t units, int sms, cudaStream_t stream);
int few_clusters(int ctas, int sms);

}  // namespace fp8
}  // namespace nep

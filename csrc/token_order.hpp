// Launch interface of the token order: a batch sorted by expert and back, on one GPU without a peer window (token_order.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace nep {
namespace order {

constexpr int kMaxExperts = 1024, kMaxTopk = 32;
enum OrderStatus : uint32_t { kBadExpertId = 105 };

struct PlanArgs {
    const int64_t* topk_idx;   // [choices] expert of each choice, -1 = masked
    int* slots;                // [choices] row of the choice, -1 = masked
    int* slot_map;             // [capacity] choice of the row, -1 = padding
    int64_t* expert_counts;    // [experts]
    int64_t* expert_offsets;   // [experts + 1]
    int64_t choices, capacity;
    int experts;
    int64_t alignment;
    uint32_t* status;
};
cudaError_t launch_plan(const PlanArgs& args, cudaStream_t stream);

// rows[slots[t, k]] = x[t]; a second tensor of the same rows (their scales) travels along.
struct SortArgs {
    const void* x;         // [tokens] rows of row_bytes
    void* rows;            // [capacity] rows of row_bytes
    const void* extra;     // or null: [tokens] rows of extra_bytes
    void* extra_rows;
    const int* slots;      // [tokens, topk]
    const int* slot_map;   // [capacity]
    int64_t tokens, capacity;
    int topk;
    int64_t row_bytes, extra_bytes;
    bool zero_padding;
};
cudaError_t launch_sort(const SortArgs& args, cudaStream_t stream);

enum Type : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

// out[t] = bias[t] + sum over k of weights[t, k] * y[slots[t, k]]
struct UnsortArgs {
    const void* y;          // [capacity, hidden]
    const int* slots;       // [tokens, topk]
    const float* weights;   // or null: [tokens, topk]
    const void* bias;       // or null: [tokens, hidden]
    void* out;              // [tokens, hidden]
    int64_t tokens, capacity;
    int topk, hidden;
    bool aligned;           // hidden % 8 == 0 and every pointer on a 16-byte boundary
};
cudaError_t launch_unsort(const UnsortArgs& args, Type type, cudaStream_t stream);

// grad_y[slots[t, k]] = weights[t, k] * grad_out[t], zero in rows without a choice; grad_weights[t, k] = <grad_out[t], y[slots[t, k]]>
struct UnsortGradArgs {
    const void* grad_out;   // [tokens, hidden]
    const void* y;          // [capacity, hidden]; used for grad_weights
    const int* slots;
    const int* slot_map;
    const float* weights;   // or null: ones
    void* grad_y;           // [capacity, hidden]
    float* grad_weights;    // or null: [tokens, topk]
    int64_t tokens, capacity;
    int topk, hidden;
    bool aligned;
};
cudaError_t launch_unsort_grad(const UnsortGradArgs& args, Type type, cudaStream_t stream);

}  // namespace order
}  // namespace nep

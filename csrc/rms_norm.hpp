// Launch interface of the norm and of the rows' 8-bit form (rms_norm.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

namespace nep {
namespace norm {

enum Type : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

struct NormArgs {
    const void* x;          // [tokens, hidden]
    const void* residual;   // or null
    const void* weight;     // [hidden], of x's type or (weight_f32) 32 bits
    void* stream_out;       // x + residual in x's type, where there is a residual
    void* y;                // or null
    uint8_t* q;             // or null: e4m3 [tokens, hidden]
    float* scales;          // [tokens, ceil(hidden / 128)]
    float* rstd;            // or null: [tokens]
    int64_t tokens;
    int hidden;
    float eps;
    bool weight_f32;
    bool aligned;           // hidden % 8 == 0 and every pointer on a 16-byte boundary
};
cudaError_t launch_norm(const NormArgs& args, Type type, int sms, cudaStream_t stream);

struct NormGradArgs {
    const void* grad_y;         // [tokens, hidden]
    const void* h;              // what was normalised, [tokens, hidden]
    const void* weight;
    const float* rstd;          // [tokens]
    const void* grad_stream;    // or null: gradient of the residual stream behind the norm
    void* grad_x;               // [tokens, hidden]
    float* partial;             // [grad_blocks, hidden]
    void* grad_weight;          // [hidden]
    int64_t tokens;
    int hidden;
    bool weight_f32;
    bool aligned;
};
// Blocks that the gradient of the weight is summed in.
int grad_blocks(int64_t tokens, int sms);
cudaError_t launch_norm_grad(const NormGradArgs& args, Type type, int sms, cudaStream_t stream);

struct QuantizeArgs {
    const void* x;  // [rows, columns]
    uint8_t* q;
    float* scales;  // [rows, ceil(columns / 128)]
    int64_t rows;
    int columns;
    bool aligned;
};
cudaError_t launch_quantize(const QuantizeArgs& args, Type type, cudaStream_t stream);

}  // namespace norm
}  // namespace nep

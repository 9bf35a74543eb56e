// Python bindings of the operators around 8-bit experts: norm, token order, block-scaled product.  They check their arguments,
// allocate what they return on the caller's stream and launch there; none of them waits for the device.
#include "op_api.hpp"

#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include "fp8_gemm_sm100.hpp"
#include "peer_window.hpp"
#include "rms_norm.hpp"
#include "token_order.hpp"

namespace nep {
namespace {

// Messages hold no numbers but through std::to_string: numeric operator<< on iostreams is avoided throughout this extension.
static_assert(order::kMaxTopk == 32 && order::kMaxExperts == 1024 && fp8::kMaxExperts == 1024, "limits named in messages");

using OptTensor = c10::optional<at::Tensor>;

// A tensor on the device of `like` without the dispatcher: a small call's time is the host's, about a microsecond a tensor.
at::Tensor make_empty(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& like) {
    return at::Tensor(at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt));
}

// Element types in the numbering that norm::Type and order::Type share.
int row_type(const at::Tensor& t, const char* name) {
    const auto s = t.scalar_type();
    TORCH_CHECK(s == at::kBFloat16 || s == at::kHalf || s == at::kFloat, name, " must be bfloat16, float16 or float32");
    return s == at::kBFloat16 ? 0 : s == at::kHalf ? 1 : 2;
}

void check_rows(const at::Tensor& t, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.dim() == 2 && t.is_contiguous(), name, " must be a contiguous two-dimensional CUDA tensor");
}

void check_like(const OptTensor& t, const at::Tensor& x, const char* name) {
    if (!t.has_value()) return;
    TORCH_CHECK(t->is_cuda() && t->device() == x.device() && t->scalar_type() == x.scalar_type() && t->sizes() == x.sizes() && t->is_contiguous(), name,
                " must be a contiguous tensor of the rows' shape, type and device");
}

void check_status_tensor(const at::Tensor& status, const at::Tensor& x) {
    TORCH_CHECK(status.is_cuda() && status.device() == x.device() && status.scalar_type() == at::kInt && status.is_contiguous() && status.numel() >= 2,
                "status must be an int32 tensor on the operands' device");
}

bool on16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool on16(const OptTensor& t) { return !t.has_value() || on16(t->data_ptr()); }
const void* pointer(const OptTensor& t) { return t.has_value() ? t->data_ptr() : nullptr; }
int64_t blocks_of(int64_t columns) { return (columns + 127) / 128; }
int sm_count() { return at::cuda::getCurrentDeviceProperties()->multiProcessorCount; }

void launched(cudaError_t e, const char* what) {
    TORCH_CHECK(e == cudaSuccess, what, " launch failed: ", cudaGetErrorString(e));
    PeerWindow::launches += 1;
}

void check_weight(const at::Tensor& weight, const at::Tensor& x) {
    TORCH_CHECK(weight.is_cuda() && weight.device() == x.device() && weight.dim() == 1 && weight.is_contiguous() && weight.size(0) == x.size(1),
                "weight must be a contiguous tensor of hidden entries on the rows' device");
    TORCH_CHECK(weight.scalar_type() == x.scalar_type() || weight.scalar_type() == at::kFloat, "weight must have the rows' type or be float32");
}

void check_hidden(const at::Tensor& x) {
    TORCH_CHECK(x.size(1) >= 1 && x.size(1) <= (int64_t(1) << 28), "rows must have 1 to 2^28 columns");
    TORCH_CHECK(x.size(0) < (int64_t(1) << 31), "at most 2^31 - 1 rows");
}

// (y, q, scales, stream, rstd), undefined where not asked for
std::vector<OptTensor> rms_norm(const at::Tensor& x, const at::Tensor& weight, const OptTensor& residual, double eps, bool quantize, bool keep, bool save) {
    check_rows(x, "x");
    check_hidden(x);
    const int type = row_type(x, "x");
    check_weight(weight, x);
    check_like(residual, x, "residual");
    TORCH_CHECK(eps >= 0, "eps must not be negative");
    TORCH_CHECK(quantize || keep, "neither the rows nor their 8-bit form is asked for");
    c10::cuda::CUDAGuard guard(x.device());
    OptTensor y, q, scales, stream, rstd;
    if (keep) y = make_empty(x.sizes(), x.scalar_type(), x);
    if (quantize) {
        q = make_empty(x.sizes(), at::kFloat8_e4m3fn, x);
        scales = make_empty({x.size(0), blocks_of(x.size(1))}, at::kFloat, x);
    }
    if (residual.has_value()) stream = make_empty(x.sizes(), x.scalar_type(), x);
    if (save) rstd = make_empty({x.size(0)}, at::kFloat, x);
    if (x.size(0) > 0) {
        norm::NormArgs a{};
        a.x = x.data_ptr();
        a.residual = pointer(residual);
        a.weight = weight.data_ptr();
        a.stream_out = stream.has_value() ? stream->data_ptr() : nullptr;
        a.y = y.has_value() ? y->data_ptr() : nullptr;
        a.q = q.has_value() ? static_cast<uint8_t*>(q->data_ptr()) : nullptr;
        a.scales = scales.has_value() ? scales->data_ptr<float>() : nullptr;
        a.rstd = rstd.has_value() ? rstd->data_ptr<float>() : nullptr;
        a.tokens = x.size(0);
        a.hidden = int(x.size(1));
        a.eps = float(eps);
        a.weight_f32 = weight.scalar_type() == at::kFloat;
        a.aligned = a.hidden % 8 == 0 && on16(a.x) && on16(a.weight) && on16(residual);
        launched(norm::launch_norm(a, norm::Type(type), sm_count(), c10::cuda::getCurrentCUDAStream()), "rms_norm");
    }
    return {y, q, scales, stream, rstd};
}

std::pair<at::Tensor, at::Tensor> rms_norm_grad(const at::Tensor& grad_y, const at::Tensor& h, const at::Tensor& weight, const at::Tensor& rstd,
                                                const OptTensor& grad_stream) {
    check_rows(h, "h");
    check_hidden(h);
    const int type = row_type(h, "h");
    check_weight(weight, h);
    check_like(grad_y, h, "grad_y");
    check_like(grad_stream, h, "grad_residual");
    TORCH_CHECK(rstd.is_cuda() && rstd.device() == h.device() && rstd.scalar_type() == at::kFloat && rstd.is_contiguous() && rstd.dim() == 1 && rstd.size(0) == h.size(0),
                "rstd must be float32 [tokens] on the rows' device");
    c10::cuda::CUDAGuard guard(h.device());
    at::Tensor grad_x = make_empty(h.sizes(), h.scalar_type(), h);
    if (h.size(0) == 0) return {grad_x, at::zeros_like(weight)};
    at::Tensor grad_weight = make_empty(weight.sizes(), weight.scalar_type(), h);
    const int sms = sm_count();
    at::Tensor partial = make_empty({norm::grad_blocks(h.size(0), sms), h.size(1)}, at::kFloat, h);
    norm::NormGradArgs a{};
    a.grad_y = grad_y.data_ptr();
    a.h = h.data_ptr();
    a.weight = weight.data_ptr();
    a.rstd = rstd.data_ptr<float>();
    a.grad_stream = pointer(grad_stream);
    a.grad_x = grad_x.data_ptr();
    a.partial = partial.data_ptr<float>();
    a.grad_weight = grad_weight.data_ptr();
    a.tokens = h.size(0);
    a.hidden = int(h.size(1));
    a.weight_f32 = weight.scalar_type() == at::kFloat;
    a.aligned = a.hidden % 8 == 0 && on16(a.grad_y) && on16(a.h) && on16(a.weight) && on16(grad_stream);
    launched(norm::launch_norm_grad(a, norm::Type(type), sms, c10::cuda::getCurrentCUDAStream()), "rms_norm_grad");
    PeerWindow::launches += 1;  // and the sum of the blocks' parts
    return {grad_x, grad_weight};
}

std::pair<at::Tensor, at::Tensor> quantize_rows(const at::Tensor& x) {
    check_rows(x, "x");
    check_hidden(x);
    const int type = row_type(x, "x");
    c10::cuda::CUDAGuard guard(x.device());
    at::Tensor q = make_empty(x.sizes(), at::kFloat8_e4m3fn, x);
    at::Tensor scales = make_empty({x.size(0), blocks_of(x.size(1))}, at::kFloat, x);
    if (x.size(0) > 0) {
        norm::QuantizeArgs a{};
        a.x = x.data_ptr();
        a.q = static_cast<uint8_t*>(q.data_ptr());
        a.scales = scales.data_ptr<float>();
        a.rows = x.size(0);
        a.columns = int(x.size(1));
        a.aligned = a.columns % 8 == 0 && on16(a.x);
        launched(norm::launch_quantize(a, norm::Type(type), c10::cuda::getCurrentCUDAStream()), "quantize_rows");
    }
    return {q, scales};
}

// ------------------------------------------------------------------------------------------------ token order

// (slots, slot_map, expert_counts, expert_offsets)
std::tuple<at::Tensor, at::Tensor, at::Tensor, at::Tensor> plan_tokens(const at::Tensor& topk_idx, int64_t experts, int64_t alignment, const at::Tensor& status) {
    TORCH_CHECK(topk_idx.is_cuda() && topk_idx.scalar_type() == at::kLong && topk_idx.dim() == 2 && topk_idx.is_contiguous(),
                "topk_idx must be a contiguous int64 CUDA tensor [tokens, topk]");
    TORCH_CHECK(topk_idx.size(1) >= 1 && topk_idx.size(1) <= order::kMaxTopk, "topk must be 1 to 32");
    TORCH_CHECK(experts >= 1 && experts <= order::kMaxExperts, "num_experts must be 1 to 1024");
    TORCH_CHECK(alignment >= 1 && alignment <= 4096, "alignment must be 1 to 4096");
    check_status_tensor(status, topk_idx);
    const int64_t choices = topk_idx.numel();
    TORCH_CHECK(choices < (int64_t(1) << 30), "at most 2^30 choices");
    // every choice has a row whatever the routing: no more than min(experts, choices) ranges are rounded up
    const int64_t capacity = (choices + (std::min(experts, choices) + 1) * (alignment - 1)) / alignment * alignment;
    TORCH_CHECK(capacity < (int64_t(1) << 31), "at most 2^31 - 1 rows");
    c10::cuda::CUDAGuard guard(topk_idx.device());
    at::Tensor slots = make_empty(topk_idx.sizes(), at::kInt, topk_idx), slot_map = make_empty({capacity}, at::kInt, topk_idx);
    at::Tensor counts = make_empty({experts}, at::kLong, topk_idx), offsets = make_empty({experts + 1}, at::kLong, topk_idx);
    order::PlanArgs a{};
    a.topk_idx = topk_idx.data_ptr<int64_t>();
    a.slots = slots.data_ptr<int>();
    a.slot_map = slot_map.data_ptr<int>();
    a.expert_counts = counts.data_ptr<int64_t>();
    a.expert_offsets = offsets.data_ptr<int64_t>();
    a.choices = choices;
    a.capacity = capacity;
    a.experts = int(experts);
    a.alignment = alignment;
    a.status = reinterpret_cast<uint32_t*>(status.data_ptr<int>());
    launched(order::launch_plan(a, c10::cuda::getCurrentCUDAStream()), "plan_tokens");
    return {slots, slot_map, counts, offsets};
}

void check_order(const at::Tensor& slots, const at::Tensor& slot_map, const at::Tensor& x) {
    TORCH_CHECK(slots.is_cuda() && slots.device() == x.device() && slots.scalar_type() == at::kInt && slots.dim() == 2 && slots.is_contiguous() &&
                    slots.size(1) >= 1 && slots.size(1) <= order::kMaxTopk,
                "the order's slots must be contiguous int32 [tokens, topk] on the rows' device");
    TORCH_CHECK(slot_map.is_cuda() && slot_map.device() == x.device() && slot_map.scalar_type() == at::kInt && slot_map.dim() == 1 &&
                    slot_map.is_contiguous() && slot_map.size(0) < (int64_t(1) << 31),
                "the order's slot_map must be contiguous int32 [capacity] on the rows' device");
}

std::pair<at::Tensor, OptTensor> sort_tokens(const at::Tensor& x, const at::Tensor& slots, const at::Tensor& slot_map, const OptTensor& scales, bool zero_padding) {
    check_rows(x, "x");
    check_hidden(x);
    check_order(slots, slot_map, x);
    TORCH_CHECK(slots.size(0) == x.size(0), "x and the order must have the same tokens");
    const auto s = x.scalar_type();
    TORCH_CHECK(s == at::kBFloat16 || s == at::kHalf || s == at::kFloat || s == at::kFloat8_e4m3fn, "x must be bfloat16, float16, float32 or float8_e4m3fn");
    if (scales.has_value())
        TORCH_CHECK(scales->is_cuda() && scales->device() == x.device() && scales->scalar_type() == at::kFloat && scales->dim() == 2 && scales->is_contiguous() &&
                        scales->size(0) == x.size(0) && scales->size(1) >= 1,
                    "scales must be contiguous float32 [tokens, blocks] on the rows' device");
    c10::cuda::CUDAGuard guard(x.device());
    const int64_t capacity = slot_map.size(0);
    at::Tensor rows = make_empty({capacity, x.size(1)}, x.scalar_type(), x);
    OptTensor row_scales;
    if (scales.has_value()) row_scales = make_empty({capacity, scales->size(1)}, at::kFloat, x);
    order::SortArgs a{};
    a.x = x.data_ptr();
    a.rows = rows.data_ptr();
    if (scales.has_value()) {
        a.extra = scales->data_ptr();
        a.extra_rows = row_scales->data_ptr();
        a.extra_bytes = scales->size(1) * 4;
    }
    a.slots = slots.data_ptr<int>();
    a.slot_map = slot_map.data_ptr<int>();
    a.tokens = x.size(0);
    a.capacity = capacity;
    a.topk = int(slots.size(1));
    a.row_bytes = x.size(1) * x.element_size();
    a.zero_padding = zero_padding;
    if (capacity > 0) launched(order::launch_sort(a, c10::cuda::getCurrentCUDAStream()), "sort_tokens");
    return {rows, row_scales};
}

void check_gate(const OptTensor& weights, const at::Tensor& slots) {
    if (weights.has_value())
        TORCH_CHECK(weights->is_cuda() && weights->device() == slots.device() && weights->scalar_type() == at::kFloat && weights->sizes() == slots.sizes() &&
                        weights->is_contiguous(),
                    "weights must be contiguous float32 [tokens, topk] on the rows' device");
}

at::Tensor unsort_tokens(const at::Tensor& y, const at::Tensor& slots, const at::Tensor& slot_map, const OptTensor& weights, const OptTensor& bias) {
    check_rows(y, "y");
    check_hidden(y);
    const int type = row_type(y, "y");
    check_order(slots, slot_map, y);
    TORCH_CHECK(y.size(0) == slot_map.size(0), "y must have a row for every slot of the order");
    check_gate(weights, slots);
    if (bias.has_value())
        TORCH_CHECK(bias->is_cuda() && bias->device() == y.device() && bias->scalar_type() == y.scalar_type() && bias->dim() == 2 && bias->is_contiguous() &&
                        bias->size(0) == slots.size(0) && bias->size(1) == y.size(1),
                    "bias must be a contiguous [tokens, hidden] tensor of y's type and device");
    c10::cuda::CUDAGuard guard(y.device());
    at::Tensor out = make_empty({slots.size(0), y.size(1)}, y.scalar_type(), y);
    if (slots.size(0) == 0) return out;
    order::UnsortArgs a{};
    a.y = y.data_ptr();
    a.slots = slots.data_ptr<int>();
    a.weights = static_cast<const float*>(pointer(weights));
    a.bias = pointer(bias);
    a.out = out.data_ptr();
    a.tokens = slots.size(0);
    a.capacity = y.size(0);
    a.topk = int(slots.size(1));
    a.hidden = int(y.size(1));
    a.aligned = a.hidden % 8 == 0 && on16(a.y) && on16(bias);
    launched(order::launch_unsort(a, order::Type(type), c10::cuda::getCurrentCUDAStream()), "unsort_tokens");
    return out;
}

std::pair<at::Tensor, OptTensor> unsort_tokens_grad(const at::Tensor& grad_out, const at::Tensor& y, const at::Tensor& slots, const at::Tensor& slot_map,
                                                    const OptTensor& weights) {
    check_rows(y, "y");
    check_rows(grad_out, "grad_out");
    check_hidden(y);
    const int type = row_type(y, "y");
    check_order(slots, slot_map, y);
    check_gate(weights, slots);
    TORCH_CHECK(y.size(0) == slot_map.size(0), "y must have a row for every slot of the order");
    TORCH_CHECK(grad_out.device() == y.device() && grad_out.scalar_type() == y.scalar_type() && grad_out.size(0) == slots.size(0) && grad_out.size(1) == y.size(1),
                "grad_out must be a contiguous [tokens, hidden] tensor of y's type and device");
    c10::cuda::CUDAGuard guard(y.device());
    at::Tensor grad_y = make_empty(y.sizes(), y.scalar_type(), y);
    OptTensor grad_weights;
    if (weights.has_value()) grad_weights = make_empty(weights->sizes(), at::kFloat, y);
    order::UnsortGradArgs a{};
    a.grad_out = grad_out.data_ptr();
    a.y = y.data_ptr();
    a.slots = slots.data_ptr<int>();
    a.slot_map = slot_map.data_ptr<int>();
    a.weights = static_cast<const float*>(pointer(weights));
    a.grad_y = grad_y.data_ptr();
    a.grad_weights = grad_weights.has_value() ? grad_weights->data_ptr<float>() : nullptr;
    a.tokens = slots.size(0);
    a.capacity = y.size(0);
    a.topk = int(slots.size(1));
    a.hidden = int(y.size(1));
    a.aligned = a.hidden % 8 == 0 && on16(a.grad_out) && on16(a.y);
    if (a.tokens + a.capacity > 0) launched(order::launch_unsort_grad(a, order::Type(type), c10::cuda::getCurrentCUDAStream()), "unsort_tokens_grad");
    return {grad_y, grad_weights};
}

// ------------------------------------------------------------------------------------------------ product

using EncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                              const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Row-major 8-bit [rows, columns], or [outer, rows, columns]; box = 128 columns (one swizzle row) x box_rows rows.  What a box covers
// outside of the tensor reads as zero.
CUtensorMap e4m3_map(const void* base, int64_t columns, int64_t rows, int64_t outer, int box_rows) {
    static EncodeFn encode = [] {
        void* ptr = nullptr;
        cudaDriverEntryPointQueryResult result;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &result);
        TORCH_CHECK(e == cudaSuccess && result == cudaDriverEntryPointSuccess && ptr != nullptr, "cuTensorMapEncodeTiled is not available");
        return reinterpret_cast<EncodeFn>(ptr);
    }();
    CUtensorMap map;
    const cuuint64_t dims[3] = {cuuint64_t(columns), cuuint64_t(rows), cuuint64_t(outer)};
    const cuuint64_t strides[2] = {cuuint64_t(columns), cuuint64_t(rows) * cuuint64_t(columns)};
    const cuuint32_t box[3] = {128, cuuint32_t(box_rows), 1};
    const cuuint32_t elem[3] = {1, 1, 1};
    const CUresult r = encode(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, outer > 0 ? 3 : 2, const_cast<void*>(base), dims, strides, box, elem,
                              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    TORCH_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed");
    return map;
}

void check_e4m3(const at::Tensor& t, int dims, const char* name) {
    TORCH_CHECK(t.is_cuda() && t.scalar_type() == at::kFloat8_e4m3fn && t.is_contiguous() && t.dim() == dims, name,
                " must be a contiguous CUDA float8_e4m3fn tensor of the expected rank");
}

void check_i64(const OptTensor& t, const at::Tensor& a, int64_t entries, const char* name) {
    if (t.has_value())
        TORCH_CHECK(t->is_cuda() && t->device() == a.device() && t->scalar_type() == at::kLong && t->is_contiguous() && t->dim() == 1 && t->size(0) == entries, name,
                    " must be a contiguous int64 tensor of ", std::to_string(entries), " entries on the rows' device");
}

// Which kernel an 8-bit product runs.  tile = 128: rows as M (fp8_gemm_sm100.cu); 32 or 64: weights as M, so many rows at most as N, the K
// axis over `ctas` CTAs (fp8_gemm_few_sm100.cu).  `units`: tiles that the rows allow, whatever the offsets say.
//
// The choice is the shortest of the times that these kernels have taken, whole passes over the tiles at a time.  us a block of 128 columns: rows
// as M 0.62 on a few SMs and 0.69 on all; 32 rows as N 0.43 alone, 0.70 where all SMs stream weights from memory, 0.45 where L2 has
// them; 64 rows 0.61 and 0.86.  Behind a tile's last block: 2.7, and 2.5 + 0.3 a CTA for the exchange.  32 experts of 7168 x 2048, up, us for 32
// rows as N, 64, and rows as M: 32 rows an expert 157, 166, 172; 64 rows 199, 192, 174.  One matrix of 7168 x 4096, calls on eight such matrices by turns in a graph: one row
// 13.0 over four CTAs, 25.1 in one, 36.4; 128 rows, four CTAs, 23.1, 19.0, 41.0.  Tiles of one block of output columns instead of two (0.62 of a block's time each): one
// row 12.7 instead of 13.0, 64 rows (as 32s) 20.4 instead of 15.1.
struct Fp8Choice {
    int64_t tile, ctas, units, n_tiles;
};
Fp8Choice choose_fp8(int64_t rows, int64_t experts, int64_t most, int64_t n_blocks, bool swiglu, int64_t k_blocks, int64_t sms, int64_t tile, int64_t ctas,
                     int64_t columns) {
    // Rows of an expert: the average of the ranges, which may be padded (to 128 behind a dispatch), and at most what the caller says.  An expert of up
    // to 32 rows is one tile of any kind, so the largest of such a call counts rather than the average.
    const int64_t holders = std::min(experts, rows), spread = (rows + holders - 1) / holders;
    const int64_t average = most == 0 ? spread : most <= 32 ? most : std::min(spread, most);
    const auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
    Fp8Choice c{};
    constexpr double kHalfTile = 0.62;  // a block of a tile of 128 columns, of one of 256
    double best = -1;
    for (const int64_t t : {int64_t(32), int64_t(64), int64_t(128)}) {
        if (tile > 0 && t != tile) continue;
        for (int64_t wide = swiglu ? 1 : 2; wide >= 1; --wide) {  // blocks of 128 columns a tile: one is for calls that leave SMs idle
            if ((wide == 1 && !swiglu && t == 128) || (columns > 0 && !swiglu && t < 128 && columns != wide * 128)) continue;
            const bool half = wide == 1 && !swiglu;
            const int64_t n_tiles = up(n_blocks, wide), tiles = up(average, t), units = holders * tiles * n_tiles;
            for (int64_t s = 1; s <= (t == 128 ? 1 : 8); s *= 2) {
                if (ctas > 0 && s != ctas && t != 128) continue;
                const int64_t clusters = fp8::few_clusters(int(s), int(sms));
                const double busy = double(std::min(units, clusters) * s) / double(sms);
                double block = t == 128 ? 0.62 + 0.07 * busy : t == 64 ? 0.61 + 0.25 * busy : tiles > 1 ? 0.45 : 0.43 + 0.27 * busy;
                if (half) block *= kHalfTile;
                const double time = double(up(units, clusters)) * (double(up(k_blocks, s)) * block + (t == 128 ? 2.7 : 2.5 + 0.3 * double(s)));
                if (best >= 0 && time >= best) continue;
                best = time;
                c = Fp8Choice{t, s, (rows / t + holders) * n_tiles, n_tiles};
            }
        }
    }
    return c;
}

// (out) or (q, scales)
std::vector<at::Tensor> grouped_gemm_fp8(const at::Tensor& a, const at::Tensor& a_scales, const at::Tensor& w, const at::Tensor& w_scales,
                                         const OptTensor& expert_offsets, const OptTensor& expert_counts, const OptTensor& row_scale, bool swiglu, bool quantize,
                                         int64_t max_expert_rows, const at::Tensor& status, int64_t tile, int64_t ctas, int64_t columns) {
    check_e4m3(a, 2, "a");
    check_e4m3(w, 3, "w");
    const int64_t rows = a.size(0), K = a.size(1), E = w.size(0), halves = swiglu ? 2 : 1;
    TORCH_CHECK(w.device() == a.device() && w.size(2) == K, "w must be [experts, N, K] with the rows' K on the rows' device");
    TORCH_CHECK(E >= 1 && E <= fp8::kMaxExperts, "w must hold 1 to 1024 experts");
    TORCH_CHECK(w.size(1) % halves == 0, "w must be [experts, 2 * I, K] with swiglu");
    const int64_t n = w.size(1) / halves;
    TORCH_CHECK(K >= 16 && K % 16 == 0 && K < (int64_t(1) << 24), "K must be a multiple of 16 below 2^24");
    TORCH_CHECK(n >= 16 && n % 16 == 0 && n < (int64_t(1) << 24), "the output's columns must be a multiple of 16 below 2^24");
    TORCH_CHECK(rows < (int64_t(1) << 31) - 256 && E * w.size(1) < (int64_t(1) << 31), "at most 2^31 - 257 rows and 2^31 - 1 weight rows");
    const int64_t kb = blocks_of(K), nb = blocks_of(n);
    TORCH_CHECK(a_scales.is_cuda() && a_scales.device() == a.device() && a_scales.scalar_type() == at::kFloat && a_scales.is_contiguous() && a_scales.dim() == 2 &&
                    a_scales.size(0) == rows && a_scales.size(1) == kb,
                "a_scales must be contiguous float32 [rows, ceil(K / 128)] on the rows' device");
    TORCH_CHECK(w_scales.is_cuda() && w_scales.device() == a.device() && w_scales.scalar_type() == at::kFloat && w_scales.is_contiguous() && w_scales.dim() == 3 &&
                    w_scales.size(0) == E && w_scales.size(1) == halves * nb && w_scales.size(2) == kb,
                "w_scales must be contiguous float32 [experts, ceil(N / 128) (of each half with swiglu), ceil(K / 128)] on the rows' device");
    TORCH_CHECK(on16(a.data_ptr()) && on16(w.data_ptr()), "a and w must lie on 16-byte boundaries");
    TORCH_CHECK(expert_offsets.has_value() || E == 1, "expert_offsets is needed for more than one expert");
    check_i64(expert_offsets, a, E + 1, "expert_offsets");
    check_i64(expert_counts, a, E, "expert_counts");
    if (row_scale.has_value())
        TORCH_CHECK(!swiglu && row_scale->is_cuda() && row_scale->device() == a.device() && row_scale->scalar_type() == at::kFloat && row_scale->is_contiguous() &&
                        row_scale->dim() == 1 && row_scale->size(0) == rows,
                    "row_scale must be contiguous float32 [rows] on the rows' device (without swiglu)");
    TORCH_CHECK(max_expert_rows >= 0, "max_expert_rows must not be negative");
    TORCH_CHECK((tile == 0 || tile == 32 || tile == 64 || tile == 128) && (ctas == 0 || ctas == 1 || ctas == 2 || ctas == 4 || ctas == 8),
                "tile must be 0, 32, 64 or 128 and ctas 0, 1, 2, 4 or 8");
    TORCH_CHECK(columns == 0 || columns == 128 || columns == 256, "columns must be 0, 128 or 256");
    check_status_tensor(status, a);
    c10::cuda::CUDAGuard guard(a.device());
    std::vector<at::Tensor> out;
    if (quantize) {
        out.push_back(make_empty({rows, n}, at::kFloat8_e4m3fn, a));
        out.push_back(make_empty({rows, nb}, at::kFloat, a));
    } else {
        out.push_back(make_empty({rows, n}, at::kBFloat16, a));
    }
    if (rows == 0) return out;
    fp8::Args g{};
    g.a_scales = a_scales.data_ptr<float>();
    g.w_scales = w_scales.data_ptr<float>();
    g.expert_offsets = static_cast<const int64_t*>(pointer(expert_offsets));
    g.expert_counts = static_cast<const int64_t*>(pointer(expert_counts));
    g.row_scale = static_cast<const float*>(pointer(row_scale));
    if (quantize) {
        g.q = static_cast<uint8_t*>(out[0].data_ptr());
        g.scales = out[1].data_ptr<float>();
    } else {
        g.out = reinterpret_cast<__nv_bfloat16*>(out[0].data_ptr());
    }
    g.rows = rows;
    g.experts = int(E);
    g.n = int(n);
    g.k_blocks = int(kb);
    g.n_blocks = int(nb);
    g.swiglu = swiglu;
    g.status = reinterpret_cast<uint32_t*>(status.data_ptr<int>());
    g.timeout_ns = uint64_t(5e9);
    const int sms = sm_count();
    const Fp8Choice c = choose_fp8(rows, E, max_expert_rows, nb, swiglu, g.k_blocks, sms, tile, ctas, columns);
    g.n_tiles = int(c.n_tiles);
    TORCH_CHECK(c.units < (int64_t(1) << 31), "too many output tiles for one call");
    fp8::Maps maps{};
    maps.weights = e4m3_map(w.data_ptr(), K, n, E * halves, swiglu && c.tile == 128 ? 64 : 128);
    for (int b = 0; b < 4; ++b) maps.rows[b] = e4m3_map(a.data_ptr(), K, rows, 0, 128 >> b);
    const auto stream = c10::cuda::getCurrentCUDAStream();
    launched(c.tile == 128 ? fp8::launch(maps, g, int(std::min<int64_t>(sms, c.units)), stream) : fp8::launch_few(maps, g, int(c.tile), int(c.ctas), c.units, sms, stream),
             "grouped_gemm_fp8");
    return out;
}

// ------------------------------------------------------------------------------------------------ gradients
// The operators as nodes of autograd's graph, in C++: a node of Python's costs the host 10 us a pass each way.

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// What the backward functions compute has no graph of its own, and accumulation nodes remember the stream of the graph that made them: one that
// outlives into a capture ends the process.
void check_backward(const char* name, const char* explicit_name) {
    TORCH_CHECK(!at::GradMode::is_enabled(), name, " is differentiable once: call without create_graph");
    TORCH_CHECK(c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None, name, " is not differentiated inside a CUDA graph capture: call ",
                explicit_name, " there");
}

at::Tensor dense(const at::Tensor& t) { return t.defined() ? t.contiguous() : t; }
OptTensor optional(const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }

struct NormNode : torch::autograd::Function<NormNode> {
    // y, then the stream where there is a residual, then q and scales, then rstd
    static variable_list forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& weight, const OptTensor& residual, double eps, bool quantize) {
        at::AutoDispatchBelowADInplaceOrView below;
        const auto out = rms_norm(x, weight, residual, eps, quantize, true, true);
        ctx->saved_data["stream"] = residual.has_value();
        ctx->save_for_backward({residual.has_value() ? *out[3] : x, weight, *out[4]});
        ctx->set_materialize_grads(false);
        variable_list all{*out[0]}, fixed;
        if (residual.has_value()) all.push_back(*out[3]);
        if (quantize) fixed = {*out[1], *out[2]};
        fixed.push_back(*out[4]);
        all.insert(all.end(), fixed.begin(), fixed.end());
        ctx->mark_non_differentiable(fixed);
        return all;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_backward("rms_norm", "rms_norm_grad");
        const bool stream = ctx->saved_data["stream"].toBool();
        const at::Tensor grad_y = dense(grads[0]), grad_stream = stream ? dense(grads[1]) : at::Tensor();
        at::Tensor grad_x = grad_stream, grad_weight;
        if (grad_y.defined()) {
            const auto saved = ctx->get_saved_variables();
            std::tie(grad_x, grad_weight) = rms_norm_grad(grad_y, saved[0], saved[1], saved[2], optional(grad_stream));
        }
        return {grad_x, grad_weight, stream ? grad_x : at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

struct SortNode : torch::autograd::Function<SortNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const at::Tensor& slots, const at::Tensor& slot_map, bool zero_padding) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->save_for_backward({slots, slot_map});
        return sort_tokens(x, slots, slot_map, {}, zero_padding).first;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_backward("sort_tokens", "sort_tokens_grad");
        const auto saved = ctx->get_saved_variables();
        return {unsort_tokens(dense(grads[0]), saved[0], saved[1], {}, {}), at::Tensor(), at::Tensor(), at::Tensor()};
    }
};

struct UnsortNode : torch::autograd::Function<UnsortNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& y, const at::Tensor& slots, const at::Tensor& slot_map, const OptTensor& weights, const OptTensor& bias) {
        at::AutoDispatchBelowADInplaceOrView below;
        ctx->saved_data["weighted"] = weights.has_value();
        ctx->saved_data["biased"] = bias.has_value();
        ctx->save_for_backward({y, slots, slot_map, weights.has_value() ? *weights : at::Tensor()});
        return unsort_tokens(y, slots, slot_map, weights, bias);
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        check_backward("unsort_tokens", "unsort_tokens_grad");
        const auto saved = ctx->get_saved_variables();
        const at::Tensor grad_out = dense(grads[0]);
        at::Tensor grad_y, grad_weights;
        if (ctx->needs_input_grad(0) || (ctx->saved_data["weighted"].toBool() && ctx->needs_input_grad(3))) {
            const auto both = unsort_tokens_grad(grad_out, saved[0], saved[1], saved[2], optional(saved[3]));
            grad_y = both.first;
            if (both.second.has_value()) grad_weights = *both.second;
        }
        return {grad_y, at::Tensor(), at::Tensor(), grad_weights, ctx->saved_data["biased"].toBool() ? grad_out : at::Tensor()};
    }
};

}  // namespace

void bind_ops(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("rms_norm", &rms_norm, py::arg("x"), py::arg("weight"), py::arg("residual"), py::arg("eps"), py::arg("quantize"), py::arg("keep"), py::arg("save"));
    m.def("rms_norm_node", [](const at::Tensor& x, const at::Tensor& weight, const OptTensor& residual, double eps, bool quantize, bool save) -> std::vector<OptTensor> {
        const auto out = NormNode::apply(x, weight, residual, eps, quantize);
        size_t at = 1;
        std::vector<OptTensor> named(5);
        named[0] = out[0];
        if (residual.has_value()) named[3] = out[at++];
        if (quantize) named[1] = out[at], named[2] = out[at + 1];
        if (save) named[4] = out.back();
        return named;
    });
    m.def("sort_tokens_node", [](const at::Tensor& x, const at::Tensor& slots, const at::Tensor& slot_map, bool zero_padding) {
        return SortNode::apply(x, slots, slot_map, zero_padding);
    });
    m.def("unsort_tokens_node", [](const at::Tensor& y, const at::Tensor& slots, const at::Tensor& slot_map, const OptTensor& weights, const OptTensor& bias) {
        return UnsortNode::apply(y, slots, slot_map, weights, bias);
    });
    m.def("rms_norm_grad", &rms_norm_grad, py::arg("grad_y"), py::arg("h"), py::arg("weight"), py::arg("rstd"), py::arg("grad_stream"));
    m.def("quantize_rows", &quantize_rows, py::arg("x"));
    m.def("plan_tokens", &plan_tokens, py::arg("topk_idx"), py::arg("num_experts"), py::arg("alignment"), py::arg("status"));
    m.def("sort_tokens", &sort_tokens, py::arg("x"), py::arg("slots"), py::arg("slot_map"), py::arg("scales"), py::arg("zero_padding"));
    m.def("unsort_tokens", &unsort_tokens, py::arg("y"), py::arg("slots"), py::arg("slot_map"), py::arg("weights"), py::arg("bias"));
    m.def("unsort_tokens_grad", &unsort_tokens_grad, py::arg("grad_out"), py::arg("y"), py::arg("slots"), py::arg("slot_map"), py::arg("weights"));
    m.def("exchange_turn", [](int exchange) {
        const auto turn = fp8::exchange_turn(exchange);
        return std::make_pair(turn.at, turn.parity);
    });
    m.def("fp8_gemm_choice", [](int64_t rows, int64_t experts, int64_t most, int64_t n_blocks, bool swiglu, int64_t k_blocks, int64_t sms) {
        const Fp8Choice c = choose_fp8(rows, experts, most, n_blocks, swiglu, k_blocks, sms, 0, 0, 0);
        return std::make_tuple(c.tile, c.ctas, c.n_tiles);
    });
    m.def("grouped_gemm_fp8", &grouped_gemm_fp8, py::arg("a"), py::arg("a_scales"), py::arg("w"), py::arg("w_scales"), py::arg("expert_offsets"),
          py::arg("expert_counts"), py::arg("row_scale"), py::arg("swiglu"), py::arg("quantize"), py::arg("max_expert_rows"), py::arg("status"), py::arg("tile") = 0, py::arg("ctas") = 0, py::arg("columns") = 0);
}

}  // namespace nep

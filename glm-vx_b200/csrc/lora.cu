// Low-rank adapters of many requests beside a shared projection:
//   y[t] += s_a * B_a (A_a x[t]),   a = adapter_ids[t]  (-1: none, row t stays)
// with A_a [rank_a][cols] and B_a [rows][rank_a] taken from stacks padded to
// max_rank.  Two kernels: lora_shrink (h = A x, f32, into the workspace) and
// lora_expand (y += s B h).  Sums are f32; weights are F32, F16 or BF16 and
// widen to f32 exactly.
#include <cuda_bf16.h>

#include <algorithm>
#include <cstdint>

#include "common.cuh"

namespace glmvx {

namespace {

constexpr int kLoraMaxRank = 256;
constexpr int kLoraThreads = 256;

struct LoraArgs {
    float *y;
    const float *x;
    const int32_t *ids;
    const void *a, *b;
    const int32_t *ranks;
    const float *scales;
    float *h;
    int64_t y_stride, x_stride;
    int tokens, rows, cols, adapters, max_rank;
    int *err;
};

__device__ __forceinline__ float lora_f32(float v) { return v; }
__device__ __forceinline__ float lora_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float lora_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

// The adapter of token t, or -1; an id outside the bank is reported.
__device__ __forceinline__ int lora_adapter(const LoraArgs &p, int t) {
    const int a = p.ids[t];
    if (a < 0) return -1;
    if (a < p.adapters) return a;
    if (threadIdx.x == 0) report_device_error(p.err, kDevErrBadIndex);
    return -1;
}

__device__ __forceinline__ int lora_rank(const LoraArgs &p, int a) { return min(max(p.ranks[a], 0), p.max_rank); }

// One CTA per token, a warp per row of A.
template <class W>
__global__ void __launch_bounds__(kLoraThreads) lora_shrink_kernel(LoraArgs p) {
    const int t = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int id = lora_adapter(p, t);
    if (id < 0) return;
    const int rank = lora_rank(p, id);
    const float *x = p.x + t * p.x_stride;
    for (int r = warp; r < rank; r += kLoraThreads / 32) {
        const W *a = static_cast<const W *>(p.a) + (static_cast<int64_t>(id) * p.max_rank + r) * p.cols;
        float sum = 0.0f;
        for (int c = lane; c < p.cols; c += 32) sum = fmaf(lora_f32(a[c]), x[c], sum);
        sum = warp_sum(sum);
        if (lane == 0) p.h[static_cast<int64_t>(t) * p.max_rank + r] = sum;
    }
}

// One CTA per token and kLoraThreads rows, a thread per row of B.
template <class W>
__global__ void __launch_bounds__(kLoraThreads) lora_expand_kernel(LoraArgs p) {
    const int t = blockIdx.x, n = blockIdx.y * kLoraThreads + threadIdx.x;
    const int id = lora_adapter(p, t);
    if (id < 0 || n >= p.rows) return;
    const int rank = lora_rank(p, id);
    if (rank == 0) return;
    const W *b = static_cast<const W *>(p.b) + (static_cast<int64_t>(id) * p.rows + n) * p.max_rank;
    const float *h = p.h + static_cast<int64_t>(t) * p.max_rank;
    float sum = 0.0f;
    for (int r = 0; r < rank; ++r) sum = fmaf(lora_f32(b[r]), h[r], sum);
    float *y = p.y + t * p.y_stride + n;
    *y = fmaf(p.scales[id], sum, *y);
}

template <class W>
int32_t lora_launch(const LoraArgs &p, cudaStream_t stream) {
    lora_shrink_kernel<W><<<p.tokens, kLoraThreads, 0, stream>>>(p);
    if (const int32_t rc = launch_status("lora_shrink_kernel")) return rc;
    const dim3 grid(p.tokens, (p.rows + kLoraThreads - 1) / kLoraThreads);
    lora_expand_kernel<W><<<grid, kLoraThreads, 0, stream>>>(p);
    return launch_status("lora_expand_kernel");
}

int64_t lora_bytes(int64_t tokens, int64_t adapters, int64_t max_rank) {
    (void)adapters;
    return 4 * std::max<int64_t>(tokens, 1) * max_rank;
}

}  // namespace

}  // namespace glmvx

using namespace glmvx;

GLMVX_EXPORT int64_t glmvx_lora_workspace_bytes(int32_t tokens, int32_t adapters, int32_t max_rank) {
    if (tokens < 0 || tokens > 1 << 20 || adapters < 1 || max_rank < 1 || max_rank > kLoraMaxRank) return kInvalid;
    return lora_bytes(tokens, adapters, max_rank);
}

GLMVX_EXPORT int32_t glmvx_lora_add(float *y, int64_t y_stride, const float *x, int64_t x_stride,
                                    const int32_t *adapter_ids, int32_t kind, const void *a, const void *b,
                                    const int32_t *ranks, const float *scales, int32_t tokens, int32_t rows,
                                    int32_t cols, int32_t adapters, int32_t max_rank, void *workspace,
                                    uint64_t workspace_bytes, void *stream) {
    if (tokens < 0 || tokens > 1 << 20 || rows < 1 || cols < 1 || adapters < 1 || rows > 1 << 22)
        return set_error("lora_add: invalid dimensions"), kInvalid;
    if (max_rank < 1 || max_rank > kLoraMaxRank)
        return set_error("lora_add: max_rank must be 1..%d", kLoraMaxRank), kInvalid;
    if (kind != 0 && kind != 1 && kind != 30)
        return set_error("lora_add: adapters are kind 0 (F32), 1 (F16) or 30 (BF16), not %d", kind), kUnsupported;
    if (!tokens) return kOk;
    if (tokens > 1 && (y_stride < rows || x_stride < cols))
        return set_error("lora_add: row strides are shorter than the rows"), kInvalid;
    if (!y || !x || !adapter_ids || !a || !b || !ranks || !scales || !workspace)
        return set_error("lora_add: null pointer"), kInvalid;
    const auto bits = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
    if (((bits(y) | bits(x) | bits(adapter_ids) | bits(ranks) | bits(scales)) & 3) || (bits(workspace) & 15) ||
        ((bits(a) | bits(b)) & (kind == 0 ? 3 : 1)))
        return set_error("lora_add: misaligned pointer"), kInvalid;
    if (workspace_bytes < static_cast<uint64_t>(lora_bytes(tokens, adapters, max_rank)))
        return set_error("lora_add: workspace smaller than glmvx_lora_workspace_bytes"), kInvalid;
    const LoraArgs p{y, x, adapter_ids, a, b, ranks, scales, static_cast<float *>(workspace), y_stride, x_stride,
                     tokens, rows, cols, adapters, max_rank, device_error_word()};
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (kind == 0) return lora_launch<float>(p, s);
    if (kind == 1) return lora_launch<__half>(p, s);
    return lora_launch<__nv_bfloat16>(p, s);
}

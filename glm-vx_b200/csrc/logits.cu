// A row of logits from the model's to the chosen token, under one request's
// rules.  Per token v of row b, in f32, each operation rounded once:
//   seen in the history (or fed):  l = l > 0 ? l / repetition : l * repetition
//   c times among the output:      l = l - c * frequency; if c: l = l - presence
//   biased:                        l = l + bias   (of a token's entries the last holds)
//   outside the grammar mask:      l = -inf
// The choice is the lowest index of the largest l (a NaN counts as the
// largest, its first index is taken, as numpy's argmax does), -1 if nothing
// is above -inf.  One kernel reads the row once and writes it once.
//
// What happens to a token is gathered in one 32-bit word in shared memory:
// bits 0..19 its count among the output, bit 20 seen in the prompt, bits
// 21..31 the last bias entry that names it, plus one.  Integer atomics only, so the
// order in which threads meet a token changes nothing.
#include <cmath>
#include <cstdint>

#include "common.cuh"

namespace glmvx {

namespace {

constexpr int kSelThreads = 512;
constexpr int kSelChunk = 8192;  // tokens per pass: 32 KB of words
constexpr uint32_t kSelCount = (1u << 20) - 1, kSelPrompt = 1u << 20;
constexpr int kSelBiasShift = 21;
constexpr int kSelMaxBias = 2047, kSelMaxHistory = (1 << 20) - 2;  // the fields of a word, the fed token included

struct SelArgs {
    int32_t *selected;
    float *out;
    const float *logits;
    const int32_t *fed;
    int32_t *history, *history_lens;
    const int32_t *prompt_lens;
    const float *penalties;
    const int32_t *bias_ids;
    const float *bias_values;
    const int32_t *bias_lens;
    const uint32_t *masks;
    const int32_t *mask_rows;
    int64_t out_stride, logits_stride;
    int rows, vocab, history_capacity, bias_capacity, mask_count, mask_words;
    int *err;
};

// (v, j) replaces (best, bi): larger, or equal and earlier; a NaN is larger
// than any number, the first NaN stays.
__device__ __forceinline__ bool sel_takes(float v, int j, float best, int bi) {
    const bool vn = v != v, bn = best != best;
    return (vn && !bn) || (vn == bn && (vn ? j < bi : (v > best || (v == best && j < bi))));
}

__global__ void __launch_bounds__(kSelThreads) logits_select_kernel(SelArgs p) {
    __shared__ uint32_t words[kSelChunk];
    __shared__ float sv[kSelThreads / 32];
    __shared__ int si[kSelThreads / 32];
    const int b = blockIdx.x, tid = threadIdx.x;
    const float *in = p.logits + b * p.logits_stride;
    float *out = p.out + b * p.out_stride;
    int32_t *history = p.history ? p.history + static_cast<int64_t>(b) * p.history_capacity : nullptr;
    const int len = history ? min(max(p.history_lens[b], 0), p.history_capacity) : 0;
    const int prompt = p.prompt_lens ? p.prompt_lens[b] : 0;
    int fed = p.fed ? p.fed[b] : -1;
    if (fed >= p.vocab) {
        if (tid == 0) report_device_error(p.err, kDevErrBadIndex);
        fed = -1;
    }
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if (p.penalties) rep = p.penalties[3 * b], pres = p.penalties[3 * b + 1], freq = p.penalties[3 * b + 2];
    const int biases = p.bias_lens ? min(max(p.bias_lens[b], 0), p.bias_capacity) : 0;
    const int32_t *bias_ids = p.bias_ids + static_cast<int64_t>(b) * p.bias_capacity;
    const float *bias_values = p.bias_values + static_cast<int64_t>(b) * p.bias_capacity;
    int mrow = p.mask_rows ? p.mask_rows[b] : -1;
    const bool closed = mrow >= p.mask_count;  // no such mask: nothing is allowed
    if (closed && tid == 0) report_device_error(p.err, kDevErrBadIndex);
    const uint32_t *mask = mrow >= 0 && !closed ? p.masks + static_cast<int64_t>(mrow) * p.mask_words : nullptr;

    float best = -INFINITY;
    int bi = p.vocab;
    for (int v0 = 0; v0 < p.vocab; v0 += kSelChunk) {
        const int n = min(kSelChunk, p.vocab - v0);
        for (int i = tid; i < n; i += kSelThreads) words[i] = 0;
        __syncthreads();
        for (int i = tid; i < biases; i += kSelThreads) {
            const int v = bias_ids[i] - v0;
            if (v >= 0 && v < n) atomicMax(words + v, static_cast<uint32_t>(i + 1) << kSelBiasShift);
        }
        __syncthreads();
        if (p.penalties) {
            for (int i = tid; i < len; i += kSelThreads) {
                const int v = history[i] - v0;
                if (v < 0 || v >= n) continue;
                if (i < prompt) atomicOr(words + v, kSelPrompt);
                else atomicAdd(words + v, 1u);
            }
            if (tid == 0 && fed >= v0 && fed - v0 < n) {
                if (len < prompt) atomicOr(words + (fed - v0), kSelPrompt);
                else atomicAdd(words + (fed - v0), 1u);
            }
        }
        __syncthreads();
        for (int i = tid; i < n; i += kSelThreads) {
            const int v = v0 + i;
            const bool allowed = !closed && (!mask || (mask[v >> 5] >> (v & 31) & 1));
            float l = -INFINITY;
            if (allowed) {
                l = in[v];
                const uint32_t w = words[i];
                const uint32_t count = w & kSelCount;
                if (w & (kSelCount | kSelPrompt)) l = l > 0.0f ? __fdiv_rn(l, rep) : __fmul_rn(l, rep);
                if (count) l = __fsub_rn(__fsub_rn(l, __fmul_rn(static_cast<float>(count), freq)), pres);
                if (w >> kSelBiasShift) l = __fadd_rn(l, bias_values[(w >> kSelBiasShift) - 1]);
                if (sel_takes(l, v, best, bi)) best = l, bi = v;
            }
            out[v] = l;
        }
        __syncthreads();
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const float v = __shfl_xor_sync(0xffffffffu, best, o);
        const int j = __shfl_xor_sync(0xffffffffu, bi, o);
        if (sel_takes(v, j, best, bi)) best = v, bi = j;
    }
    if ((tid & 31) == 0) sv[tid >> 5] = best, si[tid >> 5] = bi;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kSelThreads / 32; ++w)
            if (sel_takes(sv[w], si[w], best, bi)) best = sv[w], bi = si[w];
        p.selected[b] = best == -INFINITY ? -1 : bi;
        if (history && fed >= 0 && len < p.history_capacity) {
            history[len] = fed;
            p.history_lens[b] = len + 1;
        }
    }
}

}  // namespace

}  // namespace glmvx

using namespace glmvx;

GLMVX_EXPORT int32_t glmvx_logits_select(int32_t *selected, float *out, int64_t out_stride, const float *logits,
                                         int64_t logits_stride, int32_t rows, int32_t vocab, const int32_t *fed,
                                         int32_t *history, int32_t history_capacity, int32_t *history_lens,
                                         const int32_t *prompt_lens, const float *penalties, const int32_t *bias_ids,
                                         const float *bias_values, const int32_t *bias_lens, int32_t bias_capacity,
                                         const uint32_t *masks, const int32_t *mask_rows, int32_t mask_count,
                                         void *stream) {
    if (rows < 0 || vocab < 1) return set_error("logits_select: invalid dimensions"), kInvalid;
    if (!rows) return kOk;
    if (!selected || !out || !logits) return set_error("logits_select: null pointer"), kInvalid;
    if (rows > 1 && (out_stride < vocab || logits_stride < vocab))
        return set_error("logits_select: row strides are shorter than the vocabulary"), kInvalid;
    if (out == logits && rows > 1 && out_stride != logits_stride)
        return set_error("logits_select: in place needs equal strides"), kInvalid;
    if (!history != !history_lens || (!history && (fed || prompt_lens)))
        return set_error("logits_select: a history needs its lengths, fed tokens and prompt lengths a history"), kInvalid;
    if (history && (history_capacity < 1 || history_capacity > kSelMaxHistory))
        return set_error("logits_select: history capacity must be 1..%d", kSelMaxHistory), kInvalid;
    if (!bias_ids != !bias_values || !bias_ids != !bias_lens)
        return set_error("logits_select: biases need ids, values and lengths"), kInvalid;
    if (bias_ids && (bias_capacity < 1 || bias_capacity > kSelMaxBias))
        return set_error("logits_select: bias capacity must be 1..%d", kSelMaxBias), kInvalid;
    if (!masks != !mask_rows) return set_error("logits_select: masks need the row of each sequence"), kInvalid;
    if (masks && mask_count < 1) return set_error("logits_select: no masks"), kInvalid;
    const auto bits = [](const void *q) { return reinterpret_cast<uintptr_t>(q); };
    if ((bits(selected) | bits(out) | bits(logits) | bits(fed) | bits(history) | bits(history_lens) |
         bits(prompt_lens) | bits(penalties) | bits(bias_ids) | bits(bias_values) | bits(bias_lens) | bits(masks) |
         bits(mask_rows)) & 3)
        return set_error("logits_select: misaligned pointer"), kInvalid;
    const SelArgs p{selected, out, logits, fed, history, history_lens, prompt_lens, penalties, bias_ids, bias_values,
                    bias_lens, masks, mask_rows, out_stride, logits_stride, rows, vocab, history_capacity,
                    bias_capacity, mask_count, static_cast<int>((static_cast<int64_t>(vocab) + 31) / 32),
                    device_error_word()};
    logits_select_kernel<<<rows, kSelThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launch_status("logits_select_kernel");
}

// A row of logits from the model's to the chosen token, under one request's
// rules.  Per token v of row b, in f32, each operation rounded once:
//   seen in the history (or fed):  l = l > 0 ? l / repetition : l * repetition
//   c times among the output:      l = l - c * frequency; if c: l = l - presence
//   biased:                        l = l + bias   (of a token's entries the last holds; -inf bans, whatever l is)
//   outside the grammar mask:      l = -inf
// The choice is the lowest index of the largest l (a NaN counts as the
// largest, its first index is taken, as numpy's argmax does), -1 if nothing
// is above -inf.  One kernel reads the row once and writes it once.
//
// A row is a few thousand tokens with rules and 10^5 without.  The ruled ones
// are settled first, on the side: a bitmap of the CTA's tokens, a slot for each
// set bit (its rank), the marks of all entries gathered there, the marks turned
// into the ruled logits.  Then the row streams past: a group of four tokens
// costs its load, a look at four bits, a maximum and its store.
//
// A slot's mark is one 32-bit word: bits 0..19 the token's count among the
// output, bit 20 seen in the prompt, bits 21..31 the last bias entry that names
// it, plus one.  Integer atomics only, so the order in which threads meet a
// token changes nothing.
//
// Measured in CUDA graphs, 154880 tokens a row, beside the time of a copy of the
// bytes (6.57 TB/s): 256 rows with short rules 60.9 us (48.4: 5.2 TB/s; DRAM at
// 55 % of its peak under the profiler, the schedulers issue in 58 % of the
// cycles), 64 rows with histories of 2048, biases and masks 21.9 us (12.1), 32 rows
// of tight masks 13.4 us (6.1), 1 row 8.9 us (0.2).  Many rows are bound by the
// stream, by what its warps have in flight (256 rows without rules 55.5 us, with
// half the instructions), few by the rules' phases, each a wait.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "common.cuh"

namespace glmvx {

namespace {

constexpr int kSelThreads = 512, kSelWarps = kSelThreads / 32;
constexpr int kSelMaxCluster = 8;
constexpr int kSelBlock = 128;         // tokens a warp handles at once, four a lane
constexpr int kSelDepth = 3;           // blocks a warp has in flight
constexpr int kSelBatch = 4;           // entries a thread has in flight
constexpr int kSelSmem = 200 << 10;    // shared memory a CTA may take
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
    int shift, blocks, passes, slots;  // 2^shift CTAs per row; blocks per CTA and pass; room for ruled tokens
    int eager;                         // load the logits before the mask says which are needed
    int *err;
};

// The larger, or NaN when either is.
__device__ __forceinline__ float sel_max(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

// Whether x is an element that a row's maximum m came from.
__device__ __forceinline__ bool sel_is(float x, float m) { return x == m || (m != m && x != x); }

// Stores v to this CTA's shared variable `at` in the CTA `rank` of the cluster.
__device__ __forceinline__ void cluster_store(void *at, uint32_t rank, uint32_t v) {
    asm volatile(
        "{\n\t.reg .b32 r;\n\t"
        "mapa.shared::cluster.u32 r, %0, %1;\n\t"
        "st.shared::cluster.u32 [r], %2;\n\t}" ::"r"(smem_addr(at)),
        "r"(rank), "r"(v)
        : "memory");
}

// One cluster per row.  The vocabulary goes round the cluster's CTAs, and there
// round their warps, in blocks of 128 tokens (frequent tokens have low ids:
// slices would leave the first CTA most of the history).  A lane's tokens of a
// block are four neighbours with VEC (rows on 16-byte boundaries), else 32 apart.
template <bool VEC>
__global__ void __launch_bounds__(kSelThreads, 2) logits_select_kernel(SelArgs p) {
    extern __shared__ __align__(16) uint32_t sel_smem[];
    __shared__ float warp_max[kSelWarps];
    __shared__ int warp_sum[kSelWarps];
    __shared__ int first;                                        // lowest token of this CTA that is its maximum
    __shared__ uint32_t cv[kSelMaxCluster], ci[kSelMaxCluster];  // CTA 0: every CTA's maximum and its token
    cluster_arrive();  // waited for below, before the first store to another CTA
    const int b = blockIdx.x >> p.shift, part = blockIdx.x & ((1 << p.shift) - 1);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int nwords = 4 * p.blocks;
    uint32_t *bits = sel_smem, *rank = bits + nwords;  // of the CTA's tokens: ruled; ruled ones before this word
    uint32_t *slot = rank + nwords;                    // mark, then ruled logit
    int *slot_token = reinterpret_cast<int *>(slot + p.slots);
    const float *in = p.logits + b * p.logits_stride;
    float *out = p.out + b * p.out_stride;
    int32_t *history = p.history + static_cast<int64_t>(b) * p.history_capacity;
    const int32_t *bias_ids = p.bias_ids + static_cast<int64_t>(b) * p.bias_capacity;
    // Everything that is known by address is asked for before anything is waited for.
    int len = p.history ? p.history_lens[b] : 0, biases = p.bias_ids ? p.bias_lens[b] : 0;
    const int prompt = p.prompt_lens ? p.prompt_lens[b] : 0;
    int fed = p.fed ? p.fed[b] : -1;
    const int mrow = p.mask_rows ? p.mask_rows[b] : -1;
    float rep = 1.0f, pres = 0.0f, freq = 0.0f;
    if (p.penalties) rep = p.penalties[3 * b], pres = p.penalties[3 * b + 1], freq = p.penalties[3 * b + 2];

    constexpr int kGap = VEC ? 1 : 32;  // from one of a lane's tokens to the next
    const int lane_at = VEC ? 4 * lane : lane;
    const int stride = kSelWarps * kSelBlock << p.shift;  // from a warp's block to its next
    int v_first, v_end;  // the lane's first token of the pass, the end of the pass's blocks for this warp
    const auto range = [&](int pass) {
        v_first = (((pass * p.blocks + warp) << p.shift) + part) * kSelBlock + lane_at;
        v_end = min(p.vocab, static_cast<int>(((static_cast<int64_t>(pass) + 1) * p.blocks << p.shift) * kSelBlock));
    };
    const auto load = [&](float(&x)[4], int v, uint32_t keep) {
        if (VEC) {
            float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
            if (v < v_end && keep) f = __ldcs(reinterpret_cast<const float4 *>(in + v));
            x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = v + 32 * e < v_end && (keep >> e & 1u) ? in[v + 32 * e] : 0.0f;
        }
    };
    float cur[kSelDepth][4], nxt[kSelDepth][4];
    range(0);
    if (p.eager) {
#pragma unroll
        for (int d = 0; d < kSelDepth; ++d) load(cur[d], v_first + d * stride, 15u);
    }

    len = min(max(len, 0), p.history_capacity);
    biases = min(max(biases, 0), p.bias_capacity);
    const bool closed = mrow >= p.mask_count;  // no such mask: nothing is allowed
    if (part == 0 && tid == 0 && (fed >= p.vocab || closed)) report_device_error(p.err, kDevErrBadIndex);
    if (fed >= p.vocab) fed = -1;
    const uint32_t *mask = mrow >= 0 && !closed ? p.masks + static_cast<int64_t>(mrow) * p.mask_words : nullptr;
    // The mask words of the block at v, one a lane, and from them the lane's four bits.
    const auto mask_word = [&](int v) {
        const int w = ((v - lane_at) >> 5) + (VEC ? lane >> 3 : lane & 3);
        return mask ? __ldg(mask + min(w, p.mask_words - 1)) : closed ? 0u : ~0u;
    };
    const auto allowed = [&](uint32_t word) {
        if (VEC) return word >> 4 * (lane & 7) & 15u;
        uint32_t k = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) k |= (__shfl_sync(0xffffffffu, word, e) >> lane & 1u) << e;
        return k;
    };
    // Entries: the biases, then (with penalties that do something) the history and the fed token.
    const bool neutral = rep == 1.0f && pres == 0.0f && freq == 0.0f;  // changes no logit, whatever was said
    const int entries = biases + (!neutral && (len > 0 || fed >= 0) ? len + 1 : 0);
    const auto entry_id = [&](int j) {
        return j >= entries ? -1 : j < biases ? bias_ids[j] : j - biases < len ? history[j - biases] : fed;
    };
    float top = -INFINITY;  // of this thread's tokens so far, and the block that it came from
    int top_at = 0;
    for (int pass = 0; pass < p.passes; ++pass) {
        if (pass) range(pass);
        uint32_t words[2 * kSelDepth];  // mask words of the blocks in flight and of the next ones
#pragma unroll
        for (int d = 0; d < 2 * kSelDepth; ++d) words[d] = mask_word(v_first + d * stride);
        if (pass || !p.eager) {
#pragma unroll
            for (int d = 0; d < kSelDepth; ++d) load(cur[d], v_first + d * stride, allowed(words[d]));
        }
        if (entries) {
            const int base = (pass * p.blocks << p.shift) * kSelBlock;
            // Where token id stands among the CTA's tokens of this pass, or -1.  An id before them, and a negative one,
            // wraps around and lies behind them.
            const auto place = [&](int id) {
                const uint32_t u = id, d = u - base, blk = d >> 7;
                const uint32_t turn = blk >> p.shift;
                return u < static_cast<uint32_t>(p.vocab) && ((blk ^ part) & ((1u << p.shift) - 1)) == 0 &&
                               turn < static_cast<uint32_t>(p.blocks)
                           ? static_cast<int>(turn * kSelBlock + (d & 127))
                           : -1;
            };
            for (int i = tid; i < nwords; i += kSelThreads) bits[i] = 0;
            int id[kSelBatch];
            const auto fetch = [&](int j0) {
#pragma unroll
                for (int u = 0; u < kSelBatch; ++u) id[u] = entry_id(j0 + u * kSelThreads);
            };
            fetch(tid);
            __syncthreads();
            for (int j0 = tid; j0 < entries; j0 += kSelBatch * kSelThreads) {
                if (j0 != tid) fetch(j0);
#pragma unroll
                for (int u = 0; u < kSelBatch; ++u) {
                    const int at = place(id[u]);
                    if (at >= 0) atomicOr(bits + (at >> 5), 1u << (at & 31));
                }
            }
            __syncthreads();
            // Ranks: a prefix sum over the words, a run of them per thread.
            const int run = (nwords + kSelThreads - 1) / kSelThreads;
            const int w0 = min(tid * run, nwords), w1 = min(w0 + run, nwords);
            int sum = 0;
            for (int w = w0; w < w1; ++w) sum += __popc(bits[w]);
            int before = sum;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(0xffffffffu, before, o);
                if (lane >= o) before += up;
            }
            if (lane == 31) warp_sum[warp] = before;
            before -= sum;
            __syncthreads();
            int count = 0;
#pragma unroll
            for (int w = 0; w < kSelWarps; ++w) {
                if (w == warp) before += count;
                count += warp_sum[w];
            }
            for (int w = w0; w < w1; ++w) {
                rank[w] = before;
                before += __popc(bits[w]);
            }
            for (int i = tid; i < count; i += kSelThreads) slot[i] = 0;
            __syncthreads();
            if (entries > kSelBatch * kSelThreads) fetch(tid);  // else the ids are still there
            for (int j0 = tid; j0 < entries; j0 += kSelBatch * kSelThreads) {
                if (j0 != tid) fetch(j0);
#pragma unroll
                for (int u = 0; u < kSelBatch; ++u) {
                    const int j = j0 + u * kSelThreads, at = place(id[u]);
                    if (at < 0) continue;
                    const int r = rank[at >> 5] + __popc(bits[at >> 5] & ((1u << (at & 31)) - 1));
                    slot_token[r] = id[u];
                    if (j >= biases) {
                        if (j - biases >= prompt) atomicAdd(slot + r, 1u);
                        else atomicOr(slot + r, kSelPrompt);
                        continue;
                    }
                    const uint32_t entry = static_cast<uint32_t>(j + 1);  // the last entry stays, whatever the order
                    uint32_t w = slot[r], seen;
                    do {
                        seen = w;
                        if (seen >> kSelBiasShift >= entry) break;
                        w = atomicCAS(slot + r, seen, (seen & ((1u << kSelBiasShift) - 1)) | entry << kSelBiasShift);
                    } while (w != seen);
                }
            }
            __syncthreads();
            for (int r = tid; r < count; r += kSelThreads) {
                const uint32_t w = slot[r], n = w & kSelCount, entry = w >> kSelBiasShift;
                float x = in[slot_token[r]];
                if (w & (kSelCount | kSelPrompt)) x = x > 0.0f ? __fdiv_rn(x, rep) : __fmul_rn(x, rep);
                if (n) x = __fsub_rn(__fsub_rn(x, __fmul_rn(static_cast<float>(n), freq)), pres);
                if (entry) {
                    const float bias = p.bias_values[static_cast<int64_t>(b) * p.bias_capacity + entry - 1];
                    x = bias == -INFINITY ? bias : __fadd_rn(x, bias);  // a ban, of an infinite logit too
                }
                slot[r] = __float_as_uint(x);
            }
            __syncthreads();
        }
        // The warp's i-th block, of the lane's tokens from v on.
        const auto finish = [&](float(&x)[4], int v, int i, uint32_t k) {
            if (entries) {
                const int w = 4 * (i * kSelWarps + warp);
                if (VEC) {
                    const uint32_t word = bits[min(w + (lane >> 3), nwords - 1)], t = word >> (v & 31) & 15u;
                    if (t && v < v_end) {
                        const uint32_t *s = slot + rank[w + (lane >> 3)] + __popc(word & ((1u << (v & 31)) - 1));
                        if (t & 1) x[0] = __uint_as_float(*s++);
                        if (t & 2) x[1] = __uint_as_float(*s++);
                        if (t & 4) x[2] = __uint_as_float(*s++);
                        if (t & 8) x[3] = __uint_as_float(*s);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t word = bits[min(w + e, nwords - 1)];
                        if ((word >> lane & 1u) && v + 32 * e < v_end)
                            x[e] = __uint_as_float(slot[rank[w + e] + __popc(word & ((1u << lane) - 1))]);
                    }
                }
            }
            if (v >= v_end) return;
            if (mask || closed) {
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = k >> e & 1u ? x[e] : -INFINITY;
            }
            if (VEC) {
                __stcs(reinterpret_cast<float4 *>(out + v), make_float4(x[0], x[1], x[2], x[3]));
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (v + 32 * e < v_end) out[v + 32 * e] = x[e];
                    else x[e] = -INFINITY;
                }
            }
            const float m = sel_max(sel_max(x[0], x[1]), sel_max(x[2], x[3]));
            if (top == top && !(m <= top)) top = m, top_at = v;  // larger, or the first NaN
        };
        for (int i = 0, v = v_first; v - lane_at < v_end; i += kSelDepth, v += kSelDepth * stride) {
#pragma unroll
            for (int d = 0; d < kSelDepth; ++d)
                load(nxt[d], v + (kSelDepth + d) * stride, p.eager ? 15u : allowed(words[kSelDepth + d]));
#pragma unroll
            for (int d = 0; d < kSelDepth; ++d) {
                finish(cur[d], v + d * stride, i + d, allowed(words[d]));
                words[d] = words[kSelDepth + d];
                words[kSelDepth + d] = mask_word(v + (2 * kSelDepth + d) * stride);
#pragma unroll
                for (int e = 0; e < 4; ++e) cur[d][e] = nxt[d][e];
            }
        }
        if (pass + 1 < p.passes) __syncthreads();  // the bitmap and the slots are free again
    }
    // The CTA's maximum, then its lowest token: only the threads that hold it look for it.
    float m = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = sel_max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) warp_max[warp] = m;
    if (tid == 0) first = p.vocab;
    __syncthreads();
    m = warp_max[lane & (kSelWarps - 1)];
#pragma unroll
    for (int o = kSelWarps / 2; o > 0; o >>= 1) m = sel_max(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m != -INFINITY && sel_is(top, m)) {
        int at = p.vocab;
#pragma unroll
        for (int e = 3; e >= 0; --e)
            if (top_at + kGap * e < p.vocab && sel_is(out[top_at + kGap * e], m)) at = top_at + kGap * e;
        atomicMin(&first, at);
    }
    __syncthreads();
    cluster_wait();  // every CTA of the cluster has started
    if (tid == 0) {
        cluster_store(cv + part, 0, __float_as_uint(m));
        cluster_store(ci + part, 0, static_cast<uint32_t>(first));
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (part == 0 && tid == 0) {
        int bi = first;
        for (int c = 1; c < 1 << p.shift; ++c) {
            const float v = __uint_as_float(cv[c]);
            const int j = static_cast<int>(ci[c]);
            if (v > m || (v != v && m == m) || (sel_is(v, m) && j < bi)) m = v, bi = j;
        }
        p.selected[b] = m == -INFINITY ? -1 : bi;
        // every CTA has read the history and its length by now
        if (p.history && fed >= 0 && len < p.history_capacity) {
            history[len] = fed;
            p.history_lens[b] = len + 1;
        }
    }
}

template <bool VEC>
int32_t sel_launch(const SelArgs &p, size_t smem, cudaStream_t stream) {
    if (const int32_t rc = allow_dynamic_smem(logits_select_kernel<VEC>, kSelSmem, "logits_select smem")) return rc;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 1 << p.shift;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(p.rows << p.shift);
    cfg.blockDim = dim3(kSelThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    GLMVX_CUDA(cudaLaunchKernelEx(&cfg, logits_select_kernel<VEC>, p));
    return launch_status("logits_select_kernel");
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
    if (rows < 0 || vocab < 1 || vocab > 1 << 30 || rows > 1 << 24)
        return set_error("logits_select: invalid dimensions"), kInvalid;
    if (!rows) return kOk;
    if (!selected || !out || !logits) return set_error("logits_select: null pointer"), kInvalid;
    if (rows > 1 && (out_stride < vocab || logits_stride < vocab))
        return set_error("logits_select: row strides are shorter than the vocabulary"), kInvalid;
    if (out == logits && rows > 1 && out_stride != logits_stride)
        return set_error("logits_select: in place needs equal strides"), kInvalid;
    if (!history != !history_lens || (!history && (fed || prompt_lens)))
        return set_error("logits_select: a history needs its lengths, fed tokens and prompt lengths a history"),
               kInvalid;
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
    const auto parts = [](int n, int of) { return (n + of - 1) / of; };
    const int all_blocks = parts(vocab, kSelBlock);
    // As many CTAs to a row as run at once, two an SM (clusters leave a few of those places empty), while each
    // warp has a block: a CTA settles its rules once, however many blocks stream past after that.  Always 8: 64 rows
    // 29.3 us against 21.9, 256 rows 104.5 against 60.9; at most 2: 1 row 15.4 against 8.9, 32 rows 20.3 against 13.4.
    int shift = 0;
    while (1 << shift < kSelMaxCluster && all_blocks > kSelWarps << shift &&
           static_cast<int64_t>(rows) << (shift + 1) <= 2 * sm_count() * 7 / 8)
        ++shift;
    // Shared memory: a bit and its rank for every token of a CTA, a slot for every token that may
    // be ruled.  What does not fit at once goes in passes.
    const int most = (penalties && history ? history_capacity + 1 : 0) + (bias_ids ? bias_capacity : 0);
    const int cta_blocks = parts(all_blocks, 1 << shift);
    int passes = 0, blocks = 0, slots = 0;
    size_t smem = 0;
    do {
        blocks = parts(cta_blocks, ++passes);
        slots = static_cast<int>(std::min<int64_t>(most, static_cast<int64_t>(blocks) * kSelBlock));
        smem = most ? 8ull * (4ull * blocks + slots) : 0;
    } while (smem > kSelSmem);
    // Masked rows load what their mask keeps, but where an SM has one CTA at most the wait for the mask would show:
    // eager everywhere 64 rows 23.4 us against 21.9 and 32 rows of tight masks 14.6 against 13.4, nowhere 17 rows of
    // 32003 tokens 10.2 against 9.75.
    const bool eager = !masks || rows << shift <= sm_count();
    const SelArgs p{selected, out, logits, fed, history, history_lens, prompt_lens, penalties, bias_ids, bias_values,
                    bias_lens, masks, mask_rows, out_stride, logits_stride, rows, vocab,
                    history ? history_capacity : 0, bias_ids ? bias_capacity : 0, mask_count, parts(vocab, 32), shift,
                    blocks, passes, slots, eager, device_error_word()};
    // Rows on 16-byte boundaries go four tokens a load, others one: 256 rows 60.9 us against 104.8.
    const bool vec = !((bits(out) | bits(logits)) & 15) && !(vocab & 3) &&
                     (rows == 1 || !((out_stride | logits_stride) & 3));
    return vec ? sel_launch<true>(p, smem, static_cast<cudaStream_t>(stream))
               : sel_launch<false>(p, smem, static_cast<cudaStream_t>(stream));
}

// Experts chosen by scores: scores, bias, groups, the best few of a token, their weights, and the rows of the matrix sorted by expert.
//
//  * score_select_kernel: a warp per token.  Choices lie next to borders, where 32 bits would tell equal from unequal by the order of their sums: scores are
//    64-bit.  A CTA's 32 tokens leave one word per expert, a bit for every token that chose it (a token chooses an expert once).
//  * score_layout_kernel: from those words the experts' segments, and every pair's row: what the words ahead count, and the bits below its own.
//    No order of arrival enters, so the rows are the same every time.
#include "spk_experts.cuh"

namespace {

constexpr int kTokens = 32;  // per CTA of the selection: the bits of a word
constexpr int kSelectWarps = 8;
constexpr int kLayoutThreads = 1024;
constexpr int kLayoutWords = 8;  // words per CTA of the layout

__device__ __forceinline__ double warp_max(double v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v = fmax(v, __shfl_xor_sync(~0u, v, o));
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
    return v;
}

// NaN counts as -infinity, +infinity as the largest finite value.
template <typename T>
__device__ __forceinline__ double logit(const T* l, int e) {
    const float f = spk_to_float<T>(l[e]);
    return f != f ? -INFINITY : static_cast<double>(fminf(f, 3.402823466e38f));
}

template <typename T>
__global__ void __launch_bounds__(kSelectWarps * 32)
score_select_kernel(const spk_route_scores_args a, uint32_t* words) {
    extern __shared__ double sm[];
    const int E = a.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    double* c = sm + static_cast<int64_t>(warp) * 2 * E;  // what the choice goes by
    double* gs = c + E;                                   // the groups' scores
    uint32_t* word = reinterpret_cast<uint32_t*>(sm + static_cast<int64_t>(kSelectWarps) * 2 * E);
    for (int e = threadIdx.x; e < E; e += blockDim.x) word[e] = 0;
    __syncthreads();
    for (int i = warp; i < kTokens; i += kSelectWarps) {
        const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + i;
        if (t >= a.n) break;
        const bool on = a.active == nullptr || a.active[t] == 1;
        const T* l = static_cast<const T*>(a.logits) + t * a.logits_stride;
        double m = 0.0, inv = 1.0;
        if (on) {
            if (a.score == SPK_SCORE_SOFTMAX) {
                double top = -INFINITY, sum = 0.0;
                for (int e = lane; e < E; e += 32) top = fmax(top, logit(l, e));
                top = warp_max(top);
                m = top == -INFINITY ? 0.0 : top;
                for (int e = lane; e < E; e += 32) sum += exp(logit(l, e) - m);
                inv = warp_sum(sum);
            }
            for (int e = lane; e < E; e += 32) {
                const double x = logit(l, e);
                double v = a.score == SPK_SCORE_SOFTMAX ? exp(x - m) / inv : 1.0 / (1.0 + exp(-x));
                if (a.bias != nullptr) v += static_cast<double>(a.bias[e]);
                c[e] = x == -INFINITY || v != v ? -INFINITY : v;
            }
            __syncwarp();
            if (a.groups > 1) {
                const int per = E / a.groups;
                for (int g = lane; g < a.groups; g += 32) {
                    double first = -INFINITY, second = -INFINITY;
                    for (int k = 0; k < per; ++k) {
                        const double v = c[g * per + k];
                        second = fmax(second, fmin(first, v));
                        first = fmax(first, v);
                    }
                    gs[g] = second == -INFINITY ? first : first + second;
                }
                __syncwarp();
                for (int g = lane; g < a.groups; g += 32) {
                    int better = 0;
                    for (int h = 0; h < a.groups; ++h) better += gs[h] > gs[g] || (gs[h] == gs[g] && h < g);
                    if (better >= a.top_groups)
                        for (int k = 0; k < per; ++k) c[g * per + k] = -INFINITY;
                }
                __syncwarp();
            }
        }
        int mine = -1;  // choice number `lane` of the token
        for (int j = 0; j < a.top && on; ++j) {
            double best = -INFINITY;
            int at = E;
            for (int e = lane; e < E; e += 32)
                if (c[e] > best) best = c[e], at = e;
#pragma unroll
            for (int o = 16; o >= 1; o >>= 1) {
                const double v = __shfl_xor_sync(~0u, best, o);
                const int w = __shfl_xor_sync(~0u, at, o);
                if (v > best || (v == best && w < at)) best = v, at = w;
            }
            if (at >= E) break;
            if (lane == j) mine = at;
            if (lane == 0) {
                c[at] = -INFINITY;
                atomicOr(word + at, 1u << i);
            }
            __syncwarp();
        }
        double s = 0.0;
        if (mine >= 0) {
            const double x = logit(l, mine);
            s = a.score == SPK_SCORE_SOFTMAX ? exp(x - m) / inv : 1.0 / (1.0 + exp(-x));
        }
        if (a.renormalize) {
            const double sum = warp_sum(s);
            s = sum > 0.0 ? s / sum : 0.0;
        }
        if (lane < a.top) {
            a.ids[t * a.top + lane] = mine;
            a.weights[t * a.top + lane] = static_cast<float>(s * static_cast<double>(a.scale));
        }
        __syncwarp();
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += blockDim.x) words[static_cast<int64_t>(blockIdx.x) * E + e] = word[e];
}

__global__ void __launch_bounds__(kLayoutThreads)
score_layout_kernel(const spk_route_scores_args a, const uint32_t* __restrict__ words, const int n_words) {
    extern __shared__ int32_t at[];  // [experts] all rows of the expert, then the first row of this CTA's tokens
    const int E = a.experts;
    int32_t* before = at + E;
    const int w0 = blockIdx.x * kLayoutWords;
    for (int e = threadIdx.x; e < 2 * E; e += kLayoutThreads) at[e] = 0;
    __syncthreads();
    for (int64_t i = threadIdx.x; i < static_cast<int64_t>(n_words) * E; i += kLayoutThreads) {
        const int e = static_cast<int>(i % E), c = __popc(words[i]);
        if (c == 0) continue;
        atomicAdd(at + e, c);
        if (i / E < w0) atomicAdd(before + e, c);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int rows = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + threadIdx.x;
            const int c = e < E ? at[e] : 0;
            const int padded = (c + kExpertAlign - 1) & ~(kExpertAlign - 1);
            int upto = padded;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(~0u, upto, o);
                if (static_cast<int>(threadIdx.x) >= o) upto += up;
            }
            if (e < E) {
                const int first = rows + upto - padded;
                at[e] = first + before[e];
                if (blockIdx.x == 0) reinterpret_cast<int2*>(a.segs)[e] = make_int2(first, c);
            }
            rows += __shfl_sync(~0u, upto, 31);
        }
    }
    __syncthreads();
    const int64_t lo = static_cast<int64_t>(w0) * kTokens * a.top, hi = min(lo + static_cast<int64_t>(kLayoutWords) * kTokens * a.top, a.n * a.top);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kLayoutThreads) {
        const int e = a.ids[i];
        int slot = -1;
        if (e >= 0) {
            const int64_t t = i / a.top;
            const int w = static_cast<int>(t / kTokens);
            slot = at[e] + __popc(words[static_cast<int64_t>(w) * E + e] & ((1u << (t % kTokens)) - 1u));
            for (int v = w0; v < w; ++v) slot += __popc(words[static_cast<int64_t>(v) * E + e]);
        }
        a.slots[i] = slot;
    }
}

int64_t words_of(int64_t n) { return (n + kTokens - 1) / kTokens; }

}  // namespace

extern "C" int64_t spk_route_scores_workspace_bytes(int64_t n, int experts) {
    if (n < 1 || experts < 1) return 0;
    return words_of(n) * experts * static_cast<int64_t>(sizeof(uint32_t));
}

extern "C" int spk_route_scores(const spk_route_scores_args* args, void* stream) {
    SpkRange nvtx_range("spk_route_scores");
    if (args == nullptr) return SPK_ERR_NULL_POINTER;
    const spk_route_scores_args& a = *args;
    if (a.n < 0 || a.experts < 1 || a.experts > 1024 || a.top < 1 || a.top > 32 || a.groups < 1 || a.experts % a.groups != 0 || a.top_groups < 1 ||
        a.top_groups > a.groups || a.top > a.experts / a.groups * a.top_groups)
        return SPK_ERR_BAD_SHAPE;
    if (a.dtype != SPK_F32 && a.dtype != SPK_BF16) return SPK_ERR_BAD_DTYPE;
    if (a.score != SPK_SCORE_SOFTMAX && a.score != SPK_SCORE_SIGMOID) return SPK_ERR_UNSUPPORTED;
    if (a.n > (1 << 24)) return SPK_ERR_TOO_LARGE;  // rows of the sorted matrix are 32-bit
    if (a.segs == nullptr) return SPK_ERR_NULL_POINTER;
    cudaStream_t s = spk_stream(stream);
    if (a.n > 0) {
        if (a.logits == nullptr || a.ids == nullptr || a.weights == nullptr || a.slots == nullptr) return SPK_ERR_NULL_POINTER;
        if (a.logits_stride < a.experts) return SPK_ERR_BAD_STRIDE;
        if (a.workspace == nullptr || a.workspace_bytes < spk_route_scores_workspace_bytes(a.n, a.experts)) return SPK_ERR_WORKSPACE_TOO_SMALL;
    }
    uint32_t* words = static_cast<uint32_t*>(a.workspace);
    const int n_words = static_cast<int>(words_of(a.n));
    if (a.n > 0) {
        const int bytes = a.experts * (kSelectWarps * 2 * 8 + 4);
        auto kernel = a.dtype == SPK_F32 ? score_select_kernel<float> : score_select_kernel<__nv_bfloat16>;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
        if (e != cudaSuccess) return spk_set_cuda_error(e);
        kernel<<<n_words, kSelectWarps * 32, bytes, s>>>(a, words);
        SPK_CHECK_LAUNCH();
    }
    const int grid = n_words == 0 ? 1 : (n_words + kLayoutWords - 1) / kLayoutWords;
    score_layout_kernel<<<grid, kLayoutThreads, 2 * sizeof(int32_t) * a.experts, s>>>(a, words, n_words);
    SPK_CHECK_LAUNCH();
    return SPK_OK;
}

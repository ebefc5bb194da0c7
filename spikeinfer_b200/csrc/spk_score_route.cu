// Experts chosen by scores: scores, bias, groups, the best few of a token, their weights, and the rows of the matrix sorted by expert.
//
// A warp per token, an expert of every 32 per lane.  Choices lie next to borders, where 32 bits would tell equal from unequal by how they were rounded, so they have to
// come out as in 64-bit arithmetic.  Nearly all of them are settled by 32-bit scores: where every difference that decides (each choice from the next, the worst group kept from
// the best one dropped) is beyond what the scores can be off by, it has the sign of the exact one.  Tokens with a difference that is not are done again in 64 bits
// (exact_choice; 64 bits for all of them: 8191 rows of 256 experts in eight groups 94 us, 64 rows 44).  Weights are 64-bit, of the chosen alone where they are divided by their sum.
//
// A CTA's 32 tokens leave one word per expert, a bit for every token that chose it (a token chooses an expert once).  A pair's row is what the words ahead count, and the
// bits below its own: no order of arrival enters, so the rows are the same every time.  Up to 256 tokens: a cluster's CTAs read one another's words, one launch.
// More: score_layout_kernel, from the words in memory.
#include "spk_experts.cuh"

namespace {

constexpr int kTokens = 32;        // per CTA of the selection: the bits of a word
constexpr int kMostCluster = 8;    // CTAs that hand out the rows among themselves
constexpr int kLayoutThreads = 1024;
constexpr int kLayoutWords = 8;    // words per CTA of the layout

// What a 32-bit score can be off by, relative to the score (and to the bias beside it): the exponent's rounding (100 * 2^-24 where the exponential is still normal), the
// exponential's 2 ulp, 13 sums and a reciprocal are under 2^-17; two of them make a difference.
constexpr float kOff = 1.52587890625e-5f;  // 2^-16

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
// Floats as integers of the same order; 0 is below all of them.
__device__ __forceinline__ uint32_t key_of(float f) {
    const uint32_t u = __float_as_uint(f);
    return u ^ ((u >> 31) != 0 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) != 0 ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ float warp_most(float f) { return of_key(__reduce_max_sync(~0u, key_of(f))); }

// NaN counts as -infinity, +infinity as the largest finite value.
template <typename T>
__device__ __forceinline__ float logit(const T* l, int e) {
    const float f = spk_to_float<T>(l[e]);
    return f != f ? -INFINITY : fminf(f, 3.402823466e38f);
}
__device__ __forceinline__ int padded(int e) { return e + (e >> 5 << 2); }  // groups of 32 side by side lie in banks of their own

// The largest logit (0 where there is none) and the sum of the exponentials.
template <typename T>
__device__ __noinline__ void exact_softmax(const T* l, int E, double& m, double& sum) {
    const int lane = threadIdx.x & 31;
    double top = -INFINITY, s = 0.0;
    for (int e = lane; e < E; e += 32) top = fmax(top, static_cast<double>(logit(l, e)));
    top = warp_max(top);
    m = top == -INFINITY ? 0.0 : top;
    for (int e = lane; e < E; e += 32) s += exp(static_cast<double>(logit(l, e)) - m);
    sum = warp_sum(s);
}

// The token's choices in 64 bits: lane j gets choice j, -1 where there is none.  c: 2 E doubles of shared memory of this warp.
template <typename T>
__device__ __noinline__ int exact_choice(const spk_route_scores_args& a, const T* l, double* c) {
    const int E = a.experts, lane = threadIdx.x & 31;
    double* gs = c + E;
    double m = 0.0, sum = 1.0;
    if (a.score == SPK_SCORE_SOFTMAX) exact_softmax(l, E, m, sum);
    __syncwarp();
    for (int e = lane; e < E; e += 32) {
        const double x = logit(l, e);
        double v = a.score == SPK_SCORE_SOFTMAX ? exp(x - m) / sum : 1.0 / (1.0 + exp(-x));
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
    int mine = -1;
    for (int j = 0; j < a.top; ++j) {
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
        if (lane == 0) c[at] = -INFINITY;
        __syncwarp();
    }
    return mine;
}

// The same by 32-bit scores; false where a difference that decides is too small for them.  x, b: this lane's logits and biases (expert lane + 32 i), c: padded(E) floats.
template <int P>
__device__ __forceinline__ bool fast_choice(const spk_route_scores_args& a, const float (&x)[P], const float (&b)[P], float bias_most, float* c, int& mine) {
    const int E = a.experts, lane = threadIdx.x & 31;
    uint32_t key[P];
    {
        float m = 0.0f, scale = 1.0f;
        float s[P];
        if (a.score == SPK_SCORE_SOFTMAX) {
            m = x[0];
#pragma unroll
            for (int i = 1; i < P; ++i) m = fmaxf(m, x[i]);
            m = warp_most(m);
            if (m == -INFINITY) m = 0.0f;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                s[i] = expf(x[i] - m);
                sum += s[i];
            }
            scale = 1.0f / spk_warp_sum(sum);
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float v = (a.score == SPK_SCORE_SOFTMAX ? s[i] * scale : 1.0f / (1.0f + expf(-x[i]))) + b[i];
            key[i] = x[i] == -INFINITY || v != v || v == -INFINITY ? 0u : key_of(v);
        }
    }
    if (a.groups > 1) {
        if (a.groups > 32) return false;
        const int per = E / a.groups;
        int L = 32;  // lanes of a group: a power of two
        while (L * a.groups > 32) L >>= 1;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (lane + 32 * i < E) c[padded(lane + 32 * i)] = key[i] != 0 ? of_key(key[i]) : -INFINITY;
        __syncwarp();
        const int g = lane / L;
        float first = -INFINITY, second = -INFINITY;
        if (g < a.groups) {
            for (int k = lane % L; k < per; k += L) {
                const float v = c[padded(g * per + k)];
                second = fmaxf(second, fminf(first, v));
                first = fmaxf(first, v);
            }
        }
        for (int o = L >> 1; o >= 1; o >>= 1) {
            const float f = __shfl_xor_sync(~0u, first, o), s = __shfl_xor_sync(~0u, second, o);
            second = fmaxf(fminf(first, f), fmaxf(second, s));
            first = fmaxf(first, f);
        }
        const float worth = second == -INFINITY ? first : first + second;
        int better = 0;
        for (int h = 0; h < a.groups; ++h) {
            const float w = __shfl_sync(~0u, worth, h * L);
            better += w > worth || (w == worth && h < g);
        }
        const bool there = g < a.groups, kept = there && better < a.top_groups;
        const float worst = -warp_most(kept ? -worth : -INFINITY), dropped = warp_most(there && !kept ? worth : -INFINITY);
        if (a.top_groups < a.groups && !(worst - dropped > 2.0f * kOff * (fabsf(worst) + 2.0f * bias_most))) return false;
        const uint32_t keep = __ballot_sync(~0u, kept);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if ((keep >> min(31, (lane + 32 * i) / per * L) & 1u) == 0) key[i] = 0;
    }
    mine = -1;
    float before = 0.0f;
    for (int j = 0; j <= a.top; ++j) {
        uint32_t most = key[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < P; ++i)
            if (key[i] > most) most = key[i], at = i;
        const uint32_t best = __reduce_max_sync(~0u, most);
        if (best == 0) break;
        const float v = of_key(best);
        if (j > 0 && !(before - v > kOff * (fabsf(before) + bias_most))) return false;
        if (j == a.top) break;
        const int who = __ffs(__ballot_sync(~0u, most == best)) - 1;
        const int e = __shfl_sync(~0u, lane + 32 * at, who);
        if (lane == who) {
#pragma unroll
            for (int i = 0; i < P; ++i)
                if (i == at) key[i] = 0;
        }
        if (lane == j) mine = e;
        before = v;
    }
    return true;
}

// Adds up what the words of the CTA's tokens and of those ahead count, and lays the segments out.  `word(w, e)`: word w of expert e.  at, before: E integers each; before[e] becomes the
// row of the first pair of this CTA's tokens (words from w0 on) that chose e.
template <typename Word>
__device__ __forceinline__ void lay_out(const spk_route_scores_args& a, int n_words, int w0, bool writes, int32_t* at, int32_t* before, Word word) {
    const int E = a.experts, threads = blockDim.x;
    for (int e = threadIdx.x; e < E; e += threads) at[e] = before[e] = 0;
    __syncthreads();
    const int wide = E < threads ? E : threads, parts = threads / wide, part = threadIdx.x / wide;
    if (part < parts) {
        for (int e = threadIdx.x % wide; e < E; e += wide) {
            int all = 0, ahead = 0;
#pragma unroll 8
            for (int w = part; w < n_words; w += parts) {
                const int c = __popc(word(w, e));
                all += c;
                if (w < w0) ahead += c;
            }
            if (all != 0) atomicAdd(at + e, all);
            if (ahead != 0) atomicAdd(before + e, ahead);
        }
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        int rows = 0;
        for (int e0 = 0; e0 < E; e0 += 32) {
            const int e = e0 + threadIdx.x;
            const int c = e < E ? at[e] : 0;
            const int pad = (c + kExpertAlign - 1) & ~(kExpertAlign - 1);
            int upto = pad;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int up = __shfl_up_sync(~0u, upto, o);
                if (static_cast<int>(threadIdx.x) >= o) upto += up;
            }
            if (e < E) {
                const int first = rows + upto - pad;
                before[e] += first;
                if (writes) reinterpret_cast<int2*>(a.segs)[e] = make_int2(first, c);
            }
            rows += __shfl_sync(~0u, upto, 31);
        }
    }
    __syncthreads();
}

__device__ __forceinline__ uint32_t cluster_load(const uint32_t* p, uint32_t rank) {
    uint32_t v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.u32 %0, [r];\n\t}\n"
                 : "=r"(v) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank) : "memory");
    return v;
}

// WHOLE: the grid is one cluster and hands out the rows as well.
template <typename T, int P, bool WHOLE>
__global__ void __launch_bounds__(1024)
score_select_kernel(const __grid_constant__ spk_route_scores_args a, uint32_t* words, const int n_words) {
    extern __shared__ double sm[];
    const int E = a.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    double* c64 = sm + static_cast<int64_t>(warp) * 2 * E;  // also the 32-bit scores
    uint32_t* word = reinterpret_cast<uint32_t*>(sm + static_cast<int64_t>(warps) * 2 * E);
    int32_t* chosen = reinterpret_cast<int32_t*>(word + E);  // WHOLE: [32][top], then 2 E integers
    for (int e = threadIdx.x; e < E; e += blockDim.x) word[e] = 0;
    float b[P], bias_most = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        b[i] = a.bias != nullptr && lane + 32 * i < E ? a.bias[lane + 32 * i] : 0.0f;
        if (fabsf(b[i]) < INFINITY) bias_most = fmaxf(bias_most, fabsf(b[i]));
    }
    bias_most = warp_most(bias_most);
    __syncthreads();
    for (int i = warp; i < kTokens; i += warps) {
        const int64_t t = static_cast<int64_t>(blockIdx.x) * kTokens + i;
        if (t >= a.n) break;
        int mine = -1;  // choice number `lane` of the token
        const T* l = static_cast<const T*>(a.logits) + t * a.logits_stride;
        double s = 0.0;
        if (a.active == nullptr || a.active[t] == 1) {
            float x[P];
#pragma unroll
            for (int k = 0; k < P; ++k) x[k] = lane + 32 * k < E ? logit(l, lane + 32 * k) : -INFINITY;
            if (!fast_choice<P>(a, x, b, bias_most, reinterpret_cast<float*>(c64), mine)) mine = exact_choice(a, l, c64);
            if (mine >= 0) atomicOr(word + mine, 1u << i);
            const double y = mine >= 0 ? static_cast<double>(logit(l, mine)) : 0.0;
            if (a.score == SPK_SCORE_SIGMOID) {
                s = 1.0 / (1.0 + exp(-y));
            } else if (a.renormalize) {  // the sum over all experts falls out of the quotient
                float top = x[0];
#pragma unroll
                for (int k = 1; k < P; ++k) top = fmaxf(top, x[k]);
                top = warp_most(top);
                s = exp(y - (top == -INFINITY ? 0.0 : static_cast<double>(top)));
            } else {
                double m, sum;
                exact_softmax(l, E, m, sum);
                s = exp(y - m) / sum;
            }
            if (mine < 0) s = 0.0;
            if (a.renormalize) {
                const double sum = warp_sum(s);
                s = sum > 0.0 ? s / sum : 0.0;
            }
        }
        if (lane < a.top) {
            a.ids[t * a.top + lane] = mine;
            a.weights[t * a.top + lane] = static_cast<float>(s * static_cast<double>(a.scale));
            if (WHOLE) chosen[i * a.top + lane] = mine;
        }
    }
    __syncthreads();
    if (!WHOLE) {
        for (int e = threadIdx.x; e < E; e += blockDim.x) words[static_cast<int64_t>(blockIdx.x) * E + e] = word[e];
        return;
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    int32_t *at = chosen + kTokens * a.top, *before = at + E;
    lay_out(a, n_words, blockIdx.x, blockIdx.x == 0, at, before, [&](int w, int e) { return cluster_load(word + e, w); });
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // the others' words have been read
    const int64_t first = static_cast<int64_t>(blockIdx.x) * kTokens;
    const int pairs = static_cast<int>(min(a.n - first, static_cast<int64_t>(kTokens))) * a.top;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const int e = chosen[i];
        a.slots[first * a.top + i] = e >= 0 ? before[e] + __popc(word[e] & ((1u << (i / a.top)) - 1u)) : -1;
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // no CTA leaves while its words are being read
}

__global__ void __launch_bounds__(kLayoutThreads)
score_layout_kernel(const spk_route_scores_args a, const uint32_t* __restrict__ words, const int n_words) {
    extern __shared__ int32_t sm32[];
    const int E = a.experts, w0 = blockIdx.x * kLayoutWords;
    int32_t *at = sm32, *before = at + E;
    spk_grid_wait();
    lay_out(a, n_words, w0, blockIdx.x == 0, at, before, [&](int w, int e) { return __ldcg(words + static_cast<int64_t>(w) * E + e); });
    const int64_t lo = static_cast<int64_t>(w0) * kTokens * a.top, hi = min(lo + static_cast<int64_t>(kLayoutWords) * kTokens * a.top, a.n * a.top);
    for (int64_t i = lo + threadIdx.x; i < hi; i += kLayoutThreads) {
        const int e = __ldcg(a.ids + i);
        int slot = -1;
        if (e >= 0) {
            const int64_t t = i / a.top;
            const int w = static_cast<int>(t / kTokens);
            slot = before[e] + __popc(__ldcg(words + static_cast<int64_t>(w) * E + e) & ((1u << (t % kTokens)) - 1u));
#pragma unroll
            for (int v = 0; v < kLayoutWords - 1; ++v)
                if (w0 + v < w) slot += __popc(__ldcg(words + static_cast<int64_t>(w0 + v) * E + e));
        }
        a.slots[i] = slot;
    }
}

int64_t words_of(int64_t n) { return (n + kTokens - 1) / kTokens; }

template <typename T, int P, bool WHOLE>
int launch_select(const spk_route_scores_args& a, uint32_t* words, int n_words, cudaStream_t s) {
    // 64-bit scores of a warp are kept in shared memory: as many warps as fit, 32 where few CTAs make the grid
    const int per = 16 * a.experts, extra = 4 * a.experts + (WHOLE ? 4 * (kTokens * a.top + 2 * a.experts) : 0);
    int warps = WHOLE || n_words <= 148 ? 32 : 16;
    while (warps * per + extra > 200 * 1024) warps /= 2;
    const int bytes = warps * per + extra;
    auto kernel = score_select_kernel<T, P, WHOLE>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim = {static_cast<unsigned>(n_words), 1, 1};
    cfg.gridDim = dim3(n_words);
    cfg.blockDim = dim3(32 * warps);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cfg.attrs = &attr;
    cfg.numAttrs = WHOLE ? 1 : 0;
    e = cudaLaunchKernelEx(&cfg, kernel, a, words, n_words);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    spk_count_launch();
    return SPK_OK;
}

template <typename T, bool WHOLE>
int select(const spk_route_scores_args& a, uint32_t* words, int n_words, cudaStream_t s) {
    if (a.experts <= 32) return launch_select<T, 1, WHOLE>(a, words, n_words, s);
    if (a.experts <= 64) return launch_select<T, 2, WHOLE>(a, words, n_words, s);
    if (a.experts <= 128) return launch_select<T, 4, WHOLE>(a, words, n_words, s);
    if (a.experts <= 256) return launch_select<T, 8, WHOLE>(a, words, n_words, s);
    if (a.experts <= 512) return launch_select<T, 16, WHOLE>(a, words, n_words, s);
    return launch_select<T, 32, WHOLE>(a, words, n_words, s);
}

}  // namespace

extern "C" int64_t spk_route_scores_workspace_bytes(int64_t n, int experts) {
    if (n <= kMostCluster * kTokens || experts < 1) return 0;
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
    uint32_t* words = static_cast<uint32_t*>(a.workspace);
    const int n_words = static_cast<int>(words_of(a.n));
    if (a.n > 0) {
        if (a.logits == nullptr || a.ids == nullptr || a.weights == nullptr || a.slots == nullptr) return SPK_ERR_NULL_POINTER;
        if (a.logits_stride < a.experts) return SPK_ERR_BAD_STRIDE;
        if (n_words <= kMostCluster) return a.dtype == SPK_F32 ? select<float, true>(a, words, n_words, s) : select<__nv_bfloat16, true>(a, words, n_words, s);
        if (a.workspace == nullptr || a.workspace_bytes < spk_route_scores_workspace_bytes(a.n, a.experts)) return SPK_ERR_WORKSPACE_TOO_SMALL;
        const int rc = a.dtype == SPK_F32 ? select<float, false>(a, words, n_words, s) : select<__nv_bfloat16, false>(a, words, n_words, s);
        if (rc != SPK_OK) return rc;
    }
    const int grid = n_words == 0 ? 1 : (n_words + kLayoutWords - 1) / kLayoutWords;
    return spk_launch(score_layout_kernel, dim3(grid), kLayoutThreads, 2 * sizeof(int32_t) * a.experts, s, n_words > 0, a, words, n_words);
}

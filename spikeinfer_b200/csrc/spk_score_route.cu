// Experts chosen by scores: scores, bias, groups, the best few of a token, their weights, and the rows of the matrix sorted by expert.
//
// A warp per token, an expert of every 32 per lane.  Choices lie next to borders, where 32 bits would tell equal from unequal by how they were rounded, so they have to
// come out as in 64-bit arithmetic.  Nearly all of them are settled by 32-bit scores: where every difference that decides (each choice from the next, the worst group kept from
// the best one dropped) is beyond what the scores can be off by, it has the sign of the exact one.  Where one is not, the groups, or the experts that can be among the chosen, are
// compared in 64 bits.  (64 bits for every token: 8191 rows of 256 experts in eight groups 94 us, 64 rows 44; for the whole of a token that is not settled: 49 and 13; so, with the layout's loads side by side, 34 and 9.5.)
//
// What bounds it: some 1300 instructions a token (scores 200, groups 250, choices 500, weights 100) and their latency; reading the logits would take 1.4 of the 35 us.  The form of more than 128 tokens
// has 64 registers (two CTAs of 512 threads on an SM) and spills 64 to 100 bytes a thread up to 256 experts, 0.2 KB up to 512, 0.9 KB beyond.
//
// A CTA's 32 tokens leave one word per expert, a bit for every token that chose it (a token chooses an expert once).  A pair's row is what the words ahead count, and the
// bits below its own: no order of arrival enters, so the rows are the same every time.  Up to 128 tokens: a cluster's CTAs read one another's words, one launch.
// More: score_layout_kernel, from the words in memory; beyond kAllWords, where every CTA's counting of all of them would grow with the square of the tokens, from counts
// by chunks of words that two more launches sum up (score_count_kernel, score_scan_kernel).
#include "spk_experts.cuh"
#include "spk_tensor.cuh"

namespace {

using namespace spk_tc;

constexpr int kTokens = 32;        // per CTA of the selection, at most: the bits of a word
constexpr int kMostCluster = 8;    // CTAs that hand out the rows among themselves
constexpr int kMostWhole = 128;    // tokens of such a launch
constexpr int kWholeTokens = kMostWhole / kMostCluster;  // of a CTA of it
constexpr int kLayoutThreads = 1024;
constexpr int kLayoutWords = 8;    // words per CTA of the layout
// Words that every CTA of the layout counts by itself; beyond, those of a chunk of kChunkWords (a multiple of kLayoutWords) are counted together.  us in all, by itself / by chunks: 32768 tokens
// of 64 experts 34 / 37, of 256 87 / 78; 65536 68 / 62 and 190 / 147; 262144 381 / 239 and 1167 / 539.
constexpr int kAllWords = 1024, kChunkWords = 64;

// What makes a difference of two 32-bit scores settled: off times the larger (and the bias beside it) and kLeast.  The exponential's argument is off by |x| 2^-23 at most (a product, or a
// difference and a product), which moves a sigmoid s by s (1 - s) |x| 2^-23 < 2^-25 and a softmax weight by d e^-d 2^-23 < 2^-24 (d: distance from the largest logit): kLeast.  The approximate
// exponential and reciprocal and the sum under it move s by 2^-21, the sums of a softmax (37 roundings of up to 1024 terms) by 2^-18.6, the bias' addition c by 2^-24, and the
// bits that a key gives up to the expert's place by 2^-20 (three bits) or 2^-18.  Twice all that for a difference, and up to the next power of two.
constexpr float kLeast = 2.384185791015625e-7f;  // 2^-22
__device__ __forceinline__ float off_of(int score, bool key, bool wide) {
    const float sigmoid = key ? wide ? 1.52587890625e-5f : 3.814697265625e-6f : 9.5367431640625e-7f;  // 2^-16, 2^-18, 2^-20
    return score == SPK_SCORE_SIGMOID ? sigmoid : wide ? 1.52587890625e-5f : 7.62939453125e-6f;        // 2^-16, 2^-17
}

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

// Lanes for each of up to 32 groups: a power of two.
__device__ __forceinline__ int lanes_of(int groups) {
    int L = 32;
    while (L * groups > 32) L >>= 1;
    return L;
}

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

// What the choice goes by, in 64 bits.
__device__ __forceinline__ double exact_score(const spk_route_scores_args& a, float logit, float bias, double m, double sum) {
    const double x = logit, v = (a.score == SPK_SCORE_SOFTMAX ? exp(x - m) / sum : 1.0 / (1.0 + exp(-x))) + static_cast<double>(bias);
    return logit == -INFINITY || v != v ? -INFINITY : v;
}

// Which groups stay, in 64 bits: a bit for the first lane of each (up to 32 groups).  c: E doubles of shared memory of this warp.
template <typename T>
__device__ __noinline__ uint32_t exact_groups(const spk_route_scores_args& a, const T* l, double* c) {
    const int E = a.experts, lane = threadIdx.x & 31, per = E / a.groups, L = lanes_of(a.groups), g = lane / L;
    double m = 0.0, sum = 1.0;
    if (a.score == SPK_SCORE_SOFTMAX) exact_softmax(l, E, m, sum);
    __syncwarp();
    for (int e = lane; e < E; e += 32) c[e] = exact_score(a, logit(l, e), a.bias != nullptr ? a.bias[e] : 0.0f, m, sum);
    __syncwarp();
    double first = -INFINITY, second = -INFINITY;
    if (g < a.groups) {
        for (int k = lane % L; k < per; k += L) {
            const double v = c[g * per + k];
            second = fmax(second, fmin(first, v));
            first = fmax(first, v);
        }
    }
    for (int o = L >> 1; o >= 1; o >>= 1) {
        const double f = __shfl_xor_sync(~0u, first, o), s = __shfl_xor_sync(~0u, second, o);
        second = fmax(fmin(first, f), fmax(second, s));
        first = fmax(first, f);
    }
    const double worth = second == -INFINITY ? first : first + second;
    int better = 0;
    for (int h = 0; h < a.groups; ++h) {
        const double w = __shfl_sync(~0u, worth, h * L);
        better += w > worth || (w == worth && h < g);
    }
    __syncwarp();
    return __ballot_sync(~0u, g < a.groups && better < a.top_groups);
}

// The order of n <= 32 experts (lane q: list[q]) in 64 bits: lane j gets the j-th of them, -1 where there is none or j >= top.
template <typename T>
__device__ __noinline__ int exact_order(const spk_route_scores_args& a, const T* l, const int* list, int n) {
    const int lane = threadIdx.x & 31, e = lane < n ? list[lane] : 0;
    double m = 0.0, sum = 1.0;
    if (a.score == SPK_SCORE_SOFTMAX) exact_softmax(l, a.experts, m, sum);
    const double c = lane < n ? exact_score(a, logit(l, e), a.bias != nullptr ? a.bias[e] : 0.0f, m, sum) : -INFINITY;
    int rank = 0;
    for (int q = 0; q < n; ++q) {
        const double w = __shfl_sync(~0u, c, q);
        const int f = __shfl_sync(~0u, e, q);
        rank += w > c || (w == c && f < e);
    }
    if (lane >= n) rank = 32;
    int mine = -1;
    for (int j = 0; j < a.top && j < n; ++j) {
        const int who = __ffs(__ballot_sync(~0u, rank == j)) - 1, got = __shfl_sync(~0u, e, who);
        if (lane == j) mine = got;
    }
    return mine;
}

// The token's choices in 64 bits: lane j gets choice j, -1 where there is none.  c: 2 E doubles of shared memory of this warp.
template <typename T>
__device__ __noinline__ int exact_choice(const spk_route_scores_args& a, const T* l, double* c) {
    const int E = a.experts, lane = threadIdx.x & 31;
    double* gs = c + E;
    double m = 0.0, sum = 1.0;
    if (a.score == SPK_SCORE_SOFTMAX) exact_softmax(l, E, m, sum);
    __syncwarp();
    for (int e = lane; e < E; e += 32) c[e] = exact_score(a, logit(l, e), a.bias != nullptr ? a.bias[e] : 0.0f, m, sum);
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

// Falling order; a network of exchanges.
template <int P>
__device__ __forceinline__ void sort_keys(uint32_t (&key)[P]) {
#pragma unroll
    for (int k = 2; k <= P; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1)
#pragma unroll
            for (int i = 0; i < P; ++i)
                if ((i & j) == 0) {
                    const uint32_t hi = max(key[i], key[i | j]), lo = min(key[i], key[i | j]);
                    key[i] = (i & k) == 0 ? hi : lo;
                    key[i | j] = (i & k) == 0 ? lo : hi;
                }
}

// The token's choices.  x, b: this lane's logits and biases (expert lane + 32 i), bit: where a group's bit is, c64: 2 E doubles of shared memory of this warp.  A key's last bits name the
// expert's place in the lane, the first of equal ones the largest.
template <typename T, int P>
__device__ __forceinline__ int choose(const spk_route_scores_args& a, const T* l, const float (&x)[P], const float (&b)[P], const int (&bit)[P], float bias_most, double* c64) {
    constexpr uint32_t PLACE = P - 1;
    if (a.groups > 32) return exact_choice(a, l, c64);
    const int E = a.experts, lane = threadIdx.x & 31;
    float* c = reinterpret_cast<float*>(c64);
    float v[P];
    {
        float m = 0.0f, scale = 1.0f;
        if (a.score == SPK_SCORE_SOFTMAX) {
            m = x[0];
#pragma unroll
            for (int i = 1; i < P; ++i) m = fmaxf(m, x[i]);
            m = warp_most(m);
            if (m == -INFINITY) m = 0.0f;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                v[i] = ex2((x[i] - m) * 1.4426950408889634f);
                sum += v[i];
            }
            scale = rcp(spk_warp_sum(sum));
        }
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const float y = (a.score == SPK_SCORE_SOFTMAX ? v[i] * scale : sigmoid_fast(x[i])) + b[i];
            v[i] = x[i] == -INFINITY || y != y ? -INFINITY : y;
        }
    }
    if (a.groups > 1 && a.top_groups < a.groups) {
        __syncwarp();
#pragma unroll
        for (int i = 0; i < P; ++i)
            if (lane + 32 * i < E) c[padded(lane + 32 * i)] = v[i];
        __syncwarp();
        const int per = E / a.groups, L = lanes_of(a.groups), g = lane / L;
        float first = -INFINITY, second = -INFINITY;
        if (g < a.groups) {
#pragma unroll 4
            for (int k = lane % L; k < per; k += L) {
                const float y = c[padded(g * per + k)];
                second = fmaxf(second, fminf(first, y));
                first = fmaxf(first, y);
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
        uint32_t keep = __ballot_sync(~0u, kept);
        if (!(worst - dropped > 2.0f * (off_of(a.score, false, P > 8) * (fabsf(worst) + 2.0f * bias_most) + kLeast))) keep = exact_groups(a, l, c64);
#pragma unroll
        for (int i = 0; i < P; ++i)
            if ((keep >> bit[i] & 1u) == 0) v[i] = -INFINITY;
    }
    uint32_t key[P];
#pragma unroll
    for (int i = 0; i < P; ++i) key[i] = v[i] == -INFINITY ? 0u : (key_of(v[i]) & ~PLACE) | (PLACE - i);
    sort_keys<P>(key);  // the lane's best is its first, and a choice moves its others up
    const float off = off_of(a.score, true, P > 8);
    int mine = -1, last = 0;
    float before = 0.0f, apart = 0.0f;
    bool settled = true;
    for (int j = 0; j <= a.top; ++j) {
        const uint32_t most = key[0], best = __reduce_max_sync(~0u, most);
        if (best == 0) {
            before = -INFINITY;  // everything there is has been chosen
            break;
        }
        const int who = __ffs(__ballot_sync(~0u, most == best)) - 1, place = PLACE - static_cast<int>(best & PLACE), e = who + 32 * place;  // equal ones by index
        const float y = of_key(best & ~PLACE);
        // experts of the very same logit and bias are equal in 64 bits too
        if (j > 0 && !(before - y > apart)) {
            const float x0 = logit(l, last), b0 = a.bias != nullptr ? a.bias[last] : 0.0f;
            if (x0 != logit(l, e) || (a.bias != nullptr && b0 != a.bias[e])) {
                settled = false;
            } else if (j == a.top && settled) {  // nor may one behind the cut, which is neither of the two, be better than they
                bool other = false;
#pragma unroll
                for (int i = 0; i < P; ++i)
                    other = other || (v[i] != -INFINITY && (key_of(v[i]) & ~PLACE) <= key_of(before) && !(v[i] < before - apart) && (x[i] != x0 || b[i] != b0));
                if (__any_sync(~0u, other)) settled = false;
            }
        }
        if (j == a.top) break;
        if (lane == who) {
#pragma unroll
            for (int i = 0; i + 1 < P; ++i) key[i] = key[i + 1];
            key[P - 1] = 0;
        }
        if (lane == j) mine = e;
        before = y;
        apart = off * (fabsf(y) + bias_most) + kLeast;
        last = e;
    }
    if (settled) return mine;
    // Those that can be among the chosen, in 64 bits.
    const float from = before - apart;  // NaN (infinite biases): all of them
    int* list = reinterpret_cast<int*>(c64);
    int n = 0;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < P; ++i) {
        const bool in = v[i] != -INFINITY && !(v[i] < from);
        const uint32_t all = __ballot_sync(~0u, in);
        const int at = n + __popc(all & ((1u << lane) - 1u));
        if (in && at < 32) list[at] = lane + 32 * i;
        n += __popc(all);
    }
    __syncwarp();
    return n <= 32 ? exact_order(a, l, list, n) : exact_choice(a, l, c64);
}

// Lays the segments out.  at: all pairs of every expert; before: its pairs ahead of this CTA's tokens, which becomes the row of the first pair of theirs.  sums: 32 integers.
__device__ __forceinline__ void lay_out(const spk_route_scores_args& a, bool writes, const int32_t* at, int32_t* before, int32_t* sums) {
    const int E = a.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5, chunks = (E + 31) / 32;
    auto scan = [&](int v) {  // of the lanes up to this one
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(~0u, v, o);
            if (lane >= o) v += up;
        }
        return v;
    };
    auto rows_of = [](int c) { return (c + kExpertAlign - 1) & ~(kExpertAlign - 1); };
    for (int k = warp; k < chunks; k += warps) {
        const int upto = scan(32 * k + lane < E ? rows_of(at[32 * k + lane]) : 0);
        if (lane == 31) sums[k] = upto;
    }
    __syncthreads();
    const int mine = lane < chunks ? sums[lane] : 0, ahead = scan(mine) - mine;  // of chunk `lane`
    for (int k = warp; k < chunks; k += warps) {
        const int e = 32 * k + lane, c = e < E ? at[e] : 0, rows = rows_of(c);
        const int first = __shfl_sync(~0u, ahead, k) + scan(rows) - rows;
        if (e < E) {
            before[e] += first;
            if (writes) reinterpret_cast<int2*>(a.segs)[e] = make_int2(first, c);
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

// WHOLE: the grid is one cluster and hands out the rows as well; at most kWholeTokens tokens, a warp each, so that a thread may have 128 registers and few spill (64 of them, a bound of
// 1024 threads: 64 tokens of 256 experts 12.4 us against 11.7, of 384 16.5 against 14.9).
template <typename T, int P, bool WHOLE>
__global__ void __launch_bounds__(512, WHOLE ? 1 : 2)
score_select_kernel(const __grid_constant__ spk_route_scores_args a, uint32_t* words, const int n_words, const int tokens) {
    extern __shared__ double sm[];
    const int E = a.experts, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    double* c64 = sm + static_cast<int64_t>(warp) * 2 * E;  // also the 32-bit scores
    uint32_t* word = reinterpret_cast<uint32_t*>(sm + static_cast<int64_t>(warps) * 2 * E);
    int32_t* chosen = reinterpret_cast<int32_t*>(word + E);  // WHOLE: [kWholeTokens][top], then 2 E + 32 integers
    for (int e = threadIdx.x; e < E; e += blockDim.x) word[e] = 0;
    float b[P], bias_most = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
        b[i] = a.bias != nullptr && lane + 32 * i < E ? a.bias[lane + 32 * i] : 0.0f;
        if (fabsf(b[i]) < INFINITY) bias_most = fmaxf(bias_most, fabsf(b[i]));
    }
    bias_most = warp_most(bias_most);
    int bit[P];
    const int per = E / a.groups, L = a.groups <= 32 ? lanes_of(a.groups) : 1, inverse = ((1 << 20) + per - 1) / per;
#pragma unroll
    for (int i = 0; i < P; ++i) bit[i] = min(31, (lane + 32 * i) * inverse / (1 << 20) * L);  // expert / per: experts and groups of up to 1024
    __syncthreads();
    for (int i = warp; i < tokens; i += warps) {
        const int64_t t = static_cast<int64_t>(blockIdx.x) * tokens + i;
        if (t >= a.n) break;
        int mine = -1;  // choice number `lane` of the token
        const T* l = static_cast<const T*>(a.logits) + t * a.logits_stride;
        float s = 0.0f;
        if (a.active == nullptr || a.active[t] == 1) {
            float x[P];
#pragma unroll
            for (int k = 0; k < P; ++k) x[k] = lane + 32 * k < E ? logit(l, lane + 32 * k) : -INFINITY;
            mine = choose<T, P>(a, l, x, b, bit, bias_most, c64);
            if (mine >= 0) atomicOr(word + mine, 1u << i);
            // 32-bit weights, every exponent at most zero.  sigmoid(y) = exp(min(y, 0)) / (1 + exp(-|y|)).  Where they are divided by their sum, a factor of all of them falls out (the sum of a
            // softmax too): the exponents count from the largest of the chosen, unless 64 bits would have had nothing left of it.
            const float y = mine >= 0 ? logit(l, mine) : -INFINITY;
            float m = 0.0f;
            if (a.score == SPK_SCORE_SIGMOID) {
                if (a.renormalize) m = warp_most(fminf(y, 0.0f));
                s = m < -745.0f ? 0.0f : expf(fminf(y, 0.0f) - m) / (1.0f + expf(-fabsf(y)));
            } else {
                float top = x[0], sum = 0.0f;
#pragma unroll
                for (int k = 1; k < P; ++k) top = fmaxf(top, x[k]);
                top = warp_most(top);
                m = a.renormalize ? warp_most(y) : top;
                s = m - top < -745.0f ? 0.0f : expf(y - m);
                if (!a.renormalize) {
#pragma unroll
                    for (int k = 0; k < P; ++k) sum += expf(x[k] - m);
                    s /= spk_warp_sum(sum);
                }
            }
            if (mine < 0) s = 0.0f;
            if (a.renormalize) {
                const float sum = spk_warp_sum(s);
                s = sum > 0.0f ? s / sum : 0.0f;
            }
        }
        if (lane < a.top) {
            a.ids[t * a.top + lane] = mine;
            a.weights[t * a.top + lane] = s * a.scale;
            if (WHOLE) chosen[i * a.top + lane] = mine;
        }
    }
    __syncthreads();
    if (!WHOLE) {
        // [expert][word], whole 16 bytes of them
        const int row = (n_words + 3) & ~3, behind = blockIdx.x + 1 == n_words ? row - n_words : 0;
        for (int e = threadIdx.x; e < E; e += blockDim.x)
            for (int k = 0; k <= behind; ++k) words[static_cast<int64_t>(e) * row + blockIdx.x + k] = k == 0 ? word[e] : 0u;
        return;
    }
    cluster_sync();
    int32_t *at = chosen + kWholeTokens * a.top, *before = at + E;
    for (int e = threadIdx.x; e < E; e += blockDim.x) {
        int all = 0, ahead = 0;
#pragma unroll
        for (int w = 0; w < kMostCluster; ++w) {
            const int c = w < n_words ? __popc(cluster_load(word + e, w)) : 0;
            all += c;
            if (w < static_cast<int>(blockIdx.x)) ahead += c;
        }
        at[e] = all;
        before[e] = ahead;
    }
    __syncthreads();
    lay_out(a, blockIdx.x == 0, at, before, before + E);
    cluster_arrive();  // the others' words have been read
    const int64_t first = static_cast<int64_t>(blockIdx.x) * tokens;
    const int pairs = static_cast<int>(min(a.n - first, static_cast<int64_t>(tokens))) * a.top;
    for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
        const int e = chosen[i];
        a.slots[first * a.top + i] = e >= 0 ? before[e] + __popc(word[e] & ((1u << (i / a.top)) - 1u)) : -1;
    }
    cluster_wait();  // no CTA leaves while its words are being read
}

// counts [chunk][expert] <- the pairs of a chunk's words, 16 lanes an expert.
__global__ void __launch_bounds__(kLayoutThreads)
score_count_kernel(const uint32_t* __restrict__ words, const int n_words, const int E, int32_t* __restrict__ counts) {
    constexpr int L = kChunkWords / 4;
    const int row = (n_words + 3) & ~3, q = blockIdx.x * L + threadIdx.x % L;
    spk_grid_wait();
    for (int e0 = 0; e0 < E; e0 += kLayoutThreads / L) {
        const int e = e0 + threadIdx.x / L;
        int c = 0;
        if (e < E && q < row / 4) {
            const uint4 u = __ldcg(reinterpret_cast<const uint4*>(words + static_cast<int64_t>(e) * row) + q);
            c = __popc(u.x) + __popc(u.y) + __popc(u.z) + __popc(u.w);
        }
        __syncwarp();
#pragma unroll
        for (int o = L / 2; o >= 1; o >>= 1) c += __shfl_xor_sync(~0u, c, o);
        if (e < E && threadIdx.x % L == 0) counts[static_cast<int64_t>(blockIdx.x) * E + e] = c;
    }
}

// counts [chunk][expert] <- the pairs ahead of a chunk, and behind the last chunk all pairs.  A lane per expert, a run of chunks per warp.
__global__ void __launch_bounds__(1024)
score_scan_kernel(int32_t* __restrict__ counts, const int chunks, const int E) {
    __shared__ int32_t runs[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int lo = static_cast<int>(static_cast<int64_t>(chunks) * warp / 32), hi = static_cast<int>(static_cast<int64_t>(chunks) * (warp + 1) / 32);
    int32_t* mine = counts + (e < E ? e : 0);
    spk_grid_wait();
    int sum = 0;
#pragma unroll 8
    for (int k = lo; k < hi; ++k) sum += e < E ? __ldcg(mine + static_cast<int64_t>(k) * E) : 0;
    runs[warp][lane] = sum;
    __syncthreads();
    int ahead = 0;
    for (int w = 0; w < warp; ++w) ahead += runs[w][lane];
#pragma unroll 8
    for (int k = lo; k < hi; ++k) {
        if (e >= E) break;
        const int c = __ldcg(mine + static_cast<int64_t>(k) * E);
        mine[static_cast<int64_t>(k) * E] = ahead;
        ahead += c;
    }
    if (warp == 31 && e < E) mine[static_cast<int64_t>(chunks) * E] = ahead;
}

// ALL: this CTA counts all words; else counts is score_scan_kernel's.
template <bool ALL>
__global__ void __launch_bounds__(kLayoutThreads)
score_layout_kernel(const spk_route_scores_args a, const uint32_t* __restrict__ words, const int n_words, const int tokens, const int32_t* __restrict__ counts, const int chunks) {
    extern __shared__ int32_t sm32[];  // [experts] twice, 32
    const int E = a.experts, w0 = blockIdx.x * kLayoutWords, row = (n_words + 3) & ~3, quads = row / 4;
    const int chunk = w0 / kChunkWords, from = ALL ? 0 : chunk * (kChunkWords / 4), upto = ALL ? quads : w0 / 4;  // what is counted here
    int32_t *at = sm32, *before = at + E;
    spk_grid_wait();
    auto load = [&](int e, int q) { return __ldcg(reinterpret_cast<const uint4*>(words + static_cast<int64_t>(e) * row) + q); };
    auto count = [](const uint4& u, int n) {  // of the first n words
        return (n > 0 ? __popc(u.x) : 0) + (n > 1 ? __popc(u.y) : 0) + (n > 2 ? __popc(u.z) : 0) + (n > 3 ? __popc(u.w) : 0);
    };
    // Lanes side by side take a row's words, 16 bytes each and about eight loads a lane: 8192 tokens' words of 256 experts in two passes.
    int side = 1;
    while (side < 32 && 8 * side < upto - from) side <<= 1;
    for (int e0 = 0; e0 < E; e0 += kLayoutThreads / side) {
        const int e = e0 + threadIdx.x / side;
        int all = 0, ahead = 0;
#pragma unroll 8
        for (int q = from + threadIdx.x % side; q < upto; q += side) {
            const int c = e < E ? count(load(e, q), 4) : 0;
            all += c;
            if (4 * q < w0) ahead += c;  // w0 is a multiple of four
        }
        __syncwarp();
        for (int o = side >> 1; o >= 1; o >>= 1) {
            all += __shfl_xor_sync(~0u, all, o);
            ahead += __shfl_xor_sync(~0u, ahead, o);
        }
        if (e < E && threadIdx.x % side == 0) {
            at[e] = ALL ? all : __ldcg(counts + static_cast<int64_t>(chunks) * E + e);
            before[e] = ALL ? ahead : ahead + __ldcg(counts + static_cast<int64_t>(chunk) * E + e);
        }
    }
    __syncthreads();
    lay_out(a, blockIdx.x == 0, at, before, before + E);
    const int64_t lo = static_cast<int64_t>(w0) * tokens * a.top;
    const int pairs = static_cast<int>(min(static_cast<int64_t>(kLayoutWords) * tokens, a.n - static_cast<int64_t>(w0) * tokens)) * a.top;
    for (int i = threadIdx.x; i < pairs; i += kLayoutThreads) {
        const int e = __ldcg(a.ids + lo + i);
        int slot = -1;
        if (e >= 0) {
            const int t = i / a.top, w = t / tokens;  // word of the CTA's
            const uint4 u = load(e, w0 / 4), v = w0 / 4 + 1 < quads ? load(e, w0 / 4 + 1) : make_uint4(0u, 0u, 0u, 0u);
            const uint32_t own = w < 4 ? (w < 2 ? (w == 0 ? u.x : u.y) : (w == 2 ? u.z : u.w)) : (w < 6 ? (w == 4 ? v.x : v.y) : (w == 6 ? v.z : v.w));
            slot = before[e] + __popc(own & ((1u << (t % tokens)) - 1u)) + count(u, w) + count(v, w - 4);
        }
        a.slots[lo + i] = slot;
    }
}

// Tokens per CTA of the selection.  Up to 128 in all: eight CTAs share them evenly (a CTA's warps share four schedulers: 64 rows of 256 experts 9.5 us, 256 rows 14.9).  More: eight each while all of
// them are on the chip at once (257 and 1024 rows 12.9 and 14.5 us, with 32 each 19.9 and 22.5).
int tokens_of(int64_t n) { return n <= kMostWhole ? static_cast<int>((n + kMostCluster - 1) / kMostCluster) : n <= 148 * 8 ? 8 : n <= 148 * 16 ? 16 : kTokens; }
int64_t words_of(int64_t n) { return n < 1 ? 0 : (n + tokens_of(n) - 1) / tokens_of(n); }
int64_t word_bytes(int64_t n, int64_t experts) { return (words_of(n) + 3) / 4 * 16 * experts; }
int64_t chunks_of(int64_t n) { return words_of(n) <= kAllWords ? 0 : (words_of(n) + kChunkWords - 1) / kChunkWords; }

template <typename T, int P, bool WHOLE>
int launch_select(const spk_route_scores_args& a, uint32_t* words, int n_words, cudaStream_t s) {
    const int tokens = tokens_of(a.n);
    // 64-bit scores of a warp are kept in shared memory: as many warps as fit
    const int per = 16 * a.experts, extra = 4 * a.experts + (WHOLE ? 4 * (kWholeTokens * a.top + 2 * a.experts + 32) : 0);
    int warps = !WHOLE ? min(tokens, 16) : tokens < 8 ? 8 : tokens;  // eight at least hand out the rows
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
    e = cudaLaunchKernelEx(&cfg, kernel, a, words, n_words, tokens);
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
    if (n <= kMostWhole || experts < 1) return 0;
    return word_bytes(n, experts) + (chunks_of(n) > 0 ? (chunks_of(n) + 1) * 4 * experts : 0);
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
        if (a.n <= kMostWhole) return a.dtype == SPK_F32 ? select<float, true>(a, words, n_words, s) : select<__nv_bfloat16, true>(a, words, n_words, s);
        if (a.workspace == nullptr || a.workspace_bytes < spk_route_scores_workspace_bytes(a.n, a.experts)) return SPK_ERR_WORKSPACE_TOO_SMALL;
        if (reinterpret_cast<uintptr_t>(a.workspace) % 16 != 0) return SPK_ERR_BAD_STRIDE;
        const int rc = a.dtype == SPK_F32 ? select<float, false>(a, words, n_words, s) : select<__nv_bfloat16, false>(a, words, n_words, s);
        if (rc != SPK_OK) return rc;
    }
    const int grid = n_words == 0 ? 1 : (n_words + kLayoutWords - 1) / kLayoutWords, chunks = static_cast<int>(chunks_of(a.n));
    const size_t bytes = sizeof(int32_t) * (2 * a.experts + 32);
    int32_t* counts = nullptr;
    if (chunks == 0) return spk_launch(score_layout_kernel<true>, dim3(grid), kLayoutThreads, bytes, s, n_words > 0, a, words, n_words, tokens_of(a.n), counts, chunks);
    counts = reinterpret_cast<int32_t*>(static_cast<uint8_t*>(a.workspace) + word_bytes(a.n, a.experts));
    int rc = spk_launch(score_count_kernel, dim3(chunks), kLayoutThreads, 0, s, true, words, n_words, a.experts, counts);
    if (rc == SPK_OK) rc = spk_launch(score_scan_kernel, dim3((a.experts + 31) / 32), 1024, 0, s, true, counts, chunks, a.experts);
    if (rc == SPK_OK) rc = spk_launch(score_layout_kernel<false>, dim3(grid), kLayoutThreads, bytes, s, true, a, words, n_words, tokens_of(a.n), counts, chunks);
    return rc;
}

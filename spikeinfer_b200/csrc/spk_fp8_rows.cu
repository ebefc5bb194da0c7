// Rows in e4m3 with one scale for every 128 columns: what the products of spk_fp8_linear.cu read.
//
//  * boundary8_kernel: x' = x + delta + the weighted rows of the token's experts, RMS norm of x' as it is stored, and the norm's output in 8 bits.
//  * quantize8_kernel: an activation and the same 8-bit form of its result.
//
// A block of 128 columns is the four-column groups of one warp, so its largest magnitude is one warp reduction away.  scale = most / 448 (448: the
// largest e4m3 value), value = round(v / scale), saturating: NaN stays NaN and is no candidate for the largest, an infinity counts as the
// largest finite value.  A block below 2^-100 is scaled as if its largest magnitude was that, so that no reciprocal overflows.
// Both quotients are what a 32-bit division gives, by Markstein's correction of a product with the reciprocal (q + (a - q b) / b, the remainder without a rounding), two values an instruction.  Products
// alone / corrected / one value an instruction, us: 8192 x 3584 boundary 38.9 / 39.9 / 40.9, gate of 8192 x 18944 131 / 125 / 128, no activation 78 / 84 / 86, gelu of 8192 x 4864 33.4 / 34.8 / 35.5.
// 16-bit values over a scale of few bits lie exactly between two e4m3 values once in a thousand, where the product alone, or a scale that is off by a unit, takes the other one.
#include <cuda_fp8.h>
#include <float.h>

#include "spk_dense.cuh"
#include "spk_tensor.cuh"

namespace {

using namespace spk_tc;

constexpr float kMostE4m3 = 448.0f;
constexpr float kLeastBlock = 7.888609052210118e-31f;  // 2^-100

// a / b; by: next to 1 / b.
__device__ __forceinline__ float quotient(float a, float b, float by) {
    const float q = a * by;
    return fmaf(fmaf(-q, b, a), by, q);
}
// Four values over b, two at a time.
__device__ __forceinline__ uint32_t pack_e4m3(const float* f, float b, float by) {
    const uint64_t nb = f2_pack(-b, -b), y = f2_pack(by, by);
    auto two = [&](const float* a) {
        const uint64_t v = f2_pack(a[0], a[1]), q = f2_mul(v, y);
        float2 r;
        f2_unpack(f2_fma(f2_fma(q, nb, v), y, q), r.x, r.y);
        return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(r, __NV_SATFINITE, __NV_E4M3));
    };
    return two(f) | two(f + 2) << 16;
}

// C columns of a thread and how they lie.  kWide: consecutive ones, all of them there or none, on a 16-byte boundary (or that of their own size).  Else C = 4 and a warp's
// elements lie side by side: kPairs (rows begin at multiples of two elements) columns 0, 1, 64 and 65 from the thread's first on, kSingle every 32nd, those that are there.
// 8192 rows of 4102 bf16: 374 us with four consecutive ones each, read one by one, 153 with every 32nd, 71 in pairs whose loads are not waited for one by one.
constexpr int kSingle = 0, kPairs = 1, kWide = 2;
template <int C>
struct Cols {
    float f[C];
};
template <int VEC>
__device__ __forceinline__ constexpr int nth(int i) {
    return VEC == kPairs ? (i >> 1) * 64 + (i & 1) : 32 * i;
}
template <int C, int VEC, typename T>
__device__ __forceinline__ Cols<C> load_cols(const T* p, int left) {
    Cols<C> r;
    if constexpr (VEC == kSingle) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            T v = spk_from_float<T>(0.0f);  // converted behind the branch, so that all loads are under way together
            if (nth<VEC>(i) < left) v = p[nth<VEC>(i)];
            r.f[i] = spk_to_float<T>(v);
        }
    } else if constexpr (VEC == kPairs) {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            if constexpr (sizeof(T) == 4) {
                float2 v = make_float2(0.0f, 0.0f);
                if (nth<VEC>(i) < left) v = *reinterpret_cast<const float2*>(p + nth<VEC>(i));
                r.f[i] = v.x, r.f[i + 1] = v.y;
            } else {
                uint32_t u = 0;
                if (nth<VEC>(i) < left) u = *reinterpret_cast<const uint32_t*>(p + nth<VEC>(i));
                r.f[i] = __uint_as_float(u << 16), r.f[i + 1] = __uint_as_float(u & 0xffff0000u);
            }
        }
    } else if constexpr (C == 4) {
        const float4 v = spk_load4<T, true>(p, left);
        r.f[0] = v.x, r.f[1] = v.y, r.f[2] = v.z, r.f[3] = v.w;
    } else if constexpr (sizeof(T) == 2) {
        uint4 v = make_uint4(0u, 0u, 0u, 0u);
        if (left > 0) v = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            r.f[2 * i] = __uint_as_float(w[i] << 16);
            r.f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    } else {
        const float4 u = spk_load4<float, true>(p, left), v = spk_load4<float, true>(p + 4, left);
        r.f[0] = u.x, r.f[1] = u.y, r.f[2] = u.z, r.f[3] = u.w, r.f[4] = v.x, r.f[5] = v.y, r.f[6] = v.z, r.f[7] = v.w;
    }
    return r;
}
template <int C, int VEC, typename T>
__device__ __forceinline__ void store_cols(T* p, const Cols<C>& r, int left) {
    if constexpr (VEC == kSingle) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (nth<VEC>(i) < left) p[nth<VEC>(i)] = spk_from_float<T>(r.f[i]);
    } else if constexpr (VEC == kPairs) {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            if (nth<VEC>(i) >= left) continue;
            if constexpr (sizeof(T) == 4) *reinterpret_cast<float2*>(p + nth<VEC>(i)) = make_float2(r.f[i], r.f[i + 1]);
            else *reinterpret_cast<uint32_t*>(p + nth<VEC>(i)) = pack_bf16(r.f[i], r.f[i + 1]);
        }
    } else if constexpr (C == 4) {
        spk_store4<T, true>(p, make_float4(r.f[0], r.f[1], r.f[2], r.f[3]), left);
    } else if constexpr (sizeof(T) == 2) {
        if (left > 0)
            *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16(r.f[0], r.f[1]), pack_bf16(r.f[2], r.f[3]), pack_bf16(r.f[4], r.f[5]), pack_bf16(r.f[6], r.f[7]));
    } else {
        spk_store4<float, true>(p, make_float4(r.f[0], r.f[1], r.f[2], r.f[3]), left);
        spk_store4<float, true>(p + 4, make_float4(r.f[4], r.f[5], r.f[6], r.f[7]), left);
    }
}
// What the stream keeps of r: as it is in 32 bits, or rounded to bf16, pairs at a time (an element at a time the conversions filled the special-function unit to 29 %).
template <int C, typename T>
__device__ __forceinline__ void round_cols(Cols<C>& r) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < C; i += 2) {
            const uint32_t u = pack_bf16(r.f[i], r.f[i + 1]);
            r.f[i] = __uint_as_float(u << 16);
            r.f[i + 1] = __uint_as_float(u & 0xffff0000u);
        }
    }
}
// First column of a thread's group, of those that begin at multiples of the block's threads.
template <int C, int VEC>
__device__ __forceinline__ int first_col(int thread) {
    return VEC == kWide ? C * thread : (thread >> 5) * 128 + (VEC == kPairs ? 2 : 1) * (thread & 31);
}
// The 8-bit form of a warp's 32 C columns (C = 4: a block; C = 8: two, a half-warp each), this thread's from column c of row t on.  The whole warp calls it.
template <int C, int VEC>
__device__ __forceinline__ void put8(void* q, int64_t q_stride, float* scales, int64_t scale_stride, int64_t t, int c, int width, Cols<C> r) {
    float most = 0.0f;  // fmaxf passes NaN over
#pragma unroll
    for (int i = 0; i < C; ++i) most = fmaxf(most, fabsf(r.f[i]));
    if constexpr (C == 4) {
        most = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(most)));  // magnitudes order like their bits
    } else {
#pragma unroll
        for (int o = 8; o >= 1; o >>= 1) most = fmaxf(most, __shfl_xor_sync(~0u, most, o));
    }
    if (c >= width) return;
    if (most > FLT_MAX) {  // an infinity has no remainder
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (fabsf(r.f[i]) > FLT_MAX) r.f[i] = copysignf(FLT_MAX, r.f[i]);
        most = FLT_MAX;
    }
    const float scale = quotient(fmaxf(most, kLeastBlock), kMostE4m3, 1.0f / kMostE4m3), by = rcp(scale);
    uint8_t* to = static_cast<uint8_t*>(q) + t * q_stride + c;
    const uint32_t lo = pack_e4m3(r.f, scale, by);
    if constexpr (VEC == kSingle) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (c + nth<VEC>(i) < width) to[nth<VEC>(i)] = static_cast<uint8_t>(lo >> (8 * i));
    } else if constexpr (VEC == kPairs) {
#pragma unroll
        for (int i = 0; i < C; i += 2)
            if (c + nth<VEC>(i) < width) *reinterpret_cast<uint16_t*>(to + nth<VEC>(i)) = static_cast<uint16_t>(lo >> (8 * i));
    } else if constexpr (C == 4) {
        *reinterpret_cast<uint32_t*>(to) = lo;
    } else {
        *reinterpret_cast<uint2*>(to) = make_uint2(lo, pack_e4m3(r.f + 4, scale, by));
    }
    if (c % 128 == 0) scales[(c >> 7) * scale_stride + t] = scale;
}

// One CTA per row, C columns a thread and group.  Everything that does not depend on the row's sum is asked for at once.  (V = 8, rows of more than 8192 fp32 or 16384 bf16 columns, keeps the row in the
// registers of up to 1024 threads: 32 or 64 of them, so that 0.5 to 2.6 KB a thread go through local memory.)
template <typename TX, typename TD, int V, int VEC, int MOST>
__global__ void __launch_bounds__(MOST)
boundary8_kernel(const spk_rms_residual_fp8_args p) {
    constexpr int C = VEC == kWide ? 16 / sizeof(TX) : 4;
    constexpr bool AHEAD = V <= 2;
    constexpr int N = AHEAD ? 2 : 1;  // expert rows at a time
    __shared__ float part[32];
    const int64_t t = blockIdx.x;
    const int width = static_cast<int>(p.width);
    auto col = [&](int v) { return first_col<C, VEC>(threadIdx.x + v * blockDim.x); };
    int64_t slot[N] = {};
    float share[N] = {};
    auto ask = [&](int j0) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            slot[j] = j0 + j < p.pair_top ? p.pair_slots[t * p.pair_top + j0 + j] : -1;
            share[j] = j0 + j < p.pair_top ? p.pair_weights[t * p.pair_top + j0 + j] : 0.0f;
        }
    };
    if (p.pairs != nullptr) ask(0);
    Cols<C> y[V], d[V], w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) {
        y[v] = load_cols<C, VEC>(static_cast<const TX*>(p.x) + t * p.width + col(v), width - col(v));
        if (p.delta != nullptr) d[v] = load_cols<C, VEC>(static_cast<const TD*>(p.delta) + t * p.width + col(v), width - col(v));
    }
    if (AHEAD) {
#pragma unroll
        for (int v = 0; v < V; ++v) w[v] = load_cols<C, VEC>(p.w + col(v), width - col(v));
    }
    if (p.delta != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < C; ++i) y[v].f[i] += d[v].f[i];
    }
    if (p.pairs != nullptr) {
        Cols<C> s[V];
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < C; ++i) s[v].f[i] = 0.0f;
        for (int j0 = 0; j0 < p.pair_top; j0 += N) {
            if (j0 > 0) ask(j0);
            Cols<C> f[N][V];
            bool in[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                in[j] = slot[j] >= 0 && slot[j] < p.pair_rows;
                if (slot[j] >= p.pair_rows && threadIdx.x == 0) spk_flag(p.status, SPK_STATUS_BAD_SLOT);
                const float* r = p.pairs + (in[j] ? slot[j] : 0) * p.width;
#pragma unroll
                for (int v = 0; v < V; ++v) f[j][v] = load_cols<C, VEC>(r + col(v), in[j] ? width - col(v) : 0);
            }
#pragma unroll
            for (int j = 0; j < N; ++j) {
                if (!in[j]) continue;  // its weight may be anything
#pragma unroll
                for (int v = 0; v < V; ++v)
#pragma unroll
                    for (int i = 0; i < C; ++i) s[v].f[i] = fmaf(share[j], f[j][v].f[i], s[v].f[i]);
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v)
#pragma unroll
            for (int i = 0; i < C; ++i) y[v].f[i] += s[v].f[i];
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
        round_cols<C, TX>(y[v]);  // the norm of what the next boundary will read
        if (p.x_out != nullptr) store_cols<C, VEC>(static_cast<TX*>(p.x_out) + t * p.width + col(v), y[v], width - col(v));
#pragma unroll
        for (int i = 0; i < C; i += 4)
            q[0] += (y[v].f[i] * y[v].f[i] + y[v].f[i + 1] * y[v].f[i + 1]) + (y[v].f[i + 2] * y[v].f[i + 2] + y[v].f[i + 3] * y[v].f[i + 3]);
    }
    spk_block_sum<1>(q, part);
    const float inv = 1.0f / sqrtf(q[0] / static_cast<float>(width) + p.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = col(v);
        if (!AHEAD) w[v] = load_cols<C, VEC>(p.w + c, width - c);
        Cols<C> f;
#pragma unroll
        for (int i = 0; i < C; ++i) f.f[i] = y[v].f[i] * inv * w[v].f[i];
        if (p.out != nullptr) {
            if (p.out_dtype == SPK_F32) store_cols<C, VEC>(static_cast<float*>(p.out) + t * p.width + c, f, width - c);
            else store_cols<C, VEC>(static_cast<__nv_bfloat16*>(p.out) + t * p.width + c, f, width - c);
        }
        put8<C, VEC>(p.q, p.q_stride, p.scales, p.scale_stride, t, c, width, f);
    }
}

// Prompt batches without expert rows: CTAs go over the rows, whose copies (cp.async.bulk) are kStages ahead; the weight stays in registers.
constexpr int kStages = 3;
template <typename TX, typename TD, int V, int T>
__global__ void __launch_bounds__(T, 768 / T)
boundary8_stream_kernel(const spk_rms_residual_fp8_args p) {
    constexpr int C = 16 / sizeof(TX);
    extern __shared__ __align__(128) uint8_t rows_s[];
    __shared__ float part[32];
    __shared__ uint64_t full[kStages];
    const int width = static_cast<int>(p.width);
    const uint32_t x_bytes = width * sizeof(TX), d_bytes = p.delta != nullptr ? width * sizeof(TD) : 0, stage = x_bytes + d_bytes;
    auto col = [&](int v) { return C * static_cast<int>(threadIdx.x + v * T); };
    auto copy = [&](int s, int64_t t) {  // by thread 0
        const uint32_t bar = smem_u32(&full[s]), dst = smem_u32(rows_s) + s * stage;
        mbar_expect(bar, stage);
        bulk_load(dst, static_cast<const TX*>(p.x) + t * p.width, x_bytes, bar);
        if (d_bytes != 0) bulk_load(dst + x_bytes, static_cast<const TD*>(p.delta) + t * p.width, d_bytes, bar);
    };
    if (threadIdx.x == 0) {
        for (int s = 0; s < kStages; ++s) mbar_init(smem_u32(&full[s]), 1);
        fence_async_shared();
        for (int s = 0; s < kStages; ++s)
            if (blockIdx.x + static_cast<int64_t>(s) * gridDim.x < p.n) copy(s, blockIdx.x + static_cast<int64_t>(s) * gridDim.x);
    }
    Cols<C> w[V];
#pragma unroll
    for (int v = 0; v < V; ++v) w[v] = load_cols<C, kWide>(p.w + col(v), width - col(v));
    __syncthreads();
    int i = 0;
    bool ok = true;
    for (int64_t t = blockIdx.x; t < p.n; t += gridDim.x, ++i) {
        const int s = i % kStages;
        ok = mbar_wait(smem_u32(&full[s]), (i / kStages) & 1) && ok;
        const TX* x = reinterpret_cast<const TX*>(rows_s + s * stage);
        const TD* d = reinterpret_cast<const TD*>(rows_s + s * stage + x_bytes);
        Cols<C> y[V];
        float q[1] = {0.0f};
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = col(v);
            y[v] = load_cols<C, kWide>(x + c, width - c);
            if (d_bytes != 0) {
                const Cols<C> f = load_cols<C, kWide>(d + c, width - c);
#pragma unroll
                for (int k = 0; k < C; ++k) y[v].f[k] += f.f[k];
            }
            round_cols<C, TX>(y[v]);
            if (p.x_out != nullptr) store_cols<C, kWide>(static_cast<TX*>(p.x_out) + t * p.width + c, y[v], width - c);
#pragma unroll
            for (int k = 0; k < C; k += 4)
                q[0] += (y[v].f[k] * y[v].f[k] + y[v].f[k + 1] * y[v].f[k + 1]) + (y[v].f[k + 2] * y[v].f[k + 2] + y[v].f[k + 3] * y[v].f[k + 3]);
        }
        spk_block_sum<1>(q, part);
        // every thread has its columns: the stage is free
        if (threadIdx.x == 0 && t + static_cast<int64_t>(kStages) * gridDim.x < p.n) copy(s, t + static_cast<int64_t>(kStages) * gridDim.x);
        const float inv = 1.0f / sqrtf(q[0] / static_cast<float>(width) + p.eps);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int c = col(v);
            Cols<C> f;
#pragma unroll
            for (int k = 0; k < C; ++k) f.f[k] = y[v].f[k] * inv * w[v].f[k];
            if (p.out != nullptr) {
                if (p.out_dtype == SPK_F32) store_cols<C, kWide>(static_cast<float*>(p.out) + t * p.width + c, f, width - c);
                else store_cols<C, kWide>(static_cast<__nv_bfloat16*>(p.out) + t * p.width + c, f, width - c);
            }
            put8<C, kWide>(p.q, p.q_stride, p.scales, p.scale_stride, t, c, width, f);
        }
    }
    if (!ok && threadIdx.x == 0) spk_flag(p.status, SPK_STATUS_DEVICE_WAIT_EXPIRED);
}

template <typename TX, typename TD, int V, int T>
int launch_stream(const spk_rms_residual_fp8_args& p, int stage, cudaStream_t s) {
    const int bytes = kStages * stage;
    auto kernel = boundary8_stream_kernel<TX, TD, V, T>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    const int fit = 220 * 1024 / (bytes + 1280), ctas = fit < 768 / T ? fit : 768 / T;
    kernel<<<static_cast<unsigned>(p.n < 148 * ctas ? p.n : 148 * ctas), T, bytes, s>>>(p);
    SPK_CHECK_LAUNCH();
    return SPK_OK;
}

// Whether a batch goes to the streaming form, and its launch: no expert rows, enough rows, and 16-bit or narrow ones (8192 rows, the form above / streaming, us: 3584 bf16 104 / 38, 896 bf16
// 16.7 / 12.3, 896 fp32 19.9 / 17.2; 3584 fp32 61 / 72).  Narrow rows have two warps each (one 14.3 and 27.1, four 14.4 and 23.4).
template <typename TX, typename TD>
bool stream_boundary8(const spk_rms_residual_fp8_args& p, cudaStream_t s, int* rc) {
    constexpr int F = sizeof(TX) / 2;
    const int groups = static_cast<int>(p.width * sizeof(TX) / 16), stage = static_cast<int>(p.width * (sizeof(TX) + (p.delta != nullptr ? sizeof(TD) : 0)));
    if (p.pairs != nullptr || p.n < 592 || kStages * stage > 110 * 1024 || groups > (F == 1 ? 1024 : 128 * F)) return false;
    // bulk copies: 16-byte boundaries (16-bit rows beside 32-bit ones of a multiple of four columns may have eight)
    if (p.delta != nullptr && (p.width * sizeof(TD) % 16 != 0 || reinterpret_cast<uintptr_t>(p.delta) % 16 != 0)) return false;
    if (groups <= 128 * F) *rc = launch_stream<TX, TD, 2 * F, 64>(p, stage, s);
    else if constexpr (F == 1) *rc = groups <= 256 ? launch_stream<TX, TD, 1, 256>(p, stage, s) : groups <= 512 ? launch_stream<TX, TD, 2, 256>(p, stage, s) : launch_stream<TX, TD, 4, 256>(p, stage, s);
    return true;
}

template <typename TX, typename TD, int VEC>
int launch_boundary8(const spk_rms_residual_fp8_args& p, cudaStream_t s) {
    constexpr int C = VEC == kWide ? 16 / sizeof(TX) : 4;
    int rc = SPK_OK;
    if constexpr (VEC == kWide)
        if (stream_boundary8<TX, TD>(p, s, &rc)) return rc;
    const unsigned grid = static_cast<unsigned>(p.n);
    // Few rows: many threads each (64 rows of 3584 fp32 with two experts: 4.6 us with 512, 6.6 with 256); many rows hide one another (8192 of them: 123 and 114).
    const int groups = static_cast<int>((p.width + C - 1) / C), most = p.n >= 592 ? 256 : 512;
    int v = 1;
    while (v < 4 && groups > most * v) v *= 2;
    if (groups > 512 * 4) v = 8;
    const int threads = ((groups + v - 1) / v + 31) / 32 * 32;
    if (v == 1) boundary8_kernel<TX, TD, 1, VEC, 512><<<grid, threads, 0, s>>>(p);
    else if (v == 2) boundary8_kernel<TX, TD, 2, VEC, 512><<<grid, threads, 0, s>>>(p);
    else if (v == 4 && threads <= 256) boundary8_kernel<TX, TD, 4, VEC, 256><<<grid, threads, 0, s>>>(p);
    else if (v == 4) boundary8_kernel<TX, TD, 4, VEC, 512><<<grid, threads, 0, s>>>(p);
    else boundary8_kernel<TX, TD, 8, VEC, 1024><<<grid, threads, 0, s>>>(p);
    SPK_CHECK_LAUNCH();
    return SPK_OK;
}

// Approximate exponential and reciprocal (2^-22 each): next to the 2^-4 of the result.  z / 2 (1 + tanh(y)) = z / (1 + exp(-2 y)), y = sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float gelu_tanh(float z) { return z * rcp(1.0f + ex2(-2.302208198f * fmaf(0.044715f * z * z, z, z))); }  // 2 sqrt(2 / pi) log2(e)
__device__ __forceinline__ float silu(float z) { return z * sigmoid_fast(z); }

constexpr int kQuantThreads = 128;  // 256: gate of 8192 x 18944 133 us against 128

// A warp (C = 4) or half-warp (C = 8) takes U blocks of 128 columns that lie one after the other; all of their loads are under way together.
template <typename T, int ACT, int VEC, int U>
__global__ void __launch_bounds__(kQuantThreads)
quantize8_kernel(const spk_quantize_fp8_args p, const uint32_t blocks, const uint32_t per_row) {
    constexpr int C = VEC == kWide ? 16 / sizeof(T) : 4, L = 128 / C;  // threads of a block
    const int width = static_cast<int>(p.width), in = first_col<C, VEC>(threadIdx.x % L);
    const uint32_t b0 = (blockIdx.x * (kQuantThreads / L) + threadIdx.x / L) * U;
    if (b0 - threadIdx.x % 32 / L * U >= blocks) return;  // the whole warp's
    Cols<C> f[U], g[U];
    int64_t t[U];
    int c[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t b = b0 + u < blocks ? b0 + u : blocks - 1;
        t[u] = b / per_row;
        c[u] = static_cast<int>(b % per_row) * 128 + in;
        const T* z = static_cast<const T*>(p.z) + t[u] * p.z_stride + c[u];
        f[u] = load_cols<C, VEC>(z, width - c[u]);
        if (ACT == SPK_ACT_SILU_GATE) g[u] = load_cols<C, VEC>(z + width, width - c[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            if (ACT == SPK_ACT_GELU_TANH) f[u].f[i] = gelu_tanh(f[u].f[i]);
            if (ACT == SPK_ACT_SILU_GATE) f[u].f[i] = silu(f[u].f[i]) * g[u].f[i];
        }
        put8<C, VEC>(p.q, p.q_stride, p.scales, p.scale_stride, t[u], b0 + u < blocks ? c[u] : width, width, f[u]);
    }
}

template <typename T, int ACT>
int launch_quantize8(const spk_quantize_fp8_args& p, cudaStream_t s) {
    const int64_t per_row = (p.width + 127) / 128, blocks = p.n * per_row;
    if (blocks > 0x3fffffffLL) return SPK_ERR_TOO_LARGE;
    auto at = [&](int e) { return p.width % e == 0 && p.z_stride % e == 0 && reinterpret_cast<uintptr_t>(p.z) % (e * sizeof(T)) == 0; };
    constexpr int e = 16 / sizeof(T);
    const bool wide = at(e);
    // One / two / four blocks at a time, us: 37 x 4864 bf16 gelu 1.64 / 1.75 / 2.47, 512 rows 4.1 / 3.7 / 4.6, 8192 rows 39.0 / 34.1 / 33.9; 8192 x 18944 gate 141 / 128 / 122, without activation 100 / 82 / 87.
    constexpr int U4 = ACT != SPK_ACT_NONE && sizeof(T) == 2 ? 4 : 2;
    const int u = blocks < 16384 ? 1 : wide && blocks >= 262144 ? U4 : 2, per = kQuantThreads / (wide ? 128 / e : 32) * u;
    const unsigned grid = static_cast<unsigned>((blocks + per - 1) / per);
    const uint32_t nb = static_cast<uint32_t>(blocks), pr = static_cast<uint32_t>(per_row);
    if (wide && u == 4) quantize8_kernel<T, ACT, kWide, U4><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    else if (wide && u == 2) quantize8_kernel<T, ACT, kWide, 2><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    else if (wide) quantize8_kernel<T, ACT, kWide, 1><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    else if (at(2) && u == 2) quantize8_kernel<T, ACT, kPairs, 2><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    else if (at(2)) quantize8_kernel<T, ACT, kPairs, 1><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    else if (u == 2) quantize8_kernel<T, ACT, kSingle, 2><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    else quantize8_kernel<T, ACT, kSingle, 1><<<grid, kQuantThreads, 0, s>>>(p, nb, pr);
    SPK_CHECK_LAUNCH();
    return SPK_OK;
}

template <typename T>
int launch_quantize8(const spk_quantize_fp8_args& p, cudaStream_t s) {
    if (p.act == SPK_ACT_NONE) return launch_quantize8<T, SPK_ACT_NONE>(p, s);
    if (p.act == SPK_ACT_GELU_TANH) return launch_quantize8<T, SPK_ACT_GELU_TANH>(p, s);
    return launch_quantize8<T, SPK_ACT_SILU_GATE>(p, s);
}

}  // namespace

extern "C" int spk_rms_residual_fp8(const spk_rms_residual_fp8_args* a, void* stream) {
    SpkRange nvtx_range("spk_rms_residual_fp8");
    if (a == nullptr) return SPK_ERR_NULL_POINTER;
    if (a->n < 0 || a->width < 1 || a->width > (1 << 15) || a->scale_stride < a->n) return SPK_ERR_BAD_SHAPE;
    const bool x32 = a->x_dtype == SPK_F32, d32 = a->delta == nullptr ? x32 : a->delta_dtype == SPK_F32;
    if ((!x32 && a->x_dtype != SPK_BF16) || (a->delta != nullptr && !d32 && a->delta_dtype != SPK_BF16) || (!x32 && d32)) return SPK_ERR_BAD_DTYPE;
    if (a->out != nullptr && a->out_dtype != SPK_F32 && a->out_dtype != SPK_BF16) return SPK_ERR_BAD_DTYPE;
    if (a->q_stride < a->width || a->q_stride % 16 != 0 || reinterpret_cast<uintptr_t>(a->q) % 16 != 0) return SPK_ERR_BAD_STRIDE;
    if (a->n == 0) return SPK_OK;
    if (a->n > 0x7fffffffLL) return SPK_ERR_TOO_LARGE;
    if (a->x == nullptr || a->w == nullptr || a->q == nullptr || a->scales == nullptr) return SPK_ERR_NULL_POINTER;
    if (a->pairs != nullptr && (a->pair_slots == nullptr || a->pair_weights == nullptr)) return SPK_ERR_NULL_POINTER;
    if (a->pairs != nullptr && (a->pair_top < 1 || a->pair_rows < 1)) return SPK_ERR_BAD_SHAPE;
    auto at = [](const void* p, size_t b) { return reinterpret_cast<uintptr_t>(p) % b == 0; };
    // e elements of every matrix are read and written at once
    auto all = [&](int64_t e) {
        const size_t xb = e * (x32 ? 4 : 2), db = e * (d32 ? 4 : 2), ob = e * (a->out_dtype == SPK_F32 ? 4 : 2), fb = e * 4;
        auto cap = [](size_t b) { return b < 16 ? b : 16; };
        return a->width % e == 0 && at(a->x, cap(xb)) && at(a->x_out, cap(xb)) && at(a->delta, cap(db)) && at(a->out, cap(ob)) && at(a->w, cap(fb)) && at(a->pairs, cap(fb));
    };
    const int vec = all(x32 ? 4 : 8) ? kWide : all(2) ? kPairs : kSingle;
    cudaStream_t s = spk_stream(stream);
#define SPK_B8(TX, TD) return vec == kWide ? launch_boundary8<TX, TD, kWide>(*a, s) : vec == kPairs ? launch_boundary8<TX, TD, kPairs>(*a, s) : launch_boundary8<TX, TD, kSingle>(*a, s)
    if (!x32) SPK_B8(__nv_bfloat16, __nv_bfloat16);
    if (d32) SPK_B8(float, float);
    SPK_B8(float, __nv_bfloat16);
#undef SPK_B8
}

extern "C" int spk_quantize_fp8(const spk_quantize_fp8_args* a, void* stream) {
    SpkRange nvtx_range("spk_quantize_fp8");
    if (a == nullptr) return SPK_ERR_NULL_POINTER;
    if (a->n < 0 || a->width < 1 || a->width > (1 << 20) || a->scale_stride < a->n) return SPK_ERR_BAD_SHAPE;
    if (a->z_stride < a->width * (a->act == SPK_ACT_SILU_GATE ? 2 : 1)) return SPK_ERR_BAD_STRIDE;
    if (a->q_stride < a->width || a->q_stride % 16 != 0 || reinterpret_cast<uintptr_t>(a->q) % 16 != 0) return SPK_ERR_BAD_STRIDE;
    if (a->dtype != SPK_F32 && a->dtype != SPK_BF16) return SPK_ERR_BAD_DTYPE;
    if (a->act < SPK_ACT_NONE || a->act > SPK_ACT_SILU_GATE) return SPK_ERR_UNSUPPORTED;
    if (a->n == 0) return SPK_OK;
    if (a->z == nullptr || a->q == nullptr || a->scales == nullptr) return SPK_ERR_NULL_POINTER;
    cudaStream_t s = spk_stream(stream);
    return a->dtype == SPK_F32 ? launch_quantize8<float>(*a, s) : launch_quantize8<__nv_bfloat16>(*a, s);
}

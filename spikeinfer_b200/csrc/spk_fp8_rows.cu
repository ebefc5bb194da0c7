// Rows in e4m3 with one scale for every 128 columns: what the products of spk_fp8_linear.cu read.
//
//  * boundary8_kernel: x' = x + delta + the weighted rows of the token's experts, RMS norm of x' as it is stored, and the norm's output in 8 bits.
//  * quantize8_kernel: an activation and the same 8-bit form of its result.
//
// A block of 128 columns is the four-column groups of one warp, so its largest magnitude is one warp reduction away.  scale = most / 448 (448: the
// largest e4m3 value), value = round(v * 448 / most), saturating: NaN stays NaN and is no candidate for the largest, an infinity counts as the
// largest finite value.  A block below 2^-100 is scaled as if its largest magnitude was that, so that no reciprocal overflows.
#include <cuda_fp8.h>
#include <float.h>

#include "spk_dense.cuh"
#include "spk_tensor.cuh"

namespace {

using namespace spk_tc;

constexpr float kMostE4m3 = 448.0f;
constexpr float kLeastBlock = 7.888609052210118e-31f;  // 2^-100

__device__ __forceinline__ float most_of(const float4& f) {  // fmaxf passes NaN over
    return fmaxf(fmaxf(fmaxf(0.0f, fabsf(f.x)), fabsf(f.y)), fmaxf(fabsf(f.z), fabsf(f.w)));
}

// Largest magnitude of the lanes' groups, as a block of 128 columns scales it.  Magnitudes order like their bits.
__device__ __forceinline__ float block_most(float mine) {
    const float m = __uint_as_float(__reduce_max_sync(~0u, __float_as_uint(mine)));
    return fminf(fmaxf(m, kLeastBlock), FLT_MAX);
}

__device__ __forceinline__ uint32_t pack_e4m3(const float4& f, float by) {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f.x * by, f.y * by), __NV_SATFINITE, __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f.z * by, f.w * by), __NV_SATFINITE, __NV_E4M3);
    return lo | hi << 16;
}

// One CTA per row, four columns a thread and group: warp w holds, of group v, the block that starts at column 128 (w + v * warps).
template <typename TX, typename TD, int V, bool VEC>
__global__ void __launch_bounds__(1024)
boundary8_kernel(const spk_rms_residual_fp8_args p) {
    __shared__ float part[32];
    const int64_t t = blockIdx.x;
    const int width = static_cast<int>(p.width);
    auto col = [&](int v) { return 4 * static_cast<int>(threadIdx.x + v * blockDim.x); };
    SpkRow<V> y;
#pragma unroll
    for (int v = 0; v < V; ++v) y.g[v] = spk_load4<TX, VEC>(static_cast<const TX*>(p.x) + t * p.width + col(v), width - col(v));
    if (p.delta != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const float4 f = spk_load4<TD, VEC>(static_cast<const TD*>(p.delta) + t * p.width + col(v), width - col(v));
            y.g[v] = make_float4(y.g[v].x + f.x, y.g[v].y + f.y, y.g[v].z + f.z, y.g[v].w + f.w);
        }
    }
    if (p.pairs != nullptr) {
        SpkRow<V> s;
#pragma unroll
        for (int v = 0; v < V; ++v) s.g[v] = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int j = 0; j < p.pair_top; ++j) {
            const int64_t slot = p.pair_slots[t * p.pair_top + j];
            if (slot < 0) continue;
            if (slot >= p.pair_rows) {
                if (threadIdx.x == 0) spk_flag(p.status, SPK_STATUS_BAD_SLOT);
                continue;
            }
            const float m = p.pair_weights[t * p.pair_top + j];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float4 f = spk_load4<float, VEC>(p.pairs + slot * p.width + col(v), width - col(v));
                s.g[v] = make_float4(fmaf(m, f.x, s.g[v].x), fmaf(m, f.y, s.g[v].y), fmaf(m, f.z, s.g[v].z), fmaf(m, f.w, s.g[v].w));
            }
        }
#pragma unroll
        for (int v = 0; v < V; ++v)
            y.g[v] = make_float4(y.g[v].x + s.g[v].x, y.g[v].y + s.g[v].y, y.g[v].z + s.g[v].z, y.g[v].w + s.g[v].w);
    }
    float q[1] = {0.0f};
#pragma unroll
    for (int v = 0; v < V; ++v) {
        if (sizeof(TX) == 2) {  // the norm of what the next boundary will read
            y.g[v].x = spk_to_float<TX>(spk_from_float<TX>(y.g[v].x));
            y.g[v].y = spk_to_float<TX>(spk_from_float<TX>(y.g[v].y));
            y.g[v].z = spk_to_float<TX>(spk_from_float<TX>(y.g[v].z));
            y.g[v].w = spk_to_float<TX>(spk_from_float<TX>(y.g[v].w));
        }
        if (p.x_out != nullptr) spk_store4<TX, VEC>(static_cast<TX*>(p.x_out) + t * p.width + col(v), y.g[v], width - col(v));
        q[0] += (y.g[v].x * y.g[v].x + y.g[v].y * y.g[v].y) + (y.g[v].z * y.g[v].z + y.g[v].w * y.g[v].w);
    }
    spk_block_sum<1>(q, part);
    const float inv = 1.0f / sqrtf(q[0] / static_cast<float>(width) + p.eps);
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const int c = col(v);
        const float4 w = spk_load4<float, VEC>(p.w + c, width - c);
        const float4 f = make_float4(y.g[v].x * inv * w.x, y.g[v].y * inv * w.y, y.g[v].z * inv * w.z, y.g[v].w * inv * w.w);
        if (p.out != nullptr) {
            if (p.out_dtype == SPK_F32) spk_store4<float, VEC>(static_cast<float*>(p.out) + t * p.width + c, f, width - c);
            else spk_store4<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p.out) + t * p.width + c, f, width - c);
        }
        const float most = block_most(most_of(f));
        if (c < width) {
            *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.q) + t * p.q_stride + c) = pack_e4m3(f, kMostE4m3 / most);
            if ((threadIdx.x & 31) == 0) p.scales[(c >> 7) * p.scale_stride + t] = most / kMostE4m3;
        }
    }
}

template <typename TX, typename TD>
int launch_boundary8(const spk_rms_residual_fp8_args& p, bool vec, cudaStream_t s) {
    int v = 1;
    const int threads = spk_row_shape(p.width, &v);
    if (threads == 0) return SPK_ERR_TOO_LARGE;
    const unsigned grid = static_cast<unsigned>(p.n);
#define SPK_B8(V_)                                                                     \
    do {                                                                               \
        if (vec) boundary8_kernel<TX, TD, V_, true><<<grid, threads, 0, s>>>(p);       \
        else boundary8_kernel<TX, TD, V_, false><<<grid, threads, 0, s>>>(p);          \
    } while (0)
    if (v == 1) SPK_B8(1);
    else if (v == 2) SPK_B8(2);
    else if (v == 4) SPK_B8(4);
    else SPK_B8(8);
#undef SPK_B8
    SPK_CHECK_LAUNCH();
    return SPK_OK;
}

// z / 2 (1 + tanh(y)) = z / (1 + exp(-2 y)), y = sqrt(2 / pi) (z + 0.044715 z^3)
__device__ __forceinline__ float gelu_tanh(float z) { return z / (1.0f + expf(-1.5957691216057308f * fmaf(0.044715f * z * z, z, z))); }

constexpr int kQuantWarps = 8;

// A warp per block of 128 columns.
template <typename T, int ACT, bool VEC>
__global__ void __launch_bounds__(kQuantWarps * 32)
quantize8_kernel(const spk_quantize_fp8_args p, const int64_t blocks, const int per_row) {
    const int64_t b = static_cast<int64_t>(blockIdx.x) * kQuantWarps + (threadIdx.x >> 5);
    if (b >= blocks) return;
    const int64_t t = b / per_row;
    const int k = static_cast<int>(b % per_row), width = static_cast<int>(p.width);
    const int c = k * 128 + 4 * (threadIdx.x & 31);
    const T* z = static_cast<const T*>(p.z) + t * p.z_stride + c;
    float4 f = spk_load4<T, VEC>(z, width - c);
    if (ACT == SPK_ACT_GELU_TANH) f = make_float4(gelu_tanh(f.x), gelu_tanh(f.y), gelu_tanh(f.z), gelu_tanh(f.w));
    if (ACT == SPK_ACT_SILU_GATE) {
        const float4 u = spk_load4<T, VEC>(z + width, width - c);
        f = make_float4(spk_silu(f.x) * u.x, spk_silu(f.y) * u.y, spk_silu(f.z) * u.z, spk_silu(f.w) * u.w);
    }
    const float most = block_most(most_of(f));
    if (c < width) *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(p.q) + t * p.q_stride + c) = pack_e4m3(f, kMostE4m3 / most);
    if ((threadIdx.x & 31) == 0) p.scales[k * p.scale_stride + t] = most / kMostE4m3;
}

template <typename T, int ACT>
int launch_quantize8(const spk_quantize_fp8_args& p, cudaStream_t s) {
    const int per_row = static_cast<int>((p.width + 127) / 128);
    const int64_t blocks = p.n * per_row, grid = (blocks + kQuantWarps - 1) / kQuantWarps;
    if (grid > 0x7fffffffLL) return SPK_ERR_TOO_LARGE;
    const bool vec = p.width % 4 == 0 && p.z_stride % 4 == 0 && reinterpret_cast<uintptr_t>(p.z) % (4 * sizeof(T)) == 0;
    if (vec) quantize8_kernel<T, ACT, true><<<static_cast<unsigned>(grid), kQuantWarps * 32, 0, s>>>(p, blocks, per_row);
    else quantize8_kernel<T, ACT, false><<<static_cast<unsigned>(grid), kQuantWarps * 32, 0, s>>>(p, blocks, per_row);
    SPK_CHECK_LAUNCH();
    return SPK_OK;
}

template <typename T>
int launch_quantize8(const spk_quantize_fp8_args& p, cudaStream_t s) {
    if (p.act == SPK_ACT_NONE) return launch_quantize8<T, SPK_ACT_NONE>(p, s);
    if (p.act == SPK_ACT_GELU_TANH) return launch_quantize8<T, SPK_ACT_GELU_TANH>(p, s);
    if (p.act == SPK_ACT_SILU_GATE) return launch_quantize8<T, SPK_ACT_SILU_GATE>(p, s);
    return SPK_ERR_UNSUPPORTED;
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
    const size_t xb = x32 ? 16 : 8, db = d32 ? 16 : 8, ob = a->out_dtype == SPK_F32 ? 16 : 8;
    const bool vec = a->width % 4 == 0 && at(a->x, xb) && at(a->x_out, xb) && at(a->delta, db) && at(a->w, 16) && at(a->pairs, 16) && at(a->out, ob);
    cudaStream_t s = spk_stream(stream);
    if (!x32) return launch_boundary8<__nv_bfloat16, __nv_bfloat16>(*a, vec, s);
    return d32 ? launch_boundary8<float, float>(*a, vec, s) : launch_boundary8<float, __nv_bfloat16>(*a, vec, s);
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

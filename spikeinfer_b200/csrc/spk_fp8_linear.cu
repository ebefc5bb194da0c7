// Products of e4m3 rows with e4m3 weights on the fifth-generation tensor cores (tcgen05, kind::f8f6f4).
//
// A block of 128 columns has one scale per row of x and one per 128 features, so its sum of products (32-bit, in TMEM) is multiplied by both and added to
// the result in registers: the accumulator of a block is a TMEM buffer of its own, read while the next block's MMAs run into another.
//
// fp8_rows_kernel: CTA = (128 features, run of TN tokens, part of k).  The weights are the M operand, the tokens the N operand: a few decoded tokens cost a
// narrow MMA.  Warp 0 copies (TMA, rows beyond the end and columns beyond k read zero), warp 1 issues MMAs, four warps have a feature per lane.  Where few
// CTAs would stream the weights, a cluster of S shares the blocks of k; the parts meet in shared memory and are added in the order of the CTAs.
#include <cuda.h>

#include "spk_dense.cuh"
#include "spk_tensor.cuh"

namespace {

using namespace spk_tc;

constexpr int kBlock = 128;              // columns with a scale, and bytes of a tile's row
constexpr int kTileW = kBlock * kBlock;  // bytes of a weight tile: 128 features
constexpr int kThreads = 192;

template <int TN>
struct Shape {
    static constexpr int kStage = kTileW + TN * kBlock;
    static constexpr int NS = TN >= 128 ? 6 : TN >= 64 ? 8 : 10;
    static constexpr int NB = 4;  // accumulators
    static constexpr int kColumns = NB * TN;
    static constexpr int kScales = 2 * TN * 4;
    static constexpr int kBytes = 1024 + NS * kStage + kScales + 512;
};

struct Bars {
    uint64_t full[10], free[10], sums[4], drained[4], done;
    int abort;
    uint32_t tmem;
};

// kind::f8f6f4 instruction descriptor: e4m3 operands, contiguous along k, fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1 : 0) : "memory");
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// What CTA `rank` of the cluster has where this CTA has `addr`.
__device__ __forceinline__ float cluster_load(uint32_t addr, uint32_t rank) {
    float v;
    asm volatile("{\n\t.reg .b32 r;\n\tmapa.shared::cluster.u32 r, %1, %2;\n\tld.shared::cluster.f32 %0, [r];\n\t}\n" : "=f"(v) : "r"(addr), "r"(rank) : "memory");
    return v;
}

__device__ __forceinline__ void put(const spk_linear_fp8_args& a, int64_t t, int64_t f, float v) {
    if (a.out_dtype == SPK_F32) static_cast<float*>(a.out)[t * a.out_stride + f] = v;
    else static_cast<__nv_bfloat16*>(a.out)[t * a.out_stride + f] = __float2bfloat16_rn(v);
}

template <int TN, int S>
__global__ void __launch_bounds__(kThreads, 1)
fp8_rows_kernel(const spk_linear_fp8_args a, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const int blocks) {
    using Sh = Shape<TN>;
    constexpr int NS = Sh::NS, NB = Sh::NB;
    static_assert(S == 1 || TN * 128 * 4 <= NS * Sh::kStage, "partial sums take the stages' place");
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float* scales = reinterpret_cast<float*>(base + NS * Sh::kStage);  // [2][TN]
    Bars* bars = reinterpret_cast<Bars*>(base + NS * Sh::kStage + Sh::kScales);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = static_cast<int>(blockIdx.x) % S;
    const int fb = blockIdx.x / S;                                              // block of 128 features
    const int64_t t0 = static_cast<int64_t>(blockIdx.y) * TN;
    const int kb = blocks * part / S, kn = blocks * (part + 1) / S - kb;        // this CTA's blocks of k, at least one
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_u32(&bars->full[i]), 1);
            mbar_init(smem_u32(&bars->free[i]), 1);
        }
        for (int i = 0; i < NB; ++i) {
            mbar_init(smem_u32(&bars->sums[i]), 1);
            mbar_init(smem_u32(&bars->drained[i]), 128);
        }
        mbar_init(smem_u32(&bars->done), 1);
        bars->abort = 0;
    }
    if (warp == 0) tmem_alloc(smem_u32(&bars->tmem), Sh::kColumns);
    fence_async_shared();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = bars->tmem;
    volatile int* abort = &bars->abort;
    if (warp == 0) {
        if (lane == 0) {
            int issued = 0;
            for (int k = 0; k < kn; ++k) {
                const int s = k % NS;
                if (k >= NS && !mbar_wait(smem_u32(&bars->free[s]), ((k / NS) - 1) & 1, abort)) break;
                const uint32_t bar = smem_u32(&bars->full[s]), dst = smem_u32(base + s * Sh::kStage);
                mbar_expect(bar, Sh::kStage);
                tma_load(dst, &w_map, (kb + k) * kBlock, fb * 128, bar);
                tma_load(dst + kTileW, &x_map, (kb + k) * kBlock, static_cast<int>(t0), bar);
                issued = k + 1;
            }
            if (*abort != 0)  // copies in flight land before the CTA's shared memory is given up
                for (int k = issued > NS ? issued - NS : 0; k < issued; ++k) mbar_wait(smem_u32(&bars->full[k % NS]), (k / NS) & 1);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            constexpr uint32_t idesc = idesc_e4m3(128, TN);
            for (int k = 0; k < kn; ++k) {
                const int s = k % NS, b = k % NB;
                if (k >= NB && !mbar_wait(smem_u32(&bars->drained[b]), ((k / NB) - 1) & 1, abort)) break;
                if (!mbar_wait(smem_u32(&bars->full[s]), (k / NS) & 1, abort)) break;
                tc_fence_after();
                const uint32_t wa = smem_u32(base + s * Sh::kStage), xa = wa + kTileW;
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    mma_e4m3(tmem + b * TN, desc_sw128(wa + i * 32, 16, 1024), desc_sw128(xa + i * 32, 16, 1024), idesc, i > 0);
                mma_commit(smem_u32(&bars->free[s]));
                mma_commit(smem_u32(&bars->sums[b]));
            }
            mma_commit(smem_u32(&bars->done));
            mbar_wait(smem_u32(&bars->done), 0);  // nothing this thread issued is in the tensor pipe any more
        }
    } else {
        const int quad = warp & 3, e = threadIdx.x - 64;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const bool has = e < TN && t0 + e < a.n;  // this thread brings the scale of token e
        const float* xs = a.x_scales + t0 + e;
        const float* ws = a.w_scales + static_cast<int64_t>(fb) * a.w_scale_stride;
        float acc[TN];
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[j] = 0.0f;
        bool ok = true;
        float next = has ? xs[kb * a.x_scale_stride] * ws[kb] : 0.0f;
        for (int k = 0; k < kn; ++k) {
            const int b = k % NB;
            float* sc = scales + (k & 1) * TN;
            if (e < TN) sc[e] = next;
            asm volatile("bar.sync 1, 128;" ::: "memory");  // a block's factors are written when those of the one before last have been used
            next = has && k + 1 < kn ? xs[(kb + k + 1) * a.x_scale_stride] * ws[kb + k + 1] : 0.0f;
            if (ok) ok = __all_sync(~0u, mbar_wait(smem_u32(&bars->sums[b]), (k / NB) & 1, abort));
            if (!ok) continue;  // keeps the barriers
            tc_fence_after();
#pragma unroll
            for (int j0 = 0; j0 < TN; j0 += 16) {
                uint32_t r[16];
                tmem_ld16(tmem + lanes + b * TN + j0, r);
#pragma unroll
                for (int j = 0; j < 16; ++j) acc[j0 + j] = fmaf(__uint_as_float(r[j]), sc[j0 + j], acc[j0 + j]);
            }
            tc_fence_before();
            mbar_arrive(smem_u32(&bars->drained[b]));
        }
        const int64_t f = static_cast<int64_t>(fb) * 128 + quad * 32 + lane;
        if (S == 1) {
#pragma unroll
            for (int j = 0; j < TN; ++j)
                if (ok && t0 + j < a.n && f < a.features) put(a, t0 + j, f, acc[j]);
        } else {
            float* sums = reinterpret_cast<float*>(base) + quad * 32 + lane;
#pragma unroll
            for (int j = 0; j < TN; ++j) sums[j * 128] = ok ? acc[j] : 0.0f;
        }
    }
    if (S > 1) {
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2) {  // every CTA adds and writes its own tokens
            constexpr int J = TN / S;
            const int quad = warp & 3;
            const uint32_t own = smem_u32(base) + 4 * (part * J * 128 + quad * 32 + lane);
            const int64_t f = static_cast<int64_t>(fb) * 128 + quad * 32 + lane;
            for (int j = 0; j < J && t0 + part * J + j < a.n; ++j) {
                float v = 0.0f;
#pragma unroll
                for (int r = 0; r < S; ++r) v += cluster_load(own + j * 512, r);
                if (f < a.features) put(a, t0 + part * J + j, f, v);
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();  // no CTA leaves while its sums are being read
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && *abort != 0) spk_flag(a.status, SPK_STATUS_DEVICE_WAIT_EXPIRED);
    if (warp == 0) tmem_dealloc(tmem, Sh::kColumns);
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*,
                                CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encoder() {
    static EncodeTiled fn = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiled>(p);
    }();
    return fn;
}

// [rows][columns] bytes, boxes of box_rows x 128 bytes, 128-byte swizzle; rows and columns beyond the end read zero.
bool encode(CUtensorMap* map, const void* p, int64_t rows, int64_t columns, int64_t row_stride, int box_rows) {
    const EncodeTiled fn = encoder();
    if (fn == nullptr) return false;
    const cuuint64_t size[2] = {static_cast<cuuint64_t>(columns), static_cast<cuuint64_t>(rows)}, stride[1] = {static_cast<cuuint64_t>(row_stride)};
    const cuuint32_t box[2] = {kBlock, static_cast<cuuint32_t>(box_rows)}, unit[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(p), size, stride, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int TN, int S>
int launch_rows(const spk_linear_fp8_args& a, cudaStream_t s) {
    constexpr int bytes = Shape<TN>::kBytes;
    static_assert(sizeof(Bars) <= 512 && bytes <= 227 * 1024, "shared memory");
    CUtensorMap w_map, x_map;
    if (!encode(&w_map, a.w, a.features, a.k, a.w_stride, 128) || !encode(&x_map, a.x, a.n, a.k, a.x_stride, TN)) return SPK_ERR_UNSUPPORTED;
    const int blocks = static_cast<int>((a.k + kBlock - 1) / kBlock);
    const int64_t fblocks = (a.features + 127) / 128, runs = (a.n + TN - 1) / TN;
    if (fblocks * S > 0x7fffffff || runs > 65535) return SPK_ERR_TOO_LARGE;
    auto kernel = fp8_rows_kernel<TN, S>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {};
    cfg.gridDim = dim3(static_cast<unsigned>(fblocks * S), static_cast<unsigned>(runs));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    cfg.attrs = attr;
    if (S > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {S, 1, 1};
        cfg.numAttrs = 1;
    }
    e = cudaLaunchKernelEx(&cfg, kernel, a, w_map, x_map, blocks);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    spk_count_launch();
    return SPK_OK;
}

template <int TN>
int dispatch(const spk_linear_fp8_args& a, cudaStream_t s) {
    const int64_t ctas = (a.features + 127) / 128 * ((a.n + TN - 1) / TN), blocks = (a.k + kBlock - 1) / kBlock;
    if (ctas * 2 <= 148 && blocks >= 4) return launch_rows<TN, 4>(a, s);
    if (ctas <= 148 && blocks >= 2) return launch_rows<TN, 2>(a, s);
    return launch_rows<TN, 1>(a, s);
}

}  // namespace

extern "C" int spk_linear_fp8(const spk_linear_fp8_args* args, void* stream) {
    SpkRange nvtx_range("spk_linear_fp8");
    if (args == nullptr) return SPK_ERR_NULL_POINTER;
    const spk_linear_fp8_args& a = *args;
    if (a.n < 0 || a.k < 1 || a.features < 1) return SPK_ERR_BAD_SHAPE;
    const int64_t blocks = (a.k + kBlock - 1) / kBlock;
    if (a.x_stride < a.k || a.w_stride < a.k || a.x_stride % 16 != 0 || a.w_stride % 16 != 0 || reinterpret_cast<uintptr_t>(a.x) % 16 != 0 ||
        reinterpret_cast<uintptr_t>(a.w) % 16 != 0 || a.x_scale_stride < a.n || a.w_scale_stride < blocks || a.out_stride < a.features)
        return SPK_ERR_BAD_STRIDE;
    if (a.out_dtype != SPK_F32 && a.out_dtype != SPK_BF16) return SPK_ERR_BAD_DTYPE;
    if (a.n == 0) return SPK_OK;
    if (a.n > 0x7fffff00LL || a.features > 0x7fffff00LL || a.k > 0x7fffff00LL || a.x_stride >= 1LL << 40 || a.w_stride >= 1LL << 40) return SPK_ERR_TOO_LARGE;
    if (a.x == nullptr || a.w == nullptr || a.x_scales == nullptr || a.w_scales == nullptr || a.out == nullptr) return SPK_ERR_NULL_POINTER;
    cudaStream_t s = spk_stream(stream);
    if (a.n <= 16) return dispatch<16>(a, s);
    if (a.n <= 32) return dispatch<32>(a, s);
    if (a.n <= 64) return dispatch<64>(a, s);
    return dispatch<128>(a, s);
}

// Products of e4m3 rows with e4m3 weights on the fifth-generation tensor cores (tcgen05, kind::f8f6f4).
//
// A block of 128 columns has one scale per row of x and one per 128 features, so its sum of products (32-bit, in TMEM) is multiplied by both and added to
// the result in registers: the accumulator of a block is a TMEM buffer of its own, read while the next block's MMAs run into another.
//
// fp8_rows_kernel (up to 64 rows): CTA = (128 features, all rows, part of k).  The weights are the M operand, the tokens the N operand: a few decoded tokens cost a
// narrow MMA and every lane of the accumulators is a feature.  Where few CTAs would stream the weights, a cluster of S shares the blocks of k; the parts meet in shared
// memory and are added in the order of the CTAs.  64 x 3584 x 18944: 17.7 us, 3.8 TB/s of weights (0.61 of the copy rate; set-up and drain are 4 us of it).
// fp8_tiles_kernel (more rows): the tokens are the M operand, below.  8192 x 3584 x 18944: 564 us, 1.97 PFLOP/s (1.18 of the library's measured bf16 rate; up to 600 where the GPU has been at its power
// limit before).
//
// What bounds the large products: two lanes of work of nearly the same length.  With parts taken out in turn, the MMAs alone (copies, barriers) were 480 us, everything but the MMAs (sums read from
// tensor memory, scaled, added, stored) 455, both 570.  480 is half the nominal e4m3 rate; why is not known.  A block of 128 x 256 is 512 cycles of MMAs at the nominal rate, its sums are read, scaled
// and added in some 500 cycles by eight warps, and with two accumulators the way from the last MMA through the writers to the next MMA into the same columns counts as well (some 1150 cycles a block).
// Scales that are powers of two for 32 columns could stay in the MMA; these are 32-bit and for 128.
// Steps on the way, us before / after for 8192 x 3584 x 18944: one accumulating warpgroup per feature block 1680; barriers for every block's scales / for eight blocks 703 / 600; products of pairs
// (fma.rn.f32x2) / one by one 656 / 606; an arrival with cluster scope on the pair's barrier / without 1240 / 640; 16 writing warps / eight 606 / 600.
#include <cuda.h>
#include <cuda_fp8.h>
#include <float.h>

#include "spk_dense.cuh"
#include "spk_tensor.cuh"

namespace {

using namespace spk_tc;

constexpr int kBlock = 128;              // columns with a scale, and bytes of a tile's row
constexpr int kTileW = kBlock * kBlock;  // bytes of a weight tile: 128 features
constexpr int kGroup = 8;                // tiles: blocks of k whose scales come together
constexpr int kGroups = 4;               // of those in the ring

// Few rows: blocks of k come in groups of kRun, each with accumulators of its own and one barrier for the group (1.3 us a block of 64 tokens with one each).
constexpr int kRun = 4;
template <int TN>
struct Shape {
    static constexpr int kStage = kTileW + TN * kBlock;
    static constexpr int NS = TN >= 64 ? 8 : 10;
    static constexpr int NB = 512 / (kRun * TN) > 4 ? 4 : 512 / (kRun * TN);  // groups with accumulators
    static constexpr int kColumns = NB * kRun * TN;
    static constexpr int kRing = 8;  // groups with factors
    static constexpr int kFactors = kRing * kRun * TN * 4;
    static constexpr int kBytes = 1024 + NS * kStage + kFactors + 1024;
    static constexpr int kWriters = TN >= 64 ? 8 : 4;
    static constexpr int kThreads = 128 + 32 * kWriters;
};

struct Bars {
    uint64_t full[10], free[10], sums[4], drained[4], factors[8], used[8], done;
    int abort;
    uint32_t tmem;
    int odd;  // rows: a token may be far
};

// kind::f8f6f4 instruction descriptor: e4m3 operands, contiguous along k, fp32 accumulator.
__host__ __device__ constexpr uint32_t idesc_e4m3(int m, int n) { return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24); }

// Issued by the lane whose `who` is set.  CG = 2: by the even CTA of a pair for both.
template <int CG>
__device__ __forceinline__ void mma_e4m3_by(uint32_t who, uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool acc) {
    if (CG == 1)
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1 : 0), "r"(who) : "memory");
    else
        asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                     "@q tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}\n"
                     ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc ? 1 : 0), "r"(who) : "memory");
}
// Arrives on `bar` (CG = 2: of both CTAs) when every MMA that lane has issued so far is complete.
template <int CG>
__device__ __forceinline__ void commit_by(uint32_t who, uint32_t bar) {
    if (CG == 1)
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n"
                     ::"r"(bar), "r"(who) : "memory");
    else
        asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %2;\n\t}\n"
                     ::"r"(bar), "r"(who), "h"(static_cast<uint16_t>(3)) : "memory");
}

__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}

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

// A block's sum is multiplied by the product of its scales.  Where that is beyond the 32-bit numbers while both scales are not (1e20 times 1e20, beside a sum of zero too), what a thread has
// added up is put aside, and its outputs are summed up here from the operands, up to 500 times as slow: a sum times the smaller scale, times the larger one, so that nothing on the way
// overflows unless the term does.  (A branch for every block in the loops that read tensor memory took 2 to 12 % of all products.)  A product below the normal numbers is taken as it is, to
// within 2^-150: scales of 2^-100 / 448, those of blocks of zeros, are met beside small ones.
__device__ __forceinline__ bool is_far(float x, float w) { return fabsf(x * w) == INFINITY && fabsf(x) <= FLT_MAX && fabsf(w) <= FLT_MAX; }
__device__ __forceinline__ bool may_be_far(float product) { return !(fabsf(product) <= FLT_MAX); }  // or one of the scales is not finite
__device__ __noinline__ bool has_far(const spk_linear_fp8_args& a, int64_t t, int64_t f, int kb, int kn) {
    if (t >= a.n || f >= a.features) return false;
    bool far = false;
    for (int b = kb; b < kb + kn && !far; ++b) far = is_far(a.x_scales[b * a.x_scale_stride + t], a.w_scales[f / kBlock * a.w_scale_stride + b]);
    return far;
}
__device__ __noinline__ float far_sum(const spk_linear_fp8_args& a, int64_t t, int64_t f, int kb, int kn) {
    if (t >= a.n || f >= a.features) return 0.0f;
    const uint8_t *x = static_cast<const uint8_t*>(a.x) + t * a.x_stride, *w = static_cast<const uint8_t*>(a.w) + f * a.w_stride;
    auto two = [](uint32_t v) { return __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(v), __NV_E4M3))); };
    float y = 0.0f;
    for (int b = kb; b < kb + kn; ++b) {
        const int64_t c0 = static_cast<int64_t>(b) * kBlock, c1 = min(c0 + kBlock, a.k);
        float s = 0.0f;
        int64_t c = c0;
        for (; c + 16 <= c1; c += 16) {
            const uint4 u = *reinterpret_cast<const uint4*>(x + c), v = *reinterpret_cast<const uint4*>(w + c);
            const uint32_t p[4] = {u.x, u.y, u.z, u.w}, q[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 e = two(p[i / 2] >> (i % 2 * 16) & 0xffffu), g = two(q[i / 2] >> (i % 2 * 16) & 0xffffu);
                s = fmaf(e.x, g.x, s);
                s = fmaf(e.y, g.y, s);
            }
        }
        for (; c < c1; ++c) s = fmaf(two(x[c]).x, two(w[c]).x, s);
        const float sx = a.x_scales[b * a.x_scale_stride + t], sw = a.w_scales[f / kBlock * a.w_scale_stride + b], m = sx * sw;
        const bool x_first = fabsf(sx) < fabsf(sw);
        y = is_far(sx, sw) ? fmaf(s * (x_first ? sx : sw), x_first ? sw : sx, y) : fmaf(s, m, y);
    }
    return y;
}

template <int TN, int S>
__global__ void __launch_bounds__(Shape<TN>::kThreads, 1)
fp8_rows_kernel(const __grid_constant__ spk_linear_fp8_args a, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const int blocks) {
    using Sh = Shape<TN>;
    constexpr int NS = Sh::NS, NB = Sh::NB;
    static_assert(S == 1 || TN * 128 * 4 <= NS * Sh::kStage, "partial sums take the stages' place");
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    float* ring = reinterpret_cast<float*>(base + NS * Sh::kStage);  // [kRing][kRun][TN]: scale of the token times scale of the features
    Bars* bars = reinterpret_cast<Bars*>(base + NS * Sh::kStage + Sh::kFactors);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = static_cast<int>(blockIdx.x) % S;
    const int fb = blockIdx.x / S;                                        // block of 128 features
    const int kb = blocks * part / S, kn = blocks * (part + 1) / S - kb;  // this CTA's blocks of k, at least one
    const int groups = (kn + kRun - 1) / kRun;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_u32(&bars->full[i]), 1);
            mbar_init(smem_u32(&bars->free[i]), 1);
        }
        for (int i = 0; i < NB; ++i) {
            mbar_init(smem_u32(&bars->sums[i]), 1);
            mbar_init(smem_u32(&bars->drained[i]), Sh::kWriters);
        }
        for (int i = 0; i < Sh::kRing; ++i) {
            mbar_init(smem_u32(&bars->factors[i]), 32);
            mbar_init(smem_u32(&bars->used[i]), Sh::kWriters);
        }
        mbar_init(smem_u32(&bars->done), 1);
        bars->abort = bars->odd = 0;
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
                tma_load(dst + kTileW, &x_map, (kb + k) * kBlock, 0, bar);
                issued = k + 1;
            }
            if (*abort != 0)  // copies in flight land before the CTA's shared memory is given up
                for (int k = issued > NS ? issued - NS : 0; k < issued; ++k) mbar_wait(smem_u32(&bars->full[k % NS]), (k / NS) & 1);
        }
    } else if (warp == 1) {
        constexpr uint32_t idesc = idesc_e4m3(128, TN);
        const uint32_t who = elect_one();
        bool go = true;
        for (int k = 0; k < kn; ++k) {
            const int s = k % NS, g = k / kRun, b = g % NB;
            go = __all_sync(~0u, (k % kRun != 0 || g < NB || mbar_wait(smem_u32(&bars->drained[b]), ((g / NB) - 1) & 1, abort)) &&
                                     mbar_wait(smem_u32(&bars->full[s]), (k / NS) & 1, abort));
            if (!go) break;
            tc_fence_after();
            const uint32_t wa = smem_u32(base + s * Sh::kStage), xa = wa + kTileW;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                mma_e4m3_by<1>(who, tmem + (b * kRun + k % kRun) * TN, desc_sw128(wa + i * 32, 16, 1024), desc_sw128(xa + i * 32, 16, 1024), idesc, i > 0);
            commit_by<1>(who, smem_u32(&bars->free[s]));
            if (k % kRun == kRun - 1 || k + 1 == kn) commit_by<1>(who, smem_u32(&bars->sums[b]));
        }
        commit_by<1>(who, smem_u32(&bars->done));
        mbar_wait(smem_u32(&bars->done), 0);  // nothing this warp issued is in the tensor pipe any more
    } else if (warp < 4) {  // scales: two warps take a group in turn, whose loads are under way together
        constexpr int R = (TN + 31) / 32;
        const float* w = a.w_scales + fb * a.w_scale_stride + kb;
        for (int g = warp - 2; g < groups; g += 2) {
            const int at = g % Sh::kRing;
            float u[kRun][R], v[kRun];
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                const int k = g * kRun + i;
                const float* x = a.x_scales + (kb + k) * a.x_scale_stride;
                v[i] = k < kn ? w[k] : 0.0f;
#pragma unroll
                for (int j = 0; j < R; ++j) u[i][j] = k < kn && 32 * j + lane < TN && 32 * j + lane < a.n ? x[32 * j + lane] : 0.0f;
            }
            if (g >= Sh::kRing && !__all_sync(~0u, mbar_wait(smem_u32(&bars->used[at]), ((g / Sh::kRing) - 1) & 1, abort))) break;
#pragma unroll
            for (int i = 0; i < kRun; ++i)
#pragma unroll
                for (int j = 0; j < R; ++j) {
                    const float m = u[i][j] * v[i];
                    if (may_be_far(m)) bars->odd = 1;
                    if (32 * j + lane < TN) ring[(at * kRun + i) * TN + 32 * j + lane] = m;
                }
            mbar_arrive(smem_u32(&bars->factors[at]));
        }
    } else {  // a feature per lane, 32 tokens (or all 16) per warp
        constexpr int C = TN < 32 ? TN : 32;
        const int quad = warp & 3, j0 = (warp - 4) / 4 * C;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        float acc[C];
#pragma unroll
        for (int j = 0; j < C; ++j) acc[j] = 0.0f;
        bool ok = true;
        for (int g = 0; g < groups; ++g) {
            const int b = g % NB, at = g % Sh::kRing;
            ok = __all_sync(~0u, mbar_wait(smem_u32(&bars->factors[at]), (g / Sh::kRing) & 1, abort) && mbar_wait(smem_u32(&bars->sums[b]), (g / NB) & 1, abort));
            if (!ok) break;
            tc_fence_after();
            const uint32_t from = tmem + lanes + b * kRun * TN + j0;
            const int in = kn - g * kRun;  // blocks left
            uint32_t r[2][C];
            auto load = [&](int i) {
                if constexpr (C == 32) tmem_ld32(from + i * TN, r[i & 1]);
                else tmem_ld16(from + i * TN, r[i & 1]);
            };
            load(0);
#pragma unroll
            for (int i = 0; i < kRun; ++i) {
                if (i >= in) break;
                if constexpr (C == 32) tmem_wait_ld(r[i & 1]);
                if (i + 1 < kRun && i + 1 < in) load((i + 1) & 3);
                const float4* m = reinterpret_cast<const float4*>(ring + (at * kRun + i) * TN + j0);
#pragma unroll
                for (int j = 0; j < C; j += 4) {
                    const float4 f = m[j / 4];
                    acc[j] = fmaf(__uint_as_float(r[i & 1][j]), f.x, acc[j]);
                    acc[j + 1] = fmaf(__uint_as_float(r[i & 1][j + 1]), f.y, acc[j + 1]);
                    acc[j + 2] = fmaf(__uint_as_float(r[i & 1][j + 2]), f.z, acc[j + 2]);
                    acc[j + 3] = fmaf(__uint_as_float(r[i & 1][j + 3]), f.w, acc[j + 3]);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(smem_u32(&bars->drained[b]));
                mbar_arrive(smem_u32(&bars->used[at]));
            }
        }
        const int64_t f = static_cast<int64_t>(fb) * 128 + quad * 32 + lane;
        if (S == 1) {
#pragma unroll
            for (int j = 0; j < C; ++j)
                if (ok && j0 + j < a.n && f < a.features) put(a, j0 + j, f, acc[j]);
            if (ok && bars->odd != 0)
                for (int j = 0; j < C; ++j)
                    if (has_far(a, j0 + j, f, kb, kn)) put(a, j0 + j, f, far_sum(a, j0 + j, f, kb, kn));
        } else {  // [token][128 features]
            float* sums = reinterpret_cast<float*>(base) + j0 * 128 + quad * 32 + lane;
#pragma unroll
            for (int j = 0; j < C; ++j) sums[j * 128] = ok ? acc[j] : 0.0f;
            if (ok && bars->odd != 0)
                for (int j = 0; j < C; ++j)
                    if (has_far(a, j0 + j, f, kb, kn)) sums[j * 128] = far_sum(a, j0 + j, f, kb, kn);
        }
    }
    if (S > 1) {
        cluster_sync();
        if (warp >= 4) {  // every CTA adds and writes its own tokens
            constexpr int J = TN / S / (Sh::kWriters / 4);
            const int quad = warp & 3, j0 = part * (TN / S) + (warp - 4) / 4 * J;
            const uint32_t own = smem_u32(base) + 4 * (j0 * 128 + quad * 32 + lane);
            const int64_t f = static_cast<int64_t>(fb) * 128 + quad * 32 + lane;
            float v[J][S];
#pragma unroll
            for (int j = 0; j < J; ++j)
#pragma unroll
                for (int r = 0; r < S; ++r) v[j][r] = j0 + j < a.n ? cluster_load(own + j * 512, r) : 0.0f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                float y = v[j][0];
#pragma unroll
                for (int r = 1; r < S; ++r) y += v[j][r];
                if (j0 + j < a.n && f < a.features) put(a, j0 + j, f, y);
            }
        }
        cluster_sync();  // no CTA leaves while its sums are being read
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && *abort != 0) spk_flag(a.status, SPK_STATUS_DEVICE_WAIT_EXPIRED);
    if (warp == 0) tmem_dealloc(tmem, Sh::kColumns);
}

// ---- many rows ---------------------------------------------------------------------------------------------------------------------------------
// Tile = (128 tokens, or 256 by a pair of CTAs; NF features).  The tokens are the M operand: a thread of the epilogue has one token and half of the tile's
// features, so a block of k has one factor per thread.  CG = 2: a pair of CTAs on two SMs, each holding its 128 tokens and half of the features' rows
// (cta_group::2); the even one issues the MMAs.  Persistent: CTAs go over the tiles, the copies of the next tile under way while this one's results are written.
// S > 1 (one tile per cluster): the cluster's CTAs are parts of k as above.
template <int NF, int CG>
struct Tile {
    static constexpr int kRowsW = NF / CG;
    static constexpr int kStage = kTileW + kRowsW * kBlock;
    static constexpr int NS = kStage > 40000 ? 4 : 6;
    static constexpr int NB = 512 / NF;
    static constexpr int kScales = kGroups * kGroup * (128 + 4) * 4;
    static constexpr int kBytes = 1024 + NS * kStage + kScales + 1024;
};
constexpr int kPanel = 16;   // tiles of tokens
constexpr int kWriters = 8;  // warps that scale and add up a block's sums
constexpr int kTileThreads = 128 + 32 * kWriters;

// The scales of `kn` blocks of k, ROWS tokens and FB runs of 128 features, into a ring [kGroups][kGroup][ROWS + 4] (tokens, then runs), kGroup blocks at a time, by two
// warps in turn with asynchronous copies.  Asked for one or two blocks ahead by the threads that use them, scales were waited for (1171 x 4864 x 896: 0.62 us a block, the
// latency of HBM over two); a barrier for every block took 0.1 us of the 0.5 that a block of 128 x 256 took, and so did copies of four bytes where rows of scales are
// aligned to 16 (`vec`).  g: groups so far; x: the first token's scale, of `rows` that exist (none: any scale); w: the first run's, of `runs`.  false where a wait ran out.
template <int ROWS, int FB>
__device__ __forceinline__ bool bring_scales(Bars* bars, float* ring, int who, int& g, int kn, const float* x, int64_t x_step, int rows, int vec, const float* w, int64_t w_run, int runs,
                                             volatile int* abort) {
    const int lane = threadIdx.x & 31;
    auto copy = [](uint32_t dst, const float* src, int count) {  // of 16 bytes: those of `count` floats, zeros behind them
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(4 * count) : "memory");
    };
    auto copy4 = [](uint32_t dst, const float* src, bool live) {
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(__cvta_generic_to_global(src)), "r"(live ? 4 : 0) : "memory");
    };
    const int left = rows - 4 * lane, count = left < 0 ? 0 : left > 4 ? 4 : left;
    for (int k0 = 0; k0 < kn; k0 += kGroup, ++g) {
        if ((g & 1) != who) continue;
        const int at = g % kGroups;
        if (g >= kGroups && !__all_sync(~0u, mbar_wait(smem_u32(&bars->used[at]), ((g / kGroups) - 1) & 1, abort))) return false;
        uint32_t dst = smem_u32(ring + at * kGroup * (ROWS + 4));
        const float* xk = x + k0 * x_step;
        for (int k = k0; k < k0 + kGroup && k < kn; ++k, xk += x_step, dst += 4 * (ROWS + 4)) {
            if (vec) {
                if (4 * lane < ROWS) copy(dst + 16 * lane, count > 0 ? xk + 4 * lane : xk, count);
            } else {
#pragma unroll
                for (int j = lane; j < ROWS; j += 32) copy4(dst + 4 * j, j < rows ? xk + j : xk, j < rows);
            }
            if (lane < FB) copy4(dst + 4 * (ROWS + lane), lane < runs ? w + lane * w_run + k : w, lane < runs);
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bars->factors[at])) : "memory");
    }
    return true;
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
// On a barrier of any CTA of the cluster.  What is handed over is tensor memory, ordered by the tcgen05 fences: no release of cluster scope, which took some 2 us.
__device__ __forceinline__ void remote_arrive(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// A copy of one of the pair, whose barrier is the even CTA's.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
// C columns of a result row, those below `left` alone; BY: all of them exist, at a multiple of so many bytes.
template <int BY, int C>
__device__ __forceinline__ void put_row(const spk_linear_fp8_args& a, int64_t t, int64_t f, const float* v, int64_t left) {
    if (BY == 0) {
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (i < left) put(a, t, f + i, v[i]);
        return;
    }
    auto store = [](uint32_t* o, const uint32_t* w) {  // eight words
        if (BY == 32) {
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(o), SPK_I8(w, 0) : "memory");
        } else {
            reinterpret_cast<uint4*>(o)[0] = make_uint4(w[0], w[1], w[2], w[3]);
            reinterpret_cast<uint4*>(o)[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
    };
    if (a.out_dtype == SPK_F32) {
        uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<float*>(a.out) + t * a.out_stride + f);
#pragma unroll
        for (int i = 0; i < C / 8; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(v[8 * i + j]);
            store(o + 8 * i, w);
        }
    } else {
        uint32_t* o = reinterpret_cast<uint32_t*>(static_cast<__nv_bfloat16*>(a.out) + t * a.out_stride + f);
#pragma unroll
        for (int i = 0; i < C / 16; ++i) {
            uint32_t w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = pack_bf16(v[16 * i + 2 * j], v[16 * i + 2 * j + 1]);
            store(o + 8 * i, w);
        }
    }
}
template <int C>
__device__ __forceinline__ void put_row(const spk_linear_fp8_args& a, int vec, int64_t t, int64_t f, const float* v) {
    const int64_t left = a.features - f;
    if (vec == 32 && left >= C) put_row<32, C>(a, t, f, v, C);
    else if (vec == 16 && left >= C) put_row<16, C>(a, t, f, v, C);
    else put_row<0, C>(a, t, f, v, left);
}

template <int NF, int CG, int S>
__global__ void __launch_bounds__(kTileThreads, 1)
fp8_tiles_kernel(const __grid_constant__ spk_linear_fp8_args a, const __grid_constant__ CUtensorMap w_map, const __grid_constant__ CUtensorMap x_map, const int blocks, const int m_tiles,
                 const int n_tiles, const int vec, const int vec_scales) {
    using Sh = Tile<NF, CG>;
    constexpr int NS = Sh::NS, NB = Sh::NB, H = 4 * NF / kWriters;  // columns of a thread
    static_assert(CG == 1 || S == 1, "a pair takes all of k");
    static_assert(S == 1 || 128 * NF * 4 <= NS * Sh::kStage, "partial sums take the stages' place");
    extern __shared__ uint8_t raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~uintptr_t(1023));
    constexpr int FB = NF / 128;
    float* ring = reinterpret_cast<float*>(base + NS * Sh::kStage);  // of bring_scales
    Bars* bars = reinterpret_cast<Bars*>(base + NS * Sh::kStage + Sh::kScales);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = CG == 2 ? static_cast<int>(cluster_rank()) : 0;
    const int part = S > 1 ? static_cast<int>(blockIdx.x) % S : 0;
    const int first = blockIdx.x / (CG * S), stride = gridDim.x / (CG * S);
    const int kb = blocks * part / S, kn = blocks * (part + 1) / S - kb;
    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            mbar_init(smem_u32(&bars->full[i]), 1);
            mbar_init(smem_u32(&bars->free[i]), 1);
        }
        for (int i = 0; i < NB; ++i) {
            mbar_init(smem_u32(&bars->sums[i]), 1);
            mbar_init(smem_u32(&bars->drained[i]), kWriters * CG);
        }
        for (int i = 0; i < kGroups; ++i) {
            mbar_init(smem_u32(&bars->factors[i]), 32);
            mbar_init(smem_u32(&bars->used[i]), kWriters);
        }
        mbar_init(smem_u32(&bars->done), 1);
        bars->abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 0) {
        if (CG == 1) {
            tmem_alloc(smem_u32(&bars->tmem), 512);
        } else {
            __syncwarp();
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        }
    }
    fence_async_shared();
    tc_fence_before();
    __syncthreads();
    if (CG == 2) {  // the pair's barriers are set up
        cluster_sync();
    }
    tc_fence_after();
    const uint32_t tmem = bars->tmem;
    volatile int* abort = &bars->abort;
    // tiles go over the tokens of a panel, then the features, then the panels: x beyond the cache is read from memory once
    const int tiles = m_tiles * n_tiles, per_panel = kPanel * n_tiles;
    auto high = [&](int tile) { return min(kPanel, m_tiles - tile / per_panel * kPanel); };
    auto m_of = [&](int tile) { return tile / per_panel * kPanel + tile % per_panel % high(tile); };
    auto n_of = [&](int tile) { return tile % per_panel / high(tile); };
    if (warp < 4) {  // 128 x 56 + 256 x 224 registers: the launch's 384 x 168
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            if (lane == 0) {
                int c = 0;
                bool go = true;
                for (int tile = first; tile < tiles && go; tile += stride) {
                    const int t0 = m_of(tile) * 128 * CG + rank * 128, f0 = n_of(tile) * NF + rank * Sh::kRowsW;
                    for (int k = 0; k < kn; ++k, ++c) {
                        const int s = c % NS;
                        if (c >= NS && !mbar_wait(smem_u32(&bars->free[s]), ((c / NS) - 1) & 1, abort)) {
                            go = false;
                            break;
                        }
                        const uint32_t dst = smem_u32(base + s * Sh::kStage);
                        if (CG == 1) {
                            const uint32_t bar = smem_u32(&bars->full[s]);
                            mbar_expect(bar, Sh::kStage);
                            tma_load(dst, &x_map, (kb + k) * kBlock, t0, bar);
                            tma_load(dst + kTileW, &w_map, (kb + k) * kBlock, f0, bar);
                        } else {
                            const uint32_t bar = at_rank(smem_u32(&bars->full[s]), 0);
                            if (rank == 0) mbar_expect(smem_u32(&bars->full[s]), 2 * Sh::kStage);
                            tma_load_pair(dst, &x_map, (kb + k) * kBlock, t0, bar);
                            tma_load_pair(dst + kTileW, &w_map, (kb + k) * kBlock, f0, bar);
                        }
                    }
                }
                // copies in flight land before the CTA's shared memory is given up
                if (*abort != 0 && rank == 0)
                    for (int k = c > NS ? c - NS : 0; k < c; ++k) mbar_wait(smem_u32(&bars->full[k % NS]), (k / NS) & 1);
            }
        } else if (warp == 1) {
            if (rank == 0) {  // in code that the whole warp runs: descriptors stay in uniform registers
                constexpr uint32_t idesc = idesc_e4m3(128 * CG, NF);
                const uint32_t who = elect_one();
                int c = 0;
                bool go = true;
                for (int tile = first; tile < tiles && go; tile += stride) {
                    for (int k = 0; k < kn; ++k, ++c) {
                        const int s = c % NS, b = c % NB;
                        go = __all_sync(~0u, (c < NB || mbar_wait(smem_u32(&bars->drained[b]), ((c / NB) - 1) & 1, abort)) &&
                                                 mbar_wait(smem_u32(&bars->full[s]), (c / NS) & 1, abort));
                        if (!go) break;
                        tc_fence_after();
                        const uint32_t xa = smem_u32(base + s * Sh::kStage), wa = xa + kTileW;
#pragma unroll
                        for (int i = 0; i < 4; ++i) mma_e4m3_by<CG>(who, tmem + b * NF, desc_sw128(xa + i * 32, 16, 1024), desc_sw128(wa + i * 32, 16, 1024), idesc, i > 0);
                        commit_by<CG>(who, smem_u32(&bars->free[s]));
                        commit_by<CG>(who, smem_u32(&bars->sums[b]));
                    }
                }
                commit_by<CG>(who, smem_u32(&bars->done));
                mbar_wait(smem_u32(&bars->done), 0);  // nothing this warp issued is in the tensor pipe any more
            }
        } else {
            int g = 0;
            for (int tile = first; tile < tiles; tile += stride) {
                const int64_t t = static_cast<int64_t>(m_of(tile)) * 128 * CG + rank * 128, fb = static_cast<int64_t>(n_of(tile)) * FB;
                if (!bring_scales<128, FB>(bars, ring, warp - 2, g, kn, a.x_scales + kb * a.x_scale_stride + (t < a.n ? t : 0), a.x_scale_stride,
                                           static_cast<int>(max(min(a.n - t, static_cast<int64_t>(128)), static_cast<int64_t>(0))), vec_scales,
                                           a.w_scales + fb * a.w_scale_stride + kb, a.w_scale_stride, static_cast<int>(min((a.features + 127) / 128 - fb, static_cast<int64_t>(FB))), abort))
                    break;
            }
            cp_async_wait_all();
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        const int quad = warp & 3, half = (warp - 4) / 4, r = quad * 32 + lane;
        const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
        const uint32_t drained = CG == 2 ? at_rank(smem_u32(&bars->drained[0]), 0) : smem_u32(&bars->drained[0]);
        int c = 0, g = 0;
        bool ok = true, odd = false;
        for (int tile = first; tile < tiles && ok; tile += stride) {
            float acc[H];
#pragma unroll
            for (int j = 0; j < H; ++j) acc[j] = 0.0f;
            for (int k = 0; k < kn; ++k, ++c) {
                const int b = c % NB;
                if (k % kGroup == 0) ok = mbar_wait(smem_u32(&bars->factors[g % kGroups]), (g / kGroups) & 1, abort);
                const float* scales = ring + (g % kGroups * kGroup + k % kGroup) * 132;
                const float m = scales[r] * scales[128 + half * H / 128];
                odd = odd || may_be_far(m);
                ok = __all_sync(~0u, ok && mbar_wait(smem_u32(&bars->sums[b]), (c / NB) & 1, abort));
                if (!ok) break;
                tc_fence_after();
                const uint32_t from = tmem + lanes + b * NF + half * H;
                const bool last = k % kGroup == kGroup - 1 || k == kn - 1;  // of its group
                uint32_t v[2][32];
                tmem_ld32(from, v[0]);
#pragma unroll
                for (int j0 = 0; j0 < H; j0 += 32) {
                    const int p = (j0 / 32) & 1;
                    tmem_wait_ld(v[p]);
                    if (j0 + 32 < H) {
                        tmem_ld32(from + j0 + 32, v[p ^ 1]);
                    } else {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) {
                            if (CG == 1) mbar_arrive(drained + 8 * b);
                            else remote_arrive(drained + 8 * b);
                            if (last) mbar_arrive(smem_u32(&bars->used[g % kGroups]));
                        }
                    }
#pragma unroll
                    for (int j = 0; j < 32; ++j) acc[j0 + j] = fmaf(__uint_as_float(v[p][j]), m, acc[j0 + j]);
                }
                if (last) ++g;
            }
            const int64_t t = static_cast<int64_t>(m_of(tile)) * 128 * CG + rank * 128 + r, f = static_cast<int64_t>(n_of(tile)) * NF + half * H;
            if (S == 1) {
                if (ok && t < a.n) {
#pragma unroll
                    for (int j = 0; j < H; j += 32) put_row<32>(a, vec, t, f + j, acc + j);
                }
            } else {  // [column][token]
                float* sums = reinterpret_cast<float*>(base) + half * H * 128 + r;
#pragma unroll
                for (int j = 0; j < H; ++j) sums[j * 128] = ok ? acc[j] : 0.0f;
                if (ok && odd && has_far(a, t, f, kb, kn))
                    for (int j = 0; j < H; ++j) sums[j * 128] = far_sum(a, t, f + j, kb, kn);
            }
        }
        if (S == 1 && ok && odd) {  // behind the last tile, where no other warp waits for this one
            for (int tile = first; tile < tiles; tile += stride) {
                const int64_t t = static_cast<int64_t>(m_of(tile)) * 128 * CG + rank * 128 + r, f = static_cast<int64_t>(n_of(tile)) * NF + half * H;
                if (has_far(a, t, f, kb, kn))
                    for (int j = 0; j < H && f + j < a.features; ++j) put(a, t, f + j, far_sum(a, t, f + j, kb, kn));
            }
        }
    }
    if (S > 1) {
        cluster_sync();
        if (warp >= 4) {  // every CTA adds and writes its own columns, two warps those of a token
            constexpr int J = NF / S / (kWriters / 4);
            const int r = (warp & 3) * 32 + lane, j0 = part * (NF / S) + (warp - 4) / 4 * J;
            const int64_t t = static_cast<int64_t>(m_of(first)) * 128 + r, f = static_cast<int64_t>(n_of(first)) * NF + j0;
            float v[J];
#pragma unroll
            for (int j = 0; j < J; ++j) {
                v[j] = cluster_load(smem_u32(base) + 4 * ((j0 + j) * 128 + r), 0);
#pragma unroll
                for (int q = 1; q < S; ++q) v[j] += cluster_load(smem_u32(base) + 4 * ((j0 + j) * 128 + r), q);
            }
            if (t < a.n) put_row<J>(a, vec, t, f, v);
        }
    }
    if (S > 1 || CG == 2) {
        cluster_sync();  // no CTA leaves while its sums are being read, or its partner works in its memory
    }
    // Behind the pair's barrier the even CTA has seen its last commit, so its arrivals here are all but made, however long the product took (a wait's limit is meant for one phase).
    if (CG == 2 && rank != 0 && warp == 1 && !mbar_wait(smem_u32(&bars->done), 0)) *abort = 1;
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0 && *abort != 0) spk_flag(a.status, SPK_STATUS_DEVICE_WAIT_EXPIRED);
    if (warp == 0) {
        if (CG == 1) {
            tmem_dealloc(tmem, 512);
        } else {
            __syncwarp();
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
        }
    }
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

int aligned_scales(const spk_linear_fp8_args& a) { return reinterpret_cast<uintptr_t>(a.x_scales) % 16 == 0 && a.x_scale_stride % 4 == 0; }

template <int TN, int S>  // n <= TN
int launch_rows(const spk_linear_fp8_args& a, cudaStream_t s) {
    constexpr int bytes = Shape<TN>::kBytes;
    static_assert(sizeof(Bars) <= 1024 && bytes <= 227 * 1024, "shared memory");
    CUtensorMap w_map, x_map;
    if (!encode(&w_map, a.w, a.features, a.k, a.w_stride, 128) || !encode(&x_map, a.x, a.n, a.k, a.x_stride, TN)) return SPK_ERR_UNSUPPORTED;
    const int blocks = static_cast<int>((a.k + kBlock - 1) / kBlock);
    const int64_t fblocks = (a.features + 127) / 128;
    if (fblocks * S > 0x7fffffff) return SPK_ERR_TOO_LARGE;
    auto kernel = fp8_rows_kernel<TN, S>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {};
    cfg.gridDim = dim3(static_cast<unsigned>(fblocks * S));
    cfg.blockDim = dim3(Shape<TN>::kThreads);
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

template <int NF, int CG, int S>
int launch_tiles(const spk_linear_fp8_args& a, cudaStream_t s) {
    using Sh = Tile<NF, CG>;
    static_assert(sizeof(Bars) <= 1024 && Sh::kBytes <= 227 * 1024, "shared memory");
    CUtensorMap w_map, x_map;
    if (!encode(&w_map, a.w, a.features, a.k, a.w_stride, Sh::kRowsW) || !encode(&x_map, a.x, a.n, a.k, a.x_stride, 128)) return SPK_ERR_UNSUPPORTED;
    const int blocks = static_cast<int>((a.k + kBlock - 1) / kBlock);
    const int64_t m = (a.n + 128 * CG - 1) / (128 * CG), tiles = m * ((a.features + NF - 1) / NF);
    if (tiles * S > 0x3fffffff) return SPK_ERR_TOO_LARGE;
    auto kernel = fp8_tiles_kernel<NF, CG, S>;
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Sh::kBytes);
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    const size_t size = a.out_dtype == SPK_F32 ? 4 : 2;
    auto at = [&](size_t b) { return reinterpret_cast<uintptr_t>(a.out) % b == 0 && a.out_stride * size % b == 0; };
    const int vec = at(32) ? 32 : at(16) ? 16 : 0;
    const int64_t groups = S > 1 || tiles < 148 / CG ? tiles : 148 / CG;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1] = {};
    cfg.gridDim = dim3(static_cast<unsigned>(groups * CG * S));
    cfg.blockDim = dim3(kTileThreads);
    cfg.dynamicSmemBytes = Sh::kBytes;
    cfg.stream = s;
    cfg.attrs = attr;
    if (S > 1 || CG > 1) {
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim = {S * CG, 1, 1};
        cfg.numAttrs = 1;
    }
    e = cudaLaunchKernelEx(&cfg, kernel, a, w_map, x_map, blocks, static_cast<int>(m), static_cast<int>(tiles / m), vec, aligned_scales(a));
    if (e != cudaSuccess) return spk_set_cuda_error(e);
    spk_count_launch();
    return SPK_OK;
}

// The form of a product: rows of a tile (16, 32, 64: fp8_rows_kernel; 128; 256: by pairs) and parts of k.
struct Form {
    int rows, parts;
};
Form form_of(int64_t n, int64_t k, int64_t features) {
    const int64_t blocks = (k + kBlock - 1) / kBlock, fblocks = (features + 127) / 128;
    if (n <= 64) {
        // Parts of k: as many as leave the clusters on the chip at once (148 SMs in groups of 16 to 18 hold 64 or more of two CTAs, 32 of four, 16 of eight).  One / two / four parts, us: 16 x 3584 x
        // 4608 11.5 / 8.7 / 12.4 (36 clusters of four: two waves), 64 x 18944 x 3584 51.8 / 28.0 / 18.8, 64 x 4864 x 896 17.7 / 11.5 / 8.8 (eight 8.0),
        // 16 x 18944 x 1024 in four / eight 13.7 / 9.7, 64 x 18944 x 2048 17.7 / 23.9, 1 x 896 x 4864 5.5 / 5.4 / 8.3 whole / in two / four.
        const int parts = fblocks <= 8 && blocks >= 16 ? 8 : fblocks <= 32 && blocks >= 8 ? 4 : fblocks <= 64 && blocks >= 4 ? 2 : 1;
        return {n <= 16 ? 16 : n <= 32 ? 32 : 64, parts};
    }
    // Tiles of 128 x 128, or of 256 x 256 by pairs of CTAs, which take 1.6 times as long a wave (8192 x 3584 x 18944: 720 / 564 us; 1171 x 896 x 4864, three waves of 380 tiles against
    // two of 95: 14.9 / 16.8).  Few tiles: parts of k as above (1171 x 4864 x 896, 70 tiles: 19.2 us whole, 15.0 in two).
    const int64_t tiles = (n + 127) / 128 * fblocks, pairs = (n + 255) / 256 * ((features + 255) / 256);
    if (tiles <= 32 && blocks >= 16) return {128, 4};
    if (tiles <= 72 && blocks >= 8) return {128, 2};
    return {8 * ((pairs + 73) / 74) < 5 * ((tiles + 147) / 148) ? 256 : 128, 1};
}

template <int TN>
int launch_parts(const spk_linear_fp8_args& a, int parts, cudaStream_t s) {
    if (parts == 8) return launch_rows<TN, 8>(a, s);
    if (parts == 4) return launch_rows<TN, 4>(a, s);
    if (parts == 2) return launch_rows<TN, 2>(a, s);
    return launch_rows<TN, 1>(a, s);
}

}  // namespace

extern "C" int spk_linear_fp8_form(int64_t n, int64_t k, int64_t features) {
    if (n < 1 || k < 1 || features < 1) return 0;
    const Form f = form_of(n, k, features);
    return f.rows * 16 + f.parts;
}

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
    const Form f = form_of(a.n, a.k, a.features);
    if (f.rows == 16) return launch_parts<16>(a, f.parts, s);
    if (f.rows == 32) return launch_parts<32>(a, f.parts, s);
    if (f.rows == 64) return launch_parts<64>(a, f.parts, s);
    if (f.parts == 4) return launch_tiles<128, 1, 4>(a, s);
    if (f.parts == 2) return launch_tiles<128, 1, 2>(a, s);
    if (f.rows == 256) return launch_tiles<256, 2, 1>(a, s);
    return launch_tiles<128, 1, 1>(a, s);
}

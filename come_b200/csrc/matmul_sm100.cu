// Products of the feed-forward half of a block on Blackwell tensor cores (sm_100a): the kernel with one 128 x 128 result tile per
// CTA (128 rows of both projections in the gated forms), the contraction of a tile split over the CTAs of a cluster.
//
//   warps 0-7 : two epilogue warpgroups, columns [0, 64) and [64, 128) of the tile.  Thread r of a warpgroup owns row r (TMEM lane r).
//               8-bit operands: every K block of 128 is a product of its own (two TMEM buffers), whose sums the thread scales by
//               a_scale[row, block] * b_scale[column block, block] and adds to float32 registers: the scales are constants of the row
//               there, so a block costs one FMA per sum.  16-bit operands: the whole contraction is summed in TMEM.
//               The sums go to shared memory, where the CTAs of the cluster read each other's: row i of the tile is finished by the
//               CTA of rank i % cluster, which adds the shares in the order of the ranks (no atomics: the same bits in every run),
//               applies the epilogue with a warp per row and stores whole rows of 128 neighbouring columns.
//   warp 8    : producer (TMA ring).      warp 9 : MMA issuer.
//
// Why a split: a block's products have few tiles where there are few tokens (1 x 2736 -> 1024: eight), and a tile's time is its
// contraction's; shares of it bring up to eight SMs per tile to read the weights (64 of 148 there).  The shares meet in shared memory, not in a workspace, so that two
// graphs captured from the same call share nothing.
//
// Measured in a graph: 1 token 2736 -> 1024 in 8 bits 6.4 us, 64 tokens 7.7, 128 tokens 9.0 (weights 2.8 MB; launch, cluster barriers and
// the first loads' latency are most of it), 1374 tokens 1024 -> 1024 10 us.  The 8-bit gated form spills 72 bytes (128 float32 sums beside
// the loads in 168 registers).
//
// Shared memory: a CTA asks for all of an SM's, so that no other CTA that needs tensor memory, of this library or of another, shares its
// SM: CTAs of two clusters that wait for each other's tensor memory while their partners wait at a cluster barrier would never end.
//
// Every wait on an mbarrier is bounded (kWaitTicks): a CTA whose wait gave up raises its abort flag and the device status word, goes
// on to the cluster's barriers, and no CTA of the cluster stores.
#include "matmul_sm100.cuh"

#include <mutex>

namespace come {

namespace {

constexpr int kEpilogueWarps = 8, kProducerWarp = 8, kIssuerWarp = 9, kThreads = 320;
constexpr int kRingBytes = 192 * 1024;
constexpr int kPartRow = kTile + 4;                // floats: rows of the shares in shared memory, no bank conflicts row to row
constexpr int kPartBytes = kTile * kPartRow * 4;
constexpr int kMaxCluster = 8;

struct SplitBarriers {
    uint64_t full[6], empty[6];
    uint64_t acc_full[2], acc_empty[2];
    uint64_t drained;
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
};
constexpr size_t kSmemBytes = 227 * 1024;
static_assert(kRingBytes + sizeof(SplitBarriers) <= kSmemBytes, "");
static_assert(2 * kPartBytes <= kRingBytes, "the shares reuse the ring");

// Four neighbouring columns of a row, `valid` of them inside the result.
__device__ __forceinline__ void store4(void *out, int64_t at, const float (&v)[4], int valid, int dtype) {
    if (dtype == COME_F32) {
        float *p = (float *)out + at;
        if (valid >= 4 && ((uintptr_t)p & 15) == 0) *reinterpret_cast<float4 *>(p) = make_float4(v[0], v[1], v[2], v[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < valid) p[i] = v[i];
        return;
    }
    const bool bf16 = dtype == COME_BF16;
    const uint32_t lo = bf16 ? pack_16<true>(v[0], v[1]) : pack_16<false>(v[0], v[1]), hi = bf16 ? pack_16<true>(v[2], v[3]) : pack_16<false>(v[2], v[3]);
    uint16_t *p = (uint16_t *)out + at;
    if (valid >= 4 && ((uintptr_t)p & 7) == 0) *reinterpret_cast<uint2 *>(p) = make_uint2(lo, hi);
    else {
        if (valid > 0) p[0] = (uint16_t)lo;
        if (valid > 1) p[1] = (uint16_t)(lo >> 16);
        if (valid > 2) p[2] = (uint16_t)hi;
        if (valid > 3) p[3] = (uint16_t)(hi >> 16);
    }
}
__device__ __forceinline__ void load4(const void *in, int64_t at, float (&v)[4], int valid, int dtype) {
    const uint16_t *p = (const uint16_t *)in + at;
    if (dtype != COME_F32 && valid >= 4 && ((uintptr_t)p & 7) == 0) {
        const uint2 raw = *reinterpret_cast<const uint2 *>(p);
        if (dtype == COME_BF16) {
            v[0] = __uint_as_float(raw.x << 16);
            v[1] = __uint_as_float(raw.x & 0xffff0000u);
            v[2] = __uint_as_float(raw.y << 16);
            v[3] = __uint_as_float(raw.y & 0xffff0000u);
        } else {
            const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&raw.x)), hi = __half22float2(*reinterpret_cast<const __half2 *>(&raw.y));
            v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < valid ? load_any(in, at + i, dtype) : 0.0f;
}

// kSelfTest: the producers of some CTAs stop before a K block, so that the waits for it run out, after a limit of the launch's own.
template <bool kE4m3, int kMode, bool kAMn, bool kBMn, bool kSelfTest>
__global__ void __launch_bounds__(kThreads, 1) matmul_split_kernel(const __grid_constant__ MatmulParams p) {
    constexpr int kMats = kMode == kMatmulPlain ? 1 : 2;
    constexpr int kN = kMats * kTile;
    constexpr int kStageBytes = kOperandBytes * (1 + kMats), kStages = kRingBytes / kStageBytes;
    constexpr int kElems = kE4m3 ? 128 : 64;  // contraction elements of a K block
    constexpr uint32_t kTmemCols = 512;
    static_assert(kStages <= 6 && 2 * kN <= kTmemCols, "");
    extern __shared__ __align__(1024) uint8_t smem[];
    SplitBarriers &sh = *reinterpret_cast<SplitBarriers *>(smem + kRingBytes);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank(), ranks = cluster_size();

    const int tile = (int)(blockIdx.x / ranks), per_problem = p.tiles_m * p.tiles_n, problem = tile / per_problem, t = tile - problem * per_problem;
    const int m0 = (t / p.tiles_n) * kTile, n0 = (t % p.tiles_n) * kTile;
    const int kb0 = (int)((int64_t)p.k_blocks * rank / ranks), kb1 = (int)((int64_t)p.k_blocks * (rank + 1) / ranks), n_kb = kb1 - kb0;
    const int rows = min(kTile, p.M - m0);

    if (warp == kProducerWarp && lane == 0) {
        prefetch_map(&p.a[problem * p.sums]);
        prefetch_map(&p.b[0]);
        if constexpr (kMats == 2) prefetch_map(&p.b[1]);
        sh.abort_flag = (*(volatile unsigned int *)p.status & kStatusMatmul) != 0 ? 1u : 0u;  // an earlier launch gave up
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.acc_full[i], 1);
            mbar_init(&sh.acc_empty[i], kEpilogueWarps);
        }
        mbar_init(&sh.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssuerWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    // All of the SM's tensor memory is allocated, so its base is column 0: the tensor-memory addresses are constants.
    constexpr uint32_t tmem = 0;
    const uint32_t ring = smem_u32(smem);
    const auto limit = [&] { return kSelfTest ? p.wait_limit : kWaitTicks; };
    const auto wait = [&](uint64_t *bar, uint32_t parity, uint32_t code) { return mbar_wait_limit(bar, parity, &sh.abort_flag, p.status, code, limit()); };
    const bool misplaced = sh.tmem_base != tmem, dead = sh.abort_flag != 0 || misplaced;
    if (misplaced && threadIdx.x == 0) atomicOr(p.status, kErrSums);

    if (!dead && warp == kProducerWarp) {
        if (lane == 0) {
            int i = 0;
            for (; i < n_kb; ++i) {
                const int st = i % kStages;
                if (!wait(&sh.empty[st], ((i / kStages) & 1) ^ 1, kErrEmpty)) break;
                if (kSelfTest && i >= p.stall_block && (p.stall_ctas >> rank & 1)) break;
                const int kb = kb0 + i, sum = kE4m3 || p.sums == 1 ? 0 : kb / p.kb_per_sum, k = (kb - sum * p.kb_per_sum) * kElems;
                const uint32_t dst = ring + st * kStageBytes;
                mbar_arrive_expect_tx(&sh.full[st], kStageBytes);
                const CUtensorMap *ma = &p.a[problem * p.sums + sum], *mb = &p.b[kAMn ? 0 : sum & 1];
                if constexpr (kAMn) {
                    tma_load_2d(dst, ma, m0, k, &sh.full[st]);
                    tma_load_2d(dst + kOperandBytes / 2, ma, m0 + 64, k, &sh.full[st]);
                } else {
                    tma_load_2d(dst, ma, k, m0, &sh.full[st]);
                }
                if constexpr (kBMn) {
                    tma_load_2d(dst + kOperandBytes, mb, n0, k, &sh.full[st]);
                    tma_load_2d(dst + kOperandBytes + kOperandBytes / 2, mb, n0 + 64, k, &sh.full[st]);
                } else {
                    tma_load_2d(dst + kOperandBytes, mb, k, n0, &sh.full[st]);
                    if constexpr (kMats == 2) tma_load_2d(dst + 2 * kOperandBytes, &p.b[1], k, n0, &sh.full[st]);
                }
            }
            for (int j = max(i - kStages, 0); j < i; ++j) mbar_drain(&sh.full[j % kStages], (j / kStages) & 1, p.status, kErrFull, limit());
            if (i == n_kb)  // the last arrivals of the products, which no other role waits for
                for (int j = max(i - kStages, 0); j < i && wait(&sh.empty[j % kStages], (j / kStages) & 1, kErrEmpty); ++j) {
                }
        }
        __syncwarp();
    } else if (!dead && warp == kIssuerWarp) {
        // Warp-uniform control flow and constant tensor-memory addresses: see matmul_pair_sm100.cu.
        const uint32_t idesc = matmul_idesc(kE4m3, p.dtype == COME_BF16, kTile, kN, kAMn, kBMn);
        constexpr uint32_t kAStep = kAMn ? 2048 >> 4 : 32 >> 4, kBStep = kBMn ? 2048 >> 4 : 32 >> 4;
        const uint64_t desc_a = operand_desc(ring, kOperandBytes / 2), desc_b = operand_desc(ring + kOperandBytes, kOperandBytes / 2);
        uint32_t st = 0, st_phase = 0, buf = 0, buf_phase = 1;
        bool ok = true;
        const auto wait_here = [&](uint64_t *bar, uint32_t parity, uint32_t code) {
            if (!mbar_try_wait(bar, parity)) ok = ok && wait(bar, parity, code);
        };
        for (int i = 0; i < n_kb; ++i) {
            if ((i & 31) == 31 && !__all_sync(0xffffffffu, ok)) break;
            wait_here(&sh.full[st], st_phase, kErrFull);
            if (kE4m3) wait_here(&sh.acc_empty[buf], buf_phase, kErrSums);
            __syncwarp();
            tc_fence_after();
            const uint64_t da = desc_a + (uint64_t)(st * (kStageBytes >> 4)), db = desc_b + (uint64_t)(st * (kStageBytes >> 4));
            if (elect_one() && ok) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t more = k > 0 || (!kE4m3 && i > 0) ? 1u : 0u;
                    if constexpr (kE4m3) tc_mma_f8_ss_1(buf * kN, da + k * kAStep, db + k * kBStep, idesc, more);
                    else tc_mma_ss_1(0, da + k * kAStep, db + k * kBStep, idesc, more);
                }
                tc_commit_1(&sh.empty[st]);
                if (kE4m3 || i == n_kb - 1) tc_commit_1(&sh.acc_full[buf]);
            }
            __syncwarp();
            if (++st == kStages) {
                st = 0;
                st_phase ^= 1u;
            }
            if (kE4m3) {
                buf ^= 1u;
                if (buf == 0) buf_phase ^= 1u;
            }
        }
        if (elect_one()) {
            tc_commit_1(&sh.drained);
            mbar_drain(&sh.drained, 0, p.status, kErrSums, limit());
        }
        __syncwarp();
    } else if (!dead) {
        const int part = warp >> 2, r = (warp & 3) * 32 + lane;  // columns [64 part, + 64) of a weight, row of the tile
        const uint32_t lanes = tmem + ((uint32_t)((warp & 3) * 32) << 16) + part * 64;
        const bool busy = (warp & 3) * 32 < rows;                // a warp without rows only keeps the barriers going
        float *share = reinterpret_cast<float *>(smem) + r * kPartRow + part * 64;
        bool ok = true;
        if constexpr (kE4m3) {
            float sum[kMats][64];
#pragma unroll
            for (int w = 0; w < kMats; ++w)
#pragma unroll
                for (int c = 0; c < 64; ++c) sum[w][c] = 0.0f;
            const float *as = p.a_scale + (int64_t)(m0 + (r < rows ? r : 0)) * p.as_row;
            const float *bs[2] = {p.b_scale[0] + (n0 / kTile) * p.bs_row[0], kMats == 2 ? p.b_scale[1] + (n0 / kTile) * p.bs_row[1] : nullptr};
            float sa = as[kb0 * p.as_block], sb[2] = {bs[0][kb0], kMats == 2 ? bs[1][kb0] : 0.0f};
            for (int i = 0; i < n_kb; ++i) {
                const int buf = i & 1;
                const float s[2] = {sa * sb[0], sa * sb[1]};
                if (i + 1 < n_kb) {
                    sa = as[(kb0 + i + 1) * p.as_block];
                    sb[0] = bs[0][kb0 + i + 1];
                    if constexpr (kMats == 2) sb[1] = bs[1][kb0 + i + 1];
                }
                ok = wait(&sh.acc_full[buf], (i >> 1) & 1, kErrSums);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (busy) {
                    tc_fence_after();
#pragma unroll
                    for (int w = 0; w < kMats; ++w)
#pragma unroll
                        for (int c = 0; c < 64; c += 32) {
                            uint32_t d[32];
                            tmem_ld32(lanes + buf * kN + w * kTile + c, d);
                            tc_wait_ld();
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[w][c + j] = fmaf(__uint_as_float(d[j]), s[w], sum[w][c + j]);
                        }
                    tc_fence_before();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.acc_empty[buf]);
            }
            // the last product has completed and with it every read of the ring: the shares may take its place
            if (ok && busy) {
#pragma unroll
                for (int w = 0; w < kMats; ++w)
#pragma unroll
                    for (int c = 0; c < 64; c += 4)
                        *reinterpret_cast<float4 *>(share + w * (kPartBytes / 4) + c) = make_float4(sum[w][c], sum[w][c + 1], sum[w][c + 2], sum[w][c + 3]);
            }
        } else {
            ok = wait(&sh.acc_full[0], 0, kErrSums);
            ok = __all_sync(0xffffffffu, ok);
            if (ok && busy) {
                tc_fence_after();
#pragma unroll
                for (int w = 0; w < kMats; ++w)
#pragma unroll
                    for (int c = 0; c < 64; c += 32) {
                        uint32_t d[32];
                        tmem_ld32(lanes + w * kTile + c, d);
                        tc_wait_ld();
#pragma unroll
                        for (int j = 0; j < 32; j += 4)
                            *reinterpret_cast<uint4 *>(share + w * (kPartBytes / 4) + c + j) = make_uint4(d[j], d[j + 1], d[j + 2], d[j + 3]);
                    }
            }
        }
    }

    const int n = n0 + 4 * lane, valid = p.N - n;  // the lane's four result columns
    float bias[kMats][4] = {};
#pragma unroll
    for (int w = 0; w < kMats; ++w)
        if (p.bias[w] && warp < kEpilogueWarps)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (i < valid) bias[w][i] = load_any(p.bias[w], n + i, p.bias_dtype);
    [[maybe_unused]] const float factor = range_factor(p.range, kMode == kMatmulPlain);
    if (misplaced && threadIdx.x == 0) sh.abort_flag = 1;  // read by the others behind the barrier
    tc_fence_before();
    cluster_sync();
    bool store = true;
    for (uint32_t s = 0; s < ranks; ++s) store &= ld_cluster_u32(map_rank(smem_u32((const void *)&sh.abort_flag), s)) == 0;
    if (store && warp < kEpilogueWarps) {
        // A warp per row, one copy of the code: a launch of a few microseconds feels every instruction that has to be fetched (four rows
        // at a time, unrolled, took 12 us where this takes 8).  Two shares are asked for together: another SM's shared memory is some
        // 200 clocks away.
#pragma unroll 1
        for (int r = (int)(rank + ranks * warp); r < rows; r += (int)ranks * kEpilogueWarps) {
            const int64_t row = m0 + r, at = row * p.out_row[problem] + n;
            [[maybe_unused]] float dh[4];
            if constexpr (kMode == kMatmulGatedGrad) {
                load4(p.dh, row * p.dh_row + n, dh, valid, p.dtype);
#pragma unroll
                for (int i = 0; i < 4; ++i) dh[i] *= factor;
            }
            float v[kMats][4];
#pragma unroll
            for (int w = 0; w < kMats; ++w)
#pragma unroll
                for (int i = 0; i < 4; ++i) v[w][i] = bias[w][i];
            const uint32_t from = ring + (r * kPartRow + 4 * lane) * 4;
#pragma unroll 1
            for (uint32_t s = 0; s < ranks; s += 2) {
                float4 x[2][kMats];
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                    for (int w = 0; w < kMats; ++w) x[j][w] = s + j < ranks ? ld_cluster(map_rank(from, s + j) + w * kPartBytes) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
                for (uint32_t j = 0; j < 2; ++j)
#pragma unroll
                    for (int w = 0; w < kMats; ++w) v[w][0] += x[j][w].x, v[w][1] += x[j][w].y, v[w][2] += x[j][w].z, v[w][3] += x[j][w].w;
            }
            if constexpr (kMode == kMatmulPlain) {
                if constexpr (!kE4m3) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[0][i] *= factor;
                }
                store4(p.out[problem], at, v[0], valid, p.out_dtype);
            } else if constexpr (kMode == kMatmulGated) {
                float h[4], top = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    h[i] = i < valid ? activation(v[0][i], p.act) * v[1][i] : 0.0f;
                    top = fmaxf(top, fabsf(h[i]));
                }
                if (p.out_dtype != COME_E4M3) {
                    store4(p.out[0], at, h, valid, p.out_dtype);
                } else {
#pragma unroll
                    for (int s = 16; s >= 1; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
                    top = fmaxf(top, kSmallestMax);
                    const float inv = inverse_scale(top);
                    const uint32_t q = pack_e4m3(h[0] * inv, h[1] * inv, h[2] * inv, h[3] * inv);
                    uint8_t *out = (uint8_t *)p.out[0] + at;  // rows start at multiples of 16 bytes
                    if (valid >= 4) {
                        *reinterpret_cast<uint32_t *>(out) = q;
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (i < valid) out[i] = (uint8_t)(q >> (8 * i));
                    }
                    if (lane == 0) p.out_scale[row * p.os_row + (n0 / kTile) * p.os_block] = top * (1.0f / kE4m3Max);
                }
            } else {
                float dg[4], du[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float a, slope;
                    activation_grad(v[0][i], p.act, a, slope);
                    dg[i] = dh[i] * v[1][i] * slope;
                    du[i] = dh[i] * a;
                }
                store4(p.out[0], at, dg, valid, p.out_dtype);
                store4(p.out[1], row * p.out_row[1] + n, du, valid, p.out_dtype);
                if (p.low_rows > 0) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        dg[i] -= p.out_dtype == COME_BF16 ? __bfloat162float(__float2bfloat16_rn(dg[i])) : __half2float(__float2half_rn(dg[i]));
                        du[i] -= p.out_dtype == COME_BF16 ? __bfloat162float(__float2bfloat16_rn(du[i])) : __half2float(__float2half_rn(du[i]));
                    }
                    store4(p.out[0], at + p.low_rows * p.out_row[0], dg, valid, p.out_dtype);
                    store4(p.out[1], (row + p.low_rows) * p.out_row[1] + n, du, valid, p.out_dtype);
                }
            }
        }
    }
    cluster_sync();  // no CTA leaves while another reads its share
    if (warp == kIssuerWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

template <bool kE4m3, int kMode, bool kAMn, bool kBMn, bool kSelfTest = false> int launch_split(const MatmulParams &p, int64_t tiles, int cluster, cudaStream_t st) {
    constexpr auto kernel = matmul_split_kernel<kE4m3, kMode, kAMn, kBMn, kSelfTest>;
    if (int rc = allow_smem<kernel>(kSmemBytes); rc != COME_OK) return rc;
    cudaLaunchAttribute attr = {};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(tiles * cluster));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = kSmemBytes;
    cfg.stream = st;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        set_error("product kernel: launch failed: %s", cudaGetErrorString(e));
        return COME_ERR_CUDA;
    }
    return COME_OK;
}

// CTAs that share a tile's contraction: as many as fill the SMs once, at least one K block each.
int pick_cluster(int64_t tiles, int64_t k_blocks) {
    int c = 1;
    while (c < kMaxCluster && tiles * c * 2 <= sm_count() && c * 2 <= k_blocks) c *= 2;
    return c;
}

int run_matmul(const MatmulArgs &a, cudaStream_t st) {
    const int mats = a.mode == kMatmulPlain ? 1 : 2;
    MatmulParams p = {};
    p.status = status_word_dev();
    if (!p.status) return COME_ERR_CUDA;
    int rc;
    for (int i = 0; i < a.sums * a.problems; ++i) {
        rc = a.a_mn ? make_rows_map(&p.a[i], a.a[i], a.e4m3, a.dtype, a.K, a.M, a.a_row[i], 64) : make_rows_map(&p.a[i], a.a[i], a.e4m3, a.dtype, a.M, a.K, a.a_row[i], kTile);
        if (rc != COME_OK) return rc;
    }
    for (int i = 0; i < (a.a_mn ? 1 : a.sums > 1 ? 2 : mats); ++i) {
        rc = a.b_mn ? make_rows_map(&p.b[i], a.b[i], a.e4m3, a.dtype, a.K, a.N, a.b_row[i], 64) : make_rows_map(&p.b[i], a.b[i], a.e4m3, a.dtype, a.N, a.K, a.b_row[i], kTile);
        if (rc != COME_OK) return rc;
    }
    p.a_scale = a.a_scale;
    p.as_row = a.as_row;
    p.as_block = a.as_block;
    for (int i = 0; i < 2; ++i) {
        p.b_scale[i] = a.b_scale[i];
        p.bs_row[i] = a.bs_row[i];
        p.bias[i] = a.bias[i];
        p.out[i] = a.out[i];
        p.out_row[i] = a.out_row[i];
    }
    p.dh = a.dh;
    p.dh_row = a.dh_row;
    p.range = a.range;
    p.out_scale = a.out_scale;
    p.os_row = a.os_row;
    p.os_block = a.os_block;
    p.M = (int)a.M;
    p.N = (int)a.N;
    const int elems = a.e4m3 ? 128 : 64;
    p.kb_per_sum = (int)((a.K + elems - 1) / elems);
    p.sums = a.sums;
    p.k_blocks = p.kb_per_sum * a.sums;
    p.low_rows = a.low_rows;
    p.problems = a.problems;
    p.wait_limit = a.wait_limit;
    p.stall_block = a.stall_block;
    p.stall_ctas = a.stall_ctas;
    p.act = a.act;
    p.dtype = a.dtype;
    p.bias_dtype = a.e4m3 ? COME_F32 : a.dtype;
    p.out_dtype = a.out_dtype;
    if (matmul_pair_takes(a)) return matmul_pair_launch(a, p, st);
    p.tiles_n = (int)((a.N + kTile - 1) / kTile);
    const int64_t per_problem = (a.M + kTile - 1) / kTile * p.tiles_n, tiles = per_problem * a.problems;
    COME_REQUIRE(tiles < (1ll << 27), "the result has %lld tiles of 128 x 128: too many for one launch", (long long)tiles);
    p.tiles_m = (int)(per_problem / p.tiles_n);
    const int cluster = pick_cluster(tiles, p.k_blocks);
    if (a.wait_limit > 0)
        return a.e4m3 ? launch_split<true, kMatmulGated, false, false, true>(p, tiles, cluster, st) : launch_split<false, kMatmulGated, false, false, true>(p, tiles, cluster, st);
    if (a.e4m3) return a.mode == kMatmulPlain ? launch_split<true, kMatmulPlain, false, false>(p, tiles, cluster, st) : launch_split<true, kMatmulGated, false, false>(p, tiles, cluster, st);
    if (a.mode == kMatmulGated) return launch_split<false, kMatmulGated, false, false>(p, tiles, cluster, st);
    if (a.mode == kMatmulGatedGrad) return launch_split<false, kMatmulGatedGrad, false, false>(p, tiles, cluster, st);
    return a.a_mn ? launch_split<false, kMatmulPlain, true, true>(p, tiles, cluster, st) : launch_split<false, kMatmulPlain, false, true>(p, tiles, cluster, st);
}

// ---- column sums (gradients of the biases) --------------------------------------------------------------------------------
// One CTA per 32 columns of one matrix: 4 lanes x 16 bytes cover a row's columns, kSumRows rows per pass and four passes in flight; a
// thread adds its rows in float32, then the threads of a column are added in their order: one launch, no workspace, the same bits in
// every run.
constexpr int kSumThreads = 512, kSumRows = kSumThreads / 4;
template <typename T>
__global__ void __launch_bounds__(kSumThreads) column_sums_kernel(const T *__restrict__ x0, const T *__restrict__ x1, int64_t row_stride, int64_t rows, int cols,
                                                                  T *__restrict__ out0, T *__restrict__ out1, const unsigned int *status,
                                                                  const uint32_t *range) {
    __shared__ float part[kSumRows][33];
    if (__syncthreads_or((*(const volatile unsigned int *)status & kStatusMatmul) != 0)) return;  // a product gave up: nothing has filled the rows
    const T *x = blockIdx.y ? x1 : x0;
    T *out = blockIdx.y ? out1 : out0;
    if (!out) return;
    const int c = blockIdx.x * 32 + (threadIdx.x & 3) * 8, r0 = threadIdx.x >> 2;
    float sum[8] = {};
    if (c + 8 <= cols) {
        for (int64_t r = r0; r < rows; r += 4 * kSumRows) {
            uint4 raw[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) raw[j] = r + j * kSumRows < rows ? *reinterpret_cast<const uint4 *>(x + (r + j * kSumRows) * row_stride + c) : make_uint4(0, 0, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const T *e = reinterpret_cast<const T *>(&raw[j]);
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] += Elem<T>::to_f32(e[i]);
            }
        }
    } else if (c < cols) {  // the last row may end with its last element
        for (int64_t r = r0; r < rows; r += kSumRows)
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (c + i < cols) sum[i] += Elem<T>::to_f32(x[r * row_stride + c + i]);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) part[r0][(threadIdx.x & 3) * 8 + i] = sum[i];
    __syncthreads();
    // 16 threads per column, then one
    const int col = threadIdx.x & 31, group = threadIdx.x >> 5;
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < kSumRows / 16; ++r) s += part[group * (kSumRows / 16) + r][col];
    __syncthreads();
    part[group][col] = s;
    __syncthreads();
    if (group == 0 && blockIdx.x * 32 + col < cols) {
        s = 0.0f;
#pragma unroll
        for (int r = 0; r < 16; ++r) s += part[r][col];
        out[blockIdx.x * 32 + col] = Elem<T>::from_f32(s * range_factor(range, true));
    }
}

// ---- largest magnitude (float16 gradients) --------------------------------------------------------------------------------
// Bits of the largest |x| as float32, an infinity or a NaN above all numbers; `largest` is zero before.  A maximum is the same in any
// order.  One pass over dh at the copy rate: with the clearing of the word 11 us for 35 MB, 5 for 2 MB.  Three CTAs per SM: with eight their
// 1184 atomics on one address cost 3 us more.
constexpr int kLargestThreads = 512;
__device__ __forceinline__ uint32_t largest_of(const uint4 &v) {  // of the even and of the odd halves
    return __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
}
__global__ void __launch_bounds__(kLargestThreads) largest_kernel(const uint16_t *__restrict__ x, int64_t rows, int64_t cols, int64_t row_stride, uint32_t *__restrict__ largest) {
    __shared__ uint32_t tops[kLargestThreads / 32];
    const bool aligned = (((uintptr_t)x | (uintptr_t)(row_stride * 2)) & 15) == 0;
    uint32_t top = 0;  // two numbers
    for (int64_t r = blockIdx.y; r < rows; r += gridDim.y) {
        const uint16_t *row = x + r * row_stride;
        const int64_t step = (int64_t)gridDim.x * kLargestThreads * 8;
        int64_t c = ((int64_t)blockIdx.x * kLargestThreads + threadIdx.x) * 8;
        if (aligned) {
            for (; c + 3 * step + 8 <= cols; c += 4 * step) {  // four loads in flight
                uint4 v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = __ldg(reinterpret_cast<const uint4 *>(row + c + j * step));
#pragma unroll
                for (int j = 0; j < 4; ++j) top = __vmaxu2(top, largest_of(v[j]));
            }
            for (; c + 8 <= cols; c += step) top = __vmaxu2(top, largest_of(__ldg(reinterpret_cast<const uint4 *>(row + c))));
        }
        for (; c < cols; c += step)
            for (int i = 0; i < 8 && c + i < cols; ++i) top = __vmaxu2(top, row[c + i] & 0x7fffu);
    }
    top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < kLargestThreads / 32; ++i) top = max(top, tops[i]);
        const uint32_t bits = __float_as_uint(__half2float(__ushort_as_half((unsigned short)top))) & 0x7fffffffu;
        if (bits > *(volatile uint32_t *)largest) atomicMax(largest, bits);
    }
}
int find_largest(const void *x, int64_t rows, int64_t cols, int64_t row_stride, uint32_t *largest, cudaStream_t st) {
    if (row_stride == cols) {  // one long row
        cols *= rows;
        rows = 1;
        row_stride = 0;
    }
    COME_CUDA(cudaMemsetAsync(largest, 0, sizeof(uint32_t), st));
    const int64_t blocks = (cols + kLargestThreads * 8 - 1) / (kLargestThreads * 8), most = 3 * sm_count();
    const int64_t gx = blocks < most ? blocks : most, gy = rows < (most + gx - 1) / gx ? rows : (most + gx - 1) / gx;
    largest_kernel<<<dim3((unsigned)gx, (unsigned)gy), kLargestThreads, 0, st>>>((const uint16_t *)x, rows, cols, row_stride, largest);
    return check_launch("come_gated_matmul_backward");
}

bool rows_ok(const void *p, int64_t row_stride, int size) { return p && (uintptr_t)p % 16 == 0 && row_stride >= 0 && row_stride * size % 16 == 0 && row_stride * size < (1ll << 40); }
bool is_16_bit(int dtype) { return dtype == COME_F16 || dtype == COME_BF16; }
constexpr int64_t kMaxExtent = (1ll << 31) - 256;

}  // namespace

}  // namespace come

#define COME_REQUIRE_SIZES(what, m, n, k)                                                                                              \
    COME_REQUIRE((m) >= 0 && (n) >= 0 && (k) > 0 && (m) < come::kMaxExtent && (n) < come::kMaxExtent && (k) < come::kMaxExtent,           \
                 what ": sizes must be positive and fit int32 (got %lld, %lld, %lld)", (long long)(m), (long long)(n), (long long)(k))
#define COME_REQUIRE_MULTIPLES(size, ...) COME_REQUIRE(come::multiples_of(size, __VA_ARGS__), "addresses must be multiples of their elements' size")
#define COME_REQUIRE_ROWS(what, ptr, stride, size, least)                                                                             \
    COME_REQUIRE(come::rows_ok(ptr, stride, size) && (stride) >= (least), what " must be given, 16-byte aligned, with a row stride of whole 16 bytes that holds its rows")

extern "C" int come_matmul_e4m3(const void *x_dev, int64_t x_row_stride, const float *x_scale_dev, int64_t x_scale_row_stride, int64_t x_scale_block_stride,
                                const void *w_dev, int64_t w_row_stride, const float *w_scale_dev, int64_t w_scale_row_stride, const float *bias_dev, int64_t tokens,
                                int64_t features, int64_t channels, void *out_dev, int64_t out_row_stride, int out_dtype, void *stream) {
    COME_REQUIRE_SIZES("come_matmul_e4m3", tokens, features, channels);
    COME_REQUIRE(out_dtype == COME_F32 || come::is_16_bit(out_dtype), "unknown dtype %d", out_dtype);
    if (tokens == 0 || features == 0) return COME_OK;
    COME_REQUIRE_ROWS("x", x_dev, x_row_stride, 1, channels);
    COME_REQUIRE_ROWS("w", w_dev, w_row_stride, 1, channels);
    COME_REQUIRE(x_scale_dev && w_scale_dev && out_dev && out_row_stride >= features, "scales and result must be given");
    COME_REQUIRE(x_scale_row_stride >= 0 && x_scale_block_stride >= 0 && w_scale_row_stride >= 0, "strides of scales must not be negative");
    COME_REQUIRE_MULTIPLES(4, {x_scale_dev, w_scale_dev, bias_dev});
    COME_REQUIRE_MULTIPLES(come::dtype_size(out_dtype), {out_dev});
    come::MatmulArgs a = {};
    a.mode = come::kMatmulPlain;
    a.e4m3 = true;
    a.M = tokens, a.N = features, a.K = channels;
    a.a[0] = x_dev, a.a_row[0] = x_row_stride;
    a.b[0] = w_dev, a.b_row[0] = w_row_stride;
    a.sums = a.problems = 1;
    a.a_scale = x_scale_dev, a.as_row = x_scale_row_stride, a.as_block = x_scale_block_stride;
    a.b_scale[0] = w_scale_dev, a.bs_row[0] = w_scale_row_stride;
    a.bias[0] = bias_dev;
    a.out[0] = out_dev, a.out_row[0] = out_row_stride;
    a.out_dtype = out_dtype;
    return come::run_matmul(a, (cudaStream_t)stream);
}

extern "C" int come_gated_matmul_e4m3(const void *x_dev, int64_t x_row_stride, const float *x_scale_dev, int64_t x_scale_row_stride,
                                      int64_t x_scale_block_stride, const void *gate_dev, int64_t gate_row_stride, const float *gate_scale_dev,
                                      int64_t gate_scale_row_stride, const void *up_dev, int64_t up_row_stride, const float *up_scale_dev,
                                      int64_t up_scale_row_stride, const float *gate_bias_dev, const float *up_bias_dev, int activation, int64_t tokens,
                                      int64_t features, int64_t channels, void *out_dev, int64_t out_row_stride, int out_dtype, float *out_scale_dev,
                                      int64_t out_scale_row_stride, int64_t out_scale_block_stride, void *stream) {
    COME_REQUIRE_SIZES("come_gated_matmul_e4m3", tokens, features, channels);
    COME_REQUIRE(out_dtype == COME_E4M3 || come::is_16_bit(out_dtype), "the result is float16, bfloat16 or 8 bits with scales (got dtype %d)", out_dtype);
    COME_REQUIRE(activation == COME_ACT_SILU || activation == COME_ACT_GELU, "unknown activation %d", activation);
    if (tokens == 0 || features == 0) return COME_OK;
    COME_REQUIRE_ROWS("x", x_dev, x_row_stride, 1, channels);
    COME_REQUIRE_ROWS("gate", gate_dev, gate_row_stride, 1, channels);
    COME_REQUIRE_ROWS("up", up_dev, up_row_stride, 1, channels);
    COME_REQUIRE(x_scale_dev && gate_scale_dev && up_scale_dev && out_dev && out_row_stride >= features, "scales and result must be given");
    COME_REQUIRE(out_dtype != COME_E4M3 || (out_scale_dev && come::rows_ok(out_dev, out_row_stride, 1)),
                 "an 8-bit result needs its scales, 16-byte aligned rows and a row stride of whole 16 bytes");
    COME_REQUIRE(x_scale_row_stride >= 0 && x_scale_block_stride >= 0 && gate_scale_row_stride >= 0 && up_scale_row_stride >= 0 &&
                     (out_dtype != COME_E4M3 || (out_scale_row_stride >= 0 && out_scale_block_stride >= 0)), "strides of scales must not be negative");
    COME_REQUIRE_MULTIPLES(4, {x_scale_dev, gate_scale_dev, up_scale_dev, gate_bias_dev, up_bias_dev, out_scale_dev});
    COME_REQUIRE_MULTIPLES(2, {out_dtype == COME_E4M3 ? nullptr : out_dev});
    come::MatmulArgs a = {};
    a.mode = come::kMatmulGated;
    a.e4m3 = true;
    a.M = tokens, a.N = features, a.K = channels;
    a.a[0] = x_dev, a.a_row[0] = x_row_stride;
    a.b[0] = gate_dev, a.b_row[0] = gate_row_stride;
    a.b[1] = up_dev, a.b_row[1] = up_row_stride;
    a.sums = a.problems = 1;
    a.a_scale = x_scale_dev, a.as_row = x_scale_row_stride, a.as_block = x_scale_block_stride;
    a.b_scale[0] = gate_scale_dev, a.bs_row[0] = gate_scale_row_stride;
    a.b_scale[1] = up_scale_dev, a.bs_row[1] = up_scale_row_stride;
    a.bias[0] = gate_bias_dev, a.bias[1] = up_bias_dev;
    a.act = activation;
    a.out[0] = out_dev, a.out_row[0] = out_row_stride;
    a.out_dtype = out_dtype;
    a.out_scale = out_scale_dev, a.os_row = out_scale_row_stride, a.os_block = out_scale_block_stride;
    return come::run_matmul(a, (cudaStream_t)stream);
}

static int gated_common(come::MatmulArgs &a, const void *x, int64_t x_row, const void *gate, int64_t gate_row, const void *up, int64_t up_row, const void *gate_bias,
                        const void *up_bias, int dtype, int activation, int64_t tokens, int64_t features, int64_t channels) {
    COME_REQUIRE_SIZES("come_gated_matmul", tokens, features, channels);
    COME_REQUIRE(come::is_16_bit(dtype), "the gated projections need float16 or bfloat16 (got dtype %d)", dtype);
    COME_REQUIRE(activation == COME_ACT_SILU || activation == COME_ACT_GELU, "unknown activation %d", activation);
    if (tokens == 0 || features == 0) return COME_OK;
    COME_REQUIRE_ROWS("x", x, x_row, 2, channels);
    COME_REQUIRE_ROWS("gate", gate, gate_row, 2, channels);
    COME_REQUIRE_ROWS("up", up, up_row, 2, channels);
    COME_REQUIRE_MULTIPLES(2, {gate_bias, up_bias});
    a.dtype = dtype;
    a.M = tokens, a.N = features, a.K = channels;
    a.a[0] = x, a.a_row[0] = x_row;
    a.b[0] = gate, a.b_row[0] = gate_row;
    a.b[1] = up, a.b_row[1] = up_row;
    a.bias[0] = gate_bias, a.bias[1] = up_bias;
    a.sums = a.problems = 1;
    a.act = activation;
    a.out_dtype = dtype;
    return COME_OK;
}

extern "C" int come_gated_matmul(const void *x_dev, int64_t x_row_stride, const void *gate_dev, int64_t gate_row_stride, const void *up_dev, int64_t up_row_stride,
                                 const void *gate_bias_dev, const void *up_bias_dev, int dtype, int activation, int64_t tokens, int64_t features,
                                 int64_t channels, void *out_dev, int64_t out_row_stride, void *stream) {
    come::MatmulArgs a = {};
    const int rc = gated_common(a, x_dev, x_row_stride, gate_dev, gate_row_stride, up_dev, up_row_stride, gate_bias_dev, up_bias_dev, dtype, activation, tokens, features, channels);
    if (rc != COME_OK || tokens == 0 || features == 0) return rc;
    COME_REQUIRE(out_dev && out_row_stride >= features, "out must be given, with a row stride that holds its rows");
    COME_REQUIRE_MULTIPLES(2, {out_dev});
    a.mode = come::kMatmulGated;
    a.out[0] = out_dev, a.out_row[0] = out_row_stride;
    return come::run_matmul(a, (cudaStream_t)stream);
}

// Gradients of few tokens, or of few elements, are sums of few rounded numbers: the error is the luck of some hundred roundings rather
// than their average (up to 1.7 times that of float32 operands after rounding, where large ones have 1.4).  There the operands keep a
// second 16-bit part, which doubles the contractions behind them.  Both sides of the rule, a step in a graph, two parts / one (bf16; error
// of dx and dW against float64 0.0017 / 0.0023 in every case): by elements, 261 / 262 tokens 392 -> 1003 45 / 40 us, 1000 tokens 64 ->
// 262 / 263 54 / 48, 95 / 96 tokens 2048 -> 2736 96 / 58; by tokens, 64 / 65 of 4096 -> 11,008 444 / 204.  Launched from Python the small
// ones take 135-143 us on either side.
extern "C" int64_t come_gated_backward_rows(int64_t tokens, int64_t features) {
    if (tokens <= 0) return 0;
    return tokens <= 64 || (features < (1ll << 18) && tokens < (1ll << 18) && tokens * features <= (1ll << 18)) ? 2 * tokens : tokens;
}

extern "C" int come_gated_matmul_backward_in_range(const void *x_dev, int64_t x_row_stride, const void *gate_dev, int64_t gate_row_stride, const void *up_dev, int64_t up_row_stride,
                                          const void *gate_bias_dev, const void *up_bias_dev, int dtype, int activation, int64_t tokens, int64_t features,
                                          int64_t channels, const void *dout_dev, int64_t dout_row_stride, void *dgate_dev, void *dup_dev, int64_t d_row_stride,
                                          void *dx_dev, int64_t dx_row_stride, void *dgate_weight_dev, void *dup_weight_dev, int64_t dw_row_stride,
                                          void *dgate_bias_dev, void *dup_bias_dev, float *range_dev,
                                                   void *stream) {
    using namespace come;
    cudaStream_t st = (cudaStream_t)stream;
    MatmulArgs a = {};
    int rc = gated_common(a, x_dev, x_row_stride, gate_dev, gate_row_stride, up_dev, up_row_stride, gate_bias_dev, up_bias_dev, dtype, activation, tokens, features, channels);
    if (rc != COME_OK) return rc;
    COME_REQUIRE(tokens > 0 && features > 0, "come_gated_matmul_backward: without tokens or features every gradient is zero or empty");
    COME_REQUIRE(dout_dev && dout_row_stride >= 0, "dout must be given");
    COME_REQUIRE_ROWS("dgate", dgate_dev, d_row_stride, 2, features);
    COME_REQUIRE_ROWS("dup", dup_dev, d_row_stride, 2, features);
    COME_REQUIRE(!dx_dev || dx_row_stride >= channels, "the row stride of dx must hold its rows");
    COME_REQUIRE((!dgate_weight_dev && !dup_weight_dev) || dw_row_stride >= channels, "the row stride of the weights' gradients must hold their rows");
    COME_REQUIRE(multiples_of(4, {range_dev}), "range_dev must be 4-byte aligned");
    COME_REQUIRE_MULTIPLES(2, {dout_dev, dx_dev, dgate_weight_dev, dup_weight_dev, dgate_bias_dev, dup_bias_dev});
    const uint32_t *range = dtype == COME_F16 ? (const uint32_t *)range_dev : nullptr;
    if (range && (rc = find_largest(dout_dev, tokens, features, dout_row_stride, (uint32_t *)range_dev, st)) != COME_OK) return rc;
    // the gradients of the projections
    a.mode = kMatmulGatedGrad;
    a.range = range;
    a.dh = dout_dev, a.dh_row = dout_row_stride;
    a.out[0] = dgate_dev, a.out[1] = dup_dev;
    a.out_row[0] = a.out_row[1] = d_row_stride;
    const int parts = (int)(come_gated_backward_rows(tokens, features) / tokens);
    a.low_rows = parts > 1 ? tokens : 0;
    const auto part = [&](const void *d, int i) { return (const void *)((const uint16_t *)d + i * tokens * d_row_stride); };
    if ((rc = run_matmul(a, st)) != COME_OK) return rc;
    if (dx_dev) {  // dx = dgate gate + dup up
        MatmulArgs b = {};
        b.dtype = b.out_dtype = dtype;
        b.range = range;
        b.b_mn = true;
        b.M = tokens, b.N = channels, b.K = features;
        for (int i = 0; i < 2 * parts; ++i) b.a[i] = part(i & 1 ? dup_dev : dgate_dev, i >> 1), b.a_row[i] = d_row_stride;
        b.b[0] = gate_dev, b.b_row[0] = gate_row_stride;
        b.b[1] = up_dev, b.b_row[1] = up_row_stride;
        b.sums = 2 * parts, b.problems = 1;
        b.out[0] = dx_dev, b.out_row[0] = dx_row_stride;
        if ((rc = run_matmul(b, st)) != COME_OK) return rc;
    }
    if (dgate_weight_dev || dup_weight_dev) {  // dgate^T x, dup^T x
        MatmulArgs b = {};
        b.dtype = b.out_dtype = dtype;
        b.range = range;
        b.a_mn = b.b_mn = true;
        b.M = features, b.N = channels, b.K = tokens;
        b.b[0] = x_dev, b.b_row[0] = x_row_stride;
        b.sums = parts;
        for (int i = 0; i < 2; ++i) {
            void *out = i ? dup_weight_dev : dgate_weight_dev;
            if (!out) continue;
            for (int j = 0; j < parts; ++j) b.a[b.problems * parts + j] = part(i ? dup_dev : dgate_dev, j), b.a_row[b.problems * parts + j] = d_row_stride;
            b.out[b.problems] = out, b.out_row[b.problems++] = dw_row_stride;
        }
        if ((rc = run_matmul(b, st)) != COME_OK) return rc;
    }
    if (dgate_bias_dev || dup_bias_dev) {
        const dim3 grid((unsigned)((features + 31) / 32), 2);
        const unsigned int *status = status_word_dev();
        if (!status) return COME_ERR_CUDA;
        if (dtype == COME_F16)
            column_sums_kernel<__half><<<grid, kSumThreads, 0, st>>>((const __half *)dgate_dev, (const __half *)dup_dev, d_row_stride, parts * tokens, (int)features, (__half *)dgate_bias_dev, (__half *)dup_bias_dev,
                                                                     status, range);
        else
            column_sums_kernel<__nv_bfloat16><<<grid, kSumThreads, 0, st>>>((const __nv_bfloat16 *)dgate_dev, (const __nv_bfloat16 *)dup_dev, d_row_stride, parts * tokens, (int)features,
                                                                            (__nv_bfloat16 *)dgate_bias_dev, (__nv_bfloat16 *)dup_bias_dev, status, range);
        return check_launch("come_gated_matmul_backward");
    }
    return COME_OK;
}

extern "C" int come_gated_matmul_backward(const void *x_dev, int64_t x_row_stride, const void *gate_dev, int64_t gate_row_stride, const void *up_dev, int64_t up_row_stride,
                                          const void *gate_bias_dev, const void *up_bias_dev, int dtype, int activation, int64_t tokens, int64_t features,
                                          int64_t channels, const void *dout_dev, int64_t dout_row_stride, void *dgate_dev, void *dup_dev, int64_t d_row_stride,
                                          void *dx_dev, int64_t dx_row_stride, void *dgate_weight_dev, void *dup_weight_dev, int64_t dw_row_stride,
                                          void *dgate_bias_dev, void *dup_bias_dev, void *stream) {
    return come_gated_matmul_backward_in_range(x_dev, x_row_stride, gate_dev, gate_row_stride, up_dev, up_row_stride, gate_bias_dev, up_bias_dev, dtype, activation, tokens, features,
                                                channels, dout_dev, dout_row_stride, dgate_dev, dup_dev, d_row_stride, dx_dev, dx_row_stride, dgate_weight_dev, dup_weight_dev, dw_row_stride,
                                                dgate_bias_dev, dup_bias_dev, nullptr, stream);
}

extern "C" int come_selftest_matmul_stall(const void *x_dev, const float *x_scale_dev, const void *gate_dev, const void *up_dev, const float *w_scale_dev, int64_t tokens,
                                          int64_t features, int64_t channels, int k_blocks, int ctas, int64_t ticks, void *out_dev, float *out_scale_dev, void *stream) {
    using namespace come;
    COME_REQUIRE(x_dev && gate_dev && up_dev && out_dev, "come_selftest_matmul_stall: x, gate, up and out must be given");
    COME_REQUIRE((x_scale_dev == nullptr) == (w_scale_dev == nullptr) && (x_scale_dev || !out_scale_dev), "come_selftest_matmul_stall: scales of both operands or of none, and no 8-bit result of 16-bit operands");
    COME_REQUIRE(tokens > 0 && tokens < (1 << 16) && features > 0 && features < (1 << 12) && features % 16 == 0 && channels > 0 && channels < (1 << 12) && channels % 128 == 0,
                 "come_selftest_matmul_stall: a small launch only (tokens below 2^16, features below 2^12 and a multiple of 16, channels below 2^12 and a multiple of 128)");
    COME_REQUIRE(k_blocks >= 0 && ctas > 0 && ctas < 256, "come_selftest_matmul_stall: k_blocks must not be negative, ctas a mask of up to 8 ranks");
    COME_REQUIRE(ticks > 0 && ticks <= (1ll << 26), "come_selftest_matmul_stall: ticks must be in (0, 2^26] (a fraction of a second)");
    const bool e4m3 = x_scale_dev != nullptr;
    const int size = e4m3 ? 1 : 2;
    COME_REQUIRE_ROWS("x", x_dev, channels, size, channels);
    COME_REQUIRE_ROWS("gate", gate_dev, channels, size, channels);
    COME_REQUIRE_ROWS("up", up_dev, channels, size, channels);
    COME_REQUIRE((uintptr_t)out_dev % 16 == 0, "come_selftest_matmul_stall: out must be 16-byte aligned");
    MatmulArgs a = {};
    a.mode = kMatmulGated;
    a.e4m3 = e4m3;
    a.dtype = COME_BF16;
    a.M = tokens, a.N = features, a.K = channels;
    a.a[0] = x_dev, a.b[0] = gate_dev, a.b[1] = up_dev;
    a.a_row[0] = a.b_row[0] = a.b_row[1] = channels;
    a.sums = a.problems = 1;
    a.a_scale = x_scale_dev, a.as_row = channels / kScaleBlock, a.as_block = 1;
    a.b_scale[0] = a.b_scale[1] = w_scale_dev, a.bs_row[0] = a.bs_row[1] = channels / kScaleBlock;
    a.act = COME_ACT_SILU;
    a.out[0] = out_dev, a.out_row[0] = features;
    a.out_dtype = out_scale_dev ? (int)COME_E4M3 : (int)COME_BF16;
    a.out_scale = out_scale_dev, a.os_row = (features + kScaleBlock - 1) / kScaleBlock, a.os_block = 1;
    a.wait_limit = ticks;
    a.stall_block = k_blocks;
    a.stall_ctas = (uint32_t)ctas;
    return run_matmul(a, (cudaStream_t)stream);
}

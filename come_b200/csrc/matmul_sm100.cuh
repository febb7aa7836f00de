// Products of the feed-forward half of a block: the problem a launch computes, and what its two kernels share.
//
//   out[m, n] = f( sum_k A[m, k] B[n, k] )       A: tokens (or the gradient of the projections), B: weights
//
// Operands are tiles of 128-byte rows (128-byte swizzle) that TMA brings to shared memory: 128 e4m3 or 64 16-bit numbers of the
// contraction per K block, or, where a 16-bit operand is stored with the contraction as its rows ("MN-major": x and W in the backward
// products), 64 contraction rows of 64 neighbouring m or n.  Both forms are read by tcgen05.mma as they lie.
#pragma once
#include "block_scale.cuh"
#include "sm100_ptx.cuh"

namespace come {

// What becomes of the sums.
enum MatmulMode : int {
    kMatmulPlain = 0,      // out = sum (+ bias)
    kMatmulGated = 1,      // two weights: out = act(gate) * up, in out_dtype or in 8 bits with scales
    kMatmulGatedGrad = 2,  // two weights and dh: out = dh * up * act'(gate), out2 = dh * act(gate)
};
struct MatmulArgs {
    int mode;
    bool e4m3;             // 8-bit operands with scales, else 16-bit ones of `dtype`
    int dtype;
    bool a_mn, b_mn;       // operand stored with the contraction as its rows (16 bits)
    int64_t M, N, K;
    // Operands.  `sums` contractions that are added and `problems` of them (plain mode): a[problem * sums + sum] times b[sum & 1], or times
    // b[0] where both are stored with the contraction as their rows; or two weights b[0], b[1] of one a[0] (gated modes).
    const void *a[4], *b[2];
    int64_t a_row[4], b_row[2];  // row strides in elements
    int sums, problems;
    int64_t low_rows;            // gated gradient: what rounding took from row r of a result goes to row r + low_rows; 0: nowhere
    // Scales of 8-bit operands: of a[0] per row and 128 contraction elements, of b[i] per 128 x 128 block.
    const float *a_scale, *b_scale[2];
    int64_t as_row, as_block, bs_row[2];
    const void *bias[2];         // float32 (8-bit operands) or `dtype`; NULL: none
    int act;
    const void *dh;              // gated gradient: `dtype`
    int64_t dh_row;
    const uint32_t *range;       // float16 gradients: bits of the largest |dh| as float32 (see range_factor); NULL: taken as they are
    void *out[2];
    int64_t out_row[2];
    int out_dtype;
    float *out_scale;            // 8-bit result: per row and 128 columns
    int64_t os_row, os_block;
    long long wait_limit;        // self-test: clock ticks after which a wait gives up; 0: an ordinary launch
    int stall_block;             // ... K block, counted over a CTA's life, before which the producers of `stall_ctas` stop
    uint32_t stall_ctas;         // ... ranks of a cluster, as bits
};

constexpr int kTile = 128;
constexpr int kKBytes = 128;                       // bytes of the contraction per K block
constexpr int kOperandBytes = kTile * kKBytes;     // 16 KiB: 128 rows of a K block

// What a launch of either kernel gets.
struct MatmulParams {
    CUtensorMap a[4], b[2];
    const float *a_scale, *b_scale[2];
    int64_t as_row, as_block, bs_row[2];
    const void *bias[2], *dh;
    const uint32_t *range;
    void *out[2];
    float *out_scale;
    int64_t dh_row, out_row[2], os_row, os_block;
    int64_t low_rows;
    int M, N, sums, kb_per_sum, k_blocks;  // K blocks of one contraction, of all
    int tiles_m, tiles_n, problems;   // grid of tiles of one problem
    int act, dtype, bias_dtype, out_dtype;
    unsigned int *status;
    long long wait_limit;  // self-test only, as in MatmulArgs
    int stall_block;
    uint32_t stall_ctas;
};

// The kernel for results with many tiles (matmul_pair_sm100.cu).
bool matmul_pair_takes(const MatmulArgs &a);
int matmul_pair_launch(const MatmulArgs &a, MatmulParams &p, cudaStream_t st);

// ---- host ---------------------------------------------------------------------------------------------------------------
// 2-D tensor map of rows of `inner` elements; box of `box_rows` rows of 128 bytes, 128-byte swizzle, zeros outside.
inline int make_rows_map(CUtensorMap *map, const void *base, bool e4m3, int dtype, int64_t rows, int64_t inner, int64_t row_stride, int box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) {
        set_error("cuTensorMapEncodeTiled is not available from the CUDA driver");
        return COME_ERR_CUDA;
    }
    const int size = e4m3 ? 1 : 2;
    cuuint64_t dims[2] = {(cuuint64_t)inner, (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)(row_stride * size)};
    cuuint32_t box[2] = {(cuuint32_t)(128 / size), (cuuint32_t)box_rows};
    cuuint32_t estr[2] = {1, 1};
    const CUtensorMapDataType type = e4m3 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : dtype == COME_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const auto encode = [&] {
        return fn(map, type, 2, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    };
    CUresult r = encode();
    if (r == CUDA_ERROR_INVALID_CONTEXT) {  // a host thread that has made no runtime call yet (an autograd worker): bind its device
        int dev = 0;
        COME_CUDA(cudaGetDevice(&dev));
        COME_CUDA(cudaSetDevice(dev));
        r = encode();
    }
    if (r != CUDA_SUCCESS) {
        set_error("cuTensorMapEncodeTiled failed with CUresult %d", (int)r);
        return COME_ERR_CUDA;
    }
    return COME_OK;
}

// The shared-memory opt-in of a kernel, once per device and instantiation and before its first launch (launches stay cheap and
// legal inside a stream capture).
template <auto kernel> int allow_smem(size_t bytes) {
    static std::mutex mu;
    static bool done[64];
    int dev = 0;
    COME_CUDA(cudaGetDevice(&dev));
    COME_REQUIRE(dev >= 0 && dev < 64, "device ordinal %d is out of the supported range", dev);
    std::lock_guard<std::mutex> lock(mu);
    if (done[dev]) return COME_OK;
    COME_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done[dev] = true;
    return COME_OK;
}

// ---- device -------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int x, int y, uint64_t *bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) { asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory"); }

__device__ __forceinline__ void tc_mma_f8_ss_1(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// Shared-memory matrix descriptor of an operand tile of 128-byte rows (128-byte swizzle, 8-row groups of 1024 bytes).  K-major:
// rows are m or n, a K step of 32 bytes advances the start address by 32.  MN-major: rows are contraction indexes, 64 m or n each;
// further 64s of m or n lie `mn_stride` bytes on, a K step of 16 rows advances the start address by 2048.
__device__ __forceinline__ uint64_t operand_desc(uint32_t saddr, uint32_t mn_stride) {
    return (uint64_t)((saddr & 0x3FFFF) >> 4) | ((uint64_t)((mn_stride >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// Instruction descriptor: float32 sums; 16-bit operands of one type, or e4m3 (format code 0).
__host__ __device__ constexpr uint32_t matmul_idesc(bool e4m3, bool bf16, int M, int N, bool a_mn, bool b_mn) {
    const uint32_t format = !e4m3 && bf16 ? 1u : 0u;
    return (1u << 4) | (format << 7) | (format << 10) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
           ((uint32_t)(M >> 4) << 24);
}

__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_rank(uint32_t saddr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(saddr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 ld_cluster(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ uint32_t ld_cluster_u32(uint32_t addr) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}

__device__ __forceinline__ void st_cluster_u32(uint32_t addr, uint32_t v) { asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory"); }

enum : uint32_t { kErrFull = 1u << 19, kErrEmpty = 1u << 20, kErrSums = 1u << 21 };
static_assert((kErrFull | kErrEmpty | kErrSums) == kStatusMatmul, "come_device_status names these bits");


// act(g) and its derivative.  silu: g s with s = 1 / (1 + e^-g), derivative s (1 + g (1 - s)); gelu: g Phi(g), derivative
// Phi(g) + g phi(g).  The logistic function is one exponential and one reciprocal of the special-function unit, each good to about
// 2^-22 (denormals flushed: where e^-g leaves the range, s is 0 or 1 to float32), so that an element costs six instructions.
__device__ __forceinline__ float logistic(float g) {
    float e, s;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(s) : "f"(1.0f + e));
    return s;
}
__device__ __forceinline__ float activation(float g, int act) {
    if (act == COME_ACT_SILU) return g * logistic(g);
    return 0.5f * g * erfcf(g * -0.70710678118654752f);
}
__device__ __forceinline__ void activation_grad(float g, int act, float &value, float &slope) {
    if (act == COME_ACT_SILU) {
        const float s = logistic(g);
        value = g * s;
        slope = fmaf(value, 1.0f - s, s);
    } else {
        const float phi = 0.3989422804014327f * __expf(-0.5f * g * g);
        const float cdf = 0.5f * erfcf(g * -0.70710678118654752f);
        value = g * cdf;
        slope = fmaf(g, phi, cdf);
    }
}

// The power of two that float16 gradients of the projections, which lie around dh, are held times, and its inverse.  Where the largest
// |dh| is below 1/2 it is brought to [1/2, 1): those of a mean over many elements would fall below the type's smallest number.  From
// 2^10 on it is brought to [2^9, 2^10): times the other projection they would pass the type's largest, while the gradients that they
// become would not.  In between, where neither is near, they stay as they are: making room for one token's would cost the others digits.
// Nothing is scaled where the largest is zero, infinite or no number.
__device__ __forceinline__ float range_factor(const uint32_t *range, bool inverse) {
    const uint32_t bits = range ? __ldg(range) : 0u, e = bits >> 23;  // exponent, biased by 127
    const uint32_t want = bits == 0 || e == 255 ? e : e < 126 ? 126 : e > 136 ? 136 : e;
    return __uint_as_float((inverse ? 127 + e - want : 127 + want - e) << 23);
}

__device__ __forceinline__ float load_any(const void *p, int64_t i, int dtype) {
    if (dtype == COME_F32) return ((const float *)p)[i];
    if (dtype == COME_F16) return __half2float(((const __half *)p)[i]);
    return __bfloat162float(((const __nv_bfloat16 *)p)[i]);
}
template <bool kBF16> __device__ __forceinline__ uint32_t pack_16(float lo, float hi) {
    if constexpr (kBF16) {
        __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    } else {
        __half2 v = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<uint32_t *>(&v);
    }
}

}  // namespace come

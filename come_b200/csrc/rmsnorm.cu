// Residual add fused with the root-mean-square norm behind it, and the 8-bit quantisers of the block-scaled products.
//
//   x_out  = x + scale * branch                        (float32, rounded once to the stream's type)
//   y      = x_out * rsqrt(mean(x_out^2) + eps) * weight   (float32, of the stream as it is stored)
//   normed = y rounded to the stream's type, or
//   q      = e4m3(y / s),  s = max(max|y|, 448 * 2^-126) / 448 over each 128 columns of a row
//
// Memory bound: both inputs are read once, both results written once.  A row is owned by a group of threads: a quarter of a warp or half
// of one (narrow rows), a warp, or several (few rows, where a row's latency counts, and wide rows, whose registers would not fit one
// warp).  Thread i of the group holds the vectors i, i + group size, ... of the row, so the 128 columns of a scale always lie in 16
// (16-bit types) or 32 (float32) neighbouring lanes, or are the whole row, and their maximum needs shuffles only.
//
// Measured: 80,672 x 1024 bf16 with residual and 8-bit result 114 us (5.1 TB/s, 78 % of the copy rate; with a bf16 result 108 us, 6.1
// TB/s), 10,534 x 1000 float32 28.7 us (5.9 TB/s).  The quantiser alone: 80,672 x 1024 bf16 60 us (4.2 TB/s), 8192 x 28,672 in pieces 187 us
// (3.8 TB/s).
#include "block_scale.cuh"

namespace come {

namespace {

struct RmsNormArgs {
    const void *x, *branch, *scale, *weight;
    int64_t rows, x_row;  // row stride of x in elements; branch, x_out and normed are contiguous
    int C;
    float eps, inv_C;
    bool norm;            // off: quantise x as it is
    void *x_out, *normed;
    uint8_t *q;
    int64_t q_row;
    float *q_scale;
    int64_t s_row, s_block;
    int64_t chunks;       // quantiser of wide rows: pieces of a row
};

// VEC elements of a row from column c on as 16 raw bytes; kAligned: one access, the row's width is a whole number of them.  kOnce: a
// row that is read once, against the scale and weight vectors that every row reads.
template <typename T, int VEC, bool kAligned, bool kOnce> __device__ __forceinline__ uint4 load_raw(const T *p, int c, int C) {
    if constexpr (kAligned) {
        return kOnce ? __ldcs(reinterpret_cast<const uint4 *>(p + c)) : __ldg(reinterpret_cast<const uint4 *>(p + c));
    } else {
        uint4 raw = make_uint4(0, 0, 0, 0);
        T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < C) e[i] = p[c + i];
        return raw;
    }
}
template <typename T, int VEC> __device__ __forceinline__ void unpack_raw(const uint4 &raw, float (&v)[VEC]) {
    const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[i] = Elem<T>::to_f32(e[i]);
}
template <typename T, int VEC> __device__ __forceinline__ uint4 pack_raw(const float (&v)[VEC]) {
    uint4 raw;
    T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
    for (int i = 0; i < VEC; ++i) e[i] = Elem<T>::from_f32(v[i]);
    return raw;
}
template <typename T, int VEC, bool kAligned> __device__ __forceinline__ void store_raw(T *p, int c, int C, const uint4 &raw) {
    if constexpr (kAligned) {
        __stcs(reinterpret_cast<uint4 *>(p + c), raw);
    } else {
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < C) p[c + i] = e[i];
    }
}

template <int VEC> __device__ __forceinline__ void store_e4m3(uint8_t *p, int c, int C, const float (&v)[VEC], float inv) {
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) w[i] = pack_e4m3(v[4 * i] * inv, v[4 * i + 1] * inv, v[4 * i + 2] * inv, v[4 * i + 3] * inv);
    if (c + VEC <= C) {  // rows are stored with a stride of whole 16 bytes
        if constexpr (VEC == 8) *reinterpret_cast<uint2 *>(p + c) = make_uint2(w[0], w[1]);
        else *reinterpret_cast<uint32_t *>(p + c) = w[0];
    } else {
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (c + i < C) p[c + i] = (uint8_t)(w[i / 4] >> (8 * (i & 3)));
    }
}

// kGroup threads own a row (part of a warp, or whole warps); a CTA of kThreads threads holds kThreads / kGroup of them.  kChunked: they own
// a piece of kGroup * NV vectors of a row instead, which is a whole number of scales: the quantiser alone needs no more of it.
template <typename T, int kGroup, int NV, int kThreads, bool kAligned, bool kChunked>
__global__ void __launch_bounds__(kThreads) residual_rmsnorm_kernel(const RmsNormArgs a) {
    constexpr int VEC = 16 / sizeof(T), kGroups = kThreads / kGroup, kSpan = kGroup * VEC;
    constexpr int kWarps = kGroup / 32, kPerWarp = kGroup < 32 ? 32 / kGroup : 1;  // warps per row, rows per warp
    __shared__ float part[kWarps > 1 ? kWarps : 1];
    const int lane = threadIdx.x & 31, warp = threadIdx.x % kGroup / 32, c0 = threadIdx.x % kGroup * VEC;
    const T *scale = (const T *)a.scale, *weight = (const T *)a.weight;
    // the loop is the warp's: rows past the last one have no columns
    int64_t first = (int64_t)blockIdx.x * kGroups + (kGroup < 32 ? threadIdx.x / 32 * kPerWarp : threadIdx.x / kGroup);
    const int64_t rows = kChunked ? a.rows * a.chunks : a.rows;
    for (; first < rows; first += (int64_t)gridDim.x * kGroups) {
        static_assert(!kChunked || (kGroup >= 32 && kSpan * NV % kScaleBlock == 0), "");
        const int64_t row = kChunked ? first / a.chunks : first + (kGroup < 32 ? lane / kGroup : 0);
        const int col0 = kChunked ? (int)(first - row * a.chunks) * (kSpan * NV) : 0;
        const int C = row >= a.rows ? 0 : kChunked ? min(a.C - col0, kSpan * NV) : a.C;
        const T *x = (const T *)a.x + row * a.x_row + col0;
        uint4 rx[NV], rb[NV];  // everything that a row reads is asked for before anything is used
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            rx[j] = make_uint4(0, 0, 0, 0);
            if (c0 + j * kSpan < C) rx[j] = load_raw<T, VEC, kAligned, true>(x, c0 + j * kSpan, C);
        }
        if (a.branch) {
            const T *branch = (const T *)a.branch + row * a.C;
#pragma unroll
            for (int j = 0; j < NV; ++j)
                if (c0 + j * kSpan < C) rb[j] = load_raw<T, VEC, kAligned, true>(branch, c0 + j * kSpan, C);
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = c0 + j * kSpan;
                if (c < C) {
                    float s[VEC], b[VEC];
                    unpack_raw<T, VEC>(rx[j], s);
                    unpack_raw<T, VEC>(rb[j], b);
                    if (scale) {
                        float g[VEC];
                        unpack_raw<T, VEC>(load_raw<T, VEC, kAligned, false>(scale, c, C), g);
#pragma unroll
                        for (int i = 0; i < VEC; ++i) s[i] = fmaf(b[i], g[i], s[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < VEC; ++i) s[i] += b[i];
                    }
                    rx[j] = pack_raw<T, VEC>(s);  // the norm is that of the stream as the next block reads it
                    if (a.x_out) store_raw<T, VEC, kAligned>((T *)a.x_out + row * a.C, c, C, rx[j]);
                }
            }
        }
        if (!a.normed && !a.q) continue;
        // From here on a row is its raw bytes, unpacked once for the sum and once for the result: registers are what limits the rows in
        // flight.
        float rstd = 1.0f;
        if (a.norm) {
            float sum = 0.0f;
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                float v[VEC];
                unpack_raw<T, VEC>(rx[j], v);
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum = fmaf(v[i], v[i], sum);
            }
#pragma unroll
            for (int m = (kGroup < 32 ? kGroup : 32) / 2; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
            if constexpr (kWarps > 1) {  // one group per CTA: a whole-CTA barrier
                static_assert(kGroups == 1, "the barrier below is the CTA's");
                if (lane == 0) part[warp] = sum;
                __syncthreads();
                sum = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) sum += part[w];
                __syncthreads();
            }
            rstd = rsqrtf(fmaf(sum, a.inv_C, a.eps));
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = c0 + j * kSpan;
            float v[VEC];
            unpack_raw<T, VEC>(rx[j], v);
            if (a.norm) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) v[i] *= rstd;
                if (weight && c < C) {
                    float w[VEC];
                    unpack_raw<T, VEC>(load_raw<T, VEC, kAligned, false>(weight, c, C), w);
#pragma unroll
                    for (int i = 0; i < VEC; ++i) v[i] *= w[i];
                }
            }
            if (a.normed) {
                if (c < C) store_raw<T, VEC, kAligned>((T *)a.normed + row * a.C, c, C, pack_raw<T, VEC>(v));
            } else {
                float top = 0.0f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) top = fmaxf(top, fabsf(v[i]));
#pragma unroll
                for (int m = (kGroup < kScaleBlock / VEC ? kGroup : kScaleBlock / VEC) / 2; m >= 1; m >>= 1)
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
                top = fmaxf(top, kSmallestMax);
                if (c < C) {
                    store_e4m3<VEC>(a.q + row * a.q_row + col0, c, C, v, inverse_scale(top));
                    if (c % kScaleBlock == 0) a.q_scale[row * a.s_row + ((col0 + c) / kScaleBlock) * a.s_block] = top * (1.0f / kE4m3Max);
                }
            }
        }
    }
}

template <typename T, bool kAligned> int launch_rmsnorm(const RmsNormArgs &a, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    const int64_t vectors = ((int64_t)a.C + VEC - 1) / VEC;
    const int64_t sms = sm_count();
    const auto grid = [&](int64_t blocks, int64_t per_sm) { return (unsigned)(blocks < sms * per_sm ? blocks : sms * per_sm); };
#define COME_RMS_LAUNCH(GROUP, NV, THREADS, PER_SM)                                                                       \
    residual_rmsnorm_kernel<T, GROUP, NV, THREADS, kAligned, false>                                                       \
        <<<grid((a.rows * GROUP + THREADS - 1) / THREADS, PER_SM), THREADS, 0, st>>>(a)
    // A warp per row up to 128 vectors, four from there on: 80,672 x 1024 bf16 (128 vectors) 114 / 134 us with one / four, 10,534 x 1000
    // float32 (250 vectors) 35 / 29.  Up to 16 vectors a warp holds two or four rows, so that its lanes have work: 1,875,000 x 64 bf16
    // (8 vectors) 471 / 164 us with one / four, 937,500 x 64 float32 (16 vectors) 229 / 161 with one / two.  Few rows take four or eight
    // warps each: a row's latency counts there.
    if (a.q && !a.norm && vectors > 2048) {  // the quantiser, of rows wider than a norm's: a warp per 128 vectors
        RmsNormArgs b = a;
        b.chunks = (vectors + 127) / 128;
        residual_rmsnorm_kernel<T, 32, 4, 128, kAligned, true><<<grid((b.rows * b.chunks + 3) / 4, 8), 128, 0, st>>>(b);
    } else if (vectors > 4 * 128 || (a.rows <= 4 * sms && vectors > 32)) {
        if (vectors <= 128) COME_RMS_LAUNCH(128, 1, 128, 16);
        else if (vectors <= 256) COME_RMS_LAUNCH(256, 1, 256, 8);
        else if (vectors <= 512) COME_RMS_LAUNCH(256, 2, 256, 6);
        else if (vectors <= 1024) COME_RMS_LAUNCH(256, 4, 256, 4);
        else if (vectors <= 2048) COME_RMS_LAUNCH(256, 8, 256, 2);
        else {
            set_error("come_residual_rmsnorm: rows of at most %d elements of this type (got %d)", 2048 * VEC, a.C);
            return COME_ERR_UNSUPPORTED;
        }
    } else if (vectors <= 8) COME_RMS_LAUNCH(8, 1, 128, 16);
    else if (vectors <= 16) COME_RMS_LAUNCH(16, 1, 128, 16);
    else if (vectors <= 32) COME_RMS_LAUNCH(32, 1, 128, 16);
    else if (vectors <= 64) COME_RMS_LAUNCH(32, 2, 128, 12);
    else if (vectors <= 128) COME_RMS_LAUNCH(32, 4, 128, 8);
    else if (vectors <= 256) COME_RMS_LAUNCH(128, 2, 128, 1 << 20);
    else COME_RMS_LAUNCH(128, 4, 128, 8);
#undef COME_RMS_LAUNCH
    return check_launch("come_residual_rmsnorm");
}

template <typename T> int dispatch_rmsnorm(const RmsNormArgs &a, cudaStream_t st) {
    constexpr int VEC = 16 / sizeof(T);
    const auto al = [](const void *p) { return (uintptr_t)p % 16 == 0; };
    const bool aligned = a.C % VEC == 0 && a.x_row % VEC == 0 && al(a.x) && al(a.branch) && al(a.scale) && al(a.weight) && al(a.x_out) && al(a.normed);
    return aligned ? launch_rmsnorm<T, true>(a, st) : launch_rmsnorm<T, false>(a, st);
}

// One CTA per 128 x 128 block of a weight, blocks of a row of blocks next to each other.  Once per weight, so the plain form: two passes of
// scalar loads, the second from L2 (2736 x 1024 float32 7 us, 28,672 x 8192 bf16 228 us, 3.1 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const T *__restrict__ w, int64_t w_row, int rows, int C, uint8_t *__restrict__ q,
                                                              int64_t q_row, float *__restrict__ q_scale, int64_t s_row) {
    __shared__ float tops[8];
    const int col_blocks = (int)(((unsigned)C + kScaleBlock - 1) / kScaleBlock), row_block = blockIdx.x / col_blocks, col_block = blockIdx.x % col_blocks;
    const int64_t r0 = (int64_t)row_block * kScaleBlock, r_end = min((int64_t)rows, r0 + kScaleBlock);
    const int c = col_block * kScaleBlock + (threadIdx.x & 127);
    float top = 0.0f;
    if (c < C)
        for (int64_t r = r0 + (threadIdx.x >> 7); r < r_end; r += 2) top = fmaxf(top, fabsf(Elem<T>::to_f32(w[r * w_row + c])));
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();
    top = kSmallestMax;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = fmaxf(top, tops[i]);
    if (threadIdx.x == 0) q_scale[row_block * s_row + col_block] = top / kE4m3Max;
    const float inv = kE4m3Max / top;
    if (c < C)
        for (int64_t r = r0 + (threadIdx.x >> 7); r < r_end; r += 2)
            q[r * q_row + c] = __nv_cvt_float_to_fp8(Elem<T>::to_f32(w[r * w_row + c]) * inv, __NV_SATFINITE, __NV_E4M3);
}

int run_rmsnorm(const RmsNormArgs &a, int dtype, cudaStream_t st) {
    switch (dtype) {
        case COME_F32: return dispatch_rmsnorm<float>(a, st);
        case COME_F16: return dispatch_rmsnorm<__half>(a, st);
        default: return dispatch_rmsnorm<__nv_bfloat16>(a, st);
    }
}

}  // namespace

}  // namespace come

extern "C" int come_residual_rmsnorm(const void *x_dev, const void *branch_dev, const void *scale_dev, int64_t rows, int64_t channels, int dtype,
                                     const void *weight_dev, float eps, void *x_out_dev, void *normed_dev, void *q_dev, int64_t q_row_stride,
                                     float *q_scale_dev, int64_t q_scale_row_stride, int64_t q_scale_block_stride, void *stream) {
    COME_REQUIRE(rows >= 0 && channels >= 0, "rows and channels must be >= 0");
    COME_REQUIRE(dtype == COME_F32 || dtype == COME_F16 || dtype == COME_BF16, "unknown dtype %d", dtype);
    COME_REQUIRE(rows < (1ll << 31) && channels < (1ll << 31), "rows and channels must fit int32");
    if (rows == 0 || channels == 0) return COME_OK;
    COME_REQUIRE(x_dev != nullptr, "x must not be NULL");
    COME_REQUIRE(branch_dev || !scale_dev, "scale without a branch");
    COME_REQUIRE(!x_out_dev || branch_dev, "x_out without a branch");
    COME_REQUIRE(!normed_dev || !q_dev, "the norm is written once: in the stream's type or in 8 bits");
    COME_REQUIRE(normed_dev || q_dev || x_out_dev, "nothing to write");
    COME_REQUIRE(!q_dev || (q_scale_dev && q_row_stride >= channels && q_row_stride % 16 == 0 && (uintptr_t)q_dev % 16 == 0),
                 "an 8-bit result needs its scales, 16-byte aligned rows and a row stride of whole 16 bytes");
    COME_REQUIRE(come::multiples_of(come::dtype_size(dtype), {x_dev, branch_dev, scale_dev, weight_dev, x_out_dev, normed_dev}) && come::multiples_of(4, {q_scale_dev}),
                 "addresses must be multiples of their elements' size");
    COME_REQUIRE(q_scale_row_stride >= 0 && q_scale_block_stride >= 0, "strides of scales must not be negative");
    come::RmsNormArgs a = {};
    a.x = x_dev;
    a.branch = branch_dev;
    a.scale = scale_dev;
    a.weight = weight_dev;
    a.rows = rows;
    a.x_row = channels;
    a.C = (int)channels;
    a.eps = eps;
    a.inv_C = 1.0f / (float)channels;
    a.norm = normed_dev || q_dev;
    a.x_out = x_out_dev;
    a.normed = normed_dev;
    a.q = (uint8_t *)q_dev;
    a.q_row = q_row_stride;
    a.q_scale = q_scale_dev;
    a.s_row = q_scale_row_stride;
    a.s_block = q_scale_block_stride;
    return come::run_rmsnorm(a, dtype, (cudaStream_t)stream);
}

extern "C" int come_quantize_rows(const void *x_dev, int dtype, int64_t rows, int64_t channels, int64_t x_row_stride, void *q_dev, int64_t q_row_stride,
                                  float *q_scale_dev, int64_t q_scale_row_stride, int64_t q_scale_block_stride, void *stream) {
    COME_REQUIRE(rows >= 0 && channels >= 0, "rows and channels must be >= 0");
    COME_REQUIRE(dtype == COME_F32 || dtype == COME_F16 || dtype == COME_BF16, "unknown dtype %d", dtype);
    COME_REQUIRE(rows < (1ll << 31) && channels < (1ll << 31), "rows and channels must fit int32");
    if (rows == 0 || channels == 0) return COME_OK;
    COME_REQUIRE(x_dev && q_dev && q_scale_dev, "x, q and q_scale must not be NULL");
    COME_REQUIRE(x_row_stride >= 0 && q_scale_row_stride >= 0 && q_scale_block_stride >= 0, "strides must not be negative");
    COME_REQUIRE(come::multiples_of(come::dtype_size(dtype), {x_dev}) && come::multiples_of(4, {q_scale_dev}), "addresses must be multiples of their elements' size");
    COME_REQUIRE(q_row_stride >= channels && q_row_stride % 16 == 0 && (uintptr_t)q_dev % 16 == 0, "q needs 16-byte aligned rows and a row stride of whole 16 bytes");
    come::RmsNormArgs a = {};
    a.x = x_dev;
    a.rows = rows;
    a.x_row = x_row_stride;
    a.C = (int)channels;
    a.q = (uint8_t *)q_dev;
    a.q_row = q_row_stride;
    a.q_scale = q_scale_dev;
    a.s_row = q_scale_row_stride;
    a.s_block = q_scale_block_stride;
    return come::run_rmsnorm(a, dtype, (cudaStream_t)stream);
}

extern "C" int come_quantize_weight(const void *w_dev, int dtype, int64_t rows, int64_t channels, int64_t w_row_stride, void *q_dev, int64_t q_row_stride,
                                    float *q_scale_dev, int64_t q_scale_row_stride, void *stream) {
    COME_REQUIRE(rows >= 0 && channels >= 0, "rows and channels must be >= 0");
    COME_REQUIRE(dtype == COME_F32 || dtype == COME_F16 || dtype == COME_BF16, "unknown dtype %d", dtype);
    COME_REQUIRE(rows < (1ll << 31) && channels < (1ll << 31) - come::kScaleBlock, "rows and channels must fit int32");
    if (rows == 0 || channels == 0) return COME_OK;
    COME_REQUIRE(w_dev && q_dev && q_scale_dev, "w, q and q_scale must not be NULL");
    COME_REQUIRE(w_row_stride >= 0 && q_row_stride >= channels && q_scale_row_stride >= 0, "bad strides");
    COME_REQUIRE(come::multiples_of(come::dtype_size(dtype), {w_dev}) && come::multiples_of(4, {q_scale_dev}), "addresses must be multiples of their elements' size");
    const int64_t grid = ((channels + come::kScaleBlock - 1) / come::kScaleBlock) * ((rows + come::kScaleBlock - 1) / come::kScaleBlock);
    COME_REQUIRE(grid < (1ll << 31), "a weight of %lld blocks of 128 x 128 is too large for one launch", (long long)grid);
    cudaStream_t st = (cudaStream_t)stream;
#define COME_QW_LAUNCH(T)                                                                                                              \
    come::quantize_weight_kernel<T><<<(unsigned)grid, 256, 0, st>>>((const T *)w_dev, w_row_stride, (int)rows, (int)channels, (uint8_t *)q_dev, \
                                                          q_row_stride, q_scale_dev, q_scale_row_stride)
    if (dtype == COME_F32) COME_QW_LAUNCH(float);
    else if (dtype == COME_F16) COME_QW_LAUNCH(__half);
    else COME_QW_LAUNCH(__nv_bfloat16);
#undef COME_QW_LAUNCH
    return come::check_launch("come_quantize_weight");
}

// Products of the feed-forward half of a block on Blackwell tensor cores (sm_100a): the kernel for results with many tiles.
//
// Persistent: one pair of CTAs (two SMs, tcgen05 cta_group::2) per 256 x 256 tile of sums (256 rows x 128 columns of both projections in
// the gated forms), tiles dealt to the pairs in turn.  CTA c of a pair holds rows [128 c, + 128) of A, half of B (columns [128 c, + 128), or
// the gate's / the up projection's weight) and the sums of its rows.
//
//   warps 0-7 : two epilogue warpgroups of 128 rows each, columns [0, 128) / [128, 256) of the tile, or in the gated forms columns [0, 64) /
//               [64, 128) of both projections, so that gate and up of an element meet in one thread.  8-bit operands: every K block of
//               128 is a product of its own in one of two TMEM buffers, scaled and added to float32 registers (two sums per instruction)
//               while the tensor cores fill the other.  16-bit operands: a tile's sums stay in TMEM; the two buffers let the next tile
//               begin under this one's epilogue.  Results are staged in 4 KB of shared memory per warp and leave as whole 128-byte rows.
//   warp 8    : producer (TMA ring, one per CTA; the loads of both CTAs complete on the first CTA's barriers).
//   warp 9    : MMA issuer (first CTA only).
//   warps 10, 11 : 8-bit operands: the scales of a K block, row x column block, two blocks ahead.
//
// What it measures and what bounds it.  8-bit operands: the hand-over of a K block, about 950 clocks where its product takes 512 (two TMEM
// buffers are all there is), then the 1 kW cap: 80,672 tokens 2736 -> 1024 313 us sustained (1450 TFLOP/s), 277 cold; gated 1024 -> 2736
// 624 us (1450), of which a tile's end is 4500 of 11,000 clocks.  What cost most on the way: an arrival with cluster release per K block
// (8192 x 16,384 x 2048: 703 us, 320 without), operands of the issuer in ordinary registers (430-550 clocks for six instructions, 180
// in uniform ones), spilled registers in the scaling loop (10-15 %).  16-bit operands: the tensor pipe, at the power cap when sustained
// (8192 x 8192 -> 2 x 2736: 1278 TFLOP/s).
//
// Why pairs: a 128 x 256 tile of one CTA reads 12 KB of shared memory per 128 x 256 x 32-byte step and TMA writes as much again, more than
// the 128 bytes per clock of an SM let pass in the step's 128 clocks; in a pair each SM holds half of B.
//
// Every wait is bounded as in matmul_sm100.cu: after one gave up, the CTA's roles go on without acting, its abort flag keeps it from
// storing, and the pair meets at the last cluster barrier.  A CTA leaves when everything that signals or writes to it has landed: loads
// and arrivals are waited for, or, after a wait gave up, given a few milliseconds.
#include "matmul_sm100.cuh"

#include <type_traits>

namespace come {

namespace {

constexpr int kProducerWarp = 8, kIssuerWarp = 9, kThreads = 384;  // three warpgroups
constexpr int kPairN = 256;                         // columns of sums per tile (192 and 128 were slower wherever they gave fuller rounds)
constexpr int kStageBytes = 2 * kOperandBytes;      // 128 rows of A and of B
constexpr int kStages = 6;
constexpr int kRingBytes = kStages * kStageBytes;
__host__ __device__ constexpr int staging_row(bool e4m3) { return e4m3 ? 64 : 128; }                // bytes; 8-bit operands: the other half holds scales
__host__ __device__ constexpr int staging_bytes(bool e4m3) { return 32 * staging_row(e4m3); }       // per epilogue warp
constexpr int kScaleSlots = 4;                      // K blocks whose scales are in shared memory
constexpr uint32_t kTmemCols = 512;

struct PairBarriers {
    uint64_t full[kStages], empty[kStages];  // full: of the first CTA, for both
    uint64_t acc_full[2], acc_empty[2];      // acc_empty: of the first CTA, for both
    uint64_t drained;
    uint32_t tmem_base;
    volatile uint32_t abort_flag;
    union {
        float top[2][2][kTile];              // 8 bits: [tile parity][warpgroup][row], largest |h| of a row's columns
        alignas(16) uint16_t bias[8][128];   // 16 bits: [warp], of its 64 columns of the gate and of the up projection
    };
};
// 8-bit operands, per K block: the product of the row's scale and that of the weight's columns [0, 128) / [128, 256), or of the gate / the
// up projection.
typedef float PairScales[kScaleSlots][2][kTile];
constexpr size_t smem_bytes(bool e4m3) { return kStages * kStageBytes + 8 * staging_bytes(e4m3) + sizeof(PairBarriers) + (e4m3 ? sizeof(PairScales) : 0); }
constexpr size_t kSmemBytes = 227 * 1024;  // all of an SM's, as in matmul_sm100.cu
static_assert(smem_bytes(true) <= kSmemBytes && smem_bytes(false) <= kSmemBytes, "");

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// ---- PTX of the pair ------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap *map, int x, int y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
template <bool kE4m3> __device__ __forceinline__ void tc_mma_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    if constexpr (kE4m3)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// Arrives at the barrier of the same offset in both CTAs when all products issued so far have completed.
__device__ __forceinline__ void tc_commit_pair(uint64_t *bar) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// ---- staged rows ------------------------------------------------------------------------------------------------------------
// A warp's 32 rows of 64 or 128 bytes, in 16-byte chunks whose places are permuted so that neither a thread writing its row nor
// neighbouring lanes reading one row meet in a bank.
template <int kRow> __device__ __forceinline__ uint4 *staged(uint8_t *base, int row, int chunk) {
    return reinterpret_cast<uint4 *>(base + row * kRow + ((chunk ^ (kRow == 128 ? row & 7 : (row >> 1) & 3)) * 16));
}

// Rows that do not start at multiples of 16 bytes leave in pieces of 8 or 4 bytes, neighbouring lanes neighbouring pieces.
template <int kBytes> struct Piece;
template <> struct Piece<8> { typedef uint2 type; };
template <> struct Piece<4> { typedef uint32_t type; };
template <> struct Piece<2> { typedef uint16_t type; };
template <> struct Piece<1> { typedef uint8_t type; };
template <int kSize, int kRow, int kPiece> __device__ __forceinline__ void store_pieces(uint8_t *base, uint8_t *out, int64_t row_bytes, int rows, int cols, int lane) {
    typedef typename Piece<kPiece>::type P;
    typedef typename Piece<kSize>::type E;
    constexpr int kPerRow = kRow / kPiece;
#pragma unroll 2
    for (int i = lane; i < 32 * kPerRow; i += 32) {
        const int r = i / kPerRow, at = i % kPerRow * kPiece, left = cols * kSize - at;
        if (r < rows && left > 0) {
            const uint8_t *from = reinterpret_cast<const uint8_t *>(staged<kRow>(base, r, at / 16)) + at % 16;
            uint8_t *to = out + r * row_bytes + at;
            if (left >= kPiece) *reinterpret_cast<P *>(to) = *reinterpret_cast<const P *>(from);
            else
#pragma unroll
                for (int j = 0; j < kPiece / kSize; ++j)
                    if (j * kSize < left) reinterpret_cast<E *>(to)[j] = reinterpret_cast<const E *>(from)[j];
        }
    }
}

// Rows [0, rows) x columns [0, cols) of elements of `kSize` bytes, kRow bytes staged per row, to out (row stride in bytes).
template <int kSize, int kRow> __device__ __forceinline__ void store_staged(uint8_t *base, uint8_t *out, int64_t row_bytes, int rows, int cols, int lane) {
    constexpr int kChunks = kRow / 16, kRowsAtOnce = 32 / kChunks, kPerChunk = 16 / kSize;
    if (rows <= 0 || cols <= 0) return;
    if ((((uintptr_t)out | (uintptr_t)row_bytes) & 15) == 0) {
        const int chunk = lane % kChunks, left = cols - chunk * kPerChunk;
        uint8_t *p = out + (lane / kChunks) * row_bytes + chunk * 16;
#pragma unroll
        for (int i = 0; i < 32 / kRowsAtOnce; ++i, p += kRowsAtOnce * row_bytes) {
            const int r = lane / kChunks + i * kRowsAtOnce;
            if (r < rows && left > 0) {
                const uint4 v = *staged<kRow>(base, r, chunk);
                if (left >= kPerChunk) *reinterpret_cast<uint4 *>(p) = v;
                else {
                    const uint8_t *e = reinterpret_cast<const uint8_t *>(&v);
#pragma unroll
                    for (int j = 0; j < kPerChunk; ++j)
                        if (j < left) {
                            if constexpr (kSize == 1) p[j] = e[j];
                            else if constexpr (kSize == 2) reinterpret_cast<uint16_t *>(p)[j] = reinterpret_cast<const uint16_t *>(e)[j];
                            else reinterpret_cast<uint32_t *>(p)[j] = reinterpret_cast<const uint32_t *>(e)[j];
                        }
                }
            }
        }
    } else if ((((uintptr_t)out | (uintptr_t)row_bytes) & 7) == 0) {
        store_pieces<kSize, kRow, 8>(base, out, row_bytes, rows, cols, lane);
    } else if ((((uintptr_t)out | (uintptr_t)row_bytes) & 3) == 0) {
        store_pieces<kSize, kRow, 4>(base, out, row_bytes, rows, cols, lane);
    } else {  // element by element, a row at a time: neighbouring lanes neighbouring elements
        for (int r = 0; r < min(rows, 32); ++r)
            for (int c = lane; c < min(cols, kRow / kSize); c += 32) {
                const uint8_t *e = reinterpret_cast<const uint8_t *>(staged<kRow>(base, r, c / kPerChunk)) + c % kPerChunk * kSize;
                typedef typename Piece<kSize>::type E;
                *reinterpret_cast<E *>(out + r * row_bytes + (int64_t)c * kSize) = *reinterpret_cast<const E *>(e);
            }
    }
}
// The way back: 64 16-bit columns of up to 32 rows to shared memory, zeros outside.  All loads are asked for before the first is used.
__device__ __forceinline__ void load_staged(uint8_t *base, const uint8_t *in, int64_t row_bytes, int rows, int cols, int lane) {
    const int chunk = lane & 7, r0 = lane >> 3, left = cols - chunk * 8;
    uint4 v[8];
    const uint8_t *p = in + r0 * row_bytes + chunk * 16;
    if ((((uintptr_t)in | (uintptr_t)row_bytes) & 15) == 0 && cols >= 64) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = r0 + 4 * i < rows ? *reinterpret_cast<const uint4 *>(p + 4 * i * row_bytes) : make_uint4(0, 0, 0, 0);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            uint32_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) e[j] = r0 + 4 * i < rows && j < left ? reinterpret_cast<const uint16_t *>(p + 4 * i * row_bytes)[j] : 0u;
            v[i] = make_uint4(e[0] | e[1] << 16, e[2] | e[3] << 16, e[4] | e[5] << 16, e[6] | e[7] << 16);
        }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) *staged<128>(base, r0 + 4 * i, chunk) = v[i];
}

template <bool kBF16> __device__ __forceinline__ void unpack_16(uint32_t v, float &lo, float &hi) {
    if constexpr (kBF16) {
        lo = __uint_as_float(v << 16);
        hi = __uint_as_float(v & 0xffff0000u);
    } else {
        const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&v));
        lo = f.x;
        hi = f.y;
    }
}
// Calls f with a compile-time truth value: a tile's loops then carry no test of what is the same for the whole launch.
template <typename F> __device__ __forceinline__ void as_constant(bool value, F f) {
    if (value) f(std::true_type{});
    else f(std::false_type{});
}
// Waits for a TMEM load; the registers pass through, so that nothing reads them earlier.
__device__ __forceinline__ void tc_wait_ld_of(uint32_t (&r)[32]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]),
                   "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]),
                   "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :: "memory");
}

// kSelfTest: the producers of some CTAs stop before a K block, so that the waits for it run out, after a limit of the launch's own.
template <bool kE4m3, int kMode, bool kAMn, bool kBMn, bool kSelfTest>
__global__ void __launch_bounds__(kThreads, 1) __cluster_dims__(2, 1, 1) matmul_pair_kernel(const __grid_constant__ MatmulParams p) {
    constexpr bool kGated = kMode != kMatmulPlain;
    constexpr int kElems = kE4m3 ? 128 : 64;  // contraction elements of a K block
    constexpr int kCols = kGated ? 64 : 128;  // result columns of a thread
    constexpr int kRow = staging_row(kE4m3);
    extern __shared__ __align__(1024) uint8_t smem[];
    PairBarriers &sh = *reinterpret_cast<PairBarriers *>(smem + kRingBytes + 8 * staging_bytes(kE4m3));
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;

    if (warp == kProducerWarp && lane == 0) {
        prefetch_map(&p.a[0]);
        prefetch_map(&p.b[kGated ? rank : 0]);
        sh.abort_flag = (*(volatile unsigned int *)p.status & kStatusMatmul) != 0 ? 1u : 0u;  // an earlier launch gave up
        for (int i = 0; i < kStages; ++i) {
            mbar_init(&sh.full[i], 1);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.acc_full[i], kE4m3 ? 3 : 1);  // the products, and the two warps that bring their scales
            mbar_init(&sh.acc_empty[i], 16);
        }
        mbar_init(&sh.drained, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kIssuerWarp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem_base)), "r"(kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    cluster_sync();  // both CTAs' barriers exist before either is signalled from the other
    tc_fence_after();
    // All of the SM's tensor memory is allocated, so its base is column 0: the tensor-memory addresses are constants.
    constexpr uint32_t tmem = 0;
    const uint32_t ring = smem_u32(smem);
    const auto limit = [&] { return kSelfTest ? p.wait_limit : kWaitTicks; };
    const auto wait = [&](uint64_t *bar, uint32_t parity, uint32_t code) { return mbar_wait_limit(bar, parity, &sh.abort_flag, p.status, code, limit()); };
    const int total = p.tiles_m * p.problems * p.tiles_n;
    struct Tile {
        int problem, m0, n0;
    };
    const auto tile_of = [&](int row, int col) {  // row and column of the grid of tiles; the second problem's rows follow the first's
        Tile w;
        w.problem = kAMn && row >= p.tiles_m ? 1 : 0;
        w.m0 = (row - w.problem * p.tiles_m) * 2 * kTile + (int)rank * kTile;
        w.n0 = col * (kGated ? kTile : kPairN);
        return w;
    };
    const auto tile_at = [&](int t) { return tile_of(t / p.tiles_n, t % p.tiles_n); };
    const int step_row = pairs / p.tiles_n, step_col = pairs - step_row * p.tiles_n;
    if (sh.tmem_base != tmem && threadIdx.x == 0) {
        sh.abort_flag = 1;
        atomicOr(p.status, kErrSums);
    }
    cluster_sync();
    // both CTAs have to agree on whether they run: a flag that only one of them saw raised would leave the other waiting (boundedly)
    const bool dead = ld_cluster_u32(map_rank(smem_u32((const void *)&sh.abort_flag), 0)) != 0 || ld_cluster_u32(map_rank(smem_u32((const void *)&sh.abort_flag), 1)) != 0;

    // 384 threads x 168 registers at launch = 64,512 = 2 x 128 x 232 + 128 x 40 = 2 x 128 x 216 + 128 x 72: the sums of 8-bit operands
    // live in registers, those of 16-bit ones in TMEM.  Every warp of a warpgroup executes its setmaxnreg.
    if (dead) {
    } else if (warp >= kProducerWarp) {
        if constexpr (kE4m3) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
        else asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        if (warp == kProducerWarp) {
            if (lane == 0) {
                int it = 0;
                bool ok = true;
                const uint32_t full0 = map_rank(smem_u32(&sh.full[0]), 0);
                for (int t = pair; t < total && ok; t += pairs) {
                    const Tile w = tile_at(t);
                    const int b0 = kGated ? w.n0 : w.n0 + (int)rank * kTile;
                    for (int i = 0; i < p.k_blocks; ++i, ++it) {
                        const int st = it % kStages;
                        ok = wait(&sh.empty[st], ((it / kStages) & 1) ^ 1, kErrEmpty);
                        if constexpr (kSelfTest) ok = ok && !(it >= p.stall_block && (p.stall_ctas >> rank & 1));
                        if (!ok) break;
                        const int sum = i >= p.kb_per_sum ? 1 : 0, k = (i - sum * p.kb_per_sum) * kElems;
                        const uint32_t dst = ring + st * kStageBytes, bar = full0 + st * 8;
                        if (rank == 0) mbar_arrive_expect_tx(&sh.full[st], 2 * kStageBytes);
                        const CUtensorMap *ma = &p.a[w.problem * p.sums + sum], *mb = &p.b[kGated ? rank : kAMn ? 0 : sum];
                        if constexpr (kAMn) {
                            tma_load_2d_pair(dst, ma, w.m0, k, bar);
                            tma_load_2d_pair(dst + kOperandBytes / 2, ma, w.m0 + 64, k, bar);
                        } else {
                            tma_load_2d_pair(dst, ma, k, w.m0, bar);
                        }
                        if constexpr (kBMn) {
                            tma_load_2d_pair(dst + kOperandBytes, mb, b0, k, bar);
                            tma_load_2d_pair(dst + kOperandBytes + kOperandBytes / 2, mb, b0 + 64, k, bar);
                        } else {
                            tma_load_2d_pair(dst + kOperandBytes, mb, k, b0, bar);
                        }
                    }
                }
                if (rank == 0)  // what was asked for has landed (both CTAs' loads complete here) before shared memory is released
                    for (int j = max(it - kStages, 0); j < it; ++j) mbar_drain(&sh.full[j % kStages], (j / kStages) & 1, p.status, kErrFull, limit());
                // The products' arrivals come to the barriers of both CTAs; those that no role waits for are waited for here, or they could
                // reach the shared memory of whatever runs next on this SM: `empty` of the last stages, and on the second CTA `drained`
                // (the first one's issuer waits for its own).
                for (int j = max(it - kStages, 0); j < it && ok; ++j) ok = wait(&sh.empty[j % kStages], (j / kStages) & 1, kErrEmpty);
                if (rank == 1 && ok) wait(&sh.drained, 0, kErrSums);
            }
            __syncwarp();
        } else if (warp == kIssuerWarp) {
            if (rank == 0) {
                // Warp-uniform control flow and constant addresses, so that the operands of the tensor-core instructions are constants or
                // uniform registers: moved from ordinary ones, a K block's six instructions took 430 to 550 clocks to issue.  `ok` is a
                // lane's own: after a wait gave up its elected lane issues nothing more; it steers the loop by a vote every 32 blocks only.
                const uint32_t idesc = matmul_idesc(kE4m3, p.dtype == COME_BF16, 2 * kTile, kPairN, kAMn, kBMn);
                constexpr uint32_t kAStep = kAMn ? 2048 >> 4 : 32 >> 4, kBStep = kBMn ? 2048 >> 4 : 32 >> 4;
                const uint64_t desc_a = operand_desc(ring, kOperandBytes / 2), desc_b = operand_desc(ring + kOperandBytes, kOperandBytes / 2);
                uint32_t st = 0, st_phase = 0, buf = 0, buf_phase = 1;
                bool ok = true, go = true;
                const auto wait_here = [&](uint64_t *bar, uint32_t parity, uint32_t code) {
                    if (!mbar_try_wait(bar, parity)) ok = ok && wait(bar, parity, code);
                };
                for (int t = pair; t < total && go; t += pairs) {
                    for (int i = 0; i < p.k_blocks; ++i) {
                        if ((i & 31) == 31 || i == 0) {
                            go = __all_sync(0xffffffffu, ok);
                            if (!go) break;
                        }
                        wait_here(&sh.full[st], st_phase, kErrFull);
                        if (kE4m3 || i == 0) wait_here(&sh.acc_empty[buf], buf_phase, kErrSums);
                        __syncwarp();
                        tc_fence_after();
                        const uint64_t da = desc_a + (uint64_t)(st * (kStageBytes >> 4)), db = desc_b + (uint64_t)(st * (kStageBytes >> 4));
                        const uint32_t d_tmem = buf * kPairN;
                        const bool last = kE4m3 || i == p.k_blocks - 1;
                        const uint32_t more = !kE4m3 && i > 0 ? 1u : 0u;
                        if (elect_one() && ok) {
                            tc_mma_pair<kE4m3>(d_tmem, da, db, idesc, more);
                            tc_mma_pair<kE4m3>(d_tmem, da + kAStep, db + kBStep, idesc, 1u);
                            tc_mma_pair<kE4m3>(d_tmem, da + 2 * kAStep, db + 2 * kBStep, idesc, 1u);
                            tc_mma_pair<kE4m3>(d_tmem, da + 3 * kAStep, db + 3 * kBStep, idesc, 1u);
                            tc_commit_pair(&sh.empty[st]);
                            if (last) tc_commit_pair(&sh.acc_full[buf]);
                        }
                        __syncwarp();
                        if (++st == kStages) {
                            st = 0;
                            st_phase ^= 1u;
                        }
                        if (last) {
                            buf ^= 1u;
                            if (buf == 0) buf_phase ^= 1u;
                        }
                    }
                }
                if (elect_one()) {
                    tc_commit_pair(&sh.drained);
                    mbar_drain(&sh.drained, 0, p.status, kErrSums, limit());
                }
            }
            __syncwarp();
        } else if constexpr (kE4m3) {
            // Warps 10, 11: the scales of a K block for 64 rows each, loaded two blocks ahead.  A warp arrives for block i after block i - 2 of
            // the same TMEM buffer has completed: then every warp has read the scales of block i - 4, whose slot block i takes.
            PairScales &scales = *reinterpret_cast<PairScales *>(&sh + 1);
            const int r0 = (warp - kProducerWarp - 2) * 64 + lane;  // rows r0, r0 + 32
            int chunk = 0;
            bool ok = true;
            float row[2][2], block[2][2];  // [parity of the K block]
            int ahead_t = pair, ahead_k = 0;
            const float *ahead_row[2] = {}, *ahead_block[2] = {};
            const auto fetch = [&](int j) {
                if (ahead_t >= total) return;
                if (ahead_k == 0) {
                    const Tile w = tile_at(ahead_t);
                    const int nb = w.n0 / kTile, last = (p.N - 1) / kTile;  // past the last column block nothing is stored
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        ahead_row[i] = p.a_scale + (int64_t)min(w.m0 + r0 + 32 * i, p.M - 1) * p.as_row;
                        ahead_block[i] = kGated ? p.b_scale[i] + nb * p.bs_row[i] : p.b_scale[0] + min(nb + i, last) * p.bs_row[0];
                    }
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    row[j][i] = *ahead_row[i];
                    block[j][i] = *ahead_block[i];
                    ahead_row[i] += p.as_block;
                    ahead_block[i] += 1;
                }
                if (++ahead_k == p.k_blocks) {
                    ahead_k = 0;
                    ahead_t += pairs;
                }
            };
            const int64_t blocks = (int64_t)((total - pair + pairs - 1) / pairs) * p.k_blocks;
            fetch(0);
            fetch(1);
            for (int64_t i0 = 0; i0 < blocks && ok; i0 += 2) {
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    if (i0 + j < blocks && ok) {
                        const int slot = chunk % kScaleSlots;
                        if (chunk >= 2) ok = wait(&sh.acc_full[j], ((chunk >> 1) - 1) & 1, kErrSums);
                        ok = __all_sync(0xffffffffu, ok);
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            scales[slot][0][r0 + 32 * i] = row[j][i] * block[j][0];
                            scales[slot][1][r0 + 32 * i] = row[j][i] * block[j][1];
                        }
                        fetch(j);
                        __syncwarp();
                        if (ok && lane == 0) mbar_arrive(&sh.acc_full[j]);
                        ++chunk;
                    }
                }
            }
        }
    } else {
        if constexpr (kE4m3) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        const int part = warp >> 2, r = (warp & 3) * 32 + lane, warp_row = (warp & 3) * 32;
        const uint32_t lanes = tmem + ((uint32_t)warp_row << 16) + part * kCols;
        uint8_t *stage = smem + kRingBytes + warp * staging_bytes(kE4m3);
        [[maybe_unused]] const PairScales &scales = *reinterpret_cast<const PairScales *>(&sh + 1);
        const uint32_t empty0 = map_rank(smem_u32(&sh.acc_empty[0]), 0);
        int chunk = 0, tiles = 0;
        bool ok = true, busy = false;
        [[maybe_unused]] const bool with_bias = p.bias[0] != nullptr || (kGated && p.bias[1] != nullptr);
        [[maybe_unused]] float *bias = reinterpret_cast<float *>(stage);  // [128]: of the gate's and the up projection's 64 columns, or of 128
        int tile_row = pair / p.tiles_n, tile_col = pair - tile_row * p.tiles_n;
        const int count = (total - pair + pairs - 1) / pairs;
        for (; tiles < count; ++tiles) {
            if constexpr (kE4m3) {
                {   // the biases of the warp's columns, before the sums
                    const Tile w = tile_of(tile_row, tile_col);
                    const int n = w.n0 + part * kCols, cols = p.N - n;
                    if (with_bias) {
                        __syncwarp();
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            const float *b = kGated ? (const float *)p.bias[c >> 1] : (const float *)p.bias[0];
                            const int col = (kGated ? (c & 1) : c) * 32 + lane;
                            bias[c * 32 + lane] = b != nullptr && col < cols ? b[n + col] : 0.0f;
                        }
                        __syncwarp();
                    }
                    busy = p.M - w.m0 - warp_row > 0;
                }
                // sums as packed pairs: [0, 32) of the gate or of columns [0, 64), [32, 64) of the up projection or of columns [64, 128)
                f32x2_t sum[64];
#pragma unroll
                for (int c = 0; c < 64; ++c) sum[c] = 0ull;
                for (int i = 0; i < p.k_blocks; ++i, ++chunk) {
                    const int buf = chunk & 1, slot = chunk % kScaleSlots;
                    ok = ok && wait(&sh.acc_full[buf], (chunk >> 1) & 1, kErrSums);
                    ok = __all_sync(0xffffffffu, ok);
                    if (ok && busy) {
                        tc_fence_after();
                        const float s0 = scales[slot][kGated ? 0 : part][r], s1 = kGated ? scales[slot][1][r] : s0;
                        const f32x2_t s0p = pack_f32x2(s0, s0), s1p = pack_f32x2(s1, s1);
                        // 16 columns at a time, two loads in flight: 32 at a time need registers that are not there (spills cost 15 %)
                        const auto column = [&](int c) { return lanes + buf * kPairN + (kGated ? (c >> 2) * kTile + (c & 3) * 16 : c * 16); };
                        uint32_t d[32];
                        tmem_ld16(column(0), d);
                        tmem_ld16(column(1), d + 16);
#pragma unroll
                        for (int c = 0; c < 8; c += 2) {
                            tc_wait_ld_of(d);
                            if (c == 6) {
                                tc_fence_before();
                                __syncwarp();
                                if (lane == 0) mbar_arrive_at(empty0 + buf * 8);  // the buffer is in registers
                            }
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
#pragma unroll
                                for (int e = 0; e < 8; ++e)
                                    sum[(c + j) * 8 + e] = fma_f32x2(pack_f32x2(__uint_as_float(d[j * 16 + 2 * e]), __uint_as_float(d[j * 16 + 2 * e + 1])), (c + j) >> 2 ? s1p : s0p, sum[(c + j) * 8 + e]);
                                if (c < 6) tmem_ld16(column(c + 2 + j), d + j * 16);
                            }
                        }
                    } else if (ok && lane == 0) {
                        mbar_arrive_at(empty0 + buf * 8);
                    }
                }
                // Where the tile lies is worked out again (the shuffles hide that they are the same numbers): kept over the loop, it costs
                // registers that the sums need.
                const Tile w = tile_of(__shfl_sync(0xffffffffu, tile_row, 0), __shfl_sync(0xffffffffu, tile_col, 0));
                const int rows = min(32, p.M - w.m0 - warp_row), n = w.n0 + part * kCols, cols = p.N - n;
                const int64_t row0 = w.m0 + warp_row;
                if constexpr (!kGated) {
                    if (ok && busy) {
                        if (with_bias) {
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                const float4 b = *reinterpret_cast<const float4 *>(bias + 4 * c);
                                sum[2 * c] = add_f32x2(sum[2 * c], pack_f32x2(b.x, b.y));
                                sum[2 * c + 1] = add_f32x2(sum[2 * c + 1], pack_f32x2(b.z, b.w));
                            }
                            __syncwarp();
                        }
                        if (p.out_dtype == COME_F32) {
                            uint8_t *out = (uint8_t *)p.out[0] + (row0 * p.out_row[0] + n) * 4;
#pragma unroll
                            for (int h = 0; h < 8; ++h) {
#pragma unroll
                                for (int c = 0; c < 4; ++c) {
                                    float v[4];
                                    unpack_f32x2(sum[h * 8 + c * 2], v[0], v[1]);
                                    unpack_f32x2(sum[h * 8 + c * 2 + 1], v[2], v[3]);
                                    *staged<kRow>(stage, lane, c) = make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
                                }
                                __syncwarp();
                                store_staged<4, kRow>(stage, out + h * kRow, p.out_row[0] * 4, rows, cols - h * 16, lane);
                                __syncwarp();
                            }
                        } else {
                            as_constant(p.out_dtype == COME_BF16, [&](auto bf16) {
                                uint8_t *out = (uint8_t *)p.out[0] + (row0 * p.out_row[0] + n) * 2;
#pragma unroll
                                for (int h = 0; h < 4; ++h) {
#pragma unroll
                                    for (int c = 0; c < 4; ++c) {
                                        uint32_t e[4];
#pragma unroll
                                        for (int j = 0; j < 4; ++j) {
                                            float lo, hi;
                                            unpack_f32x2(sum[h * 16 + c * 4 + j], lo, hi);
                                            e[j] = pack_16<decltype(bf16)::value>(lo, hi);
                                        }
                                        *staged<kRow>(stage, lane, c) = make_uint4(e[0], e[1], e[2], e[3]);
                                    }
                                    __syncwarp();
                                    store_staged<2, kRow>(stage, out + h * kRow, p.out_row[0] * 2, rows, cols - h * 32, lane);
                                    __syncwarp();
                                }
                            });
                        }
                    }
                } else {
                    float tops[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // the results take the place of the gate's sums
                    if (ok && busy) {
                        if (with_bias) {
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                const float4 b = *reinterpret_cast<const float4 *>(bias + 4 * c);
                                sum[2 * c] = add_f32x2(sum[2 * c], pack_f32x2(b.x, b.y));
                                sum[2 * c + 1] = add_f32x2(sum[2 * c + 1], pack_f32x2(b.z, b.w));
                            }
                        }
                        as_constant(p.act == COME_ACT_SILU, [&](auto silu) {
                            constexpr int act = decltype(silu)::value ? COME_ACT_SILU : COME_ACT_GELU;
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                float g0, g1, u0, u1;
                                unpack_f32x2(sum[c], g0, g1);
                                unpack_f32x2(sum[32 + c], u0, u1);
                                const float h0 = activation(g0, act) * u0, h1 = activation(g1, act) * u1;
                                tops[c & 3] = fmaxf(tops[c & 3], fmaxf(fabsf(h0), fabsf(h1)));  // under the special-function unit
                                sum[c] = pack_f32x2(h0, h1);
                            }
                        });
                        if (cols < 64) {  // columns past the end are zeros (TMA fills them), or NaN in a row whose scale is infinite: not in the maximum
                            tops[0] = tops[1] = tops[2] = tops[3] = 0.0f;
#pragma unroll
                            for (int c = 0; c < 32; ++c) {
                                float h0, h1;
                                unpack_f32x2(sum[c], h0, h1);
                                h0 = 2 * c < cols ? h0 : 0.0f;
                                h1 = 2 * c + 1 < cols ? h1 : 0.0f;
                                tops[0] = fmaxf(tops[0], fmaxf(fabsf(h0), fabsf(h1)));
                                sum[c] = pack_f32x2(h0, h1);
                            }
                        }
                        __syncwarp();
                    }
                    if (p.out_dtype == COME_E4M3) {
                        float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                        // the largest magnitude of a row's 128 columns: half of it in the other warpgroup (every warp meets here, also
                        // one that gave up; a third tile's write to the same place is two barriers away)
                        sh.top[tiles & 1][part][r] = top;
                        asm volatile("bar.sync 1, 256;" ::: "memory");
                        top = fmaxf(fmaxf(top, sh.top[tiles & 1][part ^ 1][r]), kSmallestMax);
                        if (ok && busy) {
                            const float inv = inverse_scale(top);
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                uint32_t q[4];
#pragma unroll
                                for (int j = 0; j < 4; ++j) {
                                    float e[4];
                                    unpack_f32x2(sum[c * 8 + j * 2], e[0], e[1]);
                                    unpack_f32x2(sum[c * 8 + j * 2 + 1], e[2], e[3]);
                                    q[j] = pack_e4m3(e[0] * inv, e[1] * inv, e[2] * inv, e[3] * inv);
                                }
                                *staged<kRow>(stage, lane, c) = make_uint4(q[0], q[1], q[2], q[3]);
                            }
                            __syncwarp();
                            store_staged<1, kRow>(stage, (uint8_t *)p.out[0] + row0 * p.out_row[0] + n, p.out_row[0], rows, cols, lane);
                            if (part == 0 && lane < rows) p.out_scale[(row0 + lane) * p.os_row + (w.n0 / kTile) * p.os_block] = top * (1.0f / kE4m3Max);
                            __syncwarp();
                        }
                    } else if (ok && busy) {
                        as_constant(p.out_dtype == COME_BF16, [&](auto bf16) {
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
#pragma unroll
                                for (int c = 0; c < 4; ++c) {
                                    uint32_t q[4];
#pragma unroll
                                    for (int j = 0; j < 4; ++j) {
                                        float lo, hi;
                                        unpack_f32x2(sum[half * 16 + c * 4 + j], lo, hi);
                                        q[j] = pack_16<decltype(bf16)::value>(lo, hi);
                                    }
                                    *staged<kRow>(stage, lane, c) = make_uint4(q[0], q[1], q[2], q[3]);
                                }
                                __syncwarp();
                                store_staged<2, kRow>(stage, (uint8_t *)p.out[0] + (row0 * p.out_row[0] + n + half * 32) * 2, p.out_row[0] * 2, rows, cols - half * 32, lane);
                                __syncwarp();
                            }
                        });
                    }
                }
            } else {
                const Tile w = tile_of(tile_row, tile_col);
                const int rows = min(32, p.M - w.m0 - warp_row);      // of this warp, may be <= 0
                const int n = w.n0 + part * kCols, cols = p.N - n;    // first result column of the thread, columns from there on
                busy = rows > 0;
                const int64_t row0 = w.m0 + warp_row;
                const int buf = chunk & 1;
                if (kGated && busy) {  // before the wait: the biases of this warp's 64 + 64 columns, and dh
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        const uint16_t *b = (const uint16_t *)p.bias[c >> 1];
                        const int col = (c & 1) * 32 + lane;
                        sh.bias[warp][c * 32 + lane] = b != nullptr && col < cols ? b[n + col] : (uint16_t)0;
                    }
                    if (kMode == kMatmulGatedGrad && ok && cols > 0) load_staged(stage, (const uint8_t *)p.dh + (row0 * p.dh_row + n) * 2, p.dh_row * 2, rows, cols, lane);
                    __syncwarp();
                }
                ok = ok && wait(&sh.acc_full[buf], (chunk >> 1) & 1, kErrSums);
                ok = __all_sync(0xffffffffu, ok);
                if (ok && busy) {
                    tc_fence_after();
                    const uint32_t from = lanes + buf * kPairN;
                    as_constant(p.dtype == COME_BF16, [&](auto bf16_c) {
                        constexpr bool kBF16 = decltype(bf16_c)::value;
                        [[maybe_unused]] const float factor = kBF16 ? 1.0f : range_factor(p.range, !kGated);
                        if constexpr (!kGated) {
#pragma unroll 1
                            for (int h = 0; h < kCols / 32; ++h) {
                                uint32_t d[32];
                                tmem_ld32(from + h * 32, d);
                                tc_wait_ld_of(d);
                                if (h == kCols / 32 - 1) {  // the sums are in registers: the next tile may begin
                                    tc_fence_before();
                                    __syncwarp();
                                    if (lane == 0) mbar_arrive_at(empty0 + buf * 8);
                                }
#pragma unroll
                                for (int c = 0; c < 4; ++c) {
                                    uint32_t e[4];
#pragma unroll
                                    for (int j = 0; j < 4; ++j) {
                                        const float lo = __uint_as_float(d[c * 8 + 2 * j]), hi = __uint_as_float(d[c * 8 + 2 * j + 1]);
                                        e[j] = kBF16 ? pack_16<kBF16>(lo, hi) : pack_16<kBF16>(lo * factor, hi * factor);
                                    }
                                    *staged<64>(stage + (h & 1) * 2048, lane, c) = make_uint4(e[0], e[1], e[2], e[3]);
                                }
                                __syncwarp();
                                store_staged<2, 64>(stage + (h & 1) * 2048, (uint8_t *)p.out[w.problem] + (row0 * p.out_row[w.problem] + n + h * 32) * 2, p.out_row[w.problem] * 2, rows, cols - h * 32, lane);
                            }
                            __syncwarp();
                        } else {
                            as_constant(p.act == COME_ACT_SILU, [&](auto silu) {
                                constexpr int act = decltype(silu)::value ? COME_ACT_SILU : COME_ACT_GELU;
                                [[maybe_unused]] uint32_t second[32];  // du of the row, while dg is staged
#pragma unroll
                                for (int q = 0; q < 2; ++q) {
                                    uint32_t g[32], u[32];
                                    tmem_ld32(from + q * 32, g);
                                    tmem_ld32(from + kTile + q * 32, u);
                                    tc_wait_ld_of(g);
                                    tc_wait_ld_of(u);
                                    if (q == 1) {  // the sums are in registers: the next tile may begin
                                        tc_fence_before();
                                        __syncwarp();
                                        if (lane == 0) mbar_arrive_at(empty0 + buf * 8);
                                    }
#pragma unroll
                                    for (int c = 0; c < 4; ++c) {
                                        const uint4 bg = *reinterpret_cast<const uint4 *>(&sh.bias[warp][q * 32 + c * 8]), bu = *reinterpret_cast<const uint4 *>(&sh.bias[warp][64 + q * 32 + c * 8]);
                                        const uint32_t bgs[4] = {bg.x, bg.y, bg.z, bg.w}, bus[4] = {bu.x, bu.y, bu.z, bu.w};
                                        uint32_t e[4];
                                        [[maybe_unused]] uint32_t dh[4];
                                        if constexpr (kMode == kMatmulGatedGrad) {
                                            const uint4 raw = *staged<kRow>(stage, lane, q * 4 + c);
                                            dh[0] = raw.x, dh[1] = raw.y, dh[2] = raw.z, dh[3] = raw.w;
                                        }
#pragma unroll
                                        for (int j = 0; j < 4; ++j) {
                                            float g0, g1, u0, u1;
                                            unpack_16<kBF16>(bgs[j], g0, g1);
                                            unpack_16<kBF16>(bus[j], u0, u1);
                                            g0 += __uint_as_float(g[c * 8 + 2 * j]), g1 += __uint_as_float(g[c * 8 + 2 * j + 1]);
                                            u0 += __uint_as_float(u[c * 8 + 2 * j]), u1 += __uint_as_float(u[c * 8 + 2 * j + 1]);
                                            if constexpr (kMode == kMatmulGated) {
                                                e[j] = pack_16<kBF16>(activation(g0, act) * u0, activation(g1, act) * u1);
                                            } else {
                                                float d0, d1, a0, a1, s0, s1;
                                                unpack_16<kBF16>(dh[j], d0, d1);
                                                if constexpr (!kBF16) d0 *= factor, d1 *= factor;
                                                activation_grad(g0, act, a0, s0);
                                                activation_grad(g1, act, a1, s1);
                                                e[j] = pack_16<kBF16>(d0 * u0 * s0, d1 * u1 * s1);
                                                second[(q * 4 + c) * 4 + j] = pack_16<kBF16>(d0 * a0, d1 * a1);
                                            }
                                        }
                                        *staged<kRow>(stage, lane, q * 4 + c) = make_uint4(e[0], e[1], e[2], e[3]);
                                    }
                                }
                                __syncwarp();
                                store_staged<2, kRow>(stage, (uint8_t *)p.out[0] + (row0 * p.out_row[0] + n) * 2, p.out_row[0] * 2, rows, cols, lane);
                                __syncwarp();
                                if constexpr (kMode == kMatmulGatedGrad) {
#pragma unroll
                                    for (int c = 0; c < 8; ++c) *staged<kRow>(stage, lane, c) = make_uint4(second[4 * c], second[4 * c + 1], second[4 * c + 2], second[4 * c + 3]);
                                    __syncwarp();
                                    store_staged<2, kRow>(stage, (uint8_t *)p.out[1] + (row0 * p.out_row[1] + n) * 2, p.out_row[1] * 2, rows, cols, lane);
                                    __syncwarp();
                                }
                            });
                        }
                    });
                } else if (ok) {
                    if (lane == 0) mbar_arrive_at(empty0 + buf * 8);
                }
                ++chunk;
            }
            tile_row += step_row;
            tile_col += step_col;
            if (tile_col >= p.tiles_n) {
                tile_col -= p.tiles_n;
                ++tile_row;
            }
        }
    }
    __syncwarp();
    if (sh.abort_flag != 0) st_cluster_u32(map_rank(smem_u32((const void *)&sh.abort_flag), rank ^ 1), 1);  // the other CTA learns of it
    tc_fence_before();
    cluster_sync();  // both CTAs' roles have ended: nothing more is issued, and every arrival and copy has landed unless a wait gave up
    if (sh.abort_flag != 0) {  // what was not waited for, of either CTA, gets time to land before either leaves
        const long long t0 = clock64();
        while (clock64() - t0 < (1ll << 22)) {
        }
    }
    __syncwarp();
    if (warp == kIssuerWarp) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

template <bool kE4m3, int kMode, bool kAMn, bool kBMn, bool kSelfTest = false> int launch_pair(const MatmulParams &p, cudaStream_t st) {
    constexpr auto kernel = matmul_pair_kernel<kE4m3, kMode, kAMn, kBMn, kSelfTest>;
    if (int rc = allow_smem<kernel>(kSmemBytes); rc != COME_OK) return rc;
    const int tiles = p.tiles_m * p.problems * p.tiles_n, pairs = sm_count() / 2;
    kernel<<<2 * (tiles < pairs ? tiles : pairs), kThreads, kSmemBytes, st>>>(p);
    return check_launch("product kernel");
}

}  // namespace

// A tile for every second pair of SMs is where this kernel overtakes the split one (us in a graph, split / pair): 8-bit 1374 tokens
// 1024 -> 1024, 24 tiles: 10.3 / 10.7; 2748 tokens, 44 tiles: 19.3 / 10.9; 300 tokens 4096 -> 4096, 32 tiles: 19.4 / 22.1; 16-bit gated
// 1024 -> 2736, 100 tokens, 22 tiles: 9.9 / 11.0; 300 tokens, 44 tiles: 11.7 / 11.4.  In the 8-bit gated form every fourth pair is
// enough, where the rows fill most of a tile: 700 tokens 400 -> 1003, 24 tiles: 11.6 / 10.0; 1024 -> 2736 (22 tiles) with 64 tokens
// 8.5 / 9.9, with 128 10.5 / 10.0.
bool matmul_pair_takes(const MatmulArgs &a) {
    const int64_t n = a.mode == kMatmulPlain ? kPairN : kTile, pairs = sm_count() / 2;
    const int64_t tiles = (a.M + 2 * kTile - 1) / (2 * kTile) * ((a.N + n - 1) / n) * a.problems;
    if (a.low_rows > 0 || a.sums * a.problems > 2) return false;  // few tokens: the split kernel alone has these forms
    return tiles * 2 >= pairs || (a.e4m3 && a.mode == kMatmulGated && a.M > 96 && tiles * 4 >= pairs);
}

int matmul_pair_launch(const MatmulArgs &a, MatmulParams &p, cudaStream_t st) {
    const int n = a.mode == kMatmulPlain ? kPairN : kTile;
    p.tiles_n = (int)((a.N + n - 1) / n);
    const int64_t rows = (a.M + 2 * kTile - 1) / (2 * kTile);
    COME_REQUIRE(rows * p.tiles_n * a.problems < (1ll << 30), "the result has too many tiles for one launch");
    p.tiles_m = (int)rows;
    if (a.wait_limit > 0) return a.e4m3 ? launch_pair<true, kMatmulGated, false, false, true>(p, st) : launch_pair<false, kMatmulGated, false, false, true>(p, st);
    if (a.e4m3) return a.mode == kMatmulPlain ? launch_pair<true, kMatmulPlain, false, false>(p, st) : launch_pair<true, kMatmulGated, false, false>(p, st);
    if (a.mode == kMatmulGated) return launch_pair<false, kMatmulGated, false, false>(p, st);
    if (a.mode == kMatmulGatedGrad) return launch_pair<false, kMatmulGatedGrad, false, false>(p, st);
    return a.a_mn ? launch_pair<false, kMatmulPlain, true, true>(p, st) : launch_pair<false, kMatmulPlain, false, true>(p, st);
}

}  // namespace come

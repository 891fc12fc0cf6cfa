// C[M][N] = A B^T of two NVFP4 operands on the block-scaled tensor cores of sm_100a: tcgen05.mma kind::mxf4nvf4 with an E4M3
// scale for 16 values of K, FP32 accumulators in tensor memory, operands and their block scales staged by TMA, the scales copied
// on from shared to tensor memory by tcgen05.cp in front of the MMAs that read them.
//
// The operands' rows are 128-byte swizzled panels as in the Newton-Schulz GEMM (ns_gemm_sm100.cu): 128 bytes are 256 values of K,
// four MMAs.  The block scales of 128 rows and 64 values of K are a 512-byte tile, stored as the copy wants it.
//
// What bounds it.  8192^3: the MMAs, 5.8 PFLOP/s (190 us).  Short sums: the way between L2 and the SMs.  16384 x 1600 -> 6400 in BF16, 90
// us, moves 1.18 GB through L2 (13 TB/s), loads of tiles and stores of results together; without its stores it takes 64 us, without
// its MMAs 80, without the copies of scales 89.  The same for results stored by row, by threads from shared memory or straight from
// registers in 32-byte pieces (129, 88, 87), for tiles in the other order and for cache hints.  Tiles of 256 x 192, whose
// accumulators share no columns of tensor memory, load more for a result: 108.
#include <algorithm>
#include <atomic>
#include <cstdlib>
#include <type_traits>

#include <cuda.h>

#include "common.cuh"
#include "fp4.h"
#include "fp4_block.cuh"
#include "sm100.cuh"

namespace b2 {

namespace {

constexpr uint32_t kStageK = 256;       // values of K in a pipeline stage
constexpr uint32_t kScaleTile = 512;    // bytes: 128 rows x 64 values of K
constexpr uint32_t kSlabBytes = 32 * 128;   // an epilogue warp's: 32 rows x 128 bytes of c
constexpr uint32_t kScaleBand = kStageK / 64 * kScaleTile;   // a stage's scales of 128 rows

// Set when a bounded wait ran out (b2_nvfp4_status).
__device__ uint32_t g_fp4_status;

// D (+)= A B^T over 64 values of K; the scales' addresses are columns of tensor memory
template <bool PAIR>
__device__ __forceinline__ void tc_mma_fp4(uint32_t d_tmem, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                           uint32_t accumulate) {
    if (PAIR)
        asm volatile(
            "{ .reg .pred p; setp.ne.b32 p, %6, 0; "
            "tcgen05.mma.cta_group::2.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p; }"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{ .reg .pred p; setp.ne.b32 p, %6, 0; "
            "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p; }"
            ::"r"(d_tmem), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
            : "memory");
}
// A 512-byte tile of scales from shared memory to four columns of tensor memory, the same in every lane quarter; PAIR: in both
// CTAs, each from its own shared memory.
template <bool PAIR>
__device__ __forceinline__ void tc_copy_scales(uint32_t tmem, uint64_t desc) {
    if (PAIR) asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
    else asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(tmem), "l"(desc) : "memory");
}
// Descriptor of such a tile: no swizzle, 8 rows of 16 bytes after one another.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
    return (uint64_t)((addr & 0x3ffffu) >> 4) | ((uint64_t)(128 >> 4) << 32) | ((uint64_t)1 << 46);
}
// Instruction descriptor for kind::mxf4nvf4: A and B E2M1 (1), scales UE4M3 (0), N >> 3 at bit 17, M >> 4 at bit 24.
__device__ __forceinline__ uint32_t fp4_instr_desc(uint32_t m, uint32_t n) {
    return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}

struct Epilogue {
    uint8_t *c;
    uint64_t pitch;            // bytes
    const float *scale_a;      // one, or one a row of A
    const float *scale_b;
    const float *bias;         // null or [N]
    uint32_t M, N;
    uint32_t a_rows, b_rows;   // a scale for every row of A (B)
    uint32_t type;             // of c
    uint32_t accumulate;
    // Rows of c on any boundary (see below): classes of rows (0: no map), places that the first row is off, and a next one more
    uint32_t classes, offset, step;
};

// ---- scales on top at the ends of FP32's range ----
// The product of two scales may be subnormal or out of range where the result is not.  A scale is then m p, p a power of two and m as far
// from 1: a sum (0, or 2^-20 and more, below 2^48) times both m, and then both p, leaves the range on the way only where the result is lost
// too, and otherwise has the bits of the sum times the product.  A warp whose rows need that (`far`) goes a way of its own: with these
// products done always 2048 x 1600 -> 50257 takes 160 us instead of 150 and 24 x 1600 -> 50304 10.2 instead of 9.0.  Rows of zeros beside a
// small weight look like it and are told by their sums: with half of the rows so, 16384 x 1600 -> 6400 takes 115.5 us instead of 108.5, where
// the way apart would take 1600.
struct Scale {
    float m, p;
};
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
__device__ __forceinline__ Scale split_scale(float g) {
    const int up = fabsf(g) < 0x1p-126f ? 64 : 0;   // subnormal, zero
    const float n = up ? g * 0x1p64f : g;
    const int k = ((int)(__float_as_uint(n) >> 23 & 255u) - 127 - up) >> 1;
    return {n * power_of_two(-up - k), power_of_two(k)};
}
// sum * (a * b), or (sum * a) * b
__device__ __forceinline__ float times_scales(float sum, Scale a, Scale b, bool one_by_one) {
    float m = a.m * b.m;
    asm("min.NaN.f32 %0, %0, %1;" : "+f"(m) : "f"(0x1.fffffep127f));   // (a sum of 0 stays 0)
    return (one_by_one ? sum * a.m * b.m : sum * m) * (a.p * b.p);
}
__device__ __forceinline__ bool in_range(float s) { return s >= 0x1p-126f && s <= 0x1.fffffep127f; }
__device__ __forceinline__ float scale_of_row(const Epilogue &e, uint32_t row) { return row < e.M ? e.scale_a[e.a_rows ? row : 0] : 1.0f; }

// Sums of 32 columns from `col` on, scaled (s: the scale of A's row, and B's where it has one for all) and biased (`bias`: theirs, in
// shared memory, or null).  `n` of them are there.
__device__ __forceinline__ void finish_columns(const Epilogue &e, uint32_t col, uint32_t n, const uint32_t *acc, float s, const float *bias, float (&v)[32]) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(acc[i]) * s;
    if (e.b_rows) {
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if ((uint32_t)i < n) v[i] *= e.scale_b[col + i];
    }
    if (bias) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float4 o = reinterpret_cast<const float4 *>(bias)[i];
            v[4 * i] += o.x; v[4 * i + 1] += o.y; v[4 * i + 2] += o.z; v[4 * i + 3] += o.w;
        }
    }
}
__device__ __forceinline__ void st_shared_16(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void store_value(const Epilogue &e, uint32_t row, uint32_t col, float v) {
    uint8_t *line = e.c + (uint64_t)row * e.pitch;
    if (e.type == B2_TYPE_F32) {
        float *p = reinterpret_cast<float *>(line) + col;
        *p = e.accumulate ? *p + v : v;
    } else {
        reinterpret_cast<uint16_t *>(line)[col] = (uint16_t)(e.type == B2_TYPE_F16 ? f32_to_f16_bits(v) : f32_to_bf16_bits(v));
    }
}
// The old values of 32 columns that are all there, of a row on a 16-byte boundary.
__device__ __forceinline__ void add_old(const Epilogue &e, uint32_t row, uint32_t col, float (&v)[32]) {
    const float4 *p = reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(e.c + (uint64_t)row * e.pitch) + col);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float4 o = p[i];
        v[4 * i] += o.x; v[4 * i + 1] += o.y; v[4 * i + 2] += o.z; v[4 * i + 3] += o.w;
    }
}
__device__ __forceinline__ void tma_store_2d(uint64_t map, uint32_t src, int x, int y) {
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Value by value through `slab` (32 x 32 floats of this warp, a row's columns in an order of its own), so that a store instruction of
// the warp writes neighbouring values of a row and not one value of each of 32 rows.
__device__ __forceinline__ void store_through(const Epilogue &e, uint32_t row0, uint32_t col, const float (&v)[32], float *slab) {
    const uint32_t lane = threadIdx.x & 31u;
    __syncwarp();
#pragma unroll
    for (uint32_t i = 0; i < 32; ++i) slab[lane * 32 + (i ^ lane)] = v[i];
    __syncwarp();
    const uint32_t rows = min(32u, e.M - row0);
    if (col + lane < e.N) {
#pragma unroll 8
        for (uint32_t r = 0; r < rows; ++r) store_value(e, row0 + r, col + lane, slab[r * 32 + (lane ^ r)]);
    }
    __syncwarp();
}

// ---- rows of c on any boundary ----
// A bulk store writes whole 16-byte pieces of memory.  Rows that start off such a boundary fall into classes: row r is off it by what
// row r + classes is (4 classes at most of FP32, 8 of 16-bit values).  A class's rows are a matrix on 16-byte boundaries, seen from
// the boundary in front of its first row; the three-dimensional map of c has a row's place as its first coordinate, offset + class
// step + column, the class as its second and r / classes as its third.  So a unit stores, class by class, its columns but the last
// `shift`, and in front of them as many of the unit before, which it reads out of tensor memory again.  The first unit of a tile has
// none before it: it begins at its first boundary and goes on into the next one (some values are written twice, the same both
// times).  What a tile has in front of its first boundary and behind its last one, and what is near the ends of c, goes value by value.
// 2048 x 1600 -> 50257: 148 us in FP32 and 126 in BF16; all of it value by value 174 and 182.
template <int SIZE>
__device__ __forceinline__ uint32_t shift_of(const Epilogue &e, uint32_t row) {
    return (e.offset + (row & (e.classes - 1)) * e.step) & (16 / SIZE - 1);
}
// 32 values behind four: the 32 that begin `shift` places before the first of the 32.  `ahead`: 32 values in front of four, the 32
// that begin 4 - shift places behind the first.
__device__ __forceinline__ void shift_values(const float (&side)[4], const float (&v)[32], bool ahead, uint32_t shift, uint32_t (&w)[32]) {
    const uint32_t u = 3 - shift;
    uint32_t a[36];
#pragma unroll
    for (int i = 0; i < 36; ++i) a[i] = __float_as_uint(ahead ? (i < 32 ? v[i & 31] : side[i & 3]) : (i < 4 ? side[i & 3] : v[(i - 4) & 31]));
#pragma unroll
    for (int i = 0; i < 34; ++i) a[i] = u & 1u ? a[i + 2] : a[i + 1];
#pragma unroll
    for (int i = 0; i < 32; ++i) w[i] = u & 2u ? a[i + 2] : a[i];
}
// The same for 64 16-bit values behind eight, or in front of eight: a[0 .. 35] -> a[0 .. 31]
__device__ __forceinline__ void shift_halves(uint32_t (&a)[36], uint32_t shift) {
    const uint32_t t = 8 - shift, h = t >> 1;
#pragma unroll
    for (int i = 0; i < 35; ++i) a[i] = t & 1u ? __byte_perm(a[i], a[i + 1], 0x5432) : a[i];
#pragma unroll
    for (int i = 0; i < 32; ++i) a[i] = h & 4u ? a[i + 4] : a[i];
#pragma unroll
    for (int i = 0; i < 33; ++i) a[i] = h & 2u ? a[i + 2] : a[i];
#pragma unroll
    for (int i = 0; i < 32; ++i) a[i] = h & 1u ? a[i + 1] : a[i];
}
__device__ __forceinline__ void tma_store_3d(uint64_t map, uint32_t src, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// The classes of a slab of 32 rows (class by class, 16-byte pieces in the order of the 128-byte swizzle) to columns col - shift on, or
// (`ahead`) to the first boundary from col on.
template <int SIZE>
__device__ __forceinline__ void store_classes(const Epilogue &e, uint64_t map, uint32_t row0, uint32_t col, bool ahead, uint32_t slab) {
    const uint32_t lane = threadIdx.x & 31u;
    fence_async_smem();
    __syncwarp();
    if (lane < e.classes) {
        const uint32_t x = e.offset + lane * e.step + col + (ahead ? 16 / SIZE - 1 : 0);
        tma_store_3d(map, slab + lane * (4096 / e.classes), (int)(x / (16 / SIZE) * (16 / SIZE)), (int)lane, (int)(row0 / e.classes));
    }
}
// 8 consecutive columns of 32 lanes
__device__ __forceinline__ void tc_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
}

// Tile of a CTA (128 x BN), or of a pair of CTAs (256 x BN): each holds 128 rows of A, half of the rows of B and all of B's scales.
template <bool PAIR, int BN>
struct FCfg {
    static constexpr uint32_t kTileM = PAIR ? 256 : 128;
    static constexpr uint32_t kBRows = PAIR ? BN / 2 : BN;
    static constexpr uint32_t kBands = BN / 128;
    static constexpr uint32_t kABytes = 128 * 128, kBBytes = kBRows * 128;
    static constexpr uint32_t kSfa = kABytes + kBBytes, kSfb = kSfa + kScaleBand;
    static constexpr uint32_t kStageBytes = kSfb + kBands * kScaleBand;
    static_assert(kStageBytes % 1024 == 0 && kSfa % 1024 == 0, "panels start on 1024-byte boundaries");
    // Tensor memory.  Two accumulators of 256 columns leave no room for scales, so they share 48 columns: the epilogue reads
    // these first, and the other accumulator's MMAs begin when it has.
    static constexpr uint32_t kShared = BN == 256 ? 48 : 0;
    static constexpr uint32_t kAcc1 = BN - kShared;
    static constexpr uint32_t kSfaCol = 2 * BN - kShared, kSfbCol = kSfaCol + 16;
    static_assert(kSfbCol + 16 * kBands <= 512, "tensor memory");
    static constexpr uint32_t kTmemCols = 512;
    // warps: producers of A, of B and of the scales, the MMA issuer, eight epilogue warps
    static constexpr int kProducerA = 0, kMmaWarp = 1, kEpiWarp0 = 2, kEpiWarps = 8, kProducerB = 10, kProducerS = 11;
    static constexpr int kThreads = 12 * 32;
    static constexpr uint32_t kControl = 1024;
    static constexpr uint32_t kStrip = 64 * 4;   // bytes: the bias of an epilogue warp's columns
    static constexpr uint32_t kBesides = kControl + kEpiWarps * (kSlabBytes + kStrip) + 1024;   // (the slabs start on a 1024-byte boundary)
    static constexpr uint32_t kMaxStages = ((uint32_t)kSmemLimit - kBesides) / kStageBytes;
    static constexpr uint32_t kStages = kMaxStages < 6 ? kMaxStages : 6;
    static constexpr uint32_t kSmemBytes = kStages * kStageBytes + kBesides;
};

// BULK: rows of c start and end on 16-byte boundaries
template <bool PAIR, int BN, bool BULK>
__global__ void __launch_bounds__((FCfg<PAIR, BN>::kThreads), 1)
k_fp4_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sa,
           const __grid_constant__ CUtensorMap map_sb, const __grid_constant__ CUtensorMap map_c, const __grid_constant__ Epilogue epi,
           uint32_t K, uint32_t tiles_m, uint32_t tiles) {
    using C = FCfg<PAIR, BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem + C::kStages * C::kStageBytes);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * C::kStages + 4);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    static_assert((2 * C::kStages + 4) * 8 + 8 <= C::kControl, "control region");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = PAIR ? cluster_cta_rank() : 0u;
    const uint32_t first = PAIR ? blockIdx.x / 2 : blockIdx.x, stride = PAIR ? gridDim.x / 2 : gridDim.x;
    const uint32_t bar0 = smem_u32(bars), stage0 = smem_u32(smem);
    auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (C::kStages + s); };
    auto tfull_bar = [&](uint32_t a) { return bar0 + 8u * (2 * C::kStages + a); };
    auto tempty_bar = [&](uint32_t a) { return bar0 + 8u * (2 * C::kStages + 2 + a); };

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < C::kStages; ++s) {
            mbar_init(full_bar(s), 3);   // the leader's three producers
            mbar_init(empty_bar(s), 1);
        }
        for (uint32_t a = 0; a < 2; ++a) {
            mbar_init(tfull_bar(a), 1);
            mbar_init(tempty_bar(a), PAIR ? 2 * C::kEpiWarps : C::kEpiWarps);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_sa) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_sb) : "memory");
    }
    if (warp == C::kMmaWarp) {
        if (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(C::kTmemCols) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    tc_fence_before();
    __syncthreads();
    if (PAIR) cluster_sync_all();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    stream_enter();

    const uint32_t stages = (K + kStageK - 1) / kStageK;
    // rows of B that the MMAs of a tile take: what there is of them, rounded up so that a pair's halves are whole 8-row groups
    auto mma_n = [&](uint32_t tile_n) { return min((uint32_t)BN, (epi.N - tile_n * BN + 31u) / 32u * 32u); };

    if (warp == C::kProducerA || warp == C::kProducerB || warp == C::kProducerS) {
        if (lane == 0) {
            const uint32_t leader_full = PAIR ? map_to_cta(full_bar(0), 0) : full_bar(0);
            const uint32_t bytes = (warp == C::kProducerA ? C::kABytes : warp == C::kProducerB ? C::kBBytes : (1 + C::kBands) * kScaleBand) * (PAIR ? 2u : 1u);
            uint32_t stage = 0, phase = 0;
            bool ok = true;
            for (uint32_t t = first; ok && t < tiles; t += stride) {
                const uint32_t tile_m = t % tiles_m, tile_n = t / tiles_m;
                for (uint32_t kb = 0; kb < stages; ++kb) {
                    if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) { ok = false; break; }
                    if (rank == 0) mbar_expect_tx(full_bar(stage), bytes);
                    const uint32_t dst = stage0 + stage * C::kStageBytes, fb = leader_full + 8u * stage;
                    if (warp == C::kProducerA)
                        tma_load_2d<PAIR>(dst, reinterpret_cast<uint64_t>(&map_a), fb, (int)(kb * 128), (int)(tile_m * C::kTileM + rank * 128));
                    else if (warp == C::kProducerB)
                        tma_load_2d<PAIR>(dst + C::kABytes, reinterpret_cast<uint64_t>(&map_b), fb, (int)(kb * 128),
                                          (int)(tile_n * BN + (PAIR ? rank * (mma_n(tile_n) / 2) : 0u)));
                    else {
                        tma_load_2d<PAIR>(dst + C::kSfa, reinterpret_cast<uint64_t>(&map_sa), fb, (int)(kb * (kScaleBand / 8)),
                                          (int)(tile_m * (C::kTileM / 128) + rank));
                        tma_load_2d<PAIR>(dst + C::kSfb, reinterpret_cast<uint64_t>(&map_sb), fb, (int)(kb * (kScaleBand / 8)), (int)(tile_n * C::kBands));
                    }
                    if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else if (warp == C::kMmaWarp) {
        if (rank == 0) {
            const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0);
            const uint64_t desc0 = smem_desc(__shfl_sync(0xffffffffu, stage0, 0), 0, 1024);
            const uint64_t sdesc0 = scale_desc(__shfl_sync(0xffffffffu, stage0, 0));
            uint32_t stage = 0, phase = 0, it = 0;
            bool ok = true;
            for (uint32_t t = first; ok && t < tiles; t += stride, ++it) {
                const uint32_t idesc = fp4_instr_desc(C::kTileM, mma_n(t / tiles_m));
                // the accumulator is free: its last tile has been read, and, where the two share columns, the other one's these
                if (C::kShared ? it >= 1 : it >= 2) {
                    const uint32_t prev = C::kShared ? it - 1 : it - 2;
                    if (!__all_sync(0xffffffffu, mbar_wait(tempty_bar(prev & 1u), (prev >> 1) & 1u, abort_flag))) break;
                }
                tc_fence_after();
                const uint32_t d_tmem = tmem + (it & 1u) * C::kAcc1;
                for (uint32_t kb = 0; kb < stages; ++kb) {
                    if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag))) { ok = false; break; }
                    tc_fence_after();
                    const uint64_t ad = desc0 + stage * (C::kStageBytes >> 4), bd = ad + (C::kABytes >> 4);
                    const uint64_t sd = sdesc0 + ((stage * C::kStageBytes + C::kSfa) >> 4);
                    if (elect_one()) {
                        // straight-line code: what bounds a stage is how fast one thread issues its sixteen instructions
                        auto copy = [&](uint32_t j) {
                            tc_copy_scales<PAIR>(tmem + C::kSfaCol + 4 * j, sd + j * (kScaleTile >> 4));
#pragma unroll
                            for (uint32_t b = 0; b < C::kBands; ++b)
                                tc_copy_scales<PAIR>(tmem + C::kSfbCol + 4 * (j * C::kBands + b), sd + (((1 + b) * kScaleBand + j * kScaleTile) >> 4));
                        };
                        auto mma = [&](uint32_t j) {
                            tc_mma_fp4<PAIR>(d_tmem, ad + 2 * j, bd + 2 * j, idesc, tmem + C::kSfaCol + 4 * j, tmem + C::kSfbCol + 4 * j * C::kBands,
                                             kb != 0 || j != 0 ? 1u : 0u);
                        };
                        const uint32_t steps = min(4u, (K - kb * kStageK + 63u) / 64u);
                        if (steps == 4) {
                            copy(0); copy(1); copy(2); copy(3);
                            mma(0); mma(1); mma(2); mma(3);
                        } else {
                            for (uint32_t j = 0; j < steps; ++j) {
                                copy(j);
                                mma(j);
                            }
                        }
                        tc_commit<PAIR>(empty_bar(stage));
                        if (kb + 1 == stages) tc_commit<PAIR>(tfull_bar(it & 1u));
                    }
                    __syncwarp();
                    if (++stage == C::kStages) { stage = 0; phase ^= 1u; }
                }
            }
        }
    } else {
        // Warp w reads tensor-memory lanes 32 (w % 4) .. +31, and every other unit of 64 columns.  Results go through slabs in
        // shared memory (32 rows x 128 bytes) to bulk stores of whole lines.
        const uint32_t q = warp & 3, half = (warp - C::kEpiWarp0) >> 2;
        const uint32_t tempty_leader = PAIR ? map_to_cta(tempty_bar(0), 0) : tempty_bar(0);
        uint8_t *slab_bytes = smem + C::kStages * C::kStageBytes + C::kControl + (warp - C::kEpiWarp0) * kSlabBytes;
        float *strip = reinterpret_cast<float *>(smem + C::kStages * C::kStageBytes + C::kControl + C::kEpiWarps * kSlabBytes + (warp - C::kEpiWarp0) * C::kStrip);
        const float sb = epi.b_rows ? 1.0f : *epi.scale_b;
        uint32_t it = 0;
        for (uint32_t t = first; t < tiles; t += stride, ++it) {
            const uint32_t tile_m = t % tiles_m, tile_n = t / tiles_m;
            const uint32_t row0 = tile_m * C::kTileM + rank * 128 + 32 * q, row = row0 + lane;
            const float s = scale_of_row(epi, row) * sb;
            const bool near = epi.b_rows ? s >= 0x1p-100f && s <= 0x1p70f : in_range(s);
            bool far = !__all_sync(0xffffffffu, near);
            const uint32_t n = mma_n(tile_n);
            // where the accumulators share columns, these first: the last ones of the first, the first ones of the second
            auto unit_of = [&](uint32_t i) { return C::kShared && (it & 1u) == 0 ? BN / 64 - 1 - (2 * i + half) : 2 * i + half; };
            float bias[BN / 128][2];   // read before the tile is there
#pragma unroll
            for (uint32_t i = 0; i < BN / 128; ++i)
#pragma unroll
                for (uint32_t k = 0; k < 2; ++k) {
                    const uint32_t col = tile_n * BN + unit_of(i) * 64 + 32 * k + lane;
                    bias[i][k] = epi.bias && col < epi.N ? epi.bias[col] : 0.0f;
                }
            if (!__all_sync(0xffffffffu, mbar_wait(tfull_bar(it & 1u), (it >> 1) & 1u, abort_flag))) break;
            tc_fence_after();
            const uint32_t acc = tmem_base + (it & 1u) * C::kAcc1 + ((32u * q) << 16);
            if (far) {   // not for rows of zeros, whose scale is the least that there is: these lose nothing
                uint32_t any = 0;
                for (uint32_t at = 0; at < n; at += 32) {
                    uint32_t r[32];
                    tc_ld32(acc + at, r);
                    tc_ld_wait();
#pragma unroll
                    for (uint32_t j = 0; j < 32; ++j) any |= r[j] << 1;
                }
                far = !__all_sync(0xffffffffu, near || (any == 0 && s >= 0.0f && s < 0x1p-99f));
            }
            if (far) {   // value by value
                const Scale a = split_scale(scale_of_row(epi, row));
                for (uint32_t k = 0; k < BN / 16; ++k) {
                    const uint32_t at = unit_of(k / 8) * 64 + k % 8 * 8, col0 = tile_n * BN + at;
                    if (at >= n) continue;
                    uint32_t r[8];
                    __syncwarp();
                    tc_ld8(acc + at, r);
                    tc_ld_wait();
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const uint32_t col = col0 + j;
                        if (row >= epi.M || col >= epi.N) continue;
                        const float v = times_scales(__uint_as_float(r[j]), a, split_scale(epi.scale_b[epi.b_rows ? col : 0]), epi.b_rows);
                        store_value(epi, row, col, epi.bias ? v + epi.bias[col] : v);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive_cluster(tempty_leader + 8u * (it & 1u));
                continue;
            }
#pragma unroll 1
            for (uint32_t i = 0; i < BN / 128; ++i) {
                const uint32_t unit = unit_of(i);
                const uint32_t col0 = tile_n * BN + unit * 64;
                uint32_t r[2][32], bits[8];   // bits: eight columns before these, of the first unit those behind what is stored first
                const uint32_t side_col = unit != 0 ? unit * 64 - 8 : epi.type == B2_TYPE_F32 ? 32 : 64;
                if (unit * 64 < n) {
                    tc_ld32(acc + unit * 64, r[0]);
                    if (unit * 64 + 32 < n) tc_ld32(acc + unit * 64 + 32, r[1]);
                    if (!BULK) tc_ld8(acc + side_col, bits);
                    tc_ld_wait();
                }
                if (i == (C::kShared ? 0 : BN / 128 - 1)) {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(tempty_leader + 8u * (it & 1u));
                }
                if (row0 >= epi.M || col0 >= epi.N) continue;
                if (epi.bias) {
                    strip[lane] = i == 0 ? bias[0][0] : bias[BN / 128 - 1][0];
                    strip[lane + 32] = i == 0 ? bias[0][1] : bias[BN / 128 - 1][1];
                    __syncwarp();
                }
                const bool f32 = epi.type == B2_TYPE_F32;
                if (!BULK) {
                    const uint32_t slab = smem_u32(slab_bytes);
                    const bool whole = epi.classes != 0 && row0 + 32 <= epi.M && col0 + (unit == 0 ? 72 : 64) <= epi.N;
                    const bool last = (unit + 1) * 64 == BN || col0 + 128 > epi.N;   // of the tile's whole units
                    if (lane < 8) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");   // the last stores have read the slab
                    __syncwarp();
                    if (!whole) {
#pragma unroll
                        for (uint32_t part = 0; part < 2; ++part) {
                            const uint32_t col = col0 + 32 * part;
                            if (col >= epi.N) continue;
                            float v[32];
                            finish_columns(epi, col, min(32u, epi.N - col), r[part], s, epi.bias ? strip + 32 * part : nullptr, v);
                            store_through(epi, row0, col, v, reinterpret_cast<float *>(slab_bytes));
                        }
                        continue;
                    }
                    float x[8];
#pragma unroll
                    for (uint32_t j = 0; j < 8; ++j) {
                        const uint32_t col = tile_n * BN + side_col + j;
                        x[j] = __uint_as_float(bits[j]) * s;
                        if (epi.b_rows) x[j] *= epi.scale_b[col];
                        if (epi.bias) x[j] += epi.bias[col];
                    }
                    const uint32_t log = 31 - __clz(epi.classes), place = ((lane & (epi.classes - 1)) << (5 - log)) + (lane >> log), slab_row = slab + place * 128;
                    if (f32) {
                        const uint32_t shift = shift_of<4>(epi, lane);
                        float side[4];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) side[j] = unit == 0 ? x[j] : x[4 + j];
#pragma unroll
                        for (uint32_t part = 0; part < 2; ++part) {
                            const uint32_t col = col0 + 32 * part;
                            float v[32];
                            finish_columns(epi, col, 32, r[part], s, epi.bias ? strip + 32 * part : nullptr, v);
                            uint32_t w[32];
                            const bool first = unit == 0 && part == 0, ahead = first && shift != 0;
                            shift_values(side, v, ahead, shift, w);
                            if (ahead) {   // nobody comes before
#pragma unroll
                                for (uint32_t j = 0; j < 3; ++j)
                                    if (j < 4 - shift) store_value(epi, row, col + j, v[j]);
                            }
                            if (part == 1) {
                                if (lane < 8) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                                __syncwarp();
                            }
#pragma unroll
                            for (uint32_t k = 0; k < 8; ++k) st_shared_16(slab_row + ((k ^ (place & 7u)) << 4), w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                            store_classes<4>(epi, reinterpret_cast<uint64_t>(&map_c), row0, col, first, slab);
#pragma unroll
                            for (uint32_t j = 0; j < 4; ++j) side[j] = v[28 + j];
                        }
                        if (last) {   // nobody comes after
#pragma unroll
                            for (uint32_t j = 1; j < 4; ++j)
                                if (j >= 4 - shift) store_value(epi, row, col0 + 60 + j, side[j]);
                        }
                    } else {
                        const uint32_t shift = shift_of<2>(epi, lane), f16 = epi.type == B2_TYPE_F16;
                        const bool ahead = unit == 0 && shift != 0;
                        uint32_t w[36], side[4], mine[32];
#pragma unroll
                        for (uint32_t j = 0; j < 4; ++j) side[j] = pack_operands(x[2 * j], x[2 * j + 1], f16);
#pragma unroll
                        for (uint32_t part = 0; part < 2; ++part) {
                            float v[32];
                            finish_columns(epi, col0 + 32 * part, 32, r[part], s, epi.bias ? strip + 32 * part : nullptr, v);
#pragma unroll
                            for (uint32_t j = 0; j < 16; ++j) mine[16 * part + j] = pack_operands(v[2 * j], v[2 * j + 1], f16);
                        }
                        uint16_t *line = reinterpret_cast<uint16_t *>(epi.c + (uint64_t)row * epi.pitch) + col0;
                        if (ahead) {   // nobody comes before
#pragma unroll
                            for (uint32_t j = 0; j < 7; ++j)
                                if (j < 8 - shift) line[j] = (uint16_t)(mine[j / 2] >> (16 * (j & 1)));
                        }
                        if (last) {   // nobody comes after
#pragma unroll
                            for (uint32_t j = 57; j < 64; ++j)
                                if (j >= 64 - shift) line[j] = (uint16_t)(mine[j / 2] >> (16 * (j & 1)));
                        }
#pragma unroll
                        for (uint32_t j = 0; j < 36; ++j) w[j] = ahead ? (j < 32 ? mine[j & 31] : side[j & 3]) : (j < 4 ? side[j & 3] : mine[(j - 4) & 31]);
                        shift_halves(w, shift);
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k) st_shared_16(slab_row + ((k ^ (place & 7u)) << 4), w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
                        store_classes<2>(epi, reinterpret_cast<uint64_t>(&map_c), row0, col0, unit == 0, slab);
                    }
                    continue;
                }
#pragma unroll
                for (uint32_t part = 0; part < 2; ++part) {
                    const uint32_t col = col0 + 32 * part;
                    if (col >= epi.N) continue;
                    float v[32];
                    finish_columns(epi, col, min(32u, epi.N - col), r[part], s, epi.bias ? strip + 32 * part : nullptr, v);
                    if (epi.accumulate && col + 32 > epi.N) {
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        store_through(epi, row0, col, v, reinterpret_cast<float *>(slab_bytes));
                        continue;
                    }
                    if (f32 || part == 0) {   // the store that read this slab last is through with it
                        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
                        __syncwarp();
                    }
                    const uint32_t slab = smem_u32(slab_bytes), slab_row = slab + lane * 128;
                    if (f32) {
                        if (epi.accumulate && row < epi.M) add_old(epi, row, col, v);
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k)
                            st_shared_16(slab_row + ((k ^ (lane & 7u)) << 4), __float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]),
                                         __float_as_uint(v[4 * k + 2]), __float_as_uint(v[4 * k + 3]));
                    } else {
#pragma unroll
                        for (uint32_t k = 0; k < 4; ++k) {
                            uint32_t w[4];
#pragma unroll
                            for (int j = 0; j < 4; ++j) w[j] = pack_operands(v[8 * k + 2 * j], v[8 * k + 2 * j + 1], epi.type == B2_TYPE_F16);
                            st_shared_16(slab_row + (((4 * part + k) ^ (lane & 7u)) << 4), w[0], w[1], w[2], w[3]);
                        }
                        if (part == 0 && col + 32 < epi.N) continue;
                    }
                    fence_async_smem();
                    __syncwarp();
                    if (lane == 0) tma_store_2d(reinterpret_cast<uint64_t>(&map_c), slab, (int)(f32 ? col : col0), (int)row0);
                }
            }
        }
        if (lane < 8) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 4096; ++i) __nanosleep(512);   // what is in flight lands
        if (threadIdx.x == 0) atomicExch(&g_fp4_status, 1u);
        __syncthreads();
    }
    if (PAIR) cluster_sync_all();
    if (warp == C::kMmaWarp) {
        if (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::kTmemCols) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(C::kTmemCols) : "memory");
    }
}

// ---- few rows of A -----------------------------------------------------------------------------------------------------
// A step of generation: up to 64 rows of A against all of B, which is read once.  A CTA takes 128 rows of B as the MMA's M side and
// the rows of A as its N side.  Where that leaves SMs without work, the CTAs of a cluster share K: rows of A go in groups of four,
// each CTA sends its sums of group j to the CTA of rank j % split, which adds them up in the order of the ranks.
// TYPE >= 0: A is up to eight rows of plain values, which every CTA quantises for itself while its first tiles of B are on their
// way, and the quantiser's launch and its way through memory are saved.
// (The same with B decoded to FP16 for mma.sync, without tensor memory and maps, spent five instructions on a code: 31 us for
// 1 x 1600 -> 50304, and 7.2 for 1 x 1600 -> 4800.)
constexpr uint32_t kFewRows = 64, kFusedRows = 8;
constexpr uint32_t kFewSplit = 8;       // CTAs of a cluster at most
constexpr uint32_t kFewMaxStages = 12;
constexpr uint32_t kFewControl = 1024;
constexpr int kFewThreads = 256;

__device__ __forceinline__ void st_cluster_16(uint32_t addr, const uint32_t *v) {
    asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}

template <bool FAR>
__device__ __forceinline__ float times(float sum, float ga, float gb) {
    return FAR ? times_scales(sum, split_scale(ga), split_scale(gb), false) : sum * (ga * gb);
}

struct FewShape {
    uint32_t K;
    uint32_t n;            // rows of A, rounded up to a multiple of 8
    uint32_t split;        // CTAs of a cluster
    uint32_t stages;       // of the pipeline
    uint32_t share;        // stages of K that a CTA has at most
    uint32_t tmem_cols;
    // plain values
    const uint8_t *x;
    uint64_t x_pitch;      // bytes
    uint32_t x_cols, x_access;
};
// Shared memory behind the 1024 bytes of barriers and the rows' scales: the pipeline's stages; TYPE >= 0: codes and scales of the
// rows of A for the CTA's part of K; the sums that the cluster sends.
struct FewLayout {
    uint32_t at_a, at_sb, at_sa, stage_bytes;   // in a stage: 128 rows of B (at 0), rows of A, scales
    uint32_t at_x, at_xs, at_sums, bytes;
};
__host__ __device__ inline FewLayout few_layout(const FewShape &f, bool fused) {
    FewLayout l;
    l.at_a = 128 * 128;
    l.at_sb = l.at_a + (fused ? 0u : f.n * 128);
    l.at_sa = l.at_sb + kScaleBand;
    l.stage_bytes = l.at_sa + (fused ? 0u : kScaleBand);
    l.stage_bytes = (l.stage_bytes + 1023) / 1024 * 1024;
    l.at_x = kFewControl + f.stages * l.stage_bytes;
    l.at_xs = l.at_x + (fused ? f.share * 1024 : 0u);
    l.at_sums = l.at_xs + (fused ? f.share * 512 + 512 : 0u);
    l.bytes = l.at_sums + (f.split > 1 ? f.split * (((f.n + 3) / 4 + f.split - 1) / f.split) * 2048 : 0u);
    return l;
}

template <int TYPE>
__global__ void __launch_bounds__(kFewThreads)
k_fp4_few(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_sa,
          const __grid_constant__ CUtensorMap map_sb, const __grid_constant__ Epilogue epi, const __grid_constant__ FewShape shape) {
    constexpr bool kFused = TYPE >= 0;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t n = shape.n, split = shape.split, pipe = shape.stages;
    const FewLayout lay = few_layout(shape, kFused);
    uint64_t *bars = reinterpret_cast<uint64_t *>(smem);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(bars + 2 * kFewMaxStages + 2);
    volatile uint32_t *abort_flag = tmem_slot + 1;
    uint32_t *maxima = tmem_slot + 2;                              // of up to eight rows of plain values
    uint32_t *ends = maxima + kFusedRows;                          // the least and the greatest of the rows' scales, of 32 rows each
    float *tops = reinterpret_cast<float *>(smem + 512);           // the rows of A's scales
    static_assert((2 * kFewMaxStages + 2) * 8 + 8 + kFusedRows * 4 + 16 <= 512 && kFewRows * 4 <= 512, "control region");
    const uint32_t stage0 = smem_u32(smem) + kFewControl;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = split > 1 ? cluster_cta_rank() : 0u, tile = blockIdx.x / split;
    const uint32_t bar0 = smem_u32(bars);
    auto full_bar = [&](uint32_t s) { return bar0 + 8u * s; };
    auto empty_bar = [&](uint32_t s) { return bar0 + 8u * (kFewMaxStages + s); };
    const uint32_t done_bar = bar0 + 8u * (2 * kFewMaxStages), x_bar = done_bar + 8u;
    // this CTA's part of K, in stages
    const uint32_t all = (shape.K + kStageK - 1) / kStageK;
    const uint32_t kb0 = all * rank / split, kb1 = all * (rank + 1) / split;

    if (threadIdx.x == 0) {
        for (uint32_t s = 0; s < pipe; ++s) {
            mbar_init(full_bar(s), kFused ? 1 : 2);
            mbar_init(empty_bar(s), 1);
        }
        mbar_init(done_bar, 1);
        mbar_init(x_bar, kFewThreads - 64);
        *abort_flag = 0;
        for (uint32_t i = 0; i < kFusedRows; ++i) maxima[i] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async_smem();
        if (!kFused) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_a) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&map_sa) : "memory");
        }
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_b) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_sb) : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(shape.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *tmem_slot;
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this CTA runs: it can be sent to
    stream_enter();

    auto ends_of = [&](uint32_t j, float top) {   // by two warps, j = 0 .. 63
        const uint32_t least = __reduce_min_sync(0xffffffffu, __float_as_uint(top)), greatest = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
        if ((j & 31u) == 0) {
            ends[j / 16] = least;
            ends[j / 16 + 1] = greatest;
        }
    };
    // whether no product of a row's scale and this one is far out (a scale that is negative or NaN counts as that)
    auto near = [&](float sb) {
        bool all = true;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) all = all && in_range(__uint_as_float(ends[i]) * sb);
        return all;
    };
    if (warp == 0 || (!kFused && warp == 2)) {
        if (lane == 0) {
            for (uint32_t kb = kb0; kb < kb1; ++kb) {
                const uint32_t i = kb - kb0, stage = i % pipe, phase = i / pipe & 1u;
                if (!mbar_wait(empty_bar(stage), phase ^ 1u, abort_flag)) break;
                const uint32_t dst = stage0 + stage * lay.stage_bytes;
                if (warp == 0) {
                    mbar_expect_tx(full_bar(stage), 128 * 128 + kScaleBand);
                    tma_load_2d<false>(dst, reinterpret_cast<uint64_t>(&map_b), full_bar(stage), (int)(kb * 128), (int)(tile * 128));
                    tma_load_2d<false>(dst + lay.at_sb, reinterpret_cast<uint64_t>(&map_sb), full_bar(stage), (int)(kb * (kScaleBand / 8)), (int)tile);
                } else {
                    mbar_expect_tx(full_bar(stage), n * 128 + kScaleBand);
                    tma_load_2d<false>(dst + lay.at_a, reinterpret_cast<uint64_t>(&map_a), full_bar(stage), (int)(kb * 128), 0);
                    tma_load_2d<false>(dst + lay.at_sa, reinterpret_cast<uint64_t>(&map_sa), full_bar(stage), (int)(kb * (kScaleBand / 8)), 0);
                }
            }
        }
    } else if (warp == 1) {
        const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_base, 0), idesc = fp4_instr_desc(128, n);
        const uint32_t sb_col = tmem + (n + 31) / 32 * 32, sa_col = sb_col + 16;
        const uint64_t desc0 = smem_desc(stage0, 0, 1024), sdesc0 = scale_desc(stage0);
        bool ok = !kFused || __all_sync(0xffffffffu, mbar_wait(x_bar, 0, abort_flag));
        for (uint32_t kb = kb0; ok && kb < kb1; ++kb) {
            const uint32_t i = kb - kb0, stage = i % pipe, phase = i / pipe & 1u;
            if (!__all_sync(0xffffffffu, mbar_wait(full_bar(stage), phase, abort_flag))) break;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t at = stage * lay.stage_bytes;
                const uint64_t bd = desc0 + (at >> 4), sbd = sdesc0 + ((at + lay.at_sb) >> 4);
                const uint64_t ad = kFused ? smem_desc(smem_u32(smem) + lay.at_x + i * 1024, 0, 1024) : bd + (lay.at_a >> 4);
                const uint64_t sad = kFused ? scale_desc(smem_u32(smem) + lay.at_xs + i * 512) : sdesc0 + ((at + lay.at_sa) >> 4);
                const uint32_t steps = min(4u, (shape.K - kb * kStageK + 63u) / 64u);
                for (uint32_t j = 0; j < steps; ++j) {
                    tc_copy_scales<false>(sb_col + 4 * j, sbd + j * (kScaleTile >> 4));
                    tc_copy_scales<false>(sa_col + 4 * j, sad + j * ((kFused ? 128u : kScaleTile) >> 4));
                }
                for (uint32_t j = 0; j < steps; ++j)
                    tc_mma_fp4<false>(tmem, bd + 2 * j, ad + 2 * j, idesc, sb_col + 4 * j, sa_col + 4 * j, kb != kb0 || j != 0 ? 1u : 0u);
                tc_commit<false>(empty_bar(stage));
                if (kb + 1 == kb1) tc_commit<false>(done_bar);
            }
            __syncwarp();
        }
    } else if (kFused) {
        // Rows' maxima over all of K, then this CTA's part of K: codes as 8 rows of 128 bytes in the 128-byte swizzle for a stage, a
        // scale tile of 128 bytes for 64 values (rows 0 .. 7; what the copy reads behind them belongs to rows that do not exist).
        constexpr int T = kFused ? TYPE : 0;
        const uint32_t t = threadIdx.x - 64, blocks = shape.K / 16;
        auto load = [&](Raw<T> &r, uint32_t row, uint32_t blk) {
            if (blk * 16 >= shape.x_cols) r.clear();
            else r.load(shape.x + row * shape.x_pitch + (uint64_t)blk * 16 * Raw<T>::kSize, (int)min(shape.x_cols - blk * 16, 16u), shape.x_access);
        };
        for (uint32_t i = t; i < epi.M * blocks; i += kFewThreads - 64) {
            Raw<T> r;
            load(r, i / blocks, i % blocks);
            atomicMax(maxima + i / blocks, r.amax_bits());
        }
        asm volatile("bar.sync 1, %0;" ::"n"(kFewThreads - 64) : "memory");
        const uint32_t first = kb0 * (kStageK / 16), mine = min((blocks + 3) / 4 * 4, kb1 * (kStageK / 16)) - first;
        for (uint32_t i = t; i < epi.M * mine; i += kFewThreads - 64) {
            const uint32_t row = i / mine, blk = i % mine;
            const float g = top_scale(maxima[row]), inv = top_inverse(g);
            Raw<T> r;
            load(r, row, first + blk);
            uint2 codes;
            const uint32_t s = encode_block(r, r.amax_bits(), g, inv, codes);
            const uint32_t in_stage = blk % (kStageK / 16);
            *reinterpret_cast<uint2 *>(smem + lay.at_x + blk / (kStageK / 16) * 1024 + row * 128 + (((in_stage >> 1) ^ row) << 4) + (in_stage & 1u) * 8) = codes;
            smem[lay.at_xs + blk / 4 * 128 + row * 16 + (blk & 3u)] = (uint8_t)s;
        }
        if (t < epi.M) tops[t] = top_scale(maxima[t]);
        fence_async_smem();   // the tensor core reads what these threads have written
        mbar_arrive(x_bar);
        if (t < 64) ends_of(t, t < epi.M ? top_scale(maxima[t]) : 1.0f);
    } else if (warp >= 4) {
        const uint32_t j = threadIdx.x - 128;
        const float top = j < epi.M ? epi.scale_a[epi.a_rows ? j : 0] : 1.0f;
        if (j < epi.M) tops[j] = top;
        if (j < 64) ends_of(j, top);
    }
    bool ok = true;
    if (warp >= 4) ok = __all_sync(0xffffffffu, mbar_wait(done_bar, 0, abort_flag));
    __syncthreads();
    tc_fence_after();
    const uint32_t groups = (epi.M + 3) / 4, held = (groups + split - 1) / split;   // groups of four rows, and those a CTA adds up
    if (split > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (warp >= 4 && ok) {
        const uint32_t q = warp & 3, at = 32 * q + lane, col_n = tile * 128 + at;   // a row of B: a column of C
        const float sb = col_n < epi.N ? epi.scale_b[epi.b_rows ? col_n : 0] : 0.0f;
        const float bias = epi.bias && col_n < epi.N ? epi.bias[col_n] : 0.0f;
        const uint32_t to = smem_u32(smem) + lay.at_sums + (rank * held * 128 + at) * 16;
        auto rows = [&](auto is_far) {
            constexpr bool FAR = decltype(is_far)::value;
            for (uint32_t j0 = 0; j0 < epi.M; j0 += 32) {
                uint32_t r[32];
                tc_ld32(tmem_base + ((32u * q) << 16) + j0, r);
                tc_ld_wait();
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j) {
                    const uint32_t group = j0 / 4 + j;
                    if (group >= groups) break;
                    if (split > 1) {
                        st_cluster_16(map_to_cta(to + group / split * 2048, group % split), r + 4 * j);
                    } else if (col_n < epi.N) {
#pragma unroll
                        for (uint32_t i = 0; i < 4; ++i)
                            if (4 * group + i < epi.M) store_value(epi, 4 * group + i, col_n, times<FAR>(__uint_as_float(r[4 * j + i]), tops[4 * group + i], sb) + bias);
                    }
                }
            }
        };
        if (__all_sync(0xffffffffu, split > 1 || col_n >= epi.N || near(sb))) rows(std::false_type{});
        else rows(std::true_type{});
        tc_fence_before();
    }
    if (split > 1) {
        const uint32_t at = threadIdx.x & 127u, col_n = tile * 128 + at;
        const float sb = col_n < epi.N ? epi.scale_b[epi.b_rows ? col_n : 0] : 1.0f, bias = epi.bias && col_n < epi.N ? epi.bias[col_n] : 0.0f;
        const bool plain = near(sb);
        cluster_sync_all();
        if (col_n < epi.N) {
            auto rows = [&](auto is_far) {
                constexpr bool FAR = decltype(is_far)::value;
                for (uint32_t group = rank + threadIdx.x / 128 * split; group < groups; group += 2 * split) {
                    float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                    for (uint32_t p = 0; p < split; ++p) {
                        const float4 o = *reinterpret_cast<const float4 *>(smem + lay.at_sums + ((p * held + group / split) * 128 + at) * 16);
                        v[0] += o.x; v[1] += o.y; v[2] += o.z; v[3] += o.w;
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        if (4 * group + i < epi.M) store_value(epi, 4 * group + i, col_n, times<FAR>(v[i], tops[4 * group + i], sb) + bias);
                }
            };
            if (plain) rows(std::false_type{});
            else rows(std::true_type{});
        }
    }
    __syncthreads();
    if (*abort_flag) {
        for (int i = 0; i < 4096; ++i) __nanosleep(512);   // what is in flight lands
        if (threadIdx.x == 0) atomicExch(&g_fp4_status, 1u);
        __syncthreads();
    }
    if (warp == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(shape.tmem_cols) : "memory");
}

// ---- host ---------------------------------------------------------------------------------------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                   const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion,
                                   CUtensorMapFloatOOBfill);
EncodeTiledFn encode_tiled() {
    static const EncodeTiledFn fn = [] {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess) p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    return fn;
}
// Codes: rows of cols / 2 bytes (bytes behind them read as zero), boxes of 128 bytes x box_rows, 128-byte swizzle.
bool codes_map(CUtensorMap *m, const b2_nvfp4_operand &o, uint32_t box_rows) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const cuuint64_t dims[2] = {o.cols / 2, o.rows}, strides[1] = {o.row_bytes};
    const cuuint32_t box[2] = {128, box_rows}, step[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, o.bytes, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Scales: a row of 8-byte words for every band of 128 rows, boxes of a stage's worth x box_bands.
bool scales_map(CUtensorMap *m, const b2_nvfp4_operand &o, uint32_t box_bands) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const uint64_t tiles = (o.cols / 16 + 3) / 4;
    const cuuint64_t dims[2] = {tiles * (kScaleTile / 8), ((uint64_t)o.rows + 127) / 128}, strides[1] = {tiles * kScaleTile};
    const cuuint32_t box[2] = {kScaleBand / 8, box_bands}, step[2] = {1, 1};
    return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT64, 2, o.scales, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// C: boxes of 32 rows x 128 bytes, as the epilogue's slabs hold them.
bool result_map(CUtensorMap *m, const b2_matrix &c) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const uint32_t size = c.type == B2_TYPE_F32 ? 4 : 2;
    const cuuint64_t dims[2] = {c.cols, c.rows}, strides[1] = {c.ld * size};
    const cuuint32_t box[2] = {128 / size, 32}, step[2] = {1, 1};
    return fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, c.data, dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// C with rows on any boundary: boxes of 128 bytes x the rows of a class in a slab.
bool classes_map(CUtensorMap *m, const b2_matrix &c, const Epilogue &e) {
    const EncodeTiledFn fn = encode_tiled();
    if (!fn) return false;
    const uint32_t size = c.type == B2_TYPE_F32 ? 4 : 2;
    const cuuint64_t dims[3] = {(uint64_t)e.offset + (e.classes - 1) * e.step + c.cols, e.classes, (c.rows + e.classes - 1) / e.classes};
    const cuuint64_t strides[2] = {e.pitch / 16 * 16, e.pitch * e.classes};
    const cuuint32_t box[3] = {128 / size, 1, 32 / e.classes}, step[3] = {1, 1, 1};
    return fn(m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, e.c - e.offset * size, dims, strides, box, step,
              CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <bool PAIR, int BN, bool BULK>
cudaError_t gemm_launch(const b2_nvfp4_operand &a, const b2_nvfp4_operand &b, const b2_matrix &c, const Epilogue &epi, int sm_count, cudaStream_t s) {
    using C = FCfg<PAIR, BN>;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(k_fp4_gemm<PAIR, BN, BULK>, C::kSmemBytes, done);
    if (e != cudaSuccess) return e;
    CUtensorMap map_a, map_b, map_sa, map_sb, map_c = {};
    if (!codes_map(&map_a, a, 128) || !codes_map(&map_b, b, C::kBRows) || !scales_map(&map_sa, a, 1) || !scales_map(&map_sb, b, C::kBands) ||
        (BULK && !result_map(&map_c, c)) || (!BULK && epi.classes != 0 && !classes_map(&map_c, c, epi)))
        return cudaErrorInvalidValue;
    const uint32_t tiles_m = (a.rows + C::kTileM - 1) / C::kTileM, tiles_n = (b.rows + BN - 1) / BN;
    const uint64_t tiles = (uint64_t)tiles_m * tiles_n;
    if (tiles > 0x7fffffffu) return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = 2;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = PAIR ? 2 : 1;
    const uint32_t groups = (uint32_t)std::min<uint64_t>(tiles, PAIR ? sm_count / 2 : sm_count);
    cfg.gridDim = dim3(PAIR ? 2 * groups : groups);
    cfg.blockDim = dim3(C::kThreads);
    cfg.dynamicSmemBytes = C::kSmemBytes;
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, k_fp4_gemm<PAIR, BN, BULK>, map_a, map_b, map_sa, map_sb, map_c, epi, a.cols, tiles_m, (uint32_t)tiles);
}

template <bool PAIR, int BN>
cudaError_t gemm_impl(const b2_nvfp4_operand &a, const b2_nvfp4_operand &b, const b2_matrix &c, const Epilogue &epi, int sm_count, cudaStream_t s) {
    // a bulk store writes whole 16-byte pieces: where a row's last one is not all its own, the bytes behind the row would change
    const uint32_t size = c.type == B2_TYPE_F32 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(c.data);
    if (at % 16 == 0 && epi.pitch % 16 == 0 && (uint64_t)c.cols * size % 16 == 0) return gemm_launch<PAIR, BN, true>(a, b, c, epi, sm_count, s);
    Epilogue moved = epi;
    if (!epi.accumulate && c.cols > 64 && c.rows >= 32) {   // (old values are added value by value)
        moved.classes = 1;
        while (moved.classes * (epi.pitch % 16) % 16 != 0) moved.classes *= 2;
        moved.offset = (uint32_t)(at % 16 / size);
        moved.step = (uint32_t)(epi.pitch % 16 / size);
    }
    return gemm_launch<PAIR, BN, false>(a, b, c, moved, sm_count, s);
}

// `x`: plain values in A's place (TYPE is theirs), else null
template <int TYPE>
cudaError_t few_impl(const b2_nvfp4_operand *a, const b2_matrix *x, const b2_nvfp4_operand &b, const Epilogue &epi, int sm_count, cudaStream_t s) {
    constexpr bool kFused = TYPE >= 0;
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_smem(k_fp4_few<TYPE>, (uint32_t)kSmemLimit, done);
    if (e != cudaSuccess) return e;
    FewShape f = {};
    f.K = b.cols;
    f.n = (epi.M + 7) / 8 * 8;
    if (kFused) {
        f.x = static_cast<const uint8_t *>(x->data);
        f.x_pitch = x->ld * Raw<kFused ? TYPE : 0>::kSize;
        f.x_cols = x->cols;
        f.x_access = access_of(x->data, f.x_pitch);
    }
    const uint32_t tiles = (b.rows + 127) / 128, all = (b.cols + kStageK - 1) / kStageK;
    f.split = std::max(1u, std::min({kFewSplit, all, (uint32_t)sm_count / tiles}));
#ifdef B2_MEASURE
    if (const char *v = getenv("B2_FP4_SPLIT")) f.split = std::min((uint32_t)atoi(v), all);
#endif
    f.share = (all + f.split - 1) / f.split;
    // where there are tiles for several CTAs an SM, a short pipeline leaves room for them
    f.stages = std::min({kFewMaxStages, f.share, tiles * f.split > (uint32_t)sm_count ? 3u : kFewMaxStages});
#ifdef B2_MEASURE
    if (const char *v = getenv("B2_FP4_STAGES")) f.stages = std::min((uint32_t)atoi(v), f.share);
#endif
    while (f.stages > 1 && few_layout(f, kFused).bytes > (uint32_t)kSmemLimit - 1024) --f.stages;
    f.tmem_cols = 32;
    while (f.tmem_cols < (f.n + 31) / 32 * 32 + 32) f.tmem_cols *= 2;
    // A CTA keeps its tensor memory while it waits for the others of its cluster, so none of them may have to wait for tensor
    // memory in turn: every launch takes at least the share of an SM's shared memory (228 KB, 1 KB of it for the system) that it
    // takes of the tensor memory, and more than a Newton-Schulz CTA that holds all of it leaves; with a cluster, more than other
    // programs' tensor-core kernels do that take half of an SM's shared memory (two such launches still fit an SM, so that one begins
    // while the other ends).
    const uint32_t bytes = std::max({few_layout(f, kFused).bytes + 1024, 228u * 1024 / 512 * f.tmem_cols - 1024, (f.split > 1 ? 108u : 40u) * 1024});
    CUtensorMap map_a = {}, map_b, map_sa = {}, map_sb;
    if ((!kFused && (!codes_map(&map_a, *a, f.n) || !scales_map(&map_sa, *a, 1))) || !codes_map(&map_b, b, 128) || !scales_map(&map_sb, b, 1))
        return cudaErrorInvalidValue;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = f.split;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = f.split > 1 ? 2 : 1;
    cfg.gridDim = dim3(tiles * f.split);
    cfg.blockDim = dim3(kFewThreads);
    cfg.dynamicSmemBytes = bytes;
    cfg.stream = s;
    return cudaLaunchKernelEx(&cfg, k_fp4_few<TYPE>, map_a, map_b, map_sa, map_sb, epi, f);
}

Epilogue epilogue_of(const b2_nvfp4_operand &b, const b2_matrix &c, const float *bias, bool accumulate) {
    Epilogue epi = {};
    epi.c = static_cast<uint8_t *>(c.data);
    epi.pitch = c.ld * (c.type == B2_TYPE_F32 ? 4 : 2);
    epi.scale_b = b.scale;
    epi.bias = bias;
    epi.M = c.rows;
    epi.N = c.cols;
    epi.b_rows = b.scale_count != 1;
    epi.type = c.type;
    epi.accumulate = accumulate;
    return epi;
}

}  // namespace

cudaError_t launch_fp4_matmul(const b2_nvfp4_operand &a, const b2_nvfp4_operand &b, const b2_matrix &c, const float *bias, bool accumulate,
                              int sm_count, cudaStream_t s) {
    Epilogue epi = epilogue_of(b, c, bias, accumulate);
    epi.scale_a = a.scale;
    epi.a_rows = a.scale_count != 1;
#ifdef B2_MEASURE
    if (const char *v = getenv("B2_FP4_SHAPE")) {
        const int k = atoi(v);
        if (k == 0 && a.rows <= kFewRows) return few_impl<-1>(&a, nullptr, b, epi, sm_count, s);
        if (k == 1) return gemm_impl<false, 128>(a, b, c, epi, sm_count, s);
        if (k == 3) return gemm_impl<true, 256>(a, b, c, epi, sm_count, s);
    }
#endif
    // Few rows: 24 x 1600 -> 50304 takes 8.7 us, in tiles 15.0; 24 x 6400 -> 1600, eight CTAs sharing K, 5.8 and 10.8; 16 x 768 ->
    // 2304 is about even (4.3, 3.8).  From 33 rows on only a long K pays: 64 x 6400 -> 1600 7.2 and 11.1, 64 x 1600 -> 4800 7.6 and 5.5.
    if (a.rows <= kFewRows / 2 || (a.rows <= kFewRows && a.cols >= 4096)) return few_impl<-1>(&a, nullptr, b, epi, sm_count, s);
    // Tiles of one CTA while every one of them has an SM to itself (777 x 1600 -> 1600 6.0 us, in pairs 7.0; 1000 x 768 -> 2304 4.7
    // and 5.8), else pairs, which take in half as much for an operation (200 x 1600 -> 50304 20.9 and 14.8; 2000 x 6400 -> 1600 20.8
    // and 13.3; 512 x 1600 -> 4800, 152 tiles, 8.0 and 7.2).
    const uint64_t tiles = (uint64_t)((a.rows + 127) / 128) * ((b.rows + 127) / 128);
    if (tiles > (uint64_t)sm_count) return gemm_impl<true, 256>(a, b, c, epi, sm_count, s);
    return gemm_impl<false, 128>(a, b, c, epi, sm_count, s);
}

// Quantised on the way and as a launch of its own: 1 x 1600 -> 4800 5.4 us and 6.6, 4 x 1600 -> 4800 6.4 and 6.8, 8 x 1600 -> 4800 7.6
// and 7.0, 1 x 6400 -> 1600 6.8 and 7.2, 2 x 6400 -> 1600 7.8 and 7.4.
bool fp4_linear_fused(uint32_t rows, uint32_t cols) { return rows <= kFusedRows && (uint64_t)rows * cols <= 8192; }

cudaError_t launch_fp4_linear(const b2_matrix &x, const b2_nvfp4_operand &b, const b2_matrix &c, const float *bias, int sm_count, cudaStream_t s) {
    const Epilogue epi = epilogue_of(b, c, bias, false);
    if (x.type == B2_TYPE_F32) return few_impl<B2_TYPE_F32>(nullptr, &x, b, epi, sm_count, s);
    if (x.type == B2_TYPE_BF16) return few_impl<B2_TYPE_BF16>(nullptr, &x, b, epi, sm_count, s);
    return few_impl<B2_TYPE_F16>(nullptr, &x, b, epi, sm_count, s);
}

cudaError_t fp4_gemm_status(uint32_t *status, cudaStream_t s) {
    uint32_t *word = nullptr;
    cudaError_t e = cudaGetSymbolAddress(reinterpret_cast<void **>(&word), g_fp4_status);
    if (e == cudaSuccess) e = cudaMemcpyAsync(status, word, sizeof *status, cudaMemcpyDeviceToHost, s);
    if (e == cudaSuccess) e = cudaMemsetAsync(word, 0, sizeof *word, s);
    if (e == cudaSuccess) e = cudaStreamSynchronize(s);
    return e;
}

}  // namespace b2

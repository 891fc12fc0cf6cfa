// Quantisation of activations and gradients to NVFP4 by rows and by columns, reading 4-bit tensors back, and the paged cache.
// All of it streams: the bytes bound these kernels from below, and at 220 instructions a block the quantisers' arithmetic is about as
// long, so they issue in 60 to 70 % of the cycles.
//
// The work is 16 values a thread, a whole block, so its maximum needs no exchange.  Measured, BF16, inputs partly in L2 as a layer's
// are; in brackets the bytes at the rate of a copy: 16384 x 1600 by rows 12.8 us (10.3); by columns 19.4, 8 of them the maximum
// (10.3, 18.3 with x read twice); decode by rows 14.3, of 1600 x 16384 10.6 (10.3); 32768 tokens of two 16 x 64 vectors written to the
// cache 35 us (26.5), as many read back 31 (26.5).
#include <algorithm>

#include "common.cuh"
#include "fp4.h"
#include "fp4_block.cuh"

namespace b2 {

namespace {

// ---- a tensor's maximum -----------------------------------------------------------------------------------------------------
struct MaximaJob {
    const uint8_t *x;        // rows without gaps are one row
    uint64_t ld_bytes, cols;
    uint32_t rows, ctas;
    const float *tops;       // or what is known already: scales on top of parts of the tensor
    uint32_t top_count, access;
    float *maxima;           // a scale for every CTA's part
};
// Part `cta` of job.ctas, in CTAs of 256 threads or 512.
template <int TYPE>
__device__ __forceinline__ void part_of_maximum(const MaximaJob &j, uint32_t cta) {
    __shared__ uint32_t part[16];
    const uint32_t threads = blockDim.x, warps = threads / 32;
    uint32_t m = 0;
    const uint64_t blocks = (j.cols + 15) / 16;
    const uint32_t access = j.access;
    auto take = [&](const uint8_t *src, uint64_t blk) {
        Raw<TYPE> r;
        r.load(src + blk * 16 * Raw<TYPE>::kSize, j.cols - blk * 16 < 16 ? (int)(j.cols - blk * 16) : 16, access);
        m = max_bits(m, r.amax_bits());
    };
    if (j.tops) {
        for (uint32_t i = cta * threads + threadIdx.x; i < j.top_count; i += j.ctas * threads) m = max_bits(m, __float_as_uint(j.tops[i]));
    } else if (j.rows == 1) {
#pragma unroll 4
        for (uint64_t blk = cta * (uint64_t)threads + threadIdx.x; blk < blocks; blk += j.ctas * (uint64_t)threads) take(j.x, blk);
    } else {
        for (uint32_t row = cta * warps + (threadIdx.x >> 5); row < j.rows; row += j.ctas * warps)
#pragma unroll 4
            for (uint64_t blk = threadIdx.x & 31u; blk < blocks; blk += 32) take(j.x + (uint64_t)row * j.ld_bytes, blk);
    }
    m = warp_max_bits(m);
    if ((threadIdx.x & 31u) == 0) part[threadIdx.x >> 5] = m;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < warps; ++i) m = max_bits(m, part[i]);
        j.maxima[cta] = j.tops ? __uint_as_float(m) : top_scale(m);
    }
}

// ---- by rows ----------------------------------------------------------------------------------------------------------------
// The row's maximum has to be there before its first code: the row waits in registers.  WPR warps a row; a thread holds kHeld blocks of it, so a row of up to WPR * 32 * kHeld blocks is read once.  A longer one
// (HELD false) is read twice, the second time out of L2 where it fits.  CTAs behind row_ctas take the maximum of another tensor.
constexpr int kHeld = 4;
template <int TYPE, int WPR, bool HELD>
__global__ void __launch_bounds__(WPR == 16 ? 512 : 256)
k_fp4_quantize_rows(const uint8_t *x, uint64_t ld_bytes, uint32_t rows, uint32_t cols, uint32_t access, uint8_t *bytes, uint64_t row_bytes,
                    uint8_t *scales, float *scale, uint32_t row_ctas, const __grid_constant__ MaximaJob other) {
    stream_enter();
    if (blockIdx.x >= row_ctas) {
        part_of_maximum<TYPE>(other, blockIdx.x - row_ctas);
        return;
    }
    constexpr int kWarps = WPR == 16 ? 16 : 8, kRowsPerCta = kWarps / WPR, kThreadsPerRow = 32 * WPR;
    __shared__ uint32_t part[kWarps];
    const uint32_t warp = threadIdx.x >> 5, in_row = threadIdx.x % kThreadsPerRow;
    const uint32_t row = blockIdx.x * kRowsPerCta + threadIdx.x / kThreadsPerRow;
    const bool there = row < rows;
    const uint32_t blocks = (cols + 15) / 16, tiles = (blocks + 3) / 4;
    const uint8_t *src = x + (uint64_t)row * ld_bytes;
    auto fetch = [&](Raw<TYPE> &r, uint32_t blk) {
        if (there && blk < blocks) r.load(src + (uint64_t)blk * 16 * Raw<TYPE>::kSize, (int)min(cols - blk * 16u, 16u), access);
        else r.clear();
    };
    Raw<TYPE> held[HELD ? kHeld : 1];
    uint32_t m = 0;
    if (HELD) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i) fetch(held[i], in_row + i * kThreadsPerRow);
#pragma unroll
        for (int i = 0; i < kHeld; ++i) m = max_bits(m, held[i].amax_bits());
    } else {
        for (uint32_t blk = in_row; blk < blocks; blk += kThreadsPerRow) {
            fetch(held[0], blk);
            m = max_bits(m, held[0].amax_bits());
        }
    }
    m = warp_max_bits(m);
    if (WPR > 1) {
        if ((threadIdx.x & 31u) == 0) part[warp] = m;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < WPR; ++i) m = max_bits(m, part[warp / WPR * WPR + i]);
    }
    const float g = top_scale(m), inv = top_inverse(g);
    if (there && in_row == 0) scale[row] = g;
    auto store = [&](const Raw<TYPE> &r, uint32_t blk) {
        uint2 codes;
        uint32_t s = encode_block(r, r.amax_bits(), g, inv, codes);
        if (there && blk < blocks) *reinterpret_cast<uint2 *>(bytes + (uint64_t)row * row_bytes + (uint64_t)blk * 8) = codes;
        s |= __shfl_down_sync(0xffffffffu, s, 1) << 8;   // four blocks' scales, one word of a 512-byte tile
        s |= __shfl_down_sync(0xffffffffu, s, 2) << 16;
        if (there && (blk & 3u) == 0 && blk < tiles * 4u) *reinterpret_cast<uint32_t *>(scales + sm100_scale_offset(row, blk, tiles)) = s;
    };
    if (HELD) {
#pragma unroll
        for (int i = 0; i < kHeld; ++i)
            if (i * kThreadsPerRow < (int)blocks) store(held[i], in_row + i * kThreadsPerRow);
    } else {
        const uint32_t turns = (blocks + kThreadsPerRow - 1) / kThreadsPerRow;
        for (uint32_t i = 0; i < turns; ++i) {
            fetch(held[0], in_row + i * kThreadsPerRow);
            store(held[0], in_row + i * kThreadsPerRow);
        }
    }
}

// ---- by columns -------------------------------------------------------------------------------------------------------------
// Both gradients' operands go through these in one launch: blockIdx.y is the tensor.
struct MaximaJobs {
    MaximaJob job[2];
};
template <int TYPE>
__global__ void __launch_bounds__(256, TYPE == B2_TYPE_F32 ? 4 : 6)
k_fp4_maxima(const __grid_constant__ MaximaJobs jobs) {
    stream_enter();
    if (blockIdx.x < jobs.job[blockIdx.y].ctas) part_of_maximum<TYPE>(jobs.job[blockIdx.y], blockIdx.x);
}

// A CTA transposes tiles of 128 rows x 128 columns: a warp takes 16 rows, a lane four columns of them, so that a thread holds
// four whole blocks of the transpose and their codes only change places on the way to memory, through shared memory.
constexpr int kTile = 128;
struct ColumnsJob {
    const uint8_t *x;
    uint64_t ld_bytes;
    uint32_t rows, cols;
    uint8_t *bytes;
    uint64_t row_bytes;
    uint8_t *scales;
    float *scale;
    const float *maxima;   // scales on top of parts of the tensor: theirs is the largest
    uint32_t count, vec;
};
struct ColumnsJobs {
    ColumnsJob job[2];
};
// (Four CTAs an SM: with three, 74 registers a thread, 16384 x 1600 takes 20.2 us instead of 19.5, 2048 x 50257 190 instead of 145.)
template <int TYPE>
__global__ void __launch_bounds__(256, TYPE == B2_TYPE_F32 ? 2 : 4)
k_fp4_quantize_columns(const __grid_constant__ ColumnsJobs jobs) {
    stream_enter();
    __shared__ uint2 codes_tile[kTile * 8];   // [column][block of 16 rows], the blocks of a column in an order of its own
    __shared__ __align__(16) uint8_t scales_tile[2 * 512];
    __shared__ uint32_t part[8];
    const ColumnsJob &job = jobs.job[blockIdx.y];
    const uint32_t rows = job.rows, cols = job.cols;
    const uint64_t ld_bytes = job.ld_bytes;
    const bool vec = job.vec != 0;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
    float g = 0.0f, inv = 0.0f;
    constexpr int kSize = Raw<TYPE>::kSize;
    const uint32_t blocks = (rows + 15) / 16, chunks = (blocks + 3) / 4;
    const uint32_t tiles_r = (rows + kTile - 1) / kTile, tiles_c = (cols + kTile - 1) / kTile;
    for (uint64_t tile = blockIdx.x; tile < (uint64_t)tiles_r * tiles_c; tile += gridDim.x) {
        const uint32_t tr = (uint32_t)(tile / tiles_c), tc = (uint32_t)(tile % tiles_c);
        const uint32_t r0 = tr * kTile + warp * 16, c0 = tc * kTile + lane * 4;
        const uint8_t *src = job.x + (uint64_t)r0 * ld_bytes + (uint64_t)c0 * kSize;
        // word [i][k]: two values (16-bit) or one (FP32) of row r0 + i
        uint32_t w[16][kSize];
        if (vec && c0 + 4 <= cols) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if (r0 + i >= rows) {
#pragma unroll
                    for (int k = 0; k < kSize; ++k) w[i][k] = 0u;
                } else if (kSize == 4) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(src + (uint64_t)i * ld_bytes);
                    w[i][0] = v.x; w[i][1] = v.y; w[i][2 % kSize] = v.z; w[i][3 % kSize] = v.w;
                } else {
                    const uint2 v = *reinterpret_cast<const uint2 *>(src + (uint64_t)i * ld_bytes);
                    w[i][0] = v.x; w[i][1] = v.y;
                }
            }
        } else {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const bool in = r0 + i < rows;
                const uint8_t *p = src + (uint64_t)i * ld_bytes;
#pragma unroll
                for (int k = 0; k < kSize; ++k) {
                    if (kSize == 4) {
                        w[i][k] = in && c0 + k < cols ? reinterpret_cast<const uint32_t *>(p)[k] : 0u;
                    } else {
                        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
                        w[i][k] = (in && c0 + 2 * k < cols ? (uint32_t)h[2 * k] : 0u) |
                                  (in && c0 + 2 * k + 1 < cols ? (uint32_t)h[2 * k + 1] << 16 : 0u);
                    }
                }
            }
        }
        if (tile == blockIdx.x) {   // the scale on top, while the first tile is on its way
            uint32_t m = 0;
            for (uint32_t i = threadIdx.x; i < job.count; i += 256) m = max_bits(m, __float_as_uint(job.maxima[i]));
            m = warp_max_bits(m);
            if (lane == 0) part[warp] = m;
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 8; ++i) m = max_bits(m, part[i]);
            g = __uint_as_float(m);
            inv = top_inverse(g);
            if (blockIdx.x == 0 && threadIdx.x == 0) job.scale[0] = g;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            Raw<TYPE> r;   // column c0 + j
#pragma unroll
            for (int i = 0; i < Raw<TYPE>::kWords; ++i) {
                if (kSize == 4) r.w[i] = w[i][j % kSize];
                else r.w[i] = __byte_perm(w[(2 * i) % 16][j >> 1], w[(2 * i + 1) % 16][j >> 1], j & 1 ? 0x7632 : 0x5410);
            }
            uint2 codes;
            const uint32_t s = encode_block(r, r.amax_bits(), g, inv, codes);
            const uint32_t c = lane * 4 + j;
            codes_tile[c * 8 + (warp ^ (lane & 7u))] = codes;
            scales_tile[(warp >> 2) * 512 + (c & 31u) * 16 + (c >> 5) * 4 + (warp & 3u)] = (uint8_t)s;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const uint32_t c = threadIdx.x / 8 + 32 * k, blk = threadIdx.x & 7u;
            if (tc * kTile + c < cols && tr * 8 + blk < blocks)
                *reinterpret_cast<uint2 *>(job.bytes + (uint64_t)(tc * kTile + c) * job.row_bytes + (uint64_t)(tr * 8 + blk) * 8) =
                    codes_tile[c * 8 + (blk ^ (c >> 2 & 7u))];
        }
        // four scales a thread, of row (t / 4) % 32 + 32 (t % 4) of the band; those behind the last row are not this tensor's
        if (tr * 2 + threadIdx.x / 128 < chunks && tc * kTile + (threadIdx.x / 4 & 31u) + 32 * (threadIdx.x & 3u) < cols)
            reinterpret_cast<uint32_t *>(job.scales + ((uint64_t)tc * chunks + tr * 2) * 512)[threadIdx.x] =
                reinterpret_cast<const uint32_t *>(scales_tile)[threadIdx.x];
        __syncthreads();
    }
}

// ---- reading back -----------------------------------------------------------------------------------------------------------
// A thread a block, as many threads a row as it has blocks (up to a CTA): values leave in 32-byte pieces, side by side.
struct DecodeJob {
    const uint8_t *bytes;
    uint64_t row_bytes;
    const uint8_t *scales;
    uint32_t layout;
    const float *scale;
    uint32_t per_row, rows, blocks, threads_per_row;
    uint8_t *out;
    uint64_t ld_bytes;
    uint32_t cols, access;
};
// Whether the header of CSF storage describes at least `groups` scales, and its records are of a size that there is (csf_load_scale goes
// where it says).
__device__ __forceinline__ bool csf_holds(const uint8_t *s, uint64_t groups) {
    const uint32_t k = reinterpret_cast<const uint32_t *>(s)[0], rows = reinterpret_cast<const uint32_t *>(s)[1];
    if (k == 0 || k % 128 != 0 || groups > (uint64_t)rows * (k / 16)) return false;
    return rows == 1 ? s[8] == 255 : s[8] != 255 && (s[9] == 7 || s[9] == 8);
}
template <int TYPE>
__device__ __forceinline__ void decode_rows(const DecodeJob &j) {
    const uint32_t row = blockIdx.x * (256u / j.threads_per_row) + threadIdx.x / j.threads_per_row;
    if (row >= j.rows) return;
    const uint32_t tiles = (j.blocks + 3) / 4;
    const float g = j.scale[j.per_row ? row : 0];
    auto codes_of = [&](uint32_t blk) { return *reinterpret_cast<const uint2 *>(j.bytes + (uint64_t)row * j.row_bytes + (uint64_t)blk * 8); };
    auto scale_of = [&](uint32_t blk) -> uint32_t {
        const uint64_t flat = (uint64_t)row * j.blocks + blk;
        return j.layout == B2_SCALES_SM100 ? j.scales[sm100_scale_offset(row, blk, tiles)]
               : j.layout == B2_SCALES_RAW ? j.scales[flat] : csf_holds(j.scales, (uint64_t)j.rows * j.blocks) ? csf_load_scale(j.scales, (uint32_t)flat) : 0x7fu;
    };
    for (uint32_t blk = threadIdx.x % j.threads_per_row; blk < j.blocks; blk += j.threads_per_row) {
        const uint2 codes = codes_of(blk);
        const uint32_t s = scale_of(blk);
        float v[16];
        decode_block<TYPE == B2_TYPE_F32 ? kNearest : kTruncate>(codes, s, g, v);
        store_block<TYPE>(j.out + (uint64_t)row * j.ld_bytes + (uint64_t)blk * 16 * Raw<TYPE>::kSize, v, (int)min(j.cols - blk * 16u, 16u), j.access);
    }
    if (TYPE == B2_TYPE_BF16 && fabsf(g) < 0x1p-126f) {   // (FP16 has 0 for all of these)
        uint16_t *line = reinterpret_cast<uint16_t *>(j.out + (uint64_t)row * j.ld_bytes);
#pragma unroll 1
        for (uint32_t i = threadIdx.x % j.threads_per_row * 16; i < j.cols; i = (i + 1) % 16 != 0 ? i + 1 : i + 1 + (j.threads_per_row - 1) * 16) {
            const uint2 codes = codes_of(i / 16);
            const float a = e2m1_value((i & 8u ? codes.y : codes.x) >> 4 * (i & 7u)) * e4m3_value((uint16_t)scale_of(i / 16));
            line[i] = (uint16_t)f32_to_bf16_bits(product_to_odd(a, g));
        }
    }
}
__global__ void __launch_bounds__(256)
k_fp4_decode(const __grid_constant__ DecodeJob job) {
    stream_enter();
    decode_rows<B2_TYPE_F32>(job);
}
// (eight CTAs an SM: left alone, the compiler takes registers for six or seven, 50304 x 768 24.4 us instead of 21.9 in F16)
template <int TYPE>
__global__ void __launch_bounds__(256, 8)
k_fp4_decode_16(const __grid_constant__ DecodeJob job) {
    stream_enter();
    decode_rows<TYPE>(job);
}

// ---- the paged cache --------------------------------------------------------------------------------------------------------
// Quotients by a divisor of the launch, for dividends below 2^31: with 2^(l-1) < d <= 2^l and m = floor(2^(31+l) / d) + 1 the
// product n m exceeds n 2^(31+l) / d by n at most, less than what is missing to the next multiple of 2^(31+l).
struct Divisor {
    uint32_t d, m, shift;
    __device__ __forceinline__ uint32_t of(uint32_t n) const { return d == 1u ? n : __umulhi(n, m) >> shift; }
};
Divisor divisor(uint32_t d) {
    uint32_t l = 0;
    while ((1ull << l) < d) ++l;
    return {d, d == 1 ? 0u : (uint32_t)((1ull << (31 + l)) / d + 1), d == 1 ? 0u : l - 1};
}
// blockIdx.y is the tensor: keys, values.
struct CacheSide {
    b2_nvfp4_cache cache;
    b2_vectors vectors;
    Divisor heads, blocks;
    uint32_t group;   // lanes of a vector when it is written
    uint32_t access;
};
struct CachePair {
    CacheSide side[2];
    Divisor page_size[2];
};
// A vector's blocks lie in `group` neighbouring lanes (a power of two, at least dim / 16 of them up to a warp; TWO: vectors of more
// than 512 values take two blocks a lane), which share its maximum.
template <int TYPE, bool TWO>
__global__ void __launch_bounds__(256)
k_fp4_cache_write(const __grid_constant__ CachePair p, const int64_t *slots, uint32_t token_count) {
    stream_enter();
    const CacheSide &side = p.side[blockIdx.y];
    const b2_nvfp4_cache &c = side.cache;
    const uint32_t group = side.group, vector = (blockIdx.x * 256u + threadIdx.x) / group, lane = threadIdx.x & (group - 1);
    const uint32_t blocks = side.blocks.d, token = side.heads.of(vector), head = vector - token * c.heads;
    int64_t slot = -1;
    if (token < token_count) slot = slots[token];
    const bool there = slot >= 0 && slot < (int64_t)c.pages * c.page_size;
    const uint8_t *src = static_cast<const uint8_t *>(side.vectors.data) + (token * side.vectors.token_stride + head * side.vectors.head_stride) * Raw<TYPE>::kSize;
    Raw<TYPE> r[TWO ? 2 : 1];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < (TWO ? 2 : 1); ++i) {
        const uint32_t blk = lane + i * group;
        if (there && blk < blocks) r[i].load(src + blk * 16 * Raw<TYPE>::kSize, 16, side.access);
        else r[i].clear();
        m = max_bits(m, r[i].amax_bits());
    }
    for (uint32_t o = group / 2; o > 0; o >>= 1) m = max_bits(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (!there) return;
    const float g = top_scale(m), inv = top_inverse(g);
    const uint64_t at = (uint64_t)slot * c.heads + head;
    if (lane == 0) c.exponents[at] = (uint8_t)(__float_as_uint(g) >> 23);
#pragma unroll
    for (int i = 0; i < (TWO ? 2 : 1); ++i) {
        const uint32_t blk = lane + i * group;
        if (blk >= blocks) break;
        uint2 codes;
        const uint32_t s = encode_block(r[i], r[i].amax_bits(), g, inv, codes);
        *reinterpret_cast<uint2 *>(c.bytes + (at * blocks + blk) * 8) = codes;
        c.scales[at * blocks + blk] = (uint8_t)s;
    }
}

// One CTA takes some tokens of a sequence; a thread reads a block at a time.
template <int TYPE>
__global__ void __launch_bounds__(256)
k_fp4_cache_read(const __grid_constant__ CachePair p, const int32_t *table, uint32_t table_width, const int32_t *lengths,
                 uint32_t max_tokens, uint32_t tokens_per_cta) {
    stream_enter();
    const CacheSide &side = p.side[blockIdx.y];
    const b2_nvfp4_cache &c = side.cache;
    const uint32_t sequence = blockIdx.z, blocks = side.blocks.d, per_token = c.heads * blocks;
    const uint64_t most = min((uint64_t)max_tokens, (uint64_t)table_width * c.page_size);
    const int32_t length = lengths[sequence];
    const uint32_t tokens = length <= 0 ? 0u : (uint32_t)min((uint64_t)length, most);
    const uint32_t t0 = blockIdx.x * tokens_per_cta;
    if (t0 >= tokens) return;
    const uint32_t work = min(tokens_per_cta, tokens - t0) * per_token;
    const int32_t *pages = table + (uint64_t)sequence * table_width;
    uint8_t *out = static_cast<uint8_t *>(side.vectors.data) + sequence * side.vectors.sequence_stride * Raw<TYPE>::kSize;
#pragma unroll 2
    for (uint32_t i = threadIdx.x; i < work; i += 256) {
        const uint32_t vector = side.blocks.of(i), blk = i - vector * blocks, token = side.heads.of(vector), head = vector - token * c.heads;
        const uint32_t t = t0 + token, in = p.page_size[blockIdx.y].of(t);
        const int32_t page = pages[in];
        uint2 codes = make_uint2(0u, 0u);
        uint32_t s = 0, e = 255;
        if (page >= 0 && (uint32_t)page < c.pages) {
            const uint64_t at = ((uint64_t)page * c.page_size + (t - in * c.page_size)) * c.heads + head;
            codes = *reinterpret_cast<const uint2 *>(c.bytes + (at * blocks + blk) * 8);
            s = c.scales[at * blocks + blk];
            e = c.exponents[at];
        }
        float v[16];
        decode_block<kNearest>(codes, s, e == 255u ? __uint_as_float(0x7fffffffu) : e == 0u ? 0x1p-127f : __uint_as_float(e << 23), v);
        store_block<TYPE>(out + (t * side.vectors.token_stride + head * side.vectors.head_stride + blk * 16) * Raw<TYPE>::kSize, v, 16, side.access);
    }
}

uint64_t type_size(uint32_t type) { return type == B2_TYPE_F32 ? 4 : 2; }
bool aligned(const void *p, uint64_t step_bytes, uint64_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0 && step_bytes % to == 0; }

#define B2_FOR_TYPE(type, F, ...)                                      \
    if ((type) == B2_TYPE_F32) return F<B2_TYPE_F32>(__VA_ARGS__);     \
    if ((type) == B2_TYPE_BF16) return F<B2_TYPE_BF16>(__VA_ARGS__);   \
    return F<B2_TYPE_F16>(__VA_ARGS__);

// The maximum of x, in as many CTAs as there is work for, up to six an SM; `maxima`: a scale of each.
MaximaJob maximum_of(const b2_matrix &x, float *maxima, int sm_count) {
    const uint64_t ld = x.ld * type_size(x.type);
    const bool flat = x.ld == x.cols || x.rows == 1;
    MaximaJob j = {};
    j.x = static_cast<const uint8_t *>(x.data);
    j.ld_bytes = ld;
    j.rows = flat ? 1u : x.rows;
    j.cols = flat ? (uint64_t)x.rows * x.cols : x.cols;
    j.access = access_of(x.data, flat ? 0 : ld);
    const uint64_t warps = flat ? (j.cols + 511) / 512 : j.rows, most = std::min(B2_NVFP4_MAXIMA, sm_count * 6);
    j.ctas = (uint32_t)std::min((warps + 7) / 8, most);
    j.maxima = maxima;
    return j;
}
template <int TYPE>
cudaError_t rows_impl(const b2_matrix &x, const b2_nvfp4_operand &out, const MaximaJob &other, cudaStream_t s) {
    const uint64_t ld = x.ld * Raw<TYPE>::kSize;
    const uint32_t access = access_of(x.data, ld);
    const uint32_t blocks = out.cols / 16;
    auto go = [&](auto kernel, uint32_t rows_per_cta, int threads) {
        const uint32_t ctas = (x.rows + rows_per_cta - 1) / rows_per_cta;
        return overlapped_launch(kernel, dim3(ctas + other.ctas), threads, 0, s, static_cast<const uint8_t *>(x.data), ld, x.rows, x.cols, access,
                                 out.bytes, out.row_bytes, out.scales, out.scale, ctas, other);
    };
    if (blocks <= 32 * kHeld) return go(k_fp4_quantize_rows<TYPE, 1, true>, 8, 256);
    if (blocks <= 4 * 32 * kHeld) return go(k_fp4_quantize_rows<TYPE, 4, true>, 2, 256);
    if (blocks <= 16 * 32 * kHeld) return go(k_fp4_quantize_rows<TYPE, 16, true>, 1, 512);
    return go(k_fp4_quantize_rows<TYPE, 16, false>, 1, 512);
}
template <int TYPE>
cudaError_t columns_impl(const ColumnsTask *tasks, uint32_t count, float *maxima, int sm_count, cudaStream_t s) {
    MaximaJobs m = {};
    ColumnsJobs c = {};
    uint32_t parts = 0, tiles = 0;
    for (uint32_t i = 0; i < count; ++i) {
        const b2_matrix &x = *tasks[i].x;
        const b2_nvfp4_operand &out = *tasks[i].out;
        const uint64_t ld = x.ld * Raw<TYPE>::kSize;
        MaximaJob &j = m.job[i];
        j = maximum_of(x, maxima + i * B2_NVFP4_MAXIMA, sm_count);
        const bool few = tasks[i].tops && tasks[i].top_count <= kFewTops;
        if (tasks[i].tops) {
            j.tops = tasks[i].tops;
            j.top_count = tasks[i].top_count;
            j.ctas = few ? 0 : 8;
        }
        parts = std::max(parts, j.ctas);
        ColumnsJob &q = c.job[i];
        q.x = static_cast<const uint8_t *>(x.data);
        q.ld_bytes = ld;
        q.rows = x.rows;
        q.cols = x.cols;
        q.bytes = out.bytes;
        q.row_bytes = out.row_bytes;
        q.scales = out.scales;
        q.scale = out.scale;
        q.maxima = few ? tasks[i].tops : j.maxima;
        q.count = few ? tasks[i].top_count : j.ctas;
        q.vec = aligned(x.data, ld, 4 * Raw<TYPE>::kSize);
        const uint64_t t = (uint64_t)((x.rows + kTile - 1) / kTile) * ((x.cols + kTile - 1) / kTile);
        tiles = std::max(tiles, (uint32_t)std::min<uint64_t>(t, 1u << 20));
    }
    if (parts != 0) {
        const cudaError_t e = overlapped_launch(k_fp4_maxima<TYPE>, dim3(parts, count), 256, 0, s, m);
        if (e != cudaSuccess) return e;
    }
    return overlapped_launch(k_fp4_quantize_columns<TYPE>, dim3(tiles, count), 256, 0, s, c);
}
template <int TYPE>
cudaError_t decode_impl(const b2_nvfp4_operand &in, uint32_t layout, const b2_matrix &out, cudaStream_t s) {
    const uint64_t ld = out.ld * Raw<TYPE>::kSize;
    const uint32_t blocks = in.cols / 16;
    uint32_t tpr = 1;
    while (tpr < blocks && tpr < 256) tpr *= 2;
    const uint32_t per_cta = 256 / tpr;
    const DecodeJob j = {in.bytes, in.row_bytes, in.scales, layout, in.scale, in.scale_count != 1, in.rows, blocks, tpr,
                         static_cast<uint8_t *>(out.data), ld, out.cols, access_of(out.data, ld)};
    const dim3 grid((in.rows + per_cta - 1) / per_cta);
    if constexpr (TYPE == B2_TYPE_F32) return overlapped_launch(k_fp4_decode, grid, 256, 0, s, j);
    else return overlapped_launch(k_fp4_decode_16<TYPE>, grid, 256, 0, s, j);
}
CachePair cache_pair(const b2_nvfp4_cache *caches, const b2_vectors *vectors, uint32_t count) {
    CachePair p = {};
    for (uint32_t i = 0; i < count; ++i) {
        CacheSide &side = p.side[i];
        side.cache = caches[i];
        side.vectors = vectors[i];
        side.heads = divisor(caches[i].heads);
        side.blocks = divisor(caches[i].dim / 16);
        p.page_size[i] = divisor(caches[i].page_size);
        for (side.group = 1; side.group < side.blocks.d && side.group < 32;) side.group *= 2;
        const uint64_t size = type_size(vectors[i].type);
        const uint64_t strides = (vectors[i].sequence_stride | vectors[i].token_stride | vectors[i].head_stride) * size;
        side.access = access_of(vectors[i].data, strides);
    }
    return p;
}
template <int TYPE>
cudaError_t write_impl(const CachePair &p, uint32_t count, const int64_t *slots, uint32_t token_count, cudaStream_t s) {
    uint64_t threads = 0;
    bool two = false;
    for (uint32_t i = 0; i < count; ++i) {
        threads = std::max(threads, (uint64_t)token_count * p.side[i].cache.heads * p.side[i].group);
        two = two || p.side[i].blocks.d > 32;
    }
    if (threads > 0x7fffff00u) return cudaErrorInvalidValue;   // threads and vectors are counted in 31 bits
    const dim3 grid((unsigned)((threads + 255) / 256), count);
    if (two) return overlapped_launch(k_fp4_cache_write<TYPE, true>, grid, 256, 0, s, p, slots, token_count);
    return overlapped_launch(k_fp4_cache_write<TYPE, false>, grid, 256, 0, s, p, slots, token_count);
}
template <int TYPE>
cudaError_t read_impl(const CachePair &p, uint32_t count, const int32_t *table, uint32_t table_width, const int32_t *lengths,
                      uint32_t sequences, uint32_t max_tokens, cudaStream_t s) {
    uint32_t per_token = 0;
    for (uint32_t i = 0; i < count; ++i) per_token = std::max(per_token, p.side[i].cache.heads * p.side[i].blocks.d);
    const uint32_t tokens = std::max(1u, 1024u / per_token);   // about four blocks a thread
    return overlapped_launch(k_fp4_cache_read<TYPE>, dim3((max_tokens + tokens - 1) / tokens, count, sequences), 256, 0, s, p, table,
                             table_width, lengths, max_tokens, tokens);
}

}  // namespace

cudaError_t launch_fp4_quantize_rows(const b2_matrix &x, const b2_nvfp4_operand &out, cudaStream_t s) {
    const MaximaJob none = {};
    B2_FOR_TYPE(x.type, rows_impl, x, out, none, s)
}
uint32_t fp4_maximum_parts(const b2_matrix &x, int sm_count) { return maximum_of(x, nullptr, sm_count).ctas; }
cudaError_t launch_fp4_quantize_rows_and_maximum(const b2_matrix &x, const b2_nvfp4_operand &out, const b2_matrix &other, float *maxima,
                                                 int sm_count, cudaStream_t s) {
    const MaximaJob job = maximum_of(other, maxima, sm_count);
    B2_FOR_TYPE(x.type, rows_impl, x, out, job, s)
}
cudaError_t launch_fp4_quantize_columns(const ColumnsTask *tasks, uint32_t count, float *maxima, int sm_count, cudaStream_t s) {
    if (count == 2 && tasks[0].x->type != tasks[1].x->type) {
        const cudaError_t e = launch_fp4_quantize_columns(tasks, 1, maxima, sm_count, s);
        return e != cudaSuccess ? e : launch_fp4_quantize_columns(tasks + 1, 1, maxima + B2_NVFP4_MAXIMA, sm_count, s);
    }
    B2_FOR_TYPE(tasks[0].x->type, columns_impl, tasks, count, maxima, sm_count, s)
}
cudaError_t launch_fp4_decode(const b2_nvfp4_operand &in, uint32_t layout, const b2_matrix &out, cudaStream_t s) {
    B2_FOR_TYPE(out.type, decode_impl, in, layout, out, s)
}
cudaError_t launch_fp4_cache_write(const b2_nvfp4_cache *caches, const b2_vectors *tokens, uint32_t count, const int64_t *slots,
                                   uint32_t token_count, cudaStream_t s) {
    const CachePair p = cache_pair(caches, tokens, count);
    B2_FOR_TYPE(tokens[0].type, write_impl, p, count, slots, token_count, s)
}
cudaError_t launch_fp4_cache_read(const b2_nvfp4_cache *caches, const b2_vectors *out, uint32_t count, const int32_t *table,
                                  uint32_t table_width, const int32_t *lengths, uint32_t sequences, uint32_t max_tokens, cudaStream_t s) {
    const CachePair p = cache_pair(caches, out, count);
    B2_FOR_TYPE(out[0].type, read_impl, p, count, table, table_width, lengths, sequences, max_tokens, s)
}

}  // namespace b2

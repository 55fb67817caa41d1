// cm_fp8.cu -- quantisation to block-scaled 8-bit floating point, alone (cm_quant_fp8) and as the
// output of an RMS norm with the residual's addition (cm_rmsnorm_fp8).
//
// Both are HBM-bound: every input is read once and every output written once, all arithmetic in
// fp32 registers.  What stands in the way of the bandwidth is the issue rate, so the work that a
// block needs once (the reduction of its maximum, the divisions) is spread over as few lanes as
// the loads allow: a row's 128-column block belongs to 4 neighbouring lanes of 32 values each.
// Chunk i of lane l is the 8 columns from 8 * (4 * i + l): the 4 lanes of a block read 64
// neighbouring bytes of a 2-byte type with one load and write one 32-byte sector with one store;
// the maximum is two shuffles, and of the two quotients lane 0 takes A / F and the others F / A.
// (With 16 lanes a block and 8 values each, 8192 x 4096 bf16 took 30.9 us instead of 20.3; 17.7 us,
// 5.7 TB/s, by now, and 39 us, 6.0 TB/s, normed with the residual's addition.)
// Values stay in their own type until they are needed, fp32 works on pairs, and the next rows'
// loads are issued before the current rows are worked on.
// Rows whose base or pitch is not a multiple of the vector sizes keep this layout: a chunk is cut out
// of the two (fp32: three) aligned 16-byte words that hold it, and 8-bit and 16-bit results leave as
// aligned 32-bit words put together from neighbouring lanes' (8192 x 1001 bf16, one element an access:
// 26.9 us quantised and 55.7 us normed; this way 9.7 and 24).  What lies behind a row's end in its
// last words is cleared where the values are used: done at the load, or by blocks that take another
// path than whole ones, it cost 8192 x 2000 bf16 normed 31 us instead of 22.
#include <algorithm>
#include <cmath>

#include "cm_fp8.cuh"

namespace cm {
namespace {

constexpr uint32_t kLanes = 4;                       // lanes of a block
constexpr uint32_t kVals = kFp8Block / kLanes;       // values of a lane
constexpr uint32_t kChunks = kVals / 8;

// column of a lane's value j
__device__ __forceinline__ uint32_t column(uint32_t col0, uint32_t l, uint32_t j) { return col0 + 8 * (kLanes * (j / 8) + l) + j % 8; }

// A lane's 32 values as they lie in memory; 0 past the row's end, once trimmed.
template <typename T>
struct Raw {
    static constexpr uint32_t W = sizeof(T) / 2;     // 16-byte words of a chunk
    uint4 w[kChunks * W];

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (uint32_t i = 0; i < kChunks * W; ++i) w[i] = make_uint4(0, 0, 0, 0);
    }
    // VEC: rows start on 16-byte boundaries
    template <bool VEC>
    __device__ __forceinline__ void load(const T* row, uint32_t col0, uint32_t l, uint32_t cols) {
        // Aligned words around each chunk; one that holds none of its values is not read, and one that
        // holds any lies in the row's own memory page.
        constexpr uint32_t N = VEC ? W : W + 1;
        const uint32_t skip = VEC ? 0u : (uint32_t)((uintptr_t)(row + col0 + 8 * l) & 15u);    // the same for all chunks of a row
        uint4 v[kChunks][N];
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i) {
            const uint32_t c = column(col0, l, 8 * i);
            const uint32_t bytes = c < cols ? min(8u, cols - c) * (uint32_t)sizeof(T) : 0u;
            const uint4* p = reinterpret_cast<const uint4*>(reinterpret_cast<const uint8_t*>(row + c) - skip);
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) v[i][k] = bytes && 16 * k < skip + bytes ? p[k] : make_uint4(0, 0, 0, 0);
        }
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i) {
            uint32_t x[4 * N];
#pragma unroll
            for (uint32_t k = 0; k < N; ++k) { x[4 * k] = v[i][k].x; x[4 * k + 1] = v[i][k].y; x[4 * k + 2] = v[i][k].z; x[4 * k + 3] = v[i][k].w; }
            if (!VEC) {
#pragma unroll
                for (uint32_t j = 0; j + 2 < 4 * N; ++j) x[j] = skip & 8u ? x[j + 2] : x[j];
#pragma unroll
                for (uint32_t j = 0; j + 3 < 4 * N; ++j) x[j] = skip & 4u ? x[j + 1] : x[j];
                if (sizeof(T) == 2) {
#pragma unroll
                    for (uint32_t j = 0; j < 4 * W; ++j) x[j] = __funnelshift_r(x[j], x[j + 1], skip & 2u ? 16u : 0u);
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < W; ++k) w[i * W + k] = make_uint4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
        }
    }
    // Clears what `load` took from behind the row's end in the last words.  Apart from it, so that
    // nothing waits for the values between their load and their use.
    __device__ __forceinline__ void trim(uint32_t col0, uint32_t l, uint32_t cols) {
        // no sum that wraps: rows end within 128 columns of 2^32 too (a lane behind the row holds zeros already)
        if (cols - col0 >= kFp8Block || cols % 8 == 0) return;
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i) {
            const uint32_t c = column(col0, l, 8 * i), n = c < cols ? min(8u, cols - c) : 0u;
#pragma unroll
            for (uint32_t j = 0; j < 4 * W; ++j) {
                uint32_t& x = reinterpret_cast<uint32_t*>(w)[4 * W * i + j];
                if (sizeof(T) == 4) x = j < n ? x : 0u;
                else x = 2 * j + 1 < n ? x : 2 * j < n ? x & 0xffffu : 0u;
            }
        }
    }
    __device__ __forceinline__ uint32_t word(uint32_t i) const {
        const uint4& v = w[i / 4];
        return i % 4 == 0 ? v.x : i % 4 == 1 ? v.y : i % 4 == 2 ? v.z : v.w;
    }
    // values 2 p and 2 p + 1 in fp32 (p a constant)
    __device__ __forceinline__ uint64_t pair(uint32_t p) const;
    // max(|v|) of the lane; a NaN among them is the result, so that it reaches the block's scale
    __device__ __forceinline__ float max_abs() const;
};

__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}
__device__ __forceinline__ float max_abs3(float m, float a, float b) {
    asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(a), "f"(b));
    return m;
}

template <> __device__ __forceinline__ uint64_t Raw<float>::pair(uint32_t p) const { return pack2(word(2 * p), word(2 * p + 1)); }
template <> __device__ __forceinline__ uint64_t Raw<__nv_bfloat16>::pair(uint32_t p) const {
    return pack2(word(p) << 16, word(p) & 0xffff0000u);        // bf16 is the upper half of fp32
}
template <> __device__ __forceinline__ uint64_t Raw<__half>::pair(uint32_t p) const {
    const uint32_t u = word(p);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u));
    return pack2(f.x, f.y);
}
template <> __device__ __forceinline__ uint64_t Raw<int16_t>::pair(uint32_t p) const {
    const uint32_t u = word(p);
    return pack2(to_f32((int16_t)(u & 0xffffu)), to_f32((int16_t)(u >> 16)));
}

template <> __device__ __forceinline__ float Raw<float>::max_abs() const {
    float m = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kVals; i += 2) m = max_abs3(m, __uint_as_float(word(i)), __uint_as_float(word(i + 1)));
    return m;
}
// magnitudes of 16-bit IEEE types order as integers, infinities above every finite value and NaN
// above infinity, so two of them compare in one instruction
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
    uint32_t m;
    asm("max.u16x2 %0, %1, %2;" : "=r"(m) : "r"(a), "r"(b));
    return m;
}
template <> __device__ __forceinline__ float Raw<__nv_bfloat16>::max_abs() const {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < kVals / 2; ++i) m = max_u16x2(m, word(i) & 0x7fff7fffu);
    return __uint_as_float(max(m & 0xffffu, m >> 16) << 16);
}
template <> __device__ __forceinline__ float Raw<__half>::max_abs() const {
    uint32_t m = 0;
#pragma unroll
    for (uint32_t i = 0; i < kVals / 2; ++i) m = max_u16x2(m, word(i) & 0x7fff7fffu);
    return __half2float(__ushort_as_half((unsigned short)max(m & 0xffffu, m >> 16)));
}
template <> __device__ __forceinline__ float Raw<int16_t>::max_abs() const {
    float m = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < kVals / 2; ++i) {
        float a, b;
        unpack2(pair(i), a, b);
        m = max_abs3(m, a, b);
    }
    return m;
}

// fp32 pairs -> 32-bit words of T
template <typename T>
__device__ __forceinline__ uint32_t to_word(uint64_t v);
template <> __device__ __forceinline__ uint32_t to_word<__nv_bfloat16>(uint64_t v) {
    float lo, hi;
    unpack2(v, lo, hi);
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}
template <> __device__ __forceinline__ uint32_t to_word<__half>(uint64_t v) {
    float lo, hi;
    unpack2(v, lo, hi);
    const __half2 b = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
}

// Stores the words of a lane's chunks (N of 32 bits each, from `chunk(i, x)`) to elements of S bytes at
// any alignment.  VEC: as one access a chunk.  Else a chunk starts `odd` bytes (0 to 3, the same for a whole row) behind a 32-bit
// boundary; its words are shifted up by them, and the chunk before it -- the lane before, or lane 3's
// last one -- gives the bytes that the first word lacks.  What has no neighbour in the block (its
// first bytes, its last, and the last ones of a row) is stored by elements.  The four lanes of a block
// arrive together.
template <uint32_t S, uint32_t N, bool VEC, typename F>
__device__ __forceinline__ void store_words(uint8_t* row, uint32_t col0, uint32_t l, uint32_t cols, F chunk) {
    const uint32_t odd = (uint32_t)((uintptr_t)row + (uintptr_t)col0 * S) & 3u;      // 8 elements are a multiple of 4 bytes
    const uint32_t lanes = 0xfu << (threadIdx.x & 28u);
    auto bytes = [&](uint8_t* p, uint32_t word, uint32_t from, uint32_t to) {           // bytes from .. to - 1 of a word, at p + from
        for (uint32_t k = from; k < to; k += S) {
            if (S == 1) p[k] = (uint8_t)(word >> (8 * k));
            else *reinterpret_cast<uint16_t*>(p + k) = (uint16_t)(word >> (8 * k));
        }
    };
    uint32_t x[N], before = 0;                 // before: the last word of this lane's chunk before
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
        chunk(i, x);
        const uint32_t c = column(col0, l, 8 * i), n = c < cols ? min(8u, cols - c) : 0u, at = kLanes * i + l;
        uint8_t* p = row + (uint64_t)c * S;
        uint32_t last = 0;
        if (!VEC) {
            last = __shfl_sync(lanes, l == kLanes - 1 ? before : x[N - 1], (l + kLanes - 1) % kLanes, kLanes);
            before = x[N - 1];
        }
        if (VEC && n == 8) {
            if constexpr (N == 4) *reinterpret_cast<uint4*>(p) = make_uint4(x[0], x[1], x[2], x[3]);
            else *reinterpret_cast<uint2*>(p) = make_uint2(x[0], x[1]);
        } else if (n == 8) {
            uint32_t* a = reinterpret_cast<uint32_t*>(p - odd);
            if (odd == 0 || at > 0) a[0] = __funnelshift_l(last, x[0], 8 * odd);
            else bytes(p, x[0], 0, 4 - odd);
#pragma unroll
            for (uint32_t j = 1; j < N; ++j) a[j] = __funnelshift_l(x[j - 1], x[j], 8 * odd);
            if (odd && (at == kLanes * kChunks - 1 || cols - c < 16)) bytes(p + 4 * (N - 1), x[N - 1], 4 - odd, 4);
        } else if (n) {
#pragma unroll
            for (uint32_t j = 0; j < N; ++j)
                if (4 * j < n * S) bytes(p + 4 * j, x[j], 0, min(4u, n * S - 4 * j));
        }
    }
}

// a lane's 32 values in fp32 pairs -> row of T
template <typename T, bool VEC>
__device__ __forceinline__ void store32(T* row, uint32_t col0, uint32_t l, uint32_t cols, const uint64_t (&v)[kVals / 2]) {
    if constexpr (sizeof(T) == 2) {
        store_words<2, 4, VEC>(reinterpret_cast<uint8_t*>(row), col0, l, cols, [&](uint32_t i, uint32_t (&x)[4]) {
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) x[j] = to_word<T>(v[4 * i + j]);
        });
    } else {
        // As store_words does it, in 16-byte words: a chunk starts `odd` values behind a boundary.
        const uint32_t odd = VEC ? 0u : (uint32_t)((uintptr_t)(row + col0) / 4) & 3u, lanes = 0xfu << (threadIdx.x & 28u);
        float before[3] = {};
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i) {
            const uint32_t c = column(col0, l, 8 * i), n = c < cols ? min(8u, cols - c) : 0u, at = kLanes * i + l;
            float x[11];                 // the chunk, behind the last three values of the one before it
#pragma unroll
            for (uint32_t j = 0; j < 4; ++j) unpack2(v[4 * i + j], x[3 + 2 * j], x[4 + 2 * j]);
            T* p = row + c;
            if (!VEC) {
#pragma unroll
                for (uint32_t j = 0; j < 3; ++j) {
                    x[j] = __shfl_sync(lanes, l == kLanes - 1 ? before[j] : x[8 + j], (l + kLanes - 1) % kLanes, kLanes);
                    before[j] = x[8 + j];
                }
            }
            if (n < 8 || (!VEC && at == 0)) {
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                    if (j < n) p[j] = x[3 + j];
                continue;
            }
            const bool end = !VEC && (at == kLanes * kChunks - 1 || cols - c < 16);
#pragma unroll
            for (uint32_t j = 0; j < 3; ++j)
                if (end && 3 - j <= odd) p[5 + j] = x[8 + j];
            if (!VEC) {
#pragma unroll
                for (uint32_t j = 0; j + 2 < 11; ++j) x[j] = odd & 2u ? x[j] : x[j + 2];
#pragma unroll
                for (uint32_t j = 0; j + 3 < 11; ++j) x[j] = odd & 1u ? x[j] : x[j + 1];
            }
            constexpr uint32_t f = VEC ? 3 : 0;
            float4* a = reinterpret_cast<float4*>(p - odd);
            a[0] = make_float4(x[f], x[f + 1], x[f + 2], x[f + 3]);
            a[1] = make_float4(x[f + 4], x[f + 5], x[f + 6], x[f + 7]);
        }
    }
}

// the 8-bit values of a lane's 32 (`value(p)`: pair p), times inv
template <bool VEC, typename V>
__device__ __forceinline__ void store_q32(uint8_t* row, uint32_t col0, uint32_t l, uint32_t cols, uint32_t format, float inv, V value) {
    const uint64_t inv2 = pack2(inv, inv);
    auto chunk = [&](uint32_t i, uint32_t (&x)[2]) {
        uint32_t p[4];
#pragma unroll
        for (uint32_t j = 0; j < 4; ++j) {
            float lo, hi;
            unpack2(mul2(value(4 * i + j), inv2), lo, hi);
            p[j] = cvt_fp8x2(format, lo, hi);
        }
        x[0] = p[0] | (p[1] << 16);
        x[1] = p[2] | (p[3] << 16);
    };
    store_words<1, 2, VEC>(row, col0, l, cols, chunk);
}

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100

// From a lane's max(|v|): F / A of its block in every lane, and A / F in lane 0.
__device__ __forceinline__ float block_scale(float m, uint32_t l, float F, float& scale) {
#pragma unroll
    for (uint32_t o = kLanes / 2; o; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    m = max_nan(m, kTiny);
    const float r = (l == 0 ? m : F) / (l == 0 ? F : m);
    scale = r;
    return __shfl_sync(0xffffffffu, r, 1, kLanes);
}

// ---- cm_quant_fp8, one scale per row and 128 columns -------------------------------------------
struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* scale;
    uint32_t rows, cols;
    uint64_t ldx, ldq, lds, x_bs, q_bs, s_bs;
    uint32_t row_tiles, col_tiles, tiles, step;   // row tiles a matrix, column tiles, row tiles of the batch, row tiles a pass
    uint32_t wide;                                // log2 of the column blocks of a CTA's tile
    FastDiv fd_row, fd_col;
};

// A warp takes 8 rows of a column block -- their scales lie side by side and fill one 32-byte
// sector --, a CTA 8 rows x 8 column blocks, 2 KB of a row of a 2-byte type, and then the rows
// `step` tiles on.  Where that many column blocks would leave warps idle in a narrow matrix or in the
// last column tile, the tile is 4, 2 or 1 blocks wide and 2, 4 or 8 times as high (8192 x 100 bf16: 6.5 -> 4.1 us).
constexpr uint32_t kQRows = 8, kQWarps = 8;

template <typename T>
constexpr uint32_t quant_ctas(bool vec) { return sizeof(T) == 4 ? 2 : vec ? 4 : 3; }     // resident an SM: two tiles' values are in registers

template <typename T, bool VEC, uint32_t FMT>
__global__ void __launch_bounds__(256, quant_ctas<T>(VEC)) quant_rows_kernel(const QuantArgs g) {
    griddep_wait();
    const uint32_t rt0 = g.fd_col.div(blockIdx.x), ct = blockIdx.x - rt0 * g.col_tiles;
    const uint32_t lane = threadIdx.x % 32, l = lane % kLanes;
    const uint32_t warp = threadIdx.x / 32, first = (warp >> g.wide) * kQRows + lane / kLanes, tile_rows = (kQWarps >> g.wide) * kQRows;
    const uint32_t cb = (ct << g.wide) + (warp & ((1u << g.wide) - 1)), col0 = cb * kFp8Block;
    if (col0 >= g.cols) return;                        // the whole warp
    const float F = fp8_largest(FMT);
    auto fetch = [&](uint32_t t, Raw<T>& v, uint32_t& z, uint32_t& row) {
        z = g.fd_row.div(t);
        row = (t - z * g.row_tiles) * tile_rows + first;
        if (row < g.rows) v.template load<VEC>((const T*)g.x + (uint64_t)z * g.x_bs + row * g.ldx, col0, l, g.cols);
        else v.clear();
    };
    Raw<T> next;
    uint32_t nz, nrow;
    fetch(rt0, next, nz, nrow);
    for (uint32_t t = rt0; t < g.tiles; t += g.step) {
        Raw<T> v = next;
        const uint32_t z = nz, row = nrow;
        if (t + g.step < g.tiles) fetch(t + g.step, next, nz, nrow);
        v.trim(col0, l, g.cols);
        float scale;
        const float inv = block_scale(v.max_abs(), l, F, scale);
        if (row < g.rows) {
            store_q32<VEC>(g.q + (uint64_t)z * g.q_bs + row * g.ldq, col0, l, g.cols, FMT, inv, [&](uint32_t p) { return v.pair(p); });
            if (l == 0) g.scale[(uint64_t)z * g.s_bs + cb * g.lds + row] = scale;
        }
    }
}

// ---- cm_quant_fp8, one scale per 128 x 128 block -----------------------------------------------
// A CTA of 512 threads holds its whole block in registers (32 values a thread), so it is read once.
template <typename T, bool VEC, uint32_t FMT>
__global__ void __launch_bounds__(512) quant_blocks_kernel(const QuantArgs g) {
    griddep_wait();
    __shared__ float top[16];
    const uint32_t rbz = g.fd_col.div(blockIdx.x), cb = blockIdx.x - rbz * g.col_tiles;
    const uint32_t z = g.fd_row.div(rbz), rb = rbz - z * g.row_tiles;
    const uint32_t l = threadIdx.x % kLanes, row = rb * kFp8Block + threadIdx.x / kLanes, col0 = cb * kFp8Block;
    const bool live = row < g.rows;
    Raw<T> v;
    if (live) v.template load<VEC>((const T*)g.x + (uint64_t)z * g.x_bs + row * g.ldx, col0, l, g.cols);
    else v.clear();
    v.trim(col0, l, g.cols);
    float m = v.max_abs();
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
    __syncthreads();
    m = max_nan(top[threadIdx.x % 16], kTiny);
#pragma unroll
    for (int o = 8; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float F = fp8_largest(FMT);
    if (live)
        store_q32<VEC>(g.q + (uint64_t)z * g.q_bs + row * g.ldq, col0, l, g.cols, FMT, F / m, [&](uint32_t p) { return v.pair(p); });
    if (threadIdx.x == 0) g.scale[(uint64_t)z * g.s_bs + rb * g.lds + cb] = m / F;
}

// ---- cm_rmsnorm_fp8 ----------------------------------------------------------------------------
// h = x + resid;  resid_out = h;  y = h / sqrt(mean(h^2) + eps) * weight;  q, scale = blocks of y.
// The sum stays unrounded in fp32 for the norm (resid_out alone is rounded to the tensors' type),
// and squares are summed in fp32 per lane, then over lanes and warps as a tree.
struct NormArgs {
    const void* x;
    const void* resid;
    const void* weight;
    void* resid_out;
    void* y;
    uint8_t* q;
    float* scale;
    uint32_t rows, cols, format, weight_type, per_row;
    uint64_t ldx, ldr, ldo, ldy, ldq, lds;
    float eps;
};

// per_row threads share a row, which stays in their registers, a block to 4 of them, and then take
// the row gridDim rows on: a part of a warp, or all warps of the CTA.  16-bit weights stay in the
// threads' registers for all their rows; others (WT = float: the weight is fp32, or of the other
// 16-bit type) are read again for each row.  BIG: rows of so many threads that there are registers for
// neither the weight nor the next row's loads.
template <typename T>
constexpr uint32_t norm_threads() { return sizeof(T) == 4 ? 384 : 512; }     // an SM's, at 168 and 128 registers each

template <typename T, typename WT, bool VEC, uint32_t THREADS>
__global__ void __launch_bounds__(THREADS, 1) rmsnorm_kernel(const NormArgs g) {
    griddep_wait();
    constexpr bool BIG = THREADS > norm_threads<T>(), KEEP = sizeof(WT) == 2 && !BIG;
    __shared__ float part[2][32];
    const bool whole = g.per_row > 32;           // all warps of the CTA on one row
    const uint32_t t = whole ? threadIdx.x : threadIdx.x & (g.per_row - 1), l = t % kLanes, blk = t / kLanes, col0 = blk * kFp8Block;
    const uint32_t per_cta = whole ? 1u : blockDim.x / g.per_row, warps = blockDim.x / 32;
    const bool mine = col0 < g.cols;
    uint32_t row = blockIdx.x * per_cta + (whole ? 0u : threadIdx.x / g.per_row);
    const uint32_t step = gridDim.x * per_cta;
    Raw<T> x, r;
    x.clear();
    r.clear();
    auto fetch = [&](uint64_t i) {
        if (!mine || i >= g.rows) return;
        x.template load<VEC>((const T*)g.x + i * g.ldx, col0, l, g.cols);
        if (g.resid) r.template load<VEC>((const T*)g.resid + i * g.ldr, col0, l, g.cols);
    };
    if (!BIG) fetch(row);
    Raw<WT> w;
    if (KEEP) {
        w.clear();
        if (mine && g.weight) w.template load<VEC>((const WT*)g.weight, col0, l, g.cols);
        w.trim(col0, l, g.cols);
    }
    const float F = fp8_largest(g.format), inv_cols = 1.0f / (float)g.cols;
    // every thread of a CTA makes the same number of passes: the barrier below is the CTA's
    for (uint32_t first = blockIdx.x * per_cta, pass = 0; first < g.rows; first += step, row += step, pass ^= 1) {
        const bool in = mine && row < g.rows;
        uint64_t h[kVals / 2];
        if (BIG) fetch(row);
        x.trim(col0, l, g.cols);
        r.trim(col0, l, g.cols);
        if (g.resid) {
#pragma unroll
            for (uint32_t p = 0; p < kVals / 2; ++p) h[p] = add2(x.pair(p), r.pair(p));
        } else {
#pragma unroll
            for (uint32_t p = 0; p < kVals / 2; ++p) h[p] = x.pair(p);
        }
        if (!BIG) fetch((uint64_t)row + step);
        // sum over the row of a thread's v^2; `set`: the partial sums' place
        auto squares = [&](auto v, uint32_t set) {
            uint64_t s2[4] = {};
#pragma unroll
            for (uint32_t p = 0; p < kVals / 2; ++p) s2[p % 4] = fma2(v(p), v(p), s2[p % 4]);
            float ss, other;
            unpack2(add2(add2(s2[0], s2[1]), add2(s2[2], s2[3])), ss, other);
            ss += other;
            for (uint32_t o = min(g.per_row, 32u) / 2; o; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            if (whole) {
                // two sets of partial sums in turn: one barrier a row is enough
                if (threadIdx.x % 32 == 0) part[set][threadIdx.x / 32] = ss;
                __syncthreads();
                ss = threadIdx.x % 32 < warps ? part[set][threadIdx.x % 32] : 0.0f;
#pragma unroll
                for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            }
            return ss;
        };
        float ms = fmaf(squares([&](uint32_t p) { return h[p]; }, pass), inv_cols, g.eps), rms = 1.0f, after = 1.0f;
        // Squares that leave fp32 (|h| from 2^64 / sqrt(cols) on, or mean and eps both below 2^-90, where squares
        // lose bits): the row is summed again times 2^-100 or 2^100, which the output takes back, where it is 2^100 in two
        // steps.  The branch is a warp's, and where a row has all warps of the CTA, the same for each of them.
        constexpr uint32_t kInf = 0x7f800000u, kSmall = (127u - 90u) << 23;
        const bool again = __any_sync(0xffffffffu, __float_as_uint(ms) - kSmall >= kInf - kSmall);
        if (again) {
            const bool large = isinf(ms), small = ms < __uint_as_float(kSmall);
            const float by = large ? 7.888609052210118e-31f : small ? 1.2676506002282294e30f : 1.0f;      // 2^-100, 2^100
            ms = fmaf(squares([&](uint32_t p) { return mul2(h[p], pack2(by, by)); }, pass ^ 1u), inv_cols, g.eps * by * by);
            if (whole) __syncthreads();                                           // the next row's sums go to the same place
            rms = small ? 1.180591620717411303424e21f : 1.0f;                        // 2^70
            after = small ? 1073741824.0f : by;                                     // 2^30
        }
        rms /= sqrtf(ms);
        if (in && g.resid_out) store32<T, VEC>((T*)g.resid_out + (uint64_t)row * g.ldo, col0, l, g.cols, h);
        auto by_factor = [&](float f) {
#pragma unroll
            for (uint32_t p = 0; p < kVals / 2; ++p) h[p] = mul2(h[p], pack2(f, f));
        };
        by_factor(rms);
        if (again) by_factor(after);
        auto times = [&](const auto& v) {
#pragma unroll
            for (uint32_t p = 0; p < kVals / 2; ++p) h[p] = mul2(h[p], v.pair(p));
        };
        auto times_read = [&](auto type) {
            using U = decltype(type);
            Raw<U> v;
            v.clear();
            if (mine) v.template load<VEC>((const U*)g.weight, col0, l, g.cols);
            v.trim(col0, l, g.cols);
            times(v);
        };
        if (g.weight) {
            if constexpr (KEEP) times(w);
            else if constexpr (sizeof(WT) == 2) times_read(WT{});
            else if (g.weight_type == CM_T_F32) times_read(float{});
            else if (g.weight_type == CM_T_F16) times_read(__half{});
            else times_read(__nv_bfloat16{});
        }
        if (in && g.y) store32<T, VEC>((T*)g.y + (uint64_t)row * g.ldy, col0, l, g.cols, h);
        if (!g.q) continue;
        if (col0 + kFp8Block > g.cols && rms > 3.4028234663852886e38f) {   // columns past the row's end hold no value: 0 * inf would be one
#pragma unroll
            for (uint32_t j = 0; j < kVals; j += 2) {
                float lo, hi;
                unpack2(h[j / 2], lo, hi);
                h[j / 2] = pack2(column(col0, l, j) < g.cols ? lo : 0.0f, column(col0, l, j + 1) < g.cols ? hi : 0.0f);
            }
        }
        float m = 0.0f, scale;
#pragma unroll
        for (uint32_t p = 0; p < kVals / 2; ++p) {
            float lo, hi;
            unpack2(h[p], lo, hi);
            m = max_abs3(m, lo, hi);
        }
        const float inv = block_scale(m, l, F, scale);
        if (in) {
            uint8_t* q = g.q + (uint64_t)row * g.ldq;
            auto value = [&](uint32_t p) { return h[p]; };
            if (g.format == CM_F8_E4M3) store_q32<VEC>(q, col0, l, g.cols, CM_F8_E4M3, inv, value);
            else store_q32<VEC>(q, col0, l, g.cols, CM_F8_E5M2, inv, value);
            if (l == 0) g.scale[blk * g.lds + row] = scale;
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
bool aligned(const void* p, uint64_t pitch_bytes, unsigned to) { return ((uintptr_t)p % to) == 0 && pitch_bytes % to == 0; }

// Whether the matrices of a batch do not overlap: each behind the one before, or their rows side by side.
bool apart(uint64_t rows, uint64_t ld, uint64_t cols, uint64_t batch, uint64_t stride) {
    return stride >= (rows - 1) * ld + cols || (stride >= cols && ld >= (batch - 1) * stride + cols);
}

template <typename T, bool VEC, uint32_t FMT>
void launch_quant(const QuantArgs& g, bool blocks, unsigned grid, cudaStream_t s) {
    if (blocks) launch_k(quant_blocks_kernel<T, VEC, FMT>, grid, 512, 0, s, g);
    else launch_k(quant_rows_kernel<T, VEC, FMT>, grid, 256, 0, s, g);
}

template <typename T>
void launch_quant_type(const QuantArgs& g, bool blocks, bool vec, unsigned format, unsigned grid, cudaStream_t s) {
    if (vec && format == CM_F8_E4M3) launch_quant<T, true, CM_F8_E4M3>(g, blocks, grid, s);
    else if (vec) launch_quant<T, true, CM_F8_E5M2>(g, blocks, grid, s);
    else if (format == CM_F8_E4M3) launch_quant<T, false, CM_F8_E4M3>(g, blocks, grid, s);
    else launch_quant<T, false, CM_F8_E5M2>(g, blocks, grid, s);
}

template <typename T, typename WT, bool VEC>
void launch_norm(const Context* cx, NormArgs g, cudaStream_t s) {
    // threads a row: four a block; below a warp a power of two, then whole warps
    const uint32_t need = (g.cols + kFp8Block - 1) / kFp8Block * kLanes;
    g.per_row = need > 32 ? (need + 31) / 32 * 32 : 4;
    while (g.per_row < need) g.per_row *= 2;
    const uint32_t threads = need > 32 ? g.per_row : 128, rows = threads / g.per_row;
    const uint32_t hold = (uint32_t)cx->sm_count * std::max(1u, norm_threads<T>() / threads);
    const uint32_t grid = std::min((g.rows + rows - 1) / rows, hold);
    if (threads <= norm_threads<T>()) launch_k(rmsnorm_kernel<T, WT, VEC, norm_threads<T>()>, grid, threads, 0, s, g);
    else if (threads <= 512) launch_k(rmsnorm_kernel<T, WT, VEC, 512>, grid, threads, 0, s, g);
    else launch_k(rmsnorm_kernel<T, WT, VEC, 1024>, grid, threads, 0, s, g);
}

template <typename T>
void launch_norm_type(const Context* cx, const NormArgs& g, bool vec, bool same, cudaStream_t s) {
    if (vec && same) launch_norm<T, T, true>(cx, g, s);
    else if (vec) launch_norm<T, float, true>(cx, g, s);
    else if (same) launch_norm<T, T, false>(cx, g, s);
    else launch_norm<T, float, false>(cx, g, s);
}

constexpr uint32_t kNormMaxCols = 1024 * kVals;

}  // namespace
}  // namespace cm

using namespace cm;

extern "C" int cm_quant_fp8_async(const void* x, unsigned x_type, uint8_t* q, float* scale, unsigned rows, unsigned cols,
                                  unsigned batch, uint64_t ldx, uint64_t ldq, uint64_t lds, uint64_t x_batch_stride,
                                  uint64_t q_batch_stride, uint64_t scale_batch_stride, unsigned format,
                                  unsigned block_rows, cm_stream_t stream) {
    const unsigned size = type_size(x_type);
    if (!size) return set_error(CM_EINVAL, "cm_quant_fp8: x_type %u", x_type);
    if (format > CM_F8_E5M2) return set_error(CM_EINVAL, "cm_quant_fp8: format %u", format);
    if (block_rows != 1 && block_rows != kFp8Block) return set_error(CM_EINVAL, "cm_quant_fp8: block_rows %u (1 or 128)", block_rows);
    const bool blocks = block_rows != 1;
    const uint64_t cb = (cols + 127ull) / 128, rb = (rows + 127ull) / 128;
    const uint64_t s_outer = blocks ? rb : cb, s_inner = blocks ? cb : rows;
    if (rows && cols && batch) {
        if (!x || !q || !scale) return set_error(CM_EINVAL, "cm_quant_fp8: null buffer");
        if ((uintptr_t)x % size || (uintptr_t)scale % 4) return set_error(CM_EINVAL, "cm_quant_fp8: buffer not aligned to its elements");
        if ((rows > 1 && (ldx < cols || ldq < cols)) || (s_outer > 1 && lds < s_inner))
            return set_error(CM_EINVAL, "cm_quant_fp8: a row pitch is shorter than its row");
        if (!extent_ok(rows, ldx, cols, size) || !extent_ok(rows, ldq, cols, 1) || !extent_ok(s_outer, lds, s_inner, 4) ||
            !extent_ok(batch, x_batch_stride, 0, size) || !extent_ok(batch, q_batch_stride, 0, 1) || !extent_ok(batch, scale_batch_stride, 0, 4))
            return set_error(CM_EINVAL, "cm_quant_fp8: sizes overflow");
        if (batch > 1 && (!apart(rows, ldq, cols, batch, q_batch_stride) || !apart(s_outer, lds, s_inner, batch, scale_batch_stride)))
            return set_error(CM_EINVAL, "cm_quant_fp8: the outputs of two batch steps overlap");
    }
    const Context* cx;
    int rc = enter(&cx);
    if (rc) return rc;
    if (rows == 0 || cols == 0 || batch == 0) return CM_OK;
    QuantArgs g{x, q, scale, rows, cols, ldx, ldq, lds, x_batch_stride, q_batch_stride, scale_batch_stride};
    for (g.wide = 3; g.wide && ((cb - 1) >> g.wide) + 1 > (cb + cb / 8) >> g.wide; --g.wide) {}     // at most an eighth of the warps idle
    const uint64_t tile_rows = (kQWarps >> g.wide) * kQRows;
    g.row_tiles = (uint32_t)(blocks ? rb : (rows + tile_rows - 1) / tile_rows);
    g.col_tiles = (uint32_t)(blocks ? cb : ((cb - 1) >> g.wide) + 1);
    const uint64_t tiles = (uint64_t)g.row_tiles * batch;
    if (tiles >= (1u << 30) || tiles * g.col_tiles >= (1u << 31)) return set_error(CM_EUNSUPPORTED, "cm_quant_fp8: more than 2^31 tiles");
    g.tiles = (uint32_t)tiles;
    // blocks: one CTA each; rows: as many CTAs as the SMs hold, each walking down its column tile
    const bool vec = aligned(x, ldx * size, 16) && aligned(q, ldq, 8) &&
                     (batch == 1 || (x_batch_stride * size % 16 == 0 && q_batch_stride % 8 == 0));
    const uint32_t hold = (x_type == CM_T_F32 ? quant_ctas<float>(vec) : quant_ctas<__half>(vec)) * cx->sm_count;
    g.step = blocks ? g.tiles : std::min(g.tiles, std::max(1u, hold / g.col_tiles));
    g.fd_row = FastDiv(g.row_tiles);
    g.fd_col = FastDiv(g.col_tiles);
    const unsigned grid = g.step * g.col_tiles;
    const cudaStream_t s = (cudaStream_t)stream;
    {
        ProfScope ps_(PK_FP8_QUANT, s);
        switch (x_type) {
            case CM_T_Q88: launch_quant_type<int16_t>(g, blocks, vec, format, grid, s); break;
            case CM_T_F32: launch_quant_type<float>(g, blocks, vec, format, grid, s); break;
            case CM_T_F16: launch_quant_type<__half>(g, blocks, vec, format, grid, s); break;
            default: launch_quant_type<__nv_bfloat16>(g, blocks, vec, format, grid, s); break;
        }
    }
    count_launch();
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CM_OK : cuda_error(e, "cm_quant_fp8");
}

extern "C" int cm_quant_fp8(const void* x, unsigned x_type, uint8_t* q, float* scale, unsigned rows, unsigned cols,
                            unsigned batch, uint64_t ldx, uint64_t ldq, uint64_t lds, uint64_t x_batch_stride,
                            uint64_t q_batch_stride, uint64_t scale_batch_stride, unsigned format, unsigned block_rows) {
    int rc = cm_quant_fp8_async(x, x_type, q, scale, rows, cols, batch, ldx, ldq, lds, x_batch_stride, q_batch_stride,
                                scale_batch_stride, format, block_rows, nullptr);
    return rc ? rc : finish_sync(nullptr);
}

extern "C" int cm_rmsnorm_fp8_async(const void* x, const void* resid, const void* weight, void* resid_out, void* y,
                                    uint8_t* q, float* scale, unsigned rows, unsigned cols, uint64_t ldx, uint64_t ldr,
                                    uint64_t ldo, uint64_t ldy, uint64_t ldq, uint64_t lds, unsigned type,
                                    unsigned weight_type, float eps, unsigned format, cm_stream_t stream) {
    const unsigned size = type_size(type), wsize = type_size(weight_type);
    if (!size || (weight && !wsize)) return set_error(CM_EINVAL, "cm_rmsnorm_fp8: type %u, weight type %u", type, weight_type);
    if (type == CM_T_Q88 || (weight && weight_type == CM_T_Q88)) return set_error(CM_EUNSUPPORTED, "cm_rmsnorm_fp8: Q8.8 tensors");
    if (format > CM_F8_E5M2) return set_error(CM_EINVAL, "cm_rmsnorm_fp8: format %u", format);
    if (!(eps >= 0.0f) || std::isinf(eps)) return set_error(CM_EINVAL, "cm_rmsnorm_fp8: eps must be finite and not negative");
    if (cols > kNormMaxCols) return set_error(CM_EUNSUPPORTED, "cm_rmsnorm_fp8: %u columns (at most %u)", cols, kNormMaxCols);
    const uint64_t cb = (cols + 127ull) / 128;
    if (rows && cols) {
        if (!x || (!y && !q)) return set_error(CM_EINVAL, "cm_rmsnorm_fp8: null buffer");
        if (!q != !scale) return set_error(CM_EINVAL, "cm_rmsnorm_fp8: q and scale go together");
        if (resid_out && !resid) return set_error(CM_EINVAL, "cm_rmsnorm_fp8: resid_out without resid");
        if ((uintptr_t)x % size || (uintptr_t)resid % size || (uintptr_t)resid_out % size || (uintptr_t)y % size ||
            (weight && (uintptr_t)weight % wsize) || (uintptr_t)scale % 4)
            return set_error(CM_EINVAL, "cm_rmsnorm_fp8: buffer not aligned to its elements");
        if ((rows > 1 && (ldx < cols || (resid && ldr < cols) || (resid_out && ldo < cols) || (y && ldy < cols) || (q && ldq < cols))) ||
            (q && cb > 1 && lds < rows))
            return set_error(CM_EINVAL, "cm_rmsnorm_fp8: a row pitch is shorter than its row");
        if (!extent_ok(rows, ldx, cols, size) || (resid && !extent_ok(rows, ldr, cols, size)) ||
            (resid_out && !extent_ok(rows, ldo, cols, size)) || (y && !extent_ok(rows, ldy, cols, size)) ||
            (q && (!extent_ok(rows, ldq, cols, 1) || !extent_ok(cb, lds, rows, 4))))
            return set_error(CM_EINVAL, "cm_rmsnorm_fp8: sizes overflow");
        if (rows >= (1u << 31)) return set_error(CM_EUNSUPPORTED, "cm_rmsnorm_fp8: more than 2^31 rows");
    }
    const Context* cx;
    int rc = enter(&cx);
    if (rc) return rc;
    if (rows == 0 || cols == 0) return CM_OK;
    NormArgs g{x, resid, weight, resid_out, y, q, scale, rows, cols, format, weight_type, 0, ldx, ldr, ldo, ldy, ldq, lds, eps};
    const cudaStream_t s = (cudaStream_t)stream;
    const bool vec = aligned(x, ldx * size, 16) && (!resid || aligned(resid, ldr * size, 16)) &&
                     (!resid_out || aligned(resid_out, ldo * size, 16)) && (!y || aligned(y, ldy * size, 16)) &&
                     (!q || aligned(q, ldq, 8)) && (!weight || aligned(weight, 0, 16));
    {
        ProfScope ps_(PK_FP8_QUANT, s);
        const bool same = !weight || weight_type == type;
        switch (type) {
            case CM_T_F32: launch_norm_type<float>(cx, g, vec, same, s); break;
            case CM_T_F16: launch_norm_type<__half>(cx, g, vec, same, s); break;
            default: launch_norm_type<__nv_bfloat16>(cx, g, vec, same, s); break;
        }
    }
    count_launch();
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CM_OK : cuda_error(e, "cm_rmsnorm_fp8");
}

extern "C" int cm_rmsnorm_fp8(const void* x, const void* resid, const void* weight, void* resid_out, void* y, uint8_t* q,
                              float* scale, unsigned rows, unsigned cols, uint64_t ldx, uint64_t ldr, uint64_t ldo,
                              uint64_t ldy, uint64_t ldq, uint64_t lds, unsigned type, unsigned weight_type, float eps,
                              unsigned format) {
    int rc = cm_rmsnorm_fp8_async(x, resid, weight, resid_out, y, q, scale, rows, cols, ldx, ldr, ldo, ldy, ldq, lds, type,
                                  weight_type, eps, format, nullptr);
    return rc ? rc : finish_sync(nullptr);
}

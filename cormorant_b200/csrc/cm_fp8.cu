// cm_fp8.cu -- quantisation to block-scaled 8-bit floating point, alone (cm_quant_fp8) and as the
// output of an RMS norm with the residual's addition (cm_rmsnorm_fp8).
//
// Both are HBM-bound: every input is read once and every output written once, all arithmetic in
// fp32 registers.  A row's 128-column block is the work of 16 neighbouring lanes of 8 values each
// (one 16-byte load of a 2-byte type), so the block's maximum is four shuffles inside a half warp
// and the 8-bit values leave as one 8-byte store a lane.  Rows whose pitch or base is not a
// multiple of those sizes run the same kernel with one-element accesses in which 16 neighbouring
// lanes touch 16 neighbouring elements.
#include <cmath>

#include "cm_fp8.cuh"

namespace cm {
namespace {

// ---- eight values of a 128-column block held by lane l (0..15) of a half warp ------------------
// VEC: columns col0 + 8*l .. +7;  else columns col0 + l + 16*j, j < 8.
template <typename T>
__device__ __forceinline__ void unpack8(const uint4 (&w)[sizeof(T) / 2], float (&v)[8]) {
    const T* t = reinterpret_cast<const T*>(w);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = to_f32(t[j]);
}

template <bool VEC>
__device__ __forceinline__ uint32_t column(uint32_t col0, uint32_t l, uint32_t j) {
    return VEC ? col0 + 8 * l + j : col0 + l + 16 * j;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* row, uint32_t col0, uint32_t l, uint32_t cols, float (&v)[8]) {
    if (VEC && col0 + 8 * l + 8 <= cols) {
        uint4 w[sizeof(T) / 2];
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(row + col0 + 8 * l)[i];
        unpack8<T>(w, v);
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t c = column<VEC>(col0, l, j);
        v[j] = c < cols ? to_f32(row[c]) : 0.0f;
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* row, uint32_t col0, uint32_t l, uint32_t cols, const float (&v)[8]) {
    if (VEC && col0 + 8 * l + 8 <= cols) {
        uint4 w[sizeof(T) / 2];
        T* t = reinterpret_cast<T*>(w);
#pragma unroll
        for (int j = 0; j < 8; ++j) from_f32(v[j], t[j]);
#pragma unroll
        for (uint32_t i = 0; i < sizeof(T) / 2; ++i) reinterpret_cast<uint4*>(row + col0 + 8 * l)[i] = w[i];
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t c = column<VEC>(col0, l, j);
        if (c < cols) from_f32(v[j], row[c]);
    }
}

// Bits of the largest magnitude: IEEE magnitudes order as integers, infinities above every finite
// value and NaN above infinity, so a NaN of the block reaches its scale.
__device__ __forceinline__ uint32_t max_bits(const float (&v)[8], uint32_t m) {
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[j]) & 0x7fffffffu);
    return m;
}

constexpr uint32_t kTinyBits = (127u - 100u) << 23;   // 2^-100

template <bool VEC>
__device__ __forceinline__ void store_q8(uint8_t* row, uint32_t col0, uint32_t l, uint32_t cols, uint32_t format,
                                         float inv, const float (&v)[8]) {
    uint32_t p[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = cvt_fp8x2(format, v[2 * j] * inv, v[2 * j + 1] * inv);
    if (VEC && col0 + 8 * l + 8 <= cols) {
        *reinterpret_cast<uint2*>(row + col0 + 8 * l) = make_uint2(p[0] | (p[1] << 16), p[2] | (p[3] << 16));
        return;
    }
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j) {
        const uint32_t c = column<VEC>(col0, l, j);
        if (c < cols) row[c] = (uint8_t)(p[j / 2] >> (8 * (j & 1)));
    }
}

// ---- cm_quant_fp8, one scale per row and 128 columns -------------------------------------------
struct QuantArgs {
    const void* x;
    uint8_t* q;
    float* scale;
    uint32_t rows, cols, format;
    uint64_t ldx, ldq, lds, x_bs, q_bs, s_bs;
    uint32_t row_tiles, col_tiles;   // tiles per matrix
};

// A CTA takes 8 rows x 4 column blocks: each row piece is 1 KB of a 2-byte type (whole DRAM
// bursts), and the 8 scales of a column block, which lie side by side, fill one 32-byte sector.
constexpr uint32_t kQRows = 8, kQCols = 4;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(QuantArgs g) {
    griddep_wait();
    const uint32_t ct = blockIdx.x % g.col_tiles, rest = blockIdx.x / g.col_tiles;
    const uint32_t rt = rest % g.row_tiles, z = rest / g.row_tiles;
    const uint32_t hw = threadIdx.x / 16, l = threadIdx.x % 16;
    const T* x = (const T*)g.x + (uint64_t)z * g.x_bs;
    constexpr uint32_t N = kQRows * kQCols / 16;
    float v[N][8];
    uint32_t row[N], cb[N];
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        const uint32_t item = hw + 16 * i;
        row[i] = rt * kQRows + item / kQCols;
        cb[i] = ct * kQCols + item % kQCols;
        if (row[i] < g.rows && cb[i] * kFp8Block < g.cols) {
            load8<T, VEC>(x + row[i] * g.ldx, cb[i] * kFp8Block, l, g.cols, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
    }
    const float F = fp8_largest(g.format);
#pragma unroll
    for (uint32_t i = 0; i < N; ++i) {
        uint32_t m = max_bits(v[i], kTinyBits);
#pragma unroll
        for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (row[i] >= g.rows || cb[i] * kFp8Block >= g.cols) continue;
        const float A = __uint_as_float(m);
        store_q8<VEC>(g.q + (uint64_t)z * g.q_bs + row[i] * g.ldq, cb[i] * kFp8Block, l, g.cols, g.format, F / A, v[i]);
        if (l == 0) g.scale[(uint64_t)z * g.s_bs + cb[i] * g.lds + row[i]] = A / F;
    }
}

// ---- cm_quant_fp8, one scale per 128 x 128 block -----------------------------------------------
// A CTA holds its whole block in registers (64 values a thread), so it is read once.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_blocks_kernel(QuantArgs g) {
    griddep_wait();
    __shared__ uint32_t top[8];
    const uint32_t cb = blockIdx.x % g.col_tiles, rest = blockIdx.x / g.col_tiles;
    const uint32_t rb = rest % g.row_tiles, z = rest / g.row_tiles;
    const uint32_t hw = threadIdx.x / 16, l = threadIdx.x % 16;
    const T* x = (const T*)g.x + (uint64_t)z * g.x_bs;
    float v[8][8];
    uint32_t m = kTinyBits;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = rb * kFp8Block + hw + 16 * i;
        if (row < g.rows) {
            load8<T, VEC>(x + row * g.ldx, cb * kFp8Block, l, g.cols, v[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) m = max_bits(v[i], m);
    m = __reduce_max_sync(0xffffffffu, m);
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) m = max(m, top[w]);
    const float F = fp8_largest(g.format), A = __uint_as_float(m), inv = F / A;
#pragma unroll
    for (uint32_t i = 0; i < 8; ++i) {
        const uint32_t row = rb * kFp8Block + hw + 16 * i;
        if (row < g.rows)
            store_q8<VEC>(g.q + (uint64_t)z * g.q_bs + row * g.ldq, cb * kFp8Block, l, g.cols, g.format, inv, v[i]);
    }
    if (threadIdx.x == 0) g.scale[(uint64_t)z * g.s_bs + rb * g.lds + cb] = A / F;
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
    uint32_t rows, cols, format, weight_type;
    uint64_t ldx, ldr, ldo, ldy, ldq, lds;
    float eps;
};

template <bool VEC>
__device__ __forceinline__ void load_weight8(const void* w, uint32_t type, uint32_t col0, uint32_t l, uint32_t cols, float (&v)[8]) {
    if (type == CM_T_F32) load8<float, VEC>((const float*)w, col0, l, cols, v);
    else if (type == CM_T_F16) load8<__half, VEC>((const __half*)w, col0, l, cols, v);
    else load8<__nv_bfloat16, VEC>((const __nv_bfloat16*)w, col0, l, cols, v);
}

// G threads share a row, which stays in their registers: at most NI chunks of 8 values each.
constexpr uint32_t kNormChunks = 4;

template <typename T, uint32_t G, bool VEC>
__global__ void __launch_bounds__(G < 128 ? 128 : G) rmsnorm_kernel(NormArgs g) {
    griddep_wait();
    constexpr uint32_t NI = kNormChunks, ROWS = G < 128 ? 128 / G : 1;
    __shared__ float part[32];
    const uint32_t t = threadIdx.x % G;
    const uint32_t row = blockIdx.x * ROWS + threadIdx.x / G;
    const bool live = row < g.rows;
    const uint32_t l = t % 16;
    const uint64_t r = live ? row : 0;
    float h[NI][8];
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
        const uint32_t col0 = (t / 16 + i * (G / 16)) * kFp8Block;
        if (live && col0 < g.cols) {
            load8<T, VEC>((const T*)g.x + r * g.ldx, col0, l, g.cols, h[i]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] = 0.0f;
        }
    }
    if (g.resid) {
#pragma unroll
        for (uint32_t i = 0; i < NI; ++i) {
            const uint32_t col0 = (t / 16 + i * (G / 16)) * kFp8Block;
            if (!live || col0 >= g.cols) continue;
            float v[8];
            load8<T, VEC>((const T*)g.resid + r * g.ldr, col0, l, g.cols, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) h[i][j] += v[j];
        }
    }
    float ss = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = fmaf(h[i][j], h[i][j], s);
        ss += s;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (G > 32) {
        if (threadIdx.x % 32 == 0) part[threadIdx.x / 32] = ss;
        __syncthreads();
        ss = threadIdx.x % 32 < G / 32 ? part[threadIdx.x % 32] : 0.0f;
#pragma unroll
        for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    const float rms = 1.0f / sqrtf(ss / (float)g.cols + g.eps);
    const float F = fp8_largest(g.format);
#pragma unroll
    for (uint32_t i = 0; i < NI; ++i) {
        const uint32_t blk = t / 16 + i * (G / 16), col0 = blk * kFp8Block;
        const bool in = live && col0 < g.cols;
        if (in && g.resid_out) store8<T, VEC>((T*)g.resid_out + r * g.ldo, col0, l, g.cols, h[i]);
        float y[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) y[j] = h[i][j] * rms;
        if (in && g.weight) {
            float w[8];
            load_weight8<VEC>(g.weight, g.weight_type, col0, l, g.cols, w);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= w[j];
        }
        if (in && g.y) store8<T, VEC>((T*)g.y + r * g.ldy, col0, l, g.cols, y);
        if (g.q) {
            if (!VEC || col0 + 8 * l + 8 > g.cols) {   // columns past the row's end hold no value (an infinite rms would make 0 * inf of them)
#pragma unroll
                for (uint32_t j = 0; j < 8; ++j)
                    if (column<VEC>(col0, l, j) >= g.cols) y[j] = 0.0f;
            }
            uint32_t m = max_bits(y, kTinyBits);
#pragma unroll
            for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
            if (in) {
                const float A = __uint_as_float(m);
                store_q8<VEC>(g.q + r * g.ldq, col0, l, g.cols, g.format, F / A, y);
                if (l == 0) g.scale[blk * g.lds + r] = A / F;
            }
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
bool aligned(const void* p, uint64_t pitch_bytes, unsigned to) { return ((uintptr_t)p % to) == 0 && pitch_bytes % to == 0; }

template <bool VEC>
void launch_quant(const QuantArgs& g, unsigned type, bool blocks, unsigned grid, cudaStream_t s) {
#define CM_QUANT(T)                                                        \
    do {                                                                   \
        if (blocks) launch_k(quant_blocks_kernel<T, VEC>, grid, 256, 0, s, g); \
        else launch_k(quant_rows_kernel<T, VEC>, grid, 256, 0, s, g);      \
    } while (0)
    switch (type) {
        case CM_T_Q88: CM_QUANT(int16_t); break;
        case CM_T_F32: CM_QUANT(float); break;
        case CM_T_F16: CM_QUANT(__half); break;
        default: CM_QUANT(__nv_bfloat16); break;
    }
#undef CM_QUANT
}

template <typename T, bool VEC>
void launch_norm(const Context* cx, const NormArgs& g, cudaStream_t s) {
    // Threads a row: enough for the row to fit their registers (32 values each); rows that do not
    // fill the GPU take one chunk a thread instead, so that a row's loads are all in flight at once.
    const bool few = (uint64_t)g.rows < 4ull * cx->sm_count;
    const uint32_t need = (g.cols + 7) / 8;             // chunks of 8 values
    const uint32_t fit = few ? need : (need + kNormChunks - 1) / kNormChunks;
    if (fit <= 32 && need <= 32 * kNormChunks) launch_k(rmsnorm_kernel<T, 32, VEC>, (g.rows + 3) / 4, 128, 0, s, g);
    else if (fit <= 128 && need <= 128 * kNormChunks) launch_k(rmsnorm_kernel<T, 128, VEC>, g.rows, 128, 0, s, g);
    else if (fit <= 512 && need <= 512 * kNormChunks) launch_k(rmsnorm_kernel<T, 512, VEC>, g.rows, 512, 0, s, g);
    else launch_k(rmsnorm_kernel<T, 1024, VEC>, g.rows, 1024, 0, s, g);
}

template <bool VEC>
void launch_norm_type(const Context* cx, const NormArgs& g, unsigned type, cudaStream_t s) {
    switch (type) {
        case CM_T_F32: launch_norm<float, VEC>(cx, g, s); break;
        case CM_T_F16: launch_norm<__half, VEC>(cx, g, s); break;
        default: launch_norm<__nv_bfloat16, VEC>(cx, g, s); break;
    }
}

constexpr uint32_t kNormMaxCols = 1024 * 8 * kNormChunks;

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
        if (batch > 1 && (q_batch_stride < (rows - 1) * ldq + cols || scale_batch_stride < (s_outer - 1) * lds + s_inner))
            return set_error(CM_EINVAL, "cm_quant_fp8: the outputs of two batch steps overlap");
    }
    const Context* cx;
    int rc = enter(&cx);
    if (rc) return rc;
    if (rows == 0 || cols == 0 || batch == 0) return CM_OK;
    QuantArgs g{x, q, scale, rows, cols, format, ldx, ldq, lds, x_batch_stride, q_batch_stride, scale_batch_stride, 0, 0};
    g.row_tiles = (uint32_t)(blocks ? rb : (rows + (uint64_t)kQRows - 1) / kQRows);
    g.col_tiles = (uint32_t)(blocks ? cb : (cb + kQCols - 1) / kQCols);
    const unsigned __int128 grid = (unsigned __int128)g.row_tiles * g.col_tiles * batch;
    if (grid >= (1u << 31)) return set_error(CM_EUNSUPPORTED, "cm_quant_fp8: more than 2^31 tiles");
    const cudaStream_t s = (cudaStream_t)stream;
    const bool vec = aligned(x, ldx * size, 16) && aligned(q, ldq, 8) &&
                     (batch == 1 || (x_batch_stride * size % 16 == 0 && q_batch_stride % 8 == 0));
    {
        ProfScope ps_(PK_FP8_QUANT, s);
        if (vec) launch_quant<true>(g, x_type, blocks, (unsigned)grid, s);
        else launch_quant<false>(g, x_type, blocks, (unsigned)grid, s);
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
    NormArgs g{x, resid, weight, resid_out, y, q, scale, rows, cols, format, weight_type, ldx, ldr, ldo, ldy, ldq, lds, eps};
    const cudaStream_t s = (cudaStream_t)stream;
    const bool vec = aligned(x, ldx * size, 16) && (!resid || aligned(resid, ldr * size, 16)) &&
                     (!resid_out || aligned(resid_out, ldo * size, 16)) && (!y || aligned(y, ldy * size, 16)) &&
                     (!q || aligned(q, ldq, 8)) && (!weight || aligned(weight, 0, 16));
    {
        ProfScope ps_(PK_FP8_QUANT, s);
        if (vec) launch_norm_type<true>(cx, g, type, s);
        else launch_norm_type<false>(cx, g, type, s);
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

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
// (With 16 lanes a block and 8 values each, 8192 x 4096 bf16 took 30.9 us instead of 20.3.)
// Rows whose pitch or base is not a multiple of the vector sizes run the same kernel with
// one-element accesses, column l + 4 * j of the block.
#include <cmath>

#include "cm_fp8.cuh"

namespace cm {
namespace {

constexpr uint32_t kLanes = 4;                       // lanes of a block
constexpr uint32_t kVals = kFp8Block / kLanes;       // values of a lane
constexpr uint32_t kChunks = kVals / 8;

template <bool VEC>
__device__ __forceinline__ uint32_t column(uint32_t col0, uint32_t l, uint32_t j) {
    return VEC ? col0 + 8 * (kLanes * (j / 8) + l) + j % 8 : col0 + l + kLanes * j;
}

// 32 values of a lane, 0 past the row's end
template <typename T, bool VEC>
__device__ __forceinline__ void load32(const T* row, uint32_t col0, uint32_t l, uint32_t cols, float (&v)[kVals]) {
    if (VEC && col0 + kFp8Block <= cols) {
        uint4 w[kChunks][sizeof(T) / 2];
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i)
#pragma unroll
            for (uint32_t k = 0; k < sizeof(T) / 2; ++k)
                w[i][k] = reinterpret_cast<const uint4*>(row + col0 + 8 * (kLanes * i + l))[k];
#pragma unroll
        for (uint32_t i = 0; i < kChunks; ++i) {
            const T* t = reinterpret_cast<const T*>(w[i]);
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) v[8 * i + j] = to_f32(t[j]);
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
        if (VEC && column<VEC>(col0, l, 8 * i) + 8 <= cols) {    // a whole chunk of the last, partial block
            uint4 w[sizeof(T) / 2];
#pragma unroll
            for (uint32_t k = 0; k < sizeof(T) / 2; ++k) w[k] = reinterpret_cast<const uint4*>(row + column<VEC>(col0, l, 8 * i))[k];
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) v[8 * i + j] = to_f32(reinterpret_cast<const T*>(w)[j]);
            continue;
        }
#pragma unroll
        for (uint32_t j = 8 * i; j < 8 * i + 8; ++j) {
            const uint32_t c = column<VEC>(col0, l, j);
            v[j] = c < cols ? to_f32(row[c]) : 0.0f;
        }
    }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store32(T* row, uint32_t col0, uint32_t l, uint32_t cols, const float (&v)[kVals]) {
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
        if (VEC && column<VEC>(col0, l, 8 * i) + 8 <= cols) {
            uint4 w[sizeof(T) / 2];
            T* t = reinterpret_cast<T*>(w);
#pragma unroll
            for (uint32_t j = 0; j < 8; ++j) from_f32(v[8 * i + j], t[j]);
#pragma unroll
            for (uint32_t k = 0; k < sizeof(T) / 2; ++k) reinterpret_cast<uint4*>(row + column<VEC>(col0, l, 8 * i))[k] = w[k];
            continue;
        }
#pragma unroll
        for (uint32_t j = 8 * i; j < 8 * i + 8; ++j) {
            const uint32_t c = column<VEC>(col0, l, j);
            if (c < cols) from_f32(v[j], row[c]);
        }
    }
}

// max(|v|) and a floor; a NaN among them is the result, so that it reaches the block's scale
__device__ __forceinline__ float max_abs(const float (&v)[kVals], float m) {
#pragma unroll
    for (uint32_t j = 0; j < kVals; j += 2)
        asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(v[j]), "f"(v[j + 1]));
    return m;
}
__device__ __forceinline__ float max_nan(float a, float b) {
    float m;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
    return m;
}

constexpr float kTiny = 7.888609052210118e-31f;   // 2^-100

template <bool VEC>
__device__ __forceinline__ void store_q32(uint8_t* row, uint32_t col0, uint32_t l, uint32_t cols, uint32_t format, float inv,
                                          const float (&v)[kVals]) {
    uint32_t p[kVals / 2];
    if (format == CM_F8_E4M3) {
#pragma unroll
        for (uint32_t j = 0; j < kVals / 2; ++j) p[j] = cvt_fp8x2(CM_F8_E4M3, v[2 * j] * inv, v[2 * j + 1] * inv);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kVals / 2; ++j) p[j] = cvt_fp8x2(CM_F8_E5M2, v[2 * j] * inv, v[2 * j + 1] * inv);
    }
#pragma unroll
    for (uint32_t i = 0; i < kChunks; ++i) {
        if (VEC && column<VEC>(col0, l, 8 * i) + 8 <= cols) {
            *reinterpret_cast<uint2*>(row + column<VEC>(col0, l, 8 * i)) =
                make_uint2(p[4 * i] | (p[4 * i + 1] << 16), p[4 * i + 2] | (p[4 * i + 3] << 16));
            continue;
        }
#pragma unroll
        for (uint32_t j = 8 * i; j < 8 * i + 8; ++j) {
            const uint32_t c = column<VEC>(col0, l, j);
            if (c < cols) row[c] = (uint8_t)(p[j / 2] >> (8 * (j & 1)));
        }
    }
}

// From a lane's max(|v|): F / A of its block in every lane, and A / F in lane 0.
__device__ __forceinline__ float block_scale(float m, uint32_t l, float F, float& scale) {
#pragma unroll
    for (uint32_t o = kLanes / 2; o; o /= 2) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float r = (l == 0 ? m : F) / (l == 0 ? F : m);
    scale = r;
    return __shfl_sync(0xffffffffu, r, 1, kLanes);
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

// A warp takes 8 rows of a column block -- their scales lie side by side and fill one 32-byte
// sector --, a CTA 8 rows x 8 column blocks, 2 KB of a row of a 2-byte type.
constexpr uint32_t kQRows = 8, kQCols = 8;

template <typename T, bool VEC>
__global__ void __launch_bounds__(256) quant_rows_kernel(QuantArgs g) {
    griddep_wait();
    const uint32_t ct = blockIdx.x % g.col_tiles, rest = blockIdx.x / g.col_tiles;
    const uint32_t rt = rest % g.row_tiles, z = rest / g.row_tiles;
    const uint32_t lane = threadIdx.x % 32, l = lane % kLanes;
    const uint32_t row = rt * kQRows + lane / kLanes, cb = ct * kQCols + threadIdx.x / 32, col0 = cb * kFp8Block;
    if (col0 >= g.cols) return;                        // the whole warp
    const bool live = row < g.rows;
    float v[kVals];
    if (live) {
        load32<T, VEC>((const T*)g.x + (uint64_t)z * g.x_bs + row * g.ldx, col0, l, g.cols, v);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kVals; ++j) v[j] = 0.0f;
    }
    float scale;
    const float inv = block_scale(max_abs(v, kTiny), l, fp8_largest(g.format), scale);
    if (!live) return;
    store_q32<VEC>(g.q + (uint64_t)z * g.q_bs + row * g.ldq, col0, l, g.cols, g.format, inv, v);
    if (l == 0) g.scale[(uint64_t)z * g.s_bs + cb * g.lds + row] = scale;
}

// ---- cm_quant_fp8, one scale per 128 x 128 block -----------------------------------------------
// A CTA of 512 threads holds its whole block in registers (32 values a thread), so it is read once.
template <typename T, bool VEC>
__global__ void __launch_bounds__(512) quant_blocks_kernel(QuantArgs g) {
    griddep_wait();
    __shared__ float top[16];
    const uint32_t cb = blockIdx.x % g.col_tiles, rest = blockIdx.x / g.col_tiles;
    const uint32_t rb = rest % g.row_tiles, z = rest / g.row_tiles;
    const uint32_t l = threadIdx.x % kLanes, row = rb * kFp8Block + threadIdx.x / kLanes, col0 = cb * kFp8Block;
    const bool live = row < g.rows;
    float v[kVals];
    if (live) {
        load32<T, VEC>((const T*)g.x + (uint64_t)z * g.x_bs + row * g.ldx, col0, l, g.cols, v);
    } else {
#pragma unroll
        for (uint32_t j = 0; j < kVals; ++j) v[j] = 0.0f;
    }
    float m = max_abs(v, kTiny);
#pragma unroll
    for (int o = 16; o; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (threadIdx.x % 32 == 0) top[threadIdx.x / 32] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 16; ++w) m = max_nan(m, top[w]);
    const float F = fp8_largest(g.format);
    if (live) store_q32<VEC>(g.q + (uint64_t)z * g.q_bs + row * g.ldq, col0, l, g.cols, g.format, F / m, v);
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
    uint32_t rows, cols, format, weight_type;
    uint64_t ldx, ldr, ldo, ldy, ldq, lds;
    float eps;
};

template <bool VEC>
__device__ __forceinline__ void load_weight(const void* w, uint32_t type, uint32_t col0, uint32_t l, uint32_t cols, float (&v)[kVals]) {
    if (type == CM_T_F32) load32<float, VEC>((const float*)w, col0, l, cols, v);
    else if (type == CM_T_F16) load32<__half, VEC>((const __half*)w, col0, l, cols, v);
    else load32<__nv_bfloat16, VEC>((const __nv_bfloat16*)w, col0, l, cols, v);
}

// G threads share a row, which stays in their registers, a block to 4 of them.
template <typename T, uint32_t G, bool VEC>
__global__ void __launch_bounds__(G < 128 ? 128 : G) rmsnorm_kernel(NormArgs g) {
    griddep_wait();
    constexpr uint32_t ROWS = G < 128 ? 128 / G : 1;
    __shared__ float part[32];
    const uint32_t t = threadIdx.x % G, l = t % kLanes, blk = t / kLanes, col0 = blk * kFp8Block;
    const uint32_t row = blockIdx.x * ROWS + threadIdx.x / G;
    const bool in = row < g.rows && col0 < g.cols;
    const uint64_t r = row;
    float h[kVals];
#pragma unroll
    for (uint32_t j = 0; j < kVals; ++j) h[j] = 0.0f;
    if (in) {
        load32<T, VEC>((const T*)g.x + r * g.ldx, col0, l, g.cols, h);
        if (g.resid) {
            float v[kVals];
            load32<T, VEC>((const T*)g.resid + r * g.ldr, col0, l, g.cols, v);
#pragma unroll
            for (uint32_t j = 0; j < kVals; ++j) h[j] += v[j];
        }
    }
    float ss = 0.0f;
    {
        float s[4] = {};
#pragma unroll
        for (uint32_t j = 0; j < kVals; ++j) s[j % 4] = fmaf(h[j], h[j], s[j % 4]);
        ss = (s[0] + s[1]) + (s[2] + s[3]);
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
    if (in && g.resid_out) store32<T, VEC>((T*)g.resid_out + r * g.ldo, col0, l, g.cols, h);
#pragma unroll
    for (uint32_t j = 0; j < kVals; ++j) h[j] *= rms;
    if (in && g.weight) {
        float w[kVals];
        load_weight<VEC>(g.weight, g.weight_type, col0, l, g.cols, w);
#pragma unroll
        for (uint32_t j = 0; j < kVals; ++j) h[j] *= w[j];
    }
    if (in && g.y) store32<T, VEC>((T*)g.y + r * g.ldy, col0, l, g.cols, h);
    if (g.q) {
        if (col0 + kFp8Block > g.cols) {   // columns past the row's end hold no value (an infinite rms would make 0 * inf of them)
#pragma unroll
            for (uint32_t j = 0; j < kVals; ++j)
                if (column<VEC>(col0, l, j) >= g.cols) h[j] = 0.0f;
        }
        float scale;
        const float inv = block_scale(max_abs(h, kTiny), l, fp8_largest(g.format), scale);
        if (in) {
            store_q32<VEC>(g.q + r * g.ldq, col0, l, g.cols, g.format, inv, h);
            if (l == 0) g.scale[blk * g.lds + r] = scale;
        }
    }
}

// ---- host ---------------------------------------------------------------------------------------
bool aligned(const void* p, uint64_t pitch_bytes, unsigned to) { return ((uintptr_t)p % to) == 0 && pitch_bytes % to == 0; }

template <bool VEC>
void launch_quant(const QuantArgs& g, unsigned type, bool blocks, unsigned grid, cudaStream_t s) {
#define CM_QUANT(T)                                                        \
    do {                                                                   \
        if (blocks) launch_k(quant_blocks_kernel<T, VEC>, grid, 512, 0, s, g); \
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
void launch_norm(const NormArgs& g, cudaStream_t s) {
    // threads a row: the fewest that hold it (32 values each)
    if (g.cols <= 32 * kVals) launch_k(rmsnorm_kernel<T, 32, VEC>, (g.rows + 3) / 4, 128, 0, s, g);
    else if (g.cols <= 128 * kVals) launch_k(rmsnorm_kernel<T, 128, VEC>, g.rows, 128, 0, s, g);
    else if (g.cols <= 256 * kVals) launch_k(rmsnorm_kernel<T, 256, VEC>, g.rows, 256, 0, s, g);
    else if (g.cols <= 512 * kVals) launch_k(rmsnorm_kernel<T, 512, VEC>, g.rows, 512, 0, s, g);
    else launch_k(rmsnorm_kernel<T, 1024, VEC>, g.rows, 1024, 0, s, g);
}

template <bool VEC>
void launch_norm_type(const NormArgs& g, unsigned type, cudaStream_t s) {
    switch (type) {
        case CM_T_F32: launch_norm<float, VEC>(g, s); break;
        case CM_T_F16: launch_norm<__half, VEC>(g, s); break;
        default: launch_norm<__nv_bfloat16, VEC>(g, s); break;
    }
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
        if (vec) launch_norm_type<true>(g, type, s);
        else launch_norm_type<false>(g, type, s);
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

// cm_fp8_gemm.cu -- matrix products of block-scaled 8-bit floating point operands:
//   c[i][j] = sum over 128-deep blocks t of  a_scale[t][i] * b_scale[j / 128][t] * (a[i][t] . b[j][t])
// dense (cm_matmul_fp8) and grouped by expert (cm_matmul_fp8_grouped: rows offsets[g] ..
// offsets[g+1] - 1 of a and c use b[g]).  A block's products are summed in fp32, scaled, and the
// scaled blocks are summed in fp32; one rounding to the output type.
#include <algorithm>

#include "cm_fp8.cuh"

namespace cm {
namespace {

struct Fp8Args {
    const uint8_t* a;
    const uint8_t* b;
    const float* as;
    const float* bs;
    void* c;
    const int32_t* offsets;          // null: one group of all rows
    uint32_t groups, n, k, m, a_format, b_format, c_type;
    uint64_t lda, a_lds, ldb, b_lds, b_gs, bs_gs, ldc;
};

__device__ __forceinline__ float fp8_f32(uint32_t format, uint8_t v) {
    uint32_t h;
    if (format == CM_F8_E4M3) asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
    else asm("cvt.rn.f16x2.e5m2x2 %0, %1;" : "=r"(h) : "h"((uint16_t)v));
    return __half2float(__ushort_as_half((unsigned short)(h & 0xffffu)));
}

__device__ __forceinline__ void store_c(void* c, uint32_t type, uint64_t i, float v) {
    switch (type) {
        case CM_T_Q88: from_f32(v, ((int16_t*)c)[i]); break;
        case CM_T_F32: from_f32(v, ((float*)c)[i]); break;
        case CM_T_F16: from_f32(v, ((__half*)c)[i]); break;
        default: from_f32(v, ((__nv_bfloat16*)c)[i]); break;
    }
}

constexpr uint32_t ST = 64, SK = 32;

__global__ void __launch_bounds__(256) fp8_simple_kernel(Fp8Args g) {
    griddep_wait();
    __shared__ float as[ST][SK + 1], bs[ST][SK + 1];
    uint32_t row0 = blockIdx.y * ST, row1 = g.n, group = 0;
    if (g.offsets) {
        // this CTA's token tile: groups in order, each in whole tiles; offsets are held to 0..n and
        // to increasing order, so that no value of theirs can reach outside a and c
        uint32_t left = blockIdx.y, lo = (uint32_t)min(max(g.offsets[0], 0), (int)g.n);
        for (;; ++group) {
            if (group == g.groups) return;
            const uint32_t hi = max(lo, (uint32_t)min(max(g.offsets[group + 1], 0), (int)g.n));
            const uint32_t tiles = (hi - lo + ST - 1) / ST;
            if (left < tiles) { row0 = lo + left * ST; row1 = hi; break; }
            left -= tiles;
            lo = hi;
        }
    }
    const uint32_t col0 = blockIdx.x * ST;
    const uint8_t* b = g.b + group * g.b_gs;
    const float* bsc = g.bs + group * g.bs_gs;
    const uint32_t tx = threadIdx.x % 16, ty = threadIdx.x / 16;
    float acc[4][4] = {}, part[4][4] = {};
    for (uint32_t k0 = 0; k0 < g.k; k0 += SK) {
        for (uint32_t e = threadIdx.x; e < ST * SK; e += 256) {
            const uint32_t r = e / SK, kk = e % SK;
            as[r][kk] = row0 + r < row1 && k0 + kk < g.k ? fp8_f32(g.a_format, g.a[(row0 + r) * g.lda + k0 + kk]) : 0.0f;
            bs[r][kk] = col0 + r < g.m && k0 + kk < g.k ? fp8_f32(g.b_format, b[(col0 + r) * g.ldb + k0 + kk]) : 0.0f;
        }
        __syncthreads();
        for (uint32_t kk = 0; kk < SK; ++kk)
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) part[i][j] = fmaf(as[ty + 16 * i][kk], bs[tx + 16 * j][kk], part[i][j]);
        __syncthreads();
        if ((k0 + SK) % kFp8Block == 0 || k0 + SK >= g.k) {
            const uint32_t kb = k0 / kFp8Block;
            for (int i = 0; i < 4; ++i)
                for (int j = 0; j < 4; ++j) {
                    const uint32_t r = row0 + ty + 16 * i, cc = col0 + tx + 16 * j;
                    const float s = r < row1 && cc < g.m ? g.as[kb * g.a_lds + r] * bsc[(cc / kFp8Block) * g.b_lds + kb] : 0.0f;
                    acc[i][j] = fmaf(part[i][j], s, acc[i][j]);
                    part[i][j] = 0.0f;
                }
        }
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4; ++j) {
            const uint32_t r = row0 + ty + 16 * i, cc = col0 + tx + 16 * j;
            if (r < row1 && cc < g.m) store_c(g.c, g.c_type, r * g.ldc + cc, acc[i][j]);
        }
}

constexpr uint32_t kMaxGroups = 1024;

int fp8_check(const char* who, const Fp8Args& g) {
    const unsigned size = type_size(g.c_type);
    if (!size) return set_error(CM_EINVAL, "%s: c_type %u", who, g.c_type);
    if (g.a_format > CM_F8_E5M2 || g.b_format > CM_F8_E5M2) return set_error(CM_EINVAL, "%s: format %u, %u", who, g.a_format, g.b_format);
    if (g.n == 0 || g.m == 0 || g.groups == 0) return CM_OK;
    const uint64_t kb = (g.k + 127ull) / 128, mb = (g.m + 127ull) / 128;
    if (!g.c || (g.k && (!g.a || !g.b || !g.as || !g.bs))) return set_error(CM_EINVAL, "%s: null buffer", who);
    if ((uintptr_t)g.c % size || (uintptr_t)g.as % 4 || (uintptr_t)g.bs % 4 || (uintptr_t)g.offsets % 4)
        return set_error(CM_EINVAL, "%s: buffer not aligned to its elements", who);
    if ((g.n > 1 && (g.lda < g.k || g.ldc < g.m)) || (g.m > 1 && g.ldb < g.k) || (kb > 1 && g.a_lds < g.n) || (mb > 1 && g.b_lds < kb))
        return set_error(CM_EINVAL, "%s: a row pitch is shorter than its row", who);
    if (!extent_ok(g.n, g.lda, g.k, 1) || !extent_ok(g.m, g.ldb, g.k, 1) || !extent_ok(g.n, g.ldc, g.m, size) ||
        !extent_ok(kb, g.a_lds, g.n, 4) || !extent_ok(mb, g.b_lds, kb, 4) || !extent_ok(g.groups, g.b_gs, 0, 1) ||
        !extent_ok(g.groups, g.bs_gs, 0, 4))
        return set_error(CM_EINVAL, "%s: sizes overflow", who);
    if (g.n >= (1u << 31) || g.k >= (1u << 31) || g.m >= (1u << 31)) return set_error(CM_EUNSUPPORTED, "%s: a size above 2^31 - 1", who);
    return CM_OK;
}

int fp8_launch(const char* who, const Context* cx, const Fp8Args& g, cudaStream_t s) {
    (void)cx;
    const dim3 grid((g.m + ST - 1) / ST, (unsigned)(g.offsets ? (uint64_t)g.n / ST + g.groups : (g.n + ST - 1) / ST));
    {
        ProfScope ps_(PK_FP8_GEMM, s);
        launch_k(fp8_simple_kernel, grid, 256, 0, s, g);
    }
    count_launch();
    cudaError_t e = cudaGetLastError();
    return e == cudaSuccess ? CM_OK : cuda_error(e, who);
}

}  // namespace
}  // namespace cm

using namespace cm;

extern "C" int cm_matmul_fp8_async(const uint8_t* a, const float* a_scale, const uint8_t* b, const float* b_scale, void* c,
                                   unsigned n, unsigned k, unsigned m, uint64_t lda, uint64_t a_scale_ld, uint64_t ldb,
                                   uint64_t b_scale_ld, uint64_t ldc, unsigned a_format, unsigned b_format,
                                   unsigned c_type, cm_stream_t stream) {
    Fp8Args g{a, b, a_scale, b_scale, c, nullptr, 1, n, k, m, a_format, b_format, c_type, lda, a_scale_ld, ldb, b_scale_ld, 0, 0, ldc};
    int rc = fp8_check("cm_matmul_fp8", g);
    const Context* cx;
    if (!rc) rc = enter(&cx);
    if (rc) return rc;
    if (n == 0 || m == 0) return CM_OK;
    return fp8_launch("cm_matmul_fp8", cx, g, (cudaStream_t)stream);
}

extern "C" int cm_matmul_fp8(const uint8_t* a, const float* a_scale, const uint8_t* b, const float* b_scale, void* c,
                             unsigned n, unsigned k, unsigned m, uint64_t lda, uint64_t a_scale_ld, uint64_t ldb,
                             uint64_t b_scale_ld, uint64_t ldc, unsigned a_format, unsigned b_format, unsigned c_type) {
    int rc = cm_matmul_fp8_async(a, a_scale, b, b_scale, c, n, k, m, lda, a_scale_ld, ldb, b_scale_ld, ldc, a_format, b_format,
                                 c_type, nullptr);
    return rc ? rc : finish_sync(nullptr);
}

extern "C" int cm_matmul_fp8_grouped_async(const uint8_t* a, const float* a_scale, const uint8_t* b, const float* b_scale,
                                           void* c, const int32_t* offsets, unsigned groups, unsigned n, unsigned k,
                                           unsigned m, uint64_t lda, uint64_t a_scale_ld, uint64_t ldb, uint64_t b_scale_ld,
                                           uint64_t b_group_stride, uint64_t b_scale_group_stride, uint64_t ldc,
                                           unsigned a_format, unsigned b_format, unsigned c_type, cm_stream_t stream) {
    Fp8Args g{a, b, a_scale, b_scale, c, offsets, groups, n, k, m, a_format, b_format, c_type,
              lda, a_scale_ld, ldb, b_scale_ld, b_group_stride, b_scale_group_stride, ldc};
    int rc = fp8_check("cm_matmul_fp8_grouped", g);
    if (!rc && groups && !offsets) rc = set_error(CM_EINVAL, "cm_matmul_fp8_grouped: null offsets");
    if (!rc && groups > kMaxGroups) rc = set_error(CM_EUNSUPPORTED, "cm_matmul_fp8_grouped: %u groups (at most %u)", groups, kMaxGroups);
    const Context* cx;
    if (!rc) rc = enter(&cx);
    if (rc) return rc;
    if (n == 0 || m == 0 || groups == 0) return CM_OK;
    return fp8_launch("cm_matmul_fp8_grouped", cx, g, (cudaStream_t)stream);
}

extern "C" int cm_matmul_fp8_grouped(const uint8_t* a, const float* a_scale, const uint8_t* b, const float* b_scale, void* c,
                                     const int32_t* offsets, unsigned groups, unsigned n, unsigned k, unsigned m,
                                     uint64_t lda, uint64_t a_scale_ld, uint64_t ldb, uint64_t b_scale_ld,
                                     uint64_t b_group_stride, uint64_t b_scale_group_stride, uint64_t ldc,
                                     unsigned a_format, unsigned b_format, unsigned c_type) {
    int rc = cm_matmul_fp8_grouped_async(a, a_scale, b, b_scale, c, offsets, groups, n, k, m, lda, a_scale_ld, ldb, b_scale_ld,
                                         b_group_stride, b_scale_group_stride, ldc, a_format, b_format, c_type, nullptr);
    return rc ? rc : finish_sync(nullptr);
}

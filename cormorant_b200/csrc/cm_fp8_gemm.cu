// cm_fp8_gemm.cu -- matrix products of block-scaled 8-bit floating point operands:
//   c[i][j] = sum over 128-deep blocks t of  a_scale[t][i] * b_scale[j / 128][t] * (a[i][t] . b[j][t])
// dense (cm_matmul_fp8) and grouped by expert (cm_matmul_fp8_grouped: rows offsets[g] ..
// offsets[g+1] - 1 of a and c use b[g]).
//
// A block's product is a fresh accumulator (4 MMAs, 32 deep); epilogue warps take it out of TMEM and
// add it, times token scale * weight scale, to fp32 sums in registers while the next blocks' MMAs run
// into other TMEM buffers.  There are two layouts:
//   few tokens   The weights are the tensor cores' 128-row operand and TN = 16, 32 or 64 tokens their
//                N operand: D[128 weight rows (TMEM lanes)][TN tokens (TMEM columns)].  A single token
//                costs a 16-column tile instead of a 128-row one, the weight scale is one number a
//                block, and an output column is 32 neighbouring lanes: its stores are whole sectors.
//   many (TOK)   Two SMs share a tile of 256 tokens (the M operand) and TN = 128 or 256 weight rows:
//                D[128 tokens a CTA][TN weight rows].  A thread's columns are of one weight block, so a
//                block's scale is one number a thread, and each SM stages half of the N operand.
//                (128 x 128 tiles of one SM, which stage both operands whole and read a scale a
//                column, took 19.8 us at 300 x 4096 x 4096, and 256 x 128 tiles of two 14.7.)
// What bounds it: one token is the weights' HBM read and the launch (4096 x 4096: 7.4 us).  Middle
// sizes are whole waves of tiles whose blocks take 0.19 to 0.3 us against 0.12 to 0.15 us of MMAs
// measured alone: accumulators change hands, and an SM takes its operands from L2 at up to 100 KB a
// microsecond.  8192 x 4096 x 11008 (335 us, 2.2 PFLOP/s; 390 us in a long run, at the clocks of the
// power limit) is the exchange of the two accumulators that TMEM holds: a block of 0.28 us of MMAs
// takes 0.38 to 0.42 us.  Accumulators handed over in halves (353 us) and blocks fetched into a second
// set of registers while the one before is added (in 256 x 128 tiles: 396 -> 489 us) were slower.
//
// Warps: 0 TMA producer, 1 MMA issuer (of the pair's leader), 2-3 token scales (global memory ->
// times the weight scale -> a ring in shared memory), 4.. epilogue.  Every mbarrier wait is bounded
// by %globaltimer, as in cm_gemm.cu.
#include <algorithm>
#include <atomic>

#include "cm_fp8.cuh"
#include "cm_tcgen05.cuh"

namespace cm {
namespace {

constexpr uint32_t kMaxGroups = 1024;

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

// What the kernel needs beside its two tensor maps.
struct KArgs {
    const float* as;
    const float* bs;
    void* c;
    const int32_t* offsets;
    uint64_t a_lds, b_lds, bs_gs, ldc;
    uint32_t groups, n, m, c_type, kb, ksteps, tiles_m, tiles_t, total, idesc, group_step;
    FastDiv fd_m;
    int* status;
    uint64_t timeout_ns;
};

template <int TN>
struct F8Cfg {
    static constexpr bool TOK = TN >= 128;                    // token rows are the M operand; such tiles take a pair of SMs
    static constexpr int CG = TOK ? 2 : 1;
    // Eight epilogue warps.  TOK: four for each half of the columns.  Else the K blocks go to the two
    // fours in turn, which add their sums at the end of a tile (a block costs a warp some 500 cycles of
    // waiting whatever its width).
    static constexpr int EPI_WARPS = 8;
    static constexpr int TURNS = TOK ? 1 : 2;
    static constexpr int COLS = TN / 2 * TURNS;              // accumulator columns of an epilogue warp
    static constexpr int THREADS = 128 + 32 * EPI_WARPS;
    static constexpr uint32_t TOKENS = TOK ? 128 * CG : TN;  // token rows of a tile
    static constexpr uint32_t WEIGHTS = TOK ? TN : 128 * CG; // weight rows of a tile
    static constexpr bool SPLIT_REGS = TN == 256;            // 128 sums a thread: registers move to the epilogue warps
    static constexpr int A_TILE = 128 * 128, B_TILE = TN / CG * 128;
    static constexpr int STAGE = A_TILE + B_TILE;
    static constexpr int STAGES = TN == 256 ? 6 : TN == 128 ? 8 : TN == 64 ? 7 : TN == 32 ? 9 : 10;
    static constexpr int NBUF = TN == 256 ? 2 : 4;           // accumulators in TMEM
    // scale ring: K blocks (not TOK: in groups of 4 with a barrier each way)
    static constexpr int SLOTS = TOK ? 2 * NBUF + 4 : 8;
    static constexpr int GROUPS = SLOTS / 4;
    static constexpr uint32_t TMEM_COLS = NBUF * TN;
    static constexpr int TABLES = (2 * (kMaxGroups + 1) * 4 + 15) / 16 * 16;
    static_assert((STAGES * STAGE + SLOTS * TN * 4) % 16 == 0, "what follows the ring is 16-byte aligned");
    // output staging, 32 rows x 64 bytes a warp; or the sums that the two fours exchange
    static constexpr int OUT = TOK ? EPI_WARPS * 2048 : TN * 128 * 4;
    static constexpr int SMEM = 1024 + STAGES * STAGE + SLOTS * TN * 4 + 512 + TABLES + OUT;
    static_assert(SMEM <= 232448 && 2 * SMEM > 232448, "one CTA an SM");
    static_assert(TOK || TN * 512 <= STAGES * STAGE, "partial sums of a split tile fit the stages");
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
// the same, completing on the pair leader's barrier (bar is a shared::cluster address)
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
        "l"((uint64_t)map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

template <int CG>
__device__ __forceinline__ void umma_f8(uint32_t d_tmem, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    if (CG == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "setp.ne.b32 p, %4, 0;\n\t"
            "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
            "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
            : "memory");
}

// 16, 32 or 2 x 32 accumulator columns of this warp's 32 lanes.  A load writes its registers until its
// wait, so the two are one statement: nothing that the compiler makes of the code around it -- a copy, a
// spill -- can come between them and read a register too early.
#define CM_O(i) "=r"(r[i])
#define CM_O0(i) "=&r"(r0[i])
#define CM_O1(i) "=r"(r1[i])
#define CM_IO1(i) "+&r"(r1[i])
#define CM_ACC(i) "+&f"(acc[i])
#define CM_8(X, o) X(o), X(o + 1), X(o + 2), X(o + 3), X(o + 4), X(o + 5), X(o + 6), X(o + 7)
#define CM_32(X) CM_8(X, 0), CM_8(X, 8), CM_8(X, 16), CM_8(X, 24)
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : CM_8(CM_O, 0), CM_8(CM_O, 8)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_get(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : CM_32(CM_O)
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void tmem_get(uint32_t taddr0, uint32_t taddr1, uint32_t (&r0)[32], uint32_t (&r1)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : CM_32(CM_O0), CM_32(CM_O1)
        : "r"(taddr0), "r"(taddr1)
        : "memory");
}
// acc += r1 * one between the load of r0 and the load of the next r1
__device__ __forceinline__ void tmem_get_adding(uint32_t taddr0, uint32_t taddr1, uint32_t (&r0)[32], uint32_t (&r1)[32], float* acc, float one) {
#define CM_FMA(a, r) "fma.rn.f32 %" #a ", %" #r ", %98, %" #a ";\n\t"
#define CM_FMA4(a, b, c, d, p, q, r, s) CM_FMA(a, p) CM_FMA(b, q) CM_FMA(c, r) CM_FMA(d, s)
    asm volatile(
        "{\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%96];\n\t"
        CM_FMA4(64, 65, 66, 67, 32, 33, 34, 35)
        CM_FMA4(68, 69, 70, 71, 36, 37, 38, 39)
        CM_FMA4(72, 73, 74, 75, 40, 41, 42, 43)
        CM_FMA4(76, 77, 78, 79, 44, 45, 46, 47)
        CM_FMA4(80, 81, 82, 83, 48, 49, 50, 51)
        CM_FMA4(84, 85, 86, 87, 52, 53, 54, 55)
        CM_FMA4(88, 89, 90, 91, 56, 57, 58, 59)
        CM_FMA4(92, 93, 94, 95, 60, 61, 62, 63)
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"
        "%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, "
        "%48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%97];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t}"
        : CM_32(CM_O0), CM_32(CM_IO1), CM_32(CM_ACC)
        : "r"(taddr0), "r"(taddr1), "f"(one)
        : "memory");
#undef CM_FMA
#undef CM_FMA4
}
#undef CM_O
#undef CM_O0
#undef CM_O1
#undef CM_IO1
#undef CM_ACC
#undef CM_8
#undef CM_32

// One thread of a converged warp.  The compiler knows that a branch on it holds one thread and keeps
// the operands of the MMA and copy instructions in uniform registers; behind `lane == 0` it moves
// them there for every instruction (measured: 4 MMAs and their commit take 157 cycles to issue
// behind an elected branch, 817 behind a comparison, whatever the tile's width).
__device__ __forceinline__ bool elect_one() {
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "elect.sync _|p, 0xffffffff;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(r));
    return r != 0;
}

// An arrival by the lanes with `on`, without a branch; on a barrier of this CTA, or of the cluster
// (a shared::cluster address).
__device__ __forceinline__ void arrive_if(bool on, uint32_t bar) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(bar), "r"((uint32_t)on)
                 : "memory");
}
__device__ __forceinline__ void arrive_cluster_if(bool on, uint32_t bar) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %1, 0;\n\t@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n\t}" ::"r"(bar), "r"((uint32_t)on)
                 : "memory");
}

// Whether the phase is complete, without waiting (try_wait may hold the thread for a while).
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}

// 16 bytes of another CTA's shared memory (of this cluster; between two cluster barriers)
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// a barrier of the epilogue warps alone
template <int THREADS>
__device__ __forceinline__ void epilogue_sync() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }

struct TileF8 {
    uint32_t m0;             // first weight row
    uint32_t row0, row1;     // token rows row0 .. row1 - 1, at most a tile's used
    uint32_t group;
};

// Tile t: groups in order; within a group, bands of kBand token tiles are walked weight tile by
// weight tile, so that the tiles in flight share a few operand panels in L2.
constexpr uint32_t kBand = 8;

template <typename C>
__device__ __forceinline__ TileF8 decode_tile(const KArgs& g, const uint32_t* first, const uint32_t* ends, uint32_t t) {
    uint32_t local = t, tt = g.tiles_t, row0 = 0, row1 = g.n, group = 0;
    if (g.offsets) {
        const uint32_t q = g.fd_m.div(t);                     // token tile over all groups
        uint32_t lo = 0, hi = g.groups;                        // the last group with first[] <= q
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            if (first[mid] <= q) lo = mid;
            else hi = mid;
        }
        group = lo;
        tt = first[lo + 1] - first[lo];
        local = t - first[lo] * g.tiles_m;
        row0 = ends[lo];
        row1 = ends[lo + 1];
    }
    const uint32_t per = kBand * g.tiles_m, band = local / per, r = local - band * per;
    const uint32_t size = min(kBand, tt - band * kBand), mt = r / size;
    TileF8 c;
    c.m0 = mt * C::WEIGHTS;
    c.row0 = row0 + (band * kBand + r - mt * size) * C::TOKENS;
    c.row1 = row1;
    c.group = group;
    return c;
}

template <typename T, int COLS>
__device__ __forceinline__ void store_cols(const KArgs& g, const TileF8& tc, uint32_t col0, uint32_t mrow, const float* acc) {
    if (mrow >= g.m) return;
    const uint32_t tok = tc.row0 + col0;
    T* p = (T*)g.c + (uint64_t)tok * g.ldc + mrow;
    const uint32_t live = tc.row1 > tok ? tc.row1 - tok : 0u;
#pragma unroll
    for (uint32_t j = 0; j < COLS; ++j) {
        if (j < live) from_f32(acc[j], *p);
        p += g.ldc;
    }
}

// 16 / sizeof(T) values in 16 bytes
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v);
template <>
__device__ __forceinline__ uint4 pack16<float>(const float* v) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <>
__device__ __forceinline__ uint4 pack16<__nv_bfloat16>(const float* v) {
    union {
        __nv_bfloat162 h[4];
        uint4 u;
    } o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.h[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
    return o.u;
}
template <>
__device__ __forceinline__ uint4 pack16<__half>(const float* v) {
    union {
        __half2 h[4];
        uint4 u;
    } o;
#pragma unroll
    for (int j = 0; j < 4; ++j) o.h[j] = __floats2half2_rn(v[2 * j], v[2 * j + 1]);
    return o.u;
}
template <>
__device__ __forceinline__ uint4 pack16<int16_t>(const float* v) {
    union {
        int16_t h[8];
        uint4 u;
    } o;
#pragma unroll
    for (int j = 0; j < 8; ++j) from_f32(v[j], o.h[j]);
    return o.u;
}

// TOK: 32 token rows of 128 columns, a row a lane.  64 bytes of each row go through shared memory
// at a time (16-byte pieces XOR-swizzled over the bank groups), so that a store covers whole
// 64-byte runs of eight rows instead of 16 bytes of 32.  The code is passed through once a tile, at
// the pace of instruction fetches, so what counts is its length.
template <typename T, int COLS>
__device__ __forceinline__ void store_rows(const KArgs& g, uint32_t row0, uint32_t row1, uint32_t mcol, uint8_t* stage, uint32_t lane,
                                           const float (&acc)[COLS]) {
    constexpr uint32_t W = 64 / sizeof(T), P = W / 4;          // columns of a pass and of a piece
    const bool vec = (uintptr_t)g.c % 16 == 0 && g.ldc * sizeof(T) % 16 == 0;
    const uint32_t rows = row1 > row0 ? row1 - row0 : 0u, sw = (lane >> 1) & 3u, rsw = (lane >> 3) & 3u;
    uint8_t* in = stage + lane * 64;                           // this lane's row
    const uint8_t* out = stage + lane / 4 * 64 + ((lane ^ rsw) & 3u) * 16;   // piece lane % 4 of rows lane / 4, + 8, ..
    T* d = (T*)g.c + (uint64_t)(row0 + lane / 4) * g.ldc + mcol + lane % 4 * P;
    const uint64_t down = 8 * g.ldc;
#pragma unroll
    for (uint32_t c0 = 0; c0 < COLS; c0 += W) {
        if (mcol + c0 >= g.m) break;                            // the whole warp
        __syncwarp();
#pragma unroll
        for (uint32_t p = 0; p < 4; ++p) *reinterpret_cast<uint4*>(in + ((p ^ sw) & 3u) * 16) = pack16<T>(acc + c0 + p * P);
        __syncwarp();
        if (vec && mcol + c0 + W <= g.m) {
            T* e = d + c0;
#pragma unroll
            for (uint32_t i = 0; i < 4; ++i) {
                const uint4 v = *reinterpret_cast<const uint4*>(out + i * 512);
                if (8 * i + lane / 4 < rows) *reinterpret_cast<uint4*>(e) = v;
                e += down;
            }
        } else {
            // rows at any pitch, or the last columns: an element a lane, so that a store covers whole
            // runs all the same
#pragma unroll 8
            for (uint32_t r0 = 0; r0 < W; ++r0) {               // 32 / W rows at a time
                const uint32_t r = r0 * (32 / W) + lane / W, e = lane % W;
                const T v = *reinterpret_cast<const T*>(stage + r * 64 + ((e / P ^ (r >> 1)) & 3u) * 16 + e % P * sizeof(T));
                if (r < rows && mcol + c0 + e < g.m) ((T*)g.c)[(uint64_t)(row0 + r) * g.ldc + mcol + c0 + e] = v;
            }
        }
    }
}

__device__ __forceinline__ void store_one(const KArgs& g, uint64_t i, float v) {
    switch (g.c_type) {
        case CM_T_Q88: from_f32(v, ((int16_t*)g.c)[i]); break;
        case CM_T_F32: from_f32(v, ((float*)g.c)[i]); break;
        case CM_T_F16: from_f32(v, ((__half*)g.c)[i]); break;
        default: from_f32(v, ((__nv_bfloat16*)g.c)[i]); break;
    }
}

// The token scales of one (tile, K block), as a scale warp holds them on their way from global
// memory: the loads of a group of four are issued while the group before it waits for room.
template <int TN>
struct ScaleRegs {
    float v[TN < 32 ? 1 : TN / 32];
    float sb;
};

// KS: the CTAs of a cluster share one tile, each a contiguous part of its K blocks, and add their
// sums through distributed shared memory, in the order of their ranks.
template <int TN, bool KS>
__global__ void __launch_bounds__(F8Cfg<TN>::THREADS, 1)
    gemm_f8_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmT, const KArgs g) {
    using C = F8Cfg<TN>;
    constexpr bool TOK = C::TOK;
    constexpr int CG = C::CG;
    static_assert(TN == 16 || !KS, "only the narrowest tiles split K");
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* smem = (uint8_t*)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    float* ring = (float*)(smem + C::STAGES * C::STAGE);
    uint64_t* bars = (uint64_t*)(ring + C::SLOTS * TN);
    uint64_t* full_b = bars;
    uint64_t* empty_b = full_b + C::STAGES;
    uint64_t* accf_b = empty_b + C::STAGES;
    uint64_t* acce_b = accf_b + C::NBUF;
    uint64_t* sfull_b = acce_b + C::NBUF;
    uint64_t* sempty_b = sfull_b + C::GROUPS;
    uint64_t* done_b = sempty_b + C::GROUPS;
    volatile uint32_t* tmem_slot = (volatile uint32_t*)(done_b + 1);
    volatile int* abort_flag = (volatile int*)(tmem_slot + 1);
    uint32_t* first = (uint32_t*)((uint8_t*)bars + 512);      // grouped: first token tile of each group
    uint32_t* ends = first + kMaxGroups + 1;                   // grouped: offsets, held to 0..n and in order

    const uint32_t warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const uint32_t crank = CG == 2 || KS ? cluster_rank() : 0u;
    uint32_t csize = 1;
    if (KS) asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    const uint32_t rank = CG == 2 ? crank : 0u;
    const bool leader = rank == 0;
    const uint32_t per_tile = CG == 2 ? 2u : csize;            // CTAs of a tile
    const uint32_t cid = blockIdx.x / per_tile, ncl = gridDim.x / per_tile;
    const uint32_t kb0 = KS ? (uint32_t)((uint64_t)g.kb * crank / csize) : 0u;
    const uint32_t kb1 = KS ? (uint32_t)((uint64_t)g.kb * (crank + 1) / csize) : g.kb;
    constexpr uint16_t kPairMask = 0x3;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmW) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"((uint64_t)&tmT) : "memory");
        for (int s = 0; s < C::STAGES; ++s) {
            mbar_init(smem_u32(&full_b[s]), 1);
            mbar_init(smem_u32(&empty_b[s]), 1);
        }
        for (int b = 0; b < C::NBUF; ++b) {
            mbar_init(smem_u32(&accf_b[b]), TOK ? 2 : 1);     // TOK: its MMAs and its scales
            mbar_init(smem_u32(&acce_b[b]), C::EPI_WARPS / C::TURNS * CG);
        }
        for (int s = 0; s < C::GROUPS; ++s) {        // not used by TOK
            mbar_init(smem_u32(&sfull_b[s]), 2);
            mbar_init(smem_u32(&sempty_b[s]), C::EPI_WARPS);
        }
        mbar_init(smem_u32(done_b), 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        if (CG == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)),
                         "r"(C::TMEM_COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_slot)),
                         "r"(C::TMEM_COLS)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
        tc_fence_before();
    }
    // up to here nothing of the kernel before this one is touched
    griddep_wait();
    griddep_launch_dependents();   // all CTAs are resident
    if (g.offsets) {
        // the offsets in one round of loads; then one warp's running maximum of them, held to 0..n, and
        // running sum of the groups' token tiles: whatever the offsets hold, no row outside 0..n-1 is reached
        for (uint32_t i = threadIdx.x; i <= g.groups; i += C::THREADS) ends[i] = (uint32_t)min(max(g.offsets[i], 0), (int)g.n);
        __syncthreads();
        if (warp == 2) {
            uint32_t high = 0, tiles = 0;
            for (uint32_t base = 0; base <= g.groups; base += 32) {
                const uint32_t i = base + lane;
                uint32_t e = i <= g.groups ? ends[i] : 0u;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const uint32_t p = __shfl_up_sync(0xffffffffu, e, o);
                    if (lane >= (uint32_t)o) e = max(e, p);
                }
                e = max(e, high);
                uint32_t before = __shfl_up_sync(0xffffffffu, e, 1);
                if (lane == 0) before = high;
                // tiles of the group that ends at offset i (none ends at offset 0)
                uint32_t cnt = i > 0 ? (e - before + C::TOKENS - 1) / C::TOKENS : 0u;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const uint32_t p = __shfl_up_sync(0xffffffffu, cnt, o);
                    if (lane >= (uint32_t)o) cnt += p;
                }
                if (i <= g.groups) {
                    ends[i] = e;
                    first[i] = tiles + cnt;
                }
                high = __shfl_sync(0xffffffffu, e, 31);
                tiles += __shfl_sync(0xffffffffu, cnt, 31);
            }
        }
    }
    __syncthreads();
    if (CG == 2) cluster_sync_all();      // both CTAs' barriers exist before any remote arrival
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t total = g.offsets ? first[g.groups] * g.tiles_m : g.total;
    const WaitCtl wc{abort_flag, g.status, g.timeout_ns};

    // The first four warps hand registers to the epilogue warps: 168 a thread at launch,
    // 128 x 56 + 256 x 224 = 384 x 168.  A warpgroup's warps execute one and the same instruction for
    // it, so the roles branch after it.
    if (warp < 4) {
        if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        if (warp == 0) {
            if (elect_one()) {
                uint32_t s = 0, phase = 1, it = 0;
                bool ok = true;
                for (uint32_t t = cid; ok && t < total; t += ncl) {
                    const TileF8 tc = decode_tile<C>(g, first, ends, t);
                    for (uint32_t kb = kb0; kb < kb1; ++kb, ++it) {
                        if (!mbar_wait(smem_u32(&empty_b[s]), phase, wc)) { ok = false; break; }
                        const uint32_t st = smem_u32(smem + s * C::STAGE);
                        if (CG == 2) {
                            const uint32_t full = map_to_rank(smem_u32(&full_b[s]), 0);
                            if (leader) mbar_expect_tx(smem_u32(&full_b[s]), 2 * C::STAGE);
                            // each CTA its 128 rows of the M operand and its half of the N operand
                            tma_load_2d_pair(st, &tmT, full, (int)(kb * 128), (int)(tc.row0 + rank * 128));
                            tma_load_3d_pair(st + C::A_TILE, &tmW, full, (int)(kb * 128), (int)(tc.m0 + rank * (TN / CG)), (int)(tc.group * g.group_step));
                        } else {
                            const uint32_t full = smem_u32(&full_b[s]);
                            mbar_expect_tx(full, C::STAGE);
                            tma_load_3d(st, &tmW, full, (int)(kb * 128), (int)tc.m0, (int)(tc.group * g.group_step));
                            tma_load_2d(st + C::A_TILE, &tmT, full, (int)(kb * 128), (int)tc.row0);
                        }
                        if (++s == C::STAGES) { s = 0; phase ^= 1; }
                    }
                }
                if (*abort_flag && leader) {
                    // let copies already in flight land before the CTA exits
                    const uint32_t from = it > C::STAGES ? it - C::STAGES : 0u;
                    volatile int never = 0;
                    WaitCtl drain{&never, g.status, g.timeout_ns};
                    for (uint32_t k = from; k < it; ++k) mbar_wait(smem_u32(&full_b[k % C::STAGES]), (k / C::STAGES) & 1u, drain);
                }
            }
        } else if (warp == 1) {
            if (leader && elect_one()) {
                // What a block's MMAs need is worked out before the wait for its accumulator, which is the
                // short side of the loop: descriptors advance by a stage, barriers by their address.
                constexpr uint32_t DSTEP = C::STAGE >> 4;
                const uint64_t da0 = sdesc(smem_u32(smem)), db0 = sdesc(smem_u32(smem + C::A_TILE));
                uint32_t s = 0, phase = 0, buf = 0, bphase = 1;
                bool ok = true;
                for (uint32_t t = cid; ok && t < total; t += ncl) {
                    for (uint32_t steps = g.ksteps - kb0 * 4, left = kb1 - kb0; left; --left, steps -= 4) {
                        const uint64_t da = da0 + s * DSTEP, db = db0 + s * DSTEP;
                        const uint32_t d = tmem + buf * TN, full = smem_u32(&full_b[s]), empty = smem_u32(&empty_b[s]);
                        const uint32_t accf = smem_u32(&accf_b[buf]), acce = smem_u32(&acce_b[buf]);
                        if (!mbar_test(full, phase) && !mbar_wait(full, phase, wc)) { ok = false; break; }
                        if (!mbar_test(acce, bphase) && !mbar_wait(acce, bphase, wc)) { ok = false; break; }
                        tc_fence_after();
                        if (steps >= 4) {
#pragma unroll
                            for (uint32_t kk = 0; kk < 4; ++kk) umma_f8<CG>(d, da + 2 * kk, db + 2 * kk, g.idesc, kk != 0);
                        } else {                        // the last block's 32-deep steps with any column below k
                            for (uint32_t kk = 0; kk < steps; ++kk) umma_f8<CG>(d, da + 2 * kk, db + 2 * kk, g.idesc, kk != 0);
                        }
                        if (CG == 2) {
                            umma_commit_pair(accf, kPairMask);
                            umma_commit_pair(empty, kPairMask);
                        } else {
                            umma_commit(accf);
                            umma_commit(empty);
                        }
                        if (++s == C::STAGES) { s = 0; phase ^= 1; }
                        if (++buf == C::NBUF) { buf = 0; bphase ^= 1; }
                    }
                }
                // every MMA issued by this thread has completed once `done` fires
                if (CG == 2) umma_commit_pair(smem_u32(done_b), 0x1);
                else umma_commit(smem_u32(done_b));
                volatile int never = 0;
                WaitCtl drain{&never, g.status, g.timeout_ns};
                mbar_wait(smem_u32(done_b), 0, drain);
            }
        } else {
            if constexpr (TOK) {
                // Scale warps: K blocks are counted over all tiles of this CTA; warp 2 has the even ones,
                // warp 3 the odd ones.  A block's barrier
                // completes with its MMAs and with its scales' arrival here, so the epilogue waits once.
                // When block i - NBUF is complete, its MMAs were issued, so every epilogue warp has given
                // back the accumulator of block i - 2 NBUF and has read that block's scales: block i + 4
                // may take their place in the ring.
                const uint32_t par = warp - 2;
                uint32_t t = cid, kb = 0, wblocks = 0;       // the next block to load
                TileF8 tc{};
                const float* sbp = nullptr;
                bool fresh = true;
                float sa[2][4], sb[2][2];                    // two blocks on their way
                auto step = [&](uint32_t by) {
                    for (uint32_t i = 0; i < by; ++i)
                        if (++kb == g.kb) { kb = 0; t += ncl; fresh = true; }
                };
                auto load = [&](float (&a4)[4], float (&b2)[2]) {
                    if (t >= total) return;
                    if (fresh) {
                        tc = decode_tile<C>(g, first, ends, t);
                        tc.row0 += rank * 128;
                        wblocks = (g.m - tc.m0 + 127) / 128;       // of which a tile has two at most
                        sbp = g.bs + tc.group * g.bs_gs + (uint64_t)(tc.m0 / 128) * g.b_lds;
                        fresh = false;
                    }
                    b2[0] = __ldg(sbp + kb);
                    b2[1] = TN == 256 && wblocks > 1 ? __ldg(sbp + g.b_lds + kb) : 0.0f;
                    const float* a = g.as + (uint64_t)kb * g.a_lds + tc.row0;
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) a4[q] = tc.row0 + lane + 32 * q < tc.row1 ? __ldg(a + lane + 32 * q) : 0.0f;
                    step(2);
                };
                uint32_t place = par;                        // in the ring, of the next block stored
                auto store = [&](const float (&a4)[4], const float (&b2)[2]) {
                    float* dst = ring + place * TN;
                    place += 2;
                    if (place >= C::SLOTS) place -= C::SLOTS;
#pragma unroll
                    for (uint32_t q = 0; q < 4; ++q) {
                        dst[lane + 32 * q] = a4[q] * b2[0];
                        if (TN == 256) dst[128 + lane + 32 * q] = a4[q] * b2[1];
                    }
                };
                const uint64_t items = (uint64_t)(cid < total ? (total - cid + ncl - 1) / ncl : 0u) * g.kb;
                uint32_t buf = par, phase = 1;               // of block i - NBUF; there is none before the first
                step(par);
                load(sa[0], sb[0]);
                load(sa[1], sb[1]);
                if (par < items) store(sa[0], sb[0]);
                load(sa[0], sb[0]);
                if (par + 2 < items) store(sa[1], sb[1]);
                for (uint64_t i = par; i < items; i += 2) {
                    const uint32_t accf = smem_u32(&accf_b[buf]);
                    if (i >= C::NBUF && !__all_sync(0xffffffffu, mbar_wait(accf, phase, wc))) break;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(accf);
                    if (i + 4 < items) store(sa[0], sb[0]);
                    load(sa[0], sb[0]);
                    buf += 2;
                    if (buf >= C::NBUF) { buf -= C::NBUF; phase ^= 1; }
                }
            } else {
                // Scale warps: of a tile's K blocks, in groups of four, 2 takes the even ones and 3 the odd
                // ones; the next group's loads are in flight while this one waits for room.
                const uint32_t nkb = kb1 - kb0, per = (nkb + 3) / 4;
                ScaleRegs<TN> regs[2];
                bool have[2] = {false, false};
                uint32_t t = cid, at = 0;            // the next group: tile and place in it
                TileF8 tc{};
                const float* sbp = nullptr;
                auto fetch = [&]() {
                    if (t >= total) return;
                    if (at == 0) {
                        tc = decode_tile<C>(g, first, ends, t);
                        sbp = g.bs + tc.group * g.bs_gs + (uint64_t)(tc.m0 / 128) * g.b_lds;
                    }
#pragma unroll
                    for (uint32_t p = 0; p < 2; ++p) {
                        const uint32_t i = at * 4 + 2 * p + warp - 2, kb = kb0 + i;
                        have[p] = i < nkb;
                        if (!have[p]) continue;
                        ScaleRegs<TN>& r = regs[p];
                        r.sb = __ldg(sbp + kb);
                        const float* a = g.as + (uint64_t)kb * g.a_lds + tc.row0;
#pragma unroll
                        for (uint32_t q = 0; q < sizeof(r.v) / 4; ++q) {
                            const uint32_t j = lane + 32 * q;
                            r.v[q] = j < TN && tc.row0 + j < tc.row1 ? __ldg(a + j) : 0.0f;
                        }
                    }
                    if (++at == per) { at = 0; t += ncl; }
                };
                const uint64_t groups = (uint64_t)(cid < total ? (total - cid + ncl - 1) / ncl : 0u) * per;
                fetch();
                for (uint64_t grp = 0; grp < groups; ++grp) {
                    const uint32_t gs = (uint32_t)grp % C::GROUPS, use = (uint32_t)(grp / C::GROUPS);
                    if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&sempty_b[gs]), (use & 1u) ^ 1u, wc))) break;
#pragma unroll
                    for (uint32_t p = 0; p < 2; ++p) {
                        float* dst = ring + (gs * 4 + 2 * p + warp - 2) * TN;
                        if (!have[p]) continue;
#pragma unroll
                        for (uint32_t q = 0; q < sizeof(regs[p].v) / 4; ++q) {
                            const uint32_t j = lane + 32 * q;
                            if (j < TN) dst[j] = regs[p].v[q] * regs[p].sb;
                        }
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sfull_b[gs]));
                    fetch();
                }
            }
        }
    } else {
        if constexpr (C::SPLIT_REGS) asm volatile("setmaxnreg.inc.sync.aligned.u32 224;");
        if constexpr (TOK) {
            // A lane is a token row and the warp's 128 columns are one weight block, so a block's scale is
            // one number a thread.
            //
            // 128 sums leave registers for half of a block's columns: the second half is fetched as the
            // first is added, and the accumulator is given back when it is here, before it is added.
            // 64 sums take a block's columns at once.
            constexpr int CW = 32;
            const uint32_t quarter = warp & 3u, half = (warp - 4) / 4;
            const uint32_t acce0 = map_to_rank(smem_u32(&acce_b[0]), 0), accf0 = smem_u32(&accf_b[0]);
            const uint32_t d0 = tmem + half * C::COLS + (quarter << 21);
            const float* sc = ring + half * (TN / 256 * 128) + quarter * 32 + lane;
            uint32_t buf = 0, bphase = 0, slot = 0;
            bool ok = true;
            for (uint32_t t = cid; t < total; t += ncl) {
                const TileF8 tc = decode_tile<C>(g, first, ends, t);
                float acc[C::COLS];
#pragma unroll
                for (int j = 0; j < C::COLS; ++j) acc[j] = 0.0f;
                uint32_t r0[CW], r1[CW];
                float one = 0.0f;
                auto begin = [&]() {                 // the block's accumulator and scales are there: fetch its first 64 columns
                    ok = __all_sync(0xffffffffu, mbar_wait(accf0 + 8 * buf, bphase, wc));
                    if (!ok) return;
                    tc_fence_after();
                    one = sc[slot * TN];
                    tmem_get(d0 + buf * TN, d0 + buf * TN + CW, r0, r1);
                };
                begin();
                if (!ok) break;
                auto add = [&](int c, const uint32_t (&r)[CW]) {
#pragma unroll
                    for (int j = 0; j < CW; ++j) acc[c * CW + j] = fmaf(__uint_as_float(r[j]), one, acc[c * CW + j]);
                };
                for (uint32_t left = g.kb; left; --left) {
                    const uint32_t d = d0 + buf * TN, acce = acce0 + 8 * buf;
                    if constexpr (TN == 256) {
                        add(0, r0);
                        tmem_get_adding(d + 2 * CW, d + 3 * CW, r0, r1, acc + CW, one);
                    }
                    tc_fence_before();
                    __syncwarp();
                    arrive_cluster_if(lane == 0, acce);      // the accumulator's columns are in registers
                    add(TN == 256 ? 2 : 0, r0);
                    add(TN == 256 ? 3 : 1, r1);
                    buf = (buf + 1u) % C::NBUF;
                    if (buf == 0) bphase ^= 1u;
                    slot = (slot + 1u) % C::SLOTS;
                    if (left > 1) begin();
                    if (!ok) break;
                }
                if (!ok) break;
                uint8_t* stage = (uint8_t*)bars + 512 + C::TABLES + (warp - 4) * 2048;
                const uint32_t row0 = tc.row0 + rank * 128 + quarter * 32, mcol = tc.m0 + half * C::COLS;
                switch (g.c_type) {
                    case CM_T_Q88: store_rows<int16_t, C::COLS>(g, row0, tc.row1, mcol, stage, lane, acc); break;
                    case CM_T_F32: store_rows<float, C::COLS>(g, row0, tc.row1, mcol, stage, lane, acc); break;
                    case CM_T_F16: store_rows<__half, C::COLS>(g, row0, tc.row1, mcol, stage, lane, acc); break;
                    default: store_rows<__nv_bfloat16, C::COLS>(g, row0, tc.row1, mcol, stage, lane, acc); break;
                }
            }
        } else {
            const uint32_t quarter = warp & 3u, turn = (warp - 4) / 4;
            const uint32_t nkb = kb1 - kb0;
            uint32_t item = 0, grp = 0;          // K blocks and groups of scales before this tile
            bool ok = true;
            constexpr int CW = C::COLS < 32 ? 16 : 32, NC = C::COLS / CW;
            static_assert(NC == 1 || NC == 2, "chunks of a warp's columns");
            for (uint32_t t = cid; t < total; t += ncl, item += nkb) {
                const TileF8 tc = decode_tile<C>(g, first, ends, t);
                float acc[C::COLS];
#pragma unroll
                for (int j = 0; j < C::COLS; ++j) acc[j] = 0.0f;
                uint32_t r0[CW], r1[CW];
                for (uint32_t g4 = 0; ok && g4 < nkb; g4 += 4, ++grp) {
                    const uint32_t gs = grp % C::GROUPS;
                    ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sfull_b[gs]), (grp / C::GROUPS) & 1u, wc));
                    for (uint32_t q = turn; ok && q < 4 && g4 + q < nkb; q += C::TURNS) {
                        const uint32_t it = item + g4 + q, buf = it % C::NBUF;
                        ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&accf_b[buf]), (it / C::NBUF) & 1u, wc));
                        if (!ok) break;
                        tc_fence_after();
                        const uint32_t d = tmem + buf * TN + (quarter << 21);
                        if constexpr (NC > 1) tmem_get(d, d + CW, r0, r1);
                        else tmem_get(d, r0);
                        tc_fence_before();
                        __syncwarp();
                        arrive_if(lane == 0, smem_u32(&acce_b[buf]));
                        const float* sc = ring + (gs * 4 + q) * TN;      // a scale a column
#pragma unroll
                        for (int j = 0; j < C::COLS; j += 4) {
                            const float4 s4 = *reinterpret_cast<const float4*>(sc + j);
                            const uint32_t* r = j < CW ? r0 + j : r1 + (j - CW);
                            acc[j] = fmaf(__uint_as_float(r[0]), s4.x, acc[j]);
                            acc[j + 1] = fmaf(__uint_as_float(r[1]), s4.y, acc[j + 1]);
                            acc[j + 2] = fmaf(__uint_as_float(r[2]), s4.z, acc[j + 2]);
                            acc[j + 3] = fmaf(__uint_as_float(r[3]), s4.w, acc[j + 3]);
                        }
                    }
                    __syncwarp();
                    arrive_if(lane == 0, smem_u32(&sempty_b[gs]));
                }
                // each four finishes half of the columns, adding what the other one summed of them
                constexpr int H = TN / 2;
                float* mine = (float*)((uint8_t*)bars + 512 + C::TABLES) + quarter * 32 + lane;
#pragma unroll
                for (int j = 0; j < H; ++j) mine[(turn * H + j) * 128] = turn ? acc[j] : acc[H + j];
                epilogue_sync<C::EPI_WARPS * 32>();
#pragma unroll
                for (int j = 0; j < H; ++j) acc[j] = (turn ? acc[H + j] : acc[j]) + mine[((turn ^ 1u) * H + j) * 128];
                if (t + ncl < total) epilogue_sync<C::EPI_WARPS * 32>();      // read before the next tile writes
                const uint32_t own0 = turn * H;
                if (KS) {
                    // this CTA's part, [column][weight row], over the stages: their copies have landed and
                    // the MMAs that read them are complete (this tile is the CTA's only one)
                    float* part = (float*)smem + quarter * 32 + lane;
#pragma unroll
                    for (int j = 0; j < H; ++j) part[(own0 + j) * 128] = acc[j];
                } else if (ok) {
                    const uint32_t mrow = tc.m0 + quarter * 32 + lane;
                    switch (g.c_type) {
                        case CM_T_Q88: store_cols<int16_t, H>(g, tc, own0, mrow, acc); break;
                        case CM_T_F32: store_cols<float, H>(g, tc, own0, mrow, acc); break;
                        case CM_T_F16: store_cols<__half, H>(g, tc, own0, mrow, acc); break;
                        default: store_cols<__nv_bfloat16, H>(g, tc, own0, mrow, acc); break;
                    }
                }
            }
        }
    }
    __syncthreads();
    if (KS) {
        __syncwarp();
        cluster_sync_all();                 // every CTA's part is written
        if (cid < total) {
            const TileF8 tc = decode_tile<C>(g, first, ends, cid);
            const uint32_t lo = TN * crank / csize, hi = TN * (crank + 1) / csize;
            const uint32_t base = smem_u32(smem);
            for (uint32_t e = threadIdx.x; e < (hi - lo) * 32; e += C::THREADS) {
                const uint32_t col = lo + e / 32, r = e % 32 * 4;
                if (tc.row0 + col >= tc.row1 || tc.m0 + r >= g.m) continue;
                float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (uint32_t p = 0; p < csize; p += 2) {          // 2, 4 or 8 parts, in order
                    const float4 x = ld_cluster4(map_to_rank(base + (col * 128 + r) * 4, p));
                    const float4 y = ld_cluster4(map_to_rank(base + (col * 128 + r) * 4, p + 1));
                    v.x = v.x + x.x + y.x;
                    v.y = v.y + x.y + y.y;
                    v.z = v.z + x.z + y.z;
                    v.w = v.w + x.w + y.w;
                }
                const uint64_t i = (uint64_t)(tc.row0 + col) * g.ldc + tc.m0 + r;
                const uint32_t live = g.m - tc.m0 - r;
                store_one(g, i, v.x);
                if (live > 1) store_one(g, i + 1, v.y);
                if (live > 2) store_one(g, i + 2, v.z);
                if (live > 3) store_one(g, i + 3, v.w);
            }
        }
    }
    // CTAs of a cluster use each other's shared memory and barriers until here
    if (CG == 2 || KS) {
        __syncwarp();
        cluster_sync_all();
    }
    if (warp == 1) {
        tc_fence_after();
        if (CG == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(C::TMEM_COLS) : "memory");
    }
}

// Rows of 8-bit values that do not start on 16-byte boundaries, copied to rows that do.  Each
// thread makes 16 bytes from the five aligned words that hold them (words without a byte of the
// row are not read).
__global__ void __launch_bounds__(256) align_rows_kernel(const uint8_t* __restrict__ src, uint64_t ld, uint64_t gs, uint32_t rows,
                                                         uint32_t cols, uint8_t* __restrict__ dst, uint64_t dst_ld, uint64_t total) {
    griddep_wait();
    const uint32_t chunks = (uint32_t)(dst_ld / 16);
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (uint64_t)gridDim.x * 256) {
        const uint64_t row = e / chunks;
        const uint32_t c0 = (uint32_t)(e - row * chunks) * 16;
        const uint64_t z = row / rows, r = row - z * rows;
        const uint8_t* p = src + z * gs + r * ld + c0;
        const uint32_t n = min(16u, cols - c0), shift = (uint32_t)((uintptr_t)p & 3u);
        const uint32_t* w = (const uint32_t*)(p - shift);
        uint32_t v[5];
#pragma unroll
        for (uint32_t i = 0; i < 5; ++i) v[i] = 4 * i < n + shift ? w[i] : 0u;
        uint4 o;
        o.x = __funnelshift_r(v[0], v[1], 8 * shift);
        o.y = __funnelshift_r(v[1], v[2], 8 * shift);
        o.z = __funnelshift_r(v[2], v[3], 8 * shift);
        o.w = __funnelshift_r(v[3], v[4], 8 * shift);
        *(uint4*)(dst + row * dst_ld + c0) = o;
    }
}

// c = 0 (k = 0): the rows of the groups, or all of them.
__global__ void __launch_bounds__(256) zero_rows_kernel(const KArgs g, uint64_t total) {
    griddep_wait();
    uint32_t lo = 0, hi = g.n;
    if (g.offsets) {
        // the running maximum ends at the largest offset; the first one opens the range
        lo = (uint32_t)min(max(g.offsets[0], 0), (int)g.n);
        hi = lo;
        for (uint32_t i = 1; i <= g.groups; ++i) hi = max(hi, (uint32_t)min(max(g.offsets[i], 0), (int)g.n));
    }
    for (uint64_t e = (uint64_t)blockIdx.x * 256 + threadIdx.x; e < total; e += (uint64_t)gridDim.x * 256) {
        const uint64_t row = e / g.m;
        if (row >= lo && row < hi) store_one(g, row * g.ldc + (e - row * g.m), 0.0f);
    }
}

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

int make_map(CUtensorMap* map, const uint8_t* base, uint32_t k, uint64_t ld, uint32_t rows, uint32_t groups, uint64_t gs, uint32_t box_rows,
             uint32_t dims) {
    EncodeTiledFn enc = encode_fn();
    if (!enc) return set_error(CM_ECUDA, "cuTensorMapEncodeTiled unavailable");
    const cuuint64_t size[3] = {k, rows, groups};
    const cuuint64_t strides[2] = {ld, gs};
    const cuuint32_t box[3] = {128, box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, dims, (void*)base, size, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? CM_OK : set_error(CM_ECUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
}

// Clusters of `size` CTAs of this kernel that the GPU holds at once.
template <int TN, bool KS>
int resident_clusters(const Context* cx, uint32_t size, int* out) {
    static std::atomic<int> known[16][9] = {};      // by device and size (function attributes are a device's own); first calls may come from several threads
    const int dev = cx->device < 16 ? cx->device : 15;
    int n = dev == 15 ? 0 : known[dev][size].load();
    if (!n) {
        const auto kern = gemm_f8_kernel<TN, KS>;
        cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, F8Cfg<TN>::SMEM);
        if (e != cudaSuccess) return cuda_error(e, "cudaFuncSetAttribute(gemm_f8)");
        n = cx->sm_count / (int)size;
        if (size > 1) {
            cudaLaunchConfig_t q{};
            q.gridDim = dim3(size * n);
            q.blockDim = dim3(F8Cfg<TN>::THREADS);
            q.dynamicSmemBytes = F8Cfg<TN>::SMEM;
            cudaLaunchAttribute at{};
            at.id = cudaLaunchAttributeClusterDimension;
            at.val.clusterDim.x = size; at.val.clusterDim.y = 1; at.val.clusterDim.z = 1;
            q.attrs = &at; q.numAttrs = 1;
            int r = 0;
            if (cudaOccupancyMaxActiveClusters(&r, kern, &q) == cudaSuccess && r > 0) n = std::min(n, r);
            cudaGetLastError();
        }
        known[dev][size].store(n);
    }
    *out = n;
    return CM_OK;
}

template <int TN, bool KS>
int launch_tiles(const Context* cx, const CUtensorMap& tw, const CUtensorMap& tt, const KArgs& g, uint32_t size, uint64_t most, cudaStream_t s) {
    int resident = 0;
    int rc = resident_clusters<TN, KS>(cx, size, &resident);
    if (rc) return rc;
    const unsigned clusters = (unsigned)std::min<uint64_t>(most, KS ? most : (uint64_t)resident);
    cudaLaunchConfig_t q{};
    q.gridDim = dim3(size * clusters);
    q.blockDim = dim3(F8Cfg<TN>::THREADS);
    q.dynamicSmemBytes = F8Cfg<TN>::SMEM;
    q.stream = s;
    cudaLaunchAttribute at[2]{};
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = g_pdl ? 1 : 0;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = size; at[1].val.clusterDim.y = 1; at[1].val.clusterDim.z = 1;
    q.attrs = at; q.numAttrs = size > 1 ? 2 : 1;
    cudaError_t e;
    {
        ProfScope ps_(PK_FP8_GEMM, s);
        e = cudaLaunchKernelEx(&q, gemm_f8_kernel<TN, KS>, tw, tt, g);
    }
    count_launch();
    return e == cudaSuccess ? CM_OK : cuda_error(e, "gemm_f8 launch");
}

template <int TN>
int run_tiles(const Context* cx, const uint8_t* a, uint64_t lda, const uint8_t* b, uint64_t ldb, uint64_t b_gs, const Fp8Args& f, KArgs g,
              cudaStream_t s) {
    using C = F8Cfg<TN>;
    constexpr bool TOK = C::TOK;
    constexpr int CG = C::CG;
    g.tiles_m = (f.m + C::WEIGHTS - 1) / C::WEIGHTS;
    g.tiles_t = (f.n + C::TOKENS - 1) / C::TOKENS;
    // a group's last tile may be partial, so grouped rows make at most n / TOKENS + groups tiles
    const uint64_t token_tiles = f.offsets ? std::min<uint64_t>((uint64_t)f.n / C::TOKENS + f.groups, f.n) : g.tiles_t;
    const uint64_t most = token_tiles * g.tiles_m;
    if (most >= (1ull << 31)) return set_error(CM_EUNSUPPORTED, "cm_matmul_fp8: more than 2^31 tiles");
    g.total = (uint32_t)most;
    g.fd_m = FastDiv(g.tiles_m);
    // D fp32; M operand and N operand (weights and tokens, TOK: tokens and weights), both K-major;
    // M = 128 a CTA, N = TN
    const uint32_t mf = TOK ? f.a_format : f.b_format, nf = TOK ? f.b_format : f.a_format;
    g.idesc = (1u << 4) | (mf << 7) | (nf << 10) | ((uint32_t)(TN >> 3) << 17) | ((uint32_t)(CG * 128 >> 4) << 24);
    const uint32_t stored_groups = f.offsets && b_gs ? f.groups : 1u;
    g.group_step = stored_groups > 1 ? 1u : 0u;
    CUtensorMap tw, tt;
    int rc = make_map(&tw, b, f.k, ldb, f.m, stored_groups, stored_groups > 1 ? b_gs : (uint64_t)f.m * ldb, C::WEIGHTS / CG, 3);
    if (!rc) rc = make_map(&tt, a, f.k, lda, f.n, 1, 0, C::TOKENS / CG, 2);
    if (rc) return rc;
    if constexpr (TN == 16) {
        // Few tiles (wider ones are taken only where narrow ones fill the SMs): a cluster of CTAs to a
        // tile, as many as are resident at once, where the blocks that a CTA is spared cost more than
        // the cluster's launch, barriers and additions.  (Hundredths of a
        // microsecond: one token, m = k = 4096, 32 blocks of 0.18 us: 9.7 us on one CTA a tile, 8.3 on
        // two, 7.4 on four; m = k = 1024, 8 blocks: 4.3, 5.0 and 4.8.)
        constexpr uint32_t block = 18, extra = 180;
        uint32_t best = 1, least = g.kb * block;
        for (uint32_t size = 2; size <= 8 && size <= g.kb && most * size <= (uint64_t)cx->sm_count; size *= 2) {
            const uint32_t cost = (g.kb + size - 1) / size * block + extra;
            int resident = 0;
            if (cost >= least) continue;
            rc = resident_clusters<TN, true>(cx, size, &resident);
            if (rc) return rc;
            if (most <= (uint64_t)resident) { best = size; least = cost; }
        }
        if (best > 1) return launch_tiles<TN, true>(cx, tw, tt, g, best, most, s);
    }
    return launch_tiles<TN, false>(cx, tw, tt, g, CG, most, s);
}

// The tile: 16 to 64 tokens x 128 weight rows on one SM, or 256 x 128 or 256 x 256 on two.  A wider
// tile reads the operands less often and does more a block, but a block takes it longer and there are
// fewer tiles to spread over the SMs.  The one is taken whose whole waves cost least: waves x (K
// blocks x time of a block + time of a tile's output), in hundredths of a microsecond, fitted to 127
// measured sizes from 1 x 512 x 512 to 8192 x 4096 x 11008 and groups of 1 to 512 rows; the choice is
// within a tenth of the best of the five at each of them.  m = k = 4096, in tiles of 16, 32, 64, 256 x
// 128 and 256 x 256: 100 tokens 16.6, 10.5, 11.9, 12.5 and 18.0 us; 200: 23.1, 17.7, 11.9, 12.9 and
// 18.3; 512: 49.7, 32.3, 21.4, 13.6 and 18.3; 1000: 96, 54, 39.5, 22.5 and 19.7.
uint32_t pick_tile(const Context* cx, const Fp8Args& f, uint32_t kb) {
    static const struct { uint32_t tokens, weights, sms, block, out; } kinds[] = {
        {16, 128, 1, 19, 30}, {32, 128, 1, 22, 70}, {64, 128, 1, 25, 80}, {256, 128, 2, 30, 100}, {256, 256, 2, 47, 220}};
    uint32_t best = 0;
    uint64_t least = ~0ull;
    for (uint32_t kind = 0; kind < 5; ++kind) {
        const auto& t = kinds[kind];
        // groups: their sizes are on the device; on average half a tile of each is not filled
        uint64_t token_tiles = (f.n + (uint64_t)t.tokens - 1) / t.tokens;
        if (f.offsets) token_tiles = std::min<uint64_t>(f.n, f.n / t.tokens + (f.groups + 1) / 2 + 1);
        const uint64_t tiles = token_tiles * ((f.m + (uint64_t)t.weights - 1) / t.weights);
        const uint64_t at_once = (uint64_t)cx->sm_count / t.sms;
        const uint64_t cost = (tiles + at_once - 1) / at_once * ((uint64_t)kb * t.block + t.out);
        if (cost < least) { least = cost; best = kind; }
    }
    return best;
}

int fp8_launch(const char* who, const Context* cx, const Fp8Args& f, cudaStream_t s) {
    KArgs g{};
    g.as = f.as; g.bs = f.bs; g.c = f.c; g.offsets = f.offsets;
    g.a_lds = f.a_lds; g.b_lds = f.b_lds; g.bs_gs = f.bs_gs; g.ldc = f.ldc;
    g.groups = f.groups; g.n = f.n; g.m = f.m; g.c_type = f.c_type;
    g.kb = (f.k + 127) / 128; g.ksteps = (f.k + 31) / 32;
    g.status = cx->status; g.timeout_ns = cx->timeout_ns;
    if (f.k == 0) {
        const uint64_t total = (uint64_t)f.n * f.m;
        launch_k(zero_rows_kernel, grid_for(cx, total, 256, 8), 256, 0, s, g, total);
        count_launch();
        cudaError_t e = cudaGetLastError();
        return e == cudaSuccess ? CM_OK : cuda_error(e, who);
    }
    // TMA reads rows that start on 16-byte boundaries (pitches below 2^40); others are copied first
    const uint64_t k16 = (f.k + 15ull) & ~15ull;
    const uint64_t lda = f.n > 1 ? f.lda : k16, ldb = f.m > 1 ? f.ldb : k16;
    const bool one = !f.offsets || f.groups == 1 || f.b_gs == 0;
    const bool a_ok = (uintptr_t)f.a % 16 == 0 && lda % 16 == 0 && lda < (1ull << 40);
    const bool b_ok = (uintptr_t)f.b % 16 == 0 && ldb % 16 == 0 && ldb < (1ull << 40) && (one || (f.b_gs % 16 == 0 && f.b_gs < (1ull << 40)));
    const uint64_t b_count = one ? 1 : f.groups;
    const uint64_t a_bytes = a_ok ? 0 : f.n * k16, b_bytes = b_ok ? 0 : b_count * f.m * k16;
    uint8_t* scratch = nullptr;
    int rc = scratch_alloc((void**)&scratch, a_bytes + b_bytes, s);
    if (rc) return rc;
    auto align_rows = [&](const uint8_t* src, uint64_t ld, uint64_t gs, uint32_t rows, uint64_t count, uint8_t* dst) {
        const uint64_t total = count * rows * (k16 / 16);
        ProfScope ps_(PK_FP8_QUANT, s);
        launch_k(align_rows_kernel, grid_for(cx, total, 256, 8), 256, 0, s, src, ld, gs, rows, f.k, dst, k16, total);
        count_launch();
    };
    if (a_bytes) align_rows(f.a, lda, 0, f.n, 1, scratch);
    if (b_bytes) align_rows(f.b, ldb, one ? 0 : f.b_gs, f.m, b_count, scratch + a_bytes);
    const uint8_t* a = a_bytes ? scratch : f.a;
    const uint8_t* b = b_bytes ? scratch + a_bytes : f.b;
    const uint64_t pa = a_bytes ? k16 : lda, pb = b_bytes ? k16 : ldb, gsb = one ? 0 : b_bytes ? f.m * k16 : f.b_gs;
    switch (pick_tile(cx, f, g.kb)) {
        case 0: rc = run_tiles<16>(cx, a, pa, b, pb, gsb, f, g, s); break;
        case 1: rc = run_tiles<32>(cx, a, pa, b, pb, gsb, f, g, s); break;
        case 2: rc = run_tiles<64>(cx, a, pa, b, pb, gsb, f, g, s); break;
        case 3: rc = run_tiles<128>(cx, a, pa, b, pb, gsb, f, g, s); break;
        default: rc = run_tiles<256>(cx, a, pa, b, pb, gsb, f, g, s); break;
    }
    scratch_free(scratch, s);
    if (rc) return rc;
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

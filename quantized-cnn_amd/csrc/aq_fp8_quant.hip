// Matrices of 8-bit floating point codes (e4m3) with a power-of-two scale per block of 128: made from plain matrices, along
// their rows, along their columns (the transpose, for the products of a backward pass) or both from one read, turned round, and
// read back.  Per block: amax over the finite magnitudes, scale 2^e with the smallest e that brings amax to 448 or less, codes
// x * 2^-e rounded to nearest even.  Scaling by a power of two is exact, so the code's rounding is the only one.
#include "aq_fp8.h"

namespace aq {

// Row blocks of 1 x 128: 16 lanes with 8 elements each hold a block, its maximum comes from four lane exchanges.
template <typename T>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T *__restrict__ x, long long ldx, uint8_t *__restrict__ q, long long ldq,
                                                       void *__restrict__ qs, long long ldqs, uint32_t nblk, uint32_t total, int cols, int scale_f32)
{
    constexpr int U = 4;
    const int c0 = (threadIdx.x & 15) * 8;
    const uint32_t g0 = blockIdx.x * (16 * U) + (threadIdx.x >> 4);
    float v[U][8];
    uint32_t row[U], blk[U];
    int n[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const uint32_t g = g0 + 16 * u;
        row[u] = g / nblk;
        blk[u] = g - row[u] * nblk;
        n[u] = g < total ? min(8, max(0, cols - (int)(blk[u] * FP8_BLK) - c0)) : 0;
    }
    // (the same test in all lanes, so that a workgroup inside the matrix has all its loads in flight at once)
    if (cols % FP8_BLK == 0 && (blockIdx.x + 1) * (16 * U) <= total) {
#pragma unroll
        for (int u = 0; u < U; ++u) load8(x + (long long)row[u] * ldx + blk[u] * FP8_BLK + c0, v[u]);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) load_n(x + (long long)row[u] * ldx + blk[u] * FP8_BLK + c0, n[u], v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        float a = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[u][i]));
        const int e = scale_exponent(max16(a));
        if (g0 + 16 * u >= total) continue;
        store_codes(q + (long long)row[u] * ldq + blk[u] * FP8_BLK + c0, n[u], e4m3x8(v[u], exp2_int(-e)));
        if (c0 == 0) store_scale(qs, (long long)row[u] * ldqs + blk[u], e, scale_f32);
    }
}

struct TileArgs {
    const void *x, *xs;        // source; xs: scales of a source that is in the format already
    long long ldx, ldxs;
    uint8_t *q, *qt;           // codes of x / of its transpose (NULL: not wanted)
    void *qs, *qts;
    long long ldq, ldqs, ldqt, ldqts;
    double *part;              // [row tiles, cols] partial column sums (NULL: not wanted)
    long long rows, cols;
    uint32_t tiles_c;
    int scale_f32;
};

// One workgroup per tile of 128 x 128.  Thread (rg, cg) holds rows 8 rg .. 8 rg + 7 and columns 8 cg .. 8 cg + 7: the 16 lanes
// of a row read it with 16 bytes each, and eight codes of a column are eight neighbouring bytes of the transpose.
//   SQUARE: one scale for the tile.  Otherwise 1 x 128 blocks along the rows for q and along the columns for qt.
//   T = e4m3_el: the source is in the format.  SQUARE turns its codes round unchanged, otherwise its values are quantised anew.
template <typename T, bool SQUARE>
__global__ __launch_bounds__(256) void fp8_tile_kernel(const TileArgs a)
{
    constexpr bool CODES = sizeof(T) == 1;
    constexpr int PITCH = 136;  // bytes of a transposed row in LDS
    __shared__ __attribute__((aligned(16))) uint8_t turned[FP8_BLK * PITCH];
    __shared__ double sums[16 * FP8_BLK];
    __shared__ float colmax[16][FP8_BLK];
    __shared__ int colexp[FP8_BLK];
    const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4;
    const long long tr = blockIdx.x / a.tiles_c, tc = blockIdx.x % a.tiles_c;
    const long long r0 = tr * FP8_BLK, cbase = tc * FP8_BLK;
    const long long c0 = cbase + 8 * cg;
    const int ncol = (int)min(8LL, max(0LL, a.cols - c0));
    float v[8][8];
    const T *p = static_cast<const T *>(a.x) + (r0 + 8 * rg) * a.ldx + c0;
    if (r0 + FP8_BLK <= a.rows && cbase + FP8_BLK <= a.cols) {  // the same in all lanes: all loads in flight at once
#pragma unroll
        for (int i = 0; i < 8; ++i) load8(p + i * a.ldx, v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) load_n(p + i * a.ldx, r0 + 8 * rg + i < a.rows ? ncol : 0, v[i]);
    }
    if (CODES && !SQUARE) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const long long r = r0 + 8 * rg + i;
            const float s = r < a.rows ? load_scale(a.xs, r * a.ldxs + tc, a.scale_f32) : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) v[i][j] *= s;
        }
    }
    if (SQUARE) {
        int e = 0;
        if (!CODES) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[i][j]));
            m = max16(m);
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if ((tid & 63) == 0) colmax[0][tid >> 6] = m;
            __syncthreads();
            e = scale_exponent(fmaxf(fmaxf(colmax[0][0], colmax[0][1]), fmaxf(colmax[0][2], colmax[0][3])));
            __syncthreads();
        }
        const float inv = exp2_int(-e);
        if (!CODES && a.q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const long long r = r0 + 8 * rg + i;
                if (r < a.rows) store_codes(a.q + r * a.ldq + c0, ncol, e4m3x8(v[i], inv));
            }
            if (tid == 0) store_scale(a.qs, tr * a.ldqs + tc, e, a.scale_f32);
        }
        if (!a.qt) return;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float col[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
            *reinterpret_cast<u2_t *>(turned + (8 * cg + j) * PITCH + 8 * rg) = e4m3x8(col, inv);
        }
        if (tid == 0) {
            if (!CODES) store_scale(a.qts, tc * a.ldqts + tr, e, a.scale_f32);
            else if (a.scale_f32) static_cast<float *>(a.qts)[tc * a.ldqts + tr] = static_cast<const float *>(a.xs)[tr * a.ldxs + tc];
            else static_cast<uint8_t *>(a.qts)[tc * a.ldqts + tr] = static_cast<const uint8_t *>(a.xs)[tr * a.ldxs + tc];
        }
    } else {
        if (!CODES && a.q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                float m = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(v[i][j]));
                const int e = scale_exponent(max16(m));
                const long long r = r0 + 8 * rg + i;
                if (r < a.rows) {
                    store_codes(a.q + r * a.ldq + c0, ncol, e4m3x8(v[i], exp2_int(-e)));
                    if (cg == 0) store_scale(a.qs, r * a.ldqs + tc, e, a.scale_f32);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, finite_abs(v[i][j]));
            colmax[rg][8 * cg + j] = m;
        }
        if (!CODES && a.part) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                double s = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += (double)v[i][j];
                sums[rg * FP8_BLK + 8 * cg + j] = s;
            }
        }
        __syncthreads();
        if (tid < FP8_BLK) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) m = fmaxf(m, colmax[i][tid]);
            const int e = scale_exponent(m);
            colexp[tid] = e;
            if (cbase + tid < a.cols) store_scale(a.qts, (cbase + tid) * a.ldqts + tr, e, a.scale_f32);
        } else if (!CODES && a.part && cbase + tid - FP8_BLK < a.cols) {
            const int c = tid - FP8_BLK;
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < 16; ++i) s += sums[i * FP8_BLK + c];
            a.part[tr * a.cols + cbase + c] = s;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float col[8] = {v[0][j], v[1][j], v[2][j], v[3][j], v[4][j], v[5][j], v[6][j], v[7][j]};
            *reinterpret_cast<u2_t *>(turned + (8 * cg + j) * PITCH + 8 * rg) = e4m3x8(col, exp2_int(-colexp[8 * cg + j]));
        }
    }
    __syncthreads();
    // 16 lanes write the 128 codes of a transposed row
    const int nrow = (int)min(8LL, max(0LL, a.rows - r0 - 8 * cg));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = 16 * i + rg;
        if (cbase + c < a.cols)
            store_codes(a.qt + (cbase + c) * a.ldqt + r0 + 8 * cg, nrow, *reinterpret_cast<const u2_t *>(turned + c * PITCH + 8 * cg));
    }
}

__global__ __launch_bounds__(256) void column_sums_kernel(const double *__restrict__ part, long long tiles, long long cols, float *__restrict__ out)
{
    const long long c = (long long)blockIdx.x * 256 + threadIdx.x;
    if (c >= cols) return;
    double s = 0.0;
    for (long long t = 0; t < tiles; ++t) s += part[t * cols + c];
    out[c] = (float)s;
}

// eight codes per thread
template <typename T>
__global__ __launch_bounds__(256) void fp8_values_kernel(const uint8_t *__restrict__ q, long long ldq, const void *__restrict__ qs, long long ldqs,
                                                         long long rows, int cols, uint32_t chunks, int shift, int scale_f32, T *__restrict__ y,
                                                         long long ldy)
{
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long r = t / chunks;
    const int c = (int)(t - r * chunks) * 8;
    if (r >= rows) return;
    const float s = load_scale(qs, (r >> shift) * ldqs + c / FP8_BLK, scale_f32);
    const int n = min(8, cols - c);
    float v[8];
    const e4m3_el *p = reinterpret_cast<const e4m3_el *>(q) + r * ldq + c;
    load_n(p, n, v);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] *= s;
    T *o = y + r * ldy + c;
    store_n(o, n, v);
}

static long long blocks_of(long long n, int b) { return (n + b - 1) / b; }

template <typename T> static void launch_tiles(const TileArgs &a, long long tiles, bool square, hipStream_t st)
{
    const dim3 g((unsigned)tiles), b(256);
    if (square) hipLaunchKernelGGL((fp8_tile_kernel<T, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((fp8_tile_kernel<T, false>), g, b, 0, st, a);
}

} // namespace aq

extern "C" {

size_t aq_fp8_quantize_workspace_bytes(long long rows, long long cols)
{
    return rows > 0 && cols > 0 ? (size_t)aq::blocks_of(rows, aq::FP8_BLK) * (size_t)cols * sizeof(double) : 0;
}

int aq_fp8_quantize(const void *x, int xtype, long long rows, long long cols, long long ldx, uint8_t *q, long long ldq, void *qs,
                    long long ldqs, uint8_t *qt, long long ldqt, void *qts, long long ldqts, int block_rows, int scale_type,
                    float *colsum, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(is_type(xtype), -EINVAL, "aq_fp8_quantize: unknown element type %d", xtype);
    AQ_REQUIRE(scale_type == AQ_SCALE_POW2 || scale_type == AQ_SCALE_F32, -EINVAL, "aq_fp8_quantize: unknown scale type %d", scale_type);
    AQ_REQUIRE(block_rows == 1 || block_rows == FP8_BLK, -EINVAL, "aq_fp8_quantize: blocks of %d rows: 1 or %d", block_rows, FP8_BLK);
    AQ_REQUIRE(rows >= 0 && cols >= 0 && cols < (1LL << 31) - 256, -EINVAL, "aq_fp8_quantize: bad sizes %lld x %lld", rows, cols);
    AQ_REQUIRE(rows == 0 || q || qt, -EINVAL, "aq_fp8_quantize: no output is wanted");
    AQ_REQUIRE(!colsum || ((rows == 0 || qt) && block_rows == 1), -EINVAL, "aq_fp8_quantize: column sums come with the transposed form in 1 x 128 blocks only");
    const long long nblk = blocks_of(cols, FP8_BLK), rblk = blocks_of(rows, FP8_BLK);
    // a launch holds fewer than 2^32 threads: 16 for a row block, 256 for a tile
    AQ_REQUIRE(nblk == 0 || (rows < (1LL << 27) / nblk && rblk * nblk < (1LL << 24)), -E2BIG, "aq_fp8_quantize: %lld x %lld is too large for one call", rows, cols);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (cols == 0 || (rows == 0 && !colsum)) return 0;
    AQ_REQUIRE((rows == 0 || x) && (!q || qs) && (!qt || qts), -EFAULT, "aq_fp8_quantize: NULL pointer");
    AQ_REQUIRE(ldx >= cols && (!q || (ldq >= cols && ldqs >= nblk)) && (!qt || (ldqt >= rows && ldqts >= rblk)), -EINVAL,
               "aq_fp8_quantize: a pitch is smaller than its row");
    if (colsum) {
        const size_t need = aq_fp8_quantize_workspace_bytes(rows, cols);
        AQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 7) == 0), -ENOSPC,
                   "aq_fp8_quantize: workspace of %zu bytes (8-byte aligned) needed, %zu given", need, workspace_bytes);
    }
    const int scale_f32 = scale_type == AQ_SCALE_F32;
    if (rows > 0) {
        if (!qt && block_rows == 1) {
            const long long total = rows * nblk;
            const dim3 g((unsigned)blocks_of(total, 64)), b(256);
            by_type(xtype, [&](auto *t) {
                using T = std::remove_pointer_t<decltype(t)>;
                hipLaunchKernelGGL((fp8_rows_kernel<T>), g, b, 0, st, static_cast<const T *>(x), ldx, q, ldq, qs, ldqs, (uint32_t)nblk, (uint32_t)total,
                                   (int)cols, scale_f32);
                return 0;
            });
        } else {
            const TileArgs a = {x, nullptr, ldx, 0, q, qt, qs, qts, ldq, ldqs, ldqt, ldqts, colsum ? static_cast<double *>(workspace) : nullptr,
                                rows, cols, (uint32_t)nblk, scale_f32};
            by_type(xtype, [&](auto *t) {
                launch_tiles<std::remove_pointer_t<decltype(t)>>(a, nblk * rblk, block_rows != 1, st);
                return 0;
            });
        }
        if (int rc = check_launch("aq_fp8_quantize")) return rc;
    }
    if (colsum) {
        hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)blocks_of(cols, 256)), dim3(256), 0, st, static_cast<const double *>(workspace), rblk, cols,
                           colsum);
        return check_launch("aq_fp8_quantize");
    }
    return 0;
}

int aq_fp8_transpose(const uint8_t *a, long long lda, const void *as, long long ldas, long long rows, long long cols, uint8_t *at,
                     long long ldat, void *ats, long long ldats, int block_rows, int scale_type, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(scale_type == AQ_SCALE_POW2 || scale_type == AQ_SCALE_F32, -EINVAL, "aq_fp8_transpose: unknown scale type %d", scale_type);
    AQ_REQUIRE(block_rows == 1 || block_rows == FP8_BLK, -EINVAL, "aq_fp8_transpose: blocks of %d rows: 1 or %d", block_rows, FP8_BLK);
    AQ_REQUIRE(rows >= 0 && cols >= 0 && cols < (1LL << 31) - 256, -EINVAL, "aq_fp8_transpose: bad sizes %lld x %lld", rows, cols);
    if (rows == 0 || cols == 0) return 0;
    const long long nblk = blocks_of(cols, FP8_BLK), rblk = blocks_of(rows, FP8_BLK);
    AQ_REQUIRE(rblk * nblk < (1LL << 24), -E2BIG, "aq_fp8_transpose: %lld x %lld is too large for one call", rows, cols);
    AQ_REQUIRE(a && as && at && ats, -EFAULT, "aq_fp8_transpose: NULL pointer");
    AQ_REQUIRE(lda >= cols && ldas >= nblk && ldat >= rows && ldats >= rblk, -EINVAL, "aq_fp8_transpose: a pitch is smaller than its row");
    const TileArgs t = {a, as, lda, ldas, nullptr, at, nullptr, ats, 0, 0, ldat, ldats, nullptr, rows, cols, (uint32_t)nblk, scale_type == AQ_SCALE_F32};
    launch_tiles<e4m3_el>(t, nblk * rblk, block_rows != 1, static_cast<hipStream_t>(stream));
    return check_launch("aq_fp8_transpose");
}

int aq_fp8_dequantize(const uint8_t *q, long long ldq, const void *qs, long long ldqs, long long rows, long long cols, int block_rows,
                      int scale_type, void *y, int ytype, long long ldy, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(is_type(ytype), -EINVAL, "aq_fp8_dequantize: unknown element type %d", ytype);
    AQ_REQUIRE(scale_type == AQ_SCALE_POW2 || scale_type == AQ_SCALE_F32, -EINVAL, "aq_fp8_dequantize: unknown scale type %d", scale_type);
    AQ_REQUIRE(block_rows == 1 || block_rows == FP8_BLK, -EINVAL, "aq_fp8_dequantize: blocks of %d rows: 1 or %d", block_rows, FP8_BLK);
    AQ_REQUIRE(rows >= 0 && cols >= 0 && cols < (1LL << 31) - 256, -EINVAL, "aq_fp8_dequantize: bad sizes %lld x %lld", rows, cols);
    if (rows == 0 || cols == 0) return 0;
    const long long chunks = blocks_of(cols, 8);
    AQ_REQUIRE(rows < (1LL << 32) / chunks - 256, -E2BIG, "aq_fp8_dequantize: %lld x %lld is too large for one call", rows, cols);
    AQ_REQUIRE(q && qs && y, -EFAULT, "aq_fp8_dequantize: NULL pointer");
    AQ_REQUIRE(ldq >= cols && ldqs >= blocks_of(cols, FP8_BLK) && ldy >= cols, -EINVAL, "aq_fp8_dequantize: a pitch is smaller than its row");
    const dim3 g((unsigned)blocks_of(rows * chunks, 256)), b(256);
    const int shift = block_rows == 1 ? 0 : 7, scale_f32 = scale_type == AQ_SCALE_F32;
    hipStream_t st = static_cast<hipStream_t>(stream);
    by_type(ytype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        hipLaunchKernelGGL((fp8_values_kernel<T>), g, b, 0, st, q, ldq, qs, ldqs, rows, (int)cols, (uint32_t)chunks, shift, scale_f32,
                           static_cast<T *>(y), ldy);
        return 0;
    });
    return check_launch("aq_fp8_dequantize");
}

} // extern "C"

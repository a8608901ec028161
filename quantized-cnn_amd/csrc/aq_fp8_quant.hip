// Matrices of 8-bit floating point codes (e4m3) with a power-of-two scale per block of 128: made from plain matrices, along
// their rows, along their columns (the transpose, for the products of a backward pass) or both from one read, turned round, and
// read back.  Per block: amax over the finite magnitudes, scale 2^e with the smallest e that brings amax to 448 or less, codes
// x * 2^-e rounded to nearest even.  Scaling by a power of two is exact, so the code's rounding is the only one.
// All are bound by memory bandwidth: 8192 x 8192 bf16 to codes along both axes 56 us (268 MB, 4.7 TB/s; a copy of 1 GiB runs at
// 5.1 TB/s), codes to bf16 values 38 us (201 MB, 5.2 TB/s).
#include "aq_fp8.h"

namespace aq {

// Row blocks of 1 x 128: 16 lanes with 8 elements each hold a block, its maximum comes from four lane exchanges.
template <typename T, bool NT>
__global__ __launch_bounds__(256) void fp8_rows_kernel(const T *__restrict__ x, long long ldx, uint8_t *__restrict__ q, long long ldq,
                                                       void *__restrict__ qs, long long ldqs, uint32_t nblk, uint32_t total, int cols, int scale_f32)
{
    constexpr int U = 4;
    const int c0 = (threadIdx.x & 15) * 8;
    const uint32_t g0 = blockIdx.x * (16 * U) + (threadIdx.x >> 4);
    raw8<T> v[U];
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
        for (int u = 0; u < U; ++u) v[u] = load_raw<NT>(x + (long long)row[u] * ldx + blk[u] * FP8_BLK + c0);
    } else if (cols >= 8) {
        const uint32_t last = (total - 1) / nblk;
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_row_chunk<NT>(x + (long long)min(row[u], last) * ldx, blk[u] * FP8_BLK + c0, cols);
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = row_chunk(v[u], n[u] > 0 ? blk[u] * FP8_BLK + c0 : cols, cols);
    } else {
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = load_raw_n(x + (long long)row[u] * ldx + blk[u] * FP8_BLK + c0, n[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int e = scale_exponent(max16(amax8(v[u])));
        if (g0 + 16 * u >= total) continue;
        const float f[8] = {value(v[u], 0), value(v[u], 1), value(v[u], 2), value(v[u], 3), value(v[u], 4), value(v[u], 5), value(v[u], 6), value(v[u], 7)};
        store_codes<NT>(q + (long long)row[u] * ldq + blk[u] * FP8_BLK + c0, n[u], e4m3x8(f, exp2_int(-e)));
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
    uint32_t tiles_c, tiles_r;
    int scale_f32;
};

// One workgroup per tile of 128 x 128.  Thread (rg, cg) holds rows 8 rg .. 8 rg + 7 and columns 8 cg .. 8 cg + 7, as they lie in
// memory: the 16 lanes of a row read it with 16 bytes each, and eight codes of a column are eight neighbouring bytes of the
// transpose.
//   SQUARE: one scale for the tile.  Otherwise 1 x 128 blocks along the rows for q and along the columns for qt.
//   T = e4m3_el: the source is in the format.  SQUARE turns its codes round unchanged, otherwise its values are quantised anew.
template <typename T, bool SQUARE, bool NT>
__global__ __launch_bounds__(256) void fp8_tile_kernel(const TileArgs a)
{
    constexpr bool CODES = sizeof(T) == 1;
    constexpr int PITCH = 136;  // bytes of a transposed row in LDS
    __shared__ __attribute__((aligned(16))) uint8_t turned[FP8_BLK * PITCH];
    __shared__ float colmax[16][FP8_BLK];
    __shared__ int colexp[FP8_BLK];
    const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4;
    // the tiles go in bands of 8 tile rows, column by column of the band: workgroups that run together then write neighbouring
    // pieces of the transpose's rows as well as read and write neighbouring pieces of x's
    const uint32_t band = blockIdx.x / (8 * a.tiles_c), height = min(8u, a.tiles_r - 8 * band), in = blockIdx.x - band * 8 * a.tiles_c;
    const long long tr = band * 8 + in % height, tc = in / height;
    const long long r0 = tr * FP8_BLK, cbase = tc * FP8_BLK;
    const long long c0 = cbase + 8 * cg;
    const int ncol = (int)min(8LL, max(0LL, a.cols - c0));
    raw8<T> x[8];
    float rscale[8];
    const T *p = static_cast<const T *>(a.x) + (r0 + 8 * rg) * a.ldx + c0;
    if (r0 + FP8_BLK <= a.rows && cbase + FP8_BLK <= a.cols) {  // the same in all lanes: all loads in flight at once
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = load_raw<NT>(p + i * a.ldx);
    } else if (a.cols >= 8) {
        const T *first = static_cast<const T *>(a.x);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = load_row_chunk<NT>(first + min(r0 + 8 * rg + i, a.rows - 1) * a.ldx, c0, a.cols);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = row_chunk(x[i], r0 + 8 * rg + i < a.rows ? c0 : a.cols, a.cols);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = load_raw_n(p + i * a.ldx, r0 + 8 * rg + i < a.rows ? ncol : 0);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const long long r = r0 + 8 * rg + i;
        rscale[i] = CODES && !SQUARE && r < a.rows ? load_scale(a.xs, r * a.ldxs + tc, a.scale_f32) : 0.0f;
    }
    auto at = [&](int i, int j) { return CODES && !SQUARE ? value(x[i], j) * rscale[i] : value(x[i], j); };
    auto turn = [&](int j, float inv) {
        const float col[8] = {at(0, j), at(1, j), at(2, j), at(3, j), at(4, j), at(5, j), at(6, j), at(7, j)};
        *reinterpret_cast<u2_t *>(turned + (8 * cg + j) * PITCH + 8 * rg) = e4m3x8(col, inv);
    };
    auto row_codes = [&](int i, float inv) {
        const float v[8] = {at(i, 0), at(i, 1), at(i, 2), at(i, 3), at(i, 4), at(i, 5), at(i, 6), at(i, 7)};
        const long long r = r0 + 8 * rg + i;
        if (r < a.rows) store_codes<NT>(a.q + r * a.ldq + c0, ncol, e4m3x8(v, inv));
    };
    if (SQUARE) {
        int e = 0;
        if (!CODES) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, amax8(x[i]));
            m = max16(m);
            m = fmaxf(m, __shfl_xor(m, 16, 64));
            m = fmaxf(m, __shfl_xor(m, 32, 64));
            if ((tid & 63) == 0) colmax[0][tid >> 6] = m;
            __syncthreads();
            e = scale_exponent(fmaxf(fmaxf(colmax[0][0], colmax[0][1]), fmaxf(colmax[0][2], colmax[0][3])));
        }
        const float inv = exp2_int(-e);
        if (!CODES && a.q) {
#pragma unroll
            for (int i = 0; i < 8; ++i) row_codes(i, inv);
            if (tid == 0) store_scale(a.qs, tr * a.ldqs + tc, e, a.scale_f32);
        }
        if (!a.qt) return;
#pragma unroll
        for (int j = 0; j < 8; ++j) turn(j, inv);
        if (tid == 0) {
            if (!CODES) store_scale(a.qts, tc * a.ldqts + tr, e, a.scale_f32);
            else if (a.scale_f32) static_cast<float *>(a.qts)[tc * a.ldqts + tr] = static_cast<const float *>(a.xs)[tr * a.ldxs + tc];
            else static_cast<uint8_t *>(a.qts)[tc * a.ldqts + tr] = static_cast<const uint8_t *>(a.xs)[tr * a.ldxs + tc];
        }
    } else {
        float cm[8];
        if constexpr (CODES) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v[8] = {at(0, j), at(1, j), at(2, j), at(3, j), at(4, j), at(5, j), at(6, j), at(7, j)};
                cm[j] = amax8(v);
            }
        } else {
            column_amax8(x, cm);
            if (a.q) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int e = scale_exponent(max16(amax8(x[i])));
                    row_codes(i, exp2_int(-e));
                    const long long r = r0 + 8 * rg + i;
                    if (cg == 0 && r < a.rows) store_scale(a.qs, r * a.ldqs + tc, e, a.scale_f32);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) colmax[rg][8 * cg + j] = cm[j];
        double *sums = reinterpret_cast<double *>(turned);  // [16][128], before the codes go there
        if (!CODES && a.part) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                double s = 0.0;
#pragma unroll
                for (int i = 0; i < 8; ++i) s += (double)at(i, j);
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
        for (int j = 0; j < 8; ++j) turn(j, exp2_int(-colexp[8 * cg + j]));
    }
    __syncthreads();
    // 16 lanes write the 128 codes of a transposed row
    const int nrow = (int)min(8LL, max(0LL, a.rows - r0 - 8 * cg));
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int c = 16 * i + rg;
        if (cbase + c < a.cols)
            store_codes<NT>(a.qt + (cbase + c) * a.ldqt + r0 + 8 * cg, nrow, *reinterpret_cast<const u2_t *>(turned + c * PITCH + 8 * cg));
    }
}

// 64 columns and 16 runs of row tiles a workgroup, in a fixed order
__global__ __launch_bounds__(1024) void column_sums_kernel(const double *__restrict__ part, long long tiles, long long cols, float *__restrict__ out)
{
    __shared__ double sh[16][64];
    const int lane = threadIdx.x & 63, run = threadIdx.x >> 6;
    const long long c = (long long)blockIdx.x * 64 + lane;
    double s = 0.0;
    if (c < cols)
        for (long long t = run; t < tiles; t += 16) s += part[t * cols + c];
    sh[run][lane] = s;
    __syncthreads();
    if (run || c >= cols) return;
    for (int i = 1; i < 16; ++i) s += sh[i][lane];
    out[c] = (float)s;
}

// 16 codes per thread
template <typename T, bool NT>
__global__ __launch_bounds__(256) void fp8_values_kernel(const uint8_t *__restrict__ q, long long ldq, const void *__restrict__ qs, long long ldqs,
                                                         uint32_t rows, int cols, uint32_t chunks, int shift, int scale_f32, T *__restrict__ y,
                                                         long long ldy)
{
    const uint32_t t = blockIdx.x * 256 + threadIdx.x, r = t / chunks;
    const int c = (int)(t - r * chunks) * 16;
    if (r >= rows) return;
    const float s = load_scale(qs, (long long)(r >> shift) * ldqs + c / FP8_BLK, scale_f32);
    const e4m3_el *p = reinterpret_cast<const e4m3_el *>(q) + (long long)r * ldq + c;
    T *o = y + (long long)r * ldy + c;
    if (c + 16 <= cols) {
        const raw8<e4m3_el> lo = load_raw<NT>(p), hi = load_raw<NT>(p + 8);
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = value(lo, i) * s, b[i] = value(hi, i) * s;
        store8_any<NT>(o, a);
        store8_any<NT>(o + 8, b);
        return;
    }
    for (int i = 0; c + i < cols; ++i) o[i] = from_f32<T>(to_f32(p[i]) * s);
}

// 16 codes per thread (8192 x 8191: 23 us, 5.8 TB/s)
__global__ __launch_bounds__(256) void fp8_repitch_kernel(const uint8_t *__restrict__ q, long long ldq, uint32_t rows, int cols, uint32_t chunks,
                                                          uint8_t *__restrict__ p, long long ldp)
{
    const uint32_t t = blockIdx.x * 256 + threadIdx.x, r = t / chunks;
    const int c = (int)(t - r * chunks) * 16;
    if (r >= rows) return;
    const e4m3_el *row = reinterpret_cast<const e4m3_el *>(q) + (long long)r * ldq;
    raw8<e4m3_el> lo, hi;
    if (cols >= 8) {
        lo = load_row_chunk<false>(row, c, cols), hi = load_row_chunk<false>(row, c + 8, cols);
        lo = row_chunk(lo, c, cols), hi = row_chunk(hi, c + 8, cols);
    } else {
        lo = load_raw_n(row + c, cols - c), hi = {};
    }
    *reinterpret_cast<u4_t *>(p + (long long)r * ldp + c) = u4_t{lo.a[0], lo.a[1], hi.a[0], hi.a[1]};
}

static long long blocks_of(long long n, int b) { return (n + b - 1) / b; }

template <typename T> static void launch_tiles(const TileArgs &a, long long tiles, bool square, hipStream_t st)
{
    const dim3 g((unsigned)tiles), b(256);
    const bool stream = a.rows * a.cols * (long long)(sizeof(T) + (a.q ? 1 : 0) + (a.qt ? 1 : 0)) > STREAM_BYTES && rows16(a.x, a.ldx, sizeof(T)) &&
                        rows16(a.q, a.ldq, 1) && rows16(a.qt, a.ldqt, 1);
    if (square) hipLaunchKernelGGL((fp8_tile_kernel<T, true, false>), g, b, 0, st, a);  // weights: the codes are read soon
    else if (stream) hipLaunchKernelGGL((fp8_tile_kernel<T, false, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((fp8_tile_kernel<T, false, false>), g, b, 0, st, a);
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
                if (rows * cols * (long long)(sizeof(T) + 1) > STREAM_BYTES && rows16(x, ldx, sizeof(T)) && rows16(q, ldq, 1))
                    hipLaunchKernelGGL((fp8_rows_kernel<T, true>), g, b, 0, st, static_cast<const T *>(x), ldx, q, ldq, qs, ldqs, (uint32_t)nblk, (uint32_t)total,
                                       (int)cols, scale_f32);
                else
                    hipLaunchKernelGGL((fp8_rows_kernel<T, false>), g, b, 0, st, static_cast<const T *>(x), ldx, q, ldq, qs, ldqs, (uint32_t)nblk, (uint32_t)total,
                                       (int)cols, scale_f32);
                return 0;
            });
        } else {
            const TileArgs a = {x, nullptr, ldx, 0, q, qt, qs, qts, ldq, ldqs, ldqt, ldqts, colsum ? static_cast<double *>(workspace) : nullptr,
                                rows, cols, (uint32_t)nblk, (uint32_t)rblk, scale_f32};
            by_type(xtype, [&](auto *t) {
                launch_tiles<std::remove_pointer_t<decltype(t)>>(a, nblk * rblk, block_rows != 1, st);
                return 0;
            });
        }
        if (int rc = check_launch("aq_fp8_quantize")) return rc;
    }
    if (colsum) {
        hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)blocks_of(cols, 64)), dim3(1024), 0, st, static_cast<const double *>(workspace), rblk, cols,
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
    const TileArgs t = {a, as, lda, ldas, nullptr, at, nullptr, ats, 0, 0, ldat, ldats, nullptr, rows, cols, (uint32_t)nblk, (uint32_t)rblk, scale_type == AQ_SCALE_F32};
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
    const long long chunks = blocks_of(cols, 16);
    AQ_REQUIRE(rows < (1LL << 32) / chunks - 256, -E2BIG, "aq_fp8_dequantize: %lld x %lld is too large for one call", rows, cols);
    AQ_REQUIRE(q && qs && y, -EFAULT, "aq_fp8_dequantize: NULL pointer");
    AQ_REQUIRE(ldq >= cols && ldqs >= blocks_of(cols, FP8_BLK) && ldy >= cols, -EINVAL, "aq_fp8_dequantize: a pitch is smaller than its row");
    const dim3 g((unsigned)blocks_of(rows * chunks, 256)), b(256);
    const int shift = block_rows == 1 ? 0 : 7, scale_f32 = scale_type == AQ_SCALE_F32;
    hipStream_t st = static_cast<hipStream_t>(stream);
    by_type(ytype, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (rows * cols * (long long)(1 + sizeof(T)) > STREAM_BYTES && rows16(q, ldq, 1) && rows16(y, ldy, sizeof(T)))
            hipLaunchKernelGGL((fp8_values_kernel<T, true>), g, b, 0, st, q, ldq, qs, ldqs, (uint32_t)rows, (int)cols, (uint32_t)chunks, shift, scale_f32,
                               static_cast<T *>(y), ldy);
        else
            hipLaunchKernelGGL((fp8_values_kernel<T, false>), g, b, 0, st, q, ldq, qs, ldqs, (uint32_t)rows, (int)cols, (uint32_t)chunks, shift, scale_f32,
                               static_cast<T *>(y), ldy);
        return 0;
    });
    return check_launch("aq_fp8_dequantize");
}

int aq_fp8_repitch(const uint8_t *q, long long ldq, long long rows, long long cols, uint8_t *p, long long ldp, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(rows >= 0 && cols >= 0 && cols < (1LL << 31) - 256, -EINVAL, "aq_fp8_repitch: bad sizes %lld x %lld", rows, cols);
    if (rows == 0 || cols == 0) return 0;
    const long long chunks = blocks_of(cols, 16);
    AQ_REQUIRE(rows < (1LL << 32) / chunks - 256, -E2BIG, "aq_fp8_repitch: %lld x %lld is too large for one call", rows, cols);
    AQ_REQUIRE(q && p, -EFAULT, "aq_fp8_repitch: NULL pointer");
    AQ_REQUIRE(ldq >= cols && ldp >= chunks * 16, -EINVAL, "aq_fp8_repitch: a pitch is smaller than its row");
    AQ_REQUIRE(((uintptr_t)p & 15) == 0 && ldp % 16 == 0, -EINVAL, "aq_fp8_repitch: rows of the output have to start at multiples of 16 bytes");
    hipLaunchKernelGGL(fp8_repitch_kernel, dim3((unsigned)blocks_of(rows * chunks, 256)), dim3(256), 0, static_cast<hipStream_t>(stream), q, ldq, (uint32_t)rows,
                       (int)cols, (uint32_t)chunks, p, ldp);
    return check_launch("aq_fp8_repitch");
}

} // extern "C"

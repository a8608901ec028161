// Root-mean-square norm over the rows of a matrix, with the residual's addition in front and, where it is wanted, e4m3 codes
// with a scale per 1 x 128 block behind; and its gradients.
//   h = round(x + res);  rstd = 1 / sqrt(mean(h^2) + eps);  y = (h * rstd) * w
//   n = h * rstd, g = dy * w:  dx = rstd * (g - n * mean(g * n)) + dh,  dw = sum over rows of dy * n
// The squares are summed in double: rstd is then the correctly rounded one whatever the order of the sum, and codes next to
// a rounding border do not depend on the launch's shape.  One pass: a row stays in the registers of its workgroup between the
// statistics and the outputs, so the traffic is what the operands hold and the kernels are bound by memory bandwidth: 16384 x 8192
// bf16 with residual to codes 168 us (939 MB, 5.6 TB/s), 8192 x 5120 backward 64 us + 6 us for dw's second stage (335 MB, 5.2 TB/s).
#include <algorithm>

#include "aq_fp8.h"

namespace aq {

template <typename S> __device__ inline S wave_sum(S v)
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    return v;
}
// sum over the workgroup, the same value in every thread; sh: 16 elements, free to be used again on return
template <typename S> __device__ inline S group_sum(S v, S *sh)
{
    v = wave_sum(v);
    const int waves = (int)blockDim.x / 64;
    if (waves == 1) return v;
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    S s = sh[0];
    for (int i = 1; i < waves; ++i) s += sh[i];
    __syncthreads();
    return s;
}

struct NormArgs {
    const void *x, *res;
    const float *w;
    void *y, *h, *qs;
    uint8_t *q;
    float *rstd;
    long long ldx, ldres, ldy, ldh, ldq, ldqs, rows, cols;
    double eps;
    int scale_f32;
};

template <bool NT, typename T>
__device__ inline void norm_outputs(const NormArgs &a, long long r, long long c, int n, const float (&hv)[8], const raw8<float> &w, float rs)
{
    float o[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = (hv[j] * rs) * value(w, j);
    if (a.y) store_n<NT>(static_cast<T *>(a.y) + r * a.ldy + c, n, o);
    if (a.q) {
        const int e = scale_exponent(max16(amax8(o)));  // 16 lanes with 8 elements each: one block
        store_codes<NT>(a.q + r * a.ldq + c, n, e4m3x8(o, exp2_int(-e)));
        if ((threadIdx.x & 15) == 0 && n > 0) store_scale(a.qs, r * a.ldqs + c / FP8_BLK, e, a.scale_f32);
    }
}

// one workgroup per row; a thread holds V chunks of 8 columns
template <typename T, int V, bool NT>
__global__ __launch_bounds__(1024) void rms_norm_fwd_kernel(const NormArgs a)
{
    __shared__ double sh[16];
    const long long r = blockIdx.x;
    const int T0 = (int)blockDim.x;
    const T *x = static_cast<const T *>(a.x) + r * a.ldx, *res = static_cast<const T *>(a.res) + r * a.ldres;
    raw8<T> xv[V], rv[V];
    raw8<float> wv[V];
    if (a.cols >= 8) {  // the same in all lanes: all loads in flight at once
#pragma unroll
        for (int i = 0; i < V; ++i) xv[i] = load_row_chunk<NT>(x, (i * T0 + threadIdx.x) * 8, a.cols);
        if (a.res)
#pragma unroll
            for (int i = 0; i < V; ++i) rv[i] = load_row_chunk<NT>(res, (i * T0 + threadIdx.x) * 8, a.cols);
#pragma unroll
        for (int i = 0; i < V; ++i) wv[i] = load_row_chunk<false>(a.w, (i * T0 + threadIdx.x) * 8, a.cols);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (i * T0 + threadIdx.x) * 8;
            xv[i] = row_chunk(xv[i], c, a.cols);
            if (a.res) rv[i] = row_chunk(rv[i], c, a.cols);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (i * T0 + threadIdx.x) * 8, n = (int)min(8LL, a.cols - c);
            xv[i] = load_raw_n(x + c, n);
            if (a.res) rv[i] = load_raw_n(res + c, n);
            wv[i] = load_raw_n(a.w + c, n);
        }
    }
    float hv[V][8];
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hv[i][j] = a.res ? to_f32(from_f32<T>(value(xv[i], j) + value(rv[i], j))) : value(xv[i], j);
            s = __builtin_fma((double)hv[i][j], (double)hv[i][j], s);
        }
        const int c = (i * T0 + threadIdx.x) * 8;
        if (a.h) store_n<NT>(static_cast<T *>(a.h) + r * a.ldh + c, (int)min(8LL, a.cols - c), hv[i]);
    }
    const float rs = (float)(1.0 / sqrt(group_sum(s, sh) / (double)a.cols + a.eps));
    if (a.rstd && threadIdx.x == 0) a.rstd[r] = rs;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (i * T0 + threadIdx.x) * 8;
        norm_outputs<NT, T>(a, r, c, (int)max(0LL, min(8LL, a.cols - c)), hv[i], a.cols >= 8 ? row_chunk(wv[i], c, a.cols) : wv[i], rs);
    }
}

// Short rows (of a head, of a small layer): LPR lanes per row, four rows for each with all their loads in flight, and sums that need no LDS
// (2^20 rows of 128 bf16: 94 us for 537 MB, 404 us with a workgroup a row; 2^20 rows of 64, half of whose lanes idle: 102 us).
template <typename T, int LPR, bool NT>
__global__ __launch_bounds__(256) void rms_norm_fwd_short_kernel(const NormArgs a)
{
    constexpr int U = 4, G = 256 / LPR;
    const int c = (int)(threadIdx.x % LPR) * 8, k = (int)max(0LL, min(8LL, a.cols - c));
    const long long r0 = (long long)blockIdx.x * (G * U) + threadIdx.x / LPR;
    const bool whole = a.cols >= 8;
    auto load = [&](const void *p, long long r, long long ld) {
        const T *row = static_cast<const T *>(p) + min(r, a.rows - 1) * ld;
        return whole ? load_row_chunk<NT>(row, c, a.cols) : load_raw_n(row + c, k);
    };
    raw8<T> xv[U], rv[U];
#pragma unroll
    for (int u = 0; u < U; ++u) xv[u] = load(a.x, r0 + u * G, a.ldx);
    if (a.res)
#pragma unroll
        for (int u = 0; u < U; ++u) rv[u] = load(a.res, r0 + u * G, a.ldres);
    const raw8<float> w = load_raw_n(a.w + c, k);
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const long long r = r0 + u * G;
        if (whole) xv[u] = row_chunk(xv[u], c, a.cols);
        if (whole && a.res) rv[u] = row_chunk(rv[u], c, a.cols);
        float hv[8];
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            hv[j] = a.res ? to_f32(from_f32<T>(value(xv[u], j) + value(rv[u], j))) : value(xv[u], j);
            s = __builtin_fma((double)hv[j], (double)hv[j], s);
        }
#pragma unroll
        for (int m = LPR / 2; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
        const float rs = (float)(1.0 / sqrt(s / (double)a.cols + a.eps));
        const int n = r < a.rows ? k : 0;
        if (a.h) store_n<NT>(static_cast<T *>(a.h) + r * a.ldh + c, n, hv);
        if (a.rstd && c == 0 && r < a.rows) a.rstd[r] = rs;
        norm_outputs<NT, T>(a, r, c, n, hv, w, rs);
    }
}

// rows too long for the registers: read twice
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_fwd_long_kernel(const NormArgs a)
{
    __shared__ double sh[16];
    const long long r = blockIdx.x;
    const T *x = static_cast<const T *>(a.x) + r * a.ldx, *res = static_cast<const T *>(a.res) + r * a.ldres;
    T *h = static_cast<T *>(a.h) + r * a.ldh;
    const long long chunks = (a.cols + 1023 * 8 + 7) / (1024 * 8);
    double s = 0.0;
    auto row_chunk = [&](long long c, int n, float(&hv)[8]) {
        load_n(x + c, n, hv);
        if (!a.res) return;
        float rv[8];
        load_n(res + c, n, rv);
#pragma unroll
        for (int j = 0; j < 8; ++j) hv[j] = to_f32(from_f32<T>(hv[j] + rv[j]));
    };
    for (long long i = 0; i < chunks; ++i) {
        const long long c = (i * 1024 + threadIdx.x) * 8;
        const int n = (int)max(0LL, min(8LL, a.cols - c));
        float hv[8];
        row_chunk(c, n, hv);
        if (a.h) store_n(h + c, n, hv);
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fma((double)hv[j], (double)hv[j], s);
    }
    const float rs = (float)(1.0 / sqrt(group_sum(s, sh) / (double)a.cols + a.eps));
    if (a.rstd && threadIdx.x == 0) a.rstd[r] = rs;
    for (long long i = 0; i < chunks; ++i) {
        const long long c = (i * 1024 + threadIdx.x) * 8;
        const int n = (int)max(0LL, min(8LL, a.cols - c));
        float hv[8];
        if (a.h) load_n(static_cast<const T *>(h) + c, n, hv);  // (its own store: h may be x or res itself)
        else row_chunk(c, n, hv);
        norm_outputs<false, T>(a, r, c, n, hv, load_raw_n(a.w + c, n), rs);
    }
}

struct NormBwdArgs {
    const void *dy, *dh, *h;
    const float *w, *rstd;
    void *dx;
    float *part;  // [grid, cols] partial dw (NULL: not wanted)
    long long lddy, lddh, ldh, lddx, rows, cols;
};

// A fixed number of workgroups, each over every gridDim.x-th row: the columns' partial dw stay in registers from row to row, and
// (V = 1) a row's operands are on their way while the row before it is computed.
template <typename T, int V, bool NT>
__global__ __launch_bounds__(1024) void rms_norm_bwd_kernel(const NormBwdArgs a)
{
    __shared__ float sh[16];
    const int T0 = (int)blockDim.x;
    float wv[V][8], acc[V][8];
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (i * T0 + threadIdx.x) * 8;
        load_n(a.w + c, (int)max(0LL, min(8LL, a.cols - c)), wv[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[i][j] = 0.0f;
    }
    const bool shifted = V == 1 && a.cols >= 8;  // two chunks shifted, or two of dh read early, do not fit the 128 registers of a thread
    const float inv = 1.0f / (float)a.cols;
    raw8<T> dyn[V], hn[V], dhn[V];
    float rsn = 0.0f;
    auto load = [&](long long r) {
        const T *dy = static_cast<const T *>(a.dy) + r * a.lddy, *h = static_cast<const T *>(a.h) + r * a.ldh;
        const T *dh = static_cast<const T *>(a.dh) + r * a.lddh;
        rsn = a.rstd[r];
        if (shifted) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (i * T0 + threadIdx.x) * 8;
                dyn[i] = load_row_chunk<NT>(dy, c, a.cols);
                hn[i] = load_row_chunk<NT>(h, c, a.cols);
                if (a.dh && a.dx) dhn[i] = load_row_chunk<NT>(dh, c, a.cols);
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const int c = (i * T0 + threadIdx.x) * 8, k = (int)max(0LL, min(8LL, a.cols - c));
                dyn[i] = load_raw_n(dy + c, k);
                hn[i] = load_raw_n(h + c, k);
                if (V == 1 && a.dh && a.dx) dhn[i] = load_raw_n(dh + c, k);
            }
        }
    };
    if (V == 1) load(blockIdx.x);  // (the grid has no more workgroups than there are rows)
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        raw8<T> dyv[V], hv[V], dhv[V];
        if (V > 1) load(r);
        const float rs = rsn;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (i * T0 + threadIdx.x) * 8;
            dyv[i] = shifted ? row_chunk(dyn[i], c, a.cols) : dyn[i];
            hv[i] = shifted ? row_chunk(hn[i], c, a.cols) : hn[i];
            if (V == 1 && a.dh && a.dx) dhv[i] = shifted ? row_chunk(dhn[i], c, a.cols) : dhn[i];
        }
        if (V == 1 && r + gridDim.x < a.rows) load(r + gridDim.x);
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = value(dyv[i], j), n = value(hv[i], j) * rs;
                acc[i][j] = __builtin_fmaf(d, n, acc[i][j]);
                s = __builtin_fmaf(d * wv[i][j], n, s);
            }
        if (!a.dx) continue;
        const float m = group_sum(s, sh) * inv;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (i * T0 + threadIdx.x) * 8;
            const int k = (int)max(0LL, min(8LL, a.cols - c));
            if (V > 1 && a.dh) dhv[i] = load_raw_n(static_cast<const T *>(a.dh) + r * a.lddh + c, k);
            float o[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float d = rs * __builtin_fmaf(-(value(hv[i], j) * rs), m, value(dyv[i], j) * wv[i][j]);
                o[j] = a.dh ? d + value(dhv[i], j) : d;
            }
            store_n<NT>(static_cast<T *>(a.dx) + r * a.lddx + c, k, o);
        }
    }
    if (!a.part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = (i * T0 + threadIdx.x) * 8;
        store_n(a.part + (long long)blockIdx.x * a.cols + c, (int)max(0LL, min(8LL, a.cols - c)), acc[i]);
    }
}

// Few rows: one launch.  The first workgroups have a row of dx each; the others 128 columns of dw each, for which they read all rows
// again (rstd is known, so dw needs nothing of dx).  dw's terms are summed in double.  A call of 256 x 4096 takes 11.6 us, 15.3 us with a second
// launch for dw and a workspace for its parts; 512 x 8192 bf16 13 against 21 us; at 1000 x 200, where a workgroup has 32 rows in turn
// for each of its lanes, 19 against 15 us.
constexpr int NORM_SMALL_ROWS = 512;
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_bwd_small_kernel(const NormBwdArgs a, float *__restrict__ dw)
{
    __shared__ float sh[16];
    __shared__ double sums[16][16][8];
    const int rows = (int)a.rows, dx_groups = a.dx ? rows : 0;
    const bool whole = a.cols >= 8;
    auto load = [&](const void *p, long long row, long long ld, int c) {
        const T *at = static_cast<const T *>(p) + row * ld;
        return whole ? load_row_chunk<false>(at, c, a.cols) : load_raw_n(at + c, (int)max(0LL, min(8LL, a.cols - c)));
    };
    auto placed = [&](const raw8<T> &v, int c) { return whole ? row_chunk(v, c, a.cols) : v; };
    if ((int)blockIdx.x < dx_groups) {
        const int r = blockIdx.x, c = threadIdx.x * 8, k = (int)max(0LL, min(8LL, a.cols - c));
        raw8<T> dy = load(a.dy, r, a.lddy, c), h = load(a.h, r, a.ldh, c), dh = {};
        if (a.dh) dh = load(a.dh, r, a.lddh, c);
        float wv[8];
        load_n(a.w + c, k, wv);
        const float rs = a.rstd[r];
        dy = placed(dy, c), h = placed(h, c);
        if (a.dh) dh = placed(dh, c);
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) s = __builtin_fmaf(value(dy, j) * wv[j], value(h, j) * rs, s);
        const float m = group_sum(s, sh) * (1.0f / (float)a.cols);
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = rs * __builtin_fmaf(-(value(h, j) * rs), m, value(dy, j) * wv[j]);
            o[j] = a.dh ? d + value(dh, j) : d;
        }
        store_n(static_cast<T *>(a.dx) + r * a.lddx + c, k, o);
        return;
    }
    // 16 lanes along a row, blockDim / 16 rows at a time
    const int lane = threadIdx.x & 15, c = ((int)blockIdx.x - dx_groups) * 128 + lane * 8, step = (int)blockDim.x / 16;
    double acc[8] = {};
#pragma unroll 4
    for (int r = (int)threadIdx.x >> 4; r < rows; r += step) {
        const raw8<T> dy = placed(load(a.dy, r, a.lddy, c), c), h = placed(load(a.h, r, a.ldh, c), c);
        const float rs = a.rstd[r];
#pragma unroll
        for (int j = 0; j < 8; ++j) acc[j] = __builtin_fma((double)value(dy, j), (double)(value(h, j) * rs), acc[j]);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        acc[j] += __shfl_xor(acc[j], 16, 64);
        acc[j] += __shfl_xor(acc[j], 32, 64);
    }
    if ((threadIdx.x & 63) < 16) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sums[threadIdx.x >> 6][lane][j] = acc[j];
    }
    __syncthreads();
    const long long col = ((long long)blockIdx.x - dx_groups) * 128 + threadIdx.x;
    if (threadIdx.x >= 128 || col >= a.cols) return;
    double s = 0.0;
    for (int i = 0; i < (int)blockDim.x / 64; ++i) s += sums[i][threadIdx.x >> 3][threadIdx.x & 7];
    dw[col] = (float)s;
}

// Short rows: LPR lanes per row, the row behind on its way, as above; the workgroup's groups of lanes join their dw at the end, in double
// (2^20 rows of 128 bf16: 147 us for 805 MB, 651 us with a workgroup a row).
template <typename T, int LPR, bool NT>
__global__ __launch_bounds__(256) void rms_norm_bwd_short_kernel(const NormBwdArgs a)
{
    constexpr int G = 256 / LPR;
    __shared__ float sums[G][LPR * 8];
    const int c = (int)(threadIdx.x % LPR) * 8, k = (int)max(0LL, min(8LL, a.cols - c)), g = threadIdx.x / LPR;
    const bool whole = a.cols >= 8;
    float wv[8], acc[8] = {};
    load_n(a.w + c, k, wv);
    auto load1 = [&](const void *p, long long r, long long ld) {
        const T *row = static_cast<const T *>(p) + r * ld;
        return whole ? load_row_chunk<NT>(row, c, a.cols) : load_raw_n(row + c, k);
    };
    raw8<T> dyn = {}, hn = {}, dhn = {};
    float rsn = 0.0f;
    auto load = [&](long long r) {
        rsn = a.rstd[r];
        dyn = load1(a.dy, r, a.lddy);
        hn = load1(a.h, r, a.ldh);
        if (a.dh && a.dx) dhn = load1(a.dh, r, a.lddh);
    };
    const float inv = 1.0f / (float)a.cols;
    const long long step = (long long)gridDim.x * G;
    long long r = (long long)blockIdx.x * G + g;
    if (r < a.rows) load(r);
    for (; r < a.rows; r += step) {  // (the lanes of a row end together)
        const raw8<T> dy = whole ? row_chunk(dyn, c, a.cols) : dyn, h = whole ? row_chunk(hn, c, a.cols) : hn;
        raw8<T> dh = {};
        if (a.dh && a.dx) dh = whole ? row_chunk(dhn, c, a.cols) : dhn;
        const float rs = rsn;
        if (r + step < a.rows) load(r + step);
        float s = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = value(dy, j), n = value(h, j) * rs;
            acc[j] = __builtin_fmaf(d, n, acc[j]);
            s = __builtin_fmaf(d * wv[j], n, s);
        }
        if (!a.dx) continue;
#pragma unroll
        for (int m = LPR / 2; m >= 1; m >>= 1) s += __shfl_xor(s, m, 64);
        const float m = s * inv;
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float d = rs * __builtin_fmaf(-(value(h, j) * rs), m, value(dy, j) * wv[j]);
            o[j] = a.dh ? d + value(dh, j) : d;
        }
        store_n<NT>(static_cast<T *>(a.dx) + r * a.lddx + c, k, o);
    }
    if (!a.part) return;
#pragma unroll
    for (int j = 0; j < 8; ++j) sums[g][c + j] = acc[j];
    __syncthreads();
    for (int col = threadIdx.x; col < (int)a.cols; col += 256) {
        double s = 0.0;
#pragma unroll
        for (int i = 0; i < G; ++i) s += (double)sums[i][col];
        a.part[(long long)blockIdx.x * a.cols + col] = (float)s;
    }
}

// rows too long for the registers: dx reads its row twice, dw is a sum over a slice of rows for 256 columns a workgroup
template <typename T>
__global__ __launch_bounds__(1024) void rms_norm_dx_long_kernel(const NormBwdArgs a)
{
    __shared__ float sh[16];
    const long long r = blockIdx.x;
    const T *dy = static_cast<const T *>(a.dy) + r * a.lddy, *h = static_cast<const T *>(a.h) + r * a.ldh;
    const T *dh = static_cast<const T *>(a.dh) + r * a.lddh;
    const float rs = a.rstd[r];
    float s = 0.0f;
    for (long long c = threadIdx.x; c < a.cols; c += 1024) s = __builtin_fmaf(to_f32(dy[c]) * a.w[c], to_f32(h[c]) * rs, s);
    const float m = group_sum(s, sh) / (float)a.cols;
    for (long long c = threadIdx.x; c < a.cols; c += 1024) {
        const float d = rs * __builtin_fmaf(-to_f32(h[c]) * rs, m, to_f32(dy[c]) * a.w[c]);
        static_cast<T *>(a.dx)[r * a.lddx + c] = from_f32<T>(a.dh ? d + to_f32(dh[c]) : d);
    }
}
template <typename T>
__global__ __launch_bounds__(256) void rms_norm_dw_long_kernel(const NormBwdArgs a, int slices)
{
    const long long c = (long long)(blockIdx.x / slices) * 256 + threadIdx.x;
    const int slice = blockIdx.x % slices;
    if (c >= a.cols) return;
    float s = 0.0f;
    for (long long r = slice; r < a.rows; r += slices)
        s = __builtin_fmaf(to_f32(static_cast<const T *>(a.dy)[r * a.lddy + c]), to_f32(static_cast<const T *>(a.h)[r * a.ldh + c]) * a.rstd[r], s);
    a.part[(long long)slice * a.cols + c] = s;
}

// dw: 16 columns and 64 runs of the partial rows a workgroup, summed in double in a fixed order
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const float *__restrict__ part, int n, long long cols, float *__restrict__ dw)
{
    __shared__ double sh[64][16];
    const int lane = threadIdx.x & 15, run = threadIdx.x >> 4;
    const long long c = (long long)blockIdx.x * 16 + lane;
    double s = 0.0;
    if (c < cols) {
#pragma unroll 4
        for (int i = run; i < n; i += 64) s += (double)part[i * cols + c];
    }
    sh[run][lane] = s;
    __syncthreads();
    for (int half = 32; half >= 1; half >>= 1) {
        if (run < half) sh[run][lane] += sh[run + half][lane];
        __syncthreads();
    }
    if (run == 0 && c < cols) dw[c] = (float)sh[0][lane];
}

constexpr long long NORM_SHORT = 256;
constexpr long long NORM_LONG = 1024 * 4 * 8, NORM_BWD_LONG = 1024 * 2 * 8;  // columns that fit the registers of a workgroup
// threads for `cols` columns in chunks of 8, v of them a thread: whole wavefronts
static unsigned norm_threads(long long cols, int v) { return (unsigned)((cols + 8 * v - 1) / (8 * v) + 63) / 64 * 64; }

static bool norm_small(long long rows, long long cols) { return rows > 0 && rows <= NORM_SMALL_ROWS && cols <= 1024 * 8; }
// workgroups of the backward kernel (= rows of partial dw)
static int norm_parts(long long rows, long long cols)
{
    if (cols <= NORM_SHORT) return (int)std::min<long long>((rows + 7) / 8, 2048);  // (eight or sixteen rows a workgroup at a time)
    return (int)std::min<long long>(rows, cols > NORM_BWD_LONG ? 64 : cols <= 1024 ? 2048 : 512);
}

} // namespace aq

extern "C" {

int aq_rms_norm_fwd(const void *x, long long ldx, const void *res, long long ldres, int type, const float *w, long long rows,
                    long long cols, double eps, void *y, long long ldy, uint8_t *q, long long ldq, void *qs, long long ldqs, int scale_type,
                    void *h, long long ldh, float *rstd, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(type == AQ_F32 || type == AQ_BF16 || type == AQ_F16, -EINVAL, "aq_rms_norm_fwd: unknown element type %d", type);
    AQ_REQUIRE(scale_type == AQ_SCALE_POW2 || scale_type == AQ_SCALE_F32, -EINVAL, "aq_rms_norm_fwd: unknown scale type %d", scale_type);
    AQ_REQUIRE(rows >= 0 && cols >= 1 && cols < (1LL << 31) - 16384, -EINVAL, "aq_rms_norm_fwd: bad sizes %lld x %lld", rows, cols);
    AQ_REQUIRE(rows < (cols <= NORM_SHORT ? 1LL << 28 : 1LL << 22), -E2BIG, "aq_rms_norm_fwd: %lld rows of %lld are too many for one call", rows, cols);
    AQ_REQUIRE(eps >= 0, -EDOM, "aq_rms_norm_fwd: eps=%g is negative", eps);
    if (rows == 0) return 0;
    AQ_REQUIRE(x && w && (y || q || h || rstd) && (!q || qs), -EFAULT, "aq_rms_norm_fwd: NULL pointer");
    AQ_REQUIRE(ldx >= cols && (!res || ldres >= cols) && (!y || ldy >= cols) && (!q || (ldq >= cols && ldqs >= (cols + FP8_BLK - 1) / FP8_BLK)) &&
                   (!h || ldh >= cols), -EINVAL, "aq_rms_norm_fwd: a pitch is smaller than its row");
    const NormArgs a = {x, res, w, y, h, qs, q, rstd, ldx, ldres, ldy, ldh, ldq, ldqs, rows, cols, eps, scale_type == AQ_SCALE_F32};
    hipStream_t st = static_cast<hipStream_t>(stream);
    by_type(type, [&](auto *t) {
        using T = std::remove_pointer_t<decltype(t)>;
        if (cols > NORM_LONG) {
            hipLaunchKernelGGL((rms_norm_fwd_long_kernel<T>), dim3((unsigned)rows), dim3(1024), 0, st, a);
            return 0;
        }
        // few chunks a thread while a workgroup stays small enough to have several of them on a compute unit
        const long long each = cols * type_size(type);
        const bool stream = rows * (each + (res ? each : 0) + (h ? each : 0) + (y ? each : 0) + (q ? cols : 0)) > STREAM_BYTES &&
                            rows16(x, ldx, sizeof(T)) && rows16(res, ldres, sizeof(T)) && rows16(y, ldy, sizeof(T)) && rows16(h, ldh, sizeof(T)) && rows16(q, ldq, 1);
        const dim3 g((unsigned)rows);
        auto launch = [&](auto v) {
            constexpr int V = decltype(v)::value;
            if (stream) hipLaunchKernelGGL((rms_norm_fwd_kernel<T, V, true>), g, dim3(norm_threads(cols, V)), 0, st, a);
            else hipLaunchKernelGGL((rms_norm_fwd_kernel<T, V, false>), g, dim3(norm_threads(cols, V)), 0, st, a);
        };
        auto launch_short = [&](auto lanes) {
            constexpr int LPR = decltype(lanes)::value, ROWS = 4 * 256 / LPR;
            const dim3 gs((unsigned)((rows + ROWS - 1) / ROWS)), b(256);
            if (stream) hipLaunchKernelGGL((rms_norm_fwd_short_kernel<T, LPR, true>), gs, b, 0, st, a);
            else hipLaunchKernelGGL((rms_norm_fwd_short_kernel<T, LPR, false>), gs, b, 0, st, a);
        };
        if (cols <= 128) launch_short(std::integral_constant<int, 16>{});
        else if (cols <= NORM_SHORT) launch_short(std::integral_constant<int, 32>{});
        else if (cols <= 256 * 8) launch(std::integral_constant<int, 1>{});
        else if (cols <= 512 * 2 * 8) launch(std::integral_constant<int, 2>{});
        else launch(std::integral_constant<int, 4>{});
        return 0;
    });
    return check_launch("aq_rms_norm_fwd");
}

size_t aq_rms_norm_bwd_workspace_bytes(long long rows, long long cols)
{
    return rows > 0 && cols > 0 && !aq::norm_small(rows, cols) ? (size_t)aq::norm_parts(rows, cols) * (size_t)cols * sizeof(float) : 0;
}

int aq_rms_norm_bwd(const void *dy, long long lddy, const void *dh, long long lddh, const void *h, long long ldh, int type, const float *w,
                    const float *rstd, long long rows, long long cols, void *dx, long long lddx, float *dw, void *workspace,
                    size_t workspace_bytes, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(type == AQ_F32 || type == AQ_BF16 || type == AQ_F16, -EINVAL, "aq_rms_norm_bwd: unknown element type %d", type);
    AQ_REQUIRE(rows >= 0 && cols >= 1 && cols < (1LL << 31) - 16384, -EINVAL, "aq_rms_norm_bwd: bad sizes %lld x %lld", rows, cols);
    AQ_REQUIRE(rows < (cols <= NORM_SHORT ? 1LL << 28 : 1LL << 22), -E2BIG, "aq_rms_norm_bwd: %lld rows of %lld are too many for one call", rows, cols);
    AQ_REQUIRE(dx || dw, -EINVAL, "aq_rms_norm_bwd: no output is wanted");
    AQ_REQUIRE(rows == 0 || (dy && h && w && rstd), -EFAULT, "aq_rms_norm_bwd: NULL pointer");
    AQ_REQUIRE(rows == 0 || (lddy >= cols && ldh >= cols && (!dh || lddh >= cols) && (!dx || lddx >= cols)), -EINVAL,
               "aq_rms_norm_bwd: a pitch is smaller than its row");
    const int parts = norm_parts(rows, cols);
    if (dw && rows) {
        const size_t need = aq_rms_norm_bwd_workspace_bytes(rows, cols);
        AQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), -ENOSPC,
                   "aq_rms_norm_bwd: workspace of %zu bytes (16-byte aligned) needed, %zu given", need, workspace_bytes);
    }
    const NormBwdArgs a = {dy, dh, h, w, rstd, dx, dw ? static_cast<float *>(workspace) : nullptr, lddy, lddh, ldh, lddx, rows, cols};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (norm_small(rows, cols)) {
        const unsigned groups = (unsigned)((dx ? rows : 0) + (dw ? (cols + 127) / 128 : 0));
        const dim3 b(std::max(512u, norm_threads(cols, 1)));
        by_type(type, [&](auto *t) {
            hipLaunchKernelGGL((rms_norm_bwd_small_kernel<std::remove_pointer_t<decltype(t)>>), dim3(groups), b, 0, st, a, dw);
            return 0;
        });
        return check_launch("aq_rms_norm_bwd");
    }
    if (rows > 0) {
        by_type(type, [&](auto *t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (cols > NORM_BWD_LONG) {
                if (dx) hipLaunchKernelGGL((rms_norm_dx_long_kernel<T>), dim3((unsigned)rows), dim3(1024), 0, st, a);
                if (dw) hipLaunchKernelGGL((rms_norm_dw_long_kernel<T>), dim3((unsigned)((cols + 255) / 256 * parts)), dim3(256), 0, st, a, parts);
                return 0;
            }
            const long long each = cols * type_size(type);
            const bool stream = rows * (2 * each + (dh ? each : 0) + (dx ? each : 0)) > STREAM_BYTES && rows16(dy, lddy, sizeof(T)) &&
                                rows16(h, ldh, sizeof(T)) && rows16(dh, lddh, sizeof(T)) && rows16(dx, lddx, sizeof(T));
            auto launch = [&](auto v) {
                constexpr int V = decltype(v)::value;
                if (stream) hipLaunchKernelGGL((rms_norm_bwd_kernel<T, V, true>), dim3((unsigned)parts), dim3(norm_threads(cols, V)), 0, st, a);
                else hipLaunchKernelGGL((rms_norm_bwd_kernel<T, V, false>), dim3((unsigned)parts), dim3(norm_threads(cols, V)), 0, st, a);
            };
            auto launch_short = [&](auto lanes) {
                constexpr int LPR = decltype(lanes)::value;
                if (stream) hipLaunchKernelGGL((rms_norm_bwd_short_kernel<T, LPR, true>), dim3((unsigned)parts), dim3(256), 0, st, a);
                else hipLaunchKernelGGL((rms_norm_bwd_short_kernel<T, LPR, false>), dim3((unsigned)parts), dim3(256), 0, st, a);
            };
            if (cols <= 128) launch_short(std::integral_constant<int, 16>{});
            else if (cols <= NORM_SHORT) launch_short(std::integral_constant<int, 32>{});
            else if (cols <= 1024 * 8) launch(std::integral_constant<int, 1>{});
            else launch(std::integral_constant<int, 2>{});
            return 0;
        });
        if (int rc = check_launch("aq_rms_norm_bwd")) return rc;
    }
    if (dw) hipLaunchKernelGGL(rms_norm_dw_kernel, dim3((unsigned)((cols + 15) / 16)), dim3(1024), 0, st, a.part, parts, cols, dw);
    return check_launch("aq_rms_norm_bwd");
}

} // extern "C"

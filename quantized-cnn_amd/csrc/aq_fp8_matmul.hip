// y [M, N] = A [M, K] . B [N, K]^T (+ bias), A and B in e4m3 codes with a scale per block of 128 along K.
//
//   y[m, n] = bias[n] + sum over blocks b of  sA[m, b] * sB[n, b] * sum_{k in b} a[m, k] * b[n, k]
//
// The matrix instruction takes B's rows as its first operand and A's as its second: a lane then holds four neighbouring
// columns n of one row m.  Three ways to the sum over a block:
//   POW2:  power-of-two scales go into the scaled 16x16x128 instruction itself; one instruction per block, fp32 accumulator.
//   FP32S: scales of any value: the block's sum from a zero accumulator, then acc += sum * (sA * sB) in fp32.
//   EXACT: fp32 outputs.  The 8-bit instruction aligns the products of 8 neighbouring k to the largest of them and drops what
//          lies 2^-14 below it (measured; 1.5e-5 of a sum of 128 normally distributed products): nothing beside the rounding of
//          a 16-bit output, too much for an fp32 one.  The codes, which are exact in fp16, go through the 16x16x32 fp16
//          instruction instead (measured 1e-8), then as FP32S.
#include <algorithm>

#include "aq_fp8.h"

namespace aq {

typedef int i8_t __attribute__((ext_vector_type(8)));
typedef int i4_t __attribute__((ext_vector_type(4)));
typedef _Float16 h8_t __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));

enum { POW2 = 0, FP32S = 1, EXACT = 2 };

struct MatArgs {
    const uint8_t *a, *b;
    const void *as, *bs;
    const float *bias;
    void *y;
    long long lda, ldb, ldas, ldbs, ldy;
    int M, N, K;
    int ashift, bshift;  // rows that share a scale: 2^shift
    int scale_f32;
    uint32_t tiles_m, tiles_n;
};

// zero what lies at K or behind it in 16 codes that start at k
__device__ inline i4_t mask16(i4_t v, int k, int K)
{
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const int left = K - (k + 4 * d);
        if (left < 4) v[d] = left <= 0 ? 0 : v[d] & ((1 << 8 * left) - 1);
    }
    return v;
}

__device__ inline h8_t codes_to_fp16(int lo, int hi)
{
    const h2_t a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
    const h2_t c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
    return h8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <int MODE> __device__ inline f4_t block_product(const i8_t &b, const i8_t &a, f4_t acc, int sb, int sa)
{
    if (MODE == POW2) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 0, 0, 0, sb, 0, sa);
    f4_t s = {0.f, 0.f, 0.f, 0.f};
    if (MODE == FP32S) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, s, 0, 0, 0, 127, 0, 127);
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_fp16(b[2 * i], b[2 * i + 1]), codes_to_fp16(a[2 * i], a[2 * i + 1]), s, 0, 0, 0);
    return s;
}

template <typename T> __device__ inline void store4(T *p, int n, const f4_t &v)
{
    if (n >= 4) {
        if constexpr (sizeof(T) == 4) *reinterpret_cast<f4_any *>(p) = v;
        else *reinterpret_cast<u2_any *>(p) = u2_t{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
        return;
    }
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (i < n) p[i] = from_f32<T>(v[i]);
}

// Tiles of BM x BN, WM x WN wavefronts, K in steps of one block of 128 bytes.  Operands go from memory to LDS without passing
// registers, 16 bytes a lane; row r of a tile lies at 128 r with its 16-byte chunk c at place c ^ (r & 7), which spreads the
// 16 rows that a fragment reads over all banks.  A lane of a fragment takes chunks g and g + 4 of its row (g = lane / 16): the
// same K order for both operands, which is all that a sum over k needs.
template <int BM, int BN, int WM, int WN, int MODE, typename T>
__global__ __launch_bounds__(WM *WN * 64) void fp8_matmul_kernel(const MatArgs p)
{
    constexpr int THREADS = WM * WN * 64, WAVES = WM * WN;
    constexpr int TM = BM / WM / 16, TN = BN / WN / 16;
    constexpr int LOADS = (BM + BN) / 8 / WAVES;  // 1 KiB loads of 8 rows per wavefront and step
    static_assert((BM + BN) % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0 && BM + BN <= THREADS, "");
    __shared__ __attribute__((aligned(16))) uint8_t tile[2][(BM + BN) * FP8_BLK];
    __shared__ __attribute__((aligned(16))) uint32_t scale[2][BM + BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int m0 = (int)(blockIdx.x % p.tiles_m) * BM, n0 = (int)(blockIdx.x / p.tiles_m) * BN;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK, kround = (p.K + 15) & ~15;

    // sources of this lane's 16-byte loads: rows past the end read the last row (their results are not stored)
    const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
    const uint8_t *src[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
        const int r = (i * WAVES + wave) * 8 + (lane >> 3);  // tile rows: A's, then B's (uniform over the wavefront's eight)
        src[i] = r < BM ? p.a + (long long)min(m0 + r, p.M - 1) * p.lda : p.b + (long long)min(n0 + r - BM, p.N - 1) * p.ldb;
    }
    // the scale of one tile row per thread
    const uint8_t *ssrc = nullptr;
    if (tid < BM + BN) {
        const long long i = tid < BM ? (long long)(min(m0 + tid, p.M - 1) >> p.ashift) * p.ldas : (long long)(min(n0 + tid - BM, p.N - 1) >> p.bshift) * p.ldbs;
        ssrc = static_cast<const uint8_t *>(tid < BM ? p.as : p.bs) + i * (p.scale_f32 ? 4 : 1);
    }
    auto read_scale = [&](int kb) -> uint32_t {
        if (tid >= BM + BN) return 0;
        if (MODE == POW2) return ssrc[kb];
        return __float_as_uint(load_scale(ssrc, kb, p.scale_f32));
    };
    auto fetch = [&](int kb, int buf) {
        const int k = kb * FP8_BLK + chunk;
        const int at = k < kround ? k : 0;  // a chunk past the row's end reads its first one and is masked below
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void *)(src[i] + at),
                                             (__attribute__((address_space(3))) void *)(tile[buf] + (i * WAVES + wave) * 1024), 16, 0, 0);
    };

    f4_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};

    const int g = lane >> 4, off = (lane & 15) * FP8_BLK + ((g ^ (lane & 7)) * 16);
    auto compute = [&](int kb, int buf, bool tail) {
        const uint8_t *ta = tile[buf] + wm * FP8_BLK, *tb = tile[buf] + (BM + wn) * FP8_BLK;
        const uint32_t *sa = scale[buf] + wm, *sb = scale[buf] + BM + wn;
        auto fragment = [&](const uint8_t *t, int i) {
            i4_t lo = *reinterpret_cast<const i4_t *>(t + i * 2048 + off), hi = *reinterpret_cast<const i4_t *>(t + i * 2048 + (off ^ 64));
            if (tail) {
                lo = mask16(lo, kb * FP8_BLK + g * 16, p.K);
                hi = mask16(hi, kb * FP8_BLK + g * 16 + 64, p.K);
            }
            return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
        };
        i8_t af[TM];
        uint32_t av[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            af[i] = fragment(ta, i);
            av[i] = sa[16 * i + (lane & 15)];
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const i8_t bf = fragment(tb, j);
            if (MODE == POW2) {
                const int bv = (int)sb[16 * j + (lane & 15)];
#pragma unroll
                for (int i = 0; i < TM; ++i) acc[i][j] = block_product<MODE>(bf, af[i], acc[i][j], bv, (int)av[i]);
            } else {
                const f4_t bv = *reinterpret_cast<const f4_t *>(sb + 16 * j + 4 * g);
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const f4_t s = block_product<MODE>(bf, af[i], acc[i][j], 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(s[e], bv[e] * __uint_as_float(av[i]), acc[i][j][e]);
                }
            }
        }
    };

    fetch(0, 0);
    if (tid < BM + BN) scale[0][tid] = read_scale(0);
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    for (int kb = 0; kb < nkb; ++kb) {
        const int buf = kb & 1;
        uint32_t next = 0;
        if (kb + 1 < nkb) {
            fetch(kb + 1, buf ^ 1);
            next = read_scale(kb + 1);
        }
        if ((kb + 1) * FP8_BLK <= p.K) compute(kb, buf, false);
        else compute(kb, buf, true);
        if (tid < BM + BN) scale[buf ^ 1][tid] = next;
        __builtin_amdgcn_s_waitcnt(0);  // the next step's tile is in LDS before anybody passes the barrier
        __syncthreads();
    }

    T *y = static_cast<T *>(p.y);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = n0 + wn + 16 * j + 4 * g;
        f4_t bias = {0.f, 0.f, 0.f, 0.f};
        if (p.bias)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < p.N) bias[e] = p.bias[n + e];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int m = m0 + wm + 16 * i + (lane & 15);
            if (m < p.M) store4(y + (long long)m * p.ldy + n, p.N - n, acc[i][j] + bias);
        }
    }
}

template <int MODE, typename T> static void launch_matmul(MatArgs p, hipStream_t st)
{
    constexpr int BM = 64, BN = 64;
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    hipLaunchKernelGGL((fp8_matmul_kernel<BM, BN, 2, 2, MODE, T>), dim3(p.tiles_m * p.tiles_n), dim3(256), 0, st, p);
}

} // namespace aq

extern "C" {

size_t aq_fp8_matmul_workspace_bytes(long long M, long long N, long long K)
{
    (void)M, (void)N, (void)K;
    return 0;
}

int aq_fp8_matmul(const uint8_t *a, long long lda, const void *as, long long ldas, int a_block_rows, const uint8_t *b, long long ldb,
                  const void *bs, long long ldbs, int b_block_rows, long long M, long long N, long long K, int scale_type,
                  const float *bias, void *y, int ytype, long long ldy, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(is_type(ytype), -EINVAL, "aq_fp8_matmul: unknown element type %d", ytype);
    AQ_REQUIRE(scale_type == AQ_SCALE_POW2 || scale_type == AQ_SCALE_F32, -EINVAL, "aq_fp8_matmul: unknown scale type %d", scale_type);
    AQ_REQUIRE((a_block_rows == 1 || a_block_rows == FP8_BLK) && (b_block_rows == 1 || b_block_rows == FP8_BLK), -EINVAL,
               "aq_fp8_matmul: blocks of %d and %d rows: 1 or %d", a_block_rows, b_block_rows, FP8_BLK);
    AQ_REQUIRE(M >= 0 && N >= 0 && K >= 1, -EINVAL, "aq_fp8_matmul: bad sizes M=%lld N=%lld K=%lld", M, N, K);
    // a launch holds fewer than 2^32 threads, row and column numbers stay below 2^31
    AQ_REQUIRE(M < (1LL << 30) && N < (1LL << 30) && K < (1LL << 30) && ((M + 63) / 64) * ((N + 63) / 64) < (1LL << 22), -E2BIG,
               "aq_fp8_matmul: M=%lld N=%lld K=%lld is too large for one call", M, N, K);
    if (M == 0 || N == 0) return 0;
    AQ_REQUIRE(a && as && b && bs && y, -EFAULT, "aq_fp8_matmul: NULL pointer");
    const long long nkb = (K + FP8_BLK - 1) / FP8_BLK;
    AQ_REQUIRE(lda >= K && ldb >= K && ldas >= nkb && ldbs >= nkb && ldy >= N, -EINVAL, "aq_fp8_matmul: a pitch is smaller than its row");
    AQ_REQUIRE(((uintptr_t)a & 15) == 0 && ((uintptr_t)b & 15) == 0 && lda % 16 == 0 && ldb % 16 == 0, -EINVAL,
               "aq_fp8_matmul: codes and their pitches (%lld, %lld) have to be multiples of 16 bytes", lda, ldb);
    const size_t need = aq_fp8_matmul_workspace_bytes(M, N, K);
    AQ_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 15) == 0), -ENOSPC,
               "aq_fp8_matmul: workspace of %zu bytes (16-byte aligned) needed, %zu given", need, workspace_bytes);
    const MatArgs p = {a, b, as, bs, bias, y, lda, ldb, ldas, ldbs, ldy, (int)M, (int)N, (int)K, a_block_rows == 1 ? 0 : 7, b_block_rows == 1 ? 0 : 7,
                       scale_type == AQ_SCALE_F32, 0, 0};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (ytype == AQ_F32) launch_matmul<EXACT, float>(p, st);
    else if (scale_type == AQ_SCALE_POW2) ytype == AQ_BF16 ? launch_matmul<POW2, bf16_el>(p, st) : launch_matmul<POW2, f16_el>(p, st);
    else ytype == AQ_BF16 ? launch_matmul<FP32S, bf16_el>(p, st) : launch_matmul<FP32S, f16_el>(p, st);
    return check_launch("aq_fp8_matmul");
}

} // extern "C"

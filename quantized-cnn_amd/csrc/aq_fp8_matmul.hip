// y [M, N] = A [M, K] . B [N, K]^T (+ bias), A and B in e4m3 codes with a scale per block of 128 along K.
//
//   y[m, n] = bias[n] + sum over blocks b of  sA[m, b] * sB[n, b] * sum_{k in b} a[m, k] * b[n, k]
//
// The matrix instruction takes B's rows as its first operand and A's as its second: a lane then holds four neighbouring
// columns n of one row m.  Three ways to the sum over a block:
//   POW2:  power-of-two scales go into the scaled 16x16x128 instruction itself; one instruction per block, fp32 accumulator.
//   FP32S: scales of any value: the block's sum from a zero accumulator, then acc += sum * (sA * sB) in fp32 (add_scaled() where
//          sA * sB leaves fp32's normal numbers).
//   EXACT: fp32 outputs.  The 8-bit instruction adds the products of 8 neighbouring k as multiples of 2^(E - 13), each cut towards zero,
//          E the largest sum of two codes' exponents among them (measured: a product of 2^-13 beside one of 1 is kept, one of 2^-14 is
//          not; subnormal codes count with -6, zeros not at all; 1.5e-5 of a sum of 128 normally distributed products): little beside the
//          rounding of a 16-bit output, too much for an fp32 one.  The codes, which are exact in fp16, go through the 16x16x32 fp16
//          instruction instead (measured 1e-8), then as FP32S.
//   WIDE:  the same for large products with power-of-two scales: code * scale is exact in bf16 (for scales of 2^-124 to 2^119; what has
//          others is computed as EXACT at the end), so the scales go into the conversion, the blocks' sums into
//          one accumulator through the bf16 instruction, and the fp32 multiplications per block are saved.
//
// What bounds them, measured: 8192^3 to bf16 0.43 ms, 2.56 PFLOP/s (a library product of fp8 matrices with one scale: 2.64): the power
// limit (a loop of nothing but these instructions on random codes reaches 3.8 PFLOP/s).  4096^3 to fp32 0.118 ms, 1.16 PFLOP/s
// (a library product of bf16 matrices: 1.23).  Few rows: the reading of B, 8192 x 8192 for one row in 14.8 us, 4.5 TB/s.
#include <algorithm>

#include "aq_fp8.h"

#pragma clang diagnostic ignored "-Wint-to-pointer-cast"  // LDS addresses have 32 bits; the host pass does not know
#pragma clang diagnostic ignored "-Winline-asm"  // m0 among the clobbers: no register for the allocator, but instruction selection writes it too

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
    int splits, split_blocks;  // fp8_matmul_large_kernel: K in `splits` parts of `split_blocks` blocks, sums to `part`
    float *part;
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

typedef __bf16 b8_t __attribute__((ext_vector_type(8)));
typedef __bf16 b2_t __attribute__((ext_vector_type(2)));
__device__ inline b8_t codes_to_bf16(int lo, int hi, float scale)
{
    const b2_t a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, scale, true);
    const b2_t c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, scale, true);
    return b8_t{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// MODE: POW2, or the block's own sum (FP32S, EXACT)
template <int MODE> __device__ inline f4_t block_product(const i8_t &b, const i8_t &a, f4_t acc, int sb, int sa)
{
    if (MODE == POW2) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, acc, 0, 0, 0, sb, 0, sa);
    f4_t s = {0.f, 0.f, 0.f, 0.f};
    if (MODE == FP32S) return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, s, 0, 0, 0, 127, 0, 127);
#pragma unroll
    for (int i = 0; i < 4; ++i) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_to_fp16(b[2 * i], b[2 * i + 1]), codes_to_fp16(a[2 * i], a[2 * i + 1]), s, 0, 0, 0);
    return s;
}

// |scale| may be multiplied with another such one: 2^-63 .. 2^63, whose products are normal fp32 numbers (0, infinities and NaN are
// outside as well)
__device__ inline bool outside(uint32_t bits) { return (bits & 0x7fffffffu) - 0x20000000u > 0x3f000000u; }
// acc + sum * sa * sb for scales of any value.  Where sa * sb is no normal number, the mantissas are multiplied and the exponents added:
// a sum of zeros stays zero, and what the scales bring back to an ordinary size is kept.
__device__ inline float add_scaled(float acc, float sum, float sa, float sb)
{
    const float s = sa * sb, a = fabsf(s);
    if (a >= 0x1p-126f && a < __builtin_inff()) return __builtin_fmaf(sum, s, acc);
    const float m = __builtin_amdgcn_frexp_mantf(sa) * __builtin_amdgcn_frexp_mantf(sb);
    return acc + __builtin_ldexpf(sum * m, __builtin_amdgcn_frexp_expf(sa) + __builtin_amdgcn_frexp_expf(sb));
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

typedef float f16_t __attribute__((ext_vector_type(16)));

// 64 lanes x 16 bytes (or one byte, widened to four, or four) from base + off (per lane) to LDS address lds + 16 * lane (4 * lane).  Inline,
// because the compiler would wait for every such load before any LDS read that follows; the wait is written where the
// pipeline needs it.
__device__ inline void load_to_lds(uint32_t lds, uint32_t off, const uint8_t *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
__device__ inline void load_byte_to_lds(uint32_t lds, uint32_t off, const uint8_t *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_ubyte %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
__device__ inline void load_word_to_lds(uint32_t lds, uint32_t off, const uint8_t *base)
{
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, %2" ::"s"(lds), "v"(off), "s"(base) : "m0", "memory");
}
template <typename P> __device__ inline uint32_t lds_address(P *p) { return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) P *)p; }

// tile number -> tile: each XCD (workgroups go round the 8 of them) takes a contiguous run of numbers, and a run walks the
// tile grid in bands of 8 tile rows, so that the workgroups of an XCD share operand panels in its L2
__device__ inline void tile_of(uint32_t id, uint32_t tiles_m, uint32_t tiles_n, int &tm, int &tn)
{
    const uint32_t total = tiles_m * tiles_n, share = total / 8, rest = total % 8, xcd = id % 8;
    const uint32_t t = xcd * share + min(xcd, rest) + id / 8;
    const uint32_t band = t / (8 * tiles_n), height = min(8u, tiles_m - band * 8), in = t - band * 8 * tiles_n;
    tm = (int)(band * 8 + in % height);
    tn = (int)(in / height);
}

// Large products with power-of-two scales.  NS stages of LDS, each a block of K of all tile rows; WM x WN wavefronts.  Half a block
// (64 codes) is multiplied from registers while the next half is read from LDS:
//   half 0 of block b:  read half 1 of b;  then wait for block b + 1 in LDS, and for everybody to have read b;
//   half 1 of block b:  load block b + NS into the stage that b has left;  read half 0 of b + 1.
// Reads, loads and matrix instructions stand in the order written (the scheduling fences hold them there): a fragment of B is
// overwritten by its successor right behind its last use, those of A alternate between two sets.
template <int BM, int BN, int WM, int WN, int NS, bool SPLIT, typename T>
__global__ __launch_bounds__(WM *WN * 64, WM *WN / 4) void fp8_matmul_large_kernel(MatArgs p)
{
    constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;  // 32 x 32 fragments of a wavefront
    constexpr int LOADS = (BM + BN) / 8 / WAVES;                          // 1 KiB loads of 8 rows per wavefront and block
    constexpr int SLOADS = ((BM + BN) / 64 + WAVES - 1) / WAVES;          // loads of 64 scales per wavefront and block, at most
    constexpr int STAGE = (BM + BN) * FP8_BLK;
    static_assert((BM + BN) % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0 && BM % 64 == 0 && BN % 64 == 0, "");
    static_assert(BM * BN * 2 <= NS * STAGE, "the output tile passes through the stages");
    __shared__ __attribute__((aligned(128))) uint8_t tile[NS * STAGE];
    __shared__ uint32_t scale[NS][BM + BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    const uint32_t tiles = p.tiles_m * p.tiles_n, part = SPLIT ? blockIdx.x / tiles : 0;
    tile_of(SPLIT ? blockIdx.x - part * tiles : blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    if (SPLIT) {  // this part of K as if it were the whole
        const int first = (int)part * p.split_blocks;
        p.a += (long long)first * FP8_BLK;
        p.b += (long long)first * FP8_BLK;
        p.as = static_cast<const uint8_t *>(p.as) + first;
        p.bs = static_cast<const uint8_t *>(p.bs) + first;
        p.K = min(p.K - first * FP8_BLK, p.split_blocks * FP8_BLK);
    }
    // the last tile of a row or column moves back inside the matrix (M >= BM, N >= BN): it computes some outputs again, the same way
    const int m0 = min(tm * BM, p.M - BM), n0 = min(tn * BN, p.N - BN);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK, kround = (p.K + 15) & ~15;

    // 16-byte chunk c of tile row r lies at place c ^ (r / 2 & 7): the 16 rows that a fragment reads at a time lie in different
    // banks.
    const int chunk = ((lane & 7) ^ (4 * (wave & 1) + (lane >> 4))) * 16;
    const uint32_t aoff = (uint32_t)(lane >> 3) * (uint32_t)p.lda, boff = (uint32_t)(lane >> 3) * (uint32_t)p.ldb;
    const uint8_t *abase = p.a + (long long)(m0 + wave * 8) * p.lda, *bbase = p.b + (long long)(n0 + wave * 8) * p.ldb;
    const uint32_t lds0 = lds_address(tile) + wave * 1024, slds0 = lds_address(&scale[0][0]) + wave * 256;
    // load i of block kb; what lies past a row's end reads the block's first chunk, masked below
    auto fetch = [&](int i, int kb, int stage) {
        const int k = kb * FP8_BLK, r = i * WAVES * 8;
        const uint32_t c = k + chunk < kround ? chunk : 0;
        if (r < BM) load_to_lds(lds0 + (stage * BM + r) * FP8_BLK, aoff + c, abase + (long long)r * p.lda + k);
        else load_to_lds(lds0 + (NS * BM + stage * BN + r - BM) * FP8_BLK, boff + c, bbase + (long long)(r - BM) * p.ldb + k);
    };
    uint32_t soff[SLOADS];
    const uint8_t *sbase[SLOADS];
#pragma unroll
    for (int i = 0; i < SLOADS; ++i) {
        const int r = min((i * WAVES + wave) * 64, BM + BN - 64);  // (the wavefront's 64 rows are all A's or all B's)
        const bool is_a = r < BM;
        const int first = is_a ? m0 + r : n0 + r - BM, shift = is_a ? p.ashift : p.bshift;
        const long long ld = is_a ? p.ldas : p.ldbs;
        sbase[i] = static_cast<const uint8_t *>(is_a ? p.as : p.bs) + (long long)(first >> shift) * ld;
        soff[i] = (uint32_t)(((first + lane) >> shift) - (first >> shift)) * (uint32_t)ld;
    }
    auto fetch_scales = [&](int kb, int stage) {
#pragma unroll
        for (int i = 0; i < SLOADS; ++i)
            if ((BM + BN) % (64 * WAVES) == 0 || (i * WAVES + wave) * 64 < BM + BN) load_byte_to_lds(slds0 + stage * (BM + BN) * 4 + i * WAVES * 256, soff[i], sbase[i] + kb);
    };

    f16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    // LDS: A of all stages, then B of all, so that stage and fragment are constants in the reads' offset field; one address for
    // each 16-byte part of a half and operand (kept in registers: the compiler would otherwise keep many more)
    const int row = lane & 31, gg = lane >> 5;
    const int o = row * FP8_BLK + ((gg ^ (row >> 1 & 7)) * 16);
    uint32_t aread[4], bread[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {
        aread[x] = lds_address(tile) + wm * FP8_BLK + (o ^ (32 * x));
        bread[x] = lds_address(tile) + (NS * BM + wn) * FP8_BLK + (o ^ (32 * x));
        asm("" : "+v"(aread[x]), "+v"(bread[x]));
    }
    typedef const __attribute__((address_space(3))) i4_t *lds_i4;
    typedef const __attribute__((address_space(3))) uint32_t *lds_u1;
    auto read_a = [&](int i, int stage, int h) {
        const i4_t lo = *(lds_i4)(aread[2 * h] + stage * BM * FP8_BLK + i * 4096), hi = *(lds_i4)(aread[2 * h + 1] + stage * BM * FP8_BLK + i * 4096);
        return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    auto read_b = [&](int j, int stage, int h) {
        const i4_t lo = *(lds_i4)(bread[2 * h] + stage * BN * FP8_BLK + j * 4096), hi = *(lds_i4)(bread[2 * h + 1] + stage * BN * FP8_BLK + j * 4096);
        return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    uint32_t asread = lds_address(&scale[0][0]) + (wm + row) * 4, bsread = lds_address(&scale[0][0]) + (BM + wn + row) * 4;
    asm("" : "+v"(asread), "+v"(bsread));
    auto read_sa = [&](int i, int stage) { return *(lds_u1)(asread + stage * (BM + BN) * 4 + i * 128); };
    auto read_sb = [&](int j, int stage) { return *(lds_u1)(bsread + stage * (BM + BN) * 4 + j * 128); };
    i8_t a0[TM], a1[TM], b[TN];
    uint32_t sa[TM], sb[TN], sa1[TM];
    // the matrix instructions of a half; next(t): what goes out behind the t-th of them
    auto multiply = [&](const i8_t(&a)[TM], auto next) {
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                acc[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a[i], acc[i][j], 0, 0, 0, (int)sb[j], 0, (int)sa[i]);
                next(j * TM + i);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    constexpr int LPER = (LOADS + TM * TN - 1) / (TM * TN);
    auto block = [&](int kb, int stage) {
        multiply(a0, [&](int t) {
            if (t < TM) a1[t] = read_a(t, stage, 1);
            if (t % TM == TM - 1) b[t / TM] = read_b(t / TM, stage, 1);
        });
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * LOADS) : "memory");  // block kb + 1 is here, NS - 2 later ones on their way
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        multiply(a1, [&](int t) {
            if (t < TM) {
                a0[t] = read_a(t, (stage + 1) % NS, 0);
                sa1[t] = read_sa(t, (stage + 1) % NS);
            }
            if (t % TM == TM - 1) {
                b[t / TM] = read_b(t / TM, (stage + 1) % NS, 0);
                sb[t / TM] = read_sb(t / TM, (stage + 1) % NS);
            }
#pragma unroll
            for (int e = 0; e < LPER; ++e)
                if (t * LPER + e < LOADS) fetch(t * LPER + e, min(kb + NS, nkb - 1), stage);
            if (t == TM * TN - 1) fetch_scales(min(kb + NS, nkb - 1), stage);
        });
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i] = sa1[i];
    };

#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) fetch(i, min(s, nkb - 1), s);
        fetch_scales(min(s, nkb - 1), s);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * LOADS) : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    auto begin = [&](int stage) {
#pragma unroll
        for (int i = 0; i < TM; ++i) a0[i] = read_a(i, stage, 0), sa[i] = read_sa(i, stage);
#pragma unroll
        for (int j = 0; j < TN; ++j) b[j] = read_b(j, stage, 0), sb[j] = read_sb(j, stage);
    };
    // Zeros in LDS for what lies at K or behind it in the last block.  Everybody has it in LDS when it is cut, and reads its first half
    // again.
    auto cut = [&](int kb, int stage) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        for (int t = tid; t < (BM + BN) * 8; t += WAVES * 64) {
            const int r = t >> 3, c = t & 7, k = kb * FP8_BLK + 16 * c;
            if (k + 16 <= p.K) continue;
            i4_t *at = reinterpret_cast<i4_t *>(tile + (r < BM ? (stage * BM + r) * FP8_BLK : (NS * BM + stage * BN + r - BM) * FP8_BLK) + (c ^ (r >> 1 & 7)) * 16);
            *at = mask16(*at, k, p.K);
        }
        __syncthreads();
        begin(stage);
    };
    begin(0);
    const int whole = p.K / FP8_BLK;
    int kb = 0;
    for (; kb + NS <= whole; kb += NS) {
#pragma unroll
        for (int s = 0; s < NS; ++s) block(kb + s, s);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (kb + s < nkb) {
            if (kb + s >= whole) cut(kb + s, s);
            block(kb + s, s);
        }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();

    if (SPLIT) {
        float *to = p.part + (long long)part * p.M * p.N;
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < TM; ++i)
                    *reinterpret_cast<f4_any *>(to + (long long)(m0 + wm + 32 * i + row) * p.N + n0 + wn + 32 * j + 8 * q + 4 * gg) =
                        f4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
        return;
    }
    // Through LDS to rows: a wavefront's part of the tile, 16-byte chunk c of its row m at place c ^ (m & mask), then whole rows of
    // it leave with 16 bytes a lane.
    constexpr int CH = BN / WN / 8;  // chunks of a row
    T *out = reinterpret_cast<T *>(tile) + wave * (BM / WM) * (BN / WN);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = 32 * j + 8 * q + 4 * gg;
            f4_t bias = {0.f, 0.f, 0.f, 0.f};
            if (p.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n0 + wn + n + e < p.N) bias[e] = p.bias[n0 + wn + n + e];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const int m = 32 * i + row;
                const f4_t v = f4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]} + bias;
                *reinterpret_cast<u2_t *>(out + m * (BN / WN) + ((n / 8) ^ (m & (CH - 1))) * 8 + 4 * gg) = u2_t{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
            }
        }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    T *y = static_cast<T *>(p.y);
    const int c = lane & (CH - 1);
#pragma unroll
    for (int i = 0; i < BM / WM * CH / 64; ++i) {
        const int m = i * (64 / CH) + lane / CH, gm = m0 + wm + m, gn = n0 + wn + 8 * c, left = p.N - gn;
        const u4_t v = *reinterpret_cast<const u4_t *>(out + m * (BN / WN) + (c ^ (m & (CH - 1))) * 8);
        T *to = y + (long long)gm * p.ldy + gn;
        if (left >= 8) *reinterpret_cast<u4_any *>(to) = v;
        else
#pragma unroll
            for (int e = 0; e < 7; ++e)
                if (e < left) to[e] = T{(uint16_t)(v[e >> 1] >> 16 * (e & 1))};
    }
}

// The kernels below multiply the scales of a block in fp32, or put them into bf16 values.  Wavefronts that meet scales so far from 1 that
// this loses something compute, behind their stores, the outputs of these rows and columns again, block by block from memory with
// add_scaled().  Which outputs that are depends on the scales of their own row and column alone, so that tiles that overlap leave the
// same values.
// Where there are no such scales the watch costs 1 to 2 % (any scales, 4096^3: 16-bit output 83 -> 85 us, fp32 150 -> 153 us; 64 x 8192 x 4096 18.2 -> 18.8 us).
// power-of-two scales with which all codes are bf16 numbers: the smallest code is 2^-9 and bf16's smallest step 2^-133, the largest code 448
constexpr uint32_t BF16_LOW = 127 - 124, BF16_HIGH = 127 + 119;
template <typename T> __device__ inline void careful_part(const MatArgs &p, int m0, int n0, int lane)
{
    asm volatile("" : "+v"(lane));  // (nothing of this is worked out ahead, in registers that the kernel's own loop needs)
    auto far = [&](const void *s, long long i) {
        if (p.scale_f32) {
            const uint32_t u = static_cast<const uint32_t *>(s)[i], v = u & 0x7fffffffu;
            return outside(u) && v != 0 && v < 0x7f800000u;
        }
        const uint32_t e = static_cast<const uint8_t *>(s)[i];
        return e < BF16_LOW || (e > BF16_HIGH && e != 255);
    };
    const long long as = (long long)((m0 + lane) >> p.ashift) * p.ldas, bs = (long long)(min(n0 + lane, p.N - 1) >> p.bshift) * p.ldbs;
    bool row_far = false, col_far = false;
    for (int kb = 0; kb * FP8_BLK < p.K; ++kb) row_far |= far(p.as, as + kb), col_far |= far(p.bs, bs + kb);
    const uint64_t rows = __ballot(row_far), cols = __ballot(col_far);
    if (!(rows | cols)) return;  // (zeros, infinities or NaN)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores of the same outputs
    const int r = lane & 15, g = lane >> 4, kround = (p.K + 15) & ~15;
    auto piece = [&](const uint8_t *row, int k) {
        i4_t v = {0, 0, 0, 0};
        if (k < kround) v = *reinterpret_cast<const i4_t *>(row + k);
        return mask16(v, k, p.K);
    };
    auto fragment = [&](const uint8_t *row, int k) {
        const i4_t lo = piece(row, k + 16 * g), hi = piece(row, k + 16 * g + 64);
        return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
#pragma unroll 1
    for (int f = 0; f < 16; ++f) {  // 16 x 16 outputs: four columns n of row m in every lane
        const uint32_t fr = (uint32_t)(rows >> 16 * (f & 3)) & 0xffff, fc = (uint32_t)(cols >> 16 * (f >> 2)) & 0xffff;
        if (!(fr | fc)) continue;
        const int m = m0 + 16 * (f & 3) + r, nf = n0 + 16 * (f >> 2), n = nf + 4 * g;
        const uint8_t *ar = p.a + (long long)m * p.lda, *br = p.b + (long long)min(nf + r, p.N - 1) * p.ldb;
        f4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
        for (int kb = 0; kb * FP8_BLK < p.K; ++kb) {
            const f4_t sum = block_product<EXACT>(fragment(br, kb * FP8_BLK), fragment(ar, kb * FP8_BLK), acc, 0, 0);
            const float sa = load_scale(p.as, (long long)(m >> p.ashift) * p.ldas + kb, p.scale_f32);
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[e] = add_scaled(acc[e], sum[e], sa, load_scale(p.bs, (long long)(min(n + e, p.N - 1) >> p.bshift) * p.ldbs + kb, p.scale_f32));
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < p.N && ((fr >> r | fc >> (4 * g + e)) & 1))
                static_cast<T *>(p.y)[(long long)m * p.ldy + n + e] = from_f32<T>(p.bias ? acc[e] + p.bias[n + e] : acc[e]);
    }
}

// Large products with scales of any value and fp32 outputs: the tile's blocks of K in two stages of LDS as above; per block and pair of
// fragments the block's sum from zero, through fp16, then acc += sum * (sA * sB).
template <int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM *WN * 64, 2) void fp8_matmul_block_kernel(const MatArgs p)
{
    constexpr int WAVES = WM * WN, TM = BM / WM / 32, TN = BN / WN / 32;
    constexpr int LOADS = (BM + BN) / 8 / WAVES, STAGE = (BM + BN) * FP8_BLK;
    static_assert((BM + BN) % (8 * WAVES) == 0 && BM % (8 * WAVES) == 0 && BM + BN <= WAVES * 64, "");
    static_assert(TM == 2 && TN == 2, "careful_part() has 64 x 64 outputs");
    __shared__ __attribute__((aligned(128))) uint8_t tile[2 * STAGE];
    __shared__ __attribute__((aligned(16))) float scale[2][BM + BN];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = min(tm * BM, p.M - BM), n0 = min(tn * BN, p.N - BN);
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK, kround = (p.K + 15) & ~15;
    const int chunk = ((lane & 7) ^ (4 * (wave & 1) + (lane >> 4))) * 16;
    const uint32_t aoff = (uint32_t)(lane >> 3) * (uint32_t)p.lda, boff = (uint32_t)(lane >> 3) * (uint32_t)p.ldb;
    const uint8_t *abase = p.a + (long long)(m0 + wave * 8) * p.lda, *bbase = p.b + (long long)(n0 + wave * 8) * p.ldb;
    const uint32_t lds0 = lds_address(tile) + wave * 1024;
    auto fetch = [&](int kb, int stage) {
        const int k = kb * FP8_BLK;
        const uint32_t c = k + chunk < kround ? chunk : 0;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int r = i * WAVES * 8;
            if (r < BM) load_to_lds(lds0 + stage * STAGE + r * FP8_BLK, aoff + c, abase + (long long)r * p.lda + k);
            else load_to_lds(lds0 + stage * STAGE + r * FP8_BLK, boff + c, bbase + (long long)(r - BM) * p.ldb + k);
        }
    };
    // the scale of one tile row per thread
    const void *ssrc = nullptr;
    long long sfirst = 0;
    if (tid < BM) ssrc = p.as, sfirst = (long long)((m0 + tid) >> p.ashift) * p.ldas;
    else if (tid < BM + BN) ssrc = p.bs, sfirst = (long long)((n0 + tid - BM) >> p.bshift) * p.ldbs;
    auto read_scale = [&](int kb) { return tid < BM + BN ? static_cast<const float *>(ssrc)[sfirst + kb] : 1.0f; };
    bool far = false;  // one of the scales that passed through this thread is outside()

    f16_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
    const int row = lane & 31, gg = lane >> 5;
    const int o = row * FP8_BLK + ((gg ^ (row >> 1 & 7)) * 16);
    constexpr int W = 4;  // matrix instructions of a half block
    struct half_t {
        h8_t fp16[W];
    };
    auto read_half = [&](const uint8_t *t, int kb, int h, bool tail) {
        i4_t lo = *reinterpret_cast<const i4_t *>(t + (o ^ (64 * h))), hi = *reinterpret_cast<const i4_t *>(t + (o ^ (64 * h) ^ 32));
        if (tail) {
            lo = mask16(lo, kb * FP8_BLK + 64 * h + 16 * gg, p.K);
            hi = mask16(hi, kb * FP8_BLK + 64 * h + 16 * gg + 32, p.K);
        }
        return half_t{{codes_to_fp16(lo[0], lo[1]), codes_to_fp16(lo[2], lo[3]), codes_to_fp16(hi[0], hi[1]), codes_to_fp16(hi[2], hi[3])}};
    };
    auto block = [&](int kb, int stage, bool tail) {
        const uint8_t *ta = tile + stage * STAGE + wm * FP8_BLK, *tb = tile + stage * STAGE + (BM + wn) * FP8_BLK;
        half_t a[TM][2];
        float sa[TM];
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            sa[i] = scale[stage][wm + 32 * i + row];
            a[i][0] = read_half(ta + i * 4096, kb, 0, tail);
            a[i][1] = read_half(ta + i * 4096, kb, 1, tail);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const half_t b0 = read_half(tb + j * 4096, kb, 0, tail), b1 = read_half(tb + j * 4096, kb, 1, tail);
            f16_t sum[TM];
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) sum[i][e] = 0.0f;
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int i = 0; i < TM; ++i) sum[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b0.fp16[w], a[i][0].fp16[w], sum[i], 0, 0, 0);
#pragma unroll
            for (int w = 0; w < W; ++w)
#pragma unroll
                for (int i = 0; i < TM; ++i) sum[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(b1.fp16[w], a[i][1].fp16[w], sum[i], 0, 0, 0);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f4_t sb = *reinterpret_cast<const f4_t *>(&scale[stage][BM + wn + 32 * j + 8 * q + 4 * gg]);
#pragma unroll
                for (int i = 0; i < TM; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = __builtin_fmaf(sum[i][4 * q + e], sa[i] * sb[e], acc[i][j][4 * q + e]);
            }
        }
    };

    fetch(0, 0);
    const float first = read_scale(0);
    if (tid < BM + BN) scale[0][tid] = first;
    far |= outside(__float_as_uint(first));
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    for (int kb = 0; kb < nkb; ++kb) {
        const int stage = kb & 1;
        // the next block's scale is asked for before its codes, so that the wait for the one is not a wait for the other
        const float next = kb + 1 < nkb ? read_scale(kb + 1) : 1.0f;
        if (kb + 1 < nkb) fetch(kb + 1, stage ^ 1);
        if ((kb + 1) * FP8_BLK <= p.K) block(kb, stage, false);
        else block(kb, stage, true);
        if (tid < BM + BN) scale[stage ^ 1][tid] = next;
        far |= outside(__float_as_uint(next));
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    }
    const bool watch = __syncthreads_or(far);
    float *y = static_cast<float *>(p.y);
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wn + 32 * j + 8 * q + 4 * gg;
            f4_t bias = {0.f, 0.f, 0.f, 0.f};
            if (p.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) bias[e] = p.bias[n + e];
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                const f4_t v = {acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
                store4(y + (long long)(m0 + wm + 32 * i + row) * p.ldy + n, 4, v + bias);
            }
        }
    if (watch) careful_part<float>(p, m0 + wm, n0 + wn, lane);
}

// Large products with scales of any value and 16-bit outputs: tiles of 128 x BN, wavefronts with 64 x 64 each, loads and reads
// as in fp8_matmul_large_kernel with NS stages of LDS.  A block's sums start from zero in half 0 and are complete after half 1; they are scaled into the
// accumulators in half 0 of the next block, each right before its registers are needed again, while the matrix instruction of
// the one before runs.  BTILE: B's scales are of 128 x 128 tiles, one for the 32 columns of a fragment (tiles start at multiples of 32
// columns: the last one of a row reaches past N, reads row N - 1 there and stores nothing).
template <int BN, int NS, bool BTILE, typename T>
__global__ __launch_bounds__(BN * 2, 2) void fp8_matmul_scaled_kernel(const MatArgs p)
{
    constexpr int BM = 128, WAVES = BN / 32, LOADS = (BM + BN) / 8 / WAVES, STAGE = (BM + BN) * FP8_BLK;
    __shared__ __attribute__((aligned(128))) uint8_t tile[NS * STAGE];
    __shared__ __attribute__((aligned(16))) float scale[4][WAVES * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = min(tm * BM, p.M - BM), n0 = min(tn * BN, (p.N + 31) / 32 * 32 - BN);
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK, kround = (p.K + 15) & ~15, whole = p.K / FP8_BLK;

    const int chunk = ((lane & 7) ^ (4 * (wave & 1) + (lane >> 4))) * 16;
    const uint32_t aoff = (uint32_t)(lane >> 3) * (uint32_t)p.lda;
    const uint8_t *abase = p.a + (long long)(m0 + wave * 8) * p.lda, *bbase = p.b + (long long)n0 * p.ldb;
    const int brow = wave * 8 + (lane >> 3), blast = p.N - 1 - n0;
    const uint32_t lds0 = lds_address(tile) + wave * 1024;
    auto fetch = [&](int i, int kb, int stage) {
        const int k = kb * FP8_BLK, r = i * WAVES * 8;
        const uint32_t c = k + chunk < kround ? chunk : 0;
        if (r < BM) load_to_lds(lds0 + stage * STAGE + r * FP8_BLK, aoff + c, abase + (long long)r * p.lda + k);
        else load_to_lds(lds0 + stage * STAGE + r * FP8_BLK, (uint32_t)min(r - BM + brow, blast) * (uint32_t)p.ldb + c, bbase + k);
    };
    // 64 scales for each of the first six wavefronts (the others load some again, to a place that nobody reads)
    const int srow = min(wave * 64, BM + BN - 64);
    const int sfirst = srow < BM ? m0 + srow : n0 + srow - BM, sshift = srow < BM ? p.ashift : p.bshift;
    const long long sld = srow < BM ? p.ldas : p.ldbs;
    const int slast = (srow < BM ? p.M : p.N) - 1;
    const uint8_t *sbase = reinterpret_cast<const uint8_t *>(static_cast<const float *>(srow < BM ? p.as : p.bs) + (long long)(min(sfirst, slast) >> sshift) * sld);
    const uint32_t soff = (uint32_t)((min(sfirst + lane, slast) >> sshift) - (min(sfirst, slast) >> sshift)) * (uint32_t)sld * 4;
    const uint32_t slds0 = lds_address(&scale[0][0]) + wave * 256;
    auto fetch_scales = [&](int kb) { load_word_to_lds(slds0 + (kb & 3) * WAVES * 256, soff, sbase + (long long)min(kb, nkb - 1) * 4); };
    f16_t acc[2][2], sum[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = sum[i][j][e] = 0.0f;
    const int row = lane & 31, gg = lane >> 5;
    const uint32_t o = row * FP8_BLK + ((gg ^ (row >> 1 & 7)) * 16);
    const uint32_t aread = lds_address(tile) + wm * FP8_BLK + o, bread = lds_address(tile) + (BM + wn) * FP8_BLK + o;
    typedef const __attribute__((address_space(3))) i4_t *lds_i4;
    auto read = [&](uint32_t base, int f, int stage, int h) {
        uint32_t p0 = base, p1;
        if (h) asm volatile("v_xor_b32 %0, 64, %1" : "=v"(p0) : "v"(base));
        if (h) asm volatile("v_xor_b32 %0, 0x60, %1" : "=v"(p1) : "v"(base));
        else asm volatile("v_xor_b32 %0, 32, %1" : "=v"(p1) : "v"(base));
        const i4_t lo = *(lds_i4)(p0 + stage * STAGE + f * 4096), hi = *(lds_i4)(p1 + stage * STAGE + f * 4096);
        return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    // scales of the block whose sums wait: of this lane's rows m, and (BTILE) of the fragments' columns; before the first block zeros
    float sa[2] = {0.f, 0.f}, sb[2] = {0.f, 0.f};
    if (!BTILE) scale[3][tid] = 0.0f;
    float least = 1.0f, most = 1.0f;  // magnitudes of this wavefront's scales
    auto read_scales = [&](int kb) {
        const float *sc = scale[kb & 3];
        sa[0] = sc[wm + row], sa[1] = sc[wm + 32 + row];
        float b0, b1;
        if (BTILE) b0 = sb[0] = sc[BM + wn], b1 = sb[1] = sc[BM + wn + 32];
        else b0 = b1 = sc[BM + wn + lane];
        least = fminf(fminf(fminf(least, fabsf(sa[0])), fminf(fabsf(sa[1]), fabsf(b0))), fabsf(b1));
        most = fmaxf(fmaxf(fmaxf(most, fabsf(sa[0])), fmaxf(fabsf(sa[1]), fabsf(b0))), fabsf(b1));
    };
    // sums of block kb into the accumulators
    auto scale_in = [&](int i, int j, int kb) {
        if (BTILE) {
            const float s = sa[i] * sb[j];
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = __builtin_fmaf(sum[i][j][e], s, acc[i][j][e]);
        } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f4_t v = *reinterpret_cast<const f4_t *>(&scale[kb & 3][BM + wn + 32 * j + 8 * q + 4 * gg]);
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] = __builtin_fmaf(sum[i][j][4 * q + e], sa[i] * v[e], acc[i][j][4 * q + e]);
            }
        }
    };
    i8_t a0[2], a1[2], b[2];
    auto block = [&](int kb, int stage) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int i = t & 1, j = t >> 1;
            scale_in(i, j, kb - 1);
            sum[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a0[i], f16_t{}, 0, 0, 0, 127, 0, 127);
            if (t < 2) a1[t] = read(aread, t, stage, 1);
            if (i == 1) b[j] = read(bread, j, stage, 1);
            __builtin_amdgcn_sched_barrier(0);
        }
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * (LOADS + 1)) : "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const int i = t & 1, j = t >> 1;
            sum[i][j] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(b[j], a1[i], sum[i][j], 0, 0, 0, 127, 0, 127);
            if (t == 0) read_scales(kb);
            if (t < 2) a0[t] = read(aread, t, (stage + 1) % NS, 0);
            if (i == 1) b[j] = read(bread, j, (stage + 1) % NS, 0);
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (2 * t + e < LOADS) fetch(2 * t + e, min(kb + NS, nkb - 1), stage);
            if (t == 3) fetch_scales(kb + NS);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) fetch(i, min(s, nkb - 1), s);
        fetch_scales(s);
    }
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 1) * (LOADS + 1)) : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    auto begin = [&](int stage) {
#pragma unroll
        for (int f = 0; f < 2; ++f) a0[f] = read(aread, f, stage, 0), b[f] = read(bread, f, stage, 0);
    };
    // zeros for what lies at K or behind it in the last block, whose first half is then read again
    auto cut = [&](int kb, int stage) {
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        for (int t = tid; t < (BM + BN) * 8; t += WAVES * 64) {
            const int r = t >> 3, c = t & 7, k = kb * FP8_BLK + 16 * c;
            if (k + 16 <= p.K) continue;
            i4_t *at = reinterpret_cast<i4_t *>(tile + stage * STAGE + r * FP8_BLK + (c ^ (r >> 1 & 7)) * 16);
            *at = mask16(*at, k, p.K);
        }
        __syncthreads();
        begin(stage);
    };
    begin(0);
    int kb = 0;
    for (; kb + NS <= whole; kb += NS) {
#pragma unroll
        for (int s = 0; s < NS; ++s) block(kb + s, s);
    }
#pragma unroll
    for (int s = 0; s < NS; ++s)
        if (kb + s < nkb) {
            if (kb + s >= whole) cut(kb + s, s);
            block(kb + s, s);
        }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
#pragma unroll
    for (int t = 0; t < 4; ++t) scale_in(t & 1, t >> 1, nkb - 1);
    const bool watch = __any(outside(__float_as_uint(least)) || outside(__float_as_uint(most)));
    T *y = static_cast<T *>(p.y);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wn + 32 * j + 8 * q + 4 * gg;
            f4_t bias = {0.f, 0.f, 0.f, 0.f};
            if (p.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < p.N) bias[e] = p.bias[n + e];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                store4(y + (long long)(m0 + wm + 32 * i + row) * p.ldy + n, p.N - n,
                       f4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]} + bias);
        }
    if (watch) careful_part<T>(p, m0 + wm, n0 + wn, lane);
}

// Large products with power-of-two scales and fp32 outputs: tiles of 128 x BN, wavefronts with 64 x 64 each.  K in half blocks of 64;
// three things go on at once, one behind each of the 16 matrix instructions of a half:
//   the matrix instructions of half s;  the conversion to bf16 of half s + 1, four codes' pairs at a time;  the LDS reads of half s + 2,
//   into the registers that the conversion has emptied.
// At the start of block b, block b + 1 is in LDS, everybody has read b, and the load of b + NS takes its place.
template <int BN, int NS>
__global__ __launch_bounds__(BN * 2, 2) void fp8_matmul_wide_kernel(const MatArgs p)
{
    constexpr int BM = 128, WAVES = BN / 32, LOADS = (BM + BN) / 8 / WAVES, STAGE = (BM + BN) * FP8_BLK;
    __shared__ __attribute__((aligned(128))) uint8_t tile[NS * STAGE];
    __shared__ uint32_t scale[NS][WAVES * 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int tm, tn;
    tile_of(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
    const int m0 = min(tm * BM, p.M - BM), n0 = min(tn * BN, p.N - BN);
    const int wm = (wave & 1) * 64, wn = (wave >> 1) * 64;
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK, kround = (p.K + 15) & ~15, whole = p.K / FP8_BLK;

    const int chunk = ((lane & 7) ^ (4 * (wave & 1) + (lane >> 4))) * 16;  // as in fp8_matmul_large_kernel
    const uint32_t aoff = (uint32_t)(lane >> 3) * (uint32_t)p.lda, boff = (uint32_t)(lane >> 3) * (uint32_t)p.ldb;
    const uint8_t *abase = p.a + (long long)(m0 + wave * 8) * p.lda, *bbase = p.b + (long long)(n0 + wave * 8) * p.ldb;
    const uint32_t lds0 = lds_address(tile) + wave * 1024;
    auto fetch = [&](int i, int kb, int stage) {
        const int k = kb * FP8_BLK, r = i * WAVES * 8;
        const uint32_t c = k + chunk < kround ? chunk : 0;
        if (r < BM) load_to_lds(lds0 + stage * STAGE + r * FP8_BLK, aoff + c, abase + (long long)r * p.lda + k);
        else load_to_lds(lds0 + stage * STAGE + r * FP8_BLK, boff + c, bbase + (long long)(r - BM) * p.ldb + k);
    };
    // 64 scales for each of the first six wavefronts (the others load some again, to a place that nobody reads)
    const int srow = min(wave * 64, BM + BN - 64);
    const int sfirst = srow < BM ? m0 + srow : n0 + srow - BM, sshift = srow < BM ? p.ashift : p.bshift;
    const long long sld = srow < BM ? p.ldas : p.ldbs;
    const uint8_t *sbase = static_cast<const uint8_t *>(srow < BM ? p.as : p.bs) + (long long)(sfirst >> sshift) * sld;
    const uint32_t soff = (uint32_t)(((sfirst + lane) >> sshift) - (sfirst >> sshift)) * (uint32_t)sld;
    const uint32_t slds0 = lds_address(&scale[0][0]) + wave * 256;
    auto fetch_scales = [&](int kb, int stage) {
        load_byte_to_lds(slds0 + stage * WAVES * 256, soff, sbase + kb);
    };
    auto cut = [&](int kb, int stage) {  // zeros for what lies at K or behind it
        for (int t = tid; t < (BM + BN) * 8; t += WAVES * 64) {
            const int r = t >> 3, c = t & 7, k = kb * FP8_BLK + 16 * c;
            if (k + 16 <= p.K) continue;
            i4_t *at = reinterpret_cast<i4_t *>(tile + stage * STAGE + r * FP8_BLK + (c ^ (r >> 1 & 7)) * 16);
            *at = mask16(*at, k, p.K);
        }
        __syncthreads();
    };

    f16_t acc[2][2];
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

    const int row = lane & 31, gg = lane >> 5;
    const uint32_t o = row * FP8_BLK + ((gg ^ (row >> 1 & 7)) * 16);
    const uint32_t aread = lds_address(tile) + wm * FP8_BLK + o, bread = lds_address(tile) + (BM + wn) * FP8_BLK + o;
    typedef const __attribute__((address_space(3))) i4_t *lds_i4;
    typedef const __attribute__((address_space(3))) uint32_t *lds_u1;
    const uint32_t asread = lds_address(&scale[0][0]) + (wm + row) * 4, bsread = lds_address(&scale[0][0]) + (BM + wn + row) * 4;
    // fragments: 0, 1 of A, 2, 3 of B
    i4_t raw[4][2];
    b8_t even[4][4], odd[4][4];
    uint32_t sc[NS][4];
    auto read_raw = [&](int f, int stage, int h) {
        const uint32_t base = f < 2 ? aread : bread;
        uint32_t p0 = base, p1;  // (turned at the read: there are no registers to keep the four addresses)
        if (h) asm volatile("v_xor_b32 %0, 64, %1" : "=v"(p0) : "v"(base));
        if (h) asm volatile("v_xor_b32 %0, 0x60, %1" : "=v"(p1) : "v"(base));
        else asm volatile("v_xor_b32 %0, 32, %1" : "=v"(p1) : "v"(base));
        raw[f][0] = *(lds_i4)(p0 + stage * STAGE + (f & 1) * 4096);
        raw[f][1] = *(lds_i4)(p1 + stage * STAGE + (f & 1) * 4096);
    };
    uint32_t least = 127, most = 127;
    auto read_scales = [&](int stage) {
#pragma unroll
        for (int f = 0; f < 4; ++f) sc[stage][f] = *(lds_u1)((f < 2 ? asread : bsread) + stage * WAVES * 256 + (f & 1) * 128);
#pragma unroll
        for (int f = 0; f < 4; ++f) least = min(least, sc[stage][f]), most = max(most, sc[stage][f]);
    };
    auto convert = [&](b8_t(&to)[4][4], int f, int w, uint32_t s) {  // (the conversion takes the exponent field alone: 2^(b - 127) for b = 0 too)
        to[f][w] = codes_to_bf16(raw[f][w >> 1][2 * (w & 1)], raw[f][w >> 1][2 * (w & 1) + 1], __uint_as_float(s << 23));
    };
    auto half = [&](const b8_t(&now)[4][4], b8_t(&next)[4][4], const uint32_t(&s)[4], int rstage, int h, int kb, int fstage) {
#pragma unroll
        for (int t = 0; t < 16; ++t) {
            const int w = t >> 2, i = t >> 1 & 1, j = t & 1;
            acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(now[2 + j][w], now[i][w], acc[i][j], 0, 0, 0);
            convert(next, t >> 2, t & 3, s[t >> 2]);
            if ((t & 3) == 3) read_raw(t >> 2, rstage, h);
            if (h == 0 && t < LOADS) fetch(t, min(kb + NS, nkb - 1), fstage);
            if (h == 0 && t == LOADS) fetch_scales(min(kb + NS, nkb - 1), fstage);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto block = [&](int kb, int stage) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((NS - 2) * (LOADS + 1)) : "memory");
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if (kb + 1 == whole && whole < nkb) cut(kb + 1, (stage + 1) % NS);
        read_scales((stage + 1) % NS);
        half(even, odd, sc[stage], (stage + 1) % NS, 0, kb, stage);
        half(odd, even, sc[(stage + 1) % NS], (stage + 1) % NS, 1, kb, stage);
    };

#pragma unroll
    for (int s = 0; s < NS; ++s) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) fetch(i, min(s, nkb - 1), s);
        fetch_scales(min(s, nkb - 1), s);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NS - 1) * (LOADS + 1)) : "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (whole == 0) cut(0, 0);
    read_scales(0);
#pragma unroll
    for (int f = 0; f < 4; ++f) {
        read_raw(f, 0, 0);
#pragma unroll
        for (int w = 0; w < 4; ++w) convert(even, f, w, sc[0][f]);
        read_raw(f, 0, 1);
    }
    for (int kb = 0; kb < nkb; kb += NS) {
#pragma unroll
        for (int s = 0; s < NS; ++s)
            if (kb + s < nkb) block(kb + s, s);
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    const bool watch = __any(least < BF16_LOW || most > BF16_HIGH);
    float *y = static_cast<float *>(p.y);
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = n0 + wn + 32 * j + 8 * q + 4 * gg;
            f4_t bias = {0.f, 0.f, 0.f, 0.f};
            if (p.bias)
#pragma unroll
                for (int e = 0; e < 4; ++e) bias[e] = p.bias[n + e];
#pragma unroll
            for (int i = 0; i < 2; ++i)
                *reinterpret_cast<f4_any *>(y + (long long)(m0 + wm + 32 * i + row) * p.ldy + n) =
                    f4_t{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]} + bias;
        }
    if (watch) careful_part<float>(p, m0 + wm, n0 + wn, lane);
}

// Few rows: bound by the reading of B.  A workgroup has 16 TN columns and 16 TM rows, its wavefronts share out the blocks of K, U
// neighbouring ones at a time with all their loads in flight, fragments straight from memory (a row's 128 bytes come in one
// piece); the wavefronts' sums meet in LDS, in a fixed order.
template <int TM, int TN, int U, int MODE, typename T>
__global__ __launch_bounds__(512, 2) void fp8_matmul_rows_kernel(const MatArgs p)
{
    constexpr int WAVES = 8;
    __shared__ __attribute__((aligned(16))) f4_t sums[WAVES][TM * TN][64];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n0 = (int)(blockIdx.x % p.tiles_n) * 16 * TN, m0 = (int)(blockIdx.x / p.tiles_n) * 16 * TM;
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK, kround = (p.K + 15) & ~15;
    const int r = lane & 15, g = lane >> 4;
    // rows past the end read the last row (their results are not stored)
    const uint8_t *arow[TM], *brow[TN];
    long long as[TM], bs[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int m = min(m0 + 16 * i + r, p.M - 1);
        arow[i] = p.a + (long long)m * p.lda + 16 * g;
        as[i] = (long long)(m >> p.ashift) * p.ldas;
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) {
        const int n = min(n0 + 16 * j + r, p.N - 1);
        brow[j] = p.b + (long long)n * p.ldb + 16 * g;
        bs[j] = (long long)(n >> p.bshift) * p.ldbs;
    }
    f4_t acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f4_t{0.f, 0.f, 0.f, 0.f};

    auto load_scale_bits = [&](const void *s, long long i) -> uint32_t {
        return MODE == POW2 ? static_cast<const uint8_t *>(s)[i] : __float_as_uint(load_scale(s, i, p.scale_f32));
    };
    auto multiply = [&](const i8_t(&af)[TM], const i8_t(&bf)[TN], const uint32_t(&sa)[TM], const uint32_t(&sb)[TN]) {
        bool far = false;
        if (MODE != POW2) {
#pragma unroll
            for (int i = 0; i < TM; ++i) far |= outside(sa[i]);
#pragma unroll
            for (int j = 0; j < TN; ++j) far |= outside(sb[j]);
            far = __any(far);
        }
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            if (MODE == POW2) {
#pragma unroll
                for (int i = 0; i < TM; ++i) acc[i][j] = block_product<MODE>(bf[j], af[i], acc[i][j], (int)sb[j], (int)sa[i]);
            } else {
                f4_t sn;  // the scales of the four columns that this lane's results belong to
#pragma unroll
                for (int e = 0; e < 4; ++e) sn[e] = __uint_as_float(__shfl((int)sb[j], 4 * g + e, 64));
#pragma unroll
                for (int i = 0; i < TM; ++i) {
                    const f4_t s = block_product<MODE>(bf[j], af[i], acc[i][j], 0, 0);
                    if (far) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) acc[i][j][e] = add_scaled(acc[i][j][e], s[e], __uint_as_float(sa[i]), sn[e]);
                        continue;
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[i][j][e] = __builtin_fmaf(s[e], sn[e] * __uint_as_float(sa[i]), acc[i][j][e]);
                }
            }
        }
    };
    const int whole = p.K / FP8_BLK;
    for (int kb = wave * U; kb < nkb; kb += WAVES * U) {
        if (kb + U <= whole) {
            i8_t af[U][TM], bf[U][TN];
            uint32_t sa[U][TM], sb[U][TN];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = (kb + u) * FP8_BLK;
                auto fragment = [&](const uint8_t *row) {
                    const i4_t lo = *reinterpret_cast<const i4_t *>(row + k), hi = *reinterpret_cast<const i4_t *>(row + k + 64);
                    return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                };
#pragma unroll
                for (int j = 0; j < TN; ++j) bf[u][j] = fragment(brow[j]), sb[u][j] = load_scale_bits(p.bs, bs[j] + kb + u);
#pragma unroll
                for (int i = 0; i < TM; ++i) af[u][i] = fragment(arow[i]), sa[u][i] = load_scale_bits(p.as, as[i] + kb + u);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) multiply(af[u], bf[u], sa[u], sb[u]);
            continue;
        }
        for (int at = kb; at < min(kb + U, nkb); ++at) {  // the last blocks; what lies past the row's end reads as zero
            const int k = at * FP8_BLK;
            auto fragment = [&](const uint8_t *row) {
                i4_t lo = {0, 0, 0, 0}, hi = {0, 0, 0, 0};
                if (k + 16 * g < kround) lo = *reinterpret_cast<const i4_t *>(row + k);
                if (k + 16 * g + 64 < kround) hi = *reinterpret_cast<const i4_t *>(row + k + 64);
                lo = mask16(lo, k + 16 * g, p.K);
                hi = mask16(hi, k + 16 * g + 64, p.K);
                return i8_t{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            };
            i8_t af[TM], bf[TN];
            uint32_t sa[TM], sb[TN];
#pragma unroll
            for (int j = 0; j < TN; ++j) bf[j] = fragment(brow[j]), sb[j] = load_scale_bits(p.bs, bs[j] + at);
#pragma unroll
            for (int i = 0; i < TM; ++i) af[i] = fragment(arow[i]), sa[i] = load_scale_bits(p.as, as[i] + at);
            multiply(af, bf, sa, sb);
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) sums[wave][i * TN + j][lane] = acc[i][j];
    __syncthreads();
    T *y = static_cast<T *>(p.y);
    for (int t = tid; t < TM * TN * 64; t += 512) {
        const int f = t >> 6, l = t & 63, m = m0 + 16 * (f / TN) + (l & 15), n = n0 + 16 * (f % TN) + 4 * (l >> 4);
        f4_t v = sums[0][f][l];
#pragma unroll
        for (int w = 1; w < WAVES; ++w) v += sums[w][f][l];
        if (p.bias)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (n + e < p.N) v[e] += p.bias[n + e];
        if (m < p.M) store4(y + (long long)m * p.ldy + n, p.N - n, v);
    }
}

template <int TM, int TN, int U, int MODE, typename T> static void launch_rows(MatArgs p, hipStream_t st)
{
    p.tiles_m = (p.M + 16 * TM - 1) / (16 * TM);
    p.tiles_n = (p.N + 16 * TN - 1) / (16 * TN);
    hipLaunchKernelGGL((fp8_matmul_rows_kernel<TM, TN, U, MODE, T>), dim3(p.tiles_m * p.tiles_n), dim3(512), 0, st, p);
}

// y = the sum of the parts of K, in their order, + bias; four columns a thread
template <typename T>
__global__ __launch_bounds__(256) void fp8_matmul_join_kernel(const float *__restrict__ part, int splits, int M, int N, const float *__restrict__ bias,
                                                              T *__restrict__ y, long long ldy)
{
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x, quads = (N + 3) / 4;
    const int m = (int)(t / quads), n = (int)(t - m * quads) * 4;
    if (m >= M) return;
    const float *p = part + (long long)m * N + n;
    f4_t v = {0.f, 0.f, 0.f, 0.f};
    if (n + 4 <= N) {
#pragma unroll 4
        for (int s = 0; s < splits; ++s) v += *reinterpret_cast<const f4_any *>(p + (long long)s * M * N);
    } else {
        for (int s = 0; s < splits; ++s)
            for (int e = 0; n + e < N; ++e) v[e] += p[(long long)s * M * N + e];
    }
    if (bias)
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (n + e < N) v[e] += bias[n + e];
    store4(y + (long long)m * ldy + n, N - n, v);
}

template <int BM, int BN, int WM, int WN, int NS, typename T> static void launch_large(MatArgs p, hipStream_t st)
{
    p.tiles_m = (p.M + BM - 1) / BM;
    p.tiles_n = (p.N + BN - 1) / BN;
    hipLaunchKernelGGL((fp8_matmul_large_kernel<BM, BN, WM, WN, NS, false, T>), dim3(p.tiles_m * p.tiles_n), dim3(WM * WN * 64), 0, st, p);
}

static long long tiles_of(long long M, long long N, long long bm, long long bn) { return (M + bm - 1) / bm * ((N + bn - 1) / bn); }
// Parts of K for the 64 x 128 tiles: as many as bring the launch to 256 workgroups, none shorter than four blocks.  Writing and joining
// them costs 8 to 10 us and a block of K 0.4 us, so they have to save 24 blocks (256 x 2048 x 8192, 64 tiles: 27 -> 16 us; 128 x 8192 x 8192,
// 128 tiles: 28 -> 23 us; 256 x 4096 x 4096, 128 tiles: 17 us whole, 19 us in two parts).
static int matmul_splits(long long M, long long N, long long K)
{
    const long long tiles = tiles_of(M, N, 64, 128), nkb = (K + FP8_BLK - 1) / FP8_BLK;
    if (M <= 64 || N < 128 || tiles > 128) return 1;
    const long long parts = std::min(256 / tiles, nkb / 4);
    return parts > 1 && nkb * (parts - 1) / parts >= 24 ? (int)parts : 1;
}

// Tiles by how many of them there are for the 256 compute units (times at 4096-long rows unless stated):
//   256 x 256 from three quarters of a round on (4096 x 4096: 57 us against 75 us in 128 x 128; 2048 x 4096, half a round: 47 against 38).
//   Products so large that they run at the power limit (2^38 multiplications and more) with four wavefronts of 128 x 128, which read a third less
//   from LDS, smaller ones with eight of 64 x 128, whose waits overlap (8192^3: 429 against 462 us, 16384 x 8192 x 2048: 270 against 285 us;
//   8192 x 8192 x 2048: 120 against 117.5 us, 5000^3: 145 against 141 us).
//   Not for a round and a few tiles more (2316 x 6403 x 1632, 260 tiles: 58 us, 44 us in 128 x 128; 4352 x 4096 x 1024, 272: 33.5 against 30 us;
//   from 321 on again: 5120 x 4352 x 1024, 340: 34.6 against 35.2 us, 4608 x 4864 x 2048, 342: 53.5 against 54, 4096 x 6144 x 4096, 384: 95 against 101 us);
//   128 x 128 with two stages, two workgroups on a unit, for more than a round (1500 x 5000 x 2560: 25 us against 30 us with four stages);
//   128 x 128 with four stages for up to a round (1024 x 4096: 22 against 28 us with two);
//   64 x 128 for fewer (512 x 4096: 17 us; 1000 x 1000 x 1000: 8 against 11 us), K in parts for very few.
template <typename T> static void launch_pow2(MatArgs p, hipStream_t st)
{
    if (p.N < 128) return launch_rows<4, 2, 2, POW2, T>(p, st);
    const long long big = tiles_of(p.M, p.N, 256, 256);
    if (p.M >= 256 && p.N >= 256 && big >= 192 && (big <= 256 || big > 320))
        return (double)p.M * p.N * p.K >= 0x1p38 ? launch_large<256, 256, 2, 2, 2, T>(p, st) : launch_large<256, 256, 4, 2, 2, T>(p, st);
    if (p.M >= 128 && tiles_of(p.M, p.N, 128, 128) > 256) return launch_large<128, 128, 2, 2, 2, T>(p, st);
    if (p.M >= 128 && tiles_of(p.M, p.N, 64, 128) > 256) return launch_large<128, 128, 2, 2, 4, T>(p, st);
    const int splits = matmul_splits(p.M, p.N, p.K), nkb = (p.K + FP8_BLK - 1) / FP8_BLK;
    if (splits == 1) return launch_large<64, 128, 1, 4, 4, T>(p, st);
    p.split_blocks = (nkb + splits - 1) / splits;
    p.splits = (nkb + p.split_blocks - 1) / p.split_blocks;
    p.tiles_m = (p.M + 63) / 64;
    p.tiles_n = (p.N + 127) / 128;
    hipLaunchKernelGGL((fp8_matmul_large_kernel<64, 128, 1, 4, 4, true, T>), dim3(p.tiles_m * p.tiles_n * p.splits), dim3(256), 0, st, p);
    const long long quads = (long long)p.M * ((p.N + 3) / 4);
    hipLaunchKernelGGL((fp8_matmul_join_kernel<T>), dim3((unsigned)((quads + 255) / 256)), dim3(256), 0, st, p.part, p.splits, p.M, p.N, p.bias,
                       static_cast<T *>(p.y), p.ldy);
}

template <int MODE, typename T> static void launch_block(MatArgs p, hipStream_t st)
{
    // Two workgroups of 128 x 128 on a compute unit run past each other's barriers (fp32 output 512 x 4096 x 4096: 30 us against 46 us for one
    // of 128 x 256, any scales 28 against 34 us); with scales in fp32 arithmetic the larger tile wins once there are two
    // rounds of it (4096^3: 16-bit output 84 against 86 us, fp32 output 152 against 191 us).  In one nearly full round it gains where the
    // round is full and loses where it is not (16-bit output, 1500 x 5000 x 2560, 240 tiles: 34.4 against 31.5 us; 2048 x 4096 x 4096, 256: 43
    // against 45.5 us), and is not taken.
    const bool wide = p.scale_f32 && p.N >= 256 && tiles_of(p.M, p.N, 128, 256) >= 512;
    p.tiles_m = (p.M + 127) / 128;
    p.tiles_n = wide ? (p.N + 255) / 256 : (p.N + 127) / 128;
    const dim3 g(p.tiles_m * p.tiles_n);
    if constexpr (MODE == EXACT) {
        if (wide) hipLaunchKernelGGL((fp8_matmul_block_kernel<128, 256, 2, 4>), g, dim3(512), 0, st, p);
        else if (p.scale_f32) hipLaunchKernelGGL((fp8_matmul_block_kernel<128, 128, 2, 2>), g, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((fp8_matmul_wide_kernel<128, 2>), g, dim3(256), 0, st, p);
    } else if (wide) {
        if (p.bshift) hipLaunchKernelGGL((fp8_matmul_scaled_kernel<256, 3, true, T>), g, dim3(512), 0, st, p);
        else hipLaunchKernelGGL((fp8_matmul_scaled_kernel<256, 3, false, T>), g, dim3(512), 0, st, p);
    } else {
        if (p.bshift) hipLaunchKernelGGL((fp8_matmul_scaled_kernel<128, 2, true, T>), g, dim3(256), 0, st, p);
        else hipLaunchKernelGGL((fp8_matmul_scaled_kernel<128, 2, false, T>), g, dim3(256), 0, st, p);
    }
}

// Streamed fragments: the smallest tiles whose workgroups fit the 256 compute units once, since a workgroup's time goes with the rows of A and
// B that it reads (128 x 1024 x 4096: 9.1 us in 16 x 32, 11.2 in 32 x 32, 16 in 64 x 32, 10.8 in 64 x 128 and parts of K; 64 x 1000 x 2048: 5.8 us
// in 16 x 16, 8.6 in 64 x 16; 64 x 8192 x 4096: 17 us in 64 x 32, 19 in 32 x 32, 26 in 64 x 16).  Up to 16 rows the reading of B is all, which
// two rounds of narrow tiles do as fast (1 x 8192 x 8192: 14.8 us, 17.8 in 16 x 32).  With more than 64 rows, power-of-two scales and long rows
// the parts of K win (512 x 512 x 8192: 15.6 against 19 us).  False: there are more, and other kernels for them.
template <int MODE, typename T> static bool launch_streamed(const MatArgs &p, hipStream_t st)
{
    const int nkb = (p.K + FP8_BLK - 1) / FP8_BLK;
    const bool parts = MODE == POW2 && p.M > 64;
    auto once = [&](int bm, int bn, int most) { return tiles_of(p.M, p.N, bm, bn) <= 256 && (!parts || nkb <= most); };
    if (once(16, 16, 64) || (p.M <= 16 && tiles_of(p.M, p.N, 16, 16) <= 512)) launch_rows<1, 1, 4, MODE, T>(p, st);
    else if (once(16, 32, 64) || p.M <= 16) launch_rows<1, 2, 4, MODE, T>(p, st);
    else if (once(32, 32, 32) || p.M <= 32) launch_rows<2, 2, MODE == POW2 ? 4 : 2, MODE, T>(p, st);
    else if (p.M <= 64) launch_rows<4, 2, 2, MODE, T>(p, st);
    else return false;
    return true;
}

template <int MODE, typename T> static void launch_matmul(MatArgs p, hipStream_t st)
{
    if (launch_streamed<MODE, T>(p, st)) return;
    if constexpr (MODE == POW2) {
        launch_pow2<T>(p, st);
    } else {
        // Tiles of 64 x 32 that fit once are still streamed (512 x 1024 x 4096: 19 us, in 32 x 32 23 us, through LDS 28 us; 512 x 2048 x 4096: 35 us,
        // through LDS 28 us); fp32 outputs with any scales, whose LDS kernel is the slowest, for twice as many (36 against 48 us).
        const long long few = MODE == EXACT && p.scale_f32 ? 512 : 256;
        if (p.M < 128 || p.N < 128 || tiles_of(p.M, p.N, 64, 32) <= few) return launch_rows<4, 2, 2, MODE, T>(p, st);
        launch_block<MODE, T>(p, st);
    }
}

} // namespace aq

extern "C" {

size_t aq_fp8_matmul_workspace_bytes(long long M, long long N, long long K)
{
    if (M <= 0 || N <= 0 || K <= 0) return 0;
    const int splits = aq::matmul_splits(M, N, K);
    return splits == 1 ? 0 : (size_t)splits * (size_t)M * (size_t)N * sizeof(float);
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
    // a launch holds fewer than 2^32 threads; offsets within a tile have 32 bits
    AQ_REQUIRE(M < (1LL << 26) && N < (1LL << 26) && M * N < (1LL << 38), -E2BIG, "aq_fp8_matmul: M=%lld N=%lld K=%lld is too large for one call", M, N, K);
    AQ_REQUIRE(lda < (1LL << 24) && ldb < (1LL << 24), -E2BIG, "aq_fp8_matmul: a pitch of %lld bytes is too large", std::max(lda, ldb));
    AQ_REQUIRE(ldas < (1LL << 24) && ldbs < (1LL << 24), -E2BIG, "aq_fp8_matmul: a pitch of %lld scales is too large", std::max(ldas, ldbs));
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
                       scale_type == AQ_SCALE_F32, 0, 0, 1, 0, static_cast<float *>(workspace)};
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (ytype == AQ_F32) launch_matmul<EXACT, float>(p, st);
    else if (scale_type == AQ_SCALE_POW2) ytype == AQ_BF16 ? launch_matmul<POW2, bf16_el>(p, st) : launch_matmul<POW2, f16_el>(p, st);
    else ytype == AQ_BF16 ? launch_matmul<FP32S, bf16_el>(p, st) : launch_matmul<FP32S, f16_el>(p, st);
    return check_launch("aq_fp8_matmul");
}

} // extern "C"

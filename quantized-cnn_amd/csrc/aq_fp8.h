// Shared pieces of the 8-bit floating point kernels: element types, vector access, the power-of-two block scale.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "../../include/aq_hip.h"
#include "aq_common.h"

namespace aq {

constexpr int FP8_BLK = 128;  // elements along a row that share a scale

typedef float f4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
typedef float f2_t __attribute__((ext_vector_type(2)));

struct bf16_el { uint16_t b; };
struct f16_el { uint16_t b; };
struct e4m3_el { uint8_t b; };

__device__ inline float to_f32(float v) { return v; }
__device__ inline float to_f32(bf16_el v) { return __uint_as_float((uint32_t)v.b << 16); }
__device__ inline float to_f32(f16_el v) { return (float)__builtin_bit_cast(_Float16, v.b); }
__device__ inline float to_f32(e4m3_el v) { return __builtin_amdgcn_cvt_f32_fp8((int)v.b, 0); }
template <typename T> __device__ inline T from_f32(float v);
template <> __device__ inline float from_f32<float>(float v) { return v; }
template <> __device__ inline bf16_el from_f32<bf16_el>(float v) { return bf16_el{__builtin_bit_cast(uint16_t, (__bf16)v)}; }
template <> __device__ inline f16_el from_f32<f16_el>(float v) { return f16_el{__builtin_bit_cast(uint16_t, (_Float16)v)}; }

// Eight neighbouring elements, at any address that is a multiple of the element's size: the global memory path takes 16-byte
// accesses at any address, so rows of odd lengths need no variant of their own.
typedef f4_t f4_any __attribute__((aligned(4)));
typedef u4_t u4_any __attribute__((aligned(2)));
typedef u2_t u2_any __attribute__((aligned(1)));
__device__ inline void load8(const float *p, float (&v)[8])
{
    const f4_t a = *reinterpret_cast<const f4_any *>(p), b = *reinterpret_cast<const f4_any *>(p + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = a[i], v[4 + i] = b[i];
}
__device__ inline void load8(const bf16_el *p, float (&v)[8])
{
    const u4_t a = *reinterpret_cast<const u4_any *>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(a[i] << 16), v[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
}
__device__ inline void load8(const f16_el *p, float (&v)[8])
{
    typedef _Float16 h8 __attribute__((ext_vector_type(8)));
    const h8 a = __builtin_bit_cast(h8, (u4_t) * reinterpret_cast<const u4_any *>(p));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)a[i];
}
__device__ inline void load8(const e4m3_el *p, float (&v)[8])
{
    const u2_t a = *reinterpret_cast<const u2_any *>(p);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const f2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)a[i], true);
        v[4 * i] = lo[0], v[4 * i + 1] = lo[1], v[4 * i + 2] = hi[0], v[4 * i + 3] = hi[1];
    }
}
template <typename T> __device__ inline uint32_t pack2(float a, float b) { return (uint32_t)from_f32<T>(a).b | (uint32_t)from_f32<T>(b).b << 16; }
// the same, eight elements as they lie in memory (half the registers for 16-bit types), and their values one by one
template <typename T> struct raw8 { u4_t a; };
template <> struct raw8<float> { f4_t a, b; };
template <> struct raw8<e4m3_el> { u2_t a; };
#define AQ_ACCESS(V, ANY)                                                                                                     \
    template <bool NT> __device__ inline V load_any(const ANY *p) { return NT ? __builtin_nontemporal_load(p) : *p; }            \
    template <bool NT> __device__ inline void store_any(V v, ANY *p)                                                             \
    {                                                                                                                            \
        if (NT) __builtin_nontemporal_store(v, p);                                                                               \
        else *p = v;                                                                                                             \
    }
AQ_ACCESS(f4_t, f4_any)
AQ_ACCESS(u4_t, u4_any)
AQ_ACCESS(u2_t, u2_any)
#undef AQ_ACCESS
// NT: streaming (nontemporal) accesses, for calls that move more than the last-level cache holds
template <bool NT> __device__ inline raw8<float> load_raw(const float *p)
{
    return {load_any<NT>(reinterpret_cast<const f4_any *>(p)), load_any<NT>(reinterpret_cast<const f4_any *>(p + 4))};
}
template <bool NT> __device__ inline raw8<bf16_el> load_raw(const bf16_el *p) { return {load_any<NT>(reinterpret_cast<const u4_any *>(p))}; }
template <bool NT> __device__ inline raw8<f16_el> load_raw(const f16_el *p) { return {load_any<NT>(reinterpret_cast<const u4_any *>(p))}; }
template <bool NT> __device__ inline raw8<e4m3_el> load_raw(const e4m3_el *p) { return {load_any<NT>(reinterpret_cast<const u2_any *>(p))}; }
// the first n (0..8); the others zero
__device__ inline raw8<float> load_raw_n(const float *p, int n)
{
    if (n >= 8) return load_raw<false>(p);
    raw8<float> r = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) (i < 4 ? r.a : r.b)[i & 3] = p[i];
    return r;
}
template <typename T> __device__ inline raw8<T> load_raw_n(const T *p, int n)
{
    if (n >= 8) return load_raw<false>(p);
    constexpr int PER = 4 / sizeof(T);
    raw8<T> r = {};
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) r.a[i / PER] |= (uint32_t)p[i].b << 32 / PER * (i % PER);
    return r;
}
// A row's eight elements from column c, for rows of eight elements or more, whose end may lie within them or before them: the eight are
// read from where the row's last eight begin at the latest, so every lane has one whole access in flight and waits at its use,
// where row_chunk() moves the elements to their places and puts zeros behind the row's end.
template <bool NT, typename T> __device__ inline raw8<T> load_row_chunk(const T *row, long long c, long long cols)
{
    return load_raw<NT>(row + (c < cols - 8 ? c : cols - 8));
}
template <typename T> __device__ inline raw8<T> row_chunk(raw8<T> r, long long c, long long cols)
{
    const long long over = c - (cols - 8);
    if (over <= 0) return r;
    constexpr int N = 2 * sizeof(T);  // 32-bit words
    uint32_t w[N];
    __builtin_memcpy(w, &r, sizeof(w));
    const int bytes = over >= 8 ? 8 * (int)sizeof(T) : (int)over * (int)sizeof(T);
#pragma unroll
    for (int step = N; step >= 1; step >>= 1)
        if (bytes & 4 * step) {
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = i + step < N ? w[i + step < N ? i + step : 0] : 0;
        }
    const int bits = (bytes & 3) * 8;
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __builtin_amdgcn_alignbit(i + 1 < N ? w[i + 1 < N ? i + 1 : 0] : 0, w[i], bits);
    __builtin_memcpy(&r, w, sizeof(w));
    return r;
}
__device__ inline float value(const raw8<float> &r, int i) { return i < 4 ? r.a[i & 3] : r.b[i & 3]; }
__device__ inline float value(const raw8<bf16_el> &r, int i) { return __uint_as_float(i & 1 ? r.a[i >> 1] & 0xffff0000u : r.a[i >> 1] << 16); }
__device__ inline float value(const raw8<f16_el> &r, int i) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(r.a[i >> 1] >> 16 * (i & 1))); }
__device__ inline float value(const raw8<e4m3_el> &r, int i)
{
    const int w = (int)r.a[i >> 2];
    return (i & 3) == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0) : (i & 3) == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1)
         : (i & 3) == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2) : __builtin_amdgcn_cvt_f32_fp8(w, 3);
}
template <bool NT> __device__ inline void store8_any(float *p, const float (&v)[8])
{
    store_any<NT>(f4_t{v[0], v[1], v[2], v[3]}, reinterpret_cast<f4_any *>(p));
    store_any<NT>(f4_t{v[4], v[5], v[6], v[7]}, reinterpret_cast<f4_any *>(p + 4));
}
template <bool NT, typename T> __device__ inline void store8_any(T *p, const float (&v)[8])
{
    store_any<NT>(u4_t{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7])}, reinterpret_cast<u4_any *>(p));
}
// Calls that move more than this many bytes (half the last-level cache, the rest being what other kernels have there) stream.
// Measured at 134 + 134 MB of the quantiser: 66 us with plain accesses, 57 us streaming; at 34 + 34 MB no difference.  Rows that do
// not start at multiples of 16 bytes never stream: their accesses share lines, which streaming fetches again (norm backward,
// 4096 x 4097 bf16: 49 us streaming against 30).
constexpr long long STREAM_BYTES = 128LL << 20;

// the first n (0..8) of eight elements; the others read as zero and are not written
template <typename T> __device__ inline void load_n(const T *p, int n, float (&v)[8])
{
    if (n >= 8) {
        load8(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = 0.0f;
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) v[i] = to_f32(p[i]);
}
template <bool NT = false, typename T> __device__ inline void store_n(T *p, int n, const float (&v)[8])
{
    if (n >= 8) {
        store8_any<NT>(p, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) p[i] = from_f32<T>(v[i]);
}

// |v| where v is finite, 0 elsewhere
__device__ inline float finite_abs(float v)
{
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}
// Exponent e of the block scale 2^e, the smallest with amax <= 448 * 2^e: amax = (1 + f) 2^E, 448 = 1.75 * 2^8, so
// e = E - 8, one more where 1 + f > 1.75.  At least -126, the smallest whose scale and reciprocal are normal fp32 numbers.
__device__ inline int scale_exponent(float amax)
{
    const uint32_t b = __float_as_uint(amax);
    if (b == 0) return 0;
    const int e = (int)(b >> 23) - 127 - 8 + ((b & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < -126 ? -126 : e;
}
__device__ inline float exp2_int(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // -126 <= e <= 127
// four codes from four values that lie within +-448 (or are not finite: NaN)
__device__ inline uint32_t e4m3x4(float a, float b, float c, float d)
{
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
}
__device__ inline u2_t e4m3x8(const float (&v)[8], float inv)
{
    u2_t r;
    r[0] = e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv);
    r[1] = e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv);
    return r;
}
template <bool NT = false> __device__ inline void store_codes(uint8_t *p, int n, u2_t c)  // the first n (0..8) of eight codes
{
    if (n >= 8) {
        store_any<NT>(c, reinterpret_cast<u2_any *>(p));
        return;
    }
#pragma unroll
    for (int i = 0; i < 7; ++i)
        if (i < n) p[i] = (uint8_t)(c[i >> 2] >> 8 * (i & 3));
}
__device__ inline void store_scale(void *s, long long i, int e, int scale_f32)
{
    if (scale_f32) static_cast<float *>(s)[i] = exp2_int(e);
    else static_cast<uint8_t *>(s)[i] = (uint8_t)(e + 127);
}
// byte b of a power-of-two scale: 2^(b - 127); b = 0 is the subnormal 2^-127, 255 NaN
__device__ inline float pow2_scale(uint32_t b) { return b == 0 ? 0x1p-127f : b == 255 ? __builtin_nanf("") : __uint_as_float(b << 23); }
__device__ inline float load_scale(const void *s, long long i, int scale_f32)
{
    return scale_f32 ? static_cast<const float *>(s)[i] : pow2_scale(static_cast<const uint8_t *>(s)[i]);
}
// max over the 16 lanes of an aligned group of 16, of numbers that are not negative
__device__ inline float max16(float v)
{
    uint32_t u = __float_as_uint(v);
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) u = max(u, (uint32_t)__shfl_xor((int)u, m, 64));
    return __uint_as_float(u);
}
// Largest finite magnitude of eight values.  Magnitudes compare like their bit patterns as whole numbers, two 16-bit ones at a
// time; patterns from infinity on are not finite, and only where there is one the values are looked at singly.
__device__ inline float amax8(const float (&v)[8])
{
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    if (m < 0x7f800000u) return __uint_as_float(m);
    float a = 0.0f;
    for (int i = 0; i < 8; ++i) a = fmaxf(a, finite_abs(v[i]));
    return a;
}
typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
__device__ inline us2_t abs2(uint32_t w) { return __builtin_bit_cast(us2_t, w & 0x7fff7fffu); }
template <typename T> __device__ constexpr uint32_t infinity16() { return std::is_same<T, bf16_el>::value ? 0x7f80 : 0x7c00; }
template <typename T> __device__ inline float amax8(const raw8<T> &r)
{
    if constexpr (sizeof(T) == 2) {
        const us2_t m = __builtin_elementwise_max(__builtin_elementwise_max(abs2(r.a[0]), abs2(r.a[1])), __builtin_elementwise_max(abs2(r.a[2]), abs2(r.a[3])));
        const uint32_t u = max((uint32_t)m[0], (uint32_t)m[1]);
        if (u < infinity16<T>()) return to_f32(T{(uint16_t)u});
    }
    const float v[8] = {value(r, 0), value(r, 1), value(r, 2), value(r, 3), value(r, 4), value(r, 5), value(r, 6), value(r, 7)};
    return amax8(v);
}
// the same for each of the eight columns of eight rows
template <typename T> __device__ inline void column_amax8(const raw8<T> (&r)[8], float (&m)[8])
{
    if constexpr (sizeof(T) == 2) {
        us2_t c[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            c[k] = abs2(r[0].a[k]);
#pragma unroll
            for (int i = 1; i < 8; ++i) c[k] = __builtin_elementwise_max(c[k], abs2(r[i].a[k]));
        }
        const us2_t t = __builtin_elementwise_max(__builtin_elementwise_max(c[0], c[1]), __builtin_elementwise_max(c[2], c[3]));
        if (max((uint32_t)t[0], (uint32_t)t[1]) < infinity16<T>()) {
#pragma unroll
            for (int j = 0; j < 8; ++j) m[j] = to_f32(T{c[j >> 1][j & 1]});
            return;
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float v[8] = {value(r[0], j), value(r[1], j), value(r[2], j), value(r[3], j), value(r[4], j), value(r[5], j), value(r[6], j), value(r[7], j)};
        m[j] = amax8(v);
    }
}

inline bool rows16(const void *p, long long ld, int size) { return !p || (((uintptr_t)p & 15) == 0 && ld * size % 16 == 0); }

template <typename F> inline int by_type(int type, F f)
{
    return type == AQ_F32 ? f((float *)nullptr) : type == AQ_BF16 ? f((bf16_el *)nullptr) : f((f16_el *)nullptr);
}
inline bool is_type(int t) { return t == AQ_F32 || t == AQ_BF16 || t == AQ_F16; }
inline int type_size(int t) { return t == AQ_F32 ? 4 : 2; }

} // namespace aq

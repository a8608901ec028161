// Norm of all gradients of a model together, and clipping: norm = sqrt(sum g^2), g' = g * min(1, max_norm / (norm + 1e-6)).
// Squares are formed and summed in double (no overflow for large fp32 gradients, and the order does not show in the result's
// fp32 digits).  A tensor is cut into chunks and the chunks of all tensors are dealt to at most GRAD_PARTS workgroups, each of
// which leaves one partial sum.  The scaling launch adds the partial sums up again in every workgroup, in the same order
// everywhere: two launches for 64 tensors, no atomics, no host round trip.  Both passes are bound by memory bandwidth: 400 M fp32
// elements 246 us (1.6 GB, 6.5 TB/s) and 594 us (3.2 GB, 5.4 TB/s).  16-byte accesses that are neighbours across the lanes matter
// there: with two per lane side by side the streaming stores took 693 us.
#include <algorithm>

#include "aq_fp8.h"

namespace aq {

constexpr int GRAD_MAX = 64;           // tensors per launch (the table travels in the kernel arguments)
constexpr int GRAD_CHUNK = 256 * 32;   // elements
constexpr int GRAD_PARTS = 2048;       // workgroups of one summing launch
constexpr int GRAD_SELF = 4096;        // partial sums that every workgroup of the scaling launch adds up by itself

struct GradTab {
    const void *p[GRAD_MAX];
    void *o[GRAD_MAX];
    long long n[GRAD_MAX];
    int blk0[GRAD_MAX + 1];  // first chunk of every tensor
    uint8_t type[GRAD_MAX];
    int count;
};

__device__ inline int grad_tensor(const GradTab &t, int chunk)
{
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (chunk >= t.blk0[mid]) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ inline double grad_block_sum(double v, double *sh)  // 256 threads, fixed order, the same value in every thread
{
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    const double s = (sh[0] + sh[1]) + (sh[2] + sh[3]);
    __syncthreads();
    return s;
}

// 16 bytes of elements and their values
template <typename T> constexpr int PER16 = 16 / (int)sizeof(T);
__device__ inline float value16(u4_t v, int i, float) { return __uint_as_float(v[i]); }
__device__ inline float value16(u4_t v, int i, bf16_el) { return __uint_as_float(i & 1 ? v[i >> 1] & 0xffff0000u : v[i >> 1] << 16); }
__device__ inline float value16(u4_t v, int i, f16_el) { return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[i >> 1] >> 16 * (i & 1))); }

template <bool NT, typename T> __device__ inline double chunk_squares(const T *p, long long n)
{
    constexpr int P = PER16<T>, ITER = GRAD_CHUNK / (256 * P);
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    if (n >= GRAD_CHUNK) {
        u4_t v[ITER];
#pragma unroll
        for (int i = 0; i < ITER; ++i) v[i] = load_any<NT>(reinterpret_cast<const u4_any *>(p + (i * 256 + threadIdx.x) * P));
#pragma unroll
        for (int i = 0; i < ITER; ++i)
#pragma unroll
            for (int j = 0; j < P; ++j) {
                const double d = (double)value16(v[i], j, T{});
                s[j & 3] = __builtin_fma(d, d, s[j & 3]);
            }
    } else {
        for (int c = threadIdx.x; c < n; c += 256) {
            const double d = (double)to_f32(p[c]);
            s[0] = __builtin_fma(d, d, s[0]);
        }
    }
    return (s[0] + s[1]) + (s[2] + s[3]);
}

template <bool NT>
__global__ __launch_bounds__(256) void grad_squares_kernel(const GradTab t, double *__restrict__ part)
{
    __shared__ double sh[4];
    double s = 0.0;
    for (int c = blockIdx.x; c < t.blk0[t.count]; c += gridDim.x) {
        const int i = grad_tensor(t, c);
        const long long lo = (long long)(c - t.blk0[i]) * GRAD_CHUNK, n = t.n[i] - lo;
        if (t.type[i] == AQ_F32) s += chunk_squares<NT>(static_cast<const float *>(t.p[i]) + lo, n);
        else if (t.type[i] == AQ_BF16) s += chunk_squares<NT>(static_cast<const bf16_el *>(t.p[i]) + lo, n);
        else s += chunk_squares<NT>(static_cast<const f16_el *>(t.p[i]) + lo, n);
    }
    s = grad_block_sum(s, sh);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// out[0] = sum of the partial sums, norm[0] its root
__global__ __launch_bounds__(256) void grad_finish_kernel(const double *__restrict__ part, int n, double *__restrict__ out, float *__restrict__ norm)
{
    __shared__ double sh[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
    s = grad_block_sum(s, sh);
    if (threadIdx.x == 0) {
        if (out) out[0] = s;
        if (norm) norm[0] = (float)sqrt(s);
    }
}

template <bool NT, typename T> __device__ inline void chunk_scale(const T *p, T *o, long long n, float k)
{
    constexpr int P = PER16<T>, ITER = GRAD_CHUNK / (256 * P);
    if (n >= GRAD_CHUNK) {
        u4_t v[ITER];
#pragma unroll
        for (int i = 0; i < ITER; ++i) v[i] = load_any<NT>(reinterpret_cast<const u4_any *>(p + (i * 256 + threadIdx.x) * P));
#pragma unroll
        for (int i = 0; i < ITER; ++i) {
            u4_t r;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if constexpr (P == 4) r[j] = __float_as_uint(value16(v[i], j, T{}) * k);
                else r[j] = pack2<T>(value16(v[i], 2 * j, T{}) * k, value16(v[i], 2 * j + 1, T{}) * k);
            }
            store_any<NT>(r, reinterpret_cast<u4_any *>(o + (i * 256 + threadIdx.x) * P));
        }
        return;
    }
    for (int c = threadIdx.x; c < n; c += 256) o[c] = from_f32<T>(to_f32(p[c]) * k);
}

template <bool NT>
__global__ __launch_bounds__(256) void grad_scale_kernel(const GradTab t, const double *__restrict__ part, int nparts, double max_norm,
                                                         float *__restrict__ norm)
{
    __shared__ double sh[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < nparts; i += 256) s += part[i];
    const double total = sqrt(grad_block_sum(s, sh));
    if (norm && blockIdx.x == 0 && threadIdx.x == 0) norm[0] = (float)total;
    const double c = max_norm / (total + 1e-6);
    const float k = c >= 1.0 ? 1.0f : (float)c;  // (NaN stays NaN)
    // the last chunks first: they are what the caches still hold of the summing pass
    for (int b = t.blk0[t.count] - 1 - (int)blockIdx.x; b >= 0; b -= gridDim.x) {
        const int i = grad_tensor(t, b);
        if (k == 1.0f && t.p[i] == t.o[i]) continue;  // in place and not clipped
        const long long lo = (long long)(b - t.blk0[i]) * GRAD_CHUNK, n = t.n[i] - lo;
        if (t.type[i] == AQ_F32) chunk_scale<NT>(static_cast<const float *>(t.p[i]) + lo, static_cast<float *>(t.o[i]) + lo, n, k);
        else if (t.type[i] == AQ_BF16) chunk_scale<NT>(static_cast<const bf16_el *>(t.p[i]) + lo, static_cast<bf16_el *>(t.o[i]) + lo, n, k);
        else chunk_scale<NT>(static_cast<const f16_el *>(t.p[i]) + lo, static_cast<f16_el *>(t.o[i]) + lo, n, k);
    }
}

static long long grad_chunks(long long n) { return (n + GRAD_CHUNK - 1) / GRAD_CHUNK; }
// partial sums that the launch for tensors base .. base + GRAD_MAX - 1 leaves
static long long grad_parts(const long long *sizes, int base, int n)
{
    long long chunks = 0;
    for (int i = base; i < std::min(n, base + GRAD_MAX); ++i) chunks += grad_chunks(sizes[i]);
    return std::min<long long>(chunks, GRAD_PARTS);
}

} // namespace aq

extern "C" {

size_t aq_clip_grad_norm_workspace_bytes(const long long *sizes, int n)
{
    long long parts = 1;
    for (int base = 0; sizes && base < n; base += aq::GRAD_MAX) parts += aq::grad_parts(sizes, base, n);
    return (size_t)parts * sizeof(double);
}

int aq_clip_grad_norm(const void *const *tensors, void *const *outs, const long long *sizes, const int *types, int n, double max_norm,
                      float *norm, void *workspace, size_t workspace_bytes, void *stream)
{
    using namespace aq;
    AQ_REQUIRE(n >= 0 && (n == 0 || (tensors && sizes && types)) && norm, -EINVAL, "aq_clip_grad_norm: bad arguments");
    AQ_REQUIRE(!outs || max_norm >= 0, -EDOM, "aq_clip_grad_norm: max_norm=%g is negative", max_norm);
    for (int i = 0; i < n; ++i) {
        AQ_REQUIRE(types[i] == AQ_F32 || types[i] == AQ_BF16 || types[i] == AQ_F16, -EINVAL, "aq_clip_grad_norm: unknown element type %d", types[i]);
        AQ_REQUIRE(sizes[i] >= 0 && sizes[i] < (1LL << 37) && (sizes[i] == 0 || (tensors[i] && (!outs || outs[i]))), -EINVAL, "aq_clip_grad_norm: bad tensor %d", i);
    }
    const size_t need = aq_clip_grad_norm_workspace_bytes(sizes, n);
    AQ_REQUIRE(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 7) == 0, -ENOSPC,
               "aq_clip_grad_norm: workspace of %zu bytes (8-byte aligned) needed, %zu given", need, workspace_bytes);
    hipStream_t st = static_cast<hipStream_t>(stream);
    double *sum = static_cast<double *>(workspace), *part = sum + 1;
    auto table = [&](int base, GradTab &t) {
        long long chunks = 0;
        t.count = std::min(GRAD_MAX, n - base);
        for (int i = 0; i < t.count; ++i) {
            t.p[i] = tensors[base + i];
            t.o[i] = outs ? outs[base + i] : nullptr;
            t.n[i] = sizes[base + i];
            t.type[i] = (uint8_t)types[base + i];
            t.blk0[i] = (int)chunks;
            chunks += grad_chunks(sizes[base + i]);
        }
        t.blk0[t.count] = (int)chunks;
        return chunks;
    };
    long long total = 0, bytes = 0;
    for (int i = 0; i < n; ++i) bytes += sizes[i] * type_size(types[i]);
    const bool streaming = bytes > STREAM_BYTES;
    for (int base = 0; base < n; base += GRAD_MAX) {
        GradTab t = {};
        AQ_REQUIRE(table(base, t) < (1LL << 31) - GRAD_PARTS, -E2BIG, "aq_clip_grad_norm: too many elements");
        const long long parts = grad_parts(sizes, base, n);
        if (parts == 0) continue;
        if (streaming) hipLaunchKernelGGL((grad_squares_kernel<true>), dim3((unsigned)parts), dim3(256), 0, st, t, part + total);
        else hipLaunchKernelGGL((grad_squares_kernel<false>), dim3((unsigned)parts), dim3(256), 0, st, t, part + total);
        if (int rc = check_launch("aq_clip_grad_norm")) return rc;
        total += parts;
    }
    const bool self = outs && total > 0 && total <= GRAD_SELF;
    if (!self) {
        hipLaunchKernelGGL(grad_finish_kernel, dim3(1), dim3(256), 0, st, part, (int)total, sum, norm);
        if (int rc = check_launch("aq_clip_grad_norm")) return rc;
    }
    for (int base = 0; outs && base < n; base += GRAD_MAX) {
        GradTab t = {};
        const long long chunks = table(base, t);
        if (chunks == 0) continue;
        const dim3 g((unsigned)std::min<long long>(chunks, GRAD_PARTS));
        if (streaming) hipLaunchKernelGGL((grad_scale_kernel<true>), g, dim3(256), 0, st, t, self ? part : sum, self ? (int)total : 1, max_norm, self ? norm : nullptr);
        else hipLaunchKernelGGL((grad_scale_kernel<false>), g, dim3(256), 0, st, t, self ? part : sum, self ? (int)total : 1, max_norm, self ? norm : nullptr);
        if (int rc = check_launch("aq_clip_grad_norm")) return rc;
    }
    return 0;
}

} // extern "C"

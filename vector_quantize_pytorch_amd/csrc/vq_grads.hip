// vq_grads.hip -- the global norm of many gradients, and their clipping.
#include "vq_elem.h"

#include <algorithm>
#include <math.h>
#include <stdlib.h>

// norm = sqrt(sum of all squares): squares and sums in 64 bits, so that neither 1e30 nor 1e-30 leaves the range.  The tensors travel as
// kernel arguments, GRAD_TENSORS to a launch (4 KB of arguments); a tensor is cut into chunks, a workgroup and a partial sum each.
// Bound by HBM: one read for the norm, one read and one write to clip.  Clipping goes through the tensors from the last to the first, since
// the last ones read are the ones still in the memory-side cache.
#define GRAD_TENSORS 100
#define GRAD_CHUNK 4096            // (16384: 311 tensors of 90e6 elements 173 us of kernels instead of 159, 8 of 262144 15 instead of 12)
struct GradTensor { const void *src; void *dst; int64_t n; unsigned first; int dtype; };        // first: its first workgroup in the launch
struct GradArgs { GradTensor t[GRAD_TENSORS]; int count; };

__device__ __forceinline__ const GradTensor &grad_tensor(const GradArgs &a, unsigned block)
{
    int lo = 0, hi = a.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.t[mid].first <= block) lo = mid; else hi = mid - 1;
    }
    return a.t[lo];
}

__device__ double grad_block_sum(double v)
{
    __shared__ double red[16];
    v = vq_wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0;
    for (unsigned w = 0; w < blockDim.x / 64; ++w) v += red[w];
    return v;
}

// 16-byte loads, four in flight a thread (of a chunk's 512 vectors of a 16-bit type two are a thread's own, the other two read its first again);
// what is left of a tensor's end one by one
template <typename T> __device__ double grad_sumsq(const T *src, int64_t n)
{
    constexpr int N = 16 / sizeof(T);
    double s = 0.0;
    const int64_t whole = n / N;
    for (int64_t i = threadIdx.x; i < whole; i += 4 * 256) {
        VqVec<T, N> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
            v[u] = vq_ldv<T, N>(src + (i + u * 256 < whole ? i + u * 256 : i) * N);           // (unconditional: four in flight)
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * 256 < whole)
#pragma unroll
                for (int k = 0; k < N; ++k) { const double f = (double)(float)v[u].v[k]; s = fma(f, f, s); }
    }
    const int64_t i = whole * N + threadIdx.x;
    if (i < n) { const double f = (double)(float)src[i]; s = fma(f, f, s); }
    return s;
}

__global__ void __launch_bounds__(256) vq_grad_norm_kernel(const GradArgs a, double *partial)
{
    const GradTensor &t = grad_tensor(a, blockIdx.x);
    const int64_t at = (int64_t)(blockIdx.x - t.first) * GRAD_CHUNK, n = t.n - at < GRAD_CHUNK ? t.n - at : GRAD_CHUNK;
    double s = t.dtype == VQHIP_F32 ? grad_sumsq((const float *)t.src + at, n) : t.dtype == VQHIP_BF16 ? grad_sumsq((const __bf16 *)t.src + at, n) : grad_sumsq((const _Float16 *)t.src + at, n);
    s = grad_block_sum(s);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// norm, and coef = min(1, max_norm / (norm + eps)): one workgroup, 8 partial sums in flight a thread
__global__ void __launch_bounds__(1024) vq_grad_coef_kernel(const double *partial, int64_t n, double max_norm, double eps, float *norm, float *coef)
{
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += 8 * 1024) {
        double v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = i + u * 1024 < n ? partial[i + u * 1024] : 0.0;
#pragma unroll
        for (int u = 0; u < 8; ++u) s += v[u];
    }
    s = sqrt(grad_block_sum(s));
    if (threadIdx.x == 0) {
        const double c = max_norm == INFINITY && s == INFINITY ? 1.0 : max_norm / (s + eps);
        norm[0] = (float)s;
        coef[0] = c > 1.0 ? 1.f : (float)c;             // (a norm that is not a number: neither comparison holds, NaN goes through)
    }
}

template <typename T> __device__ void grad_scale(const T *src, T *dst, int64_t n, float coef)
{
    constexpr int N = 16 / sizeof(T);
    const int64_t whole = n / N;
    for (int64_t i = threadIdx.x; i < whole; i += 4 * 256) {
        VqVec<T, N> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = vq_ldv<T, N>(src + (i + u * 256 < whole ? i + u * 256 : i) * N);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i + u * 256 < whole) {
#pragma unroll
                for (int k = 0; k < N; ++k) v[u].v[k] = (T)((float)v[u].v[k] * coef);
                vq_stv<T, N>(dst + (i + u * 256) * N, v[u]);
            }
    }
    const int64_t i = whole * N + threadIdx.x;
    if (i < n) dst[i] = (T)((float)src[i] * coef);
}

__global__ void __launch_bounds__(256) vq_grad_scale_kernel(const GradArgs a, const float *coef_p)
{
    const GradTensor &t = grad_tensor(a, blockIdx.x);
    const float coef = *coef_p;
    if (coef == 1.f && t.src == t.dst) return;          // in place and nothing to clip: g * 1 is g
    const int64_t at = (int64_t)(blockIdx.x - t.first) * GRAD_CHUNK, n = t.n - at < GRAD_CHUNK ? t.n - at : GRAD_CHUNK;
    if (t.dtype == VQHIP_F32) grad_scale((const float *)t.src + at, (float *)t.dst + at, n, coef);
    else if (t.dtype == VQHIP_BF16) grad_scale((const __bf16 *)t.src + at, (__bf16 *)t.dst + at, n, coef);
    else grad_scale((const _Float16 *)t.src + at, (_Float16 *)t.dst + at, n, coef);
}

// every dst is its own src or shares no byte with a tensor of the call, and no src occurs twice: 1, or 0 with an overlap, -1 without memory
static int grad_apart(const vqhip_grad_t *g, int64_t count)
{
    struct Span { uintptr_t first, behind; bool written; };
    Span *s = (Span *)malloc(sizeof(Span) * 2 * (size_t)count);
    if (!s) return -1;
    size_t n = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (g[i].n <= 0) continue;
        const uintptr_t bytes = (uintptr_t)g[i].n * vq_elem_bytes(g[i].dtype), src = (uintptr_t)g[i].src, dst = (uintptr_t)g[i].dst;
        s[n++] = Span{src, src + bytes, src == dst};
        if (dst && dst != src) s[n++] = Span{dst, dst + bytes, true};
    }
    std::sort(s, s + n, [](const Span &a, const Span &b) { return a.first < b.first; });
    uintptr_t any = 0, written = 0, last = 0;                 // behind the last byte of any span, of a written one; the last first byte
    int ok = 1;
    for (size_t i = 0; i < n && ok; ++i) {
        if (s[i].first < (s[i].written ? any : written) || (i && s[i].first == last)) ok = 0;
        last = s[i].first;
        any = std::max(any, s[i].behind);
        if (s[i].written) written = std::max(written, s[i].behind);
    }
    free(s);
    return ok;
}

static int64_t grad_blocks(const vqhip_grad_t *g, int64_t count)
{
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) n += g[i].n > 0 ? (g[i].n + GRAD_CHUNK - 1) / GRAD_CHUNK : 0;
    return n;
}

extern "C" size_t vqhip_clip_grads_workspace_bytes(const vqhip_grad_t *grads, int64_t count)
{
    return grads && count > 0 ? (size_t)grad_blocks(grads, count) * 8 + 16 : 16;
}

extern "C" int vqhip_clip_grads(const vqhip_grad_t *grads, int64_t count, double max_norm, double eps, float *norm, void *workspace,
                                size_t workspace_bytes, void *stream)
{
    if (count < 0 || (count > 0 && !grads) || !norm || !workspace) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: %lld tensors, null pointer", (long long)count);
    if (!(max_norm >= 0.0) || !(eps >= 0.0)) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: max_norm %g, eps %g", max_norm, eps);
    bool write = false;
    for (int64_t i = 0; i < count; ++i) {
        if (!vq_elem_bytes(grads[i].dtype) || grads[i].n < 0 || grads[i].n > ((int64_t)1 << 44)) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: tensor %lld: dtype %lld, %lld elements", (long long)i, (long long)grads[i].dtype, (long long)grads[i].n);
        if (grads[i].n > 0 && !grads[i].src) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: tensor %lld: null pointer", (long long)i);
        write |= grads[i].n > 0 && grads[i].dst;
    }
    const int64_t blocks = grad_blocks(grads, count);
    if (blocks >= 1 << 24) VQ_FAIL(VQHIP_EDIM, "vqhip_clip_grads: too many elements");              // (2^32 threads)
    if (workspace_bytes < (size_t)blocks * 8 + 16) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: workspace of %zu bytes", workspace_bytes);
    if ((uintptr_t)workspace & 15) VQ_FAIL(VQHIP_EALIGN, "vqhip_clip_grads: workspace not 16-byte aligned");
    const int apart = count > 0 ? grad_apart(grads, count) : 1;
    if (apart < 0) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: no host memory");
    if (!apart) VQ_FAIL(VQHIP_EINVAL, "vqhip_clip_grads: a tensor occurs twice, or a result shares memory with another tensor");
    hipStream_t st = (hipStream_t)stream;
    float *coef = (float *)workspace;
    double *partial = (double *)((char *)workspace + 16);
    for (int pass = 0; pass < (write ? 2 : 1); ++pass) {
        int64_t done = 0;
        for (int64_t i = 0; i < count;) {
            GradArgs a;
            a.count = 0;
            unsigned nb = 0;
            for (; i < count && a.count < GRAD_TENSORS; ++i) {
                const vqhip_grad_t &g = grads[pass == 0 ? i : count - 1 - i];
                if (g.n <= 0 || (pass == 1 && !g.dst)) continue;
                a.t[a.count++] = GradTensor{g.src, g.dst, g.n, nb, (int)g.dtype};
                nb += (unsigned)((g.n + GRAD_CHUNK - 1) / GRAD_CHUNK);
            }
            if (!nb) continue;
            if (pass == 0) vq_grad_norm_kernel<<<dim3(nb), 256, 0, st>>>(a, partial + done);
            else vq_grad_scale_kernel<<<dim3(nb), 256, 0, st>>>(a, coef);
            done += nb;
        }
        if (pass == 0) vq_grad_coef_kernel<<<1, 1024, 0, st>>>(partial, done, max_norm, eps, norm, coef);
    }
    return vq_launch_status("vqhip_clip_grads");
}

// vq_group_norm.hip -- group norm with an activation on channels-last rows, forward and backward: the normalisation ahead of a quantizer
// that reads rows [b, n, c].
#include "vq_elem.h"

#include <math.h>

// y = act((x - mean) rstd w + bias), mean and variance over the live rows and the C / G channels of a group; rows that `lens` or `mask`
// leave out are neither read into the statistics nor normalised: their output is zero, whatever they hold.
struct GnArgs {
    const void *x; int64_t xb, xn;                      // element strides of batch and row
    const void *weight, *bias;
    const int64_t *lens; const uint8_t *mask;           // either or none
    void *y; float *mean, *rstd;
    const void *grad; void *dx; float *dws, *dbs;       // backward: grad and dx contiguous; [B, C] sums each
    int64_t N; int C, G, act, wdtype;
    double eps;
};

__device__ __forceinline__ float gn_param(const void *p, int dtype, int c, float none)
{
    if (!p) return none;
    return dtype == VQHIP_F32 ? ((const float *)p)[c] : dtype == VQHIP_BF16 ? (float)((const __bf16 *)p)[c] : (float)((const _Float16 *)p)[c];
}

__device__ __forceinline__ bool gn_live(const GnArgs &a, int64_t b, int64_t n)
{
    return a.lens ? n < a.lens[b] : a.mask ? a.mask[b * a.N + n] != 0 : true;
}

__device__ double gn_block_sum(double v, double *red)
{
    red[threadIdx.x] = v;
    __syncthreads();
    for (int o = 128; o; o >>= 1) {
        if ((int)threadIdx.x < o) red[threadIdx.x] += red[threadIdx.x + o];
        __syncthreads();
    }
    v = red[0];
    __syncthreads();
    return v;
}

template <typename T> __global__ void __launch_bounds__(256) vq_group_norm_kernel(const GnArgs a)
{
    __shared__ double red[256];
    const int64_t b = blockIdx.x / a.G;
    const int g = blockIdx.x % a.G, cg = a.C / a.G;
    const T *x = (const T *)a.x + b * a.xb + g * cg;
    const int64_t total = a.N * cg;
    double s = 0.0, n = 0.0;
    for (int64_t i = threadIdx.x; i < total; i += 256)
        if (gn_live(a, b, i / cg)) { s += (double)(float)x[(i / cg) * a.xn + i % cg]; n += 1.0; }
    n = gn_block_sum(n, red);
    const double mean = n > 0.0 ? gn_block_sum(s, red) / n : 0.0;
    s = 0.0;
    for (int64_t i = threadIdx.x; i < total; i += 256)
        if (gn_live(a, b, i / cg)) { const double d = (double)(float)x[(i / cg) * a.xn + i % cg] - mean; s += d * d; }
    const double rstd = n > 0.0 ? 1.0 / sqrt(gn_block_sum(s, red) / n + a.eps) : 0.0;
    if (threadIdx.x == 0) {
        a.mean[blockIdx.x] = (float)mean;
        a.rstd[blockIdx.x] = (float)rstd;
    }
    for (int64_t i = threadIdx.x; i < total; i += 256) {
        const int64_t r = i / cg;
        const int c = g * cg + (int)(i % cg);
        float y = 0.f;
        if (gn_live(a, b, r)) {
            const float xh = (float)(((double)(float)x[r * a.xn + i % cg] - mean) * rstd);
            y = fmaf(xh, gn_param(a.weight, a.wdtype, c, 1.f), gn_param(a.bias, a.wdtype, c, 0.f));
            if (a.act == VQHIP_ACT_SILU) y = y / (1.f + expf(-y));
        }
        ((T *)a.y)[(b * a.N + r) * a.C + c] = (T)y;
    }
}

// dz = grad act'(z); db = sum dz, dw = sum dz xh over the live rows; dx = rstd (dz w - mean(dz w) - xh mean(dz w xh)), 0 in padding rows
template <typename T> __global__ void __launch_bounds__(256) vq_group_norm_bwd_kernel(const GnArgs a)
{
    __shared__ double red[256];
    const int64_t b = blockIdx.x / a.G;
    const int g = blockIdx.x % a.G, cg = a.C / a.G;
    const T *x = (const T *)a.x + b * a.xb;
    const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
    double s1 = 0.0, s2 = 0.0, n = 0.0;
    for (int c = g * cg; c < (g + 1) * cg; ++c) {
        const float w = gn_param(a.weight, a.wdtype, c, 1.f), bias = gn_param(a.bias, a.wdtype, c, 0.f);
        double db = 0.0, dw = 0.0;
        n = 0.0;
        for (int64_t r = threadIdx.x; r < a.N; r += 256)
            if (gn_live(a, b, r)) {
                const float xh = ((float)x[r * a.xn + c] - mean) * rstd, z = fmaf(xh, w, bias);
                float dz = (float)((const T *)a.grad)[(b * a.N + r) * a.C + c];
                if (a.act == VQHIP_ACT_SILU) { const float q = 1.f / (1.f + expf(-z)); dz *= q * (1.f + z * (1.f - q)); }
                db += dz; dw += (double)dz * xh; n += 1.0;
            }
        db = gn_block_sum(db, red);
        dw = gn_block_sum(dw, red);
        n = gn_block_sum(n, red);
        s1 += db * w; s2 += dw * w;
        if (threadIdx.x == 0) { a.dbs[b * a.C + c] = (float)db; a.dws[b * a.C + c] = (float)dw; }
    }
    if (!a.dx) return;
    n *= cg;
    const float m1 = n > 0.0 ? (float)(s1 / n) : 0.f, m2 = n > 0.0 ? (float)(s2 / n) : 0.f;
    for (int64_t i = threadIdx.x; i < a.N * cg; i += 256) {
        const int64_t r = i / cg;
        const int c = g * cg + (int)(i % cg);
        float d = 0.f;
        if (gn_live(a, b, r)) {
            const float w = gn_param(a.weight, a.wdtype, c, 1.f);
            const float xh = ((float)x[r * a.xn + c] - mean) * rstd, z = fmaf(xh, w, gn_param(a.bias, a.wdtype, c, 0.f));
            float dz = (float)((const T *)a.grad)[(b * a.N + r) * a.C + c];
            if (a.act == VQHIP_ACT_SILU) { const float q = 1.f / (1.f + expf(-z)); dz *= q * (1.f + z * (1.f - q)); }
            d = rstd * (dz * w - m1 - xh * m2);
        }
        ((T *)a.dx)[(b * a.N + r) * a.C + c] = (T)d;
    }
}

// dweight[c] = sum_b dws[b, c], dbias likewise, in 64 bits and in the order of b
__global__ void __launch_bounds__(256) vq_group_norm_params_kernel(const float *dws, const float *dbs, int64_t B, int C, void *dweight, void *dbias, int dtype)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    double w = 0.0, q = 0.0;
    for (int64_t b = 0; b < B; ++b) { w += dws[b * C + c]; q += dbs[b * C + c]; }
    for (int k = 0; k < 2; ++k) {
        void *out = k ? dbias : dweight;
        const float v = (float)(k ? q : w);
        if (!out) continue;
        if (dtype == VQHIP_F32) ((float *)out)[c] = v;
        else if (dtype == VQHIP_BF16) ((__bf16 *)out)[c] = (__bf16)v;
        else ((_Float16 *)out)[c] = (_Float16)v;
    }
}

static int gn_check(const vqhip_group_norm_t *p, const char *what)
{
    if (!p) VQ_FAIL(VQHIP_EINVAL, "%s: null argument", what);
    if (!vq_elem_bytes(p->dtype) || !vq_elem_bytes(p->param_dtype)) VQ_FAIL(VQHIP_EINVAL, "%s: dtype %lld, parameters of %lld", what, (long long)p->dtype, (long long)p->param_dtype);
    if (p->B < 0 || p->N < 0 || p->C < 1 || p->groups < 1 || p->C % p->groups || !(p->eps >= 0.0)) VQ_FAIL(VQHIP_EINVAL, "%s: B %lld, N %lld, C %lld in %lld groups, eps %g", what, (long long)p->B, (long long)p->N, (long long)p->C, (long long)p->groups, p->eps);
    if (p->activation != VQHIP_ACT_NONE && p->activation != VQHIP_ACT_SILU) VQ_FAIL(VQHIP_EINVAL, "%s: activation %lld", what, (long long)p->activation);
    if (p->C > VQHIP_NORM_MAX_C || p->B > 0x7fffffff / p->C || p->N > ((int64_t)1 << 40) / p->C) VQ_FAIL(VQHIP_EDIM, "%s: %lld x %lld rows of %lld channels (at most %d)", what, (long long)p->B, (long long)p->N, (long long)p->C, VQHIP_NORM_MAX_C);
    if (p->lens && p->mask) VQ_FAIL(VQHIP_EINVAL, "%s: lens and mask", what);
    if (p->B > 0 && p->N > 0 && (!p->x || !p->mean || !p->rstd)) VQ_FAIL(VQHIP_EINVAL, "%s: null pointer", what);
    if (p->workspace_bytes < vqhip_group_norm_workspace_bytes(p->B, p->N, p->C, p->groups) || (!p->workspace && p->workspace_bytes)) VQ_FAIL(VQHIP_EINVAL, "%s: workspace of %zu bytes", what, p->workspace_bytes);
    return 0;
}

static GnArgs gn_args(const vqhip_group_norm_t *p)
{
    GnArgs a;
    a.x = p->x; a.xb = p->stride_b; a.xn = p->stride_n; a.weight = p->weight; a.bias = p->bias; a.lens = p->lens; a.mask = p->mask;
    a.y = nullptr; a.mean = p->mean; a.rstd = p->rstd; a.grad = nullptr; a.dx = nullptr; a.dws = a.dbs = nullptr;
    a.N = p->N; a.C = (int)p->C; a.G = (int)p->groups; a.act = (int)p->activation; a.wdtype = (int)p->param_dtype; a.eps = p->eps;
    return a;
}

extern "C" size_t vqhip_group_norm_workspace_bytes(int64_t B, int64_t N, int64_t C, int64_t groups)
{
    (void)N; (void)groups;
    return B > 0 && C > 0 ? (size_t)B * C * 8 : 0;
}

#define GN_BY_TYPE(dtype, kernel, ...)                                        \
    do {                                                                      \
        if ((dtype) == VQHIP_F32) kernel<float> __VA_ARGS__;                  \
        else if ((dtype) == VQHIP_BF16) kernel<__bf16> __VA_ARGS__;           \
        else kernel<_Float16> __VA_ARGS__;                                    \
    } while (0)

extern "C" int vqhip_group_norm(const vqhip_group_norm_t *p, void *y, void *stream)
{
    int rc = gn_check(p, "vqhip_group_norm");
    if (rc) return rc;
    if (p->B == 0 || p->N == 0) return 0;
    if (!y) VQ_FAIL(VQHIP_EINVAL, "vqhip_group_norm: null pointer");
    GnArgs a = gn_args(p);
    a.y = y;
    GN_BY_TYPE(p->dtype, vq_group_norm_kernel, <<<dim3((unsigned)(p->B * p->groups)), 256, 0, (hipStream_t)stream>>>(a));
    return vq_launch_status("vqhip_group_norm");
}

extern "C" int vqhip_group_norm_bwd(const vqhip_group_norm_t *p, const void *grad, void *dx, void *dweight, void *dbias, void *stream)
{
    int rc = gn_check(p, "vqhip_group_norm_bwd");
    if (rc) return rc;
    if (!dx && !dweight && !dbias) return 0;
    const bool some = p->B > 0 && p->N > 0;
    if (some && !grad) VQ_FAIL(VQHIP_EINVAL, "vqhip_group_norm_bwd: null pointer");
    GnArgs a = gn_args(p);
    a.grad = grad; a.dx = dx; a.dws = (float *)p->workspace; a.dbs = a.dws + p->B * p->C;
    if (some) GN_BY_TYPE(p->dtype, vq_group_norm_bwd_kernel, <<<dim3((unsigned)(p->B * p->groups)), 256, 0, (hipStream_t)stream>>>(a));
    if (dweight || dbias)
        vq_group_norm_params_kernel<<<dim3((unsigned)((p->C + 255) / 256)), 256, 0, (hipStream_t)stream>>>(a.dws, a.dbs, some ? p->B : 0, a.C, dweight, dbias, a.wdtype);
    return vq_launch_status("vqhip_group_norm_bwd");
}

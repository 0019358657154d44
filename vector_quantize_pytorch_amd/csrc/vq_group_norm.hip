// vq_group_norm.hip -- group norm with an activation on channels-last rows, forward and backward: the normalisation ahead of a quantizer
// that reads rows [b, n, c].
//
// y = act((x - mean) rstd w + bias), mean and variance over the live rows and the C / G channels of a group; rows that `lens` or `mask`
// leave out are neither read into the statistics nor normalised: their output is zero, whatever they hold.
//
// Two launches each way, both over (batch entry, chunk of rows): the first leaves each chunk's statistics (backward: its sums), the
// second joins them -- in every workgroup, S * G pairs from cache; beyond GN_JOIN in a small launch between -- and writes the rows.  Bound by HBM, with the second read of x from
// the memory-side cache where it fits.  A thread keeps VEC channels of every row it visits (16 bytes where C divides so), so parameters and
// statistics stay in registers and rows of any stride are read in whole lines.  All sums have one order: no atomics.
#include "vq_elem.h"

#include <math.h>

#define GN_T 512                   // threads of a workgroup
#define GN_FLUSH 32                // rows that a thread sums about one pivot
// pairs (chunks x groups) of a batch row that every workgroup of the second launch joins for itself; more are joined in a launch between.
// Apply kernel against join and apply: 64 x 8 9.5 and 3.9 + 8.2 us, 128 x 32 26.9 and 4.0 + 22.5, 170 x 32 36.2 and 4.6 + 32.4, 256 x 32 19.7 and
// 3.8 + 11.4; a launch more costs its 3 us of host besides.
#define GN_JOIN 6144

struct GnArgs {
    const void *x; int64_t xb, xn;                      // element strides of batch and row
    const void *weight, *bias;
    const int64_t *lens; const uint8_t *mask;           // either or none
    void *y; float *mean, *rstd;
    const void *grad; void *dx, *dweight, *dbias;       // backward: grad and dx contiguous
    float2 *pair, *joined; float *chan, *live;          // per chunk: [B * S, G] pairs, (backward) [B * S, 2, C] sums, [B * S] live rows; joined [B, G] or null
    int64_t N, B, rows; int C, G, act, wdtype, S;       // S chunks of `rows` rows
    double eps;
};

__device__ __forceinline__ float gn_param(const void *p, int dtype, int c, float none)
{
    if (!p) return none;
    return dtype == VQHIP_F32 ? ((const float *)p)[c] : dtype == VQHIP_BF16 ? (float)((const __bf16 *)p)[c] : (float)((const _Float16 *)p)[c];
}

// VEC parameters from channel c on, in one load (one by one, each waits for the one before it)
template <int VEC> __device__ __forceinline__ void gn_params(const void *p, int dtype, int c, float none, float *out)
{
    if (!p) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = none;
    } else if (dtype == VQHIP_F32) {
        const VqVec<float, VEC> v = vq_ldv<float, VEC>((const float *)p + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = v.v[i];
    } else {
        const VqVec<uint16_t, VEC> v = vq_ldv<uint16_t, VEC>((const uint16_t *)p + c);
#pragma unroll
        for (int i = 0; i < VEC; ++i) out[i] = dtype == VQHIP_BF16 ? (float)__builtin_bit_cast(__bf16, v.v[i]) : (float)__builtin_bit_cast(_Float16, v.v[i]);
    }
}

__device__ __forceinline__ void gn_store_param(void *p, int dtype, int c, float v)
{
    if (dtype == VQHIP_F32) ((float *)p)[c] = v;
    else if (dtype == VQHIP_BF16) ((__bf16 *)p)[c] = (__bf16)v;
    else ((_Float16 *)p)[c] = (_Float16)v;
}

// rows [0, gn_len) of an entry may be live, with a mask (template parameter MASKED) those that it names
__device__ __forceinline__ int64_t gn_len(const GnArgs &a, int64_t b)
{
    const int64_t len = a.lens ? a.lens[b] : a.N;
    return len < 0 ? 0 : len < a.N ? len : a.N;
}

__device__ __forceinline__ float gn_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504f)); }

// what a thread visits: rows first + lane, + step, ...; VEC channels from vector column col0 + (t % width), pass after pass of `width` columns
struct GnShape { int cols, width, lanes; };
template <int VEC> __device__ __forceinline__ GnShape gn_shape(int C)
{
    const int cols = C / VEC, width = cols < GN_T ? cols : GN_T;
    return GnShape{cols, width, GN_T / width};
}

// the groups of channels that follow each other: one division, then steps
struct GnGroup {
    int g, r, cg;
    __device__ GnGroup(int c, int cg_) : g(c / cg_), r(c - c / cg_ * cg_), cg(cg_) {}
    __device__ __forceinline__ void next() { if (++r == cg) { r = 0; ++g; } }
};

// sums over the channels of each group that lies in [c0, c1): f(lane entry) -> v[NV] doubles, entries = lanes x channels.  A group that
// goes on in the next pass is carried there (two places, since one pass may read and write it).  done(g, v) by one thread a group.
template <int NV, typename F, typename D> __device__ __forceinline__ void gn_groups(int c0, int c1, int cg, int lanes, const double *carry_in, double *carry_out, F &&entry, D &&done)
{
    const int g0 = c0 / cg, g1 = (c1 - 1) / cg, ng = g1 - g0 + 1;
    int tg = 64;                                        // threads a group: a power of two within a wave
    while (tg > 1 && tg * ng > GN_T) tg >>= 1;
    const int per = GN_T / tg;
    const bool from_before = c0 % cg != 0, goes_on = c1 % cg != 0;
    for (int base = 0; base < ng; base += per) {
        const int g = g0 + base + (int)threadIdx.x / tg, q = threadIdx.x % tg;
        double v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = 0.0;
        if (g <= g1) {
            const int lo = g * cg < c0 ? c0 : g * cg, hi = (g + 1) * cg > c1 ? c1 : (g + 1) * cg, wide = hi - lo;
            for (int l = q / wide, c = q - l * wide; l < lanes;) {             // entry l * wide + c, then tg further
                entry(l, lo + c, v);
                for (c += tg; c >= wide; c -= wide) ++l;
            }
        }
        for (int o = tg >> 1; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += __shfl_xor(v[i], o, 64);
        if (g <= g1 && q == 0) {
            if (g == g0 && from_before)
#pragma unroll
                for (int i = 0; i < NV; ++i) v[i] += carry_in[i];
            if (g == g1 && goes_on) {
#pragma unroll
                for (int i = 0; i < NV; ++i) carry_out[i] = v[i];
            } else
                done(g, v);
        }
    }
}

// ---- forward, first launch: each chunk's (mean, variance) of every group ------------------------------------------
// A thread sums x - p and (x - p)^2 of a channel over up to GN_FLUSH rows, p the first of them: p is one of the values, so what cancels is
// at most the number of rows -- an outlier or a far mean costs nothing.  Blocks, threads and channels join by counts, means and squared
// deviations, the last in 64 bits.
template <typename T, int VEC, bool MASKED> __global__ void __launch_bounds__(GN_T) vq_gn_stats_kernel(const GnArgs a)
{
    __shared__ float em[GN_T * VEC], ed[GN_T * VEC], en[GN_T];
    __shared__ double carry[2][3];
    const int chunk = blockIdx.x % (unsigned)a.S, t = threadIdx.x;
    const int64_t b = blockIdx.x / (unsigned)a.S, len = gn_len(a, b), r0 = (int64_t)chunk * a.rows, r1 = r0 + a.rows < len ? r0 + a.rows : len;
    const GnShape sh = gn_shape<VEC>(a.C);
    const int lane = t / sh.width, cg = a.C / a.G;
    const bool whole = cg % VEC == 0;
    const T *x = (const T *)a.x + b * a.xb;
    const uint8_t *mask = MASKED ? a.mask + b * a.N : nullptr;
    float2 *out = a.pair + (int64_t)blockIdx.x * a.G;
    for (int col0 = 0, pass = 0; col0 < sh.cols; col0 += sh.width, ++pass) {
        const int col = col0 + t % sh.width;
        float n = 0.f, mean[VEC], dev[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) mean[i] = dev[i] = 0.f;
        if (lane < sh.lanes && col < sh.cols) {
            const T *xc = x + (int64_t)col * VEC;
            for (int64_t r = r0 + lane; r < r1; r += (int64_t)GN_FLUSH * sh.lanes) {
                float p[VEC], s[VEC], q[VEC], m = 0.f;
#pragma unroll
                for (int i = 0; i < VEC; ++i) p[i] = s[i] = q[i] = 0.f;
                for (int k = 0; k < GN_FLUSH; k += 4) {
                    VqVec<T, VEC> v[4];
                    bool live[4];
                    const int64_t at = r + (int64_t)k * sh.lanes;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int64_t row = at + u * sh.lanes, in = row < r1 ? row : r1 - 1;
                        live[u] = row < r1 && (!MASKED || mask[in]);
                        v[u] = vq_ldv<T, VEC>(xc + in * a.xn);                     // (loads without conditions: four in flight)
                    }
                    if (m == 0.f) {                           // the first live one of these is the pivot
#pragma unroll
                        for (int u = MASKED ? 3 : 0; u >= 0; --u)
                            if (live[u])
#pragma unroll
                                for (int i = 0; i < VEC; ++i) p[i] = (float)v[u].v[i];
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
                        if (live[u]) {
                            m += 1.f;
#pragma unroll
                            for (int i = 0; i < VEC; ++i) {
                                const float d = (float)v[u].v[i] - p[i];
                                s[i] += d;
                                q[i] = fmaf(d, d, q[i]);
                            }
                        }
                    if (at + 4 * sh.lanes >= r1) break;
                }
                if (m > 0.f) {
                    const float all = n + m, inv = 1.f / m, part = m / all, cross = n * part;
#pragma unroll
                    for (int i = 0; i < VEC; ++i) {
                        const float mb = s[i] * inv, db = fmaxf(fmaf(-s[i], mb, q[i]), 0.f), d = p[i] + mb - mean[i];
                        dev[i] += fmaf(d * d, cross, db);
                        mean[i] = n > 0.f ? fmaf(d, part, mean[i]) : p[i] + mb;
                    }
                    n = all;
                }
            }
        }
        // a thread's channels in one group are joined here: an entry a thread instead of VEC
        if (whole) {
            float m = 0.f, d = 0.f;
#pragma unroll
            for (int i = 0; i < VEC; ++i) m += mean[i] * (1.f / VEC);
#pragma unroll
            for (int i = 0; i < VEC; ++i) d += fmaf((mean[i] - m) * (mean[i] - m), n, dev[i]);
            em[t] = m;
            ed[t] = d;
        } else
#pragma unroll
            for (int i = 0; i < VEC; ++i) { em[t * VEC + i] = mean[i]; ed[t * VEC + i] = dev[i]; }
        en[t] = n;
        __syncthreads();
        if (t == 0 && col0 == 0) {
            float rows = 0.f;
            for (int l = 0; l < sh.lanes; ++l) rows += en[l * sh.width];
            a.live[blockIdx.x] = rows;
        }
        // 64-bit sums about zero: count, count * mean, squared deviations + count * mean^2
        const int per = whole ? 1 : VEC, last = col0 + sh.width < sh.cols ? col0 + sh.width : sh.cols;
        gn_groups<3>(col0 * per, last * per, whole ? cg / VEC : cg, sh.lanes, carry[pass & 1], carry[~pass & 1],
            [&](int l, int c, double *v) {
                const int k = c - col0 * per, e = l * sh.width * per + k;
                const double w = whole ? en[e] * VEC : en[l * sh.width + k / VEC], m = em[e];
                v[0] += w;
                v[1] = fma(w, m, v[1]);
                v[2] += fma(w * m, m, (double)ed[e]);
            },
            [&](int g, const double *v) {
                const double m = v[0] > 0.0 ? v[1] / v[0] : 0.0, d = v[0] > 0.0 ? (v[2] - v[1] * m) / v[0] : 0.0;
                out[g] = make_float2((float)m, (float)(d > 0.0 ? d : 0.0));
            });
        __syncthreads();
    }
}

// ---- the chunks of a batch entry joined, 64-bit sums: forward to (mean, rstd), backward to (mean(dz w), mean(dz w xh)) of a group --------
template <bool BWD> __device__ __forceinline__ void gn_add(const GnArgs &a, int64_t chunk, int g, double *v)
{
    const float2 p = a.pair[chunk * a.G + g];
    const double k = a.live[chunk];
    v[0] += k;
    if (BWD) {
        v[1] += p.x;
        v[2] += p.y;
    } else {
        v[1] = fma(k, (double)p.x, v[1]);
        v[2] += k * fma((double)p.x, (double)p.x, (double)p.y);
    }
}
template <bool BWD> __device__ __forceinline__ float2 gn_joined(const GnArgs &a, const double *v)
{
    if (BWD) {
        const double inv = v[0] > 0.0 ? 1.0 / (v[0] * (a.C / a.G)) : 0.0;
        return make_float2((float)(v[1] * inv), (float)(v[2] * inv));
    }
    const double m = v[0] > 0.0 ? v[1] / v[0] : 0.0, d = v[0] > 0.0 ? (v[2] - v[1] * m) / v[0] : 0.0;
    return make_float2((float)m, (float)(1.0 / sqrt((d > 0.0 ? d : d == d ? 0.0 : d) + a.eps)));
}

// many chunks: a launch of its own, a wave each (batch entry, group)
template <bool BWD> __global__ void __launch_bounds__(256) vq_gn_join_kernel(const GnArgs a)
{
    const int64_t bg = (int64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (bg >= a.B * a.G) return;
    const int64_t b = bg / a.G;
    const int g = (int)(bg - b * a.G);
    double v[3] = {0.0, 0.0, 0.0};
#pragma unroll 4
    for (int s = threadIdx.x & 63; s < a.S; s += 64) gn_add<BWD>(a, b * a.S + s, g, v);
#pragma unroll
    for (int i = 0; i < 3; ++i) v[i] = vq_wave_sum(v[i]);
    if ((threadIdx.x & 63) == 0) a.joined[bg] = gn_joined<BWD>(a, v);
}

// few: every workgroup for itself, into LDS
template <bool BWD> __device__ __forceinline__ void gn_join(const GnArgs &a, int64_t b, float2 *stat)
{
    const int S = a.S, G = a.G;
    if (a.joined) {
        for (int g = threadIdx.x; g < G; g += GN_T) stat[g] = a.joined[b * G + g];
        return;
    }
    int tg = 64;
    while (tg > 1 && (tg * G > GN_T || tg / 2 >= S)) tg >>= 1;
    for (int g = (int)threadIdx.x / tg; g < (G + GN_T / tg - 1) / (GN_T / tg) * (GN_T / tg); g += GN_T / tg) {
        double v[3] = {0.0, 0.0, 0.0};
        if (g < G)
#pragma unroll 8
            for (int s = threadIdx.x % tg; s < S; s += tg) gn_add<BWD>(a, b * S + s, g, v);
        for (int o = tg >> 1; o; o >>= 1)
#pragma unroll
            for (int i = 0; i < 3; ++i) v[i] += __shfl_xor(v[i], o, 64);
        if (g < G && threadIdx.x % tg == 0) stat[g] = gn_joined<BWD>(a, v);
    }
}

// ---- forward, second launch --------------------------------------------------------------------------------------------------------
// rows [from, to) x VEC channels of zeros, what padding gives
template <typename T, int VEC> __device__ __forceinline__ void gn_zero_rows(T *p, int64_t from, int64_t to, int step, int64_t stride)
{
    VqVec<T, VEC> o;
#pragma unroll
    for (int i = 0; i < VEC; ++i) o.v[i] = (T)0.f;
    for (int64_t r = from; r < to; r += step) vq_stv<T, VEC>(p + r * stride, o);
}

template <typename T, int VEC, bool SILU, bool MASKED> __global__ void __launch_bounds__(GN_T) vq_gn_apply_kernel(const GnArgs a)
{
    extern __shared__ __align__(16) float2 stat[];      // (mean, rstd) [G]
    const int chunk = blockIdx.x % (unsigned)a.S, t = threadIdx.x;
    const int64_t b = blockIdx.x / (unsigned)a.S, len = gn_len(a, b), r0 = (int64_t)chunk * a.rows, end = r0 + a.rows < a.N ? r0 + a.rows : a.N, r1 = end < len ? end : len;
    const int G = a.G, cg = a.C / G;
    gn_join<false>(a, b, stat);
    __syncthreads();
    if (chunk == 0)
        for (int g = t; g < G; g += GN_T) { a.mean[b * G + g] = stat[g].x; a.rstd[b * G + g] = stat[g].y; }
    const GnShape sh = gn_shape<VEC>(a.C);
    const int lane = t / sh.width;
    if (lane >= sh.lanes) return;
    const T *x = (const T *)a.x + b * a.xb;
    const uint8_t *mask = MASKED ? a.mask + b * a.N : nullptr;
    T *y = (T *)a.y + b * a.N * a.C;
    // (x - mean) scale + bias, the mean first: bias - mean scale would round a number |mean| rstd times the result's size, and flat rows far from
    // zero would lose their bias to it (values of 1000 and a bias of 0.2: 0.212).  6 x 65536 x 128 bf16 57 us a call either way
    for (int col = t % sh.width; col < sh.cols; col += sh.width) {
        float mean[VEC], scale[VEC], shift[VEC];
        gn_params<VEC>(a.weight, a.wdtype, col * VEC, 1.f, scale);
        gn_params<VEC>(a.bias, a.wdtype, col * VEC, 0.f, shift);
        GnGroup of(col * VEC, cg);
#pragma unroll
        for (int i = 0; i < VEC; ++i, of.next()) {
            const float2 st = stat[of.g];
            mean[i] = st.x;
            scale[i] *= st.y;
        }
        const T *xc = x + (int64_t)col * VEC;
        T *yc = y + (int64_t)col * VEC;
        for (int64_t r = r0 + lane; r < r1; r += 4 * sh.lanes) {
            VqVec<T, VEC> v[4];
            bool live[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = r + (int64_t)u * sh.lanes, in = at < r1 ? at : r1 - 1;
                live[u] = at < r1 && (!MASKED || mask[in]);
                v[u] = vq_ldv<T, VEC>(xc + in * a.xn);
            }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int64_t at = r + (int64_t)u * sh.lanes;
                if (at >= r1) break;
                VqVec<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    float z = fmaf((float)v[u].v[i] - mean[i], scale[i], shift[i]);
                    if (SILU) z *= gn_sigmoid(z);
                    o.v[i] = !MASKED || live[u] ? (T)z : (T)0.f;
                }
                vq_stv<T, VEC>(yc + at * a.C, o);
            }
        }
        gn_zero_rows<T, VEC>(yc, (r0 > len ? r0 : len) + lane, end, sh.lanes, a.C);
    }
}

// ---- forward, small slabs in one launch -----------------------------------------------------------------------------------------------
// A workgroup keeps all rows of a span of whole groups (128 bytes of a row or more, a power of two of columns) in registers, U rows a
// thread: x is read once.  The mean first, then the deviations from it, whose own mean corrects it; 32 bits hold both.  A wave's rows
// join by shuffles, the waves in LDS, and every thread sums its groups' channels for itself.  Bound by latency and by the instructions of a
// wave: 1 x 256 x 512 bf16 12 us of kernels in two launches, 10 in one with 8 workgroups of 64 KB, 5.7 with 32 of 8 KB.
template <typename T, int VEC, int U, bool SILU, bool MASKED> __global__ void __launch_bounds__(GN_T) vq_gn_one_kernel(const GnArgs a, int span)
{
    constexpr int WAVES = GN_T / 64;
    __shared__ float part[2][WAVES][64 * VEC], chan[2][64 * VEC], count[WAVES];
    const int t = threadIdx.x, cols = span / VEC, lanes = GN_T / cols, lane = t / cols, cg = a.C / a.G, spans = a.C / span, wave = t >> 6;
    const int64_t b = blockIdx.x / (unsigned)spans;
    const int c0 = (int)(blockIdx.x % (unsigned)spans) * span, own = t % cols * VEC, c = c0 + own;
    const int N = (int)a.N, len = (int)gn_len(a, b);
    const T *x = (const T *)a.x + b * a.xb + c;
    const uint8_t *mask = MASKED ? a.mask + b * a.N : nullptr;
    VqVec<T, VEC> v[U];
    bool live[U];
    float n = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = lane + u * lanes, at = r < N ? r : N - 1;
        v[u] = vq_ldv<T, VEC>(x + (int64_t)at * a.xn);
        live[u] = r < len && (!MASKED || mask[at]);
        n += live[u] ? 1.f : 0.f;
    }
    float scale[VEC], shift[VEC], mean[VEC];
    gn_params<VEC>(a.weight, a.wdtype, c, 1.f, scale);
    gn_params<VEC>(a.bias, a.wdtype, c, 0.f, shift);
    if (MASKED) {
        for (int o = cols; o < 64; o <<= 1) n += __shfl_xor(n, o, 64);
        if ((t & 63) == 0) count[wave] = n;
    } else
        n = (float)len;
#pragma unroll
    for (int i = 0; i < VEC; ++i) mean[i] = 0.f;
    float inv = 0.f, unit = 1.f, rstd[VEC];             // unit: 1 / sqrt(count), so that squares sum to the variance, in its range
    const int parts = cg % VEC == 0 ? 1 : VEC;          // a thread's channels in one group: summed here, in the place of its first
    if (parts == 1)
        for (int k = t; k < 2 * span; k += GN_T) (&chan[0][0])[(k >= span) * 64 * VEC + (k >= span ? k - span : k)] = 0.f;
    for (int pass = 0; pass < 2; ++pass) {              // 0: sums; 1: sums of deviations and of their squares
        float s[VEC], q[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            s[i] = q[i] = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (live[u]) {
                    const float d = ((float)v[u].v[i] - mean[i]) * unit;
                    s[i] += d;
                    if (pass) q[i] = fmaf(d, d, q[i]);
                }
        }
        if (parts == 1)
#pragma unroll
            for (int i = 1; i < VEC; ++i) { s[0] += s[i]; q[0] += q[i]; }
#pragma unroll
        for (int i = 0; i < VEC; ++i)
            if (i < parts) {
                for (int o = cols; o < 64; o <<= 1) {
                    s[i] += __shfl_xor(s[i], o, 64);
                    q[i] += __shfl_xor(q[i], o, 64);
                }
                if ((t & 63) < cols) { part[0][wave][own + i] = s[i]; part[1][wave][own + i] = q[i]; }
            }
        __syncthreads();
        const int step = parts == 1 ? VEC : 1;
        for (int k = t * step; k < 2 * span; k += GN_T * step) {
            const int w = k >= span, e = k - w * span;
            float r = 0.f;
#pragma unroll
            for (int l = 0; l < WAVES; ++l) r += part[w][l][e];
            chan[w][e] = r;
        }
        if (!pass) {
            if (MASKED) {
                n = 0.f;
#pragma unroll
                for (int l = 0; l < WAVES; ++l) n += count[l];
            }
            inv = n > 0.f ? 1.f / (n * (float)cg) : 0.f;
        }
        __syncthreads();
        const float back = pass ? unit : inv;
        unit = sqrtf(inv);
        GnGroup of(own, cg);
        float m = 0.f, d = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i, of.next()) {
            if (i == 0 || of.r == 0) {
                float r = 0.f;
                m = 0.f;
                for (int k = 0; k < cg; k += step) { m += chan[0][of.g * cg + k]; r += chan[1][of.g * cg + k]; }
                m *= back;
                d = fmaf(-m, m, r);
                if (pass) d = 1.f / sqrtf((d > 0.f ? d : d == d ? 0.f : d) + (float)a.eps);
            }
            mean[i] += m;
            rstd[i] = d;
        }
    }
    if (lane == 0) {                                    // the groups that begin among this thread's channels
        GnGroup of(own, cg);
#pragma unroll
        for (int i = 0; i < VEC; ++i, of.next())
            if (of.r == 0) {
                a.mean[b * a.G + c0 / cg + of.g] = mean[i];
                a.rstd[b * a.G + c0 / cg + of.g] = rstd[i];
            }
    }
#pragma unroll
    for (int i = 0; i < VEC; ++i) scale[i] *= rstd[i];
    T *y = (T *)a.y + b * a.N * a.C + c;
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int r = lane + u * lanes;
        if (r >= N) break;
        VqVec<T, VEC> o;
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            float z = fmaf((float)v[u].v[i] - mean[i], scale[i], shift[i]);
            if (SILU) z *= gn_sigmoid(z);
            o.v[i] = live[u] ? (T)z : (T)0.f;
        }
        vq_stv<T, VEC>(y + (int64_t)r * a.C, o);
    }
}

// ---- backward --------------------------------------------------------------------------------------------------------------------------
// dz = grad act'(z); db = sum dz, dw = sum dz xh over the live rows; dx = rstd (dz w - mean(dz w) - xh mean(dz w xh)), 0 in padding rows
template <bool SILU> __device__ __forceinline__ float gn_dz(float g, float xh, float w, float bias)
{
    if (!SILU) return g;
    const float z = fmaf(xh, w, bias), q = gn_sigmoid(z);
    return g * q * fmaf(z, 1.f - q, 1.f);
}

// first launch: each chunk's sums of dz and dz xh of every channel, and of w times them of every group
template <typename T, int VEC, bool SILU, bool MASKED> __global__ void __launch_bounds__(GN_T) vq_gn_bwd_sums_kernel(const GnArgs a)
{
    __shared__ float e0[GN_T * VEC], e1[GN_T * VEC], en[GN_T];
    __shared__ double carry[2][2];
    const int chunk = blockIdx.x % (unsigned)a.S, t = threadIdx.x, G = a.G, cg = a.C / G;
    const int64_t b = blockIdx.x / (unsigned)a.S, len = gn_len(a, b), r0 = (int64_t)chunk * a.rows, r1 = r0 + a.rows < len ? r0 + a.rows : len;
    const GnShape sh = gn_shape<VEC>(a.C);
    const int lane = t / sh.width;
    const T *x = (const T *)a.x + b * a.xb, *gr = (const T *)a.grad + b * a.N * a.C;
    const uint8_t *mask = MASKED ? a.mask + b * a.N : nullptr;
    float2 *pair = a.pair + (int64_t)blockIdx.x * G;
    float *chan = a.chan + (int64_t)blockIdx.x * a.C * 2;
    for (int col0 = 0, pass = 0; col0 < sh.cols; col0 += sh.width, ++pass) {
        const int col = col0 + t % sh.width;
        float s0[VEC], s1[VEC], n = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) s0[i] = s1[i] = 0.f;
        if (lane < sh.lanes && col < sh.cols) {
            float mean[VEC], rstd[VEC], w[VEC], bias[VEC];
            gn_params<VEC>(a.weight, a.wdtype, col * VEC, 1.f, w);
            gn_params<VEC>(a.bias, a.wdtype, col * VEC, 0.f, bias);
            GnGroup of(col * VEC, cg);
#pragma unroll
            for (int i = 0; i < VEC; ++i, of.next()) {
                mean[i] = a.mean[b * G + of.g];
                rstd[i] = a.rstd[b * G + of.g];
            }
            for (int64_t r = r0 + lane; r < r1; r += 4 * sh.lanes) {
                VqVec<T, VEC> v[4], d[4];
                bool live[4];
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int64_t at = r + (int64_t)u * sh.lanes, in = at < r1 ? at : r1 - 1;
                    live[u] = at < r1 && (!MASKED || mask[in]);
                    v[u] = vq_ldv<T, VEC>(x + in * a.xn + (int64_t)col * VEC);
                    d[u] = vq_ldv<T, VEC>(gr + in * a.C + (int64_t)col * VEC);
                }
#pragma unroll
                for (int u = 0; u < 4; ++u)
                    if (live[u]) {
                        n += 1.f;
#pragma unroll
                        for (int i = 0; i < VEC; ++i) {
                            const float xh = ((float)v[u].v[i] - mean[i]) * rstd[i], dz = gn_dz<SILU>((float)d[u].v[i], xh, w[i], bias[i]);
                            s0[i] += dz;
                            s1[i] = fmaf(dz, xh, s1[i]);
                        }
                    }
            }
        }
#pragma unroll
        for (int i = 0; i < VEC; ++i) { e0[t * VEC + i] = s0[i]; e1[t * VEC + i] = s1[i]; }
        en[t] = n;
        __syncthreads();
        const int c0 = col0 * VEC, c1 = (col0 + sh.width < sh.cols ? col0 + sh.width : sh.cols) * VEC, wide = sh.width * VEC;
        if (t == 0 && col0 == 0) {
            float rows = 0.f;
            for (int l = 0; l < sh.lanes; ++l) rows += en[l * sh.width];
            a.live[blockIdx.x] = rows;
        }
        for (int c = c0 + t; c < c1; c += GN_T) {
            float q0 = 0.f, q1 = 0.f;
            for (int l = 0; l < sh.lanes; ++l) { q0 += e0[l * wide + c - c0]; q1 += e1[l * wide + c - c0]; }
            chan[c] = q0;
            chan[a.C + c] = q1;
            e0[c - c0] = q0;                            // (row 0 of the entries, read here alone: the groups sum from it)
            e1[c - c0] = q1;
        }
        __syncthreads();
        gn_groups<2>(c0, c1, cg, 1, carry[pass & 1], carry[~pass & 1],
            [&](int, int c, double *v) {
                const double w = gn_param(a.weight, a.wdtype, c, 1.f);
                v[0] = fma(w, (double)e0[c - c0], v[0]);
                v[1] = fma(w, (double)e1[c - c0], v[1]);
            },
            [&](int g, const double *v) { pair[g] = make_float2((float)v[0], (float)v[1]); });
        __syncthreads();
    }
}

// second launch: the first workgroups sum dweight and dbias over chunks and batch (GN_PARAM channels each), the others write dx
#define GN_PARAM 16
template <typename T, int VEC, bool SILU, bool MASKED> __global__ void __launch_bounds__(GN_T) vq_gn_bwd_apply_kernel(const GnArgs a, unsigned param_blocks)
{
    extern __shared__ __align__(16) float2 stat[];      // (mean(dz w), mean(dz w xh)) [G]; the first workgroups' partial sums
    const int t = threadIdx.x, G = a.G, cg = a.C / G;
    if (blockIdx.x < param_blocks) {
        double (*red)[GN_T / GN_PARAM][GN_PARAM] = (double (*)[GN_T / GN_PARAM][GN_PARAM])stat;          // (with it, 8192 groups would pass 64 KB)
        const int c = blockIdx.x * GN_PARAM + t % GN_PARAM, q = t / GN_PARAM;
        double v0 = 0.0, v1 = 0.0;
        if (c < a.C)
#pragma unroll 8
            for (int64_t s = q; s < a.B * a.S; s += GN_T / GN_PARAM) { v0 += a.chan[s * a.C * 2 + c]; v1 += a.chan[s * a.C * 2 + a.C + c]; }
        red[0][q][t % GN_PARAM] = v0;
        red[1][q][t % GN_PARAM] = v1;
        __syncthreads();
        if (q == 0 && c < a.C) {
            for (int k = 1; k < GN_T / GN_PARAM; ++k) { v0 += red[0][k][t]; v1 += red[1][k][t]; }
            if (a.dbias) gn_store_param(a.dbias, a.wdtype, c, (float)v0);
            if (a.dweight) gn_store_param(a.dweight, a.wdtype, c, (float)v1);
        }
        return;
    }
    const unsigned block = blockIdx.x - param_blocks;
    const int chunk = block % (unsigned)a.S;
    const int64_t b = block / (unsigned)a.S, len = gn_len(a, b), r0 = (int64_t)chunk * a.rows, end = r0 + a.rows < a.N ? r0 + a.rows : a.N, r1 = end < len ? end : len;
    gn_join<true>(a, b, stat);
    __syncthreads();
    const GnShape sh = gn_shape<VEC>(a.C);
    const int lane = t / sh.width;
    if (lane >= sh.lanes) return;
    const T *x = (const T *)a.x + b * a.xb, *gr = (const T *)a.grad + b * a.N * a.C;
    T *dx = (T *)a.dx + b * a.N * a.C;
    const uint8_t *mask = MASKED ? a.mask + b * a.N : nullptr;
    for (int col = t % sh.width; col < sh.cols; col += sh.width) {
        float mean[VEC], rstd[VEC], w[VEC], bias[VEC], m1[VEC], m2[VEC];
        gn_params<VEC>(a.weight, a.wdtype, col * VEC, 1.f, w);
        gn_params<VEC>(a.bias, a.wdtype, col * VEC, 0.f, bias);
        GnGroup of(col * VEC, cg);
#pragma unroll
        for (int i = 0; i < VEC; ++i, of.next()) {
            mean[i] = a.mean[b * G + of.g];
            rstd[i] = a.rstd[b * G + of.g];
            m1[i] = stat[of.g].x;
            m2[i] = stat[of.g].y;
        }
        for (int64_t r = r0 + lane; r < r1; r += 2 * sh.lanes) {
            VqVec<T, VEC> v[2], d[2];
            bool live[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t at = r + (int64_t)u * sh.lanes, in = at < r1 ? at : r1 - 1;
                live[u] = at < r1 && (!MASKED || mask[in]);
                v[u] = vq_ldv<T, VEC>(x + in * a.xn + (int64_t)col * VEC);
                d[u] = vq_ldv<T, VEC>(gr + in * a.C + (int64_t)col * VEC);
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const int64_t at = r + (int64_t)u * sh.lanes;
                if (at >= r1) break;
                VqVec<T, VEC> o;
#pragma unroll
                for (int i = 0; i < VEC; ++i) {
                    const float xh = ((float)v[u].v[i] - mean[i]) * rstd[i], dz = gn_dz<SILU>((float)d[u].v[i], xh, w[i], bias[i]);
                    o.v[i] = !MASKED || live[u] ? (T)(rstd[i] * (fmaf(dz, w[i], -m1[i]) - xh * m2[i])) : (T)0.f;
                }
                vq_stv<T, VEC>(dx + at * a.C + (int64_t)col * VEC, o);
            }
        }
        gn_zero_rows<T, VEC>(dx + (int64_t)col * VEC, (r0 > len ? r0 : len) + lane, end, sh.lanes, a.C);
    }
}

__global__ void __launch_bounds__(256) vq_gn_zero_params_kernel(void *dweight, void *dbias, int dtype, int C)
{
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= C) return;
    if (dweight) gn_store_param(dweight, dtype, c, 0.f);
    if (dbias) gn_store_param(dbias, dtype, c, 0.f);
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
// Two workgroups a CU in all, at most 256 chunks of an entry, at least 8192 elements each.  (6 x 65536 x 128 bf16, second launch: 45 us with
// 1020 workgroups of 256 threads that each join 170 chunks, 38 us with half as many.)
static void gn_plan(int64_t B, int64_t N, int64_t C, int64_t *S, int64_t *rows)
{
    int64_t s = B >= 512 ? 1 : 512 / B;
    if (s > 256) s = 256;
    const int64_t least = C >= 8192 ? 1 : 8192 / C;
    int64_t r = (N + s - 1) / s;
    if (r < least) r = least;
    *rows = r;
    *S = (N + r - 1) / r;
}

static int gn_check(const vqhip_group_norm_t *p, const char *what)
{
    if (!p) VQ_FAIL(VQHIP_EINVAL, "%s: null argument", what);
    if (!vq_elem_bytes(p->dtype) || !vq_elem_bytes(p->param_dtype)) VQ_FAIL(VQHIP_EINVAL, "%s: dtype %lld, parameters of %lld", what, (long long)p->dtype, (long long)p->param_dtype);
    if (p->B < 0 || p->N < 0 || p->C < 1 || p->groups < 1 || p->C % p->groups || !(p->eps >= 0.0)) VQ_FAIL(VQHIP_EINVAL, "%s: B %lld, N %lld, C %lld in %lld groups, eps %g", what, (long long)p->B, (long long)p->N, (long long)p->C, (long long)p->groups, p->eps);
    if (p->activation != VQHIP_ACT_NONE && p->activation != VQHIP_ACT_SILU) VQ_FAIL(VQHIP_EINVAL, "%s: activation %lld", what, (long long)p->activation);
    if (p->C > VQHIP_NORM_MAX_C || p->B > (1 << 22) || p->N > ((int64_t)1 << 31) / p->C * 256) VQ_FAIL(VQHIP_EDIM, "%s: %lld x %lld rows of %lld channels (at most 2^22 entries, 2^39 elements each, %d channels)", what, (long long)p->B, (long long)p->N, (long long)p->C, VQHIP_NORM_MAX_C);
    if (p->lens && p->mask) VQ_FAIL(VQHIP_EINVAL, "%s: lens and mask", what);
    if (p->B > 0 && p->N > 0 && (!p->x || !p->mean || !p->rstd)) VQ_FAIL(VQHIP_EINVAL, "%s: null pointer", what);
    const size_t need = vqhip_group_norm_workspace_bytes(p->B, p->N, p->C, p->groups);
    if (p->workspace_bytes < need || (need && !p->workspace)) VQ_FAIL(VQHIP_EINVAL, "%s: workspace of %zu bytes, needs %zu", what, p->workspace_bytes, need);
    if ((uintptr_t)p->workspace & 15) VQ_FAIL(VQHIP_EALIGN, "%s: workspace not 16-byte aligned", what);
    return 0;
}

static GnArgs gn_args(const vqhip_group_norm_t *p)
{
    GnArgs a;
    int64_t S, rows;
    gn_plan(p->B, p->N, p->C, &S, &rows);
    a.x = p->x; a.xb = p->stride_b; a.xn = p->stride_n; a.weight = p->weight; a.bias = p->bias; a.lens = p->lens; a.mask = p->mask;
    a.y = nullptr; a.mean = p->mean; a.rstd = p->rstd; a.grad = nullptr; a.dx = a.dweight = a.dbias = nullptr;
    a.N = p->N; a.B = p->B; a.C = (int)p->C; a.G = (int)p->groups; a.act = (int)p->activation; a.wdtype = (int)p->param_dtype;
    a.S = (int)S; a.rows = rows; a.eps = p->eps;
    a.pair = (float2 *)p->workspace; a.joined = a.pair + p->B * S * p->groups; a.chan = (float *)(a.joined + p->B * p->groups); a.live = a.chan + p->B * S * 2 * p->C;
    if (S == 1 || S * p->groups <= GN_JOIN) a.joined = nullptr;           // (more chunks than one: B <= 256)
    return a;
}

// the span of vq_gn_one_kernel and its rows a thread; U 0: two launches.  The widest of up to 128 bytes that leaves a workgroup to every CU,
// else the narrowest: a small map wants its rows over as many CUs as there are.  One launch and two, us a call, C channels in G groups:
//   a launch saved, all small maps       1 x 256 x 512 / 32 bf16 14.1 and 16.6, 16 x 1024 x 256 / 32 fp32 14.5 and 16.9
//   x read once from HBM                 122 x 256 x 512 / 32 fp32 24 and 36, 4096 x 256 x 64 / 8 fp32 104 and 162
//   a thread of more than 64 values      122 x 1024 x 256 / 32 bf16 45 and 37: not taken
//   stripes of less than half a line     122 x 4096 x 64 / 8 fp32 (32 bytes) 126 and 66, threads whose channels lie in several groups 1953 x 64 x
//                                        128 / 32 bf16 70 and 47: taken up to 4 MB, what an XCD's L2 holds
//   many small workgroups                3906 x 16 x 256 / 32 bf16 (2 KB each) 109 and 71: not taken, beyond what the CUs hold at once, below 32 KB
//                                        each and where two spans do not make a row (7812 x 16 x 64 / 8 bf16 57 and 140)
struct GnOne { int span, U; };
static GnOne gn_one(int64_t B, int64_t N, int C, int G, int elem)
{
    const int cg = C / G, vec = 16 / elem;
    GnOne best{0, 0};
    if (C % vec || cg > 64 || N > GN_T * 16 || B > (1 << 22) / G) return best;          // (a launch takes fewer than 2^32 threads)
    for (int k = 1; k <= G; ++k) {
        const int span = cg * k, cols = span / vec;
        if (cols > 64 || (best.span && (span * elem > 128 || B * (C / span) < 256))) break;
        if (G % k || span % vec || cols & (cols - 1)) continue;
        const int lanes = GN_T / cols, rows = (int)((N + lanes - 1) / lanes);
        if (rows > 16) break;
        best = GnOne{span, rows <= 1 ? 1 : rows <= 4 ? 4 : 16};
    }
    if (!best.span) return best;
    const int64_t slab = N * best.span * elem, slabs = B * (C / best.span);
    if (best.U * vec > 64 || (slabs * slab > (4 << 20) && (best.span * elem < 64 || cg % vec)) || (slabs > 2048 && slab < 32768 && 2 * best.span < C)) best.U = 0;
    return best;
}

template <typename T, int VEC, int U> static void gn_one_launch(const GnArgs &a, int span, hipStream_t st)
{
    const dim3 grid((unsigned)(a.B * (a.C / span)));
    if (a.act == VQHIP_ACT_SILU) {
        if (a.mask) vq_gn_one_kernel<T, VEC, U, true, true><<<grid, GN_T, 0, st>>>(a, span);
        else vq_gn_one_kernel<T, VEC, U, true, false><<<grid, GN_T, 0, st>>>(a, span);
    } else {
        if (a.mask) vq_gn_one_kernel<T, VEC, U, false, true><<<grid, GN_T, 0, st>>>(a, span);
        else vq_gn_one_kernel<T, VEC, U, false, false><<<grid, GN_T, 0, st>>>(a, span);
    }
}
template <typename T> static void gn_one_rows(const GnArgs &a, const GnOne &o, hipStream_t st)
{
    constexpr int VEC = 16 / sizeof(T);
    if (o.U == 1) gn_one_launch<T, VEC, 1>(a, o.span, st);
    else if (o.U == 4) gn_one_launch<T, VEC, 4>(a, o.span, st);
    else if constexpr (sizeof(T) == 4) gn_one_launch<T, VEC, 16>(a, o.span, st);
}

extern "C" size_t vqhip_group_norm_workspace_bytes(int64_t B, int64_t N, int64_t C, int64_t groups)
{
    if (B <= 0 || N <= 0 || C <= 0 || groups <= 0) return 0;
    int64_t S, rows;
    gn_plan(B, N, C, &S, &rows);
    return ((size_t)(B * S) * (size_t)(1 + 2 * groups + 2 * C) + (size_t)(B * groups) * 2) * 4;
}

// channels of a thread: 16 bytes where C divides so, fewer where not
#define GN_BY_VEC(T, MOST, C, call)                                                                       \
    do {                                                                                                  \
        if ((C) % (MOST) == 0) { constexpr int VEC = MOST; call; }                                        \
        else if ((C) % 2 == 0) { constexpr int VEC = 2; call; }                                           \
        else { constexpr int VEC = 1; call; }                                                             \
    } while (0)
#define GN_BY_MASK(mask, call)                                                                            \
    do {                                                                                                  \
        if (mask) { constexpr bool MASKED = true; call; } else { constexpr bool MASKED = false; call; }   \
    } while (0)
#define GN_BY_TYPE(dtype, C, call)                                                                        \
    do {                                                                                                  \
        if ((dtype) == VQHIP_F32) { using T = float; GN_BY_VEC(T, 4, C, call); }                          \
        else if ((dtype) == VQHIP_BF16) { using T = __bf16; GN_BY_VEC(T, 8, C, call); }                   \
        else { using T = _Float16; GN_BY_VEC(T, 8, C, call); }                                            \
    } while (0)

extern "C" int vqhip_group_norm(const vqhip_group_norm_t *p, void *y, void *stream)
{
    int rc = gn_check(p, "vqhip_group_norm");
    if (rc) return rc;
    if (p->B == 0 || p->N == 0) return 0;
    if (!y) VQ_FAIL(VQHIP_EINVAL, "vqhip_group_norm: null pointer");
    GnArgs a = gn_args(p);
    a.y = y;
    hipStream_t st = (hipStream_t)stream;
    const GnOne one = gn_one(a.B, a.N, a.C, a.G, vq_elem_bytes(p->dtype));
    if (one.U) {
        if (p->dtype == VQHIP_F32) gn_one_rows<float>(a, one, st);
        else if (p->dtype == VQHIP_BF16) gn_one_rows<__bf16>(a, one, st);
        else gn_one_rows<_Float16>(a, one, st);
        return vq_launch_status("vqhip_group_norm");
    }
    const dim3 grid((unsigned)(a.B * a.S));
    const size_t sm = (size_t)a.G * 8;
    GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_stats_kernel<T, VEC, MASKED><<<grid, GN_T, 0, st>>>(a))));
    if (a.joined) vq_gn_join_kernel<false><<<dim3((unsigned)((a.B * a.G + 3) / 4)), 256, 0, st>>>(a);
    if (a.act == VQHIP_ACT_SILU) GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_apply_kernel<T, VEC, true, MASKED><<<grid, GN_T, sm, st>>>(a))));
    else GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_apply_kernel<T, VEC, false, MASKED><<<grid, GN_T, sm, st>>>(a))));
    return vq_launch_status("vqhip_group_norm");
}

extern "C" int vqhip_group_norm_bwd(const vqhip_group_norm_t *p, const void *grad, void *dx, void *dweight, void *dbias, void *stream)
{
    int rc = gn_check(p, "vqhip_group_norm_bwd");
    if (rc) return rc;
    if (!dx && !dweight && !dbias) return 0;
    hipStream_t st = (hipStream_t)stream;
    if (p->B == 0 || p->N == 0) {
        if (dweight || dbias) vq_gn_zero_params_kernel<<<dim3((unsigned)((p->C + 255) / 256)), 256, 0, st>>>(dweight, dbias, (int)p->param_dtype, (int)p->C);
        return vq_launch_status("vqhip_group_norm_bwd");
    }
    if (!grad) VQ_FAIL(VQHIP_EINVAL, "vqhip_group_norm_bwd: null pointer");
    GnArgs a = gn_args(p);
    a.grad = grad; a.dx = dx; a.dweight = dweight; a.dbias = dbias;
    const dim3 grid((unsigned)(a.B * a.S));
    const unsigned params = dweight || dbias ? (unsigned)((a.C + GN_PARAM - 1) / GN_PARAM) : 0;
    const dim3 both(params + (dx ? (unsigned)(a.B * a.S) : 0));
    const size_t sums = (size_t)2 * GN_T * 8, sm = (size_t)a.G * 8 > sums ? (size_t)a.G * 8 : sums;
    if (a.act == VQHIP_ACT_SILU) {
        GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_bwd_sums_kernel<T, VEC, true, MASKED><<<grid, GN_T, 0, st>>>(a))));
        if (a.joined && dx) vq_gn_join_kernel<true><<<dim3((unsigned)((a.B * a.G + 3) / 4)), 256, 0, st>>>(a);
        GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_bwd_apply_kernel<T, VEC, true, MASKED><<<both, GN_T, sm, st>>>(a, params))));
    } else {
        GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_bwd_sums_kernel<T, VEC, false, MASKED><<<grid, GN_T, 0, st>>>(a))));
        if (a.joined && dx) vq_gn_join_kernel<true><<<dim3((unsigned)((a.B * a.G + 3) / 4)), 256, 0, st>>>(a);
        GN_BY_TYPE(p->dtype, a.C, GN_BY_MASK(a.mask, (vq_gn_bwd_apply_kernel<T, VEC, false, MASKED><<<both, GN_T, sm, st>>>(a, params))));
    }
    return vq_launch_status("vqhip_group_norm_bwd");
}

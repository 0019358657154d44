// vq_beam.hip -- beam search over codes (or any vocabulary): the selection over beams and continuations with its gradient, and the
// reordering of the beams' states with its gradient.
#include "vq_elem.h"

#include <math.h>

// ---- selection -------------------------------------------------------------------------------------------------------------------
// c[b, j, v] = s[b, j] + (l[b, j, v] - lse[b, j]) (normalize) or s + l; a finished beam has one continuation, c = s at end_token; what
// the mask leaves out, and every sum that is not a number, is -inf.  Out: the K largest c of a batch entry, equal ones by ascending
// j * V + v.  Sums and comparisons are 64-bit: two continuations of different beams may be closer than fp32 resolves.
struct SelArgs {
    const void *logits; int64_t lb, lj;                 // element strides of batch and beam
    const float *scores;                                // [B, J] or null (zeros)
    const uint8_t *mask; int64_t mb, mj;                // byte strides; null: everything admitted
    const uint8_t *finished;                            // [B, J] or null
    float *scores_out; int64_t *parents_out, *tokens_out; double *lse_out;
    int64_t B; int J, V, K, end_token, normalize;
};

__device__ __forceinline__ double sel_sum(double score, double x)
{
    const double c = score + x;
    return c != c ? -INFINITY : c;
}

template <typename T> __global__ void __launch_bounds__(256) vq_beam_select_kernel(const SelArgs a)
{
    extern __shared__ double smem[];
    double *lse = smem, *red = smem + a.J;              // [J], [256]
    int *redi = (int *)(red + 256);                     // [256]
    const int64_t b = blockIdx.x;
    const int t = threadIdx.x, J = a.J, V = a.V;
    const T *lg = (const T *)a.logits + b * a.lb;
    const uint8_t *mk = a.mask ? a.mask + b * a.mb : nullptr;
    for (int j = 0; j < J; ++j) {
        double out = 0.0;
        if (a.normalize) {
            const T *row = lg + j * a.lj;
            const uint8_t *m = mk ? mk + j * a.mj : nullptr;
            double mx = -INFINITY;
            for (int v = t; v < V; v += 256)
                if (!m || m[v]) mx = fmax(mx, (double)(float)row[v]);
            red[t] = mx;
            __syncthreads();
            for (int o = 128; o; o >>= 1) {
                if (t < o) red[t] = fmax(red[t], red[t + o]);
                __syncthreads();
            }
            mx = red[0];
            __syncthreads();
            double s = 0.0;
            for (int v = t; v < V; v += 256)
                if (!m || m[v]) s += exp((double)(float)row[v] - mx);
            red[t] = s;
            __syncthreads();
            for (int o = 128; o; o >>= 1) {
                if (t < o) red[t] += red[t + o];
                __syncthreads();
            }
            out = mx + log(red[0]);
            __syncthreads();
        }
        if (t == 0) {
            lse[j] = out;
            if (a.lse_out) a.lse_out[b * J + j] = out;
        }
    }
    __syncthreads();
    double last = INFINITY;
    int lasti = -1;
    const int total = J * V;
    for (int k = 0; k < a.K; ++k) {
        double best = -INFINITY;
        int bi = 0x7fffffff;
        for (int i = t; i < total; i += 256) {
            const int j = i / V, v = i - j * V;
            const double s = a.scores ? (double)a.scores[b * J + j] : 0.0;
            double c;
            if (a.finished && a.finished[b * J + j]) c = sel_sum(s, v == a.end_token ? 0.0 : -INFINITY);
            else if (mk && !mk[j * a.mj + v]) c = -INFINITY;
            else c = sel_sum(s, (double)(float)lg[j * a.lj + v] - lse[j]);
            const bool open = c < last || (c == last && i > lasti);
            if (open && (c > best || (c == best && i < bi))) { best = c; bi = i; }
        }
        red[t] = best;
        redi[t] = bi;
        __syncthreads();
        for (int o = 128; o; o >>= 1) {
            if (t < o && (red[t + o] > red[t] || (red[t + o] == red[t] && redi[t + o] < redi[t]))) { red[t] = red[t + o]; redi[t] = redi[t + o]; }
            __syncthreads();
        }
        last = red[0];
        lasti = redi[0];
        __syncthreads();
        if (t == 0) {
            a.scores_out[b * a.K + k] = (float)last;
            a.parents_out[b * a.K + k] = lasti / V;
            a.tokens_out[b * a.K + k] = lasti % V;
        }
    }
}

static int sel_check(const vqhip_beam_select_t *p, const char *what)
{
    if (!p) VQ_FAIL(VQHIP_EINVAL, "%s: null argument", what);
    if (!vq_elem_bytes(p->dtype)) VQ_FAIL(VQHIP_EINVAL, "%s: dtype %lld", what, (long long)p->dtype);
    if (p->B < 0 || p->J < 1 || p->V < 1 || p->K < 1) VQ_FAIL(VQHIP_EINVAL, "%s: B %lld, J %lld, V %lld, K %lld", what, (long long)p->B, (long long)p->J, (long long)p->V, (long long)p->K);
    if (p->J > VQHIP_BEAM_MAX || p->K > VQHIP_BEAM_MAX || p->B > 0x7fffffff || p->V > 0x7fffffff / p->J || p->K > p->J * p->V)
        VQ_FAIL(VQHIP_EDIM, "%s: %lld beams, %lld kept of %lld x %lld continuations: at most %d beams, %d kept, 2^31 - 1 continuations", what,
                (long long)p->J, (long long)p->K, (long long)p->J, (long long)p->V, VQHIP_BEAM_MAX, VQHIP_BEAM_MAX);
    if (p->finished && (p->end_token < 0 || p->end_token >= p->V)) VQ_FAIL(VQHIP_EINVAL, "%s: end token %lld outside [0, %lld)", what, (long long)p->end_token, (long long)p->V);
    if (p->B > 0 && (!p->logits || !p->parents || !p->tokens || !p->out_scores)) VQ_FAIL(VQHIP_EINVAL, "%s: null pointer", what);
    return 0;
}

extern "C" size_t vqhip_beam_select_workspace_bytes(int64_t B, int64_t J, int64_t V, int64_t K)
{
    (void)B; (void)J; (void)V; (void)K;
    return 0;
}

extern "C" int vqhip_beam_select(const vqhip_beam_select_t *p, void *stream)
{
    int rc = sel_check(p, "vqhip_beam_select");
    if (rc) return rc;
    if (p->B == 0) return 0;
    SelArgs a;
    a.logits = p->logits; a.lb = p->stride_b; a.lj = p->stride_j; a.scores = p->scores;
    a.mask = p->mask; a.mb = p->mask_stride_b; a.mj = p->mask_stride_j; a.finished = p->finished;
    a.scores_out = p->out_scores; a.parents_out = p->parents; a.tokens_out = p->tokens; a.lse_out = p->lse;
    a.B = p->B; a.J = (int)p->J; a.V = (int)p->V; a.K = (int)p->K; a.end_token = (int)p->end_token; a.normalize = p->normalize != 0;
    const size_t sm = (size_t)(a.J + 256) * 8 + 256 * 4;
    const dim3 grid((unsigned)p->B);
    if (p->dtype == VQHIP_F32) vq_beam_select_kernel<float><<<grid, 256, sm, (hipStream_t)stream>>>(a);
    else if (p->dtype == VQHIP_BF16) vq_beam_select_kernel<__bf16><<<grid, 256, sm, (hipStream_t)stream>>>(a);
    else vq_beam_select_kernel<_Float16><<<grid, 256, sm, (hipStream_t)stream>>>(a);
    return vq_launch_status("vqhip_beam_select");
}

// d_scores[b, j] = sum of g over the kept continuations of beam j; d_logits[b, j, v] = sum of g over those with token v, minus (normalize)
// d_scores[b, j] * softmax(l)[b, j, v].  A continuation of score -inf is none: its g counts as 0.  Finished beams pass nothing on to logits.
struct SelBwdArgs {
    const void *logits; int64_t lb, lj;
    const uint8_t *mask; int64_t mb, mj;
    const uint8_t *finished; const double *lse;
    const float *scores_out; const int64_t *parents, *tokens; const float *grad;
    void *d_logits; float *d_scores;
    int64_t B; int J, V, K, normalize;
};

template <typename T> __global__ void __launch_bounds__(256) vq_beam_select_bwd_kernel(const SelBwdArgs a)
{
    __shared__ float g[VQHIP_BEAM_MAX];
    __shared__ int tok[VQHIP_BEAM_MAX];
    __shared__ int n;
    __shared__ float onto;
    const int64_t b = blockIdx.x / a.J;
    const int j = blockIdx.x % a.J, t = threadIdx.x, V = a.V;
    if (t == 0) {
        int m = 0;
        float s = 0.f;
        for (int k = 0; k < a.K; ++k)
            if (a.parents[b * a.K + k] == j && a.scores_out[b * a.K + k] > -INFINITY) {
                g[m] = a.grad[b * a.K + k];
                tok[m] = (int)a.tokens[b * a.K + k];
                s += g[m++];
            }
        if (a.d_scores) a.d_scores[b * a.J + j] = s;
        onto = s;
        n = a.finished && a.finished[b * a.J + j] ? -1 : m;
    }
    __syncthreads();
    if (!a.d_logits) return;
    const T *row = (const T *)a.logits + b * a.lb + j * a.lj;
    const uint8_t *mk = a.mask ? a.mask + b * a.mb + j * a.mj : nullptr;
    T *out = (T *)a.d_logits + (b * a.J + j) * (int64_t)V;
    const double lse = a.normalize ? a.lse[b * a.J + j] : 0.0;
    for (int v = t; v < V; v += 256) {
        float d = 0.f;
        if (n > 0 && (!mk || mk[v])) {
            for (int i = 0; i < n; ++i)
                if (tok[i] == v) d += g[i];
            if (a.normalize) d -= onto * (float)exp((double)(float)row[v] - lse);
        }
        out[v] = (T)d;
    }
}

extern "C" int vqhip_beam_select_bwd(const vqhip_beam_select_t *p, const float *grad, void *d_logits, float *d_scores, void *stream)
{
    int rc = sel_check(p, "vqhip_beam_select_bwd");
    if (rc) return rc;
    if (p->B == 0 || (!d_logits && !d_scores)) return 0;
    if (!grad || (p->normalize && d_logits && !p->lse)) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_select_bwd: null pointer");
    if (p->B * p->J > 0x7fffffff) VQ_FAIL(VQHIP_EDIM, "vqhip_beam_select_bwd: %lld x %lld rows", (long long)p->B, (long long)p->J);
    SelBwdArgs a;
    a.logits = p->logits; a.lb = p->stride_b; a.lj = p->stride_j; a.mask = p->mask; a.mb = p->mask_stride_b; a.mj = p->mask_stride_j;
    a.finished = p->finished; a.lse = p->lse; a.scores_out = p->out_scores; a.parents = p->parents; a.tokens = p->tokens; a.grad = grad;
    a.d_logits = d_logits; a.d_scores = d_scores;
    a.B = p->B; a.J = (int)p->J; a.V = (int)p->V; a.K = (int)p->K; a.normalize = p->normalize != 0;
    const dim3 grid((unsigned)(p->B * p->J));
    if (p->dtype == VQHIP_F32) vq_beam_select_bwd_kernel<float><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else if (p->dtype == VQHIP_BF16) vq_beam_select_bwd_kernel<__bf16><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    else vq_beam_select_bwd_kernel<_Float16><<<grid, 256, 0, (hipStream_t)stream>>>(a);
    return vq_launch_status("vqhip_beam_select_bwd");
}

// ---- reordering ------------------------------------------------------------------------------------------------------------------
// out[b, i] = state[b, parents[b, i]] for every state of the call in one launch; a parent outside [0, J) gives zeros.  A state's row is
// n1 pieces of `run` contiguous bytes, s1 bytes apart (a cache whose rows are cut to the positions in use); out is contiguous.
struct ReorderState { const char *src; char *dst; int64_t sb, sj, s1, run; int64_t n1; };
struct ReorderArgs {
    ReorderState s[VQHIP_BEAM_STATES];
    const int64_t *parents;
    int64_t B; int J, K;
};

__global__ void __launch_bounds__(256) vq_beam_reorder_kernel(const ReorderArgs a)
{
    const ReorderState s = a.s[blockIdx.y];
    const int64_t row = s.n1 * s.run, total = a.B * a.K * row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / row, w = i - r * row, b = r / a.K, n = w / s.run;
        const int64_t p = a.parents[r];
        s.dst[i] = p < 0 || p >= a.J ? 0 : s.src[b * s.sb + p * s.sj + n * s.s1 + (w - n * s.run)];
    }
}

// d_state[b, j] = sum of grad[b, i] over parents[b, i] == j, ascending i, in 32 bits and rounded once; both contiguous
struct ReorderBwdState { const void *grad; void *out; int64_t row; int dtype; };
struct ReorderBwdArgs {
    ReorderBwdState s[VQHIP_BEAM_STATES];
    const int64_t *parents;
    int64_t B; int J, K;
};

template <typename T> __device__ __forceinline__ void reorder_bwd_at(const ReorderBwdArgs &a, const ReorderBwdState &s, int64_t i)
{
    const int64_t r = i / s.row, w = i - r * s.row, b = r / a.J;
    const int j = (int)(r - b * a.J);
    float d = 0.f;
    for (int k = 0; k < a.K; ++k)
        if (a.parents[b * a.K + k] == j) d += (float)((const T *)s.grad)[(b * a.K + k) * s.row + w];
    ((T *)s.out)[i] = (T)d;
}

__global__ void __launch_bounds__(256) vq_beam_reorder_bwd_kernel(const ReorderBwdArgs a)
{
    const ReorderBwdState s = a.s[blockIdx.y];
    const int64_t total = a.B * a.J * s.row;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        if (s.dtype == VQHIP_F32) reorder_bwd_at<float>(a, s, i);
        else if (s.dtype == VQHIP_BF16) reorder_bwd_at<__bf16>(a, s, i);
        else reorder_bwd_at<_Float16>(a, s, i);
    }
}

static int reorder_check(int64_t n, const void *states, const int64_t *parents, int64_t B, int64_t J, int64_t K, const char *what)
{
    if (n < 0 || n > VQHIP_BEAM_STATES || B < 0 || J < 1 || K < 1) VQ_FAIL(VQHIP_EINVAL, "%s: %lld states (at most %d), B %lld, J %lld, K %lld", what, (long long)n, VQHIP_BEAM_STATES, (long long)B, (long long)J, (long long)K);
    if (J > 0x7fffffff || K > 0x7fffffff || B > 0x7fffffff / J || B > 0x7fffffff / K) VQ_FAIL(VQHIP_EDIM, "%s: %lld x %lld rows from %lld x %lld", what, (long long)B, (long long)K, (long long)B, (long long)J);
    if (n > 0 && B > 0 && (!states || !parents)) VQ_FAIL(VQHIP_EINVAL, "%s: null pointer", what);
    return 0;
}

extern "C" int vqhip_beam_reorder(const vqhip_beam_state_t *states, int64_t n, const int64_t *parents, int64_t B, int64_t J, int64_t K, void *stream)
{
    int rc = reorder_check(n, states, parents, B, J, K, "vqhip_beam_reorder");
    if (rc) return rc;
    ReorderArgs a;
    int m = 0;
    int64_t most = 0;
    for (int64_t i = 0; i < n && B > 0; ++i) {
        const vqhip_beam_state_t &s = states[i];
        if (s.pieces < 0 || s.piece_bytes < 0) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder: state %lld: %lld pieces of %lld bytes", (long long)i, (long long)s.pieces, (long long)s.piece_bytes);
        if (s.pieces == 0 || s.piece_bytes == 0) continue;
        if (!s.src || !s.dst) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder: state %lld: null pointer", (long long)i);
        a.s[m++] = ReorderState{(const char *)s.src, (char *)s.dst, s.stride_b, s.stride_j, s.piece_stride, s.piece_bytes, s.pieces};
        const int64_t tot = B * K * s.pieces * s.piece_bytes;
        if (tot > most) most = tot;
    }
    if (m == 0) return 0;
    a.parents = parents; a.B = B; a.J = (int)J; a.K = (int)K;
    const int64_t blocks = (most + 256 * 16 - 1) / (256 * 16);
    vq_beam_reorder_kernel<<<dim3((unsigned)(blocks > 65536 ? 65536 : blocks), (unsigned)m), 256, 0, (hipStream_t)stream>>>(a);
    return vq_launch_status("vqhip_beam_reorder");
}

extern "C" int vqhip_beam_reorder_bwd(const vqhip_beam_state_t *states, const int64_t *dtypes, int64_t n, const int64_t *parents, int64_t B, int64_t J, int64_t K, void *stream)
{
    int rc = reorder_check(n, states, parents, B, J, K, "vqhip_beam_reorder_bwd");
    if (rc) return rc;
    if (n > 0 && !dtypes) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder_bwd: null pointer");
    ReorderBwdArgs a;
    int m = 0;
    int64_t most = 0;
    for (int64_t i = 0; i < n && B > 0; ++i) {
        const vqhip_beam_state_t &s = states[i];
        const int eb = vq_elem_bytes(dtypes[i]);
        if (!eb || s.pieces < 0 || s.piece_bytes < 0 || s.piece_bytes % eb) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder_bwd: state %lld: dtype %lld, %lld pieces of %lld bytes", (long long)i, (long long)dtypes[i], (long long)s.pieces, (long long)s.piece_bytes);
        if (s.pieces == 0 || s.piece_bytes == 0) continue;
        if (!s.src || !s.dst) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder_bwd: state %lld: null pointer", (long long)i);
        a.s[m++] = ReorderBwdState{s.src, s.dst, s.pieces * s.piece_bytes / eb, (int)dtypes[i]};
        const int64_t tot = B * J * s.pieces * s.piece_bytes / eb;
        if (tot > most) most = tot;
    }
    if (m == 0) return 0;
    a.parents = parents; a.B = B; a.J = (int)J; a.K = (int)K;
    const int64_t blocks = (most + 256 * 4 - 1) / (256 * 4);
    vq_beam_reorder_bwd_kernel<<<dim3((unsigned)(blocks > 65536 ? 65536 : blocks), (unsigned)m), 256, 0, (hipStream_t)stream>>>(a);
    return vq_launch_status("vqhip_beam_reorder_bwd");
}

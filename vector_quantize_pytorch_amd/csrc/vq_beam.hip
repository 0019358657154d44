// vq_beam.hip -- beam search over codes (or any vocabulary): the selection over beams and continuations with its gradient, and the
// reordering of the beams' states with its gradient.
#include "vq_elem.h"

#include <math.h>

// ---- selection -------------------------------------------------------------------------------------------------------------------
// c[b, j, v] = s[b, j] + (l[b, j, v] - lse[b, j]) (normalize) or s + l; a finished beam has one continuation, c = s at end_token; what
// the mask leaves out, and every sum that is not a number, is -inf.  Out: the K largest c of a batch entry, equal ones by ascending
// j * V + v.  Sums and comparisons are 64-bit: two continuations of different beams may be closer than fp32 resolves.
//
// Within a row c grows with l, so the K best of a row are the K largest l (where 64 bits tell their c apart, see sel_places).  Two
// launches: vq_beam_rows_kernel reads every logit once (its tile stays in registers), and leaves of each tile the log-sum's maximum and
// sum and its K largest logits; vq_beam_merge_kernel joins the tiles of a batch entry's rows.  Bound by the read of the logits.
// vq_beam_small_kernel and vq_beam_entry_kernel do entries of up to 64 and SEL_ENTRY continuations in one launch.
struct SelArgs {
    const void *logits; int64_t lb, lj;                 // element strides of batch and beam
    int dtype;
    const float *scores;                                // [B, J] or null (zeros)
    const uint8_t *mask; int64_t mb, mj;                // byte strides; null: everything admitted
    const uint8_t *finished;                            // [B, J] or null
    float *scores_out; int64_t *parents_out, *tokens_out; double *lse_out;
    int64_t B; int J, V, K, end_token, normalize;
    // per (row, tile): the K largest (logit, token), unused ones -inf; maximum and sum of exp(l - maximum)
    int2 *part; double *part_sum; float *part_max; int tiles;
};

__device__ __forceinline__ double sel_sum(double score, double x)
{
    const double c = score + x;
    return c != c ? -INFINITY : c;
}

// the log-sum as it is handed out: none for a beam whose logits are not used (no tile of it need have been summed)
__device__ __forceinline__ double sel_lse(double lse, double score, bool finished) { return !finished && score > -INFINITY ? lse : (double)NAN; }

__device__ __forceinline__ bool sel_before(double c, int i, double d, int k) { return c > d || (c == d && i < k); }

// the entry's last survivors where fewer than K continuations are above -inf: the first places, by number, that are not among the `found`
// ones.  One thread.
__device__ void sel_fill(const SelArgs &a, int64_t b, int found)
{
    int place = 0;
    for (int r = found; r < a.K; ++r, ++place) {
        for (bool taken = true; taken;) {
            taken = false;
            for (int i = 0; i < found; ++i)
                if (a.parents_out[b * a.K + i] * a.V + a.tokens_out[b * a.K + i] == place) taken = true;
            if (taken) ++place;
        }
        a.scores_out[b * a.K + r] = -INFINITY;
        a.parents_out[b * a.K + r] = place / a.V;
        a.tokens_out[b * a.K + r] = place % a.V;
    }
}

// ---- small entries: J * V <= 64, W = a power of two >= J * V lanes of a wave each, one continuation a lane.  A survivor's rank is the
// number of continuations before it.  Bound by the launch.
template <typename T> __global__ void __launch_bounds__(256) vq_beam_small_kernel(const SelArgs a, int W)
{
    const int lane = threadIdx.x & 63, i = lane & (W - 1), base = lane - i, J = a.J, V = a.V;
    const int64_t b = ((int64_t)blockIdx.x * 256 + threadIdx.x) / W;
    const bool in = b < a.B && i < J * V;
    const int64_t bb = b < a.B ? b : 0;
    const int j = in ? i / V : 0, v = in ? i - j * V : 0;
    double x = -INFINITY, s = 0.0;
    bool fin = false;
    if (in) {
        if (a.scores) s = a.scores[bb * J + j];
        fin = a.finished && a.finished[bb * J + j];
        if (!fin && (!a.mask || a.mask[bb * a.mb + j * a.mj + v])) x = (double)(float)((const T *)a.logits)[bb * a.lb + j * a.lj + v];
    }
    if (a.normalize) {
        const int row = base + j * V;
        double m = -INFINITY, e = 0.0;
        for (int t = 0; t < V; ++t) m = fmax(m, __shfl(x, row + t, 64));
        const double mine = exp(x - m);
        for (int t = 0; t < V; ++t) e += __shfl(mine, row + t, 64);
        const double lse = m + log(e);
        if (in && v == 0 && a.lse_out) a.lse_out[bb * J + j] = sel_lse(lse, s, fin);
        x -= lse;
    }
    if (fin) x = v == a.end_token ? 0.0 : -INFINITY;
    const double c = in ? sel_sum(s, x) : -INFINITY;
    int rank = 0;
    for (int t = 0; t < J * V; ++t) rank += sel_before(__shfl(c, base + t, 64), t, c, i) ? 1 : 0;
    if (in && rank < a.K) {
        a.scores_out[b * a.K + rank] = (float)c;
        a.parents_out[b * a.K + rank] = j;
        a.tokens_out[b * a.K + rank] = v;
    }
}

// ---- rows -------------------------------------------------------------------------------------------------------------------------
#define SEL_CAP 512            // continuations of a tile that the first bound lets through before it is made exact

__device__ __forceinline__ unsigned sel_order(float f)       // ascending like f; NaN never gets here
{
    const unsigned u = __float_as_uint(f + 0.f);              // (-0 + 0 = 0: the zeros are equal)
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float sel_value(unsigned u) { return __uint_as_float(u & 0x80000000u ? u ^ 0x80000000u : ~u); }

// a value that at least K (<= 64) of the wave's 64 values (sel_order's bits) are not below, the K-th largest cut to its upper 20 bits:
// bisection over the bits, a ballot each.  -inf where fewer than K are above it.
__device__ __forceinline__ float sel_kth(unsigned mine, int K)
{
    unsigned kth = 0;
#pragma unroll
    for (int bit = 31; bit >= 12; --bit) {
        const unsigned want = kth | 1u << bit;
        if (__popcll(__ballot(mine >= want)) >= K) kth = want;
    }
    return kth <= 0x007fffffu ? -INFINITY : sel_value(kth);
}

// exp(x) for x <= 0 (NaN stays NaN, -inf gives 0).  The product's rounding grows with |x|, but so falls the term: a term of weight e^-5
// is off by 5 steps of fp32, e^-5 of one in the sum.  Measured on normal logits of deviation 1 to 4, 1000 to 131071 of them: log-sums off
// by 2e-8 to 5e-8 rms, most of it the same for every row (the rounding of log2 e).
__device__ __forceinline__ float sel_exp(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504f); }

// i / of and i % of along i, i + step, ...: the divisions once
struct SelWalk {
    int q, r, dq, dr, of;
    __device__ SelWalk(int i, int of_, int step) : q(i / of_), r(i - q * of_), dq(step / of_), dr(step - dq * of_), of(of_) {}
    __device__ __forceinline__ void next() { q += dq; r += dr; if (r >= of) { r -= of; ++q; } }
};

// like sel_order in 64 bits, for scores
__device__ __forceinline__ unsigned long long sel_order64(double c)
{
    const unsigned long long u = (unsigned long long)__double_as_longlong(c + 0.0);
    return u >> 63 ? ~u : u | 1ull << 63;
}

// Where too many scores reach a first bound: a cut (value, last place among those equal to it) that at least K and at most `cap` (> K)
// are not behind.  Bisection over the ordered bits until that holds, among equal ones over the places (`places` in all).
// count(pred): how many of the workgroup's scores above -inf fulfil pred(ordered bits, place).
struct SelCut { unsigned long long value; int place; };
template <typename Count> __device__ __forceinline__ SelCut sel_cut(int K, int cap, int places, Count &&count)
{
    SelCut cut{0, 0x7fffffff};
#pragma unroll 1
    for (int bit = 63; bit >= 0; --bit) {
        const unsigned long long want = cut.value | 1ull << bit;
        const int n = count([&](unsigned long long o, int) { return o >= want; });
        if (n >= K) {
            cut.value = want;
            if (n <= cap) return cut;
        }
    }
    const unsigned long long kth = cut.value;
    const int above = count([&](unsigned long long o, int) { return o > kth; });
    int lo = 0, hi = places - 1;
    while (lo < hi) {                                         // the least place with `above` + (equal ones up to it) >= K
        const int mid = lo + (hi - lo) / 2;
        if (above + count([&](unsigned long long o, int p) { return o == kth && p <= mid; }) >= K) hi = mid; else lo = mid + 1;
    }
    cut.place = lo;
    return cut;
}
__device__ __forceinline__ bool sel_within(const SelCut &cut, unsigned long long o, int place) { return o > cut.value || (o == cut.value && place <= cut.place); }

// the sum of c over a workgroup of NT threads, for all of them; `red` holds NT / 64 ints
template <int NT> __device__ __forceinline__ int sel_count(int c, int *red)
{
    c = vq_wave_sum(c);
    if (NT == 64) return c;
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = c;
    __syncthreads();
    c = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) c += red[w];
    return c;
}

// ---- entries of up to NT * E continuations in one launch ------------------------------------------------------------------------------
// A workgroup (a wave for up to 1024) holds an entry's continuations, i = u * NT + t of thread t, as 64-bit scores; for the rows' log-sums the
// logits lie in LDS once, where lanes of a power of two sum a row.  The K best by a bound from 64 groups, sel_cut where more than CAP reach it
// (K near 64: 300 of 1024 or more do, and almost every entry of one wave takes it), and ranks.  Bound by instructions and the latency of its
// steps, so few waves an entry: 8192 entries of 32 x 32 fp32 with log-sums, K 32, 36 us with 16 a lane of one wave, 45 and 54 with 2 and 4 waves;
// 16384 of 16 x 16, K 16, 28 us with 4 a lane, 33 with 8.  Here and in two launches as below, us a call, 8192 entries:
//   16 x 16 K 16 17 and 143     32 x 32 K 32 40 and 323     4 x 1024 K 4 90 and 134, K 64 274 and 1056
//   8 x 512 K 4 88 and 77, K 16 99 and 95, K 32 118 and 140     2 x 2048 K 4 97 and 88, K 16 108 and 99, K 64 284 and 349
// and 256 entries of each with K up to 16 14.6 and 19.8: a launch saved where entries are few, a tenth lost where many have rows that fit a tile.
#define SEL_ENTRY 4096
template <typename T, int NT, int E> __global__ void __launch_bounds__(NT) vq_beam_entry_kernel(const SelArgs a)
{
    constexpr int CAP = NT == 64 ? 128 : 256;
    __shared__ float tile[NT * E + NT * E / 32];              // (a word more every 32: rows of 32 logits lie in different banks)
    __shared__ double base[VQHIP_BEAM_MAX], log_sum[VQHIP_BEAM_MAX], cs[CAP];
    __shared__ float group_max[64];
    __shared__ int ps[CAP], red[NT / 64], found;
    __shared__ uint8_t fin[VQHIP_BEAM_MAX];
    const int t = threadIdx.x, J = a.J, V = a.V, K = a.K, total = J * V;
    const SelWalk start(t, V, NT);
    const int64_t b = blockIdx.x;
    const T *lg = (const T *)a.logits + b * a.lb;
    const uint8_t *mk = a.mask ? a.mask + b * a.mb : nullptr;
    float x[E];
    {
        T raw[E];
        bool live[E];
        SelWalk at = start;
#pragma unroll
        for (int u = 0; u < E; ++u, at.next()) {              // loads without conditions; past the end, the first one again
            const bool in = u * NT + t < total;
            const int j = in ? at.q : 0, v = in ? at.r : 0;
            raw[u] = lg[j * a.lj + v];
            live[u] = in && (!mk || mk[j * a.mj + v]);
        }
#pragma unroll
        for (int u = 0; u < E; ++u) x[u] = live[u] ? (float)raw[u] : -INFINITY;
    }
    if (a.normalize)
#pragma unroll
        for (int u = 0; u < E; ++u) {
            const int i = u * NT + t;
            if (i < total) tile[i + (i >> 5)] = x[u];
        }
    if (t == 0) found = 0;
    __syncthreads();
    int w = 64;                                               // lanes of a row
    while (w > 1 && w * J > NT) w >>= 1;
    for (int j = t / w; j < (J + NT / w - 1) / (NT / w) * (NT / w); j += NT / w) {
        const bool row = j < J;
        double lse = 0.0;
        if (a.normalize) {
            float top = -INFINITY;
            double sum = 0.0;
            if (row)
#pragma unroll 8
                for (int v = t % w; v < V; v += w) { const int i = j * V + v; top = fmaxf(top, tile[i + (i >> 5)]); }
            for (int o = w >> 1; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
            if (row)
                for (int v = t % w; v < V; v += 8 * w) {      // 8 terms in 32 bits, the rest in 64
                    float q = 0.f;
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int i = j * V + (v + k * w < V ? v + k * w : v);
                        const float e = sel_exp(tile[i + (i >> 5)] - top);
                        q += v + k * w < V ? e : 0.f;
                    }
                    sum += q;
                }
            for (int o = w >> 1; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
            lse = (double)top + log(sum);                     // (no logit admitted, one of +inf or NaN: not finite)
        }
        if (row && t % w == 0) {
            const double s = a.scores ? (double)a.scores[b * J + j] : 0.0;
            const bool f = a.finished && a.finished[b * J + j];
            fin[j] = f;
            base[j] = f || (s > -INFINITY && lse > -INFINITY && lse < INFINITY) ? s : -INFINITY;
            log_sum[j] = lse;
            if (a.lse_out) a.lse_out[b * J + j] = sel_lse(lse, s, f);
        }
    }
    __syncthreads();
    double c[E], best = -INFINITY;
    {
        SelWalk at = start;
#pragma unroll
        for (int u = 0; u < E; ++u, at.next()) {
            c[u] = -INFINITY;
            if (u * NT + t < total) {
                const double s = base[at.q];
                if (fin[at.q]) c[u] = at.r == a.end_token ? sel_sum(s, 0.0) : -INFINITY;
                else if (s > -INFINITY && x[u] > -INFINITY) c[u] = sel_sum(s, (double)x[u] - log_sum[at.q]);
            }
            best = fmax(best, c[u]);
        }
    }
    float low = __double2float_rd(best);                      // (32 bits, rounded down: a bound need not be exact)
    if (NT > 64) {
#pragma unroll
        for (int o = 1; o < NT / 64; o <<= 1) low = fmaxf(low, __shfl_xor(low, o, 64));
        if (t % (NT / 64) == 0) group_max[t / (NT / 64)] = low;
        __syncthreads();
        low = group_max[t & 63];
    }
    const double bound = (double)sel_kth(sel_order(low), K);
    auto collect = [&](auto &&pred) {
#pragma unroll
        for (int u = 0; u < E; ++u)
            if (c[u] > -INFINITY && pred(c[u], u * NT + t)) {
                const int at = atomicAdd(&found, 1);
                if (at < CAP) { cs[at] = c[u]; ps[at] = u * NT + t; }
            }
    };
    collect([&](double d, int) { return d >= bound; });
    __syncthreads();
    int n = found;
    if (n > CAP) {
        const SelCut cut = sel_cut(K, CAP, total, [&](auto &&pred) {
            int k = 0;
#pragma unroll
            for (int u = 0; u < E; ++u) k += c[u] > -INFINITY && pred(sel_order64(c[u]), u * NT + t) ? 1 : 0;
            return sel_count<NT>(k, red);
        });
        __syncthreads();
        if (t == 0) found = 0;
        __syncthreads();
        collect([&](double d, int p) { return sel_within(cut, sel_order64(d), p); });
        __syncthreads();
        n = found;
    }
    for (int i = t; i < n; i += NT) {
        const double d = cs[i];
        const int p = ps[i];
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < n; ++k) rank += sel_before(cs[k], ps[k], d, p) ? 1 : 0;
        if (rank < K) {
            a.scores_out[b * K + rank] = (float)d;
            a.parents_out[b * K + rank] = p / V;
            a.tokens_out[b * K + rank] = p % V;
        }
    }
    __syncthreads();
    if (t == 0 && n < K) sel_fill(a, b, n);
}

// NT threads hold a tile of NT * E logits in registers, 8 consecutive ones of every NT * 8 each.  The K best:
//   1. a bound: the threads form 64 groups; the K-th largest of the groups' maxima has at least K logits at or above it;
//   2. what reaches the bound is collected: on unordered data the sum of 64 / (64 - i) over i < K on average, 4 for K 4, 18 for 16, 44 for 32, 304 for 64;
//   3. where more than SEL_CAP do (ties, runs), the K-th largest is found by bisection over value and place, and exactly K collected;
//   4. each collected one's rank is the number of those before it.
template <typename T, int NT, int E, bool MASKED> __global__ void __launch_bounds__(NT) vq_beam_rows_kernel(const SelArgs a)
{
    constexpr int NW = NT / 64, NU = E / 8;
    __shared__ float group_max[64], bound_s;
    __shared__ double wave_sum[NW];
    __shared__ int wave_cnt[NW], found;
    __shared__ int2 list[SEL_CAP];
    const int t = threadIdx.x, V = a.V, K = a.K;
    const unsigned row = blockIdx.x / (unsigned)a.tiles, tile = blockIdx.x - row * a.tiles, b = row / (unsigned)a.J, j = row - b * a.J;
    // a finished beam's logits are not used, nor are those of a beam without a score: the merge knows
    if (a.finished && a.finished[row]) return;
    if (a.scores && !(a.scores[row] > -INFINITY)) return;
    const T *lg = (const T *)a.logits + b * a.lb + j * a.lj;
    const uint8_t *mk = MASKED ? a.mask + b * a.mb + j * a.mj : nullptr;
    const int first = (int)tile * (NT * E);
    // all loads first: whole vectors, the ones past the row's end moved back into it and put right below
    VqVec<T, 8> raw[NU];
    unsigned long long live[NU];
    if (V >= 8) {
        if (MASKED)
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                const int at = first + (u * NT + t) * 8;
                const VqVec<uint8_t, 8> m = vq_ldv<uint8_t, 8>(mk + (at < V - 8 ? at : V - 8));
                __builtin_memcpy(&live[u], &m, 8);
            }
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int at = first + (u * NT + t) * 8;
            if (!MASKED || live[u]) raw[u] = vq_ldv<T, 8>(lg + (at < V - 8 ? at : V - 8));
        }
    }
    float x[E], most[NU];                                     // the logits, the largest of each 8
#pragma unroll
    for (int u = 0; u < NU; ++u)
#pragma unroll
        for (int i = 0; i < 8; ++i) x[u * 8 + i] = !MASKED || ((live[u] >> (8 * i)) & 0xff) ? (float)raw[u].v[i] : -INFINITY;
    if (first + NT * E > V) {
#pragma unroll
        for (int u = 0; u < NU; ++u) {
            const int at = first + (u * NT + t) * 8;
            if (at + 8 > V)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[u * 8 + i] = at + i < V && (!MASKED || mk[at + i]) ? (float)lg[at + i] : -INFINITY;
        }
    }
    float gm = -INFINITY;
#pragma unroll
    for (int u = 0; u < NU; ++u) {
        most[u] = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) most[u] = fmaxf(most[u], x[u * 8 + i]);                 // (a NaN is passed over)
        gm = fmaxf(gm, most[u]);
    }
    // 1. 64 groups of NT / 64 threads: each wave finds the largest of all, one of them the K-th
#pragma unroll
    for (int o = 1; o < NT / 64; o <<= 1) gm = fmaxf(gm, __shfl_xor(gm, o, 64));
    if (t % (NT / 64) == 0) group_max[t / (NT / 64)] = gm;
    if (t == 0) found = 0;
    __syncthreads();
    gm = group_max[t & 63];
    const float mx = vq_wave_max(gm);
    if (t >> 6 == NW - 1) {
        const float k = sel_kth(sel_order(gm), K);
        if ((t & 63) == 0) bound_s = k;
    }
    // the log-sum: 8 terms in 32 bits, the rest in 64; a logit of +inf or NaN makes it NaN
    if (a.normalize) {
        double s = 0.0;
        if (mx > -INFINITY) {
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                float q = 0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) q += sel_exp(x[u * 8 + i] - mx);
                s += q;
            }
        } else {                                              // no number at all: the sum is 0, or NaN where one is NaN
#pragma unroll
            for (int i = 0; i < E; ++i) s += x[i] != x[i] ? (double)NAN : 0.0;
        }
        s = vq_wave_sum(s);
        if ((t & 63) == 0) wave_sum[t >> 6] = s;
    }
    __syncthreads();
    // 2.
    const float bound = bound_s;
#pragma unroll
    for (int u = 0; u < NU; ++u)
        if (most[u] >= bound && most[u] > -INFINITY) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (x[u * 8 + i] >= bound && x[u * 8 + i] > -INFINITY) {
                    const int at = atomicAdd(&found, 1);
                    if (at < SEL_CAP) list[at] = make_int2(__float_as_int(x[u * 8 + i]), first + (u * NT + t) * 8 + i);
                }
        }
    __syncthreads();
    int n = found;
    if (n > SEL_CAP) {
        // 3. the K-th largest value, then the last place among those equal to it.  The logits are read again (from cache): kept in registers
        // for this rare way they would cost every tile a third of the waves that fit a CU.
        auto each = [&](auto &&f) {
#pragma unroll 1
            for (int u = 0; u < NU; ++u) {
                const int at = first + (u * NT + t) * 8;
                if (at >= V) break;
                VqVec<T, 8> r;
                if (at + 8 <= V) r = vq_ldv<T, 8>(lg + at);
                else
                    for (int i = 0; i < 8; ++i) r.v[i] = at + i < V ? lg[at + i] : (T)0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = at + i < V && (!MASKED || mk[at + i]) ? (float)r.v[i] : -INFINITY;
                    if (v > -INFINITY) f(v, sel_order(v), (unsigned)(at + i));
                }
            }
        };
        auto count = [&](auto &&pred) {
            int c = 0;
            each([&](float, unsigned o, unsigned p) { c += pred(o, p) ? 1 : 0; });
            c = vq_wave_sum(c);
            __syncthreads();
            if ((t & 63) == 0) wave_cnt[t >> 6] = c;
            __syncthreads();
            c = 0;
#pragma unroll
            for (int w = 0; w < NW; ++w) c += wave_cnt[w];
            return c;
        };
        unsigned kth = 0;
        for (unsigned bit = 0x80000000u; bit; bit >>= 1) {
            const unsigned want = kth | bit;
            if (count([&](unsigned o, unsigned) { return o >= want; }) >= K) kth = want;
        }
        const int above = count([&](unsigned o, unsigned) { return o > kth; });
        unsigned lo = (unsigned)first, hi = (unsigned)(first + NT * E < V ? first + NT * E : V) - 1;
        while (lo < hi) {                                     // the least place with `above` + (equal ones up to it) >= K
            const unsigned mid = lo + (hi - lo) / 2;
            if (above + count([&](unsigned o, unsigned p) { return o == kth && p <= mid; }) >= K) hi = mid; else lo = mid + 1;
        }
        __syncthreads();
        if (t == 0) found = 0;
        __syncthreads();
        each([&](float v, unsigned o, unsigned p) {
            if (o > kth || (o == kth && p <= lo)) list[atomicAdd(&found, 1)] = make_int2(__float_as_int(v), (int)p);
        });
        __syncthreads();
        n = found;
    }
    // 4.
    int2 *out = a.part + blockIdx.x * (int64_t)K;
    for (int i = t; i < n; i += NT) {
        const int2 me = list[i];
        const float f = __int_as_float(me.x);
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < n; ++k) {
            const int2 o = list[k];
            const float g = __int_as_float(o.x);
            rank += g > f || (g == f && o.y < me.y) ? 1 : 0;
        }
        if (rank < K) out[rank] = me;
    }
    for (int i = n + t; i < K; i += NT) out[i] = make_int2(__float_as_int(-INFINITY), 0);
    if (t == 0) {
        double s = 0.0;
        if (a.normalize)
            for (int w = 0; w < NW; ++w) s += wave_sum[w];
        a.part_max[blockIdx.x] = mx;
        a.part_sum[blockIdx.x] = s;
    }
}

// The lists hold a tile's K largest logits, yet under a score of -1e30, or around a logit of 1e-20, different logits have one and the same c,
// and the places decide.  Where the cut between the survivors and the rest goes through such a c (one step of a logit further down it is
// still the same), the survivors at the cut are the first places that have it, found by going through the entry's logits again.  `at`: the
// survivors above the cut.  The test for it costs a merge 0.7 us.
__device__ void sel_places(const SelArgs &a, int64_t b, double cut, int at, const double *base, const double *log_sum, const uint8_t *fin, int *wave_cnt)
{
    const int t = threadIdx.x, V = a.V;
    for (int j = 0; j < a.J && at < a.K; ++j) {
        if (!(base[j] > -INFINITY)) continue;
        for (int v0 = fin[j] ? a.end_token / 256 * 256 : 0; v0 < V && at < a.K; v0 += 256) {
            const int v = v0 + t;
            bool hit = false;
            if (fin[j]) hit = v == a.end_token && sel_sum(base[j], 0.0) == cut;
            else if (v < V && (!a.mask || a.mask[b * a.mb + j * a.mj + v])) {
                const int64_t i = b * a.lb + j * a.lj + v;
                const float l = a.dtype == VQHIP_F32 ? ((const float *)a.logits)[i] : a.dtype == VQHIP_BF16 ? (float)((const __bf16 *)a.logits)[i] : (float)((const _Float16 *)a.logits)[i];
                hit = sel_sum(base[j], (double)l - log_sum[j]) == cut;
            }
            const unsigned long long hits = __ballot(hit);
            __syncthreads();
            if ((t & 63) == 0) wave_cnt[t >> 6] = __popcll(hits);
            __syncthreads();
            int rank = at + __popcll(hits & ((1ull << (t & 63)) - 1));
            for (int w = 0; w < 4; ++w) {
                if (w < t >> 6) rank += wave_cnt[w];
                at += wave_cnt[w];
            }
            if (hit && rank < a.K) {
                a.scores_out[b * a.K + rank] = (float)cut;
                a.parents_out[b * a.K + rank] = j;
                a.tokens_out[b * a.K + rank] = v;
            }
            if (fin[j]) break;
        }
    }
}

// ---- merge: one workgroup per batch entry -------------------------------------------------------------------------------------------
// The rows' log-sums from their tiles (16 lanes a row), then the K best of J * tiles * K (and the finished beams') by the same bound and
// ranks in 64 bits; sel_cut where more than SEL_CAP reach the bound.  Bound by latency: the first SEL_HELD list entries of a thread are on
// their way while the log-sums are formed, and stay in registers.
#define SEL_HELD 4
__global__ void __launch_bounds__(256) vq_beam_merge_kernel(const SelArgs a)
{
    __shared__ double base[VQHIP_BEAM_MAX], log_sum[VQHIP_BEAM_MAX], cs[SEL_CAP];       // base: a row's s, -inf: no continuation
    __shared__ float ls[SEL_CAP];
    __shared__ unsigned group_max[64];
    __shared__ int ps[SEL_CAP], found, red[4];
    __shared__ double cut_s;
    __shared__ uint8_t fin[VQHIP_BEAM_MAX];
    const int t = threadIdx.x, J = a.J, S = a.tiles, K = a.K;
    const int64_t b = blockIdx.x;
    const int per = S * K, total = J * per;
    const int2 *lists = a.part + b * total;                   // (rows that no workgroup listed hold anything: base tells)
    int2 held[SEL_HELD];
#pragma unroll
    for (int h = 0; h < SEL_HELD; ++h) held[h] = h * 256 + t < total ? lists[h * 256 + t] : make_int2(0, 0);
    for (int j = t >> 4; j < J; j += 16) {
        const int64_t row = b * J + j;
        const double s = a.scores ? (double)a.scores[row] : 0.0;
        const bool f = a.finished && a.finished[row], live = !f && s > -INFINITY;
        double lse = 0.0;
        if (a.normalize) {
            float top = -INFINITY;
            for (int q = t & 15; q < S; q += 16) top = fmaxf(top, a.part_max[row * S + q]);
            for (int o = 8; o; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
            double sum = 0.0;
            for (int q = t & 15; q < S; q += 16) {
                const double p = a.part_sum[row * S + q];
                sum += p == 0.0 ? 0.0 : p * exp((double)a.part_max[row * S + q] - (double)top);
            }
            for (int o = 8; o; o >>= 1) sum += __shfl_xor(sum, o, 64);
            lse = (double)top + log(sum);                      // (no logit admitted: not finite)
        }
        if ((t & 15) == 0) {
            fin[j] = f;
            base[j] = f ? s : live && lse > -INFINITY && lse < INFINITY ? s : -INFINITY;
            log_sum[j] = lse;
            if (a.lse_out) a.lse_out[row] = sel_lse(lse, s, f);
        }
    }
    if (t == 0) found = 0;
    if (t < 64) group_max[t] = sel_order(-INFINITY);
    __syncthreads();
    // candidate i: list entry row.r of row row.q, a finished beam's first one is its only continuation; entry list.r of list list.q
    SelWalk row(t, per, 256), list(t, K, 256);
    auto value = [&](const SelWalk &row, int2 q, int &place) -> double {
        const int j = row.q;
        const double s = base[j];
        if (fin[j]) {
            place = j * a.V + a.end_token;
            return row.r == 0 ? sel_sum(s, 0.0) : -INFINITY;
        }
        const double l = (double)__int_as_float(q.x);
        place = j * a.V + q.y;
        return s > -INFINITY && l > -INFINITY ? sel_sum(s, l - log_sum[j]) : -INFINITY;
    };
    // 64 groups: lists and, where there are fewer than 64 of them, ranks modulo R.  A list falls, so its first R entries are the largest of
    // their groups.  (32 bits, rounded down: a bound need not be exact)
    const int R = J * S < 64 ? 64 / (J * S) : 1;
    auto group = [&](double c) {
        if (list.r < R && c > -INFINITY) atomicMax(&group_max[(list.q * R + list.r) & 63], sel_order(__double2float_rd(c)));
    };
    double c_held[SEL_HELD];
    int p_held[SEL_HELD], place;
#pragma unroll
    for (int h = 0; h < SEL_HELD; ++h, row.next(), list.next()) {
        c_held[h] = h * 256 + t < total ? value(row, held[h], p_held[h]) : -INFINITY;
        group(c_held[h]);
    }
    const SelWalk behind = row;
    for (int i = SEL_HELD * 256 + t; i < total; i += 256, row.next(), list.next())
        if (list.r < R) group(value(row, lists[i], place));
    __syncthreads();
    const double bound = (double)sel_kth(group_max[t & 63], K);
    auto each = [&](auto &&f) {                               // f(score, place, logit) of this thread's candidates above -inf
#pragma unroll
        for (int h = 0; h < SEL_HELD; ++h)
            if (c_held[h] > -INFINITY) f(c_held[h], p_held[h], __int_as_float(held[h].x));
        SelWalk row = behind;
        for (int i = SEL_HELD * 256 + t; i < total; i += 256, row.next()) {
            const int2 q = lists[i];
            const double c = value(row, q, place);
            if (c > -INFINITY) f(c, place, __int_as_float(q.x));
        }
    };
    auto collect = [&](auto &&pred) {
        each([&](double c, int p, float l) {
            if (pred(c, p)) {
                const int k = atomicAdd(&found, 1);
                if (k < SEL_CAP) { cs[k] = c; ps[k] = p; ls[k] = l; }
            }
        });
    };
    collect([&](double c, int) { return c >= bound; });
    __syncthreads();
    // whether a logit below l, which no list may hold, has l's c (the cut's) too
    auto more = [&](int j, float l) { return !fin[j] && sel_sum(base[j], (double)nextafterf(l, -INFINITY) - log_sum[j]) == cut_s; };
    int n = found;
    const bool many = n > SEL_CAP;
    if (many) {
        const SelCut cut = sel_cut(K, SEL_CAP, J * a.V, [&](auto &&pred) {
            int k = 0;
            each([&](double c, int p, float) { k += pred(sel_order64(c), p) ? 1 : 0; });
            return sel_count<256>(k, red);
        });
        __syncthreads();
        if (t == 0) found = 0;
        __syncthreads();
        collect([&](double c, int p) { return sel_within(cut, sel_order64(c), p); });
        __syncthreads();
        n = found;
    }
    for (int i = t; i < n; i += 256) {
        const double c = cs[i];
        const int p = ps[i];
        int rank = 0;
#pragma unroll 8
        for (int k = 0; k < n; ++k) rank += sel_before(cs[k], ps[k], c, p) ? 1 : 0;
        if (rank < K) {
            a.scores_out[b * K + rank] = (float)c;
            a.parents_out[b * K + rank] = p / a.V;
            a.tokens_out[b * K + rank] = p % a.V;
        }
        if (rank == K - 1) cut_s = c;
    }
    __syncthreads();
    if (n < K) {
        if (t == 0) sel_fill(a, b, n);
        return;
    }
    bool open = false;
    if (many) each([&](double c, int p, float l) { open |= c == cut_s && more(p / a.V, l); });
    else
        for (int i = t; i < n; i += 256) open |= cs[i] == cut_s && more(ps[i] / a.V, ls[i]);
    if (__syncthreads_or(open)) {
        int above = 0;
        for (int k = 0; k < n; ++k) above += cs[k] > cut_s ? 1 : 0;
        sel_places(a, b, cut_s, above, base, log_sum, fin, red);
    }
}

// Workgroups of a launch, which takes fewer than 2^32 threads; larger batches go in several, one after the other with the same workspace.  An
// entry has at most 2^19 + 64 tiles.
#define SEL_LAUNCH (1 << 23)

// small: 1 a lane, 2 a wave or a workgroup an entry.  Tiles of the rows: one wave for rows of up to 512 logits; 8192 logits a workgroup where that gives each CU two, else 2048.  Rows and
// merge with 8192 and 2048: 128 rows of 131071 bf16 14.6 + 6.5 and 21.0 + 15.9 us, 160 rows of 8193 masked 8.2 + 5.3 and 5.4 + 6.0.
struct SelPlan { int small, threads, per_thread, tiles; };           // (tiles: of a row)
static SelPlan sel_plan(int64_t B, int64_t J, int64_t V)
{
    if (J * V <= 64) return SelPlan{1, 0, 0, 0};
    if (J * V <= SEL_ENTRY) return SelPlan{2, 0, 0, 0};
    if (V <= 512) return SelPlan{0, 64, 8, 1};
    const bool big = B * J * ((V + 8191) / 8192) >= 512;
    return SelPlan{0, 256, big ? 32 : 8, (int)(big ? (V + 8191) / 8192 : (V + 2047) / 2048)};
}

// batch entries of a launch with `per` workgroups an entry
static int64_t sel_most(int64_t B, int64_t per) { return B < SEL_LAUNCH / per ? B : SEL_LAUNCH / per; }

template <typename T> static void sel_rows(const SelArgs &a, const SelPlan &p, hipStream_t st)
{
    const dim3 grid((unsigned)(a.B * a.J * p.tiles));
    if (p.threads == 64) {
        if (a.mask) vq_beam_rows_kernel<T, 64, 8, true><<<grid, 64, 0, st>>>(a); else vq_beam_rows_kernel<T, 64, 8, false><<<grid, 64, 0, st>>>(a);
    } else if (p.per_thread == 8) {
        if (a.mask) vq_beam_rows_kernel<T, 256, 8, true><<<grid, 256, 0, st>>>(a); else vq_beam_rows_kernel<T, 256, 8, false><<<grid, 256, 0, st>>>(a);
    } else {
        if (a.mask) vq_beam_rows_kernel<T, 256, 32, true><<<grid, 256, 0, st>>>(a); else vq_beam_rows_kernel<T, 256, 32, false><<<grid, 256, 0, st>>>(a);
    }
}

template <typename T> static void sel_entries(const SelArgs &a, hipStream_t st)
{
    const dim3 grid((unsigned)a.B);
    const int n = a.J * a.V;
    if (n <= 256) vq_beam_entry_kernel<T, 64, 4><<<grid, 64, 0, st>>>(a);
    else if (n <= 512) vq_beam_entry_kernel<T, 64, 8><<<grid, 64, 0, st>>>(a);
    else if (n <= 1024) vq_beam_entry_kernel<T, 64, 16><<<grid, 64, 0, st>>>(a);
    else if (n <= 2048) vq_beam_entry_kernel<T, 128, 16><<<grid, 128, 0, st>>>(a);
    else vq_beam_entry_kernel<T, 256, 16><<<grid, 256, 0, st>>>(a);
}

static int sel_check(const vqhip_beam_select_t *p, const char *what)
{
    if (!p) VQ_FAIL(VQHIP_EINVAL, "%s: null argument", what);
    if (!vq_elem_bytes(p->dtype)) VQ_FAIL(VQHIP_EINVAL, "%s: dtype %lld", what, (long long)p->dtype);
    if (p->B < 0 || p->J < 1 || p->V < 1 || p->K < 1) VQ_FAIL(VQHIP_EINVAL, "%s: B %lld, J %lld, V %lld, K %lld", what, (long long)p->B, (long long)p->J, (long long)p->V, (long long)p->K);
    if (p->J > VQHIP_BEAM_MAX || p->K > VQHIP_BEAM_MAX || p->V > (1 << 30) / p->J || p->K > p->J * p->V || p->B > 0x7fffffff)
        VQ_FAIL(VQHIP_EDIM, "%s: %lld entries, %lld kept of %lld x %lld continuations: fewer than 2^31 entries, at most %d beams, %d kept, 2^30 continuations an entry",
                what, (long long)p->B, (long long)p->K, (long long)p->J, (long long)p->V, VQHIP_BEAM_MAX, VQHIP_BEAM_MAX);
    if (p->finished && (p->end_token < 0 || p->end_token >= p->V)) VQ_FAIL(VQHIP_EINVAL, "%s: end token %lld outside [0, %lld)", what, (long long)p->end_token, (long long)p->V);
    if (p->B > 0 && (!p->logits || !p->parents || !p->tokens || !p->out_scores)) VQ_FAIL(VQHIP_EINVAL, "%s: null pointer", what);
    return 0;
}

extern "C" size_t vqhip_beam_select_workspace_bytes(int64_t B, int64_t J, int64_t V, int64_t K)
{
    if (B <= 0 || J <= 0 || V <= 0 || K <= 0 || B > 0x7fffffff || J > VQHIP_BEAM_MAX || V > (1 << 30) / J) return 0;
    const int64_t per = J * sel_plan(B, J, V).tiles;
    return per ? (size_t)(sel_most(B, per) * per) * (size_t)(8 * K + 12) : 0;
}

extern "C" int vqhip_beam_select(const vqhip_beam_select_t *p, void *stream)
{
    int rc = sel_check(p, "vqhip_beam_select");
    if (rc) return rc;
    if (p->B == 0) return 0;
    const size_t need = vqhip_beam_select_workspace_bytes(p->B, p->J, p->V, p->K);
    if (p->workspace_bytes < need || (need && !p->workspace)) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_select: workspace of %zu bytes, needs %zu", p->workspace_bytes, need);
    if ((uintptr_t)p->workspace & 15) VQ_FAIL(VQHIP_EALIGN, "vqhip_beam_select: workspace not 16-byte aligned");
    SelArgs a;
    a.lb = p->stride_b; a.lj = p->stride_j; a.dtype = (int)p->dtype; a.mb = p->mask_stride_b; a.mj = p->mask_stride_j;
    a.J = (int)p->J; a.V = (int)p->V; a.K = (int)p->K; a.end_token = (int)p->end_token; a.normalize = p->normalize != 0;
    const SelPlan plan = sel_plan(p->B, p->J, p->V);
    hipStream_t st = (hipStream_t)stream;
    const int64_t most = sel_most(p->B, plan.small ? 1 : p->J * plan.tiles);
    for (int64_t b = 0; b < p->B; b += most) {
        a.B = p->B - b < most ? p->B - b : most;
        a.logits = (const char *)p->logits + b * p->stride_b * vq_elem_bytes(p->dtype);
        a.scores = p->scores ? p->scores + b * p->J : nullptr;
        a.mask = p->mask ? p->mask + b * p->mask_stride_b : nullptr;
        a.finished = p->finished ? p->finished + b * p->J : nullptr;
        a.scores_out = p->out_scores + b * p->K; a.parents_out = p->parents + b * p->K; a.tokens_out = p->tokens + b * p->K;
        a.lse_out = p->lse ? p->lse + b * p->J : nullptr;
        if (plan.small == 2) {
            if (p->dtype == VQHIP_F32) sel_entries<float>(a, st);
            else if (p->dtype == VQHIP_BF16) sel_entries<__bf16>(a, st);
            else sel_entries<_Float16>(a, st);
        } else if (plan.small) {
            int W = 1;
            while (W < a.J * a.V) W <<= 1;
            const dim3 grid((unsigned)((a.B * W + 255) / 256));
            if (p->dtype == VQHIP_F32) vq_beam_small_kernel<float><<<grid, 256, 0, st>>>(a, W);
            else if (p->dtype == VQHIP_BF16) vq_beam_small_kernel<__bf16><<<grid, 256, 0, st>>>(a, W);
            else vq_beam_small_kernel<_Float16><<<grid, 256, 0, st>>>(a, W);
        } else {
            const int64_t lists = most * a.J * plan.tiles;
            a.tiles = plan.tiles;
            a.part = (int2 *)p->workspace; a.part_sum = (double *)(a.part + lists * a.K); a.part_max = (float *)(a.part_sum + lists);
            if (p->dtype == VQHIP_F32) sel_rows<float>(a, plan, st);
            else if (p->dtype == VQHIP_BF16) sel_rows<__bf16>(a, plan, st);
            else sel_rows<_Float16>(a, plan, st);
            vq_beam_merge_kernel<<<dim3((unsigned)a.B), 256, 0, st>>>(a);
        }
    }
    return vq_launch_status("vqhip_beam_select");
}

// d_scores[b, j] = sum of g over the kept continuations of beam j; d_logits[b, j, v] = sum of g over those with token v, minus (normalize)
// d_scores[b, j] * softmax(l)[b, j, v].  A continuation of score -inf is none: its g counts as 0.  Finished beams pass nothing on to logits.
// One pass: a workgroup reads SEL_BWD logits of a row and writes their gradients; a row without a survivor is written and not read.
struct SelBwdArgs {
    const void *logits; int64_t lb, lj;
    const uint8_t *mask; int64_t mb, mj;
    const uint8_t *finished; const double *lse;
    const float *scores_out; const int64_t *parents, *tokens; const float *grad;
    void *d_logits; float *d_scores;
    int64_t B; int J, V, K, normalize, tiles;
};
#define SEL_BWD 4096

template <typename T, bool MASKED> __global__ void __launch_bounds__(256) vq_beam_select_bwd_kernel(const SelBwdArgs a)
{
    __shared__ float g[VQHIP_BEAM_MAX];
    __shared__ int tok[VQHIP_BEAM_MAX], n_s;
    __shared__ float onto_s;
    const unsigned tile = blockIdx.x % a.tiles;
    const int64_t row = blockIdx.x / a.tiles, b = row / a.J;
    const int j = (int)(row - b * a.J), t = threadIdx.x, V = a.V;
    const int first = (int)tile * SEL_BWD, last = V - first < SEL_BWD ? V : first + SEL_BWD;
    if (t < 64) {                                             // lane k looks at survivor k; the list keeps this tile's
        const int64_t k = b * a.K + t;
        const bool mine = t < a.K && a.parents[k] == j && a.scores_out[k] > -INFINITY;
        const float gk = mine ? a.grad[k] : 0.f;
        const int tk = mine ? (int)a.tokens[k] : -1;
        const bool here = mine && tk >= first && tk < last;
        const unsigned long long hs = __ballot(here);
        if (here) {
            const int at = __popcll(hs & ((1ull << t) - 1));
            g[at] = gk;
            tok[at] = tk;
        }
        const float onto = (float)vq_wave_sum((double)gk);     // (64 bits: the gradients of a beam's survivors may cancel)
        const bool any = __ballot(mine) != 0;
        if (t == 0) {
            if (a.d_scores && tile == 0) a.d_scores[row] = onto;
            onto_s = onto;
            n_s = (a.finished && a.finished[row]) || !any ? -1 : __popcll(hs);
        }
    }
    __syncthreads();
    if (!a.d_logits) return;
    const int n = n_s;
    const float onto = onto_s;
    const T *lg = (const T *)a.logits + b * a.lb + j * a.lj;
    const uint8_t *mk = MASKED ? a.mask + b * a.mb + j * a.mj : nullptr;
    T *out = (T *)a.d_logits + row * V;
    const double lse = a.normalize && n >= 0 ? a.lse[row] : 0.0;
    const float lh = (float)lse, ll = (float)(lse - (double)lh);             // l - lse in two steps of 32 bits
#pragma unroll
    for (int u = 0; u < SEL_BWD / 2048; ++u) {
        const int at = first + (u * 256 + t) * 8;
        if (at >= last) break;
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = 0.f;
        const int have = last - at < 8 ? last - at : 8;
        if (n >= 0) {
            if (a.normalize) {
                VqVec<T, 8> r;
                if (have == 8) r = vq_ldv<T, 8>(lg + at);
                else
                    for (int i = 0; i < 8; ++i) r.v[i] = i < have ? lg[at + i] : (T)0.f;
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = -onto * sel_exp(((float)r.v[i] - lh) - ll);
            }
            for (int k = 0; k < n; ++k) {
                const int w = tok[k] - at;
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] += w == i ? g[k] : 0.f;
            }
            if (MASKED)
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = i < have && mk[at + i] ? d[i] : 0.f;
        }
        if (have == 8) {
            VqVec<T, 8> o;
#pragma unroll
            for (int i = 0; i < 8; ++i) o.v[i] = (T)d[i];
            vq_stv<T, 8>(out + at, o);
        } else
            for (int i = 0; i < have; ++i) out[at + i] = (T)d[i];
    }
}

// Entries of up to SEL_ENTRY continuations: a workgroup (a wave for up to 1024) each.  The survivors' gradients are put in their places in LDS,
// no two of them in one.  8192 entries of 16 x 16 fp32: 9.3 us, with a workgroup a row 117.
template <typename T, int NT> __global__ void __launch_bounds__(NT) vq_beam_select_bwd_entry_kernel(const SelBwdArgs a)
{
    extern __shared__ __align__(16) float put[];              // [J * V]
    __shared__ float g[VQHIP_BEAM_MAX], onto[VQHIP_BEAM_MAX], lh[VQHIP_BEAM_MAX], ll[VQHIP_BEAM_MAX];
    __shared__ int from[VQHIP_BEAM_MAX];
    __shared__ uint8_t dead[VQHIP_BEAM_MAX];
    const int t = threadIdx.x, J = a.J, V = a.V, K = a.K, total = J * V;
    const int64_t b = blockIdx.x;
    int place = -1;
    if (t < K) {
        const int64_t j = a.parents[b * K + t], v = a.tokens[b * K + t];
        const bool some = a.scores_out[b * K + t] > -INFINITY && j >= 0 && j < J && v >= 0 && v < V;
        g[t] = some ? a.grad[b * K + t] : 0.f;
        from[t] = some ? (int)j : -1;
        if (some) place = (int)(j * V + v);
    }
    if (a.d_logits)
        for (int i = t; i < total; i += NT) put[i] = 0.f;
    __syncthreads();
    if (place >= 0 && a.d_logits) put[place] = g[t];
    if (t < J) {
        double sum = 0.0;                                     // (64 bits: the gradients of a beam's survivors may cancel)
        bool any = false;
        for (int k = 0; k < K; ++k)
            if (from[k] == t) { sum += (double)g[k]; any = true; }
        any = any && !(a.finished && a.finished[b * J + t]);
        const double lse = a.normalize && any && a.lse ? a.lse[b * J + t] : 0.0;
        if (a.d_scores) a.d_scores[b * J + t] = (float)sum;
        onto[t] = (float)sum;
        dead[t] = !any;
        lh[t] = (float)lse;
        ll[t] = (float)(lse - (double)lh[t]);
    }
    __syncthreads();
    if (!a.d_logits) return;
    const T *lg = (const T *)a.logits + b * a.lb;
    const uint8_t *mk = a.mask ? a.mask + b * a.mb : nullptr;
    T *out = (T *)a.d_logits + b * total;
    SelWalk at(t, V, NT);
    for (int i = t; i < total; i += 4 * NT) {
        T l[4];
        uint8_t live[4];
        int row[4];
#pragma unroll
        for (int u = 0; u < 4; ++u, at.next()) {              // loads without conditions; past the end, the first one again
            const bool in = i + u * NT < total;
            const int j = in ? at.q : 0, v = in ? at.r : 0;
            row[u] = j;
            l[u] = lg[j * a.lj + v];
            live[u] = mk ? mk[j * a.mj + v] : 1;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int p = i + u * NT, j = row[u];
            if (p >= total) break;
            float d = put[p];
            if (a.normalize) d -= onto[j] * sel_exp(((float)l[u] - lh[j]) - ll[j]);
            out[p] = (T)(live[u] && !dead[j] ? d : 0.f);
        }
    }
}

template <typename T> static void sel_bwd(const SelBwdArgs &a, hipStream_t st)
{
    const int total = a.J * a.V;
    if (total <= SEL_ENTRY) {
        const size_t sm = a.d_logits ? (size_t)total * 4 : 0;
        if (total <= 1024) vq_beam_select_bwd_entry_kernel<T, 64><<<dim3((unsigned)a.B), 64, sm, st>>>(a);
        else vq_beam_select_bwd_entry_kernel<T, 256><<<dim3((unsigned)a.B), 256, sm, st>>>(a);
        return;
    }
    const dim3 grid((unsigned)(a.B * a.J * a.tiles));
    if (a.mask) vq_beam_select_bwd_kernel<T, true><<<grid, 256, 0, st>>>(a);
    else vq_beam_select_bwd_kernel<T, false><<<grid, 256, 0, st>>>(a);
}

extern "C" int vqhip_beam_select_bwd(const vqhip_beam_select_t *p, const float *grad, void *d_logits, float *d_scores, void *stream)
{
    int rc = sel_check(p, "vqhip_beam_select_bwd");
    if (rc) return rc;
    if (p->B == 0 || (!d_logits && !d_scores)) return 0;
    if (!grad || (p->normalize && d_logits && !p->lse)) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_select_bwd: null pointer");
    const int eb = vq_elem_bytes(p->dtype);
    SelBwdArgs a;
    a.lb = p->stride_b; a.lj = p->stride_j; a.mb = p->mask_stride_b; a.mj = p->mask_stride_j;
    a.J = (int)p->J; a.V = (int)p->V; a.K = (int)p->K; a.normalize = p->normalize != 0;
    a.tiles = d_logits ? (a.V + SEL_BWD - 1) / SEL_BWD : 1;
    hipStream_t st = (hipStream_t)stream;
    const int64_t most = sel_most(p->B, p->J * p->V <= SEL_ENTRY ? 1 : p->J * a.tiles);
    for (int64_t b = 0; b < p->B; b += most) {
        a.B = p->B - b < most ? p->B - b : most;
        a.logits = (const char *)p->logits + b * p->stride_b * eb;
        a.mask = p->mask ? p->mask + b * p->mask_stride_b : nullptr;
        a.finished = p->finished ? p->finished + b * p->J : nullptr;
        a.lse = p->lse ? p->lse + b * p->J : nullptr;
        a.scores_out = p->out_scores + b * p->K; a.parents = p->parents + b * p->K; a.tokens = p->tokens + b * p->K; a.grad = grad + b * p->K;
        a.d_logits = d_logits ? (char *)d_logits + b * p->J * p->V * eb : nullptr;
        a.d_scores = d_scores ? d_scores + b * p->J : nullptr;
        if (p->dtype == VQHIP_F32) sel_bwd<float>(a, st);
        else if (p->dtype == VQHIP_BF16) sel_bwd<__bf16>(a, st);
        else sel_bwd<_Float16>(a, st);
    }
    return vq_launch_status("vqhip_beam_select_bwd");
}

// ---- reordering ------------------------------------------------------------------------------------------------------------------
// out[b, i] = state[b, parents[b, i]] for every state of the call in one launch; a parent outside [0, J) gives zeros.  A state's row is
// n1 pieces of `run` contiguous bytes, s1 bytes apart (a cache whose rows are cut to the positions in use); out is contiguous.
//
// A copy, bound by HBM.  A piece is cut into units of 16 bytes (the largest power of two <= run where that is less); the last unit ends
// with the piece and may overlap the one before it, so that no length needs a tail.  A workgroup moves REO_UNITS units that follow each
// other over rows and pieces, whatever the rows' size; one 64-bit division finds its first row, 32-bit ones the rest.
#define REO_PER_THREAD 4
#define REO_UNITS (256 * REO_PER_THREAD)
struct ReorderState {
    const char *src; char *dst;
    int64_t sb, sj, s1, run;
    unsigned n1, per_piece, per_row, unit;              // pieces of a row; units of a piece, of a row; bytes of a unit
    unsigned first;                                     // first workgroup in the launch
};
struct ReorderArgs {
    ReorderState s[VQHIP_BEAM_STATES];
    const int64_t *parents;
    int64_t B; int J, K, n;
};

template <typename Args> __device__ __forceinline__ int reo_state(const Args &a, unsigned block)
{
    int lo = 0, hi = a.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.s[mid].first <= block) lo = mid; else hi = mid - 1;
    }
    return lo;
}

template <int BYTES> __device__ __forceinline__ void reo_move(const ReorderArgs &a, const ReorderState &s)
{
    using U = VqVec<uint8_t, BYTES>;
    const int64_t rows = a.B * a.K;
    const int64_t id0 = (int64_t)(blockIdx.x - s.first) * REO_UNITS, row0 = id0 / s.per_row;
    const unsigned off0 = (unsigned)(id0 - row0 * s.per_row);
    const unsigned here = row0 + (off0 + REO_UNITS - 1) / s.per_row < rows ? REO_UNITS : (unsigned)(rows * s.per_row - id0);
    U v[REO_PER_THREAD];
    int64_t dst[REO_PER_THREAD];
    bool some[REO_PER_THREAD];
#pragma unroll
    for (int u = 0; u < REO_PER_THREAD; ++u) {                // loads without conditions, so that all are in flight: the workgroup's last unit again
        const unsigned want = u * 256 + threadIdx.x, off = off0 + (want < here ? want : here - 1), skip = off / s.per_row, in_row = off - skip * s.per_row;
        const int64_t row = row0 + skip;
        const unsigned piece = s.n1 == 1 ? 0 : in_row / s.per_piece;
        int64_t at = (int64_t)(in_row - piece * s.per_piece) * BYTES;
        at = at + BYTES <= s.run ? at : s.run - BYTES;
        const int64_t b = (int64_t)((unsigned)row / (unsigned)a.K), p = a.parents[row];
        some[u] = p >= 0 && p < a.J;
        dst[u] = (row * s.n1 + piece) * s.run + at;
        v[u] = *(const U *)(s.src + b * s.sb + (some[u] ? p : 0) * s.sj + piece * s.s1 + at);
    }
#pragma unroll
    for (int u = 0; u < REO_PER_THREAD; ++u)
        if (u * 256 + threadIdx.x < here) {
            if (!some[u])
#pragma unroll
                for (int i = 0; i < BYTES; ++i) v[u].v[i] = 0;
            *(U *)(s.dst + dst[u]) = v[u];
        }
}

__global__ void __launch_bounds__(256) vq_beam_reorder_kernel(const ReorderArgs a)
{
    const ReorderState &s = a.s[reo_state(a, blockIdx.x)];
    switch (s.unit) {
    case 16: reo_move<16>(a, s); break;
    case 8: reo_move<8>(a, s); break;
    case 4: reo_move<4>(a, s); break;
    case 2: reo_move<2>(a, s); break;
    default: reo_move<1>(a, s);
    }
}

// d_state[b, j] = sum of grad[b, i] over parents[b, i] == j, ascending i, in 32 bits and rounded once; both contiguous.  The same units,
// now of 4 or 8 elements: an overlapping unit writes the same sums again.
struct ReorderBwdState { const void *grad; void *out; int64_t row; unsigned per_row, unit, first; int dtype; };       // row, unit: elements
struct ReorderBwdArgs {
    ReorderBwdState s[VQHIP_BEAM_STATES];
    const int64_t *parents;
    int64_t B; int J, K, n;
};

template <typename T, int N> __device__ __forceinline__ void reo_sum(const ReorderBwdArgs &a, const ReorderBwdState &s)
{
    const int64_t rows = a.B * a.J;
    const int64_t id0 = (int64_t)(blockIdx.x - s.first) * REO_UNITS, row0 = id0 / s.per_row, b0 = row0 / a.J;
    const unsigned off0 = (unsigned)(id0 - row0 * s.per_row), j0 = (unsigned)(row0 - b0 * a.J);
#pragma unroll
    for (int u = 0; u < REO_PER_THREAD; ++u) {
        const unsigned off = off0 + u * 256 + threadIdx.x, skip = off / s.per_row, in_row = off - skip * s.per_row;
        const int64_t row = row0 + skip;
        if (row >= rows) break;
        int64_t at = (int64_t)in_row * N;
        at = at + N <= s.row ? at : s.row - N;
        const unsigned further = (j0 + skip) / (unsigned)a.J;
        const int64_t j = (int64_t)(j0 + skip - further * (unsigned)a.J), k0 = (b0 + further) * a.K;
        const T *g = (const T *)s.grad + k0 * s.row + at;
        float d[N];
#pragma unroll
        for (int i = 0; i < N; ++i) d[i] = 0.f;
        for (int k = 0; k < a.K; k += 4) {                    // four parents at a time, their gradients loaded together
            bool hit[4];
            VqVec<T, N> v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) hit[q] = k + q < a.K && a.parents[k0 + k + q] == j;
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (hit[q]) v[q] = vq_ldv<T, N>(g + (k + q) * s.row);
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (hit[q])
#pragma unroll
                    for (int i = 0; i < N; ++i) d[i] += (float)v[q].v[i];
        }
        VqVec<T, N> o;
#pragma unroll
        for (int i = 0; i < N; ++i) o.v[i] = (T)d[i];
        vq_stv<T, N>((T *)s.out + row * s.row + at, o);
    }
}

__global__ void __launch_bounds__(256) vq_beam_reorder_bwd_kernel(const ReorderBwdArgs a)
{
    const ReorderBwdState &s = a.s[reo_state(a, blockIdx.x)];
    if (s.dtype == VQHIP_F32) {
        if (s.unit == 4) reo_sum<float, 4>(a, s); else reo_sum<float, 1>(a, s);
    } else if (s.dtype == VQHIP_BF16) {
        if (s.unit == 8) reo_sum<__bf16, 8>(a, s); else reo_sum<__bf16, 1>(a, s);
    } else {
        if (s.unit == 8) reo_sum<_Float16, 8>(a, s); else reo_sum<_Float16, 1>(a, s);
    }
}

static int reorder_check(int64_t n, const void *states, const int64_t *parents, int64_t B, int64_t J, int64_t K, const char *what)
{
    if (n < 0 || n > VQHIP_BEAM_STATES || B < 0 || J < 1 || K < 1) VQ_FAIL(VQHIP_EINVAL, "%s: %lld states (at most %d), B %lld, J %lld, K %lld", what, (long long)n, VQHIP_BEAM_STATES, (long long)B, (long long)J, (long long)K);
    if (J > 0x7fffffff || K > 0x7fffffff || B > 0x7fffffff / K)          // (B * J: a state's units are counted, reorder_blocks)
        VQ_FAIL(VQHIP_EDIM, "%s: %lld x %lld rows from %lld x %lld", what, (long long)B, (long long)K, (long long)B, (long long)J);
    if (n > 0 && B > 0 && (!states || !parents)) VQ_FAIL(VQHIP_EINVAL, "%s: null pointer", what);
    return 0;
}

// workgroups of `rows` rows of per_row units; a launch takes fewer than 2^32 threads
static int reorder_blocks(int64_t rows, int64_t per_row, unsigned *first, unsigned *total, const char *what)
{
    if (per_row > 0x40000000 || rows > (((int64_t)1 << 62) / per_row)) VQ_FAIL(VQHIP_EDIM, "%s: rows of %lld units", what, (long long)per_row);
    const int64_t blocks = (rows * per_row + REO_UNITS - 1) / REO_UNITS;
    if (blocks > ((1 << 24) - 1) - (int64_t)*total) VQ_FAIL(VQHIP_EDIM, "%s: too many bytes", what);
    *first = *total;
    *total += (unsigned)blocks;
    return 0;
}

extern "C" int vqhip_beam_reorder(const vqhip_beam_state_t *states, int64_t n, const int64_t *parents, int64_t B, int64_t J, int64_t K, void *stream)
{
    int rc = reorder_check(n, states, parents, B, J, K, "vqhip_beam_reorder");
    if (rc) return rc;
    ReorderArgs a;
    unsigned total = 0;
    a.n = 0;
    for (int64_t i = 0; i < n && B > 0; ++i) {
        const vqhip_beam_state_t &s = states[i];
        if (s.pieces < 0 || s.piece_bytes < 0) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder: state %lld: %lld pieces of %lld bytes", (long long)i, (long long)s.pieces, (long long)s.piece_bytes);
        if (s.pieces == 0 || s.piece_bytes == 0) continue;
        if (!s.src || !s.dst) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder: state %lld: null pointer", (long long)i);
        int unit = 16;
        while (unit > s.piece_bytes) unit >>= 1;
        const int64_t per_piece = (s.piece_bytes + unit - 1) / unit;
        if (s.pieces > 0x40000000 || per_piece > 0x40000000) VQ_FAIL(VQHIP_EDIM, "vqhip_beam_reorder: state %lld: %lld pieces of %lld bytes", (long long)i, (long long)s.pieces, (long long)s.piece_bytes);
        ReorderState &d = a.s[a.n];
        d = ReorderState{(const char *)s.src, (char *)s.dst, s.stride_b, s.stride_j, s.piece_stride, s.piece_bytes, (unsigned)s.pieces, (unsigned)per_piece, (unsigned)(s.pieces * per_piece), (unsigned)unit, 0};
        rc = reorder_blocks(B * K, s.pieces * per_piece, &d.first, &total, "vqhip_beam_reorder");
        if (rc) return rc;
        ++a.n;
    }
    if (a.n == 0) return 0;
    a.parents = parents; a.B = B; a.J = (int)J; a.K = (int)K;
    vq_beam_reorder_kernel<<<dim3(total), 256, 0, (hipStream_t)stream>>>(a);
    return vq_launch_status("vqhip_beam_reorder");
}

extern "C" int vqhip_beam_reorder_bwd(const vqhip_beam_state_t *states, const int64_t *dtypes, int64_t n, const int64_t *parents, int64_t B, int64_t J, int64_t K, void *stream)
{
    int rc = reorder_check(n, states, parents, B, J, K, "vqhip_beam_reorder_bwd");
    if (rc) return rc;
    if (n > 0 && !dtypes) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder_bwd: null pointer");
    ReorderBwdArgs a;
    unsigned total = 0;
    a.n = 0;
    for (int64_t i = 0; i < n && B > 0; ++i) {
        const vqhip_beam_state_t &s = states[i];
        const int eb = vq_elem_bytes(dtypes[i]);
        if (!eb || s.pieces < 0 || s.piece_bytes < 0 || s.piece_bytes % eb) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder_bwd: state %lld: dtype %lld, %lld pieces of %lld bytes", (long long)i, (long long)dtypes[i], (long long)s.pieces, (long long)s.piece_bytes);
        if (s.pieces == 0 || s.piece_bytes == 0) continue;
        if (!s.src || !s.dst) VQ_FAIL(VQHIP_EINVAL, "vqhip_beam_reorder_bwd: state %lld: null pointer", (long long)i);
        if (s.pieces > 0x40000000 || s.piece_bytes > ((int64_t)1 << 40) / s.pieces) VQ_FAIL(VQHIP_EDIM, "vqhip_beam_reorder_bwd: state %lld: %lld pieces of %lld bytes", (long long)i, (long long)s.pieces, (long long)s.piece_bytes);
        const int64_t row = s.pieces * s.piece_bytes / eb;
        const int unit = row < 16 / eb ? 1 : 16 / eb;
        const int64_t per_row = (row + unit - 1) / unit;
        ReorderBwdState &d = a.s[a.n];
        d = ReorderBwdState{s.src, s.dst, row, (unsigned)per_row, (unsigned)unit, 0, (int)dtypes[i]};
        rc = reorder_blocks(B * J, per_row, &d.first, &total, "vqhip_beam_reorder_bwd");
        if (rc) return rc;
        ++a.n;
    }
    if (a.n == 0) return 0;
    a.parents = parents; a.B = B; a.J = (int)J; a.K = (int)K;
    vq_beam_reorder_bwd_kernel<<<dim3(total), 256, 0, (hipStream_t)stream>>>(a);
    return vq_launch_status("vqhip_beam_reorder_bwd");
}

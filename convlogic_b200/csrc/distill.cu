// The loss of a row of scores against a teacher's list of top logits, and its gradient.
//
// With a = s / T, q = softmax(a); the teacher's list has classes i_k with probabilities p_k and, if its rest is known, the probability r of all the others
// together (q_r is the student's):
//     loss = T^2 [ sum_k p_k (log p_k - log q_{i_k}) + r (log r - log q_r) ]
//     d loss / d s_j = T (q_j - sum of p_k with i_k = j)            for a listed class
//                    = T (q_r - r) exp(a_j - log sum_unlisted exp a)  for any other
// The sums over listed and unlisted classes are kept apart from the start: q_r = 1 - sum of the listed q would lose what is left of a confident row.
// Per row the forward keeps (m, coefficient), unlisted gradient = coefficient * exp((s_j - m) / T), and the gradient of each listed class, weights
// and the mean's divisor included: with these the backward needs the scores and the upstream gradient, and no sum again.
#include "clb_scores.cuh"

using namespace clb;
using namespace clb_host;

namespace {

constexpr int kChunk = 32768; // classes whose "listed" bits fit the block's table at a time

struct DistillArgs {
    long long stride, rows;
    int classes, k;
    float temperature, c, scale; // c = log2(e) / T; scale: T, over the rows for a mean
};

// the bits of the listed classes in [lo, lo + kChunk)
__device__ __forceinline__ void mark_listed(uint32_t *bits, const int64_t *idx, int k, int lo, int hi)
{
    for (int i = threadIdx.x; i < kChunk / 32; i += 256) bits[i] = 0;
    __syncthreads();
    for (int n = threadIdx.x; n < k; n += 256) {
        const long long j = idx[n];
        if (j >= lo && j < hi) atomicOr(&bits[(j - lo) >> 5], 1u << ((j - lo) & 31));
    }
    __syncthreads();
}

template <typename T>
__global__ void __launch_bounds__(256) distill_fwd_kernel(const T *__restrict__ x, const float *__restrict__ values, const int64_t *__restrict__ indices,
                                                          const float *__restrict__ rest, const float *__restrict__ weight, float *__restrict__ row_loss,
                                                          float *__restrict__ stats, float *__restrict__ listed, DistillArgs a)
{
    __shared__ uint32_t bits[kChunk / 32];
    __shared__ ExpSum part[8];
    __shared__ float sv[CLB_TOP_MAX], tv[CLB_TOP_MAX], pv[CLB_TOP_MAX];
    __shared__ int64_t iv[CLB_TOP_MAX];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *row = x + r * a.stride;
        const int64_t *idx = indices + r * a.k;
        const float w = weight ? weight[r] : 1.f;
        __syncthreads();
        for (int n = threadIdx.x; n < a.k; n += 256) {
            const long long j = idx[n];
            const bool there = j >= 0 && j < a.classes;
            iv[n] = there ? j : -1;
            sv[n] = there ? to_f(row[j]) : -INFINITY;
            tv[n] = there ? values[r * a.k + n] : -INFINITY;
        }
        ExpSum s{-INFINITY, 0.f};
        for (int lo = 0; lo < a.classes; lo += kChunk) {
            const int hi = min(a.classes, lo + kChunk);
            mark_listed(bits, idx, a.k, lo, hi);
            for (int i = lo + threadIdx.x; i < hi; i += 256) {
                const float v = to_f(row[i]);
                if (!((bits[(i - lo) >> 5] >> ((i - lo) & 31)) & 1)) s = merge(s, single(v), a.c);
            }
            __syncthreads();
        }
        s = warp_merge(s, a.c);
        if (lane == 0) part[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int n = 1; n < 8; ++n) s = merge(s, part[n], a.c);
            // the teacher: mass Z = (tm, tl) of its list and rest
            ExpSum t{-INFINITY, 0.f}, u = s;
            for (int n = 0; n < a.k; ++n) {
                t = merge(t, single(tv[n]), a.c);
                bool first = iv[n] >= 0;
                for (int o = 0; o < n; ++o) first = first && iv[o] != iv[n];
                if (first) u = merge(u, single(sv[n]), a.c);
            }
            const float tt = a.temperature;
            const float rs = rest ? rest[r] : -INFINITY;
            const float tz = t.m == -INFINITY ? -INFINITY : t.m / tt;
            const float tm = fmaxf(tz, rs);
            float loss = 0.f, coef = 0.f, log_ul = 0.f;
            const bool there = w != 0.f && !(tm == -INFINITY && t.l == 0.f && !(rs != rs)) && !(u.m == -INFINITY && u.l == 0.f);
            if (there) {
                const float tl = (t.m == -INFINITY ? t.l : t.l * expf(tz - tm)) + expf(rs - tm);
                log_ul = logf(u.l);
                const float log_tl = logf(tl);
                for (int n = 0; n < a.k; ++n) {
                    const float lp = (tv[n] / tt - tm) - log_tl, lq = (sv[n] - u.m) / tt - log_ul;
                    pv[n] = tv[n] == -INFINITY ? 0.f : expf(lp);
                    if (pv[n] > 0.f || pv[n] != pv[n]) loss += pv[n] * (lp - lq);
                }
                const float lr = (rs - tm) - log_tl, rp = expf(lr);
                const float lqr = (s.m == -INFINITY ? -INFINITY : (s.m - u.m) / tt + logf(s.l)) - log_ul;
                if (rp > 0.f || rp != rp) loss += rp * (lr - lqr);
                if (s.m != -INFINITY || s.l != 0.f) coef = w * a.scale * (expf(lqr) - rp) / s.l;
            }
            row_loss[r] = there ? loss * w * a.scale * tt : 0.f;
            stats[2 * r] = finite_or_zero(s.m), stats[2 * r + 1] = coef;
            for (int n = 0; n < a.k; ++n) {
                float g = 0.f;
                if (there && iv[n] >= 0) {
                    float p = 0.f;
                    for (int o = 0; o < a.k; ++o)
                        if (iv[o] == iv[n]) p += pv[o];
                    g = w * a.scale * (expf((sv[n] - u.m) / tt - log_ul) - p);
                }
                listed[r * a.k + n] = g;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(256) distill_bwd_kernel(const T *__restrict__ x, const int64_t *__restrict__ indices, const float *__restrict__ stats,
                                                          const float *__restrict__ listed, const float *__restrict__ up, int up_stride, T *__restrict__ gx,
                                                          DistillArgs a)
{
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *row = x + r * a.stride;
        T *out = gx + r * a.classes;
        const float g = up[r * up_stride], m = stats[2 * r], coef = stats[2 * r + 1] * g;
        for (int i = threadIdx.x; i < a.classes; i += 256) out[i] = from_f<T>(coef == 0.f ? 0.f : coef * exp_diff(to_f(row[i]), m, a.c));
        __syncthreads();
        for (int n = threadIdx.x; n < a.k; n += 256) {
            const long long j = indices[r * a.k + n];
            if (j >= 0 && j < a.classes) out[j] = from_f<T>(listed[r * a.k + n] * g);
        }
    }
}

__global__ void __launch_bounds__(1024) distill_sum_kernel(const float *__restrict__ row_loss, float *__restrict__ loss, long long rows)
{
    __shared__ double red[1024];
    double mine = 0.0;
    for (long long r = threadIdx.x; r < rows; r += 1024) mine += row_loss[r];
    red[threadIdx.x] = mine;
    __syncthreads();
    for (int half = 512; half >= 1; half >>= 1) {
        if ((int)threadIdx.x < half) red[threadIdx.x] += red[threadIdx.x + half];
        __syncthreads();
    }
    if (threadIdx.x == 0) *loss = (float)red[0];
}

bool sizes_ok(int64_t rows, int64_t classes, int64_t row_stride, int k, double temperature, int dtype)
{
    return rows >= 0 && classes > 0 && row_stride >= 0 && k > 0 && temperature >= 1e-30 && temperature <= 1e30 && (dtype == CLB_F32 || dtype == CLB_F16 || dtype == CLB_BF16);
}
DistillArgs make_args(int64_t rows, int64_t classes, int64_t row_stride, int k, double temperature, int reduction)
{
    return {row_stride, rows, (int)classes, k, (float)temperature, (float)(1.4426950408889634 / temperature),
            (float)(reduction == CLB_REDUCE_MEAN && rows > 0 ? temperature / (double)rows : temperature)};
}

} // namespace

extern "C" size_t clb_distill_scratch_bytes(int64_t rows, int64_t classes, int k)
{
    if (rows <= 0 || classes <= 0 || k <= 0) return 0;
    return (size_t)rows * 4;
}

extern "C" int clb_distill_fwd(const void *scores, int64_t row_stride, const float *values, const int64_t *indices, const float *rest, const float *weight,
                               float *loss, float *stats, float *listed, void *scratch, size_t scratch_bytes, int64_t rows, int64_t classes, int k,
                               double temperature, int reduction, int dtype, void *stream)
{
    if (!loss || !sizes_ok(rows, classes, row_stride, k, temperature, dtype)) return CLB_ERR_ARG;
    if (reduction != CLB_REDUCE_NONE && reduction != CLB_REDUCE_MEAN && reduction != CLB_REDUCE_SUM) return CLB_ERR_ARG;
    if (k > CLB_TOP_MAX || classes > 0x7fffffff) return CLB_ERR_TOO_LARGE;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows > 0) {
        if (!scores || !values || !indices || !stats || !listed) return CLB_ERR_ARG;
        if (reduction != CLB_REDUCE_NONE && (!scratch || scratch_bytes < clb_distill_scratch_bytes(rows, classes, k))) return CLB_ERR_SCRATCH;
        float *row_loss = reduction == CLB_REDUCE_NONE ? loss : (float *)scratch;
        with_score_type(dtype, [&](auto t) {
            using T = decltype(t);
            CLB_TRACED("distill_fwd_kernel", st,
                       distill_fwd_kernel<T><<<(unsigned)(rows < (1 << 20) ? rows : (1 << 20)), 256, 0, st>>>(
                           (const T *)scores, values, indices, rest, weight, row_loss, stats, listed,
                           make_args(rows, classes, row_stride, k, temperature, reduction)));
        });
    }
    if (reduction == CLB_REDUCE_NONE) return rows > 0 ? check_launch() : CLB_OK;
    CLB_TRACED("distill_sum_kernel", st, distill_sum_kernel<<<1, 1024, 0, st>>>((const float *)scratch, loss, rows));
    return check_launch(rows > 0 ? 2 : 1);
}

extern "C" int clb_distill_bwd(const void *scores, int64_t row_stride, const int64_t *indices, const float *stats, const float *listed, const float *upstream,
                               int upstream_per_row, void *grad, int64_t rows, int64_t classes, int k, double temperature, int dtype, void *stream)
{
    if (!sizes_ok(rows, classes, row_stride, k, temperature, dtype)) return CLB_ERR_ARG;
    if (k > CLB_TOP_MAX || classes > 0x7fffffff) return CLB_ERR_TOO_LARGE;
    if (rows == 0) return CLB_OK;
    if (!scores || !indices || !stats || !listed || !upstream || !grad) return CLB_ERR_ARG;
    cudaStream_t st = (cudaStream_t)stream;
    with_score_type(dtype, [&](auto t) {
        using T = decltype(t);
        CLB_TRACED("distill_bwd_kernel", st,
                   distill_bwd_kernel<T><<<(unsigned)(rows < (1 << 20) ? rows : (1 << 20)), 256, 0, st>>>(
                       (const T *)scores, indices, stats, listed, upstream, upstream_per_row ? 1 : 0, (T *)grad,
                       make_args(rows, classes, row_stride, k, temperature, CLB_REDUCE_SUM)));
    });
    return check_launch();
}

// Counts per expert and the balance loss of rows of logits, and its gradient; the experts of a gate layer are its 16 operations.
//
// p = softmax(x); a kept row is one that `keep` names (or any) and that has a logit above -inf, M of them.  c_e: kept rows that have expert e among their k
// largest logits, ties to the lowest index, never a logit of -inf.
//     loss = E / (M k) sum_e c_e P_e,  P_e = (1 / M) sum of p_e over the kept rows
//     d loss / d x_j = p_j (h_j - sum_e p_e h_e),  h_e = E / (M^2 k) (c_e - mean of c)    (the counts have no gradient)
// A constant taken off every h_e changes nothing; with the mean off, the difference of two nearly equal numbers in a balanced layer is taken in 64 bits.
// Simple form: a warp per row.
#include "clb_scores.cuh"

using namespace clb;
using namespace clb_host;

namespace {

constexpr int kWarps = 8;
constexpr int kMaxBlocks = 1024;
constexpr int kSlots = CLB_BALANCE_MAX_EXPERTS / 32; // columns of a lane

int balance_blocks(long long rows) { return (int)(rows < (long long)kMaxBlocks * kWarps ? (rows + kWarps - 1) / kWarps : kMaxBlocks); }

// the row's soft-max in place (columns lane, lane + 32, ...); false for a row that is not kept
__device__ __forceinline__ bool row_softmax(float (&v)[kSlots], int lane, int experts)
{
    float m = -INFINITY;
    bool nan = false;
    for (int s = 0; s * 32 < experts; ++s) {
        m = fmaxf(m, v[s]);
        nan = nan || v[s] != v[s];
    }
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (m == -INFINITY && !__any_sync(0xffffffffu, nan)) return false;
    float l = 0.f;
    for (int s = 0; s * 32 < experts; ++s) {
        v[s] = lane + s * 32 < experts ? expf(v[s] - m) : 0.f;
        l += v[s];
    }
    l = warp_sum<float>(l);
    for (int s = 0; s * 32 < experts; ++s) v[s] /= l;
    return true;
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) balance_fwd_kernel(const T *__restrict__ x, long long stride, const uint8_t *__restrict__ keep,
                                                                  float *__restrict__ sums, int *__restrict__ counts, int *__restrict__ kept, long long rows,
                                                                  int experts, int k)
{
    __shared__ float psum[CLB_BALANCE_MAX_EXPERTS];
    __shared__ int cnt[CLB_BALANCE_MAX_EXPERTS], all;
    for (int e = threadIdx.x; e < experts; e += kWarps * 32) psum[e] = 0.f, cnt[e] = 0;
    if (threadIdx.x == 0) all = 0;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float acc[kSlots];
    int own[kSlots], mine = 0;
    for (int s = 0; s < kSlots; ++s) acc[s] = 0.f, own[s] = 0;
    for (long long r = (long long)blockIdx.x * kWarps + warp; r < rows; r += (long long)gridDim.x * kWarps) {
        if (keep && !keep[r]) continue;
        const T *row = x + r * stride;
        float v[kSlots], raw[kSlots];
        for (int s = 0; s * 32 < experts; ++s) raw[s] = v[s] = lane + s * 32 < experts ? to_f(row[lane + s * 32]) : -INFINITY;
        if (!row_softmax(v, lane, experts)) continue;
        ++mine;
        for (int s = 0; s * 32 < experts; ++s) acc[s] += v[s];
        unsigned long long last = ~0ull;
        for (int n = 0; n < k; ++n) {
            unsigned long long best = 0;
            for (int s = 0; s * 32 < experts; ++s) {
                const int e = lane + s * 32;
                const unsigned long long p = ((unsigned long long)order_key(raw[s]) << 32) | (0xffffffffu - (uint32_t)e);
                if (e < experts && raw[s] != -INFINITY && p < last && p > best) best = p;
            }
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
                if (other > best) best = other;
            }
            if (!best) break;
            last = best;
            const uint32_t e = 0xffffffffu - (uint32_t)best;
            if ((e & 31) == (uint32_t)lane) ++own[e >> 5];
        }
    }
    for (int w = 0; w < kWarps; ++w) { // warps add in turn: the same sums every time
        __syncthreads();
        if (w == warp) {
            for (int s = 0; s * 32 < experts; ++s)
                if (lane + s * 32 < experts) psum[lane + s * 32] += acc[s], cnt[lane + s * 32] += own[s];
            if (lane == 0) all += mine;
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kWarps * 32) {
        sums[(long long)blockIdx.x * experts + e] = psum[e];
        counts[(long long)blockIdx.x * experts + e] = cnt[e];
    }
    if (threadIdx.x == 0) kept[blockIdx.x] = all;
}

__global__ void __launch_bounds__(256) balance_finish_kernel(const float *__restrict__ sums, const int *__restrict__ counts, const int *__restrict__ kept,
                                                             float *__restrict__ loss, int64_t *__restrict__ total, float *__restrict__ share, int blocks,
                                                             int experts, int k)
{
    __shared__ double red[256];
    double dot = 0.0, m = 0.0, picked = 0.0;
    for (int b = 0; b < blocks; ++b) m += kept[b];
    for (int e = threadIdx.x; e < experts; e += 256) {
        double p = 0.0;
        long long c = 0;
        for (int b = 0; b < blocks; ++b) p += sums[(long long)b * experts + e], c += counts[(long long)b * experts + e];
        total[e] = c;
        dot += (double)c * p;
        picked += (double)c;
    }
    for (int round = 0; round < 2; ++round) {
        red[threadIdx.x] = round ? picked : dot;
        __syncthreads();
        for (int half = 128; half >= 1; half >>= 1) {
            if ((int)threadIdx.x < half) red[threadIdx.x] += red[threadIdx.x + half];
            __syncthreads();
        }
        if (round) picked = red[0];
        else dot = red[0];
        __syncthreads();
    }
    const double factor = m > 0.0 ? experts / (m * m * k) : 0.0;
    if (threadIdx.x == 0) *loss = (float)(factor * dot);
    for (int e = threadIdx.x; e < experts; e += 256) share[e] = (float)(factor * ((double)total[e] - picked / experts));
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) balance_bwd_kernel(const T *__restrict__ x, long long stride, const uint8_t *__restrict__ keep,
                                                                  const float *__restrict__ share, const float *__restrict__ up, T *__restrict__ gx,
                                                                  long long rows, int experts)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float g = *up;
    for (long long r = (long long)blockIdx.x * kWarps + warp; r < rows; r += (long long)gridDim.x * kWarps) {
        const T *row = x + r * stride;
        float v[kSlots];
        for (int s = 0; s * 32 < experts; ++s) v[s] = lane + s * 32 < experts ? to_f(row[lane + s * 32]) : -INFINITY;
        const bool there = (!keep || keep[r]) && row_softmax(v, lane, experts);
        float dot = 0.f;
        if (there)
            for (int s = 0; s * 32 < experts; ++s)
                if (lane + s * 32 < experts) dot += v[s] * share[lane + s * 32];
        dot = warp_sum<float>(dot);
        for (int s = 0; s * 32 < experts; ++s)
            if (lane + s * 32 < experts) gx[r * experts + lane + s * 32] = from_f<T>(there ? g * v[s] * (share[lane + s * 32] - dot) : 0.f);
    }
}

} // namespace

extern "C" size_t clb_balance_scratch_bytes(int64_t rows, int64_t experts)
{
    if (rows <= 0 || experts <= 0 || experts > CLB_BALANCE_MAX_EXPERTS) return 0;
    return (size_t)balance_blocks(rows) * (size_t)(8 * experts + 4);
}

extern "C" int clb_balance_fwd(const void *x, int64_t row_stride, const uint8_t *keep, float *loss, int64_t *counts, float *share, void *scratch,
                               size_t scratch_bytes, int64_t rows, int64_t experts, int k, int dtype, void *stream)
{
    if (!loss || !counts || !share || rows < 0 || experts <= 0 || row_stride < 0 || k <= 0) return CLB_ERR_ARG;
    if (dtype != CLB_F32 && dtype != CLB_F16 && dtype != CLB_BF16) return CLB_ERR_ARG;
    if (k > experts) return CLB_ERR_SHAPE;
    if (experts > CLB_BALANCE_MAX_EXPERTS || k > CLB_BALANCE_MAX_TOP || rows > 0x7fffffff) return CLB_ERR_TOO_LARGE;
    if (rows > 0 && !x) return CLB_ERR_ARG;
    if (rows > 0 && (!scratch || scratch_bytes < clb_balance_scratch_bytes(rows, experts))) return CLB_ERR_SCRATCH;
    cudaStream_t st = (cudaStream_t)stream;
    const int blocks = balance_blocks(rows);
    float *sums = (float *)scratch;
    int *cnt = (int *)(sums + (long long)blocks * experts), *kept = cnt + (long long)blocks * experts;
    if (rows > 0)
        with_score_type(dtype, [&](auto t) {
            using T = decltype(t);
            CLB_TRACED("balance_fwd_kernel", st,
                       balance_fwd_kernel<T><<<blocks, kWarps * 32, 0, st>>>((const T *)x, row_stride, keep, sums, cnt, kept, rows, (int)experts, k));
        });
    CLB_TRACED("balance_finish_kernel", st, balance_finish_kernel<<<1, 256, 0, st>>>(sums, cnt, kept, loss, counts, share, blocks, (int)experts, k));
    return check_launch(rows > 0 ? 2 : 1);
}

extern "C" int clb_balance_bwd(const void *x, int64_t row_stride, const uint8_t *keep, const float *share, const float *upstream, void *grad, int64_t rows,
                               int64_t experts, int dtype, void *stream)
{
    if (rows < 0 || experts <= 0 || row_stride < 0 || (dtype != CLB_F32 && dtype != CLB_F16 && dtype != CLB_BF16)) return CLB_ERR_ARG;
    if (experts > CLB_BALANCE_MAX_EXPERTS || rows > 0x7fffffff) return CLB_ERR_TOO_LARGE;
    if (rows == 0) return CLB_OK;
    if (!x || !share || !upstream || !grad) return CLB_ERR_ARG;
    cudaStream_t st = (cudaStream_t)stream;
    with_score_type(dtype, [&](auto t) {
        using T = decltype(t);
        CLB_TRACED("balance_bwd_kernel", st,
                   balance_bwd_kernel<T><<<balance_blocks(rows), kWarps * 32, 0, st>>>((const T *)x, row_stride, keep, share, upstream, (T *)grad, rows,
                                                                                     (int)experts));
    });
    return check_launch();
}

// The k largest logits of every row and the mass of the others, for losses against a teacher's lists.
//
// A row's classes are ordered by value, ties by index; the first k are the list, and rest = log sum over the others of exp(x / T).
// Simple form: a block per row that looks for the next class after the last one, k times.
#include "clb_scores.cuh"

using namespace clb;
using namespace clb_host;

namespace {

// (order of the value, index) as one number: larger comes first in a row's list
__device__ __forceinline__ unsigned long long place(float v, long long i) { return ((unsigned long long)order_key(v) << 32) | (0xffffffffu - (uint32_t)i); }

template <typename T>
__global__ void __launch_bounds__(256) top_logits_kernel(const T *__restrict__ x, long long stride, float *__restrict__ values, int64_t *__restrict__ indices,
                                                         float *__restrict__ rest, long long rows, int classes, int k, float temperature, float c)
{
    __shared__ unsigned long long best[8];
    __shared__ ExpSum part[8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (long long r = blockIdx.x; r < rows; r += gridDim.x) {
        const T *row = x + r * stride;
        unsigned long long last = ~0ull;
        for (int n = 0; n < k; ++n) {
            unsigned long long mine = 0;
            for (int i = threadIdx.x; i < classes; i += 256) {
                const unsigned long long p = place(to_f(row[i]), i);
                if (p < last && p > mine) mine = p;
            }
            for (int o = 16; o > 0; o >>= 1) {
                const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
                if (other > mine) mine = other;
            }
            if (lane == 0) best[warp] = mine;
            __syncthreads();
            for (int w = 0; w < 8; ++w)
                if (w == 0 || best[w] > mine) mine = best[w];
            __syncthreads();
            last = mine;
            if (threadIdx.x == 0) {
                const uint32_t i = 0xffffffffu - (uint32_t)last;
                values[r * k + n] = to_f(row[i]);
                indices[r * k + n] = i;
            }
        }
        ExpSum s{-INFINITY, 0.f};
        bool inf = false;
        for (int i = threadIdx.x; i < classes; i += 256) {
            const float v = to_f(row[i]);
            if (place(v, i) >= last) continue;
            if (v == INFINITY) inf = true;
            else s = merge(s, single(v), c);
        }
        inf = __syncthreads_or(inf);
        s = warp_merge(s, c);
        if (lane == 0) part[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < 8; ++w) s = merge(s, part[w], c);
            rest[r] = inf && s.l == s.l ? INFINITY : s.m / temperature + logf(s.l);
        }
        __syncthreads();
    }
}

} // namespace

extern "C" int clb_top_logits(const void *x, int64_t row_stride, float *values, int64_t *indices, float *rest, int64_t rows, int64_t classes, int k,
                              double temperature, int dtype, void *stream)
{
    if (!x || !values || !indices || !rest || rows < 0 || classes <= 0 || row_stride < 0 || k <= 0 || !(temperature >= 1e-30 && temperature <= 1e30)) return CLB_ERR_ARG;
    if (k > classes) return CLB_ERR_SHAPE;
    if (k > CLB_TOP_MAX || classes > CLB_CLASSES_MAX) return CLB_ERR_TOO_LARGE;
    if (dtype != CLB_F32 && dtype != CLB_F16 && dtype != CLB_BF16) return CLB_ERR_ARG;
    if (rows == 0) return CLB_OK;
    cudaStream_t st = (cudaStream_t)stream;
    with_score_type(dtype, [&](auto t) {
        using T = decltype(t);
        CLB_TRACED("top_logits_kernel", st,
                   top_logits_kernel<T><<<(unsigned)(rows < (1 << 20) ? rows : (1 << 20)), 256, 0, st>>>(
                       (const T *)x, row_stride, values, indices, rest, rows, (int)classes, k, (float)temperature, (float)(1.4426950408889634 / temperature)));
    });
    return check_launch();
}

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
//
// A team of threads holds the row in registers (clb_rows.cuh): one read of the scores, a maximum, a sum, and the gradient from the same registers.  Listed
// classes are struck out there (a bit per value in shared memory, set by the threads that hold the list), so that the sums over listed and unlisted
// classes are kept apart from the start.
#include <cooperative_groups.h>

#include "clb_rows.cuh"

using namespace clb;
using namespace clb_host;

namespace {

struct DistillArgs {
    long long stride, rows;
    int classes, k;
    float temperature, c, scale; // c = log2(e) / T; scale: T, over the rows for a mean
};

template <typename T> struct Entry { // one class of a list: cls < 0: does not exist
    int cls;
    float t, s;
};
template <typename T>
__device__ __forceinline__ Entry<T> list_entry(const T *row, const int64_t *idx, const float *val, int n, int classes)
{
    const long long j = idx[n];
    Entry<T> e{-1, -INFINITY, -INFINITY};
    if (j >= 0 && j < classes) e.cls = (int)j, e.t = val[n], e.s = to_f(row[j]);
    return e;
}

// TH threads a row (4 to 32: teams of a block of 256; more: the block), NV pieces a thread.  CLUSTER: the blocks of a cluster share a row.
// grad: where d loss / d scores goes for an upstream gradient of one, or NULL.
template <typename T, int TH, int NV, bool CLUSTER>
__global__ void __launch_bounds__(TH <= 32 ? 256 : TH, TH <= 32 ? 4 : 1024 / TH)
    distill_fwd_kernel(const T *__restrict__ x, const float *__restrict__ values, const int64_t *__restrict__ indices, const float *__restrict__ rest,
                       const float *__restrict__ weight, float *__restrict__ row_loss, float *__restrict__ stats, float *__restrict__ listed, T *grad, DistillArgs a)
{
    namespace cg = cooperative_groups;
    constexpr int BLOCK = TH <= 32 ? 256 : TH, TEAMS = BLOCK / TH, EV = kPiece<T>, WORDS = NV * EV <= 32 ? 1 : 2; // bits of a thread's values
    __shared__ uint32_t bits[WORDS][BLOCK];
    __shared__ float red[3][3 * 32];
    __shared__ float peer[2][16];
    const int t = threadIdx.x % TH, team = threadIdx.x / TH;
    const int ranks = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1, rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0;
    const long long groups = (long long)(gridDim.x / ranks) * TEAMS;
    auto team_sync = [] {
        if (TH <= 32) __syncwarp();
        else __syncthreads();
    };
    if (CLUSTER) cg::this_cluster().barrier_arrive(); // no block writes to another's memory before that one runs
    // every team of a warp takes every turn, on its last row again where it has none left
    const long long turns = (a.rows + groups - 1) / groups;
    for (long long turn = 0; turn < turns; ++turn) {
        const long long r0 = turn * groups + (long long)(blockIdx.x / ranks) * TEAMS + team;
        const bool live = r0 < a.rows;
        const long long r = live ? r0 : a.rows - 1;
        const RowPieces<T> row(x + r * a.stride, a.classes);
        const int64_t *idx = indices + r * a.k;
        const float *val = values + r * a.k;
        const float w = weight ? weight[r] : 1.f, rs = rest ? rest[r] : -INFINITY, tt = a.temperature;
        const int chunks = TH <= 32 ? 1 : (row.pieces + ranks * TH * NV - 1) / (ranks * TH * NV);
        uint32_t raw[NV][4];
        bool twice = false;
        Entry<T> own{-1, -INFINITY, -INFINITY};
        if (t < a.k) own = list_entry(row.row, idx, val, t, a.classes);
        auto entry = [&](int n) { return n == t ? own : list_entry(row.row, idx, val, n, a.classes); };
        auto fetch = [&](int chunk) { // the thread's pieces, without the listed classes
            const int base = (chunk * ranks + rank) * TH * NV;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const uint4 q = row.load(base + v * TH + t);
                raw[v][0] = q.x, raw[v][1] = q.y, raw[v][2] = q.z, raw[v][3] = q.w;
            }
#pragma unroll
            for (int i = 0; i < WORDS; ++i) bits[i][threadIdx.x] = 0;
            team_sync();
            for (int n = t; n < a.k; n += TH) {
                const int cls = entry(n).cls;
                const int j = cls < 0 ? -1 : row.piece_of(cls) - base;
                if (j < 0 || j >= TH * NV) continue;
                const int bit = j / TH * EV + row.place_of(cls);
                const uint32_t old = atomicOr(&bits[bit >> 5][team * TH + j % TH], 1u << (bit & 31));
                twice = twice || ((old >> (bit & 31)) & 1);
            }
            team_sync();
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                const uint32_t m = bits[(v * EV) >> 5][threadIdx.x] >> ((v * EV) & 31);
                if (m & ((1u << EV) - 1))
#pragma unroll
                    for (int e = 0; e < EV; ++e)
                        if ((m >> e) & 1) drop_value<T>(raw[v], e);
            }
        };
        // ---- maxima: unlisted scores, listed scores, the teacher's list, and whether a class is listed twice
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, 0.f};
        uint32_t top = low_word<T>();
        for (int ch = 0; ch < chunks; ++ch) {
            fetch(ch);
#pragma unroll
            for (int v = 0; v < NV; ++v)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = Word<T>::max(top, raw[v][i]);
        }
        {
            float f[Word<T>::n];
            Word<T>::get(top, f);
#pragma unroll
            for (int i = 0; i < Word<T>::n; ++i) mx[0] = fmaxf(mx[0], f[i]);
        }
        for (int n = t; n < a.k; n += TH) {
            const Entry<T> e = entry(n);
            mx[1] = fmaxf(mx[1], e.s), mx[2] = fmaxf(mx[2], e.t);
        }
        mx[3] = twice ? 1.f : 0.f;
        team_reduce<TH, true, 4>(mx, red[0]);
        if (CLUSTER) {
            auto cl = cg::this_cluster();
            if (turn == 0) cl.barrier_wait();
            if (threadIdx.x < ranks) {
                float *to = cl.map_shared_rank(&peer[0][0], threadIdx.x);
                to[rank] = mx[0], to[8 + rank] = mx[3];
            }
            cl.sync();
            for (int i = 0; i < ranks; ++i) mx[0] = fmaxf(mx[0], peer[0][i]), mx[3] = fmaxf(mx[3], peer[0][8 + i]);
        }
        const float m = finite_or_zero(mx[0]), mk = finite_or_zero(mx[1]), mt = finite_or_zero(mx[2]);
        const bool dup = mx[3] != 0.f;
        // ---- sums
        float sum[3] = {0.f, 0.f, 0.f};
        for (int ch = 0; ch < chunks; ++ch) {
            if (chunks > 1) fetch(ch);
            const int base = (ch * ranks + rank) * TH * NV;
#pragma unroll
            for (int v = 0; v < NV; ++v) {
                if (base + v * TH >= row.pieces) break;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    float f[Word<T>::n];
                    Word<T>::get(raw[v][i], f);
#pragma unroll
                    for (int q = 0; q < Word<T>::n; ++q) sum[0] += ex2((f[q] - m) * a.c);
                }
            }
        }
        for (int n = t; n < a.k; n += TH) {
            const Entry<T> e = entry(n);
            if (e.cls < 0) continue;
            bool first = true;
            if (dup)
                for (int o = 0; o < n; ++o) first = first && idx[o] != e.cls;
            if (first) sum[1] += expf((e.s - mk) / tt);
            sum[2] += expf((e.t - mt) / tt);
        }
        team_reduce<TH, false, 3>(sum, red[1]);
        if (CLUSTER) {
            auto cl = cg::this_cluster();
            if (threadIdx.x < ranks) cl.map_shared_rank(&peer[1][0], threadIdx.x)[rank] = sum[0];
            cl.sync();
            sum[0] = 0.f;
            for (int i = 0; i < ranks; ++i) sum[0] += peer[1][i];
        }
        // ---- the row's numbers, in every thread
        const bool no_rest = mx[0] == -INFINITY && sum[0] == 0.f, no_list = mx[1] == -INFINITY && sum[1] == 0.f;
        const float um = finite_or_zero(fmaxf(mx[0], mx[1]));
        const float ul = (no_rest ? 0.f : sum[0] * expf((m - um) / tt)) + (no_list ? 0.f : sum[1] * expf((mk - um) / tt));
        const float tz = mx[2] == -INFINITY ? -INFINITY : mt / tt, tm = finite_or_zero(fmaxf(tz, rs));
        const float tl = (mx[2] == -INFINITY ? sum[2] : sum[2] * expf(tz - tm)) + expf(rs - tm);
        const bool there = w != 0.f && tl != 0.f && !(no_rest && no_list);
        const float log_ul = logf(ul), log_tl = logf(tl);
        const float lr = (rs - tm) - log_tl, rp = expf(lr);
        const float lqr = no_rest ? -INFINITY : ((m - um) / tt + logf(sum[0])) - log_ul;
        const float coef = there && !no_rest ? w * a.scale * (expf(lqr) - rp) / sum[0] : 0.f;
        T *out = grad ? grad + r * a.classes : nullptr;
        const bool aligned = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
        if (grad)
            for (int ch = 0; ch < chunks; ++ch) {
                if (chunks > 1) fetch(ch);
                const int base = (ch * ranks + rank) * TH * NV;
#pragma unroll
                for (int v = 0; v < NV; ++v) {
                    const int j = base + v * TH + t;
                    if (j >= row.pieces || !live) continue;
                    uint4 q = make_uint4(0, 0, 0, 0);
                    uint32_t *o = &q.x;
                    if (coef != 0.f)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float f[Word<T>::n];
                            Word<T>::get(raw[v][i], f);
#pragma unroll
                            for (int z = 0; z < Word<T>::n; ++z) f[z] = coef * ex2((f[z] - m) * a.c);
                            o[i] = Word<T>::put(f);
                        }
                    row.store(out, aligned, j, q);
                }
                }
        // ---- the list: loss, and the gradient of its classes
        if (grad) team_sync(); // a listed class is written after the piece that it lies in
        float loss[1] = {0.f};
        for (int n = t; n < a.k; n += TH) {
            const Entry<T> e = entry(n);
            float g = 0.f;
            if (there && e.cls >= 0) {
                const float lp = ((e.t / tt) - tm) - log_tl, lq = (e.s - um) / tt - log_ul, p = expf(lp);
                if (p > 0.f || p != p) loss[0] += p * (lp - lq);
                float mass = p;
                if (dup) { // both entries' probability, in the list's order
                    mass = 0.f;
                    for (int o = 0; o < a.k; ++o)
                        if (idx[o] == e.cls) mass += expf(((val[o] / tt) - tm) - log_tl);
                }
                g = w * a.scale * (expf(lq) - mass);
            }
            if (rank == 0 && live) listed[r * a.k + n] = g;
            if (grad && live && e.cls >= 0) {
                const int j = row.piece_of(e.cls) / (TH * NV);
                if (!CLUSTER || j % ranks == rank) out[e.cls] = from_f<T>(g);
            }
        }
        team_reduce<TH, false, 1>(loss, red[2]);
        if (t == 0 && rank == 0 && live) {
            if (there && (rp > 0.f || rp != rp)) loss[0] += rp * (lr - lqr);
            row_loss[r] = there ? loss[0] * w * a.scale * tt : 0.f;
            stats[2 * r] = m, stats[2 * r + 1] = coef;
        }
        // (the tables are used again: each has a barrier of its team, or of the cluster, between the last read of this turn and the next turn's write)
    }
}

// The gradient from what the forward kept: a block takes TH * NV pieces of a row (or rows, for teams of a warp) at a time.
template <typename T, int TH, int NV>
__global__ void __launch_bounds__(256) distill_bwd_kernel(const T *__restrict__ x, const int64_t *__restrict__ indices, const float *__restrict__ stats,
                                                          const float *__restrict__ listed, const float *__restrict__ up, int up_stride, int unit_done,
                                                          T *__restrict__ gx, int parts, DistillArgs a)
{
    constexpr int TEAMS = 256 / TH;
    if (unit_done && *up == 1.f) return; // the forward has written this gradient
    const int t = threadIdx.x % TH, team = threadIdx.x / TH;
    const long long items = a.rows * parts, groups = (long long)gridDim.x * TEAMS, turns = (items + groups - 1) / groups;
    for (long long turn = 0; turn < turns; ++turn) {
        const long long item = turn * groups + (long long)blockIdx.x * TEAMS + team;
        const bool live = item < items;
        const long long r = (live ? item : items - 1) / parts;
        const int base = (int)((live ? item : items - 1) - r * parts) * TH * NV;
        const RowPieces<T> row(x + r * a.stride, a.classes);
        T *out = gx + r * a.classes;
        const bool aligned = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
        uint4 raw[NV];
#pragma unroll
        for (int v = 0; v < NV; ++v) raw[v] = row.load(base + v * TH + t);
        const float g = up[r * up_stride], m = stats[2 * r], coef = stats[2 * r + 1] * g;
#pragma unroll
        for (int v = 0; v < NV; ++v) {
            const int j = base + v * TH + t;
            if (j >= row.pieces || !live) continue;
            uint32_t *o = &raw[v].x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float f[Word<T>::n];
                Word<T>::get(o[i], f);
#pragma unroll
                for (int z = 0; z < Word<T>::n; ++z) f[z] = coef == 0.f ? 0.f : coef * ex2((f[z] - m) * a.c);
                o[i] = Word<T>::put(f);
            }
            row.store(out, aligned, j, raw[v]);
        }
        if (TH <= 32) __syncwarp();
        else __syncthreads();
        for (int n = t; n < a.k && live; n += TH) {
            const long long cls = indices[r * a.k + n];
            if (cls < 0 || cls >= a.classes) continue;
            const int j = row.piece_of((int)cls) - base;
            if (j >= 0 && j < TH * NV) out[cls] = from_f<T>(listed[r * a.k + n] * g);
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
    return rows >= 0 && classes > 0 && row_stride >= 0 && k > 0 && temperature >= 1e-30 && temperature <= 1e30 &&
           (dtype == CLB_F32 || dtype == CLB_F16 || dtype == CLB_BF16);
}
DistillArgs make_args(int64_t rows, int64_t classes, int64_t row_stride, int k, double temperature, int reduction)
{
    return {row_stride, rows, (int)classes, k, (float)temperature, (float)(1.4426950408889634 / temperature),
            (float)(reduction == CLB_REDUCE_MEAN && rows > 0 ? temperature / (double)rows : temperature)};
}

struct FwdPointers {
    const float *values;
    const int64_t *indices;
    const float *rest, *weight;
    float *row_loss, *stats, *listed;
};

template <typename T, int TH, int NV, bool CLUSTER>
cudaError_t launch_fwd(const T *x, const FwdPointers &p, T *grad, const DistillArgs &a, int cluster, cudaStream_t st)
{
    constexpr int BLOCK = TH <= 32 ? 256 : TH, TEAMS = BLOCK / TH;
    const long long groups = (a.rows + TEAMS - 1) / TEAMS, most = (1 << 20) / cluster;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((groups < most ? groups : most) * cluster)), cfg.blockDim = dim3(BLOCK), cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)cluster, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = CLUSTER ? 1 : 0;
    cudaError_t rc;
    CLB_TRACED("distill_fwd_kernel", st,
               rc = cudaLaunchKernelEx(&cfg, distill_fwd_kernel<T, TH, NV, CLUSTER>, x, p.values, p.indices, p.rest, p.weight, p.row_loss, p.stats, p.listed,
                                       grad, a));
    return rc;
}
template <typename T> cudaError_t run_fwd(const T *x, const FwdPointers &p, T *grad, const DistillArgs &a, cudaStream_t st)
{
    const long long pieces = (a.classes + 2LL * kPiece<T> - 2) / kPiece<T>;
    if (pieces <= 4) return launch_fwd<T, 4, 1, false>(x, p, grad, a, 1, st);
    if (pieces <= 32) return launch_fwd<T, 8, 4, false>(x, p, grad, a, 1, st);
    if (pieces <= 256) return launch_fwd<T, 32, 8, false>(x, p, grad, a, 1, st);
    if (pieces <= 1024) return launch_fwd<T, 128, 8, false>(x, p, grad, a, 1, st);
    if (pieces <= 2048) return launch_fwd<T, 256, 8, false>(x, p, grad, a, 1, st);
    if (pieces <= 4096) return launch_fwd<T, 512, 8, false>(x, p, grad, a, 1, st);
    if (pieces <= 8 * 4096) return launch_fwd<T, 512, 8, true>(x, p, grad, a, pieces <= 2 * 4096 ? 2 : pieces <= 4 * 4096 ? 4 : 8, st);
    return launch_fwd<T, 1024, 8, true>(x, p, grad, a, 8, st);
}

template <typename T, int TH, int NV>
void launch_bwd(const T *x, const int64_t *indices, const float *stats, const float *listed, const float *up, int per_row, int unit_done, T *grad,
                const DistillArgs &a, long long pieces, cudaStream_t st)
{
    const long long parts = (pieces + TH * NV - 1) / (TH * NV), blocks = (a.rows * parts + 256 / TH - 1) / (256 / TH), most = 8LL * sm_count();
    CLB_TRACED("distill_bwd_kernel", st,
               distill_bwd_kernel<T, TH, NV><<<(unsigned)(blocks < most ? blocks : most), 256, 0, st>>>(x, indices, stats, listed, up, per_row, unit_done, grad,
                                                                                                      (int)parts, a));
}

} // namespace

extern "C" size_t clb_distill_scratch_bytes(int64_t rows, int64_t classes, int k)
{
    if (rows <= 0 || classes <= 0 || k <= 0) return 0;
    return (size_t)rows * 4;
}

extern "C" int clb_distill_fwd(const void *scores, int64_t row_stride, const float *values, const int64_t *indices, const float *rest, const float *weight,
                               float *loss, float *stats, float *listed, void *grad, void *scratch, size_t scratch_bytes, int64_t rows, int64_t classes, int k,
                               double temperature, int reduction, int dtype, void *stream)
{
    if (!loss || !sizes_ok(rows, classes, row_stride, k, temperature, dtype)) return CLB_ERR_ARG;
    if (reduction != CLB_REDUCE_NONE && reduction != CLB_REDUCE_MEAN && reduction != CLB_REDUCE_SUM) return CLB_ERR_ARG;
    if (k > CLB_TOP_MAX || classes > CLB_CLASSES_MAX) return CLB_ERR_TOO_LARGE;
    cudaStream_t st = (cudaStream_t)stream;
    if (rows > 0) {
        if (!scores || !values || !indices || !stats || !listed) return CLB_ERR_ARG;
        if (reduction != CLB_REDUCE_NONE && (!scratch || scratch_bytes < clb_distill_scratch_bytes(rows, classes, k))) return CLB_ERR_SCRATCH;
        const FwdPointers p{values, indices, rest, weight, reduction == CLB_REDUCE_NONE ? loss : (float *)scratch, stats, listed};
        cudaError_t rc = cudaSuccess;
        with_score_type(dtype, [&](auto t) {
            using T = decltype(t);
            rc = run_fwd<T>((const T *)scores, p, (T *)grad, make_args(rows, classes, row_stride, k, temperature, reduction), st);
        });
        if (rc != cudaSuccess) return check_launch(0);
    }
    if (reduction == CLB_REDUCE_NONE) return rows > 0 ? check_launch() : CLB_OK;
    CLB_TRACED("distill_sum_kernel", st, distill_sum_kernel<<<1, 1024, 0, st>>>((const float *)scratch, loss, rows));
    return check_launch(rows > 0 ? 2 : 1);
}

extern "C" int clb_distill_bwd(const void *scores, int64_t row_stride, const int64_t *indices, const float *stats, const float *listed, const float *upstream,
                               int upstream_per_row, int unit_done, void *grad, int64_t rows, int64_t classes, int k, double temperature, int dtype,
                               void *stream)
{
    if (!sizes_ok(rows, classes, row_stride, k, temperature, dtype) || (unit_done && upstream_per_row)) return CLB_ERR_ARG;
    if (k > CLB_TOP_MAX || classes > CLB_CLASSES_MAX) return CLB_ERR_TOO_LARGE;
    if (rows == 0) return CLB_OK;
    if (!scores || !indices || !stats || !listed || !upstream || !grad) return CLB_ERR_ARG;
    cudaStream_t st = (cudaStream_t)stream;
    with_score_type(dtype, [&](auto t) {
        using T = decltype(t);
        const DistillArgs a = make_args(rows, classes, row_stride, k, temperature, CLB_REDUCE_SUM);
        const long long pieces = (classes + 2LL * kPiece<T> - 2) / kPiece<T>;
        auto go = [&](auto launch) { launch((const T *)scores, indices, stats, listed, upstream, upstream_per_row ? 1 : 0, unit_done ? 1 : 0, (T *)grad, a, pieces, st); };
        if (pieces <= 4) go(launch_bwd<T, 4, 1>);
        else if (pieces <= 32) go(launch_bwd<T, 8, 4>);
        else if (pieces <= 128) go(launch_bwd<T, 32, 4>);
        else go(launch_bwd<T, 256, 4>);
    });
    return check_launch();
}

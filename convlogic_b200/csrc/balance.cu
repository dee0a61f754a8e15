// Counts per expert and the balance loss of rows of logits, and its gradient; the experts of a gate layer are its 16 operations.
//
// p = softmax(x); a kept row is one that `keep` names (or any) and that has a logit above -inf, M of them.  c_e: kept rows that have expert e among their k
// largest logits, ties to the lowest index, never a logit of -inf.
//     loss = E / (M k) sum_e c_e P_e,  P_e = (1 / M) sum of p_e over the kept rows
//     d loss / d x_j = p_j (h_j - sum_e p_e h_e),  h_e = E / (M^2 k) (c_e - C)    (the counts have no gradient)
// A constant C changes nothing.  With the mean of c under the average probabilities, the difference of two nearly equal numbers in a balanced layer is taken in
// 64 bits: 673550 rows of 16 experts, one of them masked, 7 chosen: 1.4e-4 off with C = 0, 1.2e-5 with the plain mean, 2e-7 so.
//
// G lanes (1 to 32) hold a row, 16 or 32 columns each and always the same ones, so that a lane adds up its columns' probabilities and counts in registers over
// all its rows: no atomics on floats, the same sums every time.  The backward pass goes through the rows from the last one on, which is what the L2 still
// holds.  2621440 rows of 16 fp32, one choice: 41 us (4.1 TB/s) and 59 us (5.7 TB/s, reading and writing); 65536 of 128 bf16, eight choices: 25 us, issue.
#include <algorithm>
#include <cooperative_groups.h>
#include <type_traits>

#include "clb_rows.cuh"

using namespace clb;
using namespace clb_host;

namespace cg = cooperative_groups;

namespace {

template <int NC> constexpr int kThreads = NC > 16 ? 128 : 256; // of a block (32 columns a lane: what four warps' sums take of shared memory)
template <int G, int NC> constexpr int kResident = NC > 16 || G == 1 ? 4 : 3; // blocks an SM, which is how many are launched
constexpr float kLog2e = 1.44269504f;

// The columns of lane t of G: pieces of 16 bytes (VEC: rows at multiples of 16 bytes, whole pieces), or every G-th column.  Ascending either way.
template <typename T, int G, int NC, bool VEC> __device__ __forceinline__ int column(int i, int t)
{
    constexpr int EV = kPiece<T>;
    return VEC ? (i / EV * G + t) * EV + i % EV : i * G + t;
}
template <typename T, int G, int NC, bool VEC> __device__ __forceinline__ void load_row(float (&v)[NC], const T *row, int t, int experts)
{
    constexpr int EV = kPiece<T>;
    if constexpr (VEC) {
        uint4 q[NC / EV];
#pragma unroll
        for (int i = 0; i < NC / EV; ++i) {
            q[i] = make_uint4(low_word<T>(), low_word<T>(), low_word<T>(), low_word<T>());
            if ((i * G + t) * EV < experts) q[i] = *reinterpret_cast<const uint4 *>(row + (i * G + t) * EV);
        }
#pragma unroll
        for (int i = 0; i < NC / EV; ++i) {
            const uint32_t w[4] = {q[i].x, q[i].y, q[i].z, q[i].w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float f[Word<T>::n];
                Word<T>::get(w[j], f);
#pragma unroll
                for (int z = 0; z < Word<T>::n; ++z) v[i * EV + j * Word<T>::n + z] = f[z];
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = i * G + t < experts ? to_f(row[i * G + t]) : -INFINITY;
    }
}
// v becomes the row's probabilities; 0 for a row without a logit above -inf (whose v is then NaN), NaN for one that holds NaN
template <int G, int NC> __device__ __forceinline__ float soft_max(float (&v)[NC])
{
    float m = v[0];
#pragma unroll
    for (int i = 1; i < NC; ++i) m = fmaxf(m, v[i]);
    m = lanes_max<G>(m);
    const float ref = finite_or_zero(m);
    float l = 0.f;
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        v[i] = ex2((v[i] - ref) * kLog2e);
        l += v[i];
    }
    l = lanes_sum<G>(l);
    const float inv = 1.f / l;
#pragma unroll
    for (int i = 0; i < NC; ++i) v[i] *= inv;
    return l;
}

// Adds the k largest of a row to the bytes of `own`: equal ones by column, never one of -inf.  One after the other: the largest, the first of equal ones, then it
// becomes -inf.
template <typename T, int G, int NC, bool VEC> __device__ __forceinline__ void choose_in_turn(float (&u)[NC], uint32_t (&own)[NC / 4], int t, int k)
{
    for (int n = 0; n < k; ++n) {
        float best = u[0];
        int at = 0;
#pragma unroll
        for (int i = 1; i < NC; ++i)
            if (u[i] > best) best = u[i], at = i;
        float top = best;
        if (G > 1) {
            top = lanes_max<G>(best);
            const int col = column<T, G, NC, VEC>(at, t);
            int first = best == top ? col : 0x7fffffff;
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1) first = min(first, __shfl_xor_sync(0xffffffffu, first, o));
            if (first != col) at = -1;
        }
        if (top == -INFINITY) at = -1; // nothing is left to choose
#pragma unroll
        for (int i = 0; i < NC / 4; ++i) own[i] += at >> 2 == i ? 1u << ((at & 3) * 8) : 0u;
        if (n + 1 < k)
#pragma unroll
            for (int i = 0; i < NC; ++i) u[i] = i == at ? -INFINITY : u[i];
    }
}
// The same by the k-th largest value: every lane sorts its own, the team takes the first of a lane's k times.  What is above it is chosen, then as many of
// those that equal it as are missing.
template <typename T, int G, int NC, bool VEC> __device__ __forceinline__ void choose_sorted(const float (&u)[NC], uint32_t (&own)[NC / 4], int t, int k)
{
    const int lane = threadIdx.x & 31;
    float w[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) w[i] = u[i];
    odd_even_merges<NC>([&](int i, int j) {
        const float hi = fmaxf(w[i], w[j]);
        w[j] = fminf(w[i], w[j]), w[i] = hi;
    });
    float bound = w[0];
    if (G == 1) {
#pragma unroll
        for (int i = 1; i < NC; ++i) bound = i == k - 1 ? w[i] : bound;
    } else {
        constexpr uint32_t kTeam = G == 32 ? 0xffffffffu : (1u << G) - 1;
        for (int n = 0; n < k; ++n) {
            bound = lanes_max<G>(w[0]);
            const uint32_t holders = __ballot_sync(0xffffffffu, w[0] == bound) & (kTeam << (lane & ~(G - 1)));
            const bool taken = (holders & (0u - holders)) == 1u << lane;
#pragma unroll
            for (int i = 0; i < NC - 1; ++i) w[i] = taken ? w[i + 1] : w[i];
            w[NC - 1] = taken ? -INFINITY : w[NC - 1];
        }
    }
    bound = fmaxf(bound, -3.402823466e38f);
    int above = 0, equal = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) above += u[i] > bound, equal += u[i] == bound;
    if (G > 1) {
        int both = above | equal << 16;
#pragma unroll
        for (int o = G / 2; o > 0; o >>= 1) both += __shfl_xor_sync(0xffffffffu, both, o);
        above = both & 0xffff, equal = both >> 16;
    }
    int missing = min(k - above, equal);
    if (G > 1 && !__any_sync(0xffffffffu, missing < equal)) {
#pragma unroll
        for (int i = 0; i < NC; ++i) own[i / 4] += u[i] >= bound ? 1u << (i % 4 * 8) : 0u;
        return;
    }
    // columns ascend with a lane's i: each piece of 16 bytes (each column) after those of the lanes before
    constexpr int RUN = VEC ? kPiece<T> : 1;
#pragma unroll
    for (int i0 = 0; i0 < NC; i0 += RUN) {
        int here = 0, before = 0;
#pragma unroll
        for (int i = i0; i < i0 + RUN; ++i) here += u[i] == bound;
        int upto = here;
        if (G > 1) {
#pragma unroll
            for (int o = 1; o < G; o *= 2) {
                const int n = __shfl_up_sync(0xffffffffu, upto, o, G);
                upto += t >= o ? n : 0;
            }
            before = upto - here;
            upto = __shfl_sync(0xffffffffu, upto, G - 1, G);
        }
#pragma unroll
        for (int i = i0; i < i0 + RUN; ++i) {
            const bool same = u[i] == bound;
            own[i / 4] += u[i] > bound || (same && before < missing) ? 1u << (i % 4 * 8) : 0u;
            before += same;
        }
        missing -= upto;
    }
}

// A row's choices are counted as bytes in a lane's registers, handed to the block every 255 rows (NaN counts as +inf).
template <typename T, int G, int NC, bool VEC, bool SORT>
__global__ void __launch_bounds__(kThreads<NC>, kResident<G, NC>) balance_fwd_kernel(const T *__restrict__ x, long long stride, const uint8_t *__restrict__ keep,
                                                               float *__restrict__ sums, int *__restrict__ counts, int *__restrict__ kept, int rows, int experts,
                                                               int k)
{
    constexpr int TEAMS = kThreads<NC> / G, WARPS = kThreads<NC> / 32;
    __shared__ float psum[WARPS][G * NC];
    __shared__ int cnt[G * NC], all[WARPS];
    const int t = threadIdx.x % G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int e = threadIdx.x; e < G * NC; e += kThreads<NC>) cnt[e] = 0;
    __syncthreads();
    float acc[NC];
    uint32_t own[NC / 4];
    int mine = 0, since = 0;
#pragma unroll
    for (int i = 0; i < NC; ++i) acc[i] = 0.f;
#pragma unroll
    for (int i = 0; i < NC / 4; ++i) own[i] = 0;
    auto hand_over = [&] { // (whole numbers: any order)
#pragma unroll
        for (int i = 0; i < NC; ++i) {
            int n = (own[i / 4] >> (i % 4 * 8)) & 0xff;
            if (G == 1) n = __reduce_add_sync(0xffffffffu, n);
            if (n && (G > 1 || lane == 0)) atomicAdd(&cnt[column<T, G, NC, VEC>(i, t)], n);
        }
#pragma unroll
        for (int i = 0; i < NC / 4; ++i) own[i] = 0;
        since = 0;
    };
    // the teams of a warp take their turns together
    const int of_warp = blockIdx.x * TEAMS + (G < 32 ? warp * (32 / G) : warp);
    for (long long r0 = of_warp; r0 < rows; r0 += (long long)gridDim.x * TEAMS) {
        const long long r = r0 + lane / G;
        const bool live = r < rows && (!keep || keep[r]);
        float v[NC], u[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = -INFINITY;
        if (live) load_row<T, G, NC, VEC>(v, x + r * stride, t, experts);
#pragma unroll
        for (int i = 0; i < NC; ++i) u[i] = v[i];
        const float l = soft_max<G, NC>(v);
        if (l != 0.f) mine += t == 0; // (NaN is a row, too)
        if (l != l)
#pragma unroll
            for (int i = 0; i < NC; ++i) u[i] = u[i] != u[i] ? INFINITY : u[i];
#pragma unroll
        for (int i = 0; i < NC; ++i) acc[i] += l != 0.f ? v[i] : 0.f;
        if constexpr (SORT) choose_sorted<T, G, NC, VEC>(u, own, t, k);
        else choose_in_turn<T, G, NC, VEC>(u, own, t, k);
        if (++since == 255) hand_over();
    }
    hand_over();
    // probabilities: the teams of a warp, then the warps, each in order
#pragma unroll
    for (int i = 0; i < NC; ++i) {
#pragma unroll
        for (int o = 16; o >= G; o >>= 1) acc[i] += __shfl_xor_sync(0xffffffffu, acc[i], o);
        if (lane < G) psum[warp][column<T, G, NC, VEC>(i, t)] = acc[i];
    }
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) all[warp] = mine;
    __syncthreads();
    for (int e = threadIdx.x; e < experts; e += kThreads<NC>) {
        float p = 0.f;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) p += psum[w][e];
        sums[(long long)blockIdx.x * experts + e] = p;
        counts[(long long)blockIdx.x * experts + e] = cnt[e];
    }
    if (threadIdx.x == 0) {
        int m = 0;
        for (int w = 0; w < WARPS; ++w) m += all[w];
        kept[blockIdx.x] = m;
    }
}

// Adds up the blocks' sums: one block, or a cluster of blocks where there are many (what a single SM takes in would be the time).  `per` threads an expert and
// block, each its share of the sums in order, then a tree over the threads, then the cluster's blocks in order.
constexpr int kFinishBlocks = 8;
__global__ void __launch_bounds__(1024) balance_finish_kernel(const float *__restrict__ sums, const int *__restrict__ counts, const int *__restrict__ kept,
                                                              float *__restrict__ loss, int64_t *__restrict__ total, float *__restrict__ share, int blocks,
                                                              int experts, int per, int k)
{
    __shared__ double ps[1024];
    __shared__ long long cs[1024];
    __shared__ double red[4][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const cg::cluster_group cluster = cg::this_cluster();
    const int rank = blockIdx.x, ranks = gridDim.x; // one cluster
    // thread = part * experts + e: neighbours read neighbouring experts
    const int e = threadIdx.x % experts, part = threadIdx.x / experts;
    double p = 0.0;
    long long c = 0;
    if (part < per)
        for (int b = rank * per + part; b < blocks; b += ranks * per) p += sums[(long long)b * experts + e], c += counts[(long long)b * experts + e];
    ps[threadIdx.x] = p, cs[threadIdx.x] = c;
    double m = 0.0;
    if (rank == 0)
        for (int b = threadIdx.x; b < blocks; b += 1024) m += kept[b];
    __syncthreads();
    for (int n = per; n > 1; n = (n + 1) / 2) { // n parts: the upper ones are added to the lower ones
        if (part + (n + 1) / 2 < n) ps[threadIdx.x] += ps[threadIdx.x + (n + 1) / 2 * experts], cs[threadIdx.x] += cs[threadIdx.x + (n + 1) / 2 * experts];
        __syncthreads();
    }
    if (ranks > 1) {
        cluster.sync();
        if (rank > 0) {
            cluster.sync(); // its sums are read until here
            return;
        }
    }
    p = 0.0, c = 0;
    if (threadIdx.x < experts) p = ps[threadIdx.x], c = cs[threadIdx.x];
    if (threadIdx.x < experts)
        for (int i = 1; i < ranks; ++i) p += cluster.map_shared_rank(ps, i)[threadIdx.x], c += cluster.map_shared_rank(cs, i)[threadIdx.x];
    if (ranks > 1) cluster.sync();
    double v[4] = {(double)c * p, (double)c, m, p};
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (lane == 0)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[i][warp] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = red[i][lane];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    const double factor = v[2] > 0.0 ? experts / (v[2] * v[2] * k) : 0.0;
    if (threadIdx.x == 0) *loss = (float)(factor * v[0]);
    const double centre = v[3] > 0.0 ? v[0] / v[3] : v[1] / experts; // (the plain mean where a row holds NaN: it has no say in the others' gradients)
    if (threadIdx.x < experts) total[threadIdx.x] = c, share[threadIdx.x] = (float)(factor * ((double)c - centre));
}

template <typename T, int G, int NC, bool VEC>
__global__ void __launch_bounds__(kThreads<NC>, kResident<G, NC>) balance_bwd_kernel(const T *__restrict__ x, long long stride, const uint8_t *__restrict__ keep,
                                                               const float *__restrict__ share, const float *__restrict__ up, T *__restrict__ gx, int rows,
                                                               int experts)
{
    constexpr int TEAMS = kThreads<NC> / G, EV = kPiece<T>;
    const int t = threadIdx.x % G, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const float g = *up;
    float h[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) {
        const int e = column<T, G, NC, VEC>(i, t);
        h[i] = e < experts ? share[e] : 0.f;
    }
    const int of_warp = blockIdx.x * TEAMS + (G < 32 ? warp * (32 / G) : warp);
    for (long long r0 = of_warp; r0 < rows; r0 += (long long)gridDim.x * TEAMS) {
        const long long r = rows - 1 - (r0 + lane / G);
        const bool kept = r >= 0 && (!keep || keep[r]);
        float v[NC];
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = -INFINITY;
        if (kept) load_row<T, G, NC, VEC>(v, x + r * stride, t, experts);
        const bool there = soft_max<G, NC>(v) != 0.f && kept;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < NC; ++i) dot += v[i] * h[i];
        dot = lanes_sum<G>(dot);
#pragma unroll
        for (int i = 0; i < NC; ++i) v[i] = there ? g * (v[i] * (h[i] - dot)) : 0.f;
        if (r < 0) continue;
        T *out = gx + r * experts;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < NC / EV; ++i) {
                uint32_t w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float f[Word<T>::n];
#pragma unroll
                    for (int z = 0; z < Word<T>::n; ++z) f[z] = v[i * EV + j * Word<T>::n + z];
                    w[j] = Word<T>::put(f);
                }
                if ((i * G + t) * EV < experts) __stcs(reinterpret_cast<uint4 *>(out + (i * G + t) * EV), make_uint4(w[0], w[1], w[2], w[3]));
            }
        } else {
#pragma unroll
            for (int i = 0; i < NC; ++i)
                if (i * G + t < experts) out[i * G + t] = from_f<T>(v[i]);
        }
    }
}

// f(G, NC) for so many experts, as compile-time numbers: a thread a row up to 16, more lanes of 16 columns up to 512, then 32 columns
template <typename F> void with_team(int64_t experts, F &&f)
{
    using std::integral_constant;
    if (experts <= 8) f(integral_constant<int, 1>(), integral_constant<int, 8>());
    else if (experts <= 16) f(integral_constant<int, 1>(), integral_constant<int, 16>());
    else if (experts <= 32) f(integral_constant<int, 2>(), integral_constant<int, 16>());
    else if (experts <= 64) f(integral_constant<int, 4>(), integral_constant<int, 16>());
    else if (experts <= 128) f(integral_constant<int, 8>(), integral_constant<int, 16>());
    else if (experts <= 256) f(integral_constant<int, 16>(), integral_constant<int, 16>());
    else if (experts <= 512) f(integral_constant<int, 32>(), integral_constant<int, 16>());
    else f(integral_constant<int, 32>(), integral_constant<int, 32>());
}
// Blocks of the forward pass: those that are resident.  (Of 148 SMs: what the scratch is for.)  With the sums held to 512 KB, when one block finished them, most SMs were
// idle from 384 experts on, us, k = 8, forward and finish: 65536 rows of 384 132 + 11, now 75 + 13; of 1024 919 + 11, now 228 + 21; 4096 of 1024 58 + 11, now 22 + 20.
int balance_blocks(int64_t rows, int64_t experts)
{
    int64_t n = 0;
    with_team(experts, [&](auto G, auto NC) {
        const int64_t teams = kThreads<decltype(NC)::value> / decltype(G)::value;
        n = std::min<int64_t>((rows + teams - 1) / teams, 148 * kResident<decltype(G)::value, decltype(NC)::value>);
    });
    return (int)n;
}
template <typename T> bool whole_pieces(const void *x, int64_t stride, int64_t experts)
{
    return experts % kPiece<T> == 0 && stride % kPiece<T> == 0 && (reinterpret_cast<uintptr_t>(x) & 15) == 0;
}

} // namespace

extern "C" size_t clb_balance_scratch_bytes(int64_t rows, int64_t experts)
{
    if (rows <= 0 || experts <= 0 || experts > CLB_BALANCE_MAX_EXPERTS) return 0;
    return (size_t)balance_blocks(rows, experts) * (size_t)(8 * experts + 4);
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
    const int blocks = rows > 0 ? balance_blocks(rows, experts) : 0;
    float *sums = (float *)scratch;
    int *cnt = (int *)(sums + (long long)blocks * experts), *kept = cnt + (long long)blocks * experts;
    if (rows > 0)
        with_score_type(dtype, [&](auto t) {
            using T = decltype(t);
            with_team(experts, [&](auto G, auto NC) {
                constexpr int LANES = decltype(G)::value, COLUMNS = decltype(NC)::value;
                auto go = [&](auto vec, auto sort) {
                    constexpr bool VEC = decltype(vec)::value, SORT = decltype(sort)::value;
                    CLB_TRACED("balance_fwd_kernel", st,
                               balance_fwd_kernel<T, LANES, COLUMNS, VEC, SORT><<<blocks, kThreads<COLUMNS>, 0, st>>>(
                                   (const T *)x, row_stride, keep, sums, cnt, kept, (int)rows, (int)experts, k));
                };
                auto chosen = [&](auto sort) {
                    if (whole_pieces<T>(x, row_stride, experts)) go(std::true_type(), sort);
                    else go(std::false_type(), sort);
                };
                if constexpr (COLUMNS == 16) {
                    // in turn / sorted, 16 million logits: k = 2 30 / 43 us (16 experts), 31 / 38 (128); k = 4 40 / 42, 44 / 41; k = 8 62 / 42, 71 / 48
                    if (k >= (LANES == 1 ? 5 : 4)) return chosen(std::true_type());
                }
                chosen(std::false_type());
            });
        });
    const int ranks = blocks * experts > 32768 ? kFinishBlocks : 1; // one / eight, us: 592 sums of 30 experts 7 / 8, 444 of 60 9 / 7, 256 of 256 12 / 8
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks), cfg.blockDim = dim3(1024), cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)ranks, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    CLB_TRACED("balance_finish_kernel", st, cudaLaunchKernelEx(&cfg, balance_finish_kernel, (const float *)sums, (const int *)cnt, (const int *)kept, loss, counts,
                                                               share, blocks, (int)experts, (int)(1024 / experts), k));
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
        with_team(experts, [&](auto G, auto NC) {
            constexpr int LANES = decltype(G)::value;
            const int64_t teams = kThreads<decltype(NC)::value> / LANES;
            const int blocks = (int)std::min<int64_t>((rows + teams - 1) / teams, kResident<LANES, decltype(NC)::value> * (int64_t)sm_count());
            auto go = [&](auto vec) {
                constexpr bool VEC = decltype(vec)::value;
                CLB_TRACED("balance_bwd_kernel", st,
                           balance_bwd_kernel<T, LANES, decltype(NC)::value, VEC><<<blocks, kThreads<decltype(NC)::value>, 0, st>>>((const T *)x, row_stride, keep, share, upstream,
                                                                                                             (T *)grad, (int)rows, (int)experts));
            };
            if (whole_pieces<T>(x, row_stride, experts) && (reinterpret_cast<uintptr_t>(grad) & 15) == 0) go(std::true_type());
            else go(std::false_type());
        });
    });
    return check_launch();
}

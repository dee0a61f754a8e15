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
// classes are struck out there: a bit per value in shared memory, set by the threads that hold the list.  Many rows that are longer than a block's registers go
// through a block twice (distill_stream_kernel).  With the gradient: 8192 rows of 1000 fp32 22 us (3.0 TB/s; bound by issue, the list costs a warp as much as its
// row), 2048 of 131072 bf16 243 us (4.4 TB/s; reading, reading again from the L2 and writing alone take 203).
#include <cooperative_groups.h>

#include "clb_rows.cuh"

using namespace clb;
using namespace clb_host;

namespace {

struct DistillArgs {
    long long stride, rows;
    int classes, k;
    float temperature, c, scale; // c = log2(e) / T; scale: T, over the rows for a mean
    float inv, inv_low;          // 1 / T in two parts
    int chunks, ranks_log;       // forward: how often a cluster comes back for more of a row; its blocks
};

struct Entry { // one class of a list: cls < 0: does not exist
    int cls;
    float t, s;
};

// What a teacher's list comes to.  Everything is taken with respect to its largest value m: values far from zero (counts in the thousands) lose nothing but what
// their own rounding lost.  p of value t is exp(log_p(t)).
struct TeacherNumbers {
    float m, ref, tl; // its mass is tl * exp(m / T + ref)
    float d;          // log of the rest's mass, less m / T
    float rest;       // probability of the rest
    float listed;     // and of all that is listed
    float factor;     // of the row's loss / T and gradient; 0: the row adds nothing
    __device__ __forceinline__ float log_p(float t, float tt, float log_tl) const { return ((t - m) / tt - ref) - log_tl; }
};
__device__ __forceinline__ TeacherNumbers teacher_numbers(ExpSum teach, float rs, float w, const DistillArgs &a)
{
    TeacherNumbers q;
    const bool none = teach.m == -INFINITY;
    q.m = finite_or_zero(teach.m);
    if (fabsf(rs) < INFINITY) { // m / T by a reciprocal in two parts: rounded, it would be off by 2^-24 of itself
        const float of_m = __fmul_rn(q.m, a.inv); // (not to become part of the difference, which takes what it is rounded by on its own)
        q.d = fabsf(of_m) < INFINITY ? fminf((rs - of_m) - fmaf(q.m, a.inv, -of_m) - q.m * a.inv_low, 3.402823466e38f) : copysignf(3.402823466e38f, -of_m);
    } else
        q.d = rs == -INFINITY ? rs : rs - rs;
    q.ref = finite_or_zero(fmaxf(none ? -INFINITY : 0.f, q.d));
    const float re = ex2((q.d - q.ref) * 1.44269504f);
    const float all = none ? teach.l : teach.l * ex2(-q.ref * 1.44269504f);
    q.tl = all + re;
    q.rest = __fdividef(re, q.tl), q.listed = __fdividef(all, q.tl);
    q.factor = q.tl != 0.f ? w * a.scale : 0.f;
    return q;
}
// A class's share of the loss, p log(p / q) - p + q with delta = log(p / q): what is added to p log(p / q) comes to nothing over all classes, but for what the logarithms
// of the sums are off, and takes the cancellation out: no share is below 0, and an error of a logarithm counts with p - q, not with p.  (A list that holds little of
// the mass, or a student near its teacher: losses of 1e-4 were 1e-2 off.)
__device__ __forceinline__ float share_of(float p, float delta, float q)
{
    if (p == 0.f) return q;
    if (!(fabsf(delta) < 0.25f)) return p * (delta - 1.f) + q;
    const float d = delta; // exp(-d) - 1 + d, Taylor's to d^7: the next term is 2e-8 of the first
    float f = fmaf(d, -1.f / 5040, 1.f / 720);
    f = fmaf(d, f, -1.f / 120), f = fmaf(d, f, 1.f / 24), f = fmaf(d, f, -1.f / 6), f = fmaf(d, f, 0.5f);
    return p * (d * d) * f;
}
// What a row's sums come to: unlisted scores `rest`, distinct listed ones `list`.
struct RowNumbers {
    float m, l, coef;  // of the unlisted scores: reference and sum; gradient = coef * exp((s - m) / T).  The list's = factor * (q - p)
    float um, ul;      // of all scores; ul = 0: there are none
    float qr;          // probability of the unlisted ones
    __device__ __forceinline__ float rest_share(const TeacherNumbers &q, float tt, float log_tl, float log_ul) const // of the row's loss / (factor * T)
    {
        const float log_qr = l == 0.f ? -INFINITY : ((m - um) / tt + logf(l)) - log_ul;
        return share_of(q.rest, ((q.d - q.ref) - log_tl) - log_qr, qr);
    }
};
__device__ __forceinline__ RowNumbers row_numbers(ExpSum rest, ExpSum list, const TeacherNumbers &q, const DistillArgs &a)
{
    RowNumbers n; // (a sum of 0 has no terms: the largest adds 1)
    n.m = finite_or_zero(rest.m), n.um = finite_or_zero(fmaxf(rest.m, list.m)), n.l = rest.l;
    const float of_rest = rest.l == 0.f ? 0.f : rest.l * exp_of(n.m, n.um, a.c);
    const float of_list = list.l == 0.f ? 0.f : list.l * exp_of(finite_or_zero(list.m), n.um, a.c);
    n.ul = of_rest + of_list;
    n.qr = __fdividef(of_rest, n.ul);
    // q_r - r, or the same by what is listed where that is less: two numbers near one leave 2^-24 of one
    const float more = n.qr + q.rest > 1.f ? q.listed - __fdividef(of_list, n.ul) : n.qr - q.rest;
    n.coef = q.factor == 0.f || rest.l == 0.f ? 0.f : q.factor * __fdividef(more, rest.l);
    return n;
}

constexpr int kValues = 64; // of a row in a thread's registers, as fp32

// TH threads a row (4 to 32: teams of a block of 256; more: the block), NV pieces a thread.  CLUSTER: the blocks of a cluster share a row.
// grad: where d loss / d scores goes for an upstream gradient of one, or NULL.
//
// A thread takes the exponentials of its values with respect to its own maximum and keeps them, so that there is one exchange in the team, of pairs (maximum,
// sum), and the gradient is the kept exponential times a factor of the thread's: one exponential a value.
template <typename T, int TH, int NV, bool CLUSTER>
__global__ void __launch_bounds__(TH <= 32 ? 256 : TH, TH > 32 ? 512 / TH : NV * kPiece<T> > 32 ? 2 : 4)
    distill_fwd_kernel(const T *__restrict__ x, const float *__restrict__ values, const int64_t *__restrict__ indices, const float *__restrict__ rest,
                       const float *__restrict__ weight, float *__restrict__ row_loss, float *__restrict__ stats, float *__restrict__ listed, T *grad, DistillArgs a)
{
    namespace cg = cooperative_groups;
    constexpr int BLOCK = TH <= 32 ? 256 : TH, TEAMS = BLOCK / TH, EV = kPiece<T>, LANES = TH < 32 ? TH : 32, WARPS = TH / LANES, RANKS = CLUSTER ? 8 : 1, WORDS = NV * EV <= 32 ? 1 : 2;
    static_assert(NV * EV <= kValues, "a bit for each value");
    __shared__ uint32_t bits[WORDS][BLOCK];
    __shared__ int4 classes[TEAMS][CLB_TOP_MAX / 4]; // of the list, -1 behind its end
    __shared__ ExpSum part[2][RANKS * WARPS]; // of the unlisted scores, for even and odd turns: each warp of each block of the cluster
    __shared__ float4 list_part[4];           // of the list: maximum and sum of its scores, of the teacher's values
    __shared__ float loss_part[4];
    const int t = threadIdx.x % TH, team = threadIdx.x / TH, lane = threadIdx.x & 31, warp = t / 32;
    const int ranks = CLUSTER ? 1 << a.ranks_log : 1, rank = CLUSTER ? blockIdx.x & (ranks - 1) : 0;
    const int list_warps = TH > 32 ? (a.k + 31) / 32 : 1;
    const int groups = (int)(gridDim.x >> (CLUSTER ? a.ranks_log : 0)) * TEAMS;
    auto team_sync = [] {
        if (TH <= 32) __syncwarp();
        else __syncthreads();
    };
    if (CLUSTER) { // no block writes to another's memory before that one runs and has cleared what a cluster of fewer blocks does not write
        for (int i = threadIdx.x; i < 2 * RANKS * WARPS; i += BLOCK) part[0][i] = ExpSum{-INFINITY, 0.f};
        cg::this_cluster().sync();
    }
    // (the teams of a warp take every turn together, on the last row again where one has none left)
    const long long first_row = (long long)(blockIdx.x >> (CLUSTER ? a.ranks_log : 0)) * TEAMS;
    const int of_warp = TH < 32 ? team & ~(32 / TH - 1) : team;
    int turn = 0;
    for (long long r_warp = first_row + of_warp; r_warp < a.rows; r_warp += groups, ++turn) {
        const bool live = TH >= 32 || r_warp + (team - of_warp) < a.rows;
        const long long r = live ? r_warp + (team - of_warp) : a.rows - 1;
        const RowPieces<T> row(x + r * a.stride, a.classes);
        const int64_t *idx = indices + r * a.k;
        const float *val = values + r * a.k;
        const int chunks = CLUSTER ? a.chunks : 1; // (one unless the row is longer than the cluster's registers)
        auto class_of = [&](int n) {
            const long long j = idx[n];
            return j >= 0 && j < a.classes ? (int)j : -1;
        };
        // (what lies elsewhere is asked for before the row)
        const float w = weight ? weight[r] : 1.f, rs = rest ? rest[r] : -INFINITY, tt = a.temperature;
        Entry own{-1, -INFINITY, -INFINITY};
        if (t < a.k) own.cls = class_of(t), own.t = val[t];
        int *const list = reinterpret_cast<int *>(classes[team]);
        auto entry = [&](int n) { // of the threads that hold the list, t + TH * i
            if (n == t) return own;
            Entry e{list[n], -INFINITY, -INFINITY};
            if (e.cls >= 0) e.t = val[n], e.s = to_f(row.row[e.cls]);
            return e;
        };
        float v[NV * EV]; // the thread's values, later their exponentials
        auto fetch = [&](int chunk) {
            const int base = (chunk * ranks + rank) * TH * NV;
            uint4 raw[NV];
            row.load(raw, base + t, TH);
#pragma unroll
            for (int i = 0; i < WORDS; ++i) bits[i][threadIdx.x] = 0;
            team_sync();
            for (int n = t; n < ((a.k + 3) & ~3); n += TH) { // the listed classes are struck out where they lie
                const int cls = n == t ? own.cls : n < a.k ? class_of(n) : -1;
                if (chunk == 0) list[n] = cls;
                const int j = cls < 0 ? -1 : row.piece_of(cls) - base;
                if (j < 0 || j >= TH * NV) continue;
                const int bit = j / TH * EV + row.place_of(cls);
                atomicOr(&bits[bit >> 5][team * TH + j % TH], 1u << (bit & 31));
            }
            if (chunk == 0 && own.cls >= 0) own.s = to_f(row.row[own.cls]);
            team_sync();
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    float f[Word<T>::n];
                    Word<T>::get(w[q], f);
#pragma unroll
                    for (int z = 0; z < Word<T>::n; ++z) v[i * EV + q * Word<T>::n + z] = f[z];
                }
            }
#pragma unroll
            for (int half = 0; half < WORDS; ++half)
                if (const uint32_t m = bits[half][threadIdx.x])
#pragma unroll
                    for (int i = half * 32; i < (half + 1) * 32 && i < NV * EV; ++i)
                        if ((m >> (i & 31)) & 1) v[i] = -INFINITY;
        };
        auto exponentials = [&](float m) { // v = exp of v with respect to m; their sum
            float l = 0.f;
#pragma unroll
            for (int i = 0; i < NV * EV; ++i) {
                v[i] = exp_of(v[i], m, a.c);
                l += v[i];
            }
            return l;
        };
        ExpSum mine{-INFINITY, 0.f};
        for (int ch = 0; ch < chunks; ++ch) {
            fetch(ch);
            float m = v[0];
#pragma unroll
            for (int i = 1; i < NV * EV; ++i) m = fmaxf(m, v[i]);
            m = fmaxf(m, -INFINITY); // (NaN alone)
            const float l = exponentials(finite_or_zero(m));
            if (chunks == 1) mine = {m, l};
            else mine = merge(mine, ExpSum{m, l}, a.c);
        }
        if (own.cls < 0) own.t = -INFINITY;
        // ---- the list: distinct classes' scores, the teacher's values
        float4 sums = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
        uint32_t firsts = 0, twins = 0; // bit i: entry t + TH * i is the first of its class; its class is listed twice
        auto compare = [&](int n, int cls) {
            int before = 0, same = 0;
            for (int o = 0; o < a.k; o += 4) {
                const int4 q = classes[team][o / 4];
                const int hits = (q.x == cls) + (q.y == cls) + (q.z == cls) + (q.w == cls);
                same += hits;
                before += o + 4 <= n ? hits : (q.x == cls && o < n) + (q.y == cls && o + 1 < n) + (q.z == cls && o + 2 < n);
            }
            firsts |= (uint32_t)(before == 0) << (n / TH), twins |= (uint32_t)(same > 1) << (n / TH);
        };
        if (TH <= 32 || warp < list_warps) {
            for (int n = t; n < a.k; n += TH) {
                const Entry e = entry(n);
                sums.x = fmaxf(sums.x, e.s), sums.z = fmaxf(sums.z, e.t);
            }
            sums.x = lanes_max<LANES>(sums.x), sums.z = lanes_max<LANES>(sums.z);
            for (int n = t; n < a.k; n += TH) {
                const Entry e = entry(n);
                if (e.cls < 0) continue;
                compare(n, e.cls);
                if ((firsts >> (n / TH)) & 1) sums.y += exp_of(e.s, finite_or_zero(sums.x), a.c);
                sums.w += exp_of(e.t, finite_or_zero(sums.z), a.c);
            }
            sums.y = lanes_sum<LANES>(sums.y), sums.w = lanes_sum<LANES>(sums.w);
        }
        // ---- the team's
        const float own_max = mine.m;
        mine = lanes_merge<LANES>(mine, a.c);
        if (TH > 32) {
            if (warp < list_warps && lane == 0) list_part[warp] = sums;
            ExpSum *parts = part[turn & 1];
            if (CLUSTER) {
                if (lane < ranks) cg::this_cluster().map_shared_rank(parts, lane)[rank * WARPS + warp] = mine;
                cg::this_cluster().sync();
            } else {
                if (lane == 0) parts[warp] = mine;
                __syncthreads();
            }
            constexpr int N = RANKS * WARPS;
            mine = parts[lane % N];
#pragma unroll
            for (int i = 32; i < N; i += 32) mine = merge(mine, parts[lane + i], a.c);
            mine = lanes_merge<(N < 32 ? N : 32)>(mine, a.c);
            ExpSum s{list_part[0].x, list_part[0].y}, u{list_part[0].z, list_part[0].w};
            for (int i = 1; i < list_warps; ++i) {
                s = merge(s, ExpSum{list_part[i].x, list_part[i].y}, a.c);
                u = merge(u, ExpSum{list_part[i].z, list_part[i].w}, a.c);
            }
            sums = make_float4(s.m, s.l, u.m, u.l);
        }
        const TeacherNumbers teach = teacher_numbers(ExpSum{sums.z, sums.w}, rs, w, a);
        const RowNumbers num = row_numbers(mine, ExpSum{sums.x, sums.y}, teach, a);
        const float m = num.m, coef = num.coef;
        const bool there = teach.factor != 0.f && num.ul != 0.f;
        T *out = grad ? grad + r * a.classes : nullptr;
        if (grad) {
            const bool aligned = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
            for (int ch = 0; ch < chunks; ++ch) {
                float scale = coef;
                if (chunks == 1) scale = coef == 0.f ? 0.f : coef * exp_of(own_max, m, a.c);
                else {
                    fetch(ch);
                    exponentials(m);
                }
                if (coef == 0.f) // (a row that adds nothing may hold NaN and infinities)
#pragma unroll
                    for (int i = 0; i < NV * EV; ++i) v[i] = 0.f;
                const int base = (ch * ranks + rank) * TH * NV;
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    const int j = base + i * TH + t;
                    uint32_t o[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float f[Word<T>::n];
#pragma unroll
                        for (int z = 0; z < Word<T>::n; ++z) f[z] = scale * v[i * EV + q * Word<T>::n + z];
                        o[q] = Word<T>::put(f);
                    }
                    if (j < row.pieces && live) row.store(out, aligned, j, make_uint4(o[0], o[1], o[2], o[3]));
                }
            }
        }
        // ---- the list again: its loss, and the gradient of its classes
        float loss = 0.f, own_grad = 0.f;
        float log_tl = 0.f, log_ul = 0.f;
        if (TH <= 32 || warp < list_warps) log_tl = logf(teach.tl), log_ul = logf(num.ul);
        auto gradient_of = [&](int n, const Entry &e) {
            if (!there || e.cls < 0) return 0.f;
            const float lp = teach.log_p(e.t, tt, log_tl), lq = (e.s - num.um) / tt - log_ul, p = expf(lp), q = expf(lq);
            float mass = p;
            if ((twins >> (n / TH)) & 1) { // a class that is listed twice has both entries' probability
                mass = 0.f;
                for (int o = 0; o < a.k; ++o)
                    if (list[o] == e.cls) mass += expf(teach.log_p(val[o], tt, log_tl));
                loss += (p == 0.f ? 0.f : p * (lp - lq - 1.f)) + ((firsts >> (n / TH)) & 1 ? q : 0.f);
            } else
                loss += share_of(p, lp - lq, q);
            return teach.factor * (q - mass);
        };
        if (TH > 32) {
            if (warp < list_warps) {
                if (t < a.k) own_grad = gradient_of(t, own);
                loss = lanes_sum<32>(loss);
                if (lane == 0) loss_part[warp] = loss;
            }
            __syncthreads(); // a listed class is written after the piece that it lies in
        } else
            __syncwarp();
        for (int n = t; n < a.k; n += TH) {
            const Entry e = entry(n);
            const float g = TH > 32 ? own_grad : gradient_of(n, e);
            if (rank == 0 && live) listed[r * a.k + n] = g;
            if (grad && live && e.cls >= 0 && (!CLUSTER || ((row.piece_of(e.cls) / (TH * NV)) & (ranks - 1)) == rank)) out[e.cls] = from_f<T>(g);
        }
        if (TH <= 32) loss = lanes_sum<LANES>(loss);
        if (t == 0 && rank == 0 && live) {
            if (TH > 32) {
                loss = 0.f;
                for (int i = 0; i < list_warps; ++i) loss += loss_part[i];
            }
            row_loss[r] = there ? (loss + num.rest_share(teach, tt, log_tl, log_ul)) * teach.factor * tt : 0.f;
            stats[2 * r] = m, stats[2 * r + 1] = coef;
        }
        team_sync(); // the tables are used again
    }
}

constexpr int kTripPieces = 8; // of a thread

// Rows that are longer than a block's registers, many of them: a block a row, twice, the second time for the gradient, backwards and from the L2 (which is why
// no more rows are in flight than fit there).  The last warp does what a row's list asks for while the others read or write: its sums before the barrier
// between the passes; loss, gradients and the next row's bits before the one behind them.  The bit of a listed class is in a table of the whole row, one for
// rows of even and one for rows of odd number; a thread's values of a trip have 32 neighbouring bits, or two words.
template <typename T, int TH>
__global__ void __launch_bounds__(TH, 1024 / TH)
    distill_stream_kernel(const T *__restrict__ x, const float *__restrict__ values, const int64_t *__restrict__ indices, const float *__restrict__ rest,
                          const float *__restrict__ weight, float *__restrict__ row_loss, float *__restrict__ stats, float *__restrict__ listed, T *grad,
                          DistillArgs a)
{
    constexpr int MT = TH - 32, NV = kTripPieces, EV = kPiece<T>, WORDS = NV * EV / 32, EACH = CLB_TOP_MAX / 32;
    extern __shared__ uint32_t tables[]; // [2][trips][WORDS][MT]
    const int words = a.chunks * WORDS * MT;
    __shared__ ExpSum part[32];
    __shared__ float4 from_list; // maximum and sum of the distinct listed scores, the teacher's probability of the rest, the gradient's factor
    __shared__ float p_listed;   // the teacher's probability of all listed classes
    __shared__ int list[CLB_TOP_MAX];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const float tt = a.temperature;
    for (int i = t; i < 2 * words; i += TH) tables[i] = 0;
    if (t < 32) part[t] = ExpSum{-INFINITY, 0.f};
    __syncthreads();
    if (warp == MT / 32) { // ---------------- the list
        // Two rows ahead: classes and values are asked for; one ahead: their scores, and they are marked.  Each has a row's time to arrive.
        struct {
            int cls[EACH];
            float t[EACH], s[EACH], w, rest;
        } now, next;
        long long ahead_cls[EACH];
        float ahead_t[EACH], ahead_w = 1.f, ahead_rest = -INFINITY, g[EACH];
        auto ask = [&](long long r) {
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const int n = lane + 32 * i;
                const bool there = r < a.rows && n < a.k;
                ahead_cls[i] = there ? indices[r * a.k + n] : -1;
                ahead_t[i] = there ? values[r * a.k + n] : -INFINITY;
            }
            if (r < a.rows && weight) ahead_w = weight[r];
            if (r < a.rows && rest) ahead_rest = rest[r];
        };
        auto take = [&](long long r) { // what was asked for becomes the next row
            next.w = ahead_w, next.rest = ahead_rest;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                const bool there = ahead_cls[i] >= 0 && ahead_cls[i] < a.classes;
                next.cls[i] = there ? (int)ahead_cls[i] : -1, next.t[i] = there ? ahead_t[i] : -INFINITY;
                next.s[i] = there ? to_f(x[r * a.stride + next.cls[i]]) : -INFINITY;
            }
        };
        auto place = [&](const T *row, int c) { // bit of a class in a table
            const int v = c + (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)), j = v / EV;
            const int bit = j / MT % NV * EV + v % EV;
            return (((j / (MT * NV)) * WORDS + (bit >> 5)) * MT + j % MT) * 32 + (bit & 31);
        };
        auto mark = [&](long long r, uint32_t *table) { // the next row's classes; is one listed twice?
            bool twice = false;
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                if (next.cls[i] >= 0) {
                    const int at = place(x + r * a.stride, next.cls[i]);
                    const uint32_t before = atomicOr(&table[at >> 5], 1u << (at & 31));
                    twice = twice || ((before >> (at & 31)) & 1);
                }
            return (bool)__any_sync(0xffffffffu, twice);
        };
        ask(blockIdx.x);
        take(blockIdx.x);
        ask((long long)blockIdx.x + gridDim.x);
        bool dup = false, next_dup = mark(blockIdx.x, tables);
        int odd = 0;
        __syncthreads();
        for (long long r = blockIdx.x; r < a.rows; r += gridDim.x, odd ^= 1) {
            const T *row = x + r * a.stride;
            now = next, dup = next_dup;
            int(&cls)[EACH] = now.cls;
            float(&tv)[EACH] = now.t;
            float(&sv)[EACH] = now.s;
            const float w = now.w, rs = now.rest;
            take(r + gridDim.x);
            ask(r + 2 * (long long)gridDim.x);
            if (dup) { // (rare)
                __syncwarp();
#pragma unroll
                for (int i = 0; i < EACH; ++i) list[lane + 32 * i] = cls[i];
                __syncwarp();
            }
            ExpSum sk{-INFINITY, 0.f}, tk{-INFINITY, 0.f};
#pragma unroll
            for (int i = 0; i < EACH; ++i) sk.m = fmaxf(sk.m, sv[i]), tk.m = fmaxf(tk.m, tv[i]);
            sk.m = lanes_max<32>(sk.m), tk.m = lanes_max<32>(tk.m);
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                if (cls[i] < 0) continue;
                bool first = true;
                if (dup)
                    for (int o = 0; o < lane + 32 * i; ++o) first = first && list[o] != cls[i];
                if (first) sk.l += exp_of(sv[i], finite_or_zero(sk.m), a.c);
                tk.l += exp_of(tv[i], finite_or_zero(tk.m), a.c);
            }
            sk.l = lanes_sum<32>(sk.l), tk.l = lanes_sum<32>(tk.l);
            const TeacherNumbers q = teacher_numbers(tk, rs, w, a);
            if (lane == 0) from_list = make_float4(sk.m, sk.l, q.rest, q.factor), p_listed = q.listed;
            __syncthreads(); // ------------ all sums are there
            const RowNumbers n = row_numbers(lanes_merge<32>(part[lane], a.c), sk, q, a);
            const bool there = q.factor != 0.f && n.ul != 0.f;
            const float log_tl = logf(q.tl), log_ul = logf(n.ul);
            float loss = n.rest_share(q, tt, log_tl, log_ul); // (beside the list's terms, not behind their sum)
            loss = lane == 0 ? loss : 0.f;
#pragma unroll
            for (int i = 0; i < EACH; ++i) {
                g[i] = 0.f;
                if (there && cls[i] >= 0) {
                    const float lp = q.log_p(tv[i], tt, log_tl), lq = (sv[i] - n.um) / tt - log_ul, p = expf(lp), qk = expf(lq);
                    float mass = p;
                    if (dup) { // a class that is listed twice has both entries' probability
                        mass = 0.f;
                        bool first = true;
                        for (int o = 0; o < a.k; ++o)
                            if (list[o] == cls[i]) mass += expf(q.log_p(values[r * a.k + o], tt, log_tl)), first = first && o >= lane + 32 * i;
                        loss += (p == 0.f ? 0.f : p * (lp - lq - 1.f)) + (first ? qk : 0.f);
                    } else
                        loss += share_of(p, lp - lq, qk);
                    g[i] = q.factor * (qk - mass);
                }
                if (lane + 32 * i < a.k) listed[r * a.k + lane + 32 * i] = g[i];
            }
            loss = lanes_sum<32>(loss);
            if (lane == 0) {
                row_loss[r] = there ? loss * q.factor * tt : 0.f;
                stats[2 * r] = n.m, stats[2 * r + 1] = n.coef;
            }
            next_dup = mark(r + gridDim.x, tables + (odd ^ 1) * words);
            __syncthreads(); // ------------ the row is written, the next one is marked
            T *out = grad ? grad + r * a.classes : nullptr;
#pragma unroll
            for (int i = 0; i < EACH; ++i)
                if (cls[i] >= 0) {
                    if (grad) out[cls[i]] = from_f<T>(g[i]);
                    const int at = place(row, cls[i]);
                    atomicAnd(&tables[odd * words + (at >> 5)], ~(1u << (at & 31)));
                }
        }
        return;
    }
    // -------------------------------------------- the row
    int odd = 0;
    uint4 raw[NV];
    if (blockIdx.x < a.rows) RowPieces<T>(x + blockIdx.x * a.stride, a.classes).template load<NV, false>(raw, t, MT);
    __syncthreads();
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x, odd ^= 1) {
        const RowPieces<T> row(x + r * a.stride, a.classes);
        const uint32_t *const table = tables + odd * words;
        auto strike = [&](int trip) {
#pragma unroll
            for (int h = 0; h < WORDS; ++h) strike_out<T>(raw + h * (NV / WORDS), table[(trip * WORDS + h) * MT + t], NV / WORDS);
        };
        ExpSum mine{-INFINITY, 0.f};
        for (int trip = 0; trip < a.chunks; ++trip) {
            if (trip > 0) row.template load<NV, false>(raw, trip * MT * NV + t, MT);
            strike(trip);
            uint32_t top = low_word<T>();
#pragma unroll
            for (int i = 0; i < NV; ++i) top = piece_max<T>(top, raw[i]);
            const float m = fmaxf(mine.m, word_max<T>(top)), ref = finite_or_zero(m);
            const float before = mine.l * exp_of(mine.m, ref, a.c);
            const ExpRef er = exp_ref(ref, a.c);
            float sum = 0.f;
            if (!er.far) {
                Pair l[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
#pragma unroll
                for (int i = 0; i < NV; ++i) piece_exp_sum<T>(l, raw[i], pair_of(-er.R, -er.R), pair_of(a.c, a.c));
                float even, rest_of;
                split(l[0] + l[1], even, rest_of);
                sum = (even + rest_of) * er.fix;
            } else {
#pragma unroll 1
                for (int i = 0; i < NV; ++i) {
                    const uint4 p = raw[0];
#pragma unroll
                    for (int n = 1; n < NV; ++n) raw[n - 1] = raw[n];
                    raw[NV - 1] = p; // (a rotation: no register is named by a number that varies)
                    const uint32_t o[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        float f[Word<T>::n];
                        Word<T>::get(o[q], f);
#pragma unroll
                        for (int z = 0; z < Word<T>::n; ++z) sum += exp_of(f[z], ref, a.c);
                    }
                }
            }
            mine = {m, before + sum};
        }
        mine = lanes_merge<32>(mine, a.c);
        if (lane == 0) part[warp] = mine;
        __syncthreads(); // ---------------- all sums are there
        if (grad) {
            const float4 l = from_list;
            TeacherNumbers q;
            q.rest = l.z, q.factor = l.w, q.listed = p_listed;
            const RowNumbers n = row_numbers(lanes_merge<32>(part[lane], a.c), ExpSum{l.x, l.y}, q, a);
            T *out = grad + r * a.classes;
            const bool aligned = ((reinterpret_cast<uintptr_t>(out) ^ reinterpret_cast<uintptr_t>(row.row)) & 15) == 0;
            RowTrips<T, MT, NV> to(out, a.classes);
            if (!aligned) to.hi = 0;
            const ExpRef er = exp_ref(n.m, a.c);
            const Pair c2 = pair_of(a.c, a.c), minus_R = pair_of(-er.R, -er.R), fixed = pair_of(n.coef * er.fix, n.coef * er.fix);
            for (int trip = a.chunks - 1; trip >= 0; --trip) {
                if (trip < a.chunks - 1) {
                    row.load(raw, trip * MT * NV + t, MT);
                    strike(trip);
                }
                auto gradients = [&](auto of_pair) {
#pragma unroll
                    for (int q = 0; q < NV; ++q) {
                        Pair v[kPairs<T>];
                        piece_pairs<T>(raw[q], v);
#pragma unroll
                        for (int z = 0; z < kPairs<T>; ++z) v[z] = of_pair(v[z]);
                        raw[q] = pairs_piece<T>(v);
                    }
                };
                if (n.coef == 0.f) gradients([](Pair) { return pair_of(0.f, 0.f); }); // (a row that adds nothing may hold NaN)
                else if (!er.far) gradients([&](Pair v) { return fixed * ex2(fma2(v, c2, minus_R)); });
                else gradients([&](Pair v) { return pair_of(n.coef, n.coef) * ex2((v + pair_of(-n.m, -n.m)) * c2); });
                if (to.whole(trip)) {
                    char *o = const_cast<char *>(to.at(trip));
#pragma unroll
                    for (int q = 0; q < NV; ++q) __stcs(reinterpret_cast<uint4 *>(o + q * MT * 16), raw[q]);
                } else {
                    const int base = trip * MT * NV + t;
#pragma unroll
                    for (int q = 0; q < NV; ++q)
                        if (base + q * MT < row.pieces) row.store(out, aligned, base + q * MT, raw[q]);
                }
            }
        }
        if (r + gridDim.x < a.rows) RowPieces<T>(x + (r + gridDim.x) * a.stride, a.classes).template load<NV, false>(raw, t, MT);
        __syncthreads(); // ---------------- the row is written, the next one is marked
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
        row.load(raw, base + t, TH);
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

// Sums of `n` numbers in a fixed order: block b those of its part, in 64 bits.  One block up to 2^18 rows (65536: 3 us), else 128 and then one over theirs.
constexpr int kSumParts = 128;
constexpr long long kOneSum = 1 << 18;
template <typename In, typename Out> __global__ void __launch_bounds__(1024) distill_sum_kernel(const In *__restrict__ in, Out *__restrict__ out, long long n)
{
    __shared__ double red[32];
    const long long lo = n * blockIdx.x / gridDim.x, hi = n * (blockIdx.x + 1) / gridDim.x;
    double mine = 0.0;
    for (long long r = lo + threadIdx.x; r < hi; r += 16 * 1024) {
        In v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = r + i * 1024 < hi ? in[r + i * 1024] : In(0);
#pragma unroll
        for (int i = 0; i < 16; ++i) mine += v[i];
    }
    mine = warp_sum<double>(mine);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = mine;
    __syncthreads();
    if (threadIdx.x < 32) {
        mine = warp_sum<double>(red[threadIdx.x]);
        if (threadIdx.x == 0) out[blockIdx.x] = (Out)mine;
    }
}
size_t sums_at(int64_t rows) { return (size_t)((rows * 4 + 7) & ~7ll); } // of the parts' sums, behind the rows' losses

bool sizes_ok(int64_t rows, int64_t classes, int64_t row_stride, int k, double temperature, int dtype)
{
    return rows >= 0 && classes > 0 && row_stride >= 0 && k > 0 && temperature >= 1e-30 && temperature <= 1e30 &&
           (dtype == CLB_F32 || dtype == CLB_F16 || dtype == CLB_BF16);
}
DistillArgs make_args(int64_t rows, int64_t classes, int64_t row_stride, int k, double temperature, int reduction)
{
    const float inv = (float)(1.0 / temperature);
    return {row_stride, rows, (int)classes, k, (float)temperature, (float)(1.4426950408889634 / temperature),
            (float)(reduction == CLB_REDUCE_MEAN && rows > 0 ? temperature / (double)rows : temperature), inv, (float)(1.0 / temperature - inv)};
}

constexpr long long kMostBlocks = 1 << 16; // then they take one row after another

struct FwdPointers {
    const float *values;
    const int64_t *indices;
    const float *rest, *weight;
    float *row_loss, *stats, *listed;
};

template <typename T, int TH, int NV, bool CLUSTER>
cudaError_t launch_fwd(const T *x, const FwdPointers &p, T *grad, DistillArgs a, int ranks_log, long long pieces, cudaStream_t st)
{
    const int cluster = 1 << ranks_log;
    a.ranks_log = ranks_log, a.chunks = (int)((pieces + (long long)cluster * TH * NV - 1) / ((long long)cluster * TH * NV));
    constexpr int BLOCK = TH <= 32 ? 256 : TH, TEAMS = BLOCK / TH;
    const long long groups = (a.rows + TEAMS - 1) / TEAMS, most = kMostBlocks / cluster;
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
// pieces of the longest row: rows at a multiple of 16 bytes all begin at the first one's place in its piece
template <typename T> long long most_pieces(const T *x, const DistillArgs &a)
{
    const int phase = a.rows == 1 || a.stride % kPiece<T> == 0 ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : kPiece<T> - 1;
    return ((long long)a.classes + phase + kPiece<T> - 1) / kPiece<T>;
}
template <typename T, int TH> cudaError_t launch_stream(const T *x, const FwdPointers &p, T *grad, DistillArgs a, long long pieces, cudaStream_t st)
{
    constexpr int MT = TH - 32;
    a.chunks = (int)((pieces + MT * kTripPieces - 1) / (MT * kTripPieces));
    const int bytes = 2 * a.chunks * MT * kTripPieces * kPiece<T> / 8;
    const cudaError_t rc = ensure_dynamic_smem(distill_stream_kernel<T, TH>, bytes);
    if (rc != cudaSuccess) return rc;
    const long long most = (long long)sm_count() * (1024 / TH);
    CLB_TRACED("distill_stream_kernel", st,
               distill_stream_kernel<T, TH><<<(unsigned)(a.rows < most ? a.rows : most), TH, bytes, st>>>(x, p.values, p.indices, p.rest, p.weight, p.row_loss,
                                                                                                        p.stats, p.listed, grad, a));
    return cudaPeekAtLastError();
}
template <typename T> cudaError_t run_fwd(const T *x, const FwdPointers &p, T *grad, const DistillArgs &a, cudaStream_t st)
{
    constexpr int NV = kValues / kPiece<T>;
    const long long pieces = most_pieces(x, a), block = 256 * NV;
    if (pieces <= 4) return launch_fwd<T, 4, 1, false>(x, p, grad, a, 0, pieces, st);
    if (pieces <= 8 * NV / 4) return launch_fwd<T, 8, NV / 4, false>(x, p, grad, a, 0, pieces, st);
    if (pieces <= 16 * NV / 2) return launch_fwd<T, 16, NV / 2, false>(x, p, grad, a, 0, pieces, st);
    if (pieces <= 32 * NV / 2) return launch_fwd<T, 32, NV / 2, false>(x, p, grad, a, 0, pieces, st);
    if (pieces <= 32 * NV) return launch_fwd<T, 32, NV, false>(x, p, grad, a, 0, pieces, st);
    // A row of up to 16384 values in a block's registers where it fills most of them, else through the block twice.  134 million values with their gradient and
    // lists of 64, registers / twice: 8192 of 8192 values fp32 260 / 285 us, bf16 206 / 251; 16384 of 16384 249 / 219, bf16 203 / 217; 4096 of 8192 418 / 382, bf16
    // 371 / 246.  A few rows are shared by clusters instead, which is even at 64 rows and twice the time from 150 on.  Clusters / twice, bf16: 64 rows of 50257 14 / 18,
    // of 131072 21 / 24, of 390000 78 / 49; 100 rows 21 / 18, 36 / 26, 109 / 53; 148 rows 28 / 19, 44 / 26, 154 / 66; 296 rows 46 / 24, 84 / 42, 302 / 126.
    const long long room = (pieces <= 128 * NV ? 128 : 256) * NV;
    const bool many = a.rows >= 64 && a.classes <= 400000; // (two tables of 49 KB)
    if (pieces <= block && (!many || 10 * pieces >= 7 * room))
        return pieces <= 128 * NV ? launch_fwd<T, 128, NV, false>(x, p, grad, a, 0, pieces, st) : launch_fwd<T, 256, NV, false>(x, p, grad, a, 0, pieces, st);
    if (many)
        return pieces <= 768     ? launch_stream<T, 128>(x, p, grad, a, pieces, st)
               : pieces <= 8192  ? launch_stream<T, 256>(x, p, grad, a, pieces, st)
               : pieces <= 16384 ? launch_stream<T, 512>(x, p, grad, a, pieces, st)
                                 : launch_stream<T, 1024>(x, p, grad, a, pieces, st);
    if (pieces <= 8 * block) return launch_fwd<T, 256, NV, true>(x, p, grad, a, pieces <= 2 * block ? 1 : pieces <= 4 * block ? 2 : 3, pieces, st);
    return launch_fwd<T, 512, NV, true>(x, p, grad, a, 3, pieces, st);
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
    return sums_at(rows) + (rows > kOneSum ? kSumParts * 8 : 0);
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
        if (rc != cudaSuccess) { // (whatever the last error is by now)
            set_last_cuda_error((int)rc);
            cudaGetLastError();
            return CLB_ERR_LAUNCH;
        }
    }
    if (reduction == CLB_REDUCE_NONE) return rows > 0 ? check_launch() : CLB_OK;
    if (rows <= kOneSum) {
        CLB_TRACED("distill_sum_kernel", st, distill_sum_kernel<float, float><<<1, 1024, 0, st>>>((const float *)scratch, loss, rows));
        return check_launch(rows > 0 ? 2 : 1);
    }
    double *const parts = (double *)((char *)scratch + sums_at(rows));
    CLB_TRACED("distill_sum_kernel", st, distill_sum_kernel<float, double><<<kSumParts, 1024, 0, st>>>((const float *)scratch, parts, rows));
    CLB_TRACED("distill_sum_kernel", st, distill_sum_kernel<double, float><<<1, 1024, 0, st>>>(parts, loss, kSumParts));
    return check_launch(3);
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
        const long long pieces = most_pieces((const T *)scores, a);
        auto go = [&](auto launch) { launch((const T *)scores, indices, stats, listed, upstream, upstream_per_row ? 1 : 0, unit_done ? 1 : 0, (T *)grad, a, pieces, st); };
        if (pieces <= 4) go(launch_bwd<T, 4, 1>);
        else if (pieces <= 32) go(launch_bwd<T, 8, 4>);
        else if (pieces <= 128) go(launch_bwd<T, 32, 4>);
        else go(launch_bwd<T, 256, 4>);
    });
    return check_launch();
}

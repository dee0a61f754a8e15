// The k largest logits of every row and the mass of the others, for losses against a teacher's lists.
//
// A row's classes are ordered by value, ties by index; the first k are the list, and rest = log sum over the others of exp(x / T).
//
// One read of the logits.  Short rows are sorted whole: by counting pairs or in a warp's lanes.  Else a team of threads (a warp for rows of up to 1024 fp32 or 2048 half values; a block for longer ones, or for a segment of at
// most 32 KB, so that one row, too, fills part of the GPU) holds its values in registers:
//   1. The k-th largest of the threads' own maxima, rounded down to 16 bits of its order, is a bound that at least k values reach, and few more: with 256 maxima
//      of 64 values about 75 for k = 64.  One warp finds it by bisection.
//   2. The values that reach the bound go to a list in shared memory; the others are added up as exponentials with respect to the bound.
//   3. Each value's place in the list is the number of those above it, equal ones by index.
// Values that tie in great numbers, more than the list holds, take a second way: bisection over all values for the k-th largest, then over the indices of those
// that equal it.  Segments leave their k largest and the sum of their others; a block a row puts them together.
//
// Bound by issue: 16384 rows of 1000 bf16, k = 20: 27 us; 1024 of 128000, k = 64: 97 us for the segments (2.7 TB/s), 9 for the rows.
#include <algorithm>

#include "clb_rows.cuh"

using namespace clb;
using namespace clb_host;

namespace {

typedef unsigned long long u64;
constexpr uint32_t kMasked = 0x007fffffu; // order_key(-inf)
constexpr int kBlock = 256;

// (order of the value, index) as one number: larger comes first in a row's list; 0: nothing
__device__ __forceinline__ u64 place_of(uint32_t key, uint32_t i) { return ((u64)key << 32) | (0xffffffffu - i); }
__device__ __forceinline__ uint32_t index_of(u64 place) { return 0xffffffffu - (uint32_t)place; }
__device__ __forceinline__ float value_of(uint32_t key) // of order_key
{
    return key == 0xfffffffeu ? __uint_as_float(0x7fc00000u) : __uint_as_float((key & 0x80000000u) ? key & 0x7fffffffu : ~key);
}

// The largest bound of 16 bits that at least k of the N * 32 keys of a warp reach (0 if k of them are 0).
template <int N> __device__ __forceinline__ uint32_t bound_of(const uint32_t (&key)[N], int k)
{
    uint32_t any = key[0], all = key[0];
#pragma unroll
    for (int i = 1; i < N; ++i) any |= key[i], all &= key[i];
    any = __reduce_or_sync(0xffffffffu, any), all = __reduce_and_sync(0xffffffffu, all);
    if (!((any ^ all) >> 16)) return all & 0xffff0000u;
    uint32_t bit = 0x80000000u >> __clz(any ^ all); // (what is above is the same in all keys)
    uint32_t bound = all & ~(2 * bit - 1);
#pragma unroll 1
    for (; bit >= 0x10000u; bit >>= 1) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < N; ++i) n += key[i] >= (bound | bit);
        n = __reduce_add_sync(0xffffffffu, n);
        if (n >= k) bound |= bit;
        if ((uint32_t)(n - k) <= 4) break; // near enough (up to a quarter of k more cost a long list 10 to 30 %, to save a step or two)
    }
    return bound;
}

struct TopArgs {
    long long stride, rows;
    int classes, k, segments;
    int slots, longer; // pieces of each thread in a segment, one more in the first `longer` segments
    float temperature, c; // c = log2(e) / T
};

// Counts, flags and sums over a team of TH threads: of a warp, or of the block through `box` (TH / 32 + 1 words).
template <int TH> __device__ __forceinline__ void team_sync()
{
    if (TH == 32) __syncwarp();
    else __syncthreads();
}
template <int TH> __device__ __forceinline__ int team_count(int n, int *box)
{
    n = __reduce_add_sync(0xffffffffu, n);
    if (TH == 32) return n;
    if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = n;
    __syncthreads();
    n = 0;
#pragma unroll
    for (int w = 0; w < TH / 32; ++w) n += box[w];
    __syncthreads();
    return n;
}
template <int TH> __device__ __forceinline__ ExpSum team_merge(ExpSum s, ExpSum *box, float c)
{
    s = lanes_merge<32>(s, c);
    if (TH == 32) return s;
    __syncthreads();
    if ((threadIdx.x & 31) == 0) box[threadIdx.x >> 5] = s;
    __syncthreads();
    return lanes_merge<TH / 32>(box[threadIdx.x % (TH / 32)], c);
}

// order_key for values of 16 bits, in 16 bits, and back
template <typename T> __device__ __forceinline__ uint32_t short_key(T v)
{
    const uint32_t b = raw_bits(v);
    const float f = to_f(v);
    return f != f ? 0xffffu : f == 0.f ? 0x8000u : b & 0x8000u ? ~b & 0xffffu : b | 0x8000u;
}
template <typename T> __device__ __forceinline__ float value_of_short(uint32_t key)
{
    float f[2];
    two_values<T>(key == 0xffffu ? 0x7fffu : key & 0x8000u ? key & 0x7fffu : ~key & 0xffffu, f);
    return f[0];
}

// Candidates of a team, as 32-bit numbers of their order, 0 behind the last one up to a multiple of four.  Values of 16 bits share theirs with the class (counted
// from the segment's first), so that no two are alike; for floats, which tie seldom, the class stands beside it and is asked for only where two are alike.
template <typename T, int CAP> struct Candidates {
    static constexpr bool kShared = sizeof(T) == 2;
    uint4 four[CAP / 4 + 1];
    uint32_t cls[kShared ? 1 : CAP];
    __device__ __forceinline__ uint32_t *one() { return reinterpret_cast<uint32_t *>(four); }
    __device__ __forceinline__ void put(int n, float v, int c) // c: from the segment's first class
    {
        if constexpr (kShared) {
            one()[n] = short_key(from_f<T>(v)) << 16 | (0xffffu - (uint32_t)c);
        } else
            one()[n] = order_key(v), cls[n] = c;
    }
    __device__ __forceinline__ float value(uint32_t o) const
    {
        if constexpr (kShared) return value_of_short<T>(o >> 16);
        else return value_of(o);
    }
    __device__ __forceinline__ int class_at(int n) const
    {
        if constexpr (kShared) return (int)(0xffffu - (reinterpret_cast<const uint32_t *>(four)[n] & 0xffffu));
        else return (int)cls[n];
    }
};
// the place of each of `count` candidates among them, its value and class handed to `f`
template <int TH, typename T, int CAP, typename F> __device__ __forceinline__ void ranked(Candidates<T, CAP> &c, int count, int t, F &&f)
{
    for (int i = t; i < count; i += TH) {
        const uint32_t mine = c.one()[i];
        const int cls = c.class_at(i);
        int above = 0, same = 0;
#pragma unroll 4
        for (int j = 0; j < count; j += 4) {
            const uint4 q = c.four[j / 4];
            above += (q.x > mine) + (q.y > mine) + (q.z > mine) + (q.w > mine);
            if (!c.kShared) same += (q.x == mine) + (q.y == mine) + (q.z == mine) + (q.w == mine);
        }
        if (same > 1)
            for (int j = 0; j < count; ++j) above += c.one()[j] == mine && c.class_at(j) < cls;
        f(above, c.value(mine), cls);
    }
}
// the same of 64-bit places
template <typename F> __device__ __forceinline__ void ranked_places(const u64 *cand, int count, int t, F &&f)
{
    for (int i = t; i < count; i += kBlock) {
        const u64 mine = cand[i];
        int above = 0;
#pragma unroll 4
        for (int j = 0; j < count; j += 2) { // (the list is padded with a 0)
            const ulonglong2 two = *reinterpret_cast<const ulonglong2 *>(cand + j);
            above += (two.x > mine) + (two.y > mine);
        }
        f(above, mine);
    }
}

// TH threads a row (32: teams of a block of 256; 64 to 256: a block) or a segment of one (256), NV pieces a thread.  TH * SUB groups.
template <typename T, int TH, int NV, int SUB>
__global__ void __launch_bounds__(TH == 32 ? kBlock : TH, TH == 32 ? 4 : 4 * kBlock / TH) top_select_kernel(const T *__restrict__ x, float *__restrict__ values, int64_t *__restrict__ indices,
                                                               float *__restrict__ rest, u64 *__restrict__ places, ExpSum *__restrict__ sums, TopArgs a)
{
    constexpr int TEAMS = TH == 32 ? kBlock / TH : 1, EV = kPiece<T>, CAP = TH == 32 ? 256 : 512;
    static_assert(NV % SUB == 0 || 2 * NV == SUB || 4 * NV == SUB, "groups of whole pieces, of half a piece, or of one word");
    __shared__ Candidates<T, CAP> cand_all[TEAMS];
    __shared__ uint32_t keys_all[TEAMS][TH == 32 ? 2 : TH * SUB];
    __shared__ float extra_all[TEAMS][CAP];
    __shared__ int count_all[TEAMS], box[TH / 32 + 1];
    __shared__ uint32_t bound_all[TEAMS];
    __shared__ ExpSum sum_box[TH / 32];
    __shared__ float l_box[TH / 32];
    const int t = threadIdx.x % TH, team = threadIdx.x / TH;
    Candidates<T, CAP> &cand = cand_all[team];
    const long long items = a.rows * a.segments;
    for (long long item = (long long)blockIdx.x * TEAMS + team; item < items; item += (long long)gridDim.x * TEAMS) {
        const long long r = a.segments == 1 ? item : item / a.segments;
        const int seg = a.segments == 1 ? 0 : (int)(item - r * a.segments);
        const RowPieces<T> row(x + r * a.stride, a.classes);
        // (segments of like lengths: what a last one of a few classes lists is all candidates, which takes the second way: 1973 rows of 17000 bf16, k = 100: 1091 us)
        const int slots = TH == kBlock ? a.slots + (seg < a.longer) : NV;
        const int base = TH == kBlock ? (seg * a.slots + min(seg, a.longer)) * TH : 0;
        uint4 raw[NV];
        row.template load<NV, false, TH == kBlock>(raw, base + t, TH, base + slots * TH);
        // the class of value e of the thread's piece i, -1 for none
        auto class_of = [&](int i, int e) {
            const int c = row.first(base + i * TH + t) + e;
            return c >= 0 && c < a.classes && i < slots ? c : -1;
        };
        auto value_at = [&](int i, int e) {
            const uint32_t w = (&raw[i].x)[sizeof(T) == 4 ? e & 3 : e >> 1];
            float f[Word<T>::n];
            Word<T>::get(w, f);
            return f[Word<T>::n == 1 ? 0 : e & 1];
        };
        // ---- 1: the bound
        // pieces from i * TH on are not there if that is not below `used` (rows of blocks of 64 and 128 threads fill most of theirs)
        const int used = TH == 32 ? row.pieces : slots * TH;
        uint32_t tops[NV], key[SUB], bound;
#pragma unroll
        for (int i = 0; i < NV; ++i) tops[i] = i * TH < used ? piece_max_nan<T>(raw[i]) : low_word<T>();
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
            uint32_t top;
            if constexpr (NV >= SUB) {
                top = tops[s * (NV / SUB)];
#pragma unroll
                for (int i = 1; i < NV / SUB; ++i) top = max_nan<T>(top, tops[s * (NV / SUB) + i]);
            } else if constexpr (2 * NV == SUB)
                top = s & 1 ? max_nan<T>(raw[s / 2].z, raw[s / 2].w) : max_nan<T>(raw[s / 2].x, raw[s / 2].y);
            else
                top = (&raw[s / 4].x)[s % 4];
            key[s] = word_key<T>(top);
        }
        if constexpr (TH == 32)
            bound = bound_of(key, a.k);
        else {
#pragma unroll
            for (int s = 0; s < SUB; ++s) keys_all[team][s * TH + t] = key[s];
            if (t == 0) count_all[team] = 0;
            for (int i = t; i < CAP / 4 + 1; i += TH) cand.four[i] = make_uint4(0, 0, 0, 0); // (what is behind the list's end)
            __syncthreads();
            if (t < 32) {
                uint32_t all[TH * SUB / 32];
#pragma unroll
                for (int i = 0; i < TH * SUB / 32; ++i) all[i] = keys_all[team][i * 32 + t];
                bound = bound_of(all, a.k);
                if (t == 0) bound_all[team] = bound;
            }
            __syncthreads();
            bound = bound_all[team];
        }
        if (bound <= kMasked) bound = kMasked + 1; // fewer than k groups have a value: all values are candidates, and the first k of the masked
        const bool few = bound == kMasked + 1;
        const float reach = value_of(bound);
        // ---- 2: candidates, and the sum of the others
        const int own_first = base == 0 ? 0 : row.first(base); // the segment's first class
        auto push = [&](float v, int cls) {
            const int n = atomicAdd(&count_all[team], 1);
            if (n < CAP) cand.put(n, v, cls - own_first);
        };
        const ExpRef er = exp_ref(reach, a.c);
        float l = 0.f;
        uint32_t which_all[NV * EV / 32]; // the thread's candidates
#pragma unroll
        for (int i = 0; i < NV * EV / 32; ++i) which_all[i] = 0;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (i * TH >= used) continue;
            const uint32_t w[4] = {raw[i].x, raw[i].y, raw[i].z, raw[i].w};
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                float g[Word<T>::n];
                Word<T>::get(w[q], g);
#pragma unroll
                for (int z = 0; z < Word<T>::n; ++z) {
                    if (g[z] < reach) l += ex2(fmaf(g[z], a.c, -er.R));
                    else which_all[(i * EV + q * Word<T>::n + z) / 32] |= 1u << (i * EV + q * Word<T>::n + z) % 32;
                }
            }
        }
        if (few)
#pragma unroll
            for (int i = 0; i < NV; ++i)
#pragma unroll
                for (int e = 0; e < EV; ++e) {
                    const int cls = class_of(i, e);
                    if (cls >= own_first && cls < own_first + a.k) which_all[(i * EV + e) / 32] |= 1u << (i * EV + e) % 32;
                }
        int count = 0;
#pragma unroll
        for (int i = 0; i < NV * EV / 32; ++i) count += __popc(which_all[i]);
        if (__any_sync(0xffffffffu, count > 0)) { // where the thread's go: behind the lanes before it, a block's warps as they come
            int n = -count;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int before = __shfl_up_sync(0xffffffffu, count, o);
                count += (t & 31) >= o ? before : 0;
            }
            n += count;
            if constexpr (TH > 32) {
                int first = 0;
                if ((t & 31) == 31) first = atomicAdd(&count_all[team], count);
                n += __shfl_sync(0xffffffffu, first, 31);
            } else
                count = __shfl_sync(0xffffffffu, count, 31);
#pragma unroll
            for (int i = 0; i < NV * EV / 32; ++i)
                for (uint32_t which = which_all[i]; which; which &= which - 1, ++n) {
                    const int at = i * 32 + __ffs(which) - 1, cls = row.first(base + at / EV * TH + t) + at % EV;
                    // (read again: no register is named by a number that varies.  Beyond the row only where the bound is NaN and all are candidates, too many then.)
                    if (n < CAP && cls >= 0 && cls < a.classes) cand.put(n, to_f(row.row[cls]), cls - own_first);
                }
        }
        l = lanes_sum<32>(l * er.fix);
        if (TH > 32 && (t & 31) == 0) l_box[t >> 5] = l;
        team_sync<TH>();
        if constexpr (TH > 32) {
            count = count_all[team];
            l = 0.f;
#pragma unroll
            for (int w = 0; w < TH / 32; ++w) l += l_box[w];
        }
        // f(value, class) for each of the thread's values; code of its own, as what follows is rare (a rotation: no register is named by a number that varies)
        auto for_each = [&](auto f) {
#pragma unroll 1
            for (int i = 0; i < NV; ++i) {
                const uint4 q = raw[0];
#pragma unroll
                for (int n = 1; n < NV; ++n) raw[n - 1] = raw[n];
                raw[NV - 1] = q;
#pragma unroll
                for (int e = 0; e < EV; ++e)
                    if (class_of(i, e) >= 0) f(value_at(NV - 1, e), class_of(i, e));
            }
        };
        const bool overflow = count > CAP;
        if (overflow) { // ---- the k-th largest key, then the last index of those that equal it
            uint32_t key = 0, last = 0;
            int n;
            for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
                n = 0;
                for_each([&](float v, int) { n += order_key(v) >= (key | bit); });
                if (team_count<TH>(n, box) >= a.k) key |= bit;
            }
            n = 0;
            for_each([&](float v, int) { n += order_key(v) > key; });
            const int need = a.k - team_count<TH>(n, box);
            for (uint32_t bit = 1u << 30; bit; bit >>= 1) { // the largest class that fewer than `need` of them are below
                n = 0;
                for_each([&](float v, int cls) { n += (uint32_t)cls < (last | bit) && order_key(v) == key; });
                if (team_count<TH>(n, box) < need) last |= bit;
            }
            if (t == 0) count_all[team] = 0;
            team_sync<TH>();
            for_each([&](float v, int cls) {
                if (order_key(v) > key || (order_key(v) == key && (uint32_t)cls <= last)) push(v, cls);
            });
            team_sync<TH>();
            count = count_all[team];
        }
        if (TH == 32 || overflow) {
            if (t < 4) cand.one()[count + t] = 0;
            team_sync<TH>();
        }
        // ---- 3: their places
        const long long at = item * a.k;
        uint32_t *const kth_box = keys_all[team];
        ranked<TH>(cand, count, t, [&](int rank, float v, int c) {
            const int cls = own_first + c;
            if (rank < a.k) {
                if (a.segments == 1) values[at + rank] = v, indices[at + rank] = cls;
                else places[at + rank] = place_of(order_key(v), cls);
                if (rank == a.k - 1) kth_box[0] = order_key(v), kth_box[1] = cls;
            } else
                extra_all[team][rank - a.k] = v;
        });
        team_sync<TH>();
        auto finish = [&](ExpSum others) {
            if (a.segments == 1) rest[r] = others.m / a.temperature + logf(others.l);
            else sums[item] = others;
        };
        if (overflow || er.far || !(reach < INFINITY) || (!(l > 1e-20f) && count <= a.k)) {
            // the bound is no reference for the others (they are far below it), or they are not all counted: once more, with respect to their own largest
            const u64 kth = place_of(kth_box[0], kth_box[1]);
            ExpSum others{-INFINITY, 0.f};
            bool inf = false;
            for_each([&](float v, int cls) {
                if (place_of(order_key(v), cls) >= kth) return;
                if (v == INFINITY) inf = true;
                else others = merge(others, single(v), a.c);
            });
            others = team_merge<TH>(others, sum_box, a.c);
            if (team_count<TH>(inf, box) && others.l == others.l) others = ExpSum{INFINITY, 1.f};
            if (t == 0) finish(others);
        } else if (t < 32) {
            ExpSum others{reach, t == 0 ? l : 0.f};
            bool inf = false;
            for (int i = t; i < count - a.k; i += 32) { // in the order of their places, whatever the order in which they came to the list
                const float v = extra_all[team][i];
                if (v == INFINITY) inf = true;
                else others = merge(others, single(v), a.c);
            }
            others = lanes_merge<32>(others, a.c);
            if (__any_sync(0xffffffffu, inf) && others.l == others.l) others = ExpSum{INFINITY, 1.f};
            if (t == 0) finish(others);
        }
        team_sync<TH>(); // the tables are used again
    }
}

// Rows of up to 64 classes: G lanes a row (1 to 4), 16 neighbouring classes each.  A class's place is the number of classes before it, counted over all pairs; with
// a warp a row 40759 rows of 3 classes took 78 us, so 7.6.
constexpr int kFew = 16;
template <typename T, int G>
__global__ void __launch_bounds__(kBlock) top_few_kernel(const T *__restrict__ x, float *__restrict__ values, int64_t *__restrict__ indices,
                                                         float *__restrict__ rest, TopArgs a)
{
    const int t = threadIdx.x % G, lane = threadIdx.x & 31;
    for (long long r0 = (long long)blockIdx.x * (kBlock / G) + (threadIdx.x - lane) / G; r0 < a.rows; r0 += (long long)gridDim.x * (kBlock / G)) {
        const long long r = r0 + lane / G;
        const bool live = r < a.rows;
        uint32_t key[kFew]; // 0: no class
        int before[kFew];
#pragma unroll
        for (int i = 0; i < kFew; ++i) {
            const int c = t * kFew + i;
            key[i] = live && c < a.classes ? order_key(to_f(x[r * a.stride + c])) : 0;
            before[i] = 0;
        }
#pragma unroll
        for (int i = 0; i < kFew; ++i)
#pragma unroll
            for (int j = 0; j < kFew; ++j)
                if (j != i) before[i] += j < i ? key[j] >= key[i] : key[j] > key[i];
#pragma unroll 1
        for (int g = 1; g < G; ++g) { // the other lanes' classes; an equal one of an earlier lane is before
            const int from = (t + g) % G;
#pragma unroll
            for (int j = 0; j < kFew; ++j) {
                const uint32_t other = __shfl_sync(0xffffffffu, key[j], (lane - t) + from) + (from < t);
#pragma unroll
                for (int i = 0; i < kFew; ++i) before[i] += other > key[i];
            }
        }
        float m = -INFINITY;
#pragma unroll
        for (int i = 0; i < kFew; ++i) {
            if (!key[i]) continue;
            const float v = value_of(key[i]);
            if (before[i] < a.k) values[r * a.k + before[i]] = v, indices[r * a.k + before[i]] = t * kFew + i;
            else m = fmaxf(m, v);
        }
        m = lanes_max<G>(m);
        const float ref = finite_or_zero(m);
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < kFew; ++i) {
            if (!key[i] || before[i] < a.k) continue;
            const float v = value_of(key[i]);
            l += m == INFINITY && v == v ? (v == INFINITY ? 1.f : 0.f) : exp_of(v, ref, a.c);
        }
        l = lanes_sum<G>(l);
        if (live && t == 0) rest[r] = m / a.temperature + logf(l);
    }
}

// Rows of up to 32 * N classes, short lists: a warp a row, N classes a lane, sorted there; the row's list is taken off the lanes' heads one by one, and what is left
// in the lanes are the others.  An element is its order and class in one number (values of 16 bits), or the order with the class beside it.  Bound by issue:
// 65536 rows of 100 classes, k = 10: 43 us (bf16 37), k = 100: 198 (124).
template <typename T, int N>
__global__ void __launch_bounds__(kBlock) top_short_kernel(const T *__restrict__ x, float *__restrict__ values, int64_t *__restrict__ indices,
                                                           float *__restrict__ rest, TopArgs a)
{
    constexpr bool SHARED = sizeof(T) == 2;
    const int lane = threadIdx.x & 31;
    for (long long r = (long long)blockIdx.x * (kBlock / 32) + threadIdx.x / 32; r < a.rows; r += (long long)gridDim.x * (kBlock / 32)) {
        uint32_t key[N], cls[SHARED ? 1 : N]; // 0: no class
        T raw[N];
#pragma unroll
        for (int i = 0; i < N; ++i) raw[i] = i * 32 + lane < a.classes ? x[r * a.stride + i * 32 + lane] : from_f<T>(0.f);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = i * 32 + lane;
            if constexpr (SHARED) key[i] = c < a.classes ? short_key(raw[i]) << 16 | (0xffffu - c) : 0;
            else key[i] = c < a.classes ? order_key(raw[i]) : 0, cls[i] = c;
        }
        if constexpr (SHARED) {
            odd_even_merges<N>([&](int i, int j) {
                const uint32_t hi = max(key[i], key[j]);
                key[j] = min(key[i], key[j]), key[i] = hi;
            });
        } else {
            odd_even_merges<N>([&](int i, int j) {
                const bool swap = key[j] > key[i] || (key[j] == key[i] && cls[j] < cls[i]);
                const uint32_t k = key[i], c = cls[i];
                key[i] = swap ? key[j] : k, cls[i] = swap ? cls[j] : c;
                key[j] = swap ? k : key[j], cls[j] = swap ? c : cls[j];
            });
        }
        auto value = [](uint32_t key) {
            if constexpr (SHARED) return value_of_short<T>(key >> 16);
            else return value_of(key);
        };
        for (int n0 = 0; n0 < a.k; n0 += 32) {
            const int many = min(32, a.k - n0);
            uint32_t place = 0, place_cls = 0; // of the list's next 32 the lane-th
            for (int n = 0; n < many; ++n) {
                const uint32_t top = __reduce_max_sync(0xffffffffu, key[0]);
                bool taken = key[0] == top;
                uint32_t first = 0;
                if constexpr (!SHARED) {
                    first = __reduce_min_sync(0xffffffffu, taken ? cls[0] : 0xffffffffu);
                    taken = taken && cls[0] == first;
                }
                if (lane == n) place = top, place_cls = first;
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    key[i] = taken ? (i + 1 < N ? key[i + 1] : 0) : key[i];
                    if constexpr (!SHARED)
                        if (i + 1 < N) cls[i] = taken ? cls[i + 1] : cls[i];
                }
            }
            if (lane < many) {
                const long long at = r * a.k + n0 + lane;
                values[at] = value(place), indices[at] = SHARED ? 0xffffu - (place & 0xffffu) : place_cls;
            }
        }
        float m = -INFINITY, v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = key[i] ? value(key[i]) : -INFINITY, m = fmaxf(m, v[i]);
        m = lanes_max<32>(m);
        const float ref = finite_or_zero(m);
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) l += m == INFINITY && v[i] == v[i] ? (v[i] == INFINITY ? 1.f : 0.f) : exp_of(v[i], ref, a.c);
        l = lanes_sum<32>(l);
        if (lane == 0) rest[r] = m / a.temperature + logf(l);
    }
}

// A row's segments put together: a block a row.  places [rows][segments * k], sums [rows][segments].
__global__ void __launch_bounds__(kBlock) top_merge_kernel(const u64 *__restrict__ places, const ExpSum *__restrict__ sums, float *__restrict__ values,
                                                           int64_t *__restrict__ indices, float *__restrict__ rest, TopArgs a)
{
    constexpr int CAP = 512, WARPS = kBlock / 32;
    __shared__ __align__(16) u64 cand[CAP + 2];
    __shared__ uint32_t keys[kBlock], bound_box;
    __shared__ int count_box, box[WARPS];
    __shared__ u64 kth_box, best[WARPS];
    __shared__ ExpSum sum_box[WARPS];
    const int t = threadIdx.x, n = a.segments * a.k;
    for (long long r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const u64 *p = places + r * n;
        uint32_t top = 0;
        for (int i = 0; i < n; i += kBlock) { // (the segments' lists are in order: turned, so that a thread's are from different places of theirs, and the bound is near)
            const int j = i + ((t + 37 * (i / kBlock)) & (kBlock - 1));
            if (j < n) top = max(top, (uint32_t)(p[j] >> 32));
        }
        keys[t] = top;
        if (t == 0) count_box = 0;
        __syncthreads();
        if (t < 32) {
            uint32_t key[WARPS];
#pragma unroll
            for (int i = 0; i < WARPS; ++i) key[i] = keys[i * 32 + t];
            const uint32_t b = bound_of(key, a.k);
            if (t == 0) bound_box = b;
        }
        __syncthreads();
        const uint32_t bound = bound_box;
        for (int i = t; i < n; i += kBlock)
            if ((uint32_t)(p[i] >> 32) >= bound) {
                const int c = atomicAdd(&count_box, 1);
                if (c < CAP) cand[c] = p[i];
            }
        __syncthreads();
        const int count = count_box;
        if (count <= CAP) {
            if (t == 0) cand[count] = cand[count + 1] = 0;
            __syncthreads();
            ranked_places(cand, count, t, [&](int rank, u64 place) {
                if (rank >= a.k) return;
                values[r * a.k + rank] = value_of((uint32_t)(place >> 32)), indices[r * a.k + rank] = index_of(place);
                if (rank == a.k - 1) kth_box = place;
            });
        } else { // values that tie in great numbers: the next one after the last, k times
            u64 last = ~0ull;
            for (int i = 0; i < a.k; ++i) {
                u64 mine = 0;
                for (int j = t; j < n; j += kBlock)
                    if (p[j] < last && p[j] > mine) mine = p[j];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mine = max(mine, __shfl_xor_sync(0xffffffffu, mine, o));
                if ((t & 31) == 0) best[t >> 5] = mine;
                __syncthreads();
                last = 0;
#pragma unroll
                for (int w = 0; w < WARPS; ++w) last = max(last, best[w]);
                if (t == 0) values[r * a.k + i] = value_of((uint32_t)(last >> 32)), indices[r * a.k + i] = index_of(last);
                __syncthreads();
            }
            if (t == 0) kth_box = last;
        }
        __syncthreads();
        const u64 kth = kth_box;
        ExpSum others{-INFINITY, 0.f};
        bool inf = false;
        auto add = [&](ExpSum s) {
            if (s.m == INFINITY) inf = true;
            else others = merge(others, s, a.c);
        };
        for (int i = t; i < n; i += kBlock)
            if (p[i] < kth) add(single(value_of((uint32_t)(p[i] >> 32))));
        for (int i = t; i < a.segments; i += kBlock) add(sums[r * a.segments + i]);
        others = team_merge<kBlock>(others, sum_box, a.c);
        if (team_count<kBlock>(inf, box) && others.l == others.l) others = ExpSum{INFINITY, 1.f};
        if (t == 0) rest[r] = others.m / a.temperature + logf(others.l);
        __syncthreads(); // the tables are used again
    }
}

constexpr int kPieces = 8; // of a thread: 32 KB a block of 256

// pieces of the longest row (rows at a multiple of 16 bytes all begin at the first one's place in its piece; with `any`, at the worst)
template <typename T> long long most_pieces(const void *x, int64_t stride, int64_t rows, int64_t classes, bool any = false)
{
    const int phase = !any && (rows == 1 || stride % kPiece<T> == 0) ? (int)((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(T)) : kPiece<T> - 1;
    return (classes + phase + kPiece<T> - 1) / kPiece<T>;
}
int slots_of(long long pieces) { return (int)((pieces + kBlock - 1) / kBlock); } // pieces of each thread of a block
int segments_of(long long pieces) { return (slots_of(pieces) + kPieces - 1) / kPieces; }

} // namespace

extern "C" size_t clb_top_logits_scratch_bytes(int64_t rows, int64_t classes, int k, int dtype)
{
    if (rows <= 0 || classes <= 0 || k <= 0 || classes > CLB_CLASSES_MAX) return 0;
    int segments = 0;
    with_score_type(dtype, [&](auto t) { segments = segments_of(most_pieces<decltype(t)>(nullptr, 1, rows, classes, true)); });
    return segments > 1 ? (size_t)rows * segments * (8 * (size_t)k + sizeof(ExpSum)) : 0;
}

extern "C" int clb_top_logits(const void *x, int64_t row_stride, float *values, int64_t *indices, float *rest, void *scratch, size_t scratch_bytes, int64_t rows,
                              int64_t classes, int k, double temperature, int dtype, void *stream)
{
    if (!x || !values || !indices || !rest || rows < 0 || classes <= 0 || row_stride < 0 || k <= 0 || !(temperature >= 1e-30 && temperature <= 1e30))
        return CLB_ERR_ARG;
    if (k > classes) return CLB_ERR_SHAPE;
    if (k > CLB_TOP_MAX || classes > CLB_CLASSES_MAX) return CLB_ERR_TOO_LARGE;
    if (dtype != CLB_F32 && dtype != CLB_F16 && dtype != CLB_BF16) return CLB_ERR_ARG;
    if (rows == 0) return CLB_OK;
    if (scratch_bytes < clb_top_logits_scratch_bytes(rows, classes, k, dtype) || (!scratch && clb_top_logits_scratch_bytes(rows, classes, k, dtype)))
        return CLB_ERR_SCRATCH;
    cudaStream_t st = (cudaStream_t)stream;
    int launches = 1;
    with_score_type(dtype, [&](auto v) {
        using T = decltype(v);
        const long long pieces = most_pieces<T>(x, row_stride, rows, classes);
        const int segments = segments_of(pieces);
        TopArgs a{row_stride, rows, (int)classes, k, segments, slots_of(pieces) / segments, slots_of(pieces) % segments, (float)temperature, (float)(1.4426950408889634 / temperature)};
        u64 *const places = (u64 *)scratch;
        ExpSum *const sums = (ExpSum *)(places + (a.segments > 1 ? rows * a.segments * k : 0));
        auto blocks = [](long long n) { return (unsigned)(n < (1 << 16) ? n : (1 << 16)); }; // (then they take one row after another)
        // all pairs / short / select, us, 65536 rows (fp32, bf16), k = 10: 32 classes 21 19 / 31 29 / -; 64 44 43 / 31 28 / -; 100 - / 43 37 / 88 98; 256 - / 72 56 / 94 89;
        // 300 - / 104 88 (16 a lane) / 99 104.  A bound from groups of four classes needs more of them than the list has, or every value is a candidate: 400 classes, k = 80 and 100:
        // select 434 295, 3705 2487, short 475 260, 562 307.
        const bool few = classes <= 2 * kFew || (classes <= 4 * kFew && k > 20);
        if (!few && (classes <= 256 || (classes <= 512 && 9 * k > 2 * classes))) {
            auto go = [&](auto kernel) {
                CLB_TRACED("top_short_kernel", st, kernel<<<blocks((rows + 7) / 8), kBlock, 0, st>>>((const T *)x, values, indices, rest, a));
            };
            if (classes <= 64) go(top_short_kernel<T, 2>);
            else if (classes <= 128) go(top_short_kernel<T, 4>);
            else if (classes <= 256) go(top_short_kernel<T, 8>);
            else go(top_short_kernel<T, 16>);
            return;
        }
        if (few) {
            const int lanes = classes <= kFew ? 1 : classes <= 2 * kFew ? 2 : 4;
            const unsigned n = blocks((rows * lanes + kBlock - 1) / kBlock);
            auto go = [&](auto kernel) { CLB_TRACED("top_few_kernel", st, kernel<<<n, kBlock, 0, st>>>((const T *)x, values, indices, rest, a)); };
            if (lanes == 1) go(top_few_kernel<T, 1>);
            else if (lanes == 2) go(top_few_kernel<T, 2>);
            else go(top_few_kernel<T, 4>);
            return;
        }
        auto go = [&](auto kernel, long long n, int threads) {
            CLB_TRACED("top_select_kernel", st, kernel<<<blocks(n), threads, 0, st>>>((const T *)x, values, indices, rest, places, sums, a));
        };
        // Groups: more of them make a tighter bound and a longer search for it.  Where few more than k of them have values, the bound lets through more values than the
        // list holds and the row takes the second way.  Plain / twice as many groups, us, 33 million values, by groups / k: fp32 257 classes k = 32 (1.0) 423 / 136, k = 16
        // (2.1) 93 / 101; 513 k = 128 (1.0) 4185 / 518, k = 64 (2.0) 229 / 239; 640 k = 90 (1.8) 294 / 260; bf16 1025 k = 128 (1.0) 2987 / 228, 2049 k = 90 (1.4) 132 / 111,
        // k = 64 (2.0) 90 / 101.  Lists of 90 are even from 2.1 on, longer ones always shorter by the tighter bound: fp32 1000 k = 110 (2.3) 239 / 199.
        auto enough = [&](long long groups) { return 5 * groups >= 9 * k; };
        auto groups = [&](int threads, int pieces_each, int subs) { // that have values
            long long n = 0;
            for (int s = 0, first = 0; s < subs && subs < pieces_each; ++s, first += pieces_each / subs * threads) n += std::max(0ll, std::min<long long>(threads, pieces - first));
            return subs < pieces_each ? n : pieces * (subs / pieces_each);
        };
        auto warps = [&](auto few, auto many, auto most, int pieces_each) {
            const long long n = (rows + 7) / 8;
            if (k <= 32 && enough(groups(32, pieces_each, 4))) go(few, n, kBlock);
            else if (k <= 96 && enough(groups(32, pieces_each, 8))) go(many, n, kBlock);
            else go(most, n, kBlock);
        };
        constexpr int SHORT = sizeof(T) == 2 ? 4 : kPieces; // half types: 1024 values of a warp, or 2048
        if (pieces <= 32 * SHORT) warps(top_select_kernel<T, 32, SHORT, 4>, top_select_kernel<T, 32, SHORT, 8>, top_select_kernel<T, 32, SHORT, 16>, SHORT);
        else if (pieces <= 32 * kPieces) warps(top_select_kernel<T, 32, kPieces, 4>, top_select_kernel<T, 32, kPieces, 8>, top_select_kernel<T, 32, kPieces, 16>, kPieces);
        else if (pieces <= 64 * kPieces) go(k <= 96 && enough(groups(64, kPieces, 4)) ? top_select_kernel<T, 64, kPieces, 4> : top_select_kernel<T, 64, kPieces, 8>, rows, 64);
        else if (pieces <= 128 * kPieces) go(k <= 96 && enough(groups(128, kPieces, 2)) ? top_select_kernel<T, 128, kPieces, 2> : top_select_kernel<T, 128, kPieces, 4>, rows, 128);
        else go(top_select_kernel<T, kBlock, kPieces, 1>, rows * a.segments, kBlock);
        if (a.segments > 1) {
            CLB_TRACED("top_merge_kernel", st, top_merge_kernel<<<blocks(rows), kBlock, 0, st>>>(places, sums, values, indices, rest, a));
            launches = 2;
        }
    });
    return check_launch(launches);
}

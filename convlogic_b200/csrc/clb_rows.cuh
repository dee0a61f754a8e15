// Rows of scores in registers (distill.cu, top_logits.cu): a team of threads holds a row as 16-byte pieces, so that what needs the row's maximum or its sum
// first (a soft-max, a gradient) reads it once.
//
// A team is 4 to 32 lanes of a warp, a block, or a cluster of blocks.  Piece j of a row are the 16 / sizeof(T) values from the 16-byte boundary j * 16 bytes
// after the one at or before the row's first value; the first and the last piece may hold fewer values, and those are read one by one (no byte
// outside the row is touched, whatever its address and length).  Values that are not there are -inf, which adds nothing to a maximum or to a sum of
// exponentials.
#pragma once

#include "clb_scores.cuh"

namespace clb {

__device__ __forceinline__ float ex2(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

// Two floats at once: one instruction for two sums, products or fused multiply-adds.
struct Pair {
    unsigned long long v;
};
__device__ __forceinline__ Pair pair_of(float a, float b)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split(Pair p, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair operator+(Pair a, Pair b)
{
    Pair p;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
    return p;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b)
{
    Pair p;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
    return p;
}
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c)
{
    Pair p;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return p;
}
__device__ __forceinline__ Pair ex2(Pair p)
{
    float a, b;
    split(p, a, b);
    return pair_of(ex2(a), ex2(b));
}

template <typename T> constexpr int kPiece = 16 / (int)sizeof(T); // values of a piece
template <typename T> __device__ __forceinline__ constexpr uint32_t low_bits() { return sizeof(T) == 4 ? 0xff800000u : 0u; }
template <> __device__ __forceinline__ constexpr uint32_t low_bits<__half>() { return 0xfc00u; }
template <> __device__ __forceinline__ constexpr uint32_t low_bits<__nv_bfloat16>() { return 0xff80u; }
template <typename T> __device__ __forceinline__ constexpr uint32_t low_word() { return sizeof(T) == 4 ? low_bits<T>() : low_bits<T>() * 0x10001u; } // -inf everywhere

__device__ __forceinline__ uint32_t raw_bits(float v) { return __float_as_uint(v); }
__device__ __forceinline__ uint32_t raw_bits(__half v) { return __half_as_ushort(v); }
__device__ __forceinline__ uint32_t raw_bits(__nv_bfloat16 v) { return __bfloat16_as_ushort(v); }

// the values of one 32-bit word of a piece: one float, or two of 16 bits
template <typename T> struct Word;
template <> struct Word<float> {
    static constexpr int n = 1;
    static __device__ __forceinline__ void get(uint32_t w, float (&v)[1]) { v[0] = __uint_as_float(w); }
    static __device__ __forceinline__ uint32_t put(const float (&v)[1]) { return __float_as_uint(v[0]); }
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b))); }
};
template <> struct Word<__half> {
    static constexpr int n = 2;
    static __device__ __forceinline__ __half2 of(uint32_t w) { return *reinterpret_cast<__half2 *>(&w); }
    static __device__ __forceinline__ uint32_t to(__half2 h) { return *reinterpret_cast<uint32_t *>(&h); }
    static __device__ __forceinline__ void get(uint32_t w, float (&v)[2])
    {
        const float2 f = __half22float2(of(w));
        v[0] = f.x, v[1] = f.y;
    }
    static __device__ __forceinline__ uint32_t put(const float (&v)[2]) { return to(__floats2half2_rn(v[0], v[1])); }
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return to(__hmax2(of(a), of(b))); }
};
template <> struct Word<__nv_bfloat16> {
    static constexpr int n = 2;
    static __device__ __forceinline__ __nv_bfloat162 of(uint32_t w) { return *reinterpret_cast<__nv_bfloat162 *>(&w); }
    static __device__ __forceinline__ uint32_t to(__nv_bfloat162 h) { return *reinterpret_cast<uint32_t *>(&h); }
    static __device__ __forceinline__ void get(uint32_t w, float (&v)[2]) { v[0] = __uint_as_float(w << 16), v[1] = __uint_as_float(w & 0xffff0000u); }
    static __device__ __forceinline__ uint32_t put(const float (&v)[2]) { return to(__floats2bfloat162_rn(v[0], v[1])); }
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b) { return to(__hmax2(of(a), of(b))); }
};

// (as function templates: the float case has one value a word, and never calls them)
template <typename T> __device__ __forceinline__ void two_values(uint32_t w, float (&f)[2])
{
    if constexpr (sizeof(T) == 2) Word<T>::get(w, f);
}
template <typename T> __device__ __forceinline__ uint32_t two_word(const float (&f)[2])
{
    if constexpr (sizeof(T) == 2) return Word<T>::put(f);
    return 0;
}

// where the pieces of a row lie
template <typename T> struct RowPieces {
    const T *row;
    int classes, phase, pieces; // phase: values that the first piece lacks
    __device__ __forceinline__ RowPieces(const T *r, int n) : row(r), classes(n)
    {
        phase = (int)((reinterpret_cast<uintptr_t>(r) & 15) / sizeof(T));
        pieces = (int)(((long long)n + phase + kPiece<T> - 1) / kPiece<T>);
    }
    __device__ __forceinline__ int first(int j) const { return j * kPiece<T> - phase; } // class of the piece's first value, below 0 for one that is not there
    __device__ __forceinline__ bool whole(int j) const { return first(j) >= 0 && first(j) <= classes - kPiece<T>; }
    __device__ __forceinline__ int piece_of(int cls) const { return (cls + phase) / kPiece<T>; }
    __device__ __forceinline__ int place_of(int cls) const { return (cls + phase) % kPiece<T>; }
    // piece j, one that lies across an end of the row value by value
    __device__ __forceinline__ uint4 edge(int j) const
    {
        uint32_t w[4] = {low_word<T>(), low_word<T>(), low_word<T>(), low_word<T>()};
        if (j < pieces)
#pragma unroll
            for (int e = 0; e < kPiece<T>; ++e) {
                const int i = first(j) + e;
                if (i >= 0 && i < classes) {
                    const uint32_t b = raw_bits(row[i]);
                    if (sizeof(T) == 4) w[e & 3] = b;
                    else w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | b << 16 : (w[e >> 1] & 0xffff0000u) | b;
                }
            }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
    // pieces j, j + step, ...: the whole ones are asked for before anything waits.  LAST: not read again.  BOUND: none from `end` on (of the same step as those)
    template <int NV, bool LAST = true, bool BOUND = false> __device__ __forceinline__ void load(uint4 (&q)[NV], int j, int step, int end = 0) const
    {
        const T *const from = row + first(j);
        auto get = [&](int i) {
            const uint4 *p = reinterpret_cast<const uint4 *>(from + (long long)i * step * kPiece<T>);
            return LAST ? __ldcs(p) : __ldg(p);
        };
        if (inside<NV>(j, step) && (!BOUND || j + (NV - 1) * step < end)) {
#pragma unroll
            for (int i = 0; i < NV; ++i) q[i] = get(i);
            return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            q[i] = make_uint4(low_word<T>(), low_word<T>(), low_word<T>(), low_word<T>());
            if (whole(j + i * step) && (!BOUND || j + i * step < end)) q[i] = get(i);
        }
        if (j == 0 && !whole(0)) q[0] = edge(0); // (a first piece is some thread's first)
        const int last = pieces - 1, i = last - j;
        if (last > 0 && i >= 0 && i < NV * step && i % step == 0 && (!BOUND || last < end) && !whole(last)) {
            const uint4 e = edge(last);
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const bool here = n * step == i;
                q[n].x = here ? e.x : q[n].x, q[n].y = here ? e.y : q[n].y, q[n].z = here ? e.z : q[n].z, q[n].w = here ? e.w : q[n].w;
            }
        }
    }
    // are pieces j, j + step, ..., NV of them, all whole?
    template <int NV> __device__ __forceinline__ bool inside(int j, int step) const { return first(j) >= 0 && first(j + (NV - 1) * step) <= classes - kPiece<T>; }
    // writes a piece's values to the row `out` of as many classes; `aligned`: out has this row's phase
    __device__ __forceinline__ void store(T *out, bool aligned, int j, const uint4 &v) const
    {
        if (aligned && whole(j)) {
            __stcs(reinterpret_cast<uint4 *>(out + first(j)), v);
            return;
        }
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < kPiece<T>; ++e) {
            const int i = first(j) + e;
            if (i >= 0 && i < classes) {
                if (sizeof(T) == 4) reinterpret_cast<uint32_t *>(out)[i] = w[e & 3];
                else reinterpret_cast<uint16_t *>(out)[i] = (uint16_t)(w[e >> 1] >> ((e & 1) * 16));
            }
        }
    }
};

// value e of a piece becomes -inf
template <typename T> __device__ __forceinline__ void drop_value(uint4 &q, int e)
{
    uint32_t w[4] = {q.x, q.y, q.z, q.w};
    if (sizeof(T) == 4) w[e & 3] = low_bits<T>();
    else w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | low_bits<T>() << 16 : (w[e >> 1] & 0xffff0000u) | low_bits<T>();
    q = make_uint4(w[0], w[1], w[2], w[3]);
}
// a piece's values in pairs
template <typename T> constexpr int kPairs = kPiece<T> / 2;
template <typename T> __device__ __forceinline__ void piece_pairs(const uint4 &p, Pair (&v)[kPairs<T>])
{
    const uint32_t w[4] = {p.x, p.y, p.z, p.w};
#pragma unroll
    for (int i = 0; i < kPairs<T>; ++i) {
        if (sizeof(T) == 4) v[i] = pair_of(__uint_as_float(w[2 * i & 3]), __uint_as_float(w[2 * i + 1 & 3]));
        else {
            float f[2];
            two_values<T>(w[i & 3], f);
            v[i] = pair_of(f[0], f[1]);
        }
    }
}
template <typename T> __device__ __forceinline__ uint4 pairs_piece(const Pair (&v)[kPairs<T>])
{
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < kPairs<T>; ++i) {
        float f[2];
        split(v[i], f[0], f[1]);
        if (sizeof(T) == 4) w[2 * i & 3] = __float_as_uint(f[0]), w[2 * i + 1 & 3] = __float_as_uint(f[1]);
        else w[i & 3] = two_word<T>(f);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}
// adds the exponentials of a piece's values with respect to R / c
template <typename T> __device__ __forceinline__ void piece_exp_sum(Pair (&l)[2], const uint4 &p, Pair minus_R, Pair c)
{
    Pair v[kPairs<T>];
    piece_pairs<T>(p, v);
#pragma unroll
    for (int i = 0; i < kPairs<T>; ++i) l[i & 1] = l[i & 1] + ex2(fma2(v[i], c, minus_R));
}
// the classes whose bits are set become -inf
template <typename T> __device__ __forceinline__ void strike_out(uint4 *q, uint32_t bits, int pieces)
{
    if (bits)
#pragma unroll
        for (int i = 0; i < pieces; ++i)
            if ((bits >> (i * kPiece<T>)) & ((1u << kPiece<T>) - 1))
#pragma unroll
                for (int e = 0; e < kPiece<T>; ++e)
                    if ((bits >> (i * kPiece<T> + e)) & 1) drop_value<T>(q[i], e);
}
template <typename T> __device__ __forceinline__ uint32_t piece_max(uint32_t top, const uint4 &q)
{
    return Word<T>::max(Word<T>::max(top, Word<T>::max(q.x, q.y)), Word<T>::max(q.z, q.w));
}
template <typename T> __device__ __forceinline__ float word_max(uint32_t w)
{
    float f[Word<T>::n];
    Word<T>::get(w, f);
    return fmaxf(f[0], f[Word<T>::n - 1]);
}

// the larger of two words' values, NaN above all
template <typename T> __device__ __forceinline__ uint32_t max_nan(uint32_t a, uint32_t b);
template <> __device__ __forceinline__ uint32_t max_nan<float>(uint32_t a, uint32_t b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(__uint_as_float(a)), "f"(__uint_as_float(b)));
    return __float_as_uint(r);
}
template <> __device__ __forceinline__ uint32_t max_nan<__half>(uint32_t a, uint32_t b) { return Word<__half>::to(__hmax2_nan(Word<__half>::of(a), Word<__half>::of(b))); }
template <> __device__ __forceinline__ uint32_t max_nan<__nv_bfloat16>(uint32_t a, uint32_t b)
{
    return Word<__nv_bfloat16>::to(__hmax2_nan(Word<__nv_bfloat16>::of(a), Word<__nv_bfloat16>::of(b)));
}
template <typename T> __device__ __forceinline__ uint32_t piece_max_nan(const uint4 &q) { return max_nan<T>(max_nan<T>(q.x, q.y), max_nan<T>(q.z, q.w)); }
// order_key of the larger value of such a word
template <typename T> __device__ __forceinline__ uint32_t word_key(uint32_t w)
{
    float f[Word<T>::n];
    Word<T>::get(w, f);
    const uint32_t a = order_key(f[0]);
    return Word<T>::n == 1 ? a : max(a, order_key(f[Word<T>::n - 1]));
}

// ---- (m, l) of exponents over lanes
__device__ __forceinline__ float exp_of(float v, float m, float c) { return ex2((v - m) * c); } // of v with respect to a finite m
// One fused multiply-add a value instead of a difference and a product: exp((v - m) / T) = exp2(v c - R) * fix with R = m c, rounded, and fix = 2^(R - m c),
// which the rounding of R left out.  Not where that rounding is no small number (from 2^27 on it may be above 8, from 2^31 on 2^(R - m c) leaves the floats, and an
// infinite factor makes NaN of a sum of 0): classes masked with -1e10 or the type's lowest value, or a bound far below all values.
struct ExpRef {
    float R, fix;
    bool far;
};
__device__ __forceinline__ ExpRef exp_ref(float m, float c)
{
    ExpRef r;
    r.R = m * c, r.far = !(fabsf(m) < 1e38f && fabsf(r.R) < 0x1p27f), r.fix = ex2(-fmaf(m, c, -r.R));
    return r;
}
template <int LANES> __device__ __forceinline__ float lanes_max(float v) // NaN is passed over
{
    if constexpr (LANES == 32) { // one instruction for the warp
        float r;
        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
        return r;
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
        return v;
    }
}
template <int LANES> __device__ __forceinline__ float lanes_sum(float v)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
// the lanes' exponents as one: every lane of LANES neighbours gets it
template <int LANES> __device__ __forceinline__ ExpSum lanes_merge(ExpSum s, float c)
{
    const float m = lanes_max<LANES>(s.m);
    return {m, lanes_sum<LANES>(s.l * exp_of(s.m, finite_or_zero(m), c))};
}

// A row cut into trips of TH * NV pieces: those from `lo` on and below `hi` are whole, whichever thread asks.
template <typename T, int TH, int NV> struct RowTrips {
    static constexpr int kBytes = TH * NV * 16;
    const char *first; // the thread's piece 0 of trip 0 (not to be read unless trip 0 is whole)
    int lo, hi;
    RowTrips() = default;
    __device__ __forceinline__ RowTrips(const T *row, int classes)
    {
        const int phase = (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
        first = reinterpret_cast<const char *>(row) - phase * (int)sizeof(T) + threadIdx.x * 16;
        lo = phase ? 1 : 0, hi = (int)(((long long)classes + phase) / (kBytes / (int)sizeof(T)));
    }
    __device__ __forceinline__ bool whole(int trip) const { return trip >= lo && trip < hi; }
    __device__ __forceinline__ const char *at(int trip) const { return first + (long long)trip * kBytes; }
};

// Batcher's odd-even merge sort of N elements: `order(i, j)`, i < j, puts the pair in order
template <int N, typename F> __device__ __forceinline__ void odd_even_merges(F &&order)
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int d = p; d >= 1; d /= 2)
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i >= d % p && (i - d % p) / d % 2 == 0 && i + d < N && i / (2 * p) == (i + d) / (2 * p)) order(i, i + d);
}

} // namespace clb

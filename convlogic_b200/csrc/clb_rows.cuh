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
    __device__ __forceinline__ uint4 load(int j) const
    {
        if (whole(j)) return __ldcs(reinterpret_cast<const uint4 *>(row + first(j)));
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
template <typename T> __device__ __forceinline__ void drop_value(uint32_t (&w)[4], int e)
{
    if (sizeof(T) == 4) w[e & 3] = low_bits<T>();
    else w[e >> 1] = (e & 1) ? (w[e >> 1] & 0xffffu) | low_bits<T>() << 16 : (w[e >> 1] & 0xffff0000u) | low_bits<T>();
}

// ---- sums and maxima over a team of TH threads
template <int TH, bool MAX, int N> __device__ __forceinline__ void lanes_reduce(float (&v)[N])
{
#pragma unroll
    for (int o = (TH < 32 ? TH : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float other = __shfl_xor_sync(0xffffffffu, v[i], o);
            v[i] = MAX ? fmaxf(v[i], other) : v[i] + other;
        }
}
// `red`: N * 32 floats of the block, not in use by an earlier reduction that some thread may still read
template <int TH, bool MAX, int N> __device__ __forceinline__ void team_reduce(float (&v)[N], float *red)
{
    lanes_reduce<TH, MAX, N>(v);
    if (TH > 32) {
        constexpr int W = TH > 32 ? TH / 32 : 1;
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (lane == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) red[i * 32 + warp] = v[i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = red[i * 32 + lane % W];
        lanes_reduce<W, MAX, N>(v);
    }
}

} // namespace clb

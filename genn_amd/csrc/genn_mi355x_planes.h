// Part of libgenn_mi355x.so: matrix products of fp32 accuracy on the bf16 matrix instructions.
//
// A float is a sum of three bf16 values without a rest ("planes").  Of the nine products of two such sums the six whose planes' numbers add up to 2 at most are taken.  What the others are
// depends on how the planes were cut.  Rounded to the nearest, they leave at most 2^-8 and 2^-17 of the float's power of two, of either sign: the others are together 2^-24 of the product of the powers of two at most.
// Cut off, they leave up to 2^-7 and 2^-15, of the float's sign: 2^-21, and always too little, which does not average out.  So in every product of three planes by more than one an operand
// is rounded: 2^-24 if both are (or the other one is an fp16 input), 3 x 2^-24 if the other one is cut off, of either sign.  Where the other one is a single plane nothing is left out, and cutting off takes
// fewer cycles (prompts of 4096 rows x 32 heads in bf16: 217.5 us so, 223.5 with all rounded).  Rounded floats from 2^128 - 2^119 on count as an overflow.  A bf16 input is one plane, an fp16
// input two, so that most products take three to five instructions: 16 x 16 x 32 in 16 cycles each, where the same on the fp32 matrix
// instructions takes eight of 32.
#ifndef GENN_MI355X_PLANES_H
#define GENN_MI355X_PLANES_H

#include "genn_mi355x_elements.h"

namespace gennmi_planes
{
using gennmi_elements::bf16;
using gennmi_elements::f16;
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

template<typename T> constexpr int planesOf = 3;
template<> constexpr int planesOf<f16> = 2;
template<> constexpr int planesOf<bf16> = 1;

// Eight values along the axis that is summed over: an operand of one lane
template<int N> struct Planes { union { uint32_t word[4]; bf16x8 v; } plane[N]; };

// Takes the upper plane of a pair of values off them: its bits, the first value's below
template<bool ROUNDED> __device__ inline uint32_t takePlane(float &a, float &b)
{
    if constexpr(ROUNDED) {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        const uint32_t plane = __builtin_bit_cast(uint32_t, bf16x2{(bf16)a, (bf16)b});
        a -= __uint_as_float(plane << 16);
        b -= __uint_as_float(plane & 0xffff0000u);
        return plane;
    }
    const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
    a -= __uint_as_float(x & 0xffff0000u);
    b -= __uint_as_float(y & 0xffff0000u);
    return __builtin_amdgcn_perm(y, x, 0x07060302u);
}
// (the last plane: what is left has no more bits than a bf16, and nothing of it is needed afterwards)
__device__ inline uint32_t lastPlane(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
// (two planes hold an fp16 input without a rest, rounded or not)
template<int N, bool ROUNDED> __device__ inline void splitPair(float a, float b, uint32_t (&words)[N])
{
    #pragma unroll
    for(int p = 0; p < N; p++) { words[p] = p + 1 < N ? takePlane<ROUNDED>(a, b) : lastPlane(a, b); }
}
// Four values, N planes of 8 bytes
template<int N, bool ROUNDED = N == 3> __device__ inline void splitFour(const float (&x)[4], uint2 (&out)[N])
{
    uint32_t low[N], high[N];
    splitPair<N, ROUNDED>(x[0], x[1], low);
    splitPair<N, ROUNDED>(x[2], x[3], high);
    #pragma unroll
    for(int p = 0; p < N; p++) { out[p] = make_uint2(low[p], high[p]); }
}
// Eight values of one lane, four of each of two tiles of a result, which become an operand: see rowIn()
template<int N, bool ROUNDED = N == 3> __device__ inline Planes<N> split(const f32x4 &a, const f32x4 &b)
{
    Planes<N> out;
    const float x[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    #pragma unroll
    for(int i = 0; i < 4; i++) {
        uint32_t words[N];
        splitPair<N, ROUNDED>(x[2 * i], x[2 * i + 1], words);
        #pragma unroll
        for(int p = 0; p < N; p++) { out.plane[p].word[i] = words[p]; }
    }
    return out;
}
// A lane of a result tile has rows 4 (lane / 16) + 0 .. 3 of it, column lane % 16; an operand's lane has eight neighbours (8 (lane / 16) + 0 .. 7) along the axis that
// is summed over.  So that results become operands where they are, two tiles t, t + 1 (t even) hold 32 rows in this order: row i of tile t is row
// 8 (i / 4) + 4 (t % 2) + i % 4 of them.  A lane's eight values of both are neighbours then.
__device__ inline uint32_t rowIn(uint32_t t, uint32_t i) { return 32 * (t / 2) + 8 * (i / 4) + 4 * (t % 2) + i % 4; }

// Rows of WIDTH elements of 16 bits in LDS without a gap, units of 16 bytes in an order that differs from row to row, so that neither reads of a unit from 8 rows
// in that order, two a row, nor reads of four elements from each of four rows meet in a bank (64 of 4 bytes: 16 units).
template<int WIDTH> __device__ inline uint32_t unitAt(uint32_t row, uint32_t unit)
{
    constexpr int UNITS = WIDTH / 8;
    static_assert(UNITS == 4 || UNITS == 8 || UNITS == 16, "");
    const uint32_t turn = (UNITS == 16 ? (row & 3) << 2 : UNITS == 8 ? (row & 2) << 1 : 0) | ((row >> 2) & 2);
    return row * WIDTH + ((unit ^ turn) << 3);
}
// One unit of every plane
template<int N> __device__ inline Planes<N> fetch(const uint16_t *at, uint32_t stride)
{
    Planes<N> out;
    #pragma unroll
    for(int p = 0; p < N; p++) {
        out.plane[p].v = *(const bf16x8*)(at + p * stride);
    }
    return out;
}
// Four neighbouring rows of one column.  The lanes of a quarter of the wavefront each name four neighbours of a row, lane l those that begin at column 4 (l % 4) of row l / 4; lane l gets
// column l of the four rows.
__device__ inline uint2 readColumn(const uint16_t *at)
{
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    const s16x4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)at);
    return __builtin_bit_cast(uint2, x);
}
// Eight neighbouring rows of one column of every plane: `first` names rows 0 .. 3 of them, `second` rows 4 .. 7
template<int N> __device__ inline Planes<N> fetchColumn(const uint16_t *first, const uint16_t *second, uint32_t stride)
{
    Planes<N> out;
    #pragma unroll
    for(int p = 0; p < N; p++) {
        const uint2 a = readColumn(first + p * stride), b = readColumn(second + p * stride);
        out.plane[p].word[0] = a.x; out.plane[p].word[1] = a.y; out.plane[p].word[2] = b.x; out.plane[p].word[3] = b.y;
    }
    return out;
}
// sum += a b, the smallest products first
template<int NA, int NB> __device__ inline f32x4 multiply(const Planes<NA> &a, const Planes<NB> &b, f32x4 sum)
{
    #pragma unroll
    for(int total = 2; total >= 0; total--) {
        #pragma unroll
        for(int i = 0; i < NA; i++) {
            if(total - i >= 0 && total - i < NB) { sum = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.plane[i].v, b.plane[total - i].v, sum, 0, 0, 0); }
        }
    }
    return sum;
}
// sum[m] += a[m] b for several tiles: product after product, so that none waits for the one before it (a product takes 16 cycles, its sum is there after more than that)
template<int NA, int NB, int M> __device__ inline void multiplyAll(const Planes<NA> (&a)[M], const Planes<NB> &b, f32x4 (&sum)[M])
{
    #pragma unroll
    for(int total = 2; total >= 0; total--) {
        #pragma unroll
        for(int i = 0; i < NA; i++) {
            if(total - i < 0 || total - i >= NB) { continue; }
            #pragma unroll
            for(int m = 0; m < M; m++) { sum[m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[m].plane[i].v, b.plane[total - i].v, sum[m], 0, 0, 0); }
        }
    }
}
// Three sums at once, in turn
template<int NA> __device__ inline void multiplyThree(const Planes<NA> &a, const Planes<3> &b, f32x4 &x, const Planes<3> &c, const Planes<3> &d, f32x4 &y, const Planes<3> &e, const Planes<3> &f, f32x4 &z)
{
    #pragma unroll
    for(int total = 2; total >= 0; total--) {
        #pragma unroll
        for(int i = 0; i <= total; i++) {
            if(i < NA) { x = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a.plane[i].v, b.plane[total - i].v, x, 0, 0, 0); }
            y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(c.plane[i].v, d.plane[total - i].v, y, 0, 0, 0);
            z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e.plane[i].v, f.plane[total - i].v, z, 0, 0, 0);
        }
    }
}
// sum += a b for 16 x 16 tiles in fp32: a's lane has row lane % 16, its columns 4 (lane / 16) + 0 .. 3; b is a result
__device__ inline f32x4 multiply(const f32x4 &a, const f32x4 &b, f32x4 sum)
{
    #pragma unroll
    for(int e = 0; e < 4; e++) { sum = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], sum, 0, 0, 0); }
    return sum;
}
// Eight neighbouring elements, as they lie in memory
template<typename T> struct Eight
{
    u32x4 word[sizeof(T) / 2];
    __device__ T at(int i) const
    {
        const int byte = i * sizeof(T);
        const uint32_t w = word[byte / 16][byte % 16 / 4];
        if constexpr(sizeof(T) == 4) { return __builtin_bit_cast(T, w); }
        else { return __builtin_bit_cast(T, (uint16_t)(w >> (byte % 4 * 8))); }
    }
};
// `valid` of them, one by one, zero behind those
template<typename T> __device__ inline Eight<T> loadEight(const T *at, uint32_t valid)
{
    Eight<T> out{};
    #pragma unroll
    for(int i = 0; i < 8; i++) {
        if((uint32_t)i >= valid) { continue; }
        const int byte = i * sizeof(T);
        if constexpr(sizeof(T) == 4) { out.word[byte / 16][byte % 16 / 4] = __builtin_bit_cast(uint32_t, at[i]); }
        else { out.word[byte / 16][byte % 16 / 4] |= (uint32_t)__builtin_bit_cast(uint16_t, at[i]) << (byte % 4 * 8); }
    }
    return out;
}
// All or none, from an address on 16 bytes where something lies; or one by one
template<typename T> __device__ inline Eight<T> loadUnit(const T *at, uint32_t valid, bool wide)
{
    if(!wide) { return loadEight(at, valid); }
    Eight<T> out = *(const Eight<T>*)at;
    if(!valid) { out = Eight<T>{}; }
    return out;
}
// A unit of every plane
template<typename T> __device__ inline void storeUnit(uint16_t *to, uint32_t stride, const Eight<T> &x)
{
    constexpr int N = planesOf<T>;
    if constexpr(N == 1) { *(u32x4*)to = x.word[0]; }
    else {
        float low[4], high[4];
        #pragma unroll
        for(int e = 0; e < 4; e++) { low[e] = gennmi_elements::widen(x.at(e)); high[e] = gennmi_elements::widen(x.at(4 + e)); }
        uint2 a[N], b[N];
        splitFour<N>(low, a);
        splitFour<N>(high, b);
        #pragma unroll
        for(int p = 0; p < N; p++) { *(u32x4*)(to + p * stride) = u32x4{a[p].x, a[p].y, b[p].x, b[p].y}; }
    }
}
}

#endif

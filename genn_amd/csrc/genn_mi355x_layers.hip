// Layer norm with its gradients, and dropout.
#include <cmath>
#include <type_traits>

#define GENNMI_ROWS_THROUGHPUT
#include "genn_mi355x_elements.h"
#include "genn_mi355x_lanes.h"
#include "genn_mi355x_rows.h"

using namespace gennmi_elements;
using gennmi_detail::fail;
using gennmi_lanes::partner;

namespace
{
// ---- layer norm
// A row lies in the registers of the lanes that share it: 16 or 64 of a wavefront, or several wavefronts, each with 8 or 16 elements of it, so that it is read once and its
// statistics are those of its elements as they are: first the mean, then what is left of the elements, its squares and its own mean, which is what the first mean was rounded by: of rows far from zero
// (1000 and a spread of 0.01, say) steps of a mean in fp32 are as large as what is left.  Where wavefronts share a row, each finds these for its own part, and the parts are joined
// (Chan, Golub, LeVeque: sum of squares = sum over parts of their own and of count (mean of the part - mean)^2): one barrier a row instead of two.
struct NormArgs
{
    gennmi_rows_t x, gate, out;
    const float *weight, *bias;
    uint32_t rows, length, channels, rms, lanes;        // lanes: of a row
    float epsilon, share;           // 1 / channels
    gennmi_rows_t dout, dx, dgate;
    float *sums;                    // of each work-group: weight's and bias's, [2][channels]
};
template<typename T> __device__ inline T *normRow(const gennmi_rows_t &r, uint32_t sequence, uint32_t row) { return (T*)r.data + (uint64_t)sequence * r.sequenceStride + (uint64_t)row * r.rowStride; }

// Where a thread stands: `lane` of the `lanes` of the row of `group`, one of `groups` of the work-group
struct NormPlace { uint32_t lanes, lane, group, groups; };
template<int LANES> __device__ inline NormPlace normPlace(const NormArgs &a)
{
    constexpr uint32_t OWN = LANES ? LANES : 1;
    if(LANES) { return NormPlace{OWN, threadIdx.x % OWN, threadIdx.x / OWN, 256u / OWN}; }
    // (wavefronts have one row each)
    const uint32_t group = __builtin_amdgcn_readfirstlane(threadIdx.x / a.lanes);
    return NormPlace{a.lanes, threadIdx.x - group * a.lanes, group, blockDim.x / a.lanes};
}
template<int LANES> __device__ inline float sumOfLanes(float x)
{
    x += partner<1>(x); x += partner<2>(x); x += partner<4>(x); x += partner<8>(x);
    if(LANES != 16) { x += partner<16>(x); x += partner<32>(x); }
    return x;
}
// What a row's wavefronts found; two places in LDS are used in turn, so that one barrier does
constexpr int NORM_APART = 1024;        // a lane's sums in LDS, in elements: a constant costs no register a place
struct NormShared { float4 found[2][16]; };

template<typename T, int E, int VEC> struct NormRow { Pack<T, VEC> part[E / VEC]; };
template<typename T, int E, int VEC> __device__ inline NormRow<T, E, VEC> requestRow(const T *row, const NormPlace &at, uint32_t channels, bool valid)
{
    NormRow<T, E, VEC> x;
    #pragma unroll
    for(int i = 0; i < E / VEC; i++) {
        const uint32_t c = (i * at.lanes + at.lane) * VEC;
        x.part[i] = Pack<T, VEC>{};
        if(valid && c < channels) { x.part[i] = *(const Pack<T, VEC>*)(row + c); }
    }
    return x;
}
template<typename T, int E, int VEC> __device__ inline void takeRow(const NormRow<T, E, VEC> &from, float (&x)[E])
{
    #pragma unroll
    for(int e = 0; e < E; e++) { x[e] = widen(from.part[e / VEC].v[e % VEC]); }
}
template<typename T, int E, int VEC> __device__ inline void storeRow(T *row, const NormPlace &at, uint32_t channels, const float (&x)[E])
{
    #pragma unroll
    for(int i = 0; i < E / VEC; i++) {
        const uint32_t c = (i * at.lanes + at.lane) * VEC;
        if(c >= channels) { continue; }
        Pack<T, VEC> p;
        #pragma unroll
        for(int e = 0; e < VEC; e++) { p.v[e] = narrow<T>(x[i * VEC + e]); }
        *(Pack<T, VEC>*)(row + c) = p;
    }
}
template<int E, int VEC> __device__ inline void loadParameters(const float *from, float without, const NormPlace &at, uint32_t channels, float (&x)[E])
{
    constexpr int EACH = VEC < 4 ? 1 : 4;
    const bool wide = (uintptr_t)from % 16 == 0;
    #pragma unroll
    for(int i = 0; i < E; i += EACH) {
        const uint32_t c = (i / VEC * at.lanes + at.lane) * VEC + i % VEC;
        #pragma unroll
        for(int e = 0; e < EACH; e++) { x[i + e] = c < channels ? without : 0.0f; }
        if(!from || c >= channels) { continue; }
        if(wide) {
            const Pack<float, EACH> p = *(const Pack<float, EACH>*)(from + c);
            #pragma unroll
            for(int e = 0; e < EACH; e++) { x[i + e] = p.v[e]; }
        }
        else {
            #pragma unroll
            for(int e = 0; e < EACH; e++) { x[i + e] = from[c + e]; }
        }
    }
}
template<int E, int VEC> __device__ inline bool hasElement(const NormPlace &at, int e, uint32_t channels) { return (e / VEC * at.lanes + at.lane) * VEC + e % VEC < channels; }
// Elements that a row's wavefront has
template<int E, int VEC> __device__ inline float elementsOf(const NormPlace &at, uint32_t wave, uint32_t channels)
{
    uint32_t n = 0;
    #pragma unroll
    for(int i = 0; i < E / VEC; i++) {
        const uint32_t first = (i * at.lanes + 64 * wave) * VEC;
        n += first < channels ? min(channels - first, 64u * VEC) : 0;
    }
    return (float)n;
}

// x becomes x'; what it is divided by is returned as a factor
template<int LANES, int E, int VEC> __device__ inline float normalise(const NormArgs &a, float (&x)[E], const NormPlace &at, NormShared &shared, uint32_t &turn, float inWave, float inWaveShare)
{
    float left = 0.0f, square = 0.0f, mean = 0.0f;
    const float share = LANES ? a.share : inWaveShare;
    if(a.rms) {
        #pragma unroll
        for(int e = 0; e < E; e++) { square = __builtin_fmaf(x[e], x[e], square); }
    }
    else {
        float sum = 0.0f;
        #pragma unroll
        for(int e = 0; e < E; e++) { sum += x[e]; }
        mean = sumOfLanes<LANES>(sum) * share;
        #pragma unroll
        for(int i = 0; i < E; i += VEC) {
            if(!hasElement<E, VEC>(at, i, a.channels)) { continue; }
            #pragma unroll
            for(int e = i; e < i + VEC; e++) {
                x[e] -= mean;
                square = __builtin_fmaf(x[e], x[e], square);
                left += x[e];
            }
        }
    }
    square = sumOfLanes<LANES>(square);
    float off = 0.0f;               // of what is left
    if(!a.rms) {
        left = sumOfLanes<LANES>(left);
        off = left * share;
        square = __builtin_fmaf(-left, off, square);
    }
    if(LANES == 0 && at.lanes > 64) {
        const uint32_t waves = at.lanes >> 6, first = at.group * waves, mine = threadIdx.x >> 6, other = threadIdx.x & 15;
        if((threadIdx.x & 63) == 0) { shared.found[turn][mine] = make_float4(mean, square, off, inWave); }
        __syncthreads();
        // (a lane of each 16 has one wavefront's)
        const float4 f = other < waves ? shared.found[turn][first + other] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if(a.rms) { square = sumOfLanes<16>(f.y); }
        else {
            const float whole = sumOfLanes<16>(f.w * f.x) * a.share, o = f.x - whole + f.z;
            const float all = sumOfLanes<16>(f.w * o);
            square = __builtin_fmaf(-all, all * a.share, sumOfLanes<16>(__builtin_fmaf(f.w * o, o, f.y)));
            // (x is without this wavefront's mean, not the row's)
            off = all * a.share - (mean - whole);
        }
        turn ^= 1;
    }
    if(square < 0.0f) { square = 0.0f; }        // (what was taken off twice is as large as all of it)
    // (a root and a division, and what both were rounded by: r is in all elements of the row)
    const float variance = __builtin_fmaf(square, a.share, a.epsilon);
    float r = 1.0f / sqrtf(variance);
    const float one = variance * r, less = __builtin_fmaf(-one, r, 1.0f) - __builtin_fmaf(variance, r, -one) * r;
    if(fabsf(less) < 1.0f) { r = __builtin_fmaf(0.5f * r, less, r); }
    // (of elements behind the last channel something is left: their weights and what comes in for them are zero, and nothing of them is stored)
    #pragma unroll
    for(int e = 0; e < E; e++) { x[e] = (x[e] - off) * r; }
    return r;
}
// s = sigmoid(z) and 1 - s.  For results in 16 bits the hardware's exponential of a rounded product (off by |z| / 2 half steps of fp32) and its reciprocal are more than enough; a division and an exponential to
// the last bit were a third of the instructions of a gated row.  For fp32: of u = exp(-z), a power of two and a rest below one half whose product with log2(e) has two parts, s is 1 / (1 + u) and 1 - s is
// u / (1 + u): both are within a few half steps of themselves.
struct Logistic { float s, rest; };
template<typename T> __device__ inline Logistic logistic(float z)
{
    if constexpr(sizeof(T) < 4) {
        const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(z * -1.44269504f));
        return Logistic{s, 1.0f - s};
    }
    // (behind 200 u is 0 or infinite; a z that is no number is one in what s is multiplied with)
    const float m = fmaxf(fminf(z, 200.0f), -200.0f), whole = rintf(m * -1.44269502f), part = __builtin_fmaf(m, -1.925963e-8f, __builtin_fmaf(m, -1.44269502f, -whole));
    const float u = __builtin_ldexpf(__builtin_amdgcn_exp2f(part), (int)whole), s = __builtin_amdgcn_rcpf(1.0f + u);
    return Logistic{s, fminf(u * s, 1.0f)};         // (1 where u is infinite)
}

// Bound by memory: each row is read once and written once.  Work-groups of 256 threads where 16 lanes or a wavefront have a row, else of what rows take; each walks rows that are a grid apart,
// with the parameters in registers and the next row asked for while one is worked on.  4096 x 4096 in bf16: 62 us with a row a work-group (its parameters are four times the row), 13.9 so (4.8 TB/s);
// 131,072 heads of 128 with a gate 20.5 (4.9 TB/s).
template<typename T, int LANES, int E, int VEC, bool GATE>
__global__ __launch_bounds__(LANES ? 256 : 1024)
void normKernel(NormArgs a)
{
    __shared__ NormShared shared;
    uint32_t turn = 0;
    const NormPlace at = normPlace<LANES>(a);
    float weight[E], bias[E];
    loadParameters<E, VEC>(a.weight, 1.0f, at, a.channels, weight);
    loadParameters<E, VEC>(a.bias, 0.0f, at, a.channels, bias);
    const float inWave = LANES ? 0.0f : elementsOf<E, VEC>(at, at.lane >> 6, a.channels), inWaveShare = inWave > 0.0f ? 1.0f / inWave : 0.0f;
    const uint64_t step = (uint64_t)gridDim.x * at.groups;
    // (a gate's elements one by one, with the places of them all, are more than the registers of 16 wavefronts hold ahead of time)
    constexpr bool AHEAD = LANES || VEC > 1;
    NormRow<T, E, VEC> nextX, nextZ{};
    const auto request = [&](uint64_t n, bool x, bool z) {
        const bool valid = n < a.rows;
        const uint32_t sequence = valid ? (uint32_t)n / a.length : 0, row = valid ? (uint32_t)n - sequence * a.length : 0;
        if(x) { nextX = requestRow<T, E, VEC>(normRow<const T>(a.x, sequence, row), at, a.channels, valid); }
        if constexpr(GATE) { if(z) { nextZ = requestRow<T, E, VEC>(normRow<const T>(a.gate, sequence, row), at, a.channels, valid); } }
    };
    uint64_t first = (uint64_t)blockIdx.x * at.groups;
    request(first + at.group, true, AHEAD);
    for(; first < a.rows; first += step) {
        const uint64_t n = first + at.group;
        float x[E], z[E];
        takeRow(nextX, x);
        if constexpr(GATE && AHEAD) { takeRow(nextZ, z); }
        request(n + step, true, AHEAD);
        normalise<LANES, E, VEC>(a, x, at, shared, turn, inWave, inWaveShare);
        if constexpr(GATE && !AHEAD) { request(n, false, true); takeRow(nextZ, z); }
        #pragma unroll
        for(int e = 0; e < E; e++) {
            x[e] = __builtin_fmaf(x[e], weight[e], bias[e]);
            if constexpr(GATE) { x[e] *= z[e] * logistic<T>(z[e]).s; }
        }
        if(n < a.rows) {
            const uint32_t sequence = (uint32_t)n / a.length, row = (uint32_t)n - sequence * a.length;
            storeRow<T, E, VEC>(normRow<T>(a.out, sequence, row), at, a.channels, x);
        }
    }
}

// With y = x' weight + bias, s the gate's factor z sigmoid(z) and d = dout s:
// Bound by memory: 16384 x 2048 in bf16 51 us with the closing sums (3.9 TB/s), 134 with a row's sums over its work-group one behind another.
//   dgate = dout y s',  dweight += d x',  dbias += d,  dx = (v - x' mean(v x') - mean(v)) / length, v = d weight (without the last mean for `rms`)
template<typename T, int LANES, int E, int VEC, bool GATE>
__global__ __launch_bounds__(LANES ? 256 : 1024)
void normBackwardKernel(NormArgs a)
{
    __shared__ NormShared shared;
    extern __shared__ float rows[];
    uint32_t turn = 0;
    const NormPlace at = normPlace<LANES>(a);
    // (16 elements a lane, above 8192 channels, leave 16 wavefronts no registers for the sums, which lie in LDS, nor for the next row or a gate's bias)
    constexpr bool LARGE = LANES == 0 && E == 16, BIAS_AGAIN = LARGE && VEC == 8;
    float weight[E], bias[GATE ? E : 1], dweight[LARGE ? 1 : E] = {}, dbias[LARGE ? 1 : E] = {};
    constexpr int APART = NORM_APART;
    float *const sums[2] = {rows + threadIdx.x, rows + E * APART + threadIdx.x};
    if constexpr(LARGE) {
        #pragma unroll
        for(int e = 0; e < E; e++) { sums[0][e * APART] = sums[1][e * APART] = 0.0f; }
    }
    loadParameters<E, VEC>(a.weight, 1.0f, at, a.channels, weight);
    if constexpr(GATE && !BIAS_AGAIN) { loadParameters<E, VEC>(a.bias, 0.0f, at, a.channels, bias); }
    const float inWave = LANES ? 0.0f : elementsOf<E, VEC>(at, at.lane >> 6, a.channels), inWaveShare = inWave > 0.0f ? 1.0f / inWave : 0.0f;
    const uint64_t step = (uint64_t)gridDim.x * at.groups;
    NormRow<T, E, VEC> nextX, nextD;
    const auto request = [&](uint64_t n) {
        const bool valid = n < a.rows;
        const uint32_t sequence = valid ? (uint32_t)n / a.length : 0, row = valid ? (uint32_t)n - sequence * a.length : 0;
        nextX = requestRow<T, E, VEC>(normRow<const T>(a.x, sequence, row), at, a.channels, valid);
        nextD = requestRow<T, E, VEC>(normRow<const T>(a.dout, sequence, row), at, a.channels, valid);
    };
    uint64_t first = (uint64_t)blockIdx.x * at.groups;
    if(!LARGE) { request(first + at.group); }
    for(; first < a.rows; first += step) {
        const uint64_t n = first + at.group;
        const bool valid = n < a.rows;
        if(LARGE) { request(n); }
        const uint32_t sequence = valid ? (uint32_t)n / a.length : 0, row = valid ? (uint32_t)n - sequence * a.length : 0;
        float x[E], d[E];
        takeRow(nextX, x);
        takeRow(nextD, d);
        NormRow<T, E, VEC> gate{};
        if constexpr(GATE && !LARGE) { gate = requestRow<T, E, VEC>(normRow<const T>(a.gate, sequence, row), at, a.channels, valid); }
        if(!LARGE) { request(n + step); }
        const float r = normalise<LANES, E, VEC>(a, x, at, shared, turn, inWave, inWaveShare);
        if constexpr(GATE) {
            if constexpr(BIAS_AGAIN) { loadParameters<E, VEC>(a.bias, 0.0f, at, a.channels, bias); }
            // the gate's element becomes its gradient
            const auto pass = [&](int e, float &z) {
                const Logistic l = logistic<T>(z);
                const float y = __builtin_fmaf(x[e], weight[e], bias[e]), dz = d[e] * y * (l.s * __builtin_fmaf(z, l.rest, 1.0f));
                d[e] *= z * l.s;
                z = dz;
            };
            if constexpr(LARGE && sizeof(T) == 4) {
                // (no registers for a whole row of it and what fp32 takes for each: four elements at a time)
                const T *const from = normRow<const T>(a.gate, sequence, row);
                T *const to = normRow<T>(a.dgate, sequence, row);
                #pragma unroll
                for(int i = 0; i < E; i += 4) {
                    __builtin_amdgcn_sched_barrier(0);
                    Pack<T, VEC> z[4 / VEC];
                    #pragma unroll
                    for(int k = 0; k < 4; k += VEC) {
                        z[k / VEC] = Pack<T, VEC>{};
                        if(valid && hasElement<E, VEC>(at, i + k, a.channels)) { z[k / VEC] = *(const Pack<T, VEC>*)(from + ((i + k) / VEC * at.lanes + at.lane) * VEC); }
                    }
                    #pragma unroll
                    for(int k = 0; k < 4; k++) { pass(i + k, z[k / VEC].v[k % VEC]); }
                    #pragma unroll
                    for(int k = 0; k < 4; k += VEC) {
                        if(a.dgate.data && valid && hasElement<E, VEC>(at, i + k, a.channels)) { *(Pack<T, VEC>*)(to + ((i + k) / VEC * at.lanes + at.lane) * VEC) = z[k / VEC]; }
                    }
                }
            }
            else {
                if constexpr(LARGE) { gate = requestRow<T, E, VEC>(normRow<const T>(a.gate, sequence, row), at, a.channels, valid); }
                float z[E];
                takeRow(gate, z);
                #pragma unroll
                for(int e = 0; e < E; e++) {
                    if(LARGE && e % 4 == 0) { __builtin_amdgcn_sched_barrier(0); }
                    pass(e, z[e]);
                }
                if(a.dgate.data && valid) { storeRow<T, E, VEC>(normRow<T>(a.dgate, sequence, row), at, a.channels, z); }
            }
        }
        // (of a row that is not there d is zero)
        float along = 0.0f, mean = 0.0f;
        #pragma unroll
        for(int e = 0; e < E; e++) {
            if constexpr(LARGE) {
                if(e % 4 == 0) { __builtin_amdgcn_sched_barrier(0); }
                sums[0][e * APART] = __builtin_fmaf(d[e], x[e], sums[0][e * APART]);
                sums[1][e * APART] += d[e];
            }
            else {
                if(valid) { dweight[e] = __builtin_fmaf(d[e], x[e], dweight[e]); }
                dbias[e] += d[e];
            }
            d[e] *= weight[e];
            along = __builtin_fmaf(d[e], x[e], along);
            mean += d[e];
        }
        if(!a.dx.data) { continue; }
        along = sumOfLanes<LANES>(along);
        mean = sumOfLanes<LANES>(mean);
        if constexpr(LANES == 0) {
            const uint32_t waves = at.lanes >> 6;
            if((threadIdx.x & 63) == 0) { shared.found[turn][threadIdx.x >> 6] = make_float4(along, mean, 0.0f, 0.0f); }
            __syncthreads();
            along = mean = 0.0f;
            for(uint32_t w = 0; w < waves; w++) { const float4 f = shared.found[turn][at.group * waves + w]; along += f.x; mean += f.y; }
            turn ^= 1;
        }
        along *= a.share;
        mean = a.rms ? 0.0f : mean * a.share;
        #pragma unroll
        for(int e = 0; e < E; e++) { x[e] = r * (__builtin_fmaf(-x[e], along, d[e]) - mean); }
        if(valid) { storeRow<T, E, VEC>(normRow<T>(a.dx, sequence, row), at, a.channels, x); }
    }
    if(!a.sums) { return; }
    float *const to = a.sums + (uint64_t)blockIdx.x * 2 * a.channels;
    #pragma unroll
    for(int which = 0; which < 2; which++) {
        float (&sum)[LARGE ? 1 : E] = which ? dbias : dweight;
        if constexpr(LARGE) {
            #pragma unroll
            for(int e = 0; e < E; e++) { if(hasElement<E, VEC>(at, e, a.channels)) { to[which * a.channels + (e / VEC * at.lanes + at.lane) * VEC + e % VEC] = sums[which][e * APART]; } }
            continue;
        }
        else if(at.groups > 1) {
            // (the rows of a work-group one after another)
            __syncthreads();
            #pragma unroll
            for(int e = 0; e < E; e++) { rows[e * blockDim.x + threadIdx.x] = sum[e]; }
            __syncthreads();
            if(at.group) { continue; }
            // (in 64 bits: in 32 their roundings were as much of the result's error as all of the rows')
            #pragma unroll 1
            for(int e = 0; e < E; e += 4) {
                double whole[4];
                #pragma unroll
                for(int i = 0; i < 4; i++) { whole[i] = rows[(e + i) * blockDim.x + at.lane]; }
                for(uint32_t k = 1; k < at.groups; k++) {
                    #pragma unroll
                    for(int i = 0; i < 4; i++) { whole[i] += rows[(e + i) * blockDim.x + k * at.lanes + at.lane]; }
                }
                #pragma unroll
                for(int i = 0; i < 4; i++) { rows[(e + i) * blockDim.x + at.lane] = (float)whole[i]; }
            }
            #pragma unroll
            for(int e = 0; e < E; e++) { sum[e] = rows[e * blockDim.x + at.lane]; }
        }
        if constexpr(!LARGE) {
            #pragma unroll
            for(int e = 0; e < E; e++) { if(hasElement<E, VEC>(at, e, a.channels)) { to[which * a.channels + (e / VEC * at.lanes + at.lane) * VEC + e % VEC] = sum[e]; } }
        }
    }
}

// ---- dropout
struct DropoutArgs
{
    gennmi_rows_t x, residual, out;
    const uint64_t *callDevice;
    uint64_t call;
    uint32_t k0, k1, items, groups, length, channels, dropped;
    float factor;
};
// A thread has eight neighbouring elements and draws once for them, 16 bits each (ten rounds of two wide products and four exclusive ors; a draw for four would take longer than the memory).
// Arrays beyond the caches are bound by memory: 32768 x 16384 in bf16 onto a residual 532 us, 6.06 TB/s, which is what adding the two takes (534).  Of what the last cache holds the draws are the limit, with the
// vector units 92 to 96 % busy: 16384 x 2048 31.3 us where adding takes 29.3; 38 with the arrays of other calls between.
template<typename T, bool WIDE>
__global__ __launch_bounds__(256)
void dropoutKernel(DropoutArgs a)
{
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    if(item >= a.items) { return; }
    const uint32_t n = item / a.groups, c = (item - n * a.groups) * 8, sequence = n / a.length, row = n - sequence * a.length;
    const uint64_t call = a.call + (a.callDevice ? *a.callDevice : 0);
    const T *const x = normRow<const T>(a.x, sequence, row) + c, *const residual = a.residual.data ? normRow<const T>(a.residual, sequence, row) + c : nullptr;
    T *const out = normRow<T>(a.out, sequence, row) + c;
    constexpr int EACH = WIDE ? 16 / sizeof(T) : 1;
    typedef Pack<T, EACH> P;
    P in[8 / EACH], more[8 / EACH] = {};
    #pragma unroll
    for(int i = 0; i < 8 / EACH; i++) {
        in[i] = P{};
        if(c + i * EACH < a.channels) {
            in[i] = *(const P*)(x + i * EACH);
            if(residual) { more[i] = *(const P*)(residual + i * EACH); }
        }
    }
    const gennmi_rows::Words words = gennmi_rows::philox4x32(item, 0, (uint32_t)call, (uint32_t)(call >> 32), a.k0, a.k1);
    #pragma unroll
    for(int i = 0; i < 8 / EACH; i++) {
        #pragma unroll
        for(int e = 0; e < EACH; e++) {
            const int k = i * EACH + e;
            const uint32_t bits = k % 2 ? words.w[k / 2] >> 16 : words.w[k / 2] & 0xffff;
            const float kept = bits >= a.dropped ? widen(in[i].v[e]) * a.factor : 0.0f;
            in[i].v[e] = narrow<T>(residual ? widen(more[i].v[e]) + kept : kept);
        }
        if(c + i * EACH < a.channels) { *(P*)(out + i * EACH) = in[i]; }
    }
}

// ---- what the entry points check
int checkPlainRows(const char *what, const gennmi_sequences_t &s)
{
    if(s.offsets || s.slots) { return fail(GENNMI_EINVAL, std::string(what) + ": rows are not packed here and have no slots"); }
    return checkSequences(what, s, false);
}
int checkNorm(const char *what, const gennmi_layer_norm_t *c, bool gradients)
{
    if(!c) { return fail(GENNMI_EINVAL, std::string(what) + ": null descriptor"); }
    const auto refuse = [&](int code, const char *why) { return fail(code, std::string(what) + why); };
    const uint32_t size = sizeOf(c->type);
    if(!size) { return refuse(GENNMI_EUNSUPPORTED, ": unknown element type"); }
    if(c->channels < 1 || c->channels > GENNMI_MAX_NORM_CHANNELS) { return refuse(GENNMI_EUNSUPPORTED, ": number of channels"); }
    if(!(c->epsilon >= 0.0f) || std::isinf(c->epsilon)) { return refuse(GENNMI_EINVAL, ": epsilon"); }
    if(const int rc = checkPlainRows(what, c->sequences)) { return rc; }
    if(const int rc = checkRows(what, "x", c->x, c->sequences, c->channels, size)) { return rc; }
    if(c->gate.data) { if(const int rc = checkRows(what, "gate", c->gate, c->sequences, c->channels, size)) { return rc; } }
    if(!gradients) { if(const int rc = checkWrittenRows(what, "out", c->out, c->sequences, c->channels, size)) { return rc; } }
    if((uintptr_t)c->weight % 4 || (uintptr_t)c->bias % 4) { return refuse(GENNMI_EINVAL, ": weight or bias not aligned"); }
    return GENNMI_OK;
}
// An array that may be written in place: element for element the same
Region unlessSameRows(const Region &r, const gennmi_rows_t &a, const gennmi_rows_t &written)
{
    return a.data == written.data && a.rowStride == written.rowStride && a.sequenceStride == written.sequenceStride ? Region{r.name, 0, 0, 0, 0, 0, 0, 0} : r;
}
// Rows one behind another are one sequence: what holds of every array of a call
bool oneBehindAnother(const gennmi_sequences_t &s, std::initializer_list<const gennmi_rows_t*> arrays)
{
    for(const gennmi_rows_t *r : arrays) { if(r->data && s.count > 1 && r->sequenceStride != s.length * r->rowStride) { return false; } }
    return true;
}
// Elements of an access: 16 bytes where every row of every array lies so, else one
uint32_t vectorOf(uint32_t size, uint32_t channels, std::initializer_list<const gennmi_rows_t*> arrays)
{
    const uint32_t vector = 16 / size;
    bool whole = channels % vector == 0;
    for(const gennmi_rows_t *r : arrays) { whole = whole && (!r->data || ((uintptr_t)r->data % 16 == 0 && r->rowStride % vector == 0 && r->sequenceStride % vector == 0)); }
    return whole ? vector : 1;
}
struct NormPlan { uint32_t each, lanes, rowLanes, groups, threads, blocks; };       // lanes 0: wavefronts share a row, rowLanes of them
// Rows of up to 128 channels: 16 lanes with 8 elements each; of up to 512: a wavefront.  Above that wavefronts share a row in the forward pass, 16 elements a lane; gradients of up to 1024 channels
// (2048 without a gate) stay with one wavefront, whose rows need no barrier, as long as its registers hold four arrays of them.  us in bf16: 16384 x 2048 a wavefront a row
// and two, forward 32, 28, gradients 50, 62; gradients of 16384 x 1024 29, 35, of 8192 x 2048 with a gate 67, 48
// (all of them before what the mean leaves was taken off: now forward 24, gradients 45, 27, 45 from the caches).
// Work-groups: as many as the chip holds at once, or a quarter of the rows where that is less, as each leaves a sum for every channel; more, where a lane would add up more than 256 rows in fp32 (what its
// lanes and the work-groups found is added up in 64 bits).
NormPlan normPlan(const gennmi_layer_norm_t &c, bool gradients)
{
    const uint64_t rows = totalRows(c.sequences);
    const bool gate = c.gate.data != nullptr;
    NormPlan p;
    p.lanes = c.channels <= 128 ? 16 : c.channels <= 512 || (gradients && c.channels <= (gate ? 1024u : 2048u)) ? 64 : 0;
    p.each = p.lanes ? (c.channels <= 512 ? 8 : c.channels <= 1024 ? 16 : 32) : gradients && c.channels <= 8192 ? 8 : 16;
    p.rowLanes = p.lanes ? p.lanes : ((c.channels + p.each - 1) / p.each + 63) / 64 * 64;
    p.groups = p.lanes ? 256 / p.lanes : std::max(1u, (gradients ? 512 : 256) / p.rowLanes);
    p.threads = p.groups * p.rowLanes;
    const uint64_t needed = (rows + p.groups - 1) / p.groups, most = gradients ? (p.each == 8 && (p.lanes || !gate) ? 768 : 512) : p.lanes ? 2048 : 1024;
    p.blocks = (uint32_t)std::min<uint64_t>(gradients ? (needed + 3) / 4 : needed, gradients ? std::max(most, std::min((needed + 255) / 256, mostBlocks(p.threads))) : most);
    return p;
}
template<bool GRADIENTS, int VEC, typename F> int withNormLayout(const NormPlan &p, F &&f)
{
    typedef std::integral_constant<int, VEC> Vec;
    const std::integral_constant<int, 8> eight;
    const std::integral_constant<int, 16> sixteen;
    if(p.lanes == 16) { return f(sixteen, eight, Vec{}); }
    if(p.lanes == 64) {
        const std::integral_constant<int, 64> wave;
        if constexpr(GRADIENTS) {
            if(p.each == 32) { return f(wave, std::integral_constant<int, 32>{}, Vec{}); }
            if(p.each == 16) { return f(wave, sixteen, Vec{}); }
        }
        return f(wave, eight, Vec{});
    }
    const std::integral_constant<int, 0> several;
    if constexpr(GRADIENTS) { if(p.each == 8) { return f(several, eight, Vec{}); } }
    return f(several, sixteen, Vec{});
}
template<bool GRADIENTS, typename F> int withNorm(const gennmi_layer_norm_t &c, const NormPlan &p, uint32_t vector, F &&f)
{
    return withType(c.type, [&](auto t) {
        typedef decltype(t) T;
        const auto g = [&](auto lanes, auto each, auto vec) {
            if(!c.gate.data) { return f(t, lanes, each, vec, std::false_type{}); }
            // (with a gate rows of 32 elements a lane are not planned)
            if constexpr(decltype(each)::value <= 16) { return f(t, lanes, each, vec, std::true_type{}); }
            else { return (int)GENNMI_EUNSUPPORTED; }
        };
        if(vector > 1) { return withNormLayout<GRADIENTS, 16 / sizeof(T)>(p, g); }
        return withNormLayout<GRADIENTS, 1>(p, g);
    });
}
NormArgs normArgs(const gennmi_layer_norm_t &c, const NormPlan &p, bool flat)
{
    NormArgs a{};
    a.x = c.x; a.gate = c.gate; a.out = c.out;
    a.weight = c.weight; a.bias = c.bias;
    a.rows = (uint32_t)totalRows(c.sequences);
    a.length = flat ? a.rows : c.sequences.length;
    a.channels = c.channels; a.rms = c.rms; a.lanes = p.rowLanes;
    a.epsilon = c.epsilon; a.share = 1.0f / (float)c.channels;
    return a;
}
}

extern "C" {

int gennmi_layer_norm(const gennmi_layer_norm_t *norm, void *stream)
{
    const char *what = "layer_norm";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkNorm(what, norm, false)) { return rc; }
        const gennmi_sequences_t &s = norm->sequences;
        const uint32_t size = sizeOf(norm->type);
        const uint64_t bytes = norm->channels * 4ull;
        if(const int rc = checkApart(what, {regionOf("out", norm->out, s, norm->channels, size)}, {},
                                     {unlessSameRows(regionOf("x", norm->x, s, norm->channels, size), norm->x, norm->out), unlessSameRows(regionOf("gate", norm->gate, s, norm->channels, size), norm->gate, norm->out),
                                      regionOf("weight", norm->weight, bytes), regionOf("bias", norm->bias, bytes)})) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, s.device)) { return rc; }
        if(!totalRows(s)) { return (int)GENNMI_OK; }
        const NormPlan p = normPlan(*norm, false);
        const auto arrays = {&norm->x, &norm->gate, &norm->out};
        const NormArgs a = normArgs(*norm, p, oneBehindAnother(s, arrays));
        const int rc = withNorm<false>(*norm, p, vectorOf(size, norm->channels, arrays), [&](auto t, auto lanes, auto each, auto vec, auto gate) {
            normKernel<decltype(t), decltype(lanes)::value, decltype(each)::value, decltype(vec)::value, decltype(gate)::value><<<dim3(p.blocks), dim3(p.threads), 0, (hipStream_t)stream>>>(a);
            return gennmi_detail::afterLaunch(what);
        });
        if(rc) { return rc; }
        noteRows(norm->out, s, norm->channels, size);
        return (int)GENNMI_OK;
    });
}

int gennmi_layer_norm_backward_workspace(const gennmi_layer_norm_t *norm, size_t *bytes)
{
    return gennmi_detail::guarded("layer_norm_backward_workspace", [&] {
        if(const int rc = checkNorm("layer_norm_backward_workspace", norm, true)) { return rc; }
        if(!bytes) { return fail(GENNMI_EINVAL, "layer_norm_backward_workspace: null result pointer"); }
        *bytes = (size_t)normPlan(*norm, true).blocks * 2 * norm->channels * sizeof(float);
        return (int)GENNMI_OK;
    });
}

int gennmi_layer_norm_backward(const gennmi_layer_norm_t *norm, const gennmi_layer_norm_gradient_t *gradient, void *workspace, size_t workspaceBytes, void *stream)
{
    const char *what = "layer_norm_backward";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkNorm(what, norm, true)) { return rc; }
        if(!gradient) { return fail(GENNMI_EINVAL, "layer_norm_backward: null gradient"); }
        const gennmi_layer_norm_gradient_t &g = *gradient;
        const gennmi_sequences_t &s = norm->sequences;
        const uint32_t size = sizeOf(norm->type), channels = norm->channels;
        const uint64_t bytes = channels * 4ull;
        if(const int rc = checkRows(what, "the gradient of out", g.out, s, channels, size)) { return rc; }
        if(g.x.data) { if(const int rc = checkWrittenRows(what, "the gradient of x", g.x, s, channels, size)) { return rc; } }
        if(g.gate.data) { if(const int rc = checkWrittenRows(what, "the gradient of gate", g.gate, s, channels, size)) { return rc; } }
        if(g.gate.data && !norm->gate.data) { return fail(GENNMI_EINVAL, "layer_norm_backward: a gradient of gate without gate"); }
        if((uintptr_t)g.weight % 4 || (uintptr_t)g.bias % 4) { return fail(GENNMI_EINVAL, "layer_norm_backward: an array of fp32 is not aligned"); }
        const NormPlan p = normPlan(*norm, true);
        const bool sums = g.weight || g.bias;
        const size_t need = sums ? (size_t)p.blocks * 2 * channels * sizeof(float) : 0;
        if(const int rc = checkWorkspace(what, workspace, workspaceBytes, need)) { return rc; }
        if(const int rc = checkApart(what, {regionOf("the gradient of x", g.x, s, channels, size), regionOf("the gradient of gate", g.gate, s, channels, size), regionOf("the workspace", workspace, need)},
                                     {regionOf("the gradient of weight", g.weight, bytes), regionOf("the gradient of bias", g.bias, bytes)},
                                     {regionOf("x", norm->x, s, channels, size), regionOf("gate", norm->gate, s, channels, size), regionOf("the gradient of out", g.out, s, channels, size),
                                      regionOf("weight", norm->weight, bytes), regionOf("bias", norm->bias, bytes)})) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, s.device)) { return rc; }
        const auto arrays = {&norm->x, &norm->gate, &g.out, &g.x, &g.gate};
        NormArgs a = normArgs(*norm, p, oneBehindAnother(s, arrays));
        a.dout = g.out; a.dx = g.x; a.dgate = g.gate;
        a.sums = sums ? (float*)workspace : nullptr;
        if(a.rows) {
            const int rc = withNorm<true>(*norm, p, vectorOf(size, channels, arrays), [&](auto t, auto lanes, auto each, auto vec, auto gate) {
                constexpr int LANES = decltype(lanes)::value, E = decltype(each)::value;
                const auto kernel = normBackwardKernel<decltype(t), LANES, E, decltype(vec)::value, decltype(gate)::value>;
                const size_t lds = LANES == 0 && E == 16 ? 2 * E * NORM_APART * sizeof(float) : sums && p.groups > 1 ? p.threads * E * sizeof(float) : 0;
                if(const int rcLds = withLds(what, kernel, lds)) { return rcLds; }
                kernel<<<dim3(p.blocks), dim3(p.threads), lds, (hipStream_t)stream>>>(a);
                return gennmi_detail::afterLaunch(what);
            });
            if(rc) { return rc; }
        }
        if(sums) {
            if(const int rc = launchChunkSum(what, {a.sums, g.weight, {g.bias, nullptr}, p.blocks, channels, 1, 2}, (hipStream_t)stream)) { return rc; }
        }
        noteRows(g.x, s, channels, size);
        noteRows(g.gate, s, channels, size);
        if(g.weight) { gennmi_detail::noteDeviceWrite(g.weight, bytes); }
        if(g.bias) { gennmi_detail::noteDeviceWrite(g.bias, bytes); }
        return (int)GENNMI_OK;
    });
}

int gennmi_dropout(const gennmi_dropout_t *dropout, void *stream)
{
    const char *what = "dropout";
    return gennmi_detail::guarded(what, [&] {
        if(!dropout) { return fail(GENNMI_EINVAL, "dropout: null descriptor"); }
        const gennmi_sequences_t &s = dropout->sequences;
        const uint32_t size = sizeOf(dropout->type), channels = dropout->channels;
        if(!size) { return fail(GENNMI_EUNSUPPORTED, "dropout: unknown element type"); }
        if(channels < 1 || channels > (1u << 24)) { return fail(GENNMI_EINVAL, "dropout: number of channels"); }
        if(!(dropout->probability >= 0.0 && dropout->probability <= 1.0)) { return fail(GENNMI_EINVAL, "dropout: probability is not between 0 and 1"); }
        if(const int rc = checkPlainRows(what, s)) { return rc; }
        if(const int rc = checkRows(what, "x", dropout->x, s, channels, size)) { return rc; }
        if(dropout->residual.data) { if(const int rc = checkRows(what, "residual", dropout->residual, s, channels, size)) { return rc; } }
        if(const int rc = checkWrittenRows(what, "out", dropout->out, s, channels, size)) { return rc; }
        if((uintptr_t)dropout->callDevice % 8) { return fail(GENNMI_EINVAL, "dropout: callDevice is not aligned"); }
        const uint64_t groups = (channels + 7) / 8, items = totalRows(s) * groups;
        if((items + 255) / 256 > mostBlocks(256)) { return tooMany(what); }
        if(const int rc = checkApart(what, {regionOf("out", dropout->out, s, channels, size)}, {},
                                     {unlessSameRows(regionOf("x", dropout->x, s, channels, size), dropout->x, dropout->out),
                                      unlessSameRows(regionOf("residual", dropout->residual, s, channels, size), dropout->residual, dropout->out), regionOf("callDevice", dropout->callDevice, 8)})) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, s.device)) { return rc; }
        if(!items) { return (int)GENNMI_OK; }
        const auto arrays = {&dropout->x, &dropout->residual, &dropout->out};
        DropoutArgs a{};
        a.x = dropout->x; a.residual = dropout->residual; a.out = dropout->out;
        a.callDevice = dropout->callDevice;
        a.call = dropout->call;
        a.k0 = (uint32_t)dropout->seed; a.k1 = (uint32_t)(dropout->seed >> 32);
        a.items = (uint32_t)items; a.groups = (uint32_t)groups; a.channels = channels;
        a.length = oneBehindAnother(s, arrays) ? (uint32_t)totalRows(s) : s.length;
        a.dropped = (uint32_t)std::floor(dropout->probability * 65536.0 + 0.5);
        a.factor = a.dropped < 65536 ? (float)(65536.0 / (65536 - a.dropped)) : 0.0f;
        const int rc = withType(dropout->type, [&](auto t) {
            typedef decltype(t) T;
            const dim3 grid((uint32_t)((items + 255) / 256));
            if(vectorOf(size, channels, arrays) > 1) { dropoutKernel<T, true><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a); }
            else { dropoutKernel<T, false><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a); }
            return gennmi_detail::afterLaunch(what);
        });
        if(rc) { return rc; }
        noteRows(dropout->out, s, channels, size);
        return (int)GENNMI_OK;
    });
}

int gennmi_abi_layer_sizes(size_t sizes[5])
{
    if(!sizes) { return fail(GENNMI_EINVAL, "abi_layer_sizes: null result pointer"); }
    const size_t all[] = {sizeof(gennmi_delta_rule_t), sizeof(gennmi_delta_rule_gradient_t), sizeof(gennmi_layer_norm_t), sizeof(gennmi_layer_norm_gradient_t), sizeof(gennmi_dropout_t)};
    for(int i = 0; i < 5; i++) { sizes[i] = all[i]; }
    return GENNMI_OK;
}

}

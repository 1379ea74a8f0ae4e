// AdamW over many tensors in one launch, with states in 32 bits or in 8.
//
// Bound by memory: a weight is read and written with its gradient and states, 28 bytes in 32 bits with fp32 gradients, 16 in 8 bits, for some
// 25 to 60 operations.  A work-group takes CHUNK neighbouring weights of one tensor (a table says which), four a lane in one access each.  In
// 8 bits the 256 weights that share a scale are one wavefront's four a lane, so their maxima are found in registers and codes are written by the
// pass that made the states.  The number of the step is the device's: the work-group that ends last counts it, so a captured step counts as well.
//
// 80 M weights in 32 bits (fp32 weights, bf16 gradients and copy) take 382 to 390 us, 130 M in 8 bits (bf16 gradients) 313: 5.7 to 5.9 and 5.8 TB/s, where a large copy reaches 4.7.
// One access an array and lane, and many short work-groups: without the streaming accesses, and with more arithmetic in 8 bits, CHUNK 1024, 2048, 4096, 8192
// took 411, 428, 441, 449 us and 369, 373, 410, 409; work-groups that stay and go through the table 466 and more; the next
// block's loads ahead of the arithmetic 436 and 457 (registers).
#include <cmath>
#include <new>
#include <type_traits>
#include <vector>

#include "genn_mi355x_elements.h"
#include "genn_mi355x_lanes.h"

using namespace gennmi_elements;
using gennmi_detail::fail;

namespace
{
constexpr uint32_t CHUNK = 1024;        // weights of a work-group: a block each for its four wavefronts
static_assert(GENNMI_ADAMW_BLOCK == 256, "a block is the four weights a lane of one wavefront");

struct ParameterDev
{
    void *weight; const void *gradient; void *copy; void *m, *v; float *mScale, *vScale;
    uint64_t count;
    uint32_t weightType, gradientType, copyType, whole;         // whole: four neighbouring weights are one aligned access in every array
    double weightDecay;
};
struct ChunkDev { uint32_t parameter, index; };
constexpr uint64_t STREAM_BYTES = 64ull << 20;      // of a step, from which nothing of it stays in the L2 caches (32 MiB) for whoever comes next
// What the device knows of time: for the step to come, beta^t and 1 / (1 - beta^t); and work-groups that have ended, counted in GROUPS places (cache
// lines of their own) and the places that are full in another: one place takes 86 million counts a second, fewer than work-groups can end
constexpr uint32_t GROUPS = 32, LINE = 32;
struct CounterDev { double power1, power2; unsigned long long step; float correct1, correct2; uint32_t pad[LINE - 8]; uint32_t ended[(GROUPS + 1) * LINE]; };
// ... from beta^(t - 1)
__host__ __device__ inline void setCounter(CounterDev &c, double beta1, double beta2, double before1, double before2, unsigned long long step)
{
    c.power1 = before1 * beta1;
    c.power2 = before2 * beta2;
    c.correct1 = (float)(1.0 / (1.0 - c.power1));
    c.correct2 = (float)(1.0 / (1.0 - c.power2));
    c.step = step;
}

struct StepArgs
{
    const ParameterDev *parameters; const ChunkDev *chunks; CounterDev *counter;
    uint32_t numChunks, pad;
    double beta1, beta2, rate;
    float epsilon;
    const float *rateDevice, *gradientScale; const uint32_t *skip;
};

// Four neighbouring elements; STREAM: which nobody reads again soon
template<bool STREAM, typename P> __device__ inline P loadPack(const P *from)
{
    if constexpr(!STREAM) { return *from; }
    else {
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof(P) / 4)));
        const Words w = __builtin_nontemporal_load((const Words*)from);
        return __builtin_bit_cast(P, w);
    }
}
template<bool STREAM, typename P> __device__ inline void storePack(P *to, const P &p)
{
    if constexpr(!STREAM) { *to = p; }
    else {
        typedef uint32_t Words __attribute__((ext_vector_type(sizeof(P) / 4)));
        __builtin_nontemporal_store(__builtin_bit_cast(Words, p), (Words*)to);
    }
}
template<bool STREAM, typename T> __device__ inline void load4(const void *array, uint64_t at, uint32_t there, bool whole, float (&x)[4])
{
    const T *from = (const T*)array + at;
    if(whole && there == 4) {
        const Pack<T, 4> p = loadPack<STREAM>((const Pack<T, 4>*)from);
        #pragma unroll
        for(int k = 0; k < 4; k++) { x[k] = widen(p.v[k]); }
    }
    else {
        #pragma unroll
        for(int k = 0; k < 4; k++) { x[k] = k < (int)there ? widen(from[k]) : 0.0f; }
    }
}
template<bool STREAM> __device__ inline void load4(const void *array, uint32_t type, uint64_t at, uint32_t there, bool whole, float (&x)[4])
{
    if(type == GENNMI_TYPE_F32) { load4<STREAM, float>(array, at, there, whole, x); }
    else if(type == GENNMI_TYPE_F16) { load4<STREAM, f16>(array, at, there, whole, x); }
    else { load4<STREAM, bf16>(array, at, there, whole, x); }
}
template<bool STREAM, typename T> __device__ inline void store4(void *array, uint64_t at, uint32_t there, bool whole, const float (&x)[4])
{
    T *to = (T*)array + at;
    if(whole && there == 4) {
        Pack<T, 4> p;
        #pragma unroll
        for(int k = 0; k < 4; k++) { p.v[k] = narrow<T>(x[k]); }
        storePack<STREAM>((Pack<T, 4>*)to, p);
    }
    else {
        #pragma unroll
        for(int k = 0; k < 4; k++) { if(k < (int)there) { to[k] = narrow<T>(x[k]); } }
    }
}
template<bool STREAM> __device__ inline void store4(void *array, uint32_t type, uint64_t at, uint32_t there, bool whole, const float (&x)[4])
{
    if(type == GENNMI_TYPE_F32) { store4<STREAM, float>(array, at, there, whole, x); }
    else if(type == GENNMI_TYPE_F16) { store4<STREAM, f16>(array, at, there, whole, x); }
    else { store4<STREAM, bf16>(array, at, there, whole, x); }
}
template<bool STREAM> __device__ inline uint32_t loadCodes(const void *array, uint64_t at, uint32_t there, bool whole)
{
    const uint8_t *from = (const uint8_t*)array + at;
    if(whole && there == 4) { return loadPack<STREAM>((const uint32_t*)from); }
    uint32_t codes = 0;
    #pragma unroll
    for(int k = 0; k < 4; k++) { if(k < (int)there) { codes |= (uint32_t)from[k] << (8 * k); } }
    return codes;
}
template<bool STREAM> __device__ inline void storeCodes(void *array, uint64_t at, uint32_t there, bool whole, uint32_t codes)
{
    uint8_t *to = (uint8_t*)array + at;
    if(whole && there == 4) { storePack<STREAM>((uint32_t*)to, codes); }
    else {
        #pragma unroll
        for(int k = 0; k < 4; k++) { if(k < (int)there) { to[k] = (uint8_t)(codes >> (8 * k)); } }
    }
}
__device__ inline void decode(uint32_t codes, float (&c)[4])
{
    const auto low = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false), high = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
    c[0] = low[0]; c[1] = low[1]; c[2] = high[0]; c[3] = high[1];
}
__device__ inline uint32_t encode(const float (&r)[4])
{
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false), true);
}
// A 64-bit value in 24 bits such that rounding it once more, to fewer bits, gives what rounding the value itself would: the last bit is set
// where the result is not exact (of the two neighbours the odd one)
__device__ inline float roundToOdd(double r)
{
    const float f = (float)r;
    const double off = r - (double)f;
    const uint32_t bits = __float_as_uint(f);
    if(off == 0.0 || off != off || (bits & 1)) { return f; }
    return __uint_as_float((off > 0.0) == (r > 0.0) ? bits + 1 : bits - 1);
}
template<bool EIGHT, bool STREAM>
__global__ __launch_bounds__(256)
void adamwKernel(StepArgs a)
{
    if(a.skip && *a.skip) { return; }
    const ChunkDev chunk = a.chunks[blockIdx.x];
    const ParameterDev p = a.parameters[chunk.parameter];
    const double before1 = a.counter->power1, before2 = a.counter->power2;
    const unsigned long long stepsBefore = a.counter->step;
    const uint64_t block = (uint64_t)chunk.index * (CHUNK / 256) + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), at = block * 256 + (threadIdx.x & 63) * 4;
    if(block * 256 < p.count) {
        const double rate = a.rateDevice ? (double)*a.rateDevice : a.rate;
        const float scale = a.gradientScale ? *a.gradientScale : 1.0f, step = (float)rate, keep = (float)(1.0 - rate * p.weightDecay);
        const float correct1 = a.counter->correct1, correct2 = a.counter->correct2;
        const uint32_t there = at < p.count ? (uint32_t)(p.count - at < 4 ? p.count - at : 4) : 0;
        const bool whole = p.whole;
        float w[4], g[4], m[4], v[4];
        load4<STREAM>(p.weight, p.weightType, at, there, whole, w);
        load4<STREAM>(p.gradient, p.gradientType, at, there, whole, g);
        #pragma unroll
        for(int i = 0; i < 4; i++) { g[i] *= scale; }
        if(!EIGHT) {
            load4<STREAM, float>(p.m, at, there, whole, m);
            load4<STREAM, float>(p.v, at, there, whole, v);
            #pragma unroll
            for(int i = 0; i < 4; i++) {
                m[i] = __builtin_fmaf((float)a.beta1, m[i], (float)(1.0 - a.beta1) * g[i]);
                v[i] = __builtin_fmaf((float)a.beta2, v[i], (float)(1.0 - a.beta2) * g[i] * g[i]);
            }
            store4<STREAM, float>(p.m, at, there, whole, m);
            store4<STREAM, float>(p.v, at, there, whole, v);
        }
        else {
            // States in 64 bits (as fast here as 32), so that the scales are those of the formula and not of its rounding errors.  The codes are found in
            // 32 bits, from values 2^-20 of themselves below and above: where the two differ, a border between codes lies so near that 64 bits have to
            // say on which side (one wavefront in 60).
            decode(loadCodes<STREAM>(p.m, at, there, whole), m);
            decode(loadCodes<STREAM>(p.v, at, there, whole), v);
            const double unitM = a.beta1 * ((double)p.mScale[block] * (1.0 / 448.0)), unitV = a.beta2 * ((double)p.vScale[block] * (1.0 / (448.0 * 448.0)));
            double m64[4], v64[4];
            uint32_t bitsM = 0, bitsV = 0;
            #pragma unroll
            for(int i = 0; i < 4; i++) {
                const double gradient = g[i];
                m64[i] = __builtin_fma((double)m[i], unitM, (1.0 - a.beta1) * gradient);
                v64[i] = __builtin_fma((1.0 - a.beta2) * gradient, gradient, (double)(v[i] * v[i]) * unitV);
                m[i] = (float)m64[i];
                v[i] = (float)v64[i];
                bitsM = max(bitsM, __float_as_uint(fabsf(m[i])));
                bitsV = max(bitsV, __float_as_uint(v[i]));
            }
            gennmi_lanes::maxOfLanes(bitsM, bitsV);
            const float M = __uint_as_float(bitsM), V = __uint_as_float(bitsV);
            constexpr float BELOW = 448.0f * (1.0f - 0x1p-20f), ABOVE = 448.0f * (1.0f + 0x1p-20f), LEAST = 0x1p-18f / (448.0f * 448.0f);
            const float inverseM = M > 0.0f ? __builtin_amdgcn_rcpf(M) : M, inverseV = V > 0.0f ? __builtin_amdgcn_rcpf(V) : V;
            const float belowM = BELOW * inverseM, aboveM = ABOVE * inverseM;
            float lowM[4], highM[4], lowV[4], highV[4];
            #pragma unroll
            for(int i = 0; i < 4; i++) {
                lowM[i] = m[i] * belowM;
                highM[i] = m[i] * aboveM;
                // (a positive v has a code of its own: at least the root of LEAST)
                const float share = v[i] * inverseV, root = __builtin_amdgcn_sqrtf(v[i] > 0.0f && share < LEAST ? LEAST : share);
                lowV[i] = root * BELOW;
                highV[i] = root * ABOVE;
            }
            uint32_t codesM = encode(lowM), codesV = encode(lowV);
            // (nor do quotients of 32 bits do where the largest of a block are so small that inverses or others' are subnormal, or so large that their inverses are)
            const auto extreme = [](float most) { return (most > 0.0f && most < 1e-25f) || (most > 0x1p125f && most < __builtin_inff()); };
            const bool near = codesM != encode(highM) || codesV != encode(highV) || extreme(M) || extreme(V);
            if(__ballot(near)) {
                #pragma unroll
                for(int i = 0; i < 4; i++) {
                    if(M > 0.0f) { lowM[i] = roundToOdd(m64[i] * (448.0 / (double)M)); }
                    if(V > 0.0f) { lowV[i] = roundToOdd(448.0 * sqrt(v64[i] / (double)V)); }
                    lowV[i] = v[i] > 0.0f && lowV[i] < 0x1p-9f ? 0x1p-9f : lowV[i];
                }
                codesM = encode(lowM);
                codesV = encode(lowV);
            }
            storeCodes<STREAM>(p.m, at, there, whole, codesM);
            storeCodes<STREAM>(p.v, at, there, whole, codesV);
            if((threadIdx.x & 63) == 0) { p.mScale[block] = M; p.vScale[block] = V; }
        }
        if(a.epsilon >= 1e-12f) {
            // (one instruction each for root and inverse: their last bit, and subnormal second moments, do not matter beside epsilon)
            #pragma unroll
            for(int i = 0; i < 4; i++) {
                const float change = m[i] * correct1 * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[i] * correct2) + a.epsilon);
                w[i] = __builtin_fmaf(-step, change, w[i] * keep);
            }
        }
        else {
            #pragma unroll
            for(int i = 0; i < 4; i++) {
                const float change = m[i] * correct1 / (sqrtf(v[i] * correct2) + a.epsilon);
                w[i] = __builtin_fmaf(-step, change, w[i] * keep);
            }
        }
        store4<STREAM>(p.weight, p.weightType, at, there, whole, w);
        if(p.copy) { store4<STREAM>(p.copy, p.copyType, at, there, whole, w); }
    }
    // (every wavefront has read what it needs of the counter before its work-group is counted; what it wrote need not have arrived)
    __builtin_amdgcn_s_barrier();
    if(threadIdx.x) { return; }
    if(gridDim.x > GROUPS) {
        uint32_t *const place = a.counter->ended + (1 + blockIdx.x % GROUPS) * LINE;
        if(atomicAdd(place, 1u) != (gridDim.x - 1 - blockIdx.x % GROUPS) / GROUPS) { return; }
        *place = 0;
    }
    if(atomicAdd(a.counter->ended, 1u) == min(gridDim.x, GROUPS) - 1) {
        a.counter->ended[0] = 0;
        setCounter(*a.counter, a.beta1, a.beta2, before1, before2, stepsBefore + 1);
    }
}

}

struct gennmi_optimiser
{
    gennmi_adamw_t settings{};
    std::vector<gennmi_parameter_t> parameters;
    std::vector<ParameterDev> table;
    uint64_t bytes = 0;             // that a step reads and writes
    ParameterDev *dParameters = nullptr; ChunkDev *dChunks = nullptr; CounterDev *dCounter = nullptr;
    uint32_t numChunks = 0, device = 0;         // device: 1 + the one that was current when the table was uploaded
    bool finalised = false;
    void freeTables()
    {
        (void)gennmi_free(dParameters); (void)gennmi_free(dChunks); (void)gennmi_free(dCounter);
        dParameters = nullptr; dChunks = nullptr; dCounter = nullptr;
    }
    ~gennmi_optimiser() { freeTables(); }
};

extern "C" {

int gennmi_optimiser_create(gennmi_optimiser **optimiser, const gennmi_adamw_t *settings)
{
    return gennmi_detail::guarded("optimiser_create", [&] {
        if(!optimiser || !settings) { return fail(GENNMI_EINVAL, "optimiser_create: null argument"); }
        *optimiser = nullptr;
        if(settings->stateBits != 8 && settings->stateBits != 32) { return fail(GENNMI_EUNSUPPORTED, "optimiser_create: states have 8 or 32 bits"); }
        if(!(settings->beta1 >= 0.0 && settings->beta1 < 1.0 && settings->beta2 >= 0.0 && settings->beta2 < 1.0 && settings->epsilon >= 0.0 && std::isfinite(settings->epsilon))) {
            return fail(GENNMI_EINVAL, "optimiser_create: needs 0 <= beta < 1 and epsilon >= 0");
        }
        gennmi_optimiser *o = new gennmi_optimiser;
        o->settings = *settings;
        *optimiser = o;
        return (int)GENNMI_OK;
    });
}

int gennmi_optimiser_destroy(gennmi_optimiser *optimiser)
{
    return gennmi_detail::guarded("optimiser_destroy", [&] { delete optimiser; return (int)GENNMI_OK; });
}

int gennmi_optimiser_push(gennmi_optimiser *optimiser, const gennmi_parameter_t *parameter, uint32_t *idx)
{
    return gennmi_detail::guarded("optimiser_push", [&] {
        if(!optimiser || !parameter) { return fail(GENNMI_EINVAL, "optimiser_push: null argument"); }
        if(optimiser->finalised) { return fail(GENNMI_ESTATE, "optimiser_push: the optimiser is finalised"); }
        const gennmi_parameter_t &p = *parameter;
        const bool eight = optimiser->settings.stateBits == 8;
        const uint32_t weightSize = sizeOf(p.weightType), gradientSize = sizeOf(p.gradientType), copySize = p.copy ? sizeOf(p.copyType) : 2;
        if(!weightSize || !gradientSize || copySize != 2) { return fail(GENNMI_EUNSUPPORTED, "optimiser_push: unknown element type"); }
        if(p.count > (1ull << 40)) { return fail(GENNMI_EINVAL, "optimiser_push: number of weights"); }
        if(p.count && (!p.weight || !p.gradient || !p.m || !p.v || (eight && (!p.mScale || !p.vScale)))) { return fail(GENNMI_EINVAL, "optimiser_push: an array is missing"); }
        if((uintptr_t)p.weight % weightSize || (uintptr_t)p.gradient % gradientSize || (uintptr_t)p.copy % 2 ||
           (!eight && ((uintptr_t)p.m % 4 || (uintptr_t)p.v % 4)) || (eight && ((uintptr_t)p.mScale % 4 || (uintptr_t)p.vScale % 4))) {
            return fail(GENNMI_EINVAL, "optimiser_push: an array is not aligned to its elements");
        }
        if(!std::isfinite(p.weightDecay)) { return fail(GENNMI_EINVAL, "optimiser_push: weight decay"); }
        // (work-groups do not wait for one another: nothing that a step writes may be anything else that it reads or writes)
        const auto shared = [&](const gennmi_parameter_t &x, const gennmi_parameter_t &y) {
            struct Range { const void *ptr; size_t bytes; };
            const auto ranges = [&](const gennmi_parameter_t &q, Range (&r)[7]) {
                const size_t stateSize = eight ? 1 : 4, scales = eight ? (q.count + GENNMI_ADAMW_BLOCK - 1) / GENNMI_ADAMW_BLOCK * sizeof(float) : 0;
                const Range all[7] = {{q.weight, q.count * sizeOf(q.weightType)}, {q.m, q.count * stateSize}, {q.v, q.count * stateSize}, {q.copy, q.copy ? q.count * 2 : 0},
                                      {q.mScale, scales}, {q.vScale, scales}, {q.gradient, q.count * sizeOf(q.gradientType)}};
                for(int k = 0; k < 7; k++) { r[k] = all[k]; }
            };
            Range a[7], b[7];
            ranges(x, a);
            ranges(y, b);
            for(int i = 0; i < 7; i++) {
                for(int j = 0; j < 7; j++) {
                    if((i == 6 && j == 6) || (&x == &y && i == j)) { continue; }        // (gradients are only read)
                    if((uintptr_t)a[i].ptr < (uintptr_t)b[j].ptr + b[j].bytes && (uintptr_t)b[j].ptr < (uintptr_t)a[i].ptr + a[i].bytes) { return true; }
                }
            }
            return false;
        };
        if(shared(p, p)) { return fail(GENNMI_EINVAL, "optimiser_push: weight, gradient, states, scales and copy are arrays of their own"); }
        for(const gennmi_parameter_t &q : optimiser->parameters) {
            if(shared(p, q)) { return fail(GENNMI_EINVAL, "optimiser_push: overlaps a tensor that was pushed before"); }
        }
        const size_t stateSize = eight ? 1 : 4;
        ParameterDev d{p.weight, p.gradient, p.copy, p.m, p.v, p.mScale, p.vScale, p.count, p.weightType, p.gradientType, p.copyType, 0, p.weightDecay};
        d.whole = (uintptr_t)p.weight % (4 * weightSize) == 0 && (uintptr_t)p.gradient % (4 * gradientSize) == 0 && (uintptr_t)p.copy % 8 == 0 &&
                  (uintptr_t)p.m % (4 * stateSize) == 0 && (uintptr_t)p.v % (4 * stateSize) == 0;
        optimiser->bytes += p.count * (2 * weightSize + gradientSize + 4 * stateSize + (p.copy ? 2 : 0));
        optimiser->parameters.push_back(p);
        optimiser->table.push_back(d);
        if(idx) { *idx = (uint32_t)optimiser->parameters.size() - 1; }
        return (int)GENNMI_OK;
    });
}

int gennmi_optimiser_finalise(gennmi_optimiser *optimiser)
{
    return gennmi_detail::guarded("optimiser_finalise", [&] {
        if(!optimiser) { return fail(GENNMI_EINVAL, "optimiser_finalise: null argument"); }
        if(optimiser->finalised) { return fail(GENNMI_ESTATE, "optimiser_finalise: the optimiser is finalised"); }
        std::vector<ChunkDev> chunks;
        for(size_t k = 0; k < optimiser->table.size(); k++) {
            const uint64_t of = (optimiser->table[k].count + CHUNK - 1) / CHUNK;
            if(chunks.size() + of > mostBlocks(256)) { return fail(GENNMI_EINVAL, "optimiser_finalise: more weights than one launch covers"); }
            for(uint64_t c = 0; c < of; c++) { chunks.push_back({(uint32_t)k, (uint32_t)c}); }
        }
        if(chunks.empty()) { chunks.push_back({(uint32_t)optimiser->table.size(), 0}); }        // (a step of nothing counts: a tensor without weights)
        std::vector<ParameterDev> table = optimiser->table;
        table.push_back(ParameterDev{});
        std::vector<CounterDev> counter(1, CounterDev{});
        setCounter(counter[0], optimiser->settings.beta1, optimiser->settings.beta2, 1.0, 1.0, 0);
        const auto upload = [&](auto **to, const auto &from) {
            if(const int rc = gennmi_malloc((void**)to, from.size() * sizeof(from[0]))) { return rc; }
            return gennmi_memcpy_to_device(*to, from.data(), from.size() * sizeof(from[0]));
        };
        int device = 0, rc = upload(&optimiser->dParameters, table);
        if(!rc) { rc = upload(&optimiser->dChunks, chunks); }
        if(!rc) { rc = upload(&optimiser->dCounter, counter); }
        if(!rc) { if(const hipError_t e = hipGetDevice(&device)) { rc = fail(GENNMI_EHIP, std::string("optimiser_finalise: ") + hipGetErrorString(e)); } }
        if(rc) { optimiser->freeTables(); return rc; }          // (another attempt begins anew)
        optimiser->device = 1 + (uint32_t)device;
        optimiser->numChunks = (uint32_t)chunks.size();
        optimiser->finalised = true;
        return (int)GENNMI_OK;
    });
}

int gennmi_optimiser_step(gennmi_optimiser *optimiser, const gennmi_adamw_step_t *step, void *stream)
{
    return gennmi_detail::guarded("optimiser_step", [&] {
        if(!optimiser || !step) { return fail(GENNMI_EINVAL, "optimiser_step: null argument"); }
        if(!optimiser->finalised) { return fail(GENNMI_ESTATE, "optimiser_step: the optimiser is not finalised"); }
        if(!step->rateDevice && !std::isfinite(step->rate)) { return fail(GENNMI_EINVAL, "optimiser_step: learning rate"); }
        for(const void *p : {(const void*)step->rateDevice, (const void*)step->gradientScale, (const void*)step->skip}) {
            if((uintptr_t)p % 4) { return fail(GENNMI_EINVAL, "optimiser_step: a device value is not aligned"); }
        }
        const gennmi_optimiser &o = *optimiser;
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, o.device)) { return rc; }
        const StepArgs a{o.dParameters, o.dChunks, o.dCounter, o.numChunks, 0, o.settings.beta1, o.settings.beta2, step->rate, (float)o.settings.epsilon,
                         step->rateDevice, step->gradientScale, step->skip};
        const dim3 grid(o.numChunks);
        const bool eight = o.settings.stateBits == 8, streaming = o.bytes > STREAM_BYTES;
        if(eight && streaming) { adamwKernel<true, true><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a); }
        else if(eight) { adamwKernel<true, false><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a); }
        else if(streaming) { adamwKernel<false, true><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a); }
        else { adamwKernel<false, false><<<grid, dim3(256), 0, (hipStream_t)stream>>>(a); }
        if(const int rc = gennmi_detail::afterLaunch("optimiser_step")) { return rc; }
        if(!gennmi_detail::anyRunners()) { return (int)GENNMI_OK; }         // (dozens of tensors: asked once)
        for(const gennmi_parameter_t &p : o.parameters) {
            if(p.count) { gennmi_detail::noteDeviceWrite(p.weight, p.count * sizeOf(p.weightType)); }
        }
        return (int)GENNMI_OK;
    });
}

int gennmi_optimiser_get_step(gennmi_optimiser *optimiser, uint64_t *step)
{
    return gennmi_detail::guarded("optimiser_get_step", [&] {
        if(!optimiser || !step) { return fail(GENNMI_EINVAL, "optimiser_get_step: null argument"); }
        if(!optimiser->finalised) { return fail(GENNMI_ESTATE, "optimiser_get_step: the optimiser is not finalised"); }
        if(const int rc = gennmi_synchronize()) { return rc; }
        CounterDev counter;
        if(const int rc = gennmi_memcpy_from_device(&counter, optimiser->dCounter, sizeof(counter))) { return rc; }
        *step = counter.step;
        return (int)GENNMI_OK;
    });
}

int gennmi_optimiser_set_step(gennmi_optimiser *optimiser, uint64_t step)
{
    return gennmi_detail::guarded("optimiser_set_step", [&] {
        if(!optimiser) { return fail(GENNMI_EINVAL, "optimiser_set_step: null argument"); }
        if(!optimiser->finalised) { return fail(GENNMI_ESTATE, "optimiser_set_step: the optimiser is not finalised"); }
        if(const int rc = gennmi_synchronize()) { return rc; }
        CounterDev counter{};
        const double beta1 = optimiser->settings.beta1, beta2 = optimiser->settings.beta2;
        setCounter(counter, beta1, beta2, std::pow(beta1, (double)step), std::pow(beta2, (double)step), step);
        return gennmi_memcpy_to_device(optimiser->dCounter, &counter, sizeof(counter));
    });
}

int gennmi_abi_operator_sizes(size_t sizes[9])
{
    const size_t values[9] = {sizeof(gennmi_rows_t), sizeof(gennmi_sequences_t), sizeof(gennmi_causal_conv_t), sizeof(gennmi_causal_conv_gradient_t), sizeof(gennmi_scan_t),
                              sizeof(gennmi_scan_gradient_t), sizeof(gennmi_adamw_t), sizeof(gennmi_parameter_t), sizeof(gennmi_adamw_step_t)};
    if(!sizes) { return fail(GENNMI_EINVAL, "abi_operator_sizes: null result pointer"); }
    for(int k = 0; k < 9; k++) { sizes[k] = values[k]; }
    return GENNMI_OK;
}

}

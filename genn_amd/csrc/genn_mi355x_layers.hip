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
// A row lies in the registers of the lanes that share it: 16 or 64 of a wavefront, or a work-group, each with up to 16 elements of it, so that it is read once and its
// statistics are those of its elements as they are: first the mean, then the squares of what is left.
struct NormArgs
{
    gennmi_rows_t x, gate, out;
    const float *weight, *bias;
    uint32_t rows, length, channels, rms;
    float epsilon, share;           // 1 / channels
    gennmi_rows_t dout, dx, dgate;
    float *sums;                    // of each work-group: weight's and bias's, [2][channels]
};
template<typename T> __device__ inline T *normRow(const gennmi_rows_t &r, uint32_t sequence, uint32_t row) { return (T*)r.data + (uint64_t)sequence * r.sequenceStride + (uint64_t)row * r.rowStride; }

// Sums of N values over the lanes of a row.  `LANES` 0: over the work-group, through LDS; two of its places are used in turn, so that one barrier a sum does.
template<int LANES, int N> __device__ inline void sumOfRow(float (&v)[N], float (*found)[2][16], uint32_t &turn)
{
    #pragma unroll
    for(int n = 0; n < N; n++) {
        v[n] += partner<1>(v[n]); v[n] += partner<2>(v[n]); v[n] += partner<4>(v[n]); v[n] += partner<8>(v[n]);
        if(LANES != 16) { v[n] += partner<16>(v[n]); v[n] += partner<32>(v[n]); }
    }
    if constexpr(LANES == 0) {
        const uint32_t wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
        if((threadIdx.x & 63) == 0) { for(int n = 0; n < N; n++) { found[turn][n][wave] = v[n]; } }
        __syncthreads();
        for(int n = 0; n < N; n++) {
            float sum = 0.0f;
            for(uint32_t w = 0; w < waves; w++) { sum += found[turn][n][w]; }
            v[n] = sum;
        }
        turn ^= 1;
    }
}
template<typename T, int E, int VEC> __device__ inline void loadRow(const T *row, uint32_t lane, uint32_t lanes, uint32_t channels, float (&x)[E])
{
    #pragma unroll
    for(int i = 0; i < E / VEC; i++) {
        const uint32_t c = (i * lanes + lane) * VEC;
        Pack<T, VEC> p{};
        if(c < channels) { p = *(const Pack<T, VEC>*)(row + c); }
        #pragma unroll
        for(int e = 0; e < VEC; e++) { x[i * VEC + e] = widen(p.v[e]); }
    }
}
template<typename T, int E, int VEC> __device__ inline void storeRow(T *row, uint32_t lane, uint32_t lanes, uint32_t channels, const float (&x)[E])
{
    #pragma unroll
    for(int i = 0; i < E / VEC; i++) {
        const uint32_t c = (i * lanes + lane) * VEC;
        if(c >= channels) { continue; }
        Pack<T, VEC> p;
        #pragma unroll
        for(int e = 0; e < VEC; e++) { p.v[e] = narrow<T>(x[i * VEC + e]); }
        *(Pack<T, VEC>*)(row + c) = p;
    }
}
template<int E, int VEC> __device__ inline void loadParameters(const float *from, float without, uint32_t lane, uint32_t lanes, uint32_t channels, float (&x)[E])
{
    #pragma unroll
    for(int i = 0; i < E / VEC; i++) {
        #pragma unroll
        for(int e = 0; e < VEC; e++) {
            const uint32_t c = (i * lanes + lane) * VEC + e;
            x[i * VEC + e] = c < channels ? from ? from[c] : without : 0.0f;
        }
    }
}
// x becomes x', its length before is returned as a factor
template<int LANES, int E, int VEC> __device__ inline float normalise(const NormArgs &a, float (&x)[E], uint32_t lane, uint32_t lanes, float (*found)[2][16], uint32_t &turn)
{
    if(!a.rms) {
        float sum[1] = {0.0f};
        #pragma unroll
        for(int e = 0; e < E; e++) { sum[0] += x[e]; }
        sumOfRow<LANES>(sum, found, turn);
        const float mean = sum[0] * a.share;
        #pragma unroll
        for(int e = 0; e < E; e++) { x[e] = (uint32_t)(((e / VEC) * lanes + lane) * VEC + e % VEC) < a.channels ? x[e] - mean : 0.0f; }
    }
    float square[1] = {0.0f};
    #pragma unroll
    for(int e = 0; e < E; e++) { square[0] = __builtin_fmaf(x[e], x[e], square[0]); }
    sumOfRow<LANES>(square, found, turn);
    const float r = 1.0f / sqrtf(__builtin_fmaf(square[0], a.share, a.epsilon));
    #pragma unroll
    for(int e = 0; e < E; e++) { x[e] *= r; }
    return r;
}
__device__ inline float logistic(float z) { return 1.0f / (1.0f + expf(-z)); }

// Work-groups of 256 threads where 16 lanes or a wavefront have a row, else of as many as a row takes; each walks rows that are a grid apart, with the parameters in registers.
template<typename T, int LANES, int E, int VEC>
__global__ __launch_bounds__(LANES ? 256 : 1024)
void normKernel(NormArgs a)
{
    __shared__ float found[2][2][16];
    uint32_t turn = 0;
    const uint32_t lanes = LANES ? LANES : blockDim.x, lane = threadIdx.x % lanes, each = LANES ? 256 / LANES : 1;
    float weight[E], bias[E];
    loadParameters<E, VEC>(a.weight, 1.0f, lane, lanes, a.channels, weight);
    loadParameters<E, VEC>(a.bias, 0.0f, lane, lanes, a.channels, bias);
    for(uint64_t n = (uint64_t)blockIdx.x * each + threadIdx.x / lanes; n < a.rows; n += (uint64_t)gridDim.x * each) {
        const uint32_t sequence = (uint32_t)n / a.length, row = (uint32_t)n - sequence * a.length;
        float x[E], z[E];
        loadRow<T, E, VEC>(normRow<const T>(a.x, sequence, row), lane, lanes, a.channels, x);
        if(a.gate.data) { loadRow<T, E, VEC>(normRow<const T>(a.gate, sequence, row), lane, lanes, a.channels, z); }
        normalise<LANES, E, VEC>(a, x, lane, lanes, found, turn);
        #pragma unroll
        for(int e = 0; e < E; e++) {
            x[e] = __builtin_fmaf(x[e], weight[e], bias[e]);
            if(a.gate.data) { x[e] *= z[e] * logistic(z[e]); }
        }
        storeRow<T, E, VEC>(normRow<T>(a.out, sequence, row), lane, lanes, a.channels, x);
    }
}

// With y = x' weight + bias, s the gate's factor z sigmoid(z) and d = dout s:
//   dgate = dout y s',  dweight += d x',  dbias += d,  dx = (v - x' mean(v x') - mean(v)) / length, v = d weight (without the last mean for `rms`)
template<typename T, int LANES, int E, int VEC>
__global__ __launch_bounds__(LANES ? 256 : 1024)
void normBackwardKernel(NormArgs a)
{
    __shared__ float found[2][2][16];
    __shared__ float shared[LANES ? 256 * E : 1];
    uint32_t turn = 0;
    const uint32_t lanes = LANES ? LANES : blockDim.x, lane = threadIdx.x % lanes, each = LANES ? 256 / LANES : 1;
    float weight[E], bias[E], dweight[E] = {}, dbias[E] = {};
    loadParameters<E, VEC>(a.weight, 1.0f, lane, lanes, a.channels, weight);
    loadParameters<E, VEC>(a.bias, 0.0f, lane, lanes, a.channels, bias);
    for(uint64_t n = (uint64_t)blockIdx.x * each + threadIdx.x / lanes; n < a.rows; n += (uint64_t)gridDim.x * each) {
        const uint32_t sequence = (uint32_t)n / a.length, row = (uint32_t)n - sequence * a.length;
        float x[E], d[E];
        loadRow<T, E, VEC>(normRow<const T>(a.x, sequence, row), lane, lanes, a.channels, x);
        loadRow<T, E, VEC>(normRow<const T>(a.dout, sequence, row), lane, lanes, a.channels, d);
        const float r = normalise<LANES, E, VEC>(a, x, lane, lanes, found, turn);
        if(a.gate.data) {
            float z[E];
            loadRow<T, E, VEC>(normRow<const T>(a.gate, sequence, row), lane, lanes, a.channels, z);
            #pragma unroll
            for(int e = 0; e < E; e++) {
                const float s = logistic(z[e]), y = __builtin_fmaf(x[e], weight[e], bias[e]), dz = d[e] * y * (s * __builtin_fmaf(z[e], 1.0f - s, 1.0f));
                d[e] *= z[e] * s;
                z[e] = dz;
            }
            if(a.dgate.data) { storeRow<T, E, VEC>(normRow<T>(a.dgate, sequence, row), lane, lanes, a.channels, z); }
        }
        float means[2] = {0.0f, 0.0f};
        #pragma unroll
        for(int e = 0; e < E; e++) {
            dweight[e] = __builtin_fmaf(d[e], x[e], dweight[e]);
            dbias[e] += d[e];
            d[e] *= weight[e];
            means[0] = __builtin_fmaf(d[e], x[e], means[0]);
            means[1] += d[e];
        }
        if(!a.dx.data) { continue; }
        sumOfRow<LANES>(means, found, turn);
        const float along = means[0] * a.share, mean = a.rms ? 0.0f : means[1] * a.share;
        #pragma unroll
        for(int e = 0; e < E; e++) { x[e] = r * (__builtin_fmaf(-x[e], along, d[e]) - mean); }
        storeRow<T, E, VEC>(normRow<T>(a.dx, sequence, row), lane, lanes, a.channels, x);
    }
    if(!a.sums) { return; }
    float *const to = a.sums + (uint64_t)blockIdx.x * 2 * a.channels;
    #pragma unroll
    for(int which = 0; which < 2; which++) {
        float (&sum)[E] = which ? dbias : dweight;
        if constexpr(LANES != 0) {
            // (the rows of a work-group one after another)
            __syncthreads();
            #pragma unroll
            for(int e = 0; e < E; e++) { shared[e * 256 + threadIdx.x] = sum[e]; }
            __syncthreads();
            if(threadIdx.x >= LANES) { continue; }
            #pragma unroll
            for(int e = 0; e < E; e++) { for(uint32_t k = 1; k < each; k++) { sum[e] += shared[e * 256 + k * LANES + lane]; } }
        }
        #pragma unroll
        for(int e = 0; e < E; e++) {
            const uint32_t c = ((e / VEC) * lanes + lane) * VEC + e % VEC;
            if(c < a.channels) { to[which * a.channels + c] = sum[e]; }
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
// Bound by memory: a thread has eight neighbouring elements and draws once for them, 16 bits each (ten rounds of two wide products and four
// exclusive ors; a draw for four would take longer than the memory).
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
struct NormPlan { uint32_t lanes, threads, blocks; };       // lanes 0: a work-group a row
NormPlan normPlan(const gennmi_layer_norm_t &c, bool gradients)
{
    const uint64_t rows = totalRows(c.sequences);
    NormPlan p;
    p.lanes = c.channels <= 128 ? 16 : c.channels <= 1024 ? 64 : 0;
    p.threads = p.lanes ? 256 : ((c.channels + 15) / 16 + 63) / 64 * 64;
    const uint64_t each = p.lanes ? 256 / p.lanes : 1, most = gradients ? 1024 : 4096;
    p.blocks = (uint32_t)std::min<uint64_t>((rows + each - 1) / each, most);
    return p;
}
template<typename T, int VEC, typename F> int withNormLayout(const NormPlan &p, uint32_t channels, F &&f)
{
    typedef std::integral_constant<int, VEC> Vec;
    if(p.lanes == 16) { return f(std::integral_constant<int, 16>{}, std::integral_constant<int, 8>{}, Vec{}); }
    if(p.lanes == 64 && channels <= 512) { return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 8>{}, Vec{}); }
    if(p.lanes == 64) { return f(std::integral_constant<int, 64>{}, std::integral_constant<int, 16>{}, Vec{}); }
    return f(std::integral_constant<int, 0>{}, std::integral_constant<int, 16>{}, Vec{});
}
template<typename F> int withNorm(const gennmi_layer_norm_t &c, const NormPlan &p, uint32_t vector, F &&f)
{
    return withType(c.type, [&](auto t) {
        typedef decltype(t) T;
        const auto g = [&](auto lanes, auto each, auto vec) { return f(t, lanes, each, vec); };
        if(vector > 1) { return withNormLayout<T, 16 / sizeof(T)>(p, c.channels, g); }
        return withNormLayout<T, 1>(p, c.channels, g);
    });
}
NormArgs normArgs(const gennmi_layer_norm_t &c, bool flat)
{
    NormArgs a{};
    a.x = c.x; a.gate = c.gate; a.out = c.out;
    a.weight = c.weight; a.bias = c.bias;
    a.rows = (uint32_t)totalRows(c.sequences);
    a.length = flat ? a.rows : c.sequences.length;
    a.channels = c.channels; a.rms = c.rms;
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
        const NormArgs a = normArgs(*norm, oneBehindAnother(s, arrays));
        const int rc = withNorm(*norm, p, vectorOf(size, norm->channels, arrays), [&](auto t, auto lanes, auto each, auto vec) {
            normKernel<decltype(t), decltype(lanes)::value, decltype(each)::value, decltype(vec)::value><<<dim3(p.blocks), dim3(p.threads), 0, (hipStream_t)stream>>>(a);
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
        NormArgs a = normArgs(*norm, oneBehindAnother(s, arrays));
        a.dout = g.out; a.dx = g.x; a.dgate = g.gate;
        a.sums = sums ? (float*)workspace : nullptr;
        if(a.rows) {
            const int rc = withNorm(*norm, p, vectorOf(size, channels, arrays), [&](auto t, auto lanes, auto each, auto vec) {
                normBackwardKernel<decltype(t), decltype(lanes)::value, decltype(each)::value, decltype(vec)::value><<<dim3(p.blocks), dim3(p.threads), 0, (hipStream_t)stream>>>(a);
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

// Operators on sequences: a short causal convolution and a selective state space scan, with their gradients, for whole sequences and for
// single tokens.  Entry points and their checks; the kernels are in the headers included below.
#include <cmath>
#include <type_traits>

#include "genn_mi355x_elements.h"

using namespace gennmi_elements;
using gennmi_detail::fail;

namespace
{
// Sums over chunks, sums[number][n][channel], in 64 bits: there may be thousands, of either sign.  Row n of the sums goes to out[channel][n] for n < width,
// behind those to more[0][channel] and more[1][channel].  The 16 wavefronts of a work-group have 64 channels and a sixteenth of the numbers each;
// what they found is added up in the order of the numbers.
struct ChunkSums { const float *sums; float *out, *more[2]; uint32_t numbers, channels, width, rows; };
__global__ __launch_bounds__(1024)
void chunkSumKernel(ChunkSums a)
{
    __shared__ double found[16][64];
    const uint32_t parts = (a.channels + 63) / 64, n = blockIdx.x / parts, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t channel = (blockIdx.x - n * parts) * 64 + lane;
    const uint32_t each = (a.numbers + 15) / 16, first = min(wave * each, a.numbers), last = min(first + each, a.numbers);
    double sum = 0.0;
    if(channel < a.channels) {
        const float *at = a.sums + (uint64_t)n * a.channels + channel;
        #pragma unroll 8
        for(uint32_t k = first; k < last; k++) { sum += at[(uint64_t)k * a.rows * a.channels]; }
    }
    found[wave][lane] = sum;
    __syncthreads();
    if(wave || channel >= a.channels) { return; }
    #pragma unroll
    for(int k = 1; k < 16; k++) { sum += found[k][lane]; }
    if(n < a.width) { if(a.out) { a.out[(uint64_t)channel * a.width + n] = (float)sum; } }
    else if(a.more[n - a.width]) { a.more[n - a.width][channel] = (float)sum; }
}
uint64_t chunkSumBlocks(uint32_t rows, uint32_t channels) { return (uint64_t)rows * ((channels + 63) / 64); }
int launchChunkSum(const char *what, const ChunkSums &a, hipStream_t stream)
{
    chunkSumKernel<<<dim3((uint32_t)chunkSumBlocks(a.rows, a.channels)), dim3(1024), 0, stream>>>(a);
    return gennmi_detail::afterLaunch(what);
}
int tooMany(const char *what) { return fail(GENNMI_EINVAL, std::string(what) + ": more rows than one launch covers"); }
}

#include "genn_mi355x_lanes.h"
#include "genn_mi355x_causal_conv_kernels.h"
#include "genn_mi355x_scan_kernels.h"

namespace
{
Sequences sequencesOf(const gennmi_sequences_t &s, uint32_t chunk)
{
    Sequences d{};
    d.offsets = s.offsets;
    d.slots = s.slots;
    d.rows = s.rows;
    d.count = s.count;
    d.length = s.length;
    d.numSlots = s.numSlots;
    d.chunk = chunk;
    d.perSequence = std::max(1u, (s.length + chunk - 1) / chunk);
    return d;
}
// Chunk numbers: see Sequences.  Without sequences none, however many rows packed arrays hold: kernels look for the sequence of a number.
uint64_t chunkNumbers(const gennmi_sequences_t &s, uint32_t chunk)
{
    if(!s.count) { return 0; }
    return s.offsets ? s.rows / chunk + s.count : (uint64_t)s.count * std::max(1u, (s.length + chunk - 1) / chunk);
}
uint64_t totalRows(const gennmi_sequences_t &s) { return s.offsets ? s.rows : (uint64_t)s.count * s.length; }

// ---- causal convolution
// Rows of a chunk: at least taps - 1, so that only the first chunk reads the initial state
constexpr uint32_t CONV_ROWS = 16, CONV_GRADIENT_ROWS = 64, CONV_GRADIENT_THREADS = 1u << 17;

int checkConv(const char *what, const gennmi_causal_conv_t *c, bool gradients)
{
    if(!c) { return fail(GENNMI_EINVAL, std::string(what) + ": null descriptor"); }
    const auto refuse = [&](int code, const char *why) { return fail(code, std::string(what) + why); };
    const uint32_t size = sizeOf(c->type);
    if(!size) { return refuse(GENNMI_EUNSUPPORTED, ": unknown element type"); }
    if(c->taps < 1 || c->taps > GENNMI_MAX_TAPS) { return refuse(GENNMI_EUNSUPPORTED, ": number of taps"); }
    if(c->channels < 1 || c->channels > (1u << 24)) { return refuse(GENNMI_EINVAL, ": number of channels"); }
    if(const int rc = checkSequences(what, c->sequences, gradients)) { return rc; }
    if(const int rc = checkRows(what, "x", c->x, c->sequences, c->channels, size)) { return rc; }
    if(!gradients) {
        if(const int rc = checkWrittenRows(what, "out", c->out, c->sequences, c->channels, size)) { return rc; }
        if(c->out.data && c->out.data == c->x.data) { return refuse(GENNMI_EINVAL, ": out and x are the same array"); }
    }
    if(!c->weight || (uintptr_t)c->weight % 4 || (uintptr_t)c->bias % 4) { return refuse(GENNMI_EINVAL, ": weight is missing, or weight or bias not aligned"); }
    if((uintptr_t)c->initialState % size || (uintptr_t)c->finalState % size) { return refuse(GENNMI_EINVAL, ": a state is not aligned to its elements"); }
    return GENNMI_OK;
}
Region offsetsOf(const gennmi_sequences_t &s) { return regionOf("offsets", s.offsets, (s.count + 1ull) * 4); }
Region slotsOf(const gennmi_sequences_t &s) { return regionOf("slots", s.slots, s.count * 4ull); }
// An array that a call may write in place of the one it reads
Region unlessSame(const Region &r, const void *written) { return (uintptr_t)written == (uintptr_t)r.begin ? Region{r.name, 0, 0, 0, 0, 0, 0, 0} : r; }
int convApart(const char *what, const gennmi_causal_conv_t &c)
{
    const gennmi_sequences_t &s = c.sequences;
    const uint32_t size = sizeOf(c.type);
    const uint64_t states = statesOf(s) * (c.taps - 1) * c.channels * size, channels = c.channels * 4ull;
    return checkApart(what, {regionOf("out", c.out, s, c.channels, size), regionOf("the final state", c.finalState, states)}, {},
                      {regionOf("x", c.x, s, c.channels, size), regionOf("weight", c.weight, channels * c.taps), regionOf("bias", c.bias, channels),
                       unlessSame(regionOf("the initial state", c.initialState, states), c.finalState), offsetsOf(s), slotsOf(s)});
}
int convApart(const char *what, const gennmi_causal_conv_t &c, const gennmi_causal_conv_gradient_t &g, const void *workspace, size_t workspaceBytes)
{
    const gennmi_sequences_t &s = c.sequences;
    const uint32_t size = sizeOf(c.type);
    const uint64_t states = statesOf(s) * (c.taps - 1) * c.channels * size, channels = c.channels * 4ull;
    return checkApart(what, {regionOf("the gradient of x", g.x, s, c.channels, size), regionOf("the gradient of the initial state", g.initialState, states),
                             regionOf("the workspace", workspace, workspaceBytes)},
                      {regionOf("the gradient of weight", g.weight, channels * c.taps), regionOf("the gradient of bias", g.bias, channels)},
                      {regionOf("x", c.x, s, c.channels, size), regionOf("the gradient of out", g.out, s, c.channels, size), regionOf("weight", c.weight, channels * c.taps),
                       regionOf("bias", c.bias, channels), unlessSame(regionOf("the initial state", c.initialState, states), g.initialState),
                       regionOf("the gradient of the final state", g.finalState, states), offsetsOf(s)});
}
// Channels of a thread: four, for gradients two, where every row and state of them is one aligned access, else one.  (Gradients keep four rows of
// taps a channel in registers: with four channels a thread two wavefronts fit a SIMD, and 8 x 2048 rows of 2048 channels take 67 us instead of 60.)
uint32_t convVector(const gennmi_causal_conv_t &c, const gennmi_causal_conv_gradient_t *g)
{
    const uint32_t vector = g ? 2 : 4, bytes = vector * sizeOf(c.type);
    bool whole = c.channels % vector == 0;
    auto rows = [&](const gennmi_rows_t &r) { whole = whole && (uintptr_t)r.data % bytes == 0 && r.rowStride % vector == 0 && r.sequenceStride % vector == 0; };
    auto array = [&](const void *p) { whole = whole && (uintptr_t)p % bytes == 0; };
    rows(c.x);
    array(c.initialState);
    if(g) { rows(g->out); rows(g->x); array(g->initialState); array(g->finalState); }
    else { rows(c.out); array(c.finalState); }
    return whole ? vector : 1;
}
// Gradients walk taps - 1 rows beyond a chunk and write a sum for every tap behind it: the longer the chunks the better, as long as there are threads
// for the whole chip (the case above with 16, 32 and 64 rows: 73, 60 and 53 us).  The forward pass has neither (15, 16 and 22 us for 4096 x 4096).
uint32_t convChunk(const gennmi_causal_conv_t &c, bool gradients)
{
    if(!gradients) { return CONV_ROWS; }
    uint32_t chunk = CONV_GRADIENT_ROWS;
    while(chunk > CONV_ROWS && totalRows(c.sequences) / chunk * (c.channels / 2) < CONV_GRADIENT_THREADS) { chunk /= 2; }
    return chunk;
}
ConvArgs convArgs(const gennmi_causal_conv_t &c, uint32_t vector, uint32_t chunk)
{
    ConvArgs a{};
    a.sequences = sequencesOf(c.sequences, chunk);
    a.x = c.x;
    a.out = c.out;
    a.weight = c.weight;
    a.bias = c.bias;
    a.initialState = c.initialState;
    a.finalState = c.finalState;
    a.channels = c.channels;
    a.taps = c.taps;
    a.silu = c.silu;
    a.vectors = c.channels / vector;
    a.numbers = (uint32_t)chunkNumbers(c.sequences, chunk);
    return a;
}
#define EACH_TAPS TAPS(1) TAPS(2) TAPS(3) TAPS(4) TAPS(5) TAPS(6) TAPS(7) TAPS(8)
template<typename T, int VEC> void launchConv(const ConvArgs &a, dim3 grid, hipStream_t stream)
{
#define TAPS(K) case K: causalConvKernel<T, K, VEC><<<grid, dim3(256), 0, stream>>>(a); break;
    switch(a.taps) { EACH_TAPS }
#undef TAPS
}
template<typename T, int VEC> void launchConvBackward(const ConvArgs &a, const ConvGradientArgs &g, dim3 grid, hipStream_t stream)
{
#define TAPS(K) case K: causalConvBackwardKernel<T, K, VEC><<<grid, dim3(256), 0, stream>>>(a, g); break;
    switch(a.taps) { EACH_TAPS }
#undef TAPS
}
#undef EACH_TAPS
uint64_t convBlocks(const gennmi_causal_conv_t &c, uint32_t vector, uint32_t chunk) { return (chunkNumbers(c.sequences, chunk) * (c.channels / vector) + 255) / 256; }
int runConv(const char *what, const gennmi_causal_conv_t &c, uint32_t vector, const ConvGradientArgs *g, hipStream_t stream)
{
    const uint32_t chunk = convChunk(c, g != nullptr);
    const ConvArgs a = convArgs(c, vector, chunk);
    const uint64_t blocks = convBlocks(c, vector, chunk);
    if(!blocks) { return GENNMI_OK; }
    return withType(c.type, [&](auto t) {
        const dim3 grid((uint32_t)blocks);
        if(g) { if(vector == 2) { launchConvBackward<decltype(t), 2>(a, *g, grid, stream); } else { launchConvBackward<decltype(t), 1>(a, *g, grid, stream); } }
        else if(vector == 4) { launchConv<decltype(t), 4>(a, grid, stream); }
        else { launchConv<decltype(t), 1>(a, grid, stream); }
        return gennmi_detail::afterLaunch(what);
    });
}
size_t convWorkspace(const gennmi_causal_conv_t &c) { return (size_t)chunkNumbers(c.sequences, convChunk(c, true)) * (c.taps + 1) * c.channels * sizeof(float); }

// ---- selective scan
int checkScan(const char *what, const gennmi_scan_t *c, bool gradients)
{
    if(!c) { return fail(GENNMI_EINVAL, std::string(what) + ": null descriptor"); }
    const auto refuse = [&](int code, const char *why) { return fail(code, std::string(what) + why); };
    const uint32_t size = sizeOf(c->type);
    if(!size) { return refuse(GENNMI_EUNSUPPORTED, ": unknown element type"); }
    if(c->states < 1 || c->states > GENNMI_MAX_SCAN_STATES) { return refuse(GENNMI_EUNSUPPORTED, ": number of states"); }
    if(c->channels < 1 || c->channels > (1u << 24) || c->groups < 1 || c->channels % c->groups) { return refuse(GENNMI_EINVAL, ": number of channels or groups"); }
    if(const int rc = checkSequences(what, c->sequences, gradients)) { return rc; }
    if(const int rc = checkRows(what, "u", c->u, c->sequences, c->channels, size)) { return rc; }
    if(const int rc = checkRows(what, "delta", c->delta, c->sequences, c->channels, size)) { return rc; }
    if(const int rc = checkRows(what, "B", c->B, c->sequences, c->groups * c->states, size)) { return rc; }
    if(const int rc = checkRows(what, "C", c->C, c->sequences, c->groups * c->states, size)) { return rc; }
    if(c->z.data) { if(const int rc = checkRows(what, "z", c->z, c->sequences, c->channels, size)) { return rc; } }
    if(!gradients) {
        if(const int rc = checkWrittenRows(what, "out", c->out, c->sequences, c->channels, size)) { return rc; }
        for(const void *p : {c->u.data, c->delta.data, c->z.data, c->B.data, c->C.data}) {
            if(p && p == c->out.data) { return refuse(GENNMI_EINVAL, ": out is an array of its own"); }
        }
    }
    if(!c->A) { return refuse(GENNMI_EINVAL, ": A is missing"); }
    for(const void *p : {(const void*)c->A, (const void*)c->D, (const void*)c->deltaBias, (const void*)c->initialState, (const void*)c->finalState}) {
        if((uintptr_t)p % 4) { return refuse(GENNMI_EINVAL, ": an array of fp32 is not aligned"); }
    }
    return GENNMI_OK;
}

int scanApart(const char *what, const gennmi_scan_t &c, const void *workspace, size_t workspaceBytes)
{
    const gennmi_sequences_t &s = c.sequences;
    const uint32_t size = sizeOf(c.type), width = c.groups * c.states;
    const uint64_t channels = c.channels * 4ull, states = statesOf(s) * channels * c.states;
    return checkApart(what, {regionOf("out", c.out, s, c.channels, size), regionOf("the final state", c.finalState, states), regionOf("the workspace", workspace, workspaceBytes)}, {},
                      {regionOf("u", c.u, s, c.channels, size), regionOf("delta", c.delta, s, c.channels, size), regionOf("z", c.z, s, c.channels, size), regionOf("B", c.B, s, width, size),
                       regionOf("C", c.C, s, width, size), regionOf("A", c.A, channels * c.states), regionOf("D", c.D, channels), regionOf("delta's bias", c.deltaBias, channels),
                       unlessSame(regionOf("the initial state", c.initialState, states), c.finalState), offsetsOf(s), slotsOf(s)});
}
int scanApart(const char *what, const gennmi_scan_t &c, const gennmi_scan_gradient_t &g, const void *workspace, size_t workspaceBytes)
{
    const gennmi_sequences_t &s = c.sequences;
    const uint32_t size = sizeOf(c.type), width = c.groups * c.states;
    const uint64_t channels = c.channels * 4ull, states = statesOf(s) * channels * c.states;
    return checkApart(what, {regionOf("the gradient of u", g.u, s, c.channels, size), regionOf("the gradient of delta", g.delta, s, c.channels, size),
                             regionOf("the gradient of z", g.z, s, c.channels, size), regionOf("the gradient of B", g.B, s, width, size), regionOf("the gradient of C", g.C, s, width, size),
                             regionOf("the gradient of the initial state", g.initialState, states), regionOf("the workspace", workspace, workspaceBytes)},
                      {regionOf("the gradient of A", g.A, channels * c.states), regionOf("the gradient of D", g.D, channels), regionOf("the gradient of delta's bias", g.deltaBias, channels)},
                      {regionOf("u", c.u, s, c.channels, size), regionOf("delta", c.delta, s, c.channels, size), regionOf("z", c.z, s, c.channels, size), regionOf("B", c.B, s, width, size),
                       regionOf("C", c.C, s, width, size), regionOf("the gradient of out", g.out, s, c.channels, size), regionOf("A", c.A, channels * c.states), regionOf("D", c.D, channels),
                       regionOf("delta's bias", c.deltaBias, channels), unlessSame(regionOf("the initial state", c.initialState, states), g.initialState),
                       unlessSame(regionOf("the gradient of the final state", g.finalState, states), g.initialState), offsetsOf(s)});
}

struct ScanPlan { uint32_t slab, slabs, chunk; bool split; };
constexpr uint32_t SCAN_BLOCK_ROWS = 8;
// Blocks of rows of a chunk of gradients: what is kept of each takes 4 KiB of LDS a wavefront, and eight wavefronts of one, or of a work-group of
// several, should fit a compute unit's 160
constexpr uint32_t gradientBlocks(uint32_t slabs) { return slabs > 1 ? 2 : 4; }

uint32_t scanTiles(const gennmi_scan_t &c) { return c.groups * ((c.channels / c.groups + 63) / 64); }
// States of a wavefront, wavefronts of a work-group, rows of a chunk
ScanPlan scanPlan(const gennmi_scan_t &c, bool gradients)
{
    ScanPlan p;
    p.slab = c.states <= 8 ? 8 : 16;
    p.slabs = (c.states + p.slab - 1) / p.slab;
    // The chunk (or, of a forward scan, the whole sequence, which is walked once instead of twice) that the busiest SIMD is through with first.  A row takes a
    // wavefront's SIMD a certain time however many share it, but a quarter more where one is alone; a chunk takes as long as 4 rows more, and in the walk
    // over the chunks as long as an eighth of a row.  4096 rows x 2048 channels in chunks of 32, 64, 128: 93, 90, 106 us; 33 sequences of 8011 rows in all x
    // 1002 channels in chunks of 32, 48, 64, 96: 108, 108, 118, 134 us.  Gradients of 3 sequences of 301 rows x 511 channels in chunks of 32 and 8: 64, 39 us,
    // of one of 7900 rows x 65 channels in chunks of 8 and 32: 213, 125 us.
    constexpr uint64_t SIMDS = 1024;
    const uint64_t rows = totalRows(c.sequences), wavesEach = (uint64_t)scanTiles(c) * p.slabs, length = std::max(1u, c.sequences.length);
    const auto cost = [&](uint32_t chunk) {
        // (how packed sequences fall into chunks is the device's to know: half a share for what does not come out even)
        const double chunks = c.sequences.offsets ? (double)rows / chunk + 0.5 * c.sequences.count : (double)c.sequences.count * ((length + chunk - 1) / chunk);
        const double even = chunks * wavesEach / SIMDS, share = c.sequences.offsets ? even + 0.5 : std::ceil(even);
        return std::max(1.25, share) * (chunk + 4) + 0.13 * (length / chunk);
    };
    if(gradients) {
        p.chunk = SCAN_BLOCK_ROWS;
        for(uint32_t blocks = 2; blocks <= gradientBlocks(p.slabs); blocks *= 2) {
            if(cost(SCAN_BLOCK_ROWS * blocks) < cost(p.chunk)) { p.chunk = SCAN_BLOCK_ROWS * blocks; }
        }
    }
    else {
        p.chunk = (uint32_t)length;
        double best = std::max(1.25, std::ceil((double)c.sequences.count * wavesEach / SIMDS)) * length * 0.55;
        for(uint32_t chunk = 32; chunk <= 1024 && chunk < length; chunk += chunk < 256 ? 8 : 64) {
            if(cost(chunk) < best) { best = cost(chunk); p.chunk = chunk; }
        }
    }
    p.split = c.sequences.length > p.chunk;
    return p;
}
struct ScanSpace { size_t state, time, gradient, sums, sumBC, bytes; };
ScanSpace scanSpace(const gennmi_scan_t &c, const ScanPlan &p, bool gradients)
{
    ScanSpace s{};
    const uint64_t numbers = chunkNumbers(c.sequences, p.chunk);
    auto take = [&](uint64_t floats) { const size_t at = s.bytes; s.bytes += (floats * sizeof(float) + 255) / 256 * 256; return at; };
    if(p.split) {
        s.state = take(numbers * c.states * c.channels);
        s.time = take(numbers * c.channels);
    }
    if(gradients) {
        if(p.split) { s.gradient = take(numbers * c.states * c.channels); }
        s.sums = take(numbers * (c.states + 2) * c.channels);
        s.sumBC = take((uint64_t)scanTiles(c) * totalRows(c.sequences) * 2 * c.states);
    }
    return s;
}
// A token's states are shared by that many lanes, four each
uint32_t tokenLanes(uint32_t states) { return states <= 4 ? 1 : states <= 8 ? 2 : states <= 16 ? 4 : states <= 32 ? 8 : states <= 64 ? 16 : 32; }
uint64_t tokenBlocks(const gennmi_scan_t &c) { return ((uint64_t)c.sequences.count * c.channels * tokenLanes(c.states) + 255) / 256; }
// Whether the launches of a pass, but for the closing sums of gradients, cover it
bool scanFits(const gennmi_scan_t &c, const ScanPlan &p, bool gradients)
{
    if(!gradients && c.sequences.length <= 1) { return tokenBlocks(c) <= mostBlocks(256); }
    const bool join = p.split && (uint64_t)c.sequences.count * c.states * ((c.channels + 63) / 64) > mostBlocks(64);
    return chunkNumbers(c.sequences, p.chunk) * scanTiles(c) <= mostBlocks(64 * p.slabs) && !join;
}
ScanArgs scanArgs(const gennmi_scan_t &c, const ScanPlan &p)
{
    ScanArgs a{};
    const uint64_t numbers = chunkNumbers(c.sequences, p.chunk), tiles = scanTiles(c);
    a.sequences = sequencesOf(c.sequences, p.chunk);
    a.u = c.u; a.delta = c.delta; a.z = c.z; a.out = c.out; a.B = c.B; a.C = c.C;
    a.A = c.A; a.D = c.D; a.deltaBias = c.deltaBias;
    a.initialState = c.initialState; a.finalState = c.finalState;
    a.channels = c.channels; a.states = c.states; a.groups = c.groups; a.softplus = c.softplus;
    a.groupChannels = c.channels / c.groups;
    a.groupTiles = (a.groupChannels + 63) / 64;
    a.tiles = (uint32_t)tiles;
    a.numbers = (uint32_t)numbers;
    a.slabs = p.slabs;
    return a;
}
int checkWorkspace(const char *what, const void *workspace, size_t have, size_t need)
{
    if(need && (!workspace || have < need)) { return fail(GENNMI_EINVAL, std::string(what) + ": workspace is missing or too small"); }
    return (uintptr_t)workspace % 16 ? fail(GENNMI_EINVAL, std::string(what) + ": workspace is not 16-byte aligned") : GENNMI_OK;
}

template<typename T, int NP, bool SLABS> int launchScan(const ScanArgs &a, const ScanPlan &p, hipStream_t stream)
{
    const dim3 grid(a.numbers * a.tiles), threads(64 * p.slabs);
    if(p.split) {
        scanChunkKernel<T, NP, false, SLABS><<<grid, threads, 0, stream>>>(a, ScanGradientArgs{});
        if(const int rc = gennmi_detail::afterLaunch("selective_scan")) { return rc; }
        scanJoinKernel<false><<<dim3(a.sequences.count * a.states * ((a.channels + 63) / 64)), dim3(64), 0, stream>>>(a, ScanGradientArgs{});
        if(const int rc = gennmi_detail::afterLaunch("selective_scan")) { return rc; }
    }
    scanKernel<T, NP, SLABS><<<grid, threads, 0, stream>>>(a);
    return gennmi_detail::afterLaunch("selective_scan");
}
template<typename T, int LANES> int launchToken(const ScanArgs &a, uint32_t blocks, hipStream_t stream)
{
    // four states a lane in one access, where every array lies so
    const auto fours = [](const void *p, uint32_t size) { return (uintptr_t)p % (4 * size) == 0; };
    const auto rows = [&](const gennmi_rows_t &r) { return fours(r.data, sizeof(T)) && r.rowStride % 4 == 0 && r.sequenceStride % 4 == 0; };
    const bool quads = a.states % 4 == 0 && fours(a.A, 4) && fours(a.initialState, 4) && fours(a.finalState, 4) && rows(a.B) && rows(a.C);
    const dim3 grid(blocks);
    if(quads) { scanTokenKernel<T, LANES, true><<<grid, dim3(256), 0, stream>>>(a); } else { scanTokenKernel<T, LANES, false><<<grid, dim3(256), 0, stream>>>(a); }
    return gennmi_detail::afterLaunch("selective_scan");
}
template<typename T, int NP, bool SLABS> int launchScanBackward(const ScanArgs &a, const ScanGradientArgs &g, const ScanPlan &p, hipStream_t stream)
{
    const dim3 grid(a.numbers * a.tiles), threads(64 * p.slabs);
    if(p.split) {
        scanChunkKernel<T, NP, true, SLABS><<<grid, threads, 0, stream>>>(a, g);
        if(const int rc = gennmi_detail::afterLaunch("selective_scan_backward")) { return rc; }
        scanJoinKernel<true><<<dim3(a.sequences.count * a.states * ((a.channels + 63) / 64)), dim3(64), 0, stream>>>(a, g);
        if(const int rc = gennmi_detail::afterLaunch("selective_scan_backward")) { return rc; }
    }
    constexpr uint32_t BLOCKS = gradientBlocks(SLABS ? 2 : 1);
    const size_t lds = sizeof(float) * (p.slabs * (BLOCKS * NP * 64 + SCAN_BLOCK_ROWS * (2 * NP * 2 + 64)) + (SLABS ? p.slabs * SCAN_BLOCK_ROWS * 3 * 64 : 0));
    auto kernel = scanBackwardKernel<T, NP, (int)SCAN_BLOCK_ROWS, (int)BLOCKS, SLABS>;
    if(lds > 65536) {
        const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
        if(e != hipSuccess) { return fail(GENNMI_EHIP, std::string("selective_scan_backward: ") + hipGetErrorString(e)); }
    }
    kernel<<<grid, threads, lds, stream>>>(a, g);
    return gennmi_detail::afterLaunch("selective_scan_backward");
}
// Picks the instance: states of a wavefront, and whether several wavefronts share a channel
template<typename F> int withStates(const ScanPlan &p, F &&f)
{
    if(p.slabs > 1) { return f(std::integral_constant<int, 16>{}, std::true_type{}); }
    if(p.slab == 16) { return f(std::integral_constant<int, 16>{}, std::false_type{}); }
    return f(std::integral_constant<int, 8>{}, std::false_type{});
}
}

extern "C" {

int gennmi_stream_is_capturing(void *stream, int *capturing)
{
    if(!capturing) { return fail(GENNMI_EINVAL, "stream_is_capturing: null result pointer"); }
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if(stream) {
        const hipError_t e = hipStreamIsCapturing((hipStream_t)stream, &status);
        if(e != hipSuccess) { return fail(GENNMI_EHIP, std::string("stream_is_capturing: ") + hipGetErrorString(e)); }
    }
    *capturing = status != hipStreamCaptureStatusNone;
    return GENNMI_OK;
}

int gennmi_current_device(int *device)
{
    if(!device) { return fail(GENNMI_EINVAL, "current_device: null result pointer"); }
    const hipError_t e = hipGetDevice(device);
    return e == hipSuccess ? (int)GENNMI_OK : fail(GENNMI_EHIP, std::string("current_device: ") + hipGetErrorString(e));
}

int gennmi_causal_conv(const gennmi_causal_conv_t *conv, void *stream)
{
    return gennmi_detail::guarded("causal_conv", [&] {
        if(const int rc = checkConv("causal_conv", conv, false)) { return rc; }
        const uint32_t vector = convVector(*conv, nullptr);
        if(convBlocks(*conv, vector, convChunk(*conv, false)) > mostBlocks(256)) { return tooMany("causal_conv"); }
        if(const int rc = convApart("causal_conv", *conv)) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, conv->sequences.device)) { return rc; }
        if(const int rc = runConv("causal_conv", *conv, vector, nullptr, (hipStream_t)stream)) { return rc; }
        const uint32_t size = sizeOf(conv->type);
        noteRows(conv->out, conv->sequences, conv->channels, size);
        if(conv->finalState) { gennmi_detail::noteDeviceWrite(conv->finalState, statesOf(conv->sequences) * (conv->taps - 1) * conv->channels * size); }
        return (int)GENNMI_OK;
    });
}

int gennmi_causal_conv_backward_workspace(const gennmi_causal_conv_t *conv, size_t *bytes)
{
    return gennmi_detail::guarded("causal_conv_backward_workspace", [&] {
        if(const int rc = checkConv("causal_conv_backward_workspace", conv, true)) { return rc; }
        if(!bytes) { return fail(GENNMI_EINVAL, "causal_conv_backward_workspace: null result pointer"); }
        *bytes = convWorkspace(*conv);
        return (int)GENNMI_OK;
    });
}

int gennmi_causal_conv_backward(const gennmi_causal_conv_t *conv, const gennmi_causal_conv_gradient_t *gradient, void *workspace, size_t workspaceBytes,
                                void *stream)
{
    const char *what = "causal_conv_backward";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkConv(what, conv, true)) { return rc; }
        if(!gradient) { return fail(GENNMI_EINVAL, "causal_conv_backward: null gradient"); }
        const gennmi_causal_conv_gradient_t &g = *gradient;
        const uint32_t size = sizeOf(conv->type);
        if(const int rc = checkRows(what, "the gradient of out", g.out, conv->sequences, conv->channels, size)) { return rc; }
        if(g.x.data) {
            if(const int rc = checkWrittenRows(what, "the gradient of x", g.x, conv->sequences, conv->channels, size)) { return rc; }
            if(g.x.data == g.out.data || g.x.data == conv->x.data) { return fail(GENNMI_EINVAL, "causal_conv_backward: the gradient of x is an array of its own"); }
        }
        if((uintptr_t)g.finalState % size || (uintptr_t)g.initialState % size || (uintptr_t)g.weight % 4 || (uintptr_t)g.bias % 4) {
            return fail(GENNMI_EINVAL, "causal_conv_backward: an array is not aligned to its elements");
        }
        if(g.initialState && g.initialState == g.finalState) { return fail(GENNMI_EINVAL, "causal_conv_backward: the gradient of initialState is an array of its own"); }
        const bool sums = g.weight || g.bias;
        const uint32_t vector = convVector(*conv, gradient);
        if(convBlocks(*conv, vector, convChunk(*conv, true)) > mostBlocks(256) || (sums && chunkSumBlocks(conv->taps + 1, conv->channels) > mostBlocks(1024))) { return tooMany(what); }
        const size_t need = sums ? convWorkspace(*conv) : 0;
        if(const int rc = checkWorkspace(what, workspace, workspaceBytes, need)) { return rc; }
        if(const int rc = convApart(what, *conv, g, workspace, need)) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, conv->sequences.device)) { return rc; }
        ConvGradientArgs a{};
        a.out = g.out;
        a.x = g.x;
        a.finalState = g.finalState;
        a.initialState = g.initialState;
        a.partial = sums ? (float*)workspace : nullptr;
        if(const int rc = runConv(what, *conv, vector, &a, (hipStream_t)stream)) { return rc; }
        if(sums) {
            const ChunkSums c{a.partial, g.weight, {g.bias, nullptr}, (uint32_t)chunkNumbers(conv->sequences, convChunk(*conv, true)), conv->channels, conv->taps, conv->taps + 1};
            if(const int rc = launchChunkSum(what, c, (hipStream_t)stream)) { return rc; }
        }
        noteRows(g.x, conv->sequences, conv->channels, size);
        if(g.initialState) { gennmi_detail::noteDeviceWrite(g.initialState, (uint64_t)conv->sequences.count * (conv->taps - 1) * conv->channels * size); }
        if(g.weight) { gennmi_detail::noteDeviceWrite(g.weight, (uint64_t)conv->channels * conv->taps * sizeof(float)); }
        if(g.bias) { gennmi_detail::noteDeviceWrite(g.bias, conv->channels * sizeof(float)); }
        return (int)GENNMI_OK;
    });
}

int gennmi_selective_scan_workspace(const gennmi_scan_t *scan, size_t *bytes)
{
    return gennmi_detail::guarded("selective_scan_workspace", [&] {
        if(const int rc = checkScan("selective_scan_workspace", scan, false)) { return rc; }
        if(!bytes) { return fail(GENNMI_EINVAL, "selective_scan_workspace: null result pointer"); }
        const ScanPlan p = scanPlan(*scan, false);
        if(!scanFits(*scan, p, false)) { return tooMany("selective_scan_workspace"); }
        *bytes = scanSpace(*scan, p, false).bytes;
        return (int)GENNMI_OK;
    });
}

int gennmi_selective_scan(const gennmi_scan_t *scan, void *workspace, size_t workspaceBytes, void *stream)
{
    const char *what = "selective_scan";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkScan(what, scan, false)) { return rc; }
        const ScanPlan p = scanPlan(*scan, false);
        if(!scanFits(*scan, p, false)) { return tooMany(what); }
        const ScanSpace space = scanSpace(*scan, p, false);
        if(const int rc = checkWorkspace(what, workspace, workspaceBytes, space.bytes)) { return rc; }
        if(const int rc = scanApart(what, *scan, workspace, space.bytes)) { return rc; }
        ScanArgs a = scanArgs(*scan, p);
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, scan->sequences.device)) { return rc; }
        if(!scan->sequences.count) { return (int)GENNMI_OK; }
        if(p.split) {
            a.chunkState = (float*)((char*)workspace + space.state);
            a.chunkTime = (float*)((char*)workspace + space.time);
        }
        const int rc = withType(scan->type, [&](auto t) {
            typedef decltype(t) T;
            if(scan->sequences.length <= 1) {
                const uint32_t blocks = (uint32_t)tokenBlocks(*scan);
                switch(tokenLanes(a.states)) {
                case 1: return launchToken<T, 1>(a, blocks, (hipStream_t)stream);
                case 2: return launchToken<T, 2>(a, blocks, (hipStream_t)stream);
                case 4: return launchToken<T, 4>(a, blocks, (hipStream_t)stream);
                case 8: return launchToken<T, 8>(a, blocks, (hipStream_t)stream);
                case 16: return launchToken<T, 16>(a, blocks, (hipStream_t)stream);
                default: return launchToken<T, 32>(a, blocks, (hipStream_t)stream);
                }
            }
            return withStates(p, [&](auto np, auto slabs) { return launchScan<T, decltype(np)::value, decltype(slabs)::value>(a, p, (hipStream_t)stream); });
        });
        if(rc) { return rc; }
        noteRows(scan->out, scan->sequences, scan->channels, sizeOf(scan->type));
        if(scan->finalState) { gennmi_detail::noteDeviceWrite(scan->finalState, statesOf(scan->sequences) * scan->channels * scan->states * sizeof(float)); }
        return (int)GENNMI_OK;
    });
}

int gennmi_selective_scan_backward_workspace(const gennmi_scan_t *scan, size_t *bytes)
{
    return gennmi_detail::guarded("selective_scan_backward_workspace", [&] {
        if(const int rc = checkScan("selective_scan_backward_workspace", scan, true)) { return rc; }
        if(!bytes) { return fail(GENNMI_EINVAL, "selective_scan_backward_workspace: null result pointer"); }
        const ScanPlan p = scanPlan(*scan, true);
        if(!scanFits(*scan, p, true)) { return tooMany("selective_scan_backward_workspace"); }
        *bytes = scanSpace(*scan, p, true).bytes;
        return (int)GENNMI_OK;
    });
}

int gennmi_selective_scan_backward(const gennmi_scan_t *scan, const gennmi_scan_gradient_t *gradient, void *workspace, size_t workspaceBytes, void *stream)
{
    const char *what = "selective_scan_backward";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkScan(what, scan, true)) { return rc; }
        if(!gradient) { return fail(GENNMI_EINVAL, "selective_scan_backward: null gradient"); }
        const gennmi_scan_gradient_t &in = *gradient;
        const uint32_t size = sizeOf(scan->type), width = scan->groups * scan->states;
        if(const int rc = checkRows(what, "the gradient of out", in.out, scan->sequences, scan->channels, size)) { return rc; }
        const struct { const char *which; const gennmi_rows_t *rows; uint32_t width; } written[] = {
            {"the gradient of u", &in.u, scan->channels}, {"the gradient of delta", &in.delta, scan->channels}, {"the gradient of z", &in.z, scan->channels},
            {"the gradient of B", &in.B, width}, {"the gradient of C", &in.C, width}};
        for(const auto &w : written) {
            if(!w.rows->data) { continue; }
            if(const int rc = checkWrittenRows(what, w.which, *w.rows, scan->sequences, w.width, size)) { return rc; }
            const void *others[] = {scan->u.data, scan->delta.data, scan->z.data, scan->B.data, scan->C.data, in.out.data,
                                    w.rows == &in.u ? nullptr : in.u.data, w.rows == &in.delta ? nullptr : in.delta.data, w.rows == &in.z ? nullptr : in.z.data, w.rows == &in.B ? nullptr : in.B.data};
            for(const void *p : others) {
                if(p == w.rows->data) { return fail(GENNMI_EINVAL, std::string(what) + ": " + w.which + " is an array of its own"); }
            }
        }
        if(in.z.data && !scan->z.data) { return fail(GENNMI_EINVAL, "selective_scan_backward: a gradient of z without z"); }
        for(const void *p : {(const void*)in.finalState, (const void*)in.initialState, (const void*)in.A, (const void*)in.D, (const void*)in.deltaBias}) {
            if((uintptr_t)p % 4) { return fail(GENNMI_EINVAL, "selective_scan_backward: an array of fp32 is not aligned"); }
        }
        const ScanPlan p = scanPlan(*scan, true);
        const uint64_t rows = totalRows(scan->sequences), rowSumBlocks = in.B.data || in.C.data ? (rows * 2 * width + 255) / 256 : 0;
        const uint64_t sumBlocks = in.A || in.D || in.deltaBias ? chunkSumBlocks(scan->states + 2, scan->channels) : 0;
        if(!scanFits(*scan, p, true) || rowSumBlocks > mostBlocks(256) || sumBlocks > mostBlocks(1024)) { return tooMany(what); }
        const ScanSpace space = scanSpace(*scan, p, true);
        if(const int rc = checkWorkspace(what, workspace, workspaceBytes, space.bytes)) { return rc; }
        if(const int rc = scanApart(what, *scan, in, workspace, space.bytes)) { return rc; }
        ScanArgs a = scanArgs(*scan, p);
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, scan->sequences.device)) { return rc; }
        auto at = [&](size_t offset) { return (float*)((char*)workspace + offset); };
        a.finalState = nullptr;
        ScanGradientArgs g{};
        g.out = in.out; g.u = in.u; g.delta = in.delta; g.z = in.z; g.B = in.B; g.C = in.C;
        g.finalState = in.finalState; g.initialState = in.initialState;
        if(p.split) {
            a.chunkState = at(space.state);
            a.chunkTime = at(space.time);
            g.chunkGradient = at(space.gradient);
        }
        g.sums = at(space.sums);
        g.sumBC = at(space.sumBC);      // (written whatever gradients are asked for)
        g.rows = rows;
        const hipStream_t s = (hipStream_t)stream;
        if(a.numbers) {
            const int rc = withType(scan->type, [&](auto t) {
                typedef decltype(t) T;
                const int rcScan = withStates(p, [&](auto np, auto slabs) { return launchScanBackward<T, decltype(np)::value, decltype(slabs)::value>(a, g, p, s); });
                if(rcScan || !rowSumBlocks) { return rcScan; }
                scanRowSumKernel<T><<<dim3((uint32_t)rowSumBlocks), dim3(256), 0, s>>>(a, g);
                return gennmi_detail::afterLaunch(what);
            });
            if(rc) { return rc; }
        }
        if(in.A || in.D || in.deltaBias) {
            if(const int rc = launchChunkSum(what, {g.sums, in.A, {in.D, in.deltaBias}, a.numbers, a.channels, a.states, a.states + 2}, s)) { return rc; }
            const struct { float *out; uint64_t count; } sums[] = {{in.A, (uint64_t)a.channels * a.states}, {in.D, a.channels}, {in.deltaBias, a.channels}};
            for(const auto &c : sums) { if(c.out) { gennmi_detail::noteDeviceWrite(c.out, c.count * sizeof(float)); } }
        }
        for(const auto &w : written) { noteRows(*w.rows, scan->sequences, w.width, size); }
        if(in.initialState) { gennmi_detail::noteDeviceWrite(in.initialState, (uint64_t)scan->sequences.count * scan->channels * scan->states * sizeof(float)); }
        return (int)GENNMI_OK;
    });
}

}

// Part of libgenn_mi355x.so: element types, rows and sequences, as the operators' translation units share them.
#ifndef GENN_MI355X_ELEMENTS_H
#define GENN_MI355X_ELEMENTS_H

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <utility>

#include "genn_mi355x.h"

namespace gennmi_detail
{
// (defined beside the runner)
int fail(int code, const std::string &msg);
void noteDeviceWrite(const void *dev, size_t bytes);
bool anyRunners();          // that would have to be told
int flushQueuedSteps();
bool stepsQueued();

// What every operator does before it launches: it makes sure of the device (0, or 1 + the arrays'), and steps queued in runners run first.
// Under capture they cannot: their launches would join the null stream's order, which a capture forbids.
inline int beforeLaunch(hipStream_t stream, uint32_t device)
{
    if(device) {
        int current = -1;
        const hipError_t e = hipGetDevice(&current);
        if(e != hipSuccess) { return fail(GENNMI_EHIP, std::string("current device: ") + hipGetErrorString(e)); }
        if((uint32_t)current != device - 1) { return fail(GENNMI_ESTATE, "the current device is " + std::to_string(current) + ", the arrays are on device " + std::to_string(device - 1)); }
    }
    if(!stepsQueued()) { return GENNMI_OK; }
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    if(stream && hipStreamIsCapturing(stream, &status) == hipSuccess && status != hipStreamCaptureStatusNone) {
        return fail(GENNMI_ESTATE, "steps are queued in a runner while the stream is captured: call gennmi_flush before");
    }
    return flushQueuedSteps();
}
inline int afterLaunch(const char *what)
{
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? GENNMI_OK : fail(GENNMI_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}
// An entry point's body: no C++ exception leaves the library
template<typename F> int guarded(const char *what, F &&body)
{
    try { return body(); }
    catch(const std::exception &e) { try { return fail(GENNMI_EHIP, std::string(what) + ": " + e.what()); } catch(...) { return GENNMI_EHIP; } }
    catch(...) { return GENNMI_EHIP; }
}
}

namespace gennmi_elements
{
// Types are converted by the hardware's instructions, to fewer bits with ties to even
typedef __bf16 bf16;
typedef _Float16 f16;
template<typename T> __device__ inline float widen(T x) { return (float)x; }
template<typename T> __device__ inline T narrow(float x) { return (T)x; }

inline uint32_t sizeOf(uint32_t type) { return type == GENNMI_TYPE_F32 ? 4 : (type == GENNMI_TYPE_F16 || type == GENNMI_TYPE_BF16) ? 2 : 0; }

// Calls f with a value of the element type, which picks the instance
template<typename F> int withType(uint32_t type, F &&f)
{
    switch(type) {
    case GENNMI_TYPE_F32: return f(float{});
    case GENNMI_TYPE_F16: return f(f16{});
    default: return f(bf16{});
    }
}

// N neighbouring elements in one access
template<typename T, int N> struct alignas(sizeof(T) * N) Pack { T v[N]; };

// Which rows a work-group owns.  Sequences are cut into chunks of `chunk` rows; a packed sequence's chunks are numbered from
// offsets[s] / chunk + s, so that rows / chunk + count numbers do for any lengths, and every sequence (also one without rows) has one.
struct Sequences
{
    const uint32_t *offsets;
    const int32_t *slots;
    uint64_t rows;
    uint32_t count, length, numSlots, chunk, perSequence;      // perSequence: chunk numbers of a sequence that is not packed
};
struct Place
{
    uint64_t first;         // packed: the sequence's first row; else 0
    uint32_t sequence, index, length;       // index: number of the chunk in its sequence
    int32_t state;
};
__device__ inline uint64_t firstRow(const Sequences &s, uint32_t sequence)
{
    const uint64_t at = s.offsets[sequence];
    return at < s.rows ? at : s.rows;
}
__device__ inline uint64_t firstChunk(const Sequences &s, uint32_t sequence)
{
    return s.offsets ? firstRow(s, sequence) / s.chunk + sequence : (uint64_t)sequence * s.perSequence;
}
// false: padding, nothing to do
__device__ inline bool describe(const Sequences &s, uint32_t sequence, Place &p)
{
    p.sequence = sequence;
    p.first = 0;
    p.length = s.length;
    if(s.offsets) {
        p.first = firstRow(s, sequence);
        const uint64_t end = firstRow(s, sequence + 1);
        p.length = end > p.first ? (uint32_t)(end - p.first < s.length ? end - p.first : s.length) : 0;
    }
    p.state = s.slots ? s.slots[sequence] : (int32_t)sequence;
    return !s.slots || (p.state >= 0 && (uint32_t)p.state < s.numSlots);
}
// The sequence that chunk number `number` belongs to (uniform over the wavefront); 64 candidates are looked at a time
__device__ inline bool locate(const Sequences &s, uint32_t number, Place &p)
{
    uint32_t sequence;
    if(!s.offsets) {
        sequence = number / s.perSequence;
        p.index = number - sequence * s.perSequence;
    }
    else {
        const uint32_t lane = threadIdx.x & 63;
        uint32_t low = 0, span = s.count;       // the answer is in low .. low + span - 1
        while(span > 1) {
            const uint32_t step = (span + 63) / 64;
            const uint32_t candidate = low + lane * step;
            const bool below = lane * step < span && firstChunk(s, candidate) <= number;
            const uint64_t votes = __ballot(below);
            const uint32_t last = votes ? 63 - __clzll((long long)votes) : 0;
            low += last * step;
            span = min(step, span - last * step);
        }
        sequence = __builtin_amdgcn_readfirstlane(low);
        p.index = __builtin_amdgcn_readfirstlane(number - (uint32_t)firstChunk(s, sequence));
    }
    if(sequence >= s.count || !describe(s, sequence, p)) { return false; }
    return (uint64_t)p.index * s.chunk < p.length || p.index == 0;
}
template<typename T> __device__ inline T *rowsOf(const gennmi_rows_t &r, const Sequences &s, const Place &p)
{
    return (T*)r.data + (s.offsets ? p.first * r.rowStride : (uint64_t)p.sequence * r.sequenceStride);
}

// A thread's number in its launch of 256 a work-group, divided by `by` (32 bits do: see mostBlocks)
__device__ inline void divideItem(uint32_t by, uint32_t &quotient, uint32_t &rest)
{
    const uint32_t item = blockIdx.x * 256 + threadIdx.x;
    quotient = item / by;
    rest = item - quotient * by;
}

// Work-groups of that many threads that one launch takes: its threads are numbered in 32 bits
constexpr uint64_t mostBlocks(uint32_t threads) { return 0xffffffffull / threads; }

// host side (a call of a few microseconds: texts are put together for a refusal only)
inline int checkSequences(const char *what, const gennmi_sequences_t &s, bool gradients)
{
    const auto refuse = [&](const char *why) { return gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + why); };
    if(s.slots && gradients) { return refuse(": slots are not for gradients"); }
    if(s.count > (1u << 24) || s.length > 0x7fffffffu || (s.offsets ? s.rows : (uint64_t)s.count * s.length) > 0x7fffffffull) { return refuse(": more sequences or rows than the kernels number"); }
    if(s.slots && s.numSlots == 0) { return refuse(": slots, but no states (numSlots is 0)"); }
    if((uintptr_t)s.offsets % 4 || (uintptr_t)s.slots % 4) { return refuse(": offsets or slots not aligned"); }
    return GENNMI_OK;
}
inline int checkRows(const char *what, const char *which, const gennmi_rows_t &r, const gennmi_sequences_t &s, uint32_t width, uint32_t size)
{
    const auto refuse = [&](const char *why) { return gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + ": " + which + why); };
    if(!(s.offsets ? s.rows : (uint64_t)s.count * s.length)) { return GENNMI_OK; }       // (nothing of it is touched)
    if(!r.data) { return refuse(" is missing"); }
    if((uintptr_t)r.data % size) { return refuse(" is not aligned to its elements"); }
    if(s.length > 1 && r.rowStride < width) { return refuse(": rows overlap (rowStride)"); }
    if((r.rowStride > 0xffffffffull && (s.length > 1 || s.offsets)) || r.sequenceStride > (1ull << 50)) { return refuse(": stride out of range"); }
    return GENNMI_OK;
}
// What is written: one row of a sequence and another must not share elements either
inline int checkWrittenRows(const char *what, const char *which, const gennmi_rows_t &r, const gennmi_sequences_t &s, uint32_t width, uint32_t size)
{
    if(const int rc = checkRows(what, which, r, s, width, size)) { return rc; }
    const bool overlap = s.count > 1 && (s.offsets ? s.rows : s.length) && (s.offsets ? r.rowStride < width : r.sequenceStride < width);
    return overlap ? gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + ": " + which + ": sequences overlap") : GENNMI_OK;
}

// What a call reads or writes, in bytes: `outer` times `inner` runs of `width`, the larger of the strides outside
struct Region
{
    const char *name;
    int64_t begin, end;             // of all of it; nothing: both 0
    int64_t width, inner, innerStride, outer, outerStride;
};
inline Region regionOf(const char *name, const void *data, uint64_t width, uint64_t inner = 1, uint64_t innerStride = 0, uint64_t outer = 1, uint64_t outerStride = 0)
{
    if(innerStride > outerStride) { std::swap(inner, outer); std::swap(innerStride, outerStride); }
    if(innerStride == 0) { inner = std::min<uint64_t>(inner, 1); }
    if(outerStride == 0) { outer = std::min<uint64_t>(outer, 1); }
    const unsigned __int128 bytes = (unsigned __int128)(inner - 1) * innerStride + (unsigned __int128)(outer - 1) * outerStride + width;
    // (what no address space holds is none of this check's business)
    if(!data || !width || !inner || !outer || bytes > (1ull << 60)) { return Region{name, 0, 0, 0, 0, 0, 0, 0}; }
    return Region{name, (int64_t)(uintptr_t)data, (int64_t)(uintptr_t)data + (int64_t)bytes, (int64_t)width, (int64_t)inner, (int64_t)innerStride, (int64_t)outer, (int64_t)outerStride};
}
inline Region regionOf(const char *name, const gennmi_rows_t &r, const gennmi_sequences_t &s, uint64_t width, uint32_t size)
{
    if(s.offsets) { return regionOf(name, r.data, width * size, s.rows, r.rowStride * size); }
    return regionOf(name, r.data, width * size, s.length, r.rowStride * size, s.count, r.sequenceStride * size);
}
inline int64_t floorOf(int64_t a, int64_t by) { return a / by - (a % by < 0); }
// Whether a run of r's lies in part in low .. high - 1
inline bool meets(const Region &r, int64_t low, int64_t high)
{
    const int64_t run = (r.inner - 1) * r.innerStride + r.width;
    low -= r.begin;
    high -= r.begin;
    const int64_t first = r.outerStride ? std::max<int64_t>(0, floorOf(low - run, r.outerStride) + 1) : 0;
    const int64_t last = r.outerStride ? std::min(r.outer - 1, floorOf(high - 1, r.outerStride)) : 0;
    for(int64_t o = first; o <= last; o++) {
        const int64_t from = low - o * r.outerStride, to = high - o * r.outerStride;
        const int64_t i = r.innerStride ? std::max<int64_t>(0, floorOf(from - r.width, r.innerStride) + 1) : 0;
        if(i < r.inner && i * r.innerStride < to && i * r.innerStride + r.width > from) { return true; }
    }
    return false;
}
// The places of r's runs, seen from each other
inline Region differences(const Region &r, int64_t outerFrom, int64_t outerTo)
{
    Region d = r;
    d.begin = outerFrom * r.outerStride - (r.inner - 1) * r.innerStride;
    d.inner = 2 * r.inner - 1;
    d.outer = outerTo - outerFrom + 1;
    return d;
}
inline bool overlap(const Region &a, const Region &b)
{
    if(a.begin >= b.end || b.begin >= a.end) { return false; }
    if(a.inner == b.inner && a.outer == b.outer && a.innerStride == b.innerStride && a.outerStride == b.outerStride) {
        const Region d = differences(b, 1 - b.outer, b.outer - 1);
        return meets(d, a.begin - b.begin, a.begin - b.begin + a.width);
    }
    // (sequences equally far apart, in which the rows of one array lie behind those of the other)
    const auto sequencesOf = [](Region r) { r.width += (r.inner - 1) * r.innerStride; r.inner = 1; r.innerStride = 0; return r; };
    if(a.inner * b.inner > 1 && a.outer == b.outer && a.outerStride == b.outerStride && !overlap(sequencesOf(a), sequencesOf(b))) { return false; }
    // (one array's rows between another's that are not as far apart: looked at one by one)
    const Region &few = a.inner * a.outer <= b.inner * b.outer ? a : b, &many = &few == &a ? b : a;
    for(int64_t o = 0; o < few.outer; o++) {
        for(int64_t i = 0; i < few.inner; i++) {
            const int64_t at = few.begin + o * few.outerStride + i * few.innerStride;
            if(meets(many, at, at + few.width)) { return true; }
        }
    }
    return false;
}
// Runs of one array that overlap each other
inline bool overlapsItself(const Region &r)
{
    if(r.inner > 1 && r.innerStride < r.width) { return true; }
    return r.outer > 1 && meets(differences(r, 1, r.outer - 1), 0, r.width);
}
// Work-groups do not wait for one another: what a call writes is nothing else that it reads or writes.  `last`: written when everything has been read.
inline int checkApart(const char *what, std::initializer_list<Region> written, std::initializer_list<Region> last, std::initializer_list<Region> read)
{
    const auto refuse = [&](const Region &a, const char *why, const char *other) { return gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + ": " + a.name + why + other); };
    for(const Region *w = written.begin(); w != written.end(); w++) {
        if(overlapsItself(*w)) { return refuse(*w, ": sequences overlap", ""); }
        for(const Region *x = w + 1; x != written.end(); x++) { if(overlap(*w, *x)) { return refuse(*w, " overlaps ", x->name); } }
        for(const Region &x : read) { if(overlap(*w, x)) { return refuse(*w, " overlaps ", x.name); } }
    }
    for(const Region *l = last.begin(); l != last.end(); l++) {
        for(const Region *x = l + 1; x != last.end(); x++) { if(overlap(*l, *x)) { return refuse(*l, " overlaps ", x->name); } }
        for(const Region &x : written) { if(overlap(*l, x)) { return refuse(*l, " overlaps ", x.name); } }
    }
    return GENNMI_OK;
}
inline void noteRows(const gennmi_rows_t &r, const gennmi_sequences_t &s, uint32_t width, uint32_t size)
{
    const uint64_t rows = s.offsets ? s.rows : s.length;
    if(!r.data || !rows || !s.count) { return; }
    const uint64_t last = (rows - 1) * r.rowStride + (s.offsets ? 0 : (s.count - 1) * r.sequenceStride);
    gennmi_detail::noteDeviceWrite(r.data, (last + width) * size);
}
inline uint64_t statesOf(const gennmi_sequences_t &s) { return s.slots ? s.numSlots : s.count; }

inline Sequences sequencesOf(const gennmi_sequences_t &s, uint32_t chunk)
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
inline uint64_t chunkNumbers(const gennmi_sequences_t &s, uint32_t chunk)
{
    if(!s.count) { return 0; }
    return s.offsets ? s.rows / chunk + s.count : (uint64_t)s.count * std::max(1u, (s.length + chunk - 1) / chunk);
}
inline uint64_t totalRows(const gennmi_sequences_t &s) { return s.offsets ? s.rows : (uint64_t)s.count * s.length; }
inline Region offsetsOf(const gennmi_sequences_t &s) { return regionOf("offsets", s.offsets, (s.count + 1ull) * 4); }
inline Region slotsOf(const gennmi_sequences_t &s) { return regionOf("slots", s.slots, s.count * 4ull); }
// An array that a call may write in place of the one it reads
inline Region unlessSame(const Region &r, const void *written) { return (uintptr_t)written == (uintptr_t)r.begin ? Region{r.name, 0, 0, 0, 0, 0, 0, 0} : r; }
// Kernels ask for more LDS than a launch has without being told
template<typename K> int withLds(const char *what, K kernel, size_t bytes)
{
    if(bytes <= 65536) { return GENNMI_OK; }
    const hipError_t e = hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    return e == hipSuccess ? (int)GENNMI_OK : gennmi_detail::fail(GENNMI_EHIP, std::string(what) + ": " + hipGetErrorString(e));
}
inline int checkWorkspace(const char *what, const void *workspace, size_t have, size_t need)
{
    if(need && (!workspace || have < need)) { return gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + ": workspace is missing or too small"); }
    return (uintptr_t)workspace % 16 ? gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + ": workspace is not 16-byte aligned") : GENNMI_OK;
}
inline int tooMany(const char *what) { return gennmi_detail::fail(GENNMI_EINVAL, std::string(what) + ": more rows than one launch covers"); }

// Sums over chunks, sums[number][n][channel], in 64 bits: there may be thousands, of either sign.  Row n of the sums goes to out[channel][n] for n < width,
// behind those to more[0][channel] and more[1][channel].  The 16 wavefronts of a work-group have 64 channels and a sixteenth of the numbers each;
// what they found is added up in the order of the numbers.
struct ChunkSums { const float *sums; float *out, *more[2]; uint32_t numbers, channels, width, rows; };
inline uint64_t chunkSumBlocks(uint32_t rows, uint32_t channels) { return (uint64_t)rows * ((channels + 63) / 64); }
int launchChunkSum(const char *what, const ChunkSums &a, hipStream_t stream);       // (defined beside the scan)
}

#endif

// Part of libgenn_mi355x.so: included by genn_mi355x_sequence.hip only.
//
// Selective state space scan.  A channel d drives N leaky units:
//   h[t][n] = exp(dt A[n]) h[t - 1][n] + dt u B[t][n],   y = sum_n C[t][n] h[t][n] + D u,   out = y z sigmoid(z)
// B and C are those of the channel's group.
//
// Layout: a lane is a channel, with NP of its states in registers, and walks rows one after another; a wavefront has 64 neighbouring
// channels, so every access to a row of channels is one run of memory, sums over the states stay in a lane, and B and C are the same for all
// lanes (staged in LDS in fp32, read as broadcasts).  More than NP states are the work of several wavefronts of a work-group, whose sums
// over the states meet in LDS.  Where channels and sequences are too few to fill the chip, sequences are cut into chunks: one kernel
// finds what each chunk adds to a state that comes in as zero (and the sum of dt, which says what becomes of one that does not), a second
// walks over the chunks, and the third does the work from the right state.
//
// Bound by vector instructions, not by memory: a state takes a row a product and an exponential (two slots of a SIMD's issue) for its decay, a product and a sum
// for what comes in, a sum for y, 6 slots, of which the first kernel of a split scan needs 5 as well.  At 39.3 T lane-slots a second 4096 rows x 2048 channels x 16
// states are 38 us of these alone, their 68 MB 12 us.  They take 77 us in bf16: 36 the first kernel, 8 the second, 42 the third, with the vector
// units busy for four fifths of the time (softplus, gate and conversions are a fifth of their instructions).  What there is to gain by matrix instructions is
// nothing: every state of every channel has decays of its own.
#ifndef GENN_MI355X_SCAN_KERNELS_H
#define GENN_MI355X_SCAN_KERNELS_H

namespace
{
constexpr float LOG2E = 1.44269504f, LN2 = 0.693147181f;

struct ScanArgs
{
    Sequences sequences;
    gennmi_rows_t u, delta, z, out, B, C;
    const float *A, *D, *deltaBias;
    const float *initialState; float *finalState;
    uint32_t channels, states, groups, softplus;
    uint32_t groupChannels, groupTiles, tiles;      // channels of a group; tiles of 64 of them; of all groups
    uint32_t numbers, slabs;                        // chunk numbers; wavefronts that share the states of a channel
    float *chunkState;                              // [numbers][states][channels]: what a chunk adds, then the state it starts from; NULL: one chunk a sequence
    float *chunkTime;                               // [numbers][channels]: sum of dt
};
struct ScanGradientArgs
{
    gennmi_rows_t out, u, delta, z, B, C;
    const float *finalState; float *initialState;
    float *chunkGradient;           // [numbers][states][channels]: what a chunk's rows give the state before it, then the gradient of the state behind it
    float *sums;                    // [numbers][states + 2][channels]: sums over a chunk, for A, D and the bias
    float *sumBC;                   // [tiles][rows][2][states]: sums over a tile's channels, of B's gradient and of C's
    uint64_t rows;                  // rows of sumBC
};

__device__ inline float exp2Of(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ inline float logistic(float x) { return __builtin_amdgcn_rcpf(1.0f + exp2Of(x * -LOG2E)); }
// log(1 + exp(x)) = max(x, 0) + log(1 + e), e = exp(-|x|).  Where e is small, f = 1 + e as rounded has lost most of it: log(1 + e) = log(f) + log((1 + e) / f),
// and the second is e - (f - 1) to the last bits (that difference is exact, below 2^-24, and f is at most 2).
__device__ inline float softplusOf(float x)
{
    const float e = exp2Of(fabsf(x) * -LOG2E), f = 1.0f + e;
    return fmaxf(x, 0.0f) + __builtin_fmaf(__builtin_amdgcn_logf(f), LN2, e - (f - 1.0f));
}

// Where a work-group is: a chunk and a tile of channels
struct ScanPlace
{
    Place place;
    uint32_t tile, group, channel, first, rows;     // first row of the chunk in its sequence, and how many
    uint32_t firstState, numStates;                 // of the wavefront
    bool valid, active;                             // there is a chunk; the lane has a channel (else it reads the last one's and writes nothing)
};
template<int NP> __device__ inline ScanPlace scanPlace(const ScanArgs &a, uint32_t &number)
{
    ScanPlace s;
    number = blockIdx.x / a.tiles;
    s.tile = blockIdx.x - number * a.tiles;
    s.group = s.tile / a.groupTiles;
    const uint32_t within = (s.tile - s.group * a.groupTiles) * 64 + (threadIdx.x & 63);
    s.active = within < a.groupChannels;
    s.channel = s.group * a.groupChannels + min(within, a.groupChannels - 1);
    const uint32_t slab = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    s.firstState = slab * NP;
    s.numStates = min((uint32_t)NP, a.states - s.firstState);
    s.valid = locate(a.sequences, number, s.place);
    s.first = s.place.index * a.sequences.chunk;
    s.rows = s.valid && s.place.length > s.first ? min(a.sequences.chunk, s.place.length - s.first) : 0;
    return s;
}

// B and C of R rows, of a wavefront's states, in LDS as [row][B, C][NP], zero where there is no row or state.  A lane fetches
// R * 2 * NP / 64 of the values, of B or of C and of one state all of them, a block of rows before they are needed.
template<typename T, int NP, int R> struct StagedBC
{
    static constexpr int EACH = R * 2 * NP / 64, LANES = 2 * NP;        // LANES: that a row takes
    const T *at;
    uint32_t stride;
    bool here;
    T raw[EACH];
    __device__ inline StagedBC(const T *B, const T *C, const ScanArgs &a, uint32_t numStates)
    {
        const uint32_t lane = threadIdx.x & 63, n = lane % NP;
        const bool isC = (lane / NP) & 1;
        at = (isC ? C : B) + min(n, numStates - 1);
        stride = (uint32_t)(isC ? a.C.rowStride : a.B.rowStride);
        here = n < numStates;
    }
    __device__ static inline uint32_t rowOf(int q) { return q * (64 / LANES) + (threadIdx.x & 63) / LANES; }
    __device__ inline void fetch(uint32_t row, uint32_t end)
    {
        #pragma unroll
        for(int q = 0; q < EACH; q++) { raw[q] = at[(uint64_t)min(row + rowOf(q), end - 1) * stride]; }
    }
    __device__ inline void store(float *lds, uint32_t row, uint32_t end) const
    {
        #pragma unroll
        for(int q = 0; q < EACH; q++) { lds[q * 64 + (threadIdx.x & 63)] = here && row + rowOf(q) < end ? widen(raw[q]) : 0.0f; }
    }
};
// What one wavefront wrote to LDS is read by its other lanes: LDS accesses of a wavefront are done in order, only the compiler has to keep it
__device__ inline void waveFence() { __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront"); __builtin_amdgcn_wave_barrier(); }

// An element of a row.  The row's address is the same for all lanes, the element's place in it (in bytes) fits 32 bits: loads and stores take the two so,
// without 64-bit arithmetic in every lane, if the compiler does not get to see how the row's address is made.
template<typename T> __device__ inline uint64_t rowAddress(T *rows, uint32_t t, uint64_t stride)
{
    uint64_t address = (uint64_t)(rows + (uint64_t)t * stride);
    asm("" : "+s"(address));
    return address;
}
template<typename T> __device__ inline T loadAt(const T *rows, uint32_t t, uint64_t stride, uint32_t place)
{
    return *(const __attribute__((address_space(1))) T*)((const __attribute__((address_space(1))) char*)rowAddress(rows, t, stride) + place);
}
template<typename T> __device__ inline void storeAt(T *rows, uint32_t t, uint64_t stride, uint32_t place, T value)
{
    *(__attribute__((address_space(1))) T*)((__attribute__((address_space(1))) char*)rowAddress(rows, t, stride) + place) = value;
}
// Reads of LDS behind this point wait for the four values.  (Left alone, the compiler gathers the reads of many rows in front of all arithmetic, puts off
// sums that nothing waits for until behind it, and spills hundreds of registers.)
__device__ inline void readAfter(float &a, float &b, float &c, float &d) { asm volatile("" : "+v"(a), "+v"(b), "+v"(c), "+v"(d) : : "memory"); }

__device__ inline void readAfter(float &a, float &b) { asm volatile("" : "+v"(a), "+v"(b) : : "memory"); }
// ... COUNT values from the one at `first` on
template<int COUNT, int N> __device__ inline void readAfter(float (&x)[N], int first = 0)
{
    #pragma unroll
    for(int n = 0; n < COUNT; n += 2) { readAfter(x[first + n], x[first + n + 1]); }
}

// A lane's states of its channel, which are neighbours in memory: four an access where they lie so (a quarter of the trips through the cache, whose
// lines hold the states of two lanes or so), else one; a wavefront with fewer than NP reads its last one again instead
template<int NP> __device__ inline void loadNeighbours(const float *from, uint32_t count, bool fours, float (&x)[NP])
{
    if(fours) {
        #pragma unroll
        for(int n = 0; n < NP; n += 4) {
            const Pack<float, 4> p = *(const Pack<float, 4>*)(from + n);
            #pragma unroll
            for(int k = 0; k < 4; k++) { x[n + k] = p.v[k]; }
        }
    }
    else {
        #pragma unroll
        for(int n = 0; n < NP; n++) { x[n] = from[min((uint32_t)n, count - 1)]; }
    }
}
template<int NP> __device__ inline bool inFours(const ScanArgs &a, const ScanPlace &s, const float *states)
{
    return s.numStates == NP && a.states % 4 == 0 && (uint64_t)states % 16 == 0;
}
// What exp2 takes of A.  An infinite one (a unit that forgets everything) as the largest number: no time at all, which rows behind the end and sequences without
// rows take, is not to change a state, and any other is the same.
__device__ inline float exponentOf(float A)
{
    const float x = A * LOG2E;
    return fabsf(x) == __builtin_inff() ? __builtin_copysignf(3.402823466e38f, x) : x;
}
template<int NP> __device__ inline void loadA(const ScanArgs &a, const ScanPlace &s, float (&A)[NP])
{
    loadNeighbours<NP>(a.A + (uint64_t)s.channel * a.states + s.firstState, s.numStates, inFours<NP>(a, s, a.A), A);
    #pragma unroll
    for(int n = 0; n < NP; n++) { A[n] = n < (int)s.numStates ? exponentOf(A[n]) : 0.0f; }
}
template<int NP> __device__ inline void loadState(const ScanArgs &a, const ScanPlace &s, const float *state, uint64_t which, float (&h)[NP])
{
    #pragma unroll
    for(int n = 0; n < NP; n++) { h[n] = 0.0f; }
    if(state) { loadNeighbours<NP>(state + (which * a.channels + s.channel) * a.states + s.firstState, s.numStates, inFours<NP>(a, s, state), h); }
}
template<int NP> __device__ inline void storeState(const ScanArgs &a, const ScanPlace &s, float *state, uint64_t which, const float (&h)[NP])
{
    if(!state || !s.active) { return; }
    float *const to = state + (which * a.channels + s.channel) * a.states + s.firstState;
    if(inFours<NP>(a, s, state)) {
        #pragma unroll
        for(int n = 0; n < NP; n += 4) { *(Pack<float, 4>*)(to + n) = Pack<float, 4>{{h[n], h[n + 1], h[n + 2], h[n + 3]}}; }
    }
    else {
        #pragma unroll
        for(int n = 0; n < NP; n++) { if(n < (int)s.numStates) { to[n] = h[n]; } }
    }
}
template<int NP> __device__ inline void loadChunk(const ScanArgs &a, const ScanPlace &s, const float *chunks, uint32_t number, float (&h)[NP])
{
    const float *from = chunks + ((uint64_t)number * a.states + s.firstState) * a.channels;
    #pragma unroll
    for(int n = 0; n < NP; n++) { h[n] = (from + (uint64_t)min((uint32_t)n, s.numStates - 1) * a.channels)[s.channel]; }
}
template<int NP> __device__ inline void storeChunk(const ScanArgs &a, const ScanPlace &s, float *chunks, uint32_t number, const float (&h)[NP])
{
    if(!s.active) { return; }
    float *to = chunks + ((uint64_t)number * a.states + s.firstState) * a.channels;
    #pragma unroll
    for(int n = 0; n < NP; n++) {
        if(n < (int)s.numStates) { (to + (uint64_t)n * a.channels)[s.channel] = h[n]; }
    }
}

// One row of a channel's array, R of them, fetched a block of rows before they are needed (rows behind the last one are that one again).  Strides of rows fit 32 bits: two
// scalar products for an address instead of four (a scan of 4096 rows x 2048 channels 81.5 -> 79.3 us; the same in the walk back of the gradients: 870 -> 907, other registers)
template<typename T, int R> struct StagedRows
{
    T raw[R];
    __device__ inline void fetch(const T *rows, uint32_t stride, uint32_t place, uint32_t row, uint32_t end)
    {
        #pragma unroll
        for(int r = 0; r < R; r++) { raw[r] = loadAt(rows, min(row + r, end - 1), stride, place); }
    }
};
// dt and dt u of a block of rows; zero behind the end, which leaves every state as it is
template<typename T, int R>
__device__ inline void times(const ScanArgs &a, const StagedRows<T, R> &delta, const StagedRows<T, R> &u, float bias, uint32_t there, float (&dt)[R], float (&w)[R])
{
    #pragma unroll
    for(int r = 0; r < R; r++) { dt[r] = widen(delta.raw[r]) + bias; }
    if(a.softplus) {
        #pragma unroll
        for(int r = 0; r < R; r++) { dt[r] = softplusOf(dt[r]); }
    }
    #pragma unroll
    for(int r = 0; r < R; r++) { w[r] = dt[r] * widen(u.raw[r]); }
    if(there < R) {
        #pragma unroll
        for(int r = 0; r < R; r++) { if(r >= (int)there) { dt[r] = w[r] = 0.0f; } }
    }
}
// The gate, z sigmoid(z)
template<typename T, int R> __device__ inline void gates(const StagedRows<T, R> &z, float (&gate)[R])
{
    #pragma unroll
    for(int r = 0; r < R; r++) { const float x = widen(z.raw[r]); gate[r] = x * logistic(x); }
}

// Whether a lane has an infinite value
template<int R> __device__ inline bool anyInfinite(const float (&w)[R])
{
    float most = 0.0f;
    #pragma unroll
    for(int r = 0; r < R; r++) { most = fmaxf(most, fabsf(w[r])); }
    return __any(most == __builtin_inff());
}

// First kernel of a split scan: every chunk from a state of zero.  With GRADIENT also sum_t (prod_{s <= t} exp(dt_s A)) C_t g_t, what the chunk's rows
// give the gradient of the state before it.
template<typename T, int NP, bool GRADIENT, bool SLABS>
__global__ __launch_bounds__(SLABS ? 512 : 64)
void scanChunkKernel(ScanArgs a, ScanGradientArgs g)
{
    constexpr int R = 8;
    __shared__ float staged[SLABS ? 8 : 1][R * 2 * NP];
    uint32_t number;
    const ScanPlace s = scanPlace<NP>(a, number);
    if(!s.valid) { return; }
    float *const bc = staged[__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)];
    const uint32_t channel = s.channel, place = channel * (uint32_t)sizeof(T);
    const T *u = rowsOf<const T>(a.u, a.sequences, s.place), *delta = rowsOf<const T>(a.delta, a.sequences, s.place);
    const uint32_t bcAt = s.group * a.states + s.firstState;
    const T *B = rowsOf<const T>(a.B, a.sequences, s.place) + bcAt, *C = rowsOf<const T>(a.C, a.sequences, s.place) + bcAt;
    const T *dout = GRADIENT ? rowsOf<const T>(g.out, a.sequences, s.place) : nullptr;
    const T *z = GRADIENT && a.z.data ? rowsOf<const T>(a.z, a.sequences, s.place) : nullptr;
    const float bias = a.deltaBias ? a.deltaBias[channel] : 0.0f;
    float A[NP], h[NP], G[NP], P[NP], time = 0.0f;
    loadA<NP>(a, s, A);
    #pragma unroll
    for(int n = 0; n < NP; n++) { h[n] = G[n] = 0.0f; P[n] = 1.0f; }
    const uint32_t end = s.first + s.rows;
    StagedBC<T, NP, R> stage(B, C, a, s.numStates);
    StagedRows<T, R> rawU, rawDelta, rawOut, rawZ;
    const auto fetch = [&](uint32_t row) {
        stage.fetch(row, end);
        rawU.fetch(u, a.u.rowStride, place, row, end);
        rawDelta.fetch(delta, a.delta.rowStride, place, row, end);
        if(GRADIENT) { rawOut.fetch(dout, g.out.rowStride, place, row, end); }
        if(GRADIENT && z) { rawZ.fetch(z, a.z.rowStride, place, row, end); }
    };
    if(s.rows) { fetch(s.first); }
    for(uint32_t row = s.first; row < end; row += R) {
        float dt[R], w[R], gy[R];
        times<T, R>(a, rawDelta, rawU, bias, end - row, dt, w);
        if(GRADIENT) {
            #pragma unroll
            for(int r = 0; r < R; r++) { gy[r] = r < (int)(end - row) ? widen(rawOut.raw[r]) : 0.0f; }
            if(z) {
                float gate[R];
                gates<T, R>(rawZ, gate);
                #pragma unroll
                for(int r = 0; r < R; r++) { gy[r] *= gate[r]; }
            }
        }
        waveFence();
        stage.store(bc, row, end);
        waveFence();
        fetch(row + R);         // (behind the last block: its last row, for nothing)
        float nextB[NP], nextC[NP];
        #pragma unroll
        for(int n = 0; n < NP; n++) { nextB[n] = bc[n]; if(GRADIENT) { nextC[n] = bc[NP + n]; } }
        #pragma unroll
        for(int r = 0; r < R; r++) {
            float Bn[NP], Cn[NP];
            #pragma unroll
            for(int n = 0; n < NP; n++) { Bn[n] = nextB[n]; Cn[n] = nextC[n]; }
            if(r + 1 < R) {
                // (a row's inputs are read while the row before is worked on, and no sooner)
                readAfter<NP>(h);
                if(GRADIENT) { readAfter<NP>(G); readAfter<NP>(P); }
                #pragma unroll
                for(int n = 0; n < NP; n++) { nextB[n] = bc[(r + 1) * 2 * NP + n]; if(GRADIENT) { nextC[n] = bc[((r + 1) * 2 + 1) * NP + n]; } }
            }
            time += dt[r];
            #pragma unroll
            for(int n = 0; n < NP; n++) {
                const float decay = exp2Of(dt[r] * A[n]);
                h[n] = __builtin_fmaf(decay, h[n], w[r] * Bn[n]);
                if(GRADIENT) {
                    P[n] *= decay;
                    G[n] = __builtin_fmaf(P[n], gy[r] * Cn[n], G[n]);
                }
            }
        }
    }
    storeChunk<NP>(a, s, a.chunkState, number, h);
    if(s.firstState == 0 && s.active) { a.chunkTime[(uint64_t)number * a.channels + channel] = time; }
    if(GRADIENT) { storeChunk<NP>(a, s, g.chunkGradient, number, G); }
}

// One walk over the chunks of a state, forwards or backwards: what a chunk adds is replaced by what there was before it.  A trip to memory is as long as
// dozens of chunks' arithmetic, so what AHEAD chunks add is fetched before the AHEAD before those are worked on.
template<bool BACKWARDS> __device__ inline float walkChunks(float *state, uint64_t stride, const float *time, uint32_t channels, uint32_t chunks, float A, float h)
{
    constexpr uint32_t AHEAD = 8;
    const auto chunk = [&](uint32_t k) { return BACKWARDS ? chunks - 1 - min(k, chunks - 1) : min(k, chunks - 1); };
    float adds[AHEAD], times[AHEAD];
    #pragma unroll
    for(uint32_t k = 0; k < AHEAD; k++) { adds[k] = state[chunk(k) * stride]; times[k] = time[(uint64_t)chunk(k) * channels]; }
    for(uint32_t first = 0; first < chunks; first += AHEAD) {
        float nextAdds[AHEAD], nextTimes[AHEAD];
        #pragma unroll
        for(uint32_t k = 0; k < AHEAD; k++) { nextAdds[k] = state[chunk(first + AHEAD + k) * stride]; nextTimes[k] = time[(uint64_t)chunk(first + AHEAD + k) * channels]; }
        #pragma unroll
        for(uint32_t k = 0; k < AHEAD; k++) {
            if(first + k < chunks) {
                state[chunk(first + k) * stride] = h;
                // (a chunk's decay may be infinite, where A is positive, or round to zero: of nothing, nothing is left all the same, and of what is infinite all)
                constexpr int ZERO_OR_INFINITE = 0x20 | 0x40 | 0x4 | 0x200;
                const float sum = h + adds[k], next = __builtin_fmaf(exp2Of(times[k] * A), h, adds[k]);
                h = __builtin_amdgcn_classf(h, ZERO_OR_INFINITE) ? sum : next;
            }
            adds[k] = nextAdds[k];
            times[k] = nextTimes[k];
        }
    }
    return h;
}
// Second kernel: a lane has one state of one channel of one sequence and walks over the chunks, leaving in each one's place the state it starts from,
// and (GRADIENT) back again, leaving the gradient of the state behind each.
template<bool GRADIENT>
__global__ __launch_bounds__(64)
void scanJoinKernel(ScanArgs a, ScanGradientArgs g)
{
    const uint32_t parts = (a.channels + 63) / 64;
    const uint32_t part = blockIdx.x % parts, rest = blockIdx.x / parts;
    const uint32_t n = rest % a.states, sequence = rest / a.states;
    const uint32_t channel = part * 64 + threadIdx.x;
    Place p;
    if(!describe(a.sequences, sequence, p) || channel >= a.channels) { return; }
    const uint64_t chunk0 = firstChunk(a.sequences, sequence), stride = (uint64_t)a.states * a.channels;
    const uint32_t chunks = max(1u, (uint32_t)(((uint64_t)p.length + a.sequences.chunk - 1) / a.sequences.chunk));
    const float A = exponentOf(a.A[(uint64_t)channel * a.states + n]);
    const uint64_t at = ((uint64_t)p.state * a.channels + channel) * a.states + n, first = (chunk0 * a.states + n) * a.channels + channel;
    const float *time = a.chunkTime + chunk0 * a.channels + channel;
    const float h = walkChunks<false>(a.chunkState + first, stride, time, a.channels, chunks, A, a.initialState ? a.initialState[at] : 0.0f);
    if(!GRADIENT) { if(a.finalState) { a.finalState[at] = h; } }
    else {
        const float r = walkChunks<true>(g.chunkGradient + first, stride, time, a.channels, chunks, A, g.finalState ? g.finalState[at] : 0.0f);
        if(g.initialState) { g.initialState[at] = r; }
    }
}

// Third kernel, or the only one: the outputs.
template<typename T, int NP, bool SLABS>
__global__ __launch_bounds__(SLABS ? 512 : 64)
void scanKernel(ScanArgs a)
{
    constexpr int R = 8;
    __shared__ float staged[SLABS ? 8 : 1][R * 2 * NP];
    __shared__ float sums[SLABS ? 2 : 1][SLABS ? 8 : 1][SLABS ? R : 1][64];     // [alternating][slab][row][lane]
    uint32_t number;
    const ScanPlace s = scanPlace<NP>(a, number);
    if(!s.valid) { return; }
    const uint32_t slab = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, channel = s.channel, place = channel * (uint32_t)sizeof(T);
    float *const bc = staged[slab];
    const T *u = rowsOf<const T>(a.u, a.sequences, s.place), *delta = rowsOf<const T>(a.delta, a.sequences, s.place);
    const T *z = a.z.data ? rowsOf<const T>(a.z, a.sequences, s.place) : nullptr;
    T *out = rowsOf<T>(a.out, a.sequences, s.place);
    const uint32_t bcAt = s.group * a.states + s.firstState;
    const T *B = rowsOf<const T>(a.B, a.sequences, s.place) + bcAt, *C = rowsOf<const T>(a.C, a.sequences, s.place) + bcAt;
    const float bias = a.deltaBias ? a.deltaBias[channel] : 0.0f, skip = a.D ? a.D[channel] : 0.0f;
    float A[NP], h[NP];
    loadA<NP>(a, s, A);
    if(a.chunkState) { loadChunk<NP>(a, s, a.chunkState, number, h); } else { loadState<NP>(a, s, a.initialState, s.place.state, h); }
    // States that are not there have decay 1 and B = C = 0, and are 0 for as long as what they are multiplied with is finite
    #pragma unroll
    for(int n = 0; n < NP; n++) { h[n] = n < (int)s.numStates ? h[n] : 0.0f; }
    const uint32_t end = s.first + s.rows;
    StagedBC<T, NP, R> stage(B, C, a, s.numStates);
    StagedRows<T, R> rawU, rawDelta, rawZ;
    const auto fetch = [&](uint32_t row) {
        stage.fetch(row, end);
        rawU.fetch(u, a.u.rowStride, place, row, end);
        rawDelta.fetch(delta, a.delta.rowStride, place, row, end);
        if(z) { rawZ.fetch(z, a.z.rowStride, place, row, end); }
    };
    if(s.rows) { fetch(s.first); }
    uint32_t turn = 0;
    for(uint32_t row = s.first; row < end; row += R, turn ^= 1) {
        float dt[R], w[R], y[R], gate[R], direct[R];
        times<T, R>(a, rawDelta, rawU, bias, end - row, dt, w);
        #pragma unroll
        for(int r = 0; r < R; r++) { direct[r] = a.D ? skip * widen(rawU.raw[r]) : 0.0f; gate[r] = 1.0f; }
        if(z) { gates<T, R>(rawZ, gate); }
        waveFence();
        stage.store(bc, row, end);
        waveFence();
        fetch(row + R);         // (behind the last block: its last row, for nothing)
        if(s.numStates < NP && anyInfinite<R>(w)) {
            // (rare: the states that are there, one row after another)
            #pragma unroll
            for(int r = 0; r < R; r++) { y[r] = 0.0f; }
            #pragma nounroll
            for(int r = 0; r < R; r++) {
                float time = 0.0f, in = 0.0f, y0 = 0.0f, y1 = 0.0f;
                #pragma unroll
                for(int k = 0; k < R; k++) { time = k == r ? dt[k] : time; in = k == r ? w[k] : in; y0 = k == r && !SLABS ? direct[k] : y0; }
                #pragma unroll
                for(int n = 0; n < NP; n++) {
                    if(n >= (int)s.numStates) { break; }
                    h[n] = __builtin_fmaf(exp2Of(time * A[n]), h[n], in * bc[r * 2 * NP + n]);
                    const float c = bc[(r * 2 + 1) * NP + n];
                    if(n & 1) { y1 = __builtin_fmaf(h[n], c, y1); } else { y0 = __builtin_fmaf(h[n], c, y0); }
                }
                #pragma unroll
                for(int k = 0; k < R; k++) { y[k] = k == r ? y0 + y1 : y[k]; }
            }
        }
        else {
            float nextB[NP], nextC[NP];
            #pragma unroll
            for(int n = 0; n < NP; n++) { nextB[n] = bc[n]; nextC[n] = bc[NP + n]; }
            #pragma unroll
            for(int r = 0; r < R; r++) {
                float Bn[NP], Cn[NP];
                #pragma unroll
                for(int n = 0; n < NP; n++) { Bn[n] = nextB[n]; Cn[n] = nextC[n]; }
                if(r + 1 < R) {
                    // (a row's inputs are read while the row before is worked on, and no sooner)
                    readAfter<NP>(h);
                    if(r) { readAfter(y[r - 1], h[0], h[1], h[2]); }
                    #pragma unroll
                    for(int n = 0; n < NP; n++) { nextB[n] = bc[(r + 1) * 2 * NP + n]; nextC[n] = bc[((r + 1) * 2 + 1) * NP + n]; }
                }
                float y0 = SLABS ? 0.0f : direct[r], y1 = 0.0f;
                #pragma unroll
                for(int n = 0; n < NP; n++) {
                    h[n] = __builtin_fmaf(exp2Of(dt[r] * A[n]), h[n], w[r] * Bn[n]);
                    if(n & 1) { y1 = __builtin_fmaf(h[n], Cn[n], y1); } else { y0 = __builtin_fmaf(h[n], Cn[n], y0); }
                }
                y[r] = y0 + y1;
            }
        }
        if(SLABS) {
            #pragma unroll
            for(int r = 0; r < R; r++) { sums[turn][slab][r][lane] = y[r]; }
            __syncthreads();        // (the other half of `sums` is written next, so one barrier a block of rows does)
            #pragma unroll
            for(int r = 0; r < R; r++) {
                if(r % a.slabs == slab) {
                    y[r] = direct[r];
                    for(uint32_t k = 0; k < a.slabs; k++) { y[r] += sums[turn][k][r][lane]; }
                }
            }
        }
        if(s.active) {
            #pragma unroll
            for(int r = 0; r < R; r++) {
                if(row + r < end && (!SLABS || r % a.slabs == slab)) { storeAt(out, row + r, (uint32_t)a.out.rowStride, place, narrow<T>(y[r] * gate[r])); }
            }
        }
    }
    if(!a.chunkState) { storeState<NP>(a, s, a.finalState, s.place.state, h); }
}

// One row a sequence (a token): the states of a sequence's channel are neighbours in memory, and reading and writing them is all there is to it.
// LANES lanes have four each; what they give the output is added up between them.  256 sequences of 4096 channels of 16 states take 31 us (4.6 TB/s), with
// two or four sequences a lane (which share A) 32 and 38.
template<typename T, int LANES, bool QUADS>
__global__ __launch_bounds__(256)
void scanTokenKernel(ScanArgs a)
{
    uint32_t sequence, channel;
    divideItem(a.channels * LANES, sequence, channel);
    const uint32_t part = threadIdx.x % LANES, n0 = part * 4;
    channel /= LANES;
    if(sequence >= a.sequences.count) { return; }
    Place p;
    if(!describe(a.sequences, sequence, p)) { return; }
    const uint32_t bcAt = (channel / a.groupChannels) * a.states + n0;
    const bool here = n0 < a.states;
    const auto load4 = [&](const auto *from, float (&to)[4]) {
        typedef std::remove_cv_t<std::remove_reference_t<decltype(*from)>> E;
        #pragma unroll
        for(int k = 0; k < 4; k++) { to[k] = 0.0f; }
        if(QUADS) {
            if(here) {
                const Pack<E, 4> q = *(const Pack<E, 4>*)from;
                #pragma unroll
                for(int k = 0; k < 4; k++) { to[k] = widen(q.v[k]); }
            }
        }
        else {
            #pragma unroll
            for(int k = 0; k < 4; k++) { if(n0 + k < a.states) { to[k] = widen(from[k]); } }
        }
    };
    const uint64_t at = ((uint64_t)p.state * a.channels + channel) * a.states + n0;
    float h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if(a.initialState) { load4(a.initialState + at, h); }
    if(p.length) {          // (a packed sequence may have none)
        float A[4], B[4], C[4], y = 0.0f;
        load4(rowsOf<const T>(a.B, a.sequences, p) + bcAt, B);
        load4(rowsOf<const T>(a.C, a.sequences, p) + bcAt, C);
        load4(a.A + (uint64_t)channel * a.states + n0, A);
        const float u = widen(rowsOf<const T>(a.u, a.sequences, p)[channel]), z = a.z.data ? widen(rowsOf<const T>(a.z, a.sequences, p)[channel]) : 0.0f;
        float time = widen(rowsOf<const T>(a.delta, a.sequences, p)[channel]) + (a.deltaBias ? a.deltaBias[channel] : 0.0f);
        if(a.softplus) { time = softplusOf(time); }
        float w = time * u;
        if(!here) { time = w = 0.0f; }          // (what is infinite, times nothing)
        #pragma unroll
        for(int k = 0; k < 4; k++) {
            if(QUADS || n0 + k < a.states) {
                h[k] = __builtin_fmaf(exp2Of(time * (A[k] * LOG2E)), h[k], w * B[k]);
                y = __builtin_fmaf(h[k], C[k], y);
            }
        }
        // (lanes behind the last state have added zeros)
        if constexpr(LANES > 1) { y += gennmi_lanes::partner<1>(y); }
        if constexpr(LANES > 2) { y += gennmi_lanes::partner<2>(y); }
        if constexpr(LANES > 4) { y += gennmi_lanes::partner<4>(y); }
        if constexpr(LANES > 8) { y += gennmi_lanes::partner<8>(y); }
        if constexpr(LANES > 16) { y += gennmi_lanes::partner<16>(y); }
        if(part == 0) {
            if(a.D) { y = __builtin_fmaf(a.D[channel], u, y); }
            if(a.z.data) { y *= z * logistic(z); }
            rowsOf<T>(a.out, a.sequences, p)[channel] = narrow<T>(y);
        }
    }
    if(a.finalState && here) {
        float *state = a.finalState + at;
        if(QUADS) { *(Pack<float, 4>*)state = Pack<float, 4>{{h[0], h[1], h[2], h[3]}}; }
        else {
            #pragma unroll
            for(int k = 0; k < 4; k++) { if(n0 + k < a.states) { state[k] = h[k]; } }
        }
    }
}

// Gradients of a chunk, from the state before it and the gradient of the state behind it.  The states in between are made again, a block of
// R rows at a time: first one walk forward that keeps the state before every block (LDS), then from the last block to the first one walk
// forward through a block that keeps its states in registers, and one back:
//   dh = C gy + (what comes from the row behind);  dC = gy h, dB = dh dt u (summed over channels);  q = sum dh B, x = dh exp(dt A) h', r = sum x A
//   du = dt q + D gy;  d(dt) = u q + r;  dA += x dt;  and exp(dt A) dh for the row before
// A block's walks take PART of the states at a time, so that R * PART of them, and as many decays, fit the registers of two wavefronts a SIMD.
//
// Bound by vector instructions: 420 a row and wavefront of 16 states, an eighth of them the sums over channels (all of them in registers: 444 and 690 us), and units
// busy for three quarters of the time (252 registers, so two wavefronts a SIMD; 20 KiB of LDS each, all that there is for eight).  8 sequences of 2048 rows x 2048 channels in bf16: this kernel 671 to 676 us, the first 206, the second 57 (memory, 4.8 TB/s), sums
// over tiles 23 and over chunks 16.  PART 4 spills (813 us), so do three wavefronts a SIMD (1240), without the ties of readAfter it was 9.4 ms.
template<typename T, int NP, int R, int BLOCKS, bool SLABS>
__global__ __launch_bounds__(SLABS ? 512 : 64) __attribute__((amdgpu_waves_per_eu(2, 2)))
void scanBackwardKernel(ScanArgs a, ScanGradientArgs g)
{
    constexpr int PART = 2, PARTS = NP / PART;
    constexpr int SPACE = BLOCKS * NP * 64 + R * 2 * NP * 2 + R * 64;        // floats of LDS a wavefront
    static_assert(PART == 2 && R == 8, "the lanes' shares of a part's sums are eight values a lane");
    extern __shared__ __attribute__((aligned(16))) float lds[];
    uint32_t number;
    const ScanPlace s = scanPlace<NP>(a, number);
    const uint32_t slab = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, channel = s.channel, place = channel * (uint32_t)sizeof(T);
    float *const kept = lds + (size_t)slab * SPACE;       // [block][part][lane][PART]: the states before a block
    float *const bc = kept + BLOCKS * NP * 64, *const rowSums = bc + R * 2 * NP;     // both [row][B, C][NP]
    float *const shares = rowSums + R * 2 * NP;             // [row][lane]: of a part's sums over the lanes, 16 lanes for each of B's two and C's two
    float *const sums = lds + (size_t)a.slabs * SPACE;      // SLABS: [slab][row][q, r, y][lane]
    const auto keep = [&](uint32_t b, const float (&h)[NP]) {
        #pragma unroll
        for(int n = 0; n < NP; n++) { kept[((b * PARTS + n / PART) * 64 + lane) * PART + n % PART] = h[n]; }
    };
    float dA[NP], dD = 0.0f, dBias = 0.0f;
    #pragma unroll
    for(int n = 0; n < NP; n++) { dA[n] = 0.0f; }
    if(s.valid) {
        const T *u = rowsOf<const T>(a.u, a.sequences, s.place), *delta = rowsOf<const T>(a.delta, a.sequences, s.place);
        const T *z = a.z.data ? rowsOf<const T>(a.z, a.sequences, s.place) : nullptr, *dout = rowsOf<const T>(g.out, a.sequences, s.place);
        T *du = g.u.data ? rowsOf<T>(g.u, a.sequences, s.place) : nullptr, *ddelta = g.delta.data ? rowsOf<T>(g.delta, a.sequences, s.place) : nullptr;
        T *dz = z && g.z.data ? rowsOf<T>(g.z, a.sequences, s.place) : nullptr;
        const uint32_t bcAt = s.group * a.states + s.firstState;
        const T *B = rowsOf<const T>(a.B, a.sequences, s.place) + bcAt, *C = rowsOf<const T>(a.C, a.sequences, s.place) + bcAt;
        const float bias = a.deltaBias ? a.deltaBias[channel] : 0.0f, skip = a.D ? a.D[channel] : 0.0f;
        const uint64_t sumRow = (uint64_t)s.tile * g.rows + (a.sequences.offsets ? s.place.first : (uint64_t)s.place.sequence * a.sequences.length);
        // Sums over the lanes of what a part gives B and C: folded in registers as far as two exchanges go, the rest through LDS for all rows of the block at once, where
        // a lane adds up half of the 16 shares of one value of one row
        float *const rowSum = rowSums + lane / 8 * 2 * NP + lane % 8 / 4 * NP + lane % 4 / 2;
        const auto addShares = [&](int part) {
            float x[8];
            const Pack<float, 4> *const from = (const Pack<float, 4>*)(shares + lane * 8);
            const Pack<float, 4> low = from[0], high = from[1];
            #pragma unroll
            for(int k = 0; k < 4; k++) { x[k] = low.v[k] + high.v[k]; }
            const float sum = (x[0] + x[2]) + (x[1] + x[3]);
            rowSum[part * PART] = sum + gennmi_lanes::partner<1>(sum);
        };
        float A[NP], h[NP], carry[NP];
        loadA<NP>(a, s, A);
        if(a.chunkState) { loadChunk<NP>(a, s, a.chunkState, number, h); loadChunk<NP>(a, s, g.chunkGradient, number, carry); }
        else { loadState<NP>(a, s, a.initialState, s.place.state, h); loadState<NP>(a, s, g.finalState, s.place.state, carry); }
        const uint32_t end = s.first + s.rows, blocks = (s.rows + R - 1) / R;
        StagedBC<T, NP, R> stage(B, C, a, s.numStates);
        for(uint32_t b = 0; b + 1 < blocks; b++) {
            const uint32_t row = s.first + b * R;
            T rawU[R], rawDelta[R];
            #pragma unroll
            for(int r = 0; r < R; r++) {
                rawU[r] = loadAt(u, row + r, a.u.rowStride, place);
                rawDelta[r] = loadAt(delta, row + r, a.delta.rowStride, place);
            }
            stage.fetch(row, end);
            keep(b, h);
            waveFence();
            stage.store(bc, row, end);
            waveFence();
            float nextB[NP];
            #pragma unroll
            for(int n = 0; n < NP; n++) { nextB[n] = bc[n]; }
            #pragma unroll
            for(int r = 0; r < R; r++) {
                float dt = widen(rawDelta[r]) + bias, Bn[NP];
                dt = a.softplus ? softplusOf(dt) : dt;
                const float w = dt * widen(rawU[r]);
                readAfter<NP>(h);
                #pragma unroll
                for(int n = 0; n < NP; n++) {
                    Bn[n] = nextB[n];
                    if(r + 1 < R) { nextB[n] = bc[(r + 1) * 2 * NP + n]; }
                }
                #pragma unroll
                for(int n = 0; n < NP; n++) { h[n] = __builtin_fmaf(exp2Of(dt * A[n]), h[n], w * Bn[n]); }
            }
        }
        if(blocks) { keep(blocks - 1, h); }
        for(uint32_t b = blocks; b-- > 0; ) {
            const uint32_t row = s.first + b * R;
            stage.fetch(row, end);
            float dt[R], uu[R], gy[R], q[R], rr[R], y[R];
            {
                T rawDelta[R], rawU[R], rawOut[R], rawZ[R];
                #pragma unroll
                for(int r = 0; r < R; r++) {
                    const uint32_t t = min(row + r, end - 1);
                    rawDelta[r] = loadAt(delta, t, a.delta.rowStride, place);
                    rawU[r] = loadAt(u, t, a.u.rowStride, place);
                    rawOut[r] = loadAt(dout, t, g.out.rowStride, place);
                }
                if(z) {
                    #pragma unroll
                    for(int r = 0; r < R; r++) { rawZ[r] = loadAt(z, min(row + r, end - 1), a.z.rowStride, place); }
                    #pragma unroll
                    for(int r = 0; r < R; r++) { const float zr = widen(rawZ[r]); gy[r] = widen(rawOut[r]) * (zr * logistic(zr)); }
                }
                else {
                    #pragma unroll
                    for(int r = 0; r < R; r++) { gy[r] = widen(rawOut[r]); }
                }
                #pragma unroll
                for(int r = 0; r < R; r++) {
                    // (rows behind the end, and lanes without a channel: dt, u and gradient 0 leave everything as it is)
                    const bool there = row + r < end && s.active;
                    const float raw = widen(rawDelta[r]) + bias;
                    const float time = a.softplus ? softplusOf(raw) : raw;
                    dt[r] = there ? time : 0.0f;
                    uu[r] = there ? widen(rawU[r]) : 0.0f;
                    gy[r] = there ? gy[r] : 0.0f;
                    q[r] = rr[r] = y[r] = 0.0f;
                }
            }
            waveFence();
            stage.store(bc, row, end);
            waveFence();
            // what a row's channel gets, when its sums over the states are there
            const auto finish = [&](int r) {
                const uint32_t t = row + r;
                if(!s.active) { return; }
                if(du) { storeAt(du, t, g.u.rowStride, place, narrow<T>(__builtin_fmaf(dt[r], q[r], skip * gy[r]))); }
                float d = __builtin_fmaf(uu[r], q[r], rr[r] * LN2);
                if(a.softplus) { d *= logistic(widen(loadAt(delta, t, a.delta.rowStride, place)) + bias); }
                if(ddelta) { storeAt(ddelta, t, g.delta.rowStride, place, narrow<T>(d)); }
                if(dz) {
                    const float zr = widen(loadAt(z, t, a.z.rowStride, place)), sig = logistic(zr), dd = widen(loadAt(dout, t, g.out.rowStride, place));
                    storeAt(dz, t, g.z.rowStride, place, narrow<T>(dd * __builtin_fmaf(skip, uu[r], y[r]) * (sig * (1.0f + zr * (1.0f - sig)))));
                }
                dBias += d;
                dD = __builtin_fmaf(gy[r], uu[r], dD);
            };
            #pragma unroll
            for(int part = 0; part < PARTS; part++) {
                float hs[R][PART], decay[R][PART], start[PART];
                waveFence();
                #pragma unroll
                for(int k = 0; k < PART; k++) { start[k] = kept[((b * PARTS + part) * 64 + lane) * PART + k]; }
                float nextB[PART], nextC[PART], terms[2 * PART];
                #pragma unroll
                for(int k = 0; k < PART; k++) { nextB[k] = bc[part * PART + k]; }
                if(part) { addShares(part - 1); }           // (of the part before: its trip through LDS is one with that of this part's states)
                #pragma unroll
                for(int r = 0; r < R; r++) {
                    const float w = dt[r] * uu[r];
                    float (&before)[PART] = r ? hs[r - 1] : start, Bn[PART];
                    readAfter<PART>(before);
                    #pragma unroll
                    for(int k = 0; k < PART; k++) {
                        Bn[k] = nextB[k];
                        if(r + 1 < R) { nextB[k] = bc[(r + 1) * 2 * NP + part * PART + k]; }
                    }
                    #pragma unroll
                    for(int k = 0; k < PART; k++) {
                        const int n = part * PART + k;
                        decay[r][k] = exp2Of(dt[r] * A[n]);
                        hs[r][k] = __builtin_fmaf(decay[r][k], before[k], w * Bn[k]);
                    }
                }
                #pragma unroll
                for(int k = 0; k < PART; k++) { terms[k] = terms[PART + k] = 0.0f; nextB[k] = bc[(R - 1) * 2 * NP + part * PART + k]; nextC[k] = bc[((R - 1) * 2 + 1) * NP + part * PART + k]; }
                #pragma unroll
                for(int r = R - 1; r >= 0; r--) {
                    const float w = dt[r] * uu[r];
                    const float (&before)[PART] = r ? hs[r - 1] : start;
                    float Bn[PART], Cn[PART];
                    if(r < R - 1) {
                        readAfter(q[r + 1], rr[r + 1], y[r + 1], carry[part * PART]);
                        readAfter<2 * PART>(terms);
                    }
                    readAfter<PART>(dA, part * PART);
                    // (the sums of the row behind: a chain of dependent steps, which this row's arithmetic fills)
                    if(r < R - 1) { shares[(r + 1) * 64 + lane] = gennmi_lanes::shareOfLanes<2 * PART>(terms); }
                    #pragma unroll
                    for(int k = 0; k < PART; k++) {
                        Bn[k] = nextB[k];
                        Cn[k] = nextC[k];
                        if(r) { nextB[k] = bc[(r - 1) * 2 * NP + part * PART + k]; nextC[k] = bc[((r - 1) * 2 + 1) * NP + part * PART + k]; }
                    }
                    #pragma unroll
                    for(int k = 0; k < PART; k++) {
                        const int n = part * PART + k;
                        const float dh = __builtin_fmaf(gy[r], Cn[k], carry[n]);
                        y[r] = __builtin_fmaf(Cn[k], hs[r][k], y[r]);
                        terms[k] = dh * w;
                        terms[PART + k] = gy[r] * hs[r][k];
                        q[r] = __builtin_fmaf(dh, Bn[k], q[r]);
                        carry[n] = decay[r][k] * dh;
                        const float x = carry[n] * before[k];
                        dA[n] = __builtin_fmaf(x, dt[r], dA[n]);
                        rr[r] = __builtin_fmaf(x, A[n], rr[r]);
                    }
                    if(r == 0) { shares[lane] = gennmi_lanes::shareOfLanes<2 * PART>(terms); }
                    if(part == PARTS - 1 && row + r < end) {
                        if(SLABS) {
                            sums[((slab * R + r) * 3) * 64 + lane] = q[r];
                            sums[((slab * R + r) * 3 + 1) * 64 + lane] = rr[r];
                            sums[((slab * R + r) * 3 + 2) * 64 + lane] = y[r];
                        }
                        else { finish(r); }
                    }
                }
            }
            waveFence();
            addShares(PARTS - 1);
            waveFence();
            #pragma unroll
            for(int e = 0; e < R * 2 * NP / 64; e++) {
                const uint32_t at = e * 64 + lane, r = at / (2 * NP), which = (at / NP) % 2, n = at % NP;
                if(row + r < end && n < s.numStates) { (g.sumBC + (sumRow + row + r) * 2 * a.states)[which * a.states + s.firstState + n] = rowSums[at]; }
            }
            if(SLABS) {
                __syncthreads();
                #pragma unroll
                for(int r = 0; r < R; r++) {
                    if(r % a.slabs == slab && row + r < end) {
                        q[r] = rr[r] = y[r] = 0.0f;
                        for(uint32_t k = 0; k < a.slabs; k++) {
                            q[r] += sums[((k * R + r) * 3) * 64 + lane];
                            rr[r] += sums[((k * R + r) * 3 + 1) * 64 + lane];
                            y[r] += sums[((k * R + r) * 3 + 2) * 64 + lane];
                        }
                        finish(r);
                    }
                }
                __syncthreads();
            }
        }
        if(!a.chunkState) { storeState<NP>(a, s, g.initialState, s.place.state, carry); }
    }
    // Sums over the chunk (numbers without a chunk leave zeros)
    float *const to = g.sums + (uint64_t)number * (a.states + 2) * a.channels;
    if(s.active) {
        #pragma unroll
        for(int n = 0; n < NP; n++) { if(n < (int)s.numStates) { (to + (uint64_t)(s.firstState + n) * a.channels)[channel] = dA[n]; } }
    }
    if(SLABS) {
        sums[(slab * 2) * 64 + lane] = dD;
        sums[(slab * 2 + 1) * 64 + lane] = dBias;
        __syncthreads();
        if(slab == 0) {
            dD = dBias = 0.0f;
            for(uint32_t k = 0; k < a.slabs; k++) { dD += sums[(k * 2) * 64 + lane]; dBias += sums[(k * 2 + 1) * 64 + lane]; }
        }
    }
    if(slab == 0 && s.active) {
        (to + (uint64_t)a.states * a.channels)[channel] = dD;
        (to + (uint64_t)(a.states + 1) * a.channels)[channel] = dBias;
    }
}

// Sums over a group's tiles of what belongs to a row
template<typename T>
__global__ __launch_bounds__(256)
void scanRowSumKernel(ScanArgs a, ScanGradientArgs g)
{
    const uint32_t width = a.groups * a.states;
    const uint64_t item = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    const uint64_t row = item / (2 * width);
    if(row >= g.rows) { return; }
    const uint32_t e = (uint32_t)(item - row * 2 * width), which = e / width, group = (e - which * width) / a.states, n = e % a.states;
    uint32_t sequence = 0;
    uint64_t t = row;
    if(!a.sequences.offsets) { sequence = (uint32_t)(row / a.sequences.length); t = row - (uint64_t)sequence * a.sequences.length; }
    else {
        // rows of no sequence (in front of the first, behind one that was cut, behind the last) are left as they were
        uint32_t low = 0, high = a.sequences.count;
        while(high - low > 1) {
            const uint32_t middle = low + (high - low) / 2;
            if(firstRow(a.sequences, middle) <= row) { low = middle; } else { high = middle; }
        }
        Place p;
        if(!describe(a.sequences, low, p) || row < p.first || row - p.first >= p.length) { return; }
    }
    float sum = 0.0f;
    for(uint32_t k = 0; k < a.groupTiles; k++) { sum += g.sumBC[(((uint64_t)(group * a.groupTiles + k) * g.rows + row) * 2 + which) * a.states + n]; }
    const gennmi_rows_t &to = which ? g.C : g.B;
    if(!to.data) { return; }
    T *at = (T*)to.data + (a.sequences.offsets ? row * to.rowStride : (uint64_t)sequence * to.sequenceStride + t * to.rowStride);
    at[group * a.states + n] = narrow<T>(sum);
}
}
#endif

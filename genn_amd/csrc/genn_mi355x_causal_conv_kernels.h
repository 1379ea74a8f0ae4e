// Part of libgenn_mi355x.so: included by genn_mi355x_sequence.hip only.
//
// Short causal convolution of every channel by itself:  s[t] = bias + sum_k w[k] x[t - (K - 1) + k],  out = s or s sigmoid(s).
// Bound by memory: 2 K + 6 operations for one element read and one written.  A thread owns a few neighbouring channels (VEC of
// them, one access a row) and a chunk of rows, which it walks with the last K inputs in registers, so that a row is read once but for
// the K - 1 rows before a chunk.  4096 rows x 4096 channels x 4 taps in bf16: 14.8 us, 4.5 TB/s (with 8 channels a thread 17.8, 8 rows ahead 16.0).
#ifndef GENN_MI355X_CAUSAL_CONV_KERNELS_H
#define GENN_MI355X_CAUSAL_CONV_KERNELS_H

namespace
{
struct ConvArgs
{
    Sequences sequences;
    gennmi_rows_t x, out;
    const float *weight, *bias;
    const void *initialState; void *finalState;
    uint32_t channels, taps, silu, vectors;         // vectors: threads a row
    uint32_t numbers;                               // chunk numbers
};
struct ConvGradientArgs
{
    gennmi_rows_t out, x;
    const void *finalState; void *initialState;
    float *partial;                 // [numbers][taps + 1][channels]: sums over a chunk for the weights and the bias; or NULL
};

__device__ inline float sigmoid(float x) { return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(x * -1.44269504f)); }

template<typename T, int VEC> __device__ inline void widenRow(const Pack<T, VEC> &p, float (&to)[VEC])
{
    #pragma unroll
    for(int v = 0; v < VEC; v++) { to[v] = widen(p.v[v]); }
}
template<typename T, int VEC> __device__ inline void loadRow(const T *from, float (&to)[VEC]) { widenRow<T, VEC>(*(const Pack<T, VEC>*)from, to); }
// AHEAD rows on their way while as many before them are worked on; behind row `last` that one again
constexpr int AHEAD = 4;
template<typename T, int VEC> struct RowsAhead
{
    Pack<T, VEC> raw[AHEAD];
    __device__ inline void fetch(const T *rows, uint64_t stride, uint32_t row, uint32_t last)
    {
        #pragma unroll
        for(int r = 0; r < AHEAD; r++) { raw[r] = *(const Pack<T, VEC>*)(rows + (uint64_t)min(row + r, last) * stride); }
    }
};
template<typename T, int VEC> __device__ inline void storeRow(T *to, const float (&from)[VEC])
{
    Pack<T, VEC> p;
    #pragma unroll
    for(int v = 0; v < VEC; v++) { p.v[v] = narrow<T>(from[v]); }
    *(Pack<T, VEC>*)to = p;
}
// (a thread's weights are neighbours in memory: taken four at a time where they lie so)
template<int K, int VEC> __device__ inline void loadWeights(const ConvArgs &a, uint32_t channel, float (&w)[K][VEC], float (&bias)[VEC])
{
    const float *from = a.weight + (uint64_t)channel * K;
    if(K * VEC % 4 == 0 && (uintptr_t)a.weight % 16 == 0) {
        #pragma unroll
        for(int i = 0; i < K * VEC / 4; i++) {
            const Pack<float, 4> p = *(const Pack<float, 4>*)(from + 4 * i);
            #pragma unroll
            for(int j = 0; j < 4; j++) { w[(4 * i + j) % K][(4 * i + j) / K] = p.v[j]; }
        }
    }
    else {
        #pragma unroll
        for(int i = 0; i < K * VEC; i++) { w[i % K][i / K] = from[i]; }
    }
    #pragma unroll
    for(int v = 0; v < VEC; v++) { bias[v] = a.bias ? a.bias[channel + v] : 0.0f; }
}
// The K - 1 rows before row `first` of the sequence, as window[1 ..]
template<typename T, int K, int VEC>
__device__ inline void loadWindow(const ConvArgs &a, const T *x, const Place &p, uint32_t first, uint32_t channel, float (&window)[K][VEC])
{
    const T *state = (const T*)a.initialState;
    #pragma unroll
    for(int j = 1; j < K; j++) {
        #pragma unroll
        for(int v = 0; v < VEC; v++) { window[j][v] = 0.0f; }
        const long long t = (long long)first - (K - j);
        if(t >= 0) { loadRow<T, VEC>(x + (uint64_t)t * a.x.rowStride + channel, window[j]); }
        else if(state) { loadRow<T, VEC>(state + ((uint64_t)p.state * (K - 1) + (uint64_t)(K - 1 + t)) * a.channels + channel, window[j]); }
    }
}
// The final state: rows length - (K - 1) .. length - 1, of which negative ones are the initial state's, still in the window of the first
// chunk.  One thread reads what it needs of the initial state before it writes: the two may be the same array.
template<typename T, int K, int VEC>
__device__ inline void storeState(const ConvArgs &a, const T *x, const Place &p, uint32_t channel, const float (&window)[K][VEC])
{
    T *to = (T*)a.finalState + (uint64_t)p.state * (K - 1) * a.channels + channel;
    float rows[K][VEC];         // (all read before the first is written: one trip to memory)
    #pragma unroll
    for(int j = 1; j < K; j++) {
        const long long t = (long long)p.length - (K - j);
        if(t >= 0) { loadRow<T, VEC>(x + (uint64_t)t * a.x.rowStride + channel, rows[j]); }
        else {
            // row t lies -t rows before the first: window[K + t]
            #pragma unroll
            for(int i = 1; i < K; i++) {
                #pragma unroll
                for(int v = 0; v < VEC; v++) { rows[j][v] = i == 1 || i == K + t ? window[i][v] : rows[j][v]; }
            }
        }
    }
    #pragma unroll
    for(int j = 1; j < K; j++) { storeRow<T, VEC>(to + (uint64_t)(j - 1) * a.channels, rows[j]); }
}

template<int K, int VEC>
__device__ inline void product(const float (&w)[K][VEC], const float (&window)[K][VEC], const float (&bias)[VEC], float (&s)[VEC])
{
    #pragma unroll
    for(int v = 0; v < VEC; v++) {
        s[v] = bias[v];
        #pragma unroll
        for(int k = 0; k < K; k++) { s[v] = __builtin_fmaf(w[k][v], window[k][v], s[v]); }
    }
}
// One row on: what is at k + 1 moves to k
template<int K, int VEC> __device__ inline void shift(float (&window)[K][VEC])
{
    #pragma unroll
    for(int k = 0; k < K - 1; k++) {
        #pragma unroll
        for(int v = 0; v < VEC; v++) { window[k][v] = window[k + 1][v]; }
    }
}

// (the chunk of a thread; lanes of a wavefront may lie in two chunks, so nothing here is uniform)
__device__ inline bool convPlace(const ConvArgs &a, uint32_t number, Place &p)
{
    uint32_t sequence;
    if(!a.sequences.offsets) {
        sequence = number / a.sequences.perSequence;
        p.index = number - sequence * a.sequences.perSequence;
    }
    else {
        uint32_t low = 0, high = a.sequences.count;         // firstChunk(low) <= number
        while(high - low > 1) {
            const uint32_t middle = low + (high - low) / 2;
            if(firstChunk(a.sequences, middle) <= number) { low = middle; } else { high = middle; }
        }
        sequence = low;
        p.index = number - (uint32_t)firstChunk(a.sequences, sequence);
    }
    if(sequence >= a.sequences.count || !describe(a.sequences, sequence, p)) { return false; }
    return (uint64_t)p.index * a.sequences.chunk < p.length || p.index == 0;
}

template<typename T, int K, int VEC>
__global__ __launch_bounds__(256)
void causalConvKernel(ConvArgs a)
{
    uint32_t number, channel;
    divideItem(a.vectors, number, channel);
    channel *= VEC;
    Place p;
    if(number >= a.numbers || !convPlace(a, number, p)) { return; }
    const T *x = rowsOf<const T>(a.x, a.sequences, p);
    T *out = rowsOf<T>(a.out, a.sequences, p) + channel;
    const uint32_t first = p.index * a.sequences.chunk, last = (uint32_t)min((uint64_t)first + a.sequences.chunk, (uint64_t)p.length);
    float w[K][VEC], window[K][VEC], bias[VEC];
    RowsAhead<T, VEC> next;
    if(first < last) { next.fetch(x + channel, a.x.rowStride, first, last - 1); }
    loadWindow<T, K, VEC>(a, x, p, first, channel, window);
    loadWeights<K, VEC>(a, channel, w, bias);
    if(K > 1 && p.index == 0 && a.finalState) { storeState<T, K, VEC>(a, x, p, channel, window); }
    for(uint32_t t = first; t < last; t += AHEAD) {
        const RowsAhead<T, VEC> rows = next;
        if(t + AHEAD < last) { next.fetch(x + channel, a.x.rowStride, t + AHEAD, last - 1); }
        #pragma unroll
        for(int r = 0; r < AHEAD; r++) {
            shift<K, VEC>(window);
            widenRow<T, VEC>(rows.raw[r], window[K - 1]);
            float s[VEC];
            product<K, VEC>(w, window, bias, s);
            if(a.silu) {
                #pragma unroll
                for(int v = 0; v < VEC; v++) { s[v] *= sigmoid(s[v]); }
            }
            if(t + r < last) { storeRow<T, VEC>(out + (uint64_t)(t + r) * a.out.rowStride, s); }
        }
    }
}

// Gradients.  With ds[t] = dout[t] f'(s[t]):  dx[p] = sum_k w[k] ds[p + (K - 1) - k], which is complete when ds[p + K - 1] is there, so a
// thread walks K - 1 rows further than its chunk, with the last K inputs and the last K ds in registers, and writes row t - (K - 1)
// at row t; in front of a sequence's first chunk these are the rows of the initial state.  dw[k] = sum ds[t] x[t - (K - 1) + k] and
// dbias are summed over the chunk and then over chunks by a kernel of their own, always in the same order.  8 x 2048 rows x 2048 channels x 4 taps in bf16 take 54 us
// with the sums (5 of them), 3.7 TB/s for what has to be read and written; vector units are busy for 87 % of the time (44 instructions an element).
template<typename T, int K, int VEC>
__global__ __launch_bounds__(256)
void causalConvBackwardKernel(ConvArgs a, ConvGradientArgs g)
{
    uint32_t number, channel;
    divideItem(a.vectors, number, channel);
    channel *= VEC;
    if(number >= a.numbers) { return; }
    float w[K][VEC], window[K][VEC], bias[VEC], ds[K][VEC], dw[K][VEC], db[VEC];
    #pragma unroll
    for(int v = 0; v < VEC; v++) {
        db[v] = 0.0f;
        #pragma unroll
        for(int k = 0; k < K; k++) { dw[k][v] = ds[k][v] = 0.0f; }
    }
    Place p;
    if(convPlace(a, number, p)) {
        const T *x = rowsOf<const T>(a.x, a.sequences, p), *dout = rowsOf<const T>(g.out, a.sequences, p);
        T *dx = g.x.data ? rowsOf<T>(g.x, a.sequences, p) : nullptr;
        T *dstate = (T*)g.initialState;
        const T *dfinal = (const T*)g.finalState;
        const uint32_t first = p.index * a.sequences.chunk, last = (uint32_t)min((uint64_t)first + a.sequences.chunk, (uint64_t)p.length);
        RowsAhead<T, VEC> nextX, nextOut;
        if(p.length) {
            nextX.fetch(x + channel, a.x.rowStride, first, p.length - 1);
            nextOut.fetch(dout + channel, g.out.rowStride, first, p.length - 1);
        }
        loadWindow<T, K, VEC>(a, x, p, first, channel, window);
        loadWeights<K, VEC>(a, channel, w, bias);
        // (dx of rows before `last`; in the first chunk of rows -(K - 1) on)
        const long long from = p.index == 0 ? -(long long)(K - 1) : (long long)first;
        const uint32_t walk = last + (K - 1);
        for(uint32_t group = first; group < walk; group += AHEAD) {
            const RowsAhead<T, VEC> rowsX = nextX, rowsOut = nextOut;
            if(group + AHEAD < walk && p.length) {
                nextX.fetch(x + channel, a.x.rowStride, group + AHEAD, p.length - 1);
                nextOut.fetch(dout + channel, g.out.rowStride, group + AHEAD, p.length - 1);
            }
            // Rows that need no looking after: all of the chunk's own, and so are those whose dx is complete with them
            const bool plain = (long long)group - (K - 1) >= (long long)first && group + AHEAD <= last;
            const auto walkRows = [&](auto known) {
                constexpr bool PLAIN = decltype(known)::value;
                #pragma unroll
                for(int r = 0; r < AHEAD; r++) {
                    const uint32_t t = group + r;
                    shift<K, VEC>(window);
                    shift<K, VEC>(ds);
                    // (ds of rows that are not there is zero, and their inputs, which may be anything, count for nothing)
                    widenRow<T, VEC>(rowsX.raw[r], window[K - 1]);
                    widenRow<T, VEC>(rowsOut.raw[r], ds[K - 1]);
                    if(a.silu) {
                        float s[VEC];
                        product<K, VEC>(w, window, bias, s);
                        #pragma unroll
                        for(int v = 0; v < VEC; v++) { const float q = sigmoid(s[v]); ds[K - 1][v] *= q * (1.0f + s[v] * (1.0f - q)); }
                    }
                    if(!PLAIN && t >= p.length) {
                        #pragma unroll
                        for(int v = 0; v < VEC; v++) { ds[K - 1][v] = 0.0f; }
                    }
                    if(PLAIN || t < last) {
                        #pragma unroll
                        for(int v = 0; v < VEC; v++) {
                            db[v] += ds[K - 1][v];
                            #pragma unroll
                            for(int k = 0; k < K; k++) { dw[k][v] = __builtin_fmaf(ds[K - 1][v], window[k][v], dw[k][v]); }
                        }
                    }
                    const long long row = (long long)t - (K - 1);
                    if(!PLAIN && !(row >= from && t < walk)) { continue; }
                    float d[VEC];
                    #pragma unroll
                    for(int v = 0; v < VEC; v++) {
                        d[v] = 0.0f;
                        #pragma unroll
                        for(int k = 0; k < K; k++) { d[v] = __builtin_fmaf(w[k][v], ds[K - 1 - k][v], d[v]); }
                    }
                    const long long behind = row - ((long long)p.length - (K - 1));         // its place in the final state
                    if(!PLAIN && dfinal && behind >= 0) {
                        float f[VEC];
                        loadRow<T, VEC>(dfinal + ((uint64_t)p.state * (K - 1) + (uint64_t)behind) * a.channels + channel, f);
                        #pragma unroll
                        for(int v = 0; v < VEC; v++) { d[v] += f[v]; }
                    }
                    if(PLAIN || row >= 0) { if(dx) { storeRow<T, VEC>(dx + (uint64_t)row * g.x.rowStride + channel, d); } }
                    else if(dstate) { storeRow<T, VEC>(dstate + ((uint64_t)p.state * (K - 1) + (uint64_t)(row + K - 1)) * a.channels + channel, d); }
                }
            };
            if(__all(plain)) { walkRows(std::true_type{}); } else { walkRows(std::false_type{}); }
        }
    }
    if(g.partial) {
        float *to = g.partial + (uint64_t)number * (K + 1) * a.channels + channel;
        #pragma unroll
        for(int v = 0; v < VEC; v++) {
            #pragma unroll
            for(int k = 0; k < K; k++) { to[(uint64_t)k * a.channels + v] = dw[k][v]; }
            to[(uint64_t)K * a.channels + v] = db[v];
        }
    }
}
}
#endif

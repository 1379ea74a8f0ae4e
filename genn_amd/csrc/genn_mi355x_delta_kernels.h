// Part of genn_mi355x_delta.hip: kernels of the gated delta rule.
//
// Of one head, with unit keys k^ and queries q^, a[t] = exp(g[t]):
//   S[t] = a[t] S[t-1] + k^[t] u[t]',   u[t] = beta[t] w[t],   w[t] = v[t] - a[t] S[t-1]' k^[t],   out[t] = scale S[t]' q^[t]
// Over a chunk of rows that begins with the state S, with G[i] = exp(sum of g up to row i) and D[i][j] = G[i] / G[j] for i >= j:
//   w[i] = v[i] - G[i] S' k^[i] - sum_{j<i} M[i][j] beta[j] w[j],   M[i][j] = D[i][j] k^[i].k^[j]
// so that w = (I + M beta)^-1 r with r = v - G k^ S, and the inverse is I - N beta with (I + M beta) N = M.  Then
//   out = scale G q^ S + P u,   P[i][j] = scale D[i][j] q^[i].k^[j] for i >= j,   S behind the chunk = G[last] S + sum_j D[last][j] k^[j] u[j]'.
// The transposed inverse of the gradients, (I + beta M')^-1, is I - beta N': N serves both, and no beta is divided by.
//
// M, N and P do not need the state: a work-group a chunk and key head finds them (deltaChunkKernel).  Then a state's columns do not need each other:
// a wavefront owns 16 of them, all rows in registers, and walks the chunks (walkForwards, walkBackwards).  Its results become operands of the next product
// without leaving the registers; what multiplies them (keys, N, P) is shared by the work-group's wavefronts through LDS.  Products have fp32 accuracy (genn_mi355x_planes.h).
#ifndef GENN_MI355X_DELTA_KERNELS_H
#define GENN_MI355X_DELTA_KERNELS_H

#include "genn_mi355x_lanes.h"
#include "genn_mi355x_planes.h"

namespace gennmi_delta
{
using namespace gennmi_elements;
using namespace gennmi_planes;
using gennmi_lanes::partner;

// Keeps the compiler from asking for all of LDS's operands at once, which costs more registers than there are
__device__ inline void inTurn() { __builtin_amdgcn_sched_barrier(0); }

// What the rows of a chunk need of one head
template<int C> struct alignas(16) RowTable
{
    float keyState[C];      // G / |k|: times the key and the state
    float beta[C];
    float keyEnd[C];        // D[last] / |k|: times the key and u, what the row leaves in the state behind the chunk
    float queryState[C];    // scale G / |q|
    float keyUnit[C], queryUnit[C];     // 1 / |k|, 1 / |q|
    double sum[C];          // of g, since the chunk's beginning
};
// The first four of them, in LDS; four rows that are a lane's in a result an access
template<int C> struct RowFactors
{
    float *at;
    __device__ f32x4 four(int which, uint32_t row) const { return *(const f32x4*)(at + which * C + row); }
    __device__ f32x4 keyState(uint32_t row) const { return four(0, row); }
    __device__ f32x4 beta(uint32_t row) const { return four(1, row); }
    __device__ f32x4 keyEnd(uint32_t row) const { return four(2, row); }
    __device__ f32x4 queryState(uint32_t row) const { return four(3, row); }
};
struct ChunkTable { float decay; uint32_t bad; };          // G[last]; first row from which nothing is finite, or the chunk's rows

struct DeltaArgs
{
    Sequences chunks, segments;
    gennmi_rows_t q, k, v, out, g, beta;
    const float *initialState;
    float *finalState;
    uint32_t heads, keyHeads, group, keys, values, normalise, wide, wideValues, columnBlocks;
    uint32_t padded;                // values, up to a multiple of 32: the width of what is kept of them
    float scale, epsilon;
    float *correction, *score;      // of each chunk number and head: -N and P, [C][C]
    void *rows;                     // RowTable
    ChunkTable *table;
    uint32_t segmentNumbers, moveBlocks;        // moveBlocks: of the columns of a segment's `move`
    float *segmentStates, *segmentMoves;        // of each segment and head [DK][padded], [DK][DK]; NULL: sequences are not cut
    float *states, *errors;         // kept for gradients, of each chunk number and head: the state in front of it [DK][padded], w [C][padded]
};

// Gates below this are as good as minus infinity (exp(-1e6) is 0), and sums of them are finite
__device__ inline float clampGate(float g) { return g < -1e6f ? -1e6f : g; }
__device__ inline float decayOver(double sum) { return __builtin_amdgcn_exp2f((float)(sum * 1.4426950408889634)); }
__device__ inline bool finite(float x) { return fabsf(x) < __builtin_inff(); }

template<typename T> __device__ inline const T *rowAt(const gennmi_rows_t &r, const Sequences &s, const Place &p, uint32_t row) { return rowsOf<const T>(r, s, p) + (uint64_t)row * r.rowStride; }

// ---- what a chunk needs that does not depend on the state
// FOLDED: for outputs alone, -N beta and P beta (I - N beta) are left, which r is multiplied with at once; else, for gradients, -N and P.
// (M and P lie where the keys and queries were)
// What bounds it is waiting (three quarters of a wavefront's cycles): loads, then a triangle solved row by row by one wavefront.  Hence four work-groups a compute unit, whose pauses fill each other, at the price of 18 registers
// that are spilled: 64 chunks x 32 heads of 128 keys in bf16 39 us, 256 x 16 for gradients 108 (180 MB written).
template<typename T, int C, int DK> constexpr uint32_t chunkSquares() { const uint32_t keys = 2 * planesOf<T> * C * DK * 2, squares = 2 * C * (C + 4) * 4; return keys > squares ? keys : squares; }
template<typename T, int C, int DK> constexpr uint32_t chunkLds() { return chunkSquares<T, C, DK>() + C * (8 + 3 * 4) + 16; }

template<typename T, int C, int DK, bool FOLDED>
__global__ __launch_bounds__(256, 4)
void deltaChunkKernel(DeltaArgs a)
{
    constexpr int NP = planesOf<T>, B = C / 16, PLANE = C * DK, MP = C + 4, TILES = B * B / 4;
    extern __shared__ __align__(16) char lds[];
    uint16_t *const keyPlanes = (uint16_t*)lds, *const queryPlanes = keyPlanes + NP * PLANE;
    float *const m = (float*)lds, *const scores = m + C * MP;
    double *const sums = (double*)(lds + chunkSquares<T, C, DK>());
    float *const keyUnit = (float*)(sums + C), *const queryUnit = keyUnit + C, *const beta = queryUnit + C;
    uint32_t *const bad = (uint32_t*)(beta + C);
    const uint32_t number = blockIdx.x / a.keyHeads, keyHead = blockIdx.x - number * a.keyHeads;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n16 = lane & 15, g = lane >> 4;
    Place p;
    if(!locate(a.chunks, number, p)) { return; }
    const uint32_t begin = p.index * C, count = min((uint32_t)C, p.length - min(p.length, begin));
    if(!count) { return; }

    // keys and queries as planes, and what they are divided by
    #pragma unroll
    for(int item = 0; item < C * DK / 8; item += 256) {
        const uint32_t i = item + tid, row = i / (DK / 8), at = i % (DK / 8) * 8;
        if(C * DK / 8 < 256 && i >= C * DK / 8) { break; }
        const uint32_t valid = row < count && at < a.keys ? min(8u, a.keys - at) : 0;
        #pragma unroll
        for(int which = 0; which < 2; which++) {
            const gennmi_rows_t &r = which ? a.q : a.k;
            const Eight<T> x = loadUnit(rowAt<T>(r, a.chunks, p, valid ? begin + row : begin) + (valid ? keyHead * a.keys + at : 0), valid, a.wide);
            float sum = 0.0f;
            #pragma unroll
            for(int e = 0; e < 8; e++) { const float f = widen(x.at(e)); sum = __builtin_fmaf(f, f, sum); }
            storeUnit((which ? queryPlanes : keyPlanes) + unitAt<DK>(row, at / 8), PLANE, x);
            sum += partner<1>(sum);
            sum += partner<2>(sum);
            sum += partner<4>(sum);
            if(DK == 128) { sum += partner<8>(sum); }
            if(at == 0) { (which ? queryUnit : keyUnit)[row] = row >= count ? 0.0f : a.normalise ? 1.0f / sqrtf(sum + a.epsilon) : 1.0f; }
        }
    }
    __syncthreads();

    // products of all keys with all keys and queries; tiles above the diagonal are left out
    f32x4 kk[TILES], qk[TILES];
    const auto tileRow = [&](int t) { return C == 64 ? wave : wave >> 1; };
    const auto tileColumn = [&](int t) { return C == 64 ? (uint32_t)t : wave & 1; };
    // (a walk has the first 32 rows of a square without the columns behind them)
    const auto isRead = [](uint32_t tileRow, uint32_t tileColumn) { return tileRow >= 2 || tileColumn < 2; };
    #pragma unroll
    for(int t = 0; t < TILES; t++) {
        kk[t] = qk[t] = f32x4{0, 0, 0, 0};
        if(tileColumn(t) > tileRow(t)) { continue; }
        #pragma unroll
        for(int s = 0; s < DK / 32; s++) {
            inTurn();
            const uint32_t ra = unitAt<DK>(tileRow(t) * 16 + n16, 4 * s + g), rb = unitAt<DK>(tileColumn(t) * 16 + n16, 4 * s + g);
            const Planes<NP> kb = fetch<NP>(keyPlanes + rb, PLANE);
            kk[t] = multiply(fetch<NP>(keyPlanes + ra, PLANE), kb, kk[t]);
            qk[t] = multiply(fetch<NP>(queryPlanes + ra, PLANE), kb, qk[t]);
        }
    }

    for(uint32_t inGroup = 0; inGroup < a.group; inGroup++) {
        const uint32_t head = keyHead * a.group + inGroup;
        const uint64_t at = (uint64_t)number * a.heads + head;
        RowTable<C> *const rows = (RowTable<C>*)a.rows + at;
        if(tid == 0) { *bad = C; }
        float decay = 0.0f;
        if(wave == 0) {
            const bool valid = lane < count;
            const float b = valid ? rowAt<float>(a.beta, a.chunks, p, begin + lane)[head] : 0.0f;
            double sum = valid ? (double)clampGate(rowAt<float>(a.g, a.chunks, p, begin + lane)[head]) : 0.0;
            #pragma unroll
            for(int w = 1; w < C; w *= 2) {
                const double before = __shfl_up(sum, w);
                if(lane >= (uint32_t)w) { sum += before; }
            }
            const double last = __shfl(sum, C - 1);
            decay = decayOver(last);
            if(lane < C) {
                const float since = decayOver(sum), until = decayOver(last - sum), ku = keyUnit[lane], qu = queryUnit[lane];
                sums[lane] = sum;
                beta[lane] = b;
                rows->keyState[lane] = since * ku;
                rows->beta[lane] = b;
                rows->keyEnd[lane] = until * ku;
                rows->queryState[lane] = a.scale * since * qu;
                rows->keyUnit[lane] = ku;
                rows->queryUnit[lane] = qu;
                rows->sum[lane] = sum;
                // (sum, b and the key's length: what makes a row's errors no numbers, also in a chunk's first row)
                if(valid && !(finite(b) && finite(since) && finite(ku))) { atomicMin(bad, lane); }
            }
        }
        __syncthreads();
        float *const score = a.score + at * C * C, *const correction = a.correction + at * C * C;
        #pragma unroll
        for(int t = 0; t < TILES; t++) {
            const uint32_t column = tileColumn(t) * 16 + n16;
            const double sum = sums[column];
            const float ku = keyUnit[column];
            #pragma unroll
            for(int r = 0; r < 4; r++) {
                const uint32_t row = tileRow(t) * 16 + 4 * g + r;
                const float d = row >= column ? decayOver(sums[row] - sum) : 0.0f;
                const float x = row > column ? d * (keyUnit[row] * kk[t][r] * ku) : 0.0f;
                const float y = row >= column ? d * (a.scale * (queryUnit[row] * qk[t][r] * ku)) : 0.0f;
                if(!finite(x)) { atomicMin(bad, row); }
                m[row * MP + column] = x;
                if(FOLDED) { scores[row * MP + column] = y; } else if(isRead(row / 16, column / 16)) { score[row * C + column] = y; }
            }
        }
        __syncthreads();
        const uint32_t from = *bad;
        if(from < C) {      // (nothing finite from that row on: the rows before it must not meet it)
            for(uint32_t i = from * C + tid; i < C * C; i += 256) {
                m[i / C * MP + i % C] = 0.0f;
                if(FOLDED) { scores[i / C * MP + i % C] = 0.0f; } else { score[i] = 0.0f; }
            }
            if(tid >= from && tid < C) { beta[tid] = 0.0f; }
            __syncthreads();
        }
        if(tid == 0) { a.table[at] = ChunkTable{decay, from}; }
        // N's blocks on the diagonal: a lane solves one column, row after row
        if(wave == 0 && lane < C) {
            const uint32_t block = lane & ~15u;
            float x[16];
            #pragma unroll
            for(int i = 0; i < 16; i++) {
                x[i] = m[(block + i) * MP + lane];
                #pragma unroll
                for(int j = 0; j < i; j++) { x[i] = __builtin_fmaf(-m[(block + i) * MP + block + j] * beta[block + j], x[j], x[i]); }
            }
            #pragma unroll
            for(int i = 0; i < 16; i++) { m[(block + i) * MP + lane] = x[i]; }
        }
        __syncthreads();
        // Below it: N[r] = Y - N[r][r] beta Y with Y = M[r] - sum_{s<r} M[r][s] beta N[s], a block column a wavefront
        if(wave < B) {
            f32x4 found[B];
            const auto result = [&](uint32_t row) { f32x4 x; for(int r = 0; r < 4; r++) { x[r] = m[(row * 16 + 4 * g + r) * MP + wave * 16 + n16]; } return x; };
            const auto operand = [&](uint32_t row, uint32_t column) {
                f32x4 x;
                #pragma unroll
                for(int e = 0; e < 4; e++) { x[e] = -m[(row * 16 + n16) * MP + column * 16 + 4 * g + e] * beta[column * 16 + 4 * g + e]; }
                return x;
            };
            #pragma unroll
            for(int r = 0; r < B; r++) {
                if((uint32_t)r < wave) { found[r] = f32x4{0, 0, 0, 0}; continue; }
                found[r] = result(r);
                if((uint32_t)r == wave) { continue; }
                #pragma unroll
                for(int s = 0; s < r; s++) { if((uint32_t)s >= wave) { found[r] = multiply(operand(r, s), found[s], found[r]); } }
                found[r] = multiply(operand(r, r), found[r], found[r]);
            }
            const float betaColumn = FOLDED ? beta[wave * 16 + n16] : 1.0f;
            #pragma unroll
            for(int r = 0; r < B; r++) {
                #pragma unroll
                for(int e = 0; e < 4; e++) {
                    found[r][e] *= -betaColumn;
                    if(isRead(r, wave)) { correction[(r * 16 + 4 * g + e) * C + wave * 16 + n16] = found[r][e]; }
                }
            }
            if constexpr(FOLDED) {
                // P beta (I - N beta), the same block column
                #pragma unroll
                for(int r = 0; r < B; r++) {
                    f32x4 y = {0, 0, 0, 0};
                    if((uint32_t)r >= wave) {
                        #pragma unroll
                        for(int e = 0; e < 4; e++) { y[e] = scores[(r * 16 + 4 * g + e) * MP + wave * 16 + n16] * betaColumn; }
                        #pragma unroll
                        for(int t = 0; t <= r; t++) {
                            if((uint32_t)t < wave) { continue; }
                            f32x4 x;
                            #pragma unroll
                            for(int e = 0; e < 4; e++) { x[e] = scores[(r * 16 + n16) * MP + t * 16 + 4 * g + e] * beta[t * 16 + 4 * g + e]; }
                            y = multiply(x, found[t], y);
                        }
                    }
                    if(!isRead(r, wave)) { continue; }
                    #pragma unroll
                    for(int e = 0; e < 4; e++) { score[(r * 16 + 4 * g + e) * C + wave * 16 + n16] = y[e]; }
                }
            }
        }
        __syncthreads();
    }
}

// ---- the walk over chunks
// Writes outputs; keeps states and errors for gradients; or finds what a segment of a sequence does to the state in front of it, S behind = move S + its own.
enum { WALK_OUTPUTS, WALK_KEEP, WALK_SUMMARY };

// A lower triangle of C rows and columns in LDS: blocks of 32 rows, each as wide as it has to be
template<int C> struct Triangle
{
    static constexpr uint32_t elements = C == 64 ? 3 * 1024 : 1024;
    // unit of a row
    __device__ static uint32_t at(uint32_t row, uint32_t unit) { return C == 64 && row >= 32 ? 1024 + unitAt<64>(row - 32, unit) : unitAt<32>(row, unit); }
    // which four neighbours of [C][C] item k is, of 8 of each of the first 32 rows and 16 of the others
    static constexpr int items = C == 64 ? 768 : 256;
    __device__ static uint32_t row(uint32_t k) { return k < 256 ? k / 8 : 32 + (k - 256) / 16; }
    __device__ static uint32_t column(uint32_t k) { return (k < 256 ? k % 8 : (k - 256) % 16) * 4; }
};
// LDS of a walk, in elements of 16 bits: keys, queries, -N, P, factors of rows
template<typename T, int C, int DK, bool QUERIES> struct WalkLayout
{
    static constexpr int NP = planesOf<T>;
    static constexpr uint32_t keys = 0, queries = keys + NP * C * DK, correction = queries + (QUERIES ? NP * C * DK : 0), score = correction + 3 * Triangle<C>::elements,
        table = score + (QUERIES ? 3 * Triangle<C>::elements : 0), bytes = table * 2 + C * 16;
};
constexpr int WALK_THREADS = 256;
// What the next chunk needs, on its way to LDS
template<typename T, int C, int DK, bool QUERIES> struct WalkStage
{
    typedef WalkLayout<T, C, DK, QUERIES> L;
    static constexpr int EACH = C * DK / 8 / WALK_THREADS, SQUARES = Triangle<C>::items / WALK_THREADS;
    Eight<T> keys[EACH], queries[QUERIES ? EACH : 1];
    f32x4 corrections[SQUARES], scores[QUERIES ? SQUARES : 1], rows;

    static constexpr uint32_t STEP = WALK_THREADS * 8 / DK;         // rows between a thread's units
    __device__ static uint32_t rowOf(int i) { return threadIdx.x / (DK / 8) + i * STEP; }
    __device__ static uint32_t column() { return threadIdx.x % (DK / 8) * 8; }
    // Units that are not there are asked for at another place, and become zero in store(): no branch a unit, with which the compiler would wait for each
    __device__ void requestKeys(const DeltaArgs &a, const Place &p, uint32_t keyHead, uint32_t first, uint32_t count)
    {
        const T *const key = rowsOf<const T>(a.k, a.chunks, p) + (uint64_t)first * a.k.rowStride + keyHead * a.keys, *const query = rowsOf<const T>(a.q, a.chunks, p) + (uint64_t)first * a.q.rowStride + keyHead * a.keys;
        if(a.wide && count == C) {
            // (an offset of 32 bits a lane, the rest is the scalar unit's)
            const uint32_t at0 = column() < a.keys ? column() : 0, keyOffset = rowOf(0) * (uint32_t)a.k.rowStride + at0, queryOffset = rowOf(0) * (uint32_t)a.q.rowStride + at0;
            #pragma unroll
            for(int i = 0; i < EACH; i++) {
                keys[i] = *(const Eight<T>*)((key + i * STEP * a.k.rowStride) + keyOffset);
                if(QUERIES) { queries[i] = *(const Eight<T>*)((query + i * STEP * a.q.rowStride) + queryOffset); }
            }
        }
        else {
            const uint32_t valid = column() < a.keys ? min(8u, a.keys - column()) : 0, at0 = valid ? column() : 0;
            #pragma unroll
            for(int i = 0; i < EACH; i++) {
                const uint64_t row = min(rowOf(i), count - 1);
                keys[i] = a.wide ? *(const Eight<T>*)(key + row * a.k.rowStride + at0) : loadEight(key + row * a.k.rowStride + at0, valid);
                if(QUERIES) { queries[i] = a.wide ? *(const Eight<T>*)(query + row * a.q.rowStride + at0) : loadEight(query + row * a.q.rowStride + at0, valid); }
            }
        }
    }
    __device__ void requestSquares(const DeltaArgs &a, uint64_t at)
    {
        #pragma unroll
        for(int i = 0; i < SQUARES; i++) {
            const uint32_t item = threadIdx.x + i * WALK_THREADS, offset = Triangle<C>::row(item) * C + Triangle<C>::column(item);
            corrections[i] = *(const f32x4*)(a.correction + at * C * C + offset);
            if(QUERIES) { scores[i] = *(const f32x4*)(a.score + at * C * C + offset); }
        }
        if(threadIdx.x < C) { rows = ((const f32x4*)((const RowTable<C>*)a.rows + at))[threadIdx.x]; }
    }
    __device__ static void storeSquare(uint16_t *to, uint32_t item, const f32x4 &x)
    {
        const float f[4] = {x[0], x[1], x[2], x[3]};
        uint2 words[3];
        splitFour<3, (planesOf<T> > 1)>(f, words);
        const uint32_t column = Triangle<C>::column(item);
        to += Triangle<C>::at(Triangle<C>::row(item), column / 8) + column % 8;
        #pragma unroll
        for(int k = 0; k < 3; k++) { *(uint2*)(to + k * Triangle<C>::elements) = words[k]; }
    }
    __device__ void store(const DeltaArgs &a, uint16_t *planes, uint32_t count)
    {
        if(count < C || a.keys <= DK - 8) {
            #pragma unroll
            for(int i = 0; i < EACH; i++) {
                if(rowOf(i) < count && column() < a.keys) { continue; }
                keys[i] = Eight<T>{};
                if(QUERIES) { queries[i] = Eight<T>{}; }
            }
        }
        #pragma unroll
        for(int i = 0; i < EACH; i++) {
            const uint32_t to = unitAt<DK>(rowOf(i), column() / 8);
            storeUnit(planes + L::keys + to, C * DK, keys[i]);
            if(QUERIES) { storeUnit(planes + L::queries + to, C * DK, queries[i]); }
        }
        #pragma unroll
        for(int i = 0; i < SQUARES; i++) {
            storeSquare(planes + L::correction, threadIdx.x + i * WALK_THREADS, corrections[i]);
            if(QUERIES) { storeSquare(planes + L::score, threadIdx.x + i * WALK_THREADS, scores[i]); }
        }
        if(threadIdx.x < C) { ((f32x4*)(planes + L::table))[threadIdx.x] = rows; }
    }
};
// (What a lane's place makes of them is worked out anew for every product: kept over the walk, as the compiler would have it, it costs registers that there are not.)
// Operands of a walk.  Tile t of a result has rows in the order of rowIn(): of keys (or queries, of the chunk's rows), times what is summed over keys 32 s ..; of a triangle, summed over
// rows 32 s ..; of their transposes, summed over the chunk's rows 32 s ..
template<typename T, int C, int DK, bool ANEW = true> struct WalkOperands
{
    static constexpr int NP = planesOf<T>;
    uint32_t n16, g;
    __device__ WalkOperands(uint32_t lane) { if(ANEW) { asm volatile("" : "+v"(lane)); } n16 = lane & 15; g = lane >> 4; }
    __device__ Planes<NP> rows(const uint16_t *from, int t, int s) const { return fetch<NP>(from + unitAt<DK>(rowIn(t, n16), 4 * s + g), C * DK); }
    __device__ Planes<NP> columns(const uint16_t *from, int t, int s) const
    {
        const uint32_t row = 32 * s + 8 * g + n16 / 4, unit = 4 * (t / 2) + n16 % 4, half = 4 * (t % 2);
        return fetchColumn<NP>(from + unitAt<DK>(row, unit) + half, from + unitAt<DK>(row + 4, unit) + half, C * DK);
    }
    __device__ Planes<3> triangle(const uint16_t *from, int t, int s) const { return fetch<3>(from + Triangle<C>::at(rowIn(t, n16), 4 * s + g), Triangle<C>::elements); }
    __device__ Planes<3> triangleColumns(const uint16_t *from, int t, int s) const
    {
        const uint32_t row = 32 * s + 8 * g + n16 / 4, unit = 4 * (t / 2) + n16 % 4, half = 4 * (t % 2);
        return fetchColumn<3>(from + Triangle<C>::at(row, unit) + half, from + Triangle<C>::at(row + 4, unit) + half, Triangle<C>::elements);
    }
};

// The first row of a column from which nothing is finite; rows of the chunk, if all are
template<int C> __device__ inline uint32_t firstBad(const f32x4 (&x)[C / 16], uint32_t g)
{
    uint32_t first = C;
    #pragma unroll
    for(int t = C / 16 - 1; t >= 0; t--) {
        #pragma unroll
        for(int r = 3; r >= 0; r--) { if(!finite(x[t][r])) { first = min(first, rowIn(t, r) + 8 * g); } }
    }
    first = min(first, (uint32_t)__shfl_xor((int)first, 16));
    return min(first, (uint32_t)__shfl_xor((int)first, 32));
}

// Rows of values at a lane's column, in the order of a result: row 4 g + r of tile t.  What differs between lanes is an offset of 32 bits (strides are
// below 2^25 here), the rest is the scalar unit's.  Behind `count` rows, or the last column: zero.
template<typename T, int TILES> struct Result { T v[TILES][4]; };
template<typename T, int TILES> __device__ inline Result<T, TILES> requestResult(const T *rows, uint64_t stride, uint32_t g, uint32_t column, bool inside, uint32_t count)
{
    Result<T, TILES> x;
    const uint32_t offset = 8 * g * (uint32_t)stride + (inside ? column : 0);
    if(count >= 16 * TILES) {       // (all there: without a branch a row; columns behind the last read the first)
        #pragma unroll
        for(int t = 0; t < TILES; t++) {
            #pragma unroll
            for(int r = 0; r < 4; r++) { x.v[t][r] = (rows + rowIn(t, r) * stride)[offset]; }
        }
        return x;
    }
    #pragma unroll
    for(int t = 0; t < TILES; t++) {
        #pragma unroll
        for(int r = 0; r < 4; r++) {
            x.v[t][r] = (T)0.0f;
            if((int)rowIn(t, r) < (int)(count - 8 * g)) { x.v[t][r] = (rows + rowIn(t, r) * stride)[offset]; }
        }
    }
    return x;
}
template<typename T, int TILES> __device__ inline void takeResult(const Result<T, TILES> &from, bool inside, f32x4 (&x)[TILES])
{
    #pragma unroll
    for(int t = 0; t < TILES; t++) {
        #pragma unroll
        for(int r = 0; r < 4; r++) { x[t][r] = inside ? widen(from.v[t][r]) : 0.0f; }
    }
}
template<typename T, int C> __device__ inline void loadResult(const T *rows, uint64_t stride, uint32_t g, uint32_t column, bool inside, uint32_t count, f32x4 (&x)[C / 16])
{
    takeResult(requestResult<T, C / 16>(rows, stride, g, column, inside, count), inside, x);
}
template<typename T, int C> __device__ inline void storeResult(T *rows, uint64_t stride, uint32_t g, uint32_t column, bool inside, uint32_t count, const f32x4 (&x)[C / 16])
{
    const uint32_t offset = 8 * g * (uint32_t)stride + column;
    if(!inside) { return; }
    if(count >= C) {
        #pragma unroll
        for(int t = 0; t < C / 16; t++) {
            #pragma unroll
            for(int r = 0; r < 4; r++) { (rows + rowIn(t, r) * stride)[offset] = narrow<T>(x[t][r]); }
        }
        return;
    }
    #pragma unroll
    for(int t = 0; t < C / 16; t++) {
        #pragma unroll
        for(int r = 0; r < 4; r++) { if((int)rowIn(t, r) < (int)(count - 8 * g)) { (rows + rowIn(t, r) * stride)[offset] = narrow<T>(x[t][r]); } }
    }
}

// Which head, columns and segment a work-group of a walk has.  Those of one segment and key head read the same keys, queries and squares: they go to one of the eight parts of the chip with an L2 of
// its own, to which the hardware hands work-groups in turn.
struct WalkPlace { uint32_t segment, head, block; bool valid; };
__device__ inline WalkPlace walkPlace(const DeltaArgs &a, uint32_t blocks)
{
    const uint32_t each = a.group * blocks, slot = blockIdx.x / 8, outer = slot / each * 8 + blockIdx.x % 8, inner = slot % each, segment = outer / a.keyHeads;
    return WalkPlace{segment, (outer - segment * a.keyHeads) * a.group + inner / blocks, inner % blocks, segment < a.segmentNumbers};
}

// A work-group walks a sequence (or a segment of it) of one head with 16 columns of the state a wavefront.  What bounds it: a wavefront's five products of a chunk wait for each other (14,000 cycles alone on a SIMD,
// of which matrix instructions 3,500), and of as many vector instructions as take the same time (5.4 to 5.9 for each matrix instruction: most of them cut floats into planes, the same squares in every work-group of a head),
// so that two work-groups share a compute unit.  One prompt of 64 chunks x 32 heads of 128 x 128 in bf16, in 8 segments: what they do to a state 92 us, outputs 79 (all 256 registers, 19 spilled, 65 scalars in lanes).
template<typename T, int C, int DK, int MODE, bool FOLDED> __device__ __forceinline__ void walkForwards(const DeltaArgs &a)
{
    constexpr bool OUTPUTS = MODE == WALK_OUTPUTS;
    typedef WalkLayout<T, C, DK, OUTPUTS> L;
    constexpr int NP = planesOf<T>, TILES = C / 16, STATE = DK / 16, WAVES = WALK_THREADS / 64;
    extern __shared__ __align__(16) char lds[];
    uint16_t *const planes = (uint16_t*)lds;
    const RowFactors<C> table{(float*)(planes + L::table)};
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4;
    const WalkPlace mine = walkPlace(a, a.columnBlocks + (MODE == WALK_SUMMARY ? a.moveBlocks : 0));
    const uint32_t block = mine.block, head = mine.head, segment = mine.segment, keyHead = head / a.group;
    Place p;
    if(!mine.valid || !locate(a.segments, segment, p)) { return; }
    const uint32_t begin = p.index * a.segments.chunk, end = min(p.length, begin + a.segments.chunk);
    // (what is behind the last segment nobody asks)
    if(MODE == WALK_SUMMARY && end == p.length) { return; }
    const bool move = MODE == WALK_SUMMARY && block >= a.columnBlocks;
    const uint32_t firstColumn = ((move ? block - a.columnBlocks : block) * WAVES + wave) * 16, column = firstColumn + n16;
    const bool active = firstColumn < (move ? (uint32_t)DK : OUTPUTS ? a.values : a.padded), inside = !move && column < a.values;
    const uint32_t chunks = end > begin ? (end - begin + C - 1) / C : 0;
    const uint64_t firstNumber = firstChunk(a.chunks, p.sequence) + begin / C, segmentAt = (uint64_t)segment * a.heads + head;

    f32x4 state[STATE];
    #pragma unroll
    for(int t = 0; t < STATE; t++) { state[t] = f32x4{0, 0, 0, 0}; }
    if(MODE == WALK_SUMMARY) {
        #pragma unroll
        for(int t = 0; t < STATE; t++) {
            #pragma unroll
            for(int r = 0; r < 4; r++) { if(move && (int)rowIn(t, r) == (int)(column - 8 * g)) { state[t][r] = 1.0f; } }
        }
    }
    else if(a.segmentStates) {
        if(active) { loadResult<float, DK>(a.segmentStates + segmentAt * DK * a.padded, a.padded, g, column, true, DK, state); }
    }
    else if(a.initialState) { loadResult<float, DK>(a.initialState + ((uint64_t)p.state * a.heads + head) * a.keys * a.values, a.values, g, column, inside, a.keys, state); }

    WalkStage<T, C, DK, OUTPUTS> stage;
    if(chunks) { stage.requestKeys(a, p, keyHead, begin, min((uint32_t)C, end - begin)); stage.requestSquares(a, firstNumber * a.heads + head); }
    for(uint32_t n = 0; n < chunks; n++) {
        const uint32_t first = begin + n * C, count = min((uint32_t)C, end - first);
        const uint64_t at = (firstNumber + n) * a.heads + head;
        const ChunkTable chunk = a.table[at];
        Result<T, TILES> values;
        if(active) { values = requestResult<T, TILES>(rowsOf<const T>(a.v, a.chunks, p) + (uint64_t)first * a.v.rowStride + head * a.values, a.v.rowStride, g, column, inside, move ? 0 : count); }
        __syncthreads();
        stage.store(a, planes, count);
        __syncthreads();
        const auto requestKeys = [&] { if(n + 1 < chunks) { stage.requestKeys(a, p, keyHead, first + C, min((uint32_t)C, end - first - C)); } };
        const auto requestSquares = [&] { if(n + 1 < chunks) { stage.requestSquares(a, at + a.heads); } };
        if(!active) { requestKeys(); requestSquares(); continue; }

        // r = v - G k^ S, and the part of the outputs that the state in front has: x's first tiles and the others
        constexpr int ROWS = OUTPUTS ? 2 * TILES : TILES;
        f32x4 w[TILES], x[ROWS];
        if(MODE == WALK_KEEP) { storeResult<float, DK>(a.states + at * DK * a.padded, a.padded, g, column, true, DK, state); }
        #pragma unroll
        for(int t = 0; t < ROWS; t++) { x[t] = f32x4{0, 0, 0, 0}; }
        #pragma unroll
        for(int s = 0; s < DK / 32; s++) {
            inTurn();
            const WalkOperands<T, C, DK, OUTPUTS> operand(lane);
            Planes<NP> rows[ROWS];
            #pragma unroll
            for(int t = 0; t < ROWS; t++) { rows[t] = operand.rows(planes + (t < TILES ? L::keys : L::queries), t % TILES, s); }
            multiplyAll(rows, split<3, (NP > 1)>(state[2 * s], state[2 * s + 1]), x);
        }
        inTurn();
        takeResult(values, inside, w);
        float notFinite = 0.0f;
        #pragma unroll
        for(int t = 0; t < TILES; t++) {
            const f32x4 keyState = table.keyState(rowIn(t, 4 * g));
            if(OUTPUTS) { x[TILES + t] *= table.queryState(rowIn(t, 4 * g)); }
            #pragma unroll
            for(int r = 0; r < 4; r++) {
                w[t][r] = __builtin_fmaf(-keyState[r], x[t][r], w[t][r]);
                notFinite = __builtin_fmaf(w[t][r], 0.0f, notFinite);
            }
        }
        uint32_t bad = chunk.bad;
        if(__builtin_expect(__ballot(notFinite != 0.0f) != 0 || bad < C, 0)) {
            // (what is not finite must not reach rows before it: 0 times it is not 0)
            bad = min(bad, firstBad<C>(w, g));
            #pragma unroll
            for(int t = 0; t < TILES; t++) {
                #pragma unroll
                for(int r = 0; r < 4; r++) { if((int)rowIn(t, r) >= (int)(bad - 8 * g)) { w[t][r] = 0.0f; } }
            }
        }
        // w = r - N beta r and out += P beta w; tiles above the diagonal are zero
        {
            Planes<3> b[TILES / 2];
            #pragma unroll
            for(int s = 0; s < TILES / 2; s++) {
                f32x4 y[2] = {w[2 * s], w[2 * s + 1]};
                if(!FOLDED) {
                    #pragma unroll
                    for(int h = 0; h < 2; h++) { y[h] *= table.beta(rowIn(2 * s + h, 4 * g)); }
                }
                b[s] = split<3>(y[0], y[1]);
            }
            #pragma unroll
            for(int s = 0; s < TILES / 2; s++) {
                #pragma unroll
                for(int t = 2 * s; t < TILES; t += 2) {
                    inTurn();
                    const WalkOperands<T, C, DK, OUTPUTS> operand(lane);
                    constexpr int SQUARES = OUTPUTS ? 4 : 2;
                    Planes<3> rows[SQUARES];
                    f32x4 sum[SQUARES];
                    #pragma unroll
                    for(int i = 0; i < SQUARES; i++) {
                        rows[i] = operand.triangle(planes + (i < 2 ? L::correction : L::score), t + i % 2, s);
                        sum[i] = i < 2 ? w[t + i] : x[TILES + t + i % 2];
                    }
                    multiplyAll(rows, b[s], sum);
                    #pragma unroll
                    for(int i = 0; i < SQUARES; i++) { (i < 2 ? w[t + i] : x[ROWS - TILES + t + i % 2]) = sum[i]; }
                }
            }
        }
        inTurn();
        if(__builtin_expect(bad < C, 0)) {
            const float no = __builtin_nanf("");
            #pragma unroll
            for(int t = 0; t < TILES; t++) {
                #pragma unroll
                for(int r = 0; r < 4; r++) { if((int)rowIn(t, r) >= (int)(bad - 8 * g)) { w[t][r] = x[ROWS - TILES + t][r] = no; } }
            }
        }
        if(MODE == WALK_KEEP) { storeResult<float, C>(a.errors + at * C * a.padded, a.padded, g, column, true, C, w); }
        if(OUTPUTS) { storeResult<T, C>(rowsOf<T>(a.out, a.chunks, p) + (uint64_t)first * a.out.rowStride + head * a.values, a.out.rowStride, g, column, inside, count, *(const f32x4 (*)[TILES])(x + ROWS - TILES)); }
        // the state behind the chunk; meanwhile the next one's operands are on their way (asked for before this they cost registers that there are not)
        requestKeys();
        #pragma unroll
        for(int t = 0; t < STATE; t++) { state[t] *= chunk.decay; }
        #pragma unroll
        for(int s = 0; s < TILES / 2; s++) {
            inTurn();
            f32x4 left[2];
            #pragma unroll
            for(int h = 0; h < 2; h++) { left[h] = w[2 * s + h] * table.beta(rowIn(2 * s + h, 4 * g)) * table.keyEnd(rowIn(2 * s + h, 4 * g)); }
            const WalkOperands<T, C, DK, OUTPUTS> operand(lane);
            Planes<NP> columns[STATE];
            #pragma unroll
            for(int t = 0; t < STATE; t++) { columns[t] = operand.columns(planes + L::keys, t, s); }
            multiplyAll(columns, split<3, (NP > 1)>(left[0], left[1]), state);
        }
        inTurn();
        requestSquares();
        if(__builtin_expect(bad < C, 0)) {
            const float no = __builtin_nanf("");
            #pragma unroll
            for(int t = 0; t < STATE; t++) { state[t] = f32x4{no, no, no, no}; }
        }
    }
    if(!active) { return; }
    if(MODE == WALK_SUMMARY) {
        float *const to = move ? a.segmentMoves + segmentAt * DK * DK : a.segmentStates + segmentAt * DK * a.padded;
        storeResult<float, DK>(to, move ? DK : a.padded, g, column, true, DK, state);
    }
    if(MODE == WALK_OUTPUTS && a.finalState && end == p.length) {
        storeResult<float, DK>(a.finalState + ((uint64_t)p.state * a.heads + head) * a.keys * a.values, a.values, g, column, inside, a.keys, state);
    }
}

// (what segments of two planes do to a state fits the registers of three work-groups a compute unit, with two registers less than the compiler takes by itself: 33 sequences of 8011 rows in fp16 195 us, with two 216)
template<typename T, int C, int DK, int MODE, bool FOLDED>
__global__ __launch_bounds__(WALK_THREADS, MODE == WALK_SUMMARY && planesOf<T> == 2 ? 3 : 2)
void deltaStateKernel(DeltaArgs a) { walkForwards<T, C, DK, MODE, FOLDED>(a); }

// From what each segment does: the state in front of each, in place of its own share: S = move S + own in fp32.  A work-group has 16 columns; its four wavefronts share the rows of
// `move`, and hand each other what they found through LDS.  32 heads of 128 keys, 8 segments: 38 us with one share in registers, tiles of a head all over the chip; 27 so.
template<int DK>
__global__ __launch_bounds__(256, 1)
void deltaJoinKernel(DeltaArgs a)
{
    constexpr int STATE = DK / 16, MINE = STATE / 4;
    __shared__ f32x4 found[STATE][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4, tiles = a.padded / 16;
    // (those that read one `move` on one part of the chip, as in walkPlace)
    const uint32_t slot = blockIdx.x / 8, tile = slot % tiles, outer = slot / tiles * 8 + blockIdx.x % 8, sequence = outer / a.heads, head = outer - sequence * a.heads, column = tile * 16 + n16;
    Place p;
    if(sequence >= a.segments.count || !describe(a.segments, sequence, p)) { return; }
    f32x4 state[STATE];
    #pragma unroll
    for(int t = 0; t < STATE; t++) { state[t] = f32x4{0, 0, 0, 0}; }
    if(a.initialState) { loadResult<float, DK>(a.initialState + ((uint64_t)p.state * a.heads + head) * a.keys * a.values, a.values, g, column, column < a.values, a.keys, state); }
    const uint32_t segments = max(1u, (p.length + a.segments.chunk - 1) / a.segments.chunk);
    const uint64_t first = firstChunk(a.segments, sequence) * a.heads + head;
    // (this wavefront's tiles of `move` and of a segment's own share; those of the next segment are on their way while one is joined)
    struct Share { f32x4 move[MINE][STATE], own[MINE]; } shares[2];
    const auto request = [&](uint32_t n, Share &to) {
        const uint64_t at = first + (uint64_t)n * a.heads;
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            const uint32_t rows = wave * MINE + m;
            #pragma unroll
            for(int r = 0; r < 4; r++) { to.own[m][r] = a.segmentStates[at * DK * a.padded + rowIn(rows, 4 * g + r) * a.padded + column]; }
            #pragma unroll
            for(int t = 0; t < STATE; t++) { to.move[m][t] = *(const f32x4*)(a.segmentMoves + at * DK * DK + rowIn(rows, n16) * DK + rowIn(t, 4 * g)); }
        }
    };
    const auto join = [&](uint32_t n, const Share &share, Share &ahead) {
        // (behind the last segment but one nobody asks)
        if(n + 2 < segments) { request(n + 1, ahead); }
        f32x4 next[MINE];
        if(n + 1 < segments) {
            #pragma unroll
            for(int m = 0; m < MINE; m++) { next[m] = share.own[m]; }
            #pragma unroll
            for(int t = 0; t < STATE; t++) {
                #pragma unroll
                for(int m = 0; m < MINE; m++) { next[m] = multiply(share.move[m][t], state[t], next[m]); }
            }
        }
        // (own shares have been read: the state goes in their place)
        float *const to = a.segmentStates + (first + (uint64_t)n * a.heads) * DK * a.padded + column;
        #pragma unroll
        for(int t = 0; t < STATE; t++) {
            if((uint32_t)t / MINE != wave) { continue; }
            #pragma unroll
            for(int r = 0; r < 4; r++) { to[rowIn(t, 4 * g + r) * a.padded] = state[t][r]; }
        }
        if(n + 1 == segments) { return; }
        __syncthreads();
        #pragma unroll
        for(int m = 0; m < MINE; m++) { found[wave * MINE + m][lane] = next[m]; }
        __syncthreads();
        #pragma unroll
        for(int t = 0; t < STATE; t++) { state[t] = found[t][lane]; }
    };
    if(segments > 1) { request(0, shares[0]); }
    for(uint32_t n = 0; n < segments; n += 2) {
        join(n, shares[0], shares[1]);
        if(n + 1 < segments) { join(n + 1, shares[1], shares[0]); }
    }
}

// ---- gradients: the same walk from the other end
// dR = (I - beta N')' of dU, row by row what the loss says of u through everything behind it; v's gradient is beta dR.
struct DeltaGradientArgs
{
    gennmi_rows_t out, q, k, v, g, beta;
    const float *finalState;
    float *initialState;
    float *states, *errors;         // the gradient of the state behind each chunk [DK][padded], dR [C][padded]
    float *shared;                  // where heads share keys: each one's gradients of unit queries and keys, [2][C][DK]
};
template<typename T, int C, int DK, bool ALONE> __device__ __forceinline__ void walkBackwards(const DeltaArgs &a, const DeltaGradientArgs &d)
{
    typedef WalkLayout<T, C, DK, true> L;
    constexpr int NP = planesOf<T>, TILES = C / 16, STATE = DK / 16, WAVES = WALK_THREADS / 64;
    extern __shared__ __align__(16) char lds[];
    uint16_t *const planes = (uint16_t*)lds;
    const RowFactors<C> table{(float*)(planes + L::table)};
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n16 = lane & 15, g = lane >> 4;
    const WalkPlace mine = walkPlace(a, a.columnBlocks);
    const uint32_t block = mine.block, head = mine.head, segment = mine.segment, keyHead = head / a.group;
    Place p;
    if(!mine.valid || !locate(a.segments, segment, p)) { return; }
    const uint32_t begin = p.index * a.segments.chunk, end = min(p.length, begin + a.segments.chunk);
    const uint32_t column = (block * WAVES + wave) * 16 + n16;
    const bool active = (block * WAVES + wave) * 16 < a.padded, inside = column < a.values;
    const uint32_t chunks = end > begin ? (end - begin + C - 1) / C : 0;
    const uint64_t firstNumber = firstChunk(a.chunks, p.sequence) + begin / C;

    f32x4 state[STATE];
    #pragma unroll
    for(int t = 0; t < STATE; t++) { state[t] = f32x4{0, 0, 0, 0}; }
    if(d.finalState) { loadResult<float, DK>(d.finalState + ((uint64_t)p.sequence * a.heads + head) * a.keys * a.values, a.values, g, column, inside, a.keys, state); }
    // two tiles of a triangle's transpose
    const auto timesTriangle = [&](uint32_t from, int t, int s, const auto &b, f32x4 (&to)[TILES]) {
        inTurn();
        const WalkOperands<T, C, DK, !ALONE> operand(lane);
        const Planes<3> rows[2] = {operand.triangleColumns(planes + from, t, s), operand.triangleColumns(planes + from, t + 1, s)};
        f32x4 sum[2] = {to[t], to[t + 1]};
        multiplyAll(rows, b, sum);
        to[t] = sum[0];
        to[t + 1] = sum[1];
    };
    WalkStage<T, C, DK, true> stage;
    if(chunks) { const uint32_t last = begin + (chunks - 1) * C; stage.requestKeys(a, p, keyHead, last, end - last); stage.requestSquares(a, (firstNumber + chunks - 1) * a.heads + head); }
    for(uint32_t left = chunks; left > 0; left--) {
        const uint32_t n = left - 1, first = begin + n * C, count = min((uint32_t)C, end - first);
        const uint64_t at = (firstNumber + n) * a.heads + head;
        const float decay = a.table[at].decay;
        Result<T, TILES> douts;
        if(active) { douts = requestResult<T, TILES>(rowsOf<const T>(d.out, a.chunks, p) + (uint64_t)first * d.out.rowStride + head * a.values, d.out.rowStride, g, column, inside, count); }
        __syncthreads();
        stage.store(a, planes, count);
        __syncthreads();
        const auto requestKeys = [&] { if(n > 0) { stage.requestKeys(a, p, keyHead, first - C, C); } };
        const auto requestSquares = [&] { if(n > 0) { stage.requestSquares(a, at - a.heads); } };
        if(!active) { requestKeys(); requestSquares(); continue; }

        f32x4 dout[TILES], du[TILES];
        #pragma unroll
        for(int t = 0; t < TILES; t++) { du[t] = f32x4{0, 0, 0, 0}; }
        storeResult<float, DK>(d.states + at * DK * a.padded, a.padded, g, column, true, DK, state);
        // dU = D[last] k^ dS + P' dout
        #pragma unroll
        for(int s = 0; s < DK / 32; s++) {
            inTurn();
            const WalkOperands<T, C, DK, !ALONE> operand(lane);
            Planes<NP> rows[TILES];
            #pragma unroll
            for(int t = 0; t < TILES; t++) { rows[t] = operand.rows(planes + L::keys, t, s); }
            multiplyAll(rows, split<3, (NP > 1)>(state[2 * s], state[2 * s + 1]), du);
        }
        inTurn();
        takeResult(douts, inside, dout);
        #pragma unroll
        for(int t = 0; t < TILES; t++) {
            du[t] *= table.keyEnd(rowIn(t, 4 * g));
        }
        #pragma unroll
        for(int s = 0; s < TILES / 2; s++) {
            inTurn();
            const Planes<NP> b = split<NP>(dout[2 * s], dout[2 * s + 1]);
            #pragma unroll
            for(int t = 0; t < 2 * s + 2; t += 2) { timesTriangle(L::score, t, s, b, du); }
        }
        // dR = dU - N' beta dU
        {
            Planes<3> b[TILES / 2];
            #pragma unroll
            for(int s = 0; s < TILES / 2; s++) {
                inTurn();
                f32x4 y[2];
                #pragma unroll
                for(int h = 0; h < 2; h++) { y[h] = du[2 * s + h] * table.beta(rowIn(2 * s + h, 4 * g)); }
                b[s] = split<3>(y[0], y[1]);
            }
            #pragma unroll
            for(int s = 0; s < TILES / 2; s++) {
                inTurn();
                #pragma unroll
                for(int t = 0; t < 2 * s + 2; t += 2) { timesTriangle(L::correction, t, s, b[s], du); }
            }
        }
        storeResult<float, C>(d.errors + at * C * a.padded, a.padded, g, column, true, C, du);
        requestKeys();
        // dS in front of the chunk = G[last] dS + (scale G q^)' dout - (G k^)' (beta dR)
        #pragma unroll
        for(int t = 0; t < STATE; t++) { state[t] *= decay; }
        #pragma unroll
        for(int s = 0; s < TILES / 2; s++) {
            inTurn();
            f32x4 x[2], y[2];
            #pragma unroll
            for(int h = 0; h < 2; h++) {
                const uint32_t row = rowIn(2 * s + h, 4 * g);
                x[h] = dout[2 * s + h] * table.queryState(row);
                du[2 * s + h] *= table.beta(row);
                y[h] = -table.keyState(row) * du[2 * s + h];
            }
            #pragma unroll
            for(int which = 0; which < 2; which++) {
                inTurn();
                const WalkOperands<T, C, DK, !ALONE> operand(lane);
                Planes<NP> columns[STATE];
                #pragma unroll
                for(int t = 0; t < STATE; t++) { columns[t] = operand.columns(planes + (which ? L::keys : L::queries), t, s); }
                multiplyAll(columns, which ? split<3, (NP > 1)>(y[0], y[1]) : split<3, (NP > 1)>(x[0], x[1]), state);
            }
        }
        inTurn();
        requestSquares();
        if(d.v.data) { storeResult<T, C>(rowsOf<T>(d.v, a.chunks, p) + (uint64_t)first * d.v.rowStride + head * a.values, d.v.rowStride, g, column, inside, count, du); }
    }
    if(d.initialState && active && begin == 0) { storeResult<float, DK>(d.initialState + ((uint64_t)p.sequence * a.heads + head) * a.keys * a.values, a.values, g, column, inside, a.keys, state); }
}

// Neither walk of a gradient needs the other: both at once, so that a compute unit has a work-group of each, and one works where the other waits.  8 sequences of 2048 rows x 16 heads of 128 x 128 in bf16:
// one behind the other 530 us, both at once 393 (1.4 GB moved, 3.6 TB/s: memory counts as much as the wait; over 500 scalars of the two walks' descriptors are kept in lanes: 7.9 vector instructions a matrix instruction);
// 3 of 301 rows x 3 heads of 33 x 47 in fp32: 75, 48.  ALONE: not more work-groups in all than compute units; each may have all registers of one.
template<typename T, int C, int DK, bool ALONE>
__global__ __launch_bounds__(WALK_THREADS, ALONE ? 1 : 2)
void deltaWalksKernel(DeltaArgs a, DeltaGradientArgs d)
{
    if(blockIdx.y == 0) { walkBackwards<T, C, DK, ALONE>(a, d); }
    else { walkForwards<T, C, DK, WALK_KEEP, false>(a); }
}

// ---- gradients of a chunk, once the state in front of it, w, the gradient of the state behind it and dR are known
//   dq^ = scale G (dout S') + sum_j dQK[i][j] k^[j],   dQK[i][j] = scale D[i][j] dout[i].u[j] for i >= j
//   dk^ = beta (D[last] w dS' - G dR S') + sum_i dQK[i][j] q^[i] + sum_j (dKK + dKK')[i][j] k^[j],   dKK[i][j] = -D[i][j] beta[i] beta[j] dR[i].w[j] for i > j
//   dbeta[i] = w[i].dR[i]
// and g[t]'s is what of the loss carries the decay of row t, term by term, so that it vanishes with that decay and no two large numbers cancel:
//   dg[t] = sum_{i>=t} (q^[i].scale G dout S' - k^[i].beta G dR S')[i] + sum_{i>=t>j} (dQK[i][j] q^[i].k^[j] + dKK[i][j] k^[i].k^[j])
//           + sum_{j<t} k^[j].beta D[last] w dS'[j] + G[last] S.dS
// A work-group has a chunk and a head.  Products are summed over the values, 32 at a time, with what multiplies S and dS
// in LDS; a wavefront has the results' columns of a quarter of the keys, S' and dS' straight from memory.  What bounds it is waiting, for memory and at barriers: two work-groups
// of four wavefronts fit a compute unit and fill each other's pauses.  256 chunks x 16 heads of 128 x 128 in bf16: 447 us, some 1.15 GB (2.6 TB/s).  Sums over keys and within a chunk's square are in fp32 (each term of a gate's gradient carries its decay, so nothing is lost with it), over a chunk's rows in 64 bits.  Where heads share keys, what each finds for them is left for deltaSharedKernel to add up.
template<typename T, int C, int DK> struct GradientLayout
{
    static constexpr int NP = planesOf<T>;
    static constexpr uint32_t keys = 0, queries = keys + NP * C * DK, stage = queries + NP * C * DK, staged = (NP + 6) * C * 32, square = 3 * C * C,
        floats = stage + (staged > square ? staged : square), bytes = floats * 2 + C * 8 + C * 4 * (5 + 2 * 4) + 4 * 256 + 32;
    static_assert((staged > square ? staged : square) * 2 >= 4 * (C * (C + 1) + 256), "");          // (the crossings and their columns' sums lie there as well)
};

template<typename T, int C, int DK>
__global__ __launch_bounds__(256, 2)
void deltaGradientKernel(DeltaArgs a, DeltaGradientArgs d)
{
    typedef GradientLayout<T, C, DK> L;
    constexpr int NP = planesOf<T>, TILES = C / 16, MINE = DK / 64, SQUARES = C == 64 ? 4 : 1, UNITS = C * DK / 8, VP = C * 32, ITEMS = C / 32;
    extern __shared__ __align__(16) char lds[];
    uint16_t *const planes = (uint16_t*)lds, *const stage = planes + L::stage;
    uint16_t *const doutPlanes = stage, *const dRPlanes = stage + NP * VP, *const wPlanes = dRPlanes + 3 * VP;
    double *const sums = (double*)(planes + L::floats);
    float *const since = (float*)(sums + C), *const until = since + C, *const beta = until + C, *const keyUnit = beta + C, *const queryUnit = keyUnit + C;
    float *const queryDots = queryUnit + C, *const keyDots = queryDots + 4 * C, *const crossingDots = keyDots + 4 * C, *const ends = crossingDots + 256;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n16 = lane & 15, g = lane >> 4;
    const uint32_t number = blockIdx.x / a.heads, head = blockIdx.x - number * a.heads, keyHead = head / a.group;
    const uint64_t at = (uint64_t)number * a.heads + head;
    Place p;
    if(!locate(a.chunks, number, p)) { return; }
    const uint32_t begin = p.index * C, count = min((uint32_t)C, p.length - min(p.length, begin));
    if(!count) { return; }

    // this wavefront's columns of keys; squares: of 64 rows a column of tiles a wavefront, of 32 a tile
    const auto keyOf = [&](int m) { return (wave * MINE + m) * 16 + n16; };
    const auto squareRow = [&](int q) { return C == 64 ? (uint32_t)q : wave >> 1; };
    const uint32_t squareColumn = C == 64 ? wave : wave & 1;

    // keys and queries
    Eight<T> units[2 * UNITS / 256];
    #pragma unroll
    for(int i = 0; i < 2 * UNITS / 256; i++) {
        const uint32_t item = (tid + i * 256) % UNITS, row = item / (DK / 8), column = item % (DK / 8) * 8, valid = row < count && column < a.keys ? min(8u, a.keys - column) : 0;
        const gennmi_rows_t &r = i < UNITS / 256 ? a.k : a.q;
        units[i] = loadUnit(rowAt<T>(r, a.chunks, p, valid ? begin + row : begin) + (valid ? keyHead * a.keys + column : 0), valid, a.wide);
    }
    // what multiplies S and dS: eight threads a row, four values each
    const float *const stateRows = a.states + at * DK * a.padded, *const dStateRows = d.states + at * DK * a.padded;
    typedef Pack<T, 4> Four;
    f32x4 inDR[ITEMS], inW[ITEMS];
    Four inDout[ITEMS];
    const auto rowOfItem = [&](int i) { return tid / 8 + 32 * i; };
    const uint32_t stageAt = tid % 8 * 4;
    const T *const douts = rowsOf<const T>(d.out, a.chunks, p) + (uint64_t)begin * d.out.rowStride + head * a.values;
    const auto request = [&](uint32_t v) {
        #pragma unroll
        for(int i = 0; i < ITEMS; i++) {
            inDR[i] = *(const f32x4*)(d.errors + (at * C + rowOfItem(i)) * a.padded + v + stageAt);
            inW[i] = *(const f32x4*)(a.errors + (at * C + rowOfItem(i)) * a.padded + v + stageAt);
        }
        // (rows and values that are not there: others, and nothing of them is used; no branch an access, with which the compiler would wait for each)
        if(a.wideValues) {
            const uint32_t there = v + stageAt < a.values ? v + stageAt : 0;
            #pragma unroll
            for(int i = 0; i < ITEMS; i++) {
                const uint64_t row = min(rowOfItem(i), count - 1);
                inDout[i] = *(const Four*)(douts + row * d.out.rowStride + there);
            }
        }
        else {
            #pragma unroll
            for(int i = 0; i < ITEMS; i++) {
                const uint64_t row = min(rowOfItem(i), count - 1);
                #pragma unroll
                for(int e = 0; e < 4; e++) {
                    const uint32_t there = v + stageAt + e < a.values ? v + stageAt + e : 0;
                    inDout[i].v[e] = douts[row * d.out.rowStride + there];
                }
            }
        }
    };
    #pragma unroll
    for(int i = 0; i < 2 * UNITS / 256; i++) {
        const uint32_t item = (tid + i * 256) % UNITS;
        storeUnit(planes + (i < UNITS / 256 ? L::keys : L::queries) + unitAt<DK>(item / (DK / 8), item % (DK / 8)), C * DK, units[i]);
    }
    const float decay = a.table[at].decay;
    if(tid < C) {
        const RowTable<C> &rows = ((const RowTable<C>*)a.rows)[at];
        const double sum = rows.sum[tid], last = rows.sum[C - 1];
        sums[tid] = sum;
        since[tid] = decayOver(sum);
        until[tid] = decayOver(last - sum);
        beta[tid] = rows.beta[tid];
        keyUnit[tid] = rows.keyUnit[tid];
        queryUnit[tid] = rows.queryUnit[tid];
    }
    // the keys' (or queries') values at this lane's column, four rows of a tile
    const auto valuesAt = [&](uint32_t from, uint32_t tile, int m) {
        f32x4 x = {0, 0, 0, 0};
        #pragma unroll
        for(int k = 0; k < NP; k++) {
            const uint2 w = readColumn(planes + from + k * C * DK + unitAt<DK>(tile * 16 + 4 * g + n16 / 4, 2 * (wave * MINE + m) + n16 % 4 / 2) + n16 % 2 * 4);
            x[0] += __uint_as_float(w.x << 16); x[1] += __uint_as_float(w.x & 0xffff0000u);
            x[2] += __uint_as_float(w.y << 16); x[3] += __uint_as_float(w.y & 0xffff0000u);
        }
        return x;
    };
    const auto fourRows = [&](const float *from, uint32_t tile) { return *(const f32x4*)(from + tile * 16 + 4 * g); };
    const auto sumOf16 = [](float x) { x += partner<1>(x); x += partner<2>(x); x += partner<4>(x); return x + partner<8>(x); };

    f32x4 dq[MINE][TILES], rS[MINE][TILES], dk[MINE][TILES], dqk[SQUARES], dkk[SQUARES];
    #pragma unroll
    for(int m = 0; m < MINE; m++) {
        #pragma unroll
        for(int t = 0; t < TILES; t++) { dq[m][t] = rS[m][t] = dk[m][t] = f32x4{0, 0, 0, 0}; }
    }
    #pragma unroll
    for(int q = 0; q < SQUARES; q++) { dqk[q] = dkk[q] = f32x4{0, 0, 0, 0}; }
    float stateDot = 0.0f, betaDot[ITEMS] = {};
    for(uint32_t v = 0; v < a.padded; v += 32) {
        request(v);
        f32x4 s0[MINE][2], ds[MINE][2];
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            #pragma unroll
            for(int h = 0; h < 2; h++) {
                const uint32_t offset = keyOf(m) * a.padded + v + 8 * g + 4 * h;
                s0[m][h] = *(const f32x4*)(stateRows + offset);
                ds[m][h] = *(const f32x4*)(dStateRows + offset);
            }
        }
        __syncthreads();
        #pragma unroll
        for(int i = 0; i < ITEMS; i++) {
            float dr[4], w[4], dout[4];
            #pragma unroll
            for(int e = 0; e < 4; e++) {
                const bool row = rowOfItem(i) < count, there = row && v + stageAt + e < a.values;
                dr[e] = row ? inDR[i][e] : 0.0f;
                w[e] = row ? inW[i][e] : 0.0f;
                dout[e] = there ? widen(inDout[i].v[e]) : 0.0f;
                betaDot[i] = __builtin_fmaf(w[e], dr[e], betaDot[i]);
            }
            uint2 words[3], own[NP];
            uint16_t *const to = stage + unitAt<32>(rowOfItem(i), stageAt / 8) + stageAt % 8;
            splitFour<NP>(dout, own);
            #pragma unroll
            for(int k = 0; k < NP; k++) { *(uint2*)(to + k * VP) = own[k]; }
            splitFour<3>(dr, words);
            #pragma unroll
            for(int k = 0; k < 3; k++) { *(uint2*)(to + (NP + k) * VP) = words[k]; }
            splitFour<3>(w, words);
            #pragma unroll
            for(int k = 0; k < 3; k++) { *(uint2*)(to + (NP + 3 + k) * VP) = words[k]; }
        }
        __syncthreads();
        {
            const Planes<3> other = fetch<3>(wPlanes + unitAt<32>(squareColumn * 16 + n16, g), VP);
            #pragma unroll
            for(int q = 0; q < SQUARES; q++) {
                inTurn();
                if(squareRow(q) < squareColumn) { continue; }
                const uint32_t offset = unitAt<32>(squareRow(q) * 16 + n16, g);
                dqk[q] = multiply(fetch<NP>(doutPlanes + offset, VP), other, dqk[q]);
                dkk[q] = multiply(fetch<3>(dRPlanes + offset, VP), other, dkk[q]);
            }
        }
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            inTurn();
            #pragma unroll
            for(int h = 0; h < 2; h++) {
                #pragma unroll
                for(int e = 0; e < 4; e++) { stateDot = __builtin_fmaf(s0[m][h][e], ds[m][h][e], stateDot); }
            }
            const Planes<3> state = split<3, (NP > 1)>(s0[m][0], s0[m][1]), dState = split<3, (NP > 1)>(ds[m][0], ds[m][1]);
            #pragma unroll
            for(int t = 0; t < TILES; t++) {
                inTurn();
                const uint32_t offset = unitAt<32>(t * 16 + n16, g);
                const Planes<NP> out = fetch<NP>(doutPlanes + offset, VP);
                const Planes<3> r = fetch<3>(dRPlanes + offset, VP), w = fetch<3>(wPlanes + offset, VP);
                multiplyThree(out, state, dq[m][t], r, state, rS[m][t], w, dState, dk[m][t]);
            }
        }
        inTurn();
    }
    // what the rows' factors make of them; for the gates, what each row has of the state in front and what it leaves in the state behind (where the lengths' gradients find place afterwards)
    #pragma unroll
    for(int t = 0; t < TILES; t++) {
        const f32x4 grown = fourRows(since, t), by = fourRows(beta, t), last = fourRows(until, t) * by, keyLength = fourRows(keyUnit, t), queryLength = fourRows(queryUnit, t);
        f32x4 front = {0, 0, 0, 0}, end = {0, 0, 0, 0};
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            const f32x4 k = valuesAt(L::keys, t, m) * keyLength, back = grown * by * rS[m][t];
            dq[m][t] *= a.scale * grown;
            dk[m][t] *= last;
            front += valuesAt(L::queries, t, m) * queryLength * dq[m][t] - k * back;
            end += k * dk[m][t];
            dk[m][t] -= back;
        }
        #pragma unroll
        for(int r = 0; r < 4; r++) { front[r] = sumOf16(front[r]); end[r] = sumOf16(end[r]); }
        if(n16 == 0) { *(f32x4*)(queryDots + wave * C + t * 16 + 4 * g) = front; *(f32x4*)(keyDots + wave * C + t * 16 + 4 * g) = end; }
    }
    {
        const uint32_t column = squareColumn * 16 + n16;
        const float betaColumn = beta[column];
        const double sumColumn = sums[column];
        #pragma unroll
        for(int q = 0; q < SQUARES; q++) {
            const f32x4 by = fourRows(beta, squareRow(q));
            #pragma unroll
            for(int r = 0; r < 4; r++) {
                const uint32_t row = squareRow(q) * 16 + 4 * g + r;
                const float between = row >= column ? decayOver(sums[row] - sumColumn) : 0.0f;
                dqk[q][r] = row >= column ? a.scale * between * (dqk[q][r] * betaColumn) : 0.0f;
                dkk[q][r] = row > column ? -between * (by[r] * betaColumn * dkk[q][r]) : 0.0f;
            }
        }
    }
    #pragma unroll
    for(int w = 1; w < 64; w *= 2) { stateDot += __shfl_xor(stateDot, w); }
    if(lane == 0) { ends[wave] = decay * stateDot; }
    #pragma unroll
    for(int i = 0; i < ITEMS; i++) {
        const uint32_t row = rowOfItem(i);
        betaDot[i] += partner<1>(betaDot[i]); betaDot[i] += partner<2>(betaDot[i]); betaDot[i] += partner<4>(betaDot[i]);
        if(stageAt == 0 && d.beta.data && row < count) { (rowsOf<float>(d.beta, a.chunks, p) + (uint64_t)(begin + row) * d.beta.rowStride)[head] = betaDot[i]; }
    }

    __syncthreads();
    if(d.g.data) {
        // crossings[i][j], i > j: what goes from row j to row i.  Sums over the rows from t on of each column, first of a part of the rows, then over the columns before t.
        constexpr int PARTS = 256 / C, EACH = C / PARTS, PITCH = C + 1;
        float *const crossings = (float*)stage, *const columnSums = crossings + C * PITCH;
        #pragma unroll
        for(int q = 0; q < SQUARES; q++) {
            if(squareRow(q) < squareColumn) { continue; }
            const uint32_t column = squareColumn * 16 + n16;
            f32x4 kk = {0, 0, 0, 0}, qk = {0, 0, 0, 0};
            #pragma unroll
            for(int s = 0; s < DK / 32; s++) {
                inTurn();
                const uint32_t rows = unitAt<DK>(squareRow(q) * 16 + n16, 4 * s + g);
                const Planes<NP> columns = fetch<NP>(planes + L::keys + unitAt<DK>(column, 4 * s + g), C * DK);
                kk = multiply(fetch<NP>(planes + L::keys + rows, C * DK), columns, kk);
                qk = multiply(fetch<NP>(planes + L::queries + rows, C * DK), columns, qk);
            }
            const float length = keyUnit[column];
            const f32x4 x = (dqk[q] * (fourRows(queryUnit, squareRow(q)) * qk) + dkk[q] * (fourRows(keyUnit, squareRow(q)) * kk)) * length;
            #pragma unroll
            for(int r = 0; r < 4; r++) {
                const uint32_t row = squareRow(q) * 16 + 4 * g + r;
                crossings[row * PITCH + column] = row > column ? x[r] : 0.0f;
            }
        }
        __syncthreads();
        const uint32_t of = tid % C, part = tid / C;
        float below = 0.0f;
        #pragma unroll
        for(int i = EACH - 1; i >= 0; i--) {
            const uint32_t row = part * EACH + i;
            if(row <= of) { break; }
            crossings[row * PITCH + of] = below += crossings[row * PITCH + of];
        }
        columnSums[part * C + of] = below;
        __syncthreads();
        float across = 0.0f;
        #pragma unroll
        for(int i = 0; i < EACH; i++) {
            const uint32_t column = part * EACH + i;
            if(column >= of) { break; }
            float sum = crossings[of * PITCH + column];
            for(uint32_t behind = of / EACH + 1; behind < PARTS; behind++) { sum += columnSums[behind * C + column]; }
            across += sum;
        }
        crossingDots[part * C + of] = across;
        __syncthreads();
        if(wave == 0) {
            double front = 0.0, end = 0.0, sum = 0.0;
            if(lane < C) {
                #pragma unroll
                for(int w = 0; w < 4; w++) { front += queryDots[w * C + lane]; end += keyDots[w * C + lane]; sum += ends[w]; }
                #pragma unroll
                for(int w = 0; w < PARTS; w++) { sum += crossingDots[w * C + lane]; }
            }
            #pragma unroll
            for(int w = 1; w < C; w *= 2) {
                const double behind = __shfl_down(front, w), before = __shfl_up(end, w);
                if(lane + w < C) { front += behind; }
                if(lane >= (uint32_t)w) { end += before; }
            }
            const double before = __shfl_up(end, 1);
            if(lane > 0) { sum += before; }
            if(lane < count) { (rowsOf<float>(d.g, a.chunks, p) + (uint64_t)(begin + lane) * d.g.rowStride)[head] = (float)(sum + front); }
        }
    }
    if(!d.q.data && !d.k.data) { return; }

    // squares times queries and keys
    const auto storeSquares = [&](bool transposed, const f32x4 (&square)[SQUARES], const float *rowFactor, const float *columnFactor) {
        #pragma unroll
        for(int q = 0; q < SQUARES; q++) {
            const uint32_t column = squareColumn * 16 + n16, row = squareRow(q) * 16 + 4 * g;
            const f32x4 scaled = square[q] * (rowFactor ? fourRows(rowFactor, squareRow(q)) : f32x4{1, 1, 1, 1} * columnFactor[column]);
            const float x[4] = {scaled[0], scaled[1], scaled[2], scaled[3]};
            uint2 words[3];
            splitFour<3, (NP > 1)>(x, words);
            #pragma unroll
            for(int k = 0; k < 3; k++) {
                uint16_t *const to = stage + k * C * C;
                if(transposed) { *(uint2*)(to + unitAt<C>(column, row / 8) + row % 8) = words[k]; }
                else {
                    to[unitAt<C>(row, column / 8) + column % 8] = (uint16_t)words[k].x;
                    to[unitAt<C>(row + 1, column / 8) + column % 8] = (uint16_t)(words[k].x >> 16);
                    to[unitAt<C>(row + 2, column / 8) + column % 8] = (uint16_t)words[k].y;
                    to[unitAt<C>(row + 3, column / 8) + column % 8] = (uint16_t)(words[k].y >> 16);
                }
            }
        }
    };
    // (`lower`, `upper`: whether the square has blocks of 32 rows and columns below the diagonal's, and above them)
    const auto timesColumns = [&](uint32_t from, f32x4 (&to)[MINE][TILES], bool lower, bool upper) {
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            #pragma unroll
            for(int s = 0; s < TILES / 2; s++) {
                inTurn();
                const uint32_t row = 32 * s + 8 * g + n16 / 4, unit = 2 * (wave * MINE + m) + n16 % 4 / 2, half = n16 % 2 * 4;
                const Planes<NP> b = fetchColumn<NP>(planes + from + unitAt<DK>(row, unit) + half, planes + from + unitAt<DK>(row + 4, unit) + half, C * DK);
                #pragma unroll
                for(int t = 0; t < TILES; t += 2) {
                    if((t / 2 < s && !upper) || (t / 2 > s && !lower)) { continue; }
                    const Planes<3> rows[2] = {fetch<3>(stage + unitAt<C>(t * 16 + n16, 4 * s + g), C * C), fetch<3>(stage + unitAt<C>(t * 16 + 16 + n16, 4 * s + g), C * C)};
                    f32x4 sum[2] = {to[m][t], to[m][t + 1]};
                    multiplyAll(rows, b, sum);
                    to[m][t] = sum[0];
                    to[m][t + 1] = sum[1];
                }
            }
        }
    };
    storeSquares(false, dqk, nullptr, keyUnit);
    __syncthreads();
    timesColumns(L::keys, dq, true, false);
    // q^.dq^, for the queries' lengths
    if(a.normalise && a.group == 1) {
        #pragma unroll
        for(int t = 0; t < TILES; t++) {
            const f32x4 queryLength = fourRows(queryUnit, t);
            f32x4 dot = {0, 0, 0, 0};
            #pragma unroll
            for(int m = 0; m < MINE; m++) { dot += valuesAt(L::queries, t, m) * queryLength * dq[m][t]; }
            #pragma unroll
            for(int r = 0; r < 4; r++) { dot[r] = sumOf16(dot[r]); }
            if(n16 == 0) { *(f32x4*)(queryDots + wave * C + t * 16 + 4 * g) = dot; }
        }
    }
    __syncthreads();
    storeSquares(true, dqk, queryUnit, nullptr);
    __syncthreads();
    timesColumns(L::queries, dk, false, true);
    __syncthreads();
    // (both triangles of what is symmetric)
    storeSquares(true, dkk, keyUnit, nullptr);
    __syncthreads();
    timesColumns(L::keys, dk, false, true);
    __syncthreads();
    storeSquares(false, dkk, nullptr, keyUnit);
    __syncthreads();
    timesColumns(L::keys, dk, true, false);
    if(a.group > 1) {
        float *const to = d.shared + at * 2 * C * DK;
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            #pragma unroll
            for(int t = 0; t < TILES; t++) {
                #pragma unroll
                for(int r = 0; r < 4; r++) {
                    to[(t * 16 + 4 * g + r) * DK + keyOf(m)] = dq[m][t][r];
                    to[(C + t * 16 + 4 * g + r) * DK + keyOf(m)] = dk[m][t][r];
                }
            }
        }
        return;
    }

    // through the lengths of queries and keys
    if(a.normalise) {
        #pragma unroll
        for(int t = 0; t < TILES; t++) {
            const f32x4 keyLength = fourRows(keyUnit, t);
            f32x4 dot = {0, 0, 0, 0};
            #pragma unroll
            for(int m = 0; m < MINE; m++) { dot += valuesAt(L::keys, t, m) * keyLength * dk[m][t]; }
            #pragma unroll
            for(int r = 0; r < 4; r++) { dot[r] = sumOf16(dot[r]); }
            if(n16 == 0) { *(f32x4*)(keyDots + wave * C + t * 16 + 4 * g) = dot; }
        }
        __syncthreads();
    }
    #pragma unroll
    for(int t = 0; t < TILES; t++) {
        const f32x4 queryLength = fourRows(queryUnit, t), keyLength = fourRows(keyUnit, t);
        f32x4 queryDot = {0, 0, 0, 0}, keyDot = {0, 0, 0, 0};
        if(a.normalise) {
            #pragma unroll
            for(int w = 0; w < 4; w++) { queryDot += fourRows(queryDots + w * C, t); keyDot += fourRows(keyDots + w * C, t); }
        }
        #pragma unroll
        for(int m = 0; m < MINE; m++) {
            const f32x4 x = (dq[m][t] - valuesAt(L::queries, t, m) * queryLength * queryDot) * queryLength, y = (dk[m][t] - valuesAt(L::keys, t, m) * keyLength * keyDot) * keyLength;
            const uint32_t key = keyOf(m);
            #pragma unroll
            for(int r = 0; r < 4; r++) {
                const uint32_t row = t * 16 + 4 * g + r;
                if(row < count && key < a.keys) {
                    if(d.q.data) { (rowsOf<T>(d.q, a.chunks, p) + (uint64_t)(begin + row) * d.q.rowStride)[keyHead * a.keys + key] = narrow<T>(x[r]); }
                    if(d.k.data) { (rowsOf<T>(d.k, a.chunks, p) + (uint64_t)(begin + row) * d.k.rowStride)[keyHead * a.keys + key] = narrow<T>(y[r]); }
                }
            }
        }
    }
}

// Gradients of keys and queries that heads share: the heads' one after another, then through the lengths.  A wavefront a row of a key head, lane l its keys l and l + 64.
template<typename T, int C, int DK>
__global__ __launch_bounds__(256)
void deltaSharedKernel(DeltaArgs a, DeltaGradientArgs d)
{
    const uint32_t lane = threadIdx.x & 63, row = blockIdx.x % (C / 4) * 4 + (threadIdx.x >> 6), chunk = blockIdx.x / (C / 4);
    const uint32_t number = chunk / a.keyHeads, keyHead = chunk - number * a.keyHeads;
    Place p;
    if(!locate(a.chunks, number, p)) { return; }
    const uint32_t begin = p.index * C, count = min((uint32_t)C, p.length - min(p.length, begin));
    const float *const from = d.shared + ((uint64_t)number * a.heads + keyHead * a.group) * 2 * C * DK;
    if(row < count) {
        #pragma unroll
        for(int which = 0; which < 2; which++) {
            const gennmi_rows_t &in = which ? a.k : a.q, &out = which ? d.k : d.q;
            if(!out.data) { continue; }
            float x[DK / 64], hat[DK / 64], square = 0.0f, dot = 0.0f;
            #pragma unroll
            for(int i = 0; i < DK / 64; i++) {
                const uint32_t key = lane + 64 * i;
                x[i] = 0.0f;
                for(uint32_t h = 0; h < a.group; h++) { x[i] += from[(h * 2 + which) * C * DK + row * DK + key]; }
                hat[i] = key < a.keys ? widen(rowAt<T>(in, a.chunks, p, begin + row)[keyHead * a.keys + key]) : 0.0f;
                square = __builtin_fmaf(hat[i], hat[i], square);
            }
            float unit = 1.0f;
            if(a.normalise) {
                #pragma unroll
                for(int w = 1; w < 64; w *= 2) { square += __shfl_xor(square, w); }
                unit = 1.0f / sqrtf(square + a.epsilon);
                #pragma unroll
                for(int i = 0; i < DK / 64; i++) { hat[i] *= unit; dot = __builtin_fmaf(hat[i], x[i], dot); }
                #pragma unroll
                for(int w = 1; w < 64; w *= 2) { dot += __shfl_xor(dot, w); }
                #pragma unroll
                for(int i = 0; i < DK / 64; i++) { x[i] -= hat[i] * dot; }
            }
            T *const to = rowsOf<T>(out, a.chunks, p) + (uint64_t)(begin + row) * out.rowStride + keyHead * a.keys;
            #pragma unroll
            for(int i = 0; i < DK / 64; i++) { if(lane + 64 * i < a.keys) { to[lane + 64 * i] = narrow<T>(x[i] * unit); } }
        }
    }
}

// ---- a token of every running sequence
// Bound by the state, which is read and written once: a work-group has a head's columns of 8 lanes times VEC, a lane the rows with its number (of 32) in them, in registers
// between reading and writing.  One sum over the rows does for everything: with S' k, S' q, |k|^2, |q|^2 and k.q
//   u = beta (v - a S' k^),   out = scale (a S' q^ + (k^.q^) u).
// 32 heads of 128 x 128 in bf16: one sequence 5.3 us (the launch), 32 33, 128 131, 256 232 (4.7 TB/s past the caches, 249 through them).
__device__ inline float eightApart(float x) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x128, 0xf, 0xf, true)); }      // row_ror:8
template<typename T, int ROWS, int VEC, bool STREAM>
__global__ __launch_bounds__(256)
void deltaTokenKernel(DeltaArgs a)
{
    constexpr int SUMS = 2 * VEC + 3;
    __shared__ float sums[4][8][SUMS];
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, inRow = tid & 7, part = tid >> 3;
    const uint32_t block = blockIdx.x % a.columnBlocks, rest = blockIdx.x / a.columnBlocks, head = rest % a.heads, sequence = rest / a.heads, keyHead = head / a.group;
    const uint32_t column = (block * 8 + inRow) * VEC;
    const bool inside = column < a.values;
    Place p;
    if(!describe(a.chunks, sequence, p)) { return; }
    const uint64_t stateAt = ((uint64_t)p.state * a.heads + head) * a.keys * a.values + column;
    typedef Pack<float, VEC> Columns;
    typedef float Stream __attribute__((ext_vector_type(VEC)));
    Columns s[ROWS];
    #pragma unroll
    for(int i = 0; i < ROWS; i++) {
        const uint32_t row = part + 32 * i;
        s[i] = Columns{};
        if(a.initialState && row < a.keys && inside) {
            const float *const from = a.initialState + stateAt + (uint64_t)row * a.values;
            if constexpr(STREAM) { s[i] = __builtin_bit_cast(Columns, __builtin_nontemporal_load((const Stream*)from)); }
            else { s[i] = *(const Columns*)from; }
        }
    }
    if(p.length) {
        const T *const keys = rowsOf<const T>(a.k, a.chunks, p) + keyHead * a.keys, *const queries = rowsOf<const T>(a.q, a.chunks, p) + keyHead * a.keys;
        const float beta = rowsOf<const float>(a.beta, a.chunks, p)[head], decay = decayOver(clampGate(rowsOf<const float>(a.g, a.chunks, p)[head]));
        float v[VEC], k[ROWS], q[ROWS], sum[SUMS] = {};
        #pragma unroll
        for(int e = 0; e < VEC; e++) { v[e] = inside && column + e < a.values ? widen((rowsOf<const T>(a.v, a.chunks, p) + head * a.values)[column + e]) : 0.0f; }
        #pragma unroll
        for(int i = 0; i < ROWS; i++) {
            const uint32_t row = part + 32 * i;
            k[i] = row < a.keys ? widen(keys[row]) : 0.0f;
            q[i] = row < a.keys ? widen(queries[row]) : 0.0f;
        }
        #pragma unroll
        for(int i = 0; i < ROWS; i++) {
            #pragma unroll
            for(int e = 0; e < VEC; e++) { sum[e] = __builtin_fmaf(s[i].v[e], k[i], sum[e]); sum[VEC + e] = __builtin_fmaf(s[i].v[e], q[i], sum[VEC + e]); }
            sum[2 * VEC] = __builtin_fmaf(k[i], k[i], sum[2 * VEC]);
            sum[2 * VEC + 1] = __builtin_fmaf(q[i], q[i], sum[2 * VEC + 1]);
            sum[2 * VEC + 2] = __builtin_fmaf(k[i], q[i], sum[2 * VEC + 2]);
        }
        #pragma unroll
        for(int n = 0; n < SUMS; n++) {
            // (over the eight parts of the wavefront: lanes 8, 16 and 32 apart)
            sum[n] += eightApart(sum[n]);
            sum[n] += partner<16>(sum[n]);
            sum[n] += partner<32>(sum[n]);
            if(lane < 8) { sums[wave][inRow][n] = sum[n]; }
        }
        __syncthreads();
        #pragma unroll
        for(int n = 0; n < SUMS; n++) { sum[n] = (sums[0][inRow][n] + sums[1][inRow][n]) + (sums[2][inRow][n] + sums[3][inRow][n]); }
        const float keyUnit = a.normalise ? 1.0f / sqrtf(sum[2 * VEC] + a.epsilon) : 1.0f, queryUnit = a.normalise ? 1.0f / sqrtf(sum[2 * VEC + 1] + a.epsilon) : 1.0f;
        float u[VEC];
        #pragma unroll
        for(int e = 0; e < VEC; e++) { u[e] = beta * __builtin_fmaf(-decay * keyUnit, sum[e], v[e]); }
        if(part == 0 && inside) {
            T *const out = rowsOf<T>(a.out, a.chunks, p) + head * a.values;
            const float both = keyUnit * sum[2 * VEC + 2];
            #pragma unroll
            for(int e = 0; e < VEC; e++) { if(column + e < a.values) { out[column + e] = narrow<T>(a.scale * queryUnit * __builtin_fmaf(both, u[e], decay * sum[VEC + e])); } }
        }
        #pragma unroll
        for(int i = 0; i < ROWS; i++) {
            #pragma unroll
            for(int e = 0; e < VEC; e++) { s[i].v[e] = __builtin_fmaf(k[i] * keyUnit, u[e], decay * s[i].v[e]); }
        }
    }
    if(!a.finalState || !inside) { return; }
    #pragma unroll
    for(int i = 0; i < ROWS; i++) {
        const uint32_t row = part + 32 * i;
        if(row >= a.keys) { continue; }
        float *const to = a.finalState + stateAt + (uint64_t)row * a.values;
        if constexpr(STREAM) { __builtin_nontemporal_store(__builtin_bit_cast(Stream, s[i]), (Stream*)to); }
        else { *(Columns*)to = s[i]; }
    }
}
}

#endif

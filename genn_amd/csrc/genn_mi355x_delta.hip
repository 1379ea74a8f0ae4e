// The gated delta rule, for whole sequences (with gradients) and for single tokens.  Entry points and their checks; the kernels are in the header included below.
#include <algorithm>
#include <type_traits>

#include "genn_mi355x_delta_kernels.h"

using namespace gennmi_elements;
using namespace gennmi_delta;
using gennmi_detail::fail;

namespace
{
// Rows of a chunk: 64 where keys are one plane of 16 bits; with two or three, what a chunk needs of LDS would pass a compute unit's 160 KiB
uint32_t chunkRows(uint32_t type) { return type == GENNMI_TYPE_BF16 ? 64 : 32; }
uint32_t paddedKeys(uint32_t keys) { return keys <= 64 ? 64 : 128; }
uint32_t paddedValues(uint32_t values) { return (values + 31) / 32 * 32; }
// Calls f with the element type, the rows of a chunk and the keys that the kernels have room for
template<typename F> int withSizes(const gennmi_delta_rule_t &c, F &&f)
{
    const auto keys = [&](auto t, auto rows) {
        return paddedKeys(c.keys) == 64 ? f(t, rows, std::integral_constant<int, 64>{}) : f(t, rows, std::integral_constant<int, 128>{});
    };
    switch(c.type) {
    case GENNMI_TYPE_F32: return keys(float{}, std::integral_constant<int, 32>{});
    case GENNMI_TYPE_F16: return keys(f16{}, std::integral_constant<int, 32>{});
    default: return keys(bf16{}, std::integral_constant<int, 64>{});
    }
}
constexpr uint32_t WALK_COLUMNS = WALK_THREADS / 64 * 16;         // of a work-group of a walk
uint32_t blocksOf(uint32_t columns) { return (columns + WALK_COLUMNS - 1) / WALK_COLUMNS; }

// Work-groups that share what they read go to one of the chip's eight parts: of segments and key heads (of sequences and heads) eight at a time, so many work-groups each
uint64_t walkGrid(uint64_t outer, uint64_t each) { return (outer + 7) / 8 * 8 * each; }

int checkDelta(const char *what, const gennmi_delta_rule_t *c, bool gradients)
{
    if(!c) { return fail(GENNMI_EINVAL, std::string(what) + ": null descriptor"); }
    const auto refuse = [&](int code, const char *why) { return fail(code, std::string(what) + why); };
    const uint32_t size = sizeOf(c->type);
    if(!size) { return refuse(GENNMI_EUNSUPPORTED, ": unknown element type"); }
    if(c->keys < 1 || c->keys > GENNMI_MAX_DELTA_KEYS) { return refuse(GENNMI_EUNSUPPORTED, ": number of keys"); }
    if(c->values < 1 || c->values > GENNMI_MAX_DELTA_VALUES) { return refuse(GENNMI_EUNSUPPORTED, ": number of values"); }
    if(c->heads < 1 || c->heads > (1u << 16) || c->keyHeads < 1 || c->heads % c->keyHeads) { return refuse(GENNMI_EINVAL, ": number of heads or key heads"); }
    if(const int rc = checkSequences(what, c->sequences, gradients)) { return rc; }
    const struct { const char *which; const gennmi_rows_t *rows; uint32_t width, size; } read[] = {
        {"q", &c->q, c->keyHeads * c->keys, size}, {"k", &c->k, c->keyHeads * c->keys, size}, {"v", &c->v, c->heads * c->values, size}, {"g", &c->g, c->heads, 4}, {"beta", &c->beta, c->heads, 4}};
    for(const auto &r : read) { if(const int rc = checkRows(what, r.which, *r.rows, c->sequences, r.width, r.size)) { return rc; } }
    if(!gradients) { if(const int rc = checkWrittenRows(what, "out", c->out, c->sequences, c->heads * c->values, size)) { return rc; } }
    for(const gennmi_rows_t *r : {&c->q, &c->k, &c->v, &c->out}) {
        if(c->sequences.length > 1 && r->data && r->rowStride >= GENNMI_MAX_DELTA_STRIDE) { return refuse(GENNMI_EINVAL, ": stride of q, k, v or out out of range"); }
    }
    if((uintptr_t)c->initialState % 4 || (uintptr_t)c->finalState % 4) { return refuse(GENNMI_EINVAL, ": a state is not aligned"); }
    return GENNMI_OK;
}
uint64_t stateBytes(const gennmi_delta_rule_t &c) { return (uint64_t)c.heads * c.keys * c.values * 4; }
int deltaApart(const char *what, const gennmi_delta_rule_t &c, const void *workspace, size_t workspaceBytes)
{
    const gennmi_sequences_t &s = c.sequences;
    const uint32_t size = sizeOf(c.type), keys = c.keyHeads * c.keys, values = c.heads * c.values;
    const uint64_t states = statesOf(s) * stateBytes(c);
    return checkApart(what, {regionOf("out", c.out, s, values, size), regionOf("the final state", c.finalState, states), regionOf("the workspace", workspace, workspaceBytes)}, {},
                      {regionOf("q", c.q, s, keys, size), regionOf("k", c.k, s, keys, size), regionOf("v", c.v, s, values, size), regionOf("g", c.g, s, c.heads, 4), regionOf("beta", c.beta, s, c.heads, 4),
                       unlessSame(regionOf("the initial state", c.initialState, states), c.finalState), offsetsOf(s), slotsOf(s)});
}
int deltaApart(const char *what, const gennmi_delta_rule_t &c, const gennmi_delta_rule_gradient_t &g, const void *workspace, size_t workspaceBytes)
{
    const gennmi_sequences_t &s = c.sequences;
    const uint32_t size = sizeOf(c.type), keys = c.keyHeads * c.keys, values = c.heads * c.values;
    const uint64_t states = statesOf(s) * stateBytes(c);
    return checkApart(what, {regionOf("the gradient of q", g.q, s, keys, size), regionOf("the gradient of k", g.k, s, keys, size), regionOf("the gradient of v", g.v, s, values, size),
                             regionOf("the gradient of g", g.g, s, c.heads, 4), regionOf("the gradient of beta", g.beta, s, c.heads, 4),
                             regionOf("the gradient of the initial state", g.initialState, states), regionOf("the workspace", workspace, workspaceBytes)}, {},
                      {regionOf("q", c.q, s, keys, size), regionOf("k", c.k, s, keys, size), regionOf("v", c.v, s, values, size), regionOf("g", c.g, s, c.heads, 4), regionOf("beta", c.beta, s, c.heads, 4),
                       regionOf("the gradient of out", g.out, s, values, size), regionOf("the initial state", c.initialState, states),
                       unlessSame(regionOf("the gradient of the final state", g.finalState, states), g.initialState), offsetsOf(s)});
}

// Segments that a sequence is cut into, so that there are work-groups for the whole chip: what each does to the state is found for all of them at once (the state's columns and
// those of a unit matrix), then joined, then outputs are found for all of them at once.  The number is the one that should take the shortest, in units of a chunk's step of a walk alone on the chip (5.7 us for 64 rows in bf16;
// one unit for all types):
// two work-groups fit a compute unit, and with all 512 a step takes 1.8 units; what a segment does takes 0.57 of that a step; a segment's join and what else comes with it 0.8 units.  One prompt of 64 chunks x 32 heads
// in 1, 2, 4, 8, 16 segments: 375, 330, 223, 207, 237 us, x 8 heads 358, 314, 181, 125, 122; 33 sequences of 8011 rows in all x 6 heads (fp16) in 1, 2, 4, 8, 16: 261, 247, 184, 197, 206
// (the rule takes 5 there, as the steps of 32 rows are shorter than it has them).
uint32_t segmentsOf(const gennmi_delta_rule_t &c, uint32_t columns)
{
    const uint32_t C = chunkRows(c.type), chunks = (c.sequences.length + C - 1) / C;
    const double all = (double)chunkNumbers(c.sequences, C) / std::max(1u, chunks) * c.heads, room = 512.0, blocks = blocksOf(columns), both = blocks + blocksOf(paddedKeys(c.keys));
    const auto step = [&](double groups) { return (1.0 + 0.8 * std::min(1.0, groups / room)) * std::max(1.0, groups / room); };
    uint32_t best = 1;
    double least = chunks * step(all * blocks);
    for(uint32_t n = 2; n <= std::min(chunks, 64u); n++) {
        const uint32_t each = (chunks + n - 1) / n;
        const double cost = each * (step(all * blocks * n) + 0.57 * step(all * both * (n - 1))) + 0.8 * n + 0.5;
        if(cost < least) { least = cost; best = n; }
    }
    return best;
}
// Rows of a segment: a multiple of a chunk's
uint32_t segmentRows(const gennmi_delta_rule_t &c, bool gradients)
{
    const uint32_t C = chunkRows(c.type), chunks = std::max(1u, (c.sequences.length + C - 1) / C), segments = gradients ? 1 : segmentsOf(c, c.values);
    return (chunks + segments - 1) / segments * C;
}
bool isCut(const gennmi_delta_rule_t &c, bool gradients) { return c.sequences.length > segmentRows(c, gradients); }
uint32_t moveBlocks(const gennmi_delta_rule_t &c) { return blocksOf(paddedKeys(c.keys)); }
struct DeltaSpace { size_t correction, score, rows, table, segmentStates, segmentMoves, states, errors, gradientStates, gradientErrors, shared, bytes; };
DeltaSpace deltaSpace(const gennmi_delta_rule_t &c, bool gradients)
{
    DeltaSpace s{};
    const uint64_t C = chunkRows(c.type), numbers = chunkNumbers(c.sequences, (uint32_t)C) * c.heads, padded = paddedValues(c.values);
    if(!gradients && c.sequences.length <= 1) { return s; }
    const auto take = [&](uint64_t bytes) { const size_t at = s.bytes; s.bytes += (bytes + 255) / 256 * 256; return at; };
    s.correction = take(numbers * C * C * 4);
    s.score = take(numbers * C * C * 4);
    s.rows = take(numbers * C * 32);
    s.table = take(numbers * sizeof(ChunkTable));
    if(isCut(c, gradients)) {
        const uint64_t segments = chunkNumbers(c.sequences, segmentRows(c, gradients)) * c.heads;
        s.segmentStates = take(segments * paddedKeys(c.keys) * padded * 4);
        s.segmentMoves = take(segments * paddedKeys(c.keys) * paddedKeys(c.keys) * 4);
    }
    if(gradients) {
        s.states = take(numbers * paddedKeys(c.keys) * padded * 4);
        s.errors = take(numbers * C * padded * 4);
        s.gradientStates = take(numbers * paddedKeys(c.keys) * padded * 4);
        s.gradientErrors = take(numbers * C * padded * 4);
        if(c.heads > c.keyHeads) { s.shared = take(numbers * 2 * C * paddedKeys(c.keys) * 4); }
    }
    return s;
}
uint32_t tokenVector(const gennmi_delta_rule_t &c) { return c.values % 4 == 0 && (uintptr_t)c.initialState % 16 == 0 && (uintptr_t)c.finalState % 16 == 0 ? 4 : 1; }
uint64_t tokenBlocks(const gennmi_delta_rule_t &c) { const uint32_t columns = 8 * tokenVector(c); return (uint64_t)c.sequences.count * c.heads * ((c.values + columns - 1) / columns); }
bool deltaFits(const gennmi_delta_rule_t &c, bool gradients)
{
    if(!gradients && c.sequences.length <= 1) { return tokenBlocks(c) <= mostBlocks(256); }
    const uint32_t columns = gradients ? paddedValues(c.values) : c.values;
    return chunkNumbers(c.sequences, chunkRows(c.type)) * c.heads * (gradients && c.heads > c.keyHeads ? 8 : 1) <= mostBlocks(512) &&
        walkGrid(chunkNumbers(c.sequences, segmentRows(c, gradients)) * c.keyHeads, (uint64_t)(c.heads / c.keyHeads) * (gradients ? 2 * blocksOf(columns) : blocksOf(columns) + moveBlocks(c))) <= mostBlocks(WALK_THREADS) &&
        walkGrid((uint64_t)c.sequences.count * c.heads, paddedValues(c.values) / 16) <= mostBlocks(256);
}
DeltaArgs deltaArgs(const gennmi_delta_rule_t &c, const DeltaSpace &space, void *workspace, bool gradients)
{
    DeltaArgs a{};
    a.chunks = sequencesOf(c.sequences, chunkRows(c.type));
    a.segments = sequencesOf(c.sequences, segmentRows(c, gradients));
    a.q = c.q; a.k = c.k; a.v = c.v; a.out = c.out; a.g = c.g; a.beta = c.beta;
    a.initialState = c.initialState;
    a.finalState = gradients ? nullptr : c.finalState;
    a.heads = c.heads; a.keyHeads = c.keyHeads; a.group = c.heads / c.keyHeads; a.keys = c.keys; a.values = c.values; a.normalise = c.normalise;
    a.padded = paddedValues(c.values);
    a.columnBlocks = blocksOf(gradients ? a.padded : a.values);
    a.segmentNumbers = (uint32_t)chunkNumbers(c.sequences, segmentRows(c, gradients));
    a.scale = c.scale; a.epsilon = c.epsilon;
    const uint32_t size = sizeOf(c.type);
    const auto wide = [&](const gennmi_rows_t &r) { return (uintptr_t)r.data % 16 == 0 && r.rowStride * size % 16 == 0 && r.sequenceStride * size % 16 == 0; };
    a.wide = c.keys % 8 == 0 && wide(c.q) && wide(c.k);
    const auto at = [&](size_t offset) { return (char*)workspace + offset; };
    a.correction = (float*)at(space.correction);
    a.score = (float*)at(space.score);
    a.rows = at(space.rows);
    a.table = (ChunkTable*)at(space.table);
    if(isCut(c, gradients)) {
        a.segmentStates = (float*)at(space.segmentStates);
        a.segmentMoves = (float*)at(space.segmentMoves);
        a.moveBlocks = moveBlocks(c);
    }
    if(gradients) {
        a.states = (float*)at(space.states);
        a.errors = (float*)at(space.errors);
    }
    return a;
}

template<typename T, int C, int DK, bool FOLDED> int launchChunks(const char *what, const DeltaArgs &a, uint64_t numbers, hipStream_t stream)
{
    const auto kernel = deltaChunkKernel<T, C, DK, FOLDED>;
    constexpr size_t lds = chunkLds<T, C, DK>();
    if(const int rc = withLds(what, kernel, lds)) { return rc; }
    kernel<<<dim3((uint32_t)(numbers * a.keyHeads)), dim3(256), lds, stream>>>(a);
    return gennmi_detail::afterLaunch(what);
}
template<typename T, int C, int DK, int MODE, bool FOLDED> int launchWalk(const char *what, const DeltaArgs &a, uint64_t segments, hipStream_t stream)
{
    const auto kernel = deltaStateKernel<T, C, DK, MODE, FOLDED>;
    constexpr size_t lds = WalkLayout<T, C, DK, MODE == WALK_OUTPUTS>::bytes;
    if(const int rc = withLds(what, kernel, lds)) { return rc; }
    kernel<<<dim3((uint32_t)walkGrid(segments * a.keyHeads, a.group * (a.columnBlocks + (MODE == WALK_SUMMARY ? a.moveBlocks : 0)))), dim3(WALK_THREADS), lds, stream>>>(a);
    return gennmi_detail::afterLaunch(what);
}
// The state in front of every segment
template<typename T, int C, int DK, bool FOLDED> int launchSegments(const char *what, const DeltaArgs &a, uint64_t segments, hipStream_t stream)
{
    if(!a.segmentStates) { return GENNMI_OK; }
    if(const int rc = launchWalk<T, C, DK, WALK_SUMMARY, FOLDED>(what, a, segments, stream)) { return rc; }
    deltaJoinKernel<DK><<<dim3((uint32_t)walkGrid((uint64_t)a.chunks.count * a.heads, a.padded / 16)), dim3(256), 0, stream>>>(a);
    return gennmi_detail::afterLaunch(what);
}
template<typename T, int C, int DK> int launchGradients(const char *what, const DeltaArgs &a, const DeltaGradientArgs &d, uint64_t numbers, uint64_t segments, hipStream_t stream)
{
    if(const int rc = launchChunks<T, C, DK, false>(what, a, numbers, stream)) { return rc; }
    const uint64_t grid = walkGrid(segments * a.keyHeads, a.group * a.columnBlocks);
    const auto walks = 2 * grid <= 256 ? deltaWalksKernel<T, C, DK, true> : deltaWalksKernel<T, C, DK, false>;
    constexpr size_t walksLds = WalkLayout<T, C, DK, true>::bytes;
    if(const int rc = withLds(what, walks, walksLds)) { return rc; }
    walks<<<dim3((uint32_t)grid, 2), dim3(WALK_THREADS), walksLds, stream>>>(a, d);
    const int rc = gennmi_detail::afterLaunch(what);
    if(rc || !(d.q.data || d.k.data || d.g.data || d.beta.data)) { return rc; }
    const auto kernel = deltaGradientKernel<T, C, DK>;
    constexpr size_t lds = GradientLayout<T, C, DK>::bytes;
    if(const int rcLds = withLds(what, kernel, lds)) { return rcLds; }
    kernel<<<dim3((uint32_t)(numbers * a.heads)), dim3(256), lds, stream>>>(a, d);
    if(const int rcGradient = gennmi_detail::afterLaunch(what)) { return rcGradient; }
    if(a.group == 1 || !(d.q.data || d.k.data)) { return GENNMI_OK; }
    deltaSharedKernel<T, C, DK><<<dim3((uint32_t)(numbers * a.keyHeads * (C / 4))), dim3(256), 0, stream>>>(a, d);
    return gennmi_detail::afterLaunch(what);
}
// States of more than the last cache holds (256 MiB) pass the caches by
bool streams(const gennmi_delta_rule_t &c) { return tokenVector(c) == 4 && c.sequences.count * stateBytes(c) > (256ull << 20); }
template<typename T, int VEC, bool STREAM> int launchToken(const char *what, const DeltaArgs &a, uint32_t blocks, hipStream_t stream)
{
    const dim3 grid(blocks), threads(256);
    if(a.keys <= 32) { deltaTokenKernel<T, 1, VEC, STREAM><<<grid, threads, 0, stream>>>(a); }
    else if(a.keys <= 64) { deltaTokenKernel<T, 2, VEC, STREAM><<<grid, threads, 0, stream>>>(a); }
    else { deltaTokenKernel<T, 4, VEC, STREAM><<<grid, threads, 0, stream>>>(a); }
    return gennmi_detail::afterLaunch(what);
}
}

extern "C" {

int gennmi_delta_rule_workspace(const gennmi_delta_rule_t *rule, size_t *bytes)
{
    return gennmi_detail::guarded("delta_rule_workspace", [&] {
        if(const int rc = checkDelta("delta_rule_workspace", rule, false)) { return rc; }
        if(!bytes) { return fail(GENNMI_EINVAL, "delta_rule_workspace: null result pointer"); }
        if(!deltaFits(*rule, false)) { return tooMany("delta_rule_workspace"); }
        *bytes = deltaSpace(*rule, false).bytes;
        return (int)GENNMI_OK;
    });
}

int gennmi_delta_rule(const gennmi_delta_rule_t *rule, void *workspace, size_t workspaceBytes, void *stream)
{
    const char *what = "delta_rule";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkDelta(what, rule, false)) { return rc; }
        if(!deltaFits(*rule, false)) { return tooMany(what); }
        const DeltaSpace space = deltaSpace(*rule, false);
        if(const int rc = checkWorkspace(what, workspace, workspaceBytes, space.bytes)) { return rc; }
        if(const int rc = deltaApart(what, *rule, workspace, space.bytes)) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, rule->sequences.device)) { return rc; }
        if(!rule->sequences.count) { return (int)GENNMI_OK; }
        DeltaArgs a = deltaArgs(*rule, space, workspace, false);
        const hipStream_t s = (hipStream_t)stream;
        int rc;
        if(rule->sequences.length <= 1) {
            const uint32_t vector = tokenVector(*rule), blocks = (uint32_t)tokenBlocks(*rule);
            a.columnBlocks = (rule->values + 8 * vector - 1) / (8 * vector);
            rc = withType(rule->type, [&](auto t) {
                typedef decltype(t) T;
                if(vector == 1) { return launchToken<T, 1, false>(what, a, blocks, s); }
                return streams(*rule) ? launchToken<T, 4, true>(what, a, blocks, s) : launchToken<T, 4, false>(what, a, blocks, s);
            });
        }
        else {
            rc = withSizes(*rule, [&](auto t, auto rows, auto keys) {
                typedef decltype(t) T;
                constexpr int C = decltype(rows)::value, DK = decltype(keys)::value;
                if(const int rcChunks = launchChunks<T, C, DK, true>(what, a, chunkNumbers(rule->sequences, C), s)) { return rcChunks; }
                const uint64_t segments = chunkNumbers(rule->sequences, a.segments.chunk);
                if(const int rcSegments = launchSegments<T, C, DK, true>(what, a, segments, s)) { return rcSegments; }
                return launchWalk<T, C, DK, WALK_OUTPUTS, true>(what, a, segments, s);
            });
        }
        if(rc) { return rc; }
        noteRows(rule->out, rule->sequences, rule->heads * rule->values, sizeOf(rule->type));
        if(rule->finalState) { gennmi_detail::noteDeviceWrite(rule->finalState, statesOf(rule->sequences) * stateBytes(*rule)); }
        return (int)GENNMI_OK;
    });
}

int gennmi_delta_rule_backward_workspace(const gennmi_delta_rule_t *rule, size_t *bytes)
{
    return gennmi_detail::guarded("delta_rule_backward_workspace", [&] {
        if(const int rc = checkDelta("delta_rule_backward_workspace", rule, true)) { return rc; }
        if(!bytes) { return fail(GENNMI_EINVAL, "delta_rule_backward_workspace: null result pointer"); }
        if(!deltaFits(*rule, true)) { return tooMany("delta_rule_backward_workspace"); }
        *bytes = deltaSpace(*rule, true).bytes;
        return (int)GENNMI_OK;
    });
}

int gennmi_delta_rule_backward(const gennmi_delta_rule_t *rule, const gennmi_delta_rule_gradient_t *gradient, void *workspace, size_t workspaceBytes, void *stream)
{
    const char *what = "delta_rule_backward";
    return gennmi_detail::guarded(what, [&] {
        if(const int rc = checkDelta(what, rule, true)) { return rc; }
        if(!gradient) { return fail(GENNMI_EINVAL, "delta_rule_backward: null gradient"); }
        const gennmi_delta_rule_gradient_t &in = *gradient;
        const uint32_t size = sizeOf(rule->type), keys = rule->keyHeads * rule->keys, values = rule->heads * rule->values;
        if(const int rc = checkRows(what, "the gradient of out", in.out, rule->sequences, values, size)) { return rc; }
        const struct { const char *which; const gennmi_rows_t *rows; uint32_t width, size; } written[] = {
            {"the gradient of q", &in.q, keys, size}, {"the gradient of k", &in.k, keys, size}, {"the gradient of v", &in.v, values, size},
            {"the gradient of g", &in.g, rule->heads, 4}, {"the gradient of beta", &in.beta, rule->heads, 4}};
        for(const auto &w : written) {
            if(!w.rows->data) { continue; }
            if(const int rc = checkWrittenRows(what, w.which, *w.rows, rule->sequences, w.width, w.size)) { return rc; }
        }
        if(rule->sequences.length > 1 && (in.out.rowStride >= GENNMI_MAX_DELTA_STRIDE || (in.v.data && in.v.rowStride >= GENNMI_MAX_DELTA_STRIDE))) {
            return fail(GENNMI_EINVAL, "delta_rule_backward: stride of the gradients of v or out out of range");
        }
        if((uintptr_t)in.finalState % 4 || (uintptr_t)in.initialState % 4) { return fail(GENNMI_EINVAL, "delta_rule_backward: a state is not aligned"); }
        if(!deltaFits(*rule, true)) { return tooMany(what); }
        const DeltaSpace space = deltaSpace(*rule, true);
        if(const int rc = checkWorkspace(what, workspace, workspaceBytes, space.bytes)) { return rc; }
        if(const int rc = deltaApart(what, *rule, in, workspace, space.bytes)) { return rc; }
        if(const int rc = gennmi_detail::beforeLaunch((hipStream_t)stream, rule->sequences.device)) { return rc; }
        if(!rule->sequences.count) { return (int)GENNMI_OK; }
        DeltaArgs a = deltaArgs(*rule, space, workspace, true);
        const auto fours = [&](const gennmi_rows_t &r) { return (uintptr_t)r.data % (4 * size) == 0 && r.rowStride % 4 == 0 && r.sequenceStride % 4 == 0; };
        a.wideValues = rule->values % 4 == 0 && fours(in.out);
        DeltaGradientArgs d{};
        d.out = in.out; d.q = in.q; d.k = in.k; d.v = in.v; d.g = in.g; d.beta = in.beta;
        d.finalState = in.finalState; d.initialState = in.initialState;
        d.states = (float*)((char*)workspace + space.gradientStates);
        d.errors = (float*)((char*)workspace + space.gradientErrors);
        d.shared = (float*)((char*)workspace + space.shared);
        const int rc = withSizes(*rule, [&](auto t, auto rows, auto keysRoom) {
            typedef decltype(t) T;
            constexpr int C = decltype(rows)::value, DK = decltype(keysRoom)::value;
            return launchGradients<T, C, DK>(what, a, d, chunkNumbers(rule->sequences, C), chunkNumbers(rule->sequences, a.segments.chunk), (hipStream_t)stream);
        });
        if(rc) { return rc; }
        for(const auto &w : written) { noteRows(*w.rows, rule->sequences, w.width, w.size); }
        if(in.initialState) { gennmi_detail::noteDeviceWrite(in.initialState, (uint64_t)rule->sequences.count * stateBytes(*rule)); }
        return (int)GENNMI_OK;
    });
}

}

// Attention of new tokens over a key/value cache with a length per sequence, the new tokens being the nodes of a drafted
// tree (or a chain, or one), and the attention weight that every cached row receives.  fp32 in and out.
//
// Node i of sequence b sees the cached rows j < lengths[b] and those new rows j < counts[b] whose bit is set in
// visible[b, i] (NULL: bits 0..i, a chain).  With s_j = scale q_i . k_j over what it sees,
//   m = max s_j,  l = sum exp(s_j - m),  out = sum exp(s_j - m) v_j / l;     nothing seen: out = 0, m = -inf, l = 0.
// Query head h reads key head h * kvHeads / heads.
#include "common.hpp"

#include <cmath>

namespace bf {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

struct TreeParams {
    const float* q; const float* kNew; const float* vNew; const float* k; const float* v;
    const int* lengths; const int* counts; const unsigned long long* visible;
    float* out; float* m; float* l;
    const float* weightsIn; float* weightsOut;
    int batch, heads, kvHeads, groups, nodes, capacity, hd;
    float scale;
};

// What the device-side counters say, held inside what the tensors have room for
__device__ __forceinline__ int rowsInUse(const TreeParams& p, int b) { return min(max(p.lengths[b], 0), p.capacity); }
__device__ __forceinline__ int nodesInUse(const TreeParams& p, int b) { return p.counts ? min(max(p.counts[b], 0), p.nodes) : p.nodes; }
// the new rows node i sees, as bits below `count`
__device__ __forceinline__ unsigned long long newRowsSeen(const TreeParams& p, int b, int i, int count) {
    const unsigned long long upTo = count >= 64 ? ~0ull : (1ull << count) - 1;
    const unsigned long long bits = p.visible ? p.visible[size_t(b) * p.nodes + i] : (i >= 63 ? ~0ull : (2ull << i) - 1);
    return bits & upTo;
}

// One wavefront per (sequence, head, node), a key at a time.
__global__ void __launch_bounds__(256) treeAttentionKernel(TreeParams p) {
    const int lane = threadIdx.x & 63;
    const size_t row = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= size_t(p.batch) * p.heads * p.nodes) return;
    const int i = int(row % p.nodes), h = int(row / p.nodes % p.heads), b = int(row / p.nodes / p.heads);
    const int length = rowsInUse(p, b), count = nodesInUse(p, b);
    if (i >= count) return;
    const int kvDim = p.kvHeads * p.hd, kh = h / (p.heads / p.kvHeads);
    const unsigned long long seen = newRowsSeen(p, b, i, count);
    const float* q = p.q + (size_t(b) * p.nodes + i) * p.heads * p.hd + size_t(h) * p.hd;
    float qr[4], acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int u = 0; u < 4; ++u) qr[u] = lane + 64 * u < p.hd ? q[lane + 64 * u] : 0.0f;
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j < length + count; ++j) {
        const bool fresh = j >= length;
        if (fresh && !(seen >> (j - length) & 1)) continue;
        const size_t at = (fresh ? size_t(b) * p.nodes + (j - length) : size_t(b) * p.capacity + j) * kvDim + size_t(kh) * p.hd;
        const float* kr = (fresh ? p.kNew : p.k) + at;
        const float* vr = (fresh ? p.vNew : p.v) + at;
        float dot = 0.0f;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (lane + 64 * u < p.hd) dot += qr[u] * kr[lane + 64 * u];
        const float s = waveSum(dot) * p.scale;
        const float mm = fmaxf(m, s);
        const float keep = m == -INFINITY ? 0.0f : expf(m - mm), w = s == -INFINITY ? 0.0f : expf(s - mm);
        l = l * keep + w;
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (lane + 64 * u < p.hd) acc[u] = acc[u] * keep + w * vr[lane + 64 * u];
        m = mm;
    }
    float* out = p.out + (size_t(b) * p.nodes + i) * p.heads * p.hd + size_t(h) * p.hd;
#pragma unroll
    for (int u = 0; u < 4; ++u)
        if (lane + 64 * u < p.hd) out[lane + 64 * u] = l == 0.0f ? 0.0f : acc[u] / l;
    if (lane == 0) {
        const size_t stat = (size_t(b) * p.heads + h) * p.nodes + i;
        p.m[stat] = m;
        p.l[stat] = l;
    }
}

// One wavefront per (sequence, group, row of the cache): the row's weight from the statistics of the pass above.
__global__ void __launch_bounds__(256) treeWeightsKernel(TreeParams p) {
    const int lane = threadIdx.x & 63;
    const size_t row = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= size_t(p.batch) * p.groups * p.capacity) return;
    const int j = int(row % p.capacity), g = int(row / p.capacity % p.groups), b = int(row / p.capacity / p.groups);
    const int length = rowsInUse(p, b), count = nodesInUse(p, b);
    if (j >= length + count) return;
    const bool fresh = j >= length;
    const int kvDim = p.kvHeads * p.hd, share = p.heads / p.kvHeads, perGroup = p.heads / p.groups;
    const float* rows = fresh ? p.kNew + (size_t(b) * p.nodes + (j - length)) * kvDim : p.k + (size_t(b) * p.capacity + j) * kvDim;
    float sum = 0.0f;
    for (int h = g * perGroup; h < (g + 1) * perGroup; ++h) {
        const float* kr = rows + size_t(h / share) * p.hd;
        for (int i = 0; i < count; ++i) {
            if (fresh && !(newRowsSeen(p, b, i, count) >> (j - length) & 1)) continue;
            const float* q = p.q + (size_t(b) * p.nodes + i) * p.heads * p.hd + size_t(h) * p.hd;
            float dot = 0.0f;
            for (int d = lane; d < p.hd; d += 64) dot += q[d] * kr[d];
            const float s = waveSum(dot) * p.scale;
            const size_t stat = (size_t(b) * p.heads + h) * p.nodes + i;
            if (p.l[stat] > 0.0f) sum += expf(s - p.m[stat]) / p.l[stat];
        }
    }
    if (lane == 0) p.weightsOut[row] = (!fresh && p.weightsIn ? p.weightsIn[row] : 0.0f) + sum;
}

struct KeyWeightParams {
    const float* q; const float* k; const float* m; const float* l;
    const int* counts; const float* weightsIn; float* weightsOut;
    int batch, heads, kvHeads, groups, newLen, totalLen, kvRows, hd, oldLen, weightRows;
    float scale;
};

// One wavefront per (sequence, group, key).
__global__ void __launch_bounds__(256) keyWeightsKernel(KeyWeightParams p) {
    const int lane = threadIdx.x & 63;
    const size_t row = size_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (row >= size_t(p.batch) * p.groups * p.totalLen) return;
    const int j = int(row % p.totalLen), g = int(row / p.totalLen % p.groups), b = int(row / p.totalLen / p.groups);
    const int count = p.counts ? min(max(p.counts[b], 0), p.newLen) : p.newLen;
    const int share = p.heads / p.kvHeads, perGroup = p.heads / p.groups;
    float sum = 0.0f;
    for (int h = g * perGroup; h < (g + 1) * perGroup; ++h) {
        const float* kr = p.k + (size_t(b) * p.kvRows + j) * p.kvHeads * p.hd + size_t(h / share) * p.hd;
        for (int i = max(0, j - p.oldLen); i < count; ++i) {
            const float* q = p.q + (size_t(b) * p.newLen + i) * p.heads * p.hd + size_t(h) * p.hd;
            float dot = 0.0f;
            for (int d = lane; d < p.hd; d += 64) dot += q[d] * kr[d];
            const float s = waveSum(dot) * p.scale;
            const size_t stat = (size_t(b) * p.heads + h) * p.newLen + i;
            if (p.l[stat] > 0.0f) sum += expf(s - p.m[stat]) / p.l[stat];
        }
    }
    const size_t at = (size_t(b) * p.groups + g) * p.weightRows + j;
    if (lane == 0) p.weightsOut[at] = (p.weightsIn ? p.weightsIn[at] : 0.0f) + sum;
}

int checkHeads(const char* fn, size_t heads, size_t kvHeads, size_t groups, size_t headDim) {
    if (heads == 0 || kvHeads == 0 || heads % kvHeads != 0)
        return failInvalid(fn, "kvHeads (" + std::to_string(kvHeads) + ") must divide the number of heads (" + std::to_string(heads) + ")");
    if (groups == 0 || kvHeads % groups != 0)
        return failInvalid(fn, "groups (" + std::to_string(groups) + ") must divide kvHeads (" + std::to_string(kvHeads) + ")");
    if (headDim > 256) return failInvalid(fn, "headDim (" + std::to_string(headDim) + ") exceeds the supported limit (256)");
    if (heads >= (size_t(1) << 16)) return failInvalid(fn, "shape too large");
    return BF_OK;
}

int treeAttention(const char* fn, TreeParams p, size_t batch, size_t heads, size_t kvHeads, size_t groups, size_t nodes, size_t capacity,
                  size_t headDim, bool weights, bf_stream_t stream) {
    int st = checkHeads(fn, heads, kvHeads, groups, headDim);
    if (st != BF_OK) return st;
    if (nodes > 64) return failInvalid(fn, "a tree has at most 64 nodes, got " + std::to_string(nodes));
    if (batch >= (size_t(1) << 16) || capacity >= (size_t(1) << 30)) return failInvalid(fn, "shape too large");
    if (batch == 0 || nodes == 0 || headDim == 0) return BF_OK;
    if (!p.q || !p.kNew || !p.vNew || !p.lengths || !p.out || (capacity != 0 && (!p.k || !p.v)) || (weights && capacity != 0 && !p.weightsOut))
        return failInvalid(fn, "NULL pointer");
    p.batch = int(batch); p.heads = int(heads); p.kvHeads = int(kvHeads); p.groups = int(groups); p.nodes = int(nodes);
    p.capacity = int(capacity); p.hd = int(headDim);
    hipStream_t s = asStream(stream);
    const size_t stats = batch * heads * nodes;
    Scratch own(p.m && p.l ? 0 : 2 * stats * sizeof(float));
    if (own.status != BF_OK) return own.status;
    if (!p.m) p.m = own.as<float>();
    if (!p.l) p.l = own.as<float>() + stats;
    treeAttentionKernel<<<unsigned((stats + 3) / 4), 256, 0, s>>>(p);
    BF_LAUNCH_CHECK();
    if (weights && capacity != 0) {
        treeWeightsKernel<<<unsigned((batch * groups * capacity + 3) / 4), 256, 0, s>>>(p);
        BF_LAUNCH_CHECK();
    }
    return BF_OK;
}

}  // namespace
}  // namespace bf

using namespace bf;

extern "C" {

int bf_hip_attention_tree(const float* q, const float* kNew, const float* vNew, const float* kCache, const float* vCache, const int* lengths,
                          const int* counts, const uint64_t* visible, float* out, float* m, float* l, size_t batch, size_t heads, size_t kvHeads,
                          size_t nodes, size_t capacity, size_t headDim, float scale, bf_stream_t stream) {
    TreeParams p{};
    p.q = q; p.kNew = kNew; p.vNew = vNew; p.k = kCache; p.v = vCache; p.lengths = lengths; p.counts = counts;
    p.visible = reinterpret_cast<const unsigned long long*>(visible);
    p.out = out; p.m = m; p.l = l; p.scale = scale;
    return treeAttention(__func__, p, batch, heads, kvHeads, 1, nodes, capacity, headDim, false, stream);
}

int bf_hip_attention_tree_weights(const float* q, const float* kNew, const float* vNew, const float* kCache, const float* vCache, const int* lengths,
                                  const int* counts, const uint64_t* visible, float* out, float* m, float* l, const float* weightsIn,
                                  float* weightsOut, size_t batch, size_t heads, size_t kvHeads, size_t groups, size_t nodes, size_t capacity,
                                  size_t headDim, float scale, bf_stream_t stream) {
    TreeParams p{};
    p.q = q; p.kNew = kNew; p.vNew = vNew; p.k = kCache; p.v = vCache; p.lengths = lengths; p.counts = counts;
    p.visible = reinterpret_cast<const unsigned long long*>(visible);
    p.out = out; p.m = m; p.l = l; p.weightsIn = weightsIn; p.weightsOut = weightsOut; p.scale = scale;
    return treeAttention(__func__, p, batch, heads, kvHeads, groups, nodes, capacity, headDim, true, stream);
}

int bf_hip_attention_key_weights(const float* q, const float* k, const float* m, const float* l, const int* counts, const float* weightsIn,
                                 float* weightsOut, size_t batch, size_t heads, size_t kvHeads, size_t groups, size_t newLen, size_t totalLen,
                                 size_t kvRows, size_t headDim, float scale, size_t oldLen, size_t weightRows, bf_stream_t stream) {
    int st = checkHeads(__func__, heads, kvHeads, groups, headDim);
    if (st != BF_OK) return st;
    BF_REQUIRE(kvRows >= totalLen && weightRows >= totalLen, "kvRows and weightRows must be at least totalLen");
    BF_REQUIRE(batch < (size_t(1) << 16) && kvRows < (size_t(1) << 30) && weightRows < (size_t(1) << 30) && newLen < (size_t(1) << 30) &&
                   oldLen < (size_t(1) << 30), "shape too large");
    if (batch == 0 || totalLen == 0) return BF_OK;
    BF_REQUIRE(weightsOut && ((q && k && m && l) || newLen == 0 || headDim == 0), "NULL pointer");
    KeyWeightParams p{};
    p.q = q; p.k = k; p.m = m; p.l = l; p.counts = counts; p.weightsIn = weightsIn; p.weightsOut = weightsOut;
    p.batch = int(batch); p.heads = int(heads); p.kvHeads = int(kvHeads); p.groups = int(groups); p.newLen = headDim == 0 ? 0 : int(newLen);
    p.totalLen = int(totalLen); p.kvRows = int(kvRows); p.hd = int(headDim); p.oldLen = int(oldLen); p.weightRows = int(weightRows);
    p.scale = scale;
    keyWeightsKernel<<<unsigned((batch * groups * totalLen + 3) / 4), 256, 0, asStream(stream)>>>(p);
    BF_LAUNCH_CHECK();
    return BF_OK;
}

}  // extern "C"

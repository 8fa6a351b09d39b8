#pragma once
// Decoding over caches with a length per sequence: attention of drafted trees, the attention weight of cached rows,
// eviction by it, verification of a draft.  No counterparts in the reference, whose generation loop takes one token at a
// time and keeps every position (src/main.cpp:594-617).  The semantics are those of the C entry points (bf_hip.h).
#include <cstddef>
#include <cstdint>
#include <string>
#include <utility>
#include <vector>

#include "blackforge/backend/hip/device_tensor.hpp"
#include "blackforge/backend/hip/fused_attention.hpp"

namespace blackforge::backend::hip {

// A small array of integers on the device (lengths, counts, node indices: int; masks of tree nodes: std::uint64_t).
template <typename T>
class DeviceArray {
public:
    DeviceArray() = default;
    explicit DeviceArray(std::size_t count) : store_({(count * sizeof(T) + sizeof(float) - 1) / sizeof(float)}), count_(count) {}
    explicit DeviceArray(const std::vector<T>& host) : DeviceArray(host.size()) {
        check(bf_hip_memcpy_h2d(store_.data(), host.data(), host.size() * sizeof(T)));
    }
    [[nodiscard]] T* data() { return reinterpret_cast<T*>(store_.data()); }
    [[nodiscard]] const T* data() const { return reinterpret_cast<const T*>(store_.data()); }
    [[nodiscard]] std::size_t size() const { return count_; }
    [[nodiscard]] std::vector<T> toHost() const {
        std::vector<T> host(count_);
        check(bf_hip_memcpy_d2h(host.data(), store_.data(), count_ * sizeof(T)));
        return host;
    }

private:
    DeviceTensor store_;
    std::size_t count_ = 0;
};

// One attention layer's keys and values, [batch, capacity, kvHeads * headDim], and, if account is kept of it, the attention
// weight of their rows, [batch, groups, capacity] (an empty tensor: none).  How many rows of a sequence are in use is the
// same for all layers of a model and lies beside them, one int per sequence on the device.
struct DecodeLayer {
    DeviceTensor k;
    DeviceTensor v;
    DeviceTensor weights;

    DecodeLayer(std::size_t batch, std::size_t capacity, std::size_t dim, std::size_t groups = 0)
        : k({batch, capacity, dim}), v({batch, capacity, dim}) {
        if (groups != 0) weights = DeviceTensor::zeros({batch, groups, capacity});
    }
    [[nodiscard]] std::size_t batch() const { return k.dim(0); }
    [[nodiscard]] std::size_t capacity() const { return k.dim(1); }
};

// Masks for treeAttention from the nodes' parents, [batch, nodes] (a parent comes before its child, a root's is negative):
// a node sees its ancestors and itself.
inline std::vector<std::uint64_t> treeVisibility(const std::vector<int>& parents, std::size_t nodes) {
    require(nodes >= 1 && nodes <= 64 && parents.size() % nodes == 0, "treeVisibility: one parent per node, at most 64 nodes");
    std::vector<std::uint64_t> masks(parents.size());
    for (std::size_t at = 0; at < parents.size(); ++at) {
        const std::size_t node = at % nodes;
        require(parents[at] < static_cast<int>(node), "treeVisibility: node " + std::to_string(node) + " comes before its parent");
        masks[at] = std::uint64_t{1} << node;
        if (parents[at] >= 0) masks[at] |= masks[at - node + static_cast<std::size_t>(parents[at])];
    }
    return masks;
}

// Attention of new tokens, the nodes of a tree (visible == nullptr: of a chain), over a layer's cache; their keys and values
// are not in the cache yet.  A layer that keeps account of the weights has them updated.  Rows past counts[b] are zero.
inline FusedAttentionForwardResult treeAttention(const DeviceTensor& q, const DeviceTensor& kNew, const DeviceTensor& vNew, DecodeLayer& layer,
                                                 const DeviceArray<int>& lengths, std::size_t numHeads, std::size_t kvHeads, float scaleFactor,
                                                 const DeviceArray<int>* counts = nullptr, const DeviceArray<std::uint64_t>* visible = nullptr) {
    require(q.rank() == 3 && numHeads != 0 && q.dim(2) % numHeads == 0, "treeAttention: q must be [batch, nodes, heads * headDim]");
    const std::size_t batch = q.dim(0), nodes = q.dim(1), headDim = q.dim(2) / numHeads, kvDim = kvHeads * headDim;
    require(kNew.shape() == std::vector<std::size_t>({batch, nodes, kvDim}) && vNew.shape() == kNew.shape(), "treeAttention: incompatible new keys and values");
    require(layer.k.rank() == 3 && layer.k.shape() == layer.v.shape() && layer.batch() == batch && layer.k.dim(2) == kvDim, "treeAttention: incompatible cache");
    require(lengths.size() == batch && (counts == nullptr || counts->size() == batch) && (visible == nullptr || visible->size() == batch * nodes),
            "treeAttention: one length and one count per sequence, one mask per node");
    auto make = [&](std::vector<std::size_t> shape) { return counts == nullptr ? DeviceTensor(std::move(shape)) : DeviceTensor::zeros(std::move(shape)); };
    FusedAttentionForwardResult r{make(q.shape()), make({batch, numHeads, nodes}), make({batch, numHeads, nodes})};
    const int* c = counts != nullptr ? counts->data() : nullptr;
    const std::uint64_t* seen = visible != nullptr ? visible->data() : nullptr;
    if (layer.weights.rank() == 3) {
        require(layer.weights.dim(0) == batch && layer.weights.dim(2) == layer.capacity(), "treeAttention: weights must be [batch, groups, capacity]");
        check(bf_hip_attention_tree_weights(q.data(), kNew.data(), vNew.data(), layer.k.data(), layer.v.data(), lengths.data(), c, seen, r.output.data(),
                                            r.m.data(), r.l.data(), layer.weights.data(), layer.weights.data(), batch, numHeads, kvHeads,
                                            layer.weights.dim(1), nodes, layer.capacity(), headDim, scaleFactor, nullptr));
    } else {
        check(bf_hip_attention_tree(q.data(), kNew.data(), vNew.data(), layer.k.data(), layer.v.data(), lengths.data(), c, seen, r.output.data(), r.m.data(),
                                    r.l.data(), batch, numHeads, kvHeads, nodes, layer.capacity(), headDim, scaleFactor, nullptr));
    }
    return r;
}

// The weight that the keys of a pass that has run received (fusedAttentionForward's q, k, m, l), added to weights [batch,
// groups, rows >= k's]; queries i >= counts[b] do not count.
inline void attentionKeyWeights(const DeviceTensor& q, const DeviceTensor& k, const DeviceTensor& m, const DeviceTensor& l, std::size_t numHeads,
                                std::size_t kvHeads, float scaleFactor, std::size_t oldLen, DeviceTensor& weights,
                                const DeviceArray<int>* counts = nullptr) {
    require(q.rank() == 3 && k.rank() == 3 && numHeads != 0 && q.dim(2) % numHeads == 0 && k.dim(0) == q.dim(0) &&
                k.dim(2) == kvHeads * (q.dim(2) / numHeads), "attentionKeyWeights: incompatible q and k");
    const std::size_t batch = q.dim(0), newLen = q.dim(1);
    require(m.shape() == std::vector<std::size_t>({batch, numHeads, newLen}) && l.shape() == m.shape(), "attentionKeyWeights: statistics must be [batch, heads, newLen]");
    require(weights.rank() == 3 && weights.dim(0) == batch && weights.dim(2) >= k.dim(1), "attentionKeyWeights: weights must be [batch, groups, rows]");
    require(counts == nullptr || counts->size() == batch, "attentionKeyWeights: one count per sequence");
    check(bf_hip_attention_key_weights(q.data(), k.data(), m.data(), l.data(), counts != nullptr ? counts->data() : nullptr, weights.data(), weights.data(),
                                       batch, numHeads, kvHeads, weights.dim(1), newLen, k.dim(1), k.dim(1), q.dim(2) / numHeads, scaleFactor, oldLen,
                                       weights.dim(2), nullptr));
}

// Every layer's cache cut down in place to `budget` rows a sequence, the most recent and the heaviest, and the lengths with
// them.  The lengths are cut with the last layer, so all are checked before the first: cut in part, the caches and their
// lengths would no longer agree.
inline void evictKeyValues(std::vector<DecodeLayer>& layers, DeviceArray<int>& lengths, std::size_t kvHeads, std::size_t budget, std::size_t recent) {
    require(kvHeads != 0 && recent <= budget, "evictKeyValues: more recent rows than the budget holds, or no heads");
    for (const DecodeLayer& x : layers) {
        require(x.k.rank() == 3 && x.v.shape() == x.k.shape() && x.weights.rank() == 3 && x.weights.dim(0) == x.batch() &&
                    x.weights.dim(2) == x.capacity() && lengths.size() == x.batch(),
                "evictKeyValues: every layer needs weights [batch, groups, capacity], every sequence a length");
        require(x.k.dim(2) % kvHeads == 0 && x.weights.dim(1) != 0 && kvHeads % x.weights.dim(1) == 0, "evictKeyValues: incompatible heads and groups");
        require(budget <= x.capacity(), "evictKeyValues: the budget does not fit the capacity");
    }
    for (std::size_t i = 0; i < layers.size(); ++i) {
        DecodeLayer& x = layers[i];
        check(bf_hip_kv_evict(x.k.data(), x.v.data(), x.weights.data(), lengths.data(), x.k.data(), x.v.data(), x.weights.data(),
                              i + 1 == layers.size() ? lengths.data() : nullptr, nullptr, x.batch(), kvHeads, x.weights.dim(1), x.k.dim(2) / kvHeads,
                              x.capacity(), x.capacity(), budget, recent, nullptr));
    }
}

struct AcceptedPath {
    DeviceArray<int> path;     // [batch, nodes], -1 past the path
    DeviceArray<int> counts;   // [batch]
    DeviceTensor next;         // [batch] token ids
};

// The path of a drafted tree that greedy choices confirm: logits [batch, nodes, vocab], tokens [batch, nodes].
inline AcceptedPath treeAccept(const DeviceTensor& logits, const DeviceTensor& tokens, const DeviceArray<int>& parents,
                               const DeviceArray<int>* counts = nullptr) {
    require(logits.rank() == 3 && tokens.elementCount() == logits.dim(0) * logits.dim(1) && parents.size() == tokens.elementCount() &&
                (counts == nullptr || counts->size() == logits.dim(0)), "treeAccept: needs logits [batch, nodes, vocab] and a token and a parent per node");
    const std::size_t batch = logits.dim(0), nodes = logits.dim(1);
    AcceptedPath r{DeviceArray<int>(batch * nodes), DeviceArray<int>(batch), DeviceTensor::zeros({batch})};
    if (nodes == 0) check(bf_hip_fill_zero(r.counts.data(), batch * sizeof(int), nullptr));   // the call writes nothing: no node is accepted
    check(bf_hip_tree_accept(logits.data(), tokens.data(), parents.data(), counts != nullptr ? counts->data() : nullptr, r.path.data(), r.counts.data(),
                             r.next.data(), batch, nodes, logits.dim(2), nullptr));
    return r;
}

// The accepted nodes' keys and values, of every layer [batch, nodes, dim], appended to its cache; the lengths move on.
inline void commitPath(std::vector<DecodeLayer>& layers, const std::vector<DeviceTensor>& kNew, const std::vector<DeviceTensor>& vNew,
                       const AcceptedPath& accepted, DeviceArray<int>& lengths) {
    require(!layers.empty() && kNew.size() == layers.size() && vNew.size() == layers.size(), "commitPath: one pair of tensors per layer");
    const std::size_t batch = layers[0].batch(), capacity = layers[0].capacity(), dim = layers[0].k.dim(2);
    const std::size_t groups = layers[0].weights.rank() == 3 ? layers[0].weights.dim(1) : 0;
    require(kNew[0].rank() == 3 && lengths.size() == batch && accepted.counts.size() == batch && accepted.path.size() == batch * kNew[0].dim(1) &&
                (groups == 0 || dim % groups == 0), "commitPath: one path per sequence");
    std::vector<float*> k, v, w;
    std::vector<const float*> kn, vn;
    for (std::size_t i = 0; i < layers.size(); ++i) {
        DecodeLayer& x = layers[i];
        require(x.k.shape() == layers[0].k.shape() && x.v.shape() == x.k.shape() && kNew[i].shape() == std::vector<std::size_t>({batch, kNew[0].dim(1), dim}) &&
                    vNew[i].shape() == kNew[i].shape() && (groups == 0 ? x.weights.rank() != 3 : x.weights.shape() == std::vector<std::size_t>({batch, groups, capacity})),
                "commitPath: the layers differ in shape");
        k.push_back(x.k.data());
        v.push_back(x.v.data());
        kn.push_back(kNew[i].data());
        vn.push_back(vNew[i].data());
        if (groups != 0) w.push_back(x.weights.data());
    }
    const std::size_t heads = groups == 0 ? 1 : groups;   // how the rows divide into heads does not matter to the copy
    check(bf_hip_kv_commit(k.data(), v.data(), kn.data(), vn.data(), groups != 0 ? w.data() : nullptr, layers.size(), accepted.path.data(),
                           accepted.counts.data(), lengths.data(), lengths.data(), batch, heads, heads, kNew[0].dim(1), capacity, dim / heads, nullptr));
}

}  // namespace blackforge::backend::hip

// Tests of decode_cache.hpp: what is refused leaves every layer and the lengths as they were.
// Built by blackforge_amd/host/Makefile, run on a GPU by tests/test_gpu_decode_cache_layers.py.
#include <cstdio>
#include <functional>
#include <stdexcept>
#include <vector>

#include "blackforge/backend/hip/decode_cache.hpp"

namespace hip = blackforge::backend::hip;
using blackforge::runtime::Tensor;
using hip::DeviceTensor;

namespace {
int failures = 0;
void expect(bool ok, const char* what) {
    if (!ok) { ++failures; std::printf("FAILED: %s\n", what); }
}
DeviceTensor counted(std::vector<std::size_t> shape) {   // every element its own value
    std::size_t n = 1;
    for (std::size_t d : shape) n *= d;
    std::vector<float> x(n);
    for (std::size_t i = 0; i < n; ++i) x[i] = static_cast<float>(i * 7 % 1009);
    return DeviceTensor::fromHost(Tensor(std::move(shape), std::move(x)));
}

// the third of three layers changed by `spoil`, evicted: refused, nothing cut
void refused(const char* what, const std::function<void(hip::DecodeLayer&)>& spoil, std::size_t budget = 12, std::size_t recent = 3, std::size_t kvHeads = 4) {
    const std::size_t batch = 2, capacity = 30, dim = 16, groups = 2;
    std::vector<hip::DecodeLayer> layers;
    for (int i = 0; i < 3; ++i) {
        layers.emplace_back(batch, capacity, dim, groups);
        layers.back().k = counted({batch, capacity, dim});
        layers.back().v = counted({batch, capacity, dim});
        layers.back().weights = counted({batch, groups, capacity});
    }
    spoil(layers[2]);
    hip::DeviceArray<int> lengths(std::vector<int>{30, 20});
    const Tensor k = layers[0].k.toHost(), v = layers[0].v.toHost(), w = layers[0].weights.toHost();
    bool thrown = false;
    try {
        hip::evictKeyValues(layers, lengths, kvHeads, budget, recent);
    } catch (const std::invalid_argument&) {
        thrown = true;
    }
    expect(thrown, what);
    for (int i = 0; i < 2; ++i)
        expect(layers[i].k.toHost().data() == k.data() && layers[i].v.toHost().data() == v.data() && layers[i].weights.toHost().data() == w.data(), what);
    expect(lengths.toHost() == std::vector<int>({30, 20}), what);
}
}  // namespace

int main() {
    const auto keep = [](hip::DecodeLayer&) {};
    refused("values of another shape", [](hip::DecodeLayer& x) { x.v = counted({2, 29, 16}); });
    refused("weights of fewer sequences", [](hip::DecodeLayer& x) { x.weights = counted({1, 2, 30}); });
    refused("weights of another capacity", [](hip::DecodeLayer& x) { x.weights = counted({2, 2, 29}); });
    refused("groups that do not divide the heads", [](hip::DecodeLayer& x) { x.weights = counted({2, 3, 30}); });
    refused("no weights", [](hip::DecodeLayer& x) { x.weights = DeviceTensor(); });
    refused("a capacity below the budget", [](hip::DecodeLayer& x) {
        x.k = counted({2, 11, 16});
        x.v = counted({2, 11, 16});
        x.weights = counted({2, 2, 11});
    });
    refused("rows that do not divide into heads", [](hip::DecodeLayer& x) {
        x.k = counted({2, 30, 18});
        x.v = counted({2, 30, 18});
    });
    refused("another number of sequences", [](hip::DecodeLayer& x) {
        x.k = counted({3, 30, 16});
        x.v = counted({3, 30, 16});
        x.weights = counted({3, 2, 30});
    });
    refused("a budget past the capacity", keep, 31);
    refused("more recent rows than the budget", keep, 12, 13);
    refused("no heads", keep, 12, 3, 0);

    // a draft without nodes: none is accepted, whatever the counts' memory held before
    { const hip::DeviceArray<int> dirty(std::vector<int>{9, 9, 9}); }
    const auto accepted = hip::treeAccept(DeviceTensor({3, 0, 50}), DeviceTensor({3, 0}), hip::DeviceArray<int>(0));
    expect(accepted.counts.toHost() == std::vector<int>({0, 0, 0}), "treeAccept without nodes");
    std::printf(failures == 0 ? "all passed\n" : "%d failed\n", failures);
    return failures != 0;
}

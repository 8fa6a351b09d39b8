// Tests of decode_cache.hpp: a two-layer round of draft, verification, append and eviction against plain loops on the host.
// Built by blackforge_amd/host/Makefile, run on a GPU by tests/test_gpu_decode_cache.py.
#include <algorithm>
#include <cmath>
#include <cstdio>
#include <random>
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
std::mt19937 gen(7);
std::vector<float> normal(std::size_t n) {
    std::normal_distribution<float> d;
    std::vector<float> x(n);
    for (float& y : x) y = d(gen);
    return x;
}
DeviceTensor dev(std::vector<std::size_t> shape, const std::vector<float>& data) { return DeviceTensor::fromHost(Tensor(std::move(shape), data)); }
}  // namespace

int main() {
    const std::size_t batch = 2, heads = 4, kvHeads = 2, hd = 32, kvDim = kvHeads * hd, dim = heads * hd, capacity = 64, nodes = 4, vocab = 11;
    const std::vector<int> lengths = {40, 9}, parents = {-1, 0, 0, 2, -1, 0, 1, 2};
    const auto masks = hip::treeVisibility(parents, nodes);
    expect(masks == std::vector<std::uint64_t>({1, 3, 5, 13, 1, 3, 7, 15}), "treeVisibility");
    bool thrown = false;
    try { (void)hip::treeVisibility({-1, 1}, 2); } catch (const std::invalid_argument&) { thrown = true; }
    expect(thrown, "treeVisibility refuses a node before its parent");

    std::vector<hip::DecodeLayer> layers;
    std::vector<std::vector<float>> k, v, kn, vn;
    std::vector<DeviceTensor> kNew, vNew;
    for (int i = 0; i < 2; ++i) {
        k.push_back(normal(batch * capacity * kvDim));
        v.push_back(normal(batch * capacity * kvDim));
        kn.push_back(normal(batch * nodes * kvDim));
        vn.push_back(normal(batch * nodes * kvDim));
        layers.emplace_back(batch, capacity, kvDim, kvHeads);
        layers.back().k = dev({batch, capacity, kvDim}, k.back());
        layers.back().v = dev({batch, capacity, kvDim}, v.back());
        kNew.push_back(dev({batch, nodes, kvDim}, kn.back()));
        vNew.push_back(dev({batch, nodes, kvDim}, vn.back()));
    }
    hip::DeviceArray<int> devLengths(lengths), devParents(parents);
    hip::DeviceArray<std::uint64_t> devMasks(masks);
    const std::vector<float> q = normal(batch * nodes * dim);
    const DeviceTensor devQ = dev({batch, nodes, dim}, q);
    const float scale = 1.0F / std::sqrt(static_cast<float>(hd));

    std::vector<std::vector<double>> received(2, std::vector<double>(batch * kvHeads * capacity, 0.0));
    for (std::size_t i = 0; i < 2; ++i) {
        const auto got = hip::treeAttention(devQ, kNew[i], vNew[i], layers[i], devLengths, heads, kvHeads, scale, nullptr, &devMasks);
        const Tensor out = got.output.toHost();
        double worst = 0.0;
        for (std::size_t b = 0; b < batch; ++b)
            for (std::size_t h = 0; h < heads; ++h)
                for (std::size_t n = 0; n < nodes; ++n) {
                    const std::size_t L = static_cast<std::size_t>(lengths[b]), g = h / 2;
                    std::vector<double> s(L + nodes, -INFINITY);
                    double top = -INFINITY, total = 0.0;
                    auto row = [&](const std::vector<float>& c, const std::vector<float>& f, std::size_t j) {
                        return j < L ? &c[(b * capacity + j) * kvDim + g * hd] : &f[(b * nodes + j - L) * kvDim + g * hd];
                    };
                    for (std::size_t j = 0; j < L + nodes; ++j) {
                        if (j >= L && !(masks[b * nodes + n] >> (j - L) & 1)) continue;
                        s[j] = 0.0;
                        for (std::size_t d = 0; d < hd; ++d) s[j] += double(q[(b * nodes + n) * dim + h * hd + d]) * row(k[i], kn[i], j)[d];
                        s[j] *= scale;
                        top = std::max(top, s[j]);
                    }
                    for (double& x : s) total += x = std::exp(x - top);
                    for (std::size_t j = 0; j < L + nodes; ++j) received[i][(b * kvHeads + g) * capacity + j] += s[j] / total;
                    for (std::size_t d = 0; d < hd; ++d) {
                        double want = 0.0;
                        for (std::size_t j = 0; j < L + nodes; ++j) want += s[j] / total * row(v[i], vn[i], j)[d];
                        worst = std::max(worst, std::fabs(want - double(out.data()[(b * nodes + n) * dim + h * hd + d])));
                    }
                }
        expect(worst < 2e-5, "treeAttention");   // 44 rows, scores below 10: 2 (3 * 36 * 10 + 60) 2^-24 times 4 at the very most
    }

    // logits that follow node 0 -> 2 -> 3 in sequence 0 and 0 -> 1 in sequence 1
    std::vector<float> logits(batch * nodes * vocab, 0.0F);
    const std::vector<float> tokens = {5, 1, 7, 3, 5, 2, 4, 6};
    auto choose = [&](std::size_t b, std::size_t n, std::size_t token) { logits[(b * nodes + n) * vocab + token] = 1.0F; };
    choose(0, 0, 7); choose(0, 2, 3); choose(0, 3, 9);
    choose(1, 0, 2); choose(1, 1, 10);
    const auto accepted = hip::treeAccept(dev({batch, nodes, vocab}, logits), dev({batch, nodes}, tokens), devParents);
    expect(accepted.path.toHost() == std::vector<int>({0, 2, 3, -1, 0, 1, -1, -1}), "treeAccept's path");
    expect(accepted.counts.toHost() == std::vector<int>({3, 2}), "treeAccept's counts");
    expect(accepted.next.toHost().data() == std::vector<float>({9, 10}), "treeAccept's next token");
    hip::commitPath(layers, kNew, vNew, accepted, devLengths);
    expect(devLengths.toHost() == std::vector<int>({43, 11}), "commitPath's lengths");
    const std::vector<std::vector<std::size_t>> paths = {{0, 2, 3}, {0, 1}};
    for (std::size_t i = 0; i < 2; ++i) {
        for (std::size_t b = 0; b < batch; ++b)
            for (std::size_t n = 0; n < paths[b].size(); ++n) {
                const std::size_t at = (b * capacity + static_cast<std::size_t>(lengths[b]) + n) * kvDim, from = (b * nodes + paths[b][n]) * kvDim;
                std::copy_n(&kn[i][from], kvDim, &k[i][at]);
                std::copy_n(&vn[i][from], kvDim, &v[i][at]);
                for (std::size_t g = 0; g < kvHeads; ++g) {
                    double* w = &received[i][(b * kvHeads + g) * capacity + static_cast<std::size_t>(lengths[b])];
                    w[n] = w[paths[b][n]];
                }
            }
        expect(layers[i].k.toHost().data() == k[i] && layers[i].v.toHost().data() == v[i], "commitPath");
        const Tensor w = layers[i].weights.toHost();
        double worst = 0.0;
        for (std::size_t b = 0; b < batch; ++b)
            for (std::size_t g = 0; g < kvHeads; ++g)
                for (std::size_t j = 0; j < static_cast<std::size_t>(lengths[b]) + paths[b].size(); ++j)
                    worst = std::max(worst, std::fabs(received[i][(b * kvHeads + g) * capacity + j] - double(w.data()[(b * kvHeads + g) * capacity + j])));
        expect(worst < 2e-5, "weights after commitPath");
    }

    const std::size_t budget = 12, recent = 4;
    std::vector<Tensor> before;
    for (auto& x : layers) before.push_back(x.weights.toHost());
    hip::evictKeyValues(layers, devLengths, kvHeads, budget, recent);
    expect(devLengths.toHost() == std::vector<int>({12, 11}), "evictKeyValues' lengths");
    for (std::size_t i = 0; i < 2; ++i) {
        const Tensor gotK = layers[i].k.toHost(), gotV = layers[i].v.toHost(), gotW = layers[i].weights.toHost();
        bool same = true;
        for (std::size_t g = 0; g < kvHeads; ++g) {
            std::vector<std::size_t> order(43 - recent), kept;
            for (std::size_t j = 0; j < order.size(); ++j) order[j] = j;
            const float* w = &before[i].data()[g * capacity];
            std::stable_sort(order.begin(), order.end(), [&](std::size_t a, std::size_t b) { return w[a] > w[b]; });
            kept.assign(order.begin(), order.begin() + static_cast<long>(budget - recent));
            std::sort(kept.begin(), kept.end());
            for (std::size_t j = 43 - recent; j < 43; ++j) kept.push_back(j);
            for (std::size_t j = 0; j < budget; ++j) {
                same = same && gotW.data()[g * capacity + j] == w[kept[j]];
                for (std::size_t d = 0; d < hd; ++d)
                    same = same && gotK.data()[j * kvDim + g * hd + d] == k[i][kept[j] * kvDim + g * hd + d] &&
                           gotV.data()[j * kvDim + g * hd + d] == v[i][kept[j] * kvDim + g * hd + d];
            }
        }
        expect(same, "evictKeyValues");
    }

    // a prompt's account: two queries, the second sees both keys
    const DeviceTensor pq = dev({1, 2, hd}, normal(2 * hd)), pk = dev({1, 2, hd}, normal(2 * hd)), pv = dev({1, 2, hd}, normal(2 * hd));
    const auto full = hip::fusedAttentionForward(pq, pk, pv, 1, scale, 0);
    DeviceTensor w = DeviceTensor::zeros({1, 1, 5});
    hip::attentionKeyWeights(pq, pk, full.m, full.l, 1, 1, scale, 0, w);
    const Tensor got = w.toHost();
    expect(std::fabs(got.data()[0] + got.data()[1] - 2.0F) < 1e-5F && got.data()[0] > 1.0F && got.data()[2] == 0.0F, "attentionKeyWeights");
    thrown = false;
    try { hip::attentionKeyWeights(pq, pk, full.m, full.l, 1, 2, scale, 0, w); } catch (const std::invalid_argument&) { thrown = true; }
    expect(thrown, "attentionKeyWeights refuses heads that do not fit");
    std::printf(failures == 0 ? "all passed\n" : "%d failed\n", failures);
    return failures != 0;
}

// Upkeep of a key/value cache: eviction by accumulated attention weight, and the verification of a drafted tree (which
// of its nodes the model's own choices confirm, and their rows appended to the caches of all layers).
//
// All of it moves rows or reads logits once: HBM-bound where it is large, launch-bound where it is not.  No kernel adds
// floating-point numbers, so every result is exact.
#include "common.hpp"

#include <algorithm>
#include <climits>
#include <initializer_list>

namespace bf {
namespace {

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- eviction ----------------------------------------------------------------------------------
struct EvictParams {
    const float* k; const float* v; const float* weights; const int* lengths;
    float* kOut; float* vOut; float* weightsOut; int* lengthsOut;
    int* kept;       // [batch, groups, budget] source rows, ascending
    int* left;       // [batch] rows that remain, written by the selection for the kernel that moves rows
    int batch, groups, capacity, outCapacity, budget, recent;
    int slab;        // floats of a row that belong to one group
};

// Unsigned integers in the order of the floats; NaN as -infinity, -0 as +0
__device__ __forceinline__ unsigned weightKey(float w) {
    if (w != w) w = -INFINITY;
    const unsigned u = __float_as_uint(w + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// One workgroup per (sequence, group): which rows stay.  The rows before the most recent `recent` compete for budget -
// recent places.  Three passes over their weights, 11 + 11 + 10 bits from the top, find the key of the last place (each
// pass a histogram of the next digit among the keys that share the digits found so far); equal keys go to the lowest
// rows.  Two more passes write the kept rows in order: the wavefronts own consecutive stretches, count, and then emit at
// the offsets that the counts before them give.  Last the kept rows' weights move up, a tile at a time, all of a
// tile's reads before its writes: row i comes from a row at or after i, so a call in place overwrites nothing unread.
// With NK > 0 the capacity is at most 1024 NK and a thread keeps its NK keys in registers, so the weights are read once
// (8 sequences of 16384 rows, 16 groups: 33 us reading them in every pass, 17 with NK = 16); NK = 0 reads them again.
template <int NK>
__global__ void __launch_bounds__(1024) evictSelectKernel(EvictParams p) {
    constexpr int BINS = 2048, WAVES = 16;
    __shared__ unsigned hist[BINS];
    __shared__ unsigned total[WAVES];
    __shared__ unsigned sDigit, sAbove;
    __shared__ int sGreater[WAVES], sEqual[WAVES];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int b = blockIdx.x / p.groups, g = blockIdx.x % p.groups;
    const int length = min(max(p.lengths[b], 0), p.capacity);
    const int left = min(length, p.budget);
    const float* w = p.weights + (size_t(b) * p.groups + g) * p.capacity;
    int* kept = p.kept + (size_t(b) * p.groups + g) * p.budget;
    if (g == 0 && t == 0) p.left[b] = left;
    if (length <= p.budget) {
        for (int i = t; i < left; i += 1024) kept[i] = i;
    } else {
        const int n = length - p.recent, places = p.budget - p.recent;   // n > places >= 0
        // wavefront's stretch; element e of a lane is row from + 64 e + lane
        const int stretch = NK > 0 ? NK * 64 : ((n + WAVES - 1) / WAVES + 63) / 64 * 64;
        const int from = min(wave * stretch, n), to = min(from + stretch, n);
        unsigned key[NK > 0 ? NK : 1];
        if constexpr (NK > 0) {
            float x[NK];
#pragma unroll
            for (int e = 0; e < NK; ++e) x[e] = w[min(from + 64 * e + lane, n - 1)];
#pragma unroll
            for (int e = 0; e < NK; ++e) key[e] = weightKey(x[e]);
        }
        auto each = [&](auto f) {   // f(row, key, the row exists): called by whole wavefronts
            if constexpr (NK > 0) {
#pragma unroll
                for (int e = 0; e < NK; ++e)
                    if (from + 64 * e < to) f(from + 64 * e + lane, key[e], from + 64 * e + lane < to);
            } else {
                for (int i0 = from; i0 < to; i0 += 64) f(i0 + lane, weightKey(w[min(i0 + lane, n - 1)]), i0 + lane < to);
            }
        };
        unsigned prefix = 0;     // the digits found so far
        int need = places;       // places left for keys that share them
        int shift = 32;
        if (places > 0) {
            for (int pass = 0; pass < 3; ++pass) {
                const int bits = pass < 2 ? 11 : 10;
                shift -= bits;
                for (int i = t; i < BINS; i += 1024) hist[i] = 0;
                __syncthreads();
                each([&](int, unsigned x, bool in) {
                    if (in && (pass == 0 || x >> (shift + bits) == prefix)) atomicAdd(&hist[x >> shift & ((1u << bits) - 1)], 1u);
                });
                __syncthreads();
                // thread t owns a pair of bins, 2 t bins from the top: the bin that holds place `need`
                const int hi = BINS - 1 - 2 * t, lo = hi - 1;
                const unsigned a = hist[hi], c = hist[lo];
                unsigned sum = a + c;
#pragma unroll
                for (int off = 1; off < 64; off <<= 1) {
                    const unsigned o = __shfl_up(sum, off, 64);
                    if (lane >= off) sum += o;
                }
                if (lane == 63) total[wave] = sum;
                __syncthreads();
                unsigned before = sum - a - c;
#pragma unroll
                for (int x = 0; x < WAVES; ++x) before += x < wave ? total[x] : 0u;
                if (before < unsigned(need) && before + a >= unsigned(need)) { sDigit = hi; sAbove = before; }
                else if (before + a < unsigned(need) && before + a + c >= unsigned(need)) { sDigit = lo; sAbove = before + a; }
                __syncthreads();
                prefix = prefix << bits | sDigit;
                need -= int(sAbove);
                __syncthreads();
            }
        }
        // keys above `prefix` stay, and the first `need` of those equal to it
        int greater = 0, equal = 0;
        if (places > 0) {
            each([&](int, unsigned x, bool in) {
                greater += __popcll(__ballot(in && x > prefix));
                equal += __popcll(__ballot(in && x == prefix));
            });
        }
        if (lane == 0) { sGreater[wave] = greater; sEqual[wave] = equal; }
        __syncthreads();
        int at = 0, equalBefore = 0;
#pragma unroll
        for (int x = 0; x < WAVES; ++x) {
            if (x < wave) {
                at += sGreater[x] + min(max(need - equalBefore, 0), sEqual[x]);
                equalBefore += sEqual[x];
            }
        }
        if (places > 0) {
            const unsigned long long below = (1ull << lane) - 1;
            each([&](int i, unsigned x, bool in) {
                const unsigned long long eq = __ballot(in && x == prefix);
                const bool stays = in && (x > prefix || (x == prefix && equalBefore + __popcll(eq & below) < need));
                const unsigned long long st = __ballot(stays);
                if (stays) kept[at + __popcll(st & below)] = i;
                at += __popcll(st);
                equalBefore += __popcll(eq);
            });
        }
        for (int i = t; i < p.recent; i += 1024) kept[places + i] = n + i;
    }
    __syncthreads();   // kept[] is read back below by other threads of this workgroup
    float* wOut = p.weightsOut + (size_t(b) * p.groups + g) * p.outCapacity;
    for (int i0 = 0; i0 < left; i0 += 4096) {
        float x[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) x[u] = i0 + 1024 * u + t < left ? w[kept[i0 + 1024 * u + t]] : 0.0f;
        __syncthreads();
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (i0 + 1024 * u + t < left) wOut[i0 + 1024 * u + t] = x[u];
    }
}

// The kept rows moved up.  A workgroup owns 16 accesses' width (256 bytes with 16-byte accesses) of one group's share of
// the rows, of the keys or of the values, and takes tiles of 128 rows in order, `splits` workgroups dealing them out
// among themselves when the result goes to other tensors (each tile is then on its own).  In place one workgroup walks
// all the tiles: a tile's reads come before the barrier, its writes after it, and what later tiles read lies at or
// after their own first row.  That leaves few workgroups and a load's latency bare in every tile: 8 ragged sequences of up
// to 16384 rows cut to 4096, 16 heads of 128, 335 us with the selection where the call to other tensors takes 186; one such
// sequence 202 and 40.
template <int VEC, bool NT>
__global__ void __launch_bounds__(256) evictMoveKernel(EvictParams p, int slices, int splits) {
    constexpr int ROWS = 16, U = 8, TILE = ROWS * U;
    const int slice = blockIdx.x % slices, side = blockIdx.x / slices % 2, split = blockIdx.x / slices / 2;
    const int g = blockIdx.y, b = blockIdx.z;
    const int left = p.left[b];
    if (g == 0 && blockIdx.x == 0 && threadIdx.x == 0 && p.lengthsOut) p.lengthsOut[b] = left;
    const int column = (slice * 16 + int(threadIdx.x & 15)) * VEC, r0 = threadIdx.x >> 4;
    const bool live = column < p.slab;
    const size_t rowFloats = size_t(p.groups) * p.slab;
    const float* src = (side ? p.v : p.k) + size_t(b) * p.capacity * rowFloats + size_t(g) * p.slab + column;
    float* dst = (side ? p.vOut : p.kOut) + size_t(b) * p.outCapacity * rowFloats + size_t(g) * p.slab + column;
    const int* kept = p.kept + (size_t(b) * p.groups + g) * p.budget;
    const bool inPlace = src == dst;
    for (int i0 = split * TILE; i0 < left; i0 += splits * TILE) {
        // ascending rows: if the tile's last row stays where it is, all of them do
        const int last = min(i0 + TILE, left) - 1;
        if (inPlace && kept[last] == last) continue;
        float x[U][VEC];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * ROWS + r0;
            if (live && i < left) {
                const float* from = src + size_t(kept[i]) * rowFloats;
                if constexpr (VEC == 4) {
                    const float4v f = ldf4<NT>(from);
                    x[u][0] = f.x; x[u][1] = f.y; x[u][2] = f.z; x[u][3] = f.w;
                } else {
                    x[u][0] = *from;
                }
            }
        }
        if (inPlace) __syncthreads();
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int i = i0 + u * ROWS + r0;
            if (live && i < left) {
                float* to = dst + size_t(i) * rowFloats;
                if constexpr (VEC == 4) stf4<NT>(to, float4v{x[u][0], x[u][1], x[u][2], x[u][3]});
                else *to = x[u][0];
            }
        }
    }
}

// ---- verification of a drafted tree ------------------------------------------------------------
// Lowest index of each row's maximum, by the loop "best = 0; if (row[c] > row[best]) best = c": a NaN is never chosen unless
// it is element 0, which is then never beaten.  The logits are read once, 16 bytes a thread and four loads in flight, and
// compared in groups of four: of the best group only the value and the place are kept until the end.  `pieces` workgroups
// share a row where there are few rows (26 rows of 50257: 13.7 us with one each, 4.4 with three); 1536 rows of 32000 take 31 us, 6.3 TB/s.
struct Best { float value; int at; };   // at: INT_MAX, nothing above -infinity seen
__device__ __forceinline__ void take(Best& mine, float value, int at) {
    if (value > mine.value || (value == mine.value && at < mine.at)) { mine.value = value; mine.at = at; }
}
__global__ void __launch_bounds__(256) treeChoiceKernel(const float* __restrict__ logits, const int* __restrict__ counts, Best* __restrict__ best,
                                                        int nodes, int vocab, int pieces) {
    __shared__ Best sBest[4];
    const int row = blockIdx.x / pieces, piece = blockIdx.x % pieces, b = row / nodes, i = row % nodes;
    if (counts && i >= counts[b]) return;
    const float* x = logits + size_t(row) * vocab;
    // groups of four from the 16-byte boundary at or below the row's first element; the row's ends are taken one by one
    const int shift = int((reinterpret_cast<uintptr_t>(x) >> 2) & 3), groups = (vocab + shift + 3) / 4;
    const int per = (groups + pieces - 1) / pieces, from = piece * per, to = min(from + per, groups);
    auto whole = [&](int group) { return group * 4 >= shift && group * 4 + 4 <= vocab + shift; };
    auto load = [&](int group) {
        if (whole(group)) return loadf4(x + (group * 4 - shift));
        float4v v;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int c = group * 4 - shift + j;
            v[j] = c >= 0 && c < vocab ? x[c] : -INFINITY;
        }
        return v;
    };
    Best mine{-INFINITY, INT_MAX};
    for (int g0 = from + int(threadIdx.x); g0 < to; g0 += 1024) {
        float4v v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = g0 + 256 * u < to ? load(g0 + 256 * u) : float4v{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const float most = fmaxf(fmaxf(v[u].x, v[u].y), fmaxf(v[u].z, v[u].w));   // fmaxf passes over NaN
            if (most > mine.value) { mine.value = most; mine.at = g0 + 256 * u; }
        }
    }
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float value = __shfl_xor(mine.value, off, 64);
        const int at = __shfl_xor(mine.at, off, 64);
        take(mine, value, at);
    }
    if ((threadIdx.x & 63) == 0) sBest[threadIdx.x >> 6] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) take(mine, sBest[w].value, sBest[w].at);
        if (mine.at != INT_MAX) {
            const float4v v = load(mine.at);
            int j = 0;
            while (j < 3 && !(v[j] == mine.value)) ++j;
            mine.at = mine.at * 4 - shift + j;
        }
        if (piece == 0 && x[0] != x[0]) mine = Best{INFINITY, 0};
        best[blockIdx.x] = mine;
    }
}

// One wavefront per sequence, a lane per node: from the root, the lowest-numbered child that carries the token chosen at
// the node, until there is none.  Children come after their parent, so the walk ends.
__global__ void __launch_bounds__(64) treeWalkKernel(const Best* __restrict__ best, int pieces, const float* __restrict__ tokens, const int* __restrict__ parents,
                                                     const int* __restrict__ counts, int* __restrict__ path, int* __restrict__ pathCounts,
                                                     float* __restrict__ next, int nodes) {
    const int lane = threadIdx.x, b = blockIdx.x;
    const int count = counts ? min(max(counts[b], 0), nodes) : nodes;
    const size_t at = size_t(b) * nodes + lane;
    const bool live = lane < count;
    const int parent = live ? parents[at] : -1;
    const long token = live ? lroundf(tokens[at]) : -1;
    Best chosenHere{-INFINITY, INT_MAX};
    for (int x = 0; live && x < pieces; ++x) {
        const Best piece = best[at * pieces + x];
        take(chosenHere, piece.value, piece.at);
    }
    const int mine = chosenHere.at == INT_MAX ? 0 : chosenHere.at;   // nothing above -infinity: element 0 was never beaten
    int found = 0, cur = 0, step = -1;     // `step`: what this lane writes into path[lane]
    if (count > 0) {
        for (;;) {
            if (lane == found) step = cur;
            ++found;
            const int chosen = __shfl(mine, cur, 64);
            const unsigned long long fits = __ballot(live && lane > cur && parent == cur && token == chosen);
            if (fits == 0) {
                if (lane == 0) next[b] = float(chosen);
                break;
            }
            cur = __ffsll(fits) - 1;
        }
    }
    if (lane < nodes) path[at] = step;
    if (lane == 0) pathCounts[b] = found;
}

constexpr int kCommitLayers = 48;   // layers per launch: their pointers travel as kernel arguments
struct CommitParams {
    float* k[kCommitLayers]; float* v[kCommitLayers];
    const float* kNew[kCommitLayers]; const float* vNew[kCommitLayers];
    float* weights[kCommitLayers];   // all NULL: none kept
    const int* path; const int* pathCounts; const int* lengths; int* lengthsOut;   // lengthsOut NULL: not written here
    int nodes, capacity, rowFloats, groups;
};

// True if the sequence's path fits: every entry a node, and the cache has room.  Uniform over the wavefront.
__device__ __forceinline__ bool pathFits(const CommitParams& p, int b, int length, int count) {
    if (count < 0 || count > p.nodes || length < 0 || length > p.capacity - count) return false;
    const int lane = threadIdx.x & 63;
    const int node = lane < count ? p.path[size_t(b) * p.nodes + lane] : 0;
    return __ballot(node < 0 || node >= p.nodes) == 0;
}

// blockIdx.x: pieces of the rows, .y: layer * 2 + side, .z: sequence
template <int VEC>
__global__ void __launch_bounds__(256) kvCommitKernel(CommitParams p) {
    const int b = blockIdx.z, layer = blockIdx.y >> 1, side = blockIdx.y & 1;
    const int length = p.lengths[b], count = p.pathCounts[b];
    const bool fits = pathFits(p, b, length, count);
    if (p.lengthsOut && blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) p.lengthsOut[b] = fits ? length + count : length;
    if (!fits) return;
    const int units = p.rowFloats / VEC;
    const float* src = (side ? p.vNew[layer] : p.kNew[layer]) + size_t(b) * p.nodes * p.rowFloats;
    float* dst = (side ? p.v[layer] : p.k[layer]) + (size_t(b) * p.capacity + length) * p.rowFloats;
    for (int e = blockIdx.x * 256 + threadIdx.x; e < count * units; e += gridDim.x * 256) {
        const int i = e / units, c = (e - i * units) * VEC;
        const float* from = src + size_t(p.path[size_t(b) * p.nodes + i]) * p.rowFloats + c;
        float* to = dst + size_t(i) * p.rowFloats + c;
        if constexpr (VEC == 4) storef4(to, loadf4(from));
        else *to = *from;
    }
    if (p.weights[layer] && side == 0 && blockIdx.x == 0 && threadIdx.x < 64) {
        // one wavefront, a lane per accepted node: its load is complete before any lane's store is issued
        const int lane = threadIdx.x;
        const int node = lane < count ? p.path[size_t(b) * p.nodes + lane] : 0;
        for (int g = 0; g < p.groups; ++g) {
            float* w = p.weights[layer] + (size_t(b) * p.groups + g) * p.capacity + length;
            const float x = lane < count && length + node < p.capacity ? w[node] : 0.0f;   // past the capacity none was kept
            if (lane < count) w[lane] = x;
        }
    }
}

__global__ void __launch_bounds__(64) commitLengthsKernel(CommitParams p) {
    const int b = blockIdx.x, length = p.lengths[b], count = p.pathCounts[b];
    const bool fits = pathFits(p, b, length, count);
    if (threadIdx.x == 0) p.lengthsOut[b] = fits ? length + count : length;
}

}  // namespace
}  // namespace bf

using namespace bf;

extern "C" {

int bf_hip_kv_evict(const float* kCache, const float* vCache, const float* weights, const int* lengths, float* kOut, float* vOut, float* weightsOut,
                    int* lengthsOut, int* kept, size_t batch, size_t kvHeads, size_t groups, size_t headDim, size_t capacity, size_t outCapacity,
                    size_t budget, size_t recent, bf_stream_t stream) {
    BF_REQUIRE(kvHeads > 0 && groups > 0 && kvHeads % groups == 0, "groups must divide kvHeads");
    BF_REQUIRE(recent <= budget, "more recent rows than the budget holds");
    BF_REQUIRE(budget <= outCapacity, "the budget does not fit the result's capacity");
    BF_REQUIRE(batch < (size_t(1) << 16) && groups < (size_t(1) << 16) && kvHeads * headDim < (size_t(1) << 24) && capacity < (size_t(1) << 30) &&
                   outCapacity < (size_t(1) << 30), "shape too large");
    if (batch == 0 || headDim == 0) return BF_OK;
    BF_REQUIRE(lengths && ((kCache && vCache && weights) || capacity == 0) && ((kOut && vOut && weightsOut) || budget == 0), "NULL pointer");
    const bool inPlace = kOut == kCache;
    // (of caches without rows only the lengths are left to write)
    BF_REQUIRE(capacity == 0 || ((vOut == vCache) == inPlace && (weightsOut == weights) == inPlace),
               "keys, values and weights go in place together or not at all");
    BF_REQUIRE(capacity == 0 || !inPlace || outCapacity == capacity, "a call in place keeps the capacity");
    EvictParams p{};
    p.k = kCache; p.v = vCache; p.weights = weights; p.lengths = lengths; p.kOut = kOut; p.vOut = vOut; p.weightsOut = weightsOut;
    p.lengthsOut = lengthsOut; p.batch = int(batch); p.groups = int(groups); p.capacity = int(capacity); p.outCapacity = int(outCapacity);
    p.budget = int(budget); p.recent = int(recent); p.slab = int(kvHeads / groups * headDim);
    const bool vec = p.slab % 4 == 0 && aligned16(kCache) && aligned16(vCache) && aligned16(kOut) && aligned16(vOut);
    const int slices = std::max(1, (p.slab / (vec ? 4 : 1) + 15) / 16);
    const size_t tiles = std::max<size_t>(1, (std::min(budget, capacity) + 127) / 128);
    const int splits = inPlace ? 1 : int(std::min<size_t>(tiles, 64));
    const size_t gridX = size_t(slices) * 2 * size_t(splits);
    BF_REQUIRE(batch * groups <= mostBlocks(1024) && gridX <= mostBlocks(256), "shape too large");
    hipStream_t s = asStream(stream);
    const size_t keptInts = kept ? 0 : batch * groups * budget;
    Scratch own((batch + keptInts) * sizeof(int));
    if (own.status != BF_OK) return own.status;
    p.left = own.as<int>();
    p.kept = kept ? kept : p.left + batch;
    const unsigned pairs = unsigned(batch * groups);
    if (capacity <= 4 * 1024) evictSelectKernel<4><<<pairs, 1024, 0, s>>>(p);
    else if (capacity <= 16 * 1024) evictSelectKernel<16><<<pairs, 1024, 0, s>>>(p);
    else if (capacity <= 64 * 1024) evictSelectKernel<64><<<pairs, 1024, 0, s>>>(p);
    else evictSelectKernel<0><<<pairs, 1024, 0, s>>>(p);
    BF_LAUNCH_CHECK();
    const dim3 grid{unsigned(gridX), unsigned(groups), unsigned(batch)};
    // rows that stream past the last-level cache carry the non-temporal hint (0.9 GB moved: 195 -> 185 us with the selection)
    const size_t moved = batch * std::min(budget, capacity) * groups * size_t(p.slab) * 4 * sizeof(float);
    if (vec && streamsPastCache(moved)) evictMoveKernel<4, true><<<grid, 256, 0, s>>>(p, slices, splits);
    else if (vec) evictMoveKernel<4, false><<<grid, 256, 0, s>>>(p, slices, splits);
    else evictMoveKernel<1, false><<<grid, 256, 0, s>>>(p, slices, splits);
    BF_LAUNCH_CHECK();
    return BF_OK;
}

int bf_hip_tree_accept(const float* logits, const float* tokens, const int* parents, const int* counts, int* path, int* pathCounts, float* next,
                       size_t batch, size_t nodes, size_t vocab, bf_stream_t stream) {
    BF_REQUIRE(nodes <= 64, "a tree has at most 64 nodes, got " + std::to_string(nodes));
    BF_REQUIRE(batch < (size_t(1) << 16), "shape too large");
    if (batch == 0 || nodes == 0) return BF_OK;
    BF_REQUIRE(vocab > 0, "empty logits");
    BF_REQUIRE(vocab <= (size_t(1) << 24), "a token id beyond 2^24 has no exact float");
    BF_REQUIRE(logits && tokens && parents && path && pathCounts && next, "NULL pointer");
    hipStream_t s = asStream(stream);
    // two workgroups a compute unit, as long as each has 4096 logits
    const size_t rows = batch * nodes, wanted = (2 * size_t(computeUnits()) + rows - 1) / rows;
    const size_t pieces = std::max<size_t>(1, std::min<size_t>({wanted, vocab / 4096, 32}));
    Scratch best(rows * pieces * sizeof(Best));
    if (best.status != BF_OK) return best.status;
    treeChoiceKernel<<<unsigned(rows * pieces), 256, 0, s>>>(logits, counts, best.as<Best>(), int(nodes), int(vocab), int(pieces));
    BF_LAUNCH_CHECK();
    treeWalkKernel<<<unsigned(batch), 64, 0, s>>>(best.as<Best>(), int(pieces), tokens, parents, counts, path, pathCounts, next, int(nodes));
    BF_LAUNCH_CHECK();
    return BF_OK;
}

int bf_hip_kv_commit(float* const* kCaches, float* const* vCaches, const float* const* kNew, const float* const* vNew, float* const* weights,
                     size_t layers, const int* path, const int* pathCounts, const int* lengths, int* lengthsOut, size_t batch, size_t kvHeads,
                     size_t groups, size_t nodes, size_t capacity, size_t headDim, bf_stream_t stream) {
    BF_REQUIRE(nodes <= 64, "a tree has at most 64 nodes, got " + std::to_string(nodes));
    BF_REQUIRE(!weights || (groups > 0 && kvHeads > 0 && kvHeads % groups == 0), "groups must divide kvHeads");
    BF_REQUIRE(batch < (size_t(1) << 16) && capacity < (size_t(1) << 30) && kvHeads * headDim < (size_t(1) << 24), "shape too large");
    if (batch == 0) return BF_OK;
    BF_REQUIRE(pathCounts && lengths && (path || nodes == 0), "NULL pointer");
    const size_t rowFloats = kvHeads * headDim;
    const bool rows = layers > 0 && nodes > 0 && rowFloats > 0;
    BF_REQUIRE(!rows || (kCaches && vCaches && kNew && vNew), "NULL pointer");
    bool vec = rowFloats % 4 == 0;
    for (size_t i = 0; rows && i < layers; ++i) {
        BF_REQUIRE(((kCaches[i] && vCaches[i]) || capacity == 0) && kNew[i] && vNew[i] && (!weights || weights[i] || capacity == 0),
                   "NULL pointer in layer " + std::to_string(i));
        vec = vec && aligned16(kCaches[i]) && aligned16(vCaches[i]) && aligned16(kNew[i]) && aligned16(vNew[i]);
    }
    hipStream_t s = asStream(stream);
    CommitParams p{};
    p.path = path; p.pathCounts = pathCounts; p.lengths = lengths;
    p.nodes = int(nodes); p.capacity = int(capacity); p.rowFloats = int(rowFloats); p.groups = int(groups);
    // the new lengths ride on the first launch unless they replace the ones that every workgroup reads
    bool lengthsDone = lengthsOut == nullptr;
    for (size_t first = 0; rows && first < layers; first += kCommitLayers) {
        const size_t n = std::min<size_t>(kCommitLayers, layers - first);
        for (size_t i = 0; i < n; ++i) {
            p.k[i] = kCaches[first + i]; p.v[i] = vCaches[first + i]; p.kNew[i] = kNew[first + i]; p.vNew[i] = vNew[first + i];
            p.weights[i] = weights ? weights[first + i] : nullptr;
        }
        p.lengthsOut = !lengthsDone && lengthsOut != lengths ? lengthsOut : nullptr;
        lengthsDone = lengthsDone || p.lengthsOut != nullptr;
        // workgroups for four rows at once: a path is rarely longer, and a workgroup without a row still costs its launch
        // (32 sequences, 12 layers: 15 us with a workgroup for every row there might be)
        const unsigned pieces = unsigned(std::min<size_t>(16, (std::min<size_t>(nodes, 4) * rowFloats / (vec ? 4 : 1) + 255) / 256));
        const dim3 grid(std::max(1u, pieces), unsigned(2 * n), unsigned(batch));
        if (vec) kvCommitKernel<4><<<grid, 256, 0, s>>>(p);
        else kvCommitKernel<1><<<grid, 256, 0, s>>>(p);
        BF_LAUNCH_CHECK();
    }
    if (!lengthsDone) {
        p.lengthsOut = lengthsOut;
        commitLengthsKernel<<<unsigned(batch), 64, 0, s>>>(p);
        BF_LAUNCH_CHECK();
    }
    return BF_OK;
}

}  // extern "C"

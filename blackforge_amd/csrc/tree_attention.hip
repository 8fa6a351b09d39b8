// Attention of new tokens over a key/value cache with a length per sequence, the new tokens being the nodes of a drafted
// tree (or a chain, or one), and the attention weight that every cached row receives.  fp32 in and out.
//
// Node i of sequence b sees the cached rows j < lengths[b] and those new rows j < counts[b] whose bit is set in
// visible[b, i] (NULL: bits 0..i, a chain).  With s_j = scale q_i . k_j over what it sees,
//   m = max s_j,  l = sum exp(s_j - m),  out = sum exp(s_j - m) v_j / l;     nothing seen: out = 0, m = -inf, l = 0.
// Query head h reads key head h * kvHeads / heads.
#include "common.hpp"

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <type_traits>

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

// ---- the pass over the cache -------------------------------------------------------------------
// The rows of one key head, all its queries of all nodes (row = node * share + head within the share), times the cache is a
// pair of matrix products with a softmax between them, and the cache is read once: 8 bytes of keys and values against four
// flops a row; fp32 matrix instructions (v_mfma_f32_16x16x4_f32) keep up with the memory up to about 32 rows.
//
// A wavefront holds RT tiles of 16 rows (the queries as B operands, the output as accumulators) and takes 16 keys at a
// time: S^T = K Q^T leaves a lane with 4 keys of one row, which is already the B operand of O^T += V^T P^T, so neither
// scores nor probabilities leave their registers.  Keys and values go from memory straight into A operands, 16 bytes a
// lane and no LDS: a dot product does not care about the order of its terms, nor do the rows of O^T, so lane (i, g) of
// 16 x 4 loads head columns 16 s + 4 g .. of key i, and columns 4 i .. of the values of keys 4 g ...  The loads of the
// next keys are issued as soon as the products have read the registers of these.
//
// Softmax about a reference that moves only when a score outgrows it by 2^8 (common for the first keys, then rare), so a
// tile normally needs no maximum across lanes and no rescaling.  d = c dot - ref in one fused operation, c = scale log2(e):
// the error of d is relative to d, not to the score.  The true maximum is kept beside it for the statistics.
//
// Measured: 26 nodes, 16 heads of 128, 120011 rows 322 us = 6.1 TB/s with the join (HBM); 32 ragged sequences of up to 4032 rows,
// 12 heads of 64, 64 nodes 147 us (427 MB, 10.3 GFLOP: the matrix pipe is busy for half of the time, and the call takes 22 us
// over empty caches, the start and end of a workgroup and the join); one node over 701 rows 10 us (two dependent launches).
struct TilePlan {
    int target;          // chunks per (key head, group of row tiles) that the launch wants in total over the sequences
    int minChunk;        // keys a chunk has at least
    float slots;         // chunks (per key head and group of row tiles) that run at once; 0: even shares of `target`
    int items;           // workgroups along the sequences' chunks: at least the number of chunks there will be
    int rowGroups;       // groups of RT row tiles
    float4v* partStat;   // [item][kvHeads][rows]: ref, l, largest dot product
    float* partOut;      // [item][kvHeads][rows][partPitch], relative to ref
    float2* rowStat;     // [batch][kvHeads][rows]: ref, 1 / l over all chunks, for a launch that makes weights (NULL: not kept)
    int2* span;          // [batch]: first item and number of items of a sequence
    float* scores;       // [batch][kvHeads][rows][scorePitch] dot products with the cached rows (NULL: not kept)
    float* newScores;    // [batch][kvHeads][rows][64] and with the new ones, -infinity where not seen
    int scorePitch, partPitch, keyBlocks;
    float c;             // |scale| log2(e); 1 if that is 0
    float sign;          // that of the scale, which the queries take; 0 with c: a scale of 0 makes every score it sees 0
    unsigned magic;      // 2^32 / (heads / kvHeads), rounded up
};

// Where the products bound the pass, what a chunk size costs is the number of rounds its workgroups take on the device's
// slots times the length of a round, and neighbouring sizes differ much (32 equal sequences, 12 heads, 512 slots: three
// chunks each are 1152 workgroups, 3 rounds of a third; four are 1536, 3 rounds of a quarter).  Lane c of the wavefront tries one
// size, from half as much again as fills the slots once down to a third of it; the cheapest is taken, the larger on a tie.
// Lane 0's makes slots / 1.5 + batch chunks at most, which `target`, 3 slots + batch, always has room for.
__device__ __forceinline__ int bestChunk(const TreeParams& p, const TilePlan& plan, int length, int total) {
    const int lane = threadIdx.x & 63, mine = (length + 63) / 64;
    const float base = float(total) / plan.slots;            // units of 64 keys that fill the slots once
    const int least = plan.minChunk / 64;
    const float size = fminf(fmaxf(float(least), ceilf(base * 1.5f * 18.0f / (18.0f + float(lane)))), 16777216.0f);   // 2^30 keys
    const float over = 1.0f / size;
    float chunks = 0.0f;
    for (int b = 0; b < p.batch; ++b) chunks += fmaxf(1.0f, ceilf(float(__builtin_amdgcn_readlane(mine, b)) * over - 1e-4f));
    float cost = ceilf(chunks / plan.slots - 1e-4f) * (size + 2.0f);   // 2: what a chunk costs beside its keys
    if (chunks > float(plan.target)) cost = INFINITY;        // more than there will be workgroups
    int best = int(size);
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const float otherCost = __shfl_xor(cost, off, 64);
        const int other = __shfl_xor(best, off, 64);
        if (otherCost < cost || (otherCost == cost && other > best)) { cost = otherCost; best = other; }
    }
    return best;
}

// Chunk sizes from the lengths themselves: about `target` chunks of equal size over all sequences, at least one for each (a
// sequence without nodes has nothing to read).  Returns this item's sequence (-1: there is none) and its chunk.
struct Chunk { int b, first, count, start, end, queries; };
__device__ __forceinline__ Chunk findChunk(const TreeParams& p, const TilePlan& plan, int item) {
    const int lane = threadIdx.x & 63;
    auto sequence = [&](int b, int& rows, int& nodes) {
        nodes = b < p.batch ? nodesInUse(p, b) : 0;
        rows = nodes > 0 ? rowsInUse(p, b) : 0;
    };
    int length0, count0;
    sequence(lane, length0, count0);
    long long total = (length0 + 63) / 64;   // in units of 64 rows
    for (int b0 = 64; b0 < p.batch; b0 += 64) {
        int length, count;
        sequence(b0 + lane, length, count);
        total += (length + 63) / 64;
    }
    if (p.batch > 1) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
    } else {
        total = __shfl(total, 0, 64);
    }
    int units = int(min((total + plan.target - 1) / plan.target, (long long)(1 << 24)));
    // (lengths that fill the slots with the shortest chunks at most need no choice)
    if (plan.slots > 0 && p.batch <= 64 && float(total) > plan.slots * float(plan.minChunk / 64)) units = bestChunk(p, plan, length0, int(total));
    const int size = max(plan.minChunk, units * 64);
    Chunk c{-1, 0, 0, 0, 0, 0};
    int before = 0;
    for (int b0 = 0; b0 < p.batch; b0 += 64) {
        const bool on = b0 + lane < p.batch;
        int length = length0, count = count0;
        if (b0 != 0) sequence(b0 + lane, length, count);
        const int mine = on ? max(1, (length + size - 1) / size) : 0;
        int upTo = mine;
        if (p.batch > 1) {
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const int o = __shfl_up(upTo, off, 64);
                if (lane >= off) upTo += o;
            }
        }
        const unsigned long long past = __ballot(on && before + upTo > item);
        if (past != 0) {
            const int at = __ffsll(past) - 1;
            c.b = __builtin_amdgcn_readfirstlane(b0 + at);
            c.count = __builtin_amdgcn_readlane(mine, at);
            c.first = before + __builtin_amdgcn_readlane(upTo, at) - c.count;
            c.queries = __builtin_amdgcn_readlane(count, at);
            const int len = __builtin_amdgcn_readlane(length, at);
            // a sequence's chunks are of one size, a multiple of 64 rows
            const int each = ((len + c.count - 1) / c.count + 63) / 64 * 64;
            c.start = min((item - c.first) * each, len);
            c.end = min(c.start + each, len);
            return c;
        }
        before += __builtin_amdgcn_readlane(upTo, 63);
    }
    return c;
}

// Columns d .. of a row.  MODE 2: headDim == HDP, 16-byte aligned; 1: a multiple of 4, aligned; 0: anything.  `sure`: the
// caller's form is for head dims that all have these columns.  With mode 1 the columns past the row's end hold any others of
// it, and the caller takes them out where it uses them: a select behind a load waits for it (head dim 100, 4 x 8192 rows, 8
// heads: 60 us with the select here, 48 without; 160: 100 and 72; one element at a time the select is better, 33: 34 and 40).
template <int MODE, int W>
__device__ __forceinline__ void fetchColumns(float (&x)[W], const float* row, int d, int hd, bool sure = false) {
    if constexpr (MODE == 0) {
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = sure || d + j < hd ? row[d + j] : 0.0f;
    } else {
        const float* at = row + (MODE == 2 || sure || d < hd ? d : 0);
        if constexpr (W == 4) {
            const float4v f = loadf4(at);
            x[0] = f.x; x[1] = f.y; x[2] = f.z; x[3] = f.w;
        } else {
            const float2v f = *reinterpret_cast<const float2v*>(at);
            x[0] = f.x; x[1] = f.y;
        }
    }
}
template <int MODE, int W>
__device__ __forceinline__ void clearPastEnd(float (&x)[W], int d, int hd) {
    if constexpr (MODE == 1) {
#pragma unroll
        for (int j = 0; j < W; ++j) x[j] = d < hd ? x[j] : 0.0f;
    }
}
template <int MODE, int W>
__device__ __forceinline__ void loadColumns(float (&x)[W], const float* row, int d, int hd) {
    fetchColumns<MODE>(x, row, d, hd);
    clearPastEnd<MODE>(x, d, hd);
}

// A row's statistics from its reference, the sum about it and its largest dot product
__device__ __forceinline__ void finishStats(const TreeParams& p, const TilePlan& plan, int b, int kh, int row, float ref, float sum, float top) {
    const int share = p.heads / p.kvHeads;
    const size_t stat = (size_t(b) * p.heads + kh * share + row % share) * p.nodes + row / share;
    const bool empty = sum == 0.0f;
    if (plan.rowStat) plan.rowStat[(size_t(b) * p.kvHeads + kh) * p.nodes * share + row] = make_float2(ref, empty ? 0.0f : 1.0f / sum);
    if (p.m) p.m[stat] = empty ? -INFINITY : top * fabsf(p.scale);
    if (p.l) p.l[stat] = empty ? 0.0f : sum * __builtin_amdgcn_exp2f(-fmaf(top, plan.c, -ref));
}

constexpr float kNoRef = -3.402823466e38f;   // a reference below every score: the first real one moves it
constexpr float kRefSlack = 8.0f;

// The node of a row and its head among the heads that share its key head; `magic` is 2^32 / share rounded up
__device__ __forceinline__ int nodeOf(const TilePlan& plan, int share, int row) { return share == 1 ? row : int(__umulhi(unsigned(row), plan.magic)); }

// wavefronts per SIMD that the registers of a form allow
constexpr int tileWaves(int hdp, int rt) { return hdp * rt <= 96 ? 3 : hdp * rt <= 256 && hdp <= 128 ? 2 : 1; }
template <int HDP, int RT, int MODE, bool SCORES>
__global__ void __launch_bounds__(256, tileWaves(HDP, RT)) treeTilesKernel(TreeParams p, TilePlan plan) {
    constexpr int KS = HDP / 16;                    // 16-column steps of the dot products
    constexpr int LEAST = HDP == 256 ? 192 : HDP == 192 ? 128 : HDP == 32 ? 0 : HDP - 32;   // head dims of this form are above
    constexpr int VW = HDP % 64 == 0 ? 4 : 2;       // value columns a lane loads at once
    constexpr int VU = HDP / (16 * VW);             // such loads
    constexpr int PITCH = HDP + 4;
    extern __shared__ float smem[];                 // [wavefront][row][PITCH]: the outputs to be joined
    __shared__ float4v sStat[4][RT * 16];
    __shared__ unsigned sOdd[4];   // new rows of each 16 that hold a value which is not finite
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), i16 = lane & 15, g = lane >> 4;
    // the row groups of one chunk next to each other on one XCD (workgroups go to the 8 XCDs in turn), where they share its reads
    const unsigned perXcd = blockIdx.x / 8, flat = perXcd / plan.rowGroups * 8 + blockIdx.x % 8;
    const int rowGroup = perXcd % plan.rowGroups;
    const int kh = flat % p.kvHeads, item = flat / p.kvHeads;
    if (item >= plan.items) return;
    const Chunk ch = findChunk(p, plan, item);
    if (ch.b < 0) return;
    const int b = ch.b, share = p.heads / p.kvHeads, rows = p.nodes * share, hd = p.hd;
    const int count = ch.queries, live = count * share;     // rows past `live` belong to no node
    if (item == ch.first && kh == 0 && rowGroup == 0 && threadIdx.x == 0) plan.span[b] = make_int2(ch.first, ch.count);
    const int row0 = rowGroup * RT * 16;
    if (row0 >= live) return;
    const int tiles = min(RT, (live - row0 + 15) / 16);
    const unsigned kvDim = unsigned(p.kvHeads) * hd;
    if (threadIdx.x < 4) sOdd[threadIdx.x] = 0;
    __syncthreads();

    // The wavefront's tiles of 16 keys: every fourth of the chunk's, and with the sequence's last chunk 16 of the new rows,
    // starting with the wavefront that has the fewest cached ones.
    const int from = ch.start + wave * 16, cachedTiles = max(0, (ch.end - from + 63) / 64);
    const int newTile = (wave - (ch.end - ch.start + 15) / 16) & 3;
    const bool hasNew = item == ch.first + ch.count - 1 && newTile * 16 < count;
    const size_t firstCached = (size_t(b) * p.capacity + from) * kvDim + size_t(kh) * hd;
    const size_t firstNew = (size_t(b) * p.nodes + newTile * 16) * kvDim + size_t(kh) * hd;
    float k[KS][4], v[VU][4][VW];
    // a tile from its first row, of which rows 0 .. last exist; the addresses are a uniform base and a 32-bit offset
    auto loadK = [&](const float* base, int last) {
        const float* src = reinterpret_cast<const float*>(reinterpret_cast<const char*>(base) + 4u * (__umul24(unsigned(min(i16, last)), kvDim) + 4 * g));
#pragma unroll
        for (int s = 0; s < KS; ++s) fetchColumns<MODE>(k[s], src - 4 * g, 16 * s + 4 * g, hd, 16 * s + 16 <= LEAST);
    };
    auto loadV = [&](const float* base, int last) {
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const float* src = reinterpret_cast<const float*>(reinterpret_cast<const char*>(base) + 4u * __umul24(unsigned(min(4 * g + r, last)), kvDim));
#pragma unroll
            for (int u = 0; u < VU; ++u) fetchColumns<MODE>(v[u][r], src, u * 16 * VW + i16 * VW, hd, (u + 1) * 16 * VW <= LEAST);   // past the end: columns that nobody reads
        }
    };
    unsigned seen[RT];   // bits 0..3: new rows 16 newTile + 4 g .. that this lane's row of tile t sees
    float q[RT][KS][4];
    const float sign = plan.sign;
    const float* qBase = p.q + size_t(b) * p.nodes * p.heads * hd + size_t(kh) * share * hd;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        const int row = row0 + t * 16 + i16;
        const bool on = row < live;
        const int node = on ? nodeOf(plan, share, row) : 0, h = on ? row - node * share : 0;
        const float* src = qBase + unsigned(node * p.heads + h) * unsigned(hd);
        seen[t] = hasNew && on ? unsigned(newRowsSeen(p, b, node, count) >> (newTile * 16 + 4 * g)) & 15u : 0u;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            loadColumns<MODE, 4>(q[t][s], src, 16 * s + 4 * g, hd);
#pragma unroll
            for (int c = 0; c < 4; ++c) q[t][s][c] *= on ? sign : 0.0f;
        }
    }
    float4v o[RT][VU][VW];
    float ref[RT], l[RT], top[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        ref[t] = kNoRef; l[t] = 0.0f; top[t] = -INFINITY;
#pragma unroll
        for (int u = 0; u < VU; ++u)
#pragma unroll
            for (int w = 0; w < VW; ++w) o[t][u][w] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
    }
    const int newLast = min(15, count - 1 - newTile * 16);
    auto clearKeys = [&]() {
#pragma unroll
        for (int s = 0; s < KS; ++s)
            if (16 * s + 16 > LEAST) clearPastEnd<MODE>(k[s], 16 * s + 4 * g, hd);
    };
    auto dotProducts = [&](int t) {
        float4v even = {0.0f, 0.0f, 0.0f, 0.0f}, odd = even;   // two chains: half the error, and none waits for the one before
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            even = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][0], q[t][s][0], even, 0, 0, 0);
            odd = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][1], q[t][s][1], odd, 0, 0, 0);
            even = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][2], q[t][s][2], even, 0, 0, 0);
            odd = __builtin_amdgcn_mfma_f32_16x16x4f32(k[s][3], q[t][s][3], odd, 0, 0, 0);
        }
        return even + odd;
    };
    // dot products of N tiles to probabilities about ref (-infinity: not seen)
    auto probabilities = [&](auto tileCount, float (&x)[RT][4]) {
        constexpr int N = decltype(tileCount)::value;
        float d[N][4];
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < N; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) d[t][r] = fmaf(x[t][r], plan.c, -ref[t]);
            top[t] = fmaxf(top[t], fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3])));
            most = fmaxf(most, fmaxf(fmaxf(d[t][0], d[t][1]), fmaxf(d[t][2], d[t][3])));
        }
        if (__any(most > kRefSlack)) {
#pragma unroll
            for (int t = 0; t < N; ++t) {
                float mx = fmaxf(fmaxf(x[t][0], x[t][1]), fmaxf(x[t][2], x[t][3]));
                mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
                mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
                const float moved = mx == -INFINITY ? ref[t] : fmaxf(ref[t], mx * plan.c);
                const float keep = __builtin_amdgcn_exp2f(ref[t] - moved);
                ref[t] = moved;
                l[t] *= keep;
#pragma unroll
                for (int u = 0; u < VU; ++u)
#pragma unroll
                    for (int w = 0; w < VW; ++w) o[t][u][w] = o[t][u][w] * keep;
#pragma unroll
                for (int r = 0; r < 4; ++r) d[t][r] = fmaf(x[t][r], plan.c, -moved);
            }
        }
#pragma unroll
        for (int t = 0; t < N; ++t) {
#pragma unroll
            for (int r = 0; r < 4; ++r) x[t][r] = __builtin_amdgcn_exp2f(d[t][r]);
            l[t] += (x[t][0] + x[t][1]) + (x[t][2] + x[t][3]);
        }
    };
    auto addValues = [&](int t, const float (&x)[4]) {
#pragma unroll
        for (int r = 0; r < 4; ++r)       // products of one key after another's: none waits for the accumulator of the one before
#pragma unroll
            for (int u = 0; u < VU; ++u)
#pragma unroll
                for (int w = 0; w < VW; ++w) o[t][u][w] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[u][r][w], x[r], o[t][u][w], 0, 0, 0);
    };

    // The cached tiles.  The body is straight-line code for the number of row tiles in use, and no load in it stands behind a
    // branch (the waits for the loads before it would have to assume the worst); the last tile fetches the new rows'.
    auto walk = [&](auto tileCount) {
        constexpr int N = decltype(tileCount)::value;
        if (cachedTiles + int(hasNew) == 0) return;
        const float* kAt = cachedTiles > 0 ? p.k + firstCached : p.kNew + firstNew;
        const float* vAt = cachedTiles > 0 ? p.v + firstCached : p.vNew + firstNew;
        const int lastAt = cachedTiles > 0 ? min(15, ch.end - 1 - from) : newLast;
        loadK(kAt, lastAt);
        loadV(vAt, lastAt);
        for (int n = 0; n < cachedTiles; ++n) {
            const int key = from + n * 64;
            const bool more = n + 1 < cachedTiles;
            const float* kNext = more ? kAt + size_t(64) * kvDim : hasNew ? p.kNew + firstNew : kAt;
            const float* vNext = more ? vAt + size_t(64) * kvDim : hasNew ? p.vNew + firstNew : vAt;
            const int lastNext = more ? min(15, ch.end - 1 - key - 64) : hasNew ? newLast : 0;
            float x[RT][4];
            clearKeys();
#pragma unroll
            for (int t = 0; t < N; ++t) {
                const float4v dots = dotProducts(t);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[t][r] = dots[r];
            }
            loadK(kNext, lastNext);
            if (key + 16 > ch.end) {     // values of keys past the end: whatever lies there must not meet a weight of zero
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = key + 4 * g + r < ch.end;
#pragma unroll
                    for (int t = 0; t < N; ++t) x[t][r] = in ? x[t][r] : -INFINITY;
#pragma unroll
                    for (int u = 0; u < VU; ++u)
#pragma unroll
                        for (int w = 0; w < VW; ++w) v[u][r][w] = in ? v[u][r][w] : 0.0f;
                }
            }
            if constexpr (SCORES) {
#pragma unroll
                for (int t = 0; t < N; ++t) {
                    const int row = row0 + t * 16 + i16;
                    if (row < live) storef4(plan.scores + ((size_t(b) * p.kvHeads + kh) * rows + row) * plan.scorePitch + key + 4 * g, float4v{x[t][0], x[t][1], x[t][2], x[t][3]});
                }
            }
            probabilities(tileCount, x);
#pragma unroll
            for (int t = 0; t < N; ++t) addValues(t, x[t]);
            loadV(vNext, lastNext);
            kAt = kNext;
            vAt = vNext;
        }
        if (hasNew) {
            const int j0 = newTile * 16;
            // A value that is not finite must not meet the weight zero of a row that does not see it: taken out here, added to
            // the rows that do when the results are written.
            unsigned notFinite = 0;
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int u = 0; u < VU; ++u)
#pragma unroll
                    for (int w = 0; w < VW; ++w) {
                        const bool in = j0 + 4 * g + r < count, finite = fabsf(v[u][r][w]) < INFINITY;
                        if (in && !finite) notFinite |= 1u << (4 * g + r);
                        v[u][r][w] = in && finite ? v[u][r][w] : 0.0f;
                    }
            if (notFinite) atomicOr(&sOdd[newTile], notFinite);
            float x[RT][4];
            clearKeys();
#pragma unroll
            for (int t = 0; t < N; ++t) {
                const float4v dots = dotProducts(t);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[t][r] = seen[t] >> r & 1 ? dots[r] : -INFINITY;
                const int row = row0 + t * 16 + i16;
                if (plan.newScores && row < live)
                    storef4(plan.newScores + ((size_t(b) * p.kvHeads + kh) * rows + row) * 64 + j0 + 4 * g, float4v{x[t][0], x[t][1], x[t][2], x[t][3]});
            }
            probabilities(tileCount, x);
#pragma unroll
            for (int t = 0; t < N; ++t) addValues(t, x[t]);
        }
    };
    if (tiles == RT) walk(std::integral_constant<int, RT>{});
    if constexpr (RT >= 2) { if (tiles == 1) walk(std::integral_constant<int, 1>{}); }
    if constexpr (RT >= 4) {
        if (tiles == 2) walk(std::integral_constant<int, 2>{});
        if (tiles == 3) walk(std::integral_constant<int, 3>{});
    }

    // the four wavefronts' states joined through LDS
#pragma unroll
    for (int t = 0; t < RT; ++t) {
        if (t < tiles) {
            float sum = l[t], mx = top[t];
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            if (g == 0) sStat[wave][t * 16 + i16] = float4v{ref[t], sum, mx, 0.0f};
            float* mine = smem + (wave * RT * 16 + t * 16 + i16) * PITCH;
#pragma unroll
            for (int u = 0; u < VU; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float* to = mine + u * 16 * VW + (4 * g + e) * VW;
                    if constexpr (VW == 4) storef4(to, float4v{o[t][u][0][e], o[t][u][1][e], o[t][u][2][e], o[t][u][3][e]});
                    else *reinterpret_cast<float2v*>(to) = float2v{o[t][u][0][e], o[t][u][1][e]};
                }
        }
    }
    __syncthreads();
    const bool only = ch.count == 1;
    const unsigned long long odd = (unsigned long long)(sOdd[0] | sOdd[1] << 16) | (unsigned long long)(sOdd[2] | sOdd[3] << 16) << 32;
    const int liveHere = min(live - row0, tiles * 16);
    const size_t entry = (size_t(item) * p.kvHeads + kh) * rows;
    float* outBase = only ? p.out + size_t(b) * p.nodes * p.heads * hd + size_t(kh) * share * hd : plan.partOut + entry * plan.partPitch;
    // sixteen threads a row, four columns at a time
    for (int e = threadIdx.x; e < liveHere * 16; e += 256) {
        const int r = e >> 4, part = e & 15, row = row0 + r;
        float4v st[4];
        float most = kNoRef, mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            st[w] = sStat[w][r];
            most = fmaxf(most, st[w].x);
            mx = fmaxf(mx, st[w].z);
        }
        float f[4], sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            f[w] = __builtin_amdgcn_exp2f(st[w].x - most);
            sum += st[w].y * f[w];
        }
        const int node = nodeOf(plan, share, row), h = row - node * share;
        if (only) {
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
#pragma unroll
            for (int w = 0; w < 4; ++w) f[w] *= inv;
        }
        float* dst = outBase + (only ? unsigned(node * p.heads + h) * unsigned(hd) : unsigned(row) * unsigned(plan.partPitch));
        for (int d = part * 4; d < hd; d += 64) {
            float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < 4; ++w) acc = acc + *reinterpret_cast<const float4v*>(smem + (w * RT * 16 + r) * PITCH + d) * f[w];
            if (odd != 0) {
                for (unsigned long long left = odd & newRowsSeen(p, b, node, count); left != 0; left &= left - 1) {
                    const float* src = p.vNew + (size_t(b) * p.nodes + __ffsll(left) - 1) * kvDim + size_t(kh) * hd + d;
                    for (int j = 0; j < 4; ++j)
                        if (d + j < hd && !(fabsf(src[j]) < INFINITY)) acc[j] += src[j];
                }
            }
            if (MODE != 0 || !only) {
                storef4(dst + d, acc);
            } else {
                for (int j = 0; j < 4; ++j)
                    if (d + j < hd) dst[d + j] = acc[j];
            }
        }
        if (part == 0) {
            if (only) finishStats(p, plan, b, kh, row, most, sum, mx);
            if (plan.partStat) plan.partStat[entry + row] = float4v{most, sum, mx, 0.0f};
        }
    }
}

// A row's reference and sum over its chunks, by LANES neighbouring lanes; `at` + c * `step` is chunk c's entry
template <int LANES>
__device__ __forceinline__ float2 joinedSum(const TilePlan& plan, size_t at, size_t step, int chunks, float& mx) {
    const int lane = threadIdx.x % LANES;
    float most = kNoRef, sum = 0.0f;
    for (int c = lane; c < chunks; c += LANES) most = fmaxf(most, plan.partStat[at + c * step].x);
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, 64));
    mx = -INFINITY;
    for (int c = lane; c < chunks; c += LANES) {
        const float4v st = plan.partStat[at + c * step];
        sum += st.y * __builtin_amdgcn_exp2f(st.x - most);
        mx = fmaxf(mx, st.z);
    }
#pragma unroll
    for (int off = LANES / 2; off > 0; off >>= 1) {
        sum += __shfl_xor(sum, off, 64);
        mx = fmaxf(mx, __shfl_xor(mx, off, 64));
    }
    return make_float2(most, sum);
}

// The weights of a block of 1024 cached rows, four a thread, from the kept dot products of the group's rows, of which there
// are four at most; the block of the first ones also makes the new rows'.  The statistics are put together here once more, a
// row by each wavefront, rather than waited for in a launch of their own.
__device__ __forceinline__ void weightsFromScores(const TreeParams& p, const TilePlan& plan, int index) {
    __shared__ float2 sStat[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int block = index % plan.keyBlocks, g = index / plan.keyBlocks % p.groups, b = index / plan.keyBlocks / p.groups;
    const int share = p.heads / p.kvHeads, rows = p.nodes * share, length = rowsInUse(p, b), count = nodesInUse(p, b), live = count * share;
    if (block != 0 && block * 1024 >= length) return;
    const int perGroup = p.kvHeads / p.groups, kh0 = g * perGroup, all = perGroup * live;
    const size_t at = (size_t(b) * p.groups + g) * p.capacity, step = size_t(p.kvHeads) * rows;
    const int j = block * 1024 + int(threadIdx.x) * 4, fresh = threadIdx.x;
    const bool cached = j < length, isNew = block == 0 && fresh < count && length + fresh < p.capacity;
    if (wave < all) {
        const int2 span = plan.span[b];
        float mx;
        const float2 st = joinedSum<64>(plan, size_t(span.x) * step + size_t(kh0 + wave / live) * rows + wave % live, step, span.y, mx);
        if (lane == 0) sStat[wave] = make_float2(st.x, st.y == 0.0f ? 0.0f : 1.0f / st.y);
    }
    __syncthreads();
    float4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
    float newSum = 0.0f;
#pragma unroll 4
    for (int n = 0; n < all; ++n) {
        const size_t row = (size_t(b) * p.kvHeads + kh0 + n / live) * rows + n % live;
        const float2 st = sStat[n];
        if (cached) {
            const float4v x = loadf4(plan.scores + row * plan.scorePitch + j);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += __builtin_amdgcn_exp2f(fmaf(x[e], plan.c, -st.x)) * st.y;
        }
        if (isNew) newSum += __builtin_amdgcn_exp2f(fmaf(plan.newScores[row * 64 + fresh], plan.c, -st.x)) * st.y;
    }
    if (cached) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (j + e < length) p.weightsOut[at + j + e] = (p.weightsIn ? p.weightsIn[at + j + e] : 0.0f) + sum[e];
    }
    if (isNew) p.weightsOut[at + length + fresh] = newSum;
}

// The weights of 64 cached rows from the kept dot products and the rows' statistics, or (block 0) those of the new rows, in
// a launch of its own: sixteen lanes have four keys each, and the sixteen such groups take every sixteenth row.
__global__ void __launch_bounds__(256) rowWeightsKernel(TreeParams p, TilePlan plan) {
    __shared__ float4v sSum[16][17];
    const int sub = threadIdx.x & 15, part = threadIdx.x >> 4;
    const int block = blockIdx.x % plan.keyBlocks, g = blockIdx.x / plan.keyBlocks % p.groups, b = blockIdx.x / plan.keyBlocks / p.groups;
    const int share = p.heads / p.kvHeads, rows = p.nodes * share, length = rowsInUse(p, b), count = nodesInUse(p, b), live = count * share;
    const int first = block == 0 ? 0 : (block - 1) * 64, keys = block == 0 ? min(count, p.capacity - length) : min(64, length - first);
    if (keys <= 0) return;
    const int perGroup = p.kvHeads / p.groups;
    const size_t pitch = block == 0 ? 64 : plan.scorePitch, row0 = (size_t(b) * p.kvHeads + size_t(g) * perGroup) * rows;
    const float* from = (block == 0 ? plan.newScores : plan.scores) + row0 * pitch + min(first + sub * 4, int(pitch) - 4);
    const float2* stat = plan.rowStat + row0;
    const int over = max(1, live), khStep = 16 / over, rowStep = 16 % over;
    int kh = part / over, row = part % over;
    float4v sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int n = part; n < perGroup * live; n += 16) {
        const size_t at = size_t(kh) * rows + row;
        const float2 st = stat[at];
        const float4v x = loadf4(from + at * pitch);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += __builtin_amdgcn_exp2f(fmaf(x[e], plan.c, -st.x)) * st.y;
        row += rowStep;
        kh += khStep + (row >= live);
        row -= row >= live ? live : 0;
    }
    sSum[part][sub] = sum;
    __syncthreads();
    if (int(threadIdx.x) >= keys) return;
    const int of = threadIdx.x / 4, e = threadIdx.x % 4;
    float all = 0.0f;
#pragma unroll
    for (int n = 0; n < 16; ++n) all += sSum[n][of][e];
    const size_t at = (size_t(b) * p.groups + g) * p.capacity + (block == 0 ? length : first) + threadIdx.x;
    p.weightsOut[at] = block != 0 && p.weightsIn ? p.weightsIn[at] + all : all;
}

// A step without new tokens: the weights of the rows in use carried over (zeros without weightsIn).
__global__ void __launch_bounds__(256) carryWeightsKernel(TreeParams p) {
    const int j = int(blockIdx.x) * 256 + int(threadIdx.x), g = blockIdx.y, b = blockIdx.z;
    if (j >= rowsInUse(p, b)) return;
    const size_t at = (size_t(b) * p.groups + g) * p.capacity + j;
    p.weightsOut[at] = p.weightsIn ? p.weightsIn[at] : 0.0f;
}

// The chunks of a row put together.  LPR lanes hold a row's columns, four each.  Few chunks a row (MANY false): every LPR
// lanes have a row of their own and take its chunks in turn, so that few wavefronts wait out the chain of loads (24000 rows
// of three chunks: 15 us with a wavefront each).  Many: a workgroup a row, 256 / LPR chunks at once.  Workgroups past
// `joinBlocks` make the weights.
template <int LPR, bool MANY>
__global__ void __launch_bounds__(256) treeJoinKernel(TreeParams p, TilePlan plan, unsigned joinBlocks) {
    constexpr int STEP = MANY ? 256 / LPR : 1;
    __shared__ float4v sAcc[4][LPR];
    if (blockIdx.x >= joinBlocks) {
        weightsFromScores(p, plan, int(blockIdx.x - joinBlocks));
        return;
    }
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, share = p.heads / p.kvHeads, rows = p.nodes * share, sub = lane % LPR;
    const size_t flat = MANY ? blockIdx.x : size_t(blockIdx.x) * (256 / LPR) + threadIdx.x / LPR;
    if (flat >= size_t(p.batch) * p.kvHeads * rows) return;
    const int row = int(flat % rows), kh = int(flat / rows % p.kvHeads), b = int(flat / rows / p.kvHeads);
    const int2 span = plan.span[b];
    if (row >= nodesInUse(p, b) * share || span.y == 1) return;   // no such row, or written by its only chunk
    const size_t step = size_t(p.kvHeads) * rows, at = size_t(span.x) * step + size_t(kh) * rows + row;
    float mx;
    const float2 total = joinedSum<MANY ? 64 : LPR>(plan, at, step, span.y, mx);
    float4v acc = {0.0f, 0.0f, 0.0f, 0.0f};
    const bool on = sub * 4 < p.hd;
#pragma unroll 4
    for (int c = MANY ? int(threadIdx.x) / LPR : 0; c < span.y; c += STEP) {
        const float f = __builtin_amdgcn_exp2f(plan.partStat[at + c * step].x - total.x);
        const float4v x = on ? loadf4(plan.partOut + (at + c * step) * plan.partPitch + sub * 4) : float4v{0.0f, 0.0f, 0.0f, 0.0f};
        acc = acc + x * f;
    }
    if constexpr (MANY) {
#pragma unroll
        for (int off = LPR; off < 64; off <<= 1)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] += __shfl_xor(acc[j], off, 64);
        if (lane < LPR) sAcc[wave][lane] = acc;
        __syncthreads();
        if (threadIdx.x >= LPR) return;
        acc = (sAcc[0][sub] + sAcc[1][sub]) + (sAcc[2][sub] + sAcc[3][sub]);
    }
    const float inv = total.y == 0.0f ? 0.0f : 1.0f / total.y;
    float* dst = p.out + (size_t(b) * p.nodes + row / share) * p.heads * p.hd + size_t(kh * share + row % share) * p.hd + sub * 4;
#pragma unroll
    for (int j = 0; j < 4; ++j)
        if (sub * 4 + j < p.hd) dst[j] = acc[j] * inv;
    if (sub == 0) finishStats(p, plan, b, kh, row, total.x, total.y, mx);
}

// ---- the weight of keys from statistics --------------------------------------------------------
struct KeyWeightParams {
    const float* q; const float* k; const float* m; const float* l;
    const int* counts;     // queries of each sequence that count (NULL: all)
    const int* lengths;    // keys of each sequence that are in use (NULL: totalLen)
    const float* weightsIn; float* weightsOut;
    float* part;           // [batch][heads][queryChunks][totalLen] sums over a chunk of queries
    int batch, heads, kvHeads, groups, newLen, totalLen, kvRows, hd, oldLen, weightRows;
    int keyBlocks, queryChunk, queryChunks;
    float scale;
};

// What sequence b has in use
__device__ __forceinline__ int queriesOf(const KeyWeightParams& p, int b) { return p.counts ? min(max(p.counts[b], 0), p.newLen) : p.newLen; }
__device__ __forceinline__ int keysOf(const KeyWeightParams& p, int b) { return p.lengths ? min(max(p.lengths[b], 0), p.totalLen) : p.totalLen; }
// Queries of chunk c that see a key of a block starting at `key`: [from, to), empty if from >= to
__device__ __forceinline__ int2 queriesOfChunk(const KeyWeightParams& p, int queries, int c, int key) {
    return make_int2(max(c * p.queryChunk, (key - p.oldLen) & ~15), min((c + 1) * p.queryChunk, queries));
}

// sum_i exp(s_ij - m_i) / l_i with the keys' owner as the workgroup: a wavefront holds KT tiles of 16 keys as B operands and
// walks the queries 16 at a time, S = Q K^T leaving a lane with 4 queries of one key, whose probabilities it adds up; no
// lane needs another's until the end.  For few queries (a tree's), where reading the keys bounds the pass, and head dims
// above 128; the prompts of 8192 and 1934 tokens below took 2.7 ms with it (54 TFLOP/s, its queries' loads exposed).
// The four wavefronts of a workgroup take neighbouring keys and the same queries.
template <int HDP, int KT, int MODE>
__global__ void __launch_bounds__(256, 2) keyWeightTilesKernel(KeyWeightParams p) {
    constexpr int KS = HDP / 16;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, g = lane >> 4;
    // chunks of queries outermost and the blocks of keys with the most queries (the lowest) first
    const size_t pairs = size_t(p.batch) * p.heads;
    const size_t flat = blockIdx.x;
    const int h = int(flat % pairs % p.heads), b = int(flat % pairs / p.heads);
    const int block = int(flat / pairs) % p.keyBlocks, chunk = int(flat / pairs) / p.keyBlocks;
    const int keys = keysOf(p, b), key0 = block * KT * 64, mine = key0 + wave * KT * 16;
    const int2 span = queriesOfChunk(p, queriesOf(p, b), chunk, key0);
    if (mine >= keys || span.x >= span.y) return;
    const int hd = p.hd, kh = h / (p.heads / p.kvHeads);
    const size_t kvDim = size_t(p.kvHeads) * hd, dim = size_t(p.heads) * hd;
    float k[KT][KS][4];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const float* src = p.k + (size_t(b) * p.kvRows + min(mine + t * 16 + i16, keys - 1)) * kvDim + size_t(kh) * hd;
#pragma unroll
        for (int s = 0; s < KS; ++s) loadColumns<MODE, 4>(k[t][s], src, 16 * s + 4 * g, hd);
    }
    const float* qb = p.q + size_t(b) * p.newLen * dim + size_t(h) * hd;
    const float* mb = p.m + (size_t(b) * p.heads + h) * p.newLen;
    const float* lb = p.l + (size_t(b) * p.heads + h) * p.newLen;
    float q[KS][4], m[4], l[4], sum[KT] = {};
    auto load = [&](int i) {
        const float* src = qb + size_t(min(i + i16, span.y - 1)) * dim;
#pragma unroll
        for (int s = 0; s < KS; ++s) fetchColumns<MODE>(q[s], src, 16 * s + 4 * g, hd);   // past the end they meet zeros of the keys
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = min(i + 4 * g + r, span.y - 1);
            m[r] = mb[row];
            l[r] = lb[row];
        }
    };
    // queries below `mine - oldLen` see none of this wavefront's keys
    int i = max(span.x, (mine - p.oldLen) & ~15);
    if (i < span.y) load(i);
    for (; i < span.y; i += 16) {
        const bool whole = i + 16 <= span.y && mine + KT * 16 - 1 <= p.oldLen + i;   // every pair seen
        float4v dots[KT];
        float top[4], over[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            over[r] = l[r] != 0.0f ? __builtin_amdgcn_rcpf(l[r]) : 0.0f;
            top[r] = l[r] != 0.0f ? m[r] : INFINITY;      // a row that saw nothing gives nothing
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            float4v even = {0.0f, 0.0f, 0.0f, 0.0f}, odd = even;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                even = __builtin_amdgcn_mfma_f32_16x16x4f32(q[s][0], k[t][s][0], even, 0, 0, 0);
                odd = __builtin_amdgcn_mfma_f32_16x16x4f32(q[s][1], k[t][s][1], odd, 0, 0, 0);
                even = __builtin_amdgcn_mfma_f32_16x16x4f32(q[s][2], k[t][s][2], even, 0, 0, 0);
                odd = __builtin_amdgcn_mfma_f32_16x16x4f32(q[s][3], k[t][s][3], odd, 0, 0, 0);
            }
            dots[t] = even + odd;
        }
        if (i + 16 < span.y) load(i + 16);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            float w[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) w[r] = __builtin_amdgcn_exp2f((dots[t][r] * p.scale - top[r]) * kLog2e) * over[r];
            if (!whole) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = i + 4 * g + r;
                    w[r] = row < span.y && mine + t * 16 + i16 <= p.oldLen + row ? w[r] : 0.0f;
                }
            }
            sum[t] += (w[0] + w[1]) + (w[2] + w[3]);
        }
    }
    float* dst = p.part + ((size_t(b) * p.heads + h) * p.queryChunks + chunk) * p.totalLen;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        sum[t] += __shfl_xor(sum[t], 16, 64);
        sum[t] += __shfl_xor(sum[t], 32, 64);
        const int key = mine + t * 16 + i16;
        if (g == 0 && key < keys) dst[key] = sum[t];
    }
}

// The same with every fp32 product as six bf16 ones (v_mfma_f32_16x16x32_bf16), for passes of many queries, which are
// bound by the matrix instruction: an fp32 value is the exact sum of three bf16 terms, x = h + m + l, and h h', h m', m h',
// h l', l h', m m' hold everything above 2^-24 of the product, at 6/16 of the fp32 instruction's time.  h h' and the rest
// are two accumulators, so that the small terms are added among themselves first.
//
// The keys' terms stay in registers; 32 queries at a time are split once for the four wavefronts and handed over through
// LDS (two buffers, one barrier a step, the next step's rows in flight in registers meanwhile), their maxima and reciprocal
// sums beside them.  2 prompts of 8192 and 1934 tokens, 16 heads of 128: 1.03 ms = 141 TFLOP/s of fp32 products, 0.85 PFLOP/s
// of bf16 ones; 8 of 1024, 12 heads of 64: 51 us.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
struct Terms { bf16x8 t[3]; };
__device__ __forceinline__ Terms splitTerms(const float (&x)[8]) {
    Terms out;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const __bf16 h = static_cast<__bf16>(x[j]);
        const float r1 = x[j] - static_cast<float>(h);
        const __bf16 m = static_cast<__bf16>(r1);
        out.t[0][j] = h;
        out.t[1][j] = m;
        out.t[2][j] = static_cast<__bf16>(r1 - static_cast<float>(m));
    }
    return out;
}
template <int HDP, int KT, int MODE>
__global__ void __launch_bounds__(256, 2) keyWeightSplitKernel(KeyWeightParams p) {
    constexpr int ST = HDP / 32, PITCH = HDP + 8, ROWS = 32, CHUNKS = ROWS * HDP / 8, PER = (CHUNKS + 255) / 256;
    __shared__ __attribute__((aligned(16))) __bf16 sQ[2][3][ROWS][PITCH];
    __shared__ __attribute__((aligned(16))) float sTop[2][ROWS], sOver[2][ROWS];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, i16 = lane & 15, g = lane >> 4;
    const size_t pairs = size_t(p.batch) * p.heads;
    const size_t flat = blockIdx.x;
    const int h = int(flat % pairs % p.heads), b = int(flat % pairs / p.heads);
    const int block = int(flat / pairs) % p.keyBlocks, chunk = int(flat / pairs) / p.keyBlocks;
    const int keys = keysOf(p, b), key0 = block * KT * 64, mine = key0 + wave * KT * 16;
    const int2 span = queriesOfChunk(p, queriesOf(p, b), chunk, key0);
    if (key0 >= keys || span.x >= span.y) return;
    const int hd = p.hd, kh = h / (p.heads / p.kvHeads);
    const size_t kvDim = size_t(p.kvHeads) * hd, dim = size_t(p.heads) * hd;
    Terms k[KT][ST];
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        const float* src = p.k + (size_t(b) * p.kvRows + min(mine + t * 16 + i16, keys - 1)) * kvDim + size_t(kh) * hd;
#pragma unroll
        for (int s = 0; s < ST; ++s) {
            float x[2][4], y[8];
            loadColumns<MODE, 4>(x[0], src, 32 * s + 8 * g, hd);
            loadColumns<MODE, 4>(x[1], src, 32 * s + 8 * g + 4, hd);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] = x[j / 4][j % 4];
            k[t][s] = splitTerms(y);
        }
    }
    const float* qb = p.q + size_t(b) * p.newLen * dim + size_t(h) * hd;
    const float* mb = p.m + (size_t(b) * p.heads + h) * p.newLen;
    const float* lb = p.l + (size_t(b) * p.heads + h) * p.newLen;
    float q[PER][2][4], m = 0.0f, l = 0.0f, sum[KT] = {};
    auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int e = int(threadIdx.x) + 256 * u, row = e / (HDP / 8), col = e % (HDP / 8) * 8;
            if (CHUNKS % 256 == 0 || e < CHUNKS) {
                const float* src = qb + size_t(min(i0 + row, span.y - 1)) * dim;
                fetchColumns<MODE>(q[u][0], src, col, hd);       // past the end they meet zeros of the keys
                fetchColumns<MODE>(q[u][1], src, col + 4, hd);
            }
        }
        if (threadIdx.x < ROWS) {
            const int row = min(i0 + int(threadIdx.x), span.y - 1);
            m = mb[row];
            l = lb[row];
        }
    };
    auto stage = [&](int buf) {
#pragma unroll
        for (int u = 0; u < PER; ++u) {
            const int e = int(threadIdx.x) + 256 * u, row = e / (HDP / 8), col = e % (HDP / 8) * 8;
            if (CHUNKS % 256 == 0 || e < CHUNKS) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = q[u][j / 4][j % 4];
                const Terms t = splitTerms(y);
#pragma unroll
                for (int x = 0; x < 3; ++x) *reinterpret_cast<bf16x8*>(&sQ[buf][x][row][col]) = t.t[x];
            }
        }
        if (threadIdx.x < ROWS) {
            sTop[buf][threadIdx.x] = l != 0.0f ? m : INFINITY;      // a row that saw nothing gives nothing
            sOver[buf][threadIdx.x] = l != 0.0f ? __builtin_amdgcn_rcpf(l) : 0.0f;
        }
    };
    load(span.x);
    stage(0);
    __syncthreads();
    int buf = 0;
    for (int i0 = span.x; i0 < span.y; i0 += ROWS, buf ^= 1) {
        const bool more = i0 + ROWS < span.y;
        if (more) load(i0 + ROWS);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int i = i0 + half * 16;
            // none of these queries counts, or sees one of this wavefront's keys
            if (mine >= keys || i >= span.y || i + 15 + p.oldLen < mine) continue;
            const bool whole = i + 16 <= span.y && mine + KT * 16 - 1 <= p.oldLen + i;
            float4v large[KT], small[KT];
#pragma unroll
            for (int t = 0; t < KT; ++t) large[t] = small[t] = float4v{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < ST; ++s) {
                bf16x8 a[3];
#pragma unroll
                for (int x = 0; x < 3; ++x) a[x] = *reinterpret_cast<const bf16x8*>(&sQ[buf][x][half * 16 + i16][32 * s + 8 * g]);
#pragma unroll
                for (int t = 0; t < KT; ++t) {
                    small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[2], k[t][s].t[0], small[t], 0, 0, 0);
                    large[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], k[t][s].t[0], large[t], 0, 0, 0);
                }
#pragma unroll
                for (int t = 0; t < KT; ++t) small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], k[t][s].t[2], small[t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < KT; ++t) small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], k[t][s].t[1], small[t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < KT; ++t) small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[1], k[t][s].t[0], small[t], 0, 0, 0);
#pragma unroll
                for (int t = 0; t < KT; ++t) small[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[0], k[t][s].t[1], small[t], 0, 0, 0);
            }
            const float4v top = *reinterpret_cast<const float4v*>(&sTop[buf][half * 16 + 4 * g]);
            const float4v over = *reinterpret_cast<const float4v*>(&sOver[buf][half * 16 + 4 * g]);
#pragma unroll
            for (int t = 0; t < KT; ++t) {
                const float4v dots = large[t] + small[t];
                float w[4];
#pragma unroll
                for (int r = 0; r < 4; ++r) w[r] = __builtin_amdgcn_exp2f(fmaf(dots[r], p.scale, -top[r]) * kLog2e) * over[r];
                if (!whole) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int row = i + 4 * g + r;
                        w[r] = row < span.y && mine + t * 16 + i16 <= p.oldLen + row ? w[r] : 0.0f;
                    }
                }
                sum[t] += (w[0] + w[1]) + (w[2] + w[3]);
            }
        }
        if (more) stage(buf ^ 1);
        __syncthreads();
    }
    float* dst = p.part + ((size_t(b) * p.heads + h) * p.queryChunks + chunk) * p.totalLen;
#pragma unroll
    for (int t = 0; t < KT; ++t) {
        sum[t] += __shfl_xor(sum[t], 16, 64);
        sum[t] += __shfl_xor(sum[t], 32, 64);
        const int key = mine + t * 16 + i16;
        if (g == 0 && key < keys) dst[key] = sum[t];
    }
}

// The sums of a group's heads and of the chunks of queries added up, in order.
__global__ void __launch_bounds__(256) keyWeightJoinKernel(KeyWeightParams p, int keysPerBlock) {
    const int j = int(blockIdx.x) * 256 + int(threadIdx.x), g = blockIdx.y, b = blockIdx.z;
    if (j >= keysOf(p, b)) return;
    const int queries = queriesOf(p, b), perGroup = p.heads / p.groups, key0 = j / keysPerBlock * keysPerBlock;
    float sum = 0.0f;
    for (int h = g * perGroup; h < (g + 1) * perGroup; ++h) {
        const float* src = p.part + (size_t(b) * p.heads + h) * p.queryChunks * p.totalLen + j;
        for (int c = 0; c < p.queryChunks; ++c) {
            const int2 span = queriesOfChunk(p, queries, c, key0);
            if (span.x < span.y) sum += src[size_t(c) * p.totalLen];
        }
    }
    const size_t at = (size_t(b) * p.groups + g) * p.weightRows + j;
    p.weightsOut[at] = (p.weightsIn ? p.weightsIn[at] : 0.0f) + sum;
}

// ---- launches ----------------------------------------------------------------------------------
bool aligned16(std::initializer_list<const void*> ptrs) {
    uintptr_t bits = 0;
    for (const void* x : ptrs) bits |= reinterpret_cast<uintptr_t>(x);
    return (bits & 15u) == 0;
}
int paddedHeadDim(size_t hd) { return hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 128 ? 128 : hd <= 192 ? 192 : 256; }

template <int HDP, int KT>
int launchKeyTiles(const KeyWeightParams& p, int mode, size_t grid, hipStream_t s) {
    if (mode == 2) keyWeightTilesKernel<HDP, KT, 2><<<unsigned(grid), 256, 0, s>>>(p);
    else if (mode == 1) keyWeightTilesKernel<HDP, KT, 1><<<unsigned(grid), 256, 0, s>>>(p);
    else keyWeightTilesKernel<HDP, KT, 0><<<unsigned(grid), 256, 0, s>>>(p);
    BF_LAUNCH_CHECK();
    return BF_OK;
}

template <int HDP, int KT>
int launchKeySplit(const KeyWeightParams& p, int mode, size_t grid, hipStream_t s) {
    if (mode == 2) keyWeightSplitKernel<HDP, KT, 2><<<unsigned(grid), 256, 0, s>>>(p);
    else if (mode == 1) keyWeightSplitKernel<HDP, KT, 1><<<unsigned(grid), 256, 0, s>>>(p);
    else keyWeightSplitKernel<HDP, KT, 0><<<unsigned(grid), 256, 0, s>>>(p);
    BF_LAUNCH_CHECK();
    return BF_OK;
}

// many queries: bound by the products, which the bf16 route does faster; few: by reading the keys
bool splitProducts(const KeyWeightParams& p) { return paddedHeadDim(size_t(p.hd)) <= 128 && p.newLen > 64; }
int keysPerBlock(const KeyWeightParams& p) {
    const int hdp = paddedHeadDim(size_t(p.hd));
    return (hdp > 128 || (splitProducts(p) && hdp == 128) ? 2 : 4) * 64;
}

// The chunks of queries; a shape too large is refused here, before anything is launched
int planKeyWeights(const char* fn, KeyWeightParams& p) {
    p.keyBlocks = (p.totalLen + keysPerBlock(p) - 1) / keysPerBlock(p);
    const size_t pairs = size_t(p.batch) * p.heads, blocks = pairs * p.keyBlocks;
    // Queries a workgroup walks: as many as leave three workgroups a compute unit (8 prompts of 1024 tokens, 12 heads: 62, 56, 53,
    // 67 us with 128, 256, 512, 1024; one of 4096: 101, 95, 92, 158 with 256 to 2048)
    int chunk = 2048;
    while (chunk > 128 && blocks * size_t((p.newLen + chunk - 1) / chunk) < size_t(computeUnits()) * 3) chunk /= 2;
    while (chunk < p.newLen && chunk < (1 << 30) && pairs * size_t((p.newLen + chunk - 1) / chunk) * p.totalLen > (size_t(1) << 28)) chunk *= 2;   // sums of 1 GiB, or one chunk's
    p.queryChunk = chunk;
    p.queryChunks = std::max(1, (p.newLen + chunk - 1) / chunk);
    return blocks * p.queryChunks > mostBlocks(256) ? failInvalid(fn, "shape too large") : BF_OK;
}

int keyWeights(KeyWeightParams p, hipStream_t s) {
    const int hdp = paddedHeadDim(size_t(p.hd));
    const bool split = splitProducts(p);
    const size_t pairs = size_t(p.batch) * p.heads, grid = pairs * p.keyBlocks * p.queryChunks;
    Scratch part(pairs * p.queryChunks * p.totalLen * sizeof(float));
    if (part.status != BF_OK) return part.status;
    p.part = part.as<float>();
    if (p.newLen > 0) {
        const int mode = p.hd % 4 != 0 || !aligned16({p.q, p.k}) ? 0 : p.hd == hdp ? 2 : 1;
        int st = BF_OK;
        if (split) {
            st = hdp == 32 ? launchKeySplit<32, 4>(p, mode, grid, s) : hdp == 64 ? launchKeySplit<64, 4>(p, mode, grid, s) : launchKeySplit<128, 2>(p, mode, grid, s);
        } else switch (hdp) {
            case 32: st = launchKeyTiles<32, 4>(p, mode, grid, s); break;
            case 64: st = launchKeyTiles<64, 4>(p, mode, grid, s); break;
            case 128: st = launchKeyTiles<128, 4>(p, mode, grid, s); break;
            case 192: st = launchKeyTiles<192, 2>(p, mode, grid, s); break;
            default: st = launchKeyTiles<256, 2>(p, mode, grid, s); break;
        }
        if (st != BF_OK) return st;
    }
    keyWeightJoinKernel<<<dim3(unsigned((p.totalLen + 255) / 256), unsigned(p.groups), unsigned(p.batch)), 256, 0, s>>>(p, keysPerBlock(p));
    BF_LAUNCH_CHECK();
    return BF_OK;
}

template <int HDP, int RT, int MODE, bool SCORES>
int launchTilesOf(const TreeParams& p, const TilePlan& plan, unsigned grid, hipStream_t s) {
    constexpr size_t smem = size_t(4) * RT * 16 * (HDP + 4) * sizeof(float);
    const int st = allowDynamicSharedMemory(reinterpret_cast<const void*>(treeTilesKernel<HDP, RT, MODE, SCORES>), smem);
    if (st != BF_OK) return st;
    treeTilesKernel<HDP, RT, MODE, SCORES><<<grid, 256, smem, s>>>(p, plan);
    BF_LAUNCH_CHECK();
    return BF_OK;
}
template <int HDP, int RT>
int launchTilesMode(const TreeParams& p, const TilePlan& plan, int mode, unsigned grid, hipStream_t s) {
    if (plan.scores) {
        if (mode == 2) return launchTilesOf<HDP, RT, 2, true>(p, plan, grid, s);
        if (mode == 1) return launchTilesOf<HDP, RT, 1, true>(p, plan, grid, s);
        return launchTilesOf<HDP, RT, 0, true>(p, plan, grid, s);
    }
    if (mode == 2) return launchTilesOf<HDP, RT, 2, false>(p, plan, grid, s);
    if (mode == 1) return launchTilesOf<HDP, RT, 1, false>(p, plan, grid, s);
    return launchTilesOf<HDP, RT, 0, false>(p, plan, grid, s);
}
template <int HDP>
int launchTilesRows(const TreeParams& p, const TilePlan& plan, int rt, int mode, unsigned grid, hipStream_t s) {
    if constexpr (HDP <= 64) {
        if (rt == 4) return launchTilesMode<HDP, 4>(p, plan, mode, grid, s);
    }
    if constexpr (HDP <= 192) {
        if (rt == 2) return launchTilesMode<HDP, 2>(p, plan, mode, grid, s);
    }
    return launchTilesMode<HDP, 1>(p, plan, mode, grid, s);
}
int launchTiles(const TreeParams& p, const TilePlan& plan, int hdp, int rt, int mode, unsigned grid, hipStream_t s) {
    switch (hdp) {
        case 32: return launchTilesRows<32>(p, plan, rt, mode, grid, s);
        case 64: return launchTilesRows<64>(p, plan, rt, mode, grid, s);
        case 96: return launchTilesRows<96>(p, plan, rt, mode, grid, s);
        case 128: return launchTilesRows<128>(p, plan, rt, mode, grid, s);
        case 192: return launchTilesRows<192>(p, plan, rt, mode, grid, s);
        default: return launchTilesRows<256>(p, plan, rt, mode, grid, s);
    }
}

template <int LPR>
int launchJoinOf(const TreeParams& p, const TilePlan& plan, size_t rows, size_t weightBlocks, hipStream_t s) {
    // A workgroup a row where there is room for more than four chunks a sequence, unless the rows' lanes alone give every SIMD
    // two wavefronts (their sequences then have 17 chunks at most).  A workgroup each against lanes each: one node over 8000
    // rows, 8 heads of 64, 13 against 21 us, 64 nodes 21 and 24; 26 nodes over 120011 rows, 16 heads of 128, 322 and 333; more
    // lanes than the bound: 64 nodes over 32 ragged sequences, 12 heads, 181 and 154, over 16 x 4000 rows, 8 heads of 128, 173
    // and 161.  Up to four chunks it is the same within 5 %; close below the bound the workgroups lose up to 10 % (64 nodes
    // over 8 x 4000 rows, 16 heads of 64: 101 and 91).
    const bool many = size_t(plan.items) > size_t(p.batch) * 4 && rows * LPR <= size_t(computeUnits()) * 512;
    const size_t blocks = size_t(plan.items) == size_t(p.batch) ? 0 : many ? rows : (rows * LPR + 255) / 256;   // one chunk each: nothing to join
    if (blocks + weightBlocks == 0) return BF_OK;
    if (many) treeJoinKernel<LPR, true><<<unsigned(blocks + weightBlocks), 256, 0, s>>>(p, plan, unsigned(blocks));
    else treeJoinKernel<LPR, false><<<unsigned(blocks + weightBlocks), 256, 0, s>>>(p, plan, unsigned(blocks));
    BF_LAUNCH_CHECK();
    return BF_OK;
}
int joinLanes(size_t hd) { return hd <= 32 ? 8 : hd <= 64 ? 16 : hd <= 128 ? 32 : 64; }
int launchJoin(const TreeParams& p, const TilePlan& plan, size_t rows, size_t weightBlocks, hipStream_t s) {
    switch (joinLanes(size_t(p.hd))) {
        case 8: return launchJoinOf<8>(p, plan, rows, weightBlocks, s);
        case 16: return launchJoinOf<16>(p, plan, rows, weightBlocks, s);
        case 32: return launchJoinOf<32>(p, plan, rows, weightBlocks, s);
        default: return launchJoinOf<64>(p, plan, rows, weightBlocks, s);
    }
}

int checkHeads(const char* fn, size_t heads, size_t kvHeads, size_t groups, size_t headDim) {
    if (heads == 0 || kvHeads == 0 || heads % kvHeads != 0)
        return failInvalid(fn, "kvHeads (" + std::to_string(kvHeads) + ") must divide the number of heads (" + std::to_string(heads) + ")");
    if (groups == 0 || kvHeads % groups != 0)
        return failInvalid(fn, "groups (" + std::to_string(groups) + ") must divide kvHeads (" + std::to_string(kvHeads) + ")");
    if (headDim > 256) return failInvalid(fn, "headDim (" + std::to_string(headDim) + ") exceeds the supported limit (256)");
    if (heads >= (size_t(1) << 16) || heads / kvHeads > 4096) return failInvalid(fn, "shape too large");
    return BF_OK;
}

int treeAttention(const char* fn, TreeParams p, size_t batch, size_t heads, size_t kvHeads, size_t groups, size_t nodes, size_t capacity,
                  size_t headDim, bool weights, bf_stream_t stream) {
    int st = checkHeads(fn, heads, kvHeads, groups, headDim);
    if (st != BF_OK) return st;
    if (nodes > 64) return failInvalid(fn, "a tree has at most 64 nodes, got " + std::to_string(nodes));
    if (batch >= (size_t(1) << 16) || capacity >= (size_t(1) << 30)) return failInvalid(fn, "shape too large");
    if (batch == 0) return BF_OK;
    if (nodes == 0 || headDim == 0) {
        if (!weights || capacity == 0) return BF_OK;
        if (!p.lengths || !p.weightsOut) return failInvalid(fn, "NULL pointer");
        if (p.weightsIn == p.weightsOut) return BF_OK;
        p.groups = int(groups); p.capacity = int(capacity);
        carryWeightsKernel<<<dim3(unsigned((capacity + 255) / 256), unsigned(groups), unsigned(batch)), 256, 0, asStream(stream)>>>(p);
        BF_LAUNCH_CHECK();
        return BF_OK;
    }
    if (!p.q || !p.kNew || !p.vNew || !p.lengths || !p.out || (capacity != 0 && (!p.k || !p.v)) || (weights && capacity != 0 && !p.weightsOut))
        return failInvalid(fn, "NULL pointer");
    p.batch = int(batch); p.heads = int(heads); p.kvHeads = int(kvHeads); p.groups = int(groups); p.nodes = int(nodes);
    p.capacity = int(capacity); p.hd = int(headDim);
    const size_t share = heads / kvHeads, rows = nodes * share;
    // The weights come from the dot products that the pass leaves in a workspace, up to 1 GiB of it (or 64 bytes a key and key
    // head); past that they are made again from the keys (20 nodes over 4 x 8100 rows, 8 heads of 64: 44 us against 60; 64
    // nodes 72 against 95; 512 rows to a key head 481 against 510), which takes sums of 4 bytes a key and query head, one part
    // in `nodes` of what is kept: with three nodes or fewer that saves too little (one node over 500000 rows, 128 heads on one
    // key head of 128: 0.39 ms kept, 5.0 made again; three 1.2 and 5.8; 32 heads on one of 64, 1000000 rows: 0.20 and 1.4).
    const size_t scoreBytes = batch * kvHeads * rows * ((capacity + 15) / 16 * 16) * sizeof(float);
    const bool keepScores = weights && capacity != 0 && (nodes <= 3 || rows <= 16 || scoreBytes <= size_t(1) << 30);
    const bool recompute = weights && capacity != 0 && !keepScores;
    // Row tiles a wavefront holds: what the rows fill, up to the registers there are (two tiles of 192 columns halve the reads,
    // 98 -> 90 us for 17 nodes over 4 x 8192 rows, 8 heads; of 256 they spill and take two thirds longer).  With less to do, two
    // at most, and one where the tiles of all sequences are half the compute units at most: more workgroups, and each starts and ends sooner.  The
    // measure is keys (by the capacity) x row tiles x columns, 0.75 and 2 times 2^18 of them a compute unit.  53 nodes over 700 rows, 8
    // heads of 64: 12, 14, 19 us with one, two, four; over 30000 rows 48, 51, 53; over 10 x 2000 55, 49, 50; 64 nodes over 32
    // ragged sequences, 12 heads: 193, 157, 154; heads of 128, 24 nodes over 3 x 8000 rows: 43, 50, 53 nodes 79, 73.  Lengths far
    // below the capacity are not known here: 64 nodes over 4 x 256 rows of room for 8192, 8 heads of 64: 15, 18, 24 us.
    const int hdp = headDim > 64 && headDim <= 96 ? 96 : paddedHeadDim(headDim);
    const size_t device = size_t(computeUnits()), tiles = batch * kvHeads * ((rows + 15) / 16);
    const double work = double(tiles) * double(capacity) * hdp / double(device << 18);
    const int most = work <= 0.75 && tiles * 2 <= device ? 1 : hdp <= 64 && work > 2.0 ? 4 : hdp <= 192 ? 2 : 1;
    const int rt = std::min(most, rows <= 16 ? 1 : rows <= 32 ? 2 : 4);
    TilePlan plan{};
    plan.rowGroups = int((rows + 16 * rt - 1) / (16 * rt));
    plan.minChunk = 128;
    // Chunk sizes by the rounds they make (bestChunk): with several row tiles on the workgroups whose registers a compute unit
    // holds (even shares of four a compute unit measured 337 us where that gives 327, 26 nodes over 120011 rows, and 160 where it
    // gives 151, 50000 rows), with one on the compute units, since longer chunks cost less than they lose in loads under way (one
    // node over 100000 rows, 2 heads of 64: 26 us, and 45 with even shares of eight a compute unit; 4 x 8192 rows, 8 heads of
    // 192: 84 and 109).  Many sequences: a chunk more or less of each matters too much, and the even shares of eight balance
    // them better (16 ragged sequences of up to 16000 rows, 16 heads of 128: 376 us, by rounds 387).
    const size_t pairs = kvHeads * size_t(plan.rowGroups);
    if (rt == 1 && batch * pairs * 2 > device) {
        plan.target = int(std::max<size_t>(1, device * 8 / pairs));
    } else {
        plan.slots = float(device * (rt == 1 ? 1 : hdp * rt <= 128 ? 3 : hdp <= 128 ? 2 : 1)) / float(pairs);
        plan.target = int(std::max<size_t>(1, size_t(3.0f * plan.slots + 0.5f))) + int(batch);
    }
    // Even shares are at most target + batch chunks, and so are those of bestChunk, whose own count may miss one a sequence
    const size_t chunksAtMost = batch * std::max<size_t>(1, (capacity + plan.minChunk - 1) / plan.minChunk);
    plan.items = int(std::min(chunksAtMost, size_t(plan.target) + batch));
    plan.c = float(std::fabs(double(p.scale)) * 1.4426950408889634074);
    plan.sign = plan.c == 0.0f ? 0.0f : p.scale < 0.0f ? -1.0f : 1.0f;
    if (plan.c == 0.0f) plan.c = 1.0f;      // what a row does not see stays at -inf, which 0 would turn into NaN
    plan.magic = unsigned(((size_t(1) << 32) + share - 1) / share);
    plan.scorePitch = int((capacity + 15) / 16 * 16);
    plan.partPitch = int((headDim + 3) / 4 * 4);
    const bool join = size_t(plan.items) > batch;
    const size_t slots = size_t(plan.items) * kvHeads * rows, rowsAll = batch * kvHeads * rows;
    // The join's launch makes the weights too where a group has a row for each wavefront of its workgroups at most: they put the
    // statistics together themselves (1024 rows, 12 groups of one head: 11 us against 14).  Else a launch of its own with the
    // statistics from the join (12 nodes, one group of 12 heads: 16 us against 123; 8 groups, 8192 rows: 46 against 48).
    const bool apart = recompute || (keepScores && kvHeads / groups * rows > 4);
    plan.keyBlocks = !keepScores ? 1 : apart ? int((capacity + 63) / 64) + 1 : int((capacity + 1023) / 1024);
    const size_t weightBlocks = weights && capacity != 0 ? batch * groups * size_t(plan.keyBlocks) : 0;
    const size_t grid = (size_t(plan.items) * kvHeads + 7) / 8 * 8 * size_t(plan.rowGroups);
    // (a workgroup a row joins where there are few rows only)
    const size_t joinBlocks = join ? (rowsAll * size_t(joinLanes(headDim)) + 255) / 256 : 0;
    if (grid > mostBlocks(256) || joinBlocks > mostBlocks(256) || joinBlocks * !apart + weightBlocks > mostBlocks(256))
        return failInvalid(fn, "shape too large");
    KeyWeightParams w{};
    if (recompute) {
        w.q = p.q; w.k = p.k; w.counts = p.counts; w.lengths = p.lengths; w.weightsIn = p.weightsIn; w.weightsOut = p.weightsOut;
        w.batch = p.batch; w.heads = p.heads; w.kvHeads = p.kvHeads; w.groups = p.groups; w.newLen = p.nodes; w.totalLen = p.capacity;
        w.kvRows = p.capacity; w.hd = p.hd; w.oldLen = p.capacity; w.weightRows = p.capacity; w.scale = p.scale;
        st = planKeyWeights(fn, w);
        if (st != BF_OK) return st;
    }
    const size_t need[] = {join || (weights && !apart) ? slots * sizeof(float4v) : 0, join ? slots * plan.partPitch * sizeof(float) : 0, batch * sizeof(int2),
                           keepScores ? rowsAll * size_t(plan.scorePitch) * sizeof(float) : 0, weights ? rowsAll * 64 * sizeof(float) : 0,
                           recompute && !(p.m && p.l) ? 2 * rowsAll * sizeof(float) : 0, apart ? rowsAll * sizeof(float2) : 0};
    hipStream_t s = asStream(stream);
    size_t bytes = 0, offset[7];
    for (int i = 0; i < 7; ++i) {
        offset[i] = bytes;
        bytes += (need[i] + 255) / 256 * 256;
    }
    Scratch own(bytes);
    if (own.status != BF_OK) return own.status;
    auto part = [&](int i) { return need[i] != 0 ? own.as<char>() + offset[i] : nullptr; };
    plan.partStat = reinterpret_cast<float4v*>(part(0));
    plan.partOut = reinterpret_cast<float*>(part(1));
    plan.span = reinterpret_cast<int2*>(part(2));
    plan.scores = reinterpret_cast<float*>(part(3));
    plan.newScores = reinterpret_cast<float*>(part(4));
    plan.rowStat = reinterpret_cast<float2*>(part(6));
    if (float* own2 = reinterpret_cast<float*>(part(5))) {
        if (!p.m) p.m = own2;
        if (!p.l) p.l = own2 + rowsAll;
    }
    const int mode = headDim % 4 != 0 || !aligned16({p.q, p.kNew, p.vNew, p.k, p.v, p.out}) ? 0 : headDim == size_t(hdp) ? 2 : 1;
    st = launchTiles(p, plan, hdp, rt, mode, unsigned(grid), s);
    if (st != BF_OK) return st;
    // the new rows' weights, and the cached rows' where their dot products were kept, ride on the launch that joins
    st = launchJoin(p, plan, rowsAll, apart ? 0 : weightBlocks, s);
    if (st != BF_OK) return st;
    if (apart) {
        rowWeightsKernel<<<unsigned(weightBlocks), 256, 0, s>>>(p, plan);
        BF_LAUNCH_CHECK();
    }
    if (recompute) {
        w.m = p.m; w.l = p.l;
        return keyWeights(w, s);
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
    st = planKeyWeights(__func__, p);
    return st != BF_OK ? st : keyWeights(p, asStream(stream));
}

}  // extern "C"

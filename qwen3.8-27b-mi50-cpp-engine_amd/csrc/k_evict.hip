// k_evict.hip -- eviction from a paged key/value cache by accumulated attention weight.
//
// Per sequence: acc[i] = decay acc[i] + sum over the accepted rows of w[row][i] (keys that came since the last call start
// at 0); where the cache has grown past `high` positions, the newest `recent` keys and the heaviest others stay, `budget`
// in all, ties to the lowest index. Attention does not care for the order of the keys, so nothing is shifted: the keys
// behind `budget` that stay move into the places of those before it that go, both in ascending order, as many bytes as
// can be. Source and target positions are disjoint, so the moves need no staging.
#include "q27x_paged.h"

namespace q27x {

struct EvictArgs {
    PagedArgs kv;
    const float* w; int w_stride; const int32_t* n_acc; int nrows; float decay;
    float* acc; int32_t* ord; int stride; int32_t* state;
    int high, budget, recent, max_len;
    int32_t* new_lens;
    uint32_t* rank;                 // [n_seq][max_len] the keys' order: larger stays
    int2* pairs;                    // [n_seq][max_len / 2 + 1] (from, to)
    int32_t* npairs;                // [n_seq]
    uint32_t *parts;                // [n_seq][blocks of k_evict_sums][3] its newest keys, least and largest other rank
    uint64_t *stay, *same;          // [n_seq][max_len / 64] a bit per key: above the cut, of the cut's rank
    int fused;                      // the kernel that picks also moves
};
constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / 64;

// Floats as unsigned numbers of the same order: -0 as 0, what is not a number below all others; the newest above all, and
// 0 for a place without a key.
constexpr uint32_t kNewest = 0xFFFFFFFFu, kNaN = 1u;
__device__ __forceinline__ uint32_t rank_of(float x) {
    if (x != x) return kNaN;
    const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

constexpr int kTiles = 32, kBins = 2048;
constexpr int kMaxKeys = 0x7fffffff - 64 * kEvThreads;     // (indexes run over by less than that)

// Exclusive prefix sum over the block's first n <= 1024 values, one a thread; the sum of all in `sum`.
__device__ __forceinline__ uint32_t scan_block(uint32_t x, uint32_t* red, uint32_t& sum) {
    const int l = threadIdx.x & 63, wv = threadIdx.x >> 6;
    uint32_t y = x;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t z = __shfl_up(y, o, 64);
        y += l >= o ? z : 0u;
    }
    __syncthreads();
    if (l == 63) red[wv] = y;
    __syncthreads();
    uint32_t before = 0;
    sum = 0;
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
        const uint32_t z = red[i];
        before += i < wv ? z : 0u;
        sum += z;
    }
    return before + y - x;
}

// A block's sequence.
struct EvictSeq {
    int first, rows, len, known, total, now, fresh;   // its rows of w, keys, keys with a sum, arrivals before and now, the first of the newest
    bool over;
    float* acc;
    int32_t* ord;
    int2* pairs;
};
__device__ __forceinline__ EvictSeq evict_seq(const EvictArgs& a, int b) {
    EvictSeq q;
    int n;
    paged_rows(a.kv, b, q.first, n);
    const long long cap = paged_cap(a.kv);
    int len = min(a.kv.lens[b], a.max_len);
    len = len < cap ? len : (int)cap;
    q.len = len < 0 ? 0 : len;
    const int known = max(a.state[2 * b], 0);
    q.known = min(known, q.len);
    q.total = a.state[2 * b + 1] - (known - q.known);         // (keys that were taken back came last: their numbers are free again)
    q.now = q.total + q.len - q.known;
    q.rows = a.w ? min(n, a.nrows - q.first) : 0;
    if (a.n_acc) q.rows = min(q.rows, a.n_acc[b]);
    q.over = q.len > a.high;
    q.fresh = q.now - a.recent;
    q.acc = a.acc + (size_t)b * a.stride;
    q.ord = a.ord + (size_t)b * a.stride;
    q.pairs = a.pairs + (size_t)b * (a.max_len / 2 + 1);
    return q;
}
// The thread's sums of keys i, i + 1024 .. , eight with their loads together, and their ranks. q.len > 0.
__device__ __forceinline__ void add_up(const EvictArgs& a, const EvictSeq& q, int i0, uint32_t (&key)[8]) {
    float x[8];
    int o[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int j = min(i0 + u * kEvThreads, q.len - 1);
        x[u] = q.acc[j];
        o[u] = q.ord[j];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kEvThreads;
        x[u] = i < q.known ? x[u] * a.decay : 0.0f;
        o[u] = i < q.known ? o[u] : q.total + i - q.known;
    }
    for (int r = 0; r < q.rows; ++r) {
        const float* w = a.w + (size_t)(q.first + r) * a.w_stride;
        float y[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) y[u] = w[min(i0 + u * kEvThreads, q.len - 1)];
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] += y[u];
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kEvThreads;
        if (i < q.len) {
            q.acc[i] = x[u];
            if (i >= q.known) q.ord[i] = o[u];
        }
        key[u] = i < q.len ? (o[u] >= q.fresh ? kNewest : rank_of(x[u])) : 0u;
    }
}
// The sequence's state after its sums; every thread has read what it was.
__device__ __forceinline__ void set_state(const EvictArgs& a, const EvictSeq& q, int b) {
    const int left = q.over ? a.budget : q.len;
    a.new_lens[b] = left;
    a.state[2 * b] = left;
    a.state[2 * b + 1] = q.now;
    if (!q.over) a.npairs[b] = 0;
}

// The budget-th largest of a block's ranks: a histogram of 2048 equal steps of the range between the smallest and the
// largest, then of the step that holds it, three at most -- digits of the rank itself meet in a few counters, as sums share
// their exponents, and LDS adds to one address come one after another (4097 keys: 53 us with eight bits a pass).
struct Cut {
    uint32_t top, left, same;       // that rank, how many of that rank stay, how many there are
};
// `each(f)`: f(rank) for every rank of this thread (0: no key); fixed, lo, hi: this thread's count of the newest (this
// wave's, rather) and the smallest and largest of its other ranks.
template <class Each>
__device__ __forceinline__ Cut find_cut(int budget, uint32_t fixed, uint32_t lo, uint32_t hi, uint32_t* red, const Each& each) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t red2[3][kEvWaves];
    __shared__ uint32_t s_bin, s_left, s_same;
    const int t = threadIdx.x, wv = __builtin_amdgcn_readfirstlane(t >> 6);
    lo = min_xor64(lo);
    hi = ~min_xor64(~hi);
    if ((t & 63) == 0) { red2[0][wv] = fixed; red2[1][wv] = lo; red2[2][wv] = hi; }
    __syncthreads();
    fixed = 0; lo = kNewest; hi = 0;
#pragma unroll
    for (int i = 0; i < kEvWaves; ++i) {
        fixed += red2[0][i];
        lo = min(lo, red2[1][i]);
        hi = max(hi, red2[2][i]);
    }
    Cut cut{kNewest, (uint32_t)budget, fixed};
    if (fixed >= (uint32_t)budget) return cut;
    cut.left = (uint32_t)budget - fixed;
    uint32_t span = hi - lo;
    for (;;) {
        const int bits = span ? 32 - __builtin_clz(span) : 0, shift = bits > 11 ? bits - 11 : 0;
        hist[t] = 0;
        hist[t + kEvThreads] = 0;
        __syncthreads();
        each([&](uint32_t key) __attribute__((always_inline)) {
            const uint32_t x = key - lo;
            if (x <= span && key != kNewest && key != 0) atomicAdd(&hist[x >> shift], 1u);
        });
        __syncthreads();
        const uint32_t h1 = hist[kBins - 1 - 2 * t], h0 = hist[kBins - 2 - 2 * t];     // from the top
        uint32_t sum;
        const uint32_t before = scan_block(h1 + h0, red, sum);
        if (before < cut.left && cut.left <= before + h1 + h0) {
            const bool second = cut.left > before + h1;
            s_bin = (uint32_t)(kBins - 1 - 2 * t - (second ? 1 : 0));
            s_left = cut.left - before - (second ? h1 : 0);
            s_same = second ? h0 : h1;
        }
        __syncthreads();
        lo += s_bin << shift;
        cut.left = s_left;
        cut.same = s_same;
        if (shift == 0) break;
        span = (1u << shift) - 1;
    }
    cut.top = lo;
    return cut;
}

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
// Moved positions by one wave: their keys, values and scales.
template <int U>
__device__ __forceinline__ void move_rows(const PagedArgs& kv, int b, const int2 (&p)[U], int n) {
    const int l = threadIdx.x & 63;
    const size_t width = (size_t)kv.nkv * kv.hd * (kv.G ? 1 : 2);           // bytes, whole 128s
    const int ng = kv.G ? kv.nkv * (kv.hd / kv.G) : 0;
    int from[U], to[U];                               // (where there is nothing to move, position 0 is read and not stored)
    bool is[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        from[u] = u < n ? paged_slot(kv, b, p[u].x) : -1;
        to[u] = u < n ? paged_slot(kv, b, p[u].y) : -1;
        is[u] = from[u] >= 0 && to[u] >= 0;
        from[u] = is[u] ? from[u] : 0;
    }
    for (size_t x = 16 * (size_t)l; x < width; x += 1024) {
        u32x4 k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = *(const u32x4*)((const char*)kv.k + (size_t)from[u] * width + x);
            v[u] = *(const u32x4*)((const char*)kv.v + (size_t)from[u] * width + x);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (is[u]) {
                *(u32x4*)((char*)kv.k + (size_t)to[u] * width + x) = k[u];
                *(u32x4*)((char*)kv.v + (size_t)to[u] * width + x) = v[u];
            }
    }
    for (int x = l; x < ng; x += 64) {
        float k[U], v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            k[u] = kv.ks[(size_t)from[u] * ng + x];
            v[u] = kv.vs[(size_t)from[u] * ng + x];
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (is[u]) {
                kv.ks[(size_t)to[u] * ng + x] = k[u];
                kv.vs[(size_t)to[u] * ng + x] = v[u];
            }
    }
}

// A bounded cache's steady state: as many keys go as a step brought, found one after another as the smallest rank left (of
// equal ones the highest place). The keys behind budget that stay are at most as many; one wave pairs them with the
// places that fall free. 4097 keys of which one goes: 18.7 us by the histograms below, 8 here.
constexpr int kFew = 8;
__device__ __forceinline__ void few_go(const EvictArgs& a, const uint32_t (&key)[kTiles], int len, int tiles, float* acc, int32_t* ord, int2* pairs) {
    const int b = blockIdx.x, t = threadIdx.x, l = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    __shared__ uint32_t s_key[2][kEvWaves], s_at[2][kEvWaves];
    __shared__ int s_gone[kFew], s_hole[kFew];
    __shared__ int2 s_pair[kFew];
    const int budget = a.budget, go = len - budget;
    uint32_t gone = 0;                                // bit r: this thread's key of tile r went
    for (int k = 0; k < go; ++k) {
        uint32_t best = 0xFFFFFFFFu, at = 0xFFFFFFFFu;    // at: 2^31 - 1 - place, so that the highest is the least
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
            if (r < tiles) {
                const int i = r * kEvThreads + t;
                const bool take = i < len && !((gone >> r) & 1) && key[r] <= best;
                best = take ? key[r] : best;
                at = take ? 0x7FFFFFFFu - (uint32_t)i : at;
            }
        const uint32_t wbest = min_xor64(best);
        const uint32_t wat = min_xor64(best == wbest ? at : 0xFFFFFFFFu);
        if (l == 0) { s_key[k & 1][wv] = wbest; s_at[k & 1][wv] = wat; }
        __syncthreads();
        uint32_t mk = 0xFFFFFFFFu, ma = 0xFFFFFFFFu;
#pragma unroll
        for (int w = 0; w < kEvWaves; ++w) {
            const uint32_t x = s_key[k & 1][w], y = s_at[k & 1][w];
            ma = x < mk ? y : x == mk ? min(ma, y) : ma;
            mk = min(mk, x);
        }
        const int place = (int)(0x7FFFFFFFu - ma);
        if ((place & (kEvThreads - 1)) == t) gone |= 1u << (place / kEvThreads);
        if (t == 0) s_gone[k] = place;
    }
    __syncthreads();
    int moves = 0;
    if (wv == 0) {
        const int mine = l < go ? s_gone[l] : 0x7FFFFFFF;      // lane l: the l-th that went, and the l-th place behind budget
        int rank = 0;
        bool went = false;
        for (int k = 0; k < go; ++k) {
            rank += s_gone[k] < mine ? 1 : 0;
            went = went || s_gone[k] == budget + l;
        }
        const uint64_t movers = __ballot(l < go && !went);
        if (l < go && mine < budget) s_hole[rank] = mine;
        __builtin_amdgcn_wave_barrier();
        if ((movers >> l) & 1) {
            const int m = __popcll(movers & ((1ull << l) - 1)), from = budget + l, to = s_hole[m];
            s_pair[m] = make_int2(from, to);
            pairs[m] = make_int2(from, to);
            acc[to] = acc[from];
            ord[to] = ord[from];
        }
        moves = __popcll(movers);
        if (l == 0) a.npairs[b] = moves;
    }
    if (a.fused) {
        if (l == 0) s_key[0][wv] = (uint32_t)moves;
        __syncthreads();
        moves = (int)s_key[0][0];
        for (int i = wv; i < moves; i += kEvWaves) {
            const int2 p[1] = {s_pair[i]};
            move_rows<1>(a.kv, b, p, 1);
        }
    }
}

// The sums of up to kTiles x 1024 keys of a sequence by one block, the keys' ranks in registers (thread t: keys t, t + 1024
// ..), read once. Bound by latency: loads, then about ten barriers a pass; with one block a sequence, not by memory.
__global__ __launch_bounds__(kEvThreads) void k_evict(EvictArgs a) {
    const int b = blockIdx.x, t = threadIdx.x, l = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    __shared__ uint64_t s_stay[kTiles * kEvWaves], s_same[kTiles * kEvWaves];
    __shared__ uint32_t red[kEvWaves];
    extern __shared__ uint32_t holes[];               // the places that fall free, in order; above them the keys that move in
    const EvictSeq q = evict_seq(a, b);
    const int len = q.len, budget = a.budget;
    float* acc = q.acc;
    int32_t* ord = q.ord;
    uint32_t key[kTiles];
#pragma unroll
    for (int r0 = 0; r0 < kTiles; r0 += 8) {
        uint32_t some[8] = {};
        if (r0 * kEvThreads < len) add_up(a, q, r0 * kEvThreads + t, some);
#pragma unroll
        for (int u = 0; u < 8; ++u) key[r0 + u] = some[u];
    }
    __syncthreads();                                  // (the state is read by every thread before it changes)
    if (t == 0) set_state(a, q, b);
    if (!q.over) return;
    const int tiles = (len + kEvThreads - 1) / kEvThreads;
    int2* pairs = q.pairs;
    if (len - budget <= kFew) {
        few_go(a, key, len, tiles, acc, ord, pairs);
        return;
    }
    uint32_t lo = kNewest, hi = 0, fixed = 0;
#pragma unroll
    for (int r = 0; r < kTiles; ++r) {
        if (r < tiles) {
            const uint32_t x = key[r];
            fixed += (uint32_t)__popcll(__ballot(x == kNewest));
            if (x != 0 && x != kNewest) {
                lo = min(lo, x);
                hi = max(hi, x);
            }
        }
    }
    const Cut cut = find_cut(budget, fixed, lo, hi, red, [&](auto f) __attribute__((always_inline)) {
#pragma unroll
        for (int r = 0; r < kTiles; ++r)
            if (r < tiles) f(key[r]);
    });
    const uint32_t top = cut.top, left = cut.left;
    // Which keys stay, a bit each: a tile's ballot is two words of 32 keys, word t then thread t's. Of the keys of rank `top`
    // the lowest places stay, if not all do. (Ballots and counts per tile all the way: 16 us more at 32001 keys.)
#pragma unroll
    for (int r = 0; r < kTiles; ++r)
        if (r < tiles) {
            const uint64_t more = __ballot(key[r] > top), as = __ballot(key[r] == top);
            if (l == 0) {
                s_stay[r * kEvWaves + wv] = more;
                s_same[r * kEvWaves + wv] = as;
            }
        }
    __syncthreads();
    const bool mine = t < tiles * (kEvThreads / 32);
    uint32_t stay = mine ? ((const uint32_t*)s_stay)[t] : 0u, eq = mine ? ((const uint32_t*)s_same)[t] : 0u, sum;
    if (cut.same == left) {
        stay |= eq;
    } else {
        const uint32_t n = (uint32_t)__popc(eq), before = scan_block(n, red, sum);
        for (uint32_t k = before < left ? min(n, left - before) : 0u; k > 0; --k) {
            stay |= eq & (0u - eq);
            eq &= eq - 1u;
        }
    }
    // the places before budget that fall free and the keys behind it that stay, counted (low and high half) and listed in order
    const int in = min(max(budget - 32 * t, 0), 32);              // keys of the word before budget
    const uint32_t head = in == 32 ? ~0u : (1u << in) - 1u;
    uint32_t hole = ~stay & head, mover = stay & ~head;
    const uint32_t before = scan_block((uint32_t)__popc(hole) | ((uint32_t)__popc(mover) << 16), red, sum);
    for (uint32_t m = before & 0xFFFFu; hole; ++m, hole &= hole - 1u) holes[m] = (uint32_t)(32 * t + __builtin_ctz(hole));
    __syncthreads();
    for (uint32_t m = before >> 16; mover; ++m, mover &= mover - 1u) holes[m] |= (uint32_t)(32 * t + __builtin_ctz(mover)) << 16;
    __syncthreads();
    const int moves = (int)(sum & 0xFFFFu);
    if (t == 0) a.npairs[b] = moves;
    for (int m0 = t; m0 < moves; m0 += 8 * kEvThreads) {
        uint32_t p[8];
        float x[8];
        int o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            p[u] = holes[min(m0 + u * kEvThreads, moves - 1)];
            x[u] = acc[p[u] >> 16];
            o[u] = ord[p[u] >> 16];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (m0 + u * kEvThreads < moves) {
                const int from = (int)(p[u] >> 16), to = (int)(p[u] & 0xFFFFu);
                pairs[m0 + u * kEvThreads] = make_int2(from, to);
                acc[to] = x[u];
                ord[to] = o[u];
            }
    }
    if (a.fused) {                                    // a few moves at most: no second launch
        __syncthreads();
        for (int i = wv; i < moves; i += kEvWaves) {
            const int2 p[1] = {pairs[i]};
            move_rows<1>(a.kv, b, p, 1);
        }
    }
}

// The same for longer sequences in two launches, the ranks in memory: sums and ranks by a block for every 8192 keys, then
// the choice by one block a sequence, each wave walking a run of 64-key steps in order, 16 with their loads together.
// 131071 keys of which one goes: 95 us, of which all but 16000 go 112 (sums in the one block, digits of eight bits: 343). Bound
// by the one block's instructions, some 25 a step of 64 keys and walk, and its LDS adds. A limit above the budget has it done
// once in many steps.
__device__ __forceinline__ int sum_blocks(int max_len) { return (max_len + 8 * kEvThreads - 1) / (8 * kEvThreads); }
__device__ __forceinline__ int mask_words(int max_len) { return (max_len + 63) / 64; }
__global__ __launch_bounds__(kEvThreads) void k_evict_sums(EvictArgs a) {
    const int b = blockIdx.y, t = threadIdx.x, i0 = (int)blockIdx.x * 8 * kEvThreads + t;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    __shared__ uint32_t red[3][kEvWaves];
    const EvictSeq q = evict_seq(a, b);
    if (i0 - t >= q.len) return;
    uint32_t* rank = a.rank + (size_t)b * a.max_len;
    uint32_t key[8];
    add_up(a, q, i0, key);
    if (!q.over) return;
    uint32_t lo = kNewest, hi = 0, fixed = 0;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        if (i0 + u * kEvThreads < q.len) rank[i0 + u * kEvThreads] = key[u];
        fixed += (uint32_t)__popcll(__ballot(key[u] == kNewest));
        if (key[u] != 0 && key[u] != kNewest) {
            lo = min(lo, key[u]);
            hi = max(hi, key[u]);
        }
    }
    lo = min_xor64(lo);
    hi = ~min_xor64(~hi);
    if ((t & 63) == 0) { red[0][wv] = fixed; red[1][wv] = lo; red[2][wv] = hi; }
    __syncthreads();
    if (t == 0) {
        fixed = 0; lo = kNewest; hi = 0;
        for (int i = 0; i < kEvWaves; ++i) {
            fixed += red[0][i];
            lo = min(lo, red[1][i]);
            hi = max(hi, red[2][i]);
        }
        uint32_t* part = a.parts + ((size_t)b * sum_blocks(a.max_len) + blockIdx.x) * 3;
        part[0] = fixed; part[1] = lo; part[2] = hi;
    }
}
__global__ __launch_bounds__(kEvThreads) void k_evict_long(EvictArgs a) {
    const int b = blockIdx.x, t = threadIdx.x, l = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    __shared__ uint32_t red[kEvWaves];
    const EvictSeq q = evict_seq(a, b);
    const int len = q.len, budget = a.budget;
    const uint32_t* rank = a.rank + (size_t)b * a.max_len;
    __syncthreads();                                  // (the state is read by every thread before it changes)
    if (t == 0) set_state(a, q, b);
    if (!q.over) return;
    const int steps = (len + 63) / 64, run = (steps + kEvWaves - 1) / kEvWaves;
    const int s0 = wv * run, s1 = min(s0 + run, steps);
    constexpr int kDeep = 16;
    // f(step, rank) for the keys of this wave's run in order; the rank is 0 where there is no key
    auto walk = [&](auto f) __attribute__((always_inline)) {
        for (int st = s0; st < s1; st += kDeep) {
            uint32_t x[kDeep];
#pragma unroll
            for (int u = 0; u < kDeep; ++u) x[u] = rank[min(64 * (st + u) + l, len - 1)];
#pragma unroll
            for (int u = 0; u < kDeep; ++u) f(st + u, st + u < s1 && 64 * (st + u) + l < len ? x[u] : 0u);
        }
    };
    uint32_t lo = kNewest, hi = 0, fixed = 0, sum;
    for (int i = t; i < sum_blocks(len); i += kEvThreads) {
        const uint32_t* part = a.parts + ((size_t)b * sum_blocks(a.max_len) + i) * 3;
        fixed += part[0];
        lo = min(lo, part[1]);
        hi = max(hi, part[2]);
    }
    scan_block(fixed, red, sum);
    const Cut cut = find_cut(budget, wv == 0 ? sum : 0u, lo, hi, red, [&](auto f) __attribute__((always_inline)) {
        walk([&](int, uint32_t x) __attribute__((always_inline)) { f(x); });
    });
    uint64_t *stays = a.stay + (size_t)b * mask_words(a.max_len), *sames = a.same + (size_t)b * mask_words(a.max_len);
    walk([&](int st, uint32_t x) __attribute__((always_inline)) {
        const uint64_t more = __ballot(x > cut.top), as = __ballot(x == cut.top);
        if (l == 0 && st < s1) {
            stays[st] = more;
            sames[st] = as;
        }
    });
    __syncthreads();
    // as in k_evict, 1024 words of 32 keys at a time: sames so far, places that fall free and keys that move
    uint32_t eq0 = 0, h0 = 0, m0 = 0;
    for (int w0 = 0; w0 < 2 * steps; w0 += kEvThreads) {
        const int w = w0 + t;
        uint32_t stay = w < 2 * steps ? ((const uint32_t*)stays)[w] : 0u, eq = w < 2 * steps ? ((const uint32_t*)sames)[w] : 0u;
        if (cut.same == cut.left) {
            stay |= eq;
        } else {
            const uint32_t n = (uint32_t)__popc(eq), before = eq0 + scan_block(n, red, sum);
            eq0 += sum;
            for (uint32_t k = before < cut.left ? min(n, cut.left - before) : 0u; k > 0; --k) {
                stay |= eq & (0u - eq);
                eq &= eq - 1u;
            }
        }
        const int in = min(max(budget - 32 * w, 0), 32);
        const uint32_t head = in == 32 ? ~0u : (1u << in) - 1u;
        uint32_t hole = ~stay & head, mover = stay & ~head;
        const uint32_t before = scan_block((uint32_t)__popc(hole) | ((uint32_t)__popc(mover) << 16), red, sum);
        for (uint32_t h = h0 + (before & 0xFFFFu); hole; ++h, hole &= hole - 1u) q.pairs[h].y = 32 * w + __builtin_ctz(hole);
        for (uint32_t m = m0 + (before >> 16); mover; ++m, mover &= mover - 1u) q.pairs[m].x = 32 * w + __builtin_ctz(mover);
        h0 += sum & 0xFFFFu;
        m0 += sum >> 16;
    }
    __syncthreads();
    if (t == 0) a.npairs[b] = (int)h0;
    for (uint32_t i0 = (uint32_t)t; i0 < h0; i0 += 8 * kEvThreads) {
        int2 p[8];
        float x[8];
        int o[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            p[u] = q.pairs[min(i0 + u * kEvThreads, h0 - 1u)];
            x[u] = q.acc[p[u].x];
            o[u] = q.ord[p[u].x];
        }
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (i0 + u * kEvThreads < h0) {
                q.acc[p[u].y] = x[u];
                q.ord[p[u].y] = o[u];
            }
    }
}

// The moved positions of a sequence, kMoves a wave. Bound by memory.
constexpr int kMoves = 4;
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a) {
    const int b = blockIdx.y;
    const int i = (blockIdx.x * 4 + (threadIdx.x >> 6)) * kMoves, n = a.npairs[b] - i;
    if (n <= 0) return;
    const int2* pairs = a.pairs + (size_t)b * (a.max_len / 2 + 1) + i;
    int2 p[kMoves];
#pragma unroll
    for (int u = 0; u < kMoves; ++u) p[u] = pairs[u < n ? u : 0];
    move_rows<kMoves>(a.kv, b, p, n);
}

struct EvictWork { size_t pairs, stay, same, parts, rank, npairs, total; };      // bytes; those of longer sequences, if any may be
static EvictWork evict_work(int n_seq, int max_len) {
    const size_t n = (size_t)n_seq, more = max_len > kTiles * kEvThreads ? n : 0;
    EvictWork w{};
    w.pairs = 0;
    w.stay = w.pairs + n * ((size_t)max_len / 2 + 1) * sizeof(int2);
    w.same = w.stay + more * (((size_t)max_len + 63) / 64) * 8;
    w.parts = w.same + more * (((size_t)max_len + 63) / 64) * 8;
    w.rank = w.parts + more * (((size_t)max_len + 8 * kEvThreads - 1) / (8 * kEvThreads)) * 12;
    w.npairs = w.rank + more * max_len * 4;
    w.total = w.npairs + n * 4;
    return w;
}

}  // namespace q27x

using namespace q27x;
extern "C" size_t q27x_paged_evict_work_bytes(int n_seq, int max_len) {
    return n_seq >= 1 && n_seq <= 65535 && max_len >= 1 && max_len <= kMaxKeys ? evict_work(n_seq, max_len).total : 0;
}
extern "C" int q27x_paged_evict(const q27x_paged_kv_t* kv, const float* w, int w_stride, const int32_t* n_acc, int nrows,
                                float decay, float* acc, int32_t* ord, int acc_stride, int32_t* state, int high, int budget,
                                int recent, int max_len, void* work, int32_t* new_lens, q27x_stream_t s) {
    const char* who = "q27x_paged_evict";
    EvictArgs a{};
    if (int rc = paged_args(kv, who, &a.kv)) return rc;
    if (!acc || !ord || !state || !work || !new_lens) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if ((uintptr_t)work & 15) { set_error("%s: work must be 16-byte aligned", who); return Q27X_E_ARG; }
    if (max_len < 1 || max_len > kMaxKeys || acc_stride < max_len || (w && (w_stride < max_len || nrows < 1))) {
        set_error("%s: bad counts (max_len=%d acc_stride=%d w_stride=%d nrows=%d)", who, max_len, acc_stride, w_stride, nrows);
        return Q27X_E_ARG;
    }
    if (recent < 0 || budget < 1 || budget < recent || high < budget || !(decay >= 0.0f && decay <= 1.0f)) {
        set_error("%s: bad limits (recent=%d <= budget=%d <= high=%d, decay=%g in 0 .. 1)", who, recent, budget, high, (double)decay);
        return Q27X_E_ARG;
    }
    a.w = w; a.w_stride = w_stride; a.n_acc = n_acc; a.nrows = nrows; a.decay = decay;
    a.acc = acc; a.ord = ord; a.stride = acc_stride; a.state = state;
    a.high = high; a.budget = budget; a.recent = recent; a.max_len = max_len; a.new_lens = new_lens;
    const EvictWork ew = evict_work(a.kv.n_seq, max_len);
    a.pairs = (int2*)((char*)work + ew.pairs);
    a.rank = (uint32_t*)((char*)work + ew.rank);
    a.parts = (uint32_t*)((char*)work + ew.parts);
    a.stay = (uint64_t*)((char*)work + ew.stay);
    a.same = (uint64_t*)((char*)work + ew.same);
    a.npairs = (int32_t*)((char*)work + ew.npairs);
    const int most = max_len > high ? min(budget, max_len - budget) : 0;       // moves of a sequence
    if (max_len <= kTiles * kEvThreads) {
        Q27X_HIP(allow_lds<k_evict>(kTiles * kEvThreads * 2));
        a.fused = most <= kEvWaves;
        hipLaunchKernelGGL(k_evict, dim3((unsigned)a.kv.n_seq), dim3(kEvThreads), (size_t)most * 4, (hipStream_t)s, a);
    } else {
        const unsigned per = 8 * kEvThreads;
        hipLaunchKernelGGL(k_evict_sums, dim3(((unsigned)max_len + per - 1) / per, (unsigned)a.kv.n_seq), dim3(kEvThreads), 0, (hipStream_t)s, a);
        Q27X_HIP(hipGetLastError());
        hipLaunchKernelGGL(k_evict_long, dim3((unsigned)a.kv.n_seq), dim3(kEvThreads), 0, (hipStream_t)s, a);
    }
    Q27X_HIP(hipGetLastError());
    if (most > 0 && !a.fused) {
        const unsigned per = 4 * kMoves;
        hipLaunchKernelGGL(k_evict_move, dim3((unsigned)((most + per - 1) / per), (unsigned)a.kv.n_seq), dim3(256), 0, (hipStream_t)s, a);
        Q27X_HIP(hipGetLastError());
    }
    return Q27X_OK;
}

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
};
constexpr int kEvThreads = 1024, kEvWaves = kEvThreads / 64;

// Floats as unsigned numbers of the same order: -0 as 0, what is not a number below all others; the newest above all.
__device__ __forceinline__ uint32_t rank_of(float x) {
    if (x != x) return 0u;
    const uint32_t u = __float_as_uint(x == 0.0f ? 0.0f : x);
    return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// exclusive prefix sums over the block's waves of one count per wave; total in *sum
__device__ __forceinline__ int scan_waves(int mine, int wv, int* red, int& sum) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[wv] = mine;
    __syncthreads();
    int before = 0;
    sum = 0;
    for (int i = 0; i < kEvWaves; ++i) {
        const int x = red[i];
        before += i < wv ? x : 0;
        sum += x;
    }
    return before;
}

__global__ __launch_bounds__(kEvThreads) void k_evict_pick(EvictArgs a) {
    const int b = blockIdx.x, t = threadIdx.x, l = t & 63;
    const int wv = __builtin_amdgcn_readfirstlane(t >> 6);
    __shared__ uint32_t hist[256];
    __shared__ int red[kEvWaves];
    __shared__ uint32_t s_digit;
    __shared__ int s_left;
    int first, n;
    paged_rows(a.kv, b, first, n);
    const long long cap = paged_cap(a.kv);
    int len = min(a.kv.lens[b], a.max_len);
    len = len < cap ? len : (int)cap;
    len = len < 0 ? 0 : len;
    int known = a.state[2 * b], total = a.state[2 * b + 1];
    known = min(known < 0 ? 0 : known, len);
    const int now = total + len - known;
    int rows = a.w ? min(n, a.nrows - first) : 0;
    if (a.n_acc) rows = min(rows, a.n_acc[b]);
    float* acc = a.acc + (size_t)b * a.stride;
    int32_t* ord = a.ord + (size_t)b * a.stride;
    uint32_t* rank = a.rank + (size_t)b * a.max_len;
    const bool over = len > a.high;
    const int fresh = now - a.recent;                 // the first of the newest keys
    for (int i = t; i < len; i += kEvThreads) {
        float x = i < known ? acc[i] * a.decay : 0.0f;
        for (int r = 0; r < rows; ++r) x += a.w[(size_t)(first + r) * a.w_stride + i];
        acc[i] = x;
        int o = total + i - known;
        if (i < known) o = ord[i];
        else ord[i] = o;
        if (over) rank[i] = o >= fresh ? 0xFFFFFFFFu : rank_of(x);
    }
    __syncthreads();                                  // (known and total are read by every thread before they change)
    if (t == 0) {
        const int left = over ? a.budget : len;
        a.new_lens[b] = left;
        a.state[2 * b] = left;
        a.state[2 * b + 1] = now;
        if (!over) a.npairs[b] = 0;
    }
    if (!over) return;
    // the budget-th largest rank, eight bits at a time; left: how many of that rank stay
    uint32_t top = 0;
    int left = a.budget;
    for (int sh = 24; sh >= 0; sh -= 8) {
        if (t < 256) hist[t] = 0;
        __syncthreads();
        for (int i = t; i < len; i += kEvThreads) {
            const uint32_t x = rank[i];
            if (sh == 24 || (x >> (sh + 8)) == (top >> (sh + 8))) atomicAdd(&hist[(x >> sh) & 255u], 1u);
        }
        __syncthreads();
        if (t == 0) {
            int d = 255, k = left;
            while (d > 0 && (int)hist[d] < k) k -= (int)hist[d--];
            s_digit = (uint32_t)d;
            s_left = k;
        }
        __syncthreads();
        top |= s_digit << sh;
        left = s_left;
    }
    // Each wave walks a run of 64-key steps in order: how many of rank `top` come before it tells which of those stay;
    // then the places that fall free before budget and the keys that stay behind it, each counted in order.
    const int steps = (len + 63) / 64, run = (steps + kEvWaves - 1) / kEvWaves;
    const int s0 = wv * run, s1 = min(s0 + run, steps);
    int count = 0, sum = 0;
    for (int s = s0; s < s1; ++s) {
        const int i = 64 * s + l;
        count += __popcll(__ballot(i < len && rank[i] == top));
    }
    const int eq0 = scan_waves(count, wv, red, sum);
    const uint64_t below = (1ull << l) - 1;
    int2* pairs = a.pairs + (size_t)b * (a.max_len / 2 + 1);
    int holes = 0, movers = 0, h0 = 0, m0 = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int eq = eq0, h = h0, m = m0;
        for (int s = s0; s < s1; ++s) {
            const int i = 64 * s + l;
            const uint32_t x = i < len ? rank[i] : 0u;
            const uint64_t same = __ballot(i < len && x == top);
            const bool stays = i < len && (x > top || (x == top && eq + __popcll(same & below) < left));
            eq += __popcll(same);
            const uint64_t hole = __ballot(i < len && !stays && i < a.budget), mover = __ballot(stays && i >= a.budget);
            if (pass) {
                if ((hole >> l) & 1) pairs[h + __popcll(hole & below)].y = i;
                if ((mover >> l) & 1) pairs[m + __popcll(mover & below)].x = i;
            }
            h += __popcll(hole);
            m += __popcll(mover);
        }
        if (!pass) {
            h0 = scan_waves(h, wv, red, holes);
            m0 = scan_waves(m, wv, red, movers);
        }
    }
    __syncthreads();
    if (t == 0) a.npairs[b] = holes;
    for (int i = t; i < holes; i += kEvThreads) {
        const int2 p = pairs[i];
        acc[p.y] = acc[p.x];
        ord[p.y] = ord[p.x];
    }
}

// One wave a moved position: its key, its value and their scales.
__global__ __launch_bounds__(256) void k_evict_move(EvictArgs a) {
    const int b = blockIdx.y, l = threadIdx.x & 63;
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= a.npairs[b]) return;
    const int2 p = a.pairs[(size_t)b * (a.max_len / 2 + 1) + i];
    const int from = paged_slot(a.kv, b, p.x), to = paged_slot(a.kv, b, p.y);
    if (from < 0 || to < 0) return;
    const size_t width = (size_t)a.kv.nkv * a.kv.hd * (a.kv.G ? 1 : 2);     // bytes, whole 128s
    for (size_t x = 16 * (size_t)l; x < width; x += 1024) {
        const uint4 k = *(const uint4*)((const char*)a.kv.k + (size_t)from * width + x);
        const uint4 v = *(const uint4*)((const char*)a.kv.v + (size_t)from * width + x);
        *(uint4*)((char*)a.kv.k + (size_t)to * width + x) = k;
        *(uint4*)((char*)a.kv.v + (size_t)to * width + x) = v;
    }
    if (a.kv.G) {
        const int ng = a.kv.nkv * (a.kv.hd / a.kv.G);
        for (int x = l; x < ng; x += 64) {
            const float k = a.kv.ks[(size_t)from * ng + x], v = a.kv.vs[(size_t)from * ng + x];
            a.kv.ks[(size_t)to * ng + x] = k;
            a.kv.vs[(size_t)to * ng + x] = v;
        }
    }
}

struct EvictWork { size_t rank, pairs, npairs, total; };      // bytes
static EvictWork evict_work(int n_seq, int max_len) {
    EvictWork w{};
    w.pairs = 0;
    w.rank = w.pairs + (size_t)n_seq * ((size_t)max_len / 2 + 1) * sizeof(int2);
    w.npairs = w.rank + (size_t)n_seq * max_len * 4;
    w.total = w.npairs + (size_t)n_seq * 4;
    return w;
}

}  // namespace q27x

using namespace q27x;
extern "C" size_t q27x_paged_evict_work_bytes(int n_seq, int max_len) {
    return n_seq >= 1 && n_seq <= 65535 && max_len >= 1 ? evict_work(n_seq, max_len).total : 0;
}
extern "C" int q27x_paged_evict(const q27x_paged_kv_t* kv, const float* w, int w_stride, const int32_t* n_acc, int nrows,
                                float decay, float* acc, int32_t* ord, int acc_stride, int32_t* state, int high, int budget,
                                int recent, int max_len, void* work, int32_t* new_lens, q27x_stream_t s) {
    const char* who = "q27x_paged_evict";
    EvictArgs a{};
    if (int rc = paged_args(kv, who, &a.kv)) return rc;
    if (!acc || !ord || !state || !work || !new_lens) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if ((uintptr_t)work & 15) { set_error("%s: work must be 16-byte aligned", who); return Q27X_E_ARG; }
    if (max_len < 1 || max_len > 0x7fffffff - 64 || acc_stride < max_len || (w && (w_stride < max_len || nrows < 1))) {
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
    a.npairs = (int32_t*)((char*)work + ew.npairs);
    hipLaunchKernelGGL(k_evict_pick, dim3((unsigned)a.kv.n_seq), dim3(kEvThreads), 0, (hipStream_t)s, a);
    Q27X_HIP(hipGetLastError());
    if (max_len > high) {
        const int most = min(budget, max_len - budget);
        hipLaunchKernelGGL(k_evict_move, dim3((unsigned)((most + 3) / 4), (unsigned)a.kv.n_seq), dim3(256), 0, (hipStream_t)s, a);
        Q27X_HIP(hipGetLastError());
    }
    return Q27X_OK;
}

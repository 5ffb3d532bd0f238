// k_sample.hip -- a token a row from its logits, by temperature, top-k, top-p and min-p, with given random numbers.
//
// A row's tokens in order: logits falling, of equal ones the lowest index first; those that are not finite are left out. With l0 the
// largest, w = e^((l - l0) / t). Kept: the first k; of these the fewest first ones whose weights reach p of their sum; of these
// those with w >= m. With S the sum of what is kept: the first token whose running sum passes u S.
//
// Every kept set is a beginning of the order, so a cut is a sum of weights, and the cuts and the draw are searches for the place
// where a running count or sum passes a target. Weights are whole numbers, 2^-z rounded to a multiple of 2^-44 (z = (l0 - l) log2(e) /
// t, the power in fp64 to 2^-46): sums are exact, whatever their order, and nothing depends on atomics' order or on the grid. A
// token of z >= 48 weighs 0 and is never drawn.
//
//   k_sample_max: the largest logit of each 4096.
//   k_sample_bins: bins of z (a 16th of a binary order up to 16 of them, a quarter up to 48): a slice's tokens by bin, and each
//     bin's weight; up to 16 slices a row.
//   k_sample_draw: a row's bins summed and searched. Where all that can be drawn is 256 tokens or fewer, each of them counts and
//     sums those before it, and the cuts and the draw are comparisons; else the bin that a search ends in is narrowed to 64 tokens, by a
//     256th of its z and then by (logit, index) in steps of 8 bits, and these are counted like that.
//   k_sample_one: all of that by one block, for rows of up to 4096 logits (7.8 us for 300, 8 to 11 for 4000, by the settings).
//
// Bound by latency: 62080 logits, 1 row, 16.4 to 18.1 us, of which k_sample_max has 2.5, k_sample_bins 6, k_sample_draw 8 (2.9 to read, 2.2
// to sum the bins, 2 to count 117 tokens); their bytes take 0.05. 64 rows of every kind 33 to 39 us: 4.8, 15.1 (the exponentials and the
// atomics 2.6 each; what the rest of these waits for was not measured), and for the slowest row, whose cuts and draw are three searches (k
// = 1000 alone 24.5 us), or one in a bin of thousands of tokens, which are read twice (p = 0.99, nothing before it: 29; by the ranks'
// range from the start, three times: 35).
// All that can be drawn held in LDS and searched there: 32 us against 25 for a row of k = 1000; ranks alone held, 4096 of them, and
// weights computed anew: 26.5. A search down to 128 or 256 tokens in place of 64: 25.9 and 28.3 us. One copy of the bins: atomics of
// a wave wait for one another.
#include "q27x_dev.h"
#include "q27x_int.h"

namespace q27x {

typedef unsigned long long u64;
constexpr int kMaxPart = 4096;                    // logits of a block of k_sample_max
constexpr int kLeastSlice = 4096, kMostSlices = 16, kMostSlice = 32768, kCopies = 4;
constexpr int kBins = 384, kOffs = kBins + 8;     // a slice's list offsets by bin, in u16
constexpr int kDrawThreads = 256, kHeld = 2048;   // (tokens that LDS holds)
constexpr int kFew = 256, kLeft = 64;             // tokens counted among each other at once, and at a search's end
constexpr int kAhead = 64, kBatch = 8;            // tokens of each slice's list read ahead; held tokens compared at a time
constexpr int kAheadOf = kMostSlices * kAhead / kDrawThreads, kOffLoads = (kMostSlices * kOffs / 8 + kDrawThreads - 1) / kDrawThreads;    // of a thread
constexpr u64 kUnit = 1ull << 44;                 // the weight of the largest logit
constexpr int kMaxTokens = 1 << 19;               // (their weights' sum fits 64 bits, 16 slices hold them)

struct SampleArgs {
    const void* logits; int bf16, n, ld, nr, ns, slice, parts;
    const float* temperature; const int32_t* top_k; const float* top_p; const float* min_p; const float* u;
    float* smax;                                  // [nr][parts] their largest logits, -inf without a finite one
    u64* bw;                                      // [nr][ns][kBins] weights
    uint16_t* off;                                // [nr][ns][kOffs] where a bin begins in the slice's list, and its end
    uint16_t* list;                               // [nr][ns][slice] tokens of the slice by bin
    float* ahead;                                 // [nr][ns][kAhead] logits of the first of them
    int32_t* idx; float* prob;
};

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ float logit_at(const SampleArgs& a, int row, int i) {
    const size_t at = (size_t)row * a.ld + i;
    return a.bf16 ? bf2f(((const uint16_t*)a.logits)[at]) : ((const float*)a.logits)[at];
}
// log2(e) / t, or of a greedy row (t not above 0) 0 with greedy set
__device__ __forceinline__ double inv_temp(const SampleArgs& a, int row, bool& greedy) {
    const float t = a.temperature ? a.temperature[row] : 1.0f;
    greedy = !(t > 0.0f);
    return greedy ? 1.0 : 1.4426950408889634074 / (double)t;
}
// the row's largest logit, in every lane of the calling wave
__device__ __forceinline__ float row_max(const SampleArgs& a, int row) {
    float m = -__builtin_huge_valf();
    for (int s = threadIdx.x & 63; s < a.parts; s += 64) m = fmaxf(m, a.smax[(size_t)row * a.parts + s]);
    return max_xor(m, 64);
}
__device__ __forceinline__ double order_of(float l, double l0, double c) { return (l0 - (double)l) * c; }
__device__ __forceinline__ int bin_of(double z) { return z < 16.0 ? (int)(z * 16.0) : 256 + (int)((z - 16.0) * 4.0); }
// 2^-z in units of 2^-44, z in [0, 48): 2^f, f = rint(z) - z in [-1/2, 1/2], by its series in f ln 2 up to the 11th power (the
// next term is below 2^-47)
__device__ __forceinline__ u64 weight(double z) {
    const double k = __builtin_rint(z), x = (k - z) * 0.69314718055994530942;
    double p = 1.0 / 39916800.0;
    p = __builtin_fma(p, x, 1.0 / 3628800.0);
    p = __builtin_fma(p, x, 1.0 / 362880.0);
    p = __builtin_fma(p, x, 1.0 / 40320.0);
    p = __builtin_fma(p, x, 1.0 / 5040.0);
    p = __builtin_fma(p, x, 1.0 / 720.0);
    p = __builtin_fma(p, x, 1.0 / 120.0);
    p = __builtin_fma(p, x, 1.0 / 24.0);
    p = __builtin_fma(p, x, 1.0 / 6.0);
    p = __builtin_fma(p, x, 0.5);
    p = __builtin_fma(p, x, 1.0);
    p = __builtin_fma(p, x, 1.0);
    // (2^8 + w: the sum's last place is 2^-44)
    const double w = __builtin_ldexp(p, -(int)k) + 256.0;
    return (u64)(__double_as_longlong(w) - __double_as_longlong(256.0));
}
// ascending in the row's order: the logit's bits, falling, then the index
__device__ __forceinline__ u64 rank_of(float l, int i) {
    const uint32_t b = __float_as_uint(l + 0.0f);                // (-0 is 0)
    const uint32_t up = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (u64)~up << 32 | (uint32_t)i;
}

__device__ __forceinline__ float logit_of(u64 rank) {
    const uint32_t up = ~(uint32_t)(rank >> 32);
    return __uint_as_float(up & 0x80000000u ? up & 0x7FFFFFFFu : ~up);
}

// four logits from i on, those behind the row as NaN
__device__ __forceinline__ void logits4(const SampleArgs& a, int row, int i, float (&v)[4]) {
    typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
    typedef uint32_t u32x2h __attribute__((ext_vector_type(2), aligned(2)));
    const size_t at = (size_t)row * a.ld + i;
    if (i + 4 <= a.n) {
        if (a.bf16) {
            const u32x2h x = *(const u32x2h*)((const uint16_t*)a.logits + at);
            v[0] = __uint_as_float(x[0] << 16); v[1] = __uint_as_float(x[0] & 0xFFFF0000u);
            v[2] = __uint_as_float(x[1] << 16); v[3] = __uint_as_float(x[1] & 0xFFFF0000u);
        } else {
            const f32x4u x = *(const f32x4u*)((const float*)a.logits + at);
            v[0] = x[0]; v[1] = x[1]; v[2] = x[2]; v[3] = x[3];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = i + j < a.n ? logit_at(a, row, i + j) : __builtin_nanf("");
    }
}

__global__ __launch_bounds__(256) void k_sample_max(SampleArgs a) {
    const int s = blockIdx.x, row = blockIdx.y;
    float v[kMaxPart / 1024][4], m = -__builtin_huge_valf();
#pragma unroll
    for (int j = 0; j < kMaxPart / 1024; ++j) logits4(a, row, s * kMaxPart + 1024 * j + 4 * (int)threadIdx.x, v[j]);
#pragma unroll
    for (int j = 0; j < kMaxPart / 1024; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) m = is_finite(v[j][k]) ? fmaxf(m, v[j][k]) : m;
    __shared__ float s_m[4];
    m = max_xor(m, 64);
    if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.smax[(size_t)row * a.parts + s] = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
}

// Inclusive running sum over the wave, by DPP: the 16 lanes of a row, then the rows' ends.
__device__ __forceinline__ uint32_t scan_wave(uint32_t x) {
#define Q27X_STEP(CTRL, ROWS) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, true)
    Q27X_STEP(0x111, 0xF); Q27X_STEP(0x112, 0xF); Q27X_STEP(0x114, 0xF); Q27X_STEP(0x118, 0xF);
    Q27X_STEP(0x142, 0xA); Q27X_STEP(0x143, 0xC);
#undef Q27X_STEP
    return x;
}
__device__ __forceinline__ u64 scan_wave(u64 x) {
#define Q27X_STEP(CTRL, ROWS) x += (u64)(uint32_t)__builtin_amdgcn_update_dpp(0, (int)(x >> 32), CTRL, ROWS, 0xF, true) << 32 | \
                                   (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xF, true)
    Q27X_STEP(0x111, 0xF); Q27X_STEP(0x112, 0xF); Q27X_STEP(0x114, 0xF); Q27X_STEP(0x118, 0xF);
    Q27X_STEP(0x142, 0xA); Q27X_STEP(0x143, 0xC);
#undef Q27X_STEP
    return x;
}

// The bins of T threads: of each, the waves that have some, and the threads that store their wave's count (a wave without bins has
// none, as blocks of 512 and 1024 have: there is no place for it).
template <int T>
struct BinThreads {
    static constexpr int kEach = (kBins + T - 1) / T, kWaves = (kBins + 64 * kEach - 1) / (64 * kEach);
    static __host__ __device__ constexpr bool has_sum(int t) { return (t & 63) == 63 && t >> 6 < kWaves; }
    static constexpr bool sums_within(int places) {
        for (int t = 0; t < T; ++t)
            if (has_sum(t) && t >> 6 >= places) return false;
        return true;
    }
};
struct BinShared {
    u64 w[kBins * kCopies];
    uint32_t n[kBins * kCopies], part[(kBins + 63) / 64];
};
// A slice of T PER tokens (MANY: some times that) from `begin` on by bin: list, where each bin begins in it (off, and its end behind the
// last), the bins' weights, the first tokens' logits (if `ahead`); how many there are. x: the slice's first logits, 4 (j T + t) .. + 3 of this thread.
// Bins are kept four times, by lane, as a wave's 64 tokens lie in some 70 bins at most: adding to one place waits for one another.
// Counting gives a token its place in its bin at once. From z = 16 on a slice's weights of a bin are below 2^43: the count has room
// above them, one addition for both.
template <int T, int PER, bool MANY>
__device__ __forceinline__ uint32_t bins_of(const SampleArgs& a, BinShared& sh, uint16_t* list, int row, int begin, float (&x)[PER / 4][4], double l0,
                                            double c, uint16_t* off, u64* bw, float* ahead) {
    constexpr int kTail = 256 * kCopies;          // places of z >= 16
    const int t = threadIdx.x, copy = t & (kCopies - 1);
    uint32_t place[PER];                          // of a token: its bin's copy, and how many came before it there; ~0: left out
    auto take = [&](bool add) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const float l = x[j / 4][j % 4];
            const double z = order_of(l, l0, c);
            place[j] = ~0u;
            if (is_finite(l) && z < 48.0) {
                const int b = bin_of(z) * kCopies + copy;
                uint32_t before;
                if (add && b >= kTail) {
                    before = (uint32_t)(atomicAdd(&sh.w[b], weight(z) | 1ull << 48) >> 48);
                } else {
                    if (add) atomicAdd(&sh.w[b], weight(z));
                    before = atomicAdd(&sh.n[b], 1u);
                }
                place[j] = (uint32_t)b << 16 | before;
            }
        }
    };
    auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
        for (int j = 0; j < PER / 4; ++j) logits4(a, row, begin + i0 + 4 * (j * T + t), x[j]);
    };
    take(true);
    if constexpr (MANY)
        for (int i0 = PER * T; i0 < a.slice; i0 += PER * T) {
            load(i0);
            take(true);
        }
    __syncthreads();
    // where each bin begins
    constexpr int kEach = BinThreads<T>::kEach, kWaves = BinThreads<T>::kWaves;
    static_assert(BinThreads<T>::sums_within(sizeof(sh.part) / sizeof(sh.part[0])), "a place for each sum that is stored");
    uint32_t n[kEach][kCopies], run = 0;
    if (t * kEach < kBins) {
#pragma unroll
        for (int e = 0; e < kEach; ++e)
#pragma unroll
            for (int k = 0; k < kCopies; ++k) {
                const int at = (t * kEach + e) * kCopies + k;
                n[e][k] = at >= kTail ? (uint32_t)(sh.w[at] >> 48) : sh.n[at];
                run += n[e][k];
            }
    }
    const uint32_t mine = run;
    run = scan_wave(run);
    if (BinThreads<T>::has_sum(t)) sh.part[t >> 6] = run;
    run -= mine;
    __syncthreads();
    uint32_t total = 0;
#pragma unroll
    for (int k = 0; k < kWaves; ++k) {
        run += k < t >> 6 ? sh.part[k] : 0;
        total += sh.part[k];
    }
    if (t * kEach < kBins) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int bin = t * kEach + e;
            off[bin] = (uint16_t)run;
            u64 w = 0;
#pragma unroll
            for (int k = 0; k < kCopies; ++k) {
                const u64 wk = sh.w[bin * kCopies + k];
                w += bin * kCopies >= kTail ? wk & ((1ull << 48) - 1) : wk;
                sh.n[bin * kCopies + k] = run;
                run += n[e][k];
            }
            bw[bin] = w;
            if (bin == kBins - 1) off[kBins] = (uint16_t)run;
        }
    }
    __syncthreads();
    if constexpr (!MANY) {
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (place[j] != ~0u) {
                const uint32_t at = sh.n[place[j] >> 16] + (place[j] & 0xFFFFu);
                list[at] = (uint16_t)(4 * (j / 4 * T + t) + j % 4);
                if (ahead && at < kAhead) ahead[at] = x[j / 4][j % 4];
            }
    } else {
        for (int i0 = 0; i0 < a.slice; i0 += PER * T) {
            load(i0);
            take(false);                          // (the bins' beginnings count on)
#pragma unroll
            for (int j = 0; j < PER; ++j)
                if (place[j] != ~0u) {
                    const uint32_t at = place[j] & 0xFFFFu;
                    list[at] = (uint16_t)(i0 + 4 * (j / 4 * T + t) + j % 4);
                    if (ahead && at < kAhead) ahead[at] = x[j / 4][j % 4];
                }
        }
    }
    __syncthreads();
    return total;
}
template <int T, int PER, bool MANY>
__global__ __launch_bounds__(T) void k_sample_bins(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) uint16_t s_list[];
    __shared__ BinShared sh;
    __shared__ float s_ahead[kAhead];
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x, begin = s * a.slice;
    float x[PER / 4][4];
#pragma unroll
    for (int j = 0; j < PER / 4; ++j) logits4(a, row, begin + 4 * (j * T + t), x[j]);       // (requested before the maximum that they wait for)
    for (int b = t; b < kBins * kCopies; b += T) { sh.w[b] = 0; sh.n[b] = 0; }
    bool greedy;
    const double l0 = (double)row_max(a, row), c = inv_temp(a, row, greedy);
    __syncthreads();
    const size_t at = (size_t)row * a.ns + s;
    const uint32_t total = bins_of<T, PER, MANY>(a, sh, s_list, row, begin, x, l0, c, a.off + at * kOffs, a.bw + at * kBins, s_ahead);
    if (t < kAhead) a.ahead[at * kAhead + t] = s_ahead[t];       // (behind the list's end: anything)
    for (uint32_t i = 8 * t; i < total; i += 8 * T) *(uint4*)(a.list + at * a.slice + i) = *(const uint4*)&s_list[i];
}

struct Sum { uint32_t n; u64 w; };
__device__ __forceinline__ u64 shfl_xor64(u64 x, int o) {
    const uint32_t lo = __shfl_xor((uint32_t)x, o, 64), hi = __shfl_xor((uint32_t)(x >> 32), o, 64);
    return (u64)hi << 32 | lo;
}

template <int SLICES>
struct DrawShared {
    u64 bw[kBins + 1];                            // running weights and counts of the row's bins
    uint32_t bn[kBins + 1];
    __attribute__((aligned(16))) uint16_t off[SLICES][kOffs];         // the slices' lists by bin
    Sum part[kBins / 128];
    u64 hw[256];                                  // a narrowing step's digits
    uint32_t hn[256];
    ulonglong2 qw[kHeld + 4 * kBatch];            // candidates: rank, weight
    u64 lo[4], hi[4], found_q, found_w, found_end, digit_w, end_k, end_p, end_m;
    uint32_t held, digit, digit_n, left, heavy;
    int bk, bp;
};

// The row's tokens by bin: in the slices' lists, or (ONE) a single list and its logits in LDS.
template <bool ONE>
struct Lists {
    const SampleArgs& a;
    int row;
    const uint16_t* list;
    const float* x;
    double l0, c;
    __device__ __forceinline__ double z_of(u64 rank) const { return order_of(logit_of(rank), l0, c); }
    // f(rank, weight, z) for each of bins b0 .. b1, the block's threads side by side
    template <typename SH, typename F>
    __device__ __forceinline__ void each(const SH& sh, int b0, int b1, F f) const {
        if constexpr (ONE) {
            for (int i = sh.off[0][b0] + (int)threadIdx.x; i < sh.off[0][b1 + 1]; i += kDrawThreads) {
                const int id = list[i];
                const double z = order_of(x[id], l0, c);
                f(rank_of(x[id], id), weight(z), z);
            }
        } else {
            // a wave's slices, 64 tokens of each requested at once (what lies behind a list's end is left out)
            constexpr int kOf = kMostSlices * 64 / kDrawThreads;
            const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
            for (int i0 = 0;; i0 += 64) {
                int id[kOf];
                float l[kOf];
                bool is[kOf], any = false;
#pragma unroll
                for (int j = 0; j < kOf; ++j) {
                    const int s = min(wave + j * (kDrawThreads / 64), a.ns - 1), i = sh.off[s][b0] + i0 + lane;
                    is[j] = wave + j * (kDrawThreads / 64) < a.ns && i < sh.off[s][b1 + 1];
                    any |= is[j];
                    id[j] = s * a.slice + a.list[((size_t)row * a.ns + s) * a.slice + min(i, a.slice - 1)];
                }
                if (!__ballot(any)) break;
#pragma unroll
                for (int j = 0; j < kOf; ++j) l[j] = logit_at(a, row, is[j] ? id[j] : 0);          // (idle lanes at one place)
#pragma unroll
                for (int j = 0; j < kOf; ++j)
                    if (is[j]) {
                        const double z = order_of(l[j], l0, c);
                        f(rank_of(l[j], id[j]), weight(z), z);
                    }
            }
        }
    }
};
// Four, two or one threads a token: the held token that this thread is one of, and what comes before it among the n held ones
// (a call's threads past the last one's batches have put ranks behind all others there).
struct Counted { bool is; u64 q, w; Sum before; };
template <typename SH>
__device__ __forceinline__ Counted count_held(const SH& sh, uint32_t n) {
    const uint32_t t = threadIdx.x, parts = n <= 64 ? 4 : n <= 128 ? 2 : 1, i = t / parts;
    Counted x;
    x.is = i < n && t % parts == 0;
    const ulonglong2 mine = sh.qw[i < n ? i : 0];
    x.q = mine.x;
    x.w = mine.y;
    x.before = {0, 0};
    for (uint32_t j0 = t % parts; j0 < n; j0 += parts * kBatch) {
        ulonglong2 y[kBatch];
#pragma unroll
        for (int k = 0; k < kBatch; ++k) y[k] = sh.qw[j0 + parts * k];       // (behind the n: ranks that come after all)
#pragma unroll
        for (int k = 0; k < kBatch; ++k) {
            const bool first = y[k].x < x.q;
            x.before.n += first ? 1u : 0u;
            x.before.w += first ? y[k].y : 0;
        }
    }
    if (parts >= 2) {
        x.before.n += __shfl_xor(x.before.n, 1, 64);
        x.before.w += shfl_xor64(x.before.w, 1);
    }
    if (parts == 4) {
        x.before.n += __shfl_xor(x.before.n, 2, 64);
        x.before.w += shfl_xor64(x.before.w, 2);
    }
    return x;
}

// The token of bin b at which the running count (by_count) or weight, from the bin's beginning on, reaches `target` (at least 1, at
// most the bin's): its rank, its weight and the running weight up to it, in sh. Of many tokens first those of a 256th of the bin's z are
// left, then of these those of a 256th of their ranks' range, until there are few.
template <typename SH, typename LISTS>
__device__ __forceinline__ void search(SH& sh, const LISTS& lists, bool by_count, int b, u64 target) {
    const int t = threadIdx.x;
    uint32_t n = sh.bn[b + 1] - sh.bn[b];
    u64 before = 0;                               // weight before what is left
    bool held = n <= kHeld;
    const bool split = n > kLeft;
    int part = 0;
    auto part_of = [&](double z) __attribute__((always_inline)) {          // (as bin_of: z and the tokens have one order)
        const double y = b < 256 ? z * 16.0 - (double)b : (z - 16.0) * 4.0 - (double)(b - 256);
        return min(max((int)(y * 256.0), 0), 255);
    };
    auto clear = [&]() __attribute__((always_inline)) { sh.hw[t] = 0; sh.hn[t] = 0; };
    // the part that `target` is in, by a wave, four parts a lane
    auto choose = [&]() __attribute__((always_inline)) {
        __syncthreads();
        if (t < 64) {
            Sum x = {0, 0};
#pragma unroll
            for (int k = 0; k < 4; ++k) { x.n += sh.hn[4 * t + k]; x.w += sh.hw[4 * t + k]; }
            Sum run = {scan_wave(x.n) - x.n, scan_wave(x.w) - x.w};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const uint32_t pn = sh.hn[4 * t + k];
                const u64 pw = sh.hw[4 * t + k];
                if (by_count ? run.n < target && target <= run.n + pn : run.w < target && target <= run.w + pw) {
                    sh.digit = 4 * t + k;
                    sh.digit_n = run.n;
                    sh.digit_w = run.w;
                    sh.left = pn;
                }
                run.n += pn;
                run.w += pw;
            }
            if (t == 0) sh.held = 0;
        }
        __syncthreads();
        before += sh.digit_w;
        target -= by_count ? sh.digit_n : sh.digit_w;
    };
    auto each = [&](auto f) {                     // of what is left in the part
        if (held) for (uint32_t i = t; i < n; i += kDrawThreads) f(sh.qw[i].x, sh.qw[i].y);
        else lists.each(sh, b, b, [&](u64 q, u64 w, double z) { if (part_of(z) == part) f(q, w); });
    };
    // those that stay to the front, or into LDS once they fit
    auto keep = [&](auto stays) {
        const uint32_t left = sh.left;
        if (held) {
            ulonglong2 x[kHeld / kDrawThreads];
#pragma unroll
            for (int k = 0; k < kHeld / kDrawThreads; ++k) {
                const uint32_t i = t + k * kDrawThreads;
                x[k] = sh.qw[i];
                if (i >= n || !stays(x[k].x)) x[k].x = ~0ull;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kHeld / kDrawThreads; ++k)
                if (x[k].x != ~0ull) sh.qw[atomicAdd(&sh.held, 1u)] = x[k];
        } else if (left <= kHeld) {
            each([&](u64 q, u64 w) { if (stays(q)) sh.qw[atomicAdd(&sh.held, 1u)] = make_ulonglong2(q, w); });
        } else {
            return;
        }
        held = true;
        n = left;
        __syncthreads();
    };
    __syncthreads();
    clear();
    if (t == 0) sh.held = 0;
    __syncthreads();
    if (held || split)
        lists.each(sh, b, b, [&](u64 q, u64 w, double z) {
            if (held) sh.qw[atomicAdd(&sh.held, 1u)] = make_ulonglong2(q, w);
            if (split) {
                const int k = part_of(z);
                atomicAdd(&sh.hw[k], w);
                atomicAdd(&sh.hn[k], 1u);
            }
        });
    if (split) {
        choose();
        part = sh.digit;
        keep([&](u64 q) { return part_of(lists.z_of(q)) == part; });
    } else {
        __syncthreads();
    }
    u64 lo = 0, hi = ~0ull;
    while (n > kLeft) {
        // the range of what is left, in 256 parts
        u64 least = ~0ull, most = 0;
        each([&](u64 q, u64) {
            if (q >= lo && q <= hi) {
                least = q < least ? q : least;
                most = q > most ? q : most;
            }
        });
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const u64 x = shfl_xor64(least, o), y = shfl_xor64(most, o);
            least = x < least ? x : least;
            most = y > most ? y : most;
        }
        __syncthreads();
        if ((t & 63) == 0) { sh.lo[t >> 6] = least; sh.hi[t >> 6] = most; }
        clear();
        __syncthreads();
        lo = min(min(sh.lo[0], sh.lo[1]), min(sh.lo[2], sh.lo[3]));
        hi = max(max(sh.hi[0], sh.hi[1]), max(sh.hi[2], sh.hi[3]));
        const int shift = max(0, 64 - __builtin_clzll((hi - lo) | 1) - 8);
        each([&](u64 q, u64 w) {
            if (q >= lo && q <= hi) {
                atomicAdd(&sh.hw[(q - lo) >> shift], w);
                atomicAdd(&sh.hn[(q - lo) >> shift], 1u);
            }
        });
        choose();
        lo += (u64)sh.digit << shift;
        hi = min(hi, lo + ((1ull << shift) - 1));
        keep([&](u64 q) { return q >= lo && q <= hi; });
    }
    if (t < 4 * kBatch) sh.qw[n + t].x = ~0ull;
    __syncthreads();
    const Counted x = count_held(sh, n);
    if (x.is && (by_count ? x.before.n + 1 == target : x.before.w < target && target <= x.before.w + x.w)) {
        sh.found_q = x.q;
        sh.found_w = x.w;
        sh.found_end = before + x.before.w + x.w;
    }
    __syncthreads();
}

// The bin in which the running weight of the row reaches `target`.
template <typename SH>
__device__ __forceinline__ int bin_that_reaches(const SH& sh, u64 target) {
    int lo = 0, hi = kBins - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        if (sh.bw[mid + 1] >= target) hi = mid; else lo = mid + 1;
    }
    return lo;
}
// the whole number that a running weight has to reach to be at least (PASS: more than) share x kept, of 1 .. kept
template <bool PASS>
__device__ __forceinline__ u64 share_of(float share, u64 kept) {
    const double want = share > 0.0f ? (double)share * (double)kept : 0.0;
    if (!(want < (double)kept)) return kept;
    const u64 x = PASS ? (u64)want + 1 : (u64)__builtin_ceil(want);
    return min(max(x, (u64)1), kept);
}

// A row's settings.
struct Cuts {
    int k;
    float p, m, u;
    double c;
    u64 least;                                    // the weight that min_p asks for: above 1 one that no token has
    int bm0, bm1;                                 // bins around those that tokens of this weight are in (the logarithm is rounded)
    __device__ __forceinline__ Cuts(const SampleArgs& a, int row) {
        bool greedy;
        c = inv_temp(a, row, greedy);
        k = greedy ? 1 : a.top_k ? a.top_k[row] : 0;
        p = a.top_p ? a.top_p[row] : 1.0f;
        m = a.min_p ? a.min_p[row] : 0.0f;
        u = a.u[row];
        least = m <= 1.0f ? (u64)__builtin_ceil((double)m * (double)kUnit) : kUnit + 1;
        const double z = m < 1.0f ? -(double)__builtin_amdgcn_logf(m) : 0.0;
        const int bm = z < 48.0 ? bin_of(z) : kBins - 1;
        bm0 = bm > 0 ? bm - 1 : 0;
        bm1 = bm + 1 < kBins ? bm + 1 : kBins - 1;
    }
};

// The row's token, from its bins: this thread's are 2 t and 2 t + 1, of n0, n1 tokens and weights w0, w1. push(upto): the tokens of
// bins 0 .. upto into sh.qw.
template <typename SH, typename LISTS, typename PUSH>
__device__ __forceinline__ void draw_row(const SampleArgs& a, SH& sh, int row, const LISTS& lists, const Cuts& cuts, uint32_t n0, uint32_t n1, u64 w0, u64 w1,
                                         PUSH push) {
    const int t = threadIdx.x;
    Sum run = {0, 0};
    if (t < kBins / 2) {
        run = {scan_wave(n0 + n1), scan_wave(w0 + w1)};
        if ((t & 63) == 63) sh.part[t >> 6] = run;
    }
    if (t == 0) { sh.held = 0; sh.heavy = 0; sh.bk = sh.bp = kBins - 1; }
    __syncthreads();
    const Sum all = {sh.part[0].n + sh.part[1].n + sh.part[2].n, sh.part[0].w + sh.part[1].w + sh.part[2].w};
    static_assert(kBins / 128 == 3, "three waves of bins");
    u64 kept = all.w;                             // the weight of what is kept
    const int k = cuts.k;
    const bool by_k = k >= 1 && (uint32_t)k < all.n, by_p = cuts.p < 1.0f, by_m = cuts.m > 0.0f;
    if (t < kBins / 2) {
        if (t >= 64) { run.n += sh.part[0].n; run.w += sh.part[0].w; }
        if (t >= 128) { run.n += sh.part[1].n; run.w += sh.part[1].w; }
        const uint32_t na = run.n - n0 - n1, nb = run.n - n1;
        const u64 wa = run.w - w0 - w1, wb = run.w - w1;
        sh.bn[2 * t] = na;
        sh.bn[2 * t + 1] = nb;
        sh.bw[2 * t] = wa;
        sh.bw[2 * t + 1] = wb;
        if (t == kBins / 2 - 1) { sh.bn[kBins] = run.n; sh.bw[kBins] = run.w; }
        // the bins in which the cuts end (by weight, of all)
        if (by_k && na < (uint32_t)k && (uint32_t)k <= run.n) sh.bk = 2 * t + ((uint32_t)k > nb);
        const u64 target = share_of<false>(cuts.p, kept);
        if (by_p && wa < target && target <= run.w) sh.bp = 2 * t + (target > wb);
    }
    __syncthreads();
    const int bk = sh.bk, upto = by_k ? bk : by_p ? sh.bp : by_m ? cuts.bm1 : kBins - 1;
    const uint32_t n = sh.bn[upto + 1];
    if (n <= kFew) {
        push(upto);                               // (all that can be drawn)
        if (t < 4 * kBatch) sh.qw[n + t].x = ~0ull;
        __syncthreads();
        const Counted x = count_held(sh, n);
        const u64 end = x.before.w + x.w;
        if (by_k && x.is && x.before.n + 1 == (uint32_t)k) sh.end_k = end;
        const uint32_t heavy = (uint32_t)__popcll(__ballot(x.is && x.w >= cuts.least));
        if ((t & 63) == 0 && heavy) atomicAdd(&sh.heavy, heavy);
        __syncthreads();
        if (by_k) kept = sh.end_k;
        const u64 want = share_of<false>(cuts.p, kept);
        if (by_p && x.is && x.before.w < want && want <= end) sh.end_p = end;
        if (by_m && x.is && x.before.n + 1 == max(sh.heavy, 1u)) sh.end_m = end;       // (one at least)
        __syncthreads();
        u64 cut = kept;
        if (by_p) cut = min(cut, sh.end_p);
        if (by_m) cut = min(cut, sh.end_m);
        const u64 target = share_of<true>(cuts.u, cut);
        if (x.is && x.before.w < target && target <= end) {
            a.idx[row] = (int32_t)(uint32_t)x.q;
            if (a.prob) a.prob[row] = (float)((double)x.w / (double)cut);
        }
        return;
    }
    u64 cut = 0;
#pragma unroll 1
    for (int stage = 0; stage < 3; ++stage) {     // top-k, top-p, the draw (behind min-p): searches in one bin each
        u64 target;
        int b = bk;
        if (stage == 0) {
            if (!by_k) continue;
            if (sh.bn[bk + 1] == (uint32_t)k) { kept = sh.bw[bk + 1]; continue; }
            target = (u64)k - sh.bn[bk];
        } else {
            if (stage == 1) {
                cut = kept;
                if (!by_p) continue;
            } else if (by_m) {
                u64 sum = 0;
                lists.each(sh, cuts.bm0, cuts.bm1, [&](u64, u64 w, double) { sum += w >= cuts.least ? w : 0; });
                __syncthreads();
                if (t == 0) sh.found_w = 0;
                __syncthreads();
                if (sum) atomicAdd(&sh.found_w, sum);
                __syncthreads();
                cut = min(cut, max(sh.bw[cuts.bm0] + sh.found_w, kUnit));       // (one at least: the largest, of weight 1)
                __syncthreads();
            }
            target = stage == 1 ? share_of<false>(cuts.p, kept) : share_of<true>(cuts.u, cut);
            b = bin_that_reaches(sh, target);
            target -= sh.bw[b];
        }
        search(sh, lists, stage == 0, b, target);
        const u64 end = sh.bw[b] + sh.found_end;
        if (stage == 0) kept = end;
        else if (stage == 1) cut = min(cut, end);
    }
    if (t == 0) {
        a.idx[row] = (int32_t)(uint32_t)sh.found_q;
        if (a.prob) a.prob[row] = (float)((double)sh.found_w / (double)cut);
    }
}

__global__ __launch_bounds__(kDrawThreads) void k_sample_draw(SampleArgs a) {
    const int row = blockIdx.x, t = threadIdx.x;
    __shared__ DrawShared<kMostSlices> sh;
    const size_t first = (size_t)row * a.ns;
    // Requested at once, as each is a trip to memory: the first tokens of each slice's list and their logits, its offsets, bins 2 t and
    // 2 t + 1 of each. (What lies behind a list's end is read too, and not used.)
    int id[kAheadOf];
    float ahead[kAheadOf];
    uint4 off[kOffLoads];
    ulonglong2 bw[kMostSlices];
#pragma unroll
    for (int j = 0; j < kAheadOf; ++j) {
        const int s = min((t >> 6) + 4 * j, a.ns - 1);
        id[j] = s * a.slice + (int)a.list[(first + s) * a.slice + (t & 63)];
        ahead[j] = a.ahead[(first + s) * kAhead + (t & 63)];
    }
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < kOffLoads; ++j) off[j] = ((const uint4*)(a.off + first * kOffs))[min(t + j * kDrawThreads, a.ns * (kOffs / 8) - 1)];
#pragma unroll
    for (int s = 0; s < kMostSlices; ++s)
        bw[s] = *(const ulonglong2*)(a.bw + (first + min(s, a.ns - 1)) * kBins + 2 * min(t, kBins / 2 - 1));
    __builtin_amdgcn_sched_barrier(0);
    const float top = row_max(a, row);
    const Cuts cuts(a, row);
#pragma unroll
    for (int j = 0; j < kOffLoads; ++j)
        if (t + j * kDrawThreads < kMostSlices * (kOffs / 8)) ((uint4*)sh.off)[t + j * kDrawThreads] = off[j];
    u64 w0 = 0, w1 = 0;
#pragma unroll
    for (int s = 0; s < kMostSlices; ++s)
        if (s < a.ns) {
            w0 += bw[s].x;
            w1 += bw[s].y;
        }
    if (!is_finite(top)) {                        // (no finite logit)
        if (t == 0) { a.idx[row] = 0; if (a.prob) a.prob[row] = 0.0f; }
        return;
    }
    __syncthreads();
    uint32_t n0 = 0, n1 = 0;
    if (t < kBins / 2)
        for (int s = 0; s < a.ns; ++s) {
            const uint32_t o0 = sh.off[s][2 * t], o1 = sh.off[s][2 * t + 1], o2 = sh.off[s][2 * t + 2];
            n0 += o1 - o0;
            n1 += o2 - o1;
        }
    const Lists<false> lists = {a, row, nullptr, nullptr, (double)top, cuts.c};
    draw_row(a, sh, row, lists, cuts, n0, n1, w0, w1, [&](int upto) {
        // what was read ahead, and the rest of a longer list
        for (int s = t >> 6, j = 0; s < a.ns; s += 4, ++j) {
            const size_t at = (first + s) * a.slice;
            const int end = sh.off[s][upto + 1];
            for (int i = t & 63; i < end; i += 64) {
                int of = 0;
                float x = 0.0f;
                if (i < kAhead) {
#pragma unroll
                    for (int y = 0; y < kAheadOf; ++y) {
                        of = y == j ? id[y] : of;
                        x = y == j ? ahead[y] : x;
                    }
                } else {
                    of = s * a.slice + a.list[at + i];
                    x = logit_at(a, row, of);
                }
                sh.qw[atomicAdd(&sh.held, 1u)] = make_ulonglong2(rank_of(x, of), weight(order_of(x, lists.l0, lists.c)));
            }
        }
    });
}

// Rows of one slice: all three steps by a block, the bins and the list in LDS.
struct OneShared {
    DrawShared<1> draw;
    BinShared bins;
    u64 bw[kBins];
    __attribute__((aligned(16))) float x[kLeastSlice];
    uint16_t list[kLeastSlice];
    float m[4];
};
__global__ __launch_bounds__(kDrawThreads) void k_sample_one(SampleArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    OneShared& sh = *(OneShared*)lds;
    constexpr int kPer = kLeastSlice / kDrawThreads;
    const int row = blockIdx.x, t = threadIdx.x;
    float x[kPer / 4][4], top = -__builtin_huge_valf();
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) logits4(a, row, 4 * (j * kDrawThreads + t), x[j]);
    const Cuts cuts(a, row);
    for (int b = t; b < kBins * kCopies; b += kDrawThreads) { sh.bins.w[b] = 0; sh.bins.n[b] = 0; }
#pragma unroll
    for (int j = 0; j < kPer / 4; ++j) {
#pragma unroll
        for (int k = 0; k < 4; ++k) top = is_finite(x[j][k]) ? fmaxf(top, x[j][k]) : top;
        *(float4*)&sh.x[4 * (j * kDrawThreads + t)] = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
    }
    top = max_xor(top, 64);
    if ((t & 63) == 0) sh.m[t >> 6] = top;
    __syncthreads();
    top = fmaxf(fmaxf(sh.m[0], sh.m[1]), fmaxf(sh.m[2], sh.m[3]));
    if (!is_finite(top)) {                        // (no finite logit)
        if (t == 0) { a.idx[row] = 0; if (a.prob) a.prob[row] = 0.0f; }
        return;
    }
    bins_of<kDrawThreads, kPer, false>(a, sh.bins, sh.list, row, 0, x, (double)top, cuts.c, sh.draw.off[0], sh.bw, nullptr);
    uint32_t n0 = 0, n1 = 0;
    u64 w0 = 0, w1 = 0;
    if (t < kBins / 2) {
        const uint32_t o0 = sh.draw.off[0][2 * t], o1 = sh.draw.off[0][2 * t + 1], o2 = sh.draw.off[0][2 * t + 2];
        n0 = o1 - o0;
        n1 = o2 - o1;
        w0 = sh.bw[2 * t];
        w1 = sh.bw[2 * t + 1];
    }
    const Lists<true> lists = {a, row, sh.list, sh.x, (double)top, cuts.c};
    draw_row(a, sh.draw, row, lists, cuts, n0, n1, w0, w1, [&](int upto) {
        lists.each(sh.draw, 0, upto, [&](u64 q, u64 w, double) { sh.draw.qw[atomicAdd(&sh.draw.held, 1u)] = make_ulonglong2(q, w); });
    });
}

struct SampleLayout { size_t bw, smax, off, list, ahead, total; int slice, ns, parts; };
static SampleLayout sample_layout(int n, int nr) {
    SampleLayout w{};
    w.slice = kLeastSlice;
    while ((n + w.slice - 1) / w.slice > kMostSlices) w.slice *= 2;
    w.ns = (n + w.slice - 1) / w.slice;
    w.parts = (n + kMaxPart - 1) / kMaxPart;
    const size_t at = (size_t)nr * w.ns;
    w.bw = 0;
    w.list = w.bw + at * kBins * 8;
    w.off = w.list + at * w.slice * 2;
    w.ahead = w.off + at * kOffs * 2;
    w.smax = w.ahead + at * kAhead * 4;
    w.total = w.smax + (size_t)nr * w.parts * 4;
    return w;
}
static bool sample_shape(int n, int nr) { return n >= 1 && n <= kMaxTokens && nr >= 1 && nr <= 65535; }

}  // namespace q27x

// ---------------------------------------------------------------- C ABI (kernel tier)
using namespace q27x;
extern "C" size_t q27x_sample_work_bytes(int n, int nr) { return sample_shape(n, nr) ? sample_layout(n, nr).total : 0; }
extern "C" int q27x_sample_rows(const void* logits, int logits_bf16, int n, int ld, int nr, const float* temperature,
                                const int32_t* top_k, const float* top_p, const float* min_p, const float* u, void* work,
                                int32_t* idx, float* prob, q27x_stream_t s) {
    const char* who = "q27x_sample_rows";
    if (!logits || !u || !work || !idx) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if (!sample_shape(n, nr)) { set_error("%s: unsupported shape (n=%d: 1 to %d; nr=%d: 1 to 65535)", who, n, kMaxTokens, nr); return Q27X_E_SHAPE; }
    if ((uintptr_t)work & 15) { set_error("%s: work must be 16-byte aligned", who); return Q27X_E_ARG; }
    if (nr > 1 && ld < n) { set_error("%s: ld=%d below n=%d", who, ld, n); return Q27X_E_ARG; }
    const SampleLayout wl = sample_layout(n, nr);
    char* p = (char*)work;
    SampleArgs a{};
    a.logits = logits; a.bf16 = logits_bf16 ? 1 : 0; a.n = n; a.ld = nr > 1 ? ld : 0; a.nr = nr;
    a.ns = wl.ns; a.slice = wl.slice; a.parts = wl.parts;
    a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.u = u;
    a.bw = (u64*)(p + wl.bw); a.list = (uint16_t*)(p + wl.list); a.off = (uint16_t*)(p + wl.off);
    a.ahead = (float*)(p + wl.ahead); a.smax = (float*)(p + wl.smax);
    a.idx = idx; a.prob = prob;
    if (a.ns == 1) {
        Q27X_HIP(allow_lds<k_sample_one>((int)sizeof(OneShared)));
        hipLaunchKernelGGL(k_sample_one, dim3((unsigned)nr), dim3(kDrawThreads), sizeof(OneShared), (hipStream_t)s, a);
        Q27X_HIP(hipGetLastError());
        return Q27X_OK;
    }
    const dim3 grid((unsigned)a.ns, (unsigned)nr);
    hipLaunchKernelGGL(k_sample_max, dim3((unsigned)a.parts, (unsigned)nr), dim3(256), 0, (hipStream_t)s, a);
    Q27X_HIP(hipGetLastError());
    if (a.slice == kLeastSlice && (long long)a.ns * nr <= 256) {          // (a compute unit for each block: 1 row 16.2 us, by 512 threads 16.8; 64 rows of every kind 35.2 and 34.3)
        hipLaunchKernelGGL((k_sample_bins<1024, 4, false>), grid, dim3(1024), 2 * a.slice, (hipStream_t)s, a);
    } else if (a.slice == kLeastSlice) {
        hipLaunchKernelGGL((k_sample_bins<512, 8, false>), grid, dim3(512), 2 * a.slice, (hipStream_t)s, a);
    } else if (a.slice == 8192) {
        hipLaunchKernelGGL((k_sample_bins<1024, 8, false>), grid, dim3(1024), 2 * a.slice, (hipStream_t)s, a);
    } else if (a.slice == 16384) {
        Q27X_HIP((allow_lds<k_sample_bins<1024, 16, false>>(2 * kMostSlice)));
        hipLaunchKernelGGL((k_sample_bins<1024, 16, false>), grid, dim3(1024), 2 * a.slice, (hipStream_t)s, a);
    } else {
        Q27X_HIP((allow_lds<k_sample_bins<1024, 16, true>>(2 * kMostSlice)));
        hipLaunchKernelGGL((k_sample_bins<1024, 16, true>), grid, dim3(1024), 2 * a.slice, (hipStream_t)s, a);
    }
    Q27X_HIP(hipGetLastError());
    hipLaunchKernelGGL(k_sample_draw, dim3((unsigned)nr), dim3(kDrawThreads), 0, (hipStream_t)s, a);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}

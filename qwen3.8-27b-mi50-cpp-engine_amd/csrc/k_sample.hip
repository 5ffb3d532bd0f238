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
//   k_sample_max: the largest logit of each slice of 4096.
//   k_sample_bins: bins of z (a 16th of a binary order up to 16 of them, a quarter up to 48): a slice's tokens by bin, and each
//     bin's weight.
//   k_sample_draw: a row's bins summed and searched; the bin that a search ends in is searched by (logit, index) in steps of 10 bits.
#include "q27x_dev.h"
#include "q27x_int.h"

namespace q27x {

typedef unsigned long long u64;
constexpr int kSlice = 4096, kBins = 384, kBinThreads = 512, kPer = kSlice / kBinThreads;
constexpr int kOffs = kBins + 8;                  // a slice's list offsets by bin, in u16
constexpr int kDrawThreads = 1024, kHeld = 2048;  // candidates that LDS holds
constexpr u64 kUnit = 1ull << 44;                 // the weight of the largest logit
constexpr int kMaxTokens = 1 << 19;               // (their weights' sum fits 64 bits)

struct SampleArgs {
    const void* logits; int bf16, n, ld, nr, ns;
    const float* temperature; const int32_t* top_k; const float* top_p; const float* min_p; const float* u;
    float* smax;                                  // [nr][ns] slices' largest logits, -inf without a finite one
    u64* bw;                                      // [nr][ns][kBins] weights
    uint16_t* off;                                // [nr][ns][kOffs] where a bin begins in the slice's list, and its end
    uint16_t* list;                               // [nr][ns][kSlice] tokens of the slice by bin
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
    for (int s = threadIdx.x & 63; s < a.ns; s += 64) m = fmaxf(m, a.smax[(size_t)row * a.ns + s]);
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

__global__ __launch_bounds__(256) void k_sample_max(SampleArgs a) {
    const int s = blockIdx.x, row = blockIdx.y, end = min(a.n, (s + 1) * kSlice);
    float m = -__builtin_huge_valf();
    for (int i = s * kSlice + threadIdx.x; i < end; i += 256) {
        const float l = logit_at(a, row, i);
        m = is_finite(l) ? fmaxf(m, l) : m;
    }
    __shared__ float s_m[4];
    m = max_xor(m, 64);
    if ((threadIdx.x & 63) == 0) s_m[threadIdx.x >> 6] = m;
    __syncthreads();
    if (threadIdx.x == 0) a.smax[(size_t)row * a.ns + s] = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
}

__global__ __launch_bounds__(kBinThreads) void k_sample_bins(SampleArgs a) {
    const int s = blockIdx.x, row = blockIdx.y, t = threadIdx.x, begin = s * kSlice;
    __shared__ u64 s_w[kBins];
    __shared__ uint32_t s_n[kBins], s_at[kBins];
    __shared__ uint32_t s_part[kBinThreads / 64];
    __shared__ __attribute__((aligned(16))) uint16_t s_list[kSlice];
    for (int b = t; b < kBins; b += kBinThreads) { s_w[b] = 0; s_n[b] = 0; }
    const float top = row_max(a, row);
    bool greedy;
    const double c = inv_temp(a, row, greedy), l0 = (double)top;
    __syncthreads();
    int bin[kPer];
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
        const int i = begin + j * kBinThreads + t;
        const float l = i < a.n ? logit_at(a, row, i) : __builtin_huge_valf();
        const double z = order_of(l, l0, c);
        bin[j] = is_finite(l) && z < 48.0 ? bin_of(z) : -1;
        if (bin[j] >= 0) {
            atomicAdd(&s_w[bin[j]], weight(z));
            atomicAdd(&s_n[bin[j]], 1u);
        }
    }
    __syncthreads();
    // where each bin begins
    const size_t at = (size_t)row * a.ns + s;
    uint32_t n = t < kBins ? s_n[t] : 0, run = n;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t y = __shfl_up(run, o, 64);
        run += (t & 63) >= o ? y : 0;
    }
    if ((t & 63) == 63) s_part[t >> 6] = run;
    __syncthreads();
    for (int k = 0; k < t >> 6; ++k) run += s_part[k];
    if (t < kBins) {
        s_at[t] = run - n;
        a.off[at * kOffs + t] = (uint16_t)(run - n);
        a.bw[at * kBins + t] = s_w[t];
        if (t == kBins - 1) a.off[at * kOffs + kBins] = (uint16_t)run;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kPer; ++j)
        if (bin[j] >= 0) s_list[atomicAdd(&s_at[bin[j]], 1u)] = (uint16_t)(j * kBinThreads + t);
    __syncthreads();
    uint32_t total = 0;
    for (int k = 0; k < kBinThreads / 64; ++k) total += s_part[k];
    for (uint32_t i = 2 * t; i < total; i += 2 * kBinThreads) *(uint32_t*)(a.list + at * kSlice + i) = *(const uint32_t*)&s_list[i];
}

// Exclusive running sums over the block's threads of a count and a weight.
struct Sum { uint32_t n; u64 w; };
__device__ __forceinline__ u64 shfl_up64(u64 x, int o) {
    const uint32_t lo = __shfl_up((uint32_t)x, o, 64), hi = __shfl_up((uint32_t)(x >> 32), o, 64);
    return (u64)hi << 32 | lo;
}
__device__ __forceinline__ Sum scan_block(Sum x, Sum* part) {
    const int t = threadIdx.x, l = t & 63;
    Sum run = x;
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t n = __shfl_up(run.n, o, 64);
        const u64 w = shfl_up64(run.w, o);
        if (l >= o) { run.n += n; run.w += w; }
    }
    __syncthreads();                              // (the parts before are read)
    if (l == 63) part[t >> 6] = run;
    __syncthreads();
    for (int k = 0; k < t >> 6; ++k) { run.n += part[k].n; run.w += part[k].w; }
    run.n -= x.n;
    run.w -= x.w;
    return run;
}

struct DrawShared {
    u64 bw[kBins + 1];                            // running weights and counts of the row's bins
    uint32_t bn[kBins + 1];
    Sum part[kDrawThreads / 64];
    u64 hw[1024];                                 // a search step's digits
    uint32_t hn[1024];
    u64 q[kHeld], w[kHeld];                       // candidates
    u64 lo, hi, found_q, found_w, found_before;
    u64 before_w;
    uint32_t held, before_n, digit, left;
};

// The token of bin b at which the running count (BY_COUNT) or weight, from the bin's beginning on, reaches `target` (at least 1, at
// most the bin's): its rank, its weight and the running weight before it, in sh.
template <bool BY_COUNT>
__device__ void search(const SampleArgs& a, DrawShared& sh, int row, int b, u64 target, double l0, double c) {
    const int t = threadIdx.x, wv = t >> 6, l = t & 63;
    const uint32_t count = sh.bn[b + 1] - sh.bn[b];
    const bool held = count <= kHeld;
    // every token of the bin, slices to waves in turn
    auto each_listed = [&](auto f) {
        for (int s = wv; s < a.ns; s += kDrawThreads / 64) {
            const size_t at = (size_t)row * a.ns + s;
            const int end = a.off[at * kOffs + b + 1];
            for (int i = a.off[at * kOffs + b] + l; i < end; i += 64) {
                const int id = s * kSlice + a.list[at * kSlice + i];
                const float x = logit_at(a, row, id);
                f(rank_of(x, id), weight(order_of(x, l0, c)));
            }
        }
    };
    __syncthreads();
    if (t == 0) { sh.held = 0; sh.lo = ~0ull; sh.hi = 0; }
    __syncthreads();
    u64 lo = ~0ull, hi = 0;
    each_listed([&](u64 q, u64 w) {
        lo = q < lo ? q : lo;
        hi = q > hi ? q : hi;
        if (held) {
            const uint32_t k = atomicAdd(&sh.held, 1u);
            sh.q[k] = q;
            sh.w[k] = w;
        }
    });
    atomicMin(&sh.lo, lo);
    atomicMax(&sh.hi, hi);
    __syncthreads();
    lo = sh.lo;
    hi = sh.hi;
    auto each = [&](auto f) {
        if (held) {
            for (uint32_t i = t; i < count; i += kDrawThreads) f(sh.q[i], sh.w[i]);
        } else {
            each_listed(f);
        }
    };
    u64 before = 0;                               // weight before the digits that are left
    int shift = max(0, 64 - __builtin_clzll((hi - lo) | 1) - 10);
    for (;;) {
        sh.hw[t] = 0;
        sh.hn[t] = 0;
        __syncthreads();
        each([&](u64 q, u64 w) {
            if (q >= lo && q <= hi) {
                atomicAdd(&sh.hw[(q - lo) >> shift], w);
                atomicAdd(&sh.hn[(q - lo) >> shift], 1u);
            }
        });
        __syncthreads();
        const Sum mine = {sh.hn[t], sh.hw[t]}, run = scan_block(mine, sh.part);
        const bool here = BY_COUNT ? run.n < target && target <= run.n + mine.n : run.w < target && target <= run.w + mine.w;
        if (here) {
            sh.digit = t;
            sh.before_n = run.n;
            sh.before_w = run.w;
            sh.left = mine.n;
        }
        __syncthreads();
        const u64 first = lo + ((u64)sh.digit << shift);
        before += sh.before_w;
        target -= BY_COUNT ? sh.before_n : sh.before_w;
        const bool last = sh.left == 1 || shift == 0;
        lo = first;
        hi = min(hi, first + ((1ull << shift) - 1));
        if (last) break;
        shift = max(0, shift - 10);
        __syncthreads();                          // (the choice is read)
    }
    each([&](u64 q, u64 w) {
        if (q >= lo && q <= hi) { sh.found_q = q; sh.found_w = w; }
    });
    if (t == 0) sh.found_before = before;
    __syncthreads();
}

// The bin in which the running count or weight of the row reaches `target`.
template <bool BY_COUNT>
__device__ int bin_that_reaches(const DrawShared& sh, u64 target) {
    int lo = 0, hi = kBins - 1;
    while (lo < hi) {
        const int mid = (lo + hi) / 2;
        const u64 upto = BY_COUNT ? (u64)sh.bn[mid + 1] : sh.bw[mid + 1];
        if (upto >= target) hi = mid; else lo = mid + 1;
    }
    return lo;
}

__global__ __launch_bounds__(kDrawThreads) void k_sample_draw(SampleArgs a) {
    const int row = blockIdx.x, t = threadIdx.x;
    __shared__ DrawShared sh;
    const float top = row_max(a, row);
    if (!is_finite(top)) {                        // (no finite logit)
        if (t == 0) { a.idx[row] = 0; if (a.prob) a.prob[row] = 0.0f; }
        return;
    }
    bool greedy;
    const double c = inv_temp(a, row, greedy), l0 = (double)top;
    Sum mine = {0, 0};
    if (t < kBins)
        for (int s = 0; s < a.ns; ++s) {
            const size_t at = (size_t)row * a.ns + s;
            mine.n += (uint32_t)a.off[at * kOffs + t + 1] - a.off[at * kOffs + t];
            mine.w += a.bw[at * kBins + t];
        }
    const Sum run = scan_block(mine, sh.part);
    if (t <= kBins) { sh.bn[t] = run.n; sh.bw[t] = run.w; }
    __syncthreads();
    u64 kept = sh.bw[kBins];                      // the weight of what is kept
    const int k = greedy ? 1 : a.top_k ? a.top_k[row] : 0;
    if (k >= 1 && (uint32_t)k < sh.bn[kBins]) {
        const int b = bin_that_reaches<true>(sh, (u64)k);
        if (sh.bn[b + 1] == (uint32_t)k) {
            kept = sh.bw[b + 1];
        } else {
            search<true>(a, sh, row, b, (u64)k - sh.bn[b], l0, c);
            kept = sh.bw[b] + sh.found_before + sh.found_w;
        }
    }
    const float p = a.top_p ? a.top_p[row] : 1.0f;
    if (p < 1.0f) {
        const double want = p > 0.0f ? (double)p * (double)kept : 0.0;
        const u64 target = max((u64)1, (u64)__builtin_ceil(want));
        const int b = bin_that_reaches<false>(sh, target);
        search<false>(a, sh, row, b, target - sh.bw[b], l0, c);
        kept = min(kept, sh.bw[b] + sh.found_before + sh.found_w);
    }
    const float m = a.min_p ? a.min_p[row] : 0.0f;
    if (m > 0.0f) {
        const u64 least = m < 1.0f ? (u64)__builtin_ceil((double)m * (double)kUnit) : kUnit;
        // the last bin that holds a weight of at least `least`: its tokens' share
        __syncthreads();
        if (t == 0) sh.found_w = 0;
        __syncthreads();
        const double z = m < 1.0f ? -log2((double)m) : 0.0;
        const int bm = z < 48.0 ? bin_of(z) : kBins - 1;
        const int b0 = bm > 0 ? bm - 1 : 0, b1 = bm + 1 < kBins ? bm + 1 : kBins - 1;     // (its logarithm is rounded)
        u64 sum = 0;
        for (int s = t >> 6; s < a.ns; s += kDrawThreads / 64) {
            const size_t at = (size_t)row * a.ns + s;
            const int end = a.off[at * kOffs + b1 + 1];
            for (int i = a.off[at * kOffs + b0] + (t & 63); i < end; i += 64) {
                const u64 w = weight(order_of(logit_at(a, row, s * kSlice + a.list[at * kSlice + i]), l0, c));
                sum += w >= least ? w : 0;
            }
        }
        if (sum) atomicAdd(&sh.found_w, sum);
        __syncthreads();
        kept = min(kept, sh.bw[b0] + sh.found_w);
    }
    const float u = a.u[row];
    double want = u > 0.0f ? (double)u * (double)kept : 0.0;
    if (!(want < (double)kept)) want = (double)kept;
    const u64 target = min((u64)want + 1, kept);  // passes u S: reaches the next whole number
    const int b = bin_that_reaches<false>(sh, target);
    search<false>(a, sh, row, b, target - sh.bw[b], l0, c);
    if (t == 0) {
        a.idx[row] = (int32_t)(uint32_t)sh.found_q;
        if (a.prob) a.prob[row] = (float)((double)sh.found_w / (double)kept);
    }
}

struct SampleLayout { size_t bw, smax, off, list, total; };
static SampleLayout sample_layout(int n, int nr) {
    const size_t at = (size_t)nr * (((size_t)n + kSlice - 1) / kSlice);
    SampleLayout w{};
    w.bw = 0;
    w.list = w.bw + at * kBins * 8;
    w.off = w.list + at * kSlice * 2;
    w.smax = w.off + at * kOffs * 2;
    w.total = w.smax + at * 4;
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
    a.logits = logits; a.bf16 = logits_bf16 ? 1 : 0; a.n = n; a.ld = nr > 1 ? ld : 0; a.nr = nr; a.ns = (n + kSlice - 1) / kSlice;
    a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.u = u;
    a.bw = (u64*)(p + wl.bw); a.list = (uint16_t*)(p + wl.list); a.off = (uint16_t*)(p + wl.off); a.smax = (float*)(p + wl.smax);
    a.idx = idx; a.prob = prob;
    const dim3 grid((unsigned)a.ns, (unsigned)nr);
    hipLaunchKernelGGL(k_sample_max, grid, dim3(256), 0, (hipStream_t)s, a);
    Q27X_HIP(hipGetLastError());
    hipLaunchKernelGGL(k_sample_bins, grid, dim3(kBinThreads), 0, (hipStream_t)s, a);
    Q27X_HIP(hipGetLastError());
    hipLaunchKernelGGL(k_sample_draw, dim3((unsigned)nr), dim3(kDrawThreads), 0, (hipStream_t)s, a);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}

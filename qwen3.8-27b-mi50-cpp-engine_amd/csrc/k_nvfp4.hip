// k_nvfp4.hip -- projections of 1 to 8 rows through NVFP4 weights, and gate | up with SwiGLU and the quantizer behind it.
//
// Weights: E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), the even one of a byte in its low nibble, an E4M3 scale
// per 16. Activations: int8 codes, an fp32 scale per 16. With s over the 16-wide slabs of K:
//   y[n][r] = alpha sum_s dot_s (ws[r][s] xs[n][s]),  dot_s = sum of 16 products code x code, exact (multiples of 1/2 below 2^14).
//
// The codes go into the matrix instructions as they lie in memory: v_mfma_scale_f32_16x16x128_f8f6f4 takes one operand in E2M1
// and the other in E4M3. An int8 code is 16 h + l, l its low nibble (0 .. 15) and h = h' - 8: E4M3 reads a byte 0 .. 15 as that
// many 2^-9 exactly (subnormals, then the first binade), so nibbles are operands without a conversion, the instruction's own
// power of two per operand (E8M0) supplies 2^9 and the 16, and the -8 comes from a constant operand, -8 where the others
// hold codes. A slab has scales of its own on both sides, so slabs may not be summed by the instruction: row 4 n + i of the
// activation operand holds slab i of row n and zeros elsewhere, and the 16 x 16 result has the dots of 4 slabs of 4 rows with
// 16 weight rows. A quarter of the operand's lanes hold something; the matrix cores have the time.
#include "q27x_dev.h"
#include "q27x_int.h"

namespace q27x {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4u __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(1)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2u __attribute__((ext_vector_type(2), aligned(1)));

struct Nvfp4Args {
    const uint8_t* w[2]; const uint8_t* s[2]; float alpha[2];    // the matrix, or gate and up
    int rows, K;
    const int8_t* xq; int xstride; const float* xs; int nr;
    void* y; int ystride, out_bf16; const void* res; int res_bf16, rstride; float rs;
    int8_t* oq; float* os; float g;                              // SwiGLU: codes and scales of v / in_scale, g = 1 / in_scale
};

constexpr int kNvTile = 128;          // weights of a row that a matrix instruction takes
constexpr int kNvWaves = 8;           // waves of a block at most; they share K

// Tile kt's operands of a wave: lane (c, g) = (lane & 15, lane >> 4) has the codes 32 g .. of weight row c, the scales of that
// row, slabs g and 4 + g of activation row c / 4 if c % 4 == g, and the scales of activation row g.
template <int RT, int SETS>
struct Nvfp4Tile {
    u32x4 w[RT];
    u32x2 ws[RT];
    u32x4 x[SETS][2];
    f32x4 xs[SETS][2];
};

template <int RT, int SETS, bool SWIGLU>
struct Nvfp4Wave {
    using Tile = Nvfp4Tile<RT, SETS>;
    const uint8_t* w[RT]; const uint8_t* s[RT];
    const int8_t* x[SETS]; const float* xs[SETS];
    bool has[SETS];                                  // this lane holds activation codes
    int g;
    float acc[RT][SETS];                             // activation row g (of each four), weight row c

    __device__ __forceinline__ void begin(const Nvfp4Args& a, int l) {
        const int c = l & 15;
        g = l >> 4;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            const int r = SWIGLU ? (int)blockIdx.x * 16 + c : ((int)blockIdx.x * RT + t) * 16 + c;
            const size_t row = (size_t)(r < a.rows ? r : a.rows - 1);       // (rows past the last read it again)
            w[t] = a.w[SWIGLU ? t : 0] + row * (size_t)(a.K >> 1);
            s[t] = a.s[SWIGLU ? t : 0] + row * (size_t)(a.K >> 4);
        }
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            const int rx = 4 * u + (c >> 2), ry = 4 * u + g;
            has[u] = (c & 3) == g && rx < a.nr;
            x[u] = a.xq + (size_t)(rx < a.nr ? rx : 0) * a.xstride;
            xs[u] = a.xs + (size_t)(ry < a.nr ? ry : 0) * (a.xstride >> 4);
#pragma unroll
            for (int t = 0; t < RT; ++t) acc[t][u] = 0.0f;
        }
    }
    __device__ __forceinline__ void load(Tile& b, int kt) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            b.w[t] = __builtin_nontemporal_load((const u32x4u*)(w[t] + (size_t)kt * 64 + 16 * g));
            b.ws[t] = *(const u32x2u*)(s[t] + (size_t)kt * 8);
        }
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                b.x[u][h] = u32x4{0, 0, 0, 0};
                if (has[u]) b.x[u][h] = *(const u32x4u*)(x[u] + (size_t)kt * 128 + 64 * h + 16 * g);
                b.xs[u][h] = *(const f32x4u*)(xs[u] + (size_t)kt * 8 + 4 * h);
            }
        }
    }
    // a last tile of n (1 to 7) slabs: zeros behind them
    __device__ __forceinline__ void load_end(Tile& b, int kt, int n) const {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                u32x2 v = {0, 0};
                if (2 * g + h < n) v = *(const u32x2u*)(w[t] + (size_t)kt * 64 + 16 * g + 8 * h);
                b.w[t][2 * h] = v[0];
                b.w[t][2 * h + 1] = v[1];
                uint32_t e = 0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if (4 * h + j < n) e |= (uint32_t)s[t][(size_t)kt * 8 + 4 * h + j] << (8 * j);
                b.ws[t][h] = e;
            }
        }
#pragma unroll
        for (int u = 0; u < SETS; ++u)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                b.x[u][h] = u32x4{0, 0, 0, 0};
                if (has[u] && 4 * h + g < n) b.x[u][h] = *(const u32x4u*)(x[u] + (size_t)kt * 128 + 64 * h + 16 * g);
#pragma unroll
                for (int j = 0; j < 4; ++j) b.xs[u][h][j] = 4 * h + j < n ? xs[u][(size_t)kt * 8 + 4 * h + j] : 0.0f;
            }
    }
    static __device__ __forceinline__ f32x4 dots(const i32x8& x, const u32x4& w, const f32x4& c, int scale) {
        const i32x8 b = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
        return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, b, c, 0, 4, 0, scale, 0, 127);
    }
    // slabs 0 .. 3 (H = 0) or 4 .. 7 of the activation operand: its first or second half
    template <int H>
    static __device__ __forceinline__ i32x8 half(const u32x4& v) {
        if constexpr (H == 0) return i32x8{(int)v[0], (int)v[1], (int)v[2], (int)v[3], 0, 0, 0, 0};
        else return i32x8{0, 0, 0, 0, (int)v[0], (int)v[1], (int)v[2], (int)v[3]};
    }
    template <int H>
    __device__ __forceinline__ void add_half(const Tile& b, const float (&sc)[RT][8]) {
        constexpr int kOne = 127 + 9, k16 = kOne + 4;               // bytes are 2^-9 each
        i32x8 lo[SETS], hi[SETS], minus[SETS];
#pragma unroll
        for (int u = 0; u < SETS; ++u) {
            const uint32_t eight = has[u] ? 0x08080808u : 0u;
            u32x4 l4, h4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                l4[i] = b.x[u][H][i] & 0x0F0F0F0Fu;
                h4[i] = ((b.x[u][H][i] >> 4) & 0x0F0F0F0Fu) ^ eight;
            }
            lo[u] = half<H>(l4);
            hi[u] = half<H>(h4);
            const uint32_t m = has[u] ? 0x88888888u : 0u;
            minus[u] = half<H>(u32x4{m, m, m, m});
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int u = 0; u < SETS; ++u) {
                f32x4 d = dots(minus[u], b.w[t], f32x4{0.0f, 0.0f, 0.0f, 0.0f}, k16);
                d = dots(lo[u], b.w[t], d, kOne);
                d = dots(hi[u], b.w[t], d, k16);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[t][u] = __builtin_fmaf(d[j], sc[t][4 * H + j] * b.xs[u][H][j], acc[t][u]);
            }
    }
    __device__ __forceinline__ void add(const Tile& b) {
        float sc[RT][8];
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const auto p = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.ws[t][h], false), q = __builtin_amdgcn_cvt_pk_f32_fp8((int)b.ws[t][h], true);
                sc[t][4 * h] = p[0]; sc[t][4 * h + 1] = p[1]; sc[t][4 * h + 2] = q[0]; sc[t][4 * h + 3] = q[1];
            }
        add_half<0>(b, sc);
        add_half<1>(b, sc);
    }
};

// Block = 16 RT weight rows (SWIGLU: 16 of gate and the same 16 of up), its waves take K's tiles in turn and are summed in
// wave order.
template <int RT, int SETS, bool SWIGLU>
__global__ __launch_bounds__(64 * kNvWaves) void k_nvfp4(Nvfp4Args a) {
    __shared__ float s_sum[kNvWaves][RT][SETS][64];
    const int t = threadIdx.x, l = t & 63, wv = __builtin_amdgcn_readfirstlane(t >> 6), waves = (int)blockDim.x >> 6;
    Nvfp4Wave<RT, SETS, SWIGLU> v;
    v.begin(a, l);
    const int full = a.K / kNvTile, rest = (a.K % kNvTile) >> 4;
    typename Nvfp4Wave<RT, SETS, SWIGLU>::Tile cur, next;
    if (wv < full) v.load(cur, wv);
    for (int kt = wv; kt < full; kt += waves) {
        if (kt + waves < full) v.load(next, kt + waves);
        v.add(cur);
        cur = next;
    }
    if (rest && wv == full % waves) {
        v.load_end(cur, full, rest);
        v.add(cur);
    }
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int u = 0; u < SETS; ++u) s_sum[wv][i][u][l] = v.acc[i][u];
    __syncthreads();
    constexpr int kOut = SWIGLU ? SETS * 64 : RT * SETS * 64;
    for (int i = t; i < kOut; i += (int)blockDim.x) {
        const int c = i & 15, n = (i >> 4) % (4 * SETS), tile = SWIGLU ? 0 : i / (64 * SETS);
        auto total = [&](int tl) {
            float y = 0.0f;
            for (int k = 0; k < waves; ++k) y = y + s_sum[k][tl][n >> 2][(n & 3) * 16 + c];
            return y;
        };
        if constexpr (SWIGLU) {
            const float gate = a.alpha[0] * total(0), up = a.alpha[1] * total(1);
            const float z = gate / (1.0f + qexp(-gate)) * up * a.g;
            const float sc = max_xor(fabsf(z), 16) * (1.0f / 127.0f);
            const float inv = sc > 0.0f ? 1.0f / sc : 0.0f;
            if (n < a.nr) {
                const size_t at = (size_t)n * a.rows + (size_t)blockIdx.x * 16 + c;
                a.oq[at] = qcode(z, inv);
                if (c == 0) a.os[at >> 4] = sc;
            }
        } else {
            const int r = ((int)blockIdx.x * RT + tile) * 16 + c;
            if (n < a.nr && r < a.rows) {
                float y = a.alpha[0] * total(tile);
                if (a.res) {
                    const size_t at = (size_t)n * a.rstride + r;
                    y = __builtin_fmaf(a.rs, a.res_bf16 ? bf2f(((const uint16_t*)a.res)[at]) : ((const float*)a.res)[at], y);
                }
                const size_t at = (size_t)n * a.ystride + r;
                if (a.out_bf16) ((uint16_t*)a.y)[at] = f2bf(y);
                else ((float*)a.y)[at] = y;
            }
        }
    }
}

template <int RT, bool SWIGLU>
static int launch_nvfp4(const Nvfp4Args& a, hipStream_t s) {
    const int tiles = (a.K + kNvTile - 1) / kNvTile;
    int waves = kNvWaves;
    while (waves > 1 && waves > tiles) waves >>= 1;
    const dim3 grid((unsigned)(SWIGLU ? a.rows / 16 : (a.rows + 16 * RT - 1) / (16 * RT)));
    if (a.nr <= 4) hipLaunchKernelGGL((k_nvfp4<RT, 1, SWIGLU>), grid, dim3(64 * waves), 0, s, a);
    else hipLaunchKernelGGL((k_nvfp4<RT, 2, SWIGLU>), grid, dim3(64 * waves), 0, s, a);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}

// the caller's matrix and rows, checked
static int nvfp4_args(const q27x_nvfp4_t* w, const char* who, const int8_t* xq, int xstride, const float* xs, int nr) {
    if (!w || !w->w || !w->s || !xq || !xs) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if (w->rows < 1 || w->rows > 0x7fffffff - 64 || w->K < 16 || (w->K & 15) || w->K > 0x7fffffff - kNvTile) {
        set_error("%s: unsupported shape (rows=%d K=%d: K a multiple of 16)", who, w->rows, w->K);
        return Q27X_E_SHAPE;
    }
    if (nr < 1 || nr > kMaxRows) { set_error("%s: nr=%d: 1 to %d rows", who, nr, kMaxRows); return Q27X_E_SHAPE; }
    if (nr > 1 && (xstride < w->K || (xstride & 15))) {
        set_error("%s: xstride=%d: at least K=%d, a multiple of 16", who, xstride, w->K);
        return Q27X_E_ARG;
    }
    return Q27X_OK;
}

}  // namespace q27x

// ---------------------------------------------------------------- C ABI (kernel tier)
using namespace q27x;
extern "C" int q27x_proj_nvfp4_rows(const q27x_nvfp4_t* w, const int8_t* xq, int xstride, const float* xs, void* y,
                                    int ystride, int out_bf16, const void* res, int res_bf16, int rstride, float rs,
                                    int nr, q27x_stream_t s) {
    const char* who = "q27x_proj_nvfp4_rows";
    if (int rc = nvfp4_args(w, who, xq, xstride, xs, nr)) return rc;
    if (!y) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if (nr > 1 && (ystride < w->rows || (res && rstride < w->rows))) {
        set_error("%s: bad strides (ystride=%d rstride=%d rows=%d)", who, ystride, rstride, w->rows);
        return Q27X_E_ARG;
    }
    Nvfp4Args a{};
    a.w[0] = w->w; a.s[0] = w->s; a.alpha[0] = w->alpha; a.rows = w->rows; a.K = w->K;
    a.xq = xq; a.xstride = nr > 1 ? xstride : 0; a.xs = xs; a.nr = nr;
    a.y = y; a.ystride = nr > 1 ? ystride : 0; a.out_bf16 = out_bf16 ? 1 : 0;
    a.res = res; a.res_bf16 = res_bf16 ? 1 : 0; a.rstride = nr > 1 ? rstride : 0; a.rs = rs;
    return launch_nvfp4<1, false>(a, (hipStream_t)s);
}
extern "C" int q27x_swiglu_nvfp4_rows(const q27x_nvfp4_t* gate, const q27x_nvfp4_t* up, const int8_t* xq, int xstride,
                                      const float* xs, int8_t* oq, float* os, float in_scale, int nr, q27x_stream_t s) {
    const char* who = "q27x_swiglu_nvfp4_rows";
    if (int rc = nvfp4_args(gate, who, xq, xstride, xs, nr)) return rc;
    if (int rc = nvfp4_args(up, who, xq, xstride, xs, nr)) return rc;
    if (!oq || !os || !(in_scale > 0.0f)) { set_error("%s: null output, or in_scale=%g not above 0", who, in_scale); return Q27X_E_ARG; }
    if (gate->rows != up->rows || gate->K != up->K || (gate->rows & 15)) {
        set_error("%s: gate [%d][%d] and up [%d][%d]: equal, rows a multiple of 16", who, gate->rows, gate->K, up->rows, up->K);
        return Q27X_E_SHAPE;
    }
    Nvfp4Args a{};
    a.w[0] = gate->w; a.s[0] = gate->s; a.alpha[0] = gate->alpha;
    a.w[1] = up->w; a.s[1] = up->s; a.alpha[1] = up->alpha;
    a.rows = gate->rows; a.K = gate->K;
    a.xq = xq; a.xstride = nr > 1 ? xstride : 0; a.xs = xs; a.nr = nr;
    a.oq = oq; a.os = os; a.g = 1.0f / in_scale;
    return launch_nvfp4<2, true>(a, (hipStream_t)s);
}

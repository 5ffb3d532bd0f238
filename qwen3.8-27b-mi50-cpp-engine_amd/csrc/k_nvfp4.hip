// k_nvfp4.hip -- projections of 1 to 8 rows through NVFP4 weights, and gate | up with SwiGLU and the quantizer behind it.
//
// Weights: E2M1 codes (0, .5, 1, 1.5, 2, 3, 4, 6 and their negatives), the even one of a byte in its low nibble, an E4M3 scale
// per 16. Activations: int8 codes, an fp32 scale per 16. With s over the 16-wide slabs of K:
//   y[n][r] = alpha sum_s dot_s (ws[r][s] xs[n][s]),  dot_s = sum of 16 products code x code, exact (multiples of 1/2 below 2^14).
//
// The codes go into the matrix instructions as they lie in memory: v_mfma_scale_f32_16x16x128_f8f6f4 takes one operand in E2M1
// and the other in E4M3. An int8 code is 16 h + l, l its low nibble (0 .. 15) and h = -8 .. 7: E4M3 reads a byte 0 .. 15 as that
// many 2^-9 exactly (subnormals, then the first binade), so nibbles are operands without a conversion, h as sign and size, and the
// instruction's own power of two per operand (E8M0) supplies 2^9 and the 16. A slab has scales of its own on both sides, so
// slabs may not be summed by the instruction: row 8 n + i of the activation operand holds slab i of row n and zeros elsewhere, and the
// 16 x 16 result has the dots of 8 slabs of a pair of rows with 16 weight rows. An eighth of the operand holds something; the
// matrix cores have the time.
//
// Up to 4 rows the bound is memory: 62080 x 5120, 1 row, 179 MB in 30.8 us where no cache holds them (5.8 TB/s), 28.9 over and over (a
// kernel that only reads them so, 26.0). What it takes: whole 128-byte lines of 8 rows a load, exchanged in registers (16 rows by 64
// bytes, which are operands at once, read at 5.0 TB/s and no more); scales of several steps in one load (one a step: +9 us of 39); blocks
// that stay and keep the activations, prepared, in LDS (a block a tile: 49.5 us, a third of it spent on them); the next tile on its way
// while one is worked on.
// Chunks of K shorter than 5 steps: 33 us (3), 39 (2), 58 (1).
//
// From 5 rows on tiles of 32 weight rows, and v_mfma_scale_f32_32x32x64_f8f6f4 with the nibbles in E2M3, whose codes 0 .. 15 are as many
// eighths: row 4 n + i of the operand holds slab i of row n, so one instruction serves 8 rows. It takes 40 cycles, the 16 x 16 x 128
// with E4M3, two rows, 42: 8 rows 36 to 37 us, where those tiles take 45 to 48. Left are the scales' products and sums (2 operations a slab, row
// and weight row) and the masks of the operands: without the sums 33.8 us; without preparing the activations 36.9.
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

constexpr int kNvStep = 256;          // weights of a row that a wave takes at a time: a 128-byte line of codes
constexpr int kNvSteps = 5;           // steps of a wave in registers
constexpr int kNvWaves = 16;          // waves of a block at most
constexpr int kNvLds = 160 * 1024;
constexpr int kNvMaxRows = 0x7fffffff - (1 << 19);      // (a block's next tile, and its rows, keep in 31 bits: 256 x 16 blocks of 4 tiles)
constexpr int kNvMaxK = 57344;        // (45 slots: their sums of gate and up, 8 rows, have room in LDS beside 20 steps of 4 rows: 157 KB)

// LDS of a block: activation nibbles of its rows as operands, [steps][rows][low | high][256], and their scales, [steps][rows]
// [16]; before them what lanes without activation codes read; behind them the waves' scales, the sums, [2][groups]
// [slots][32 PAIRS], and the weights of a last step that K does not fill, for each group codes [16][128] and scales [16][16].
struct Nvfp4Lds {
    static constexpr int kZeros = 1024 * (kMaxRows / 2 - 1) + 512;
    int xs, ws, sums, tail, total;
    __host__ __device__ __forceinline__ Nvfp4Lds(int rows, int steps, int per, int groups, int waves, int slots, int outs, bool ends_inside) {
        xs = kZeros + 512 * rows * steps;
        ws = xs + 64 * rows * steps;
        sums = ws + 256 * (per | 1) * groups * waves;
        tail = sums + 8 * groups * slots * outs;
        total = tail + (ends_inside ? 2304 * groups : 0);
    }
};

// Loads from `bytes` bytes at p, the same in every lane; what lies behind them reads as 0, without a branch.
struct Span {
    __amdgpu_buffer_rsrc_t r;
    __device__ __forceinline__ Span(const void* p, uint32_t bytes) {
        const uint64_t x = (uint64_t)(uintptr_t)p;
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)x), hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(x >> 32));
        r = __builtin_amdgcn_make_buffer_rsrc((void*)(uintptr_t)((uint64_t)hi << 32 | lo), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00027000);
    }
    __device__ __forceinline__ u32x4 ld16(uint32_t at) const { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 0)); }
    __device__ __forceinline__ u32x4 ld16_nt(uint32_t at) const { return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)at, 0, 2)); }
    __device__ __forceinline__ float ldf(uint32_t at) const { return __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, (int)at, 0, 0)); }
};

// Rows first .. first + ROWS - 1 of a matrix, of which those from `end` on are read as 0.
template <int ROWS>
struct Nvfp4Tile {
    Span w, s;
    __device__ __forceinline__ Nvfp4Tile(const uint8_t* w_, const uint8_t* s_, int K, int first, int end)
        : w(w_ + (size_t)first * (size_t)(K >> 1), (uint32_t)max(0, min(ROWS, end - first)) * (uint32_t)(K >> 1)),
          s(s_ + (size_t)first * (size_t)(K >> 4), (uint32_t)max(0, min(ROWS, end - first)) * (uint32_t)(K >> 4)) {}
    // its last step, of `rest` slabs, into LDS by `threads` threads: codes [ROWS][128], scales [ROWS][16], zeros behind K
    static __device__ void bring(const uint8_t* w_, const uint8_t* s_, int K, int first, int end, char* lds, int rest, int t, int threads) {
        for (int i = t; i < ROWS * 16; i += threads) {
            const int k = i & 15, row = first + (i >> 4);
            u32x2 v = {0, 0};
            uint8_t e = 0;
            if (k < rest && row < end) {
                const size_t slab = (size_t)(K >> 4) - rest + k;
                v = *(const u32x2u*)(w_ + (size_t)row * (size_t)(K >> 1) + 8 * slab);
                e = s_[(size_t)row * (size_t)(K >> 4) + slab];
            }
            *(u32x2*)(lds + 8 * i) = v;
            lds[ROWS * 128 + i] = (char)e;
        }
    }
};

// A wave's codes: up to kNvSteps steps of 16 rows, as they come: lane l has the codes 128 (l / 4 % 2) + 32 (l / 16) .. of a
// step of rows r and 8 + r, r = l % 4 + 4 (l / 8 % 2), so a load covers 8 rows of a whole line. Exchanged between lanes 4
// apart, register h has codes 128 h + 32 (l / 16) .. of row row_of(l % 16): an operand. The scales of all steps come together,
// 16 per bytes of a row after another, and go through the wave's own LDS, [16][16 (per | 1)] (an odd number of 16 bytes apart).
__device__ __forceinline__ int nvfp4_row_of(int c) { return 8 * ((c >> 2) & 1) + 4 * ((c >> 3) & 1) + (c & 3); }
struct Nvfp4Weights {
    static constexpr int kScales = (16 * kNvSteps + 63) / 64;
    u32x4 w[kNvSteps][2];
    u32x4 s[kScales];
    uint32_t at[2], sat[kScales], sto[kScales];      // this lane's bytes from the tile's beginning, and in LDS

    __device__ __forceinline__ void begin(int K, int per) {
        const int l = threadIdx.x & 63, r = (l & 3) + 4 * ((l >> 3) & 1), piece = 4 * ((l >> 2) & 1) + (l >> 4);
        at[0] = (uint32_t)r * (uint32_t)(K >> 1) + 16 * piece;
        at[1] = at[0] + 8 * (uint32_t)(K >> 1);
#pragma unroll
        for (int i = 0; i < kScales; ++i) {
            const uint32_t k = (uint32_t)(l + 64 * i), row = k / (uint32_t)per, j = k - row * (uint32_t)per;
            sat[i] = row < 16 ? row * (uint32_t)(K >> 4) + 16 * j : 0x40000000u;
            sto[i] = row < 16 ? (row * (uint32_t)(per | 1) + j) * 16 : ~0u;
        }
    }
    // step st of the tile into place j, if `is` (rows behind the last are 0). Always the same loads: where there is no step they
    // read nothing, so that the waits for others know how many are on their way.
    __device__ __forceinline__ void load(const Nvfp4Tile<16>& from, int j, int st, bool is) {
        const uint32_t wo = is ? (uint32_t)st * 128 : 0x80000000u;
        w[j][0] = from.w.ld16_nt(at[0] + wo);
        w[j][1] = from.w.ld16_nt(at[1] + wo);
    }
    // the scales of steps st .. (those of whole steps: `most` bytes of a row are)
    __device__ __forceinline__ void load_scales(const Nvfp4Tile<16>& from, int st, int per, int full) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < kScales; ++i) {
            const uint32_t k = (uint32_t)(l + 64 * i), j = k % (uint32_t)per;
            s[i] = from.s.ld16(st + (int)j < full ? sat[i] + (uint32_t)st * 16 : 0x80000000u);
        }
    }
    __device__ __forceinline__ void store_scales(char* lds) const {
#pragma unroll
        for (int i = 0; i < kScales; ++i)
            if (sto[i] != ~0u) *(u32x4*)(lds + sto[i]) = s[i];
    }
    __device__ __forceinline__ void take(const char* lds, int j) {
        const int l = threadIdx.x & 63, r = (l & 3) + 4 * ((l >> 3) & 1), piece = 4 * ((l >> 2) & 1) + (l >> 4);
        w[j][0] = *(const u32x4*)(lds + 128 * r + 16 * piece);
        w[j][1] = *(const u32x4*)(lds + 128 * (8 + r) + 16 * piece);
    }
    __device__ __forceinline__ u32x4 operand(int j, int h) const {
        u32x4 v;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int x = (int)w[j][0][i], y = (int)w[j][1][i];
            v[i] = (uint32_t)(h == 0 ? __builtin_amdgcn_update_dpp(x, y, 0x114, 0xF, 0xA, false) : __builtin_amdgcn_update_dpp(y, x, 0x104, 0xF, 0x5, false));
        }
        return v;
    }
};

// A thread's share of some activation rows: up to ITEMS slabs.
template <int ITEMS>
struct Nvfp4Rows {
    u32x4 x[ITEMS];
    float xs[ITEMS];
    // slabs first .. + count - 1 of rows r0 .. + n - 1 (zeros behind K and of rows that are not); items from `item` on
    __device__ __forceinline__ void load(const Nvfp4Args& a, int r0, int n, int first, int count, int item) {
        const Span xq_(a.xq, (uint32_t)(a.nr - 1) * (uint32_t)a.xstride + (uint32_t)a.K);
        const Span xs_(a.xs, (uint32_t)(a.nr - 1) * (uint32_t)(a.xstride >> 2) + (uint32_t)(a.K >> 2));
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t k = (uint32_t)(item + (int)threadIdx.x + i * (int)blockDim.x), r = k / (uint32_t)count, slab = first + (k - r * (uint32_t)count);
            const bool there = (int)r < n && r0 + (int)r < a.nr && (int)slab < (a.K >> 4);
            const uint32_t off = (uint32_t)(r0 + (int)r) * (uint32_t)a.xstride + slab * 16;
            x[i] = xq_.ld16(there ? off : 0x80000000u);
            xs[i] = xs_.ldf(there ? off >> 2 : 0x80000000u);
        }
    }
    // codes 16 h + l: l = 0 .. 15, h = -8 .. 7 as sign and size
    __device__ __forceinline__ void store(char* lds, const Nvfp4Lds& L, int n, int count, int item) const {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t k = (uint32_t)(item + (int)threadIdx.x + i * (int)blockDim.x), r = k / (uint32_t)count, slab = k - r * (uint32_t)count;
            if ((int)r >= n) continue;
            u32x4 lo, hi;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lo[j] = x[i][j] & 0x0F0F0F0Fu;
                const uint32_t h = (x[i][j] >> 4) & 0x0F0F0F0Fu, minus = h & 0x08080808u, one = minus >> 3;
                hi[j] = ((h ^ ((minus << 1) - one)) + one) | (minus << 4);
            }
            const uint32_t at = (slab >> 4) * (uint32_t)n + r;
            char* to = lds + Nvfp4Lds::kZeros + at * 512 + (slab & 15) * 16;
            *(u32x4*)to = lo;
            *(u32x4*)(to + 256) = hi;
            *(float*)(lds + L.xs + at * 64 + 4 * (slab & 15)) = xs[i];
        }
    }
    // the same in E2M3: 6 bits a code, 12 bytes a slab
    __device__ __forceinline__ void store_e2m3(char* codes, char* scales, int n, int count, int item) const {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const uint32_t k = (uint32_t)(item + (int)threadIdx.x + i * (int)blockDim.x), r = k / (uint32_t)count, slab = k - r * (uint32_t)count;
            if ((int)r >= n) continue;
            uint32_t lo[4], hi[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t h = (x[i][j] >> 4) & 0x0F0F0F0Fu, minus = h & 0x08080808u, one = minus >> 3;
                lo[j] = six(x[i][j] & 0x0F0F0F0Fu);
                hi[j] = six(((h ^ ((minus << 1) - one)) + one) | (minus << 2));
            }
            const uint32_t at = (slab >> 2) * (uint32_t)n + r;
            char* to = codes + ((slab >> 2) * (uint32_t)n + at) * 64 + (slab & 3) * 16;
            *(u32x4*)to = u32x4{lo[0] | lo[1] << 24, lo[1] >> 8 | lo[2] << 16, lo[2] >> 16 | lo[3] << 8, 0};
            *(u32x4*)(to + 64 * n) = u32x4{hi[0] | hi[1] << 24, hi[1] >> 8 | hi[2] << 16, hi[2] >> 16 | hi[3] << 8, 0};
            *(float*)(scales + at * 16 + 4 * (slab & 3)) = xs[i];
        }
    }
    static __device__ __forceinline__ uint32_t six(uint32_t v) {           // four bytes below 64 as 24 bits
        const uint32_t u = (v & 0x003F003Fu) | ((v >> 2) & 0x0FC00FC0u);
        return (u & 0xFFFu) | ((u >> 4) & 0xFFF000u);
    }
};

__device__ __forceinline__ f32x4 nvfp4_dots(const i32x8& x, const u32x4& w, const f32x4& c, int scale) {
    const i32x8 b = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, b, c, 0, 4, 0, scale, 0, 127);
}

// What a block's sums [group][slot][row][COLS] come to: `wide` tiles of `each` of ROWS outputs, the first ones `first`, first + stride .. With SWIGLU
// gate and up are groups in turn, or the halves of a group's columns.
template <int PAIRS, bool SWIGLU, int ROWS, int COLS>
__device__ __forceinline__ void nvfp4_finish(const Nvfp4Args& a, const float* sums, int first, int each, int stride, int wide, int slots) {
    const int outs = wide * 2 * PAIRS * ROWS;
    constexpr bool kHalves = SWIGLU && COLS != ROWS;
    for (int i = threadIdx.x; i < (outs + 63) / 64 * 64; i += (int)blockDim.x) {
        const int r = i % ROWS, n = i / ROWS % (2 * PAIRS), k = min(i / (2 * PAIRS * ROWS), wide - 1), row = first + k * stride + r;
        auto total = [&](int gr, int at = 0) {
            float y = 0.0f;
            for (int v = 0; v < slots; ++v) y = y + sums[((gr * slots + v) * 2 * PAIRS + n) * COLS + at + r];
            return y;
        };
        const bool is = i < outs && n < a.nr && r < each && row < a.rows;
        if constexpr (SWIGLU) {
            const float gate = a.alpha[0] * (kHalves ? total(k) : total(2 * k)), up = a.alpha[1] * (kHalves ? total(k, ROWS) : total(2 * k + 1));
            const float z = gate / (1.0f + qexp(-gate)) * up * a.g;
            // (a maximum passes over what is not a number: a group that has such a value has it as its scale, and codes of 0)
            const bool none = (__ballot(z != z) >> (threadIdx.x & 48)) & 0xFFFF;
            const float mx = max_xor(fabsf(z), 16), sc = none ? __builtin_nanf("") : mx * (1.0f / 127.0f);
            const float inv = sc > 0.0f ? 1.0f / sc : 0.0f;
            if (is) {
                const size_t at = (size_t)n * a.rows + row;
                a.oq[at] = qcode(none ? 0.0f : z, inv);
                if ((r & 15) == 0) a.os[at >> 4] = sc;
            }
        } else if (is) {
            float y = a.alpha[0] * total(k);
            if (a.res) {
                const size_t at = (size_t)n * a.rstride + row;
                y = __builtin_fmaf(a.rs, a.res_bf16 ? bf2f(((const uint16_t*)a.res)[at]) : ((const float*)a.res)[at], y);
            }
            const size_t at = (size_t)n * a.ystride + row;
            if (a.out_bf16) ((uint16_t*)a.y)[at] = y == y ? f2bf(y) : (uint16_t)0x7FC0;       // (rounded, one with all its bits set would be a 0)
            else ((float*)a.y)[at] = y;
        }
    }
}

// A block goes through tiles of up to 16 weight rows, `groups` side by side (SWIGLU: 16 of gate beside 16 of up). K is cut into
// `slots` of `per` steps; a group's waves take one each, `turn` steps together, then the next ones. Activation rows go in pairs.
// RESIDENT: all of them are in LDS, once for all tiles; else a pair's turn is brought when it comes. The weights of the next turn or
// tile are requested as this one's are used. An output is the sum of its slots in order, whatever the waves, so its bits do not
// depend on nr.
template <int PAIRS, bool SWIGLU, bool RESIDENT>
__global__ __launch_bounds__((RESIDENT ? 64 : 32) * kNvWaves) void k_nvfp4(Nvfp4Args a, int tile_rows, int groups, int waves, int per, int slots) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int t = threadIdx.x, l = t & 63, c = l & 15, g = l >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), grp = __builtin_amdgcn_readfirstlane((t >> 6) / waves), wv = wave - grp * waves;
    const int full = a.K / kNvStep, rest = (a.K % kNvStep) >> 4, steps = full + (rest != 0);
    const int turn = waves * per, held = RESIDENT ? steps : turn, count = 16 * held;
    const int wide = SWIGLU ? groups >> 1 : groups, each = SWIGLU ? 16 : tile_rows;
    constexpr int kIn = RESIDENT || PAIRS == 1 ? PAIRS : 2, kPasses = (PAIRS + kIn - 1) / kIn;        // pairs of a pass over the weights, and passes
    constexpr int kItems = !RESIDENT ? 5 : PAIRS <= 2 ? 4 : 3;       // (3 rows of 17408 at once: 18.6 us, by 3 items 19.5)
    const int rows_held = RESIDENT ? a.nr : min(a.nr, 2 * kIn);
    const Nvfp4Lds L(rows_held, held, per, groups, waves, slots, 32 * PAIRS, rest != 0);
    const uint8_t* wp = SWIGLU && (grp & 1) ? a.w[1] : a.w[0];
    const uint8_t* sp = SWIGLU && (grp & 1) ? a.s[1] : a.s[0];
    const int mine = SWIGLU ? grp >> 1 : grp;        // this group's tile of `wide`
    char* tail = lds + L.tail + 2304 * grp;
    for (int i = 16 * t; i < Nvfp4Lds::kZeros; i += 16 * (int)blockDim.x) *(u32x4*)(lds + i) = u32x4{0, 0, 0, 0};
    Nvfp4Rows<kItems> x;
    Nvfp4Weights w;
    w.begin(a.K, per);
    char* scales = lds + L.ws + 256 * (per | 1) * wave;
    x.load(a, 0, rows_held, 0, count, 0);
    __builtin_amdgcn_sched_barrier(0);               // (requested first: loads come in order)
    const int stride = (int)gridDim.x * each, turn_rows = stride * wide;
    int row = (int)blockIdx.x * each + mine * stride;        // of the tile
    {
        const Nvfp4Tile<16> from(wp, sp, a.K, row, min(row + each, a.rows));
        w.load_scales(from, wv * per, per, full);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kNvSteps; ++j) w.load(from, j, wv * per + j, j < per && wv * per + j < full);
    }
    __builtin_amdgcn_sched_barrier(0);
    if constexpr (RESIDENT) {
        x.store(lds, L, a.nr, count, 0);
        for (int item = kItems * (int)blockDim.x; item < a.nr * count; item += kItems * (int)blockDim.x) {
            x.load(a, 0, a.nr, 0, count, item);
            x.store(lds, L, a.nr, count, item);
        }
        __syncthreads();
    }
    // the operand's row c holds slab c % 8 of row c / 8 of a pair, in lanes g = c % 4, in its first or second half; the other lanes
    // read zeros (an odd last row's neighbour reads what lies behind it, for outputs that are not)
    int opa[2], per_step[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const bool has = (c & 3) == g && ((c >> 2) & 1) == h;
        opa[h] = has ? Nvfp4Lds::kZeros + 512 * (wv * per * rows_held + (c >> 3)) + (c & 7) * 16 : 0;
        per_step[h] = has ? 512 * rows_held : 0;
    }
    const int xsa = L.xs + 64 * (wv * per * rows_held + (g >> 1)) + 16 * (g & 1);
    int parity = 0;
    for (int first = (int)blockIdx.x * each; first < a.rows; first += turn_rows, parity ^= 1) {
        if (rest) {
            Nvfp4Tile<16>::bring(wp, sp, a.K, row, min(row + each, a.rows), tail, rest, t - 64 * grp * waves, 64 * waves);
            __syncthreads();
        }
        float* sums = (float*)(lds + L.sums) + parity * groups * slots * 32 * PAIRS;       // [group][slot][row][16], of two tiles in turn
        for (int s0 = 0, slot = wv; s0 < steps; s0 += turn, slot += waves) {
            float acc[PAIRS] = {};                   // row 2 p + g / 2, slabs 4 (g % 2) .. of each 128 weights, weight row of lane c
            const bool last = s0 + turn >= steps;    // (of the tile)
            const int to = last ? row + turn_rows : row;
            const Nvfp4Tile<16> next(wp, sp, a.K, to, min(to + each, a.rows));
            const int from = last ? wv * per : s0 + turn + wv * per;   // the steps after these
            const int sa = L.ws + 256 * (per | 1) * wave + 16 * (per | 1) * nvfp4_row_of(c) + 4 * (g & 1);
            w.store_scales(scales);
#pragma unroll
            for (int p = 0; p < kPasses; ++p) {
                int o0 = opa[0], o1 = opa[1], ox = xsa;
                if constexpr (RESIDENT) {
                    o0 += per_step[0] * s0;
                    o1 += per_step[1] * s0;
                    ox += 64 * rows_held * s0;
                }
                asm volatile("" : "+v"(o0), "+v"(o1), "+v"(ox));      // (opaque: operands kept over the loop would spill)
                if constexpr (!RESIDENT) {
                    __syncthreads();                  // (the rows before are read)
                    x.store(lds, L, rows_held, count, 0);
                    for (int item = kItems * (int)blockDim.x; item < rows_held * count; item += kItems * (int)blockDim.x) {
                        x.load(a, 2 * kIn * p, rows_held, 16 * s0, count, item);
                        x.store(lds, L, rows_held, count, item);
                    }
                    __syncthreads();
                    if (p + 1 < kPasses) x.load(a, 2 * kIn * (p + 1), rows_held, 16 * s0, count, 0);
                    else x.load(a, 0, rows_held, last ? 0 : 16 * (s0 + turn), count, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                if (p + 1 == kPasses) {
                    w.load_scales(next, from, per, full);
                    __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int j = 0; j < kNvSteps; ++j) {
                    const int st = s0 + wv * per + j;
                    int sj = sa + 16 * j;
                    if (j < per && st < steps) {
                        if (st == full) {
                            w.take(tail, j);
                            sj = L.tail + 2304 * grp + 2048 + 16 * nvfp4_row_of(c) + 4 * (g & 1);
                        }
                        constexpr int kOne = 127 + 9, k16 = kOne + 4;       // bytes are 2^-9 each
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const u32x4 q = w.operand(j, h);
                            const int e = *(const int*)(lds + sj + 8 * h);
                            const auto e0 = __builtin_amdgcn_cvt_pk_f32_fp8(e, false), e1 = __builtin_amdgcn_cvt_pk_f32_fp8(e, true);
#pragma unroll
                            for (int i = 0; i < kIn; ++i) {
                                if (p * kIn + i >= PAIRS) continue;
                                auto operand = [&](int at) __attribute__((always_inline)) {
                                    const u32x4 y = *(const u32x4*)(lds + o0 + at), z = *(const u32x4*)(lds + o1 + at);
                                    return i32x8{(int)y[0], (int)y[1], (int)y[2], (int)y[3], (int)z[0], (int)z[1], (int)z[2], (int)z[3]};
                                };
                                const i32x8 lo = operand(1024 * i + 128 * h), hi = operand(1024 * i + 256 + 128 * h);
                                const f32x4 xs = *(const f32x4*)(lds + ox + 128 * i + 32 * h);
                                const f32x4 d = nvfp4_dots(hi, q, nvfp4_dots(lo, q, f32x4{0.0f, 0.0f, 0.0f, 0.0f}, kOne), k16);
                                float& y = acc[p * kIn + i];
                                y = __builtin_fmaf(d[0], e0[0] * xs[0], y);
                                y = __builtin_fmaf(d[1], e0[1] * xs[1], y);
                                y = __builtin_fmaf(d[2], e1[0] * xs[2], y);
                                y = __builtin_fmaf(d[3], e1[1] * xs[3], y);
                            }
                        }
                    }
                    o0 += per_step[0];
                    o1 += per_step[1];
                    ox += 64 * rows_held;
                    if (p + 1 == kPasses) w.load(next, j, from + j, j < per && from + j < full);
                }
            }
            if (slot < slots) {
#pragma unroll
                for (int p = 0; p < PAIRS; ++p) {
                    const float y = acc[p] + xor16(acc[p]);
                    if (!(g & 1)) sums[((grp * slots + slot) * 2 * PAIRS + 2 * p + (g >> 1)) * 16 + nvfp4_row_of(c)] = y;
                }
            }
        }
        __syncthreads();
        nvfp4_finish<PAIRS, SWIGLU, 16, 16>(a, sums, first, each, stride, wide, slots);
        row += turn_rows;
    }
}

// ---- Tiles of 32 weight rows (SWIGLU: 16 of gate and 16 of up, side by side: with tiles of both in groups of their own a block has half as
// many, and the last round of 17408 rows is longer, 30.7 us against 29.0). 8 waves, for the registers: 80 hold weights on their way.
// The operands are read 64 weights ahead, in a place for each row whether it is or not, so that their offsets are constants.
constexpr int kNvWideWaves = 8, kWidePairs = 3;
struct Nvfp4WideLds {                 // operands [4 steps][low | high][rows][4 slabs][12, 4 unused]; scales [4 steps][rows][4]; then as Nvfp4Lds
    int xs, ws, sums, tail, total;
    __host__ __device__ __forceinline__ Nvfp4WideLds(int rows, int steps, int per, int groups, int waves, int slots, bool ends_inside) {
        xs = 512 * rows * steps;
        ws = xs + 64 * rows * steps;
        sums = ws + 512 * (per | 1) * groups * waves;
        tail = sums + 8 * groups * slots * 32 * rows;
        total = tail + (ends_inside ? 4608 * groups : 0);
    }
};
// As Nvfp4Weights, of 32 rows: lane l's loads are of rows 8 i + l % 8, codes 32 (2 (l / 8 % 4) + l / 32) ..; exchanged between lanes 16 and 8
// apart, register q has codes 64 q + 32 (l / 32) .. of row l % 32.
template <int MATS>
struct Nvfp4WideWeights {
    static constexpr int kRows = 32 / MATS, kScales = (kRows * kNvSteps + 63) / 64;
    u32x4 w[kNvSteps][4], s[MATS][kScales];
    uint32_t at, rows8, sat[kScales], sto[kScales];

    __device__ __forceinline__ void begin(int K, int per) {
        const int l = threadIdx.x & 63;
        rows8 = 8 * (uint32_t)(K >> 1);
        at = (uint32_t)(l & 7) * (uint32_t)(K >> 1) + 16 * (2 * ((l >> 3) & 3) + (l >> 5));
#pragma unroll
        for (int i = 0; i < kScales; ++i) {
            const uint32_t k = (uint32_t)(l + 64 * i), row = k / (uint32_t)per, j = k - row * (uint32_t)per;
            sat[i] = row < kRows ? row * (uint32_t)(K >> 4) + 16 * j : 0x40000000u;
            sto[i] = row < kRows ? (row * (uint32_t)(per | 1) + j) * 16 : ~0u;
        }
    }
    template <typename TILES>
    __device__ __forceinline__ void load(const TILES& from, int j, int st, bool is) {
        const uint32_t wo = is ? at + (uint32_t)st * 128 : 0x80000000u;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[j][i] = from[i * MATS / 4].w.ld16_nt(wo + (i * 8 % kRows / 8) * rows8);
    }
    template <typename TILES>
    __device__ __forceinline__ void load_scales(const TILES& from, int st, int per, int full) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < kScales; ++i) {
            const uint32_t k = (uint32_t)(l + 64 * i), j = k % (uint32_t)per;
#pragma unroll
            for (int m = 0; m < MATS; ++m) s[m][i] = from[m].s.ld16(st + (int)j < full ? sat[i] + (uint32_t)st * 16 : 0x80000000u);
        }
    }
    __device__ __forceinline__ void store_scales(char* lds, int per) const {
#pragma unroll
        for (int i = 0; i < kScales; ++i)
#pragma unroll
            for (int m = 0; m < MATS; ++m)
                if (sto[i] != ~0u) *(u32x4*)(lds + m * kRows * (per | 1) * 16 + sto[i]) = s[m][i];
    }
    __device__ __forceinline__ void take(const char* lds, int j) {
        const int l = threadIdx.x & 63;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            w[j][i] = *(const u32x4*)(lds + i * MATS / 4 * (kRows * 144) + 128 * (i * 8 % kRows + (l & 7)) + 16 * (2 * ((l >> 3) & 3) + (l >> 5)));
    }
    __device__ __forceinline__ void operands(int j, u32x4 (&q)[4]) const {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const auto x = __builtin_amdgcn_permlane16_swap(w[j][0][d], w[j][2][d], false, false);
            const auto y = __builtin_amdgcn_permlane16_swap(w[j][1][d], w[j][3][d], false, false);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                q[2 * h][d] = (uint32_t)__builtin_amdgcn_update_dpp((int)x[h], (int)y[h], 0x118, 0xF, 0xC, false);
                q[2 * h + 1][d] = (uint32_t)__builtin_amdgcn_update_dpp((int)y[h], (int)x[h], 0x108, 0xF, 0x3, false);
            }
        }
    }
};
typedef float f32x16 __attribute__((ext_vector_type(16)));
template <int PAIRS, bool SWIGLU, bool RESIDENT>
__global__ __launch_bounds__(64 * kNvWideWaves) void k_nvfp4_wide(Nvfp4Args a, int tile_rows, int groups, int waves, int per, int slots) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int kMats = SWIGLU ? 2 : 1, kRows = 32 / kMats, kIn = 2 * PAIRS, kItems = RESIDENT ? 5 : 2;       // (5 spill there: 38.8 us, 34.7)
    using Weights = Nvfp4WideWeights<kMats>;
    using Tile = Nvfp4Tile<kRows>;
    const int t = threadIdx.x, l = t & 63, c = l & 31, g = l >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6), grp = __builtin_amdgcn_readfirstlane((t >> 6) / waves), wv = wave - grp * waves;
    const int full = a.K / kNvStep, rest = (a.K % kNvStep) >> 4, steps = full + (rest != 0);
    const int turn = waves * per, held = RESIDENT ? steps : turn, count = 16 * held;
    const int each = SWIGLU ? kRows : tile_rows;
    const Nvfp4WideLds L(kIn, held, per, groups, waves, slots, rest != 0);
    char* tail = lds + L.tail + 4608 * grp;
    Nvfp4Rows<kItems> x;
    Weights w;
    w.begin(a.K, per);
    char* scales = lds + L.ws + 512 * (per | 1) * wave;
    x.load(a, 0, kIn, 0, count, 0);
    __builtin_amdgcn_sched_barrier(0);
    const int stride = (int)gridDim.x * each, turn_rows = stride * groups;
    int row = (int)blockIdx.x * each + grp * stride;        // of the tile
    {
        const Tile from[2] = {Tile(a.w[0], a.s[0], a.K, row, min(row + each, a.rows)), Tile(a.w[kMats - 1], a.s[kMats - 1], a.K, row, min(row + each, a.rows))};
        w.load_scales(from, wv * per, per, full);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < kNvSteps; ++j) w.load(from, j, wv * per + j, j < per && wv * per + j < full);
    }
    __builtin_amdgcn_sched_barrier(0);
    auto store = [&](int slab) __attribute__((always_inline)) {        // what x has, and the rest of these rows
        x.store_e2m3(lds, lds + L.xs, kIn, count, 0);
        for (int item = kItems * (int)blockDim.x; item < kIn * count; item += kItems * (int)blockDim.x) {
            x.load(a, 0, kIn, slab, count, item);
            x.store_e2m3(lds, lds + L.xs, kIn, count, item);
        }
        __syncthreads();
    };
    if constexpr (RESIDENT) store(0);
    // row c of the operand holds slab c % 4 of row c / 4, in lanes g = c % 4 / 2, in its first or second half; zeros elsewhere
    const bool has = ((c >> 1) & 1) == g && (c >> 2) < kIn;
    const uint32_t even = has && !(c & 1) ? ~0u : 0, odd = has && (c & 1) ? ~0u : 0;
    const int opa = 512 * kIn * wv * per + 16 * (c & (4 * kIn - 1 < 16 ? 4 * kIn - 1 : 31)), xsa = L.xs + 64 * kIn * wv * per + 16 * g;
    int parity = 0;
    for (int first = (int)blockIdx.x * each; first < a.rows; first += turn_rows, parity ^= 1) {
        if (rest) {
#pragma unroll
            for (int m = 0; m < kMats; ++m)
                Tile::bring(a.w[m], a.s[m], a.K, row, min(row + each, a.rows), tail + m * kRows * 144, rest, t - 64 * grp * waves, 64 * waves);
            __syncthreads();
        }
        float* sums = (float*)(lds + L.sums) + parity * groups * slots * 32 * kIn;
        for (int s0 = 0, slot = wv; s0 < steps; s0 += turn, slot += waves) {
            float acc[PAIRS][2] = {};                // row 2 p + g; even and odd 64 weights
            const bool last = s0 + turn >= steps;
            const int from = last ? wv * per : s0 + turn + wv * per, to = last ? row + turn_rows : row;
            const Tile next[2] = {Tile(a.w[0], a.s[0], a.K, to, min(to + each, a.rows)), Tile(a.w[kMats - 1], a.s[kMats - 1], a.K, to, min(to + each, a.rows))};
            w.store_scales(scales, per);
            int o = opa + (RESIDENT ? 512 * kIn * s0 : 0), ox = xsa + (RESIDENT ? 64 * kIn * s0 : 0), sa = L.ws + 512 * (per | 1) * wave + 16 * (per | 1) * c;
            asm volatile("" : "+v"(o), "+v"(ox));
            if constexpr (!RESIDENT) {
                __syncthreads();                      // (the turn before is read)
                store(16 * s0);
                x.load(a, 0, kIn, last ? 0 : 16 * (s0 + turn), count, 0);
                __builtin_amdgcn_sched_barrier(0);
            }
            w.load_scales(next, from, per, full);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < kNvSteps; ++j) {
                const int st = s0 + wv * per + j;
                if (j < per && st < steps) {
                    int sj = sa + 16 * j;
                    if (st == full) {
                        w.take(tail, j);
                        sj = L.tail + 4608 * grp + c / kRows * (kRows * 144) + kRows * 128 + 16 * (c % kRows);
                    }
                    constexpr int kOne = 127 + 3, k16 = kOne + 4;       // codes are eighths
                    u32x4 y[2][2];                   // 64 weights' operands ahead
                    f32x4 xs[2][PAIRS];
                    auto bring = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) y[i & 1][h] = *(const u32x4*)(lds + o + (2 * i + h) * 64 * kIn);
                    };
                    auto bring_scales = [&](int i) __attribute__((always_inline)) {
#pragma unroll
                        for (int p = 0; p < PAIRS; ++p) xs[i & 1][p] = *(const f32x4*)(lds + ox + 16 * kIn * i + 32 * p);
                    };
                    auto operand = [&](const u32x4& v) __attribute__((always_inline)) {
                        return i32x8{(int)(v[0] & even), (int)(v[1] & even), (int)(v[2] & even), (int)(v[0] & odd), (int)(v[1] & odd), (int)(v[2] & odd), 0, 0};
                    };
                    f32x16 d[2];
                    bring(0);
                    const u32x4 e = *(const u32x4*)(lds + sj);
                    bring_scales(0);
                    u32x4 q[4];
                    w.operands(j, q);
                    auto sum = [&](int i) __attribute__((always_inline)) {
                        const auto e0 = __builtin_amdgcn_cvt_pk_f32_fp8((int)e[i], false), e1 = __builtin_amdgcn_cvt_pk_f32_fp8((int)e[i], true);
#pragma unroll
                        for (int p = 0; p < PAIRS; ++p) {
                            const f32x4& z = xs[i & 1][p];
                            float& r = acc[p][i & 1];
                            r = __builtin_fmaf(d[i & 1][4 * p], e0[0] * z[0], r);
                            r = __builtin_fmaf(d[i & 1][4 * p + 1], e0[1] * z[1], r);
                            r = __builtin_fmaf(d[i & 1][4 * p + 2], e1[0] * z[2], r);
                            r = __builtin_fmaf(d[i & 1][4 * p + 3], e1[1] * z[3], r);
                        }
                    };
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const i32x8 b = {(int)q[i][0], (int)q[i][1], (int)q[i][2], (int)q[i][3], 0, 0, 0, 0};
                        const i32x8 lo = operand(y[i & 1][0]), hi = operand(y[i & 1][1]);
                        if (i < 3) bring(i + 1);
                        d[i & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(lo, b, f32x16{}, 2, 4, 0, kOne, 0, 127);
                        d[i & 1] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(hi, b, d[i & 1], 2, 4, 0, k16, 0, 127);
                        __builtin_amdgcn_sched_barrier(0);
                        if (i > 0) sum(i - 1);
                        if (i < 3) bring_scales(i + 1);
                        __builtin_amdgcn_sched_barrier(0);
                    }
                    sum(3);
                    o += 512 * kIn;
                    ox += 64 * kIn;
                }
                w.load(next, j, from + j, j < per && from + j < full);
            }
            if (slot < slots) {
#pragma unroll
                for (int p = 0; p < PAIRS; ++p) sums[((grp * slots + slot) * kIn + 2 * p + g) * 32 + c] = acc[p][0] + acc[p][1];
            }
        }
        __syncthreads();
        nvfp4_finish<PAIRS, SWIGLU, kRows, 32>(a, sums, first, each, stride, groups, slots);
        row += turn_rows;
    }
}

// Tiles side by side in a block, that share its activations: up to 1, 2, 4 or 4 for 1 to 4 pairs of rows, while there are as many for every
// compute unit. Three tiles a unit are one block's: in blocks of two a unit has two or four (3 rows of 10240 x 5120 12.3 us, so 11.3; 5
// rows of 9001 x 5136 17.0 and 14.8; 3 rows of 9216 x 16384 27.1 and 22.7).
static constexpr int nvfp4_groups(int pairs, int least, int tiles) {
    int groups = pairs == 1 ? 1 : pairs == 2 ? 2 : 4;
    if (groups < least) groups = least;
    while (groups > least && tiles * least < 256 * groups) groups >>= 1;
    return least == 1 && groups == 2 && tiles > 512 && tiles <= 768 ? 3 : groups;
}
// (up to four tiles a unit, where LDS has room for a block's: every unit's are whole blocks; from five on rounds run into one another)
static constexpr bool nvfp4_shares_are_even() {
    for (int pairs = 1; pairs <= kMaxRows / 2; ++pairs)
        for (int tiles = 1; tiles <= 4 * 256; ++tiles)
            if ((tiles + 255) / 256 % nvfp4_groups(pairs, 1, tiles)) return false;
    return true;
}
static_assert(nvfp4_shares_are_even(), "a compute unit's tiles are whole blocks");
struct Nvfp4Plan { int per, slots, groups, waves, bytes, tile_rows, tiles; };
template <int PAIRS, bool SWIGLU, bool RESIDENT>
static int launch_nvfp4_wide(const Nvfp4Args& a, const Nvfp4Plan& p, hipStream_t s) {
    const int tiles = (a.rows + p.tile_rows - 1) / p.tile_rows, units = (tiles + p.groups - 1) / p.groups, grid = units < 256 ? units : 256;
    Q27X_HIP((allow_lds<k_nvfp4_wide<PAIRS, SWIGLU, RESIDENT>>(kNvLds)));
    hipLaunchKernelGGL((k_nvfp4_wide<PAIRS, SWIGLU, RESIDENT>), dim3((unsigned)grid), dim3(64 * p.groups * p.waves), p.bytes, s, a, p.tile_rows,
                       p.groups, p.waves, p.per, p.slots);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}
template <int PAIRS, bool SWIGLU, bool RESIDENT>
static int launch_nvfp4_form(const Nvfp4Args& a, const Nvfp4Plan& p, hipStream_t s) {
    const int wide = SWIGLU ? p.groups / 2 : p.groups, units = (p.tiles + wide - 1) / wide;
    int fit = kNvLds / p.bytes;                      // blocks of a compute unit
    const int room = (RESIDENT ? kNvWaves : kNvWaves / 2) / (p.groups * p.waves);
    fit = fit < room ? fit : room;
    fit = fit < 1 ? 1 : fit;
    const int grid = 256 * fit < units ? 256 * fit : units;
    Q27X_HIP((allow_lds<k_nvfp4<PAIRS, SWIGLU, RESIDENT>>(kNvLds)));
    hipLaunchKernelGGL((k_nvfp4<PAIRS, SWIGLU, RESIDENT>), dim3((unsigned)grid), dim3(64 * p.groups * p.waves), p.bytes, s, a, p.tile_rows, p.groups,
                       p.waves, p.per, p.slots);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}
template <int PAIRS, bool SWIGLU>
static int launch_nvfp4_pairs(const Nvfp4Args& a, hipStream_t s) {
    const int steps = (a.K + kNvStep - 1) / kNvStep, tiles = (a.rows + 15) / 16;
    const bool ends_inside = a.K % kNvStep != 0;
    constexpr int least = SWIGLU ? 2 : 1;
    Nvfp4Plan p;
    p.per = steps <= 4 ? 1 : steps <= 8 ? 2 : kNvSteps;
    p.slots = (steps + p.per - 1) / p.per;
    // tiles of fewer rows, as many for every compute unit (cold weights, 5120 x 17408, 1 row: 10 of 16 rows 14.4 us, all 16 16.7; 5120 x
    // 5120, 3 rows 8.3 and 8.9; 17408 x 5120, five tiles a unit, 15.6 and 16.0; 34816 x 5120, nine, the same; where a unit has one at most it
    // is no gain: 1024 x 768 4.2 and 3.9)
    const int n = SWIGLU || tiles <= 256 ? 0 : (tiles + 255) / 256;
    p.tile_rows = n ? (a.rows - 1) / (256 * n) + 1 : 16;
    p.tiles = (a.rows + p.tile_rows - 1) / p.tile_rows;
    const int side = nvfp4_groups(PAIRS, least, p.tiles);
    auto fits = [&](int groups) {                    // all activations in LDS, tiles side by side that share them
        const int most = kNvWaves / groups, turns = (p.slots + most - 1) / most;
        p.groups = groups;
        p.waves = (p.slots + turns - 1) / turns;
        p.bytes = Nvfp4Lds(a.nr, steps, p.per, groups, p.waves, p.slots, 32 * PAIRS, ends_inside).total;
        return p.bytes <= kNvLds;
    };
    const int tiles32 = SWIGLU ? tiles : (tiles + 1) / 2;
    auto fits_wide = [&](int most, bool resident) {
        const int turns = (p.slots + most - 1) / most;
        p.waves = (p.slots + turns - 1) / turns;
        p.bytes = Nvfp4WideLds(2 * PAIRS, resident ? steps : p.waves * p.per, p.per, p.groups, p.waves, p.slots, ends_inside).total;
        return p.bytes <= kNvLds;
    };
    // 5 rows and more: tiles of 32 weight rows, where there are enough of them. Against those of 16: 62080 x 5120, 8 rows 37 us (45), 5
    // rows 36 (39); gate | up 17408 x 5120 29.6 (36.8), 29 (32); 5120 x 5120 11.9 (15.3), 11.6 (11.5); with fewer tiles than here
    // 1024 x 768 5.6 (4.8), and 9001 x 5136, 5 rows 19.8 (14.8); 3 rows 33.4 (33.2) and 26.8 (24.8). Not where three tiles of 16 are a
    // unit's: cold weights, 9001 x 5136, 8 rows 20.8 (16.6), 10240 x 1024 8.5 (7.4), 12288 x 5120 16.4 (16.2).
    if constexpr (PAIRS >= kWidePairs) {
        if (tiles32 >= (PAIRS == 4 ? 160 : 512) && !(side == 3 && fits(3))) {
            const Nvfp4Plan narrow = p;
            p.groups = tiles32 < 512 ? 1 : 2;        // (tiles for every compute unit)
            p.tile_rows = SWIGLU ? 16 : 32;
            if (fits_wide(kNvWideWaves / p.groups, true)) return launch_nvfp4_wide<PAIRS, SWIGLU, true>(a, p, s);
            p = narrow;
        }
    }
    for (int groups = side;; groups = groups == 3 ? 2 : groups >> 1) {
        if (fits(groups)) return launch_nvfp4_form<PAIRS, SWIGLU, true>(a, p, s);
        if (groups == least) break;
    }
    // activations in turns: 32 weight rows where that is a tile for each compute unit at most, or 5 or 6 rows, or gate | up; and 4 waves have
    // room beside the sums. Against 16: 5120 x 17408, 5 rows 24.9 us (34.3), 8 rows 34.7 (37.6), 9001 x 17408 42 (49), 63 (54), gate |
    // up 17408 x 12288 96 (112), 115 (122), 5120 x 57344 81 (92), 170 (101; 2 waves)
    if constexpr (PAIRS >= kWidePairs) {
        if (tiles32 >= 160 && (PAIRS == 3 || SWIGLU || tiles32 <= 256)) {
            const Nvfp4Plan narrow = p;
            p.groups = 1;
            const int shares = (tiles32 + 255) / 256;
            p.tile_rows = SWIGLU ? 16 : (a.rows - 1) / (256 * shares) + 1;
            for (int most = kNvWideWaves; most >= 4; --most)
                if (fits_wide(most, false)) return launch_nvfp4_wide<PAIRS, SWIGLU, false>(a, p, s);
            p = narrow;
        }
    }
    const int most = kNvWaves / 2 / least, turns = (p.slots + most - 1) / most;
    p.waves = (p.slots + turns - 1) / turns;
    p.bytes = Nvfp4Lds(a.nr < 4 ? a.nr : 4, p.waves * p.per, p.per, p.groups, p.waves, p.slots, 32 * PAIRS, ends_inside).total;
    if (p.bytes > kNvLds) { set_error("nvfp4: K=%d: %d bytes of LDS", a.K, p.bytes); return Q27X_E_SHAPE; }
    return launch_nvfp4_form<PAIRS, SWIGLU, false>(a, p, s);
}
template <bool SWIGLU>
static int launch_nvfp4(const Nvfp4Args& a, hipStream_t s) {
    switch ((a.nr + 1) / 2) {
        case 1: return launch_nvfp4_pairs<1, SWIGLU>(a, s);
        case 2: return launch_nvfp4_pairs<2, SWIGLU>(a, s);
        case 3: return launch_nvfp4_pairs<3, SWIGLU>(a, s);
        default: return launch_nvfp4_pairs<4, SWIGLU>(a, s);
    }
}

// the caller's matrix and rows, checked
static int nvfp4_args(const q27x_nvfp4_t* w, const char* who, const int8_t* xq, int xstride, const float* xs, int nr) {
    if (!w || !w->w || !w->s || !xq || !xs) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if (w->rows < 1 || w->rows > kNvMaxRows || w->K < 16 || (w->K & 15) || w->K > kNvMaxK) {
        set_error("%s: unsupported shape (rows=%d K=%d: K a multiple of 16 up to %d)", who, w->rows, w->K, kNvMaxK);
        return Q27X_E_SHAPE;
    }
    if (nr < 1 || nr > kMaxRows) { set_error("%s: nr=%d: 1 to %d rows", who, nr, kMaxRows); return Q27X_E_SHAPE; }
    if (nr > 1 && (xstride < w->K || (xstride & 15))) {
        set_error("%s: xstride=%d: at least K=%d, a multiple of 16", who, xstride, w->K);
        return Q27X_E_ARG;
    }
    if ((long long)(nr - 1) * (nr > 1 ? xstride : 0) + w->K > 0x7fffffffLL) {
        set_error("%s: rows of activations over more than 2^31 - 1 bytes", who);
        return Q27X_E_RANGE;
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
    return launch_nvfp4<false>(a, (hipStream_t)s);
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
    return launch_nvfp4<true>(a, (hipStream_t)s);
}

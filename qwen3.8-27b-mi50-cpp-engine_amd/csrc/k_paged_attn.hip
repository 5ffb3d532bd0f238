// k_paged_attn.hip -- attention of new rows over a paged key/value cache.
//
// Row i of a sequence's n new rows sees keys 0 .. len - n + i of its cache. For every query head, with x = q.k / sqrt(hd):
// out = sum e^(x - M) v / sum e^(x - M), M = max x, times sigmoid(gate); a row that sees nothing gets zeros.
//
// Keys are cut into fixed splits of 256 and these into chunks of 64, so a row's result depends on its own keys alone,
// whatever else is in the batch. A wave takes a chunk for up to 16 RT columns, the pairs
// of a row and a query head of its kv head: it has the chunk's scores before it needs their maximum, so the chunk has one
// maximum and one exponential, and leaves (m, l, o). Chunks are joined in order, (m, l, o) <- (m', l e^(m - m') + l_c e^(m_c
// - m'), ..), m' = max(m, m_c); k_paged_join joins the splits. Two forms of the same arithmetic, the same bits:
//   PAR: block = a split's chunks, one a wave, joined through LDS: as many waves as can be, for few keys.
//   else: a wave walks a split's chunks and joins them in registers; waves are independent (no barrier), each with the
//     next chunk's keys and values on their way, for many keys.
//
// Scores on v_mfma_f32_16x16x32_bf16 as K Q^T: lane (c, g) = (lane & 15, lane >> 4) holds dims 32 i + 8 g .. + 7 of key
// c, and gets keys 4 g .. 4 g + 3 of column c. Codes and queries are bf16 exactly; the fp32 sum of each scale group
// is multiplied by the key's scale afterwards, so scores carry no rounding but fp32's. One dword a lane holds a tile's
// scales (key 4 g + c % 4, group c / 4), handed to the row's lanes by DPP.
// P.V as V^T P^T: the columns' weights are already where the second product wants them (slots 8 g .. of column c: keys
// 4 g .. of two tiles), and lane (c, g) loads dims c HD/16 .. of keys 4 g .. + 3, so V needs no transpose: byte t of the
// eight keys is row c of dim tile t. A value is code x scale rounded to fp16, scales first brought to [1, 2) by the power
// of two of the largest in the chunk and group (undone in fp32), weights (at most 1) are rounded to fp16: 2^-11 each, below
// the bf16 output's 2^-8, but 2^-25 of the chunk's largest weight or scale where less than 2^-14 of it is left. The chunk's
// largest is that of the keys that a row sees: where a later row's key would change it so that it shows, the
// rows' products run one after another. One fp16 term each is a choice: of 16 x 4099 keys the outputs are 1.662e-3 from
// the 64-bit ones (relative, whole tensor), 1.646e-3 with two terms each, which is the bf16 output's own rounding; two cost
// 14 to 19% (16 x 4099 keys, 3 rows, 256-wide 77 -> 91 us, 32 x 4097 keys, 128-wide 75.5 -> 89.7), and two for the weights alone
// change next to nothing (1.659e-3, 77 -> 82 us). bf16 pages: values exact, weights as two bf16 terms (2^-16).
//
// Loads: a vector load costs the texture addresser about 2.3 to 4 cycles per row of the cache that it touches (measured:
// 8 bytes a lane over 16 rows 67 cycles, over 4 rows 18; 16 bytes a lane over 8 rows 21), so K comes by LDS DMA in whole
// rows of a head, swizzled so that the operand reads of 16 rows meet distinct banks, and V in rows over 16 lanes. K read
// straight into operands, 32 bytes of 16 rows at a time, held 64 x 8000 keys to 3.2 TB/s.
//
// Bound: bf16 pages by memory (64 x 4000 keys, 1.05 GB: 191 us, 5.5 TB/s; its loads without the arithmetic 189). int8 pages
// by both sides, which overlap for the most part (32 x 4097 keys, 302 MB: 76 us; the loads alone 63, the arithmetic on
// keys in the L2 59). Two column tiles of 256-wide heads by one wave's latencies (16 x 4099 keys, 3 rows, 151 MB: 78 us, the
// arithmetic alone 74): it has its SIMD to itself, and vector instructions fill half of its time, matrix ones a twelfth.
#include <math.h>

#include "q27x_paged.h"

namespace q27x {

constexpr int kPSplit = 256;
constexpr int kCUs = 256;             // compute units of an MI355X
constexpr int kChunk = 64, kChunks = kPSplit / kChunk;
constexpr int kCounted = 256;          // sequences whose splits the split kernel counts before it begins

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct PAttnArgs {
    const uint16_t* qh; const uint16_t* qkv; int qkv_stride;
    PagedArgs kv;
    int nq, gate, max_len, max_rows, nrows, ns;      // ns: splits of max_len
    float sl2e;                                      // log2(e) / sqrt(hd)
    float* po; float* pm; float* pl;                 // splits' outputs [row][head][ns][hd], maxima and sums [row][head][ns]
    float* pp; float* pmc; float* fin;               // with w: e^(x - m) [row][head][ns 256], chunk maxima [row][head][ns chunks], (M, l)
    uint16_t* out; int8_t* xq; float* xs;
    float* w; int w_stride;
    int par;                                         // PAR throughout: sequences of one split are finished by it
};

// lane n of the 16-lane row, in every lane of it, and lane j of every quad in its four lanes (n, j constants after
// unrolling)
__device__ __forceinline__ float row_bcast(float x, int n) {
    const int v = __float_as_int(x);
#define Q27X_RB(N) case N: return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x150 + N, 0xF, 0xF, false))
    switch (n & 15) {
        Q27X_RB(0); Q27X_RB(1); Q27X_RB(2); Q27X_RB(3); Q27X_RB(4); Q27X_RB(5); Q27X_RB(6); Q27X_RB(7);
        Q27X_RB(8); Q27X_RB(9); Q27X_RB(10); Q27X_RB(11); Q27X_RB(12); Q27X_RB(13); Q27X_RB(14);
        default: return __int_as_float(__builtin_amdgcn_mov_dpp(v, 0x15F, 0xF, 0xF, false));
    }
#undef Q27X_RB
}
__device__ __forceinline__ float byte_f(uint32_t x, int i) { return (float)(int8_t)(x >> (8 * i)); }
// two floats that bf16 holds exactly
__device__ __forceinline__ uint32_t pack_bf(float lo, float hi) {
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const h2 v = {(_Float16)lo, (_Float16)hi};
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ bool finite_f(float x) { return (__float_as_uint(x) & 0x7F800000u) != 0x7F800000u; }
__device__ __forceinline__ float max_cols(float x) { x = fmaxf(x, xor16(x)); return fmaxf(x, xor32(x)); }
__device__ __forceinline__ float sum_cols(float x) { x = x + xor16(x); return x + xor32(x); }
// e^(x - M) of the base-2 logits, 0 where no key was seen (m = -inf); M is finite or no split saw any
__device__ __forceinline__ float weight_of(float m, float M) {
    return m == -__builtin_huge_valf() ? 0.0f : __builtin_amdgcn_exp2f(m - M);
}

// out = o / l x sigmoid(gate) as bf16, and if wanted its per-16 codes: 16 neighbouring lanes hold 16 neighbouring dims
__device__ __forceinline__ void put_out(const PAttnArgs& a, int hd, size_t row, int head, int d, float o, float l) {
    float v = l == 0.0f ? 0.0f : o / l;
    if (a.gate) v = v * qsigmoid(bf2f(a.qkv[row * a.qkv_stride + (size_t)head * 2 * hd + hd + d]));
    const uint16_t vb = f2bf(v);
    const size_t k = (row * a.nq + head) * hd + d;
    a.out[k] = vb;
    if (a.xq) {
        const float yv = bf2f(vb);
        const float sc = max_xor(fabsf(yv), 16) * (1.0f / 127.0f);
        a.xq[k] = qcode(yv, sc > 0.0f ? 1.0f / sc : 0.0f);
        if ((d & 15) == 0) a.xs[k >> 4] = sc;
    }
}

// Keys of sequence b that a call reads, and its rows (first, n; nr of them computed).
struct SeqOf { int first, n, nr, raw, len; };
__device__ __forceinline__ SeqOf seq_of(const PAttnArgs& a, int b) {
    SeqOf q;
    paged_rows(a.kv, b, q.first, q.n);
    q.nr = min(min(q.n, a.max_rows), a.nrows - q.first);
    q.raw = a.kv.lens[b];
    const long long cap = paged_cap(a.kv);
    q.len = min(q.raw, a.max_len);
    q.len = q.len < cap ? q.len : (int)cap;
    return q;
}

// The same of a sequence that all lanes ask for, by scalar loads.
__device__ __forceinline__ SeqOf seq_of_all(const PAttnArgs& a, int b) {
    SeqOf q;
    q.first = a.kv.row_start ? ld_uniform(a.kv.row_start + b) : b;
    q.n = a.kv.row_start ? ld_uniform(a.kv.row_start + b + 1) - q.first : 1;
    if (q.n < 0 || q.first < 0) q.n = 0;
    q.nr = min(min(q.n, a.max_rows), a.nrows - q.first);
    q.raw = ld_uniform(a.kv.lens + b);
    const long long cap = paged_cap(a.kv);
    q.len = min(q.raw, a.max_len);
    q.len = q.len < cap ? q.len : (int)cap;
    return q;
}
__device__ __forceinline__ int splits_of(const SeqOf& q) {
    return q.nr <= 0 ? 0 : q.len <= kPSplit ? 1 : (q.len + kPSplit - 1) / kPSplit;
}
// The call's (sequence, split) pairs in order, without those that are empty, 64 sequences at a time: lane l holds the running
// count up to sequence base + l. A wave walks them forwards only.
struct Items {
    int base, before, upto;                          // sequences and pairs before these 64; upto: this lane's running count
    __device__ __forceinline__ void load(const PAttnArgs& a, int b0, int n0) {
        base = b0;
        before = n0;
        const int b = b0 + (int)(threadIdx.x & 63);
        int x = b < a.kv.n_seq ? splits_of(seq_of(a, b)) : 0;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int y = __shfl_up(x, o, 64);
            x += (int)(threadIdx.x & 63) >= o ? y : 0;
        }
        upto = n0 + x;
    }
    // pair `item` (not smaller than the last one asked for): false behind the last
    __device__ __forceinline__ bool find(const PAttnArgs& a, int item, int& b, int& sp) {
        int last = __builtin_amdgcn_readlane(upto, 63);
        while (item >= last) {
            if (base + 64 >= a.kv.n_seq) return false;
            load(a, base + 64, last);
            last = __builtin_amdgcn_readlane(upto, 63);
        }
        const int k = __popcll(__ballot(upto <= item));
        b = base + k;
        sp = item - (k ? __builtin_amdgcn_readlane(upto, k - 1) : before);
        return true;
    }
};

// Units side by side for a kv head's columns. More than 32 of them (16 RT at a time) read the keys again: 16 x 4099 keys of 24 / 4
// heads take 55 us with one row (6 columns), 78 with three (18), 133 with eight (48, two units).
__host__ __device__ __forceinline__ int column_blocks(const PAttnArgs& a, int rt) {
    return (a.max_rows * (a.nq / a.kv.nkv) + 16 * rt - 1) / (16 * rt);
}

template <int HD, int G, int RT, bool PAR>
struct AttnShape {
    static constexpr int NCH = kChunks, CH = kChunk;
    static constexpr int KB = HD * (G ? 1 : 2);                                    // bytes of a key's row
    static constexpr int kWaves = PAR ? NCH : 4;
    static constexpr int kKeyBytes = CH * KB;                                      // a wave's K in LDS
    static constexpr int kOffs = PAR ? CH : kPSplit;                               // and its keys' positions
    static constexpr int CG = HD == 128 ? 8 : 4;                                   // columns joined at a time (PAR)
    static constexpr int kWaveBytes = kKeyBytes + 8 * kOffs;
    static constexpr int kJoinBytes = PAR ? kWaves * 16 * RT * 8 : 0;
    static constexpr int kLds = kWaves * kWaveBytes + kJoinBytes;                  // (not PAR: no less than PAR's)
    static constexpr int kXBytes = kWaves * CG * (HD + 4) * 4;                     // (the exchange lies over the keys)
    static_assert(!PAR || kXBytes <= kWaves * kWaveBytes, "exchange");
    // Waves of a SIMD that the registers are cut for. More in flight is not more: 64 x 4000 keys on bf16 pages take 192 us
    // with two waves a SIMD (not PAR), 207 with three; int8 PAR 89 with two, 85 with three, 98 with four. 256-wide heads (32 x
    // 4099 keys, one, two waves): groups of 32 89 / 81, of 64 83 / 69; of 16 107 / 194, the second wave's registers spill.
    // Some forms spill a little all the same, in bytes a lane (not PAR): two tiles of 256 dims by 16 368, of 128 dims by 16 116,
    // of 128 dims bf16 32, one tile of 256 dims by 32 12. Their times beside groups that do not: 16 x 4099 keys, 3 rows,
    // 256-wide by 16 113 us, by 32 78, by 64 72; 32 x 4097 keys, 8 rows, 128-wide by 16 145, by 32 124, bf16 155 (1.8 times
    // the bytes).
    static constexpr int kOcc = HD == 128 ? (RT == 1 && G && PAR ? 3 : 2) : RT == 1 && G && (G != 16 || PAR) ? 2 : 1;
    static constexpr int kBlocks = kCUs / 8 * (160 * 1024 / kLds < 4 * kOcc / kWaves ? 160 * 1024 / kLds : 4 * kOcc / kWaves);    // an XCD's at once
    // Units a block that are left to PAR at most, rather than a round of waves of their own. Measured (PAR / not, us, join
    // and all): one tile, 128-wide int8, 64 blocks of an XCD: 136 units 30 / 36, 204 units 40 / 37; bf16 the same way, 136
    // units 35 / 39, 204 units 46 / 43. A wave a SIMD (bf16, 256-wide), 32 blocks: 34 units 36 / 41, 68 units 53 / 44. Two
    // tiles (the joins double, and a wave's registers), 256-wide, 32 blocks: 42 units left 102 / 94, 68 units 74 / 52.
    static constexpr unsigned kTail = RT == 2 ? 1 : kOcc == 1 ? 2 : 3;
};

// One wave's work on one chunk after another: the split's running (m, l, o) of its columns, and the chunk's K, V and scales.
template <int HD, int G, int RT, bool PAR>
struct Chunker {
    using S = AttnShape<HD, G, RT, PAR>;
    static constexpr int E = HD / 16;                // dims of V a lane holds
    static constexpr int NM = HD / 32;               // products of a score tile
    static constexpr int NG = G ? HD / G : 1;        // scale groups of a head
    static constexpr int NS = NG > 4 ? NG / 4 : 1;   // scale registers of a tile
    static constexpr int VW = G ? E / 4 : E / 2;     // registers of a key's V dims
    static constexpr int NT = S::CH / 16, NU = S::CH / 32;
    static constexpr int SL = S::KB / 16;            // 16-byte pieces of a key's row
    static constexpr int kVLoads = NT * 4 * (VW > 4 ? VW / 4 : 1);
    static constexpr float kNone = -__builtin_huge_valf();
    typedef uint32_t vvec __attribute__((ext_vector_type(VW)));

    const PAttnArgs& a;
    char* keys;                                      // this wave's LDS: K
    uint64_t* offs;                                  // and its keys' positions in the pool, in elements
    int l, c, g;
    uint64_t width, hoff;
    float ksc[NT][NS], vsc[NT][NS];                  // scales of key 16 ti + 4 g + c % 4
    uint32_t vx[NT][4][VW];                          // V: dims E c .. of key 16 ti + 4 g + j
    u32x4 qx[RT][NM];                                // queries: dims 32 i + 8 g .. of column c
    int last[RT];                                    // the last key that the column sees
    size_t prow[RT];                                 // its (row, head)
    bool on[RT];
    float m[RT], lsum[RT];
    f32x4 o[RT][E];

    __device__ __forceinline__ Chunker(const PAttnArgs& args) : a(args) {}

    __device__ __forceinline__ void begin() {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            m[rt] = kNone;
            lsum[rt] = 0.0f;
#pragma unroll
            for (int e = 0; e < E; ++e) o[rt][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
    }
    __device__ __forceinline__ void columns(const SeqOf& q, int kvh, int col0, int ncol, int grp) {
        hoff = (uint64_t)kvh * HD;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            on[rt] = 16 * rt + c < ncol;
            const int col = on[rt] ? col0 + 16 * rt + c : 0;
            last[rt] = on[rt] ? q.raw - q.n + col / grp : -1;
            prow[rt] = (size_t)(q.first + col / grp) * a.nq + (size_t)kvh * grp + col % grp;
            const uint16_t* p = a.qh + prow[rt] * HD + 8 * g;
            typedef uint32_t u32x4u __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                const u32x4 x = *(const u32x4u*)(p + 32 * i);
                qx[rt][i] = on[rt] ? x : u32x4{0, 0, 0, 0};
            }
        }
    }
    // K of the chunk whose keys' positions begin at offs[k], on its way into LDS, and its scales into registers. Piece s
    // of key r lies at place s ^ f(r), f(r) = r / 2 % 8 for rows of 128 bytes and r % 16 for longer ones: 16 rows' reads
    // of one piece then meet all banks.
    __device__ __forceinline__ int place(int r, int s) const { return s ^ (SL == 8 ? (r >> 1) & 7 : r & 15); }
    __device__ __forceinline__ void load_k(int k) {
        if constexpr (G != 0) {
#pragma unroll
            for (int ti = 0; ti < NT; ++ti) {
                const uint64_t srow = (offs[k + 16 * ti + 4 * g + (c & 3)] + hoff) / G;
#pragma unroll
                for (int u = 0; u < NS; ++u) ksc[ti][u] = a.kv.ks[srow + (NG >= 4 ? (c >> 2) + 4 * u : (c >> 2) % NG)];   // groups c / 4 + 4 u
            }
        }
        const uint32_t lds = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)keys);
        constexpr int RD = 64 / SL;                  // rows of a transfer
#pragma unroll
        for (int i = 0; i < S::CH / RD; ++i) {
            const int r = RD * i + l / SL;
            const char* p = (const char*)a.kv.k + (offs[k + r] + hoff) * (G ? 1 : 2) + 16 * place(r, l % SL);
            lds_dma16_nt(p, lds + 1024 * i);
        }
    }
    __device__ __forceinline__ vvec v_at(int k) const {
        const uint64_t at = offs[k] + hoff + E * c;
        return __builtin_nontemporal_load((const vvec*)((const char*)a.kv.v + (G ? at : 2 * at)));
    }
    __device__ __forceinline__ void load_v(int k) {
        if constexpr (G != 0) {
#pragma unroll
            for (int ti = 0; ti < NT; ++ti) {
                const uint64_t srow = (offs[k + 16 * ti + 4 * g + (c & 3)] + hoff) / G;
#pragma unroll
                for (int u = 0; u < NS; ++u) vsc[ti][u] = a.kv.vs[srow + (NG >= 4 ? (c >> 2) * NS + u : (c >> 2) * NG / 4)];  // the quad's dims' groups
            }
        }
#pragma unroll
        for (int ti = 0; ti < NT; ++ti)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const vvec x = v_at(k + 16 * ti + 4 * g + j);
#pragma unroll
                for (int u = 0; u < VW; ++u) vx[ti][j][u] = x[u];
            }
    }

    float s[RT][NT][4];
    // Scores of the chunk (times nothing yet). The caller has waited for K.
    typedef uint32_t kvec __attribute__((ext_vector_type(G ? 2 : 4)));
    // dims 32 i + 8 g .. of key r
    __device__ __forceinline__ kvec k_at(int r, int i) const {
        const char* row = keys + r * S::KB;
        if constexpr (G == 0) return *(const kvec*)(row + 16 * place(r, 4 * i + g));
        else return *(const kvec*)(row + 16 * place(r, 2 * i + (g >> 1)) + 8 * (g & 1));
    }
    __device__ __forceinline__ void scores() {
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        kvec first = k_at(c, 0);
#pragma unroll
        for (int ti = 0; ti < NT; ++ti) {
            __builtin_amdgcn_sched_barrier(0);        // (tiles widened ahead of their products spill)
            uint32_t low = g < 2 ? ~0u : 0u;           // (opaque: masked queries are not worth registers of their own)
            if constexpr (G == 16) asm volatile("" : "+v"(low));
            // products of a group after another, a group's scales applied while the next one's product runs
            constexpr int NP = G == 16 ? 2 * NM : NM, PG = G == 0 ? NP : G == 16 ? 1 : G / 32;    // products, and of a group
            f32x4 acc[2][RT];
            u32x4 kb;
            kvec x = first;
            auto scale = [&](int gr) __attribute__((always_inline)) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float k = row_bcast(ksc[ti][gr >> 2], 4 * (gr & 3) + j);
                        s[rt][ti][j] = gr == 0 ? acc[gr & 1][rt][j] * k : __builtin_fmaf(acc[gr & 1][rt][j], k, s[rt][ti][j]);
                    }
            };
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const int i = G == 16 ? p / 2 : p, gr = p / PG;
                if constexpr (G != 0) __builtin_amdgcn_sched_barrier(0);
                if (G != 16 || p % 2 == 0) {
                    // the operand after this one is requested first
                    const kvec now = x;
                    if (i + 1 < NM) x = k_at(16 * ti + c, i + 1);
                    else if (ti + 1 < NT) first = k_at(16 * ti + 16 + c, 0);
                    if constexpr (G == 0) {
                        kb = now;
                    } else {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            kb[2 * h] = pack_bf(byte_f(now[h], 0), byte_f(now[h], 1));
                            kb[2 * h + 1] = pack_bf(byte_f(now[h], 2), byte_f(now[h], 3));
                        }
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    // (a group of 16: the other half of the lanes' queries zeroed)
                    const u32x4 qm = G != 16 ? qx[rt][i] : qx[rt][i] & (p % 2 ? ~low : low);
                    acc[gr & 1][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, kb), __builtin_bit_cast(bf16x8, qm),
                                                                              p % PG ? acc[gr & 1][rt] : zero, 0, 0, 0);
                }
                if (G != 0 && p % PG == 0 && gr > 0) scale(gr - 1);
            }
            if constexpr (G != 0) {
                scale(NP / PG - 1);
            } else {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[rt][ti][j] = acc[0][rt][j];
            }
            // (pinned here: moved behind the next branch, the products and scales would all be kept until then)
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(s[rt][ti][j]));
        }
    }
    // V and its scales have come: what follows does not wait for loads issued later
    __device__ __forceinline__ void v_here() {
#pragma unroll
        for (int ti = 0; ti < NT; ++ti) {
            if constexpr (G != 0) {
#pragma unroll
                for (int u = 0; u < NS; ++u) asm volatile("" : "+v"(vsc[ti][u]));
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int u = 0; u < VW; ++u) asm volatile("" : "+v"(vx[ti][j][u]));
        }
    }

    uint32_t pw[RT][NU][4], plo[RT][NU][G == 0 ? 4 : 1];
    float f1[RT], f2[RT];
    // The chunk's weights e^(x - m), 0 for keys that the row does not see, and what the join multiplies: keys k0 .. of
    // the sequence, `valid` those that are there.
    __device__ __forceinline__ void weights(const SeqOf& q, int k0, uint64_t valid, int chunk0) {
        const bool full = valid == ~0ull && k0 + S::CH - 1 <= q.raw - q.n;
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (!full) {
                const int see = last[rt] - k0 - 4 * g;    // keys 16 ti + j of this lane up to here
#pragma unroll
                for (int ti = 0; ti < NT; ++ti) {
                    const uint32_t there = (uint32_t)(valid >> (16 * ti)) >> (4 * g);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[rt][ti][j] = (16 * ti + j <= see && ((there >> j) & 1)) ? s[rt][ti][j] : kNone;
                }
            }
            float mx = kNone;
#pragma unroll
            for (int ti = 0; ti < NT; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[rt][ti][j] *= a.sl2e;
                    mx = fmaxf(mx, s[rt][ti][j]);
                }
            mx = max_cols(mx);
            const float base = mx == kNone ? 0.0f : mx;
            float sum = 0.0f;
#pragma unroll
            for (int ti = 0; ti < NT; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[rt][ti][j] = __builtin_amdgcn_exp2f(s[rt][ti][j] - base);
                    sum += s[rt][ti][j];
                }
            sum = sum_cols(sum);
            const float mn = fmaxf(m[rt], mx);
            f1[rt] = weight_of(m[rt], mn);
            f2[rt] = weight_of(mx, mn);
            m[rt] = mn;
            lsum[rt] = __builtin_fmaf(sum, f2[rt], lsum[rt] * f1[rt]);
            if (a.w && on[rt]) {
                float* pp = a.pp + prow[rt] * ((size_t)a.ns * kPSplit) + (size_t)chunk0 * S::CH + 4 * g;
#pragma unroll
                for (int ti = 0; ti < NT; ++ti) *(f32x4*)(pp + 16 * ti) = f32x4{s[rt][ti][0], s[rt][ti][1], s[rt][ti][2], s[rt][ti][3]};
                if (g == 0) a.pmc[prow[rt] * ((size_t)a.ns * S::NCH) + chunk0] = mx;
            }
#pragma unroll
            for (int ti = 0; ti < NT; ++ti)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p0 = s[rt][ti][2 * h], p1 = s[rt][ti][2 * h + 1];
                    if constexpr (G != 0) {
                        pw[rt][ti >> 1][2 * (ti & 1) + h] = pack_f16(p0, p1);
                    } else {
                        const float h0 = bfr(p0), h1 = bfr(p1);
                        pw[rt][ti >> 1][2 * (ti & 1) + h] = pack_bf(h0, h1);
                        plo[rt][ti >> 1][2 * (ti & 1) + h] = pack_bf(bfr(p0 - h0), bfr(p1 - h1));
                    }
                }
        }
    }

    float fac[NS], back[NS];
    // the scale of this lane's dims at key j of the quad's four
    __device__ __forceinline__ float key_scale(const float (&v)[NS], int j) const {
        float x = quad_bcast(v[0], j);
#pragma unroll
        for (int u = 1; u < NS; ++u) {
            const float y = quad_bcast(v[u], j);      // (in every lane: a lane reads its neighbours')
            x = (c & 3) >= u * (4 / NS) ? y : x;
        }
        return x;
    }
    // V of the keys in `in` (others 0) times the weights, joined to o. ONE: added to what is joined, in the columns of the row
    // whose last key is `key`.
    template <bool ONE>
    __device__ __forceinline__ void product(uint64_t in, int key) {
        float vs[NT][NS];
        if constexpr (G != 0) {
#pragma unroll
            for (int ti = 0; ti < NT; ++ti)
#pragma unroll
                for (int u = 0; u < NS; ++u) vs[ti][u] = vsc[ti][u] * fac[u];
        }
        if (in != ~0ull) {
#pragma unroll
            for (int ti = 0; ti < NT; ++ti) {
                const uint32_t keep = (uint32_t)(in >> (16 * ti)) >> (4 * g);
                if constexpr (G != 0) {
#pragma unroll
                    for (int u = 0; u < NS; ++u) vs[ti][u] = (keep >> (c & 3)) & 1 ? vs[ti][u] : 0.0f;
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int u = 0; u < VW; ++u) vx[ti][j][u] = (keep >> j) & 1 ? vx[ti][j][u] : 0u;
                }
            }
        }
        float fb[RT][4];                              // the join's factor of output rows 4 g + j
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int j = 0; j < 4; ++j) fb[rt][j] = G ? f2[rt] * back[j * NS / 4] : f2[rt];
        // a dim tile's products are joined to o while the next tile's run
        f32x4 acc[2][RT];
        auto join = [&](int e) __attribute__((always_inline)) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float x = acc[e & 1][rt][j];
                    if constexpr (!ONE) o[rt][e][j] = __builtin_fmaf(x, fb[rt][j], o[rt][e][j] * f1[rt]);
                    else o[rt][e][j] = key == last[rt] ? __builtin_fmaf(x, fb[rt][j], o[rt][e][j]) : o[rt][e][j];
                }
        };
#pragma unroll
        for (int e = 0; e < E; ++e) {
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[e & 1][rt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < NU; ++u) {
                u32x4 va;
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const int ti = 2 * u + (h >> 1), j = 2 * (h & 1);
                    if constexpr (G != 0) {
                        va[h] = pack_f16(byte_f(vx[ti][j][e / 4], e & 3) * key_scale(vs[ti], j), byte_f(vx[ti][j + 1][e / 4], e & 3) * key_scale(vs[ti], j + 1));
                    } else {
                        va[h] = __builtin_amdgcn_perm(vx[ti][j + 1][e / 2], vx[ti][j][e / 2], (e & 1) ? 0x07060302u : 0x05040100u);
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    const u32x4 pb = {pw[rt][u][0], pw[rt][u][1], pw[rt][u][2], pw[rt][u][3]};
                    if constexpr (G != 0) {
                        acc[e & 1][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, va), __builtin_bit_cast(f16x8, pb), acc[e & 1][rt], 0, 0, 0);
                    } else {
                        const u32x4 pl = {plo[rt][u][0], plo[rt][u][1], plo[rt][u][2], plo[rt][u][3]};
                        acc[e & 1][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, pb), acc[e & 1][rt], 0, 0, 0);
                        acc[e & 1][rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, pl), acc[e & 1][rt], 0, 0, 0);
                    }
                }
            }
            if (e > 0) join(e - 1);
        }
        join(E - 1);
    }
    // The largest finite scale among the keys in `in` of group u of the quad's dims.
    __device__ __forceinline__ float top_scale(uint64_t in, int u) const {
        float mx = 0.0f;
#pragma unroll
        for (int ti = 0; ti < NT; ++ti) {
            const bool is = (in >> (16 * ti + 4 * g + (c & 3))) & 1;
            mx = fmaxf(mx, is && finite_f(vsc[ti][u]) ? fabsf(vsc[ti][u]) : 0.0f);
        }
        return max_cols(max_quad(mx));
    }
    __device__ __forceinline__ static int exponent_of(float x) {
        const int ex = (int)(__float_as_uint(x) >> 23);
        return ex < 1 ? 1 : ex > 253 ? 253 : ex;
    }
    // The power of two that brings the largest finite scale of each of the quad's groups to [1, 2), among the keys in `in`,
    // and its inverse for the output rows 4 g + j (the dims of quad g).
    __device__ __forceinline__ void factors(uint64_t in) {
        if constexpr (G != 0) {
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                const int ex = exponent_of(top_scale(in, u));
                fac[u] = __uint_as_float((uint32_t)(254 - ex) << 23);
                back[u] = __shfl(__uint_as_float((uint32_t)ex << 23), (l & 48) + 4 * g, 64);
            }
        }
    }
    // Whether the rows of the call have to be taken one by one, because a key that only later rows see would change what
    // the rows before it get. Its weight there is 0, but it counts where it is not finite, and where its scale changes the
    // factor: powers of two change nothing by themselves, so that takes a value that the larger factor's fp16 holds with
    // fewer bits (a scale below 2^-14 of the largest), or a factor of the join that fp32 does (from 2^-126 on; the bounds
    // here are far above). `first`: the keys of the first row that sees any.
    __device__ __forceinline__ bool apart(uint64_t valid, uint64_t first, uint64_t later) const {
        bool odd = false;
        if constexpr (G != 0) {
            bool moved = false, low = false;
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                const int ex = exponent_of(top_scale(valid, u)), ex0 = exponent_of(top_scale(first, u));
                moved = moved || ex != ex0;
                low = low || (ex != ex0 && ex0 < 64);
#pragma unroll
                for (int ti = 0; ti < NT; ++ti) {
                    const int bit = 16 * ti + 4 * g + (c & 3);
                    const uint32_t x = __float_as_uint(vsc[ti][u]) & 0x7FFFFFFFu;
                    odd = odd || (((later >> bit) & 1) && x >= 0x7F800000u);
                    low = low || (ex != ex0 && ((valid >> bit) & 1) && x != 0 && (int)(x >> 23) < ex - 14);
                }
            }
            if (__ballot(moved)) {
                odd = odd || low;
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) odd = odd || (f2[rt] != 0.0f && f2[rt] < 0x1p-60f);
            }
        } else {
#pragma unroll
            for (int ti = 0; ti < NT; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    if ((later >> (16 * ti + 4 * g + j)) & 1) {
#pragma unroll
                        for (int u = 0; u < VW; ++u)
                            odd = odd || (vx[ti][j][u] & 0x7F80u) == 0x7F80u || (vx[ti][j][u] & 0x7F800000u) == 0x7F800000u;
                    }
        }
        return __ballot(odd) != 0;
    }
    // The chunk's values joined to o: those of keys that are there (the others read something else, maybe not finite). All
    // rows at once where that gives each what it would get alone; else o joins nothing and each row adds its own keys,
    // values and scales read again: the same roundings, so a row's result is that of its own keys.
    __device__ __forceinline__ void values(const SeqOf& q, int k0, uint64_t valid, int k) {
        const int from = q.raw - q.n + 1 - k0;        // the first key that row 0 does not see
        uint64_t enter = valid;
        if (from < S::CH) {
            const uint64_t first = from <= 0 ? valid & 1 : valid & ((1ull << from) - 1), later = from <= 0 ? valid : valid & ~first;
            if (later && apart(valid, first, later)) enter = 0;
        }
        factors(enter);
        product<false>(enter, 0);
        if (enter == valid) return;
#pragma unroll 1
        for (int i = 0; i < q.nr; ++i) {
            const int end = from - 1 + i;             // row i's last key of the chunk
            if (end < 0) continue;
            const uint64_t in = end >= S::CH - 1 ? valid : valid & ((2ull << end) - 1);
            asm volatile("" : "+v"(k), "+v"(c), "+v"(g));     // (opaque: nothing is kept over the loop, which spills)
            load_v(k);
            __builtin_amdgcn_sched_barrier(0);
            if constexpr (G != 0) v_here();
            factors(in);
            product<true>(in, k0 + end);
        }
    }
};

// This block's (PAR) or wave's units from `unit` on, `step` apart, below `end`.
template <int HD, int G, int RT, bool PAR>
__device__ __forceinline__ void attn_units(const PAttnArgs& a, char* lds, Items& items, unsigned unit, unsigned step, unsigned end) {
    using S = AttnShape<HD, G, RT, PAR>;
    using C = Chunker<HD, G, RT, PAR>;
    const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const PagedArgs& kv = a.kv;
    const int grp = a.nq / kv.nkv, per = kv.nkv * column_blocks(a, RT);
    char* mine = lds + wv * S::kWaveBytes;
    for (; unit < end; unit += step) {
        const int sub = (int)(unit % (unsigned)per);
        int b, sp;
        if (!items.find(a, (int)(unit / (unsigned)per * 8u + (blockIdx.x & 7u)), b, sp)) return;
        const int kvh = sub % kv.nkv, col0 = sub / kv.nkv * 16 * RT;
        const SeqOf q = seq_of_all(a, b);
        const int ncol = min(q.nr * grp - col0, 16 * RT);        // this unit's columns
        if (ncol <= 0) continue;
        int t;
        C ch(a);
        auto lanes = [&]() __attribute__((always_inline)) {   // (opaque: what follows from it is not kept over a loop, which spills)
            t = threadIdx.x;
            asm volatile("" : "+v"(t));
            ch.l = t & 63;
            ch.c = t & 15;
            ch.g = (t >> 4) & 3;
        };
        lanes();
        ch.keys = mine;
        ch.offs = (uint64_t*)(mine + S::kKeyBytes);
        ch.width = (uint64_t)kv.nkv * HD;
        const int l = ch.l;
        const int k0 = sp * kPSplit + (PAR ? wv * S::CH : 0);
        if constexpr (PAR) __syncthreads();           // the unit before is read out of LDS
        // the positions of this wave's keys: lane l looks k0 + l, k0 + 64 + l .. up
        constexpr int NL = S::kOffs / 64;
        uint64_t there[NL];
#pragma unroll
        for (int u = 0; u < NL; ++u) {
            const int k = 64 * u + l;
            const int slot = k0 + k < q.len ? paged_slot(kv, b, k0 + k) : -1;
            there[u] = __ballot(slot >= 0);
            // (a key that is not there reads position 0 of the pool)
            ch.offs[k] = slot < 0 ? 0 : (uint64_t)(unsigned)slot * ch.width;
        }
        __builtin_amdgcn_wave_barrier();
        ch.begin();
        const int nch = PAR ? (there[0] != 0) : max(0, (min(q.len - sp * kPSplit, kPSplit) + S::CH - 1) / S::CH);
        auto valid_of = [&](int ci) __attribute__((always_inline)) {
            return ci == 0 ? there[0] : ci == 1 ? there[1 % NL] : ci == 2 ? there[2 % NL] : there[3 % NL];
        };
        ch.columns(q, kvh, col0, ncol, grp);
        if (nch > 0) {
            ch.load_k(0);
            ch.load_v(0);
        }
#pragma unroll 1
        for (int ci = 0; ci < nch; ++ci) {
            lanes();
            // K is behind by at least the V loads issued after it
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(C::kVLoads) : "memory");
            ch.scores();
            ch.v_here();
            if (ci + 1 < nch) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // (the operand reads of this chunk's K are done)
                ch.load_k((ci + 1) * S::CH);
            }
            const uint64_t valid = valid_of(ci);
            ch.weights(q, k0 + ci * S::CH, valid, sp * S::NCH + (PAR ? wv : ci));
            ch.values(q, k0 + ci * S::CH, valid, ci * S::CH);
            if (ci + 1 < nch) ch.load_v((ci + 1) * S::CH);
        }
        lanes();
        const int c = ch.c, g = ch.g;
        if constexpr (!PAR) {
            // lane (c, g): dims 4 E g .. of column c
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                if (!ch.on[rt]) continue;
                const size_t at = ch.prow[rt];
                const int d0 = 4 * C::E * g;
                if (g == 0) {
                    a.pm[at * a.ns + sp] = ch.m[rt];
                    a.pl[at * a.ns + sp] = ch.lsum[rt];
                }
                float* p = a.po + (at * a.ns + sp) * HD + d0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < C::E; e += 4)
                        *(f32x4*)(p + C::E * j + e) = f32x4{ch.o[rt][e][j], ch.o[rt][e + 1][j], ch.o[rt][e + 2][j], ch.o[rt][e + 3][j]};
            }
        } else {
            // the chunks joined in order, CG columns at a time
            float* s_m = (float*)(lds + S::kWaves * S::kWaveBytes);
            float* s_l = s_m + S::kWaves * 16 * RT;
            float* s_o = (float*)lds;
            constexpr int OS = HD + 4;
            const bool whole = a.par && q.len <= kPSplit;      // the sequence has no other split: finished here
            if (g == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    s_m[wv * 16 * RT + 16 * rt + c] = ch.m[rt];
                    s_l[wv * 16 * RT + 16 * rt + c] = ch.lsum[rt];
                    if (a.w && ch.on[rt] && nch == 0) a.pmc[ch.prow[rt] * ((size_t)a.ns * S::NCH) + sp * S::NCH + wv] = C::kNone;
                }
            }
#pragma unroll
            for (int cg = 0; cg < 16 * RT / S::CG; ++cg) {
                if (cg * S::CG < ncol) {              // (the same in every wave)
                    __syncthreads();                  // keys, or the columns before, are read out of LDS
                    constexpr int PT = 16 / S::CG;
                    if (c / S::CG == cg % PT) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int e = 0; e < C::E; e += 4) {
                                const f32x4* src = ch.o[cg / PT];
                                *(f32x4*)&s_o[(wv * S::CG + c % S::CG) * OS + C::E * (4 * g + j) + e] = f32x4{src[e][j], src[e + 1][j], src[e + 2][j], src[e + 3][j]};
                            }
                    }
                    __syncthreads();
                    const int nc = min(S::CG, ncol - cg * S::CG);
                    for (int i = t; i < nc * HD; i += 64 * S::kWaves) {
                        const int cc = i / HD, d = i % HD, col = cg * S::CG + cc;
                        float M = C::kNone, L = 0.0f, v = 0.0f;
#pragma unroll
                        for (int w = 0; w < S::kWaves; ++w) {
                            const float mw = s_m[w * 16 * RT + col], mn = fmaxf(M, mw);
                            const float f1 = weight_of(M, mn), f2 = weight_of(mw, mn);
                            M = mn;
                            L = __builtin_fmaf(s_l[w * 16 * RT + col], f2, L * f1);
                            v = __builtin_fmaf(s_o[(w * S::CG + cc) * OS + d], f2, v * f1);
                        }
                        const int gc = col0 + col;
                        const size_t row = (size_t)(q.first + gc / grp);
                        const int head = kvh * grp + gc % grp;
                        const size_t at = row * a.nq + head;
                        if (whole) put_out(a, HD, row, head, d, v, L);
                        else a.po[(at * a.ns + sp) * HD + d] = v;
                        if (d == 0) {
                            a.pm[at * a.ns + sp] = M;
                            a.pl[at * a.ns + sp] = L;
                        }
                    }
                }
            }
        }
    }
}

// Blocks j and j + 8 run on the same XCD: XCD x takes the pairs x, x + 8, .. with all their kv heads, which share the lines
// of the scales; its blocks (waves) take its (pair, head, columns) units in turn. ALL: every unit as PAR. Else the rounds
// that fill every wave, then what is left as PAR, if that is kTail units a block or fewer, as one more round of waves
// otherwise: 16 sequences of 4099 keys with 3 rows on 256-wide heads are 136 units for an XCD's 128 waves, 92 us in two rounds,
// 78 with 8 units left to PAR; 32 of 4097 keys on 128-wide ones 544 for 256, 76 with 32 left, 87 all as PAR. Where the rest is
// two units a block and some, the some go to the waves of as many blocks as they need, in the time of the others' two: 48
// sequences of 8 to 8190 keys, 128 or 136 units for 64 blocks, 34.6 us, 39 with a third round (a batch that is known to be that
// small from max_len is better off as PAR with three, 136 units in bf16 34.7 / 38.9).
template <int HD, int G, int RT, bool ALL>
__global__ __launch_bounds__((64 * AttnShape<HD, G, RT, ALL>::kWaves), (AttnShape<HD, G, RT, ALL>::kOcc)) void k_paged_attn(PAttnArgs a) {
    using S = AttnShape<HD, G, RT, ALL>;
    static_assert(S::kLds >= AttnShape<HD, G, RT, true>::kLds, "the tail's LDS");
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const unsigned xcd = blockIdx.x & 7u, block = blockIdx.x >> 3, blocks = gridDim.x >> 3;
    Items items;
    items.load(a, 0, 0);
    if constexpr (ALL) {
        attn_units<HD, G, RT, true>(a, lds, items, block, blocks, ~0u);
    } else {
        const unsigned wv = (unsigned)__builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), waves = blocks * S::kWaves;
        unsigned tail = ~0u, wide = 0;                // the rest's first unit, and the blocks whose waves take one each of it
        if (a.kv.n_seq <= kCounted) {                 // (more sequences are not worth their counting)
            unsigned n = (unsigned)__builtin_amdgcn_readlane(items.upto, 63);
            for (int b = 64; b < a.kv.n_seq; b += 64) {
                Items more;
                more.load(a, b, (int)n);
                n = (unsigned)__builtin_amdgcn_readlane(more.upto, 63);
            }
            n = n > xcd ? (n - xcd + 7u) / 8u * (unsigned)(a.kv.nkv * column_blocks(a, RT)) : 0u;
            const unsigned rest = n % waves;
            if (rest <= S::kTail * blocks) tail = n - rest;
            if (S::kTail == 3 && tail != ~0u && rest > 2 * blocks) wide = (rest - 2 * blocks + 1) / 2;
        }
        const unsigned first = tail + wide * S::kWaves;              // of the units that go as PAR
        attn_units<HD, G, RT, false>(a, lds, items, block * S::kWaves + wv, waves, block < wide ? first : tail);
        if (tail != ~0u && block >= wide) attn_units<HD, G, RT, true>(a, lds, items, first + block - wide, blocks - wide, ~0u);
    }
}

// The splits of a (row, head) joined. Split s belongs to class s % 16; a class is added up in split order, the classes as
// ((0 + 1) + (2 + 3)) and so on by fours, then the four fours in order: one order for both forms. X lanes hold 4 X dims of
// a head, so wave w's lanes have 64 / X of its classes 4 w .. 4 w + 3 side by side and X / 16 each in a row. X = 16: a block
// joins 64 dims with every class in lanes of its own, for few (row, head) pairs (24 heads of 126 splits: 4.8 us, 43 with one
// thread per dim). X = hd/4: a block joins a head, fewer blocks of more work for many (48 rows of 24 heads and 17
// splits: 20.8 us with X = 16). A thread's first eight splits are requested before the maximum is known.
template <int X>
__global__ __launch_bounds__(256) void k_paged_join(PAttnArgs a) {
    const int b = blockIdx.y / a.max_rows, i = blockIdx.y % a.max_rows;
    const SeqOf q = seq_of_all(a, b);
    if (i >= q.nr) return;
    constexpr int NA = X / 16, B = 8 / NA;            // classes of a lane, splits of each requested at a time
    const int hd = a.kv.hd, parts = hd / (4 * X);
    const int head = blockIdx.x / parts, d0 = (blockIdx.x % parts) * 4 * X;
    const int t = threadIdx.x, x = t % X, y = 4 * (t >> 6) + (t & 63) / X * NA;      // the lane's first class
    const int ns = splits_of(q);
    const bool done = ns == 1 && a.par;               // (finished by the split kernel: with weights, its sums are noted)
    if (done && !(a.w && d0 == 0)) return;
    const size_t row = (size_t)(q.first + i), at = row * a.nq + head;
    const float* pm = a.pm + at * a.ns;
    const float* pl = a.pl + at * a.ns;
    const f32x4* po = (const f32x4*)(a.po + at * a.ns * hd + d0) + x;
    __shared__ float s_red[4], s_l[4];
    __shared__ float s_sum[4][4 * X];
    f32x4 ov[B][NA];
    float mv[B][NA], lv[B][NA], M = -__builtin_huge_valf();
    auto batch = [&](int s0) __attribute__((always_inline)) {
#pragma unroll
        for (int u = 0; u < B; ++u)
#pragma unroll
            for (int k = 0; k < NA; ++k) {
                const int s = s0 + 16 * u + k, r = s < ns ? s : 0;
                const float m = pm[r], l = pl[r];
                const f32x4 o = po[(unsigned)(r * (hd >> 2))];
                mv[u][k] = s < ns ? m : -__builtin_huge_valf();
                lv[u][k] = s < ns ? l : 0.0f;
                ov[u][k] = s < ns ? o : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
    };
    batch(y);
#pragma unroll
    for (int u = 0; u < B; ++u)
#pragma unroll
        for (int k = 0; k < NA; ++k) M = fmaxf(M, mv[u][k]);
    for (int s = 16 * B + t; s < ns; s += 256) M = fmaxf(M, pm[s]);
    M = max_xor(M, 64);
    if ((t & 63) == 0) s_red[t >> 6] = M;
    __syncthreads();
    M = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
    float L[NA] = {};
    f32x4 o[NA] = {};
    for (int s0 = y;; ) {
#pragma unroll
        for (int u = 0; u < B; ++u)
#pragma unroll
            for (int k = 0; k < NA; ++k) {
                const float f = weight_of(mv[u][k], M);
                L[k] = __builtin_fmaf(lv[u][k], f, L[k]);
#pragma unroll
                for (int e = 0; e < 4; ++e) o[k][e] = __builtin_fmaf(ov[u][k][e], f, o[k][e]);
            }
        s0 += 16 * B;
        if (s0 - y >= ns) break;
        batch(s0);
    }
#pragma unroll
    for (int k = 1; k < NA; k *= 2)
#pragma unroll
        for (int n = 0; n < NA; n += 2 * k) {
            L[n] = L[n] + L[n + k];
            o[n] = o[n] + o[n + k];
        }
    if constexpr (X == 16) {
        L[0] = L[0] + xor16(L[0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][e] = o[0][e] + xor16(o[0][e]);
    }
    if constexpr (X <= 32) {
        L[0] = L[0] + xor32(L[0]);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[0][e] = o[0][e] + xor32(o[0][e]);
    }
    if ((t & 63) < X) {
        *(f32x4*)&s_sum[t >> 6][4 * x] = o[0];
        if (x == 0) s_l[t >> 6] = L[0];
    }
    __syncthreads();
    if (t >= 4 * X) return;
    const float l = ((s_l[0] + s_l[1]) + s_l[2]) + s_l[3];
    if (!done) put_out(a, hd, row, head, d0 + t, ((s_sum[0][t] + s_sum[1][t]) + s_sum[2][t]) + s_sum[3][t], l);
    if (a.w && d0 == 0 && t == 0) {
        a.fin[2 * at] = M;
        a.fin[2 * at + 1] = l;
    }
}

// The weight that each key of split sp got from row i, summed over the query heads in order: w[row][key] = sum over h of
// e^(x - M_h) / l_h, from the split kernel's e^(x - m) of its chunks: one factor per (head, chunk), made first. Keys up
// to the sequence's length are written (0 where the row does not see them, or the table does not reach: such chunks left
// nothing behind), nothing further. Bound by the 4 nq bytes per key that it reads.
constexpr int kWHeads = 64;
__global__ __launch_bounds__(256) void k_paged_weights(PAttnArgs a) {
    const int sp = blockIdx.x, b = blockIdx.y / a.max_rows, i = blockIdx.y % a.max_rows, t = threadIdx.x, key = sp * kPSplit + t;
    const SeqOf q = seq_of_all(a, b);
    if (i >= q.nr || sp * kPSplit >= min(q.raw, a.max_len)) return;
    const size_t at = (size_t)(q.first + i) * a.nq;
    const bool live = sp * kPSplit < q.len;           // (behind the table's end nothing was split)
    __shared__ float2 s_f[kWHeads][kChunks];          // a chunk's factor, and what is added where it has no weights
    float w = 0.0f;
    for (int h0 = 0; h0 < a.nq && live; h0 += kWHeads) {
        const int nh = min(kWHeads, a.nq - h0);
        __syncthreads();
        if (t < kChunks * nh) {
            const int h = t / kChunks, y = t % kChunks;
            const size_t r = at + h0 + h;
            const float m = a.pmc[(r * a.ns + sp) * kChunks + y], M = a.fin[2 * r], L = a.fin[2 * r + 1];
            // (a chunk without a key that is there has no weights written: its share is 0, or not a number with the row's sum)
            const float f = L == 0.0f ? 0.0f : weight_of(m, M) / L;
            s_f[h][y] = make_float2(f, m == -__builtin_huge_valf() || f != f ? f : 0.0f);
        }
        __syncthreads();
        const float* pp = a.pp + ((at + h0) * a.ns + sp) * kPSplit + t;
        const size_t step = (size_t)a.ns * kPSplit;
        for (int u0 = 0; u0 < nh; u0 += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = u0 + u < nh ? pp[(u0 + u) * step] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (u0 + u < nh) {
                    const float2 k = s_f[u0 + u][t / kChunk];
                    w = k.x == 0.0f || k.x != k.x ? w + k.y : __builtin_fmaf(v[u], k.x, w);
                }
        }
    }
    if (key < min(q.raw, a.max_len)) a.w[(size_t)(q.first + i) * a.w_stride + key] = key > q.raw - q.n + i || key >= q.len ? 0.0f : w;
}

struct WorkLayout { size_t po, pp, pm, pl, pmc, fin, total; };
static WorkLayout work_layout(int nq, int hd, int max_len, int nrows, int weights) {
    const size_t n = (size_t)nrows * nq, ns = ((size_t)max_len + kPSplit - 1) / kPSplit;
    WorkLayout w{};
    w.po = 0;
    w.pp = w.po + n * ns * hd;
    w.pm = w.pp + (weights ? n * ns * kPSplit : 0);
    w.pl = w.pm + n * ns;
    w.pmc = w.pl + n * ns;
    w.fin = w.pmc + (weights ? n * ns * kChunks : 0);
    w.total = w.fin + (weights ? 2 * n : 0);
    return w;
}

template <int HD, int G, int RT, bool ALL>
static int launch_split_form(const PAttnArgs& a, long long units, hipStream_t s) {
    using S = AttnShape<HD, G, RT, ALL>;
    Q27X_HIP((allow_lds<k_paged_attn<HD, G, RT, ALL>>(S::kLds)));
    // as many blocks as fit at once, or fewer units, in eights (one per XCD)
    const long long need = ALL ? units : (units + S::kWaves - 1) / S::kWaves;
    hipLaunchKernelGGL((k_paged_attn<HD, G, RT, ALL>), dim3((unsigned)(8 * (need < S::kBlocks ? need : S::kBlocks))), dim3(64 * S::kWaves), S::kLds, s, a);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}
template <int HD, int G, int RT>
static int launch_split_rt(PAttnArgs& a, hipStream_t s) {
    using S = AttnShape<HD, G, RT, false>;
    const long long units = ((long long)a.kv.n_seq * a.ns + 7) / 8 * a.kv.nkv * column_blocks(a, RT);      // of an XCD, if all sequences have max_len keys
    a.par = units <= S::kTail * S::kBlocks;
    return a.par ? launch_split_form<HD, G, RT, true>(a, units, s) : launch_split_form<HD, G, RT, false>(a, units, s);
}
template <int HD, int G>
static int launch_split(PAttnArgs& a, hipStream_t s) {
    return a.max_rows * (a.nq / a.kv.nkv) <= 16 ? launch_split_rt<HD, G, 1>(a, s) : launch_split_rt<HD, G, 2>(a, s);
}
static int launch_paged_attn(PAttnArgs& a, hipStream_t s) {
    int rc;
    switch (a.kv.hd * 100 + a.kv.G) {
        case 12800: rc = launch_split<128, 0>(a, s); break;
        case 12816: rc = launch_split<128, 16>(a, s); break;
        case 12832: rc = launch_split<128, 32>(a, s); break;
        case 12864: rc = launch_split<128, 64>(a, s); break;
        case 25600: rc = launch_split<256, 0>(a, s); break;
        case 25616: rc = launch_split<256, 16>(a, s); break;
        case 25632: rc = launch_split<256, 32>(a, s); break;
        default: rc = launch_split<256, 64>(a, s); break;
    }
    if (rc) return rc;
    const unsigned rows = (unsigned)(a.kv.n_seq * a.max_rows);
    if (a.ns > 1 || !a.par || a.w) {
        if ((long long)rows * a.nq < 2 * kCUs) hipLaunchKernelGGL(k_paged_join<16>, dim3((unsigned)(a.nq * (a.kv.hd / 64)), rows), dim3(256), 0, s, a);
        else if (a.kv.hd == 128) hipLaunchKernelGGL(k_paged_join<32>, dim3((unsigned)a.nq, rows), dim3(256), 0, s, a);
        else hipLaunchKernelGGL(k_paged_join<64>, dim3((unsigned)a.nq, rows), dim3(256), 0, s, a);
        Q27X_HIP(hipGetLastError());
    }
    if (a.w) {
        hipLaunchKernelGGL(k_paged_weights, dim3((unsigned)a.ns, rows), dim3(256), 0, s, a);
        Q27X_HIP(hipGetLastError());
    }
    return Q27X_OK;
}

}  // namespace q27x

using namespace q27x;
static bool paged_attn_shape(int nq, int hd, int max_len, int nrows) {
    return nq >= 1 && nq <= 1024 && (hd == 128 || hd == 256) && max_len >= 1 && max_len <= 0x7fffffff - kPSplit && nrows >= 1 && nrows <= 65535 * kMaxRows;
}
extern "C" size_t q27x_paged_attn_work_bytes(int nq, int hd, int max_len, int nrows, int weights) {
    return paged_attn_shape(nq, hd, max_len, nrows) ? work_layout(nq, hd, max_len, nrows, weights).total * 4 : 0;
}
extern "C" int q27x_paged_attn_rows(const uint16_t* qh, const uint16_t* qkv_gate, int qkv_stride, const q27x_paged_kv_t* kv,
                                    int nq, int gate, int max_len, int max_rows, int nrows, void* work, uint16_t* out,
                                    int8_t* xq, float* xs, float* w, int w_stride, q27x_stream_t s) {
    const char* who = "q27x_paged_attn_rows";
    PAttnArgs a{};
    if (int rc = paged_args(kv, who, &a.kv)) return rc;
    if (!qh || (gate && !qkv_gate) || !work || !out || (xq && !xs)) { set_error("%s: null argument", who); return Q27X_E_ARG; }
    if ((uintptr_t)work & 15) { set_error("%s: work must be 16-byte aligned", who); return Q27X_E_ARG; }
    if (!paged_attn_shape(nq, a.kv.hd, max_len, nrows) || nq % a.kv.nkv) {
        set_error("%s: unsupported shape (nq=%d nkv=%d hd=%d max_len=%d nrows=%d)", who, nq, a.kv.nkv, a.kv.hd, max_len, nrows);
        return Q27X_E_SHAPE;
    }
    if (max_rows < 1 || max_rows > kMaxRows) {
        set_error("%s: max_rows=%d: 1 to %d rows of a sequence", who, max_rows, kMaxRows);
        return Q27X_E_SHAPE;
    }
    if ((long long)a.kv.n_seq * max_rows > 65535) { set_error("%s: n_seq x max_rows = %lld: at most 65535", who, (long long)a.kv.n_seq * max_rows); return Q27X_E_RANGE; }
    if (qkv_stride < 0 || (w && w_stride < max_len)) { set_error("%s: bad strides (qkv_stride=%d w_stride=%d max_len=%d)", who, qkv_stride, w_stride, max_len); return Q27X_E_ARG; }
    a.qh = qh; a.qkv = qkv_gate; a.qkv_stride = qkv_stride; a.nq = nq; a.gate = gate ? 1 : 0;
    a.max_len = max_len; a.max_rows = max_rows; a.nrows = nrows; a.ns = (max_len + kPSplit - 1) / kPSplit;
    a.sl2e = (float)((1.0 / sqrt((double)a.kv.hd)) * 1.4426950408889634);
    const WorkLayout wl = work_layout(nq, a.kv.hd, max_len, nrows, w != nullptr);
    float* p = (float*)work;
    a.po = p + wl.po; a.pm = p + wl.pm; a.pl = p + wl.pl;
    if (w) { a.pp = p + wl.pp; a.pmc = p + wl.pmc; a.fin = p + wl.fin; }
    a.out = out; a.xq = xq; a.xs = xs; a.w = w; a.w_stride = w_stride;
    return launch_paged_attn(a, (hipStream_t)s);
}

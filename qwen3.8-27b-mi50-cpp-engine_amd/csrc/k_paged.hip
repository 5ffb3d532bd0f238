// k_paged.hip -- one paged key/value cache for many sequences: preparing their new rows (norm, rotary positions of
// several axes, append) and attention of those rows over the pages.
#include <math.h>

#include <type_traits>

#include "q27x_paged.h"

namespace q27x {

int paged_args(const q27x_paged_kv_t* kv, const char* who, PagedArgs* out) {
    if (!kv || !kv->k || !kv->v || !kv->table || !kv->lens) { set_error("%s: null cache, pool, table or lens", who); return Q27X_E_ARG; }
    if (kv->kv_group != 0 && (!kv->ks || !kv->vs)) { set_error("%s: int8 pages need scales", who); return Q27X_E_ARG; }
    if (((uintptr_t)kv->k | (uintptr_t)kv->v) & 15) { set_error("%s: pages must be 16-byte aligned", who); return Q27X_E_ARG; }
    if ((kv->hd != 128 && kv->hd != 256) || kv->nkv < 1 || kv->nkv > 1024 ||
        (kv->kv_group != 0 && kv->kv_group != 16 && kv->kv_group != 32 && kv->kv_group != 64)) {
        set_error("%s: unsupported cache (nkv=%d hd=%d kv_group=%d: hd 128 or 256, kv_group 16, 32, 64 or 0 for bf16)", who,
                  kv->nkv, kv->hd, kv->kv_group);
        return Q27X_E_SHAPE;
    }
    if (kv->page < 1 || (kv->page & (kv->page - 1)) || kv->n_pages < 1 || kv->table_stride < 1 || kv->n_seq < 1 ||
        (kv->page_stride != 0 && kv->page_stride < kv->page)) {
        set_error("%s: bad pages (page=%d, a power of two; page_stride=%d, 0 or at least page; n_pages=%d table_stride=%d n_seq=%d)",
                  who, kv->page, kv->page_stride, kv->n_pages, kv->table_stride, kv->n_seq);
        return Q27X_E_ARG;
    }
    const int stride = kv->page_stride ? kv->page_stride : kv->page;
    if ((long long)kv->n_pages * stride > 0x7fffffffLL || (long long)kv->table_stride * kv->page > 0x7fffffffLL || kv->n_seq > 65535) {
        set_error("%s: a pool or table of more than 2^31 - 1 positions, or more than 65535 sequences", who);
        return Q27X_E_RANGE;
    }
    PagedArgs a{};
    a.k = kv->k; a.v = kv->v; a.ks = kv->ks; a.vs = kv->vs; a.G = kv->kv_group; a.nkv = kv->nkv; a.hd = kv->hd;
    a.n_pages = kv->n_pages; a.shift = __builtin_ctz((unsigned)kv->page); a.stride = stride;
    a.table = kv->table; a.table_stride = kv->table_stride; a.lens = kv->lens; a.row_start = kv->row_start; a.n_seq = kv->n_seq;
    *out = a;
    return Q27X_OK;
}

// ---------------------------------------------------------------- prep
// Per head of a row: y = x / sqrt(mean x^2 + eps) (1 + w), then pair i of the first rot dims (dims i and i + rot/2)
// turned by the angle of position pos[axis of i][row]: (a, b) -> (a c - b s, b c + a s). Keys (normed, turned) and values
// (as they are) go to the row's position in the pages, int8 codes with a scale per group (s = max|v| / 127, code =
// rint(v / s)) or bf16.
//
// Block = (row, 16 heads of q | k | v), 16 lanes a head: a lane holds HD/16 neighbouring dims, so a group's maximum and the
// head's sum of squares are a few DPP steps and four heads share a wave's root and division. The row's angles are read
// once per block into LDS; the partner dims of a turn come through LDS too, so rot can be any even number.
struct PrepArgs {
    const uint16_t* qkv; int qkv_stride;
    const uint16_t* q_norm_w; const uint16_t* k_norm_w;
    const float* rope_cos; const float* rope_sin; int rot, n_pos;
    const int32_t* pos; int pos_stride, n_axes;
    uint32_t axes[8];               // the axis of pair i in bits 2 (i % 16) of word i / 16
    uint16_t* qh; int nq, gate; float eps; int nrows;
    PagedArgs kv;
};

// E bf16 values from p (aligned to 2 bytes)
template <int E>
__device__ __forceinline__ void ld_bf16(const uint16_t* p, float (&v)[E]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        const u32x4 x = *(const u32x4*)(p + 8 * i);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[8 * i + 2 * j] = __uint_as_float(x[j] << 16);
            v[8 * i + 2 * j + 1] = __uint_as_float(x[j] & 0xFFFF0000u);
        }
    }
}
template <int E>
__device__ __forceinline__ void st_bf16(uint16_t* p, const float (&v)[E]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        u32x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = (uint32_t)f2bf(v[8 * i + 2 * j]) | ((uint32_t)f2bf(v[8 * i + 2 * j + 1]) << 16);
        *(u32x4*)(p + 8 * i) = x;
    }
}
// sum over the 16 lanes of a DPP row, in every lane of it
__device__ __forceinline__ float sum16(float x) {
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0xB1, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x4E, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x141, 0xF, 0xF, false));
    x += __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(x), 0x140, 0xF, 0xF, false));
    return x;
}
// The sequence of row r, or -1: the count of sequences that end at or before it (row_start does not decrease), by every
// wave of the block for itself, 64 sequences a step.
__device__ __forceinline__ int seq_of_row(const PagedArgs& a, int r) {
    if (!a.row_start) return r < a.n_seq ? r : -1;
    const int l = threadIdx.x & 63;
    int b = 0;
    for (int j = 0; j < a.n_seq; j += 64) {
        const bool ends = j + l < a.n_seq && a.row_start[j + l + 1] <= r;
        b += __popcll(__ballot(ends));
    }
    return b < a.n_seq && a.row_start[b] <= r && a.row_start[b] >= 0 && r < a.row_start[b + 1] ? b : -1;
}

template <int HD, int G>
__device__ __forceinline__ void st_kv(const PagedArgs& a, void* pool, float* scales, size_t slot, int head, int c,
                                      const float (&v)[HD / 16]) {
    constexpr int E = HD / 16;
    const size_t at = slot * ((size_t)a.nkv * HD) + (size_t)head * HD + E * c;
    if constexpr (G == 0) {
        st_bf16<E>((uint16_t*)pool + at, v);
    } else {
        float mx = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) mx = fmaxf(mx, fabsf(v[e]));
        mx = max_xor(mx, G / E);
        const float sc = mx * (1.0f / 127.0f);
        const float inv = (sc > 0.0f) ? (1.0f / sc) : 0.0f;
        uint32_t w[E / 4];
#pragma unroll
        for (int e = 0; e < E; e += 4) w[e / 4] = pack4(qcode(v[e], inv), qcode(v[e + 1], inv), qcode(v[e + 2], inv), qcode(v[e + 3], inv));
        int8_t* p = (int8_t*)pool + at;
        if constexpr (E == 16) *(uint4*)p = make_uint4(w[0], w[1], w[2], w[3]);
        else *(uint2*)p = make_uint2(w[0], w[1]);
        if ((E * c) % G == 0) scales[at / G] = sc;
    }
}

template <int HD, int G>
__global__ __launch_bounds__(256) void k_paged_prep(PrepArgs a) {
    constexpr int E = HD / 16;
    const int r = blockIdx.x, t = threadIdx.x, c = t & 15, slotw = t >> 4;
    const int half = a.rot >> 1;
    __shared__ float cs[2][HD / 2];
    __shared__ float ex[16][HD];
    // the row's angles: thread t < rot takes the cosine (t < half) or sine of pair t % half
    if (t < a.rot) {
        const int f = t < half ? t : t - half;
        const int axis = (a.axes[f >> 4] >> (2 * (f & 15))) & 3;
        int p = a.pos[(size_t)axis * a.pos_stride + r];
        p = p < 0 ? 0 : (p >= a.n_pos ? a.n_pos - 1 : p);
        cs[t >= half][f] = (t < half ? a.rope_cos : a.rope_sin)[(size_t)p * half + f];
    }
    const int b = seq_of_row(a.kv, r);
    if (b < 0) return;                               // (the same in every wave: a row behind the last sequence)
    const int u = blockIdx.y * 16 + slotw;           // q heads, then k, then v
    const bool isq = u < a.nq, isk = !isq && u < a.nq + a.kv.nkv, isv = !isq && !isk && u < a.nq + 2 * a.kv.nkv;
    const int head = isq ? u : isk ? u - a.nq : u - a.nq - a.kv.nkv;
    const int qw = a.gate ? 2 * HD : HD;
    float y[E];
    if (isq || isk || isv) {
        const uint16_t* src = a.qkv + (size_t)r * a.qkv_stride +
                              (isq ? (size_t)head * qw : (size_t)a.nq * qw + ((size_t)(isv ? a.kv.nkv : 0) + head) * HD) + E * c;
        ld_bf16<E>(src, y);
    }
    if (isq || isk) {
        float w[E];
        ld_bf16<E>((isq ? a.q_norm_w : a.k_norm_w) + E * c, w);
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = __builtin_fmaf(y[e], y[e], ss);
        ss = sum16(ss);
        const float inv = rsqrt_cr(ss * (1.0f / (float)HD) + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = y[e] * inv * (1.0f + w[e]);
#pragma unroll
        for (int e = 0; e < E; ++e) ex[slotw][E * c + e] = y[e];
    }
    __syncthreads();
    if ((isq || isk) && E * c < a.rot) {
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = E * c + e;
            if (d >= a.rot) break;
            const int f = d < half ? d : d - half;
            const float o = ex[slotw][d < half ? d + half : d - half];
            y[e] = d < half ? y[e] * cs[0][f] - o * cs[1][f] : y[e] * cs[0][f] + o * cs[1][f];
        }
    }
    if (isq) {
        st_bf16<E>(a.qh + ((size_t)r * a.nq + head) * HD + E * c, y);
    } else if (isk || isv) {
        int first, n;
        paged_rows(a.kv, b, first, n);
        const int slot = paged_slot(a.kv, b, a.kv.lens[b] - n + (r - first));
        if (slot < 0) return;
        st_kv<HD, G>(a.kv, isk ? a.kv.k : a.kv.v, isk ? a.kv.ks : a.kv.vs, (size_t)slot, head, c, y);
    }
}

static int launch_prep(const PrepArgs& a, hipStream_t s) {
    const dim3 grid((unsigned)a.nrows, (unsigned)((a.nq + 2 * a.kv.nkv + 15) / 16));
#define Q27X_PP(H, GG) hipLaunchKernelGGL((k_paged_prep<H, GG>), grid, dim3(256), 0, s, a)
    switch (a.kv.hd * 100 + a.kv.G) {
        case 12800: Q27X_PP(128, 0); break;
        case 12816: Q27X_PP(128, 16); break;
        case 12832: Q27X_PP(128, 32); break;
        case 12864: Q27X_PP(128, 64); break;
        case 25600: Q27X_PP(256, 0); break;
        case 25616: Q27X_PP(256, 16); break;
        case 25632: Q27X_PP(256, 32); break;
        default: Q27X_PP(256, 64); break;
    }
#undef Q27X_PP
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}

// ---------------------------------------------------------------- attention
// Row i of a sequence's n new rows sees keys 0 .. len - n + i of its cache. For every query head, with x = q.k / sqrt(hd):
// out = sum e^(x - M) v / sum e^(x - M), M = max x, times sigmoid(gate); a row that sees nothing gets zeros.
//
// Keys are cut into fixed splits of kPSplit, a split into four chunks of 64, so a row's result depends on its own keys
// alone, whatever else is in the batch. Block = (split, kv head, up to 16 RT columns: the pairs of a row and a query head
// of that kv head), a wave = one chunk. A wave has its 64 keys' scores before it needs their maximum, so there is no
// running rescale: one maximum, one exponential, then P.V; the block joins its four chunks in order in LDS and writes
// the split's (m, l, o), which k_paged_combine joins in split order (a sequence of one split is finished here).
//
// Scores on v_mfma_f32_16x16x32_bf16 as K Q^T: lane (c, g) = (lane & 15, lane >> 4) holds dims 32 i + 8 g .. + 7 of key
// c, and gets keys 4 g .. 4 g + 3 of column c. Codes and queries are bf16 exactly; the fp32 sum of each scale group
// is multiplied by the key's scale afterwards, so scores carry no rounding but fp32's. One dword a lane holds a tile's
// scales (key 4 g + c % 4, group c / 4), handed to the row's lanes by DPP.
// P.V as V^T P^T: the columns' weights are already where the second product wants them (slots 8 g .. of column c: keys
// 4 g .. of two tiles), and lane (c, g) loads dims c HD/16 .. of keys 4 g .. + 3, so V needs no transpose: byte t of the
// eight keys is row c of dim tile t. A value is code x scale rounded to fp16, scales first brought to [1, 2) by the power
// of two of the group's largest (undone in fp32), weights (at most 1) are rounded to fp16: 2^-11 each, below the bf16
// output's 2^-8. bf16 pages: values exact, weights as two bf16 terms (2^-16).
constexpr int kPSplit = 256;
constexpr int kCUs = 256;             // compute units of an MI355X

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

struct PAttnArgs {
    const uint16_t* qh; const uint16_t* qkv; int qkv_stride;
    PagedArgs kv;
    int nq, gate, max_len, max_rows, nrows, ns;      // ns: splits of max_len
    float sl2e;                                      // log2(e) / sqrt(hd)
    float* po; float* pm; float* pl;                 // splits' outputs [row][head][ns][hd], maxima and sums [row][head][ns]
    float* pp; float* pm64; float* fin;              // with w: e^(x - m) [row][head][ns 256], chunk maxima [row][head][ns 4], (M, 1/l)
    uint16_t* out; int8_t* xq; float* xs;
    float* w; int w_stride;
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

// blocks of a compute unit, and the registers that leaves a lane (512 / it)
template <int HD, int G, int RT>
struct AttnOcc { static constexpr int n = HD == 128 ? (RT == 1 && G ? 4 : 2) : RT == 1 ? 2 : 1; };

template <int HD, int G, int RT>
__global__ __launch_bounds__(256, (AttnOcc<HD, G, RT>::n)) void k_paged_attn(PAttnArgs a) {
    constexpr int E = HD / 16;                       // dims of V a lane holds
    constexpr int NM = HD / 32;                      // products of a score tile
    constexpr int NG = G ? HD / G : 1;               // scale groups of a head
    constexpr int NS = NG > 4 ? NG / 4 : 1;          // scale registers of a tile
    constexpr int VW = G ? E / 4 : E / 2;            // registers of a key's V dims
    constexpr int CG = 8;                            // columns joined at a time
    constexpr float kNone = -__builtin_huge_valf();
    const int wv = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
    const PagedArgs& kv = a.kv;
    const int grp = a.nq / kv.nkv;
    // Blocks j and j + 8 run on the same XCD: XCD x takes the pairs x, x + 8, .. with all their kv heads, which share the
    // lines of the scales; its blocks take its (pair, head, columns) units in turn.
    const int ncb = (a.max_rows * grp + 16 * RT - 1) / (16 * RT), per = kv.nkv * ncb;
    __shared__ uint64_t s_off[4][64];
    __shared__ float s_m[4][16 * RT], s_l[4][16 * RT];
    __shared__ float s_o[4][CG][HD + 4];
    Items items;
    items.load(a, 0, 0);
    const uint64_t width = (uint64_t)kv.nkv * HD;    // elements of a position
    for (unsigned unit = blockIdx.x >> 3;; unit += gridDim.x >> 3) {
    const int sub = (int)(unit % (unsigned)per);
    int b, sp;
    if (!items.find(a, (int)(unit / (unsigned)per * 8u + (blockIdx.x & 7u)), b, sp)) return;
    const int kvh = sub % kv.nkv, cb = sub / kv.nkv;
    const SeqOf q = seq_of(a, b);
    const int ncol = min(q.nr * grp - cb * 16 * RT, 16 * RT);    // this unit's columns
    if (ncol <= 0) continue;
    const int k0 = sp * kPSplit + 64 * wv;
    int t = threadIdx.x;                              // (opaque: what follows from it is not kept over the loop, which spills)
    asm volatile("" : "+v"(t));
    const int l = t & 63, c = l & 15, g = l >> 4;
    __syncthreads();                                  // the unit before is read out of LDS

    // this wave's keys: lane l looks key k0 + l up
    const int my = k0 + l < q.len ? paged_slot(kv, b, k0 + l) : -1;
    const uint64_t valid = __ballot(my >= 0);
    s_off[wv][l] = my < 0 ? 0 : (uint64_t)(unsigned)my * width;     // (a key that is not there reads position 0 of the pool)
    __builtin_amdgcn_wave_barrier();

    float m[RT], lsum[RT];
    f32x4 o[RT][E];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = kNone;
        lsum[rt] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) o[rt][e] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    if (valid) {
        const uint64_t hoff = (uint64_t)kvh * HD;
        u32x4 kx[4][NM];                              // K: dims 32 i + 8 g .. of key 16 ti + c (int8: the low two words)
        uint32_t vx[4][4][VW];                        // V: dims E c .. of key 16 ti + 4 g + j
        float ksc[4][NS], vsc[4][NS];                 // scales of key 16 ti + 4 g + c % 4
#pragma unroll
        for (int ti = 0; ti < 4; ++ti) {
            const uint64_t at = s_off[wv][16 * ti + c] + hoff;
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                if constexpr (G == 0) {
                    kx[ti][i] = *(const u32x4*)((const uint16_t*)kv.k + at + 32 * i + 8 * g);
                } else {
                    const uint2 x = *(const uint2*)((const int8_t*)kv.k + at + 32 * i + 8 * g);
                    kx[ti][i] = u32x4{x.x, x.y, 0, 0};
                }
            }
            if constexpr (G != 0) {
                const uint64_t srow = (s_off[wv][16 * ti + 4 * g + (c & 3)] + hoff) / G;
#pragma unroll
                for (int u = 0; u < NS; ++u) {
                    ksc[ti][u] = kv.ks[srow + (NG >= 4 ? (c >> 2) + 4 * u : (c >> 2) % NG)];     // groups c / 4 + 4 u
                    vsc[ti][u] = kv.vs[srow + (NG >= 4 ? (c >> 2) * NS + u : (c >> 2) * NG / 4)]; // the quad's dims' groups
                }
            }
        }
        typedef uint32_t vvec __attribute__((ext_vector_type(VW)));
        auto v_at = [&](int k) __attribute__((always_inline)) {
            const uint64_t at = s_off[wv][k] + hoff + E * c;
            return *(const vvec*)(G == 0 ? (const char*)kv.v + 2 * at : (const char*)kv.v + at);
        };
        auto load_v = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int ti = 0; ti < 4; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const vvec x = v_at(16 * ti + 4 * g + j);
#pragma unroll
                    for (int u = 0; u < VW; ++u) vx[ti][j][u] = x[u];
                }
        };
        // (256-wide bf16 rows: K and V together are all of a lane's registers)
        constexpr bool kLateV = G == 0 && HD == 256;
        if constexpr (!kLateV) load_v();
        // the columns' queries: dims 32 i + 8 g .. + 7 of column c
        u32x4 qx[RT][NM];
        int last[RT];                                 // the last key that the column sees
        size_t prow[RT];                              // its (row, head)
        bool on[RT];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            on[rt] = 16 * rt + c < ncol;
            const int col = on[rt] ? cb * 16 * RT + 16 * rt + c : 0;
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
        // scores
        const f32x4 zero = {0.0f, 0.0f, 0.0f, 0.0f};
        float s[RT][4][4];
#pragma unroll
        for (int ti = 0; ti < 4; ++ti) {
            __builtin_amdgcn_sched_barrier(0);        // (tiles widened ahead of their products spill)
            uint32_t low = g < 2 ? ~0u : 0u;           // (opaque: masked queries are not worth registers of their own)
            if constexpr (G == 16) asm volatile("" : "+v"(low));
            f32x4 acc[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) {
                acc[rt] = zero;
#pragma unroll
                for (int i = 0; i < 4; ++i) s[rt][ti][i] = 0.0f;
            }
#pragma unroll
            for (int i = 0; i < NM; ++i) {
                u32x4 kb;
                if constexpr (G == 0) {
                    kb = kx[ti][i];
                } else {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t x = kx[ti][i][h];
                        kb[2 * h] = pack_bf(byte_f(x, 0), byte_f(x, 1));
                        kb[2 * h + 1] = pack_bf(byte_f(x, 2), byte_f(x, 3));
                    }
                }
                const bf16x8 ka = __builtin_bit_cast(bf16x8, kb);
                // a group of 16: two products, the other half of the lanes' queries zeroed
                constexpr int NH = G == 16 ? 2 : 1;
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    if constexpr (NH == 2) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) {
                        const u32x4 qm = NH == 1 ? qx[rt][i] : qx[rt][i] & (h ? ~low : low);
                        acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka, __builtin_bit_cast(bf16x8, qm), acc[rt], 0, 0, 0);
                    }
                    if constexpr (G != 0) {
                        const int done = 32 * i + (NH == 2 ? 16 * (h + 1) : 32);
                        if (done % G == 0) {          // the group is whole: times the keys' scales
                            const int gr = done / G - 1;
#pragma unroll
                            for (int rt = 0; rt < RT; ++rt) {
#pragma unroll
                                for (int j = 0; j < 4; ++j)
                                    s[rt][ti][j] = __builtin_fmaf(acc[rt][j], row_bcast(ksc[ti][gr >> 2], 4 * (gr & 3) + j), s[rt][ti][j]);
                                acc[rt] = zero;
                            }
                        }
                    }
                }
            }
            if constexpr (G == 0) {
#pragma unroll
                for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[rt][ti][j] = acc[rt][j];
            }
        }
        if constexpr (kLateV) load_v();
        // weights: e^(x - m) of the 64 keys, those that the row does not see 0
        const bool full = valid == ~0ull && k0 + 63 <= q.raw - q.n;
        uint32_t pw[RT][2][4], plo[RT][2][G == 0 ? 4 : 1];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            if (!full) {
                const int see = last[rt] - k0 - 4 * g;    // keys 16 ti + j of this lane up to here
#pragma unroll
                for (int ti = 0; ti < 4; ++ti) {
                    const uint32_t there = (uint32_t)(valid >> (16 * ti)) >> (4 * g);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        s[rt][ti][j] = (16 * ti + j <= see && ((there >> j) & 1)) ? s[rt][ti][j] : kNone;
                }
            }
            float mx = kNone;
#pragma unroll
            for (int ti = 0; ti < 4; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[rt][ti][j] *= a.sl2e;
                    mx = fmaxf(mx, s[rt][ti][j]);
                }
            mx = max_cols(mx);
            m[rt] = mx;
            const float base = mx == kNone ? 0.0f : mx;
            float sum = 0.0f;
#pragma unroll
            for (int ti = 0; ti < 4; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[rt][ti][j] = __builtin_amdgcn_exp2f(s[rt][ti][j] - base);
                    sum += s[rt][ti][j];
                }
            lsum[rt] = sum_cols(sum);
            if (a.w && on[rt]) {
                float* pp = a.pp + (prow[rt] * a.ns + sp) * kPSplit + 64 * wv + 4 * g;
#pragma unroll
                for (int ti = 0; ti < 4; ++ti) *(f32x4*)(pp + 16 * ti) = f32x4{s[rt][ti][0], s[rt][ti][1], s[rt][ti][2], s[rt][ti][3]};
            }
#pragma unroll
            for (int ti = 0; ti < 4; ++ti)
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
        // The keys whose values enter: keys that are not there read something else, maybe not finite. Keys that only
        // later rows see enter too (their weight is 0 in the rows before), unless they hold something that is not finite:
        // those enter one by one, in the columns that see them.
        uint64_t enter = valid, later = 0;
        if (q.raw - q.n < k0 + 63) {
            const int from = q.raw - q.n + 1 - k0;    // the first key that row 0 does not see
            later = from <= 0 ? valid : valid & ~((1ull << from) - 1);
        }
        if (later) {
            bool odd = false;
#pragma unroll
            for (int ti = 0; ti < 4; ++ti) {
                if constexpr (G != 0) {
                    if ((later >> (16 * ti + 4 * g + (c & 3))) & 1) {
#pragma unroll
                        for (int u = 0; u < NS; ++u) odd |= !finite_f(vsc[ti][u]);
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if ((later >> (16 * ti + 4 * g + j)) & 1) {
#pragma unroll
                            for (int u = 0; u < VW; ++u)
                                odd |= (vx[ti][j][u] & 0x7F80u) == 0x7F80u || (vx[ti][j][u] & 0x7F800000u) == 0x7F800000u;
                        }
                }
            }
            if (__ballot(odd)) enter &= ~later;
            else later = 0;
        }
        // the power of two that brings the largest finite scale of each of the quad's groups to [1, 2), and its inverse
        // for the output rows 4 g + j (the dims of quad g)
        float fac[NS], back[NS];
        if constexpr (G != 0) {
#pragma unroll
            for (int u = 0; u < NS; ++u) {
                float mx = 0.0f;
#pragma unroll
                for (int ti = 0; ti < 4; ++ti) {
                    const bool in = (valid >> (16 * ti + 4 * g + (c & 3))) & 1;
                    mx = fmaxf(mx, in && finite_f(vsc[ti][u]) ? fabsf(vsc[ti][u]) : 0.0f);
                }
                mx = max_cols(max_quad(mx));
                int ex = (int)(__float_as_uint(mx) >> 23);
                ex = ex < 1 ? 1 : ex > 253 ? 253 : ex;
                fac[u] = __uint_as_float((uint32_t)(254 - ex) << 23);
                back[u] = __shfl(__uint_as_float((uint32_t)ex << 23), (l & 48) + 4 * g, 64);
            }
        }
        // V' of the given keys (others 0), both 32-key halves of a dim tile, into one product chain per column tile: added to
        // o, or (single) to the columns that see the key
        // the scale of this lane's dims at key j of the quad's four
        auto key_scale = [&](const float (&v)[NS], int j) __attribute__((always_inline)) {
            float x = quad_bcast(v[0], j);
#pragma unroll
            for (int u = 1; u < NS; ++u) {
                const float y = quad_bcast(v[u], j);  // (in every lane: a lane reads its neighbours')
                x = (c & 3) >= u * (4 / NS) ? y : x;
            }
            return x;
        };
        auto pv = [&](uint64_t keys, auto single, int key) __attribute__((always_inline)) {
            float vs[4][NS];
            uint32_t keep[4] = {15, 15, 15, 15};
            if constexpr (G != 0) {
#pragma unroll
                for (int ti = 0; ti < 4; ++ti)
#pragma unroll
                    for (int u = 0; u < NS; ++u) vs[ti][u] = vsc[ti][u] * fac[u];
            }
            if (keys != ~0ull) {
#pragma unroll
                for (int ti = 0; ti < 4; ++ti) {
                    keep[ti] = (uint32_t)(keys >> (16 * ti)) >> (4 * g);
                    if constexpr (G != 0) {
#pragma unroll
                        for (int u = 0; u < NS; ++u) vs[ti][u] = (keep[ti] >> (c & 3)) & 1 ? vs[ti][u] : 0.0f;
                    }
                }
                if constexpr (G == 0) {
#pragma unroll
                    for (int ti = 0; ti < 4; ++ti)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
#pragma unroll
                            for (int u = 0; u < VW; ++u) vx[ti][j][u] = (keep[ti] >> j) & 1 ? vx[ti][j][u] : 0u;
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                __builtin_amdgcn_sched_barrier(0);
                f32x4 acc[RT];
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) acc[rt] = single ? zero : o[rt][e];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
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
                            acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, va), __builtin_bit_cast(f16x8, pb), acc[rt], 0, 0, 0);
                        } else {
                            const u32x4 pl = {plo[rt][u][0], plo[rt][u][1], plo[rt][u][2], plo[rt][u][3]};
                            acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, pb), acc[rt], 0, 0, 0);
                            acc[rt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, va), __builtin_bit_cast(bf16x8, pl), acc[rt], 0, 0, 0);
                        }
                    }
                }
#pragma unroll
                for (int rt = 0; rt < RT; ++rt) {
                    if (!single) o[rt][e] = acc[rt];
                    else if (key <= last[rt]) o[rt][e] = o[rt][e] + acc[rt];
                }
            }
        };
        pv(enter, std::false_type{}, 0);
        while (later) {
            const int k = __builtin_ctzll(later);
            later &= later - 1;
            const vvec x = v_at(k);
#pragma unroll
            for (int ti = 0; ti < 4; ++ti)
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int u = 0; u < VW; ++u) vx[ti][j][u] = k == 16 * ti + 4 * g + j ? x[u] : 0u;
            pv(1ull << k, std::true_type{}, k0 + k);
        }
        if constexpr (G != 0) {
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[rt][e][j] = o[rt][e][j] * back[j * NS / 4];
        }
    }
    // the four chunks joined in order
    if (g == 0) {
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) { s_m[wv][16 * rt + c] = m[rt]; s_l[wv][16 * rt + c] = lsum[rt]; }
    }
    const bool whole = q.len <= kPSplit;              // the sequence has no other split
#pragma unroll
    for (int cg = 0; cg < 2 * RT; ++cg) {
        if (cg * CG < ncol) {                         // (the same in every wave)
            if (cg) __syncthreads();
            if ((c >> 3) == (cg & 1)) {
#pragma unroll
                for (int j = 0; j < 4; ++j)
#pragma unroll
                    for (int e = 0; e < E; e += 4)
                        *(f32x4*)&s_o[wv][c & 7][E * (4 * g + j) + e] =
                            f32x4{o[cg >> 1][e][j], o[cg >> 1][e + 1][j], o[cg >> 1][e + 2][j], o[cg >> 1][e + 3][j]};
            }
            __syncthreads();
            const int nc = min(CG, ncol - cg * CG);
            for (int i = t; i < nc * HD; i += 256) {
                const int cc = i / HD, d = i % HD, col = cg * CG + cc;
                const float M = fmaxf(fmaxf(s_m[0][col], s_m[1][col]), fmaxf(s_m[2][col], s_m[3][col]));
                float L = 0.0f, v = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = weight_of(s_m[w][col], M);
                    L = __builtin_fmaf(s_l[w][col], f, L);
                    v = __builtin_fmaf(s_o[w][cc][d], f, v);
                }
                const int gc = cb * 16 * RT + col;
                const size_t row = (size_t)(q.first + gc / grp);
                const int head = kvh * grp + gc % grp;
                const size_t at = row * a.nq + head;
                if (whole) put_out(a, HD, row, head, d, v, L);
                else a.po[(at * a.ns + sp) * HD + d] = v;
                if (d == 0) {
                    a.pm[at * a.ns + sp] = M;
                    a.pl[at * a.ns + sp] = L;
                }
                if (a.w && d < 4) a.pm64[(at * a.ns + sp) * 4 + d] = s_m[d][col];
            }
        }
    }
    }
}

// The splits of a (row, head) joined. Split s belongs to class s % 16; a class is added up in split order, the classes as
// ((0 + 1) + (2 + 3)) and so on by fours, then the four fours in order: one order for both forms. X lanes hold 4 X dims of
// a head, so wave w's lanes have 64 / X of its classes 4 w .. 4 w + 3 side by side and X / 16 each in a row. X = 16: a block
// joins 64 dims with every class in lanes of its own, for few (row, head) pairs (24 heads of 126 splits: 4.8 us, 43 with one
// thread per dim). X = hd/4: a block joins a head, fewer blocks of more work for many (48 rows of 24 heads and 17
// splits: 20.8 us with X = 16). A thread's first eight splits are requested before the maximum is known.
// A sequence of one split was finished above: with weights, only its maximum and sum are noted.
template <int X>
__global__ __launch_bounds__(256) void k_paged_combine(PAttnArgs a) {
    constexpr int NA = X / 16, B = 8 / NA;            // classes of a lane, splits of each requested at a time
    const int hd = a.kv.hd, parts = hd / (4 * X);
    const int head = blockIdx.x / parts, d0 = (blockIdx.x % parts) * 4 * X, b = blockIdx.y / a.max_rows, i = blockIdx.y % a.max_rows;
    const int t = threadIdx.x, x = t % X, y = 4 * (t >> 6) + (t & 63) / X * NA;      // the lane's first class
    const SeqOf q = seq_of(a, b);
    if (i >= q.nr) return;
    const int ns = splits_of(q);
    if (ns == 1 && !(a.w && d0 == 0)) return;
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
                const int s = s0 + 16 * u + k;
                mv[u][k] = s < ns ? pm[s] : -__builtin_huge_valf();
                lv[u][k] = s < ns ? pl[s] : 0.0f;
                ov[u][k] = s < ns && ns > 1 ? po[(size_t)s * (hd >> 2)] : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
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
    if (ns > 1) put_out(a, hd, row, head, d0 + t, ((s_sum[0][t] + s_sum[1][t]) + s_sum[2][t]) + s_sum[3][t], l);
    if (a.w && d0 == 0 && t == 0) {
        a.fin[2 * at] = M;
        a.fin[2 * at + 1] = l;
    }
}

// The weight that each key got from a row, summed over the query heads in order: w[row][key] = sum over h of
// e^(x - M_h) / l_h, from the split kernel's e^(x - m) of 64-key chunks: one factor per (head, chunk), made first. Keys
// up to the sequence's length are written (0 where the row does not see them), nothing behind. Bound by the 4 nq bytes
// per key that it reads.
constexpr int kWHeads = 64;
__global__ __launch_bounds__(256) void k_paged_weights(PAttnArgs a) {
    const int sp = blockIdx.x, b = blockIdx.y / a.max_rows, i = blockIdx.y % a.max_rows, t = threadIdx.x;
    const SeqOf q = seq_of(a, b);
    const int key = sp * kPSplit + t;
    if (i >= q.nr || sp * kPSplit >= min(q.raw, a.max_len)) return;
    const size_t at = (size_t)(q.first + i) * a.nq;
    const bool live = sp * kPSplit < q.len;           // (behind the table's end nothing was split)
    __shared__ float2 s_f[kWHeads][4];                // a chunk's factor, and what its sums are multiplied by where it has none
    float w = 0.0f;
    for (int h0 = 0; h0 < a.nq && live; h0 += kWHeads) {
        const int nh = min(kWHeads, a.nq - h0);
        __syncthreads();
        if (t < 4 * nh) {
            const size_t r = at + h0 + (t >> 2);
            const float m = a.pm64[(r * a.ns + sp) * 4 + (t & 3)], M = a.fin[2 * r], L = a.fin[2 * r + 1];
            // (a chunk without a key that is there has no weights written: its share is 0, or not a number with the row's sum)
            const float f = L == 0.0f ? 0.0f : weight_of(m, M) / L;
            s_f[t >> 2][t & 3] = make_float2(f, m == -__builtin_huge_valf() || f != f ? f : 0.0f);
        }
        __syncthreads();
        const float* pp = a.pp + ((at + h0) * a.ns + sp) * kPSplit + t;
        const size_t step = (size_t)a.ns * kPSplit;
        for (int h = 0; h < nh; h += 8) {
            float v[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) v[u] = h + u < nh ? pp[(h + u) * step] : 0.0f;
#pragma unroll
            for (int u = 0; u < 8; ++u)
                if (h + u < nh) {
                    const float2 f = s_f[h + u][t >> 6];
                    w = f.x == 0.0f || f.x != f.x ? w + f.y : __builtin_fmaf(v[u], f.x, w);
                }
        }
    }
    if (key < min(q.raw, a.max_len)) a.w[(size_t)(q.first + i) * a.w_stride + key] = key > q.raw - q.n + i ? 0.0f : w;
}

struct WorkLayout { size_t po, pp, pm, pl, pm64, fin, total; };
static WorkLayout work_layout(int nq, int hd, int max_len, int nrows, int weights) {
    const size_t n = (size_t)nrows * nq, ns = ((size_t)max_len + kPSplit - 1) / kPSplit;
    WorkLayout w{};
    w.po = 0;
    w.pp = w.po + n * ns * hd;
    w.pm = w.pp + (weights ? n * ns * kPSplit : 0);
    w.pl = w.pm + n * ns;
    w.pm64 = w.pl + n * ns;
    w.fin = w.pm64 + (weights ? n * ns * 4 : 0);
    w.total = w.fin + (weights ? 2 * n : 0);
    return w;
}

template <int HD, int G, int RT>
static int launch_split_rt(const PAttnArgs& a, hipStream_t s) {
    // as many blocks as fit at once, or fewer units: those of max_len keys in every sequence, in eights (one per XCD)
    const int ncb = (a.max_rows * (a.nq / a.kv.nkv) + 16 * RT - 1) / (16 * RT);
    const long long units = ((long long)a.kv.n_seq * a.ns + 7) / 8 * a.kv.nkv * ncb;
    const long long most = (long long)kCUs / 8 * AttnOcc<HD, G, RT>::n;
    hipLaunchKernelGGL((k_paged_attn<HD, G, RT>), dim3((unsigned)(8 * (units < most ? units : most))), dim3(256), 0, s, a);
    Q27X_HIP(hipGetLastError());
    return Q27X_OK;
}
template <int HD, int G>
static int launch_split(const PAttnArgs& a, hipStream_t s) {
    return a.max_rows * (a.nq / a.kv.nkv) <= 16 ? launch_split_rt<HD, G, 1>(a, s) : launch_split_rt<HD, G, 2>(a, s);
}
static int launch_paged_attn(const PAttnArgs& a, hipStream_t s) {
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
    if (rc || (a.ns == 1 && !a.w)) return rc;
    const unsigned rows = (unsigned)(a.kv.n_seq * a.max_rows);
    if ((long long)rows * a.nq < 2 * kCUs) hipLaunchKernelGGL(k_paged_combine<16>, dim3((unsigned)(a.nq * (a.kv.hd / 64)), rows), dim3(256), 0, s, a);
    else if (a.kv.hd == 128) hipLaunchKernelGGL(k_paged_combine<32>, dim3((unsigned)a.nq, rows), dim3(256), 0, s, a);
    else hipLaunchKernelGGL(k_paged_combine<64>, dim3((unsigned)a.nq, rows), dim3(256), 0, s, a);
    Q27X_HIP(hipGetLastError());
    if (a.w) {
        hipLaunchKernelGGL(k_paged_weights, dim3((unsigned)a.ns, rows), dim3(256), 0, s, a);
        Q27X_HIP(hipGetLastError());
    }
    return Q27X_OK;
}

}  // namespace q27x

using namespace q27x;
extern "C" int q27x_paged_prep_rows(const uint16_t* qkv, int qkv_stride, const uint16_t* q_norm_w, const uint16_t* k_norm_w,
                                    const float* rope_cos, const float* rope_sin, int rot, int n_pos, const int32_t* pos,
                                    int pos_stride, int n_axes, const uint8_t* pair_axis, const q27x_paged_kv_t* kv,
                                    uint16_t* qh, int nq, int gate, float eps, int nrows, q27x_stream_t s) {
    const char* who = "q27x_paged_prep_rows";
    PrepArgs a{};
    if (int rc = paged_args(kv, who, &a.kv)) return rc;
    if (!qkv || !q_norm_w || !k_norm_w || !rope_cos || !rope_sin || !pos || !qh || (n_axes > 1 && !pair_axis)) {
        set_error("%s: null argument", who);
        return Q27X_E_ARG;
    }
    if (nq < 1 || nq > 1024 || nq % a.kv.nkv || rot < 2 || (rot & 1) || rot > a.kv.hd) {
        set_error("%s: unsupported shape (nq=%d nkv=%d hd=%d rot=%d: rot even, at most hd)", who, nq, a.kv.nkv, a.kv.hd, rot);
        return Q27X_E_SHAPE;
    }
    if (n_pos < 1 || n_axes < 1 || n_axes > 4 || nrows < 1 || (n_axes > 1 && pos_stride < nrows) || qkv_stride < 0) {
        set_error("%s: bad counts (n_pos=%d n_axes=%d pos_stride=%d nrows=%d qkv_stride=%d)", who, n_pos, n_axes, pos_stride, nrows, qkv_stride);
        return Q27X_E_ARG;
    }
    for (int i = 0; i < rot / 2; ++i) {
        const int axis = pair_axis ? pair_axis[i] : 0;
        if (axis >= n_axes) { set_error("%s: pair %d turns by axis %d of %d", who, i, axis, n_axes); return Q27X_E_ARG; }
        a.axes[i >> 4] |= (uint32_t)axis << (2 * (i & 15));
    }
    a.qkv = qkv; a.qkv_stride = qkv_stride; a.q_norm_w = q_norm_w; a.k_norm_w = k_norm_w;
    a.rope_cos = rope_cos; a.rope_sin = rope_sin; a.rot = rot; a.n_pos = n_pos;
    a.pos = pos; a.pos_stride = pos_stride; a.n_axes = n_axes;
    a.qh = qh; a.nq = nq; a.gate = gate ? 1 : 0; a.eps = eps; a.nrows = nrows;
    return launch_prep(a, (hipStream_t)s);
}

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
    if (w) { a.pp = p + wl.pp; a.pm64 = p + wl.pm64; a.fin = p + wl.fin; }
    a.out = out; a.xq = xq; a.xs = xs; a.w = w; a.w_stride = w_stride;
    return launch_paged_attn(a, (hipStream_t)s);
}

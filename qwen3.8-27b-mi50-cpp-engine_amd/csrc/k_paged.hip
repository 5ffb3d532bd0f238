// k_paged.hip -- one paged key/value cache for many sequences: its handle, and preparing new rows (norm, rotary positions of
// several axes, append).

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
// Wave = 4 heads of q | k | v of a row, 16 lanes a head: a lane holds HD/16 neighbouring dims, so a group's maximum and the
// head's sum of squares are a few DPP steps and four heads share a wave's root and division. Waves are independent: each
// reads its row's angles into its own LDS (a row's are 2 rot floats, from L1 after the first wave), and the partner dims of
// a turn come through LDS too, so rot can be any even number. Bound by latency (row -> sequence -> page and position -> angle are
// chains of loads), so the row's values are requested before anything else and both chains run beside the norm.
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
// two floats as bf16 (to nearest even, by the hardware)
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 v = {(__bf16)lo, (__bf16)hi};
    return __builtin_bit_cast(uint32_t, v);
}
template <int E>
__device__ __forceinline__ void st_bf16(uint16_t* p, const float (&v)[E]) {
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));
#pragma unroll
    for (int i = 0; i < E / 8; ++i) {
        u32x4 x;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[j] = pack_bf16(v[8 * i + 2 * j], v[8 * i + 2 * j + 1]);
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
    const int r = blockIdx.x, t = threadIdx.x, l = t & 63, c = t & 15, wv = t >> 6, slotw = t >> 4;
    const int half = a.rot >> 1;
    __shared__ __attribute__((aligned(16))) float s_cs[4][2][HD / 2];
    __shared__ __attribute__((aligned(16))) float s_ex[16][HD];
    const int u = blockIdx.y * 16 + slotw;           // q heads, then k, then v
    const bool isq = u < a.nq, isk = !isq && u < a.nq + a.kv.nkv, isv = !isq && !isk && u < a.nq + 2 * a.kv.nkv;
    const int head = isq ? u : isk ? u - a.nq : u - a.nq - a.kv.nkv;
    const int qw = a.gate ? 2 * HD : HD;
    float y[E], w[E];
    // (lanes past the last head read the first one's)
    const uint16_t* src = a.qkv + (size_t)r * a.qkv_stride + E * c +
                          (isq ? (size_t)head * qw : isk || isv ? (size_t)a.nq * qw + ((size_t)(isv ? a.kv.nkv : 0) + head) * HD : 0);
    ld_bf16<E>(src, y);
    ld_bf16<E>((isq ? a.q_norm_w : a.k_norm_w) + E * c, w);
    // the row's angles: lane l takes the cosines, then the sines of pairs l, l + 64 ..
    int p[HD / 128];
#pragma unroll
    for (int i = 0; i < HD / 128; ++i) {
        const int f = l + 64 * i < half ? l + 64 * i : 0;
        const int axis = (a.axes[f >> 4] >> (2 * (f & 15))) & 3;
        p[i] = a.pos[(size_t)axis * a.pos_stride + r];
    }
    const int b = seq_of_row(a.kv, r);
    if (b < 0) return;                               // (a row behind the last sequence)
    int slot = -1;
    if (isk || isv) {
        int first, n;
        paged_rows(a.kv, b, first, n);
        slot = paged_slot(a.kv, b, a.kv.lens[b] - n + (r - first));
    }
#pragma unroll
    for (int i = 0; i < HD / 128; ++i) {
        const int f = l + 64 * i;
        if (f < half) {
            const int q = p[i] < 0 ? 0 : (p[i] >= a.n_pos ? a.n_pos - 1 : p[i]);
            s_cs[wv][0][f] = a.rope_cos[(size_t)q * half + f];
            s_cs[wv][1][f] = a.rope_sin[(size_t)q * half + f];
        }
    }
    const bool turns = (isq || isk) && E * c < a.rot;
    if (isq || isk) {
        float ss = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) ss = __builtin_fmaf(y[e], y[e], ss);
        ss = sum16(ss);
        const float inv = rsqrt_cr(ss * (1.0f / (float)HD) + a.eps);
#pragma unroll
        for (int e = 0; e < E; ++e) y[e] = y[e] * inv * (1.0f + w[e]);
        if (turns) {
#pragma unroll
            for (int e = 0; e < E; ++e) s_ex[slotw][E * c + e] = y[e];
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (turns && half % E == 0) {                    // a lane's dims are one half's, its partners and angles neighbours
        const int d = E * c, f = d < half ? d : d - half;
        const float4* o4 = (const float4*)&s_ex[slotw][d < half ? d + half : f];
        const float4 *c4 = (const float4*)&s_cs[wv][0][f], *s4 = (const float4*)&s_cs[wv][1][f];
        const float sign = d < half ? -1.0f : 1.0f;
#pragma unroll
        for (int e = 0; e < E; e += 4) {
            const float4 o = o4[e / 4], k = c4[e / 4], n = s4[e / 4];
            y[e] = __builtin_fmaf(sign * o.x, n.x, y[e] * k.x);
            y[e + 1] = __builtin_fmaf(sign * o.y, n.y, y[e + 1] * k.y);
            y[e + 2] = __builtin_fmaf(sign * o.z, n.z, y[e + 2] * k.z);
            y[e + 3] = __builtin_fmaf(sign * o.w, n.w, y[e + 3] * k.w);
        }
    } else if (turns) {
#pragma unroll 1
        for (int e = 0; e < E; ++e) {
            const int d = E * c + e, f = d < half ? d : d - half;
            if (d < a.rot) {
                const float o = s_ex[slotw][d < half ? d + half : f], k = s_cs[wv][1][f];
                const float z = __builtin_fmaf(o, d < half ? -k : k, s_ex[slotw][d] * s_cs[wv][0][f]);
#pragma unroll
                for (int x = 0; x < E; ++x) y[x] = x == e ? z : y[x];
            }
        }
    }
    if (isq) st_bf16<E>(a.qh + ((size_t)r * a.nq + head) * HD + E * c, y);
    else if (slot >= 0) st_kv<HD, G>(a.kv, isk ? a.kv.k : a.kv.v, isk ? a.kv.ks : a.kv.vs, (size_t)slot, head, c, y);
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

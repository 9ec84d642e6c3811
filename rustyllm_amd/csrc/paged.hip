// paged.hip — the paged 4-bit KV cache: rows of many sessions appended with
// their rotation, read back, and attended to.
//
// Values.  32 consecutive channels of a row form a group with one half-
// precision scale d and 32 codes c (0..15); the group's values are d (c - 8),
// those of GGUF's Q4_0.  With e the group's value of largest magnitude (the
// positive one at a tie), d = half(clamp(e / -8, +-8188)), so e itself sits on
// code 0 (value -8 d) and |d (c - 8)| <= 65504 stays a finite half; c = 8 +
// clamp(rne(x * r), -8, 7) with r = f32(1 / d), 0 where d is 0.  A NaN makes
// its whole group NaN, infinities saturate.  Products of the rotation are
// rounded before they are added (no FMA), as the other RoPE kernels do, so a
// code depends on nothing but the definition.
//
// Layout.  A page holds ps tokens; for each kv head it is one block of
// ps * 18 * G bytes, where G = 2, 4 or 8 groups cover the head size: ps * 16 *
// G bytes of codes, then scales [ps][G].  16 tokens of codes are 256 G
// contiguous bytes from which every lane l of a wave loads 4 G contiguous
// bytes that are its matrix operand:
//   K: token l % 16, dwords [kc = l / 16][g], nibble n = channel 32 g + 8 kc + n
//      (A[m = token][k = 8 kc + .] of a 16x16x32 product per group)
//   V: tokens 4 (l / 16) + t, bytes [c = l % 16][t][g], low nibble = channel
//      32 g + c, high nibble = channel 32 g + 16 + c (a 16x16x32 product per
//      group and nibble, k = token, transposed by byte permutes alone)
#pragma once

#include "common.hpp"

namespace rh {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8v __attribute__((ext_vector_type(8)));
typedef float f32x4v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4v __attribute__((ext_vector_type(4)));

struct PagedDev {
    uint8_t *k, *v;
    const int32_t *table;     // [n_seqs][stride] page ids
    const int32_t *kv_lens;   // [n_seqs]
    const int32_t *q_starts;  // [n_seqs + 1]
    int32_t n_pages, ps, n_kv, hd, vd, n_seqs, stride, n_tokens;
    uint32_t tile_mul, tile_shift;  // 16-token tile -> page, see page_of_tile
    int64_t block;                  // bytes of one (page, kv head)
};

// n / d for n < 2^31 as (n * mul) >> shift: shift = 31 + ceil(log2 d), mul =
// ceil(2^shift / d) <= 2^32 - 1 for d > 1, whose excess over 2^shift / d is below
// 2^ceil(log2 d) / d, too little to reach the next quotient.  (An integer division
// is about 25 instructions.)
__host__ __device__ __forceinline__ int page_of_tile(const PagedDev &P, int tile) {
    return P.tile_mul ? (int)((uint64_t)(uint32_t)tile * P.tile_mul >> P.tile_shift) : tile;
}

// Session of row t of the batch, wave-uniform: the last start at or below t, found
// by 64 lanes at a time.  False for rows of no session: rows behind the last one,
// and starts that do not ascend.
__device__ __forceinline__ bool paged_session(const PagedDev &P, int t, int *seq, int *start, int *end) {
    const int lane = threadIdx.x & 63;
    int n = 0;
    for (int base = 0; base <= P.n_seqs; base += 64) {
        const int i = base + lane;
        n += __popcll(__ballot(i <= P.n_seqs && P.q_starts[i <= P.n_seqs ? i : 0] <= t));
    }
    const int s = n - 1;
    if (s < 0 || s >= P.n_seqs) return false;
    *seq = s;
    *start = P.q_starts[s];
    *end = P.q_starts[s + 1];
    return t >= *start && t < *end;
}

// Session and position of the N rows from t on (a session's rows are its last
// ones), -1 for rows of no session and for positions below zero.  One pass over the
// starts, and the N rows' loads in flight together.
template <int N>
__device__ __forceinline__ void paged_rows(const PagedDev &P, int t, int *seq, int *pos) {
    const int lane = threadIdx.x & 63;
    int n[N] = {};
    for (int base = 0; base <= P.n_seqs; base += 64) {
        const int i = base + lane, start = P.q_starts[i <= P.n_seqs ? i : 0];
#pragma unroll
        for (int j = 0; j < N; j++) n[j] += __popcll(__ballot(i <= P.n_seqs && start <= t + j));
    }
    int a[N], b[N], len[N];
#pragma unroll
    for (int j = 0; j < N; j++) {
        seq[j] = n[j] > 0 && n[j] <= P.n_seqs ? n[j] - 1 : 0;
        a[j] = P.q_starts[seq[j]];
        b[j] = P.q_starts[seq[j] + 1];
        len[j] = P.kv_lens[seq[j]];
    }
#pragma unroll
    for (int j = 0; j < N; j++) {
        const int64_t p = (int64_t)len[j] - ((int64_t)b[j] - (t + j));
        const bool ok = n[j] > 0 && n[j] <= P.n_seqs && t + j < P.n_tokens && t + j >= a[j] && t + j < b[j] && p >= 0;
        pos[j] = ok ? (int)p : -1;
    }
}

// Page of a position, or -1: outside the table's row or the pool.  *off: token in it.
__device__ __forceinline__ int paged_page(const PagedDev &P, int seq, int pos, int *off) {
    const int i = page_of_tile(P, pos >> 4);
    *off = pos - i * P.ps;
    const int page = P.table[(int64_t)seq * P.stride + (i < P.stride ? i : 0)];
    return i < P.stride && page >= 0 && page < P.n_pages ? page : -1;
}
// wave-uniform values into scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// ---- element access: rows of f32 or bf16 ----------------------------------------
__device__ __forceinline__ void row_load4(const float *p, float *x) {
    const float4 a = *(const float4 *)p;
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}
__device__ __forceinline__ void row_load4(const uint16_t *p, float *x) {
    const float4 a = bf16x4_load(p);
    x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w;
}
__device__ __forceinline__ void row_store4(float *p, const float *x) {
    *(float4 *)p = make_float4(x[0], x[1], x[2], x[3]);
}
__device__ __forceinline__ void row_store4(uint16_t *p, const float *x) {
    uint2 u;
    u.x = f32_to_bf16(x[0]) | (uint32_t)f32_to_bf16(x[1]) << 16;
    u.y = f32_to_bf16(x[2]) | (uint32_t)f32_to_bf16(x[3]) << 16;
    *(uint2 *)p = u;
}

// ---- append -------------------------------------------------------------------------
struct PagedAppend {
    const void *q, *k, *v;
    void *q_out;
    int64_t q_stride, k_stride, v_stride, qo_stride;  // elements between rows
    const float *cos_t, *sin_t;                       // [max_pos][rot / 2]
    int32_t n_heads, max_pos, rot, neox;
    int32_t q_segs, kv_segs;                          // waves for a row's q, and for its k (= for its v)
};

// Eight rotated channels ch.. of a head (ch a multiple of 8; rot a multiple of
// 16, so both halves of a NeoX pair are whole chunks).
template <class T>
__device__ __forceinline__ void paged_rotated8(const PagedAppend &A, const T *head, int ch, int pos, float *x) {
    row_load4(head + ch, x);
    row_load4(head + ch + 4, x + 4);
    if (ch >= A.rot) return;
    const int half = A.rot >> 1;
    const float *ct = A.cos_t + (int64_t)pos * half, *st = A.sin_t + (int64_t)pos * half;
    if (A.neox) {
        const bool up = ch >= half;
        const int p = up ? ch - half : ch;
        float y[8], c[8], s[8];
        row_load4(head + (up ? p : ch + half), y);
        row_load4(head + (up ? p : ch + half) + 4, y + 4);
        row_load4(ct + p, c);
        row_load4(ct + p + 4, c + 4);
        row_load4(st + p, s);
        row_load4(st + p + 4, s + 4);
#pragma unroll
        for (int j = 0; j < 8; j++) x[j] = up ? y[j] * s[j] + x[j] * c[j] : x[j] * c[j] - y[j] * s[j];
    } else {
        float c[4], s[4];
        row_load4(ct + (ch >> 1), c);
        row_load4(st + (ch >> 1), s);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float a = x[2 * j], b = x[2 * j + 1];
            x[2 * j] = a * c[j] - b * s[j];
            x[2 * j + 1] = a * s[j] + b * c[j];
        }
    }
}

// Codes (0..15) of this lane's eight channels; the four lanes of a quad hold one
// group and agree on its scale.
__device__ __forceinline__ uint16_t paged_codes(const float *x, uint32_t *c) {
    float top = x[0], low = x[0];
    int bad = x[0] != x[0];
#pragma unroll
    for (int j = 1; j < 8; j++) {
        top = fmaxf(top, x[j]);
        low = fminf(low, x[j]);
        bad |= x[j] != x[j];
    }
    top = fmaxf(top, __builtin_bit_cast(float, dpp_i<0xB1>(__builtin_bit_cast(int, top))));
    low = fminf(low, __builtin_bit_cast(float, dpp_i<0xB1>(__builtin_bit_cast(int, low))));
    bad |= dpp_i<0xB1>(bad);
    top = fmaxf(top, __builtin_bit_cast(float, dpp_i<0x4E>(__builtin_bit_cast(int, top))));
    low = fminf(low, __builtin_bit_cast(float, dpp_i<0x4E>(__builtin_bit_cast(int, low))));
    bad |= dpp_i<0x4E>(bad);
    float e = (top >= -low ? top : low) * -0.125f;
    e = fminf(fmaxf(e, -8188.0f), 8188.0f);
    const _Float16 d = (_Float16)(e + 0.0f);  // -0 becomes 0
    const float r = bad ? __builtin_nanf("") : (float)d == 0.0f ? 0.0f : 1.0f / (float)d;  // NaN: all codes 0
#pragma unroll
    for (int j = 0; j < 8; j++) c[j] = (uint32_t)((int)fminf(fmaxf(rintf(x[j] * r), -8.0f), 7.0f) + 8);
    return bad ? 0x7E00 : __builtin_bit_cast(uint16_t, d);
}

// One wave per (row, up to 64 units of eight channels): first the row's queries,
// then its keys, then its values.  A row's bytes are read and written once; what
// bounds it is the traffic for prompts (10496 f32 rows of 40 + 8 + 8 heads of 128
// channels: 111 us, 4.8 TB/s) and the chain of dependent loads (starts, length, page)
// for single tokens (one row 3.2 us, 200 rows 5.0 us).
template <int G, class T>
__global__ __launch_bounds__(256) void paged_append_kernel(PagedDev P, PagedAppend A) {
    __shared__ uint32_t s_v[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int segs = A.q_segs + 2 * A.kv_segs;
    const int64_t w = (int64_t)blockIdx.x * 4 + wave;
    const int t = (int)(w / segs);
    int seg = (int)(w % segs);
    if (t >= P.n_tokens) return;
    int seq, pos;
    paged_rows<1>(P, t, &seq, &pos);
    if (pos < 0 || pos >= A.max_pos) return;
    if (seg < A.q_segs) {
        // whole heads per wave: q_out may be q, where a lane's partner chunk is
        // another lane's output, and the wave's loads are all done before it stores
        const int lanes = P.hd >> 3, heads = 64 / lanes;
        const int mine = lane / lanes, head = seg * heads + mine, c = (lane - mine * lanes) * 8;
        if (mine >= heads || head >= A.n_heads) return;
        float x[8];
        paged_rotated8(A, (const T *)A.q + (int64_t)t * A.q_stride + (int64_t)head * P.hd, c, pos, x);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        T *o = (T *)A.q_out + (int64_t)t * A.qo_stride + (int64_t)head * P.hd + c;
        row_store4(o, x);
        row_store4(o + 4, x + 4);
        return;
    }
    seg -= A.q_segs;
    int off;
    const int page = paged_page(P, seq, pos, &off);
    if (page < 0) return;
    const bool is_v = seg >= A.kv_segs;
    const int u = (is_v ? seg - A.kv_segs : seg) * 64 + lane;
    const int head = u / (4 * G), g = (u % (4 * G)) >> 2, i = u & 3;
    const bool on = head < P.n_kv;
    uint8_t *blk = (is_v ? P.v : P.k) + ((int64_t)page * P.n_kv + (on ? head : 0)) * P.block;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    uint32_t c[8];
    if (!is_v) {
        const int ch = 32 * g + 8 * i;
        if (on && ch < P.hd)
            paged_rotated8(A, (const T *)A.k + (int64_t)t * A.k_stride + (int64_t)head * P.hd, ch, pos, x);
        const uint16_t d = paged_codes(x, c);
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 8; j++) word |= c[j] << (4 * j);
        if (on) {
            *(uint32_t *)(blk + (int64_t)off * (16 * G) + (i * G + g) * 4) = word;
            if (i == 0) *(uint16_t *)(blk + (int64_t)P.ps * (16 * G) + (off * G + g) * 2) = d;
        }
        return;
    }
    // values: channels 4 i.. and 16 + 4 i.. of the group make four bytes, which
    // the wave's LDS turns from [g][c] to the page's [c][g]
    const int ch = 32 * g + 4 * i;
    const T *row = (const T *)A.v + (int64_t)t * A.v_stride + (int64_t)head * P.vd;
    if (on && ch < P.vd) row_load4(row + ch, x);
    if (on && ch + 16 < P.vd) row_load4(row + ch + 16, x + 4);
    const uint16_t d = paged_codes(x, c);
    uint8_t *s = (uint8_t *)s_v[wave];
#pragma unroll
    for (int j = 0; j < 4; j++) s[(lane / (4 * G)) * (16 * G) + (4 * i + j) * G + g] = (uint8_t)(c[j] | c[4 + j] << 4);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const uint32_t word = s_v[wave][lane];
    if (!on) return;
    const int b = (lane % (4 * G)) * 4, cc = b / G;  // this lane's four bytes of the row
    uint8_t *dst = blk + (int64_t)((off >> 2) * 64 + cc * 4 + (off & 3)) * G + b % G;
    if (G >= 4) {
        *(uint32_t *)dst = word;
    } else {
        *(uint16_t *)dst = (uint16_t)word;
        *(uint16_t *)(dst + 4 * G) = (uint16_t)(word >> 16);
    }
    if (i == 0) *(uint16_t *)(blk + (int64_t)P.ps * (16 * G) + (off * G + g) * 2) = d;
}

// ---- read ---------------------------------------------------------------------------
struct PagedRead {
    void *k, *v;
    int64_t k_stride, v_stride;
    int32_t kv_segs;
};

// One wave per (N rows, up to 64 dwords of keys or of values of each), the rows'
// loads in flight together.  A lane puts out 16 bytes at a time, so that a store
// covers 1 KB without gaps (eight f32 channels per lane, in two stores of every other
// 16 bytes, took 53 us for 20001 rows instead of 50).
template <int G, class T, int N>
__global__ __launch_bounds__(256) void paged_read_kernel(PagedDev P, PagedRead A) {
    __shared__ uint32_t s_v[4][N][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t w = (int64_t)blockIdx.x * 4 + wave;
    const int t = (int)(w / (2 * A.kv_segs)) * N, seg = (int)(w % (2 * A.kv_segs));
    if (t >= P.n_tokens) return;
    const bool is_v = seg >= A.kv_segs;
    if (is_v ? !A.v : !A.k) return;
    int seq[N], pos[N], page[N], off[N];
    paged_rows<N>(P, t, seq, pos);
#pragma unroll
    for (int j = 0; j < N; j++) {  // (a row that has no page reads page 0)
        page[j] = paged_page(P, seq[j], pos[j] < 0 ? 0 : pos[j], &off[j]);
        if (pos[j] < 0) page[j] = -1;
        if (page[j] < 0) off[j] = 0;
    }
    const uint8_t *pool = is_v ? P.v : P.k;
    const int first = (is_v ? seg - A.kv_segs : seg) * (64 / (4 * G)), dim = is_v ? P.vd : P.hd;  // first head
    const int64_t stride = is_v ? A.v_stride : A.k_stride;
    T *out = (T *)(is_v ? A.v : A.k);
    if (is_v) {
        // [c][g] bytes of four channels' pairs to LDS
        const int head = first + lane / (4 * G), b = (lane % (4 * G)) * 4, cc = b / G;
        uint32_t word[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const uint8_t *src = pool + ((int64_t)(page[j] < 0 ? 0 : page[j]) * P.n_kv + (head < P.n_kv ? head : 0)) * P.block +
                                 (int64_t)((off[j] >> 2) * 64 + cc * 4 + (off[j] & 3)) * G + b % G;
            if (G >= 4)
                word[j] = *(const uint32_t *)src;
            else
                word[j] = *(const uint16_t *)src | (uint32_t)*(const uint16_t *)(src + 4 * G) << 16;
        }
#pragma unroll
        for (int j = 0; j < N; j++) s_v[wave][j][lane] = word[j];
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
    }
    // C channels, 16 bytes of output, per lane and pass
    constexpr int C = 16 / sizeof(T);
#pragma unroll
    for (int pass = 0; pass < 8 / C; pass++) {
        const int u = 64 * pass + lane, head = first + u / (32 * G / C), r = u % (32 * G / C), g = r / (32 / C);
        const int ch = r % (32 / C) * C;  // in the group
        const bool on = head < P.n_kv && C * r < dim;
        uint32_t code[N];
        float d[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            const uint8_t *blk = pool + ((int64_t)(page[j] < 0 ? 0 : page[j]) * P.n_kv + (head < P.n_kv ? head : 0)) * P.block;
            d[j] = h2f(*(const uint16_t *)(blk + (int64_t)P.ps * (16 * G) + (off[j] * G + g) * 2));
            const uint8_t *src = blk + (int64_t)off[j] * (16 * G) + ((ch >> 3) * G + g) * 4;
            if (!is_v) code[j] = C == 8 ? *(const uint32_t *)src : *(const uint16_t *)(src + (ch & 4) / 2);
        }
#pragma unroll
        for (int j = 0; j < N; j++) {
            float x[C];
            const uint8_t *s = (const uint8_t *)s_v[wave][j] + (u / (32 * G / C) * 16 + (ch & 15)) * G + g;
#pragma unroll
            for (int n = 0; n < C; n++) {
                const uint32_t c = is_v ? (uint32_t)s[n * G] >> (ch >> 4) * 4 : code[j] >> (4 * n);
                x[n] = d[j] * (float)((int)(c & 15) - 8);
            }
            if (!on || page[j] < 0) continue;
            T *o = out + (int64_t)(t + j) * stride + (int64_t)head * dim + C * r;
#pragma unroll
            for (int n = 0; n < C; n += 4) row_store4(o + n, x + n);
        }
    }
}

}  // namespace rh

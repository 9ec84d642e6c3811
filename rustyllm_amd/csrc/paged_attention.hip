// paged_attention.hip — attention over the paged 4-bit KV cache (paged.hip).
//
//   out = sum_t p_t v_t / (sum_t p_t + 2^(sink - m)),  p_t = 2^(s_t - m),
//   s_t = scale log2(e) q . k_t,   pos - window < t <= pos
//
// One pass over the cache: the running maximum m and sum of each row are kept
// in f32, the accumulators rescaled where m grows.
#pragma once

#include "paged.hip"

namespace rh {

typedef float f32x16v __attribute__((ext_vector_type(16)));

struct PagedAttn {
    const void *q;
    void *out;
    const float *sinks;  // [n_heads] or null
    float *part;         // [split][token][head][32 G] sums, or null with one split
    float *ml;           // [split][token][head][2]: maximum (base 2) and sum
    int64_t q_stride, o_stride;
    float scale;         // times log2(e)
    int32_t n_heads, kv_mul, window;
    int32_t n_chunk;     // 16 query heads of a kv head at a time
    int32_t inv16, inv;  // ceil(256 / heads) of a full chunk and of the last: row / heads for row < 16
    int32_t tok_tile;    // tokens of a row tile
    int32_t n_splits;    // most splits of a row tile's range
    int32_t split_steps; // 64-token steps of a split, more where n_splits would not cover the range
    int32_t short_q;     // sessions of up to so many rows are row tiles of their own (paged_attn_rows_kernel)
    int32_t both;        // 1: the others are paged_attn_tile_kernel's; 0: all are of one kind
};

// A row tile: its session, first token (of the session) and tokens, the session's
// first row, and the first token's position.
struct PagedTile {
    int seq, tok, n, row0, pos0;
};
__device__ __forceinline__ bool paged_tile_of(const PagedDev &P, const PagedAttn &A, int seq, int tok, PagedTile *T) {
    T->seq = uniform(seq);
    T->tok = uniform(tok);
    const int a = uniform(P.q_starts[T->seq]), b = uniform(P.q_starts[T->seq + 1]);
    if (a < 0 || b > P.n_tokens || T->tok < 0 || b - a <= T->tok) return false;
    T->n = b - a - T->tok < A.tok_tile ? b - a - T->tok : A.tok_tile;
    T->row0 = a;
    const int64_t pos = (int64_t)uniform(P.kv_lens[T->seq]) - (b - a) + T->tok;
    T->pos0 = (int)(pos < -(1 << 30) ? -(1 << 30) : pos);
    return !A.both || (b - a <= A.short_q) == (A.tok_tile == A.short_q);
}
// Tile x of the sessions with more than short_q rows (of all, unless both): 64
// sessions per turn, each lane one session's tile count.
__device__ __forceinline__ bool paged_tile(const PagedDev &P, const PagedAttn &A, int x, PagedTile *T) {
    const int lane = threadIdx.x & 63, least = A.both ? A.short_q : 0;
    int before = 0;
    for (int base = 0; base < P.n_seqs; base += 64) {
        const int i = base + lane;
        int c = 0;
        if (i < P.n_seqs) {
            const int64_t len = (int64_t)P.q_starts[i + 1] - P.q_starts[i];
            c = len > least && len <= P.n_tokens ? ((int)len + A.tok_tile - 1) / A.tok_tile : 0;
        }
        int sum = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int up = __shfl_up(sum, o, 64);
            if (lane >= o) sum += up;
        }
        const uint64_t here = __ballot(before + sum > x);
        if (here) {
            const int l = __ffsll((unsigned long long)here) - 1;
            return paged_tile_of(P, A, base + l, (x - before - __shfl(sum - c, l, 64)) * A.tok_tile, T);
        }
        before += __shfl(sum, 63, 64);
    }
    return false;
}

// Cached positions [lo, hi) that any of a tile's rows attends to.
struct PagedRange {
    int lo, hi, first;  // first: the 16-token tile that lo is in
    int steps;          // 64-token steps from first to hi
};
__device__ __forceinline__ PagedRange paged_range(const PagedDev &P, const PagedAttn &A, int pos0, int n) {
    PagedRange r;
    const int64_t table = (int64_t)P.stride * P.ps, most = 0x7FFFFF00, room = table < most ? table : most;
    const int64_t hi = (int64_t)pos0 + n;
    r.hi = (int)(hi < room ? hi : room);
    const int64_t lo = A.window > 0 ? (int64_t)pos0 - A.window + 1 : 0;
    r.lo = lo > 0 ? (int)(lo < room ? lo : room) : 0;
    r.first = r.lo & ~15;
    r.steps = r.hi > r.lo ? (int)(((int64_t)r.hi - r.first + 63) >> 6) : 0;
    return r;
}

__device__ __forceinline__ half2v paged_h2(uint32_t w) { return __builtin_bit_cast(half2v, w); }

// Codes as exact halves c - 8: a nibble or-ed into 1024 (bits 0..3) or 64 (bits
// 4..7) makes the half 1024 + c or 64 + c.  The two constants live in vector
// registers of their own, so mask and or are one instruction (a VALU instruction
// reads one scalar register or literal).
struct PagedMagic {
    uint32_t lo = 0x64006400u, hi = 0x54005400u;
    __device__ __forceinline__ PagedMagic() { asm("" : "+v"(lo), "+v"(hi)); }
    __device__ __forceinline__ uint32_t low(uint32_t w) const {
        const half2v o = {(_Float16)-1032.0f, (_Float16)-1032.0f};
        return __builtin_bit_cast(uint32_t, paged_h2((w & 0x000F000Fu) | lo) + o);
    }
    __device__ __forceinline__ uint32_t high(uint32_t w) const {
        const half2v o = {(_Float16)-72.0f, (_Float16)-72.0f};
        return __builtin_bit_cast(uint32_t, paged_h2((w & 0x00F000F0u) | hi) + o);
    }
    // the 8 codes of a K dword, in the order nibble 0 4 1 5 2 6 3 7
    __device__ __forceinline__ half8v k8(uint32_t w) const {
        const u32x4v r = {low(w), high(w), low(w >> 8), high(w >> 8)};
        return __builtin_bit_cast(half8v, r);
    }
};

template <int CTRL>
__device__ __forceinline__ float paged_dpp(float v) {
    return __builtin_bit_cast(float, dpp_i<CTRL>(__builtin_bit_cast(int, v)));
}
// Where a wave's next 16 steps' tiles lie: lane j looks up tile j % 4 of the
// wave's step j / 4.
struct PagedWhere {
    uint64_t codes;   // byte offset of the tile's codes
    uint64_t scales;  // and of its scales
    uint64_t ok;      // one bit per tile: inside the range, its page inside the pool
};
template <int G>
__device__ __forceinline__ PagedWhere paged_where(const PagedDev &P, const PagedRange &rg, int seq, int64_t head_off,
                                                  int step, int step_by, int s_hi) {
    const int lane = threadIdx.x & 63;
    const int s = step + (lane >> 2) * step_by;
    const int t = rg.first + s * 64 + (lane & 3) * 16;
    const bool in = s < s_hi && t < rg.hi;
    int off = 0;
    const int page = in ? paged_page(P, seq, t, &off) : -1;
    if (page < 0) off = 0;
    const uint64_t at = (uint64_t)(page < 0 ? 0 : page) * (uint64_t)(P.n_kv * P.block) + (uint64_t)head_off;
    PagedWhere w;
    w.codes = at + (uint32_t)off * (16 * G);
    w.scales = at + (uint32_t)(P.ps * (16 * G) + off * (2 * G));
    w.ok = __ballot(page >= 0);
    return w;
}
__device__ __forceinline__ uint64_t lane_u64(uint64_t v, int l) {
    return (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)v, l) |
           (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), l) << 32;
}
__device__ __forceinline__ uint64_t shfl_u64(uint64_t v, int l) {
    return (uint32_t)__shfl((int)(uint32_t)v, l, 64) | (uint64_t)(uint32_t)__shfl((int)(uint32_t)(v >> 32), l, 64) << 32;
}

// Row tiles of at most R = 4, 8 or 16 rows (tokens x query heads of one kv head):
// single tokens, and short runs of them.
//
// The 16 columns of a 16x16x32 product hold 16 / R copies of the rows, copy i for
// the i-th of 16 / R tiles of 16 tokens: copy i's queries are zero in the other
// columns, so the products of all tiles accumulate in one result whose lane
// (column n, quarter c) holds the scores of row n % R against tokens 4 c + r of
// tile n / R.  No lane's softmax work is spent on padding.  Codes go into the
// products as the exact integers c - 8; each group's K product is scaled by d of
// its (token, group) in f32, and V's scale goes into p: p d 2^E as one half (two
// for f32 rows: 22 bits), where E, the same for the wave, keeps the largest |d| seen
// near 2^14, so p d leaves the normal halves only 2^28 below the largest.
//
// The W = 4 waves of a workgroup take a tile's steps in turn and join their results;
// W = 1 is for many short sessions.  Neighbouring workgroups are the kv heads of one
// tile, so the sessions spread over the 8 XCDs (a session each made the XCD with the
// longest ones last).
//
// What bounds it: for bf16 rows the cache's bytes (one session of 131072 positions, 8 kv
// heads of 128 channels: 33 us, 4.6 TB/s); for f32 rows, whose p takes two halves, the
// issue of about 520 VALU and 64 matrix instructions per wave and step (48 sessions of
// up to 8192: 78 us, 3.4 TB/s); below some 10 steps the start of one wave (7.5 us).
template <int G, int R, bool F32, int W>
__global__ __launch_bounds__(64 * W, G == 8 ? 1 : G == 4 ? (R == 4 && !F32 ? 3 : 2) : R == 4 ? 4 : 3) void paged_attn_rows_kernel(PagedDev P, PagedAttn A) {
    constexpr int NT = 16 / R;  // token tiles per score result
    constexpr int NU = 4 / NT;  // score results per 64-token step
    constexpr int DV = 32 * G;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4, copy = col / R;
    const int heads_y = P.n_kv * A.n_chunk, tile = (int)(blockIdx.x / (uint32_t)heads_y);
    const int head_y = (int)(blockIdx.x - (uint32_t)tile * (uint32_t)heads_y);
    const int kvh = A.n_chunk == 1 ? head_y : head_y / A.n_chunk, h0 = A.n_chunk == 1 ? 0 : head_y % A.n_chunk * 16;
    const bool last = A.kv_mul - h0 < 16;
    const int heads = last ? A.kv_mul - h0 : 16, inv = last ? A.inv : A.inv16;
    const int split = blockIdx.y;
    PagedTile T;
    if (!paged_tile_of(P, A, tile, 0, &T)) return;
    const int seq = T.seq, n_tok = T.n, row0 = T.row0, pos0 = T.pos0;
    const PagedRange rg = paged_range(P, A, pos0, n_tok);

    // the splits' and then the waves' share of the steps
    int per = A.split_steps;
    if ((int64_t)per * A.n_splits < rg.steps) per = (rg.steps + A.n_splits - 1) / A.n_splits;
    const int64_t s_at = (int64_t)split * per;
    const int s_lo = (int)(s_at < rg.steps ? s_at : rg.steps);
    const int s_hi = s_lo + per < rg.steps ? s_lo + per : rg.steps;
    const int s_first = s_lo + wave;
    const int n_mine = s_hi > s_first ? (s_hi - s_first + W - 1) / W : 0;  // steps s_first + W k
    const int64_t head_off = (int64_t)kvh * P.block;
    PagedWhere at = paged_where<G>(P, rg, seq, head_off, s_first, W, s_hi);

    // this lane's row: token and head of column col
    const int row = col % R, my_tok = row * inv >> 8, my_head = row - my_tok * heads;
    const bool on = my_tok < n_tok;
    const int my_pos = pos0 + my_tok;
    int rhi = on ? my_pos + 1 : 0, rlo = A.window > 0 && my_pos - A.window + 1 > 0 ? my_pos - A.window + 1 : 0;
    if (rhi > rg.hi) rhi = rg.hi;

    // Codes and scales of one step.  16-row tiles need every token's scales in every
    // lane: those are loaded where they are used.
    constexpr bool KEEP = R < 16;
    uint32_t kc[4][G], vc[4][G], ks[KEEP ? NU : 1][2 * G], vs[KEEP ? NU : 1][2 * G];
    const uint32_t k_lane = (uint32_t)((lane & 15) * 16 * G + quad * 4 * G);
    const uint32_t v_lane = (uint32_t)(quad * 64 * G + (lane & 15) * 4 * G);
    auto load_codes = [&](const uint8_t *pool, uint32_t mine, int k, uint32_t (&to)[4][G])
                          __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < 4; i++)
            __builtin_memcpy(to[i], pool + lane_u64(at.codes, 4 * k + i) + mine, 4 * G);
    };
    auto scales_at = [&](int k, int u) __attribute__((always_inline)) {
        return shfl_u64(at.scales, 4 * k + u * NT + copy) + (uint32_t)(quad * 8 * G);
    };
    auto load_k = [&](int k) __attribute__((always_inline)) {
        load_codes(P.k, k_lane, k, kc);
        if (KEEP)
#pragma unroll
            for (int u = 0; u < NU; u++) __builtin_memcpy(ks[KEEP ? u : 0], P.k + scales_at(k, u), 8 * G);
    };
    auto load_v = [&](int k) __attribute__((always_inline)) {
        load_codes(P.v, v_lane, k, vc);
        if (KEEP)
#pragma unroll
            for (int u = 0; u < NU; u++) __builtin_memcpy(vs[KEEP ? u : 0], P.v + scales_at(k, u), 8 * G);
    };
    if (n_mine > 0) {
        load_k(0);
        load_v(0);
    }

    // queries: f16 of q 2^-e with 2^e above the row's largest (and the rest of it in
    // a second f16 for f32 inputs, 22 bits in all), zero in the other tiles' columns
    // (in LDS where they would take 32 registers or more)
    constexpr int TERMS = F32 ? 2 : 1;
    constexpr bool QLDS = NT * G * TERMS >= 8;
    half8v qr[QLDS ? 1 : TERMS][QLDS ? 1 : NT][QLDS ? 1 : G];
    __shared__ half8v s_q[QLDS ? TERMS : 1][QLDS ? G : 1][QLDS ? 65 : 1];  // [lane], then zero
    float qf;
    {
        float x[G][8], big = 0.0f;
        // a lane without a row or channel reads another's: the loads of all groups
        // are in flight together, which a branch around each would prevent
        const int64_t from = (int64_t)(row0 + (on ? my_tok : 0)) * A.q_stride +
                             (int64_t)(kvh * A.kv_mul + h0 + my_head) * P.hd;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int ch = 32 * g + 8 * quad, c = ch < P.hd ? ch : 0;
            if (F32) {
                row_load4((const float *)A.q + from + c, x[g]);
                row_load4((const float *)A.q + from + c + 4, x[g] + 4);
            } else {
                row_load4((const uint16_t *)A.q + from + c, x[g]);
                row_load4((const uint16_t *)A.q + from + c + 4, x[g] + 4);
            }
        }
#pragma unroll
        for (int g = 0; g < G; g++) {
#pragma unroll
            for (int j = 0; j < 8; j++) x[g][j] = on && 32 * g + 8 * quad < P.hd ? x[g][j] : 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(x[g][j]));
        }
        big = fmaxf(big, __shfl_xor(big, 16, 64));
        big = fmaxf(big, __shfl_xor(big, 32, 64));
        int e = 0;
        if (big > 0.0f && big < __builtin_inff()) (void)frexpf(big, &e);
        qf = A.scale * ldexpf(1.0f, e);
        const float down = ldexpf(1.0f, -(e >> 1)), more = ldexpf(1.0f, -(e - (e >> 1)));  // 2^-e may not be normal
        const int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for (int g = 0; g < G; g++) {
            if (QLDS && g % W != wave) continue;  // a wave each
            half8v hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = x[g][order[j]] * down * more;
                hi[j] = (_Float16)v;
                lo[j] = (_Float16)(v - (float)hi[j]);
            }
            const half8v zero = {0, 0, 0, 0, 0, 0, 0, 0};
            if (!QLDS) {
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    qr[0][QLDS ? 0 : i][QLDS ? 0 : g] = copy == i ? hi : zero;
                    if (F32) qr[QLDS ? 0 : TERMS - 1][QLDS ? 0 : i][QLDS ? 0 : g] = copy == i ? lo : zero;
                }
            } else {
                half8v *to = s_q[0][QLDS ? g : 0];
                to[lane] = hi;
                if (lane == 0) to[64] = zero;
                if (F32) {
                    to = s_q[QLDS ? TERMS - 1 : 0][QLDS ? g : 0];
                    to[lane] = lo;
                    if (lane == 0) to[64] = zero;
                }
            }
        }
    }
    if (QLDS) __syncthreads();

    float m = -__builtin_inff(), l = 0.0f, E = 0.0f, d2_most = 0.0f;
    f32x4v acc[G][2];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int h = 0; h < 2; h++) acc[g][h] = f32x4v{0, 0, 0, 0};
    // rows whose masks the whole step passes need no masking
    const int full_lo = rg.lo + (A.window > 0 ? n_tok - 1 : 0), full_hi = rg.hi - (n_tok - 1);

    const PagedMagic magic;
    for (int k = 0; k < n_mine; k++) {
        const int t0 = rg.first + (s_first + W * k) * 64;
        const uint32_t okm = (uint32_t)(at.ok >> (4 * (k & 15))) & 15;
        const bool full = t0 >= full_lo && t0 + 64 <= full_hi && okm == 15, more = k + 1 < n_mine;
        // what this lane's row does not see may hold anything: its scales become 0
        auto clear = [&](int u, uint32_t (&d)[2 * G]) __attribute__((always_inline)) {
            const bool page = (okm >> (u * NT + copy)) & 1;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = t0 + 16 * (u * NT + copy) + 4 * quad + r;
                const bool out = t < rlo || t >= rhi || !page;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const int e = r * G + g;
                    d[e >> 1] &= out ? (e & 1 ? 0x0000FFFFu : 0xFFFF0000u) : 0xFFFFFFFFu;
                }
            }
        };

        // scores
        int q_at = lane;
        asm volatile("" : "+v"(q_at));  // keeps the reads in the loop, out of registers before it
        auto query = [&](int term, int i, int g) __attribute__((always_inline)) {
            if (QLDS)
                return s_q[QLDS ? term : 0][QLDS ? g : 0][QLDS ? (copy == i ? q_at : 64) : 0];
            return qr[QLDS ? 0 : term][QLDS ? 0 : i][QLDS ? 0 : g];
        };
        float sc[NU][4], mx = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < NU; u++) {
            uint32_t late[2 * G];
            if (!KEEP) __builtin_memcpy(late, P.k + scales_at(k & 15, u), 8 * G);
            const uint32_t(&kd)[2 * G] = KEEP ? ks[KEEP ? u : 0] : late;
#pragma unroll
            for (int r = 0; r < 4; r++) sc[u][r] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++) {
                f32x4v d = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const half8v k8 = magic.k8(kc[u * NT + i][g]);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, query(0, i, g), d, 0, 0, 0);
                    if (F32) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, query(TERMS - 1, i, g), d, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int e = r * G + g;
                    sc[u][r] = fmaf((float)paged_h2(kd[e >> 1])[e & 1], d[r], sc[u][r]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) sc[u][r] *= qf;
            if (!full) {
                const bool page = (okm >> (u * NT + copy)) & 1;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int t = t0 + 16 * (u * NT + copy) + 4 * quad + r;
                    if (t < rlo || t >= rhi || !page) sc[u][r] = -__builtin_inff();
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, sc[u][r]);
        }
        // the registers are free again: the next step's keys, under this one's values
        // (the last step loads its own again: with a branch around them the waits for
        // the values would count these loads as well)
        if (KEEP) {
            if (more && ((k + 1) & 15) == 0)
                at = paged_where<G>(P, rg, seq, head_off, s_first + W * (k + 1), W, s_hi);
            load_k((more ? k + 1 : k) & 15);
        }

        float d2 = 0.0f;
#pragma unroll
        for (int u = 0; u < NU; u++) {
            uint32_t late[2 * G];
            if (!KEEP) __builtin_memcpy(late, P.v + scales_at(k & 15, u), 8 * G);
            uint32_t(&vd)[2 * G] = KEEP ? vs[KEEP ? u : 0] : late;
            if (!full) clear(u, vd);
#pragma unroll
            for (int j = 0; j < 2 * G; j++) d2 = __builtin_amdgcn_fdot2(paged_h2(vd[j]), paged_h2(vd[j]), d2, false);
        }
        if (__ballot(mx > m || d2 > d2_most)) {
            // a row's scores lie in the lanes of all tiles and quarters
            if (NT >= 4) mx = fmaxf(mx, paged_dpp<0x124>(mx));
            if (NT >= 2) mx = fmaxf(mx, paged_dpp<0x128>(mx));
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            mx = fmaxf(mx, m);
            d2 = wave_max(d2);
            const float was = m - E;
            if (d2 > d2_most) {
                int e;
                (void)frexpf(d2, &e);  // |d| <= 2^(e / 2)
                E = (float)(14 - ((e + 1) >> 1));
                d2_most = ldexpf(1.0f, 2 * (15 - (int)E));
            }
            const float a = m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(was - (mx - E));
            m = mx;
            l *= a;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int h = 0; h < 2; h++) acc[g][h] *= a;
        }
        const float base = (m == -__builtin_inff() ? 0.0f : m) - E;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                sc[u][r] = __builtin_amdgcn_exp2f(sc[u][r] - base);
                l += sc[u][r];
            }

        // values, 32 tokens (two tiles) per product
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            constexpr int UU = NU > 1 ? NU / 2 : 1;  // score results of these 32 tokens
            uint32_t late[2][2 * G];
            if (!KEEP)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    __builtin_memcpy(late[x], P.v + scales_at(k & 15, 2 * k2 + x), 8 * G);
                    if (!full) clear(2 * k2 + x, late[x]);
                }
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t ph[UU][2], pl[UU][2];
#pragma unroll
                for (int v = 0; v < UU; v++)
#pragma unroll
                    for (int r = 0; r < 4; r += 2) {
                        const int u = NU > 1 ? k2 * UU + v : 0;
                        half2v hi, lo;
#pragma unroll
                        for (int x = 0; x < 2; x++) {
                            const int e = (r + x) * G + g;
                            const uint32_t w = KEEP ? vs[KEEP ? u : 0][e >> 1] : late[v & 1][e >> 1];
                            const _Float16 d = paged_h2(w)[e & 1];
                            hi[x] = (_Float16)fmaf(sc[u][r + x], (float)d, 0.0f);
                            if (F32) lo[x] = (_Float16)fmaf(sc[u][r + x], (float)d, -(float)hi[x]);
                        }
                        ph[v][r >> 1] = __builtin_bit_cast(uint32_t, hi);
                        if (F32) pl[v][r >> 1] = __builtin_bit_cast(uint32_t, lo);
                    }
                u32x4v bh, bl = {0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int i = (2 * k2 + x) % NT, v = NU > 1 ? (2 * k2 + x) / NT - k2 * UU : 0;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        // copy i's columns to the first R (row_ror by 16 - R i)
                        auto turn = [&](uint32_t y) -> uint32_t {
                            if (i == 0) return y;
                            if (i * R == 4) return (uint32_t)dpp_i<0x12C>((int)y);
                            if (i * R == 8) return (uint32_t)dpp_i<0x128>((int)y);
                            return (uint32_t)dpp_i<0x124>((int)y);
                        };
                        bh[2 * x + h] = turn(ph[v][h]);
                        if (F32) bl[2 * x + h] = turn(pl[v][h]);
                    }
                }
                u32x4v va, vb;
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int b0 = (2 * h) * G + g, b1 = (2 * h + 1) * G + g;
                        const uint32_t w = __builtin_amdgcn_perm(vc[2 * k2 + x][b1 >> 2], vc[2 * k2 + x][b0 >> 2],
                                                                 0x0C000C00u | (uint32_t)(b0 & 3) |
                                                                     (uint32_t)(4 + (b1 & 3)) << 16);
                        va[2 * x + h] = magic.low(w);
                        vb[2 * x + h] = magic.high(w);
                    }
                const half8v p8 = __builtin_bit_cast(half8v, bh);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const half8v v8 = __builtin_bit_cast(half8v, h ? vb : va);
                    acc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, p8, acc[g][h], 0, 0, 0);
                    if (F32)
                        acc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8, __builtin_bit_cast(half8v, bl),
                                                                           acc[g][h], 0, 0, 0);
                }
            }
        }
        if (!KEEP) {
            if (more && ((k + 1) & 15) == 0)
                at = paged_where<G>(P, rg, seq, head_off, s_first + W * (k + 1), W, s_hi);
            load_k((more ? k + 1 : k) & 15);
        }
        load_v((more ? k + 1 : k) & 15);
    }

    if (NT >= 4) l += paged_dpp<0x124>(l);
    if (NT >= 2) l += paged_dpp<0x128>(l);
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    // scores of NaN pass the maximum by, also where there is no other: with +inf the row
    // is no empty one, and its weight is NaN in every join
    if (l != l) m = __builtin_inff();
    if (W == 1) {  // one split, and the lanes hold whole results: four channels of a row each
        if (col >= R || !on) return;
        const int hd = kvh * A.kv_mul + h0 + my_head;
        const int64_t token = row0 + my_tok;
        const bool none = m == -__builtin_inff();
        const float one = ldexpf(1.0f, -(int)E);
        float f = none ? 0.0f : 1.0f / l;
        if (A.sinks && !none) {
            const float sink = A.sinks[hd] * 1.44269504f, top = fmaxf(m, sink), a = __builtin_amdgcn_exp2f(m - top);
            f = a * one / fmaf(l * one, a, __builtin_amdgcn_exp2f(sink - top));
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int ch = 32 * g + 16 * h + 4 * quad;
                if (ch >= P.vd) continue;
                float y[4];
#pragma unroll
                for (int j = 0; j < 4; j++) y[j] = none ? 0.0f : acc[g][h][j] * f;
                const int64_t to = token * A.o_stride + (int64_t)hd * P.vd + ch;
                if (F32)
                    row_store4((float *)A.out + to, y);
                else
                    row_store4((uint16_t *)A.out + to, y);
            }
        return;
    }
    const float unit = ldexpf(1.0f, -(int)E);
    __shared__ float s_acc[W][R][DV + 4];
    __shared__ float s_m[W][R], s_l[W][R];
    if (col < R) {
        if (quad == 0) {
            s_m[wave][col] = m;
            s_l[wave][col] = l * unit;
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                *(f32x4v *)&s_acc[wave][col][32 * g + 16 * h + 4 * quad] = acc[g][h] * unit;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * DV; i += 64 * W) {
        const int r = i / DV, ch = i % DV;
        const int tk = r * inv >> 8, hd = kvh * A.kv_mul + h0 + r - tk * heads;
        if (tk >= n_tok) break;
        float top = s_m[0][r];
#pragma unroll
        for (int w = 1; w < W; w++) top = fmaxf(top, s_m[w][r]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < W; w++) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][r] - base);
            sum = fmaf(f, s_l[w][r], sum);
            o = fmaf(f, s_acc[w][r][ch], o);
        }
        const int64_t token = row0 + tk;
        if (A.n_splits > 1) {
            const int64_t to = ((int64_t)split * P.n_tokens + token) * A.n_heads + hd;
            if (top != -__builtin_inff()) A.part[to * DV + ch] = o;
            if (ch == 0) {
                A.ml[to * 2] = top;
                A.ml[to * 2 + 1] = sum;
            }
            continue;
        }
        if (ch >= P.vd) continue;
        if (A.sinks) {
            const float sink = A.sinks[hd] * 1.44269504f;
            const float to = fmaxf(base, sink), f = __builtin_amdgcn_exp2f(base - to);
            sum = fmaf(sum, f, __builtin_amdgcn_exp2f(sink - to));
            o *= f;
        }
        const float y = top == -__builtin_inff() ? 0.0f : o / sum;
        const int64_t to = token * A.o_stride + (int64_t)hd * P.vd + ch;
        if (F32)
            ((float *)A.out)[to] = y;
        else
            ((uint16_t *)A.out)[to] = f32_to_bf16(y);
    }
}

// Prompts and longer chunks: tiles of up to 128 rows (tokens x query heads of one kv
// head), 32 per wave, whose keys and values the workgroup unpacks once per 64 cached
// tokens into LDS: K as halves [token][channel], V as halves [channel][token] times
// 2^E, where E keeps the largest |d| of the steps so far at 2^12.  Scores are
// 32x32x16 products K q^T, so that a lane holds one row's p against 16 tokens of each
// 32 and feeds them to V^T p without leaving its registers: V's tokens lie in LDS in
// the order (quads 0 2 1 3 of 16) in which the scores come.  LDS holds two steps: one
// is unpacked while the other is worked on, with one barrier per step (one step of f32
// rows from 128 channels on, so that two workgroups fit a CU).  For f32 rows q, K, p
// and V are two halves each and the products of their small parts are left out (2^-22
// of the result).
//
// What bounds it: a wave's step of 32 rows x 64 tokens x 128 channels (bf16) is 32
// products of 32 clocks and about 370 VALU instructions, 147 of them for the softmax
// (32 exponentials at a quarter of the rate) and 142 for unpacking, and the two add up
// also across the waves of a SIMD: 2900 clocks by the counters' busy cycles, 3020
// measured.  Eight waves that share the unpacking (half per wave) waited longer at the
// barrier than that saved: 92 us for a mixed step of 64-channel heads, 84 with four.
__host__ __device__ constexpr int paged_tiles_per_cu(int G) { return G == 8 ? 1 : G == 4 ? 2 : 3; }
template <int G, bool F32>
__global__ __launch_bounds__(256, paged_tiles_per_cu(G)) void paged_attn_tile_kernel(PagedDev P, PagedAttn A) {
    constexpr int DV = 32 * G, N = F32 ? 2 : 1, NB = G >= 4 && F32 ? 1 : 2;
    __shared__ half8v s_k[NB][N][64 * DV / 8], s_v[NB][N][DV * 64 / 8];
    __shared__ uint32_t s_most[2][4], s_page[2][4];
    __shared__ uint8_t s_bad[2][64][G];
    // Row r's 16-byte piece c lies at r * pieces + (c ^ h(r)): the 16 rows that a
    // quarter wave reads at one c, and the 4 x 4 (row, piece) it writes, fall on
    // different banks.
    auto k_at = [](int r, int c) __attribute__((always_inline)) {
        const int h = G == 2 ? ((r >> 1) & 1) << 2 | ((r >> 2) & 3) : (r & 3) << 2 | ((r >> 2) & 3);
        return r * (DV / 8) + (c ^ h);
    };
    auto v_at = [](int r, int c) __attribute__((always_inline)) { return r * 8 + (c ^ ((r >> 1) & 7)); };
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int heads_y = P.n_kv * A.n_chunk, n_tiles = (int)(gridDim.x / (uint32_t)heads_y);
    const int x = (int)(blockIdx.x / (uint32_t)heads_y), head_y = (int)blockIdx.x - x * heads_y;
    const int kvh = A.n_chunk == 1 ? head_y : head_y / A.n_chunk, h0 = A.n_chunk == 1 ? 0 : head_y % A.n_chunk * 16;
    const bool last = A.kv_mul - h0 < 16;
    const int heads = last ? A.kv_mul - h0 : 16, inv = last ? A.inv : A.inv16;
    PagedTile T;
    // later tiles of a prompt see more keys: they start first
    if (!paged_tile(P, A, n_tiles - 1 - x, &T)) return;
    const int seq = T.seq, tok = T.tok, n_tok = T.n, row0 = T.row0, pos0 = T.pos0;
    const PagedRange rg = paged_range(P, A, pos0, n_tok);
    const int split = blockIdx.y;
    int per = A.split_steps;
    if ((int64_t)per * A.n_splits < rg.steps) per = (rg.steps + A.n_splits - 1) / A.n_splits;
    const int64_t s_at = (int64_t)split * per;
    const int s_lo = (int)(s_at < rg.steps ? s_at : rg.steps);
    const int s_hi = s_lo + per < rg.steps ? s_lo + per : rg.steps;
    const int64_t head_off = (int64_t)kvh * P.block;

    // a wave unpacks the 16-token tile wave of each step; lane j looks up where it lies
    // in step j of the next 64
    uint64_t where = 0, ok = 0;
    int off_tok = 0;
    auto look = [&](int s) __attribute__((always_inline)) {
        const int t = rg.first + (s + lane) * 64 + 16 * wave;
        const bool in = s + lane < s_hi && t < rg.hi;
        int off = 0;
        const int page = in ? paged_page(P, seq, t, &off) : -1;
        off_tok = page < 0 ? 0 : off;
        where = (uint64_t)(page < 0 ? 0 : page) * (uint64_t)(P.n_kv * P.block) + (uint64_t)head_off;
        ok = __ballot(page >= 0);
    };
    uint32_t kr[G], vr[G], kd[G / 2], vd[2 * G];  // a step as it is stored: codes and scales of keys and values
    bool here = false;
    const int kt = lane >> 2, kc = lane & 3, quad = lane >> 4, vc = lane & 15;
    auto load = [&](int s) __attribute__((always_inline)) {
        const int l = (s - s_lo) & 63;
        const uint64_t at = lane_u64(where, l);
        const uint32_t off = (uint32_t)__builtin_amdgcn_readlane(off_tok, l), sc = (uint32_t)P.ps * (16 * G);
        here = (ok >> l) & 1;
        __builtin_memcpy(kr, P.k + at + (uint32_t)((off + kt) * (16 * G) + kc * (4 * G)), 4 * G);
        __builtin_memcpy(kd, P.k + at + sc + (off + kt) * (2 * G), 2 * G);
        __builtin_memcpy(vr, P.v + at + (uint32_t)(off * (16 * G) + quad * (64 * G) + vc * (4 * G)), 4 * G);
        __builtin_memcpy(vd, P.v + at + sc + (off + 4 * quad) * (2 * G), 8 * G);
    };
    if (s_lo < s_hi) {
        look(s_lo);
        load(s_lo);
    }

    // this lane's row and its queries: B[k = 8 half + .][n = col] of each 16 channels
    const int row = 32 * wave + col, my_tok = row * inv >> 16, my_head = row - my_tok * heads;
    const bool on = my_tok < n_tok;
    const int my_pos = pos0 + my_tok;
    int rhi = on ? my_pos + 1 : 0, rlo = A.window > 0 && my_pos - A.window + 1 > 0 ? my_pos - A.window + 1 : 0;
    if (rhi > rg.hi) rhi = rg.hi;
    half8v q[N][2 * G];
    float qf;
    {
        float v[2 * G][8], big = 0.0f;
        const int64_t from = (int64_t)(row0 + tok + (on ? my_tok : 0)) * A.q_stride +
                             (int64_t)(kvh * A.kv_mul + h0 + my_head) * P.hd;
#pragma unroll
        for (int k = 0; k < 2 * G; k++) {
            const int ch = 16 * k + 8 * half, c = ch < P.hd ? ch : 0;
            if (F32) {
                row_load4((const float *)A.q + from + c, v[k]);
                row_load4((const float *)A.q + from + c + 4, v[k] + 4);
            } else {
                row_load4((const uint16_t *)A.q + from + c, v[k]);
                row_load4((const uint16_t *)A.q + from + c + 4, v[k] + 4);
            }
        }
#pragma unroll
        for (int k = 0; k < 2 * G; k++) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                v[k][j] = on && 16 * k + 8 * half < P.hd ? v[k][j] : 0.0f;
                big = fmaxf(big, fabsf(v[k][j]));
            }
        }
        big = fmaxf(big, __shfl_xor(big, 32, 64));
        int e = 0;
        if (big > 0.0f && big < __builtin_inff()) (void)frexpf(big, &e);
        // qf > 0, so that a maximum of products is one of scores
        qf = fmaxf(fabsf(A.scale) * ldexpf(1.0f, e), 1.17549435e-38f);
        const float down = ldexpf(1.0f, -(e >> 1)), sign = A.scale > 0.0f ? 1.0f : A.scale < 0.0f ? -1.0f : 0.0f;
        const float more = ldexpf(sign, -(e - (e >> 1)));
        const int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for (int k = 0; k < 2 * G; k++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = v[k][order[j]] * down * more;
                q[0][k][j] = (_Float16)y;
                if (F32) q[N - 1][k][j] = (_Float16)(y - (float)q[0][k][j]);
            }
    }

    float m = -__builtin_inff(), l = 0.0f;
    int E = 0;
    uint32_t limit = 0;  // the half's bits of the largest |d| that E holds
    f32x16v acc[G];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < 16; i++) acc[g][i] = 0.0f;
    const int full_lo = rg.lo + (A.window > 0 ? n_tok - 1 : 0), full_hi = rg.hi - (n_tok - 1);
    const PagedMagic magic;

    // Before the barrier in front of a step's unpacking: the values' scales that no
    // row sees become 0, the largest of the others and the page's presence are told.
    auto tell = [&](int s) __attribute__((always_inline)) {
        const int t0 = rg.first + s * 64 + 16 * wave;
        if (!(t0 >= rg.lo && t0 + 16 <= rg.hi && here)) {
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const int t = t0 + 4 * quad + r;
                const bool out = t < rg.lo || t >= rg.hi || !here;
#pragma unroll
                for (int g = 0; g < G; g++) {
                    const int e = r * G + g;
                    vd[e >> 1] &= out ? (e & 1 ? 0x0000FFFFu : 0xFFFF0000u) : 0xFFFFFFFFu;
                }
            }
        }
        typedef uint16_t u16x2v __attribute__((ext_vector_type(2)));
        u16x2v top = {0, 0};
#pragma unroll
        for (int j = 0; j < 2 * G; j++) {
            const uint32_t a = vd[j] & 0x7FFF7FFFu;
            top = __builtin_elementwise_max(top, __builtin_bit_cast(u16x2v, a));
        }
        uint32_t most = top[0] > top[1] ? top[0] : top[1];
        if (__ballot(most > limit)) {
            for (int o = 32; o > 0; o >>= 1) {
                const uint32_t y = (uint32_t)__shfl_xor((int)most, o, 64);
                most = most > y ? most : y;
            }
        }
        if (lane == 0) {
            s_most[s & 1][wave] = most;
            s_page[s & 1][wave] = here ? 1u << wave : 0u;
        }
    };
    // Behind it: E and the pages of the step.  True where some scales are NaN or
    // infinite.
    uint32_t pages = 0, pages_next = 0;  // a bit per 16-token tile
    auto decide = [&](int s, int *e_new) __attribute__((always_inline)) {
        const uint32_t *pg = s_page[s & 1];
        pages_next = (uint32_t)uniform((int)(pg[0] | pg[1] | pg[2] | pg[3]));
        uint32_t top = s_most[s & 1][0];
#pragma unroll
        for (int w = 1; w < 4; w++) top = top > s_most[s & 1][w] ? top : s_most[s & 1][w];
        top = (uint32_t)uniform((int)top);
        *e_new = E;
        if (top <= limit) return false;
        const bool bad = top >= 0x7C00u;
        if (bad) top = 0x7BFFu;
        if (top > limit) {
            // |d| < 2^e, |d| 2^E <= 2^12, |d (c - 8)| 2^E <= 2^15
            int e;
            (void)frexpf(h2f((uint16_t)top), &e);
            *e_new = 12 - e < 30 ? 12 - e : 30;
            limit = e < 15 ? (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)ldexpf(1.0f, e)) : 0x7BFFu;
        }
        return bad;
    };
    auto unpack = [&](int s, int b, int e_new, bool bad) __attribute__((always_inline)) {
        {  // token kt's channels 32 g + 8 kc ..
            const int t = 16 * wave + kt;
#pragma unroll
            for (int g = 0; g < G; g++) {
                const _Float16 d = paged_h2(kd[g >> 1])[g & 1];
                const half2v d2 = {d, d};
                // in the order 0 4 1 5 2 6 3 7 of each eight channels, as the queries
                const u32x4v c = __builtin_bit_cast(u32x4v, magic.k8(kr[g]));
                u32x4v hi, lo;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t cj = c[j];
                    const half2v p = paged_h2(cj) * d2;
                    hi[j] = __builtin_bit_cast(uint32_t, p);
                    if (F32) {
                        half2v r;
#pragma unroll
                        for (int y = 0; y < 2; y++) r[y] = (_Float16)fmaf((float)paged_h2(cj)[y], (float)d, -(float)p[y]);
                        lo[j] = __builtin_bit_cast(uint32_t, r);
                    }
                }
                s_k[b][0][k_at(t, 4 * g + kc)] = __builtin_bit_cast(half8v, hi);
                if (F32) s_k[b][N - 1][k_at(t, 4 * g + kc)] = __builtin_bit_cast(half8v, lo);
            }
        }
        {  // quad's four tokens, channels 32 g + vc and 32 g + 16 + vc
            if (bad) {
                // such groups become 0 here and NaN to the rows that see them
#pragma unroll
                for (int r = 0; r < 4; r++)
#pragma unroll
                    for (int g = 0; g < G; g++) {
                        const int e = r * G + g;
                        const bool is = ((vd[e >> 1] >> (16 * (e & 1))) & 0x7FFFu) >= 0x7C00u;
                        if (vc == 0) s_bad[s & 1][16 * wave + 4 * quad + r][g] = is;
                        vd[e >> 1] &= is ? (e & 1 ? 0x0000FFFFu : 0xFFFF0000u) : 0xFFFFFFFFu;
                    }
            }
            // d 2^E in two exact steps (E - E / 2 <= 15)
            const _Float16 u1 = (_Float16)ldexpf(1.0f, e_new / 2), u2 = (_Float16)ldexpf(1.0f, e_new - e_new / 2);
            const half2v up1 = {u1, u1}, up2 = {u2, u2};
            uint32_t dv[2 * G];
#pragma unroll
            for (int j = 0; j < 2 * G; j++) dv[j] = __builtin_bit_cast(uint32_t, paged_h2(vd[j]) * up1 * up2);
            const int piece = 2 * wave + (quad & 1);
#pragma unroll
            for (int g = 0; g < G; g++) {
                uint32_t hi[2][2], lo[2][2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const int b0 = 2 * h * G + g, b1 = (2 * h + 1) * G + g;
                    const uint32_t w = __builtin_amdgcn_perm(vr[b1 >> 2], vr[b0 >> 2],
                                                             0x0C000C00u | (uint32_t)(b0 & 3) |
                                                                 (uint32_t)(4 + (b1 & 3)) << 16);
                    const half2v dd = paged_h2(__builtin_amdgcn_perm(dv[b1 >> 1], dv[b0 >> 1],
                                                                     (b0 & 1 ? 0x0302u : 0x0100u) |
                                                                         (b1 & 1 ? 0x07060000u : 0x05040000u)));
                    const uint32_t cw[2] = {magic.low(w), magic.high(w)};
#pragma unroll
                    for (int n = 0; n < 2; n++) {
                        const half2v c = paged_h2(cw[n]), y = c * dd;
                        hi[n][h] = __builtin_bit_cast(uint32_t, y);
                        if (F32) {
                            half2v r;
                            r[0] = (_Float16)fmaf((float)c[0], (float)dd[0], -(float)y[0]);
                            r[1] = (_Float16)fmaf((float)c[1], (float)dd[1], -(float)y[1]);
                            lo[n][h] = __builtin_bit_cast(uint32_t, r);
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < 2; n++) {
                    const int at = v_at(32 * g + 16 * n + vc, piece);
                    ((uint2 *)&s_v[b][0][at])[quad >> 1] = make_uint2(hi[n][0], hi[n][1]);
                    if (F32) ((uint2 *)&s_v[b][N - 1][at])[quad >> 1] = make_uint2(lo[n][0], lo[n][1]);
                }
            }
        }
    };
    // the load behind a step's unpacking (the last step's is not used)
    auto load_next = [&](int s) __attribute__((always_inline)) {
        if (((s - s_lo) & 63) == 0 && s < s_hi) look(s);
        load(s < s_hi ? s : s_hi - 1);
    };

    bool bad = false, bad_next = false;
    int e_next = 0;
    if (s_lo < s_hi) {
        tell(s_lo);
        __syncthreads();
        bad = decide(s_lo, &E);
        unpack(s_lo, s_lo & (NB - 1), E, bad);
        load_next(s_lo + 1);
    }
    for (int s = s_lo; s < s_hi; s++) {
        const int t0 = rg.first + s * 64, b = s & (NB - 1);
        const bool more = s + 1 < s_hi;
        if (NB == 2 && more) tell(s + 1);
        __syncthreads();  // step s is in LDS; nobody reads step s - 1 any more
        pages = pages_next;
        const bool full = t0 >= full_lo && t0 + 64 <= full_hi && pages == 15;
        e_next = E;
        if (NB == 2 && more) bad_next = decide(s + 1, &e_next);

        // scores of 64 tokens: [32-token tile][16]
        f32x16v sc[2];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) sc[u][i] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2 * G; k++)
#pragma unroll
            for (int u = 0; u < 2; u++) {
                const half8v a = s_k[b][0][k_at(32 * u + col, 2 * k + half)];
                sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[0][k], sc[u], 0, 0, 0);
                if (F32) {
                    const half8v c = s_k[b][N - 1][k_at(32 * u + col, 2 * k + half)];
                    sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q[N - 1][k], sc[u], 0, 0, 0);
                    sc[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(c, q[0][k], sc[u], 0, 0, 0);
                }
            }
        if (NB == 2 && more) {
            unpack(s + 1, b ^ 1, e_next, bad_next);
            load_next(s + 2);
        }
        if (!full) {
            const float none = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < 2; u++)
#pragma unroll
                for (int i = 0; i < 16; i++) {
                    const int t = t0 + 32 * u + 8 * (i >> 2) + 4 * half + (i & 3);
                    const bool in = (t >= rlo) & (t < rhi) & ((pages >> (2 * u + (i >> 3))) & 1);
                    sc[u][i] = in ? sc[u][i] : none;
                }
        }
        float mx = sc[0][0];
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int i = 0; i < 16; i++) mx = fmaxf(mx, sc[u][i]);
        mx *= qf;
        // m follows the maximum only when it is 8 behind: p 2^6 stays at or below 2^14,
        // and keeps all its bits as a half down to 2^-28 of that
        if (__ballot(mx > m + 8.0f || (m == -__builtin_inff() && mx > m))) {
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            mx = fmaxf(mx, m);
            const float a = m == -__builtin_inff() ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
            m = mx;
            l *= a;
#pragma unroll
            for (int g = 0; g < G; g++) acc[g] *= a;
        }
        const float base = (m == -__builtin_inff() ? 0.0f : m) - 6.0f;
        float l4[4] = {0, 0, 0, 0};
#pragma unroll
        for (int c = 0; c < 4; c++) {
            half8v ph, pl;
#pragma unroll
            for (int i = 0; i < 8; i++) {
                const float p = __builtin_amdgcn_exp2f(fmaf(sc[c >> 1][8 * (c & 1) + i], qf, -base));
                l4[i & 3] += p;
                ph[i] = (_Float16)p;
                if (F32) pl[i] = (_Float16)(p - (float)(_Float16)p);
            }
#pragma unroll
            for (int g = 0; g < G; g++) {
                const half8v a = s_v[b][0][v_at(32 * g + col, 2 * c + half)];
                acc[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, ph, acc[g], 0, 0, 0);
                if (F32) {
                    const half8v d = s_v[b][N - 1][v_at(32 * g + col, 2 * c + half)];
                    acc[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, pl, acc[g], 0, 0, 0);
                    acc[g] = __builtin_amdgcn_mfma_f32_32x32x16_f16(d, ph, acc[g], 0, 0, 0);
                }
            }
        }
        l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
        if (bad) {
#pragma unroll 1
            for (int g = 0; g < G; g++) {
                bool sees = false;
#pragma unroll 1
                for (int k = 0; k < 64; k++) sees |= s_bad[s & 1][k][g] && t0 + k >= rlo && t0 + k < rhi;
                const float add = sees ? __builtin_nanf("") : 0.0f;
#pragma unroll
                for (int h = 0; h < G; h++) acc[h] += h == g ? add : 0.0f;
            }
        }
        if (NB == 1 && more) {
            tell(s + 1);
            __syncthreads();
            bad_next = decide(s + 1, &e_next);
            unpack(s + 1, 0, e_next, bad_next);
            load_next(s + 2);
        }
        if (e_next != E) {
            const float a = ldexpf(1.0f, e_next - E);
#pragma unroll
            for (int g = 0; g < G; g++) acc[g] *= a;
            E = e_next;
        }
        bad = bad_next;
    }

    l += __shfl_xor(l, 32, 64);
    l *= 1.0f / 64.0f;
    if (l != l) m = __builtin_inff();  // as in the row tiles
    if (!on) return;
    const float unit = ldexpf(1.0f, -E - 6);
    // the arguments used from here on are read here: kept through the loop, they
    // pushed others out of the scalar registers (25 lane reads per step)
    static_assert(sizeof(PagedDev) % alignof(PagedAttn) == 0, "the second argument follows the first");
    typedef __attribute__((address_space(4))) const uint8_t kernarg_t;
    kernarg_t *args = (kernarg_t *)__builtin_amdgcn_kernarg_segment_ptr() + sizeof(PagedDev);
    asm volatile("" : "+s"(args));
    const auto &B = *(__attribute__((address_space(4))) const PagedAttn *)args;
    const int hd = kvh * B.kv_mul + h0 + my_head;
    const int64_t token = row0 + tok + my_tok;
    const bool none = m == -__builtin_inff();
    if (B.n_splits > 1) {
        const int64_t to = ((int64_t)split * P.n_tokens + token) * B.n_heads + hd;
        if (half == 0) {
            B.ml[to * 2] = m;
            B.ml[to * 2 + 1] = l;
        }
        if (!none)
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const float y[4] = {acc[g][i] * unit, acc[g][i + 1] * unit, acc[g][i + 2] * unit, acc[g][i + 3] * unit};
                    row_store4(B.part + to * DV + 32 * g + 2 * i + 4 * half, y);
                }
        return;
    }
    float f = none ? 0.0f : unit / l;
    if (B.sinks && !none) {
        const float sink = B.sinks[hd] * 1.44269504f, top = fmaxf(m, sink), a = __builtin_amdgcn_exp2f(m - top);
        f = unit * a / fmaf(l, a, __builtin_amdgcn_exp2f(sink - top));
    }
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {
            const int ch = 32 * g + 2 * i + 4 * half;
            if (ch >= P.vd) continue;
            const float y[4] = {none ? 0.0f : acc[g][i] * f, none ? 0.0f : acc[g][i + 1] * f,
                                none ? 0.0f : acc[g][i + 2] * f, none ? 0.0f : acc[g][i + 3] * f};
            const int64_t to = token * B.o_stride + (int64_t)hd * P.vd + ch;
            if (F32)
                row_store4((float *)B.out + to, y);
            else
                row_store4((uint16_t *)B.out + to, y);
        }
}

// Joins the splits of the sessions that are row tiles.  One workgroup per (session,
// row of it, query head): the splits' weights first, then each of 256 / DV groups of
// threads sums every so-manieth split, eight loads in flight, and the groups' sums
// are added in their order.  Its loads' latency bounds it (one row of 32 heads in 94
// parts: 8.1 us; 48 rows in two: 5.0).
template <int G, bool F32>
__global__ __launch_bounds__(256) void paged_attn_join_rows_kernel(PagedDev P, PagedAttn A) {
    constexpr int DV = 32 * G, N = 256 / DV;
    __shared__ float s_f[256], s_o[N][DV], s_red[4];
    const uint32_t r = blockIdx.x / (uint32_t)A.n_heads;
    const int hd = (int)(blockIdx.x - r * (uint32_t)A.n_heads);
    const int seq = (int)(r / (uint32_t)A.short_q), tk = (int)(r - (uint32_t)seq * (uint32_t)A.short_q);
    const int a = P.q_starts[seq], b = P.q_starts[seq + 1];
    if (a < 0 || b > P.n_tokens || tk >= b - a || (A.both && b - a > A.short_q)) return;
    const int64_t rows = (int64_t)P.n_tokens * A.n_heads, token = a + tk, w = token * A.n_heads + hd;
    const int i = threadIdx.x;  // at most 256 splits
    float m = -__builtin_inff(), part = 0.0f;
    if (i < A.n_splits) {
        m = A.ml[(i * rows + w) * 2];
        part = A.ml[(i * rows + w) * 2 + 1];
    }
    const float top = block_max_256(m, s_red);
    const bool none = top == -__builtin_inff();
    float base = none ? 0.0f : top, sink = 0.0f;
    if (A.sinks) {
        sink = A.sinks[hd] * 1.44269504f;
        base = none ? sink : fmaxf(base, sink);
        sink = __builtin_amdgcn_exp2f(sink - base);
    }
    const float f = m == -__builtin_inff() ? 0.0f : __builtin_amdgcn_exp2f(m - base);
    s_f[i] = f;
    const float sum = block_sum_256(f == 0.0f ? 0.0f : f * part, s_red) + sink;  // the barriers order s_f too
    const int ch = i % DV;
    float o[4] = {0, 0, 0, 0};
    for (int s = i / DV; s < A.n_splits; s += 8 * N) {
        float x[8], f8[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int at = s + j * N < A.n_splits ? s + j * N : 0;
            f8[j] = s + j * N < A.n_splits ? s_f[at] : 0.0f;
            x[j] = A.part[(at * rows + w) * DV + ch];
        }
#pragma unroll
        for (int j = 0; j < 8; j++)  // a split without keys wrote no sums
            o[j & 3] = f8[j] != 0.0f ? fmaf(f8[j], x[j], o[j & 3]) : o[j & 3];
    }
    s_o[i / DV][ch] = (o[0] + o[1]) + (o[2] + o[3]);
    __syncthreads();
    if (i >= DV || ch >= P.vd) return;
    float y = s_o[0][ch];
#pragma unroll
    for (int j = 1; j < N; j++) y += s_o[j][ch];
    y = none ? 0.0f : y / sum;
    const int64_t to = token * A.o_stride + (int64_t)hd * P.vd + ch;
    if (F32)
        ((float *)A.out)[to] = y;
    else
        ((uint16_t *)A.out)[to] = f32_to_bf16(y);
}

// The same for the rows of larger tiles, of which there are many with few splits:
// one wave per (row, four query heads), their loads in flight together (512 rows of 32
// heads of 128 channels in two f32 parts: 7.4 us, in four 10.4).
template <int G, bool F32>
__global__ __launch_bounds__(256) void paged_attn_join_tiles_kernel(PagedDev P, PagedAttn A) {
    constexpr int DV = 32 * G, N = DV / 64, H = 4;
    const int lane = threadIdx.x & 63;
    const int64_t rows = (int64_t)P.n_tokens * A.n_heads, w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int groups = (A.n_heads + H - 1) / H;
    const int token = (int)(w / groups), hd = (int)(w - (int64_t)token * groups) * H;
    if (token >= P.n_tokens) return;
    int seq, a, b;
    // rows of no session stay as they are
    if (!paged_session(P, token, &seq, &a, &b) || (A.both && b - a <= A.short_q)) return;
    int64_t at[H];
    float top[H], base[H], sum[H], o[H][N];
#pragma unroll
    for (int h = 0; h < H; h++) {
        at[h] = (int64_t)token * A.n_heads + (hd + h < A.n_heads ? hd + h : hd);
        top[h] = -__builtin_inff();
    }
    for (int s = 0; s < A.n_splits; s++)
#pragma unroll
        for (int h = 0; h < H; h++) top[h] = fmaxf(top[h], A.ml[(s * rows + at[h]) * 2]);
#pragma unroll
    for (int h = 0; h < H; h++) {
        base[h] = top[h] == -__builtin_inff() ? 0.0f : top[h];
        sum[h] = 0.0f;
        if (A.sinks) {
            const float sink = A.sinks[hd + h < A.n_heads ? hd + h : hd] * 1.44269504f;
            base[h] = top[h] == -__builtin_inff() ? sink : fmaxf(top[h], sink);
            sum[h] = __builtin_amdgcn_exp2f(sink - base[h]);
        }
#pragma unroll
        for (int n = 0; n < N; n++) o[h][n] = 0.0f;
    }
    for (int s = 0; s < A.n_splits; s++) {
        float x[H][N], m[H], l[H];
#pragma unroll
        for (int h = 0; h < H; h++) {
            m[h] = A.ml[(s * rows + at[h]) * 2];
            l[h] = A.ml[(s * rows + at[h]) * 2 + 1];
#pragma unroll
            for (int n = 0; n < N; n++) x[h][n] = A.part[(s * rows + at[h]) * DV + lane + 64 * n];
        }
#pragma unroll
        for (int h = 0; h < H; h++) {
            // a split without keys wrote no sums
            const bool has = m[h] != -__builtin_inff();
            const float f = has ? __builtin_amdgcn_exp2f(m[h] - base[h]) : 0.0f;
            sum[h] = has ? fmaf(f, l[h], sum[h]) : sum[h];
#pragma unroll
            for (int n = 0; n < N; n++) o[h][n] = has ? fmaf(f, x[h][n], o[h][n]) : o[h][n];
        }
    }
#pragma unroll
    for (int h = 0; h < H; h++)
#pragma unroll
        for (int n = 0; n < N; n++) {
            const int ch = lane + 64 * n;
            if (ch >= P.vd || hd + h >= A.n_heads) continue;
            const float y = top[h] == -__builtin_inff() ? 0.0f : o[h][n] / sum[h];
            const int64_t to = token * A.o_stride + (int64_t)(hd + h) * P.vd + ch;
            if (F32)
                ((float *)A.out)[to] = y;
            else
                ((uint16_t *)A.out)[to] = f32_to_bf16(y);
        }
}

}  // namespace rh

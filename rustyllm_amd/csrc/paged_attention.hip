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

struct PagedAttn {
    const void *q;
    void *out;
    const float *sinks;  // [n_heads] or null
    float *part;         // [split][token][head][32 G] sums, or null with one split
    float *ml;           // [split][token][head][2]: maximum (base 2) and sum
    int64_t q_stride, o_stride;
    float scale;         // times log2(e)
    int32_t n_heads, kv_mul, window;
    int32_t tok_tile;    // tokens of a row tile
    int32_t n_splits;    // most splits of a row tile's range
    int32_t split_steps; // 64-token steps of a split, more where n_splits would not cover the range
    int32_t by_seq;      // 1: tile x is session x (at most one tile each)
};

// Row tile x of the batch: its session, first token (of the session) and tokens.
// Wave-uniform; 64 sessions per turn, each lane one session's tile count.
__device__ __forceinline__ bool paged_tile(const PagedDev &P, const PagedAttn &A, int x, int *seq, int *tok,
                                           int *n) {
    const int lane = threadIdx.x & 63;
    if (A.by_seq) {
        *seq = x;
        *tok = 0;
    } else {
        int before = 0, found = -1;
        for (int base = 0; base < P.n_seqs; base += 64) {
            const int i = base + lane;
            int c = 0;
            if (i < P.n_seqs) {
                const int64_t len = (int64_t)P.q_starts[i + 1] - P.q_starts[i];
                c = len > 0 && len <= P.n_tokens ? ((int)len + A.tok_tile - 1) / A.tok_tile : 0;
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
                found = base + l;
                *tok = (x - before - __shfl(sum - c, l, 64)) * A.tok_tile;
                break;
            }
            before += __shfl(sum, 63, 64);
        }
        if (found < 0) return false;
        *seq = found;
    }
    const int a = P.q_starts[*seq], b = P.q_starts[*seq + 1];
    if (a < 0 || b > P.n_tokens || *tok < 0 || b - a <= *tok) return false;
    *n = b - a - *tok < A.tok_tile ? b - a - *tok : A.tok_tile;
    return true;
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

// 8 codes of a K dword as exact halves c - 8, in the order nibble 0 4 1 5 2 6 3 7:
// or-ing a nibble into 1024 (bits 0..3) or 64 (bits 4..7) makes the half 1024 + c
// or 64 + c, so the dword needs one shift.
__device__ __forceinline__ half8v paged_k8(uint32_t w) {
    const half2v a = {(_Float16)-1032.0f, (_Float16)-1032.0f}, b = {(_Float16)-72.0f, (_Float16)-72.0f};
    u32x4v r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (w & 0x000F000Fu) | 0x64006400u) + a);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (w & 0x00F000F0u) | 0x54005400u) + b);
    w >>= 8;
    r[2] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (w & 0x000F000Fu) | 0x64006400u) + a);
    r[3] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(half2v, (w & 0x00F000F0u) | 0x54005400u) + b);
    return __builtin_bit_cast(half8v, r);
}

// bf16 pair (round to nearest even), low half first.
__device__ __forceinline__ uint32_t paged_bf16x2(float a, float b) {
    typedef __bf16 bf16x2v __attribute__((ext_vector_type(2)));
    bf16x2v r = {(__bf16)a, (__bf16)b};
    return __builtin_bit_cast(uint32_t, r);
}

template <int CTRL>
__device__ __forceinline__ float paged_dpp(float v) {
    return __builtin_bit_cast(float, dpp_i<CTRL>(__builtin_bit_cast(int, v)));
}

// Row tiles of at most R = 4, 8 or 16 rows (tokens x query heads of one kv head):
// single tokens, and short runs of them.
//
// The 16 columns of a 16x16x32 product hold 16 / R copies of the rows, copy i for
// the i-th of 16 / R tiles of 16 tokens: copy i's queries are zero in the other
// columns, so the products of all tiles accumulate in one result whose lane
// (column n, quarter c) holds the scores of row n % R against tokens 4 c + r of
// tile n / R.  No lane's softmax work is spent on padding.  K codes stay integers:
// each group's product is scaled by d of its (token, group) in f32.  For V the
// scale goes into p (p d rounded to bf16, for f32 outputs in two terms), and the
// codes are bf16 128 + c with a product against the constant -136 before each, so
// the large offset never outlives a tile.
template <int G, int R, bool F32>
__global__ __launch_bounds__(256, G == 8 ? 1 : 2) void paged_attn_rows_kernel(PagedDev P, PagedAttn A) {
    constexpr int NT = 16 / R;  // token tiles per score result
    constexpr int NU = 4 / NT;  // score results per 64-token step
    constexpr int DV = 32 * G;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, quad = lane >> 4;
    const int n_chunk = (A.kv_mul + 15) / 16;  // kv_mul > 16: 16 query heads at a time
    const int kvh = blockIdx.y / n_chunk, h0 = (blockIdx.y % n_chunk) * 16;
    const int heads = A.kv_mul - h0 < 16 ? A.kv_mul - h0 : 16;
    const int split = blockIdx.z;
    int seq, tok, n_tok;
    if (!paged_tile(P, A, blockIdx.x, &seq, &tok, &n_tok)) return;
    const int row0 = P.q_starts[seq];
    const int64_t pos_end = P.kv_lens[seq];
    const int64_t pos0l = pos_end - (P.q_starts[seq + 1] - row0) + tok;  // position of the tile's first token
    const int pos0 = (int)(pos0l < -(1 << 30) ? -(1 << 30) : pos0l);
    const PagedRange rg = paged_range(P, A, pos0, n_tok);

    // this lane's row: token and head of column col
    const int row = col % R, my_tok = row / heads, my_head = row % heads;
    const bool on = my_tok < n_tok;
    const int my_pos = pos0 + my_tok;
    int rhi = on ? my_pos + 1 : 0, rlo = A.window > 0 && my_pos - A.window + 1 > 0 ? my_pos - A.window + 1 : 0;
    if (rhi > rg.hi) rhi = rg.hi;

    // queries: f16 of q 2^-e with 2^e above the row's largest (and the rest of it in
    // a second f16 for f32 inputs, 22 bits in all), zero in the other tiles' columns
    half8v qh[NT][G], ql[F32 ? NT : 1][F32 ? G : 1];
    float qf;
    {
        float x[G][8], big = 0.0f;
        const int64_t at = (int64_t)(row0 + tok + my_tok) * A.q_stride + (int64_t)(kvh * A.kv_mul + h0 + my_head) * P.hd;
#pragma unroll
        for (int g = 0; g < G; g++) {
            const int ch = 32 * g + 8 * quad;
#pragma unroll
            for (int j = 0; j < 8; j++) x[g][j] = 0.0f;
            if (on && ch < P.hd) {
                if (F32) {
                    row_load4((const float *)A.q + at + ch, x[g]);
                    row_load4((const float *)A.q + at + ch + 4, x[g] + 4);
                } else {
                    row_load4((const uint16_t *)A.q + at + ch, x[g]);
                    row_load4((const uint16_t *)A.q + at + ch + 4, x[g] + 4);
                }
            }
#pragma unroll
            for (int j = 0; j < 8; j++) big = fmaxf(big, fabsf(x[g][j]));
        }
        big = fmaxf(big, __shfl_xor(big, 16, 64));
        big = fmaxf(big, __shfl_xor(big, 32, 64));
        int e = 0;
        if (big > 0.0f && big < __builtin_inff()) (void)frexpf(big, &e);
        qf = A.scale * ldexpf(1.0f, e);
        const int order[8] = {0, 4, 1, 5, 2, 6, 3, 7};
#pragma unroll
        for (int g = 0; g < G; g++) {
            half8v hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = ldexpf(x[g][order[j]], -e);
                hi[j] = (_Float16)v;
                lo[j] = (_Float16)(v - (float)hi[j]);
            }
            const half8v zero = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < NT; i++) {
                qh[i][g] = col / R == i ? hi : zero;
                if (F32) ql[i][g] = col / R == i ? lo : zero;
            }
        }
    }

    // the splits' and then the waves' share of the steps
    int per = A.split_steps;
    if ((int64_t)per * A.n_splits < rg.steps) per = (rg.steps + A.n_splits - 1) / A.n_splits;
    const int s_lo = split * per < rg.steps ? split * per : rg.steps;
    const int s_hi = s_lo + per < rg.steps ? s_lo + per : rg.steps;

    float m = -__builtin_inff(), l = 0.0f;
    f32x4v acc[G][2];
#pragma unroll
    for (int g = 0; g < G; g++)
#pragma unroll
        for (int h = 0; h < 2; h++) acc[g][h] = f32x4v{0, 0, 0, 0};
    u32x4v bias_u = {0xC308C308u, 0xC308C308u, 0xC308C308u, 0xC308C308u};
    const bf16x8v bias = __builtin_bit_cast(bf16x8v, bias_u);

    // rows whose masks the whole step passes need no masking
    const int full_lo = rg.lo + (A.window > 0 ? n_tok - 1 : 0), full_hi = rg.hi - (n_tok - 1);
    const uint32_t k_lane = (uint32_t)((lane & 15) * 16 * G + quad * 4 * G);
    const uint32_t v_lane = (uint32_t)(quad * 64 * G + (lane & 15) * 4 * G);
    const int64_t head_off = (int64_t)kvh * P.block, page_bytes = (int64_t)P.n_kv * P.block;

    for (int s = s_lo + wave; s < s_hi; s += 4) {
        const int t0 = rg.first + s * 64;
        uint32_t kc[4][G], vc[4][G], ks[NU][2 * G], vs[NU][2 * G];
        int pg[4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int t = t0 + 16 * i;
            pg[i] = t < rg.hi ? __builtin_amdgcn_readfirstlane(paged_page(P, seq, t)) : -1;
            const int64_t at = (int64_t)(pg[i] < 0 ? 0 : pg[i]) * page_bytes + head_off + (int64_t)(t % P.ps) * (16 * G);
            __builtin_memcpy(kc[i], P.k + at + k_lane, 4 * G);
            __builtin_memcpy(vc[i], P.v + at + v_lane, 4 * G);
        }
#pragma unroll
        for (int u = 0; u < NU; u++) {
            int page = pg[u * NT];
#pragma unroll
            for (int i = 1; i < NT; i++) page = col / R == i ? pg[u * NT + i] : page;
            const int t = t0 + 16 * (u * NT + col / R) + 4 * quad;
            const int64_t at = (int64_t)(page < 0 ? 0 : page) * page_bytes + head_off + (int64_t)P.ps * (16 * G) +
                               (int64_t)(t % P.ps) * (2 * G);
            __builtin_memcpy(ks[u], P.k + at, 8 * G);
            __builtin_memcpy(vs[u], P.v + at, 8 * G);
        }
        const bool full = t0 >= full_lo && t0 + 64 <= full_hi && pg[0] >= 0 && pg[1] >= 0 && pg[2] >= 0 && pg[3] >= 0;

        // scores
        float sc[NU][4];
        float mx = -__builtin_inff();
#pragma unroll
        for (int u = 0; u < NU; u++) {
#pragma unroll
            for (int r = 0; r < 4; r++) sc[u][r] = 0.0f;
#pragma unroll
            for (int g = 0; g < G; g++) {
                f32x4v d = {0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < NT; i++) {
                    const half8v k8 = paged_k8(kc[u * NT + i][g]);
                    d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, qh[i][g], d, 0, 0, 0);
                    if (F32) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(k8, ql[i][g], d, 0, 0, 0);
                }
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int e = r * G + g;
                    const float f = h2f((uint16_t)(ks[u][e >> 1] >> (16 * (e & 1))));
                    sc[u][r] = fmaf(f, d[r], sc[u][r]);
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) sc[u][r] *= qf;
            if (!full) {
                int page = pg[u * NT];
#pragma unroll
                for (int i = 1; i < NT; i++) page = col / R == i ? pg[u * NT + i] : page;
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int t = t0 + 16 * (u * NT + col / R) + 4 * quad + r;
                    if (t < rlo || t >= rhi || page < 0) sc[u][r] = -__builtin_inff();
                }
            }
#pragma unroll
            for (int r = 0; r < 4; r++) mx = fmaxf(mx, sc[u][r]);
        }
        if (__ballot(mx > m)) {
            // a row's scores lie in the lanes of all tiles and quarters
            if (NT >= 4) mx = fmaxf(mx, paged_dpp<0x124>(mx));
            if (NT >= 2) mx = fmaxf(mx, paged_dpp<0x128>(mx));
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            mx = fmaxf(mx, m);
            const float a = m == mx ? 1.0f : __builtin_amdgcn_exp2f(m - mx);
            m = mx;
            l *= a;
#pragma unroll
            for (int g = 0; g < G; g++)
#pragma unroll
                for (int h = 0; h < 2; h++) acc[g][h] *= a;
        }
        const float base = m == -__builtin_inff() ? 0.0f : m;
#pragma unroll
        for (int u = 0; u < NU; u++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                sc[u][r] = __builtin_amdgcn_exp2f(sc[u][r] - base);
                l += sc[u][r];
            }

        // values, 32 tokens (two tiles) per product
#pragma unroll
        for (int g = 0; g < G; g++) {
            uint32_t ph[NU][2], pl[NU][2];
#pragma unroll
            for (int u = 0; u < NU; u++) {
                float f[4];
#pragma unroll
                for (int r = 0; r < 4; r++) {
                    const int e = r * G + g;
                    f[r] = sc[u][r] * h2f((uint16_t)(vs[u][e >> 1] >> (16 * (e & 1))));
                    // a masked token's page may hold anything, NaN among it
                    if (!full) f[r] = sc[u][r] == 0.0f ? 0.0f : f[r];
                }
                ph[u][0] = paged_bf16x2(f[0], f[1]);
                ph[u][1] = paged_bf16x2(f[2], f[3]);
                if (F32) {
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const uint32_t w = ph[u][r >> 1];
                        f[r] -= __builtin_bit_cast(float, r & 1 ? w & 0xFFFF0000u : w << 16);
                    }
                    pl[u][0] = paged_bf16x2(f[0], f[1]);
                    pl[u][1] = paged_bf16x2(f[2], f[3]);
                }
            }
#pragma unroll
            for (int k = 0; k < 2; k++) {
                u32x4v bh, bl = {0, 0, 0, 0};
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const int i = (2 * k + x) % NT, u = (2 * k + x) / NT;
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        // copy i's columns to the first R (row_ror by 16 - R i)
                        auto turn = [&](uint32_t v) -> uint32_t {
                            if (i == 0) return v;
                            if (i * R == 4) return (uint32_t)dpp_i<0x12C>((int)v);
                            if (i * R == 8) return (uint32_t)dpp_i<0x128>((int)v);
                            return (uint32_t)dpp_i<0x124>((int)v);
                        };
                        bh[2 * x + h] = turn(ph[u][h]);
                        if (F32) bl[2 * x + h] = turn(pl[u][h]);
                    }
                }
                u32x4v va, vb;
#pragma unroll
                for (int x = 0; x < 2; x++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int b0 = (2 * h) * G + g, b1 = (2 * h + 1) * G + g;
                        const uint32_t w = __builtin_amdgcn_perm(vc[2 * k + x][b1 >> 2], vc[2 * k + x][b0 >> 2],
                                                                 0x0C000C00u | (uint32_t)(b0 & 3) |
                                                                     (uint32_t)(4 + (b1 & 3)) << 16);
                        va[2 * x + h] = (w & 0x000F000Fu) | 0x43004300u;
                        vb[2 * x + h] = ((w >> 4) & 0x000F000Fu) | 0x43004300u;
                    }
                const bf16x8v p8 = __builtin_bit_cast(bf16x8v, bh);
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const bf16x8v v8 = __builtin_bit_cast(bf16x8v, h ? vb : va);
                    acc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bias, p8, acc[g][h], 0, 0, 0);
                    acc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v8, p8, acc[g][h], 0, 0, 0);
                    if (F32) {
                        const bf16x8v l8 = __builtin_bit_cast(bf16x8v, bl);
                        acc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(bias, l8, acc[g][h], 0, 0, 0);
                        acc[g][h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v8, l8, acc[g][h], 0, 0, 0);
                    }
                }
            }
        }
    }

    // the four waves' results through LDS
    if (NT >= 4) l += paged_dpp<0x124>(l);
    if (NT >= 2) l += paged_dpp<0x128>(l);
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
    __shared__ float s_acc[4][R][DV + 4];
    __shared__ float s_m[4][R], s_l[4][R];
    if (col < R) {
        if (quad == 0) {
            s_m[wave][col] = m;
            s_l[wave][col] = l;
        }
#pragma unroll
        for (int g = 0; g < G; g++)
#pragma unroll
            for (int h = 0; h < 2; h++)
                *(f32x4v *)&s_acc[wave][col][32 * g + 16 * h + 4 * quad] = acc[g][h];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < R * DV; i += 256) {
        const int r = i / DV, ch = i % DV;
        const int tk = r / heads, hd = kvh * A.kv_mul + h0 + r % heads;
        if (tk >= n_tok) break;
        float top = fmaxf(fmaxf(s_m[0][r], s_m[1][r]), fmaxf(s_m[2][r], s_m[3][r]));
        const float base = top == -__builtin_inff() ? 0.0f : top;
        float sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][r] - base);
            sum = fmaf(f, s_l[w][r], sum);
            o = fmaf(f, s_acc[w][r][ch], o);
        }
        const int64_t token = row0 + tok + tk;
        if (A.n_splits > 1) {
            const int64_t at = ((int64_t)split * P.n_tokens + token) * A.n_heads + hd;
            if (top != -__builtin_inff()) A.part[at * DV + ch] = o;
            if (ch == 0) {
                A.ml[at * 2] = top;
                A.ml[at * 2 + 1] = sum;
            }
            continue;
        }
        if (ch >= P.vd) continue;
        if (A.sinks) {
            const float sink = A.sinks[hd] * 1.44269504f;
            const float to = fmaxf(base, sink), f = __builtin_amdgcn_exp2f(base - to);
            if (top == -__builtin_inff()) {
                o = 0.0f, sum = 1.0f;
            } else {
                sum = fmaf(sum, f, __builtin_amdgcn_exp2f(sink - to));
                o *= f;
            }
        }
        const float y = top == -__builtin_inff() ? 0.0f : o / sum;
        const int64_t to = token * A.o_stride + (int64_t)hd * P.vd + ch;
        if (F32)
            ((float *)A.out)[to] = y;
        else
            ((uint16_t *)A.out)[to] = f32_to_bf16(y);
    }
}

// Joins a row's splits in their order.  One wave per (token, query head).
template <int G, bool F32>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedDev P, PagedAttn A) {
    constexpr int DV = 32 * G;
    const int lane = threadIdx.x & 63;
    const int64_t w = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int64_t rows = (int64_t)P.n_tokens * A.n_heads;
    if (w >= rows) return;
    const int token = (int)(w / A.n_heads), hd = (int)(w % A.n_heads);
    int seq, a, b;
    // rows of no tile stay as they are
    if (!paged_session(P, token, &seq, &a, &b) || (A.by_seq && token - a >= A.tok_tile)) return;
    float top = -__builtin_inff();
    for (int s = 0; s < A.n_splits; s++) top = fmaxf(top, A.ml[(s * rows + w) * 2]);
    const bool none = top == -__builtin_inff();
    float base = none ? 0.0f : top, sum = 0.0f;
    if (A.sinks) {
        const float sink = A.sinks[hd] * 1.44269504f;
        base = none ? sink : fmaxf(base, sink);
        sum = __builtin_amdgcn_exp2f(sink - base);
    }
    float o[DV / 64] = {};
    for (int s = 0; s < A.n_splits; s++) {
        const float m = A.ml[(s * rows + w) * 2];
        if (m == -__builtin_inff()) continue;
        const float f = __builtin_amdgcn_exp2f(m - base);
        sum = fmaf(f, A.ml[(s * rows + w) * 2 + 1], sum);
#pragma unroll
        for (int j = 0; j < DV / 64; j++) o[j] = fmaf(f, A.part[(s * rows + w) * DV + lane + 64 * j], o[j]);
    }
#pragma unroll
    for (int j = 0; j < DV / 64; j++) {
        const int ch = lane + 64 * j;
        if (ch >= P.vd) continue;
        const float y = none ? 0.0f : o[j] / sum;
        const int64_t to = token * A.o_stride + (int64_t)hd * P.vd + ch;
        if (F32)
            ((float *)A.out)[to] = y;
        else
            ((uint16_t *)A.out)[to] = f32_to_bf16(y);
    }
}

}  // namespace rh

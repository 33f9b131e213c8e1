// Attention of query rows over the paged 8-bit key/value cache.
//
//   out[r] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q_r . k_j - running maximum)
//
// in one pass over the keys.  A row of the kernels is one (token, query head) pair of one sequence and key/value head: all heads
// of a group read the same keys, so they are rows of one tile.  Everything is computed transposed, S^T = K Q^T and
// O^T = V^T P^T, with v_mfma_f32_16x16x32_f16: in its result a lane holds tokens 4 g + 0..3 (g = lane / 16) of row lane % 16, which
// is the share of the second product's operand that the lane needs when the operand's 8 tokens are taken as 4 of the block's first
// 16 tokens and 4 of its second 16.  The cache stores values in that order, so probabilities go from one product to the next in the
// registers they were formed in.
//
// Precision.  Codes are exact in f16, scales stay fp32: a key block's scale multiplies the fp32 products, a value block's the
// fp32 probabilities.  Queries and probabilities of fp32 calls are split in two f16 terms (hi + lo, 22 bits) and cost two matrix
// instructions each; one term would leave errors of 2^-12 of a probability, 100 times what an fp32 result should have.
// bf16 calls use one term (a query's 8 bits are exact, a probability's 11 are 3 more than the result keeps).  Queries
// are scaled by a power of two of their row's maximum, the value scales by one of the largest in reach, so that neither
// leaves f16's range; both are undone in fp32.
#include <algorithm>
#include <climits>

#include "kv_dev.h"

namespace smx {

namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kSegBlocks = 128;          // blocks whose places and scales are looked up at a time
constexpr float kLazy = 8.0f;            // the running maximum follows only steps of more than 2^8
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxPieces = 1024;
constexpr float kNoMax = -1e30f;         // running maximum of a row that has seen no key

struct AttnArgs {
    KvArgs kv;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    float* part;        // [rows * q_heads][pieces][dim64] unnormalised sums
    float2* part_ml;    // [rows * q_heads][pieces] maximum and sum of the probabilities
    int q_heads, group, window;
    int piece;          // tokens per piece (a multiple of 32)
    int pieces;         // of the longest sequence
    int row_tiles;
    int paired;         // (see attn_tile_kernel)
    float scale;        // times log2(e)
    int vec;            // rows may be read and written 16 bytes (bf16: 8) at a time
};

// Keys that the rows of one sequence see, and how they are split.
struct Span {
    KvSeq q;
    int first;    // first token in reach of any row, rounded down to a block
    int pieces;
};
__device__ __forceinline__ Span seq_span(const AttnArgs& A, int s) {
    Span x;
    x.q = kv_seq(A.kv, s);
    x.first = A.window > 0 ? max(x.q.len - x.q.n - A.window + 1, 0) & ~(SMX_KV_BLOCK - 1) : 0;
    x.pieces = min((x.q.len - x.first + A.piece - 1) / A.piece, A.pieces);
    return x;
}

// 4 signed bytes -> 4 f16 in two registers: v + 128 as the low mantissa bits of 1024 + (v + 128), then minus 1152.  Exact.
__device__ __forceinline__ void widen4(unsigned w, unsigned* o) {
    w ^= 0x80808080u;
    const unsigned a = __builtin_amdgcn_perm(0x64646464u, w, 0x04010400u), b = __builtin_amdgcn_perm(0x64646464u, w, 0x04030402u);
    const v2h off = {(_Float16)1152.f, (_Float16)1152.f};
    o[0] = __builtin_bit_cast(unsigned, __builtin_bit_cast(v2h, a) - off);
    o[1] = __builtin_bit_cast(unsigned, __builtin_bit_cast(v2h, b) - off);
}
__device__ __forceinline__ v8h widen8(unsigned lo, unsigned hi) {
    uint4 r;
    unsigned* p = (unsigned*)&r;
    widen4(lo, p);
    widen4(hi, p + 2);
    return __builtin_bit_cast(v8h, r);
}

// A value that is the same in every lane of a wave, in scalar registers.
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const unsigned lo = __builtin_amdgcn_readfirstlane((int)(unsigned)v), hi = __builtin_amdgcn_readfirstlane((int)(unsigned)((uint64_t)v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}

// The two values whose larger (sum) a step of a reduction over the four lanes of a row (lane, ^ 16, ^ 32, ^ 48) takes: rows of 16 lanes, or
// halves, swapped between two copies.
__device__ __forceinline__ float2 swap32(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float2 swap16(float v) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return make_float2(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float row_max(float v) {
    float2 s = swap32(v);
    s = swap16(fmaxf(s.x, s.y));
    return fmaxf(s.x, s.y);
}
__device__ __forceinline__ float row_sum(float v) {
    float2 s = swap32(v);
    s = swap16(s.x + s.y);
    return s.x + s.y;
}

// The query rows of one column tile as the B operand of S^T = K Q^T: lane (row lane % 16, g) holds channels 64 c + 16 g + 0..15 of
// its row, scaled by a power of two; *unit is what a product of them with codes times a key scale is multiplied by.
template <int DC, int NT, bool BF16>
__device__ __forceinline__ void load_query(const AttnArgs& A, bool live, int64_t at, v8h (&qf)[NT][DC * 2], float* unit) {
    const int g = (threadIdx.x & 63) >> 4;
    float x[DC][16];
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < DC; c++) {
        const int d0 = c * 64 + g * 16;
        if (A.vec && live && d0 + 16 <= A.kv.dim) {
            if (BF16) {
                const uint4* p = (const uint4*)((const uint16_t*)A.q + at + d0);
#pragma unroll
                for (int j = 0; j < 2; j++) {
                    const uint4 w = p[j];
                    const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        x[c][j * 8 + 2 * i] = __uint_as_float(u[i] << 16);
                        x[c][j * 8 + 2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
                    }
                }
            } else {
                const float4* p = (const float4*)((const float*)A.q + at + d0);
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 w = p[j];
                    x[c][4 * j] = w.x; x[c][4 * j + 1] = w.y; x[c][4 * j + 2] = w.z; x[c][4 * j + 3] = w.w;
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; j++) x[c][j] = live && d0 + j < A.kv.dim ? load_elem<BF16>(A.q, at + d0 + j) : 0.f;
        }
#pragma unroll
        for (int j = 0; j < 16; j++) top = fmaxf(top, fabsf(x[c][j]));
    }
    top = row_max(top);
    // 2^e with top * 2^e in [2^14, 2^15): f16's largest power of two; 0, inf and subnormal maxima keep e in range
    int e = 14 - (int)((__float_as_uint(top) >> 23) & 255) + 127;
    e = min(max(e, -115), 120);
    const float up = __uint_as_float((unsigned)(e + 127) << 23);
    *unit = A.scale * __uint_as_float((unsigned)(127 - e) << 23);
#pragma unroll
    for (int c = 0; c < DC; c++)
#pragma unroll
        for (int h = 0; h < 2; h++) {
            v8h hi, lo;
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float y = x[c][h * 8 + j] * up;
                hi[j] = (_Float16)y;
                lo[j] = (_Float16)(y - (float)hi[j]);
            }
            qf[0][c * 2 + h] = hi;
            if (NT == 2) qf[NT - 1][c * 2 + h] = lo;
        }
}

// Places and scales of up to kSegBlocks blocks of a sequence, looked up by the whole workgroup at once.
struct Segment {
    int64_t place[kSegBlocks];
    float ks[kSegBlocks], vs[kSegBlocks];
    float top[4];   // largest value scale, per wave
};
template <int THREADS>
__device__ __forceinline__ void load_segment(const AttnArgs& A, Segment& seg, int s, int head, int blk0, int n) {
    float top = 0.f;
    for (int i = threadIdx.x; i < n; i += THREADS) {
        const int64_t p = kv_block(A.kv, s, head, blk0 + i);
        seg.place[i] = p;
        seg.ks[i] = A.kv.ks[p];
        const float v = A.kv.vs[p];
        seg.vs[i] = v;
        top = fmaxf(top, v);   // (a NaN scale does not count)
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) top = fmaxf(top, __shfl_xor(top, o));
    if ((threadIdx.x & 63) == 0) seg.top[threadIdx.x >> 6] = top;
}
// Exponent that brings value scales up to `top` under 2^6 (times probabilities of up to 2^8 under 2^14).
__device__ __forceinline__ int value_exponent(float top) {
    const int e = 5 - (int)((__float_as_uint(top) >> 23) & 255) + 127;
    return top > 0.f ? min(max(e, -100), 100) : 0;
}
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }

// One block of 32 tokens against CT column tiles: scores to probabilities, with the running maximum m and sum l of each row, the
// sums O rescaled when a maximum moves.  t: [CT][8] scores in base 2 of tokens 4 g + i % 4 + 16 (i / 4) (masked: -inf).
template <int CT, int NO>
__device__ __forceinline__ void rescale(const float (&mx)[CT], float (&m)[CT], float (&l)[CT], v4f (&o)[CT][NO]) {
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const bool up = mx[ct] > m[ct] + kLazy;
        if (__ballot(up)) {
            const float nm = up ? mx[ct] : m[ct];
            const float f = __builtin_amdgcn_exp2f(m[ct] - nm);
            m[ct] = nm;
            l[ct] *= f;
#pragma unroll
            for (int i = 0; i < NO; i++) o[ct][i] *= f;
        }
    }
}
template <int NT>
__device__ __forceinline__ void split_prob(const float (&p)[8], v8h (&pf)[NT]) {
#pragma unroll
    for (int j = 0; j < 8; j += 2) {
        const v2h hi = {(_Float16)p[j], (_Float16)p[j + 1]};   // one packed conversion
        pf[0][j] = hi[0];
        pf[0][j + 1] = hi[1];
        if (NT == 2) {   // p - hi is exact; an FMA takes the f16 operand as it is
            const v2h lo = {(_Float16)fmaf((float)hi[0], -1.0f, p[j]), (_Float16)fmaf((float)hi[1], -1.0f, p[j + 1])};
            pf[NT - 1][j] = lo[0];
            pf[NT - 1][j + 1] = lo[1];
        }
    }
}

// Where row r (of n * group) of the sequence is: its element offset in q and out divided by its head's, and its position.
struct RowAt {
    int row, head, pos;
    bool live;
};
__device__ __forceinline__ RowAt row_at(const AttnArgs& A, const KvSeq& q, int kvh, int r) {
    RowAt x;
    const int tok = r / A.group;
    x.live = tok < q.n;
    x.row = q.row + min(tok, max(q.n - 1, 0));
    x.head = kvh * A.group + (r - tok * A.group);
    x.pos = q.len - q.n + tok;
    return x;
}
// 4 channels d.. of one row of the result
template <bool BF16>
__device__ __forceinline__ void store_out(const AttnArgs& A, const RowAt& r, int d, v4f o) {
    const int64_t at = (int64_t)r.row * A.ldo + (int64_t)r.head * A.kv.dim + d;
    if (A.vec && d + 4 <= A.kv.dim) {
        if (BF16) *(uint2*)((uint16_t*)A.out + at) = make_uint2(f32_to_bf16(o[0]) | (unsigned)f32_to_bf16(o[1]) << 16, f32_to_bf16(o[2]) | (unsigned)f32_to_bf16(o[3]) << 16);
        else *(float4*)((float*)A.out + at) = make_float4(o[0], o[1], o[2], o[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++)
            if (d + i < A.kv.dim) store_elem<BF16>(A.out, at + i, o[i]);
    }
}
// A piece's share of one row: the result itself where the sequence is one piece, else sums for attn_join_kernel.
template <bool BF16>
__device__ __forceinline__ void put_row(const AttnArgs& A, const RowAt& r, int piece, int pieces, int d, v4f o, float m, float l, bool first) {
    if (!r.live) return;
    if (pieces == 1) {
        const float inv = l > 0.f ? 1.0f / l : l == l ? 0.f : l;   // (a NaN stays one)
        store_out<BF16>(A, r, d, o * inv);
        return;
    }
    const int64_t at = ((int64_t)r.row * A.q_heads + r.head) * A.pieces + piece;
    if (first) A.part_ml[at] = make_float2(m, l);
    *(float4*)(A.part + at * A.kv.dim64 + d) = make_float4(o[0], o[1], o[2], o[3]);
}

// ---- few rows: a decode step, a handful of drafted tokens.  Workgroup (head and tile of 16 CT rows, piece of the context,
// sequence); its four waves take the piece's blocks in turn, straight from memory into the matrix instructions' registers (one block
// ahead), and add up through LDS at the end.
template <int DC, int CT, int NT, bool BF16>
__global__ __launch_bounds__(256, CT == 2 ? 2 : DC <= 1 ? 4 : DC == 2 ? 3 : 2) void attn_rows_kernel(const AttnArgs A) {
    constexpr int D64 = DC * 64, NO = DC * 4;
    __shared__ Segment seg;
    __shared__ float wm[4][16 * CT], wl[4][16 * CT];
    extern __shared__ float wo[];   // [4][16][D64 + 4], one column tile at a time
    const int s = blockIdx.z, piece = blockIdx.y;
    const int kvh = blockIdx.x % A.kv.kv_heads, tile = blockIdx.x / A.kv.kv_heads;
    const Span sp = seq_span(A, s);
    const int rows = sp.q.n * A.group;
    if (tile * 16 * CT >= rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    RowAt at[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) at[ct] = row_at(A, sp.q, kvh, (tile * CT + ct) * 16 + (lane & 15));
    if (piece >= sp.pieces) {
        if (piece == 0 && wave == 0) {   // a sequence without a token in the cache
#pragma unroll
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int i = 0; i < NO; i++) put_row<BF16>(A, at[ct], 0, 1, i * 16 + g * 4, v4f{0.f, 0.f, 0.f, 0.f}, 0.f, 0.f, false);
        }
        return;
    }
    const int tok0 = sp.first + piece * A.piece, tok1 = min(tok0 + A.piece, sp.q.len);
    const int b0 = tok0 / SMX_KV_BLOCK, b1 = (tok1 + SMX_KV_BLOCK - 1) / SMX_KV_BLOCK;
    v8h qf[CT][NT][DC * 2];
    float unit[CT], m[CT], l[CT];
    v4f o[CT][NO];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        load_query<DC, NT, BF16>(A, at[ct].live, (int64_t)at[ct].row * A.ldq + (int64_t)at[ct].head * A.kv.dim, qf[ct], &unit[ct]);
        m[ct] = kNoMax;
        l[ct] = 0.f;
#pragma unroll
        for (int i = 0; i < NO; i++) o[ct][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    // every row of the tile sees keys [all_lo, all_hi]: blocks inside need no mask
    const int first_pos = sp.q.len - sp.q.n + tile * 16 * CT / A.group, last_pos = sp.q.len - sp.q.n + min(tile * 16 * CT + 16 * CT - 1, rows - 1) / A.group;
    const int all_hi = first_pos, all_lo = A.window > 0 ? last_pos - A.window + 1 : 0;
    int vexp = 0;
    for (int c0 = b0; c0 < b1; c0 += kSegBlocks) {
        const int n = min(kSegBlocks, b1 - c0);
        if (c0 != b0) __syncthreads();
        load_segment<256>(A, seg, s, kvh, c0, n);
        __syncthreads();
        const int e = value_exponent(fmaxf(fmaxf(seg.top[0], seg.top[1]), fmaxf(seg.top[2], seg.top[3])));
        if (e != vexp) {
            const float f = pow2(min(max(e - vexp, -126), 127));
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int i = 0; i < NO; i++) o[ct][i] *= f;
            vexp = e;
        }
        const float vup = pow2(vexp);
        // a block's bytes are asked for as soon as the registers of the one in front are free: keys behind its scores, values behind
        // its second product
        uint4 kb[2 * DC], vb[2 * DC];
        auto fetch = [&](uint4 (&to)[2 * DC], const int8_t* plane, int i) {
            const int8_t* base = plane + uniform(seg.place[i]) * (SMX_KV_BLOCK * D64);
#pragma unroll
            for (int j = 0; j < 2 * DC; j++) to[j] = *(const uint4*)(base + (unsigned)(j * 1024 + lane * 16));
        };
        if (wave < n) {
            fetch(kb, A.kv.k, wave);
            fetch(vb, A.kv.v, wave);
        }
        for (int i = wave; i < n; i += 4) {
            v4f sc[CT][2];
#pragma unroll
            for (int tt = 0; tt < 2; tt++) {
                v8h kf[DC * 2];
#pragma unroll
                for (int c = 0; c < DC; c++) {
                    const uint4 w = kb[tt * DC + c];
                    kf[c * 2] = widen8(w.x, w.y);
                    kf[c * 2 + 1] = widen8(w.z, w.w);
                }
#pragma unroll
                for (int ct = 0; ct < CT; ct++) {
                    sc[ct][tt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int nt = NT - 1; nt >= 0; nt--)   // the small terms first: fewer roundings of large sums
#pragma unroll
                        for (int k = 0; k < DC * 2; k++) sc[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], qf[ct][nt][k], sc[ct][tt], 0, 0, 0);
                }
            }
            const float ks = seg.ks[i], vs = seg.vs[i] * vup;
            const int next = i + 4;
            if (next < n) fetch(kb, A.kv.k, next);
            const int tok = (c0 + i) * SMX_KV_BLOCK;
            const bool edge = tok + SMX_KV_BLOCK - 1 > all_hi || tok < all_lo;
            float t[CT][8], mx[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float f = unit[ct] * ks;
                mx[ct] = kNoMax;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    t[ct][j] = sc[ct][j >> 2][j & 3] * f;
                    if (edge) {
                        const int key = tok + 16 * (j >> 2) + 4 * g + (j & 3);
                        if (key > at[ct].pos || (A.window > 0 && key <= at[ct].pos - A.window)) t[ct][j] = -INFINITY;
                    }
                    mx[ct] = fmaxf(mx[ct], t[ct][j]);
                }
                mx[ct] = row_max(mx[ct]);
            }
            rescale<CT, NO>(mx, m, l, o);
            v8h pf[CT][NT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float p[8], sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float e2 = __builtin_amdgcn_exp2f(t[ct][j] - m[ct]);
                    sum += e2;
                    p[j] = edge && t[ct][j] == -INFINITY ? 0.f : e2 * vs;   // (a masked token's value scale may be NaN)
                }
                l[ct] += sum;
                split_prob<NT>(p, pf[ct]);
            }
#pragma unroll
            for (int j = 0; j < 2 * DC; j++) {
                const v8h v0 = widen8(vb[j].x, vb[j].y), v1 = widen8(vb[j].z, vb[j].w);
#pragma unroll
                for (int ct = 0; ct < CT; ct++)
#pragma unroll
                    for (int nt = NT - 1; nt >= 0; nt--) {
                        o[ct][2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, pf[ct][nt], o[ct][2 * j], 0, 0, 0);
                        o[ct][2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, pf[ct][nt], o[ct][2 * j + 1], 0, 0, 0);
                    }
            }
            if (next < n) fetch(vb, A.kv.v, next);
        }
    }
    // the four waves' shares
    const float down = pow2(-vexp);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        l[ct] = row_sum(l[ct]);
        if (g == 0) {
            wm[wave][ct * 16 + lane] = m[ct];
            wl[wave][ct * 16 + lane] = l[ct];
        }
    }
    constexpr int PITCH = D64 + 4;
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        __syncthreads();
        const int r = ct * 16 + (lane & 15);
        const float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
        const float f = __builtin_amdgcn_exp2f(m[ct] - M) * down;
#pragma unroll
        for (int i = 0; i < NO; i++) *(v4f*)&wo[(wave * 16 + (lane & 15)) * PITCH + i * 16 + g * 4] = o[ct][i] * f;
        float L = 0.f;
#pragma unroll
        for (int w = 0; w < 4; w++) L += wl[w][r] * __builtin_amdgcn_exp2f(wm[w][r] - M);
        __syncthreads();
        // wave w writes channels [w * D64 / 4, ...)
#pragma unroll
        for (int i = 0; i < DC; i++) {
            const int d = (wave * DC + i) * 16 + g * 4;
            v4f acc = *(v4f*)&wo[(lane & 15) * PITCH + d];
#pragma unroll
            for (int w = 1; w < 4; w++) acc += *(v4f*)&wo[(w * 16 + (lane & 15)) * PITCH + d];
            put_row<BF16>(A, at[ct], piece, sp.pieces, d, acc, M, L, wave == 0 && i == 0 && g == 0);
        }
    }
}

// ---- many rows: a prompt chunk.  Workgroup (head and tile of 64 CT rows, piece, sequence); a wave holds 16 CT rows, and the four
// share tiles of TB blocks that are widened to f16 on their way into LDS (each byte once per workgroup), two of them in turn; the tile
// behind the next one is in flight in registers.
// A block's scores are formed one step ahead: the matrix unit works on the next block's while the vector unit turns this block's into
// probabilities (exp, two f16 terms: about ten instructions a score, as long as the matrix instructions of the score take).
template <int DC, int CT, int NT, bool BF16>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(const AttnArgs A) {
    constexpr int D64 = DC * 64, NO = DC * 4, KF = DC * 2, TB = DC <= 2 ? 2 : 1;
    constexpr int UNITS = TB * 2 * DC, PER = (UNITS + 3) / 4;      // 1 KB units of a tile's keys (and values); of them a wave's
    constexpr int KEYS = TB * 2 * KF * 64, TILE = KEYS + TB * NO * 64;   // 16-byte words: keys [block][token / 16][KF][lane], values [block][NO][lane]
    __shared__ Segment seg;
    extern __shared__ uint4 stage[];   // [2][TILE]
    const int s = blockIdx.z, piece = blockIdx.y;
    const int kvh = blockIdx.x % A.kv.kv_heads;
    // The longest rows first.  Where every workgroup has a place at once (two on a CU), the second half goes the other way round, so that
    // each CU has a long and a short one.
    int tile = blockIdx.x / A.kv.kv_heads;
    if (!A.paired || tile < (A.row_tiles + 1) / 2) tile = A.row_tiles - 1 - tile;
    else tile -= (A.row_tiles + 1) / 2;
    const Span sp = seq_span(A, s);
    const int rows = sp.q.n * A.group, row0 = tile * 64 * CT;
    if (row0 >= rows) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int wrow0 = row0 + wave * 16 * CT;
    RowAt at[CT];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) at[ct] = row_at(A, sp.q, kvh, wrow0 + ct * 16 + (lane & 15));
    if (piece >= sp.pieces && piece > 0) return;
    const int pos0 = sp.q.len - sp.q.n;
    const int last_pos = pos0 + min(row0 + 64 * CT - 1, rows - 1) / A.group;
    // tokens of the piece in reach of the tile's rows
    const int reach = A.window > 0 ? max(pos0 + row0 / A.group - A.window + 1, 0) & ~(SMX_KV_BLOCK - 1) : 0;
    const int tok0 = max(sp.first + piece * A.piece, reach), tok1 = min(min(sp.first + (piece + 1) * A.piece, sp.q.len), last_pos + 1);
    v8h qf[CT][NT][KF];
    float unit[CT], m[CT], l[CT];
    v4f o[CT][NO];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        load_query<DC, NT, BF16>(A, at[ct].live, (int64_t)at[ct].row * A.ldq + (int64_t)at[ct].head * A.kv.dim, qf[ct], &unit[ct]);
        m[ct] = kNoMax;
        l[ct] = 0.f;
#pragma unroll
        for (int i = 0; i < NO; i++) o[ct][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    // this wave's rows: every one sees [all_lo, all_hi]; none sees a token outside [any_lo, any_hi]
    const int wfirst = pos0 + wrow0 / A.group, wlast = pos0 + min(wrow0 + 16 * CT - 1, rows - 1) / A.group;
    const int all_hi = wfirst, all_lo = A.window > 0 ? wlast - A.window + 1 : 0;
    const int any_hi = wrow0 < rows ? wlast : -1, any_lo = A.window > 0 ? wfirst - A.window + 1 : 0;
    int vexp = 0;
    const int b0 = tok0 / SMX_KV_BLOCK, b1 = tok1 > tok0 ? (tok1 + SMX_KV_BLOCK - 1) / SMX_KV_BLOCK : b0;
    for (int c0 = b0; c0 < b1; c0 += kSegBlocks) {
        const int n = min(kSegBlocks, b1 - c0), tiles = (n + TB - 1) / TB;
        __syncthreads();
        load_segment<256>(A, seg, s, kvh, c0, n);
        __syncthreads();
        const int e = value_exponent(fmaxf(fmaxf(seg.top[0], seg.top[1]), fmaxf(seg.top[2], seg.top[3])));
        if (e != vexp) {
            const float f = pow2(min(max(e - vexp, -126), 127));
            for (int ct = 0; ct < CT; ct++)
#pragma unroll
                for (int i = 0; i < NO; i++) o[ct][i] *= f;
            vexp = e;
        }
        const float vup = pow2(vexp);
        uint4 kb[PER], vb[PER];
        // this wave's units of a tile: u = wave + 4 j (a last tile's missing block is its first again, and masked)
        auto fetch = [&](int t) {
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int u = wave + 4 * j;
                if (UNITS % 4 && u >= UNITS) break;
                const int64_t base = uniform(seg.place[min(t * TB + u / (2 * DC), n - 1)]) * (SMX_KV_BLOCK * D64) + (u % (2 * DC)) * 1024;
                kb[j] = *(const uint4*)(A.kv.k + base + (unsigned)lane * 16);
                vb[j] = *(const uint4*)(A.kv.v + base + (unsigned)lane * 16);
            }
        };
        auto put = [&](int t) {
            uint4* to = stage + (t & 1) * TILE + lane;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int u = wave + 4 * j;
                if (UNITS % 4 && u >= UNITS) break;
                uint4* kd = to + ((u / DC) * KF + (u % DC) * 2) * 64;     // (block, token / 16), chunk d / 64 -> fragments 2 c, 2 c + 1
                kd[0] = __builtin_bit_cast(uint4, widen8(kb[j].x, kb[j].y));
                kd[64] = __builtin_bit_cast(uint4, widen8(kb[j].z, kb[j].w));
                uint4* vd = to + KEYS + (2 * u) * 64;                     // (block, d / 32) -> channel tiles 2 (d / 32), + 1
                vd[0] = __builtin_bit_cast(uint4, widen8(vb[j].x, vb[j].y));
                vd[64] = __builtin_bit_cast(uint4, widen8(vb[j].z, vb[j].w));
            }
        };
        auto needed = [&](int i) {
            const int tok = (c0 + i) * SMX_KV_BLOCK;
            return i < n && tok <= any_hi && tok + SMX_KV_BLOCK > any_lo;
        };
        auto scores = [&](v4f (&sc)[CT][2], int i) {
            const uint4* kt = stage + ((i / TB) & 1) * TILE + (i % TB) * 2 * KF * 64 + lane;
#pragma unroll
            for (int tt = 0; tt < 2; tt++) {
                v8h kf[KF];
#pragma unroll
                for (int k = 0; k < KF; k++) kf[k] = __builtin_bit_cast(v8h, kt[(tt * KF + k) * 64]);
#pragma unroll
                for (int ct = 0; ct < CT; ct++) sc[ct][tt] = v4f{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int nt = NT - 1; nt >= 0; nt--)   // the small terms first: fewer roundings of large sums
#pragma unroll
                    for (int k = 0; k < KF; k++)
#pragma unroll
                        for (int ct = 0; ct < CT; ct++) sc[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[k], qf[ct][nt][k], sc[ct][tt], 0, 0, 0);
            }
        };
        // probabilities times value scale of block i, 2^(scores * f + base), and their product with its values; the sums of
        // probabilities take the scale out again (per_vs)
        auto weigh = [&](const v4f (&sc)[CT][2], const float (&f)[CT], const float (&base)[CT], float per_vs, float poison, int i) {
            v8h pf[CT][NT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                float p[8], sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    p[j] = __builtin_amdgcn_exp2f(fmaf(sc[ct][j >> 2][j & 3], f[ct], base[ct]));
                    sum += p[j];
                }
                l[ct] = fmaf(sum, per_vs, l[ct]) + (sum > 0.f ? poison : 0.f);
                split_prob<NT>(p, pf[ct]);
            }
            const uint4* vt = stage + ((i / TB) & 1) * TILE + KEYS + (i % TB) * NO * 64 + lane;
#pragma unroll
            for (int k = 0; k < NO; k++) {
                const v8h vf = __builtin_bit_cast(v8h, vt[k * 64]);
#pragma unroll
                for (int nt = NT - 1; nt >= 0; nt--)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) o[ct][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf[ct][nt], o[ct][k], 0, 0, 0);
            }
        };
        // scores(nxt, i + 1) and weigh(cur, i) in one, in the order the instructions are to leave: a pair of probabilities between every
        // MS matrix instructions of the next block's scores, then the product with the values.  The operands pass through a ring of KF
        // registers' worth of LDS reads, each asked for when the one in its place has been used last.
        auto both = [&](const v4f (&cur)[CT][2], v4f (&nxt)[CT][2], const float (&f)[CT], const float (&base)[CT], float per_vs, float poison, int i) {
            constexpr int TT = KF * NT * CT, MS = 2 * TT / (4 * CT);   // matrix instructions of 16 tokens; between two pairs
            const uint4* kt = stage + (((i + 1) / TB) & 1) * TILE + ((i + 1) % TB) * 2 * KF * 64 + lane;
            const uint4* vt = stage + ((i / TB) & 1) * TILE + KEYS + (i % TB) * NO * 64 + lane;
            v8h ring[KF], pf[CT][NT];
            float sum[CT];
#pragma unroll
            for (int k = 0; k < KF; k++) ring[k] = __builtin_bit_cast(v8h, kt[k * 64]);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                sum[ct] = 0.f;
                nxt[ct][0] = nxt[ct][1] = v4f{0.f, 0.f, 0.f, 0.f};
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int pair = 0; pair < 4 * CT; pair++) {
                const int pc = pair % CT, j = pair / CT * 2;
                float p[2];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    p[h] = __builtin_amdgcn_exp2f(fmaf(cur[pc][(j + h) >> 2][(j + h) & 3], f[pc], base[pc]));
                    sum[pc] += p[h];
                }
                const v2h hi = {(_Float16)p[0], (_Float16)p[1]};
                pf[pc][0][j] = hi[0];
                pf[pc][0][j + 1] = hi[1];
                if (NT == 2) {
                    const v2h lo = {(_Float16)fmaf((float)hi[0], -1.0f, p[0]), (_Float16)fmaf((float)hi[1], -1.0f, p[1])};
                    pf[pc][NT - 1][j] = lo[0];
                    pf[pc][NT - 1][j + 1] = lo[1];
                }
#pragma unroll
                for (int q = pair * MS; q < pair * MS + MS; q++) {
                    const int tt = q / TT, r = q % TT, nt = NT - 1 - r / (KF * CT), k = r / CT % KF, ct = r % CT;
                    nxt[ct][tt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[k], qf[ct][nt][k], nxt[ct][tt], 0, 0, 0);
                    if (nt == 0 && ct == CT - 1) ring[k] = __builtin_bit_cast(v8h, tt == 0 ? kt[(KF + k) * 64] : vt[k * 64]);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int ct = 0; ct < CT; ct++) l[ct] = fmaf(sum[ct], per_vs, l[ct]) + (sum[ct] > 0.f ? poison : 0.f);
#pragma unroll
            for (int k = 0; k < NO; k++) {
#pragma unroll
                for (int nt = NT - 1; nt >= 0; nt--)
#pragma unroll
                    for (int ct = 0; ct < CT; ct++) o[ct][k] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ring[k % KF], pf[ct][nt], o[ct][k], 0, 0, 0);
                if (k + KF < NO) ring[k % KF] = __builtin_bit_cast(v8h, vt[(k + KF) * 64]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        // block i, whose scores are in `cur`; the next block's go to `nxt`
        auto step = [&](v4f (&cur)[CT][2], v4f (&nxt)[CT][2], int i) {
            if (i % TB == TB - 1 && i / TB + 1 < tiles) {
                __syncthreads();   // everyone is done with the tile in front of this one
                put(i / TB + 1);
                if (i / TB + 2 < tiles) fetch(i / TB + 2);
                __syncthreads();
            }
            const bool now = needed(i), then = needed(i + 1);
            if (!now) {
                if (then) scores(nxt, i + 1);
                return;
            }
            const int tok = (c0 + i) * SMX_KV_BLOCK;
            const bool edge = tok + SMX_KV_BLOCK - 1 > all_hi || tok < all_lo;
            const float ks = seg.ks[i];
            // a value scale of 0 stands for codes of 0; a NaN one is for the rows that see a token of the block
            const float scale = seg.vs[i] * vup, vs = fmaxf(scale, 0x1p-60f), poison = scale == scale ? 0.f : scale;
            const float log_vs = __builtin_amdgcn_logf(vs), per_vs = __builtin_amdgcn_rcpf(vs);
            float f[CT], base[CT], mx[CT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                f[ct] = unit[ct] * ks;
                if (edge) {
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const int key = tok + 16 * (j >> 2) + 4 * g + (j & 3);
                        const bool out = key > at[ct].pos || (A.window > 0 && key <= at[ct].pos - A.window);
                        cur[ct][j >> 2][j & 3] = out ? -INFINITY : cur[ct][j >> 2][j & 3] * f[ct];
                    }
                    f[ct] = 1.0f;
                }
                mx[ct] = kNoMax;
#pragma unroll
                for (int j = 0; j < 8; j++) mx[ct] = fmaxf(mx[ct], cur[ct][j >> 2][j & 3]);
                mx[ct] = row_max(mx[ct]) * f[ct];
            }
            rescale<CT, NO>(mx, m, l, o);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) base[ct] = log_vs - m[ct];
            if (then) both(cur, nxt, f, base, per_vs, poison, i);
            else weigh(cur, f, base, per_vs, poison, i);
        };
        fetch(0);
        put(0);
        if (tiles > 1) fetch(1);
        __syncthreads();
        v4f s0[CT][2], s1[CT][2];
        if (needed(0)) scores(s0, 0);
        for (int i = 0; i < n; i += 2) {
            step(s0, s1, i);
            if (i + 1 < n) step(s1, s0, i + 1);
        }
    }
    const float down = pow2(-vexp);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const float L = row_sum(l[ct]);
#pragma unroll
        for (int i = 0; i < NO; i++) put_row<BF16>(A, at[ct], piece, max(sp.pieces, 1), i * 16 + g * 4, o[ct][i] * down, m[ct], L, i == 0 && g == 0);
    }
}

// Workgroup (row, head): the pieces of a long sequence joined.  Every piece's factor is formed first, so that nothing stands between
// the loads of their sums; 16 bytes for each thread, several pieces at a time.
template <bool BF16>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs A) {
    __shared__ float factor[kMaxPieces], red[2][4];
    __shared__ v4f sums[256];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    int s = row;
    if (A.kv.row0) {
        int lo = 0, hi = A.kv.nseq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (A.kv.row0[mid] <= row) lo = mid; else hi = mid - 1;
        }
        s = lo;
    }
    const Span sp = seq_span(A, s);
    if (sp.pieces <= 1 || row >= sp.q.row + sp.q.n) return;
    const int64_t at = ((int64_t)row * A.q_heads + head) * A.pieces;
    float M = kNoMax;
    for (int i = tid; i < sp.pieces; i += 256) M = fmaxf(M, A.part_ml[at + i].x);
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) M = fmaxf(M, __shfl_xor(M, o));
    if (lane == 0) red[0][wave] = M;
    __syncthreads();
    M = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float L = 0.f;
    for (int i = tid; i < sp.pieces; i += 256) {
        const float2 ml = A.part_ml[at + i];
        const float f = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);   // (a piece without a key for the row)
        factor[i] = f;
        L += ml.y * f;
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) L += __shfl_xor(L, o);
    if (lane == 0) red[1][wave] = L;
    __syncthreads();
    L = red[1][0] + red[1][1] + red[1][2] + red[1][3];
    const int quads = A.kv.dim64 / 4, groups = 256 / quads, g = tid / quads, d = (tid - g * quads) * 4;   // quads: 16, 32, 48 or 64
    v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
    if (g < groups) {
        const float* from = A.part + at * A.kv.dim64 + d;
#pragma unroll 4
        for (int i = g; i < sp.pieces; i += groups) acc += *(const v4f*)(from + (int64_t)i * A.kv.dim64) * factor[i];
    }
    sums[tid] = acc;
    __syncthreads();
    if (g != 0) return;
    for (int w = 1; w < groups; w++) acc += sums[w * quads + tid];
    const float inv = L > 0.f ? 1.0f / L : L == L ? 0.f : L;
    RowAt r;
    r.row = row; r.head = head; r.pos = 0; r.live = true;
    store_out<BF16>(A, r, d, acc * inv);
}

template <int DC, int CT, int NT, bool BF16>
int launch_rows(smx_ctx* c, const AttnArgs& A, dim3 grid) {
    const size_t lds = 4 * 16 * (DC * 64 + 4) * 4;
    int rc;
    if ((rc = set_dyn_lds(c, attn_rows_kernel<DC, CT, NT, BF16>, lds)) != SMX_OK) return rc;
    hipLaunchKernelGGL((attn_rows_kernel<DC, CT, NT, BF16>), grid, dim3(256), lds, c->stream, A);
    return SMX_OK;
}
template <int DC, int CT, int NT, bool BF16>
int launch_tile(smx_ctx* c, const AttnArgs& A, dim3 grid) {
    const size_t lds = 2 * (DC <= 2 ? 2 : 1) * (2 * DC * 2 + DC * 4) * 1024;
    int rc;
    if ((rc = set_dyn_lds(c, attn_tile_kernel<DC, CT, NT, BF16>, lds)) != SMX_OK) return rc;
    hipLaunchKernelGGL((attn_tile_kernel<DC, CT, NT, BF16>), grid, dim3(256), lds, c->stream, A);
    return SMX_OK;
}
// Column tiles of a wave: as many as leave two waves a SIMD their registers (queries and sums are 8 CT DC NT and 16 CT DC of 256).
constexpr int rows_tiles(int dc) { return dc <= 2 ? 2 : 1; }
constexpr int wave_tiles(int dc) { return dc <= 2 ? 2 : 1; }
template <int DC>
int launch_dim(smx_ctx* c, const AttnArgs& A, dim3 grid, bool bf16, int form) {
    if (form == 0) return bf16 ? launch_rows<DC, 1, 1, true>(c, A, grid) : launch_rows<DC, 1, 2, false>(c, A, grid);
    if (form == 1) return bf16 ? launch_rows<DC, rows_tiles(DC), 1, true>(c, A, grid) : launch_rows<DC, rows_tiles(DC), 2, false>(c, A, grid);
    return bf16 ? launch_tile<DC, wave_tiles(DC), 1, true>(c, A, grid) : launch_tile<DC, wave_tiles(DC), 2, false>(c, A, grid);
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" int smx_attn_dev(smx_ctx* c, const smx_kv_cache* cache, const smx_kv_batch* batch, int type, const void* q, size_t ldq, size_t q_heads,
                            float scale, size_t window, void* out, size_t ldo) {
    if (!c) return SMX_ERR_ARG;
    AttnArgs A{};
    int rc;
    if ((rc = kv_args(c, "attn_dev", cache, batch, &A.kv)) != SMX_OK) return rc;
    if (type != SMX_TYPE_F32 && type != SMX_TYPE_BF16) return fail(c, SMX_ERR_ARG, "attn_dev: element type %d", type);
    if (q_heads == 0 || q_heads > 65535 || q_heads % cache->kv_heads)
        return fail(c, SMX_ERR_ARG, "attn_dev: %zu query heads for %zu key/value heads", q_heads, cache->kv_heads);
    const size_t width = q_heads * cache->head_dim;
    if (ldq < width || ldo < width) return fail(c, SMX_ERR_ARG, "attn_dev: rows of %zu elements, ldq %zu, ldo %zu", width, ldq, ldo);
    if (batch->nseq == 0 || batch->rows == 0) return SMX_OK;
    if (!q || !out) return fail(c, SMX_ERR_ARG, "attn_dev: null queries or result");
    const bool bf16 = type == SMX_TYPE_BF16;
    A.q = q; A.out = out; A.ldq = (int64_t)ldq; A.ldo = (int64_t)ldo;
    A.q_heads = (int)q_heads;
    A.group = (int)(q_heads / cache->kv_heads);
    A.window = (int)std::min<size_t>(window, INT_MAX / 2);
    A.scale = scale * kLog2e;
    const size_t per16 = bf16 ? 8 : 4;
    A.vec = cache->head_dim % 16 == 0 && ldq % per16 == 0 && ldo % per16 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0;
    const size_t tile_rows = batch->max_rows * (size_t)A.group;
    const int form = tile_rows <= 16 ? 0 : tile_rows <= 64 ? 1 : 2;
    const int dc = A.kv.dim64 / 64;
    const size_t per_tile = form == 0 ? 16 : form == 1 ? 16 * rows_tiles(dc) : 64 * wave_tiles(dc);
    A.row_tiles = (int)((tile_rows + per_tile - 1) / per_tile);
    // tokens in reach of one sequence's rows, and how many workgroups they make without a split
    const size_t reach = window ? std::min<size_t>(A.kv.max_len, window + batch->max_rows + SMX_KV_BLOCK) : (size_t)A.kv.max_len;
    const size_t groups = batch->nseq * cache->kv_heads * (size_t)A.row_tiles;
    const size_t want = 512, least = 128;
    size_t split = std::min<size_t>(groups >= want ? 1 : (want + groups - 1) / groups, kMaxPieces);
    size_t piece = (std::max<size_t>(reach, 1) + split - 1) / split;
    piece = std::max<size_t>((piece + 127) & ~size_t(127), least);
    A.piece = (int)std::min<size_t>(piece, size_t(1) << 30);
    A.pieces = (int)std::max<size_t>((reach + piece - 1) / piece, 1);
    if (A.pieces > 1) {
        const size_t n = batch->rows * q_heads * (size_t)A.pieces;
        if ((rc = ensure(c, c->work, n * ((size_t)A.kv.dim64 * 4 + 8))) != SMX_OK) return rc;
        A.part = (float*)c->work.p;
        A.part_ml = (float2*)(A.part + n * A.kv.dim64);
    }
    A.paired = groups * (size_t)A.pieces <= 2 * (size_t)c->num_cu && A.pieces == 1;
    const dim3 grid((unsigned)(cache->kv_heads * A.row_tiles), (unsigned)A.pieces, (unsigned)batch->nseq);
    ProfScope ps(c, form < 2 ? "attn_rows" : "attn_tile");
    switch (A.kv.dim64 / 64) {
        case 1: rc = launch_dim<1>(c, A, grid, bf16, form); break;
        case 2: rc = launch_dim<2>(c, A, grid, bf16, form); break;
        case 3: rc = launch_dim<3>(c, A, grid, bf16, form); break;
        default: rc = launch_dim<4>(c, A, grid, bf16, form); break;
    }
    if (rc != SMX_OK) return rc;
    SMX_HIP(c, hipGetLastError());
    if (A.pieces > 1) {
        const dim3 jg((unsigned)batch->rows, (unsigned)q_heads);
        if (bf16) hipLaunchKernelGGL(attn_join_kernel<true>, jg, dim3(256), 0, c->stream, A);
        else hipLaunchKernelGGL(attn_join_kernel<false>, jg, dim3(256), 0, c->stream, A);
        SMX_HIP(c, hipGetLastError());
    }
    return SMX_OK;
}

// Attention of query rows over the paged 8-bit key/value cache.
//
//   out[r] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale * q_r . k_j - reference)
//
// in one pass over the keys.  A row of the kernels is one (token, query head) pair of one sequence and key/value head: all heads
// of a group read the same keys, so they are rows of one tile.  Everything is computed transposed, S^T = K Q^T and
// O^T = V^T P^T, with v_mfma_f32_16x16x32_f16: in its result a lane holds tokens 4 g + 0..3 (g = lane / 16) of row lane % 16, which
// is the share of the second product's operand that the lane needs when the operand's 8 tokens are taken as 4 of the block's first
// 16 tokens and 4 of its second 16.  The cache stores values in that order, so probabilities go from one product to the next in the
// registers they were formed in.
//
// Precision.  Codes are exact in f16, scales stay fp32: a key block's scale multiplies the fp32 products, a value block's the
// fp32 probabilities.  Queries and weights (probabilities times value scales) of fp32 calls are split in two f16 terms (hi + lo, 22
// bits) and cost two matrix instructions each; one term would leave errors of 2^-12 of a weight, 100 times what an fp32 result should have.
// bf16 calls use one term (a query's 8 bits are exact, a weight's 11 are 3 more than the result keeps).
// f16's range: queries are scaled by a power of two of their row's maximum.  A weight is p_j 2^e u with the value scale's exponent e and
// u in [1, 2); the reference of the exponentials is the running maximum of score + e (base 2), so a row's largest weight is
// near 2^5 whatever its probability and scale are, and blocks of far larger values with tiny probabilities (or out of a row's sight) take no
// bits from the others.  Sums of probabilities take 2^e out again in fp32, which holds while the value scales of a sequence are within
// 2^100 of each other and above 2^-90: smaller ones are taken for 2^-100 of the largest (2^-90) in these sums.
#pragma once
#include "kv_dev.h"

namespace smx {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kSegBlocks = 256;          // blocks whose places and scales are looked up at a time
constexpr float kLazy = 8.0f;            // the reference follows only steps of more than 2^8
constexpr int kLift = 5;                 // weights are 2^kLift times what the reference makes of them: up to 2^14
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxPieces = 1024;
constexpr float kNoMax = -3.402823466e38f;   // reference of a row that has seen no key: no finite score is below it

struct AttnArgs {
    KvArgs kv;
    const void* q;
    void* out;
    int64_t ldq, ldo;
    float* part;        // unnormalised sums of pieces, [dim64] each: [sums_of()][pieces]
    float2* part_ml;    // their references and sums of probabilities
    unsigned* count;    // few rows: finished pieces of each (sequence, head, tile); 0 between launches
    int join;           // few rows: the last workgroup of a row tile to finish joins its pieces
    int tile_rows;
    int few_rows;       // places that each sequence's rows of a key/value head have for their sums; 0: each of the call's rows has one (see sums_of)
    int above, upto;    // sequences of more than `above` and up to `upto` rows of a key/value head are this launch's
    int listed;         // many rows: workgroups z serve the z-th of the sequences that are this launch's
    int q_heads, group, window;
    int piece;          // tokens per piece (a multiple of 32)
    int pieces;         // of the longest sequence
    int row_tiles;
    int paired;         // (see attn_tile_kernel)
    int lone;           // few rows: workgroups of one wave
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
    const int64_t rows = (int64_t)x.q.n * A.group;
    if (rows <= A.above || rows > A.upto) x.q.n = 0;
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
// Of 16 lanes by DPP moves: neighbours, pairs of them, the half row's mirror, the row's.  (Shuffles go through LDS: four of them one behind
// the other are a fifth of a microsecond of every workgroup's start.)
template <int CTRL>
__device__ __forceinline__ float dpp_max(float v) {
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, false)));
}
__device__ __forceinline__ float wave_max(float v) {
    v = dpp_max<0xb1>(v);
    v = dpp_max<0x4e>(v);
    v = dpp_max<0x141>(v);
    v = dpp_max<0x140>(v);
    return row_max(v);
}
__device__ __forceinline__ float row_sum(float v) {
    float2 s = swap32(v);
    s = swap16(s.x + s.y);
    return s.x + s.y;
}

// The query rows of one column tile as the B operand of S^T = K Q^T: lane (row lane % 16, g) holds channels 64 c + 16 g + 0..15 of
// its row, times a power of two and the sign of the call's scale; *unit (not negative) is what a product of them with codes times
// a key scale is multiplied by.
// (load_query: the channels as they are; set_query: the operand.)
template <int DC, bool BF16>
__device__ __forceinline__ void load_query(const AttnArgs& A, bool live, int64_t at, float (&x)[DC][16]) {
    const int g = (threadIdx.x & 63) >> 4;
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
    }
}
template <int DC, int NT>
__device__ __forceinline__ void set_query(const AttnArgs& A, const float (&x)[DC][16], v8h (&qf)[NT][DC * 2], float* unit) {
    float top = 0.f;
#pragma unroll
    for (int c = 0; c < DC; c++)
#pragma unroll
        for (int j = 0; j < 16; j++) top = fmaxf(top, fabsf(x[c][j]));
    top = row_max(top);
    // 2^e with top * 2^e in [2^14, 2^15): f16's largest power of two; 0, inf and subnormal maxima keep e in range
    int e = 14 - (int)((__float_as_uint(top) >> 23) & 255) + 127;
    e = min(max(e, -115), 120);
    // (the sign of the call's scale goes into the operand, so that a larger product is a larger score)
    const float up = copysignf(__uint_as_float((unsigned)(e + 127) << 23), A.scale);
    *unit = fabsf(A.scale) * __uint_as_float((unsigned)(127 - e) << 23);
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
static_assert(kSegBlocks == 256, "a block for each of 4 waves' threads");
// (two steps, so that other loads can be on their way between the page table and the scales; a barrier follows)
__device__ __forceinline__ int64_t find_segment(const AttnArgs& A, int s, int head, int blk0, int n) {
    return (int)threadIdx.x < n ? kv_block(A.kv, s, head, blk0 + threadIdx.x) : 0;
}
__device__ __forceinline__ void load_segment(const AttnArgs& A, Segment& seg, int64_t place, int n) {
    float top = 0.f;
    if ((int)threadIdx.x < n) {
        const float k = A.kv.ks[place], v = A.kv.vs[place];
        seg.place[threadIdx.x] = place;
        seg.ks[threadIdx.x] = k;
        seg.vs[threadIdx.x] = v;
        top = fmaxf(v, 0.f);   // (a NaN scale does not count)
    }
    top = wave_max(top);
    if ((threadIdx.x & 63) == 0) seg.top[threadIdx.x >> 6] = top;
}
template <int WAVES>
__device__ __forceinline__ float segment_top(const Segment& seg) { return WAVES == 1 ? seg.top[0] : fmaxf(fmaxf(seg.top[0], seg.top[1]), fmaxf(seg.top[2], seg.top[3])); }
__device__ __forceinline__ float pow2(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float v) { return (int)(__float_as_uint(v) >> 23) - 127; }   // of a v >= 0
// What value scales below it (0 and NaN among them) lend their exponent from, where the largest one is `top`.
__device__ __forceinline__ float least_scale(float top) { return pow2(max(exponent_of(top) - 100, -90)); }

// References m that the maxima mx of a block's score + e have left behind follow them, and the sums l and o of each row with them.
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
// Where the sums of a row's pieces are, in units of all its pieces; r: the row among its sequence's of the key/value head.  A launch for few
// rows goes by its sequences where the call's other rows, a prompt chunk beside decode steps say, are many times its own.
__device__ __forceinline__ int64_t sums_of(const AttnArgs& A, int s, int kvh, int r, int row, int head) {
    return A.few_rows ? ((int64_t)s * A.kv.kv_heads + kvh) * A.few_rows + r : (int64_t)row * A.q_heads + head;
}
__device__ __forceinline__ int64_t sums_of(const AttnArgs& A, int s, const KvSeq& q, int row, int head) {
    const int kvh = head / A.group;
    return sums_of(A, s, kvh, (row - q.row) * A.group + (head - kvh * A.group), row, head);
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
// A piece's share of one row (of many): the result itself where the sequence is one piece, else sums for attn_join_kernel.
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

// Few rows of each sequence (attn_rows.hip): workgroups of the launch, and the launch with its join.
int rows_per_tile(int dim64, size_t rows);
int rows_residents(int dim64, int tile_rows);   // workgroups of four waves on a CU
int launch_attn_rows(smx_ctx* c, AttnArgs& A, size_t rows, bool bf16);   // rows: of a key/value head, as most sequences have them

}  // namespace smx

// Attention over the paged 8-bit key/value cache: prompt chunks, and the entry point (see attn_dev.h for the arithmetic).
#include <algorithm>
#include <climits>

#include "attn_dev.h"

namespace smx {

namespace {

// The n-th (from 0) of the sequences that are this launch's (or would be, were all their tokens within max_len: looked up by their rows
// alone); -1: there are fewer.
__device__ __forceinline__ int nth_sequence(const AttnArgs& A, int n) {
    for (int base = 0; base < A.kv.nseq; base += 64) {   // a wave looks at 64 at a time
        const int s = base + (threadIdx.x & 63);
        unsigned long long hit = __ballot(s < A.kv.nseq && kv_rows(A.kv, s).n * (int64_t)A.group > A.above);
        const int found = __popcll(hit);
        if (n < found) {
            for (; n > 0; n--) hit &= hit - 1;
            return base + __ffsll((long long)hit) - 1;
        }
        n -= found;
    }
    return -1;
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
    __shared__ float4 value[kSegBlocks];   // of a block's value scale: exponent e, log2(scale 2^(kLift - e)), 1 / (scale 2^kLift), the scale itself
    __shared__ float key_top[4];           // largest key scale of each wave's blocks of the segment
    extern __shared__ uint4 stage[];       // [2][TILE]
    const int s = A.listed ? nth_sequence(A, blockIdx.z) : blockIdx.z, piece = blockIdx.y;
    if (s < 0) return;
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
    float unit[CT], m[CT], l[CT], unit_top = 0.f;
    v4f o[CT][NO];
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        float x[DC][16];
        load_query<DC, BF16>(A, at[ct].live, (int64_t)at[ct].row * A.ldq + (int64_t)at[ct].head * A.kv.dim, x);
        set_query<DC, NT>(A, x, qf[ct], &unit[ct]);
        unit_top = fmaxf(unit_top, unit[ct]);
        m[ct] = kNoMax;
        l[ct] = 0.f;
#pragma unroll
        for (int i = 0; i < NO; i++) o[ct][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    unit_top = wave_max(unit_top);
    // this wave's rows: every one sees [all_lo, all_hi]; none sees a token outside [any_lo, any_hi]
    const int wfirst = pos0 + wrow0 / A.group, wlast = pos0 + min(wrow0 + 16 * CT - 1, rows - 1) / A.group;
    const int all_hi = wfirst, all_lo = A.window > 0 ? wlast - A.window + 1 : 0;
    const int any_hi = wrow0 < rows ? wlast : -1, any_lo = A.window > 0 ? wfirst - A.window + 1 : 0;
    float least = 0.f;
    const int b0 = tok0 / SMX_KV_BLOCK, b1 = tok1 > tok0 ? (tok1 + SMX_KV_BLOCK - 1) / SMX_KV_BLOCK : b0;
    for (int c0 = b0; c0 < b1; c0 += kSegBlocks) {
        const int n = min(kSegBlocks, b1 - c0), tiles = (n + TB - 1) / TB;
        __syncthreads();
        load_segment(A, seg, find_segment(A, s, kvh, c0, n), n);
        const float top = wave_max((int)threadIdx.x < n ? seg.ks[threadIdx.x] : 0.f);   // (a thread's own)
        if (lane == 0) key_top[wave] = top;
        __syncthreads();
        // Scores may be so large that the rounding of the reference is more than what an exponential may exceed it by: they are rounded as it was, on
        // the way of blocks with masks, where a reference of up to 2^24 takes a product that only the FMA rounds.
        const bool far = __ballot(fmaxf(fmaxf(key_top[0], key_top[1]), fmaxf(key_top[2], key_top[3])) * unit_top * (32768.0f * 127 * D64) > 0x1p24f) != 0;
        const int plain_hi = __builtin_amdgcn_readfirstlane(far ? -1 : all_hi);   // blocks up to here need no mask
        least = fmaxf(least, least_scale(segment_top<4>(seg)));
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
        // weights of block i, 2^(scores * f + base), and their product with its values; the sums of probabilities take the value scale
        // out again (per_vs)
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
            const bool edge = tok + SMX_KV_BLOCK - 1 > plain_hi || tok < all_lo;
            const float ks = seg.ks[i];
            const float4 vs = value[i];
            const float exponent = vs.x, log_rest = vs.y, per_vs = vs.z, poison = vs.w == vs.w ? 0.f : vs.w;
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
                mx[ct] = row_max(mx[ct]) * f[ct] + exponent;
            }
            rescale<CT, NO>(mx, m, l, o);
#pragma unroll
            for (int ct = 0; ct < CT; ct++) base[ct] = (exponent - m[ct]) + log_rest;
            if (then) both(cur, nxt, f, base, per_vs, poison, i);
            else weigh(cur, f, base, per_vs, poison, i);
        };
        fetch(0);
        if ((int)threadIdx.x < n) {
            // (a value scale of 0 stands for codes of 0; a NaN one is for the rows that see a token of the block)
            const float scale = seg.vs[threadIdx.x], vs = fmaxf(scale, least);
            const int e = exponent_of(vs);
            value[threadIdx.x] = make_float4((float)e, __builtin_amdgcn_logf(vs * pow2(kLift - e)), __builtin_amdgcn_rcpf(vs) * (1.0f / (1 << kLift)), scale);
        }
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
    constexpr float down = 1.0f / (1 << kLift);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        const float L = row_sum(l[ct]);
#pragma unroll
        for (int i = 0; i < NO; i++) put_row<BF16>(A, at[ct], piece, max(sp.pieces, 1), i * 16 + g * 4, o[ct][i] * down, m[ct], L, i == 0 && g == 0);
    }
}

// The sequence of a row.
__device__ __forceinline__ int seq_of_row(const KvArgs& a, int row) {
    if (!a.row0) return row;
    int lo = 0, hi = a.nseq - 1;   // the last one that starts at or before the row
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (a.row0[mid] <= row) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// Up to kJoinFew pieces: dim64 / 4 threads for a (row, head), each with 4 channels of every piece.  A workgroup for each (row, head) as
// below / this: 96 rows of 16 sequences in 2 pieces 47 / 34 us with the attention, 24 rows of 4 in 7 pieces 25 / 21; more pieces than that
// (64 for one row) 58 / 64.
constexpr int kJoinFew = 16;
template <bool BF16>
__global__ __launch_bounds__(256) void attn_join_few_kernel(const AttnArgs A) {
    const int quads = A.kv.dim64 >> 2, nth = threadIdx.x / quads, units = 256 / quads, d = (threadIdx.x - nth * quads) * 4;   // quads: 16, 32, 48 or 64
    const int unit = blockIdx.x * units + nth, row = unit / A.q_heads, head = unit - row * A.q_heads;
    if (nth >= units || row >= A.kv.rows) return;
    const int s = seq_of_row(A.kv, row);
    const Span sp = seq_span(A, s);
    if (sp.pieces <= 1 || row >= sp.q.row + sp.q.n) return;
    const int64_t at = sums_of(A, s, sp.q, row, head) * A.pieces;
    float M = kNoMax, L = 0.f;
#pragma unroll 4
    for (int i = 0; i < sp.pieces; i++) M = fmaxf(M, A.part_ml[at + i].x);
    v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
    const float* from = A.part + at * A.kv.dim64 + d;
#pragma unroll 4
    for (int i = 0; i < sp.pieces; i++) {
        const float2 ml = A.part_ml[at + i];
        const float f = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);   // (a piece without a key for the row)
        acc += *(const v4f*)(from + (int64_t)i * A.kv.dim64) * f;
        L += ml.y * f;
    }
    RowAt r;
    r.row = row; r.head = head; r.pos = 0; r.live = true;
    store_out<BF16>(A, r, d, acc * (L > 0.f ? 1.0f / L : L == L ? 0.f : L));
}

// Workgroup (row, head): the pieces of a long sequence joined.  Every piece's factor is formed first, so that nothing stands between
// the loads of their sums; 16 bytes for each thread, several pieces at a time.
template <bool BF16>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnArgs A) {
    __shared__ float factor[kMaxPieces], red[2][4];
    __shared__ v4f sums[256];
    const int row = blockIdx.x, head = blockIdx.y, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int s = seq_of_row(A.kv, row);
    const Span sp = seq_span(A, s);
    if (sp.pieces <= 1 || row >= sp.q.row + sp.q.n) return;
    const int64_t at = sums_of(A, s, sp.q, row, head) * A.pieces;
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
int launch_tile(smx_ctx* c, const AttnArgs& A, dim3 grid) {
    const size_t lds = 2 * (DC <= 2 ? 2 : 1) * (2 * DC * 2 + DC * 4) * 1024;
    int rc;
    if ((rc = set_dyn_lds(c, attn_tile_kernel<DC, CT, NT, BF16>, lds)) != SMX_OK) return rc;
    hipLaunchKernelGGL((attn_tile_kernel<DC, CT, NT, BF16>), grid, dim3(256), lds, c->stream, A);
    return SMX_OK;
}
// Column tiles of a wave: as many as leave two waves a SIMD their registers (queries and sums are 8 CT DC NT and 16 CT DC of 256).
// f32 rows of 65..128 channels spill 47 of them: values that are reloaded once a tile or a segment, none between the matrix instructions.
constexpr int most_wave_tiles(int dc) { return dc <= 2 ? 2 : 1; }
// Rows of a workgroup in units of 64: 128 (they share each widened byte), or 64 where the work does not fill the chip for long, which makes
// more workgroups with a shorter way each.  The measure is pairs of a row and a key for each CU; f32 rows of 65..128 channels stay with 64
// for longer, since 128 of them spill some registers.  us at 64 / 128 rows, 32 heads over 8 key/value heads of 128 channels, bf16 and f32:
// 32 tokens behind 4000 21 / 26 and 23 / 30, 40 tokens of 4 sequences of 4000 41 / 40 and 49 / 59, 96 of 4 of 16000 230 / 158 and
// 296 / 218, 512 of 4 of 16000 882 / 658 and 1135 / 978.
int tile_waves(const smx_ctx* c, const AttnArgs& A, size_t nseq, size_t rows, size_t reach, bool bf16) {
    const int dc = A.kv.dim64 / 64;
    const double pairs = (double)nseq * A.kv.kv_heads * (double)rows * (double)reach / c->num_cu;
    return pairs < (dc == 2 && !bf16 ? 4e5 : 1e5) ? 1 : most_wave_tiles(dc);
}
template <int DC>
int launch_dim(smx_ctx* c, const AttnArgs& A, dim3 grid, bool bf16) {
    if (A.tile_rows == 64) return bf16 ? launch_tile<DC, 1, 1, true>(c, A, grid) : launch_tile<DC, 1, 2, false>(c, A, grid);
    return bf16 ? launch_tile<DC, most_wave_tiles(DC), 1, true>(c, A, grid) : launch_tile<DC, most_wave_tiles(DC), 2, false>(c, A, grid);
}

// Tokens that are worth a second workgroup on a CU (a workgroup's start and its share of the join cost as much as some 200).  us at one
// workgroup a CU / two, with the pieces' tokens.  Few rows (24 of 80 channels, 4 key/value heads): 1 sequence of 16000 tokens
// 18.2 / 20.5 (256 / 128), 5 of 4000 18.9 / 20.3 (384 / 256), 20 of 4000 31.1 / 31.0 (1408 / 768), 5 of 16000 29.7 / 29.2
// (1408 / 640); 72 rows, 20 of 16000 174 / 120.  Many rows (40 tokens of 32 heads of 128 channels, 8 key/value heads): 1 of 4000
// 27.8 / 31.0 (256 / 128), 1 of 16000 47 / 40 (1024 / 512), 4 of 4000 52 / 45 (1024 / 512).
constexpr size_t kWorthFew = 512, kWorthMany = 256;
// Contexts that are not split at all: the join costs more than it shortens.  Whole / in pieces of 128 tokens, 4 sequences: one row of 200
// tokens 8.8 / 10.2, of 350 9.8 / 10.3, of 600 11.8 / 11.4; 64 rows of 200 15.6 / 22.3, of 350 19.7 / 22.7, of 600 26.4 / 26.1.
constexpr size_t kWhole = 384;

// Contexts up to which (sequence, key/value head) pairs, where they are more than workgroups of four waves have places at once, take a wave
// each: four waves of a pair have a block or two each and then their sums to put together.  Four waves / one, one row of 32/8 heads of
// 128 channels: 128 sequences of 50 tokens 15 / 10, of 200 21 / 16, 1000 of 100 98 / 53, of 300 154 / 133, of 500 208 / 203, of 800
// 307 / 305, of 20..800 188 / 192.  Where it loses: two column tiles or 64 channels, 350..512 tokens and few more pairs than places (96/4 heads of
// 64, 564 pairs of 512 tokens 24 / 28), and 256 channels at four times the places (109 / 124).
// A window makes longer contexts alike too.  There single waves win while four would begin a second round that does not fill the chip (up to
// 2 rounds), if together they have bytes enough on the way, which goes by pairs times channels (kLoneBytes).  Four waves / one, windows of
// 512, 1024 and 2048:
//   16/8 heads of 256, bf16 (512 places): 640 pairs 44/38 73/67 133/126, 768 48/44 85/83 150/149, 1024 58/56 108/107 195/193, 1280 77/71 132/131 239/247
//   32/8 heads of 128, f32 (768 places): 896 32/26 49/44 99/94, 1024 34/27 54/48 108/100, 1280 38/36 67/67 130/130, 3200 97/99 166/182 310/345
//   16/8 heads of 192, bf16 (512): 576 35/30 53/48 103/101, 768 40/33 63/58 123/114, 1024 46/41 86/80 150/147
//   96/4 heads of 128, f32 (512, two column tiles: only the shorter windows): 576 39/41 52/67 88/122, 896 47/41 65/69 120/130, 1024 48/42 74/69 131/138
//   32/4 heads of 64, bf16 (1024): 1280 24/24 36/38 70/78, 1600 27/24 41/39 85/86, 2048 31/27 51/48 105/103
// and at a window of 4096, which stays with four: 128 channels 183/177, 197/190, 240/250; 256 245/234, 280/281, 373/371.
constexpr size_t kLone = 512, kLoneWindow = 2112, kLoneWindowTwo = 576, kLoneBytes = 7 << 14;
// Tokens of 128 channels of a piece, however many sequences there are: the call knows the longest only, and one long sequence among short ones
// would keep a few workgroups busy for long after the others.  One row each of 64 sequences of 500 tokens and one of 131072: 145 us, without
// 1163; 64 of 33..32768 430 / 462; where all are alike it costs a little: 64 of 16384 394 / 370.
constexpr size_t kLongest = 8192, kMostSums = size_t(256) << 20;

// Rows of a key/value head up to which attn_rows_kernel serves a sequence, and sequences up to which a launch's own are looked up among them.
constexpr size_t kFewRows = 64, kListed = 4096;

// One kernel's share of a call and the join behind it.  nseq, rows: sequences and their rows of a key/value head, as far as the call tells
// (what is split how follows from them; the kernels go by the device's arrays).
int attend(smx_ctx* c, AttnArgs A, size_t nseq, size_t rows, size_t reach, bool few, bool bf16) {
    int rc;
    const int dc = A.kv.dim64 / 64;
    const size_t all = A.kv.nseq, top = few ? std::min<size_t>((size_t)A.kv.max_rows * A.group, kFewRows) : (size_t)A.kv.max_rows * A.group;
    A.tile_rows = few ? rows_per_tile(A.kv.dim64, rows) : 64 * tile_waves(c, A, nseq, rows, reach, bf16);
    A.row_tiles = (int)((top + A.tile_rows - 1) / A.tile_rows);
    // how many workgroups the sequences make without a split
    const size_t groups = nseq * A.kv.kv_heads * ((rows + A.tile_rows - 1) / A.tile_rows);
    // one to a CU, or two where that leaves each enough tokens; never a few more than that, which would wait for a round of their own
    const size_t cus = c->num_cu, span = std::max<size_t>(reach, 1);
    size_t split = std::max<size_t>(1, cus / groups);
    if (span <= kWhole) split = 1;
    else if (2 * cus / groups > split && span / (2 * cus / groups) >= (few ? kWorthFew : kWorthMany)) split = 2 * cus / groups;
    // and no piece is longer than kLongest to 2 kLongest; all of it as far as there is room for the pieces' sums.  Each of the call's rows has a
    // place for its own; of few rows beside many it is each that a sequence may have (one chunk of 8192 rows and a decode step of 32 heads of
    // 128 channels at 100000 tokens: 4.4 GB the first way, 17 MB the second)
    const size_t outputs = (size_t)A.kv.rows * A.q_heads, each = (size_t)A.kv.dim64 * 4 + 8, by_seq = all * A.kv.kv_heads * top;
    A.few_rows = few && by_seq < outputs ? (int)top : 0;
    const size_t kept = A.few_rows ? by_seq : outputs;
    split = std::max(split, span * A.kv.dim64 / 128 / kLongest);
    split = std::min({split, std::max<size_t>(1, kMostSums / (kept * each)), (size_t)kMaxPieces});
    const size_t places = cus * rows_residents(A.kv.dim64, A.tile_rows);
    const bool alike = A.window > 0 && span <= (A.tile_rows == 16 ? kLoneWindow : kLoneWindowTwo) && groups <= 2 * places && groups * A.kv.dim64 >= kLoneBytes;
    A.lone = few && groups > places && (span <= kLone || alike);
    const size_t piece = std::max<size_t>(((span + split - 1) / split + 127) & ~size_t(127), 128);
    A.piece = (int)std::min<size_t>(piece, size_t(1) << 30);
    A.pieces = (int)std::max<size_t>((reach + piece - 1) / piece, 1);
    if (A.pieces > 1) {
        const size_t n = kept * (size_t)A.pieces;
        if ((rc = ensure(c, c->work, n * each)) != SMX_OK) return rc;
        A.part = (float*)c->work.p;
        A.part_ml = (float2*)(A.part + n * A.kv.dim64);
    }
    if (few) {
        rc = launch_attn_rows(c, A, rows, bf16);
    } else {
        A.paired = groups * (size_t)A.pieces <= 2 * cus && A.pieces == 1;
        const size_t z = A.listed ? std::min<size_t>(all, std::max<size_t>(1, (size_t)A.kv.rows * A.group / (A.above + 1))) : all;
        const dim3 grid((unsigned)(A.kv.kv_heads * A.row_tiles), (unsigned)A.pieces, (unsigned)z);
        ProfScope ps(c, "attn_tile");
        switch (dc) {
            case 1: rc = launch_dim<1>(c, A, grid, bf16); break;
            case 2: rc = launch_dim<2>(c, A, grid, bf16); break;
            case 3: rc = launch_dim<3>(c, A, grid, bf16); break;
            default: rc = launch_dim<4>(c, A, grid, bf16); break;
        }
    }
    if (rc != SMX_OK) return rc;
    SMX_HIP(c, hipGetLastError());
    if (A.pieces > 1 && !A.join) {
        ProfScope ps(c, "attn_join");
        if (A.pieces <= kJoinFew) {
            const size_t units = 256 / (A.kv.dim64 / 4);
            const dim3 jg((unsigned)((outputs + units - 1) / units));
            if (bf16) hipLaunchKernelGGL(attn_join_few_kernel<true>, jg, dim3(256), 0, c->stream, A);
            else hipLaunchKernelGGL(attn_join_few_kernel<false>, jg, dim3(256), 0, c->stream, A);
        } else {
            const dim3 jg((unsigned)A.kv.rows, (unsigned)A.q_heads);
            if (bf16) hipLaunchKernelGGL(attn_join_kernel<true>, jg, dim3(256), 0, c->stream, A);
            else hipLaunchKernelGGL(attn_join_kernel<false>, jg, dim3(256), 0, c->stream, A);
        }
        SMX_HIP(c, hipGetLastError());
    }
    return SMX_OK;
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
    // (rows of a head's group are counted in 32 bits)
    if (batch->rows * q_heads >= (size_t(1) << 31)) return fail(c, SMX_ERR_LIMIT, "attn_dev: %zu rows of %zu query heads (2^31 in all)", batch->rows, q_heads);
    if (!q || !out) return fail(c, SMX_ERR_ARG, "attn_dev: null queries or result");
    const bool bf16 = type == SMX_TYPE_BF16;
    A.q = q; A.out = out; A.ldq = (int64_t)ldq; A.ldo = (int64_t)ldo;
    A.q_heads = (int)q_heads;
    A.group = (int)(q_heads / cache->kv_heads);
    A.window = (int)std::min<size_t>(window, INT_MAX / 2);
    A.scale = scale * kLog2e;
    const size_t per16 = bf16 ? 8 : 4;
    A.vec = cache->head_dim % 16 == 0 && ldq % per16 == 0 && ldo % per16 == 0 && (((uintptr_t)q | (uintptr_t)out) & 15) == 0;
    // tokens in reach of one sequence's rows
    const size_t reach = window ? std::min<size_t>(A.kv.max_len, (size_t)A.window + batch->max_rows + SMX_KV_BLOCK) : (size_t)A.kv.max_len;
    const size_t most = batch->max_rows * (size_t)A.group;
    A.upto = INT_MAX;
    if (most <= kFewRows) return attend(c, A, batch->nseq, most, reach, true, bf16);
    // Sequences of few rows in a call that has longer ones get the launch for few rows to themselves (in tiles of 64 or 128 rows, 63 decode
    // steps beside a prompt chunk took 1169 us where each alone takes 100).  A call whose rows are all alike has none.
    if (batch->rows < batch->nseq * batch->max_rows && (size_t)A.group <= kFewRows) {
        AttnArgs F = A;
        F.upto = (int)kFewRows;
        if ((rc = attend(c, F, batch->nseq, A.group, reach, true, bf16)) != SMX_OK) return rc;
        A.above = (int)kFewRows;
        A.listed = batch->nseq <= kListed;
        // the longer ones, were the others of one row and these of max_rows
        const size_t longer = (batch->rows - std::min(batch->rows, batch->nseq) + batch->max_rows - 2) / (batch->max_rows - 1);
        return attend(c, A, std::max<size_t>(longer, 1), most, reach, false, bf16);
    }
    return attend(c, A, batch->nseq, most, reach, false, bf16);
}

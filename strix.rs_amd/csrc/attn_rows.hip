// Attention over the paged 8-bit key/value cache for few rows of each sequence: a decode step, a handful of drafted tokens (see
// attn_dev.h for the arithmetic).  Bound by the cache that it reads, once for all rows of a tile: 541 MB (64 sequences of
// 33..8192 tokens) in 120 us, the same in sequences of one length in 101 us (5.4 TB/s), one sequence of 65536 tokens (269 MB)
// in 52 us + 4.5 us for joining its pieces.  What the ragged batch loses is the longest sequences' end, where less than all of the
// chip reads.  Pieces of 4096, 2048 and 1024 tokens instead of whole sequences took 119, 126 and 121 us (and 115, 109 and 121 us for
// the even batch): what a better balance wins, the starts of more workgroups lose.  All blocks dealt out evenly to
// workgroups that stay took 141 us.
#include <algorithm>

#include "attn_dev.h"

namespace smx {

namespace {

// The pieces of a row tile are joined by the last of its workgroups to finish where they are few, by a launch of their own else: sums
// that another XCD shall see are written and read word by word.  One sequence, 8 key/value heads of 128 channels, us inside /
// us launched: 4 rows in 4 pieces 11.0 / 12.6, in 8 pieces 11.8 / 12.8, in 16 pieces 13.3 / 13.4; 8 rows in 4 pieces 12.2 / 12.8, in
// 8 pieces 13.0 / 13.2; 16 rows in 4 pieces 14.0 / 12.9, in 8 pieces 15.8 / 12.5.
constexpr int kJoinInside = 16;      // pieces
constexpr int kJoinRows = 32;        // rows times pieces

// Sums pass from workgroup to workgroup as words that are atomic at device scope: written to, and read from, where all XCDs see them, each
// thread's waited for before the workgroup counts itself.  That such a store has arrived once it has been waited for is the hardware's
// (gfx950 writes it through its L2); in the language's terms it is no release, which would write the XCD's whole L2 back instead.
__device__ __forceinline__ void give(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float take(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ float row16_max(float v) {   // of 16 lanes
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float over(float L) { return L > 0.f ? 1.0f / L : L == L ? 0.f : L; }   // (a NaN stays one)

// Waves on a SIMD: what the registers leave.  (f32 rows of 193..256 channels spill 24 of them, in front of the loop over blocks and behind it.)
constexpr int residents(int dc, int ct) { return ct == 2 ? 2 : dc <= 1 ? 4 : dc == 2 ? 3 : 2; }

// Workgroup (head and tile of 16 CT rows, piece of the context, sequence); its four waves (or one) take the piece's blocks in turn, straight
// from memory into the matrix instructions' registers (one block ahead), and add up through LDS at the end.
template <int DC, int CT, int NT, int WAVES, bool BF16>
__global__ __launch_bounds__(WAVES * 64, residents(DC, CT)) void attn_rows_kernel(const AttnArgs A) {
    constexpr int D64 = DC * 64, NO = DC * 4, ROWS = 16 * CT, PITCH = D64 + 4, SEG = kSegBlocks * WAVES / 4;
    __shared__ Segment seg;
    __shared__ float wm[WAVES][ROWS], wl[WAVES][ROWS];
    __shared__ unsigned last;
    extern __shared__ float wo[];   // [WAVES][16][PITCH], one column tile at a time
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4;
    const int s = blockIdx.z, piece = blockIdx.y;
    // (Sequences of fewer rows leave tiles empty: which of a sequence's workgroups those are goes round, since workgroups go to the parts of the
    // chip in turn, and one in four at work would meet on a quarter of it: 188 us where all sequences of one row take 96.)
    const int kvh = blockIdx.x % A.kv.kv_heads, tile = (blockIdx.x / A.kv.kv_heads + s) % A.row_tiles;
    const Span sp = seq_span(A, s);
    const int rows = sp.q.n * A.group;
    if (tile * ROWS >= rows) return;
    if (piece >= sp.pieces) {
        if (piece == 0) {   // a sequence without a token in the cache
            for (int it = threadIdx.x; it < min(ROWS, rows - tile * ROWS) * (D64 / 4); it += WAVES * 64) {
                const int r = it / (D64 / 4);
                store_out<BF16>(A, row_at(A, sp.q, kvh, tile * ROWS + r), (it - r * (D64 / 4)) * 4, v4f{0.f, 0.f, 0.f, 0.f});
            }
        }
        return;
    }
    RowAt at[CT];
    v8h qf[CT][NT][DC * 2];
    float unit[CT], m[CT], l[CT];
    v4f o[CT][NO];
    // every row of the tile sees keys [all_lo, all_hi]: blocks inside need no mask
    const int pos0 = sp.q.len - sp.q.n;
    const int all_hi = pos0 + tile * ROWS / A.group, all_lo = A.window > 0 ? pos0 + min(tile * ROWS + ROWS - 1, rows - 1) / A.group - A.window + 1 : 0;
    float least = 0.f;
    const int tok0 = sp.first + piece * A.piece, tok1 = min(tok0 + A.piece, sp.q.len);
    const int b0 = tok0 / SMX_KV_BLOCK, b1 = (tok1 + SMX_KV_BLOCK - 1) / SMX_KV_BLOCK;
    // a block's bytes are asked for as soon as the registers of the one in front are free: keys behind its scores, values behind
    // its second product
    uint4 kb[2 * DC], vb[2 * DC];
    auto fetch = [&](uint4 (&to)[2 * DC], const int8_t* plane, int i) {
        const int8_t* base = plane + uniform(seg.place[i]) * (SMX_KV_BLOCK * D64);
#pragma unroll
        for (int j = 0; j < 2 * DC; j++) to[j] = *(const uint4*)(base + (unsigned)(j * 1024 + lane * 16));
    };
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        float x[DC][16];
        at[ct] = row_at(A, sp.q, kvh, (tile * CT + ct) * 16 + (lane & 15));
        load_query<DC, BF16>(A, at[ct].live, (int64_t)at[ct].row * A.ldq + (int64_t)at[ct].head * A.kv.dim, x);
        set_query<DC, NT>(A, x, qf[ct], &unit[ct]);
        m[ct] = kNoMax;
        l[ct] = 0.f;
#pragma unroll
        for (int i = 0; i < NO; i++) o[ct][i] = v4f{0.f, 0.f, 0.f, 0.f};
    }
    for (int c0 = b0; c0 < b1; c0 += SEG) {
        const int n = min(SEG, b1 - c0);
        if (c0 != b0) __syncthreads();
        load_segment(A, seg, find_segment(A, s, kvh, c0, n), n);
        __syncthreads();
        if (wave < n) {
            fetch(kb, A.kv.k, wave);
            fetch(vb, A.kv.v, wave);
        }
        least = fmaxf(least, least_scale(segment_top<WAVES>(seg)));
        for (int i = wave; i < n; i += WAVES) {
            v4f sc[CT][2];
#pragma unroll
            for (int tt = 0; tt < 2; tt++) {
                v8h kf[DC * 2];
#pragma unroll
                for (int c = 0; c < DC; c++) {
                    const uint4 u = kb[tt * DC + c];
                    kf[c * 2] = widen8(u.x, u.y);
                    kf[c * 2 + 1] = widen8(u.z, u.w);
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
            const float ks = seg.ks[i], vs = seg.vs[i];
            const int e = exponent_of(fmaxf(vs, least));
            const float exponent = (float)e, rest = vs * pow2(kLift - e), inverse = pow2(-e);
            const int next = i + WAVES;
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
                mx[ct] = row_max(mx[ct]) + exponent;
            }
            rescale<CT, NO>(mx, m, l, o);
            v8h pf[CT][NT];
#pragma unroll
            for (int ct = 0; ct < CT; ct++) {
                const float base = exponent - m[ct];
                float p[8], sum = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    const float e2 = __builtin_amdgcn_exp2f(t[ct][j] + base);
                    sum += e2;
                    p[j] = edge && t[ct][j] == -INFINITY ? 0.f : e2 * rest;   // (a masked token's value scale may be NaN)
                }
                l[ct] = fmaf(sum, inverse, l[ct]);
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
    // the four waves' shares of the piece
    constexpr float down = 1.0f / (1 << kLift);
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        l[ct] = row_sum(l[ct]);
        if (g == 0) {
            wm[wave][ct * 16 + lane] = m[ct];
            wl[wave][ct * 16 + lane] = l[ct];
        }
    }
#pragma unroll
    for (int ct = 0; ct < CT; ct++) {
        __syncthreads();
        const int r = ct * 16 + (lane & 15);
        float M = wm[0][r];
#pragma unroll
        for (int v = 1; v < WAVES; v++) M = fmaxf(M, wm[v][r]);
        const float f = __builtin_amdgcn_exp2f(m[ct] - M) * down;
#pragma unroll
        for (int i = 0; i < NO; i++) *(v4f*)&wo[(wave * 16 + (lane & 15)) * PITCH + i * 16 + g * 4] = o[ct][i] * f;
        float L = 0.f;
#pragma unroll
        for (int v = 0; v < WAVES; v++) L += wl[v][r] * __builtin_amdgcn_exp2f(wm[v][r] - M);
        __syncthreads();
        if (!at[ct].live) continue;
        const int64_t mine = sums_of(A, s, kvh, tile * ROWS + r, at[ct].row, at[ct].head) * A.pieces + piece;
        if (sp.pieces > 1 && wave == 0 && g == 0) {
            give(&A.part_ml[mine].x, M);
            give(&A.part_ml[mine].y, L);
        }
        // wave w writes channels [w * D64 / WAVES, ...)
#pragma unroll
        for (int i = 0; i < NO / WAVES; i++) {
            const int d = (wave * (NO / WAVES) + i) * 16 + g * 4;
            v4f acc = *(v4f*)&wo[(lane & 15) * PITCH + d];
#pragma unroll
            for (int v = 1; v < WAVES; v++) acc += *(v4f*)&wo[(v * 16 + (lane & 15)) * PITCH + d];
            if (sp.pieces == 1) {
                store_out<BF16>(A, at[ct], d, acc * over(L));
            } else {
                float* to = A.part + mine * D64 + d;
                if (A.join) {
#pragma unroll
                    for (int j = 0; j < 4; j++) give(to + j, acc[j]);
                } else {
                    *(v4f*)to = acc;
                }
            }
        }
    }
    if (sp.pieces == 1 || !A.join) return;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // this thread's words have arrived
    __syncthreads();
    unsigned* count = A.count + ((int64_t)s * A.kv.kv_heads * A.row_tiles + blockIdx.x);
    if (threadIdx.x == 0) last = atomicAdd(count, 1u) == (unsigned)sp.pieces - 1;
    __syncthreads();
    if (!last) return;
    if (threadIdx.x == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    // factors of all (row, piece) first, so that nothing stands between the loads of the sums
    const int live = min(ROWS, rows - tile * ROWS);
    float2* factor = (float2*)wo;   // [ROWS][kJoinInside], x: the factor, y: the piece's share of the row's sum
    for (int it = threadIdx.x; it < live * kJoinInside; it += WAVES * 64) {
        const int r = it / kJoinInside, i = it - r * kJoinInside;
        float2 ml = make_float2(kNoMax, 0.f);
        if (i < sp.pieces) {
            const RowAt x = row_at(A, sp.q, kvh, tile * ROWS + r);
            const float2* from = A.part_ml + sums_of(A, s, kvh, tile * ROWS + r, x.row, x.head) * A.pieces + i;
            ml = make_float2(take(&from->x), take(&from->y));
        }
        const float M = row16_max(ml.x);
        const float f = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - M);   // (a piece without a key for the row)
        factor[it] = make_float2(f, ml.y * f);
    }
    __syncthreads();
    constexpr int QUADS = D64 / 4, GROUPS = WAVES * 64 / QUADS;
    const int gr = threadIdx.x / QUADS, d = (threadIdx.x - gr * QUADS) * 4;
    for (int r = gr; r < live && gr < GROUPS; r += GROUPS) {
        const RowAt x = row_at(A, sp.q, kvh, tile * ROWS + r);
        const float* from = A.part + sums_of(A, s, kvh, tile * ROWS + r, x.row, x.head) * A.pieces * D64 + d;
        v4f acc = v4f{0.f, 0.f, 0.f, 0.f};
        float L = 0.f;
        for (int i = 0; i < sp.pieces; i += 4) {
            v4f t[4];
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float* p = from + min(i + k, sp.pieces - 1) * D64;
                t[k] = v4f{take(p), take(p + 1), take(p + 2), take(p + 3)};
            }
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float2 f = i + k < sp.pieces ? factor[r * kJoinInside + i + k] : make_float2(0.f, 0.f);
                if (i + k < sp.pieces) acc += t[k] * f.x;
                L += f.y;
            }
        }
        store_out<BF16>(A, x, d, acc * over(L));
    }
}

__global__ __launch_bounds__(256) void clear_kernel(unsigned* p, size_t n) {
    const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (i < n) p[i] = 0;
}

template <int DC, int CT, int NT, int WAVES, bool BF16>
int launch(smx_ctx* c, const AttnArgs& A, dim3 grid) {
    const size_t lds = WAVES * 16 * (DC * 64 + 4) * 4;
    int rc;
    if ((rc = set_dyn_lds(c, attn_rows_kernel<DC, CT, NT, WAVES, BF16>, lds)) != SMX_OK) return rc;
    hipLaunchKernelGGL((attn_rows_kernel<DC, CT, NT, WAVES, BF16>), grid, dim3(WAVES * 64), lds, c->stream, A);
    return SMX_OK;
}
// Two column tiles to a wave where their registers leave two waves a SIMD (and the second tile's products share the widened bytes).
constexpr int most_tiles(int dc) { return dc <= 2 ? 2 : 1; }
template <int DC, int WAVES>
int launch_tiles(smx_ctx* c, const AttnArgs& A, dim3 grid, bool bf16) {
    if (A.tile_rows == 16) return bf16 ? launch<DC, 1, 1, WAVES, true>(c, A, grid) : launch<DC, 1, 2, WAVES, false>(c, A, grid);
    return bf16 ? launch<DC, most_tiles(DC), 1, WAVES, true>(c, A, grid) : launch<DC, most_tiles(DC), 2, WAVES, false>(c, A, grid);
}
template <int DC>
int launch_dim(smx_ctx* c, const AttnArgs& A, dim3 grid, bool bf16) {
    return A.lone ? launch_tiles<DC, 1>(c, A, grid, bf16) : launch_tiles<DC, 4>(c, A, grid, bf16);
}

}  // namespace

int rows_per_tile(int dim64, size_t rows) { return rows <= 16 ? 16 : 16 * most_tiles(dim64 / 64); }

int rows_residents(int dim64, int tile_rows) { return residents(dim64 / 64, tile_rows / 16); }

int launch_attn_rows(smx_ctx* c, AttnArgs& A, size_t rows, bool bf16) {
    int rc;
    const size_t items = (size_t)A.kv.nseq * A.kv.kv_heads * A.row_tiles;
    A.join = A.pieces > 1 && A.pieces <= kJoinInside && (size_t)A.pieces * rows <= (size_t)kJoinRows;
    if (A.join) {
        const size_t had = c->counts.cap;
        if ((rc = ensure(c, c->counts, items * 4)) != SMX_OK) return rc;
        if (c->counts.cap != had) {
            const size_t words = c->counts.cap / 4;
            hipLaunchKernelGGL(clear_kernel, dim3((unsigned)((words + 255) / 256)), dim3(256), 0, c->stream, (unsigned*)c->counts.p, words);
            SMX_HIP(c, hipGetLastError());
        }
        A.count = (unsigned*)c->counts.p;
    }
    const dim3 grid((unsigned)(A.kv.kv_heads * A.row_tiles), (unsigned)A.pieces, (unsigned)A.kv.nseq);
    ProfScope ps(c, "attn_rows");
    switch (A.kv.dim64 / 64) {
        case 1: rc = launch_dim<1>(c, A, grid, bf16); break;
        case 2: rc = launch_dim<2>(c, A, grid, bf16); break;
        case 3: rc = launch_dim<3>(c, A, grid, bf16); break;
        default: rc = launch_dim<4>(c, A, grid, bf16); break;
    }
    if (rc != SMX_OK) return rc;
    SMX_HIP(c, hipGetLastError());
    return SMX_OK;
}

}  // namespace smx

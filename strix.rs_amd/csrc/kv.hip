// The paged 8-bit key/value cache: a step's keys and values appended with their position rotation, stored values read back.
#include <algorithm>
#include <climits>
#include <type_traits>

#include "kv_dev.h"

namespace smx {

int kv_args(smx_ctx* c, const char* who, const smx_kv_cache* cache, const smx_kv_batch* b, KvArgs* out) {
    if (!cache || !b) return fail(c, SMX_ERR_ARG, "%s: null cache or batch", who);
    if (!cache->k || !cache->v || !cache->k_scale || !cache->v_scale) return fail(c, SMX_ERR_ARG, "%s: null cache plane", who);
    size_t code_bytes, scales;
    if (smx_kv_sizes(cache->pages, cache->page_tokens, cache->kv_heads, cache->head_dim, &code_bytes, &scales) != SMX_OK)
        return fail(c, SMX_ERR_ARG, "%s: cache of %zu pages of %zu tokens (a multiple of %d), %zu heads of %zu channels (even, up to %d)", who,
                    cache->pages, cache->page_tokens, SMX_KV_BLOCK, cache->kv_heads, cache->head_dim, SMX_KV_MAX_HEAD_DIM);
    if (((uintptr_t)cache->k | (uintptr_t)cache->v) & 15) return fail(c, SMX_ERR_ARG, "%s: code planes must be 16-byte aligned", who);
    if (b->nseq == 0) return SMX_OK;   // nothing to do
    if (!b->len || !b->table) return fail(c, SMX_ERR_ARG, "%s: null length or page table", who);
    if (b->table_ld == 0) return fail(c, SMX_ERR_ARG, "%s: empty page table", who);
    if (!b->row0 && (b->rows != b->nseq || b->max_rows != 1))
        return fail(c, SMX_ERR_ARG, "%s: %zu rows (at most %zu each) of %zu sequences without row0", who, b->rows, b->max_rows, b->nseq);
    if (b->max_rows > b->rows || (b->max_rows == 0 && b->rows > 0)) return fail(c, SMX_ERR_ARG, "%s: max_rows %zu of %zu rows", who, b->max_rows, b->rows);
    if (b->nseq > 65535 || b->rows > (size_t(1) << 24) || b->max_len > (size_t(1) << 28) || b->table_ld > (size_t(1) << 26) || cache->pages > INT_MAX)
        return fail(c, SMX_ERR_LIMIT, "%s: %zu sequences (65535), %zu rows (2^24), %zu tokens (2^28), %zu pages (2^31 - 1)", who, b->nseq, b->rows,
                    b->max_len, cache->pages);
    KvArgs a;
    a.k = cache->k; a.v = cache->v; a.ks = cache->k_scale; a.vs = cache->v_scale;
    a.len = b->len; a.row0 = b->row0; a.table = b->table;
    a.table_ld = (int)b->table_ld; a.pages = (int)cache->pages; a.page_blocks = (int)(cache->page_tokens / SMX_KV_BLOCK);
    a.kv_heads = (int)cache->kv_heads; a.dim = (int)cache->head_dim; a.dim64 = (int)((cache->head_dim + 63) & ~size_t(63));
    a.nseq = (int)b->nseq; a.rows = (int)b->rows; a.max_rows = (int)b->max_rows;
    // a sequence holds no more tokens than its page table names
    a.max_len = (int)std::min<size_t>(b->max_len, b->table_ld * cache->page_tokens);
    *out = a;
    return SMX_OK;
}

namespace {

struct AppendArgs {
    KvArgs kv;
    const void *k, *v, *q;
    void* qo;
    int64_t ldk, ldv, ldq, ldqo;
    const float2* rope;   // [n_pos][rot / 2]; null: no rotation
    int n_pos, rot, q_heads;
    int touched;          // workgroups along x that serve cache blocks; the ones behind them rotate queries
};

// Channels are worked on W pairs at a time: of 16-byte loads where rows, halves and addresses allow it, else a pair.
template <bool BF16, bool VEC>
constexpr int kPairs = VEC ? (BF16 ? 8 : 4) : 1;
constexpr int kQueryItems = 512;   // groups of W pairs for each workgroup of the query rotation

// 2 W channels of a row: a[j], b[j] is pair j of group i (pairs W i ..), rotated.  da, db: channel of a[0], b[0]; the others follow
// them (PAIRS and channels behind the rotated ones: a[j], b[j] are neighbours, a[j] at da + 2 j).
template <bool BF16, bool PAIRS, bool VEC>
struct Group {
    static constexpr int W = kPairs<BF16, VEC>;
    float a[W], b[W];
    float2 c[W];
    uint4 p, q;
    int da, db;
    bool split;   // a and b lie half a rotation apart

    __device__ __forceinline__ void place(int i, int rot) {
        const int half = rot >> 1;
        split = !PAIRS && i * W < half;
        da = split ? i * W : 2 * i * W;
        db = split ? i * W + half : 2 * i * W + 1;
    }
    // asked for: the channels' bytes, and the position's {cos, sin} of the group's pairs (cs: of pair 0; group i is one of the rotated)
    __device__ __forceinline__ void fetch(const void* x, int64_t at) {
        const int64_t second = VEC && !split ? at + da + W : at + db;
        if constexpr (VEC) {
            p = BF16 ? *(const uint4*)((const uint16_t*)x + at + da) : *(const uint4*)((const float*)x + at + da);
            q = BF16 ? *(const uint4*)((const uint16_t*)x + second) : *(const uint4*)((const float*)x + second);
        } else {
            p.x = BF16 ? ((const uint16_t*)x)[at + da] : ((const unsigned*)x)[at + da];
            q.x = BF16 ? ((const uint16_t*)x)[second] : ((const unsigned*)x)[second];
        }
    }
    __device__ __forceinline__ void fetch_turn(const float2* __restrict__ cs, int i) {
#pragma unroll
        for (int j = 0; j < W; j++) c[j] = cs[i * W + j];
    }
    // what has been asked for, as numbers
    __device__ __forceinline__ void open() {
        if constexpr (!VEC) {
            a[0] = __uint_as_float(BF16 ? p.x << 16 : p.x);
            b[0] = __uint_as_float(BF16 ? q.x << 16 : q.x);
        } else {
            float v[2 * W];
            const unsigned u[8] = {p.x, p.y, p.z, p.w, q.x, q.y, q.z, q.w};
#pragma unroll
            for (int j = 0; j < 8; j++) {
                if constexpr (BF16) {
                    v[2 * j] = __uint_as_float(u[j] << 16);
                    v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
                } else {
                    v[j] = __uint_as_float(u[j]);
                }
            }
#pragma unroll
            for (int j = 0; j < W; j++) {
                a[j] = split ? v[j] : v[2 * j];
                b[j] = split ? v[W + j] : v[2 * j + 1];
            }
        }
    }
    __device__ __forceinline__ void turn() {
#pragma clang fp contract(off)
#pragma unroll
        for (int j = 0; j < W; j++) {
            const float x = a[j], y = b[j];
            a[j] = x * c[j].x - y * c[j].y;
            b[j] = x * c[j].y + y * c[j].x;
        }
    }
    // the 2 W channels in memory order: first W at da, the others at second()
    __device__ __forceinline__ int second() const { return split ? db : da + W; }
    __device__ __forceinline__ void ordered(float (&v)[2 * W]) const {
#pragma unroll
        for (int j = 0; j < W; j++) {
            if (split) { v[j] = a[j]; v[W + j] = b[j]; }
            else { v[2 * j] = a[j]; v[2 * j + 1] = b[j]; }
        }
    }
    __device__ __forceinline__ void store(void* y, int64_t at) const {
        if constexpr (!VEC) {
            store_elem<BF16>(y, at + da, a[0]);
            store_elem<BF16>(y, at + db, b[0]);
        } else {
            float v[2 * W];
            ordered(v);
            if constexpr (BF16) {
                unsigned u[8];
#pragma unroll
                for (int j = 0; j < 8; j++) u[j] = f32_to_bf16(v[2 * j]) | (unsigned)f32_to_bf16(v[2 * j + 1]) << 16;
                *(uint4*)((uint16_t*)y + at + da) = make_uint4(u[0], u[1], u[2], u[3]);
                *(uint4*)((uint16_t*)y + at + second()) = make_uint4(u[4], u[5], u[6], u[7]);
            } else {
                *(float4*)((float*)y + at + da) = make_float4(v[0], v[1], v[2], v[3]);
                *(float4*)((float*)y + at + second()) = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
    }
};

// The largest |value| as its bits: NaN and infinity order above every finite value.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Which part of the batch a workgroup serves: block x of those that the sequences' rows lie in, in order.
struct BlockRows {
    int s, blk;       // sequence, block
    int t0, t1;       // the block's tokens that are rows of the batch: [t0, t1), none if t1 <= t0
    int row;          // row of the block's token 0 (may lie in front of the batch's)
};
__device__ __forceinline__ BlockRows block_rows(const KvArgs& a, int x) {
    BlockRows r;
    r.s = x;
    int nth = 0;
    if (a.row0) {   // a wave looks at 64 sequences at a time
        const int lane = threadIdx.x & 63;
        int base = 0, left = x;
        for (;; base += 64) {
            if (base >= a.nseq) { r.t0 = r.t1 = 0; r.s = r.blk = r.row = 0; return r; }
            int n = 0;
            if (base + lane < a.nseq) {
                const KvSeq q = kv_seq(a, base + lane);
                const int first = max(q.len - q.n, 0);
                n = q.len > first ? (q.len - 1) / SMX_KV_BLOCK - first / SMX_KV_BLOCK + 1 : 0;
            }
            int upto = n;
#pragma unroll
            for (int o = 1; o < 64; o <<= 1) {
                const int v = __shfl_up(upto, o);
                if (lane >= o) upto += v;
            }
            const unsigned long long hit = __ballot(upto > left);
            if (hit) {
                const int l = __ffsll((long long)hit) - 1;
                r.s = __builtin_amdgcn_readfirstlane(base + l);
                nth = __builtin_amdgcn_readfirstlane(left - __shfl(upto - n, l));
                break;
            }
            left -= __shfl(upto, 63);
        }
    }
    const KvSeq q = kv_seq(a, r.s);
    const int start = q.len - q.n;                 // may be negative: rows in front of position 0 are left out
    r.blk = max(start, 0) / SMX_KV_BLOCK + nth;
    r.t0 = max(max(start, 0) - r.blk * SMX_KV_BLOCK, 0);
    r.t1 = min(q.len - r.blk * SMX_KV_BLOCK, SMX_KV_BLOCK);
    r.row = q.row + r.blk * SMX_KV_BLOCK - start;
    return r;
}
// Workgroups enough for every block: n rows from the last token of a block on touch (n + 62) / 32.
int touched_blocks(const smx_kv_batch* b) { return b->row0 ? (int)((b->rows + 62 * b->nseq) / SMX_KV_BLOCK) : (int)b->nseq; }

// Workgroup (x, head, keys | values): x < touched is one block of 32 tokens that the step writes into, the others rotate
// kQueryItems groups of channel pairs of the queries each (head and z choose among those).
//
// A block is one workgroup's alone, so its scale, the rounding of earlier codes under a scale that grew and the new codes need no
// atomics: the block's new values stay in registers, their largest gives the scale, and the codes go through LDS (in the layout's
// order) to leave in its 16-byte units (a token's 16 channels of keys; 8 tokens of 2 channels of values).  In a block that is only
// partly new, values go by 4 tokens or single bytes, so that nothing is read back unless the scale grew.
// Bytes bound a prompt chunk (2048 rows of 16 + 16 heads of 256 bf16 channels, 59 MB: 17 us, 20 with the new values in LDS as fp32 and
// loads asked for one group at a time), the launch and a chain of three loads (the step's arrays, its rows, the page) a decode step
// (64 rows of 32 + 16 heads of 128: 6.0 us): what does not depend on another load is asked for in front of it.
template <bool BF16, bool PAIRS, bool VEC>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs A) {
#pragma clang fp contract(off)
    constexpr int W = kPairs<BF16, VEC>, ROUNDS = SMX_KV_BLOCK * SMX_KV_MAX_HEAD_DIM / (2 * W * 256), TURNS = kQueryItems / 256;
    extern __shared__ __align__(16) int8_t image[];   // [SMX_KV_BLOCK * dim64]: the block's new codes
    __shared__ unsigned red[4];
    const KvArgs& a = A.kv;
    const int tid = threadIdx.x, groups = a.dim / (2 * W);
    if ((int)blockIdx.x >= A.touched) {
        const int64_t items = (int64_t)a.rows * A.q_heads * groups;
        const int64_t first = ((((int64_t)blockIdx.x - A.touched) * gridDim.y + blockIdx.y) * gridDim.z + blockIdx.z) * kQueryItems;
        if (first >= items) return;
        // (one division of 64 bits for the workgroup, the threads' own are of 32)
        const unsigned per_row = (unsigned)A.q_heads * (unsigned)groups;   // < 2^23
        const int r0 = (int)(first / per_row);
        const unsigned i0 = (unsigned)(first - (int64_t)r0 * per_row), left = (unsigned)min(items - first, (int64_t)kQueryItems);
        Group<BF16, PAIRS, VEC> g[TURNS];
        int row[TURNS], head[TURNS], nth[TURNS];
#pragma unroll
        for (int j = 0; j < TURNS; j++) {   // (a thread without an item takes the last one and stores nothing)
            const unsigned it = i0 + min(j * 256u + tid, left - 1), over = it / per_row, in = it - over * per_row;
            row[j] = r0 + (int)over;
            head[j] = (int)(in / (unsigned)groups);
            nth[j] = (int)in - head[j] * groups;
            g[j].place(nth[j], A.rot);
            g[j].fetch(A.q, (int64_t)row[j] * A.ldq + (int64_t)head[j] * a.dim);
        }
        if (A.rope) {
#pragma unroll
            for (int j = 0; j < TURNS; j++) {
                int s = row[j];
                if (a.row0) {   // the last sequence that starts at or before the row
                    int lo = 0, hi = a.nseq - 1;
                    while (lo < hi) {
                        const int mid = (lo + hi + 1) >> 1;
                        if (a.row0[mid] <= row[j]) lo = mid; else hi = mid - 1;
                    }
                    s = lo;
                }
                const KvSeq q = kv_seq(a, s);
                const int pos = max(q.len - q.n + row[j] - q.row, 0);
                if (nth[j] * W < A.rot >> 1) g[j].fetch_turn(A.rope + (int64_t)min(pos, A.n_pos - 1) * (A.rot >> 1), nth[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < TURNS; j++) {
            g[j].open();
            if (A.rope && nth[j] * W < A.rot >> 1) g[j].turn();
            if (j * 256u + tid < left) g[j].store(A.qo, (int64_t)row[j] * A.ldqo + (int64_t)head[j] * a.dim);
        }
        return;
    }
    const BlockRows br = block_rows(a, blockIdx.x);
    const int t0 = br.t0, t1 = br.t1;
    if (t1 <= t0) return;
    const int head = blockIdx.y;
    const bool keys = blockIdx.z == 0;
    const int rot = keys && A.rope ? A.rot : 0, n = (t1 - t0) * groups;
    Group<BF16, PAIRS, VEC> g[ROUNDS];
    int tok[ROUNDS], nth[ROUNDS];
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {   // (a thread without an item takes the last one again)
        if (j * 256 >= n) continue;
        const int it = min(j * 256 + tid, n - 1);
        tok[j] = t0 + it / groups;
        nth[j] = it - (tok[j] - t0) * groups;
        g[j].place(nth[j], rot);
        g[j].fetch(keys ? A.k : A.v, (int64_t)(br.row + tok[j]) * (keys ? A.ldk : A.ldv) + (int64_t)head * a.dim);
        if (nth[j] * W < rot >> 1) g[j].fetch_turn(A.rope + (int64_t)min(br.blk * SMX_KV_BLOCK + tok[j], A.n_pos - 1) * (rot >> 1), nth[j]);
    }
    const KvPlace at = kv_place(a, br.s, head, br.blk);
    const int64_t bi = at.block;
    float* sp = (keys ? a.ks : a.vs) + bi;
    const float before = t0 > 0 ? *sp : 0.0f;
    for (int u = tid; u < 2 * a.dim64; u += 256) ((uint4*)image)[u] = make_uint4(0, 0, 0, 0);
    unsigned most = 0;
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {
        if (j * 256 >= n) continue;
        g[j].open();
        if (nth[j] * W < rot >> 1) g[j].turn();
#pragma unroll
        for (int w = 0; w < W; w++) most = max(most, max(abs_bits(g[j].a[w]), abs_bits(g[j].b[w])));
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) most = max(most, (unsigned)__shfl_xor((int)most, o));
    if ((tid & 63) == 0) red[tid >> 6] = most;
    __syncthreads();   // (every thread has read the old scale, too)
    if (at.page < 0 || at.page >= a.pages) return;   // (the same for the workgroup) the clamped one is another sequence's
    most = max(max(red[0], red[1]), max(red[2], red[3]));
    const float top = __uint_as_float(most);
    const float fresh = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : top >= 0x1p-96f ? top / 127.0f : 0.0f;
    float scale = fresh, ratio = 1.0f;
    bool grown = false;
    if (t0 > 0) {
        if (before != before || fresh != fresh) scale = __uint_as_float(0x7fc00000u);
        else if (before < fresh) { ratio = before / fresh; grown = true; }
        else scale = before;
    }
    if (tid == 0) *sp = scale;
    const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
    // round-half-even(v * inv) within +-127 as the low byte of 1.5 * 2^23 + it (a block without inv has codes of 0: the image as it is; one
    // with it holds finite values only)
    auto code = [&](float v) -> unsigned { return __float_as_uint(__builtin_amdgcn_fmed3f(v * inv, -127.0f, 127.0f) + 12582912.0f); };
#pragma unroll
    for (int j = 0; j < ROUNDS; j++) {
        if (j * 256 >= n || inv == 0.0f) continue;
        const int t = tok[j];
        float v[2 * W];
        g[j].ordered(v);
#pragma unroll
        for (int h = 0; h < 2; h++) {   // W channels in memory order from d on (VEC: of one 16)
            const int d = h == 0 ? g[j].da : VEC ? g[j].second() : g[j].db;
            unsigned b[W];
#pragma unroll
            for (int w = 0; w < W; w++) b[w] = code(v[h * W + w]);
            if (!keys) {
                int8_t* to = &image[kv_v_byte(t, d)];   // (of one 16: 16 bytes from channel to channel)
#pragma unroll
                for (int w = 0; w < W; w++) to[w * 16] = (int8_t)b[w];
            } else if constexpr (VEC) {
                unsigned* to = (unsigned*)&image[kv_k_byte(a.dim64, t, d)];
#pragma unroll
                for (int w = 0; w < W; w += 4)
                    to[w / 4] = __builtin_amdgcn_perm(b[w + 1], b[w], 0x0c0c0400u) | __builtin_amdgcn_perm(b[w + 3], b[w + 2], 0x04000c0cu);
            } else {
                image[kv_k_byte(a.dim64, t, d)] = (int8_t)b[0];
            }
        }
    }
    __syncthreads();
    auto again = [&](unsigned b) -> unsigned { return (unsigned)(int)rintf((float)(int8_t)b * ratio) & 255u; };
    const int w0 = grown ? 0 : t0;   // tokens whose codes change
    if (keys) {
        int8_t* dst = a.k + bi * (SMX_KV_BLOCK * (int64_t)a.dim64);
        // units of 16 channels of a token, in memory order: (token / 16, d / 64, d / 16 % 4, token % 16); all 32 tokens are gone through
        const int units = 2 * a.dim64;
        for (int u = tid; u < units; u += 256) {
            const int c = u >> 6, dc = a.dim64 >> 6, tt = c / dc;
            const int t = tt * 16 + (u & 15), d0 = (c - tt * dc) * 64 + ((u >> 4) & 3) * 16;
            if (t < w0 || t >= t1 || d0 >= a.dim) continue;
            uint4* p = (uint4*)(dst + (int64_t)u * 16);
            if (t >= t0) {
                *p = ((const uint4*)image)[u];
                continue;
            }
            const uint4 old = *p;
            const unsigned ow[4] = {old.x, old.y, old.z, old.w};
            unsigned w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int j = 0; j < 16; j++) w[j >> 2] |= again(ow[j >> 2] >> (8 * (j & 3))) << (8 * (j & 3));
            *p = make_uint4(w[0], w[1], w[2], w[3]);
        }
        return;
    }
    int8_t* dst = a.v + bi * (SMX_KV_BLOCK * (int64_t)a.dim64);
    if (t0 == 0 && t1 == SMX_KV_BLOCK) {
        // units of 8 tokens of channels d and d + 16, in memory order: (d / 32, token / 4 % 4, d % 16)
        for (int u = tid; u < 2 * a.dim64; u += 256)
            if ((u >> 6) * 32 + (u & 15) < a.dim) *(uint4*)(dst + (int64_t)u * 16) = ((const uint4*)image)[u];
        return;
    }
    const int g0 = w0 >> 2, quads = ((t1 + 3) >> 2) - g0;   // groups of 4 tokens of a channel
    for (int it = tid; it < quads * a.dim; it += 256) {
        const int q = it / a.dim, t = (g0 + q) * 4, d = it - q * a.dim, at = kv_v_byte(t, d);
        int8_t* p = dst + at;
        if (!grown && (t < t0 || t + 4 > t1)) {
            for (int j = max(t0 - t, 0); j < min(t1 - t, 4); j++) p[j] = image[at + j];
            continue;
        }
        unsigned w = *(const unsigned*)&image[at];   // (0 for tokens outside [t0, t1))
        if (t < t0) {
            const unsigned old = *(const unsigned*)p;
            for (int j = 0; j < min(t0 - t, 4); j++) w |= again(old >> (8 * j)) << (8 * j);
        }
        *(unsigned*)p = w;
    }
}

// Workgroup (x, head, keys | values): the stored values of one block's rows.  A thread takes 4 tokens of 4 channels, four words of
// the layout (a token's channels of keys, a channel's tokens of values), so that a wave's stores are whole pieces of rows: the
// values are four times the bytes of the codes, and 16-byte stores to 64 rows at once took 26 us for 34 MB, these 9.5.
template <bool VEC>
__global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs a, float* __restrict__ k, float* __restrict__ v) {
    const bool keys = blockIdx.z == 0;
    float* out = keys ? k : v;
    if (!out) return;
    const BlockRows br = block_rows(a, blockIdx.x);
    const int t0 = br.t0, t1 = br.t1, head = blockIdx.y;
    if (t1 <= t0) return;
    const int64_t bi = kv_block(a, br.s, head, br.blk);
    const int8_t* src = (keys ? a.k : a.v) + bi * (SMX_KV_BLOCK * (int64_t)a.dim64);
    const float scale = (keys ? a.ks : a.vs)[bi];
    const int64_t ld = (int64_t)a.kv_heads * a.dim;
    float* base = out + (int64_t)br.row * ld + (int64_t)head * a.dim;   // of the block's token 0
    const int quads = (a.dim + 3) >> 2;
    for (int it = threadIdx.x; it < 8 * quads; it += 256) {
        const int tq = it / quads, t = tq * 4, d = (it - tq * quads) * 4;
        if (t >= t1 || t + 4 <= t0) continue;
        unsigned w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = *(const unsigned*)(src + (keys ? kv_k_byte(a.dim64, t + j, d) : kv_v_byte(t, d + j)));
#pragma unroll
        for (int j = 0; j < 4; j++) {   // token t + j
            if (t + j < t0 || t + j >= t1) continue;
            float f[4];
#pragma unroll
            for (int i = 0; i < 4; i++) f[i] = (float)(int8_t)(keys ? w[j] >> (8 * i) : w[i] >> (8 * j)) * scale;
            float* to = base + (t + j) * ld + d;
            if (VEC) {
                *(float4*)to = make_float4(f[0], f[1], f[2], f[3]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (d + i < a.dim) to[i] = f[i];
            }
        }
    }
}

__global__ __launch_bounds__(256) void rope_table_kernel(double log_base, int half, int64_t n, float2* __restrict__ out) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const double angle = (double)(i / half) * exp(-log_base * (double)(i % half) / (double)half);
    double sn, cs;
    sincos(angle, &sn, &cs);
    out[i] = make_float2((float)cs, (float)sn);
}

}  // namespace
}  // namespace smx

using namespace smx;

extern "C" {

int smx_rope_table_dev(smx_ctx* c, float base, size_t rot_dim, size_t n_pos, float* table_dev) {
    if (!c) return SMX_ERR_ARG;
    if (!table_dev) return fail(c, SMX_ERR_ARG, "rope_table_dev: null argument");
    if (!(base > 0) || rot_dim == 0 || rot_dim % 2 || rot_dim > SMX_KV_MAX_HEAD_DIM || n_pos == 0 || n_pos > (size_t(1) << 30))
        return fail(c, SMX_ERR_ARG, "rope_table_dev: base %g, %zu channels (even, up to %d), %zu positions (1..2^30)", (double)base, rot_dim,
                    SMX_KV_MAX_HEAD_DIM, n_pos);
    const int64_t n = (int64_t)n_pos * (int64_t)(rot_dim / 2);
    hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, c->stream, log((double)base), (int)(rot_dim / 2), n,
                       (float2*)table_dev);
    SMX_HIP(c, hipGetLastError());
    return SMX_OK;
}

int smx_kv_sizes(size_t pages, size_t page_tokens, size_t kv_heads, size_t head_dim, size_t* code_bytes, size_t* scales) {
    if (!code_bytes || !scales) return SMX_ERR_ARG;
    if (pages == 0 || page_tokens == 0 || page_tokens % SMX_KV_BLOCK || page_tokens > (size_t(1) << 20) || kv_heads == 0 || kv_heads > 65535 ||
        head_dim == 0 || head_dim % 2 || head_dim > SMX_KV_MAX_HEAD_DIM || pages > (size_t(1) << 31))
        return SMX_ERR_ARG;
    const size_t blocks = pages * kv_heads * (page_tokens / SMX_KV_BLOCK);   // < 2^62
    if (blocks > size_t(1) << 48) return SMX_ERR_ARG;                        // (and their bytes would pass 64 bits)
    *code_bytes = blocks * SMX_KV_BLOCK * ((head_dim + 63) & ~size_t(63));
    *scales = blocks;
    return SMX_OK;
}

int smx_kv_append_dev(smx_ctx* c, const smx_kv_cache* cache, const smx_kv_batch* batch, int type, const void* k, size_t ldk, const void* v, size_t ldv,
                      const smx_rope* rope, const void* q, size_t ldq, size_t q_heads, void* q_out, size_t ldqo) {
    if (!c) return SMX_ERR_ARG;
    AppendArgs A{};
    int rc;
    if ((rc = kv_args(c, "kv_append_dev", cache, batch, &A.kv)) != SMX_OK) return rc;
    if (type != SMX_TYPE_F32 && type != SMX_TYPE_BF16) return fail(c, SMX_ERR_ARG, "kv_append_dev: element type %d", type);
    if (batch->nseq == 0 || batch->rows == 0 || batch->max_len == 0) return SMX_OK;
    if (!k || !v) return fail(c, SMX_ERR_ARG, "kv_append_dev: null keys or values");
    const size_t kvw = cache->kv_heads * cache->head_dim, qw = q_heads * cache->head_dim;
    if (ldk < kvw || ldv < kvw) return fail(c, SMX_ERR_ARG, "kv_append_dev: rows of %zu elements, ldk %zu, ldv %zu", kvw, ldk, ldv);
    if (rope && (!rope->table || rope->n_pos == 0 || rope->n_pos > (size_t(1) << 30) || rope->rot_dim == 0 || rope->rot_dim % 2 || rope->rot_dim > cache->head_dim))
        return fail(c, SMX_ERR_ARG, "kv_append_dev: rotation of %zu channels (even, up to %zu) with %zu positions", rope->rot_dim, cache->head_dim, rope->n_pos);
    if (q && (!q_out || q_heads == 0 || q_heads > 65535 || ldq < qw || ldqo < qw))
        return fail(c, SMX_ERR_ARG, "kv_append_dev: queries of %zu elements a row, ldq %zu, ldqo %zu", qw, ldq, ldqo);
    A.k = k; A.v = v; A.ldk = (int64_t)ldk; A.ldv = (int64_t)ldv;
    if (rope) {
        A.rope = (const float2*)rope->table;
        A.n_pos = (int)rope->n_pos;
        A.rot = (int)rope->rot_dim;
    }
    A.touched = touched_blocks(batch);
    const bool bf = type == SMX_TYPE_BF16, pairs = rope && rope->interleaved;
    const size_t W = bf ? 8 : 4, half = rope ? rope->rot_dim / 2 : 0;
    bool vec = cache->head_dim % (2 * W) == 0 && half % W == 0 && ldk % W == 0 && ldv % W == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    if (q) vec = vec && ldq % W == 0 && ldqo % W == 0 && (((uintptr_t)q | (uintptr_t)q_out) & 15) == 0;
    size_t extra = 0;
    if (q) {
        A.q = q; A.qo = q_out; A.ldq = (int64_t)ldq; A.ldqo = (int64_t)ldqo; A.q_heads = (int)q_heads;
        const size_t items = batch->rows * q_heads * (cache->head_dim / (vec ? 2 * W : 2)), per = (size_t)kQueryItems * cache->kv_heads * 2;
        extra = (items + per - 1) / per;
    }
    if (batch->rows * q_heads >= (size_t(1) << 31) || A.touched + extra > INT_MAX)
        return fail(c, SMX_ERR_LIMIT, "kv_append_dev: %zu rows of %zu query heads", batch->rows, q_heads);
    const dim3 grid((unsigned)(A.touched + extra), (unsigned)cache->kv_heads, 2);
    const size_t lds = SMX_KV_BLOCK * (size_t)A.kv.dim64;
    ProfScope ps(c, "kv_append");
    auto pick = [&](auto bf16, auto two) {
        return vec ? kv_append_kernel<decltype(bf16)::value, decltype(two)::value, true> : kv_append_kernel<decltype(bf16)::value, decltype(two)::value, false>;
    };
    std::true_type yes;
    std::false_type no;
    auto kern = bf ? (pairs ? pick(yes, yes) : pick(yes, no)) : (pairs ? pick(no, yes) : pick(no, no));
    hipLaunchKernelGGL(kern, grid, dim3(256), lds, c->stream, A);
    SMX_HIP(c, hipGetLastError());
    return SMX_OK;
}

int smx_kv_read_dev(smx_ctx* c, const smx_kv_cache* cache, const smx_kv_batch* batch, float* k, float* v) {
    if (!c) return SMX_ERR_ARG;
    KvArgs a{};
    int rc;
    if ((rc = kv_args(c, "kv_read_dev", cache, batch, &a)) != SMX_OK) return rc;
    if (batch->nseq == 0 || batch->rows == 0) return SMX_OK;
    if (!k && !v) return fail(c, SMX_ERR_ARG, "kv_read_dev: nothing to read into");
    ProfScope ps(c, "kv_read");
    const bool vec = cache->head_dim % 4 == 0 && (((uintptr_t)k | (uintptr_t)v) & 15) == 0;
    hipLaunchKernelGGL(vec ? kv_read_kernel<true> : kv_read_kernel<false>, dim3((unsigned)touched_blocks(batch), (unsigned)cache->kv_heads, 2), dim3(256), 0,
                       c->stream, a, k, v);
    SMX_HIP(c, hipGetLastError());
    return SMX_OK;
}

}  // extern "C"

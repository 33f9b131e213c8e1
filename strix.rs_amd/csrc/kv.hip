// The paged 8-bit key/value cache: a step's keys and values appended with their position rotation, stored values read back.
#include <algorithm>
#include <climits>

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
    if (b->max_rows > b->rows) return fail(c, SMX_ERR_ARG, "%s: max_rows %zu of %zu rows", who, b->max_rows, b->rows);
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

constexpr int kQueryItems = 1024;   // channel pairs per workgroup of the query rotation

// Pair i of a head's dim / 2 channel pairs, rotated: channels *da, *db of the row.  Pairs behind the rotated ones are
// neighbouring channels that pass through.
template <bool BF16, bool PAIRS>
__device__ __forceinline__ float2 rotated_pair(const AppendArgs& A, const void* x, int64_t at, int pos, int i, int* da, int* db) {
#pragma clang fp contract(off)
    const int half = A.rot >> 1;
    const bool turn = i < half;
    *da = turn ? (PAIRS ? 2 * i : i) : 2 * i;
    *db = turn ? (PAIRS ? 2 * i + 1 : i + half) : 2 * i + 1;
    const float a = load_elem<BF16>(x, at + *da), b = load_elem<BF16>(x, at + *db);
    if (!turn) return make_float2(a, b);
    const float2 cs = A.rope[(int64_t)min(pos, A.n_pos - 1) * half + i];
    return make_float2(a * cs.x - b * cs.y, a * cs.y + b * cs.x);
}

// The largest |value| as its bits: NaN and infinity order above every finite value.
__device__ __forceinline__ unsigned abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Workgroup (x, head, keys | values): x < touched is one block of 32 tokens that the step writes into, the others rotate
// kQueryItems channel pairs of the queries each (head and z choose among those).
//
// A block is one workgroup's alone, so its scale, the rounding of earlier codes under a scale that grew and the new codes need no
// atomics: the block's new values go through LDS as fp32, their largest gives the scale, and whole groups of bytes are written
// (4 tokens of a channel for values, 16 channels of a token for keys).
template <bool BF16, bool PAIRS>
__global__ __launch_bounds__(256) void kv_append_kernel(const AppendArgs A) {
#pragma clang fp contract(off)
    extern __shared__ float vals[];   // [32][dim + 1]
    __shared__ unsigned red[4];
    const KvArgs& a = A.kv;
    const int tid = threadIdx.x, half = a.dim >> 1;
    if ((int)blockIdx.x >= A.touched) {
        const int64_t items = (int64_t)a.rows * A.q_heads * half;
        const int64_t group = ((int64_t)(blockIdx.x - A.touched) * gridDim.y + blockIdx.y) * gridDim.z + blockIdx.z;
        for (int64_t it = group * kQueryItems + tid; it < min((group + 1) * kQueryItems, items); it += 256) {
            const int64_t rh = it / half;
            const int row = (int)(rh / A.q_heads), h = (int)(rh - (int64_t)row * A.q_heads), i = (int)(it - rh * half);
            int s = row;
            if (a.row0) {   // the last sequence that starts at or before the row
                int lo = 0, hi = a.nseq - 1;
                while (lo < hi) {
                    const int mid = (lo + hi + 1) >> 1;
                    if (a.row0[mid] <= row) lo = mid; else hi = mid - 1;
                }
                s = lo;
            }
            const KvSeq q = kv_seq(a, s);
            const int pos = max(q.len - q.n + row - q.row, 0);
            int da, db;
            const float2 r = rotated_pair<BF16, PAIRS>(A, A.q, (int64_t)row * A.ldq + (int64_t)h * a.dim, pos, i, &da, &db);
            const int64_t at = (int64_t)row * A.ldqo + (int64_t)h * a.dim;
            store_elem<BF16>(A.qo, at + da, r.x);
            store_elem<BF16>(A.qo, at + db, r.y);
        }
        return;
    }
    // which sequence, and which of the blocks that it touches
    int s = blockIdx.x, nth = 0;
    if (a.row0) {
        int left = blockIdx.x;
        for (s = 0; s < a.nseq; s++) {
            const KvSeq q = kv_seq(a, s);
            const int first = max(q.len - q.n, 0);
            const int blocks = q.len > first ? (q.len - 1) / SMX_KV_BLOCK - first / SMX_KV_BLOCK + 1 : 0;
            if (left < blocks) break;
            left -= blocks;
        }
        if (s == a.nseq) return;
        nth = left;
    }
    const KvSeq q = kv_seq(a, s);
    const int start = q.len - q.n;                 // may be negative: rows in front of position 0 are left out
    const int blk = max(start, 0) / SMX_KV_BLOCK + nth;
    const int t0 = max(max(start, 0) - blk * SMX_KV_BLOCK, 0), t1 = min(q.len - blk * SMX_KV_BLOCK, SMX_KV_BLOCK);
    if (t1 <= t0) return;
    const int head = blockIdx.y;
    const bool keys = blockIdx.z == 0;
    const int64_t bi = kv_block(a, s, head, blk);
    const int row = q.row + blk * SMX_KV_BLOCK - start;   // of the block's token 0
    const int pitch = a.dim + 1;
    unsigned most = 0;
    const int items = (t1 - t0) * half;
    for (int it = tid; it < items; it += 256) {
        const int t = t0 + it / half, i = it % half;
        float2 r;
        int da, db;
        if (keys && A.rope) {
            r = rotated_pair<BF16, PAIRS>(A, A.k, (int64_t)(row + t) * A.ldk + (int64_t)head * a.dim, blk * SMX_KV_BLOCK + t, i, &da, &db);
        } else {
            const int64_t at = (keys ? (int64_t)(row + t) * A.ldk : (int64_t)(row + t) * A.ldv) + (int64_t)head * a.dim;
            da = 2 * i; db = 2 * i + 1;
            r = make_float2(load_elem<BF16>(keys ? A.k : A.v, at + da), load_elem<BF16>(keys ? A.k : A.v, at + db));
        }
        vals[t * pitch + da] = r.x;
        vals[t * pitch + db] = r.y;
        most = max(most, max(abs_bits(r.x), abs_bits(r.y)));
    }
    for (int o = 1; o < 64; o <<= 1) most = max(most, (unsigned)__shfl_xor((int)most, o));
    if ((tid & 63) == 0) red[tid >> 6] = most;
    __syncthreads();
    most = max(max(red[0], red[1]), max(red[2], red[3]));
    const float top = __uint_as_float(most);
    const float fresh = most >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : top >= 0x1p-96f ? top / 127.0f : 0.0f;
    float* sp = (keys ? a.ks : a.vs) + bi;
    float scale = fresh, ratio = 1.0f;
    bool grown = false;
    if (t0 > 0) {
        const float before = *sp;
        if (before != before || fresh != fresh) scale = __uint_as_float(0x7fc00000u);
        else if (before < fresh) { ratio = before / fresh; grown = true; }
        else scale = before;
    }
    __syncthreads();   // every thread has read the old scale
    if (tid == 0) *sp = scale;
    const float inv = scale > 0.0f ? 1.0f / scale : 0.0f;
    const int w0 = grown ? 0 : t0;   // tokens whose codes change
    auto code = [&](int t, int d) -> int {
        const float y = rintf(vals[t * pitch + d] * inv);
        return y == y ? (int)fminf(fmaxf(y, -127.0f), 127.0f) & 255 : 0;
    };
    auto again = [&](unsigned b) -> int { return (int)rintf((float)(int8_t)b * ratio) & 255; };
    if (keys) {
        int8_t* dst = a.k + bi * (SMX_KV_BLOCK * (int64_t)a.dim64);
        const int quads = (a.dim + 3) >> 2;
        for (int it = tid; it < (t1 - w0) * quads; it += 256) {
            const int t = w0 + it / quads, d = it % quads * 4;
            unsigned* p = (unsigned*)(dst + kv_k_byte(a.dim64, t, d));
            unsigned w = 0;
            if (t < t0) {
                const unsigned old = *p;
                for (int j = 0; j < 4; j++) w |= (unsigned)again(old >> (8 * j)) << (8 * j);
            } else {
                for (int j = 0; j < 4; j++)
                    if (d + j < a.dim) w |= (unsigned)code(t, d + j) << (8 * j);
            }
            *p = w;
        }
    } else {
        int8_t* dst = a.v + bi * (SMX_KV_BLOCK * (int64_t)a.dim64);
        const int g0 = w0 >> 2, groups = ((t1 + 3) >> 2) - g0;   // groups of 4 tokens
        for (int it = tid; it < groups * a.dim; it += 256) {
            const int t = (g0 + it / a.dim) * 4, d = it % a.dim;
            unsigned* p = (unsigned*)(dst + kv_v_byte(t, d));
            unsigned w = 0;
            const unsigned old = t < t0 ? *p : 0u;
            for (int j = 0; j < 4; j++) {
                unsigned b = 0;
                if (t + j < t0) b = grown ? (unsigned)again(old >> (8 * j)) : (old >> (8 * j)) & 255u;
                else if (t + j < t1) b = (unsigned)code(t + j, d);
                w |= b << (8 * j);
            }
            *p = w;
        }
    }
}

// Workgroup (row, key/value heads): the stored values of one row.
__global__ __launch_bounds__(256) void kv_read_kernel(const KvArgs a, float* __restrict__ k, float* __restrict__ v) {
    const int row = blockIdx.x;
    int s = row;
    if (a.row0) {
        int lo = 0, hi = a.nseq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (a.row0[mid] <= row) lo = mid; else hi = mid - 1;
        }
        s = lo;
    }
    const KvSeq q = kv_seq(a, s);
    const int pos = q.len - q.n + row - q.row;
    for (int it = threadIdx.x; it < a.kv_heads * a.dim; it += 256) {
        const int head = it / a.dim, d = it % a.dim;
        const int64_t at = (int64_t)row * a.kv_heads * a.dim + it;
        float kval = 0.f, vval = 0.f;
        if (pos >= 0 && pos < q.len) {
            const int64_t bi = kv_block(a, s, head, pos / SMX_KV_BLOCK);
            const int64_t base = bi * (SMX_KV_BLOCK * (int64_t)a.dim64);
            const int t = pos % SMX_KV_BLOCK;
            if (k) kval = (float)a.k[base + kv_k_byte(a.dim64, t, d)] * a.ks[bi];
            if (v) vval = (float)a.v[base + kv_v_byte(t, d)] * a.vs[bi];
        }
        if (k) k[at] = kval;
        if (v) v[at] = vval;
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
    const size_t blocks = pages * kv_heads * (page_tokens / SMX_KV_BLOCK);
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
    // a sequence of n rows touches at most (n + 61) / 32 blocks
    A.touched = batch->row0 ? (int)((batch->rows + 61 * batch->nseq) / SMX_KV_BLOCK) : (int)batch->nseq;
    size_t extra = 0;
    if (q) {
        A.q = q; A.qo = q_out; A.ldq = (int64_t)ldq; A.ldqo = (int64_t)ldqo; A.q_heads = (int)q_heads;
        const size_t items = batch->rows * q_heads * (cache->head_dim / 2), per = (size_t)kQueryItems * cache->kv_heads * 2;
        extra = (items + per - 1) / per;
    }
    const dim3 grid((unsigned)(A.touched + extra), (unsigned)cache->kv_heads, 2);
    const size_t lds = SMX_KV_BLOCK * (cache->head_dim + 1) * 4;
    ProfScope ps(c, "kv_append");
    const bool bf = type == SMX_TYPE_BF16, pairs = rope && rope->interleaved;
    auto kern = bf ? (pairs ? kv_append_kernel<true, true> : kv_append_kernel<true, false>) : (pairs ? kv_append_kernel<false, true> : kv_append_kernel<false, false>);
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
    hipLaunchKernelGGL(kv_read_kernel, dim3((unsigned)batch->rows), dim3(256), 0, c->stream, a, k, v);
    SMX_HIP(c, hipGetLastError());
    return SMX_OK;
}

}  // extern "C"

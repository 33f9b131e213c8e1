// Sampling: one token for each row of logits by temperature, top-k, top-p and min-p from a given uniform number.
//
// A token's weight is a whole number, floor(exp((x - max) / T) * 2^40), so every sum below is exact and has one value in any
// order: the cut of top_p and the pick are the same however a row is split over workgroups.  (With fp32 sums a pick would change
// with the split in about one row of 50 of an unfiltered 262144-token row.)
//
// Rows are ordered by (logit descending, index ascending), and nothing sorts a row.  Four launches over parts of rows:
//   1  the largest logit
//   2  rows with top_k or top_p: a histogram over kBins steps of distance from it, of tokens (top_k) or of weight (top_p)
//   3  the bin that the cut falls into; what lies above it is totalled per chunk of kChunk tokens (top_k: listed), the bin's own
//      tokens are listed
//   4  one workgroup for each row sorts the list (up to kList tokens), which places the cut at one token, finds the chunk that
//      the pick falls into from the totals and the pick in the chunk
// A row is read three times (without top_k and top_p: twice), every other launch from its end, where the one in front has left
// the caches.  A list that does not fit (thousands of equal logits at the cut, or a cut more than kReach below the largest logit) is
// found by bisection over the logits instead.
#include <algorithm>
#include <climits>
#include <cmath>

#include "smx_internal.h"

namespace smx {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;   // of the row's own workgroup (launch 4)
constexpr int kChunk = 1024;                             // tokens whose kept weight is totalled together
constexpr int kMaxVocab = SMX_SAMPLE_MAX_VOCAB, kMaxChunks = kMaxVocab / kChunk;
constexpr int kBins = 2048;
constexpr float kReach = 28.0f;                          // exp(-28) < 2^-40: beyond it there is no weight
constexpr int kList = 4096;

struct SampleArgs {
    const float* logits;
    int64_t ld;
    int rows, vocab, chunks, parts, part_chunks;   // part_chunks: chunks per part of a row
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* ids;
    float* prob;
    // workspace
    uint2* best;                    // [rows][parts] key and index of the part's largest logit
    unsigned long long* hist;       // [rows][kBins] weight; top_k rows: tokens
    unsigned long long* totals;     // [rows][chunks] kept weight above the cut's bin
    unsigned long long* list;       // [rows][kList] ~key : index
    unsigned* listed;               // [rows]
};

// Order-preserving key of a logit: NaN and -inf are 0, below every other; -0 is +0.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    const unsigned k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float of_key(unsigned k) { return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// exp((x - max) / T) of a candidate (x > -inf), 1 for the largest (so that a +inf maximum has a share)
__device__ __forceinline__ float share(float x, float mx, float T) {
#pragma clang fp contract(off)
    return x == mx ? 1.0f : expf((x - mx) / T);
}
__device__ __forceinline__ unsigned long long weight(float e) { return (unsigned long long)(e * 0x1p40f); }
// Bin of a candidate: steps of distance below the largest logit.  Rounding is monotone in x, so a smaller bin means a larger logit.
__device__ __forceinline__ int bin_of(float x, float mx, float T) {
#pragma clang fp contract(off)
    const float y = x == mx ? 0.0f : (mx - x) / T;
    return (int)fminf(y * ((float)kBins / kReach), (float)(kBins - 1));
}

// What a row asks for, and its largest logit.
enum Mode { kNone, kGreedy, kFree, kTopK, kTopP };   // kNone: no candidate at all
struct Ask {
    Mode mode;
    unsigned best_at;
    float mx, T, top_p, min_p;
    float bin_T;      // divides distances in bin_of: T, or 1 where tokens are counted
    int top_k;
};
__device__ __forceinline__ uint2 better(uint2 a, uint2 b) { return b.x > a.x || (b.x == a.x && b.y < a.y) ? b : a; }
__device__ __forceinline__ uint2 wave_best(uint2 v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v = better(v, make_uint2(__shfl_xor(v.x, o), __shfl_xor(v.y, o)));
    return v;
}
__device__ __forceinline__ Ask ask_of(const SampleArgs& A, int row) {
    // every wave reads the parts' candidates for itself: no barrier
    uint2 b = make_uint2(0u, 0xffffffffu);
    for (int i = threadIdx.x & 63; i < A.parts; i += 64) b = better(b, A.best[(int64_t)row * A.parts + i]);
    b = wave_best(b);
    Ask q;
    q.best_at = b.y;
    q.mx = of_key(b.x);
    q.T = A.temperature ? A.temperature[row] : 1.0f;
    q.top_k = A.top_k ? A.top_k[row] : 0;
    q.top_p = A.top_p ? A.top_p[row] : 1.0f;
    q.min_p = A.min_p ? fminf(A.min_p[row], 1.0f) : 0.0f;
    const bool k = q.top_k > 0 && q.top_k < A.vocab;
    q.mode = b.x == 0 ? kNone : !(q.T > 0.0f) || q.top_k == 1 || q.top_p <= 0.0f ? kGreedy : k ? kTopK : q.top_p < 1.0f ? kTopP : kFree;
    q.bin_T = q.mode == kTopK ? 1.0f : q.T;
    return q;
}

// The chunk's 16 tokens of each lane: token chunk * kChunk + 256 j + 4 lane + i (-inf past the row).
template <bool VEC>
__device__ __forceinline__ void load_chunk(const float* __restrict__ x, int vocab, int chunk, float (&v)[16]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = chunk * kChunk + 256 * j + 4 * lane;
        if (VEC && i + 4 <= vocab) {
            const float4 f = *(const float4*)(x + i);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        } else {
#pragma unroll
            for (int t = 0; t < 4; t++) v[4 * j + t] = i + t < vocab ? x[i + t] : -INFINITY;
        }
    }
}
__device__ __forceinline__ int token_of(int chunk, int n) { return chunk * kChunk + 256 * (n >> 2) + 4 * (int)(threadIdx.x & 63) + (n & 3); }

// Launch 1.  Workgroup (part, row); also clears what launches 2 and 3 add to.
template <bool VEC>
__global__ __launch_bounds__(1024) void sample_best_kernel(const SampleArgs A) {
    __shared__ uint2 red[16];
    const int row = blockIdx.y, part = blockIdx.x, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const float* x = A.logits + (int64_t)row * A.ld;
    for (int i = part * blockDim.x + threadIdx.x; i < kBins; i += A.parts * blockDim.x) A.hist[(int64_t)row * kBins + i] = 0;
    if (part == 0 && threadIdx.x == 0) A.listed[row] = 0;
    uint2 b = make_uint2(0u, 0xffffffffu);
    const int c1 = min((part + 1) * A.part_chunks, A.chunks);
    for (int c = part * A.part_chunks + wave; c < c1; c += waves) {
        float v[16];
        load_chunk<VEC>(x, A.vocab, c, v);
#pragma unroll
        for (int n = 0; n < 16; n++) {   // (ascending tokens of a lane: the first of equals stays)
            const unsigned k = key_of(v[n]);
            if (k > b.x) b = make_uint2(k, (unsigned)token_of(c, n));
        }
    }
    b = wave_best(b);
    if ((threadIdx.x & 63) == 0) red[wave] = b;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < waves; w++) b = better(b, red[w]);
        A.best[(int64_t)row * A.parts + part] = b;
    }
}

// Launch 2.  Workgroup (part, row), from the last to the first.
template <bool VEC>
__global__ __launch_bounds__(1024) void sample_hist_kernel(const SampleArgs A) {
    __shared__ unsigned long long hist[kBins];
    const int row = A.rows - 1 - blockIdx.y, part = A.parts - 1 - blockIdx.x, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const Ask q = ask_of(A, row);
    if (q.mode != kTopK && q.mode != kTopP) return;
    const float* x = A.logits + (int64_t)row * A.ld;
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) hist[i] = 0;
    __syncthreads();
    const int c0 = part * A.part_chunks, c1 = min(c0 + A.part_chunks, A.chunks);
    for (int c = c1 - 1 - wave; c >= c0; c -= waves) {
        float v[16];
        load_chunk<VEC>(x, A.vocab, c, v);
#pragma unroll
        for (int n = 0; n < 16; n++) {
            if (!(v[n] > -INFINITY)) continue;
            const int b = bin_of(v[n], q.mx, q.bin_T);
            const unsigned long long w = q.mode == kTopK ? 1ull : weight(share(v[n], q.mx, q.T));
            if (w) atomicAdd(&hist[b], w);
        }
    }
    __syncthreads();
    unsigned long long* out = A.hist + (int64_t)row * kBins;
    for (int i = threadIdx.x; i < kBins; i += blockDim.x) {
        const unsigned long long w = hist[i];
        if (w) atomicAdd(&out[i], w);
    }
}

__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v) {   // inclusive
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned long long r = __shfl_up(v, o);
        if (lane >= o) v += r;
    }
    return v;
}

// The cut's bin: the first whose running total reaches `limit` (top_k tokens, or floor(top_p * all weight)), and what lies above it.
struct Cut {
    int bin;
    unsigned long long above, limit;
};
// Every thread of the workgroup (256..1024); red: 17 words of LDS.
__device__ __forceinline__ Cut find_cut(const SampleArgs& A, const Ask& q, int row, unsigned long long* red) {
    const unsigned long long* h = A.hist + (int64_t)row * kBins;
    const int per = kBins / blockDim.x, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;   // bins of a thread: up to 8
    unsigned long long mine[8], sum = 0;
    for (int i = 0; i < per; i++) {
        mine[i] = h[threadIdx.x * per + i];
        sum += mine[i];
    }
    unsigned long long run = wave_scan(sum);
    if ((threadIdx.x & 63) == 63) red[wave] = run;
    __syncthreads();
    unsigned long long total = 0, front = 0;
    for (int w = 0; w < waves; w++) {
        if (w < wave) front += red[w];
        total += red[w];
    }
    run += front - sum;   // in front of this thread's bins
    Cut c;
    c.limit = q.mode == kTopK ? (unsigned long long)q.top_k : (unsigned long long)((double)q.top_p * (double)total);
    c.bin = kBins;        // fewer candidates than top_k: every one
    c.above = 0;
    __syncthreads();
    if (threadIdx.x == 0) { red[0] = kBins; red[1] = total; }
    __syncthreads();
    // the running total first reaches the limit in one thread's bins (a limit of 0: in the first bin)
    if (run < c.limit && run + sum >= c.limit) {
        for (int i = 0; i < per; i++) {
            if (run + mine[i] >= c.limit) {
                red[0] = threadIdx.x * per + i;
                red[1] = run;
                break;
            }
            run += mine[i];
        }
    }
    if (c.limit == 0 && threadIdx.x == 0) { red[0] = 0; red[1] = 0; }
    __syncthreads();
    c.bin = (int)red[0];
    c.above = red[1];
    return c;
}

// Launch 3.  Workgroup (part, row).
template <bool VEC>
__global__ __launch_bounds__(1024) void sample_gather_kernel(const SampleArgs A) {
    __shared__ unsigned long long red[17];
    const int row = blockIdx.y, part = blockIdx.x, wave = threadIdx.x >> 6, waves = blockDim.x >> 6, lane = threadIdx.x & 63;
    const Ask q = ask_of(A, row);
    if (q.mode <= kGreedy) return;
    int cut = -1;
    if (q.mode != kFree) cut = find_cut(A, q, row, red).bin;
    const float* x = A.logits + (int64_t)row * A.ld;
    const int c1 = min((part + 1) * A.part_chunks, A.chunks);
    for (int c = part * A.part_chunks + wave; c < c1; c += waves) {
        float v[16];
        load_chunk<VEC>(x, A.vocab, c, v);
        unsigned long long total = 0;
#pragma unroll
        for (int n = 0; n < 16; n++) {
            const bool live = v[n] > -INFINITY;
            const int b = q.mode != kFree ? bin_of(v[n], q.mx, q.bin_T) : -1;
            if (live && q.mode != kTopK && (q.mode == kFree || b < cut)) {
                const float e = share(v[n], q.mx, q.T);
                if (e >= q.min_p) total += weight(e);
            }
            const bool put = live && (q.mode == kTopK ? b <= cut : q.mode == kTopP && b == cut);
            const unsigned long long who = __ballot(put);
            if (who) {
                unsigned at = 0;
                if (lane == 0) at = atomicAdd(&A.listed[row], (unsigned)__popcll(who));
                at = __builtin_amdgcn_readfirstlane(at) + __popcll(who & ((1ull << lane) - 1));
                if (put && at < (unsigned)kList)
                    A.list[(int64_t)row * kList + at] = (unsigned long long)~key_of(v[n]) << 32 | (unsigned)token_of(c, n);
            }
        }
        if (q.mode != kTopK) {
            total = wave_sum(total);
            if (lane == 0) A.totals[(int64_t)row * A.chunks + c] = total;
        }
    }
}

struct Reduce {
    unsigned long long a[kWaves];
};
__device__ __forceinline__ unsigned long long block_sum(Reduce& r, unsigned long long v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.a[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long t = 0;
    for (int w = 0; w < kWaves; w++) t += r.a[w];
    return t;
}
// inclusive, over the workgroup's threads
__device__ __forceinline__ unsigned long long block_scan(Reduce& r, unsigned long long v) {
    v = wave_scan(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 63) r.a[threadIdx.x >> 6] = v;
    __syncthreads();
    for (int w = 0; w < (int)(threadIdx.x >> 6); w++) v += r.a[w];
    return v;
}

// Sorts a[0, n) upwards; n a power of two, up to kList.
__device__ void sort_list(unsigned long long* a, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            for (int t = threadIdx.x; t < n / 2; t += kThreads) {
                const int i = ((t & ~(j - 1)) << 1) | (t & (j - 1));
                const unsigned long long p = a[i], r = a[i | j];
                const bool up = (i & k) == 0;
                if ((p > r) == up) { a[i] = r; a[i | j] = p; }
            }
        }
    __syncthreads();
}
__device__ __forceinline__ int pow2_at_least(int n) { return n <= 1 ? 1 : 1 << (32 - __clz(n - 1)); }

// The last token that the cut keeps; tokens with a larger key, or its key and an index up to its own, are kept.
struct Last {
    unsigned key, at;
};
__device__ __forceinline__ bool kept(const Last& l, unsigned k, unsigned i) { return k > l.key || (k == l.key && i <= l.at); }

// The cut of a row whose list overflowed, by bisection over the keys and then over the indices of the key's tokens.
__device__ Last cut_by_bisection(const SampleArgs& A, const Ask& q, int row, Reduce& red) {
    const float* x = A.logits + (int64_t)row * A.ld;
    const int V = A.vocab;
    // tokens and weight of keys > k
    auto count_above = [&](unsigned k) {
        unsigned long long t = 0;
        for (int i = threadIdx.x; i < V; i += kThreads) t += key_of(x[i]) > k;
        return block_sum(red, t);
    };
    auto weight_above = [&](unsigned k) {
        unsigned long long t = 0;
        for (int i = threadIdx.x; i < V; i += kThreads) {
            const float v = x[i];
            if (key_of(v) > k) t += weight(share(v, q.mx, q.T));
        }
        return block_sum(red, t);
    };
    // index of the n-th (from 1) token of key k, the last one if there are fewer
    auto nth = [&](unsigned k, unsigned long long n) {
        unsigned lo = 0, hi = (unsigned)V - 1;
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2;
            unsigned long long t = 0;
            for (unsigned i = threadIdx.x; i <= mid; i += kThreads) t += key_of(x[i]) == k;
            if (block_sum(red, t) >= n) hi = mid; else lo = mid + 1;
        }
        return lo;
    };
    Last l = {0u, 0xffffffffu};
    unsigned long long ties = 0;   // kept tokens of key l.key
    const unsigned top = key_of(q.mx);
    if (q.mode == kTopK) {
        unsigned lo = 0, hi = top;
        while (lo < hi) {          // the smallest key with fewer than top_k keys above it
            const unsigned mid = lo + (hi - lo) / 2;
            if (count_above(mid) < (unsigned long long)q.top_k) hi = mid; else lo = mid + 1;
        }
        if (lo == 0) lo = 1;       // (fewer candidates than top_k: all of them)
        ties = min((unsigned long long)q.top_k - count_above(lo), count_above(lo - 1) - count_above(lo));
        l.key = lo;
        l.at = ties ? nth(lo, ties) : 0u;
    }
    if (q.top_p < 1.0f) {
        const unsigned long long w_key = l.key ? weight(share(of_key(l.key), q.mx, q.T)) : 0;
        const unsigned long long total = weight_above(l.key) + ties * w_key;
        const unsigned long long limit = (unsigned long long)((double)q.top_p * (double)total);
        unsigned lo = l.key, hi = top;
        while (lo < hi) {          // the smallest key with less than `limit` above it
            const unsigned mid = lo + (hi - lo) / 2;
            if (weight_above(mid) < limit) hi = mid; else lo = mid + 1;
        }
        if (limit == 0) return Last{top, q.best_at};
        const unsigned long long w = lo ? weight(share(of_key(lo), q.mx, q.T)) : 0;
        const unsigned long long n = w ? (limit - weight_above(lo) + w - 1) / w : 0;
        if (lo != l.key || n < ties) {
            l.key = lo;
            l.at = n ? nth(lo, n) : 0u;
        }
    }
    return l;
}

// Launch 4.  Workgroup: a row.
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(const SampleArgs A) {
    __shared__ Reduce red;
    __shared__ unsigned long long list[kList];
    __shared__ unsigned long long totals[kMaxChunks];
    __shared__ unsigned long long found[3];
    const int row = blockIdx.x, tid = threadIdx.x;
    const float* x = A.logits + (int64_t)row * A.ld;
    const Ask q = ask_of(A, row);
    if (q.mode <= kGreedy) {
        if (tid == 0) {
            A.ids[row] = q.mode == kNone ? 0 : (int)q.best_at;
            if (A.prob) A.prob[row] = q.mode == kNone ? 0.0f : 1.0f;
        }
        return;
    }
    const double u = A.u[row];
    Last last = {0u, 0xffffffffu};
    int n = 0;
    bool fits = true;
    Cut cut = {kBins, 0, 0};
    if (q.mode != kFree) {
        cut = find_cut(A, q, row, list);
        const unsigned listed = A.listed[row];
        fits = listed <= (unsigned)kList;
        if (fits) {
            n = (int)listed;
            const int size = pow2_at_least(n);
            __syncthreads();
            for (int i = tid; i < size; i += kThreads) list[i] = i < n ? A.list[(int64_t)row * kList + i] : ~0ull;
            sort_list(list, size);
        } else {
            last = cut_by_bisection(A, q, row, red);
        }
    }
    constexpr int PER = kList / kThreads;
    unsigned long long w[PER];
    if (fits && q.mode != kFree) {
        // the list's tokens in order: thread t has PER of them
        unsigned long long sum = 0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const int i = tid * PER + j;
            w[j] = i < n && (q.mode != kTopK || i < q.top_k) ? weight(share(of_key(~(unsigned)(list[i] >> 32)), q.mx, q.T)) : 0;
            sum += w[j];
        }
        unsigned long long ahead = block_scan(red, sum) - sum;
        int keep = q.mode == kTopK ? min(n, q.top_k) : n;
        if (q.top_p < 1.0f) {
            unsigned long long limit = cut.limit;
            if (q.mode == kTopK) {   // of what top_k has kept
                const unsigned long long total = block_sum(red, sum);
                limit = (unsigned long long)((double)q.top_p * (double)total);
            } else {
                ahead += cut.above;
            }
            unsigned long long c = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                c += tid * PER + j < keep && ahead < limit;
                ahead += w[j];
            }
            keep = max((int)block_sum(red, c), 1);
        }
        __syncthreads();
        if (tid == 0) found[0] = keep;
        if (q.mode == kTopK) {
            // the pick in index order, among the list's first `keep`
            const int size = pow2_at_least(keep);
            unsigned long long mine[PER];
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int i = tid + j * kThreads;
                mine[j] = i < keep ? list[i] << 32 | list[i] >> 32 : ~0ull;   // index : ~key
            }
            __syncthreads();
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (tid + j * kThreads < size) list[tid + j * kThreads] = mine[j];
            sort_list(list, size);
            sum = 0;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const int i = tid * PER + j;
                w[j] = 0;
                if (i < keep) {
                    const float e = share(of_key(~(unsigned)list[i]), q.mx, q.T);
                    if (e >= q.min_p) w[j] = weight(e);
                }
                sum += w[j];
            }
            const unsigned long long total = block_sum(red, sum);
            const unsigned long long target = min((unsigned long long)fmax(u * (double)total, 0.0), total - 1);
            unsigned long long run = block_scan(red, sum) - sum;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                if (run <= target && target < run + w[j]) {   // one token
                    A.ids[row] = (int)(list[tid * PER + j] >> 32);
                    if (A.prob) A.prob[row] = (float)((double)w[j] / (double)total);
                }
                run += w[j];
            }
            return;
        }
        last = Last{~(unsigned)(list[keep - 1] >> 32), (unsigned)list[keep - 1]};
    }
    // the chunks' totals
    for (int c = tid; c < A.chunks; c += kThreads) totals[c] = fits ? A.totals[(int64_t)row * A.chunks + c] : 0;
    __syncthreads();
    if (!fits) {
        for (int c = tid >> 6; c < A.chunks; c += kWaves) {
            unsigned long long t = 0;
            for (int i = c * kChunk + (tid & 63); i < min((c + 1) * kChunk, A.vocab); i += 64) {
                const float v = x[i];
                if (v > -INFINITY && kept(last, key_of(v), (unsigned)i)) {
                    const float e = share(v, q.mx, q.T);
                    if (e >= q.min_p) t += weight(e);
                }
            }
            t = wave_sum(t);
            if ((tid & 63) == 0) totals[c] = t;
        }
    } else if (q.mode == kTopP) {
        const int keep = (int)found[0];
        for (int i = tid; i < keep; i += kThreads) {
            const float e = share(of_key(~(unsigned)(list[i] >> 32)), q.mx, q.T);
            if (e >= q.min_p) atomicAdd(&totals[(unsigned)list[i] / kChunk], weight(e));
        }
    }
    __syncthreads();
    constexpr int CPT = kMaxChunks / kThreads;
    unsigned long long t[CPT], sum = 0;
#pragma unroll
    for (int j = 0; j < CPT; j++) {
        const int c = tid * CPT + j;
        t[j] = c < A.chunks ? totals[c] : 0;
        sum += t[j];
    }
    unsigned long long run = block_scan(red, sum);
    if (tid == kThreads - 1) found[0] = run;
    __syncthreads();
    const unsigned long long total = found[0];
    const unsigned long long target = min((unsigned long long)fmax(u * (double)total, 0.0), total - 1);
    run -= sum;
#pragma unroll
    for (int j = 0; j < CPT; j++) {
        if (run <= target && target < run + t[j]) { found[1] = tid * CPT + j; found[2] = target - run; }
        run += t[j];
    }
    __syncthreads();
    // the pick in its chunk: one token for each thread
    static_assert(kChunk == kThreads, "a token for each thread");
    const unsigned i = (unsigned)found[1] * kChunk + tid;
    const unsigned long long left = found[2];
    const float v = i < (unsigned)A.vocab ? x[i] : -INFINITY;
    unsigned long long mine = 0;
    if (v > -INFINITY && kept(last, key_of(v), i)) {
        const float e = share(v, q.mx, q.T);
        if (e >= q.min_p) mine = weight(e);
    }
    const unsigned long long upto = block_scan(red, mine);
    if (upto - mine <= left && left < upto) {
        A.ids[row] = (int)i;
        if (A.prob) A.prob[row] = (float)((double)mine / (double)total);
    }
}

}  // namespace

int launch_sample(smx_ctx* c, const float* logits, size_t rows, size_t vocab, size_t ld, const smx_sample_params* p, const float* u, int32_t* ids, float* prob) {
    SampleArgs A{};
    A.logits = logits; A.ld = (int64_t)ld; A.rows = (int)rows; A.vocab = (int)vocab;
    A.chunks = (int)((vocab + kChunk - 1) / kChunk);
    if (p) { A.temperature = p->temperature; A.top_k = p->top_k; A.top_p = p->top_p; A.min_p = p->min_p; }
    A.u = u; A.ids = ids; A.prob = prob;
    // Parts of a row: 512 workgroups in all (two a CU), of at least one chunk a wave.  Few rows take workgroups of 4 waves, so that
    // a single row spreads over as many CUs as it has chunks for.
    const bool few = rows * (size_t)A.chunks < 512 * 16;
    const int threads = few ? 256 : 1024;
    const size_t want = 512, most = ((size_t)A.chunks + threads / 64 - 1) / (threads / 64);
    size_t parts = std::max<size_t>(1, std::min(most, (want + rows - 1) / rows));
    A.part_chunks = (int)((A.chunks + parts - 1) / parts);
    A.parts = (A.chunks + A.part_chunks - 1) / A.part_chunks;
    // workspace of up to kRowsAtOnce rows (the launches of a larger call follow one another)
    constexpr size_t kRowsAtOnce = 4096;
    const size_t group = std::min(rows, kRowsAtOnce);
    const size_t per_row = (size_t)kBins * 8 + (size_t)A.chunks * 8 + (size_t)kList * 8 + (size_t)A.parts * 8 + 4;
    int rc;
    if ((rc = ensure(c, c->work, group * per_row + 64)) != SMX_OK) return rc;
    A.hist = (unsigned long long*)c->work.p;
    A.totals = A.hist + group * kBins;
    A.list = A.totals + group * A.chunks;
    A.best = (uint2*)(A.list + group * kList);
    A.listed = (unsigned*)(A.best + group * A.parts);
    const bool vec = ld % 4 == 0 && ((uintptr_t)logits & 15) == 0;
    // Without top_k and top_p arrays no row has a cut: no histogram.
    const bool cuts = A.top_k || A.top_p;
    ProfScope ps(c, "sample");
    for (size_t r = 0; r < rows; r += group) {
        SampleArgs G = A;
        const size_t n = std::min(group, rows - r);
        G.rows = (int)n;
        G.logits += r * ld;
        G.temperature = A.temperature ? A.temperature + r : nullptr;
        G.top_k = A.top_k ? A.top_k + r : nullptr;
        G.top_p = A.top_p ? A.top_p + r : nullptr;
        G.min_p = A.min_p ? A.min_p + r : nullptr;
        G.u += r; G.ids += r;
        if (prob) G.prob += r;
        const dim3 grid((unsigned)A.parts, (unsigned)n);
        hipLaunchKernelGGL(vec ? sample_best_kernel<true> : sample_best_kernel<false>, grid, dim3(threads), 0, c->stream, G);
        if (cuts) hipLaunchKernelGGL(vec ? sample_hist_kernel<true> : sample_hist_kernel<false>, grid, dim3(threads), 0, c->stream, G);
        hipLaunchKernelGGL(vec ? sample_gather_kernel<true> : sample_gather_kernel<false>, grid, dim3(threads), 0, c->stream, G);
        hipLaunchKernelGGL(sample_pick_kernel, dim3((unsigned)n), dim3(kThreads), 0, c->stream, G);
        SMX_HIP(c, hipGetLastError());
    }
    return SMX_OK;
}

}  // namespace smx

using namespace smx;

extern "C" int smx_sample_dev(smx_ctx* c, const float* logits, size_t rows, size_t vocab, size_t ld, const smx_sample_params* params, const float* u,
                              int32_t* ids, float* prob) {
    if (!c) return SMX_ERR_ARG;
    if (rows == 0) return SMX_OK;
    if (!logits || !u || !ids) return fail(c, SMX_ERR_ARG, "sample_dev: null argument");
    if (vocab == 0 || ld < vocab) return fail(c, SMX_ERR_ARG, "sample_dev: %zu tokens, %zu elements from row to row", vocab, ld);
    if (vocab > (size_t)kMaxVocab || rows > (size_t(1) << 24)) return fail(c, SMX_ERR_LIMIT, "sample_dev: %zu tokens (%d), %zu rows (2^24)", vocab, SMX_SAMPLE_MAX_VOCAB, rows);
    return launch_sample(c, logits, rows, vocab, ld, params, u, ids, prob);
}

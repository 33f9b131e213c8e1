// Sampling: one token for each row of logits by temperature, top-k, top-p and min-p from a given uniform number.
//
// A token's weight is a whole number, floor(exp((x - max) / T) * 2^40), so every sum below is exact and has one value in any
// order: the cut of top_p and the pick are the same however a row is split over threads.  (With fp32 sums a pick would change
// with the split in about one row of 50 of an unfiltered 262144-token row.)
//
// Rows are ordered by (logit descending, index ascending).  A prefix of that order is a pair (key, ties): every token whose key is
// larger and the first `ties` of those whose key is equal, so neither top-k nor top-p sorts.
#include <algorithm>
#include <climits>
#include <cmath>

#include "smx_internal.h"

namespace smx {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kChunks = 1024;   // parts of a row whose kept weight is totalled, in index order

struct SampleArgs {
    const float* logits;
    int64_t ld;
    int vocab, chunk;   // chunk: tokens per part (a multiple of 64)
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* ids;
    float* prob;
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

struct Reduce {
    unsigned long long a[kWaves];
};
__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ unsigned long long block_sum(Reduce& r, unsigned long long v) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.a[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long t = 0;
    for (int w = 0; w < kWaves; w++) t += r.a[w];
    return t;
}

__global__ __launch_bounds__(kThreads) void sample_row_kernel(const SampleArgs A) {
    __shared__ Reduce red;
    __shared__ unsigned bv[kWaves], bi[kWaves];
    __shared__ unsigned long long above[kChunks];
    __shared__ unsigned ties_in[kChunks];
    __shared__ unsigned long long found[3];
    const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const float* x = A.logits + (int64_t)row * A.ld;
    const int V = A.vocab;
    // the largest logit, lowest index on equal ones
    unsigned bk = 0, at = 0xffffffffu;
    for (int i = tid; i < V; i += kThreads) {
        const unsigned k = key_of(x[i]);
        if (k > bk) { bk = k; at = i; }
    }
    for (int o = 1; o < 64; o <<= 1) {
        const unsigned k = __shfl_xor(bk, o), i = __shfl_xor(at, o);
        if (k > bk || (k == bk && i < at)) { bk = k; at = i; }
    }
    if (lane == 0) { bv[wave] = bk; bi[wave] = at; }
    __syncthreads();
    bk = bv[0]; at = bi[0];
    for (int w = 1; w < kWaves; w++)
        if (bv[w] > bk || (bv[w] == bk && bi[w] < at)) { bk = bv[w]; at = bi[w]; }
    const float T = A.temperature ? A.temperature[row] : 1.0f;
    const int top_k = A.top_k ? A.top_k[row] : 0;
    const float top_p = A.top_p ? A.top_p[row] : 1.0f;
    const float min_p = A.min_p ? fminf(A.min_p[row], 1.0f) : 0.0f;
    if (bk == 0 || !(T > 0.0f) || top_k == 1) {
        if (tid == 0) {
            A.ids[row] = bk == 0 ? 0 : (int)at;
            if (A.prob) A.prob[row] = bk == 0 ? 0.0f : 1.0f;
        }
        return;
    }
    const float mx = of_key(bk);
    unsigned tau = 0;              // the prefix kept so far: keys above tau, and `ties` tokens of key tau
    unsigned long long ties = ~0ull;
    auto weight_above = [&](unsigned k, unsigned least) {   // total weight of keys > k, and >= least
        unsigned long long t = 0;
        for (int i = tid; i < V; i += kThreads) {
            const float v = x[i];
            const unsigned kk = key_of(v);
            if (kk > k && kk >= least) t += weight(share(v, mx, T));
        }
        return block_sum(red, t);
    };
    auto count_above = [&](unsigned k) {
        unsigned long long t = 0;
        for (int i = tid; i < V; i += kThreads) t += key_of(x[i]) > k;
        return block_sum(red, t);
    };
    if (top_k > 0 && top_k < V) {
        // smallest key with fewer than top_k keys above it
        unsigned lo = 0, hi = bk;
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2;
            if (count_above(mid) < (unsigned long long)top_k) hi = mid; else lo = mid + 1;
        }
        tau = lo;
        ties = (unsigned long long)top_k - count_above(tau);
    }
    unsigned long long w_tau = tau ? weight(share(of_key(tau), mx, T)) : 0;
    if (tau) ties = min(ties, count_above(tau - 1) - count_above(tau));
    if (top_p < 1.0f) {
        const unsigned long long total = weight_above(tau, 0) + (tau ? ties * w_tau : 0);
        const unsigned long long limit = top_p > 0.0f ? (unsigned long long)((double)top_p * (double)total) : 0;
        // smallest key with less than `limit` above it
        unsigned lo = tau, hi = bk;
        while (lo < hi) {
            const unsigned mid = lo + (hi - lo) / 2;
            if (weight_above(mid, 0) < limit) hi = mid; else lo = mid + 1;
        }
        const unsigned long long ahead = weight_above(lo, 0);
        if (limit == 0) {
            tau = bk;
            ties = 1;
        } else {
            const unsigned long long w = lo ? weight(share(of_key(lo), mx, T)) : 0;
            const unsigned long long n = w ? (limit - ahead + w - 1) / w : ~0ull;
            ties = lo == tau ? min(ties, n) : n;
            tau = lo;
        }
        w_tau = tau ? weight(share(of_key(tau), mx, T)) : 0;
    }
    if (tau && share(of_key(tau), mx, T) < min_p) ties = 0;
    // what each part of the row keeps: weight above tau, tokens at tau
    for (int c = wave; c < kChunks; c += kWaves) {
        unsigned long long t = 0;
        unsigned n = 0;
        for (int64_t i = (int64_t)c * A.chunk + lane; i < min((int64_t)(c + 1) * A.chunk, (int64_t)V); i += 64) {
            const float v = x[i];
            const unsigned k = key_of(v);
            if (k > tau) {
                const float e = share(v, mx, T);
                if (e >= min_p) t += weight(e);
            }
            n += k == tau && tau;
        }
        t = wave_sum(t);
        n = (unsigned)wave_sum(n);
        if (lane == 0) { above[c] = t; ties_in[c] = n; }
    }
    __syncthreads();
    if (tid == 0) {
        unsigned long long total = 0, seen = 0;
        for (int c = 0; c < kChunks; c++) {
            const unsigned long long n = seen < ties ? min((unsigned long long)ties_in[c], ties - seen) : 0;
            total += above[c] + n * w_tau;
            seen += ties_in[c];
        }
        const unsigned long long target = min((unsigned long long)fmax((double)A.u[row] * (double)total, 0.0), total - 1);
        unsigned long long run = 0;
        seen = 0;
        int c = 0;
        for (; c < kChunks - 1; c++) {
            const unsigned long long n = seen < ties ? min((unsigned long long)ties_in[c], ties - seen) : 0;
            const unsigned long long next = run + above[c] + n * w_tau;
            if (next > target) break;
            run = next;
            seen += ties_in[c];
        }
        found[0] = (unsigned)c;
        found[1] = target - run;
        found[2] = seen;
        above[0] = total;
    }
    __syncthreads();
    if (wave != 0) return;
    // the part that holds the pick, 64 tokens at a time
    const int c = (int)found[0];
    unsigned long long left = found[1], seen = found[2];
    const unsigned long long total = above[0];
    for (int64_t base = (int64_t)c * A.chunk; base < min((int64_t)(c + 1) * A.chunk, (int64_t)V); base += 64) {
        const int64_t i = base + lane;
        const float v = i < V ? x[i] : -INFINITY;
        const unsigned k = key_of(v);
        const bool tie = tau && k == tau;
        const unsigned long long tied = __ballot(tie);
        const unsigned long long before = seen + __popcll(tied & ((1ull << lane) - 1));
        unsigned long long w = 0;
        if (k > tau) {
            const float e = share(v, mx, T);
            if (e >= min_p) w = weight(e);
        } else if (tie && before < ties) {
            w = w_tau;
        }
        unsigned long long run = w;
        for (int o = 1; o < 64; o <<= 1) {
            const unsigned long long r = __shfl_up(run, o);
            if (lane >= o) run += r;
        }
        const unsigned long long hit = __ballot(run > left);
        if (hit) {
            if (lane == __ffsll((long long)hit) - 1) {
                A.ids[row] = (int)i;
                if (A.prob) A.prob[row] = (float)((double)w / (double)total);
            }
            return;
        }
        left -= __shfl(run, 63);
        seen += __popcll(tied);
    }
}

}  // namespace

int launch_sample(smx_ctx* c, const float* logits, size_t rows, size_t vocab, size_t ld, const smx_sample_params* p, const float* u, int32_t* ids, float* prob) {
    SampleArgs A{};
    A.logits = logits; A.ld = (int64_t)ld; A.vocab = (int)vocab;
    A.chunk = (int)(((vocab + kChunks - 1) / kChunks + 63) & ~size_t(63));
    if (p) { A.temperature = p->temperature; A.top_k = p->top_k; A.top_p = p->top_p; A.min_p = p->min_p; }
    A.u = u; A.ids = ids; A.prob = prob;
    ProfScope ps(c, "sample");
    hipLaunchKernelGGL(sample_row_kernel, dim3((unsigned)rows), dim3(kThreads), 0, c->stream, A);
    SMX_HIP(c, hipGetLastError());
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
    if (vocab > (size_t(1) << 22) || rows > (size_t(1) << 24)) return fail(c, SMX_ERR_LIMIT, "sample_dev: %zu tokens (2^22), %zu rows (2^24)", vocab, rows);
    return launch_sample(c, logits, rows, vocab, ld, params, u, ids, prob);
}

// Sampling: one token for each row of logits by temperature, top-k, top-p and min-p from a given uniform number.
//
// A token's weight is a whole number, floor(exp((x - max) / T) * 2^40), so every sum below is exact and has one value in any
// order: the cut of top_p and the pick are the same however a row is split over workgroups.  (With fp32 sums a pick would change
// with the split in about one row of 50 of an unfiltered 262144-token row.)
//
// Rows are ordered by (logit descending, index ascending), and nothing sorts a row.  Four launches over parts of rows:
//   1  the largest logit
//   2  rows with top_k or top_p: a histogram over kBins steps of distance from it, of tokens (top_k) or of weight (top_p), and in it
//      the bin that the cut falls into
//   3  what lies above the bin is totalled per chunk of kChunk tokens (top_k: listed), the bin's own tokens are listed
//   4  one workgroup for each row sorts the list (up to kList tokens), which places the cut at one token, finds the chunk that
//      the pick falls into from the totals and the pick in the chunk
// A row is read three times (without top_k and top_p: twice), every other launch from its end, where the one in front has left
// the caches.  256 rows of 262144 (268 MB) with top_p on 3 rows of 4: 52 + 53 + 53 + 12 us; one row with top_k and top_p:
// 4 + 8 + 4 + 4.  A list that does not fit (top_k of thousands, thousands of equal logits at the cut, or a cut more than kReach below
// the largest logit) is done without: the row's own workgroup looks for the cut in steps of the logits' keys.
#include <algorithm>
#include <climits>
#include <cmath>
#include <type_traits>

#include "smx_internal.h"

namespace smx {

namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;    // of the row's own workgroup (launch 4)
constexpr int kPartThreads = 512, kPartWaves = kPartThreads / 64;   // of a part's (launches 1 to 3)
constexpr int kChunk = 1024;                             // tokens whose kept weight is totalled together
constexpr int kMaxVocab = SMX_SAMPLE_MAX_VOCAB;   // (its chunks' totals are held in LDS)
constexpr int kBins = 2048;
constexpr float kReach = 28.0f;                          // exp(-28) < 2^-40: beyond it there is no weight
constexpr int kList = 4096;
constexpr int kSteps = 1024;                             // of a long list's keys

struct SampleArgs {
    const float* logits;
    int64_t ld;
    int rows, vocab, chunks, parts, part_chunks;   // part_chunks: chunks per part of a row
    const float *temperature, *top_p, *min_p, *u;
    const int* top_k;
    int* ids;
    float* prob;
    // workspace
    unsigned long long* best;       // [rows][parts] candidate() of the part's largest logit
    unsigned long long* hist;       // [rows][kBins] weight; top_k rows: tokens
    unsigned long long* totals;     // [rows][chunks] kept weight above the cut's bin
    unsigned long long* list;       // [rows][kList] ~key : index
    struct RowCut* cuts;            // [rows]
};

// Where a row's cut is, found by the last workgroup of launch 2 to finish the row.
struct RowCut {
    unsigned long long above, limit;   // weight in front of the cut's bin; floor(top_p * all weight)   (top_p rows)
    float total_from, list_from;       // logits from total_from on are kept, the ones below it from list_from on are the cut's bin
    unsigned done;                     // workgroups of launch 2 that have added their part
    unsigned listed;                   // tokens of the list
};

// Order-preserving key of a logit: NaN and -inf are 0, below every other; -0 is +0.
__device__ __forceinline__ unsigned key_of(float x) {
    const unsigned b = __float_as_uint(x + 0.0f);
    const unsigned k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return x > -INFINITY ? k : 0u;
}
__device__ __forceinline__ float of_key(unsigned k) { return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

// (x - max) / T, correctly rounded, in five operations where the general division alone takes eleven: with a = x - max,
// r = RN(1 / T), q = RN(a r) is within one unit of a / T, the remainder a - q T is exact in an FMA, and RN(q + remainder r) is the
// correctly rounded quotient (Markstein's theorem, for divisors whose mantissa is not all ones).  Distances of more than 200 T count
// as 200 T (exp(-200) is 0 in fp32, and so are the exponentials of all beyond); remainders lose bits to underflow only where
// |a / T| < 2^-40 (exponential 1).  A largest logit of +inf has distance 0 from itself and so a share.
struct Temp {
    float mx, T, r, far;
    bool quick;
};
__device__ __forceinline__ Temp temp_of(float T, float mx) {
    const unsigned b = __float_as_uint(T);
    return Temp{mx, T, 1.0f / T, -200.0f * T, T > 0x1p-60f && T < 0x1p60f && (b & 0x7fffffu) != 0x7fffffu && mx < INFINITY};
}
__device__ __forceinline__ float depth(float x, const Temp& t) {
#pragma clang fp contract(off)
    if (!t.quick) return x == t.mx ? 0.0f : (x - t.mx) / t.T;   // (the same for the whole row)
    const float a = __builtin_amdgcn_fmed3f(x - t.mx, t.far, 0.0f), q = a * t.r;
    return fmaf(fmaf(-q, t.T, a), t.r, q);
}
// floor(e * 2^40) of an e in [0, 1]: below 2^52, so the low bits of the double 2^52 + it are the number (shifts of 64 bits by e's
// exponent instead: launch 2 with 256 rows of 262144 71 us, with this 65)
__device__ __forceinline__ unsigned long long weight(float e) {
    return __builtin_bit_cast(unsigned long long, (double)truncf(e * 0x1p40f) + 0x1p52) & 0xfffffffffffffull;
}
// Bin of a depth: steps of distance below the largest logit.  Every rounding is monotone in x, so a smaller bin means a larger logit.
__device__ __forceinline__ int bin_of(float z) {
#pragma clang fp contract(off)
    return (int)fminf(z * -((float)kBins / kReach), (float)(kBins - 1));
}

// Steps over the lanes of a wave as DPP moves (a shuffle through LDS takes ten times as long, and launch 4 is a chain of them).
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp64(unsigned long long v) {   // 0 where no lane is moved from
    const unsigned lo = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)v, CTRL, ROWS, 0xf, false);
    const unsigned hi = (unsigned)__builtin_amdgcn_update_dpp(0, (int)(unsigned)(v >> 32), CTRL, ROWS, 0xf, false);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ unsigned long long wave_last(unsigned long long v) {   // lane 63's, in every lane
    const unsigned lo = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)v, 63), hi = (unsigned)__builtin_amdgcn_readlane((int)(unsigned)(v >> 32), 63);
    return (unsigned long long)hi << 32 | lo;
}
__device__ __forceinline__ unsigned long long wave_scan(unsigned long long v) {   // inclusive sum
    v += dpp64<0x111, 0xf>(v);   // row_shr 1, 2, 4, 8: sums inside each row of 16 lanes
    v += dpp64<0x112, 0xf>(v);
    v += dpp64<0x114, 0xf>(v);
    v += dpp64<0x118, 0xf>(v);
    v += dpp64<0x142, 0xa>(v);   // row_bcast 15 into rows 1 and 3, row_bcast 31 into rows 2 and 3
    v += dpp64<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ unsigned long long wave_sum(unsigned long long v) { return wave_last(wave_scan(v)); }
template <int CTRL, int ROWS>
__device__ __forceinline__ unsigned long long dpp_max(unsigned long long v) {
    const unsigned long long o = dpp64<CTRL, ROWS>(v);
    return o > v ? o : v;
}
__device__ __forceinline__ unsigned long long wave_max(unsigned long long v) {
    v = dpp_max<0x111, 0xf>(v);
    v = dpp_max<0x112, 0xf>(v);
    v = dpp_max<0x114, 0xf>(v);
    v = dpp_max<0x118, 0xf>(v);
    v = dpp_max<0x142, 0xa>(v);
    v = dpp_max<0x143, 0xc>(v);
    return wave_last(v);
}
// A candidate for the largest logit: the larger word wins, on equal keys the lower index.
__device__ __forceinline__ unsigned long long candidate(unsigned key, unsigned index) { return (unsigned long long)key << 32 | ~index; }

// What a row asks for, and its largest logit.
enum Mode { kNone, kGreedy, kFree, kTopK, kTopP };   // kNone: no candidate at all
struct Ask {
    Mode mode;
    unsigned best_at;
    float mx, top_p, min_p;
    Temp T, bin_T;    // bin_T divides distances for bin_of: T, or 1 where tokens are counted
    int top_k;
    __device__ float share(float x) const { return expf(depth(x, T)); }
    __device__ int bin(float x) const { return bin_of(depth(x, bin_T)); }
};
__device__ __forceinline__ Ask ask_of(const SampleArgs& A, int row) {
    // every wave reads the parts' candidates for itself: no barrier
    unsigned long long b = 0;
    for (int i = threadIdx.x & 63; i < A.parts; i += 64) b = max(b, A.best[(int64_t)row * A.parts + i]);
    b = wave_max(b);
    const unsigned top = (unsigned)(b >> 32);
    Ask q;
    q.best_at = ~(unsigned)b;
    q.mx = of_key(top);
    const float T = A.temperature ? A.temperature[row] : 1.0f;
    q.T = temp_of(T, q.mx);
    q.top_k = A.top_k ? A.top_k[row] : 0;
    q.top_p = A.top_p ? A.top_p[row] : 1.0f;
    q.min_p = A.min_p && A.min_p[row] > 0.0f ? fminf(A.min_p[row], 1.0f) : 0.0f;   // (off where the comparison does not hold: NaN, too)
    const bool k = q.top_k > 0 && q.top_k < A.vocab;
    q.mode = top == 0 ? kNone : !(T > 0.0f) || q.top_k == 1 || q.top_p <= 0.0f ? kGreedy : k ? kTopK : q.top_p < 1.0f ? kTopP : kFree;
    q.bin_T = q.mode == kTopK ? temp_of(1.0f, q.mx) : q.T;
    return q;
}

// A row in chunks of kChunk tokens that start at 16-byte boundaries of memory: chunk c holds tokens kChunk c - skew ..., skew (0..3)
// being how far the row's first token is behind such a boundary.
struct Row {
    const float* x;
    int vocab, skew;
};
__device__ __forceinline__ Row row_of(const SampleArgs& A, int row) {
    const float* x = A.logits + (int64_t)row * A.ld;
    return Row{x, A.vocab, (int)((uintptr_t)x >> 2) & 3};
}
// A lane's 16 tokens of a chunk: token first_of + 256 j + i is v[4 j + i] (-inf outside the row).
__device__ __forceinline__ int first_of(const Row& r, int chunk) { return chunk * kChunk - r.skew + 4 * (int)(threadIdx.x & 63); }
__device__ __forceinline__ int token_of(int first, int n) { return first + 256 * (n >> 2) + (n & 3); }
__device__ __forceinline__ void load_chunk(const Row& r, int chunk, float (&v)[16]) {
    const int first = first_of(r, chunk);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const int i = first + 256 * j;
        if (i >= 0 && i + 4 <= r.vocab) {
            const float4 f = *(const float4*)(r.x + i);
            v[4 * j] = f.x; v[4 * j + 1] = f.y; v[4 * j + 2] = f.z; v[4 * j + 3] = f.w;
        } else {
#pragma unroll
            for (int t = 0; t < 4; t++) v[4 * j + t] = i + t >= 0 && i + t < r.vocab ? r.x[i + t] : -INFINITY;
        }
    }
}

// Which part of which row a workgroup of launches 1 to 3 serves.  Workgroups go to the 8 XCDs in turn, so the same part is the same XCD's
// in every launch (calls of up to a few tens of MB find their logits in its L2), from the end too (`back`: for larger ones, whose last
// parts are still in the memory-side cache); and rows change places in groups of 8, so that rows that ask for alike work and recur with
// a period of 2, 4 or 8 are not all one XCD's.
struct Place {
    int row, part;
};
__device__ __forceinline__ Place place_of(const SampleArgs& A, bool back) {
    int id = blockIdx.y * A.parts + blockIdx.x;
    if (back) {
        const int whole = A.rows * A.parts & ~7;
        if (id < whole) id = (whole - 8 - (id & ~7)) | (id & 7);
    }
    const int y = id / A.parts;
    return Place{(y | 7) < A.rows ? (y & ~7) | ((y + (y >> 3)) & 7) : y, id - y * A.parts};
}

// Launch 1.  Workgroup (part, row); also clears what launches 2 and 3 add to.
__global__ __launch_bounds__(kPartThreads) void sample_best_kernel(const SampleArgs A) {
    __shared__ unsigned long long red[kPartWaves];
    const Place at = place_of(A, false);
    const int row = at.row, part = at.part, wave = threadIdx.x >> 6;
    const Row x = row_of(A, row);
    for (int i = part * kPartThreads + threadIdx.x; i < kBins; i += A.parts * kPartThreads) A.hist[(int64_t)row * kBins + i] = 0;
    if (part == 0 && threadIdx.x == 0) { A.cuts[row].done = 0; A.cuts[row].listed = 0; }
    unsigned bk = 0, bi = 0;
    const int c1 = min((part + 1) * A.part_chunks, A.chunks);
    for (int c = part * A.part_chunks + wave; c < c1; c += kPartWaves) {
        float v[16];
        load_chunk(x, c, v);
        const int first = first_of(x, c);
#pragma unroll
        for (int n = 0; n < 16; n++) {   // (a lane's tokens ascend: the first of equals stays)
            const unsigned k = key_of(v[n]);
            if (k > bk) { bk = k; bi = (unsigned)token_of(first, n); }
        }
    }
    unsigned long long b = wave_max(candidate(bk, bi));
    if ((threadIdx.x & 63) == 0) red[wave] = b;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kPartWaves; w++) b = max(b, red[w]);
        A.best[(int64_t)row * A.parts + part] = b;
    }
}

// The smallest logit whose bin is below `bin` (comparing with it replaces a division for each token); NaN if there is none.
// A wave tries 64 keys at a time.
__device__ __forceinline__ float floor_of_bin(const Ask& q, int bin) {
    const int lane = threadIdx.x & 63;
    unsigned lo = key_of(-3.402823466e38f), hi = key_of(q.mx) + 1;   // none below lo; hi stands for none at all
    const unsigned none = hi;
    while (lo < hi) {
        const unsigned step = (hi - lo + 63) / 64, k = min(lo + lane * step, hi);
        const unsigned long long yes = __ballot(k == hi || q.bin(of_key(k)) < bin);
        const int f = yes ? __ffsll((long long)yes) - 1 : 64;
        const unsigned base = lo;
        if (f > 0) lo = base + (f - 1) * step + 1;
        if (f < 64) hi = min(base + f * step, hi);
    }
    return lo == none ? __uint_as_float(0x7fc00000u) : of_key(lo);
}

// Launch 2.  Workgroup (part, row), from the last to the first.  The last one of a row to finish reads the whole histogram: the
// cut's bin is the first whose running total reaches top_k tokens, or floor(top_p * all weight).  Bound by some 35 instructions a
// token, the LDS atomic among them: 160 rows of 262144 with top_p and 96 without 53 us.
__global__ __launch_bounds__(kPartThreads) void sample_hist_kernel(const SampleArgs A) {
    __shared__ unsigned long long hist[kBins], red[kPartWaves];
    __shared__ unsigned done;
    const Place at = place_of(A, true);
    const int row = at.row, part = at.part, wave = threadIdx.x >> 6;
    const Ask q = ask_of(A, row);
    if (q.mode != kTopK && q.mode != kTopP) return;
    const Row x = row_of(A, row);
    for (int i = threadIdx.x; i < kBins; i += kPartThreads) hist[i] = 0;
    __syncthreads();
    const int c0 = part * A.part_chunks, c1 = min(c0 + A.part_chunks, A.chunks);
    for (int c = c1 - 1 - wave; c >= c0; c -= kPartWaves) {
        float v[16];
        load_chunk(x, c, v);
#pragma unroll
        for (int n = 0; n < 16; n++) {
            const float z = depth(v[n], q.bin_T);
            const unsigned long long w = q.mode == kTopK ? 1ull : weight(expf(z));
            if (w && v[n] > -INFINITY) atomicAdd(&hist[bin_of(z)], w);
        }
    }
    __syncthreads();
    unsigned long long* all = A.hist + (int64_t)row * kBins;
    RowCut* cut = A.cuts + row;
    for (int i = threadIdx.x; i < kBins; i += kPartThreads) {
        const unsigned long long w = hist[i];
        if (w) atomicAdd(&all[i], w);
    }
    // What passes between workgroups is atomic at device scope, performed where all XCDs see it: this thread's additions are
    // waited for, then the workgroup counts itself; the reads below are atomic too.  That an atomic has been performed once it has been
    // waited for is the hardware's; in the language's terms this is no release.  (A fence by each wave would be one and write its XCD's L2
    // back: 256 rows of 262144 329 us instead of 75.)
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (threadIdx.x == 0) done = atomicAdd(&cut->done, 1u);
    __syncthreads();
    if (done != (unsigned)A.parts - 1) return;
    constexpr int PER = kBins / kPartThreads;   // neighbouring bins for each thread
    unsigned long long bins[PER], sum = 0;
#pragma unroll
    for (int j = 0; j < PER; j++)   // (all in flight at once)
        bins[j] = __hip_atomic_load(&all[threadIdx.x * PER + j], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int j = 0; j < PER; j++) {
        hist[threadIdx.x * PER + j] = bins[j];
        sum += bins[j];
    }
    unsigned long long run = wave_scan(sum);
    if ((threadIdx.x & 63) == 63) red[wave] = run;
    __syncthreads();
    unsigned long long total = 0, front = 0;
    for (int w = 0; w < kPartWaves; w++) {
        if (w < wave) front += red[w];
        total += red[w];
    }
    run += front - sum;   // in front of this thread's bins
    const unsigned long long limit = q.mode == kTopK ? (unsigned long long)q.top_k : (unsigned long long)((double)q.top_p * (double)total);
    // where the running total first reaches the limit; a limit of 0: the first bin; fewer candidates than top_k: behind the last bin
    __shared__ int bin;
    __shared__ unsigned long long above;
    if (threadIdx.x == 0) { bin = limit == 0 ? 0 : kBins; above = limit == 0 ? 0 : total; }
    __syncthreads();
    if (run < limit && run + sum >= limit) {
        int i = threadIdx.x * PER;
        while (run + hist[i] < limit) run += hist[i++];
        bin = i;
        above = run;
    }
    __syncthreads();
    if (wave < 2) {
        const float f = floor_of_bin(q, bin + wave);
        if ((threadIdx.x & 63) == 0) *(wave == 0 ? &cut->total_from : &cut->list_from) = wave == 0 && q.mode == kTopK ? __uint_as_float(0x7fc00000u) : f;
    }
    if (threadIdx.x == 0) { cut->above = above; cut->limit = limit; }
}

// Launch 3.  Workgroup (part, row).  Tokens below the cut's bin take one comparison, the ones above it an exponential, the bin's own
// (few) an LDS atomic.  256 rows of 262144, 224 of them to be read (235 MB), 160 with top_p: 53 us.  Its scalar registers are kept to what lets
// 8 waves share a SIMD (7, and so a workgroup less on each CU, took 83 us where this took 63).
__global__ __launch_bounds__(kPartThreads, 8) void sample_gather_kernel(const SampleArgs A) {
    __shared__ unsigned long long list[kList];
    __shared__ unsigned found, start;
    const Place at = place_of(A, false);
    const int row = at.row, part = at.part, wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const Ask q = ask_of(A, row);
    if (q.mode <= kGreedy) return;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    // (NaN: none; top_k rows list everything that they keep)
    const float total_from = q.mode == kFree ? -3.402823466e38f : A.cuts[row].total_from;
    const float list_from = q.mode == kFree ? total_from : A.cuts[row].list_from;
    const Row x = row_of(A, row);
    const int c1 = min((part + 1) * A.part_chunks, A.chunks);
    for (int c = part * A.part_chunks + wave; c < c1; c += kPartWaves) {
        float v[16];
        load_chunk(x, c, v);
        const int first = first_of(x, c);
        double sum = 0;   // of 16 whole numbers up to 2^40: exact
#pragma unroll
        for (int n = 0; n < 16; n++) {
            if (v[n] >= list_from) {
                if (v[n] >= total_from) {
                    const float e = q.share(v[n]);
                    if (e >= q.min_p) sum += (double)truncf(e * 0x1p40f);
                } else {
                    const unsigned at = atomicAdd(&found, 1u);
                    if (at < (unsigned)kList) list[at] = (unsigned long long)~key_of(v[n]) << 32 | (unsigned)token_of(first, n);
                }
            }
        }
        if (q.mode != kTopK) {
            const unsigned long long total = wave_sum((unsigned long long)sum);
            if (lane == 0) A.totals[(int64_t)row * A.chunks + c] = total;
        }
    }
    // behind the other parts' tokens in the row's list (what does not fit is only counted)
    __syncthreads();
    const unsigned n = found;
    if (n == 0) return;
    if (threadIdx.x == 0) start = atomicAdd(&A.cuts[row].listed, n);
    __syncthreads();
    for (unsigned i = threadIdx.x; i < n && start + i < (unsigned)kList; i += kPartThreads) A.list[(int64_t)row * kList + start + i] = list[i];
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
__device__ __forceinline__ unsigned long long block_max(Reduce& r, unsigned long long v) {
    v = wave_max(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) r.a[threadIdx.x >> 6] = v;
    __syncthreads();
    unsigned long long t = 0;
    for (int w = 0; w < kWaves; w++) t = max(t, r.a[w]);
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

// Sorts 2^m words upwards, word tid + kThreads e of them in v[e] of thread tid (bitonic; n <= kThreads E, the rest idle).  Steps of
// less than a wave are exchanges between lanes, steps of kThreads and more are a thread's own, the ones between go through LDS.
__device__ __forceinline__ unsigned long long lane_xor(unsigned long long v, int o) { return __shfl_xor(v, o); }
template <int E>
__device__ void sort_words(unsigned long long (&v)[E], unsigned long long* lds, int n) {
    for (int k = 2; k <= n; k <<= 1)
        for (int j = k >> 1; j > 0; j >>= 1) {
            if (j >= kThreads) {
                const int ej = j / kThreads;
#pragma unroll
                for (int e = 0; e < E; e++)
#pragma unroll
                    for (int f = e + 1; f < E; f++)
                        if (f == (e ^ ej)) {
                            const bool up = ((e * kThreads) & k) == 0;
                            const unsigned long long p = v[e], r = v[f];
                            if ((p > r) == up) { v[e] = r; v[f] = p; }
                        }
            } else {
                unsigned long long o[E];
                if (j < 64) {
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = lane_xor(v[e], j);
                } else {
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < E; e++) lds[e * kThreads + threadIdx.x] = v[e];
                    __syncthreads();
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = lds[e * kThreads + (threadIdx.x ^ j)];
                }
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int i = e * kThreads + threadIdx.x;
                    const bool up = (i & k) == 0, low = (i & j) == 0;
                    v[e] = (v[e] < o[e]) == (up == low) ? v[e] : o[e];
                }
            }
        }
    __syncthreads();
}
// The n words that from(i) gives, sorted upwards in a[0, n); n <= kList.
template <class F>
__device__ __forceinline__ void sort_list(unsigned long long* a, int n, F&& from) {
    const int tid = threadIdx.x;
    auto run = [&](auto tag, int size) {
        constexpr int E = decltype(tag)::value;
        unsigned long long v[E];
#pragma unroll
        for (int e = 0; e < E; e++) v[e] = e * kThreads + tid < n ? from(e * kThreads + tid) : ~0ull;
        __syncthreads();   // `from` may have read a
        sort_words<E>(v, a, size);
#pragma unroll
        for (int e = 0; e < E; e++) a[e * kThreads + tid] = v[e];
        __syncthreads();
    };
    const int size = n <= 1 ? 1 : 1 << (32 - __clz(n - 1));
    static_assert(kList <= 16 * kThreads, "16 words for each thread");
    if (size <= kThreads) run(std::integral_constant<int, 1>{}, size);
    else if (size <= 4 * kThreads) run(std::integral_constant<int, 4>{}, size);
    else run(std::integral_constant<int, 16>{}, size);
}

// The last token that the cut keeps; tokens with a larger key, or its key and an index up to its own, are kept.
struct Last {
    unsigned key, at;
};
__device__ __forceinline__ bool kept(const Last& l, unsigned k, unsigned i) { return k > l.key || (k == l.key && i <= l.at); }

// The same for a list's word
__device__ __forceinline__ bool kept(const Last& l, unsigned long long word) { return kept(l, ~(unsigned)(word >> 32), (unsigned)word); }
__device__ __forceinline__ unsigned long long list_weight(const Ask& q, unsigned long long word) {
    return weight(q.share(of_key(~(unsigned)(word >> 32))));
}

// Where the list's words that `bound` keeps, taken in order with `front` in front of them, reach `limit` (weight, or their number):
// the last word with less than `limit` in front of it, at least the first one.  The words go into kSteps steps of their keys; the step
// that the limit falls into is ordered by itself (thousands of equal logits: by index).
__device__ Last place(const SampleArgs& A, const Ask& q, Reduce& red, const unsigned long long* list, int n, unsigned long long* step,
                      unsigned long long* members, unsigned long long* found, Last bound, bool weighed, unsigned long long front, unsigned long long limit) {
    const int tid = threadIdx.x;
    unsigned lo = 0xffffffffu, hi = 0;
    for (int i = tid; i < n; i += kThreads) {
        lo = min(lo, (unsigned)(list[i] >> 32));
        hi = max(hi, (unsigned)(list[i] >> 32));
    }
    lo = ~(unsigned)block_max(red, ~lo);
    hi = (unsigned)block_max(red, hi);
    const int shift = max(0, 22 - __clz(hi - lo | 1));   // (hi - lo) >> shift < kSteps
    for (int i = tid; i < kSteps; i += kThreads) step[i] = 0;
    if (tid == 0) { found[0] = kSteps; found[1] = 0; found[2] = 0; }
    __syncthreads();
    for (int i = tid; i < n; i += kThreads) {
        const unsigned long long w = list[i];
        if (kept(bound, w)) atomicAdd(&step[((unsigned)(w >> 32) - lo) >> shift], weighed ? list_weight(q, w) : 1ull);
    }
    __syncthreads();
    constexpr int PER = kSteps / kThreads;
    unsigned long long sum = 0;
    for (int i = 0; i < PER; i++) sum += step[tid * PER + i];
    unsigned long long run = front + block_scan(red, sum) - sum;
    if (run < limit && run + sum >= limit) {
        int i = tid * PER;
        while (run + step[i] < limit) run += step[i++];
        found[0] = i;
        found[1] = run;
    }
    __syncthreads();
    const unsigned at = limit <= front ? 0u : (unsigned)found[0];   // (nothing fits: the first word alone, which is in the first step)
    if (at == kSteps) return bound;                                  // everything fits
    run = limit <= front ? front : found[1];
    for (int i = tid; i < n; i += kThreads) {
        const unsigned long long w = list[i];
        if (kept(bound, w) && ((unsigned)(w >> 32) - lo) >> shift == at) members[atomicAdd((unsigned*)&found[2], 1u)] = w;
    }
    __syncthreads();
    const int m = (int)found[2];
    unsigned long long mine = ~0ull, best = 0;
    if (m <= kThreads) {
        if (tid < m) mine = members[tid];
        __syncthreads();
        ulonglong2* const pairs = (ulonglong2*)members;
        pairs[tid] = make_ulonglong2(mine, tid < m ? weighed ? list_weight(q, mine) : 1ull : 0ull);
        __syncthreads();
        bool first = true;
#pragma unroll 8
        for (int i = 0; i < m; i++) {
            const ulonglong2 o = pairs[i];
            const bool before = o.x < mine;
            first = first && !before;
            run += before ? o.y : 0;
        }
        if (tid < m && (first || run < limit)) best = mine;
    } else {
        sort_list(members, m, [&](int i) { return members[i]; });
        const int per = (m + kThreads - 1) / kThreads, i0 = min(tid * per, m), i1 = min(i0 + per, m);
        sum = 0;
        for (int i = i0; i < i1; i++) sum += weighed ? list_weight(q, members[i]) : 1ull;
        run += block_scan(red, sum) - sum;
        for (int i = i0; i < i1; i++) {
            if (i == 0 || run < limit) best = members[i];
            run += weighed ? list_weight(q, members[i]) : 1ull;
        }
    }
    best = block_max(red, best);
    return Last{~(unsigned)(best >> 32), (unsigned)best};
}

// f(logit, index) for every token of a lane's share of a chunk, 4 at a time (a row's own workgroup has other uses for registers).
template <class F>
__device__ __forceinline__ void each_token(const Row& r, int chunk, F&& f) {
    const int first = first_of(r, chunk);
#pragma unroll 1
    for (int j = 0; j < 4; j++) {
        const int i = first + 256 * j;
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (i >= 0 && i + 4 <= r.vocab) {
            v = *(const float4*)(r.x + i);
        } else {
            if (i >= 0 && i < r.vocab) v.x = r.x[i];
            if (i + 1 >= 0 && i + 1 < r.vocab) v.y = r.x[i + 1];
            if (i + 2 >= 0 && i + 2 < r.vocab) v.z = r.x[i + 2];
            if (i + 3 >= 0 && i + 3 < r.vocab) v.w = r.x[i + 3];
        }
        f(v.x, (unsigned)i);
        f(v.y, (unsigned)i + 1);
        f(v.z, (unsigned)i + 2);
        f(v.w, (unsigned)i + 3);
    }
}

// The cut of a row whose list overflowed, in steps of kBins ranges of keys (three at most) and then by the index among the last key's tokens.
// bins [kBins], counts [chunks].  A row of 262144 with top_k = 20000 0.6 ms, with top_p in it 1.1 (bisection over the keys 5.0 and 9.3).
__device__ Last cut_by_steps(const SampleArgs& A, const Ask& q, const Row& r, Reduce& red, unsigned long long* bins, unsigned long long* counts,
                             unsigned long long* found) {
    const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
    const unsigned top = key_of(q.mx);
    // index of the n-th (from 1) token of a key that the bound keeps
    auto nth = [&](unsigned key, unsigned long long n, Last bound) {
        for (int c = wave; c < A.chunks; c += kWaves) {
            unsigned m = 0;
            each_token(r, c, [&](float v, unsigned i) { m += key_of(v) == key && kept(bound, key, i); });
            const unsigned long long t = wave_sum(m);
            if (lane == 0) counts[c] = t;
        }
        __syncthreads();
        const int per = (A.chunks + kThreads - 1) / kThreads, c0 = min(tid * per, A.chunks), c1 = min(c0 + per, A.chunks);
        unsigned long long sum = 0;
        for (int c = c0; c < c1; c++) sum += counts[c];
        unsigned long long run = block_scan(red, sum) - sum;
        if (run < n && n <= run + sum) {
            int c = c0;
            while (run + counts[c] < n) run += counts[c++];
            found[0] = c;
            found[1] = n - run;
        }
        __syncthreads();
        const int first = (int)found[0] * kChunk - r.skew + tid * (kChunk / kThreads);
        const unsigned long long left = found[1];
        sum = 0;
        for (int e = 0; e < kChunk / kThreads; e++) sum += first + e >= 0 && first + e < r.vocab && key_of(r.x[first + e]) == key;
        run = block_scan(red, sum) - sum;
        if (run < left && left <= run + sum) {
            int e = 0;
            for (; run < left; e++) run += first + e >= 0 && first + e < r.vocab && key_of(r.x[first + e]) == key;
            found[0] = first + e - 1;
        }
        __syncthreads();
        const unsigned at = (unsigned)found[0];
        __syncthreads();   // (the next cut writes found again)
        return at;
    };
    // the last of the bound's tokens, in order, with less than the limit in front of it: `limit` tokens, or (weighed) top_p of their weight
    auto cut = [&](Last bound, bool weighed, unsigned long long limit) {
        unsigned lo = max(bound.key, 1u), hi = top;
        unsigned long long front = 0;
        for (bool whole = true;; whole = false) {
            const int shift = max(0, 21 - __clz(hi - lo | 1));   // (hi - lo) >> shift < kBins
            for (int i = tid; i < kBins; i += kThreads) bins[i] = 0;
            if (tid == 0) found[0] = kBins;
            __syncthreads();
            for (int c = wave; c < A.chunks; c += kWaves)
                each_token(r, c, [&](float v, unsigned i) {
                    const unsigned k = key_of(v);
                    if (k < lo || k > hi || !kept(bound, k, i)) return;
                    const unsigned long long w = weighed ? weight(q.share(v)) : 1ull;
                    if (w) atomicAdd(&bins[(hi - k) >> shift], w);
                });
            __syncthreads();
            constexpr int PER = kBins / kThreads;
            unsigned long long sum = 0;
            for (int i = 0; i < PER; i++) sum += bins[tid * PER + i];
            if (whole && weighed) {
                limit = (unsigned long long)((double)q.top_p * (double)block_sum(red, sum));
                if (limit == 0) return Last{top, q.best_at};
            }
            unsigned long long run = front + block_scan(red, sum) - sum;
            if (run < limit && run + sum >= limit) {
                int i = tid * PER;
                while (run + bins[i] < limit) run += bins[i++];
                found[0] = i;
                found[1] = run;
            }
            __syncthreads();
            const unsigned b = (unsigned)found[0];
            if (b == kBins) return bound;   // everything fits
            front = found[1];
            hi -= b << shift;
            lo = hi - min((1u << shift) - 1, hi - lo);
            __syncthreads();
            if (shift == 0) break;
        }
        const unsigned long long w = weighed ? weight(q.share(of_key(hi))) : 1ull;
        return Last{hi, nth(hi, (limit - front + w - 1) / w, bound)};
    };
    Last l = {0u, 0xffffffffu};
    if (q.mode == kTopK) l = cut(l, false, (unsigned long long)q.top_k);
    return q.top_p < 1.0f ? cut(l, true, 0) : l;
}

// Launch 4.  Workgroup: a row.
__global__ __launch_bounds__(kThreads) void sample_pick_kernel(const SampleArgs A) {
    __shared__ Reduce red;
    __shared__ unsigned long long found[3];
    extern __shared__ __align__(16) unsigned long long room[];   // list [kList], members [kList], totals [chunks] or steps [kSteps]
    unsigned long long *const list = room, *const members = room + kList, *const totals = room + 2 * kList, *const step = totals;
    unsigned long long* const ws = members;         // weights of a chunk
    ulonglong2* const pairs = (ulonglong2*)members; // words and weights of a short list
    const int row = blockIdx.x, tid = threadIdx.x;
    const Row r = row_of(A, row);
    const float* x = r.x;
    const RowCut cut = A.cuts[row];   // (asked for with the row's parameters; means something where there is a cut)
    const double u = A.u[row];
    const Ask q = ask_of(A, row);
    if (q.mode <= kGreedy) {
        if (tid == 0) {
            A.ids[row] = q.mode == kNone ? 0 : (int)q.best_at;
            if (A.prob) A.prob[row] = q.mode == kNone ? 0.0f : 1.0f;
        }
        return;
    }
    Last last = {0u, 0xffffffffu};
    bool fits = true;
    int keep = 0;   // of the list, in order
    if (q.mode != kFree) {
        const unsigned long long* from = A.list + (int64_t)row * kList;
        fits = cut.listed <= (unsigned)kList;
        const int n = fits ? (int)cut.listed : 0;
        if (!fits) {
            last = cut_by_steps(A, q, r, red, members, totals, found);
        } else if (n <= kThreads) {
            // a token for each thread; its rank and the weight in front of it by comparing with every other
            const unsigned long long mine = tid < n ? from[tid] : ~0ull;
            const unsigned long long w = tid < n ? weight(q.share(of_key(~(unsigned)(mine >> 32)))) : 0;
            list[tid] = mine;
            pairs[tid] = make_ulonglong2(mine, w);
            __syncthreads();
            int rank = 0;
            unsigned long long ahead = 0;
#pragma unroll 8
            for (int i = 0; i < n; i++) {
                const ulonglong2 o = pairs[i];
                const bool before = o.x < mine;
                rank += before;
                ahead += before ? o.y : 0;
            }
            bool stay = tid < n && (q.mode != kTopK || rank < q.top_k);
            if (q.top_p < 1.0f) {
                unsigned long long limit = cut.limit;
                if (q.mode == kTopK) limit = (unsigned long long)((double)q.top_p * (double)block_sum(red, stay ? w : 0));
                else ahead += cut.above;
                stay = stay && (rank == 0 || ahead < limit);
            }
            if (q.mode == kTopK) {
                const float e = q.share(of_key(~(unsigned)(mine >> 32)));
                const unsigned long long kw = stay && e >= q.min_p ? w : 0;
                const unsigned long long total = block_sum(red, kw);
                const unsigned long long target = min((unsigned long long)fmax(u * (double)total, 0.0), total - 1);
                pairs[tid] = make_ulonglong2((unsigned)mine, kw);   // (read by everyone: block_sum has met since)
                __syncthreads();
                unsigned long long run = 0;   // kept weight of tokens in front of this one by index
#pragma unroll 8
                for (int i = 0; i < n; i++) {
                    const ulonglong2 o = pairs[i];
                    run += o.x < (unsigned)mine ? o.y : 0;
                }
                if (run <= target && target < run + kw) {
                    A.ids[row] = (int)(unsigned)mine;
                    if (A.prob) A.prob[row] = (float)((double)kw / (double)total);
                }
                return;
            }
            const int count = (int)block_sum(red, stay);
            if (stay && rank == count - 1) found[0] = mine;
            __syncthreads();
            last = Last{~(unsigned)(found[0] >> 32), (unsigned)found[0]};
            keep = n;
        } else {
            for (int i = tid; i < n; i += kThreads) list[i] = from[i];
            __syncthreads();
            // (a cut in LDS: the list by kSteps steps of its keys, then the step's own tokens)
            if (q.mode == kTopK) {
                last = place(A, q, red, list, n, step, members, found, last, false, 0, (unsigned long long)q.top_k);
                if (q.top_p < 1.0f) {
                    unsigned long long t = 0;
                    for (int i = tid; i < n; i += kThreads) t += kept(last, list[i]) ? list_weight(q, list[i]) : 0;
                    const unsigned long long limit = (unsigned long long)((double)q.top_p * (double)block_sum(red, t));   // of what top_k has kept
                    last = place(A, q, red, list, n, step, members, found, last, true, 0, limit);
                }
            } else {
                last = place(A, q, red, list, n, step, members, found, last, true, cut.above, cut.limit);
            }
            keep = n;
        }
    }
    // the chunks' totals
    for (int c = tid; c < A.chunks; c += kThreads) totals[c] = fits && q.mode != kTopK ? A.totals[(int64_t)row * A.chunks + c] : 0;
    __syncthreads();
    if (!fits) {
        for (int c = tid >> 6; c < A.chunks; c += kWaves) {
            double t = 0;   // of 16 whole numbers up to 2^40: exact
            each_token(r, c, [&](float v, unsigned i) {
                if (!(v > -INFINITY) || !kept(last, key_of(v), i)) return;
                const float e = q.share(v);
                if (e >= q.min_p) t += (double)truncf(e * 0x1p40f);
            });
            const unsigned long long total = wave_sum((unsigned long long)t);
            if ((tid & 63) == 0) totals[c] = total;
        }
    } else {
        for (int i = tid; i < keep; i += kThreads) {   // the list's kept tokens (none without a cut)
            const float e = q.share(of_key(~(unsigned)(list[i] >> 32)));
            if (kept(last, list[i]) && e >= q.min_p) atomicAdd(&totals[((unsigned)list[i] + r.skew) / kChunk], weight(e));
        }
    }
    __syncthreads();
    const int per = (A.chunks + kThreads - 1) / kThreads, c0 = min(tid * per, A.chunks), c1 = min(c0 + per, A.chunks);
    unsigned long long sum = 0;
    for (int c = c0; c < c1; c++) sum += totals[c];
    const unsigned long long total = block_sum(red, sum);
    const unsigned long long target = min((unsigned long long)fmax(u * (double)total, 0.0), total - 1);
    unsigned long long run = block_scan(red, sum) - sum;
    if (run <= target && target < run + sum) {
        int c = c0;
        while (run + totals[c] <= target) run += totals[c++];
        found[0] = c;
        found[1] = target - run;
    }
    __syncthreads();
    // the pick in its chunk: neighbouring tokens for each thread
    constexpr int PICK = kChunk / kThreads;
    const int first = (int)found[0] * kChunk + tid * PICK - r.skew;
    const unsigned long long left = found[1];
    float v[PICK];
#pragma unroll
    for (int j = 0; j < PICK; j++) v[j] = first + j >= 0 && first + j < A.vocab ? x[first + j] : -INFINITY;
    float* const vs = (float*)list;
#pragma unroll
    for (int j = 0; j < PICK; j++) vs[tid * PICK + j] = v[j];   // (a thread's own: a rolled loop over registers)
    sum = 0;
#pragma unroll 1
    for (int j = tid * PICK; j < tid * PICK + PICK; j++) {
        unsigned long long w = 0;
        if (vs[j] > -INFINITY && kept(last, key_of(vs[j]), (unsigned)(first + j - tid * PICK))) {
            const float e = q.share(vs[j]);
            if (e >= q.min_p) w = weight(e);
        }
        ws[j] = w;
        sum += w;
    }
    run = block_scan(red, sum) - sum;
    if (run <= left && left < run + sum) {
        int j = tid * PICK;
        while (run + ws[j] <= left) run += ws[j++];
        A.ids[row] = first + j - tid * PICK;
        if (A.prob) A.prob[row] = (float)((double)ws[j] / (double)total);
    }
}

}  // namespace

int launch_sample(smx_ctx* c, const float* logits, size_t rows, size_t vocab, size_t ld, const smx_sample_params* p, const float* u, int32_t* ids, float* prob) {
    SampleArgs A{};
    A.logits = logits; A.ld = (int64_t)ld; A.rows = (int)rows; A.vocab = (int)vocab;
    // (rows that do not all start at 16-byte boundaries may lie up to 3 tokens into their first chunk)
    const size_t skew = ld % 4 == 0 ? ((uintptr_t)logits >> 2) & 3 : 3;
    A.chunks = (int)((vocab + skew + kChunk - 1) / kChunk);
    if (p) { A.temperature = p->temperature; A.top_k = p->top_k; A.top_p = p->top_p; A.min_p = p->min_p; }
    A.u = u; A.ids = ids; A.prob = prob;
    // Parts of a row: workgroups of 8 waves, of at least one chunk a wave.  More of them balance rows that ask for different work (greedy
    // ones end at once), but each adds a histogram to its row's.  512 / 1024 / 2048 in all, us of the four launches, rows that ask for
    // different things and, behind them, alike: 20 x 262144 41.6 / 41.5 / 41.8 and 43 / 43 / 43, 40 x 262144 57 / 57 / 58 and
    // 56 / 63 / 62, 64 x 262144 70 / 66 / 73 and 70 / 67 / 78, 256 x 262144 203 / 185 / 170 and 198 / 180 / 182,
    // 1000 x 50000 226 / 167 / 159 and 215 / 162 / 175.
    const size_t all = rows * (size_t)A.chunks, waves = kPartWaves, most = ((size_t)A.chunks + waves - 1) / waves;
    const size_t want = all >= 2048 * 32 ? 2048 : all >= 1024 * 12 ? 1024 : 512;
    size_t parts = std::max<size_t>(1, std::min(most, (want + rows - 1) / rows));
    // whole rounds of the waves
    A.part_chunks = (int)std::max<size_t>(waves, ((A.chunks + parts - 1) / parts + waves / 2) / waves * waves);
    A.parts = (A.chunks + A.part_chunks - 1) / A.part_chunks;
    // workspace of up to kRowsAtOnce rows (the launches of a larger call follow one another)
    constexpr size_t kRowsAtOnce = 4096;
    const size_t group = std::min(rows, kRowsAtOnce);
    const size_t per_row = (size_t)kBins * 8 + (size_t)A.chunks * 8 + (size_t)kList * 8 + (size_t)A.parts * 8 + sizeof(RowCut);
    int rc;
    if ((rc = ensure(c, c->work, group * per_row + 64)) != SMX_OK) return rc;
    A.hist = (unsigned long long*)c->work.p;
    A.totals = A.hist + group * kBins;
    A.list = A.totals + group * A.chunks;
    A.best = A.list + group * kList;
    A.cuts = (RowCut*)(A.best + group * A.parts);
    // Without top_k and top_p arrays no row has a cut: no histogram.
    const bool cuts = A.top_k || A.top_p;
    const size_t lds = (2 * (size_t)kList + std::max(A.chunks, kSteps)) * 8;
    if ((rc = set_dyn_lds(c, sample_pick_kernel, lds)) != SMX_OK) return rc;
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
        hipLaunchKernelGGL(sample_best_kernel, grid, dim3(kPartThreads), 0, c->stream, G);
        if (cuts) hipLaunchKernelGGL(sample_hist_kernel, grid, dim3(kPartThreads), 0, c->stream, G);
        hipLaunchKernelGGL(sample_gather_kernel, grid, dim3(kPartThreads), 0, c->stream, G);
        hipLaunchKernelGGL(sample_pick_kernel, dim3((unsigned)n), dim3(kThreads), lds, c->stream, G);
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

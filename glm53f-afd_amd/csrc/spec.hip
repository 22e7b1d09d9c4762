// The two ends of a speculative round (gfx950): softmax rows of the LM head's logits, and the verification of drafted
// tokens. Both are bound by the rows of the vocabulary that they read; a row is cut into segments, a workgroup each, so
// that one row alone reaches many CUs, and a second launch joins the segments. A thread takes eight or sixteen entries of its
// segment and requests them all before it looks at the first.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ext/glm53f_spec.h"

namespace spec {
namespace {

constexpr int kInvalid = 1;                       // hipErrorInvalidValue
constexpr int THREADS = 256, WAVES = THREADS / 64;
constexpr int kMostVocab = 1 << 30;

typedef long long ll;

// Vectors at any address that their elements may have: global memory takes 128 bits from there.
typedef float f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4), aligned(2)));

// N consecutive entries of a row as f32, `fill` from entry `left` on.
template <int N>
__device__ __forceinline__ void load(const float* p, int left, float fill, float (&x)[N]) {
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(p + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[i + e] = v[e];
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? p[i] : fill;
    }
}
template <int N>
__device__ __forceinline__ void load(const uint16_t* p, int left, float fill, float (&x)[N]) {
    if (left >= N) {
#pragma unroll
        for (int i = 0; i < N; i += 8) {
            const u32x4 v = *reinterpret_cast<const u32x4*>(p + i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[i + 2 * e] = __uint_as_float(v[e] << 16);
                x[i + 2 * e + 1] = __uint_as_float(v[e] & 0xffff0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = i < left ? __uint_as_float((uint32_t)p[i] << 16) : fill;
    }
}

// ---------------------------------------------------------------------------------------------------- probabilities

// A segment's greatest logit and where it first stands, and the sum of exp((x - greatest) / T) over it.
struct Part {
    float top, sum;
    int at, pad;
};

constexpr float kNone = -__builtin_inff();

__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

__device__ __forceinline__ float rate_of(const float* temperature, int r) {
    const float t = temperature ? temperature[r] : 1.0f;
    if (!(t > 0.0f)) return 0.0f;                 // the greatest logit alone
    // finite, so that 0 times it is 0; above 0, since 0 stands for the case above (an infinite temperature: all alike)
    return fmaxf(fminf(1.0f / t, 3.0e38f), 1.0e-45f);
}

// exp((x - top) * rate), 0 for -inf (also where nothing else is there and top is -inf).
__device__ __forceinline__ float share(float x, float top, float rate) { return x == kNone ? 0.0f : expf((x - top) * rate); }

__device__ __forceinline__ void wave_top(float& top, int& at) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        const float x = __shfl_xor(top, m, 64);
        const int i = __shfl_xor(at, m, 64);
        if (before(x, i, top, at)) top = x, at = i;
    }
}
__device__ __forceinline__ float wave_sum(float x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
}

// Groups of four (f32) or eight (bf16) entries go around the threads, so that a wave's access is contiguous.
template <typename L> constexpr int kGroup = 16 / sizeof(L);

// OWN: entries per thread, THREADS times as many per segment.
template <typename L, int OWN>
__global__ void __launch_bounds__(THREADS) probs_parts_kernel(int vocab, const L* logits, ll ldl, const float* temperature,
                                                              Part* parts) {
    constexpr int G = kGroup<L>, SEG = THREADS * OWN;
    const int r = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const L* row = logits + r * ldl;
    float x[OWN / G][G];
#pragma unroll
    for (int j = 0; j < OWN / G; ++j) {
        const int i = seg * SEG + (j * THREADS + t) * G;
        load<G>(row + i, vocab - i, kNone, x[j]);
    }
    const float rate = rate_of(temperature, r);
    float top = kNone;
    int at = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < OWN / G; ++j)
#pragma unroll
        for (int e = 0; e < G; ++e)
            if (x[j][e] > top) top = x[j][e], at = seg * SEG + (j * THREADS + t) * G + e;
    __shared__ float tops[WAVES], sums[WAVES];
    __shared__ int ats[WAVES];
    wave_top(top, at);
    if ((t & 63) == 0) tops[t >> 6] = top, ats[t >> 6] = at;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        if (before(tops[w], ats[w], top, at)) top = tops[w], at = ats[w];
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < OWN / G; ++j)
#pragma unroll
        for (int e = 0; e < G; ++e) sum += share(x[j][e], top, rate);
    sum = wave_sum(sum);
    if ((t & 63) == 0) sums[t >> 6] = sum;
    __syncthreads();
    if (t == 0) parts[(ll)r * gridDim.x + seg] = {top, (sums[0] + sums[1]) + (sums[2] + sums[3]), at, 0};
}

// The probabilities go past the caches (nontemporal), which keep the logits that the first pass has read: 384 rows of 151,936 f32
// 114 us against 140.
template <typename L, int OWN>
__global__ void __launch_bounds__(THREADS) probs_write_kernel(int vocab, const L* logits, ll ldl, const float* temperature,
                                                              float* probs, ll ldp, const Part* parts) {
    constexpr int G = kGroup<L>, SEG = THREADS * OWN;
    const int r = blockIdx.y, seg = blockIdx.x, segs = gridDim.x, t = threadIdx.x, lane = t & 63;
    const L* row = logits + r * ldl;
    float x[OWN / G][G];
#pragma unroll
    for (int j = 0; j < OWN / G; ++j) {
        const int i = seg * SEG + (j * THREADS + t) * G;
        load<G>(row + i, vocab - i, kNone, x[j]);
    }
    const float rate = rate_of(temperature, r);
    const Part* p = parts + (ll)r * segs;
    float top = kNone;
    int at = 0x7fffffff;
    for (int i = lane; i < segs; i += 64)         // every wave for itself
        if (before(p[i].top, p[i].at, top, at)) top = p[i].top, at = p[i].at;
    wave_top(top, at);
    float* dst = probs + r * ldp;
    float by = 0.0f;
    if (rate != 0.0f) {
        float sum = 0.0f;
        for (int i = lane; i < segs; i += 64) sum += share(p[i].top, top, rate) * p[i].sum;
        sum = wave_sum(sum);
        by = sum == 0.0f ? 0.0f : 1.0f / sum;
    }
#pragma unroll
    for (int j = 0; j < OWN / G; ++j) {
        const int i = seg * SEG + (j * THREADS + t) * G;
        float y[G];
#pragma unroll
        for (int e = 0; e < G; ++e)
            y[e] = rate != 0.0f ? share(x[j][e], top, rate) * by : i + e == at && top > kNone ? 1.0f : 0.0f;
        if (vocab - i >= G) {
#pragma unroll
            for (int e = 0; e < G; e += 4)
                __builtin_nontemporal_store(f32x4{y[e], y[e + 1], y[e + 2], y[e + 3]}, reinterpret_cast<f32x4*>(dst + i + e));
        } else {
#pragma unroll
            for (int e = 0; e < G; ++e)
                if (i + e < vocab) dst[i + e] = y[e];
        }
    }
}

// ---------------------------------------------------------------------------------------------------- verification

// Two launches: sums of segments and every request's outcome, then one workgroup per request that finds the token. 64 windows of up
// to nine rows over 151,936 entries: 18.6 and 5.3 us (78 MB: 4.2 TB/s in the first), one window 3.9 and 4.7 (launches and chains).
// Eight entries per thread: what a round waits for is the chain of loads (the windows, the tokens, their probabilities, the rows'
// weights), so the rows are spread widely (one window 8.8 us, with sixteen 10.1; 64 windows 23.7 and 25.4).
constexpr int OWN = 8, SEG = THREADS * OWN;

__device__ __forceinline__ double weight(float p) { return p > 0.0f && p < __builtin_inff() ? (double)p : 0.0; }

struct Accept {
    int vocab;
    const int32_t* cu_rows;
    const int32_t* tokens;
    const float* target;
    ll p_stride;
    const float* draft;
    ll q_stride;
    const float* uniform;
};

// Request b's outcome: `kept` rows, and whether the row behind them was rejected. Every wave computes it, 64 drafted rows
// at a time.
struct Outcome {
    int kept;
    bool rejected;
};

__device__ __forceinline__ Outcome outcome(const Accept& a, ll first, int n) {
    if (n <= 0) return {0, false};
    const int lane = threadIdx.x & 63;
    for (int i0 = 1; i0 < n; i0 += 64) {
        const int i = i0 + lane;
        bool yes = true;
        if (i < n) {
            const ll r = first + i;
            const int x = a.tokens[r];
            yes = x >= 0 && x < a.vocab &&
                  (double)a.uniform[r] * (a.draft ? weight(a.draft[r * a.q_stride + x]) : 1.0) <
                      weight(a.target[(r - 1) * a.p_stride + x]);
        }
        const unsigned long long no = __ballot(!yes);
        if (no) return {i0 + __builtin_ctzll(no), true};
    }
    return {n, false};
}

// What the next token is drawn from: p of the last kept row, less q where a draft was rejected behind it.
struct Weights {
    const float* p;
    const float* q;                               // NULL: none
    int without;                                  // a certain draft's token, -1: none

    // The weights of N entries from i on, 0 behind the vocabulary.
    template <int N>
    __device__ __forceinline__ void get(int i, int vocab, double (&w)[N]) const {
        float x[N], y[N];
        load<N>(p + i, vocab - i, 0.0f, x);
        if (q) load<N>(q + i, vocab - i, 0.0f, y);
#pragma unroll
        for (int e = 0; e < N; ++e) {
            w[e] = weight(x[e]);
            if (q) w[e] = fmax(w[e] - weight(y[e]), 0.0);
            if (i + e == without) w[e] = 0.0;
        }
    }
};

__device__ __forceinline__ Weights weights(const Accept& a, ll first, Outcome o) {
    const ll last = first + o.kept - 1;
    Weights w{a.target + last * a.p_stride, nullptr, -1};
    if (o.rejected) {
        if (a.draft) w.q = a.draft + (last + 1) * a.q_stride;
        else w.without = a.tokens[last + 1];
    }
    return w;
}

__device__ __forceinline__ double wave_sum(double x) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
}

// Each segment's sum of weights, and with the first segment the request's outcome.
__global__ void __launch_bounds__(THREADS) accept_parts_kernel(const Accept a, double* parts, int32_t* outcomes) {
    const int b = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const ll first = a.cu_rows[b];
    const Outcome o = outcome(a, first, a.cu_rows[b + 1] - (int)first);
    __shared__ double sums[WAVES];
    double sum = 0.0;
    if (o.kept > 0) {
        const Weights w = weights(a, first, o);
        double x[OWN / 4][4];
#pragma unroll
        for (int j = 0; j < OWN / 4; ++j) w.get<4>(seg * SEG + (j * THREADS + t) * 4, a.vocab, x[j]);
#pragma unroll
        for (int j = 0; j < OWN / 4; ++j) sum += (x[j][0] + x[j][1]) + (x[j][2] + x[j][3]);
    }
    sum = wave_sum(sum);
    if ((t & 63) == 0) sums[t >> 6] = sum;
    __syncthreads();
    if (t == 0) {
        parts[(ll)b * gridDim.x + seg] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
        if (seg == 0) outcomes[b] = o.rejected ? -o.kept : o.kept;
    }
}

struct Scratch {
    double sums[WAVES];
    int over[WAVES], some[WAVES];
};

// The sum over the threads before this one, and over all of them. Every thread calls it.
__device__ __forceinline__ double scan(double own, double& all, Scratch& s) {
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    double x = own;
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) {
        const double y = __shfl_up(x, m, 64);
        if (lane >= m) x += y;
    }
    __syncthreads();
    if (lane == 63) s.sums[wave] = x;
    __syncthreads();
    all = 0.0;
    double ahead = 0.0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        if (w < wave) ahead += s.sums[w];
        all += s.sums[w];
    }
    const double y = __shfl_up(x, 1, 64);
    return ahead + (lane > 0 ? y : 0.0);
}

// The least `over` of all threads (0x7fffffff: none), or where there is none the greatest `some` (-1: none).
__device__ __forceinline__ int pick(int over, int some, Scratch& s) {
    const int t = threadIdx.x;
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        over = min(over, __shfl_xor(over, m, 64));
        some = max(some, __shfl_xor(some, m, 64));
    }
    __syncthreads();
    if ((t & 63) == 0) s.over[t >> 6] = over, s.some[t >> 6] = some;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) over = min(over, s.over[w]), some = max(some, s.some[w]);
    return over != 0x7fffffff ? over : some;
}

// The lowest entry of the segment from `lo` on whose weight brings `sum` over `edge`; where rounding leaves none, the last
// one with a weight. `sum` gets the segment's added.
__device__ __forceinline__ int crossing(const Weights& w, int lo, int vocab, double& sum, double edge, Scratch& s, bool& over_edge) {
    const int mine = lo + threadIdx.x * OWN;
    double x[OWN], own = 0.0, all;
    w.get<OWN>(mine, vocab, x);
#pragma unroll
    for (int e = 0; e < OWN; ++e) own += x[e];
    double run = sum + scan(own, all, s);
    int over = 0x7fffffff, some = -1;
#pragma unroll
    for (int e = 0; e < OWN; ++e) {
        run += x[e];
        if (x[e] > 0.0) some = mine + e;
        if (run > edge && over == 0x7fffffff && x[e] > 0.0) over = mine + e;
    }
    const int best = pick(over, some, s);
    sum += all;
    over_edge = sum > edge;
    return best;
}

__global__ void __launch_bounds__(THREADS) accept_pick_kernel(const Accept a, int segs, const double* parts,
                                                              const int32_t* outcomes, int32_t* keep, int32_t* next) {
    const int b = blockIdx.x, t = threadIdx.x;
    __shared__ Scratch s;
    const int code = outcomes[b];
    const Outcome o{code < 0 ? -code : code, code < 0};
    const ll first = a.cu_rows[b];
    int token = -1;
    if (o.kept > 0) {
        Weights w = weights(a, first, o);
        const double* p = parts + (ll)b * segs;
        const double u = a.uniform[first];
        // a run of consecutive segments per thread
        const int run = (segs + THREADS - 1) / THREADS, lo = min(t * run, segs), hi = min(lo + run, segs);
        double own = 0.0, all;
        for (int i = lo; i < hi; ++i) own += p[i];
        const double ahead = scan(own, all, s);
        bool done;
        if (all > 0.0) {
            const double edge = u * all;
            double sum = ahead;
            int over = 0x7fffffff, some = -1;
            for (int i = lo; i < hi; ++i) {
                sum += p[i];
                if (p[i] > 0.0) some = i;
                if (sum > edge && over == 0x7fffffff && p[i] > 0.0) over = i;
            }
            const int seg = pick(over, some, s);
            // the sum ahead of that segment, from the thread that has it
            __shared__ double start;
            if (seg >= lo && seg < hi) {
                double x = ahead;
                for (int i = lo; i < seg; ++i) x += p[i];
                start = x;
            }
            __syncthreads();
            double from = start;
            token = crossing(w, seg * SEG, a.vocab, from, edge, s, done);
        } else if (o.rejected) {
            // the draft covers the target everywhere: p itself, all of it here
            w.q = nullptr, w.without = -1;
            double whole = 0.0, sum = 0.0;
            for (int seg = 0; seg < segs; ++seg) (void)crossing(w, seg * SEG, a.vocab, whole, 0.0, s, done);
            const double edge = u * whole;
            done = false;
            for (int seg = 0; seg < segs && !done; ++seg) {
                const int x = crossing(w, seg * SEG, a.vocab, sum, edge, s, done);
                if (x >= 0) token = x;
            }
        }
    }
    if (t == 0) keep[b] = o.kept, next[b] = token;
}

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline ll segments(int vocab, int seg) { return ((ll)vocab + seg - 1) / seg; }

// Entries per thread of the probabilities' passes: eight where sixteen would leave CUs without two workgroups (one row of 151,936 bf16
// 7.8 us against 8.6), sixteen otherwise (384 rows f32 114 us against 130).
inline int entries(int rows, int vocab) { return rows * segments(vocab, 16 * THREADS) < 512 ? 8 : 16; }

// Both passes over a part of the rows at a time where the logits are more than the cache behind the L2 holds, so that the second
// pass finds there what the first has read.
constexpr ll kCached = 224LL << 20;

template <typename L, int OWN>
int32_t probs(int rows, int vocab, const void* logits, ll ldl, const float* temperature, float* out, ll ldp, Part* parts,
              hipStream_t stream) {
    const L* x = static_cast<const L*>(logits);
    const ll slabs = ((ll)rows * vocab * (ll)sizeof(L) + kCached - 1) / kCached;
    const int most = (int)((rows + slabs - 1) / slabs);
    for (int r = 0; r < rows; r += most) {
        const dim3 grid((unsigned)segments(vocab, THREADS * OWN), (unsigned)(rows - r < most ? rows - r : most));
        const float* t = temperature ? temperature + r : nullptr;
        probs_parts_kernel<L, OWN><<<grid, THREADS, 0, stream>>>(vocab, x + r * ldl, ldl, t, parts);
        probs_write_kernel<L, OWN><<<grid, THREADS, 0, stream>>>(vocab, x + r * ldl, ldl, t, out + r * ldp, ldp, parts);
    }
    return (int32_t)hipGetLastError();
}

}  // namespace
}  // namespace spec

extern "C" int64_t glm53f_spec_probs_workspace_bytes(int32_t rows, int32_t vocab) {
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab > spec::kMostVocab) return -1;
    // Fewer rows may be cut more finely: the most that any number up to `rows` needs, so that one workspace serves them all.
    const int64_t whole = spec::segments(vocab, 16 * spec::THREADS), halves = spec::segments(vocab, 8 * spec::THREADS);
    const int64_t few = 511 / whole < rows ? 511 / whole : rows;
    const int64_t fine = few * halves, coarse = few < rows ? rows * whole : 0;
    return (fine > coarse ? fine : coarse) * (int64_t)sizeof(spec::Part);
}

extern "C" int32_t glm53f_spec_probs(int32_t rows, int32_t vocab, const void* logits, int32_t logits_f32, int64_t ldl,
                                     const float* temperature, float* probs, int64_t ldp, void* workspace,
                                     int64_t workspace_bytes, ihipStream_t* stream) {
    using namespace spec;
    if (rows < 0 || rows > 65535 || vocab < 1 || vocab > kMostVocab || ldl < vocab || ldp < vocab) return kInvalid;
    if (rows == 0) return 0;
    if (!logits || !probs || !workspace || !aligned(logits, logits_f32 ? 4 : 2) || !aligned(probs, 4) ||
        !aligned(temperature, 4) || !aligned(workspace, 16) || workspace_bytes < glm53f_spec_probs_workspace_bytes(rows, vocab))
        return kInvalid;
    if (logits == probs && (!logits_f32 || ldl != ldp)) return kInvalid;
    Part* parts = static_cast<Part*>(workspace);
    auto* call = entries(rows, vocab) == 8 ? (logits_f32 ? &spec::probs<float, 8> : &spec::probs<uint16_t, 8>)
                                           : (logits_f32 ? &spec::probs<float, 16> : &spec::probs<uint16_t, 16>);
    return call(rows, vocab, logits, ldl, temperature, probs, ldp, parts, stream);
}

extern "C" int64_t glm53f_spec_accept_workspace_bytes(int32_t batch, int32_t vocab) {
    if (batch < 0 || batch > 65535 || vocab < 1 || vocab > spec::kMostVocab) return -1;
    return batch * (spec::segments(vocab, spec::SEG) * (int64_t)sizeof(double) + (int64_t)sizeof(int32_t));
}

extern "C" int32_t glm53f_spec_accept(int32_t batch, int32_t vocab, const int32_t* cu_rows, const int32_t* tokens,
                                      const float* target, int64_t p_stride, const float* draft, int64_t q_stride,
                                      const float* uniform, int32_t* keep, int32_t* next, void* workspace,
                                      int64_t workspace_bytes, ihipStream_t* stream) {
    using namespace spec;
    if (batch < 0 || batch > 65535 || vocab < 1 || vocab > kMostVocab || p_stride < vocab || (draft && q_stride < vocab)) return kInvalid;
    if (batch == 0) return 0;
    if (!cu_rows || !tokens || !target || !uniform || !keep || !next || !workspace || !aligned(cu_rows, 4) ||
        !aligned(tokens, 4) || !aligned(target, 4) || !aligned(draft, 4) || !aligned(uniform, 4) || !aligned(keep, 4) ||
        !aligned(next, 4) || !aligned(workspace, 16) || workspace_bytes < glm53f_spec_accept_workspace_bytes(batch, vocab))
        return kInvalid;
    const int segs = (int)segments(vocab, SEG);
    double* parts = static_cast<double*>(workspace);
    int32_t* outcomes = reinterpret_cast<int32_t*>(parts + (ll)batch * segs);
    const Accept a{vocab, cu_rows, tokens, target, p_stride, draft, q_stride, uniform};
    accept_parts_kernel<<<dim3((unsigned)segs, (unsigned)batch), THREADS, 0, stream>>>(a, parts, outcomes);
    accept_pick_kernel<<<dim3((unsigned)batch), THREADS, 0, stream>>>(a, segs, parts, outcomes, keep, next);
    return (int32_t)hipGetLastError();
}

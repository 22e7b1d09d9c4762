// The two ends of a speculative round (gfx950): softmax rows of the LM head's logits, and the verification of drafted
// tokens. Both are bound by the rows of the vocabulary that they read; a row is cut into segments, a workgroup each, so
// that one row alone reaches many CUs, and a second launch joins the segments.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ext/glm53f_spec.h"

namespace spec {
namespace {

constexpr int kInvalid = 1;                       // hipErrorInvalidValue
constexpr int THREADS = 256;
constexpr int SEG = 4096;                         // entries of a row per workgroup

typedef long long ll;

__device__ __forceinline__ float widen(uint16_t b) { return __uint_as_float((uint32_t)b << 16); }
__device__ __forceinline__ float get(const float* p, ll i) { return p[i]; }
__device__ __forceinline__ float get(const uint16_t* p, ll i) { return widen(p[i]); }

// A segment's greatest logit and where it first stands, and the sum of exp((x - greatest) / T) over it.
struct Part {
    float top, sum;
    int at, pad;
};

__device__ __forceinline__ bool before(float x, int i, float y, int j) { return x > y || (x == y && i < j); }

__device__ __forceinline__ float rate_of(const float* temperature, int r) {
    const float t = temperature ? temperature[r] : 1.0f;
    if (!(t > 0.0f)) return 0.0f;                 // the greatest logit alone
    return fminf(1.0f / t, 3.0e38f);              // finite, so that 0 times it is 0
}

// exp((x - top) * rate), 0 for -inf (also where nothing else is there and top is -inf).
__device__ __forceinline__ float share(float x, float top, float rate) {
    return x == -__builtin_inff() ? 0.0f : expf((x - top) * rate);
}

template <typename L>
__global__ void __launch_bounds__(THREADS) probs_parts_kernel(int vocab, const L* logits, ll ldl, const float* temperature,
                                                              Part* parts) {
    const int r = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const L* row = logits + r * ldl;
    const int lo = seg * SEG, hi = min(vocab - lo, SEG) + lo;
    const float rate = rate_of(temperature, r);
    float top = -__builtin_inff();
    int at = 0x7fffffff;
    for (int i = lo + t; i < hi; i += THREADS) {
        const float x = get(row, i);
        if (before(x, i, top, at)) top = x, at = i;
    }
    __shared__ float tops[4], sums[4];
    __shared__ int ats[4];
    for (int m = 32; m >= 1; m >>= 1) {
        const float x = __shfl_xor(top, m, 64);
        const int i = __shfl_xor(at, m, 64);
        if (before(x, i, top, at)) top = x, at = i;
    }
    if ((t & 63) == 0) tops[t >> 6] = top, ats[t >> 6] = at;
    __syncthreads();
    for (int w = 0; w < 4; ++w)
        if (before(tops[w], ats[w], top, at)) top = tops[w], at = ats[w];
    float sum = 0.0f;
    for (int i = lo + t; i < hi; i += THREADS) sum += share(get(row, i), top, rate);
    for (int m = 32; m >= 1; m >>= 1) sum += __shfl_xor(sum, m, 64);
    if ((t & 63) == 0) sums[t >> 6] = sum;
    __syncthreads();
    if (t == 0) parts[(ll)r * gridDim.x + seg] = {top, (sums[0] + sums[1]) + (sums[2] + sums[3]), at, 0};
}

template <typename L>
__global__ void __launch_bounds__(THREADS) probs_write_kernel(int vocab, const L* logits, ll ldl, const float* temperature,
                                                              float* probs, ll ldp, const Part* parts) {
    const int r = blockIdx.y, seg = blockIdx.x, segs = gridDim.x, t = threadIdx.x;
    const Part* p = parts + (ll)r * segs;
    float top = -__builtin_inff();
    int at = 0x7fffffff;
    for (int i = 0; i < segs; ++i)
        if (before(p[i].top, p[i].at, top, at)) top = p[i].top, at = p[i].at;
    const float rate = rate_of(temperature, r);
    const int lo = seg * SEG, hi = min(vocab - lo, SEG) + lo;
    float* dst = probs + r * ldp;
    if (rate == 0.0f) {
        for (int i = lo + t; i < hi; i += THREADS) dst[i] = i == at && top > -__builtin_inff() ? 1.0f : 0.0f;
        return;
    }
    float sum = 0.0f;
    for (int i = 0; i < segs; ++i) sum += share(p[i].top, top, rate) * p[i].sum;
    const float by = sum == 0.0f ? 0.0f : 1.0f / sum;
    const L* row = logits + r * ldl;
    for (int i = lo + t; i < hi; i += THREADS) dst[i] = share(get(row, i), top, rate) * by;
}

// ---------------------------------------------------------------------------------------------------------------

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

// Request b's outcome: `kept` rows, the last of them global row `last`, and whether row last + 1 was rejected. Every
// thread of the workgroup computes it (a wave at a time looks at 64 drafted rows).
struct Outcome {
    ll last;
    int kept;
    bool rejected;
};

__device__ __forceinline__ Outcome outcome(const Accept& a, int b) {
    const ll first = a.cu_rows[b];
    const int n = a.cu_rows[b + 1] - (int)first;
    if (n <= 0) return {first, 0, false};
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
        if (no) {
            const int kept = i0 + __builtin_ctzll(no);
            return {first + kept - 1, kept, true};
        }
    }
    return {first + n - 1, n, false};
}

// What the next token is drawn from: p of the last kept row, less q where a draft was rejected behind it.
struct Weights {
    const float* p;
    const float* q;                               // NULL: none
    int without;                                  // a certain draft's token, -1: none
    __device__ __forceinline__ double at(int i) const {
        double w = weight(p[i]);
        if (q) w = fmax(w - weight(q[i]), 0.0);
        return i == without ? 0.0 : w;
    }
};

__device__ __forceinline__ Weights weights(const Accept& a, const Outcome& o) {
    Weights w{a.target + o.last * a.p_stride, nullptr, -1};
    if (o.rejected) {
        if (a.draft) w.q = a.draft + (o.last + 1) * a.q_stride;
        else w.without = a.tokens[o.last + 1];
    }
    return w;
}

__device__ __forceinline__ double wave_sum(double x) {
    for (int m = 32; m >= 1; m >>= 1) x += __shfl_xor(x, m, 64);
    return x;
}

__global__ void __launch_bounds__(THREADS) accept_parts_kernel(const Accept a, double* parts) {
    const int b = blockIdx.y, seg = blockIdx.x, t = threadIdx.x;
    const Outcome o = outcome(a, b);
    __shared__ double sums[4];
    double sum = 0.0;
    if (o.kept > 0) {
        const Weights w = weights(a, o);
        const int lo = seg * SEG, hi = min(a.vocab - lo, SEG) + lo;
        for (int i = lo + t; i < hi; i += THREADS) sum += w.at(i);
    }
    sum = wave_sum(sum);
    if ((t & 63) == 0) sums[t >> 6] = sum;
    __syncthreads();
    if (t == 0) parts[(ll)b * gridDim.x + seg] = (sums[0] + sums[1]) + (sums[2] + sums[3]);
}

// The lowest entry of [lo, hi) whose weight brings `sum` over `edge`, or the last entry with a weight where rounding
// leaves none. Each thread takes a run of consecutive entries; the threads' sums meet in LDS.
__device__ int crossing(const Weights& w, int lo, int hi, double sum, double edge, double* sums, int* found) {
    const int t = threadIdx.x, run = (hi - lo + THREADS - 1) / THREADS;
    const int mine = min(lo + t * run, hi), end = min(mine + run, hi);
    double own = 0.0;
    int some = -1;
    for (int i = mine; i < end; ++i) {
        const double x = w.at(i);
        own += x;
        if (x > 0.0) some = i;
    }
    sums[t] = own;
    if (t == 0) found[0] = 0x7fffffff, found[1] = -1;
    __syncthreads();
    for (int i = 0; i < t; ++i) sum += sums[i];
    if (some >= 0) atomicMax(&found[1], some);
    for (int i = mine; i < end; ++i) {
        sum += w.at(i);
        if (sum > edge) {
            atomicMin(&found[0], i);
            break;
        }
    }
    __syncthreads();
    return found[0] != 0x7fffffff ? found[0] : found[1];
}

__global__ void __launch_bounds__(THREADS) accept_pick_kernel(const Accept a, int segs, const double* parts, int32_t* keep,
                                                              int32_t* next) {
    const int b = blockIdx.x, t = threadIdx.x;
    const Outcome o = outcome(a, b);
    __shared__ double sums[THREADS];
    __shared__ int found[2];
    int token = -1;
    if (o.kept > 0) {
        Weights w = weights(a, o);
        const double* p = parts + (ll)b * segs;
        const double u = a.uniform[a.cu_rows[b]];
        double all = 0.0;
        for (int i = 0; i < segs; ++i) all += p[i];
        if (all > 0.0) {
            const double edge = u * all;
            double sum = 0.0, start = 0.0;
            int seg = -1;
            for (int i = 0; i < segs; ++i) {
                if (p[i] > 0.0) seg = i, start = sum;
                sum += p[i];
                if (sum > edge) break;
            }
            token = crossing(w, seg * SEG, min(a.vocab - seg * SEG, SEG) + seg * SEG, start, edge, sums, found);
        } else if (o.rejected) {
            // the draft covers the target everywhere: p itself
            w.q = nullptr, w.without = -1;
            double own = 0.0;
            for (int i = t; i < a.vocab; i += THREADS) own += w.at(i);
            sums[t] = own;
            __syncthreads();
            for (int i = 0; i < THREADS; ++i) all += sums[i];
            __syncthreads();
            if (all > 0.0) token = crossing(w, 0, a.vocab, 0.0, u * all, sums, found);
        }
    }
    if (t == 0) keep[b] = o.kept, next[b] = token;
}

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline ll segments(int vocab) { return ((ll)vocab + SEG - 1) / SEG; }

}  // namespace
}  // namespace spec

extern "C" int64_t glm53f_spec_probs_workspace_bytes(int32_t rows, int32_t vocab) {
    if (rows < 0 || vocab < 1) return -1;
    return rows * spec::segments(vocab) * (int64_t)sizeof(spec::Part);
}

extern "C" int32_t glm53f_spec_probs(int32_t rows, int32_t vocab, const void* logits, int32_t logits_f32, int64_t ldl,
                                     const float* temperature, float* probs, int64_t ldp, void* workspace,
                                     int64_t workspace_bytes, ihipStream_t* stream) {
    using namespace spec;
    if (rows < 0 || rows > 65535 || vocab < 1 || ldl < vocab || ldp < vocab) return kInvalid;
    if (rows == 0) return 0;
    if (!logits || !probs || !workspace || !aligned(logits, logits_f32 ? 4 : 2) || !aligned(probs, 4) ||
        !aligned(temperature, 4) || !aligned(workspace, 16) || workspace_bytes < glm53f_spec_probs_workspace_bytes(rows, vocab))
        return kInvalid;
    if (logits == probs && (!logits_f32 || ldl != ldp)) return kInvalid;
    Part* parts = static_cast<Part*>(workspace);
    const dim3 grid((unsigned)segments(vocab), (unsigned)rows);
    if (logits_f32) {
        probs_parts_kernel<float><<<grid, THREADS, 0, stream>>>(vocab, static_cast<const float*>(logits), ldl, temperature, parts);
        probs_write_kernel<float><<<grid, THREADS, 0, stream>>>(vocab, static_cast<const float*>(logits), ldl, temperature, probs, ldp, parts);
    } else {
        probs_parts_kernel<uint16_t><<<grid, THREADS, 0, stream>>>(vocab, static_cast<const uint16_t*>(logits), ldl, temperature, parts);
        probs_write_kernel<uint16_t><<<grid, THREADS, 0, stream>>>(vocab, static_cast<const uint16_t*>(logits), ldl, temperature, probs, ldp, parts);
    }
    return (int32_t)hipGetLastError();
}

extern "C" int64_t glm53f_spec_accept_workspace_bytes(int32_t batch, int32_t vocab) {
    if (batch < 0 || vocab < 1) return -1;
    return batch * spec::segments(vocab) * (int64_t)sizeof(double);
}

extern "C" int32_t glm53f_spec_accept(int32_t batch, int32_t vocab, const int32_t* cu_rows, const int32_t* tokens,
                                      const float* target, int64_t p_stride, const float* draft, int64_t q_stride,
                                      const float* uniform, int32_t* keep, int32_t* next, void* workspace,
                                      int64_t workspace_bytes, ihipStream_t* stream) {
    using namespace spec;
    if (batch < 0 || batch > 65535 || vocab < 1 || p_stride < vocab || (draft && q_stride < vocab)) return kInvalid;
    if (batch == 0) return 0;
    if (!cu_rows || !tokens || !target || !uniform || !keep || !next || !workspace || !aligned(cu_rows, 4) ||
        !aligned(tokens, 4) || !aligned(target, 4) || !aligned(draft, 4) || !aligned(uniform, 4) || !aligned(keep, 4) ||
        !aligned(next, 4) || !aligned(workspace, 16) || workspace_bytes < glm53f_spec_accept_workspace_bytes(batch, vocab))
        return kInvalid;
    double* parts = static_cast<double*>(workspace);
    const Accept a{vocab, cu_rows, tokens, target, p_stride, draft, q_stride, uniform};
    const int segs = (int)segments(vocab);
    accept_parts_kernel<<<dim3((unsigned)segs, (unsigned)batch), THREADS, 0, stream>>>(a, parts);
    accept_pick_kernel<<<dim3((unsigned)batch), THREADS, 0, stream>>>(a, segs, parts, keep, next);
    return (int32_t)hipGetLastError();
}

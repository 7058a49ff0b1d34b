// What is kept of a row of logits x while it goes by:
//
//   m = max x,   s = sum e^(x - m) - 1,   t = sum (x - m) e^(x - m)
//
//   log probability of x_k:  (x_k - m) - log(1 + s)        entropy:  log(1 + s) - t / (1 + s)        of the most likely token:  - log(1 + s)
//
// The largest logit's own term, 1, is left out of s: where that token is nearly certain the others' sum keeps its digits (with them the 1 left five of seven,
// and log probabilities near zero were off by 1e-5 of themselves).  t is taken about the maximum for the same reason: sum x p would lose the digits that a
// common offset takes.  A logit of minus infinity (a masked token) adds nothing.  m = -infinity: nothing seen yet.  Everything is fp32; a NaN, or plus
// infinity, ends up as a NaN in s or as m = infinity.
#pragma once

#include "common.cuh"

#define LP_LOG2E 1.4426950408889634f

__device__ __forceinline__ float lp_exp2(float x) {  // results below 2^-126 are zeros: nothing beside the largest term
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

struct LogitSums {
    float m, s, t;
    __device__ __forceinline__ void clear() { m = -INFINITY, s = 0.f, t = 0.f; }
    __device__ __forceinline__ void join(const LogitSums& o, bool first = true) {  // first: of two equal maxima this one is kept
        const bool mine = first ? m >= o.m : m > o.m;
        const float hm = mine ? m : o.m, hs = mine ? s : o.s, ht = mine ? t : o.t, lm = mine ? o.m : m, ls = mine ? o.s : s, lt = mine ? o.t : t;
        const float d = lm - hm, f = lm == -INFINITY ? 0.f : lp_exp2(d * LP_LOG2E), sum = 1.f + ls;
        m = hm;
        s = fmaf(sum, f, hs);
        t = ht + (f > 0.f ? fmaf(sum, d, lt) * f : 0.f);  // d may be minus infinity
    }
    __device__ __forceinline__ void join_lanes(int lanes) {  // of a warp's first `lanes` (a power of two): the same result, to the bit, on each
        for (int o = lanes >> 1; o > 0; o >>= 1) {
            const LogitSums other{__shfl_xor_sync(0xffffffffu, m, o), __shfl_xor_sync(0xffffffffu, s, o), __shfl_xor_sync(0xffffffffu, t, o)};
            join(other, (threadIdx.x & o) == 0);
        }
    }
    __device__ __forceinline__ bool bad() const { return isnan(s) || m == INFINITY; }
    __device__ __forceinline__ float norm() const { return m == -INFINITY ? 0.f : log1pf(s); }
};

// What is asked for and where the answers go; shared by the kernels that see logits and those that make them.
struct TokenScores {
    const void* tokens;
    float* logprob; float* entropy; float* best;
    int tokens_64;
    uint32_t* status;
};

// The token whose log probability a row asks for, -1: none.
__device__ __forceinline__ int lp_token(const TokenScores& a, int row, int vocab, bool report) {
    const int64_t k = a.tokens_64 ? reinterpret_cast<const int64_t*>(a.tokens)[row] : reinterpret_cast<const int*>(a.tokens)[row];
    if (k >= 0 && k < vocab) return (int)k;
    if (k != -1 && report) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
    return -1;
}

// `x`: the token's logit, meaningless where k < 0.
__device__ __forceinline__ void lp_store(const TokenScores& a, int row, const LogitSums& sums, bool bad, int k, float x) {
    const float norm = sums.norm(), none = __int_as_float(0x7fffffff);
    const bool empty = sums.m == -INFINITY;
    a.logprob[row] = bad || k < 0 ? none : x == -INFINITY ? -INFINITY : (x - sums.m) - norm;
    a.entropy[row] = bad ? none : empty ? 0.f : norm - sums.t / (1.f + sums.s);
    a.best[row] = bad ? none : empty ? -INFINITY : -norm;
    if (bad) raise_status(a.status, GLMB_STATUS_NONFINITE);
}

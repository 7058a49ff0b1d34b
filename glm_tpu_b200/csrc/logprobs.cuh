// What is kept of a row of logits x while it goes by:
//
//   m = max x,   s = sum e^(x - m),   t = sum (x - m) e^(x - m)
//
//   log probability of x_k:  (x_k - m) - log s        entropy:  log s - t / s        of the most likely token:  - log s
//
// t is taken about the running maximum: sum x p would lose the digits that a large common offset of the logits takes.  A logit of minus infinity
// (a masked token) adds nothing to s and t.  Everything is fp32.
#pragma once

#include "common.cuh"

#define LP_LOG2E 1.4426950408889634f

struct LogitSums {
    float m, s, t;
    __device__ __forceinline__ void clear() { m = -INFINITY, s = 0.f, t = 0.f; }
    // The sums about another, not smaller maximum.
    __device__ __forceinline__ void rebase(float next) {
        if (next == m) return;
        if (s != 0.f) {
            const float d = m - next, f = exp2f(d * LP_LOG2E);
            t = f > 0.f ? (t + s * d) * f : 0.f;
            s *= f;
        }
        m = next;
    }
    __device__ __forceinline__ void add(float x) {  // x <= m
        const float d = x - m, e = exp2f(d * LP_LOG2E);
        s += e;
        t += e > 0.f ? d * e : 0.f;
    }
    __device__ __forceinline__ void join(float om, float os, float ot) {
        const float next = fmaxf(m, om);
        LogitSums other{om, os, ot};
        rebase(next);
        other.rebase(next);
        s += other.s;
        t += other.t;
    }
};

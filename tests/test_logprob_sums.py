"""The sums that are kept of logits, joined across the lanes of a warp: the header compiled for the CPU, a thread a lane."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "glm_tpu_b200" / "csrc"

STAND_IN = r"""
#pragma once
#include <math.h>
#include <pthread.h>
#include <stdint.h>
#include <string.h>
#define __device__
#define __forceinline__ inline
enum : uint32_t { GLMB_STATUS_BAD_INDEX = 2, GLMB_STATUS_NONFINITE = 4 };
struct Index { unsigned x; };
static thread_local Index threadIdx;
static float passed[32];
static pthread_barrier_t meet;
static inline float __shfl_xor_sync(unsigned, float v, int o) {
    passed[threadIdx.x] = v;
    pthread_barrier_wait(&meet);
    const float other = passed[threadIdx.x ^ o];
    pthread_barrier_wait(&meet);
    return other;
}
static inline float __int_as_float(int i) { float f; memcpy(&f, &i, 4); return f; }
static inline void raise_status(uint32_t*, uint32_t) {}
"""

MAIN = r"""
#include <stdio.h>
#include <stdlib.h>
static LogitSums lanes[32];
static void* lane(void* at) {
    threadIdx.x = (unsigned)(size_t)at;
    lanes[threadIdx.x].join_lanes(32);
    return nullptr;
}
int main() {
    pthread_barrier_init(&meet, nullptr, 32);
    srand(1);
    auto uniform = [] { return rand() / (float)RAND_MAX; };
    for (int round = 0; round < 60; ++round) {
        double s = 0, t = 0, m = -INFINITY;
        LogitSums before[32];
        for (auto& l : lanes) {  // maxima that are often equal; some lanes have seen nothing
            l.clear();
            if (uniform() < 0.9f) l = LogitSums{(float)(rand() % (1 + round % 5)), uniform() * 7.f, -uniform() * 3.f};
            if (l.m > m) m = l.m;
        }
        memcpy(before, lanes, sizeof lanes);
        for (const auto& l : before)
            if (l.m > -INFINITY) s += (1 + (double)l.s) * exp(l.m - m), t += ((double)l.t + (1 + (double)l.s) * (l.m - m)) * exp(l.m - m);
        pthread_t id[32];
        for (size_t i = 0; i < 32; ++i) pthread_create(id + i, nullptr, lane, (void*)i);
        for (auto& i : id) pthread_join(i, nullptr);
        for (const auto& l : lanes)
            if (memcmp(&l, lanes, sizeof l)) return printf("round %d: lanes differ\n", round), 1;
        // five joins: a rounding of 2^-24 for each factor, product and sum, of terms of one sign
        const double bound = 5 * 6 * 5.97e-8;
        if (lanes[0].m != m || fabs(lanes[0].s - (s - 1)) > bound * s || fabs(lanes[0].t - t) > bound * (fabs(t) + 4 * s)) return printf("round %d: %g %g, not %g %g\n", round, lanes[0].s, lanes[0].t, s - 1, t), 1;
    }
    return 0;
}
"""


def test_lanes_join_to_the_same_bits(tmp_path):
    compiler = shutil.which("g++")
    if compiler is None:
        pytest.skip("no C++ compiler")
    source, exponentials = re.subn(r'asm\("ex2[^;]*;"[^;]*;', "y = exp2f(x);", (CSRC / "logprobs.cuh").read_text())
    assert exponentials == 1 or 'asm("ex2' not in source
    (tmp_path / "common.cuh").write_text(STAND_IN)
    (tmp_path / "logprobs.cuh").write_text(source)
    (tmp_path / "sums.cpp").write_text('#include "logprobs.cuh"\n' + MAIN)
    subprocess.run([compiler, "-std=c++17", "-O1", "-w", "-pthread", "sums.cpp", "-o", "sums"], cwd=tmp_path, check=True)
    ran = subprocess.run([tmp_path / "sums"], capture_output=True, text=True, timeout=120)
    assert ran.returncode == 0, ran.stdout

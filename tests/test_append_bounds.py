"""Which addresses ``append`` reads and writes: the kernel's source compiled for the CPU, every buffer ending at a page that cannot be touched.

The threads run one after another, so that a shuffle gives a thread its own value back: results mean nothing here, addresses do not depend on them."""

import re
import shutil
import subprocess
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "glm_tpu_b200" / "csrc"

STAND_IN = r"""
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>
#include <algorithm>
#include <vector_functions.h>
#include <vector_types.h>
#undef __device__
#undef __global__
#undef __forceinline__
#undef __grid_constant__
#undef __launch_bounds__
#define __device__
#define __global__
#define __forceinline__ inline
#define __grid_constant__
#define __launch_bounds__(...)
#define GLMB_API extern "C"
#define GLMB_PDL_PROLOGUE() do {} while (0)
#define GLMB_STATUS_BAD_INDEX 2u
using std::max;
using std::min;
#define cudaGetLastError() 0
struct bf16 { uint16_t bits; };
static uint3 threadIdx, blockIdx;
static dim3 gridDim;
static inline float of_bits(uint32_t u) { float f; memcpy(&f, &u, 4); return f; }
static inline float bf16_lo(uint32_t u) { return of_bits(u << 16); }
static inline float bf16_hi(uint32_t u) { return of_bits(u & 0xffff0000u); }
static inline float to_f32(bf16 v) { return of_bits((uint32_t)v.bits << 16); }
static inline uint32_t pack_bf16(float, float) { return 0; }
static inline uint4 ld_stream16(const void* p) { return *reinterpret_cast<const uint4*>(p); }
static inline float2 __fmul2_rn(float2 a, float2 b) { return make_float2(a.x * b.x, a.y * b.y); }
static inline float2 __ffma2_rn(float2 a, float2 b, float2 c) { return make_float2(a.x * b.x + c.x, a.y * b.y + c.y); }
static inline float __shfl_xor_sync(uint32_t, float v, int) { return v; }
static inline float rsqrtf(float x) { return 1.f / sqrtf(x); }
static inline void raise_status(uint32_t* status, uint32_t bits) { if (status) *status |= bits; }
static inline int ceil_div(int a, int b) { return (a + b - 1) / b; }
#define GLMB_LAUNCH(kernel, grid, block, smem, stream, a)                                                                          \
    do {                                                                                                                           \
        gridDim = grid;                                                                                                            \
        for (blockIdx.x = 0; blockIdx.x < gridDim.x; ++blockIdx.x)                                                                 \
            for (blockIdx.y = 0; blockIdx.y < gridDim.y; ++blockIdx.y)                                                             \
                for (threadIdx.x = 0; threadIdx.x < (block); ++threadIdx.x) kernel(a);                                             \
    } while (0)
"""

MAIN = r"""
#include <signal.h>
#include <stdio.h>
#include <stdlib.h>
#include <sys/mman.h>
#include <unistd.h>
static void outside(int) { static const char text[] = "an address out of range\n"; (void)!write(1, text, sizeof text - 1); _exit(1); }
template <typename T> static T* ends_at_a_guard(size_t count) {
    const size_t bytes = count * sizeof(T), page = 4096, whole = (bytes + page - 1) / page * page;
    char* at = (char*)mmap(nullptr, whole + 2 * page, PROT_READ | PROT_WRITE, MAP_PRIVATE | MAP_ANONYMOUS, -1, 0);
    mprotect(at, page, PROT_NONE), mprotect(at + page + whole, page, PROT_NONE);
    return (T*)(at + page + whole - bytes);
}
int main(int, char** arg) {
    signal(SIGSEGV, outside), signal(SIGBUS, outside);
    const int rows = atoi(arg[1]), H = atoi(arg[2]), G = atoi(arg[3]), dim = atoi(arg[4]), vdim = atoi(arg[5]), rot = atoi(arg[6]), pairs = atoi(arg[7]), norm = atoi(arg[8]), want_q = atoi(arg[9]);
    const int page = 8, pages = 1 + (rows - 1) / page;
    PagedAppendArgs a = {};
    PagedArgs& c = a.cache;
    c.k = ends_at_a_guard<bf16>((size_t)pages * page * G * dim), c.k_page = page * G * dim, c.k_slot = G * dim, c.k_head = dim;
    c.v = ends_at_a_guard<bf16>((size_t)pages * page * G * vdim), c.v_page = page * G * vdim, c.v_slot = G * vdim, c.v_head = vdim;
    int* table = ends_at_a_guard<int>(pages);
    for (int i = 0; i < pages; ++i) table[i] = i;
    c.table = table, c.table_stride = pages, c.seqs = 1, c.per_seq = pages, c.pages = pages, c.page = page, c.G = G, c.dim = dim, c.vdim = vdim;
    a.qkv_stride = H * dim + G * (dim + vdim), a.qkv = ends_at_a_guard<bf16>(rows * a.qkv_stride);
    if (norm) a.q_norm = ends_at_a_guard<bf16>(dim), a.k_norm = ends_at_a_guard<bf16>(dim);
    if (rot) a.rot = ends_at_a_guard<float2>((size_t)rows * rot / 2), a.rot_dims = rot, a.rot_rows = rows;
    a.pairs = pairs;
    int *positions = ends_at_a_guard<int>(rows), *slots = ends_at_a_guard<int>(rows);
    for (int r = 0; r < rows; ++r) positions[r] = slots[r] = r;
    a.positions = positions, a.slots = slots, a.row_seq = ends_at_a_guard<int>(rows);
    if (want_q) a.q = ends_at_a_guard<bf16>((size_t)rows * H * dim), a.q_stride = H * dim;
    a.rows = rows, a.H = H, a.eps = 1e-6f;
    uint32_t status = 0;
    a.status = &status;
    const int code = glmb_paged_append(&a, nullptr);
    printf("code %d status %u\n", code, status);
    return code || status ? 2 : 0;
}
"""


@pytest.fixture(scope="module")
def append_on_the_cpu(tmp_path_factory):
    compiler = shutil.which("g++")
    include = Path("/usr/local/cuda/include")
    if compiler is None or not (include / "vector_types.h").exists():
        pytest.skip("no C++ compiler, or no CUDA headers")
    at = tmp_path_factory.mktemp("append")
    source = (CSRC / "paged_append.cu").read_text()
    source, loads = re.subn(r'asm volatile\("ld\.global\.nc[^;]*;"[^;]*;', "v = *reinterpret_cast<const uint2*>(p);", source)
    assert loads == 1
    for name, text in (("common.cuh", STAND_IN), ("vec8.cuh", ""), ("paged.cuh", (CSRC / "paged.cuh").read_text()), ("append.cpp", source + MAIN)):
        (at / name).write_text(text)
    subprocess.run([compiler, "-std=c++17", "-O1", "-w", f"-I{include}", "append.cpp", "-o", "append"], cwd=at, check=True)
    return at / "append"


@pytest.mark.parametrize("pairs, want_q", [(0, 1), (1, 1), (0, 0)])
@pytest.mark.parametrize("rows, H, G, dim, vdim, rot", [
    (1, 1, 1, 16, 16, 2), (1, 1, 1, 16, 16, 16), (1, 4, 2, 32, 32, 2), (6, 4, 2, 32, 16, 30), (1, 3, 1, 48, 48, 20), (2, 9, 2, 64, 64, 34), (1, 5, 3, 80, 64, 40), (1, 5, 3, 80, 64, 20),
    (1, 1, 1, 128, 128, 90), (3, 70, 8, 128, 128, 128), (1, 1, 1, 256, 16, 34), (1, 33, 5, 256, 256, 0), (1, 17, 7, 16, 256, 6), (9, 2, 1, 96, 32, 46)])
def test_append_stays_inside_its_buffers(append_on_the_cpu, rows, H, G, dim, vdim, rot, pairs, want_q):
    for norm in (0, 1):
        ran = subprocess.run([append_on_the_cpu, *map(str, (rows, H, G, dim, vdim, rot, pairs, norm, want_q))], capture_output=True, text=True, timeout=60)
        assert ran.returncode == 0, (norm, ran.stdout)

// Log probability of given tokens, entropy and the most likely tokens of rows of logits (bf16 or fp32), one pass over them (logprobs.cuh: what is kept).
//
// A row belongs to a cluster of one to eight CTAs, each with a run of 16-byte vectors of it, which a warp brings in by bulk copies through a ring.  The
// maximum is a warp's: it moves about log(groups) times, on a branch.  (With one for each thread some lane was on that branch most of the time.)  The most
// likely tokens: every warp keeps a sorted list, one entry a lane, of 64-bit keys (the logit's order above the id's complement: ties go to the lowest id), and a
// logit enters only if it reaches a bound that n of the CTA's logits reach: the n-th largest of the threads' maxima so far, found anew after 1, 3, 9, 33 ..
// stages, at 3.3 thousand clocks.  Of 131,072 logits some 150 enter for n = 20, at 900 clocks.  (With a bound for each warp it was ten times as many.)  Sums and
// lists meet in the CTA, then in the cluster's first.  2,048 rows of 131,072 fp32 logits: 157 us without alternatives, 168 with one (6.4 TB/s, the bytes their
// bound), 197 with twenty; bf16 113, 145, 188.  333 rows of 65,521, five: 28.5 us, 18.7 without alternatives.  Where fewer of a CTA's logits than alternatives are
// above minus infinity the bound keeps none away, and every masked one is offered: the 2,048 rows with five tokens left and twenty alternatives take 5.7 ms.
//
// A row with a NaN or an infinite logit above zero has no probabilities: its numbers are NaN, its ids -1, and GLMB_STATUS_NONFINITE is raised.  A row
// of minus infinities alone (its mask leaves nothing): log probabilities minus infinity, entropy 0, the lowest ids.  A token of -1 asks for nothing
// (NaN); any other one outside the vocabulary is NaN too and raises GLMB_STATUS_BAD_INDEX.
#include <cooperative_groups.h>

#include "logprobs.cuh"
#include "tcgen05.cuh"

namespace cg = cooperative_groups;

#define LP_TOP 32      // most alternatives of a row: an entry a lane
#define LP_THREADS 256
#define LP_WARPS (LP_THREADS / 32)
#define LP_STAGE 1024  // vectors (16 KB) of a stage of the ring
#define LP_STAGES 3
#define LP_RING (LP_STAGES * LP_STAGE * 16)
#define LP_SM 233472   // bytes of shared memory of an SM
#define LP_PARTS 8     // CTAs of a row, at most

struct TokenLogprobsArgs {
    const void* logits; int64_t stride;
    TokenScores scores;
    int* top_ids; float* top_logprobs;
    int rows, vocab, top;
    int is_f32;
};

typedef unsigned long long u64;

template <typename T> struct LpVector;
template <> struct LpVector<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void get(const uint4& u, float (&x)[4]) {
        x[0] = __uint_as_float(u.x), x[1] = __uint_as_float(u.y), x[2] = __uint_as_float(u.z), x[3] = __uint_as_float(u.w);
    }
    static __device__ __forceinline__ float one(const float* p) { return *p; }
};
template <> struct LpVector<bf16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void get(const uint4& u, float (&x)[8]) {
        x[0] = bf16_lo(u.x), x[1] = bf16_hi(u.x), x[2] = bf16_lo(u.y), x[3] = bf16_hi(u.y);
        x[4] = bf16_lo(u.z), x[5] = bf16_hi(u.z), x[6] = bf16_lo(u.w), x[7] = bf16_hi(u.w);
    }
    static __device__ __forceinline__ float one(const bf16* p) { return __bfloat162float(*p); }
};

// Sums of a warp about a maximum that its lanes share: the warp's s and t are the sums of the lanes' (t in units of the binary logarithm).
struct WarpSums {
    float m, s, t;
    bool bad;
    // E more logits of every lane.  `top`: their maximum, or a NaN.  Returns nothing new: a new maximum is met about log(groups) times.
    template <int E>
    __device__ __forceinline__ void take(const float (&x)[E], float top, int lane) {
        if (!__all_sync(0xffffffffu, top <= m)) {
            bad |= isnan(top);
            const float next = fmaxf(m, warp_max(top));
            bool skip = false;
            if (next > m) {
                skip = lane == __ffs(__ballot_sync(0xffffffffu, top == next)) - 1;  // this lane's first such logit is the one whose term stays out of s
                if (m != -INFINITY) {
                    const float z = fmaxf((m - next) * LP_LOG2E, -1000.f), f = lp_exp2(z), sum = s + (skip ? 1.f : 0.f);
                    s = sum * f;
                    t = fmaf(sum, z, t) * f;
                }
                m = next;
            }
            if (m == -INFINITY) return;
#pragma unroll
            for (int i = 0; i < E; ++i) {
                const float d = x[i] - m, z = fmaxf(d * LP_LOG2E, -1000.f), e = lp_exp2(z);
                if (skip && d == 0.f) {
                    skip = false;
                } else {
                    s += e;
                    t = fmaf(z, e, t);
                }
            }
            return;
        }
        if (m == -INFINITY) return;
        if constexpr (E == 1) {
            const float z = fmaxf((x[0] - m) * LP_LOG2E, -1000.f), e = lp_exp2(z);
            s += e;
            t = fmaf(z, e, t);
        } else {
            const float2 minus_m = make_float2(-m, -m), log2e = make_float2(LP_LOG2E, LP_LOG2E);
            float2 s2 = make_float2(0.f, 0.f), t2 = s2;
#pragma unroll
            for (int i = 0; i < E; i += 2) {
                float2 z = __fmul2_rn(__fadd2_rn(make_float2(x[i], x[i + 1]), minus_m), log2e);
                z = make_float2(fmaxf(z.x, -1000.f), fmaxf(z.y, -1000.f));  // not minus infinity: its product with zero
                const float2 e = make_float2(lp_exp2(z.x), lp_exp2(z.y));
                s2 = __fadd2_rn(s2, e);
                t2 = __ffma2_rn(z, e, t2);
            }
            s += s2.x + s2.y;
            t += t2.x + t2.y;
        }
    }
    __device__ __forceinline__ LogitSums all() const { return LogitSums{m, warp_sum(s), warp_sum(t) * 0.6931471805599453f}; }
};
__device__ __forceinline__ float lp_max_nan(float a, float b) {  // a NaN if there is one
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// ---- sorted lists of keys, one entry a lane, largest first ------------------------------------------------
__device__ __forceinline__ void lp_insert(u64& list, u64 key, int lane) {
    const int at = __popc(__ballot_sync(0xffffffffu, list > key));
    const u64 above = __shfl_up_sync(0xffffffffu, list, 1);
    list = lane < at ? list : lane == at ? key : above;
}
// The 32 largest of two lists; `other`: the second one from its last entry to its first.
__device__ __forceinline__ void lp_merge(u64& list, u64 other, int lane) {
    list = list > other ? list : other;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const u64 with = __shfl_xor_sync(0xffffffffu, list, o);
        const bool larger = (lane & o) == 0;
        list = (list > with) == larger ? list : with;
    }
}
// All threads: `count` (a power of two, at most one for each warp) lists become lists[0].
__device__ __forceinline__ void lp_merge_all(u64 (*lists)[32], int count, int warp, int lane) {
    for (int step = count >> 1; step > 0; step >>= 1) {
        if (warp < step) {
            u64 list = lists[warp][lane];
            lp_merge(list, lists[warp + step][31 - lane], lane);
            lists[warp][lane] = list;
        }
        __syncthreads();
    }
}
// The n-th largest of the values that the threads of warps 0 - 7 have, on each of them; n <= 32.
__device__ __forceinline__ float lp_nth_of_cta(float v, float (*tops)[32], int warp, int lane, int n) {
#pragma unroll
    for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
        for (int j = k >> 1; j > 0; j >>= 1) {
            const float with = __shfl_xor_sync(0xffffffffu, v, j);
            v = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(v, with) : fminf(v, with);
        }
    tops[warp][lane] = v;  // largest first
    for (int step = LP_WARPS >> 1; step > 0; step >>= 1) {
        asm volatile("bar.sync 1, %0;" ::"n"(LP_THREADS) : "memory");
        if (warp < step) {
            v = fmaxf(v, tops[warp + step][31 - lane]);
#pragma unroll
            for (int j = 16; j > 0; j >>= 1) {
                const float with = __shfl_xor_sync(0xffffffffu, v, j);
                v = (lane & j) == 0 ? fmaxf(v, with) : fminf(v, with);
            }
            tops[warp][lane] = v;
        }
    }
    asm volatile("bar.sync 1, %0;" ::"n"(LP_THREADS) : "memory");
    const float nth = tops[0][n - 1];
    asm volatile("bar.sync 1, %0;" ::"n"(LP_THREADS) : "memory");  // before the next time
    return nth;
}
__device__ __forceinline__ float lp_key_value(u64 key) {
    const uint32_t u = (uint32_t)(key >> 32);
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// grid: rows x parts, cluster: parts.  Warps 0 - 7 take the logits, warp 8 brings them in.
template <typename T, bool TOP>
__global__ void __launch_bounds__(LP_THREADS + 32, 4) token_logprobs_kernel(TokenLogprobsArgs a, int parts) {
    constexpr int N = LpVector<T>::N, GROUP = 16 / N, E = 16;  // vectors and logits that a thread takes at once
    extern __shared__ __align__(16) uint4 ring[];
    __shared__ __align__(8) uint64_t full[LP_STAGES], empty[LP_STAGES];
    __shared__ u64 lists[LP_WARPS][32];
    __shared__ LogitSums sums_s[LP_WARPS], cta_sums;
    __shared__ int cta_bad;
    __shared__ float tops_s[LP_WARPS][32];
    if (threadIdx.x == 0) {
        for (int s = 0; s < LP_STAGES; ++s) mbar_init(full + s, 1), mbar_init(empty + s, LP_WARPS);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    GLMB_PDL_PROLOGUE();
    __syncthreads();
    const int row = blockIdx.x / parts, part = blockIdx.x % parts, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.stride;
    const int pre = min(a.vocab, (int)((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / (int)sizeof(T));
    const int vectors = (a.vocab - pre) / N, loose = a.vocab - vectors * N;  // elements before the first vector and behind the last
    const int begin = (int)((int64_t)vectors * part / parts), end = (int)((int64_t)vectors * (part + 1) / parts);
    const uint4* v = reinterpret_cast<const uint4*>(x + pre);
    const int stages = (end - begin + LP_STAGE - 1) / LP_STAGE;

    WarpSums mine{-INFINITY, 0.f, 0.f, false};
    u64 list = 0, last = 0;          // this warp's most likely tokens, and the entry that a further one has to beat
    int token = -1;
    float token_logit = 0.f;
    if (warp == LP_WARPS) {
        if (lane == 0) {
            int i = 0;
            for (; i < stages; ++i) {
                const int s = i % LP_STAGES, lap = i / LP_STAGES, at = begin + i * LP_STAGE;
                if (lap > 0 && !mbar_wait(empty + s, (lap - 1) & 1)) break;  // the others' waits run out too, and say so
                const uint32_t bytes = (uint32_t)min(LP_STAGE, end - at) * 16;
                mbar_expect_tx(full + s, bytes);
                asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                             ::"r"(smem_u32(ring + s * LP_STAGE)), "l"(v + at), "r"(bytes), "r"(smem_u32(full + s)) : "memory");
            }
            for (int k = max(0, i - LP_STAGES); k < i; ++k) mbar_wait(full + k % LP_STAGES, (k / LP_STAGES) & 1);  // nobody leaves while copies are under way
        }
        __syncwarp();
    } else {
        if (part == 0 && threadIdx.x == 0) {
            token = lp_token(a.scores, row, a.vocab, true);
            if (token >= 0) token_logit = LpVector<T>::one(x + token);
        }
        __syncwarp();
        float floor = -INFINITY, lane_top = -INFINITY;  // a logit below `floor` is not among the most likely
        // Every lane's logits whose bits are set in `mask`, bit e: value(e) of token id(e); the whole warp.
        auto offer = [&](uint32_t mask, auto value, auto id) {
            uint32_t who;
            while ((who = __ballot_sync(0xffffffffu, mask != 0)) != 0) {
                const int e = mask ? __ffs(mask) - 1 : 0;
                const u64 mine_now = mask ? candidate_key(value(e), id(e)) : 0;
                mask &= mask - 1;
                while (who) {  // the first of every lane's
                    const u64 k = __shfl_sync(0xffffffffu, mine_now, __ffs(who) - 1);
                    who &= who - 1;
                    if (k > last) {
                        lp_insert(list, k, lane);
                        last = __shfl_sync(0xffffffffu, list, a.top - 1);
                    }
                }
            }
        };
        if (part == 0 && warp == 0 && loose) {
            const int at = lane < pre ? lane : vectors * N + lane;
            float one[1] = {lane < loose ? LpVector<T>::one(x + at) : -INFINITY};
            mine.take(one, one[0], lane);
            if (TOP) offer(lane < loose, [&](int) { return one[0]; }, [&](int) { return at; });
        }
        bool ok = true;
        int refresh = 0;  // the stage at which the bound is found anew
        for (int i = 0; i < stages; ++i) {
            const int s = i % LP_STAGES, here = min(LP_STAGE, end - begin - i * LP_STAGE), id0 = pre + (begin + i * LP_STAGE) * N;
            if (ok && !mbar_wait_warp(full + s, (i / LP_STAGES) & 1)) {  // this warp goes on to the barriers, with no more logits
                if (lane == 0) raise_status(a.scores.status, GLMB_STATUS_WAIT_TIMEOUT);
                mine.bad = true;
                ok = false;
            }
            const uint4* tile = ring + s * LP_STAGE;
#pragma unroll 1
            for (int base = 0; base < here; base += LP_THREADS * GROUP) {
                float val[E];
                float top;
                const bool whole = ok && base + LP_THREADS * GROUP <= here;  // of the CTA
#pragma unroll
                for (int u = 0; u < GROUP; ++u) {
                    const int j = base + u * LP_THREADS + threadIdx.x;
                    float w[N];
                    if (whole || (ok && j < here)) {
                        LpVector<T>::get(tile[j], w);
#pragma unroll
                        for (int e = 0; e < N; ++e) val[u * N + e] = w[e];
                    } else {
#pragma unroll
                        for (int e = 0; e < N; ++e) val[u * N + e] = -INFINITY;
                    }
                }
                top = val[0];
#pragma unroll
                for (int e = 1; e < E; ++e) top = lp_max_nan(top, val[e]);
                mine.take(val, top, lane);
                if (TOP) {
                    if (a.top == 1) {
                        floor = mine.m;
                    } else {
                        lane_top = fmaxf(lane_top, top);
                        if (i == refresh && base == 0) floor = fmaxf(floor, lp_nth_of_cta(lane_top, tops_s, warp, lane, a.top));
                    }
                    if (__any_sync(0xffffffffu, top >= floor)) {
                        uint32_t mask = 0;
#pragma unroll
                        for (int u = 0; u < GROUP; ++u) {
                            const bool live = ok && base + u * LP_THREADS + (int)threadIdx.x < here;
#pragma unroll
                            for (int e = 0; e < N; ++e) mask |= live && val[u * N + e] >= floor ? 1u << (u * N + e) : 0u;
                        }
                        auto at = [&](int e) { return (base + e / N * LP_THREADS + (int)threadIdx.x) * N + e % N; };  // in the stage
                        offer(mask, [&](int e) { return LpVector<T>::one(reinterpret_cast<const T*>(tile) + at(e)); }, [&](int e) { return id0 + at(e); });
                        if (last) floor = fmaxf(floor, lp_key_value(last));
                    }
                }
            }
            if (i == refresh) refresh = i ? i * 4 : 2;
            __syncwarp();
            if (lane == 0) mbar_arrive(empty + s);
        }
    }
    LogitSums sums = mine.all();
    bool bad = mine.bad || sums.bad();
    if (warp < LP_WARPS) {
        if (lane == 0) sums_s[warp] = sums;
        if (TOP) lists[warp][lane] = list;
    }
    const int any_bad = __syncthreads_or(bad);
    if (TOP) lp_merge_all(lists, LP_WARPS, warp, lane);
    if (warp == 0) {
        sums = sums_s[lane & (LP_WARPS - 1)];
        sums.join_lanes(LP_WARPS);
        bad = any_bad;
    }
    if (parts > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        if (threadIdx.x == 0) cta_sums = sums, cta_bad = any_bad;
        cluster.sync();
        if (part == 0) {
            if (TOP && warp > 0 && warp < parts) lists[warp][lane] = cluster.map_shared_rank(&lists[0][0], warp)[lane];
            if (warp == 0) {
                sums.clear();
                bad = false;
                if (lane < parts) sums = *cluster.map_shared_rank(&cta_sums, lane), bad = *cluster.map_shared_rank(&cta_bad, lane) != 0;
                sums.join_lanes(LP_PARTS);
                bad = __any_sync(0xffffffffu, bad);
            }
        }
        cluster.sync();  // nobody leaves, or goes on, before what it holds has been read
        if (part != 0) return;
        if (TOP) lp_merge_all(lists, parts, warp, lane);
    }
    if (warp != 0) return;
    sums = LogitSums{__shfl_sync(0xffffffffu, sums.m, 0), __shfl_sync(0xffffffffu, sums.s, 0), __shfl_sync(0xffffffffu, sums.t, 0)};
    bad |= sums.bad();
    if (lane == 0) lp_store(a.scores, row, sums, bad, token, token_logit);
    if (TOP && lane < a.top) {
        const u64 key = lists[0][lane];
        const float value = lp_key_value(key);
        a.top_ids[(int64_t)row * a.top + lane] = bad ? -1 : candidate_id(key);
        a.top_logprobs[(int64_t)row * a.top + lane] = bad ? __int_as_float(0x7fffffff) : value == -INFINITY ? -INFINITY : (value - sums.m) - sums.norm();
    }
}

GLMB_API size_t glmb_token_logprobs_args_sizeof() { return sizeof(TokenLogprobsArgs); }

GLMB_API int glmb_token_logprobs(const TokenLogprobsArgs* args, cudaStream_t stream) {
    const TokenLogprobsArgs a = *args;
    if (a.rows < 0 || a.vocab < 1 || a.vocab > 0x7ffffff0 || a.top < 0 || a.top > LP_TOP || a.top > a.vocab || a.stride < 0 || a.rows > 0x7fffffff / LP_PARTS) return 1;
    if (a.rows == 0) return 0;
    // CTAs of a row: as many as run at once (three to four an SM), with 2,048 logits or more each.  Every CTA has its start, its bound and its merge to pay for:
    // 333 rows of 65,521 in fp32, five alternatives, 1, 2, 4 and 8 CTAs a row: 28.6, 34.5, 40, 50 us; 108 of 82,183: 23, 20, 20, 26; 40 of 154,880 in bf16: 32, 22, 17,
    // 15.6; one with twenty: 33, 23, 15.7, 12.3.
    int parts = 1;
    while (parts < LP_PARTS && (int64_t)a.rows * parts * 2 <= 148 * 3 && a.vocab / (2 * parts) >= 2048) parts *= 2;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * parts));
    cfg.blockDim = dim3(LP_THREADS + 32);
    // Evenly over the SMs: left to themselves four CTAs go to one while another has two, so each asks for as much shared memory as keeps a further one away (333
    // rows 33.1 -> 28.6 us, 200 rows 23.0 -> 20.4, 30 rows in eights 13.8 -> 11.7).  Clusters lie in one of eight groups of SMs, each of which may have parts - 1
    // places over: without room for them 16 rows in eights go in two rounds (11.1 -> 17.6).
    const int per_sm = ceil_div(a.rows * parts + (parts > 2 ? 8 * (parts - 1) : 0), 148);
    cfg.dynamicSmemBytes = per_sm < 4 ? LP_SM / (per_sm + 1) : LP_RING;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = g_glmb_pdl_enabled ? 1 : 0;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = parts;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaError_t e;
    static DeviceOnce once;
    const int dev = once.pending();
    if (dev != DeviceOnce::SET) {
        for (const void* k : {(const void*)token_logprobs_kernel<float, true>, (const void*)token_logprobs_kernel<float, false>, (const void*)token_logprobs_kernel<bf16, true>,
                              (const void*)token_logprobs_kernel<bf16, false>}) {
            e = cudaFuncSetAttribute(k, cudaFuncAttributeMaxDynamicSharedMemorySize, LP_SM / 2);
            if (e != cudaSuccess) return (int)e;
        }
        once.mark(dev);
    }
    if (a.is_f32) e = a.top ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<float, true>, a, parts) : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<float, false>, a, parts);
    else e = a.top ? cudaLaunchKernelEx(&cfg, token_logprobs_kernel<bf16, true>, a, parts) : cudaLaunchKernelEx(&cfg, token_logprobs_kernel<bf16, false>, a, parts);
    return e != cudaSuccess ? (int)e : (int)cudaGetLastError();
}

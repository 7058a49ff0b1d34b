// Log probabilities of given tokens straight from hidden states: x = hidden . head^T on tcgen05, of which only maximum, sums and the given token's logit
// leave the chip (logprobs.cuh: what is kept).  bf16 operands, fp32 sums.
//
// A tile is 256 tokens of the vocabulary by 128 rows on one SM (up to 128 rows in all: the table's bytes are the bound), or by 256 rows on a pair of SMs
// (cta_group::2: each CTA stages its own 128 rows and half of the tokens).  Workers with different row blocks walk the same tokens, so that they share a piece
// of the table in L2; where the workers divide among the row blocks with little left over, each keeps its row block and its sums in registers until
// the end, else it leaves the sums of every tile.  A second launch joins them, a warp a row.
//
// Bound: up to some 150 rows the table's bytes (16 rows of 4,096 against 131,072 tokens 168 us, 6.4 TB/s), above that the tensor core (2,048 rows 1,570 -
// 1,660 us, 1,325 - 1,400 TFLOP/s by the power the chip may draw), with narrow hidden states the sums (1,024 rows of 512: 124 - 174 us).
//
// The tensor core does not round its running sum to nearest: over K = 4,096 that is a bias of 3.7e-6 of a logit, eight times what fp32 loses otherwise.  So
// a sum stays there for 512 products only; the epilogue's threads keep their 128 logits in registers and add (at K = 512 the bias is 3.5e-7).  TMEM holds two
// accumulators, so that this runs beside the next products.
//
//   warp 0      TMA producer of this CTA's operands (pairs: all bytes are counted on the first CTA's barrier)
//   warp 1      TMEM allocation; issues the MMAs (of a pair: in the first CTA)
//   warps 2-9   sums: a thread a row, two warps a quarter of the rows, each half of the tokens
//
// Every wait is bounded; one that runs out raises GLMB_STATUS_WAIT_TIMEOUT, makes the rows whose sums are missing NaN, and the CTA still releases its TMEM.
#include "logprobs.cuh"
#include "tcgen05.cuh"

#define HL_COLS 256
#define HL_BOX 32      // tokens of a copy: a smaller tile reads no more than it needs
#define HL_CHUNK 8     // k steps of 64 between two additions
#define HL_THREADS 320
#define HL_STAGES 16   // at most
#define HL_RING (12 * 16384)
#define HL_SMEM (HL_RING + 16384 + 1024)  // a product reads 128 rows, of which a stage may hold fewer: what lies behind them, also behind the last stage
#define HL_MERGE_WARPS 4

struct HeadLogprobsArgs {
    const void* hidden; int64_t hidden_stride;
    const void* head; int64_t head_stride;
    TokenScores scores;
    float4* part;       // [rows][parts]: m, s, t
    float* given;       // [rows]: the token's logit
    int64_t parts;
    int rows, vocab, width;
};

// How the work is dealt.  keeps: worker w has row block w % blocks and the w / blocks-th run of tokens, of `run` each, in tiles of 256 and a smaller last one.
// Else worker w takes tiles w, w + workers, ..; tile i is row block i % blocks and tokens 256 (i / blocks) ..
// A stage of the ring holds `a_rows` rows and `b_rows` tokens of 64 columns.
struct HeadPlan { int blocks, tiles, workers, keeps, run, parts, a_rows, b_rows, stages; };
struct HeadTile { int block, token0, tokens, part; };
__device__ __forceinline__ bool hl_tile(const HeadPlan& plan, int vocab, int worker, int n, HeadTile& t) {  // the n-th tile of a worker
    if (plan.keeps) {
        t.block = worker % plan.blocks, t.part = worker / plan.blocks;
        const int end = (int)min((int64_t)vocab, (int64_t)(t.part + 1) * plan.run);
        const int64_t from = (int64_t)t.part * plan.run + (int64_t)n * HL_COLS;
        t.token0 = (int)min(from, (int64_t)end);
        t.tokens = min(HL_COLS, end - t.token0);
        return from < end;
    }
    const int64_t i = worker + (int64_t)n * plan.workers;
    t.block = (int)(i % plan.blocks), t.part = (int)(i / plan.blocks);
    if (t.part >= plan.tiles) return false;
    t.token0 = t.part * HL_COLS, t.tokens = min(HL_COLS, vocab - t.token0);
    return true;
}

__device__ __forceinline__ uint32_t hl_in_first_cta(uint32_t addr) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(at) : "r"(addr));
    return at;
}
__device__ __forceinline__ float hl_max_nan(float a, float b) {
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ void hl_tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
    __syncwarp();  // the whole warp's, as every access to tensor memory
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr) : "memory");
}

struct HeadRing {  // a place in the ring of stages
    uint32_t at = 0, lap = 0;
    __device__ __forceinline__ void next(uint32_t stages) {
        if (++at == stages) at = 0, ++lap;
    }
};

// What differs between one SM and a pair.
template <bool PAIR> struct HeadCta {
    static constexpr int UNIT = PAIR ? 2 * HL_BOX : HL_BOX;  // tokens that a tile is a multiple of
    static __device__ __forceinline__ void load(void* dst, const CUtensorMap* map, uint64_t* bar, int x, int y) {
        if constexpr (PAIR)
            asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
                         ::"r"(smem_u32(dst)), "l"(map), "r"(hl_in_first_cta(smem_u32(bar))), "r"(x), "r"(y) : "memory");
        else tma_load_2d(dst, map, bar, x, y);
    }
    static __device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, int columns, uint32_t accumulate) {
        if constexpr (PAIR)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(d), "l"(a), "l"(b), "r"(umma_idesc_bf16(256, columns)), "r"(accumulate) : "memory");
        else umma_bf16(d, a, b, umma_idesc_bf16(128, columns), accumulate);
    }
    static __device__ __forceinline__ void commit(uint64_t* bar) {  // pairs: at this barrier of both CTAs
        if constexpr (PAIR)
            asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(smem_u32(bar)), "h"((uint16_t)3) : "memory");
        else umma_commit(bar);
    }
    static __device__ __forceinline__ void sync() {
        if constexpr (PAIR) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
};

template <bool PAIR>
__device__ __forceinline__ void head_logprobs_cta(const CUtensorMap& map_a, const CUtensorMap& map_b, const CUtensorMap& map_rest, const HeadLogprobsArgs& p, const HeadPlan& plan) {
    typedef HeadCta<PAIR> C;
    GLMB_PDL_PROLOGUE();
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t full[HL_STAGES], empty[HL_STAGES], acc_full[2], acc_empty[2], drained;
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t fail;
    unsigned char* ring = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const int rank = PAIR ? blockIdx.x & 1 : 0, worker = PAIR ? blockIdx.x >> 1 : blockIdx.x;
    const int kblocks = (p.width + 63) >> 6, a_bytes = plan.a_rows * 128, stage = a_bytes + plan.b_rows * 128;
    constexpr int ROWS = PAIR ? 256 : 128;

    if (threadIdx.x == 0) {
        for (int s = 0; s < plan.stages; ++s) mbar_init(full + s, 1), mbar_init(empty + s, 1);
        for (int a = 0; a < 2; ++a) mbar_init(acc_full + a, 1), mbar_init(acc_empty + a, PAIR ? 16 : 8);
        mbar_init(&drained, 1);
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    C::sync();  // the barriers of both CTAs are ready
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;

    if (warp == 0) {
        HeadRing g, last;  // last: the place of the last stage but plan.stages
        int issued = 0;
        bool ok = true;
        HeadTile t;
        for (int n = 0; ok && hl_tile(plan, p.vocab, worker, n, t); ++n) {
            const int columns = (t.tokens + C::UNIT - 1) / C::UNIT * C::UNIT, mine = PAIR ? columns >> 1 : columns;
            const int a_row = t.block * ROWS + rank * 128, b_row = t.token0 + rank * mine;
            const bool whole = mine == plan.b_rows;
            for (int kb = 0; kb < kblocks; ++kb, g.next(plan.stages)) {
                const uint32_t s = g.at;
                if (g.lap > 0 && !mbar_wait_warp(empty + s, (g.lap - 1) & 1)) { fail = 1; ok = false; break; }
                if (elect_one()) {
                    unsigned char* dst = ring + s * stage;
                    if (rank == 0) mbar_expect_tx(full + s, (PAIR ? 2 : 1) * (a_bytes + mine * 128));
                    C::load(dst, &map_a, full + s, kb * 64, a_row);
                    if (whole) C::load(dst + a_bytes, &map_b, full + s, kb * 64, b_row);
                    else
                        for (int r = 0; r < mine; r += HL_BOX) C::load(dst + a_bytes + r * 128, &map_rest, full + s, kb * 64, b_row + r);
                }
                __syncwarp();
                if (++issued > plan.stages) last.next(plan.stages);
            }
        }
        // nobody leaves while copies are under way, not after a timeout either (of a pair the first CTA knows)
        for (int i = min(issued, plan.stages); rank == 0 && i > 0; --i, last.next(plan.stages)) mbar_wait_warp(full + last.at, last.lap & 1);
    } else if (warp == 1) {
        HeadRing g;
        uint32_t used = 0;  // accumulators so far
        bool ok = rank == 0;
        HeadTile t;
        for (int n = 0; ok && hl_tile(plan, p.vocab, worker, n, t); ++n) {
            const int columns = (t.tokens + C::UNIT - 1) / C::UNIT * C::UNIT;
            for (int k0 = 0; k0 < kblocks && ok; k0 += HL_CHUNK, ++used) {
                const uint32_t acc = used & 1, use = used >> 1;
                if (use > 0 && !mbar_wait_warp(acc_empty + acc, (use - 1) & 1)) { fail = 1; ok = false; break; }
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const int upto = min(kblocks, k0 + HL_CHUNK);
                for (int kb = k0; kb < upto; ++kb, g.next(plan.stages)) {
                    const uint32_t s = g.at;
                    if (!mbar_wait_warp(full + s, g.lap & 1)) { fail = 1; ok = false; break; }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t a_addr = smem_u32(ring + s * stage), b_addr = a_addr + a_bytes;
                    if (elect_one()) {
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            C::mma(tmem + acc * HL_COLS, umma_desc_sw128(a_addr + k * 32), umma_desc_sw128(b_addr + k * 32), columns, (kb > k0 || k > 0) ? 1u : 0u);
                        C::commit(empty + s);
                    }
                    __syncwarp();
                }
                if (ok && elect_one()) C::commit(acc_full + acc);  // of a pair the other CTA too takes what is announced for complete: abandoned sums never are
                __syncwarp();
            }
        }
        if (rank == 0 && elect_one()) C::commit(&drained);  // nor while products are
        __syncwarp();
        mbar_wait_warp(&drained, 0);
    } else {
        const int quarter = warp & 3, half = warp >= 6;
        const uint32_t at = tmem + half * 128 + ((uint32_t)(quarter * 32) << 16);
        LogitSums kept;
        kept.clear();
        uint32_t used = 0;
        bool ok = true;
        int row = -1, token = -1, n = 0;
        HeadTile t;
        for (; ok && hl_tile(plan, p.vocab, worker, n, t); ++n) {
            const int now = t.block * ROWS + rank * 128 + quarter * 32 + lane;
            if (now != row) row = now, token = row < p.rows ? lp_token(p.scores, row, p.vocab, false) : -1;
            const int token0 = t.token0 + half * 128, here = t.tokens - half * 128;  // tokens of this half: what lies behind them is of nobody
            float x[128];
            for (int k0 = 0; k0 < kblocks; k0 += HL_CHUNK, ++used) {
                const uint32_t acc = used & 1;
                ok = mbar_wait_warp(acc_full + acc, (used >> 1) & 1) && !__any_sync(0xffffffffu, fail);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                if (here > 0 && k0 == 0) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) hl_tmem_ld32_nowait(at + acc * HL_COLS + c * 32, reinterpret_cast<uint32_t*>(x) + c * 32);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                } else if (here > 0) {
#pragma unroll
                    for (int c = 0; c < 4; ++c) {
                        uint32_t y[32];
                        tmem_ld32(at + acc * HL_COLS + c * 32, y);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const float2 z = __fadd2_rn(make_float2(x[c * 32 + e], x[c * 32 + e + 1]), make_float2(__uint_as_float(y[e]), __uint_as_float(y[e + 1])));
                            x[c * 32 + e] = z.x, x[c * 32 + e + 1] = z.y;
                        }
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) {
                    if constexpr (PAIR)
                        asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(hl_in_first_cta(smem_u32(acc_empty + acc))) : "memory");
                    else mbar_arrive(acc_empty + acc);
                }
            }
            if (!ok) break;
            if (here > 0) {
                if (here < 128) {
#pragma unroll
                    for (int e = 0; e < 128; ++e)
                        if (e >= here) x[e] = -INFINITY;
                }
                const int wanted = token < 0 ? -1 : token - token0;
                if (__any_sync(0xffffffffu, wanted >= 0 && wanted < min(here, 128))) {
#pragma unroll
                    for (int e = 0; e < 128; ++e)
                        if (e == wanted && e < here) p.given[row] = x[e];
                }
                float top[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) top[e] = x[e];
#pragma unroll
                for (int e = 8; e < 128; ++e) top[e & 7] = hl_max_nan(top[e & 7], x[e]);
#pragma unroll
                for (int o = 4; o > 0; o >>= 1)
#pragma unroll
                    for (int e = 0; e < o; ++e) top[e] = hl_max_nan(top[e], top[e + o]);
                LogitSums tile{top[0], 0.f, 0.f};
                if (tile.m != -INFINITY) {  // a NaN ends up in s
                    // the sum without the terms of the maximum, and with them: their difference is how many there are
                    const float2 minus_m = make_float2(-tile.m, -tile.m), log2e = make_float2(LP_LOG2E, LP_LOG2E), zero = make_float2(0.f, 0.f);
                    float2 s[2] = {zero, zero}, all[2] = {zero, zero}, u[2] = {zero, zero};
#pragma unroll
                    for (int e = 0; e < 128; e += 2) {
                        const int c = (e >> 1) & 1;
                        float2 z = __fmul2_rn(__fadd2_rn(make_float2(x[e], x[e + 1]), minus_m), log2e);
                        z = make_float2(hl_max_nan(z.x, -1000.f), hl_max_nan(z.y, -1000.f));  // not minus infinity: its product with zero
                        const float2 w = make_float2(lp_exp2(z.x), lp_exp2(z.y));
                        all[c] = __fadd2_rn(all[c], w);
                        s[c] = __fadd2_rn(s[c], make_float2(z.x == 0.f ? 0.f : w.x, z.y == 0.f ? 0.f : w.y));
                        u[c] = __ffma2_rn(z, w, u[c]);
                    }
                    const float others = (s[0].x + s[0].y) + (s[1].x + s[1].y), sum = (all[0].x + all[0].y) + (all[1].x + all[1].y);
                    tile.s = others + (rintf(sum - others) - 1.f);
                    tile.t = ((u[0].x + u[0].y) + (u[1].x + u[1].y)) * 0.6931471805599453f;
                    if (isnan(tile.m)) tile.m = INFINITY, tile.s = tile.m - tile.m;
                }
                kept.join(tile);
            }
            if (!plan.keeps) {
                if (row < p.rows) p.part[(int64_t)row * plan.parts + t.part * 2 + half] = make_float4(kept.m, kept.s, kept.t, 0.f);
                kept.clear();
            }
        }
        if (!ok) {
            fail = 1;
            if (lane == 0) raise_status(p.scores.status, GLMB_STATUS_WAIT_TIMEOUT);
            do {  // no numbers where sums are missing: NaN in the rows of this tile and of those that will not be taken any more
                const int lost = t.block * ROWS + rank * 128 + quarter * 32 + lane;
                if (lost < p.rows) p.part[(int64_t)lost * plan.parts + t.part * 2 + half] = make_float4(INFINITY, __int_as_float(0x7fffffff), 0.f, 0.f);
            } while (!plan.keeps && hl_tile(plan, p.vocab, worker, ++n, t));
        } else if (plan.keeps && row >= 0 && row < p.rows) {
            p.part[(int64_t)row * plan.parts + t.part * 2 + half] = make_float4(kept.m, kept.s, kept.t, 0.f);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    C::sync();  // neither CTA leaves while the other may still signal it or read its operands
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HL_THREADS, 1)
head_logprobs_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_rest,
                          const __grid_constant__ HeadLogprobsArgs p, const __grid_constant__ HeadPlan plan) {
    head_logprobs_cta<true>(map_a, map_b, map_rest, p, plan);
}
__global__ void __launch_bounds__(HL_THREADS, 1)
head_logprobs_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const __grid_constant__ CUtensorMap map_rest,
                     const __grid_constant__ HeadLogprobsArgs p, const __grid_constant__ HeadPlan plan) {
    head_logprobs_cta<false>(map_a, map_b, map_rest, p, plan);
}

// A warp a row.
__global__ void __launch_bounds__(HL_MERGE_WARPS * 32) head_logprobs_merge_kernel(const __grid_constant__ HeadLogprobsArgs p, int parts) {
    GLMB_PDL_PROLOGUE();
    const int lane = threadIdx.x & 31, row = blockIdx.x * HL_MERGE_WARPS + (threadIdx.x >> 5);
    if (row >= p.rows) return;
    LogitSums sums;
    sums.clear();
    bool bad = false;
    for (int i0 = 0; i0 < parts; i0 += 128) {
        float4 v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = i0 + u * 32 + lane;
            v[u] = i < parts ? p.part[(int64_t)row * parts + i] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const LogitSums part{v[u].x, v[u].y, v[u].z};
            bad |= part.bad();
            sums.join(part);
        }
    }
    bad = __any_sync(0xffffffffu, bad);
    sums.join_lanes(32);
    if (lane != 0) return;
    const int k = lp_token(p.scores, row, p.vocab, true);
    lp_store(p.scores, row, sums, bad || sums.bad(), k, k >= 0 ? p.given[row] : 0.f);
}

// ---- host side ----------------------------------------------------------------------------------------------
static HeadPlan head_plan(int rows, int vocab, bool& pair) {
    // Pairs multiply up to 1.13 times as fast, in steps of 256 rows: 300 rows of 2,048 against 65,521 tokens 99 us on pairs (512 rows), 93 on single SMs (384); 600 of
    // 4,096 against 131,072 556 - 585 (768), 534 - 549 (640); at 256 rows and fewer than 129 left over pairs read the table once.
    pair = rows > 128 && 256 * ceil_div(rows, 256) * 100 <= 128 * ceil_div(rows, 128) * 113;
    HeadPlan plan;
    plan.blocks = ceil_div(rows, pair ? 256 : 128);
    plan.tiles = ceil_div(vocab, HL_COLS);
    const int all = pair ? 74 : 148, unit = pair ? HeadCta<true>::UNIT : HeadCta<false>::UNIT;
    // Row blocks and sums are kept to the end where at most a twentieth of the workers stays idle for it; a run of tokens is then as long for every one
    // of them.  (In whole tiles, 16 rows of 4,096 against 131,072 tokens took four rounds of 148 for 512 tiles: 204 us, 168 in equal runs.)
    const int groups = min(all / plan.blocks, ceil_div(vocab, unit));
    plan.keeps = all / plan.blocks * plan.blocks * 20 >= all * 19;
    plan.run = plan.keeps ? ceil_div(ceil_div(vocab, groups), unit) * unit : 0;
    plan.workers = plan.keeps ? ceil_div(vocab, plan.run) * plan.blocks : (int)min((int64_t)all, (int64_t)plan.blocks * plan.tiles);
    plan.parts = 2 * (plan.keeps ? plan.workers / plan.blocks : plan.tiles);
    // Few rows, or few tokens for each worker: smaller stages and more of them.
    plan.a_rows = rows < 128 ? ceil_div(rows, 8) * 8 : 128;
    plan.b_rows = (plan.keeps && plan.run < HL_COLS ? plan.run : HL_COLS) / (pair ? 2 : 1);
    plan.stages = min(HL_STAGES, HL_RING / ((plan.a_rows + plan.b_rows) * 128));
    return plan;
}
static int head_map(CUtensorMap* map, const void* base, int rows, int width, int64_t stride, int box_rows) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return 1;
    const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)stride * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, elem[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : 2;
}

GLMB_API size_t glmb_head_logprobs_args_sizeof() { return sizeof(HeadLogprobsArgs); }

// Sums of a row that are left for the second launch, four floats each.
GLMB_API int64_t glmb_head_logprobs_parts(int rows, int vocab) {
    bool pair;
    return rows < 1 || vocab < 1 ? 0 : head_plan(rows, vocab, pair).parts;
}

GLMB_API int glmb_head_logprobs(const HeadLogprobsArgs* args, cudaStream_t stream) {
    const HeadLogprobsArgs a = *args;
    if (a.rows < 0 || a.vocab < 1 || a.vocab > 0x7ffffe00 || a.width < 8 || a.width % 8 || a.hidden_stride % 8 || a.head_stride % 8) return 1;
    if (a.rows == 0) return 0;
    bool pair;
    const HeadPlan plan = head_plan(a.rows, a.vocab, pair);
    if (a.parts < plan.parts ) return 1;
    CUtensorMap map_a, map_b, map_rest;  // the table in whole tiles and in pieces
    if (head_map(&map_a, a.hidden, a.rows, a.width, a.hidden_stride, plan.a_rows) || head_map(&map_b, a.head, a.vocab, a.width, a.head_stride, plan.b_rows) ||
        head_map(&map_rest, a.head, a.vocab, a.width, a.head_stride, HL_BOX))
        return 3;
    static DeviceOnce once;
    const int dev = once.pending();
    if (dev != DeviceOnce::SET) {
        cudaError_t e = cudaFuncSetAttribute(head_logprobs_pair_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, HL_SMEM);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(head_logprobs_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, HL_SMEM);
        if (e != cudaSuccess) return (int)e;
        once.mark(dev);
    }
    if (pair) GLMB_LAUNCH(head_logprobs_pair_kernel, 2 * plan.workers, HL_THREADS, HL_SMEM, stream, map_a, map_b, map_rest, a, plan);
    else GLMB_LAUNCH(head_logprobs_kernel, plan.workers, HL_THREADS, HL_SMEM, stream, map_a, map_b, map_rest, a, plan);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return (int)e;
    GLMB_LAUNCH(head_logprobs_merge_kernel, ceil_div(a.rows, HL_MERGE_WARPS), HL_MERGE_WARPS * 32, 0, stream, a, plan.parts);
    return (int)cudaGetLastError();
}

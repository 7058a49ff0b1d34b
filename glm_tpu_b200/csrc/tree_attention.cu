// Attention of a few drafted tokens per sequence over a paged cache (bf16) on the 5th-generation tensor cores.
//
// Row j of a sequence, whose committed tokens lie in slots 0 .. length - 1 and whose drafted tokens in slots length, length + 1, ..:
//
//   o = sum_i p_i v_i,   p_i = e^(scale q . k_i) / (sum e^(scale q . k) + e^sink)
//
// over every committed slot and the drafted slots t (those of this call's rows) with bit t of the row's mask: its ancestors in the tree and itself.
// A row that sees nothing gives zeros.  A slot whose page the table does not know counts as not attended and raises GLMB_STATUS_BAD_INDEX, as does a
// sequence whose rows or length are out of range.
//
// A tile is up to 128 (drafted row, head) pairs of one key head: the M of both products.  A unit is a sequence's key head with one tile, or with two that
// take turns on the tensor core; its keys come in blocks of 128 or 64.  The blocks of all units, one after another, are dealt to one CTA per SM in equal runs, so
// that unequal sequences keep every SM streaming; a run may begin and end inside a unit.  For each block of a tile:
//
//   S = Q K^T       both operands K-major in shared memory (TMA, 128-byte swizzle), fp32 scores in TMEM
//   softmax         128 threads, one row each, running maximum and sum in fp32; weights back into TMEM where the scores were, in bf16
//   O += P V        A = weights from TMEM, B = values as they lie in memory
//
// A tile of up to 64 or 32 pairs is there two or four times among the 128 rows: each copy weighs its own half or quarter of every block (its weights of the rest
// are zeros), so that all threads have a part of the exponentials; the copies' sums meet like those of different runs, or in shared memory.
//
// The maximum is only followed when it grows by more than 2^8 (the weights stay finite, the division at the end removes the difference).  A weight is two bf16
// pieces, the second one the remainder of the first, so that 16 bits of it reach the product in every form: a row's digits do not depend on how many rows its call
// has.  One piece, a rounding of 2^-8 each beside that of the result, took 101 in place of 108 us for 4 x 16 drafts at 30,000 and 287 in place of 369 for 60 at 131,000;
// its error there was 2.3e-3 of the largest output, where the result's own rounding is 1.7e-3.
//
// Tiles that share a unit (PAIR) keep both groups of softmax threads busy, and the tensor core.  What bounds them is one warp that issues for both: a block of 128
// keys of two tiles takes some 2.7 thousand cycles of softmax (2.0 of them exponentials) and 3.1 of products at the tensor core's own rate
// (shared memory feeds S at half of it).  60 drafts of 8 heads at 131,000 slots: 369 us, tensor pipe active 57 %.  Measured with one piece, beside 303 (287 since the softmax threads have
// the registers that their scores need and the start of a unit counts in the runs): two buffers of scores, blocks of 64 keys 424 us, with two issuing warps 303;
// blocks of 128 with two issuing warps 357; exponentials of the two groups in turns 346.
// A tile alone has the two groups take alternate blocks, each with its own sums, which meet at the end of the run.  Heads wider than 128 (WIDE): blocks of 64 keys,
// one group, and two buffers of scores, so that the next ones are there when a softmax ends (40 drafts of 4 heads of 192 at 100,000 slots: 258 us, with one buffer
// 320).
//
//   warps 0-3, 4-7   softmax and output of group 0 and 1 (warp w reads TMEM lanes 32 (w % 4) ..)
//   warp 8           issues every tcgen05.mma, owns the TMEM allocation
//   warps 9, 10      look pages up, bring queries and keys, and values, in by TMA
//
// One warp issues for both groups and so waits for every block, in order: a warp that skipped the other group's blocks could take an older phase of a barrier
// for the one it waits for.
//
// What a row does not see must not reach it, and a weight of zero times NaN is NaN.  Slots behind the last one, and pages that do not exist, are read as zeros
// (out of the tensor map's range) or cleared in shared memory before the product; drafted values that are not finite are cleared too, and the rows
// that do see them add their product afterwards, one by one.
//
// Runs that share a unit, and copies, leave their sums in memory; a second launch joins them, and clears the rows of no sequence where asked to.  A cache of
// at most four blocks a sequence is dealt in whole units and needs none (JOINS: the copies meet in shared memory, which costs a stage of the ring: 64 pairs
// at 30,000 slots 109 us so, 103 otherwise): 36 requests of three tokens over 12 slots, 16 heads, 18.2 -> 14.1 us, one token of 8 heads of 64 13.2 -> 9.4.
// Every wait is bounded and a whole warp's, so that its lanes take one branch; one that runs out raises GLMB_STATUS_WAIT_TIMEOUT, makes the rows
// whose sums are missing NaN, and the CTA still releases its TMEM.
#include "paged.cuh"
#include "tcgen05.cuh"
#include "vec8.cuh"

#define TA_LOG2E 1.4426950408889634f
#define TA_MAX_DRAFTS 64  // bits of a mask
#define TA_SLACK 8.0f     // log2 of how far the weights may exceed one before the maximum is followed
#define TA_JOIN 68        // floats of a row of joined sums: 64 columns, padded
#define TA_WHOLE_BLOCKS 4 // caches of so few blocks a sequence: units are not split
#define TA_LONG_RUN 8     // blocks a CTA from which on the start of a unit counts
#define TA_START 4        // as so many
#define TA_NOTES 8        // blocks whose pages are remembered: the producer is at most five ahead of the softmax

enum { TA_PAIR = 0, TA_SINGLE = 1, TA_WIDE = 2 };

// Rows and committed slots of a sequence, within what there is.
struct TreeSeq {
    int row0, rows, drafts, length;
    __device__ __forceinline__ int blocks(int keys) const { return rows ? (length + drafts + keys - 1) / keys : 0; }
};
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttentionArgs& a, int b, bool report) {
    TreeSeq s;
    const int from = a.starts[b], to = a.starts[b + 1], length = a.lengths[b];
    s.row0 = min(max(from, 0), a.rows);
    s.rows = max(min(to, a.rows) - s.row0, 0);
    s.length = min(max(length, 0), a.cache.per_seq * a.cache.page);
    if (report && (from != s.row0 || to < from || to > a.rows || s.rows > a.max_rows || s.length != length)) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
    s.rows = min(s.rows, a.max_rows);
    s.drafts = s.rows;
    return s;
}

// How units are made: `heads` of a tile (of `head_blocks` of a key head), `tile_rows` drafted rows of a tile, tiles of a unit.
struct TreeShape {
    int per, heads, head_blocks, tile_rows, in_unit, copies, keys, ctas, units_max;  // units_max: of a key head of the largest sequence
    int whole;  // runs are whole units, as many for every CTA: nothing is left to join
    int start;  // blocks that the start of a unit counts for: a CTA's turn from one unit to the next
    // What a unit counts for in the runs: places, of which the first `start` hold no block.
    __device__ __forceinline__ int places(const TreeSeq& s) const { return whole ? 1 : s.blocks(keys) + start; }
    // The place of a tile's sums of a segment; a row's lie behind it.
    __device__ __forceinline__ int64_t part(int64_t segment, int tile_of_unit, int copy) const { return ((segment * in_unit + tile_of_unit) * copies + copy) * (heads * tile_rows); }
    // What a sequence's units count for in the runs.
    __device__ __forceinline__ int64_t share_of(const TreeSeq& s, int G) const { return s.rows ? (int64_t)places(s) * units(s.rows) * G : 0; }
    __device__ __forceinline__ int tiles(int rows) const { return (rows + tile_rows - 1) / tile_rows * head_blocks; }
    __device__ __forceinline__ int units(int rows) const { return (tiles(rows) + in_unit - 1) / in_unit; }
};

// Whose a row is: the last sequence that begins at or before it has it among its rows.  Also what the units of all sequences count for, and those of
// the sequences that begin no later; the whole warp.
struct TreeRow { TreeSeq seq; int b, j; bool mine; int64_t total, upto; };
__device__ __forceinline__ TreeRow tree_row(const TreeAttentionArgs& a, const TreeShape& sh, int row, int lane) {
    TreeRow r{{0, 0, 0, 0}, -1, 0, false, 0, 0};
    for (int b0 = 0; b0 < a.cache.seqs; b0 += 32) {
        bool begun = false;
        if (b0 + lane < a.cache.seqs) {
            const int64_t mine = sh.share_of(tree_seq(a, b0 + lane, false), a.cache.G);
            begun = a.starts[b0 + lane] <= row;
            r.total += mine;
            r.upto += begun ? mine : 0;
        }
        r.b += __popc(__ballot_sync(0xffffffffu, begun));
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        r.total += __shfl_xor_sync(0xffffffffu, r.total, o);
        r.upto += __shfl_xor_sync(0xffffffffu, r.upto, o);
    }
    if (r.b >= 0) r.seq = tree_seq(a, r.b, false);
    r.j = row - r.seq.row0;
    r.mine = r.b >= 0 && r.j >= 0 && r.j < r.seq.rows;
    return r;
}

// The part of a CTA's run that lies in one unit.
struct TreeSegment {
    TreeSeq seq;
    int b, g, unit;       // unit of the sequence's key head
    int block0, blocks;   // of `of` blocks of the unit
    int of;
};
// Walks a run.
struct TreeWalk {
    int64_t left;  // places
    int b, at;     // the sequence, and how many of its (key head, unit) pairs are done
    int block0;
    __device__ __forceinline__ bool next(const TreeAttentionArgs& a, const TreeShape& sh, TreeSegment& s) {
        while (left > 0 && b < a.cache.seqs) {
            s.seq = tree_seq(a, b, false);
            s.of = s.seq.blocks(sh.keys);
            const int units = s.of ? sh.units(s.seq.rows) : 0;
            if (at >= units * a.cache.G) {
                ++b, at = 0, block0 = 0;
                continue;
            }
            s.b = b, s.g = at / units, s.unit = at % units, s.block0 = block0;
            s.blocks = sh.whole ? s.of : (int)min((int64_t)(s.of - block0), left);
            left -= (sh.whole ? 1 : s.blocks) + sh.start;  // and the places at the start of the next unit
            ++at, block0 = 0;
            return true;
        }
        return false;
    }
};

__device__ __forceinline__ void ta_tmem_ld32_nowait(uint32_t taddr, uint32_t* r) {
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
__device__ __forceinline__ void ta_tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void ta_tma_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(smem_u32(smem_dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void ta_tma_4d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int x, int y, int z, int w) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
                 ::"r"(smem_u32(smem_dst)), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// MN-major operand, 128-byte swizzle: 64 columns (128 bytes) per K row, 8 K rows per 1024-byte group, 64-column boxes `box` bytes apart
__device__ __forceinline__ uint64_t ta_desc_mn(uint32_t smem_addr, uint32_t box) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | ((uint64_t)(box >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
__device__ __forceinline__ float ta_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Whether the condition holds for any of the 128 threads of a group; a barrier of theirs.
__device__ __forceinline__ bool ta_any_of_group(bool here) {
    uint32_t any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbar.red.or.pred q, 1, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(any) : "r"((uint32_t)here) : "memory");
    return any != 0;
}

// Bits i of a word of 32 keys whose first lies `ahead` slots behind the first drafted one (negative: before it): committed, or drafted and in the mask.
__device__ __forceinline__ uint32_t ta_visible(int ahead, uint64_t mask) {
    if (ahead >= 64) return 0u;
    if (ahead >= 0) return (uint32_t)(mask >> ahead);
    if (ahead <= -32) return ~0u;
    return (uint32_t)(mask << -ahead) | ((1u << -ahead) - 1u);
}

template <int MODE, int COPIES, bool JOINS> struct TreeMode {
    static constexpr int KEYS = MODE == TA_WIDE ? 64 : 128, ROWS = 128 / COPIES, COLS = KEYS / COPIES;  // rows of the tile, keys of a block that a thread weighs
    static constexpr int GROUPS = MODE == TA_WIDE ? 1 : 2, QTILES = MODE == TA_PAIR ? 2 : 1, SCORES = MODE == TA_WIDE ? 2 : 1;  // buffers
    static constexpr int STAGES = MODE == TA_SINGLE && !JOINS ? 3 : 2, BOXES = MODE == TA_WIDE ? 4 : 2;
    static constexpr int THREADS = MODE == TA_PAIR ? 384 : 352;  // a pair's last warp is there to give its registers away
    static constexpr int Q_BOX = 128 * 128, KV_BOX = KEYS * 128;  // bytes of a box of 64 columns
    static constexpr int JOIN = JOINS ? 128 * TA_JOIN * 4 : 0;  // 64 columns of the copies' sums
    static constexpr int SMEM = QTILES * BOXES * Q_BOX + 2 * STAGES * BOXES * KV_BOX + JOIN + 1024;

    // Of group t in a segment: its tile, whether nobody else has keys of the tile's rows, and else where their sums go.
    static __device__ __forceinline__ int tile_of(const TreeShape& sh, const TreeSegment& s, int t) { return s.unit * sh.in_unit + (MODE == TA_PAIR ? t : 0); }
    static __device__ __forceinline__ bool alone(const TreeSegment& s) { return (JOINS || COPIES == 1) && s.blocks == s.of; }
    static __device__ __forceinline__ int64_t part_of(const TreeAttentionArgs& a, const TreeShape& sh, const TreeSegment& s, int t, int copy) {
        return sh.part(((int64_t)s.b * a.cache.G + s.g) * sh.units_max + s.unit + blockIdx.x, MODE == TA_PAIR ? t : 0, JOINS ? 0 : copy);
    }
};

// After a lost wait: no numbers where sums are missing.  NaN in the thread's row of this segment and of those that will not be taken any more.
template <int MODE, int COPIES, bool JOINS>
__device__ __noinline__ void tree_lost(const TreeAttentionArgs& a, const TreeShape& sh, TreeWalk walk, TreeSegment s, int t, int row) {
    typedef TreeMode<MODE, COPIES, JOINS> T;
    const int copy = row / T::ROWS, in = row % T::ROWS;
    const float none = __int_as_float(0x7fffffff);
    do {
        const int tile = T::tile_of(sh, s, t), j = tile / sh.head_blocks * sh.tile_rows + in / sh.heads, hh = tile % sh.head_blocks * sh.heads + in % sh.heads;
        if (in >= sh.heads * sh.tile_rows || tile >= sh.tiles(s.seq.rows) || j >= s.seq.rows || hh >= sh.per || (JOINS && copy)) continue;
        if (!T::alone(s)) {  // the launch that joins them sees it
            *reinterpret_cast<float2*>(a.part_ml + (T::part_of(a, sh, s, t, copy) + in) * 2) = make_float2(none, none);
            continue;
        }
        bf16* dst = a.out + (int64_t)(s.seq.row0 + j) * a.out_row + (int64_t)(s.g * sh.per + hh) * a.out_head;
        for (int x = 0; x < a.cache.vdim; x += 8) *reinterpret_cast<uint4*>(dst + x) = make_uint4(~0u, ~0u, ~0u, ~0u);
    } while (walk.next(a, sh, s));
}

template <int MODE, int COPIES, bool JOINS>
__global__ void __launch_bounds__(TreeMode<MODE, COPIES, JOINS>::THREADS, 1)
tree_attention_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                      const __grid_constant__ TreeAttentionArgs a, const __grid_constant__ TreeShape sh, int slots_first_k, int slots_first_v, int chunk) {
    typedef TreeMode<MODE, COPIES, JOINS> T;
    constexpr int KEYS = T::KEYS, STAGES = T::STAGES, WORDS = KEYS / 32;
    extern __shared__ unsigned char smem_raw[];
    __shared__ __align__(8) uint64_t q_full, q_empty, k_full[STAGES], k_empty[STAGES], v_full[STAGES], v_empty[STAGES];
    __shared__ __align__(8) uint64_t s_full[2][2], p_full[2][2], o_full[2], o_free[2], pv_done[2], ml_full, drained;  // of a group (and of its buffer of scores)
    __shared__ uint32_t tmem_slot;
    __shared__ volatile uint32_t fail;
    __shared__ uint32_t page_bits[TA_NOTES][WORDS];  // keys of a block whose page exists
    __shared__ unsigned long long broken[4];         // drafted values of a segment that are not finite
    __shared__ float ml_s[128][2], copy_s[128][2], scale_s[128];
    __shared__ int64_t run_s[3];
    const int warp = uniform_warp(), lane = threadIdx.x & 31;
    const PagedArgs& c = a.cache;
    const int kboxes = (c.dim + 63) / 64, vboxes = (c.vdim + 63) / 64;
    unsigned char* q_s = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    unsigned char* k_s = q_s + T::QTILES * T::BOXES * T::Q_BOX;
    unsigned char* v_s = k_s + STAGES * T::BOXES * T::KV_BOX;
    float* join_s = reinterpret_cast<float*>(v_s + STAGES * T::BOXES * T::KV_BOX);

    if (threadIdx.x == 0) {
        mbar_init(&q_full, 1), mbar_init(&q_empty, 1), mbar_init(&ml_full, 4), mbar_init(&drained, 1);
        for (int i = 0; i < 2; ++i) {
            mbar_init(o_full + i, 1), mbar_init(o_free + i, 4), mbar_init(pv_done + i, 1);
            for (int e = 0; e < 2; ++e) mbar_init(&s_full[i][e], 1), mbar_init(&p_full[i][e], 4);
        }
        for (int i = 0; i < STAGES; ++i) mbar_init(k_full + i, 1), mbar_init(k_empty + i, 1), mbar_init(v_full + i, 1), mbar_init(v_empty + i, 1);
        for (int i = 0; i < 4; ++i) broken[i] = 0;
        fail = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (const CUtensorMap* map : {&map_q, &map_k, &map_v}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    }
    GLMB_PDL_PROLOGUE();  // before the TMEM allocation: a kernel still running may need the columns to finish
    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_slot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 9) {  // this CTA's run: equal numbers of blocks, in the order of the sequences
        auto blocks_of = [&](int b) {
            if (b >= c.seqs) return (int64_t)0;
            return sh.share_of(tree_seq(a, b, blockIdx.x == 0), c.G);
        };
        int64_t mine = blocks_of(lane), total = mine;
        for (int b = lane + 32; b < c.seqs; b += 32) total += blocks_of(b);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        const int64_t share = (total + sh.ctas - 1) / sh.ctas, first = min(total, share * (int)blockIdx.x), count = min(share, total - first);
        int64_t before = 0;
        int found = -1;
        for (int seq = 0; seq < c.seqs && found < 0; seq += 32) {
            if (seq > 0) mine = blocks_of(seq + lane);
            int64_t upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int64_t add = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += add;
            }
            const uint32_t who = __ballot_sync(0xffffffffu, mine > 0 && first < before + upto && first >= before + upto - mine);
            if (who) {
                found = seq + __ffs(who) - 1;
                const int64_t rest = first - (before + __shfl_sync(0xffffffffu, upto - mine, __ffs(who) - 1));
                if (lane == 0) run_s[1] = found, run_s[2] = rest;
            }
            before += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) run_s[0] = found < 0 ? 0 : count;
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = tmem_slot;  // scores of the groups at columns 0 and 128 (a second buffer 64 behind), O_0, O_1 at 256 and 384

    TreeWalk walk{run_s[0], 0, 0, 0};
    if (walk.left > 0) {
        walk.b = (int)run_s[1];
        const int places = sh.places(tree_seq(a, walk.b, false));
        const int place = (int)(run_s[2] % places) - sh.start;
        walk.at = (int)(run_s[2] / places), walk.block0 = max(place, 0), walk.left += min(place, 0);
    }
    // blocks of a segment that group t takes, and the n-th of them (counted from the segment's first)
    auto group_blocks = [&](const TreeSegment& s, int t) {
        if (MODE == TA_PAIR) return s.unit * 2 + t < sh.tiles(s.seq.rows) ? s.blocks : 0;
        if (MODE == TA_SINGLE) return (s.blocks + 1 - t) >> 1;
        return t == 0 ? s.blocks : 0;
    };
    auto nth = [&](int t, int n) { return MODE == TA_SINGLE ? 2 * n + t : n; };

    TreeSegment s;
    uint32_t gone = 0;  // blocks of the segments before this one
    int segment = 0;
    if (MODE == TA_PAIR) {  // 384 x 168 registers at the launch: 256 x 200 and 128 x 104
        if (warp >= 8) asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        else asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
    }
    if (warp == 11) {  // of a pair
    } else if (warp >= 9) {  // keys (and queries), values
        const bool keys = warp == 9;
        const int boxes = keys ? kboxes : vboxes, chunks = KEYS / chunk;
        const CUtensorMap* map = keys ? &map_k : &map_v;
        const bool slots_first = keys ? slots_first_k : slots_first_v;
        unsigned char* ring = keys ? k_s : v_s;
        uint64_t *full = keys ? k_full : v_full, *empty = keys ? k_empty : v_empty;
        uint32_t issued = 0;  // blocks
        int queries = 0;
        bool ok = true;
        for (; ok && walk.next(a, sh, s); gone += s.blocks, ++segment) {
            if (keys) {
                if (segment > 0 && !mbar_wait_warp(&q_empty, (segment - 1) & 1)) { fail = 1; break; }
                const int tiles = MODE == TA_PAIR ? min(2, sh.tiles(s.seq.rows) - s.unit * 2) : 1;
                ++queries;
                if (lane == 0) broken[segment & 3] = 0;
                __syncwarp();
                if (elect_one()) {
                    mbar_expect_tx(&q_full, tiles * kboxes * COPIES * sh.heads * sh.tile_rows * 128);
                    for (int t = 0; t < tiles; ++t) {
                        const int tile = s.unit * sh.in_unit + t;
                        for (int x = 0; x < kboxes * COPIES; ++x)
                            ta_tma_3d(q_s + (t * kboxes + x / COPIES) * T::Q_BOX + x % COPIES * T::ROWS * 128, &map_q, &q_full, x / COPIES * 64,
                                      s.g * sh.per + tile % sh.head_blocks * sh.heads, s.seq.row0 + tile / sh.head_blocks * sh.tile_rows);
                    }
                }
                __syncwarp();
            }
            const int last = s.seq.length + s.seq.drafts;  // slots from `last` on hold nothing
            auto page_of = [&](int block) {  // lane i: the page of the i-th chunk, or one behind the last (read as zeros)
                const int slot = (s.block0 + block) * KEYS + lane * chunk;
                if (block >= s.blocks || lane >= chunks || slot >= last) return c.pages;
                const int page = paged_page(c, s.b, slot);
                if (page < 0 && keys) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
                return page < 0 ? c.pages : page;
            };
            int page = page_of(0);
            for (int j = 0; j < s.blocks; ++j) {
                const uint32_t n = gone + j, st = n % STAGES, lap = n / STAGES;
                const int next_page = page_of(j + 1), in_page = ((s.block0 + j) * KEYS + lane * chunk) % c.page;
                if (lap > 0 && !mbar_wait_warp(empty + st, (lap - 1) & 1)) { fail = 1; ok = false; break; }
                if (keys) {
                    const uint32_t there = __ballot_sync(0xffffffffu, page < c.pages);
                    if (lane < WORDS) {
                        uint32_t bits = 0;
                        for (int i = 0; i < 32; i += 8) bits |= there >> ((lane * 32 + i) / chunk) & 1u ? 0xffu << i : 0u;
                        page_bits[n % TA_NOTES][lane] = bits;
                    }
                    __syncwarp();
                }
                if (lane == 0) mbar_expect_tx(full + st, boxes * T::KV_BOX);  // releases the notes too
                __syncwarp();
                if (lane < chunks)
                    for (int x = 0; x < boxes; ++x)
                        ta_tma_4d(ring + (st * boxes + x) * T::KV_BOX + lane * chunk * 128, map, full + st, x * 64, slots_first ? in_page : s.g, slots_first ? s.g : in_page, page);
                __syncwarp();
                page = next_page;
                ++issued;
            }
        }
        // nobody leaves while copies are under way, not after a timeout either
        for (uint32_t n = issued > STAGES ? issued - STAGES : 0; n < issued; ++n) mbar_wait_warp(full + n % STAGES, (n / STAGES) & 1);
        if (queries) mbar_wait_warp(&q_full, (queries - 1) & 1);
    } else if (warp == 8) {
        const uint32_t idesc_s = umma_idesc_bf16(128, KEYS), idesc_o = umma_idesc_bf16(128, c.vdim) | (1u << 16);  // bit 16: B is MN-major
        uint32_t made[2] = {0, 0}, done[2] = {0, 0}, uses[2] = {0, 0};  // blocks of scores, of outputs, and segments of a group so far
        bool ok = true;
        for (; ok && walk.next(a, sh, s); gone += s.blocks, ++segment) {
            const int count[2] = {group_blocks(s, 0), group_blocks(s, 1)}, most = max(count[0], count[1]);
            if (!mbar_wait_warp(&q_full, segment & 1)) { fail = 1; break; }
            auto last_of_block = [&](int t) { return MODE != TA_PAIR || t == 1 || count[1] == 0; };
            auto scores = [&](int t, int j) {  // S_t = Q_t K^T
                const uint32_t n = gone + nth(t, j), st = n % STAGES, buffer = T::SCORES == 2 ? made[t] & 1 : 0;
                if (!mbar_wait_warp(k_full + st, (n / STAGES) & 1)) return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t q_at = umma_desc_sw128(smem_u32(q_s + (MODE == TA_PAIR ? t : 0) * kboxes * T::Q_BOX)), k_at = umma_desc_sw128(smem_u32(k_s + st * kboxes * T::KV_BOX));
                const uint32_t s_at = tmem + t * 128 + buffer * 64;
                if (elect_one()) {
                    for (int x = 0; x < kboxes; ++x)  // a step of 16 columns: 32 bytes, 2 in the descriptor
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (x * 64 + k * 16 < c.dim)
                                umma_bf16(s_at, q_at + x * (T::Q_BOX / 16) + k * 2, k_at + x * (T::KV_BOX / 16) + k * 2, idesc_s, (x > 0 || k > 0) ? 1u : 0u);
                    umma_commit(&s_full[t][buffer]);
                    if (last_of_block(t)) umma_commit(k_empty + st);
                    if (nth(t, j) + 1 == s.blocks && last_of_block(t)) umma_commit(&q_empty);  // the segment's last scores
                }
                __syncwarp();
                ++made[t];
                return true;
            };
            auto outputs = [&](int t, int j) {  // O_t += P_t V
                const uint32_t n = gone + nth(t, j), st = n % STAGES, buffer = T::SCORES == 2 ? done[t] & 1 : 0, use = T::SCORES == 2 ? done[t] >> 1 : done[t];
                if (!((j > 0 || uses[t] == 0 || mbar_wait_warp(o_free + t, (uses[t] - 1) & 1)) && mbar_wait_warp(&p_full[t][buffer], use & 1) &&
                      mbar_wait_warp(v_full + st, (n / STAGES) & 1)))
                    return false;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t v_at = ta_desc_mn(smem_u32(v_s + st * vboxes * T::KV_BOX), T::KV_BOX);
                const uint32_t p_addr = tmem + t * 128 + buffer * 64;
                if (elect_one()) {
#pragma unroll
                    for (int piece = 0; piece < 2; ++piece)  // of the weights
#pragma unroll
                        for (int k = 0; k < KEYS / 16; ++k)
                            umma_bf16_ts(tmem + 256 + t * 128, p_addr + piece * (KEYS / 2) + k * 8, v_at + k * 128, idesc_o, (j > 0 || piece > 0 || k > 0) ? 1u : 0u);
                    if (T::SCORES == 2) umma_commit(pv_done + t);
                    if (last_of_block(t)) umma_commit(v_empty + st);  // the values may be replaced once they have been read
                    if (j + 1 == count[t]) umma_commit(o_full + t);
                }
                __syncwarp();
                ++done[t];
                if (j + 1 == count[t]) ++uses[t];
                return true;
            };
            for (int j = -1; j < most && ok; ++j) {
                if (T::SCORES == 2) {  // the next scores are there before the softmax asks for them
#pragma unroll
                    for (int t = 0; t < T::GROUPS; ++t) ok = ok && (j + 1 >= count[t] || scores(t, j + 1));
#pragma unroll
                    for (int t = 0; t < T::GROUPS; ++t) ok = ok && (j < 0 || j >= count[t] || outputs(t, j));
                } else {
#pragma unroll
                    for (int t = 0; t < T::GROUPS; ++t) {
                        ok = ok && (j < 0 || j >= count[t] || outputs(t, j));
                        ok = ok && (j + 1 >= count[t] || scores(t, j + 1));
                    }
                }
                if (!ok || __any_sync(0xffffffffu, fail)) { fail = 1; ok = false; }
            }
        }
        if (elect_one()) umma_commit(&drained);  // nor while products are
        __syncwarp();
        mbar_wait_warp(&drained, 0);
    } else {
        const int t = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane, copy = row / T::ROWS, in = row % T::ROWS, col0 = copy * T::COLS;
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const float scale2 = a.scale * TA_LOG2E;
        const bool fixes = MODE != TA_PAIR || t == 0;  // of two tiles the first one's products come first
        uint32_t seen = 0, used[2] = {0, 0}, joined = 0;  // blocks of this group, segments of each group, segments in which both had blocks
        bool ok = true;
        for (; ok && walk.next(a, sh, s); gone += s.blocks, ++segment) {
            const int count = group_blocks(s, t), other = MODE == TA_SINGLE ? group_blocks(s, 1 - t) : 0;
            if (count == 0) {
                if (other) ++used[1 - t];
                continue;
            }
            const int tile = T::tile_of(sh, s, t), j0 = tile / sh.head_blocks * sh.tile_rows, h0 = tile % sh.head_blocks * sh.heads;
            const int j = j0 + in / sh.heads, hh = h0 + in % sh.heads;
            const bool live = in < sh.heads * sh.tile_rows && j < s.seq.rows && hh < sh.per, warp_live = __any_sync(0xffffffffu, live);
            const uint64_t drafts = s.seq.drafts >= 64 ? ~0ull : (1ull << s.seq.drafts) - 1ull;
            const uint64_t mask = live ? (uint64_t)a.masks[s.seq.row0 + j] & drafts : 0;
            float m = -INFINITY, l = 0.f;
            for (int n = 0; n < count; ++n) {
                const int block = s.block0 + nth(t, n), base = block * KEYS;
                const uint32_t number = gone + nth(t, n), st = number % STAGES;
                const uint32_t buffer = T::SCORES == 2 ? seen & 1 : 0, s_addr = tmem + t * 128 + buffer * 64 + lanes;
                if (!mbar_wait_warp(&s_full[t][buffer], (T::SCORES == 2 ? seen >> 1 : seen) & 1) || __any_sync(0xffffffffu, fail)) { ok = false; break; }
                ++seen;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                uint32_t there = ~0u;
#pragma unroll
                for (int w = 0; w < WORDS; ++w) there &= page_bits[number % TA_NOTES][w];
                const bool drafted = base + KEYS > s.seq.length;
                if (warp_live) {
                    float x[T::COLS];
                    constexpr int PARTS = (T::COLS + 31) / 32;  // loads of 32 columns
#pragma unroll
                    for (int i = 0; i < PARTS; ++i) ta_tmem_ld32_nowait(s_addr + col0 + i * 32, reinterpret_cast<uint32_t*>(x) + i * 32);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    if (drafted || there != ~0u) {
#pragma unroll
                        for (int w = 0; w < PARTS; ++w) {
                            const uint32_t sees = ta_visible(base + col0 + w * 32 - s.seq.length, mask) & page_bits[number % TA_NOTES][col0 / 32 + w];
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(sees >> i & 1)) x[w * 32 + i] = -INFINITY;
                        }
                    }
                    float top[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) top[i] = x[i];
#pragma unroll
                    for (int i = 8; i < T::COLS; ++i) top[i & 7] = fmaxf(top[i & 7], x[i]);
#pragma unroll
                    for (int i = 4; i > 0; i >>= 1)
#pragma unroll
                        for (int e = 0; e < i; ++e) top[e] = fmaxf(top[e], top[e + i]);
                    const float most = top[0] * scale2;
                    if (n == 0) {
                        m = most;
                    } else if (__any_sync(0xffffffffu, most > m + TA_SLACK)) {
                        if (T::SCORES == 2) {  // the product before this block's may still be adding
                            if (!mbar_wait_warp(pv_done + t, (seen - 2) & 1)) ok = false;
                            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        }
                        const float next = fmaxf(m, most), fix = next == -INFINITY ? 1.f : ta_exp2(m - next);
                        m = next;
                        l *= fix;
                        for (int x0 = 0; x0 < c.vdim; x0 += 16) {
                            uint32_t o[16];
                            tmem_ld16(tmem + 256 + t * 128 + lanes + x0, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * fix);
                            ta_tmem_st16(tmem + 256 + t * 128 + lanes + x0, o);
                        }
                    }
                    const float from = m == -INFINITY ? 0.f : m;
                    const float2 scale_2 = make_float2(scale2, scale2), from_2 = make_float2(-from, -from);
                    float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                    __syncwarp();  // before the stores
#pragma unroll
                    for (int w = 0; w < PARTS; ++w) {
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const float2 z = __ffma2_rn(make_float2(x[w * 32 + 2 * i], x[w * 32 + 2 * i + 1]), scale_2, from_2), p = make_float2(ta_exp2(z.x), ta_exp2(z.y));
                            sum[i & 1] = __fadd2_rn(sum[i & 1], p);
                            hi[i] = pack_bf16(p.x, p.y);
                            const float2 rest = __fadd2_rn(p, make_float2(-bf16_lo(hi[i]), -bf16_hi(hi[i])));
                            lo[i] = pack_bf16(rest.x, rest.y);
                        }
                        ta_tmem_st16(s_addr + col0 / 2 + w * 16, hi);
                        ta_tmem_st16(s_addr + KEYS / 2 + col0 / 2 + w * 16, lo);
                    }
                    if constexpr (COPIES > 1) {  // the other copies' keys are not this row's
                        const uint32_t none[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
                        for (int at = 0; at < KEYS / 2; at += 16)
                            if (at < col0 / 2 || at >= col0 / 2 + T::COLS / 2) {
                                ta_tmem_st16(s_addr + at, none);
                                ta_tmem_st16(s_addr + KEYS / 2 + at, none);
                            }
                    }
                    l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                    asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                }
                if (drafted && fixes) {  // values that nobody, or not everybody, may multiply
                    if (!mbar_wait_warp(v_full + st, (number / STAGES) & 1)) { ok = false; break; }
                    const int key = (KEYS / 4) * quarter + lane, draft = base + key - s.seq.length;
                    if (lane < KEYS / 4 && draft >= 0) {
                        unsigned char* at = v_s + st * vboxes * T::KV_BOX + key * 128;
                        bool clear = draft >= s.seq.drafts;
                        for (int x = 0; x < vboxes * 8 && !clear; ++x) {
                            const uint4 u = *reinterpret_cast<const uint4*>(at + (x >> 3) * T::KV_BOX + (((x & 7) ^ (key & 7)) << 4));
                            for (uint32_t word : {u.x, u.y, u.z, u.w}) clear |= (word & 0x7f80u) == 0x7f80u || (word & 0x7f800000u) == 0x7f800000u;
                        }
                        if (clear) {
                            for (int x = 0; x < vboxes * 8; ++x) *reinterpret_cast<uint4*>(at + (x >> 3) * T::KV_BOX + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
                            if (draft < s.seq.drafts) atomicOr(&broken[segment & 3], 1ull << draft);
                        }
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                }
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[t][buffer]);
                if (!ok) break;
            }
            // the output of the segment: group 0 of a single tile takes what group 1 has along
            if (MODE == TA_SINGLE && t == 1) {
                if (ok && (used[1] == 0 || mbar_wait_warp(o_free + 1, (used[1] - 1) & 1))) {
                    ml_s[row][0] = m, ml_s[row][1] = l;
                    __syncwarp();
                    if (lane == 0) mbar_arrive(&ml_full);
                } else {
                    ok = false;
                }
                ++used[0], ++used[1];
                if (!ok) break;
                continue;
            }
            const bool both = MODE == TA_SINGLE && other > 0;
            if (ok) ok = mbar_wait_warp(o_full + t, used[t] & 1) && !__any_sync(0xffffffffu, fail);
            if (ok && both) ok = mbar_wait_warp(o_full + 1, used[1] & 1) && mbar_wait_warp(&ml_full, joined & 1) && !__any_sync(0xffffffffu, fail);
            ++used[t];
            if (both) ++used[1], ++joined;
            if (!ok) fail = 1;
            if (!ok && !JOINS) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const uint64_t lost = broken[segment & 3] & mask;
            const bool whole = T::alone(s);  // nobody else has keys of this row
            float f0 = 1.f, f1 = 0.f;
            if (both) {
                const float m1 = ml_s[row][0], l1 = ml_s[row][1], next = fmaxf(m, m1);
                f0 = m == next ? 1.f : ta_exp2(m - next);
                f1 = m1 == next ? 1.f : ta_exp2(m1 - next);
                l = l * f0 + l1 * f1;
                m = isnan(m1) ? m1 : next;
            }
            const int head = s.g * sh.per + hh, out_row = s.seq.row0 + j;
            const int64_t part = T::part_of(a, sh, s, t, copy);
            if constexpr (JOINS) {  // every copy learns the sums of the row's keys
                copy_s[row][0] = m, copy_s[row][1] = l;
                ok = !ta_any_of_group(!ok);  // the four warps go on together, or none of them does: those that did would wait for the others without a limit
                if (!ok) break;
                float next = m, all = 0.f;
#pragma unroll
                for (int k = 0; k < COPIES; ++k) next = fmaxf(next, copy_s[k * T::ROWS + in][0]);
#pragma unroll
                for (int k = 0; k < COPIES; ++k) {
                    const float mk = copy_s[k * T::ROWS + in][0], lk = copy_s[k * T::ROWS + in][1];
                    all += mk == next ? lk : lk * ta_exp2(mk - next);
                }
                const float f = m == next ? 1.f : ta_exp2(m - next);
                f0 *= f, f1 *= f, m = next, l = all;
            }
            float scale = 1.f;
            if (whole) {
                const float sink2 = a.sink && live ? a.sink[head] * TA_LOG2E : -INFINITY;
                if (sink2 != -INFINITY) {
                    const float next = fmaxf(m, sink2), f = m == -INFINITY ? 0.f : ta_exp2(m - next);
                    scale = f / (l * f + ta_exp2(sink2 - next));
                } else {
                    scale = l == 0.f ? 0.f : 1.f / l;
                }
            }
            if (live && !whole) *reinterpret_cast<float2*>(a.part_ml + (part + in) * 2) = make_float2(m, l);
            if (JOINS && copy == 0) scale_s[in] = scale;
            for (int x1 = 0; x1 < c.vdim; x1 += 64) {
                const int upto = min(c.vdim, x1 + 64);
                if (warp_live)
                    for (int x0 = x1; x0 < upto; x0 += 16) {
                        uint32_t o[16];
                        tmem_ld16(tmem + 256 + t * 128 + lanes + x0, o);
                        float y[16];
#pragma unroll
                        for (int i = 0; i < 16; ++i) y[i] = __uint_as_float(o[i]) * f0;
                        if (both) {
                            tmem_ld16(tmem + 384 + lanes + x0, o);
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = fmaf(__uint_as_float(o[i]), f1, y[i]);
                        }
                        if (!live) continue;
                        for (uint64_t left = lost; left; left &= left - 1) {  // drafted values that were left out of the product
                            const int drafted_slot = s.seq.length + __ffsll(left) - 1, page = paged_page(c, s.b, drafted_slot);
                            if (drafted_slot % KEYS / T::COLS != copy) continue;
                            const bf16* k = c.k + page * c.k_page + (drafted_slot % c.page) * c.k_slot + s.g * c.k_head;
                            const bf16* v = c.v + page * c.v_page + (drafted_slot % c.page) * c.v_slot + s.g * c.v_head + x0;
                            const bf16* q = a.q + (int64_t)out_row * a.q_row + (int64_t)head * a.q_head;
                            float dot = 0.f;
                            for (int d = 0; d < c.dim; ++d) dot = fmaf(to_f32(q[d]), to_f32(k[d]), dot);
                            const float p = ta_exp2(fmaf(dot, scale2, -m));
#pragma unroll
                            for (int i = 0; i < 16; ++i) y[i] = fmaf(p, to_f32(v[i]), y[i]);
                        }
                        if (JOINS) {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(join_s + row * TA_JOIN + x0 - x1 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                        } else if (whole) {
                            uint32_t w[8];
#pragma unroll
                            for (int i = 0; i < 8; ++i) w[i] = pack_bf16(y[2 * i] * scale, y[2 * i + 1] * scale);
                            bf16* dst = a.out + (int64_t)out_row * a.out_row + (int64_t)head * a.out_head;
                            *reinterpret_cast<uint4*>(dst + x0) = make_uint4(w[0], w[1], w[2], w[3]);
                            *reinterpret_cast<uint4*>(dst + x0 + 8) = make_uint4(w[4], w[5], w[6], w[7]);
                        } else {
#pragma unroll
                            for (int i = 0; i < 16; i += 4) *reinterpret_cast<float4*>(a.part_o + (part + in) * c.vdim + x0 + i) = make_float4(y[i], y[i + 1], y[i + 2], y[i + 3]);
                        }
                    }
                if constexpr (JOINS) {
                    asm volatile("bar.sync 1, 128;" ::: "memory");
                    const int pieces = (upto - x1) >> 2;  // of four columns
                    for (int i = row; i < sh.heads * sh.tile_rows * pieces; i += 128) {
                        const int r = i / pieces, d = i % pieces * 4, jr = j0 + r / sh.heads, hr = h0 + r % sh.heads;
                        if (jr >= s.seq.rows || hr >= sh.per) continue;
                        float4 y = *reinterpret_cast<const float4*>(join_s + r * TA_JOIN + d);
#pragma unroll
                        for (int k = 1; k < COPIES; ++k) {
                            const float4 z = *reinterpret_cast<const float4*>(join_s + (k * T::ROWS + r) * TA_JOIN + d);
                            y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
                        }
                        const float f = scale_s[r];
                        *reinterpret_cast<uint2*>(a.out + (int64_t)(s.seq.row0 + jr) * a.out_row + (int64_t)(s.g * sh.per + hr) * a.out_head + x1 + d) =
                            make_uint2(pack_bf16(y.x * f, y.y * f), pack_bf16(y.z * f, y.w * f));
                    }
                    if (upto < c.vdim) asm volatile("bar.sync 1, 128;" ::: "memory");  // before the next columns
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(o_free + t);
                if (both) mbar_arrive(o_free + 1);
            }
        }
        if (!ok) {
            fail = 1;
            if (lane == 0) raise_status(a.status, GLMB_STATUS_WAIT_TIMEOUT);
            if (MODE != TA_SINGLE || t == 0) tree_lost<MODE, COPIES, JOINS>(a, sh, walk, s, t, quarter * 32 + lane);
        }
        if (sh.whole && a.clear_rest)  // there is no second launch
            for (int r = blockIdx.x * 8 + warp; r < a.rows; r += gridDim.x * 8) {
                const TreeRow of = tree_row(a, sh, r, lane);
                if (!of.mine)
                    for (int i = lane; i < a.H * (c.vdim >> 3); i += 32)
                        *reinterpret_cast<uint4*>(a.out + (int64_t)r * a.out_row + (int64_t)(i / (c.vdim >> 3)) * a.out_head + i % (c.vdim >> 3) * 8) = make_uint4(0, 0, 0, 0);
            }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 8) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Joins the sums that several runs or copies left of a row's heads, or clears the row where it belongs to no sequence.  A warp a head, sixteen sums and their
// scales on their way at once: with few rows its latency is its cost, with many the search for the row's sequence, which a CTA does once for its heads.
// grid (rows, parts of the heads).
__global__ void __launch_bounds__(256, 2) tree_merge_kernel(const __grid_constant__ TreeAttentionArgs a, const __grid_constant__ TreeShape sh) {
    GLMB_PDL_PROLOGUE();
    constexpr int BATCH = 16;
    const PagedArgs& c = a.cache;
    const int lane = threadIdx.x & 31, row = blockIdx.x, h0 = blockIdx.y * 8 + (threadIdx.x >> 5), step = gridDim.y * 8;
    const TreeRow of = tree_row(a, sh, row, lane);
    bf16* dst = a.out + (int64_t)row * a.out_row;
    if (!of.mine) {
        if (a.clear_rest)
            for (int h = h0; h < a.H; h += step)
                for (int d = lane * 8; d < c.vdim; d += 256) *reinterpret_cast<uint4*>(dst + (int64_t)h * a.out_head + d) = make_uint4(0, 0, 0, 0);
        return;
    }
    const int64_t share = (of.total + sh.ctas - 1) / sh.ctas;
    const int j = of.j, places = sh.places(of.seq), units = sh.units(of.seq.rows), row_block = j / sh.tile_rows * sh.head_blocks;
    const int rows_of = sh.heads * sh.tile_rows, segment = sh.in_unit * sh.copies * rows_of, shift = sh.copies == 4 ? 2 : sh.copies - 1;
    auto offset = [&](int k) { return (k >> shift) * segment + (k & (sh.copies - 1)) * rows_of; };  // places of the k-th sum behind the first
    for (int h = h0; h < a.H; h += step) {
        const int g = h / sh.per, hh = h % sh.per, tile = row_block + hh / sh.heads, unit = tile / sh.in_unit;
        const int64_t from = of.upto - (int64_t)places * units * c.G + ((int64_t)g * units + unit) * places;
        const int first = (int)((from + sh.start) / share), last = (int)((from + places - 1) / share), parts = (last - first + 1) * sh.copies;  // CTAs with keys of the unit
        if (parts == 1) continue;  // written already
        const int64_t place = sh.part(((int64_t)of.b * c.G + g) * sh.units_max + unit + first, tile % sh.in_unit, 0) + j % sh.tile_rows * sh.heads + hh % sh.heads;
        const float* part_ml = a.part_ml + place * 2;
        const float* part_o = a.part_o + place * c.vdim;
#pragma unroll 1
        for (int d = lane * 4; d - lane * 4 < c.vdim; d += 128) {
            float m = a.sink ? a.sink[h] * TA_LOG2E : -INFINITY, l = m == -INFINITY ? 0.f : 1.f;  // the same in every lane
            float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
            for (int k0 = 0; k0 < parts; k0 += BATCH) {
                float4 v[BATCH];
#pragma unroll
                for (int u = 0; u < BATCH; ++u) {
                    v[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (k0 + u < parts && d < c.vdim) v[u] = *reinterpret_cast<const float4*>(part_o + offset(k0 + u) * c.vdim + d);
                }
                float2 ml = make_float2(-INFINITY, 0.f);
                if (lane < BATCH && k0 + lane < parts) ml = *reinterpret_cast<const float2*>(part_ml + offset(k0 + lane) * 2);
                const float next = fmaxf(m, warp_max(ml.x)), fix = m == next ? 1.f : ta_exp2(m - next);
                const float w = ml.x == -INFINITY && ml.y == 0.f ? 0.f : ml.x == next ? 1.f : ta_exp2(ml.x - next);  // saw nothing there: zeros
                m = next;
                l = l * fix + warp_sum(w == 0.f ? 0.f : ml.y * w);
                o = make_float4(o.x * fix, o.y * fix, o.z * fix, o.w * fix);
#pragma unroll
                for (int u = 0; u < BATCH; ++u) {
                    const float wu = __shfl_sync(0xffffffffu, w, u);
                    o.x = fmaf(wu, v[u].x, o.x), o.y = fmaf(wu, v[u].y, o.y), o.z = fmaf(wu, v[u].z, o.z), o.w = fmaf(wu, v[u].w, o.w);
                }
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            if (d < c.vdim) *reinterpret_cast<uint2*>(dst + (int64_t)h * a.out_head + d) = make_uint2(pack_bf16(o.x * inv, o.y * inv), pack_bf16(o.z * inv, o.w * inv));
        }
    }
}

// ---- host side ----------------------------------------------------------------------------------------------
static TreeShape tree_shape(const TreeAttentionArgs& a, int& mode) {
    TreeShape sh;
    sh.per = a.H / a.cache.G;
    sh.heads = sh.per < 128 ? sh.per : 128;
    sh.head_blocks = ceil_div(sh.per, sh.heads);
    sh.tile_rows = min(128 / sh.heads, a.max_rows);
    const int tiles = ceil_div(a.max_rows, sh.tile_rows) * sh.head_blocks;
    mode = a.cache.dim > 128 || a.cache.vdim > 128 ? TA_WIDE : tiles > 1 ? TA_PAIR : TA_SINGLE;
    sh.in_unit = mode == TA_PAIR ? 2 : 1;
    sh.keys = mode == TA_WIDE ? 64 : 128;
    sh.ctas = 148;
    sh.units_max = ceil_div(tiles, sh.in_unit);
    const int tile = sh.heads * sh.tile_rows;
    sh.copies = mode == TA_PAIR || tile > 64 ? 1 : tile > 32 || mode == TA_WIDE ? 2 : 4;
    sh.whole = (int64_t)a.cache.per_seq * a.cache.page <= TA_WHOLE_BLOCKS * sh.keys;
    if (sh.whole && mode == TA_WIDE) sh.copies = 1;  // no room to join copies in
    // A CTA that goes on from one unit to the next spends some 5 - 7 us on it, four blocks' time: its run is shorter for that.  (48 sequences of up to 8 drafts
    // 151.5 -> 146.8 us; with weights of one piece 4 x 64 drafts at 30,000 165 -> 156 and 1 x 60 at 131,000 295 -> 290.5.  Runs of few blocks would get longer: there
    // it counts nothing.)  By the table's width: the host does not know the lengths.
    sh.start = !sh.whole && (int64_t)a.cache.per_seq * a.cache.page / sh.keys * a.cache.seqs * a.cache.G * sh.units_max >= TA_LONG_RUN * sh.ctas ? TA_START : 0;
    return sh;
}
// Sums that all segments may leave: one for each unit and one more for each CTA.
static int64_t tree_parts(const TreeAttentionArgs& a, const TreeShape& sh) {
    return sh.whole ? 0 : ((int64_t)a.cache.seqs * a.cache.G * sh.units_max + sh.ctas) * sh.in_unit * sh.copies * sh.heads * sh.tile_rows;
}
static int tree_refuses(const TreeAttentionArgs& a) {
    const PagedArgs& c = a.cache;
    return a.rows < 0 || c.G < 1 || a.H < 1 || a.H % c.G || c.dim < 16 || c.dim > 256 || c.dim % 16 || c.vdim < 16 || c.vdim > 256 || c.vdim % 16 || c.page < 8 || c.page % 8 ||
           a.max_rows < 1 || a.max_rows > TA_MAX_DRAFTS || c.seqs < 0 || c.pages < 1 || !(a.scale > 0.f) || (int64_t)c.per_seq * c.page > 0x7fffff00;
}

static int tree_pool_map(CUtensorMap* map, const void* base, const PagedArgs& c, int width, int64_t page, int64_t slot, int64_t head, int rows, int& slots_first) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return 1;
    slots_first = slot < head;  // the smaller stride first
    const cuuint64_t dims[4] = {(cuuint64_t)width, (cuuint64_t)(slots_first ? c.page : c.G), (cuuint64_t)(slots_first ? c.G : c.page), (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)(slots_first ? slot : head) * 2, (cuuint64_t)(slots_first ? head : slot) * 2, (cuuint64_t)page * 2};
    const cuuint32_t box[4] = {64, (cuuint32_t)(slots_first ? rows : 1), (cuuint32_t)(slots_first ? 1 : rows), 1}, elem[4] = {1, 1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : 2;
}
static int tree_query_map(CUtensorMap* map, const TreeAttentionArgs& a, const TreeShape& sh) {
    EncodeTiledFn fn = encode_tiled();
    if (!fn) return 1;
    const cuuint64_t dims[3] = {(cuuint64_t)a.cache.dim, (cuuint64_t)a.H, (cuuint64_t)a.rows}, strides[2] = {(cuuint64_t)a.q_head * 2, (cuuint64_t)a.q_row * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)sh.heads, (cuuint32_t)sh.tile_rows}, elem[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<bf16*>(a.q), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS ? 0 : 2;
}

template <int MODE, int COPIES, bool JOINS>
static int tree_launch(const TreeAttentionArgs& a, const TreeShape& sh, cudaStream_t stream) {
    typedef TreeMode<MODE, COPIES, JOINS> T;
    int chunk = 8;  // slots that lie in one page wherever a block begins
    while (chunk < T::KEYS && a.cache.page % (2 * chunk) == 0) chunk *= 2;
    const PagedArgs& c = a.cache;
    CUtensorMap map_q, map_k, map_v;
    int first_k, first_v;
    if (tree_query_map(&map_q, a, sh) || tree_pool_map(&map_k, c.k, c, c.dim, c.k_page, c.k_slot, c.k_head, chunk, first_k) ||
        tree_pool_map(&map_v, c.v, c, c.vdim, c.v_page, c.v_slot, c.v_head, chunk, first_v))
        return 3;
    static DeviceOnce once;
    const int dev = once.pending();
    if (dev != DeviceOnce::SET) {
        const cudaError_t e = cudaFuncSetAttribute((const void*)tree_attention_kernel<MODE, COPIES, JOINS>, cudaFuncAttributeMaxDynamicSharedMemorySize, T::SMEM);
        if (e != cudaSuccess) return (int)e;
        once.mark(dev);
    }
    GLMB_LAUNCH((tree_attention_kernel<MODE, COPIES, JOINS>), sh.ctas, T::THREADS, T::SMEM, stream, map_q, map_k, map_v, a, sh, first_k, first_v, chunk);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess || sh.whole) return (int)e;
    const int heads_at_once = min(ceil_div(a.H, 8), ceil_div(148 * 2, a.rows));
    GLMB_LAUNCH(tree_merge_kernel, dim3(a.rows, heads_at_once), 256, 0, stream, a, sh);
    return (int)cudaGetLastError();
}

GLMB_API size_t glmb_tree_attention_args_sizeof() { return sizeof(TreeAttentionArgs); }

// Sums that a call needs room for: each vdim + 2 floats; -1: the call is refused.
GLMB_API int64_t glmb_tree_attention_parts(const TreeAttentionArgs* args) {
    if (tree_refuses(*args)) return -1;
    int mode;
    const TreeShape sh = tree_shape(*args, mode);
    return tree_parts(*args, sh);
}

GLMB_API int glmb_tree_attention(const TreeAttentionArgs* args, cudaStream_t stream) {
    const TreeAttentionArgs a = *args;
    if (tree_refuses(a)) return 1;
    if (a.cache.seqs == 0 || a.rows == 0) return 0;
    int mode;
    const TreeShape sh = tree_shape(a, mode);
    if (a.parts < tree_parts(a, sh) || (!sh.whole && (!a.part_o || !a.part_ml))) return 1;
    if (mode == TA_PAIR) return tree_launch<TA_PAIR, 1, false>(a, sh, stream);
    if (mode == TA_WIDE) return sh.copies == 1 ? tree_launch<TA_WIDE, 1, false>(a, sh, stream) : tree_launch<TA_WIDE, 2, false>(a, sh, stream);
    if (sh.copies == 1) return tree_launch<TA_SINGLE, 1, false>(a, sh, stream);
    if (sh.copies == 2) return sh.whole ? tree_launch<TA_SINGLE, 2, true>(a, sh, stream) : tree_launch<TA_SINGLE, 2, false>(a, sh, stream);
    return sh.whole ? tree_launch<TA_SINGLE, 4, true>(a, sh, stream) : tree_launch<TA_SINGLE, 4, false>(a, sh, stream);
}

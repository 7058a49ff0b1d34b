// Attention of a few drafted tokens per sequence over a paged cache (bf16; scores, softmax and sums fp32).
//
// Row j of a sequence, whose committed tokens lie in slots 0 .. length - 1 and whose drafted tokens in slots length, length + 1, ..:
//
//   o = sum_i p_i v_i,   p_i = e^(scale q . k_i) / (sum e^(scale q . k) + e^sink)
//
// over every committed slot and the drafted slots t (those of this call's rows) with bit t of the row's mask: its ancestors in the tree and itself.
// What a row does not attend to is never multiplied, so NaN there stays there.  Nothing attended: zeros.  A slot whose page the table does not know
// counts as not attended and raises GLMB_STATUS_BAD_INDEX, as does a sequence whose rows or length are out of range.
#include "paged.cuh"
#include "vec8.cuh"

#define TA_LOG2E 1.4426950408889634f
#define TA_MAX_DRAFTS 64  // bits of a mask

// Rows and committed slots of a sequence, within what there is.
struct TreeSeq { int row0, rows, length; };
__device__ __forceinline__ TreeSeq tree_seq(const TreeAttentionArgs& a, int b, bool report) {
    TreeSeq s;
    const int from = a.starts[b], to = a.starts[b + 1], length = a.lengths[b];
    s.row0 = min(max(from, 0), a.rows);
    s.rows = max(min(to, a.rows) - s.row0, 0);
    s.length = min(max(length, 0), a.cache.per_seq * a.cache.page);
    if (report && (from != s.row0 || to < from || to > a.rows || s.rows > a.max_rows || s.length != length)) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
    return s;
}

// grid (heads, max_rows, sequences); a warp takes every fourth key.
__global__ void __launch_bounds__(128) tree_attention_kernel(TreeAttentionArgs a) {
    GLMB_PDL_PROLOGUE();
    __shared__ float o_s[4][256], ml_s[4][2];
    const int h = blockIdx.x, j = blockIdx.y, b = blockIdx.z, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedArgs& c = a.cache;
    const TreeSeq seq = tree_seq(a, b, h == 0 && j == 0 && threadIdx.x == 0);
    if (a.clear_rest && j == 0) {
        const int last = b + 1 == c.seqs ? a.rows : seq.row0 + seq.rows, first = seq.row0 + min(seq.rows, a.max_rows);
        for (int r = b == 0 ? 0 : first; r < last; ++r)
            if (r < seq.row0 || r >= first)
                for (int d = threadIdx.x; d < c.vdim; d += 128) a.out[(int64_t)r * a.out_row + (int64_t)h * a.out_head + d] = __float2bfloat16_rn(0.f);
    }
    if (j >= seq.rows) return;
    const int row = seq.row0 + j, g = h / (a.H / c.G), drafts = min(seq.rows, min(a.max_rows, TA_MAX_DRAFTS));
    const int64_t mask = a.masks[row];
    const bf16* q = a.q + (int64_t)row * a.q_row + (int64_t)h * a.q_head;
    float qv[8], o[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        qv[i] = lane + 32 * i < c.dim ? to_f32(q[lane + 32 * i]) : 0.f;
        o[i] = 0.f;
    }
    const float scale2 = a.scale * TA_LOG2E;
    float m = -INFINITY, l = 0.f;
    for (int s = warp; s < seq.length + drafts; s += 4) {
        if (s >= seq.length && !((mask >> (s - seq.length)) & 1)) continue;
        const int page = paged_page(c, b, s);
        if (page < 0) {
            if (lane == 0) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
            continue;
        }
        const bf16* k = c.k + page * c.k_page + (s % c.page) * c.k_slot + g * c.k_head;
        const bf16* v = c.v + page * c.v_page + (s % c.page) * c.v_slot + g * c.v_head;
        float dot = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < c.dim) dot = fmaf(qv[i], to_f32(k[lane + 32 * i]), dot);
        const float x = warp_sum(dot) * scale2, next = fmaxf(m, x);
        const float fix = m == next ? 1.f : exp2f(m - next), p = exp2f(x - next);
        m = next;
        l = l * fix + p;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (lane + 32 * i < c.vdim) o[i] = o[i] * fix + p * to_f32(v[lane + 32 * i]);
    }
    if (lane == 0) ml_s[warp][0] = m, ml_s[warp][1] = l;
    for (int i = 0; i < 8; ++i) o_s[warp][lane + 32 * i] = o[i];
    __syncthreads();
    const float sink2 = a.sink ? a.sink[h] * TA_LOG2E : -INFINITY;
    float top = sink2, total = 0.f, f[4];
    for (int w = 0; w < 4; ++w) top = fmaxf(top, ml_s[w][0]);
    for (int w = 0; w < 4; ++w) {
        f[w] = ml_s[w][1] == 0.f ? 0.f : exp2f(ml_s[w][0] - top);
        total += f[w] * ml_s[w][1];
    }
    if (a.sink) total += exp2f(sink2 - top);
    for (int d = threadIdx.x; d < c.vdim; d += 128) {
        float sum = 0.f;
        for (int w = 0; w < 4; ++w)
            if (f[w] != 0.f) sum += f[w] * o_s[w][d];
        a.out[(int64_t)row * a.out_row + (int64_t)h * a.out_head + d] = __float2bfloat16_rn(total == 0.f ? 0.f : sum / total);
    }
}

GLMB_API size_t glmb_tree_attention_args_sizeof() { return sizeof(TreeAttentionArgs); }

GLMB_API int glmb_tree_attention(const TreeAttentionArgs* args, cudaStream_t stream) {
    const TreeAttentionArgs a = *args;
    const PagedArgs& c = a.cache;
    if (a.rows < 0 || c.G < 1 || a.H < 1 || a.H % c.G || c.dim < 16 || c.dim > 256 || c.dim % 16 || c.vdim < 16 || c.vdim > 256 || c.vdim % 16 || c.page < 1 ||
        a.max_rows < 1 || a.max_rows > TA_MAX_DRAFTS || c.seqs < 0 || c.seqs > 65535 || (int64_t)c.per_seq * c.page > 0x7fffff00)
        return 1;
    if (c.seqs == 0 || a.rows == 0) return 0;
    GLMB_LAUNCH(tree_attention_kernel, dim3(a.H, a.max_rows, c.seqs), 128, 0, stream, a);
    return (int)cudaGetLastError();
}

// Rows of a fused q | k | v projection on their way to attention over a paged cache, one launch:
//
//   n = x rsqrt(mean(x^2) + eps) w            per head of q and k, where weights are given
//   (a, b) -> (a cos - b sin, a sin + b cos)  on the leading rot channels of q and k; (a, b) are channels (d, d + rot / 2), or (2 j, 2 j + 1)
//   k, v -> slot of the sequence, q -> a buffer
//
// fp32 between the bf16 row and the one rounding of the result.  A row whose slot is negative stores no key and value.  A sequence, slot, table entry
// or position out of range raises GLMB_STATUS_BAD_INDEX, the row stores nothing in the cache, and its queries are zeros.
#include "paged.cuh"
#include "vec8.cuh"

// One warp per (row, head).
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppendArgs a) {
    GLMB_PDL_PROLOGUE();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.H + 2 * a.cache.G;
    const int64_t unit = (int64_t)blockIdx.x * 8 + warp;
    if (unit >= (int64_t)a.rows * heads) return;
    const int row = (int)(unit / heads), h = (int)(unit % heads);
    const int kind = h < a.H ? 0 : h < a.H + a.cache.G ? 1 : 2, head = kind == 0 ? h : kind == 1 ? h - a.H : h - a.H - a.cache.G;
    const int dim = kind == 2 ? a.cache.vdim : a.cache.dim;
    if (kind == 0 && !a.q) return;
    const int pos = a.rot ? a.positions[row] : 0, slot = a.slots[row], seq = a.row_seq[row];
    bool bad = pos < 0 || (a.rot && pos >= a.rot_rows);
    int page = -1;
    if (slot >= 0) {
        if (seq >= 0 && seq < a.cache.seqs) page = paged_page(a.cache, seq, slot);
        bad |= page < 0;
    }
    if (bad && lane == 0) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
    bf16* dst;
    if (kind == 0) {
        dst = a.q + (int64_t)row * a.q_stride + (int64_t)head * dim;
    } else {
        if (bad || slot < 0) return;
        const int in = slot % a.cache.page;
        dst = kind == 1 ? a.cache.k + page * a.cache.k_page + in * a.cache.k_slot + head * a.cache.k_head
                        : a.cache.v + page * a.cache.v_page + in * a.cache.v_slot + head * a.cache.v_head;
    }
    const bf16* src = a.qkv + (int64_t)row * a.qkv_stride + (kind == 2 ? (int64_t)(a.H + a.cache.G) * a.cache.dim + (int64_t)head * dim : (int64_t)h * dim);
    const bf16* w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    const float2* rot = kind < 2 && a.rot && !bad ? a.rot + (int64_t)pos * (a.rot_dims / 2) : nullptr;
    float inv = 1.f;
    if (w) {
        float sum = 0.f;
        for (int d = lane; d < dim; d += 32) {
            const float x = to_f32(src[d]);
            sum = fmaf(x, x, sum);
        }
        inv = 1.0f / sqrtf(warp_sum(sum) / dim + a.eps);
    }
    const int half = a.rot_dims / 2;
    for (int d = lane; d < dim; d += 32) {
        auto value = [&](int i) { return to_f32(src[i]) * (w ? inv * to_f32(w[i]) : 1.f); };
        float y = value(d);
        if (rot && d < a.rot_dims) {
            const bool second = a.pairs ? d & 1 : d >= half;
            const int other = a.pairs ? d ^ 1 : second ? d - half : d + half;
            const float2 cs = rot[a.pairs ? d >> 1 : second ? d - half : d];
            y = second ? value(other) * cs.y + y * cs.x : y * cs.x - value(other) * cs.y;
        }
        dst[d] = __float2bfloat16_rn(bad ? 0.f : y);
    }
}

GLMB_API size_t glmb_paged_append_args_sizeof() { return sizeof(PagedAppendArgs); }

GLMB_API int glmb_paged_append(const PagedAppendArgs* args, cudaStream_t stream) {
    const PagedAppendArgs a = *args;
    if (a.rows < 0 || a.H < 0 || a.cache.G < 1 || a.cache.dim < 1 || a.cache.vdim < 1 || a.cache.page < 1 || a.rot_dims < 0 || (a.rot_dims & 1) ||
        a.rot_dims > a.cache.dim)
        return 1;
    const int64_t blocks = ((int64_t)a.rows * (a.H + 2 * a.cache.G) + 7) / 8;
    if (blocks > 0x7fffffff) return 1;
    if (blocks == 0) return 0;
    GLMB_LAUNCH(paged_append_kernel, (unsigned)blocks, 256, 0, stream, a);
    return (int)cudaGetLastError();
}

// Rows of a fused q | k | v projection on their way to attention over a paged cache, one launch:
//
//   n = x rsqrt(mean(x^2) + eps) w            per head of q and k, where weights are given
//   (a, b) -> (a cos - b sin, a sin + b cos)  on the leading rot channels of q and k; (a, b) are channels (d, d + rot / 2), or (2 j, 2 j + 1)
//   k, v -> slot of the sequence, q -> a buffer
//
// fp32 between the bf16 row and the one rounding of the result.  A row whose slot is negative stores no key and value.  A sequence, slot, table entry
// or position out of range raises GLMB_STATUS_BAD_INDEX, the row stores nothing in the cache, and its queries are zeros.
//
// A thread has eight channels (16 bytes) of a head, the next power of two of threads a head, and keeps the same channels for every head that it takes: the
// row's angles and the norm's weights are read once.  Halves of a rotation change places by shuffles.
#include "paged.cuh"
#include "vec8.cuh"

#define PA_THREADS 256
#define PA_UNROLL 2  // heads of a thread on their way

// grid (rows, parts of a row); `width`: threads a head (a power of two).
__global__ void __launch_bounds__(PA_THREADS, 4) paged_append_kernel(PagedAppendArgs a, int width) {
    GLMB_PDL_PROLOGUE();
    const PagedArgs& c = a.cache;
    const int row = blockIdx.x, lane = threadIdx.x & 31, mine = threadIdx.x & (width - 1), vectors = c.dim >> 3;
    const int at_once = PA_THREADS / width, first = (a.q ? 0 : a.H) + threadIdx.x / width, heads = a.H + c.G, step = at_once * gridDim.y;
    const bool live = mine < vectors;
    const bf16* src = a.qkv + (int64_t)row * a.qkv_stride;
    auto load = [&](int h) { return live && h < heads ? ld_stream16(src + (int64_t)h * c.dim + mine * 8) : make_uint4(0, 0, 0, 0); };
    uint4 raw[PA_UNROLL];
#pragma unroll
    for (int u = 0; u < PA_UNROLL; ++u) raw[u] = load(first + (int)blockIdx.y * at_once + u * step);  // on their way before the row's place is known

    const int pos = a.rot ? a.positions[row] : 0, slot = a.slots[row], seq = a.row_seq[row];
    bool bad = pos < 0 || (a.rot && pos >= a.rot_rows);
    int page = -1;
    if (slot >= 0) {
        if (seq >= 0 && seq < c.seqs) page = paged_page(c, seq, slot);
        bad |= page < 0;
    }
    if (bad && threadIdx.x == 0 && blockIdx.y == 0) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
    const bool stores = !bad && slot >= 0;
    const int in = slot >= 0 ? slot % c.page : 0;

    const int half = a.rot && !bad ? a.rot_dims >> 1 : 0, hv = half >> 3;
    const bool swap = half && !a.pairs && !(half & 7);  // halves whose vectors pair up
    const float2* rot = a.rot + (int64_t)(bad ? 0 : pos) * (a.rot_dims >> 1);
    float2 cs[8];  // of this thread's channels: of each, or (pairs) of every second
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        cs[e] = make_float2(1.f, 0.f);
        if (!live) continue;
        const int d = mine * 8 + e;
        if (a.pairs ? e < 4 && mine * 4 + e < half : d < 2 * half) cs[e] = rot[a.pairs ? mine * 4 + e : d < half ? d : d - half];
    }
    const uint4 ones = make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
    const uint4 wq = live && a.q_norm ? ld_hot16(a.q_norm + mine * 8) : ones, wk = live && a.k_norm ? ld_hot16(a.k_norm + mine * 8) : ones;
    const int partner = (lane & ~(width - 1)) | (mine < hv ? mine + hv : mine < 2 * hv ? mine - hv : mine);  // the thread with the other half

    for (int h0 = first + (int)blockIdx.y * at_once; h0 - threadIdx.x / width < heads; h0 += PA_UNROLL * step) {  // the same number of times for every thread
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) {
            const int h = h0 + u * step;
            if (h - (int)threadIdx.x / width >= heads) break;
            const bool is_q = h < a.H;
            float x[8] = {bf16_lo(raw[u].x), bf16_hi(raw[u].x), bf16_lo(raw[u].y), bf16_hi(raw[u].y), bf16_lo(raw[u].z), bf16_hi(raw[u].z), bf16_lo(raw[u].w), bf16_hi(raw[u].w)};
            float inv = 1.f;
            if (a.q_norm || a.k_norm) {
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < 8; ++e) sum = fmaf(x[e], x[e], sum);
                for (int o = width >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (is_q ? a.q_norm : a.k_norm) inv = rsqrtf(sum / c.dim + a.eps);
            }
            const uint4 w4 = is_q ? wq : wk;
            const float w8[8] = {bf16_lo(w4.x), bf16_hi(w4.x), bf16_lo(w4.y), bf16_hi(w4.y), bf16_lo(w4.z), bf16_hi(w4.z), bf16_lo(w4.w), bf16_hi(w4.w)};
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] *= inv * w8[e];
            if (swap) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float other = __shfl_sync(0xffffffffu, x[e], partner);
                    x[e] = mine < hv ? x[e] * cs[e].x - other * cs[e].y : other * cs[e].y + x[e] * cs[e].x;
                }
            } else if (half && a.pairs) {
#pragma unroll
                for (int e = 0; e < 8; e += 2) {
                    const float p = x[e], q = x[e + 1];
                    x[e] = p * cs[e >> 1].x - q * cs[e >> 1].y;
                    x[e + 1] = p * cs[e >> 1].y + q * cs[e >> 1].x;
                }
            } else if (half && live && h < heads) {  // halves that begin inside a vector: the other channel is read again
                const bf16* head = src + (int64_t)h * c.dim;
                const bf16* w = is_q ? a.q_norm : a.k_norm;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int d = mine * 8 + e;
                    if (d >= 2 * half) continue;
                    const int o = d < half ? d + half : d - half;
                    const float other = to_f32(head[o]) * (inv * (w ? to_f32(w[o]) : 1.f));
                    x[e] = d < half ? x[e] * cs[e].x - other * cs[e].y : other * cs[e].y + x[e] * cs[e].x;
                }
            }
            if (live && h < heads) {
                if (is_q) {
                    if (bad)
#pragma unroll
                        for (int e = 0; e < 8; ++e) x[e] = 0.f;
                    store8(a.q + (int64_t)row * a.q_stride + (int64_t)h * c.dim + mine * 8, x);
                } else if (stores) {
                    store8(c.k + page * c.k_page + in * c.k_slot + (h - a.H) * c.k_head + mine * 8, x);
                }
            }
        }
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) raw[u] = load(h0 + (PA_UNROLL + u) * step);
    }
    if (!stores) return;
    const int pieces = c.vdim >> 3;
    for (int i = threadIdx.x + (int)blockIdx.y * PA_THREADS; i < c.G * pieces; i += PA_THREADS * gridDim.y) {
        const int g = i / pieces, d = i % pieces * 8;
        *reinterpret_cast<uint4*>(c.v + page * c.v_page + in * c.v_slot + g * c.v_head + d) = ld_stream16(src + (int64_t)heads * c.dim + (int64_t)g * c.vdim + d);
    }
}

GLMB_API size_t glmb_paged_append_args_sizeof() { return sizeof(PagedAppendArgs); }

GLMB_API int glmb_paged_append(const PagedAppendArgs* args, cudaStream_t stream) {
    const PagedAppendArgs a = *args;
    const PagedArgs& c = a.cache;
    if (a.rows < 0 || a.H < 0 || c.G < 1 || c.dim < 8 || c.dim > 256 || c.dim % 8 || c.vdim < 8 || c.vdim % 8 || c.page < 1 || a.rot_dims < 0 || (a.rot_dims & 1) ||
        a.rot_dims > c.dim)
        return 1;
    if (a.rows == 0) return 0;
    int width = 1;
    while (width < c.dim / 8) width *= 2;
    // a row is dealt to several CTAs while there are fewer rows than four for each SM
    const int passes = ceil_div(a.H + c.G, PA_THREADS / width), parts = min(min(passes, ceil_div(148 * 4, a.rows)), 65535);
    GLMB_LAUNCH(paged_append_kernel, dim3(a.rows, parts), PA_THREADS, 0, stream, a, width);
    return (int)cudaGetLastError();
}

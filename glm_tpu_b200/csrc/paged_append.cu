// Rows of a fused q | k | v projection on their way to attention over a paged cache, one launch:
//
//   n = x rsqrt(mean(x^2) + eps) w            per head of q and k, where weights are given
//   (a, b) -> (a cos - b sin, a sin + b cos)  on the leading rot channels of q and k; (a, b) are channels (d, d + rot / 2), or (2 j, 2 j + 1)
//   k, v -> slot of the sequence, q -> a buffer
//
// fp32 between the bf16 row and the one rounding of the result.  A row whose slot is negative stores no key and value.  A sequence, slot, table entry
// or position out of range raises GLMB_STATUS_BAD_INDEX, the row stores nothing in the cache, and its queries are zeros.
//
// A thread has eight channels (16 bytes) of a head, WIDTH (a power of two) threads a head, and keeps the same channels for every head that it takes:
// weights and angles become two factors a channel, once for the row's q and once for its k, so that a normalized head costs two packed instructions for a
// pair of channels.  Of a rotation by halves a thread has four channels and the four that they turn with, so that nothing is exchanged.  The first heads and
// values are on their way before the row's place in the cache is known.  8,191 rows of 64 + 8 + 8 heads of 128: turned by pairs 69.5 us, 4.8 TB/s, by
// halves 68.6, neither norm nor turn 56, by odd halves (90 channels; their partners are read once more) 157.  Bound: what a row costs before its heads do.  A CTA of 64 threads takes 18 rounds of heads with the same factors (256
// threads and 5 rounds 78; 128 threads 71.5), 16 of them an SM (20, with fewer registers: 83); the angles' loads go out with the table's and wait for no
// branch (behind the page's 85).  Rows in turn, the next one's place looked up ahead, 94; a ring of bulk copies 192.
#include "paged.cuh"
#include "vec8.cuh"

#define PA_THREADS 64

enum { PA_PLAIN = 0, PA_PAIRS = 1, PA_HALVES = 2, PA_ODD_HALVES = 3 };  // odd: halves that are no multiple of four channels

__device__ __forceinline__ uint2 ld_stream8(const void* p) {
    uint2 v;
    asm volatile("ld.global.nc.L1::no_allocate.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// What a thread does with its channels of a head: y = n own + n' other, n' being the channel that n turns with.
template <int WIDTH, int TURN>
struct AppendFactors {
    float2 own[4], other[TURN == PA_PLAIN ? 1 : 4];
    int first, second, half, turns;  // the thread's channels: four from `first` on, and four from `second` on; how many of the eight turn
    bool live, norm;
    float eps, inv_dim;

    __device__ __forceinline__ void place(int thread, int dim, int rot_dims) {
        half = rot_dims >> 1, live = thread * 8 < dim;
        first = thread * 8, second = first + 4;
        turns = live ? min(max(rot_dims - first, 0), 8) : 0;
        if (TURN == PA_HALVES && turns) first = thread * 4, second = half + first;
    }
    __device__ __forceinline__ bool turned(int e) const { return e < turns; }
    __device__ __forceinline__ uint4 load(const bf16* head) const {
        if (TURN != PA_HALVES) return ld_stream16(head + first);
        const uint2 a = ld_stream8(head + first), b = ld_stream8(head + second);
        return make_uint4(a.x, a.y, b.x, b.y);
    }
    __device__ __forceinline__ void store(bf16* head, const uint4& y) const {
        if (TURN == PA_HALVES) *reinterpret_cast<uint2*>(head + first) = make_uint2(y.x, y.y), *reinterpret_cast<uint2*>(head + second) = make_uint2(y.z, y.w);
        else *reinterpret_cast<uint4*>(head + first) = y;
    }

    // Two channels a register pair: neighbours, or (pairs that turn) even ones in x[0], x[1] and the odd ones that they turn with in x[2], x[3]
    static __device__ __forceinline__ void widen(const uint4& u, float2 (&x)[4]) {
        if (TURN == PA_PAIRS) {
            x[0] = make_float2(bf16_lo(u.x), bf16_lo(u.y)), x[1] = make_float2(bf16_lo(u.z), bf16_lo(u.w));
            x[2] = make_float2(bf16_hi(u.x), bf16_hi(u.y)), x[3] = make_float2(bf16_hi(u.z), bf16_hi(u.w));
        } else {
            x[0] = make_float2(bf16_lo(u.x), bf16_hi(u.x)), x[1] = make_float2(bf16_lo(u.y), bf16_hi(u.y));
            x[2] = make_float2(bf16_lo(u.z), bf16_hi(u.z)), x[3] = make_float2(bf16_lo(u.w), bf16_hi(u.w));
        }
    }
    static __device__ __forceinline__ uint4 narrow(const float2 (&y)[4]) {
        if (TURN == PA_PAIRS) return make_uint4(pack_bf16(y[0].x, y[2].x), pack_bf16(y[0].y, y[2].y), pack_bf16(y[1].x, y[3].x), pack_bf16(y[1].y, y[3].y));
        return make_uint4(pack_bf16(y[0].x, y[0].y), pack_bf16(y[1].x, y[1].y), pack_bf16(y[2].x, y[2].y), pack_bf16(y[3].x, y[3].y));
    }

    // `weights`: the norm's, or null; `rot`: the row's angles.
    __device__ __forceinline__ void set(const bf16* weights, const float2* rot) {
        norm = weights != nullptr;
        const uint4 u = norm && live ? load(weights) : make_uint4(0x3f803f80u, 0x3f803f80u, 0x3f803f80u, 0x3f803f80u);
        widen(u, own);
        if (TURN == PA_PAIRS || TURN == PA_HALVES) {
            float2 cs[4];
            if (TURN == PA_HALVES) {  // whole groups of four turn, or none; loads that depend on no branch
                const float4* at = reinterpret_cast<const float4*>(rot + (turns ? first : 0));
                const float4 a = at[0], b = at[1];
                cs[0] = make_float2(a.x, a.y), cs[1] = make_float2(a.z, a.w), cs[2] = make_float2(b.x, b.y), cs[3] = make_float2(b.z, b.w);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) cs[e] = rot[min((first >> 1) + e, half - 1)];
            }
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (!turned(2 * e)) cs[e] = make_float2(1.f, 0.f);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float2 w0 = own[e], w1 = own[e + 2], cs0 = cs[2 * e], cs1 = cs[2 * e + 1];
                own[e] = make_float2(w0.x * cs0.x, w0.y * cs1.x), other[e] = make_float2(w1.x * -cs0.y, w1.y * -cs1.y);
                own[e + 2] = make_float2(w1.x * cs0.x, w1.y * cs1.x), other[e + 2] = make_float2(w0.x * cs0.y, w0.y * cs1.y);
            }
        } else if (TURN == PA_ODD_HALVES) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float o[2] = {own[e].x, own[e].y}, t[2] = {0.f, 0.f};
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    if (turned(2 * e + i)) {
                        const int d = first + 2 * e + i;
                        const float2 cs = rot[d < half ? d : d - half];
                        const float w = norm ? to_f32(weights[d < half ? d + half : d - half]) : 1.f;
                        o[i] *= cs.x, t[i] = d < half ? -w * cs.y : w * cs.y;
                    }
                own[e] = make_float2(o[0], o[1]), other[e] = make_float2(t[0], t[1]);
            }
        }
    }

    // One head: what was loaded -> what is stored; the whole warp.  head: where it lies (odd halves read the other channels there, if it `exists`: a warp's last
    // round may have more places than there are heads).
    __device__ __forceinline__ uint4 apply(const uint4& raw, const bf16* head, bool exists) const {
        float2 x[4];
        widen(raw, x);
        float inv = 1.f;
        if (norm) {
            float2 s = __fmul2_rn(x[0], x[0]);
#pragma unroll
            for (int e = 1; e < 4; ++e) s = __ffma2_rn(x[e], x[e], s);
            float sum = s.x + s.y;
#pragma unroll
            for (int o = WIDTH >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = rsqrtf(fmaf(sum, inv_dim, eps));
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __fmul2_rn(x[e], make_float2(inv, inv));
        }
        float2 y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = __fmul2_rn(x[e], own[e]);
        if (TURN == PA_PAIRS || TURN == PA_HALVES) {
            if (turns == 8) {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __ffma2_rn(x[e ^ 2], other[e], y[e]);
            } else if (TURN == PA_PAIRS && turns) {  // what does not turn meets no other channel, whose infinity times zero would be NaN
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (turned(4 * (e & 1))) y[e].x = fmaf(x[e ^ 2].x, other[e].x, y[e].x);
                    if (turned(4 * (e & 1) + 2)) y[e].y = fmaf(x[e ^ 2].y, other[e].y, y[e].y);
                }
            }
        } else if (TURN == PA_ODD_HALVES) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int d = first + 2 * e;
                if (exists && turned(2 * e)) y[e].x = fmaf(to_f32(head[d < half ? d + half : d - half]) * inv, other[e].x, y[e].x);
                if (exists && turned(2 * e + 1)) y[e].y = fmaf(to_f32(head[d + 1 < half ? d + 1 + half : d + 1 - half]) * inv, other[e].y, y[e].y);
            }
        }
        return narrow(y);
    }
};

// grid (rows, parts of a row).
template <int WIDTH, int TURN>
__global__ void __launch_bounds__(PA_THREADS, 16) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
    GLMB_PDL_PROLOGUE();
    constexpr int AT_ONCE = PA_THREADS / WIDTH, UNROLL = TURN == PA_ODD_HALVES ? 2 : 4;  // heads of q of a thread on their way
    const PagedArgs& c = a.cache;
    const int row = blockIdx.x, heads = a.q ? a.H : 0;
    // this thread's heads of q and of k: head0, head0 + step, ..; its warp's first one decides whether the warp has any left
    const int step = AT_ONCE * (int)gridDim.y, head0 = (int)threadIdx.x / WIDTH + AT_ONCE * (int)blockIdx.y, warp0 = (int)(threadIdx.x & ~31u) / WIDTH + AT_ONCE * (int)blockIdx.y;
    AppendFactors<WIDTH, TURN> t;
    t.place(threadIdx.x & (WIDTH - 1), c.dim, TURN == PA_PLAIN ? 0 : a.rot_dims);
    t.eps = a.eps, t.inv_dim = 1.f / c.dim;
    const bf16* src = a.qkv + (int64_t)row * a.qkv_stride;
    const int far = step * c.dim, q_at = head0 * c.dim, k_at = (a.H + head0) * c.dim;  // channels between a thread's heads, and before its first one of q and of k
    const uint4 none = make_uint4(0, 0, 0, 0);
    uint4 raw[UNROLL];
#pragma unroll
    for (int u = 0; u < UNROLL; ++u) raw[u] = t.live && head0 + u * step < heads ? t.load(src + q_at + u * far) : none;
    uint4 key = t.live && head0 < c.G ? t.load(src + k_at) : none;
    const int pieces = c.vdim >> 3, values = c.G * pieces, first_value = (int)(threadIdx.x + blockIdx.y * PA_THREADS);
    const bf16* value_src = src + (a.H + c.G) * c.dim;
    const uint4 value = first_value < values ? ld_stream16(value_src + first_value * 8) : none;

    const int pos = a.rot ? a.positions[row] : 0, slot = a.slots[row], seq = a.row_seq[row];
    const bool bad_pos = pos < 0 || (a.rot && pos >= a.rot_rows);
    const int page = slot >= 0 && seq >= 0 && seq < c.seqs ? paged_page(c, seq, slot) : -1;
    const float2* rot = a.rot + (int64_t)(bad_pos ? 0 : pos) * t.half;
    t.set(a.q ? a.q_norm : a.k_norm, rot);  // its loads go out with the table's
    const bool bad = bad_pos || (slot >= 0 && page < 0);
    bf16* q = a.q + (int64_t)row * a.q_stride;
    if (bad) {
        if (threadIdx.x == 0 && blockIdx.y == 0) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
        for (int h = head0; h < heads; h += step)
            if (t.live) t.store(q + h * c.dim, none);
        return;
    }
    if (warp0 < heads) {
        int h = head0, at = q_at;
        for (int left = (heads - warp0 + step - 1) / step; left > 0; left -= UNROLL) {
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                if (u >= left) break;
                const uint4 y = t.apply(raw[u], src + at, h < heads);
                if (t.live && h < heads) t.store(q + at, y);
                h += step, at += far;
            }
            if (left <= UNROLL) break;
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (t.live && h + u * step < heads) raw[u] = t.load(src + at + u * far);
        }
    }
    if (slot < 0) return;
    const int in = slot % c.page;
    if (warp0 < c.G) {
        if (a.q && a.q_norm != a.k_norm) t.set(a.k_norm, rot);
        bf16* k = c.k + page * c.k_page + in * c.k_slot;
        int h = head0, at = k_at;
        for (int left = (c.G - warp0 + step - 1) / step; left > 0; --left) {
            const uint4 y = t.apply(key, src + at, h < c.G);
            if (t.live && h < c.G) t.store(k + h * c.k_head, y);
            h += step, at += far;
            if (t.live && h < c.G) key = t.load(src + at);
        }
    }
    bf16* v = c.v + page * c.v_page + in * c.v_slot;
    for (int i = first_value; i < values; i += PA_THREADS * (int)gridDim.y)
        *reinterpret_cast<uint4*>(v + i / pieces * c.v_head + i % pieces * 8) = i == first_value ? value : ld_stream16(value_src + i * 8);
}

template <int WIDTH>
static void append_launch(const PagedAppendArgs& a, int turn, cudaStream_t stream) {
    const int at_once = PA_THREADS / WIDTH, rounds = (a.q ? ceil_div(a.H, at_once) : 0) + ceil_div(a.cache.G, at_once);
    // a row is dealt to several CTAs while there are fewer rows than run at once
    const dim3 grid(a.rows, min(rounds, ceil_div(148 * 16, a.rows)));
    if (turn == PA_PLAIN) GLMB_LAUNCH((paged_append_kernel<WIDTH, PA_PLAIN>), grid, PA_THREADS, 0, stream, a);
    else if (turn == PA_PAIRS) GLMB_LAUNCH((paged_append_kernel<WIDTH, PA_PAIRS>), grid, PA_THREADS, 0, stream, a);
    else if (turn == PA_HALVES) GLMB_LAUNCH((paged_append_kernel<WIDTH, PA_HALVES>), grid, PA_THREADS, 0, stream, a);
    else GLMB_LAUNCH((paged_append_kernel<WIDTH, PA_ODD_HALVES>), grid, PA_THREADS, 0, stream, a);
}

GLMB_API size_t glmb_paged_append_args_sizeof() { return sizeof(PagedAppendArgs); }

GLMB_API int glmb_paged_append(const PagedAppendArgs* args, cudaStream_t stream) {
    const PagedAppendArgs a = *args;
    const PagedArgs& c = a.cache;
    if (a.rows < 0 || a.H < 0 || c.G < 1 || c.dim < 8 || c.dim > 256 || c.dim % 8 || c.vdim < 8 || c.vdim % 8 || c.page < 1 || a.rot_dims < 0 || (a.rot_dims & 1) ||
        a.rot_dims > c.dim || (a.rot && a.rot_rows < 1) || (int64_t)(a.H + c.G) * c.dim + (int64_t)c.G * c.vdim > 1 << 30)
        return 1;
    if (a.rows == 0) return 0;
    const int turn = !a.rot || !a.rot_dims ? PA_PLAIN : a.pairs ? PA_PAIRS : a.rot_dims % 8 ? PA_ODD_HALVES : PA_HALVES;
    if (c.dim <= 16) append_launch<2>(a, turn, stream);
    else if (c.dim <= 32) append_launch<4>(a, turn, stream);
    else if (c.dim <= 64) append_launch<8>(a, turn, stream);
    else if (c.dim <= 128) append_launch<16>(a, turn, stream);
    else append_launch<32>(a, turn, stream);
    return (int)cudaGetLastError();
}

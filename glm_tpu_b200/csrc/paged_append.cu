// Rows of a fused q | k | v projection on their way to attention over a paged cache, one launch:
//
//   n = x rsqrt(mean(x^2) + eps) w            per head of q and k, where weights are given
//   (a, b) -> (a cos - b sin, a sin + b cos)  on the leading rot channels of q and k; (a, b) are channels (d, d + rot / 2), or (2 j, 2 j + 1)
//   k, v -> slot of the sequence, q -> a buffer
//
// fp32 between the bf16 row and the one rounding of the result.  A row whose slot is negative stores no key and value.  A sequence, slot, table entry
// or position out of range raises GLMB_STATUS_BAD_INDEX, the row stores nothing in the cache, and its queries are zeros.
//
// A thread has eight channels (16 bytes) of a head, WIDTH (a power of two) threads a head, and keeps the same channels for every head that it takes: the row's
// angles and the norm's weights are read and widened once.  Halves of a rotation change places by shuffles.  The first heads and values are on their way before the row's
// place in the cache is known.  8,191 rows of 64 + 8 + 8 heads of 128: 85 us, 4 TB/s, the issue of some 80 instructions for a vector its bound (117 us with
// twice as many; five CTAs an SM instead of four 95 -> 85; rows in turn with the next one's place looked up ahead 94, a ring of bulk copies 192).
#include "paged.cuh"
#include "vec8.cuh"

#define PA_THREADS 256
#define PA_UNROLL 3  // heads of a thread on their way

enum { PA_PLAIN = 0, PA_PAIRS = 1, PA_HALVES = 2, PA_ODD_HALVES = 3 };  // odd: halves that begin inside a vector

template <int WIDTH, int TURN>
struct AppendHeads {
    float2 cs[TURN == PA_PLAIN ? 1 : TURN == PA_PAIRS ? 4 : 8];  // (cos, sin) of this thread's channels, or of their pairs
    int mine, half, partner;
    bool live;
    float eps, inv_dim;

    // One head: what was loaded -> what is stored.  `norm`: whether w holds weights; head: where the head lies (odd halves read the other channels again).
    __device__ __forceinline__ uint4 turn(const uint4& raw, const float2 (&w)[4], bool norm, const bf16* head, const bf16* weights) const {
        float2 x[4] = {make_float2(bf16_lo(raw.x), bf16_hi(raw.x)), make_float2(bf16_lo(raw.y), bf16_hi(raw.y)), make_float2(bf16_lo(raw.z), bf16_hi(raw.z)),
                       make_float2(bf16_lo(raw.w), bf16_hi(raw.w))};
        float inv = 1.f;
        if (norm) {
            float2 s = __fmul2_rn(x[0], x[0]);
#pragma unroll
            for (int e = 1; e < 4; ++e) s = __ffma2_rn(x[e], x[e], s);
            float sum = s.x + s.y;
#pragma unroll
            for (int o = WIDTH >> 1; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            inv = rsqrtf(fmaf(sum, inv_dim, eps));
            const float2 inv2 = make_float2(inv, inv);
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __fmul2_rn(x[e], __fmul2_rn(w[e], inv2));
        }
        if (TURN == PA_PAIRS) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 c = make_float2(cs[e].x, cs[e].x), s = make_float2(-cs[e].y, cs[e].y), swapped = make_float2(x[e].y, x[e].x);
                x[e] = __ffma2_rn(swapped, s, __fmul2_rn(x[e], c));
            }
        } else if (TURN == PA_HALVES) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float2 other = make_float2(__shfl_sync(0xffffffffu, x[e].x, partner), __shfl_sync(0xffffffffu, x[e].y, partner));
                const float2 c = make_float2(cs[2 * e].x, cs[2 * e + 1].x), s = make_float2(cs[2 * e].y, cs[2 * e + 1].y);  // sin: negative in the first half
                x[e] = __ffma2_rn(other, s, __fmul2_rn(x[e], c));
            }
        } else if (TURN == PA_ODD_HALVES && live) {
            float y[8] = {x[0].x, x[0].y, x[1].x, x[1].y, x[2].x, x[2].y, x[3].x, x[3].y};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int d = mine * 8 + e, o = d < half ? d + half : d - half;
                if (d < 2 * half) y[e] = fmaf(to_f32(head[o]) * (inv * (weights ? to_f32(weights[o]) : 1.f)), cs[e].y, y[e] * cs[e].x);
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = make_float2(y[2 * e], y[2 * e + 1]);
        }
        return make_uint4(pack_bf16(x[0].x, x[0].y), pack_bf16(x[1].x, x[1].y), pack_bf16(x[2].x, x[2].y), pack_bf16(x[3].x, x[3].y));
    }
};

// grid (rows, parts of a row).
template <int WIDTH, int TURN>
__global__ void __launch_bounds__(PA_THREADS, 5) paged_append_kernel(const __grid_constant__ PagedAppendArgs a) {
    GLMB_PDL_PROLOGUE();
    constexpr int AT_ONCE = PA_THREADS / WIDTH;
    const PagedArgs& c = a.cache;
    const int row = blockIdx.x, lane = threadIdx.x & 31, first = (int)threadIdx.x / WIDTH, heads = a.H + c.G;
    AppendHeads<WIDTH, TURN> t;
    t.mine = threadIdx.x & (WIDTH - 1), t.live = t.mine < (c.dim >> 3), t.eps = a.eps, t.inv_dim = 1.f / c.dim;
    const bf16* src = a.qkv + (int64_t)row * a.qkv_stride;
    const bf16* mine = src + t.mine * 8;
    // rounds of heads: those of q, then those of k (a round is never of both)
    const int q_rounds = a.q ? (a.H + AT_ONCE - 1) / AT_ONCE : 0, rounds = q_rounds + (c.G + AT_ONCE - 1) / AT_ONCE;
    auto head_of = [&](int r) { return r < q_rounds ? r * AT_ONCE + first : a.H + (r - q_rounds) * AT_ONCE + first; };
    auto there = [&](int r) { return t.live && r < rounds && head_of(r) < (r < q_rounds ? a.H : heads); };
    uint4 raw[PA_UNROLL];
#pragma unroll
    for (int u = 0; u < PA_UNROLL; ++u) {
        const int r = (int)blockIdx.y + u * (int)gridDim.y;
        raw[u] = there(r) ? ld_stream16(mine + (int64_t)head_of(r) * c.dim) : make_uint4(0, 0, 0, 0);
    }
    const int pieces = c.vdim >> 3, values = c.G * pieces, first_value = (int)(threadIdx.x + blockIdx.y * PA_THREADS), value_step = PA_THREADS * (int)gridDim.y;
    const bf16* value_src = src + (int64_t)heads * c.dim;
    const uint4 value = first_value < values ? ld_stream16(value_src + first_value * 8) : make_uint4(0, 0, 0, 0);

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
    if (TURN != PA_PLAIN) {
        t.half = a.rot_dims >> 1;
        const float2* rot = a.rot + (int64_t)(bad ? 0 : pos) * t.half;
        const int hv = t.half >> 3;
        t.partner = (lane & ~(WIDTH - 1)) | (t.mine < hv ? t.mine + hv : t.mine < 2 * hv ? t.mine - hv : t.mine);  // the thread with the other half
#pragma unroll
        for (int e = 0; e < (TURN == PA_PAIRS ? 4 : 8); ++e) {
            t.cs[e] = make_float2(1.f, 0.f);
            const int d = TURN == PA_PAIRS ? t.mine * 4 + e : t.mine * 8 + e;
            if (t.live && d < (TURN == PA_PAIRS ? t.half : 2 * t.half)) {
                t.cs[e] = rot[TURN != PA_PAIRS && d >= t.half ? d - t.half : d];
                if (TURN != PA_PAIRS && d < t.half) t.cs[e].y = -t.cs[e].y;
            }
        }
    }
    float2 w[4];
    auto weights = [&](const bf16* from) {
        const uint4 u = t.live && from ? ld_hot16(from + t.mine * 8) : make_uint4(0, 0, 0, 0);
        w[0] = make_float2(bf16_lo(u.x), bf16_hi(u.x)), w[1] = make_float2(bf16_lo(u.y), bf16_hi(u.y));
        w[2] = make_float2(bf16_lo(u.z), bf16_hi(u.z)), w[3] = make_float2(bf16_lo(u.w), bf16_hi(u.w));
    };
    bf16* q = a.q + (int64_t)row * a.q_stride + t.mine * 8;
    bf16* k = c.k + page * c.k_page + in * c.k_slot + t.mine * 8;
    const bf16* now = a.q_norm;
    weights(now);
    for (int r0 = blockIdx.y; r0 < rounds; r0 += PA_UNROLL * (int)gridDim.y) {
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) {
            const int r = r0 + u * (int)gridDim.y, h = head_of(r);
            if (r >= rounds) break;
            const bool is_q = r < q_rounds;
            if (!is_q && now != a.k_norm) now = a.k_norm, weights(now);
            uint4 y = t.turn(raw[u], w, now != nullptr, src + (int64_t)h * c.dim, now);
            if (bad) y = make_uint4(0, 0, 0, 0);
            if (there(r) && is_q) *reinterpret_cast<uint4*>(q + h * c.dim) = y;
            else if (there(r) && stores) *reinterpret_cast<uint4*>(k + (h - a.H) * c.k_head) = y;
        }
#pragma unroll
        for (int u = 0; u < PA_UNROLL; ++u) {
            const int r = r0 + (PA_UNROLL + u) * (int)gridDim.y;
            if (there(r)) raw[u] = ld_stream16(mine + (int64_t)head_of(r) * c.dim);
        }
    }
    if (!stores) return;
    bf16* v = c.v + page * c.v_page + in * c.v_slot;
    for (int i = first_value; i < values; i += value_step)
        *reinterpret_cast<uint4*>(v + i / pieces * c.v_head + i % pieces * 8) = i == first_value ? value : ld_stream16(value_src + i * 8);
}

template <int WIDTH>
static void append_launch(const PagedAppendArgs& a, int turn, cudaStream_t stream) {
    const int at_once = PA_THREADS / WIDTH, rounds = (a.q ? ceil_div(a.H, at_once) : 0) + ceil_div(a.cache.G, at_once);
    // a row is dealt to several CTAs while there are fewer rows than four for each SM
    const dim3 grid(a.rows, min(rounds, ceil_div(148 * 4, a.rows)));
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
        a.rot_dims > c.dim)
        return 1;
    if (a.rows == 0) return 0;
    const int turn = !a.rot || !a.rot_dims ? PA_PLAIN : a.pairs ? PA_PAIRS : a.rot_dims % 16 ? PA_ODD_HALVES : PA_HALVES;
    if (c.dim <= 16) append_launch<2>(a, turn, stream);
    else if (c.dim <= 32) append_launch<4>(a, turn, stream);
    else if (c.dim <= 64) append_launch<8>(a, turn, stream);
    else if (c.dim <= 128) append_launch<16>(a, turn, stream);
    else append_launch<32>(a, turn, stream);
    return (int)cudaGetLastError();
}

// Log probability of given tokens, entropy and the most likely tokens of rows of logits (bf16 or fp32; fp32 arithmetic, see logprobs.cuh).
//
// A row with a NaN or an infinite logit above zero has no probabilities: its numbers are NaN, its ids -1, and GLMB_STATUS_NONFINITE is raised.  A row
// of minus infinities alone (its mask leaves nothing): log probabilities minus infinity, entropy 0, the lowest ids.  A token of -1 asks for nothing
// (NaN); any other one outside the vocabulary is NaN too and raises GLMB_STATUS_BAD_INDEX.
#include "logprobs.cuh"

#define LP_TOP 32  // most alternatives of a row

struct TokenLogprobsArgs {
    const void* logits; int64_t stride;
    const void* tokens;
    float* logprob; float* entropy; float* best;
    int* top_ids; float* top_logprobs;
    int rows, vocab, top;
    int is_f32, tokens_64;
    uint32_t* status;
};

__device__ __forceinline__ float lp_value(const bf16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float lp_value(const float* p) { return *p; }

// The token whose log probability is asked for; -1: none.
__device__ __forceinline__ int lp_token(const TokenLogprobsArgs& a, int row) {
    const int64_t k = a.tokens_64 ? reinterpret_cast<const int64_t*>(a.tokens)[row] : reinterpret_cast<const int*>(a.tokens)[row];
    if (k >= 0 && k < a.vocab) return (int)k;
    if (k != -1) raise_status(a.status, GLMB_STATUS_BAD_INDEX);
    return -1;
}

// One CTA a row: the sums in one pass, each alternative in a further one.
template <typename T>
__global__ void __launch_bounds__(256) token_logprobs_kernel(TokenLogprobsArgs a) {
    GLMB_PDL_PROLOGUE();
    __shared__ float part_s[8][3];
    __shared__ unsigned long long key_s[8];
    const int row = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.stride;
    LogitSums sums;
    sums.clear();
    bool bad = false;
    for (int i = threadIdx.x; i < a.vocab; i += 256) {
        const float v = lp_value(x + i);
        bad |= isnan(v) || v == INFINITY;
        if (v > sums.m) sums.rebase(v);
        if (v != -INFINITY) sums.add(v);
    }
    bad = __syncthreads_or(bad);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        sums.join(__shfl_xor_sync(0xffffffffu, sums.m, o), __shfl_xor_sync(0xffffffffu, sums.s, o), __shfl_xor_sync(0xffffffffu, sums.t, o));
    if (lane == 0) part_s[warp][0] = sums.m, part_s[warp][1] = sums.s, part_s[warp][2] = sums.t;
    __syncthreads();
    sums.clear();
    for (int w = 0; w < 8; ++w) sums.join(part_s[w][0], part_s[w][1], part_s[w][2]);
    const float norm = sums.s > 0.f ? logf(sums.s) : 0.f;
    if (threadIdx.x == 0) {
        const int k = lp_token(a, row);
        const float v = k >= 0 ? lp_value(x + k) : NAN;
        a.logprob[row] = bad || k < 0 ? NAN : v == -INFINITY ? -INFINITY : (v - sums.m) - norm;
        a.entropy[row] = bad ? NAN : sums.s > 0.f ? norm - sums.t / sums.s : 0.f;
        a.best[row] = bad ? NAN : sums.s > 0.f ? -norm : -INFINITY;
        if (bad) raise_status(a.status, GLMB_STATUS_NONFINITE);
    }
    unsigned long long below = ~0ull;  // a key above every candidate's
    for (int n = 0; n < a.top; ++n) {
        unsigned long long key = 0;
        if (!bad)
            for (int i = threadIdx.x; i < a.vocab; i += 256) {
                const unsigned long long mine = candidate_key(lp_value(x + i), i);
                if (mine < below && mine > key) key = mine;
            }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
            key = other > key ? other : key;
        }
        __syncthreads();
        if (lane == 0) key_s[warp] = key;
        __syncthreads();
        for (int w = 0; w < 8; ++w) key = key_s[w] > key ? key_s[w] : key;
        below = key;
        if (threadIdx.x == 0) {
            const int id = candidate_id(key);
            const float v = bad ? NAN : lp_value(x + id);
            a.top_ids[(int64_t)row * a.top + n] = bad ? -1 : id;
            a.top_logprobs[(int64_t)row * a.top + n] = bad ? NAN : v == -INFINITY ? -INFINITY : (v - sums.m) - norm;
        }
    }
}

GLMB_API size_t glmb_token_logprobs_args_sizeof() { return sizeof(TokenLogprobsArgs); }

GLMB_API int glmb_token_logprobs(const TokenLogprobsArgs* args, cudaStream_t stream) {
    const TokenLogprobsArgs a = *args;
    if (a.rows < 0 || a.vocab < 1 || a.top < 0 || a.top > LP_TOP || a.top > a.vocab || a.stride < 0) return 1;
    if (a.rows == 0) return 0;
    if (a.is_f32) GLMB_LAUNCH(token_logprobs_kernel<float>, a.rows, 256, 0, stream, a);
    else GLMB_LAUNCH(token_logprobs_kernel<bf16>, a.rows, 256, 0, stream, a);
    return (int)cudaGetLastError();
}

// Log-probabilities of given tokens from rows of logits: ln softmax at the token, the row's
// entropy, the token's rank and the greatest logits with their indices.
//
// With m the row's maximum, s = sum e^(x - m) and t = sum (x - m) e^(x - m): ln p = x_t - m -
// ln s, H = ln s - t / s.  The greatest are found as 64-bit keys (value, lower index first).
#include "common.cuh"

namespace {

constexpr int LP_THREADS = 512;
constexpr int LP_MAX_TOP = 32;

// A logit and its index as one unsigned number that grows with the logit and falls with the
// index: equal logits (-0 is 0) go by the lower index.  NaN stands below every number.
__device__ __forceinline__ unsigned long long lp_key(float x, unsigned i) {
    unsigned b = __float_as_uint(x + 0.f);
    b = (int)b < 0 ? ~b : b | 0x80000000u;
    if (x != x) b = 0;
    return (unsigned long long)b << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float lp_value(unsigned long long key) {
    const unsigned b = (unsigned)(key >> 32);
    if (b == 0) return __uint_as_float(0x7fffffffu);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ unsigned long long warp_max_u64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long t = __shfl_xor_sync(0xffffffffu, v, o);
        v = t > v ? t : v;
    }
    return v;
}

struct Logprobs {
    const void* logits;
    long long ld;
    int V, top;
    const int* tokens;
    float *logprob, *entropy;
    int* rank;
    int* top_ids;
    float* top_logprobs;
};

template <typename T>
__global__ void __launch_bounds__(LP_THREADS) logprobs_kernel(Logprobs a) {
    pdl_wait();
    pdl_launch_next();
    __shared__ float scratch[32];
    __shared__ unsigned long long best[32];
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* x = (const T*)a.logits + (long long)row * a.ld;
    const int t = a.tokens[row];
    const bool has = t >= 0 && t < a.V;
    const float xt = has ? to_f32(x[t]) : 0.f;
    float m = -INFINITY;
    for (int i = tid; i < a.V; i += LP_THREADS) m = fmaxf(m, to_f32(x[i]));
    m = block_max(m, scratch);
    float s = 0.f, w = 0.f, ahead = 0.f;
    for (int i = tid; i < a.V; i += LP_THREADS) {
        const float v = to_f32(x[i]), d = v - m, e = expf(d);
        s += e;
        if (e > 0.f) w += e * d;
        ahead += v > xt || (v == xt && i < t);
    }
    s = block_sum(s, scratch);
    w = block_sum(w, scratch);
    ahead = block_sum(ahead, scratch);
    const float ls = logf(s);
    if (tid == 0) {
        a.logprob[row] = has ? xt - m - ls : __uint_as_float(0x7fffffffu);
        a.entropy[row] = ls - w / s;
        a.rank[row] = has ? (int)ahead + 1 : 0;
    }
    unsigned long long below = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        unsigned long long mine = 0;
        for (int i = tid; i < a.V; i += LP_THREADS) {
            const unsigned long long key = lp_key(to_f32(x[i]), i);
            if (key < below && key > mine) mine = key;
        }
        mine = warp_max_u64(mine);
        __syncthreads();
        if ((tid & 31) == 0) best[tid >> 5] = mine;
        __syncthreads();
        below = warp_max_u64((tid & 31) < LP_THREADS / 32 ? best[tid & 31] : 0ull);
        if (tid == 0) {
            a.top_ids[(size_t)row * a.top + k] = (int)(0xffffffffu - (unsigned)below);
            a.top_logprobs[(size_t)row * a.top + k] = lp_value(below) - m - ls;
        }
    }
}

}  // namespace

// Rows of logits [R, V] (row stride ld): logprob, entropy, rank [R]; top_ids, top_logprobs
// [R, top], greatest first, equal ones by index.  tokens[r] outside 0 .. V - 1 stands for no
// token: logprob NaN, rank 0.
AGV_API int agv_token_logprobs(const void* logits, long long ld, int dtype, int R, int V,
                               const int* tokens, int top, float* logprob, float* entropy, int* rank,
                               int* top_ids, float* top_logprobs, cudaStream_t stream) {
    AGV_REQUIRE(R >= 0 && V > 0 && ld >= 0 && (ld >= V || R <= 1), "token_logprobs: bad sizes R=%d V=%d", R, V);
    AGV_REQUIRE(top >= 0 && top <= LP_MAX_TOP && top <= V, "token_logprobs: top %d must lie in 0..%d", top,
                V < LP_MAX_TOP ? V : LP_MAX_TOP);
    AGV_REQUIRE(dtype == AGV_F32 || dtype == AGV_BF16, "token_logprobs: bad dtype");
    if (R == 0) return 0;
    Logprobs a{logits, ld, V, top, tokens, logprob, entropy, rank, top_ids, top_logprobs};
    if (dtype == AGV_F32) agv_launch(logprobs_kernel<float>, R, LP_THREADS, 0, stream, a);
    else agv_launch(logprobs_kernel<__nv_bfloat16>, R, LP_THREADS, 0, stream, a);
    AGV_LAUNCH_OK("logprobs_kernel");
    return 0;
}

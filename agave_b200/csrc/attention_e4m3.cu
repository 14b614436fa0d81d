// Decode attention over the 8-bit cache: one query per sequence.
//
// o_a = sum_j w_aj v_j with w_aj = exp(s_aj - m) / (sum_j exp(s_aj - m) + exp(sink_a - m)),
// s_aj = cap(scale * q_a . k_j) + bias; one pass over the keys with a running maximum m.
#include "e4m3.cuh"

namespace {

constexpr int AE_THREADS = 128;
constexpr int AE_MAX_DIM = 256;

struct AttendE4 {
    const void* q;
    long long ldq;
    void* out;
    const unsigned char *k_pool, *v_pool;
    const float *k_scale, *v_scale;
    const int *table, *slots, *positions;
    int n_slots, max_pages, n_pages, page, cap, nh, nkv, hd, hdv, window, keep_first;
    float scale, softcap;
    const float *sinks, *dist_bias;
    int n_dist;
};

// One CTA per sequence and query head: a warp walks every fourth key.
template <typename T>
__global__ void __launch_bounds__(AE_THREADS) attend_e4m3_kernel(AttendE4 a) {
    pdl_wait();
    pdl_launch_next();
    __shared__ float acc[AE_THREADS / 32][AE_MAX_DIM];
    __shared__ float stat[AE_THREADS / 32][2];
    const int b = blockIdx.y, h = blockIdx.x, g = h / (a.nh / a.nkv);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    T* out = (T*)a.out + ((size_t)b * a.nh + h) * a.hdv;
    const int slot = a.slots[b], p = a.positions[b];
    if (slot < 0 || slot >= a.n_slots || p < 0) {
        for (int i = threadIdx.x; i < a.hdv; i += AE_THREADS) out[i] = from_f32<T>(0.f);
        return;
    }
    const int lo = max(first_visible(p, a.window), p - a.cap + 1);
    const int kept = p < a.cap ? min(a.keep_first, lo) : 0;
    const T* q = (const T*)a.q + (long long)b * a.ldq + (long long)h * a.hd;
    float o[AE_MAX_DIM / 32] = {}, m = -INFINITY, l = 0.f;
    for (int i = warp; i < kept + p - lo + 1; i += AE_THREADS / 32) {
        const int j = i < kept ? i : lo + i - kept, row = j % a.cap;
        const int page = a.table[(size_t)slot * a.max_pages + row / a.page];
        if (page < 0 || page >= a.n_pages) continue;
        const size_t at = ((size_t)page * a.page + row % a.page) * a.nkv + g;
        float s = 0.f;
        for (int d = lane; d < a.hd; d += 32) s = fmaf(to_f32(q[d]), e4m3_to_float2(a.k_pool[at * a.hd + d]).x, s);
        s = warp_sum(s) * a.k_scale[(size_t)page * a.nkv + g] * a.scale;
        if (a.softcap > 0.f) s = soft_capped(s, a.softcap);
        if (a.dist_bias) s += a.dist_bias[(size_t)h * a.n_dist + min(p - j, a.n_dist - 1)];
        const float mn = fmaxf(m, s), keep = mn == -INFINITY ? 1.f : expf(m - mn);
        const float w = mn == -INFINITY ? 0.f : expf(s - mn);
        const float vs = w * a.v_scale[(size_t)page * a.nkv + g];
        l = l * keep + w;
        m = mn;
#pragma unroll
        for (int e = 0; e < AE_MAX_DIM / 32; ++e) {
            const int d = lane + 32 * e;
            if (d < a.hdv) o[e] = o[e] * keep + vs * e4m3_to_float2(a.v_pool[at * a.hdv + d]).x;
        }
    }
    for (int e = 0; e < AE_MAX_DIM / 32; ++e) acc[warp][lane + 32 * e] = o[e];
    if (lane == 0) { stat[warp][0] = m; stat[warp][1] = l; }
    __syncthreads();
    float M = a.sinks ? a.sinks[h] : -INFINITY, L;
    for (int w = 0; w < AE_THREADS / 32; ++w) M = fmaxf(M, stat[w][0]);
    L = a.sinks ? expf(a.sinks[h] - M) : 0.f;
    for (int w = 0; w < AE_THREADS / 32; ++w)
        if (stat[w][0] != -INFINITY || stat[w][1] != 0.f) L += stat[w][1] * expf(stat[w][0] - M);
    for (int d = threadIdx.x; d < a.hdv; d += AE_THREADS) {
        float v = 0.f;
        for (int w = 0; w < AE_THREADS / 32; ++w)
            if (stat[w][0] != -INFINITY || stat[w][1] != 0.f) v += acc[w][d] * expf(stat[w][0] - M);
        out[d] = from_f32<T>(L == 0.f ? 0.f : v / L);
    }
}

}  // namespace

// One query per batch entry, q [B, nh * hd] (row stride ldq), against the 8-bit cache; out
// [B, nh * hdv] in q's type.  The query stands at positions[b] and its own key is stored.
// window as first_visible has it; keep_first: the first keys stay visible behind a window;
// sinks [nh] or null; dist_bias [nh, n_dist] or null, added to the score of a key at distance
// min(p - j, n_dist - 1); softcap > 0: the scaled score s becomes softcap * tanh(s / softcap).
// Entries with slots[b] < 0 get zeros.
AGV_API int agv_attention_decode_e4m3(const void* q, long long ldq, void* out, int dtype,
                                      const void* k_pool, const void* v_pool, const float* k_scale,
                                      const float* v_scale, const int* table, int n_slots, int max_pages,
                                      int page, int cap, int n_pages, const int* slots,
                                      const int* positions, int B, int nh, int nkv, int hd, int hdv,
                                      float scale, int window, int keep_first, const float* sinks,
                                      const float* dist_bias, int n_dist, float softcap, int max_keys,
                                      float* partial, long long partial_floats, cudaStream_t stream) {
    AGV_REQUIRE(B >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0 && n_slots > 0 && n_pages > 0,
                "attention_decode_e4m3: bad sizes (%d query heads over %d)", nh, nkv);
    AGV_REQUIRE(hd > 0 && hd % 16 == 0 && hd <= AE_MAX_DIM && hdv > 0 && hdv % 16 == 0 && hdv <= AE_MAX_DIM,
                "attention_decode_e4m3: head sizes %d and %d must be multiples of 16 up to %d", hd, hdv, AE_MAX_DIM);
    AGV_REQUIRE(page > 0 && page % 16 == 0 && cap > 0 && cap % page == 0 && cap / page <= max_pages,
                "attention_decode_e4m3: bad cache geometry (page %d, cap %d, table of %d)", page, cap, max_pages);
    AGV_REQUIRE(dtype == AGV_F32 || dtype == AGV_BF16, "attention_decode_e4m3: bad dtype");
    AGV_REQUIRE(agv_aligned(k_pool, 16) && agv_aligned(v_pool, 16), "attention_decode_e4m3: unaligned pool");
    AGV_REQUIRE(keep_first >= 0 && softcap >= 0.f && (!dist_bias || n_dist > 0), "attention_decode_e4m3: bad options");
    AGV_REQUIRE(B <= 65535, "attention_decode_e4m3: %d sequences exceed the grid", B);
    if (B == 0) return 0;
    AttendE4 a{q, ldq, out, (const unsigned char*)k_pool, (const unsigned char*)v_pool, k_scale, v_scale,
               table, slots, positions, n_slots, max_pages, n_pages, page, cap, nh, nkv, hd, hdv,
               window, window ? keep_first : 0, scale, softcap, sinks, dist_bias, n_dist};
    if (dtype == AGV_F32) agv_launch(attend_e4m3_kernel<float>, dim3(nh, B), AE_THREADS, 0, stream, a);
    else agv_launch(attend_e4m3_kernel<__nv_bfloat16>, dim3(nh, B), AE_THREADS, 0, stream, a);
    AGV_LAUNCH_OK("attend_e4m3_kernel");
    return 0;
}

// 32-bit values of scratch that agv_attention_decode_e4m3 wants for these sizes.
AGV_API long long agv_attention_decode_e4m3_scratch(int B, int nh, int nkv, int hd, int hdv, int max_keys) {
    return 0;
}

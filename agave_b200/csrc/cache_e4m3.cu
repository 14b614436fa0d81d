// The store of new keys and values in the 8-bit cache.
//
// One CTA takes one page of one sequence and one kv head's keys or values: the greatest
// magnitude of the new rows there gives the scale, the rows are rounded to codes.  Where the
// page already holds earlier tokens of the sequence the scale never shrinks, and if it
// grows their codes are rounded to the greater one.
#include "e4m3.cuh"

namespace {

constexpr int CE_THREADS = 128;

struct StoreE4 {
    const void* x[2];              // keys, values: rows of nkv heads
    long long ld[2];
    unsigned char* pool[2];        // [pages, page, nkv, dim]
    float* scale[2];               // [pages, nkv]
    int dim[2];
    const int *cu, *slots, *lens, *table;
    int T, n_slots, max_pages, n_pages, page, cap, nkv;
};

template <typename T>
__global__ void __launch_bounds__(CE_THREADS) store_e4m3_kernel(StoreE4 a) {
    pdl_wait();
    pdl_launch_next();
    __shared__ float scratch[32];
    const int b = blockIdx.z, which = blockIdx.y & 1, g = blockIdx.y >> 1, tid = threadIdx.x;
    const int slot = a.slots[b], c0 = a.cu[b], n = a.cu[b + 1] - c0, len = a.lens[b];
    if (slot < 0 || slot >= a.n_slots || n <= 0 || c0 < 0 || c0 > a.T - n || len < n) return;
    const int start = len - n, last = (len - 1) / a.page;
    const int first = max(start / a.page, last - a.cap / a.page + 1);
    const int dim = a.dim[which];
    const T* x = (const T*)a.x[which] + (size_t)g * dim;
    for (int j = first + blockIdx.x; j <= last; j += gridDim.x) {
        const int p0 = max(start, j * a.page), p1 = min(len, (j + 1) * a.page);
        const int page = a.table[(size_t)slot * a.max_pages + j % (a.cap / a.page)];
        if (page < 0 || page >= a.n_pages) continue;
        const T* src = x + (long long)(c0 + p0 - start) * a.ld[which];
        unsigned char* dst = a.pool[which] + (((size_t)page * a.page) * a.nkv + g) * dim;
        float* sc = a.scale[which] + (size_t)page * a.nkv + g;
        const int pairs = (p1 - p0) * dim / 2, half = dim / 2;
        float amax = 0.f;
        for (int i = tid; i < pairs; i += CE_THREADS) {
            const T* e = src + (long long)(i / half) * a.ld[which] + i % half * 2;
            amax = fmaxf(amax, fmaxf(e4m3_magnitude(to_f32(e[0])), e4m3_magnitude(to_f32(e[1]))));
        }
        amax = block_max(amax, scratch);
        float s = e4m3_scale(amax);
        const int r0 = p0 - j * a.page;
        if (r0 > 0) {
            const float old = *sc;
            s = fmaxf(s, old);
            if (s != old) {
                const float f = old * e4m3_inverse(s);
                for (int i = tid; i < r0 * half; i += CE_THREADS) {
                    unsigned short* e = (unsigned short*)(dst + (size_t)(i / half) * a.nkv * dim) + i % half;
                    const float2 v = e4m3_to_float2(*e);
                    *e = (unsigned short)e4m3_pair(v.x * f, v.y * f);
                }
            }
        }
        __syncthreads();                           // everyone has read the old scale
        if (tid == 0) *sc = s;
        const float inv = e4m3_inverse(s);
        for (int i = tid; i < pairs; i += CE_THREADS) {
            const T* e = src + (long long)(i / half) * a.ld[which] + i % half * 2;
            ((unsigned short*)(dst + (size_t)(r0 + i / half) * a.nkv * dim))[i % half] =
                (unsigned short)e4m3_pair(to_f32(e[0]) * inv, to_f32(e[1]) * inv);
        }
    }
}

}  // namespace

// Stores k [T, nkv * hd] and v [T, nkv * hdv] (row strides ldk, ldv) in the pages of the
// sequences they belong to: entry b brings tokens cu[b] .. cu[b + 1] and has length lens[b]
// after them; slots[b] < 0 brings nothing to store.  Position p lives in row p % cap of the
// slot's page table; of a sequence longer than cap only the last cap / page pages are stored.
// No slot twice in one call.  max_new (the most tokens an entry brings) sizes the grid.
AGV_API int agv_cache_store_e4m3(const void* k, long long ldk, const void* v, long long ldv, int dtype,
                                 const int* cu, const int* slots, const int* lens, int B, int T,
                                 int max_new, int nkv, int hd, int hdv, void* k_pool, void* v_pool,
                                 float* k_scale, float* v_scale, const int* table, int n_slots,
                                 int max_pages, int page, int cap, int n_pages, cudaStream_t stream) {
    AGV_REQUIRE(B >= 0 && T >= 0 && nkv > 0 && n_slots > 0 && n_pages > 0, "cache_store_e4m3: bad sizes");
    AGV_REQUIRE(hd > 0 && hd % 16 == 0 && hdv > 0 && hdv % 16 == 0,
                "cache_store_e4m3: head sizes %d and %d must be multiples of 16", hd, hdv);
    AGV_REQUIRE(page > 0 && cap > 0 && cap % page == 0 && cap / page <= max_pages,
                "cache_store_e4m3: bad cache geometry (page %d, cap %d, table of %d)", page, cap, max_pages);
    AGV_REQUIRE(dtype == AGV_F32 || dtype == AGV_BF16, "cache_store_e4m3: bad dtype");
    AGV_REQUIRE(agv_aligned(k_pool, 16) && agv_aligned(v_pool, 16), "cache_store_e4m3: unaligned pool");
    AGV_REQUIRE(B <= 65535 && nkv <= 32767, "cache_store_e4m3: %d sequences, %d heads exceed the grid", B, nkv);
    if (B == 0 || T == 0) return 0;
    StoreE4 a{{k, v}, {ldk, ldv}, {(unsigned char*)k_pool, (unsigned char*)v_pool}, {k_scale, v_scale},
              {hd, hdv}, cu, slots, lens, table, T, n_slots, max_pages, n_pages, page, cap, nkv};
    const int most = max_new < 1 ? 1 : max_new > T ? T : max_new;
    int blocks = most == 1 ? 1 : (most + page - 2) / page + 1;
    if (blocks > cap / page) blocks = cap / page;
    const dim3 grid(blocks, 2 * nkv, B);
    if (dtype == AGV_F32) agv_launch(store_e4m3_kernel<float>, grid, CE_THREADS, 0, stream, a);
    else agv_launch(store_e4m3_kernel<__nv_bfloat16>, grid, CE_THREADS, 0, stream, a);
    AGV_LAUNCH_OK("store_e4m3_kernel");
    return 0;
}

// The store of new keys and values in the 8-bit cache.
//
// One CTA takes one page of one sequence and one kv head's keys or values: the greatest
// magnitude of the new rows there gives the scale, the rows are rounded to codes.  Where the
// page already holds earlier tokens of the sequence the scale never shrinks, and if it
// grows their codes are rounded to the greater one.
//
// What bounds it is reading the rows once and writing a byte for each value.  Prompts: a page's
// rows (64 of 256 values: 32 KB of bfloat16) stay in registers between the maximum and the
// rounding, read 16 bytes at a time.  Single tokens, and rows that do not start on 16 bytes, go two values
// at a time and are read twice (the second time from L1); there it is the launch that counts.
#include "e4m3.cuh"
#include <type_traits>

namespace {

constexpr int CE_THREADS = 128;

struct StoreE4 {
    const void* x[2];              // keys, values: rows of nkv heads
    long long ld[2];
    unsigned char* pool[2];        // [pages, page, nkv, dim]
    float* scale[2];               // [pages, nkv]
    int dim[2];
    const int *cu, *slots, *lens, *table;
    int T, n_slots, max_pages, n_pages, page_bits, ring, nkv;      // a sequence's pages: a ring of so many
};

// Scale of a page and head from the new rows' magnitude and, where the page goes on (r0 rows of it
// are held), the scale it has; the held codes move to it if it grows.  All threads of the CTA.
__device__ __forceinline__ float settle_scale(float amax, float* sc, int r0, unsigned char* codes, size_t row, int dim) {
    float s = e4m3_scale(amax);
    if (r0 > 0) {
        const float old = *sc;
        s = fmaxf(s, old);
        if (s != old) {
            const float f = old * e4m3_inverse(s);
            const int quads = dim / 4;
            for (int i = threadIdx.x; i < r0 * quads; i += blockDim.x) {
                unsigned* e = (unsigned*)(codes + (size_t)(i / quads) * row) + i % quads;
                const unsigned w = *e;
                const float2 lo = e4m3_to_float2(w), hi = e4m3_to_float2(w >> 16);
                *e = e4m3_pair(lo.x * f, lo.y * f) | e4m3_pair(hi.x * f, hi.y * f) << 16;
            }
        }
        __syncthreads();                           // everyone has read the old scale
    }
    if (threadIdx.x == 0) *sc = s;
    return s;
}

template <typename T>
__global__ void __launch_bounds__(CE_THREADS) store_e4m3_kernel(const StoreE4 a) {
    pdl_wait();
    pdl_launch_next();
    __shared__ float scratch[32];
    // (the heads of a page beside each other on the grid: together their rows are whole)
    const int b = blockIdx.z >> 1, which = blockIdx.z & 1, g = blockIdx.x, tid = threadIdx.x;
    const int slot = a.slots[b], c0 = a.cu[b], n = a.cu[b + 1] - c0, len = a.lens[b];
    if (slot < 0 || slot >= a.n_slots || n <= 0 || c0 < 0 || c0 > a.T - n || len < n) return;
    const int start = len - n, last = (len - 1) >> a.page_bits;
    const int first = max(start >> a.page_bits, last - a.ring + 1);
    const int dim = a.dim[which];
    const T* x = (const T*)a.x[which] + (size_t)g * dim;
    for (int j = first + blockIdx.y; j <= last; j += gridDim.y) {
        const int p0 = max(start, j << a.page_bits), p1 = min(len, (j + 1) << a.page_bits);
        const int page = a.table[(size_t)slot * a.max_pages + (j < a.ring ? j : j % a.ring)];
        if (page < 0 || page >= a.n_pages) continue;
        const T* src = x + (long long)(c0 + p0 - start) * a.ld[which];
        unsigned char* dst = a.pool[which] + (((size_t)page << a.page_bits) * a.nkv + g) * dim;
        float* sc = a.scale[which] + (size_t)page * a.nkv + g;
        const int pairs = (p1 - p0) * dim / 2, half = dim / 2;
        float amax = 0.f;
        for (int i = tid; i < pairs; i += CE_THREADS) {
            const T* e = src + (long long)(i / half) * a.ld[which] + i % half * 2;
            amax = fmaxf(amax, fmaxf(e4m3_magnitude(to_f32(e[0])), e4m3_magnitude(to_f32(e[1]))));
        }
        amax = block_max(amax, scratch);
        const int r0 = p0 - (j << a.page_bits);
        const float s = settle_scale(amax, sc, r0, dst, (size_t)a.nkv * dim, dim);
        const float inv = e4m3_inverse(s);
        for (int i = tid; i < pairs; i += CE_THREADS) {
            const T* e = src + (long long)(i / half) * a.ld[which] + i % half * 2;
            ((unsigned short*)(dst + (size_t)(r0 + i / half) * a.nkv * dim))[i % half] =
                (unsigned short)e4m3_pair(to_f32(e[0]) * inv, to_f32(e[1]) * inv);
        }
    }
}

// The same for rows of 16-byte pieces, pages of at most 64 positions and dimensions of at most 256:
// the page's rows in registers.

// The greatest magnitude of 16 bytes of values (infinity if one is infinite; NaN does not count).
__device__ __forceinline__ float piece_max(const uint4& u, float) {
    return fmaxf(fmaxf(fabsf(__uint_as_float(u.x)), fabsf(__uint_as_float(u.y))),
                 fmaxf(fabsf(__uint_as_float(u.z)), fabsf(__uint_as_float(u.w))));
}
__device__ __forceinline__ __nv_bfloat162 pair_of(unsigned w) {
    return *reinterpret_cast<const __nv_bfloat162*>(&w);
}
__device__ __forceinline__ float piece_max(const uint4& u, __nv_bfloat16) {
    const __nv_bfloat162 m = __hmax2(__hmax2(__habs2(pair_of(u.x)), __habs2(pair_of(u.y))),
                                     __hmax2(__habs2(pair_of(u.z)), __habs2(pair_of(u.w))));
    return fmaxf(__low2float(m), __high2float(m));
}
template <typename T>
__device__ __forceinline__ void piece_values(const uint4& u, float (&x)[16 / sizeof(T)]) {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) {
            x[i] = __uint_as_float(w[i]);
        } else {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
}
// (an infinity saturates here: for values that are known to have none)
__device__ __forceinline__ unsigned e4m3_quad_finite(float a, float b, float c, float d) {
    unsigned r;
    asm("{.reg .b16 l, h;\n cvt.rn.satfinite.e4m3x2.f32 l, %2, %1;\n cvt.rn.satfinite.e4m3x2.f32 h, %4, %3;\n"
        " mov.b32 %0, {l, h};}" : "=r"(r) : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
}

// WHOLE: the pieces of a row are a power of two, so a thread's pieces are all in one column.
template <typename T, int PIECES, int THREADS, bool WHOLE>
__global__ void __launch_bounds__(THREADS, (WHOLE || THREADS > 256 ? 1024 : 768) / THREADS)
store_pages_e4m3_kernel(const StoreE4 a) {
    constexpr int N = 16 / sizeof(T);
    pdl_wait();
    pdl_launch_next();
    __shared__ float scratch[32];
    // (the heads of a page beside each other on the grid: together their rows are whole)
    const int b = blockIdx.z >> 1, which = blockIdx.z & 1, g = blockIdx.x, tid = threadIdx.x;
    const int slot = a.slots[b], c0 = a.cu[b], n = a.cu[b + 1] - c0, len = a.lens[b];
    if (slot < 0 || slot >= a.n_slots || n <= 0 || c0 < 0 || c0 > a.T - n || len < n) return;
    const int start = len - n, last = (len - 1) >> a.page_bits;
    const int first = max(start >> a.page_bits, last - a.ring + 1);
    const int dim = a.dim[which], per_row = dim / N;
    // this thread's pieces, THREADS apart in the order of rows: the first one's row and column, and
    // the steps to the next
    int row0, col0, row_step, col_step;
    if (WHOLE) {
        const int bits = __ffs(per_row) - 1;
        row0 = tid >> bits, col0 = tid & (per_row - 1), row_step = THREADS >> bits, col_step = 0;
    } else {
        row0 = tid / per_row, col0 = tid % per_row, row_step = THREADS / per_row, col_step = THREADS % per_row;
    }
    const long long ld = a.ld[which], drow = (long long)a.nkv * dim;
    // (a page of codes, and so the steps in it, are within 32 bits)
    const long long x_step = row_step * ld + col_step * N, x_wrap = ld - dim;
    const int y_step = row_step * (int)drow + col_step * N, y_wrap = (int)drow - dim;
    for (int j = first + blockIdx.y; j <= last; j += gridDim.y) {
        const int p0 = max(start, j << a.page_bits), rows = min(len, (j + 1) << a.page_bits) - p0;
        const T* src = (const T*)a.x[which] + (c0 + p0 - start + row0) * ld + (size_t)g * dim + col0 * N;
        uint4 u[PIECES];
        int r = row0, c = col0;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) {
            u[i] = r < rows ? __ldg(reinterpret_cast<const uint4*>(src)) : make_uint4(0, 0, 0, 0);
            r += row_step;
            c += col_step;
            src += x_step;
            if (!WHOLE && c >= per_row) {
                c -= per_row;
                ++r;
                src += x_wrap;
            }
        }
        const int page = a.table[(size_t)slot * a.max_pages + (j < a.ring ? j : j % a.ring)];
        if (page < 0 || page >= a.n_pages) continue;
        float amax = 0.f;
#pragma unroll
        for (int i = 0; i < PIECES; ++i) amax = fmaxf(amax, piece_max(u[i], T{}));
        amax = block_max(amax, scratch);
        const bool infinite = amax == INFINITY;
        if (infinite) {                            // the greatest of the finite ones
            amax = 0.f;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                float x[N];
                piece_values<T>(u[i], x);
#pragma unroll
                for (int e = 0; e < N; ++e) amax = fmaxf(amax, e4m3_magnitude(x[e]));
            }
            amax = block_max(amax, scratch);
        }
        unsigned char* dst = a.pool[which] + (((size_t)page << a.page_bits) * a.nkv + g) * dim;
        const int r0 = p0 - (j << a.page_bits);
        const float inv = e4m3_inverse(settle_scale(amax, a.scale[which] + (size_t)page * a.nkv + g, r0, dst, drow, dim));
        const f32x2 inv2 = pack2(inv, inv);
        dst += (r0 + row0) * drow + col0 * N;
        r = row0;
        c = col0;
        auto codes = [&](float x0, float x1, float x2, float x3, auto any) {
            unpack2(mul2(pack2(x0, x1), inv2), x0, x1);
            unpack2(mul2(pack2(x2, x3), inv2), x2, x3);
            if constexpr (decltype(any)::value) return e4m3_pair(x0, x1) | e4m3_pair(x2, x3) << 16;
            else return e4m3_quad_finite(x0, x1, x2, x3);
        };
        auto write = [&](auto any) {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                if (r < rows) {
                    float x[N];
                    piece_values<T>(u[i], x);
                    const unsigned w = codes(x[0], x[1], x[2], x[3], any);
                    if constexpr (N == 8)
                        *reinterpret_cast<uint2*>(dst) = make_uint2(w, codes(x[N - 4], x[N - 3], x[N - 2], x[N - 1], any));
                    else
                        *reinterpret_cast<unsigned*>(dst) = w;
                }
                r += row_step;
                c += col_step;
                dst += y_step;
                if (!WHOLE && c >= per_row) {
                    c -= per_row;
                    ++r;
                    dst += y_wrap;
                }
            }
        };
        if (infinite) write(std::true_type{});
        else write(std::false_type{});
    }
}
// Eight pieces a thread (in the greatest page) and threads by the dimension: every size has the 128 KB
// under way on an SM that its 1024 threads of 64 registers hold (dimension 128 in 32 bits, 16000 positions
// of 16 heads: 72 us with four pieces of 512 threads, 52 with eight of 256).
template <typename T, bool WHOLE>
void launch_pages(const StoreE4& a, dim3 grid, cudaStream_t stream) {
    constexpr int T64 = 32 * sizeof(T);
    const int dim = a.dim[0] > a.dim[1] ? a.dim[0] : a.dim[1];
    if (dim > 128) agv_launch(store_pages_e4m3_kernel<T, 8, 4 * T64, WHOLE>, grid, 4 * T64, 0, stream, a);
    else if (dim > 64) agv_launch(store_pages_e4m3_kernel<T, 8, 2 * T64, WHOLE>, grid, 2 * T64, 0, stream, a);
    else agv_launch(store_pages_e4m3_kernel<T, 8, T64, WHOLE>, grid, T64, 0, stream, a);
}
template <typename T>
void launch_pages(const StoreE4& a, dim3 grid, cudaStream_t stream) {
    if ((a.dim[0] & (a.dim[0] - 1)) == 0 && (a.dim[1] & (a.dim[1] - 1)) == 0) launch_pages<T, true>(a, grid, stream);
    else launch_pages<T, false>(a, grid, stream);
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
    AGV_REQUIRE(page > 0 && (page & (page - 1)) == 0 && cap > 0 && cap % page == 0 && cap / page <= max_pages,
                "cache_store_e4m3: bad cache geometry (page %d, cap %d, table of %d)", page, cap, max_pages);
    AGV_REQUIRE(dtype == AGV_F32 || dtype == AGV_BF16, "cache_store_e4m3: bad dtype");
    AGV_REQUIRE(agv_aligned(k_pool, 16) && agv_aligned(v_pool, 16), "cache_store_e4m3: unaligned pool");
    AGV_REQUIRE(B <= 32767, "cache_store_e4m3: %d sequences exceed the grid", B);
    if (B == 0 || T == 0) return 0;
    int page_bits = 0;
    while (1 << page_bits < page) ++page_bits;
    StoreE4 a{{k, v}, {ldk, ldv}, {(unsigned char*)k_pool, (unsigned char*)v_pool}, {k_scale, v_scale},
              {hd, hdv}, cu, slots, lens, table, T, n_slots, max_pages, n_pages, page_bits, cap / page, nkv};
    const int most = max_new < 1 ? 1 : max_new > T ? T : max_new;
    int blocks = most == 1 ? 1 : (most + page - 2) / page + 1;
    if (blocks > cap / page) blocks = cap / page;
    const dim3 grid(nkv, blocks < 65535 ? blocks : 65535, 2 * B);
    const size_t esz = dtype == AGV_F32 ? 4 : 2;
    const int most_dim = hd > hdv ? hd : hdv;
    if (most > 1 && page <= 64 && most_dim <= 256 && (long long)page * nkv * most_dim <= 0x7fffffff &&
        agv_aligned(k, 16) && agv_aligned(v, 16) && ldk * esz % 16 == 0 && ldv * esz % 16 == 0) {
        if (dtype == AGV_F32) launch_pages<float>(a, grid, stream);
        else launch_pages<__nv_bfloat16>(a, grid, stream);
        AGV_LAUNCH_OK("store_pages_e4m3_kernel");
        return 0;
    }
    if (dtype == AGV_F32) agv_launch(store_e4m3_kernel<float>, grid, CE_THREADS, 0, stream, a);
    else agv_launch(store_e4m3_kernel<__nv_bfloat16>, grid, CE_THREADS, 0, stream, a);
    AGV_LAUNCH_OK("store_e4m3_kernel");
    return 0;
}

// Decode attention over the 8-bit cache: one query per sequence.
//
// o_a = sum_j w_aj v_j with w_aj = exp(s_aj - m) / (sum_j exp(s_aj - m) + exp(sink_a - m)),
// s_aj = cap(scale * q_a . k_j) + bias; one pass over the keys with a running maximum m.
//
// What bounds it is reading each key and value once, hd + hdv bytes a position and kv head.  The
// work, (sequence, kv head, up to 8 of its query heads) x pages of 64 positions, lies on one
// line and every CTA takes an equal stretch of it whatever the sequences' lengths are; a CTA
// whose stretch begins or ends inside a row leaves a partial result (sum, maximum, normaliser),
// and a second kernel joins those.  The stretches follow from the positions on the device, so a
// recorded launch serves every length.
//
// In a CTA each of four warps takes 16 of a page's positions and runs for itself: its copies
// (16-byte cp.async, ring of AE_STAGES tiles), its running maximum, its sums; the warps meet only at
// the end of a row.  Scores are the product K q^T with 16 positions as rows and 8 heads as
// columns, the sums V^T w with the head's dimensions as rows: e4m3 codes become half floats in
// registers (exactly), straight in the layout of the matrix instruction, because the order of
// dimensions along an inner product, and of rows in the result, is free: a thread converts the
// bytes that it has read 16 at a time.
//
// Precision: codes are exact in half; a query is scaled by a power of two and split into two
// halves (22 bits) where it is 32-bit, a bfloat16 one fits in one.  Weights are 32-bit, split the same
// way for 32-bit queries and rounded to 11 bits for bfloat16 ones, whose results keep 8.  The
// scale of a page's values is part of the weights, relative to the greatest one so far and times
// 2^14: a half holds a weight of up to 2^14 and, 11 bits, down to 2^-14.
#include "e4m3.cuh"

namespace {

constexpr int AE_WARPS = 4;
constexpr int AE_THREADS = 32 * AE_WARPS;
constexpr int AE_TILE = 16 * AE_WARPS;        // positions that a CTA's warps take together
constexpr int AE_HEADS = 8;                   // query heads of a row
constexpr int AE_MAX_DIM = 256;

struct AttendE4 {
    const void* q;
    long long ldq;
    void* out;
    const unsigned char *k_pool, *v_pool;
    const float *k_scale, *v_scale;
    const int *table, *slots, *positions;
    int B, n_slots, max_pages, n_pages, page, cap, nh, nkv, hd, hdv, window, keep_first;
    float scale, softcap;
    const float *sinks, *dist_bias;
    int n_dist, q_vec;
    int row_blocks;                           // blocks of 8 query heads of a kv head
    float* partial;                           // null: a CTA takes whole rows
};

// Head sizes are padded with zeros to DIM = 64, 128 or 256.
template <int DIM>
struct Tile {
    static constexpr int STAGES = DIM == 64 ? 4 : 3;
    static constexpr int CTAS = DIM == 256 ? 2 : DIM == 128 ? 3 : 5;     // resident on an SM
    // Row strides by which a warp's 16-byte reads meet every bank once: two key rows of 64 bytes,
    // four value rows of 32.
    static constexpr int KS = DIM == 64 ? 64 : DIM + 64, VS = DIM + 16;
    static constexpr int STAGE = 16 * (KS + VS);
    static constexpr int RED = DIM + 4;                                   // floats
    static constexpr int SMEM = AE_WARPS * STAGES * STAGE;
    static_assert(SMEM >= AE_WARPS * AE_HEADS * RED * 4, "the join of the warps uses the same memory");
    // a partial result: sums [8][DIM], then (maximum, normaliser) of the 8 heads
    static constexpr int PART = AE_HEADS * DIM + 2 * AE_HEADS;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ unsigned half2_of(float lo, float hi) {
    unsigned r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 float2_of(unsigned h) {
    float lo, hi;
    asm("{.reg .b16 a, b;\n mov.b32 {a, b}, %2;\n cvt.f32.f16 %0, a;\n cvt.f32.f16 %1, b;}"
        : "=f"(lo), "=f"(hi) : "r"(h));
    return make_float2(lo, hi);
}
__device__ __forceinline__ unsigned transposed(unsigned v) {              // of an 8 x 8 matrix of halves
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ void mma16816(float (&c)[4], unsigned a0, unsigned a1, unsigned a2, unsigned a3,
                                         unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 16 bytes to shared memory, zeros in the place of those behind the first ``bytes``
__device__ __forceinline__ void copy16(unsigned smem, const void* gmem, int bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem), "l"(gmem), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy4(unsigned smem, const void* gmem) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem), "l"(gmem) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// What a sequence's query sees: the positions first .. p and those below kept, in tiles of
// AE_TILE: tiles 0 .. kept_tiles - 1, then from first_tile on.
struct Seen {
    int slot, p, first, kept, kept_tiles, first_tile, tiles;
};
__device__ __forceinline__ Seen seen_by(const AttendE4& a, int b) {
    Seen s;
    s.slot = a.slots[b];
    s.p = a.positions[b];
    if (s.slot < 0 || s.slot >= a.n_slots || s.p < 0) {          // padding: one tile of nothing
        s.slot = -1;
        s.first = s.kept = s.kept_tiles = s.first_tile = 0;
        s.tiles = 1;
        return s;
    }
    s.first = max(first_visible(s.p, a.window), s.p - a.cap + 1);
    s.kept = s.p < a.cap ? min(a.keep_first, s.first) : 0;
    s.first_tile = s.first / AE_TILE;
    s.kept_tiles = min((s.kept + AE_TILE - 1) / AE_TILE, s.first_tile);
    s.tiles = s.kept_tiles + s.p / AE_TILE - s.first_tile + 1;
    return s;
}

// The sequences' tiles on one line.  ``scan``: 8 ints of shared memory.  All threads of a CTA of
// AE_THREADS take part and get the result.
__device__ __forceinline__ int all_tiles(const AttendE4& a, int* scan) {
    int n = 0;
    for (int b = threadIdx.x; b < a.B; b += AE_THREADS) n += seen_by(a, b).tiles;
    n = __reduce_add_sync(0xffffffffu, n);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) scan[threadIdx.x >> 5] = n;
    __syncthreads();
    return scan[0] + scan[1] + scan[2] + scan[3];
}
// The sequence that tile y of the line belongs to, and the tiles before it.
__device__ __forceinline__ void find_tile(const AttendE4& a, int y, int* scan, int& seq, int& before) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int done = 0;
    for (int base = 0; base < a.B; base += AE_THREADS) {
        const int b = base + threadIdx.x;
        const int n = b < a.B ? seen_by(a, b).tiles : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        __syncthreads();
        if (lane == 31) scan[warp] = upto;
        __syncthreads();
        int total = 0;
#pragma unroll
        for (int w = 0; w < AE_WARPS; ++w) {
            if (w < warp) upto += scan[w];
            total += scan[w];
        }
        if (y < done + total) {
            if (y >= done + upto - n && y < done + upto) { scan[4] = b; scan[5] = done + upto - n; }
            break;
        }
        done += total;
    }
    __syncthreads();
    seq = scan[4];
    before = scan[5];
}
__device__ __forceinline__ long long stretch_start(long long units, int cta, int ctas) {
    return units * cta / ctas;
}

// ---------------------------------------------------------------- the walk over the keys
template <typename T, int DIM>
__global__ void __launch_bounds__(AE_THREADS, Tile<DIM>::CTAS) attend_e4m3_kernel(const AttendE4 a) {
    using S = Tile<DIM>;
    constexpr bool SPLIT = sizeof(T) == 4;                       // two halves for a 32-bit value
    constexpr int NQ = DIM / 64, NT = DIM / 16;
    constexpr int VB = DIM >= 128 ? 16 : 8, NV = DIM / (8 * VB); // bytes of values at a time, times
    extern __shared__ __align__(128) unsigned char smem[];
    __shared__ int scan[8];
    __shared__ float stat[AE_WARPS][AE_HEADS][2];
    __shared__ float meta[AE_WARPS][S::STAGES][4];               // scales of keys and values, page is there
    pdl_wait();
    pdl_launch_next();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
    const int R = a.nkv * a.row_blocks, group = a.nh / a.nkv;
    unsigned char* mine = smem + warp * S::STAGES * S::STAGE;
    const unsigned mine_at = (unsigned)__cvta_generic_to_shared(mine);

    // this CTA's stretch
    int b, before, row;
    long long left;                                              // units still to do
    int tile;
    if (a.partial) {
        const int total = all_tiles(a, scan);
        const long long units = (long long)total * R;
        const long long x0 = stretch_start(units, blockIdx.x, gridDim.x);
        left = stretch_start(units, blockIdx.x + 1, gridDim.x) - x0;
        if (left == 0) return;
        find_tile(a, (int)(x0 / R), scan, b, before);
        const int n = seen_by(a, b).tiles;
        const long long in = x0 - (long long)before * R;
        row = (int)(in / n);
        tile = (int)(in - (long long)row * n);
    } else {
        b = blockIdx.x / R;
        row = blockIdx.x % R;
        tile = 0;
        left = seen_by(a, b).tiles;
    }
    int segment = 0;
    while (left > 0) {
        const Seen s = seen_by(a, b);
        const int g = row / a.row_blocks, h0 = g * group + row % a.row_blocks * AE_HEADS;
        const int heads = min(AE_HEADS, (g + 1) * group - h0);
        const int n = (int)min((long long)(s.tiles - tile), left);   // tiles of this segment
        const bool whole = n == s.tiles;
        if (s.slot < 0) {
            T* out = (T*)a.out + ((size_t)b * a.nh + h0) * a.hdv;
            for (int i = tid; i < heads * a.hdv; i += AE_THREADS) out[i] = from_f32<T>(0.f);
        } else {
            const int* table = a.table + (size_t)s.slot * a.max_pages;
            const size_t krow = (size_t)a.nkv * a.hd, vrow = (size_t)a.nkv * a.hdv;
            // position of this warp's part of tile i of the segment, and the page it lies in
            auto place = [&](int i) {
                const int t = tile + i;
                return (t < s.kept_tiles ? t : s.first_tile + t - s.kept_tiles) * AE_TILE + warp * 16;
            };
            auto page_of = [&](int i) {
                if (i >= n) return -1;
                const int j = place(i);
                return j <= s.p ? table[j % a.cap / a.page] : -1;
            };
            constexpr int LPR = DIM / 16, RPI = 32 / LPR;        // lanes a row, rows an instruction
            const int crow = lane / LPR, ccol = lane % LPR * 16;
            auto issue = [&](int i, int pg, int stage) {
                if (i < n) {
                    const int j0 = place(i);
                    const bool there = pg >= 0 && pg < a.n_pages;
                    const int page = there ? pg : 0;
                    const size_t at = (size_t)page * a.page + j0 % a.cap % a.page;
                    const unsigned char* k = a.k_pool + at * krow + (size_t)g * a.hd;
                    const unsigned char* v = a.v_pool + at * vrow + (size_t)g * a.hdv;
                    const unsigned ks = mine_at + stage * S::STAGE, vs = ks + 16 * S::KS;
                    const bool all = there && j0 >= s.first && j0 + 15 <= s.p;
#pragma unroll
                    for (int q = 0; q < 16 / RPI; ++q) {
                        const int rr = q * RPI + crow, j = j0 + rr;
                        const bool ok = all || (there && j <= s.p && (j >= s.first || j < s.kept));
                        const int kb = ok && ccol < a.hd ? 16 : 0, vb = ok && ccol < a.hdv ? 16 : 0;
                        copy16(ks + rr * S::KS + ccol, kb ? k + rr * krow + ccol : a.k_pool, kb);
                        copy16(vs + rr * S::VS + ccol, vb ? v + rr * vrow + ccol : a.v_pool, vb);
                    }
                    if (lane == 0) {
                        const unsigned at = (unsigned)__cvta_generic_to_shared(meta[warp][stage]);
                        copy4(at, a.k_scale + (size_t)page * a.nkv + g);
                        copy4(at + 4, a.v_scale + (size_t)page * a.nkv + g);
                        meta[warp][stage][2] = there ? 1.f : 0.f;
                    }
                }
                copies_commit();
            };
#pragma unroll
            for (int i = 0; i < S::STAGES - 1; ++i) issue(i, page_of(i), i);
            int next_page = page_of(S::STAGES - 1);

            // the queries: head r, dimensions i * 64 + c * 16 .. + 15
            unsigned qh[NQ][8], ql[SPLIT ? NQ : 1][8];
            float qf;                                            // what the scaled query was divided by
            {
                float x[NQ][16];
                const T* q = (const T*)a.q + (long long)b * a.ldq + (long long)(h0 + r) * a.hd;
                float most = 0.f;
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    const int d = i * 64 + c * 16;
                    const bool have = r < heads && d < a.hd;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[i][e] = 0.f;
                    if (have && a.q_vec) {
                        constexpr int PER = 16 / sizeof(T);
#pragma unroll
                        for (int e = 0; e < 16; e += PER) {
                            const uint4 u = *reinterpret_cast<const uint4*>(q + d + e);
                            const T* p = reinterpret_cast<const T*>(&u);
#pragma unroll
                            for (int f = 0; f < PER; ++f) x[i][e + f] = to_f32(p[f]);
                        }
                    } else if (have) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) x[i][e] = to_f32(q[d + e]);
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) most = fmaxf(most, fabsf(x[i][e]));
                }
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // to 2^9 .. 2^10 by a power of two (2^120 at most)
                const int e = (int)(__float_as_uint(most) >> 23) - 127;
                const int k = most > 0.f && e < 128 ? min(9 - e, 120) : 0;
                const float up = __uint_as_float((unsigned)(k + 127) << 23);
                qf = __uint_as_float((unsigned)(127 - k) << 23);
#pragma unroll
                for (int i = 0; i < NQ; ++i)
#pragma unroll
                    for (int f = 0; f < 8; ++f) {
                        const float u = x[i][2 * f] * up, v = x[i][2 * f + 1] * up;
                        qh[i][f] = half2_of(u, v);
                        if (SPLIT) {
                            const float2 w = float2_of(qh[i][f]);
                            ql[i][f] = half2_of(u - w.x, v - w.y);
                        }
                    }
            }
            // this thread's columns of the scores and sums: heads 2 c and 2 c + 1
            const float f0 = __shfl_sync(0xffffffffu, qf, 8 * c) * a.scale;
            const float f1 = __shfl_sync(0xffffffffu, qf, 8 * c + 4) * a.scale;
            const float* bias = a.dist_bias ? a.dist_bias + (size_t)min(h0 + 2 * c, a.nh - 1) * a.n_dist : nullptr;
            const float* bias1 = a.dist_bias ? a.dist_bias + (size_t)min(h0 + 2 * c + 1, a.nh - 1) * a.n_dist : nullptr;
            constexpr float LOG2E = 1.4426950408889634f;

            float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f, vref = 0.f, vlast = -1.f, vf = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;

            int stage = 0;
            for (int i = 0; i < n; ++i) {
                const int ahead = stage == 0 ? S::STAGES - 1 : stage - 1;
                issue(i + S::STAGES - 1, next_page, ahead);
                next_page = page_of(i + S::STAGES);
                copies_wait<S::STAGES - 1>();
                __syncwarp();
                const int j0 = place(i);
                if (j0 <= s.p && meta[warp][stage][2] != 0.f) {
                    const unsigned char* K = mine + stage * S::STAGE;
                    const unsigned char* V = K + 16 * S::KS;
                    const float ks = meta[warp][stage][0], vs = meta[warp][stage][1];
                    float x[2][4] = {};
                    float y[2][4] = {};
#pragma unroll
                    for (int q = 0; q < NQ; ++q) {
                        const uint4 ka = *reinterpret_cast<const uint4*>(K + r * S::KS + q * 64 + c * 16);
                        const uint4 kb = *reinterpret_cast<const uint4*>(K + (r + 8) * S::KS + q * 64 + c * 16);
                        const unsigned wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                        for (int f = 0; f < 4; ++f) {
                            const unsigned a0 = e4m3_to_half2(wa[f]), a2 = e4m3_to_half2(wa[f] >> 16);
                            const unsigned a1 = e4m3_to_half2(wb[f]), a3 = e4m3_to_half2(wb[f] >> 16);
                            mma16816(x[f & 1], a0, a1, a2, a3, qh[q][2 * f], qh[q][2 * f + 1]);
                            if (SPLIT) mma16816(y[f & 1], a0, a1, a2, a3, ql[q][2 * f], ql[q][2 * f + 1]);
                        }
                    }
                    // scores of positions j0 + r, j0 + r + 8 in units of ln 2
                    float p[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float v = x[0][e] + x[1][e];
                        if (SPLIT) v += y[0][e] + y[1][e];
                        const int j = j0 + r + (e >> 1) * 8;
                        v *= ks * (e & 1 ? f1 : f0);
                        if (a.softcap > 0.f) v = soft_capped(v, a.softcap);
                        if (a.dist_bias) v += (e & 1 ? bias1 : bias)[min(max(s.p - j, 0), a.n_dist - 1)];
                        const bool ok = j <= s.p && (j >= s.first || j < s.kept);
                        p[e] = ok ? v * LOG2E : -INFINITY;
                    }
                    float t0 = fmaxf(p[0], p[2]), t1 = fmaxf(p[1], p[3]);
#pragma unroll
                    for (int w = 4; w < 32; w <<= 1) {
                        t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, w));
                        t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, w));
                    }
                    t0 = fmaxf(t0, m0);
                    t1 = fmaxf(t1, m1);
                    const float u0 = t0 == -INFINITY ? 0.f : t0, u1 = t1 == -INFINITY ? 0.f : t1;
                    float k0 = ex2(m0 - u0), k1 = ex2(m1 - u1);
                    m0 = t0;
                    m1 = t1;
                    l0 *= k0;
                    l1 *= k1;
                    if (vs != vlast) {
                        vlast = vs;
                        if (!(vs <= vref)) {                      // the greatest scale so far
                            k0 *= vref / vs;
                            k1 *= vref / vs;
                            vref = vs;
                        }
                        vf = vs / vref * 16384.f;
                    }
                    if (__any_sync(0xffffffffu, k0 != 1.f || k1 != 1.f)) {
#pragma unroll
                        for (int t = 0; t < NT; ++t) {
                            o[t][0] *= k0;
                            o[t][1] *= k1;
                            o[t][2] *= k0;
                            o[t][3] *= k1;
                        }
                    }
                    p[0] = ex2(p[0] - u0);
                    p[1] = ex2(p[1] - u1);
                    p[2] = ex2(p[2] - u0);
                    p[3] = ex2(p[3] - u1);
                    l0 += p[0] + p[2];
                    l1 += p[1] + p[3];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] *= vf;
                    const unsigned h0w = half2_of(p[0], p[1]), h1w = half2_of(p[2], p[3]);
                    const unsigned b0 = transposed(h0w), b1 = transposed(h1w);
                    unsigned c0 = 0, c1 = 0;
                    if (SPLIT) {
                        const float2 w0 = float2_of(h0w), w1 = float2_of(h1w);
                        c0 = transposed(half2_of(p[0] - w0.x, p[1] - w0.y));
                        c1 = transposed(half2_of(p[2] - w1.x, p[3] - w1.y));
                    }
                    // values: dimensions q * 8 VB + r * VB .. of positions 2 c, 2 c + 1, 2 c + 8, 2 c + 9
#pragma unroll
                    for (int q = 0; q < NV; ++q) {
                        unsigned w[4][VB / 4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const unsigned char* at = V + (2 * c + (e & 1) + (e >> 1) * 8) * S::VS + q * 8 * VB + r * VB;
                            if constexpr (VB == 16) {
                                const uint4 u = *reinterpret_cast<const uint4*>(at);
                                w[e][0] = u.x; w[e][1] = u.y; w[e][2] = u.z; w[e][3] = u.w;
                            } else {
                                const uint2 u = *reinterpret_cast<const uint2*>(at);
                                w[e][0] = u.x; w[e][1] = u.y;
                            }
                        }
#pragma unroll
                        for (int f = 0; f < VB / 4; ++f) {
                            const unsigned la = __byte_perm(w[0][f], w[1][f], 0x5140), lb = __byte_perm(w[0][f], w[1][f], 0x7362);
                            const unsigned ha = __byte_perm(w[2][f], w[3][f], 0x5140), hb = __byte_perm(w[2][f], w[3][f], 0x7362);
                            const int t = q * (VB / 2) + 2 * f;
                            {
                                const unsigned a0 = e4m3_to_half2(la), a1 = e4m3_to_half2(la >> 16);
                                const unsigned a2 = e4m3_to_half2(ha), a3 = e4m3_to_half2(ha >> 16);
                                mma16816(o[t], a0, a1, a2, a3, b0, b1);
                                if (SPLIT) mma16816(o[t], a0, a1, a2, a3, c0, c1);
                            }
                            {
                                const unsigned a0 = e4m3_to_half2(lb), a1 = e4m3_to_half2(lb >> 16);
                                const unsigned a2 = e4m3_to_half2(hb), a3 = e4m3_to_half2(hb >> 16);
                                mma16816(o[t + 1], a0, a1, a2, a3, b0, b1);
                                if (SPLIT) mma16816(o[t + 1], a0, a1, a2, a3, c0, c1);
                            }
                        }
                    }
                }
                __syncwarp();                                    // the stage may be written again
                stage = stage + 1 == S::STAGES ? 0 : stage + 1;
            }
            // ---- the warps' results together
            copies_wait<0>();
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, w);
                l1 += __shfl_xor_sync(0xffffffffu, l1, w);
            }
            if (r == 0) {
                stat[warp][2 * c][0] = m0;
                stat[warp][2 * c][1] = l0;
                stat[warp][2 * c + 1][0] = m1;
                stat[warp][2 * c + 1][1] = l1;
            }
            __syncthreads();
            float M0 = -INFINITY, M1 = -INFINITY;
#pragma unroll
            for (int w = 0; w < AE_WARPS; ++w) {
                M0 = fmaxf(M0, stat[w][2 * c][0]);
                M1 = fmaxf(M1, stat[w][2 * c + 1][0]);
            }
            const float back = vref * (1.f / 16384.f);
            const float k0 = (M0 == -INFINITY ? 1.f : ex2(m0 - M0)) * back;
            const float k1 = (M1 == -INFINITY ? 1.f : ex2(m1 - M1)) * back;
            float* red = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                float* d0 = red + (warp * AE_HEADS + 2 * c) * S::RED + q * 8 * VB + r * VB;
                float* d1 = d0 + S::RED;
#pragma unroll
                for (int e = 0; e < VB / 4; ++e) {
                    const int t = q * (VB / 2) + 2 * e;
                    *reinterpret_cast<float4*>(d0 + 4 * e) =
                        make_float4(o[t][0] * k0, o[t][2] * k0, o[t + 1][0] * k0, o[t + 1][2] * k0);
                    *reinterpret_cast<float4*>(d1 + 4 * e) =
                        make_float4(o[t][1] * k1, o[t][3] * k1, o[t + 1][1] * k1, o[t + 1][3] * k1);
                }
            }
            __syncthreads();
            float* part = a.partial ? a.partial + (size_t)(2 * blockIdx.x + (segment > 0)) * S::PART : nullptr;
            for (int i = tid; i < heads * DIM; i += AE_THREADS) {
                const int h = i / DIM, d = i % DIM;
                if (d >= a.hdv) continue;
                float v = 0.f, L = 0.f, M = -INFINITY;
#pragma unroll
                for (int w = 0; w < AE_WARPS; ++w) {
                    v += red[(w * AE_HEADS + h) * S::RED + d];
                    M = fmaxf(M, stat[w][h][0]);
                }
#pragma unroll
                for (int w = 0; w < AE_WARPS; ++w)
                    L += stat[w][h][1] * (stat[w][h][0] == M || M == -INFINITY ? 1.f : ex2(stat[w][h][0] - M));
                if (!whole) {
                    part[h * DIM + d] = v;
                    if (d == 0) {
                        part[AE_HEADS * DIM + 2 * h] = M;
                        part[AE_HEADS * DIM + 2 * h + 1] = L;
                    }
                    continue;
                }
                if (a.sinks) {
                    const float sink = a.sinks[h0 + h] * LOG2E, N = fmaxf(M, sink);
                    const float f = M == -INFINITY ? 0.f : ex2(M - N);
                    L = L * f + ex2(sink - N);
                    v *= f;
                }
                ((T*)a.out)[((size_t)b * a.nh + h0 + h) * a.hdv + d] = from_f32<T>(L == 0.f ? 0.f : v / L);
            }
            __syncthreads();
        }
        // the next segment: the next row from its first tile on
        left -= n;
        ++segment;
        tile = 0;
        if (++row == R) {
            row = 0;
            ++b;
        }
    }
}

// ---------------------------------------------------------------- rows of several CTAs
// CTA (i, h) joins, for head h of 8, the row inside which the stretch of CTA i + 1 begins, if it is
// the first to begin there.
template <typename T, int DIM>
__global__ void __launch_bounds__(AE_THREADS) join_e4m3_kernel(const AttendE4 a, int ctas) {
    using S = Tile<DIM>;
    __shared__ int scan[8];
    pdl_wait();
    pdl_launch_next();
    const int R = a.nkv * a.row_blocks, group = a.nh / a.nkv, head = blockIdx.y, tid = threadIdx.x;
    const int total = all_tiles(a, scan);
    const long long units = (long long)total * R;
    const int i = blockIdx.x + 1;
    const long long x = stretch_start(units, i, ctas);
    if (x >= units) return;
    int b, before;
    find_tile(a, (int)(x / R), scan, b, before);
    const int n = seen_by(a, b).tiles;
    const int row = (int)((x - (long long)before * R) / n);
    const long long begin = (long long)before * R + (long long)row * n, end = begin + n;
    if (x == begin || stretch_start(units, i - 1, ctas) > begin) return;      // not inside, not the first
    const int g = row / a.row_blocks, h0 = g * group + row % a.row_blocks * AE_HEADS;
    if (h0 + head >= (g + 1) * group) return;
    constexpr int PER = (DIM + AE_THREADS - 1) / AE_THREADS;
    float v[PER] = {}, M = -INFINITY, L = 0.f;
    for (int j = i - 1; j < ctas; ++j) {
        const long long from = stretch_start(units, j, ctas);
        if (from >= end) break;
        if (stretch_start(units, j + 1, ctas) == from) continue;              // no work
        const float* part = a.partial + (size_t)(2 * j + (from < begin)) * S::PART;
        const float m = part[AE_HEADS * DIM + 2 * head], l = part[AE_HEADS * DIM + 2 * head + 1];
        const float N = fmaxf(M, m);
        const float f0 = N == -INFINITY ? 1.f : ex2(M - N), f1 = N == -INFINITY ? 1.f : ex2(m - N);
        M = N;
        L = L * f0 + l * f1;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            const int d = tid + e * AE_THREADS;
            if (d < a.hdv) v[e] = v[e] * f0 + part[head * DIM + d] * f1;
        }
    }
    if (a.sinks) {
        const float sink = a.sinks[h0 + head] * 1.4426950408889634f, N = fmaxf(M, sink);
        const float f = M == -INFINITY ? 0.f : ex2(M - N);
        L = L * f + ex2(sink - N);
#pragma unroll
        for (int e = 0; e < PER; ++e) v[e] *= f;
    }
    T* out = (T*)a.out + ((size_t)b * a.nh + h0 + head) * a.hdv;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const int d = tid + e * AE_THREADS;
        if (d < a.hdv) out[d] = from_f32<T>(L == 0.f ? 0.f : v[e] / L);
    }
}

struct Plan {
    int dim, ctas;             // padded head size; CTAs of the launch
    bool split;                // stretches of an equal number of tiles, joined afterwards
};
int sm_count() {
    static int n = 0;
    if (n == 0) {
        int dev = 0, v = 0;
        if (cudaGetDevice(&dev) == cudaSuccess &&
            cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
            n = v;
    }
    return n > 0 ? n : 148;
}
Plan plan_of(int B, int nh, int nkv, int hd, int hdv, int max_keys) {
    Plan p;
    const int most = hd > hdv ? hd : hdv;
    p.dim = most <= 64 ? 64 : most <= 128 ? 128 : 256;
    const long long rows = (long long)B * nkv * ((nh / nkv + AE_HEADS - 1) / AE_HEADS);
    const long long tiles = (max_keys + AE_TILE - 1) / AE_TILE + 1;
    const int resident = sm_count() * (p.dim == 256 ? Tile<256>::CTAS : p.dim == 128 ? Tile<128>::CTAS : Tile<64>::CTAS);
    p.split = tiles > 8;
    p.ctas = (int)(!p.split || rows * tiles < resident ? (p.split ? rows * tiles : rows) : resident);
    return p;
}
template <typename T, int DIM>
int launch(const AttendE4& a, const Plan& p, cudaStream_t stream) {
    AGV_CUDA_OK(cudaFuncSetAttribute(attend_e4m3_kernel<T, DIM>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     Tile<DIM>::SMEM));
    agv_launch(attend_e4m3_kernel<T, DIM>, p.ctas, AE_THREADS, Tile<DIM>::SMEM, stream, a);
    AGV_LAUNCH_OK("attend_e4m3_kernel");
    if (p.split && p.ctas > 1) {
        const int heads = a.nh / a.nkv < AE_HEADS ? a.nh / a.nkv : AE_HEADS;
        agv_launch(join_e4m3_kernel<T, DIM>, dim3(p.ctas - 1, heads), AE_THREADS, 0, stream, a, p.ctas);
        AGV_LAUNCH_OK("join_e4m3_kernel");
    }
    return 0;
}
template <typename T>
int launch_dim(const AttendE4& a, const Plan& p, cudaStream_t stream) {
    if (p.dim == 64) return launch<T, 64>(a, p, stream);
    if (p.dim == 128) return launch<T, 128>(a, p, stream);
    return launch<T, 256>(a, p, stream);
}

}  // namespace

// 32-bit values of scratch that agv_attention_decode_e4m3 wants for these sizes.
AGV_API long long agv_attention_decode_e4m3_scratch(int B, int nh, int nkv, int hd, int hdv, int max_keys) {
    AGV_REQUIRE(B >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0, "attention_decode_e4m3: bad sizes (%d query heads over %d)", nh, nkv);
    const Plan p = plan_of(B, nh, nkv, hd, hdv, max_keys);
    return p.split ? 2ll * p.ctas * (AE_HEADS * p.dim + 2 * AE_HEADS) : 0;
}

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
    if (B == 0) return 0;
    const Plan plan = plan_of(B, nh, nkv, hd, hdv, max_keys);
    AGV_REQUIRE(!plan.split || (partial && partial_floats >= agv_attention_decode_e4m3_scratch(B, nh, nkv, hd, hdv, max_keys)),
                "attention_decode_e4m3: %lld floats of scratch are too few", partial_floats);
    const size_t esz = dtype == AGV_F32 ? 4 : 2;
    const int q_vec = agv_aligned(q, 16) && (size_t)ldq * esz % 16 == 0;
    AttendE4 a{q, ldq, out, (const unsigned char*)k_pool, (const unsigned char*)v_pool, k_scale, v_scale,
               table, slots, positions, B, n_slots, max_pages, n_pages, page, cap, nh, nkv, hd, hdv,
               window, window ? keep_first : 0, scale, softcap, sinks, dist_bias, n_dist, q_vec,
               (nh / nkv + AE_HEADS - 1) / AE_HEADS, plan.split ? partial : nullptr};
    return dtype == AGV_F32 ? launch_dim<float>(a, plan, stream) : launch_dim<__nv_bfloat16>(a, plan, stream);
}

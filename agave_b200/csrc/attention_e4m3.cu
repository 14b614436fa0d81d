// Decode attention over the 8-bit cache: one query per sequence.
//
// o_a = sum_j w_aj v_j with w_aj = exp(s_aj - m) / (sum_j exp(s_aj - m) + exp(sink_a - m)),
// s_aj = cap(scale * q_a . k_j) + bias; one pass over the keys with a running maximum m.
//
// What bounds it is reading each key and value once, hd + hdv bytes a position and kv head.  The
// pages of all sequences, 64 positions each, lie on one line, which is cut into equal stretches
// whatever the sequences' lengths are; a CTA takes a stretch for one kv head and up to 8 of its query heads,
// and where that begins or ends inside a sequence it leaves a partial result (output, maximum,
// normaliser), which a second kernel joins.  The stretches follow from the positions on the device,
// so a recorded launch serves every length.  The CTAs of a stretch, a head each, lie beside each
// other on the grid and go through it together: a head's 64 to 256 bytes of a position are a part
// of what DRAM opens for it, and together they are all of it (64 sequences up to 8192 with 16
// kv heads of 128: 238 us with stretches that lay along the heads, 191 like this).
//
// In a CTA each of four warps takes 16 of a page's positions and runs for itself: its copies
// (16-byte cp.async, a ring of 3 or 4 tiles), its running maximum, its sums; the warps meet only at
// the end of a row.  Scores are the product K q^T with 16 positions as rows and 8 heads as
// columns, the sums V^T w with the head's dimensions as rows: e4m3 codes become half floats in
// registers (exactly), straight in the layout of the matrix instruction, because the order of
// dimensions along an inner product, and of rows in the result, is free: a thread converts the
// bytes that it has read 16 at a time.  (The conversions run on the integer pipe and are the most of
// what keeps it half busy; V's by shifts instead were slower, 281 us against 247.)
// The next tile's products stand beside a tile's softmax and fill its waits (247 us, 238 with).
//
// Precision: codes are exact in half; a query is scaled by a power of two and split into two
// halves (22 bits) where it is 32-bit; a bfloat16 one fits in one (elements below 2^-26 of a head's
// greatest keep fewer bits: they are off by up to 2^-34 of it).  Weights are 32-bit, split the same
// way for 32-bit queries and rounded to 11 bits for bfloat16 ones, whose results keep 8.  The scale 2^e
// of a page's values is part of the weights that are multiplied with them: the products e^s 2^e have
// a reference of their own, the greatest so far, apart from the maximum of the scores, which the
// normaliser goes by (so a page with a great scale and no weight takes no bits from the others).
// Against it and times 2^14 a half holds a product of up to 2^14 and, 11 bits, down to 2^-14; what is
// smaller is off by 2^-39 of the greatest.  A warp's sums are divided by the normaliser before they
// leave their reference: they are values again, in 32 bits as those are, and joining them
// takes nothing but the maxima and normalisers.
#include "e4m3.cuh"
#include <atomic>
#include <cfloat>

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
    int n_dist, q_vec, page_bits;
    int row_blocks;                           // blocks of 8 query heads of a kv head
    int cluster;                              // CTAs that share a row where there are no stretches
    float* partial;                           // null: no stretches
};

// Head sizes are padded with zeros to DIM = 64, 128 or 256.
template <int DIM>
struct Tile {
    // Tiles of a warp's ring and CTAs resident on an SM: what registers (a row's sums are DIM / 4 of a
    // thread's) and shared memory allow.  More warps with fewer registers were slower (256: three CTAs
    // 67 us where two take 61; 128: four 261 us, three 250), more tiles the same.
    static constexpr int STAGES = DIM == 64 ? 4 : 3;
    static constexpr int CTAS = DIM == 256 ? 2 : DIM == 128 ? 3 : 5;
    // A warp's 16-byte reads meet every bank once: of two key rows 64 bytes each, which lie in
    // different halves of 128 bytes (odd rows of 128 bytes or more have them exchanged), of four
    // value rows 32 bytes each, by the stride.
    static constexpr int KS = DIM, VS = DIM + 16;
    static constexpr int STAGE = 16 * (KS + VS);
    static constexpr int RED = DIM + 4;                                   // floats
    static constexpr int SMEM = AE_WARPS * STAGES * STAGE;
    static_assert(SMEM >= AE_WARPS * AE_HEADS * RED * 4, "the join of the warps uses the same memory");
    // a partial result: outputs [8][DIM], then (maximum, normaliser) of the 8 heads
    static constexpr int PART = AE_HEADS * DIM + 2 * AE_HEADS;
};

// 2^(d + e) for d <= 0 and a whole number e as two factors, neither of which leaves the range where their
// product with something does not; d = -inf: 0.
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((unsigned)(max(e, -126) + 127) << 23); }
__device__ __forceinline__ float2 two_factors(float d, float e) {
    const float whole = fmaxf(rintf(d), -500.f);
    const int t = (int)(whole + e), half = t >> 1;
    return make_float2(power_of_two(half), ex2(d - whole) * power_of_two(t - half));
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

__device__ __forceinline__ int stretch_start(int total, int part, int stretches) {
    return (int)((long long)total * part / stretches);
}
// Where a stretch begins: the tiles of all sequences, the stretch's first one and its end, the sequence
// it lies in and the tiles before that sequence.
struct Start {
    int total, x0, x1, seq, before, tiles;
};
// The sequences' tiles on one line, and on it the stretch ``part`` of so many.  All AE_THREADS of
// the CTA take part and get the result (seq -1 where it begins behind the last tile).
__device__ __forceinline__ Start find_stretch(const AttendE4& a, int part, int stretches) {
    __shared__ int sums[AE_WARPS], found[3];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Start at;
    // up to AE_THREADS sequences in one go, else all of them first and then one group after the other
    int n = 0, b = threadIdx.x;
    if (a.B <= AE_THREADS) {
        n = b < a.B ? seen_by(a, b).tiles : 0;
    } else {
        int all = 0;
        for (; b < a.B; b += AE_THREADS) all += seen_by(a, b).tiles;
        all = __reduce_add_sync(0xffffffffu, all);
        if (lane == 0) sums[warp] = all;
        __syncthreads();
        at.total = 0;
#pragma unroll
        for (int w = 0; w < AE_WARPS; ++w) at.total += sums[w];
        __syncthreads();
    }
    at.seq = -1;
    int done = 0;
    for (int base = 0; base < a.B; base += AE_THREADS) {
        b = base + threadIdx.x;
        if (a.B > AE_THREADS) n = b < a.B ? seen_by(a, b).tiles : 0;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        if (lane == 31) sums[warp] = upto;
        __syncthreads();
        int group = 0;
#pragma unroll
        for (int w = 0; w < AE_WARPS; ++w) {
            if (w < warp) upto += sums[w];
            group += sums[w];
        }
        if (a.B <= AE_THREADS) at.total = group;
        at.x0 = stretch_start(at.total, part, stretches);
        at.x1 = stretch_start(at.total, part + 1, stretches);
        if (at.x0 >= at.total) return at;                        // (the same for every thread)
        const bool here = at.x0 < done + group;
        if (here && at.x0 >= done + upto - n && at.x0 < done + upto) {
            found[0] = b;
            found[1] = done + upto - n;
            found[2] = n;
        }
        __syncthreads();
        if (here) break;
        done += group;
    }
    at.seq = found[0];
    at.before = found[1];
    at.tiles = found[2];
    return at;
}

__device__ __forceinline__ void cluster_meet() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ float peer_f32(const void* mine, int rank) {
    unsigned at;
    float v;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"((unsigned)__cvta_generic_to_shared(mine)), "r"(rank));
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
    return v;
}
// The CTAs of a cluster join their results for a row: each brings its warps' outputs together in its
// own shared memory, and writes its share of the row's from everybody's.  ml: the maximum and normaliser
// of each head in this CTA.
template <typename T, int DIM>
__device__ __forceinline__ void share_row(const AttendE4& a, float* red, const float (*ml)[2], int b, int h0,
                                          int heads) {
    using S = Tile<DIM>;
    __shared__ float2 weight[AE_HEADS][16];
    const int tid = threadIdx.x, C = a.cluster, rank = blockIdx.x % C;
    for (int i = tid; i < heads * DIM; i += AE_THREADS) {
        float* at = red + i / DIM * S::RED + i % DIM;
        float v = 0.f;
#pragma unroll
        for (int w = 0; w < AE_WARPS; ++w) v += at[w * AE_HEADS * S::RED];
        *at = v;
    }
    cluster_meet();
    // a thread a (head, CTA): what the CTA's outputs are multiplied by
    static_assert(AE_THREADS == 16 * AE_HEADS, "16 CTAs at most for each of the heads");
    {
        const int h = tid >> 4, r = tid & 15;
        float m = -INFINITY, l = 0.f;
        if (r < C) {
            m = peer_f32(&ml[h][0], r);
            l = peer_f32(&ml[h][1], r);
        }
        float M = m;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
        const float sink = a.sinks && h < heads ? a.sinks[h0 + h] * 1.4426950408889634f : -INFINITY;
        M = fmaxf(M, sink);
        if (M == -INFINITY) M = 0.f;
        float L = l * ex2(m - M);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) L += __shfl_xor_sync(0xffffffffu, L, o);
        L += ex2(sink - M);
        const float2 f = two_factors(m - M, 0.f);
        weight[h][r] = make_float2(f.x, L == 0.f ? 0.f : f.y * __fdividef(l, L));
    }
    __syncthreads();
    T* out = (T*)a.out + ((size_t)b * a.nh + h0) * a.hdv;
    for (int i = rank * AE_THREADS + tid; i < heads * a.hdv; i += C * AE_THREADS) {
        const int h = i / a.hdv, d = i % a.hdv;
        float v = 0.f;
#pragma unroll 4
        for (int r = 0; r < C; ++r) v += peer_f32(red + h * S::RED + d, r) * weight[h][r].x * weight[h][r].y;
        out[i] = from_f32<T>(v);
    }
    cluster_meet();                            // (a CTA's memory stays until its peers have read it)
}

// ---------------------------------------------------------------- the walk over the keys
// EXTRAS: a soft cap or a bias by distance.
template <typename T, int DIM, bool EXTRAS>
__global__ void __launch_bounds__(AE_THREADS, Tile<DIM>::CTAS) attend_e4m3_kernel(const AttendE4 a) {
    using S = Tile<DIM>;
    constexpr bool SPLIT = sizeof(T) == 4;                       // two halves for a 32-bit value
    constexpr int NQ = DIM / 64, NT = DIM / 16;
    constexpr int VB = DIM >= 128 ? 16 : 8, NV = DIM / (8 * VB); // bytes of values at a time, times
    extern __shared__ __align__(128) unsigned char smem[];
    // maxima and normalisers of the heads, each warp's and the CTA's
    __shared__ __align__(16) float stat[AE_WARPS][AE_HEADS][2], ml[AE_HEADS][2];
    __shared__ float meta[AE_WARPS][S::STAGES][4];               // scales of keys and values, page is there
    pdl_wait();
    pdl_launch_next();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, r = lane >> 2, c = lane & 3;
    const int R = a.nkv * a.row_blocks, group = a.nh / a.nkv;
    unsigned char* mine = smem + warp * S::STAGES * S::STAGE;
    const unsigned mine_at = (unsigned)__cvta_generic_to_shared(mine);

    // this CTA's row (a kv head and up to 8 of its query heads), sequence, tile and tiles left to do
    int b, row, tile, left;
    if (a.partial) {
        const int stretches = gridDim.x / R, part = blockIdx.x / R;
        row = blockIdx.x % R;
        const Start at = find_stretch(a, part, stretches);
        // (what the join has to know of the stretch)
        if (row == 0 && tid == 0)
            reinterpret_cast<int4*>(a.partial)[part] =
                make_int4(at.seq, at.before, at.seq < 0 ? 0 : at.before + at.tiles, at.total);
        b = at.seq;
        tile = at.x0 - at.before;
        left = at.x1 - at.x0;
        if (b < 0 || left == 0) return;
    } else {
        const int unit = blockIdx.x / a.cluster, part = blockIdx.x % a.cluster;
        b = unit / R;
        row = unit % R;
        const int n = seen_by(a, b).tiles;
        tile = n * part / a.cluster;
        left = n * (part + 1) / a.cluster - tile;
    }
    const bool shared_row = !a.partial && a.cluster > 1;
    int segment = 0;
    while (left > 0 || (shared_row && segment == 0)) {
        const Seen s = seen_by(a, b);
        const int g = row / a.row_blocks, h0 = g * group + row % a.row_blocks * AE_HEADS;
        const int heads = min(AE_HEADS, (g + 1) * group - h0);
        const int n = min(s.tiles - tile, left);                     // tiles of this segment
        const bool whole = n == s.tiles;
        if (s.slot < 0) {
            // padding (of a cluster the CTA that has its one tile)
            T* out = (T*)a.out + ((size_t)b * a.nh + h0) * a.hdv;
            for (int i = tid; i < heads * a.hdv && left > 0; i += AE_THREADS) out[i] = from_f32<T>(0.f);
        } else {
            const int* table = a.table + (size_t)s.slot * a.max_pages;
            const size_t krow = (size_t)a.nkv * a.hd, vrow = (size_t)a.nkv * a.hdv;
            // The tiles are visited in order, this warp's 16 positions of each: their first position and
            // its row of the ring, one step after the other (a division only where the kept tiles end).
            struct Place {
                int t, j, row;
            };
            auto start = [&](int t) {
                Place at;
                at.t = t;
                at.j = (t < s.kept_tiles ? t : s.first_tile + t - s.kept_tiles) * AE_TILE + warp * 16;
                at.row = at.j % a.cap;
                return at;
            };
            auto advance = [&](Place& at) {
                if (++at.t == s.kept_tiles) {
                    at = start(at.t);
                } else {
                    at.j += AE_TILE;
                    at.row += AE_TILE;
                    while (at.row >= a.cap) at.row -= a.cap;
                }
            };
            const int t_end = tile + n;
            auto page_of = [&](const Place& at) {
                return at.t < t_end && at.j <= s.p ? table[at.row >> a.page_bits] : -1;
            };
            constexpr int LPR = DIM / 16, RPI = 32 / LPR;        // lanes a row, rows an instruction
            const int crow = lane / LPR, ccol = lane % LPR * 16;
            const int flip = DIM > 64 ? (crow & 1) * 64 : 0;
            const unsigned copy_at = mine_at + crow * S::KS + (ccol ^ flip);
            const unsigned copy_vat = mine_at + 16 * S::KS + crow * S::VS + ccol;
            const int k_bytes = ccol < a.hd ? 16 : 0, v_bytes = ccol < a.hdv ? 16 : 0;
            const unsigned char* k_from = a.k_pool + (size_t)crow * krow + (size_t)g * a.hd + (k_bytes ? ccol : 0);
            const unsigned char* v_from = a.v_pool + (size_t)crow * vrow + (size_t)g * a.hdv + (v_bytes ? ccol : 0);
            auto issue = [&](const Place& at, int pg, int stage) {
                if (at.t < t_end) {
                    const bool there = pg >= 0 && pg < a.n_pages;
                    const int page = there ? pg : 0;
                    const size_t from = ((size_t)page << a.page_bits) + (at.row & (a.page - 1));
                    const unsigned char *k = k_from + from * krow, *v = v_from + from * vrow;
                    const unsigned ks = copy_at + stage * S::STAGE, vs = copy_vat + stage * S::STAGE;
                    if (there && at.j >= s.first && at.j + 15 <= s.p) {
#pragma unroll
                        for (int q = 0; q < 16 / RPI; ++q) {
                            copy16(ks + q * RPI * S::KS, k, k_bytes);
                            copy16(vs + q * RPI * S::VS, v, v_bytes);
                            k += RPI * krow;
                            v += RPI * vrow;
                        }
                    } else {
                        // (rows that are not seen become zeros: whatever their codes are, they add nothing)
#pragma unroll
                        for (int q = 0; q < 16 / RPI; ++q) {
                            const int j = at.j + q * RPI + crow;
                            const bool ok = there && j <= s.p && (j >= s.first || j < s.kept);
                            copy16(ks + q * RPI * S::KS, k, ok ? k_bytes : 0);
                            copy16(vs + q * RPI * S::VS, v, ok ? v_bytes : 0);
                            k += RPI * krow;
                            v += RPI * vrow;
                        }
                    }
                    if (lane == 0) {
                        const unsigned to = (unsigned)__cvta_generic_to_shared(meta[warp][stage]);
                        copy4(to, a.k_scale + (size_t)page * a.nkv + g);
                        copy4(to + 4, a.v_scale + (size_t)page * a.nkv + g);
                        meta[warp][stage][2] = there ? 1.f : 0.f;
                    }
                }
                copies_commit();
            };
            Place now = start(tile), next = now;
#pragma unroll
            for (int i = 0; i < S::STAGES - 1; ++i) {
                issue(next, page_of(next), i);
                advance(next);
            }
            int next_page = page_of(next);

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
            constexpr float LOG2E = 1.4426950408889634f;
            // (the cap by its exponential, off by some 2^-22 of the cap at most: as much as a score of its size
            // is in 32 bits, and 4.6 of 16 us less than tanhf and a division took for 66 rows of 1500 keys)
            const float cap_unit = EXTRAS && a.softcap > 0.f ? 2.f * LOG2E / a.softcap : 0.f;
            const float unit = EXTRAS ? a.scale : a.scale * LOG2E;
            const float f0 = __shfl_sync(0xffffffffu, qf, 8 * c) * unit;
            const float f1 = __shfl_sync(0xffffffffu, qf, 8 * c + 4) * unit;
            const float* bias = a.dist_bias ? a.dist_bias + (size_t)min(h0 + 2 * c, a.nh - 1) * a.n_dist : nullptr;
            const float* bias1 = a.dist_bias ? a.dist_bias + (size_t)min(h0 + 2 * c + 1, a.nh - 1) * a.n_dist : nullptr;

            float o[NT][4], m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
            // the sums' references: e^u0 2^e0, e^u1 2^e1; the maxima above u0, u1
            float u0 = -INFINITY, u1 = -INFINITY, e0 = 0.f, e1 = 0.f, g0 = 0.f, g1 = 0.f;
#pragma unroll
            for (int t = 0; t < NT; ++t) o[t][0] = o[t][1] = o[t][2] = o[t][3] = 0.f;

            // K q^T of a stage: positions r, r + 8 of heads 2 c, 2 c + 1, without any factor
            auto products = [&](int stage, float (&s)[4]) {
                const unsigned char* K = mine + stage * S::STAGE + r * S::KS + c * 16;
                const int half = DIM > 64 ? (r & 1) * 64 : 0;
                float x[2][4] = {};
                float y[2][4] = {};
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    const unsigned char* at = K + q * 64 + (q & 1 ? -half : half);
                    const uint4 ka = *reinterpret_cast<const uint4*>(at);
                    const uint4 kb = *reinterpret_cast<const uint4*>(at + 8 * S::KS);
                    const unsigned wa[4] = {ka.x, ka.y, ka.z, ka.w}, wb[4] = {kb.x, kb.y, kb.z, kb.w};
#pragma unroll
                    for (int f = 0; f < 4; ++f) {
                        unsigned a0, a1, a2, a3;
                        e4m3_word(wa[f], a0, a2);
                        e4m3_word(wb[f], a1, a3);
                        mma16816(x[f & 1], a0, a1, a2, a3, qh[q][2 * f], qh[q][2 * f + 1]);
                        if (SPLIT) mma16816(y[f & 1], a0, a1, a2, a3, ql[q][2 * f], ql[q][2 * f + 1]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) s[e] = x[0][e] + x[1][e] + (SPLIT ? y[0][e] + y[1][e] : 0.f);
            };
            copies_wait<S::STAGES - 2>();
            __syncwarp();
            float p[4];
            products(0, p);
            int stage = 0;
            while (now.t < t_end) {
                issue(next, next_page, stage == 0 ? S::STAGES - 1 : stage - 1);
                advance(next);
                next_page = page_of(next);
                copies_wait<S::STAGES - 2>();                    // the tile after this one is there
                __syncwarp();
                // Its products are independent of what follows, this tile's softmax and sums, whose
                // chains of instructions they fill (behind the last tile: of anything, and not used).
                const int after = stage + 1 == S::STAGES ? 0 : stage + 1;
                float p_after[4];
                products(after, p_after);

                const int j0 = now.j;
                const unsigned char* V = mine + stage * S::STAGE + 16 * S::KS;
                const bool there = meta[warp][stage][2] != 0.f;
                const float ks = meta[warp][stage][0], vs = there ? meta[warp][stage][1] : 0.f;
                // the values' scale as vf 2^ve (vf is 1 for a power of two), 2^14 with it
                const unsigned vb = min(__float_as_uint(vs) >> 23 & 0xffu, 253u);
                const float ve = __uint_as_float(0x4b000000u | vb) - 8388735.f;      // (2^23 + vb) - 2^23 - 127
                const float vf = vs * __uint_as_float((254u - vb) << 23) * 16384.f;
                const float s0 = ks * f0, s1 = ks * f1;
                // scores of positions j0 + r, j0 + r + 8 in units of ln 2
                const int ja = j0 + r, jb = ja + 8;
                const bool see_a = there && ja <= s.p && (ja >= s.first || ja < s.kept);
                const bool see_b = there && jb <= s.p && (jb >= s.first || jb < s.kept);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    p[e] *= e & 1 ? s1 : s0;
                    if (EXTRAS) {
                        if (a.softcap > 0.f) p[e] = soft_capped_ex2(p[e], cap_unit, a.softcap);
                        if (a.dist_bias) p[e] += (e & 1 ? bias1 : bias)[min(max(s.p - (e >> 1 ? jb : ja), 0), a.n_dist - 1)];
                        // (a finite score stays finite: a bias of the type's lowest value is no -inf, and
                        // where every key has it they weigh the same)
                        const float x = p[e] * LOG2E;
                        p[e] = x == -INFINITY && p[e] != -INFINITY ? -FLT_MAX : x;
                    }
                    if (!(e >> 1 ? see_b : see_a)) p[e] = -INFINITY;
                }
                float t0 = fmaxf(p[0], p[2]), t1 = fmaxf(p[1], p[3]);
#pragma unroll
                for (int w = 4; w < 32; w <<= 1) {
                    t0 = fmaxf(t0, __shfl_xor_sync(0xffffffffu, t0, w));
                    t1 = fmaxf(t1, __shfl_xor_sync(0xffffffffu, t1, w));
                }
                // A greater maximum, a greater product of a weight and its scale than any before (neither is so where
                // no key is seen), or a scale so far above the reference's that products matter where the
                // weights, as 32-bit numbers, are 0?
                const float d0 = ve - e0, d1 = ve - e1;
                float x0 = g0 + d0, x1 = g1 + d1;
                const float up0 = (t0 - u0) + d0, up1 = (t1 - u1) + d1;
                bool far = false;
                if (__any_sync(0xffffffffu, t0 > m0 || t1 > m1 || up0 > 0.f || up1 > 0.f || fmaxf(x0, x1) > 60.f)) {
                    if (t0 > m0) {
                        l0 *= ex2(m0 - t0);
                        m0 = t0;
                    }
                    if (t1 > m1) {
                        l1 *= ex2(m1 - t1);
                        m1 = t1;
                    }
                    float k0 = 1.f, k1 = 1.f;
                    if (up0 > 0.f) {
                        k0 = ex2(-up0);
                        u0 = t0;
                        e0 = ve;
                    }
                    if (up1 > 0.f) {
                        k1 = ex2(-up1);
                        u1 = t1;
                        e1 = ve;
                    }
                    g0 = m0 == u0 ? 0.f : m0 - u0;               // (both -inf: nothing seen yet)
                    g1 = m1 == u1 ? 0.f : m1 - u1;
                    x0 = g0 + (ve - e0);
                    x1 = g1 + (ve - e1);
                    far = __any_sync(0xffffffffu, fmaxf(x0, x1) > 60.f);
#pragma unroll
                    for (int t = 0; t < NT; ++t) {
                        o[t][0] *= k0;
                        o[t][1] *= k1;
                        o[t][2] *= k0;
                        o[t][3] *= k1;
                    }
                }
                const float n0 = m0 == -INFINITY ? 0.f : m0, n1 = m1 == -INFINITY ? 0.f : m1;
                if (!far) {
                    const float k0 = ex2(x0) * vf, k1 = ex2(x1) * vf;
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] = ex2(p[e] - (e & 1 ? n1 : n0));
                    l0 += p[0] + p[2];
                    l1 += p[1] + p[3];
#pragma unroll
                    for (int e = 0; e < 4; ++e) p[e] *= e & 1 ? k1 : k0;
                } else {
                    const float w0 = u0 == -INFINITY ? 0.f : u0, w1 = u1 == -INFINITY ? 0.f : u1;
                    l0 += ex2(p[0] - n0) + ex2(p[2] - n0);
                    l1 += ex2(p[1] - n1) + ex2(p[3] - n1);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        p[e] = ex2((p[e] - (e & 1 ? w1 : w0)) + (ve - (e & 1 ? e1 : e0))) * vf;
                }
                const unsigned h0w = half2_of(p[0], p[1]), h1w = half2_of(p[2], p[3]);
                const unsigned b0 = transposed(h0w), b1 = transposed(h1w);
                unsigned c0 = 0, c1 = 0;
                if (SPLIT) {
                    const float2 x0 = float2_of(h0w), x1 = float2_of(h1w);
                    c0 = transposed(half2_of(p[0] - x0.x, p[1] - x0.y));
                    c1 = transposed(half2_of(p[2] - x1.x, p[3] - x1.y));
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
                        const unsigned la = __byte_perm(w[0][f], w[1][f], 0x5140);
                        const unsigned lb = __byte_perm(w[0][f], w[1][f], 0x7362);
                        const unsigned ha = __byte_perm(w[2][f], w[3][f], 0x5140);
                        const unsigned hb = __byte_perm(w[2][f], w[3][f], 0x7362);
                        const int t = q * (VB / 2) + 2 * f;
                        unsigned a0, a1, a2, a3;
                        e4m3_word(la, a0, a1);
                        e4m3_word(ha, a2, a3);
                        mma16816(o[t], a0, a1, a2, a3, b0, b1);
                        if (SPLIT) mma16816(o[t], a0, a1, a2, a3, c0, c1);
                        e4m3_word(lb, a0, a1);
                        e4m3_word(hb, a2, a3);
                        mma16816(o[t + 1], a0, a1, a2, a3, b0, b1);
                        if (SPLIT) mma16816(o[t + 1], a0, a1, a2, a3, c0, c1);
                    }
                }
                __syncwarp();                                    // the stage may be written again
                stage = after;
                advance(now);
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = p_after[e];
            }
            // ---- the warps' results together
            copies_wait<0>();
#pragma unroll
            for (int w = 4; w < 32; w <<= 1) {
                l0 += __shfl_xor_sync(0xffffffffu, l0, w);
                l1 += __shfl_xor_sync(0xffffffffu, l1, w);
            }
            if (r == 0) *reinterpret_cast<float4*>(stat[warp][2 * c]) = make_float4(m0, l0, m1, l1);
            __syncthreads();
            // the CTA's, with the sink where this is all of the row
            float M0 = -INFINITY, M1 = -INFINITY, L0, L1;
            {
                float4 of[AE_WARPS];
#pragma unroll
                for (int w = 0; w < AE_WARPS; ++w) {
                    of[w] = *reinterpret_cast<const float4*>(stat[w][2 * c]);
                    M0 = fmaxf(M0, of[w].x);
                    M1 = fmaxf(M1, of[w].z);
                }
                float sink0 = -INFINITY, sink1 = -INFINITY;
                if (a.sinks && whole && !shared_row) {
                    if (2 * c < heads) sink0 = a.sinks[h0 + 2 * c] * LOG2E;
                    if (2 * c + 1 < heads) sink1 = a.sinks[h0 + 2 * c + 1] * LOG2E;
                    M0 = fmaxf(M0, sink0);
                    M1 = fmaxf(M1, sink1);
                }
                const float n0 = M0 == -INFINITY ? 0.f : M0, n1 = M1 == -INFINITY ? 0.f : M1;
                L0 = ex2(sink0 - n0);
                L1 = ex2(sink1 - n1);
#pragma unroll
                for (int w = 0; w < AE_WARPS; ++w) {
                    L0 = fmaf(of[w].y, ex2(of[w].x - n0), L0);
                    L1 = fmaf(of[w].w, ex2(of[w].z - n1), L1);
                }
                if (tid < 4) *reinterpret_cast<float4*>(ml[2 * c]) = make_float4(M0, L0, M1, L1);
                M0 = n0;
                M1 = n1;
            }
            // what brings this warp's sums to outputs: 2^-14 e^(u - maximum) 2^e / normaliser
            float2 k0 = two_factors(u0 - M0, e0), k1 = two_factors(u1 - M1, e1);
            k0.y *= L0 == 0.f ? 0.f : __fdividef(1.f / 16384.f, L0);
            k1.y *= L1 == 0.f ? 0.f : __fdividef(1.f / 16384.f, L1);
            float* red = reinterpret_cast<float*>(smem);
#pragma unroll
            for (int q = 0; q < NV; ++q) {
                float* d0 = red + (warp * AE_HEADS + 2 * c) * S::RED + q * 8 * VB + r * VB;
                float* d1 = d0 + S::RED;
#pragma unroll
                for (int e = 0; e < VB / 4; ++e) {
                    const int t = q * (VB / 2) + 2 * e;
                    *reinterpret_cast<float4*>(d0 + 4 * e) =
                        make_float4(o[t][0] * k0.y * k0.x, o[t][2] * k0.y * k0.x, o[t + 1][0] * k0.y * k0.x,
                                    o[t + 1][2] * k0.y * k0.x);
                    *reinterpret_cast<float4*>(d1 + 4 * e) =
                        make_float4(o[t][1] * k1.y * k1.x, o[t][3] * k1.y * k1.x, o[t + 1][1] * k1.y * k1.x,
                                    o[t + 1][3] * k1.y * k1.x);
                }
            }
            __syncthreads();
            float* part = nullptr;
            if (a.partial) part = a.partial + gridDim.x / R * 4 + (size_t)(2 * blockIdx.x + (segment > 0)) * S::PART;
            if (shared_row) {
                share_row<T, DIM>(a, red, ml, b, h0, heads);
                return;
            }
            for (int i = tid; i < heads * DIM; i += AE_THREADS) {
                const int h = i / DIM, d = i % DIM;
                if (d >= a.hdv) continue;
                float v = 0.f;
#pragma unroll
                for (int w = 0; w < AE_WARPS; ++w) v += red[(w * AE_HEADS + h) * S::RED + d];
                if (whole) {
                    ((T*)a.out)[((size_t)b * a.nh + h0 + h) * a.hdv + d] = from_f32<T>(v);
                    continue;
                }
                part[h * DIM + d] = v;
                if (d < 2) part[AE_HEADS * DIM + 2 * h + d] = ml[h][d];
            }
            __syncthreads();
        }
        // the next segment: the next sequence from its first tile on
        left -= n;
        ++segment;
        tile = 0;
        ++b;
    }
}

// ---------------------------------------------------------------- rows of several CTAs
// CTA (i, h, r) joins, for head h of 8 of row r (and every gridDim.y-th after it), the sequence inside
// which stretch i + 1 begins, if it is the first to begin there.  First the partial results' weights, a thread each, then the sums:
// DIM / 4 threads take a partial result, the CTA 8 to 32 of them at a time.
constexpr int AE_JOIN_THREADS = 512;
constexpr int AE_MAX_STRETCHES = 1024;
template <typename T, int DIM>
__global__ void __launch_bounds__(AE_JOIN_THREADS) join_e4m3_kernel(const AttendE4 a, int stretches) {
    using S = Tile<DIM>;
    __shared__ float2 weight[AE_MAX_STRETCHES];
    __shared__ int slot[AE_MAX_STRETCHES];
    __shared__ float scratch[32];
    __shared__ float4 sums[AE_JOIN_THREADS];
    pdl_wait();
    pdl_launch_next();
    const int R = a.nkv * a.row_blocks, group = a.nh / a.nkv, row = blockIdx.z, tid = threadIdx.x;
    const int g = row / a.row_blocks, h0 = g * group + row % a.row_blocks * AE_HEADS;
    const int i = blockIdx.x + 1;
    const int4 at = reinterpret_cast<const int4*>(a.partial)[i];               // of the stretch: (sequence, its tiles, all)
    const int b = at.x, begin = at.y, end = at.z, total = at.w;
    // (one behind the last tile; one that begins with the sequence; not the first to begin inside it)
    if (b < 0 || stretch_start(total, i, stretches) == begin || stretch_start(total, i - 1, stretches) > begin) return;
    // the stretches i - 1 .. last have a part of the sequence (but for empty ones)
    const int last = (int)(((long long)end * stretches - 1) / total), parts = last - i + 2;
    const float* partial = a.partial + 4 * stretches;
    for (int head = blockIdx.y; head < AE_HEADS && h0 + head < (g + 1) * group; head += gridDim.y) {
        __syncthreads();                           // (the head before has been read)
        float M = -INFINITY;
        for (int j = tid; j < parts; j += AE_JOIN_THREADS) {
            const int part = i - 1 + j, from = stretch_start(total, part, stretches);
            const int at = from == stretch_start(total, part + 1, stretches) ? -1 : 2 * (part * R + row) + (from < begin);
            slot[j] = at;
            weight[j] = at < 0 ? make_float2(-INFINITY, 0.f) : *reinterpret_cast<const float2*>(
                                     partial + (size_t)at * S::PART + AE_HEADS * DIM + 2 * head);
            M = fmaxf(M, weight[j].x);
        }
        M = block_max(M, scratch);
        const float sink = a.sinks ? a.sinks[h0 + head] * 1.4426950408889634f : -INFINITY;
        M = fmaxf(M, sink);
        if (M == -INFINITY) M = 0.f;
        float L = 0.f;
        for (int j = tid; j < parts; j += AE_JOIN_THREADS) {
            const float2 ml = weight[j], f = two_factors(ml.x - M, 0.f);
            L = fmaf(ml.y, ex2(ml.x - M), L);
            weight[j] = make_float2(f.x, f.y * ml.y);
        }
        L = block_sum(L, scratch);                 // (with barriers: the weights are there)
        L += ex2(sink - M);
        const float inverse = L == 0.f ? 0.f : 1.f / L;
        constexpr int LANES = DIM / 4, GROUPS = AE_JOIN_THREADS / LANES;
        const int d = tid % LANES * 4;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (d < a.hdv) {
#pragma unroll 4
            for (int j = tid / LANES; j < parts; j += GROUPS) {
                const int at = slot[j];
                if (at < 0) continue;
                const float4 u = *reinterpret_cast<const float4*>(partial + (size_t)at * S::PART + head * DIM + d);
                const float f = weight[j].x, w = weight[j].y * inverse;
                v.x = fmaf(u.x * f, w, v.x);
                v.y = fmaf(u.y * f, w, v.y);
                v.z = fmaf(u.z * f, w, v.z);
                v.w = fmaf(u.w * f, w, v.w);
            }
        }
        sums[tid] = v;
        __syncthreads();
        const float* flat = reinterpret_cast<const float*>(sums);
        T* out = (T*)a.out + ((size_t)b * a.nh + h0 + head) * a.hdv;
        for (int e = tid; e < a.hdv; e += AE_JOIN_THREADS) {
            float o = 0.f;
#pragma unroll
            for (int q = 0; q < GROUPS; ++q) o += flat[q * DIM + e];
            out[e] = from_f32<T>(o);
        }
    }
}

struct Plan {
    int dim, ctas;             // padded head size; CTAs of the launch
    bool split;                // stretches of an equal number of tiles, joined afterwards
    int stretches;             // so many for each row
    int cluster;               // else: CTAs that share a row
    int sms;                   // of the device
};
// Of the current device, asked once for each (148 where there is none to ask, as in a plan made on the host).
int sm_count() {
    static std::atomic<int> counts[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return 148;
    std::atomic<int>& known = counts[dev & 63];          // (of devices from 64 on nothing is kept)
    if (dev < 64 && (n = known.load()) > 0) return n;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n < 1) return 148;
    if (dev < 64) known.store(n);
    return n;
}
Plan plan_of(int B, int nh, int nkv, int hd, int hdv, int max_keys) {
    Plan p;
    const int most = hd > hdv ? hd : hdv;
    p.dim = most <= 64 ? 64 : most <= 128 ? 128 : 256;
    const int R = nkv * ((nh / nkv + AE_HEADS - 1) / AE_HEADS);
    const long long rows = (long long)B * R;
    const long long tiles = ((long long)max_keys + AE_TILE - 1) / AE_TILE + 1;
    p.sms = sm_count();
    const int resident = p.sms * (p.dim == 256 ? Tile<256>::CTAS : p.dim == 128 ? Tile<128>::CTAS : Tile<64>::CTAS);
    // A row is the work of a cluster where that leaves each of its CTAs a few tiles: one launch, and the
    // join goes through shared memory.  As many CTAs as run at a time, 16 only where those are few
    // (one row of 2000 keys: 32 us with one, 14 with four, 11 with eight, 9.7 with 16; 32 rows of 1000: 19, 12, 11, 26).
    // Else stretches, which cost the second launch and about 3 us of finding them (4 rows of 4000 keys: 14 us and
    // 11 with 16 CTAs a row, of 16000: 21 and 23; 256 rows of 1500: 40 and 36 with one CTA a row, of
    // 4000: 62 and 75).
    p.cluster = 1;
    while (p.cluster < 16 && p.cluster < tiles && rows * p.cluster * 2 <= (p.cluster < 8 ? resident : p.sms))
        p.cluster *= 2;
    p.split = tiles > (p.cluster < 8 ? 40 * p.cluster : 240);
    long long stretches = resident / R;                          // all CTAs at a time
    if (stretches > B * tiles) stretches = B * tiles;
    if (stretches > AE_MAX_STRETCHES) stretches = AE_MAX_STRETCHES;
    p.stretches = !p.split ? 0 : stretches < 1 ? 1 : (int)stretches;
    p.ctas = p.split ? p.stretches * R : (int)(rows * p.cluster);
    return p;
}
template <typename T, int DIM, bool EXTRAS>
int launch(const AttendE4& a, const Plan& p, cudaStream_t stream) {
    static std::atomic<unsigned long long> ready{0};             // devices on which the kernel has been set up
    const auto kern = attend_e4m3_kernel<T, DIM, EXTRAS>;
    int dev = 0;
    AGV_CUDA_OK(cudaGetDevice(&dev));
    if (!(ready.load() >> (dev & 63) & 1)) {
        AGV_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Tile<DIM>::SMEM));
        AGV_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        ready.fetch_or(1ull << (dev & 63));
    }
    agv_launch_cluster(kern, p.ctas, AE_THREADS, Tile<DIM>::SMEM, stream, dim3(p.split ? 1 : p.cluster), a);
    AGV_LAUNCH_OK("attend_e4m3_kernel");
    if (p.stretches > 1) {
        // (a CTA a head while that makes no more CTAs than run at a time)
        const int R = a.nkv * a.row_blocks, heads = a.nh / a.nkv < AE_HEADS ? a.nh / a.nkv : AE_HEADS;
        const int y = 4 * p.sms / ((p.stretches - 1) * R);
        agv_launch(join_e4m3_kernel<T, DIM>, dim3(p.stretches - 1, y < 1 ? 1 : y < heads ? y : heads, R), AE_JOIN_THREADS, 0,
                   stream, a, p.stretches);
        AGV_LAUNCH_OK("join_e4m3_kernel");
    }
    return 0;
}
template <typename T, int DIM>
int launch_extras(const AttendE4& a, const Plan& p, cudaStream_t stream) {
    if (a.softcap > 0.f || a.dist_bias) return launch<T, DIM, true>(a, p, stream);
    return launch<T, DIM, false>(a, p, stream);
}
template <typename T>
int launch_dim(const AttendE4& a, const Plan& p, cudaStream_t stream) {
    if (p.dim == 64) return launch_extras<T, 64>(a, p, stream);
    if (p.dim == 128) return launch_extras<T, 128>(a, p, stream);
    return launch_extras<T, 256>(a, p, stream);
}

}  // namespace

// 32-bit values of scratch that agv_attention_decode_e4m3 wants for these sizes.
AGV_API long long agv_attention_decode_e4m3_scratch(int B, int nh, int nkv, int hd, int hdv, int max_keys) {
    AGV_REQUIRE(B >= 0 && nh > 0 && nkv > 0 && nh % nkv == 0,
                "attention_decode_e4m3: bad sizes (%d query heads over %d)", nh, nkv);
    const Plan p = plan_of(B, nh, nkv, hd, hdv, max_keys);
    return p.split ? 4ll * p.stretches + 2ll * p.ctas * (AE_HEADS * p.dim + 2 * AE_HEADS) : 0;
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
    AGV_REQUIRE(page >= 16 && (page & (page - 1)) == 0 && cap > 0 && cap % page == 0 && cap / page <= max_pages,
                "attention_decode_e4m3: bad cache geometry (page %d, cap %d, table of %d)", page, cap, max_pages);
    AGV_REQUIRE(dtype == AGV_F32 || dtype == AGV_BF16, "attention_decode_e4m3: bad dtype");
    AGV_REQUIRE(agv_aligned(k_pool, 16) && agv_aligned(v_pool, 16), "attention_decode_e4m3: unaligned pool");
    AGV_REQUIRE(keep_first >= 0 && softcap >= 0.f && (!dist_bias || n_dist > 0), "attention_decode_e4m3: bad options");
    if (B == 0) return 0;
    const Plan plan = plan_of(B, nh, nkv, hd, hdv, max_keys);
    const long long wanted = agv_attention_decode_e4m3_scratch(B, nh, nkv, hd, hdv, max_keys);
    AGV_REQUIRE(!plan.split || (partial && agv_aligned(partial, 16) && partial_floats >= wanted),
                "attention_decode_e4m3: %lld floats of scratch are too few", partial_floats);
    const size_t esz = dtype == AGV_F32 ? 4 : 2;
    int page_bits = 0;
    while (1 << page_bits < page) ++page_bits;
    const int q_vec = agv_aligned(q, 16) && (size_t)ldq * esz % 16 == 0;
    AttendE4 a{q, ldq, out, (const unsigned char*)k_pool, (const unsigned char*)v_pool, k_scale, v_scale,
               table, slots, positions, B, n_slots, max_pages, n_pages, page, cap, nh, nkv, hd, hdv,
               window, window ? keep_first : 0, scale, softcap, sinks, dist_bias, n_dist, q_vec,
               page_bits, (nh / nkv + AE_HEADS - 1) / AE_HEADS, plan.cluster, plan.split ? partial : nullptr};
    return dtype == AGV_F32 ? launch_dim<float>(a, plan, stream) : launch_dim<__nv_bfloat16>(a, plan, stream);
}

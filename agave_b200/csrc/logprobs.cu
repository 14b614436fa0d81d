// Log-probabilities of given tokens from rows of logits: ln softmax at the token, the row's
// entropy, the token's rank and the greatest logits with their indices.
//
// With a reference c, d = x - c, s = sum e^d and t = sum d e^d: ln p = x_t - c - ln s and H = ln s -
// t / s.  Every thread's reference is the greatest logit it has seen; sums move to another
// reference c' as s' = s e^(c - c'), t' = (t + (c - c') s) e^(c - c').  (x - c comes before the factor
// log2 e of the exponential: logits may be the type's lowest value.)
//
// What bounds it is reading the logits once.  A row is the work of a cluster of 1 to 8 CTAs; a
// thread takes every LP_THREADS-th 16 bytes of its CTA's slice, four of them while the next four are
// under way, and keeps a running maximum, the two sums and the count of logits ahead of the
// token's; the arithmetic goes two values an instruction where there is one for two.
//
// The greatest: a logit and its index are one 64-bit key.  Every thread knows its maximum and in
// which four pieces it stood, that is, a key that its greatest logit reaches.  Of the greatest
// such keys of LP_GROUPS groups of threads the top-th is a bound that at least ``top`` keys of the
// slice reach, and few others do (of 64 groups and top 20 some 4 more).  The pieces of the threads
// that may reach it are read once more (from L2) and what does is ranked; the cluster's first CTA
// merges the slices' lists.
//
// Logits are 32-bit, as the decoder's head makes them, or bfloat16, for callers that hold their own so.
#include "common.cuh"

namespace {

constexpr int LP_MAX_TOP = 32;
constexpr int LP_MAX_CLUSTER = 8;
constexpr int LP_GROUPS = 64;
constexpr int LP_LIST = 2048;             // keys at or above the bound that a CTA can list
constexpr float LOG2E = 1.4426950408889634f;

typedef unsigned long long u64;

// A logit and its index as one unsigned number that grows with the logit and falls with the
// index: equal logits (-0 is 0) go by the lower index.  NaN stands below every number; no key is 0.
__device__ __forceinline__ u64 lp_key(float x, unsigned i) {
    unsigned b = __float_as_uint(x + 0.f);
    b = (int)b < 0 ? ~b : b | 0x80000000u;
    if (x != x) b = 0;
    return (u64)b << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ float lp_value(u64 key) {
    const unsigned b = (unsigned)(key >> 32);
    if (b == 0) return __uint_as_float(0x7fffffffu);
    return __uint_as_float((b & 0x80000000u) ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ u64 greater(u64 a, u64 b) { return a > b ? a : b; }

__device__ __forceinline__ float max_nan(float a, float b) {        // NaN if either is
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// s and t relative to the reference c (-inf: nothing yet).
struct Sums {
    float c, s, t;
    __device__ __forceinline__ void move(float to) {
        // (a reference of -inf has sums of 0, or NaN, which stay that)
        const float d = fmaxf(c - to, -1e4f), f = ex2(d * LOG2E);
        t = f * fmaf(d, s, t);
        s *= f;
        c = to;
    }
};
// Sums of WIDTH neighbouring lanes (a power of two), all relative to their greatest reference, in every one.
template <int WIDTH>
__device__ __forceinline__ void join_lanes(Sums& a) {
    float to = a.c;
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) to = fmaxf(to, __shfl_xor_sync(0xffffffffu, to, o));
    if (to != -INFINITY) a.move(to);               // (else nothing but NaN can be in them)
#pragma unroll
    for (int o = WIDTH / 2; o > 0; o >>= 1) {
        a.s += __shfl_xor_sync(0xffffffffu, a.s, o);
        a.t += __shfl_xor_sync(0xffffffffu, a.t, o);
    }
}

struct Logprobs {
    const void* logits;
    long long ld;
    int V, top, cluster_bits;                  // 2^cluster_bits CTAs a row
    const int* tokens;
    float *logprob, *entropy;
    int* rank;
    int* top_ids;
    float* top_logprobs;
};

// What the CTAs of a cluster hand to its first one.
struct Slice {
    float c, s, t;
    int ahead;
    u64 keys[LP_MAX_TOP];
};

__device__ __forceinline__ unsigned lp_cluster_rank() {
    unsigned r;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void lp_cluster_arrive() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void lp_cluster_wait() {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned in_first_cta(const void* mine) {
    unsigned p;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(p) : "r"((unsigned)__cvta_generic_to_shared(mine)));
    return p;
}
__device__ __forceinline__ void put(unsigned at, float v) {
    asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(v) : "memory");
}
__device__ __forceinline__ void put(unsigned at, int v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
}
__device__ __forceinline__ void put(unsigned at, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(at), "l"(v) : "memory");
}

// 16 bytes of logits as pairs of 32-bit values, and the greatest of them.
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ void values(const uint4& u, float* x) {
        x[0] = __uint_as_float(u.x); x[1] = __uint_as_float(u.y);
        x[2] = __uint_as_float(u.z); x[3] = __uint_as_float(u.w);
    }
    // (the pieces' sums below: what a value under -1e37 adds is 0 where ``tame`` is asked for)
    static __device__ __forceinline__ uint4 tame(const uint4& u) { return u; }
    static constexpr bool TAMES = false;
    // values above, or at or above, the bound
    static __device__ __forceinline__ f32x2 above(const uint4& u, float than, bool or_equal) {
        const float x[4] = {__uint_as_float(u.x), __uint_as_float(u.y), __uint_as_float(u.z), __uint_as_float(u.w)};
        float n[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (or_equal) asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(n[i]) : "f"(x[i]), "f"(than));
            else asm("set.gt.f32.f32 %0, %1, %2;" : "=f"(n[i]) : "f"(x[i]), "f"(than));
        }
        return add2(pack2(n[0], n[1]), pack2(n[2], n[3]));
    }
    static __device__ __forceinline__ float greatest(const uint4& u) {
        return fmaxf(fmaxf(__uint_as_float(u.x), __uint_as_float(u.y)), fmaxf(__uint_as_float(u.z), __uint_as_float(u.w)));
    }
};
template <> struct Piece<__nv_bfloat16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ void values(const uint4& u, float* x) {
        const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static constexpr bool TAMES = true;
    static __device__ __forceinline__ unsigned at_least(unsigned w) {
        unsigned r;
        asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xfcf1fcf1u));       // -1e37 twice
        return r;
    }
    static __device__ __forceinline__ uint4 tame(const uint4& u) {
        return make_uint4(at_least(u.x), at_least(u.y), at_least(u.z), at_least(u.w));
    }
    static __device__ __forceinline__ f32x2 above(const uint4& u, float than, bool or_equal) {
        const __nv_bfloat162 b = __float2bfloat162_rn(than);      // (a logit's own value: exact)
        __nv_bfloat162 n;
        if (or_equal)
            n = __hadd2(__hadd2(__hge2(pair(u.x), b), __hge2(pair(u.y), b)),
                        __hadd2(__hge2(pair(u.z), b), __hge2(pair(u.w), b)));
        else
            n = __hadd2(__hadd2(__hgt2(pair(u.x), b), __hgt2(pair(u.y), b)),
                        __hadd2(__hgt2(pair(u.z), b), __hgt2(pair(u.w), b)));
        return pack2(__low2float(n), __high2float(n));
    }
    static __device__ __forceinline__ __nv_bfloat162 pair(unsigned w) {
        return *reinterpret_cast<const __nv_bfloat162*>(&w);
    }
    static __device__ __forceinline__ float greatest(const uint4& u) {
        const __nv_bfloat162 m = __hmax2(__hmax2(pair(u.x), pair(u.y)), __hmax2(pair(u.z), pair(u.w)));
        return fmaxf(__low2float(m), __high2float(m));
    }
};
__device__ __forceinline__ uint4 piece_at(const void* p) { return __ldg(reinterpret_cast<const uint4*>(p)); }

template <typename T, bool TOP, int LP_THREADS>
__global__ void __launch_bounds__(LP_THREADS, 1024 / LP_THREADS) logprobs_kernel(const Logprobs a) {
    constexpr int LP_WARPS = LP_THREADS / 32, LP_GROUP_LANES = LP_THREADS / LP_GROUPS;
    constexpr int N = Piece<T>::N, BATCH = 4;
    __shared__ Sums wsum[LP_WARPS];
    __shared__ int wahead[LP_WARPS];
    __shared__ Slice slices[LP_MAX_CLUSTER];               // the first CTA's count
    __shared__ u64 group_best[TOP ? LP_GROUPS : 1];
    __shared__ u64 list[TOP ? LP_LIST : 1];
    __shared__ u64 greatest[TOP ? LP_MAX_TOP : 1];         // of the slice, in order
    __shared__ u64 warp_best[TOP ? LP_WARPS : 1];
    __shared__ int n_list;
    __shared__ u64 bound_key;
    const int C = 1 << a.cluster_bits;
    if (C > 1) lp_cluster_arrive();                        // (a CTA's memory is written to once it runs)
    pdl_wait();
    pdl_launch_next();
    const int row = blockIdx.x >> a.cluster_bits, rank = C > 1 ? (int)lp_cluster_rank() : 0;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const T* x = (const T*)a.logits + (long long)row * a.ld;
    // the row as 16-byte pieces behind a head that ends at a 16-byte boundary
    const int head = min(a.V, (int)((16 - (uintptr_t)x % 16) % 16 / sizeof(T)));
    const int pieces = (a.V - head) / N, per = (pieces + C - 1) >> a.cluster_bits;
    const int v0 = min(pieces, rank * per), v1 = min(pieces, v0 + per);
    const T* body = x + head;

    int v = v0 + tid;
    uint4 next[BATCH];
    auto fetch = [&]() {
#pragma unroll
        for (int q = 0; q < BATCH; ++q)
            if (v + q * LP_THREADS < v1) next[q] = piece_at(body + (size_t)(v + q * LP_THREADS) * N);
    };
    fetch();                                               // (before the token's logit is asked for)
    const int tok = a.tokens[row];
    const bool has = tok >= 0 && tok < a.V;
    const float xt = has ? to_f32(x[tok]) : INFINITY;

    Sums sum{-INFINITY, 0.f, 0.f};
    float m = -INFINITY;
    int m_at = -1;                                         // index where the pieces with the maximum begin
    int ahead = 0;
    // the values of n pieces, LP_THREADS apart, that begin at index i
    auto take = [&](const uint4* u, auto n_const, int i) {
        constexpr int n = decltype(n_const)::value;
        float bm = Piece<T>::greatest(u[0]);
#pragma unroll
        for (int q = 1; q < n; ++q) bm = fmaxf(bm, Piece<T>::greatest(u[q]));
        if (bm > m || (bm == m && m_at < 0)) m_at = i;
        if (bm > m) {
            m = bm;
            sum.move(m);
        }
        const float c = sum.c == -INFINITY ? 0.f : sum.c;
        const f32x2 minus_c = pack2(-c, -c), log2e = pack2(LOG2E, LOG2E);
        f32x2 s = pack2(0.f, 0.f), w = pack2(0.f, 0.f);
        auto add = [&](auto tame) {
#pragma unroll
            for (int q = 0; q < n; ++q) {
                float x[N];
                Piece<T>::values(decltype(tame)::value ? Piece<T>::tame(u[q]) : u[q], x);
#pragma unroll
                for (int e = 0; e < N; e += 2) {
                    f32x2 d = add2(pack2(x[e], x[e + 1]), minus_c);
                    float y0, y1;
                    if constexpr (!decltype(tame)::value) {
                        // (at e^-150 a term is 0 and its product with d is, too)
                        unpack2(d, y0, y1);
                        d = pack2(max_nan(y0, -150.f), max_nan(y1, -150.f));
                    }
                    unpack2(mul2(d, log2e), y0, y1);
                    const f32x2 p = pack2(ex2(y0), ex2(y1));
                    s = add2(s, p);
                    w = fma2(p, d, w);
                }
            }
        };
        // Where the reference is no extreme number, bfloat16 values are held above -1e37, two an
        // instruction: d is then finite, and such a value's term 0 as ever.
        if (Piece<T>::TAMES && fabsf(c) < 1e30f) add(std::integral_constant<bool, Piece<T>::TAMES>{});
        else add(std::false_type{});
        float lo, hi;
        unpack2(s, lo, hi);
        sum.s += lo + hi;
        unpack2(w, lo, hi);
        sum.t += lo + hi;
        if (bm >= xt) {
            const int end = i + (n - 1) * LP_THREADS * N + N;
            if (i > tok || end <= tok) {
                f32x2 count = pack2(0.f, 0.f);
                if (i > tok) {
#pragma unroll
                    for (int q = 0; q < n; ++q) count = add2(count, Piece<T>::above(u[q], xt, false));
                } else {
#pragma unroll
                    for (int q = 0; q < n; ++q) count = add2(count, Piece<T>::above(u[q], xt, true));
                }
                unpack2(count, lo, hi);
                ahead += (int)(lo + hi);
            } else {
#pragma unroll
                for (int q = 0; q < n; ++q) {
                    float x[N];
                    Piece<T>::values(u[q], x);
#pragma unroll
                    for (int e = 0; e < N; ++e) ahead += x[e] > xt || (x[e] == xt && i + q * LP_THREADS * N + e < tok);
                }
            }
        }
    };
    while (v < v1) {
        uint4 u[BATCH];
#pragma unroll
        for (int q = 0; q < BATCH; ++q) u[q] = next[q];
        const int i = head + v * N, left = v1 - v;
        v += BATCH * LP_THREADS;
        fetch();
        if (left > (BATCH - 1) * LP_THREADS) {
            take(u, std::integral_constant<int, BATCH>{}, i);
        } else {
#pragma unroll
            for (int q = 0; q < BATCH - 1; ++q)
                if (q * LP_THREADS < left) take(u + q, std::integral_constant<int, 1>{}, i + q * LP_THREADS * N);
        }
    }
    // the head and what is left behind the last piece: a thread of the first CTA each
    const int tail = a.V - head - pieces * N;
    int edge = -1;
    if (rank == 0 && tid < head + tail) edge = tid < head ? tid : a.V - tail + tid - head;
    float xe = 0.f;
    if (edge >= 0) {
        xe = to_f32(x[edge]);
        if (xe > m || (xe == m && m_at < 0)) m_at = edge;
        if (xe > m) {
            m = xe;
            sum.move(m);
        }
        const float d = max_nan(xe - (sum.c == -INFINITY ? 0.f : sum.c), -150.f), p = ex2(d * LOG2E);
        sum.s += p;
        sum.t = fmaf(p, d, sum.t);
        ahead += xe > xt || (xe == xt && edge < tok);
    }
    // ---- sums and counts of the CTA
    join_lanes<32>(sum);
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    if (lane == 0) {
        wsum[warp] = sum;
        wahead[warp] = ahead;
    }
    // The maximum stands at m_at or up to SPAN indices behind it: a key it reaches, and one that
    // nothing of the thread exceeds.
    constexpr unsigned SPAN = (BATCH - 1) * LP_THREADS * N + N - 1;
    const u64 reached = m_at < 0 ? 0 : lp_key(m, m_at + SPAN), most = m_at < 0 ? 0 : lp_key(m, m_at);
    if (TOP) {
        u64 k = reached;
#pragma unroll
        for (int o = 1; o < LP_GROUP_LANES; o <<= 1) k = greater(k, __shfl_xor_sync(0xffffffffu, k, o));
        if (tid % LP_GROUP_LANES == 0) group_best[tid / LP_GROUP_LANES] = k;
        if (tid == 0) {
            n_list = 0;
            bound_key = 0;
        }
        if (tid < LP_MAX_TOP) greatest[tid] = 0;
    }
    __syncthreads();
    if (warp == LP_WARPS - 1) {
        Sums all = wsum[lane & (LP_WARPS - 1)];
        int n = wahead[lane & (LP_WARPS - 1)];
        join_lanes<LP_WARPS>(all);
#pragma unroll
        for (int o = LP_WARPS / 2; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        sum = all;                                         // handed on below
        ahead = n;
    }
    if (TOP) {
        if (tid < LP_GROUPS) {
            const u64 k = group_best[tid];
            int before = 0;
#pragma unroll 8
            for (int j = 0; j < LP_GROUPS; ++j) before += group_best[j] > k;
            if (before == a.top - 1 && k) bound_key = k;
        }
        __syncthreads();
        const u64 bound = bound_key;
        auto note = [&](u64 key) {
            if (key < bound) return;
            const int at = atomicAdd(&n_list, 1);
            if (at < LP_LIST) list[at] = key;
        };
        if (edge >= 0) note(lp_key(xe, edge));
        // the pieces of a thread that may reach the bound, a lane each
        for (unsigned who = __ballot_sync(0xffffffffu, most >= bound); who; who &= who - 1) {
            const int first = v0 + (tid & ~31) + __ffs(who) - 1;
            for (int p = first + lane * LP_THREADS; p < v1; p += 32 * LP_THREADS) {
                float w[N];
                Piece<T>::values(piece_at(body + (size_t)p * N), w);
#pragma unroll
                for (int e = 0; e < N; ++e) note(lp_key(w[e], head + p * N + e));
            }
        }
        __syncthreads();
        const int n = n_list;
        if (n <= LP_LIST) {
            for (int i = tid; i < n; i += LP_THREADS) {
                const u64 key = list[i];
                int before = 0;
#pragma unroll 4
                for (int j = 0; j < n; ++j) before += list[j] > key;
                if (before < a.top) greatest[before] = key;
            }
        } else {
            // more than the list holds: one after the other from the logits
            u64 below = ~0ull;
            for (int q = 0; q < a.top; ++q) {
                u64 mine = edge >= 0 && lp_key(xe, edge) < below ? lp_key(xe, edge) : 0;
                for (int p = v0 + tid; p < v1; p += LP_THREADS) {
                    float w[N];
                    Piece<T>::values(piece_at(body + (size_t)p * N), w);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const u64 key = lp_key(w[e], head + p * N + e);
                        if (key < below) mine = greater(mine, key);
                    }
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) mine = greater(mine, __shfl_xor_sync(0xffffffffu, mine, o));
                if (lane == 0) warp_best[warp] = mine;
                __syncthreads();
                below = warp_best[0];
                for (int w = 1; w < LP_WARPS; ++w) below = greater(below, warp_best[w]);
                if (tid == 0) greatest[q] = below;
                __syncthreads();
            }
        }
        __syncthreads();
    }
    // ---- to the first CTA of the cluster
    if (C > 1) lp_cluster_wait();
    Slice* at = &slices[rank];
    if (tid == LP_THREADS - 1) {
        put(in_first_cta(&at->c), sum.c);
        put(in_first_cta(&at->s), sum.s);
        put(in_first_cta(&at->t), sum.t);
        put(in_first_cta(&at->ahead), ahead);
    }
    if (TOP && tid < a.top) put(in_first_cta(&at->keys[tid]), greatest[tid]);
    if (C > 1) {
        lp_cluster_arrive();
        lp_cluster_wait();
    } else {
        __syncthreads();
    }
    if (rank != 0) return;
    // (every warp for itself: lane r has slice r's)
    Sums all{-INFINITY, 0.f, 0.f};
    int n_ahead = 0;
    if ((lane & (LP_MAX_CLUSTER - 1)) < C) {
        const Slice& from = slices[lane & (LP_MAX_CLUSTER - 1)];
        all = Sums{from.c, from.s, from.t};
        n_ahead = from.ahead;
    }
    join_lanes<LP_MAX_CLUSTER>(all);
#pragma unroll
    for (int o = LP_MAX_CLUSTER / 2; o > 0; o >>= 1) n_ahead += __shfl_xor_sync(0xffffffffu, n_ahead, o);
    const float nan = __uint_as_float(0x7fffffffu);
    const float ls = all.s > 0.f ? logf(all.s) : nan;     // (no softmax: NaN, or nothing but -inf)
    if (tid == 0) {
        a.logprob[row] = has ? xt - all.c - ls : nan;
        a.entropy[row] = ls - all.t / all.s;
        a.rank[row] = has ? n_ahead + 1 : 0;
    }
    if (TOP) {
        // a key's place: its place in its own list and the keys ahead of it in the others
        for (int i = tid; i < C * a.top; i += LP_THREADS) {
            const int mine = i / a.top;
            const u64 key = slices[mine].keys[i % a.top];
            if (key == 0) continue;
            int place = i % a.top;
            for (int r = 0; r < C; ++r) {
                if (r == mine) continue;
                int lo = 0, hi = a.top;                    // keys ahead of it in list r
                while (lo < hi) {
                    const int mid = (lo + hi) / 2;
                    if (slices[r].keys[mid] > key) lo = mid + 1;
                    else hi = mid;
                }
                place += lo;
            }
            if (place < a.top) {
                a.top_ids[(size_t)row * a.top + place] = (int)(0xffffffffu - (unsigned)key);
                a.top_logprobs[(size_t)row * a.top + place] = lp_value(key) - all.c - ls;
            }
        }
    }
}

// CTAs for a row: as many, up to 8, as leave slices of some thousand logits and at most about the 296 CTAs
// of 512 threads that run at a time (64 rows of 262144: 35 us with one CTA a row, 23 with two, 22
// with four, 35 with eight; one row: 27, 18, 13, 11; 64 rows of 32001: 9.2, 8.7, 10.3, 19).
int lp_cluster_bits(int R, int V) {
    int bits = 0;
    while (bits < 3 && (long long)R << (bits + 1) <= 296 && V >> (bits + 1) >= 8000) ++bits;
    return bits;
}

// Threads of a CTA.  An SM takes 1024: 512 a CTA where that holds all CTAs at a time (296), and for long rows; 256 up
// to 592; above that the CTAs come in rounds, and what one does besides reading runs under the others' reads, of
// which rows up to 28000 logits have most with 128 threads, longer ones with 256 (us with 128, 256 and 512
// threads, five alternatives; 32-bit, then bfloat16: 300 rows of 32001 19, 15, 18 and 15, 15, 17; 777 of 9000 14, 16,
// 20 and 14, 16, 19; of 16384 17, 20, 23 and 17, 19, 25; of 24000 23, 24, 28 and 22, 23, 28; of 32001 29, 31, 32 and 26,
// 25, 31; of 48000 39, 41, 38 and 34, 31, 36; 1500 of 16384 30, 31, 40 and 25, 29, 43; of 24000 39, 39, 48 and 32, 35, 47; of
// 32001 50, 47, 53 and 38, 41, 54; of 65000 92, 80, 81 and 58, 58, 70; 600 of 100000 in 32 bits 78, 65, 59).
int lp_threads(long long ctas, int V) {
    return ctas <= 296 || V > 65536 ? 512 : ctas <= 592 || V > 28000 ? 256 : 128;
}

template <typename T, bool TOP, int THREADS>
int lp_launch(const Logprobs& a, int R, cudaStream_t stream) {
    auto kern = logprobs_kernel<T, TOP, THREADS>;
    agv_launch_cluster(kern, dim3((unsigned)R << a.cluster_bits), THREADS, 0, stream,
                       dim3(1u << a.cluster_bits), a);
    AGV_LAUNCH_OK("logprobs_kernel");
    return 0;
}
template <typename T>
int lp_launch(const Logprobs& a, int R, cudaStream_t stream) {
    const int threads = lp_threads((long long)R << a.cluster_bits, a.V);
    if (threads == 128) return a.top ? lp_launch<T, true, 128>(a, R, stream) : lp_launch<T, false, 128>(a, R, stream);
    if (threads == 256) return a.top ? lp_launch<T, true, 256>(a, R, stream) : lp_launch<T, false, 256>(a, R, stream);
    return a.top ? lp_launch<T, true, 512>(a, R, stream) : lp_launch<T, false, 512>(a, R, stream);
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
    Logprobs a{logits, ld, V, top, lp_cluster_bits(R, V), tokens, logprob, entropy, rank, top_ids, top_logprobs};
    return dtype == AGV_F32 ? lp_launch<float>(a, R, stream) : lp_launch<__nv_bfloat16>(a, R, stream);
}

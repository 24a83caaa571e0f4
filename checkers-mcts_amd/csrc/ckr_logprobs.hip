// ckr_logprobs.hip -- log probabilities of given actions, the entropy and the top alternatives of rows of logits, and their gradient.
//
// Row x[0 .. V), temperature 1 / it, allowed set A (the mask's, without logits of -inf):
//     d_j = x_j - max_A x,   S = sum_A exp(it d_j),   log p_j = it d_j - ln S   (-inf outside A)
//     H = -sum_A p_j log p_j = ln S - it (sum_A exp(it d_j) d_j) / S            (two terms >= 0: nothing cancels)
//     gradient for g_k = dL/d log p(a_k) and h = dL/dH:
//     dx_j = it [ sum_k g_k [j = a_k] - p_j sum_k g_k - h p_j (log p_j + H) ]   (0 outside A)
// Sums, statistics and outputs are float32; the gradient is rounded once, to the logits' type.
// An empty A: log p = -inf, H = 0, no alternatives, gradient 0.  NaN or +inf in A: NaN, and no alternatives.
//
// What bounds it: the bytes of the logits.  Forward, 4096 x 32768 bf16: 47 us = 5.7 TB/s (a large copy reaches 4.7-5.4), with 5 alternatives
// 52 us; 8192 x 16384 float32: 95 us = 5.6 TB/s.  Gradient, 4096 x 32768 bf16: 96 us = 5.6 TB/s read and written.  A launch of few or
// short rows is a chain of waits: one position (512) with 8 alternatives 5.3 us, 4096 positions with 5 8.5 us, one row of 131072 with 20
// alternatives 10.0 + 5.8 us.  Six VALU operations an element, one of them the exponential: at 7.5 TB/s they would be the bound.
#include "ckr_host.h"
#include "ckr_device.hip.h"
#include <cmath>

namespace ckr {

constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.44269504088896340736f;

typedef ckr_logprobs_args Args;

constexpr float FLOOR = -1e30f;               // differences below it are that: exp is 0 anyway, and 0 x -inf would be NaN
// 16 bytes of logits that start at any element
template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

template <int MASK> __device__ __forceinline__ bool is_allowed(const Args& A, long long row, int j) {
    if constexpr (MASK == CKR_MASK_BYTES) return static_cast<const uint8_t*>(A.mask)[row * A.mask_stride + j] != 0;
    if constexpr (MASK == CKR_MASK_LEGAL) {
        const uint32_t* m = static_cast<const uint32_t*>(A.mask) + row * A.mask_stride;
        const int x = (j >> 3) & 7, y = j & 7;
        return ((x ^ y) & 1) && ((m[j >> 6] >> (4 * x + (y >> 1))) & 1u);
    }
    return true;
}

// elements j .. j + N - 1 as float32, -inf where they are masked or not below `end`; `raw`: their logits, if all are below it
template <typename T, int MASK>
__device__ __forceinline__ void values(const Args& A, long long row, const T* x, int j, int end, const typename Vec<T>::type raw, float* out) {
    constexpr int N = Vec<T>::N;
    if (j + N <= end) {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = (float)raw[e];
        if constexpr (MASK == CKR_MASK_BYTES) {
            typedef uint8_t bytes __attribute__((ext_vector_type(N), aligned(1)));
            const bytes m = *reinterpret_cast<const bytes*>(static_cast<const uint8_t*>(A.mask) + row * A.mask_stride + j);
#pragma unroll
            for (int e = 0; e < N; ++e) out[e] = m[e] ? out[e] : -__builtin_huge_valf();
        }
        if constexpr (MASK == CKR_MASK_LEGAL) {                                   // j is a multiple of N: one word, four bits of it
            const uint32_t w = static_cast<const uint32_t*>(A.mask)[row * A.mask_stride + (j >> 6)] >> (4 * ((j >> 3) & 7));
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const int y = (j & 7) + e;
                out[e] = ((((j >> 3) ^ y) & 1) && ((w >> (y >> 1)) & 1u)) ? out[e] : -__builtin_huge_valf();
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) out[e] = j + e < end && is_allowed<MASK>(A, row, j + e) ? (float)x[j + e] : -__builtin_huge_valf();
    }
}
template <typename T> __device__ __forceinline__ typename Vec<T>::type load_vec(const T* x, int j, int end) {
    typename Vec<T>::type v = {};
    if (j + Vec<T>::N <= end) v = *reinterpret_cast<const typename Vec<T>::type*>(x + j);
    return v;
}

__device__ __forceinline__ long long action_at(const Args& A, long long i) {
    return A.action_bytes == 8 ? static_cast<const long long*>(A.actions)[i] : (long long)static_cast<const int*>(A.actions)[i];
}

__device__ __forceinline__ float wave_max_f32(float v) {
    v = fmaxf(v, bfly_f32<1>(v)); v = fmaxf(v, bfly_f32<2>(v)); v = fmaxf(v, bfly_f32<4>(v)); v = fmaxf(v, bfly_f32<8>(v));
    const int i = __float_as_int(v);
    return fmaxf(fmaxf(__int_as_float(__builtin_amdgcn_readlane(i, 0)), __int_as_float(__builtin_amdgcn_readlane(i, 16))),
                 fmaxf(__int_as_float(__builtin_amdgcn_readlane(i, 32)), __int_as_float(__builtin_amdgcn_readlane(i, 48))));
}
__device__ __forceinline__ float wave_sum_f32(float v) {
    v += bfly_f32<1>(v); v += bfly_f32<2>(v); v += bfly_f32<4>(v); v += bfly_f32<8>(v);
    const int i = __float_as_int(v);
    return (__int_as_float(__builtin_amdgcn_readlane(i, 0)) + __int_as_float(__builtin_amdgcn_readlane(i, 16))) +
           (__int_as_float(__builtin_amdgcn_readlane(i, 32)) + __int_as_float(__builtin_amdgcn_readlane(i, 48)));
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }          // 1 ulp; denormal results are 0

// ---- a wavefront's k best (value, index) so far: lane r holds the one of rank r; larger value first, then lower index --------------
struct TopList {
    float v = -__builtin_huge_valf();
    int i = -1;
    // what a candidate has to come before: the entry of rank k - 1
    float tau = -__builtin_huge_valf();
    int tau_i = -1;

    __device__ __forceinline__ void insert(float x, int j, int k) {               // x, j: the same in all lanes
        const int pos = __popcll(__ballot(v > x || (v == x && i < j)));
        const float vs = __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x138, 0xF, 0xF, false));      // wave_shr:1
        const int is = __builtin_amdgcn_update_dpp(0, i, 0x138, 0xF, 0xF, false);
        const int lane = lane_id();
        v = lane < pos ? v : lane == pos ? x : vs;
        i = lane < pos ? i : lane == pos ? j : is;
        const float kv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k - 1));
        if (kv > -__builtin_huge_valf()) { tau = kv; tau_i = __builtin_amdgcn_readlane(i, k - 1); }
    }
    // every lane's candidate (x, j); -inf and NaN are none
    __device__ __forceinline__ void offer(float x, int j, int k) {
        if (!__any(x >= tau)) return;
        unsigned long long m = __ballot(x > tau || (x == tau && j < tau_i));
        while (m) {
            const int l = first_lane(m);
            m &= m - 1;
            const float xl = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(x), l));
            const int jl = __builtin_amdgcn_readlane(j, l);
            if (xl > tau || (xl == tau && jl < tau_i)) insert(xl, jl, k);
        }
    }
    // The list of the candidates (x, j) of lanes 0 .. n - 1, one each, where it is empty so far; the other lanes have none (-inf).  Few ranks: the
    // largest is taken out k times, 20 instructions that wait for each other.  Many: a lane's rank is the number of lanes before it,
    // counted over n broadcasts that do not wait, and the values go to the lanes of their ranks, 350 instructions for 64.
    __device__ __forceinline__ void build(float x, int j, int k, int n) {
        if (8 * k < n) {
            for (int r = 0; r < k; ++r) {
                const float best = wave_max_f32(x);
                if (!(best > -__builtin_huge_valf())) return;
                unsigned long long m = __ballot(x == best);
                int l = first_lane(m), jl = __builtin_amdgcn_readlane(j, l);
                for (m &= m - 1; m; m &= m - 1) {                                 // several: the lowest index
                    const int l2 = first_lane(m), j2 = __builtin_amdgcn_readlane(j, l2);
                    if (j2 < jl) { l = l2; jl = j2; }
                }
                v = lane_id() == r ? best : v;
                i = lane_id() == r ? jl : i;
                x = lane_id() == l ? -__builtin_huge_valf() : x;
                if (r == k - 1) { tau = best; tau_i = jl; }
            }
            return;
        }
        const bool have = x > -__builtin_huge_valf();
        const int bits = __float_as_int(x + 0.0f);                                // (-0 as 0)
        const unsigned hi = bits < 0 ? ~(unsigned)bits : (unsigned)bits | 0x80000000u, lo = ~(unsigned)j;
        const unsigned long long key = (unsigned long long)hi << 32 | lo, mine = __ballot(have);
        int rank = 0;
        for (int l = 0; l < n; ++l) {
            const unsigned long long other = (unsigned long long)(unsigned)__builtin_amdgcn_readlane((int)hi, l) << 32 | (unsigned)__builtin_amdgcn_readlane((int)lo, l);
            rank += other > key ? 1 : 0;
        }
        const unsigned long long below = (1ull << lane_id()) - 1ull;
        if (!have) rank = __popcll(mine) + __popcll(~mine & below);               // none: behind the others, in their own order
        v = __int_as_float(__builtin_amdgcn_ds_permute(rank << 2, __float_as_int(x)));
        i = __builtin_amdgcn_ds_permute(rank << 2, have ? j : -1);
        const float kv = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), k - 1));
        if (kv > -__builtin_huge_valf()) { tau = kv; tau_i = __builtin_amdgcn_readlane(i, k - 1); }
    }
    // ... of M candidates a lane, in the order of their indexes j(0) < j(1) < ...
    template <int M, typename J> __device__ __forceinline__ void build_of(const float (&x)[M], J j, int k, int n) {
        float best = -__builtin_huge_valf();
        int at = 0;
#pragma unroll
        for (int e = 0; e < M; ++e) best = fmaxf(best, x[e]);
#pragma unroll
        for (int e = M - 1; e >= 0; --e) at = x[e] == best ? e : at;
        build(best, j(at), k, n);
#pragma unroll
        for (int e = 0; e < M; ++e) offer(at == e ? -__builtin_huge_valf() : x[e], j(e), k);
    }
};

// ---- forward: what a wavefront knows of its part of a row --------------------------------------------------------------------------
// m: the maximum, S = sum exp(it (x - m)), D = sum exp(it (x - m)) (x - m), per lane until they are joined.  One pass: where a tile raises a
// lane's maximum, its sums are carried over to the new one, S' = f S, D' = f (D + (m - m') S) with f = exp(it (m - m')).
struct Sums { float m, S, D; };

__device__ __forceinline__ void carry(Sums& s, float m, float c) {
    const float d = fmaxf(s.m - m, FLOOR), f = exp2_fast(d * c);
    s.D = f * __builtin_fmaf(d, s.S, s.D);
    s.S *= f;
    s.m = m;
}

// A lane's best vector so far (its largest element, and the vector's number in the part) and the largest element of its second best: nothing
// in a tile waits for other lanes.  Lane l of every wavefront has the vectors l, l + 64, ..., so that lanes can be joined over wavefronts.
struct Best {
    float v = -__builtin_huge_valf(), second = -__builtin_huge_valf();
    int i = -1;
    __device__ __forceinline__ void take(float x, int j) {                        // j rises
        second = __builtin_amdgcn_fmed3f(x, v, second);
        i = x > v ? j : i;
        v = fmaxf(v, x);
    }
    __device__ __forceinline__ void join(float v2, float second2, int i2) {
        second = fmaxf(fminf(v, v2), fmaxf(second, second2));
        i = v2 > v || (v2 == v && (unsigned)i2 < (unsigned)i) ? i2 : i;           // (-1, no vector, is the largest)
        v = fmaxf(v, v2);
    }
};

constexpr int GROUP = 4;                      // wavefronts of a workgroup
constexpr int IN_TILE = 4;                    // vectors a lane holds at a time
struct Shared {                               // what the wavefronts of a workgroup that share a part tell the first one
    float vm[GROUP][IN_TILE][64];             // the vectors' largest elements, if each had one tile only
    float v[GROUP][64], second[GROUP][64];
    int i[GROUP][64];
    float4 sums[GROUP];
};

// The alternatives of a part.  The k best elements are in the k best vectors: any other vector's best element has k elements before it, of a
// larger value or, as vectors are numbered like their elements, of the same value and a lower index.  The k best vectors are among the
// lanes' best ones and the others of those lanes whose second best reaches the list (k^2 / 128 lanes on average; one that only equals
// the list's last value lies 64 vectors behind the lane's best, if that equals it too), which the wavefront reads again unless
// all are at hand (vm: `rows` times 64 of them, by `stride` wavefronts in turn).  At the end lane r reads the vector of rank r for its elements.
template <typename T, int MASK>
__device__ __forceinline__ void alternatives(const Args& A, long long row, int begin, int end, const Best& mine, const float (*vm)[IN_TILE][64], int stride, TopList& list) {
    constexpr int N = Vec<T>::N;
    const T* x = static_cast<const T*>(A.logits) + row * A.row_stride;
    const int lane = lane_id(), k = A.top, vectors = (end - begin + N - 1) / N, rows = (vectors + 63) / 64;
    TopList vecs;
    vecs.build(mine.v, mine.i, k, 64);
    if (rows <= IN_TILE * stride) {
        for (int r = 0; r < rows; ++r)
            vecs.offer(r * 64 + lane == mine.i ? -__builtin_huge_valf() : vm[r % stride][r / stride][lane], r * 64 + lane, k);
    } else for (unsigned long long more = __ballot(mine.second > vecs.tau || (mine.second == vecs.tau && mine.second > -__builtin_huge_valf() &&
                                                                       !(mine.v == vecs.tau && mine.i + 64 >= vecs.tau_i))); more; more &= more - 1) {
        const int l = first_lane(more), known = __builtin_amdgcn_readlane(mine.i, l);
        for (int i0 = l; i0 < vectors; i0 += 64 * 64) {
            const int i = i0 + lane * 64, j = begin + i * N;
            const bool have = i < vectors && i != known;
            float e[N], m = -__builtin_huge_valf();
            values<T, MASK>(A, row, x, j, have ? end : 0, load_vec<T>(x, j, have ? end : 0), e);
#pragma unroll
            for (int q = 0; q < N; ++q) m = fmaxf(m, e[q]);
            vecs.offer(m, i, k);
        }
    }
    float e[N];
    const bool have = lane < k && vecs.i >= 0;
    const int j = have ? begin + vecs.i * N : 0;                                  // (a lane without a vector: no element is below 0)
    values<T, MASK>(A, row, x, j, have ? end : 0, load_vec<T>(x, j, have ? end : 0), e);
    list.build_of(e, [&](int i) { return j + i; }, k, k);
}

// A wavefront's share of elements begin .. end - 1: the vectors of every `stride`-th 64, from the `first` 64 on.
template <typename T, int MASK, bool TOP>
__device__ __forceinline__ void scan(const Args& A, long long row, int begin, int end, int first, int stride, Sums& s, Best& best, float (*vm)[64]) {
    constexpr int N = Vec<T>::N, U = IN_TILE, SPAN = 64 * N;
    const T* x = static_cast<const T*>(A.logits) + row * A.row_stride;
    const int lane = lane_id(), step = stride * SPAN;
    const float c = A.inv_temperature * LOG2E;
    s.m = LOWEST; s.S = 0.0f; s.D = 0.0f;
    typename Vec<T>::type raw[U];
    int j0 = begin + first * SPAN;
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_vec<T>(x, j0 + u * step + lane * N, end);
    for (; j0 < end; j0 += U * step) {
        float v[U * N], m[U], tm = -__builtin_huge_valf();
        const int left = (end - j0 + step - 1) / step;                            // vectors of this tile that hold anything
#pragma unroll
        for (int u = 0; u < U; ++u) {
            m[u] = -__builtin_huge_valf();
            if (u < left) {
                values<T, MASK>(A, row, x, j0 + u * step + lane * N, end, raw[u], v + u * N);
#pragma unroll
                for (int e = 0; e < N; ++e) m[u] = fmaxf(m[u], v[u * N + e]);
            }
            tm = fmaxf(tm, m[u]);
        }
        if (end - j0 > U * step)                                                  // the next tile is on its way while this one is summed
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u] = load_vec<T>(x, j0 + (U + u) * step + lane * N, end);
        if (__any(tm > s.m)) carry(s, fmaxf(tm, s.m), c);
        float S = 0.0f, D = 0.0f;                                                 // of the tile first: fewer roundings of the long sum
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (u < left) {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float d = v[u * N + e] - s.m, p = exp2_fast(d * c);
                    S += p;
                    D = __builtin_fmaf(p, fmaxf(d, FLOOR), D);
                }
            }
        s.S += S; s.D += D;
        if constexpr (TOP) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                best.take(m[u], (j0 + u * step - begin) / N + lane);
                vm[u][lane] = m[u];
            }
        }
    }
}

__device__ __forceinline__ void join_sums(Sums& s, Sums t, float c) {
    const float m = fmaxf(s.m, t.m);
    carry(s, m, c);
    carry(t, m, c);
    s.S += t.S; s.D += t.D;
}
// the lanes' sums over one maximum
__device__ __forceinline__ void join_lanes(Sums& s, float c) {
    carry(s, wave_max_f32(s.m), c);
    s.S = wave_sum_f32(s.S); s.D = wave_sum_f32(s.D);
}

// (x - max) it from halves: x - max itself may not fit (lowest against largest values) where the product does
__device__ __forceinline__ float scaled(float x, float m, float it) { return (0.5f * x - 0.5f * m) * (2.0f * it); }

template <typename T, int MASK, bool TOP>
__device__ __forceinline__ void write_row(const Args& A, long long row, const Sums& s, const TopList& list) {
    const int lane = lane_id();
    const float it = A.inv_temperature;
    const bool empty = s.S == 0.0f, bad = !(s.S < __builtin_huge_valf());
    const float lnS = empty ? 0.0f : logf(s.S), H = empty ? 0.0f : lnS - it * s.D / s.S;
    if (lane == 0) {
        A.entropy[row] = H;
        if (A.stats) *reinterpret_cast<float4*>(A.stats + 4 * row) = make_float4(s.m, s.S, H, 0.0f);
    }
    if (lane < A.n_given) {
        const long long a = action_at(A, row * A.n_given + lane);
        const T* x = static_cast<const T*>(A.logits) + row * A.row_stride;
        float lp;
        if (a < 0) lp = 0.0f;
        else if (a >= A.v || bad) lp = __builtin_nanf("");
        else lp = !empty && is_allowed<MASK>(A, row, (int)a) ? scaled((float)x[a], s.m, it) - lnS : -__builtin_huge_valf();
        A.logp[row * A.n_given + lane] = lp;
    }
    if (TOP && lane < A.top) {
        A.top_action[row * A.top + lane] = bad ? -1 : list.i;
        A.top_logp[row * A.top + lane] = bad ? __builtin_nanf("") : list.i < 0 ? -__builtin_huge_valf() : scaled(list.v, s.m, it) - lnS;
    }
}

// SHARE false: a wavefront per row.  SHARE true: a workgroup per part of a row, `parts` of `length` elements (whole 64 vectors) each; its first
// wavefront joins the four and writes the row, or, if there are more parts, their sums and list to the scratch memory for
// k_logprobs_join: float4 [rows][parts], values and indexes [rows][top][parts].
template <typename T, int MASK, bool TOP, bool SHARE>
__global__ __launch_bounds__(256, 4) void k_logprobs(const Args A, long long row0, int parts, int length) {
    __shared__ Shared sh;
    const int wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), lane = lane_id();
    const float c = A.inv_temperature * LOG2E;
    if constexpr (!SHARE) {
        const long long row = row0 + (long long)blockIdx.x * GROUP + wave;
        if (row >= A.n) return;
        Sums s;
        Best best;
        TopList list;
        scan<T, MASK, TOP>(A, row, 0, (int)A.v, 0, 1, s, best, sh.vm[wave]);
        if constexpr (TOP) alternatives<T, MASK>(A, row, 0, (int)A.v, best, sh.vm + wave, 1, list);
        join_lanes(s, c);
        write_row<T, MASK, TOP>(A, row, s, list);
    } else {
        const long long row = row0 + (parts == 1 ? blockIdx.x : blockIdx.y);
        const int part = parts == 1 ? 0 : (int)blockIdx.x, begin = part * length, end = (int)A.v - begin < length ? (int)A.v : begin + length;
        Sums s;
        Best best;
        scan<T, MASK, TOP>(A, row, begin, end, wave, GROUP, s, best, sh.vm[wave]);
        join_lanes(s, c);
        if (wave && lane == 0) sh.sums[wave] = make_float4(s.m, s.S, s.D, 0.0f);
        if (TOP && wave) { sh.v[wave][lane] = best.v; sh.second[wave][lane] = best.second; sh.i[wave][lane] = best.i; }
        __syncthreads();
        if (wave) return;
        TopList list;
        for (int w = 1; w < GROUP; ++w) {
            join_sums(s, {sh.sums[w].x, sh.sums[w].y, sh.sums[w].z}, c);
            if constexpr (TOP) best.join(sh.v[w][lane], sh.second[w][lane], sh.i[w][lane]);
        }
        if constexpr (TOP) alternatives<T, MASK>(A, row, begin, end, best, sh.vm, GROUP, list);
        if (parts == 1) { write_row<T, MASK, TOP>(A, row, s, list); return; }
        const long long at = row * parts + part;
        float4* sums = static_cast<float4*>(A.scratch);
        if (lane == 0) sums[at] = make_float4(s.m, s.S, s.D, 0.0f);
        if (TOP && lane < A.top) {
            float* tv = reinterpret_cast<float*>(sums + A.n * parts);
            int* ti = reinterpret_cast<int*>(tv + A.n * parts * A.top);
            const long long slot = (row * A.top + lane) * parts + part;
            tv[slot] = list.v;
            ti[slot] = list.i;
        }
    }
}

template <typename T, int MASK, bool TOP>
__global__ __launch_bounds__(64) void k_logprobs_join(const Args A, int parts) {
    const int lane = lane_id();
    const float c = A.inv_temperature * LOG2E;
    const float4* sums = static_cast<const float4*>(A.scratch);
    const float* tv = reinterpret_cast<const float*>(sums + A.n * parts);
    const int* ti = reinterpret_cast<const int*>(tv + A.n * parts * A.top);
    for (long long row = blockIdx.x; row < A.n; row += gridDim.x) {
        Sums s = {LOWEST, 0.0f, 0.0f};
        for (int p = lane; p < parts; p += 64) {
            const float4 o = sums[row * parts + p];
            Sums t = {o.x, o.y, o.z};
            join_sums(s, t, c);
        }
        join_lanes(s, c);
        TopList list;
        if constexpr (TOP) {                                                      // rank by rank: where no part's next one can enter, none behind it can
            const int n = parts * A.top;
            const float* v = tv + row * n;
            const int* i = ti + row * n;
            float x = lane < n ? v[lane] : -__builtin_huge_valf();
            int j = lane < n ? i[lane] : -1, idle = 0;
            for (int q = 0; q < n && idle < parts; q += 64) {
                const int next = q + 64 + lane;
                const float x1 = next < n ? v[next] : -__builtin_huge_valf();
                const int j1 = next < n ? i[next] : -1;
                if (q == 0) list.build(x, j, A.top, n < 64 ? n : 64);
                else {
                    const bool any = __any(x >= list.tau && x > -__builtin_huge_valf());
                    idle = any ? 0 : idle + 64;
                    if (any) list.offer(x, j, A.top);
                }
                x = x1; j = j1;
            }
        }
        write_row<T, MASK, TOP>(A, row, s, list);
    }
}

// ---- backward: a wavefront has BWD_PER_LANE elements a lane of one row ----------------------------------------------------------------
constexpr int BWD_PER_LANE = 16, BWD_TILE = 64 * BWD_PER_LANE;
// A gradient of this many bytes is stored past the caches (STREAMS), which keep no more than its end for whoever reads it.  Forward, backward and
// a reduction of the gradient, bf16 rows of 32768, with the caches and past them: 128 MiB 148 and 167 us, 144 MiB 173 and 183 us, 160 MiB 206
// and 198 us, 206 MiB 257 and 247 us, 256 MiB 320 and 303 us; with the product that a linear layer's gradient is in place of the reduction:
// 160 MiB 175 and 166 us, 206 MiB 221 and 207 us, 256 MiB 260 and 243 us.
constexpr long long STREAMED = 160ll << 20;

template <typename T, int MASK, bool STREAMS>
__global__ __launch_bounds__(256) void k_logprobs_bwd(const Args A) {
    constexpr int N = Vec<T>::N, U = BWD_PER_LANE / N;
    const int lane = lane_id(), wave = __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), V = (int)A.v;
    const int j0 = ((int)blockIdx.x * 4 + wave) * BWD_TILE;
    if (j0 >= V) return;
    const float it = A.inv_temperature, c = it * LOG2E;
    for (long long row = blockIdx.y; row < A.n; row += gridDim.y) {
        const T* x = static_cast<const T*>(A.logits) + row * A.row_stride;
        T* out = static_cast<T*>(A.grad) + row * A.grad_stride;
        float v[BWD_PER_LANE], given[BWD_PER_LANE];
        typename Vec<T>::type raw[U];
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u] = load_vec<T>(x, j0 + (u * 64 + lane) * N, V);
#pragma unroll
        for (int u = 0; u < U; ++u) values<T, MASK>(A, row, x, j0 + (u * 64 + lane) * N, V, raw[u], v + u * N);
        const float4 st = *reinterpret_cast<const float4*>(A.stats + 4 * row);
        const float m = st.x, rS = 1.0f / st.y, lnS = logf(st.y), H = st.z, h = A.g_entropy ? A.g_entropy[row] : 0.0f;
        // lane k has the k-th given action; those of this tile go to the lanes that hold their elements, in the order of k
        long long a = -1;
        float g = 0.0f;
        if (lane < A.n_given) {
            a = action_at(A, row * A.n_given + lane);
            g = a < 0 ? 0.0f : a >= V ? __builtin_nanf("") : A.g_logp[row * A.n_given + lane];
        }
        const float G = wave_sum_f32(g);
#pragma unroll
        for (int e = 0; e < BWD_PER_LANE; ++e) given[e] = 0.0f;
        for (unsigned long long mine = __ballot(a >= j0 && a < (long long)j0 + BWD_TILE && a < V); mine; mine &= mine - 1) {
            const int l = first_lane(mine);
            const int off = __builtin_amdgcn_readlane((int)a, l) - j0 - lane * N;
            const float gl = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(g), l));
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int e = 0; e < N; ++e) given[u * N + e] += off == u * 64 * N + e ? gl : 0.0f;
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            typename Vec<T>::type r;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float x1 = v[u * N + e], d = x1 - m, p = exp2_fast(d * c) * rS;
                const float lp = fmaxf(__builtin_fmaf(d, it, -lnS), -200.0f);         // p is 0 below -104: any finite number does
                const float q = p * __builtin_fmaf(h, lp + H, G);
                r[e] = (T)(x1 == -__builtin_huge_valf() ? 0.0f : it * (given[u * N + e] - q));
            }
            const int j = j0 + (u * 64 + lane) * N;
            if (j + N <= V) {
                if constexpr (STREAMS) __builtin_nontemporal_store(r, reinterpret_cast<typename Vec<T>::type*>(out + j));
                else *reinterpret_cast<typename Vec<T>::type*>(out + j) = r;
            } else
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (j + e < V) out[j + e] = r[e];
        }
    }
}

// How a row is shared.  A row of one tile is a wavefront's.  A longer one is a workgroup's if its wavefronts get two tiles each: one of four
// makes the row's list while other workgroups read (4096 x 32768 bf16: 47 us, with 5 alternatives 52 us, against 51 and 56 us of a wavefront per
// row; 8192 x 16384 float32: 95 and 101 us against 101 and 106; but 16384 x 4096 bf16, half a tile each: 32 and 49 us against 25 and 36), or if
// there are too few rows to fill the card otherwise.  Rows fewer than about 1024 are cut into parts, which a second launch joins; where each has
// to make a list, a part has a tile for each wavefront at least (one row of 131072 bf16 with 20 alternatives: 9.8 + 5.8 us for 16 parts, 8.8 +
// 7.7 us for 64; 517 rows of 50001 fp16 under a mask with 10: 26.3 + 4.3 us at 1024 workgroups, 30.2 at 500, 27.8 + 5.1 us at 2560).
static bool split(const Args& A, int& parts, int& length) {
    constexpr long long GROUPS = 1024;
    const int span = 64 * (A.dtype == CKR_F32 ? Vec<float>::N : Vec<_Float16>::N);                // 64 vectors
    const long long n = A.n > 0 ? A.n : 1, rows = (A.v + span - 1) / span;
    parts = 1;
    length = (int)A.v;
    if (rows <= IN_TILE || (n >= 2 * GROUPS && rows < 2 * IN_TILE * GROUP)) return false;
    const long long want = n >= GROUPS ? 1 : (GROUPS + n / 2) / n, least = A.top ? GROUP * IN_TILE : GROUP;
    const long long each = rows <= want * least ? least : (rows + want - 1) / want;
    parts = (int)((rows + each - 1) / each);
    length = parts == 1 ? (int)A.v : (int)each * span;
    return true;
}

template <typename T, int MASK, bool TOP> int forward_tmk(const Args& A, hipStream_t s) {
    int parts, length;
    const bool share = split(A, parts, length);
    const long long most = 1 << 23, each = share ? most : most * GROUP;           // rows of a launch: a grid has less than 2^24 workgroups of this size
    for (long long row0 = 0; row0 < A.n; row0 += each) {
        const long long rows = A.n - row0 < each ? A.n - row0 : each;
        if (!share)
            hipLaunchKernelGGL((k_logprobs<T, MASK, TOP, false>), dim3((unsigned)((rows + GROUP - 1) / GROUP)), dim3(64 * GROUP), 0, s, A, row0, parts, length);
        else if constexpr (MASK != CKR_MASK_LEGAL)                                // (512 actions are one tile)
            hipLaunchKernelGGL((k_logprobs<T, MASK, TOP, true>), parts == 1 ? dim3((unsigned)rows) : dim3((unsigned)parts, (unsigned)rows), dim3(64 * GROUP), 0, s,
                               A, row0, parts, length);
        CKR_HIP(hipGetLastError());
    }
    if (parts > 1) {                                                              // (fewer than 1024 rows)
        hipLaunchKernelGGL((k_logprobs_join<T, MASK, TOP>), dim3((unsigned)A.n), dim3(64), 0, s, A, parts);
        CKR_HIP(hipGetLastError());
    }
    return CKR_OK;
}
template <typename T> int forward_t(const Args& A, hipStream_t s) {
    if (A.mask_kind == CKR_MASK_NONE) return A.top ? forward_tmk<T, CKR_MASK_NONE, true>(A, s) : forward_tmk<T, CKR_MASK_NONE, false>(A, s);
    if (A.mask_kind == CKR_MASK_BYTES) return A.top ? forward_tmk<T, CKR_MASK_BYTES, true>(A, s) : forward_tmk<T, CKR_MASK_BYTES, false>(A, s);
    return A.top ? forward_tmk<T, CKR_MASK_LEGAL, true>(A, s) : forward_tmk<T, CKR_MASK_LEGAL, false>(A, s);
}
template <typename T, int MASK> void backward_tm(const Args& A, hipStream_t s) {
    const dim3 grid((unsigned)((A.v + 4 * BWD_TILE - 1) / (4 * BWD_TILE)), (unsigned)(A.n < 65535 ? A.n : 65535)), block(256);
    if (A.n * A.v * (long long)sizeof(T) >= STREAMED) hipLaunchKernelGGL((k_logprobs_bwd<T, MASK, true>), grid, block, 0, s, A);
    else hipLaunchKernelGGL((k_logprobs_bwd<T, MASK, false>), grid, block, 0, s, A);
}
template <typename T> int backward_t(const Args& A, hipStream_t s) {
    if (A.mask_kind == CKR_MASK_NONE) backward_tm<T, CKR_MASK_NONE>(A, s);
    else if (A.mask_kind == CKR_MASK_BYTES) backward_tm<T, CKR_MASK_BYTES>(A, s);
    else backward_tm<T, CKR_MASK_LEGAL>(A, s);
    CKR_HIP(hipGetLastError());
    return CKR_OK;
}

static int check_args(const Args* a, const char* who) {
    if (!a) return fail(CKR_ERR_INVALID, "%s: null argument", who);
    if (a->n < 0 || a->n > (1ll << 32) || a->v < 1 || a->v > (1ll << 30)) return fail(CKR_ERR_INVALID, "%s: n in 0 .. 2^32, v in 1 .. 2^30", who);
    if (a->dtype < CKR_F32 || a->dtype > CKR_F16) return fail(CKR_ERR_INVALID, "%s: unknown type %d", who, (int)a->dtype);
    if (a->mask_kind < CKR_MASK_NONE || a->mask_kind > CKR_MASK_LEGAL || (a->n && a->mask_kind != CKR_MASK_NONE && !a->mask) || a->mask_stride < 0)
        return fail(CKR_ERR_INVALID, "%s: bad mask", who);
    if (a->mask_kind == CKR_MASK_LEGAL && a->v != 512) return fail(CKR_ERR_INVALID, "%s: legal-move words belong to 512 actions", who);
    if (a->n_given < 0 || a->n_given > CKR_LOGPROBS_MOST || a->top < 0 || a->top > CKR_LOGPROBS_MOST)
        return fail(CKR_ERR_INVALID, "%s: at most %d given actions and alternatives a row", who, CKR_LOGPROBS_MOST);
    if (a->n && a->n_given && (!a->actions || (a->action_bytes != 4 && a->action_bytes != 8))) return fail(CKR_ERR_INVALID, "%s: bad actions", who);
    if (!(a->inv_temperature >= 9.9e-7f && a->inv_temperature <= 1.01e6f)) return fail(CKR_ERR_INVALID, "%s: the temperature must be from 1e-6 to 1e6", who);
    if ((reinterpret_cast<uintptr_t>(a->stats) | reinterpret_cast<uintptr_t>(a->scratch)) & 15) return fail(CKR_ERR_INVALID, "%s: stats and scratch begin at multiples of 16 bytes", who);
    if (a->row_stride < 0 || (a->n && !a->logits)) return fail(CKR_ERR_INVALID, "%s: bad logits", who);
    return CKR_OK;
}

}  // namespace ckr

extern "C" {

int64_t ckr_logprobs_scratch(const ckr_logprobs_args* a) {
    if (int rc = ckr::check_args(a, "ckr_logprobs_scratch")) return rc;
    int parts, length;
    ckr::split(*a, parts, length);
    return parts == 1 ? 0 : a->n * parts * (16 + 8 * (int64_t)a->top);
}

int ckr_logprobs_forward(const ckr_logprobs_args* a, void* stream) {
    if (int rc = ckr::check_args(a, "ckr_logprobs_forward")) return rc;
    if (a->n && (!a->entropy || (a->n_given && !a->logp) || (a->top && (!a->top_action || !a->top_logp))))
        return ckr::fail(CKR_ERR_INVALID, "ckr_logprobs_forward: null output");
    const int64_t scratch = ckr_logprobs_scratch(a);
    if (scratch > 0 && (!a->scratch || a->scratch_bytes < scratch)) return ckr::fail(CKR_ERR_INVALID, "ckr_logprobs_forward: %lld bytes of scratch memory needed", (long long)scratch);
    if (int rc = ckr::require_device()) return rc;
    if (!a->n) return CKR_OK;
    if (a->dtype == CKR_F32) return ckr::forward_t<float>(*a, (hipStream_t)stream);
    if (a->dtype == CKR_BF16) return ckr::forward_t<__bf16>(*a, (hipStream_t)stream);
    return ckr::forward_t<_Float16>(*a, (hipStream_t)stream);
}

int ckr_logprobs_backward(const ckr_logprobs_args* a, void* stream) {
    if (int rc = ckr::check_args(a, "ckr_logprobs_backward")) return rc;
    if (a->n && (!a->stats || !a->grad || a->grad_stride < a->v || (a->n_given && !a->g_logp)))
        return ckr::fail(CKR_ERR_INVALID, "ckr_logprobs_backward: bad argument");
    if (int rc = ckr::require_device()) return rc;
    if (!a->n) return CKR_OK;
    if (a->dtype == CKR_F32) return ckr::backward_t<float>(*a, (hipStream_t)stream);
    if (a->dtype == CKR_BF16) return ckr::backward_t<__bf16>(*a, (hipStream_t)stream);
    return ckr::backward_t<_Float16>(*a, (hipStream_t)stream);
}

}  // extern "C"

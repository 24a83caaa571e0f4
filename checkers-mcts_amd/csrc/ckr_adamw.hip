// ckr_adamw.hip -- one AdamW update of many tensors, with the moments in 32 or in 8 bits.
//
//     norm = sqrt(sum g^2) over all tensors (float64),  c = min(1, max_norm / (norm + 1e-6)),  g := c g        (where clipping is on)
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   t = t + 1
//     w = w (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
// Parameters of 16 bits have a float32 master copy w; the parameter is its rounding.
//
// 8-bit moments: blocks of 128 elements, each with a scale byte b (2^(b - 127): the power of two of the block's largest value, or the
// next one; 255: the block holds a value that is not finite and reads back as NaN).  A code is a small float below that scale,
//     m: sign, 4 exponent bits, 3 mantissa bits   value (1 + M / 8) 2^(E - 15) 2^(b - 127)
//     v: 5 exponent bits, 3 mantissa bits         value (1 + M / 8) 2^(E - 31) 2^(b - 127)
// code 0 is 0.  A value of v below the smallest code is raised to it: as 0 it would divide by eps alone.
// The rounding to 3 mantissa bits is stochastic.  With 1 - b2 = 0.001, v moves by a thousandth of itself a step and a code is 1/8 to
// 1/16 wide: to the nearest code it would not move at all, whatever the gradients.  16 dither bits per value, from Philox4x32-10 with
// key = seed and counter = (group of 8 elements, step): whoever knows the seed can repeat a run, and graphs replay with fresh bits.
// The moments themselves are computed in float64 on this path, so that which code a value falls to is decided by the formula and not
// by the order of float32 operations (a v_fma_f64 issues at the rate of a v_fma_f32 here).
// The price of so few bits is noise: v fluctuates by about 20 % around its average, its root, which divides, by 10 %.
//
// What bounds it: memory.  134 M bf16 parameters with master copies and 8-bit moments: 440 us = 4.9 TB/s (a large copy reaches 4.7-5.4); with 32-bit
// moments 9 M float16 in 170 tensors: 51 us = 4.9 TB/s; the 48 tensors of the policy / value network (1.3 M float32): 11 us, of which a
// launch, the table and the tickets are 5.  In 8 bits the 90 VALU operations an element (20 of them Philox, shared by 8 elements) would
// allow 7 TB/s.
#include "ckr_host.h"
#include "ckr_device.hip.h"
#include <cmath>
#include <cstring>

namespace ckr {

constexpr int CHUNK = 2048;                   // elements of one tensor that a workgroup takes at a time: 256 threads x 8
constexpr int BLOCKS = 2048;                  // at most (8 workgroups of 256 threads on each of 256 CUs)
constexpr int M_TOP = 15, V_TOP = 31;

// The tensors of one launch travel in the kernel's arguments (4 KB): the step takes 128 of them, the norm, which reads gradients only, 240.
constexpr int STEP_TENSORS = 128, NORM_TENSORS = 240;
template <int CAP, bool STEP> struct TensorTable {
    static constexpr int MOST = CAP;
    const void* g[CAP];
    void* p[STEP ? CAP : 1];
    unsigned block[STEP ? CAP : 1];           // of the states: the tensor's first block of 128
    unsigned first[CAP + 1];                  // chunks before tensor i
    uint16_t tail[CAP];                       // elements of its last chunk
    int tensors;
    __device__ __forceinline__ long long size(int i) const { return (long long)(first[i + 1] - first[i] - 1) * CHUNK + tail[i]; }
};
typedef TensorTable<STEP_TENSORS, true> StepTable;
typedef TensorTable<NORM_TENSORS, false> NormTable;

struct Hyper {
    float* master; void* m; void* v; uint8_t* m_scale; uint8_t* v_scale;
    int* step; unsigned* ticket;
    const float* d_lr; const double* norm;    // norm[0], the factor c norm[1]
    double lr, beta1, beta2, ln_beta1, ln_beta2, weight_decay;
    unsigned long long seed;
    float eps;
};

// The tensor that chunk c belongs to, from one load of the whole table: kernel arguments lie in host memory, and each step of a bisection
// would wait for them anew.
template <typename Table> __device__ __forceinline__ int tensor_of(const Table& T, unsigned c) {
    int n = 0;
#pragma unroll
    for (int q = 0; q < Table::MOST; q += 64) {
        const int i = q + lane_id();
        n += __popcll(__ballot(i < T.tensors && T.first[min(i, T.tensors)] <= c));
    }
    return __builtin_amdgcn_readfirstlane(n - 1);
}

// True in the workgroup that arrives last of `total` (numbered `number`).  All threads call it; what a workgroup did before is done, and what
// other workgroups are to read of it has been stored with device-scope atomics (no cache is written back for it).  One counter for
// all of them would be their queue: 690 arrivals took 8 us.  32 counters, a cache line each, and one for their last ones.  All are 0 again afterwards.
__device__ __forceinline__ bool arrives_last(unsigned* tickets, unsigned number, unsigned total) {
    __shared__ unsigned last;
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    if (!threadIdx.x) {
        const unsigned line = number & 31u, of_line = (total - line + 31u) / 32u, lines = total < 32u ? total : 32u;
        last = 0u;
        if (__hip_atomic_fetch_add(tickets + 32 * (1 + line), 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == of_line - 1u) {
            __hip_atomic_store(tickets + 32 * (1 + line), 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            if (__hip_atomic_fetch_add(tickets, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == lines - 1u) {
                __hip_atomic_store(tickets, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                last = 1u;
            }
        }
    }
    __syncthreads();
    return last != 0u;
}

// ---- the 8-bit formats, on the high word of a double: 11 exponent bits, the first 20 bits of the mantissa ---------------------------
__device__ __forceinline__ unsigned high_word(double x) { return (unsigned)__double2hiint(x) & 0x7FFFFFFFu; }

// The scale byte of a block whose largest high word is h: one power above it (room = 1), so that a dithered rounding upwards stays in range;
// from already rounded values (room = 0), the power they need, so that what codes hold is written back as it is.
__device__ __forceinline__ int scale_byte(unsigned h, int room = 1) {
    const int b = (int)(h >> 20) - 1023 + room + 127;
    return b > 254 ? 255 : b < 1 ? 1 : b;
}
template <int TOP> __device__ __forceinline__ int encode(unsigned h, int scale, unsigned dither17) {      // magnitude only, <= 0: below the smallest code
    return (int)((h + dither17) >> 17) - ((scale - 127 + 1023 - TOP) << 3);
}
__device__ __forceinline__ unsigned encode_m(double x, int scale, unsigned dither17) {
    const int c = encode<M_TOP>(high_word(x), scale, dither17);
    return c <= 0 ? 0u : (unsigned)c | (__double2hiint(x) < 0 ? 128u : 0u);
}
__device__ __forceinline__ unsigned encode_v(double x, int scale, unsigned dither17) {
    const unsigned h = high_word(x);
    const int c = encode<V_TOP>(h, scale, dither17);
    return h == 0u ? 0u : c < 1 ? 1u : (unsigned)c;
}
template <int TOP> __device__ __forceinline__ double decode(unsigned c, int scale) {
    const int h = ((int)c + ((scale - 127 + 1023 - TOP) << 3)) << 17;
    const double x = __hiloint2double(c ? h : 0, 0);
    return scale == 255 ? (double)__builtin_nanf("") : x;
}
__device__ __forceinline__ double decode_m(unsigned c, int scale) {
    const double x = decode<M_TOP>(c & 127u, scale);
    return c & 128u ? -x : x;
}
__device__ __forceinline__ double decode_v(unsigned c, int scale) { return decode<V_TOP>(c, scale); }

__device__ __forceinline__ unsigned row16_max(unsigned v) {                       // over the 16 lanes (of 8 elements) of a block of 128
    v = max(v, (unsigned)bfly_i32<1>((int)v)); v = max(v, (unsigned)bfly_i32<2>((int)v));
    v = max(v, (unsigned)bfly_i32<4>((int)v)); v = max(v, (unsigned)bfly_i32<8>((int)v));
    return v;
}

// ---- 8 consecutive elements of a thread, in 16-byte accesses that start at any element -------------------------------------------------
template <typename T> struct Eight { typedef T type __attribute__((ext_vector_type(8), aligned(sizeof(T)))); };
template <bool WHOLE, typename T> __device__ __forceinline__ void load8(const T* p, long long left, float* out) {       // left <= 0: none of them, zeros
    if (WHOLE || left >= 8) {
        const typename Eight<T>::type v = *reinterpret_cast<const typename Eight<T>::type*>(p);
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = (float)v[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) out[j] = j < left ? (float)p[j] : 0.0f;
    }
}
template <bool WHOLE, typename T> __device__ __forceinline__ void store8(T* p, long long left, const float* x) {
    if (WHOLE || left >= 8) {
        typename Eight<T>::type v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = (T)x[j];
        *reinterpret_cast<typename Eight<T>::type*>(p) = v;
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < left) p[j] = (T)x[j];
    }
}

// chunks [c, end) of this workgroup: an even share, in one piece, so that a tensor is looked up once
__device__ __forceinline__ unsigned share(unsigned chunks, unsigned b) { return (unsigned)((unsigned long long)chunks * b / gridDim.x); }

// ---- the update: a thread has 8 consecutive elements, 16 lanes a block of 128 --------------------------------------------------------
struct Factors { double c; float decay, rate, rs; int t; };      // of the gradient; 1 - lr wd, lr / (1 - b1^t), 1 / sqrt(1 - b2^t) of the weight

// elements e0 .. e0 + 7 of a tensor of n, states at off + e0.  WHOLE: the chunk has all its elements; otherwise every access asks whether it has
// (the question keeps the loads of a thread from being under way together).
template <typename T, int BITS, bool WHOLE>
__device__ __forceinline__ void update(const Hyper& H, const Factors& F, T* p, const T* g, long long e0, long long n, long long off) {
    const long long left = n - e0, s0 = off + e0;
    const bool in = WHOLE || e0 < (n + 127) / 128 * 128;                          // of the states: whole blocks of 128
    float w[8], gr[8], mf[8], vf[8];
    load8<WHOLE>(g + e0, left, gr);
    if constexpr (sizeof(T) == 4) load8<WHOLE>(p + e0, left, w);
    else load8<WHOLE>(H.master + s0, in ? 8 : 0, w);
    if constexpr (BITS == 32) {
        float* const m = static_cast<float*>(H.m) + s0;
        float* const v = static_cast<float*>(H.v) + s0;
        const float b1 = (float)H.beta1, b2 = (float)H.beta2, a1 = (float)(1.0 - H.beta1), a2 = (float)(1.0 - H.beta2), cf = (float)F.c;
        load8<WHOLE>(m, in ? 8 : 0, mf);
        load8<WHOLE>(v, in ? 8 : 0, vf);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float x = gr[j] * cf;
            mf[j] = b1 * mf[j] + a1 * x;
            vf[j] = b2 * vf[j] + a2 * x * x;
        }
        store8<WHOLE>(m, in ? 8 : 0, mf);
        store8<WHOLE>(v, in ? 8 : 0, vf);
    } else {
        uint2* const m = reinterpret_cast<uint2*>(static_cast<uint8_t*>(H.m) + s0);
        uint2* const v = reinterpret_cast<uint2*>(static_cast<uint8_t*>(H.v) + s0);
        uint2 mc = make_uint2(0, 0), vc = make_uint2(0, 0);
        int ms = 1, vs = 1;
        if (in) { mc = *m; vc = *v; ms = H.m_scale[s0 / 128]; vs = H.v_scale[s0 / 128]; }
        double md[8], vd[8];
        unsigned hm = 0, hv = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const double x = (double)gr[j] * F.c;
            md[j] = H.beta1 * decode_m(((j < 4 ? mc.x : mc.y) >> (8 * (j & 3))) & 255u, ms) + (1.0 - H.beta1) * x;
            vd[j] = H.beta2 * decode_v(((j < 4 ? vc.x : vc.y) >> (8 * (j & 3))) & 255u, vs) + (1.0 - H.beta2) * x * x;
            hm = max(hm, high_word(md[j])); hv = max(hv, high_word(vd[j]));
            mf[j] = (float)md[j]; vf[j] = (float)vd[j];
        }
        const int ms1 = scale_byte(row16_max(hm)), vs1 = scale_byte(row16_max(hv));
        const unsigned long long grp = (unsigned long long)s0 / 8;
        const u32x4 r = philox((unsigned)H.seed, (unsigned)(H.seed >> 32), (unsigned)grp, (unsigned)(grp >> 32), (unsigned)F.t, 0u);
        const unsigned rw[4] = {r.x, r.y, r.z, r.w};
        unsigned mo[2] = {0, 0}, vo[2] = {0, 0};
#pragma unroll
        for (int j = 0; j < 8; ++j) {                                             // 16 of 32 random bits for v, the others for m: 2 r + 1 of 2^17
            const unsigned lo = rw[j >> 1] & 0xFFFFu, hi = rw[j >> 1] >> 16;
            mo[j >> 2] |= encode_m(md[j], ms1, 2u * (j & 1 ? lo : hi) + 1u) << (8 * (j & 3));
            vo[j >> 2] |= encode_v(vd[j], vs1, 2u * (j & 1 ? hi : lo) + 1u) << (8 * (j & 3));
        }
        if (in) {
            *m = make_uint2(mo[0], mo[1]);
            *v = make_uint2(vo[0], vo[1]);
            if ((threadIdx.x & 15) == 0) { H.m_scale[s0 / 128] = (uint8_t)ms1; H.v_scale[s0 / 128] = (uint8_t)vs1; }
        }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = w[j] * F.decay - F.rate * (mf[j] / (sqrtf(vf[j]) * F.rs + H.eps));
    if constexpr (sizeof(T) != 4) store8<WHOLE>(H.master + s0, left < 8 ? left : 8, w);
    store8<WHOLE>(p + e0, left, w);
}

template <typename T, int BITS>
__global__ __launch_bounds__(256) void k_adamw(const StepTable tab, const Hyper H) {
    const double lr = H.d_lr ? (double)*H.d_lr : H.lr;
    Factors F;
    F.c = H.norm ? H.norm[1] : 1.0;
    F.decay = (float)(1.0 - lr * H.weight_decay);
    const unsigned chunks = tab.first[tab.tensors], end = share(chunks, blockIdx.x + 1);
    unsigned ch = share(chunks, blockIdx.x);
    for (int i = tensor_of(tab, ch); ch < end; ++i) {                             // (tensors without a gradient have no chunks)
        const unsigned begin = tab.first[i], after = tab.first[i + 1], stop = min(end, after);
        if (ch >= stop) continue;
        F.t = H.step[i] + 1;
        F.rate = (float)(lr / -expm1(F.t * H.ln_beta1));
        F.rs = (float)(1.0 / sqrt(-expm1(F.t * H.ln_beta2)));
        T* const p = static_cast<T*>(tab.p[i]);
        const T* const g = static_cast<const T*>(tab.g[i]);
        const long long n = tab.size(i), off = (long long)tab.block[i] * 128;
        for (; ch < stop; ++ch) {
            const long long e0 = (long long)(ch - begin) * CHUNK + threadIdx.x * 8;
            if (ch + 1 < after || tab.tail[i] == CHUNK) update<T, BITS, true>(H, F, p, g, e0, n, off);
            else update<T, BITS, false>(H, F, p, g, e0, n, off);
        }
    }
    // The workgroup that ends last advances the step counters: by then every other one has read them.
    if (!arrives_last(H.ticket, blockIdx.x, gridDim.x)) return;
    for (int i = threadIdx.x; i < tab.tensors; i += 256)
        if (tab.g[i]) H.step[i] += 1;
}

// ---- the global norm: every workgroup's sum of squares in parts[base + blockIdx], the last of all `total` workgroups adds them in order --
__device__ __forceinline__ double workgroup_sum(double s, double* red) {          // 256 threads, in a fixed order; red: 4 doubles of LDS
    s = wave_sum_f64(s);
    if (lane_id() == 0) red[threadIdx.x >> 6] = s;
    __syncthreads();
    return (red[0] + red[1]) + (red[2] + red[3]);
}

template <typename T>
__global__ __launch_bounds__(256) void k_grad_norm(const NormTable tab, double max_norm, double* __restrict__ parts, int base, int total,
                                                   unsigned* __restrict__ ticket, double* __restrict__ out) {
    __shared__ double red[4];
    double s = 0.0;
    const unsigned chunks = tab.first[tab.tensors], end = share(chunks, blockIdx.x + 1);
    unsigned ch = share(chunks, blockIdx.x);
    for (int i = tensor_of(tab, ch); ch < end; ++i) {
        const unsigned stop = min(end, tab.first[i + 1]);
        if (ch >= stop) continue;
        const T* const g = static_cast<const T*>(tab.g[i]) + threadIdx.x * 8;
        const long long n = tab.size(i) - threadIdx.x * 8;
        const unsigned begin = tab.first[i], full = tab.first[i + 1] - (tab.tail[i] == CHUNK ? 0u : 1u);
        while (ch < stop) {                                                       // four chunks' loads at a time
            const long long e0 = (long long)(ch - begin) * CHUNK;
            float x[4][8];
            const unsigned take = ch + 4 <= min(stop, full) ? 4u : 1u;
            if (take == 4u)
#pragma unroll
                for (int q = 0; q < 4; ++q) load8<true>(g + e0 + q * CHUNK, 8, x[q]);
            else {
                load8<false>(g + e0, n - e0, x[0]);
#pragma unroll
                for (int q = 1; q < 4; ++q)
#pragma unroll
                    for (int j = 0; j < 8; ++j) x[q][j] = 0.0f;
            }
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int j = 0; j < 8; ++j) s = __builtin_fma((double)x[q][j], (double)x[q][j], s);
            ch += take;
        }
        ch = stop;
    }
    s = workgroup_sum(s, red);
    if (!threadIdx.x) __hip_atomic_store(parts + base + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (!arrives_last(ticket, (unsigned)base + blockIdx.x, (unsigned)total)) return;
    s = 0.0;
    for (int b = threadIdx.x; b < total; b += 256) s += __hip_atomic_load(parts + b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = workgroup_sum(s, red);
    if (threadIdx.x) return;
    const double norm = sqrt(s), c = max_norm / (norm + 1e-6);
    out[0] = norm;
    out[1] = c >= 1.0 ? 1.0 : c;                                                  // NaN stays NaN
}

// ---- reading and writing 8-bit moments (n a multiple of 128) -------------------------------------------------------------------------
// A lane has four elements at a time, so that a wavefront stores whole lines: 134 M in 215-235 us = 5.7-6.2 TB/s written and read, 280 us with
// eight (half a line a store).
__global__ __launch_bounds__(256) void k_moments_read(const uint8_t* __restrict__ m, const uint8_t* __restrict__ v, const uint8_t* __restrict__ m_scale,
                                                      const uint8_t* __restrict__ v_scale, long long n, float* __restrict__ m_out, float* __restrict__ v_out) {
    typedef float four __attribute__((ext_vector_type(4), aligned(4)));
    for (long long i0 = (long long)blockIdx.x * 2048 + threadIdx.x * 4; i0 < n; i0 += (long long)gridDim.x * 2048)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const long long i = i0 + q * 1024;
            if (i >= n) break;
            const unsigned mc = *reinterpret_cast<const unsigned*>(m + i), vc = *reinterpret_cast<const unsigned*>(v + i);
            const int ms = m_scale[i / 128], vs = v_scale[i / 128];
            four mo, vo;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                mo[j] = (float)decode_m((mc >> (8 * j)) & 255u, ms);
                vo[j] = (float)decode_v((vc >> (8 * j)) & 255u, vs);
            }
            *reinterpret_cast<four*>(m_out + i) = mo;
            *reinterpret_cast<four*>(v_out + i) = vo;
        }
}
__global__ __launch_bounds__(256) void k_moments_write(const float* __restrict__ m_in, const float* __restrict__ v_in, long long n, uint8_t* __restrict__ m,
                                                       uint8_t* __restrict__ v, uint8_t* __restrict__ m_scale, uint8_t* __restrict__ v_scale) {
    // whole blocks of 128 are whole rows of 16 lanes: the lanes of a row take part in its maximum together
    for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 8; i < n; i += (long long)gridDim.x * 2048) {
        unsigned hm = 0, hv = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) { hm = max(hm, high_word((double)m_in[i + j])); hv = max(hv, high_word((double)v_in[i + j])); }
        const int ms = scale_byte(row16_max(hm) + 0x10000u, 0), vs = scale_byte(row16_max(hv) + 0x10000u, 0);
#pragma unroll
        for (int j = 0; j < 8; ++j) {                                             // to nearest: half a step is 2^16 of 2^17
            m[i + j] = (uint8_t)encode_m((double)m_in[i + j], ms, 0x10000u);
            v[i + j] = (uint8_t)encode_v((double)v_in[i + j], vs, 0x10000u);
        }
        if ((threadIdx.x & 15) == 0) { m_scale[i / 128] = (uint8_t)ms; v_scale[i / 128] = (uint8_t)vs; }
    }
}

// tensors [k, end) of the call, as many of them as the table takes
template <int CAP, bool STEP>
static void fill_table(TensorTable<CAP, STEP>& T, int end, int k, const int64_t* sizes, const int64_t* offsets, void* const* params, const void* const* grads) {
    T.tensors = end - k < CAP ? end - k : CAP;
    unsigned chunks = 0;
    for (int i = 0; i < T.tensors; ++i) {
        T.g[i] = grads[k + i];
        if (STEP) {
            T.p[i] = params[k + i];
            T.block[i] = (unsigned)(offsets[k + i] / 128);
        }
        T.first[i] = chunks;
        T.tail[i] = (uint16_t)((sizes[k + i] - 1) % CHUNK + 1);
        chunks += T.g[i] ? (unsigned)((sizes[k + i] + CHUNK - 1) / CHUNK) : 0u;
    }
    T.first[T.tensors] = chunks;
}
template <typename Table> static unsigned grid_of(const Table& T, unsigned each) {
    const unsigned c = (T.first[T.tensors] + each - 1) / each;
    return c < 1u ? 1u : c < (unsigned)BLOCKS ? c : (unsigned)BLOCKS;
}

static int check_tensors(const char* who, int count, const int64_t* sizes, const void* const* grads, int dtype) {
    if (count <= 0 || !sizes || !grads) return fail(CKR_ERR_INVALID, "%s: no tensors", who);
    if (dtype < CKR_F32 || dtype > CKR_F16) return fail(CKR_ERR_INVALID, "%s: unknown type %d", who, dtype);
    for (int i = 0; i < count; ++i)
        if (sizes[i] < 1 || sizes[i] > (1ll << 36)) return fail(CKR_ERR_INVALID, "%s: tensor %d has %lld elements: 1 .. 2^36", who, i, (long long)sizes[i]);
    return CKR_OK;
}

}  // namespace ckr

extern "C" {

int ckr_adamw_step(const ckr_adamw_args* a, void* stream) {
    using namespace ckr;
    if (!a) return fail(CKR_ERR_INVALID, "ckr_adamw_step: null argument");
    if (int rc = check_tensors("ckr_adamw_step", a->count, a->sizes, a->grads, a->dtype)) return rc;
    if (!a->offsets || !a->params || !a->m || !a->v || !a->d_step || !a->d_ticket) return fail(CKR_ERR_INVALID, "ckr_adamw_step: null pointer");
    if (a->state_bits != 32 && a->state_bits != 8) return fail(CKR_ERR_INVALID, "ckr_adamw_step: states have 32 or 8 bits");
    if (a->state_bits == 8 && (!a->m_scale || !a->v_scale)) return fail(CKR_ERR_INVALID, "ckr_adamw_step: 8-bit states need their scales");
    if (a->dtype != CKR_F32 && !a->master) return fail(CKR_ERR_INVALID, "ckr_adamw_step: parameters of 16 bits need a master copy");
    if (!(a->beta1 >= 0.0 && a->beta1 < 1.0 && a->beta2 >= 0.0 && a->beta2 < 1.0) || !(a->eps > 0.0f)) return fail(CKR_ERR_INVALID, "ckr_adamw_step: betas in [0, 1), eps > 0");
    for (int i = 0; i < a->count; ++i) {
        if (a->grads[i] && !a->params[i]) return fail(CKR_ERR_INVALID, "ckr_adamw_step: tensor %d has a gradient and no parameter", i);
        if (a->offsets[i] < 0 || a->offsets[i] % 128 || a->offsets[i] >> 38) return fail(CKR_ERR_INVALID, "ckr_adamw_step: offsets are multiples of 128 below 2^38");
    }
    if (int rc = require_device()) return rc;
    hipStream_t s = (hipStream_t)stream;
    for (int k = 0; k < a->count; k += STEP_TENSORS) {
        StepTable T;
        fill_table(T, a->count, k, a->sizes, a->offsets, a->params, a->grads);
        if (!T.first[T.tensors]) continue;
        const Hyper H = {a->master, a->m, a->v, a->m_scale, a->v_scale, a->d_step + k, a->d_ticket, a->d_lr, a->d_norm, a->lr, a->beta1, a->beta2,
                         std::log(a->beta1), std::log(a->beta2), a->weight_decay, (unsigned long long)a->seed, a->eps};
        static_assert(sizeof(T) + sizeof(H) <= 4096, "kernel arguments");
        const dim3 grid(grid_of(T, 1)), block(256);
#define CKR_ADAMW(TYPE)                                                                                       \
        do {                                                                                                  \
            if (a->state_bits == 32) hipLaunchKernelGGL((k_adamw<TYPE, 32>), grid, block, 0, s, T, H);         \
            else hipLaunchKernelGGL((k_adamw<TYPE, 8>), grid, block, 0, s, T, H);                              \
        } while (0)
        if (a->dtype == CKR_F32) CKR_ADAMW(float);
        else if (a->dtype == CKR_BF16) CKR_ADAMW(__bf16);
        else CKR_ADAMW(_Float16);
#undef CKR_ADAMW
        CKR_HIP(hipGetLastError());
    }
    return CKR_OK;
}

int ckr_grad_norm(int32_t count, const int64_t* sizes, const void* const* grads, const int32_t* dtypes, double max_norm, double* d_parts, int64_t parts,
                  uint32_t* d_ticket, double* d_out, void* stream) {
    using namespace ckr;
    if (int rc = check_tensors("ckr_grad_norm", count, sizes, grads, CKR_F32)) return rc;
    if (!dtypes || !d_parts || !d_ticket || !d_out || !(max_norm > 0.0)) return fail(CKR_ERR_INVALID, "ckr_grad_norm: bad argument");
    // launches: runs of tensors of one type, at most NORM_TENSORS each
    int64_t total = 0;
    for (int pass = 0; pass < 2; ++pass) {
        int64_t base = 0;
        for (int k = 0; k < count;) {
            int end = k;
            while (end < count && end - k < NORM_TENSORS && dtypes[end] == dtypes[k]) ++end;
            if (dtypes[k] < CKR_F32 || dtypes[k] > CKR_F16) return fail(CKR_ERR_INVALID, "ckr_grad_norm: unknown type %d", (int)dtypes[k]);
            NormTable T;
            fill_table(T, end, k, sizes, nullptr, nullptr, grads);
            const unsigned grid = grid_of(T, 4);
            if (pass) {
                hipStream_t s = (hipStream_t)stream;
                if (dtypes[k] == CKR_F32) hipLaunchKernelGGL((k_grad_norm<float>), dim3(grid), dim3(256), 0, s, T, max_norm, d_parts, (int)base, (int)total, d_ticket, d_out);
                else if (dtypes[k] == CKR_BF16) hipLaunchKernelGGL((k_grad_norm<__bf16>), dim3(grid), dim3(256), 0, s, T, max_norm, d_parts, (int)base, (int)total, d_ticket, d_out);
                else hipLaunchKernelGGL((k_grad_norm<_Float16>), dim3(grid), dim3(256), 0, s, T, max_norm, d_parts, (int)base, (int)total, d_ticket, d_out);
                CKR_HIP(hipGetLastError());
            }
            base += grid;
            k = end;
        }
        if (!pass) {
            total = base;
            if (total > parts) return fail(CKR_ERR_INVALID, "ckr_grad_norm: %lld partial sums, room for %lld", (long long)total, (long long)parts);
            if (int rc = require_device()) return rc;
        }
    }
    return CKR_OK;
}

int ckr_adamw_read_moments(const uint8_t* m, const uint8_t* v, const uint8_t* m_scale, const uint8_t* v_scale, int64_t n, float* m_out, float* v_out, void* stream) {
    using namespace ckr;
    if (!m || !v || !m_scale || !v_scale || !m_out || !v_out || n <= 0 || n % 128) return fail(CKR_ERR_INVALID, "ckr_adamw_read_moments: bad argument");
    if (int rc = require_device()) return rc;
    const long long blocks = (n + 2047) / 2048;
    hipLaunchKernelGGL(k_moments_read, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, (hipStream_t)stream, m, v, m_scale, v_scale, (long long)n, m_out, v_out);
    CKR_HIP(hipGetLastError());
    return CKR_OK;
}

int ckr_adamw_write_moments(const float* m_in, const float* v_in, int64_t n, uint8_t* m, uint8_t* v, uint8_t* m_scale, uint8_t* v_scale, void* stream) {
    using namespace ckr;
    if (!m || !v || !m_scale || !v_scale || !m_in || !v_in || n <= 0 || n % 128) return fail(CKR_ERR_INVALID, "ckr_adamw_write_moments: bad argument");
    if (int rc = require_device()) return rc;
    const long long blocks = (n + 2047) / 2048;
    hipLaunchKernelGGL(k_moments_write, dim3((unsigned)(blocks < 65536 ? blocks : 65536)), dim3(256), 0, (hipStream_t)stream, m_in, v_in, (long long)n, m, v, m_scale, v_scale);
    CKR_HIP(hipGetLastError());
    return CKR_OK;
}

}  // extern "C"

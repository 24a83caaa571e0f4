// ckr_logprobs.hip -- log probabilities of given actions, the entropy and the top alternatives of rows of logits, and their gradient.
//
// Row x[0 .. V), temperature 1 / it, allowed set A (the mask's, without logits of -inf):
//     d_j = x_j - max_A x,   S = sum_A exp(it d_j),   log p_j = it d_j - ln S   (-inf outside A)
//     H = -sum_A p_j log p_j = ln S - it (sum_A exp(it d_j) d_j) / S            (two terms >= 0: nothing cancels)
//     gradient for g_k = dL/d log p(a_k) and h = dL/dH:
//     dx_j = it [ sum_k g_k [j = a_k] - p_j sum_k g_k - h p_j (log p_j + H) ]   (0 outside A)
// Sums, statistics and outputs are float32; the gradient is rounded once, to the logits' type.
// An empty A: log p = -inf, H = 0, no alternatives, gradient 0.  NaN or +inf in A: NaN, and no alternatives.
#include "ckr_host.h"
#include "ckr_device.hip.h"
#include <cmath>

namespace ckr {

constexpr float LOWEST = -3.402823466e38f, LOG2E = 1.44269504088896340736f;

typedef ckr_logprobs_args Args;

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }

template <int MASK> __device__ __forceinline__ bool is_allowed(const Args& A, long long row, int j) {
    if constexpr (MASK == CKR_MASK_BYTES) return static_cast<const uint8_t*>(A.mask)[row * A.mask_stride + j] != 0;
    if constexpr (MASK == CKR_MASK_LEGAL) {
        const uint32_t* m = static_cast<const uint32_t*>(A.mask) + row * A.mask_stride;
        const int x = (j >> 3) & 7, y = j & 7;
        return ((x ^ y) & 1) && ((m[j >> 6] >> (4 * x + (y >> 1))) & 1u);
    }
    return true;
}

__device__ __forceinline__ long long action_at(const Args& A, long long i) {
    return A.action_bytes == 8 ? static_cast<const long long*>(A.actions)[i] : (long long)static_cast<const int*>(A.actions)[i];
}

__device__ __forceinline__ float wave_max_f32(float v) {
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ float wave_sum_f32(float v) {
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// One wavefront per row: the maximum, then the sums, then every alternative by a pass of its own (the largest element behind the
// last one in the order "larger value, lower index").
template <typename T, int MASK>
__global__ __launch_bounds__(256) void k_logprobs(const Args A) {
    const int lane = lane_id(), V = (int)A.v;
  for (long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); row < A.n; row += 4ll * gridDim.x) {
    const T* x = static_cast<const T*>(A.logits) + row * A.row_stride;
    const float it = A.inv_temperature;
    float m = LOWEST;
    for (int j = lane; j < V; j += 64)
        if (is_allowed<MASK>(A, row, j)) m = fmaxf(m, to_f32(x[j]));
    m = wave_max_f32(m);
    float S = 0.0f, D = 0.0f;
    for (int j = lane; j < V; j += 64)
        if (is_allowed<MASK>(A, row, j)) {
            const float d = to_f32(x[j]) - m, e = exp2f(d * (it * LOG2E));
            S += e;
            D += e > 0.0f ? e * d : 0.0f;
        }
    S = wave_sum_f32(S); D = wave_sum_f32(D);
    const bool empty = S == 0.0f, bad = !(S < __builtin_huge_valf());
    const float lnS = empty ? 0.0f : logf(S), H = empty ? 0.0f : lnS - it * D / S;
    if (lane == 0) {
        A.entropy[row] = H;
        if (A.stats) { float* st = A.stats + 4 * row; st[0] = m; st[1] = S; st[2] = H; st[3] = 0.0f; }
    }
    for (int k = lane; k < A.n_given; k += 64) {
        const long long a = action_at(A, row * A.n_given + k);
        float lp;
        if (a < 0) lp = 0.0f;
        else if (a >= V || bad) lp = __builtin_nanf("");
        else lp = !empty && is_allowed<MASK>(A, row, (int)a) ? (to_f32(x[a]) - m) * it - lnS : -__builtin_huge_valf();
        A.logp[row * A.n_given + k] = lp;
    }
    float last = __builtin_huge_valf();
    int last_j = -1;
    for (int k = 0; k < A.top; ++k) {
        float best = -__builtin_huge_valf();
        int best_j = -1;
        if (!bad)
            for (int j = lane; j < V; j += 64)
                if (is_allowed<MASK>(A, row, j)) {
                    const float v = to_f32(x[j]);
                    if ((v < last || (v == last && j > last_j)) && v > best) { best = v; best_j = j; }
                }
        const float top = wave_max_f32(best);
        int j = best_j >= 0 && best == top ? best_j : 0x7FFFFFFF;
        for (int o = 32; o; o >>= 1) j = min(j, __shfl_xor(j, o));
        const bool none = j == 0x7FFFFFFF;
        if (lane == 0) {
            A.top_action[row * A.top + k] = none ? -1 : j;
            A.top_logp[row * A.top + k] = bad ? __builtin_nanf("") : none ? -__builtin_huge_valf() : (top - m) * it - lnS;
        }
        last = none ? -__builtin_huge_valf() : top; last_j = none ? V : j;
    }
  }
}

template <typename T, int MASK>
__global__ __launch_bounds__(256) void k_logprobs_bwd(const Args A) {
    const int V = (int)A.v;
    const float it = A.inv_temperature;
    for (long long row = blockIdx.x; row < A.n; row += gridDim.x) {
        const float* st = A.stats + 4 * row;
        const float m = st[0], S = st[1], H = st[2], h = A.g_entropy ? A.g_entropy[row] : 0.0f;
        const float lnS = logf(S);
        const T* x = static_cast<const T*>(A.logits) + row * A.row_stride;
        T* out = static_cast<T*>(A.grad) + row * A.grad_stride;
        float G = 0.0f;
        for (int k = 0; k < A.n_given; ++k) {
            const long long a = action_at(A, row * A.n_given + k);
            if (a >= V) G = __builtin_nanf("");
            else if (a >= 0) G += A.g_logp[row * A.n_given + k];
        }
        for (int j = threadIdx.x; j < V; j += 256) {
            const float v = to_f32(x[j]);
            float dx = 0.0f;
            if (is_allowed<MASK>(A, row, j) && v != -__builtin_huge_valf()) {
                const float d = v - m, p = exp2f(d * (it * LOG2E)) / S;
                float given = 0.0f;
                for (int k = 0; k < A.n_given; ++k)
                    if (action_at(A, row * A.n_given + k) == j) given += A.g_logp[row * A.n_given + k];
                const float c = p > 0.0f ? G + h * ((d * it - lnS) + H) : p * G;
                dx = it * (given - p * c);
            }
            out[j] = (T)dx;
        }
    }
}

template <typename T> int forward_t(const Args& A, hipStream_t s) {
    const dim3 grid((unsigned)(A.n < (1 << 22) ? (A.n + 3) / 4 : 1 << 20)), block(256);
    if (A.mask_kind == CKR_MASK_NONE) hipLaunchKernelGGL((k_logprobs<T, CKR_MASK_NONE>), grid, block, 0, s, A);
    else if (A.mask_kind == CKR_MASK_BYTES) hipLaunchKernelGGL((k_logprobs<T, CKR_MASK_BYTES>), grid, block, 0, s, A);
    else hipLaunchKernelGGL((k_logprobs<T, CKR_MASK_LEGAL>), grid, block, 0, s, A);
    CKR_HIP(hipGetLastError());
    return CKR_OK;
}
template <typename T> int backward_t(const Args& A, hipStream_t s) {
    const dim3 grid((unsigned)(A.n < (1 << 20) ? A.n : 1 << 20)), block(256);
    if (A.mask_kind == CKR_MASK_NONE) hipLaunchKernelGGL((k_logprobs_bwd<T, CKR_MASK_NONE>), grid, block, 0, s, A);
    else if (A.mask_kind == CKR_MASK_BYTES) hipLaunchKernelGGL((k_logprobs_bwd<T, CKR_MASK_BYTES>), grid, block, 0, s, A);
    else hipLaunchKernelGGL((k_logprobs_bwd<T, CKR_MASK_LEGAL>), grid, block, 0, s, A);
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
    if (!(a->inv_temperature > 0.0f) || !(a->inv_temperature < __builtin_huge_valf())) return fail(CKR_ERR_INVALID, "%s: the temperature must be positive and finite", who);
    if (a->row_stride < 0 || (a->n && !a->logits)) return fail(CKR_ERR_INVALID, "%s: bad logits", who);
    return CKR_OK;
}

}  // namespace ckr

extern "C" {

int64_t ckr_logprobs_scratch(const ckr_logprobs_args* a) {
    if (int rc = ckr::check_args(a, "ckr_logprobs_scratch")) return rc;
    return 0;
}

int ckr_logprobs_forward(const ckr_logprobs_args* a, void* stream) {
    if (int rc = ckr::check_args(a, "ckr_logprobs_forward")) return rc;
    if (a->n && (!a->entropy || (a->n_given && !a->logp) || (a->top && (!a->top_action || !a->top_logp))))
        return ckr::fail(CKR_ERR_INVALID, "ckr_logprobs_forward: null output");
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

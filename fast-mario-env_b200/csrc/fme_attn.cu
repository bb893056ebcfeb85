// fme_attn.cu - decayed linear attention with restarts: over whole sequences, forward and backward, and one token at
// a time. Sizes, layouts and the recurrence are those of include/fme.h (FmeDecayAttn).
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include "fme_host.h"

namespace fme {
namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

// ---------------------------------------------------------------- token by token
// All four products of the operator are one recurrence over a (D, D) matrix M, with an index b that is summed over and
// an index a that the output keeps:   M[b][a] += x_b y_a;   out_a = sum_b z_b M[b][a]
//   o  : forward,  M = S,   x = k, y = v,  z = q       dq : forward,  M = S^T, x = v,  y = k, z = do
//   dv : backward, M = U,   x = q, y = do, z = k       dk : backward, M = U^T, x = do, y = q, z = v
// with U_t = scale q_t do_t^T + (reset_{t+1} ? 0 : lambda U_{t+1}) the gradient of S_t. Going forward the decay comes
// before the token's own product, going backward after it.
template <typename T> struct Sweep {
    const T *x, *y, *z;
    T* out;
    int64_t xt, yt, zt, ot;
    const uint8_t* reset;
    int64_t rt;
    const float* m_in;   // element (b, a) at b * mb + a * ma
    float* m_out;
    int mb, ma;
    float lam, xs, os;
    int t;
    bool back;
};

constexpr int SEQ_THREADS = 256;

// One CTA; thread (r, a) holds D / R rows b of column a in registers. One token costs two barriers.
template <typename T, int D> __device__ void sweep(const Sweep<T>& s, float* sm) {
    constexpr int R = SEQ_THREADS / D, PER = D / R;
    const int a = threadIdx.x % D, r = threadIdx.x / D;
    float* in = sm;                 // x, y, z
    float* part = sm + 3 * D;       // R x D
    float m[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) m[i] = s.m_in ? s.m_in[(r * PER + i) * s.mb + a * s.ma] : 0.f;
    for (int u = 0; u < s.t; u++) {
        const int64_t t = s.back ? s.t - 1 - u : u;
        for (int i = threadIdx.x; i < 3 * D; i += SEQ_THREADS) {
            const int w = i / D, e = i % D;
            in[i] = w == 0 ? to_f(s.x[t * s.xt + e]) * s.xs : w == 1 ? to_f(s.y[t * s.yt + e]) : to_f(s.z[t * s.zt + e]);
        }
        const bool cut = s.reset && s.reset[t * s.rt];
        __syncthreads();
        const float y = in[D + a];
        float acc = 0.f;
#pragma unroll
        for (int i = 0; i < PER; i++) {
            if (!s.back) m[i] = cut ? 0.f : m[i] * s.lam;
            m[i] = fmaf(in[r * PER + i], y, m[i]);
            acc = fmaf(in[2 * D + r * PER + i], m[i], acc);
            if (s.back) m[i] = cut ? 0.f : m[i] * s.lam;
        }
        part[r * D + a] = acc;
        __syncthreads();
        if (r == 0) {
            float o = 0.f;
#pragma unroll
            for (int i = 0; i < R; i++) o += part[i * D + a];
            s.out[t * s.ot + a] = from_f<T>(o * s.os);
        }
    }
    if (s.m_out) {
#pragma unroll
        for (int i = 0; i < PER; i++) s.m_out[(r * PER + i) * s.mb + a * s.ma] = m[i];
    }
}

template <typename T> __device__ __forceinline__ T* at(const FmeAttnTensor& x, int64_t n, int64_t h) {
    return reinterpret_cast<T*>(x.p) + n * x.sn + h * x.sh;
}

// blockIdx.x: sequence and head; blockIdx.y: which of the sweeps (forward: o; backward: dq, dv, dk)
template <typename T, int D, bool BWD>
__global__ void __launch_bounds__(SEQ_THREADS) k_sweep(const FmeDecayAttn A) {
    __shared__ float sm[3 * D + SEQ_THREADS];
    const int64_t n = blockIdx.x / A.h, h = blockIdx.x % A.h, mat = (int64_t)blockIdx.x * D * D;
    Sweep<T> s{};
    s.reset = A.reset ? A.reset + n * A.reset_sn : nullptr;
    s.rt = A.reset_st;
    s.lam = expf(A.log_decay[h]);
    s.xs = s.os = 1.f;
    s.t = A.t;
    T *q = at<T>(A.q, n, h), *k = at<T>(A.k, n, h), *v = at<T>(A.v, n, h);
    if (!BWD) {
        s.x = k; s.xt = A.k.st; s.y = v; s.yt = A.v.st; s.z = q; s.zt = A.q.st;
        s.out = at<T>(A.o, n, h); s.ot = A.o.st; s.os = A.scale;
        s.m_in = A.s_in ? A.s_in + mat : nullptr; s.m_out = A.s_out ? A.s_out + mat : nullptr; s.mb = D; s.ma = 1;
    } else {
        T* g = at<T>(A.d_o, n, h);
        if (blockIdx.y == 0) {
            s.x = v; s.xt = A.v.st; s.y = k; s.yt = A.k.st; s.z = g; s.zt = A.d_o.st;
            s.out = at<T>(A.dq, n, h); s.ot = A.dq.st; s.os = A.scale;
            s.m_in = A.s_in ? A.s_in + mat : nullptr; s.mb = 1; s.ma = D;
        } else {
            s.back = true; s.xs = A.scale;
            s.m_in = A.ds_out ? A.ds_out + mat : nullptr;
            if (blockIdx.y == 1) {
                s.x = q; s.xt = A.q.st; s.y = g; s.yt = A.d_o.st; s.z = k; s.zt = A.k.st;
                s.out = at<T>(A.dv, n, h); s.ot = A.dv.st;
                s.m_out = A.ds_in ? A.ds_in + mat : nullptr; s.mb = D; s.ma = 1;
            } else {
                s.x = g; s.xt = A.d_o.st; s.y = q; s.yt = A.q.st; s.z = v; s.zt = A.v.st;
                s.out = at<T>(A.dk, n, h); s.ot = A.dk.st;
                s.mb = 1; s.ma = D;
            }
        }
    }
    sweep<T, D>(s, sm);
}

// ---------------------------------------------------------------- host side
int bad(const char* msg) { return host_fail(FME_E_ARG, msg); }

int check_sizes(const FmeDecayAttn* a) {
    if (!a) return bad("null decay attention arguments");
    if (a->n < 0 || a->t < 0 || a->h < 1) return bad("decay attention: n and t must be >= 0 and h >= 1");
    if ((int64_t)a->n * a->h > 0x7fffffff) return bad("decay attention: more than 2^31 - 1 (sequence, head) pairs");
    if (a->d != 32 && a->d != 64 && a->d != 128) return bad("decay attention: d must be 32, 64 or 128");
    if (a->dtype != FME_F32 && a->dtype != FME_BF16) return bad("decay attention: dtype must be FME_F32 or FME_BF16");
    return FME_OK;
}
bool rows_aligned(const FmeAttnTensor& x, int dtype) {
    const int64_t e = dtype == FME_F32 ? 4 : 2;
    return x.p && !((uintptr_t)x.p & 15) && !((x.sn * e) & 15) && !((x.st * e) & 15) && !((x.sh * e) & 15);
}
bool aligned16(const void* p) { return !((uintptr_t)p & 15); }

int check_common(const FmeDecayAttn* a) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (!a->log_decay) return bad("decay attention: null log_decay");
    if (!aligned16(a->s_in) || !aligned16(a->s_out) || !aligned16(a->ds_in) || !aligned16(a->ds_out) || !aligned16(a->saved))
        return bad("decay attention: states must be 16-byte aligned");
    if (a->n && a->t && (!rows_aligned(a->q, a->dtype) || !rows_aligned(a->k, a->dtype) || !rows_aligned(a->v, a->dtype)))
        return bad("decay attention: q, k, v must be given, with 16-byte aligned rows");
    return FME_OK;
}

template <typename T, int D> void launch_fwd(const FmeDecayAttn& a, cudaStream_t st) {
    k_sweep<T, D, false><<<dim3(a.n * a.h, 1), SEQ_THREADS, 0, st>>>(a);
}
template <typename T, int D> void launch_bwd(const FmeDecayAttn& a, cudaStream_t st) {
    k_sweep<T, D, true><<<dim3(a.n * a.h, 3), SEQ_THREADS, 0, st>>>(a);
}
#define FME_BY_TYPE(a, FN, st)                                                           \
    do {                                                                                 \
        if ((a).dtype == FME_F32) {                                                      \
            if ((a).d == 32) FN<float, 32>(a, st);                                       \
            else if ((a).d == 64) FN<float, 64>(a, st);                                  \
            else FN<float, 128>(a, st);                                                  \
        } else {                                                                         \
            if ((a).d == 32) FN<__nv_bfloat16, 32>(a, st);                               \
            else if ((a).d == 64) FN<__nv_bfloat16, 64>(a, st);                          \
            else FN<__nv_bfloat16, 128>(a, st);                                          \
        }                                                                                \
    } while (0)

}  // namespace
}  // namespace fme

using namespace fme;

extern "C" {

int64_t fme_decay_attn_bytes(const FmeDecayAttn* a, int32_t which) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (which < 0 || which > 2) return bad("decay attention: which must be 0, 1 or 2");
    return 0;
}

int fme_decay_attn_fwd(const FmeDecayAttn* a, void* stream) {
    const int rc = check_common(a);
    if (rc) return rc;
    if (a->n == 0) return FME_OK;
    if (a->t && !rows_aligned(a->o, a->dtype)) return bad("decay attention: o must be given, with 16-byte aligned rows");
    FME_BY_TYPE(*a, launch_fwd, (cudaStream_t)stream);
    return launch_status("fme_decay_attn_fwd");
}

int fme_decay_attn_bwd(const FmeDecayAttn* a, void* stream) {
    const int rc = check_common(a);
    if (rc) return rc;
    if (a->n == 0) return FME_OK;
    if (a->t && (!rows_aligned(a->d_o, a->dtype) || !rows_aligned(a->dq, a->dtype) || !rows_aligned(a->dk, a->dtype) ||
                 !rows_aligned(a->dv, a->dtype)))
        return bad("decay attention: the gradients must be given, with 16-byte aligned rows");
    FME_BY_TYPE(*a, launch_bwd, (cudaStream_t)stream);
    return launch_status("fme_decay_attn_bwd");
}

int fme_decay_attn_step(const FmeDecayAttn* a, void* stream) {
    const int rc = check_common(a);
    if (rc) return rc;
    if (a->t != 1) return bad("decay attention step: t must be 1");
    if (a->n == 0) return FME_OK;
    if (!a->s_in || !a->s_out) return bad("decay attention step: s_in and s_out are required");
    if (!rows_aligned(a->o, a->dtype)) return bad("decay attention: o must be given, with 16-byte aligned rows");
    FME_BY_TYPE(*a, launch_fwd, (cudaStream_t)stream);
    return launch_status("fme_decay_attn_step");
}

}  // extern "C"

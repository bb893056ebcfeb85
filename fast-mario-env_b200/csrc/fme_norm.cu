// fme_norm.cu - group norm with an activation for channels-last activations, forward and backward, with the backward
// pass's input kept whole or as 8-bit codes. Sizes, layouts and formulas are those of include/fme.h (FmeGroupNorm).
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

__device__ __forceinline__ float act_fwd(float z, int act) {
    return act == FME_ACT_SILU ? z / (1.f + expf(-z)) : act == FME_ACT_RELU ? (z < 0.f ? 0.f : z) : z;
}
__device__ __forceinline__ float act_bwd(float z, float dy, int act) {
    if (act == FME_ACT_SILU) { const float s = 1.f / (1.f + expf(-z)); return dy * s * (1.f + z * (1.f - s)); }
    return act == FME_ACT_RELU ? (z <= 0.f ? 0.f : dy) : dy;
}

constexpr int NT = 256;
constexpr int MAX_C = 4096;

// One CTA walks samples blockIdx.x, + gridDim.x, ...; per-channel sums in shared memory, one thread a channel.
template <typename T> __global__ void __launch_bounds__(NT) k_norm_fwd(const FmeGroupNorm A) {
    extern __shared__ float sm[];
    float *s0 = sm, *s1 = sm + A.c, *s2 = sm + 2 * A.c;
    const int cg = A.c / A.g;
    const float m = (float)((int64_t)A.p * cg);
    for (int64_t n = blockIdx.x; n < A.n; n += gridDim.x) {
        const T* x = (const T*)A.x + n * A.x_sn;
        const int64_t base = n * (int64_t)A.p * A.c;
        for (int c = threadIdx.x; c < A.c; c += NT) {
            float s = 0.f, lo = INFINITY, hi = -INFINITY;
            for (int64_t p = 0; p < A.p; p++) { const float v = to_f(x[p * A.c + c]); s += v; lo = fminf(lo, v); hi = fmaxf(hi, v); }
            s0[c] = s; s1[c] = lo; s2[c] = hi;
        }
        __syncthreads();
        for (int g = threadIdx.x; g < A.g; g += NT) {
            float s = 0.f, lo = INFINITY, hi = -INFINITY;
            for (int c = g * cg; c < (g + 1) * cg; c++) { s += s0[c]; lo = fminf(lo, s1[c]); hi = fmaxf(hi, s2[c]); }
            s /= m;
            for (int c = g * cg; c < (g + 1) * cg; c++) { s0[c] = s; s1[c] = lo; s2[c] = hi; }
            if (A.codes) { A.lo[n * A.g + g] = lo; A.hi[n * A.g + g] = hi; }
            if (A.mean) A.mean[n * A.g + g] = s;
        }
        __syncthreads();
        if (A.codes) {
            for (int c = threadIdx.x; c < A.c; c += NT) {
                const float lo = s1[c], d = s2[c] - lo, inv = d > 0.f ? __fmul_rn(__frcp_rn(d), 255.f) : 0.f;
                for (int64_t p = 0; p < A.p; p++)
                    A.codes[base + p * A.c + c] = (uint8_t)rintf(__fmul_rn(__fsub_rn(to_f(x[p * A.c + c]), lo), inv));
            }
        }
        __syncthreads();
        for (int c = threadIdx.x; c < A.c; c += NT) {
            float q = 0.f;
            for (int64_t p = 0; p < A.p; p++) { const float d = to_f(x[p * A.c + c]) - s0[c]; q = fmaf(d, d, q); }
            s1[c] = q;
        }
        __syncthreads();
        for (int g = threadIdx.x; g < A.g; g += NT) {
            float q = 0.f;
            for (int c = g * cg; c < (g + 1) * cg; c++) q += s1[c];
            const float r = rsqrtf(q / m + A.eps);
            for (int c = g * cg; c < (g + 1) * cg; c++) s2[c] = r;
            if (A.rstd) A.rstd[n * A.g + g] = r;
        }
        __syncthreads();
        for (int c = threadIdx.x; c < A.c; c += NT) {
            const float w = A.w ? A.w[c] : 1.f, b = A.b ? A.b[c] : 0.f;
            for (int64_t p = 0; p < A.p; p++)
                ((T*)A.y)[base + p * A.c + c] = from_f<T>(act_fwd(fmaf((to_f(x[p * A.c + c]) - s0[c]) * s2[c], w, b), A.act));
        }
        __syncthreads();
    }
}

template <typename T> __device__ __forceinline__ float x_of(const FmeGroupNorm& A, int64_t n, int64_t i, float lo, float step) {
    if (A.codes) return __fadd_rn(lo, __fmul_rn((float)A.codes[n * (int64_t)A.p * A.c + i], step));
    return to_f(((const T*)A.x)[n * A.x_sn + i]);
}

// As the forward kernel; a CTA's sums of dw and db over its samples go to its row of the workspace.
template <typename T> __global__ void __launch_bounds__(NT) k_norm_bwd(const FmeGroupNorm A) {
    extern __shared__ float sm[];
    float *s0 = sm, *s1 = sm + A.c, *tw = sm + 2 * A.c, *tb = sm + 3 * A.c;
    const int cg = A.c / A.g;
    const float m = (float)((int64_t)A.p * cg);
    for (int c = threadIdx.x; c < A.c; c += NT) tw[c] = tb[c] = 0.f;
    __syncthreads();
    for (int64_t n = blockIdx.x; n < A.n; n += gridDim.x) {
        const T* dy = (const T*)A.dy + n * A.dy_sn;
        for (int pass = 0; pass < 2; pass++) {
            for (int c = threadIdx.x; c < A.c; c += NT) {
                const int64_t ng = n * A.g + c / cg;
                const float mean = A.mean[ng], rstd = A.rstd[ng], w = A.w ? A.w[c] : 1.f, b = A.b ? A.b[c] : 0.f;
                const float lo = A.codes ? A.lo[ng] : 0.f, step = A.codes ? __fdiv_rn(__fsub_rn(A.hi[ng], lo), 255.f) : 0.f;
                float a1 = 0.f, a2 = 0.f;
                for (int64_t p = 0; p < A.p; p++) {
                    const int64_t i = p * A.c + c;
                    const float xh = (x_of<T>(A, n, i, lo, step) - mean) * rstd;
                    const float dz = act_bwd(fmaf(xh, w, b), to_f(dy[i]), A.act);
                    if (pass == 0) { a1 += dz; a2 = fmaf(dz, xh, a2); }
                    else ((T*)A.dx)[n * (int64_t)A.p * A.c + i] = from_f<T>(rstd * (dz * w - s0[c] - xh * s1[c]));
                }
                if (pass == 0) { s0[c] = a1; s1[c] = a2; tb[c] += a1; tw[c] += a2; }
            }
            __syncthreads();
            if (pass == 0) {
                for (int g = threadIdx.x; g < A.g; g += NT) {
                    float a1 = 0.f, a2 = 0.f;
                    for (int c = g * cg; c < (g + 1) * cg; c++) { const float w = A.w ? A.w[c] : 1.f; a1 = fmaf(s0[c], w, a1); a2 = fmaf(s1[c], w, a2); }
                    for (int c = g * cg; c < (g + 1) * cg; c++) { s0[c] = a1 / m; s1[c] = a2 / m; }
                }
                __syncthreads();
            }
        }
    }
    if (A.dw) {
        float* row = (float*)A.ws + (int64_t)blockIdx.x * 2 * A.c;
        for (int c = threadIdx.x; c < A.c; c += NT) { row[c] = tw[c]; row[A.c + c] = tb[c]; }
    }
}

__global__ void __launch_bounds__(NT) k_norm_params(const float* ws, int rows, int c, float* dw, float* db) {
    const int i = blockIdx.x * NT + threadIdx.x;
    if (i >= 2 * c) return;
    float s = 0.f;
    for (int r = 0; r < rows; r++) s += ws[(int64_t)r * 2 * c + i];
    if (i < c) dw[i] = s; else db[i - c] = s;
}

// ---------------------------------------------------------------- host side
int bad(const char* msg) { return host_fail(FME_E_ARG, msg); }
int check_sizes(const FmeGroupNorm* a) {
    if (!a) return bad("null group norm arguments");
    if (a->n < 0 || a->p < 0 || a->c < 1 || a->g < 1 || a->c % a->g) return bad("group norm: sizes must be >= 0 and g must divide c");
    if (a->c > MAX_C) return bad("group norm: c must be at most 4096");
    if (a->dtype != FME_F32 && a->dtype != FME_BF16) return bad("group norm: dtype must be FME_F32 or FME_BF16");
    if (a->act < FME_ACT_NONE || a->act > FME_ACT_SILU) return bad("group norm: unknown activation");
    return FME_OK;
}
int grid_of(const FmeGroupNorm* a) { return a->n < 592 ? a->n : 592; }

}  // namespace
}  // namespace fme

using namespace fme;

extern "C" {

int64_t fme_group_norm_bytes(const FmeGroupNorm* a, int32_t which) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (which < 0 || which > 1) return bad("group norm: which must be 0 or 1");
    return which == 1 ? (int64_t)grid_of(a) * 2 * a->c * 4 : 0;
}

int fme_group_norm_fwd(const FmeGroupNorm* a, void* stream) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (a->n == 0 || a->p == 0) return FME_OK;
    if (!a->x || !a->y) return bad("group norm: x and y are required");
    if (a->codes && (!a->lo || !a->hi)) return bad("group norm: codes need lo and hi");
    const size_t smem = (size_t)3 * a->c * 4;
    if (a->dtype == FME_F32) k_norm_fwd<float><<<grid_of(a), NT, smem, (cudaStream_t)stream>>>(*a);
    else k_norm_fwd<__nv_bfloat16><<<grid_of(a), NT, smem, (cudaStream_t)stream>>>(*a);
    return launch_status("fme_group_norm_fwd");
}

int fme_group_norm_bwd(const FmeGroupNorm* a, void* stream) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if ((a->dw == nullptr) != (a->db == nullptr)) return bad("group norm: dw and db come together");
    if (a->n == 0 || a->p == 0) {
        if (a->dw) {
            if (cudaMemsetAsync(a->dw, 0, 4 * (size_t)a->c, (cudaStream_t)stream) != cudaSuccess ||
                cudaMemsetAsync(a->db, 0, 4 * (size_t)a->c, (cudaStream_t)stream) != cudaSuccess)
                return launch_status("fme_group_norm_bwd");
        }
        return FME_OK;
    }
    if ((!a->x && !a->codes) || !a->dy || !a->dx || !a->mean || !a->rstd) return bad("group norm: x or codes, dy, dx, mean and rstd are required");
    if (a->codes && (!a->lo || !a->hi)) return bad("group norm: codes need lo and hi");
    if (a->dw && (!a->ws || a->ws_bytes < fme_group_norm_bytes(a, 1))) return bad("group norm: workspace too small");
    const size_t smem = (size_t)4 * a->c * 4;
    const int grid = grid_of(a);
    if (smem > 48 * 1024) {
        cudaFuncSetAttribute(k_norm_bwd<float>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        cudaFuncSetAttribute(k_norm_bwd<__nv_bfloat16>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    }
    if (a->dtype == FME_F32) k_norm_bwd<float><<<grid, NT, smem, (cudaStream_t)stream>>>(*a);
    else k_norm_bwd<__nv_bfloat16><<<grid, NT, smem, (cudaStream_t)stream>>>(*a);
    if (a->dw) k_norm_params<<<(2 * a->c + NT - 1) / NT, NT, 0, (cudaStream_t)stream>>>((const float*)a->ws, grid, a->c, a->dw, a->db);
    return launch_status("fme_group_norm_bwd");
}

}  // extern "C"

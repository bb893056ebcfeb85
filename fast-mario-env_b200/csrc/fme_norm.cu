// fme_norm.cu - group norm with an activation for channels-last activations, forward and backward, with the backward
// pass's input kept whole or as 8-bit codes. Sizes, layouts and formulas are those of include/fme.h (FmeGroupNorm).
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <math.h>
#include <stdint.h>

#include <type_traits>

#include "fme_host.h"

namespace fme {
namespace {

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16(x); }

namespace cg = cooperative_groups;

// sigmoid by the fast exponential and division: both are off by a few units of 2^-23, as the sums around them
__device__ __forceinline__ float sigmoid(float z) { return __fdividef(1.f, 1.f + __expf(-z)); }
__device__ __forceinline__ float act_fwd(int act, float z) {
    return act == FME_ACT_SILU ? z * sigmoid(z) : act == FME_ACT_RELU ? (z < 0.f ? 0.f : z) : z;
}
__device__ __forceinline__ float act_bwd(int act, float z, float dy) {
    if (act == FME_ACT_SILU) { const float s = sigmoid(z); return dy * s * (1.f + z * (1.f - s)); }
    return act == FME_ACT_RELU ? (z <= 0.f ? 0.f : dy) : dy;
}

template <int V> struct cuda_int { static constexpr int value = V; };
constexpr int NT = 256;
constexpr int MAX_C = 4096;

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Pack { T v[VEC]; };

// ---------------------------------------------------------------- samples held in registers
// A sample is p * c values in a row. Threads take vectors of VEC of them; R threads form a team and R * VEC is a multiple
// of c, so that a thread meets the same channels in each of its K vectors and keeps their weights in registers. A team
// holds R * K vectors. Small samples: M teams in a CTA, a sample each. Large ones: the CTAs of a cluster share a sample and
// add up their sums through distributed shared memory. So x (and dy) are read once, which is the bound: HBM bytes.
// Where no cluster can hold a sample (or so few samples would leave most SMs idle) its pieces are separate CTAs, and the
// kernel runs twice, for the sums (STATS) and, after k_norm_join*, for the values (APPLY), with a second read of the inputs.
// GR: all values of a vector belong to one group (VEC divides c / g).
enum Phase { WHOLE, STATS, APPLY };

struct Plan {
    int R, M, K, vec, parts;   // parts: CTAs that share a sample
    bool gr, cluster;
    int threads, grid;         // grid: CTAs
    size_t smem;
};

template <int NS> struct Slots {   // where the values to be summed over a group stand in shared memory
    int R, M, L, gl, rows, G, n;
    __device__ Slots(const FmeGroupNorm& A, int R_, int M_, int vec)
        : R(R_), M(M_), L(NS == 1 ? A.c / vec : A.c), gl(L / A.g), rows(R_ * NS / L), G(A.g), n(R_ * M_ * NS) {}
};

// Sum (or, for the second and third value with MM, minimum and maximum) of NV values of each (team, group), in a fixed order;
// out[v * M * G + pair]. All threads of the CTA call it.
template <int NV, int NS, bool MM>
__device__ __forceinline__ void group_reduce(const Slots<NS>& S, const float (&v)[NV][NS], bool mine, float* red, float* out) {
    if (mine) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < NS; j++) red[i * S.n + threadIdx.x * NS + j] = v[i][j];
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, members = S.rows * S.gl, pairs = S.M * S.G;
    for (int pair = threadIdx.x >> 5; pair < pairs; pair += blockDim.x >> 5) {
        const int base = (pair / S.G) * S.R * NS + (pair % S.G) * S.gl;
        float a[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) a[i] = !MM || i == 0 ? 0.f : i == 1 ? INFINITY : -INFINITY;
        for (int m = lane; m < members; m += 32) {
            const int at = base + (m / S.gl) * S.L + m % S.gl;
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const float x = red[i * S.n + at];
                a[i] = !MM || i == 0 ? a[i] + x : i == 1 ? fminf(a[i], x) : fmaxf(a[i], x);
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; i++) {
                const float x = __shfl_xor_sync(0xffffffffu, a[i], o);
                a[i] = !MM || i == 0 ? a[i] + x : i == 1 ? fminf(a[i], x) : fmaxf(a[i], x);
            }
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < NV; i++) out[i * pairs + pair] = a[i];
        }
    }
    __syncthreads();
}

// mean and rstd from the parts' means and squared distances (count of values each)
struct Moments {
    float n = 0.f, mean = 0.f, m2 = 0.f;
    __device__ __forceinline__ void add(float cnt, float mu, float q) {
        if (cnt == 0.f) return;
        const float t = n + cnt, d = mu - mean;
        mean = fmaf(d, cnt / t, mean);
        m2 += q + d * d * (n * cnt / t);
        n = t;
    }
};

__device__ __forceinline__ float rstd_of(float m2, float m, float eps) { return __frsqrt_rn(m2 / m + eps); }
__device__ __forceinline__ float code_inv(float lo, float hi) { return hi > lo ? __fmul_rn(__frcp_rn(__fsub_rn(hi, lo)), 255.f) : 0.f; }
__device__ __forceinline__ float code_step(float lo, float hi) { return __fdiv_rn(__fsub_rn(hi, lo), 255.f); }

template <typename T, int VEC, int K, bool GR, int PH>
__global__ void __launch_bounds__(512) k_norm_fwd(const FmeGroupNorm A, const int R, const int M, const int parts) {
    constexpr int NS = GR ? 1 : VEC;
    extern __shared__ float sm[];
    const Slots<NS> S(A, R, M, VEC);
    const int pairs = M * A.g, team = threadIdx.x / R, t = threadIdx.x - team * R;
    float* red = sm;                       // 3 * S.n, or 1 * S.n
    float* out = sm + 3 * S.n;             // 3 * pairs: sum, lo, hi; then mean, rstd in the first two
    float* out2 = out + 3 * pairs;         // pairs
    float* part = out2 + pairs;            // 4 * pairs: what the cluster's other CTAs read
    const int rank = blockIdx.x % parts;
    const int64_t n = (int64_t)(blockIdx.x / parts) * M + team;
    const bool mine = team < M, ok = mine && n < A.n;
    const int nvec = (int)((int64_t)A.p * A.c / VEC), v0 = rank * R * K;
    const int count = max(0, min(nvec - v0, R * K));
    const float cnt = (float)((int64_t)count * VEC / A.g);   // of each group in this CTA: whole pixels
    const T* x = (const T*)A.x + n * A.x_sn;
    Pack<T, VEC> raw[K];
#pragma unroll
    for (int k = 0; k < K; k++)
        if (ok && k * R + t < count) raw[k] = reinterpret_cast<const Pack<T, VEC>*>(x)[v0 + k * R + t];
    const int c0 = (int)((int64_t)t * VEC % A.c), cgr = A.c / A.g;
    int ch[VEC];                           // channel of each value of the vector
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        ch[j] = c0 + j;
        if (!GR) ch[j] %= A.c;
        w[j] = PH != STATS && A.w ? __ldg(A.w + ch[j]) : 1.f;
        b[j] = PH != STATS && A.b ? __ldg(A.b + ch[j]) : 0.f;
    }
    int grp[NS];
#pragma unroll
    for (int j = 0; j < NS; j++) grp[j] = team * A.g + ch[j] / cgr;
    const bool u8 = A.codes != nullptr;
    if (PH != APPLY) {
        float v[3][NS];
#pragma unroll
        for (int j = 0; j < NS; j++) { v[0][j] = 0.f; v[1][j] = INFINITY; v[2][j] = -INFINITY; }
#pragma unroll
        for (int k = 0; k < K; k++)
            if (ok && k * R + t < count) {
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const float f = to_f(raw[k].v[j]);
                    const int s = GR ? 0 : j;
                    v[0][s] += f;
                    if (u8) { v[1][s] = fminf(v[1][s], f); v[2][s] = fmaxf(v[2][s], f); }
                }
            }
        if (u8) group_reduce<3, NS, true>(S, v, mine, red, out);
        else { float s1[1][NS];
#pragma unroll
            for (int j = 0; j < NS; j++) s1[0][j] = v[0][j];
            group_reduce<1, NS, false>(S, s1, mine, red, out); }
        float mu[NS], q[1][NS];
#pragma unroll
        for (int j = 0; j < NS; j++) { mu[j] = mine && cnt > 0.f ? out[grp[j]] / cnt : 0.f; q[0][j] = 0.f; }
#pragma unroll
        for (int k = 0; k < K; k++)
            if (ok && k * R + t < count) {
#pragma unroll
                for (int j = 0; j < VEC; j++) { const int s = GR ? 0 : j; const float d = to_f(raw[k].v[j]) - mu[s]; q[0][s] = fmaf(d, d, q[0][s]); }
            }
        group_reduce<1, NS, false>(S, q, mine, red, out2);
    }
    const float m = (float)((int64_t)A.p * cgr);
    if (PH == STATS) {                     // (sample, part, group): mean, squared distances, lo, hi
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            float4* dst = reinterpret_cast<float4*>(A.ws) + ((blockIdx.x / parts) * (int64_t)parts + rank) * A.g + i;   // M is 1 here
            *dst = make_float4(cnt > 0.f ? out[i] / cnt : 0.f, out2[i], u8 ? out[pairs + i] : 0.f, u8 ? out[2 * pairs + i] : 0.f);
        }
        return;
    }
    if (PH == WHOLE) {
        if (parts == 1) {
            for (int i = threadIdx.x; i < pairs; i += blockDim.x) { out[i] = out[i] / m; out2[i] = rstd_of(out2[i], m, A.eps); }
        } else {
            cg::cluster_group cl = cg::this_cluster();
            for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
                part[i] = cnt > 0.f ? out[i] / cnt : 0.f; part[pairs + i] = out2[i];
                if (u8) { part[2 * pairs + i] = out[pairs + i]; part[3 * pairs + i] = out[2 * pairs + i]; }
            }
            cl.sync();
            for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
                Moments mo;
                float lo = INFINITY, hi = -INFINITY;
                for (int r = 0; r < parts; r++) {
                    const float* o = cl.map_shared_rank(part, r);
                    const int rc = max(0, min(nvec - r * R * K, R * K));
                    mo.add((float)((int64_t)rc * VEC / A.g), o[i], o[pairs + i]);
                    if (u8) { lo = fminf(lo, o[2 * pairs + i]); hi = fmaxf(hi, o[3 * pairs + i]); }
                }
                out[i] = mo.mean; out2[i] = rstd_of(mo.m2, m, A.eps);
                if (u8) { out[pairs + i] = lo; out[2 * pairs + i] = hi; }
            }
            cg::this_cluster().barrier_arrive();   // this CTA has read the others; it ends only when they have read it
        }
    } else {
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            const float4 f = reinterpret_cast<const float4*>(A.ws)[(int64_t)A.n * parts * A.g + (blockIdx.x / parts) * (int64_t)A.g + i];
            out[i] = f.x; out2[i] = f.y;
            if (u8) { out[pairs + i] = f.z; out[2 * pairs + i] = f.w; }
        }
    }
    __syncthreads();
    if (rank == 0) {
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            const int64_t ng = (int64_t)(blockIdx.x / parts) * pairs + i;
            if (ng < (int64_t)A.n * A.g) {
                if (A.mean) { A.mean[ng] = out[i]; A.rstd[ng] = out2[i]; }
                if (u8) { A.lo[ng] = out[pairs + i]; A.hi[ng] = out[2 * pairs + i]; }
            }
        }
    }
    if (ok) {
        float mean[NS], rstd[NS], lo[NS], inv[NS];
#pragma unroll
        for (int j = 0; j < NS; j++) {
            mean[j] = out[grp[j]]; rstd[j] = out2[grp[j]];
            if (u8) { lo[j] = out[pairs + grp[j]]; inv[j] = code_inv(lo[j], out[2 * pairs + grp[j]]); }
        }
        const int64_t base = n * nvec + v0;
        auto apply = [&](auto act) {
#pragma unroll
            for (int k = 0; k < K; k++)
                if (k * R + t < count) {
                    Pack<T, VEC> y;
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const int s = GR ? 0 : j;
                        y.v[j] = from_f<T>(act_fwd(decltype(act)::value, fmaf((to_f(raw[k].v[j]) - mean[s]) * rstd[s], w[j], b[j])));
                    }
                    reinterpret_cast<Pack<T, VEC>*>(A.y)[base + k * R + t] = y;
                }
        };
        if (u8) {
#pragma unroll
            for (int k = 0; k < K; k++)
                if (k * R + t < count) {
                    Pack<uint8_t, VEC> q;
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const int s = GR ? 0 : j;   // in 0..255 by construction; a group with NaN gets some code
                        q.v[j] = (uint8_t)__float2uint_rn(__fmul_rn(__fsub_rn(to_f(raw[k].v[j]), lo[s]), inv[s]));
                    }
                    reinterpret_cast<Pack<uint8_t, VEC>*>(A.codes)[base + k * R + t] = q;
                }
        }
        if (A.act == FME_ACT_SILU) apply(cuda_int<FME_ACT_SILU>{});
        else if (A.act == FME_ACT_RELU) apply(cuda_int<FME_ACT_RELU>{});
        else apply(cuda_int<FME_ACT_NONE>{});
    }
    if (PH == WHOLE && parts > 1) cg::this_cluster().barrier_wait();
}

// One warp a (sample, group): its parts' moments in order, to the end of the workspace.
template <typename T, int VEC> __global__ void __launch_bounds__(NT) k_norm_join_fwd(const FmeGroupNorm A, const int parts, const int per) {
    const int64_t i = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= (int64_t)A.n * A.g) return;
    const int64_t n = i / A.g;
    const int g = (int)(i % A.g), nvec = (int)((int64_t)A.p * A.c / VEC);
    Moments mo;
    float lo = INFINITY, hi = -INFINITY;
    const float4* src = reinterpret_cast<const float4*>(A.ws);
    for (int r = lane; r < parts; r += 32) {
        const float4 f = src[(n * parts + r) * A.g + g];
        mo.add((float)((int64_t)max(0, min(nvec - r * per, per)) * VEC / A.g), f.x, f.y);
        lo = fminf(lo, f.z); hi = fmaxf(hi, f.w);
    }
    for (int o = 1; o < 32; o <<= 1) {
        const float on = __shfl_down_sync(0xffffffffu, mo.n, o), om = __shfl_down_sync(0xffffffffu, mo.mean, o), oq = __shfl_down_sync(0xffffffffu, mo.m2, o);
        mo.add(on, om, oq);
        lo = fminf(lo, __shfl_down_sync(0xffffffffu, lo, o)); hi = fmaxf(hi, __shfl_down_sync(0xffffffffu, hi, o));
    }
    if (lane == 0) {
        const float m = (float)((int64_t)A.p * (A.c / A.g));
        reinterpret_cast<float4*>(A.ws)[(int64_t)A.n * parts * A.g + i] = make_float4(mo.mean, rstd_of(mo.m2, m, A.eps), lo, hi);
    }
}

// x^ = (x - mean) rstd, z = w x^ + b, dz = dy act'(z); dw = sum dz x^, db = sum dz;
// dx = rstd (w dz - mean(w dz) - x^ mean(w dz x^)), the means over the (sample, group).
// A CTA (or cluster) walks samples and keeps its channels' dw and db in registers until the end.
template <typename T, int VEC, int K, bool GR, int PH, bool U8>
__global__ void __launch_bounds__(512) k_norm_bwd(const FmeGroupNorm A, const int R, const int M, const int parts) {
    constexpr int NS = GR ? 1 : VEC;
    extern __shared__ float sm[];
    const Slots<NS> S(A, R, M, VEC);
    const int pairs = M * A.g, team = threadIdx.x / R, t = threadIdx.x - team * R;
    float* red = sm;                       // 2 * S.n (at the end 2 * threads * VEC)
    float* out = sm + 2 * R * M * VEC;     // 2 * pairs
    float* part = out + 2 * pairs;         // 2 * pairs
    const int rank = blockIdx.x % parts, nvec = (int)((int64_t)A.p * A.c / VEC), v0 = rank * R * K;
    const int count = max(0, min(nvec - v0, R * K));
    const int c0 = (int)((int64_t)t * VEC % A.c), cgr = A.c / A.g;
    const float m = (float)((int64_t)A.p * cgr);
    const bool mine = team < M;
    int ch[VEC];
    float w[VEC], b[VEC], dw[VEC], db[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        ch[j] = c0 + j;
        if (!GR) ch[j] %= A.c;
        w[j] = A.w ? __ldg(A.w + ch[j]) : 1.f;
        b[j] = A.b ? __ldg(A.b + ch[j]) : 0.f;
        dw[j] = db[j] = 0.f;
    }
    int grp[NS];
#pragma unroll
    for (int j = 0; j < NS; j++) grp[j] = ch[j] / cgr;
    for (int64_t n0 = (int64_t)(blockIdx.x / parts) * M; n0 < A.n; n0 += (int64_t)(gridDim.x / parts) * M) {
        const int64_t n = n0 + team;
        const bool ok = mine && n < A.n;
        Pack<T, VEC> rx[U8 ? 1 : K], rd[K];
        Pack<uint8_t, VEC> rc[U8 ? K : 1];
        const T* dy = (const T*)A.dy + n * A.dy_sn;
#pragma unroll
        for (int k = 0; k < K; k++)
            if (ok && k * R + t < count) {
                const int i = v0 + k * R + t;
                if (U8) rc[k] = reinterpret_cast<const Pack<uint8_t, VEC>*>(A.codes)[n * nvec + i];
                else rx[k] = reinterpret_cast<const Pack<T, VEC>*>((const T*)A.x + n * A.x_sn)[i];
                rd[k] = reinterpret_cast<const Pack<T, VEC>*>(dy)[i];
            }
        // x^ = x * xa + xb (of codes: code * xa + xb)
        float xa[NS], xb[NS], rstd[NS];
#pragma unroll
        for (int j = 0; j < NS; j++) {
            const int64_t ng = n * A.g + grp[j];
            rstd[j] = ok ? __ldg(A.rstd + ng) : 0.f;
            const float mean = ok ? __ldg(A.mean + ng) : 0.f;
            if (U8) {
                const float lo = ok ? __ldg(A.lo + ng) : 0.f, hi = ok ? __ldg(A.hi + ng) : 0.f;
                xa[j] = code_step(lo, hi) * rstd[j]; xb[j] = (lo - mean) * rstd[j];
            } else { xa[j] = rstd[j]; xb[j] = mean; }
        }
        auto hat = [&](int k, int j) {
            const int s = GR ? 0 : j;
            return U8 ? fmaf((float)rc[U8 ? k : 0].v[j], xa[s], xb[s]) : (to_f(rx[U8 ? 0 : k].v[j]) - xb[s]) * xa[s];
        };
        auto value = [&](auto act) {
            if (PH != APPLY) {
                float v[2][NS];
#pragma unroll
                for (int j = 0; j < NS; j++) v[0][j] = v[1][j] = 0.f;
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (ok && k * R + t < count) {
#pragma unroll
                        for (int j = 0; j < VEC; j++) {
                            const int s = GR ? 0 : j;
                            const float xh = hat(k, j), dz = act_bwd(decltype(act)::value, fmaf(xh, w[j], b[j]), to_f(rd[k].v[j]));
                            if (sizeof(T) == 4) rd[k].v[j] = from_f<T>(dz);   // fp32 keeps dz; bf16 would round it
                            const float wd = w[j] * dz;
                            v[0][s] += wd; v[1][s] = fmaf(wd, xh, v[1][s]);
                            db[j] += dz; dw[j] = fmaf(dz, xh, dw[j]);
                        }
                    }
                group_reduce<2, NS, false>(S, v, mine, red, out);
            }
            if (PH == STATS) {
                for (int i = threadIdx.x; i < pairs; i += blockDim.x)
                    reinterpret_cast<float2*>(A.ws)[(n0 * parts + rank) * A.g + i] = make_float2(out[i], out[pairs + i]);
                return;
            }
            if (PH == WHOLE && parts > 1) {
                cg::cluster_group cl = cg::this_cluster();
                for (int i = threadIdx.x; i < 2 * pairs; i += blockDim.x) part[i] = out[i];
                cl.sync();
                for (int i = threadIdx.x; i < 2 * pairs; i += blockDim.x) {
                    float s = 0.f;
                    for (int r = 0; r < parts; r++) s += cl.map_shared_rank(part, r)[i];
                    out[i] = s;
                }
                cl.barrier_arrive();
                __syncthreads();
            }
            if (PH == APPLY) {
                for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
                    const float2 f = reinterpret_cast<const float2*>(A.ws)[(int64_t)A.n * parts * A.g + n0 * A.g + i];
                    out[i] = f.x; out[pairs + i] = f.y;
                }
                __syncthreads();
            }
            if (ok) {
                float a1[NS], a2[NS];
#pragma unroll
                for (int j = 0; j < NS; j++) { a1[j] = out[team * A.g + grp[j]] / m; a2[j] = out[pairs + team * A.g + grp[j]] / m; }
#pragma unroll
                for (int k = 0; k < K; k++)
                    if (k * R + t < count) {
                        Pack<T, VEC> dx;
#pragma unroll
                        for (int j = 0; j < VEC; j++) {
                            const int s = GR ? 0 : j;
                            const float xh = hat(k, j);
                            const float dz = sizeof(T) == 4 && PH != APPLY ? to_f(rd[k].v[j])
                                                                           : act_bwd(decltype(act)::value, fmaf(xh, w[j], b[j]), to_f(rd[k].v[j]));
                            dx.v[j] = from_f<T>(rstd[s] * (fmaf(dz, w[j], -a1[s]) - xh * a2[s]));
                        }
                        reinterpret_cast<Pack<T, VEC>*>(A.dx)[n * nvec + v0 + k * R + t] = dx;
                    }
            }
            if (PH == WHOLE && parts > 1) cg::this_cluster().barrier_wait();   // before part is written again
        };
        if (A.act == FME_ACT_SILU) value(cuda_int<FME_ACT_SILU>{});
        else if (A.act == FME_ACT_RELU) value(cuda_int<FME_ACT_RELU>{});
        else value(cuda_int<FME_ACT_NONE>{});
        __syncthreads();   // out and red are written again
    }
    if (PH == APPLY || !A.dw) return;
    // dw and db of this CTA: slots c, c + C, ... hold channel c
    float* rw = sm;
    const int slots = R * M * VEC;
    if (mine) {
#pragma unroll
        for (int j = 0; j < VEC; j++) { rw[threadIdx.x * VEC + j] = dw[j]; rw[slots + threadIdx.x * VEC + j] = db[j]; }
    }
    __syncthreads();
    float* row = (float*)A.ws + (PH == STATS ? 2 * ((int64_t)A.n * parts * A.g + (int64_t)A.n * A.g) : 0) + (int64_t)blockIdx.x * 2 * A.c;
    for (int i = threadIdx.x; i < 2 * A.c; i += blockDim.x) {
        const float* src = rw + (i < A.c ? i : slots + i - A.c);
        float s = 0.f;
        for (int k = 0; k < slots; k += A.c) s += src[k];
        row[i] = s;
    }
}

__global__ void __launch_bounds__(NT) k_norm_join_bwd(const FmeGroupNorm A, const int parts) {
    const int64_t i = (int64_t)blockIdx.x * (NT / 32) + (threadIdx.x >> 5);
    const int lane = threadIdx.x & 31;
    if (i >= (int64_t)A.n * A.g) return;
    const int64_t n = i / A.g;
    const int g = (int)(i % A.g);
    float2 s = make_float2(0.f, 0.f);
    const float2* src = reinterpret_cast<const float2*>(A.ws);
    for (int r = lane; r < parts; r += 32) { const float2 f = src[(n * parts + r) * A.g + g]; s.x += f.x; s.y += f.y; }
    for (int o = 16; o > 0; o >>= 1) { s.x += __shfl_xor_sync(0xffffffffu, s.x, o); s.y += __shfl_xor_sync(0xffffffffu, s.y, o); }
    if (lane == 0) reinterpret_cast<float2*>(A.ws)[(int64_t)A.n * parts * A.g + i] = s;
}

// ---------------------------------------------------------------- many channels of an odd number
// Channel counts whose vectors repeat only after more than MAX_R threads (odd ones above 512, mostly): one thread a channel,
// x read three times. One CTA walks samples blockIdx.x, + gridDim.x, ...; per-channel sums in shared memory, one thread a channel.
template <typename T> __global__ void __launch_bounds__(NT) k_norm_wide_fwd(const FmeGroupNorm A) {
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
                ((T*)A.y)[base + p * A.c + c] = from_f<T>(act_fwd(A.act, fmaf((to_f(x[p * A.c + c]) - s0[c]) * s2[c], w, b)));
        }
        __syncthreads();
    }
}

template <typename T> __device__ __forceinline__ float x_of(const FmeGroupNorm& A, int64_t n, int64_t i, float lo, float step) {
    if (A.codes) return __fadd_rn(lo, __fmul_rn((float)A.codes[n * (int64_t)A.p * A.c + i], step));
    return to_f(((const T*)A.x)[n * A.x_sn + i]);
}

// As the forward kernel; a CTA's sums of dw and db over its samples go to its row of the workspace.
template <typename T> __global__ void __launch_bounds__(NT) k_norm_wide_bwd(const FmeGroupNorm A) {
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
                    const float dz = act_bwd(A.act, fmaf(xh, w, b), to_f(dy[i]));
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

// Columns of the CTAs' dw and db rows, summed in a fixed order: 32 columns a CTA, 32 threads a column.
__global__ void __launch_bounds__(1024) k_norm_params(const float* __restrict__ ws, int rows, int c, float* dw, float* db) {
    __shared__ float sm[32][33];
    const int i = blockIdx.x * 32 + threadIdx.x;
    float s = 0.f;
    if (i < 2 * c)
        for (int r = threadIdx.y; r < rows; r += 32) s += ws[(int64_t)r * 2 * c + i];
    sm[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = sm[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int col = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < 2 * c) (col < c ? dw[col] : db[col - c]) = s;
}

// ---------------------------------------------------------------- host side
constexpr int SMS = 148, MAX_R = 512;

int bad(const char* msg) { return host_fail(FME_E_ARG, msg); }
int check_sizes(const FmeGroupNorm* a) {
    if (!a) return bad("null group norm arguments");
    if (a->n < 0 || a->p < 0 || a->c < 1 || a->g < 1 || a->c % a->g) return bad("group norm: sizes must be >= 0 and g must divide c");
    if (a->c > MAX_C) return bad("group norm: c must be at most 4096");
    if ((int64_t)a->p * a->c > 0x7fffffff) return bad("group norm: a sample must have fewer than 2^31 values");
    if (a->dtype != FME_F32 && a->dtype != FME_BF16) return bad("group norm: dtype must be FME_F32 or FME_BF16");
    if (a->act < FME_ACT_NONE || a->act > FME_ACT_SILU) return bad("group norm: unknown activation");
    return FME_OK;
}
int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

// How a call is laid out. false: the kernels for many channels of an odd number.
bool make_plan(const FmeGroupNorm& a, bool bwd, Plan* P) {
    const int e = a.dtype == FME_F32 ? 4 : 2, full = 16 / e;
    const int64_t S = (int64_t)a.p * a.c;
    auto al = [&](const void* p, int64_t sn) { return !((uintptr_t)p & 15) && !((sn * e) & 15); };
    const bool wide = S % full == 0 && (bwd ? al(a.dy, a.dy_sn) && al(a.dx, 0) && (a.codes || al(a.x, a.x_sn)) : al(a.x, a.x_sn) && al(a.y, 0)) &&
                      !((uintptr_t)a.codes & 7);
    P->vec = wide ? full : 1;
    P->gr = (a.c / a.g) % P->vec == 0;
    const int per = a.c / gcd(a.c, P->vec);            // threads after which a vector's channels repeat
    if (per > MAX_R) return false;
    const int64_t nvec = S / P->vec;
    auto up = [&](int64_t x) { return (int)((x + per - 1) / per * per); };
    const int cap = MAX_R / per * per;                 // threads of a team at most
    P->parts = 1;
    P->cluster = false;
    P->M = 1;
    P->K = nvec <= 2 * (int64_t)cap ? 2 : nvec <= 4 * (int64_t)cap ? 4 : 8;
    if (nvec > 4 * (int64_t)cap) {
        int parts = 1;
        while (parts < 16 && nvec > (int64_t)parts * cap * 4) parts *= 2;
        P->K = nvec <= (int64_t)parts * cap * 4 ? 4 : 8;
        const bool fits = nvec <= (int64_t)parts * cap * 8;
        if (fits) { P->cluster = true; P->parts = parts; }
        else P->parts = (int)((nvec + cap * 8 - 1) / (cap * 8));
    }
    P->R = up((nvec + (int64_t)P->parts * P->K - 1) / ((int64_t)P->parts * P->K));
    if (P->R > cap) P->R = cap;
    if (P->R < 1) P->R = per;
    if (P->parts == 1 && P->R <= 128) {
        P->M = 256 / P->R;
        if (P->M > a.n) P->M = a.n > 0 ? a.n : 1;
    }
    P->threads = (P->R * P->M + 31) / 32 * 32;
    const int64_t groups = ((int64_t)a.n + P->M - 1) / P->M;
    const int ns = P->gr ? 1 : P->vec, pairs = P->M * a.g;
    if (bwd) {
        P->smem = 4 * ((size_t)2 * P->R * P->M * P->vec + 4 * (size_t)pairs);
        const bool walk = P->parts == 1 || P->cluster;
        const int64_t most = walk ? (int64_t)SMS * (1536 / P->threads > 8 ? 8 : 1536 / P->threads) / P->parts : groups;
        P->grid = (int)((groups < most ? groups : most) * P->parts);
    } else {
        P->smem = 4 * ((size_t)3 * P->R * P->M * ns + 8 * (size_t)pairs);
        P->grid = (int)(groups * P->parts);
    }
    return groups * P->parts <= 0x7fffffff;
}

template <typename... Args>
int launch(const char* what, void (*kernel)(Args...), const Plan& P, cudaStream_t st, std::common_type_t<Args>... args) {
    if (P.smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)P.smem);
    cudaLaunchConfig_t c{};
    c.gridDim = P.grid; c.blockDim = P.threads; c.dynamicSmemBytes = P.smem; c.stream = st;
    cudaLaunchAttribute at{};
    if (P.cluster) {
        if (P.parts > 8) cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        at.id = cudaLaunchAttributeClusterDimension;
        at.val.clusterDim.x = P.parts; at.val.clusterDim.y = at.val.clusterDim.z = 1;
        c.attrs = &at; c.numAttrs = 1;
    }
    cudaLaunchKernelEx(&c, kernel, args...);
    return launch_status(what);
}

template <typename T, int VEC, bool GR> int run_fwd(const FmeGroupNorm& a, const Plan& P, cudaStream_t st) {
    const char* what = "fme_group_norm_fwd";
    if (P.parts == 1 || P.cluster) {
        if (P.K == 2) return launch(what, k_norm_fwd<T, VEC, 2, GR, WHOLE>, P, st, a, P.R, P.M, P.parts);
        if (P.K == 4) return launch(what, k_norm_fwd<T, VEC, 4, GR, WHOLE>, P, st, a, P.R, P.M, P.parts);
        return launch(what, k_norm_fwd<T, VEC, 8, GR, WHOLE>, P, st, a, P.R, P.M, P.parts);
    }
    int rc = launch(what, k_norm_fwd<T, VEC, 8, GR, STATS>, P, st, a, P.R, P.M, P.parts);
    if (rc) return rc;
    k_norm_join_fwd<T, VEC><<<(int)(((int64_t)a.n * a.g + NT / 32 - 1) / (NT / 32)), NT, 0, st>>>(a, P.parts, P.R * P.K);
    if ((rc = launch_status(what))) return rc;
    return launch(what, k_norm_fwd<T, VEC, 8, GR, APPLY>, P, st, a, P.R, P.M, P.parts);
}
template <typename T, int VEC, bool GR, bool U8> int run_bwd(const FmeGroupNorm& a, const Plan& P, cudaStream_t st) {
    const char* what = "fme_group_norm_bwd";
    if (P.parts == 1 || P.cluster) {
        if (P.K == 2) return launch(what, k_norm_bwd<T, VEC, 2, GR, WHOLE, U8>, P, st, a, P.R, P.M, P.parts);
        if (P.K == 4) return launch(what, k_norm_bwd<T, VEC, 4, GR, WHOLE, U8>, P, st, a, P.R, P.M, P.parts);
        return launch(what, k_norm_bwd<T, VEC, 8, GR, WHOLE, U8>, P, st, a, P.R, P.M, P.parts);
    }
    int rc = launch(what, k_norm_bwd<T, VEC, 8, GR, STATS, U8>, P, st, a, P.R, P.M, P.parts);
    if (rc) return rc;
    k_norm_join_bwd<<<(int)(((int64_t)a.n * a.g + NT / 32 - 1) / (NT / 32)), NT, 0, st>>>(a, P.parts);
    if ((rc = launch_status(what))) return rc;
    return launch(what, k_norm_bwd<T, VEC, 8, GR, APPLY, U8>, P, st, a, P.R, P.M, P.parts);
}

constexpr int WIDE_GRID = 592;
bool split(const Plan& P) { return P.parts > 1 && !P.cluster; }
// floats of the workspace before the CTAs' rows of dw and db
int64_t split_floats(const FmeGroupNorm& a, const Plan& P, int each) { return split(P) ? (int64_t)each * ((int64_t)a.n * P.parts * a.g + (int64_t)a.n * a.g) : 0; }

}  // namespace
}  // namespace fme

using namespace fme;

extern "C" {

int64_t fme_group_norm_bytes(const FmeGroupNorm* a, int32_t which) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (which < 0 || which > 1) return bad("group norm: which must be 0 or 1");
    Plan P;
    const bool planned = make_plan(*a, which == 1, &P);
    if (which == 0) return planned ? 4 * split_floats(*a, P, 4) : 0;
    return 4 * ((planned ? split_floats(*a, P, 2) : 0) + (int64_t)(planned ? P.grid : WIDE_GRID) * 2 * a->c);
}

int fme_group_norm_fwd(const FmeGroupNorm* a, void* stream) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (a->n == 0 || a->p == 0) return FME_OK;
    if (!a->x || !a->y) return bad("group norm: x and y are required");
    if (a->codes && (!a->lo || !a->hi)) return bad("group norm: codes need lo and hi");
    if ((a->mean == nullptr) != (a->rstd == nullptr)) return bad("group norm: mean and rstd come together");
    if (const int64_t need = fme_group_norm_bytes(a, 0); need > 0 && (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < need))
        return bad("group norm: workspace too small or not aligned");
    cudaStream_t st = (cudaStream_t)stream;
    Plan P;
    if (!make_plan(*a, false, &P)) {
        const size_t smem = (size_t)3 * a->c * 4;
        const int grid = a->n < WIDE_GRID ? a->n : WIDE_GRID;
        if (a->dtype == FME_F32) k_norm_wide_fwd<float><<<grid, NT, smem, st>>>(*a);
        else k_norm_wide_fwd<__nv_bfloat16><<<grid, NT, smem, st>>>(*a);
        return launch_status("fme_group_norm_fwd");
    }
    if (a->dtype == FME_F32) {
        if (P.vec == 1) return run_fwd<float, 1, true>(*a, P, st);
        return P.gr ? run_fwd<float, 4, true>(*a, P, st) : run_fwd<float, 4, false>(*a, P, st);
    }
    if (P.vec == 1) return run_fwd<__nv_bfloat16, 1, true>(*a, P, st);
    return P.gr ? run_fwd<__nv_bfloat16, 8, true>(*a, P, st) : run_fwd<__nv_bfloat16, 8, false>(*a, P, st);
}

int fme_group_norm_bwd(const FmeGroupNorm* a, void* stream) {
    int rc = check_sizes(a);
    if (rc) return rc;
    if ((a->dw == nullptr) != (a->db == nullptr)) return bad("group norm: dw and db come together");
    cudaStream_t st = (cudaStream_t)stream;
    if (a->n == 0 || a->p == 0) {
        if (a->dw) {
            if (cudaMemsetAsync(a->dw, 0, 4 * (size_t)a->c, st) != cudaSuccess || cudaMemsetAsync(a->db, 0, 4 * (size_t)a->c, st) != cudaSuccess)
                return launch_status("fme_group_norm_bwd");
        }
        return FME_OK;
    }
    if ((!a->x && !a->codes) || !a->dy || !a->dx || !a->mean || !a->rstd) return bad("group norm: x or codes, dy, dx, mean and rstd are required");
    if (a->codes && (!a->lo || !a->hi)) return bad("group norm: codes need lo and hi");
    if (!a->ws || ((uintptr_t)a->ws & 15) || a->ws_bytes < fme_group_norm_bytes(a, 1)) return bad("group norm: workspace too small or not aligned");
    Plan P;
    int rows = a->n < WIDE_GRID ? a->n : WIDE_GRID;
    int64_t skip = 0;
    if (!make_plan(*a, true, &P)) {
        const size_t smem = (size_t)4 * a->c * 4;
        auto kernel = a->dtype == FME_F32 ? k_norm_wide_bwd<float> : k_norm_wide_bwd<__nv_bfloat16>;
        if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        kernel<<<rows, NT, smem, st>>>(*a);
        rc = launch_status("fme_group_norm_bwd");
    } else {
        rows = P.grid;
        skip = split_floats(*a, P, 2);
        const bool u8 = a->codes != nullptr;
        if (a->dtype == FME_F32) {
            if (P.vec == 1) rc = u8 ? run_bwd<float, 1, true, true>(*a, P, st) : run_bwd<float, 1, true, false>(*a, P, st);
            else if (P.gr) rc = u8 ? run_bwd<float, 4, true, true>(*a, P, st) : run_bwd<float, 4, true, false>(*a, P, st);
            else rc = u8 ? run_bwd<float, 4, false, true>(*a, P, st) : run_bwd<float, 4, false, false>(*a, P, st);
        } else {
            if (P.vec == 1) rc = u8 ? run_bwd<__nv_bfloat16, 1, true, true>(*a, P, st) : run_bwd<__nv_bfloat16, 1, true, false>(*a, P, st);
            else if (P.gr) rc = u8 ? run_bwd<__nv_bfloat16, 8, true, true>(*a, P, st) : run_bwd<__nv_bfloat16, 8, true, false>(*a, P, st);
            else rc = u8 ? run_bwd<__nv_bfloat16, 8, false, true>(*a, P, st) : run_bwd<__nv_bfloat16, 8, false, false>(*a, P, st);
        }
    }
    if (rc || !a->dw) return rc;
    k_norm_params<<<(2 * a->c + 31) / 32, dim3(32, 32), 0, st>>>((const float*)a->ws + skip, rows, a->c, a->dw, a->db);
    return launch_status("fme_group_norm_bwd");
}

}  // extern "C"

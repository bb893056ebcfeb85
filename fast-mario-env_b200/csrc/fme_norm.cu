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

// 1 / (1 + 2^(-z log2 e)) by the approximate exponential and reciprocal, each off by a few units of 2^-23. The product with log2 e is
// rounded before it is an exponent, so the result's relative error grows for negative z, as |z| 2^-24 (of z times it: less than
// 2^-24 in all, since z^2 e^z < 0.6). Both of +-inf come out as limits (2^inf = inf, 1 / inf = 0).
__device__ __forceinline__ float sigmoid(float z) {
    float e, r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(z * -1.44269504088896340736f));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
    return r;
}
__device__ __forceinline__ float act_fwd(int act, float z) {
    return act == FME_ACT_SILU ? z * sigmoid(z) : act == FME_ACT_RELU ? (z < 0.f ? 0.f : z) : z;
}
__device__ __forceinline__ float act_bwd(int act, float z, float dy) {
    // s (1 + z (1 - s)). The form s ((1 + z) - z s) loses the 1 from z = 2^24 on, and digits of it before
    if (act == FME_ACT_SILU) { const float s = sigmoid(z); return dy * (s * fmaf(z, 1.f - s, 1.f)); }
    return act == FME_ACT_RELU ? (z <= 0.f ? 0.f : dy) : dy;
}

constexpr int NT = 256;
constexpr int MAX_C = 4096;

// A vector of VEC values as the words that it is loaded in: values are taken out of registers, not out of memory
template <int BYTES> struct Words;
template <> struct Words<16> { using type = uint4; };
template <> struct Words<8> { using type = uint2; };
template <> struct Words<4> { using type = uint32_t; };
template <> struct Words<2> { using type = uint16_t; };
template <> struct Words<1> { using type = uint8_t; };
template <typename T, int VEC> using Pack = typename Words<(int)sizeof(T) * VEC>::type;
__device__ __forceinline__ uint32_t word(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }
__device__ __forceinline__ uint32_t word(const uint2& v, int i) { return i ? v.y : v.x; }
__device__ __forceinline__ uint32_t word(uint32_t v, int) { return v; }
__device__ __forceinline__ void set_word(uint4& v, int i, uint32_t x) { (i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w) = x; }
__device__ __forceinline__ void set_word(uint2& v, int i, uint32_t x) { (i ? v.y : v.x) = x; }
__device__ __forceinline__ void set_word(uint32_t& v, int, uint32_t x) { v = x; }

// Codes by the float32 that is 2^23 + code: adding 2^23 rounds to the nearest integer, ties to even, and leaves it in the low
// byte. Conversions between float and integer go at a quarter of that rate. (A group with NaN gets some code.)
__device__ __forceinline__ uint32_t code_of(float x, float lo, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(__fsub_rn(x, lo), inv), 8388608.f)); }
template <int VEC> __device__ __forceinline__ Pack<uint8_t, VEC> codes_of(const float (&x)[VEC], const float* lo, const float* inv, bool each) {
    Pack<uint8_t, VEC> q;
    if constexpr (VEC % 4 == 0) {
#pragma unroll
        for (int j = 0; j < VEC; j += 4) {
            uint32_t c[4];
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = code_of(x[j + i], lo[each ? j + i : 0], inv[each ? j + i : 0]);
            set_word(q, j / 4, __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410));
        }
    } else {
        static_assert(VEC == 1, "");
        q = (uint8_t)code_of(x[0], lo[0], inv[0]);
    }
    return q;
}
// The values of a vector as float32
template <typename T, int VEC> __device__ __forceinline__ void floats(float (&f)[VEC], const Pack<T, VEC>& r) {
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 1) f[0] = (float)r;
        else if constexpr (sizeof(T) == 2) f[0] = __uint_as_float((uint32_t)r << 16);
        else f[0] = __uint_as_float(r);
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            if constexpr (sizeof(T) == 1) f[j] = __uint_as_float(__byte_perm(word(r, j / 4), 0x4b000000u, 0x7540 + (j & 3))) - 8388608.f;
            else if constexpr (sizeof(T) == 2) f[j] = __uint_as_float(j & 1 ? word(r, j / 2) & 0xffff0000u : word(r, j / 2) << 16);
            else f[j] = __uint_as_float(word(r, j));
        }
    }
}
template <typename T, int VEC> __device__ __forceinline__ Pack<T, VEC> packed(const float (&f)[VEC]) {
    Pack<T, VEC> r;
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 2) r = __bfloat16_as_ushort(__float2bfloat16(f[0]));
        else r = __float_as_uint(f[0]);
    } else if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int j = 0; j < VEC; j += 2) {
            const __nv_bfloat162 two = __floats2bfloat162_rn(f[j], f[j + 1]);
            set_word(r, j / 2, *reinterpret_cast<const uint32_t*>(&two));
        }
    } else {
#pragma unroll
        for (int j = 0; j < VEC; j++) set_word(r, j, __float_as_uint(f[j]));
    }
    return r;
}

// ---------------------------------------------------------------- samples held in shared memory
// A sample is p * c values in a row. Threads take vectors of VEC of them, R threads form a team and R * VEC is a multiple of
// c, so that a thread meets the same channels in each of its vectors and keeps their weights (and, backward, their dw and db)
// in registers. Each thread copies its own vectors to shared memory (asynchronously, without registers) and reads them from
// there in every pass, so that x (and dy) come from HBM once, which is the bound: some 50 KB a CTA, four CTAs an SM, of which
// some load while others compute. Small samples: M teams in a CTA, a sample each. Large ones: the CTAs of a cluster share a
// sample and add up their sums through distributed shared memory. Where no cluster can hold a sample its pieces are separate
// CTAs, and the kernel runs twice, for the sums (STATS) and, after k_norm_join*, for the values (APPLY), with a second read.
// Measured on a B200 (HBM copy 6441 GB/s), forward + backward + sums of dw and db: 1024 x 20 x 20 x 32 fp32 21 + 35 + 8 us (4.9 and
// 4.5 TB/s); 8192 x 9 x 9 x 64 fp32 with codes 67 + 80 + 10 us (5.7 and 4.8 TB/s), bound by issue slots (65 to 72 % used: 50
// instructions a value); 37 x 84 x 84 x 48 bf16 with codes, clusters of 16: 31 + 50 + 7 us, of it 10 + 10 for HBM, bound by the sigmoid (two
// exponentials and two reciprocals a value backward) and by clusters waiting for their last CTA.
// How a group's sums are found: EACH: a vector's values may belong to several groups (VEC does not divide c / g); ONE: to one
// group; WARP: to one, and the c / VEC vectors of a pixel are a power of two up to 32, so that shuffles do most of it.
enum Phase { WHOLE, STATS, APPLY };
enum How { EACH, ONE, WARP };

struct Div {   // x / d for x < 2^16, d <= 2^12
    uint32_t d, m;
    __device__ __forceinline__ int operator()(int x) const { return d == 1 ? x : (int)__umulhi((uint32_t)x, m); }
    __device__ __forceinline__ int mod(int x) const { return x - (*this)(x) * (int)d; }
};

struct Plan {
    int R, M, vec, parts;      // parts: CTAs that share a sample
    int chunk, nvec;           // vectors of a part at most, of a sample
    int how;
    bool cluster;
    int L, gl, rows;           // what is summed over a group stands at row * L + g * gl + 0..gl-1
    Div by_r, by_c, by_cg, by_gl, by_g;
    int threads, grid;
    int tile;                  // bytes of a team's vectors
    size_t smem;
};

// Sums (MM: the second and third value's minimum and maximum) over each (team, group), in a fixed order. red: room for NV *
// threads * NS values, twice that for WARP, which alternates between halves (buf) and so needs one barrier. The result of the
// thread's own group(s) in v; in out[i * pairs + pair] as well, for EACH and ONE, and for WARP from the team's first warp
// (without a barrier after it).
template <int NV, int NS, int HOW, bool MM>
__device__ __forceinline__ void group_sums(const Plan& P, int G, float (&v)[NV][NS], const int (&grp)[NS], int team, int t, float* red, float* out, int buf) {
    auto join = [](int i, float x, float y) { return !MM || i == 0 ? x + y : i == 1 ? fminf(x, y) : fmaxf(x, y); };
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, pairs = P.M * G;
    if (HOW == WARP) {
        for (int o = 16; o >= P.L; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; i++) v[i][0] = join(i, v[i][0], __shfl_xor_sync(0xffffffffu, v[i][0], o));
        for (int o = P.gl >> 1; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; i++) v[i][0] = join(i, v[i][0], __shfl_xor_sync(0xffffffffu, v[i][0], o));
        const int warps = blockDim.x >> 5, g = P.by_gl(lane & (P.L - 1));
        float* mine = red + buf * NV * warps * G;
        if (lane < P.L && (lane & (P.gl - 1)) == 0) {
#pragma unroll
            for (int i = 0; i < NV; i++) mine[(i * warps + warp) * G + g] = v[i][0];
        }
        __syncthreads();
        const int per = P.M == 1 ? warps : P.R >> 5, w0 = P.M == 1 ? 0 : team * per;   // M > 1: a team is whole warps
#pragma unroll
        for (int i = 0; i < NV; i++) {
            const float* src = mine + (i * warps + min(w0, warps - per)) * G + g;
            float x = src[0];
            for (int w = 1; w < per; w++) x = join(i, x, src[w * G]);
            v[i][0] = x;
        }
        if (t < P.L && (t & (P.gl - 1)) == 0 && team < P.M) {
#pragma unroll
            for (int i = 0; i < NV; i++) out[i * pairs + team * G + g] = v[i][0];
        }
        return;
    }
    const int n = P.R * P.M * NS, members = P.rows * P.gl;
    __syncthreads();
    if (team < P.M) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < NS; j++) red[i * n + threadIdx.x * NS + j] = v[i][j];
    }
    __syncthreads();
    for (int pair = warp; pair < pairs; pair += blockDim.x >> 5) {
        const int tm = P.by_g(pair), base = tm * P.R * NS + (pair - tm * G) * P.gl;
        float a[NV];
#pragma unroll
        for (int i = 0; i < NV; i++) a[i] = !MM || i == 0 ? 0.f : i == 1 ? INFINITY : -INFINITY;
        for (int m = lane; m < members; m += 32) {
            const int row = P.by_gl(m), at = base + row * P.L + (m - row * P.gl);
#pragma unroll
            for (int i = 0; i < NV; i++) a[i] = join(i, a[i], red[i * n + at]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1)
#pragma unroll
            for (int i = 0; i < NV; i++) a[i] = join(i, a[i], __shfl_xor_sync(0xffffffffu, a[i], o));
        if (lane == 0) {
#pragma unroll
            for (int i = 0; i < NV; i++) out[i * pairs + pair] = a[i];
        }
    }
    __syncthreads();
    if (team < P.M) {
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int j = 0; j < NS; j++) v[i][j] = out[i * pairs + team * G + grp[j]];
    }
}

// mean and squared distances of several parts
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

__device__ __forceinline__ float rstd_of(float m2, float m, float eps) { return rsqrtf(m2 / m + eps); }
__device__ __forceinline__ float code_inv(float lo, float hi) { return hi > lo ? __fmul_rn(__frcp_rn(__fsub_rn(hi, lo)), 255.f) : 0.f; }
__device__ __forceinline__ float code_step(float lo, float hi) { return __fdiv_rn(__fsub_rn(hi, lo), 255.f); }

// a thread's vector to its place in shared memory; BYTES 16, 8 or 4 asynchronously
template <typename V> __device__ __forceinline__ void fetch(V* dst, const V* src) {
    constexpr int B = sizeof(V);
    if constexpr (B == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
    else if constexpr (B == 8 || B == 4) asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "n"(B) : "memory");
    else *dst = *src;
}
__device__ __forceinline__ void fetched() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// values of each group in part r: parts begin and end with whole pixels
__device__ __forceinline__ int part_vecs(const Plan& P, int r) { return max(0, min(P.nvec - r * P.chunk, P.chunk)); }

template <int ACT> struct act_is { static constexpr int value = ACT; };
template <typename F> __device__ __forceinline__ void by_act(int act, F f) {
    if (act == FME_ACT_SILU) f(act_is<FME_ACT_SILU>{});
    else if (act == FME_ACT_RELU) f(act_is<FME_ACT_RELU>{});
    else f(act_is<FME_ACT_NONE>{});
}

constexpr int MAX_THREADS = 512;

template <typename T, int VEC, int HOW, int PH>
__global__ void __launch_bounds__(MAX_THREADS, 2) k_norm_fwd(const FmeGroupNorm A, const __grid_constant__ Plan P) {
    constexpr int NS = HOW == EACH ? VEC : 1;
    using V = Pack<T, VEC>;
    extern __shared__ __align__(16) char sm[];
    const int pairs = P.M * A.g, team = P.M == 1 ? (threadIdx.x < P.R ? 0 : 1) : P.by_r(threadIdx.x), t = threadIdx.x - team * P.R;
    V* tile = reinterpret_cast<V*>(sm + team * P.tile);                // only for team < M
    float* out = reinterpret_cast<float*>(sm + (size_t)P.M * P.tile);  // sum, lo, hi: 3 * pairs; squared distances: pairs
    float* part = out + 4 * pairs;                                     // 4 * pairs
    float* red = part + 4 * pairs;
    const int rank = P.parts == 1 ? 0 : blockIdx.x % P.parts, block = P.parts == 1 ? blockIdx.x : blockIdx.x / P.parts;
    const int64_t n = (int64_t)block * P.M + team;
    const bool ok = team < P.M && n < A.n;
    const int v0 = rank * P.chunk, count = ok ? part_vecs(P, rank) : 0;
    const V* x = reinterpret_cast<const V*>((const T*)A.x + n * A.x_sn) + v0;
    for (int i = t; i < count; i += P.R) fetch(tile + i, x + i);
    int ch[VEC], grp[NS];
    float w[VEC], b[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        ch[j] = P.by_c.mod(t * VEC + j);
        w[j] = PH != STATS && A.w ? __ldg(A.w + ch[j]) : 1.f;
        b[j] = PH != STATS && A.b ? __ldg(A.b + ch[j]) : 0.f;
    }
#pragma unroll
    for (int j = 0; j < NS; j++) grp[j] = P.by_cg(ch[j]);
    const bool u8 = A.codes != nullptr;
    const float per_vec = (float)VEC / (float)A.g, cnt = (float)part_vecs(P, rank) * per_vec, m = (float)P.nvec * per_vec;
    float mean[NS], rstd[NS], lo[NS], hi[NS];
    fetched();
    if (PH != APPLY) {
        float v[3][NS], q[1][NS];
#pragma unroll
        for (int j = 0; j < NS; j++) { v[0][j] = 0.f; v[1][j] = INFINITY; v[2][j] = -INFINITY; q[0][j] = 0.f; }
        if (u8) {
#pragma unroll 4
            for (int i = t; i < count; i += P.R) {
                float f[VEC];
                const V r = tile[i];   // in one piece
                floats<T, VEC>(f, r);
#pragma unroll
                for (int j = 0; j < VEC; j++) {
                    const int s = NS == 1 ? 0 : j;
                    v[0][s] += f[j]; v[1][s] = fminf(v[1][s], f[j]); v[2][s] = fmaxf(v[2][s], f[j]);
                }
            }
            group_sums<3, NS, HOW, true>(P, A.g, v, grp, team, t, red, out, 0);
        } else {
            float s1[1][NS];
#pragma unroll
            for (int j = 0; j < NS; j++) s1[0][j] = 0.f;
#pragma unroll 4
            for (int i = t; i < count; i += P.R) {
                float f[VEC];
                const V r = tile[i];   // in one piece
                floats<T, VEC>(f, r);
#pragma unroll
                for (int j = 0; j < VEC; j++) s1[0][NS == 1 ? 0 : j] += f[j];
            }
            group_sums<1, NS, HOW, false>(P, A.g, s1, grp, team, t, red, out, 0);
#pragma unroll
            for (int j = 0; j < NS; j++) v[0][j] = s1[0][j];
        }
#pragma unroll
        for (int j = 0; j < NS; j++) { mean[j] = cnt > 0.f ? v[0][j] / cnt : 0.f; lo[j] = v[1][j]; hi[j] = v[2][j]; }
#pragma unroll 4
        for (int i = t; i < count; i += P.R) {
            float f[VEC];
            const V r = tile[i];
            floats<T, VEC>(f, r);
#pragma unroll
            for (int j = 0; j < VEC; j++) { const int s = NS == 1 ? 0 : j; const float d = f[j] - mean[s]; q[0][s] = fmaf(d, d, q[0][s]); }
        }
        // 3 * warps * g floats on: past what the first sums used
        group_sums<1, NS, HOW, false>(P, A.g, q, grp, team, t, HOW == WARP ? red + 3 * (blockDim.x >> 5) * A.g : red, out + 3 * pairs, 0);
#pragma unroll
        for (int j = 0; j < NS; j++) rstd[j] = rstd_of(q[0][j], m, A.eps);
        if (PH == STATS || P.parts > 1) __syncthreads();   // out, for other threads
    }
    if (PH == STATS) {                     // (sample, part, group): mean, squared distances, lo, hi; M is 1
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            float4* dst = reinterpret_cast<float4*>(A.ws) + ((int64_t)block * P.parts + rank) * A.g + i;
            *dst = make_float4(cnt > 0.f ? out[i] / cnt : 0.f, out[3 * pairs + i], u8 ? out[pairs + i] : 0.f, u8 ? out[2 * pairs + i] : 0.f);
        }
        return;
    }
    if (PH == WHOLE && P.parts > 1) {
        cg::cluster_group cl = cg::this_cluster();
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            part[i] = cnt > 0.f ? out[i] / cnt : 0.f; part[pairs + i] = out[3 * pairs + i];
            if (u8) { part[2 * pairs + i] = out[pairs + i]; part[3 * pairs + i] = out[2 * pairs + i]; }
        }
        cl.sync();
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            Moments mo;
            float l = INFINITY, h = -INFINITY;
            for (int r = 0; r < P.parts; r++) {
                const float* o = cl.map_shared_rank(part, r);
                mo.add((float)part_vecs(P, r) * per_vec, o[i], o[pairs + i]);
                if (u8) { l = fminf(l, o[2 * pairs + i]); h = fmaxf(h, o[3 * pairs + i]); }
            }
            out[i] = mo.mean; out[3 * pairs + i] = rstd_of(mo.m2, m, A.eps);
            out[pairs + i] = l; out[2 * pairs + i] = h;
        }
        cl.barrier_arrive();   // this CTA has read the others; it ends only when they have read it
        __syncthreads();
    }
    if (PH == APPLY) {
        for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
            const float4 f = reinterpret_cast<const float4*>(A.ws)[(int64_t)A.n * P.parts * A.g + (int64_t)block * A.g + i];
            out[i] = f.x; out[3 * pairs + i] = f.y; out[pairs + i] = f.z; out[2 * pairs + i] = f.w;
        }
        __syncthreads();
    }
    if (ok) {
        if (PH == APPLY || P.parts > 1) {
#pragma unroll
            for (int j = 0; j < NS; j++) { mean[j] = out[grp[j]]; rstd[j] = out[3 * pairs + grp[j]]; lo[j] = out[pairs + grp[j]]; hi[j] = out[2 * pairs + grp[j]]; }
        }
        if (rank == 0 && A.mean && t < P.L * (NS == 1 ? 1 : A.g)) {   // a group's first thread; EACH: every value of the first pixels
#pragma unroll
            for (int j = 0; j < NS; j++) {
                const int64_t ng = n * A.g + grp[j];
                const bool first = NS == 1 ? t == grp[j] * P.gl : t * VEC + j == grp[j] * P.gl;
                if (first) {
                    A.mean[ng] = mean[j]; A.rstd[ng] = rstd[j];
                    if (u8) { A.lo[ng] = lo[j]; A.hi[ng] = hi[j]; }
                }
            }
        }
        V* y = reinterpret_cast<V*>(A.y) + n * P.nvec + v0;
        Pack<uint8_t, VEC>* codes = reinterpret_cast<Pack<uint8_t, VEC>*>(A.codes) + n * P.nvec + v0;
        float inv[NS];
#pragma unroll
        for (int j = 0; j < NS; j++) inv[j] = u8 ? code_inv(lo[j], hi[j]) : 0.f;
        by_act(A.act, [&](auto act) {
            auto values = [&](auto with) {
#pragma unroll 2
                for (int i = t; i < count; i += P.R) {
                    float f[VEC], o[VEC];
                    const V r = tile[i];   // in one piece
                floats<T, VEC>(f, r);
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const int s = NS == 1 ? 0 : j;
                        o[j] = act_fwd(decltype(act)::value, fmaf((f[j] - mean[s]) * rstd[s], w[j], b[j]));
                    }
                    y[i] = packed<T, VEC>(o);
                    if (decltype(with)::value) codes[i] = codes_of<VEC>(f, lo, inv, NS > 1);
                }
            };
            if (u8) values(std::true_type{});
            else values(std::false_type{});
        });
    }
    if (PH == WHOLE && P.parts > 1) cg::this_cluster().barrier_wait();
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
// A CTA (or cluster) walks samples and keeps its channels' dw and db in registers until the end. fp32 keeps dz in dy's place in
// shared memory; bf16 would round it and computes it twice.
template <typename T, int VEC, int HOW, int PH, bool U8>
__global__ void __launch_bounds__(MAX_THREADS, 2) k_norm_bwd(const FmeGroupNorm A, const __grid_constant__ Plan P) {
    constexpr int NS = HOW == EACH ? VEC : 1;
    constexpr bool KEEP = sizeof(T) == 4 && PH != APPLY;
    using V = Pack<T, VEC>;
    using XT = typename std::conditional<U8, uint8_t, T>::type;
    using X = Pack<XT, VEC>;
    extern __shared__ __align__(16) char sm[];
    const int pairs = P.M * A.g, team = P.M == 1 ? (threadIdx.x < P.R ? 0 : 1) : P.by_r(threadIdx.x), t = threadIdx.x - team * P.R;
    V* td = reinterpret_cast<V*>(sm + team * P.tile);      // only for team < M
    X* tx = reinterpret_cast<X*>(td + P.chunk);
    float* out = reinterpret_cast<float*>(sm + (size_t)P.M * P.tile);   // 2 * pairs
    float* part = out + 2 * pairs;                                       // 2 * pairs
    float* red = part + 2 * pairs;
    const int rank = P.parts == 1 ? 0 : blockIdx.x % P.parts, block = P.parts == 1 ? blockIdx.x : blockIdx.x / P.parts;
    const int blocks = P.parts == 1 ? gridDim.x : gridDim.x / P.parts;
    const int v0 = rank * P.chunk, mine = team < P.M ? part_vecs(P, rank) : 0;
    const float inv_m = 1.f / ((float)P.nvec * ((float)VEC / (float)A.g));
    int ch[VEC], grp[NS];
    float w[VEC], b[VEC], dw[VEC], db[VEC];
#pragma unroll
    for (int j = 0; j < VEC; j++) {
        ch[j] = P.by_c.mod(t * VEC + j);
        w[j] = A.w ? __ldg(A.w + ch[j]) : 1.f;
        b[j] = A.b ? __ldg(A.b + ch[j]) : 0.f;
        dw[j] = db[j] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < NS; j++) grp[j] = P.by_cg(ch[j]);
    int buf = 0;
    for (int64_t n0 = (int64_t)block * P.M; n0 < A.n; n0 += (int64_t)blocks * P.M) {
        const int64_t n = n0 + team;
        const bool ok = team < P.M && n < A.n;
        const int count = ok ? mine : 0;
        const V* dy = reinterpret_cast<const V*>((const T*)A.dy + n * A.dy_sn) + v0;
        const X* x = U8 ? reinterpret_cast<const X*>(A.codes) + n * P.nvec + v0 : reinterpret_cast<const X*>((const T*)A.x + n * A.x_sn) + v0;
        for (int i = t; i < count; i += P.R) { fetch(tx + i, x + i); fetch(td + i, dy + i); }
        // x^ = (x - xb) xa; of codes: code * xa + xb
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
        auto hats = [&](float (&xh)[VEC], const X r) {
            floats<XT, VEC>(xh, r);
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int s = NS == 1 ? 0 : j;
                xh[j] = U8 ? fmaf(xh[j], xa[s], xb[s]) : (xh[j] - xb[s]) * xa[s];
            }
        };
        fetched();
        float v[2][NS];
        if (PH != APPLY) {
#pragma unroll
            for (int j = 0; j < NS; j++) v[0][j] = v[1][j] = 0.f;
            by_act(A.act, [&](auto act) {
#pragma unroll 2
                for (int i = t; i < count; i += P.R) {
                    float xh[VEC], dz[VEC];
                    const X r = tx[i];
                    const V g = td[i];
                    hats(xh, r);
                    floats<T, VEC>(dz, g);
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const int s = NS == 1 ? 0 : j;
                        dz[j] = act_bwd(decltype(act)::value, fmaf(xh[j], w[j], b[j]), dz[j]);
                        const float wd = w[j] * dz[j];
                        v[0][s] += wd; v[1][s] = fmaf(wd, xh[j], v[1][s]);
                        db[j] += dz[j]; dw[j] = fmaf(dz[j], xh[j], dw[j]);
                    }
                    if (KEEP && decltype(act)::value != FME_ACT_NONE) td[i] = packed<T, VEC>(dz);
                }
            });
            group_sums<2, NS, HOW, false>(P, A.g, v, grp, team, t, red, out, buf);
            buf ^= 1;
            if (PH == STATS || P.parts > 1) __syncthreads();
        }
        if (PH == STATS) {
            for (int i = threadIdx.x; i < pairs; i += blockDim.x)
                reinterpret_cast<float2*>(A.ws)[(n0 * P.parts + rank) * A.g + i] = make_float2(out[i], out[pairs + i]);
            break;   // one sample a CTA
        }
        if (PH == WHOLE && P.parts > 1) {
            cg::cluster_group cl = cg::this_cluster();
            for (int i = threadIdx.x; i < 2 * pairs; i += blockDim.x) part[i] = out[i];
            cl.sync();
            for (int i = threadIdx.x; i < 2 * pairs; i += blockDim.x) {
                float s = 0.f;
                for (int r = 0; r < P.parts; r++) s += cl.map_shared_rank(part, r)[i];
                out[i] = s;
            }
            cl.barrier_arrive();
            __syncthreads();
        }
        if (PH == APPLY) {
            for (int i = threadIdx.x; i < pairs; i += blockDim.x) {
                const float2 f = reinterpret_cast<const float2*>(A.ws)[(int64_t)A.n * P.parts * A.g + n0 * A.g + i];
                out[i] = f.x; out[pairs + i] = f.y;
            }
            __syncthreads();
        }
        if (ok) {
            float a1[NS], a2[NS];
#pragma unroll
            for (int j = 0; j < NS; j++) {
                a1[j] = inv_m * (PH == APPLY || P.parts > 1 ? out[team * A.g + grp[j]] : v[0][j]);
                a2[j] = inv_m * (PH == APPLY || P.parts > 1 ? out[pairs + team * A.g + grp[j]] : v[1][j]);
            }
            V* dx = reinterpret_cast<V*>(A.dx) + n * P.nvec + v0;
            by_act(A.act, [&](auto act) {
#pragma unroll 2
                for (int i = t; i < count; i += P.R) {
                    float xh[VEC], dz[VEC];
                    const X r = tx[i];
                    const V g = td[i];
                    hats(xh, r);
                    floats<T, VEC>(dz, g);
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const int s = NS == 1 ? 0 : j;
                        if (!KEEP) dz[j] = act_bwd(decltype(act)::value, fmaf(xh[j], w[j], b[j]), dz[j]);
                        dz[j] = rstd[s] * fmaf(-xh[j], a2[s], fmaf(dz[j], w[j], -a1[s]));
                    }
                    dx[i] = packed<T, VEC>(dz);
                }
            });
        }
        if (PH == WHOLE && P.parts > 1) cg::this_cluster().barrier_wait();   // before part is written again
        if (PH == APPLY) break;
    }
    if (PH == APPLY || !A.dw) return;
    // dw and db of this CTA: slots c, c + C, ... hold channel c
    let_next_start();
    __syncthreads();
    float* rw = reinterpret_cast<float*>(sm);
    const int slots = P.R * P.M * VEC;
    if (team < P.M) {
#pragma unroll
        for (int j = 0; j < VEC; j++) { rw[threadIdx.x * VEC + j] = dw[j]; rw[slots + threadIdx.x * VEC + j] = db[j]; }
    }
    __syncthreads();
    float* row = (float*)A.ws + (PH == STATS ? 2 * ((int64_t)A.n * P.parts * A.g + (int64_t)A.n * A.g) : 0) + (int64_t)blockIdx.x * 2 * A.c;
    for (int i = threadIdx.x; i < 2 * A.c; i += blockDim.x) {
        const float* src = rw + (i < A.c ? i : slots + i - A.c);
        float s = 0.f;
        for (int k = 0; k < slots; k += A.c) s += src[k];
        row[i] = s;
    }
}

// The parts' sums in order, to the end of the workspace
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

// ---------------------------------------------------------------- groups in a row
// p = 1 (tokens, heads): a (sample, group) is c / g values in a row, KV vectors for each of LG lanes of a warp. No shared
// memory and no barrier: shuffles. A lane keeps its channels over the samples that it walks, U of them on their way at a time, the
// next ones while these are computed; as many CTAs as the GPU holds (one more would run alone after them).
// 131072 rows of 8 heads of 64, bf16: forward 55 us (4.9 TB/s), backward 72 us (5.6 TB/s); through shared memory 113 + 282 us.
struct Rows {
    int LG, segs, tall;   // lanes of a group; groups of a CTA at once; samples of a CTA at once (0: the groups take grid.y)
    Div by_g;
    int cgv, grid, gy;
    size_t smem;
};
template <int LG> struct RowSpot {
    int lane, g, first, step;   // lane within the group, group, first sample, samples between
    bool on;
    __device__ RowSpot(const Rows& W, int G) {
        const int seg = threadIdx.x / LG;
        lane = threadIdx.x % LG;
        if (W.tall) {
            const int k = W.by_g(seg);
            g = seg - k * G;
            on = k < W.tall;
            first = blockIdx.x * W.tall + k;
            step = gridDim.x * W.tall;
        } else {
            g = blockIdx.y * W.segs + seg;
            on = g < G;
            first = blockIdx.x;
            step = gridDim.x;
        }
    }
};
template <int LG> __device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int o = LG / 2; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}
// samples on their way at a time: four vectors a lane (backward: of x and of dy each)
template <int KV> __host__ __device__ constexpr int rows_at_once() { return KV == 1 ? 4 : KV == 2 ? 2 : 1; }

template <typename T, int VEC, int KV, int LG, bool U8>
__global__ void __launch_bounds__(NT, KV == 1 ? 4 : 2) k_norm_rows_fwd(const FmeGroupNorm A, const __grid_constant__ Rows W) {
    using V = Pack<T, VEC>;
    constexpr int U = rows_at_once<KV>();
    const RowSpot<LG> S(W, A.g);
    const int cgr = W.cgv * VEC;
    const float inv_m = 1.f / (float)cgr;
    bool has[KV];
    float w[KV][VEC], b[KV][VEC];
#pragma unroll
    for (int k = 0; k < KV; k++) {
        has[k] = S.on && S.lane + k * LG < W.cgv;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int c = S.g * cgr + (S.lane + k * LG) * VEC + j;
            w[k][j] = has[k] && A.w ? __ldg(A.w + c) : 1.f;
            b[k][j] = has[k] && A.b ? __ldg(A.b + c) : 0.f;
        }
    }
    const T* x0 = (const T*)A.x + S.first * A.x_sn + S.g * cgr + S.lane * VEC;
    const int64_t xs = S.step * A.x_sn, ys = (int64_t)S.step * A.c;
    int64_t at = (int64_t)S.first * A.c + S.g * cgr + S.lane * VEC, ng = (int64_t)S.first * A.g + S.g;
    V x[U][KV];
    auto load = [&](int u, int64_t n, const T* p) {
#pragma unroll
        for (int k = 0; k < KV; k++)
            if (has[k] && n < A.n) x[u][k] = *reinterpret_cast<const V*>(p + k * LG * VEC);
    };
#pragma unroll
    for (int u = 0; u < U; u++) load(u, S.first + (int64_t)u * S.step, x0 + u * xs);
    for (int64_t n = S.first, base = 0; base < A.n; base += (int64_t)U * S.step) {   // the same trips for all lanes: shuffles
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool ok = n < A.n;
            float f[KV][VEC], s = 0.f, lo = INFINITY, hi = -INFINITY, q = 0.f;
#pragma unroll
            for (int k = 0; k < KV; k++) {
                floats<T, VEC>(f[k], x[u][k]);
                if (has[k]) {
#pragma unroll
                    for (int j = 0; j < VEC; j++) { s += f[k][j]; if (U8) { lo = fminf(lo, f[k][j]); hi = fmaxf(hi, f[k][j]); } }
                }
            }
            load(u, n + (int64_t)U * S.step, x0 + U * xs);   // on its way while the next samples are computed
            s = lanes_sum<LG>(s);
            if (U8) {
#pragma unroll
                for (int o = LG / 2; o > 0; o >>= 1) { lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o)); }
            }
            const float mean = s * inv_m;
            const float inv = U8 ? code_inv(lo, hi) : 0.f;
#pragma unroll
            for (int k = 0; k < KV; k++)
                if (has[k]) {
                    if (U8 && ok) *reinterpret_cast<Pack<uint8_t, VEC>*>(A.codes + at + k * LG * VEC) = codes_of<VEC>(f[k], &lo, &inv, false);
#pragma unroll
                    for (int j = 0; j < VEC; j++) { f[k][j] -= mean; q = fmaf(f[k][j], f[k][j], q); }
                }
            const float rstd = rsqrtf(fmaf(lanes_sum<LG>(q), inv_m, A.eps));
            if (ok && S.on) {
                if (A.mean && S.lane == 0) {
                    A.mean[ng] = mean; A.rstd[ng] = rstd;
                    if (U8) { A.lo[ng] = lo; A.hi[ng] = hi; }
                }
                by_act(A.act, [&](auto act) {
#pragma unroll
                    for (int k = 0; k < KV; k++)
                        if (has[k]) {
#pragma unroll
                            for (int j = 0; j < VEC; j++) f[k][j] = act_fwd(decltype(act)::value, fmaf(f[k][j] * rstd, w[k][j], b[k][j]));
                            *reinterpret_cast<V*>((T*)A.y + at + k * LG * VEC) = packed<T, VEC>(f[k]);
                        }
                });
            }
            n += S.step; at += ys; ng += (int64_t)S.step * A.g; x0 += xs;
        }
    }
}

template <typename T, int VEC, int KV, int LG, bool U8>
__global__ void __launch_bounds__(NT, KV == 4 ? 1 : 2) k_norm_rows_bwd(const FmeGroupNorm A, const __grid_constant__ Rows W) {
    using V = Pack<T, VEC>;
    using XT = typename std::conditional<U8, uint8_t, T>::type;
    using X = Pack<XT, VEC>;
    constexpr int U = rows_at_once<KV>();
    extern __shared__ float rw[];
    const RowSpot<LG> S(W, A.g);
    const int cgr = W.cgv * VEC;
    const float inv_m = 1.f / (float)cgr;
    bool has[KV];
    float w[KV][VEC], b[KV][VEC], dw[KV][VEC], db[KV][VEC];
#pragma unroll
    for (int k = 0; k < KV; k++) {
        has[k] = S.on && S.lane + k * LG < W.cgv;
#pragma unroll
        for (int j = 0; j < VEC; j++) {
            const int c = S.g * cgr + (S.lane + k * LG) * VEC + j;
            w[k][j] = has[k] && A.w ? __ldg(A.w + c) : 1.f;
            b[k][j] = has[k] && A.b && A.act != FME_ACT_NONE ? __ldg(A.b + c) : 0.f;   // without an activation b is not used
            dw[k][j] = db[k][j] = 0.f;
        }
    }
    const int col = S.g * cgr + S.lane * VEC;
    const T *x0 = (const T*)A.x + S.first * A.x_sn + col, *g0 = (const T*)A.dy + S.first * A.dy_sn + col;
    const int64_t xs = S.step * A.x_sn, gs = S.step * A.dy_sn, ys = (int64_t)S.step * A.c;
    int64_t at = (int64_t)S.first * A.c + col, ng = (int64_t)S.first * A.g + S.g;
    V g[U][KV];
    X x[U][KV];
    float mean[U], rstd[U], lo[U], hi[U];
    auto load = [&](int u, int64_t n, int64_t at, int64_t ng, const T* px, const T* pg) {
        const bool ok = S.on && n < A.n;
#pragma unroll
        for (int k = 0; k < KV; k++)
            if (has[k] && ok) {
                if constexpr (U8) x[u][k] = *reinterpret_cast<const X*>(A.codes + at + k * LG * VEC);
                else x[u][k] = *reinterpret_cast<const X*>(px + k * LG * VEC);
                g[u][k] = *reinterpret_cast<const V*>(pg + k * LG * VEC);
            }
        mean[u] = ok ? __ldg(A.mean + ng) : 0.f;
        rstd[u] = ok ? __ldg(A.rstd + ng) : 0.f;
        lo[u] = U8 && ok ? __ldg(A.lo + ng) : 0.f;
        hi[u] = U8 && ok ? __ldg(A.hi + ng) : 0.f;
    };
#pragma unroll
    for (int u = 0; u < U; u++) load(u, S.first + (int64_t)u * S.step, at + u * ys, ng + (int64_t)u * S.step * A.g, x0 + u * xs, g0 + u * gs);
    for (int64_t n = S.first, base = 0; base < A.n; base += (int64_t)U * S.step) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const bool ok = n < A.n;
            const float xa = U8 ? code_step(lo[u], hi[u]) * rstd[u] : rstd[u], xb = U8 ? (lo[u] - mean[u]) * rstd[u] : mean[u];
            float xh[KV][VEC], dz[KV][VEC], s1 = 0.f, s2 = 0.f;
#pragma unroll
            for (int k = 0; k < KV; k++) {
                floats<XT, VEC>(xh[k], x[u][k]);
                floats<T, VEC>(dz[k], g[u][k]);
#pragma unroll
                for (int j = 0; j < VEC; j++) xh[k][j] = U8 ? fmaf(xh[k][j], xa, xb) : (xh[k][j] - xb) * xa;
            }
            const float scale = rstd[u];
            load(u, n + (int64_t)U * S.step, at + U * ys, ng + (int64_t)U * S.step * A.g, x0 + U * xs, g0 + U * gs);   // while this one is computed
            by_act(A.act, [&](auto act) {
#pragma unroll
                for (int k = 0; k < KV; k++)
#pragma unroll
                    for (int j = 0; j < VEC; j++) dz[k][j] = act_bwd(decltype(act)::value, fmaf(xh[k][j], w[k][j], b[k][j]), dz[k][j]);
            });
#pragma unroll
            for (int k = 0; k < KV; k++)
                if (has[k] && ok) {
#pragma unroll
                    for (int j = 0; j < VEC; j++) {
                        const float wd = w[k][j] * dz[k][j];
                        s1 += wd; s2 = fmaf(wd, xh[k][j], s2);
                        db[k][j] += dz[k][j]; dw[k][j] = fmaf(dz[k][j], xh[k][j], dw[k][j]);
                    }
                }
            const float a1 = lanes_sum<LG>(s1) * inv_m, a2 = lanes_sum<LG>(s2) * inv_m;
#pragma unroll
            for (int k = 0; k < KV; k++)
                if (has[k] && ok) {
#pragma unroll
                    for (int j = 0; j < VEC; j++) dz[k][j] = scale * fmaf(-xh[k][j], a2, fmaf(dz[k][j], w[k][j], -a1));
                    *reinterpret_cast<V*>((T*)A.dx + at + k * LG * VEC) = packed<T, VEC>(dz[k]);
                }
            n += S.step; at += ys; ng += (int64_t)S.step * A.g; x0 += xs; g0 += gs;
        }
    }
    if (!A.dw) return;
    let_next_start();
    // the CTA's row of dw and db: c of each, with zeros where another grid.y has the channels
    float* row = (float*)A.ws + ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 2 * A.c;
    const int tall = W.tall ? W.tall : 1, k0 = W.tall ? (S.first - (int)blockIdx.x * W.tall) : 0;
    const int cols = W.tall ? A.c : min(W.segs, A.g - (int)blockIdx.y * W.segs) * cgr, c0 = W.tall ? 0 : blockIdx.y * W.segs * cgr;
#pragma unroll
    for (int k = 0; k < KV; k++)
        if (has[k]) {
#pragma unroll
            for (int j = 0; j < VEC; j++) {
                const int c = S.g * cgr + (S.lane + k * LG) * VEC + j - c0;
                rw[k0 * cols + c] = dw[k][j]; rw[(tall + k0) * cols + c] = db[k][j];
            }
        }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * A.c; i += NT) {
        const int c = (i < A.c ? i : i - A.c) - c0;
        float s = 0.f;
        if (c >= 0 && c < cols)
            for (int k = 0; k < tall; k++) s += rw[((i < A.c ? 0 : tall) + k) * cols + c];
        row[i] = s;
    }
}

// ---------------------------------------------------------------- calls without a plan
// What make_plan refuses: vectors whose channels repeat only after more than MAX_THREADS of them (odd channel counts above 512,
// fp32 ones above 2048, and with c > 512 whatever cannot be read in 16-byte pieces), and more groups than shared memory has
// room for the sums of. One thread a channel, x read three times. One CTA walks samples blockIdx.x, + gridDim.x, ...;
// per-channel sums in shared memory, one thread a channel, joined by one warp a group.

// A sum that carries what each addition rounds off (Kahan): a thread adds up all pixels of a channel, and without it the mean of a
// constant group of 4096 pixels came out 737 units of 2^-24 away from the constant.
struct Sum {
    float s = 0.f, c = 0.f;
    __device__ __forceinline__ void take(float y) { const float t = s + y; c = (t - s) - y; s = t; }
    __device__ __forceinline__ void add(float x) { take(x - c); }
    __device__ __forceinline__ void add(float x, float y) { take(fmaf(x, y, -c)); }
};

template <typename T> __global__ void __launch_bounds__(NT) k_norm_wide_fwd(const FmeGroupNorm A) {
    extern __shared__ float wide[];
    float *s0 = wide, *s1 = wide + A.c, *s2 = wide + 2 * A.c, *s3 = wide + 3 * A.c;
    const int cg = A.c / A.g, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const float m = (float)((int64_t)A.p * cg);
    for (int64_t n = blockIdx.x; n < A.n; n += gridDim.x) {
        const T* x = (const T*)A.x + n * A.x_sn;
        const int64_t base = n * (int64_t)A.p * A.c;
        for (int c = threadIdx.x; c < A.c; c += NT) {
            Sum s;
            float lo = INFINITY, hi = -INFINITY;
            for (int64_t p = 0; p < A.p; p++) { const float v = to_f(x[p * A.c + c]); s.add(v); lo = fminf(lo, v); hi = fmaxf(hi, v); }
            s0[c] = s.s; s3[c] = s.c; s1[c] = lo; s2[c] = hi;
        }
        __syncthreads();
        for (int g = warp; g < A.g; g += NT / 32) {
            double s = 0.;   // so that the mean is rounded once: of a constant group it is the constant
            float lo = INFINITY, hi = -INFINITY;
            for (int c = g * cg + lane; c < (g + 1) * cg; c += 32) { s += (double)s0[c] - (double)s3[c]; lo = fminf(lo, s1[c]); hi = fmaxf(hi, s2[c]); }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xffffffffu, s, o);
                lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)); hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            }
            const float mean = (float)(s / ((double)A.p * cg));
            for (int c = g * cg + lane; c < (g + 1) * cg; c += 32) { s0[c] = mean; s1[c] = lo; s2[c] = hi; }
            if (lane == 0) {
                if (A.codes) { A.lo[n * A.g + g] = lo; A.hi[n * A.g + g] = hi; }
                if (A.mean) A.mean[n * A.g + g] = mean;
            }
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
            Sum q;
            for (int64_t p = 0; p < A.p; p++) { const float d = to_f(x[p * A.c + c]) - s0[c]; q.add(d, d); }
            s1[c] = q.s;
        }
        __syncthreads();
        for (int g = warp; g < A.g; g += NT / 32) {
            Sum q;
            for (int c = g * cg + lane; c < (g + 1) * cg; c += 32) q.add(s1[c]);
            const float r = rsqrtf(lanes_sum<32>(q.s) / m + A.eps);
            for (int c = g * cg + lane; c < (g + 1) * cg; c += 32) s2[c] = r;
            if (A.rstd && lane == 0) A.rstd[n * A.g + g] = r;
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
    extern __shared__ float wide[];
    float *s0 = wide, *s1 = wide + A.c, *tw = wide + 2 * A.c, *tb = wide + 3 * A.c;
    const int cg = A.c / A.g, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
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
                Sum a1, a2;
                for (int64_t p = 0; p < A.p; p++) {
                    const int64_t i = p * A.c + c;
                    const float xh = (x_of<T>(A, n, i, lo, step) - mean) * rstd;
                    const float dz = act_bwd(A.act, fmaf(xh, w, b), to_f(dy[i]));
                    if (pass == 0) { a1.add(dz); a2.add(dz, xh); }
                    else ((T*)A.dx)[n * (int64_t)A.p * A.c + i] = from_f<T>(rstd * (dz * w - s0[c] - xh * s1[c]));
                }
                if (pass == 0) { s0[c] = a1.s; s1[c] = a2.s; tb[c] += a1.s; tw[c] += a2.s; }
            }
            __syncthreads();
            if (pass == 0) {
                for (int g = warp; g < A.g; g += NT / 32) {
                    Sum a1, a2;
                    for (int c = g * cg + lane; c < (g + 1) * cg; c += 32) { const float w = A.w ? A.w[c] : 1.f; a1.add(s0[c], w); a2.add(s1[c], w); }
                    const float m1 = lanes_sum<32>(a1.s) / m, m2 = lanes_sum<32>(a2.s) / m;
                    for (int c = g * cg + lane; c < (g + 1) * cg; c += 32) { s0[c] = m1; s1[c] = m2; }
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
    await_previous();
    if (i < 2 * c) {
        const float* p = ws + i;
        int r = threadIdx.y;
        for (; r + 7 * 32 < rows; r += 8 * 32) {
            float x[8];
#pragma unroll
            for (int k = 0; k < 8; k++) x[k] = p[(int64_t)(r + k * 32) * 2 * c];
#pragma unroll
            for (int k = 0; k < 8; k++) s += x[k];
        }
        for (; r < rows; r += 32) s += p[(int64_t)r * 2 * c];
    }
    sm[threadIdx.y][threadIdx.x] = s;
    __syncthreads();
    s = sm[threadIdx.x][threadIdx.y];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int col = blockIdx.x * 32 + threadIdx.y;
    if (threadIdx.x == 0 && col < 2 * c) (col < c ? dw[col] : db[col - c]) = s;
}

// ---------------------------------------------------------------- host side
constexpr int SMS = 148;

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
bool split_parts(const Plan& P) { return P.parts > 1 && !P.cluster; }
int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

Div divisor(int d) { return Div{(uint32_t)d, d <= 1 ? 0u : (uint32_t)((0x100000000ull + d - 1) / d)}; }
int64_t round_up(int64_t x, int64_t to) { return (x + to - 1) / to * to; }
int pow2_up(int x) { int p = 1; while (p < x) p *= 2; return p; }

int vec_of(const FmeGroupNorm& a, bool bwd) {
    const int e = a.dtype == FME_F32 ? 4 : 2, full = 16 / e;
    auto al = [&](const void* p, int64_t sn) { return !((uintptr_t)p & 15) && !((sn * e) & 15); };
    const bool wide = (int64_t)a.p * a.c % full == 0 && !((uintptr_t)a.codes & 7) &&
                      (bwd ? al(a.dy, a.dy_sn) && al(a.dx, 0) && (a.codes || al(a.x, a.x_sn)) : al(a.x, a.x_sn) && al(a.y, 0));
    return wide ? full : 1;
}

// Groups in a row: one pixel, whole vectors in a group, at most 4 of them for each lane.
bool make_rows(const FmeGroupNorm& a, bool bwd, Rows* W, int* kv) {
    const int vec = vec_of(a, bwd), cgr = a.c / a.g;
    if (a.p != 1 || vec == 1 || cgr % vec) return false;
    W->cgv = cgr / vec;
    if (W->cgv > 128) return false;
    W->LG = W->cgv > 32 ? 32 : pow2_up(W->cgv);
    *kv = W->cgv <= 32 ? 1 : W->cgv <= 64 ? 2 : 4;
    W->segs = NT / W->LG;
    W->tall = W->segs / a.g;
    W->gy = W->tall ? 1 : (a.g + W->segs - 1) / W->segs;
    W->by_g = divisor(a.g);
    const int at_once = W->tall ? W->tall : 1;
    const int64_t need = ((int64_t)a.n + at_once - 1) / at_once, most = (int64_t)SMS * (bwd ? (*kv == 4 ? 1 : 2) : (*kv == 1 ? 4 : 2)) / W->gy;
    W->grid = (int)(need < most ? need : most);   // as many CTAs as the GPU holds
    if (W->grid < 1) W->grid = 1;
    W->smem = bwd ? (size_t)8 * (W->tall ? W->tall * a.c : W->segs * cgr) : 0;
    return true;
}

// The layout with this many parts of `chunk` vectors. false: more shared memory, or more CTAs, than there are.
bool lay_out(const FmeGroupNorm& a, bool bwd, int parts, bool cluster, int64_t chunk, int per, Plan* P) {
    const int e = a.dtype == FME_F32 ? 4 : 2, vec = P->vec;
    const int64_t nvec = (int64_t)a.p * a.c / vec;
    const int bpv = vec * (bwd ? e + (a.codes ? 1 : e) : e);
    P->parts = parts;
    P->cluster = cluster;
    P->chunk = (int)(chunk < per ? per : chunk);
    P->nvec = (int)nvec;
    const bool gr = (a.c / a.g) % vec == 0, whole = a.c % vec == 0;
    const int cv = whole ? a.c / vec : 0;
    const bool pow2 = gr && cv <= 32 && (cv & (cv - 1)) == 0 && ((cv / a.g) & (cv / a.g - 1)) == 0;
    P->how = !gr ? EACH : pow2 ? WARP : ONE;
    // Twelve vectors a thread when there is much to do (8192 x 9 x 9 x 64 fp32 with codes: 66 + 78 us then, with eight 78 + 88 us, with
    // sixteen 62 + 77 us, but 1024 x 20 x 20 x 32 22 + 36 against 20 + 33 us); two when not: then the call takes as long as one CTA
    const bool busy = (int64_t)a.n * parts >= 4 * SMS;
    int64_t r = (P->chunk + (busy ? 12 : 2) - 1) / (busy ? 12 : 2);
    if (r < 32) r = P->chunk < 32 ? P->chunk : 32;
    // (64 registers a thread: four CTAs of 256, five of 192; where clusters have to fit beside each other, five)
    const int unit = P->how == WARP ? 32 : per, top = busy ? (parts > 1 ? 192 : 256) : MAX_THREADS;
    if (r > top) r = top;
    P->R = (int)round_up(r, unit);
    if (P->R > top) P->R = top / unit > 0 ? top / unit * unit : unit;
    P->M = 1;
    P->tile = (int)round_up((int64_t)P->chunk * bpv, 16);
    if (parts == 1 && P->R <= 128) {
        P->M = 256 / P->R;
        while (P->M > 1 && (int64_t)P->M * P->tile > 50 * 1024) P->M--;
        if (P->M > a.n) P->M = a.n > 0 ? a.n : 1;
    }
    P->threads = (P->R * P->M + 31) / 32 * 32;
    const int ns = P->how == EACH ? vec : 1, pairs = P->M * a.g, warps = P->threads / 32;
    P->L = ns == 1 ? a.c / vec : a.c;
    P->gl = P->L / a.g;
    P->rows = P->R * ns / P->L;
    P->by_r = divisor(P->R); P->by_c = divisor(a.c); P->by_cg = divisor(a.c / a.g); P->by_gl = divisor(P->gl); P->by_g = divisor(a.g);
    const int64_t groups = ((int64_t)a.n + P->M - 1) / P->M;
    const int nv = bwd ? 2 : 3;
    const size_t red = P->how == WARP ? (size_t)(bwd ? 4 : 4) * warps * a.g : (size_t)nv * P->R * P->M * ns;
    P->smem = (size_t)P->M * P->tile + 4 * ((bwd ? 4 : 8) * (size_t)pairs + red);
    if (bwd) {
        const size_t end = (size_t)8 * P->R * P->M * vec;
        if (P->smem < end) P->smem = end;
        int64_t at_once = (int64_t)(220 * 1024 / (P->smem + 1024)), by_threads = 1024 / P->threads;
        at_once = at_once < by_threads ? at_once : by_threads;
        if (at_once < 1) at_once = 1;
        const int64_t walk = SMS * at_once / parts;
        P->grid = (int)((split_parts(*P) || groups < walk ? groups : walk) * parts);
    } else {
        P->grid = (int)(groups * parts);
    }
    return groups * parts <= 0x7fffffff && P->smem <= 220 * 1024;
}

// How a call is laid out. false: the kernels for calls without a plan (k_norm_wide_*).
bool make_plan(const FmeGroupNorm& a, bool bwd, Plan* P) {
    const int e = a.dtype == FME_F32 ? 4 : 2;
    const int vec = vec_of(a, bwd);
    P->vec = vec;
    const int per = a.c / gcd(a.c, vec);               // threads after which a vector's channels repeat
    if (per > MAX_THREADS) return false;
    const int64_t nvec = (int64_t)a.p * a.c / vec;
    const int bpv = vec * (bwd ? e + (a.codes ? 1 : e) : e);
    // Parts of some 50 KB: four CTAs an SM. With few samples, more and smaller parts.
    const int64_t most = 50 * 1024 / bpv, bound = 200 * 1024 / bpv;
    int parts = 1;
    while (parts < 16 && (nvec > parts * most || (a.n * (int64_t)parts < 2 * SMS && nvec >= parts * 2048))) parts *= 2;
    // What a cluster cannot hold is split: parts that are too large by themselves, and parts that leave no room for the sums
    // (16 parts of up to 200 KB with 24 to 48 KB of sums beside them: bf16, 112 x 112 x 64 in 32 groups, backward)
    const int64_t part = round_up((nvec + parts - 1) / parts, per);
    if (part <= bound && lay_out(a, bwd, parts, parts > 1, part, per, P)) return true;
    if (parts == 1) return false;
    parts = (int)((nvec + most - 1) / most);
    return lay_out(a, bwd, parts, false, round_up((nvec + parts - 1) / parts, per), per, P);
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

int join_grid(const FmeGroupNorm& a) { return (int)(((int64_t)a.n * a.g + NT / 32 - 1) / (NT / 32)); }

template <typename T, int VEC, int HOW> int run_fwd(const FmeGroupNorm& a, const Plan& P, cudaStream_t st) {
    const char* what = "fme_group_norm_fwd";
    if (!split_parts(P)) return launch(what, k_norm_fwd<T, VEC, HOW, WHOLE>, P, st, a, P);
    int rc = launch(what, k_norm_fwd<T, VEC, HOW, STATS>, P, st, a, P);
    if (rc) return rc;
    k_norm_join_fwd<T, VEC><<<join_grid(a), NT, 0, st>>>(a, P.parts, P.chunk);
    if ((rc = launch_status(what))) return rc;
    return launch(what, k_norm_fwd<T, VEC, HOW, APPLY>, P, st, a, P);
}
template <typename T, int VEC, int HOW, bool U8> int run_bwd(const FmeGroupNorm& a, const Plan& P, cudaStream_t st) {
    const char* what = "fme_group_norm_bwd";
    if (!split_parts(P)) return launch(what, k_norm_bwd<T, VEC, HOW, WHOLE, U8>, P, st, a, P);
    int rc = launch(what, k_norm_bwd<T, VEC, HOW, STATS, U8>, P, st, a, P);
    if (rc) return rc;
    k_norm_join_bwd<<<join_grid(a), NT, 0, st>>>(a, P.parts);
    if ((rc = launch_status(what))) return rc;
    return launch(what, k_norm_bwd<T, VEC, HOW, APPLY, U8>, P, st, a, P);
}
template <typename T, bool U8> int run_bwd(const FmeGroupNorm& a, const Plan& P, cudaStream_t st) {
    constexpr int full = 16 / sizeof(T);
    if (P.vec == 1) return P.how == WARP ? run_bwd<T, 1, WARP, U8>(a, P, st) : run_bwd<T, 1, ONE, U8>(a, P, st);
    if (P.how == WARP) return run_bwd<T, full, WARP, U8>(a, P, st);
    return P.how == ONE ? run_bwd<T, full, ONE, U8>(a, P, st) : run_bwd<T, full, EACH, U8>(a, P, st);
}
template <typename T> int run_fwd(const FmeGroupNorm& a, const Plan& P, cudaStream_t st) {
    constexpr int full = 16 / sizeof(T);
    if (P.vec == 1) return P.how == WARP ? run_fwd<T, 1, WARP>(a, P, st) : run_fwd<T, 1, ONE>(a, P, st);
    if (P.how == WARP) return run_fwd<T, full, WARP>(a, P, st);
    return P.how == ONE ? run_fwd<T, full, ONE>(a, P, st) : run_fwd<T, full, EACH>(a, P, st);
}

template <typename T, bool U8, bool BWD, int KV, int LG> auto rows_kernel() {
    constexpr int full = 16 / sizeof(T);
    if constexpr (BWD) return &k_norm_rows_bwd<T, full, KV, LG, U8>;
    else return &k_norm_rows_fwd<T, full, KV, LG, U8>;
}
template <typename T, bool U8, bool BWD> int run_rows(const FmeGroupNorm& a, const Rows& W, int kv, cudaStream_t st) {
    auto kernel = rows_kernel<T, U8, BWD, 4, 32>();
    if (kv == 2) kernel = rows_kernel<T, U8, BWD, 2, 32>();
    if (kv == 1) kernel = W.LG == 1 ? rows_kernel<T, U8, BWD, 1, 1>() : W.LG == 2 ? rows_kernel<T, U8, BWD, 1, 2>() : W.LG == 4 ? rows_kernel<T, U8, BWD, 1, 4>()
                        : W.LG == 8 ? rows_kernel<T, U8, BWD, 1, 8>() : W.LG == 16 ? rows_kernel<T, U8, BWD, 1, 16>() : rows_kernel<T, U8, BWD, 1, 32>();
    if (W.smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)W.smem);
    kernel<<<dim3(W.grid, W.gy), NT, W.smem, st>>>(a, W);
    return launch_status(BWD ? "fme_group_norm_bwd" : "fme_group_norm_fwd");
}
template <bool BWD> int run_rows(const FmeGroupNorm& a, const Rows& W, int kv, cudaStream_t st) {
    if (a.dtype == FME_F32) return a.codes ? run_rows<float, true, BWD>(a, W, kv, st) : run_rows<float, false, BWD>(a, W, kv, st);
    return a.codes ? run_rows<__nv_bfloat16, true, BWD>(a, W, kv, st) : run_rows<__nv_bfloat16, false, BWD>(a, W, kv, st);
}

constexpr int WIDE_GRID = 592;
// floats of the workspace before the CTAs' rows of dw and db
int64_t split_floats(const FmeGroupNorm& a, const Plan& P, int each) { return split_parts(P) ? (int64_t)each * ((int64_t)a.n * P.parts * a.g + (int64_t)a.n * a.g) : 0; }

}  // namespace
}  // namespace fme

using namespace fme;

extern "C" {

int64_t fme_group_norm_bytes(const FmeGroupNorm* a, int32_t which) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (which < 0 || which > 1) return bad("group norm: which must be 0 or 1");
    Plan P;
    Rows W;
    int kv;
    if (make_rows(*a, which == 1, &W, &kv)) return which == 0 ? 0 : (int64_t)W.grid * W.gy * 2 * a->c * 4;
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
    Rows W;
    int kv;
    if (make_rows(*a, false, &W, &kv)) return run_rows<false>(*a, W, kv, st);
    if (!make_plan(*a, false, &P)) {
        const size_t smem = (size_t)4 * a->c * 4;
        const int grid = a->n < WIDE_GRID ? a->n : WIDE_GRID;
        auto kernel = a->dtype == FME_F32 ? k_norm_wide_fwd<float> : k_norm_wide_fwd<__nv_bfloat16>;
        if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        kernel<<<grid, NT, smem, st>>>(*a);
        return launch_status("fme_group_norm_fwd");
    }
    return a->dtype == FME_F32 ? run_fwd<float>(*a, P, st) : run_fwd<__nv_bfloat16>(*a, P, st);
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
    Rows W;
    int rows = a->n < WIDE_GRID ? a->n : WIDE_GRID, kv;
    int64_t skip = 0;
    const bool u8 = a->codes != nullptr;
    if (make_rows(*a, true, &W, &kv)) {
        rows = W.grid * W.gy;
        rc = run_rows<true>(*a, W, kv, st);
    } else if (!make_plan(*a, true, &P)) {
        const size_t smem = (size_t)4 * a->c * 4;
        auto kernel = a->dtype == FME_F32 ? k_norm_wide_bwd<float> : k_norm_wide_bwd<__nv_bfloat16>;
        if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
        kernel<<<rows, NT, smem, st>>>(*a);
        rc = launch_status("fme_group_norm_bwd");
    } else {
        rows = P.grid;
        skip = split_floats(*a, P, 2);
        if (a->dtype == FME_F32) rc = u8 ? run_bwd<float, true>(*a, P, st) : run_bwd<float, false>(*a, P, st);
        else rc = u8 ? run_bwd<__nv_bfloat16, true>(*a, P, st) : run_bwd<__nv_bfloat16, false>(*a, P, st);
    }
    if (rc || !a->dw) return rc;
    return launch_behind("fme_group_norm_bwd", k_norm_params, dim3((2 * a->c + 31) / 32), dim3(32, 32), 0, st, (const float*)a->ws + skip, rows, a->c, a->dw, a->db);
}

}  // extern "C"

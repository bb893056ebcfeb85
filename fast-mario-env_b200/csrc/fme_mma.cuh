// fme_mma.cuh - shared-memory tiles and matrix products of one warp, for bfloat16 and for float32.
//
// bfloat16: mma m16n8k16. float32: mma m16n8k8 in tf32 with every operand split in two tf32 numbers, x = hi + lo, and the
// products hi hi + hi lo + lo hi: 22 bits of each operand count, the dropped lo lo is 2^-22 of a term. Accumulators are
// float32, in the layout that both shapes share: acc[0..1] = (row g, columns 2c, 2c+1), acc[2..3] = (row g + 8, the same)
// with g = lane / 4 and c = lane % 4.
//
// A tile is a row-major matrix of COLS values; its 16-byte pieces are permuted within 128 bytes by the row, so that
// neither eight rows of one piece (ldmatrix) nor columns of rows 2c and 2c + 1 (transposed reads of float32) share a bank.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fme {

using bf16 = __nv_bfloat16;

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(bf16 x) { return __bfloat162float(x); }
template <typename T> __device__ __forceinline__ T from_f(float x);
template <> __device__ __forceinline__ float from_f<float>(float x) { return x; }
template <> __device__ __forceinline__ bf16 from_f<bf16>(float x) { return __float2bfloat16(x); }

__device__ __forceinline__ uint32_t pack2(float a, float b) {
    __nv_bfloat162 p = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&p);
}
__device__ __forceinline__ float2 unpack2(uint32_t p) {
    return make_float2(__uint_as_float(p << 16), __uint_as_float(p & 0xffff0000u));
}

template <typename T, int COLS> struct Tile {
    static constexpr int ROW = COLS * (int)sizeof(T);   // bytes
    static constexpr int PER = 16 / (int)sizeof(T);     // values of a 16-byte piece
    uint32_t base;                                      // shared-space address
    char* gen;                                          // generic address
    __device__ __forceinline__ Tile(void* p) : base((uint32_t)__cvta_generic_to_shared(p)), gen((char*)p) {}
    static __device__ __forceinline__ uint32_t off(int row, int col) {
        const uint32_t piece = (uint32_t)col / PER, in = ((uint32_t)col % PER) * sizeof(T);
        const uint32_t sw = ROW >= 128 ? (uint32_t)(row & 7) : (uint32_t)((row >> 1) & 3);
        return (uint32_t)row * ROW + ((piece ^ sw) << 4) + in;
    }
    // A lane's address of piece x (0 or 1) of row + its own row (row a multiple of 8, so that the permutation does not depend on
    // it), and from there the same piece `bytes` (a multiple of 32) further along the row: an exclusive or within 128 bytes
    __device__ __forceinline__ uint32_t lane(int row, int own, int x) const {
        const uint32_t sw = ROW >= 128 ? (uint32_t)(own & 7) : (uint32_t)((own >> 1) & 3);
        return base + (uint32_t)row * ROW + ((uint32_t)own * ROW + (((uint32_t)x ^ sw) << 4));
    }
    static __device__ __forceinline__ uint32_t along(uint32_t lane, int bytes) { return (lane ^ ((uint32_t)bytes & 127u)) + ((uint32_t)bytes & ~127u); }
    __device__ __forceinline__ T& at(int row, int col) const { return *reinterpret_cast<T*>(gen + off(row, col)); }
    __device__ __forceinline__ float2 two(int row, int col) const {   // col even
        if constexpr (sizeof(T) == 2) return unpack2(*reinterpret_cast<const uint32_t*>(gen + off(row, col)));
        else return *reinterpret_cast<const float2*>(gen + off(row, col));
    }
    __device__ __forceinline__ void put2(int row, int col, float a, float b) const {
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint32_t*>(gen + off(row, col)) = pack2(a, b);
        else *reinterpret_cast<float2*>(gen + off(row, col)) = make_float2(a, b);
    }
};

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
__device__ __forceinline__ void stsm4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ float lds(uint32_t addr) {
    float x;
    asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(addr));
    return x;
}
__device__ __forceinline__ uint32_t tf32(float x) {
    uint32_t r;
    asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = tf32(x);
    lo = tf32(x - __uint_as_float(hi));
}

template <typename T> struct Frag;

template <> struct Frag<bf16> {
    static constexpr int KS = 16, UNROLL = 8;   // steps of a product in one piece of code
    struct A { uint32_t r[4]; };
    struct B { uint32_t r[2]; };
    struct A2 { A hi, lo, rest; };    // a scaled operand in two bfloat16 numbers (16 bits of it count) or three (24)
    // 16 x 16 accumulators to a tile
    template <int COLS> static __device__ __forceinline__ void put16(const Tile<bf16, COLS>& s, int row, int col, const float* u, const float* v) {
        const int l = threadIdx.x & 31;
        stsm4(s.along(s.lane(row, l & 15, l >> 4), 2 * col), pack2(u[0], u[1]), pack2(u[2], u[3]), pack2(v[0], v[1]), pack2(v[2], v[3]));
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const A& a, const B& b) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a.r[0]), "r"(a.r[1]), "r"(a.r[2]), "r"(a.r[3]), "r"(b.r[0]), "r"(b.r[1]));
    }
    // d = a b where FIRST, else d += a b
    template <bool FIRST> static __device__ __forceinline__ void begin(float (&d)[4], const A& a, const B& b) {
        if constexpr (FIRST)
            asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                         : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a.r[0]), "r"(a.r[1]), "r"(a.r[2]), "r"(a.r[3]), "r"(b.r[0]), "r"(b.r[1]), "f"(0.f));
        else mma(d, a, b);
    }
    // A[m][k] = tile[m][k]
    template <int COLS> static __device__ __forceinline__ A ldA(const Tile<bf16, COLS>& s, int m, int k) {
        const int l = threadIdx.x & 31;
        A a;
        ldsm4(a.r, s.along(s.lane(m, l & 15, l >> 4), 2 * k));
        return a;
    }
    // B[k][n] = tile[n][k], 16 columns n
    template <int COLS> static __device__ __forceinline__ void ldB(const Tile<bf16, COLS>& s, int n, int k, B& b0, B& b1) {
        const int l = threadIdx.x & 31;
        uint32_t r[4];
        ldsm4(r, s.along(s.lane(n, (l & 7) + ((l >> 4) << 3), (l >> 3) & 1), 2 * k));
        b0.r[0] = r[0]; b0.r[1] = r[1]; b1.r[0] = r[2]; b1.r[1] = r[3];
    }
    // B[k][n] = tile[k][n], 16 columns n
    template <bool NAT, int COLS> static __device__ __forceinline__ void ldBt(const Tile<bf16, COLS>& s, int k, int n, B& b0, B& b1) {
        const int l = threadIdx.x & 31;
        uint32_t r[4];
        ldsm4t(r, s.along(s.lane(k, l & 15, l >> 4), 2 * n));
        b0.r[0] = r[0]; b0.r[1] = r[1]; b1.r[0] = r[2]; b1.r[1] = r[3];
    }
    // A[m][k] = weight[k] * tile[k][m], weights in shared memory
    template <int COLS> static __device__ __forceinline__ A2 ldAt(const Tile<bf16, COLS>& s, int k, int m, const float* w, bool fine) {
        const int l = threadIdx.x & 31;
        A2 a;
        ldsm4t(a.hi.r, s.along(s.lane(k, (l & 7) + ((l >> 4) << 3), (l >> 3) & 1), 2 * m));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const float2 v = unpack2(a.hi.r[i]), f = *reinterpret_cast<const float2*>(w + k + ((i >> 1) << 3) + 2 * (l & 3));
            const float x = v.x * f.x, y = v.y * f.y;
            a.hi.r[i] = pack2(x, y);
            const float2 h = unpack2(a.hi.r[i]);
            a.lo.r[i] = pack2(x - h.x, y - h.y);
            if (fine) {
                const float2 g = unpack2(a.lo.r[i]);
                a.rest.r[i] = pack2(x - h.x - g.x, y - h.y - g.y);
            }
        }
        return a;
    }
    // FINE: with 24 bits, and through a sum of its own. The tensor core cuts a sum off at the accumulator's last bit, always
    // towards zero, which adds up over many chunks, where an addition rounds to nearest. 16384 tokens: 49 and not 47 us.
    template <bool FINE> static __device__ __forceinline__ void add(float (&d)[4], const A2& a, const B& b) {
        if constexpr (FINE) {
            float t[4];
            begin<true>(t, a.rest, b);
            mma(t, a.lo, b);
            mma(t, a.hi, b);
#pragma unroll
            for (int i = 0; i < 4; i++) d[i] += t[i];
        } else {
            mma(d, a.lo, b);
            mma(d, a.hi, b);
        }
    }
    // The accumulators of 16 columns as an operand whose k runs over them
    static __device__ __forceinline__ A chain(const float (*acc)[4], int ks) {
        const float *u = acc[2 * ks], *v = acc[2 * ks + 1];
        return A{{pack2(u[0], u[1]), pack2(u[2], u[3]), pack2(v[0], v[1]), pack2(v[2], v[3])}};
    }
};

template <> struct Frag<float> {
    static constexpr int KS = 8, UNROLL = 1;    // longer steps, and code that outgrows the instruction cache stalls
    struct A { uint32_t hi[4], lo[4]; };
    struct B { uint32_t hi[2], lo[2]; };
    using A2 = A;
    template <int COLS> static __device__ __forceinline__ void put16(const Tile<float, COLS>& s, int row, int col, const float* u, const float* v) {
        const int g = (threadIdx.x & 31) >> 2, c = 2 * (threadIdx.x & 3);
        s.put2(row + g, col + c, u[0], u[1]);
        s.put2(row + g + 8, col + c, u[2], u[3]);
        s.put2(row + g, col + 8 + c, v[0], v[1]);
        s.put2(row + g + 8, col + 8 + c, v[2], v[3]);
    }
    static __device__ __forceinline__ void one(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
    }
    static __device__ __forceinline__ void mma(float (&d)[4], const A& a, const B& b) {
        one(d, a.lo, b.hi);
        one(d, a.hi, b.lo);
        one(d, a.hi, b.hi);
    }
    // d = a b
    static __device__ __forceinline__ void fresh(float (&d)[4], const A& a, const B& b) {
        asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
                     : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a.lo[0]), "r"(a.lo[1]), "r"(a.lo[2]), "r"(a.lo[3]), "r"(b.hi[0]), "r"(b.hi[1]), "f"(0.f));
        one(d, a.hi, b.lo);
        one(d, a.hi, b.hi);
    }
    template <bool> static __device__ __forceinline__ void begin(float (&d)[4], const A& a, const B& b) { mma(d, a, b); }   // d is zero at first
    // the same with the products of a remainder in sums of their own
    static __device__ __forceinline__ void mma_apart(float (&d)[4], float (&r)[4], const A& a, const B& b) {
        one(r, a.lo, b.hi);
        one(r, a.hi, b.lo);
        one(d, a.hi, b.hi);
    }
    template <int COLS> static __device__ __forceinline__ A ldA(const Tile<float, COLS>& s, int m, int k) {
        const int l = threadIdx.x & 31;
        uint32_t r[4];
        ldsm4(r, s.along(s.lane(m, l & 15, l >> 4), 4 * k));
        A a;
#pragma unroll
        for (int i = 0; i < 4; i++) split_tf32(__uint_as_float(r[i]), a.hi[i], a.lo[i]);
        return a;
    }
    template <int COLS> static __device__ __forceinline__ void ldB(const Tile<float, COLS>& s, int n, int k, B& b0, B& b1) {
        const int l = threadIdx.x & 31;
        uint32_t r[4];
        ldsm4(r, s.along(s.lane(n, (l & 7) + ((l >> 4) << 3), (l >> 3) & 1), 4 * k));
#pragma unroll
        for (int i = 0; i < 2; i++) {
            split_tf32(__uint_as_float(r[i]), b0.hi[i], b0.lo[i]);
            split_tf32(__uint_as_float(r[2 + i]), b1.hi[i], b1.lo[i]);
        }
    }
    // Which row of eight the two halves of a transposed operand take: rows c and c + 4 (NAT, to go with ldA), or rows 2c and
    // 2c + 1, to go with chain() and ldAt(), without bank conflicts
    template <bool NAT> static __device__ __forceinline__ int row_of(int i) {
        const int c = threadIdx.x & 3;
        return NAT ? c + 4 * i : 2 * c + i;
    }
    template <bool NAT, int COLS> static __device__ __forceinline__ void ldBt(const Tile<float, COLS>& s, int k, int n, B& b0, B& b1) {
        const int g = (threadIdx.x & 31) >> 2;
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const uint32_t at = s.lane(k, row_of<NAT>(i), g >> 2) + 4 * (g & 3);
            split_tf32(lds(s.along(at, 4 * n)), b0.hi[i], b0.lo[i]);
            split_tf32(lds(s.along(at, 4 * n + 32)), b1.hi[i], b1.lo[i]);
        }
    }
    template <int COLS> static __device__ __forceinline__ A2 ldAt(const Tile<float, COLS>& s, int k, int m, const float* w, bool) {
        const int g = (threadIdx.x & 31) >> 2;
        A a;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const int own = row_of<false>(i >> 1);
            split_tf32(lds(s.along(s.lane(k, own, g >> 2) + 4 * (g & 3), 4 * (m + 8 * (i & 1)))) * w[k + own], a.hi[i], a.lo[i]);
        }
        return a;
    }
    // through a sum of its own, as bf16's; at 2 x 4729 tokens the error fell from 2.7e-6 to 8e-7 (now 6e-7) for 1 % of the time
    template <bool> static __device__ __forceinline__ void add(float (&d)[4], const A2& a, const B& b) {
        float t[4];
        fresh(t, a, b);
#pragma unroll
        for (int i = 0; i < 4; i++) d[i] += t[i];
    }
    static __device__ __forceinline__ A chain(const float (*acc)[4], int ks) {
        const float* u = acc[ks];
        A a;
        split_tf32(u[0], a.hi[0], a.lo[0]);
        split_tf32(u[2], a.hi[1], a.lo[1]);
        split_tf32(u[1], a.hi[2], a.lo[2]);
        split_tf32(u[3], a.hi[3], a.lo[3]);
        return a;
    }
};

// 16 bytes from global to shared memory, zeros where !in
__device__ __forceinline__ void cp16(uint32_t dst, const void* src, bool in) {
    const int n = in ? 16 : 0;
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

}  // namespace fme

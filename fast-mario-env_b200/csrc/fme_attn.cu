// fme_attn.cu - decayed linear attention with restarts: over whole sequences, forward and backward, and one token at
// a time. Sizes, layouts and the recurrence are those of include/fme.h (FmeDecayAttn).
//
// Sequences are taken in chunks of C tokens. With S the state before a chunk, L_ij = lambda^(i-j) where j <= i and no restart
// lies in (j, i], a_i = lambda^(i+1) where none lies in [0, i], z_j = lambda^(last-j) where none lies in (j, last], all else 0:
//   o    = scale ( (q k^T . L) v + a (q S) )                      S'  = thru S + (z k)^T v
//   dq   = scale ( (do v^T . L) k + a (do S^T) )                  U   = thru U' + scale (a q)^T do
//   dk   = scale (do v^T . L)^T q + z (v U'^T)                    dv  = scale (q k^T . L)^T do + z (k U')
// with U' the gradient of the state after the chunk and U that before it. A CTA walks the chunks of one sequence and head and
// keeps S (or U) in registers, fp32, so that q, k, v (and do) are read once and o (dq, dk, dv) written once; the forward pass of a
// training step also stores S before every chunk but the first, in the operands' type, as the products read it.
// Where there are too few sequences and heads to fill the GPU, the chunks are split into segments: first every segment's own
// part of the state, then these joined in order, then all segments at once with the state that they begin with.
//
// What it has to move: forward 4 tensors, backward 7, and between them the kept states (D / C tensors written and read). At 64
// features the tensors are 1 KB and 1.8 KB a token and head in bf16 for 25 and 55 thousand flops, so HBM is the floor. Products are
// warp-level mma: every warp fetches its operands from shared memory by itself, and do v^T is found twice. The tensor pipe is busy
// for 35 % of the time; what bounds the kernels now is the rest of the instruction stream (issue slots 45 to 49 % used by 12 to 16
// warps an SM, shared memory 55 to 68 %): those fetches, masks, rounding to operands, stores. tcgen05 products, which read shared
// memory by themselves and accumulate outside the registers, would spare the fetches; they are not built.
// Measured on a B200 (HBM copy 6441 GB/s), 1024 x 128 tokens of 8 heads of 64, restarts at 2 %: bf16 forward 128 us (4.2 TB/s of the
// tensors above), backward 268 us (3.5 TB/s); fp32, 257 x 127 with states in and out: 665 us both, backward 70 % of it, bound by
// its three tf32 products and the splitting of their operands at every read (issue slots 50 %, ALU 45 %, tensor 38 %).
// Chunks of 64: with 128 (no state between two chunks of a 128-token rollout, more products within one) the same pass took 486
// us where it took 441 then. One CTA for each sequence and head: CTAs that walk several with the powers kept took 171 us forward
// where it took 153 then.
#include <math.h>

#include <type_traits>

#include "fme_host.h"
#include "fme_mma.cuh"

namespace fme {
namespace {

template <typename T> __device__ __forceinline__ T* at(const FmeAttnTensor& x, int64_t n, int64_t h) {
    return reinterpret_cast<T*>(x.p) + n * x.sn + h * x.sh;
}

// Sizes of a CTA: D / 16 warps; warp w owns rows 16 w of the state and, of a chunk's outputs, rows 16 (w % RB) and columns
// NC (w / RB). C is 64 but for D = 32 (two warps) and D = 128 in fp32 (shared memory), 32. At D = 128 the warps that share rows each
// find the scores for themselves.
template <typename T, int D> struct Shape {
    static constexpr int C = D == 32 || (D == 128 && sizeof(T) == 4) ? 32 : 64;
    static constexpr int NW = D / 16, NT = 32 * NW, RB = C / 16, CG = NW / RB, NC = D / CG;
    static constexpr int TILE = C * D * (int)sizeof(T), MAT = D * D * (int)sizeof(T);
    static constexpr int FLOATS = 2 * 72;                    // powers and weights
};

// Where a chunk restarts. Bit i: token i does; valid tokens only.
struct Cuts {
    uint64_t m;
    int n;   // tokens in the chunk
    __device__ __forceinline__ int last_up_to(int i) const {   // latest restart at or before i, -1: none
        const uint64_t x = m & (~0ull >> (63 - i));
        return 63 - __clzll((long long)x);
    }
};

struct ResetBytes {
    uint32_t a = 0, b = 0;
    __device__ __forceinline__ void load(const uint8_t* r, int64_t rt, int t0, int n) {
        const int l = threadIdx.x & 31;
        a = r && l < n ? r[(t0 + l) * rt] : 0u;
        b = r && l + 32 < n ? r[(t0 + l + 32) * rt] : 0u;
    }
    __device__ __forceinline__ uint64_t bits() const {
        const uint32_t lo = __ballot_sync(0xffffffffu, a != 0u), hi = __ballot_sync(0xffffffffu, b != 0u);
        return ((uint64_t)hi << 32) | lo;
    }
};

// rows of one operand's chunk to shared memory; rows past the sequence's end become zeros
template <typename T, int D, int C, int NT>
__device__ __forceinline__ void load_tile(const Tile<T, D>& dst, const T* src, int64_t st, int t0, int n) {
    constexpr int PIECES = D / Tile<T, D>::PER, STEP = NT / PIECES;   // STEP: rows between a thread's pieces
    const int row = threadIdx.x / PIECES, col = (threadIdx.x % PIECES) * Tile<T, D>::PER;
    const char* p = reinterpret_cast<const char*>(src + (t0 + row) * st + col);
    const int64_t step = STEP * st * (int64_t)sizeof(T);
    static_assert(STEP % 8 == 0, "the permutation repeats after eight rows");
    const uint32_t to = dst.base + dst.off(row, col);
    if (n == C) {
#pragma unroll
        for (int i = 0; i < C / STEP; i++) cp16(to + i * STEP * Tile<T, D>::ROW, p + i * step, true);
    } else {
#pragma unroll
        for (int i = 0; i < C / STEP; i++) {
            const bool in = row + i * STEP < n;
            cp16(to + i * STEP * Tile<T, D>::ROW, in ? p + i * step : reinterpret_cast<const char*>(src), in);
        }
    }
}

// Sixteen rows (n of them valid) of a tile to global memory, a row's pieces as 16 bytes each
template <typename TI, int COLS, typename T> __device__ __forceinline__ void copy_rows(const TI& s, int from, T* dst, int64_t st, int n) {
    constexpr int PIECES = COLS / TI::PER, STEP = 32 / PIECES;   // STEP: rows between a lane's pieces
    const int l = threadIdx.x & 31, row = l / PIECES, piece = l % PIECES;
    const uint32_t a = s.lane(from, row, piece);
    T* p = dst + row * st + piece * TI::PER;
    auto one = [&](int i) {   // i * STEP further down the permutation differs in bits that row does not have
        uint4 v;
        const uint32_t at = (TI::ROW >= 128 ? a ^ (((i * STEP) & 7) << 4) : a) + i * STEP * TI::ROW;
        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
        *reinterpret_cast<uint4*>(p + i * STEP * st) = v;
    };
    if (n >= 16) {
#pragma unroll
        for (int i = 0; i < 16 / STEP; i++) one(i);
    } else {
#pragma unroll
        for (int i = 0; i < 16 / STEP; i++)
            if (row + i * STEP < n) one(i);
    }
}

// A warp's 16 x NC accumulators to rows row0.. and columns col0.. of a (t, h, d) output: through shared memory, so that a row's
// pieces leave as 16 bytes each
template <typename T, int NC>
__device__ __forceinline__ void store_rows(char* stage, const float (&acc)[NC / 8][4], T* dst, int64_t st, int row0, int col0, int t0, int n) {
    constexpr int PW = NC < 32 ? 32 : NC;
    static_assert(NC >= 32, "");
    const Tile<T, PW> s(stage);
#pragma unroll
    for (int i = 0; i < NC / 8; i += 2) Frag<T>::put16(s, 0, 8 * i, acc[i], acc[i + 1]);
    __syncwarp();
    copy_rows<Tile<T, PW>, NC>(s, 0, dst + (t0 + row0) * st + col0, st, n - row0);
    __syncwarp();
}

// The same without shared memory. fp32: four lanes write a row's 32 bytes
template <int NC>
__device__ __forceinline__ void put_rows(const float (&acc)[NC / 8][4], float* dst, int64_t st, int row0, int col0, int t0, int n) {
    const int l = threadIdx.x & 31, g = l >> 2;
    float* p = dst + (int64_t)(t0 + row0 + g) * st + col0 + 2 * (l & 3);
    const int64_t down = 8 * st;
    const bool in0 = row0 + g < n, in1 = row0 + g + 8 < n;
#pragma unroll
    for (int i = 0; i < NC / 8; i++) {
        if (in0) *reinterpret_cast<float2*>(p + 8 * i) = make_float2(acc[i][0], acc[i][1]);
        if (in1) *reinterpret_cast<float2*>(p + down + 8 * i) = make_float2(acc[i][2], acc[i][3]);
    }
}
// bf16: lanes 2x and 2x + 1 hold two words each of two neighbouring blocks of 8 columns and
// trade one, so that each has 8 bytes in a row and four lanes write a row's 32 bytes
template <int NC>
__device__ __forceinline__ void put_rows(const float (&acc)[NC / 8][4], bf16* dst, int64_t st, int row0, int col0, int t0, int n) {
    const int l = threadIdx.x & 31, g = l >> 2, c = l & 3;
    const bool odd = c & 1;
    bf16* p = dst + (int64_t)(t0 + row0 + g) * st + col0 + (odd ? 8 : 0) + 4 * (c >> 1);
    const int64_t down = 8 * st;
    const bool in0 = row0 + g < n, in1 = row0 + g + 8 < n;
#pragma unroll
    for (int i = 0; i < NC / 8; i += 2) {
#pragma unroll
        for (int h = 0; h < 2; h++) {
            const uint32_t a = pack2(acc[i][2 * h], acc[i][2 * h + 1]), b = pack2(acc[i + 1][2 * h], acc[i + 1][2 * h + 1]);
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? a : b, 1);
            const uint2 w = odd ? make_uint2(got, b) : make_uint2(a, got);
            if (h ? in1 : in0) *reinterpret_cast<uint2*>(p + (h ? down : 0) + 8 * i) = w;
        }
    }
}

template <int N> __device__ __forceinline__ bool not_finite(const float (&a)[N][4]) {
    float z = 0.f;   // x * 0 is NaN unless x is finite
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) z = fmaf(a[i][j], 0.f, z);
    return z != 0.f;
}

// Rows g and g + 8 times f0 and f1. A product with 0 keeps what is not a number: such a chunk is done again, see walk()
template <int N> __device__ __forceinline__ void weigh(float (&a)[N][4], float f0, float f1) {
#pragma unroll
    for (int i = 0; i < N; i++) { a[i][0] *= f0; a[i][1] *= f0; a[i][2] *= f1; a[i][3] *= f1; }
}

template <int N> __device__ __forceinline__ void zero(float (&a)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) a[i][j] = 0.f;
}

// Sixteen rows of a tile as the left operand of several products: bf16 keeps them in registers, fp32 reads and splits them again (its
// loops have to stay rolled for the instruction cache; unrolled, with the rows in registers: 807 against 711 us, 257 x 127)
template <typename T, int D> struct Left {
    using F = Frag<T>;
    static constexpr bool KEPT = sizeof(T) == 2;
    typename F::A f[KEPT ? D / F::KS : 1];
    const Tile<T, D>& t;
    int m;
    __device__ __forceinline__ Left(const Tile<T, D>& tile, int row) : t(tile), m(row) {
        if (KEPT) {
#pragma unroll
            for (int k = 0; k < D; k += F::KS) f[k / F::KS] = F::ldA(t, m, k);
        }
    }
    __device__ __forceinline__ typename F::A get(int k) const {
        if constexpr (KEPT) return f[k / F::KS];
        else return F::ldA(t, m, k);
    }
};

// Two steps of an fp32 product, 8 NB columns from n on: acc += a0 b(0) + a1 b(1), each 16 x 8 piece through a sum of its own that an
// addition rounds. In one accumulator each of the 3 K / 8 products cuts off at its last bit, towards zero: with heads of 128
// the error against 64 bits was 1.2e-6 (now 3.7e-7) and with heads of 64 5.7e-7 to 8.9e-7 (now 3.7e-7 to 5.3e-7), 2e-7 to 3e-7
// being that of sums in fp32. load(step, i, b0, b1) gives the columns.
template <int NB, typename F, typename L>
__device__ __forceinline__ void two_steps(float (&acc)[NB][4], const typename F::A& a0, const typename F::A& a1, L load) {
#pragma unroll
    for (int i = 0; i < NB; i += 2) {
        float t[2][4];
        typename F::B b0, b1;
        load(0, i, b0, b1);
        F::fresh(t[0], a0, b0);
        F::fresh(t[1], a0, b1);
        load(1, i, b0, b1);
        F::mma(t[0], a1, b0);
        F::mma(t[1], a1, b1);
#pragma unroll
        for (int j = 0; j < 4; j++) { acc[i][j] += t[0][j]; acc[i + 1][j] += t[1][j]; }
    }
}

// acc (16 x 8 NB) = A B, B the rows of a D x D tile as columns or, TR, its columns as columns. fp32 in two steps at a time with heads of
// 128 (10 x 556 tokens of 12 heads 838 -> 826 us forward and backward); with heads of 64 that needs more registers than there are
// for three CTAs (257 x 127 tokens of 8 heads 650 -> 716 us), and half as many products are added up.
template <typename T, int NB, int D, bool TR>
__device__ __forceinline__ void product(float (&acc)[NB][4], const Left<T, D>& a, const Tile<T, D>& b, int n) {
    using F = Frag<T>;
    auto step = [&](int k, auto first) {
        const typename F::A fa = a.get(k);
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
            typename F::B b0, b1;
            if (TR) F::template ldBt<true>(b, k, n + 8 * i, b0, b1);
            else F::ldB(b, n + 8 * i, k, b0, b1);
            F::template begin<decltype(first)::value>(acc[i], fa, b0);
            F::template begin<decltype(first)::value>(acc[i + 1], fa, b1);
        }
    };
    if constexpr (sizeof(T) == 4 && D == 128) {
        zero(acc);
#pragma unroll 1
        for (int k = 0; k < D; k += 2 * F::KS) {
            const typename F::A a0 = a.get(k), a1 = a.get(k + F::KS);
            two_steps<NB, F>(acc, a0, a1, [&](int s, int i, typename F::B& b0, typename F::B& b1) {
                if (TR) F::template ldBt<true>(b, k + s * F::KS, n + 8 * i, b0, b1);
                else F::ldB(b, n + 8 * i, k + s * F::KS, b0, b1);
            });
        }
        return;
    }
    if constexpr (sizeof(T) == 2) step(0, std::true_type{});
    else zero(acc);
#pragma unroll(Frag<T>::UNROLL)
    for (int k = sizeof(T) == 2 ? F::KS : 0; k < D; k += F::KS) step(k, std::false_type{});
}

// A warp's factors of L * scale for rows row0..row0+15 of a chunk, block of 16 columns by block. UP: rows are i, columns j, from the
// diagonal down to column 0; otherwise rows are j and columns i, from the diagonal up. On the diagonal the factors are as they are.
// Elsewhere lambda^(i-j) = lambda^(i-edge) lambda^(edge-j) with the edge between rows and column, so that neither power grows, and
// from one block to the next the column's part takes lambda^16. No restart in (j, i] means none in (j, edge] and none in
// (edge, i]: the mask is a product too, and blocks beyond the nearest restart outside the sixteen rows are not visited.
template <bool UP, int C> struct Decay {
    int row0, n, lim0, lim1, lim;   // lim: the nearest restart outside the rows, lim0 and lim1 for rows g and g + 8
    uint32_t own;                // restarts within the rows
    __device__ __forceinline__ Decay(const Cuts& cuts, int row0_) : row0(row0_), n(cuts.n) {
        const int g = (threadIdx.x & 31) >> 2;
        own = (uint32_t)(cuts.m >> row0) & 0xffffu;
        if (UP) {
            const uint64_t below = cuts.m & ~(~0ull << row0);
            const uint32_t x0 = own & (0x1ffu >> (8 - g)), x1 = own & (0x1ffffu >> (8 - g));
            lim = 63 - __clzll((long long)below);
            lim0 = x0 ? row0 + 31 - __clz(x0) : lim;
            lim1 = x1 ? row0 + 31 - __clz(x1) : lim;
        } else {
            const uint64_t above = row0 + 16 >= 64 ? 0ull : cuts.m >> (row0 + 16);
            const uint32_t x0 = own >> (g + 1), x1 = own >> (g + 9);
            lim = above ? row0 + 15 + __ffsll((long long)above) : 64;
            lim0 = x0 ? row0 + g + __ffs(x0) : lim;
            lim1 = x1 ? row0 + g + 8 + __ffs(x1) : lim;
        }
    }
    __device__ __forceinline__ void diagonal(float (&f)[2][4], const float* pw, float scale) const {
        const int l = threadIdx.x & 31, g = l >> 2, c = 2 * (l & 3);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int row = g + 8 * (j >> 1), col = 8 * i + c + (j & 1), d = UP ? row - col : col - row;
                f[i][j] = d >= 0 ? pw[d < 0 ? 0 : d] * scale : 0.f;
            }
        if (own) {
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int at = row0 + 8 * i + c + (j & 1), l = j < 2 ? lim0 : lim1;
                    f[i][j] = (UP ? at >= l : at < l) ? f[i][j] : 0.f;
                }
        }
    }
    // The rows' parts, and the columns' in the block next to the diagonal
    __device__ __forceinline__ void beside(float (&rows)[2], float (&cols)[2][2], const float* pw, float scale) const {
        const int l = threadIdx.x & 31, g = l >> 2, c = 2 * (l & 3);
        const bool in0 = UP ? lim0 < row0 : lim0 > row0 + 15, in1 = UP ? lim1 < row0 : lim1 > row0 + 15;
        rows[0] = in0 ? pw[UP ? g : 15 - g] * scale : 0.f;
        rows[1] = in1 ? pw[UP ? g + 8 : 7 - g] * scale : 0.f;
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) cols[i][e] = pw[UP ? 16 - 8 * i - c - e : 1 + 8 * i + c + e];
    }
    // Columns beyond the nearest restart, in the block that holds it
    __device__ __forceinline__ void cut(float (&x)[2][2], int col0) const {
        const int c = 2 * (threadIdx.x & 3);
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const int at = col0 + 8 * i + c + e;
                x[i][e] = (UP ? at >= lim : at < lim) ? x[i][e] : 0.f;
            }
    }
    // f(col0, factors) for every block that the mask leaves
    template <typename F> __device__ __forceinline__ void blocks(const float* pw, float scale, F f) const {
        float w[2][4], rows[2], cols[2][2];
        diagonal(w, pw, scale);
        beside(rows, cols, pw, scale);
        const float step = pw[16];
        const int last = UP ? (lim < 0 ? 0 : lim & ~15) : (lim > n ? n : lim) - 1;   // a column of the last block
#pragma unroll 1
        for (int col0 = row0;;) {   // one copy of f: the code has to stay in the instruction cache
            f(col0, w);
            col0 += UP ? -16 : 16;
            if (UP ? col0 < last : col0 > last) break;
            float x[2][2] = {{cols[0][0], cols[0][1]}, {cols[1][0], cols[1][1]}};
            if (UP ? col0 < lim : col0 + 16 > lim) cut(x, col0);
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int j = 0; j < 4; j++) w[i][j] = x[i][j & 1] * rows[j >> 1];
                cols[i][0] *= step; cols[i][1] *= step;
            }
        }
    }
};

// p = (16 rows) . (rows col0..col0+15 of b) * f
template <typename T, int D>
__device__ __forceinline__ void block_scores(float (&p)[2][4], const Left<T, D>& a, const Tile<T, D>& b, int col0, const float (&f)[2][4]) {
    using F = Frag<T>;
    if constexpr (sizeof(T) == 2) {
        const typename F::A fa = a.get(0);
        typename F::B b0, b1;
        F::ldB(b, col0, 0, b0, b1);
        F::template begin<true>(p[0], fa, b0);
        F::template begin<true>(p[1], fa, b1);
    } else zero(p);
    if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = F::KS; k < D; k += F::KS) {
            const typename F::A fa = a.get(k);
            typename F::B b0, b1;
            F::ldB(b, col0, k, b0, b1);
            F::mma(p[0], fa, b0);
            F::mma(p[1], fa, b1);
        }
    } else {   // the products with a remainder are summed apart: an accumulator drops bits at its own size with each addition
               // (error against 64 bits 6.7e-7 and not 8.3e-7 then, and the sums wait less for one another: 640 against 646 us, 257 x 127)
        float r[2][4];
        zero(r);
#pragma unroll 2
        for (int k = 0; k < D; k += F::KS) {
            const typename F::A fa = a.get(k);
            typename F::B b0, b1;
            F::ldB(b, col0, k, b0, b1);
            F::mma_apart(p[0], r[0], fa, b0);
            F::mma_apart(p[1], r[1], fa, b1);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) p[i][j] += r[i][j];
    }
#pragma unroll
    for (int i = 0; i < 2; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) p[i][j] *= f[i][j];
}

// acc += p (16 x 16) times rows row..row+15 of a tile, columns n..
template <typename T, int D, int NB>
__device__ __forceinline__ void block_apply(float (&acc)[NB][4], const float (&p)[2][4], const Tile<T, D>& b, int row, int n) {
    using F = Frag<T>;
    if constexpr (sizeof(T) == 2) {
        const typename F::A fa = F::chain(p, 0);
#pragma unroll
        for (int i = 0; i < NB; i += 2) {
            typename F::B b0, b1;
            F::template ldBt<false>(b, row, n + 8 * i, b0, b1);
            F::mma(acc[i], fa, b0);
            F::mma(acc[i + 1], fa, b1);
        }
    } else {
        const typename F::A a0 = F::chain(p, 0), a1 = F::chain(p, 1);
        two_steps<NB, F>(acc, a0, a1, [&](int s, int i, typename F::B& b0, typename F::B& b1) { F::template ldBt<false>(b, row + s * F::KS, n + 8 * i, b0, b1); });
    }
}

// state (rows m0..m0+15 of the D x D matrix) += (w a)^T b over the chunk's tokens. The scaled rows of bf16 are taken in 16 bits,
// fine: in 24, where the state itself is asked for, in fp32. Two loops, the choice outside: with it at each product 3 x 5000 tokens
// of 4 heads of 128 took 168 and not 153 us, forward and backward, and 1024 x 128 of 8 heads of 64 425 and not 411 us (then).
template <typename T, int D, int C, int UNROLL>
__device__ __forceinline__ void outer(float (&s)[D / 8][4], const Tile<T, D>& a, int m0, const float* w, const Tile<T, D>& b, bool fine) {
    using F = Frag<T>;
    auto step = [&](int k, auto all) {
        const typename F::A2 fa = F::ldAt(a, k, m0, w, decltype(all)::value);
#pragma unroll
        for (int i = 0; i < D / 8; i += 2) {
            typename F::B b0, b1;
            F::template ldBt<false>(b, k, 8 * i, b0, b1);
            F::template add<decltype(all)::value>(s[i], fa, b0);
            F::template add<decltype(all)::value>(s[i + 1], fa, b1);
        }
    };
    if constexpr (sizeof(T) == 2) {
        if (!fine) {
#pragma unroll(UNROLL)
            for (int k = 0; k < C; k += F::KS) step(k, std::false_type{});
            return;
        }
    }
#pragma unroll 1
    for (int k = 0; k < C; k += F::KS) step(k, std::true_type{});
}

template <int D> __device__ __forceinline__ void keep_state(float (&s)[D / 8][4], const Cuts& cuts, const float* pw) {
    if (cuts.m) { zero(s); return; }
    const float thru = pw[cuts.n];
#pragma unroll
    for (int i = 0; i < D / 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s[i][j] *= thru;
}

// A warp's rows of the state in a tile of the operands' type
template <typename T, int D> __device__ __forceinline__ void put_state(const Tile<T, D>& m, const float (&s)[D / 8][4], int row0) {
#pragma unroll
    for (int i = 0; i < D / 8; i += 2) Frag<T>::put16(m, row0, 8 * i, s[i], s[i + 1]);
}
// ... and to or from a (d, d) fp32 matrix. FLIP: the warp's rows are the matrix's columns.
template <int D, bool FLIP, bool STORE, typename P> __device__ __forceinline__ void move_state(float (&s)[D / 8][4], P* mat, int row0) {
    const int l = threadIdx.x & 31, g = l >> 2, c = l & 3;
#pragma unroll
    for (int i = 0; i < D / 8; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const int row = row0 + g + 8 * (j >> 1), col = 8 * i + 2 * c + (j & 1);
            P* e = mat + (FLIP ? col * D + row : row * D + col);
            if constexpr (STORE) *e = s[i][j];
            else s[i][j] = *e;
        }
}
// Between the segments' kernels the state stays in the order of the registers
template <int D, int NT, bool STORE> __device__ __forceinline__ void move_part(float (&s)[D / 8][4], float* ws, int64_t item) {
    float4* p = reinterpret_cast<float4*>(ws) + item * (D / 8) * NT + threadIdx.x;
#pragma unroll
    for (int i = 0; i < D / 8; i++) {
        if (STORE) p[i * NT] = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        else { const float4 f = p[i * NT]; s[i][0] = f.x; s[i][1] = f.y; s[i][2] = f.z; s[i][3] = f.w; }
    }
}

// ---------------------------------------------------------------- token by token
// A product with 0 keeps the NaN of a masked token, so a chunk whose result is not finite is done again by the recurrence
// itself, in which a restart drops what was before. A warp holds 16 rows r of a matrix M and walks the tokens:
//   M[r][c] += x_r y_c (after the decay going forward, before it going backward),   out_r = f sum_c M[r][c] z_c
template <typename T, int D, bool BACK>
__device__ __forceinline__ void walk(float (&m)[D / 8][4], const Tile<T, D>& x, const Tile<T, D>& y, const Tile<T, D>& z, float xf, float f,
                                     int row0, const Cuts& cuts, float lam, T* out, int64_t st, int t0) {
    const int l = threadIdx.x & 31, g = l >> 2, c = l & 3;
    for (int u = 0; u < cuts.n; u++) {
        const int t = BACK ? cuts.n - 1 - u : u;
        const bool cut = (cuts.m >> t) & 1;
        const float x0 = to_f(x.at(t, row0 + g)) * xf, x1 = to_f(x.at(t, row0 + g + 8)) * xf;
        float o0 = 0.f, o1 = 0.f;
#pragma unroll
        for (int i = 0; i < D / 8; i++) {
            const float2 yy = y.two(t, 8 * i + 2 * c), zz = z.two(t, 8 * i + 2 * c);
#pragma unroll
            for (int j = 0; j < 4; j++) {
                float& s = m[i][j];
                if (!BACK) s = cut ? 0.f : s * lam;
                s = fmaf(j < 2 ? x0 : x1, j & 1 ? yy.y : yy.x, s);
                float& o = j < 2 ? o0 : o1;
                o = fmaf(s, j & 1 ? zz.y : zz.x, o);
                if (BACK) s = cut ? 0.f : s * lam;
            }
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1) { o0 += __shfl_xor_sync(0xffffffffu, o0, d); o1 += __shfl_xor_sync(0xffffffffu, o1, d); }
        if (out && c == 0) {
            out[(t0 + t) * st + row0 + g] = from_f<T>(o0 * f);
            out[(t0 + t) * st + row0 + g + 8] = from_f<T>(o1 * f);
        }
    }
}

struct Walkers {   // the grid's layout: CTA = (sequence and head) * segs + segment
    int chunks, segs, per;   // chunks of the sequence, segments, chunks of a segment
    float* parts;            // state of the segments: D * D floats each, then one float each: what a segment passes on
};

// The CTA's segment, head and sequence
struct Spot {
    int seg, h, n;
    __device__ __forceinline__ Spot(const FmeDecayAttn& A, uint32_t across) {
        const uint32_t pair = across == 1 ? blockIdx.x : blockIdx.x / across;
        seg = blockIdx.x - pair * across;
        n = pair / (uint32_t)A.h;
        h = pair - n * A.h;
    }
};

__device__ __forceinline__ void powers(float* pw, int n, float log2_lam) {
    for (int i = threadIdx.x; i < n; i += blockDim.x) pw[i] = i ? exp2f(log2_lam * (float)i) : 1.f;
}

constexpr float LOG2E = 1.44269504088896340736f;

// The forward pass of a segment (state rows: features of v). LOCAL: only its part of the state, from zero (the first: from s_in).
// P = q k^T goes from accumulators straight to operands; the state's transpose is kept, so that its accumulators, rounded to the
// operands' type, are the rows that q S reads. Rounded to bf16: P, S as q reads it; o is off by 0.0023 of its norm against 0.0017 by
// its own rounding alone. One env's 16384 tokens, 8 heads of 64, bf16: parts, join and outputs, started behind each other, 49 us.
// STAGES: 2 loads the next chunk while this one is computed, for CTAs that have an SM to themselves or nearly so.
template <typename T, int D, bool LOCAL, int STAGES, int MINB>
__global__ void __launch_bounds__(Shape<T, D>::NT, MINB) k_attn_fwd(const FmeDecayAttn A, const Walkers W) {
    using Z = Shape<T, D>;
    using Ti = Tile<T, D>;
    constexpr int C = Z::C, NT = Z::NT, NC = Z::NC;
    extern __shared__ __align__(1024) char sm[];
    constexpr int SET = (LOCAL ? 2 : 3) * Z::TILE;
    const Ti ts(sm + STAGES * SET);
    float* pw = reinterpret_cast<float*>(sm + STAGES * SET + (LOCAL ? 0 : Z::MAT));   // C + 1
    float* z = pw + 72;                                                                       // C
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, g = l >> 2;
    const Spot P(A, LOCAL ? W.segs - 1 : W.segs);
    const int seg = P.seg, h = P.h, n = P.n;
    const bool fine = A.s_out != nullptr;
    const int c0 = seg * W.per, c1 = min(c0 + W.per, W.chunks);
    const int row0 = 16 * (warp % Z::RB), col0 = NC * (warp / Z::RB), m0 = 16 * warp;
    const float g2 = A.log_decay[h] * LOG2E;
    float s[D / 8][4];
    bool some;   // whether the state before the chunk may be other than zero
    ResetBytes rb;
    auto fetch = [&](int c) {
        const int t0 = c * C, nv = min(C, A.t - t0);
        char* set = sm + (STAGES == 2 ? ((c - c0) & 1) * SET : 0);
        load_tile<T, D, C, NT>(Ti(set), at<T>(A.k, n, h), A.k.st, t0, nv);
        load_tile<T, D, C, NT>(Ti(set + Z::TILE), at<T>(A.v, n, h), A.v.st, t0, nv);
        if (!LOCAL) load_tile<T, D, C, NT>(Ti(set + 2 * Z::TILE), at<T>(A.q, n, h), A.q.st, t0, nv);
        cp_commit();
        rb.load(A.reset ? A.reset + n * A.reset_sn : nullptr, A.reset_st, t0, nv);
    };
    if (c0 < c1) fetch(c0);
    powers(pw, C + 1, g2);
    __syncthreads();
    const int64_t pair = (int64_t)n * A.h + h;
    some = true;
    if (LOCAL) let_next_start();
    else await_previous();   // the parts
    if (seg > 0 && !LOCAL) move_part<D, NT, false>(s, W.parts, pair * (W.segs - 1) + seg - 1);
    else if (seg == 0 && A.s_in) move_state<D, true, false>(s, A.s_in + pair * D * D, m0);
    else { zero(s); some = false; }
    if (!LOCAL && some) put_state(ts, s, m0);
    uint64_t any_cut = 0;
    for (int c = c0; c < c1; c++) {
        const int t0 = c * C;
        char* set = sm + (STAGES == 2 ? ((c - c0) & 1) * SET : 0);
        const Ti tk(set), tv(set + Z::TILE), tq(set + 2 * Z::TILE);
        cp_wait<0>();
        __syncthreads();
        const Cuts cuts{rb.bits(), min(C, A.t - t0)};
        if (STAGES == 2 && c + 1 < c1) fetch(c + 1);   // the other set has been read by all
        any_cut |= cuts.m;
        bool again = false;
        {
            const int j = threadIdx.x, last = cuts.last_up_to(63);
            if (j < C) z[j] = j < cuts.n && j >= last ? pw[cuts.n - 1 - j] : 0.f;
        }
        if constexpr (LOCAL) __syncthreads();
        if constexpr (!LOCAL) {
            float acc[NC / 8][4];
            bool off = false;
            if (row0 < cuts.n) {   // rows past the sequence's end have nothing to do
                const Left<T, D> lq(tq, row0);
                if (some) {
                    product<T, NC / 8, D, false>(acc, lq, ts, col0);
                    const bool in0 = cuts.last_up_to(row0 + g) < 0, in1 = cuts.last_up_to(row0 + g + 8) < 0;
                    weigh(acc, in0 ? pw[row0 + g + 1] * A.scale : 0.f, in1 ? pw[row0 + g + 9] * A.scale : 0.f);
                } else zero(acc);
                const Decay<true, C> decay(cuts, row0);
                decay.blocks(pw, A.scale, [&](int j, const float (&f)[2][4]) {
                    float p[2][4];
                    block_scores<T, D>(p, lq, tk, j, f);
                    block_apply<T, D>(acc, p, tv, j, col0);
                });
                off = not_finite(acc);
            }
            again = __syncthreads_or(off);
            // q and the old state have been read by all: the q tile takes the outputs
            if (!again && row0 < cuts.n) {
                if constexpr (sizeof(T) == 2) store_rows<T, NC>(set + 2 * Z::TILE + warp * (16 * NC * (int)sizeof(T)), acc, at<T>(A.o, n, h), A.o.st, row0, col0, t0, cuts.n);
                else put_rows<NC>(acc, at<T>(A.o, n, h), A.o.st, row0, col0, t0, cuts.n);
            }
        }
        const bool more = c + 1 < c1, save = A.saved && c + 1 < W.chunks;
        if (more || LOCAL || save || (A.s_out && c + 1 == W.chunks)) {
            if (!again) {
                keep_state<D>(s, cuts, pw);
                outer<T, D, C, 4>(s, tv, m0, z, tk, fine);
                // after a restart nothing of the state before is left: if what came out is no number, the walk starts over
                if (LOCAL) again = cuts.m && __any_sync(0xffffffffu, not_finite(s));
            }
        }
        if (again) walk<T, D, false>(s, tv, tk, LOCAL ? tk : tq, 1.f, A.scale, m0, cuts, pw[1], LOCAL ? (T*)nullptr : at<T>(A.o, n, h), A.o.st, t0);
        some = true;
        if constexpr (!LOCAL) {
            if (more || save) put_state(ts, s, m0);
            if (save) {
                __syncwarp();
                copy_rows<Ti, D>(ts, m0, reinterpret_cast<T*>(A.saved) + ((pair * (W.chunks - 1) + c) * D + m0) * D, (int64_t)D, 16);
            }
        }
        if (STAGES == 1 && more) {
            __syncthreads();   // the tiles have been read by all
            fetch(c + 1);
        }
    }
    if (LOCAL) {
        move_part<D, NT, true>(s, W.parts, blockIdx.x);
        if (threadIdx.x == 0) {
            const int len = min(c1 * C, A.t) - c0 * C;
            W.parts[(int64_t)gridDim.x * D * D + blockIdx.x] = any_cut ? -1.f : exp2f(g2 * (float)len);
        }
    } else if (A.s_out && seg == W.segs - 1) {
        move_state<D, true, true>(s, A.s_out + pair * D * D, m0);
    }
}

// The backward pass of a segment, from its last chunk to its first (state rows: features of k). LOCAL: only its part of the
// state's gradient, from zero (the last: from ds_out); segments then count from the end. TWO: ds_in is wanted.
// A warp finds do v^T twice, once by rows and once by columns: two products more, no exchange through shared memory and no barrier.
// 3 x 5000 tokens, 4 heads of 128, bf16: 153 us with the forward pass's, one CTA of 8 warps an SM, bound by latency.
template <typename T, int D, bool LOCAL, bool TWO, int MINB>
__global__ void __launch_bounds__(Shape<T, D>::NT, MINB) k_attn_bwd(const FmeDecayAttn A, const Walkers W) {
    using Z = Shape<T, D>;
    using Ti = Tile<T, D>;
    constexpr int C = Z::C, NT = Z::NT, NC = Z::NC;
    extern __shared__ __align__(1024) char sm[];
    const Ti tq(sm), tg(sm + Z::TILE), tk(sm + 2 * Z::TILE), tv(sm + 3 * Z::TILE), ts(sm + 4 * Z::TILE), tu(sm + 4 * Z::TILE + Z::MAT);
    float* pw = reinterpret_cast<float*>(sm + (LOCAL ? 2 * Z::TILE : 4 * Z::TILE + 2 * Z::MAT));
    float* a = pw + 72;
    const int warp = threadIdx.x >> 5, l = threadIdx.x & 31, g = l >> 2;
    const Spot P(A, LOCAL ? W.segs - 1 : W.segs);
    const int rseg = P.seg, seg = W.segs - 1 - rseg, h = P.h, n = P.n;   // rseg 0: the last in time
    const bool fine = A.ds_in != nullptr;
    const int c0 = seg * W.per, c1 = min(c0 + W.per, W.chunks);
    const int row0 = 16 * (warp % Z::RB), col0 = NC * (warp / Z::RB), m0 = 16 * warp;
    const float g2 = A.log_decay[h] * LOG2E;
    float u[D / 8][4];
    bool some;   // whether the gradient of the state after the chunk may be other than zero
    ResetBytes rb;
    auto fetch_rows = [&](int c) {   // q and do
        const int t0 = c * C, nv = min(C, A.t - t0);
        load_tile<T, D, C, NT>(tq, at<T>(A.q, n, h), A.q.st, t0, nv);
        load_tile<T, D, C, NT>(tg, at<T>(A.d_o, n, h), A.d_o.st, t0, nv);
        cp_commit();
        rb.load(A.reset ? A.reset + n * A.reset_sn : nullptr, A.reset_st, t0, nv);
    };
    auto fetch_keys = [&](int c) {   // k, v and the state before the chunk
        const int t0 = c * C, nv = min(C, A.t - t0);
        const int64_t pair = (int64_t)n * A.h + h;
        load_tile<T, D, C, NT>(tk, at<T>(A.k, n, h), A.k.st, t0, nv);
        load_tile<T, D, C, NT>(tv, at<T>(A.v, n, h), A.v.st, t0, nv);
        if (c > 0) load_tile<T, D, D, NT>(ts, reinterpret_cast<const T*>(A.saved) + (pair * (W.chunks - 1) + c - 1) * D * D, D, 0, D);
        else if (A.s_in) {
            for (int i = threadIdx.x; i < D * D; i += NT) ts.at(i % D, i / D) = from_f<T>(A.s_in[pair * D * D + i]);
        }
        cp_commit();
    };
    auto fetch = [&](int c) {
        fetch_rows(c);
        if (!LOCAL) fetch_keys(c);
    };
    if (c0 < c1) fetch(c1 - 1);
    powers(pw, C + 1, g2);
    const int64_t pair = (int64_t)n * A.h + h;
    some = true;
    if (LOCAL) let_next_start();
    else await_previous();   // the parts
    if (rseg > 0 && !LOCAL) move_part<D, NT, false>(u, W.parts, pair * (W.segs - 1) + rseg - 1);
    else if (rseg == 0 && A.ds_out) move_state<D, false, false>(u, A.ds_out + pair * D * D, m0);
    else { zero(u); some = false; }
    uint64_t any_cut = 0;
    for (int c = c1 - 1; c >= c0; c--) {
        const int t0 = c * C;
        if (!LOCAL && some) put_state(tu, u, m0);
        cp_wait<0>();
        __syncthreads();
        const Cuts cuts{rb.bits(), min(C, A.t - t0)};
        any_cut |= cuts.m;
        const int last = cuts.last_up_to(63);
        const bool before = c > 0 || A.s_in;   // whether the state before the chunk may be other than zero
        bool again = false;
        if constexpr (!LOCAL) {
            const int r0 = row0 + g, r1 = r0 + 8;
            auto put = [&](const float (&acc)[NC / 8][4], const FmeAttnTensor& x) {
                again |= not_finite(acc);
                put_rows<NC>(acc, at<T>(x, n, h), x.st, row0, col0, t0, cuts.n);
            };
            if (row0 < cuts.n) {   // rows past the sequence's end have nothing to do
                float acc[NC / 8][4];
                {
                    const bool z0 = r0 >= last && r0 < cuts.n, z1 = r1 >= last && r1 < cuts.n;
                    const float w0 = z0 ? pw[cuts.n - 1 - r0] : 0.f, w1 = z1 ? pw[cuts.n - 1 - r1] : 0.f;
                    const Decay<false, C> down(cuts, row0);
                    // dv, then dk: the same with k and v, q and do in each other's place
#pragma unroll(sizeof(T) == 2 ? 2 : 1)
                    for (int which = 0; which < 2; which++) {
                        const Ti rows = which ? tv : tk, cols = which ? tg : tq, other = which ? tq : tg;
                        const Left<T, D> left(rows, row0);
                        if (some) {
                            if (which) product<T, NC / 8, D, false>(acc, left, tu, col0);
                            else product<T, NC / 8, D, true>(acc, left, tu, col0);
                            weigh(acc, w0, w1);
                        } else zero(acc);
                        down.blocks(pw, A.scale, [&](int i, const float (&f)[2][4]) {
                            float p[2][4];
                            block_scores<T, D>(p, left, cols, i, f);
                            block_apply<T, D>(acc, p, other, i, col0);
                        });
                        put(acc, which ? A.dk : A.dv);
                    }
                }
                const Decay<true, C> up(cuts, row0);
                const Left<T, D> lg(tg, row0);
                if (before) {
                    product<T, NC / 8, D, true>(acc, lg, ts, col0);
                    weigh(acc, cuts.last_up_to(r0) < 0 ? pw[r0 + 1] * A.scale : 0.f, cuts.last_up_to(r1) < 0 ? pw[r1 + 1] * A.scale : 0.f);
                } else zero(acc);
                up.blocks(pw, A.scale, [&](int j, const float (&f)[2][4]) {
                    float p[2][4];
                    block_scores<T, D>(p, lg, tv, j, f);
                    block_apply<T, D>(acc, p, tk, j, col0);
                });
                put(acc, A.dq);
            }
        }
        const bool more = c > c0;
        const int j = threadIdx.x;
        if (j < C) a[j] = j < cuts.n && cuts.last_up_to(j) < 0 ? pw[j + 1] * A.scale : 0.f;
        again = __syncthreads_or(again);
        if (!LOCAL && more && !again) fetch_keys(c - 1);   // k, v and the state before have been read by all
        if (LOCAL || again || more || TWO) {
            if (LOCAL) {
                keep_state<D>(u, cuts, pw);
                outer<T, D, C, 4>(u, tq, m0, a, tg, fine);
                if (cuts.m && __any_sync(0xffffffffu, not_finite(u)))   // as in the forward pass: the walk starts over
                    walk<T, D, true>(u, tq, tg, tg, A.scale, 1.f, m0, cuts, pw[1], (T*)nullptr, 0, t0);
            } else if (!again) {
                keep_state<D>(u, cuts, pw);
                outer<T, D, C, 2>(u, tq, m0, a, tg, fine);
            } else {
                float s[D / 8][4];
                const int cc = l & 3;
                // dq: forward from the state before the chunk (rows: features of k)
#pragma unroll
                for (int i = 0; i < D / 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[i][j] = before ? to_f(ts.at(8 * i + 2 * cc + (j & 1), m0 + g + 8 * (j >> 1))) : 0.f;
                walk<T, D, false>(s, tk, tv, tg, 1.f, A.scale, m0, cuts, pw[1], at<T>(A.dq, n, h), A.dq.st, t0);
                // dv: backward, the transposed gradient (rows: features of v)
#pragma unroll
                for (int i = 0; i < D / 8; i++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[i][j] = some ? to_f(tu.at(8 * i + 2 * cc + (j & 1), m0 + g + 8 * (j >> 1))) : 0.f;
                walk<T, D, true>(s, tg, tq, tk, A.scale, 1.f, m0, cuts, pw[1], at<T>(A.dv, n, h), A.dv.st, t0);
                // dk, and the gradient itself
                walk<T, D, true>(u, tq, tg, tv, A.scale, 1.f, m0, cuts, pw[1], at<T>(A.dk, n, h), A.dk.st, t0);
            }
        }
        some = true;
        if (more) {
            __syncthreads();   // the tiles and the gradient have been read by all
            fetch_rows(c - 1);
            if (!LOCAL && again) fetch_keys(c - 1);
        }
    }
    if (LOCAL) {
        move_part<D, NT, true>(u, W.parts, blockIdx.x);
        if (threadIdx.x == 0) {
            const int len = min(c1 * C, A.t) - c0 * C;
            W.parts[(int64_t)gridDim.x * D * D + blockIdx.x] = any_cut ? -1.f : exp2f(g2 * (float)len);
        }
    } else if (TWO && rseg == W.segs - 1) {
        move_state<D, false, true>(u, A.ds_in + pair * D * D, m0);
    }
}

// The segments' parts joined: parts[s] becomes the state after segments 0..s. One thread a value; a segment's loads depend on
// nothing, so JOIN of them are on their way at a time: the time is that of two or three trips to L2.
template <int JOIN> __global__ void __launch_bounds__(128) k_attn_join(float* parts, int64_t pairs, int segs, int dd) {
    const int64_t i = (int64_t)blockIdx.x * 128 + threadIdx.x;
    let_next_start();
    await_previous();
    if (i >= pairs * dd) return;
    const int64_t pair = i / dd;
    float* p = parts + pair * segs * dd + i % dd;
    const float* keep = parts + pairs * segs * dd + pair * segs;
    float s = p[0];
    for (int b = 1; b < segs; b += JOIN) {
        float x[JOIN], f[JOIN];
#pragma unroll
        for (int j = 0; j < JOIN; j++)
            if (b + j < segs) { x[j] = p[(int64_t)(b + j) * dd]; f[j] = keep[b + j]; }   // negative: a restart
#pragma unroll
        for (int j = 0; j < JOIN; j++)
            if (b + j < segs) {
                s = f[j] < 0.f ? x[j] : fmaf(s, f[j], x[j]);
                p[(int64_t)(b + j) * dd] = s;
            }
    }
}

// An empty sequence hands its state on.
__global__ void k_attn_pass(const float* from, float* to, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (int64_t)gridDim.x * blockDim.x) to[i] = from ? from[i] : 0.f;
}

// ---------------------------------------------------------------- one token
// One CTA a (sequence, head): a thread holds D * D / 256 values of the state in pieces of four columns, all loaded before the
// first is used. Bound by HBM: the state is read and written once, 8 D * D bytes, against 4 D values of q, k, v and o. Whole rows of
// CTAs, not split ones: a sequence and head is 16 KB at 64 features, and 128 of them (16 envs) take 4 us.
// 4096 envs x 8 heads of 64, bf16: 156 us, 7.0 TB/s; 1003 x 4 heads of 128, fp32: 82 us, 6.5 TB/s (copy: 6441 GB/s).
constexpr int STEP_THREADS = 256;
template <typename T, int D> __global__ void __launch_bounds__(STEP_THREADS) k_attn_step(const FmeDecayAttn A) {
    constexpr int LANES = D / 4, R = STEP_THREADS / LANES, PER = D / R;
    __shared__ float qk[2][D];
    __shared__ float4 part[R][LANES];
    const int64_t pair = blockIdx.x, n = pair / A.h, h = pair % A.h;
    const int lane = threadIdx.x % LANES, r = threadIdx.x / LANES;
    const bool cut = A.reset && A.reset[n * A.reset_sn];
    const float4* in = reinterpret_cast<const float4*>(A.s_in + pair * D * D) + lane;
    float4* out = reinterpret_cast<float4*>(A.s_out + pair * D * D) + lane;
    float4 s[PER];
#pragma unroll
    for (int i = 0; i < PER; i++) s[i] = in[(i * R + r) * LANES];
    if (threadIdx.x < 2 * D) qk[threadIdx.x / D][threadIdx.x % D] = to_f((threadIdx.x < D ? at<T>(A.q, n, h) : at<T>(A.k, n, h))[threadIdx.x % D]);
    const T* vp = at<T>(A.v, n, h) + 4 * lane;
    const float4 v = make_float4(to_f(vp[0]), to_f(vp[1]), to_f(vp[2]), to_f(vp[3]));
    const float lam = expf(A.log_decay[h]);
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PER; i++) {
        const float q = qk[0][i * R + r], k = qk[1][i * R + r];
        float4 x = s[i];
        if (cut) x = make_float4(0.f, 0.f, 0.f, 0.f);   // not a product: what was there may not be a number
        x = make_float4(fmaf(k, v.x, x.x * lam), fmaf(k, v.y, x.y * lam), fmaf(k, v.z, x.z * lam), fmaf(k, v.w, x.w * lam));
        out[(i * R + r) * LANES] = x;
        o = make_float4(fmaf(q, x.x, o.x), fmaf(q, x.y, o.y), fmaf(q, x.z, o.z), fmaf(q, x.w, o.w));
    }
    part[r][lane] = o;
    __syncthreads();
    if (threadIdx.x < D) {
        const float* p = reinterpret_cast<const float*>(part) + threadIdx.x;
        float t = 0.f;
#pragma unroll
        for (int i = 0; i < R; i++) t += p[i * D];
        at<T>(A.o, n, h)[threadIdx.x] = from_f<T>(t * A.scale);
    }
}

// ---------------------------------------------------------------- host side
constexpr int SMS = 148;
constexpr int SEG_CHUNKS = 4;    // chunks of a segment at least

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

template <typename T, int D> struct Plan {
    using Z = Shape<T, D>;
    Walkers W;
    int64_t pairs;
    Plan(const FmeDecayAttn& a, int ctas) {   // ctas: what an SM holds
        pairs = (int64_t)a.n * a.h;
        W.chunks = (a.t + Z::C - 1) / Z::C;
        W.segs = 1;
        W.per = W.chunks;
        W.parts = (float*)a.ws;
        // Segments where half the GPU or more would idle: as many as make one wave, of four chunks at least. 3 x 5000 tokens, 4 heads
        // of 128: 168 us with 12 segments (144 CTAs on 148 SMs; now 153), 250 us with 16 (192 CTAs). Splitting costs a second read of k and v
        // (q and do), so a GPU that is more than half full is left as it is.
        const int64_t slots = (int64_t)SMS * ctas;
        if (pairs > 0 && 2 * pairs <= slots && W.chunks >= 2 * SEG_CHUNKS) {
            int64_t want = slots / pairs;
            if (want > W.chunks / SEG_CHUNKS) want = W.chunks / SEG_CHUNKS;
            W.per = (int)((W.chunks + want - 1) / want);
            W.segs = (W.chunks + W.per - 1) / W.per;
        }
    }
    int64_t ws_bytes() const { return W.segs > 1 ? pairs * (W.segs - 1) * (4 * D * D + 4) : 0; }
    int64_t saved_bytes() const { return W.chunks > 1 ? pairs * (W.chunks - 1) * D * D * (int64_t)sizeof(T) : 0; }
    static constexpr int FLOAT_BYTES = Z::FLOATS * 4;
    static constexpr int FWD = 3 * Z::TILE + Z::MAT + FLOAT_BYTES, BWD = 4 * Z::TILE + 2 * Z::MAT + FLOAT_BYTES;
    static constexpr int LOCAL_FWD = 4 * Z::TILE + FLOAT_BYTES, LOCAL_BWD = 2 * Z::TILE + FLOAT_BYTES;
};
// CTAs an SM that the registers are bounded for: what shared memory allows, and no more than keeps the accumulators in registers
template <typename T, int D> constexpr int fwd_ctas() { return D == 128 ? 1 : D == 32 ? 8 : sizeof(T) == 4 ? 3 : 4; }
template <typename T, int D> constexpr int bwd_ctas() { return D == 128 ? 1 : D == 32 ? 6 : sizeof(T) == 4 ? 2 : 3; }
template <typename T, int D> constexpr int local_ctas() { return D == 128 ? 1 : sizeof(T) == 4 ? 2 : 4; }

template <typename K> int go(const char* what, K kernel, int64_t grid, int threads, int smem, cudaStream_t st, const FmeDecayAttn& a, const Walkers& W, bool behind = false) {
    if (smem > 48 * 1024) cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (behind) return launch_behind(what, kernel, dim3((unsigned)grid), dim3(threads), smem, st, a, W);
    kernel<<<(unsigned)grid, threads, smem, st>>>(a, W);
    return launch_status(what);
}
int join(const char* what, const Walkers& W, int64_t pairs, int dd, cudaStream_t st) {
    if (W.segs == 2) return FME_OK;   // one part: nothing to add
    auto kernel = W.segs > 17 ? k_attn_join<32> : k_attn_join<16>;   // 63 parts: 8.1 against 9.7 us; 11 parts: 11.8 against 8.4 us
    return launch_behind(what, kernel, dim3((unsigned)((pairs * dd + 127) / 128)), dim3(128), 0, st, W.parts, pairs, W.segs - 1, dd);
}
bool has_ws(const FmeDecayAttn& a, int64_t need) { return need == 0 || (a.ws && !((uintptr_t)a.ws & 255) && a.ws_bytes >= need); }
int pass_on(const char* what, const FmeDecayAttn& a, const float* from, float* to, cudaStream_t st) {
    if (to && to != from) k_attn_pass<<<592, 256, 0, st>>>(from, to, (int64_t)a.n * a.h * a.d * a.d);
    return launch_status(what);
}

template <typename T, int D> int launch_fwd(const FmeDecayAttn& a, cudaStream_t st) {
    const char* what = "fme_decay_attn_fwd";
    const Plan<T, D> P(a, fwd_ctas<T, D>());
    if (a.t == 0) return pass_on(what, a, a.s_in, a.s_out, st);
    if (!has_ws(a, P.ws_bytes())) return bad("decay attention: workspace too small or not aligned");
    if (P.pairs * P.W.segs > 0x7fffffff) return bad("decay attention: too many sequences");
    constexpr int NT = Shape<T, D>::NT;
    if (P.W.segs > 1) {
        int rc = go(what, k_attn_fwd<T, D, true, 2, local_ctas<T, D>()>, P.pairs * (P.W.segs - 1), NT, Plan<T, D>::LOCAL_FWD, st, a, P.W);
        if (rc || (rc = join(what, P.W, P.pairs, D * D, st))) return rc;
        if constexpr (D == 128) return go(what, k_attn_fwd<T, D, false, 2, 1>, P.pairs * P.W.segs, NT, Plan<T, D>::FWD + 3 * Shape<T, D>::TILE, st, a, P.W, true);
    }
    return go(what, k_attn_fwd<T, D, false, 1, fwd_ctas<T, D>()>, P.pairs * P.W.segs, NT, Plan<T, D>::FWD, st, a, P.W, P.W.segs > 1);
}
template <typename T, int D> int launch_bwd(const FmeDecayAttn& a, cudaStream_t st) {
    const char* what = "fme_decay_attn_bwd";
    const Plan<T, D> P(a, bwd_ctas<T, D>());
    if (a.t == 0) return pass_on(what, a, a.ds_out, a.ds_in, st);
    if (!has_ws(a, P.ws_bytes())) return bad("decay attention: workspace too small or not aligned");
    if (P.saved_bytes() && !a.saved) return bad("decay attention: the backward pass needs what the forward pass saved");
    if (P.pairs * P.W.segs > 0x7fffffff) return bad("decay attention: too many sequences");
    constexpr int NT = Shape<T, D>::NT;
    if (P.W.segs > 1) {
        int rc = go(what, k_attn_bwd<T, D, true, true, local_ctas<T, D>()>, P.pairs * (P.W.segs - 1), NT, Plan<T, D>::LOCAL_BWD, st, a, P.W);
        if (rc || (rc = join(what, P.W, P.pairs, D * D, st))) return rc;
    }
    if (a.ds_in) return go(what, k_attn_bwd<T, D, false, true, bwd_ctas<T, D>()>, P.pairs * P.W.segs, NT, Plan<T, D>::BWD, st, a, P.W, P.W.segs > 1);
    return go(what, k_attn_bwd<T, D, false, false, bwd_ctas<T, D>()>, P.pairs * P.W.segs, NT, Plan<T, D>::BWD, st, a, P.W, P.W.segs > 1);
}
template <typename T, int D> int launch_step(const FmeDecayAttn& a, cudaStream_t st) {
    k_attn_step<T, D><<<a.n * a.h, STEP_THREADS, 0, st>>>(a);
    return launch_status("fme_decay_attn_step");
}
template <typename T, int D> int64_t sizes(const FmeDecayAttn& a, int which) {
    const Plan<T, D> P(a, which == 1 ? bwd_ctas<T, D>() : fwd_ctas<T, D>());
    return which == 2 ? P.saved_bytes() : P.ws_bytes();
}
#define FME_BY_TYPE(a, FN, arg)                                                                                              \
    ((a).dtype == FME_F32 ? ((a).d == 32 ? FN<float, 32>(a, arg) : (a).d == 64 ? FN<float, 64>(a, arg) : FN<float, 128>(a, arg)) \
                          : ((a).d == 32 ? FN<bf16, 32>(a, arg) : (a).d == 64 ? FN<bf16, 64>(a, arg) : FN<bf16, 128>(a, arg)))

}  // namespace
}  // namespace fme

using namespace fme;

extern "C" {

int64_t fme_decay_attn_bytes(const FmeDecayAttn* a, int32_t which) {
    const int rc = check_sizes(a);
    if (rc) return rc;
    if (which < 0 || which > 2) return bad("decay attention: which must be 0, 1 or 2");
    return FME_BY_TYPE(*a, sizes, which);
}

int fme_decay_attn_fwd(const FmeDecayAttn* a, void* stream) {
    const int rc = check_common(a);
    if (rc) return rc;
    if (a->n == 0) return FME_OK;
    if (a->t && !rows_aligned(a->o, a->dtype)) return bad("decay attention: o must be given, with 16-byte aligned rows");
    return FME_BY_TYPE(*a, launch_fwd, (cudaStream_t)stream);
}

int fme_decay_attn_bwd(const FmeDecayAttn* a, void* stream) {
    const int rc = check_common(a);
    if (rc) return rc;
    if (a->n == 0) return FME_OK;
    if (a->t && (!rows_aligned(a->d_o, a->dtype) || !rows_aligned(a->dq, a->dtype) || !rows_aligned(a->dk, a->dtype) ||
                 !rows_aligned(a->dv, a->dtype)))
        return bad("decay attention: the gradients must be given, with 16-byte aligned rows");
    return FME_BY_TYPE(*a, launch_bwd, (cudaStream_t)stream);
}

int fme_decay_attn_step(const FmeDecayAttn* a, void* stream) {
    const int rc = check_common(a);
    if (rc) return rc;
    if (a->t != 1) return bad("decay attention step: t must be 1");
    if (a->n == 0) return FME_OK;
    if (!a->s_in || !a->s_out) return bad("decay attention step: s_in and s_out are required");
    if (!rows_aligned(a->o, a->dtype)) return bad("decay attention: o must be given, with 16-byte aligned rows");
    return FME_BY_TYPE(*a, launch_step, (cudaStream_t)stream);
}

}  // extern "C"

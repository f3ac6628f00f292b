// Linear attention with a decay for each head (gfx950 / CDNA4, wave64):
//   S_t = g S_(t-1) + k_t^T v_t,   o_t = scale * q_t S_t,   S [dk][dv] in f32.

#include <climits>

#include <algorithm>

#include "split.h"
#include "ops.h"

namespace zjai {

namespace {

__device__ __forceinline__ long long lin_at(const LinRows& r, int width, long long s, int t) {
    const long long base = s * r.seq;
    if (width == 0) return base + t * r.pos;
    const int y = t / width;
    return base + y * r.row + (t - y * width) * r.pos;
}

// The recurrent form. A workgroup owns 4 << cl_log2 value columns of one (sequence, head): a thread
// keeps 4 columns of the NR key rows rg, rg + RG, .. (RG = 256 >> cl_log2) in registers over the
// positions, so a state is read and written once however many positions there are. q and k of a
// position go through LDS as f32; the outputs are summed over the row groups by lane exchanges and LDS.
// Bandwidth and latency: the state's and the first position's loads are all issued before anything waits.
template <typename T, bool V4, int NR>
__global__ void __launch_bounds__(256) k_linear_recurrent(LinAttnArgs a, int cl_log2, int tiles) {
    __shared__ float s_k[256], s_q[256];
    __shared__ f32x4 s_o[4][32];
    __shared__ int s_next;
    const int tid = threadIdx.x, cl = 1 << cl_log2, RG = 256 >> cl_log2;
    const int tile = blockIdx.x % tiles, b = blockIdx.x / tiles;
    const int head = b % a.heads, first = b / a.heads;
    const int col = (tile * cl + (tid & (cl - 1))) * 4, rg = tid >> cl_log2;
    int slot = first;
    if (a.slots) {
        slot = a.slots[first];
        if ((unsigned)slot >= (unsigned)a.num_slots) return;
    }
    const long long sbase = ((long long)slot * a.heads + head) * a.dk;
    f32x4 S[NR];
#pragma unroll
    for (int n = 0; n < NR; ++n) S[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    if (a.s_in) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int r = rg + n * RG;
            if (V4) {
                if (r < a.dk && col < a.dv) S[n] = *(const f32x4*)(a.s_in + (sbase + r) * a.dv + col);
            } else {  // a row and columns that exist, zeros in the place of others afterwards (a branch for each value
                      // took 2304 registers to private memory: 200 states of 16 heads of 64 x 66 1166 us, now 41)
                const float* p = a.s_in + (sbase + min(r, a.dk - 1)) * a.dv;
#pragma unroll
                for (int c = 0; c < 4; ++c) S[n][c] = p[min(col + c, a.dv - 1)];
            }
        }
        if (!V4)
#pragma unroll
            for (int n = 0; n < NR; ++n)
#pragma unroll
                for (int c = 0; c < 4; ++c) S[n][c] = rg + n * RG < a.dk && col + c < a.dv ? S[n][c] : 0.0f;
    }
    // A position's channels: a thread loads one of k or q and its four value columns. (Absent ones: a channel that
    // exists, not used.)
    const int c = tid & 127;
    T kq, v[4];
    const auto fetch = [&](int seq, int t) {
        const LinRows& src = tid < 128 ? a.k : a.q;
        kq = ((const T*)src.p)[lin_at(src, a.width, seq, t) + (long long)head * a.dk + (c < a.dk ? c : 0)];
        const T* vp = (const T*)a.v.p + lin_at(a.v, a.width, seq, t) + (long long)head * a.dv;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = vp[col + e < a.dv ? col + e : 0];
    };
    int len = a.lengths ? max(0, min(a.lengths[first], a.length)) : a.length;
    if (len > 0) fetch(first, 0);
    const float g = a.decay[head];
    s_k[tid] = s_q[tid] = 0.0f;  // rows past dk
    // Sequences of one slot follow one another: the first of them takes them all, in order.
    int next = INT_MAX;
    if (a.slots && a.seqs > 1) {
        if (tid == 0) s_next = INT_MAX;
        __syncthreads();
        int earlier = 0, later = INT_MAX;
        for (int j = tid; j < a.seqs; j += 256)
            if (a.slots[j] == slot) {
                earlier |= j < first;
                if (j > first) later = min(later, j);
            }
        if (later != INT_MAX) atomicMin(&s_next, later);
        if (__syncthreads_or(earlier)) return;
        next = s_next;
    }
    for (int cur = first;;) {
        for (int t = 0; t < len; ++t) {
            __syncthreads();
            if (c < a.dk) (tid < 128 ? s_k : s_q)[c] = to_f32(kq);
            float vf[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) vf[e] = to_f32(v[e]);
            if (t + 1 < len) fetch(cur, t + 1);
            __syncthreads();
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const float kk = s_k[(rg + n * RG) & 255], qq = s_q[(rg + n * RG) & 255];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    S[n][e] = fmaf(g, S[n][e], kk * vf[e]);
                    o[e] = fmaf(qq, S[n][e], o[e]);
                }
            }
            for (int off = cl; off < 64; off <<= 1)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], off);
            if ((tid & 63) < cl) s_o[tid >> 6][tid & 63] = o;
            __syncthreads();
            if (tid < cl) {
                T* op = (T*)a.o.p + lin_at(a.o, a.width, cur, t) + (long long)head * a.dv + col;
                const f32x4 y = (s_o[0][tid] + s_o[1][tid]) + (s_o[2][tid] + s_o[3][tid]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < a.dv) op[e] = from_f32<T>(y[e] * a.scale);
            }
        }
        if (next == INT_MAX) break;
        cur = next;
        fetch(cur, 0);
        __syncthreads();
        if (tid == 0) s_next = INT_MAX;
        __syncthreads();
        for (int j = cur + 1 + tid; j < a.seqs; j += 256)
            if (a.slots[j] == slot) {
                atomicMin(&s_next, j);
                break;
            }
        __syncthreads();
        next = s_next;
    }
    if (a.s_out) {
#pragma unroll
        for (int n = 0; n < NR; ++n) {
            const int r = rg + n * RG;
            if (r >= a.dk) continue;
            float* p = a.s_out + (sbase + r) * a.dv + col;
            if (V4) {
                if (col < a.dv) *(f32x4*)p = S[n];
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (col + e < a.dv) p[e] = S[n][e];
            }
        }
    }
}

struct RecurrentPlan {
    int cl_log2, tiles, nr;
    bool v4;
};
RecurrentPlan recurrent_plan(const LinAttnArgs& a) {
    RecurrentPlan p{};
    // Whole rows up to 128 columns: 512 bytes at a time instead of 256 took 257 sequences of 16 heads of 128 x 128 from
    // 170 to 111 us (4.9 TB/s).
    while (p.cl_log2 < 5 && (4 << p.cl_log2) < a.dv) ++p.cl_log2;
    p.tiles = (a.dv + (4 << p.cl_log2) - 1) / (4 << p.cl_log2);
    const int rg = 256 >> p.cl_log2;
    p.nr = 1;
    while (p.nr * rg < a.dk) p.nr *= 2;
    p.v4 = a.dv % 4 == 0 && (((uintptr_t)a.s_in | (uintptr_t)a.s_out) & 15) == 0;
    return p;
}

template <typename T, bool V4>
void recurrent_nr(const LinAttnArgs& a, const RecurrentPlan& p, hipStream_t s) {
    const dim3 grid((unsigned)(p.tiles * a.heads * a.seqs));
    switch (p.nr) {
        case 1: k_linear_recurrent<T, V4, 1><<<grid, 256, 0, s>>>(a, p.cl_log2, p.tiles); break;
        case 2: k_linear_recurrent<T, V4, 2><<<grid, 256, 0, s>>>(a, p.cl_log2, p.tiles); break;
        case 4: k_linear_recurrent<T, V4, 4><<<grid, 256, 0, s>>>(a, p.cl_log2, p.tiles); break;
        case 8: k_linear_recurrent<T, V4, 8><<<grid, 256, 0, s>>>(a, p.cl_log2, p.tiles); break;
        default: k_linear_recurrent<T, V4, 16><<<grid, 256, 0, s>>>(a, p.cl_log2, p.tiles);
    }
}
template <typename T>
hipError_t recurrent(const LinAttnArgs& a, hipStream_t s) {
    const RecurrentPlan p = recurrent_plan(a);
    if (p.v4) recurrent_nr<T, true>(a, p, s);
    else recurrent_nr<T, false>(a, p, s);
    return hipGetLastError();
}

const char* type_name(int dtype) { return dtype == DT_F32 ? "float" : dtype == DT_F16 ? "_Float16" : "__bf16"; }

// ------------------------------------------------------------------------------ chunked form
//
// 32 positions at a time, with the state S before them, i, j = 0..31 within the chunk:
//   o_i = scale * ( g^(i+1) q_i S + sum_{j<=i} g^(i-j) (q_i . k_j) v_j )
//   S  <- g^32 S + sum_j k_j^T (g^(31-j) v_j)
// all four products on MFMAs with f32 accumulators. A unit is one head's up to D = 32, 64 or 128 key channels by
// D value channels (wider values are several units), a workgroup each; a wave keeps the state of 16 (or 32)
// of its value columns in registers, as MFMA accumulators. Every operand comes from the accumulator layout
// itself or from LDS rows of one position: an accumulator tile holds rows 4 g + r of a column in lane
// group g, so two tiles under one another are the K slots {4 g + r, 16 + 4 g + r} of the next product's
// operand, and the other operand is read in the same order (q stored so, k^T and v through the
// transposing LDS read).
//
// f32 runs on the f32 MFMAs (16x16x4; the same slots, one register at a time). The 16-bit types run on
// 16x16x32 MFMAs, q.k on the stored values themselves. What is computed in f32 enters the matrix cores in pieces:
//  - the query products and the state, in front of an output that is rounded to 16 bits, as two bf16
//    pieces (2^-16 of them; bf16 has f32's range, which f16 q.k or states can leave), and so do the f16
//    values they meet (exactly: 11 bits), in all four products: the smallest is up to 2^-14 of the term where the
//    first pieces are cut off, always of its sign (three products: 65536 f16 positions 553 us instead of 573);
//  - the weighted values g^(31-j) v_j, which the state's f32 sums are made of, as three bf16 pieces (exactly), and the
//    f16 keys they meet as two (exactly); of the six products the smallest is left out (2^-24). (Weighted values
//    below 2^-110 lose low bits.) Two f16
//    pieces of a weighted value are two products instead of five (12 ragged sequences of 64 x 128 channels 72 us
//    instead of 81, 65536 positions of 16 heads of 128 447 instead of 547), but end at 2^-36, where a decay
//    of a half is after a chunk: a value that zeros follow is then lost from the state.
constexpr int LC = 32;

__device__ u32x4 g_lin_zero[2];  // zeros: the source of absent positions and channels

// log2 g to a few units in its last place, also for g next to 1, where log2f has the places of 1 (a memory of a
// million positions takes them): there ln g = 2 atanh s, s = (g - 1) / (g + 1), by its series to s^15 (|s| <= 1/3).
__device__ __forceinline__ float lin_log2(float g) {
    if (!(g >= 0.5f)) return log2f(g);
    const float s = (g - 1.0f) * __builtin_amdgcn_rcpf(g + 1.0f), z = s * s;
    float p = 1.0f / 15.0f;
    p = fmaf(p, z, 1.0f / 13.0f);
    p = fmaf(p, z, 1.0f / 11.0f);
    p = fmaf(p, z, 1.0f / 9.0f);
    p = fmaf(p, z, 1.0f / 7.0f);
    p = fmaf(p, z, 1.0f / 5.0f);
    p = fmaf(p, z, 1.0f / 3.0f);
    p = fmaf(p, z, 1.0f);
    return s * p * 2.88539008177792681472f;
}
// g^n for n >= 0, l2 = log2 g (-inf for g = 0).
__device__ __forceinline__ float lin_pow(float l2, int n) { return n == 0 ? 1.0f : exp2f((float)n * l2); }

// LDS rows: 16-bit ones are padded by 32 bytes, which puts the 16 rows of a b128 fragment read (q) and the 8 rows by 2
// units of a transposing read (k, v) on distinct banks; f32 ones by 16, which does it for rows r and
// r + 4 of a column read and all but a pair of the rows of a b128 read. (An XOR by row has no conflicts at
// all, but every address is then an instruction and a register of its own.)
template <typename T> __host__ __device__ constexpr int lin_row(int d) { return d + (sizeof(T) == 4 ? 4 : 16); }

// The bf16 pieces of eight values: p0 cut off (so that a finite value's is finite) or, for values of f16's range
// (ROUND), rounded as the others.
template <int N, bool ROUND = false>
__device__ __forceinline__ void lin_split(const float (&x)[8], u32x4 (&p)[N]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const unsigned a = __builtin_bit_cast(unsigned, x[2 * h]), b = __builtin_bit_cast(unsigned, x[2 * h + 1]);
        p[0][h] = ROUND ? pack_bf16(x[2 * h], x[2 * h + 1]) : __builtin_amdgcn_perm(b, a, 0x07060302);
        if (N == 1) continue;
        const unsigned ta = ROUND ? p[0][h] << 16 : a & 0xffff0000u, tb = ROUND ? p[0][h] & 0xffff0000u : b & 0xffff0000u;
        float ra = x[2 * h] - __builtin_bit_cast(float, ta), rb = x[2 * h + 1] - __builtin_bit_cast(float, tb);
#pragma unroll
        for (int n = 1; n < N; ++n) {
            p[n][h] = pack_bf16(ra, rb);
            ra -= __builtin_bit_cast(float, p[n][h] << 16);
            rb -= __builtin_bit_cast(float, p[n][h] & 0xffff0000u);
        }
    }
}

// Sums of matrix products, the tiles of an instruction group given as pairs (c, a, b), over the products of pieces (all
// of them but the smallest of an f16 key's and a weighted value's), the small ones first (zero: the sums start here, a
// constant where this is inlined). Inline assembly with the accumulators in place: the compiler renames the builtin's chains
// back to back. A block carries its own wait states, as split.h's.
#define LM(MF, c, a, b) MF "%[c" #c "], %[a" #a "], %[b" #b "], %[c" #c "]\n\t"
#define LZ(MF, c, a, b) MF "%[c" #c "], %[a" #a "], %[b" #b "], 0\n\t"
#define LIN_LIST(...) __VA_ARGS__
#define LIN_ASM(PRODUCTS_ZERO, PRODUCTS, OUT_ZERO, OUT, ...)                          \
    if (zero) asm("s_nop 1\n\t" PRODUCTS_ZERO : LIN_LIST OUT_ZERO : __VA_ARGS__);     \
    else asm("s_nop 1\n\t" PRODUCTS : LIN_LIST OUT : __VA_ARGS__);
#define LIN_F16 "v_mfma_f32_16x16x32_f16 "
#define LIN_F32 "v_mfma_f32_16x16x4_f32 "
#define LIN_F32_WAIT "s_nop 9"

// pt[j][i] += k[j] q[i] on the stored values: the three tiles that have a position of the past in them.
#define L3(X, MF) X(MF, 00, 0, 0) X(MF, 01, 0, 1) X(MF, 11, 1, 1)
#define LO3 ([c00] "=&v"(c[0][0]), [c01] "=&v"(c[0][1]), [c11] "=&v"(c[1][1]))
#define LC3 ([c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c11] "+v"(c[1][1]))
template <bool F16>
__device__ __forceinline__ void lin_scores(f32x4 (&c)[2][2], const u32x4 (&a)[2], const u32x4 (&b)[2], bool zero) {
    if constexpr (F16) {
        LIN_ASM(L3(LZ, LIN_F16) ZJAI_WAIT, L3(LM, LIN_F16) ZJAI_WAIT, LO3, LC3, [a0] "v"(a[0]), [a1] "v"(a[1]), [b0] "v"(b[0]), [b1] "v"(b[1]))
    } else {
        LIN_ASM(L3(LZ, ZJAI_MF) ZJAI_WAIT, L3(LM, ZJAI_MF) ZJAI_WAIT, LO3, LC3, [a0] "v"(a[0]), [a1] "v"(a[1]), [b0] "v"(b[0]), [b1] "v"(b[1]))
    }
}
#define L3R(X, r) X(LIN_F32, 00, 0##r, 0##r) X(LIN_F32, 01, 0##r, 1##r) X(LIN_F32, 11, 1##r, 1##r)
#define LA4(n) [a##n##0] "v"(a[n][0]), [a##n##1] "v"(a[n][1]), [a##n##2] "v"(a[n][2]), [a##n##3] "v"(a[n][3])
#define LB4(n) [b##n##0] "v"(b[n][0]), [b##n##1] "v"(b[n][1]), [b##n##2] "v"(b[n][2]), [b##n##3] "v"(b[n][3])
__device__ __forceinline__ void lin_scores_f32(f32x4 (&c)[2][2], const f32x4 (&a)[2], const f32x4 (&b)[2], bool zero) {
    LIN_ASM(L3R(LZ, 0) L3R(LM, 1) L3R(LM, 2) L3R(LM, 3) LIN_F32_WAIT, L3R(LM, 0) L3R(LM, 1) L3R(LM, 2) L3R(LM, 3) LIN_F32_WAIT, LO3, LC3,
            LA4(0), LA4(1), LB4(0), LB4(1))
}

// One of those tiles.
template <bool F16>
__device__ __forceinline__ void lin_score(f32x4& c, const u32x4& a, const u32x4& b, bool zero) {
    if constexpr (F16) {
        LIN_ASM(LZ(LIN_F16, 0, 0, 0) ZJAI_WAIT, LM(LIN_F16, 0, 0, 0) ZJAI_WAIT, ([c0] "=&v"(c)), ([c0] "+v"(c)), [a0] "v"(a), [b0] "v"(b))
    } else {
        LIN_ASM(LZ(ZJAI_MF, 0, 0, 0) ZJAI_WAIT, LM(ZJAI_MF, 0, 0, 0) ZJAI_WAIT, ([c0] "=&v"(c)), ([c0] "+v"(c)), [a0] "v"(a), [b0] "v"(b))
    }
}

// o[n][i] += a[n] b[i]: tiles of the state or of the values (one or two to a wave) with the queries or their products.
#define LO1(X, MF, p, q) X(MF, 00, 0##p, 0##q) X(MF, 01, 0##p, 1##q)
#define LO2(X, MF, p, q) LO1(X, MF, p, q) X(MF, 10, 1##p, 0##q) X(MF, 11, 1##p, 1##q)
#define OZ1 ([c00] "=&v"(c[0][0]), [c01] "=&v"(c[0][1]))
#define OZ2 ([c00] "=&v"(c[0][0]), [c01] "=&v"(c[0][1]), [c10] "=&v"(c[1][0]), [c11] "=&v"(c[1][1]))
#define OC1 ([c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]))
#define OC2 ([c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1]))
#define A1(p) [a0##p] "v"(a[0][p])
#define A2(p) A1(p), [a1##p] "v"(a[1][p])
#define B1(q) [b0##q] "v"(b[0][q])
#define B2(q) B1(q), [b1##q] "v"(b[1][q])
#define LIN_OUT(L, OZ, OC, A)                                                                                                   \
    if constexpr (NA == 1) {                                                                                                    \
        static_assert(NB == 2, "piece products");                                                                               \
        LIN_ASM(L(LZ, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, L(LM, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, OZ, OC, A(0), \
                B2(0), B2(1))                                                                                                   \
    } else if constexpr (NB == 1) {                                                                                             \
        LIN_ASM(L(LZ, ZJAI_MF, 1, 0) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, L(LM, ZJAI_MF, 1, 0) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, OZ, OC, A(0), \
                A(1), B2(0))                                                                                                    \
    } else {                                                                                                                    \
        LIN_ASM(L(LZ, ZJAI_MF, 1, 1) L(LM, ZJAI_MF, 1, 0) L(LM, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT,                  \
                L(LM, ZJAI_MF, 1, 1) L(LM, ZJAI_MF, 1, 0) L(LM, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, OZ, OC, A(0), A(1), \
                B2(0), B2(1))                                                                                                   \
    }
template <int NV, int NA, int NB>
__device__ __forceinline__ void lin_outputs(f32x4 (&c)[NV][2], const u32x4 (&a)[NV][NA], const u32x4 (&b)[2][NB], bool zero = false) {
    if constexpr (NV == 1) {
        LIN_OUT(LO1, OZ1, OC1, A1)
    } else {
        LIN_OUT(LO2, OZ2, OC2, A2)
    }
}
#define R4(L, X) L(X, LIN_F32, 0, 0) L(LM, LIN_F32, 1, 1) L(LM, LIN_F32, 2, 2) L(LM, LIN_F32, 3, 3) LIN_F32_WAIT
template <int NV>
__device__ __forceinline__ void lin_outputs_f32(f32x4 (&c)[NV][2], const f32x4 (&a)[NV], const f32x4 (&b)[2], bool zero = false) {
    if constexpr (NV == 1) {
        LIN_ASM(R4(LO1, LZ), R4(LO1, LM), OZ1, OC1, A1(0), A1(1), A1(2), A1(3), LB4(0), LB4(1))
    } else {
        LIN_ASM(R4(LO2, LZ), R4(LO2, LM), OZ2, OC2, A2(0), A2(1), A2(2), A2(3), LB4(0), LB4(1))
    }
}
// c += a b: one tile.
#define LL(X, MF, p, q) X(MF, 0, p, q)
__device__ __forceinline__ void lin_tile_f32(f32x4& c, const f32x4& a, const f32x4& b, bool zero = false) {
    LIN_ASM(R4(LL, LZ), R4(LL, LM), ([c0] "=&v"(c)), ([c0] "+v"(c)), [a0] "v"(a[0]), [a1] "v"(a[1]), [a2] "v"(a[2]), [a3] "v"(a[3]),
            [b0] "v"(b[0]), [b1] "v"(b[1]), [b2] "v"(b[2]), [b3] "v"(b[3]))
}

// c[m][n] += a[m] b[n]: two key tiles of the state.
#define LS1(X, MF, p, q) X(MF, 00, 0##p, 0##q) X(MF, 10, 1##p, 0##q)
#define LS2(X, MF, p, q) LS1(X, MF, p, q) X(MF, 01, 0##p, 1##q) X(MF, 11, 1##p, 1##q)
#define SZ1 ([c00] "=&v"(c[0][0]), [c10] "=&v"(c[1][0]))
#define SZ2 ([c00] "=&v"(c[0][0]), [c10] "=&v"(c[1][0]), [c01] "=&v"(c[0][1]), [c11] "=&v"(c[1][1]))
#define SC1 ([c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]))
#define SC2 ([c00] "+v"(c[0][0]), [c10] "+v"(c[1][0]), [c01] "+v"(c[0][1]), [c11] "+v"(c[1][1]))
// `a` is the keys or the first piece of them (b's three pieces) or the second (b's two largest).
#define LIN_STATE(L, SZ, SC, B)                                                                                                       \
    if constexpr (NB == 3) {                                                                                                          \
        LIN_ASM(L(LZ, ZJAI_MF, 0, 2) L(LM, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT,                                             \
                L(LM, ZJAI_MF, 0, 2) L(LM, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, SZ, SC, A2(0), B(0), B(1), B(2))            \
    } else {                                                                                                                          \
        LIN_ASM(L(LZ, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, L(LM, ZJAI_MF, 0, 1) L(LM, ZJAI_MF, 0, 0) ZJAI_WAIT, SZ, SC, A2(0), B(0), B(1)) \
    }
template <int NB, int NV>
__device__ __forceinline__ void lin_state(f32x4 (&c)[2][NV], const u32x4 (&a)[2][1], const u32x4 (&b)[NV][3], bool zero) {
    if constexpr (NV == 1) {
        LIN_STATE(LS1, SZ1, SC1, B1)
    } else {
        LIN_STATE(LS2, SZ2, SC2, B2)
    }
}
template <int NV>
__device__ __forceinline__ void lin_state_f32(f32x4 (&c)[2][NV], const f32x4 (&a)[2], const f32x4 (&b)[NV], bool zero) {
    if constexpr (NV == 1) {
        LIN_ASM(R4(LS1, LZ), R4(LS1, LM), SZ1, SC1, LA4(0), LA4(1), LB4(0))
    } else {
        LIN_ASM(R4(LS2, LZ), R4(LS2, LM), SZ2, SC2, LA4(0), LA4(1), LB4(0), LB4(1))
    }
}
#undef LIN_STATE
#undef SC2
#undef SC1
#undef SZ2
#undef SZ1
#undef LS2
#undef LS1
#undef LL
#undef R4
#undef LIN_OUT
#undef B2
#undef B1
#undef A2
#undef A1
#undef OC2
#undef OC1
#undef OZ2
#undef OZ1
#undef LO2
#undef LO1
#undef LB4
#undef LA4
#undef L3R
#undef LC3
#undef LO3
#undef L3
#undef LIN_ASM
#undef LIN_LIST
#undef LZ
#undef LM

// Eight channels of one position as loaded.
template <typename T> struct alignas(16) LinUnit { u32x4 v[sizeof(T) / 2]; };

// Channels 8 u .. 8 u + 7 of a head at `p` (d channels), zeros where absent. VEC: whole 16-byte loads.
template <typename T>
__device__ __forceinline__ LinUnit<T> lin_load(const T* p, int c0, int d, bool valid, bool vec) {
    LinUnit<T> r;
    constexpr int E = 16 / sizeof(T);
    if (vec) {
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            const u32x4* q = valid && c0 + h * E < d ? (const u32x4*)(p + c0 + h * E) : g_lin_zero;
            r.v[h] = *q;
        }
    } else {
        typedef T tE __attribute__((ext_vector_type(E)));
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            tE x;
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = valid && c0 + h * E + e < d ? p[c0 + h * E + e] : (T)0.0f;
            r.v[h] = __builtin_bit_cast(u32x4, x);
        }
    }
    return r;
}

// Eight f16 or bf16 values as f32.
template <typename T>
__device__ __forceinline__ void lin_floats(const u32x4& v, float (&x)[8]) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 t = __builtin_bit_cast(t8, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)t[e];
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// Transposing read: the 16 lanes of a group pass the addresses of a 4 x 16 block of 16-bit values, row (lane / 4) and
// columns 4 (lane % 4); lane n gets the four values of column n.
__device__ __forceinline__ u32x2 lds_tr(const unsigned short* p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p));
}

struct LinChunkArgs {
    LinAttnArgs a;
    float* scratch;  // sums: the state after each segment; outputs: before each but the first
    int segments, seg_len, units, tiles;
    int slots;  // states of a sequence in it: one for each segment but the last and, in place, the state before the first
    int vec_k, vec_v, vec_o;
    int even;  // vec_k and vec_v, and head sizes of whole units
};

// 16-bit planes of a chunk in LDS: k, v and, for outputs, q; f16's k and q in two pieces, for outputs as they are too.
template <typename T> __host__ __device__ constexpr int lin_lds_planes(bool out) {
    return sizeof(T) == 4 ? (out ? 6 : 4) : Elem<T>::dt == DT_F16 ? (out ? 7 : 3) : (out ? 3 : 2);
}

// D: channels of a unit; a wave has one 16-column tile of its values or, for the outputs of the widest, two: with
// eight waves to a unit instead of four, what the waves share and the barriers between so many cost more than the
// registers of one tile less give (65536 positions, 16 heads, bf16: 451 us, with two tiles 408; held to 128
// registers 526). The sums have no query products, and more waves load more (two tiles 150 us, one 113).
constexpr int lin_tiles(int d, bool out) { return out && d == 128 ? 2 : 1; }
constexpr int lin_waves(int d, bool out) { return d / 16 / lin_tiles(d, out); }
template <typename T, int D, bool OUT>
__global__ void __launch_bounds__(64 * lin_waves(D, OUT), !OUT ? 4 : D == 128 ? 2 : 3) k_linear_chunks(LinChunkArgs c) {
    constexpr bool F32 = sizeof(T) == 4, F16 = Elem<T>::dt == DT_F16;
    constexpr int NV = lin_tiles(D, OUT);
    constexpr int ROW = lin_row<T>(D), PLANE = LC * ROW;  // LDS values of a position and of a chunk of q, k or v
    constexpr int MT = D / 16, KS = D / 32;
    constexpr int QP = F16 ? 2 : 1;           // bf16 pieces of a 16-bit q, k or v
    extern __shared__ __attribute__((aligned(16))) unsigned short s_lds[];  // [lin_lds_planes][PLANE], then 64 WV floats
    const LinAttnArgs& a = c.a;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, l16 = lane & 15, g = lane >> 4;
    unsigned short* s_k = s_lds;
    unsigned short* s_v = s_k + (F32 || (F16 && !OUT) ? 2 : 1) * PLANE;
    unsigned short* s_q = s_v + (F32 ? 2 : 1) * PLANE;           // f16: the values, then their two pieces
    unsigned short* s_kp = F16 && OUT ? s_q + 3 * PLANE : s_k;  // the keys that the state's products take
    float *f_k = (float*)s_k, *f_v = (float*)s_v, *f_q = (float*)s_q;

    // Workgroups go round the eight XCDs. The units of a segment share cache lines of the positions' channels and are
    // put on one XCD, the segments dealt out one by one (a contiguous share of the sequences to an XCD
    // leaves some with the long ones); with fewer segments than XCDs, units are dealt out instead.
    const int segs = OUT ? c.segments : c.segments - 1, spread = a.seqs * segs >= 8 ? 8 : 1;
    const int b = blockIdx.x / spread, part = b / c.units * spread + blockIdx.x % spread;
    const int unit = b % c.units, seg = part % segs, seq = part / segs;
    if (seq >= a.seqs) return;
    const int len = a.lengths ? max(0, min(a.lengths[seq], a.length)) : a.length;
    const int begin = seg * c.seg_len, end = min(len, begin + c.seg_len);
    // Sums are those that a later segment starts from.
    if (OUT ? begin > len || (begin == len && seg > 0) : begin + c.seg_len >= len) return;
    const int head = unit / c.tiles, col0 = unit % c.tiles * D;
    const int colw = col0 + wave * 16 * NV;   // the wave's value columns
    // Four waves share the query products: each of three makes one tile of them, weighed and in pieces, in LDS, at the
    // price of one more barrier a chunk (12 ragged f16 sequences of 64 channels 87 -> 83 us, 65536 positions of 128
    // bf16 channels 422 -> 411 us). The two waves of 32 channels would save half a tile's work each and make their own.
    constexpr bool SHARE = OUT && D > 32;
    const bool work = SHARE || colw < a.dv;

    const T* kp = (const T*)a.k.p + (long long)seq * a.k.seq + (long long)head * a.dk;
    const T* vp = (const T*)a.v.p + (long long)seq * a.v.seq + (long long)head * a.dv + col0;
    const T* qp = OUT ? (const T*)a.q.p + (long long)seq * a.q.seq + (long long)head * a.dk : nullptr;
    T* op = OUT ? (T*)a.o.p + (long long)seq * a.o.seq + (long long)head * a.dv + colw : nullptr;
    const int vcols = a.dv - col0;

    // A thread stages NV units of eight channels of each matrix: positions row0 (and row0 + 16), unit u.
    constexpr int UPR = D / 8;
    const int row0 = t / UPR, u = t % UPR;
    LinUnit<T> rk[NV], rv[NV], rq[NV];
    // Whole chunks of evenly strided rows: running pointers, those of absent channels on zeros that stay put.
    const bool even = a.width == 0 && c.even;
    const bool on_k = u * 8 < a.dk, on_v = u * 8 < vcols;
    const T *pk[NV], *pv[NV], *pq[NV];
    constexpr int STEP = OUT ? LC : -LC;
    const long long step_k = on_k ? STEP * a.k.pos : 0, step_v = on_v ? STEP * a.v.pos : 0, step_q = on_k ? STEP * a.q.pos : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const long long p = (OUT ? begin : end - LC) + row0 + i * 16;
        pk[i] = on_k ? kp + p * a.k.pos + u * 8 : (const T*)g_lin_zero;
        pv[i] = on_v ? vp + p * a.v.pos + u * 8 : (const T*)g_lin_zero;
        pq[i] = OUT && on_k ? qp + p * a.q.pos + u * 8 : (const T*)g_lin_zero;
    }
    const auto fetch = [&](int pos) {
        if (even && pos + LC <= end) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                rk[i] = *(const LinUnit<T>*)pk[i];
                rv[i] = *(const LinUnit<T>*)pv[i];
                if (OUT) rq[i] = *(const LinUnit<T>*)pq[i];
                pk[i] += step_k;
                pv[i] += step_v;
                pq[i] += step_q;
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int p = pos + row0 + i * 16;
            const bool ok = p < end;
            const int y = a.width ? p / a.width : 0, x = a.width ? p - y * a.width : p;
            rk[i] = lin_load<T>(kp + (y * a.k.row + x * a.k.pos), u * 8, a.dk, ok, c.vec_k);
            rv[i] = lin_load<T>(vp + (y * a.v.row + x * a.v.pos), u * 8, vcols, ok, c.vec_v);
            if (OUT) rq[i] = lin_load<T>(qp + (y * a.q.row + x * a.q.pos), u * 8, a.dk, ok, c.vec_k);
        }
    };
    // Outputs go forward. Sums go backward, from the segment's last chunk to its first: the part of k and v that the
    // outputs begin with is then what the last-level cache has seen last.
    if (begin < end) fetch(OUT ? begin : end - LC);

    // The head's powers g^0..g^63, one a lane, then those a lane's rows and columns need.
    float* s_pow = (float*)(s_lds + lin_lds_planes<T>(OUT) * PLANE) + wave * 64;
    u32x4* s_p = (u32x4*)((float*)(s_lds + lin_lds_planes<T>(OUT) * PLANE) + lin_waves(D, OUT) * 64);
    if (SHARE && !F32 && wave == 0) s_p[lane] = s_p[64 + lane] = u32x4{0, 0, 0, 0};  // products with later positions
    s_pow[lane] = lin_pow(lin_log2(a.decay[head]), lane);
    __syncthreads();
    float w_v[8], w_o[2], w_d[4], w_n[4], g_c = s_pow[LC];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        w_v[r] = s_pow[LC - 1 - (4 * g + r)];
        w_v[4 + r] = s_pow[LC - 1 - (16 + 4 * g + r)];
        const int d = l16 - (4 * g + r);
        w_d[r] = s_pow[max(d, 0)] * a.scale;
        w_n[r] = s_pow[16 + d] * a.scale;
    }
    w_o[0] = s_pow[l16 + 1] * a.scale;
    w_o[1] = s_pow[l16 + 17] * a.scale;

    // The state before the segment: S[m][n][r] is key channel 16 m + 4 g + r of value column 16 n + l16.
    f32x4 S[MT][NV];
    // Where it is in the caller's arrays: the row by scalar arithmetic (one that exists), the lane's part added.
    const long long sbase = ((long long)seq * a.heads + head) * a.dk;
    const auto s_row = [&](int row) { return (sbase + min(row, a.dk - 1)) * a.dv + col0; };
    const unsigned s_lane = 4 * g * a.dv + colw - col0 + l16;
    const size_t xunit = (size_t)D * D;
    float* const x_seq = c.scratch + ((size_t)seq * c.slots * c.units + unit) * xunit + (size_t)(wave * NV * 64 + lane) * 4;
    const size_t x_seg = c.units * xunit;
    const float g_seg = OUT ? 1.0f : lin_pow(lin_log2(a.decay[head]), c.seg_len);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < NV; ++n) S[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // In place, the workgroup of a sequence's last segment writes the states that the first one's outputs start from,
    // and nothing orders the two: the sums, a launch before, keep a copy of them. (A sequence of one segment
    // is read and written by the same lanes.)
    const bool copied = a.s_in && a.s_in == a.s_out && len > c.seg_len;
    // One branch for all tiles, so that their loads are issued together (a branch for each: 16 waits one after
    // another for 128 channels; six positions with states 14.4 us, now 11.6).
    if (OUT && (seg > 0 || copied)) {
        const int slot = seg > 0 ? seg - 1 : c.segments - 1;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NV; ++n) S[m][n] = *(const f32x4*)(x_seq + slot * x_seg + (m * (D / 16) + n) * 256);
    } else if (seg == 0 && a.s_in && work) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = 16 * m + 4 * g + r < a.dk && colw + 16 * n + l16 < a.dv;
                    S[m][n][r] = a.s_in[s_row(16 * m + r) + (in ? s_lane + 16 * n : 0)];
                }
        int keys = a.dk, values = a.dv;  // compared again: 64 masks kept over the loads leave no scalar registers
        asm("" : "+s"(keys), "+s"(values));
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const bool in = 16 * m + 4 * g + r < keys && colw + 16 * n + l16 < values;
                    S[m][n][r] = in ? S[m][n][r] : 0.0f;
                }
        if (!OUT) {
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    if (copied) *(f32x4*)(x_seq + (c.segments - 1) * x_seg + (m * (D / 16) + n) * 256) = S[m][n];
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[m][n][r] *= g_seg;
                }
        }
    }

    const auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int row = row0 + i * 16;
            if constexpr (F32) {
                const int at = row * ROW + u * 8;
                *(u32x4*)(f_k + at) = rk[i].v[0];
                *(u32x4*)(f_k + at + 4) = rk[i].v[1];
                *(u32x4*)(f_v + at) = rv[i].v[0];
                *(u32x4*)(f_v + at + 4) = rv[i].v[1];
                if (OUT) {
                    *(u32x4*)(f_q + at) = rq[i].v[0];
                    *(u32x4*)(f_q + at + 4) = rq[i].v[1];
                }
            } else {
                if (OUT || !F16) *(u32x4*)(s_k + row * ROW + u * 8) = rk[i].v[0];
                if constexpr (F16) {
                    float x[8];
                    u32x4 p[2];
                    lin_floats<T>(rk[i].v[0], x);
                    lin_split<2, true>(x, p);
#pragma unroll
                    for (int n = 0; n < 2; ++n) *(u32x4*)(s_kp + n * PLANE + row * ROW + u * 8) = p[n];
                }
                *(u32x4*)(s_v + row * ROW + u * 8) = rv[i].v[0];
                if (OUT) {
                    // Channels 4 x of a 32-channel block go to unit x % 4, half x / 4.
                    unsigned short* q0 = s_q + row * ROW + ((u & ~3) + 2 * (u & 1)) * 8 + ((u >> 1) & 1) * 4;
                    const u32x4 v = rq[i].v[0];
                    *(u32x2*)q0 = u32x2{v[0], v[1]};
                    *(u32x2*)(q0 + 8) = u32x2{v[2], v[3]};
                    if constexpr (F16) {
                        float x[8];
                        u32x4 p[2];
                        lin_floats<T>(v, x);
                        lin_split<2>(x, p);
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            *(u32x2*)(q0 + (n + 1) * PLANE) = u32x2{p[n][0], p[n][1]};
                            *(u32x2*)(q0 + 8 + (n + 1) * PLANE) = u32x2{p[n][2], p[n][3]};
                        }
                    }
                }
            }
        }
    };

    T* po = OUT && a.width == 0 ? op + (begin + l16) * a.o.pos : op;  // the output of position pos + l16
    float ahead = 1.0f;  // sums: g^(positions of the segment after this chunk)
    for (int pos = OUT ? begin : end - LC; OUT ? pos < end : pos >= begin; pos += STEP) {
        __syncthreads();
        stage();
        __syncthreads();
        const int nv = min(LC, end - pos);
        if (OUT ? pos + LC < end : pos > begin) fetch(pos + STEP);
        if (!work) continue;

        const bool last = pos + LC >= end;
        const bool update = !OUT || !last || (end == len && a.s_out);
        if (update && nv < LC) {  // the last chunk of a state that is kept: weights from its own end
            g_c = s_pow[nv];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w_v[r] = s_pow[max(0, nv - 1 - (4 * g + r))];
                w_v[4 + r] = s_pow[max(0, nv - 1 - (16 + 4 * g + r))];
            }
        }
        // Transposing reads of 16-bit rows 4 g + r (and 16 + 4 g + r): the lane's part of the address.
        const int tbase = (4 * g + (l16 >> 2)) * ROW + (l16 & 3) * 4;
        const auto column16 = [&](const unsigned short* m, int un) {
            const unsigned short* p = m + tbase + un * 8;
            const u32x2 lo = lds_tr(p), hi = lds_tr(p + 16 * ROW);
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        };
        // Column col of f32 rows 16 t + 4 g + r.
        const auto column32 = [&](const float* m, int col, int t) {
            f32x4 x;
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = m[(16 * t + 4 * g + r) * ROW + col];
            return x;
        };

        // The wave's value columns 16 n + l16 at positions j = {4 g + r, 16 + 4 g + r}, and their weighted pieces.
        float x[NV][8], w[NV][8], big = 0.0f;
        u32x4 wv[NV][3];
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            const int col = wave * NV + n;
            if constexpr (F32) {
                const f32x4 t0 = column32(f_v, col * 16 + l16, 0), t1 = column32(f_v, col * 16 + l16, 1);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[n][r] = t0[r], x[n][4 + r] = t1[r];
            } else {
                lin_floats<T>(column16(s_v, col * 2), x[n]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                big = __builtin_elementwise_maximum(big, __builtin_fabsf(x[n][e]));
                w[n][e] = x[n][e] * w_v[e];
            }
            if constexpr (!F32) lin_split<3>(w[n], wv[n]);
        }

        if (OUT) {
            // A value that is infinite or NaN is left out of the products, where it would meet the zero
            // weights of the positions before it, and put on the others afterwards.
            const bool poison = __builtin_amdgcn_ballot_w64(!(big <= FLT_MAX)) != 0;
            int first[NV];
            if (poison) {
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    first[n] = LC;
#pragma unroll
                    for (int e = 7; e >= 0; --e)
                        if (!(__builtin_fabsf(x[n][e]) <= FLT_MAX)) {
                            first[n] = (e >> 2) * 16 + 4 * g + (e & 3);
                            x[n][e] = 0.0f;
                        }
                    first[n] = min(first[n], __shfl_xor(first[n], 16));
                    first[n] = min(first[n], __shfl_xor(first[n], 32));
                }
            }
            f32x4 O[NV][2];  // O[n][i], transposed: rows are value columns 16 n + 4 g + r, columns positions 16 i + l16
            f32x4 pt[2][2];  // pt[j][i]: rows are positions j of the keys, columns positions i of the queries
            const auto weighed = [&](const f32x4& t, int j, int i) {
                f32x4 p;
#pragma unroll
                for (int r = 0; r < 4; ++r)  // a select: products with later positions may be infinite
                    p[r] = j != i ? t[r] * w_n[r] : 4 * g + r <= l16 ? t[r] * w_d[r] : 0.0f;
                return p;
            };
            if constexpr (SHARE) {
                const int j = wave == 2, i = wave >= 1;
                if (wave < 3) {
                    f32x4 tile;
#pragma unroll
                    for (int s = 0; s < (F32 ? MT : KS); ++s) {
                        if constexpr (F32) {
                            lin_tile_f32(tile, *(const f32x4*)(f_k + (16 * j + l16) * ROW + (4 * s + g) * 4),
                                         *(const f32x4*)(f_q + (16 * i + l16) * ROW + (4 * s + g) * 4), s == 0);
                        } else {
                            const unsigned short* kr = s_k + (16 * j + l16) * ROW + 32 * s + 4 * g;
                            const u32x2 k_lo = *(const u32x2*)kr, k_hi = *(const u32x2*)(kr + 16);
                            lin_score<F16>(tile, u32x4{k_lo[0], k_lo[1], k_hi[0], k_hi[1]},
                                           *(const u32x4*)(s_q + (16 * i + l16) * ROW + (4 * s + g) * 8), s == 0);
                        }
                    }
                    const f32x4 p = weighed(tile, j, i);
                    if constexpr (F32) {
                        s_p[wave * 64 + lane] = __builtin_bit_cast(u32x4, p);
                    } else {
                        const float z[8] = {p[0], p[1], p[2], p[3], 0.0f, 0.0f, 0.0f, 0.0f};
                        u32x4 q[2];
                        lin_split<2>(z, q);
#pragma unroll
                        for (int n = 0; n < 2; ++n) ((u32x2*)(s_p + (2 * i + n) * 64 + lane))[j] = u32x2{q[n][0], q[n][1]};
                    }
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int s = 0; s < MT; ++s) {
                    f32x4 kf[2], qf[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = (16 * i + l16) * ROW + (4 * s + g) * 4;
                        if (!SHARE) kf[i] = *(const f32x4*)(f_k + at);
                        qf[i] = *(const f32x4*)(f_q + at);
                    }
                    if (!SHARE) lin_scores_f32(pt, kf, qf, s == 0);
                    lin_outputs_f32<NV>(O, S[s], qf, s == 0);
                }
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 qf[2], qp[2][QP], kf[2], sf[NV][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const unsigned short* qr = s_q + (16 * i + l16) * ROW + (4 * s + g) * 8;
                        const unsigned short* kr = s_k + (16 * i + l16) * ROW + 32 * s + 4 * g;
                        if (!SHARE || !F16) qf[i] = *(const u32x4*)qr;
#pragma unroll
                        for (int n = 0; n < QP; ++n) qp[i][n] = F16 ? *(const u32x4*)(qr + (n + 1) * PLANE) : qf[i];
                        if (!SHARE) {
                            const u32x2 k_lo = *(const u32x2*)kr, k_hi = *(const u32x2*)(kr + 16);
                            kf[i] = u32x4{k_lo[0], k_lo[1], k_hi[0], k_hi[1]};
                        }
                    }
#pragma unroll
                    for (int n = 0; n < NV; ++n) {
                        float z[8];
#pragma unroll
                        for (int r = 0; r < 4; ++r) z[r] = S[2 * s][n][r], z[4 + r] = S[2 * s + 1][n][r];
                        lin_split<2>(z, sf[n]);
                    }
                    if (!SHARE) lin_scores<F16>(pt, kf, qf, s == 0);
                    lin_outputs<NV>(O, sf, qp, s == 0);
                }
            }
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[n][i][r] *= w_o[i];
            // The weighed query products of positions 16 i + l16 with the positions j.
            if (SHARE) __syncthreads();
            if constexpr (F32) {
                f32x4 p[2], p11;
                if constexpr (SHARE) {
                    p[0] = __builtin_bit_cast(f32x4, s_p[lane]);
                    p[1] = __builtin_bit_cast(f32x4, s_p[64 + lane]);
                    p11 = __builtin_bit_cast(f32x4, s_p[128 + lane]);
                } else {
                    p[0] = weighed(pt[0][0], 0, 0);
                    p[1] = weighed(pt[0][1], 0, 1);
                    p11 = weighed(pt[1][1], 1, 1);
                }
                f32x4 early[NV];
#pragma unroll
                for (int n = 0; n < NV; ++n) early[n] = f32x4{x[n][0], x[n][1], x[n][2], x[n][3]};
                lin_outputs_f32<NV>(O, early, p);
#pragma unroll
                for (int n = 0; n < NV; ++n) lin_tile_f32(O[n][1], f32x4{x[n][4], x[n][5], x[n][6], x[n][7]}, p11);
            } else {
                u32x4 vf[NV][QP], P[2][2];
#pragma unroll
                for (int n = 0; n < NV; ++n) lin_split<QP>(x[n], vf[n]);
                if constexpr (SHARE) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) P[i >> 1][i & 1] = s_p[i * 64 + lane];
                } else {
                    const f32x4 p00 = weighed(pt[0][0], 0, 0), p01 = weighed(pt[0][1], 0, 1), p11 = weighed(pt[1][1], 1, 1);
                    const float z0[8] = {p00[0], p00[1], p00[2], p00[3], 0.0f, 0.0f, 0.0f, 0.0f};
                    const float z1[8] = {p01[0], p01[1], p01[2], p01[3], p11[0], p11[1], p11[2], p11[3]};
                    lin_split<2>(z0, P[0]);
                    lin_split<2>(z1, P[1]);
                }
                lin_outputs<NV>(O, vf, P);
            }
            if (poison) {
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int from = __shfl(first[n], 4 * g + r);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            if (16 * i + l16 >= from) O[n][i][r] = __builtin_nanf("");
                    }
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int p = pos + 16 * i + l16;
                if (p >= end) continue;
                T* o = po + i * 16 * a.o.pos;
                if (a.width) {
                    const int y = p / a.width;
                    o = op + (y * a.o.row + (p - y * a.width) * a.o.pos);
                }
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    const int cc = 16 * n + 4 * g;
                    if (c.vec_o) {
                        if (colw + cc < a.dv) store4<T>(o + cc, O[n][i]);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (colw + cc + r < a.dv) o[cc + r] = from_f32<T>(O[n][i][r]);
                    }
                }
            }
        }
        if (OUT && a.width == 0) po += LC * a.o.pos;
        if (!update) continue;
#pragma unroll
        for (int m = 0; m < MT; m += 2) {
            f32x4 acc[2][NV];
            if (OUT)
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int n = 0; n < NV; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[h][n][r] = S[m + h][n][r] * g_c;
            if constexpr (F32) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const f32x4 kt[2] = {column32(f_k, 16 * m + l16, i), column32(f_k, 16 * m + 16 + l16, i)};
                    f32x4 vt[NV];
#pragma unroll
                    for (int n = 0; n < NV; ++n) vt[n] = f32x4{w[n][4 * i], w[n][4 * i + 1], w[n][4 * i + 2], w[n][4 * i + 3]};
                    lin_state_f32<NV>(acc, kt, vt, !OUT && i == 0);
                }
            } else {
                if constexpr (F16) {
                    const u32x4 kt[2][1] = {{column16(s_kp + PLANE, 2 * m)}, {column16(s_kp + PLANE, 2 * m + 2)}};
                    lin_state<2, NV>(acc, kt, wv, !OUT);
                }
                const u32x4 kt[2][1] = {{column16(s_kp, 2 * m)}, {column16(s_kp, 2 * m + 2)}};
                lin_state<3, NV>(acc, kt, wv, !OUT && !F16);
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < NV; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) S[m + h][n][r] = OUT ? acc[h][n][r] : fmaf(ahead, acc[h][n][r], S[m + h][n][r]);
        }
        if (!OUT) ahead *= g_c;
    }

    if (OUT) {
        if (!a.s_out || end != len || !work) return;
#pragma unroll
        for (int n = 0; n < NV; ++n) {
            if (colw + 16 * n + l16 >= a.dv) continue;
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * m + 4 * g + r < a.dk) a.s_out[s_row(16 * m + r) + s_lane + 16 * n] = S[m][n][r];
        }
    } else {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < NV; ++n) *(f32x4*)(x_seq + seg * x_seg + (m * (D / 16) + n) * 256) = S[m][n];
    }
}

// The state before segment s + 1 from the segments' own sums: E_(s+1) = g^seg_len E_s + X_s, in place (E_1 = X_0).
// A thread holds sixteen segments of one f32x4, all loaded at once; the threads of the other sixteens join
// theirs in LDS, so that a scan is one round of loads and one of stores however many segments there are
// (64 segments of 5 states of 32 x 32: 7.2 us one sixteen after another).
constexpr int SCAN_SEGS = 16;
__global__ void __launch_bounds__(1024) k_linear_scan(LinChunkArgs c, int quads, int width) {
    __shared__ f32x4 s_total[1024];
    const int lane = threadIdx.x % width, part = threadIdx.x / width, q = blockIdx.x * width + lane;
    const int unit = blockIdx.y % c.units, seq = blockIdx.y / c.units;
    const float g = lin_pow(lin_log2(c.a.decay[unit / c.tiles]), c.seg_len);
    // A sequence has the sums of its segments but the last.
    const int len = c.a.lengths ? max(0, min(c.a.lengths[seq], c.a.length)) : c.a.length, sums = max(len - 1, 0) / c.seg_len;
    if (sums < 2) return;
    const int s0 = part * SCAN_SEGS, n = sums - s0;
    f32x4* x = (f32x4*)c.scratch + (((size_t)seq * c.slots + s0) * c.units + unit) * quads + q;
    const size_t step = (size_t)c.units * quads;
    f32x4 v[SCAN_SEGS];
#pragma unroll
    for (int k = 0; k < SCAN_SEGS; ++k) v[k] = x[k < n ? k * step : 0];
#pragma unroll
    for (int k = 1; k < SCAN_SEGS; ++k)
#pragma unroll
        for (int r = 0; r < 4; ++r) v[k][r] = fmaf(g, v[k - 1][r], v[k][r]);
    s_total[threadIdx.x] = v[SCAN_SEGS - 1];
    __syncthreads();
    float f = g;
#pragma unroll
    for (int k = 1; k < SCAN_SEGS; k *= 2) f *= f;  // g^16
    f32x4 e = {0.0f, 0.0f, 0.0f, 0.0f};  // the state before this thread's segments
    for (int p = 0; p < part; ++p) {
        const f32x4 t = s_total[p * width + lane];
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = fmaf(f, e[r], t[r]);
    }
#pragma unroll
    for (int k = 0; k < SCAN_SEGS; ++k) {
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] *= g;
        if (k < n) x[k * step] = v[k] + e;
    }
}

LinChunkArgs chunk_args(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, float* scratch) {
    LinChunkArgs c{};
    c.a = a;
    c.scratch = scratch;
    c.segments = p.segments;
    c.seg_len = p.seg_len;
    c.slots = p.slots;
    c.units = p.units;
    c.tiles = p.units / a.heads;
    const int es = dtype == DT_F32 ? 4 : 2;
    const auto aligned = [&](const LinRows& r, int d, int bytes) {
        const int e = bytes / es;
        return ((uintptr_t)r.p & (bytes - 1)) == 0 && r.seq % e == 0 && r.pos % e == 0 && r.row % e == 0 && d % e == 0;
    };
    c.vec_k = aligned(a.k, a.dk, 16) && aligned(a.q, a.dk, 16);
    c.vec_v = aligned(a.v, a.dv, 16);
    c.vec_o = aligned(a.o, a.dv, 4 * es);
    c.even = c.vec_k && c.vec_v && a.dk % 8 == 0 && a.dv % 8 == 0;
    return c;
}

template <typename T, int D, bool OUT>
void chunks_d(const LinChunkArgs& c, const dim3& grid, hipStream_t s) {
    constexpr int threads = 64 * lin_waves(D, OUT);
    const size_t lds = lin_lds_planes<T>(OUT) * LC * lin_row<T>(D) * 2 + threads * 4 + (OUT && D > 32 ? 4 * 64 * 16 : 0);
    k_linear_chunks<T, D, OUT><<<grid, threads, lds, s>>>(c);
}
template <typename T, bool OUT>
hipError_t chunks(const LinChunkArgs& c, int width, hipStream_t s) {
    const long long parts = (long long)c.a.seqs * (OUT ? c.segments : c.segments - 1);
    const dim3 grid((unsigned)((parts >= 8 ? (parts + 7) / 8 * 8 : parts) * c.units));
    if (width == 32) chunks_d<T, 32, OUT>(c, grid, s);
    else if (width == 64) chunks_d<T, 64, OUT>(c, grid, s);
    else chunks_d<T, 128, OUT>(c, grid, s);
    return hipGetLastError();
}
template <bool OUT>
hipError_t chunks_of(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, float* scratch, hipStream_t s) {
    const LinChunkArgs c = chunk_args(a, p, dtype, scratch);
    if (dtype == DT_F32) return chunks<float, OUT>(c, p.width, s);
    if (dtype == DT_F16) return chunks<_Float16, OUT>(c, p.width, s);
    return chunks<__bf16, OUT>(c, p.width, s);
}

}  // namespace

std::string linear_recurrent_name(const LinAttnArgs& a, int dtype) {
    const RecurrentPlan p = recurrent_plan(a);
    return std::string("k_linear_recurrent<") + type_name(dtype) + (p.v4 ? ", true, " : ", false, ") + std::to_string(p.nr) + ">";
}

hipError_t launch_linear_recurrent(const LinAttnArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return recurrent<float>(a, s);
    if (dtype == DT_F16) return recurrent<_Float16>(a, s);
    return recurrent<__bf16>(a, s);
}

// A position takes the recurrent form 0.7 to 3 us, a chunk costs its 32 positions whether they are there or not, but a
// state is read and written faster by the recurrent form (both, us: one f32 sequence of 4 heads of 32, no
// states: 3 positions 4.8 and 4.8, 4 5.6 and 4.9; with states 4 5.7 and 6.2, 6 7.2 and 6.2; 500 f16 sequences of
// 4 heads of 32 x 64 with states: 5 16.2 and 19.2, 6 18.2 and 19.3; 64 bf16 ones of 16 heads of 128: 5 38.0 and 39.6,
// 6 41.2 and 39.4; 500 f16 ones of 8 heads of 64 without: 3 16.1 and 22.2, 6 27.6 and 22.4).
bool linear_prefers_recurrent(const LinAttnArgs& a) { return a.length <= (a.s_in || a.s_out ? 5 : 3); }

LinChunkPlan linear_chunk_plan(const LinAttnArgs& a, size_t scratch_bytes) {
    LinChunkPlan p;
    p.width = a.dk <= 32 ? 32 : a.dk <= 64 ? 64 : 128;
    p.units = a.heads * ((a.dv + p.width - 1) / p.width);
    const long long waves = (long long)a.seqs * p.units * (p.width / 32), chunks = (a.length + LC - 1) / LC;
    const long long state = (long long)a.seqs * p.units * p.width * p.width * 4;
    // A wave for every SIMD needs no segments (2160 waves of 240 positions: 16.6 us, in two segments 22.4). With
    // fewer, k and v are read twice, and two waves to a SIMD pay for it (65536 positions, 64 waves: in 16 segments
    // 490 us, in 32 404); with lengths, half of the segments may be empty (12 ragged sequences of up to 3001: six
    // segments 90 us, eleven 83). A segment has at least as many bytes of channels as of state: 4096 positions in
    // five heads of 32, f32: one chunk a segment 16.4 us, two 17.5. The context's 33 MiB hold what 2048 waves ask for;
    // ragged batches of the widest heads get half of theirs (in 80 MiB, 12 sequences of up to 3001 in eight heads
    // of 128, f16: 139 us instead of 136; 6 of up to 9000 150 instead of 183, 30 of up to 4000 360 instead of 343).
    const long long want = waves >= 1024 ? 1 : ((a.lengths ? 4096 : 2048) + waves - 1) / waves;
    const int kept = a.s_in && a.s_in == a.s_out;  // states updated in place have a copy in the scratch
    const long long n = std::max(std::min(std::min(std::min(want, 1024LL), chunks * 32 / p.width), (long long)(scratch_bytes / state) + 1 - kept), 1LL);
    const long long per = std::max((chunks + n - 1) / n, 1LL);
    p.seg_len = (int)(per * LC);
    p.segments = (int)std::max((chunks + per - 1) / per, 1LL);
    p.slots = p.segments - 1 + kept;
    return p;
}

std::string linear_chunk_name(const LinChunkPlan& p, int dtype, bool outputs) {
    return std::string("k_linear_chunks<") + type_name(dtype) + ", " + std::to_string(p.width) + (outputs ? ", true>" : ", false>");
}

hipError_t launch_linear_sums(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, float* scratch, hipStream_t s) {
    return chunks_of<false>(a, p, dtype, scratch, s);
}
hipError_t launch_linear_scan(const LinAttnArgs& a, const LinChunkPlan& p, float* scratch, hipStream_t s) {
    const int quads = p.width * p.width / 4, parts = (p.segments - 1 + SCAN_SEGS - 1) / SCAN_SEGS;
    int width = 64;
    while (width * parts > 1024) width /= 2;
    k_linear_scan<<<dim3((unsigned)(quads / width), (unsigned)(a.seqs * p.units)), width * parts, 0, s>>>(chunk_args(a, p, DT_F32, scratch), quads, width);
    return hipGetLastError();
}
hipError_t launch_linear_outputs(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, const float* scratch, hipStream_t s) {
    return chunks_of<true>(a, p, dtype, const_cast<float*>(scratch), s);
}

}  // namespace zjai

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
    for (int n = 0; n < NR; ++n) {
        const int r = rg + n * RG;
        S[n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (a.s_in && r < a.dk) {
            const float* p = a.s_in + (sbase + r) * a.dv + col;
            if (V4) {
                if (col < a.dv) S[n] = *(const f32x4*)p;
            } else {
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    if (col + c < a.dv) S[n][c] = p[c];
            }
        }
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
    const dim3 grid((unsigned)linear_recurrent_groups(a));
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
// all four products on 16x16x32 bf16 MFMAs with f32 accumulators. A unit is one head's up to 32 WV key
// channels by 32 WV value channels (wider values are several units), the work of WV waves, each with the
// state of 32 value columns in registers as MFMA accumulators; a workgroup of four waves holds 4 / WV
// units of one stretch of a sequence. Every operand comes from the accumulator layout itself or from
// LDS rows of one position: an accumulator tile holds rows 4 g + r of a column in lane group g, so two
// tiles under one another are the K slots {4 g + r, 16 + 4 g + r} of the next product's operand, and
// the other operand is read in the same order (q stored so, k^T and v through the transposing LDS read).
//
// f32 runs on the f32 MFMAs (16x16x4; the same slots, one register at a time). The 16-bit types run on
// 16x16x32 MFMAs, q.k on the stored values themselves. What is computed in f32 enters the matrix cores in pieces:
//  - the query products and the state, in front of an output that is rounded to 16 bits, as two bf16
//    pieces (2^-16 of them; bf16 has f32's range, which f16 q.k or states can leave), and so do the f16
//    values they meet (exactly: 11 bits);
//  - the weighted values g^(31-j) v_j, which the state's f32 sums are made of, as three bf16 pieces next to
//    bf16 keys (exactly), and next to f16 keys as two f16 ones, the second times 2^11 in a sum of its own
//    (2^-23 of them; |g^n v| <= |v| stays in f16's range).
constexpr int LC = 32;

__device__ u32x4 g_lin_zero[2];  // zeros: the source of absent positions and channels

// g^n for n >= 0, l2 = log2 g (-inf for g = 0).
__device__ __forceinline__ float lin_pow(float l2, int n) { return n == 0 ? 1.0f : exp2f((float)n * l2); }

// LDS rows: 16-bit ones are padded by 32 bytes, which puts the 16 rows of a b128 fragment read (q) and the 8 rows by 2
// units of a transposing read (k, v) on distinct banks; f32 ones by 16, which does it for rows r and
// r + 4 of a column read and all but a pair of the rows of a b128 read. (An XOR by row has no conflicts at
// all, but every address is then an instruction and a register of its own.)
template <typename T> __host__ __device__ constexpr int lin_row(int d) { return d + (sizeof(T) == 4 ? 4 : 16); }

// The bf16 pieces of eight values: p0 cut off (so that a finite value's is finite), the others rounded.
template <int N>
__device__ __forceinline__ void lin_split(const float (&x)[8], u32x4 (&p)[N]) {
#pragma unroll
    for (int h = 0; h < 4; ++h) {
        const unsigned a = __builtin_bit_cast(unsigned, x[2 * h]), b = __builtin_bit_cast(unsigned, x[2 * h + 1]);
        p[0][h] = __builtin_amdgcn_perm(b, a, 0x07060302);
        if (N == 1) continue;
        float ra = x[2 * h] - __builtin_bit_cast(float, a & 0xffff0000u), rb = x[2 * h + 1] - __builtin_bit_cast(float, b & 0xffff0000u);
#pragma unroll
        for (int n = 1; n < N; ++n) {
            p[n][h] = pack_bf16(ra, rb);
            ra -= __builtin_bit_cast(float, p[n][h] << 16);
            rb -= __builtin_bit_cast(float, p[n][h] & 0xffff0000u);
        }
    }
}

// c[i][j] += a[i] b[j] over the products of pieces p + q <= 1 (up to 2 with three), the small ones first (two
// tiles of either operand; zero: the sums start here, a constant where this is inlined). Inline
// assembly with the accumulators in place: the compiler renames the builtin's chains back to back. The
// block carries its own wait states, as split.h's.
#define LM(MF, i, j, p, q) MF "%[c" #i #j "], %[a" #i #p "], %[b" #j #q "], %[c" #i #j "]\n\t"
#define LZ(MF, i, j, p, q) MF "%[c" #i #j "], %[a" #i #p "], %[b" #j #q "], 0\n\t"
#define LM4(MF, p, q) LM(MF, 0, 0, p, q) LM(MF, 0, 1, p, q) LM(MF, 1, 0, p, q) LM(MF, 1, 1, p, q)
#define LZ4(MF, p, q) LZ(MF, 0, 0, p, q) LZ(MF, 0, 1, p, q) LZ(MF, 1, 0, p, q) LZ(MF, 1, 1, p, q)
#define LC4 [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1])
#define LO4 [c00] "=&v"(c[0][0]), [c01] "=&v"(c[0][1]), [c10] "=&v"(c[1][0]), [c11] "=&v"(c[1][1])
#define LA(p) [a0##p] "v"(a[0][p]), [a1##p] "v"(a[1][p])
#define LB(p) [b0##p] "v"(b[0][p]), [b1##p] "v"(b[1][p])
#define LIN_ASM(MF, WAIT, P, Q, REST, ...)                                              \
    if (zero) asm("s_nop 1\n\t" LZ4(MF, P, Q) REST WAIT : LO4 : __VA_ARGS__);            \
    else asm("s_nop 1\n\t" LM4(MF, P, Q) REST WAIT : LC4 : __VA_ARGS__);
template <int NA, int NB>
__device__ __forceinline__ void lin_mma(f32x4 (&c)[2][2], const u32x4 (&a)[2][NA], const u32x4 (&b)[2][NB], bool zero = false) {
    if constexpr (NA == 1 && NB == 1) {
        LIN_ASM(ZJAI_MF, ZJAI_WAIT, 0, 0, , LA(0), LB(0))
    } else if constexpr (NA == 1 && NB == 2) {
        LIN_ASM(ZJAI_MF, ZJAI_WAIT, 0, 1, LM4(ZJAI_MF, 0, 0), LA(0), LB(0), LB(1))
    } else if constexpr (NA == 2 && NB == 1) {
        LIN_ASM(ZJAI_MF, ZJAI_WAIT, 1, 0, LM4(ZJAI_MF, 0, 0), LA(0), LA(1), LB(0))
    } else if constexpr (NA == 1 && NB == 3) {
        LIN_ASM(ZJAI_MF, ZJAI_WAIT, 0, 2, LM4(ZJAI_MF, 0, 1) LM4(ZJAI_MF, 0, 0), LA(0), LB(0), LB(1), LB(2))
    } else {
        static_assert(NA == 2 && NB == 2, "piece products");
        LIN_ASM(ZJAI_MF, ZJAI_WAIT, 1, 0, LM4(ZJAI_MF, 0, 1) LM4(ZJAI_MF, 0, 0), LA(0), LA(1), LB(0), LB(1))
    }
}
#define LIN_F16 "v_mfma_f32_16x16x32_f16 "
__device__ __forceinline__ void lin_mma_f16(f32x4 (&c)[2][2], const u32x4 (&a)[2][1], const u32x4 (&b)[2][1], bool zero = false) {
    LIN_ASM(LIN_F16, ZJAI_WAIT, 0, 0, , LA(0), LB(0))
}
// The f32 form: sixteen (a tile's four K slots, one register each) or, with TRI, the twelve but c[1][0]'s.
#define LIN_F32 "v_mfma_f32_16x16x4_f32 "
#define LIN_F32_WAIT "s_nop 9"
#define LM3(MF, p, q) LM(MF, 0, 0, p, q) LM(MF, 0, 1, p, q) LM(MF, 1, 1, p, q)
template <bool TRI>
__device__ __forceinline__ void lin_mma_f32(f32x4 (&c)[2][2], const f32x4 (&a)[2], const f32x4 (&b)[2], bool zero = false) {
    if constexpr (TRI) {
        if (zero) c[0][0] = c[0][1] = c[1][0] = c[1][1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        asm("s_nop 1\n\t" LM3(LIN_F32, 0, 0) LM3(LIN_F32, 1, 1) LM3(LIN_F32, 2, 2) LM3(LIN_F32, 3, 3) LIN_F32_WAIT
            : [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c11] "+v"(c[1][1])
            : LA(0), LA(1), LA(2), LA(3), LB(0), LB(1), LB(2), LB(3));
    } else {
        LIN_ASM(LIN_F32, LIN_F32_WAIT, 0, 0, LM4(LIN_F32, 1, 1) LM4(LIN_F32, 2, 2) LM4(LIN_F32, 3, 3), LA(0), LA(1), LA(2), LA(3), LB(0),
                LB(1), LB(2), LB(3))
    }
}
// c[n] += a[n] b: the values of the later sixteen positions, which only the later sixteen queries see.
__device__ __forceinline__ void lin_mma_f32_late(f32x4& c0, f32x4& c1, const f32x4 (&a)[2], const f32x4& b) {
    asm("s_nop 1\n\t" LIN_F32 "%0, %2, %10, %0\n\t" LIN_F32 "%1, %6, %10, %1\n\t" LIN_F32 "%0, %3, %11, %0\n\t" LIN_F32
        "%1, %7, %11, %1\n\t" LIN_F32 "%0, %4, %12, %0\n\t" LIN_F32 "%1, %8, %12, %1\n\t" LIN_F32 "%0, %5, %13, %0\n\t" LIN_F32
        "%1, %9, %13, %1\n\t" LIN_F32_WAIT
        : "+v"(c0), "+v"(c1)
        : "v"(a[0][0]), "v"(a[0][1]), "v"(a[0][2]), "v"(a[0][3]), "v"(a[1][0]), "v"(a[1][1]), "v"(a[1][2]), "v"(a[1][3]), "v"(b[0]),
          "v"(b[1]), "v"(b[2]), "v"(b[3]));
}
#undef LM3
#undef LIN_ASM
#undef LB
#undef LA
#undef LO4
#undef LC4
#undef LZ4
#undef LM4
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

// An f16 pair of f32 values' halves.
__device__ __forceinline__ unsigned pack_f16(float a, float b) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    f16x2 r;
    r[0] = (_Float16)a;
    r[1] = (_Float16)b;
    return __builtin_bit_cast(unsigned, r);
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
    int vec_k, vec_v, vec_o;
    int even;  // vec_k and vec_v, and head sizes of whole units
};

// 16-bit planes of a chunk in LDS: k, v and, for outputs, q (f16's in pieces too).
template <typename T> __host__ __device__ constexpr int lin_lds_planes(bool out) {
    return sizeof(T) == 4 ? (out ? 6 : 4) : Elem<T>::dt == DT_F16 ? (out ? 5 : 2) : (out ? 3 : 2);
}

template <typename T, int WV, bool OUT>
__global__ void __launch_bounds__(256, 2) k_linear_chunks(LinChunkArgs c) {
    constexpr bool F32 = sizeof(T) == 4, F16 = Elem<T>::dt == DT_F16;
    constexpr int D = 32 * WV;
    constexpr int ROW = lin_row<T>(D), PLANE = LC * ROW;  // LDS values of a position and of a chunk of q, k or v
    constexpr int MT = D / 16, KS = D / 32;
    constexpr int QP = F16 ? 2 : 1;           // bf16 pieces of a 16-bit q or v
    extern __shared__ __attribute__((aligned(16))) unsigned short s_lds[];  // [lin_lds_planes][PLANE], then 64 WV floats
    const LinAttnArgs& a = c.a;
    const int t = threadIdx.x, wave = t >> 6, lane = t & 63, l16 = lane & 15, g = lane >> 4;
    unsigned short* s_k = s_lds;
    unsigned short* s_v = s_k + (F32 ? 2 : 1) * PLANE;
    unsigned short* s_q = s_v + (F32 ? 2 : 1) * PLANE;  // f16: the values, then their two pieces
    float *f_k = (float*)s_k, *f_v = (float*)s_v, *f_q = (float*)s_q;

    // Workgroups go round the eight XCDs; neighbours in (sequence, segment, unit) share cache lines of the
    // positions' channels and are put on one XCD.
    const int segs = OUT ? c.segments : c.segments - 1;
    int b = (blockIdx.x & 7) * (gridDim.x >> 3) + (blockIdx.x >> 3);
    const int unit = b % c.units;
    b /= c.units;
    const int seg = b % segs, seq = b / segs;
    if (seq >= a.seqs) return;
    const int len = a.lengths ? max(0, min(a.lengths[seq], a.length)) : a.length;
    const int begin = seg * c.seg_len, end = min(len, begin + c.seg_len);
    // Sums are those that a later segment starts from.
    if (OUT ? begin > len || (begin == len && seg > 0) : begin + c.seg_len >= len) return;
    const int head = unit / c.tiles, col0 = unit % c.tiles * D;
    const int colw = col0 + wave * 32;        // the wave's 32 value columns
    const bool work = colw < a.dv;

    const T* kp = (const T*)a.k.p + (long long)seq * a.k.seq + (long long)head * a.dk;
    const T* vp = (const T*)a.v.p + (long long)seq * a.v.seq + (long long)head * a.dv + col0;
    const T* qp = OUT ? (const T*)a.q.p + (long long)seq * a.q.seq + (long long)head * a.dk : nullptr;
    T* op = OUT ? (T*)a.o.p + (long long)seq * a.o.seq + (long long)head * a.dv + colw : nullptr;
    const int vcols = a.dv - col0;

    // A thread stages two units of eight channels of each matrix: rows row0 and row0 + 16, unit u.
    constexpr int UPR = D / 8;
    const int row0 = t / UPR, u = t % UPR;
    LinUnit<T> rk[2], rv[2], rq[2];
    // Whole chunks of evenly strided rows: running pointers, those of absent channels on zeros that stay put.
    const bool even = a.width == 0 && c.even;
    const bool on_k = u * 8 < a.dk, on_v = u * 8 < vcols;
    const T *pk[2], *pv[2], *pq[2];
    const long long step_k = on_k ? LC * a.k.pos : 0, step_v = on_v ? LC * a.v.pos : 0, step_q = on_k ? LC * a.q.pos : 0;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const long long p = begin + row0 + i * 16;
        pk[i] = on_k ? kp + p * a.k.pos + u * 8 : (const T*)g_lin_zero;
        pv[i] = on_v ? vp + p * a.v.pos + u * 8 : (const T*)g_lin_zero;
        if (OUT) pq[i] = on_k ? qp + p * a.q.pos + u * 8 : (const T*)g_lin_zero;
    }
    const auto fetch = [&](int pos) {
        if (even && pos + LC <= end) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                rk[i] = *(const LinUnit<T>*)pk[i];
                rv[i] = *(const LinUnit<T>*)pv[i];
                pk[i] += step_k;
                pv[i] += step_v;
                if (OUT) {
                    rq[i] = *(const LinUnit<T>*)pq[i];
                    pq[i] += step_q;
                }
            }
            return;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int p = pos + row0 + i * 16;
            const bool ok = p < end;
            const int y = a.width ? p / a.width : 0, x = a.width ? p - y * a.width : p;
            rk[i] = lin_load<T>(kp + (y * a.k.row + x * a.k.pos), u * 8, a.dk, ok, c.vec_k);
            rv[i] = lin_load<T>(vp + (y * a.v.row + x * a.v.pos), u * 8, vcols, ok, c.vec_v);
            if (OUT) rq[i] = lin_load<T>(qp + (y * a.q.row + x * a.q.pos), u * 8, a.dk, ok, c.vec_k);
        }
    };
    if (begin < end) fetch(begin);

    // The head's powers g^0..g^63, one a lane, then those a lane's rows and columns need.
    float* s_pow = (float*)(s_lds + lin_lds_planes<T>(OUT) * PLANE) + wave * 64;
    s_pow[lane] = lin_pow(log2f(a.decay[head]), lane);
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

    // The state before the segment: S[mt][n][r] is key channel 16 mt + 4 g + r of value column 16 n + l16.
    f32x4 S[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) S[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const long long sbase = ((long long)seq * a.heads + head) * a.dk;
    const size_t xunit = (size_t)D * D;
    float* const x_seq = c.scratch + ((size_t)seq * (c.segments - 1) * c.units + unit) * xunit + (size_t)(wave * 64 + lane) * 4;
    const size_t x_seg = c.units * xunit;
    if (seg == 0) {
        if (a.s_in && work)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int kk = 16 * m + 4 * g + r, vv = colw + 16 * n + l16;
                        const bool in = kk < a.dk && vv < a.dv;
                        const float x = a.s_in[in ? (sbase + kk) * a.dv + vv : 0];
                        S[m][n][r] = in ? x : 0.0f;
                    }
    } else if (OUT) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n) S[m][n] = *(const f32x4*)(x_seq + (seg - 1) * x_seg + (size_t)(m * 2 + n) * WV * 256);
    }

    const auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = row0 + i * 16;
            if constexpr (F32) {
                const int at = row * ROW, u0 = u * 8, u1 = u * 8 + 4;
                *(u32x4*)(f_k + at + u0) = rk[i].v[0];
                *(u32x4*)(f_k + at + u1) = rk[i].v[1];
                *(u32x4*)(f_v + at + u0) = rv[i].v[0];
                *(u32x4*)(f_v + at + u1) = rv[i].v[1];
                if (OUT) {
                    *(u32x4*)(f_q + at + u0) = rq[i].v[0];
                    *(u32x4*)(f_q + at + u1) = rq[i].v[1];
                }
            } else {
                const int kv = row * ROW + u * 8;
                *(u32x4*)(s_k + kv) = rk[i].v[0];
                *(u32x4*)(s_v + kv) = rv[i].v[0];
                if (OUT) {
                    // Channels 4 x of a 32-channel block go to unit x % 4, half x / 4.
                    const int unit0 = (u & ~3) + 2 * (u & 1), half = ((u >> 1) & 1) * 4;
                    unsigned short* q0 = s_q + row * ROW + unit0 * 8 + half;
                    unsigned short* q1 = q0 + 8;
                    const u32x4 v = rq[i].v[0];
                    *(u32x2*)q0 = u32x2{v[0], v[1]};
                    *(u32x2*)q1 = u32x2{v[2], v[3]};
                    if constexpr (F16) {
                        float x[8];
                        u32x4 p[2];
                        lin_floats<T>(v, x);
                        lin_split<2>(x, p);
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            *(u32x2*)(q0 + (n + 1) * PLANE) = u32x2{p[n][0], p[n][1]};
                            *(u32x2*)(q1 + (n + 1) * PLANE) = u32x2{p[n][2], p[n][3]};
                        }
                    }
                }
            }
        }
    };

    for (int pos = begin; pos < end; pos += LC) {
        __syncthreads();
        stage();
        __syncthreads();
        const int nv = min(LC, end - pos);
        if (pos + LC < end) fetch(pos + LC);
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

        // The wave's value columns 16 n + l16 at positions j, in the order of P, and their weighted pieces.
        float x[2][8];
        u32x4 wv[2][3], hi[2][1], lo[2][1];
        const auto weigh = [&]() {
            float w[2][8];
#pragma unroll
            for (int n = 0; n < 2; ++n) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    w[n][e] = x[n][e] * w_v[e];
                    // The product as it is rounded to f32: contracted into v_fma_mixlo_f16 (one rounding), what the second
                    // piece is the rest of would not always be the first.
                    if (F16) asm("" : "+v"(w[n][e]));
                }
                if constexpr (F32) {
                    wv[n][0] = __builtin_bit_cast(u32x4, f32x4{w[n][0], w[n][1], w[n][2], w[n][3]});
                    wv[n][1] = __builtin_bit_cast(u32x4, f32x4{w[n][4], w[n][5], w[n][6], w[n][7]});
                } else if constexpr (F16) {
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        const unsigned top = pack_f16(w[n][2 * h], w[n][2 * h + 1]);
                        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
                        const f16x2 p = __builtin_bit_cast(f16x2, top);
                        hi[n][0][h] = top;
                        lo[n][0][h] = pack_f16((w[n][2 * h] - (float)p[0]) * 2048.0f, (w[n][2 * h + 1] - (float)p[1]) * 2048.0f);
                    }
                } else {
                    lin_split<3>(w[n], wv[n]);
                }
            }
        };
        float big = 0.0f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            if constexpr (F32) {
                const f32x4 t0 = column32(f_v, wave * 32 + 16 * n + l16, 0), t1 = column32(f_v, wave * 32 + 16 * n + l16, 1);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[n][r] = t0[r], x[n][4 + r] = t1[r];
            } else {
                lin_floats<T>(column16(s_v, wave * 4 + 2 * n), x[n]);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) big = __builtin_elementwise_maximum(big, __builtin_fabsf(x[n][e]));
        }
        weigh();

        if (OUT) {
            // A value that is infinite or NaN is left out of the products, where it would meet the zero
            // weights of the positions before it, and put on the others afterwards.
            const bool poison = __builtin_amdgcn_ballot_w64(!(big <= FLT_MAX)) != 0;
            int first[2] = {LC, LC};
            if (poison) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
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
            f32x4 O[2][2];   // O[n][i], transposed: rows are value columns 16 n + 4 g + r, columns positions 16 i + l16
            f32x4 pt[2][2];  // pt[j][i]: rows are positions j of the keys, columns positions i of the queries
            if constexpr (F32) {
#pragma unroll
                for (int s = 0; s < MT; ++s) {
                    f32x4 kf[2], qf[2], sf[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int at = (16 * i + l16) * ROW + (4 * s + g) * 4;
                        kf[i] = *(const f32x4*)(f_k + at);
                        qf[i] = *(const f32x4*)(f_q + at);
                        sf[i] = S[s][i];
                    }
                    lin_mma_f32<true>(pt, kf, qf, s == 0);
                    lin_mma_f32<false>(O, sf, qf, s == 0);
                }
            } else {
#pragma unroll
                for (int s = 0; s < KS; ++s) {
                    u32x4 qf[2][1], qp[2][QP], kf[2][1], sf[2][2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const int row = 16 * i + l16;
                        const unsigned short* qr = s_q + row * ROW + (4 * s + g) * 8;
                        const unsigned short* k0 = s_k + row * ROW + 32 * s + 4 * g;
                        qf[i][0] = *(const u32x4*)qr;
#pragma unroll
                        for (int n = 0; n < QP; ++n) qp[i][n] = F16 ? *(const u32x4*)(qr + (n + 1) * PLANE) : qf[i][0];
                        const u32x2 k_lo = *(const u32x2*)k0, k_hi = *(const u32x2*)(k0 + 16);
                        kf[i][0] = u32x4{k_lo[0], k_lo[1], k_hi[0], k_hi[1]};
                        float z[8];
#pragma unroll
                        for (int r = 0; r < 4; ++r) z[r] = S[2 * s][i][r], z[4 + r] = S[2 * s + 1][i][r];
                        lin_split<2>(z, sf[i]);
                    }
                    if constexpr (F16) lin_mma_f16(pt, kf, qf, s == 0);
                    else lin_mma(pt, kf, qf, s == 0);
                    lin_mma(O, sf, qp, s == 0);
                }
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[n][i][r] *= w_o[i];
            // Weighted query products of positions 16 i + l16 with j = {4 g + r, 16 + 4 g + r}.
            float p0[8], p1[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool seen = 4 * g + r <= l16;  // a select: products with later positions may be infinite
                p0[r] = seen ? pt[0][0][r] * w_d[r] : 0.0f;
                p0[4 + r] = 0.0f;
                p1[r] = pt[0][1][r] * w_n[r];
                p1[4 + r] = seen ? pt[1][1][r] * w_d[r] : 0.0f;
            }
            if constexpr (F32) {
                const f32x4 early[2] = {{x[0][0], x[0][1], x[0][2], x[0][3]}, {x[1][0], x[1][1], x[1][2], x[1][3]}};
                const f32x4 late[2] = {{x[0][4], x[0][5], x[0][6], x[0][7]}, {x[1][4], x[1][5], x[1][6], x[1][7]}};
                const f32x4 p[2] = {{p0[0], p0[1], p0[2], p0[3]}, {p1[0], p1[1], p1[2], p1[3]}};
                lin_mma_f32<false>(O, early, p);
                lin_mma_f32_late(O[0][1], O[1][1], late, f32x4{p1[4], p1[5], p1[6], p1[7]});
            } else {
                u32x4 vf[2][QP], P[2][2];
#pragma unroll
                for (int n = 0; n < 2; ++n) lin_split<QP>(x[n], vf[n]);
                lin_split<2>(p0, P[0]);
                lin_split<2>(p1, P[1]);
                lin_mma(O, vf, P);
            }
            if (poison) {
#pragma unroll
                for (int n = 0; n < 2; ++n)
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
                const int row = a.width ? p / a.width : 0, at = a.width ? p - row * a.width : p;
                T* o = op + (row * a.o.row + at * a.o.pos);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int cc = 16 * n + 4 * g;
                    const f32x4 v = O[n][i];
                    if (c.vec_o) {
                        if (colw + cc < a.dv) store4<T>(o + cc, v);
                    } else {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (colw + cc + r < a.dv) o[cc + r] = from_f32<T>(v[r]);
                    }
                }
            }
        }
        if (!update) continue;
#pragma unroll
        for (int m = 0; m < MT; m += 2) {
            f32x4 acc[2][2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < 2; ++n)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[h][n][r] = S[m + h][n][r] * g_c;
            if constexpr (F32) {
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    const f32x4 kt[2] = {column32(f_k, 16 * m + l16, t), column32(f_k, 16 * m + 16 + l16, t)};
                    const f32x4 vt[2] = {__builtin_bit_cast(f32x4, wv[0][t]), __builtin_bit_cast(f32x4, wv[1][t])};
                    lin_mma_f32<false>(acc, kt, vt);
                }
            } else {
                const u32x4 kt[2][1] = {{column16(s_k, 2 * m)}, {column16(s_k, 2 * m + 2)}};
                if constexpr (F16) {
                    f32x4 small[2][2];
                    lin_mma_f16(acc, kt, hi);
                    lin_mma_f16(small, kt, lo, true);
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int n = 0; n < 2; ++n)
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[h][n][r] = fmaf(small[h][n][r], 0x1p-11f, acc[h][n][r]);
                } else {
                    lin_mma(acc, kt, wv);
                }
            }
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int n = 0; n < 2; ++n) S[m + h][n] = acc[h][n];
        }
    }

    if (OUT) {
        if (!a.s_out || end != len || !work) return;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int kk = 16 * m + 4 * g + r, vv = colw + 16 * n + l16;
                    if (kk < a.dk && vv < a.dv) a.s_out[(sbase + kk) * a.dv + vv] = S[m][n][r];
                }
    } else {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n) *(f32x4*)(x_seq + seg * x_seg + (size_t)(m * 2 + n) * WV * 256) = S[m][n];
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
    const float g = lin_pow(log2f(c.a.decay[unit / c.tiles]), c.seg_len);
    const int s0 = part * SCAN_SEGS, n = c.segments - 1 - s0;
    f32x4* x = (f32x4*)c.scratch + (((size_t)seq * (c.segments - 1) + s0) * c.units + unit) * quads + q;
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

template <typename T, int WV, bool OUT>
void chunks_wv(const LinChunkArgs& c, const dim3& grid, hipStream_t s) {
    const size_t lds = lin_lds_planes<T>(OUT) * LC * lin_row<T>(32 * WV) * 2 + WV * 64 * 4;
    k_linear_chunks<T, WV, OUT><<<grid, 64 * WV, lds, s>>>(c);
}
template <typename T, bool OUT>
hipError_t chunks(const LinChunkArgs& c, int width, hipStream_t s) {
    const dim3 grid((unsigned)(((long long)c.a.seqs * (OUT ? c.segments : c.segments - 1) * c.units + 7) / 8 * 8));
    if (width == 32) chunks_wv<T, 1, OUT>(c, grid, s);
    else if (width == 64) chunks_wv<T, 2, OUT>(c, grid, s);
    else chunks_wv<T, 4, OUT>(c, grid, s);
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

long long linear_recurrent_groups(const LinAttnArgs& a) { return (long long)recurrent_plan(a).tiles * a.heads * a.seqs; }

std::string linear_recurrent_name(const LinAttnArgs& a, int dtype) {
    const RecurrentPlan p = recurrent_plan(a);
    return std::string("k_linear_recurrent<") + type_name(dtype) + (p.v4 ? ", true, " : ", false, ") + std::to_string(p.nr) + ">";
}

hipError_t launch_linear_recurrent(const LinAttnArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return recurrent<float>(a, s);
    if (dtype == DT_F16) return recurrent<_Float16>(a, s);
    return recurrent<__bf16>(a, s);
}

bool linear_prefers_recurrent(const LinAttnArgs& a) { return a.length <= 8; }

LinChunkPlan linear_chunk_plan(const LinAttnArgs& a, size_t scratch_bytes) {
    LinChunkPlan p;
    p.width = a.dk <= 32 ? 32 : a.dk <= 64 ? 64 : 128;
    p.units = a.heads * ((a.dv + p.width - 1) / p.width);
    const long long waves = (long long)a.seqs * p.units * (p.width / 32), chunks = (a.length + LC - 1) / LC;
    const long long state = (long long)a.seqs * p.units * p.width * p.width * 4;
    // A wave for every SIMD needs no segments (1080 waves of 240 positions: 21.6 us, in two segments 26.8). With
    // fewer, k and v are read twice, and two waves to a SIMD pay for it (65536 positions, 64 waves: in 16 segments
    // 636 us, in 32 434). A segment of one chunk costs more in states than it saves (4096 positions, 5 waves: 29 us,
    // with two chunks 23, with four 25).
    const long long want = waves >= 1024 ? 1 : (2048 + waves - 1) / waves;
    const long long n = std::max(std::min(std::min(std::min(want, 1024LL), chunks / 2), (long long)(scratch_bytes / state) + 1), 1LL);
    const long long per = std::max((chunks + n - 1) / n, 1LL);
    p.seg_len = (int)(per * LC);
    p.segments = (int)std::max((chunks + per - 1) / per, 1LL);
    return p;
}

std::string linear_chunk_name(const LinChunkPlan& p, int dtype, bool outputs) {
    return std::string("k_linear_chunks<") + type_name(dtype) + ", " + std::to_string(p.width / 32) + (outputs ? ", true>" : ", false>");
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

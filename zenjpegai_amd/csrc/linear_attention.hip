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
template <typename T, bool V4, int NR>
__global__ void __launch_bounds__(256) k_linear_recurrent(LinAttnArgs a, int cl_log2, int tiles) {
    __shared__ float s_k[256], s_q[256];
    __shared__ f32x4 s_o[4][16];
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
    const float g = a.decay[head];
    s_k[tid] = s_q[tid] = 0.0f;  // rows past dk
    for (int cur = first;;) {
        const int len = a.lengths ? max(0, min(a.lengths[cur], a.length)) : a.length;
        for (int t = 0; t < len; ++t) {
            const int c = tid & 127;
            __syncthreads();
            if (c < a.dk) {
                const LinRows& src = tid < 128 ? a.k : a.q;
                (tid < 128 ? s_k : s_q)[c] = to_f32(((const T*)src.p)[lin_at(src, a.width, cur, t) + (long long)head * a.dk + c]);
            }
            const T* vp = (const T*)a.v.p + lin_at(a.v, a.width, cur, t) + (long long)head * a.dv + col;
            f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (col + e < a.dv) v[e] = to_f32(vp[e]);
            __syncthreads();
            f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < NR; ++n) {
                const float kk = s_k[(rg + n * RG) & 255], qq = s_q[(rg + n * RG) & 255];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    S[n][e] = fmaf(g, S[n][e], kk * v[e]);
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
                for (int c = 0; c < 4; ++c)
                    if (col + c < a.dv) p[c] = S[n][c];
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
    while (p.cl_log2 < 4 && (4 << p.cl_log2) < a.dv) ++p.cl_log2;
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
        default: k_linear_recurrent<T, V4, 8><<<grid, 256, 0, s>>>(a, p.cl_log2, p.tiles);
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
// Every value enters the matrix cores as bf16 pieces whose sum it is: one for bf16, two for f16 and three for
// f32 inputs (exact). What is computed in f32 is split likewise: the weighted values three ways (the
// state's sums keep f32 accuracy), the query products and the state in front of an output that is
// rounded to 16 bits two ways (2^-16 of them), with f32 outputs three ways. Products of pieces below
// 2^-16 (16-bit outputs) or 2^-23 of the whole are left out.
constexpr int LC = 32;

template <typename T> struct LinPieces;
template <> struct LinPieces<__bf16> { static constexpr int in = 1, mid = 2; };
template <> struct LinPieces<_Float16> { static constexpr int in = 2, mid = 2; };
template <> struct LinPieces<float> { static constexpr int in = 3, mid = 3; };

__device__ u32x4 g_lin_zero[1];  // 16 zero bytes: the source of absent positions and channels

// g^n for n >= 0, l2 = log2 g (-inf for g = 0).
__device__ __forceinline__ float lin_pow(float l2, int n) { return n == 0 ? 1.0f : exp2f((float)n * l2); }

// LDS rows of D bf16 in 16-byte units, XORed by row: the 16 rows of a b128 fragment read (q) and the 8
// rows by 2 units of a transposing read or the 16 rows of a b64 read (k, v) fall on distinct banks.
template <int D> __device__ __forceinline__ int swz_q(int row) {
    return D == 128 ? row & 15 : D == 64 ? (row >> 1) & 7 : ((row >> 2) & 1) << 1;
}
template <int D> __device__ __forceinline__ int swz_kv(int row) {
    return (D == 128 ? (row & 7) << 1 : D == 64 ? ((row >> 1) & 3) << 1 : ((row >> 2) & 1) << 1) | ((row >> 3) & 1);
}

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

// c[i][j] += a[i] b[j] over the products of pieces p + q <= LIM, the small ones first (two tiles of either operand).
// Inline assembly with the accumulators in place: the compiler renames the builtin's chains back to
// back. The block carries its own wait states, as split.h's.
#define LM(i, j, p, q) ZJAI_MF "%[c" #i #j "], %[a" #i #p "], %[b" #j #q "], %[c" #i #j "]\n\t"
#define LM4(p, q) LM(0, 0, p, q) LM(0, 1, p, q) LM(1, 0, p, q) LM(1, 1, p, q)
#define LC4 [c00] "+v"(c[0][0]), [c01] "+v"(c[0][1]), [c10] "+v"(c[1][0]), [c11] "+v"(c[1][1])
#define LA(p) [a0##p] "v"(a[0][p]), [a1##p] "v"(a[1][p])
#define LB(p) [b0##p] "v"(b[0][p]), [b1##p] "v"(b[1][p])
template <int LIM, int NA, int NB>
__device__ __forceinline__ void lin_mma(f32x4 (&c)[2][2], const u32x4 (&a)[2][NA], const u32x4 (&b)[2][NB]) {
    if constexpr (NA == 1 && NB == 1) {
        asm("s_nop 1\n\t" LM4(0, 0) ZJAI_WAIT : LC4 : LA(0), LB(0));
    } else if constexpr (NA == 1 && NB == 2) {
        asm("s_nop 1\n\t" LM4(0, 1) LM4(0, 0) ZJAI_WAIT : LC4 : LA(0), LB(0), LB(1));
    } else if constexpr (NA == 2 && NB == 1) {
        asm("s_nop 1\n\t" LM4(1, 0) LM4(0, 0) ZJAI_WAIT : LC4 : LA(0), LA(1), LB(0));
    } else if constexpr (NA == 1 && NB == 3) {
        asm("s_nop 1\n\t" LM4(0, 2) LM4(0, 1) LM4(0, 0) ZJAI_WAIT : LC4 : LA(0), LB(0), LB(1), LB(2));
    } else if constexpr (NA == 2 && NB == 2 && LIM == 1) {
        asm("s_nop 1\n\t" LM4(1, 0) LM4(0, 1) LM4(0, 0) ZJAI_WAIT : LC4 : LA(0), LA(1), LB(0), LB(1));
    } else if constexpr (NA == 2 && NB == 3 && LIM == 2) {
        asm("s_nop 1\n\t" LM4(1, 1) LM4(0, 2) LM4(1, 0) LM4(0, 1) LM4(0, 0) ZJAI_WAIT : LC4 : LA(0), LA(1), LB(0), LB(1), LB(2));
    } else {
        static_assert(NA == 3 && NB == 3 && LIM == 2, "piece products");
        asm("s_nop 1\n\t" LM4(2, 0) LM4(1, 1) LM4(0, 2) LM4(1, 0) LM4(0, 1) LM4(0, 0) ZJAI_WAIT
            : LC4 : LA(0), LA(1), LA(2), LB(0), LB(1), LB(2));
    }
}
#undef LB
#undef LA
#undef LC4
#undef LM4
#undef LM

// Eight channels of one position as loaded.
template <typename T> struct LinUnit { u32x4 v[sizeof(T) / 2]; };

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

template <typename T, int N>
__device__ __forceinline__ void lin_pieces(const LinUnit<T>& u, u32x4 (&p)[N]) {
    if constexpr (N == 1) {
        p[0] = u.v[0];
    } else {
        float x[8];
        constexpr int E = 16 / sizeof(T);
        typedef T tE __attribute__((ext_vector_type(E)));
#pragma unroll
        for (int h = 0; h < (int)sizeof(T) / 2; ++h) {
            const tE t = __builtin_bit_cast(tE, u.v[h]);
#pragma unroll
            for (int e = 0; e < E; ++e) x[h * E + e] = (float)t[e];
        }
        lin_split<N>(x, p);
    }
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
    int segments, seg_len, units, groups, tiles;
    int vec_k, vec_v, vec_o;
};

template <typename T, int WV, bool OUT>
__global__ void __launch_bounds__(256, 2) k_linear_chunks(LinChunkArgs c) {
    constexpr int D = 32 * WV, TT = 64 * WV, TEAMS = 4 / WV, NP = LinPieces<T>::in, NM = LinPieces<T>::mid;
    constexpr int LIM = NM - 1;               // products of the outputs
    constexpr int PLANE = LC * D;             // one piece of q, k or v
    constexpr int MT = D / 16, KS = D / 32;
    constexpr int NMAT = OUT ? 3 : 2;
    __shared__ __attribute__((aligned(16))) unsigned short s_lds[TEAMS * NMAT * NP * PLANE];
    const LinAttnArgs& a = c.a;
    const int team = threadIdx.x / TT, t = threadIdx.x % TT, wave = t >> 6, lane = t & 63, l16 = lane & 15, g = lane >> 4;
    unsigned short* s_k = s_lds + team * NMAT * NP * PLANE;
    unsigned short* s_v = s_k + NP * PLANE;
    unsigned short* s_q = s_v + NP * PLANE;

    const int segs = OUT ? c.segments : c.segments - 1;
    int b = blockIdx.x;
    const int group = b % c.groups;
    b /= c.groups;
    const int seg = b % segs, seq = b / segs;
    const int len = a.lengths ? max(0, min(a.lengths[seq], a.length)) : a.length;
    const int begin = seg * c.seg_len, end = min(len, begin + c.seg_len);
    // Sums are those that a later segment starts from.
    if (OUT ? begin > len || (begin == len && seg > 0) : begin + c.seg_len >= len) return;
    const int unit = group * TEAMS + team;
    const bool live = unit < c.units;
    const int head = live ? unit / c.tiles : 0, col0 = live ? (unit % c.tiles) * D : 0;
    const int colw = col0 + wave * 32;        // the wave's 32 value columns
    const bool work = live && colw < a.dv;

    const float l2 = log2f(a.decay[head]);
    float w_v[8], w_o[2], w_d[4], w_n[4], g_c = lin_pow(l2, LC);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        w_v[r] = lin_pow(l2, LC - 1 - (4 * g + r));
        w_v[4 + r] = lin_pow(l2, LC - 1 - (16 + 4 * g + r));
        const int d = l16 - (4 * g + r);
        w_d[r] = d >= 0 ? lin_pow(l2, d) : 0.0f;
        w_n[r] = lin_pow(l2, 16 + d);
    }
    w_o[0] = lin_pow(l2, l16 + 1);
    w_o[1] = lin_pow(l2, l16 + 17);

    // The state before the segment: S[mt][n][r] is key channel 16 mt + 4 g + r of value column 16 n + l16.
    f32x4 S[MT][2];
    const long long sbase = ((long long)seq * a.heads + head) * a.dk;
    const size_t xunit = (size_t)D * D;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            S[m][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (seg == 0) {
                if (a.s_in && work)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int kk = 16 * m + 4 * g + r, vv = colw + 16 * n + l16;
                        if (kk < a.dk && vv < a.dv) S[m][n][r] = a.s_in[(sbase + kk) * a.dv + vv];
                    }
            } else if (OUT && live) {
                const float* x = c.scratch + (((size_t)seq * (c.segments - 1) + seg - 1) * c.units + unit) * xunit;
                S[m][n] = *(const f32x4*)(x + (size_t)(((m * 2 + n) * WV + wave) * 64 + lane) * 4);
            }
        }

    const T* kp = (const T*)a.k.p + (long long)seq * a.k.seq + (long long)head * a.dk;
    const T* vp = (const T*)a.v.p + (long long)seq * a.v.seq + (long long)head * a.dv + col0;
    const T* qp = OUT ? (const T*)a.q.p + (long long)seq * a.q.seq + (long long)head * a.dk : nullptr;
    T* op = OUT ? (T*)a.o.p + (long long)seq * a.o.seq + (long long)head * a.dv + colw : nullptr;
    const int vcols = a.dv - col0;

    // A thread stages two units of eight channels of each matrix: rows row0 and row0 + 16, unit u.
    constexpr int UPR = D / 8;
    const int row0 = t / UPR, u = t % UPR;
    LinUnit<T> rk[2], rv[2], rq[2];
    const auto fetch = [&](int pos) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int p = pos + row0 + i * 16;
            const bool ok = live && p < end;
            const int y = a.width ? p / a.width : 0, x = a.width ? p - y * a.width : p;
            rk[i] = lin_load<T>(kp + (y * a.k.row + x * a.k.pos), u * 8, a.dk, ok, c.vec_k);
            rv[i] = lin_load<T>(vp + (y * a.v.row + x * a.v.pos), u * 8, vcols, ok, c.vec_v);
            if (OUT) rq[i] = lin_load<T>(qp + (y * a.q.row + x * a.q.pos), u * 8, a.dk, ok, c.vec_k);
        }
    };
    const auto stage = [&]() {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int row = row0 + i * 16;
            u32x4 p[NP];
            const int kv = row * D + ((u ^ swz_kv<D>(row)) * 8);
            lin_pieces<T, NP>(rk[i], p);
#pragma unroll
            for (int n = 0; n < NP; ++n) *(u32x4*)(s_k + n * PLANE + kv) = p[n];
            lin_pieces<T, NP>(rv[i], p);
#pragma unroll
            for (int n = 0; n < NP; ++n) *(u32x4*)(s_v + n * PLANE + kv) = p[n];
            if (OUT) {
                // Channels 4 x of a 32-channel block go to unit x % 4, half x / 4.
                lin_pieces<T, NP>(rq[i], p);
                const int unit0 = (u & ~3) + 2 * (u & 1), half = ((u >> 1) & 1) * 4;
                unsigned short* q0 = s_q + row * D + ((unit0 ^ swz_q<D>(row)) * 8) + half;
                unsigned short* q1 = s_q + row * D + (((unit0 + 1) ^ swz_q<D>(row)) * 8) + half;
#pragma unroll
                for (int n = 0; n < NP; ++n) {
                    *(u32x2*)(q0 + n * PLANE) = u32x2{p[n][0], p[n][1]};
                    *(u32x2*)(q1 + n * PLANE) = u32x2{p[n][2], p[n][3]};
                }
            }
        }
    };

    if (begin < end) fetch(begin);
    for (int pos = begin; pos < end; pos += LC) {
        __syncthreads();
        stage();
        __syncthreads();
        const int nv = min(LC, end - pos);
        if (pos + LC < end) fetch(pos + LC);
        if (!work) continue;

        f32x4 O[2][2];  // O[n][i], transposed: rows are value columns 16 n + 4 g + r, columns positions 16 i + l16
        u32x4 P[2][NM]; // weighted query products of positions 16 i + l16 with j = {4 g + r, 16 + 4 g + r}
        if (OUT) {
            f32x4 pt[2][2];  // pt[j][i]: rows are positions j of the keys, columns positions i of the queries
#pragma unroll
            for (int i = 0; i < 4; ++i) pt[i >> 1][i & 1] = O[i >> 1][i & 1] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                u32x4 qf[2][NP], kf[2][NP];
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int row = 16 * i + l16;
                    const unsigned short* qr = s_q + row * D + (((4 * s + g) ^ swz_q<D>(row)) * 8);
                    const unsigned short* k0 = s_k + row * D + (((4 * s + (g >> 1)) ^ swz_kv<D>(row)) * 8) + (g & 1) * 4;
                    const unsigned short* k1 = s_k + row * D + (((4 * s + 2 + (g >> 1)) ^ swz_kv<D>(row)) * 8) + (g & 1) * 4;
#pragma unroll
                    for (int n = 0; n < NP; ++n) {
                        qf[i][n] = *(const u32x4*)(qr + n * PLANE);
                        const u32x2 lo = *(const u32x2*)(k0 + n * PLANE), hi = *(const u32x2*)(k1 + n * PLANE);
                        kf[i][n] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                    }
                }
                lin_mma<LIM>(pt, kf, qf);
                u32x4 sf[2][NM];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float x[8];
#pragma unroll
                    for (int r = 0; r < 4; ++r) x[r] = S[2 * s][n][r], x[4 + r] = S[2 * s + 1][n][r];
                    lin_split<NM>(x, sf[n]);
                }
                lin_mma<LIM>(O, sf, qf);
            }
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r) O[n][i][r] *= w_o[i];
            float x0[8], x1[8];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const bool seen = 4 * g + r <= l16;  // a select: products with later positions may be infinite
                x0[r] = seen ? pt[0][0][r] * w_d[r] : 0.0f;
                x0[4 + r] = 0.0f;
                x1[r] = pt[0][1][r] * w_n[r];
                x1[4 + r] = seen ? pt[1][1][r] * w_d[r] : 0.0f;
            }
            lin_split<NM>(x0, P[0]);
            lin_split<NM>(x1, P[1]);
        }

        const bool last = pos + LC >= end;
        const bool update = !OUT || !last || (end == len && a.s_out);
        if (update && nv < LC) {  // the last chunk of a state that is kept: weights from its own end
            g_c = lin_pow(l2, nv);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                w_v[r] = lin_pow(l2, max(0, nv - 1 - (4 * g + r)));
                w_v[4 + r] = lin_pow(l2, max(0, nv - 1 - (16 + 4 * g + r)));
            }
        }
        const int trow = 4 * g + (l16 >> 2), tcol = (l16 & 3) >> 1, thalf = (l16 & 1) * 4;
        u32x4 vf[2][NP], wv[2][3];  // the values, and their weighted values' pieces
        float big = 0.0f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
            const int un = wave * 4 + 2 * n + tcol;
#pragma unroll
            for (int p = 0; p < NP; ++p) {
                const u32x2 lo = lds_tr(s_v + p * PLANE + trow * D + ((un ^ swz_kv<D>(trow)) * 8) + thalf);
                const u32x2 hi = lds_tr(s_v + p * PLANE + (trow + 16) * D + ((un ^ swz_kv<D>(trow)) * 8) + thalf);
                vf[n][p] = u32x4{lo[0], lo[1], hi[0], hi[1]};
            }
            float x[8];
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                float lo = __builtin_bit_cast(float, vf[n][0][h] << 16), hi = __builtin_bit_cast(float, vf[n][0][h] & 0xffff0000u);
#pragma unroll
                for (int p = 1; p < NP; ++p) {
                    lo += __builtin_bit_cast(float, vf[n][p][h] << 16);
                    hi += __builtin_bit_cast(float, vf[n][p][h] & 0xffff0000u);
                }
                big = __builtin_elementwise_maximum(__builtin_elementwise_maximum(big, __builtin_fabsf(lo)), __builtin_fabsf(hi));
                x[2 * h] = lo * w_v[2 * h];
                x[2 * h + 1] = hi * w_v[2 * h + 1];
            }
            lin_split<3>(x, wv[n]);
        }
        if (OUT) {
            if (__builtin_amdgcn_ballot_w64(!(big <= FLT_MAX)) == 0) {
                lin_mma<LIM>(O, vf, P);
            } else {
                // A value that is infinite or NaN: left out of the products, where it would meet the
                // zero weights of the positions before it, and put on the others afterwards.
                int first[2] = {LC, LC};
#pragma unroll
                for (int n = 0; n < 2; ++n) {
#pragma unroll
                    for (int e = 7; e >= 0; --e) {
                        const unsigned sh = (e & 1) * 16;
                        if (((vf[n][0][e >> 1] >> sh) & 0x7f80u) == 0x7f80u) {
                            first[n] = (e >> 2) * 16 + 4 * g + (e & 3);
#pragma unroll
                            for (int p = 0; p < NP; ++p) vf[n][p][e >> 1] &= 0xffff0000u >> sh;
                        }
                    }
                    first[n] = min(first[n], __shfl_xor(first[n], 16));
                    first[n] = min(first[n], __shfl_xor(first[n], 32));
                }
                lin_mma<LIM>(O, vf, P);
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
        }
        if (update) {
#pragma unroll
            for (int m = 0; m < MT; m += 2) {
                u32x4 kt[2][NP];
                f32x4 acc[2][2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int un = 2 * (m + h) + tcol;
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        const u32x2 lo = lds_tr(s_k + p * PLANE + trow * D + ((un ^ swz_kv<D>(trow)) * 8) + thalf);
                        const u32x2 hi = lds_tr(s_k + p * PLANE + (trow + 16) * D + ((un ^ swz_kv<D>(trow)) * 8) + thalf);
                        kt[h][p] = u32x4{lo[0], lo[1], hi[0], hi[1]};
                    }
#pragma unroll
                    for (int n = 0; n < 2; ++n)
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[h][n][r] = S[m + h][n][r] * g_c;
                }
                lin_mma<2>(acc, kt, wv);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int n = 0; n < 2; ++n) S[m + h][n] = acc[h][n];
            }
        }
        if (OUT) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int p = pos + 16 * i + l16;
                if (p >= end) continue;
                const int y = a.width ? p / a.width : 0, x = a.width ? p - y * a.width : p;
                T* o = op + (y * a.o.row + x * a.o.pos);
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int cc = 16 * n + 4 * g;
                    f32x4 v = O[n][i];
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] *= a.scale;
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
    } else if (live) {
        float* x = c.scratch + (((size_t)seq * (c.segments - 1) + seg) * c.units + unit) * xunit;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int n = 0; n < 2; ++n) *(f32x4*)(x + (size_t)(((m * 2 + n) * WV + wave) * 64 + lane) * 4) = S[m][n];
    }
}

// The state before segment s + 1 from the segments' own sums: E_(s+1) = g^seg_len E_s + X_s, in place (E_1 = X_0).
__global__ void __launch_bounds__(256) k_linear_scan(LinChunkArgs c, int quads) {
    const int q = blockIdx.x * 256 + threadIdx.x;
    if (q >= quads) return;
    const int unit = blockIdx.y % c.units, seq = blockIdx.y / c.units;
    const float g = lin_pow(log2f(c.a.decay[unit / c.tiles]), c.seg_len);
    f32x4* x = (f32x4*)c.scratch + ((size_t)seq * (c.segments - 1) * c.units + unit) * quads + q;
    const size_t step = (size_t)c.units * quads;
    f32x4 e = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s = 0; s < c.segments - 1; ++s, x += step) {
        const f32x4 v = *x;
#pragma unroll
        for (int r = 0; r < 4; ++r) e[r] = fmaf(g, e[r], v[r]);
        *x = e;
    }
}

LinChunkArgs chunk_args(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, float* scratch) {
    LinChunkArgs c{};
    c.a = a;
    c.scratch = scratch;
    c.segments = p.segments;
    c.seg_len = p.seg_len;
    c.units = p.units;
    c.groups = p.groups;
    c.tiles = p.units / a.heads;
    const int es = dtype == DT_F32 ? 4 : 2;
    const auto aligned = [&](const LinRows& r, int d, int bytes) {
        const int e = bytes / es;
        return ((uintptr_t)r.p & (bytes - 1)) == 0 && r.seq % e == 0 && r.pos % e == 0 && r.row % e == 0 && d % e == 0;
    };
    c.vec_k = aligned(a.k, a.dk, 16) && aligned(a.q, a.dk, 16);
    c.vec_v = aligned(a.v, a.dv, 16);
    c.vec_o = aligned(a.o, a.dv, 4 * es);
    return c;
}

template <typename T, bool OUT>
hipError_t chunks(const LinChunkArgs& c, int width, hipStream_t s) {
    const dim3 grid((unsigned)((long long)c.a.seqs * (OUT ? c.segments : c.segments - 1) * c.groups));
    if (width == 32) k_linear_chunks<T, 1, OUT><<<grid, 256, 0, s>>>(c);
    else if (width == 64) k_linear_chunks<T, 2, OUT><<<grid, 256, 0, s>>>(c);
    else k_linear_chunks<T, 4, OUT><<<grid, 256, 0, s>>>(c);
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
    const int teams = 128 / p.width;
    p.units = a.heads * ((a.dv + p.width - 1) / p.width);
    p.groups = (p.units + teams - 1) / teams;
    const long long have = (long long)a.seqs * p.groups;
    const long long state = (long long)a.seqs * p.units * p.width * p.width * 4;
    const long long chunks = (a.length + LC - 1) / LC;
    long long n = std::min(std::min((512 + have - 1) / have, chunks / 4), (long long)(scratch_bytes / state) + 1);
    n = std::max(n, 1LL);
    const long long per = (chunks + n - 1) / n;
    p.seg_len = (int)(per * LC);
    p.segments = (int)((chunks + per - 1) / per);
    if (p.segments < 1) p.segments = 1;
    return p;
}

std::string linear_chunk_name(const LinChunkPlan& p, int dtype, bool outputs) {
    return std::string("k_linear_chunks<") + type_name(dtype) + ", " + std::to_string(p.width / 32) + (outputs ? ", true>" : ", false>");
}

hipError_t launch_linear_sums(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, float* scratch, hipStream_t s) {
    return chunks_of<false>(a, p, dtype, scratch, s);
}
hipError_t launch_linear_scan(const LinAttnArgs& a, const LinChunkPlan& p, float* scratch, hipStream_t s) {
    const int quads = p.width * p.width / 4;
    k_linear_scan<<<dim3((unsigned)((quads + 255) / 256), (unsigned)(a.seqs * p.units)), 256, 0, s>>>(chunk_args(a, p, DT_F32, scratch), quads);
    return hipGetLastError();
}
hipError_t launch_linear_outputs(const LinAttnArgs& a, const LinChunkPlan& p, int dtype, const float* scratch, hipStream_t s) {
    return chunks_of<true>(a, p, dtype, const_cast<float*>(scratch), s);
}

}  // namespace zjai

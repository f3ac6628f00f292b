// Linear attention with a decay for each head (gfx950 / CDNA4, wave64):
//   S_t = g S_(t-1) + k_t^T v_t,   o_t = scale * q_t S_t,   S [dk][dv] in f32.

#include <climits>

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

}  // namespace zjai

// The join of two residual blocks (gfx950 / CDNA4, wave64), position by position:
//   x_out = x + scale * (post_norm(y) * act(gate)),   h = pre_norm(x_out),
// post_norm in groups of channels, statistics and intermediate values in f32, one rounding each.

#include "ops.h"

namespace zjai {

namespace {

__device__ __forceinline__ long long join_at(const JoinRows& r, int width, long long i) {
    if (width == 0) return i * r.pos;
    const long long y = i / width;
    return y * r.row + (i - y * width) * r.pos;
}

__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == GATE_LINEAR) return g;
    const float d = 1.0f + expf(-g);
    return act == GATE_SIGMOID ? 1.0f / d : g / d;
}

// Sum over the workgroup's 256 threads.
__device__ __forceinline__ float block_sum(float v, float* s_red) {
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) v += __shfl_xor(v, off);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) s_red[threadIdx.x >> 6] = v;
    __syncthreads();
    return (s_red[0] + s_red[1]) + (s_red[2] + s_red[3]);
}

// Mean (0 for RMS) and 1 / sqrt(variance + eps) of the n values at s.
__device__ __forceinline__ void norm_stats(const float* s, int n, int kind, float eps, float* s_red, float* mean, float* inv) {
    float m = 0.0f;
    if (kind == NORM_LAYER) {
        for (int c = threadIdx.x; c < n; c += 256) m += s[c];
        m = block_sum(m, s_red) / (float)n;
    }
    float q = 0.0f;
    for (int c = threadIdx.x; c < n; c += 256) q = fmaf(s[c] - m, s[c] - m, q);
    *mean = m;
    *inv = 1.0f / sqrtf(block_sum(q, s_red) / (float)n + eps);
}

template <typename T>
__global__ void __launch_bounds__(256) k_join(JoinArgs a) {
    extern __shared__ float s_v[];
    __shared__ float s_red[4];
    const long long i = blockIdx.x;
    const int C = a.channels, tid = threadIdx.x;
    const T* x = (const T*)a.x.p + join_at(a.x, a.width, i);
    const T* y = (const T*)a.y.p + join_at(a.y, a.width, i);
    const T* g = a.g.p ? (const T*)a.g.p + join_at(a.g, a.width, i) : nullptr;
    T* xo = (T*)a.xo.p + join_at(a.xo, a.width, i);
    T* h = a.h.p ? (T*)a.h.p + join_at(a.h, a.width, i) : nullptr;
    for (int c = tid; c < C; c += 256) s_v[c] = to_f32(y[c]);
    __syncthreads();
    const int per = C / a.groups;
    for (int k = 0; k < a.groups; ++k) {
        float m = 0.0f, inv = 1.0f;
        if (a.post != NORM_NONE) norm_stats(s_v + k * per, per, a.post, a.post_eps, s_red, &m, &inv);
        __syncthreads();
        for (int c = k * per + tid; c < (k + 1) * per; c += 256) {
            float u = s_v[c];
            if (a.post != NORM_NONE) u = (u - m) * inv;
            if (a.post_w) u *= a.post_w[c];
            if (a.post_b) u += a.post_b[c];
            if (g) u *= gate_value(to_f32(g[c]), a.gate);
            if (a.scale) u *= a.scale[c];
            s_v[c] = to_f32(x[c]) + u;
        }
    }
    __syncthreads();
    float m = 0.0f, inv = 1.0f;
    if (h) norm_stats(s_v, C, a.pre, a.pre_eps, s_red, &m, &inv);
    for (int c = tid; c < C; c += 256) {
        const float v = s_v[c];
        xo[c] = from_f32<T>(v);
        if (h) {
            float u = (v - m) * inv;
            if (a.pre_w) u *= a.pre_w[c];
            if (a.pre_b) u += a.pre_b[c];
            h[c] = from_f32<T>(u);
        }
    }
}

template <typename T>
hipError_t join(const JoinArgs& a, hipStream_t s) {
    k_join<T><<<dim3((unsigned)a.positions), 256, sizeof(float) * a.channels, s>>>(a);
    return hipGetLastError();
}

}  // namespace

std::string join_name(const JoinArgs& a, int dtype) {
    return std::string("k_join<") + (dtype == DT_F32 ? "float" : dtype == DT_F16 ? "_Float16" : "__bf16") + ">";
}

hipError_t launch_join(const JoinArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return join<float>(a, s);
    if (dtype == DT_F16) return join<_Float16>(a, s);
    return join<__bf16>(a, s);
}

}  // namespace zjai

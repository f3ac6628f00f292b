// Selective state-space scan (gfx950 / CDNA4, wave64): for every channel and state
//   s_t = softplus(delta_t + bias),  h_t = exp(s_t a) h_(t-1) + s_t b_t x_t,
//   out_t = (sum over the states of c_t h_t + d x_t) * silu(z_t).
//
// A wave has 64 / `lanes` channels of one group, a lane `ns` states of one of them, in registers over the positions. b and c
// of a tile of positions, which all channels of a group share, go through LDS as f32.
// Sequences that leave SIMDs idle are cut into segments: what each leaves behind when it starts from nothing (its end
// states and the sum of its steps, which is all that its decays depend on), from those the states that each starts from, then the outputs of all.

#include <algorithm>

#include "sequence.h"

namespace zjai {

namespace {

constexpr float LOG2E = 1.44269504088896340736f;
constexpr int SCAN_TILE = 8;  // positions whose loads are issued together

// ln(1 + exp(s)) = max(s, 0) + 2 artanh(e / (2 + e)) with e = exp(-|s|), by the series up to the fifteenth power of
// an argument of at most 1/3 (what follows is below 2^-29 of it): small steps keep their accuracy, the hardware's 2^x
// leaves (|s| + 2) 2^-24 of e.
__device__ __forceinline__ float softplus(float s) {
    const float e = __builtin_amdgcn_exp2f(fabsf(s) * -LOG2E);
    const float q = e * __builtin_amdgcn_rcpf(2.0f + e), q2 = q * q;
    float p = fmaf(q2, 1.0f / 15.0f, 1.0f / 13.0f);
    p = fmaf(p, q2, 1.0f / 11.0f);
    p = fmaf(p, q2, 1.0f / 9.0f);
    p = fmaf(p, q2, 1.0f / 7.0f);
    p = fmaf(p, q2, 1.0f / 5.0f);
    p = fmaf(p, q2, 1.0f / 3.0f);
    p = fmaf(p, q2, 1.0f);
    return fmaxf(s, 0.0f) + 2.0f * q * p;
}

// Sum over the 2^k neighbouring lanes of one channel; every one of them gets it.
template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_sum(float v, int lanes) {
    if (lanes >= 2) v = dpp_add<0xb1>(v);    // quad_perm 1 0 3 2
    if (lanes >= 4) v = dpp_add<0x4e>(v);    // quad_perm 2 3 0 1
    if (lanes >= 8) v = dpp_add<0x141>(v);   // the other half of eight lanes
    if (lanes >= 16) v = dpp_add<0x140>(v);  // ... of sixteen
    if (lanes >= 32) v += __shfl_xor(v, 16);
    if (lanes >= 64) v += __shfl_xor(v, 32);
    return v;
}

// A segment's states in the scratch: [sequences][segments][n][channels], then the sums of steps [sequences][segments][channels].
__device__ __forceinline__ long long scan_slot(const ScanArgs& a, const ScanPlan& p, int s, int seg) {
    return ((long long)s * p.segments + seg) * a.n * a.channels;
}
__device__ __forceinline__ long long step_slot(const ScanArgs& a, const ScanPlan& p, int s, int seg) {
    return ((long long)a.seqs * p.segments * a.n + (long long)s * p.segments + seg) * a.channels;
}
__device__ __forceinline__ int live_segments(const ScanPlan& p, int len) { return max(1, (len + p.seg_len - 1) / p.seg_len); }

// OUT: the outputs of a segment; else what it leaves behind.
template <typename T, int NS, bool OUT>
__global__ void __launch_bounds__(64) k_scan(ScanArgs a, ScanPlan p, float* scratch) {
    extern __shared__ float s_bc[];  // [SCAN_TILE][2][np]
    const int lane = threadIdx.x, np = NS * p.lanes, per_seg = a.groups * p.blocks, grid_segs = OUT ? p.segments : p.segments - 1;
    int id = blockIdx.x;
    const int s = id / (per_seg * grid_segs);
    id -= s * per_seg * grid_segs;
    const int seg = id / per_seg;
    id -= seg * per_seg;
    const int g = id / p.blocks, cg = a.channels / a.groups;
    const int at = (id - g * p.blocks) * (64 / p.lanes) + lane / p.lanes, part = lane & (p.lanes - 1);
    const bool on = at < cg;
    const int c = g * cg + (on ? at : 0);
    const int len = seq_length(a.lengths, s, a.length), live = live_segments(p, len);
    if (seg >= live || (!OUT && seg + 1 >= live)) return;
    const int t0 = seg * p.seg_len, t1 = min(len, t0 + p.seg_len);

    float rate[NS], h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int n = part * NS + i;
        rate[i] = n < a.n ? a.a[(long long)c * a.n + n] * LOG2E : 0.0f;
        h[i] = 0.0f;
        if (OUT && n < a.n) {
            if (p.segments > 1) h[i] = scratch[scan_slot(a, p, s, seg) + (long long)n * a.channels + c];
            else if (a.s_in) h[i] = a.s_in[((long long)s * a.channels + c) * a.n + n];
        }
    }
    const float bias = a.bias ? a.bias[c] : 0.0f, d = OUT && a.d ? a.d[c] : 0.0f;
    double steps = 0.0;  // its rounding would grow with the positions, and what a segment keeps of its start with it
    for (int t = t0; t < t1; t += SCAN_TILE) {
        T xv[SCAN_TILE], dv[SCAN_TILE], zv[SCAN_TILE];
#pragma unroll
        for (int i = 0; i < SCAN_TILE; ++i) {
            const int u = min(t + i, t1 - 1);
            xv[i] = ((const T*)a.x.p)[seq_at(a.x, a.width, s, u) + c];
            dv[i] = ((const T*)a.delta.p)[seq_at(a.delta, a.width, s, u) + c];
            if (OUT && a.z.p) zv[i] = ((const T*)a.z.p)[seq_at(a.z, a.width, s, u) + c];
        }
        __syncthreads();
        for (int e = lane; e < SCAN_TILE * np; e += 64) {
            const int i = e / np, n = e - i * np, u = min(t + i, t1 - 1);
            const bool there = n < a.n;
            const long long k = (long long)g * a.n + (there ? n : 0);
            const float b = to_f32(((const T*)a.b.p)[seq_at(a.b, a.width, s, u) + k]);
            s_bc[2 * i * np + n] = there ? b : 0.0f;
            if (OUT) {
                const float w = to_f32(((const T*)a.c.p)[seq_at(a.c, a.width, s, u) + k]);
                s_bc[(2 * i + 1) * np + n] = there ? w : 0.0f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < SCAN_TILE; ++i) {
            if (t + i >= t1) break;
            float step = to_f32(dv[i]) + bias;
            if (a.softplus) step = softplus(step);
            if (!OUT) steps += step;
            const float x = to_f32(xv[i]), u = step * x;
            const float* b = s_bc + 2 * i * np + part * NS;
            float y = 0.0f;
#pragma unroll
            for (int k = 0; k < NS; ++k) {
                h[k] = fmaf(__builtin_amdgcn_exp2f(step * rate[k]), h[k], u * b[k]);
                if (OUT) y = fmaf(b[np + k], h[k], y);
            }
            if (OUT) {
                y = lane_sum(y, p.lanes);
                if (a.d) y = fmaf(d, x, y);
                if (a.z.p) {
                    const float z = to_f32(zv[i]);
                    y *= z * fast_sigmoid(z);
                }
                if (on && part == 0) ((T*)a.o.p)[seq_at(a.o, a.width, s, t + i) + c] = from_f32<T>(y);
            }
        }
    }
    if (!on) return;
    float* to = nullptr;
    if (!OUT) to = scratch + scan_slot(a, p, s, seg);
    else if (a.s_out && seg + 1 == live) to = a.s_out;
    if (!to) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int n = part * NS + i;
        if (n < a.n) to[OUT ? ((long long)s * a.channels + c) * a.n + n : (long long)n * a.channels + c] = h[i];
    }
    if (!OUT && part == 0) scratch[step_slot(a, p, s, seg) + c] = (float)steps;
}

// Each segment's end states become the states that it starts from.
__global__ void __launch_bounds__(256) k_scan_starts(ScanArgs a, ScanPlan p, float* scratch) {
    const long long each = (long long)a.n * a.channels, i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= a.seqs * each) return;
    const int s = (int)(i / each);
    const long long in_slot = i - s * each;
    const int n = (int)(in_slot / a.channels), c = (int)(in_slot - (long long)n * a.channels);
    const int live = live_segments(p, seq_length(a.lengths, s, a.length));
    const float rate = a.a[(long long)c * a.n + n] * LOG2E;
    float h = a.s_in ? a.s_in[((long long)s * a.channels + c) * a.n + n] : 0.0f;
    float* state = scratch + scan_slot(a, p, s, 0) + in_slot;
    const float* steps = scratch + step_slot(a, p, s, 0) + c;
    for (int k = 0; k < live; ++k) {
        const float end = k + 1 < live ? state[k * each] : 0.0f, sum = k + 1 < live ? steps[(long long)k * a.channels] : 0.0f;
        state[k * each] = h;
        h = fmaf(__builtin_amdgcn_exp2f(sum * rate), h, end);
    }
}

// One position of each sequence. `lanes` lanes have a channel, four states each.
template <typename T, bool V4>
__global__ void __launch_bounds__(256) k_scan_step(ScanArgs a, int lanes, int blocks) {
    __shared__ int s_next;
    const int first = blockIdx.x / blocks, at = (blockIdx.x - first * blocks) * (256 / lanes) + threadIdx.x / lanes;
    const int n0 = (threadIdx.x & (lanes - 1)) * 4;
    const bool on = at < a.channels && n0 < a.n;
    const int c = min(at, a.channels - 1), n_first = n0 < a.n ? n0 : 0;
    const long long g = c / (a.channels / a.groups) * a.n;
    SlotChain chain{a.slots, a.num_slots, a.seqs, &s_next};
    if (!chain.begin(first)) return;
    const long long sbase = ((long long)chain.slot * a.channels + c) * a.n;
    f32x4 h, rate;
    if (V4) {
        h = *(const f32x4*)(a.s_in + sbase + n_first);
        rate = *(const f32x4*)(a.a + (long long)c * a.n + n_first);
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int n = min(n_first + k, a.n - 1);
            h[k] = a.s_in[sbase + n];
            rate[k] = a.a[(long long)c * a.n + n];
        }
    }
    const float bias = a.bias ? a.bias[c] : 0.0f, d = a.d ? a.d[c] : 0.0f;
    for (int s = first; s != INT_MAX; s = chain.next()) {
        float step = to_f32(((const T*)a.delta.p)[(long long)s * a.delta.seq + c]) + bias;
        const float x = to_f32(((const T*)a.x.p)[(long long)s * a.x.seq + c]);
        const float z = a.z.p ? to_f32(((const T*)a.z.p)[(long long)s * a.z.seq + c]) : 0.0f;
        float b[4], w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int n = min(n_first + k, a.n - 1);
            b[k] = to_f32(((const T*)a.b.p)[(long long)s * a.b.seq + g + n]);
            w[k] = to_f32(((const T*)a.c.p)[(long long)s * a.c.seq + g + n]);
        }
        if (a.softplus) step = softplus(step);
        const float u = step * x;
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = fmaf(__builtin_amdgcn_exp2f(step * (rate[k] * LOG2E)), h[k], u * b[k]);
            if (n0 + k < a.n) y = fmaf(w[k], h[k], y);
        }
        y = lane_sum(y, lanes);
        if (a.d) y = fmaf(d, x, y);
        if (a.z.p) y *= z * fast_sigmoid(z);
        if (on && n0 == 0) ((T*)a.o.p)[(long long)s * a.o.seq + c] = from_f32<T>(y);
    }
    if (!on) return;
    if (V4) *(f32x4*)(a.s_out + sbase + n0) = h;
    else
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n0 + k < a.n) a.s_out[sbase + n0 + k] = h[k];
}

bool step_wide(const ScanArgs& a) { return a.n % 4 == 0 && (((uintptr_t)a.s_in | (uintptr_t)a.s_out | (uintptr_t)a.a) & 15) == 0; }

template <typename T>
hipError_t scan_step(const ScanArgs& a, hipStream_t s) {
    int lanes = 1;
    while (lanes * 4 < a.n) lanes *= 2;
    const int blocks = (a.channels + 256 / lanes - 1) / (256 / lanes);
    if (step_wide(a)) k_scan_step<T, true><<<(unsigned)(a.seqs * blocks), 256, 0, s>>>(a, lanes, blocks);
    else k_scan_step<T, false><<<(unsigned)(a.seqs * blocks), 256, 0, s>>>(a, lanes, blocks);
    return hipGetLastError();
}

template <typename T, bool OUT>
hipError_t scan(const ScanArgs& a, const ScanPlan& p, float* scratch, hipStream_t s) {
    const unsigned grid = (unsigned)(a.seqs * (OUT ? p.segments : p.segments - 1) * a.groups * p.blocks);
    const size_t lds = sizeof(float) * SCAN_TILE * 2 * p.ns * p.lanes;
    switch (p.ns) {
        case 1: k_scan<T, 1, OUT><<<grid, 64, lds, s>>>(a, p, scratch); break;
        case 2: k_scan<T, 2, OUT><<<grid, 64, lds, s>>>(a, p, scratch); break;
        case 4: k_scan<T, 4, OUT><<<grid, 64, lds, s>>>(a, p, scratch); break;
        case 8: k_scan<T, 8, OUT><<<grid, 64, lds, s>>>(a, p, scratch); break;
        default: k_scan<T, 16, OUT><<<grid, 64, lds, s>>>(a, p, scratch);
    }
    return hipGetLastError();
}
template <bool OUT>
hipError_t scan_any(const ScanArgs& a, const ScanPlan& p, int dtype, float* scratch, hipStream_t s) {
    if (dtype == DT_F32) return scan<float, OUT>(a, p, scratch, s);
    if (dtype == DT_F16) return scan<_Float16, OUT>(a, p, scratch, s);
    return scan<__bf16, OUT>(a, p, scratch, s);
}

}  // namespace

ScanPlan scan_plan(const ScanArgs& a, int dtype, size_t scratch_bytes) {
    ScanPlan p{};
    const int cg = a.channels / a.groups;
    p.ns = 1;
    while (p.ns < 16 && p.ns < a.n) p.ns *= 2;
    p.lanes = 1;
    while (p.ns * p.lanes < a.n) p.lanes *= 2;
    p.blocks = (cg + 64 / p.lanes - 1) / (64 / p.lanes);
    const double waves = (double)a.seqs * a.groups * p.blocks;
    const long long slot = 4LL * a.seqs * a.channels * (a.n + 1);
    // Two waves a SIMD, of 32 positions at least.
    long long segments = waves < 1 ? 1 : (long long)std::min(2048.0 / waves, a.length / 32.0);
    segments = std::min<long long>(segments, (long long)scratch_bytes / std::max(slot, 1LL));
    p.segments = (int)std::max(1LL, segments);
    p.seg_len = std::max(1, (a.length + p.segments - 1) / p.segments);
    p.seg_len = (p.seg_len + SCAN_TILE - 1) / SCAN_TILE * SCAN_TILE;
    p.segments = std::max(1, (a.length + p.seg_len - 1) / p.seg_len);
    return p;
}

std::string scan_name(const ScanPlan& p, int dtype, bool outputs) {
    return std::string("k_scan<") + type_name(dtype) + ", " + std::to_string(p.ns) + (outputs ? ", true>" : ", false>");
}
hipError_t launch_scan_ends(const ScanArgs& a, const ScanPlan& p, int dtype, float* scratch, hipStream_t s) {
    return scan_any<false>(a, p, dtype, scratch, s);
}
hipError_t launch_scan_starts(const ScanArgs& a, const ScanPlan& p, float* scratch, hipStream_t s) {
    const long long n = (long long)a.seqs * a.n * a.channels;
    k_scan_starts<<<(unsigned)((n + 255) / 256), 256, 0, s>>>(a, p, scratch);
    return hipGetLastError();
}
hipError_t launch_scan_outputs(const ScanArgs& a, const ScanPlan& p, int dtype, const float* scratch, hipStream_t s) {
    return scan_any<true>(a, p, dtype, const_cast<float*>(scratch), s);
}

std::string scan_step_name(const ScanArgs& a, int dtype) {
    return std::string("k_scan_step<") + type_name(dtype) + (step_wide(a) ? ", true>" : ", false>");
}
hipError_t launch_scan_step(const ScanArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return scan_step<float>(a, s);
    if (dtype == DT_F16) return scan_step<_Float16>(a, s);
    return scan_step<__bf16>(a, s);
}

}  // namespace zjai

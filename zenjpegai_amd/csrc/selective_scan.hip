// Selective state-space scan (gfx950 / CDNA4, wave64): the states that segments start from, single positions, and the plan of a call.
// (The kernels of whole sequences, and the mathematics: selective_scan.h.)

#include <algorithm>

#include "selective_scan.h"

namespace zjai {

namespace {

constexpr int SCAN_RUN = 16, SCAN_MAX_SEGMENTS = 256;  // segments of a thread, and of 16 threads

// The decay 2^x of many positions together, as m 2^n: where states grow it may lie past f32's range although what comes of it
// does not, and a zero stays zero. (x is cut off well past the range of an exponent. Where it is no number, neither is the end
// state that is added.)
__device__ __forceinline__ void split_power(float x, float& m, int& n) {
    x = __builtin_amdgcn_fmed3f(x, -1024.0f, 1024.0f);
    const float whole = floorf(x);
    m = __builtin_amdgcn_exp2f(x - whole);
    n = (int)whole;
}
__device__ __forceinline__ float pass_on(float start, float m, int n, float end) { return fmaf(__builtin_amdgcn_ldexpf(start, n), m, end); }

// Each segment's end states become the states that it starts from. `parts` threads of a workgroup have a state, each
// SCAN_RUN consecutive segments of it, whose loads are issued together; what a run makes of its start (a decay and an
// end) goes to the later ones through LDS.
__global__ void __launch_bounds__(256) k_scan_starts(ScanArgs a, ScanPlan p, int parts, float* scratch) {
    __shared__ float s_power[256], s_end[256];
    __shared__ int s_whole[256];
    const int items = 256 / parts, part = threadIdx.x / items, first = part * SCAN_RUN;
    const long long size = (long long)a.n * a.channels, i = (long long)blockIdx.x * items + threadIdx.x % items;
    const bool on = i < a.seqs * size;
    const int s = on ? (int)(i / size) : 0;
    const long long in_slot = on ? i - s * size : 0;
    const int n = (int)(in_slot / a.channels), c = (int)(in_slot - (long long)n * a.channels);
    const int left = live_segments(p, seq_length(a.lengths, s, a.length)) - first;  // segments of the run, or none
    float* state = scratch + scan_slot(a, p, s, 0) + in_slot;
    const float* steps = scratch + step_slot(a, p, s, 0) + c;
    float end[SCAN_RUN], power[SCAN_RUN];
#pragma unroll
    for (int k = 0; k < SCAN_RUN; ++k) {  // the last segment leaves nothing behind (the first one's values in its place, not used)
        const long long from = k + 1 < left ? first + k : 0;
        end[k] = state[from * size];
        power[k] = steps[from * a.channels];
    }
    const float rate = a.a[(long long)c * a.n + n] * LOG2E;
    float h = a.s_in ? a.s_in[((long long)s * a.channels + c) * a.n + n] : 0.0f, all = 0.0f, e = 0.0f;
    int whole[SCAN_RUN];
#pragma unroll
    for (int k = 0; k < SCAN_RUN; ++k) {
        const float x = power[k] * rate;
        all += x;
        split_power(x, power[k], whole[k]);
        e = pass_on(e, power[k], whole[k], end[k]);
    }
    split_power(all, s_power[threadIdx.x], s_whole[threadIdx.x]);
    s_end[threadIdx.x] = e;
    __syncthreads();  // (and every state has been read before one is written)
    for (int q = threadIdx.x - part * items; q < (int)threadIdx.x; q += items) h = pass_on(h, s_power[q], s_whole[q], s_end[q]);
#pragma unroll
    for (int k = 0; k < SCAN_RUN; ++k) {
        if (!on || k >= left) break;
        state[(first + k) * size] = h;
        h = pass_on(h, power[k], whole[k], end[k]);
    }
}

// One position of each sequence. `lanes` lanes have a channel, four states each. WIDE: states, rates, b and c in aligned
// quads. A workgroup for every 256 / lanes channels: four times as many states a lane gain nothing (25 us instead of 23).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(256) k_scan_step(ScanArgs a, int lanes, int blocks) {
    typedef SeqVec<T, 4> Quad;
    __shared__ int s_next;
    const int first = blockIdx.x / blocks, at = (blockIdx.x - first * blocks) * (256 / lanes) + threadIdx.x / lanes;
    const int n0 = (threadIdx.x & (lanes - 1)) * 4;
    const bool on = at < a.channels && n0 < a.n, gate = a.z.p != nullptr;
    const int c = min(at, a.channels - 1), n_first = n0 < a.n ? n0 : 0;
    const long long g = c / (a.channels / a.groups) * a.n;
    SlotChain chain{a.slots, a.num_slots, a.seqs, &s_next};
    if (!chain.enter(first)) return;
    const long long sbase = ((long long)chain.slot * a.channels + c) * a.n;
    // Quads, or their values one by one: of states past the last one, the last one's (not used).
    const auto quad = [&](const float* p) __attribute__((always_inline)) {
        if (WIDE) return *(const f32x4*)(p + n_first);
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = p[min(n_first + k, a.n - 1)];
        return v;
    };
    const auto quad_t = [&](const T* p) __attribute__((always_inline)) {
        if (WIDE) return *(const Quad*)(p + n_first);
        Quad v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v.e[k] = p[min(n_first + k, a.n - 1)];
        return v;
    };
    T dr, xr, zr;
    Quad b, w;
    const auto fetch = [&](long long s) __attribute__((always_inline)) {
        dr = ((const T*)a.delta.p)[s * a.delta.seq + c];
        xr = ((const T*)a.x.p)[s * a.x.seq + c];
        zr = gate ? ((const T*)a.z.p)[s * a.z.seq + c] : xr;
        b = quad_t((const T*)a.b.p + s * a.b.seq + g);
        w = quad_t((const T*)a.c.p + s * a.c.seq + g);
    };
    f32x4 h = quad(a.s_in + sbase);
    fetch(first);
    const f32x4 rate = quad(a.a + (long long)c * a.n) * LOG2E;
    const float bias = a.bias ? a.bias[c] : 0.0f, d = a.d ? a.d[c] : 0.0f;
    // (All these are in flight while the sequences of the slot are looked for.)
    if (!chain.alone_or_first(first)) return;
    for (int s = first; s != INT_MAX;) {
        float step = to_f32(dr) + bias;
        const float x = to_f32(xr), z = to_f32(zr);
        if (a.softplus) step = softplus(step);
        const float u = step * x;
        float y = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = fmaf(__builtin_amdgcn_exp2f(step * rate[k]), h[k], u * to_f32(b.e[k]));
            if (n0 + k < a.n) y = fmaf(to_f32(w.e[k]), h[k], y);
        }
        y = lane_sum(y, lanes);
        if (a.d) y = fmaf(d, x, y);
        if (gate) y *= z * fast_sigmoid(z);
        if (on && n0 == 0) ((T*)a.o.p)[(long long)s * a.o.seq + c] = from_f32<T>(y);
        s = chain.next();
        if (s != INT_MAX) fetch(s);
    }
    if (!on) return;
    if (WIDE) *(f32x4*)(a.s_out + sbase + n0) = h;
    else
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (n0 + k < a.n) a.s_out[sbase + n0 + k] = h[k];
}

bool step_wide(const ScanArgs& a, int es) {
    for (const LinRows* r : {&a.b, &a.c})
        if ((uintptr_t)r->p % (4 * es) || r->seq % 4) return false;
    return a.n % 4 == 0 && (((uintptr_t)a.s_in | (uintptr_t)a.s_out | (uintptr_t)a.a) & 15) == 0;
}

template <typename T>
hipError_t scan_step(const ScanArgs& a, hipStream_t s) {
    int lanes = 1;
    while (lanes * 4 < a.n) lanes *= 2;
    const int blocks = (a.channels + 256 / lanes - 1) / (256 / lanes);
    if (step_wide(a, sizeof(T))) k_scan_step<T, true><<<(unsigned)(a.seqs * blocks), 256, 0, s>>>(a, lanes, blocks);
    else k_scan_step<T, false><<<(unsigned)(a.seqs * blocks), 256, 0, s>>>(a, lanes, blocks);
    return hipGetLastError();
}

hipError_t scan_any(const ScanArgs& a, const ScanPlan& p, int dtype, bool outputs, float* scratch, hipStream_t s) {
    if (dtype == DT_F32) return launch_scan_kernels<float>(a, p, outputs, scratch, s);
    if (dtype == DT_F16) return launch_scan_kernels<_Float16>(a, p, outputs, scratch, s);
    return launch_scan_kernels<__bf16>(a, p, outputs, scratch, s);
}

}  // namespace

ScanPlan scan_plan(const ScanArgs& a, size_t scratch_bytes) {
    ScanPlan p{};
    const int cg = a.channels / a.groups;
    p.ns = a.n == 1 ? 1 : a.n <= 4 ? 4 : a.n <= 8 ? 8 : 16;
    p.lanes = 1;
    while (p.ns * p.lanes < a.n) p.lanes *= 2;
    if (p.ns == 16 && p.lanes <= 4 && 12 * p.lanes >= a.n) p.ns = 12;
    const auto waves = [&]() { return std::max(1.0, (double)a.seqs * a.groups * ((cg + 64 / p.lanes - 1) / (64 / p.lanes))); };
    // Nine to sixteen states in one lane, or, where that leaves SIMDs idle even with segments of 64 positions, in four
    // (64 x 64 positions of 320 channels x 16 states f32 36 -> 27 us, 24 of 64 11.1 -> 5.4).
    if (p.ns >= 12 && p.lanes == 1 && waves() * (std::max(a.length, 1) / 64.0) < 1024.0) {
        p.ns = 4;
        p.lanes = 4;
    }
    // Waves of a workgroup: few without a channel, and few workgroups, each of which loads b and c (half a wave's worth): 64 sequences
    // of 1000 positions of 100 channels x 16 f32 four waves 122 us, two 95. (More than sixteen states' b and c take four waves.)
    const int needed = (int)(((long long)cg * p.lanes + 63) / 64);
    const auto cost = [&](int w) { return (needed + w - 1) / w * (w + 0.5); };
    p.waves = SCAN_WAVES;
    if (p.ns * p.lanes <= 16)
        for (int w = SCAN_WAVES - 1; w > 0; --w)
            if (cost(w) < cost(p.waves)) p.waves = w;
    p.blocks = (needed + p.waves - 1) / p.waves;
    // Segments for four waves a SIMD (65536 positions of 2048 channels x 16 states bf16: two 864 us, four 832, eight 879) or,
    // where lengths may differ, which only the device knows, for eight (12 sequences of 0-3001, 1024 channels x 64 f16: two
    // 939 us, four 640, eight 518), but none of less than 32 positions (the 64 x 64 map: 64 positions 31 us, 32 27, 16 29).
    const long long slot = 4LL * a.seqs * a.channels * (a.n + 1);
    long long segments = (long long)std::min((a.lengths ? 8192 : 4096) / waves(), a.length / 32.0);
    segments = std::min<long long>({segments, (long long)scratch_bytes / std::max(slot, 1LL), SCAN_MAX_SEGMENTS});
    p.segments = (int)std::max(1LL, segments);
    p.seg_len = std::max(1, (a.length + p.segments - 1) / p.segments);
    p.seg_len = (p.seg_len + SCAN_TILE - 1) / SCAN_TILE * SCAN_TILE;
    p.segments = std::max(1, (a.length + p.seg_len - 1) / p.seg_len);
    return p;
}

std::string scan_name(const ScanPlan& p, int dtype, bool outputs) {
    return std::string("k_scan<") + type_name(dtype) + ", " + std::to_string(p.ns) + ", " + std::to_string(p.lanes) + (outputs ? ", true>" : ", false>");
}
hipError_t launch_scan_ends(const ScanArgs& a, const ScanPlan& p, int dtype, float* scratch, hipStream_t s) {
    return scan_any(a, p, dtype, false, scratch, s);
}
hipError_t launch_scan_starts(const ScanArgs& a, const ScanPlan& p, float* scratch, hipStream_t s) {
    int parts = 1;
    while (parts * SCAN_RUN < p.segments) parts *= 2;
    const long long n = (long long)a.seqs * a.n * a.channels, items = 256 / parts;
    k_scan_starts<<<(unsigned)((n + items - 1) / items), 256, 0, s>>>(a, p, parts, scratch);
    return hipGetLastError();
}
hipError_t launch_scan_outputs(const ScanArgs& a, const ScanPlan& p, int dtype, const float* scratch, hipStream_t s) {
    return scan_any(a, p, dtype, true, const_cast<float*>(scratch), s);
}

std::string scan_step_name(const ScanArgs& a, int dtype) {
    return std::string("k_scan_step<") + type_name(dtype) + (step_wide(a, dtype == DT_F32 ? 4 : 2) ? ", true>" : ", false>");
}
hipError_t launch_scan_step(const ScanArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return scan_step<float>(a, s);
    if (dtype == DT_F16) return scan_step<_Float16>(a, s);
    return scan_step<__bf16>(a, s);
}

}  // namespace zjai

// The join of two residual blocks (gfx950 / CDNA4, wave64), position by position:
//   x_out = x + scale * (post_norm(y) * act(gate)),   h = pre_norm(x_out),
// post_norm in groups of channels, statistics and intermediate values in f32, one rounding each.
//
// HBM bound: five arrays pass once (x, y, gate in, x_out, h out). A position belongs to a team of TP lanes
// (a power of two), a lane to the vectors lane + TP i of its channels, so the five weight vectors
// are loaded once and stay in registers over the positions a team walks through (up to 8192 channels); a position's whole
// arithmetic runs on registers. The next position's loads are issued before this one's sums.

#include <algorithm>

#include "ops.h"

namespace zjai {

namespace {

__device__ __forceinline__ long long join_at(const JoinRows& r, int width, long long i) {
    if (width == 0) return i * r.pos;
    const long long y = i / width;
    return y * r.row + (i - y * width) * r.pos;
}

// exp(-g) by the hardware's 2^x: relative error (|g| + 2) 2^-24, as the rounding of g log2 e leaves any.
__device__ __forceinline__ float gate_value(float g, int act) {
    if (act == GATE_LINEAR) return g;
    const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269504088896340736f));
    return act == GATE_SIGMOID ? s : g * s;
}

// How a team sums over groups of channels: all of a position; groups of 2^k lanes; or, for every other
// size, lane exchanges over the 2^k lanes that divide a group and LDS for the rest, which `join` lanes of the team
// add up together for each group (4000 positions of 9002 channels in two groups, bf16: 0.44 ms; each lane its own
// group's parts, one after another: 394).
enum SumMode : int { SUM_ALL = 0, SUM_LANES = 1, SUM_LDS = 2 };

struct JoinPlan {
    int tp, threads, mode, group_vecs, lanes;  // group_vecs: vectors of a group; lanes: 2^k of SUM_LANES / SUM_LDS
    int join;                                  // SUM_LDS: lanes (2^k) that add up a group's parts
    int wide_weights;                          // the weights are 16-byte aligned
};

template <int NV>
struct TeamSum {
    int tid, lane, tp, threads, team0;  // team0: the team's first thread
    float *s_red, *s_group;             // s_group: the team's sums of its groups
    int n_groups;

    // Of the whole team's values; every lane gets it.
    __device__ __forceinline__ float all(const float (&v)[NV]) const {
        float s = v[0];
#pragma unroll
        for (int i = 1; i < NV; ++i) s += v[i];
        const int in_wave = min(tp, 64);
        for (int off = 1; off < in_wave; off <<= 1) s += __shfl_xor(s, off);
        if (tp > 64) {
            __syncthreads();
            if ((tid & 63) == 0) s_red[tid >> 6] = s;
            __syncthreads();
            s = 0.0f;
            for (int w = team0 >> 6; w < (team0 + tp) >> 6; ++w) s += s_red[w];
        }
        return s;
    }
    // v[i]: of the group that vector i belongs to.
    __device__ __forceinline__ void groups(float (&v)[NV], const JoinPlan& p) const {
        if (p.mode == SUM_ALL) {
            const float s = all(v);
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] = s;
            return;
        }
        for (int off = 1; off < p.lanes; off <<= 1)
#pragma unroll
            for (int i = 0; i < NV; ++i) v[i] += __shfl_xor(v[i], off);
        if (p.mode == SUM_LANES) return;
        int t = tid, l = lane;
        if (NV > 4) asm volatile("" : "+v"(t), "+v"(l));  // places computed here, not kept over the positions
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if ((t & (p.lanes - 1)) == 0) s_red[i * threads + t] = v[i];
        __syncthreads();
        const int part = l & (p.join - 1), stride = p.join * p.lanes, log_tp = __builtin_ctz(tp), log_join = __builtin_ctz(p.join);
        for (int n = l >> log_join; n < n_groups; n += tp >> log_join) {
            const int first = n * p.group_vecs;
            float s = 0.0f;
            for (int k = first + part * p.lanes; k < first + p.group_vecs; k += stride)
                s += s_red[(k >> log_tp) * threads + team0 + (k & (tp - 1))];
            for (int off = 1; off < p.join; off <<= 1) s += __shfl_xor(s, off);
            if (part == 0) s_group[n] = s;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int n = (l + tp * i) / p.group_vecs;
            v[i] = s_group[min(n, n_groups - 1)];  // past the channels: nothing uses it
        }
    }
};

template <typename T, int VE> struct alignas(sizeof(T) * VE) JoinVec { T e[VE]; };

// PRE, GATE: whether h and the gate are there.
template <typename T, int VE, int NV, bool PRE, bool GATE>
__global__ void __launch_bounds__(1024) k_join(JoinArgs a, JoinPlan p) {
    typedef JoinVec<T, VE> V;
    extern __shared__ float s_red[];
    const int tid = threadIdx.x, lane = tid & (p.tp - 1), team = tid / p.tp, teams = p.threads / p.tp;
    const TeamSum<NV> sum{tid, lane, p.tp, p.threads, team * p.tp, s_red, s_red + NV * p.threads + team * a.groups, a.groups};
    const int C = a.channels;
    // Eight channels' weights stay in registers; sixteen channels', and those of single ones, are read again where a
    // position needs them. (With 1024 lanes a lane has 128 registers. What does not fit goes to private memory, for
    // which the runtime takes 686 MiB of the card at the first such launch: 9001 channels, f32.)
    constexpr bool KEEP = NV * VE <= 8 && VE > 1;
    // There, what a position's addresses are made of is not kept over the positions either (nor over its parts).
    int here = lane;
    const auto afresh = [&]() {
        if constexpr (KEEP) return;
        asm volatile("" : "+v"(here));
    };
    const auto vec = [&](int i) { return (here + p.tp * i) * VE; };
    bool on[NV];
    float pw[NV][VE], pb[NV][VE], sc[NV][VE], nw[NV][VE], nb[NV][VE];
    // w's VE values of vector i; lanes past the channels read the first ones, which nothing uses.
    const auto weights = [&](const float* w, int i, float absent, float (&to)[VE]) {
        if (!w) {
#pragma unroll
            for (int e = 0; e < VE; ++e) to[e] = absent;
            return;
        }
        if (!KEEP) asm volatile("" : "+s"(w));
        w += on[i] ? vec(i) : 0;
        if constexpr (VE % 4 == 0) {
            if (p.wide_weights) {
#pragma unroll
                for (int e = 0; e < VE; e += 4) {
                    const f32x4 q = *(const f32x4*)(w + e);
#pragma unroll
                    for (int k = 0; k < 4; ++k) to[e + k] = q[k];
                }
                return;
            }
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) to[e] = w[e];
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) on[i] = (lane + p.tp * i) * VE < C;
    const auto load_weights = [&]() {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            weights(a.post_w, i, 1.0f, pw[i]);
            weights(a.post_b, i, 0.0f, pb[i]);
            weights(a.scale, i, 1.0f, sc[i]);
            if (PRE) weights(a.pre_w, i, 1.0f, nw[i]);
            if (PRE) weights(a.pre_b, i, 0.0f, nb[i]);
        }
    };
    const float inv_group = 1.0f / (float)(C / a.groups), inv_all = 1.0f / (float)C;

    V x[NV], y[NV], g[NV];
    const auto place = [&](const JoinRows& r, long long at) {
        return (const T*)r.p + (at < a.positions ? join_at(r, a.width, at) : 0);
    };
    // (`c`: always a channel that exists.)
    const auto fetch_gate = [&](long long at) {
        const T* pg = place(a.g, at);
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = on[i] ? vec(i) : 0;
            g[i] = *(const V*)(pg + c);
        }
    };
    constexpr bool GATE_AHEAD = GATE && NV < 16;  // sixteen addresses more than there are registers for
    const auto fetch = [&](long long at) {
        const T *px = place(a.x, at), *py = place(a.y, at), *pg = GATE_AHEAD ? place(a.g, at) : nullptr;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int c = on[i] ? vec(i) : 0;
            x[i] = *(const V*)(px + c);
            y[i] = *(const V*)(py + c);
            if (GATE_AHEAD) g[i] = *(const V*)(pg + c);
        }
    };
    const long long step = (long long)gridDim.x * teams;
    long long base = (long long)blockIdx.x * teams;
    if (base < a.positions) fetch(base + team);
    if (KEEP) load_weights();
    const auto weight = [&](const float (&kept)[NV][VE], const float* w, int i, float absent, float (&to)[VE]) {
        if constexpr (KEEP) {
#pragma unroll
            for (int e = 0; e < VE; ++e) to[e] = kept[i][e];
        } else {
            weights(w, i, absent, to);
        }
    };
    for (; base < a.positions; base += step) {
        const long long at = base + team;
        afresh();
        float u[NV][VE], v[NV][VE];
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                u[i][e] = to_f32(y[i].e[e]);
                v[i][e] = to_f32(x[i].e[e]);
            }
        if (a.post != NORM_NONE) {
            float s[NV];
            if (a.post == NORM_LAYER) {
#pragma unroll
                for (int i = 0; i < NV; ++i) {
                    s[i] = 0.0f;
#pragma unroll
                    for (int e = 0; e < VE; ++e) s[i] += u[i][e];
                    s[i] = on[i] ? s[i] : 0.0f;
                }
                sum.groups(s, p);
#pragma unroll
                for (int i = 0; i < NV; ++i)
#pragma unroll
                    for (int e = 0; e < VE; ++e) u[i][e] -= s[i] * inv_group;
            }
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                s[i] = 0.0f;
#pragma unroll
                for (int e = 0; e < VE; ++e) s[i] = fmaf(u[i][e], u[i][e], s[i]);
                s[i] = on[i] ? s[i] : 0.0f;
            }
            sum.groups(s, p);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float inv = 1.0f / sqrtf(s[i] * inv_group + a.post_eps);
                float w[VE], b[VE];
                weight(pw, a.post_w, i, 1.0f, w);
                weight(pb, a.post_b, i, 0.0f, b);
#pragma unroll
                for (int e = 0; e < VE; ++e) u[i][e] = u[i][e] * inv * w[e] + b[e];
            }
        }
        if (GATE && !GATE_AHEAD) {
            afresh();
            fetch_gate(at);
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            float w[VE];
            weight(sc, a.scale, i, 1.0f, w);
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                if (GATE) u[i][e] *= gate_value(to_f32(g[i].e[e]), a.gate);
                v[i][e] += u[i][e] * w[e];
                if (!KEEP) asm volatile("" : "+v"(v[i][e]));  // before the next loads, not where it is stored
            }
        }
        afresh();
        fetch(at + step);
        afresh();
        if (at < a.positions) {
            T* po = (T*)a.xo.p + join_at(a.xo, a.width, at);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                V o;
#pragma unroll
                for (int e = 0; e < VE; ++e) o.e[e] = from_f32<T>(v[i][e]);
                if (on[i]) *(V*)(po + vec(i)) = o;
            }
        }
        if (!PRE) continue;
        float s[NV], mean = 0.0f;
        if (a.pre == NORM_LAYER) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                s[i] = 0.0f;
#pragma unroll
                for (int e = 0; e < VE; ++e) s[i] += v[i][e];
                s[i] = on[i] ? s[i] : 0.0f;
            }
            mean = sum.all(s) * inv_all;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            s[i] = 0.0f;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                v[i][e] -= mean;
                s[i] = fmaf(v[i][e], v[i][e], s[i]);
            }
            s[i] = on[i] ? s[i] : 0.0f;
        }
        const float inv = 1.0f / sqrtf(sum.all(s) * inv_all + a.pre_eps);
        afresh();
        if (at < a.positions) {
            T* ph = (T*)a.h.p + join_at(a.h, a.width, at);
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                V o;
                float w[VE], b[VE];
                weight(nw, a.pre_w, i, 1.0f, w);
                weight(nb, a.pre_b, i, 0.0f, b);
#pragma unroll
                for (int e = 0; e < VE; ++e) o.e[e] = from_f32<T>(v[i][e] * inv * w[e] + b[e]);
                if (on[i]) *(V*)(ph + vec(i)) = o;
            }
        }
    }
}

// Channels a vector holds: the most, up to 16 bytes, that divide the group and keep every row aligned.
int join_vector(const JoinArgs& a, int es) {
    int ve = 16 / es;
    const auto fits = [&](int v) {
        if (a.channels / a.groups % v) return false;
        for (const JoinRows* r : {&a.x, &a.y, &a.g, &a.xo, &a.h})
            if (r->p && (((uintptr_t)r->p % (v * es)) || r->pos % v || r->row % v)) return false;
        return true;
    };
    while (ve > 1 && !fits(ve)) ve /= 2;
    return ve;
}
// Channels a lane holds: eight, or sixteen where 1024 lanes of eight are too few.
int join_lane_channels(const JoinArgs& a) { return a.channels <= 8192 ? 8 : 16; }

JoinPlan join_plan(const JoinArgs& a, int ve, int per_lane) {
    JoinPlan p{};
    p.tp = 1;
    while (p.tp * per_lane < a.channels) p.tp *= 2;
    p.threads = std::max(p.tp, 256);
    p.group_vecs = a.channels / a.groups / ve;
    p.lanes = 1;
    while (p.lanes < std::min(p.tp, 64) && p.group_vecs % (2 * p.lanes) == 0) p.lanes *= 2;
    p.join = 1;
    while (p.join < std::min(64, p.tp / a.groups) && p.join * p.lanes < p.group_vecs) p.join *= 2;
    p.wide_weights = (((uintptr_t)a.post_w | (uintptr_t)a.post_b | (uintptr_t)a.scale | (uintptr_t)a.pre_w | (uintptr_t)a.pre_b) & 15) == 0;
    p.mode = a.groups == 1 ? SUM_ALL : p.group_vecs == p.lanes ? SUM_LANES : SUM_LDS;
    return p;
}

template <typename T, int VE, int NV>
hipError_t join(const JoinArgs& a, hipStream_t s) {
    const JoinPlan p = join_plan(a, VE, VE * NV);
    const int teams = p.threads / p.tp;
    // Four workgroups of 256 lanes to a CU (registers hold four waves to a SIMD), each over its share of the
    // positions: one to a CU leaves the loads' latency bare (16385 x 4096 f16 290 us, four 128), a workgroup for
    // every 16 positions pays for the weights as often as for the data (215 x 216 x 128 bf16 13.6 -> 14.9 us).
    const long long blocks = std::min((a.positions + teams - 1) / teams, (long long)256 * 4 * 256 / p.threads);
    const dim3 grid((unsigned)blocks), block((unsigned)p.threads);
    const size_t lds = sizeof(float) * (p.mode == SUM_LDS ? NV * p.threads + teams * a.groups : 16);
    if (a.h.p && a.g.p) k_join<T, VE, NV, true, true><<<grid, block, lds, s>>>(a, p);
    else if (a.h.p) k_join<T, VE, NV, true, false><<<grid, block, lds, s>>>(a, p);
    else if (a.g.p) k_join<T, VE, NV, false, true><<<grid, block, lds, s>>>(a, p);
    else k_join<T, VE, NV, false, false><<<grid, block, lds, s>>>(a, p);
    return hipGetLastError();
}
template <typename T, int VE>
hipError_t join_lanes(const JoinArgs& a, hipStream_t s) {
    return join_lane_channels(a) == 8 ? join<T, VE, 8 / VE>(a, s) : join<T, VE, 16 / VE>(a, s);
}
template <typename T>
hipError_t join_of(const JoinArgs& a, hipStream_t s) {
    const int ve = join_vector(a, sizeof(T));
    if constexpr (sizeof(T) == 2)
        if (ve == 8) return join_lanes<T, 8>(a, s);
    if (ve == 4) return join_lanes<T, 4>(a, s);
    if (ve == 2) return join_lanes<T, 2>(a, s);
    return join_lanes<T, 1>(a, s);
}

}  // namespace

std::string join_name(const JoinArgs& a, int dtype) {
    const int ve = join_vector(a, dtype == DT_F32 ? 4 : 2);
    return std::string("k_join<") + (dtype == DT_F32 ? "float" : dtype == DT_F16 ? "_Float16" : "__bf16") + ", " + std::to_string(ve) +
           ", " + std::to_string(join_lane_channels(a) / ve) + (a.h.p ? ", true" : ", false") + (a.g.p ? ", true>" : ", false>");
}

hipError_t launch_join(const JoinArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return join_of<float>(a, s);
    if (dtype == DT_F16) return join_of<_Float16>(a, s);
    return join_of<__bf16>(a, s);
}

}  // namespace zjai

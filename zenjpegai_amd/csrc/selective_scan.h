// Selective state-space scan (gfx950 / CDNA4, wave64): for every channel and state
//   s_t = softplus(delta_t + bias),  h_t = exp(s_t a) h_(t-1) + s_t b_t x_t,
//   out_t = (sum over the states of c_t h_t + d x_t) * silu(z_t).
//
// A lane has NS states of one channel, in registers over the positions; LANES neighbouring lanes have a channel, a workgroup of
// one to four waves 64 / LANES channels of one group for each of them. Positions pass in tiles of eight. What a tile needs for each channel
// and position (the step, its softplus, the gate) is shared out among the channel's lanes and handed round by lane
// exchanges; b and c, which all channels of a group share, go through LDS as f32. The next two tiles' loads are in
// flight meanwhile.
// Bound by the vector ALUs: four instructions of 4 cycles and a 2^x of 8 for each position, channel and state of a wave's lanes. 65536
// positions of 2048 channels x 16 states bf16: outputs 483 us with the ALUs 90 % busy, ends 347 with 98 %.
// Sequences that leave SIMDs idle are cut into segments: what each leaves behind when it starts from nothing (its end
// states and the sum of its steps, which is all that its decays depend on), from those the states that each starts from, then
// the outputs of all. The ends cost nearly as much again, so whole sequences stay whole where they fill the card.
//
// Here are the kernels of whole sequences and what the steps share with them. Those of each storage type are compiled in a file
// of their own: together they take a compiler three and a half minutes.
#pragma once

#include <type_traits>

#include "sequence.h"

namespace zjai {

// The ends (outputs: the outputs) of the segments of a plan.
template <typename T>
hipError_t launch_scan_kernels(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s);
template <>
hipError_t launch_scan_kernels<float>(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s);
template <>
hipError_t launch_scan_kernels<_Float16>(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s);
template <>
hipError_t launch_scan_kernels<__bf16>(const ScanArgs& a, const ScanPlan& p, bool outputs, float* scratch, hipStream_t s);

namespace {

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;
constexpr int SCAN_TILE = 8, SCAN_WAVES = 4;

// ln(1 + exp(s)) = max(s, 0) + ln(1 + e) with e = exp(-|s|): the logarithm of the rounded 1 + e, and what the rounding left
// of e beside it, so that small steps keep their accuracy (the hardware's 2^x leaves (|s| + 2) 2^-24 of e, its logarithm
// 2^-23 of itself next to one, too).
__device__ __forceinline__ float softplus(float s) {
    const float e = __builtin_amdgcn_exp2f(fabsf(s) * -LOG2E);
    const float u = 1.0f + e;
    return __builtin_amdgcn_fmed3f(s, 0.0f, __builtin_inff()) + fmaf(__builtin_amdgcn_logf(u), LN2, e - (u - 1.0f));
}

// Sum over the `lanes` neighbouring lanes of one channel; every one of them gets it.
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_sum(float v, int lanes) {
    if (lanes >= 2) v += dpp<0xb1>(v);    // quad_perm 1 0 3 2
    if (lanes >= 4) v += dpp<0x4e>(v);    // quad_perm 2 3 0 1
    if (lanes >= 8) v += dpp<0x141>(v);   // the other half of eight lanes
    if (lanes >= 16) v += dpp<0x140>(v);  // ... of sixteen
    if (lanes >= 32) v += __shfl_xor(v, 16);
    if (lanes >= 64) v += __shfl_xor(v, 32);
    return v;
}
// The value of lane `owner` of the LANES neighbouring ones.
template <int LANES, int OWNER>
__device__ __forceinline__ float lane_value(float v) {
    if constexpr (LANES == 1) return v;
    else if constexpr (LANES == 2) return dpp<OWNER == 0 ? 0xa0 : 0xf5>(v);  // quad_perm 0 0 2 2, 1 1 3 3
    else if constexpr (LANES == 4) return dpp<OWNER * 0x55>(v);
    else if constexpr (LANES == 8) {
        const float mine = dpp<(OWNER & 3) * 0x55>(v), other = dpp<0x141>(mine);  // of the lane's four, of the other four
        return ((threadIdx.x >> 2) & 1) == OWNER >> 2 ? mine : other;
    } else return dpp<0x150 + OWNER>(v);  // row_newbcast
}

// A segment's states in the scratch: [sequences][segments][n][channels], then the sums of steps [sequences][segments][channels].
__device__ __forceinline__ long long scan_slot(const ScanArgs& a, const ScanPlan& p, int s, int seg) {
    return ((long long)s * p.segments + seg) * a.n * a.channels;
}
__device__ __forceinline__ long long step_slot(const ScanArgs& a, const ScanPlan& p, int s, int seg) {
    return ((long long)a.seqs * p.segments * a.n + (long long)s * p.segments + seg) * a.channels;
}
__device__ __forceinline__ int live_segments(const ScanPlan& p, int len) { return max(1, (len + p.seg_len - 1) / p.seg_len); }

// Compile-time loop: f(0), f(1), .. as constants.
template <int N, int I = 0, typename F>
__device__ __forceinline__ void each(F&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each<N, I + 1>(f);
    }
}

// OUT: the outputs of a segment; else what it leaves behind.
template <typename T, int NS, int LANES, bool OUT>
__global__ void __launch_bounds__(64 * SCAN_WAVES, 2) k_scan(ScanArgs a, ScanPlan p, float* scratch) {
    constexpr int NP = NS * LANES < 4 ? 4 : NS * LANES;  // floats of a row of b or c in LDS
    constexpr int SIDES = OUT ? 2 : 1, ITEMS = SCAN_TILE * SIDES * NP / 4, PER_LANE = (ITEMS + 64 * SCAN_WAVES - 1) / (64 * SCAN_WAVES);
    constexpr int OWNERS = LANES < SCAN_TILE ? LANES : SCAN_TILE, OWN = SCAN_TILE / OWNERS;  // positions of a tile that a lane looks after
    __shared__ alignas(16) float s_bc[2][SCAN_TILE][SIDES][NP];  // read and written in quads
    const int tid = threadIdx.x, lane = tid & 63, per_seg = a.groups * p.blocks, grid_segs = OUT ? p.segments : p.segments - 1;
    int id = blockIdx.x;
    const int s = id / (per_seg * grid_segs);
    id -= s * per_seg * grid_segs;
    const int seg = id / per_seg;
    id -= seg * per_seg;
    const int g = id / p.blocks, cg = a.channels / a.groups;
    const int at = (id - g * p.blocks) * ((int)blockDim.x / LANES) + tid / LANES, part = lane & (LANES - 1);
    const bool on = at < cg;
    const bool idle = __builtin_amdgcn_readfirstlane(at) >= cg;  // a wave without channels: it loads, and waits at the barriers
    const int c = g * cg + (on ? at : 0);
    const int len = seq_length(a.lengths, s, a.length), live = live_segments(p, len);
    if (seg >= live || (!OUT && seg + 1 >= live)) return;
    const int t0 = seg * p.seg_len, t1 = min(len, t0 + p.seg_len);

    // The lane's state i: quads of states go round the channel's lanes, so that those read neighbouring quads.
    const auto state = [&](int i) { return NS < 4 ? i : ((i >> 2) * LANES + part) * 4 + (i & 3); };
    float rate[NS], h[NS];
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int n = state(i);
        rate[i] = n < a.n ? a.a[(long long)c * a.n + n] * LOG2E : 0.0f;
        h[i] = 0.0f;
        if (OUT && n < a.n) {
            if (p.segments > 1) h[i] = scratch[scan_slot(a, p, s, seg) + (long long)n * a.channels + c];
            else if (a.s_in) h[i] = a.s_in[((long long)s * a.channels + c) * a.n + n];
        }
    }
    const float bias = a.bias ? a.bias[c] : 0.0f, d = OUT && a.d ? a.d[c] : 0.0f;
    const bool gate = OUT && a.z.p;
    double steps = 0.0;  // its rounding would grow with the positions, and what a segment keeps of its start with it

    // A tile's inputs: the lane's share of x, delta and z, and of b and c in quads. Lanes without a channel or a quad of
    // their own load the first ones, which nothing uses: no load is in a branch, so that they stay in flight over the tiles.
    struct Tile {
        T x[OWN], delta[OWN], z[OWN];
        SeqVec<T, 4> bc[PER_LANE];
    };
    const int own = part & (OWNERS - 1);
    const unsigned c_bytes = (unsigned)c * (unsigned)sizeof(T);
    const auto item_of = [&](int k) { return min(tid + k * 64 * SCAN_WAVES, ITEMS - 1); };
    // The channel's offset, made anew where it is added to a place that all lanes share: as the address's own 32 bits.
    const auto channel = [&]() __attribute__((always_inline)) {
        unsigned off = c_bytes;
        asm volatile("" : "+v"(off));
        return off;
    };
    const auto load = [&](const T* at, long long pos, T (&to)[OWN]) __attribute__((always_inline)) {
        const unsigned off = channel();
#pragma unroll
        for (int k = 0; k < OWN; ++k, at += OWNERS * pos) to[k] = *(const T*)((const char*)at + off);
    };
    const auto load_quad = [&](const T* at, int q, SeqVec<T, 4>& to) __attribute__((always_inline)) {
#pragma unroll
        for (int e = 0; e < 4; ++e) to.e[e] = at[min(q + e, a.n - 1)];
    };
    // Places of the next whole tile to load; they stay at the last one.
    const LinRows gate_rows = gate ? a.z : a.x;
    const auto place = [&](const LinRows& r, long long t) { return (const T*)r.p + s * r.seq + t * r.pos; };
    const auto side = [&](int row, long long t) { return (row % SIDES ? place(a.c, t) : place(a.b, t)) + (long long)g * a.n; };
    const long long own_at = LANES == 1 ? t0 : t0 + own;  // (one lane: the same for all of them)
    const T *xp = place(a.x, own_at), *dp = place(a.delta, own_at), *zp = place(gate_rows, own_at), *bp[PER_LANE];
    long long b_move[PER_LANE];
#pragma unroll
    for (int k = 0; k < PER_LANE; ++k) {
        const int row = item_of(k) / (NP / 4);
        bp[k] = side(row, t0 + row / SIDES);
        b_move[k] = SCAN_TILE * (row % SIDES ? a.c.pos : a.b.pos);
    }
    const int whole = (t1 - t0) / SCAN_TILE;
    int ahead = 0;  // whole tiles whose loads have been issued
    const auto fetch = [&](Tile& v) __attribute__((always_inline)) {
        load(xp, a.x.pos, v.x);
        load(dp, a.delta.pos, v.delta);
        if (OUT) load(zp, gate_rows.pos, v.z);
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) load_quad(bp[k], item_of(k) % (NP / 4) * 4, v.bc[k]);
        const bool more = ++ahead < whole;
        xp += more ? SCAN_TILE * a.x.pos : 0;
        dp += more ? SCAN_TILE * a.delta.pos : 0;
        if (OUT) zp += more ? SCAN_TILE * gate_rows.pos : 0;
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) bp[k] += more ? b_move[k] : 0;
    };
    T* op = OUT ? (T*)a.o.p + s * a.o.seq + own_at * a.o.pos : nullptr;
    // n positions from t on (SCAN_TILE but for the last tile), with b and c in s_bc[buf].
    const auto tile = [&](const Tile& v, auto buf_, int n, auto next) __attribute__((always_inline)) {
        constexpr int buf = decltype(buf_)::value;
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) {
            const int item = tid + k * 64 * SCAN_WAVES, q = item_of(k) % (NP / 4) * 4, row = item_of(k) / (NP / 4);
            f32x4 f;
#pragma unroll
            for (int e = 0; e < 4; ++e) f[e] = q + e < a.n ? to_f32(v.bc[k].e[e]) : 0.0f;  // states past the last one: zeros
            if (ITEMS >= (k + 1) * 64 * SCAN_WAVES || item < ITEMS) *(f32x4*)&s_bc[buf][row / SIDES][row % SIDES][q] = f;
        }
        float step[OWN], in[OWN], z[OWN], y[OWN];  // y: begins with d x
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            step[k] = to_f32(v.delta[k]) + bias;
            in[k] = to_f32(v.x[k]);
            if (OUT) {
                y[k] = d * in[k];
                z[k] = to_f32(v.z[k]);
            }
        }
        if (a.softplus) {
#pragma unroll
            for (int k = 0; k < OWN; ++k) step[k] = softplus(step[k]);
        }
#pragma unroll
        for (int k = 0; k < OWN; ++k) in[k] *= step[k];
        __syncthreads();
        next();
        if (idle) return;
        if (!OUT) {
            float sum[OWN];
#pragma unroll
            for (int k = 0; k < OWN; ++k) sum[k] = part < OWNERS && k * OWNERS + own < n ? step[k] : 0.0f;
#pragma unroll
            for (int m = OWN / 2; m > 0; m /= 2)
#pragma unroll
                for (int k = 0; k < m; ++k) sum[k] += sum[k + m];
            steps += sum[0];
        }
        // A position's quads of states one after another. The quads of b and c are read from LDS AHEAD quads before
        // they are used (the barriers keep the compiler from reading them where it needs them, and waiting: outputs of the long
        // sequence above 552 us, with them 511).
        constexpr int QUADS = NS < 4 ? 1 : NS / 4, AHEAD = 2;
        f32x4 b[AHEAD + 1], w[AHEAD + 1];
        const auto read = [&](auto at_) __attribute__((always_inline)) {
            constexpr int at = decltype(at_)::value, i = at / QUADS, q = at % QUADS;
            if constexpr (i < SCAN_TILE) {
                b[at % (AHEAD + 1)] = *(const f32x4*)&s_bc[buf][i][0][(q * LANES + part) * 4];
                if (OUT) w[at % (AHEAD + 1)] = *(const f32x4*)&s_bc[buf][i][SIDES - 1][(q * LANES + part) * 4];
            }
        };
        each<AHEAD>(read);
        __builtin_amdgcn_sched_barrier(0);
        constexpr int REGION = NS > 4 ? 1 : 4;  // quads between which the compiler may move things about
        float st, u, o[SCAN_TILE];
        each<SCAN_TILE * QUADS>([&](auto at_) __attribute__((always_inline)) {
            constexpr int at = decltype(at_)::value, i = at / QUADS, q = at % QUADS, owner = i % OWNERS, k = i / OWNERS;
            read(std::integral_constant<int, at + AHEAD>{});
            if (q == 0) o[i] = 0.0f;
            if (n < SCAN_TILE && i >= n) return;
            if (q == 0) {
                st = lane_value<LANES, owner>(step[k]);
                u = lane_value<LANES, owner>(in[k]);
                asm volatile("" : "+v"(st));  // its products and powers are formed here, not with all of the tile's
                if (OUT && LANES == 1) o[i] = y[k];
            }
#pragma unroll
            for (int e = 0; e < 4 && q * 4 + e < NS; ++e) {
                float& x = h[q * 4 + e];
                x = fmaf(__builtin_amdgcn_exp2f(st * rate[q * 4 + e]), x, u * b[at % (AHEAD + 1)][e]);
                if (OUT) o[i] = fmaf(w[at % (AHEAD + 1)][e], x, o[i]);
            }
            if constexpr (OUT && LANES > 4 && q + 1 == QUADS) {
                const float v = lane_sum(o[i], LANES);
                y[k] += own == owner ? v : 0.0f;
            }
            if (at % REGION == REGION - 1) __builtin_amdgcn_sched_barrier(0);
        });
        if (OUT) {  // each position's sum over the channel's lanes, for the lane that looks after it
            const bool p0 = part & 1, p1 = part & 2;
            const auto pair = [&](float v0, float v1) { return (p0 ? v1 : v0) + dpp<0xb1>(p0 ? v0 : v1); };
#pragma unroll
            for (int k = 0; k < OWN; ++k) {
                if constexpr (LANES == 1) y[k] = o[k];
                else if constexpr (LANES == 2) y[k] += pair(o[2 * k], o[2 * k + 1]);
                else if constexpr (LANES == 4) {
                    const float v0 = pair(o[4 * k], o[4 * k + 1]), v1 = pair(o[4 * k + 2], o[4 * k + 3]);
                    y[k] += (p1 ? v1 : v0) + dpp<0x4e>(p1 ? v0 : v1);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < NS; ++i) asm volatile("" : "+v"(h[i]));  // done here, not behind the next tile's branches
        if (OUT) {
            if (gate)
#pragma unroll
                for (int k = 0; k < OWN; ++k) y[k] *= z[k] * fast_sigmoid(z[k]);
            T* o = op;
            const unsigned off = channel();
#pragma unroll
            for (int k = 0; k < OWN; ++k, o += OWNERS * a.o.pos) {
                if (LANES <= SCAN_TILE && n == SCAN_TILE) {
                    if (on) *(T*)((char*)o + off) = from_f32<T>(y[k]);
                } else if (on && part < OWNERS && k * OWNERS + own < n) {
                    o[c] = from_f32<T>(y[k]);
                }
            }
            op += SCAN_TILE * a.o.pos;
        }
    };
    typedef std::integral_constant<int, 0> Even;
    typedef std::integral_constant<int, 1> Odd;
    Tile even, odd;
    if (whole > 0) {
        fetch(even);
        fetch(odd);
    }
    int j = 0;
    for (; j + 1 < whole; j += 2) {
        Tile v = even;
        tile(v, Even(), SCAN_TILE, [&]() __attribute__((always_inline)) { fetch(even); });
        v = odd;
        tile(v, Odd(), SCAN_TILE, [&]() __attribute__((always_inline)) { fetch(odd); });
    }
    if (j < whole) tile(even, Even(), SCAN_TILE, []() {});
    if (const int n = (t1 - t0) - whole * SCAN_TILE; n > 0) {
        // Positions past the last one: its values, not used.
        Tile v;
        const int first = t0 + whole * SCAN_TILE;
#pragma unroll
        for (int k = 0; k < OWN; ++k) {
            const int t = min(first + k * OWNERS + own, t1 - 1);
            v.x[k] = place(a.x, t)[c];
            v.delta[k] = place(a.delta, t)[c];
            if (OUT) v.z[k] = place(gate_rows, t)[c];
        }
#pragma unroll
        for (int k = 0; k < PER_LANE; ++k) {
            const int row = item_of(k) / (NP / 4);
            load_quad(side(row, min(first + row / SIDES, t1 - 1)), item_of(k) % (NP / 4) * 4, v.bc[k]);
        }
        if (j < whole) tile(v, Odd(), n, []() {});
        else tile(v, Even(), n, []() {});
    }
    if (!OUT) {
        const float sum = lane_sum((float)steps, LANES);
        if (on && part == 0) scratch[step_slot(a, p, s, seg) + c] = sum;
    }
    if (!on) return;
    float* to = nullptr;
    if (!OUT) to = scratch + scan_slot(a, p, s, seg);
    else if (a.s_out && seg + 1 == live) to = a.s_out;
    if (!to) return;
#pragma unroll
    for (int i = 0; i < NS; ++i) {
        const int n = state(i);
        if (n < a.n) to[OUT ? ((long long)s * a.channels + c) * a.n + n : (long long)n * a.channels + c] = h[i];
    }
}

template <typename T, bool OUT>
hipError_t scan(const ScanArgs& a, const ScanPlan& p, float* scratch, hipStream_t s) {
    const unsigned grid = (unsigned)(a.seqs * (OUT ? p.segments : p.segments - 1) * a.groups * p.blocks);
    const dim3 block(64 * p.waves);
    switch (p.ns * 100 + p.lanes) {
        case 101: k_scan<T, 1, 1, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 401: k_scan<T, 4, 1, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 404: k_scan<T, 4, 4, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 801: k_scan<T, 8, 1, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1201: k_scan<T, 12, 1, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1202: k_scan<T, 12, 2, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1204: k_scan<T, 12, 4, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1601: k_scan<T, 16, 1, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1602: k_scan<T, 16, 2, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1604: k_scan<T, 16, 4, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1608: k_scan<T, 16, 8, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        case 1616: k_scan<T, 16, 16, OUT><<<grid, block, 0, s>>>(a, p, scratch); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace
}  // namespace zjai

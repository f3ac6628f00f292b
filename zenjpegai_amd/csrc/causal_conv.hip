// Short causal convolution of each channel over the positions of its sequence (gfx950 / CDNA4, wave64):
//   out_t = act(bias + sum_j w_j x_(t - taps + 1 + j)).
//
// HBM bound: inputs and outputs pass once. A lane owns four channels and walks a run of positions, the last
// inputs kept in registers, the next eight positions' loads issued together. Runs of 16 positions: longer ones leave SIMDs
// without work (135 rows of 240 positions of 384 channels bf16: 64 positions 18.2 us, 32 14.3, 16 11.9, 8 12.9, a copy
// of as many bytes 9.9), shorter ones read more of the inputs twice (12 sequences of 0-3001 of 2048 f16: 51, 44, 42, 45).
// Eight channels of 16 bits a lane halve the lanes (14.9 and 45 us); taking neighbouring runs to one XCD's L2 gains
// nothing (11.8 and 43) or leaves XCDs without work where lengths differ (48).

#include <algorithm>

#include "sequence.h"

namespace zjai {

namespace {

constexpr int CONV_AHEAD = 8;  // positions whose loads are issued together

struct ConvPlan {
    int vecs;       // accesses of a position
    int run, runs;  // positions of a run, runs of a sequence
    bool wide;      // weights and bias 16-byte aligned
};

// Weights and bias of VE channels.
template <int VE, int K>
struct ConvWeights {
    float w[VE][K], b[VE];
    __device__ __forceinline__ ConvWeights(const CausalConvArgs& a, int c, bool wide) {
        if (VE % 4 == 0 && wide) {  // 16 bytes at a time
#pragma unroll
            for (int i = 0; i < VE * K; i += 4) {
                const f32x4 v = *(const f32x4*)(a.weight + (long long)c * K + i);
#pragma unroll
                for (int k = 0; k < 4; ++k) w[(i + k) / K][(i + k) % K] = v[k];
            }
#pragma unroll
            for (int e = 0; e < VE; e += 4) {
                const f32x4 v = a.bias ? *(const f32x4*)(a.bias + c + e) : f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < 4; ++k) b[e + k] = v[k];
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < VE; ++e) {
#pragma unroll
            for (int j = 0; j < K; ++j) w[e][j] = a.weight[(long long)(c + e) * K + j];
            b[e] = a.bias ? a.bias[c + e] : 0.0f;
        }
    }
};

template <typename T, int VE, int K>
__global__ void __launch_bounds__(256) k_causal_conv(CausalConvArgs a, ConvPlan p) {
    typedef SeqVec<T, VE> V;
    const long long items = (long long)a.seqs * p.runs * p.vecs;
    for (long long item = (long long)blockIdx.x * 256 + threadIdx.x; item < items; item += (long long)gridDim.x * 256) {
        int cv, run, s;
        if (items <= INT_MAX) {
            const unsigned r = (unsigned)item / (unsigned)p.vecs;
            cv = (unsigned)item - r * p.vecs;
            s = r / (unsigned)p.runs;
            run = r - s * p.runs;
        } else {
            const long long r = item / p.vecs;
            cv = (int)(item - r * p.vecs);
            s = (int)(r / p.runs);
            run = (int)(r - (long long)s * p.runs);
        }
        const int c = cv * VE, len = seq_length(a.lengths, s, a.length), t0 = run * p.run, t1 = min(t0 + p.run, len);
        const bool keeps = run == 0 && K > 1 && a.s_out;  // a sequence's first run takes its state on as well
        if (t0 >= t1 && !keeps) continue;
        const T* x = (const T*)a.x.p + s * a.x.seq + c;
        const T* before = a.s_in && K > 1 ? (const T*)a.s_in + (long long)s * (K - 1) * a.channels + c : nullptr;
        // The input at position t of the sequence, which may lie up to K - 1 positions before the first.
        const auto input = [&](int t) {
            V v;
            if (t >= 0) {
                v = *(const V*)(x + t * a.x.pos);
            } else if (before) {
                v = *(const V*)(before + (long long)(t + K - 1) * a.channels);
            } else {
#pragma unroll
                for (int e = 0; e < VE; ++e) v.e[e] = from_f32<T>(0.0f);
            }
            return v;
        };
        if (t0 < t1) {
            const ConvWeights<VE, K> w(a, c, p.wide);
            float in[K + CONV_AHEAD - 1][VE];  // the last K - 1 inputs, then the new ones
#pragma unroll
            for (int j = 0; j < K - 1; ++j) {
                const V v = input(t0 - (K - 1) + j);
#pragma unroll
                for (int e = 0; e < VE; ++e) in[j][e] = to_f32(v.e[e]);
            }
            const T* from = x + t0 * a.x.pos;
            T* o = (T*)a.o.p + s * a.o.seq + t0 * a.o.pos + c;
            for (int t = t0; t < t1; t += CONV_AHEAD) {
                V v[CONV_AHEAD];
#pragma unroll
                for (int i = 0; i < CONV_AHEAD; ++i) {
                    v[i] = *(const V*)from;
                    if (t + i + 1 < t1) from += a.x.pos;  // past the run's last position: it once more, not used
                }
#pragma unroll
                for (int i = 0; i < CONV_AHEAD; ++i) {
                    V y;
#pragma unroll
                    for (int e = 0; e < VE; ++e) {
                        in[K - 1 + i][e] = to_f32(v[i].e[e]);
                        float sum = w.b[e];
#pragma unroll
                        for (int j = 0; j < K; ++j) sum = fmaf(w.w[e][j], in[i + j][e], sum);
                        y.e[e] = from_f32<T>(gate_act(sum, a.act));
                    }
                    if (t + i < t1) *(V*)o = y;
                    o += a.o.pos;
                }
#pragma unroll
                for (int j = 0; j < K - 1; ++j)
#pragma unroll
                    for (int e = 0; e < VE; ++e) in[j][e] = in[CONV_AHEAD + j][e];
            }
        }
        if constexpr (K > 1)
            if (keeps) {  // read before it is written: the state may be updated in place
                V last[K - 1];
#pragma unroll
                for (int j = 0; j < K - 1; ++j) last[j] = input(len - (K - 1) + j);
                T* to = (T*)a.s_out + (long long)s * (K - 1) * a.channels + c;
#pragma unroll
                for (int j = 0; j < K - 1; ++j) *(V*)(to + (long long)j * a.channels) = last[j];
            }
    }
}

// One position of each sequence: a workgroup takes a block of channels of one (or of all that share a slot).
template <typename T, int VE, int K>
__global__ void __launch_bounds__(256) k_causal_conv_step(CausalConvArgs a, int vecs, int blocks, bool wide) {
    typedef SeqVec<T, VE> V;
    __shared__ int s_next;
    const int first = blockIdx.x / blocks, cv = (blockIdx.x - first * blocks) * blockDim.x + threadIdx.x;
    SlotChain chain{a.slots, a.num_slots, a.seqs, &s_next};
    if (!chain.enter(first)) return;
    const bool on = cv < vecs;
    const int c = on ? cv * VE : 0;
    const ConvWeights<VE, K> w(a, c, wide);
    const long long sbase = (long long)chain.slot * (K - 1) * a.channels + c;
    V in[K];
#pragma unroll
    for (int j = 0; j < K - 1; ++j) in[j] = *(const V*)((const T*)a.s_in + sbase + (long long)j * a.channels);
    in[K - 1] = *(const V*)((const T*)a.x.p + (long long)first * a.x.seq + c);
    // (All these are in flight while the sequences of the slot are looked for.)
    if (!chain.alone_or_first(first)) return;
    for (int s = first; s != INT_MAX;) {
        V y;
#pragma unroll
        for (int e = 0; e < VE; ++e) {
            float sum = w.b[e];
#pragma unroll
            for (int j = 0; j < K; ++j) sum = fmaf(w.w[e][j], to_f32(in[j].e[e]), sum);
            y.e[e] = from_f32<T>(gate_act(sum, a.act));
        }
        if (on) *(V*)((T*)a.o.p + (long long)s * a.o.seq + c) = y;
#pragma unroll
        for (int j = 0; j < K - 1; ++j) in[j] = in[j + 1];
        s = chain.next();
        if (s != INT_MAX) in[K - 1] = *(const V*)((const T*)a.x.p + (long long)s * a.x.seq + c);
    }
    if (!on) return;
#pragma unroll
    for (int j = 0; j < K - 1; ++j) *(V*)((T*)a.s_out + sbase + (long long)j * a.channels) = in[j];
}

// Elements of an access: four channels, two of 16 bits, or one.
int conv_vector(const CausalConvArgs& a, int es) {
    const auto fits = [&](int v) {
        if (a.channels % v) return false;
        for (const LinRows* r : {&a.x, &a.o})
            if ((uintptr_t)r->p % (v * es) || r->pos % v || r->seq % v) return false;
        return ((uintptr_t)a.s_in | (uintptr_t)a.s_out) % (v * es) == 0;
    };
    if (fits(4)) return 4;
    return es == 2 && fits(2) ? 2 : 1;
}

template <typename T, int VE, int K>
void conv_taps(const CausalConvArgs& a, bool step, hipStream_t s) {
    const int vecs = a.channels / VE;
    const bool wide = (((uintptr_t)a.weight | (uintptr_t)a.bias) & 15) == 0;
    if (step) {
        const int threads = std::min(256, (vecs + 63) / 64 * 64), blocks = (vecs + threads - 1) / threads;
        k_causal_conv_step<T, VE, K><<<(unsigned)(a.seqs * blocks), threads, 0, s>>>(a, vecs, blocks, wide);
        return;
    }
    ConvPlan p{};
    p.vecs = vecs;
    p.run = 16;
    p.wide = wide;
    p.runs = std::max(1, (a.length + p.run - 1) / p.run);
    const long long items = (long long)a.seqs * p.runs * vecs;
    k_causal_conv<T, VE, K><<<(unsigned)std::min<long long>((items + 255) / 256, 1 << 20), 256, 0, s>>>(a, p);
}
template <typename T, int VE>
hipError_t conv_of(const CausalConvArgs& a, bool step, hipStream_t s) {
    switch (a.taps) {
        case 1: conv_taps<T, VE, 1>(a, step, s); break;
        case 2: conv_taps<T, VE, 2>(a, step, s); break;
        case 3: conv_taps<T, VE, 3>(a, step, s); break;
        case 4: conv_taps<T, VE, 4>(a, step, s); break;
        case 5: conv_taps<T, VE, 5>(a, step, s); break;
        case 6: conv_taps<T, VE, 6>(a, step, s); break;
        case 7: conv_taps<T, VE, 7>(a, step, s); break;
        default: conv_taps<T, VE, 8>(a, step, s);
    }
    return hipGetLastError();
}
template <typename T>
hipError_t conv_vec(const CausalConvArgs& a, bool step, hipStream_t s) {
    const int ve = conv_vector(a, sizeof(T));
    if (ve == 4) return conv_of<T, 4>(a, step, s);
    if constexpr (sizeof(T) == 2)
        if (ve == 2) return conv_of<T, 2>(a, step, s);
    return conv_of<T, 1>(a, step, s);
}
hipError_t conv(const CausalConvArgs& a, int dtype, bool step, hipStream_t s) {
    if (dtype == DT_F32) return conv_vec<float>(a, step, s);
    if (dtype == DT_F16) return conv_vec<_Float16>(a, step, s);
    return conv_vec<__bf16>(a, step, s);
}

}  // namespace

std::string causal_conv_name(const CausalConvArgs& a, int dtype, bool step) {
    return std::string(step ? "k_causal_conv_step<" : "k_causal_conv<") + type_name(dtype) + ", " +
           std::to_string(conv_vector(a, dtype == DT_F32 ? 4 : 2)) + ", " + std::to_string(a.taps) + ">";
}

hipError_t launch_causal_conv(const CausalConvArgs& a, int dtype, hipStream_t s) { return conv(a, dtype, false, s); }
hipError_t launch_causal_conv_step(const CausalConvArgs& a, int dtype, hipStream_t s) { return conv(a, dtype, true, s); }

}  // namespace zjai

// Rotary positions (gfx950 / CDNA4, wave64): pairs (a, b) of channels become
//   m (a cos(p f) - b sin(p f)),  m (a sin(p f) + b cos(p f)).
//
// HBM bound: every channel passes once. A workgroup takes a tile of positions: its lanes first form the tile's sines and
// cosines, one for each pair and position however many heads there are, in LDS, then walk over the channels of the
// tile's positions, which lie behind one another, 16 bytes a lane (65536 positions of 32 heads of 128 channels, 64 of them turned, bf16:
// 215 us, 5.0 TB/s, a copy 213; the 64 x 64 map of 10 heads of 32 f32: 4.5 us, a launch).

#include <algorithm>

#include "sequence.h"

namespace zjai {

namespace {

struct RotaryPlan {
    int tp;               // positions of a tile
    int turn, copy;       // accesses of a head's turned channels (a pair of them with halves) and of the others
    int tiles;            // of a sequence
};

// (magnitude cos, magnitude sin) of p f. The angle loses its whole turns in 64 bits (two products and a constant, each off by
// 2^-53 of itself, are within 2^-51 of the angle: 2^-33 of a radian at 2^18), down to an eighth of a turn to either side; there the power series up to the ninth and
// tenth order are exact to 2^-27 and 2^-31.
__device__ __forceinline__ float2 rotary_turn(int p, double f, float magnitude) {
    const double turns = (double)p * f * 0.15915494309189533577;  // 1 / (2 pi)
    const double quarter = rint(turns * 4.0);
    const float r = (float)((turns - quarter * 0.25) * 6.28318530717958647693), r2 = r * r;
    const int q = (int)(quarter - 4.0 * floor(quarter * 0.25));
    float s = fmaf(r2, 1.0f / 362880.0f, -1.0f / 5040.0f);
    s = fmaf(s, r2, 1.0f / 120.0f);
    s = fmaf(s, r2, -1.0f / 6.0f);
    s = fmaf(s * r2, r, r);
    float c = fmaf(r2, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = fmaf(c, r2, -1.0f / 720.0f);
    c = fmaf(c, r2, 1.0f / 24.0f);
    c = fmaf(c, r2, -0.5f);
    c = fmaf(c, r2, 1.0f);
    float2 v;
    v.x = (q & 1) ? s : c;
    v.y = (q & 1) ? c : s;
    if (q == 1 || q == 2) v.x = -v.x;
    if (q == 2 || q == 3) v.y = -v.y;
    v.x *= magnitude;
    v.y *= magnitude;
    return v;
}

template <typename T, int VE, bool HALVES>
__global__ void __launch_bounds__(256) k_rotary(RotaryArgs a, RotaryPlan p) {
    typedef SeqVec<T, VE> V;
    extern __shared__ float2 s_turn[];  // [tp][turned / 2]
    const int tid = threadIdx.x, pairs = a.turned / 2, per_head = p.turn + p.copy, per_pos = per_head * a.heads;
    const long long tiles = (long long)a.seqs * p.tiles;
    for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
        const int s = (int)(tile / p.tiles), t0 = (int)(tile - (long long)s * p.tiles) * p.tp;
        const int n = min(p.tp, seq_length(a.lengths, s, a.length) - t0);
        if (n <= 0) continue;
        const int start = a.starts ? a.starts[s] : 0;
        __syncthreads();  // the last tile's turns have been used
        for (int e = tid; e < n * pairs; e += 256) {
            const int t = e / pairs, i = e - t * pairs;
            int at = (int)((unsigned)(a.positions ? a.positions[(long long)s * a.length + t0 + t] : t0 + t) + (unsigned)start);
            if (a.map > 0) {
                int row = at / a.map;
                row -= at < row * a.map;  // downwards for places before the first
                at = 2 * i < pairs ? row : at - row * a.map;
            }
            s_turn[e] = rotary_turn(at, a.freq[i], a.magnitude);
        }
        __syncthreads();
        // A lane keeps its channels over the tile's positions: `beside` of these lie side by side in the workgroup.
        const int beside = max(1, 256 / per_pos), t_first = beside > 1 ? tid / per_pos : 0;
        for (int in_pos = t_first < beside ? tid - t_first * per_pos : per_pos; in_pos < per_pos; in_pos += 256) {
            const int h = in_pos / per_head, k = in_pos - h * per_head;
            for (int t = t_first; t < n; t += beside) {
                const T* x = (const T*)a.x.p + seq_at(a.x, a.width, s, t0 + t) + (long long)h * a.dim;
                T* o = (T*)a.o.p + seq_at(a.o, a.width, s, t0 + t) + (long long)h * a.dim;
                if (k >= p.turn) {
                    const int c = a.turned + (k - p.turn) * VE;
                    *(V*)(o + c) = *(const V*)(x + c);
                    continue;
                }
                if constexpr (HALVES || VE == 1) {  // two accesses, the pairs across them
                    const float2* cs = s_turn + t * pairs + k * VE;
                    const int c0 = HALVES ? k * VE : 2 * k, c1 = HALVES ? pairs + k * VE : 2 * k + 1;
                    const V va = *(const V*)(x + c0), vb = *(const V*)(x + c1);
                    V oa, ob;
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const float u = to_f32(va.e[i]), v = to_f32(vb.e[i]), sn = a.inverse ? -cs[i].y : cs[i].y;
                        oa.e[i] = from_f32<T>(fmaf(u, cs[i].x, -(v * sn)));
                        ob.e[i] = from_f32<T>(fmaf(u, sn, v * cs[i].x));
                    }
                    *(V*)(o + c0) = oa;
                    *(V*)(o + c1) = ob;
                } else {  // one, the pairs within it
                    const float2* cs = s_turn + t * pairs + k * (VE / 2);
                    const V va = *(const V*)(x + k * VE);
                    V oa;
#pragma unroll
                    for (int i = 0; i < VE / 2; ++i) {
                        const float u = to_f32(va.e[2 * i]), v = to_f32(va.e[2 * i + 1]), sn = a.inverse ? -cs[i].y : cs[i].y;
                        oa.e[2 * i] = from_f32<T>(fmaf(u, cs[i].x, -(v * sn)));
                        oa.e[2 * i + 1] = from_f32<T>(fmaf(u, sn, v * cs[i].x));
                    }
                    *(V*)(o + k * VE) = oa;
                }
            }
        }
    }
}

// Elements of an access: the most, up to 16 bytes, that divide the heads' parts and keep every place aligned.
int rotary_vector(const RotaryArgs& a, int es) {
    int ve = 16 / es;
    const auto fits = [&](int v) {
        if (a.dim % v || (a.halves ? a.turned / 2 : a.turned) % v) return false;
        for (const LinRows* r : {&a.x, &a.o})
            if ((uintptr_t)r->p % (v * es) || r->pos % v || r->seq % v || (a.width && r->row % v)) return false;
        return true;
    };
    while (ve > 1 && !fits(ve)) ve /= 2;
    return ve;
}

RotaryPlan rotary_plan(const RotaryArgs& a, int ve, int es) {
    RotaryPlan p{};
    p.turn = a.halves ? a.turned / 2 / ve : a.turned / std::max(ve, 2);
    p.copy = a.x.p == a.o.p ? 0 : (a.dim - a.turned) / ve;
    const long long per_pos = (long long)(p.turn + p.copy) * a.heads;
    // Accesses a lane: five of 16 bytes, eight of fewer. 512 MB into as many, us with four, five, eight: heads of 128 (32, bf16, from
    // packed channels) 220, 215, 215, of 160 (13, f16) 199, 204, 217, both 16 bytes; 10 heads of 100 in 8 bytes (f16) 258, 244, 237, 8 in
    // 4 bytes 297, 304, 277. Fewer where that leaves CUs idle; 16 KB of turns at most. A count that leaves lanes idle costs
    // little, as HBM is what bounds them (heads of 80 f16: 16, 160 accesses a position, 200 us; 13, 130 of them, 222).
    const long long lane = ve * es == 16 ? 5 : 8;
    const long long want = std::max<long long>(1, 256 * lane / per_pos), spread = std::max<long long>(1, (long long)a.seqs * a.length / 1024);
    p.tp = (int)std::min({want, spread, (long long)(2048 / (a.turned / 2)), (long long)a.length});
    p.tiles = (a.length + p.tp - 1) / p.tp;
    return p;
}

template <typename T, int VE>
void rotary_of(const RotaryArgs& a, hipStream_t s) {
    const RotaryPlan p = rotary_plan(a, VE, sizeof(T));
    const unsigned grid = (unsigned)std::min<long long>((long long)a.seqs * p.tiles, 1 << 16);
    const size_t lds = sizeof(float2) * p.tp * (a.turned / 2);
    if (a.halves) k_rotary<T, VE, true><<<grid, 256, lds, s>>>(a, p);
    else k_rotary<T, VE, false><<<grid, 256, lds, s>>>(a, p);
}

template <typename T>
hipError_t rotary(const RotaryArgs& a, hipStream_t s) {
    const int ve = rotary_vector(a, sizeof(T));
    if constexpr (sizeof(T) == 2)
        if (ve == 8) {
            rotary_of<T, 8>(a, s);
            return hipGetLastError();
        }
    if (ve == 4) rotary_of<T, 4>(a, s);
    else if (ve == 2) rotary_of<T, 2>(a, s);
    else rotary_of<T, 1>(a, s);
    return hipGetLastError();
}

}  // namespace

std::string rotary_name(const RotaryArgs& a, int dtype) {
    return std::string("k_rotary<") + type_name(dtype) + ", " + std::to_string(rotary_vector(a, dtype == DT_F32 ? 4 : 2)) +
           (a.halves ? ", true>" : ", false>");
}

hipError_t launch_rotary(const RotaryArgs& a, int dtype, hipStream_t s) {
    if (dtype == DT_F32) return rotary<float>(a, s);
    if (dtype == DT_F16) return rotary<_Float16>(a, s);
    return rotary<__bf16>(a, s);
}

}  // namespace zjai

// Device helpers of the operators that work on sequences of positions (rotary positions, causal convolution, selective
// scan).
#pragma once

#include <climits>

#include "device.h"
#include "ops.h"

namespace zjai {

// Offset of position t of sequence s, in elements.
__device__ __forceinline__ long long seq_at(const LinRows& r, int width, long long s, int t) {
    const long long base = s * r.seq;
    if (width == 0) return base + (long long)t * r.pos;
    const int y = t / width;
    return base + (long long)y * r.row + (long long)(t - y * width) * r.pos;
}

// Positions that sequence s has.
__device__ __forceinline__ int seq_length(const int* lengths, int s, int room) {
    return lengths ? max(0, min(lengths[s], room)) : room;
}

// 1 / (1 + exp(-v)) by the hardware's 2^x: relative error (|v| + 2) 2^-24, as the rounding of v log2 e leaves any.
__device__ __forceinline__ float fast_sigmoid(float v) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(v * -1.44269504088896340736f));
}
__device__ __forceinline__ float gate_act(float v, int act) {
    if (act == GATE_LINEAR) return v;
    const float s = fast_sigmoid(v);
    return act == GATE_SIGMOID ? s : v * s;
}

// The sequences of one slot, for a workgroup that starts at sequence `first`: the first of them takes them all, in
// order. enter: its slot, and whether there is one; alone_or_first: whether this workgroup has them (all lanes get the same
// answer); next: the sequence after the current one, or INT_MAX. The workgroup's lanes share the search (a step of 257
// sequences of 2048 channels x 16 states 20.0 us, each wave for itself, without a barrier, 21.8, without slots 16.2). Every workgroup
// reads all slots, so the search grows with the square of the sequences: 1024 of them 71 us (52 without slots), 4096 474 (243).
struct SlotChain {
    const int* slots;
    int num_slots, seqs;
    int* s_next;  // shared
    int slot = 0, after = INT_MAX;
    bool alone = false;

    __device__ __forceinline__ bool enter(int first) {
        slot = slots ? slots[first] : first;
        alone = !slots || seqs == 1;
        return !slots || (unsigned)slot < (unsigned)num_slots;
    }
    __device__ __forceinline__ bool alone_or_first(int first) {
        if (alone) return true;
        if (threadIdx.x == 0) *s_next = INT_MAX;
        __syncthreads();
        int earlier = 0, later = INT_MAX;
        for (int j = threadIdx.x; j < seqs; j += blockDim.x)
            if (slots[j] == slot) {
                earlier |= j < first;
                if (j > first) later = min(later, j);
            }
        if (later != INT_MAX) atomicMin(s_next, later);
        if (__syncthreads_or(earlier)) return false;
        after = *s_next;
        return true;
    }
    __device__ __forceinline__ int next() {
        const int cur = after;
        if (alone || cur == INT_MAX) return cur;
        __syncthreads();
        if (threadIdx.x == 0) *s_next = INT_MAX;
        __syncthreads();
        for (int j = cur + 1 + threadIdx.x; j < seqs; j += blockDim.x)
            if (slots[j] == slot) {
                atomicMin(s_next, j);
                break;
            }
        __syncthreads();
        after = *s_next;
        return cur;
    }
};

// VE elements as one access.
template <typename T, int VE> struct alignas(sizeof(T) * VE) SeqVec { T e[VE]; };

inline const char* type_name(int dtype) { return dtype == DT_F32 ? "float" : dtype == DT_F16 ? "_Float16" : "__bf16"; }

}  // namespace zjai

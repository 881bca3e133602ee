// The 4-bit KV cache: its layout and its arithmetic, shared by the kernels
// that write it, read it back and attend over it.
//
// A cache is `pages` pages of `page_size` positions (a multiple of 16).  A
// page holds one block per kv head, and a block, for D = head_dim values a
// row and NG = D / 32 groups a row:
//   K codes  [page_size][D / 2 bytes]
//   V codes  [page_size][D / 2 bytes]
//   K scales [page_size][NG] fp16
//   V scales [page_size][NG] fp16
// so a position costs D + D / 8 bytes (K and V together) and every section
// starts on a 32-byte boundary.  A group of 32 values is d * (c - 8) with
// c in 0..15.  Inside a row the codes are ordered for the attention kernel's
// matrix fragments:
//   K: word (c, g), c < 4, at byte 4 (c NG + g): dims 32 g + 8 c + i in bits 4 i
//   V: halfword (r, g), r < 8, at byte 2 (r NG + g): dims 32 g + 4 r + i in bits 4 i
#pragma once

#include "common.cuh"

namespace alj {

__device__ __forceinline__ long long kv4_block_bytes(int page_size, int head_dim) {
    return static_cast<long long>(page_size) * (head_dim + head_dim / 8);
}

// Scale of a group from its extremes: d = ext / -8 in fp16, ext the extreme
// of larger magnitude (the negative one when both are equal), so ext itself
// has code 0.  |d| saturates at 65504; a group that holds an infinity or a
// NaN gets a NaN scale, and all its values read back as NaN.
__device__ __forceinline__ __half kv4_scale(float mn, float mx, bool finite) {
    const float ext = -mn >= mx ? mn : mx;
    const float d = fminf(fmaxf(ext * -0.125f, -65504.0f), 65504.0f);
    return finite ? __float2half_rn(d) : __ushort_as_half(0x7E00);
}
// Reciprocal of the rounded scale: one division a group, and the same
// products as the definition x * (1 / d).
__device__ __forceinline__ float kv4_inverse(__half d) {
    const float f = __half2float(d);
    return f == 0.0f ? 0.0f : __fdiv_rn(1.0f, f);
}
// x / d clamped to -8..7 and rounded to the nearest integer, ties to even, as
// the sum with 1.5 * 2^23 + 8: its low four bits are the code, and less that
// number it is the code's integer c - 8.
constexpr float kKv4Round = 12582920.0f;
__device__ __forceinline__ float kv4_rounded(float x, float inv) {
    return __fadd_rn(fminf(fmaxf(__fmul_rn(x, inv), -8.0f), 7.0f), kKv4Round);
}
// The value a code stands for; exact in fp32 (4-bit x 11-bit product).  The
// added zero turns -0 into +0, as the Q4_0 dequantisation does.
__device__ __forceinline__ float kv4_value(uint32_t c, float d) {
    return __fadd_rn(__fmul_rn(static_cast<float>(static_cast<int>(c) - 8), d), 0.0f);
}

// ---------------------------------------------------------------- trees of drafted tokens
// A tree of up to kKv4MaxNodes nodes is given by parents[t] < t: -1 for a
// root, -2 for a node that is absent, as is one whose parent is.  Anything else
// is no tree: the node counts as absent and a fault is recorded.
constexpr int kKv4TreeWords = kKv4MaxNodes / 32;

__device__ __forceinline__ int tree_parent(const int* parents, int t) {
    const int up = __ldg(parents + t);
    if (up >= -2 && up < t) return up;
    record_fault(ALJ_FAULT_BOUNDS);
    return -2;
}
__device__ __forceinline__ bool tree_sees(const uint32_t* words, int node) { return (words[node >> 5] >> (node & 31)) & 1u; }
// Depth of node t, itself counted (0: absent); see: bits of the last `window` nodes of its path (0: of all of it).
__device__ __forceinline__ int tree_chain(const int* parents, int t, int window, uint32_t* see) {
    for (int i = 0; i < kKv4TreeWords; ++i) see[i] = 0u;
    int depth = 0;
    for (; t >= 0; t = parents[t], ++depth)        // parents come first: at most t steps
        if (window == 0 || depth < window) see[t >> 5] |= 1u << (t & 31);
    if (t == -1) return depth;
    for (int i = 0; i < kKv4TreeWords; ++i) see[i] = 0u;
    return 0;
}

}  // namespace alj

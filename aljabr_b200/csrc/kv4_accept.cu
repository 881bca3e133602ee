// Acceptance of a drafted tree over the 4-bit KV cache (layout and trees: kv4.cuh).
//
// Node 0 is the token that the model emitted last.  From node t the walk goes
// on to the first child u (lowest index) with drafted[u] = picked[t], the
// model's own token after t, until there is none.  The rows of the path's i-th
// node then move from position base + path[i] to base + i, base = len - nodes,
// in every layer's cache, and the sequence ends there.
//
// One launch for all layers: a CTA does some layers of one sequence and walks for
// itself.  The walk is one pass over the nodes (the lowest child that fits, by
// an atomic minimum: its result does not depend on the order) and then one
// shared-memory load a step.  A row's move is a column of 32-bit words a
// thread, in the path's order: path[i] >= i, so a row is read before another
// is written over it, also with the reads of the next rows ahead.
#include "kv4.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kThreads = 256;
constexpr int kBatch = 4;            // rows read before the first of them is written

__global__ void __launch_bounds__(kThreads) kv4_accept_kernel(const __grid_constant__ Kv4Accept p, int per_cta) {
    __shared__ int s_par[kKv4MaxNodes], s_next[kKv4MaxNodes], s_picked[kKv4MaxNodes], s_path[kKv4MaxNodes];
    __shared__ int2 s_src[kKv4MaxNodes], s_dst[kKv4MaxNodes];        // page and row in it; page -1: nothing to move
    __shared__ int s_count;
    pdl_launch_dependents();
    pdl_wait();
    const int layer0 = blockIdx.x * per_cta, b = blockIdx.y;
    const int* parents = p.parents + static_cast<long long>(b) * p.parents_stride;
    const long long row0 = static_cast<long long>(b) * p.nodes;
    const int len = __ldg(p.lens + b);
    const long long cap = p.table ? static_cast<long long>(p.table_stride) * p.page_size : p.page_size;
    if (threadIdx.x == 0 && (len < 0 || len > cap)) record_fault(ALJ_FAULT_BOUNDS);
    const int base = len >= p.nodes && len <= cap ? len - p.nodes : -1;    // -1: no tree is there
    for (int t = threadIdx.x; t < p.nodes; t += kThreads) {
        s_par[t] = tree_parent(parents, t);
        s_next[t] = p.nodes;
        s_picked[t] = __ldg(p.picked + row0 + t);
        s_path[t] = -1;
    }
    __syncthreads();
    for (int t = threadIdx.x; t < p.nodes; t += kThreads)
        if (s_par[t] >= 0 && __ldg(p.drafted + row0 + t) == s_picked[s_par[t]]) atomicMin(s_next + s_par[t], t);
    __syncthreads();
    if (threadIdx.x == 0) {
        int n = 0, last = -1;
        for (int t = base >= 0 && s_par[0] == -1 ? 0 : p.nodes; t < p.nodes; t = s_next[t]) {   // children come after their parents
            s_path[n++] = t;
            last = t;
        }
        s_count = n;
        if (layer0 == 0) {
            p.count[b] = n;
            p.token[b] = last >= 0 ? s_picked[last] : -1;
            p.new_lens[b] = base >= 0 ? base + n : len;
        }
    }
    __syncthreads();
    const int count = s_count;
    if (layer0 == 0)
        for (int t = threadIdx.x; t < p.nodes; t += kThreads) p.path[row0 + t] = s_path[t];

    // where the rows are and go, but for those in place already and pages that are not there
    for (int i = threadIdx.x; i < count; i += kThreads) {
        auto place = [&](int pos) {
            const int pi = pos / p.page_size;
            int page = p.table ? __ldg(p.table + static_cast<long long>(b) * p.table_stride + pi) : b;
            if (page < 0 || page >= p.pages) {
                record_fault(ALJ_FAULT_BOUNDS);
                page = -1;
            }
            return make_int2(page, pos - pi * p.page_size);
        };
        int2 from = make_int2(-1, 0), to = from;
        if (s_path[i] != i) from = place(base + s_path[i]), to = place(base + i);
        if (to.x < 0) from.x = -1;
        s_src[i] = from;
        s_dst[i] = to;
    }
    __syncthreads();
    // a row of a head: K codes and V codes of D / 8 words, K scales and V scales of D / 64
    const int code = p.head_dim / 8, scale = p.head_dim / 64, words = 2 * (code + scale);
    const long long block = kv4_block_bytes(p.page_size, p.head_dim) / 4, ps = p.page_size;
    const int columns = words * p.kv_heads, layers = min(per_cta, p.layers - layer0);
    for (int n = threadIdx.x; n < columns * layers; n += kThreads) {
        const int layer = n / columns, c = n - layer * columns, head = c / words, w = c - head * words;
        uint32_t* const cache = reinterpret_cast<uint32_t*>(p.cache[layer0 + layer]);
        const bool is_code = w < 2 * code;
        const int wide = is_code ? code : scale, which = is_code ? w / code : (w - 2 * code) / scale;
        const long long section = is_code ? which * ps * code : ps * (2 * code + which * scale);
        const long long word = section + (is_code ? w - which * code : w - 2 * code - which * scale);
        auto at = [&](int2 place) { return cache + (static_cast<long long>(place.x) * p.kv_heads + head) * block + word + static_cast<long long>(place.y) * wide; };
        for (int i = 1; i < count; i += kBatch) {
            uint32_t x[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (i + j < count && s_src[i + j].x >= 0) x[j] = *at(s_src[i + j]);
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (i + j < count && s_src[i + j].x >= 0) *at(s_dst[i + j]) = x[j];
        }
    }
}

}  // namespace

cudaError_t launch_kv4_accept(const Kv4Accept& p, int sms, cudaStream_t stream) {
    // as many layers a CTA as leave four CTAs an SM: with one each, 32 layers of 64 sequences took 14.4 us in two waves
    const int per_cta = std::max(1, static_cast<int>(static_cast<long long>(p.layers) * p.batch / (4 * sms)));

    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((p.layers + per_cta - 1) / per_cta, p.batch);
    cfg.blockDim = dim3(kThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_accept_kernel, p, per_cta);
}

}  // namespace alj

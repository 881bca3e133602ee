// The logits step of a decode loop, one launch for a batch of rows:
//   l <- l > 0 ? l / rep : l * rep, then l - freq * count - pres
//                               for every token in the row's history
//   l <- l + bias               for the row's listed tokens, in list order
//   l <- -inf                   where the row's mask has a zero bit
//   token <- the lowest index of the largest value (NaN never wins; -1 where
//            no token is allowed or all that are allowed are NaN)
//
// Bound: one read and one write of the row, so HBM for a batch and latency
// for one row.  A row belongs to one thread-block cluster, its vocabulary
// dealt out to the cluster's CTAs in chunks of 8192.  A CTA asks for its chunk
// first, then finds the tokens that need more than a mask: it counts the
// history's hits of the chunk in shared memory (integer atomics: their order
// is immaterial), adds the biases with one warp in list order, and lists each
// such token once.  The chunk is then streamed with a mask, a store and a
// maximum a logit; the listed tokens are finished by one thread each, so that
// their divisions are not paid by whole warps.  Measured: 96 x 128256 fp32
// logits with a mask, 4000 history entries and 64 biases a row 58 us (1.8 TB/s;
// floor 16 us); one row with 300 entries 5.7 us.  Tables read and keys formed
// for every logit: 105 us.  What bounds it now is the chain of phases in a CTA
// (load, count, stream, finish) with 2 CTAs an SM to overlap: issue slots 44 %
// busy, DRAM 12 %.  3 CTAs by 40 registers spill (76 us), halves of the chunk
// scan the history twice (80 us).
// The greedy token is reduced over the cluster through distributed shared
// memory: no workspace and no second launch.
// Every step of the arithmetic is one rounded fp32 operation, as written.
#include "common.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kLThreads = 512;
constexpr int kPer = 16;                            // logits a thread holds, in runs of 4
constexpr int kChunk = kLThreads * kPer;            // vocabulary entries counted at a time
constexpr int kSeen = 8;                            // history entries a thread holds
constexpr int kMaxCluster = 16;

__device__ __forceinline__ unsigned long long order_key(float v, int i) {
    uint32_t b = __float_as_uint(v + 0.0f);         // -0 and +0 tie
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<unsigned long long>(b) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

// A thread's kPer entries are 4-wide runs: i = base + 4 thread + 4 kLThreads j + 0..3.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, bool vec, float (&v)[4]);
template <>
__device__ __forceinline__ void load4<float>(const float* p, int n, bool vec, float (&v)[4]) {
    if (vec && n >= 4) {
        const float4 a = *reinterpret_cast<const float4*>(p);
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? p[i] : 0.0f;
    }
}
template <>
__device__ __forceinline__ void load4<__nv_bfloat16>(const __nv_bfloat16* p, int n, bool vec, float (&v)[4]) {
    if (vec && n >= 4) {
        const uint2 a = *reinterpret_cast<const uint2*>(p);
        v[0] = __uint_as_float(a.x << 16); v[1] = __uint_as_float(a.x & 0xFFFF0000u);
        v[2] = __uint_as_float(a.y << 16); v[3] = __uint_as_float(a.y & 0xFFFF0000u);
    } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = i < n ? __bfloat162float(p[i]) : 0.0f;
    }
}

// The 16-byte pieces inside [p, p + bytes) into L2.
__device__ __forceinline__ void prefetch_l2(const void* p, size_t bytes) {
    const uintptr_t first = (reinterpret_cast<uintptr_t>(p) + 15) & ~uintptr_t(15);
    const uintptr_t end = (reinterpret_cast<uintptr_t>(p) + bytes) & ~uintptr_t(15);
    for (uintptr_t at = first; at < end; at += 16384)
        asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(at), "r"(static_cast<uint32_t>(min(end - at, uintptr_t(16384))))
                     : "memory");
}

// A float as an unsigned number of the same order; -0 counts as +0.
__device__ __forceinline__ uint32_t order_bits(float v) {
    const uint32_t b = __float_as_uint(v + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <typename T>
__global__ void __launch_bounds__(kLThreads, 2) logits_kernel(const LogitsArgs a, int share, int vec_in, int vec_out, int ahead) {
    extern __shared__ uint4 s_tables[];             // hit counts [kChunk], biases [kChunk], listed tokens [kChunk] (16 bits)
    uint32_t* const s_count = reinterpret_cast<uint32_t*>(s_tables);
    float* const s_bias = reinterpret_cast<float*>(s_count + kChunk);
    uint16_t* const s_list = reinterpret_cast<uint16_t*>(s_bias + kChunk);
    __shared__ uint32_t s_mark[kChunk / 32];        // tokens in the list
    __shared__ unsigned long long s_key[kLThreads / 32];
    __shared__ unsigned long long s_best[kMaxCluster];
    __shared__ uint64_t s_bar;                      // rank 0: the cluster's keys have arrived
    __shared__ int s_listed;
    const int row = blockIdx.y, rank = blockIdx.x, ranks = gridDim.x;
    int tid = threadIdx.x;
    asm volatile("" : "+r"(tid));                  // kept in a register, not read again where it is used
    const int lane = tid & 31;
    if (tid == 0) {
        mbar_init(&s_bar, 1);
        fence_mbar_init();
        mbar_arrive_expect_tx(&s_bar, ranks * 8);
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // waited for before the first remote store
    pdl_launch_dependents();
    pdl_wait();

    const T* in = static_cast<const T*>(a.logits) + row * a.in_stride;
    float* out = a.out + row * a.out_stride;
    const int* hist = a.history + static_cast<long long>(row) * a.history_stride;
    // What the CTA that takes this one's place will read, into L2: rows come in order, `ahead` of them at a time.
    if (tid == 0 && row + ahead < a.rows) {
        const int first = min(a.vocab, rank * share), many = min(a.vocab, first + share) - first;
        prefetch_l2(static_cast<const T*>(a.logits) + (row + ahead) * a.in_stride + first, many * sizeof(T));
        if (a.allow) prefetch_l2(a.allow + static_cast<long long>(row + ahead) * a.allow_stride + first / 32, many / 8);
        if (a.history && rank == 0) prefetch_l2(a.history + static_cast<long long>(row + ahead) * a.history_stride, a.history_stride * 4u);
    }
    // everything that does not depend on the lengths is asked for along with them
    const int hist_len = a.history ? __ldg(a.history_len + row) : 0;
    const int bias_len = a.bias_tokens ? __ldg(a.bias_len + row) : 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (a.history) {
        rep = __ldg(a.penalties + row * 3LL);
        freq = __ldg(a.penalties + row * 3LL + 1);
        pres = __ldg(a.penalties + row * 3LL + 2);
    }
    int seen[kSeen];                                // the first history entries
#pragma unroll
    for (int j = 0; j < kSeen; ++j) {
        const int i = j * kLThreads + tid;
        seen[j] = i < a.history_stride ? __ldg(hist + i) : -1;   // the stride is 0 without a history
    }
    // the last warp has the biases: the first 64 entries ahead of time
    const int* bias_tokens = a.bias_tokens + static_cast<long long>(row) * a.bias_stride;
    const float* bias_values = a.bias_values + static_cast<long long>(row) * a.bias_stride;
    const bool biaser = a.bias_tokens && tid >= kLThreads - 32;
    int bt[2] = {-1, -1};
    float bv[2] = {0.0f, 0.0f};
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (biaser && j * 32 + lane < a.bias_stride) {
            bt[j] = __ldg(bias_tokens + j * 32 + lane);
            bv[j] = __ldg(bias_values + j * 32 + lane);
        }
    const uint32_t* allow = a.allow ? a.allow + static_cast<long long>(row) * a.allow_stride : nullptr;
    const int v0 = min(a.vocab, rank * share), v1 = min(a.vocab, v0 + share);
    unsigned long long best = 0ull;                 // 0: no candidate
    for (int c0 = v0; c0 < v1; c0 += kChunk) {
        const int c1 = min(v1, c0 + kChunk), n = c1 - c0;
        const bool quads = vec_in && vec_out && n % 4 == 0;   // every run of 4 is whole or absent
        float x[kPer / 4][4];
        uint32_t ok[kPer / 4];
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
            const int at = 4 * (j * kLThreads + tid), i = c0 + at;
            ok[j] = 0u;
            if (quads) {
                x[j][0] = x[j][1] = x[j][2] = x[j][3] = 0.0f;
                if (at < n) {
                    load4<T>(in + i, 4, true, x[j]);
                    ok[j] = 15u;
                    if (allow) ok[j] = __ldg(allow + (i >> 5)) >> (i & 31);
                }
            } else {
                load4<T>(in + min(i, c1), c1 - i, vec_in != 0, x[j]);
                if (at < n) ok[j] = allow ? __ldg(allow + (i >> 5)) >> (i & 31) : 15u;
                if (at + 4 > n && at < n) ok[j] &= (1u << (n - at)) - 1u;
            }
        }
        const int n_hist = max(0, min(hist_len, a.history_stride)), n_bias = max(0, min(bias_len, a.bias_stride));
        const bool special = n_hist > 0 || n_bias > 0;
        if (special) {
            const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
            const int words = (n_bias > 0 ? 2 : 1) * kChunk / 4;
            for (int i = tid; i < words; i += kLThreads) s_tables[i] = zero;
            for (int i = tid; i < kChunk / 32; i += kLThreads) s_mark[i] = 0u;
            if (tid == 0) s_listed = 0;
            __syncthreads();
            auto list = [&](int t) {
                const uint32_t bit = 1u << (t & 31);
                if (!(atomicOr(s_mark + (t >> 5), bit) & bit)) s_list[atomicAdd(&s_listed, 1)] = static_cast<uint16_t>(t);
            };
            // A thread's entries in this chunk, few of them: found together, counted one after the other
            uint32_t here = 0u;
#pragma unroll
            for (int j = 0; j < kSeen; ++j)
                if (static_cast<unsigned int>(seen[j] - c0) < static_cast<unsigned int>(n)) here |= 1u << j;
            const int mine_in = (n_hist - tid + kLThreads - 1) / kLThreads;   // this thread's entries
            if (mine_in < kSeen) here &= (1u << max(0, mine_in)) - 1u;
            while (here) {
                const int j = __ffs(here) - 1;
                here &= here - 1u;
                const int t = __ldg(hist + j * kLThreads + tid) - c0;   // read again: registers have no index
                atomicAdd(s_count + t, 1u);
                list(t);
            }
            for (int i = kSeen * kLThreads + tid; i < n_hist; i += kLThreads) {
                const int t = __ldg(hist + i) - c0;
                if (static_cast<unsigned int>(t) < static_cast<unsigned int>(n)) {
                    atomicAdd(s_count + t, 1u);
                    list(t);
                }
            }
            if (n_bias > 0 && biaser) {   // the last warp, 32 entries at a time, in order
                for (int i0 = 0; i0 < n_bias; i0 += 32) {
                    int t = -1;
                    float b = 0.0f;
                    if (i0 + lane < n_bias) {
                        t = i0 == 0 ? bt[0] : i0 == 32 ? bt[1] : __ldg(bias_tokens + i0 + lane);
                        b = i0 == 0 ? bv[0] : i0 == 32 ? bv[1] : __ldg(bias_values + i0 + lane);
                        t = static_cast<unsigned int>(t) < static_cast<unsigned int>(a.vocab) ? t - c0 : -1;
                    }
                    const bool mine = static_cast<unsigned int>(t) < static_cast<unsigned int>(n);
                    const unsigned int same = __match_any_sync(0xffffffffu, mine ? t : -1 - lane);
                    float sum = mine ? s_bias[t] : 0.0f;
                    const bool leads = (same & ((1u << lane) - 1u)) == 0u;
                    if (__any_sync(0xffffffffu, !leads)) {       // equal tokens: the lowest lane adds them in lane order
                        for (int o = 0; o < 32; ++o) {
                            const float v = __shfl_sync(0xffffffffu, b, o);
                            if ((same >> o) & 1u) sum = __fadd_rn(sum, v);
                        }
                    } else {
                        sum = __fadd_rn(sum, b);
                    }
                    if (mine && leads) {
                        s_bias[t] = sum;
                        list(t);
                    }
                    __syncwarp();
                }
            }
            __syncthreads();
        }
        // a listed token a thread: asked for before the chunk is streamed, finished after it
        const int listed = special ? s_listed : 0;
        auto finish = [&](int t, float v, uint32_t word) {
            const uint32_t hits = s_count[t];
            if (hits > 0u) {
                v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, static_cast<float>(hits))), pres);
            }
            if (n_bias > 0) v = __fadd_rn(v, s_bias[t]);
            const int i = c0 + t;
            const bool may = (word >> (i & 31)) & 1u;
            out[i] = may ? v : -INFINITY;
            if (may && v == v) best = max(best, order_key(v, i));
        };
        auto allowed = [&](int i) { return allow ? __ldg(allow + (i >> 5)) : 0xFFFFFFFFu; };   // its whole word
        int mine = -1;
        float mine_v = 0.0f;
        uint32_t mine_ok = 0u;
        if (tid < listed) {
            mine = s_list[tid];
            mine_v = static_cast<float>(in[c0 + mine]);
            mine_ok = allowed(c0 + mine);
        }
        // stream the chunk; a listed token's logit is written as it is and replaced below
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
            const int at = 4 * (j * kLThreads + tid);
            const uint32_t marks = special && at < n ? (s_mark[at >> 5] >> (at & 31)) & 15u : 0u;
            const uint32_t keep = ok[j] | marks;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[j][e] = (keep >> e) & 1u ? x[j][e] : -INFINITY;
            if (quads) {
                if (at < n) *reinterpret_cast<float4*>(out + c0 + at) = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
            } else if (vec_out && at + 4 <= n) {
                *reinterpret_cast<float4*>(out + c0 + at) = make_float4(x[j][0], x[j][1], x[j][2], x[j][3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (at + e < n) out[c0 + at + e] = x[j][e];
            }
            if (marks) {                            // no candidate here
#pragma unroll
                for (int e = 0; e < 4; ++e) x[j][e] = (marks >> e) & 1u ? -INFINITY : x[j][e];
            }
            top = fmaxf(top, fmaxf(fmaxf(x[j][0], x[j][1]), fmaxf(x[j][2], x[j][3])));   // a NaN does not count
        }
        if (special) __syncthreads();               // the logits above are written
        if (mine >= 0) finish(mine, mine_v, mine_ok);
        for (int k = kLThreads + tid; k < listed; k += kLThreads) {
            const int t = s_list[k];
            finish(t, static_cast<float>(in[c0 + t]), allowed(c0 + t));
        }
        // the warp's largest streamed candidate and its lowest index
        if (a.token) {
            const uint32_t high = __reduce_max_sync(0xffffffffu, order_bits(top));
            unsigned int first = 0xFFFFFFFFu;
            if (high == order_bits(-INFINITY)) {    // rarely: nothing above -inf; a logit of -inf that is allowed counts
                for (int j = 0; j < kPer; ++j) {
                    const int at = 4 * ((j >> 2) * kLThreads + tid) + (j & 3);
                    if (at >= n || (special && (s_mark[at >> 5] >> (at & 31)) & 1u)) continue;
                    if (((allowed(c0 + at) >> ((c0 + at) & 31)) & 1u) && out[c0 + at] == -INFINITY &&
                        (a.out != a.logits ? static_cast<float>(in[c0 + at]) == -INFINITY : true))
                        first = min(first, static_cast<unsigned int>(c0 + at));
                }
            } else if (order_bits(top) == high) {
#pragma unroll
                for (int j = kPer / 4 - 1; j >= 0; --j)
#pragma unroll
                    for (int e = 3; e >= 0; --e)
                        if (x[j][e] == top) first = c0 + 4 * (j * kLThreads + tid) + e;
            }
            first = __reduce_min_sync(0xffffffffu, first);
            if (first != 0xFFFFFFFFu) best = max(best, (static_cast<unsigned long long>(high) << 32) | (0xFFFFFFFFu - first));
        }
        if (c0 + kChunk < v1) __syncthreads();      // the tables are reused
    }
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");   // every CTA has started, its barrier is ready
    if (!a.token) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) s_key[tid >> 5] = best;
    __syncthreads();
    if (tid >= 32) return;
    best = lane < kLThreads / 32 ? s_key[lane] : 0ull;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) {                                // to rank 0, which counts the bytes: no fence over the row's stores
        uint32_t to, bar;
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(to) : "r"(smem_u32(s_best + rank)));
        asm volatile("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(bar) : "r"(smem_u32(&s_bar)));
        asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.u64 [%0], %1, [%2];" ::"r"(to), "l"(best), "r"(bar)
                     : "memory");
        if (rank == 0) {
            mbar_wait(&s_bar, 0);
            for (int k = 0; k < ranks; ++k) best = max(best, s_best[k]);
            a.token[row] = best ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best)) : -1;
        }
    }
}

template <typename T>
cudaError_t launch_typed(const LogitsArgs& a, int sms, cudaStream_t stream) {
    auto kernel = logits_kernel<T>;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    const int smem = kChunk * 10;
    if (!configured[dev & 63]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        configured[dev & 63] = true;
    }
    // 16 CTAs a row (one chunk each for vocabularies up to 131072); fewer where a row has no 1024 entries for each
    // (5 x 32003: 6.0 us with 16 CTAs a row, 7.2 with 4)
    int ranks = kMaxCluster;
    while (ranks > 1 && (a.vocab + ranks - 1) / ranks < 1024) ranks >>= 1;
    const int share = ((a.vocab + ranks - 1) / ranks + 31) / 32 * 32;   // whole words of the mask
    auto aligned = [](const void* p, long long stride, size_t bytes) {
        return (reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride) * bytes) % (4 * bytes) == 0;
    };
    const int vec_in = aligned(a.logits, a.in_stride, sizeof(T)), vec_out = aligned(a.out, a.out_stride, 4);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ranks, a.rows);
    cfg.blockDim = dim3(kLThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ranks;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    const int ahead = std::max(1, 2 * sms / ranks);   // rows under way: two CTAs an SM
    return cudaLaunchKernelEx(&cfg, kernel, a, share, vec_in, vec_out, ahead);
}

}  // namespace

cudaError_t launch_logits(const LogitsArgs& a, int sms, cudaStream_t stream) {
    return a.type == ALJ_KV_BF16 ? launch_typed<__nv_bfloat16>(a, sms, stream) : launch_typed<float>(a, sms, stream);
}

}  // namespace alj

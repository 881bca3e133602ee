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
// dealt out to the cluster's CTAs in chunks; a CTA counts the history's hits
// of its chunk in shared memory (integer atomics: their order is immaterial),
// adds the biases with one warp in list order, and streams the chunk once.
// The greedy token is reduced over the cluster through distributed shared
// memory: no workspace and no second launch.
// Every step of the arithmetic is one rounded fp32 operation, as written.
#include "common.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kLThreads = 1024;
constexpr int kPer = 8;                             // logits a thread holds
constexpr int kChunk = kLThreads * kPer;            // vocabulary entries counted at a time
constexpr int kMaxCluster = 16;

__device__ __forceinline__ unsigned long long order_key(float v, int i) {
    uint32_t b = __float_as_uint(v + 0.0f);         // -0 and +0 tie
    b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return (static_cast<unsigned long long>(b) << 32) | (0xFFFFFFFFu - static_cast<uint32_t>(i));
}

template <typename T>
__device__ __forceinline__ float as_float(T v) {
    return static_cast<float>(v);
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

template <typename T>
__global__ void __launch_bounds__(kLThreads) logits_kernel(const LogitsArgs a, int share, int vec_in, int vec_out) {
    extern __shared__ uint32_t s_count[];           // [kChunk], then the biases [kChunk]
    float* const s_bias = reinterpret_cast<float*>(s_count + kChunk);
    __shared__ unsigned long long s_key[32];
    __shared__ unsigned long long s_best[kMaxCluster];
    const int row = blockIdx.y, rank = blockIdx.x, ranks = gridDim.x;
    const int lane = threadIdx.x & 31;
    pdl_launch_dependents();
    pdl_wait();

    const T* in = static_cast<const T*>(a.logits) + row * a.in_stride;
    float* out = a.out + row * a.out_stride;
    const int* hist = a.history + static_cast<long long>(row) * a.history_stride;
    const int n_hist = a.history ? max(0, min(__ldg(a.history_len + row), a.history_stride)) : 0;
    const int n_bias = a.bias_tokens ? max(0, min(__ldg(a.bias_len + row), a.bias_stride)) : 0;
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    if (n_hist > 0) {
        rep = __ldg(a.penalties + row * 3LL);
        freq = __ldg(a.penalties + row * 3LL + 1);
        pres = __ldg(a.penalties + row * 3LL + 2);
    }
    const int v0 = min(a.vocab, rank * share), v1 = min(a.vocab, v0 + share);
    unsigned long long best = 0ull;
    for (int c0 = v0; c0 < v1; c0 += kChunk) {
        const int c1 = min(v1, c0 + kChunk);
        float x[kPer / 4][4];
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
            const int i = c0 + 4 * (j * kLThreads + static_cast<int>(threadIdx.x));
            load4<T>(in + min(i, c1), c1 - i, vec_in != 0, x[j]);
        }
        if (n_hist > 0) {
            for (int i = threadIdx.x; i < kChunk; i += kLThreads) s_count[i] = 0u;
        }
        if (n_bias > 0) {
            for (int i = threadIdx.x; i < kChunk; i += kLThreads) s_bias[i] = 0.0f;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < n_hist; i += kLThreads) {
            const int t = __ldg(hist + i);
            if (t >= c0 && t < c1) atomicAdd(s_count + (t - c0), 1u);
        }
        if (n_bias > 0 && threadIdx.x >= kLThreads - 32) {   // the last warp, 32 entries at a time, in order
            for (int i0 = 0; i0 < n_bias; i0 += 32) {
                const int i = i0 + lane;
                const int t = i < n_bias ? __ldg(a.bias_tokens + static_cast<long long>(row) * a.bias_stride + i) : -1;
                const float b = i < n_bias ? __ldg(a.bias_values + static_cast<long long>(row) * a.bias_stride + i) : 0.0f;
                const bool mine = t >= c0 && t < c1;
                const unsigned int same = __match_any_sync(0xffffffffu, mine ? t : -1 - lane);
                float sum = mine ? s_bias[t - c0] : 0.0f;
                // equal tokens of these 32: the lowest lane adds them all, in lane order
                const bool leads = (same & ((1u << lane) - 1u)) == 0u;
                for (int o = 0; o < 32; ++o) {
                    const float v = __shfl_sync(0xffffffffu, b, o);
                    if (mine && leads && ((same >> o) & 1u)) sum = __fadd_rn(sum, v);
                }
                if (mine && leads) s_bias[t - c0] = sum;
                __syncwarp();
            }
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kPer / 4; ++j) {
            const int i = c0 + 4 * (j * kLThreads + static_cast<int>(threadIdx.x));
            if (i >= c1) continue;
            const uint32_t bits = a.allow ? __ldg(a.allow + static_cast<long long>(row) * a.allow_stride + (i >> 5)) >> (i & 31) : 15u;
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float v = x[j][e];
                const int at = i - c0 + e;
                if (n_hist > 0) {
                    const uint32_t n = s_count[at];
                    if (n > 0u) {
                        v = v > 0.0f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
                        v = __fsub_rn(__fsub_rn(v, __fmul_rn(freq, static_cast<float>(n))), pres);
                    }
                }
                if (n_bias > 0) v = __fadd_rn(v, s_bias[at]);
                const bool ok = (bits >> e) & 1u;
                y[e] = ok ? v : -INFINITY;
                if (ok && i + e < c1 && v == v) best = max(best, order_key(v, i + e));
            }
            if (vec_out && i + 4 <= c1) {
                *reinterpret_cast<float4*>(out + i) = make_float4(y[0], y[1], y[2], y[3]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (i + e < c1) out[i + e] = y[e];
            }
        }
        __syncthreads();                            // the tables are reused
    }
    if (!a.token) return;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
    if (lane == 0) s_key[threadIdx.x >> 5] = best;
    // every CTA of the cluster has started before its shared memory is written
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (threadIdx.x < 32) {
        best = s_key[lane];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
        if (lane == 0) {
            uint32_t to;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(smem_u32(s_best + rank)), "r"(0));
            asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(best) : "memory");
        }
    }
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank == 0 && threadIdx.x == 0) {
        for (int k = 0; k < ranks; ++k) best = max(best, s_best[k]);
        a.token[row] = best ? static_cast<int>(0xFFFFFFFFu - static_cast<uint32_t>(best)) : -1;
    }
}

template <typename T>
cudaError_t launch_typed(const LogitsArgs& a, int sms, cudaStream_t stream) {
    auto kernel = logits_kernel<T>;
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    const int smem = kChunk * 8;
    if (!configured[dev & 63]) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return e;
        configured[dev & 63] = true;
    }
    // CTAs a row: up to 16 while that fills no more than the machine once (2
    // CTAs an SM), else 8, which every GPC can place; no more than a row has
    // 1024-entry pieces.
    int ranks = static_cast<long long>(a.rows) * kMaxCluster <= 2LL * sms ? kMaxCluster : 8;
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
    return cudaLaunchKernelEx(&cfg, kernel, a, share, vec_in, vec_out);
}

}  // namespace

cudaError_t launch_logits(const LogitsArgs& a, int sms, cudaStream_t stream) {
    return a.type == ALJ_KV_BF16 ? launch_typed<__nv_bfloat16>(a, sms, stream) : launch_typed<float>(a, sms, stream);
}

}  // namespace alj

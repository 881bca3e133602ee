// Rows into and out of the 4-bit KV cache (layout: kv4.cuh).
//
// append: K and V rows of new tokens are quantised and stored at their slots
// in one pass, and optionally returned as the values the cache now holds, so
// that the attention of a prompt sees what later decode steps will see.
// read: rows at given slots back as fp32 or bf16.
//
// Both are streams: a thread owns 8 consecutive dims of K and of V of one
// (token, kv head), a quad owns a group of 32, so the extremes need two
// shuffles and nothing is staged.  Each byte is touched once.
#include "kv4.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kRowThreads = 256;

template <typename T>
struct Wide;   // 8 consecutive elements
template <>
struct Wide<float> {
    static __device__ __forceinline__ void load(const float* p, bool vec, float (&v)[8]) {
        if (vec) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
        }
    }
    static __device__ __forceinline__ void store(float* p, bool vec, const float (&v)[8]) {
        if (vec) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = v[i];
        }
    }
};
template <>
struct Wide<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, bool vec, float (&v)[8]) {
        if (vec) {
            const uint4 a = __ldg(reinterpret_cast<const uint4*>(p));
            const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __bfloat162float(p[i]);
        }
    }
    // one rounding to bf16, the type the caller asked the values in
    static __device__ __forceinline__ void store(__nv_bfloat16* p, bool vec, const float (&v)[8]) {
        if (vec) {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&b);
            }
            *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(v[i]);
        }
    }
};

struct Where {          // one thread's place: token, head, 8 dims
    long long token;
    int head, j;        // dims 8 j ..
    int slot;           // -1: skip
};

__device__ __forceinline__ bool place(const Kv4Rows& p, Where& w) {
    const int per_row = p.head_dim / 8;
    const long long i = static_cast<long long>(blockIdx.x) * kRowThreads + threadIdx.x;
    w.j = static_cast<int>(i % per_row);
    const long long row = i / per_row;
    w.head = static_cast<int>(row % p.kv_heads);
    w.token = row / p.kv_heads;
    if (w.token >= p.tokens) return false;   // whole quads only: per_row is a multiple of 8
    w.slot = __ldg(p.slots + w.token);
    if (w.slot >= 0 && w.slot >= static_cast<long long>(p.pages) * p.page_size) {
        record_fault(ALJ_FAULT_BOUNDS);
        w.slot = -1;
    }
    return true;
}

__device__ __forceinline__ uint32_t pack8(const float (&x)[8], float inv) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) w |= kv4_code(x[i], inv) << (4 * i);
    return w;
}
__device__ __forceinline__ void unpack8(uint32_t w, float d, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv4_value((w >> (4 * i)) & 15u, d);
}

// Extremes of a group over its quad and the scale they give.  `finite` from
// x - x: zero for every finite x, NaN for an infinity or a NaN.
__device__ __forceinline__ __half group_scale(const float (&x)[8]) {
    float mn = x[0], mx = x[0], nan = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
        nan += x[i] - x[i];
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        nan += __shfl_xor_sync(0xffffffffu, nan, o);
    }
    return kv4_scale(mn, mx, nan == 0.0f);
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_append_kernel(const Kv4Rows p) {
    pdl_launch_dependents();
    pdl_wait();
    Where w;
    const bool live = place(p, w);
    const int NG = p.head_dim / 32, g = w.j >> 2, c = w.j & 3;
    const bool vec = p.vec != 0;
    float k[8] = {}, v[8] = {};
    const bool write = live && w.slot >= 0;
    if (write) {
        Wide<T>::load(static_cast<const T*>(p.k) + w.token * p.k_stride + w.head * p.head_dim + 8 * w.j, vec, k);
        Wide<T>::load(static_cast<const T*>(p.v) + w.token * p.v_stride + w.head * p.head_dim + 8 * w.j, vec, v);
    }
    // every lane takes part in the shuffles below; a skipped row's zeros are not stored
    const __half dk = group_scale(k), dv = group_scale(v);
    const uint32_t kw = pack8(k, kv4_inverse(dk)), vw = pack8(v, kv4_inverse(dv));
    // V halfwords (2 c, g) and (2 c + 1, g): lanes of groups g and g ^ 1 trade
    // one each, so a lane stores the adjacent pair (r, g & ~1), (r, g | 1)
    const uint32_t other = __shfl_xor_sync(0xffffffffu, vw, 4);
    const uint32_t vpair = g & 1 ? __byte_perm(other, vw, 0x7632) : __byte_perm(vw, other, 0x5410);
    if (write) {
        const int page = w.slot / p.page_size, off = w.slot - page * p.page_size;
        uint8_t* blk = p.cache + (static_cast<long long>(page) * p.kv_heads + w.head) * kv4_block_bytes(p.page_size, p.head_dim);
        const int row = p.head_dim / 2;
        uint8_t* kc = blk + static_cast<long long>(off) * row;
        uint8_t* vc = kc + static_cast<long long>(p.page_size) * row;
        *reinterpret_cast<uint32_t*>(kc + 4 * (c * NG + g)) = kw;
        *reinterpret_cast<uint32_t*>(vc + 2 * ((2 * c + (g & 1)) * NG + (g & ~1))) = vpair;
        __half* sc = reinterpret_cast<__half*>(blk + 2LL * p.page_size * row);
        if (c == 0) sc[static_cast<long long>(off) * NG + g] = dk;
        if (c == 1) sc[static_cast<long long>(p.page_size + off) * NG + g] = dv;
    }
    if (live && p.k_out) {
        const long long at = (w.token * p.kv_heads + w.head) * p.head_dim + 8 * w.j;
        unpack8(kw, write ? __half2float(dk) : 0.0f, k);
        unpack8(vw, write ? __half2float(dv) : 0.0f, v);
        Wide<T>::store(static_cast<T*>(p.k_out) + at, p.vec_out != 0, k);
        Wide<T>::store(static_cast<T*>(p.v_out) + at, p.vec_out != 0, v);
    }
}

template <typename T>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const Kv4Rows p) {
    pdl_launch_dependents();
    pdl_wait();
    Where w;
    if (!place(p, w)) return;
    const int NG = p.head_dim / 32, g = w.j >> 2, c = w.j & 3;
    float k[8] = {}, v[8] = {};
    if (w.slot >= 0) {
        const int page = w.slot / p.page_size, off = w.slot - page * p.page_size;
        const uint8_t* blk = p.cache + (static_cast<long long>(page) * p.kv_heads + w.head) * kv4_block_bytes(p.page_size, p.head_dim);
        const int row = p.head_dim / 2;
        const uint8_t* kc = blk + static_cast<long long>(off) * row;
        const uint8_t* vc = kc + static_cast<long long>(p.page_size) * row;
        const __half* sc = reinterpret_cast<const __half*>(blk + 2LL * p.page_size * row);
        const uint32_t kw = *reinterpret_cast<const uint32_t*>(kc + 4 * (c * NG + g));
        const uint32_t v0 = *reinterpret_cast<const uint16_t*>(vc + 2 * (2 * c * NG + g));
        const uint32_t v1 = *reinterpret_cast<const uint16_t*>(vc + 2 * ((2 * c + 1) * NG + g));
        const float dk = __half2float(sc[static_cast<long long>(off) * NG + g]);
        const float dv = __half2float(sc[static_cast<long long>(p.page_size + off) * NG + g]);
        unpack8(kw, dk, k);
        unpack8(v0 | (v1 << 16), dv, v);
    }
    const long long at = (w.token * p.kv_heads + w.head) * p.head_dim + 8 * w.j;
    if (p.k_out) Wide<T>::store(static_cast<T*>(p.k_out) + at, p.vec_out != 0, k);
    if (p.v_out) Wide<T>::store(static_cast<T*>(p.v_out) + at, p.vec_out != 0, v);
}

cudaError_t launch_rows(void (*kernel)(const Kv4Rows), const Kv4Rows& p, cudaStream_t stream) {
    const long long items = static_cast<long long>(p.tokens) * p.kv_heads * (p.head_dim / 8);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned int>((items + kRowThreads - 1) / kRowThreads));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace

bool kv4_supported(int page_size, int kv_heads, int head_dim) {
    return page_size >= 16 && page_size % 16 == 0 && kv_heads >= 1 &&
           (head_dim == 64 || head_dim == 128 || head_dim == 256);
}

long long kv4_cache_bytes(int pages, int page_size, int kv_heads, int head_dim) {
    return static_cast<long long>(pages) * kv_heads * page_size * (head_dim + head_dim / 8);
}

cudaError_t launch_kv4_append(const Kv4Rows& p, cudaStream_t stream) {
    return launch_rows(p.type == ALJ_KV_BF16 ? kv4_append_kernel<__nv_bfloat16> : kv4_append_kernel<float>, p, stream);
}

cudaError_t launch_kv4_read(const Kv4Rows& p, cudaStream_t stream) {
    return launch_rows(p.type == ALJ_KV_BF16 ? kv4_read_kernel<__nv_bfloat16> : kv4_read_kernel<float>, p, stream);
}

}  // namespace alj

// Rows into and out of the 4-bit KV cache (layout: kv4.cuh).
//
// append: K and V rows of new tokens are quantised and stored at their slots
// in one pass, and optionally returned as the values the cache now holds, so
// that the attention of a prompt sees what later decode steps will see.
// read: rows at given slots back as fp32 or bf16.
//
// Both are streams: a thread owns 8 consecutive dims of K and of V of one
// (token, kv head), a quad owns a group of 32, so the extremes need two
// shuffles and nothing is staged.  Each byte is touched once, and HBM is the
// bound as long as a thread's ~64 bytes cost it few hundred instructions:
// head_dim is a template parameter (rows by shifts), a code is four
// operations (kv4_rounded), and 40 registers let 48 warps an SM wait for
// their loads (50 registers: 48 us).  Measured: 16384 rows of 8 x 128, fp32 in
// and back, 46.4 to 47.1 us over several runs (6.1 to 6.2 TB/s, 94 to 96 % of
// the measured copy rate); 49152 rows read back as fp32 72.5 us (6.3 TB/s, 98 %).
#include "kv4.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kRowThreads = 128;   // 256 threads: 51 us in, 76 us out at the sizes above; 64: 46 and 102

// 8 consecutive elements.  `vec`: 2 for 32-byte aligned rows (one 32-byte
// access a lane, whole sectors: two 16-byte stores each cover half of every
// sector, and read-back of 49152 rows took 88 us with them), 1 for 16-byte
// aligned ones, 0 for the rest.  bf16 rows need 16 bytes a lane.
template <typename T>
struct Wide;
template <>
struct Wide<float> {
    static __device__ __forceinline__ void load(const float* p, int vec, float (&v)[8]) {
        if (vec == 2) {
            asm volatile("ld.global.nc.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
                         : "l"(p));
        } else if (vec == 1) {
            const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __ldg(p + i);
        }
    }
    static __device__ __forceinline__ void store(float* p, int vec, const float (&v)[8]) {
        if (vec == 2) {
            asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
                         "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
                         : "memory");
        } else if (vec == 1) {
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
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, int vec, float (&v)[8]) {
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
    static __device__ __forceinline__ void store(__nv_bfloat16* p, int vec, const float (&v)[8]) {
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

struct Where {          // one thread's place: token, head, 8 dims 8 j ..
    int token, head, j;
    long long block;    // its page's block for the head, in bytes; -1: skip
    int off;            // position in the page
};

template <int D>
__device__ __forceinline__ bool place(const Kv4Rows& p, Where& w) {
    constexpr int kLanes = D / 8;
    const unsigned int row = blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;   // < 2^31: checked on the host
    w.j = threadIdx.x % kLanes;
    w.token = row / static_cast<unsigned int>(p.kv_heads);
    w.head = row - w.token * p.kv_heads;
    w.block = -1;
    if (w.token >= p.tokens) return false;         // whole rows, so whole quads
    const int slot = __ldg(p.slots + w.token);
    if (slot < 0) return true;
    const int page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
    if (page >= p.pages) {
        record_fault(ALJ_FAULT_BOUNDS);
        return true;
    }
    w.off = slot - page * p.page_size;
    w.block = (static_cast<long long>(page) * p.kv_heads + w.head) * kv4_block_bytes(p.page_size, D);
    return true;
}

// Codes of 8 values as a word, and the values they stand for back in x.
__device__ __forceinline__ uint32_t encode8(float (&x)[8], float inv, float d, bool finite) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float r = kv4_rounded(x[i], inv);
        w |= (__float_as_uint(r) & 15u) << (4 * i);
        x[i] = __fadd_rn(__fmul_rn(__fadd_rn(r, -kKv4Round), d), 0.0f);   // as kv4_value
    }
    return finite ? w : 0x88888888u;
}
__device__ __forceinline__ void unpack8(uint32_t w, float d, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = kv4_value((w >> (4 * i)) & 15u, d);
}

// A group's scale from its extremes over the quad.  `finite` from x * 0: zero
// for every finite x, NaN for an infinity or a NaN.
struct Group {
    __half d;
    bool finite;
};
__device__ __forceinline__ Group group_of(const float (&x)[8]) {
    float mn = x[0], mx = x[0], nan = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        mn = fminf(mn, x[i]);
        mx = fmaxf(mx, x[i]);
        nan = fmaf(x[i], 0.0f, nan);
    }
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        nan += __shfl_xor_sync(0xffffffffu, nan, o);
    }
    Group g;
    g.finite = nan == 0.0f;
    g.d = kv4_scale(mn, mx, g.finite);
    return g;
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, 12) kv4_append_kernel(const Kv4Rows p) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int NG = D / 32;
    Where w;
    const bool live = place<D>(p, w);
    const int g = w.j >> 2, c = w.j & 3;
    float k[8] = {}, v[8] = {};
    const bool write = live && w.block >= 0;
    if (write) {
        const int col = w.head * D + 8 * w.j;
        Wide<T>::load(static_cast<const T*>(p.k) + w.token * p.k_stride + col, p.vec, k);
        Wide<T>::load(static_cast<const T*>(p.v) + w.token * p.v_stride + col, p.vec, v);
    }
    // every lane takes part in the shuffles below; a skipped row's zeros are not stored
    const Group gk = group_of(k), gv = group_of(v);
    const uint32_t kw = encode8(k, kv4_inverse(gk.d), __half2float(gk.d), gk.finite);
    const uint32_t vw = encode8(v, kv4_inverse(gv.d), __half2float(gv.d), gv.finite);
    // V halfwords (2 c, g) and (2 c + 1, g): lanes of groups g and g ^ 1 trade
    // one each, so a lane stores the adjacent pair (r, g & ~1), (r, g | 1)
    const uint32_t other = __shfl_xor_sync(0xffffffffu, vw, 4);
    const uint32_t vpair = g & 1 ? __byte_perm(other, vw, 0x7632) : __byte_perm(vw, other, 0x5410);
    if (write) {
        uint8_t* blk = p.cache + w.block;
        uint8_t* kc = blk + w.off * (D / 2LL);
        uint8_t* vc = kc + p.page_size * (D / 2LL);
        *reinterpret_cast<uint32_t*>(kc + 4 * (c * NG + g)) = kw;
        *reinterpret_cast<uint32_t*>(vc + 2 * ((2 * c + (g & 1)) * NG + (g & ~1))) = vpair;
        __half* sc = reinterpret_cast<__half*>(blk + p.page_size * static_cast<long long>(D));
        if (c == 0) sc[w.off * static_cast<long long>(NG) + g] = gk.d;
        if (c == 1) sc[(static_cast<long long>(p.page_size) + w.off) * NG + g] = gv.d;
    }
    if (live && p.k_out) {                         // a skipped row's zeros stand for zeros
        const long long at = (static_cast<long long>(w.token) * p.kv_heads + w.head) * D + 8 * w.j;
        Wide<T>::store(static_cast<T*>(p.k_out) + at, p.vec_out, k);
        Wide<T>::store(static_cast<T*>(p.v_out) + at, p.vec_out, v);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads) kv4_read_kernel(const Kv4Rows p) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int NG = D / 32;
    Where w;
    if (!place<D>(p, w)) return;
    const int g = w.j >> 2, c = w.j & 3;
    float k[8] = {}, v[8] = {};
    if (w.block >= 0) {
        const uint8_t* blk = p.cache + w.block;
        const uint8_t* kc = blk + w.off * (D / 2LL);
        const uint8_t* vc = kc + p.page_size * (D / 2LL);
        const __half* sc = reinterpret_cast<const __half*>(blk + p.page_size * static_cast<long long>(D));
        const uint32_t kw = __ldg(reinterpret_cast<const uint32_t*>(kc + 4 * (c * NG + g)));
        const uint32_t v0 = __ldg(reinterpret_cast<const uint16_t*>(vc + 2 * (2 * c * NG + g)));
        const uint32_t v1 = __ldg(reinterpret_cast<const uint16_t*>(vc + 2 * ((2 * c + 1) * NG + g)));
        const float dk = __half2float(__ldg(sc + w.off * static_cast<long long>(NG) + g));
        const float dv = __half2float(__ldg(sc + (static_cast<long long>(p.page_size) + w.off) * NG + g));
        unpack8(kw, dk, k);
        unpack8(v0 | (v1 << 16), dv, v);
    }
    const long long at = (static_cast<long long>(w.token) * p.kv_heads + w.head) * D + 8 * w.j;
    if (p.k_out) Wide<T>::store(static_cast<T*>(p.k_out) + at, p.vec_out, k);
    if (p.v_out) Wide<T>::store(static_cast<T*>(p.v_out) + at, p.vec_out, v);
}

// Decode step: split-half RoPE of one token's q and k heads (the products and
// sums of rope_store_kernel, decode.cu), then K and V into the cache at
// position *p.slots.  A thread owns dims 8 t .. and D / 2 + 8 t .. of a head,
// which RoPE pairs.
template <int D>
__global__ void __launch_bounds__(kRowThreads) kv4_rope_append_kernel(const Kv4Rows p, float* q, const float2* rope, int q_heads) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kLanes = D / 16, NG = D / 32;
    const int unit = blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes, t = threadIdx.x % kLanes;
    const int pos = __ldg(p.slots);
    const bool in_cache = pos >= 0 && pos < p.page_size, live = unit < q_heads + 2 * p.kv_heads;
    if (!in_cache && live) record_fault(ALJ_FAULT_BOUNDS);
    const bool is_q = unit < q_heads, is_v = unit >= q_heads + p.kv_heads;
    const int head = is_q ? unit : is_v ? unit - q_heads - p.kv_heads : unit - q_heads;
    float x[2][8] = {};
    if (live && in_cache) {
        const float* src = (is_q ? q : static_cast<const float*>(is_v ? p.v : p.k)) + head * D + 8 * t;
        Wide<float>::load(src, 1, x[0]);
        Wide<float>::load(src + D / 2, 1, x[1]);
        if (!is_v) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float2 cs = rope[static_cast<long long>(pos) * (D / 2) + 8 * t + i];
                const float a = x[0][i], b = x[1][i];
                x[0][i] = __fsub_rn(__fmul_rn(a, cs.x), __fmul_rn(b, cs.y));
                x[1][i] = __fadd_rn(__fmul_rn(a, cs.y), __fmul_rn(b, cs.x));
            }
        }
        if (is_q) {
            Wide<float>::store(q + head * D + 8 * t, 1, x[0]);
            Wide<float>::store(q + head * D + D / 2 + 8 * t, 1, x[1]);
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {                  // every lane takes part in the shuffles
        const int j = t + e * kLanes, g = j >> 2, c = j & 3;
        const Group gr = group_of(x[e]);
        const uint32_t w = encode8(x[e], kv4_inverse(gr.d), __half2float(gr.d), gr.finite);
        if (!live || !in_cache || is_q) continue;
        uint8_t* blk = p.cache + head * kv4_block_bytes(p.page_size, D);
        const long long at = (is_v ? static_cast<long long>(p.page_size) : 0) + pos;   // row of the block
        uint8_t* row = blk + at * (D / 2);
        if (is_v) {
            *reinterpret_cast<uint16_t*>(row + 2 * (2 * c * NG + g)) = static_cast<uint16_t>(w);
            *reinterpret_cast<uint16_t*>(row + 2 * ((2 * c + 1) * NG + g)) = static_cast<uint16_t>(w >> 16);
        } else {
            *reinterpret_cast<uint32_t*>(row + 4 * (c * NG + g)) = w;
        }
        if (c == 0)
            reinterpret_cast<__half*>(blk + p.page_size * static_cast<long long>(D))[at * NG + g] = gr.d;
    }
}

cudaError_t launch_rows(void (*kernel)(const Kv4Rows), Kv4Rows p, cudaStream_t stream) {
    p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
    const long long rows = static_cast<long long>(p.tokens) * p.kv_heads;
    const int per_cta = kRowThreads / (p.head_dim / 8);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned int>((rows + per_cta - 1) / per_cta));
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

template <typename T>
cudaError_t launch_append(const Kv4Rows& p, cudaStream_t stream) {
    if (p.head_dim == 64) return launch_rows(kv4_append_kernel<T, 64>, p, stream);
    if (p.head_dim == 128) return launch_rows(kv4_append_kernel<T, 128>, p, stream);
    return launch_rows(kv4_append_kernel<T, 256>, p, stream);
}
template <typename T>
cudaError_t launch_read(const Kv4Rows& p, cudaStream_t stream) {
    if (p.head_dim == 64) return launch_rows(kv4_read_kernel<T, 64>, p, stream);
    if (p.head_dim == 128) return launch_rows(kv4_read_kernel<T, 128>, p, stream);
    return launch_rows(kv4_read_kernel<T, 256>, p, stream);
}

cudaError_t launch_kv4_append(const Kv4Rows& p, cudaStream_t stream) {
    return p.type == ALJ_KV_BF16 ? launch_append<__nv_bfloat16>(p, stream) : launch_append<float>(p, stream);
}

cudaError_t launch_kv4_read(const Kv4Rows& p, cudaStream_t stream) {
    return p.type == ALJ_KV_BF16 ? launch_read<__nv_bfloat16>(p, stream) : launch_read<float>(p, stream);
}

cudaError_t launch_kv4_rope_append(const Kv4Rows& p, float* q, const float2* rope, int q_heads, cudaStream_t stream) {
    const int units = q_heads + 2 * p.kv_heads, per_cta = kRowThreads / (p.head_dim / 16);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((units + per_cta - 1) / per_cta);
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto kernel = p.head_dim == 64 ? kv4_rope_append_kernel<64> : p.head_dim == 128 ? kv4_rope_append_kernel<128> : kv4_rope_append_kernel<256>;
    return cudaLaunchKernelEx(&cfg, kernel, p, q, rope, q_heads);
}

}  // namespace alj

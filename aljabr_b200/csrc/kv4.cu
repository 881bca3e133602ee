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

// 8 elements as they are in memory, to be on their way in few registers.
template <typename T>
struct Raw {
    uint32_t w[2 * sizeof(T)];
    __device__ __forceinline__ void load(const T* p, int vec) {
        constexpr int kWords = 2 * sizeof(T);
        if (vec) {
#pragma unroll
            for (int i = 0; i < kWords / 4; ++i) {
                const uint4 a = __ldg(reinterpret_cast<const uint4*>(p) + i);
                w[4 * i] = a.x, w[4 * i + 1] = a.y, w[4 * i + 2] = a.z, w[4 * i + 3] = a.w;
            }
        } else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kWords; ++i) w[i] = __float_as_uint(__ldg(p + i));
        } else {
#pragma unroll
            for (int i = 0; i < kWords; ++i)
                w[i] = __bfloat16_as_ushort(p[2 * i]) | static_cast<uint32_t>(__bfloat16_as_ushort(p[2 * i + 1])) << 16;
        }
    }
    __device__ __forceinline__ void to(float (&v)[8]) const {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
            else v[i] = __uint_as_float(i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        }
    }
};

struct Where {          // one thread's place: token, head, 8 dims 8 j ..
    int token, head, j;
    long long block;    // its page's block for the head, in bytes; -1: skip
    int off;            // position in the page
};

// The block of w.head in the slot's page, -1 for none.
template <int D>
__device__ __forceinline__ void find_block(const Kv4Rows& p, int slot, Where& w) {
    w.block = -1;
    if (slot < 0) return;
    const int page = p.page_shift >= 0 ? slot >> p.page_shift : slot / p.page_size;
    if (page >= p.pages) {
        record_fault(ALJ_FAULT_BOUNDS);
        return;
    }
    w.off = slot - page * p.page_size;
    w.block = (static_cast<long long>(page) * p.kv_heads + w.head) * kv4_block_bytes(p.page_size, D);
}

template <int D>
__device__ __forceinline__ bool place(const Kv4Rows& p, Where& w) {
    constexpr int kLanes = D / 8;
    const unsigned int row = blockIdx.x * (kRowThreads / kLanes) + threadIdx.x / kLanes;   // < 2^31: checked on the host
    w.j = threadIdx.x % kLanes;
    w.token = row / static_cast<unsigned int>(p.kv_heads);
    w.head = row - w.token * p.kv_heads;
    if (w.token >= p.tokens) {                     // whole rows, so whole quads
        w.block = -1;
        return false;
    }
    find_block<D>(p, __ldg(p.slots + w.token), w);
    return true;
}

// (a, b) turned by the angle of cosine c and sine s.
__device__ __forceinline__ void turn_pair(float& a, float& b, float c, float s) {
    const float x = __fsub_rn(__fmul_rn(a, c), __fmul_rn(b, s));
    b = __fadd_rn(__fmul_rn(a, s), __fmul_rn(b, c));
    a = x;
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

// Quantises a thread's 8 dims of K and of V and stores them at w where `write`; k and v become the values that the
// codes stand for.  Every lane of the warp takes part.
template <int D>
__device__ __forceinline__ void put8(const Kv4Rows& p, const Where& w, bool write, float (&k)[8], float (&v)[8]) {
    constexpr int NG = D / 32;
    const int g = w.j >> 2, c = w.j & 3;
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
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, 12) kv4_append_kernel(const Kv4Rows p) {
    pdl_launch_dependents();
    pdl_wait();
    Where w;
    const bool live = place<D>(p, w);
    float k[8] = {}, v[8] = {};
    const bool write = live && w.block >= 0;
    if (write) {
        const int col = w.head * D + 8 * w.j;
        Wide<T>::load(static_cast<const T*>(p.k) + w.token * p.k_stride + col, p.vec, k);
        Wide<T>::load(static_cast<const T*>(p.v) + w.token * p.v_stride + col, p.vec, v);
    }
    put8<D>(p, w, write, k, v);                    // a skipped row's zeros are not stored
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

// Rows of new tokens with the position rotation on the way: q is rotated into q_out, k before it is quantised; the
// products and sums are rounded one by one, as in the decode step.  In the CTAs that have q rows a thread owns two runs
// of 8 dims that are each other's pairs (split halves) or adjacent (interleaved, and what does not turn), so nothing is
// exchanged, and keeps their 8 cosines and sines for p.span heads of its token.  The others have K and V, laid out as in
// kv4_append_kernel for the groups' shuffles.  The former wait for memory, the latter (600 instructions a warp for
// 2 KB) for issue slots, so they are spread among each other.
template <typename T, int D>
__device__ __forceinline__ void rotate_q(const Kv4Rotate& p, unsigned int block) {
    constexpr int kLanes = D / 16, kPer = kRowThreads / kLanes;
    const unsigned int row = block * kPer + threadIdx.x / kLanes;
    const int t = threadIdx.x % kLanes;
    const int token = row / static_cast<unsigned int>(p.splits);
    if (token >= p.rows.tokens) return;
    const int head0 = (row - token * p.splits) * p.span, heads = min(p.span, p.q_heads - head0);
    int pos = __ldg(p.positions + token);          // on its way while the first head is; then always the next one
    const int half8 = p.half >> 3;                 // runs of 8 in half of the turning dims
    // its runs: with split halves t and t + half8, behind the turning dims two neighbours
    const int run0 = p.interleaved || t >= half8 ? 2 * t : t, run1 = p.interleaved || t >= half8 ? 2 * t + 1 : t + half8;
    const T* q = static_cast<const T*>(p.q) + token * p.q_stride + head0 * D;
    T* out = static_cast<T*>(p.q_out) + token * p.q_out_stride + head0 * D;
    Raw<T> next0, next1;
    next0.load(q + 8 * run0, p.vec_q);
    next1.load(q + 8 * run1, p.vec_q);
    if (pos >= p.rope_positions) {
        record_fault(ALJ_FAULT_BOUNDS);
        pos = -1;
    }
    const bool turns = t < half8 && pos >= 0;
    float cs[8], sn[8];
    if (turns) {
        const float4* at = reinterpret_cast<const float4*>(p.rope + static_cast<long long>(pos) * p.half + 8 * t);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float4 f = __ldg(at + i);
            cs[2 * i] = f.x, sn[2 * i] = f.y, cs[2 * i + 1] = f.z, sn[2 * i + 1] = f.w;
        }
    }
#pragma unroll 1
    for (int h = 0; h < heads; ++h, q += D, out += D) {
        float a[8], b[8];
        next0.to(a);
        next1.to(b);
        if (h + 1 < heads) {
            next0.load(q + D + 8 * run0, p.vec_q);
            next1.load(q + D + 8 * run1, p.vec_q);
        }
        if (pos < 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.0f;
        }
        if (turns && p.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                turn_pair(a[2 * i], a[2 * i + 1], cs[i], sn[i]);
                turn_pair(b[2 * i], b[2 * i + 1], cs[4 + i], sn[4 + i]);
            }
        } else if (turns) {
#pragma unroll
            for (int i = 0; i < 8; ++i) turn_pair(a[i], b[i], cs[i], sn[i]);
        }
        Wide<T>::store(out + 8 * run0, p.vec_q_out, a);
        Wide<T>::store(out + 8 * run1, p.vec_q_out, b);
    }
}

template <typename T, int D>
__global__ void __launch_bounds__(kRowThreads, 8) kv4_rotate_append_kernel(const Kv4Rotate p) {
    pdl_launch_dependents();
    pdl_wait();
    // of every q_blocks + kv_blocks CTAs, kv_blocks evenly among the others
    const unsigned int kv_block = __umulhi(blockIdx.x, p.kv_step);
    if (__umulhi(blockIdx.x + 1, p.kv_step) == kv_block) {
        rotate_q<T, D>(p, blockIdx.x - kv_block);
        return;
    }
    // the rows are on their way while slots and positions are, whether they are used or not
    constexpr int kLanes = D / 8;
    Where w;
    const unsigned int row = kv_block * (kRowThreads / kLanes) + threadIdx.x / kLanes;
    w.j = threadIdx.x % kLanes;
    w.token = row / static_cast<unsigned int>(p.rows.kv_heads);
    w.head = row - w.token * p.rows.kv_heads;
    w.block = -1;
    const bool live = w.token < p.rows.tokens;
    const int half8 = p.half >> 3;
    const bool second = !p.interleaved && w.j >= half8, in = w.j < 2 * half8;
    float k[8] = {}, v[8] = {}, mate[8] = {};
    int pos = -1;
    if (live) {
        const int slot = __ldg(p.rows.slots + w.token);
        pos = __ldg(p.positions + w.token);
        const T* const k_row = static_cast<const T*>(p.rows.k) + w.token * p.rows.k_stride + w.head * D;
        Wide<T>::load(k_row + 8 * w.j, p.rows.vec, k);
        // split halves: the dims that pair with these, which their own thread loads too
        if (in && !p.interleaved) Wide<T>::load(k_row + 8 * (second ? w.j - half8 : w.j + half8), p.rows.vec, mate);
        Wide<T>::load(static_cast<const T*>(p.rows.v) + w.token * p.rows.v_stride + w.head * D + 8 * w.j, p.rows.vec, v);
        find_block<D>(p.rows, slot, w);
    }
    if (pos >= p.rope_positions) {
        if (w.head == 0) record_fault(ALJ_FAULT_BOUNDS);
        pos = -1;
    }
    const bool write = w.block >= 0 && pos >= 0, turns = write && in;
    float cs[8] = {}, sn[8] = {};
    if (!write) {
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = v[i] = 0.0f;
    }
    if (turns) {
        const int pair = p.interleaved ? 4 * w.j : 8 * (second ? w.j - half8 : w.j);
        const float4* at = reinterpret_cast<const float4*>(p.rope + static_cast<long long>(pos) * p.half + pair);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (i >= 2 && p.interleaved) break;
            const float4 f = __ldg(at + i);
            cs[2 * i] = f.x, sn[2 * i] = f.y, cs[2 * i + 1] = f.z, sn[2 * i + 1] = f.w;
        }
    }
    if (p.interleaved) {
        if (turns) {
#pragma unroll
            for (int i = 0; i < 4; ++i) turn_pair(k[2 * i], k[2 * i + 1], cs[i], sn[i]);
        }
    } else if (turns) {
#pragma unroll
        for (int i = 0; i < 8; ++i) k[i] = __fadd_rn(__fmul_rn(k[i], cs[i]), __fmul_rn(mate[i], second ? sn[i] : -sn[i]));
    }
    put8<D>(p.rows, w, write, k, v);               // a skipped row's zeros are not stored
    if (live && p.rows.k_out) {
        const long long at = (static_cast<long long>(w.token) * p.rows.kv_heads + w.head) * D + 8 * w.j;
        Wide<T>::store(static_cast<T*>(p.rows.k_out) + at, p.rows.vec_out, k);
        Wide<T>::store(static_cast<T*>(p.rows.v_out) + at, p.rows.vec_out, v);
    }
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

cudaError_t launch_kv4_rotate_append(const Kv4Rotate& a, int sms, cudaStream_t stream) {
    Kv4Rotate p = a;
    p.rows.page_shift = (p.rows.page_size & (p.rows.page_size - 1)) == 0 ? __builtin_ctz(p.rows.page_size) : -1;
    // q: four heads a thread where the rows still fill the GPU, else one
    const long long tokens = p.rows.tokens;
    const int per_q = kRowThreads / (p.rows.head_dim / 16), per_kv = kRowThreads / (p.rows.head_dim / 8);
    p.span = tokens * ((p.q_heads + 3) / 4) / per_q >= 8LL * sms ? 4 : 1;
    p.splits = (p.q_heads + p.span - 1) / p.span;
    const long long q_blocks = (tokens * p.splits + per_q - 1) / per_q, kv_blocks = (tokens * p.rows.kv_heads + per_kv - 1) / per_kv;
    const long long blocks = q_blocks + kv_blocks;   // < 2^31: checked on the host
    p.kv_step = static_cast<unsigned int>(((kv_blocks << 32) + blocks - 1) / blocks);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned int>(blocks));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    const bool bf16 = p.rows.type == ALJ_KV_BF16;
    auto pick = [&](auto wide, auto narrow) { return bf16 ? narrow : wide; };
    auto kernel = p.rows.head_dim == 64    ? pick(kv4_rotate_append_kernel<float, 64>, kv4_rotate_append_kernel<__nv_bfloat16, 64>)
                  : p.rows.head_dim == 128 ? pick(kv4_rotate_append_kernel<float, 128>, kv4_rotate_append_kernel<__nv_bfloat16, 128>)
                                           : pick(kv4_rotate_append_kernel<float, 256>, kv4_rotate_append_kernel<__nv_bfloat16, 256>);
    return cudaLaunchKernelEx(&cfg, kernel, p);
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

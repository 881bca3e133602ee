// Attention of a few new tokens per sequence over the 4-bit KV cache
// (layout: kv4.cuh), for batches of sequences of any lengths.
//
//   S[i, p] = scale * sum_g dK[p, g] * sum_{j in g} (cK[p, j] - 8) q[i, j]
//   (soft cap: S <- cap * tanh(S / cap)),  P = softmax over the positions
//   that row i sees,  O[i, j] = sum_p P[i, p] * dV[p, g(j)] * (cV[p, j] - 8)
//
// A row i is one (query token, query head) pair of the T x G pairs that share
// a kv head.  The cache is read once per kv head and 8 or 16 rows; a position
// costs 1.125 D bytes, so the bound is HBM until the 148 SMs cannot decode
// ~23 bytes of codes a clock each.  What is spent per code decides, hence:
//
//   * Both products run on mma.sync m16n8k16 (fp16 operands, fp32 sums).  The
//     K codes are the B operand of S^T = q K^T without being converted: a
//     nibble masked out of its word is the fp16 subnormal c * 2^-24 (or
//     16 c * 2^-24), exact, so 8 codes cost 4 LOP3 and a shift.  The slots
//     with the factor 16 have q / 16 on the other side.  The offset -8 is
//     sum_g dK[p, g] * (-8 sum_{j in g} q_j): one more MMA with the fp16
//     scales as they are stored for its B operand.
//   * q is scaled by a power of two into fp16's range.  bf16 queries are
//     exact in one part; fp32 queries take two parts in the two row halves of
//     the A operand, each a multiple of a fixed step of the row (2^-11 and
//     2^-22 of its largest value), so that the tensor cores' sums of a group
//     are exact integers and their truncation does not enter.
//   * The accumulator layout of S^T (row = query, columns = positions) is the
//     B operand layout of O^T = V^T P^T, so probabilities never leave their
//     lane.  V's group scales are folded into P before it is rounded:
//     P' = P * dV * 2^(20 - e), e the largest exponent field of the V scales
//     seen so far by the warp, so P' uses the upper part of fp16's range
//     whatever the size of V.  fp32 outputs take P' in two fp16 parts.
//   * V codes become the exact fp16 integers c - 8 (the sums then stay as
//     small as the result; adding -8 sum P' afterwards would lose 2-3 digits
//     over long contexts): (bits | 1024) - 1032, or (bits | 1024) / 16 - 72.
//     Two positions are interleaved by one PRMT, no transposing load needed.
//   * Rounding points: q parts, P' parts, the output type.  Scores, softmax
//     statistics and sums are fp32.  For fp32 outputs every tile's product is
//     added to the running sum by the CUDA cores, because the tensor cores'
//     own accumulation truncates and a long chain of it drifts.
//
// Work split: the positions of each sequence are cut into chunks of 128
// (a 16-position tile for each of the 8 warps); all chunks of all (sequence,
// kv head, row tile) items form one line that is dealt out evenly to the
// resident CTAs, whatever the lengths are (starting and ending an item counts
// as kItemCost chunks).  A CTA keeps an item's running softmax in registers;
// where an item ends inside a CTA the warps merge in shared memory, and an
// item cut over several CTAs is joined by the CTA that arrives last, in CTA
// order, so results do not depend on timing.  Each warp feeds itself through
// a private ring of tiles, four bulk copies a tile; warps meet only at item
// ends.
#include "kv4.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTilePos = 16;
constexpr int kChunkTiles = kWarps;
constexpr int kStages = 3;
constexpr int kItemCost = 2;     // chunks that an item's start and end are worth
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.0f;    // a row's maximum is raised only when a score exceeds it by 2^8

// d = a b + c; the form without c starts from zero.
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_f16_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                             uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ float half_lo(uint32_t v) { return __low2float(bits_h2(v)); }
__device__ __forceinline__ float half_hi(uint32_t v) { return __high2float(bits_h2(v)); }
__device__ __forceinline__ float pow2i(int e) {   // 2^e for normal results
    return __int_as_float((e + 127) << 23);
}
__device__ __forceinline__ unsigned int arrive_acq_rel(unsigned int* p) {
    unsigned int old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
    return old;
}

// Four outputs sum * inv at element `to`, one rounding where the type is bf16.
__device__ __forceinline__ void store4(void* out, bool bf16, long long to, float4 sum, float inv) {
    sum.x *= inv; sum.y *= inv; sum.z *= inv; sum.w *= inv;
    if (bf16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(sum.x, sum.y), b = __floats2bfloat162_rn(sum.z, sum.w);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + to) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + to) = sum;
    }
}

// NW consecutive 32-bit words from shared memory (4 NW-byte aligned).
template <int NW>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[NW]) {
    if constexpr (NW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 4; ++i) {
            const uint4 v = reinterpret_cast<const uint4*>(p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (NW == 2) {
        const uint2 v = *reinterpret_cast<const uint2*>(p);
        w[0] = v.x; w[1] = v.y;
    } else {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    }
}

// Shapes of one instantiation: NG groups of 32 dims, RT tiles of 8 rows,
// PARTS fp16 parts of q and P (2 for fp32 in and out, 1 for bf16).
template <int NG, int RT, int PARTS>
struct Cfg {
    static constexpr int D = 32 * NG;
    static constexpr int ROWS = 8 * RT;
    static constexpr int NA = PARTS == 2 ? RT : 1;          // A operands: [hi ; lo] per row tile, or both row tiles
    static constexpr int CODES = 256 * NG;                  // code bytes of a tile (K or V)
    static constexpr int SCALES = 32 * NG;
    static constexpr int STAGE = 2 * (CODES + SCALES);
    static constexpr int RING = kStages * kWarps * STAGE;
    static constexpr int SG = RT == 1 ? (NG < 4 ? NG : 4) : 2;   // groups merged at a time
    static constexpr int MROW = SG * 32 + 4;                // floats a row in the merge buffer; + 4: no bank conflicts
    static constexpr int MERGE = kWarps * ROWS * MROW * 4;
    static constexpr int QFRAG = NA * NG * 2 * 32 * 16;
    static constexpr int QSUM = NA * 32 * 16;               // offset fragments
    static constexpr int BARS = kStages * kWarps * 8;
    static constexpr int MISC = (kWarps * ROWS * 2 + kWarps + ROWS + 8) * 4;
    static constexpr int SMEM = RING + MERGE + QFRAG + QSUM + BARS + MISC;   // + the per-sequence tables
};

// One place on the line of chunks: sequence b, item h = kv head * row tiles +
// row tile, chunk ch of that item.
struct Cursor {
    int b, h, ch, chunks, len, first;   // first: the item's first tile
};

struct Tables {      // per sequence, in shared memory
    const int* pre;  // [batch + 1] chunks and item costs before it (of one item)
    const int* len;  // [batch]
};

__device__ __forceinline__ int first_tile(const Kv4Attn& p, int len) {
    return p.window > 0 ? max(0, len - p.q_len - p.window + 1) / kTilePos : 0;
}
__device__ __forceinline__ int chunks_of(const Kv4Attn& p, int len) {
    const int tiles = (len + kTilePos - 1) / kTilePos - first_tile(p, len);
    return max(1, (tiles + kChunkTiles - 1) / kChunkTiles);   // an empty sequence still has its zeros to write
}
__device__ __forceinline__ void load_seq(Cursor& c, const Kv4Attn& p, const Tables& t) {
    c.len = t.len[c.b];
    c.chunks = t.pre[c.b + 1] - t.pre[c.b] - kItemCost;
    c.first = first_tile(p, c.len);
}
__device__ __forceinline__ void step(Cursor& c, const Kv4Attn& p, const Tables& t, int items) {
    if (++c.ch < c.chunks) return;
    c.ch = 0;
    if (++c.h < items) return;
    c.h = 0;
    if (++c.b < p.batch) load_seq(c, p, t);
}

// Issue the copies of this warp's tile at cursor c into `stage`: lane 0 the K
// codes, lane 1 the V codes, lanes 2 and 3 their scales.  Returns false, with
// nothing issued, where there is no tile (past the end, or a page id outside
// the cache).
template <int NG>
__device__ __forceinline__ bool load_tile(const Kv4Attn& p, const Cursor& c, uint8_t* stage, uint64_t* bar, int warp,
                                          int lane) {
    using F = Cfg<NG, 1, 1>;
    const int pos = (c.first + c.ch * kChunkTiles + warp) * kTilePos;
    if (pos >= c.len) return false;
    const int pi = p.page_shift >= 0 ? pos >> p.page_shift : pos / p.page_size;
    const int page = p.table ? __ldg(p.table + static_cast<long long>(c.b) * p.table_stride + pi) : c.b;
    if (page < 0 || page >= p.pages) {
        record_fault(ALJ_FAULT_BOUNDS);
        return false;
    }
    if (lane == 0) mbar_arrive_expect_tx(bar, F::STAGE);
    __syncwarp();
    if (lane < 4) {
        const uint32_t off = pos - pi * p.page_size, ps = p.page_size;
        const int kvh = p.row_tiles == 1 ? c.h : c.h / p.row_tiles;
        // sections of a block start at 0, 16 NG ps, 32 NG ps and 34 NG ps bytes
        const uint32_t row = lane < 2 ? 16 * NG : 2 * NG;
        const uint32_t section = (lane < 2 ? 16 * NG * lane : 28 * NG + 2 * NG * lane);
        const uint8_t* src = p.cache + (static_cast<long long>(page) * p.kv_heads + kvh) * kv4_block_bytes(p.page_size, F::D) +
                             static_cast<unsigned long long>(section) * ps + static_cast<unsigned long long>(row) * off;
        const uint32_t dst = lane < 2 ? F::CODES * lane : 2 * F::CODES + F::SCALES * (lane - 2);
        bulk_g2s(stage + dst, src, row * kTilePos, bar);
    }
    return true;
}

template <int NG, int RT, int PARTS>
__global__ void __launch_bounds__(kThreads, NG <= 4 && RT == 1 ? 2 : 1) kv4_attn_kernel(const Kv4Attn p) {
    using F = Cfg<NG, RT, PARTS>;
    constexpr int D = F::D, ROWS = F::ROWS, NA = F::NA;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const ring = smem;
    float* const s_merge = reinterpret_cast<float*>(smem + F::RING);
    uint4* const s_q = reinterpret_cast<uint4*>(smem + F::RING + F::MERGE);
    uint4* const s_off = s_q + F::QFRAG / 16;                 // offset fragments
    uint64_t* const s_bar = reinterpret_cast<uint64_t*>(s_off + F::QSUM / 16);
    float* const s_ml = reinterpret_cast<float*>(s_bar + kStages * kWarps);   // [warp][row][max, sum]
    int* const s_e = reinterpret_cast<int*>(s_ml + kWarps * ROWS * 2);        // [warp]
    float* const s_fac = reinterpret_cast<float*>(s_e + kWarps);              // [row] score factor
    int* const s_misc = reinterpret_cast<int*>(s_fac + ROWS);
    int* const s_pre = s_misc + 8;
    int* const s_len = s_pre + p.batch + 1;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r = lane >> 2, c4 = lane & 3;
    const int R = p.q_len * p.group;               // rows that share a kv head
    const int items = p.kv_heads * p.row_tiles;    // items of a sequence
    pdl_launch_dependents();
    uint64_t* const bars = s_bar + warp * kStages;
    if (lane == 0) {
        for (int i = 0; i < kStages; ++i) mbar_init(bars + i, 1);
        fence_mbar_init();
    }
    for (int i = threadIdx.x; i < (F::QFRAG + F::QSUM) / 16; i += kThreads) s_q[i] = make_uint4(0u, 0u, 0u, 0u);
    pdl_wait();

    // lengths (clamped to what the table can address) and the prefix of chunks
    const int cap = p.table ? static_cast<int>(min(static_cast<long long>(p.table_stride) * p.page_size, 0x7fffff00LL))
                            : p.page_size;
    if (threadIdx.x == 0) s_misc[0] = 0;
    __syncthreads();
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int n = 0;
        if (b < p.batch) {
            int len = __ldg(p.lens + b) + p.len_add;
            if (len < 0 || len > cap) {
                record_fault(ALJ_FAULT_BOUNDS);
                len = len < 0 ? 0 : cap;
            }
            s_len[b] = len;
            n = chunks_of(p, len) + kItemCost;
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (lane == 31) s_e[warp] = incl;
        __syncthreads();
        int base = s_misc[0];
        for (int w = 0; w < warp; ++w) base += s_e[w];
        if (b < p.batch) s_pre[b] = base + incl - n;
        __syncthreads();
        if (threadIdx.x == kThreads - 1) s_misc[0] = base + incl;
        __syncthreads();
    }
    if (threadIdx.x == 0) s_pre[p.batch] = s_misc[0];
    __syncthreads();
    const Tables tab = {s_pre, s_len};
    const long long total = static_cast<long long>(s_pre[p.batch]) * items;
    const long long ctas = min(static_cast<long long>(gridDim.x), total);
    if (static_cast<long long>(blockIdx.x) >= ctas) return;
    // The line with its item costs is dealt out evenly; chunk numbers (u) count
    // real chunks only.
    auto chunks_before = [&](int b) { return static_cast<long long>(s_pre[b] - kItemCost * b) * items; };
    auto real = [&](long long x) {                 // real chunks before place x of the line
        if (x >= total) return chunks_before(p.batch);
        int lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (static_cast<long long>(s_pre[mid]) * items <= x) lo = mid;
            else hi = mid - 1;
        }
        const int width = s_pre[lo + 1] - s_pre[lo];
        const long long rest = x - static_cast<long long>(s_pre[lo]) * items;
        const long long h = rest / width;
        return chunks_before(lo) + h * (width - kItemCost) + max(0, static_cast<int>(rest - h * width) - kItemCost);
    };
    const long long u0 = real(total * blockIdx.x / ctas), u1 = real(total * (blockIdx.x + 1) / ctas);
    if (u0 >= u1) return;

    Cursor at;
    {
        int lo = 0, hi = p.batch - 1;              // the sequence of chunk u0
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (chunks_before(mid) <= u0) lo = mid;
            else hi = mid - 1;
        }
        at.b = lo;
        load_seq(at, p, tab);
        const long long rest = u0 - chunks_before(lo);
        at.h = static_cast<int>(rest / at.chunks);
        at.ch = static_cast<int>(rest - static_cast<long long>(at.h) * at.chunks);
    }
    Cursor ahead = at;
    uint8_t* const my_ring = ring + warp * (kStages * F::STAGE);
    long long next = u0;                           // first chunk not yet asked for
    uint32_t have = 0, phase = 0;                  // per ring slot: a tile was asked for; the barrier's next parity
    bool dead = false;                             // a copy never arrived: stop waiting, the fault is recorded
    auto ask = [&](int slot) {
        if (next >= u1) return;
        const bool some = load_tile<NG>(p, ahead, my_ring + slot * F::STAGE, bars + slot, warp, lane);
        have = some ? have | (1u << slot) : have & ~(1u << slot);
        step(ahead, p, tab, items);
        ++next;
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) ask(i);
    int fill = kStages - 1, use = 0;               // ring slots

    long long u = u0;
    while (u < u1) {
        // ---------------------------------------------------------- item start
        const int kvh = at.h / p.row_tiles, row0 = (at.h - kvh * p.row_tiles) * ROWS;
        const int item_b = at.b, len = at.len;
        const long long item0 = chunks_before(item_b) + static_cast<long long>(at.h) * at.chunks;
        const long long item1 = item0 + at.chunks;
        // the item's place on the line, for the CTAs that share it
        const long long line0 = static_cast<long long>(s_pre[item_b]) * items +
                                static_cast<long long>(at.h) * (at.chunks + kItemCost) + kItemCost;
        const long long line1 = line0 + at.chunks;
        const long long seg0 = u, seg1 = min(u1, item1);
        const int rows = min(ROWS, R - row0);
        __syncthreads();                           // the previous item's tables are read

        // q rows -> fp16 parts in A-fragment order, their group sums, their score factors
        for (int row = warp; row < ROWS; row += kWarps) {
            float x[NG];
            const int i = row0 + row;
            const bool live = row < rows;
            const int t = live ? i / p.group : 0, hd = live ? i - t * p.group : 0;
            const long long src = (static_cast<long long>(item_b) * p.q_len + t) * p.q_stride +
                                  static_cast<long long>(kvh * p.group + hd) * D;
            float big = 0.0f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                x[g] = 0.0f;
                if (live)
                    x[g] = PARTS == 2 ? static_cast<const float*>(p.q)[src + 32 * g + lane]
                                      : __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[src + 32 * g + lane]);
                big = fmaxf(big, fabsf(x[g]));
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            // big * 2^f in [2^14, 2^15); f kept where both 2^f and the factor below are normal
            const int f = big > 0.0f ? max(-100, min(126, 14 - (static_cast<int>((__float_as_uint(big) >> 23) & 255) - 127))) : 0;
            const float up = pow2i(f);
            // lane j of a group: slot (c = j / 8, i = j % 8).  MMA step (i & 3) >> 1; k index within it
            const int i8 = lane & 7, cc = lane >> 3, st = (i8 & 3) >> 1;
            const bool odd = i8 & 1;               // second k half, codes carry a factor 16
            const int half_at = i8 >> 2;           // low or high half of the pair
            const __half sixteenth = __ushort_as_half(0x2C00);
            float sum[NG];
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float y = x[g] * up;         // |y| < 2^15
                // PARTS 2: multiples of 16 and of 2^-7 -- 11 bits each, so that a group's sum of products is exact
                const __half h = __float2half_rn(PARTS == 2 ? rintf(y * 0.0625f) * 16.0f : y);
                const float hf = __half2float(h);
                const __half l = __float2half_rn(rintf((y - hf) * 128.0f) * 16.0f);
                sum[g] = PARTS == 2 ? fmaf(__half2float(l), 1.0f / 2048.0f, hf) : hf;
                const __half hs = odd ? __hmul(h, sixteenth) : h, ls = odd ? __hmul(l, sixteenth) : l;
                // register of the fragment: a0 / a2 rows 0-7, a1 / a3 rows 8-15; a2, a3 the second k half
                auto put = [&](int na, int reg, __half v) {
                    reinterpret_cast<__half*>(s_q + ((na * NG + g) * 2 + st) * 32 + (row & 7) * 4 + cc)[2 * reg + half_at] = v;
                };
                if (PARTS == 2) {
                    put(row >> 3, odd ? 2 : 0, hs);
                    put(row >> 3, odd ? 3 : 1, ls);
                } else {
                    put(0, (odd ? 2 : 0) + (row >> 3), hs);
                }
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int g = 0; g < NG; ++g) sum[g] += __shfl_xor_sync(0xffffffffu, sum[g], o);
            // offset fragment: k = g holds the group sum * 2^-6 in fp16, k = NG + g what that rounding left
            if (lane < 2 * NG) {
                float v = 0.0f;
#pragma unroll
                for (int g = 0; g < NG; ++g) v = (lane & (NG - 1)) == g ? sum[g] * 0.015625f : v;
                const __half h = __float2half_rn(v);
                const __half w = lane < NG ? h : __float2half_rn(v - __half2float(h));
                const int na = PARTS == 2 ? row >> 3 : 0;
                const int reg = (lane >= 8 ? 2 : 0) + (PARTS == 2 ? 0 : row >> 3);
                reinterpret_cast<__half*>(s_off + na * 32 + (row & 7) * 4 + ((lane & 7) >> 1))[2 * reg + (lane & 1)] = w;
            }
            if (lane == 0) s_fac[row] = p.scale * pow2i(24 - f);
        }
        __syncthreads();

        // this lane's rows (r, r + 8): the last position each sees, and the first
        int hi[RT], lo[RT];
        float fac[RT], m[RT], l[RT];
#pragma unroll
        for (int a = 0; a < RT; ++a) {
            const int row = r + 8 * a;
            hi[a] = row < rows ? len - p.q_len + (row0 + row) / p.group : -1;
            lo[a] = p.window > 0 ? hi[a] - p.window + 1 : 0;
            fac[a] = s_fac[row] * (p.soft_cap > 0.0f ? 1.0f : kLog2e);
            m[a] = -INFINITY;
            l[a] = 0.0f;
        }
        // a tile inside [all_lo, all_hi] is seen whole by every row
        const int all_hi = len - p.q_len + row0 / p.group;
        const int all_lo = p.window > 0 ? len - p.q_len + (row0 + rows - 1) / p.group - p.window + 1 : 0;
        const int any_lo = p.window > 0 ? all_hi - p.window + 1 : 0;
        constexpr bool kQRegs = NA == 1 && NG <= 4;
        uint4 qreg[kQRegs ? NG * 2 : 1];
        if constexpr (kQRegs) {
#pragma unroll
            for (int i = 0; i < NG * 2; ++i) qreg[i] = s_q[i * 32 + lane];
        }
        uint4 oreg[NA];
#pragma unroll
        for (int n = 0; n < NA; ++n) oreg[n] = s_off[n * 32 + lane];
        float acc[2 * NG][RT][4];
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
            for (int a = 0; a < RT; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][a][j] = 0.0f;
        int E = 0;                                 // exponent field the P' scaling is made for
        float sigma = pow2i(20);

        // A lane's columns of S^T and P: slots (h, j) of tile halves h are the
        // positions 8 h + 2 c4 + (j ^ (c4 & 1)).  The swap for odd c4 spreads the
        // V rows of one load over both halves of the banks.
        const int swap = c4 & 1;
        auto tile = [&](const uint8_t* st, int pos) {
            const uint8_t* kcode = st;
            const uint8_t* vcode = st + F::CODES;
            const uint8_t* kscale = st + 2 * F::CODES;
            const uint8_t* vscale = kscale + F::SCALES;
            float s[RT][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int krow = 8 * h + (r ^ ((r >> 1) & 1));     // the position of column r
                uint32_t kw[NG];
                lds_words<NG>(kcode + krow * 16 * NG + c4 * 4 * NG, kw);
                uint32_t d0w[NG / 2], d1w[NG / 2];
                lds_words<NG / 2>(kscale + (8 * h + 2 * c4 + swap) * 2 * NG, d0w);
                lds_words<NG / 2>(kscale + (8 * h + 2 * c4 + 1 - swap) * 2 * NG, d1w);
                // offset: B = the scales of position `krow`, k = g and again NG + g
                uint32_t ob = 0u;
                if (NG > 2 || c4 < 2) ob = *reinterpret_cast<const uint32_t*>(kscale + krow * 2 * NG + 4 * (c4 & (NG / 2 - 1)));
                float off[NA][4], part[NA][4];
#pragma unroll
                for (int n = 0; n < NA; ++n)
                    mma_f16_zero(off[n], oreg[n].x, oreg[n].y, oreg[n].z, oreg[n].w, ob, NG == 8 ? ob : 0u);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t w8 = kw[g] >> 8;
                    const uint32_t b0 = kw[g] & 0x000F000Fu, b1 = kw[g] & 0x00F000F0u;
                    const uint32_t b2 = w8 & 0x000F000Fu, b3 = w8 & 0x00F000F0u;
                    const float d0 = g & 1 ? half_hi(d0w[g / 2]) : half_lo(d0w[g / 2]);
                    const float d1 = g & 1 ? half_hi(d1w[g / 2]) : half_lo(d1w[g / 2]);
#pragma unroll
                    for (int n = 0; n < NA; ++n) {
                        uint4 a0, a1;
                        if constexpr (kQRegs) {
                            a0 = qreg[2 * g];
                            a1 = qreg[2 * g + 1];
                        } else {
                            a0 = s_q[((n * NG + g) * 2) * 32 + lane];
                            a1 = s_q[((n * NG + g) * 2 + 1) * 32 + lane];
                        }
                        float x[4];
                        mma_f16_zero(x, a0.x, a0.y, a0.z, a0.w, b0, b1);
                        mma_f16(x, a1.x, a1.y, a1.z, a1.w, b2, b3);
                        if (g == 0) {
                            part[n][0] = d0 * x[0];
                            part[n][1] = d1 * x[1];
                            part[n][2] = d0 * x[2];
                            part[n][3] = d1 * x[3];
                        } else {
                            part[n][0] = fmaf(d0, x[0], part[n][0]);
                            part[n][1] = fmaf(d1, x[1], part[n][1]);
                            if (PARTS == 2 || RT == 2) {
                                part[n][2] = fmaf(d0, x[2], part[n][2]);
                                part[n][3] = fmaf(d1, x[3], part[n][3]);
                            }
                        }
                    }
                }
                // offset in the units of the products: -8 * 2^6 * 2^-24
#pragma unroll
                for (int a = 0; a < RT; ++a)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const float v = PARTS == 2 ? fmaf(part[a][2 + j], 1.0f / 2048.0f, part[a][j]) : part[0][2 * a + j];
                        const float o = PARTS == 2 ? off[a][j] : off[0][2 * a + j];
                        s[a][2 * h + j] = fmaf(o, -3.0517578125e-5f, v) * fac[a];
                    }
            }
            if (p.soft_cap > 0.0f) {
#pragma unroll
                for (int a = 0; a < RT; ++a)
#pragma unroll
                    for (int j = 0; j < 4; ++j) s[a][j] = tanhf(s[a][j] / p.soft_cap) * p.soft_cap * kLog2e;
            }
            // largest V scale: the tile's scale words are dealt out over the lanes
            uint32_t top = 0u;
            if (NG >= 4 || lane < 16) {
                constexpr int NW = NG == 8 ? 2 : 1;
                uint32_t w[NW];
                lds_words<NW>(vscale + lane * 4 * NW, w);
#pragma unroll
                for (int i = 0; i < NW; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
            }
            // a tile at the edge of what some row sees: masks; what no row sees, and NaN scales, do not set the range
            uint32_t keep[RT][2];
#pragma unroll
            for (int a = 0; a < RT; ++a) keep[a][0] = keep[a][1] = 0xFFFFFFFFu;
            if (pos < all_lo || pos + kTilePos - 1 > all_hi) {
                const int word_pos = pos + (NG == 2 ? lane : lane >> 1);   // the position of the lane's scale words
                if (word_pos >= len || word_pos < any_lo || top >= 0x7C00u) top = 0u;
#pragma unroll
                for (int a = 0; a < RT; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at0 = pos + 8 * h + 2 * c4 + swap, at1 = pos + 8 * h + 2 * c4 + 1 - swap;
                        const bool see0 = at0 <= hi[a] && at0 >= lo[a], see1 = at1 <= hi[a] && at1 >= lo[a];
                        s[a][2 * h] = see0 ? s[a][2 * h] : -INFINITY;
                        s[a][2 * h + 1] = see1 ? s[a][2 * h + 1] : -INFINITY;
                        keep[a][h] = (see0 ? 0x0000FFFFu : 0u) | (see1 ? 0xFFFF0000u : 0u);
                    }
            }
            // ---- running maximum and the exponent of the V scales
            const int e_tile = static_cast<int>(__reduce_max_sync(0xffffffffu, top) >> 10);
            float mx[RT];
            bool raise = e_tile > E;
#pragma unroll
            for (int a = 0; a < RT; ++a) {
                float v = fmaxf(fmaxf(s[a][0], s[a][1]), fmaxf(s[a][2], s[a][3]));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
                v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
                mx[a] = v;
                raise |= v > m[a] + kLazy;
            }
            if (__any_sync(0xffffffffu, raise)) {
                const int e_new = max(E, e_tile);
                const float shrink = pow2i(E - e_new);
                E = e_new;
                sigma = pow2i(20 - E);
#pragma unroll
                for (int a = 0; a < RT; ++a) {
                    const float mn = fmaxf(m[a], mx[a]);
                    const float alpha = m[a] == mn ? 1.0f : ex2(m[a] - mn);
                    m[a] = mn;
                    l[a] *= alpha;
                    // the accumulator's columns are rows 2 c4 and 2 c4 + 1 of this row tile
                    const float f0 = shrink * __shfl_sync(0xffffffffu, alpha, 8 * c4);
                    const float f1 = shrink * __shfl_sync(0xffffffffu, alpha, 8 * c4 + 4);
#pragma unroll
                    for (int i = 0; i < 2 * NG; ++i) {
                        acc[i][a][0] *= f0;
                        acc[i][a][1] *= f1;
                        acc[i][a][2] *= f0;
                        acc[i][a][3] *= f1;
                    }
                }
            }
#pragma unroll
            for (int a = 0; a < RT; ++a) {
                const float ms = m[a] == -INFINITY ? 0.0f : m[a];
#pragma unroll
                for (int j = 0; j < 4; ++j) s[a][j] = ex2(s[a][j] - ms);
                l[a] += (s[a][0] + s[a][1]) + (s[a][2] + s[a][3]);
#pragma unroll
                for (int j = 0; j < 4; ++j) s[a][j] *= sigma;
            }
            // ---- output: V rows of the lane's positions, nibbles of row block r
            uint32_t vw[4][NG / 2], dv[4][NG / 2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int row = (j >> 1) * 8 + 2 * c4 + ((j & 1) ^ swap);
                lds_words<NG / 2>(vcode + row * 16 * NG + r * 2 * NG, vw[j]);
                lds_words<NG / 2>(vscale + row * 2 * NG, dv[j]);
            }
            const __half2 kOff = bits_h2(0x64086408u);          // 1032
            const __half2 kDiv = bits_h2(0x2C002C00u), kOff16 = bits_h2(0xD480D480u);   // 1/16, -72
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                uint32_t bh[RT][2], bl[RT][2];
#pragma unroll
                for (int a = 0; a < RT; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w0 = dv[2 * h][g / 2], w1 = dv[2 * h + 1][g / 2];
                        const float x0 = s[a][2 * h] * (g & 1 ? half_hi(w0) : half_lo(w0));
                        const float x1 = s[a][2 * h + 1] * (g & 1 ? half_hi(w1) : half_lo(w1));
                        const __half2 hh = __floats2half2_rn(x0, x1);
                        bh[a][h] = h2_bits(hh) & keep[a][h];       // a masked position's scale may be anything
                        if (PARTS == 2)
                            bl[a][h] = h2_bits(__floats2half2_rn(x0 - __low2float(hh), x1 - __high2float(hh))) & keep[a][h];
                    }
                uint32_t f[2][4];                  // [position half][nibble]: the integers c - 8
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t t = __byte_perm(vw[2 * h][g / 2], vw[2 * h + 1][g / 2], g & 1 ? 0x7632 : 0x5410);
                    const uint32_t t8 = t >> 8;
                    f[h][0] = h2_bits(__hsub2(bits_h2((t & 0x000F000Fu) | 0x64006400u), kOff));
                    f[h][1] = h2_bits(__hfma2(bits_h2((t & 0x00F000F0u) | 0x64006400u), kDiv, kOff16));
                    f[h][2] = h2_bits(__hsub2(bits_h2((t8 & 0x000F000Fu) | 0x64006400u), kOff));
                    f[h][3] = h2_bits(__hfma2(bits_h2((t8 & 0x00F000F0u) | 0x64006400u), kDiv, kOff16));
                }
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int a = 0; a < RT; ++a) {
                        float (&o)[4] = acc[2 * g + q2][a];
                        if constexpr (PARTS == 2) {
                            float x[4];
                            mma_f16_zero(x, f[0][2 * q2], f[0][2 * q2 + 1], f[1][2 * q2], f[1][2 * q2 + 1], bl[a][0], bl[a][1]);
                            mma_f16(x, f[0][2 * q2], f[0][2 * q2 + 1], f[1][2 * q2], f[1][2 * q2 + 1], bh[a][0], bh[a][1]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[j] += x[j];
                        } else {
                            mma_f16(o, f[0][2 * q2], f[0][2 * q2 + 1], f[1][2 * q2], f[1][2 * q2 + 1], bh[a][0], bh[a][1]);
                        }
                    }
            }
        };

        // ---------------------------------------------------------- the item's chunks
        for (; u < seg1; ++u) {
            __syncwarp();                          // the slot below was read by every lane
            ask(fill);
            fill = fill + 1 == kStages ? 0 : fill + 1;
            if ((have >> use) & 1u) {
                if (!dead) dead = !mbar_wait(bars + use, (phase >> use) & 1u);
                phase ^= 1u << use;
                tile(my_ring + use * F::STAGE, (at.first + at.ch * kChunkTiles + warp) * kTilePos);
            }
            use = use + 1 == kStages ? 0 : use + 1;
            step(at, p, tab, items);
        }

        // ---------------------------------------------------------- merge the warps
#pragma unroll
        for (int a = 0; a < RT; ++a) {
            l[a] += __shfl_xor_sync(0xffffffffu, l[a], 1);
            l[a] += __shfl_xor_sync(0xffffffffu, l[a], 2);
            if (c4 == 0) {
                s_ml[(warp * ROWS + r + 8 * a) * 2] = m[a];
                s_ml[(warp * ROWS + r + 8 * a) * 2 + 1] = l[a];
            }
        }
        __syncthreads();
        // weight of this warp for its accumulator columns
        float wgt[RT][2];
#pragma unroll
        for (int a = 0; a < RT; ++a)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int row = 8 * a + 2 * c4 + j;
                float M = -INFINITY;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) M = fmaxf(M, s_ml[(w * ROWS + row) * 2]);
                const float mine = s_ml[(warp * ROWS + row) * 2];
                wgt[a][j] = mine == -INFINITY ? 0.0f : ex2(mine - M) * pow2i(E - 20);
            }
        const bool whole = seg0 == item0 && seg1 == item1;
        const int slot = seg0 == u0 ? 0 : 1;
        float* const part = p.part + (static_cast<long long>(blockIdx.x) * 2 + slot) * (ROWS * (D + 2));
#pragma unroll
        for (int g0 = 0; g0 < NG; g0 += F::SG) {
            if (g0 > 0) __syncthreads();
#pragma unroll
            for (int g = g0; g < g0 + F::SG; ++g)
#pragma unroll
                for (int a = 0; a < RT; ++a)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float4 v;
                        v.x = acc[2 * g][a][j] * wgt[a][j];
                        v.y = acc[2 * g][a][2 + j] * wgt[a][j];
                        v.z = acc[2 * g + 1][a][j] * wgt[a][j];
                        v.w = acc[2 * g + 1][a][2 + j] * wgt[a][j];
                        *reinterpret_cast<float4*>(s_merge + (warp * ROWS + 8 * a + 2 * c4 + j) * F::MROW + (g - g0) * 32 + 4 * r) = v;
                    }
            __syncthreads();
            for (int i = threadIdx.x; i < rows * F::SG * 8; i += kThreads) {
                const int row = i / (F::SG * 8), d4 = i - row * (F::SG * 8);
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float4 v = *reinterpret_cast<const float4*>(s_merge + (w * ROWS + row) * F::MROW + d4 * 4);
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                    M = fmaxf(M, s_ml[(w * ROWS + row) * 2]);
                }
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
                    const float mw = s_ml[(w * ROWS + row) * 2], lw = s_ml[(w * ROWS + row) * 2 + 1];
                    L += mw == -INFINITY ? lw : lw * ex2(mw - M);
                }
                const int d = g0 * 32 + d4 * 4;
                if (whole) {
                    const int ri = row0 + row, t = ri / p.group, hd = ri - t * p.group;
                    const long long to = ((static_cast<long long>(item_b) * p.q_len + t) * p.kv_heads + kvh) * p.group * D +
                                         static_cast<long long>(hd) * D + d;
                    const float inv = L == 0.0f ? 0.0f : 1.0f / L;    // a row that sees nothing is zero
                    store4(p.out, PARTS == 1, to, sum, inv);
                } else {
                    *reinterpret_cast<float4*>(part + row * D + d) = sum;
                    if (d == 0) {
                        part[ROWS * D + row * 2] = M;
                        part[ROWS * D + row * 2 + 1] = L;
                    }
                }
            }
        }
        if (whole) continue;

        // ---------------------------------------------------------- join an item cut over CTAs
        const int cta0 = static_cast<int>(((line0 + 1) * ctas - 1) / total);
        const int cta1 = static_cast<int>((line1 * ctas - 1) / total);
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            const bool last = arrive_acq_rel(p.counters + cta0) == static_cast<unsigned int>(cta1 - cta0);
            if (last) p.counters[cta0] = 0;
            s_misc[1] = last;
        }
        __syncthreads();
        if (!s_misc[1]) continue;
        __threadfence();
        const int n = cta1 - cta0 + 1;
        const int slot0 = real(total * cta0 / ctas) == item0 ? 0 : 1;   // only the first CTA may hold it in its second slot
        auto base = [&](int k) { return p.part + (static_cast<long long>(cta0 + k) * 2 + (k == 0 ? slot0 : 0)) * (ROWS * (D + 2)); };
        const int outs = rows * (D / 4);
        const int ways = max(1, min(n, min(kThreads / outs, F::MERGE / 4 / (outs * 4))));   // threads that share one output
        const int way = threadIdx.x / outs;
        for (int i = ways > 1 ? threadIdx.x - way * outs : threadIdx.x; i < outs; i += ways > 1 ? outs : kThreads) {
            if (ways > 1 && way >= ways) break;
            const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
            float M = -INFINITY, L = 0.0f;
            for (int k = 0; k < n; ++k) M = fmaxf(M, __ldcg(base(k) + ROWS * D + row * 2));
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const int per = (n + ways - 1) / ways, k0 = ways > 1 ? way * per : 0, k1 = min(n, k0 + per);
#pragma unroll 4
            for (int k = k0; k < k1; ++k) {
                const float* b = base(k);
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(b + ROWS * D + row * 2));
                const float4 v = __ldcg(reinterpret_cast<const float4*>(b + row * D + d));
                const float w = ml.x == -INFINITY ? (ml.y == 0.0f ? 0.0f : 1.0f) : ex2(ml.x - M);
                L = fmaf(ml.y, w, L);
                sum.x = fmaf(v.x, w, sum.x); sum.y = fmaf(v.y, w, sum.y);
                sum.z = fmaf(v.z, w, sum.z); sum.w = fmaf(v.w, w, sum.w);
            }
            if (ways == 1) {
                const int ri = row0 + row, t = ri / p.group, hd = ri - t * p.group;
                const long long to = ((static_cast<long long>(item_b) * p.q_len + t) * p.kv_heads + kvh) * p.group * D +
                                     static_cast<long long>(hd) * D + d;
                store4(p.out, PARTS == 1, to, sum, L == 0.0f ? 0.0f : 1.0f / L);
            } else {
                reinterpret_cast<float4*>(s_merge)[way * outs + i] = sum;
                if (d == 0) s_ml[way * ROWS + row] = L;      // ways <= kWarps * 2 entries a row
            }
        }
        if (ways > 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < outs; i += kThreads) {
                const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float L = 0.0f;
                for (int k = 0; k < ways; ++k) {
                    const float4 v = reinterpret_cast<const float4*>(s_merge)[k * outs + i];
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                    L += s_ml[k * ROWS + row];
                }
                const int ri = row0 + row, t = ri / p.group, hd = ri - t * p.group;
                const long long to = ((static_cast<long long>(item_b) * p.q_len + t) * p.kv_heads + kvh) * p.group * D +
                                     static_cast<long long>(hd) * D + d;
                store4(p.out, PARTS == 1, to, sum, L == 0.0f ? 0.0f : 1.0f / L);
            }
        }
    }
}

template <int NG, int RT, int PARTS>
cudaError_t launch_cfg(Kv4Attn p, int sms, int max_ctas, cudaStream_t stream) {
    using F = Cfg<NG, RT, PARTS>;
    const int smem = F::SMEM + (2 * p.batch + 1) * static_cast<int>(sizeof(int));
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_attn_kernel<NG, RT, PARTS>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   F::SMEM + (2 * kKv4MaxBatch + 1) * static_cast<int>(sizeof(int)));
        if (e != cudaSuccess) return e;
        configured[dev & 63] = true;
    }
    // One wave: two CTAs an SM where registers and 227 KB of shared memory hold two.
    const int per_sm = NG <= 4 && RT == 1 && 2 * (smem + 1024) <= 227 * 1024 ? 2 : 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(std::min(per_sm * sms, max_ctas));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kv4_attn_kernel<NG, RT, PARTS>, p);
}

// Rows of one row tile: 8, or 16 where more than 8 rows share a kv head and
// the accumulators of 16 fit the registers (D <= 128).
int tile_rows(int rows, int head_dim) { return rows > 8 && head_dim <= 128 ? 16 : 8; }

}  // namespace

int kv4_attention_max_ctas(int sms) { return 2 * sms; }

size_t kv4_attention_workspace_bytes(int q_rows, int head_dim, int sms) {
    const size_t ctas = kv4_attention_max_ctas(sms);
    return (ctas * 4 + 255) / 256 * 256 + ctas * 2 * tile_rows(q_rows, head_dim) * (head_dim + 2) * 4;
}

cudaError_t launch_kv4_attention(const Kv4Attn& a, void* workspace, int sms, cudaStream_t stream) {
    Kv4Attn p = a;
    const int ctas = kv4_attention_max_ctas(sms);
    const int rows = p.q_len * p.group, tr = tile_rows(rows, p.head_dim);
    p.row_tiles = (rows + tr - 1) / tr;
    p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
    p.counters = static_cast<unsigned int*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (static_cast<size_t>(ctas) * 4 + 255) / 256 * 256);
    const bool wide = p.type == ALJ_KV_F32;
#define ALJ_KV4(NG, RT)                                                      \
    return wide ? launch_cfg<NG, RT, 2>(p, sms, ctas, stream) : launch_cfg<NG, RT, 1>(p, sms, ctas, stream)
    if (p.head_dim == 256) ALJ_KV4(8, 1);
    if (p.head_dim == 128) {
        if (tr == 16) ALJ_KV4(4, 2);
        ALJ_KV4(4, 1);
    }
    if (p.head_dim != 64) return cudaErrorNotSupported;
    if (tr == 16) ALJ_KV4(2, 2);
    ALJ_KV4(2, 1);
#undef ALJ_KV4
}

}  // namespace alj

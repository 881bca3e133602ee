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
//   * Both products run on mma.sync m16n8k16 (fp16 operands, fp32 sums), 16
//     positions or dims by 8 columns, a column being a row's query vector.
//     (tcgen05 has no use for 8 columns: its operands come from shared memory,
//     so every decoded tile would be written there and read again.)
//   * The K codes are the A operand of S = K q^T without being converted: a
//     nibble masked out of its word is the fp16 subnormal c * 2^-24 (or
//     16 c * 2^-24), exact, so 8 codes cost 4 LOP3 and a shift.  The slots
//     with the factor 16 have q / 16 on the other side.
//   * q is scaled by a power of two into fp16's range.  bf16 queries are
//     exact in one column; their offset -8 is sum_g dK[p, g] * (-8 sum_{j in
//     g} q_j), one more MMA with the fp16 scales as they are stored for its A
//     operand.  fp32 queries take two columns, each a multiple of a fixed step
//     of the row's group of 32 (at most 2^-10 and 2^-22 of the group's largest
//     value, so an element is off by at most 2^-23 of that).  Their groups' sums,
//     with the offset -8 sum_j q_j, are exact integers: neither the tensor
//     cores' truncation nor an outlier in another group enters.  (One step for
//     the whole row loses 1e-4 of the result where q has an outlier of 300;
//     a group's scale and offset cost 4 FFMA and a shared load, asked for ahead
//     of its products: 8 sequences of 8192, 32 fp32 heads on 8, 33.0 us against
//     32.7, D 256 53.5 against 51.5.  Loaded after the products, short contexts
//     took 0.5 us more.)
//     4 fp32 rows, as 8 bf16 ones, fill one MMA's columns.
//   * P = 2^(S - M), M the running maximum less a shift t: P lies where fp16
//     is precise, and no other scaling is kept.  One movmatrix turns the
//     accumulator layout (rows = positions) into the B operand of
//     O^T = V^T P^T.  V's group scales are folded into P: for bf16 outputs as
//     fp16 products of the rounded P, for fp32 ones in fp32, rounded into a
//     high and a low part in the row's two columns.  t follows the largest V
//     scale seen, so that P dV uses the upper part of fp16's range whatever
//     the size of V.
//   * V codes become the exact fp16 integers c - 8 (the sums then stay as
//     small as the result; adding -8 sum P dV afterwards would lose 2-3 digits
//     over long contexts): (bits | 1024) - 1032, or (bits | 1024) / 16 - 72, the
//     well-known reading of small integers as the low bits of an fp16 number.
//     Two positions are interleaved by one PRMT, no transposing load needed.
//   * Rounding points: q parts, P parts, the output type.  Scores, softmax
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
// order, so results do not depend on timing.  The ring
// of chunks is filled two chunks ahead, by the warps in turn: each lane one
// bulk copy (K codes, V codes, K scales or V scales of the tiles that share a
// page).  A ninth warp for it would cut every warp from 128 to 96 registers,
// and address arithmetic in every warp for itself was half of all
// instructions.
// For pages of 16 that is 32 copies a chunk, issued one after the other, and
// still faster than 16-byte pieces copied by every warp for itself (8 sequences
// of 8192: 33 us against 36; pages of 32: 30 against 35).
//
// Measured (1965 MHz, measured copy rate 6473 GB/s): two sequences of 131072,
// 64 query heads on 8 kv heads, D 128, bf16: 79 us, 3.8 TB/s; 32 ragged
// sequences up to 16384: 55 us, 3.3 TB/s; 4096 positions of one sequence, fp32:
// 11.6 us.  The long ones are bound by issue: 374 instructions a tile (2304
// bytes) at 2.45 a clock and SM, ALU pipe 55 % busy, DRAM 44 %; the short ones
// by the chain launch - lengths - page - tile - merge - join.  Tried and
// slower, against 80 us: scores of the next tile beside the values of this one (84 us), tiles
// asked for 3 chunks ahead (88 us), one loop with the item's start inside
// (116 us: the registers no longer hold).
#include "kv4.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
constexpr int kTilePos = 16;
constexpr int kChunkTiles = kWarps;
constexpr int kStages = 4;
constexpr int kAhead = 2;        // chunks asked for before their turn
constexpr int kItemCost = 2;     // chunks that an item's start and end are worth (4: 80.6 us for 2 x 131072, 80.0 with 2)
constexpr int kWholeItem = 4;    // chunks of the average item up to which none is cut for want of work
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 2.0f;    // a row's maximum is raised only when a score exceeds it by 2 (log2)
constexpr float kNone = -3.4e38f;  // running maximum of a row that has seen nothing: below every finite score

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
__device__ __forceinline__ void mma_f16_k8_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%7,%7,%7,%7};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(b0), "f"(0.0f));
}
// 8 x 8 transpose of 16-bit elements over the warp: lane 4 i + j holds columns 2 j, 2 j + 1 of row i.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
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
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }   // 2^e, normal
__device__ __forceinline__ unsigned int arrive_acq_rel(unsigned int* p) {
    unsigned int old;
    asm volatile("atom.add.acq_rel.gpu.global.u32 %0, [%1], 1;" : "=r"(old) : "l"(p) : "memory");
    return old;
}

// A constant the compiler keeps in a register: as an immediate it would cost
// LOP3 its place for a second one.
__device__ __forceinline__ uint32_t hide(uint32_t v) {
    asm volatile("" : "+r"(v));
    return v;
}

// Four outputs sum * inv at element `to`, one rounding where the type is bf16.
__device__ __forceinline__ void store4(void* out, bool bf16, long long to, float4 sum, float inv) {
    sum.x *= inv; sum.y *= inv; sum.z *= inv; sum.w *= inv;
    if (inv == 0.0f) sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);   // a row that sees nothing, whatever its sums are
    if (bf16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(sum.x, sum.y), b = __floats2bfloat162_rn(sum.z, sum.w);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(out) + to) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    } else {
        *reinterpret_cast<float4*>(static_cast<float*>(out) + to) = sum;
    }
}

// NW consecutive 32-bit words from shared memory (aligned to 4 NW bytes, at most 16).
template <int NW>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[NW]) {
    if constexpr (NW % 4 == 0) {
#pragma unroll
        for (int i = 0; i < NW / 4; ++i)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(w[4 * i]), "=r"(w[4 * i + 1]), "=r"(w[4 * i + 2]), "=r"(w[4 * i + 3])
                         : "r"(a + 16 * i));
    } else if constexpr (NW == 2) {
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
    } else {
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a));
    }
}

// Shapes of one instantiation: NG groups of 32 dims, CT column tiles of 8,
// PARTS columns a row (2 for fp32 in and out, 1 for bf16).  A row's columns
// are `row` (bf16), or row and row + 4 of a column tile's 4 rows (fp32).
template <int NG, int CT, int PARTS>
struct Cfg {
    static constexpr int D = 32 * NG;
    static constexpr int COLS = 8 * CT;
    static constexpr int ROWS = COLS / PARTS;
    static constexpr int CODES = 256 * NG;                  // code bytes of a tile (K or V)
    static constexpr int SCALES = 32 * NG;
    static constexpr int TILE = 2 * (CODES + SCALES);
    static constexpr int STAGE = kWarps * TILE;             // a chunk: K codes, V codes, K scales, V scales of its tiles
    static constexpr int RING = kStages * STAGE;
    static constexpr int SG = CT == 1 ? (NG < 4 ? NG : 4) : 2;   // groups merged at a time
    static constexpr int MROW = SG * 32 + 4;                // floats a column in the merge buffer; + 4: no bank conflicts
    static constexpr int MERGE = kWarps * COLS * MROW * 4;
    static constexpr int QFRAG = CT * NG * 2 * 32 * 8;
    static constexpr int QOFF = PARTS == 2 ? CT * NG * 64 : CT * 32 * 8;   // per group offsets and scales, or offset fragments
    static constexpr int BARS = kStages * 2 * 8;            // full and empty
    static constexpr int MISC = (3 * kWarps * COLS + kWarps + 2 * COLS + 8) * 4;
    static constexpr int SMEM = RING + MERGE + QFRAG + QOFF + BARS + MISC;   // + the per-sequence tables
};
// Column of a row's part, and the row of a column.
template <int PARTS>
__device__ __forceinline__ int column_of(int row, int part) {
    return PARTS == 1 ? row : (row >> 2) * 8 + (row & 3) + 4 * part;
}

// One place on the line of chunks: sequence b, item h = kv head * row tiles +
// row tile, chunk ch of that item.
struct Cursor {
    int b, h, ch, chunks, len, first;   // first: the item's first tile
};

struct Tables {      // per sequence, in shared memory
    const int* pre;  // [batch + 1] chunks and item costs before it (of one item)
    const int* len;  // [batch]
};

// First of the p.window positions before `end`: a window may be as long as an int holds, so it is only taken from what
// is longer.
__device__ __forceinline__ int window_start(const Kv4Attn& p, int end) {
    return p.window > 0 && end > p.window ? end - p.window : 0;
}
__device__ __forceinline__ int first_tile(const Kv4Attn& p, int len) {
    return window_start(p, len - p.q_len + 1) / kTilePos;
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

// A warp's pass over one chunk to load: lane 4 w + i copies section i of the
// tile of consumer w.
struct TileSource {
    int pos;     // the tile's first position; at or past the sequence's end there is no tile
    int page;    // its page, or -1
    int off;     // its place in the page
};
__device__ __forceinline__ TileSource find_tile(const Kv4Attn& p, const Cursor& c, int w) {
    TileSource t;
    t.pos = (c.first + c.ch * kChunkTiles + w) * kTilePos;
    t.page = -1;
    t.off = 0;
    if (t.pos < c.len) {
        const int pi = p.page_shift >= 0 ? t.pos >> p.page_shift : t.pos / p.page_size;
        t.page = p.table ? __ldg(p.table + static_cast<long long>(c.b) * p.table_stride + pi) : c.b;
        t.off = t.pos - pi * p.page_size;
    }
    return t;
}
template <int NG>
__device__ __forceinline__ void load_chunk(const Kv4Attn& p, const TileSource& t, int kvh, int len, uint8_t* stage,
                                           uint64_t* bar, int lane) {
    using F = Cfg<NG, 1, 1>;
    const int sec = lane & 3;
    const int w = lane >> 2;
    const bool ok = t.pos < len && t.page >= 0 && t.page < p.pages;
    const uint32_t part = sec < 2 ? F::CODES : F::SCALES;
    uint8_t* dst = stage + (sec & 1) * kWarps * part + (sec < 2 ? 0 : 2 * kWarps * F::CODES) + w * part;
    if (t.pos < len && !ok) {                      // a page id outside the cache: zero scales, so zero rows
        record_fault(ALJ_FAULT_BOUNDS);
        if (sec >= 2)
            for (int i = 0; i < F::SCALES / 16; ++i) reinterpret_cast<uint4*>(dst)[i] = make_uint4(0u, 0u, 0u, 0u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // the slot's next writer is a bulk copy
    }
    const unsigned int tiles = __popc(__ballot_sync(0xffffffffu, ok)) / 4;
    __syncwarp();
    if (lane == 0) mbar_arrive_expect_tx(bar, tiles * F::TILE);
    __syncwarp();
    // the tiles that share a page follow one another there: one copy for all of them
    if (ok && (w == 0 || t.off == 0)) {
        const int run = min(min(kChunkTiles - w, (p.page_size - t.off) / kTilePos), (len - t.pos + kTilePos - 1) / kTilePos);
        // sections of a block start at 0, 16 NG ps, 32 NG ps and 34 NG ps bytes
        const uint32_t row = sec < 2 ? 16 * NG : 2 * NG;
        const uint32_t section = sec < 2 ? 16 * NG * sec : 28 * NG + 2 * NG * sec;
        const uint8_t* src = p.cache + (static_cast<long long>(t.page) * p.kv_heads + kvh) * kv4_block_bytes(p.page_size, F::D) +
                             static_cast<unsigned long long>(section) * p.page_size + static_cast<unsigned long long>(row) * t.off;
        bulk_g2s(dst, src, run * part, bar);
    }
}

// TREE: the q_len new tokens are the nodes of a drafted tree (p.parents): a row sees the positions before the tree, its
// node's ancestors and its node.
template <int NG, int CT, int PARTS, bool TREE>
__global__ void __launch_bounds__(kThreads, NG * CT <= 4 ? 2 : 1) kv4_attn_kernel(const Kv4Attn p) {
    using F = Cfg<NG, CT, PARTS>;
    constexpr int D = F::D, ROWS = F::ROWS, COLS = F::COLS;
    extern __shared__ __align__(128) uint8_t smem[];
    uint8_t* const ring = smem;
    float* const s_merge = reinterpret_cast<float*>(smem + F::RING);
    uint2* const s_q = reinterpret_cast<uint2*>(smem + F::RING + F::MERGE);
    uint2* const s_off = s_q + F::QFRAG / 8;                  // PARTS 1: offset fragments
    float4* const s_group = reinterpret_cast<float4*>(s_off); // PARTS 2: [column tile][group][c4] offsets, scales of 2 columns
    uint64_t* const s_bar = reinterpret_cast<uint64_t*>(s_off + F::QOFF / 8);
    float* const s_m = reinterpret_cast<float*>(s_bar + 2 * kStages);   // [warp][column] running maximum
    float* const s_l = s_m + kWarps * COLS;                             // [warp][column] weighted sum
    float* const s_way = s_l + kWarps * COLS;                           // the join's sums
    int* const s_e = reinterpret_cast<int*>(s_way + kWarps * COLS);     // [warp]
    float* const s_fac = reinterpret_cast<float*>(s_e + kWarps);        // [column] score factor
    int* const s_hi = reinterpret_cast<int*>(s_fac + COLS);             // [column] last position its row sees
    int* const s_misc = s_hi + COLS;
    int* const s_pre = s_misc + 8;
    int* const s_len = s_pre + p.batch + 1;
    int* const s_par = s_len + p.batch;                                 // TREE: [node] the sequence's parents,
    uint32_t* const s_see = reinterpret_cast<uint32_t*>(s_par + kKv4MaxNodes);   // [column] bits of the nodes its row sees,
    uint32_t* const s_any = s_see + COLS * kKv4TreeWords;               // their union, and the first row's position

    const int warp = hide(threadIdx.x >> 5), lane = hide(threadIdx.x & 31);
    const int r = lane >> 2, c4 = lane & 3;
    const int R = p.q_len * p.group;               // rows that share a kv head
    const int items = p.kv_heads * p.row_tiles;    // items of a sequence
    pdl_launch_dependents();
    uint64_t* const full = s_bar;
    uint64_t* const empty = s_bar + kStages;
    if (threadIdx.x == 0) {
        for (int i = 0; i < kStages; ++i) {
            mbar_init(full + i, 1);
            mbar_init(empty + i, kWarps);
        }
        fence_mbar_init();
        s_misc[0] = 0;
    }
    for (int i = threadIdx.x; i < (F::QFRAG + F::QOFF) / 8; i += kThreads) s_q[i] = make_uint2(0u, 0u);
    __syncthreads();
    pdl_wait();

    // lengths (clamped to what the table or page can address, less what the last chunk counts past the end) and the
    // prefix of chunks and item costs
    const int cap = static_cast<int>(min(p.table ? static_cast<long long>(p.table_stride) * p.page_size : p.page_size, 0x7fffff00LL));
    int total = 0;                                 // < 2^31: checked on the host for the longest sequences
    bool longer = false;                           // than an item that is left whole
    for (int b0 = 0; b0 < p.batch; b0 += kThreads) {
        const int b = b0 + threadIdx.x;
        int n = 0;
        if (b < p.batch) {
            int len = __ldg(p.lens + b) + p.len_add;
            if (len < 0 || len > cap) {
                record_fault(ALJ_FAULT_BOUNDS);
                len = len < 0 ? 0 : cap;
            }
            if (TREE && len < p.q_len) len = 0;    // no tree is there
            s_len[b] = len;
            n = chunks_of(p, len) + kItemCost;
            longer |= n > kItemCost + kWholeItem;
        }
        int incl = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += up;
        }
        if (b0 > 0) __syncthreads();               // s_e is read
        if (lane == 31) s_e[warp] = incl;
        __syncthreads();
        int base = total;
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            const int e = s_e[w];
            if (w < warp) base += e;
            total += e;
        }
        if (b < p.batch) s_pre[b + 1] = base + incl;
    }
    if (threadIdx.x == 0) s_pre[0] = 0;
    if (TREE) longer = __syncthreads_or(longer);
    else __syncthreads();
    const Tables tab = {s_pre, s_len};
    // A chunk costs a CTA about as much as 25 parts cost the one that joins them, so where the line is short an item
    // of n places is cut into stretches of sqrt(n / 25): one kv head of 32768 positions 23 us with 256 CTAs of a
    // chunk each, 16 so.  The join itself costs as much as three chunks, so items of up to kWholeItem chunks are left
    // whole: 257 positions 9.1 us in three parts, 7.4 whole.  n is the average item: among short sequences a long one
    // is cut as they are, and dealt out over the CTAs all the same.  Of trees, whose items begin with a table of what
    // each row sees and which come with more rows, all have to be that short: 5 ragged sequences within a window of
    // 1024, 12 heads on 4, 21 nodes 25 us by the average and 20 so.
    const int width = (total + p.batch - 1) / p.batch;
    const int stretch = (TREE ? !longer : width <= kItemCost + kWholeItem) ? width : max(1, __float2int_rn(sqrtf(width / 25.0f)));
    total *= items;
    const int ctas = min(static_cast<int>(gridDim.x), (total + stretch - 1) / stretch);
    if (static_cast<int>(blockIdx.x) >= ctas) return;
    const int share = total / ctas, rem = total - share * ctas;
    auto start_of = [&](int c) { return share * c + min(c, rem); };     // CTA c's first place on the line
    auto cta_at = [&](int x) {
        const int wide = rem * (share + 1);
        return x < wide ? x / (share + 1) : rem + (x - wide) / share;
    };
    // The line with its item costs is dealt out evenly.  Lane 0 finds the place where this CTA starts, lane 1 (and
    // the others) the one where the next does: sequence, item, chunk, and the real chunks before it.
    Cursor at;
    int todo;                                      // chunks of this CTA
    {
        const int x = start_of(blockIdx.x + min(lane, 1));
        int lo = 0, hi = p.batch - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (s_pre[mid] * items <= x) lo = mid;
            else hi = mid - 1;
        }
        const int width = s_pre[lo + 1] - s_pre[lo];
        const int rest = x - s_pre[lo] * items;    // x = total: item `items`, chunk 0
        const int h = rest / width, ch = max(0, rest - h * width - kItemCost);
        const int before = (s_pre[lo] - kItemCost * lo) * items + h * (width - kItemCost) + ch;
        todo = __shfl_sync(0xffffffffu, before, 1) - __shfl_sync(0xffffffffu, before, 0);
        at.b = __shfl_sync(0xffffffffu, lo, 0);
        at.h = __shfl_sync(0xffffffffu, h, 0);
        at.ch = __shfl_sync(0xffffffffu, ch, 0);
    }
    if (todo <= 0) return;
    load_seq(at, p, tab);
    bool dead = false;                             // a chunk never arrived: stop waiting, the fault is recorded
    constexpr bool kQRegs = CT == 1 && NG <= 4;    // q fragments in registers, else read for every tile
    // PARTS 2: the other part's column is two lanes away and weighs 2^-12 where this one is the high part
    const float inv_cap = p.soft_cap > 0.0f ? 1.0f / p.soft_cap : 0.0f;
    const float own = PARTS == 1 || c4 < 2 ? 1.0f : 1.0f / 4096.0f, others = c4 < 2 ? 1.0f / 4096.0f : 1.0f;
    // e: exponent field the shift t is made for.  |dV| < 2^(e - 14) and P <= 2^(t + kLazy): P dV < 2^15, and for bf16,
    // where P itself is rounded to fp16, P <= 2^15
    auto shift_of = [](int e) { return PARTS == 2 ? 27 - e : min(13, 27 - e); };
    auto token_of = [&](int row) { return static_cast<int>((static_cast<unsigned int>(row) * p.group_magic) >> 21); };   // row / group

    // chunk number i of this CTA, at cursor c, into its slot
    auto ask = [&](int i, const Cursor& c) {
        const int slot = i % kStages, head = p.row_tiles == 1 ? c.h : c.h / p.row_tiles;
        const TileSource t = find_tile(p, c, lane >> 2);   // the page id is on its way while the slot empties
        if (i >= kStages && !dead) dead = !mbar_wait(empty + slot, (i / kStages - 1) & 1);
        if (!dead) load_chunk<NG>(p, t, head, c.len, ring + slot * F::STAGE, full + slot, lane);
    };
    if (warp < kAhead) {
        Cursor c = at;
#pragma unroll 1
        for (int i = 0; i < min(kAhead, todo); ++i) {
            if (i == warp) ask(i, c);
            step(c, p, tab, items);
        }
    }
    struct Item {
        int kvh, row0, rows;
    };
    auto item_of = [&](const Cursor& c) {
        Item it;
        it.kvh = p.row_tiles == 1 ? c.h : c.h / p.row_tiles;
        it.row0 = (c.h - it.kvh * p.row_tiles) * ROWS;
        it.rows = min(ROWS, R - it.row0);
        return it;
    };
    int done = 0;                                  // chunks of this CTA behind us
#pragma unroll 1
    while (done < todo) {
        // ---------------------------------------------------------- an item begins
        const int len = at.len;
        const int count = min(at.chunks - at.ch, todo - done);
        __syncthreads();                           // the previous item's tables are read
        int all_lo, all_hi;                        // a tile inside is seen whole by every row
        {
        const Item it = item_of(at);
        const int kvh = it.kvh, row0 = it.row0, rows = it.rows, item_b = at.b;

        // q rows -> columns in B-fragment order, their groups' sums and scales, their score factors.  A lane has NG dims
        // of one group.  (The first warps are busy with the first chunks.)
        for (int row = (warp - kAhead) & (kWarps - 1); row < ROWS; row += kWarps) {
            float x[NG];
            const int i = row0 + row;
            const bool live = row < rows;
            const int t = live ? token_of(i) : 0, hd = live ? i - t * p.group : 0;
            const long long src = (static_cast<long long>(item_b) * p.q_len + t) * p.q_stride +
                                  static_cast<long long>(kvh * p.group + hd) * D + lane * NG;
            constexpr int kSpan = 32 / NG;         // lanes of a group
            const int g = lane / kSpan;
            float big = 0.0f, big_g = 0.0f;        // largest value of the row, of the lane's group
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                x[k] = 0.0f;
                if (live)
                    x[k] = PARTS == 2 ? static_cast<const float*>(p.q)[src + k]
                                      : __bfloat162float(static_cast<const __nv_bfloat16*>(p.q)[src + k]);
                big = fmaxf(big, fabsf(x[k]));
            }
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                if (o == kSpan) big_g = big;
                big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
            }
            // v * 2^f in [2^14, 2^15)
            auto raise_of = [](float v) { return 14 - (static_cast<int>((__float_as_uint(v) >> 23) & 255) - 127); };
            // f of the row, kept where both 2^f and the factor below are normal; PARTS 2: fg of the group, at most 2^40
            // above the row's, so that d * 2^(f - fg) is normal too
            const int f = big > 0.0f ? max(-100, min(126, raise_of(big))) : 0;
            const int fg = PARTS == 2 && big_g > 0.0f ? max(-100, min(min(126, f + 40), raise_of(big_g))) : f;
            const float up = pow2i(fg);
            float sum[PARTS] = {};
#pragma unroll
            for (int k = 0; k < NG; ++k) {
                const float y = x[k] * up;         // |y| < 2^15
                // dim j of its group is slot (c = j / 8, i = j % 8): MMA step (i & 3) >> 1, k half i & 1 (where the
                // codes carry a factor 16), pair c, element i >> 2
                const int j = (lane % kSpan) * NG + k, c = j >> 3, i8 = j & 7, st = (i8 & 3) >> 1;
                // PARTS 2: multiples of 16 and of 2^-8 -- 11 bits each, so that a group's sum of products is exact
                __half v[PARTS];
                v[0] = __float2half_rn(PARTS == 2 ? rintf(y * 0.0625f) * 16.0f : y);
                if (PARTS == 2) v[PARTS - 1] = __float2half_rn(rintf((y - __half2float(v[0])) * 256.0f) * 16.0f);
#pragma unroll
                for (int e = 0; e < PARTS; ++e) {
                    const int col = column_of<PARTS>(row, e);
                    sum[e] += __half2float(v[e]);
                    reinterpret_cast<__half*>(s_q + (((col >> 3) * NG + g) * 2 + st) * 32 + (col & 7) * 4 + c)[2 * (i8 & 1) + (i8 >> 2)] =
                        __hmul(v[e], __ushort_as_half(i8 & 1 ? 0x2C00 : 0x3C00));     // 1/16 or 1
                }
            }
#pragma unroll
            for (int o = kSpan / 2; o > 0; o >>= 1)
#pragma unroll
                for (int e = 0; e < PARTS; ++e) sum[e] += __shfl_xor_sync(0xffffffffu, sum[e], o);
            if constexpr (PARTS == 2) {
                // the group's scale against the row's, and -8 * 2^-24 (the products' units) times its sum, scaled so:
                // powers of two and an integer of 20 bits, all exact
                if (lane % kSpan < 2) {
                    const int e = lane % kSpan, col = column_of<PARTS>(row, e);
                    float* const to = reinterpret_cast<float*>(s_group + ((col >> 3) * NG + g) * 4 + ((col & 7) >> 1)) + (col & 1);
                    const float u = pow2i(f - fg);
                    to[0] = (e ? sum[PARTS - 1] : sum[0]) * -4.76837158203125e-7f * u;
                    to[2] = u;
                }
            } else if (lane % kSpan < 2) {
                // offset fragment: k = g holds the group sum * 2^-6 in fp16, k = NG + g what that rounding left
                const int k = lane % kSpan * NG + g;
                const float v = sum[0] * 0.015625f;
                const __half h = __float2half_rn(v);
                reinterpret_cast<__half*>(s_off + (row >> 3) * 32 + (row & 7) * 4 + ((k & 7) >> 1))[(k >> 3) * 2 + (k & 1)] =
                    k < NG ? h : __float2half_rn(v - __half2float(h));
            }
            if (lane < PARTS) s_fac[column_of<PARTS>(row, lane)] = p.scale * pow2i(24 - f);
        }

        if constexpr (TREE) {
            const int base = len - p.q_len;
            for (int i = threadIdx.x; i < p.q_len; i += kThreads)
                s_par[i] = tree_parent(p.parents + static_cast<long long>(item_b) * p.parents_stride, i);
            if (threadIdx.x <= kKv4TreeWords) s_any[threadIdx.x] = threadIdx.x < kKv4TreeWords ? 0u : 0x7FFFFFFFu;
            __syncthreads();
            if (threadIdx.x < COLS) {              // the position that a column's row stands for, and the nodes it sees
                const int row = PARTS == 1 ? threadIdx.x : 4 * (threadIdx.x >> 3) + (threadIdx.x & 3);
                uint32_t* const see = s_see + threadIdx.x * kKv4TreeWords;
                const int depth = row < rows && base >= 0 ? tree_chain(s_par, token_of(row0 + row), p.window, see) : 0;
                s_hi[threadIdx.x] = depth > 0 ? base + depth - 1 : -1;
                if (depth > 0) {
                    for (int i = 0; i < kKv4TreeWords; ++i) atomicOr(s_any + i, see[i]);
                    atomicMin(s_any + kKv4TreeWords, static_cast<uint32_t>(base + depth - 1));
                }
            }
            all_hi = base - 1;                     // every position before the tree; rows of absent nodes need no care
            all_lo = window_start(p, len);
        }
        if (!TREE && threadIdx.x < COLS) {         // the last position a column's row sees
            const int row = PARTS == 1 ? threadIdx.x : 4 * (threadIdx.x >> 3) + (threadIdx.x & 3);
            s_hi[threadIdx.x] = row < rows ? len - p.q_len + token_of(row0 + row) : -1;
        }
        if constexpr (!TREE) {
            all_hi = len - p.q_len + token_of(row0);
            all_lo = window_start(p, len - p.q_len + token_of(row0 + rows - 1) + 1);
        }
        }
        __syncthreads();

        // this lane's columns 2 c4 and 2 c4 + 1 of each tile
        float fac[CT][2], M[CT][2], l[CT][2], acc[2 * NG][CT][4];
        uint2 qreg[kQRegs ? NG * 2 : 1];
#pragma unroll
        for (int a = 0; a < CT; ++a)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                fac[a][j] = s_fac[8 * a + 2 * c4 + j] * (p.soft_cap > 0.0f ? 1.0f : kLog2e);
                M[a][j] = kNone;
                l[a][j] = 0.0f;
            }
        if constexpr (kQRegs) {
#pragma unroll
            for (int i = 0; i < NG * 2; ++i) qreg[i] = s_q[i * 32 + lane];
        }
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i)
#pragma unroll
            for (int a = 0; a < CT; ++a)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][a][j] = 0.0f;
        int E = 0;
        float limit = shift_of(0) + kLazy;
        const uint32_t m0 = hide(0x000F000Fu), m1 = hide(0x00F000F0u), one = hide(0x64006400u);
        const uint32_t div16 = hide(0x2C002C00u), off16 = hide(0xD480D480u);     // 1/16, -72

        // The lane's places in a slot.  Row positions: krow + 8 h, with rows r and r ^ 1 swapped for every second
        // pair -- it spreads the V rows of one load over both halves of the banks.
        const int krow = r ^ ((r >> 1) & 1);
        const int vrow0 = 2 * c4 + (c4 & 1);       // and vrow0 ^ 1
        const uint32_t codes = smem_u32(ring) + warp * F::CODES;
        const uint32_t scales = smem_u32(ring) + 2 * kWarps * F::CODES + warp * F::SCALES;
        const uint32_t at_k = hide(codes + krow * 16 * NG + c4 * 4 * NG);
        const uint32_t at_v = hide(codes + kWarps * F::CODES + vrow0 * 16 * NG + r * 2 * NG);
        const uint32_t at_ks = hide(scales + krow * 2 * NG);
        const uint32_t at_vs = hide(scales + kWarps * F::SCALES + vrow0 * 2 * NG);
        const uint32_t at_top = hide(scales + kWarps * F::SCALES + lane * (NG == 8 ? 8 : 4));
        const uint32_t at_group = hide(smem_u32(s_group) + c4 * 16);
        auto q_frag = [&](int a, int g, int st) {
            if constexpr (kQRegs) return qreg[2 * g + st];
            return s_q[((a * NG + g) * 2 + st) * 32 + lane];
        };
        auto tile = [&](int slot, int pos) {
            const uint32_t st = slot * F::STAGE;
            // ---- scores: y[a][h][j] of row position krow + 8 h and column 2 c4 + j
            float y[CT][2][2];
            {
                uint32_t kw[2][NG], dw[2][NG / 2];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    lds_words<NG>(at_k + st + h * 128 * NG, kw[h]);
                    lds_words<NG / 2>(at_ks + st + h * 16 * NG, dw[h]);
                }
                float off[CT][4], part[CT][4];
                if constexpr (PARTS == 1) {        // offset: A = the scales, k = g and again NG + g
                    uint32_t o0, o1;
                    if constexpr (NG == 8) {
                        o0 = c4 & 2 ? (c4 & 1 ? dw[0][3] : dw[0][2]) : (c4 & 1 ? dw[0][1] : dw[0][0]);
                        o1 = c4 & 2 ? (c4 & 1 ? dw[1][3] : dw[1][2]) : (c4 & 1 ? dw[1][1] : dw[1][0]);
                    } else if constexpr (NG == 4) {
                        o0 = c4 & 1 ? dw[0][1] : dw[0][0];
                        o1 = c4 & 1 ? dw[1][1] : dw[1][0];
                    } else {                       // k = 4 .. 7 are empty
                        o0 = c4 < 2 ? dw[0][0] : 0u;
                        o1 = c4 < 2 ? dw[1][0] : 0u;
                    }
#pragma unroll
                    for (int a = 0; a < CT; ++a) {
                        const uint2 b = s_off[a * 32 + lane];
                        if constexpr (NG == 8) mma_f16_zero(off[a], o0, o1, o0, o1, b.x, b.y);
                        else mma_f16_k8_zero(off[a], o0, o1, b.x);
                    }
                }
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    uint32_t f[2][4];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w8 = kw[h][g] >> 8;
                        f[h][0] = kw[h][g] & m0;
                        f[h][1] = kw[h][g] & m1;
                        f[h][2] = w8 & m0;
                        f[h][3] = w8 & m1;
                    }
                    const float d0 = g & 1 ? half_hi(dw[0][g / 2]) : half_lo(dw[0][g / 2]);
                    const float d1 = g & 1 ? half_hi(dw[1][g / 2]) : half_lo(dw[1][g / 2]);
#pragma unroll
                    for (int a = 0; a < CT; ++a) {
                        const uint2 b0 = q_frag(a, g, 0), b1 = q_frag(a, g, 1);
                        float x[4];
                        uint32_t gr[4];            // the group's offsets and scales, on their way before the products
                        if constexpr (PARTS == 2) lds_words<4>(at_group + (a * NG + g) * 64, gr);
                        mma_f16_zero(x, f[0][0], f[1][0], f[0][1], f[1][1], b0.x, b0.y);
                        mma_f16(x, f[0][2], f[1][2], f[0][3], f[1][3], b1.x, b1.y);
                        if constexpr (PARTS == 2) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) x[j] = fmaf(x[j], __uint_as_float(gr[2 + (j & 1)]), __uint_as_float(gr[j & 1]));
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            part[a][j] = g == 0 ? (j < 2 ? d0 : d1) * x[j] : fmaf(j < 2 ? d0 : d1, x[j], part[a][j]);
                    }
                }
                // PARTS 1: offset in the units of the products: -8 * 2^6 * 2^-24
#pragma unroll
                for (int a = 0; a < CT; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float v = part[a][2 * h + j];
                            if constexpr (PARTS == 2) v = fmaf(v, own, __shfl_xor_sync(0xffffffffu, v, 2) * others);
                            else v = fmaf(off[a][2 * h + j], -3.0517578125e-5f, v);
                            y[a][h][j] = v * fac[a][j];
                        }
            }
            if (p.soft_cap > 0.0f) {               // one value at a time, rotated through: tanhf is long
#pragma unroll 1
                for (int k = 0; k < 4 * CT; ++k) {
                    const float v = tanhf(y[0][0][0] * inv_cap) * (p.soft_cap * kLog2e);
#pragma unroll
                    for (int n = 0; n < 4 * CT - 1; ++n) y[n >> 2][(n >> 1) & 1][n & 1] = y[(n + 1) >> 2][((n + 1) >> 1) & 1][(n + 1) & 1];
                    y[CT - 1][1][1] = v;
                }
            }
            // largest V scale of the tile: its scale words are dealt out over the lanes
            uint32_t top = 0u;
            if (NG >= 4 || lane < 16) {
                constexpr int NW = NG == 8 ? 2 : 1;
                uint32_t w[NW];
                lds_words<NW>(at_top + st, w);
#pragma unroll
                for (int i = 0; i < NW; ++i) top = max(top, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
            }
            // a tile at the edge of what some row sees: masks; what no row sees does not set the shift
            uint32_t keep[CT][2];
#pragma unroll
            for (int a = 0; a < CT; ++a) keep[a][0] = keep[a][1] = 0xFFFFFFFFu;
            if (pos < all_lo || pos + kTilePos - 1 > all_hi) {
                const int word_pos = pos + (NG == 2 ? lane : lane >> 1);   // the position of the lane's scale words
                if constexpr (TREE) {
                    const int node = word_pos - (all_hi + 1);
                    if (word_pos >= len || (node >= 0 && !tree_sees(s_any, node)) ||
                        (p.window > 0 && static_cast<int>(s_any[kKv4TreeWords]) - word_pos >= p.window))
                        top = 0u;
                } else if (word_pos >= len || (p.window > 0 && all_hi - word_pos >= p.window)) {
                    top = 0u;
                }
#pragma unroll
                for (int a = 0; a < CT; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int at_pos = pos + krow + 8 * h;
                        bool see[2];
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const int hi = s_hi[8 * a + 2 * c4 + j];
                            if constexpr (TREE) {  // hi: the position the row stands for, -1 where its node is absent
                                const int node = at_pos - (all_hi + 1);
                                if (node < 0) see[j] = hi >= 0 && (p.window == 0 || hi - at_pos < p.window);
                                else see[j] = hi >= 0 && node < p.q_len && tree_sees(s_see + (8 * a + 2 * c4 + j) * kKv4TreeWords, node);
                            } else {
                                see[j] = at_pos <= hi && (p.window == 0 || hi - at_pos < p.window);
                            }
                            y[a][h][j] = see[j] ? y[a][h][j] : -INFINITY;
                        }
                        keep[a][h] = transpose8((see[0] ? 0x0000FFFFu : 0u) | (see[1] ? 0xFFFF0000u : 0u));
                    }
            }
            // ---- P = 2^(score - M); M is moved when a score passes it by more than kLazy, or a V scale its range
            float most = -INFINITY;
#pragma unroll
            for (int a = 0; a < CT; ++a)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    most = fmaxf(most, fmaxf(y[a][0][j], y[a][1][j]) - M[a][j]);
            const bool raise = most > limit || static_cast<int>(top >> 10) > E;
            if (__any_sync(0xffffffffu, raise)) {
                if (top >= 0x7C00u) {              // a NaN scale sets no shift, but its words' other groups do
                    constexpr int NW = NG == 8 ? 2 : 1;
                    uint32_t w[NW];
                    lds_words<NW>(at_top + st, w);
                    top = 0u;
#pragma unroll
                    for (int i = 0; i < 2 * NW; ++i) {
                        const uint32_t h = (w[i >> 1] >> (16 * (i & 1))) & 0x7FFFu;
                        if (h < 0x7C00u) top = max(top, h);
                    }
                }
                const int e_new = max(E, static_cast<int>(__reduce_max_sync(0xffffffffu, top) >> 10));
                const float t_old = shift_of(E), t_new = shift_of(e_new);
                E = e_new;
                limit = t_new + kLazy;
#pragma unroll
                for (int a = 0; a < CT; ++a)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float mx = fmaxf(y[a][0][j], y[a][1][j]);
#pragma unroll
                        for (int o = 4; o < 32; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                        // the maximum M stands for is M + t; a row that has seen nothing keeps kNone
                        float now = M[a][j] == kNone ? -INFINITY : M[a][j] + t_old;
                        now = fmaxf(now, mx) - t_new;
                        now = now == -INFINITY ? kNone : now;
                        const float f = ex2(M[a][j] - now);
                        M[a][j] = now;
                        l[a][j] *= f;
#pragma unroll
                        for (int i = 0; i < 2 * NG; ++i) {
                            acc[i][a][j] *= f;
                            acc[i][a][2 + j] *= f;
                        }
                    }
            }
            uint32_t pp[CT][2];                    // fp16 P of (positions 2 c4, 2 c4 + 1 swapped as krow) x column r
            float pf[CT][2][2];                    // PARTS 2: the same in fp32
#pragma unroll
            for (int a = 0; a < CT; ++a)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float p0 = ex2(y[a][h][0] - M[a][0]), p1 = ex2(y[a][h][1] - M[a][1]);
                    l[a][0] += p0;
                    l[a][1] += p1;
                    if constexpr (PARTS == 1) {
                        pp[a][h] = transpose8(h2_bits(__floats2half2_rn(p0, p1)));
                    } else {                       // 32-bit transpose: upper and lower halves apart
                        const uint32_t u0 = __float_as_uint(p0), u1 = __float_as_uint(p1);
                        const uint32_t tu = transpose8(__byte_perm(u0, u1, 0x7632));
                        const uint32_t tl = transpose8(__byte_perm(u0, u1, 0x5410));
                        pf[a][h][0] = __uint_as_float(__byte_perm(tl, tu, 0x5410));
                        pf[a][h][1] = __uint_as_float(__byte_perm(tl, tu, 0x7632));
                    }
                }
            // ---- output: V rows of the lane's positions, nibbles of row block r
            uint32_t vw[4][NG / 2], dv[4][NG / 2];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                lds_words<NG / 2>(((at_v + st) ^ (j & 1 ? 16 * NG : 0)) + (j >> 1) * 128 * NG, vw[j]);   // slots start at even rows
                lds_words<NG / 2>(((at_vs + st) ^ (j & 1 ? 2 * NG : 0)) + (j >> 1) * 16 * NG, dv[j]);
            }
            const __half2 kOff = bits_h2(0x64086408u);          // 1032
            const __half2 kDiv = bits_h2(div16), kOff16 = bits_h2(off16);
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t pick = g & 1 ? 0x7632 : 0x5410;
                uint32_t b[CT][2];
#pragma unroll
                for (int a = 0; a < CT; ++a)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const uint32_t w0 = dv[2 * h][g / 2], w1 = dv[2 * h + 1][g / 2];
                        if constexpr (PARTS == 2) {
                            // the high column takes the product cut to 11 bits, the low one the rest
                            float x0 = pf[a][h][0] * (g & 1 ? half_hi(w0) : half_lo(w0));
                            float x1 = pf[a][h][1] * (g & 1 ? half_hi(w1) : half_lo(w1));
                            const float c0 = __uint_as_float(__float_as_uint(x0) & 0xFFFFE000u);
                            const float c1 = __uint_as_float(__float_as_uint(x1) & 0xFFFFE000u);
                            x0 = r & 4 ? x0 - c0 : c0;
                            x1 = r & 4 ? x1 - c1 : c1;
                            b[a][h] = h2_bits(__floats2half2_rn(x0, x1)) & keep[a][h];
                        } else {                   // a masked position's scale may be anything: keep clears it
                            b[a][h] = h2_bits(__hmul2(bits_h2(pp[a][h]), bits_h2(__byte_perm(w0, w1, pick)))) & keep[a][h];
                        }
                    }
                uint32_t f[2][4];                  // [position half][nibble]: the integers c - 8
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t t = __byte_perm(vw[2 * h][g / 2], vw[2 * h + 1][g / 2], pick);
                    const uint32_t t8 = t >> 8;
                    f[h][0] = h2_bits(__hsub2(bits_h2(lop3_and_or(t, m0, one)), kOff));
                    f[h][1] = h2_bits(__hfma2(bits_h2(lop3_and_or(t, m1, one)), kDiv, kOff16));
                    f[h][2] = h2_bits(__hsub2(bits_h2(lop3_and_or(t8, m0, one)), kOff));
                    f[h][3] = h2_bits(__hfma2(bits_h2(lop3_and_or(t8, m1, one)), kDiv, kOff16));
                }
#pragma unroll
                for (int q2 = 0; q2 < 2; ++q2)
#pragma unroll
                    for (int a = 0; a < CT; ++a) {
                        float (&o)[4] = acc[2 * g + q2][a];
                        if constexpr (PARTS == 2) {
                            float x[4];
                            mma_f16_zero(x, f[0][2 * q2], f[0][2 * q2 + 1], f[1][2 * q2], f[1][2 * q2 + 1], b[a][0], b[a][1]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) o[j] += x[j];
                        } else {
                            mma_f16(o, f[0][2 * q2], f[0][2 * q2 + 1], f[1][2 * q2], f[1][2 * q2 + 1], b[a][0], b[a][1]);
                        }
                    }
            }
        };

        // ---------------------------------------------------------- its chunks
        const int pos0 = (at.first + at.ch * kChunkTiles + warp) * kTilePos;
#pragma unroll 1
        for (int i = 0; i < count; ++i, ++done) {
            if (((done + kAhead) & (kWarps - 1)) == warp && done + kAhead < todo) {
                Cursor c = at;
                c.ch += i;
                for (int k = 0; k < kAhead; ++k) step(c, p, tab, items);
                ask(done + kAhead, c);
            }
            const int slot = done % kStages;
            if (!dead) dead = !mbar_wait(full + slot, (done / kStages) & 1);
            const int pos = pos0 + i * (kChunkTiles * kTilePos);
            if (pos < len) tile(slot, pos);
            __syncwarp();                          // every lane has read the slot
            if (lane == 0) mbar_arrive(empty + slot);
        }
        Cursor was = at;
        at.ch = at.chunks - 1;                     // on to the next item
        step(at, p, tab, items);
        was.h = hide(was.h);                       // found again, not held in registers over the chunks
        const Item it = item_of(was);
        const int kvh = it.kvh, row0 = it.row0, rows = it.rows;

        // ---------------------------------------------------------- merge the warps
        if constexpr (TREE) {                      // absent nodes took part in the tiles that need no masks
#pragma unroll
            for (int a = 0; a < CT; ++a)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    if (s_hi[8 * a + 2 * c4 + j] < 0) {
                        M[a][j] = kNone;
                        l[a][j] = 0.0f;
                    }
        }
        if (r == 0) {
#pragma unroll
            for (int a = 0; a < CT; ++a)
#pragma unroll
                for (int j = 0; j < 2; ++j) s_m[warp * COLS + 8 * a + 2 * c4 + j] = M[a][j];
        }
        __syncthreads();
        float wgt[CT][2];                          // this warp's weight for its columns
#pragma unroll
        for (int a = 0; a < CT; ++a)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int col = 8 * a + 2 * c4 + j;
                float top = kNone;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * COLS + col]);
                wgt[a][j] = ex2(M[a][j] - top);
                float sum = l[a][j];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (r == 0) s_l[warp * COLS + col] = sum * wgt[a][j];
            }
        const bool whole = count == was.chunks;
        // the item's place on the line, for the CTAs that share it: the first of them keeps its part in its second
        // slot (no other item can begin there and go on), the others in their first
        const int line0 = s_pre[was.b] * items + was.h * (was.chunks + kItemCost) + kItemCost;
        const int cta0 = whole ? 0 : cta_at(line0);
        float* const part = p.part + (static_cast<long long>(blockIdx.x) * 2 + (static_cast<int>(blockIdx.x) == cta0 ? 1 : 0)) * (ROWS * (D + 2));
        // element of the output that row `row`, dim d of this item has
        auto out_at = [&](int row, int d) {
            const int ri = row0 + row, t = token_of(ri), hd = ri - t * p.group;
            return (((static_cast<long long>(was.b) * p.q_len + t) * p.kv_heads + kvh) * p.group + hd) * D + d;
        };
#pragma unroll
        for (int g0 = 0; g0 < NG; g0 += F::SG) {
            if (g0 > 0) __syncthreads();
#pragma unroll
            for (int g = g0; g < g0 + F::SG; ++g)
#pragma unroll
                for (int a = 0; a < CT; ++a)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        *reinterpret_cast<float4*>(s_merge + (warp * COLS + 8 * a + 2 * c4 + j) * F::MROW + (g - g0) * 32 + 4 * r) =
                            make_float4(acc[2 * g][a][j] * wgt[a][j], acc[2 * g][a][2 + j] * wgt[a][j],
                                        acc[2 * g + 1][a][j] * wgt[a][j], acc[2 * g + 1][a][2 + j] * wgt[a][j]);
            __syncthreads();
            for (int i = threadIdx.x; i < rows * F::SG * 8; i += kThreads) {
                const int row = i / (F::SG * 8), d4 = i - row * (F::SG * 8), col = column_of<PARTS>(row, 0);
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                float L = 0.0f;
#pragma unroll
                for (int w = 0; w < kWarps; ++w) {
#pragma unroll
                    for (int e = 0; e < PARTS; ++e) {
                        const float4 v = *reinterpret_cast<const float4*>(s_merge + (w * COLS + col + 4 * e) * F::MROW + d4 * 4);
                        sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                    }
                    L += s_l[w * COLS + col];
                }
                const int d = g0 * 32 + d4 * 4;
                if (whole) {
                    store4(p.out, PARTS == 1, out_at(row, d), sum, L == 0.0f ? 0.0f : 1.0f / L);   // a row that sees nothing is zero
                } else {
                    *reinterpret_cast<float4*>(part + row * D + d) = sum;
                    if (d == 0) {
                        float top = kNone;
                        for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_m[w * COLS + col]);
                        part[ROWS * D + row * 2] = top;
                        part[ROWS * D + row * 2 + 1] = L;
                    }
                }
            }
        }
        if (whole) continue;

        // ---------------------------------------------------------- join an item cut over CTAs
        const int cta1 = cta_at(line0 + was.chunks - 1);
        __syncthreads();                           // every thread's partials, made visible by thread 0's release
        if (threadIdx.x == 0) {
            const bool last = arrive_acq_rel(p.counters + cta0) == static_cast<unsigned int>(cta1 - cta0);
            if (last) p.counters[cta0] = 0;
            s_misc[1] = last;
        }
        __syncthreads();
        if (!s_misc[1]) continue;
        const int n = cta1 - cta0 + 1;
        auto base = [&](int k) { return p.part + (static_cast<long long>(cta0 + k) * 2 + (k == 0 ? 1 : 0)) * (ROWS * (D + 2)); };
        // Threads that share one output take a run of the CTAs each.  The CTAs' weights first: w[row][k], a warp a
        // row, the rows' sums in s_way.
        const int outs = rows * (D / 4);
        const int room = (F::MERGE / 4 - rows * n - 3) / 4;
        const int ways = max(1, min(min(n, kThreads / outs), room / outs));
        const int way = ways > 1 ? threadIdx.x / outs : 0;
        const int per = (n + ways - 1) / ways, k0 = way * per, k1 = min(n, k0 + per);
        const int first = threadIdx.x - way * outs;
        float* const w = s_merge;
#pragma unroll 1
        for (int row = warp; row < rows; row += kWarps) {
            float2 ml = make_float2(kNone, 0.0f);      // the lane's CTA, and what came before it
            for (int k = lane; k < n; k += 32) {
                const float2 x = __ldcg(reinterpret_cast<const float2*>(base(k) + ROWS * D + row * 2));
                w[row * n + k] = x.x;
                const float top = fmaxf(ml.x, x.x);
                ml.y = fmaf(ml.y, ex2(ml.x - top), x.y * ex2(x.x - top));
                ml.x = top;
            }
            float top = ml.x;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const float L = warp_sum(ml.y * ex2(ml.x - top));
            for (int k = lane; k < n; k += 32) w[row * n + k] = ex2(w[row * n + k] - top);
            if (lane == 0) s_way[row] = L;
        }
        float4* const sums = reinterpret_cast<float4*>(s_merge + (rows * n + 3) / 4 * 4);
        __syncthreads();
#pragma unroll 1
        for (int i = first; i < outs && way < ways; i += kThreads) {
            const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            auto add = [&](int k, float4 v) {
                const float f = w[row * n + k];
                sum.x = fmaf(v.x, f, sum.x); sum.y = fmaf(v.y, f, sum.y);
                sum.z = fmaf(v.z, f, sum.z); sum.w = fmaf(v.w, f, sum.w);
            };
#pragma unroll 4
            for (int k = k0; k < k1; ++k) add(k, __ldcg(reinterpret_cast<const float4*>(base(k) + row * D + d)));
            if (ways == 1) store4(p.out, PARTS == 1, out_at(row, d), sum, s_way[row] == 0.0f ? 0.0f : 1.0f / s_way[row]);
            else sums[way * outs + i] = sum;
        }
        if (ways > 1) {
            __syncthreads();
            for (int i = threadIdx.x; i < outs; i += kThreads) {
                const int row = i / (D / 4), d = (i - row * (D / 4)) * 4;
                float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                for (int k = 0; k < ways; ++k) {
                    const float4 v = sums[k * outs + i];
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                store4(p.out, PARTS == 1, out_at(row, d), sum, s_way[row] == 0.0f ? 0.0f : 1.0f / s_way[row]);
            }
        }
    }
}

template <int NG, int CT, int PARTS, bool TREE>
cudaError_t launch_cfg(Kv4Attn p, int sms, int max_ctas, cudaStream_t stream) {
    using F = Cfg<NG, CT, PARTS>;
    constexpr int kTree = TREE ? (kKv4MaxNodes + F::COLS * kKv4TreeWords + kKv4TreeWords + 1) * 4 : 0;
    const int smem = F::SMEM + kTree + (2 * p.batch + 1) * static_cast<int>(sizeof(int));
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_attn_kernel<NG, CT, PARTS, TREE>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   F::SMEM + kTree + (2 * kKv4MaxBatch + 1) * static_cast<int>(sizeof(int)));
        if (e != cudaSuccess) return e;
        configured[dev & 63] = true;
    }
    // One wave: two CTAs an SM where registers and 227 KB of shared memory hold two.  At D 128 the batch's tables leave
    // room for two up to 552 sequences: 500 of 300 positions 94 us, 600 of them 164 us.
    const int per_sm = NG * CT <= 4 && 2 * (smem + 1024) <= 227 * 1024 ? 2 : 1;
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
    return cudaLaunchKernelEx(&cfg, kv4_attn_kernel<NG, CT, PARTS, TREE>, p);
}

// Rows a CTA serves at once: a column tile holds 8 bf16 or 4 fp32 rows; two
// tiles where the rows need them and the accumulators fit (D <= 128): 8
// sequences of 8192 with 16 bf16 rows 44 us in one pass of two tiles, 49 in two
// of one; 8 fp32 rows 47 against 55.  D 256 has room for one tile and one CTA
// an SM (220 registers a thread, 181 KB of ring and merge buffer): 48 us for 4
// bf16 rows of the same, 3.2 TB/s.
int tile_rows(int rows, int head_dim, bool wide) {
    const int one = wide ? 4 : 8;
    return rows > one && head_dim <= 128 ? 2 * one : one;
}

}  // namespace

int kv4_attention_max_ctas(int sms) { return 2 * sms; }

size_t kv4_attention_counter_bytes(int sms) { return (static_cast<size_t>(kv4_attention_max_ctas(sms)) * 4 + 255) / 256 * 256; }

size_t kv4_attention_workspace_bytes(int q_rows, int head_dim, int sms) {
    const size_t ctas = kv4_attention_max_ctas(sms);
    return kv4_attention_counter_bytes(sms) + ctas * 2 * tile_rows(q_rows, head_dim, false) * (head_dim + 2) * 4;
}

cudaError_t launch_kv4_attention(const Kv4Attn& a, void* workspace, int sms, cudaStream_t stream) {
    Kv4Attn p = a;
    const int ctas = kv4_attention_max_ctas(sms);
    const bool wide = p.type == ALJ_KV_F32;
    const int rows = p.q_len * p.group, tr = tile_rows(rows, p.head_dim, wide);
    const bool two = tr > (wide ? 4 : 8);
    p.row_tiles = (rows + tr - 1) / tr;
    p.group_magic = ((1u << 21) + p.group - 1) / p.group;   // row / group for row < 2048, exact as row * group < 2^21
    p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
    p.counters = static_cast<unsigned int*>(workspace);
    p.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kv4_attention_counter_bytes(sms));
#define ALJ_KV4(NG, CT)                                                                                             \
    return p.parents ? (wide ? launch_cfg<NG, CT, 2, true>(p, sms, ctas, stream) : launch_cfg<NG, CT, 1, true>(p, sms, ctas, stream)) \
                     : (wide ? launch_cfg<NG, CT, 2, false>(p, sms, ctas, stream) : launch_cfg<NG, CT, 1, false>(p, sms, ctas, stream))
    if (p.head_dim == 256) ALJ_KV4(8, 1);
    if (p.head_dim == 128) {
        if (two) ALJ_KV4(4, 2);
        ALJ_KV4(4, 1);
    }
    if (p.head_dim != 64) return cudaErrorNotSupported;
    if (two) ALJ_KV4(2, 2);
    ALJ_KV4(2, 1);
#undef ALJ_KV4
}

}  // namespace alj

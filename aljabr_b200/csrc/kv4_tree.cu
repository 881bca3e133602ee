// Attention of drafted trees over the 4-bit KV cache (layout and trees:
// kv4.cuh) on tcgen05, for bf16 queries with many rows a kv head.
//
//   S[i, p] = scale q_i . K_p  (soft cap: S <- cap tanh(S / cap)),  P = softmax
//   over what row i sees: positions before the tree, its node's ancestors, its
//   node (window: the last of these);  O_i = sum_p P[i, p] V_p
//
// A row i is one (node, query head) pair of the nodes x group pairs that share
// a kv head; 128 of them are an MMA's M.  A tile is KT positions.  Every code is
// decoded once for 128 rows, into fp16 operands in shared memory:
//   * K: d (c - 8) 2^-e, row p = the position, in the 128-byte swizzle; e, one
//     of 32 positions, puts the largest of their scales into [2^11, 2^12), so the
//     operand is below 2^15 whatever the cache holds, and scores are scaled back by
//     2^e in fp32.  d (c - 8) has 15 bits: it is rounded to fp16's 11 (2^-11 half a
//     step; the output's own rounding is 2^-8), also where another group's or
//     position's d is up to 2^25 times as large; from there on bits are lost.
//   * V: the same, transposed on the way (a row is a dim, 8 positions 16 bytes): a
//     word of two positions' codes is put together by one PRMT, as the codes of
//     four dims lie in a halfword.  Its e, one of 32 positions too, goes into P.
//   * Q: scaled by a power of two into fp16's range, exact for bf16 to 2^-38 of
//     the row's largest.
//   * P = 2^(S - M + b + e - E) in fp16: M the running maximum, raised when a
//     score passes it by 2^5, E the running largest e, b a bias that keeps P in
//     the upper part of fp16's range.  P is written over S in tensor memory and is
//     the A operand of O += P V from there.  Softmax sums are fp32, of the
//     unrounded P.
//   * A V group that is NaN counts as zeros in the product, and as NaN for the
//     rows that see it: a product with a masked position's zero would be NaN too.
//
// Roles (one CTA an SM, persistent over a line of tiles that is cut into equal parts): a producer warp (bulk copies of a
// tile's codes and scales into a ring), two that find the exponents e of K and V, two warpgroups that decode, a tile each
// in turn, one warp that issues the MMAs, and a warpgroup of softmax for each of two streams: the even and the odd tiles
// of an item have their own S, running maximum and O, so that one stream's softmax runs beside the other's products.
// (D 256: tiles of 64, one stream, as two O do not fit tensor memory beside S.)  The streams are joined when the item
// ends; items cut over CTAs are joined by a second small kernel, which all SMs share (one CTA joining 128 rows of 10 parts
// would read 0.6 MB by itself).
//
// What bounds it: the issue of instructions, most of them of the decoding and of the softmax.  A tile of 128 positions and
// 128 rows takes about 7400 warp instructions and 3400 cycles: 64 % of the issue slots at 20 warps an SM, the tensor pipe
// 35 % of the time, DRAM 14 %.  2 sequences of 65536, 64 query heads on 8, 61 nodes: 378 us by itself, 690 TFLOP/s, and 396 to
// 411 among other work; 24 ragged sequences up to 16384 with 26 nodes: 114 to 117 us.  Tried and slower for the first: tiles
// of 64 with 10 stages of codes (472 us), 8 warps for V (465), one stage of K and four of codes (398 against 388 then).
#define ALJ_OWN_FAULT_WORD     // compiled by itself, for setmaxnreg (build.py)
#include "kv4.cuh"
#include "tc_gemm.cuh"

#include <algorithm>

namespace alj {
namespace {

constexpr int kRows = 128;
constexpr int kPages = 128;           // page ids read from the table at once
// Tiles that an item's start and end are worth on the line.  24 ragged sequences up to 16384, 26 nodes, us: 2 tiles 176,
// 4 136, 6 126, 8 118, 10 120, 12 123, 16 131.
constexpr int kItemCost = 8;
// Places of a CTA: with fewer, joining them costs more than it saves.  1 sequence of 4096, 64 nodes, us: 2 places 29.9,
// 3 28, 4 29.2, 6 32.1, 8 36.
constexpr int kLeast = 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNone = -3.4e38f;     // running maximum of a row that has seen nothing
// P <= 2^(kLazy + kSlack + kBias) = 2^15, or its sum over 32 positions <= kMostSum
constexpr float kLazy = 5.0f, kMostSum = 60000.0f;
constexpr int kSlack = 2, kBias = 8;
constexpr float kMostM = 1048576.0f;  // where M's last place is 2^-3: S - M from the unrounded S is off by less

template <int NG>
struct Shape {
    static constexpr int D = 32 * NG;
    static constexpr int KT = NG == 8 ? 64 : 128;            // positions of a tile
    static constexpr int STREAMS = NG == 8 ? 1 : 2;
    // tiles of scores, of K and of V as fp16, of codes.  Codes take most: they hide the time of the loads.
    static constexpr int S_STAGES = 2, K_STAGES = 2, V_STAGES = NG == 8 ? 1 : 2, RAW = NG == 2 ? 8 : NG == 4 ? 3 : 2;
    // tiles whose exponents are kept: those of tile t + META replace t's, and its codes come once V of t + META - RAW is
    // decoded, for which the products of t + META - RAW - V_STAGES have been done, and t's softmax before them
    static constexpr int META = NG == 2 ? 16 : 8;
    static_assert(META >= RAW + V_STAGES, "exponents kept");
    static constexpr int SOFT = 4 * STREAMS;                 // softmax warps
    static constexpr int WARPS = SOFT + 12;
    // Registers a thread, of the launch's (96 for 5 warpgroups, 128 for 4) that they trade: 5 x 96 = 2 x 128 + 2 x 72 + 80,
    // 4 x 128 = 192 + 3 x 104.  Those who give come down to fewer (to ask for more there is an illegal instruction),
    // those who take wait for no more than is given.
    static constexpr int R_SOFT = STREAMS == 2 ? 128 : 192, R_DECODE = STREAMS == 2 ? 72 : 104, R_REST = STREAMS == 2 ? 80 : 104;
    static constexpr int THREADS = 32 * WARPS, R_LAUNCH = 65536 / THREADS / 8 * 8;
    static_assert(R_SOFT > R_LAUNCH && R_DECODE < R_LAUNCH && R_REST < R_LAUNCH &&
                      STREAMS * R_SOFT + 2 * R_DECODE + R_REST <= WARPS / 4 * R_LAUNCH, "registers that the warpgroups trade");
    // a raw tile: K codes, V codes, K scales, V scales, each by position
    static constexpr int V_CODES = KT * D / 2, K_SC = 2 * V_CODES, V_SC = K_SC + KT * 2 * NG, RAW_BYTES = V_SC + KT * 2 * NG;
    static constexpr int BLOCK_BYTES = 16 * (D + D / 8);     // copied for 16 positions
    static constexpr int KHAT = KT * D * 2, VHAT = KT * D * 2, Q = kRows * D * 2;
    static constexpr int AT_K = Q, AT_V = AT_K + K_STAGES * KHAT, AT_RAW = AT_V + V_STAGES * VHAT, AT_SMALL = AT_RAW + RAW * RAW_BYTES;
    static constexpr int O_COL = S_STAGES * KT;              // tensor memory: S of the tiles, then O of each stream
    static_assert(O_COL + STREAMS * D <= 512, "tensor memory");
};

template <int NG>
struct Small {                        // behind the tiles in shared memory
    using F = Shape<NG>;
    static constexpr int kMeta = F::META;
    uint64_t raw_full[F::RAW], raw_empty[F::RAW], k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], p_full[2], pv_done[2], q_full, done;
    uint64_t meta_full[kMeta];
    int abort, tmem;
    uint32_t valid[F::RAW][4];           // by raw slot: bits of the positions that some row may see
    float k_unit[kMeta][4];           // by tile and 32 positions: 2^e of K, e of V, the largest of those,
    int ev[kMeta][4];
    int e_top[kMeta];
    int nan_any[kMeta];               // and V groups that are NaN: bits by position
    uint8_t nan[kMeta][F::KT];
    uint32_t node_ok[kKv4TreeWords];  // the producer's
    int pages[kPages];
    short par_p[kKv4MaxNodes];
    short par[kKv4MaxNodes];            // the softmax warps'
    uint32_t see[kKv4TreeWords][kRows];
    float fac[kRows];
    float ml[2][kRows][2];            // M, l of each stream
    short er[2][kRows];               // E, and the row's NaN groups
    uint8_t row_nan[2][kRows];
};

template <int NG>
constexpr int smem_bytes() { return 1024 + Shape<NG>::AT_SMALL + static_cast<int>(sizeof(Small<NG>)); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float pow2i(int e) { return __int_as_float((e + 127) << 23); }   // 2^e, normal
__device__ __forceinline__ uint32_t h2_bits(__half2 v) { return *reinterpret_cast<const uint32_t*>(&v); }
__device__ __forceinline__ __half2 bits_h2(uint32_t v) { return *reinterpret_cast<const __half2*>(&v); }
__device__ __forceinline__ void sts128(uint32_t a, uint4 v) {
    asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
template <int NW>
__device__ __forceinline__ void lds_words(uint32_t a, uint32_t (&w)[NW]) {
    if constexpr (NW == 4)
        asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(a));
    else if constexpr (NW == 2)
        asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(a));
    else
        asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[0]) : "r"(a));
}
template <int NW>
__device__ __forceinline__ void sts_words(uint32_t a, const uint32_t (&w)[NW]) {
    if constexpr (NW == 4)
        asm volatile("st.shared.v4.u32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
    else if constexpr (NW == 2)
        asm volatile("st.shared.v2.u32 [%0], {%1, %2};" ::"r"(a), "r"(w[0]), "r"(w[1]) : "memory");
    else
        asm volatile("st.shared.u32 [%0], %1;" ::"r"(a), "r"(w[0]) : "memory");
}
__device__ __forceinline__ uint32_t lds_word(uint32_t a) {
    uint32_t w;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w) : "r"(a));
    return w;
}
// Waits with a limit, that also end once another role has given up.  The roles' loops have to share the instruction
// cache, so these are kept short: a count of tries, each of which the hardware suspends for some microseconds, in place of
// a clock.
constexpr int kTries = 1 << 17;
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p, q;\n .reg .b32 n, a;\n mov.b32 n, 0;\n"
        "WAIT:\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n @p bra DONE;\n"
        " ld.volatile.shared.b32 a, [%3];\n setp.ne.b32 q, a, 0;\n @q bra DONE;\n"
        " add.s32 n, n, 1;\n setp.lt.s32 q, n, %4;\n @q bra WAIT;\n"
        "DONE:\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(smem_u32(const_cast<int*>(gave_up))), "n"(kTries)
        : "memory");
    if (ok == 0u && *gave_up == 0) {
        record_fault(ALJ_FAULT_TIMEOUT);
        *gave_up = 1;
    }
    return ok != 0u;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* gave_up) {
    return __all_sync(0xffffffffu, wait_bar(bar, parity, gave_up));
}
__device__ __forceinline__ void bulk_to(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(smem_u32(bar))
                 : "memory");
}
__device__ __forceinline__ void fence_proxy_shared() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// 32 lanes x 32 columns of 32 bit from tensor memory; the wait is tied to the outputs.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,"
        "%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
// 16 columns asked for, and there: until then nothing may use the registers.
__device__ __forceinline__ void tmem_ask16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_have(uint32_t (&r)[16]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
        "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_ld8(uint32_t taddr, uint32_t (&r)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld8x2(uint32_t at0, uint32_t at1, uint32_t (&r)[8], uint32_t (&q)[8]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%16];\n"
        "tcgen05.ld.sync.aligned.32x32b.x8.b32 {%8,%9,%10,%11,%12,%13,%14,%15}, [%17];\n"
        "tcgen05.wait::ld.sync.aligned;"
        : "=&r"(r[0]), "=&r"(r[1]), "=&r"(r[2]), "=&r"(r[3]), "=&r"(r[4]), "=&r"(r[5]), "=&r"(r[6]), "=&r"(r[7]), "=&r"(q[0]),
          "=&r"(q[1]), "=&r"(q[2]), "=&r"(q[3]), "=&r"(q[4]), "=&r"(q[5]), "=&r"(q[6]), "=&r"(q[7])
        : "r"(at0), "r"(at1)
        : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&r)[8]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}
// d (+)= a b for 64 values of K (four MMAs, fp16): both operands in shared memory, or a in tensor memory.  The whole warp
// comes here and `one` of it issues, so that the operands stay in uniform registers: by a lone thread an MMA took 150
// cycles to issue.
__device__ __forceinline__ void mma64_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t one) {
    asm volatile(
        "{\n .reg .pred p, q, t;\n .reg .b64 a1, a2, a3, b1, b2, b3;\n"
        " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n setp.eq.b32 t, %3, %3;\n"
        " add.s64 a1, %1, 2;\n add.s64 a2, %1, 4;\n add.s64 a3, %1, 6;\n add.s64 b1, %2, 2;\n add.s64 b2, %2, 4;\n add.s64 b3, %2, 6;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a1, b1, %3, t;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a2, b2, %3, t;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], a3, b3, %3, t;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
}
__device__ __forceinline__ void mma64_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t add, uint32_t one) {
    asm volatile(
        "{\n .reg .pred p, q, t;\n .reg .b32 a1, a2, a3;\n .reg .b64 b1, b2, b3;\n"
        " setp.ne.b32 p, %4, 0;\n setp.ne.b32 q, %5, 0;\n setp.eq.b32 t, %3, %3;\n"
        " add.s32 a1, %1, 8;\n add.s32 a2, %1, 16;\n add.s32 a3, %1, 24;\n add.s64 b1, %2, 2;\n add.s64 b2, %2, 4;\n add.s64 b3, %2, 6;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a1], b1, %3, t;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a2], b2, %3, t;\n"
        " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [a3], b3, %3, t;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(add), "r"(one)
        : "memory");
}
__device__ __forceinline__ void commit2(uint64_t* x, uint64_t* y, uint32_t one) {
    asm volatile(
        "{\n .reg .pred q;\n setp.ne.b32 q, %2, 0;\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n"
        " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%1];\n}\n" ::"r"(smem_u32(x)),
        "r"(smem_u32(y)), "r"(one)
        : "memory");
}
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t one;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(one));
    return one;
}

// Codes to fp16.  The 8 codes of a word, each half of an output pair 16 bits
// apart: (0, 4), (1, 5), (2, 6), (3, 7), times the pair of scales d2: (bits | 1024)
// - 1032, or (bits | 1024) / 16 - 72 where the bits lie 4 higher, are c - 8.
__device__ __forceinline__ void decode8(uint32_t w, __half2 d2, uint32_t (&out)[4]) {
    const uint32_t w8 = w >> 8;
    const __half2 off = bits_h2(0x64086408u), div16 = bits_h2(0x2C002C00u), off16 = bits_h2(0xD480D480u);
    out[0] = h2_bits(__hmul2(__hsub2(bits_h2(lop3_and_or(w, 0x000F000Fu, 0x64006400u)), off), d2));
    out[1] = h2_bits(__hmul2(__hfma2(bits_h2(lop3_and_or(w, 0x00F000F0u, 0x64006400u)), div16, off16), d2));
    out[2] = h2_bits(__hmul2(__hsub2(bits_h2(lop3_and_or(w8, 0x000F000Fu, 0x64006400u)), off), d2));
    out[3] = h2_bits(__hmul2(__hfma2(bits_h2(lop3_and_or(w8, 0x00F000F0u, 0x64006400u)), div16, off16), d2));
}
// The largest fp16 magnitude of the words' halves; `finite` leaves NaN and infinity out.
template <int N>
__device__ __forceinline__ uint32_t top_of(const uint32_t (&w)[N], bool finite) {
    uint32_t m = 0u;
#pragma unroll
    for (int i = 0; i < N; ++i) {
        uint32_t x = w[i] & 0x7FFF7FFFu;
        if (finite) {
            if ((x & 0xFFFFu) >= 0x7C00u) x &= 0xFFFF0000u;
            if ((x >> 16) >= 0x7C00u) x &= 0xFFFFu;
        }
        m = __vmaxu2(m, x);
    }
    return max(m & 0xFFFFu, m >> 16);
}
// Exponent e with 2^11 <= v 2^-e < 2^12 for an fp16 magnitude's bits (subnormals: that of the smallest normal), in [-25, 4]:
// times a code, at most 8, the upper end of fp16's normal range, so that smaller scales beside it have the most of it.
__device__ __forceinline__ int exponent_of(uint32_t bits) { return max(1, static_cast<int>(bits >> 10)) - 15 - 11; }
// Two scales times 2^-e, -28 <= e <= 29, in two steps, exact where the result is normal.
struct Unit {
    __half2 a, b;
    __device__ __forceinline__ explicit Unit(int e) {
        const int x = -e / 2, y = -e - x;
        a = __half2half2(__ushort_as_half(static_cast<unsigned short>((x + 15) << 10)));
        b = __half2half2(__ushort_as_half(static_cast<unsigned short>((y + 15) << 10)));
    }
    __device__ __forceinline__ uint32_t of(uint32_t w) const { return h2_bits(__hmul2(__hmul2(bits_h2(w), a), b)); }
};

// ------------------------------------------------------------------ the line
// All tiles of all (sequence, kv head, row tile) items, kItemCost places before each.
struct Line {
    int b, h, ch;                     // the next chunk: sequence, item of it, chunk of that
    int left;                         // chunks of this CTA still to come
    int chunks, len, first;           // of sequence b
};
struct Piece {
    int b, kvh, row0, rows, len, base;
    int tile0, count;                 // first tile of the cache, tiles (0: a sequence without a tree)
    int h, ch, chunks;
};
__device__ __forceinline__ int window_start(const Kv4Attn& p, int end) { return p.window > 0 && end > p.window ? end - p.window : 0; }
__device__ __forceinline__ int length_of(const Kv4Attn& p, int b, bool& bad) {
    const int cap = static_cast<int>(min(p.table ? static_cast<long long>(p.table_stride) * p.page_size : p.page_size, 0x7fffff00LL));
    int len = __ldg(p.lens + b);
    bad = len < 0 || len > cap;
    if (bad) len = len < 0 ? 0 : cap;
    return len < p.q_len ? 0 : len;   // no tree is there
}
template <int KT>
__device__ __forceinline__ int first_tile(const Kv4Attn& p, int len) { return window_start(p, len - p.q_len + 1) / KT; }
template <int KT>
__device__ __forceinline__ int chunks_of(const Kv4Attn& p, int len) { return max(1, (len + KT - 1) / KT - first_tile<KT>(p, len)); }
template <int KT>
__device__ __forceinline__ void load_seq(Line& l, const Kv4Attn& p) {
    bool bad;
    l.len = length_of(p, l.b, bad);
    l.first = first_tile<KT>(p, l.len);
    l.chunks = chunks_of<KT>(p, l.len);
}
template <int KT>
__device__ __forceinline__ bool next_piece(Line& l, const Kv4Attn& p, int items, Piece& pc) {
    if (l.left <= 0) return false;
    const int n = min(l.chunks - l.ch, l.left);
    pc.b = l.b;
    pc.h = l.h;
    pc.ch = l.ch;
    pc.chunks = l.chunks;
    pc.kvh = l.h / p.row_tiles;
    pc.row0 = (l.h - pc.kvh * p.row_tiles) * kRows;
    pc.rows = min(kRows, p.q_len * p.group - pc.row0);
    pc.len = l.len;
    pc.base = l.len - p.q_len;
    pc.tile0 = l.first + l.ch;
    pc.count = l.len > 0 ? n : 0;
    l.left -= n;
    l.ch += n;
    if (l.ch >= l.chunks) {
        l.ch = 0;
        if (++l.h == items) {
            l.h = 0;
            if (++l.b < p.batch && l.left > 0) load_seq<KT>(l, p);
        }
    }
    return true;
}

struct Cut {                          // an item cut over CTAs: its first CTA, their number, the item
    int n, b, h;
};

template <int NG>
__global__ void __launch_bounds__(Shape<NG>::THREADS, 1) kv4_tree_kernel(const Kv4Attn p, Cut* cuts) {
    using F = Shape<NG>;
    constexpr int D = F::D, KT = F::KT;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    uint8_t* const smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    Small<NG>& s = *reinterpret_cast<Small<NG>*>(smem + F::AT_SMALL);
    constexpr int kMeta = F::META;
    volatile int* const gave_up = &s.abort;
    auto token_of = [&](int row) { return static_cast<int>((static_cast<unsigned int>(row) * p.group_magic) >> 21); };   // row / group
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    pdl_launch_dependents();
    if (threadIdx.x == 0) {
        for (int i = 0; i < F::RAW; ++i) {
            mbar_init(s.raw_full + i, 1);
            mbar_init(s.raw_empty + i, 6);
        }
        for (int i = 0; i < F::K_STAGES; ++i) {
            mbar_init(s.k_full + i, 4);
            mbar_init(s.k_empty + i, 1);
        }
        for (int i = 0; i < F::V_STAGES; ++i) mbar_init(s.v_full + i, 4);
        for (int i = 0; i < 2; ++i) mbar_init(s.v_empty + i, 1);
        for (int i = 0; i < F::S_STAGES; ++i) {
            mbar_init(s.s_full + i, 1);
            mbar_init(s.p_full + i, 4);
            mbar_init(s.pv_done + i, 1);
        }
        for (int i = 0; i < kMeta; ++i) mbar_init(s.meta_full + i, 2);
        mbar_init(&s.q_full, F::SOFT);
        mbar_init(&s.done, 1);
        s.abort = 0;
        fence_mbar_init();
    }
    if (warp == F::SOFT + 9) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s.tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tcg::tc_fence_before();
    __syncthreads();
    tcg::tc_fence_after();
    const uint32_t tmem = static_cast<uint32_t>(*reinterpret_cast<volatile int*>(&s.tmem));
    pdl_wait();

    // ---------------------------------------------------------- this CTA's part of the line
    const int items = p.kv_heads * p.row_tiles;
    // Each warp adds the sequences up for itself, 32 at a time: nothing to wait for but their lengths.
    auto width_of = [&](int b) {
        bool bad = false;
        const int n = b < p.batch ? chunks_of<KT>(p, length_of(p, b, bad)) + kItemCost : 0;
        if (bad && blockIdx.x == 0 && warp == 0) record_fault(ALJ_FAULT_BOUNDS);
        return n;
    };
    auto scan = [&](int n) {          // inclusive prefix sums of the lanes' n
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, n, o);
            if (lane >= o) n += up;
        }
        return n;
    };
    int total = 0, mine = 0, incl = 0;                    // the lane's sequence's places, and those up to its end
#pragma unroll 1
    for (int b0 = 0; b0 < p.batch; b0 += 32) {
        incl = scan(mine = width_of(b0 + lane));
        total += __shfl_sync(0xffffffffu, incl, 31);
    }
    total *= items;                   // < 2^31: checked on the host for the longest sequences
    const int ctas = min(static_cast<int>(gridDim.x), (total + kLeast - 1) / kLeast);
    const int share = total / ctas, rem = total - share * ctas;
    auto start_of = [&](int c) { return share * c + min(c, rem); };
    auto cta_at = [&](int x) {
        const int wide = rem * (share + 1);
        return x < wide ? x / (share + 1) : rem + (x - wide) / share;
    };
    if (threadIdx.x == 0) cuts[blockIdx.x].n = 0;
    Line line = {};
    int my_pre = 0;                   // places before the sequence of the first piece
    if (static_cast<int>(blockIdx.x) < ctas) {
        const int x0 = start_of(blockIdx.x), x1 = start_of(blockIdx.x + 1);
        int before = 0;               // line places before the sequences at hand, of one item
#pragma unroll 1
        for (int b0 = 0; b0 < p.batch; b0 += 32) {
            if (p.batch > 32) incl = scan(mine = width_of(b0 + lane));
            const int upto = before + incl, pre = upto - mine;
            const uint32_t here = __ballot_sync(0xffffffffu, mine > 0 && pre * items <= x0 && x0 < upto * items);
            if (here) {
                line.b = b0 + __ffs(here) - 1;
                my_pre = __shfl_sync(0xffffffffu, pre, __ffs(here) - 1);
                break;
            }
            before = __shfl_sync(0xffffffffu, upto, 31);
        }
        load_seq<KT>(line, p);
        const int width = line.chunks + kItemCost, rest = x0 - my_pre * items;
        line.h = rest / width;
        const int at = rest - line.h * width;
        line.ch = max(0, at - kItemCost);
        // the chunks between x0 and x1: places less what of the items' costs lies there
        Line l = line;
        int x = x0 - at + kItemCost + line.ch, n = 0;   // place of the next chunk
        while (x < x1) {
            const int m = min(l.chunks - l.ch, x1 - x);
            n += m;
            x += l.chunks - l.ch + kItemCost;
            l.ch = 0;
            if (++l.h == items) {
                l.h = 0;
                if (++l.b == p.batch) break;
                load_seq<KT>(l, p);
            }
        }
        line.left = n;
    }
    const uint32_t at_q = smem_u32(smem), at_k = at_q + F::AT_K, at_v = at_q + F::AT_V, at_raw = at_q + F::AT_RAW;
    Piece pc;
    bool ok = true;

    if (warp < F::SOFT) {
        // ------------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(F::R_SOFT));
        const int stream = warp >> 2, row = (warp & 3) * 32 + lane, thread = threadIdx.x;
        const uint32_t tq = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
        const float inv_cap = p.soft_cap > 0.0f ? 1.0f / p.soft_cap : 0.0f;
        const float size = fabsf(p.scale) * (p.soft_cap > 0.0f ? 1.0f : kLog2e);
        auto sync = [&] { named_bar(1, 32 * F::SOFT); };
        int tiles = 0;                // of this CTA before the piece
        int pre = my_pre, seq = line.b;
        while (next_piece<KT>(line, p, items, pc)) {
            if (pc.b != seq) {        // the line's places before sequence pc.b
                for (; seq < pc.b; ++seq) {
                    bool bad;
                    pre += chunks_of<KT>(p, length_of(p, seq, bad)) + kItemCost;
                }
            }
            const bool whole = pc.ch == 0 && (pc.count == pc.chunks || pc.count == 0);
            const int line0 = pre * items + pc.h * (pc.chunks + kItemCost) + kItemCost;
            // -------------------------------------------------- the rows' masks and Q
            // Q's rows come to their places in shared memory as they are, while the masks are made: a lane 16 bytes of a row,
            // kPer rows a pass of a warp
            constexpr int kChunks = D / 8, kPer = 32 / kChunks, kPasses = kRows / kPer / F::SOFT;
            const int j = lane % kChunks;
            auto place_of = [&](int k, int& r) {
                r = (k * F::SOFT + warp) * kPer + lane / kChunks;
                return at_q + (j >> 3) * (kRows * 128) + r * 128 + (((j & 7) ^ (r & 7)) << 4);
            };
            constexpr int kPar = kKv4MaxNodes / (32 * F::SOFT);      // nodes a thread brings
            int par[kPar];
#pragma unroll
            for (int k = 0; k < kPar; ++k) {
                const int i = k * (32 * F::SOFT) + thread;
                par[k] = i < p.q_len ? tree_parent(p.parents + static_cast<long long>(pc.b) * p.parents_stride, i) : 0;
            }
            if (pc.count > 0) {
                const bool wide = ((reinterpret_cast<uintptr_t>(p.q) | static_cast<uintptr_t>(p.q_stride * 2)) & 15) == 0;
#pragma unroll 2
                for (int k = 0; k < kPasses; ++k) {
                    int r;
                    const uint32_t place = place_of(k, r);
                    const int i = min(pc.row0 + r, p.q_len * p.group - 1), t = token_of(i), hd = i - t * p.group;
                    const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(p.q) + (static_cast<long long>(pc.b) * p.q_len + t) * p.q_stride +
                                             static_cast<long long>(pc.kvh * p.group + hd) * D + 8 * j;
                    if (wide) {
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(place), "l"(q), "r"(r < pc.rows ? 16 : 0) : "memory");
                    } else {
                        const unsigned short* h = reinterpret_cast<const unsigned short*>(q);
                        sts128(place, r < pc.rows ? make_uint4(h[0] | h[1] << 16, h[2] | h[3] << 16, h[4] | h[5] << 16, h[6] | h[7] << 16)
                                                  : make_uint4(0u, 0u, 0u, 0u));
                    }
                }
            }
#pragma unroll
            for (int k = 0; k < kPar; ++k) s.par[k * (32 * F::SOFT) + thread] = static_cast<short>(par[k]);
            sync();
            const int node = token_of(pc.row0 + row);
            int depth = 0;
            if (pc.count > 0 && row < pc.rows) {
                if (stream == 0) {
#pragma unroll 1
                    for (int i = 0; i < kKv4TreeWords; ++i) s.see[i][row] = 0u;
                }
                int t = node;
#pragma unroll 1
                for (; t >= 0; t = s.par[t], ++depth)
                    if (stream == 0 && (p.window == 0 || depth < p.window)) s.see[t >> 5][row] |= 1u << (t & 31);
                if (t != -1) depth = 0;                               // its bits are not looked at
            }
            const bool alive = depth > 0;
            const int row_lo = window_start(p, pc.base + depth);          // first position the row sees
            const int all_lo = window_start(p, pc.len);
            if (pc.count > 0) {
                asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
                for (int k = 0; k < kPasses; ++k) {               // each lane what it brought
                    int r;
                    const uint32_t place = place_of(k, r);
                    uint32_t w[4];
                    lds_words<4>(place, w);
                    float v[8], big = 0.0f;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        v[2 * i] = __uint_as_float(w[i] << 16);
                        v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
                    }
#pragma unroll
                    for (int i = 0; i < 8; ++i) big = fmaxf(big, fabsf(v[i]));
#pragma unroll
                    for (int o = 1; o < kChunks; o <<= 1) big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, o));
                    // the row times 2^f: its largest in [2^14, 2^15), where both 2^f and 2^-f are normal
                    const int f = big > 0.0f ? max(-100, min(126, 14 - (static_cast<int>((__float_as_uint(big) >> 23) & 255) - 127))) : 0;
                    const float up = p.scale < 0.0f ? -pow2i(f) : pow2i(f);
                    if (j == 0) s.fac[r] = size * pow2i(-f);
                    uint32_t out[4];                  // as decode8 orders the dims of a chunk
#pragma unroll
                    for (int i = 0; i < 4; ++i) out[i] = h2_bits(__floats2half2_rn(v[i] * up, v[i + 4] * up));
                    sts128(place, make_uint4(out[0], out[1], out[2], out[3]));
                }
            }
            fence_proxy_shared();
            __syncwarp();
            if (lane == 0 && pc.count > 0) mbar_arrive(&s.q_full);
            sync();                                               // masks and factors
            const float fac = pc.count > 0 ? s.fac[row] : 0.0f;
            float M = kNone, l = 0.0f;
            int E = -100, nan_groups = 0;
            const bool warp_lives = (warp & 3) * 32 < pc.rows;
            // bits of the positions from at on that the row sees
            auto visible = [&](int at) {
                uint32_t bits = 0u;
                const int rel = at - pc.base;
                if (rel < 0 && alive) {
                    bits = rel <= -32 ? 0xFFFFFFFFu : (1u << -rel) - 1u;
                    const int skip = row_lo - at;
                    if (skip > 0) bits = skip >= 32 ? 0u : bits & (0xFFFFFFFFu << skip);
                }
                if (rel > -32 && rel < p.q_len && alive) {
                    const int i = max(rel, 0) >> 5, sh = rel & 31;
                    const uint32_t a = s.see[i][row], b = i + 1 < kKv4TreeWords ? s.see[i + 1][row] : 0u;
                    bits |= rel < 0 ? a << -rel : __funnelshift_r(a, b, sh);
                }
                return bits;
            };
            // -------------------------------------------------- its tiles
            int last = -1;            // the stream's last tile
            for (int tile = tiles + (F::STREAMS == 2 ? (tiles ^ stream) & 1 : 0); tile < tiles + pc.count; last = tile, tile += F::STREAMS) {
                const int buf = tile % F::S_STAGES, use = tile / F::S_STAGES;
                const int meta = tile & (kMeta - 1), pos = (pc.tile0 + tile - tiles) * KT;
                const uint32_t ts = tq + buf * KT, to = tq + F::O_COL + (F::STREAMS == 2 ? stream * D : 0);
                ok = ok && warp_wait(s.s_full + buf, use & 1, gave_up);
                ok = ok && warp_wait(s.meta_full + meta, (tile / kMeta) & 1, gave_up);
                if (ok && warp_lives) {
                    tcg::tc_fence_after();
                    const bool edge = pos < all_lo || pos + KT > pc.base;
                    // O summed up so far times g
                    auto rescale = [&](float g) {
                        if (last < 0) return;
                        ok = ok && warp_wait(s.pv_done + last % F::S_STAGES, (last / F::S_STAGES) & 1, gave_up);
                        tcg::tc_fence_after();
                        tcg::tmem_wait_st();                          // an earlier call's stores: loads do not wait for them
#pragma unroll 1
                        for (int c = 0; c < 4 * NG; ++c) {
                            uint32_t v[8];
                            tmem_ld8(to + 8 * c, v);
#pragma unroll
                            for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * g);
                            tmem_st8(to + 8 * c, v);
                        }
                    };
                    const int e_new = s.e_top[meta];
                    if (e_new > E + kSlack) {                         // the same for the whole warp
                        rescale(pow2i(max(E - e_new, -126)));
                        E = e_new;
                    }
                    int c = 0;
                    if (!edge && p.soft_cap == 0.0f) {
                        // Without masks and without the maximum: P may pass 1, and the sum of 32 says whether it stays in
                        // fp16's range.  Where it does not, or M is so large that its rounding counts, the rest of the tile
                        // goes the long way.  16 columns are on their way while 16 are used.
                        uint32_t v[16], w[16];
                        tmem_ask16(ts, v);
#pragma unroll 1
                        for (; c < KT / 32; ++c) {
                            const int sh = kBias + s.ev[meta][c] - E;
                            const float fc = fac * s.k_unit[meta][c], at = static_cast<float>(sh) - M;
                            float sums[4] = {};
                            uint32_t out[16];
                            auto half = [&](const uint32_t (&x)[16], int to) {
#pragma unroll
                                for (int k = 0; k < 8; ++k) {
                                    const float a = ex2(fmaf(__uint_as_float(x[2 * k]), fc, at)), b = ex2(fmaf(__uint_as_float(x[2 * k + 1]), fc, at));
                                    sums[2 * (k & 1)] += a;
                                    sums[2 * (k & 1) + 1] += b;
                                    out[to + k] = h2_bits(__floats2half2_rn(a, b));
                                }
                            };
                            tmem_have(v);
                            tmem_ask16(ts + 32 * c + 16, w);
                            half(v, 0);
                            tmem_have(w);
                            if (c + 1 < KT / 32) tmem_ask16(ts + 32 * c + 32, v);
                            half(w, 8);
                            const float sum = (sums[0] + sums[1]) + (sums[2] + sums[3]);
                            if (__any_sync(0xffffffffu, sum > kMostSum || fabsf(M) > kMostM)) break;
                            l = fmaf(sum, pow2i(-sh), l);
                            tmem_st16(ts + 16 * c, out);              // columns that this lane has read
                        }
                        tmem_have(v);
                    }
#pragma unroll 1
                    for (; c < KT / 32; ++c) {
                        const uint32_t bits = edge ? visible(pos + 32 * c) : 0xFFFFFFFFu;
                        const int sh = kBias + s.ev[meta][c] - E;
                        float fc = fac * s.k_unit[meta][c];
                        if (p.soft_cap > 0.0f) {
#pragma unroll 1
                            for (int b = 0; b < 4; ++b) {             // S becomes the capped score
                                uint32_t v[8];
                                tmem_ld8(ts + 32 * c + 8 * b, v);
#pragma unroll
                                for (int k = 0; k < 8; ++k) v[k] = __float_as_uint(tanhf(__uint_as_float(v[k]) * fc * inv_cap) * (p.soft_cap * kLog2e));
                                tmem_st8(ts + 32 * c + 8 * b, v);
                            }
                            tcg::tmem_wait_st();
                            fc = 1.0f;
                        }
                        uint32_t v[32];
                        tmem_ld32(ts + 32 * c, v);
                        float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
                        for (int k = 0; k < 32; ++k) {
                            const float y = (bits >> k) & 1u ? __uint_as_float(v[k]) * fc : -INFINITY;
                            m[k & 1] = fmaxf(m[k & 1], y);
                            v[k] = __float_as_uint(y);
                        }
                        const float mx = fmaxf(m[0], m[1]);
                        if (__any_sync(0xffffffffu, mx > M + kLazy)) {
                            // M becomes the next integer above the score, so that what is there already, the P of the chunks
                            // before c too, is scaled by a power of two
                            const float now = mx > M + kLazy ? ceilf(mx) : M, f = ex2(M - now);
                            M = now;
                            l *= f;
                            rescale(f);
                            if (c > 0) tcg::tmem_wait_st();           // P as it was stored or scaled last
                            const __half2 f2 = __float2half2_rn(f);
#pragma unroll 1
                            for (int b = 0; b < 2 * c; ++b) {
                                uint32_t x[8];
                                tmem_ld8(ts + 8 * b, x);
#pragma unroll
                                for (int k = 0; k < 8; ++k) x[k] = h2_bits(__hmul2(bits_h2(x[k]), f2));
                                tmem_st8(ts + 8 * b, x);
                            }
                        }
                        const float at = static_cast<float>(sh) - M;
                        float sum[2] = {};
                        uint32_t out[16];
#pragma unroll
                        for (int k = 0; k < 16; ++k) {
                            const float a = ex2(__uint_as_float(v[2 * k]) + at), b = ex2(__uint_as_float(v[2 * k + 1]) + at);
                            sum[k & 1] += a + b;
                            out[k] = h2_bits(__floats2half2_rn(a, b));
                        }
                        l = fmaf(sum[0] + sum[1], pow2i(-sh), l);
                        tmem_st16(ts + 16 * c, out);
                    }
                    if (s.nan_any[meta]) {
                        for (int k = 0; k < KT; ++k) {
                            const int g = s.nan[meta][k];
                            if (g && (edge ? (visible(pos + (k & ~31)) >> (k & 31)) & 1u : alive)) nan_groups |= g;
                        }
                    }
                    tcg::tmem_wait_st();
                }
                tcg::tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s.p_full + buf);
            }
            // -------------------------------------------------- the streams' results, and the rows' outputs
            // (The stream's own last products: S of that tile has been seen, so the use of its buffer before is behind us.)
            if (last >= 0) ok = ok && warp_wait(s.pv_done + last % F::S_STAGES, (last / F::S_STAGES) & 1, gave_up);
            s.ml[stream][row][0] = M;
            s.ml[stream][row][1] = l;
            s.er[stream][row] = static_cast<short>(E);
            s.row_nan[stream][row] = static_cast<uint8_t>(nan_groups);
            sync();
            tcg::tc_fence_after();
            // which streams had a tile
            const bool has0 = pc.count > 0 && (F::STREAMS == 1 || pc.count > 1 || (tiles & 1) == 0);
            const bool has1 = F::STREAMS == 2 && (pc.count > 1 || (pc.count == 1 && (tiles & 1) == 1));
            tiles += pc.count;
            float w0 = 0.0f, w1 = 0.0f, L = 0.0f, top = kNone;
            int gone = 0;
            if (alive && pc.count > 0) {
                const float m0 = has0 ? s.ml[0][row][0] : kNone, m1 = has1 ? s.ml[1][row][0] : kNone;
                top = fmaxf(m0, m1);
                w0 = has0 ? ex2(m0 - top) : 0.0f;
                w1 = has1 ? ex2(m1 - top) : 0.0f;
                L = (has0 ? s.ml[0][row][1] * w0 : 0.0f) + (has1 ? s.ml[1][row][1] * w1 : 0.0f);
                if (has0) w0 *= pow2i(max(-126, s.er[0][row] - kBias));
                if (has1) w1 *= pow2i(max(-126, s.er[1][row] - kBias));
                gone = (has0 ? s.row_nan[0][row] : 0) | (has1 ? s.row_nan[1][row] : 0);
            }
            int slot = 0;
            if (!whole) {
                const int cta0 = cta_at(line0), cta1 = cta_at(line0 + pc.chunks - 1);
                slot = static_cast<int>(blockIdx.x) * 2 + (static_cast<int>(blockIdx.x) == cta0 ? 1 : 0);
                if (static_cast<int>(blockIdx.x) == cta0 && thread == 0) cuts[cta0] = Cut{cta1 - cta0 + 1, pc.b, pc.h};
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            constexpr int kCols = D / F::STREAMS;                     // columns of a warp
            if (ok && warp_lives) {
                // kCut columns of the warp's rows at a time through its share of Q's place, so that a row's are written side by
                // side; 16-byte pieces are swizzled by the row
                constexpr int kCut = D == 64 ? 16 : 32, kPieces = kCut / 4;
                const uint32_t stage = at_q + warp * (F::Q / F::SOFT);
                float* const part = p.part + static_cast<long long>(slot) * (kRows * (D + 2));
#pragma unroll 1
                for (int d0 = stream * kCols; d0 < (stream + 1) * kCols; d0 += kCut) {
                    const bool nan = (gone >> (d0 >> 5)) & 1;
#pragma unroll 1
                    for (int d = 0; d < kCut; d += 8) {
                        uint32_t v[8], w[8];
                        tmem_ld8x2(tq + F::O_COL + d0 + d, tq + F::O_COL + (F::STREAMS - 1) * D + d0 + d, v, w);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {             // what has not been written may be anything
                            float o = has0 ? __uint_as_float(v[k]) * w0 : 0.0f;
                            if (has1) o = fmaf(__uint_as_float(w[k]), w1, o);
                            v[k] = __float_as_uint(!alive || L == 0.0f ? 0.0f : nan ? NAN : whole ? o * inv : o);   // what sees nothing is zero
                        }
#pragma unroll
                        for (int k = 0; k < 2; ++k)
                            sts128(stage + lane * (kCut * 4) + (((d / 4 + k) ^ (lane & (kPieces - 1))) << 4),
                                   make_uint4(v[4 * k], v[4 * k + 1], v[4 * k + 2], v[4 * k + 3]));
                    }
                    __syncwarp();
#pragma unroll 1
                    for (int n = lane; n < 32 * kPieces; n += 32) {
                        const int r = n / kPieces, piece = n % kPieces, at = (warp & 3) * 32 + r, d = d0 + 4 * piece;
                        uint32_t x[4];
                        lds_words<4>(stage + r * (kCut * 4) + ((piece ^ (r & (kPieces - 1))) << 4), x);
                        if (at >= pc.rows) continue;
                        if (whole) {
                            const int t = token_of(pc.row0 + at), hd = pc.row0 + at - t * p.group;
                            const __nv_bfloat162 a = __floats2bfloat162_rn(__uint_as_float(x[0]), __uint_as_float(x[1]));
                            const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(x[2]), __uint_as_float(x[3]));
                            *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p.out) +
                                (((static_cast<long long>(pc.b) * p.q_len + t) * p.kv_heads + pc.kvh) * p.group + hd) * D + d) =
                                make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
                        } else {
                            *reinterpret_cast<uint4*>(part + at * D + d) = make_uint4(x[0], x[1], x[2], x[3]);
                        }
                    }
                    __syncwarp();
                }
                if (!whole && stream == 0 && row < pc.rows) {
                    float* const ml = p.part + static_cast<long long>(slot) * (kRows * (D + 2)) + kRows * D + row * 2;
                    ml[0] = top;
                    ml[1] = L;
                }
            }
            tcg::tc_fence_before();
            sync();                                               // tensor memory and the tables are read
        }
    } else if (warp < F::SOFT + 8) {
        // ------------------------------------------------------ K, then V, to fp16: a warpgroup every second tile
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::R_DECODE));
        const int turn = (warp - F::SOFT) >> 2;
        constexpr int GW = KT == 128 ? NG : NG / 2;               // K: groups of a warp
        const int kw = warp & 3, span = KT == 128 ? kw : kw & 1, half = KT == 128 ? 0 : kw >> 1;
        const int c = lane & 3, pos_in = (lane >> 3) + (lane & 4);
        const uint32_t k_src = (32 * span + pos_in) * (D / 2) + c * (4 * NG) + half * (4 * GW);
        const uint32_t k_sc = F::K_SC + (32 * span + pos_in) * (2 * NG) + half * (2 * GW);
        const uint32_t k_dst = (half * GW >> 1) * (KT * 128) + (32 * span + pos_in) * 128 + ((c ^ pos_in) << 4);
        // V: a thread has 8 positions, block j of 64, and a word (8 codes: 4 dims of groups g and g + 1) a pass.  Lanes read
        // different words, those that would meet on a bank the other position of a pair first; eight lanes that store
        // together have eight different j, so that their 16-byte pieces lie in different banks under the swizzle.
        constexpr int kPasses = NG == 2 ? 1 : 2;
        const int vw = warp & 3;
        const int word = NG == 8   ? (lane & 3) | (lane & 24) >> 1 | (lane & 4) << 2
                         : NG == 4 ? lane & 15
                                   : lane & 7;
        const int part = KT == 128 ? lane >> 4 : 0, flip = NG == 8 ? 0 : lane >> 4;
        const int hw0 = 2 * word;
        int tile = 0;
        while (next_piece<KT>(line, p, items, pc)) {
            for (int i = 0; i < pc.count; ++i, ++tile) {
                if ((tile & 1) != turn) continue;
                const int slot = tile % F::RAW, ks = tile % F::K_STAGES, vs = tile % F::V_STAGES;
                // the exponents are found after the codes have arrived
                ok = ok && warp_wait(s.meta_full + (tile & (kMeta - 1)), (tile / kMeta) & 1, gave_up);
                if (tile >= F::K_STAGES) ok = ok && warp_wait(s.k_empty + ks, (tile / F::K_STAGES - 1) & 1, gave_up);
                if (!ok) break;
                const uint32_t raw = at_raw + slot * F::RAW_BYTES;
                const uint32_t k_codes = raw + k_src, k_scales = raw + k_sc, k_to0 = at_k + ks * F::KHAT + k_dst, k_to1 = k_to0 ^ 64u;
#pragma unroll 2
                for (int it = 0; it < 4; ++it) {
                    uint32_t w[GW], d[GW / 2];
                    lds_words<GW>(k_codes + it * (4 * D), w);
                    lds_words<GW / 2>(k_scales + it * (16 * NG), d);
#pragma unroll
                    for (int g = 0; g < GW; ++g) {                // 16-byte piece 4 g + c of the row
                        uint32_t out[4];
                        decode8(w[g], bits_h2(__byte_perm(d[g / 2], 0u, g & 1 ? 0x3232 : 0x1010)), out);
                        sts128((g & 1 ? k_to1 : k_to0) + (g >> 1) * (KT * 128) + it * 1024, make_uint4(out[0], out[1], out[2], out[3]));
                    }
                }
                fence_proxy_shared();
                __syncwarp();
                if (lane == 0) mbar_arrive(s.k_full + ks);
                // A barrier for every second tile also where V has one place: a wait by parity has to see each phase of its
                // barrier in turn, and the other warpgroup waits for the others.
                if (const int u = tile - F::V_STAGES; u >= 0) ok = ok && warp_wait(s.v_empty + (u & 1), (u >> 1) & 1, gave_up);
                if (!ok) break;
                const uint32_t to = at_v + vs * F::VHAT + part * (D * 128);
#pragma unroll 1
                for (int n = 0; n < kPasses; ++n) {
                    const int j = (lane + (NG == 2 ? vw + ((lane & 8) >> 1) : 2 * vw + n)) & 7, pos = 64 * part + 8 * j;
                    const uint32_t blk = raw + F::V_CODES + pos * (D / 2) + 4 * word;
                    const int q = pos >> 2, turned = (q >> 3) & 1;
                    const uint32_t sc = raw + F::V_SC + ((word % (NG / 2)) * KT + 4 * (q ^ turned)) * 4;
                    uint32_t code[8], d[2][4];                    // code k: position k ^ flip
                    lds_words<4>(sc, d[0]);
                    lds_words<4>(turned ? sc - 16 : sc + 16, d[1]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) code[k] = lds_word(blk + (k & 6) * (D / 2) + (k & 1 ? (flip ^ 1) : flip) * (D / 2));
#pragma unroll 1
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t pick_d = x ? 0x7632u : 0x5410u, pick = flip ? (x ? 0x3276u : 0x1054u) : pick_d;
                        const int hw = hw0 + x, dim = 32 * (hw % NG) + 4 * (hw / NG);
                        const uint32_t at = to + dim * 128 + ((j ^ (dim & 4)) << 4);
                        uint32_t out[4][4];                       // [dim][pair of positions]
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            uint32_t v[4];
                            decode8(__byte_perm(code[2 * k], code[2 * k + 1], pick), bits_h2(__byte_perm(d[k >> 1][2 * (k & 1)], d[k >> 1][2 * (k & 1) + 1], pick_d)), v);
#pragma unroll
                            for (int m = 0; m < 4; ++m) out[m][k] = v[m];
                        }
#pragma unroll
                        for (int m = 0; m < 4; ++m)
                            sts128((at ^ (m << 4)) + m * 128, make_uint4(out[m][0], out[m][1], out[m][2], out[m][3]));
                    }
                }
                fence_proxy_shared();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(s.v_full + vs);
                    mbar_arrive(s.raw_empty + slot);
                }
            }
            if (!ok) break;
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(F::R_REST));
    if (warp == F::SOFT + 8) {
        // ------------------------------------------------------ codes and scales from the cache
        // Lane 4 n + k sees to section k of the n-th 16 positions of a tile.  Page ids come through shared memory, kPages at a
        // time: a load from the table for every tile would take as long as the tile's products.
        int tile = 0, seq = -1;
        const int blk = lane >> 2, k = lane & 3;
        const int row = k < 2 ? D / 2 : 2 * NG;                       // bytes of a position in the section
        const uint32_t to = at_raw + (k == 0 ? 0 : k == 1 ? F::V_CODES : k == 2 ? F::K_SC : F::V_SC) + 16 * blk * row;
        const long long section = static_cast<long long>(p.page_size) * (k < 2 ? k * (D / 2) : D + (k - 2) * (2 * NG));
        const long long block = kv4_block_bytes(p.page_size, D);
        while (next_piece<KT>(line, p, items, pc)) {
            const int lo = window_start(p, pc.base + 1), kept = lo / p.page_size;   // pages before `kept` may have been given back
            int pos = pc.tile0 * KT + 16 * blk, pi = pos / p.page_size, off = pos - pi * p.page_size;
            int first = 0, last = -1;                                 // pages at hand
            const uint8_t* const head = p.cache + static_cast<long long>(pc.kvh) * block + section;
#pragma unroll 1
            for (int i = 0; i < pc.count; ++i, ++tile) {
                const int slot = tile % F::RAW, pos0 = (pc.tile0 + i) * KT;
                const bool there = 16 * blk < KT && pos < pc.len;
                if (__any_sync(0xffffffffu, there && pi > last)) {
                    first = __shfl_sync(0xffffffffu, pi, 0);
                    last = first + kPages - 1;
                    const int end = (pc.len - 1) / p.page_size;
                    __syncwarp();
#pragma unroll 1
                    for (int n = lane; n < kPages && first + n <= end; n += 32) {
                        const int page = p.table ? __ldg(p.table + static_cast<long long>(pc.b) * p.table_stride + first + n) : pc.b;
                        const bool bad = page < 0 || page >= p.pages;
                        if (bad && first + n >= kept) record_fault(ALJ_FAULT_BOUNDS);
                        s.pages[n] = bad ? -1 : page;
                    }
                    __syncwarp();
                }
                const int page = there ? s.pages[pi - first] : -1;
                const bool has = page >= 0;
                const uint32_t any = __ballot_sync(0xffffffffu, has);
                uint32_t bits = has ? 0xFFFFu : 0u;                   // valid ones of the 16 positions
                if (pos0 < lo || pos0 + KT > pc.base) {               // at the window's edge, or with the tree's nodes
                    if (seq != pc.b) {                                // which of them are there: those whose ancestors all are
                        seq = pc.b;
                        __syncwarp();
#pragma unroll 1
                        for (int t = lane; t < p.q_len; t += 32)
                            s.par_p[t] = static_cast<short>(tree_parent(p.parents + static_cast<long long>(pc.b) * p.parents_stride, t));
                        __syncwarp();
#pragma unroll 1
                        for (int w = 0; w < kKv4TreeWords; ++w) {
                            int t = 32 * w + lane < p.q_len ? 32 * w + lane : -2;
                            while (t >= 0) t = s.par_p[t];
                            const uint32_t nodes = __ballot_sync(0xffffffffu, t == -1);
                            if (lane == 0) s.node_ok[w] = nodes;
                        }
                        __syncwarp();
                    }
#pragma unroll 1
                    for (int n = 0; n < 16; ++n) {
                        const int node = pos + n - pc.base;
                        const bool v = pos + n >= lo && (node < 0 || (node < p.q_len && ((s.node_ok[node >> 5] >> (node & 31)) & 1u)));
                        if (!v) bits &= ~(1u << n);
                    }
                }
                bits |= __shfl_down_sync(0xffffffffu, bits, 4) << 16;
                // the blocks that share a page follow one another there: one copy of each section for all of them
                const uint8_t* const src = head + static_cast<long long>(page) * p.kv_heads * block + static_cast<long long>(off) * row;
                const int run = min(min(KT / 16 - blk, (p.page_size - off) >> 4), (pc.len - pos + 15) >> 4);
                if (tile >= F::RAW) ok = ok && warp_wait(s.raw_empty + slot, (tile / F::RAW - 1) & 1, gave_up);
                if (!ok) break;
                if ((lane & 7) == 0) s.valid[slot][lane >> 3] = bits;
                __syncwarp();
                if (lane == 0) mbar_arrive_expect_tx(s.raw_full + slot, (__popc(any) >> 2) * F::BLOCK_BYTES);
                __syncwarp();
                if (has && (blk == 0 || off == 0)) bulk_to(to + slot * F::RAW_BYTES, src, 16 * run * row, s.raw_full + slot);
                pos += KT;
                off += KT;
                while (off >= p.page_size) {
                    off -= p.page_size;
                    ++pi;
                }
            }
            if (!ok) break;
        }
        if (!ok)                          // the copies under way end before the CTA does
            for (int t = max(0, tile - F::RAW); t < tile; ++t) mbar_wait(s.raw_full + t % F::RAW, (t / F::RAW) & 1);
    } else if (warp >= F::SOFT + 10) {
        // ------------------------------------------------------ exponents of a tile's scales, which become d 2^-e: one warp
        // K's, one V's
        const bool is_v = warp == F::SOFT + 11;
        int tile = 0;
        while (next_piece<KT>(line, p, items, pc)) {
            for (int i = 0; i < pc.count; ++i, ++tile) {
                const int slot = tile % F::RAW, meta = tile & (kMeta - 1);
                ok = ok && warp_wait(s.raw_full + slot, (tile / F::RAW) & 1, gave_up);
                if (!ok) break;
                int e_top = -100;
                bool any = false;
                uint32_t w[KT / 32][NG / 2];                      // 32 positions, a lane each
                const uint32_t at = at_raw + slot * F::RAW_BYTES + (is_v ? F::V_SC : F::K_SC);
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) lds_words<NG / 2>(at + (32 * c + lane) * (2 * NG), w[c]);
                __syncwarp();
#pragma unroll
                for (int c = 0; c < KT / 32; ++c) {
                    const bool mine = (s.valid[slot][c] >> lane) & 1u;
                    uint32_t top = __reduce_max_sync(0xffffffffu, mine ? top_of(w[c], false) : 0u);
                    if (top >= 0x7C00u) {
                        top = __reduce_max_sync(0xffffffffu, mine ? top_of(w[c], true) : 0u);
                        if (is_v) {                               // NaN groups of V count as zero, and their rows are marked
                            if (!any)
                                for (int k = lane; k < KT; k += 32) s.nan[meta][k] = 0;
                            any = true;
                            int bad = 0;
#pragma unroll
                            for (int g = 0; g < NG; ++g)
                                if (((w[c][g / 2] >> (16 * (g & 1))) & 0x7FFFu) >= 0x7C00u) {
                                    bad |= 1 << g;
                                    w[c][g / 2] &= g & 1 ? 0x0000FFFFu : 0xFFFF0000u;
                                }
                            __syncwarp();
                            if (mine) s.nan[meta][32 * c + lane] = static_cast<uint8_t>(bad);
                        }
                    }
                    const int e = exponent_of(top);
                    const Unit unit(e);
#pragma unroll
                    for (int k = 0; k < NG / 2; ++k) w[c][k] = mine ? unit.of(w[c][k]) : 0u;
                    if (is_v) {
                        // word by word, so that a thread finds 8 positions side by side; their 16-byte halves trade places
                        // in every second 32 positions, or eight threads' would meet on four banks
                        const int q = 8 * c + (lane >> 2), place = 4 * (q ^ ((q >> 3) & 1)) + (lane & 3);
#pragma unroll
                        for (int k = 0; k < NG / 2; ++k) sts_words<1>(at + (k * KT + place) * 4, reinterpret_cast<const uint32_t(&)[1]>(w[c][k]));
                    } else {
                        sts_words<NG / 2>(at + (32 * c + lane) * (2 * NG), w[c]);
                    }
                    e_top = max(e_top, e);
                    if (lane == 0) {
                        if (is_v) s.ev[meta][c] = e;
                        else s.k_unit[meta][c] = pow2i(e);
                    }
                }
                if (is_v && lane == 0) {
                    s.e_top[meta] = e_top;
                    s.nan_any[meta] = any;
                }
                fence_proxy_shared();                             // the slot's next writer is a bulk copy
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(s.meta_full + meta);
                    mbar_arrive(s.raw_empty + slot);
                }
            }
            if (!ok) break;
        }
    } else {
        // ------------------------------------------------------ MMA issue
        constexpr uint32_t kS = tcg::idesc_f16(KT), kO = tcg::idesc_f16(D);
        const uint32_t one = elect_one();
        // descriptors count 16-byte units: 2 for 16 values of K, an atom of 64 for its rows' 128 bytes
        const uint64_t q_desc = tcg::sdesc(at_q), k_desc = tcg::sdesc(at_k), v_desc = tcg::sdesc(at_v);
        int tile = 0, pieces = 0;
        while (ok && next_piece<KT>(line, p, items, pc)) {
            if (pc.count == 0) continue;
            ok = ok && warp_wait(&s.q_full, pieces & 1, gave_up);
            ++pieces;
#pragma unroll 1
            for (int i = -F::S_STAGES; ok && i < pc.count; ++i) {     // O of tile i, then S of tile i + S_STAGES
                if (i >= 0) {
                    const int t = tile + i, vs = t % F::V_STAGES, buf = t % F::S_STAGES;
                    ok = ok && warp_wait(s.v_full + vs, (t / F::V_STAGES) & 1, gave_up);
                    ok = ok && warp_wait(s.p_full + buf, (t / F::S_STAGES) & 1, gave_up);
                    if (!ok) break;
                    tcg::tc_fence_after();
                    const uint32_t to = tmem + F::O_COL + (F::STREAMS == 2 ? (t & 1) * D : 0);
                    const uint64_t v = v_desc + vs * (F::VHAT >> 4);
#pragma unroll
                    for (int h = 0; h < KT / 64; ++h)
                        mma64_ts(to, tmem + buf * KT + 32 * h, v + h * (D * 8), kO, h > 0 || i >= F::STREAMS, one);
                    commit2(s.v_empty + (t & 1), s.pv_done + buf, one);
                }
                if (i + F::S_STAGES < pc.count) {
                    const int t = tile + i + F::S_STAGES, ks = t % F::K_STAGES, buf = t % F::S_STAGES;
                    ok = ok && warp_wait(s.k_full + ks, (t / F::K_STAGES) & 1, gave_up);
                    if (!ok) break;
                    tcg::tc_fence_after();
                    const uint64_t k_at = k_desc + ks * (F::KHAT >> 4);
#pragma unroll
                    for (int h = 0; h < D / 64; ++h)
                        mma64_ss(tmem + buf * KT, q_desc + h * (kRows * 8), k_at + h * (KT * 8), kS, h > 0, one);
                    commit2(s.k_empty + ks, s.s_full + buf, one);
                }
            }
            tile += pc.count;
        }
        if (one) {
            tcg::tc_commit(&s.done);      // every MMA issued has completed before tensor memory is released
            mbar_wait(&s.done, 0);
        }
        __syncwarp();
    }
    }
    tcg::tc_fence_before();
    __syncthreads();
    if (warp == F::SOFT + 9) {
        tcg::tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// Items cut over CTAs: kJoinRows rows of one item at a time are joined by a block, in CTA order.  Every block lists the items
// that were cut, so that the grid is no larger than is resident at once; parts are asked for kJoinParts at a time.  What it
// waits for is memory.  1 x 4096 with 64 nodes, 24 ragged sequences and 2 x 65536, us: a block for each CTA and 8 rows
// 27.7, 114.4, 379; 8 rows here 27.1, 114.0, 376; 4 rows 26.2, 115.1, 377; 4 rows and 6 blocks an SM 27.4, 115.7, 378;
// 8 rows and 3 blocks 27.2, 117.5, 384.
constexpr int kJoinRows = 4, kJoinParts = 4, kJoinBlocks = 4;   // blocks an SM
template <int D>
__global__ void __launch_bounds__(256, kJoinBlocks) kv4_tree_join_kernel(const Kv4Attn p, const Cut* cuts, int ctas, unsigned int* fault_word) {
    extern __shared__ int4 s_cut[];   // [ctas] first CTA, CTAs, sequence, item
    __shared__ int s_warp[8];
    pdl_launch_dependents();
    pdl_wait();
    if (blockIdx.x == 0 && threadIdx.x == 0 && *static_cast<volatile unsigned int*>(&g_fault_word) != 0u)
        atomicOr(fault_word, atomicExch(&g_fault_word, 0u));   // what the attention recorded, to the library's word
    int count = 0;                    // listed in the order of the CTAs: all blocks have to number them alike
    for (int c0 = 0; c0 < ctas; c0 += 256) {
        const int c = c0 + threadIdx.x, warp = threadIdx.x >> 5;
        Cut cut = c < ctas ? cuts[c] : Cut{};
        // what another call has written over the list, on a stream that the workspace was not for, is not followed
        if (cut.n > 1 && (cut.n > ctas - c || static_cast<unsigned int>(cut.b) >= static_cast<unsigned int>(p.batch) ||
                          static_cast<unsigned int>(cut.h) >= static_cast<unsigned int>(p.kv_heads * p.row_tiles))) {
            if (blockIdx.x == 0) atomicOr(fault_word, ALJ_FAULT_BOUNDS);
            cut.n = 0;
        }
        const uint32_t is = __ballot_sync(0xffffffffu, cut.n > 1);
        if (c0 > 0) __syncthreads();
        if ((threadIdx.x & 31) == 0) s_warp[warp] = __popc(is);
        __syncthreads();
        int at = count + __popc(is & ((1u << (threadIdx.x & 31)) - 1u));
#pragma unroll
        for (int w = 0; w < 8; ++w) {
            if (w < warp) at += s_warp[w];
            count += s_warp[w];
        }
        if (cut.n > 1) s_cut[at] = make_int4(c, cut.n, cut.b, cut.h);
    }
    __syncthreads();
    const int groups = (min(kRows, p.q_len * p.group) + kJoinRows - 1) / kJoinRows, units = count * groups;
    const long long size = kRows * (D + 2);
    constexpr int kQuads = D / 4;
#pragma unroll 1
    for (int unit = blockIdx.x; unit < units; unit += gridDim.x) {
        const int4 cut = s_cut[unit / groups];
        const int kvh = cut.w / p.row_tiles, row0 = (cut.w - kvh * p.row_tiles) * kRows;
        const int rows = min(kRows, p.q_len * p.group - row0);
#pragma unroll 1
        for (int i = threadIdx.x; i < kJoinRows * kQuads; i += 256) {
            const int row = (unit % groups) * kJoinRows + i / kQuads, d = (i % kQuads) * 4;
            if (row >= rows) break;
            float top = kNone, L = 0.0f;
            float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 1
            for (int k0 = 0; k0 < cut.y; k0 += kJoinParts) {
                float2 ml[kJoinParts];
                float4 v[kJoinParts];
#pragma unroll
                for (int u = 0; u < kJoinParts; ++u) {
                    const int k = k0 + u;
                    const float* part = p.part + (2 * (static_cast<long long>(cut.x) + k) + (k == 0 ? 1 : 0)) * size;
                    ml[u] = k < cut.y ? __ldcg(reinterpret_cast<const float2*>(part + kRows * D + row * 2)) : make_float2(kNone, 0.0f);
                    v[u] = k < cut.y ? __ldcg(reinterpret_cast<const float4*>(part + row * D + d)) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                }
                float now = top;
#pragma unroll
                for (int u = 0; u < kJoinParts; ++u) now = fmaxf(now, ml[u].x);
                const float f = ex2(top - now);
                top = now;
                L *= f;
                sum.x *= f, sum.y *= f, sum.z *= f, sum.w *= f;
#pragma unroll
                for (int u = 0; u < kJoinParts; ++u) {
                    const float g = ex2(ml[u].x - now);
                    L = fmaf(ml[u].y, g, L);
                    sum.x = fmaf(v[u].x, g, sum.x);
                    sum.y = fmaf(v[u].y, g, sum.y);
                    sum.z = fmaf(v[u].z, g, sum.z);
                    sum.w = fmaf(v[u].w, g, sum.w);
                }
            }
            const float inv = 1.0f / L;
            const bool none = L == 0.0f;
            const __nv_bfloat162 a = __floats2bfloat162_rn(none ? 0.0f : sum.x * inv, none ? 0.0f : sum.y * inv);
            const __nv_bfloat162 b = __floats2bfloat162_rn(none ? 0.0f : sum.z * inv, none ? 0.0f : sum.w * inv);
            const int r = row0 + row, t = r / p.group, hd = r - t * p.group;
            __nv_bfloat16* out = static_cast<__nv_bfloat16*>(p.out) +
                                 (((static_cast<long long>(cut.z) * p.q_len + t) * p.kv_heads + kvh) * p.group + hd) * D + d;
            *reinterpret_cast<uint2*>(out) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
        }
    }
}

template <int NG>
cudaError_t launch_tree(const Kv4Attn& p, Cut* cuts, int sms, unsigned int* fault_word, cudaStream_t stream) {
    using F = Shape<NG>;
    static_assert(smem_bytes<NG>() <= 232448, "shared memory of a CTA");
    static bool configured[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (!configured[dev & 63]) {
        const cudaError_t e = cudaFuncSetAttribute(kv4_tree_kernel<NG>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<NG>());
        if (e != cudaSuccess) return e;
        configured[dev & 63] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(sms);
    cfg.blockDim = dim3(F::THREADS);
    cfg.dynamicSmemBytes = smem_bytes<NG>();
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaLaunchKernelEx(&cfg, kv4_tree_kernel<NG>, p, cuts);
    if (e != cudaSuccess) return e;
    cfg.gridDim = dim3(kJoinBlocks * sms);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = sms * sizeof(int4);
    return cudaLaunchKernelEx(&cfg, kv4_tree_join_kernel<F::D>, p, static_cast<const Cut*>(cuts), sms, fault_word);
}

// Which kernel.  That of 8 or 16 columns (kv4_attention.cu) has all fp32 queries, since 16-bit operands would cost them
// their accuracy.  For bf16 its time goes with the passes over the cache, one for every 16 rows (8 at D 256), and this
// one's hardly with the rows, but this one takes 17 to 26 us for the smallest call.  Measured with 8 KV heads, us, the few
// columns' first and this kernel's second:
//   8 sequences of 16384:   16 rows, D 128: 72, 107   24: 124, 107   48: 182, 108   128: 452, 111
//                           D 64: 45, 90   75, 90   106, 91   258, 93      D 256: 155, 242   225, 243   434, 248   1130, 256
//   32 sequences of 1024:   32 rows, D 64, 128, 256: 38, 47   60, 58   115, 112     48 rows: 50, 48   82, 60   166, 113
//   1 sequence of 4096:     48 rows, D 64, 128, 256: 16, 19   23, 21    29, 33     128 rows: 23, 19   32, 21    52, 34
//   1 sequence of 257:     128 rows, D 64, 128, 256: 11, 18   12, 20    12, 27
// 32 rows is where D 64 turns.  D 128 would from 17 rows on and D 256 from 25, by up to 14 % and about a fifth on long
// contexts; up to 32 rows K's codes stay exact, as attend() has them.  So this kernel has more than 32 rows, where positions
// times heads, rows and dims reach 160 million (D 64 and 128: 40 rows of 8 sequences of 257, D 128, 22 and 21 us; 64 of D 64,
// 151 million, 11 and 19) or 640 million (D 256: 64 rows there 36 and 38, 80 rows 43 and 38).  The lengths are on the GPU: what
// counts is what the block table can hold, and short sequences in a wide table cost those 7 to 15 us more, and fp16's
// rounding of K and V.
bool tree_is_wide(const Kv4Attn& a) {
    const long long rows = static_cast<long long>(a.q_len) * a.group;
    if (a.type != ALJ_KV_BF16 || rows <= 32) return false;
    const double positions = static_cast<double>(a.batch) * a.page_size * (a.table ? a.table_stride : 1);
    return positions * a.kv_heads * rows * a.head_dim >= (a.head_dim == 256 ? 640e6 : 160e6);
}

}  // namespace

size_t kv4_tree_workspace_bytes(int q_rows, int head_dim, int sms) {
    const size_t few = kv4_attention_workspace_bytes(q_rows, head_dim, sms);
    const size_t many = kv4_attention_counter_bytes(sms) + (sms * sizeof(Cut) + 255) / 256 * 256 +
                        static_cast<size_t>(sms) * 2 * kRows * (head_dim + 2) * 4;
    return std::max(few, many);
}

cudaError_t launch_kv4_tree(const Kv4Attn& a, void* workspace, int sms, unsigned int* fault_word, cudaStream_t stream) {
    if (!tree_is_wide(a)) return launch_kv4_attention(a, workspace, sms, stream);
    Kv4Attn p = a;
    p.row_tiles = (p.q_len * p.group + kRows - 1) / kRows;
    p.group_magic = ((1u << 21) + p.group - 1) / p.group;   // row / group for row < 2048, exact as row * group < 2^21
    p.page_shift = (p.page_size & (p.page_size - 1)) == 0 ? __builtin_ctz(p.page_size) : -1;
    uint8_t* at = static_cast<uint8_t*>(workspace) + kv4_attention_counter_bytes(sms);
    Cut* cuts = reinterpret_cast<Cut*>(at);
    p.part = reinterpret_cast<float*>(at + (sms * sizeof(Cut) + 255) / 256 * 256);
    if (p.head_dim == 256) return launch_tree<8>(p, cuts, sms, fault_word, stream);
    if (p.head_dim == 128) return launch_tree<4>(p, cuts, sms, fault_word, stream);
    return p.head_dim == 64 ? launch_tree<2>(p, cuts, sms, fault_word, stream) : cudaErrorNotSupported;
}

}  // namespace alj

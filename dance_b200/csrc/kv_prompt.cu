// kv_prompt.cu -- attention of many rows (prompt chunks) over the 8-bit
// key/value cache on the tcgen05 tensor cores.
//
// A block holds 256 rows (query tokens x query heads of one key/value head) as
// two tiles of 128, one tensor-memory lane per row, and walks the sequence in
// tiles of 128 tokens:
//   S = Q K^T   (A, B in shared memory, f16, sums in tensor memory)
//   P = weights (softmax threads: S from tensor memory, P back to it as f16)
//   O += P V    (A = P from tensor memory, B in shared memory)
// The two row tiles alternate.  A row's 128 logits move into registers at
// once, so one S serves both tiles: the scores of the other tile, and then of
// the next token tile, are computed while the weights are.  Tensor memory: 128
// columns of S, 2 x 64 of P, 2 x head_dim of O, full at 128 channels.
//
// Measured on 2594 rows x 32 heads over 16000 and 7100 tokens of 128 channels:
// 0.78 ms, 0.72 PFLOP/s (0.44 of the measured matrix rate).  A token tile takes
// about 4900 clocks where the tensor core works 2100: what bounds it are the
// softmax threads' 3200 clocks for a tile (two warps a scheduler, the
// exponentials half of it) and the turning of codes into halves; tensor core,
// exponentials and issue slots are each under half used.  Tried and slower:
// an S for each row tile with P over it, so that softmax and both products of a
// tile follow one another, 0.82; with two buffers of 64 columns each, 0.94 (a
// product of 64 columns takes the tensor core as long as one of 128); weights
// handed over in halves, 0.95; a quarter of the exponentials as polynomials,
// 0.95; one register buffer of raw codes instead of two, 0.84; 176 registers
// for the softmax threads, 0.86, which then spill.  What helped before: the
// logits read from tensor memory once, 1.21 -> 0.88 together with registers
// handed to the softmax threads; one short copy of the code that issues the
// products (it competes with long unrolled loops for the instruction cache),
// 0.90 -> 0.86.
//
// Warps 0-3 and 4-7 hold the rows' softmax, one thread per row and no exchange
// between threads.  Warps 8-11 turn codes into halves: a tile's raw bytes are
// loaded into registers one tile ahead, then converted and stored, a token a
// row, with a 128-byte swizzle; K is read as K-major, V, whose rows are the
// summed dimension, as MN-major.  Warp 12 issues the matrix instructions.
//
// Weights.  A row sums p = 2^(s - m) in float; the product's operand is the half
// of p sv 2^base.  Rescaling O in tensor memory is a round trip, so m and base
// stay until a logit exceeds m by 8 or a weight would pass 2^15.  base is then set so
// that the row's largest p sv becomes 2^6 to 2^7: a weight has its 11 bits down to
// 2^-20 of the row's largest p sv and is lost below 2^-31.  Both come from the
// tokens that the row sees alone, however far apart the blocks' value scales lie;
// m and base are whole numbers, which sums and outputs are scaled by exactly.
// (Weights taken relative to the split's largest value scale, with no base to
// keep, were no faster: 783 us for the call above, against 779.)
//
// Every wait on a barrier is bounded.  A block that gives up counts itself in
// g_kv_prompt_timeouts, which dance_kv_status reads, and its rows read as
// not-a-number.
#include <cuda_runtime.h>

#include <cstdlib>
#include <type_traits>

#include "kv_attention.cuh"

namespace dance
{

// Blocks that gave up waiting (0 in a healthy run).
__device__ unsigned int g_kv_prompt_timeouts;

namespace
{

constexpr int kSoftWarps = 8, kConvWarps = 4;
constexpr int kMmaWarp = kSoftWarps + kConvWarps;
// Four groups of four warps, so that registers can be handed between them (the
// last group's other warps only wait): 128 x (2 x 184 + 96 + 48) = 512 x 128.
constexpr int kThreads = 512;
constexpr int kSoftRegs = 184, kConvRegs = 96, kMmaRegs = 48;
constexpr int kTok = (int)kPromptTokens;
constexpr int kGroups = kTok / 16;    // 16 tokens share a cache block
constexpr int kFactorStages = 4;      // factors are read up to two tiles after the codes are free
constexpr float kLift = 7.0f;         // log2 of a row's largest weight when its base is set
constexpr float kSlack = 8.0f;        // how far maximum and weights may rise before they are set anew
constexpr float kMostBase = 126.0f;   // bases whose power of two, and its inverse, are normal numbers
constexpr float kTame = 24.0f, kTameBase = 48.0f; // log2 of value scales, and bases, of a plain tile, up and down
constexpr float kFar = 1048576.0f;    // logits beyond it: their unrounded products part from the rounded ones
constexpr uint32_t kWaitNs = 20000;           // how long one try may sleep
constexpr long long kWaitClocks = 2000000000; // about a second: a wait in earnest is over in microseconds

template <int D>
struct Layout
{
    static constexpr int kTileBytes = (D + 63) / 64 * kTok * 128; // 128 rows of halves, 64 channels a run of 16 KB
    static constexpr int q = 0;                     // two row tiles
    static constexpr int k = 2 * kTileBytes;        // two stages
    static constexpr int v = 4 * kTileBytes;        // two stages
    static constexpr int factors = 6 * kTileBytes;  // kFactorStages x kGroups x (logit factor, log2 of the
                                                    // value scale, position (with the sign where the scale is far from
                                                    // 1), inverse of the value scale)
    static constexpr int bars = factors + kFactorStages * kGroups * 16;
    static constexpr int misc = bars + 24 * 8;
    static constexpr int used = misc + 64 + 1024;
    // more than half of an SM's shared memory: a second block would wait for tensor memory
    static constexpr int bytes = used > 118 * 1024 ? used : 118 * 1024;
};

enum Bar : int
{
    kKFull = 0,  // 2 stages
    kVFull = 2,
    kKEmpty = 4,
    kVEmpty = 6,
    kSFull = 8,  // 2 row tiles
    kPFull = 10,
    kODone = 12,
    kSFree = 14,
    kDrain = 15
};

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;\n" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];\n" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity), "r"(kWaitNs)
                 : "memory");
    return ok != 0;
}
// Bounded wait; false (with *gave_up set for the whole block) when it ran out.  The last try comes after the time: a
// block that was switched out for longer finds its barrier ready.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, long long clocks, volatile int *gave_up)
{
    if (bar_try(bar, parity))
        return true;
    const long long begin = clock64();
    for (;;)
    {
        const bool over = clock64() - begin >= clocks || *gave_up;
        if (bar_try(bar, parity))
            return true;
        if (over)
            break;
    }
    *gave_up = 1;
    return false;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Shared-memory matrix descriptor with 128-byte swizzle: start, leading and
// stride byte offsets, descriptor version 1.  K-major: stride = from 8 rows to
// the next 8 (leading unused).  MN-major: leading = from 64 channels to the
// next 64, stride = from 8 rows (of the summed dimension) to the next 8.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading, uint32_t stride)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)((leading >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((stride >> 4) & 0x3FFFu) << 32) | (1ull << 46) | (2ull << 61);
}
// kind::f16 instruction descriptor: f32 sums, f16 operands, M = 128.
constexpr uint32_t instr_desc(int n, bool b_mn_major)
{
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
// The products of one tile, issued in one go by the lane with `leader`; of the
// descriptors only the low words, which hold the start in 16 bytes, advance.
// S = Q K^T over D channels: 16 channels are 32 bytes of a row, 64 a run.
template <int D>
__device__ __forceinline__ void mma_scores(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc, uint32_t leader)
{
#define DANCE_SS(at, acc)                                                                                        \
    "add.u32 u, %1, " #at ";\n\tadd.u32 v, %2, " #at ";\n\tmov.b64 x, {u, %5};\n\tmov.b64 y, {v, %5};\n\t"         \
    "@q tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, " #acc ";\n\t"
#define DANCE_SS_HEAD                                                                                            \
    "{\n\t.reg .pred n, p, q;\n\t.reg .b64 x, y;\n\t.reg .b32 u, v;\n\tsetp.ne.b32 q, %4, 0;\n\t"                 \
    "setp.ne.b32 n, %4, %4;\n\tsetp.eq.b32 p, %4, %4;\n\t"                                                      \
    DANCE_SS(0, n) DANCE_SS(2, p) DANCE_SS(4, p) DANCE_SS(6, p)
    static_assert(kTok * 8 == 1024, "offset of the second run");
    if constexpr (D == 128)
        asm volatile(DANCE_SS_HEAD DANCE_SS(1024, p) DANCE_SS(1026, p) DANCE_SS(1028, p) DANCE_SS(1030, p) "}\n" ::"r"(d),
                     "r"(a), "r"(b), "r"(idesc), "r"(leader), "r"(high)
                     : "memory");
    else if constexpr (D == 96)
        asm volatile(DANCE_SS_HEAD DANCE_SS(1024, p) DANCE_SS(1026, p) "}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc),
                     "r"(leader), "r"(high)
                     : "memory");
    else
        asm volatile(DANCE_SS_HEAD "}\n" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(leader), "r"(high) : "memory");
#undef DANCE_SS_HEAD
#undef DANCE_SS
}
// O (+)= P V over 128 tokens: 16 tokens are 8 columns of P and 2 KB of V.
__device__ __forceinline__ void mma_values(uint32_t d, uint32_t a, uint32_t b, uint32_t high, uint32_t idesc,
                                           uint32_t accumulate, uint32_t leader)
{
#define DANCE_TS(col, at, acc)                                                                                   \
    "add.u32 x, %1, " #col ";\n\tadd.u32 v, %2, " #at ";\n\tmov.b64 y, {v, %6};\n\t"                             \
    "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [x], y, %3, " #acc ";\n\t"
    asm volatile("{\n\t.reg .pred n, p, q;\n\t.reg .b32 x, v;\n\t.reg .b64 y;\n\tsetp.ne.b32 q, %5, 0;\n\t"
                 "setp.ne.b32 n, %4, 0;\n\tsetp.eq.b32 p, %4, %4;\n\t" DANCE_TS(0, 0, n) DANCE_TS(8, 128, p)
                     DANCE_TS(16, 256, p) DANCE_TS(24, 384, p) DANCE_TS(32, 512, p) DANCE_TS(40, 640, p)
                         DANCE_TS(48, 768, p) DANCE_TS(56, 896, p) "}\n" ::"r"(d),
                 "r"(a), "r"(b), "r"(idesc), "r"(accumulate), "r"(leader), "r"(high)
                 : "memory");
#undef DANCE_TS
}
__device__ __forceinline__ void commit(uint32_t bar, uint32_t leader)
{
    asm volatile("{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
                 "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(bar),
                 "r"(leader)
                 : "memory");
}

__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, "
                 "[%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
                   "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
                   "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
                   "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16])
{
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15}, [%16];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
// Waits for the loads in flight; what they loaded passes through, so that no
// use of it can move ahead of the wait.
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[32])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void loaded(uint32_t (&r)[32])
{
    asm volatile(""
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]),
                   "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
                   "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                   "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_wait(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;\n"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]),
                   "+r"(r[6]), "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]),
                   "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16};\n" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// Two floats in one register pair: one instruction for both.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
        "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return r;
}
// Byte offset of 16-byte chunk c (8 channels) of row r: runs of 64 channels,
// 128 bytes a row, the chunks of eight rows exchanged (128-byte swizzle) so
// that neither the threads that store a column of rows nor the tensor core
// that reads one meet on a bank.
__device__ __forceinline__ uint32_t tile_off(int r, int c)
{
    return (uint32_t)((c >> 3) * (kTok * 128) + r * 128 + (((c ^ r) & 7) << 4));
}

// What a block works on.
struct Work
{
    KvSeq s;
    uint32_t b, h, split;
    int r0, r1;           // packed rows
    int seen_lo, seen_hi; // tokens that its first and last row see
    int e0, e1, nsplits;  // cache blocks of the split
    int tiles;            // token tiles
    int base;             // position of the first token
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1) prompt_kernel(AttnParams p)
{
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = smem_raw + ((0u - smem_addr(smem_raw)) & 1023u); // the swizzle counts from 1024 bytes
    using L = Layout<D>;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    Work w;
    w.b = blockIdx.y;
    const uint32_t rt = blockIdx.x % p.row_tiles;
    w.h = (blockIdx.x / p.row_tiles) % p.c.hkv;
    w.split = blockIdx.x / p.row_tiles / p.c.hkv;
    w.s = kv_seq(p.c, w.b, p.rows);
    const int shift = (int)p.c.shift, G = (int)p.G;
    w.r0 = (int)(rt * kPromptRows);
    const int nrows = w.s.rows * G;
    if (w.r0 >= nrows)
        return;
    w.r1 = min(w.r0 + (int)kPromptRows, nrows);
    w.seen_lo = min(w.s.first + w.r0 / G + 1, w.s.len);
    w.seen_hi = min(w.s.first + (w.r1 - 1) / G + 1, w.s.len);
    const int nent = (max(w.seen_hi, 0) + (1 << shift) - 1) >> shift;
    w.nsplits = max(1, (nent + (int)p.chunk - 1) / (int)p.chunk);
    if ((int)w.split >= w.nsplits)
        return;
    w.e0 = (int)w.split * (int)p.chunk;
    w.e1 = min(w.e0 + (int)p.chunk, nent);
    w.base = w.e0 << shift;
    w.tiles = max(0, (min(w.e1 << shift, w.seen_hi) - w.base + kTok - 1) / kTok);
    const bool two = w.r1 - w.r0 > 128;

    const uint32_t sbase = smem_addr(smem);
    auto bar = [&](int i) { return sbase + L::bars + 8u * (uint32_t)i; };
    volatile int *gave_up = reinterpret_cast<volatile int *>(smem + L::misc);
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + L::misc + 4);
    int *s_last = reinterpret_cast<int *>(smem + L::misc + 8);
    float4 *s_f = reinterpret_cast<float4 *>(smem + L::factors);

    if (warp == kMmaWarp)
    {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(smem_addr(tmem_slot)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    if (tid == 0)
    {
        for (int i = 0; i < 2; ++i)
        {
            bar_init(bar(kKFull + i), 32 * kConvWarps);
            bar_init(bar(kVFull + i), 32 * kConvWarps);
            bar_init(bar(kKEmpty + i), 1);
            bar_init(bar(kVEmpty + i), 1);
            bar_init(bar(kSFull + i), 1);
            bar_init(bar(kPFull + i), 128);
            bar_init(bar(kODone + i), 1);
        }
        bar_init(bar(kSFree), 128);
        bar_init(bar(kDrain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        *gave_up = p.wait_clocks > 0 ? 0 : 1; // a limit of nothing has run out
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    // ---- q: one thread per row, as halves
    float rf = 0.0f; // logit factor of the thread's row
    int limit = 0;   // tokens that it sees
    if (warp < kSoftWarps)
    {
        const int r = w.r0 + tid;
        const bool live = r < w.r1;
        const int i = live ? r / G : 0, hd = (int)w.h * G + (live ? r % G : 0);
        const uint16_t *src = p.q + (uint64_t)(w.s.row0 + i) * p.q_row + (uint64_t)hd * p.q_head;
        uint32_t x[D / 2];
        if (live && p.q_aligned)
        {
#pragma unroll
            for (int e = 0; e < D / 8; ++e)
                *reinterpret_cast<uint4 *>(&x[4 * e]) = __ldg(reinterpret_cast<const uint4 *>(src) + e);
        }
        else
        {
#pragma unroll
            for (int e = 0; e < D / 2; ++e)
                x[e] = live ? (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16) : 0u;
        }
        float amax = 0.0f;
#pragma unroll
        for (int e = 0; e < D / 2; ++e)
            amax = fmaxf(amax, fmaxf(fabsf(kv_float<BF16>((uint16_t)x[e])), fabsf(kv_float<BF16>((uint16_t)(x[e] >> 16)))));
        const int up = row_shift(amax);
        // the sign of the logits' factor goes into q: a group's largest logit has to be that of its largest product
        const float mul = p.scale_log2 < 0.0f ? -power_of_two(up) : power_of_two(up);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
        {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = kv_pack<false>(kv_float<BF16>((uint16_t)x[4 * c + e]) * mul,
                                      kv_float<BF16>((uint16_t)(x[4 * c + e] >> 16)) * mul);
            *reinterpret_cast<uint4 *>(smem + L::q + (tid >> 7) * L::kTileBytes + tile_off(tid & 127, c)) =
                make_uint4(y[0], y[1], y[2], y[3]);
        }
        rf = live ? power_of_two(-up) * fabsf(p.scale_log2) : 0.0f;
        limit = live ? min(w.s.first + i + 1, w.s.len) : 0;
        fence_smem();
    }
    __syncthreads();
    float m = kKvNegInf, l = 0.0f, base = kMostBase, unbase = 0.0f;
    bool ok = true;

    if (warp < kSoftWarps)
    {
        // ------------------------------------------------ softmax
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;\n" ::"n"(kSoftRegs));
        const int tile = warp >> 2;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21; // tensor-memory lane in bits 16 and up
        const uint32_t s_addr = tmem + lanes, p_addr = s_addr + 128u + 64u * (uint32_t)tile;
        const uint32_t o_addr = tmem + lanes + 256u + (uint32_t)(D * tile);
        const int tile_lo = min(w.s.first + (w.r0 + 128 * tile) / G + 1, w.s.len); // least that a row of the tile sees
        for (int i = 0; i < (tile == 0 || two ? w.tiles : 0); ++i)
        {
            ok = bar_wait(bar(kSFull + tile), (uint32_t)i & 1u, p.wait_clocks, gave_up);
            if (!__all_sync(kKvFull, ok))
            {
                ok = false;
                break;
            }
            fence_after();
            const float4 *f = s_f + (i % kFactorStages) * kGroups;

            // The row's 128 logits stay in registers from the maximum to the weights.
            uint32_t x[4][32];
            tmem_ld32(s_addr, x[0]);
            tmem_ld32(s_addr + 32u, x[1]);
            bool whole = w.base + (i + 1) * kTok <= tile_lo;
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                whole &= __float_as_uint(f[g].z) < (uint32_t)kMaxPos;
            tmem_ld_wait(x[0]);
            loaded(x[1]);
            tmem_ld32(s_addr + 64u, x[2]);
            tmem_ld32(s_addr + 96u, x[3]);
            float top = kKvNegInf, heavy = kKvNegInf; // largest logit; log2 of the largest p times value scale
            float largest[kGroups];
            // the logits' factor is not negative and constant over 16 tokens
            auto maximum = [&](auto masked, int g0) {
#pragma unroll
                for (int g = g0; g < g0 + kGroups / 2; ++g)
                {
                    const float4 fg = f[g];
                    float m0 = kKvNegInf, m1 = kKvNegInf;
                    const int left = limit - (__float_as_int(fg.z) & kMaxPos); // columns of the group that the row sees
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                    {
                        const float y0 = __uint_as_float(x[g >> 1][16 * (g & 1) + e]);
                        const float y1 = __uint_as_float(x[g >> 1][16 * (g & 1) + e + 8]);
                        m0 = fmaxf(m0, !masked || e < left ? y0 : kKvNegInf);
                        m1 = fmaxf(m1, !masked || e + 8 < left ? y1 : kKvNegInf);
                    }
                    m0 = fmaxf(m0, m1);
                    float y = m0 * (fg.x * rf);
                    if constexpr (masked)
                        y = m0 == kKvNegInf ? kKvNegInf : y;
                    largest[g] = y;
                    top = fmaxf(top, y);
                    heavy = fmaxf(heavy, y - m + fg.y);
                }
            };
            // Weights p = 2^(s - m), summed, and p times value scale times 2^base, the product's operand.  Plain tiles
            // take the latter's exponent at once and the sum's terms from it; where a mask, far logits or a scale
            // that would leave the range of floats there are met, each is computed by itself.
            auto weights = [&](auto masked) {
                const float shift_m = masked && m == kKvNegInf ? 0.0f : -m;
#pragma unroll
                for (int c = 0; c < 4; ++c)
                {
                    uint32_t y[16];
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                    {
                        const float4 fg = f[2 * c + u];
                        const float kf = fg.x * rf, sm = masked ? shift_m : shift_m + (base + fg.y);
                        const float vf = masked ? exp2_fast(fminf(base + fg.y, kMostBase)) : 1.0f;
                        const int left = limit - (__float_as_int(fg.z) & kMaxPos);
                        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                        {
                            float2 z = make_float2(__uint_as_float(x[c][16 * u + 2 * e]),
                                                   __uint_as_float(x[c][16 * u + 2 * e + 1]));
                            if constexpr (masked)
                            {
                                // products rounded as the maximum's is: none exceeds it, however far
                                z.x = 2 * e < left ? __fadd_rn(__fmul_rn(z.x, kf), sm) : kKvNegInf;
                                z.y = 2 * e + 1 < left ? __fadd_rn(__fmul_rn(z.y, kf), sm) : kKvNegInf;
                            }
                            else
                                z = fma2(z, make_float2(kf, kf), make_float2(sm, sm));
                            z.x = exp2_fast(z.x);
                            z.y = exp2_fast(z.y);
                            sum.x += z.x;
                            sum.y += z.y;
                            if constexpr (masked)
                                z.x *= vf, z.y *= vf;
                            y[8 * u + e] = kv_pack<false>(z.x, z.y);
                        }
                        l = masked ? l + (sum.x + sum.y) : fmaf(sum.x + sum.y, fg.w * unbase, l);
                    }
                    tmem_st16(p_addr + 16u * c, y);
                }
            };
            if (whole)
                maximum(std::false_type{}, 0);
            else
                maximum(std::true_type{}, 0);
            tmem_ld_wait(x[2]);
            loaded(x[3]);
            fence_before();
            bar_arrive(bar(kSFree)); // the other row tile's scores may take its place
            if (whole)
                maximum(std::false_type{}, kGroups / 2);
            else
                maximum(std::true_type{}, kGroups / 2);
            // the product before is done with O and with the place of the weights
            if (i > 0)
            {
                ok = bar_wait(bar(kODone + tile), (uint32_t)(i - 1) & 1u, p.wait_clocks, gave_up);
                if (!__all_sync(kKvFull, ok))
                {
                    ok = false;
                    break;
                }
                fence_after();
            }
            if (__any_sync(kKvFull, top > m + kSlack || heavy + base > kLift + kSlack))
            {
                // m: an integer, so that powers of two are all that sums and outputs are scaled by
                const float mn = top > m + kSlack ? ceilf(top) : m; // from -inf: any maximum
                float need = kKvNegInf;
#pragma unroll
                for (int g = 0; g < kGroups; ++g)
                    need = fmaxf(need, largest[g] - mn + f[g].y);
                const float keep = fminf(base + (mn - m), kMostBase); // leaves O as it is; from -inf: kMostBase
                const float bn = need + keep > kLift + kSlack ? fmaxf(floorf(kLift - need), -kMostBase) : keep;
                const float out_down = mn != m || bn != base ? exp2_fast((m - mn) + (bn - base)) : 1.0f;
                l *= mn != m ? exp2_fast(m - mn) : 1.0f; // from -inf: 0
                m = mn;
                base = bn;
                unbase = exp2_fast(-bn);
                if (i > 0 && __any_sync(kKvFull, out_down != 1.0f))
                {
#pragma unroll 1
                    for (int c = 0; c < D / 16; ++c)
                    {
                        uint32_t o[16];
                        tmem_ld16(o_addr + 16u * c, o);
                        tmem_ld_wait(o);
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            o[e] = __float_as_uint(__uint_as_float(o[e]) * out_down);
                        tmem_st16(o_addr + 16u * c, o);
                    }
                }
            }
            if (whole && __all_sync(kKvFull, fabsf(m) < kFar && fabsf(base) <= kTameBase))
                weights(std::false_type{});
            else
                weights(std::true_type{});
            tmem_st_wait();
            fence_before();
            bar_arrive(bar(kPFull + tile));
        }
        // ------------------------------------------------ out
        if (w.tiles > 0 && ok && (tile == 0 || two))
        {
            ok = bar_wait(bar(kODone + tile), (uint32_t)(w.tiles - 1) & 1u, p.wait_clocks, gave_up);
            ok = __all_sync(kKvFull, ok);
            fence_after();
        }
        const int r = w.r0 + tid;
        const bool live = r < w.r1;
        const float lse2 = l == 0.0f ? kKvNegInf : m + log2f(l);
        float f = l == 0.0f ? 0.0f : 1.0f / l;
        if (!ok)
            f = __int_as_float(0x7FC00000);
        // unbase is apart from f: their product may leave the range of floats
        const int i = live ? r / G : 0, hd = (int)w.h * G + (live ? r % G : 0);
        const int item = (int)((w.b * p.c.hkv + w.h) * p.row_tiles + rt);
        float *part = p.part + (uint64_t)item * p.splits * kPromptRows * (D + 1);
        float *part_lse = part + (uint64_t)p.splits * kPromptRows * D;
        uint16_t *out = reinterpret_cast<uint16_t *>(p.out) + ((uint64_t)(w.s.row0 + i) * p.heads + hd) * D;
        if (live)
        {
            if (w.nsplits > 1)
                part_lse[w.split * kPromptRows + tid] = ok ? lse2 : f;
            else if (p.lse)
                p.lse[(uint64_t)(w.s.row0 + i) * p.heads + hd] = (ok ? lse2 : f) * 0.69314718056f;
        }
        if (tile == 0 || two)
        {
#pragma unroll
            for (int c = 0; c < D / 32; ++c)
            {
                uint32_t x[32];
                if (w.tiles > 0 && ok)
                {
                    tmem_ld32(o_addr + 32u * c, x);
                    tmem_ld_wait(x);
                }
                else
                {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        x[e] = 0u;
                }
                if (live && w.nsplits > 1)
                {
                    float4 *dst = reinterpret_cast<float4 *>(part + ((uint64_t)w.split * kPromptRows + tid) * D + 32 * c);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        dst[e] = make_float4(__uint_as_float(x[4 * e]) * f * unbase, __uint_as_float(x[4 * e + 1]) * f * unbase,
                                             __uint_as_float(x[4 * e + 2]) * f * unbase,
                                             __uint_as_float(x[4 * e + 3]) * f * unbase);
                }
                else if (live)
                {
                    uint4 *dst = reinterpret_cast<uint4 *>(out + 32 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            y[k] = kv_pack<BF16>(__uint_as_float(x[8 * e + 2 * k]) * f * unbase,
                                                 __uint_as_float(x[8 * e + 2 * k + 1]) * f * unbase);
                        dst[e] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
            }
        }
        if (w.nsplits > 1)
        {
            // ---- the splits are joined by the block that comes last, in their order
            __threadfence();
            asm volatile("bar.sync 1, 256;\n" ::: "memory");
            if (tid == 0)
                *s_last = atomicAdd(p.counters + item, 1u) == (uint32_t)w.nsplits - 1u;
            asm volatile("bar.sync 1, 256;\n" ::: "memory");
            if (*s_last)
            {
                __threadfence();
                if (tid == 0)
                    p.counters[item] = 0u;
                uint16_t *rows_out = reinterpret_cast<uint16_t *>(p.out);
                // a warp per row, a lane per 4 channels
                for (int r = warp; w.r0 + r < w.r1; r += kSoftWarps)
                {
                    const int i = (w.r0 + r) / G, hd = (int)w.h * G + (w.r0 + r) % G;
                    float top = kKvNegInf, sum = 0.0f;
                    for (int k = lane; k < w.nsplits; k += 32)
                        top = fmaxf(top, __ldcg(part_lse + k * kPromptRows + r));
                    for (int o = 16; o; o >>= 1)
                        top = fmaxf(top, __shfl_xor_sync(kKvFull, top, o));
                    const float ref = top == kKvNegInf ? 0.0f : top;
                    float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
                    for (int k = 0; k < w.nsplits; ++k)
                    {
                        const float wt = exp2_fast(__ldcg(part_lse + k * kPromptRows + r) - ref);
                        sum += wt;
                        if (lane < D / 4)
                        {
                            const float4 z = __ldcg(reinterpret_cast<const float4 *>(
                                part + ((uint64_t)k * kPromptRows + r) * D + 4 * lane));
                            y.x += wt * z.x, y.y += wt * z.y, y.z += wt * z.z, y.w += wt * z.w;
                        }
                    }
                    const float f = sum == 0.0f ? 0.0f : 1.0f / sum;
                    const uint64_t at = (uint64_t)(w.s.row0 + i) * p.heads + hd;
                    if (lane < D / 4)
                        *reinterpret_cast<uint2 *>(rows_out + at * D + 4 * lane) =
                            make_uint2(kv_pack<BF16>(y.x * f, y.y * f), kv_pack<BF16>(y.z * f, y.w * f));
                    if (lane == 0 && p.lse)
                        p.lse[at] = (sum == 0.0f ? kKvNegInf : ref + log2f(sum)) * 0.69314718056f;
                }
            }
        }
        fence_before();
    }
    else if (warp < kSoftWarps + kConvWarps)
    {
        // ------------------------------------------------ codes to halves
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kConvRegs));
        constexpr int kPairs = D / 16; // (8 tokens, 16 channels) units of a lane
        const int cw = warp - kSoftWarps;
        uint4 rk[kPairs], rv[kPairs];          // raw bytes, loaded a tile ahead
        int blk[2] = {-1, -1}, nblk[2]; // blocks of the warp's two groups of 16 tokens: loaded tile, next tile
        float fk = 0.0f, fv = 0.0f;
        const int bs1 = (1 << shift) - 1;
        auto look = [&](int i, int (&to)[2]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const int pos = w.base + i * kTok + cw * 32 + u * 16;
                to[u] = i < w.tiles && pos < w.seen_hi ? kv_block(p.c, w.b, pos >> shift) : -1;
            }
        };
        auto load = [&](int i, const uint8_t *pool, uint64_t stride, uint4 (&r)[kPairs]) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const int pos = w.base + i * kTok + cw * 32 + u * 16;
                const uint8_t *src = pool + (uint64_t)max(blk[u], 0) * stride +
                                     (uint64_t)(((w.h << shift) + (uint32_t)(pos & bs1)) * D) + (lane & 7) * D;
#pragma unroll
                for (int it = 0; it < kPairs; ++it)
                {
                    const int pair = it * 4 + (lane >> 3), grp = pair / (D / 16), ch = pair % (D / 16);
                    if (grp >> 1 != u)
                        continue;
                    r[it] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                    if (blk[u] >= 0)
                        r[it] = __ldg(reinterpret_cast<const uint4 *>(src + (grp & 1) * 8 * D + ch * 16));
                }
            }
        };
        auto convert = [&](uint8_t *tile, const uint4 (&r)[kPairs]) {
#pragma unroll
            for (int it = 0; it < kPairs; ++it)
            {
                const int pair = it * 4 + (lane >> 3), grp = pair / (D / 16), ch = pair % (D / 16);
                const int row = cw * 32 + grp * 8 + (lane & 7);
                const uint32_t u[4] = {r[it].x, r[it].y, r[it].z, r[it].w};
                uint32_t y[8];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    y[2 * e] = code_halves(u[e], 0x4140);
                    y[2 * e + 1] = code_halves(u[e], 0x4342);
                }
                *reinterpret_cast<uint4 *>(tile + tile_off(row, 2 * ch)) = make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4 *>(tile + tile_off(row, 2 * ch + 1)) = make_uint4(y[4], y[5], y[6], y[7]);
            }
        };
        auto factors = [&]() { // lane u of the warp: group u
            fk = fv = 0.0f;
            const int mine = lane ? blk[1] : blk[0];
            if (lane < 2 && mine >= 0)
            {
                const uint64_t si = (uint64_t)mine * p.c.hkv + w.h;
                fk = __ldg(p.c.ks + si);
                fv = __ldg(p.c.vs + si);
            }
        };
        look(0, blk);
        load(0, p.c.k, p.c.kbs, rk);
        load(0, p.c.v, p.c.vbs, rv);
        factors();
        look(1, nblk);
#pragma unroll 1
        for (int i = 0; i < w.tiles; ++i)
        {
            const int st = i & 1;
            const uint32_t par = (uint32_t)((i >> 1) + 1) & 1u; // of the stage's release before this use
            if (i >= 2)
                ok = bar_wait(bar(kKEmpty + st), par, p.wait_clocks, gave_up);
            if (!__all_sync(kKvFull, ok))
                break;
            const bool held = (lane ? blk[1] : blk[0]) >= 0;
            if (lane < 2)
            {
                const float lg = log2f(fv);
                const int pos = held ? w.base + i * kTok + cw * 32 + lane * 16 : kMaxPos;
                s_f[(i % kFactorStages) * kGroups + cw * 2 + lane] =
                    make_float4(fk, lg, __int_as_float(fabsf(lg) <= kTame ? pos : pos | (int)0x80000000), 1.0f / fv);
            }
            convert(smem + L::k + st * L::kTileBytes, rk);
            fence_smem();
            bar_arrive(bar(kKFull + st));
            if (i >= 2)
                ok = bar_wait(bar(kVEmpty + st), par, p.wait_clocks, gave_up);
            if (!__all_sync(kKvFull, ok))
                break;
            convert(smem + L::v + st * L::kTileBytes, rv);
            fence_smem();
            bar_arrive(bar(kVFull + st));
            // the next tile's loads come behind the fences, which would wait for them
            blk[0] = nblk[0];
            blk[1] = nblk[1];
            load(i + 1, p.c.k, p.c.kbs, rk);
            load(i + 1, p.c.v, p.c.vbs, rv);
            factors();
            look(i + 2, nblk);
        }
    }
    else
    {
        // ------------------------------------------------ matrix instructions
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;\n" ::"n"(kMmaRegs));
        if (warp == kMmaWarp && !__any_sync(kKvFull, *gave_up))
        {
            // The whole warp walks the loop and one lane issues: with every address the same in all lanes by
            // construction (reductions and votes), the operands stay in uniform registers.
            const uint32_t leader = lane == 0 ? 1u : 0u, tm = __reduce_max_sync(kKvFull, tmem);
            const uint32_t tiles = __reduce_max_sync(kKvFull, (unsigned)w.tiles);
            const bool both = __any_sync(kKvFull, two);
            constexpr uint32_t kIdS = instr_desc(kTok, false), kIdO = instr_desc(D, true);
            const uint64_t dk = smem_desc(0u, 16u, 1024u), dv = smem_desc(0u, kTok * 128u, 1024u);
            constexpr uint32_t kNext = L::kTileBytes / 16;
            const uint32_t aq = (sbase + L::q) >> 4, ak = ((sbase + L::k) >> 4) | (uint32_t)dk;
            const uint32_t av = ((sbase + L::v) >> 4) | (uint32_t)dv;
            auto wait = [&](int which, uint32_t parity) {
                if (__all_sync(kKvFull, bar_try(bar(which), parity)))
                    return true;
                const long long begin = clock64();
                for (;;)
                {
                    const bool over = clock64() - begin >= p.wait_clocks || *gave_up;
                    if (__all_sync(kKvFull, bar_try(bar(which), parity)))
                        return true;
                    if (__any_sync(kKvFull, over))
                        break;
                }
                *gave_up = 1;
                return false;
            };
            const uint32_t ntile = both ? 2u : 1u;
            // One copy of each piece of this code: between its turns the softmax threads' long loops pass through the
            // instruction cache.  Step n issues the scores of row tile n % ntile over token tile n / ntile, as soon as
            // the scores before have been read, and then the product with V of ntile steps before.
            const uint32_t steps = tiles * ntile;
#pragma unroll 1
            for (uint32_t n = 0; n < steps + ntile; ++n)
            {
                const uint32_t tile = both ? n & 1u : 0u, i = both ? n >> 1 : n; // scores' token tile
                const uint32_t sk = i & 1u, sv = sk ^ 1u;
                if (n < steps)
                {
                    if (tile == 0 && !wait(kKFull + (int)sk, (i >> 1) & 1u))
                        break;
                    if (n > 0 && !wait(kSFree, (n - 1u) & 1u))
                        break;
                    fence_after();
                    mma_scores<D>(tm, (aq + tile * kNext) | (uint32_t)dk, ak + sk * kNext, (uint32_t)(dk >> 32), kIdS, leader);
                    commit(bar(kSFull + (int)tile), leader);
                    if (tile + 1 == ntile)
                        commit(bar(kKEmpty + (int)sk), leader);
                }
                if (n >= ntile)
                {
                    if (tile == 0 && !wait(kVFull + (int)sv, ((i - 1u) >> 1) & 1u))
                        break;
                    if (!wait(kPFull + (int)tile, sv))
                        break;
                    fence_after();
                    mma_values(tm + 256u + (uint32_t)D * tile, tm + 128u + 64u * tile, av + sv * kNext, (uint32_t)(dv >> 32),
                               kIdO, i - 1u, leader);
                    commit(bar(kODone + (int)tile), leader);
                    if (tile + 1 == ntile)
                        commit(bar(kVEmpty + (int)sv), leader);
                }
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (*gave_up)
    {
        // matrix instructions in flight when a wait ran out get a bounded time to end
        if (tid == 32 * kMmaWarp)
        {
            atomicAdd(&g_kv_prompt_timeouts, 1u);
            commit(bar(kDrain), 1u);
            const long long begin = clock64();
            while (!bar_try(bar(kDrain), 0u) && clock64() - begin < kWaitClocks)
            {
            }
        }
        __syncthreads();
    }
    fence_after();
    __syncthreads();
    if (warp == kMmaWarp)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D, bool BF16>
int launch(const AttnParams &p, uint32_t blocks_x, cudaStream_t st)
{
    static SmemAllowed allowed;
    DANCE_CUDA(allowed.on_current(reinterpret_cast<const void *>(prompt_kernel<D, BF16>), Layout<D>::bytes));
    prompt_kernel<D, BF16><<<dim3(blocks_x, p.c.batch), kThreads, Layout<D>::bytes, st>>>(p);
    DANCE_LAUNCHED();
    return 0;
}

} // namespace

int launch_prompt(AttnParams &p, uint32_t head_dim, bool bf16, uint32_t blocks_x, cudaStream_t st)
{
    const char *limit = std::getenv("DANCE_KV_WAIT_CLOCKS");
    p.wait_clocks = limit ? std::atoll(limit) : kWaitClocks;
    p.wait_clocks = p.wait_clocks < 0 || p.wait_clocks > kWaitClocks ? kWaitClocks : p.wait_clocks;
    switch (head_dim)
    {
    case 64:
        return bf16 ? launch<64, true>(p, blocks_x, st) : launch<64, false>(p, blocks_x, st);
    case 96:
        return bf16 ? launch<96, true>(p, blocks_x, st) : launch<96, false>(p, blocks_x, st);
    default:
        return bf16 ? launch<128, true>(p, blocks_x, st) : launch<128, false>(p, blocks_x, st);
    }
}

} // namespace dance

using namespace dance;

extern "C" int dance_kv_status(void)
{
    unsigned int t = 0;
    DANCE_CUDA(cudaDeviceSynchronize());
    DANCE_CUDA(cudaMemcpyFromSymbol(&t, g_kv_prompt_timeouts, sizeof(t)));
    if (t)
    {
        const unsigned int z = 0;
        DANCE_CUDA(cudaMemcpyToSymbol(g_kv_prompt_timeouts, &z, sizeof(z)));
        return fail(-4, "key/value attention: %u blocks gave up waiting", t);
    }
    return 0;
}

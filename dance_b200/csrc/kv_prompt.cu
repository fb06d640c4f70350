// kv_prompt.cu -- attention of many rows (prompt chunks) over the 8-bit
// key/value cache on the tcgen05 tensor cores.
//
// A block holds 256 rows (query tokens x query heads of one key/value head) as
// two tiles of 128, one tensor-memory lane per row, and walks the sequence in
// tiles of 128 tokens:
//   S = Q K^T   (A, B in shared memory, f16, sums in tensor memory)
//   P = weights (softmax threads: S from tensor memory, P back over it as f16)
//   O += P V    (A = P from tensor memory, B in shared memory)
// The two row tiles alternate, so that the tensor core works on one while the
// softmax threads work on the other; tensor memory is full: 2 x 128 columns of
// S (P lies over the first half of its S) and 2 x head_dim of O.
//
// Warps 0-3 and 4-7 hold the rows' softmax, one thread per row and no exchange
// between threads.  Warps 8-11 turn codes into halves: a tile's raw bytes are
// loaded into registers one tile ahead, then converted and stored in the
// K-major core-matrix layout (8 rows x 16 bytes); the same layout read as
// MN-major serves V, whose rows are the summed dimension.  Warp 12 issues the
// matrix instructions.
//
// Rescaling O in tensor memory is a round trip, so a row keeps its reference
// maximum until the true one exceeds it by 2^8: weights are 2^(s - ref + 7) <=
// 2^15, inside a half.  The reference only shifts weights and their sum alike.
//
// Every wait on a barrier is bounded.  A block that gives up counts itself in
// g_kv_prompt_timeouts, and its rows read as not-a-number.
#include <cuda_runtime.h>

#include "kv_attention.cuh"

namespace dance
{

// Blocks that gave up waiting (0 in a healthy run).
__device__ unsigned int g_kv_prompt_timeouts;

namespace
{

constexpr int kSoftWarps = 8, kConvWarps = 4;
constexpr int kThreads = 32 * (kSoftWarps + kConvWarps + 1);
constexpr int kTok = (int)kPromptTokens;
constexpr int kGroups = kTok / 16;    // 16 tokens share a cache block
constexpr int kFactorStages = 4;      // factors are read up to two tiles after the codes are free
constexpr float kLift = 7.0f;         // log2 of the weight of a row's reference maximum
constexpr float kSlack = 8.0f;        // how far the maximum may rise above the reference
constexpr uint32_t kWaitLimit = 1u << 24;

template <int D>
struct Layout
{
    static constexpr int kTileBytes = kTok * D * 2; // 128 rows of D halves
    static constexpr int q = 0;                     // two row tiles
    static constexpr int k = 2 * kTileBytes;        // two stages
    static constexpr int v = 4 * kTileBytes;        // two stages
    static constexpr int factors = 6 * kTileBytes;  // kFactorStages x kGroups x (logit, weight, position, -)
    static constexpr int bars = factors + kFactorStages * kGroups * 16;
    static constexpr int misc = bars + 16 * 8;
    static constexpr int used = misc + 64;
    // more than half of an SM's shared memory: a second block would wait for tensor memory
    static constexpr int bytes = used > 118 * 1024 ? used : 118 * 1024;
};

enum Bar : int
{
    kKFull = 0,  // 2 stages
    kVFull = 2,
    kKEmpty = 4,
    kVEmpty = 6,
    kSFull = 8, // 2 row tiles
    kPFull = 10,
    kODone = 12,
    kDrain = 14,
    kBars = 15
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
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
                 "selp.u32 %0, 1, 0, p;\n\t}\n"
                 : "=r"(ok)
                 : "r"(bar), "r"(parity)
                 : "memory");
    return ok != 0;
}
// Bounded wait; false (with *gave_up set for the whole block) when it ran out.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int *gave_up)
{
    if (bar_try(bar, parity))
        return true;
    for (uint32_t it = 0; it < kWaitLimit; ++it)
    {
        if (bar_try(bar, parity))
            return true;
        if ((it & 255u) == 255u && *gave_up)
            return false;
    }
    *gave_up = 1;
    return false;
}
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory"); }
__device__ __forceinline__ void fence_smem() { asm volatile("fence.proxy.async.shared::cta;\n" ::: "memory"); }

// Shared-memory matrix descriptor without swizzle: start, leading and stride
// byte offsets, descriptor version 1.  K-major: leading = from one 16-byte
// column of core matrices to the next, stride = from 8 rows to the next 8.
// MN-major: leading = from 8 rows (of the summed dimension) to the next 8,
// stride = from one 16-byte column to the next.
__device__ __forceinline__ uint64_t smem_desc(uint32_t addr, uint32_t leading, uint32_t stride)
{
    return (uint64_t)((addr & 0x3FFFFu) >> 4) | ((uint64_t)((leading >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)((stride >> 4) & 0x3FFFu) << 32) | (1ull << 46);
}
// kind::f16 instruction descriptor: f32 sums, f16 operands, M = 128.
constexpr uint32_t instr_desc(int n, bool b_mn_major)
{
    return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
                 : "memory");
}
__device__ __forceinline__ void commit(uint32_t bar)
{
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n" ::"r"(bar)
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
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory"); }
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16};\n" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32])
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, "
                 "%13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, "
                 "%32};\n" ::"r"(addr),
                 "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]),
                 "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]),
                 "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
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
__device__ __forceinline__ float2 mul2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b)
{
    float2 r;
    asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
        "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}\n"
        : "=f"(r.x), "=f"(r.y)
        : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return r;
}

// Byte offset of 16-byte chunk c of row r in the core-matrix layout.
template <int D>
__device__ __forceinline__ uint32_t core_off(int r, int c)
{
    return (uint32_t)((r >> 3) * (D / 8 * 128) + c * 128 + (r & 7) * 16);
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
    extern __shared__ __align__(1024) uint8_t smem[];
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
    uint32_t *s_vmax = reinterpret_cast<uint32_t *>(smem + L::misc + 12);
    float4 *s_f = reinterpret_cast<float4 *>(smem + L::factors);

    if (warp == kSoftWarps + kConvWarps)
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
        bar_init(bar(kDrain), 1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        *gave_up = 0;
        *s_vmax = 0u;
    }
    fence_before();
    __syncthreads();
    fence_after();
    const uint32_t tmem = *tmem_slot;

    // ---- the largest value scale of the split: weights are taken relative to it
    {
        float vm = 0.0f;
        for (int e = w.e0 + tid; e < w.e1; e += kThreads)
        {
            const int blk = kv_block(p.c, w.b, e);
            if (blk >= 0)
                vm = fmaxf(vm, __ldg(p.c.vs + (uint64_t)blk * p.c.hkv + w.h));
        }
        for (int o = 16; o; o >>= 1)
            vm = fmaxf(vm, __shfl_xor_sync(kKvFull, vm, o));
        if (lane == 0 && vm > 0.0f)
            atomicMax(s_vmax, __float_as_uint(vm));
    }

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
        const float mul = power_of_two(up);
#pragma unroll
        for (int c = 0; c < D / 8; ++c)
        {
            uint32_t y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                y[e] = kv_pack<false>(kv_float<BF16>((uint16_t)x[4 * c + e]) * mul,
                                      kv_float<BF16>((uint16_t)(x[4 * c + e] >> 16)) * mul);
            *reinterpret_cast<uint4 *>(smem + L::q + (tid >> 7) * L::kTileBytes + core_off<D>(tid & 127, c)) =
                make_uint4(y[0], y[1], y[2], y[3]);
        }
        rf = live ? power_of_two(-up) * p.scale_log2 : 0.0f;
        limit = live ? min(w.s.first + i + 1, w.s.len) : 0;
        fence_smem();
    }
    __syncthreads();
    const float vref = __uint_as_float(*s_vmax);
    float m = kKvNegInf, l = 0.0f;
    bool ok = true;

    if (warp < kSoftWarps)
    {
        // ------------------------------------------------ softmax
        const int tile = warp >> 2;
        const uint32_t lanes = (uint32_t)(warp & 3) << 21; // tensor-memory lane in bits 16 and up
        const uint32_t s_addr = tmem + lanes + 128u * (uint32_t)tile;
        const uint32_t o_addr = tmem + lanes + 256u + (uint32_t)(D * tile);
        const int tile_lo = min(w.s.first + (w.r0 + 128 * tile) / G + 1, w.s.len); // least that a row of the tile sees
        for (int i = 0; i < (tile == 0 || two ? w.tiles : 0); ++i)
        {
            // the product before these scores is done as well (the tensor core works in order)
            ok = bar_wait(bar(kSFull + tile), (uint32_t)i & 1u, gave_up) &&
                 (i == 0 || bar_wait(bar(kODone + tile), (uint32_t)(i - 1) & 1u, gave_up));
            if (!__all_sync(kKvFull, ok))
            {
                ok = false;
                break;
            }
            fence_after();
            const float4 *f = s_f + (i % kFactorStages) * kGroups;
            const int pos0 = w.base + i * kTok;
            bool whole = pos0 + kTok <= tile_lo;
#pragma unroll
            for (int g = 0; g < kGroups; ++g)
                whole &= __float_as_int(f[g].z) != kMaxPos;

            // the tile's maximum; the products' factor is not negative and constant over 16 tokens
            float top = kKvNegInf;
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                uint32_t x[32];
                tmem_ld32(s_addr + 32u * c, x);
                tmem_ld_wait();
#pragma unroll
                for (int u = 0; u < 2; ++u)
                {
                    const int g = 2 * c + u;
                    const float4 fg = f[g];
                    float gm = kKvNegInf;
                    if (whole)
                    {
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            gm = fmaxf(gm, __uint_as_float(x[16 * u + e]));
                    }
                    else
                    {
                        const int left = limit - __float_as_int(fg.z); // columns of the group that the row sees
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            gm = fmaxf(gm, e < left ? __uint_as_float(x[16 * u + e]) : kKvNegInf);
                    }
                    top = fmaxf(top, gm == kKvNegInf ? kKvNegInf : gm * (fg.x * rf));
                }
            }
            const bool rise = top > m + kSlack; // from -inf: any maximum
            if (__any_sync(kKvFull, rise))
            {
                const float down = !rise ? 1.0f : exp2_fast(m - top); // from -inf: 0
                m = rise ? top : m;
                l *= down;
                if (i > 0)
                {
#pragma unroll
                    for (int c = 0; c < D / 32; ++c)
                    {
                        uint32_t x[32];
                        tmem_ld32(o_addr + 32u * c, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            x[e] = __float_as_uint(__uint_as_float(x[e]) * down);
                        tmem_st32(o_addr + 32u * c, x);
                    }
                }
            }
            const float shift_m = m == kKvNegInf ? 0.0f : kLift - m;
            // the exponent's product is not rounded where the maximum's was: beyond 2^20 that difference shows,
            // and is cut off
            const bool plain = whole && __all_sync(kKvFull, fabsf(m) < 1048576.0f);
            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
            for (int c = 0; c < 4; ++c)
            {
                uint32_t x[32], y[16];
                tmem_ld32(s_addr + 32u * c, x);
                tmem_ld_wait();
#pragma unroll
                for (int u = 0; u < 2; ++u)
                {
                    const float4 fg = f[2 * c + u];
                    const float kf = fg.x * rf;
                    const int left = plain ? 16 : limit - __float_as_int(fg.z);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                    {
                        float2 z = fma2(make_float2(__uint_as_float(x[16 * u + 2 * e]), __uint_as_float(x[16 * u + 2 * e + 1])),
                                        make_float2(kf, kf), make_float2(shift_m, shift_m));
                        if (!plain)
                        {
                            // a logit that is not a number stays one
                            z.x = z.x > kLift + kSlack ? kLift + kSlack : z.x;
                            z.y = z.y > kLift + kSlack ? kLift + kSlack : z.y;
                        }
                        z.x = exp2_fast(z.x);
                        z.y = exp2_fast(z.y);
                        if (!plain)
                        {
                            z.x = 2 * e < left ? z.x : 0.0f;
                            z.y = 2 * e + 1 < left ? z.y : 0.0f;
                        }
                        sum = add2(sum, z);
                        z = mul2(z, make_float2(fg.y, fg.y));
                        y[8 * u + e] = kv_pack<false>(z.x, z.y);
                    }
                }
                tmem_st16(s_addr + 16u * c, y);
            }
            l += sum.x + sum.y;
            tmem_st_wait();
            fence_before();
            bar_arrive(bar(kPFull + tile));
        }
        // ------------------------------------------------ out
        if (w.tiles > 0 && ok && (tile == 0 || two))
        {
            ok = bar_wait(bar(kODone + tile), (uint32_t)(w.tiles - 1) & 1u, gave_up);
            ok = __all_sync(kKvFull, ok);
            fence_after();
        }
        const int r = w.r0 + tid;
        const bool live = r < w.r1;
        const float lse2 = l == 0.0f ? kKvNegInf : m + log2f(l) - kLift;
        float f = l == 0.0f ? 0.0f : vref / l;
        if (!ok)
            f = __int_as_float(0x7FC00000);
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
                    tmem_ld_wait();
                }
                else
                {
#pragma unroll
                    for (int e = 0; e < 32; ++e)
                        x[e] = 0u;
                }
                if (!live)
                    continue;
                if (w.nsplits > 1)
                {
                    float4 *dst = reinterpret_cast<float4 *>(part + ((uint64_t)w.split * kPromptRows + tid) * D + 32 * c);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        dst[e] = make_float4(__uint_as_float(x[4 * e]) * f, __uint_as_float(x[4 * e + 1]) * f,
                                             __uint_as_float(x[4 * e + 2]) * f, __uint_as_float(x[4 * e + 3]) * f);
                }
                else
                {
                    uint4 *dst = reinterpret_cast<uint4 *>(out + 32 * c);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                    {
                        uint32_t y[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            y[k] = kv_pack<BF16>(__uint_as_float(x[8 * e + 2 * k]) * f,
                                                 __uint_as_float(x[8 * e + 2 * k + 1]) * f);
                        dst[e] = make_uint4(y[0], y[1], y[2], y[3]);
                    }
                }
            }
        }
        fence_before();
    }
    else if (warp < kSoftWarps + kConvWarps)
    {
        // ------------------------------------------------ codes to halves
        constexpr int kPairs = D / 16; // (8 tokens, 16 channels) units of a lane
        const int cw = warp - kSoftWarps;
        uint4 rk[kPairs], rv[kPairs];
        int blk[2], nblk[2];  // blocks of the warp's two groups of 16 tokens: loaded tile, next tile
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
            for (int it = 0; it < kPairs; ++it)
            {
                const int pair = it * 4 + (lane >> 3), grp = pair / (D / 16), ch = pair % (D / 16);
                const int tk = grp * 8 + (lane & 7); // token of the warp's 32
                const int at = grp >= 2 ? blk[1] : blk[0];
                const int pos = w.base + i * kTok + cw * 32 + tk;
                r[it] = make_uint4(0x80808080u, 0x80808080u, 0x80808080u, 0x80808080u);
                if (at >= 0)
                    r[it] = __ldg(reinterpret_cast<const uint4 *>(
                        pool + (uint64_t)at * stride + (uint64_t)(((w.h << shift) + (uint32_t)(pos & bs1)) * D + ch * 16)));
            }
        };
        auto convert = [&](uint8_t *tile, const uint4 (&r)[kPairs]) {
#pragma unroll
            for (int it = 0; it < kPairs; ++it)
            {
                const int pair = it * 4 + (lane >> 3), grp = pair / (D / 16), ch = pair % (D / 16);
                uint8_t *dst = tile + core_off<D>(cw * 32 + grp * 8 + (lane & 7), 2 * ch);
                const uint32_t u[4] = {r[it].x, r[it].y, r[it].z, r[it].w};
                uint32_t y[8];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                {
                    y[2 * e] = code_halves(u[e], 0x4140);
                    y[2 * e + 1] = code_halves(u[e], 0x4342);
                }
                *reinterpret_cast<uint4 *>(dst) = make_uint4(y[0], y[1], y[2], y[3]);
                *reinterpret_cast<uint4 *>(dst + 128) = make_uint4(y[4], y[5], y[6], y[7]);
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
        for (int i = 0; i < w.tiles; ++i)
        {
            const int st = i & 1;
            const uint32_t par = (uint32_t)((i >> 1) + 1) & 1u; // of the stage's release before this use
            if (i >= 2)
                ok = bar_wait(bar(kKEmpty + st), par, gave_up);
            if (!__all_sync(kKvFull, ok))
                break;
            if (lane < 2)
                s_f[(i % kFactorStages) * kGroups + cw * 2 + lane] =
                    make_float4(fk, vref > 0.0f ? fv / vref : 0.0f,
                                __int_as_float((lane ? blk[1] : blk[0]) >= 0 ? w.base + i * kTok + cw * 32 + lane * 16 : kMaxPos), 0.0f);
            convert(smem + L::k + st * L::kTileBytes, rk);
            fence_smem();
            bar_arrive(bar(kKFull + st));
            blk[0] = nblk[0];
            blk[1] = nblk[1];
            load(i + 1, p.c.k, p.c.kbs, rk);
            factors();
            if (i >= 2)
                ok = bar_wait(bar(kVEmpty + st), par, gave_up);
            if (!__all_sync(kKvFull, ok))
                break;
            convert(smem + L::v + st * L::kTileBytes, rv);
            fence_smem();
            bar_arrive(bar(kVFull + st));
            load(i + 1, p.c.v, p.c.vbs, rv);
            look(i + 2, nblk);
        }
    }
    else if (lane == 0)
    {
        // ------------------------------------------------ matrix instructions
        constexpr uint32_t kRow8 = D / 8 * 128; // from 8 rows to the next
        constexpr uint32_t kIdS = instr_desc(kTok, false), kIdO = instr_desc(D, true);
        auto scores = [&](int tile, int st) {
            const uint32_t a = sbase + L::q + (uint32_t)tile * L::kTileBytes, b = sbase + L::k + (uint32_t)st * L::kTileBytes;
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks)
                mma_ss(tmem + 128u * (uint32_t)tile, smem_desc(a + 256u * ks, 128u, kRow8),
                       smem_desc(b + 256u * ks, 128u, kRow8), kIdS, ks > 0 ? 1u : 0u);
            commit(bar(kSFull + tile));
        };
        auto values = [&](int tile, int st, bool first) {
            const uint32_t b = sbase + L::v + (uint32_t)st * L::kTileBytes;
#pragma unroll
            for (int ks = 0; ks < kTok / 16; ++ks)
                mma_ts(tmem + 256u + (uint32_t)(D * tile), tmem + 128u * (uint32_t)tile + 8u * ks,
                       smem_desc(b + 2u * kRow8 * ks, kRow8, 128u), kIdO, first && ks == 0 ? 0u : 1u);
            commit(bar(kODone + tile));
        };
        if (w.tiles > 0)
        {
            ok = bar_wait(bar(kKFull), 0u, gave_up);
            fence_after();
            if (ok)
            {
                scores(0, 0);
                if (two)
                    scores(1, 0);
                commit(bar(kKEmpty));
            }
        }
        for (int i = 0; ok && i < w.tiles; ++i)
        {
            const int st = i & 1, sn = st ^ 1;
            const uint32_t par = (uint32_t)(i >> 1) & 1u, parn = (uint32_t)((i + 1) >> 1) & 1u;
            const bool more = i + 1 < w.tiles;
            if (!(ok = bar_wait(bar(kVFull + st), par, gave_up)))
                break;
            if (!(ok = bar_wait(bar(kPFull), (uint32_t)i & 1u, gave_up)))
                break;
            fence_after();
            values(0, st, i == 0);
            if (more)
            {
                if (!(ok = bar_wait(bar(kKFull + sn), parn, gave_up)))
                    break;
                fence_after();
                scores(0, sn);
            }
            if (two)
            {
                if (!(ok = bar_wait(bar(kPFull + 1), (uint32_t)i & 1u, gave_up)))
                    break;
                fence_after();
                values(1, st, i == 0);
            }
            commit(bar(kVEmpty + st));
            if (more)
            {
                if (two)
                    scores(1, sn);
                commit(bar(kKEmpty + sn));
            }
        }
    }
    __syncwarp();
    __syncthreads();
    if (*gave_up)
    {
        // matrix instructions in flight when a wait ran out get a bounded time to end
        if (tid == 32 * (kSoftWarps + kConvWarps))
        {
            atomicAdd(&g_kv_prompt_timeouts, 1u);
            commit(bar(kDrain));
            for (uint32_t it = 0; it < kWaitLimit && !bar_try(bar(kDrain), 0u); ++it)
            {
            }
        }
        __syncthreads();
    }
    if (w.nsplits > 1)
    {
        // ---- the splits are joined by the block that comes last, in their order
        const int item = (int)((w.b * p.c.hkv + w.h) * p.row_tiles + rt);
        const float *part = p.part + (uint64_t)item * p.splits * kPromptRows * (D + 1);
        const float *part_lse = part + (uint64_t)p.splits * kPromptRows * D;
        __threadfence();
        __syncthreads();
        if (tid == 0)
            *s_last = atomicAdd(p.counters + item, 1u) == (uint32_t)w.nsplits - 1u;
        __syncthreads();
        if (*s_last)
        {
            __threadfence();
            if (tid == 0)
                p.counters[item] = 0u;
            uint16_t *out = reinterpret_cast<uint16_t *>(p.out);
            // a warp per row, a lane per 4 channels
            for (int r = warp; w.r0 + r < w.r1; r += kThreads / 32)
            {
                const int i = (w.r0 + r) / G, hd = (int)w.h * G + (w.r0 + r) % G;
                float top = kKvNegInf, sum = 0.0f;
                for (int k = 0; k < w.nsplits; ++k)
                    top = fmaxf(top, __ldcg(part_lse + k * kPromptRows + r));
                const float ref = top == kKvNegInf ? 0.0f : top;
                float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
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
                    *reinterpret_cast<uint2 *>(out + at * D + 4 * lane) =
                        make_uint2(kv_pack<BF16>(y.x * f, y.y * f), kv_pack<BF16>(y.z * f, y.w * f));
                if (lane == 0 && p.lse)
                    p.lse[at] = (sum == 0.0f ? kKvNegInf : ref + log2f(sum)) * 0.69314718056f;
            }
        }
    }
    fence_after();
    __syncthreads();
    if (warp == kSoftWarps + kConvWarps)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512u) : "memory");
}

template <int D, bool BF16>
int launch(const AttnParams &p, uint32_t blocks_x, cudaStream_t st)
{
    static const cudaError_t attr = cudaFuncSetAttribute(prompt_kernel<D, BF16>,
                                                         cudaFuncAttributeMaxDynamicSharedMemorySize, Layout<D>::bytes);
    DANCE_CUDA(attr);
    prompt_kernel<D, BF16><<<dim3(blocks_x, p.c.batch), kThreads, Layout<D>::bytes, st>>>(p);
    DANCE_LAUNCHED();
    return 0;
}

} // namespace

int launch_prompt(const AttnParams &p, uint32_t head_dim, bool bf16, uint32_t blocks_x, cudaStream_t st)
{
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

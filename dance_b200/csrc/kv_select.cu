// kv_select.cu -- the blocks of the 8-bit key/value cache that each row reads
// (dance_kv_select_blocks, include/dance_b200.h).
//
// Score.  No key of a block lies outside the block's bounds, so
//   q . k <= sum_d max(q_d low_d, q_d high_d),
// for the query in 8 bits an integer.  With c+ and c- the positive and the
// negative part of the query's codes the sum is one product of length 2 D,
//   c+ . high + c- . low,
// and the bounds' offset of 128 comes out of it as 128 * sum_d c_d.  The order
// of an integer sum does not show, so the choice is the same however it is
// summed.
//
// Floor: the bounds' 2 * head_dim bytes of every (block, head), once.  Measured:
// 32 sequences of up to 1875 blocks, 8 heads of 128 channels (54.7 MB): 28 us,
// scores 19 (2.9 TB/s), choice 6, a launch between them.  700 rows of one
// sequence, 24 heads of 96, 2049 blocks: 94 us, scores 46, choice 47;
// latency and instructions bound both there (54 and 76 % of the issue slots), not
// the 4 us that bytes and products need.
//
// scores_kernel writes the float scores of (row, head, block) from integer
// matrix instructions, choose_kernel finds each (row, head)'s threshold in
// histograms of the order-preserving keys and writes the chosen blocks in
// ascending order.
#include "kv_common.cuh"

namespace dance
{
namespace
{

constexpr int kScoreThreads = 128;
constexpr int kScoreBlocks = 128; // cache blocks of one pass of a thread block: 32 per warp
constexpr int kScoreHeads = 8;    // query heads in shared memory at once
constexpr int kChooseThreads = 256;
constexpr int kBins = 2048;
constexpr uint32_t kChooseKeys = 9728; // keys that the choice holds in shared memory

struct SelectParams
{
    KvView c;
    const uint16_t *q;
    uint64_t q_row, q_head;
    bool q_aligned;
    uint32_t rows, heads, G;
    uint32_t nblk;      // blocks that a row can see
    uint32_t width;     // floats from one (row, head)'s scores to the next
    uint32_t row_tiles; // of a sequence
    uint32_t passes;    // runs of blocks of a thread block
    uint32_t slots;     // query heads in shared memory at once
    uint32_t select, first, last;
    float *scores; // rows x hkv x nblk
    int32_t *out;
};

__device__ __forceinline__ void mma_u8s8(int (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.u8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};\n"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Bytes of a query row in shared memory: 2 D codes, padded so that two rows
// of 64 bytes lie on different banks.
template <int D>
constexpr int code_stride()
{
    return (2 * D) % 128 == 64 ? 2 * D : 2 * D + 64;
}

// Scores of 8 * NT rows of one sequence and one key/value head against
// `passes` runs of 128 blocks.  Blocks lie on the 16-row side of the matrix
// instruction, the rows of one query head on its 8-column side, so that the
// maximum over the query heads stays in the accumulator's lane.  A warp keeps
// the bounds of its 32 blocks in registers through all heads and rows; a lane
// takes adjacent bytes, the order of the channels in the sum being free.
//
// Latency bounds it (prologue, then bounds loaded in their turn), so blocks an
// SM count most: 700 rows x 24 heads x 2049 blocks of 96 channels took 61 us
// with 32 rows a block and no register bound, 53 with four blocks an SM, 46
// with 16 rows and four, 50 with five (spills); 8 and 64 rows were slower.
template <int D, int NT, bool BF16>
__global__ void __launch_bounds__(kScoreThreads, 4) scores_kernel(SelectParams p)
{
    extern __shared__ __align__(16) uint8_t smem[];
    constexpr int kRows = 8 * NT, kStride = code_stride<D>(), kChunks = 2 * D / 64;
    float *qs_s = reinterpret_cast<float *>(smem + p.slots * kRows * kStride);
    int *init_s = reinterpret_cast<int *>(qs_s + p.slots * kRows);
    const uint32_t b = blockIdx.z, h = blockIdx.y;
    const int tile = (int)(blockIdx.x % p.row_tiles), i0 = tile * kRows;
    const int jbeg = (int)(blockIdx.x / p.row_tiles) * (int)p.passes * kScoreBlocks;
    const KvSeq s = kv_seq(p.c, b, p.rows);
    if (i0 >= s.rows)
        return;
    const int i1 = min(i0 + kRows, s.rows);
    const int seen = min(s.first + i1, s.len);
    const int nb = (max(seen, 0) + (1 << p.c.shift) - 1) >> p.c.shift;
    const int jend = min(jbeg + (int)p.passes * kScoreBlocks, nb);
    if (jbeg >= nb)
        return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;

    for (int j0 = jbeg; j0 < jend; j0 += kScoreBlocks)
    {
        uint32_t w[2][2][4 * kChunks]; // bounds of blocks (tile, g or g + 8)
        float ks[2][2];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int u = 0; u < 2; ++u)
            {
                const int j = j0 + warp * 32 + mt * 16 + u * 8 + g;
                const int blk = j < jend ? kv_block(p.c, b, j) : -1;
                const uint64_t si = (uint64_t)max(blk, 0) * p.c.hkv + h;
                const uint4 *src = reinterpret_cast<const uint4 *>(p.c.bounds + si * 2 * D) + t;
#pragma unroll
                for (int i = 0; i < kChunks; ++i)
                    *reinterpret_cast<uint4 *>(&w[mt][u][4 * i]) =
                        blk >= 0 ? __ldg(src + 4 * i) : make_uint4(0u, 0u, 0u, 0u);
                ks[mt][u] = blk >= 0 ? __ldg(p.c.ks + si) : -1.0f;
            }
        float best[2][NT][4];
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
                best[mt][n][0] = best[mt][n][1] = best[mt][n][2] = best[mt][n][3] = kKvNegInf;
        for (uint32_t g0 = 0; g0 < p.G; g0 += kScoreHeads)
        {
            const int ng = (int)min((uint32_t)kScoreHeads, p.G - g0);
            if (j0 == jbeg || p.G > kScoreHeads)
            {
                __syncthreads();
                // queries in 8 bits: eight lanes a row, c- (which meets the lower bounds) before c+
                for (int e = threadIdx.x >> 3; e < ng * kRows; e += kScoreThreads / 8)
                {
                    const int hd = e / kRows, i = i0 + e % kRows, l8 = threadIdx.x & 7;
                    const bool live = i < i1;
                    const uint16_t *src = p.q + (uint64_t)(s.row0 + (live ? i : i0)) * p.q_row +
                                          (uint64_t)(h * p.G + g0 + hd) * p.q_head + l8 * (D / 8);
                    alignas(8) uint16_t raw[D / 8];
                    if (p.q_aligned) // 8 bytes at a time: D / 8 elements are 16, 24 or 32 bytes
                    {
#pragma unroll
                        for (int k = 0; k < D / 32; ++k)
                            *reinterpret_cast<uint2 *>(&raw[4 * k]) = __ldg(reinterpret_cast<const uint2 *>(src) + k);
                    }
                    else
                    {
#pragma unroll
                        for (int k = 0; k < D / 8; ++k)
                            raw[k] = __ldg(src + k);
                    }
                    float x[D / 8], amax = 0.0f;
#pragma unroll
                    for (int k = 0; k < D / 8; ++k)
                    {
                        x[k] = live ? kv_float<BF16>(raw[k]) : 0.0f;
                        amax = fmaxf(amax, kv_finite_abs(x[k]));
                    }
                    const unsigned eight = 0xFFu << (threadIdx.x & 24);
                    for (int o = 4; o; o >>= 1)
                        amax = fmaxf(amax, __shfl_xor_sync(eight, amax, o));
                    const float qs = kv_step_of(amax), inv = kv_inverse(qs);
                    int sum = 0;
                    uint8_t *dst = smem + (hd * kRows + e % kRows) * kStride + l8 * (D / 8);
#pragma unroll
                    for (int k = 0; k < D / 8; k += 4)
                    {
                        uint32_t lo = 0u, hi = 0u;
#pragma unroll
                        for (int y = 0; y < 4; ++y)
                        {
                            const int c = kv_code(x[k + y], inv);
                            sum += c;
                            lo |= ((uint32_t)min(c, 0) & 255u) << (8 * y);
                            hi |= (uint32_t)max(c, 0) << (8 * y);
                        }
                        *reinterpret_cast<uint32_t *>(dst + k) = lo;
                        *reinterpret_cast<uint32_t *>(dst + D + k) = hi;
                    }
                    for (int o = 4; o; o >>= 1)
                        sum += __shfl_xor_sync(eight, sum, o);
                    if (l8 == 0)
                    {
                        qs_s[hd * kRows + e % kRows] = qs;
                        init_s[hd * kRows + e % kRows] = -128 * sum;
                    }
                }
                __syncthreads();
            }
            for (int hd = 0; hd < ng; ++hd)
            {
#pragma unroll
                for (int n = 0; n < NT; ++n)
                {
                    const int r = hd * kRows + 8 * n;
                    const uint8_t *src = smem + (r + g) * kStride + t * 16;
                    const int2 init = *reinterpret_cast<const int2 *>(init_s + r + 2 * t);
                    const float2 qs = *reinterpret_cast<const float2 *>(qs_s + r + 2 * t);
                    int acc[2][4];
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
                    {
                        acc[mt][0] = acc[mt][2] = init.x;
                        acc[mt][1] = acc[mt][3] = init.y;
                    }
#pragma unroll
                    for (int i = 0; i < kChunks; ++i)
                    {
                        const uint4 q = *reinterpret_cast<const uint4 *>(src + 64 * i);
#pragma unroll
                        for (int mt = 0; mt < 2; ++mt)
                        {
                            mma_u8s8(acc[mt], w[mt][0][4 * i], w[mt][1][4 * i], w[mt][0][4 * i + 1],
                                     w[mt][1][4 * i + 1], q.x, q.y);
                            mma_u8s8(acc[mt], w[mt][0][4 * i + 2], w[mt][1][4 * i + 2], w[mt][0][4 * i + 3],
                                     w[mt][1][4 * i + 3], q.z, q.w);
                        }
                    }
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            best[mt][n][k] =
                                fmaxf(best[mt][n][k], __fmul_rn((float)acc[mt][k], k & 1 ? qs.y : qs.x));
                }
            }
        }
#pragma unroll
        for (int mt = 0; mt < 2; ++mt)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k)
                {
                    const int i = i0 + 8 * n + 2 * t + (k & 1);
                    const int j = j0 + warp * 32 + mt * 16 + (k >> 1) * 8 + g;
                    const float f = ks[mt][k >> 1];
                    if (i < i1 && j < jend)
                        p.scores[((uint64_t)(s.row0 + i) * p.c.hkv + h) * p.width + j] =
                            f >= 0.0f ? __fmul_rn(best[mt][n][k], f) : kKvNegInf;
                }
    }
}

// Order-preserving key of a score (-0 counts as 0).
__device__ __forceinline__ uint32_t score_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f);
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

// One thread block per (row, head).  The keys' range is cut into 2048 equal
// bins; the bin in which the count from above passes what is still needed is
// cut again until it is taken whole or holds one value (three cuts at most).
// Equal cuts of the actual range fill more bins than digits of the key would,
// whose leading bits hardly differ: fewer shared-memory atomics meet.
template <bool SHARED>
__global__ void __launch_bounds__(kChooseThreads) choose_kernel(SelectParams p)
{
    extern __shared__ uint32_t keys_s[];
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t s_red[2][kChooseThreads / 32];
    __shared__ uint32_t s_bin, s_need, s_count;
    __shared__ uint64_t s_scan[kChooseThreads / 32];
    const uint32_t b = blockIdx.y, h = blockIdx.x % p.c.hkv;
    const int i = (int)(blockIdx.x / p.c.hkv), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KvSeq s = kv_seq(p.c, b, p.rows);
    if (i >= s.rows)
        return;
    const uint64_t rh = (uint64_t)(s.row0 + i) * p.c.hkv + h;
    int32_t *out = p.out + rh * p.select;
    const int seen = min(s.first + i + 1, s.len);
    const int nb = min((max(seen, 0) + (1 << p.c.shift) - 1) >> p.c.shift, (int)p.nblk);
    const int k = (int)p.select;
    if (nb <= k)
    {
        for (int e = tid; e < k; e += kChooseThreads)
            out[e] = e < nb ? e : -1;
        return;
    }
    const float *sc = p.scores + rh * p.width;
    const int lo = (int)p.first, hi = nb - (int)p.last; // the blocks that compete
    uint32_t need = (uint32_t)(k - (int)p.first - (int)p.last);
    auto key_of = [&](int j) { return SHARED ? keys_s[j] : score_key(__ldg(sc + j)); };

    uint32_t least = 0xFFFFFFFFu, most = 0u;
    for (int j = lo + tid; j < hi; j += kChooseThreads)
    {
        const uint32_t key = score_key(__ldg(sc + j));
        if (SHARED)
            keys_s[j] = key;
        least = min(least, key);
        most = max(most, key);
    }
    for (int e = tid; e < kBins; e += kChooseThreads)
        hist[e] = 0u;
    least = __reduce_min_sync(kKvFull, least);
    most = __reduce_max_sync(kKvFull, most);
    if (lane == 0)
    {
        s_red[0][warp] = least;
        s_red[1][warp] = most;
    }
    __syncthreads();
    for (int w = 0; w < kChooseThreads / 32; ++w)
    {
        least = min(least, s_red[0][w]);
        most = max(most, s_red[1][w]);
    }
    // taken: keys above `top`; of the keys in [least, top] the first `need` in block order
    uint32_t top = need ? most : 0xFFFFFFFFu;
    if (!need)
        least = 0xFFFFFFFFu;
    while (need)
    {
        const uint32_t span = top - least;
        const int shift = max(0, 21 - __clz(span)); // span >> shift < 2048
        for (int j = lo + tid; j < hi; j += kChooseThreads)
        {
            const uint32_t key = key_of(j);
            if (key >= least && key <= top)
                atomicAdd(&hist[(key - least) >> shift], 1u);
        }
        __syncthreads();
        // thread t holds eight bins, the highest bins first
        uint32_t c[kBins / kChooseThreads], sum = 0;
#pragma unroll
        for (int e = 0; e < kBins / kChooseThreads; ++e)
        {
            uint32_t *at = &hist[kBins - 1 - tid * (kBins / kChooseThreads) - e];
            sum += c[e] = *at;
            *at = 0u;
        }
        uint32_t above = sum;
        for (int o = 1; o < 32; o <<= 1)
        {
            const uint32_t y = __shfl_up_sync(kKvFull, above, o);
            above += lane >= o ? y : 0u;
        }
        if (lane == 31)
            s_red[0][warp] = above;
        __syncthreads();
        above -= sum;
        for (int w = 0; w < warp; ++w)
            above += s_red[0][w];
#pragma unroll
        for (int e = 0; e < kBins / kChooseThreads; ++e)
        {
            if (above < need && above + c[e] >= need)
            {
                s_bin = (uint32_t)(kBins - 1 - tid * (kBins / kChooseThreads) - e);
                s_need = need - above;
                s_count = c[e];
            }
            above += c[e];
        }
        __syncthreads();
        need = s_need;
        const uint32_t base = least + (s_bin << shift);
        top = (uint32_t)min((uint64_t)top, (uint64_t)base + ((1u << shift) - 1u));
        least = base;
        if (s_count == need || shift == 0)
            break;
    }
    __syncthreads();

    // every thread writes a run of blocks, behind what the threads before it write
    const int per = ((nb + kChooseThreads - 1) / kChooseThreads) | 1;
    const int ja = min(tid * per, nb), jb = min(ja + per, nb);
    uint64_t mine = 0; // (keys in [least, top]) << 32 | (keys above, blocks always taken)
    for (int j = ja; j < jb; ++j)
    {
        const bool always = j < lo || j >= hi;
        const uint32_t key = always ? 0u : key_of(j);
        mine += always || key > top ? 1ull : (need && key >= least ? 1ull << 32 : 0ull);
    }
    uint64_t incl = mine;
    for (int o = 1; o < 32; o <<= 1)
    {
        const uint64_t y = __shfl_up_sync(kKvFull, incl, o);
        incl += lane >= o ? y : 0ull;
    }
    if (lane == 31)
        s_scan[warp] = incl;
    __syncthreads();
    uint64_t before = incl - mine;
    for (int w = 0; w < warp; ++w)
        before += s_scan[w];
    uint32_t sure = (uint32_t)before, maybe = (uint32_t)(before >> 32);
    for (int j = ja; j < jb; ++j)
    {
        const bool always = j < lo || j >= hi;
        const uint32_t key = always ? 0u : key_of(j);
        if (always || key > top)
            out[min(sure++ + min(maybe, need), (uint32_t)k - 1u)] = j;
        else if (need && key >= least && maybe++ < need)
            out[min(sure + maybe - 1u, (uint32_t)k - 1u)] = j;
    }
}

// The same choice for up to 4096 blocks, the keys in registers (KPT of a
// thread, four adjacent blocks at a time): one read of the scores, and the
// ranks of all runs from one scan of packed 16-bit counts.
template <int KPT>
__global__ void __launch_bounds__(kChooseThreads) choose_short_kernel(SelectParams p)
{
    constexpr int kRuns = KPT / 4, kPer = kBins / kChooseThreads;
    static_assert(kRuns <= 4 && kPer == 8, "16-bit fields of the ranks, two vectors of bins");
    __shared__ __align__(16) uint32_t hist[kBins];
    __shared__ uint32_t s_least[kChooseThreads / 32], s_most[kChooseThreads / 32], s_above[kChooseThreads / 32];
    __shared__ uint32_t s_bin, s_need, s_count;
    __shared__ __align__(16) uint4 s_ranks[kChooseThreads / 32];
    const uint32_t b = blockIdx.y, h = blockIdx.x % p.c.hkv;
    const int i = (int)(blockIdx.x / p.c.hkv), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KvSeq s = kv_seq(p.c, b, p.rows);
    if (i >= s.rows)
        return;
    const uint64_t rh = (uint64_t)(s.row0 + i) * p.c.hkv + h;
    int32_t *out = p.out + rh * p.select;
    const int seen = min(s.first + i + 1, s.len);
    const int nb = min((max(seen, 0) + (1 << p.c.shift) - 1) >> p.c.shift, (int)p.nblk);
    const int k = (int)p.select;
    if (nb <= k)
    {
        for (int e = tid; e < k; e += kChooseThreads)
            out[e] = e < nb ? e : -1;
        return;
    }
    const float4 *sc = reinterpret_cast<const float4 *>(p.scores + rh * p.width);
    const int lo = (int)p.first, hi = nb - (int)p.last; // the blocks that compete
    uint32_t need = (uint32_t)(k - (int)p.first - (int)p.last);
    // Blocks that are always taken get the largest key, places without a block 0: below every score's key, so that
    // comparisons of keys are all that follows.
    const int runs = (nb + 4 * kChooseThreads - 1) / (4 * kChooseThreads);
    uint32_t key[KPT], least = 0xFFFFFFFFu, most = 0u;
#pragma unroll
    for (int r = 0; r < kRuns; ++r)
    {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            key[4 * r + e] = 0u;
        if (r < runs)
        {
            const int q = tid + kChooseThreads * r;
            const float4 v = 4 * q < nb ? __ldg(sc + q) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            const float x[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
            {
                const int j = 4 * q + e;
                if (j >= lo && j < hi)
                {
                    key[4 * r + e] = min(score_key(x[e]), 0xFFFFFFFEu);
                    least = min(least, key[4 * r + e]);
                    most = max(most, key[4 * r + e]);
                }
                else if (j < nb)
                    key[4 * r + e] = 0xFFFFFFFFu;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 2; ++e)
        reinterpret_cast<uint4 *>(hist)[tid * 2 + e] = make_uint4(0u, 0u, 0u, 0u);
    least = __reduce_min_sync(kKvFull, least);
    most = __reduce_max_sync(kKvFull, most);
    if (lane == 0)
    {
        s_least[warp] = least;
        s_most[warp] = most;
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kChooseThreads / 32; ++w)
    {
        least = min(least, s_least[w]);
        most = max(most, s_most[w]);
    }
    // taken: keys above `top`; of the keys in [least, top] the first `need` in block order
    uint32_t top = need ? most : 0xFFFFFFFEu;
    if (!need)
        least = 0xFFFFFFFEu;
    while (need)
    {
        const uint32_t span = top - least;
        const int shift = max(0, 21 - __clz(span)); // span >> shift < 2048
#pragma unroll
        for (int r = 0; r < kRuns; ++r)
            if (r < runs)
            {
#pragma unroll
                for (int e = 4 * r; e < 4 * r + 4; ++e)
                    if (key[e] - least <= span)
                        atomicAdd(&hist[(key[e] - least) >> shift], 1u);
            }
        __syncthreads();
        // thread t holds eight bins, the highest bins first
        uint4 *mine = reinterpret_cast<uint4 *>(hist) + (kChooseThreads - 1 - tid) * 2;
        const uint4 c1 = mine[1], c0 = mine[0];
        const uint32_t c[kPer] = {c1.w, c1.z, c1.y, c1.x, c0.w, c0.z, c0.y, c0.x};
        mine[0] = mine[1] = make_uint4(0u, 0u, 0u, 0u);
        uint32_t sum = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e)
            sum += c[e];
        uint32_t above = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const uint32_t y = __shfl_up_sync(kKvFull, above, o);
            above += lane >= o ? y : 0u;
        }
        if (lane == 31)
            s_above[warp] = above;
        __syncthreads();
        above -= sum;
        for (int w = 0; w < warp; ++w)
            above += s_above[w];
        if (above < need && above + sum >= need)
        {
#pragma unroll
            for (int e = 0; e < kPer; ++e)
            {
                if (above < need && above + c[e] >= need)
                {
                    s_bin = (uint32_t)(kBins - 1 - tid * kPer - e);
                    s_need = need - above;
                    s_count = c[e];
                }
                above += c[e];
            }
        }
        __syncthreads();
        need = s_need;
        const uint32_t base = least + (s_bin << shift);
        top = (uint32_t)min((uint64_t)top, (uint64_t)base + ((1u << shift) - 1u));
        least = base;
        if (s_count == need || shift == 0)
            break;
    }

    // ranks in block order: run by run, thread by thread; 16 bits for each run
    const uint32_t span = top - least;
    uint32_t sure[2] = {0u, 0u}, maybe[2] = {0u, 0u};
#pragma unroll
    for (int r = 0; r < kRuns; ++r)
        if (r < runs)
        {
#pragma unroll
            for (int e = 4 * r; e < 4 * r + 4; ++e)
            {
                sure[r >> 1] += key[e] > top ? 1u << (16 * (r & 1)) : 0u;
                maybe[r >> 1] += key[e] - least <= span ? 1u << (16 * (r & 1)) : 0u;
            }
        }
    uint32_t sure_to[2] = {sure[0], sure[1]}, maybe_to[2] = {maybe[0], maybe[1]};
    constexpr int kWords = (kRuns + 1) / 2;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1)
#pragma unroll
        for (int w = 0; w < kWords; ++w)
        {
            const uint32_t y = __shfl_up_sync(kKvFull, sure_to[w], o), z = __shfl_up_sync(kKvFull, maybe_to[w], o);
            sure_to[w] += lane >= o ? y : 0u;
            maybe_to[w] += lane >= o ? z : 0u;
        }
    if (lane == 31)
        s_ranks[warp] = make_uint4(sure_to[0], sure_to[1], maybe_to[0], maybe_to[1]);
    __syncthreads();
    uint4 all = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
    for (int w = 0; w < kWords; ++w)
    {
        sure_to[w] -= sure[w];
        maybe_to[w] -= maybe[w];
    }
#pragma unroll
    for (int w = 0; w < kChooseThreads / 32; ++w)
    {
        const uint4 y = s_ranks[w];
        if (w < warp)
        {
            sure_to[0] += y.x, sure_to[1] += y.y;
            maybe_to[0] += y.z, maybe_to[1] += y.w;
        }
        all.x += y.x, all.y += y.y, all.z += y.z, all.w += y.w;
    }
    uint32_t sure_base = 0, maybe_base = 0;
#pragma unroll
    for (int r = 0; r < kRuns; ++r)
        if (r < runs)
        {
            const int sh = 16 * (r & 1);
            uint32_t a = sure_base + ((sure_to[r >> 1] >> sh) & 0xFFFFu);
            uint32_t m = maybe_base + ((maybe_to[r >> 1] >> sh) & 0xFFFFu);
#pragma unroll
            for (int e = 4 * r; e < 4 * r + 4; ++e)
            {
                const int j = 4 * (tid + kChooseThreads * r) + (e & 3);
                const bool in = key[e] - least <= span;
                if (key[e] > top || (in && m < need))
                    out[min(a + min(m, need), (uint32_t)k - 1u)] = j;
                a += key[e] > top;
                m += in;
            }
            sure_base += ((r >> 1 ? all.y : all.x) >> sh) & 0xFFFFu;
            maybe_base += ((r >> 1 ? all.w : all.z) >> sh) & 0xFFFFu;
        }
}

uint32_t score_blocks(const DanceKvCache &c, const DanceKvBatch &b)
{
    const uint64_t n = ((uint64_t)b.max_len + c.block_tokens - 1) / c.block_tokens;
    return (uint32_t)(n < b.table_width ? n : b.table_width);
}

// Floats from one (row, head)'s scores to the next: whole sectors.
uint32_t score_width(uint32_t nblk) { return (nblk + 7u) & ~7u; }

template <int D, int NT>
int launch_scores(SelectParams &p, bool bf16, cudaStream_t st)
{
    p.row_tiles = (p.c.max_rows + 8 * NT - 1) / (8 * NT);
    const uint32_t runs = (p.nblk + kScoreBlocks - 1) / kScoreBlocks;
    const uint64_t tiles = (uint64_t)p.row_tiles * p.c.hkv * p.c.batch;
    // runs of one thread block: one, unless there is work for several waves without
    p.passes = (uint32_t)(tiles * runs >= 4 * 4 * 148 ? min(4u, runs) : 1u);
    const dim3 grid(p.row_tiles * ((runs + p.passes - 1) / p.passes), p.c.hkv, p.c.batch);
    constexpr int per_head = 8 * NT * (code_stride<D>() + 8);
    static_assert(kScoreHeads * per_head <= 48 * 1024, "more shared memory would have to be asked for");
    p.slots = min(p.G, (uint32_t)kScoreHeads);
    const int smem = (int)p.slots * per_head;
    if (bf16)
        scores_kernel<D, NT, true><<<grid, kScoreThreads, smem, st>>>(p);
    else
        scores_kernel<D, NT, false><<<grid, kScoreThreads, smem, st>>>(p);
    DANCE_LAUNCHED();
    return 0;
}

template <int D>
int launch_select(SelectParams &p, bool bf16, cudaStream_t st)
{
    if (p.nblk > p.select)
        if (int rc = p.c.max_rows <= 8 ? launch_scores<D, 1>(p, bf16, st) : launch_scores<D, 2>(p, bf16, st))
            return rc;
    const dim3 grid(p.c.max_rows * p.c.hkv, p.c.batch);
    if (p.nblk <= 4 * kChooseThreads)
        choose_short_kernel<4><<<grid, kChooseThreads, 0, st>>>(p);
    else if (p.nblk <= 8 * kChooseThreads)
        choose_short_kernel<8><<<grid, kChooseThreads, 0, st>>>(p);
    else if (p.nblk <= 16 * kChooseThreads)
        choose_short_kernel<16><<<grid, kChooseThreads, 0, st>>>(p);
    else if (p.nblk <= kChooseKeys)
        choose_kernel<true><<<grid, kChooseThreads, p.nblk * 4, st>>>(p);
    else
        choose_kernel<false><<<grid, kChooseThreads, 0, st>>>(p);
    DANCE_LAUNCHED();
    return 0;
}

} // namespace

uint64_t kv_select_bytes(const DanceKvCache &c, const DanceKvBatch &b, uint32_t rows)
{
    return (uint64_t)rows * c.kv_heads * score_width(score_blocks(c, b)) * 4u;
}
uint64_t kv_attention_bytes(const DanceKvCache &c, const DanceKvBatch &b, uint32_t heads, uint32_t select);
uint64_t kv_counter_bytes();

} // namespace dance

using namespace dance;

extern "C" int dance_kv_select_blocks(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *q,
                                      uint32_t num_heads, uint32_t select, uint32_t first_blocks, uint32_t last_blocks,
                                      int32_t *d_blocks, void *d_workspace, uint64_t workspace_bytes, void *stream)
{
    if (int rc = kv_check(cache, batch))
        return rc;
    if (int rc = kv_check_rows(q, "q"))
        return rc;
    if (num_heads == 0 || num_heads % cache->kv_heads || num_heads > 65536)
        return fail(-1, "num_heads %u must be a multiple of kv_heads %u", num_heads, cache->kv_heads);
    if (select == 0 || select > 4096)
        return fail(-1, "select %u: 1 to 4096 are supported", select);
    if ((uint64_t)first_blocks + last_blocks > select)
        return fail(-1, "%u first and %u last blocks do not fit select %u", first_blocks, last_blocks, select);
    if (q->rows == 0 || batch->max_rows == 0)
        return 0;
    if (!d_blocks || (uintptr_t)d_blocks % 4)
        return fail(-1, "null or misaligned output");
    if ((uint64_t)batch->max_rows * cache->kv_heads > 0x7FFFFFFFull ||
        (uint64_t)(batch->max_rows / 8 + 1) * (score_blocks(*cache, *batch) / kScoreBlocks + 1) > 0x7FFFFFFFull)
        return fail(-1, "call too large: max_rows %u, %u heads, %u blocks", batch->max_rows, cache->kv_heads,
                    score_blocks(*cache, *batch));
    const uint64_t need = kv_counter_bytes() + kv_select_bytes(*cache, *batch, q->rows);
    if (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < need)
        return fail(-1, "workspace of %llu bytes: %llu are needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)need);
    SelectParams p;
    p.c = kv_view(*cache, *batch);
    p.q = reinterpret_cast<const uint16_t *>(q->d_data);
    p.q_row = q->row_stride;
    p.q_head = q->head_stride;
    p.q_aligned = kv_aligned(*q);
    p.rows = q->rows;
    p.heads = num_heads;
    p.G = num_heads / cache->kv_heads;
    p.nblk = score_blocks(*cache, *batch);
    p.width = score_width(p.nblk);
    p.select = select;
    p.first = first_blocks;
    p.last = last_blocks;
    p.scores = reinterpret_cast<float *>(reinterpret_cast<uint8_t *>(d_workspace) + kv_counter_bytes());
    p.out = d_blocks;
    const bool bf16 = q->dtype == DANCE_BF16;
    switch (cache->head_dim)
    {
    case 64:
        return launch_select<64>(p, bf16, as_stream(stream));
    case 96:
        return launch_select<96>(p, bf16, as_stream(stream));
    default:
        return launch_select<128>(p, bf16, as_stream(stream));
    }
}

extern "C" uint64_t dance_kv_workspace_bytes(const DanceKvCache *cache, const DanceKvBatch *batch, uint32_t rows,
                                             uint32_t num_heads, uint32_t select)
{
    if (kv_check(cache, batch) || num_heads == 0 || num_heads % cache->kv_heads || select > 4096)
        return 0;
    const uint64_t a = kv_attention_bytes(*cache, *batch, num_heads, select);
    const uint64_t s = select ? kv_counter_bytes() + kv_select_bytes(*cache, *batch, rows) : 0;
    return a > s ? a : s;
}

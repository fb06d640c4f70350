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
// scores_kernel writes the float scores of (row, head, block); choose_kernel
// finds each (row, head)'s select-th largest key by a radix search over four
// bytes and writes the chosen blocks in ascending order.
#include "kv_common.cuh"

namespace dance
{
namespace
{

constexpr int kScoreThreads = 128;
constexpr int kScoreHeads = 8; // query heads scored together
constexpr int kChooseThreads = 256;

struct SelectParams
{
    KvView c;
    const uint16_t *q;
    uint64_t q_row, q_head;
    uint32_t rows, heads, G;
    uint32_t nblk; // scores of a (row, head)
    uint32_t select, first, last;
    float *scores; // rows x hkv x nblk
    int32_t *out;
};

// One thread block per (row, head, 128 blocks), one thread per block.
template <int D, bool BF16>
__global__ void __launch_bounds__(kScoreThreads) scores_kernel(SelectParams p)
{
    __shared__ __align__(16) uint32_t c_s[kScoreHeads][D / 2]; // c+ of the channels, then c-
    __shared__ float qs_s[kScoreHeads];
    __shared__ int sum_s[kScoreHeads];
    const uint32_t b = blockIdx.z, h = blockIdx.y % p.c.hkv;
    const int i = (int)(blockIdx.y / p.c.hkv);
    const KvSeq s = kv_seq(p.c, b, p.rows);
    if (i >= s.rows)
        return;
    const int seen = min(s.first + i + 1, s.len);
    const int nb = (max(seen, 0) + (1 << p.c.shift) - 1) >> p.c.shift;
    const int j0 = (int)blockIdx.x * kScoreThreads;
    if (j0 >= nb)
        return;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int j = j0 + (int)threadIdx.x;
    const int blk = j < nb ? kv_block(p.c, b, j) : -1;
    uint4 w[D / 8];
    if (blk >= 0)
    {
        const uint4 *src = reinterpret_cast<const uint4 *>(p.c.bounds + ((uint64_t)blk * p.c.hkv + h) * 2 * D);
#pragma unroll
        for (int e = 0; e < D / 8; ++e)
            w[e] = __ldg(src + e);
    }
    const float ks = blk >= 0 ? __ldg(p.c.ks + (uint64_t)blk * p.c.hkv + h) : 0.0f;
    float best = kKvNegInf;
    for (uint32_t g0 = 0; g0 < p.G; g0 += kScoreHeads)
    {
        const int ng = (int)min((uint32_t)kScoreHeads, p.G - g0);
        __syncthreads();
        for (int g = warp; g < ng; g += kScoreThreads / 32)
        {
            const uint16_t *src = p.q + (uint64_t)(s.row0 + i) * p.q_row + (uint64_t)(h * p.G + g0 + g) * p.q_head;
            float x[D / 32], amax = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 32; ++e)
            {
                x[e] = kv_float<BF16>(src[lane + 32 * e]);
                amax = fmaxf(amax, kv_finite_abs(x[e]));
            }
            for (int o = 16; o; o >>= 1)
                amax = fmaxf(amax, __shfl_xor_sync(kKvFull, amax, o));
            const float qs = kv_scale_of(amax), inv = kv_inverse(qs);
            int sum = 0;
            int8_t *dst = reinterpret_cast<int8_t *>(c_s[g]);
#pragma unroll
            for (int e = 0; e < D / 32; ++e)
            {
                const int c = kv_code(x[e], inv);
                sum += c;
                dst[lane + 32 * e] = (int8_t)min(c, 0);
                dst[D + lane + 32 * e] = (int8_t)max(c, 0);
            }
            for (int o = 16; o; o >>= 1)
                sum += __shfl_xor_sync(kKvFull, sum, o);
            if (lane == 0)
            {
                qs_s[g] = qs;
                sum_s[g] = sum;
            }
        }
        __syncthreads();
        for (int g = 0; g < ng; ++g)
        {
            int dot = 0;
            const uint4 *c = reinterpret_cast<const uint4 *>(c_s[g]);
#pragma unroll
            for (int e = 0; e < D / 8; ++e)
            {
                const uint4 y = c[e];
                asm("dp4a.u32.s32 %0, %1, %2, %0;" : "+r"(dot) : "r"(w[e].x), "r"(y.x));
                asm("dp4a.u32.s32 %0, %1, %2, %0;" : "+r"(dot) : "r"(w[e].y), "r"(y.y));
                asm("dp4a.u32.s32 %0, %1, %2, %0;" : "+r"(dot) : "r"(w[e].z), "r"(y.z));
                asm("dp4a.u32.s32 %0, %1, %2, %0;" : "+r"(dot) : "r"(w[e].w), "r"(y.w));
            }
            best = fmaxf(best, __fmul_rn((float)(dot - 128 * sum_s[g]), qs_s[g]));
        }
    }
    if (j < nb)
        p.scores[((uint64_t)(s.row0 + i) * p.c.hkv + h) * p.nblk + j] = blk >= 0 ? __fmul_rn(best, ks) : kKvNegInf;
}

// Order-preserving key of a score; larger is better, blocks that are always
// taken come first.
__device__ __forceinline__ uint32_t score_key(float x)
{
    const uint32_t u = __float_as_uint(x + 0.0f); // -0 counts as 0
    return (u >> 31) ? ~u : (u | 0x80000000u);
}

__global__ void __launch_bounds__(kChooseThreads) choose_kernel(SelectParams p)
{
    __shared__ uint32_t hist[256];
    __shared__ uint32_t s_digit, s_need;
    __shared__ uint32_t s_cnt[2][kChooseThreads / 32];
    const uint32_t b = blockIdx.y, h = blockIdx.x % p.c.hkv;
    const int i = (int)(blockIdx.x / p.c.hkv), tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const KvSeq s = kv_seq(p.c, b, p.rows);
    if (i >= s.rows)
        return;
    const uint64_t rh = (uint64_t)(s.row0 + i) * p.c.hkv + h;
    const float *sc = p.scores + rh * p.nblk;
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
    const int lo = (int)p.first, hi = nb - (int)p.last;
    auto key_of = [&](int j) { return j < lo || j >= hi ? 0xFFFFFFFFu : score_key(__ldg(sc + j)); };
    uint32_t prefix = 0, need = (uint32_t)k;
    for (int byte = 3; byte >= 0; --byte)
    {
        for (int e = tid; e < 256; e += kChooseThreads)
            hist[e] = 0u;
        __syncthreads();
        for (int j = tid; j < nb; j += kChooseThreads)
        {
            const uint32_t key = key_of(j);
            if (byte == 3 || (key >> (8 * (byte + 1))) == prefix)
                atomicAdd(&hist[(key >> (8 * byte)) & 255u], 1u);
        }
        __syncthreads();
        if (warp == 0)
        {
            // lane holds bins 255 - 8 lane ... downwards; the digit is where the count passes need
            uint32_t c[8], tot = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e)
                tot += c[e] = hist[255 - 8 * lane - e];
            uint32_t above = tot;
            for (int o = 1; o < 32; o <<= 1)
            {
                const uint32_t y = __shfl_up_sync(kKvFull, above, o);
                above += lane >= o ? y : 0u;
            }
            above -= tot;
#pragma unroll
            for (int e = 0; e < 8; ++e)
            {
                if (above < need && above + c[e] >= need)
                {
                    s_digit = 255u - 8u * lane - e;
                    s_need = need - above;
                }
                above += c[e];
            }
        }
        __syncthreads();
        prefix = (prefix << 8) | s_digit;
        need = s_need;
        __syncthreads();
    }
    // larger keys all, equal keys the first `need` of them
    int taken = 0;
    uint32_t equal = 0;
    for (int j0 = 0; j0 < nb; j0 += kChooseThreads)
    {
        const int j = j0 + tid;
        const uint32_t key = j < nb ? key_of(j) : 0u;
        const bool gt = j < nb && key > prefix, eq = j < nb && key == prefix;
        const uint32_t mg = __ballot_sync(kKvFull, gt), me = __ballot_sync(kKvFull, eq);
        if (lane == 0)
        {
            s_cnt[0][warp] = __popc(mg);
            s_cnt[1][warp] = __popc(me);
        }
        __syncthreads();
        uint32_t g_before = 0, e_before = 0, g_all = 0, e_all = 0;
        for (int w = 0; w < kChooseThreads / 32; ++w)
        {
            if (w < warp)
                g_before += s_cnt[0][w], e_before += s_cnt[1][w];
            g_all += s_cnt[0][w], e_all += s_cnt[1][w];
        }
        const uint32_t below = (1u << lane) - 1u;
        const uint32_t e_rank = equal + e_before + __popc(me & below);
        if (gt || (eq && e_rank < need))
        {
            const uint32_t at = (uint32_t)taken + g_before + __popc(mg & below) +
                                min(e_rank, need) - min(equal, need);
            if (at < (uint32_t)k)
                out[at] = j;
        }
        taken += (int)(g_all + min(equal + e_all, need) - min(equal, need));
        equal += e_all;
        __syncthreads();
    }
}

uint32_t score_blocks(const DanceKvCache &c, const DanceKvBatch &b)
{
    const uint64_t n = ((uint64_t)b.max_len + c.block_tokens - 1) / c.block_tokens;
    return (uint32_t)(n < b.table_width ? n : b.table_width);
}

template <int D>
int launch_select(const SelectParams &p, bool bf16, cudaStream_t st)
{
    const dim3 grid((p.nblk + kScoreThreads - 1) / kScoreThreads, p.c.max_rows * p.c.hkv, p.c.batch);
    if (p.nblk > p.select)
    {
        if (bf16)
            scores_kernel<D, true><<<grid, kScoreThreads, 0, st>>>(p);
        else
            scores_kernel<D, false><<<grid, kScoreThreads, 0, st>>>(p);
        DANCE_LAUNCHED();
    }
    choose_kernel<<<dim3(p.c.max_rows * p.c.hkv, p.c.batch), kChooseThreads, 0, st>>>(p);
    DANCE_LAUNCHED();
    return 0;
}

} // namespace

uint64_t kv_select_bytes(const DanceKvCache &c, const DanceKvBatch &b, uint32_t rows)
{
    return (uint64_t)rows * c.kv_heads * score_blocks(c, b) * 4u;
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
    if (int rc = kv_check_rows(q, cache->head_dim, num_heads, "q"))
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
    const uint64_t need = kv_counter_bytes() + kv_select_bytes(*cache, *batch, q->rows);
    if (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < need)
        return fail(-1, "workspace of %llu bytes: %llu are needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)need);
    SelectParams p;
    p.c = kv_view(*cache, *batch);
    p.q = reinterpret_cast<const uint16_t *>(q->d_data);
    p.q_row = q->row_stride;
    p.q_head = q->head_stride;
    p.rows = q->rows;
    p.heads = num_heads;
    p.G = num_heads / cache->kv_heads;
    p.nblk = score_blocks(*cache, *batch);
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

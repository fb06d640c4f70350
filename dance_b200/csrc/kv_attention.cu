// kv_attention.cu -- attention over the 8-bit key/value cache, over whole
// sequences (dance_kv_attention) and over chosen blocks
// (dance_kv_sparse_attention; include/dance_b200.h).
//
// Mathematics.  With codes k = kc - 128, v = vc - 128 (integers of 8 bits,
// exact in half precision) and block scales sk, sv:
//   s_j = scale * sk * (q . k_j),   o = sum_j p_j sv v_j / sum_j p_j,
//   p_j = 2^(s_j log2 e - m), m the running maximum of the row, a whole number
//   that stays until it is exceeded by 6 (8 in prompt_kernel).
// Scales are constant in a block, so they stay out of the matrix products: sk
// multiplies the logits, sv the weights.
//
// Roundings.  q enters as halves after an exact division by a power of two
// per row (bfloat16 has fewer bits than half; what underflows is below 2^-38
// of the row's largest channel).  The weights enter the second product as
// halves of p_j sv 2^base, 11 bits.  base is a row's own, set so that its
// largest p_j sv becomes 2^7 to 2^9 here (2^6 to 2^7 in prompt_kernel), and set
// anew before one passes 2^15: a weight has its 11 bits down to 2^-21 (2^-20)
// of the largest and is lost below 2^-32 (2^-31).  It comes from the tokens
// that the row sees alone.  Products are summed in float, as are the p_j, before
// rounding, and the output.
//
// Two kernels: rows_kernel here for the few rows of decode steps, drafts and
// chosen blocks, where the cache's bytes bound the call, and prompt_kernel
// (kv_prompt.cu) from 33 rows of a sequence and key/value head, where the
// products do.  Measured (rows_kernel): one token over 2.2M tokens, 64 heads on
// 8 of 128: 755 to 770 us, 5.9 to 6.0 TB/s, 0.90 of the measured copy rate; one
// token of each of 96 sequences up to 8192 tokens, 32 heads on 8: 179 to 181 us,
// 5.2 TB/s; 64 chosen blocks of 64 tokens of each of 32 sequences: 62 us, 4.3
// TB/s (short blocks' start and end); 700 rows of 24 heads on 8 of 96 over 48
// chosen blocks of 32: 215 us, 1.65 GB out of L2, bound by instructions
// (conversion of codes) and latency; 24 sequences' drafts of up to 5 tokens over
// up to 6000: 29 us, latency.  Maximum and base that move only when they have to
// save the exchange between a row's eight lanes in most tiles, about what the
// row's own base costs: with one maximum of the value scales for all rows,
// taken and exchanged in every tile, the five took 748, 178, 62, 217 and 28.6.
#include <cuda_runtime.h>

#include <algorithm>

#include "kv_attention.cuh"

namespace dance
{
namespace
{

constexpr int kWarps = 4;
constexpr int kTile = 32;       // tokens of a warp's tile
// Tiles of a warp in flight or in use.  Two leave room for three blocks an SM at 128 channels and four below, whose
// warps hide what a third tile would (with the kernel of that time, 171 against 172 us for a step of 96 sequences, 68
// against 80 for the sparse one).
constexpr int kStages = 2;
constexpr int kEntries = 256;   // cache blocks looked up at once
constexpr float kLift = 9.0f;   // log2 of a row's largest weight when its base is set
constexpr float kSlack = 6.0f;  // how far maximum and weights may rise before they are set anew
constexpr float kMostBase = 126.0f; // bases whose power of two, and its inverse, are normal numbers
constexpr float kMostTimes = 8.507059e37f; // 2^126

__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src)
{
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;\n" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait()
{
    asm volatile("cp.async.wait_group %0;\n" ::"n"(N) : "memory");
}

__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
                 "{%0,%1,%2,%3};\n"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Transpose of an 8 x 8 matrix of halves held one pair per lane.
__device__ __forceinline__ uint32_t transpose8(uint32_t x)
{
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;\n" : "=r"(y) : "r"(x));
    return y;
}

// Byte offset of 16-byte chunk ch of a tile's token in shared memory.  Keys
// are read with four lanes along a token and eight tokens apart, values with
// eight lanes along a token and four tokens apart by two; the offsets spread
// either pattern over the banks.
template <int D>
__device__ __forceinline__ int key_off(int tok, int ch)
{
    return tok * D + (D == 128 ? (ch ^ ((tok & 1) << 2)) : ch) * 16;
}
template <int D>
__device__ __forceinline__ int value_off(int tok, int ch)
{
    if constexpr (D == 128)
        return tok * D + (ch ^ (tok & 6)) * 16;
    else if constexpr (D == 64)
        return (tok ^ ((tok >> 2) & 1)) * D + (ch ^ (tok & 2)) * 16;
    else
        return tok * D + ch * 16;
}

// Key words (4 codes) of lane t along a token: D / 16 words from t * D / 4.
template <int D>
__device__ __forceinline__ void load_key(const uint8_t *tile, int tok, int t, uint32_t (&w)[D / 16])
{
    if constexpr (D == 128)
    {
#pragma unroll
        for (int i = 0; i < 2; ++i)
            *reinterpret_cast<uint4 *>(&w[4 * i]) =
                *reinterpret_cast<const uint4 *>(tile + key_off<D>(tok, 2 * t + i));
    }
    else if constexpr (D == 96)
    {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            *reinterpret_cast<uint2 *>(&w[2 * i]) = *reinterpret_cast<const uint2 *>(tile + tok * D + t * 24 + 8 * i);
    }
    else
        *reinterpret_cast<uint4 *>(&w[0]) = *reinterpret_cast<const uint4 *>(tile + key_off<D>(tok, t));
}

// Value words of lane g along a token: D / 32 words from g * D / 8.
template <int D>
__device__ __forceinline__ void load_value(const uint8_t *tile, int tok, int g, uint32_t (&w)[D / 32])
{
    if constexpr (D == 128)
        *reinterpret_cast<uint4 *>(&w[0]) = *reinterpret_cast<const uint4 *>(tile + value_off<D>(tok, g));
    else if constexpr (D == 96)
    {
#pragma unroll
        for (int i = 0; i < 3; ++i)
            w[i] = *reinterpret_cast<const uint32_t *>(tile + tok * D + g * 12 + 4 * i);
    }
    else
        *reinterpret_cast<uint2 *>(&w[0]) =
            *reinterpret_cast<const uint2 *>(tile + value_off<D>(tok, g >> 1) + 8 * (g & 1));
}

template <int D>
constexpr int ring_bytes()
{
    return kWarps * kStages * 2 * kTile * D;
}
template <int D>
constexpr int rows_smem()
{
    return ring_bytes<D>() + kEntries * 20;
}

// Thread blocks an SM: by shared memory, and by registers for 16 rows.
template <int D, int NT>
constexpr int rows_blocks()
{
    return D == 128 ? 4 - NT : 5 - NT;
}

// The blocks that any of ntok adjacent query tokens chose, each once, with a
// mask of the tokens that chose it, to s_page and s_mask; returns their count.
// Lists in strictly ascending order (negative entries behind) are united by
// binary search; any others are strung together, each entry with its own
// token's bit, so that a block named twice counts twice.  The order is that of
// the lists, fixed by the input alone.
__device__ int unite_lists(const AttnParams &p, const KvSeq &s, uint32_t h, int tok0, int ntok, int seen, int shift,
                           int *s_page, uint32_t *s_mask, int *s_kept, int *s_raw)
{
    __shared__ int s_sum[kWarps];
    const int n = (int)p.select, total = ntok * n, tid = threadIdx.x;
    bool odd = false;
    for (int e = tid; e < total; e += kWarps * 32)
    {
        const int t = e / n;
        const int32_t *list = p.blocks + ((uint64_t)(s.row0 + tok0 + t) * p.c.hkv + h) * n;
        const int page = __ldg(list + e - t * n);
        const int before = e > t * n ? __ldg(list + e - t * n - 1) : -1;
        odd |= page >= 0 && e > t * n && (before < 0 || before >= page);
        s_raw[e] = page >= 0 && page < (kMaxPos >> shift) && (page << shift) < seen ? page : -1;
        s_mask[e] = 0u;
    }
    odd = __syncthreads_or(odd);
    for (int e = tid; e < total; e += kWarps * 32)
    {
        const int t = e / n, page = s_raw[e];
        int first = e;
        if (!odd && page >= 0)
        {
            for (int u = 0; u < t && first == e; ++u)
            {
                int lo = u * n, hi = u * n + n; // first entry that is not below page; -1 counts as above all
                while (lo < hi)
                {
                    const int mid = (lo + hi) >> 1, y = s_raw[mid];
                    if (y >= 0 && y < page)
                        lo = mid + 1;
                    else
                        hi = mid;
                }
                if (lo < u * n + n && s_raw[lo] == page)
                    first = lo;
            }
        }
        s_kept[e] = page >= 0 && first == e;
        if (page >= 0)
            atomicOr(&s_mask[first], 1u << t);
    }
    __syncthreads();
    // every thread moves a run of entries
    constexpr int kRun = kEntries / (kWarps * 32);
    int page[kRun], count = 0;
    uint32_t mask[kRun];
#pragma unroll
    for (int k = 0; k < kRun; ++k)
    {
        const int e = tid * kRun + k;
        const bool kept = e < total && s_kept[e];
        page[k] = kept ? s_raw[e] : -1;
        mask[k] = kept ? s_mask[e] : 0u;
        count += kept;
    }
    int incl = count;
    for (int o = 1; o < 32; o <<= 1)
    {
        const int y = __shfl_up_sync(kKvFull, incl, o);
        incl += (tid & 31) >= o ? y : 0;
    }
    if ((tid & 31) == 31)
        s_sum[tid >> 5] = incl;
    __syncthreads();
    int at = incl - count, all = 0;
    for (int w = 0; w < kWarps; ++w)
    {
        at += w < (tid >> 5) ? s_sum[w] : 0;
        all += s_sum[w];
    }
#pragma unroll
    for (int k = 0; k < kRun; ++k)
        if (page[k] >= 0)
        {
            s_page[at] = page[k];
            s_mask[at++] = mask[k];
        }
    __syncthreads();
    return all;
}

// Attention of at most 8 * NT rows that share a key/value head over one split
// of their tokens.  Tokens lie on the 16-row side of the matrix instruction
// and rows on its 8-column side, for both products (S^T = K Q^T, O^T = V^T
// P^T): one row per query head of a single token fills 8 columns where the
// other way round it would leave half of 16 rows empty.
//
// The codes go from shared memory straight into the operand registers: the
// order of channels in a product over channels is free, so a lane takes D / 4
// adjacent key bytes (the rows of q are laid out alike), and so is the order
// of the output's channels, so a lane takes D / 8 adjacent value bytes of its
// tokens.  Every warp streams its own tiles of 32 tokens through its own ring
// (no barrier between warps) and keeps its own maximum and sums; the warps,
// and then the splits, are joined at the end, the splits by the block that
// finishes last, in their order.
template <int D, int NT, bool SPARSE, bool BF16>
__global__ void __launch_bounds__(kWarps * 32, rows_blocks<D, NT>()) rows_kernel(AttnParams p)
{
    extern __shared__ __align__(128) uint8_t smem[];
    constexpr int kRows = 8 * NT, kSteps = D / 16, kV = D / 8;
    int *s_blk = reinterpret_cast<int *>(smem + ring_bytes<D>());
    int *s_pos = s_blk + kEntries;
    float *s_kf = reinterpret_cast<float *>(s_pos + kEntries);
    float *s_vs = s_kf + kEntries;
    uint32_t *s_mask = reinterpret_cast<uint32_t *>(s_vs + kEntries); // tokens of the group that chose the block

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t b = blockIdx.y;
    const uint32_t rt = blockIdx.x % p.row_tiles;
    uint32_t xq = blockIdx.x / p.row_tiles;
    const uint32_t h = xq % p.c.hkv;
    xq /= p.c.hkv;
    const uint32_t split = xq % p.splits;
    const int tg = SPARSE ? (int)(xq / p.splits) : 0; // sparse: group of query tokens
    const KvSeq s = kv_seq(p.c, b, p.rows);
    const int shift = (int)p.c.shift, bs = 1 << shift, G = (int)p.G;
    const int rbase = SPARSE ? tg * (int)p.group * G : 0;
    const int nrows = SPARSE ? min(s.rows * G, rbase + (int)p.group * G) : s.rows * G;
    const int r0 = rbase + (int)rt * kRows;
    if (r0 >= nrows)
        return;
    const int r1 = min(r0 + kRows, nrows);
    const int tok_lo = r0 / G, tok_hi = (r1 - 1) / G, ntok = tok_hi - tok_lo + 1;
    const int seen_lo = min(s.first + tok_lo + 1, s.len), seen_hi = min(s.first + tok_hi + 1, s.len);
    const int nent = SPARSE ? (int)p.select : (max(seen_hi, 0) + bs - 1) >> shift;
    const int nsplits = max(1, (nent + (int)p.chunk - 1) / (int)p.chunk);
    if ((int)split >= nsplits)
        return;
    const int e0 = (int)split * (int)p.chunk, e1 = min(e0 + (int)p.chunk, nent);

    // ---- q as the second operand: lane (g, t) holds channels t * D/4 ... of rows 8 j + g
    uint32_t qf[NT][2 * kSteps];
    float rf[NT][2];   // logit factor of columns 2t, 2t + 1
    int limit[NT][2];  // tokens that they see
    uint32_t chose[NT][2]; // sparse: their token's bit in the blocks' masks
    auto load_q = [&]() {
#pragma unroll
        for (int j = 0; j < NT; ++j)
        {
            const int r = r0 + 8 * j + g;
            float x[D / 4];
            const bool live = r < r1;
            const int i = r / G, hd = (int)h * G + r % G;
            const uint16_t *src = p.q + (uint64_t)(s.row0 + (live ? i : 0)) * p.q_row + (uint64_t)(live ? hd : 0) * p.q_head +
                                  t * (D / 4);
            if (p.q_aligned)
            {
#pragma unroll
                for (int e = 0; e < D / 32; ++e)
                {
                    const uint4 w = __ldg(reinterpret_cast<const uint4 *>(src) + e);
                    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int k = 0; k < 8; ++k)
                        x[8 * e + k] = kv_float<BF16>((uint16_t)(u[k >> 1] >> (16 * (k & 1))));
                }
            }
            else
            {
#pragma unroll
                for (int e = 0; e < D / 4; ++e)
                    x[e] = kv_float<BF16>(src[e]);
            }
            float amax = 0.0f;
#pragma unroll
            for (int e = 0; e < D / 4; ++e)
                amax = fmaxf(amax, fabsf(x[e]));
            amax = fmaxf(amax, __shfl_xor_sync(kKvFull, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(kKvFull, amax, 2));
            const int up = row_shift(amax);
            const float mul = power_of_two(up), back = power_of_two(-up);
#pragma unroll
            for (int e = 0; e < 2 * kSteps; ++e)
                qf[j][e] = live ? kv_pack<false>(x[2 * e] * mul, x[2 * e + 1] * mul) : 0u;
            const float f = live ? back * p.scale_log2 : 0.0f;
            rf[j][0] = __shfl_sync(kKvFull, f, (2 * t) << 2);
            rf[j][1] = __shfl_sync(kKvFull, f, (2 * t + 1) << 2);
#pragma unroll
            for (int k = 0; k < 2; ++k)
            {
                const int rr = min(r0 + 8 * j + 2 * t + k, r1 - 1);
                limit[j][k] = min(s.first + rr / G + 1, s.len);
                if (SPARSE)
                    chose[j][k] = 1u << (rr / G - tok_lo);
            }
        }
    };

    float o[kSteps][NT][4];
    float m[NT][2], l[NT][2], base[NT][2], times[NT][2]; // times: 2^base
#pragma unroll
    for (int j = 0; j < NT; ++j)
    {
        m[j][0] = m[j][1] = kKvNegInf;
        l[j][0] = l[j][1] = 0.0f;
        base[j][0] = base[j][1] = kMostBase;
        times[j][0] = times[j][1] = kMostTimes;
#pragma unroll
        for (int i = 0; i < kSteps; ++i)
            o[i][j][0] = o[i][j][1] = o[i][j][2] = o[i][j][3] = 0.0f;
    }
    uint8_t *ring = smem + warp * (kStages * 2 * kTile * D);

    for (int seg = e0; seg < e1; seg += kEntries)
    {
        int ne = min(kEntries, e1 - seg);
        if (seg > e0)
            __syncthreads();
        const bool joint = SPARSE && ntok > 1;
        if (joint)
            ne = unite_lists(p, s, h, tok_lo, ntok, seen_hi, shift, s_pos, s_mask, reinterpret_cast<int *>(s_kf),
                             reinterpret_cast<int *>(s_vs));
        const int ntiles = (ne * bs + kTile - 1) / kTile;
        const int padded = min(kEntries, max(ne, (ntiles * kTile) >> shift)); // block_tokens 16: an even count
        for (int e = threadIdx.x; e < padded; e += kWarps * 32)
        {
            int page = -1;
            if (e < ne)
            {
                if (joint)
                    page = s_pos[e];
                else if (SPARSE)
                    page = __ldg(p.blocks + ((uint64_t)(s.row0 + tok_lo) * p.c.hkv + h) * p.select + seg + e);
                else
                    page = seg + e;
            }
            int blk = -1;
            if (page >= 0 && page < (kMaxPos >> shift) && (page << shift) < seen_hi)
                blk = kv_block(p.c, b, page);
            s_blk[e] = blk;
            s_pos[e] = blk >= 0 ? page << shift : kMaxPos;
            if (SPARSE && !joint)
                s_mask[e] = 1u;
        }
        __syncthreads();

        auto issue = [&](int tile, int stage) {
            if (tile < ntiles)
            {
                const int vt = tile * kTile;
                uint8_t *kd = ring + stage * (2 * kTile * D), *vd = kd + kTile * D;
#pragma unroll
                for (int half = 0; half < 2; ++half)
                {
                    const int v0 = vt + 16 * half, e = v0 >> shift;
                    const int blk = s_blk[e];
                    if (blk < 0)
                        continue;
                    const uint64_t off = (uint64_t)(((h << shift) + (uint32_t)(v0 & (bs - 1))) * D);
                    const uint8_t *ksrc = p.c.k + (uint64_t)blk * p.c.kbs + off;
                    const uint8_t *vsrc = p.c.v + (uint64_t)blk * p.c.vbs + off;
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
                    {
                        const int cidx = lane + 32 * i, tk = 16 * half + cidx / (D / 16), ch = cidx % (D / 16);
                        cp_async16(smem_addr(kd + key_off<D>(tk, ch)), ksrc + cidx * 16);
                        cp_async16(smem_addr(vd + value_off<D>(tk, ch)), vsrc + cidx * 16);
                    }
                }
            }
            cp_async_commit();
        };

        for (int st = 0; st < kStages - 1; ++st)
            issue(warp + kWarps * st, st);
        // q and the scales, while the first tiles are on their way
        if (seg == e0)
            load_q();
        for (int e = threadIdx.x; e < padded; e += kWarps * 32)
        {
            const int blk = s_blk[e];
            const uint64_t si = (uint64_t)max(blk, 0) * p.c.hkv + h;
            s_kf[e] = blk >= 0 ? __ldg(p.c.ks + si) : 0.0f;
            s_vs[e] = blk >= 0 ? __ldg(p.c.vs + si) : 0.0f;
        }
        __syncthreads();
        int stage = 0;
        for (int tile = warp; tile < ntiles; tile += kWarps)
        {
            int next = stage + kStages - 1;
            next = next >= kStages ? next - kStages : next;
            issue(tile + kWarps * (kStages - 1), next);
            cp_async_wait<kStages - 1>();
            __syncwarp();
            const uint8_t *kt = ring + stage * (2 * kTile * D), *vtile = kt + kTile * D;
            stage = stage + 1 == kStages ? 0 : stage + 1;
            const int ea = (tile * kTile) >> shift, eb = (tile * kTile + 16) >> shift;
            const int in_page = (tile * kTile) & (bs - 1);
            const int pos[2] = {s_pos[ea] + in_page, s_pos[eb] + (eb == ea ? in_page + 16 : 0)};
            if (pos[0] >= seen_hi && pos[1] >= seen_hi)
            {
                __syncwarp();
                continue;
            }
            const float kf[2] = {s_kf[ea], s_kf[eb]}, vs[2] = {s_vs[ea], s_vs[eb]};
            const float ve[2] = {scale_exponent(vs[0]), scale_exponent(vs[1])};

            // ---- logits
            float sc[2][NT][4];
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
            {
                uint32_t ka[D / 16], kb[D / 16];
                load_key<D>(kt, 16 * mt + g, t, ka);
                load_key<D>(kt, 16 * mt + g + 8, t, kb);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    sc[mt][j][0] = sc[mt][j][1] = sc[mt][j][2] = sc[mt][j][3] = 0.0f;
#pragma unroll
                for (int i = 0; i < kSteps; ++i)
                {
                    const uint32_t a0 = code_halves(ka[i], 0x4140), a2 = code_halves(ka[i], 0x4342);
                    const uint32_t a1 = code_halves(kb[i], 0x4140), a3 = code_halves(kb[i], 0x4342);
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        mma_f16(sc[mt][j], a0, a1, a2, a3, qf[j][2 * i], qf[j][2 * i + 1]);
                }
            }
            bool whole = pos[0] + 16 <= seen_lo && pos[1] + 16 <= seen_lo;
            uint32_t chosen[2];
            if (SPARSE)
            {
                chosen[0] = s_mask[ea];
                chosen[1] = s_mask[eb];
                whole &= (chosen[0] & chosen[1]) == (1u << ntok) - 1u;
            }
            bool up = false;
            float most[NT][2][2]; // the lane's largest logits
#pragma unroll
            for (int j = 0; j < NT; ++j)
            {
#pragma unroll
                for (int k = 0; k < 2; ++k)
                {
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt)
                    {
                        const float f = kf[mt] * rf[j][k];
#pragma unroll
                        for (int u = 0; u < 2; ++u)
                        {
                            float x = sc[mt][j][2 * u + k] * f;
                            if (!whole && (pos[mt] + g + 8 * u >= limit[j][k] || (SPARSE && !(chosen[mt] & chose[j][k]))))
                                x = kKvNegInf;
                            sc[mt][j][2 * u + k] = x;
                        }
                        most[j][k][mt] = fmaxf(sc[mt][j][k], sc[mt][j][2 + k]);
                    }
                    const float a = most[j][k][0] - m[j][k], b = most[j][k][1] - m[j][k];
                    up |= fmaxf(a, b) > kSlack || fmaxf(a + ve[0], b + ve[1]) + base[j][k] > kLift + kSlack;
                }
            }
            if (__any_sync(kKvFull, up))
            {
#pragma unroll
                for (int j = 0; j < NT; ++j)
                {
                    float down[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                    {
                        float top = fmaxf(most[j][k][0], most[j][k][1]);
                        top = fmaxf(top, __shfl_xor_sync(kKvFull, top, 4));
                        top = fmaxf(top, __shfl_xor_sync(kKvFull, top, 8));
                        top = fmaxf(top, __shfl_xor_sync(kKvFull, top, 16));
                        // whole numbers: powers of two are all that sums and outputs are scaled by
                        const float mn = top > m[j][k] + kSlack ? ceilf(top) : m[j][k];
                        float need = fmaxf(most[j][k][0] - mn + ve[0], most[j][k][1] - mn + ve[1]);
                        need = fmaxf(need, __shfl_xor_sync(kKvFull, need, 4));
                        need = fmaxf(need, __shfl_xor_sync(kKvFull, need, 8));
                        need = fmaxf(need, __shfl_xor_sync(kKvFull, need, 16));
                        const float rise = mn - m[j][k]; // from -inf: inf, or not a number where it stays
                        const float keep = fminf(base[j][k] + rise, kMostBase); // leaves the output as it is
                        const float bn = need + keep > kLift + kSlack ? fmaxf(floorf(kLift - need), -kMostBase) : keep;
                        const bool none = mn == kKvNegInf;
                        l[j][k] *= none ? 1.0f : exp2_fast(-rise);
                        down[k] = none ? 1.0f : exp2_fast(bn - base[j][k] - rise);
                        m[j][k] = mn;
                        base[j][k] = bn;
                        times[j][k] = exp2_fast(bn);
                    }
#pragma unroll
                    for (int i = 0; i < kSteps; ++i)
                    {
                        o[i][j][0] *= down[0];
                        o[i][j][1] *= down[1];
                        o[i][j][2] *= down[0];
                        o[i][j][3] *= down[1];
                    }
                }
            }

            // ---- weights and their product with the values
#pragma unroll
            for (int mt = 0; mt < 2; ++mt)
            {
                uint32_t pb[NT][2];
#pragma unroll
                for (int j = 0; j < NT; ++j)
                {
                    const float m0 = m[j][0] == kKvNegInf ? 0.0f : m[j][0];
                    const float m1 = m[j][1] == kKvNegInf ? 0.0f : m[j][1];
                    // a block that the row does not see may have any scale: 0 times it has to be 0
                    const float f0 = fminf(vs[mt] * times[j][0], kMostTimes), f1 = fminf(vs[mt] * times[j][1], kMostTimes);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                    {
                        const float p0 = exp2_fast(sc[mt][j][2 * u] - m0), p1 = exp2_fast(sc[mt][j][2 * u + 1] - m1);
                        l[j][0] += p0;
                        l[j][1] += p1;
                        pb[j][u] = transpose8(kv_pack<false>(p0 * f0, p1 * f1));
                    }
                }
                uint32_t v0[D / 32], v1[D / 32], v8[D / 32], v9[D / 32];
                load_value<D>(vtile, 16 * mt + 2 * t, g, v0);
                load_value<D>(vtile, 16 * mt + 2 * t + 1, g, v1);
                load_value<D>(vtile, 16 * mt + 2 * t + 8, g, v8);
                load_value<D>(vtile, 16 * mt + 2 * t + 9, g, v9);
#pragma unroll
                for (int w = 0; w < D / 32; ++w)
                {
                    // bytes of two tokens side by side: the pair of a channel is one operand register
                    const uint32_t a_lo = __byte_perm(v0[w], v1[w], 0x5140), a_hi = __byte_perm(v0[w], v1[w], 0x7362);
                    const uint32_t b_lo = __byte_perm(v8[w], v9[w], 0x5140), b_hi = __byte_perm(v8[w], v9[w], 0x7362);
#pragma unroll
                    for (int u = 0; u < 2; ++u)
                    {
                        const uint32_t aw = u ? a_hi : a_lo, bw = u ? b_hi : b_lo;
                        const uint32_t a0 = code_halves(aw, 0x4140), a1 = code_halves(aw, 0x4342);
                        const uint32_t a2 = code_halves(bw, 0x4140), a3 = code_halves(bw, 0x4342);
#pragma unroll
                        for (int j = 0; j < NT; ++j)
                            mma_f16(o[2 * w + u][j], a0, a1, a2, a3, pb[j][0], pb[j][1]);
                    }
                }
            }
            __syncwarp();
        }
        cp_async_wait<0>();
    }

    // ---- the warps are joined: maxima and sums through shared memory, then the outputs
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            l[j][k] += __shfl_xor_sync(kKvFull, l[j][k], 4);
            l[j][k] += __shfl_xor_sync(kKvFull, l[j][k], 8);
            l[j][k] += __shfl_xor_sync(kKvFull, l[j][k], 16);
        }
    __syncthreads();
    float *s_o = reinterpret_cast<float *>(smem);         // kWarps x kRows x D
    float *s_m = s_o + kWarps * kRows * D;                // kWarps x kRows
    float *s_l = s_m + kWarps * kRows;                    // kWarps x kRows
    float *s_all = s_l + kWarps * kRows;                  // 1 / sum of the rows
    static_assert(4 * (kWarps * kRows * D + 2 * kWarps * kRows + kRows) <= ring_bytes<D>(), "join area");
    if (g == 0)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int k = 0; k < 2; ++k)
            {
                s_m[warp * kRows + 8 * j + 2 * t + k] = m[j][k];
                s_l[warp * kRows + 8 * j + 2 * t + k] = l[j][k];
            }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int k = 0; k < 2; ++k)
        {
            const int r = 8 * j + 2 * t + k;
            float top = kKvNegInf;
            for (int w = 0; w < kWarps; ++w)
                top = fmaxf(top, s_m[w * kRows + r]);
            const float f = m[j][k] == kKvNegInf ? 0.0f : exp2_fast(m[j][k] - top), unbase = exp2_fast(-base[j][k]);
            float *dst = s_o + (warp * kRows + r) * D + g * kV;
#pragma unroll
            for (int i = 0; i < kSteps; ++i)
                *reinterpret_cast<float2 *>(dst + 2 * i) = make_float2(o[i][j][k] * f * unbase, o[i][j][2 + k] * f * unbase);
        }
    __syncthreads();
    const int item = (int)((SPARSE ? ((b * p.groups + (uint32_t)tg) * p.c.hkv + h) : (b * p.c.hkv + h)) *
                               p.row_tiles + rt);
    // partial results of the item (not touched where one split covers it)
    float *part = p.part + (uint64_t)item * p.splits * kRows * (D + 1);
    float *part_lse = part + (uint64_t)p.splits * kRows * D;
    if (threadIdx.x < kRows)
    {
        const int r = threadIdx.x;
        float top = kKvNegInf, sum = 0.0f;
        for (int w = 0; w < kWarps; ++w)
            top = fmaxf(top, s_m[w * kRows + r]);
        // a maximum of -inf: no token (sum 0), or logits that are not numbers (sum NaN), which have to show
        for (int w = 0; w < kWarps; ++w)
            sum += s_m[w * kRows + r] == kKvNegInf ? s_l[w * kRows + r]
                                                   : exp2_fast(s_m[w * kRows + r] - top) * s_l[w * kRows + r];
        const float lse2 = sum == 0.0f ? kKvNegInf : top + log2f(sum);
        s_all[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
        if (nsplits > 1)
            part_lse[split * kRows + r] = lse2;
        else if (p.lse && r0 + r < r1)
        {
            const int i = (r0 + r) / G, hd = (int)h * G + (r0 + r) % G;
            p.lse[(uint64_t)(s.row0 + i) * p.heads + hd] = lse2 * 0.69314718056f;
        }
    }
    __syncthreads();
    uint16_t *out = reinterpret_cast<uint16_t *>(p.out);
    for (int e = threadIdx.x; e < kRows * D / 4; e += kWarps * 32)
    {
        const int r = e / (D / 4), d = (e % (D / 4)) * 4;
        if (r0 + r >= r1)
            break;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int w = 0; w < kWarps; ++w)
        {
            const float4 z = *reinterpret_cast<const float4 *>(s_o + (w * kRows + r) * D + d);
            y.x += z.x, y.y += z.y, y.z += z.z, y.w += z.w;
        }
        const float f = s_all[r];
        y.x *= f, y.y *= f, y.z *= f, y.w *= f;
        if (nsplits > 1)
            *reinterpret_cast<float4 *>(part + ((uint64_t)split * kRows + r) * D + d) = y;
        else
        {
            const int i = (r0 + r) / G, hd = (int)h * G + (r0 + r) % G;
            *reinterpret_cast<uint2 *>(out + ((uint64_t)(s.row0 + i) * p.heads + hd) * D + d) =
                make_uint2(kv_pack<BF16>(y.x, y.y), kv_pack<BF16>(y.z, y.w));
        }
    }
    if (nsplits == 1)
        return;

    // ---- the splits are joined by the block that comes last, in their order
    __shared__ bool s_last;
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0)
        s_last = atomicAdd(p.counters + item, 1u) == (uint32_t)nsplits - 1u;
    __syncthreads();
    if (!s_last)
        return;
    __threadfence();
    float *s_w = reinterpret_cast<float *>(smem); // nsplits x kRows: weights
    float *s_f = s_w + nsplits * kRows;           // kRows: 1 / sum
    for (int e = threadIdx.x; e < nsplits * kRows; e += kWarps * 32)
        s_w[e] = __ldcg(part_lse + e);
    __syncthreads();
    if (threadIdx.x == 0)
        p.counters[item] = 0u;
    for (int r = warp; r < kRows; r += kWarps)
    {
        float top = kKvNegInf, sum = 0.0f;
        for (int i = lane; i < nsplits; i += 32)
            top = fmaxf(top, s_w[i * kRows + r]);
        for (int o = 16; o; o >>= 1)
            top = fmaxf(top, __shfl_xor_sync(kKvFull, top, o));
        const float base = top == kKvNegInf ? 0.0f : top;
        for (int i = lane; i < nsplits; i += 32)
        {
            const float wt = exp2_fast(s_w[i * kRows + r] - base);
            s_w[i * kRows + r] = wt;
            sum += wt;
        }
        for (int o = 16; o; o >>= 1)
            sum += __shfl_xor_sync(kKvFull, sum, o);
        if (lane == 0)
        {
            s_f[r] = sum == 0.0f ? 0.0f : 1.0f / sum;
            if (p.lse && r0 + r < r1)
            {
                const int i = (r0 + r) / G, hd = (int)h * G + (r0 + r) % G;
                p.lse[(uint64_t)(s.row0 + i) * p.heads + hd] =
                    (sum == 0.0f ? kKvNegInf : base + log2f(sum)) * 0.69314718056f;
            }
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < kRows * D / 4; e += kWarps * 32)
    {
        const int r = e / (D / 4), d = (e % (D / 4)) * 4;
        if (r0 + r >= r1)
            break;
        float4 y = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 8
        for (int i = 0; i < nsplits; ++i)
        {
            const float w = s_w[i * kRows + r];
            const float4 z = __ldcg(reinterpret_cast<const float4 *>(part + ((uint64_t)i * kRows + r) * D + d));
            y.x += w * z.x, y.y += w * z.y, y.z += w * z.z, y.w += w * z.w;
        }
        const float f = s_f[r];
        const int i = (r0 + r) / G, hd = (int)h * G + (r0 + r) % G;
        *reinterpret_cast<uint2 *>(out + ((uint64_t)(s.row0 + i) * p.heads + hd) * D + d) =
            make_uint2(kv_pack<BF16>(y.x * f, y.y * f), kv_pack<BF16>(y.z * f, y.w * f));
    }
}

constexpr uint32_t kSms = 148;
constexpr uint64_t kMostSplits = 480; // their weights are joined in the ring's shared memory
static_assert((kMostSplits + 8) * 16 * 4 <= rows_smem<64>(), "weights of the splits");
// The prompt kernel takes over above this many rows (query tokens x query heads) of a sequence and key/value head.  8
// key/value heads of 128, prompt kernel against rows_kernel: 40 rows of 24 sequences of 6000 tokens 225 and 188 us, of
// one of 60000 91 and 80; 64 rows of 8 sequences of 8000 96 and 128, 128 rows 107 and 226; 256 rows of 2 of 16000 117
// and 215.  They meet between 40 and 64 rows.
constexpr uint64_t kPromptLeast = 32;

AttnPlan plan_attention(const DanceKvCache &c, const DanceKvBatch &b, uint32_t heads, uint32_t select)
{
    AttnPlan a;
    const uint32_t G = heads / c.kv_heads;
    // Sparse rows: adjacent query tokens choose much the same blocks; as many as fill 8 columns share a thread block,
    // which loads and converts what any of them chose once.  Tokens that choose nothing in common cost what they
    // would cost alone.  (16 columns halve the blocks once more where most of the choice is shared, but cost more per
    // block: with a quarter shared, 700 rows of 24 heads took 260 us, with 8 columns 244, alone 257.)
    a.group = 1;
    if (select && G <= 4 && b.max_rows > 1)
    {
        a.group = 8 / G < kEntries / select ? 8 / G : kEntries / select;
        a.group = a.group < b.max_rows ? a.group : b.max_rows;
        while (a.group > 1 && (uint64_t)(b.max_rows + a.group - 1) / a.group * b.batch * c.kv_heads < 2 * kSms)
            --a.group;
        a.group = a.group ? a.group : 1;
    }
    a.groups = (b.max_rows + a.group - 1) / a.group;
    const uint64_t rows = select ? (uint64_t)a.group * G : (uint64_t)b.max_rows * G;
    a.prompt = !select && rows > kPromptLeast;
    a.nt = rows <= 8 ? 1u : 2u;
    const uint32_t tile = a.prompt ? kPromptRows : 8 * a.nt;
    a.row_tiles = (uint32_t)((rows + tile - 1) / tile);
    const uint64_t per_b = (uint64_t)c.kv_heads * a.row_tiles * (select ? a.groups : 1u);
    const uint64_t items = per_b * b.batch;
    const uint64_t cap = (uint64_t)b.table_width * c.block_tokens;
    const uint64_t len = b.max_len < cap ? b.max_len : cap;
    const uint32_t ent = select ? select : (uint32_t)((len + c.block_tokens - 1) / c.block_tokens);
    const uint64_t tokens = (uint64_t)ent * c.block_tokens;
    uint64_t want = 1;
    uint32_t unit = c.block_tokens == 16 ? 2 : 1; // cache blocks of a tile of 32 tokens
    if (a.prompt)
    {
        // splits: what fills the waves of blocks best, a block's start and end counting like 768 tokens,
        // the joining of splits like 768 more
        unit = c.block_tokens < kPromptTokens ? kPromptTokens / c.block_tokens : 1;
        uint64_t best = ~0ull;
        for (uint64_t s = 1; s <= kSms && (s == 1 || tokens / s >= 512); ++s)
        {
            const uint64_t cost = (items * s + kSms - 1) / kSms *
                                  (tokens / s + (s > 1 ? 1536u : 768u));
            if (cost < best)
                best = cost, want = s;
        }
    }
    else
    {
        // A block's start and end count like 384 tokens of 128 channels and 8 rows, and so does joining.  One sequence, or lists of one length:
        // whole waves of equal blocks.  Sequences of unknown lengths up to max_len: the work spread over the slots,
        // and the last block's own time.  (Steps of 96 sequences up to 8192 tokens, 8 heads: 1 split 175 us, 2 171,
        // 4 165.  24 of up to 6000, 4 heads: 4 splits 26.7, 7 23.5, 13 33; of these the rule can take 4.)
        const uint32_t per_sm = c.head_dim == 128 ? 4u - a.nt : 5u - a.nt; // rows_blocks()
        const uint64_t slots = (uint64_t)kSms * per_sm;
        const uint64_t most = std::min<uint64_t>((tokens + 255) / 256, kMostSplits);
        const uint64_t fixed = 384ull * a.nt * 128 / c.head_dim;
        uint64_t best = ~0ull;
        for (uint64_t waves = 0; waves <= 8; ++waves)
        {
            uint64_t s = items ? waves * slots / items : 1;
            s = s < 1 ? 1 : s > most ? (most ? most : 1) : s;
            const uint64_t one = tokens / s + fixed;
            const uint64_t cost = (b.batch == 1 || select ? (items * s + slots - 1) / slots * one
                                                          : items * s * one / slots + one) + (s > 1 ? fixed : 0);
            if (cost < best)
                best = cost, want = s;
        }
    }
    if (want < 1 || items > kCounters || a.group > 1) // what a group chose is known to its own thread block only
        want = 1;
    a.chunk = (uint32_t)((ent + want - 1) / want);
    a.chunk = a.chunk ? (a.chunk + unit - 1) / unit * unit : unit;
    a.splits = (ent + a.chunk - 1) / a.chunk;
    a.splits = a.splits ? a.splits : 1;
    a.blocks_x = per_b * a.splits;
    a.bytes = kCounters * 4ull + (a.splits > 1 ? items * a.splits * tile * (c.head_dim + 1) * 4ull : 0ull);
    return a;
}

template <int D, int NT, bool SPARSE, bool BF16>
int launch_rows(const AttnParams &p, dim3 grid, cudaStream_t st)
{
    static SmemAllowed allowed;
    DANCE_CUDA(allowed.on_current(reinterpret_cast<const void *>(rows_kernel<D, NT, SPARSE, BF16>), rows_smem<D>()));
    rows_kernel<D, NT, SPARSE, BF16><<<grid, kWarps * 32, rows_smem<D>(), st>>>(p);
    DANCE_LAUNCHED();
    return 0;
}

template <int D>
int launch_rows_d(const AttnParams &p, uint32_t nt, bool bf16, dim3 grid, cudaStream_t st)
{
    const bool sparse = p.blocks != nullptr;
    switch ((nt - 1) * 4 + (sparse ? 2 : 0) + (bf16 ? 1 : 0))
    {
    case 0:
        return launch_rows<D, 1, false, false>(p, grid, st);
    case 1:
        return launch_rows<D, 1, false, true>(p, grid, st);
    case 2:
        return launch_rows<D, 1, true, false>(p, grid, st);
    case 3:
        return launch_rows<D, 1, true, true>(p, grid, st);
    case 4:
        return launch_rows<D, 2, false, false>(p, grid, st);
    case 5:
        return launch_rows<D, 2, false, true>(p, grid, st);
    case 6:
        return launch_rows<D, 2, true, false>(p, grid, st);
    default:
        return launch_rows<D, 2, true, true>(p, grid, st);
    }
}

int attend(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *q, uint32_t num_heads,
           const int32_t *d_blocks, uint32_t select, float scale, void *d_out, float *d_lse, void *d_workspace,
           uint64_t workspace_bytes, void *stream)
{
    if (int rc = kv_check(cache, batch))
        return rc;
    if (int rc = kv_check_rows(q, "q"))
        return rc;
    if (num_heads == 0 || num_heads % cache->kv_heads || num_heads > 65536)
        return fail(-1, "num_heads %u must be a multiple of kv_heads %u", num_heads, cache->kv_heads);
    if (q->rows == 0 || batch->max_rows == 0)
        return 0;
    if (!d_out || (uintptr_t)d_out % 16 || (uintptr_t)d_lse % 4)
        return fail(-1, "null or misaligned output");
    const AttnPlan a = plan_attention(*cache, *batch, num_heads, select);
    if (!d_workspace || (uintptr_t)d_workspace % 16 || workspace_bytes < a.bytes)
        return fail(-1, "workspace of %llu bytes: %llu are needed", (unsigned long long)workspace_bytes,
                    (unsigned long long)a.bytes);
    if (a.blocks_x > 0x7FFFFFFFull)
        return fail(-1, "call too large: %llu thread blocks per sequence", (unsigned long long)a.blocks_x);
    AttnParams p;
    p.c = kv_view(*cache, *batch);
    p.q = reinterpret_cast<const uint16_t *>(q->d_data);
    p.q_row = q->row_stride;
    p.q_head = q->head_stride;
    p.q_aligned = kv_aligned(*q);
    p.rows = q->rows;
    p.heads = num_heads;
    p.G = num_heads / cache->kv_heads;
    p.scale_log2 = scale * 1.44269504089f;
    p.blocks = d_blocks;
    p.select = select;
    p.group = a.group;
    p.groups = a.groups;
    p.chunk = a.chunk;
    p.splits = a.splits;
    p.row_tiles = a.row_tiles;
    p.out = d_out;
    p.lse = d_lse;
    p.counters = reinterpret_cast<uint32_t *>(d_workspace);
    p.part = reinterpret_cast<float *>(p.counters + kCounters);
    const dim3 grid((unsigned)a.blocks_x, batch->batch);
    const bool bf16 = q->dtype == DANCE_BF16;
    if (a.prompt)
        return launch_prompt(p, cache->head_dim, bf16, (uint32_t)a.blocks_x, as_stream(stream));
    switch (cache->head_dim)
    {
    case 64:
        return launch_rows_d<64>(p, a.nt, bf16, grid, as_stream(stream));
    case 96:
        return launch_rows_d<96>(p, a.nt, bf16, grid, as_stream(stream));
    default:
        return launch_rows_d<128>(p, a.nt, bf16, grid, as_stream(stream));
    }
}

} // namespace

uint64_t kv_counter_bytes() { return kCounters * 4ull; }
uint64_t kv_attention_bytes(const DanceKvCache &c, const DanceKvBatch &b, uint32_t heads, uint32_t select)
{
    return plan_attention(c, b, heads, select).bytes;
}

} // namespace dance

using namespace dance;

extern "C" int dance_kv_attention(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *q,
                                  uint32_t num_heads, float scale, void *d_out, float *d_lse, void *d_workspace,
                                  uint64_t workspace_bytes, void *stream)
{
    return attend(cache, batch, q, num_heads, nullptr, 0, scale, d_out, d_lse, d_workspace, workspace_bytes, stream);
}

extern "C" int dance_kv_sparse_attention(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *q,
                                         uint32_t num_heads, const int32_t *d_blocks, uint32_t select, float scale,
                                         void *d_out, float *d_lse, void *d_workspace, uint64_t workspace_bytes,
                                         void *stream)
{
    if (!d_blocks || (uintptr_t)d_blocks % 4)
        return fail(-1, "null or misaligned block selection");
    if (select == 0 || select > 4096)
        return fail(-1, "select %u: 1 to 4096 are supported", select);
    return attend(cache, batch, q, num_heads, d_blocks, select, scale, d_out, d_lse, d_workspace, workspace_bytes,
                  stream);
}

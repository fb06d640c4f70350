// kv_cache.cu -- the write into and the read out of the 8-bit key/value cache
// (dance_kv_append, dance_kv_read in include/dance_b200.h).
//
// append.  One thread block per (touched cache block, head), keys and values.
// The new rows are read once into registers; their largest finite magnitudes
// and the scales so far give the new scales.  Only where a scale grew are the
// block's earlier codes read, rounded again and written back.  The earlier
// tokens enter the bounds through the bounds themselves (rounding is monotone,
// so the rounded bounds are the bounds of the rounded codes), so that a decode
// step moves one token and 2 * head_dim bytes of bounds, not a block.
// Threads are laid out as 16 token groups x head_dim / 8 channel groups: a
// thread keeps its 8 channels through all its tokens, so the bounds are byte
// minima and maxima in registers and one reduction over 16 groups.
//
// Both kernels move each byte once.  Measured: 17106 tokens x 8 heads of 96
// channels in blocks of 32, f16: append 35 us (79 MB, 2.3 TB/s; instructions
// bound it, about 31 per element with their block's share of setup and
// reductions, 74 % of the issue slots), read 20 us (79 MB, 4.0 TB/s, 77 % of the
// issue slots).  One token of each of 64 sequences
// x 8 heads of 128: append 6 to 9 us, read 5, latency.  Taking the keys and the
// values of a block together, magnitudes as packed integers and codes by adding
// a constant brought the append from 46 us.
#include "kv_common.cuh"

namespace dance
{
namespace
{

constexpr int kTokenGroups = 16;

struct AppendParams
{
    KvView c;
    const uint16_t *x[2]; // new keys, new values
    uint64_t row_stride[2], head_stride[2];
    uint32_t rows;
    bool aligned[2];
};

// Two magnitudes at once, as the bits of two 16-bit floats without their sign:
// such bits order like the values, infinities and NaN above all.
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b)
{
    uint32_t r;
    asm("max.u16x2 %0, %1, %2;\n" : "=r"(r) : "r"(a), "r"(b));
    return r;
}

// The largest finite magnitude of eight values.
template <bool BF16>
__device__ __noinline__ float finite_max(uint4 x)
{
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
    float m = 0.0f;
    for (int e = 0; e < 4; ++e)
    {
        m = fmaxf(m, kv_finite_abs(kv_float<BF16>((uint16_t)w[e])));
        m = fmaxf(m, kv_finite_abs(kv_float<BF16>((uint16_t)(w[e] >> 16))));
    }
    return m;
}

// Four finite values at a scale as codes.  Adding 1.5 * 2^23 + 128 rounds to a
// whole number, ties to even as rint does (the sum's unit is 1 and the number
// added is even), and leaves the code in the low byte; |x * inv| is at most
// 127 up to rounding, so nothing is cut off.
template <bool BF16>
__device__ __forceinline__ uint32_t codes4(uint32_t w0, uint32_t w1, float inv)
{
    const float magic = 12582912.0f + 128.0f;
    const uint32_t a = __float_as_uint(__fadd_rn(__fmul_rn(kv_float<BF16>((uint16_t)w0), inv), magic));
    const uint32_t b = __float_as_uint(__fadd_rn(__fmul_rn(kv_float<BF16>((uint16_t)(w0 >> 16)), inv), magic));
    const uint32_t c = __float_as_uint(__fadd_rn(__fmul_rn(kv_float<BF16>((uint16_t)w1), inv), magic));
    const uint32_t d = __float_as_uint(__fadd_rn(__fmul_rn(kv_float<BF16>((uint16_t)(w1 >> 16)), inv), magic));
    return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// The same for any values; not inlined, so that it costs the common case a
// branch and no more.
template <bool BF16>
__device__ __noinline__ uint32_t codes4_any(uint32_t w0, uint32_t w1, float inv)
{
    uint32_t r = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
        r |= (uint32_t)(kv_code(kv_float<BF16>((uint16_t)((e < 2 ? w0 : w1) >> (16 * (e & 1)))), inv) + 128) << (8 * e);
    return r;
}

// The largest of two non-negative values over the thread block.
__device__ __forceinline__ float2 block_max(float2 x, float2 *s)
{
    for (int o = 16; o; o >>= 1)
    {
        x.x = fmaxf(x.x, __shfl_xor_sync(kKvFull, x.x, o));
        x.y = fmaxf(x.y, __shfl_xor_sync(kKvFull, x.y, o));
    }
    if ((threadIdx.x & 31) == 0)
        s[threadIdx.x >> 5] = x;
    __syncthreads();
    float2 m = make_float2(0.0f, 0.0f);
    for (int i = 0; i < (int)blockDim.x / 32; ++i)
        m = make_float2(fmaxf(m.x, s[i].x), fmaxf(m.y, s[i].y));
    return m;
}

// Four codes rounded again to a scale that is 1 / shrink times as large.
__device__ __noinline__ uint32_t shrink_codes(uint32_t w, float shrink)
{
    uint32_t r = 0u;
#pragma unroll
    for (int e = 0; e < 4; ++e)
    {
        const float y = __fmul_rn((float)((int)((w >> (8 * e)) & 255u) - 128), shrink);
        r |= ((uint32_t)(__float2int_rn(y) + 128) & 255u) << (8 * e);
    }
    return r;
}

// IT = block_tokens / 16 tokens per thread.
template <int D, int IT, bool BF16>
__global__ void __launch_bounds__(D / 8 * kTokenGroups, IT <= 2 ? 1536 / (D / 8 * kTokenGroups) : 1)
    append_kernel(AppendParams p)
{
    constexpr int kD8 = D / 8, kBs = IT * kTokenGroups;
    __shared__ float2 red[8];
    __shared__ uint2 lo_s[kTokenGroups][kD8], hi_s[kTokenGroups][kD8];
    const uint32_t b = blockIdx.y, h = blockIdx.x % p.c.hkv; // heads of a token side by side
    const KvSeq s = kv_seq(p.c, b, p.rows);
    const int start = max(s.first, 0), end = min(s.first + s.rows, s.len);
    const int page = start / kBs + (int)(blockIdx.x / p.c.hkv);
    const int base = page * kBs;
    const int lo = max(start, base), hi = min(end, base + kBs);
    if (lo >= hi)
        return;
    const int blk = kv_block(p.c, b, page);
    if (blk < 0)
        return;
    const int n_old = lo - base;
    const int d8 = threadIdx.x % kD8, tg = threadIdx.x / kD8;
    const uint64_t si = (uint64_t)blk * p.c.hkv + h;
    const float old[2] = {n_old ? p.c.ks[si] : 0.0f, n_old ? p.c.vs[si] : 0.0f};

    uint4 x[2][IT];
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
#pragma unroll
        for (int i = 0; i < IT; ++i)
        {
            const int pos = base + tg + kTokenGroups * i;
            x[kind][i] = make_uint4(0u, 0u, 0u, 0u);
            if (pos >= lo && pos < hi)
            {
                const uint16_t *src = p.x[kind] + (uint64_t)h * p.head_stride[kind] + d8 * 8 +
                                      (uint64_t)(s.row0 + pos - s.first) * p.row_stride[kind];
                if (p.aligned[kind])
                    x[kind][i] = __ldg(reinterpret_cast<const uint4 *>(src));
                else
                {
                    uint32_t w[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        w[e] = (uint32_t)src[2 * e] | ((uint32_t)src[2 * e + 1] << 16);
                    x[kind][i] = make_uint4(w[0], w[1], w[2], w[3]);
                }
            }
        }
    float largest[2];
    bool odd = false; // infinities or NaN among the thread's values
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
    {
        uint32_t top = 0u;
#pragma unroll
        for (int i = 0; i < IT; ++i)
        {
            top = max_u16x2(top, max_u16x2(x[kind][i].x & 0x7FFF7FFFu, x[kind][i].y & 0x7FFF7FFFu));
            top = max_u16x2(top, max_u16x2(x[kind][i].z & 0x7FFF7FFFu, x[kind][i].w & 0x7FFF7FFFu));
        }
        const uint32_t most = max(top & 0xFFFFu, top >> 16);
        largest[kind] = kv_float<BF16>((uint16_t)most);
        odd |= most >= (BF16 ? 0x7F80u : 0x7C00u);
    }
    if (odd)
    {
#pragma unroll
        for (int kind = 0; kind < 2; ++kind)
        {
            largest[kind] = 0.0f;
#pragma unroll
            for (int i = 0; i < IT; ++i)
                largest[kind] = fmaxf(largest[kind], finite_max<BF16>(x[kind][i]));
        }
    }
    const float2 both = block_max(make_float2(largest[0], largest[1]), red);

    uint32_t lo4[2] = {0xFFFFFFFFu, 0xFFFFFFFFu}, hi4[2] = {0u, 0u};
    float key_shrink = 1.0f;
    bool key_grew = false;
#pragma unroll
    for (int kind = 0; kind < 2; ++kind)
    {
        const float amax = kind ? both.y : both.x, quotient = kv_scale_of(amax);
        const float scale = fmaxf(old[kind], quotient);
        // written again (quotient == old), the same rows get the same codes
        const float step = old[kind] > quotient ? old[kind] : kv_step_of(amax);
        const float inv = kv_inverse(step);
        // a scale that was never written (NaN) cannot be told from a grown one: the comparison treats it as grown
        const bool grew = n_old > 0 && !(scale == old[kind]);
        const float shrink = step > 0.0f ? __fdiv_rn(old[kind], step) : 0.0f;
        uint8_t *codes = (kind ? p.c.v + (uint64_t)blk * p.c.vbs : p.c.k + (uint64_t)blk * p.c.kbs) +
                         (uint64_t)h * (kBs * D) + d8 * 8;
#pragma unroll
        for (int i = 0; i < IT; ++i)
        {
            const int t = tg + kTokenGroups * i, pos = base + t;
            if (pos >= lo && pos < hi)
            {
                const uint4 w = x[kind][i];
                uint32_t c2[2];
                if (odd)
                {
                    c2[0] = codes4_any<BF16>(w.x, w.y, inv);
                    c2[1] = codes4_any<BF16>(w.z, w.w, inv);
                }
                else
                {
                    c2[0] = codes4<BF16>(w.x, w.y, inv);
                    c2[1] = codes4<BF16>(w.z, w.w, inv);
                }
                *reinterpret_cast<uint2 *>(codes + t * D) = make_uint2(c2[0], c2[1]);
                if (kind == 0)
#pragma unroll
                    for (int g = 0; g < 2; ++g)
                    {
                        lo4[g] = __vminu4(lo4[g], c2[g]);
                        hi4[g] = __vmaxu4(hi4[g], c2[g]);
                    }
            }
            else if (grew && t < n_old)
            {
                const uint2 c = *reinterpret_cast<const uint2 *>(codes + t * D);
                *reinterpret_cast<uint2 *>(codes + t * D) =
                    make_uint2(shrink_codes(c.x, shrink), shrink_codes(c.y, shrink));
            }
        }
        if (threadIdx.x == 0)
            (kind ? p.c.vs : p.c.ks)[si] = scale;
        if (kind == 0)
        {
            key_shrink = shrink;
            key_grew = grew;
        }
    }
    lo_s[tg][d8] = make_uint2(lo4[0], lo4[1]);
    hi_s[tg][d8] = make_uint2(hi4[0], hi4[1]);
    __syncthreads();
    if (threadIdx.x < 2 * kD8)
    {
        const bool high = threadIdx.x >= kD8;
        const int d = high ? threadIdx.x - kD8 : threadIdx.x;
        uint2 *out = reinterpret_cast<uint2 *>(p.c.bounds + (2 * si + (high ? 1 : 0)) * D) + d;
        uint2 r = high ? make_uint2(0u, 0u) : make_uint2(0xFFFFFFFFu, 0xFFFFFFFFu);
        if (n_old)
        {
            r = *out;
            if (key_grew)
                r = make_uint2(shrink_codes(r.x, key_shrink), shrink_codes(r.y, key_shrink));
        }
        for (int g = 0; g < kTokenGroups; ++g)
        {
            const uint2 y = high ? hi_s[g][d] : lo_s[g][d];
            r.x = high ? __vmaxu4(r.x, y.x) : __vminu4(r.x, y.x);
            r.y = high ? __vmaxu4(r.y, y.y) : __vminu4(r.y, y.y);
        }
        *out = r;
    }
}

template <int D>
int launch_append(const AppendParams &p, dim3 grid, bool bf16, cudaStream_t st)
{
    const dim3 block(D / 8 * kTokenGroups);
    switch (((1u << p.c.shift) / kTokenGroups) * 2 + (bf16 ? 1 : 0))
    {
#define DANCE_APPEND_CASE(it)                                                                                    \
    case 2 * it:                                                                                                 \
        append_kernel<D, it, false><<<grid, block, 0, st>>>(p);                                                  \
        break;                                                                                                   \
    case 2 * it + 1:                                                                                             \
        append_kernel<D, it, true><<<grid, block, 0, st>>>(p);                                                   \
        break;
        DANCE_APPEND_CASE(1)
        DANCE_APPEND_CASE(2)
        DANCE_APPEND_CASE(4)
        DANCE_APPEND_CASE(8)
#undef DANCE_APPEND_CASE
    default:
        return fail(-1, "block_tokens %u", 1u << p.c.shift);
    }
    DANCE_LAUNCHED();
    return 0;
}

// One thread per 8 channels of a (row, head): 8 code bytes in, 8 values out.
template <int D, int DT>
__global__ void __launch_bounds__(256) read_kernel(KvView c, uint32_t rows, void *ko, void *vo)
{
    constexpr uint32_t kD8 = D / 8;
    const uint32_t b = blockIdx.y;
    const KvSeq s = kv_seq(c, b, rows);
    const uint64_t n = (uint64_t)s.rows * c.hkv * kD8;
    const uint32_t mask = (1u << c.shift) - 1u;
    for (uint64_t e = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; e < n; e += (uint64_t)gridDim.x * blockDim.x)
    {
        const uint32_t d8 = (uint32_t)(e % kD8), rh = (uint32_t)(e / kD8), h = rh % c.hkv, i = rh / c.hkv;
        const int pos = s.first + (int)i;
        const int blk = pos >= 0 && pos < s.len ? kv_block(c, b, pos >> c.shift) : -1;
        const uint64_t si = (uint64_t)max(blk, 0) * c.hkv + h;
        const uint64_t in = (((uint64_t)h << c.shift) + ((uint32_t)pos & mask)) * D + d8 * 8;
        const uint64_t out = ((uint64_t)(s.row0 + i) * c.hkv + h) * D + d8 * 8;
#pragma unroll
        for (int kind = 0; kind < 2; ++kind)
        {
            void *dst = kind ? vo : ko;
            if (!dst)
                continue;
            float y[8];
            uint2 w = make_uint2(0x80808080u, 0x80808080u);
            float scale = 0.0f;
            if (blk >= 0)
            {
                w = __ldg(reinterpret_cast<const uint2 *>(
                    (kind ? c.v + (uint64_t)blk * c.vbs : c.k + (uint64_t)blk * c.kbs) + in));
                scale = __ldg((kind ? c.vs : c.ks) + si);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
            {
                // the byte as the last of 2^23 + c, exactly
                const uint32_t u = __byte_perm(k < 4 ? w.x : w.y, 0x4B000000u, 0x7440 + (k & 3));
                y[k] = __fmul_rn(__fsub_rn(__uint_as_float(u), 8388608.0f + 128.0f), scale);
            }
            if constexpr (DT == DANCE_F32)
            {
                float4 *o = reinterpret_cast<float4 *>(reinterpret_cast<float *>(dst) + out);
                o[0] = make_float4(y[0], y[1], y[2], y[3]);
                o[1] = make_float4(y[4], y[5], y[6], y[7]);
            }
            else
            {
                constexpr bool bf = DT == DANCE_BF16;
                *reinterpret_cast<uint4 *>(reinterpret_cast<uint16_t *>(dst) + out) =
                    make_uint4(kv_pack<bf>(y[0], y[1]), kv_pack<bf>(y[2], y[3]), kv_pack<bf>(y[4], y[5]),
                               kv_pack<bf>(y[6], y[7]));
            }
        }
    }
}

template <int D>
int launch_read(const KvView &c, uint32_t rows, int dtype, void *ko, void *vo, cudaStream_t st)
{
    const uint64_t work = (uint64_t)c.max_rows * c.hkv * (D / 8);
    const dim3 grid((unsigned)((work + 255) / 256 < 65536 ? (work + 255) / 256 : 65536), c.batch);
    if (dtype == DANCE_F32)
        read_kernel<D, DANCE_F32><<<grid, 256, 0, st>>>(c, rows, ko, vo);
    else if (dtype == DANCE_F16)
        read_kernel<D, DANCE_F16><<<grid, 256, 0, st>>>(c, rows, ko, vo);
    else
        read_kernel<D, DANCE_BF16><<<grid, 256, 0, st>>>(c, rows, ko, vo);
    DANCE_LAUNCHED();
    return 0;
}

} // namespace
} // namespace dance

using namespace dance;

extern "C" int dance_kv_append(const DanceKvCache *cache, const DanceKvBatch *batch, const DanceKvRows *k,
                               const DanceKvRows *v, void *stream)
{
    if (int rc = kv_check(cache, batch))
        return rc;
    if (int rc = kv_check_rows(k, "k"))
        return rc;
    if (int rc = kv_check_rows(v, "v"))
        return rc;
    if (k->rows != v->rows || k->dtype != v->dtype)
        return fail(-1, "keys (%u rows, dtype %d) and values (%u rows, dtype %d) differ", k->rows, k->dtype, v->rows,
                    v->dtype);
    if (k->rows == 0 || batch->max_rows == 0)
        return 0;
    AppendParams p;
    p.c = kv_view(*cache, *batch);
    const DanceKvRows *r[2] = {k, v};
    for (int i = 0; i < 2; ++i)
    {
        p.x[i] = reinterpret_cast<const uint16_t *>(r[i]->d_data);
        p.row_stride[i] = r[i]->row_stride;
        p.head_stride[i] = r[i]->head_stride;
        p.aligned[i] = kv_aligned(*r[i]);
    }
    p.rows = k->rows;
    const uint32_t bs = cache->block_tokens;
    const dim3 grid(((batch->max_rows + bs - 2) / bs + 1) * cache->kv_heads, batch->batch);
    const bool bf16 = k->dtype == DANCE_BF16;
    switch (cache->head_dim)
    {
    case 64:
        return launch_append<64>(p, grid, bf16, as_stream(stream));
    case 96:
        return launch_append<96>(p, grid, bf16, as_stream(stream));
    default:
        return launch_append<128>(p, grid, bf16, as_stream(stream));
    }
}

extern "C" int dance_kv_read(const DanceKvCache *cache, const DanceKvBatch *batch, uint32_t rows, int dtype,
                             void *d_k_out, void *d_v_out, void *stream)
{
    if (int rc = kv_check(cache, batch))
        return rc;
    if (dtype != DANCE_F16 && dtype != DANCE_BF16 && dtype != DANCE_F32)
        return fail(-1, "output dtype %d: float16, bfloat16 and float32 are supported", dtype);
    if (((uintptr_t)d_k_out | (uintptr_t)d_v_out) % 16)
        return fail(-1, "outputs must be 16-byte aligned");
    if (rows == 0 || batch->max_rows == 0 || (!d_k_out && !d_v_out))
        return 0;
    const KvView c = kv_view(*cache, *batch);
    switch (cache->head_dim)
    {
    case 64:
        return launch_read<64>(c, rows, dtype, d_k_out, d_v_out, as_stream(stream));
    case 96:
        return launch_read<96>(c, rows, dtype, d_k_out, d_v_out, as_stream(stream));
    default:
        return launch_read<128>(c, rows, dtype, d_k_out, d_v_out, as_stream(stream));
    }
}

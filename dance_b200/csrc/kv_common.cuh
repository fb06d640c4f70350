// kv_common.cuh -- what the key/value cache kernels share: the device view of
// a cache and a batch, argument checks, and the 8-bit code arithmetic.
//
// A code c in 1..255 stands for (c - 128) * scale.  Two exact routes lead
// from codes to matrix operands:
//  * as halves: the byte under 0x64 is the half 1024 + c, and 1024 + c - 1152
//    is c - 128 without rounding (every step is an integer below 2048);
//  * as bytes of an integer product, the 128 taken out of the sum.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "../../include/dance_b200.h"
#include "func_attr.cuh"
#include "host_errors.cuh"

namespace dance
{

constexpr unsigned kKvFull = 0xFFFFFFFFu;
constexpr float kKvTiny = 1.17549435e-38f; // 2^-126: a smaller scale has no finite reciprocal and counts as 0
constexpr float kKvNegInf = -__builtin_huge_valf();

// Device view of the cache and of the call's sequences.
struct KvView
{
    uint8_t *k, *v;
    float *ks, *vs;
    uint8_t *bounds;
    uint64_t kbs, vbs; // block strides, bytes
    uint32_t num_blocks, hkv, shift;
    const int32_t *table, *lens, *offs;
    uint32_t width, batch, max_rows, max_len;
};

inline KvView kv_view(const DanceKvCache &c, const DanceKvBatch &b)
{
    uint32_t shift = 0;
    while ((1u << shift) < c.block_tokens)
        ++shift;
    return {c.d_k,         c.d_v,          c.d_k_scale,     c.d_v_scale,   c.d_k_bounds,  c.k_block_stride,
            c.v_block_stride, c.num_blocks, c.kv_heads,     shift,         b.d_block_table, b.d_seq_lens,
            b.d_row_offsets,  b.table_width, b.batch,       b.max_rows,    b.max_len};
}

// One sequence of the batch, clipped to what the launch and the tensors cover.
struct KvSeq
{
    int row0, rows, first; // first row of the call's tensors, row count, position of the first row
    int len;               // tokens held
};

__device__ __forceinline__ KvSeq kv_seq(const KvView &c, uint32_t b, uint32_t total_rows)
{
    KvSeq s;
    const int64_t cap = (int64_t)c.width << c.shift;
    const int n = c.lens[b];
    s.row0 = c.offs[b];
    s.rows = c.offs[b + 1] - s.row0;
    s.first = n - s.rows;
    s.len = (int)min((int64_t)min(n, (int)min(c.max_len, 0x7FFFFFFFu)), cap);
    if (s.row0 < 0 || s.rows < 0)
        s.row0 = 0, s.rows = 0;
    s.rows = min(s.rows, (int)min(c.max_rows, 0x7FFFFFFFu));
    s.rows = min(s.rows, max(0, (int)min((int64_t)total_rows - s.row0, (int64_t)0x7FFFFFFF)));
    return s;
}

// Physical block of position `page` of sequence b, -1 where there is none.
__device__ __forceinline__ int kv_block(const KvView &c, uint32_t b, int page)
{
    if (page < 0 || (uint32_t)page >= c.width)
        return -1;
    const int blk = __ldg(c.table + (uint64_t)b * c.width + page);
    return (uint32_t)blk < c.num_blocks ? blk : -1;
}

template <bool BF16>
__device__ __forceinline__ float kv_float(uint16_t u)
{
    if constexpr (BF16)
        return __uint_as_float((uint32_t)u << 16);
    else
        return __half2float(__ushort_as_half(u));
}

__device__ __forceinline__ uint16_t kv_round(float x, int dtype)
{
    return dtype == DANCE_BF16 ? __bfloat16_as_ushort(__float2bfloat16_rn(x)) : __half_as_ushort(__float2half_rn(x));
}

template <bool BF16>
__device__ __forceinline__ uint32_t kv_pack(float lo, float hi)
{
    if constexpr (BF16)
    {
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    else
    {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
}

// Scale of a set of finite magnitudes, and the code - 128 of a value at a
// step: 1/step is taken once, so that a value costs one product.
//
// A block's scale is the quotient amax / 127, the float nearest to it.  The step that
// codes are taken at is amax times the float nearest 1/127: the scale, or, for
// 4.6 % of all magnitudes, the float below it.  Where the two part, so do their
// codes only at half the magnitude, whose exact code 63.5 is a tie: the step
// gives the even 64, the scale for half of these magnitudes 63 (every pair of
// float16 and of bfloat16 numbers was compared with the exact quotient).
__device__ __forceinline__ float kv_scale_of(float amax)
{
    const float s = __fdiv_rn(amax, 127.0f);
    return s < kKvTiny ? 0.0f : s;
}
__device__ __forceinline__ float kv_step_of(float amax)
{
    const float s = __fmul_rn(amax, 1.0f / 127.0f);
    return s < kKvTiny ? 0.0f : s;
}
__device__ __forceinline__ float kv_inverse(float s) { return s >= kKvTiny ? __fdiv_rn(1.0f, s) : 0.0f; }
__device__ __forceinline__ int kv_code(float x, float inv)
{
    // min and max of NaN and a number give the number: NaN is told apart first
    const float y = __fmul_rn(x, inv);
    return y != y ? 0 : __float2int_rn(fminf(fmaxf(y, -127.0f), 127.0f));
}
__device__ __forceinline__ float kv_finite_abs(float x)
{
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;
}

// ------------------------------------------------------------------ host checks
inline int kv_check(const DanceKvCache *c, const DanceKvBatch *b)
{
    if (!c || !b)
        return fail(-1, "null key/value cache or batch");
    if (!c->d_k || !c->d_v || !c->d_k_scale || !c->d_v_scale || !c->d_k_bounds)
        return fail(-1, "key/value cache with a null tensor");
    if (c->head_dim != 64 && c->head_dim != 96 && c->head_dim != 128)
        return fail(-1, "head_dim %u: 64, 96 or 128 are supported", c->head_dim);
    if (c->block_tokens != 16 && c->block_tokens != 32 && c->block_tokens != 64 && c->block_tokens != 128)
        return fail(-1, "block_tokens %u: 16, 32, 64 or 128 are supported", c->block_tokens);
    if (c->kv_heads == 0 || c->kv_heads > 1024 || c->num_blocks == 0 || c->num_blocks > 0x7FFFFFFFu)
        return fail(-1, "key/value cache of %u blocks x %u heads", c->num_blocks, c->kv_heads);
    const uint64_t block = (uint64_t)c->kv_heads * c->block_tokens * c->head_dim;
    if (c->k_block_stride < block || c->v_block_stride < block || c->k_block_stride % 16 || c->v_block_stride % 16)
        return fail(-1, "block strides %llu and %llu must be multiples of 16 and hold %llu bytes",
                    (unsigned long long)c->k_block_stride, (unsigned long long)c->v_block_stride,
                    (unsigned long long)block);
    if (((uintptr_t)c->d_k | (uintptr_t)c->d_v | (uintptr_t)c->d_k_bounds) % 16)
        return fail(-1, "key/value cache tensors must be 16-byte aligned");
    if (((uintptr_t)c->d_k_scale | (uintptr_t)c->d_v_scale) % 4)
        return fail(-1, "key/value cache scales must be 4-byte aligned");
    if (!b->d_seq_lens || !b->d_row_offsets || (!b->d_block_table && b->table_width))
        return fail(-1, "batch with a null tensor");
    if (b->batch == 0 || b->batch > 65535)
        return fail(-1, "batch of %u sequences: 1 to 65535 are supported", b->batch);
    if (b->max_len > 0x40000000u || b->max_rows > 0x1000000u || b->table_width > 0x10000000u)
        return fail(-1, "batch of max_rows %u, max_len %u, table width %u is too large", b->max_rows, b->max_len,
                    b->table_width);
    return 0;
}

inline int kv_check_rows(const DanceKvRows *r, const char *name)
{
    if (!r)
        return fail(-1, "null rows %s", name);
    if (r->dtype != DANCE_F16 && r->dtype != DANCE_BF16)
        return fail(-1, "%s of dtype %d: float16 and bfloat16 are supported", name, r->dtype);
    if (r->rows == 0)
        return 0;
    if (!r->d_data || (uintptr_t)r->d_data % 2)
        return fail(-1, "null or misaligned rows %s", name);
    if (r->rows > 0x7FFFFFFFu)
        return fail(-1, "%s has too many rows", name);
    return 0;
}

// Whether every (row, head) vector of the tensor starts on 16 bytes.
inline bool kv_aligned(const DanceKvRows &r)
{
    return (uintptr_t)r.d_data % 16 == 0 && r.row_stride % 8 == 0 && r.head_stride % 8 == 0;
}

} // namespace dance

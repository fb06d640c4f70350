// kv_attention.cuh -- what the two attention kernels over the 8-bit cache
// share: parameters, code conversion, and the plan of a call.
#pragma once

#include "kv_common.cuh"

namespace dance
{

constexpr uint32_t kCounters = 1u << 16; // arrival counters at the head of the workspace
constexpr int kMaxPos = 0x3FFFFFFF;      // position of tokens that no row sees

struct AttnParams
{
    KvView c;
    const uint16_t *q;
    uint64_t q_row, q_head;
    uint32_t rows, heads, G;
    bool q_aligned;
    float scale_log2;
    const int32_t *blocks; // sparse: rows x hkv x select
    uint32_t select;
    uint32_t group;     // sparse: query tokens that share a thread block
    uint32_t groups;    // sparse: such groups of a sequence
    uint32_t chunk;     // cache blocks of one split
    uint32_t splits;    // most splits of a sequence
    uint32_t row_tiles; // row tiles of a (sequence or row, head)
    void *out;
    float *lse;
    uint32_t *counters;
    float *part; // partial outputs, then partial log-sums
    long long wait_clocks; // limit of a wait on a barrier (prompt kernel)
};

// How a call is cut: row tiles, splits, workspace.
struct AttnPlan
{
    bool prompt;  // the kernel of many rows
    uint32_t nt;  // eights of rows of a tile (few rows)
    uint32_t group, groups; // sparse: see AttnParams
    uint32_t row_tiles, chunk, splits;
    uint64_t blocks_x, bytes;
};

// Rows of a tile of the kernel of many rows (kv_prompt.cu).
constexpr uint32_t kPromptRows = 256;
constexpr uint32_t kPromptTokens = 128;
int launch_prompt(AttnParams &p, uint32_t head_dim, bool bf16, uint32_t blocks_x, cudaStream_t st);

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ float exp2_fast(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
    return y;
}

// Two bytes of w (sel 0x4140: the low two, 0x4342: the high two) as the
// halves c - 128.
__device__ __forceinline__ uint32_t code_halves(uint32_t w, uint32_t sel)
{
    const uint32_t u = __byte_perm(w, 0x64646464u, sel);
    const __half2 r = __hsub2(*reinterpret_cast<const __half2 *>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t *>(&r);
}

// The power of two that brings the largest channel of a row to [2^13, 2^14),
// as the exponent to add; rows of zeros or without a largest stay as they are.
__device__ __forceinline__ int row_shift(float amax)
{
    const int ex = (int)(__float_as_uint(amax) >> 23);
    return (ex == 255 || amax == 0.0f) ? 0 : min(126, 127 + 13 - ex);
}
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float((uint32_t)(127 + e) << 23); }
// The least whole number above log2 of a value scale; -126 for 0.
__device__ __forceinline__ float scale_exponent(float s)
{
    // the exponent's bits as the last of 2^23 + e, exactly
    return __uint_as_float((__float_as_uint(s) >> 23) | 0x4B000000u) - (8388608.0f + 126.0f);
}

} // namespace dance

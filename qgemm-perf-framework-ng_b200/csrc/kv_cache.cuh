// kv_cache.cuh -- the q4_0 key/value cache and the value formats shared by
// the kernels of the attention step (kv_plan.cu, qk_norm_rope.cu,
// kv_append.cu, attn_*.cu).
//
// A cache (K and V have one each) is [pages][heads_kv][page_size / 16] groups
// of 16 tokens.  A group of head dimension D holds 16 nibble rows of D / 2
// bytes, then 16 rows of D / 32 fp16 scales: 9 D bytes, a multiple of 16 (D is
// a multiple of 32), so any run of groups of one page and head is one
// contiguous, 16-byte aligned piece for a bulk copy.
//
// A value is d * (n - 8), d and n those of ggml's block_q4_0 (byte i of a
// block: value i in the low nibble, value i + 16 in the high one).  Within a
// token's row the bytes of its B = D / 32 blocks are interleaved so that one
// wide load gives a tensor-core thread its share of every block:
//   K: byte 4 t + e (t, e = 0..3) of block b at t * 4 B + 4 b + e
//   V: byte 2 g + e (g = 0..7, e = 0, 1) of block b at g * 2 B + 2 b + e
// With K as the A operand of m16n8k16 (rows = keys), thread t of a quad reads
// 4 B bytes: a word per block, whose masks and one shift are its A fragments
// (the order of k within a block is free as long as Q follows it).  With V^T
// as the A operand (rows = dimensions), thread group g reads 2 B bytes of a
// key: two bytes per block, so an MMA stays within a block and the block's
// scale can go into the probabilities, which leaves n - 8 exact.
#pragma once

#include <cuda_bf16.h>

#include "pfng_common.cuh"
#include "pfng_internal.h"

namespace pfng {

constexpr int kKvGroup = 16;  // tokens of a group
__host__ __device__ constexpr int kv_row_bytes(int dim) { return dim / 2; }
__host__ __device__ constexpr int kv_group_bytes(int dim) { return 9 * dim; }
__host__ __device__ constexpr int kv_scale_offset(int dim) { return 8 * dim; }

// First byte of the group that holds (page, head, offset within the page).
PFNG_DEV int64_t kv_group_offset(int64_t page, int head, int offset, int heads, int groups, int dim) {
    return ((page * heads + head) * groups + offset / kKvGroup) * kv_group_bytes(dim);
}

// ---- values in fp32 / fp16 / bf16 (the kOutF32 / kOutF16 / kOutBF16 codes) ----
PFNG_DEV int format_bytes(int fmt) { return fmt == kOutF32 ? 4 : 2; }

// N consecutive values (N = 1, 4 or 8) at element `at`; N > 1 needs the
// address aligned to N elements or 16 bytes, whichever is less.
template <int N>
PFNG_DEV void load_values(int fmt, const void *p, int64_t at, float (&v)[N]) {
    if (fmt == kOutF32) {
        const float *f = static_cast<const float *>(p) + at;
        if constexpr (N == 1) {
            v[0] = *f;
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4) {
                const float4 q = *reinterpret_cast<const float4 *>(f + i);
                v[i] = q.x, v[i + 1] = q.y, v[i + 2] = q.z, v[i + 3] = q.w;
            }
        }
        return;
    }
    const uint16_t *h = static_cast<const uint16_t *>(p) + at;
    uint32_t w[(N + 1) / 2];
    if constexpr (N == 1) {
        w[0] = *h;
    } else if constexpr (N == 4) {
        const uint2 q = *reinterpret_cast<const uint2 *>(h);
        w[0] = q.x, w[1] = q.y;
    } else {
        const uint4 q = *reinterpret_cast<const uint4 *>(h);
        w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const uint32_t b = (w[i / 2] >> (16 * (i & 1))) & 0xffffu;
        v[i] = fmt == kOutBF16 ? __uint_as_float(b << 16) : f16_bits_to_f32(b);
    }
}

PFNG_DEV uint32_t pack_values(int fmt, float a, float b) {
    if (fmt == kOutBF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&h);
    }
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// load_values in two steps, for loops that start several loads before they use
// the first: the bits, then their values.
template <int FMT, int N>
struct RawValues {
    static constexpr int kWords = FMT == kOutF32 ? N : (N + 1) / 2;
    uint32_t w[kWords];
    PFNG_DEV void zero() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) w[i] = 0;
    }
    PFNG_DEV void load(const void *p, int64_t at) {
        const uint8_t *b = static_cast<const uint8_t *>(p) + at * (FMT == kOutF32 ? 4 : 2);
        if constexpr (N == 1) {
            w[0] = FMT == kOutF32 ? *reinterpret_cast<const uint32_t *>(b) : *reinterpret_cast<const uint16_t *>(b);
        } else if constexpr (kWords == 2) {
            const uint2 q = *reinterpret_cast<const uint2 *>(b);
            w[0] = q.x, w[1] = q.y;
        } else {
#pragma unroll
            for (int i = 0; i < kWords; i += 4) {
                const uint4 q = *reinterpret_cast<const uint4 *>(b + 4 * i);
                w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
            }
        }
    }
    PFNG_DEV float operator[](int i) const {
        if constexpr (FMT == kOutF32) return __uint_as_float(w[i]);
        const uint32_t b = (w[i / 2] >> (16 * (i & 1))) & 0xffffu;
        return FMT == kOutBF16 ? __uint_as_float(b << 16) : f16_bits_to_f32(b);
    }
};

// The counterpart of load_values; fp32 -> fp16 / bf16 rounds to nearest even,
// the one rounding of a result.
template <int N>
PFNG_DEV void store_values(int fmt, void *p, int64_t at, const float (&v)[N]) {
    if (fmt == kOutF32) {
        float *f = static_cast<float *>(p) + at;
        if constexpr (N == 1) {
            *f = v[0];
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<float4 *>(f + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        }
        return;
    }
    uint16_t *h = static_cast<uint16_t *>(p) + at;
    if constexpr (N == 1) {
        *h = static_cast<uint16_t>(pack_values(fmt, v[0], 0.0f) & 0xffffu);
    } else if constexpr (N == 4) {
        *reinterpret_cast<uint2 *>(h) = make_uint2(pack_values(fmt, v[0], v[1]), pack_values(fmt, v[2], v[3]));
    } else {
        *reinterpret_cast<uint4 *>(h) = make_uint4(pack_values(fmt, v[0], v[1]), pack_values(fmt, v[2], v[3]),
                                                   pack_values(fmt, v[4], v[5]), pack_values(fmt, v[6], v[7]));
    }
}

}  // namespace pfng

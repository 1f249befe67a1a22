// kv_append.cu -- new keys and values quantized to q4_0 into the pages of the
// cache (pfng_b200_kv_append_q4_0).
//
// Per 32 values of a head (the quantizer of quantize_q4_0, bit for bit; the
// reference's quantize_row_q4_0, llama_reference.cpp:13-36): the first value m
// of largest magnitude, d = m / -8, n_i = min(15, trunc(x_i / d + 8.5)) with
// 1 / d rounded once, d stored as fp16.
//
// Four lanes hold a block, eight values each (16 or 32 bytes, one or two wide
// loads), so the search for m is two shuffle steps; each lane then trades its
// nibbles with the lane that holds the other half of its bytes and stores
// four bytes of the row.  The 16 rows of a group are contiguous, so a run of
// tokens is written in whole sectors.
#include "kv_cache.cuh"

namespace pfng {
namespace {

constexpr int kThreads = 256;

template <bool kVec>
PFNG_DEV void load8(int fmt, const void *p, int64_t at, float (&v)[8]) {
    if constexpr (kVec) {
        load_values<8>(fmt, p, at, v);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float one[1];
            load_values<1>(fmt, p, at + i, one);
            v[i] = one[0];
        }
    }
}

template <bool kVec>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendArgs p) {
    const int blocks = static_cast<int>(p.head_dim / 32);
    const int64_t per_token = p.heads_kv * blocks;  // q4_0 blocks of K (and of V) of a token
    const int64_t half = p.tokens * per_token;
    const int quad = threadIdx.x & 3;
    const int64_t id = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 2;
    const bool is_v = id >= half;
    const int64_t bi = is_v ? id - half : id;
    const bool live = bi < half;
    const int64_t token = live ? bi / per_token : 0;
    const int rest = live ? static_cast<int>(bi % per_token) : 0;
    const int head = rest / blocks, block = rest % blocks;
    const int64_t slot = live ? p.slots[token] : -1;
    const bool write = slot >= 0 && slot < p.num_pages * p.page_size;
    float v[8] = {};
    if (write)
        load8<kVec>(is_v ? p.v_format : p.k_format, is_v ? p.v : p.k,
                    token * (is_v ? p.ldv : p.ldk) + static_cast<int64_t>(head) * p.head_dim + 32 * block + 8 * quad,
                    v);
    float amax = 0.0f, smax = 0.0f;
    int first = 1 << 30;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (amax < fabsf(v[i])) amax = fabsf(v[i]), smax = v[i], first = 8 * quad + i;
#pragma unroll
    for (int o = 1; o < 4; o <<= 1) {
        const float oa = __shfl_xor_sync(0xffffffffu, amax, o), os = __shfl_xor_sync(0xffffffffu, smax, o);
        const int oi = __shfl_xor_sync(0xffffffffu, first, o);
        if (oa > amax || (oa == amax && oi < first)) amax = oa, smax = os, first = oi;
    }
    const float d = __fdiv_rn(smax, -8.0f);
    const float inv = d != 0.0f ? __fdiv_rn(1.0f, d) : 0.0f;
    uint32_t n[2] = {0, 0};  // nibbles of values 8 quad .. + 3 and + 4 .. + 7, one a byte
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        int q = __float2int_rz(__fadd_rn(__fmul_rn(v[i], inv), 8.5f));
        q = min(static_cast<int>(static_cast<int8_t>(q)), 15);
        n[i / 4] |= (static_cast<uint32_t>(q) & 15u) << (8 * (i % 4));
    }
    // bytes 8 a .. 8 a + 7 of the block are lanes a (low nibbles) and a + 2
    // (high nibbles), a = 0, 1: lane a stores the first four, lane a + 2 the
    // last four, so each needs one word of the other
    const uint32_t other = __shfl_xor_sync(0xffffffffu, quad < 2 ? n[1] : n[0], 2);
    const uint32_t bytes = quad < 2 ? n[0] | (other << 4) : other | (n[1] << 4);
    const int word = 2 * (quad & 1) + (quad >> 1);  // bytes 4 word .. 4 word + 3
    if (!write) return;
    const int64_t page = slot / p.page_size;
    const int offset = static_cast<int>(slot % p.page_size), row = offset % kKvGroup;
    const int dim = static_cast<int>(p.head_dim);
    uint8_t *group = (is_v ? p.v_cache : p.k_cache) +
                     kv_group_offset(page, head, offset, static_cast<int>(p.heads_kv),
                                     static_cast<int>(p.page_size / kKvGroup), dim);
    uint8_t *to = group + row * kv_row_bytes(dim);
    if (!is_v) {
        *reinterpret_cast<uint32_t *>(to + word * 4 * blocks + 4 * block) = bytes;
    } else {
        *reinterpret_cast<uint16_t *>(to + (2 * word) * 2 * blocks + 2 * block) = static_cast<uint16_t>(bytes);
        *reinterpret_cast<uint16_t *>(to + (2 * word + 1) * 2 * blocks + 2 * block) =
            static_cast<uint16_t>(bytes >> 16);
    }
    if (quad == 0)
        *reinterpret_cast<uint16_t *>(group + kv_scale_offset(dim) + 2 * (row * blocks + block)) = f32_to_f16_bits(d);
}

}  // namespace

cudaError_t launch_kv_append(const AppendArgs &p, cudaStream_t s) {
    const auto wide = [](const void *x, int64_t ld, int fmt) {
        return (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && ld % (fmt == kOutF32 ? 4 : 8) == 0;
    };
    const int64_t threads = 2 * p.tokens * p.heads_kv * (p.head_dim / 32) * 4;
    const unsigned grid = static_cast<unsigned>((threads + kThreads - 1) / kThreads);
    if (wide(p.k, p.ldk, p.k_format) && wide(p.v, p.ldv, p.v_format))
        kv_append_kernel<true><<<grid, kThreads, 0, s>>>(p);
    else
        kv_append_kernel<false><<<grid, kThreads, 0, s>>>(p);
    return cudaGetLastError();
}

}  // namespace pfng

// qk_norm_rope.cu -- RMS norm of every query and key head and the position
// rotation in one pass (pfng_b200_qk_norm_rope).
//
//   y = x / sqrt(mean(x^2) + eps) * w           (skipped without w)
//   (a, b) -> (a cos - b sin, b cos + a sin)    for the R / 2 pairs of a head
//
// A head of D values is D / 2 slots of two values: slot s < R / 2 is a pair
// that turns -- (s, s + R / 2), or (2 s, 2 s + 1) when interleaved -- and the
// slots behind it are the D - R values that do not.  A lane holds N
// consecutive slots, so both values of a pair are in one lane and the only
// exchange is the sum of squares over the lanes of a head.  Everything is in
// fp32 registers between one read and one write (rounded once, at the write).
#include "kv_cache.cuh"

namespace pfng {
namespace {

constexpr int kThreads = 128;

// Elements of slots s .. s + N - 1: N values from a and N from b.  Interleaved
// pairs are adjacent: 2 N values in a row, b = a + N.
template <int N>
PFNG_DEV void slot_elements(const RopeArgs &p, int s, int &a, int &b, bool &turns, bool &adjacent) {
    const int half = static_cast<int>(p.rot_dim / 2);
    turns = s < half;
    adjacent = turns && p.interleaved;
    if (turns) {
        a = p.interleaved ? 2 * s : s;
        b = p.interleaved ? 2 * s + N : s + half;
    } else {
        a = static_cast<int>(p.rot_dim) + s - half;
        b = a + static_cast<int>(p.head_dim - p.rot_dim) / 2;
    }
}

template <int N>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(const RopeArgs p, int lanes) {
    const int heads = static_cast<int>(p.heads_q + p.heads_k);
    const int lane = threadIdx.x & 31, sub = lane % lanes;
    const int slots = static_cast<int>(p.head_dim / 2);
    const int per_warp = 32 / lanes;
    const int64_t rows = p.tokens * heads;
    const int64_t row = ((static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> 5) * per_warp + lane / lanes;
    const bool live = row < rows;
    const int64_t token = live ? row / heads : 0;
    const int head = live ? static_cast<int>(row % heads) : 0;
    const bool is_q = head < p.heads_q;
    const float *weight = is_q ? p.q_weight : p.k_weight;
    float v[2][8 / N][N] = {};
    // slots of this lane: sub * N + i * lanes * N
    constexpr int kMost = 8 / N;  // head_dim <= 512: at most kMost pieces a lane
    const int pieces = (slots + lanes * N - 1) / (lanes * N);
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int s = (i * lanes + sub) * N;
        if (i < pieces && live && s < slots) {
            int a, b;
            bool turns, adjacent;
            slot_elements<N>(p, s, a, b, turns, adjacent);
            const int64_t at = token * p.ldx + static_cast<int64_t>(head) * p.head_dim;
            load_values<N>(p.in_format, p.x, at + a, v[0][i]);
            load_values<N>(p.in_format, p.x, at + b, v[1][i]);
#pragma unroll
            for (int j = 0; j < N; ++j) sum += v[0][i][j] * v[0][i][j] + v[1][i][j] * v[1][i][j];
        }
    }
    for (int o = 1; o < lanes; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (!live) return;
    const float scale = weight ? 1.0f / sqrtf(sum / static_cast<float>(p.head_dim) + p.eps) : 1.0f;
    const int64_t pos = p.positions[token];
    const bool known = pos >= 0 && pos < p.max_pos;
    void *out = is_q ? p.q_out : p.k_out;
    const int64_t to = is_q ? token * p.ldq + static_cast<int64_t>(head) * p.head_dim
                            : token * p.ldk + static_cast<int64_t>(head - p.heads_q) * p.head_dim;
    // padding rows (no position) are zeros, a position past the table is NaN
    const float blank = pos < 0 ? 0.0f : __int_as_float(0x7fffffff);
#pragma unroll
    for (int i = 0; i < kMost; ++i) {
        const int s = (i * lanes + sub) * N;
        if (i >= pieces || s >= slots) continue;
        int a, b;
        bool turns, adjacent;
        slot_elements<N>(p, s, a, b, turns, adjacent);
        float c[N], z[N], u[N], w[N];
#pragma unroll
        for (int j = 0; j < N; ++j) c[j] = 1.0f, z[j] = 0.0f;
        if (turns && known) {
            load_values<N>(kOutF32, p.cos_sin, pos * p.rot_dim + s, c);
            load_values<N>(kOutF32, p.cos_sin, pos * p.rot_dim + p.rot_dim / 2 + s, z);
        }
        // adjacent pairs come in as 2 N values in a row
        float first[N], second[N];
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int e0 = 2 * j, e1 = 2 * j + 1;
            first[j] = adjacent ? (e0 < N ? v[0][i][e0 % N] : v[1][i][e0 % N]) : v[0][i][j];
            second[j] = adjacent ? (e1 < N ? v[0][i][e1 % N] : v[1][i][e1 % N]) : v[1][i][j];
        }
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const int fa = adjacent ? a + 2 * j : a + j, sa = adjacent ? a + 2 * j + 1 : b + j;
            const float x0 = weight ? first[j] * scale * weight[fa] : first[j];
            const float x1 = weight ? second[j] * scale * weight[sa] : second[j];
            u[j] = known ? x0 * c[j] - x1 * z[j] : blank;
            w[j] = known ? x1 * c[j] + x0 * z[j] : blank;
        }
        if (adjacent) {
            float lo[N], hi[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                lo[j] = (j & 1) ? w[j / 2] : u[j / 2];
                hi[j] = ((N + j) & 1) ? w[(N + j) / 2] : u[(N + j) / 2];
            }
            store_values<N>(p.out_format, out, to + a, lo);
            store_values<N>(p.out_format, out, to + b, hi);
        } else {
            store_values<N>(p.out_format, out, to + a, u);
            store_values<N>(p.out_format, out, to + b, w);
        }
    }
}

bool aligned_to(const void *p, uintptr_t a) { return (reinterpret_cast<uintptr_t>(p) & (a - 1)) == 0; }
uintptr_t vec_bytes(int fmt) { return fmt == kOutF32 ? 16 : 8; }

}  // namespace

cudaError_t launch_qk_norm_rope(const RopeArgs &p, cudaStream_t s) {
    // Four slots a lane where every piece of four is aligned and on one side
    // of the rotated part; one slot a lane otherwise.
    const bool vec = p.rot_dim % 8 == 0 && p.head_dim % 8 == 0 && p.ldx % 4 == 0 && p.ldq % 4 == 0 &&
                     p.ldk % 4 == 0 && aligned_to(p.x, vec_bytes(p.in_format)) &&
                     aligned_to(p.q_out, vec_bytes(p.out_format)) && aligned_to(p.k_out, vec_bytes(p.out_format)) &&
                     aligned_to(p.cos_sin, 16);
    const int64_t rows = p.tokens * (p.heads_q + p.heads_k);
    const int slots = static_cast<int>(p.head_dim / 2);
    int lanes = 1;
    while (lanes < 32 && lanes * (vec ? 4 : 1) < slots) lanes *= 2;
    const int64_t per_block = kThreads / lanes;
    const unsigned grid = static_cast<unsigned>((rows + per_block - 1) / per_block);
    if (vec)
        qk_norm_rope_kernel<4><<<grid, kThreads, 0, s>>>(p, lanes);
    else
        qk_norm_rope_kernel<1><<<grid, kThreads, 0, s>>>(p, lanes);
    return cudaGetLastError();
}

}  // namespace pfng

// Pieces shared by the kernels that multiply activations by packed matrices (gfx950, wave64).
//
// A packed matrix stands for W = diag(suh) H_L X H_R diag(svh), with E4M3 labels X and H the normalised Hadamard on
// blocks of 128.  H and the scales move to the activations:
//   x W = ((xr X) H_R) * svh,   xr = (x * suh) H
// so a product reads the payload's bits and nothing wider: the rows xr go in as two bf16 pieces (hi + lo, 16 bits of
// significand), the labels are exact in bf16, sums are FP32.
#pragma once

#include "common.h"

namespace qsrt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// Rotated rows in memory: a row of K channels is K / 32 strips of 128 bytes, one for 32 payload rows: the strip's 32 hi
// pieces, then its 32 lo pieces, both in the order in which a lane of the product takes them: for lane group g = 0..3 the
// eight channels 16 h + {2g, 2g + 1, 2g + 8, 2g + 9}, h = 0, 1 (the rows that a trellis window of a tile covers).
constexpr int kStripBytes = 128;

constexpr float kHadamardScale = 0.08838834764831845f;  // 128^-1/2

template <int kControl>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kControl, 0xF, 0xF, true));
}

// One butterfly stage between lanes that differ in bit h: lower + upper in the lower, lower - upper in the upper one.
// `sign` is -1 in the upper lane.  Bits 0..3 stay within a row of 16 lanes (data-parallel moves), 16 and 32 are swaps.
template <int h>
__device__ __forceinline__ float stage(float v, float sign) {
    if constexpr (h == 1) return __builtin_fmaf(sign, v, dpp<0xB1>(v));              // quad_perm 1 0 3 2
    if constexpr (h == 2) return __builtin_fmaf(sign, v, dpp<0x4E>(v));              // quad_perm 2 3 0 1
    if constexpr (h == 4) return __builtin_fmaf(sign, v, dpp<0x1B>(dpp<0x141>(v)));  // half mirror, then quad_perm 3 2 1 0
    if constexpr (h == 8) return __builtin_fmaf(sign, v, dpp<0x128>(v));             // row rotated by 8
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto both = h == 16 ? __builtin_amdgcn_permlane16_swap(u, u, false, false)
                              : __builtin_amdgcn_permlane32_swap(u, u, false, false);
    const uint32_t lower = both[0], upper = both[1];
    return __builtin_fmaf(sign, __builtin_bit_cast(float, upper), __builtin_bit_cast(float, lower));
}

// Unnormalised 128-point Sylvester Hadamard over a wave that holds channels 2 lane and 2 lane + 1.  The 2 x 2 exact
// stages cost 7 x 2 VALU instructions and no LDS; short code matters here, as the kernels around a product run it once.
__device__ __forceinline__ void hadamard128(float& a, float& b, int lane) {
    const float x = a, y = b;
    a = x + y;
    b = x - y;
#define QSRT_STAGE(h)                                \
    {                                                \
        const float sign = (lane & h) ? -1.f : 1.f;  \
        a = stage<h>(a, sign);                       \
        b = stage<h>(b, sign);                       \
    }
    QSRT_STAGE(1) QSRT_STAGE(2) QSRT_STAGE(4) QSRT_STAGE(8) QSRT_STAGE(16) QSRT_STAGE(32)
#undef QSRT_STAGE
}

// Channels 2 lane, 2 lane + 1 of a rotated row's block of 128, split and stored in the product's order: channel rho of a
// tile's 16 lies in lane group (rho % 8) / 2, at place (rho & 1) + 2 (rho / 8) of the tile's four.
__device__ __forceinline__ void store_pieces(char* block, int lane, float a, float b) {
    const __bf16 h0 = static_cast<__bf16>(a), h1 = static_cast<__bf16>(b);
    const bf16x2 lo = {static_cast<__bf16>(a - static_cast<float>(h0)), static_cast<__bf16>(b - static_cast<float>(h1))};
    const int tile = lane >> 3, pair = lane & 7;  // channels 2 pair, 2 pair + 1 of the tile
    char* dst = block + (tile >> 1) * kStripBytes + (pair & 3) * 16 + (tile & 1) * 8 + (pair >> 2) * 4;
    *reinterpret_cast<bf16x2*>(dst) = bf16x2{h0, h1};
    *reinterpret_cast<bf16x2*>(dst + 64) = lo;
}

// Rows of one key (an expert, an adapter) in groups that one wave multiplies at once.
struct Chunk {
    int key, first, count, pad;  // rows order[first .. first + count)
};

// Head of a grouping: what the host cannot know when it launches what reads it.
struct GroupHead {
    int chunks;
    int parts[2];  // parts that the K axis of a layer's first and second product is cut into
    int pad;
};

// Cuts the K axis (`strips`) of `units` products into parts so that `waves` waves come out even: the fewest strips in turn
// on one wave, with two strips' time for what an item costs beside them.  A whole wave asks; every lane gets the answer.
__device__ __forceinline__ int choose_parts(int64_t units, int strips, int max_parts, int waves, int lane) {
    int64_t best = INT64_MAX;
    for (int s = lane + 1; s <= min(max_parts, strips); s += 64) {
        if (units * s >= int64_t(1) << 31) break;  // the product counts its items in 32 bits
        const int64_t rounds = (units * s + waves - 1) / waves;
        const int64_t cost = rounds * ((strips + s - 1) / s + 2) << 16 | s;  // ties: the fewest parts
        best = cost < best ? cost : best;
    }
    for (int h = 1; h < 64; h <<= 1) {
        const int64_t o = __shfl_xor(static_cast<long long>(best), h);
        best = o < best ? o : best;
    }
    return best == INT64_MAX ? 1 : static_cast<int>(best & 0xFFFF);
}

struct GroupArgs {
    const int* ids;
    int n, keys;
    bool none;       // rows without a key form a group of their own (key -1)
    int chunk_rows;
    GroupHead* head;
    Chunk* chunks;
    int* order;
    int* clean;      // ids with everything outside [0, keys) as -1
    int units[2], strips[2], max_parts[2];  // per product: column blocks (times matrices) a chunk has, K axis, limit
    int waves;
};

constexpr int kMaxKeys = 8191;  // their counters fit LDS

int launch_group(const GroupArgs& args, hipStream_t stream);

}  // namespace qsrt

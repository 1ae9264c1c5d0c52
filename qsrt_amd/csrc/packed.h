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
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// Rotated rows in memory: a row of K channels is K / 32 strips of 128 bytes, one for 32 payload rows: the strip's 32 hi
// pieces, then its 32 lo pieces, both in the order in which a lane of the product takes them: for lane group g = 0..3 the
// eight channels 16 h + {2g, 2g + 1, 2g + 8, 2g + 9}, h = 0, 1 (the rows that a trellis window of a tile covers).
constexpr int kStripBytes = 128;

// A wave holds 128 channels of 16 rows as v[4 a + i] = channel 16 a + 4 g + i of row n, lane = 16 g + n.
// Unnormalised 128-point Sylvester Hadamard of every row: stages over a and i in registers, over g across lanes.
__device__ __forceinline__ void hadamard128(float (&v)[32], int lane) {
#pragma unroll
    for (int h = 1; h < 32; h <<= 1) {
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            if (j & h) continue;
            const float x = v[j], y = v[j + h];
            v[j] = x + y;
            v[j + h] = x - y;
        }
    }
#pragma unroll
    for (int h = 16; h < 64; h <<= 1) {
        const bool upper = (lane & h) != 0;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const float o = __shfl_xor(v[j], h);
            v[j] = upper ? o - v[j] : v[j] + o;
        }
    }
}

constexpr float kHadamardScale = 0.08838834764831845f;  // 128^-1/2

// Channels 16 a + 4 g .. + 3 of a rotated row, split and stored in the product's order.  rho = 4 g + i lies in lane group
// (rho % 8) / 2 of its tile, at place (rho & 1) + 2 (rho / 8) of four.
__device__ __forceinline__ void store_pieces(char* block, int a, int g, float v0, float v1, float v2, float v3) {
    const float v[4] = {v0, v1, v2, v3};
    __bf16 hi[4], lo[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        hi[i] = static_cast<__bf16>(v[i]);
        lo[i] = static_cast<__bf16>(v[i] - static_cast<float>(hi[i]));
    }
    char* strip = block + (a >> 1) * kStripBytes;
#pragma unroll
    for (int p = 0; p < 2; ++p) {  // channel pairs (0, 1) and (2, 3)
        const int group = 2 * (g & 1) + p, place = 2 * (g >> 1) + 4 * (a & 1);
        char* dst = strip + group * 16 + place * 2;
        *reinterpret_cast<bf16x2*>(dst) = bf16x2{hi[2 * p], hi[2 * p + 1]};
        *reinterpret_cast<bf16x2*>(dst + 64) = bf16x2{lo[2 * p], lo[2 * p + 1]};
    }
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

// Pieces shared by the kernels that multiply activations by packed matrices (gfx950, wave64).
//
// A packed matrix stands for W = diag(suh) H_L X H_R diag(svh), with E4M3 labels X and H the normalised Hadamard on
// blocks of 128.  H and the scales move to the activations:
//   x W = ((xr X) H_R) * svh,   xr = (x * suh) H
// so a product reads the payload's bits and nothing wider: the labels are exact in bf16 and f16, the rows xr go in as pieces
// that hold the 24 bits of an FP32 value between them, sums are FP32.
//   kBf16Pieces  hi + mid + lo, 8 bits and a sign each: any FP32 value, exactly
//   kF16Pieces   hi + lo, 11 bits and a sign each, of a row scaled by a power of two so that its largest value is near the
//                top of the type: 23 bits of values down to 2^-13 of the row's bound, 2^-40 of that bound below.  Two products
//                where bf16 takes three, for calls of many rows, which the matrix cores bound; the scale needs a look at the
//                whole row first.
#pragma once

#include "common.h"

namespace qsrt {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int kBf16Pieces = 3, kF16Pieces = 2;

// Rotated rows in memory.  A row of K channels is K / 32 strips, one for 32 payload rows: 32 values of each piece, as four
// times 16 bytes, what a lane of the product takes: for lane group g = 0..3 the eight channels 16 h + {2g, 2g + 1, 2g + 8,
// 2g + 9}, h = 0, 1 (the rows that a trellis window of a tile covers).  A few rows lie one after another; more are laid out
// by 16, [16 rows][strip][piece][g][row][16 bytes], so that a wave's load is one stretch (rows apart by a multiple of 4 KiB
// came from one L2 channel: a 2048 x 5120 x 1536 product took 125 us).
struct RowLayout {
    int row, strip, piece, group;  // bytes between neighbours
    int64_t sixteen;               // bytes of 16 rows
};
__host__ __device__ constexpr int strip_bytes(int pieces) { return 64 * pieces; }  // of one row
__host__ __device__ inline RowLayout row_layout(int kb, bool grouped, int pieces) {
    const int strip = strip_bytes(pieces);
    const int64_t bytes = static_cast<int64_t>(kb) * 4 * strip;
    return grouped ? RowLayout{16, 16 * strip, 1024, 256, 16 * bytes} : RowLayout{static_cast<int>(bytes), strip, 64, 16, 16 * bytes};
}
__host__ __device__ inline int64_t row_place(const RowLayout& l, int64_t row) { return (row >> 4) * l.sixteen + (row & 15) * l.row; }

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

// The pieces of a value: each the nearest of what is left, which is exact in FP32.
__device__ __forceinline__ void split(float v, __bf16 (&piece)[kBf16Pieces]) {
#pragma unroll
    for (int i = 0; i < kBf16Pieces; ++i) {
        piece[i] = static_cast<__bf16>(v);
        v -= static_cast<float>(piece[i]);
    }
}
__device__ __forceinline__ void split(float v, _Float16 (&piece)[kF16Pieces]) {
#pragma unroll
    for (int i = 0; i < kF16Pieces; ++i) {
        piece[i] = static_cast<_Float16>(v);
        v -= static_cast<float>(piece[i]);
    }
}

// Channels 2 lane, 2 lane + 1 of a rotated row's kb-th block of 128, split and stored in the product's order: channel rho of
// a tile's 16 lies in lane group (rho % 8) / 2, at place (rho & 1) + 2 (rho / 8) of the tile's four.
template <typename P, int kPieces>
__device__ __forceinline__ void store_pairs(char* row, const RowLayout& l, int kb, int lane, float a, float b) {
    typedef P p2 __attribute__((ext_vector_type(2)));
    P pa[kPieces], pb[kPieces];
    split(a, pa);
    split(b, pb);
    const int tile = lane >> 3, pair = lane & 7;  // channels 2 pair, 2 pair + 1 of the tile
    char* dst = row + (4 * kb + (tile >> 1)) * l.strip + (pair & 3) * l.group + (tile & 1) * 8 + (pair >> 2) * 4;
#pragma unroll
    for (int i = 0; i < kPieces; ++i) *reinterpret_cast<p2*>(dst + i * l.piece) = p2{pa[i], pb[i]};
}
__device__ __forceinline__ void store_pieces(char* row, const RowLayout& l, int kb, int lane, float a, float b) {
    store_pairs<__bf16, kBf16Pieces>(row, l, kb, lane, a, b);
}

// The same for channels `lane` and 64 + lane.
__device__ __forceinline__ void store_halves(char* row, const RowLayout& l, int kb, int lane, float a, float b) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        __bf16 piece[kBf16Pieces];
        split(h ? b : a, piece);
        const int tile = 4 * h + (lane >> 4), pair = (lane & 15) >> 1;
        char* dst = row + (4 * kb + (tile >> 1)) * l.strip + (pair & 3) * l.group + (tile & 1) * 8 + (pair >> 2) * 4 + (lane & 1) * 2;
#pragma unroll
        for (int i = 0; i < kBf16Pieces; ++i) *reinterpret_cast<__bf16*>(dst + i * l.piece) = piece[i];
    }
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }

// Rows into a payload's basis: (x * suh) H in pieces.  `residual`: x is turned by the normalised Hadamard on blocks of 512
// first, as coupled weights take it.
struct RotateArgs {
    const void* x;  // [rows / x_div][ld]
    int64_t ld;
    const _Float16* suh[2];
    int64_t suh_stride[2];
    const int* ids;  // null: one scale vector for all; else row r of the result is row r / x_div of x at scale ids[r]
    int x_div;
    int every;       // not 0: that many rows of x at every scale, row r of the result is row r % every at scale r / every
    char* out[2];
    int64_t rows;
    int kb, nmat;
    RowLayout layout;
    bool residual;
    const int* exponents;  // of kF16Pieces: row r is scaled by 2^exponents[r]
};

// Entry (i, j) of the 4 x 4 Sylvester matrix, which turns blocks of 128 into blocks of 512.
__device__ __forceinline__ float sign4(int i, int j) { return __builtin_popcount(i & j) & 1 ? -1.f : 1.f; }

inline int64_t rotate_waves(const RotateArgs& p) { return (p.rows + 15) / 16 * 16 * p.kb * p.nmat; }

// The `wave`-th 128 channels of a row and matrix; neighbouring waves have the same channels of neighbouring rows.
struct RotateAt {
    int64_t row;
    int kb, mat;
};
__device__ __forceinline__ RotateAt rotate_at(const RotateArgs& p, int64_t wave) {
    const int64_t sixteen = wave >> 4, rest = sixteen / p.kb;
    return RotateAt{16 * (p.nmat == 2 ? rest >> 1 : rest) + (wave & 15), static_cast<int>(sixteen - rest * p.kb),
                    p.nmat == 2 ? static_cast<int>(rest & 1) : 0};
}

template <typename T>
__device__ __forceinline__ f32x2 rotated(const RotateArgs& p, const RotateAt& at, int lane) {
    const int64_t id = p.every ? at.row / p.every : p.ids ? max(p.ids[at.row], 0) : 0;
    const int64_t from = p.every ? at.row - id * p.every : p.x_div == 1 ? at.row : at.row / p.x_div;
    const _Float16* suh =
        (at.mat ? p.suh[1] : p.suh[0]) + id * (at.mat ? p.suh_stride[1] : p.suh_stride[0]) + 128 * at.kb;
    const T* x = static_cast<const T*>(p.x) + from * p.ld + 128 * at.kb;
    typedef T t2 __attribute__((ext_vector_type(2)));
    const f16x2 sv = reinterpret_cast<const f16x2*>(suh)[lane];
    float a, b;
    if (p.residual) {
        const int block = at.kb & 3;
        a = b = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const t2 xv = reinterpret_cast<const t2*>(x + 128 * (i - block))[lane];
            a += sign4(i, block) * static_cast<float>(xv[0]);
            b += sign4(i, block) * static_cast<float>(xv[1]);
        }
        hadamard128(a, b, lane);
        a *= 0.5f * kHadamardScale;
        b *= 0.5f * kHadamardScale;
    } else {
        const t2 xv = reinterpret_cast<const t2*>(x)[lane];
        a = static_cast<float>(xv[0]);
        b = static_cast<float>(xv[1]);
    }
    a *= static_cast<float>(sv[0]);
    b *= static_cast<float>(sv[1]);
    hadamard128(a, b, lane);
    return f32x2{a * kHadamardScale, b * kHadamardScale};
}

template <typename T>
__device__ __forceinline__ void rotate_block(const RotateArgs& p, int64_t wave, int lane) {
    const RotateAt at = rotate_at(p, wave);
    if (at.row >= p.rows) return;
    const f32x2 v = rotated<T>(p, at, lane);
    store_pieces((at.mat ? p.out[1] : p.out[0]) + row_place(p.layout, at.row), p.layout, at.kb, lane, v[0], v[1]);
}

// The same by a workgroup of four waves for rows laid out by 16, two blocks of channels at once: 16 rows by 256 channels,
// which leave in one stretch (2048 x 5120 in two pieces: 17.0 us; four blocks 24.4, one 16.4, which makes more of the stores
// short where rows are few).
constexpr int kRotateBlocks = 2;
inline int64_t rotate_quads(const RotateArgs& p) { return (p.rows + 15) / 16 * p.nmat * ((p.kb + kRotateBlocks - 1) / kRotateBlocks); }
template <typename T, int kPieces>
__device__ __forceinline__ void rotate_quad(const RotateArgs& p, int64_t quad, u32x4 (&staged)[256 * kPieces * kRotateBlocks]) {
    const int lane = threadIdx.x & 63, w = uniform(static_cast<int>(threadIdx.x >> 6));
    const int quads = (p.kb + kRotateBlocks - 1) / kRotateBlocks;
    const int64_t rest = quad / quads, sixteen = p.nmat == 2 ? rest >> 1 : rest;
    const int kb0 = kRotateBlocks * static_cast<int>(quad - rest * quads), mat = p.nmat == 2 ? static_cast<int>(rest & 1) : 0;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        const int64_t row = 16 * sixteen + 4 * w + r, from = min(row, p.rows - 1);
        f32x2 v[kRotateBlocks];
#pragma unroll
        for (int j = 0; j < kRotateBlocks; ++j)  // past the last row and channel another's; not read by anyone who counts
            v[j] = rotated<T>(p, RotateAt{from, min(kb0 + j, p.kb - 1), mat}, lane);
        char* to = reinterpret_cast<char*>(staged) + (row & 15) * p.layout.row;
#pragma unroll
        for (int j = 0; j < kRotateBlocks; ++j) {
            if constexpr (kPieces == kF16Pieces) {
                const int e = p.exponents[from];
                store_pairs<_Float16, kF16Pieces>(to, p.layout, j, lane, ldexpf(v[j][0], e), ldexpf(v[j][1], e));
            } else {
                store_pieces(to, p.layout, j, lane, v[j][0], v[j][1]);
            }
        }
    }
    __syncthreads();
    u32x4* out = reinterpret_cast<u32x4*>((mat ? p.out[1] : p.out[0]) + sixteen * p.layout.sixteen + 4 * kb0 * p.layout.strip);
    const int end = 256 * kPieces * min(kRotateBlocks, p.kb - kb0);
    for (int i = threadIdx.x; i < end; i += 256) out[i] = staged[i];
}

// At most chunk_rows rows of one key (an expert): order[first .. first + count), the first of them row0.
// Chunks follow one another; the table's rest has count 0.
struct Chunk {
    int key, first, count, row0;
};
typedef const __attribute__((address_space(4))) Chunk* ConstChunk;  // constant for the kernels that read them

struct GroupArgs {
    const int* ids;
    int n, keys;
    int chunk_rows, max_chunks;
    Chunk* chunks;
    int* order;
    int* clean;  // ids with everything outside [0, keys) as -1
};

constexpr int kMaxKeys = 8191;  // their counters fit LDS

// Chunks that n rows can make at the most.
inline int64_t most_chunks(int64_t n, int64_t keys, int64_t chunk_rows) {
    const int64_t full = (n + chunk_rows - 1) / chunk_rows;
    return n < full + keys ? n : full + keys;
}

// Groups, and rotates beside it what does not need the groups (rows 0: nothing).
int launch_group(const GroupArgs& args, const RotateArgs& beside, int dtype, hipStream_t stream);

// Router of `tokens` rows, with what else of a layer can run beside it: the rotation of the same rows (rows 0: none), and
// the grouping of the chosen experts (null: none).
struct RouterArgs {
    const void* x;
    int64_t x_ld;
    const void* weight;
    int64_t weight_ld;
    int dtype;
    int tokens, hidden, experts, k;
    const float* bias;
    int scoring, normalize;
    float scale;
    float* weights;
    int* ids;
    float* logits;
};
const char* router_fault(const RouterArgs& args);
size_t router_logit_bytes(int64_t tokens, int64_t hidden, int64_t experts);
int64_t router_blocks(int64_t tokens, int64_t hidden, int64_t experts, const RotateArgs& beside);  // of 256 threads
int launch_router(const RouterArgs& args, const RotateArgs& beside, const GroupArgs* group, hipStream_t stream);

}  // namespace qsrt

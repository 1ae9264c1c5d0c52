// Products of a few rows with packed trellis matrices, and what stands around them in a mixture-of-experts layer.
#include <algorithm>
#include <cmath>

#include "packed.h"
#include "qsrt_amd.h"

using namespace qsrt;

namespace {

// ---------------------------------------------------------------------------
// The product: part sums of xr X, decoded on the way
// ---------------------------------------------------------------------------

struct ProductArgs {
    const int16_t* words[2];
    int64_t key_stride[2];        // words between the matrices of two keys
    const int64_t* records[2];    // per record: first word << 3 | bits
    int64_t record_stride[2];     // 0: one table for every key
    const char* x[2];             // rotated rows
    RowLayout layout;
    int x_div, x_every;           // row of order entry o with key e: e x_every + o / x_div
    const Chunk* chunks;          // null: runs of kRows rows of `rows`
    const int* order;
    int max_chunks, parts;
    const uint8_t* lut[2];
    int lut_bits[2];
    int luts;
    int pass;                     // this launch's parts follow `pass` times as many
    float* part;                  // [passes * parts][nmat][rows][cols]
    int nmat, axis, kb, nb;       // 128-channel blocks of both axes
    int rows;
};

typedef const __attribute__((address_space(1))) bf16x8* gbf8;
typedef const __attribute__((address_space(1))) f16x8* gf8;

// The label tables come to LDS while a wave looks up its first item and asks for its first words; one barrier a wave.
struct Tables {
    bool ready = false;
    __device__ __forceinline__ void wait() {
        if (ready) return;
        __builtin_amdgcn_s_waitcnt(0);  // the direct loads to LDS are not ordered by the barrier alone
        __syncthreads();
        ready = true;
    }
};

// `strips` strips of 32 payload rows by 128 columns at `tiles`, of rate K, times G groups of 16 rows.  Eight successive
// positions of a tile, 8 i8 .. 8 i8 + 7, are the rows 2g + {0, 1, 8, 9} of columns i8 / 4 and i8 / 4 + 8 (g = i8 % 4): one
// window of 16 + 7 K bits of the tile's stream, two dwords.  Lane 16 g + m reads it in tile column 2 t + m / 8 of each pair
// t, for i8 = 4 (m % 8) + g; MFMA 2 t + u has its columns m % 8 + 8 u as rows.  K is a value and not a template argument:
// the same instructions with other shifts, where a body for each rate made the compiler keep a second set of sums.
// kHalf false: 16 G rows, hi, mid and lo pieces multiplied one after the other.  kHalf (G 1): up to 8 rows, the hi piece of row
// n in lanes n and the mid piece in lanes n + 8 of one product, the lo piece in lanes n of a second; `x` is then the lane's own
// piece, x_piece the way from it to the lo piece.
// kPairs (K 2 alone): `lut` holds a row of 8 bytes for each 14 bits that two successive states share, the label of the first
// state for each value x of its other bits at byte 2 x, of the second for each y at byte 2 y + 1.  A lookup costs the banks
// the same at 8 bytes as at one (7.3 clocks for 64 random lanes), so this halves what bounds the product.
template <int G, bool kHalf, bool kPairs>
__device__ __forceinline__ void multiply_strips(const char* tiles, int tile_row_bytes, int strips, int K,
                                                const char* (&x)[G], int x_strip, int x_piece, const uint8_t* lut,
                                                int lane, Tables& tables, f32x4 (&acc)[G][8]) {
    const int m = lane & 15, g = lane >> 4;
    int b0 = (8 * (4 * (m & 7) + g) + 1) * K - 16;
    if (b0 < 0) b0 += 256 * K;
    const int d0 = b0 >> 5, d1 = d0 + 1 == 8 * K ? 0 : d0 + 1;
    const uint32_t sh = b0 & 31, rsh = 32u - sh;  // sh is never 0 at K = 2, 3, 4
    const uint32_t o0 = 4 * d0 + (m >> 3) * 32 * K, o1 = 4 * d1 + (m >> 3) * 32 * K;
    const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(tiles), 0, (2 * strips - 1) * tile_row_bytes + 256 * K, 0x00027000);
    constexpr int kProducts = kHalf ? 2 : kBf16Pieces;
    uint32_t lo[8], hi[8];
    auto fetch = [&](int s, int t) {  // the pair's windows of both tile rows
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int at = (2 * s + h) * tile_row_bytes + t * 64 * K;
            lo[2 * t + h] = __builtin_amdgcn_raw_buffer_load_b32(src, o0, at, 0);
            if constexpr (!kPairs) hi[2 * t + h] = __builtin_amdgcn_raw_buffer_load_b32(src, o1, at, 0);
        }
    };
#pragma unroll
    for (int t = 0; t < 4; ++t) fetch(0, t);
    tables.wait();
    int s = 0;
    do {
        bf16x8 b[G][kProducts];
#pragma unroll
        for (int q = 0; q < G; ++q) {
#pragma unroll
            for (int p = 0; p < kProducts; ++p) b[q][p] = *(gbf8)(x[q] + p * x_piece);
            x[q] += x_strip;
        }
        if constexpr (kHalf) {
            if (m >= 8) b[0][1] = bf16x8{};
        }
        uint32_t next[16], window[2];
        uint32_t rest = 0x0C000C01u;  // the selector's fixed part, in a vector register: one instruction takes one scalar
        asm volatile("" : "+v"(rest));
        u32x2 next_row[8];
        auto gather = [&](int t) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // At K2 the windows of odd i8 lie in one dword, which is the second one of i8 - 1, 16 lanes below.
                if constexpr (kPairs)
                    hi[2 * t + h] = __builtin_amdgcn_permlane16_swap(lo[2 * t + h], lo[2 * t + h], false, false)[1];
                const uint32_t w0 = __builtin_amdgcn_alignbit(lo[2 * t + h], hi[2 * t + h], rsh);
                if constexpr (kPairs) {
                    window[h] = w0;  // 30 bits: x, 14 shared bits, y of each pair, two bits further on for the next but one
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        next_row[4 * h + j] = *reinterpret_cast<const u32x2*>(lut + ((w0 >> (13 - 4 * j)) & 0x1FFF8u));
                } else {
                    // bits 0..31 of the window, and 4 K .. 4 K + 31: four labels in each
                    const uint32_t w1 = __builtin_amdgcn_alignbit(w0, hi[2 * t + h] << sh, 32 - 4 * K);
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        next[8 * h + j] = lut[__builtin_amdgcn_ubfe(j < 4 ? w0 : w1, 16 - (j & 3) * K, 16)];
                }
            }
            fetch(min(s + 1, strips - 1), t);  // the last strip asks for itself again: no branch, so that waits stay exact
        };
        gather(0);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            uint32_t label[16], seen[2];
            u32x2 row[8];
            if constexpr (kPairs) {
#pragma unroll
                for (int j = 0; j < 8; ++j) row[j] = next_row[j];
                seen[0] = window[0];
                seen[1] = window[1];
            } else {
#pragma unroll
                for (int j = 0; j < 16; ++j) label[j] = next[j];
            }
            if (t < 3) gather(t + 1);
            bf16x8 av[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                u32x4 a;
                if constexpr (kPairs) {
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        uint32_t two[2];  // a pair's second label in byte 0, its first in byte 2
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            const int j = 2 * u + q;
                            two[q] = __builtin_amdgcn_perm(row[4 * h + j][1], row[4 * h + j][0],
                                                           ((seen[h] >> (13 - 4 * j)) & 0x00060006u) | rest);
                        }
                        const uint32_t four = __builtin_amdgcn_perm(two[1], two[0], 0x04060002u);
                        a[2 * h] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, false));
                        a[2 * h + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(four, 1.0f, true));
                    }
                } else {
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        const int j = 8 * (q >> 1) + 4 * u + 2 * (q & 1);
                        a[q] = __builtin_bit_cast(
                            uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                                          __builtin_amdgcn_perm(label[j + 1], label[j], 0x0C0C0400u), 1.0f, false));
                    }
                }
                av[u] = __builtin_bit_cast(bf16x8, a);
            }
#pragma unroll
            for (int p = 0; p < kProducts; ++p)  // hi pieces of all sums, then the next: a sum's products do not follow each other
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int q = 0; q < G; ++q)
                        acc[q][2 * t + u] =
                            __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[u], b[q][p], acc[q][2 * t + u], 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);  // two pairs' labels in registers at most
        }
    } while (++s < strips);
}

// Rows of label pairs from the K2 table: four rows a thread and turn, their first states' labels from the table's quarters.
template <int kThreads>
__device__ __forceinline__ void build_pairs(const uint8_t* table, uint8_t* rows) {
#pragma unroll
    for (int i = 0; i < (4096 + kThreads - 1) / kThreads; ++i) {
        const int c = 4 * (threadIdx.x + i * kThreads);
        if (c >= 16384) break;
        uint32_t quarter[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) quarter[x] = *reinterpret_cast<const uint32_t*>(table + 16384 * x + c);
        const u32x4 second = *reinterpret_cast<const u32x4*>(table + 4 * c);
#pragma unroll
        for (int r = 0; r < 4; r += 2) {
            u32x4 two;
#pragma unroll
            for (int d = 0; d < 4; ++d) {  // row r + d / 2: {first x, second x, first x + 1, second x + 1}, x = 2 (d % 2)
                const int at = r + (d >> 1), x = 2 * (d & 1);
                const uint32_t first = __builtin_amdgcn_perm(quarter[x + 1], quarter[x], 0x0C040C00u + 0x00010001u * at);
                const uint32_t other = __builtin_amdgcn_perm(0u, second[at], x ? 0x030C020Cu : 0x010C000Cu);
                two[d] = first | other;
            }
            *reinterpret_cast<u32x4*>(rows + 8 * (c + r)) = two;
        }
    }
}

// kTables: label tables in LDS; 0: the pairs of the K2 table.
template <int G, bool kHalf, int kWaves, int kTables>
__global__ __launch_bounds__(64 * kWaves) void product_kernel(const ProductArgs p) {
    static_assert(!kHalf || G == 1, "half a group of rows is the least there is");
    __shared__ __attribute__((aligned(16))) uint8_t lut_s[kTables ? 65536 * kTables : 131072];
    const int lane = threadIdx.x & 63;
    const int w = uniform(static_cast<int>(threadIdx.x >> 6));
    if constexpr (kTables == 0)
        build_pairs<64 * kWaves>(p.lut[0], lut_s);
    else
        for (int i = w; i < kTables * 64; i += kWaves)
            __builtin_amdgcn_global_load_lds(
                (const __attribute__((address_space(1))) void*)((i < 64 ? p.lut[0] : p.lut[1]) + 1024 * (i & 63) + 16 * lane),
                (__attribute__((address_space(3))) void*)(lut_s + 1024 * i), 16, 0, 0);
    Tables tables;

    constexpr int kRows = kHalf ? 8 : 16 * G;
    const int g = lane >> 4, n = kHalf ? lane & 7 : lane & 15, piece = kHalf ? (lane >> 3) & 1 : 0;
    const int x_piece = kHalf ? (2 - piece) * p.layout.piece : p.layout.piece;
    const int parts = p.parts;
    const uint32_t items = static_cast<uint32_t>(p.max_chunks) * p.nmat * p.nb * parts;  // below 2^31: see cut_parts
    const int64_t cols = 128 * static_cast<int64_t>(p.nb);
    const int strips = 4 * p.kb;

    // Rounds of an item a wave.
    const uint32_t grid = gridDim.x, per_round = grid * kWaves;
    uint32_t turn = blockIdx.x + 37 * w;
    for (uint32_t base = 0; base < items; base += per_round, turn += 101) {
        uint32_t item;
        int part, cb, mat, ci;
        if constexpr (G == 1) {
            // One group of rows: the items of a round are dealt out to the workgroups one by one.  The deal is turned from
            // wave to wave and round to round: column blocks come in a period that divides the grid's, and a workgroup that
            // only ever met the blocks of the highest rate would finish last (7168 x 2048 at K3 and K4 records: 1.84 ms
            // where 1.54 will do).
            item = base + w * grid + turn % grid;
            if (item >= items) break;
            uint32_t rest = item / parts;
            part = static_cast<int>(item - rest * parts);
            cb = static_cast<int>(rest % p.nb);
            rest /= p.nb;
            mat = p.nmat == 2 ? static_cast<int>(rest & 1) : 0;
            ci = static_cast<int>(p.nmat == 2 ? rest >> 1 : rest);
        } else {
            // Many rows: a strip of them is more than the payload's, so neighbouring waves, and the workgroups of one
            // chiplet (blockIdx.x % 8), take the column blocks of the same rows and find these in their caches.
            const uint32_t eighth = grid >> 3;
            const uint32_t b = (grid & 7) ? blockIdx.x : (blockIdx.x & 7) * eighth + (blockIdx.x >> 3);
            item = base + (items - base >= per_round ? b * kWaves + w : w * grid + b);
            if (item >= items) break;
            uint32_t rest = item / p.nb;
            cb = static_cast<int>(item - rest * p.nb);
            mat = p.nmat == 2 ? static_cast<int>(rest & 1) : 0;
            if (p.nmat == 2) rest >>= 1;
            ci = static_cast<int>(rest / parts);
            part = static_cast<int>(rest - ci * parts);
        }
        int key = 0, first = ci * kRows, count = min(kRows, p.rows - first), row0 = first;
        if (p.chunks) {
            const ConstChunk c = (ConstChunk)p.chunks + ci;
            key = c->key;
            first = c->first;
            count = c->count;
            row0 = c->row0;
            if (count == 0) break;  // the last chunk is behind
        }
        int s = strips * part / parts;
        const int end = strips * (part + 1) / parts;
        int row[G];
        const char* x[G];
#pragma unroll
        for (int q = 0; q < G; ++q) {  // lanes past the last row repeat it; their sums are not stored
            const int at = first + min(16 * q + n, count - 1);
            row[q] = !p.chunks ? at : count == 1 ? row0 : p.order[at];
            const int64_t from = static_cast<int64_t>(key) * p.x_every + (p.x_div == 1 ? row[q] : row[q] / p.x_div);
            x[q] = (mat ? p.x[1] : p.x[0]) + row_place(p.layout, from) + g * p.layout.group + s * p.layout.strip +
                   piece * p.layout.piece;
        }
        f32x4 acc[G][8];
#pragma unroll
        for (int q = 0; q < G; ++q)
#pragma unroll
            for (int t = 0; t < 8; ++t) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};

        const char* words =
            reinterpret_cast<const char*>((mat ? p.words[1] : p.words[0]) + key * (mat ? p.key_stride[1] : p.key_stride[0]));
        typedef const __attribute__((address_space(4))) int64_t* ConstRecord;
        const ConstRecord records = (ConstRecord)(mat ? p.records[1] : p.records[0]) +
                                    key * (mat ? p.record_stride[1] : p.record_stride[0]);
        while (s < end) {  // runs of one rate
            const int r = p.axis ? cb : s >> 2;
            const int64_t rec = records[r];
            const int bits = static_cast<int>(rec & 7);
            int stop = end;
            if (!p.axis) {  // records of one rate that follow one another are one strip of tiles
                int r1 = r + 1;
                while (4 * r1 < end && static_cast<int>(records[r1] & 7) == bits) ++r1;
                stop = min(end, 4 * r1);
            }
            const int tile = 32 * bits;
            const int tile_row = p.axis ? 8 * tile : 8 * p.nb * tile;
            const char* tiles = words + 2 * (rec >> 3) +
                                (p.axis ? static_cast<int64_t>(2 * s) * tile_row
                                        : static_cast<int64_t>(2 * (s - 4 * r)) * tile_row + 8 * cb * tile);
            if (bits == p.lut_bits[0] || (kTables > 1 && bits == p.lut_bits[1])) {
                const uint8_t* lut = kTables > 1 && bits == p.lut_bits[1] ? lut_s + 65536 : lut_s;
                multiply_strips<G, kHalf, kTables == 0>(tiles, tile_row, stop - s, bits, x, p.layout.strip, x_piece, lut, lane,
                                                        tables, acc);
            } else {  // another pass has this rate
#pragma unroll
                for (int q = 0; q < G; ++q) x[q] += (stop - s) * p.layout.strip;
            }
            s = stop;
        }
        if constexpr (kHalf) {
#pragma unroll
            for (int t = 0; t < 8; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[0][t][i] += dpp<0x128>(acc[0][t][i]);  // row rotated by 8: the other piece's
        }
        // MFMA rows 4 g .. 4 g + 3: columns 16 (2 t + g / 2) + 8 u + 4 (g % 2) + 0..3 of row n.  (Exchanging halves of the wave
        // so that a store covers 64 bytes of a row and not 32 made no difference.)
        float* out = p.part + (static_cast<int64_t>(p.pass * parts + part) * p.nmat + mat) * p.rows * cols + 128 * cb +
                     16 * (g >> 1) + 4 * (g & 1);
#pragma unroll
        for (int q = 0; q < G; ++q) {
            if (16 * q + n >= count || piece) continue;
#pragma unroll
            for (int t = 0; t < 8; ++t)
                *reinterpret_cast<f32x4*>(out + row[q] * cols + 32 * (t >> 1) + 8 * (t & 1)) = acc[q][t];
        }
    }
    tables.wait();
}

// ---------------------------------------------------------------------------
// The product of many rows: a workgroup decodes a strip once for 128 G of them
// ---------------------------------------------------------------------------

constexpr int kRowWaves = 8;

// A barrier that orders LDS alone: loads from memory stay on their way across it.
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// Eight waves of 16 G rows each over the same columns.  Wave w decodes one window a lane of every strip (tile column pair
// w / 2, tile row w % 2) into the MFMA operands of the strip in LDS, two strips ahead, and multiplies all of a strip's by its
// own rows; one barrier a strip, across which the first operands of the next are on their way.  The table reads, which bound
// the product of a few rows, fall to an eighth a row and are spread over the strip's products (all at its start, with two
// buffers of operands: 1.39 us a strip of 4 groups and 0.86 of 2, so 1.19 and 0.72).  The matrix cores take 0.95 and 0.48 of
// that at two pieces a row and the 2.2 GHz that they leave; before and after it a workgroup waits 8 us for tables and first
// rows and 6 to 12 for its sums' stores (2048 x 5120 x 1536: 70 us, 925 TFLOP/s of pieces).
template <int G>
__device__ __forceinline__ void multiply_rows(const char* tiles, int tile_row_bytes, int strips, int K, const char* (&x)[G],
                                              const uint8_t* lut, u32x2 (&frags)[3][8][128], int lane, int w, bool& ready,
                                              f32x4 (&acc)[G][8]) {
    constexpr int kStrip = 16 * strip_bytes(kF16Pieces);
    const int m = lane & 15, g = lane >> 4, t = w >> 1, h = w & 1;
    int b0 = (8 * (4 * (m & 7) + g) + 1) * K - 16;  // as in multiply_strips
    if (b0 < 0) b0 += 256 * K;
    const int d0 = b0 >> 5, d1 = d0 + 1 == 8 * K ? 0 : d0 + 1;
    const uint32_t sh = b0 & 31, rsh = 32u - sh;
    const uint32_t o0 = 4 * d0 + (m >> 3) * 32 * K + t * 64 * K, o1 = 4 * d1 + (m >> 3) * 32 * K + t * 64 * K;
    const __amdgpu_buffer_rsrc_t src = __builtin_amdgcn_make_buffer_rsrc(
        const_cast<char*>(tiles), 0, (2 * strips - 1) * tile_row_bytes + 256 * K, 0x00027000);
    uint32_t lo[2], hi[2];
    f16x8 b[G][kF16Pieces], next[G][kF16Pieces];
    auto fetch_words = [&](int s, int slot) {
        const int at = (2 * min(s, strips - 1) + h) * tile_row_bytes;
        lo[slot] = __builtin_amdgcn_raw_buffer_load_b32(src, o0, at, 0);
        hi[slot] = __builtin_amdgcn_raw_buffer_load_b32(src, o1, at, 0);
    };
    auto fetch_rows = [&](int s) {
#pragma unroll
        for (int q = 0; q < G; ++q)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                next[q][p] = *(gf8)(x[q] + static_cast<int64_t>(min(s, strips - 1)) * kStrip + 1024 * p);
    };
    uint32_t label[8], window[2];
    auto open_window = [&](int slot) {
        window[0] = __builtin_amdgcn_alignbit(lo[slot], hi[slot], rsh);
        window[1] = __builtin_amdgcn_alignbit(window[0], hi[slot] << sh, 32 - 4 * K);
    };
    auto look_up = [&](int j) { label[j] = lut[__builtin_amdgcn_ubfe(window[j >> 2], 16 - (j & 3) * K, 16)]; };
    auto write_operands = [&](int buffer) {
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            u32x2 half;
#pragma unroll
            for (int q = 0; q < 2; ++q)
                half[q] = __builtin_bit_cast(
                    uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(
                                  __builtin_amdgcn_perm(label[4 * u + 2 * q + 1], label[4 * u + 2 * q], 0x0C0C0400u), 1.0f, false));
            frags[buffer][2 * t + u][2 * lane + h] = half;
        }
    };
    fetch_words(0, 0);
    fetch_words(1, 1);
    fetch_rows(0);
    if (!ready) {
        __builtin_amdgcn_s_waitcnt(0);  // the direct loads to LDS are not ordered by the barrier alone
        ready = true;
    }
    __syncthreads();  // the tables are there, and no wave reads the operands of an earlier run
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        open_window(e);
#pragma unroll
        for (int j = 0; j < 8; ++j) look_up(j);
        write_operands(e);
        fetch_words(2 + e, e);
    }
    lds_barrier();
    int now = 0, then = 1, after = 2;  // buffers of this strip and the next two
    auto operand = [&](int buffer, int c) { return *reinterpret_cast<const u32x4*>(&frags[buffer][c][2 * lane]); };
    u32x4 ahead[2] = {operand(0, 0), operand(0, 1)};
    for (int s = 0; s < strips; s += 2) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {  // words of strips s + e + 2 in slot e
            if (s + e < strips) {
#pragma unroll
                for (int q = 0; q < G; ++q) {
                    b[q][0] = next[q][0];
                    b[q][1] = next[q][1];
                }
                fetch_rows(s + e + 1);
                open_window(e);
                fetch_words(s + e + 4, e);
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    // the labels of the strip after the next come in between, so that no operand waits behind all of them
                    if (c < 2) look_up(2 * c);
                    if (c < 2) look_up(2 * c + 1);
                    if (c >= 2 && c < 6) look_up(c + 2);
                    const f16x8 a = __builtin_bit_cast(f16x8, ahead[c & 1]);
                    ahead[c & 1] = c < 6 ? operand(now, c + 2) : operand(then, c - 6);
#pragma unroll
                    for (int p = 0; p < 2; ++p)
#pragma unroll
                        for (int q = 0; q < G; ++q)
                            acc[q][c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b[q][p], acc[q][c], 0, 0, 0);
                    __builtin_amdgcn_sched_barrier(0);
                }
                write_operands(after);  // past the last strip: the last again, which nobody uses
                lds_barrier();
                const int free = now;
                now = then;
                then = after;
                after = free;
            }
        }
    }
#pragma unroll
    for (int q = 0; q < G; ++q) x[q] += static_cast<int64_t>(strips) * kStrip;
}

template <int G, int kTables>
__global__ __launch_bounds__(64 * kRowWaves) void product_rows_kernel(const ProductArgs p) {
    __shared__ __attribute__((aligned(16))) uint8_t lut_s[65536 * kTables];
    __shared__ __attribute__((aligned(16))) u32x2 frags[3][8][128];
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int w = uniform(static_cast<int>(threadIdx.x >> 6));
    for (int i = w; i < kTables * 64; i += kRowWaves)
        __builtin_amdgcn_global_load_lds(
            (const __attribute__((address_space(1))) void*)((i < 64 ? p.lut[0] : p.lut[1]) + 1024 * (i & 63) + 16 * lane),
            (__attribute__((address_space(3))) void*)(lut_s + 1024 * i), 16, 0, 0);
    bool ready = false;
    const uint32_t items = static_cast<uint32_t>(p.max_chunks) * p.nb * p.parts, grid = gridDim.x;
    const int64_t cols = 128 * static_cast<int64_t>(p.nb);
    const int strips = 4 * p.kb, sixteens = (p.rows + 15) / 16;
    // the workgroups of one chiplet (blockIdx.x % 8) take the column blocks of the same rows and find these in their cache
    const uint32_t turn = (grid & 7) ? blockIdx.x : (blockIdx.x & 7) * (grid >> 3) + (blockIdx.x >> 3);
    for (uint32_t item = turn; item < items; item += grid) {
        uint32_t rest = item / p.nb;
        const int cb = static_cast<int>(item - rest * p.nb);
        const int ci = static_cast<int>(rest / p.parts), part = static_cast<int>(rest - ci * p.parts);
        const int first = (ci * kRowWaves + w) * G;  // in groups of 16 rows
        int s = strips * part / p.parts;
        const int end = strips * (part + 1) / p.parts;
        const char* x[G];
        f32x4 acc[G][8];
#pragma unroll
        for (int q = 0; q < G; ++q) {  // groups past the last repeat it; their sums are not stored
            x[q] = p.x[0] + min(first + q, sixteens - 1) * p.layout.sixteen + s * p.layout.strip + 16 * lane;
#pragma unroll
            for (int t = 0; t < 8; ++t) acc[q][t] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        const char* words = reinterpret_cast<const char*>(p.words[0]);
        typedef const __attribute__((address_space(4))) int64_t* ConstRecord;
        const ConstRecord records = (ConstRecord)p.records[0];
        while (s < end) {  // runs of one rate, as in product_kernel
            const int r = p.axis ? cb : s >> 2;
            const int64_t rec = records[r];
            const int bits = static_cast<int>(rec & 7);
            int stop = end;
            if (!p.axis) {
                int r1 = r + 1;
                while (4 * r1 < end && static_cast<int>(records[r1] & 7) == bits) ++r1;
                stop = min(end, 4 * r1);
            }
            const int tile = 32 * bits, tile_row = p.axis ? 8 * tile : 8 * p.nb * tile;
            const char* tiles = words + 2 * (rec >> 3) +
                                (p.axis ? static_cast<int64_t>(2 * s) * tile_row
                                        : static_cast<int64_t>(2 * (s - 4 * r)) * tile_row + 8 * cb * tile);
            if (bits == p.lut_bits[0] || (kTables > 1 && bits == p.lut_bits[1])) {
                const uint8_t* lut = kTables > 1 && bits == p.lut_bits[1] ? lut_s + 65536 : lut_s;
                multiply_rows<G>(tiles, tile_row, stop - s, bits, x, lut, frags, lane, w, ready, acc);
            } else {  // another pass has this rate
#pragma unroll
                for (int q = 0; q < G; ++q) x[q] += (stop - s) * p.layout.strip;
            }
            s = stop;
        }
        float* out = p.part + static_cast<int64_t>(p.pass * p.parts + part) * p.rows * cols + 128 * cb + 16 * (g >> 1) +
                     4 * (g & 1);
#pragma unroll
        for (int q = 0; q < G; ++q) {
            const int64_t row = 16 * static_cast<int64_t>(first + q) + n;
            if (row >= p.rows) continue;
#pragma unroll
            for (int t = 0; t < 8; ++t)
                *reinterpret_cast<f32x4*>(out + row * cols + 32 * (t >> 1) + 8 * (t & 1)) = acc[q][t];
        }
    }
    if (!ready) __builtin_amdgcn_s_waitcnt(0);  // no wave ends with loads to LDS on their way
}

// ---------------------------------------------------------------------------
// Rows into the payload's basis
// ---------------------------------------------------------------------------

template <typename T>
__global__ __launch_bounds__(256) void rotate_rows_kernel(const RotateArgs p) {
    rotate_block<T>(p, static_cast<int64_t>(blockIdx.x) * 4 + uniform(static_cast<int>(threadIdx.x >> 6)), threadIdx.x & 63);
}

// ---------------------------------------------------------------------------
// Between the two products of an expert
// ---------------------------------------------------------------------------

struct MiddleArgs {
    const float* part;  // [parts][2][pairs][inter]
    int parts;
    const int* ids;
    const _Float16* svh[2];
    int64_t svh_stride[2];
    const _Float16* suh;  // of the second product
    int64_t suh_stride;
    char* out;
    RowLayout layout;
    int pairs, ib, act;
    const float *pre_signs, *post_signs;  // [2 inter], [inter] of coupled weights; else null
};

__device__ __forceinline__ float activate(float g, float u, int act) {
    const float s = 1.0f / (1.0f + expf(-g));
    return act == 0 ? g * s * u : 4.0f * tanhf(0.25f * g) * s * (25.0f * tanhf(0.04f * u));
}

// Sum over parts first, first + step, ... of the two channels 2 lane, 2 lane + 1; the loads of eight parts go out together.
__device__ __forceinline__ f32x2 sum_parts(const float* src, int64_t stride, int first, int step, int parts) {
    f32x2 sum = {0.f, 0.f};
    int s = first;
    for (; s + 7 * step < parts; s += 8 * step) {
        f32x2 v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = *reinterpret_cast<const f32x2*>(src + (s + j * step) * stride);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += v[j];
    }
#pragma unroll 4
    for (; s < parts; s += step) sum += *reinterpret_cast<const f32x2*>(src + s * stride);
    return sum;
}

// Both sums of 128 channels over all parts; the loads of eight parts go out together.  `step`: floats from part to part.
__device__ __forceinline__ void sum_two(const float* s0, const float* s1, int64_t step, int parts, f32x2& a, f32x2& b) {
    a = b = f32x2{0.f, 0.f};
    int s = 0;
    for (; s + 8 <= parts; s += 8) {
        f32x2 v[8], t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            v[j] = *reinterpret_cast<const f32x2*>(s0 + (s + j) * step);
            t[j] = *reinterpret_cast<const f32x2*>(s1 + (s + j) * step);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            a += v[j];
            b += t[j];
        }
    }
#pragma unroll 4
    for (; s < parts; ++s) {
        a += *reinterpret_cast<const f32x2*>(s0 + s * step);
        b += *reinterpret_cast<const f32x2*>(s1 + s * step);
    }
}

// One wave for 128 middle channels of one (token, expert) pair.
__global__ __launch_bounds__(256) void middle_kernel(const MiddleArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + uniform(static_cast<int>(threadIdx.x >> 6));
    const int ib = static_cast<int>(wave % p.ib);
    const int64_t pair = wave / p.ib;
    if (pair >= p.pairs) return;
    const int id = uniform(p.ids[pair]);
    if (id < 0) return;
    const int64_t inter = 128 * static_cast<int64_t>(p.ib), rows = static_cast<int64_t>(p.pairs) * inter;
    const f16x2 sg = reinterpret_cast<const f16x2*>(p.svh[0] + id * p.svh_stride[0] + 128 * ib)[lane];
    const f16x2 su = reinterpret_cast<const f16x2*>(p.svh[1] + id * p.svh_stride[1] + 128 * ib)[lane];
    const f16x2 sd = reinterpret_cast<const f16x2*>(p.suh + id * p.suh_stride + 128 * ib)[lane];
    const float* src = p.part + pair * inter + 128 * ib + 2 * lane;
    f32x2 gs, us;
    sum_two(src, src + rows, 2 * rows, p.parts, gs, us);
    float g0 = gs[0], g1 = gs[1], u0 = us[0], u1 = us[1];
    hadamard128(g0, g1, lane);
    hadamard128(u0, u1, lane);
    float a = activate(g0 * kHadamardScale * static_cast<float>(sg[0]), u0 * kHadamardScale * static_cast<float>(su[0]), p.act) *
              static_cast<float>(sd[0]);
    float b = activate(g1 * kHadamardScale * static_cast<float>(sg[1]), u1 * kHadamardScale * static_cast<float>(su[1]), p.act) *
              static_cast<float>(sd[1]);
    hadamard128(a, b, lane);
    store_pieces(p.out + row_place(p.layout, pair), p.layout, ib, lane, a * kHadamardScale, b * kHadamardScale);
}

// The same for coupled weights.  Their gate and up channels are interleaved, the interleaved axis turned by the signed
// Hadamard on blocks of 128 (which turns back to signs * H z), and its first half is the first product's, its second half the
// second's.  So block z of the turned axis holds channels 64 z .. 64 z + 63 of both, and after turning it back lane l has gate
// and up of channel 64 z + l: no exchange between lanes.  A wave takes two such blocks, whose channels lie as l and 64 + l of
// its 128: the butterflies are the same in that order.  The second product's turn is H (signs * middle).
__global__ __launch_bounds__(256) void middle_coupled_kernel(const MiddleArgs p) {
    const int lane = threadIdx.x & 63;
    const int64_t wave = static_cast<int64_t>(blockIdx.x) * 4 + uniform(static_cast<int>(threadIdx.x >> 6));
    const int ib = static_cast<int>(wave % p.ib);
    const int64_t pair = wave / p.ib;
    if (pair >= p.pairs) return;
    const int id = uniform(p.ids[pair]);
    if (id < 0) return;
    const int64_t inter = 128 * static_cast<int64_t>(p.ib), rows = static_cast<int64_t>(p.pairs) * inter;
    const float* src[2];
    f32x2 sums[2];
    float middle[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int z = 2 * ib + h, mat = z >= p.ib;
        src[h] = p.part + mat * rows + pair * inter + 128 * (z - mat * p.ib) + 2 * lane;
    }
    sum_two(src[0], src[1], 2 * rows, p.parts, sums[0], sums[1]);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int z = 2 * ib + h, mat = z >= p.ib;
        const _Float16* svh = (mat ? p.svh[1] + id * p.svh_stride[1] : p.svh[0] + id * p.svh_stride[0]) + 128 * (z - mat * p.ib);
        const f16x2 sv = reinterpret_cast<const f16x2*>(svh)[lane];
        const f32x2 sign = reinterpret_cast<const f32x2*>(p.pre_signs + 128 * z)[lane];
        float g = sums[h][0], u = sums[h][1];
        hadamard128(g, u, lane);
        g *= kHadamardScale * static_cast<float>(sv[0]);
        u *= kHadamardScale * static_cast<float>(sv[1]);
        hadamard128(g, u, lane);
        middle[h] = activate(g * kHadamardScale * sign[0], u * kHadamardScale * sign[1], p.act) *
                    p.post_signs[128 * ib + 64 * h + lane];
    }
    float a = middle[0], b = middle[1];
    hadamard128(a, b, lane);
    const _Float16* suh = p.suh + id * p.suh_stride + 128 * ib + lane;
    a *= kHadamardScale * static_cast<float>(suh[0]);
    b *= kHadamardScale * static_cast<float>(suh[64]);
    hadamard128(a, b, lane);
    store_halves(p.out + row_place(p.layout, pair), p.layout, ib, lane, a * kHadamardScale, b * kHadamardScale);
}

// ---------------------------------------------------------------------------
// The layer's sum over a token's experts
// ---------------------------------------------------------------------------

struct CombineArgs {
    const float* part;  // [parts][pairs][hidden]
    int parts;
    const int* ids;
    const float* weights;
    const _Float16* svh;
    int64_t svh_stride;
    void* out;
    int64_t ld;
    int tokens, k, hb;
};

constexpr int kCombineWaves = 8, kCoupledShares = 4;

// (v H) * svh of 128 channels.
__device__ __forceinline__ f32x2 scaled_turn(f32x2 v, const _Float16* svh, int lane) {
    float a = v[0], b = v[1];
    hadamard128(a, b, lane);
    const f16x2 sv = reinterpret_cast<const f16x2*>(svh)[lane];
    return f32x2{a * kHadamardScale * static_cast<float>(sv[0]), b * kHadamardScale * static_cast<float>(sv[1])};
}

// One workgroup for 128 channels of one token, its waves share the token's experts.  With one svh for all experts the
// weighted sum is rotated once, with one for each every expert's.
template <typename T>
__global__ __launch_bounds__(64 * kCombineWaves) void combine_kernel(const CombineArgs p) {
    __shared__ f32x2 sums[kCombineWaves][64];
    const int lane = threadIdx.x & 63, w = uniform(static_cast<int>(threadIdx.x >> 6)), waves = blockDim.x >> 6;
    const int hb = static_cast<int>(blockIdx.x % p.hb);
    const int64_t token = blockIdx.x / p.hb;
    const int64_t hidden = 128 * static_cast<int64_t>(p.hb), stride = static_cast<int64_t>(p.tokens) * p.k * hidden;
    const bool shared = p.svh_stride == 0;
    f32x2 y = {0.f, 0.f};
    for (int j = w; j < p.k; j += waves) {
        const int64_t pair = token * p.k + j;
        const int id = uniform(p.ids[pair]);
        if (id < 0) continue;
        f32x2 v = sum_parts(p.part + pair * hidden + 128 * hb + 2 * lane, stride, 0, 1, p.parts);
        if (!shared) v = scaled_turn(v, p.svh + id * p.svh_stride + 128 * hb, lane);
        y += v * p.weights[pair];
    }
    sums[w][lane] = y;
    __syncthreads();
    if (w) return;
    for (int j = 1; j < waves; ++j) y += sums[j][lane];
    if (shared) y = scaled_turn(y, p.svh + 128 * hb, lane);
    typedef T t2 __attribute__((ext_vector_type(2)));
    reinterpret_cast<t2*>(static_cast<T*>(p.out) + token * p.ld + 128 * hb)[lane] =
        t2{static_cast<T>(y[0]), static_cast<T>(y[1])};
}

// The same for coupled weights, whose results are turned by the Hadamard on blocks of 512: a workgroup takes four blocks of
// 128 channels, wave w the w % 4-th of them for a share of the token's experts, and then one block of the result.
template <typename T>
__global__ __launch_bounds__(256 * kCoupledShares) void combine_coupled_kernel(const CombineArgs p) {
    __shared__ f32x2 sums[4 * kCoupledShares][64], turned[4][64];
    const int lane = threadIdx.x & 63, w = uniform(static_cast<int>(threadIdx.x >> 6)), shares = blockDim.x >> 8;
    const int block = w & 3, hb = 4 * static_cast<int>(blockIdx.x % (p.hb >> 2)) + block;
    const int64_t token = blockIdx.x / (p.hb >> 2);
    const int64_t hidden = 128 * static_cast<int64_t>(p.hb), stride = static_cast<int64_t>(p.tokens) * p.k * hidden;
    const bool shared = p.svh_stride == 0;
    f32x2 y = {0.f, 0.f};
    for (int j = w >> 2; j < p.k; j += shares) {
        const int64_t pair = token * p.k + j;
        const int id = uniform(p.ids[pair]);
        if (id < 0) continue;
        f32x2 v = sum_parts(p.part + pair * hidden + 128 * hb + 2 * lane, stride, 0, 1, p.parts);
        if (!shared) v = scaled_turn(v, p.svh + id * p.svh_stride + 128 * hb, lane);
        y += v * p.weights[pair];
    }
    sums[w][lane] = y;
    __syncthreads();
    if (w < 4) {
        for (int j = 1; j < shares; ++j) y += sums[4 * j + w][lane];
        turned[w][lane] = shared ? scaled_turn(y, p.svh + 128 * hb, lane) : y;
    }
    __syncthreads();
    if (w >= 4) return;
    y = f32x2{0.f, 0.f};
    for (int i = 0; i < 4; ++i) y += turned[i][lane] * sign4(i, w);
    float a = y[0], b = y[1];
    hadamard128(a, b, lane);
    typedef T t2 __attribute__((ext_vector_type(2)));
    reinterpret_cast<t2*>(static_cast<T*>(p.out) + token * p.ld + 128 * hb)[lane] =
        t2{static_cast<T>(a * 0.5f * kHadamardScale), static_cast<T>(b * 0.5f * kHadamardScale)};
}

// ---------------------------------------------------------------------------
// Low-rank adapters
// ---------------------------------------------------------------------------

constexpr int kMaxRank = 128;
constexpr int kMaxAdapters = 8191;  // what callers are promised; no kernel depends on how many there are

struct ShrinkArgs {
    const void* x;
    int64_t ld;
    const void* a;  // [adapters][rank][k]
    const int* ids;
    float* out;     // [parts][rows][rank]
    int rows, k, adapters, rank, parts;
    int shares;     // workgroups that share the adapters of 16 rows
};
constexpr int kShrinkWaves = 4, kShrinkSteps = 8;  // a workgroup's part of the K axis: 1024 channels at the most


// x A_a^T of 16 kSets rows over a part of the K axis, 16 kTiles ranks at a time, for each adapter a that these rows name and
// that is this workgroup's.  The rows are read once; a wave has up to eight steps of 32 channels, all their loads in flight
// (two sets of rows: four and four), and the waves add up in LDS in wave order.  Products of the inputs are exact, sums FP32.
template <typename T, int kTiles, int kSets>
__device__ __forceinline__ void shrink(const ShrinkArgs& p, int block, f32x4 (&sums)[kShrinkWaves][kTiles][kSets][64]) {
    const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4;
    const int w = uniform(static_cast<int>(threadIdx.x >> 6));
    const int share = block % p.shares;
    block /= p.shares;
    const int part = block % p.parts;
    block /= p.parts;
    const int groups = p.rank / (16 * kTiles), group = block % groups;
    const int row0 = 16 * kSets * (block / groups);
    const int id = lane < 16 * kSets && row0 + lane < p.rows ? p.ids[row0 + lane] : -1;  // lane r: row r's
    uint64_t left = __ballot(id >= 0 && id < p.adapters);
    if (!left) return;
    const int steps = p.k / 32, end = static_cast<int>(static_cast<int64_t>(steps) * (part + 1) / p.parts);
    const int s0 = static_cast<int>(static_cast<int64_t>(steps) * part / p.parts) + w;
    typedef T t8 __attribute__((ext_vector_type(8)));
    const t8 zero = {};
    t8 xv[kSets][kShrinkSteps];
#pragma unroll
    for (int q = 0; q < kSets; ++q) {
        const T* x = static_cast<const T*>(p.x) + min(row0 + 16 * q + n, p.rows - 1) * p.ld + 8 * g;
#pragma unroll
        for (int j = 0; j < kShrinkSteps; ++j) {
            const int s = s0 + kShrinkWaves * j;
            xv[q][j] = s < end ? *reinterpret_cast<const t8*>(x + 32 * s) : zero;
        }
    }
    for (int index = 0; left; ++index) {
        const int key = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t same = __ballot(id == key);
        left &= ~same;
        if (index % p.shares != share) continue;
        const T* a = static_cast<const T*>(p.a) + (static_cast<int64_t>(key) * p.rank + 16 * kTiles * group + n) * p.k + 8 * g;
        f32x4 acc[kTiles][kSets] = {};
        constexpr int kAhead = kShrinkSteps / kSets;
#pragma unroll
        for (int j0 = 0; j0 < kShrinkSteps; j0 += kAhead) {
            t8 av[kAhead][kTiles];
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int s = s0 + kShrinkWaves * (j0 + j);
                if (s < end) {
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
                        av[j][t] = *reinterpret_cast<const t8*>(a + static_cast<int64_t>(16 * t) * p.k + 32 * s);
                }
            }
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                if (s0 + kShrinkWaves * (j0 + j) < end) {
#pragma unroll
                    for (int t = 0; t < kTiles; ++t)
#pragma unroll
                        for (int q = 0; q < kSets; ++q) {
                            if constexpr (__is_same(T, __bf16))
                                acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[j][t], xv[q][j0 + j], acc[t][q], 0, 0, 0);
                            else
                                acc[t][q] = __builtin_amdgcn_mfma_f32_16x16x32_f16(av[j][t], xv[q][j0 + j], acc[t][q], 0, 0, 0);
                        }
                }
            }
        }
#pragma unroll
        for (int t = 0; t < kTiles; ++t)
#pragma unroll
            for (int q = 0; q < kSets; ++q) sums[w][t][q][lane] = acc[t][q];
        __syncthreads();
        for (int i = w; i < kTiles * kSets; i += kShrinkWaves) {
            const int t = i / kSets, q = i % kSets;
            f32x4 sum = sums[0][t][q][lane];
#pragma unroll
            for (int v = 1; v < kShrinkWaves; ++v) sum += sums[v][t][q][lane];
            if (same >> (16 * q + n) & 1)
                *reinterpret_cast<f32x4*>(p.out + (static_cast<int64_t>(part) * p.rows + row0 + 16 * q + n) * p.rank +
                                          16 * (kTiles * group + t) + 4 * g) = sum;
        }
        __syncthreads();
    }
}

// Scale exponents of rows that go in as f16 pieces: the largest |x suh| of a row comes to 2^11 .. 2^12, and what it can rotate
// to, 128^1/2 of it, under the type's 65504.  A row without a value, or with an infinity, is not scaled.
struct ExponentArgs {
    const void* x;
    int64_t ld;
    const _Float16* suh;
    int k;
    int* out;  // null: none are asked for
};

template <typename T>
__device__ __forceinline__ void row_exponent(const ExponentArgs& p, int64_t row, float (&most)[kShrinkWaves]) {
    const int lane = threadIdx.x & 63, w = uniform(static_cast<int>(threadIdx.x >> 6));
    typedef T t8 __attribute__((ext_vector_type(8)));
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    const T* x = static_cast<const T*>(p.x) + row * p.ld;
    float m = 0.f;
#pragma unroll 2
    for (int c = 8 * threadIdx.x; c < p.k; c += 8 * 64 * kShrinkWaves) {
        const t8 xv = *reinterpret_cast<const t8*>(x + c);
        const f16x4 s0 = *reinterpret_cast<const f16x4*>(p.suh + c), s1 = *reinterpret_cast<const f16x4*>(p.suh + c + 4);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            m = fmaxf(m, fabsf(static_cast<float>(xv[j]) * static_cast<float>(s0[j])));
            m = fmaxf(m, fabsf(static_cast<float>(xv[4 + j]) * static_cast<float>(s1[j])));
        }
    }
#pragma unroll
    for (int h = 1; h < 64; h <<= 1) m = fmaxf(m, __shfl_xor(m, h));
    if (lane == 0) most[w] = m;
    __syncthreads();
    if (threadIdx.x) return;
    for (int v = 1; v < kShrinkWaves; ++v) m = fmaxf(m, most[v]);
    const int exponent = static_cast<int>(__builtin_bit_cast(uint32_t, m) >> 23);
    p.out[row] = m == 0.f || exponent == 255 ? 0 : 11 + 127 - exponent;
}

// What an adapter projection needs before its product: the rows' rotation, and beside it the adapters' first products.  Rows
// that go in as f16 pieces are only looked at here, for their scales.
template <typename T, int kTiles, int kSets>
__global__ __launch_bounds__(64 * kShrinkWaves) void prepare_rows_kernel(const RotateArgs r, const ExponentArgs e,
                                                                         const ShrinkArgs p, int shrinks) {
    __shared__ __attribute__((aligned(16))) union {
        f32x4 sums[kShrinkWaves][kTiles][kSets][64];
        u32x4 staged[256 * kBf16Pieces * kRotateBlocks];
        float most[kShrinkWaves];
    } l;
    const int block = static_cast<int>(blockIdx.x);
    if (block < shrinks)
        shrink<T, kTiles, kSets>(p, block, l.sums);
    else if (e.out)
        row_exponent<T>(e, block - shrinks, l.most);
    else if (r.layout.row == 16)
        rotate_quad<T, kBf16Pieces>(r, block - shrinks, l.staged);
    else
        rotate_block<T>(r, static_cast<int64_t>(block - shrinks) * kShrinkWaves + uniform(static_cast<int>(threadIdx.x >> 6)),
                        threadIdx.x & 63);
}

// And their rotation, once the scales are known.
template <typename T>
__global__ __launch_bounds__(256) void rotate_scaled_kernel(const RotateArgs r) {
    __shared__ __attribute__((aligned(16))) u32x4 staged[256 * kF16Pieces * kRotateBlocks];
    rotate_quad<T, kF16Pieces>(r, blockIdx.x, staged);
}

struct FinishArgs {
    const float* part;  // [parts][rows][cols]
    int parts;
    const _Float16* svh;
    const int* ids;     // null: no adapters
    const float* low;   // [low_parts][rows][rank]
    int low_parts, adapters;
    const void* b;      // [adapters][cols][rank]
    const float* scale;
    int rank;
    void* out;
    int64_t ld;
    int rows, nb;
    const int* exponents;  // null: none; else row r's sums are 2^exponents[r] too large
};

constexpr int kFinishLd = kMaxRank + 4;  // floats; rows start in different banks

// low B^T of one adapter for 16 rows and the wave's 32 columns, on the matrix cores: low [16][rank] in three bf16 pieces, B as
// it is (bf16) or in two (f16, whose 11 bits they hold): products of the FP32 values, sums FP32.
template <typename T>
__device__ __forceinline__ void expand(const float (&low)[16][kFinishLd], const T* b, int rank, int lane, f32x4 (&acc)[2]) {
    typedef T t8 __attribute__((ext_vector_type(8)));
    const int n = lane & 15, g = lane >> 4;
    const t8 zero = {};
    t8 bv[kMaxRank / 32][2];
#pragma unroll
    for (int q = 0; q < kMaxRank / 32; ++q)
#pragma unroll
        for (int t = 0; t < 2; ++t)
            bv[q][t] = 32 * q + 8 * g < rank
                           ? *reinterpret_cast<const t8*>(b + static_cast<int64_t>(16 * t + n) * rank + 32 * q + 8 * g)
                           : zero;
#pragma unroll
    for (int q = 0; q < kMaxRank / 32; ++q) {
        if (32 * q >= rank) break;
        const bool in = 32 * q + 8 * g < rank;
        bf16x8 a[kBf16Pieces];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            __bf16 piece[kBf16Pieces];
            split(in ? low[n][32 * q + 8 * g + j] : 0.f, piece);
#pragma unroll
            for (int i = 0; i < kBf16Pieces; ++i) a[i][j] = piece[i];
        }
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            if constexpr (__is_same(T, __bf16)) {
#pragma unroll
                for (int i = 0; i < kBf16Pieces; ++i)
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], bv[q][t], acc[t], 0, 0, 0);
            } else {
                bf16x8 bh, bl;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const float v = static_cast<float>(bv[q][t][j]);
                    const __bf16 h = static_cast<__bf16>(v);
                    bh[j] = h;
                    bl[j] = static_cast<__bf16>(v - static_cast<float>(h));
                }
#pragma unroll
                for (int i = 0; i < kBf16Pieces; ++i) {
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], bh, acc[t], 0, 0, 0);
                    acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[i], bl, acc[t], 0, 0, 0);
                }
            }
        }
    }
}

// Sum of the parts, back into the output's basis, plus the adapter's second product: a workgroup of four waves for 16 rows by
// 128 columns.  Each wave has every fourth row; under four rows the waves share the parts of each instead.
template <typename T>
__global__ __launch_bounds__(256) void finish_kernel(const FinishArgs p) {
    __shared__ f32x2 sums[4][64];
    __shared__ __attribute__((aligned(16))) float low[16][kFinishLd], more[16][kFinishLd];
    const int lane = threadIdx.x & 63, w = uniform(static_cast<int>(threadIdx.x >> 6));
    const int nb = static_cast<int>(blockIdx.x % p.nb), first = 16 * static_cast<int>(blockIdx.x / p.nb);
    const int count = min(16, p.rows - first);
    const int64_t cols = 128 * static_cast<int64_t>(p.nb), stride = p.rows * cols;
    const float* src = p.part + 128 * nb + 2 * lane;
    const bool share = count < 4;
    const int mine = share ? w < count : (count - w + 3) >> 2;  // rows of this wave
    int row[4];
    f32x2 v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {  // rows past the last repeat another; not stored
        row[i] = share ? min(w, count - 1) : i < mine ? w + 4 * i : w;
        v[i] = f32x2{0.f, 0.f};
    }
    int id = p.ids && lane < count ? p.ids[first + lane] : -1;  // lane r: row r's
    if (id >= p.adapters) id = -1;
    if (p.ids) {  // the first products of all rows, scaled
        const int quads = p.rank >> 2;
        for (int i = threadIdx.x; i < count * quads; i += 256) {
            const int r = i / quads, c = 4 * (i - r * quads);
            const int key = p.ids[first + r];
            const float* at = p.low + static_cast<int64_t>(first + r) * p.rank + c;
            f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
            for (int s = 0; s < p.low_parts; ++s)
                sum += *reinterpret_cast<const f32x4*>(at + static_cast<int64_t>(s) * p.rows * p.rank);
            const bool has = key >= 0 && key < p.adapters;  // else nothing was written there
            *reinterpret_cast<f32x4*>(&low[r][c]) = has ? sum * p.scale[key] : f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }
    if (share) {
        for (int r = 0; r < count; ++r) {
            sums[w][lane] = sum_parts(src + (first + r) * cols, stride, w, 4, p.parts);
            __syncthreads();
            if (w == r) v[0] = sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
            __syncthreads();
        }
    } else {
        for (int s = 0; s < p.parts; s += 4) {  // sixteen loads in flight
            f32x2 t[4][4];
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    t[j][i] = *reinterpret_cast<const f32x2*>(src + min(s + j, p.parts - 1) * stride + (first + row[i]) * cols);
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (s + j < p.parts) v[i] += t[j][i];
        }
        __syncthreads();
    }
    const f16x2 sv = reinterpret_cast<const f16x2*>(p.svh + 128 * nb)[lane];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= mine) break;
        float a = v[i][0], b = v[i][1];
        if (p.exponents) {
            const int e = -p.exponents[first + row[i]];
            a = ldexpf(a, e);
            b = ldexpf(b, e);
        }
        hadamard128(a, b, lane);
        v[i] = f32x2{a * kHadamardScale * static_cast<float>(sv[0]), b * kHadamardScale * static_cast<float>(sv[1])};
    }
    const uint64_t with = __ballot(id >= 0);
    const int key0 = __builtin_amdgcn_readlane(id, with ? __builtin_ctzll(with) : 0);
    const uint64_t same0 = with & __ballot(id == key0), others = with & ~same0;
    const int key1 = __builtin_amdgcn_readlane(id, others ? __builtin_ctzll(others) : 0);
    const uint64_t same1 = others & __ballot(id == key1);
    typedef T t8 __attribute__((ext_vector_type(8)));
    if (with && !(others & ~same1)) {
        // Rows of one or two adapters, as in prompts: every wave reads 32 columns of them once for all rows (2048 rows of rank
        // 64 in runs: 22 us, 35 on the vector units as below).
        f32x4 sum[2] = {};
        for (int turn = 0; turn < (others ? 2 : 1); ++turn) {
            const uint32_t same = static_cast<uint32_t>(turn ? same1 : same0);
            f32x4 acc[2] = {};
            expand<T>(low, static_cast<const T*>(p.b) + (static_cast<int64_t>(turn ? key1 : key0) * cols + 128 * nb + 32 * w) * p.rank,
                      p.rank, lane, acc);
#pragma unroll
            for (int i = 0; i < 4; ++i)  // an adapter's infinities stay in its rows
                if (same >> (4 * (lane >> 4) + i) & 1) {
                    sum[0][i] = acc[0][i];
                    sum[1][i] = acc[1][i];
                }
        }
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) more[4 * (lane >> 4) + i][32 * w + 16 * t + (lane & 15)] = sum[t][i];
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (with >> row[i] & 1) v[i] += *reinterpret_cast<const f32x2*>(&more[row[i]][2 * lane]);
    } else if (with) {
        // Rows of many adapters, as in a decode batch: a wave reads 128 columns of an adapter once for those of its rows that
        // name it, four at the most, where the matrix cores would go through all of the sixteen rows' adapters (48 rows of 32
        // adapters of rank 16: 10 us, 27 on the matrix cores).  Asking for B before the sums, or for the next adapter's during
        // this one's, gained nothing.
        int key[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) key[i] = i < mine ? __builtin_amdgcn_readlane(id, row[i]) : -1;
        for (int turn = 0; turn < mine; ++turn) {
            const int k = turn == 0 ? key[0] : turn == 1 ? key[1] : turn == 2 ? key[2] : key[3];
            if (k < 0) continue;  // no adapter, or done with an earlier row
            const T* b0 = static_cast<const T*>(p.b) + (static_cast<int64_t>(k) * cols + 128 * nb + 2 * lane) * p.rank;
            t8 next[4];  // sixteen ranks of both columns, asked for one turn ahead
            auto fetch = [&](int r) {
                r = min(r, p.rank - 16);
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    next[j] = *reinterpret_cast<const t8*>(b0 + (j >> 1) * p.rank + r + 8 * (j & 1));
            };
            fetch(0);
            for (int r = 0; r < p.rank; r += 16) {
                t8 x[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) x[j] = next[j];
                fetch(r + 16);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (key[i] != k) continue;
#pragma unroll
                    for (int j = 0; j < 16; ++j) {
                        const float f = low[row[i]][r + j];
                        v[i][0] = __builtin_fmaf(f, static_cast<float>(x[j >> 3][j & 7]), v[i][0]);
                        v[i][1] = __builtin_fmaf(f, static_cast<float>(x[2 + (j >> 3)][j & 7]), v[i][1]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (key[i] == k) key[i] = -1;
        }
    }
    typedef T t2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (i >= mine) break;
        reinterpret_cast<t2*>(static_cast<T*>(p.out) + (first + row[i]) * p.ld + 128 * nb)[lane] =
            t2{static_cast<T>(v[i][0]), static_cast<T>(v[i][1])};
    }
}

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

constexpr int64_t kMaxPartBytes = int64_t(128) << 20;  // part sums of one product, unless one part alone takes more

template <int G, bool kHalf, int kTables>
int launch_product_g(const ProductArgs& args, int cus, hipStream_t stream) {
    // 128, 168 and 256 registers a lane; four groups keep up to five more in memory, read and written once a piece of work
    constexpr int kWaves = G == 1 ? 16 : G == 2 ? 12 : 8;
    const int64_t items = static_cast<int64_t>(args.max_chunks) * args.nmat * args.nb * args.parts;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(cus, items)));
    hipLaunchKernelGGL((product_kernel<G, kHalf, kWaves, kTables>), grid, dim3(64 * kWaves), 0, stream, args);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

// The next number of parts after p that makes them shorter: between the two only the turns grow.
int next_cut(int strips, int p) {
    const int length = (strips + p - 1) / p;
    return length == 1 ? strips + 1 : (strips + length - 2) / (length - 1);
}

// Parts that the K axis (`strips`) of `units` column blocks is cut into, chosen so that the compute units come out even: the
// time of a strip on one is the table reads of its wave, shared by the unit's waves; with few waves their latencies show
// (0.9 of a wave's time beside the reads of all: 16 waves decode 4.96e12 labels a second, 8 waves 4.73e12); and a part
// costs its set-up, about a strip, and its sums' way to memory and back, 0.28 strips a row.  `most`: units there can be.
int cut_parts(double units, int64_t most, int strips, int limit, int rows, int cus) {
    int best = 1;
    double least = 0.0;
    for (int p = 1; p <= std::min(limit, strips); p = next_cut(strips, p)) {
        if (most * p >= int64_t(1) << 31) break;  // the product counts its items in 32 bits
        const double turns = std::ceil(units * p / cus);
        const double cost = (turns + 0.9) * ((strips + p - 1) / p + 1.0 + 0.28 * rows);
        if (p == 1 || cost < least) {
            least = cost;
            best = p;
        }
    }
    return best;
}

template <int G, int kTables>
int launch_rows_g(const ProductArgs& args, int cus, hipStream_t stream) {
    const int64_t items = static_cast<int64_t>(args.max_chunks) * args.nb * args.parts;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(cus, items)));
    hipLaunchKernelGGL((product_rows_kernel<G, kTables>), grid, dim3(64 * kRowWaves), 0, stream, args);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

// Rows that a wave multiplies at once: `groups` times 16, or 8 with groups 0.
int chunk_rows_of(int groups) { return groups ? 16 * groups : 8; }

// All passes of a product: the tables of at most two rates fit LDS at once.  `row_groups`: as in cut_rows (0: product_kernel).
int launch_product(ProductArgs args, int groups, int row_groups, int rates, const uint8_t* const* luts, int cus, hipStream_t stream) {
    int set[3], n = 0;
    for (int b = 2; b <= 4; ++b)
        if (rates >> b & 1) set[n++] = b;
    for (int first = 0, pass = 0; first < n; first += 2, ++pass) {
        args.pass = pass;
        args.luts = std::min(2, n - first);
        for (int j = 0; j < args.luts; ++j) {
            args.lut_bits[j] = set[first + j];
            args.lut[j] = luts[set[first + j] - 2];
        }
        const bool two = args.luts > 1;
        if (row_groups) {
            const int rc = row_groups == 2 ? (two ? launch_rows_g<2, 2> : launch_rows_g<2, 1>)(args, cus, stream)
                                           : (two ? launch_rows_g<4, 2> : launch_rows_g<4, 1>)(args, cus, stream);
            if (rc != kOk) return rc;
            continue;
        }
        const bool pairs = args.luts == 1 && args.lut_bits[0] == 2;
#define QSRT_PRODUCT(G, HALF) \
    (pairs ? launch_product_g<G, HALF, 0> : two ? launch_product_g<G, HALF, 2> : launch_product_g<G, HALF, 1>)(args, cus, stream)
        const int rc = groups == 0   ? QSRT_PRODUCT(1, true)
                       : groups == 1 ? QSRT_PRODUCT(1, false)
                       : groups == 2 ? QSRT_PRODUCT(2, false)
                                     : QSRT_PRODUCT(4, false);
#undef QSRT_PRODUCT
        if (rc != kOk) return rc;
    }
    return kOk;
}

int passes_of(int rates) { return __builtin_popcount(rates & 0x1C) > 2 ? 2 : 1; }

// The same for product_rows_kernel, with the groups of 16 rows that each of a workgroup's eight waves takes.  A workgroup is an
// item; with 4 groups a strip takes it about 1.2 us, a part's sums (256 KB) as long as 16 strips, there and back, and its
// set-up 3 or more.  With 2 all of it takes 0.6 of that: half the rows, at the same reads of the payload and the tables.  So few
// rows or items go with 2 (a call of 7168 x 7168, 256 rows: 80 us, with 4 114; 5120 x 2048, 512 rows: 55 and 63), many
// with 4 (7168 x 7168, 4096 rows: 837 us, with 2 907).
struct RowCut {
    int groups, parts;
};
RowCut cut_rows(int64_t rows, int64_t nb, int strips, int limit, int cus) {
    RowCut best{4, 1};
    double least = 0.0;
    for (const int groups : {4, 2}) {
        const int64_t each = 16 * kRowWaves * groups, units = (rows + each - 1) / each * nb;
        for (int p = 1; p <= std::min(limit, strips); p = next_cut(strips, p)) {
            if (units * p >= int64_t(1) << 31) break;
            const double turns = std::ceil(static_cast<double>(units * p) / cus);
            const double cost = turns * ((strips + p - 1) / p + 19.0) * (groups == 4 ? 1.0 : 0.6);
            if (least == 0.0 || cost < least) {
                least = cost;
                best = RowCut{groups, p};
            }
        }
    }
    return best;
}

// What a workspace's size depends on; its functions take any numbers, and answer 0 where the call would refuse them.
const char* size_fault(const qsrt_packed_matrix* m) {
    if (m->rows <= 0 || m->cols <= 0 || m->rows % 128 || m->cols % 128) return "rows and cols must be multiples of 128";
    if (m->rows > (1 << 22) || m->cols > (1 << 22) || m->rows * m->cols >= int64_t(1) << 32)
        return "matrix too large (2^32 weights)";  // the kernels' offsets in a payload have 31 bits, K4 takes half a byte
    if (m->rate_axis != 0 && m->rate_axis != 1) return "rate_axis must be 0 (rows) or 1 (columns)";
    if ((m->rates & 0x1C) == 0 || (m->rates & ~0x1C)) return "rates must name K2, K3 or K4";
    return nullptr;
}

const char* matrix_fault(const qsrt_packed_matrix* m, const uint8_t* const* luts) {
    if (!m || !m->words || !m->records || !m->suh || !m->svh) return "null pointer in a matrix";
    if (const char* e = size_fault(m)) return e;
    if (m->key_stride < 0 || m->record_stride < 0 || m->suh_stride < 0 || m->svh_stride < 0) return "negative stride";
    if (reinterpret_cast<uintptr_t>(m->words) % 4 || m->key_stride % 2) return "words must be 4-byte aligned";
    if (reinterpret_cast<uintptr_t>(m->suh) % 8 || reinterpret_cast<uintptr_t>(m->svh) % 8 || m->suh_stride % 4 ||
        m->svh_stride % 4)
        return "scales must be 8-byte aligned";
    for (int b = 2; b <= 4; ++b)
        if ((m->rates >> b & 1) && (!luts || !luts[b - 2] || reinterpret_cast<uintptr_t>(luts[b - 2]) % 16))
            return "a rate's label table is missing or not 16-byte aligned";
    return nullptr;
}

// A launch has fewer than 2^32 threads.  None here takes more than one for two channels, of rows rounded up to 16, but for an
// adapter projection's, which have 2^28 more at the most (256 a row), and the layer's router, which shares its launch with a
// rotation and is looked at by itself.
bool launch_fits(int64_t rows, int64_t a, int64_t b) { return (rows + 15) / 16 * 16 * std::max(a, b) < int64_t(1) << 32; }

const char* rows_fault(const void* p, int64_t rows, int64_t ld, int64_t cols, int align) {
    if (!p) return "null rows";
    if ((rows > 1 && (ld < cols || ld % (align / 2))) || reinterpret_cast<uintptr_t>(p) % align) return "rows are not aligned";
    return nullptr;
}

struct Carve {
    char* base;
    size_t used = 0;
    template <typename T>
    T* take(int64_t n) {
        T* p = reinterpret_cast<T*>(base + used);
        used += (static_cast<size_t>(n) * sizeof(T) + 255) / 256 * 256;
        return p;
    }
};

int part_limit(int64_t row_floats, int strips) {
    const int64_t fit = kMaxPartBytes / (row_floats * 4);
    return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(fit, strips)));
}

int64_t rotated_bytes(int64_t rows, int64_t channels, int pieces) { return (rows + 15) / 16 * 16 * (channels / 32) * strip_bytes(pieces); }

struct MoeSpace {
    Chunk* chunks;
    int *order, *clean;
    char *x[2], *mid;
    float *part, *logits;
    int parts[2], passes[2], groups, max_chunks;
    bool every;  // rows are rotated at every expert's scales, before the choice is known
    size_t bytes;
};

MoeSpace moe_space(void* ws, int64_t tokens, int k, int64_t hidden, int64_t inter, int64_t experts, int rates13, int rates2,
                   bool shared, bool router, bool either, int cus) {
    MoeSpace s;
    const int64_t pairs = tokens * k;
    // An expert's rows are one chunk more often than not: 2% of experts get over 8 of 4 a head.  Larger chunks cost more a
    // strip, more chunks decode again (16 experts, 4096 x 1536 at K3, us a layer with chunks of 8, 16, 32, 64: 4 rows a head
    // 90, 90, 94, 118; 8 rows 128, 97, 104, 132; 16 rows 184, 150, 114, 140; 24 rows 247, 165, 133, 170; 32 rows 322, 204,
    // 211, 185).
    s.groups = pairs <= 4 * experts ? 0 : pairs <= 8 * experts ? 1 : pairs <= 24 * experts ? 2 : 4;
    const int chunk_rows = chunk_rows_of(s.groups);
    s.max_chunks = static_cast<int>(most_chunks(pairs, experts, chunk_rows));
    // chunks to expect under an even router; the parts are cut for them, as the host does not wait for the real ones
    const double touched = experts * (1.0 - std::pow(1.0 - 1.0 / experts, static_cast<double>(pairs)));
    const double each = pairs / touched, chunks = std::max(1.0, touched * std::ceil(each / chunk_rows));
    const int rows = static_cast<int>(std::min<double>(chunk_rows, std::ceil(each)));
    Carve c{static_cast<char*>(ws)};
    s.chunks = c.take<Chunk>(s.max_chunks);
    s.order = c.take<int>(pairs);
    s.clean = c.take<int>(pairs);
    s.logits = c.take<float>(router ? router_logit_bytes(tokens, hidden, experts) / sizeof(float) : 0);
    // Scales of their own: a row at a scale is a wave's few microseconds, and while all of them fit the chip at once beside
    // the router they save a launch behind the choice (8 experts, 256 channels: 33 -> 29 us a layer).
    s.every = !shared && router && tokens * experts * (hidden / 128) <= 1024;
    int64_t rotated = shared ? tokens : s.every ? tokens * experts : pairs;
    if (either && s.every) rotated = std::max(rotated, pairs);  // room for a call without a router too
    for (int m = 0; m < 2; ++m) s.x[m] = c.take<char>(rotated_bytes(rotated, hidden, kBf16Pieces));
    s.mid = c.take<char>(rotated_bytes(pairs, inter, kBf16Pieces));
    s.passes[0] = passes_of(rates13);
    s.passes[1] = passes_of(rates2);
    const int64_t row_floats[2] = {2 * pairs * inter * s.passes[0], pairs * hidden * s.passes[1]};
    const int64_t units[2] = {2 * inter / 128, hidden / 128}, strips[2] = {hidden / 32, inter / 32};
    int64_t floats = 0;
    for (int i = 0; i < 2; ++i) {
        s.parts[i] = cut_parts(chunks * units[i], s.max_chunks * units[i], static_cast<int>(strips[i]),
                               part_limit(row_floats[i], static_cast<int>(strips[i])), rows, cus);
        floats = std::max(floats, s.parts[i] * row_floats[i]);
    }
    s.part = c.take<float>(floats);
    s.bytes = c.used;
    return s;
}

void set_matrix(ProductArgs& a, int i, const qsrt_packed_matrix* m) {
    a.words[i] = m->words;
    a.key_stride[i] = m->key_stride;
    a.records[i] = m->records;
    a.record_stride[i] = m->record_stride;
    a.axis = m->rate_axis;
    a.kb = static_cast<int>(m->rows / 128);
    a.nb = static_cast<int>(m->cols / 128);
}

unsigned blocks_of(int64_t waves) { return static_cast<unsigned>((waves + 3) / 4); }

int launch_rotate(const RotateArgs& args, int dtype, hipStream_t stream) {
    const dim3 grid(blocks_of(rotate_waves(args)));
    if (dtype == 0)
        hipLaunchKernelGGL(rotate_rows_kernel<__bf16>, grid, dim3(256), 0, stream, args);
    else
        hipLaunchKernelGGL(rotate_rows_kernel<_Float16>, grid, dim3(256), 0, stream, args);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

const char* moe_size_fault(const qsrt_packed_matrix* w1, const qsrt_packed_matrix* w3, const qsrt_packed_matrix* w2,
                           int64_t experts, int64_t tokens, int k) {
    for (const qsrt_packed_matrix* m : {w1, w3, w2})
        if (const char* e = size_fault(m)) return e;
    if (w1->rows != w3->rows || w1->cols != w3->cols || w2->rows != w1->cols || w2->cols != w1->rows ||
        w1->rate_axis != w3->rate_axis)
        return "w1, w3 [hidden, inter] and w2 [inter, hidden] do not match";
    if ((w1->suh_stride == 0) != (w3->suh_stride == 0)) return "w1 and w3 must both share their suh, or neither";
    if (experts < 1 || experts > kMaxKeys) return "experts must be 1 .. 8191";
    if (k < 1 || k > (1 << 20) || tokens < 0 || tokens > (1 << 20) || tokens * k > (1 << 20))
        return "tokens * k must be at most 2^20";
    if (!launch_fits(tokens * k, w1->cols, w1->rows)) return "too many tokens for these matrices";
    return nullptr;
}

const char* moe_fault(const qsrt_packed_matrix* w1, const qsrt_packed_matrix* w3, const qsrt_packed_matrix* w2,
                      const uint8_t* const* luts, int64_t experts, int64_t tokens, int k) {
    for (const qsrt_packed_matrix* m : {w1, w3, w2})
        if (const char* e = matrix_fault(m, luts)) return e;
    return moe_size_fault(w1, w3, w2, experts, tokens, k);
}

struct MoeCall {
    const qsrt_packed_matrix *w1, *w3, *w2;
    const uint8_t* const* luts;
    int64_t experts;
    int activation;
    const float *pre_signs, *post_signs;
    const void* x;
    int64_t x_ld;
    int dtype;
    int64_t tokens;
    int k;
    const int32_t* ids;
    const float* weights;
    void* out;
    int64_t out_ld;
};

// The experts of a layer; with a router (its logits' place is filled in here) also its choice.
int run_moe(const char* name, const MoeCall& c, RouterArgs* router, void* ws, size_t ws_bytes, hipStream_t stream) {
    if (const char* e = moe_fault(c.w1, c.w3, c.w2, c.luts, c.experts, c.tokens, c.k))
        return fail(kBadArgument, "%s: %s", name, e);
    if (c.dtype != 0 && c.dtype != 1) return fail(kBadArgument, "%s: dtype must be 0 (bf16) or 1 (f16)", name);
    if (c.activation != 0 && c.activation != 1) return fail(kBadArgument, "%s: unknown activation", name);
    const bool coupled = c.pre_signs != nullptr;
    if (coupled != (c.post_signs != nullptr) || reinterpret_cast<uintptr_t>(c.pre_signs) % 8)
        return fail(kBadArgument, "%s: coupled weights need both sign vectors, 8-byte aligned", name);
    if (coupled && c.w1->rows % 512) return fail(kBadArgument, "%s: coupled weights need a multiple of 512 hidden channels", name);
    if (c.tokens == 0) return kOk;
    const int64_t hidden = c.w1->rows, inter = c.w1->cols, pairs = c.tokens * c.k;
    if (const char* e = rows_fault(c.x, c.tokens, c.x_ld, hidden, 8)) return fail(kBadArgument, "%s: x: %s", name, e);
    if (const char* e = rows_fault(c.out, c.tokens, c.out_ld, hidden, 8)) return fail(kBadArgument, "%s: out: %s", name, e);
    if (!c.ids || !c.weights) return fail(kBadArgument, "%s: null routing", name);
    if (router) {
        if (const char* e = router_fault(*router)) return fail(kBadArgument, "%s: %s", name, e);
        RotateArgs rows{};  // those that all experts share are rotated beside it
        rows.rows = c.w1->suh_stride == 0 ? c.tokens : 0;
        rows.kb = static_cast<int>(hidden / 128);
        rows.nmat = 2;
        if (router_blocks(c.tokens, hidden, c.experts, rows) * 256 >= int64_t(1) << 32)
            return fail(kBadArgument, "%s: too many tokens for these matrices", name);
    }
    int cus = 0;
    if (const int rc = current_cu_count(&cus)) return rc;
    const bool shared = c.w1->suh_stride == 0;
    const int rates13 = c.w1->rates | c.w3->rates;
    const MoeSpace s =
        moe_space(ws, c.tokens, c.k, hidden, inter, c.experts, rates13, c.w2->rates, shared, router != nullptr, false, cus);
    if (!ws || ws_bytes < s.bytes) return fail(kWorkspaceTooSmall, "%s: needs %zu workspace bytes", name, s.bytes);

    GroupArgs ga{};
    ga.ids = c.ids;
    ga.n = static_cast<int>(pairs);
    ga.keys = static_cast<int>(c.experts);
    ga.chunk_rows = chunk_rows_of(s.groups);
    ga.max_chunks = s.max_chunks;
    ga.chunks = s.chunks;
    ga.order = s.order;
    ga.clean = s.clean;
    RotateArgs ra{};
    ra.x = c.x;
    ra.ld = c.x_ld;
    ra.suh[0] = static_cast<const _Float16*>(c.w1->suh);
    ra.suh[1] = static_cast<const _Float16*>(c.w3->suh);
    ra.suh_stride[0] = c.w1->suh_stride;
    ra.suh_stride[1] = c.w3->suh_stride;
    ra.ids = shared || s.every ? nullptr : s.clean;
    ra.x_div = shared ? 1 : c.k;
    ra.every = s.every ? static_cast<int>(c.tokens) : 0;
    ra.out[0] = s.x[0];
    ra.out[1] = s.x[1];
    ra.rows = shared ? c.tokens : s.every ? c.tokens * c.experts : pairs;
    ra.kb = static_cast<int>(hidden / 128);
    ra.nmat = 2;
    ra.layout = row_layout(ra.kb, s.groups > 1, kBf16Pieces);
    ra.residual = coupled;
    RotateArgs beside = ra;  // rows that all experts share are rotated beside the router or the grouping
    if (!shared && !s.every) beside.rows = 0;
    if (router) {
        router->logits = s.logits;
        if (const int rc = launch_router(*router, beside, &ga, stream)) return rc;
    } else if (const int rc = launch_group(ga, beside, c.dtype, stream)) {
        return rc;
    }
    if (!shared && !s.every)
        if (const int rc = launch_rotate(ra, c.dtype, stream)) return rc;

    ProductArgs pa{};
    set_matrix(pa, 0, c.w1);
    set_matrix(pa, 1, c.w3);
    pa.x[0] = s.x[0];
    pa.x[1] = s.x[1];
    pa.x_div = shared || s.every ? c.k : 1;
    pa.x_every = ra.every;
    pa.layout = ra.layout;
    pa.chunks = s.chunks;
    pa.order = s.order;
    pa.max_chunks = s.max_chunks;
    pa.parts = s.parts[0];
    pa.part = s.part;
    pa.nmat = 2;
    pa.rows = static_cast<int>(pairs);
    if (const int rc = launch_product(pa, s.groups, 0, rates13, c.luts, cus, stream)) return rc;

    MiddleArgs ma{};
    ma.part = s.part;
    ma.parts = s.parts[0] * s.passes[0];
    ma.ids = s.clean;
    ma.svh[0] = static_cast<const _Float16*>(c.w1->svh);
    ma.svh[1] = static_cast<const _Float16*>(c.w3->svh);
    ma.svh_stride[0] = c.w1->svh_stride;
    ma.svh_stride[1] = c.w3->svh_stride;
    ma.suh = static_cast<const _Float16*>(c.w2->suh);
    ma.suh_stride = c.w2->suh_stride;
    ma.out = s.mid;
    ma.pairs = static_cast<int>(pairs);
    ma.ib = static_cast<int>(inter / 128);
    ma.layout = row_layout(ma.ib, s.groups > 1, kBf16Pieces);
    ma.act = c.activation;
    ma.pre_signs = c.pre_signs;
    ma.post_signs = c.post_signs;
    hipLaunchKernelGGL((coupled ? middle_coupled_kernel : middle_kernel), dim3(blocks_of(pairs * ma.ib)), dim3(256), 0, stream, ma);
    QSRT_HIP_TRY(hipGetLastError());

    ProductArgs pb{};
    set_matrix(pb, 0, c.w2);
    pb.x[0] = s.mid;
    pb.x_div = 1;
    pb.layout = ma.layout;
    pb.chunks = s.chunks;
    pb.order = s.order;
    pb.max_chunks = s.max_chunks;
    pb.parts = s.parts[1];
    pb.part = s.part;
    pb.nmat = 1;
    pb.rows = static_cast<int>(pairs);
    if (const int rc = launch_product(pb, s.groups, 0, c.w2->rates, c.luts, cus, stream)) return rc;

    CombineArgs ca{};
    ca.part = s.part;
    ca.parts = s.parts[1] * s.passes[1];
    ca.ids = s.clean;
    ca.weights = c.weights;
    ca.svh = static_cast<const _Float16*>(c.w2->svh);
    ca.svh_stride = c.w2->svh_stride;
    ca.out = c.out;
    ca.ld = c.out_ld;
    ca.tokens = static_cast<int>(c.tokens);
    ca.k = c.k;
    ca.hb = static_cast<int>(hidden / 128);
    const dim3 cgrid(static_cast<unsigned>(c.tokens * (coupled ? ca.hb / 4 : ca.hb)));
    const dim3 cblock(coupled ? 256 * std::min(c.k, kCoupledShares) : 64 * std::min(c.k, kCombineWaves));
    if (c.dtype == 0)
        hipLaunchKernelGGL((coupled ? combine_coupled_kernel<__bf16> : combine_kernel<__bf16>), cgrid, cblock, 0, stream, ca);
    else
        hipLaunchKernelGGL((coupled ? combine_coupled_kernel<_Float16> : combine_kernel<_Float16>), cgrid, cblock, 0, stream, ca);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

}  // namespace

extern "C" size_t qsrt_packed_moe_workspace_bytes(const qsrt_packed_matrix* w1, const qsrt_packed_matrix* w3,
                                                  const qsrt_packed_matrix* w2, int64_t experts, int64_t tokens, int k) {
    int cus = 0;
    if (!w1 || !w3 || !w2 || tokens == 0 || moe_size_fault(w1, w3, w2, experts, tokens, k) || current_cu_count(&cus)) return 0;
    return moe_space(nullptr, tokens, k, w1->rows, w1->cols, experts, w1->rates | w3->rates, w2->rates, w1->suh_stride == 0,
                     true, true, cus)
        .bytes;
}

extern "C" int qsrt_packed_moe_plan(const qsrt_packed_matrix* w1, const qsrt_packed_matrix* w3, const qsrt_packed_matrix* w2,
                                    int64_t experts, int64_t tokens, int k, int64_t* plan) {
    if (!w1 || !w3 || !w2 || !plan || tokens == 0) return fail(kBadArgument, "qsrt_packed_moe_plan: null pointer or no tokens");
    if (const char* e = moe_size_fault(w1, w3, w2, experts, tokens, k)) return fail(kBadArgument, "qsrt_packed_moe_plan: %s", e);
    int cus = 0;
    if (const int rc = current_cu_count(&cus)) return rc;
    const MoeSpace s = moe_space(nullptr, tokens, k, w1->rows, w1->cols, experts, w1->rates | w3->rates, w2->rates,
                                 w1->suh_stride == 0, true, true, cus);
    plan[0] = chunk_rows_of(s.groups);
    plan[1] = s.parts[0];
    plan[2] = s.parts[1];
    return kOk;
}

extern "C" int qsrt_packed_moe(const qsrt_packed_matrix* w1, const qsrt_packed_matrix* w3, const qsrt_packed_matrix* w2,
                               const uint8_t* const* luts, int64_t experts, int activation, const float* pre_signs,
                               const float* post_signs, const void* x, int64_t x_ld, int dtype, int64_t tokens, int k, const int32_t* ids, const float* weights, void* out,
                               int64_t out_ld, void* ws, size_t ws_bytes, void* stream) {
    const MoeCall call{w1, w3, w2, luts, experts, activation, pre_signs, post_signs, x, x_ld, dtype,
                       tokens, k, ids, weights, out, out_ld};
    return run_moe("qsrt_packed_moe", call, nullptr, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

extern "C" int qsrt_packed_moe_layer(const qsrt_packed_matrix* w1, const qsrt_packed_matrix* w3,
                                     const qsrt_packed_matrix* w2, const uint8_t* const* luts, int64_t experts,
                                     int activation, const float* pre_signs, const float* post_signs, const void* router, int64_t router_ld, const float* bias, int scoring,
                                     int normalize, float scale, const void* x, int64_t x_ld, int dtype, int64_t tokens,
                                     int k, float* weights, int32_t* ids, void* out, int64_t out_ld, void* ws,
                                     size_t ws_bytes, void* stream) {
    const MoeCall call{w1, w3, w2, luts, experts, activation, pre_signs, post_signs, x, x_ld, dtype,
                       tokens, k, ids, weights, out, out_ld};
    if (tokens < 0 || tokens > (1 << 20) || !w1 || w1->rows > (1 << 22))
        return fail(kBadArgument, "qsrt_packed_moe_layer: bad sizes");
    RouterArgs r{x, x_ld, router, router_ld, dtype, static_cast<int>(tokens), static_cast<int>(w1->rows),
                 static_cast<int>(experts), k, bias, scoring, normalize, scale, weights, ids, nullptr};
    return run_moe("qsrt_packed_moe_layer", call, &r, ws, ws_bytes, static_cast<hipStream_t>(stream));
}

namespace {

struct LinearSpace {
    char* x;
    float *low, *part;
    int* exponents;  // of rows in f16 pieces
    int low_parts, parts, passes, groups, row_groups, product_chunks, pieces;
    bool grouped;  // layout of the rotated rows
    size_t bytes;
};

LinearSpace linear_space(void* ws, int64_t rows, int64_t k, int64_t n, int rates, int64_t adapters, int64_t rank, int cus) {
    LinearSpace s{};
    Carve c{static_cast<char*>(ws)};
    // Chunks of 8, 16, 32 and 64 rows, each up to two of them: more rows a wave share a decode, fewer leave more waves to
    // share the matrix (7168 x 7168 at K3: 12 rows 31 us in one chunk of 16, 39 in two of 8; 64 rows 50 in two of 32, 57 in
    // one of 64; 128 rows 66 in two of 64, 74 in four of 32; 96 rows 63 either way).  Beyond 128 a workgroup shares each
    // decode (192 rows: 78 us, 123 without; 128 rows: 74, without 66).
    s.groups = rows <= 8 ? 0 : rows <= 16 ? 1 : rows <= 64 ? 2 : 4;
    // Rows by 16 are rotated by a quarter of the waves, which costs a microsecond or two until the reads of the product
    // outweigh it (7168 x 7168: 24 rows 42.3 us as rows, 43.5 by 16; 32 rows 43.6 and 43.9; 48 rows 48.3 and 46.4; 64 rows
    // 50.2 and 49.7).
    s.grouped = rows > 48;
    s.passes = passes_of(rates);
    const int64_t nb = n / 128;
    const int strips = static_cast<int>(k / 32), limit = part_limit(rows * n * s.passes, strips);
    if (rows > 128) {
        const RowCut cut = cut_rows(rows, nb, strips, limit, cus);
        s.row_groups = cut.groups;
        s.parts = cut.parts;
    }
    const int64_t group_rows = s.row_groups ? 16 * kRowWaves * s.row_groups : chunk_rows_of(s.groups);
    const int64_t chunks = (rows + group_rows - 1) / group_rows;
    s.product_chunks = static_cast<int>(chunks);
    if (!s.row_groups)
        s.parts = cut_parts(static_cast<double>(chunks * nb), chunks * nb, strips, limit,
                            static_cast<int>(std::min(rows, group_rows)), cus);
    if (adapters) {
        constexpr int64_t kPart = 32 * kShrinkWaves * kShrinkSteps;
        s.low_parts = static_cast<int>((k + kPart - 1) / kPart);
        s.low = c.take<float>(s.low_parts * rows * rank);
    }
    s.pieces = s.row_groups ? kF16Pieces : kBf16Pieces;
    if (s.pieces == kF16Pieces) s.exponents = c.take<int>(rows);
    s.x = c.take<char>(rotated_bytes(rows, k, s.pieces));
    s.part = c.take<float>(static_cast<int64_t>(s.parts) * s.passes * rows * n);
    s.bytes = c.used;
    return s;
}

const char* linear_size_fault(const qsrt_packed_matrix* w, int64_t rows, int64_t adapters, int64_t rank) {
    if (const char* e = size_fault(w)) return e;
    if (rows < 0 || rows > (1 << 20)) return "at most 2^20 rows";
    if (adapters < 0 || adapters > kMaxAdapters) return "at most 8191 adapters";
    if (adapters && (rank < 16 || rank > kMaxRank || rank % 16)) return "adapters need a rank 16, 32 .. 128";
    if (!launch_fits(rows, w->rows, w->cols)) return "too many rows for this matrix";
    return nullptr;
}

}  // namespace

extern "C" size_t qsrt_adapter_linear_workspace_bytes(const qsrt_packed_matrix* w, int64_t rows, int64_t adapters,
                                                      int64_t rank) {
    int cus = 0;
    if (!w || rows == 0 || linear_size_fault(w, rows, adapters, rank) || current_cu_count(&cus)) return 0;
    return linear_space(nullptr, rows, w->rows, w->cols, w->rates, adapters, rank, cus).bytes;
}

extern "C" int qsrt_adapter_linear_plan(const qsrt_packed_matrix* w, int64_t rows, int64_t adapters, int64_t rank,
                                        int64_t* plan) {
    if (!w || !plan || rows == 0) return fail(kBadArgument, "qsrt_adapter_linear_plan: null pointer or no rows");
    if (const char* e = linear_size_fault(w, rows, adapters, rank)) return fail(kBadArgument, "qsrt_adapter_linear_plan: %s", e);
    int cus = 0;
    if (const int rc = current_cu_count(&cus)) return rc;
    const LinearSpace s = linear_space(nullptr, rows, w->rows, w->cols, w->rates, adapters, rank, cus);
    plan[0] = s.row_groups ? 16 * kRowWaves * s.row_groups : chunk_rows_of(s.groups);
    plan[1] = s.parts;
    plan[2] = static_cast<int64_t>(s.product_chunks) * (w->cols / 128) * s.parts;
    return kOk;
}

extern "C" int qsrt_adapter_linear(const qsrt_packed_matrix* w, const uint8_t* const* luts, const void* a, const void* b,
                                   const float* scale, int64_t adapters, int64_t rank, const void* x, int64_t x_ld,
                                   int dtype, int64_t rows, const int32_t* ids, void* out, int64_t out_ld, void* ws,
                                   size_t ws_bytes, void* stream_) {
    if (const char* e = matrix_fault(w, luts)) return fail(kBadArgument, "qsrt_adapter_linear: %s", e);
    if (const char* e = linear_size_fault(w, rows, adapters, rank)) return fail(kBadArgument, "qsrt_adapter_linear: %s", e);
    if (dtype != 0 && dtype != 1) return fail(kBadArgument, "qsrt_adapter_linear: dtype must be 0 (bf16) or 1 (f16)");
    if (adapters && (!a || !b || !scale || !ids || reinterpret_cast<uintptr_t>(a) % 16 || reinterpret_cast<uintptr_t>(b) % 16))
        return fail(kBadArgument, "qsrt_adapter_linear: adapters need 16-byte aligned a and b, scales and ids");
    if (rows == 0) return kOk;
    const int64_t k = w->rows, n = w->cols;
    if (const char* e = rows_fault(x, rows, x_ld, k, 16)) return fail(kBadArgument, "qsrt_adapter_linear: x: %s", e);
    if (const char* e = rows_fault(out, rows, out_ld, n, 8)) return fail(kBadArgument, "qsrt_adapter_linear: out: %s", e);
    int cus = 0;
    if (const int rc = current_cu_count(&cus)) return rc;
    const LinearSpace s = linear_space(ws, rows, k, n, w->rates, adapters, rank, cus);
    if (!ws || ws_bytes < s.bytes) return fail(kWorkspaceTooSmall, "qsrt_adapter_linear: needs %zu workspace bytes", s.bytes);
    hipStream_t stream = static_cast<hipStream_t>(stream_);

    RotateArgs ra{};
    ra.x = x;
    ra.ld = x_ld;
    ra.suh[0] = reinterpret_cast<const _Float16*>(w->suh);
    ra.x_div = 1;
    ra.out[0] = s.x;
    ra.rows = rows;
    ra.kb = static_cast<int>(k / 128);
    ra.nmat = 1;
    ra.layout = row_layout(ra.kb, s.grouped, s.pieces);
    ra.exponents = s.exponents;
    const bool scaled = s.pieces == kF16Pieces;
    const ExponentArgs ea{x, x_ld, ra.suh[0], static_cast<int>(k), scaled ? s.exponents : nullptr};
    ShrinkArgs sa{};
    sa.x = x;
    sa.ld = x_ld;
    sa.a = a;
    sa.ids = ids;
    sa.out = s.low;
    sa.rows = static_cast<int>(rows);
    sa.k = static_cast<int>(k);
    sa.adapters = static_cast<int>(adapters);
    sa.rank = static_cast<int>(rank);
    sa.parts = s.low_parts;
    const int tiles = adapters && rank % 32 == 0 ? 2 : 1;  // of 16 ranks a workgroup
    int sets = 1;                                          // of 16 rows
    int64_t shrinks = 0;
    if (adapters) {
        const auto blocks = [&](int q) { return (rows + 16 * q - 1) / (16 * q) * s.low_parts * (rank / (16 * tiles)); };
        // Beyond four workgroups a unit 32 rows share the reads of A (5120 x 1536, rank 64: 2048 rows 116 us with 32, 120 with
        // 16; 1024 rows 76 and 74; 512 rows 58 and 55); below, the adapters of a workgroup's rows are shared out.
        if (tiles == 2 && blocks(1) > 4 * cus) sets = 2;
        shrinks = blocks(sets);
        sa.shares = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(16, rows), 4 * cus / shrinks)));
        shrinks *= sa.shares;
    }
    const int64_t rotates = scaled                 ? rows
                            : ra.layout.row == 16 ? rotate_quads(ra)
                                                  : (rotate_waves(ra) + kShrinkWaves - 1) / kShrinkWaves;
    const dim3 pgrid(static_cast<unsigned>(shrinks + rotates)), pblock(64 * kShrinkWaves);
#define QSRT_PREPARE(T)                                                                                              \
    hipLaunchKernelGGL((sets == 2    ? prepare_rows_kernel<T, 2, 2>                                                   \
                        : tiles == 2 ? prepare_rows_kernel<T, 2, 1>                                                   \
                                     : prepare_rows_kernel<T, 1, 1>),                                                 \
                       pgrid, pblock, 0, stream, ra, ea, sa, static_cast<int>(shrinks))
    if (dtype == 0)
        QSRT_PREPARE(__bf16);
    else
        QSRT_PREPARE(_Float16);
#undef QSRT_PREPARE
    QSRT_HIP_TRY(hipGetLastError());
    if (scaled) {
        const dim3 rgrid(static_cast<unsigned>(rotate_quads(ra)));
        if (dtype == 0)
            hipLaunchKernelGGL(rotate_scaled_kernel<__bf16>, rgrid, dim3(256), 0, stream, ra);
        else
            hipLaunchKernelGGL(rotate_scaled_kernel<_Float16>, rgrid, dim3(256), 0, stream, ra);
        QSRT_HIP_TRY(hipGetLastError());
    }

    ProductArgs pa{};
    set_matrix(pa, 0, w);
    pa.x[0] = s.x;
    pa.x_div = 1;
    pa.layout = ra.layout;
    pa.max_chunks = s.product_chunks;
    pa.parts = s.parts;
    pa.part = s.part;
    pa.nmat = 1;
    pa.rows = static_cast<int>(rows);
    if (const int rc = launch_product(pa, s.groups, s.row_groups, w->rates, luts, cus, stream)) return rc;

    FinishArgs fa{};
    fa.part = s.part;
    fa.parts = s.parts * s.passes;
    fa.svh = static_cast<const _Float16*>(w->svh);
    fa.ids = adapters ? ids : nullptr;
    fa.low = s.low;
    fa.low_parts = s.low_parts;
    fa.adapters = static_cast<int>(adapters);
    fa.b = b;
    fa.scale = scale;
    fa.rank = static_cast<int>(rank);
    fa.out = out;
    fa.ld = out_ld;
    fa.rows = static_cast<int>(rows);
    fa.nb = static_cast<int>(n / 128);
    fa.exponents = scaled ? s.exponents : nullptr;
    const dim3 fgrid(static_cast<unsigned>((rows + 15) / 16 * fa.nb));
    if (dtype == 0)
        hipLaunchKernelGGL(finish_kernel<__bf16>, fgrid, dim3(256), 0, stream, fa);
    else
        hipLaunchKernelGGL(finish_kernel<_Float16>, fgrid, dim3(256), 0, stream, fa);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

// A gated feed-forward block in dense 16-bit weights, forward and backward, on the matrix cores (gfx950, wave64).
//
//   G = x W1^T, U = x W3^T, M = act(G, U), y = M W2^T            x [T, H], W1, W3 [I, H], W2 [H, I]
//   dM = dy W2, dG = dM act_g(G, U), dU = dM act_u(G, U)
//   dx = dG W1 + dU W3, dW1 = dG^T x, dW3 = dU^T x, dW2 = dy^T M
//
// Every product is a `tile_kernel`: sums of products of two operands that each lie with the summed index innermost
// (kRows) or outermost (kCols), so no operand is ever transposed in memory.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <type_traits>

#include "common.h"
#include "qsrt_amd.h"

namespace qsrt {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short i16x4 __attribute__((ext_vector_type(4)));

template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));
template <typename T>
using vec4 = T __attribute__((ext_vector_type(4)));

template <typename T>
__device__ __forceinline__ f32x4 multiply(vec8<T> a, vec8<T> b, f32x4 c) {
    if constexpr (__is_same(T, __bf16))
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

template <typename T>
constexpr bool kScaled = std::is_same<T, _Float16>::value;  // its rows between products, in the backward pass

// ---------------------------------------------------------------- what becomes of a product
// The activation in FP32: silu(g) u or 4 tanh(g/4) sigmoid(g) 25 tanh(u/25), and its derivatives.
__device__ __forceinline__ float activate(float g, float u, int activation) {
    const float s = 1.0f / (1.0f + expf(-g));
    return activation == 0 ? g * s * u : 4.0f * tanhf(0.25f * g) * s * (25.0f * tanhf(0.04f * u));
}
// What tanh and the sigmoid leave to 1 is a factor of situ's slopes, and is not taken as a difference: next to 1 nothing would
// be left of it (6% wrong at g = 32, 190% at u = 230).  With q = exp(-2|v|): 1 - tanh(v)^2 = 4 q / (1 + q)^2; 1 - sigmoid(g) =
// sigmoid(-g).  silu's slope adds it to 1.  tanh(v) is (1 - q) / (1 + q), or near 0 its series (the next term is 2^-24 of the
// value at 0.2).  Short, with the instructions' own reciprocal and power of two (1 ulp, and 2^-23 |2 v| of q for its argument): a
// tile's ending holds it for each of a thread's sums and waits for its instructions to come; with tanhf, expf and divisions in
// their place dM of 4096 rows of 7168 x 2048 takes 151 us, not 141.
struct Tanh {
    float value, slope;
};
__device__ __forceinline__ float exp_of(float v) { return __builtin_amdgcn_exp2f(1.44269504f * v); }
__device__ __forceinline__ Tanh tanh_of(float v, float q) {
    const float r = __builtin_amdgcn_rcpf(1.0f + q), w = v * v;
    const float near = 1.0f + w * (-1.0f / 3 + w * (2.0f / 15 + w * (-17.0f / 315)));
    return {fabsf(v) < 0.2f ? v * near : copysignf((1.0f - q) * r, v), 4.0f * q * r * r};
}
__device__ __forceinline__ void activate_with_slopes(float g, float u, int activation, float& m, float& by_g, float& by_u) {
    if (activation == 0) {
        const float s = 1.0f / (1.0f + expf(-g));
        by_u = g * s;
        m = by_u * u;
        by_g = u * (s * (1.0f + g * (1.0f - s)));
    } else {
        const float q = exp_of(-0.5f * fabsf(g)), more = __builtin_amdgcn_rcpf(1.0f + q * q), less = q * q * more;
        const float s = g >= 0.f ? more : less, rest = g >= 0.f ? less : more;  // sigmoid(g), sigmoid(-g)
        const Tanh a = tanh_of(0.25f * g, q), up = tanh_of(0.04f * u, exp_of(-0.08f * fabsf(u)));
        const float b = 25.0f * up.value, f = 4.0f * a.value * s;
        m = f * b;
        by_g = b * (a.slope * s + f * rest);
        by_u = f * up.slope;
    }
}

enum Ending { kStore, kActivate, kSlopes };

// A row between two products goes on in 16 bits, as the matrix cores take it: rounded once, or as two pieces (the nearest
// 16-bit value and the nearest of what is left; `pieces_of` says when).
struct Pieces {
    void *hi, *lo;  // lo null: one
    void* plain;    // where the rows go as they are, beside the scaled ones; or null
};

// What scaled rows between products are multiplied by: dG and dU, and M.  kStore: `rows`, what the sums are.
struct Scales {
    float rows, middle;
};

struct Finish {
    // kStore: the sums, rounded once
    void* out;
    int64_t ld;
    // the others: rows [rows, inter]
    int activation;
    float *pre_g, *pre_u;     // kActivate: G and U out, or null; kSlopes: in
    Pieces middle, dg, du;    // kActivate: middle; kSlopes: all
    // f16 in the backward pass, or null
    const f32x4* bounds;  // kSlopes: of `bounds_kernel`
    float* unscale;       // kSlopes: one over each of the scales, out; kStore: the one for these sums
};

template <typename T>
__device__ __forceinline__ void store_pieces(const Pieces& to, int64_t at, f32x4 v, float scale) {
    if constexpr (kScaled<T>) {
        if (to.plain) *reinterpret_cast<vec4<T>*>(static_cast<T*>(to.plain) + at) = __builtin_convertvector(v, vec4<T>);
        v *= scale;
    }
    const vec4<T> hi = __builtin_convertvector(v, vec4<T>);
    *reinterpret_cast<vec4<T>*>(static_cast<T*>(to.hi) + at) = hi;
    if (to.lo) {
        f32x4 left = v - __builtin_convertvector(hi, f32x4);
#pragma unroll
        for (int r = 0; r < 4; ++r) left[r] = __builtin_isfinite(static_cast<float>(hi[r])) ? left[r] : 0.f;
        *reinterpret_cast<vec4<T>*>(static_cast<T*>(to.lo) + at) = __builtin_convertvector(left, vec4<T>);
    }
}

// Four neighbouring columns of one row: v the sums, u the second matrix's.
template <typename T, Ending kEnding>
__device__ __forceinline__ void finish(const Finish& f, int64_t row, int64_t col, const f32x4& v, const f32x4& u, const Scales& by) {
    const int64_t at = row * f.ld + col;
    if constexpr (kEnding == kStore) {
        *reinterpret_cast<vec4<T>*>(static_cast<T*>(f.out) + at) = __builtin_convertvector(kScaled<T> ? v * by.rows : v, vec4<T>);
    } else if constexpr (kEnding == kActivate) {
        if (f.pre_g) {
            *reinterpret_cast<f32x4*>(f.pre_g + at) = v;
            *reinterpret_cast<f32x4*>(f.pre_u + at) = u;
        }
        f32x4 m;
#pragma unroll
        for (int r = 0; r < 4; ++r) m[r] = activate(v[r], u[r], f.activation);
        store_pieces<T>(f.middle, at, m, 1.f);
    } else {
        const f32x4 g = *reinterpret_cast<const f32x4*>(f.pre_g + at), up = *reinterpret_cast<const f32x4*>(f.pre_u + at);
        f32x4 m, dg, du;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float by_g, by_u, mid;
            activate_with_slopes(g[r], up[r], f.activation, mid, by_g, by_u);
            m[r] = mid;
            dg[r] = v[r] * by_g;
            du[r] = v[r] * by_u;
        }
        store_pieces<T>(f.middle, at, m, by.middle);
        store_pieces<T>(f.dg, at, dg, by.rows);
        store_pieces<T>(f.du, at, du, by.rows);
    }
}

// The steps of f16 stop shrinking at 2^-24: of gradients of 1e-5 seven bits would be left, in two pieces no more.  So in the
// backward pass f16 rows between products are scaled by powers of two, dG and dU by one, M by another, which are divided out of
// the FP32 sums again.  Which: what takes a bound on all of them to 2^14 .. 2^15, so that none ends at 65504 for being scaled,
// but never less than 1.  The bound of M is its largest value; |dG| and |dU| are at most
//   max over rows |dy| * sqrt(H) max |W2| * the largest slope
// as no column of W2 is longer than sqrt(H) max |W2|.  That is some 2^6 to 2^12 above their usual size, of the 2^29 from 2^15 down
// to the least f16 that has all its bits.  Values that are not finite do not count.
//
// The forward pass does without: its bound would need gate and up read once more.  `bounds_kernel` is bound by memory (dy, W2, G
// and U of 4096 rows of 7168 x 2048, 154 MB, in 33 to 37 us, 4.2 to 4.7 TB/s), of few rows by its loads' way (27 rows of 5120 x
// 1536: 11).  4096 rows with gradients take 978 to 987 us, where they took 953 to 961 unscaled, 500 of 5120 x 1536 132 for 118.
constexpr int kBoundGroups = 256, kBoundWaves = 16;
struct BoundArgs {
    const void *dy, *down;
    int64_t dy_ld, down_ld, tokens, hidden, inter;
    int activation;
    const float* pre;
    f32x4* bounds;  // a workgroup's: sqrt(H) |dy| of a row, |W2|, slopes, |M|
};

__device__ __forceinline__ f32x4 most_of(f32x4 v) {  // of the wave, in each lane
#pragma unroll
    for (int apart = 32; apart > 0; apart >>= 1)
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = fmaxf(v[i], __shfl_xor(v[i], apart));
    return v;
}

__global__ __launch_bounds__(64 * kBoundWaves) void bounds_kernel(const BoundArgs p) {
    __shared__ f32x4 room[kBoundWaves];
    typedef vec8<_Float16> f16x8;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t first = blockIdx.x * kBoundWaves + wave, waves = kBoundGroups * kBoundWaves;
    f32x4 most = {};
    const auto see = [&](int i, float v) { most[i] = v <= FLT_MAX ? fmaxf(most[i], v) : most[i]; };
    // Four loads a lane on their way at a time; those past an end repeat the last.
    for (int64_t row = first; row < p.tokens; row += waves) {
        const _Float16* at = static_cast<const _Float16*>(p.dy) + row * p.dy_ld;
        float sum = 0.f;
        for (int64_t c = 8 * lane; c < p.hidden; c += 4 * 512) {
            f16x8 v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = *reinterpret_cast<const f16x8*>(at + min(c + 512 * q, p.hidden - 8));
#pragma unroll
            for (int q = 0; q < 4; ++q)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float f = static_cast<float>(v[q][i]);
                    sum += c + 512 * q < p.hidden && fabsf(f) <= FLT_MAX ? f * f : 0.f;
                }
        }
#pragma unroll
        for (int apart = 32; apart > 0; apart >>= 1) sum += __shfl_xor(sum, apart);
        see(0, sqrtf(sum * static_cast<float>(p.hidden)));
    }
    const uint32_t thread = first * 64 + lane, threads = waves * 64;
    const uint32_t across = static_cast<uint32_t>(p.inter / 8), chunks = static_cast<uint32_t>(p.hidden) * across;  // 2^31 at most
    for (uint32_t n = thread; n < chunks; n += 4 * threads) {
        f16x8 v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t k = min(n + q * threads, chunks - 1), row = k / across;
            v[q] = *reinterpret_cast<const f16x8*>(static_cast<const _Float16*>(p.down) + row * p.down_ld + 8 * (k - row * across));
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int i = 0; i < 8; ++i) see(1, fabsf(static_cast<float>(v[q][i])));
    }
    const int64_t plane = p.tokens * p.inter, step = static_cast<int64_t>(threads) * 4;
    for (int64_t n = static_cast<int64_t>(thread) * 4; n < plane; n += 2 * step) {
        f32x4 g[2], u[2];
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const int64_t at = min(n + q * step, plane - 4);
            g[q] = *reinterpret_cast<const f32x4*>(p.pre + at);
            u[q] = *reinterpret_cast<const f32x4*>(p.pre + plane + at);
        }
#pragma unroll
        for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float m, by_g, by_u;
                activate_with_slopes(g[q][i], u[q][i], p.activation, m, by_g, by_u);
                see(2, fabsf(by_g));
                see(2, fabsf(by_u));
                see(3, fabsf(m));
            }
    }
    most = most_of(most);
    if (lane == 0) room[wave] = most;
    __syncthreads();
    if (wave > 0) return;
    most = most_of(room[lane % kBoundWaves]);
    if (lane == 0) p.bounds[blockIdx.x] = most;
}

// The power of two, 1 at the least, that takes `bound` to 2^14 .. 2^15.
__device__ __forceinline__ float scale_to(float bound) {
    const int exponent = static_cast<int>(__builtin_bit_cast(uint32_t, bound) >> 23) - 127;  // (bound is not negative)
    const int up = min(max(14 - exponent, 0), 60);
    return __builtin_bit_cast(float, static_cast<uint32_t>(127 + up) << 23);
}

// For all threads of a workgroup, at its end; `first`: of the launch.
template <typename T, Ending kEnding>
__device__ __forceinline__ Scales scales_of(const Finish& f, bool first) {
    Scales by = {1.f, 1.f};
    if constexpr (kScaled<T> && kEnding == kStore) {
        if (f.unscale) by.rows = *f.unscale;
    } else if constexpr (kScaled<T> && kEnding == kSlopes) {
        if (f.bounds) {
            f32x4 most = {};
#pragma unroll
            for (int q = 0; q < kBoundGroups; q += 64) {
                const f32x4 v = f.bounds[q + (threadIdx.x & 63)];
#pragma unroll
                for (int i = 0; i < 4; ++i) most[i] = fmaxf(most[i], v[i]);
            }
            most = most_of(most);
            by = {scale_to(most[0] * most[1] * most[2]), scale_to(most[3])};
            if (first && threadIdx.x == 0) f.unscale[0] = 1.f / by.rows, f.unscale[1] = 1.f / by.middle;
        }
    }
    return by;
}

// ---------------------------------------------------------------- the product
enum Layout { kRows, kCols };

constexpr int kDepth = 64;  // of the summed index in a stage
constexpr int kSums = 4;    // products that one result adds up, at the most

struct Product {
    const void* a[kSums];
    const void* b[kSums];
    const void* b2;  // of two matrices side by side (kActivate)
    int64_t lda, ldb;
    int64_t m, n, k;
    int sums;
    int tiles_m, tiles_n;
    Finish finish;
};

constexpr int kProducts = 3;
template <int kMost>
struct TileArgs {
    Product product[kMost];
    int products;
    int parts;       // of the summed axis; > 1: sums go to `partial` [part][1 or 2][m][n]
    float* partial;
};
template <Layout kA>
using ArgsOf = TileArgs<kA == kCols ? kProducts : 1>;  // the weights' gradients go together

// f of every number from kFrom on, before kTo, as a constant.
template <int kFrom, int kTo, typename F>
__device__ __forceinline__ void count(const F& f) {
    if constexpr (kFrom < kTo) {
        f(std::integral_constant<int, kFrom>{});
        count<kFrom + 1, kTo>(f);
    }
}

// 16 bytes a lane from a buffer straight to LDS: lane l's go to `lds` + 16 l.  Written in assembly because the compiler,
// which cannot see that a stage is written while another is read, waits for all of them before any read from LDS.  Nothing
// comes back in registers; `wait_and_meet` is the wait.  m0, the LDS address, is named as written: the compiler remarks that it
// never allocates it, but it does merge its own writes of it.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
template <int kAt>
__device__ __forceinline__ void to_lds(u32x4 from, uint32_t offset, uint32_t lds) {
    asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(offset), "s"(from), "s"(lds),
                 "n"(kAt)
                 : "memory", "scc", "m0");
}
#pragma clang diagnostic pop

// All but the wave's last `kLeft` loads have landed, its reads from LDS are done, and so are the other waves'.
template <int kLeft>
__device__ __forceinline__ void wait_and_meet() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(kLeft) : "memory");
}

constexpr uint32_t kNowhere = 0x80000000u;  // past the end of every buffer here: reads zero

// A stage of one operand in LDS: kSize indices by 64 of the summed index, in 16-byte chunks of 8.
//   kRows: an index's 8 chunks in a row of 128 bytes, chunk c at place c ^ (index & 7)
//   kCols: a summed index's kSize / 8 chunks in a row, chunk c at place c ^ 2 f(k), f(k) = (k & 3) | (k >> 3 & 1) << 2
// so that a quarter of the wave's 16-byte reads, or half of its transposing 8-byte reads, hit distinct banks.  Loads to LDS
// write 16 bytes a lane in lane order, so it is the address read that is permuted.
template <Layout kLayout, int kSize, int kWaves>
struct Loader {
    static constexpr int kBytes = kSize * kDepth * 2;
    static constexpr int kLoads = kBytes / 1024 / kWaves;  // a wave's
    static constexpr int kRowBytes = kLayout == kRows ? 128 : 2 * kSize;
    static constexpr int kChunks = kRowBytes / 16;
    static_assert(kBytes % (1024 * kWaves) == 0 && kLoads >= 1, "a wave's loads are whole");
    uint32_t offset[kLoads];
    int chunk;  // kRows: of the summed index

    __device__ __forceinline__ void init(int64_t ld, int wave, int lane) {
#pragma unroll
        for (int q = 0; q < kLoads; ++q) {
            const int row = (q * kWaves + wave) * (1024 / kRowBytes) + lane / kChunks, place = lane % kChunks;
            int c;
            if constexpr (kLayout == kRows) {
                c = place ^ (row & 7);
                chunk = c;  // 8 rows a load: the same in all
            } else {
                c = place ^ (((row & 3) | (row >> 3 & 1) << 2) << 1);
            }
            offset[q] = (static_cast<uint32_t>(row) * static_cast<uint32_t>(ld) + 8 * c) * 2;
        }
    }

    // The wave's q-th load of a stage from `from`, of which `depth` summed indices are left, to kAt behind `lds` (its place of
    // the wave's first load).
    template <int kAt, int q>
    __device__ __forceinline__ void load(u32x4 from, int depth, uint32_t lds) const {
        const bool past = kLayout == kRows && 8 * chunk >= depth;
        to_lds<kAt + q * kWaves * 1024>(from, past ? kNowhere : offset[q], lds);
    }
};

// Where an operand's next stage lies: a buffer resource that ends with the last of its values, so that reads past the tile's
// end of either index are zero or feed results that are not stored.  Kept as the instruction takes it: a small tile's stage is
// short enough for scalar instructions to count.
template <Layout kLayout>
struct Feed {
    u32x4 buffer;
    uint32_t ld, span;  // bytes between rows; kRows: in the tile's rows but the last, kCols: of a row
    __device__ __forceinline__ void init(int64_t stride, int64_t size, int tile) {
        ld = static_cast<uint32_t>(stride) * 2;
        const uint32_t n = static_cast<uint32_t>(min(size, static_cast<int64_t>(tile)));
        span = kLayout == kRows ? (n - 1) * ld : n * 2;
        buffer[3] = 0x00020000;
    }
    __device__ __forceinline__ void end(int depth) {  // nothing at depth 0 and below
        const int bytes = kLayout == kRows ? static_cast<int>(span) + 2 * depth
                                           : (min(depth, kDepth) - 1) * static_cast<int>(ld) + static_cast<int>(span);
        buffer[2] = static_cast<uint32_t>(max(bytes, 0));
    }
    __device__ __forceinline__ void enter(const char* p, int depth) {
        const uint64_t at = reinterpret_cast<uint64_t>(p);
        buffer[0] = static_cast<uint32_t>(at);
        buffer[1] = static_cast<uint32_t>(at >> 32);
        end(depth);
    }
    __device__ __forceinline__ void advance(int depth) {
        const uint64_t at = (static_cast<uint64_t>(buffer[1]) << 32 | buffer[0]) +
                            (kLayout == kRows ? 2 * kDepth : static_cast<uint64_t>(ld) * kDepth);
        buffer[0] = static_cast<uint32_t>(at);
        buffer[1] = static_cast<uint32_t>(at >> 32);
        end(depth);
    }
};

// The lane's part of a 16 x 32 fragment: index lane % 16, eight summed indices from 8 (lane / 16).
template <Layout kLayout, int kSize, typename T>
struct Reader {
    uint32_t base[kLayout == kRows ? 2 : 1];
    int f;
    __device__ __forceinline__ void init(int lane) {
        if constexpr (kLayout == kRows) {
            base[0] = (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
            base[1] = base[0] ^ 64;
        } else {
            const int a = lane & 15;
            base[0] = (8 * (lane >> 4) + (a >> 2)) * (2 * kSize) + (a & 3) * 8;
            f = (a >> 2) | (lane >> 4 & 1) << 2;
        }
    }
    // `first`: a multiple of 16; `kk`: which 32 of the stage's 64
    __device__ __forceinline__ vec8<T> read(const char* lds, int first, int kk) const {
        if constexpr (kLayout == kRows) {
            return *reinterpret_cast<const vec8<T>*>(lds + first * 128 + base[kk]);
        } else {
            typedef __attribute__((address_space(3))) i16x4 lds_i16x4;
            const char* at = lds + kk * 32 * (2 * kSize) + (((first >> 4) ^ f) << 5) + base[0];
            const i16x4 half[2] = {__builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)at),
                                   __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_i16x4*)(at + 4 * 2 * kSize))};
            vec8<T> v;
            __builtin_memcpy(&v, half, sizeof(v));
            return v;
        }
    }
};

// Workgroup q of n runs on XCD q % 8: every XCD takes a run of the tile order.
__device__ __forceinline__ int xcd_slot(int q, int n) {
    const int x = q % 8, per = n / 8, rem = n % 8;
    return x * per + (x < rem ? x : rem) + q / 8;
}

// One tile of kM rows (of a) by kN columns (of b; with kActivate half of them of b, half of b2) a workgroup of kWavesM x
// kWavesN waves, kStages stages in LDS.  The first operand of the matrix instruction is b: a lane then holds four
// neighbouring columns of one row.
//
// Many rows are bound by the operands' way from L2 to LDS, with the matrix cores close behind: a stage of a 256 x 256 tile
// brings 64 KB to each compute unit in 1.66 us, 10 TB/s on the chip, 79% of it out of L2.  4096 rows of 7168 x 2048 take 187
// to 202 us for gate and up (1.2 to 1.3 PFLOP/s; 164 with the loads alone, 148 with the products and their reads from LDS
// alone, at 1.8 GHz), 110 for down, 196 for dx, 313 for the weights' gradients, and dM, in tiles of 128 x 256, 144.  64 deep:
// stages of 32 in rings of four or five cost 10%, having twice the barriers.  Eight waves of 128 x 64: four of 128 x 128 have
// nobody to load while they wait (25% slower), 32 x 32 x 16 instructions 5%.
template <typename T, Layout kA, Layout kB, Ending kEnding, int kM, int kN, int kWavesM, int kWavesN, int kStages>
__global__ __launch_bounds__(64 * kWavesM * kWavesN) void tile_kernel(const ArgsOf<kA> args) {
    constexpr int kWaves = kWavesM * kWavesN;
    constexpr bool kDual = kEnding == kActivate;
    constexpr int kNb = kDual ? kN / 2 : kN;  // of one matrix of b
    constexpr int kWm = kM / kWavesM, kWn = kN / kWavesN, kI = kWm / 16, kJ = kWn / 16, kHalf = kDual ? kJ / 2 : kJ;
    typedef Loader<kA, kM, kWaves> LoaderA;
    typedef Loader<kB, kNb, kWaves> LoaderB;
    constexpr int kStageBytes = LoaderA::kBytes + (kDual ? 2 : 1) * LoaderB::kBytes;
    constexpr int kStageLoads = LoaderA::kLoads + (kDual ? 2 : 1) * LoaderB::kLoads;
    extern __shared__ char lds[];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    int tile = xcd_slot(blockIdx.x, gridDim.x), which = 0, part = 0;
    const int parts = kA == kCols ? 1 : args.parts;  // the weights' gradients are not cut
    if constexpr (kA == kCols)
        for (; which + 1 < args.products; ++which) {
            const int tiles = args.product[which].tiles_m * args.product[which].tiles_n;
            if (tile < tiles) break;
            tile -= tiles;
        }
    const Product& p = args.product[kA == kCols ? which : 0];
    if (parts > 1) {
        const int tiles = p.tiles_m * p.tiles_n;
        part = tile / tiles;
        tile %= tiles;
    }
    // tiles in bands of four of m: the workgroups at work on an XCD at a time share operands in its L2 (bands of six: 1% less at
    // 4096 rows of 7168 x 2048 with gradients, 2% more at 4096 of 2056 x 1400; of 16 1% more)
    constexpr int kBand = 4;
    const int band = tile / (kBand * p.tiles_n), in_band = tile % (kBand * p.tiles_n);
    const int high = min(kBand, p.tiles_m - band * kBand);
    const int64_t m0 = static_cast<int64_t>(band * kBand + in_band % high) * kM, n0 = static_cast<int64_t>(in_band / high) * kNb;

    const int k = static_cast<int>(p.k), per = (k + kDepth - 1) / kDepth, stages = per * p.sums;
    const int begin = static_cast<int>(static_cast<int64_t>(stages) * part / parts);
    const int end = static_cast<int>(static_cast<int64_t>(stages) * (part + 1) / parts);

    LoaderA la;
    LoaderB lb;
    la.init(p.lda, wave, lane);
    lb.init(p.ldb, wave, lane);
    Reader<kA, kM, T> ra;
    Reader<kB, kNb, T> rb;
    ra.init(lane);
    rb.init(lane);

    // The stage to be loaded next.  Neighbouring tiles walk the sum from stages of their own, around its end: rows whose
    // distance has a high power of two would come from the same few channels of the L2 in every workgroup at once (4096 rows of
    // 7168 x 2048 with gradients: 943 us from the first stage, 933 so).  Behind the last stage come empty ones, so that what
    // is on its way is always the same number of loads.
    Feed<kA> fa;
    Feed<kB> fb, fb2;
    fa.init(p.lda, p.m - m0, kM);
    fb.init(p.ldb, p.n - n0, kNb);
    if constexpr (kDual) fb2 = fb;
    int coming = begin + tile % 8 % (end - begin), remaining = end - begin, run = 0, left, sum, depth;
    uint32_t to = 0;
    const auto enter = [&]() {  // the operands of `sum`, `depth` before their end
        const int64_t k0 = k - depth;
        const int64_t at = kB == kRows ? n0 * p.ldb + k0 : k0 * p.ldb + n0;
        fa.enter(static_cast<const char*>(p.a[sum]) + 2 * (kA == kRows ? m0 * p.lda + k0 : k0 * p.lda + m0), depth);
        fb.enter(static_cast<const char*>(p.b[sum]) + 2 * at, depth);
        if constexpr (kDual) fb2.enter(static_cast<const char*>(p.b2) + 2 * at, depth);
    };
    const uint32_t own = 1024 * static_cast<uint32_t>(wave);
    const auto load_one = [&](auto number) {  // of the wave's loads of a stage
        constexpr int q = decltype(number)::value, qb = q - LoaderA::kLoads, qb2 = qb - LoaderB::kLoads;
        if constexpr (qb < 0)
            la.template load<0, q>(fa.buffer, depth, to + own);
        else if constexpr (qb2 < 0)
            lb.template load<LoaderA::kBytes, qb>(fb.buffer, depth, to + own);
        else
            lb.template load<LoaderA::kBytes + LoaderB::kBytes, qb2>(fb2.buffer, depth, to + own);
    };
    const auto enter_run = [&]() {  // stages of one sum, one behind another
        remaining -= run;
        coming += run;
        if (remaining == 0) {
            depth = 0;
            fa.end(0);
            fb.end(0);
            if constexpr (kDual) fb2.end(0);
            left = 1 << 30;
            return;
        }
        if (coming == end) coming = begin;
        sum = coming / per;
        depth = k - (coming - sum * per) * kDepth;
        left = run = min(min(per * (sum + 1), end) - coming, remaining);
        enter();
    };
    const auto loaded = [&]() {
        to = to + kStageBytes == kStages * kStageBytes ? 0 : to + kStageBytes;
        depth = max(depth - kDepth, 0);  // times the bytes between rows: five empty stages of rows far apart would pass 2^31
        fa.advance(depth);
        fb.advance(depth);
        if constexpr (kDual) fb2.advance(depth);
        if (--left == 0) enter_run();
    };
    const auto load = [&]() {
        count<0, kStageLoads>(load_one);
        loaded();
    };

    const int wm = wave / kWavesN * kWm, wn = wave % kWavesN * (kDual ? kWn / 2 : kWn);
    f32x4 acc[kI][kJ];
#pragma unroll
    for (int i = 0; i < kI; ++i)
#pragma unroll
        for (int j = 0; j < kJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const auto read_a = [&](const char* at, int i, int kk) { return ra.read(at, wm + 16 * i, kk); };
    const auto read_b = [&](const char* at, int j, int kk) {
        return rb.read(at + LoaderA::kBytes + (j < kHalf ? 0 : LoaderB::kBytes), wn + 16 * (j % kHalf), kk);
    };

    const auto after = [](uint32_t at) { return at + kStageBytes == kStages * kStageBytes ? 0 : at + kStageBytes; };

    enter_run();
    uint32_t now = 0;
    if constexpr (kI >= 4) {
        // A stage is 2 kI steps of kJ products: fragment i of a by all of b.  Before a step's products go the reads of what
        // is used kI steps later (a's fragments in place of those just used, b's in turn), from the middle of the second
        // half on those of the next stage: then every wave has read all of this one, the next has landed, and its buffer
        // takes the one kStages on.  One wait and barrier a stage, with products before and behind it.
        vec8<T> a[kI], b[2][kJ];
#pragma unroll
        for (int s = 0; s < kStages; ++s) load();
        wait_and_meet<kStageLoads*(kStages - 1)>();
#pragma unroll
        for (int j = 0; j < kJ; ++j) b[0][j] = read_b(lds, j, 0);
#pragma unroll
        for (int i = 0; i < kI; ++i) a[i] = read_a(lds, i, 0);
        for (int s = begin; s < end; ++s) {
            const char *at = lds + now, *next = lds + (now = after(now));
#pragma unroll
            for (int i = 0; i < kI; ++i) {
                if (i > 0) a[i - 1] = read_a(at, i - 1, 1);
#pragma unroll
                for (int j = i * kJ / (kI - 1); j < (i + 1) * kJ / (kI - 1) && j < kJ; ++j) b[1][j] = read_b(at, j, 1);
#pragma unroll
                for (int j = 0; j < kJ; ++j) acc[i][j] = multiply<T>(b[0][j], a[i], acc[i][j]);
                __builtin_amdgcn_sched_barrier(0);
            }
            count<0, kI>([&](auto step) {
                constexpr int i = decltype(step)::value;
                if (i == 0) a[kI - 1] = read_a(at, kI - 1, 1);
                if (i >= 2) {
                    if (i == 2) a[0] = read_a(next, 0, 0);
                    a[i - 1] = read_a(next, i - 1, 0);
#pragma unroll
                    for (int j = (i - 2) * kJ / (kI - 2); j < (i - 1) * kJ / (kI - 2); ++j) b[0][j] = read_b(next, j, 0);
                }
#pragma unroll
                for (int j = 0; j < kJ; ++j) acc[i][j] = multiply<T>(b[1][j], a[i], acc[i][j]);
                if constexpr (i >= 2) count<(i - 2) * kStageLoads / (kI - 2), (i - 1) * kStageLoads / (kI - 2)>(load_one);
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (i == 1) {
                    wait_and_meet<kStageLoads*(kStages - 2)>();
                    __builtin_amdgcn_sched_barrier(0);
                }
            });
            loaded();
            a[kI - 1] = read_a(next, kI - 1, 0);
        }
    } else {
        // few rows: bound by reading b, with a stage on its way less
#pragma unroll
        for (int s = 0; s < kStages - 1; ++s) load();
        for (int s = begin; s < end; ++s) {
            wait_and_meet<kStageLoads*(kStages - 2)>();  // this stage has landed, the one before has been read
            load();
            const char* at = lds + now;
            now = after(now);
            vec8<T> a[2][kI], b[2][kJ];
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
                for (int j = 0; j < kJ; ++j) b[kk][j] = read_b(at, j, kk);
#pragma unroll
                for (int i = 0; i < kI; ++i) a[kk][i] = read_a(at, i, kk);
            }
#pragma unroll
            for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                for (int i = 0; i < kI; ++i)
#pragma unroll
                    for (int j = 0; j < kJ; ++j) acc[i][j] = multiply<T>(b[kk][j], a[kk][i], acc[i][j]);
        }
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no load to LDS outlives the workgroup

    Scales by = {1.f, 1.f};
    if (parts == 1) by = scales_of<T, kEnding>(p.finish, blockIdx.x == 0);
    const int64_t row0 = m0 + wm + (lane & 15), col0 = n0 + wn + 4 * (lane >> 4);
#pragma unroll
    for (int i = 0; i < kI; ++i) {
        const int64_t row = row0 + 16 * i;
        if (kEnding == kStore && parts == 1) {
            // Two tiles' columns exchanged between neighbouring groups of 16 lanes: a lane then stores eight in a row of one.
            const int odd = lane >> 4 & 1;
            const int64_t col = n0 + wn + 8 * (lane >> 5) + 16 * odd;
#pragma unroll
            for (int j = 0; j + 1 < kJ; j += 2) {
                typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
                if constexpr (kScaled<T>) acc[i][j] *= by.rows, acc[i][j + 1] *= by.rows;
                const u32x2 a = __builtin_bit_cast(u32x2, __builtin_convertvector(acc[i][j], vec4<T>));
                const u32x2 b = __builtin_bit_cast(u32x2, __builtin_convertvector(acc[i][j + 1], vec4<T>));
                const auto low = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
                const auto high = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
                const u32x4 v = {low[0], high[0], low[1], high[1]};
                if (row < p.m && col + 16 * j < p.n)  // n is a multiple of 8
                    *reinterpret_cast<u32x4*>(static_cast<T*>(p.finish.out) + row * p.finish.ld + col + 16 * j) = v;
            }
            continue;
        }
        if (row >= p.m) continue;
#pragma unroll
        for (int j = 0; j < kHalf; ++j) {
            const int64_t col = col0 + 16 * j;
            if (col >= p.n) continue;
            if (parts > 1) {
                float* to = args.partial + (part * (kDual ? 2 : 1) * p.m + row) * p.n + col;
                *reinterpret_cast<f32x4*>(to) = acc[i][j];
                if constexpr (kDual) *reinterpret_cast<f32x4*>(to + p.m * p.n) = acc[i][kHalf + j];
            } else {
                finish<T, kEnding>(p.finish, row, col, acc[i][j], acc[i][kDual ? kHalf + j : j], by);
            }
        }
    }
}

// Adds the parts up, in their order, four columns a thread.  Bound by its launch and round trips (45 rows of 1536 in eight parts
// 3.2 to 4.2 us, 500 in two 4.7), of many rows by memory (4096 rows of 2048 in two parts, with G and U read and three rows
// written: 184 MB in 31).
template <typename T, Ending kEnding>
__global__ __launch_bounds__(256) void join_kernel(const float* __restrict__ partial, int parts, int64_t m, int64_t n, const Finish f) {
    constexpr int kPlanes = kEnding == kActivate ? 2 : 1;
    const Scales by = scales_of<T, kEnding>(f, blockIdx.x == 0);
    const int64_t at = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4;
    if (at >= m * n) return;
    f32x4 sum[2] = {};
    const int64_t plane = m * n;
    int q = 0;
    // eight parts' loads go out together: few columns leave nothing else to hide them behind
    for (; q + 8 <= parts; q += 8) {
        f32x4 v[8][kPlanes];
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int h = 0; h < kPlanes; ++h) v[i][h] = *reinterpret_cast<const f32x4*>(partial + ((q + i) * kPlanes + h) * plane + at);
#pragma unroll
        for (int i = 0; i < 8; ++i)
#pragma unroll
            for (int h = 0; h < kPlanes; ++h) sum[h] += v[i][h];
    }
    for (; q < parts; ++q)
#pragma unroll
        for (int h = 0; h < kPlanes; ++h) sum[h] += *reinterpret_cast<const f32x4*>(partial + (q * kPlanes + h) * plane + at);
    finish<T, kEnding>(f, at / n, at % n, sum[0], sum[1], by);
}

// ---------------------------------------------------------------- a few rows
// Up to 16 rows of activations by a matrix whose rows lie with the summed index innermost: bound by reading the matrix once.
// A workgroup takes 16 of its rows (kActivate: eight of gate and the same eight of up), its waves a part of the sum each,
// weights straight to registers in the matrix instruction's order, the next kAhead steps of 32 always on their way; the parts
// are added in LDS, in wave order, so there is no second kernel.
//
// 7168 x 2048, one row: both products in 21.5 us, 4.1 TB/s of weights (a large copy moves 4.6).  Eight waves a workgroup for
// gate and up, whose workgroups are fewer, four for down, four steps ahead (waves, steps of the one, then the other; us at 1
// row of 7168 x 2048, 5120 x 1536, 2048 x 1024): 8, 4, 4, 4: 21.5, 15.9, 8.7; 8, 4, 8, 4: 22.0, 17.3, 8.5; 8, 7, 4, 6: 24.2,
// 17.9, 11.0; 16, 4, 8, 4: 23.0, 18.9, 8.7.  More steps ahead leave fewer waves room and reach past the end of short sums.
struct RowsArgs {
    const void* a[2];  // rows of activations; kStore: in two pieces
    const void *b, *b2;
    int64_t lda, ldb;
    int m, n, k;
    Finish finish;
};

template <typename T, Ending kEnding, int kWaves, int kAhead>
__global__ __launch_bounds__(64 * kWaves) void rows_kernel(const RowsArgs p) {
    __shared__ f32x4 sums[kWaves][64];
    constexpr bool kDual = kEnding == kActivate;
    constexpr int kPieces = kDual ? 1 : 2;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int r = lane & 15, g = lane >> 4, n0 = blockIdx.x * (kDual ? 8 : 16);
    // rows past the end repeat the last; not stored
    const T* weights = kDual ? static_cast<const T*>(r < 8 ? p.b : p.b2) + (n0 + (r & 7)) * p.ldb
                             : static_cast<const T*>(p.b) + min(n0 + r, p.n - 1) * p.ldb;
    const int64_t row = min(r, p.m - 1) * p.lda;
    const int steps = (p.k + 31) / 32, begin = steps * wave / kWaves, end = steps * (wave + 1) / kWaves;
    f32x4 acc = {};
    vec8<T> w[kAhead], x[kPieces][kAhead];
    const auto fetch = [&](int j, int step) {
        const int at = min(step * 32 + 8 * g, p.k - 8);
        w[j] = *reinterpret_cast<const vec8<T>*>(weights + at);
#pragma unroll
        for (int q = 0; q < kPieces; ++q) x[q][j] = *reinterpret_cast<const vec8<T>*>(static_cast<const T*>(p.a[q]) + row + at);
    };
    if (begin < end) {
#pragma unroll
        for (int j = 0; j < kAhead; ++j) fetch(j, min(begin + j, end - 1));
        int s = begin;
        for (; s + kAhead < end; s += kAhead)
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
#pragma unroll
                for (int q = 0; q < kPieces; ++q) acc = multiply<T>(w[j], x[q][j], acc);
                fetch(j, min(s + kAhead + j, end - 1));
            }
        const vec8<T> zero = {};
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const bool in = s + j < end && (s + j) * 32 + 8 * g < p.k;
            w[j] = in ? w[j] : zero;
#pragma unroll
            for (int q = 0; q < kPieces; ++q) acc = multiply<T>(w[j], in ? x[q][j] : zero, acc);
        }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave > 0) return;
    f32x4 sum = sums[0][lane];
#pragma unroll
    for (int q = 1; q < kWaves; ++q) sum += sums[q][lane];
    f32x4 up = sum;
    if constexpr (kDual)
#pragma unroll
        for (int q = 0; q < 4; ++q) up[q] = __shfl_xor(sum[q], 32);
    const int col = n0 + 4 * g;
    if (r < p.m && col < p.n && !(kDual && g >= 2)) finish<T, kEnding>(p.finish, r, col, sum, up, Scales{1.f, 1.f});
}

// ---------------------------------------------------------------- host
// The tiles, and what one takes on MI355X in microseconds: before and behind the sum, and for each stage of 64 while the chip
// is full (fits to 128 .. 4096 rows of 5120 x 1536 and 7168 x 2048).  A tile of 256 x 256 has two stages in LDS, one of 128 x
// 256 three, one of 128 x 128 five: the smaller it is, the more a stage's loads count, which take 1.4 us to land.
struct Shape {
    int m, n;  // rows, columns
    float fixed, stage;
};
enum { kSquare, kWide, kSmall, kFlat, kFewRows };
constexpr Shape kShapes[] = {{256, 256, 6.f, 1.66f}, {128, 256, 4.f, 1.15f}, {128, 128, 3.f, 0.68f}, {32, 128, 3.f, 0.7f}};

struct Cut {
    int shape, parts;
};

int64_t tiles_of(const Shape& s, int64_t m, int64_t n, bool dual) {
    const int64_t nb = dual ? s.n / 2 : s.n;
    return (m + s.m - 1) / s.m * ((n + nb - 1) / nb);
}

// The tile, and the parts that the sum is cut into, with the least time to expect; `products` of this size go together and
// are not cut.  Parts cost a launch, a round trip for every eight and their sums' way to memory and back.  Against 3 us and 4.6
// TB/s for that, with two workgroups of 32 rows a compute unit, in us: 24 rows of 5120 x 1536 24.6 (28.6), 333 of 2048 x 1024
// 31.2 (34.9), 200 of 5120 x 1536 36.8 (40.5); at worst 1.5% slower (4096 of 7168 x 2048 with gradients).
Cut cut(int64_t m, int64_t n, int64_t k, int sums, bool dual, int products) {
    int cus = 0;
    if (current_cu_count(&cus) != kOk) cus = 256;
    const int64_t stages = (k + kDepth - 1) / kDepth * sums;
    Cut best{kSquare, 1};
    float least = 0.f;
    for (int i = kSquare; i <= kFlat; ++i) {
        const Shape& s = kShapes[i];
        if ((i == kFlat) != (m <= 32 && products == 1)) continue;
        const int64_t tiles = tiles_of(s, m, n, dual) * products, slots = cus;
        const int64_t most = products > 1 ? 1 : std::min<int64_t>(32, stages / 2);
        for (int64_t parts = 1; parts == 1 || (parts <= most && tiles * parts <= slots); ++parts) {
            float time = static_cast<float>((tiles * parts + slots - 1) / slots) *
                         (s.fixed + s.stage * static_cast<float>((stages + parts - 1) / parts));
            if (parts > 1)
                time += 4.f + 1.2f * static_cast<float>((parts - 1) / 8) +
                        static_cast<float>(parts * (dual ? 2 : 1) * m * n) * 8.f / 3.5e6f;
            if (least == 0.f || time < least) {
                least = time;
                best = {i, static_cast<int>(parts)};
            }
        }
    }
    return best;
}

template <typename T, Layout kA, Layout kB, Ending kEnding, int kM, int kN, int kWavesM, int kWavesN, int kStages>
int launch_tiles(const ArgsOf<kA>& args, int64_t blocks, hipStream_t stream) {
    auto* kernel = tile_kernel<T, kA, kB, kEnding, kM, kN, kWavesM, kWavesN, kStages>;
    constexpr int kBytes = kStages * (kM + kN) * kDepth * 2;
    static std::atomic<uint64_t> raised{0};  // devices on which the kernel has been given its LDS
    int dev = 0;
    QSRT_HIP_TRY(hipGetDevice(&dev));
    const uint64_t bit = dev < 64 ? uint64_t{1} << dev : 0;
    if (!(raised.load(std::memory_order_relaxed) & bit)) {
        QSRT_HIP_TRY(hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kBytes));
        raised.fetch_or(bit, std::memory_order_relaxed);
    }
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks)), dim3(64 * kWavesM * kWavesN), kBytes, stream, args);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

template <typename T, Layout kA, Layout kB, Ending kEnding>
int launch_shape(const ArgsOf<kA>& args, int shape, int64_t blocks, hipStream_t stream) {
    if constexpr (kA == kRows)  // the weights' gradients go together
        if (shape == kFlat) return launch_tiles<T, kA, kB, kEnding, 32, 128, 1, 4, 4>(args, blocks, stream);
    if (shape == kSquare) return launch_tiles<T, kA, kB, kEnding, 256, 256, 2, 4, 2>(args, blocks, stream);
    if (shape == kWide) return launch_tiles<T, kA, kB, kEnding, 128, 256, 2, 4, 3>(args, blocks, stream);
    return launch_tiles<T, kA, kB, kEnding, 128, 128, 2, 4, 5>(args, blocks, stream);
}

template <typename T, Ending kEnding>
int run_rows(const Product& p, hipStream_t stream) {
    constexpr bool kDual = kEnding == kActivate;
    const RowsArgs r{{p.a[0], p.a[1]}, p.b[0], p.b2, p.lda, p.ldb, static_cast<int>(p.m), static_cast<int>(p.n),
                     static_cast<int>(p.k), p.finish};
    constexpr int kWaves = kDual ? 8 : 4, kColumns = kDual ? 8 : 16;
    const dim3 grid(static_cast<unsigned>((r.n + kColumns - 1) / kColumns));
    hipLaunchKernelGGL((rows_kernel<T, kEnding, kWaves, 4>), grid, dim3(64 * kWaves), 0, stream, r);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

template <typename T, Layout kA, Layout kB, Ending kEnding>
int run(ArgsOf<kA>& args, Cut c, hipStream_t stream) {
    if constexpr (kA == kRows && kB == kRows)
        if (c.shape == kFewRows) return run_rows<T, kEnding>(args.product[0], stream);
    const Shape& s = kShapes[c.shape];
    int64_t blocks = 0;
    for (int i = 0; i < args.products; ++i) {
        Product& p = args.product[i];
        const int nb = kEnding == kActivate ? s.n / 2 : s.n;
        p.tiles_m = static_cast<int>((p.m + s.m - 1) / s.m);
        p.tiles_n = static_cast<int>((p.n + nb - 1) / nb);
        blocks += static_cast<int64_t>(p.tiles_m) * p.tiles_n;
    }
    args.parts = c.parts;
    blocks *= c.parts;
    if (blocks >= 1 << 23) return fail(kBadArgument, "qsrt_gated_ffn: too many tiles for one launch");  // of 512 threads, 2^32 in all
    if (int rc = launch_shape<T, kA, kB, kEnding>(args, c.shape, blocks, stream)) return rc;
    if (kA == kRows && c.parts > 1) {
        const Product& p = args.product[0];
        hipLaunchKernelGGL((join_kernel<T, kEnding>), dim3(static_cast<unsigned>((p.m * p.n / 4 + 255) / 256)), dim3(256), 0,
                           stream, args.partial, c.parts, p.m, p.n, p.finish);
        QSRT_HIP_TRY(hipGetLastError());
    }
    return kOk;
}

constexpr int64_t kMaxTokens = 1 << 20, kMaxChannels = 1 << 17, kMaxLd = 1 << 22;

bool sizes_fit(int64_t tokens, int64_t hidden, int64_t inter) {
    return tokens >= 0 && tokens <= kMaxTokens && hidden > 0 && hidden <= kMaxChannels && inter > 0 && inter <= kMaxChannels &&
           hidden % 8 == 0 && inter % 8 == 0;
}

// Up to 64 rows, where reading the weights bounds a product, rows between products go on in two pieces: the result is then
// off by its own rounding alone (forward in f16 while M is over 2^-10 or so: under 2^-14 both pieces end at 2^-24, as the result
// itself does).  In one, it is off by 1.4 times as much (two roundings of one size); in two, 64 rows of 7168 x 2048 take 39.4
// us, not 35.5, 32 of 5120 x 1536 31.1, not 28.9, and 500 rows 89 us, not 73; 4096 of 7168 x 2048 395, not 304, and with
// gradients 1468, not 932.
int pieces_of(int64_t tokens) { return tokens <= 64 ? 2 : 1; }

// Up to 16 rows, one side of a matrix instruction, meet a kernel of their own.  Against tiles with parts, in us at 8, 12 and 16
// rows: 2048 x 1024 10.1, 10.7, 11.3 for 15.5, 15.8, 16.0; 5120 x 1536 20.9, 23.2, 26.2 for 24.8, 25.3, 25.3; 7168 x 2048 27.1,
// 30.3, 33.4 for 31.3, 31.6, 32.1.  With 17 to 32 the rows of activations would be read twice as often as the weights.
bool few_rows(int64_t tokens) { return tokens <= 16; }

size_t round_up(size_t n) { return (n + 255) & ~size_t{255}; }
size_t part_bytes(const Cut& c, int64_t m, int64_t n, int planes) {
    return c.parts > 1 ? round_up(sizeof(float) * c.parts * planes * m * n) : 0;
}

struct Forward {
    int pieces;
    Cut up, down;
    size_t middle, partial, bytes;
};
Forward plan_forward(int64_t tokens, int64_t hidden, int64_t inter) {
    Forward f;
    f.pieces = pieces_of(tokens);
    const Cut few{kFewRows, 1};
    f.up = few_rows(tokens) ? few : cut(tokens, inter, hidden, 1, true, 1);
    f.down = few_rows(tokens) ? few : cut(tokens, hidden, inter, f.pieces, false, 1);
    f.middle = round_up(sizeof(uint16_t) * f.pieces * tokens * inter);
    f.partial = std::max(part_bytes(f.up, tokens, inter, 2), part_bytes(f.down, tokens, hidden, 1));
    f.bytes = f.middle + f.partial;
    return f;
}

struct Backward {
    int pieces;
    Cut middle, x, weights;
    size_t rows, partial, scales, bytes;
};
Backward plan_backward(int64_t tokens, int64_t hidden, int64_t inter) {
    Backward b;
    b.pieces = pieces_of(tokens);
    b.middle = cut(tokens, inter, hidden, 1, false, 1);
    b.x = cut(tokens, hidden, inter, 2 * b.pieces, false, 1);
    b.weights = cut(inter, hidden, tokens, b.pieces, false, 3);
    b.rows = round_up(sizeof(uint16_t) * b.pieces * tokens * inter);
    b.partial = std::max(part_bytes(b.middle, tokens, inter, 1), part_bytes(b.x, tokens, hidden, 1));
    b.scales = round_up(sizeof(f32x4) * kBoundGroups + sizeof(Scales));  // of f16
    b.bytes = 3 * b.rows + b.partial + b.scales;
    return b;
}

struct Matrix {
    const void* p;
    int64_t ld, rows, cols;
    const char* name;
    int64_t apart() const { return rows > 1 ? ld : cols; }  // a lone row's leading dimension says nothing
};
int check_matrix(const char* call, const Matrix& m) {
    if (!m.p) return fail(kBadArgument, "%s: null pointer for %s", call, m.name);
    if (reinterpret_cast<uintptr_t>(m.p) % 16 || (m.rows > 1 && (m.ld % 8 || m.ld < m.cols || m.ld > kMaxLd)))
        return fail(kBadArgument, "%s: rows of %s must be 16-byte aligned, whole and at most 2^22 elements apart", call, m.name);
    return kOk;
}

struct Block {
    Matrix x, gate, up, down;
    int dtype, activation;
    int64_t tokens, hidden, inter;
};
int check_block(const char* call, const Block& b) {
    if (!sizes_fit(b.tokens, b.hidden, b.inter))
        return fail(kBadArgument, "%s: at most 2^20 tokens, and channels in multiples of 8 up to 2^17", call);
    if (b.dtype != 0 && b.dtype != 1) return fail(kBadArgument, "%s: dtype must be 0 (bf16) or 1 (f16)", call);
    if (b.activation != 0 && b.activation != 1) return fail(kBadArgument, "%s: activation must be 0 (swiglu) or 1 (situ)", call);
    if (b.tokens == 0) return kOk;
    for (const Matrix* m : {&b.x, &b.gate, &b.up, &b.down})
        if (int rc = check_matrix(call, *m)) return rc;
    return kOk;
}
int check_workspace(const char* call, const void* ws, size_t given, size_t need) {
    if (!ws || given < need) return fail(kWorkspaceTooSmall, "%s: needs %zu workspace bytes", call, need);
    if (reinterpret_cast<uintptr_t>(ws) % 16) return fail(kBadArgument, "%s: the workspace must be 16-byte aligned", call);
    return kOk;
}

Pieces pieces_at(char* ws, int64_t tokens, int64_t inter, int pieces) {
    return {ws, pieces > 1 ? ws + sizeof(uint16_t) * tokens * inter : nullptr, nullptr};
}

// One product's sums: a in pieces by b, or a by b in pieces.
void add_sums(Product& p, const Pieces& a, const void* b) {
    for (const void* piece : {a.hi, a.lo})
        if (piece) {
            p.a[p.sums] = piece;
            p.b[p.sums++] = b;
        }
}

template <typename T>
int forward(const Block& b, float* pre, const Matrix& out, char* ws, const Forward& f, hipStream_t stream) {
    TileArgs<1> args = {};
    args.products = 1;
    args.partial = reinterpret_cast<float*>(ws + f.middle);
    Product& p = args.product[0];
    const Pieces middle = pieces_at(ws, b.tokens, b.inter, f.pieces);
    p.a[0] = b.x.p;
    p.b[0] = b.gate.p;
    p.b2 = b.up.p;
    p.lda = b.x.apart();
    p.ldb = b.gate.ld;
    p.m = b.tokens;
    p.n = b.inter;
    p.k = b.hidden;
    p.sums = 1;
    p.finish = {nullptr, b.inter, b.activation, pre, pre ? pre + b.tokens * b.inter : nullptr, middle, {}, {}};
    if (int rc = run<T, kRows, kRows, kActivate>(args, f.up, stream)) return rc;
    if (!out.p) return kOk;
    p.sums = 0;
    add_sums(p, middle, b.down.p);
    p.lda = b.inter;
    p.ldb = b.down.ld;
    p.n = b.hidden;
    p.k = b.inter;
    p.finish = {const_cast<void*>(out.p), out.apart()};
    return run<T, kRows, kRows, kStore>(args, f.down, stream);
}

struct Gradients {
    Matrix dy;
    const float* pre;
    Matrix dx;
    void *gate, *up, *down;              // of the weights, in one piece each; or null
    void *gate_rows, *up_rows, *middle;  // dG, dU and M in one piece each; or null
};

template <typename T>
int backward(const Block& b, const Gradients& g, char* ws, const Backward& plan, hipStream_t stream) {
    TileArgs<1> args = {};
    args.products = 1;
    args.partial = reinterpret_cast<float*>(ws + 3 * plan.rows);
    Pieces dg = pieces_at(ws, b.tokens, b.inter, plan.pieces), du = pieces_at(ws + plan.rows, b.tokens, b.inter, plan.pieces),
           middle = pieces_at(ws + 2 * plan.rows, b.tokens, b.inter, plan.pieces);
    const bool scaled = kScaled<T> && (g.dx.p || g.gate || g.up || g.down);
    const auto hand_out = [&](Pieces& rows, void* to) {
        if (to) (scaled ? rows.plain : rows.hi) = to;
    };
    hand_out(dg, g.gate_rows);
    hand_out(du, g.up_rows);
    hand_out(middle, g.middle);
    f32x4* const bounds = scaled ? reinterpret_cast<f32x4*>(ws + 3 * plan.rows + plan.partial) : nullptr;
    float* const unscale = scaled ? reinterpret_cast<float*>(bounds + kBoundGroups) : nullptr;
    if constexpr (kScaled<T>)
        if (scaled) {
            const BoundArgs a{g.dy.p, b.down.p, g.dy.apart(), b.down.ld, b.tokens, b.hidden, b.inter, b.activation, g.pre, bounds};
            hipLaunchKernelGGL(bounds_kernel, dim3(kBoundGroups), dim3(64 * kBoundWaves), 0, stream, a);
            QSRT_HIP_TRY(hipGetLastError());
        }
    {
        Product& p = args.product[0];
        p.a[0] = g.dy.p;
        p.b[0] = b.down.p;
        p.lda = g.dy.apart();
        p.ldb = b.down.ld;
        p.m = b.tokens;
        p.n = b.inter;
        p.k = b.hidden;
        p.sums = 1;
        float* pre = const_cast<float*>(g.pre);
        p.finish = {nullptr, b.inter, b.activation, pre, pre + b.tokens * b.inter, middle, dg, du, bounds, unscale};
        if (int rc = run<T, kRows, kCols, kSlopes>(args, plan.middle, stream)) return rc;
    }
    if (g.dx.p) {
        Product& p = args.product[0];
        p.sums = 0;
        add_sums(p, dg, b.gate.p);
        add_sums(p, du, b.up.p);
        p.lda = b.inter;
        p.ldb = b.gate.ld;
        p.n = b.hidden;
        p.k = b.inter;
        p.finish = {const_cast<void*>(g.dx.p), g.dx.apart()};
        p.finish.unscale = unscale;
        if (int rc = run<T, kRows, kCols, kStore>(args, plan.x, stream)) return rc;
    }
    TileArgs<kProducts> three = {};
    const auto add = [&](const Pieces& rows, const Matrix& other, void* out, bool rows_first, float* sums_by) {
        if (!out) return;
        Product& p = three.product[three.products++];
        p = {};
        add_sums(p, rows, other.p);
        p.lda = b.inter;
        p.ldb = other.apart();
        p.m = b.inter;
        p.n = b.hidden;
        if (!rows_first) {
            std::swap_ranges(p.a, p.a + kSums, p.b);
            std::swap(p.lda, p.ldb);
            std::swap(p.m, p.n);
        }
        p.k = b.tokens;
        p.finish = {out, p.n};
        p.finish.unscale = sums_by;
    };
    add(dg, b.x, g.gate, true, unscale);
    add(du, b.x, g.up, true, unscale);
    add(middle, g.dy, g.down, false, scaled ? unscale + 1 : nullptr);
    return three.products ? run<T, kCols, kCols, kStore>(three, plan.weights, stream) : kOk;
}

}  // namespace
}  // namespace qsrt

using namespace qsrt;

extern "C" size_t qsrt_gated_ffn_workspace_bytes(int64_t tokens, int64_t hidden, int64_t inter) {
    if (tokens == 0 || !sizes_fit(tokens, hidden, inter)) return 0;
    return plan_forward(tokens, hidden, inter).bytes;
}

extern "C" int qsrt_gated_ffn(const void* x, int64_t x_ld, const void* gate, const void* up, int64_t up_ld, const void* down,
                              int64_t down_ld, int dtype, int64_t tokens, int64_t hidden, int64_t inter, int activation,
                              float* pre, void* out, int64_t out_ld, void* ws, size_t ws_bytes, void* stream) {
    constexpr const char* kCall = "qsrt_gated_ffn";
    const Block b{{x, x_ld, tokens, hidden, "x"}, {gate, up_ld, inter, hidden, "gate"}, {up, up_ld, inter, hidden, "up"},
                  {down, down_ld, hidden, inter, "down"}, dtype, activation, tokens, hidden, inter};
    if (int rc = check_block(kCall, b)) return rc;
    if (tokens == 0) return kOk;
    const Matrix y{out, out_ld, tokens, hidden, "out"};
    if (out || !pre)
        if (int rc = check_matrix(kCall, y)) return rc;
    if (reinterpret_cast<uintptr_t>(pre) % 16) return fail(kBadArgument, "%s: pre must be 16-byte aligned", kCall);
    const Forward f = plan_forward(tokens, hidden, inter);
    if (int rc = check_workspace(kCall, ws, ws_bytes, f.bytes)) return rc;
    return (dtype == 0 ? forward<__bf16> : forward<_Float16>)(b, pre, y, static_cast<char*>(ws), f, static_cast<hipStream_t>(stream));
}

extern "C" size_t qsrt_gated_ffn_backward_workspace_bytes(int64_t tokens, int64_t hidden, int64_t inter) {
    if (tokens == 0 || !sizes_fit(tokens, hidden, inter)) return 0;
    return plan_backward(tokens, hidden, inter).bytes;
}

extern "C" int qsrt_gated_ffn_backward(const void* dy, int64_t dy_ld, const void* x, int64_t x_ld, const void* gate, const void* up,
                                       int64_t up_ld, const void* down, int64_t down_ld, int dtype, int64_t tokens, int64_t hidden,
                                       int64_t inter, int activation, const float* pre, void* dx, int64_t dx_ld, void* d_gate,
                                       void* d_up, void* d_down, void* gate_rows, void* up_rows, void* middle, void* ws,
                                       size_t ws_bytes, void* stream) {
    constexpr const char* kCall = "qsrt_gated_ffn_backward";
    const Block b{{x, x_ld, tokens, hidden, "x"}, {gate, up_ld, inter, hidden, "gate"}, {up, up_ld, inter, hidden, "up"},
                  {down, down_ld, hidden, inter, "down"}, dtype, activation, tokens, hidden, inter};
    if (int rc = check_block(kCall, b)) return rc;
    if (tokens == 0) return kOk;
    const Gradients g{{dy, dy_ld, tokens, hidden, "dy"}, pre, {dx, dx_ld, tokens, hidden, "dx"}, d_gate, d_up, d_down,
                      gate_rows, up_rows, middle};
    if (int rc = check_matrix(kCall, g.dy)) return rc;
    if (dx)
        if (int rc = check_matrix(kCall, g.dx)) return rc;
    if (!pre) return fail(kBadArgument, "%s: null pointer for pre", kCall);
    for (const void* p : {static_cast<const void*>(pre), static_cast<const void*>(d_gate), static_cast<const void*>(d_up),
                          static_cast<const void*>(d_down), static_cast<const void*>(gate_rows),
                          static_cast<const void*>(up_rows), static_cast<const void*>(middle)})
        if (reinterpret_cast<uintptr_t>(p) % 16) return fail(kBadArgument, "%s: pre, gradients and rows must be 16-byte aligned", kCall);
    const Backward plan = plan_backward(tokens, hidden, inter);
    if (int rc = check_workspace(kCall, ws, ws_bytes, plan.bytes)) return rc;
    return (dtype == 0 ? backward<__bf16> : backward<_Float16>)(b, g, static_cast<char*>(ws), plan, static_cast<hipStream_t>(stream));
}

extern "C" int qsrt_gated_ffn_plan(int64_t tokens, int64_t hidden, int64_t inter, int64_t* plan) {
    constexpr const char* kCall = "qsrt_gated_ffn_plan";
    if (tokens == 0 || !sizes_fit(tokens, hidden, inter) || !plan) return fail(kBadArgument, "%s: bad sizes or no plan", kCall);
    const Forward f = plan_forward(tokens, hidden, inter);
    const Backward b = plan_backward(tokens, hidden, inter);
    for (const Cut& c : {f.up, f.down, b.middle, b.x, b.weights}) {
        *plan++ = c.shape;
        *plan++ = c.parts;
    }
    *plan = f.pieces;
    return kOk;
}

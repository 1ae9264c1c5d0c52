// The router of a mixture-of-experts layer, and the grouping of rows by expert or adapter.
#include <algorithm>

#include "packed.h"
#include "qsrt_amd.h"

namespace qsrt {
namespace {

// logits[t][e] = sum_h x[t][h] w[e][h].  One workgroup for 16 experts and 16 tokens; its 16 waves take every 16th step of
// 32 channels, products exact and sums FP32 on the matrix cores, and add up in LDS in wave order.
constexpr int kRouterWaves = 16;

template <typename T>
__global__ __launch_bounds__(64 * kRouterWaves) void router_logits_kernel(const T* __restrict__ x, int64_t ld,
                                                                          const T* __restrict__ w, int64_t w_ld,
                                                                          int tokens, int hidden, int experts,
                                                                          float* __restrict__ logits) {
    __shared__ f32x4 sums[kRouterWaves][64];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int e0 = 16 * blockIdx.x, t0 = 16 * blockIdx.y;
    typedef T t8 __attribute__((ext_vector_type(8)));
    const T* wr = w + min(e0 + m, experts - 1) * w_ld + 8 * g;  // rows past the end repeat the last; not stored
    const T* xr = x + min(t0 + m, tokens - 1) * ld + 8 * g;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](t8 a, t8 b) {
        if constexpr (__is_same(T, __bf16))
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
        else
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
    };
    constexpr int kStep = 32 * kRouterWaves, kBatch = 7;
    int h = 32 * wave;
    for (; h + (kBatch - 1) * kStep + 32 <= hidden; h += kBatch * kStep) {  // a batch of loads in flight
        t8 a[kBatch], b[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            a[j] = *reinterpret_cast<const t8*>(wr + h + j * kStep);
            b[j] = *reinterpret_cast<const t8*>(xr + h + j * kStep);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) multiply(a[j], b[j]);
    }
    const t8 zero = {};
    for (; h < hidden; h += kStep) {
        const bool in = h + 8 * g < hidden;  // hidden is a multiple of 8
        multiply(in ? *reinterpret_cast<const t8*>(wr + h) : zero, in ? *reinterpret_cast<const t8*>(xr + h) : zero);
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int v = 1; v < kRouterWaves; ++v) acc += sums[v][lane];
    const int t = t0 + m;
    if (t >= tokens) return;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (e0 + 4 * g + i < experts) logits[static_cast<int64_t>(t) * experts + e0 + 4 * g + i] = acc[i];
}

constexpr int kMaxExperts = 1024;

// Order of float keys as unsigned integers; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t sortable(float key) {
    if (!(key == key)) key = -__builtin_inff();
    key += 0.0f;
    const uint32_t u = __builtin_bit_cast(uint32_t, key);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

// Over a wave, without LDS: rows of 16 lanes by data-parallel moves, then across rows.
template <typename Op, typename V>
__device__ __forceinline__ V over_wave(V v, Op op) {
    auto with = [&](auto moved) { v = op(v, __builtin_bit_cast(V, moved)); };
    with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0xB1, 0xF, 0xF, true));
    with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x4E, 0xF, 0xF, true));
    with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x141, 0xF, 0xF, true));
    with(__builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x140, 0xF, 0xF, true));
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = op(__builtin_bit_cast(V, uint32_t(a[0])), __builtin_bit_cast(V, uint32_t(a[1])));
    const uint32_t t = __builtin_bit_cast(uint32_t, v);
    const auto b = __builtin_amdgcn_permlane32_swap(t, t, false, false);
    return op(__builtin_bit_cast(V, uint32_t(b[0])), __builtin_bit_cast(V, uint32_t(b[1])));
}
__device__ __forceinline__ float wave_max(float v) {
    return over_wave(v, [](float a, float b) { return fmaxf(a, b); });
}
__device__ __forceinline__ uint32_t wave_max(uint32_t v) {
    return over_wave(v, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}
__device__ __forceinline__ float wave_sum(float v) {
    return over_wave(v, [](float a, float b) { return a + b; });
}

struct ChooseArgs {
    const float *logits, *bias;
    int tokens, experts, k, scoring, normalize;
    float scale;
    float* weights;
    int* ids;
};

// One wave a token, expert 64 j + lane in slot j: scores, k rounds of (largest key, lowest index), weights.
template <int kSlots>
__device__ __forceinline__ void choose(const ChooseArgs& p, int token, int lane) {
    float score[kSlots];
    uint32_t key[kSlots];  // sortable; 0: none, or taken (the least of real keys, -inf, is above 0)
    float top = -__builtin_inff();
    const float* row = p.logits + static_cast<int64_t>(token) * p.experts;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
        const int e = 64 * j + lane;
        const bool in = e < p.experts;
        score[j] = in ? row[e] : -__builtin_inff();
        key[j] = in ? sortable(score[j]) : 0u;
        top = fmaxf(top, score[j]);
    }
    if (p.scoring == 0) {  // softmax over all experts
        top = wave_max(top);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            score[j] = 64 * j + lane < p.experts ? expf(score[j] - top) : 0.f;
            sum += score[j];
        }
        sum = wave_sum(sum);
#pragma unroll
        for (int j = 0; j < kSlots; ++j) score[j] /= sum;
    } else {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) score[j] = 1.0f / (1.0f + expf(-score[j]));
    }
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            const int e = 64 * j + lane;
            if (e < p.experts) key[j] = sortable(score[j] + p.bias[e]);
        }
    }
    float chosen = 0.f, total = 0.f;  // lane r: weight and expert of the r-th
    int id = 0;
    for (int r = 0; r < p.k; ++r) {
        uint32_t best = 0;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) best = key[j] > best ? key[j] : best;
        best = wave_max(best);
        uint64_t at = 0;
        float s = 0.f;
        int e = 0;
#pragma unroll
        for (int j = kSlots - 1; j >= 0; --j) {  // the lowest slot that holds it, and there the lowest lane
            const uint64_t has = __ballot(key[j] == best);
            if (has) {
                at = has;
                e = 64 * j;
                s = score[j];
            }
        }
        const int winner = __builtin_ctzll(at);
        s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), winner));
        e += winner;
        if (lane == r) {
            chosen = s;
            id = e;
        }
        total += s;
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
            if (64 * j + lane == e) key[j] = 0;
    }
    if (lane < p.k) {
        if (p.normalize) chosen /= total;
        p.weights[static_cast<int64_t>(token) * p.k + lane] = chosen * p.scale;
        p.ids[static_cast<int64_t>(token) * p.k + lane] = id;
    }
}

template <int kSlots>
__global__ __launch_bounds__(64) void choose_kernel(const ChooseArgs p) {
    choose<kSlots>(p, blockIdx.x, threadIdx.x);
}

// Rows 0 .. n - 1 by key, in one workgroup: counts, offsets, chunks of at most chunk_rows, then the rows of each key.
// Rows of a key are placed by an LDS counter, in no fixed order: no result depends on a row's neighbours in its chunk.
// A row whose key is outside [0, keys) is left out (clean = -1), or with `none` put under the key -1.
constexpr int kGroupThreads = 1024;

__global__ __launch_bounds__(kGroupThreads) void group_kernel(const GroupArgs p) {
    extern __shared__ int lds[];
    int* at = lds;  // [keys + 1]: counts, then next place
    __shared__ int waves[2][kGroupThreads / 64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slots = p.keys + 1;
    for (int i = tid; i < slots; i += kGroupThreads) at[i] = 0;
    __syncthreads();
    for (int i = tid; i < p.n; i += kGroupThreads) {
        const int id = p.ids[i];
        const bool ok = id >= 0 && id < p.keys;
        p.clean[i] = ok ? id : -1;
        if (ok || p.none) atomicAdd(&at[ok ? id : p.keys], 1);
    }
    __syncthreads();
    // each thread owns a run of keys
    const int run = (slots + kGroupThreads - 1) / kGroupThreads;
    const int k0 = min(tid * run, slots), k1 = min(k0 + run, slots);
    int rows = 0, chunks = 0;
    for (int q = k0; q < k1; ++q) {
        rows += at[q];
        chunks += (at[q] + p.chunk_rows - 1) / p.chunk_rows;
    }
    int rs = rows, cs = chunks;  // inclusive scan over the wave
    for (int h = 1; h < 64; h <<= 1) {
        const int r = __shfl_up(rs, h), c = __shfl_up(cs, h);
        if (lane >= h) {
            rs += r;
            cs += c;
        }
    }
    if (lane == 63) {
        waves[0][wave] = rs;
        waves[1][wave] = cs;
    }
    __syncthreads();
    int total = 0, r0 = rs - rows, c0 = cs - chunks;
    for (int q = 0; q < kGroupThreads / 64; ++q) {
        if (q < wave) {
            r0 += waves[0][q];
            c0 += waves[1][q];
        }
        total += waves[1][q];
    }
    for (int q = k0; q < k1; ++q) {
        const int count = at[q];
        for (int c = 0; c < count; c += p.chunk_rows)
            p.chunks[c0++] = Chunk{q == p.keys ? -1 : q, r0 + c, min(p.chunk_rows, count - c), 0};
        at[q] = r0;
        r0 += count;
    }
    __syncthreads();
    for (int i = tid; i < p.n; i += kGroupThreads) {
        const int id = p.ids[i];
        const bool ok = id >= 0 && id < p.keys;
        if (ok || p.none) p.order[atomicAdd(&at[ok ? id : p.keys], 1)] = i;
    }
    if (wave < 2) {  // how to cut the K axis: wave 0 for the first product, wave 1 for the second
        const int64_t units = static_cast<int64_t>(total) * p.units[wave];
        const int parts = choose_parts(units, p.strips[wave], p.max_parts[wave], p.waves, lane);
        if (lane == 0) {
            p.head->parts[wave] = parts;
            if (wave == 0) p.head->chunks = total;
        }
    }
}

}  // namespace

int launch_group(const GroupArgs& args, hipStream_t stream) {
    const size_t lds = sizeof(int) * (static_cast<size_t>(args.keys) + 1);
    hipLaunchKernelGGL(group_kernel, dim3(1), dim3(kGroupThreads), lds, stream, args);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

}  // namespace qsrt

using namespace qsrt;

extern "C" size_t qsrt_route_workspace_bytes(int64_t tokens, int64_t experts) {
    if (tokens <= 0 || experts <= 0) return 0;
    return static_cast<size_t>(tokens) * static_cast<size_t>(experts) * sizeof(float);
}

extern "C" int qsrt_route(const void* x, int64_t x_ld, const void* weight, int64_t weight_ld, int dtype, int64_t tokens,
                          int64_t hidden, int64_t experts, int k, const float* bias, int scoring, int normalize,
                          float scale, float* weights, int32_t* ids, void* ws, size_t ws_bytes, void* stream_) {
    if (tokens == 0) return kOk;
    if (!x || !weight || !weights || !ids || tokens < 0 || hidden <= 0 || experts <= 0)
        return fail(kBadArgument, "qsrt_route: null pointer or bad size");
    if (dtype != 0 && dtype != 1) return fail(kBadArgument, "qsrt_route: dtype must be 0 (bf16) or 1 (f16)");
    if (experts > kMaxExperts) return fail(kBadArgument, "qsrt_route: at most %d experts", kMaxExperts);
    if (k < 1 || k > 64 || k > experts) return fail(kBadArgument, "qsrt_route: k must be 1 .. min(64, experts)");
    if (scoring != 0 && scoring != 1) return fail(kBadArgument, "qsrt_route: scoring must be 0 (softmax) or 1 (sigmoid)");
    if (tokens > (1 << 20) || hidden > (1 << 24)) return fail(kBadArgument, "qsrt_route: too many tokens or channels");
    if (hidden % 8 || x_ld % 8 || weight_ld % 8 || x_ld < hidden || weight_ld < hidden ||
        reinterpret_cast<uintptr_t>(x) % 16 || reinterpret_cast<uintptr_t>(weight) % 16)
        return fail(kBadArgument, "qsrt_route: rows must be 16-byte aligned and a multiple of 8 channels");
    if (!ws || ws_bytes < qsrt_route_workspace_bytes(tokens, experts))
        return fail(kWorkspaceTooSmall, "qsrt_route: needs %zu workspace bytes",
                    qsrt_route_workspace_bytes(tokens, experts));
    hipStream_t stream = static_cast<hipStream_t>(stream_);
    const dim3 grid(static_cast<unsigned>((experts + 15) / 16), static_cast<unsigned>((tokens + 15) / 16));
    float* logits = static_cast<float*>(ws);
    if (dtype == 0)
        hipLaunchKernelGGL(router_logits_kernel<__bf16>, grid, dim3(64 * kRouterWaves), 0, stream,
                           static_cast<const __bf16*>(x), x_ld, static_cast<const __bf16*>(weight), weight_ld,
                           static_cast<int>(tokens), static_cast<int>(hidden), static_cast<int>(experts), logits);
    else
        hipLaunchKernelGGL(router_logits_kernel<_Float16>, grid, dim3(64 * kRouterWaves), 0, stream,
                           static_cast<const _Float16*>(x), x_ld, static_cast<const _Float16*>(weight), weight_ld,
                           static_cast<int>(tokens), static_cast<int>(hidden), static_cast<int>(experts), logits);
    QSRT_HIP_TRY(hipGetLastError());
    const ChooseArgs ca{logits, bias, static_cast<int>(tokens), static_cast<int>(experts), k, scoring, normalize, scale,
                        weights, ids};
    hipLaunchKernelGGL((experts <= 64    ? choose_kernel<1>
                        : experts <= 128 ? choose_kernel<2>
                        : experts <= 256 ? choose_kernel<4>
                        : experts <= 512 ? choose_kernel<8>
                                         : choose_kernel<16>),
                       dim3(static_cast<unsigned>(tokens)), dim3(64), 0, stream, ca);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

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
    const t8 zero = {};
    for (int h = 32 * wave; h < hidden; h += 32 * kRouterWaves) {
        const bool in = h + 8 * g < hidden;  // hidden is a multiple of 8
        const t8 a = in ? *reinterpret_cast<const t8*>(wr + h) : zero;
        const t8 b = in ? *reinterpret_cast<const t8*>(xr + h) : zero;
        if constexpr (sizeof(T) == 2 && __is_same(T, __bf16))
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
        else
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
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

constexpr int kMaxExperts = 1024, kPerLane = kMaxExperts / 64;

// Order of float keys as unsigned integers; NaN counts as -inf, -0 as 0.
__device__ __forceinline__ uint32_t sortable(float key) {
    if (!(key == key)) key = -__builtin_inff();
    key += 0.0f;
    const uint32_t u = __builtin_bit_cast(uint32_t, key);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float wave_max(float v) {
    for (int h = 1; h < 64; h <<= 1) v = fmaxf(v, __shfl_xor(v, h));
    return v;
}
__device__ __forceinline__ float wave_sum(float v) {
    for (int h = 1; h < 64; h <<= 1) v += __shfl_xor(v, h);
    return v;
}

// One wave a token: scores, k rounds of (largest key, lowest index), weights.
__global__ __launch_bounds__(256) void choose_kernel(const float* __restrict__ logits, const float* __restrict__ bias,
                                                     int tokens, int experts, int k, int scoring, int normalize,
                                                     float scale, float* __restrict__ weights, int* __restrict__ ids) {
    const int lane = threadIdx.x & 63;
    const int token = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (token >= tokens) return;
    float score[kPerLane];
    uint64_t key[kPerLane];  // (sortable key, ~index); 0: none, or taken
    float top = -__builtin_inff();
    const float* row = logits + static_cast<int64_t>(token) * experts;
#pragma unroll
    for (int j = 0; j < kPerLane; ++j) {
        const int e = 64 * j + lane;
        score[j] = e < experts ? row[e] : -__builtin_inff();
        key[j] = 0;
        if (e < experts) {
            key[j] = static_cast<uint64_t>(sortable(score[j])) << 32 | static_cast<uint32_t>(~e);
            top = fmaxf(top, score[j]);
        }
    }
    if (scoring == 0) {  // softmax over all experts
        top = wave_max(top);
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j)
            if (64 * j + lane < experts) {
                score[j] = expf(score[j] - top);
                sum += score[j];
            }
        sum = wave_sum(sum);
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) score[j] /= sum;
    } else {
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) score[j] = 1.0f / (1.0f + expf(-score[j]));
    }
    if (bias) {
#pragma unroll
        for (int j = 0; j < kPerLane; ++j) {
            const int e = 64 * j + lane;
            if (e < experts)
                key[j] = static_cast<uint64_t>(sortable(score[j] + bias[e])) << 32 | static_cast<uint32_t>(~e);
        }
    }
    float chosen = 0.f;  // lane j < k: weight of the j-th
    int id = 0;
    float total = 0.f;
    for (int r = 0; r < k; ++r) {
        uint64_t best = 0;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j)
            if (key[j] > best) {
                best = key[j];
                s = score[j];
            }
        uint64_t all = best;
        for (int h = 1; h < 64; h <<= 1) {
            const uint64_t o = static_cast<uint64_t>(__shfl_xor(static_cast<unsigned long long>(all), h));
            all = o > all ? o : all;
        }
        const int e = static_cast<int>(~static_cast<uint32_t>(all));
        s = __shfl(s, e & 63);  // the winner's lane holds it
        if (lane == r) {
            chosen = s;
            id = e;
        }
        total += s;
#pragma unroll
        for (int j = 0; j < kPerLane; ++j)
            if (key[j] == all) key[j] = 0;
    }
    if (lane < k) {
        if (normalize) chosen /= total;
        weights[static_cast<int64_t>(token) * k + lane] = chosen * scale;
        ids[static_cast<int64_t>(token) * k + lane] = id;
    }
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
    hipLaunchKernelGGL(choose_kernel, dim3(static_cast<unsigned>((tokens + 3) / 4)), dim3(256), 0, stream, logits, bias,
                       static_cast<int>(tokens), static_cast<int>(experts), k, scoring, normalize, scale, weights, ids);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

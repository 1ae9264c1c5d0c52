// The router of a mixture-of-experts layer, and the grouping of rows by expert.
#include <algorithm>

#include "packed.h"
#include "qsrt_amd.h"

namespace qsrt {
namespace {

// logits[split][t][e] = sum over the split's channels of x[t][h] w[e][h].  One workgroup for 16 experts, 16 tokens and one
// split; its four waves take every fourth step of 32 channels, products exact and sums FP32 on the matrix cores, and add up
// in LDS in wave order.  The splits spread a token's router over the chip; workgroups behind them rotate the same rows.
struct LogitsArgs {
    const void *x, *w;
    int64_t ld, w_ld;
    int tokens, hidden, experts, splits, etiles, ttiles;
    float* logits;
    RotateArgs beside;
};

template <typename T>
__global__ __launch_bounds__(256) void router_logits_kernel(const LogitsArgs p) {
    __shared__ f32x4 sums[4][64];
    const int lane = threadIdx.x & 63, m = lane & 15, g = lane >> 4;
    const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
    const int routers = p.etiles * p.ttiles * p.splits;
    if (static_cast<int>(blockIdx.x) >= routers) {
        rotate_block<T>(p.beside, static_cast<int64_t>(blockIdx.x - routers) * 4 + wave, lane);
        return;
    }
    const int e0 = 16 * (blockIdx.x % p.etiles), t0 = 16 * (blockIdx.x / p.etiles % p.ttiles);
    const int split = blockIdx.x / (p.etiles * p.ttiles);
    typedef T t8 __attribute__((ext_vector_type(8)));
    // rows past the end repeat the last; not stored
    const T* wr = static_cast<const T*>(p.w) + min(e0 + m, p.experts - 1) * p.w_ld;
    const T* xr = static_cast<const T*>(p.x) + min(t0 + m, p.tokens - 1) * p.ld;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](t8 a, t8 b) {
        if constexpr (__is_same(T, __bf16))
            acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, acc, 0, 0, 0);
        else
            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc, 0, 0, 0);
    };
    constexpr int kStep = 32 * 4, kBatch = 8;
    const int steps = (p.hidden + 31) / 32;
    const int end = min(p.hidden, 32 * static_cast<int>(static_cast<int64_t>(steps) * (split + 1) / p.splits));
    int h = 32 * static_cast<int>(static_cast<int64_t>(steps) * split / p.splits) + 32 * wave;
    const t8 zero = {};
    // The loads of a batch go out together, also of one that is not full (16 tokens and 64 or 384 experts, weights not cached: 4.9
    // and 5.0 us at 2048 channels, 4.9 and 5.4 at 5120, 5.0 and 5.8 at 7168; one after the other in a batch that is not full 5.7
    // and 6.3 at 5120).  Leaving out those past the end by a branch cost 96 tokens of 7168 channels 18.6 us, 17.6 so.
    for (; h < end; h += kBatch * kStep) {
        t8 a[kBatch], b[kBatch];
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int at = min(h + j * kStep + 8 * g, p.hidden - 8);  // past the end: the last, which nobody takes
            a[j] = *reinterpret_cast<const t8*>(wr + at);
            b[j] = *reinterpret_cast<const t8*>(xr + at);
        }
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
            const int from = h + j * kStep;
            if (from >= end) break;
            if (from + 32 <= end) {
                multiply(a[j], b[j]);
            } else {
                const bool in = from + 8 * g < end;  // hidden is a multiple of 8
                multiply(in ? a[j] : zero, in ? b[j] : zero);
            }
        }
    }
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave) return;
    acc = sums[0][lane] + sums[1][lane] + sums[2][lane] + sums[3][lane];
    const int t = t0 + m;
    if (t >= p.tokens) return;
    float* out = p.logits + (static_cast<int64_t>(split) * p.tokens + t) * p.experts + e0 + 4 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (e0 + 4 * g + i < p.experts) out[i] = acc[i];
}

// Splits of the channels: at most eight, whose sums the choice adds up, as many as there are compute units for, and each wave
// with half a batch of steps at the least.  The number stands in the workspace's size, which is asked for without a device: it
// counts on gfx950's 256 units.
int router_splits(int64_t tokens, int64_t hidden, int64_t experts) {
    constexpr int64_t kUnits = 256, kMost = 8, kLeast = 4 * 32 * 4;
    const int64_t tiles = ((tokens + 15) / 16) * ((experts + 15) / 16);
    return static_cast<int>(std::max<int64_t>(1, std::min({kUnits / tiles, kMost, hidden / kLeast})));
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
    int tokens, experts, splits, k, scoring, normalize;
    float scale;
    float* weights;
    int* ids;
};

// One wave a token, expert 64 j + lane in slot j: scores, k rounds of (largest key, lowest index), weights.
// `local`: a second place for the ids, in LDS (null: none).
template <int kSlots>
__device__ __forceinline__ void choose(const ChooseArgs& p, int token, int lane, int* local) {
    float score[kSlots];
    uint32_t key[kSlots];  // sortable; 0: none, or taken (the least of real keys, -inf, is above 0)
    float top = -__builtin_inff();
    const float* row = p.logits + static_cast<int64_t>(token) * p.experts;
    const int64_t step = static_cast<int64_t>(p.tokens) * p.experts;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) score[j] = 0.f;
    // The loads of a few splits go out together (one after the other the choice of 256 experts took 17 us, with eight 8);
    // fewer where the slots are many, so that all stay in registers.  Slots past the last expert repeat it.
    constexpr int kTogether = kSlots <= 4 ? 8 : 32 / kSlots;
#pragma unroll 1
    for (int q = 0; q < p.splits; q += kTogether) {
        float part[kTogether][kSlots];
#pragma unroll
        for (int i = 0; i < kTogether; ++i)
#pragma unroll
            for (int j = 0; j < kSlots; ++j)
                part[i][j] = row[min(q + i, p.splits - 1) * step + min(64 * j + lane, p.experts - 1)];
#pragma unroll
        for (int i = 0; i < kTogether; ++i)
#pragma unroll
            for (int j = 0; j < kSlots; ++j) score[j] += q + i < p.splits ? part[i][j] : 0.f;
    }
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
        const bool in = 64 * j + lane < p.experts;
        if (!in) score[j] = -__builtin_inff();
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
        uint32_t mine = 0;  // this lane's largest key, in its lowest slot
        int e = 0;
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) {
            const bool larger = key[j] > mine;
            mine = larger ? key[j] : mine;
            e = larger ? 64 * j + lane : e;
            s = larger ? score[j] : s;
        }
        const uint64_t at = __ballot(mine == wave_max(mine));
        int winner = __builtin_ctzll(at);
        if (at & (at - 1)) {  // a tie between lanes: the lowest index
            const uint32_t lowest = ~wave_max(at >> lane & 1 ? ~static_cast<uint32_t>(e) : 0u);
            winner = static_cast<int>(lowest & 63);
        }
        e = __builtin_amdgcn_readlane(e, winner);
        s = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), winner));
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
        if (local) local[token * p.k + lane] = id;
    }
}

template <int kSlots>
__global__ __launch_bounds__(64) void choose_kernel(const ChooseArgs p) {
    choose<kSlots>(p, blockIdx.x, threadIdx.x, nullptr);
}

// Rows 0 .. n - 1 by key, in one workgroup: counts, offsets, chunks of at most chunk_rows, then the rows of each key.
// Rows of a key are placed by an LDS counter, in no fixed order: no result depends on a row's neighbours in its chunk.
// A row whose key is outside [0, keys) is left out (clean = -1).
constexpr int kGroupThreads = 1024;

// Adds one to at[slot] for each active lane and returns the lane's place; lanes of the same slot share an addition for the
// first few slots (long runs of one key), the rest add by themselves.
__device__ __forceinline__ int take_place(int* at, int slot, bool active, int lane) {
    int place = -1;
    for (int round = 0; round < 4; ++round) {
        const uint64_t left = __ballot(active);
        if (!left) return place;
        const int leader = __builtin_ctzll(left);
        const int common = __builtin_amdgcn_readlane(slot, leader);
        const bool same = active && slot == common;
        const uint64_t group = __ballot(same);
        int base = 0;
        if (lane == leader) base = atomicAdd(&at[common], __popcll(group));
        base = __builtin_amdgcn_readlane(base, leader);
        if (same) {
            place = base + __popcll(group & ((uint64_t(1) << lane) - 1));
            active = false;
        }
    }
    if (active) place = atomicAdd(&at[slot], 1);
    return place;
}

struct GroupLds {
    int waves[2][kGroupThreads / 64];
    int ids[kGroupThreads], order[kGroupThreads];  // of up to kGroupThreads rows
};

// Up to 64 rows by one wave, a row a lane, keys in the order of their first rows; no LDS counters, no barriers (choice and
// grouping of a token's 8 of 384 experts 5.9 us, 8.4 by the workgroup and with two reductions a choice).
__device__ __forceinline__ void group_few(const GroupArgs& p, int id, int lane) {
    const bool ok = lane < p.n && id >= 0 && id < p.keys;
    if (lane < p.n) p.clean[lane] = ok ? id : -1;
    uint64_t left = __ballot(ok);
    int rows = 0, chunks = 0;
    while (left) {
        const int key = __builtin_amdgcn_readlane(id, __builtin_ctzll(left));
        const uint64_t same = __ballot(ok && id == key);
        const int count = __popcll(same);
        if (ok && id == key) {
            const int place = __popcll(same & ((uint64_t(1) << lane) - 1));
            p.order[rows + place] = lane;
            if (place % p.chunk_rows == 0)
                p.chunks[chunks + place / p.chunk_rows] = Chunk{key, rows + place, min(p.chunk_rows, count - place), lane};
        }
        left &= ~same;
        rows += count;
        chunks += (count + p.chunk_rows - 1) / p.chunk_rows;
    }
    for (int i = chunks + lane; i < p.max_chunks; i += 64) p.chunks[i] = Chunk{-1, 0, 0, 0};
}

// ids in l.ids already (`local`), or in memory.
__device__ __forceinline__ void group_rows(const GroupArgs& p, int* at, GroupLds& l, bool local) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slots = p.keys, padded = (p.n + 63) & ~63;
    if (p.n <= 64) {
        if (wave == 0) group_few(p, lane < p.n ? (local ? l.ids[lane] : p.ids[lane]) : -1, lane);
        return;
    }
    const bool small = p.n <= kGroupThreads;
    for (int i = tid; i < slots; i += kGroupThreads) at[i] = 0;
    __syncthreads();
    for (int i = tid; i < padded; i += kGroupThreads) {  // whole waves
        const int id = i < p.n ? (local ? l.ids[i] : p.ids[i]) : -1;
        const bool ok = id >= 0 && id < p.keys;
        if (i < p.n) {
            p.clean[i] = ok ? id : -1;
            if (small) l.ids[i] = id;
        }
        take_place(at, id, ok, lane);
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
        l.waves[0][wave] = rs;
        l.waves[1][wave] = cs;
    }
    __syncthreads();
    int total = 0, r0 = rs - rows, c0 = cs - chunks;
    for (int q = 0; q < kGroupThreads / 64; ++q) {
        if (q < wave) {
            r0 += l.waves[0][q];
            c0 += l.waves[1][q];
        }
        total += l.waves[1][q];
    }
    for (int q = k0, r = r0; q < k1; ++q) {  // counts become the next place
        const int count = at[q];
        at[q] = r;
        r += count;
    }
    __syncthreads();
    for (int i = tid; i < padded; i += kGroupThreads) {
        const int id = i < p.n ? (small ? l.ids[i] : p.ids[i]) : -1;
        const bool ok = id >= 0 && id < p.keys;
        const int place = take_place(at, id, ok, lane);
        if (ok) {
            p.order[place] = i;
            if (small) l.order[place] = i;
        }
    }
    __syncthreads();
    for (int q = k0; q < k1; ++q)  // and now the place behind the key's last row
        for (const int end = at[q]; r0 < end; r0 = min(r0 + p.chunk_rows, end))
            p.chunks[c0++] = Chunk{q, r0, min(p.chunk_rows, end - r0), small ? l.order[r0] : p.order[r0]};
    for (int i = total + tid; i < p.max_chunks; i += kGroupThreads) p.chunks[i] = Chunk{-1, 0, 0, 0};
}

// One workgroup groups; those behind it rotate rows.
template <typename T>
__global__ __launch_bounds__(kGroupThreads) void group_kernel(const GroupArgs p, const RotateArgs beside) {
    extern __shared__ int at[];  // [keys]: counts, then places
    __shared__ GroupLds l;
    if (blockIdx.x == 0)
        group_rows(p, at, l, false);
    else
        rotate_block<T>(beside, static_cast<int64_t>(blockIdx.x - 1) * (kGroupThreads / 64) +
                                    uniform(static_cast<int>(threadIdx.x >> 6)), threadIdx.x & 63);
}

// Choice and grouping of at most 16 tokens in one workgroup: a wave chooses for each token.
template <int kSlots>
__global__ __launch_bounds__(kGroupThreads) void choose_group_kernel(const ChooseArgs c, const GroupArgs p) {
    extern __shared__ int at[];
    __shared__ GroupLds l;
    const int wave = uniform(static_cast<int>(threadIdx.x >> 6));
    if (wave < c.tokens) choose<kSlots>(c, wave, threadIdx.x & 63, l.ids);
    __syncthreads();
    group_rows(p, at, l, true);
}

}  // namespace

int launch_group(const GroupArgs& args, const RotateArgs& beside, int dtype, hipStream_t stream) {
    const size_t lds = sizeof(int) * static_cast<size_t>(args.keys);
    const int64_t each = kGroupThreads / 64;
    const dim3 grid(static_cast<unsigned>(1 + (rotate_waves(beside) + each - 1) / each));
    if (dtype == 0)
        hipLaunchKernelGGL(group_kernel<__bf16>, grid, dim3(kGroupThreads), lds, stream, args, beside);
    else
        hipLaunchKernelGGL(group_kernel<_Float16>, grid, dim3(kGroupThreads), lds, stream, args, beside);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

namespace {
bool route_sizes(int64_t tokens, int64_t hidden, int64_t experts) {
    return tokens >= 0 && tokens <= 1 << 20 && hidden > 0 && hidden <= 1 << 24 && experts > 0 && experts <= kMaxExperts;
}
}  // namespace

const char* router_fault(const RouterArgs& a) {
    if (!a.x || !a.weight || !a.weights || !a.ids || a.tokens < 0 || a.hidden <= 0 || a.experts <= 0)
        return "null pointer or bad size in the router";
    if (a.dtype != 0 && a.dtype != 1) return "dtype must be 0 (bf16) or 1 (f16)";
    if (a.experts > kMaxExperts) return "the router takes at most 1024 experts";
    if (a.k < 1 || a.k > 64 || a.k > a.experts) return "k must be 1 .. min(64, experts)";
    if (a.scoring != 0 && a.scoring != 1) return "scoring must be 0 (softmax) or 1 (sigmoid)";
    const auto bad = [&](int rows, int64_t ld) { return rows > 1 && (ld % 8 || ld < a.hidden); };
    if (a.hidden % 8 || bad(a.tokens, a.x_ld) || bad(a.experts, a.weight_ld) ||
        reinterpret_cast<uintptr_t>(a.x) % 16 || reinterpret_cast<uintptr_t>(a.weight) % 16)
        return "the router's rows must be 16-byte aligned and a multiple of 8 channels";
    return nullptr;
}

size_t router_logit_bytes(int64_t tokens, int64_t hidden, int64_t experts) {
    return sizeof(float) * static_cast<size_t>(router_splits(tokens, hidden, experts)) * tokens * experts;
}

int64_t router_blocks(int64_t tokens, int64_t hidden, int64_t experts, const RotateArgs& beside) {
    return (experts + 15) / 16 * ((tokens + 15) / 16) * router_splits(tokens, hidden, experts) + (rotate_waves(beside) + 3) / 4;
}

int launch_router(const RouterArgs& a, const RotateArgs& beside, const GroupArgs* group, hipStream_t stream) {
    LogitsArgs la{a.x, a.weight, a.x_ld, a.weight_ld, a.tokens, a.hidden, a.experts,
                  router_splits(a.tokens, a.hidden, a.experts), (a.experts + 15) / 16, (a.tokens + 15) / 16, a.logits, beside};
    const int64_t blocks = router_blocks(a.tokens, a.hidden, a.experts, beside);
    if (a.dtype == 0)
        hipLaunchKernelGGL(router_logits_kernel<__bf16>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, la);
    else
        hipLaunchKernelGGL(router_logits_kernel<_Float16>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, la);
    QSRT_HIP_TRY(hipGetLastError());
    const ChooseArgs ca{a.logits, a.bias, a.tokens, a.experts, la.splits, a.k, a.scoring, a.normalize, a.scale, a.weights, a.ids};
    // Choice and grouping in one launch while one compute unit has the choices done sooner than a launch takes: a layer of
    // 384 experts 32 us for a token, apart 36; 8 tokens 77 and 79; 16 tokens 109, apart 107.5; of 64 experts, 16 tokens 65
    // and 66.  16 slots a lane do not fit the registers that a wave of a full workgroup has.
    const bool together = group && a.experts <= 512 && a.tokens <= (a.experts <= 128 ? kGroupThreads / 64 : 8);
#define QSRT_CHOOSE(SLOTS)                                                                                             \
    if (together)                                                                                                      \
        hipLaunchKernelGGL(choose_group_kernel<SLOTS>, dim3(1), dim3(kGroupThreads), sizeof(int) * group->keys,      \
                           stream, ca, *group);                                                                        \
    else                                                                                                               \
        hipLaunchKernelGGL(choose_kernel<SLOTS>, dim3(static_cast<unsigned>(a.tokens)), dim3(64), 0, stream, ca)
    if (a.experts <= 64) {
        QSRT_CHOOSE(1);
    } else if (a.experts <= 128) {
        QSRT_CHOOSE(2);
    } else if (a.experts <= 256) {
        QSRT_CHOOSE(4);
    } else if (a.experts <= 384) {
        QSRT_CHOOSE(6);
    } else if (a.experts <= 512) {
        QSRT_CHOOSE(8);
    } else {
        hipLaunchKernelGGL(choose_kernel<16>, dim3(static_cast<unsigned>(a.tokens)), dim3(64), 0, stream, ca);
    }
#undef QSRT_CHOOSE
    QSRT_HIP_TRY(hipGetLastError());
    return group && !together ? launch_group(*group, RotateArgs{}, a.dtype, stream) : kOk;
}

}  // namespace qsrt

using namespace qsrt;

extern "C" size_t qsrt_route_workspace_bytes(int64_t tokens, int64_t hidden, int64_t experts) {
    if (tokens == 0 || !route_sizes(tokens, hidden, experts)) return 0;
    return router_logit_bytes(tokens, hidden, experts);
}

extern "C" int qsrt_route(const void* x, int64_t x_ld, const void* weight, int64_t weight_ld, int dtype, int64_t tokens,
                          int64_t hidden, int64_t experts, int k, const float* bias, int scoring, int normalize,
                          float scale, float* weights, int32_t* ids, void* ws, size_t ws_bytes, void* stream) {
    if (tokens == 0) return kOk;
    if (!route_sizes(tokens, hidden, experts))
        return fail(kBadArgument, "qsrt_route: bad sizes (at most 2^20 tokens, 2^24 channels, %d experts)", kMaxExperts);
    const RouterArgs args{x, x_ld, weight, weight_ld, dtype, static_cast<int>(tokens), static_cast<int>(hidden),
                          static_cast<int>(experts), k, bias, scoring, normalize, scale, weights, ids,
                          static_cast<float*>(ws)};
    if (const char* e = router_fault(args)) return fail(kBadArgument, "qsrt_route: %s", e);
    const size_t need = router_logit_bytes(tokens, hidden, experts);
    if (!ws || ws_bytes < need) return fail(kWorkspaceTooSmall, "qsrt_route: needs %zu workspace bytes", need);
    return launch_router(args, RotateArgs{}, nullptr, static_cast<hipStream_t>(stream));
}

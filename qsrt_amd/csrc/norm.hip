// What stands between two blocks of a model: the norm behind the first, its gate, the residual with its scale and the norm
// before the second, in one pass over the rows; and its gradients in another (gfx950, wave64).
//
//   z = post * y sy, sy = (mean y^2 + eps)^-1/2   (without post: z = y)
//   h = scale * residual + gate * z
//   n = weight * h sh, sh = (mean h^2 + eps)^-1/2
//
// Bound by memory: a row stays in registers between its loads and its stores, sums and statistics are FP32, n comes from h
// before h is rounded.  The gradients, with e = weight * dn, p = post * gate and hhat = h sh (no higher power of sh stands alone:
// rows of 1e13 or, with a small eps, 1e-13 would end FP32's range there, where their gradients do not):
//   dh = dsum + sh (e - hhat mean(e hhat)),  dresidual = scale dh,  dz = gate dh
//   dy = sy (post dz - yhat mean(post dz yhat)),  yhat = y sy
//   dweight = sum over rows of dn hhat,  dpost of dz yhat,  dgate of dh z (a row's own gate: over its channels)
// mean(post dz yhat) is put together from sums that do not wait for mean(e hhat), so a row meets once:
//   sum p yhat dh = sum p yhat (dsum + sh e) - sh mean(e hhat) sum p yhat hhat
// and a gate for each channel shares its sum over the rows with post: dpost = gate S, dgate = post S, S = sum of dh yhat.
#include <algorithm>

#include "common.h"
#include "qsrt_amd.h"

namespace qsrt {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
template <typename T>
using vec8 = T __attribute__((ext_vector_type(8)));

constexpr int64_t kMaxRows = 1 << 22, kMaxHidden = 1 << 14;
enum Gate { kNone, kChannel, kRow };

struct NormArgs {
    const void *residual, *y, *weight, *post, *gate;
    int64_t residual_ld, y_ld, rows;
    int hidden, gate_kind;
    bool residual_f32, params_f32;
    float scale, eps;
    void *sum, *normed;  // sum may be null
    int64_t sum_ld, normed_ld;
    float* stats;  // [2][rows]: sy (1 without post) and sh; null where no gradient is to follow
    // backward
    const void *dsum, *dn;  // one may be null
    int64_t dsum_ld, dn_ld;
    void *dresidual, *dy;  // either may be null
    int64_t dresidual_ld, dy_ld;
    float* partial;       // [workgroup][2][hidden]: dweight, S
    void* drow;           // [rows], of a row's own gate; or null
};

__device__ __forceinline__ f32x8 load_f32(const void* p, int64_t at) {
    const f32x4* q = reinterpret_cast<const f32x4*>(static_cast<const float*>(p) + at);
    const f32x4 a = q[0], b = q[1];
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
}
template <typename T>
__device__ __forceinline__ f32x8 load8(const void* p, int64_t at, bool f32) {
    if (f32) return load_f32(p, at);
    return __builtin_convertvector(*reinterpret_cast<const vec8<T>*>(static_cast<const T*>(p) + at), f32x8);
}
template <typename T>
__device__ __forceinline__ void store8(void* p, int64_t at, const f32x8& v, bool f32) {
    if (f32) {
        f32x4* q = reinterpret_cast<f32x4*>(static_cast<float*>(p) + at);
        q[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
        q[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    } else {
        *reinterpret_cast<vec8<T>*>(static_cast<T*>(p) + at) = __builtin_convertvector(v, vec8<T>);
    }
}
template <typename T>
__device__ __forceinline__ float load1(const void* p, int64_t at, bool f32) {
    return f32 ? static_cast<const float*>(p)[at] : static_cast<float>(static_cast<const T*>(p)[at]);
}
__device__ __forceinline__ float total(const f32x8& v) { return ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7])); }

template <int kControl>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), kControl, 0xF, 0xF, true));
}
// The sum over 16 lanes, in each of them: neighbours, pairs, then mirrors of 8 and 16.
__device__ __forceinline__ float sum16(float v) {
    v += dpp<0xB1>(v);
    v += dpp<0x4E>(v);
    v += dpp<0x141>(v);
    return v + dpp<0x140>(v);
}
__device__ __forceinline__ float sum64(float v) {
    v = sum16(v);
    uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, static_cast<uint32_t>(rows[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(rows[1]));
    u = __builtin_bit_cast(uint32_t, v);
    const auto halves = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, static_cast<uint32_t>(halves[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(halves[1]));
}

constexpr int kMaxWaves = 16;
// The sums of kSums values over a workgroup, in every thread.  `room` starts at zero (the waves that are not there) and has
// two sets that are used in turn, so one barrier a call is enough.
template <int kSums>
__device__ __forceinline__ void meet(float (&v)[kSums], float (*room)[kMaxWaves], int lane, int wave) {
#pragma unroll
    for (int s = 0; s < kSums; ++s) {
        v[s] = sum64(v[s]);
        if (lane == 0) room[s][wave] = v[s];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < kSums; ++s) v[s] = sum16(room[s][lane & 15]);
}

// Eight values as they lie in memory: the next row's are on their way while a row is computed.
template <typename T, bool kF32>
struct Packed {
    vec8<T> v;
    __device__ __forceinline__ void load(const void* p, int64_t at) {
        v = *reinterpret_cast<const vec8<T>*>(static_cast<const T*>(p) + at);
    }
    __device__ __forceinline__ f32x8 get() const { return __builtin_convertvector(v, f32x8); }
};
template <typename T>
struct Packed<T, true> {
    f32x8 v;
    __device__ __forceinline__ void load(const void* p, int64_t at) { v = load_f32(p, at); }
    __device__ __forceinline__ f32x8 get() const { return v; }
};

// A workgroup walks the rows in strides, eight channels a thread and step, in as many waves as a row needs; the next row is on
// its way while this one meets.  4096 rows of 7168, the residual in 32 bits: 75 us, 4.7 TB/s, as a large copy (4.6); 8192 of
// 5120 in 16 bits 76 to 84; one row 4.2, its launch and two round trips.
template <typename T, int kSteps, bool kF32>
__global__ __launch_bounds__(1024) void norm_kernel(const NormArgs p) {
    __shared__ float room[2][1][kMaxWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, threads = blockDim.x;
    if (threadIdx.x < 2 * kMaxWaves) room[0][0][threadIdx.x] = 0.f;
    Packed<T, false> y[kSteps];
    Packed<T, kF32> residual[kSteps];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
            if (c >= p.hidden) continue;
            residual[s].load(p.residual, row * p.residual_ld + c);
            if (p.y) y[s].load(p.y, row * p.y_ld + c);
        }
    };
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        residual[s] = {};
        y[s] = {};
    }
    fetch(blockIdx.x);
    __syncthreads();
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        f32x8 r[kSteps], z[kSteps];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            r[s] = residual[s].get();
            z[s] = y[s].get();
        }
        if (row + gridDim.x < p.rows) fetch(row + gridDim.x);
        float sy = 1.f;
        if (p.post) {
            float v[1] = {0.f};
#pragma unroll
            for (int s = 0; s < kSteps; ++s) v[0] += total(z[s] * z[s]);
            meet(v, room[turn], lane, wave);
            turn ^= 1;
            sy = 1.0f / sqrtf(v[0] / static_cast<float>(p.hidden) + p.eps);
        }
        const float row_gate = p.gate_kind == kRow ? load1<T>(p.gate, row, p.params_f32) : 1.f;
        float v[1] = {0.f};
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
            if (c >= p.hidden) continue;
            if (p.post) z[s] = z[s] * sy * load8<T>(p.post, c, p.params_f32);
            if (p.gate_kind == kChannel) z[s] = z[s] * load8<T>(p.gate, c, p.params_f32);
            r[s] = p.scale * r[s] + row_gate * z[s];
            if (p.sum) store8<T>(p.sum, row * p.sum_ld + c, r[s], kF32);
            v[0] += total(r[s] * r[s]);
        }
        meet(v, room[turn], lane, wave);
        turn ^= 1;
        const float sh = 1.0f / sqrtf(v[0] / static_cast<float>(p.hidden) + p.eps);
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
            if (c < p.hidden) store8<T>(p.normed, row * p.normed_ld + c, r[s] * sh * load8<T>(p.weight, c, p.params_f32), false);
        }
        if (p.stats && threadIdx.x == 0) {
            p.stats[row] = sy;
            p.stats[p.rows + row] = sh;
        }
    }
}

// The same walk; sums over rows stay in registers until the end.  8192 rows of 5120: 109 us, 4.6 TB/s; without y (a first norm)
// 78, 3.2 TB/s.  Rows over 8192 channels take two steps, which do not fit the 128 registers that 16 waves leave a thread: the
// parameters and the next row are loaded where they are used, and of the sums, yhat, hhat and d 248 bytes a thread are spilled to
// scratch (328 with a residual in 32 bits).  2048 rows of 16384: 195 to 200 us, 2.0 TB/s; 270 in 32 bits, 2.2.
template <typename T, int kSteps, bool kF32>
__global__ __launch_bounds__(1024) void norm_gradients_kernel(const NormArgs p) {
    __shared__ float room[2][3][kMaxWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, threads = blockDim.x;
    if (threadIdx.x < 64)
        for (int i = lane; i < 2 * 3 * kMaxWaves; i += 64) room[0][0][i] = 0.f;
    const f32x8 zero = {};
    constexpr bool kKeep = kSteps == 1;
    f32x8 by_weight[kSteps], by_scale[kSteps], kept_weight, kept_pz;
    const auto weight_at = [&](int c) { return load8<T>(p.weight, c, p.params_f32); };
    const auto pz_at = [&](int c) {  // what z is yhat's multiple by, the row's gate apart
        f32x8 v = zero + 1.f;
        if (p.post) v = load8<T>(p.post, c, p.params_f32);
        return p.gate_kind == kChannel ? v * load8<T>(p.gate, c, p.params_f32) : v;
    };
    Packed<T, false> y[kSteps], dn[kSteps];
    Packed<T, kF32> residual[kSteps], dsum[kSteps];
    const auto fetch = [&](int64_t row) {
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
            if (c >= p.hidden) continue;
            residual[s].load(p.residual, row * p.residual_ld + c);
            if (p.y) y[s].load(p.y, row * p.y_ld + c);
            if (p.dn) dn[s].load(p.dn, row * p.dn_ld + c);
            if (p.dsum) dsum[s].load(p.dsum, row * p.dsum_ld + c);
        }
    };
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
        by_weight[s] = by_scale[s] = kept_weight = kept_pz = zero;
        residual[s] = dsum[s] = {};
        y[s] = dn[s] = {};
        if (!kKeep || c >= p.hidden) continue;
        kept_weight = weight_at(c);
        kept_pz = pz_at(c);
    }
    if (kKeep) fetch(blockIdx.x);
    __syncthreads();
    const float mean = 1.0f / static_cast<float>(p.hidden);
    int turn = 0;
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        const float sy = p.stats[row], sh = p.stats[p.rows + row];
        const float row_gate = p.gate_kind == kRow ? load1<T>(p.gate, row, p.params_f32) : 1.f;
        if (!kKeep) fetch(row);
        f32x8 yhat[kSteps], hhat[kSteps], d[kSteps];  // d: dsum + sh e, dh but for the row's mean
        float v[3] = {0.f, 0.f, 0.f};  // e hhat, z d, z hhat, without a row's gate: its gradient needs the same sums
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
            yhat[s] = hhat[s] = d[s] = zero;
            if (c >= p.hidden) continue;
            const f32x8 weight = kKeep ? kept_weight : weight_at(c), pz = kKeep ? kept_pz : pz_at(c);
            yhat[s] = y[s].get() * sy;
            const f32x8 z = yhat[s] * pz;
            hhat[s] = (p.scale * residual[s].get() + row_gate * z) * sh;
            const f32x8 n = dn[s].get(), e = n * weight;
            by_weight[s] += n * hhat[s];
            d[s] = dsum[s].get() + e * sh;
            v[0] += total(e * hhat[s]);
            v[1] += total(z * d[s]);
            v[2] += total(z * hhat[s]);
        }
        if (kKeep && row + gridDim.x < p.rows) fetch(row + gridDim.x);
        meet(v, room[turn], lane, wave);
        const float back = sh * (v[0] * mean);
        const float by_z = v[1] - back * v[2];  // the sum of z dh
        const float shared = p.post ? by_z * row_gate * mean : 0.f;
        if (p.drow && threadIdx.x == 0) {
            if (p.params_f32)
                static_cast<float*>(p.drow)[row] = by_z;
            else
                static_cast<T*>(p.drow)[row] = static_cast<T>(by_z);
        }
#pragma unroll
        for (int s = 0; s < kSteps; ++s) {
            const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
            if (c >= p.hidden) continue;
            const f32x8 dh = d[s] - hhat[s] * back;
            if (p.dresidual) store8<T>(p.dresidual, row * p.dresidual_ld + c, p.scale * dh, kF32);
            const f32x8 dz = row_gate * dh;
            by_scale[s] += dz * yhat[s];
            if (p.dy) store8<T>(p.dy, row * p.dy_ld + c, sy * (dz * (kKeep ? kept_pz : pz_at(c)) - yhat[s] * shared), false);
        }
    }
    float* to = p.partial + static_cast<int64_t>(blockIdx.x) * 2 * p.hidden;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
        const int c = (s * threads + static_cast<int>(threadIdx.x)) * 8;
        if (c >= p.hidden) continue;
        store8<T>(to, c, by_weight[s], true);
        store8<T>(to, p.hidden + c, by_scale[s], true);
    }
}

// Adds the workgroups' sums, 32 channels a workgroup: thread (c, q) every 32nd from q, then those in pairs.  256 sums of 5120
// channels and two planes in 4.7 us.
struct JoinArgs {
    const float* partial;
    int64_t groups;
    int hidden;
    const void *post, *gate;
    void *dweight, *dpost, *dgate;  // any may be null
    bool f32;
};
template <typename T>
__global__ __launch_bounds__(1024) void norm_join_kernel(const JoinArgs p) {
    __shared__ float sums[32][33];
    const int c = threadIdx.x & 31, q = threadIdx.x >> 5, which = blockIdx.y;
    const int64_t channel = static_cast<int64_t>(blockIdx.x) * 32 + c;
    float v = 0.f;
    if (channel < p.hidden)
#pragma unroll 4
        for (int64_t g = q; g < p.groups; g += 32) v += p.partial[(g * 2 + which) * p.hidden + channel];
    sums[q][c] = v;
    __syncthreads();
    // the transposed pair: thread (q, c) now holds part c of channel q
    v = sum16(sums[c][q]);
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __builtin_bit_cast(float, static_cast<uint32_t>(rows[0])) + __builtin_bit_cast(float, static_cast<uint32_t>(rows[1]));
    const int64_t at = static_cast<int64_t>(blockIdx.x) * 32 + q;
    if (c || at >= p.hidden) return;
    const auto put = [&](void* out, float value) {
        if (!out) return;
        if (p.f32)
            static_cast<float*>(out)[at] = value;
        else
            static_cast<T*>(out)[at] = static_cast<T>(value);
    };
    if (which == 0) {
        put(p.dweight, v);
    } else {
        put(p.dpost, p.gate ? load1<T>(p.gate, at, p.f32) * v : v);
        put(p.dgate, p.post ? load1<T>(p.post, at, p.f32) * v : v);
    }
}

// ---------------------------------------------------------------- host
// Eight channels a thread, in whole waves; over 8192 channels twice.
unsigned row_threads(int hidden) {
    const int each = hidden <= 8192 ? 512 : 1024;  // channels of a wave
    return 64 * static_cast<unsigned>((hidden + each - 1) / each);
}

// Workgroups of the gradients: 16 waves a compute unit, as many as its registers hold, but two workgroups, or four where each
// has eight rows: a workgroup leaves 8 bytes a channel behind for the second kernel.  Both kernels, in us with one, two and four
// a compute unit: 8192 rows of 1024 channels 51.6, 36.4, 30.0, 1024 rows 12.9, 12.1, 14.2; 8192 rows of 4096 98.7, 91.7, 92.6,
// of 5120 114.2, 120.1, 126.8; 1024 rows of 7168 25.3, 33.3, 47.7.
int64_t gradient_groups(int64_t rows, int64_t hidden) {
    int cus = 0;
    if (current_cu_count(&cus) != kOk) cus = 256;
    const int64_t fit = 1024 / row_threads(static_cast<int>(hidden)), most = rows >= 32 * cus ? 4 : 2;
    return std::min<int64_t>(rows, cus * std::min(fit, most));
}

// Workgroups that the chip holds at a time: 32 waves a compute unit.  With half or twice as many, 4096 rows of 7168 take 73 and
// 79 us for 75, 8192 of 5120 91 and 81 for 84.
int64_t row_groups(int hidden) {
    int cus = 0;
    if (current_cu_count(&cus) != kOk) cus = 256;
    return static_cast<int64_t>(cus) * (2048 / row_threads(hidden));
}

int check_rows(const char* call, const void* p, int64_t ld, int64_t rows, int64_t hidden, const char* name) {
    if (!p) return fail(kBadArgument, "%s: null pointer for %s", call, name);
    if (reinterpret_cast<uintptr_t>(p) % 16 || (rows > 1 && (ld % 8 || ld < hidden)))
        return fail(kBadArgument, "%s: rows of %s must be whole and 16-byte aligned", call, name);
    return kOk;
}
int check_norm(const char* call, const NormArgs& a, int dtype) {
    if (a.rows < 0 || a.rows > kMaxRows || a.hidden <= 0 || a.hidden % 8)
        return fail(kBadArgument, "%s: at most 2^22 rows, and channels in multiples of 8 up to 2^14", call);
    if (dtype != 0 && dtype != 1) return fail(kBadArgument, "%s: dtype must be 0 (bf16) or 1 (f16)", call);
    if (a.gate_kind < kNone || a.gate_kind > kRow) return fail(kBadArgument, "%s: gate must be 0 (none), 1 (channels) or 2 (rows)", call);
    if ((a.gate_kind != kNone) != (a.gate != nullptr)) return fail(kBadArgument, "%s: a gate needs its kind and its values", call);
    if (!a.y && (a.post || a.gate)) return fail(kBadArgument, "%s: without y there is nothing to norm or gate before the sum", call);
    if (!(a.eps >= 0.f)) return fail(kBadArgument, "%s: eps must not be negative", call);
    if (a.rows == 0) return kOk;
    if (int rc = check_rows(call, a.residual, a.residual_ld, a.rows, a.hidden, "residual")) return rc;
    if (a.y)
        if (int rc = check_rows(call, a.y, a.y_ld, a.rows, a.hidden, "y")) return rc;
    for (const void* v : {a.weight, a.post, a.gate_kind == kChannel ? a.gate : nullptr})
        if (reinterpret_cast<uintptr_t>(v) % 16) return fail(kBadArgument, "%s: weights must be 16-byte aligned", call);
    if (!a.weight) return fail(kBadArgument, "%s: null pointer for weight", call);
    return kOk;
}

}  // namespace
}  // namespace qsrt

using namespace qsrt;

extern "C" int qsrt_residual_norm(const void* residual, int64_t residual_ld, int residual_f32, const void* y, int64_t y_ld, int dtype,
                                  int64_t rows, int64_t hidden, const void* weight, const void* post, const void* gate,
                                  int gate_kind, int params_f32, float scale, float eps, void* sum, int64_t sum_ld, void* normed,
                                  int64_t normed_ld, float* stats, void* stream) {
    constexpr const char* kCall = "qsrt_residual_norm";
    NormArgs a = {};
    a.residual = residual, a.residual_ld = residual_ld, a.residual_f32 = residual_f32 != 0;
    a.y = y, a.y_ld = y_ld, a.rows = rows, a.hidden = hidden < 0 || hidden > kMaxHidden ? -1 : static_cast<int>(hidden);
    a.weight = weight, a.post = post, a.gate = gate, a.gate_kind = gate_kind, a.params_f32 = params_f32 != 0;
    a.scale = scale, a.eps = eps, a.sum = sum, a.sum_ld = sum_ld, a.normed = normed, a.normed_ld = normed_ld, a.stats = stats;
    if (int rc = check_norm(kCall, a, dtype)) return rc;
    if (rows == 0) return kOk;
    if (sum)
        if (int rc = check_rows(kCall, sum, sum_ld, rows, hidden, "sum")) return rc;
    if (int rc = check_rows(kCall, normed, normed_ld, rows, hidden, "normed")) return rc;
    const dim3 grid(static_cast<unsigned>(std::min<int64_t>(rows, row_groups(a.hidden))));
    const auto s = static_cast<hipStream_t>(stream);
    const dim3 threads(row_threads(a.hidden));
#define QSRT_NORM(STEPS, F32)                                                                                    \
    if (dtype == 0)                                                                                              \
        hipLaunchKernelGGL((norm_kernel<__bf16, STEPS, F32>), grid, threads, 0, s, a);                           \
    else                                                                                                         \
        hipLaunchKernelGGL((norm_kernel<_Float16, STEPS, F32>), grid, threads, 0, s, a)
    if (hidden <= 8192) {
        if (a.residual_f32) {
            QSRT_NORM(1, true);
        } else {
            QSRT_NORM(1, false);
        }
    } else if (a.residual_f32) {
        QSRT_NORM(2, true);
    } else {
        QSRT_NORM(2, false);
    }
#undef QSRT_NORM
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

extern "C" size_t qsrt_residual_norm_backward_workspace_bytes(int64_t rows, int64_t hidden) {
    if (rows <= 0 || rows > kMaxRows || hidden <= 0 || hidden > kMaxHidden || hidden % 8) return 0;
    return sizeof(float) * 2 * static_cast<size_t>(gradient_groups(rows, hidden) * hidden);
}

extern "C" int qsrt_residual_norm_backward(const void* dsum, int64_t dsum_ld, const void* dn, int64_t dn_ld, const void* residual,
                                           int64_t residual_ld, int residual_f32, const void* y, int64_t y_ld, int dtype,
                                           int64_t rows, int64_t hidden, const void* weight, const void* post, const void* gate,
                                           int gate_kind, int params_f32, float scale, const float* stats, void* dresidual,
                                           int64_t dresidual_ld, void* dy, int64_t dy_ld, void* dweight, void* dpost, void* dgate,
                                           void* ws, size_t ws_bytes, void* stream) {
    constexpr const char* kCall = "qsrt_residual_norm_backward";
    NormArgs a = {};
    a.residual = residual, a.residual_ld = residual_ld, a.residual_f32 = residual_f32 != 0;
    a.y = y, a.y_ld = y_ld, a.rows = rows, a.hidden = hidden < 0 || hidden > kMaxHidden ? -1 : static_cast<int>(hidden);
    a.weight = weight, a.post = post, a.gate = gate, a.gate_kind = gate_kind, a.params_f32 = params_f32 != 0;
    a.scale = scale, a.stats = const_cast<float*>(stats);
    a.dsum = dsum, a.dsum_ld = dsum_ld, a.dn = dn, a.dn_ld = dn_ld;
    a.dresidual = dresidual, a.dresidual_ld = dresidual_ld, a.dy = dy, a.dy_ld = dy_ld;
    a.drow = gate_kind == kRow ? dgate : nullptr;
    if (int rc = check_norm(kCall, a, dtype)) return rc;
    if (rows == 0) return kOk;
    if (!stats) return fail(kBadArgument, "%s: null pointer for stats", kCall);
    if (!y && (dy || dpost || dgate)) return fail(kBadArgument, "%s: no gradients of y, post or gate without y", kCall);
    if ((dpost && !post) || (dgate && !gate)) return fail(kBadArgument, "%s: no gradient of what is not there", kCall);
    const struct { const void* p; int64_t ld; const char* name; } given[] = {
        {dsum, dsum_ld, "dsum"}, {dn, dn_ld, "dn"}, {dresidual, dresidual_ld, "dresidual"}, {dy, dy_ld, "dy"}};
    for (const auto& g : given)
        if (g.p)
            if (int rc = check_rows(kCall, g.p, g.ld, rows, hidden, g.name)) return rc;
    const size_t need = qsrt_residual_norm_backward_workspace_bytes(rows, hidden);
    if (!ws || ws_bytes < need) return fail(kWorkspaceTooSmall, "%s: needs %zu workspace bytes", kCall, need);
    if (reinterpret_cast<uintptr_t>(ws) % 16) return fail(kBadArgument, "%s: the workspace must be 16-byte aligned", kCall);
    a.partial = static_cast<float*>(ws);
    const int64_t groups = gradient_groups(rows, hidden);
    const dim3 grid(static_cast<unsigned>(groups));
    const auto s = static_cast<hipStream_t>(stream);
    const dim3 threads(row_threads(a.hidden));
#define QSRT_NORM(STEPS, F32)                                                                                    \
    if (dtype == 0)                                                                                              \
        hipLaunchKernelGGL((norm_gradients_kernel<__bf16, STEPS, F32>), grid, threads, 0, s, a);                 \
    else                                                                                                         \
        hipLaunchKernelGGL((norm_gradients_kernel<_Float16, STEPS, F32>), grid, threads, 0, s, a)
    if (hidden <= 8192) {
        if (a.residual_f32) {
            QSRT_NORM(1, true);
        } else {
            QSRT_NORM(1, false);
        }
    } else if (a.residual_f32) {
        QSRT_NORM(2, true);
    } else {
        QSRT_NORM(2, false);
    }
#undef QSRT_NORM
    QSRT_HIP_TRY(hipGetLastError());
    const bool channels = gate_kind == kChannel;
    const JoinArgs j{a.partial, groups, a.hidden, post, channels ? gate : nullptr, dweight, dpost, channels ? dgate : nullptr,
                     a.params_f32};
    if (!j.dweight && !j.dpost && !j.dgate) return kOk;
    const dim3 columns(static_cast<unsigned>((hidden + 31) / 32), 2);
    if (dtype == 0)
        hipLaunchKernelGGL(norm_join_kernel<__bf16>, columns, dim3(1024), 0, s, j);
    else
        hipLaunchKernelGGL(norm_join_kernel<_Float16>, columns, dim3(1024), 0, s, j);
    QSRT_HIP_TRY(hipGetLastError());
    return kOk;
}

// voxel_attention.h -- attention among the rows of a window (voxel_windows.h): the kernel, for FP16 and FP32 tensors.
//
// A workgroup of four waves takes up to 64 queries of one window and a few heads, and walks over the window's keys in blocks of 64 (32
// where a head's values are many).  Keys, values and voxels of a block lie in LDS; those of the next one are gathered into registers in
// the meantime.  A wave has 16 queries; where the window has fewer than 64, waves share queries and deal the heads out.  Windows of up to
// 32 rows are a wave's own affair: their queries are their keys, which it keeps in registers, and nobody waits for anybody.  Where there are
// few queries, a workgroup has 16 of them and its waves share the keys out (shared_rows).
//
// What bounds it are vector instructions, 56 to 110 cycles for a wave's 64 scores (a distance 52, which two heads may share, a cap 28, exponential,
// maximum and sums 30), not the matrix cores, nor memory: 30 000 keys, 8 heads of 64 values, cap and distances 5.3 ms (350 TFLOP/s of products),
// 53 000 rows in windows of 16 x 16, 8 heads of 32 102 us; FP32, where the products take longer, 4 741 keys, 16 heads of 64 1.27 ms (73 TFLOP/s).
//
// Scores are taken transposed, S^T = K Q^T: a lane of the result has one query (its column) and four keys, so that maximum and sum over the
// keys are mostly the lane's own, and the weights are where the second product, O^T = V^T P^T, wants them.  Maximum and sum run along
// with the blocks; sums that are there already are rescaled only where a block raises a maximum.
#pragma once

#include <type_traits>

#include "voxel_windows.h"

namespace sessd {

struct AttentionArgs {
    const void* qkv;
    void* out;
    const float* slopes;  // or null
    WindowIndex w;
    int heads, kv_heads, dim;
    // A weight is 2^(by z - by max z), by > 0, z = f(q.k) - slope * to_slope * distance
    float by, to_slope;
    bool negate;          // the scale of the scores is negative: queries change their sign
    bool capped, series;  // series: small scores by the first terms of the series, the exponential form is not exact enough
    float in_cap;         // tanh(u) is taken of u = scale * q.k / cap: 2 u to the base 2 is q.k times this
    float cell_x, cell_y, cell_z;
    int write_pad;
};

int launch_attention_half(const AttentionArgs& a, hipStream_t stream);
int launch_attention_float(const AttentionArgs& a, hipStream_t stream);
#ifdef __HIPCC__

constexpr int kAttentionBlock = 256;
constexpr float kLog2e = 1.44269504088896340736f;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

// over the four lanes that have a query: lane, lane + 16, + 32, + 48
__device__ __forceinline__ float most_of_query(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum_of_query(float x) {
    auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

// Operands.  A row of keys or values in LDS is kPitch elements; kPer neighbouring values are 16 bytes.
template <typename T, int DP> struct Operand;

template <int DP> struct Operand<_Float16, DP> {
    static constexpr int kPer = 8, kPitch = DP + 8, kParts = DP >= 32 ? DP / 32 : 1;
    // 16x16x32: of row lane % 16 the eight values from 32 s + 8 (lane / 16) on; 16x16x16 where a head has 16 values: four from 4 (lane / 16)
    typedef std::conditional_t<(DP >= 32), v8h, v4h> Part;
    struct Row {
        Part part[kParts];
    };
    // a row's values in memory, zeros behind the last one
    static __device__ __forceinline__ Row load(const _Float16* p, int dim, int g) {
        constexpr int kEach = DP >= 32 ? 8 : 4;
        Row q;
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            q.part[s] = Part{};
            if (s * 32 + g * kEach < dim) q.part[s] = *reinterpret_cast<const Part*>(p + s * 32 + g * kEach);
        }
        return q;
    }
    static __device__ __forceinline__ v4f product(const Part& k, const Part& q, v4f acc) {
        if constexpr (DP >= 32) return __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q, acc, 0, 0, 0);
        else return __builtin_amdgcn_mfma_f32_16x16x16f16(k, q, acc, 0, 0, 0);
    }
    // 16 keys times 16 queries; keys in LDS from `k` on, or in registers
    static __device__ __forceinline__ v4f scores(const _Float16* k, const Row& q, int r, int g) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) acc = product(*reinterpret_cast<const Part*>(k + r * kPitch + s * 32 + g * (DP >= 32 ? 8 : 4)), q.part[s], acc);
        return acc;
    }
    static __device__ __forceinline__ v4f scores(const Row& k, const Row& q) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) acc = product(k.part[s], q.part[s], acc);
        return acc;
    }
    // A weight is held times 2^14.  The largest one of a row is that, and what is below FP16's steps is below 2^-39 of it: times 1, thousands of keys
    // of 2^-25 would come to nothing, or to twice what they are.  (The factor is an addend that the exponent's fma has room for, and drops out with the sum.)
    static constexpr float kLargest = 14.f;
    // The weights of 16 H keys, rounded to 11 bits: the product's own operands are FP16.  Their sum is taken by a product with ones, of the
    // weights as they are rounded.
    template <int H> struct Weights {
        std::conditional_t<H == 1, v4h, v8h> p[(H + 1) / 2];
        __device__ __forceinline__ Weights(const v4f (&z)[H]) {
#pragma unroll
            for (int e = 0; e < 4 * H; ++e) p[e / 8][e % 8] = (_Float16)z[e / 4][e % 4];
        }
    };
    typedef v4f Sum;
    template <int H> static __device__ __forceinline__ Sum add(Sum s, const Weights<H>& w) {
        constexpr _Float16 k1 = 1;
        if constexpr (H == 1) return __builtin_amdgcn_mfma_f32_16x16x16f16(v4h{k1, k1, k1, k1}, w.p[0], s, 0, 0, 0);
        else
#pragma unroll
            for (int t = 0; t < H / 2; ++t) s = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8h{k1, k1, k1, k1, k1, k1, k1, k1}, w.p[t], s, 0, 0, 0);
        return s;
    }
    static __device__ __forceinline__ float sum(const Sum& s) { return s[0]; }
    // sums of 16 values from 16 b on over 16 H keys: LDS transposes four keys' values as it reads them, a lane gets value lane % 16 of keys
    // 4 (lane / 16) .. + 3 of each 16, which is where its weights are
    template <int H> static __device__ __forceinline__ v4f values(const _Float16* v, const Weights<H>& w, v4f acc, int b, int r, int g) {
        typedef __attribute__((address_space(3))) v4s* lds;
        const _Float16* p = v + (4 * g + (r >> 2)) * kPitch + 16 * b + (r & 3) * 4;
        if constexpr (H == 1) {
            return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)p)), w.p[0], acc, 0, 0, 0);
        } else {
#pragma unroll
            for (int t = 0; t < H / 2; ++t) {
                const v4h x = __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + 32 * t * kPitch)));
                const v4h y = __builtin_bit_cast(v4h, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + (32 * t + 16) * kPitch)));
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(v8h{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, w.p[t], acc, 0, 0, 0);
            }
            return acc;
        }
    }
    static __device__ __forceinline__ void store(_Float16* p, v4f x) { *reinterpret_cast<v4h*>(p) = v4h{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]}; }
};

template <int DP> struct Operand<float, DP> {
    static constexpr int kPer = 4, kPitch = DP + 4, kParts = DP / 16;
    static constexpr float kLargest = 0.f;
    // 16x16x4: the j-th instruction of a part takes value 16 s + 4 (lane / 16) + j
    struct Row {
        v4f part[kParts];
    };
    static __device__ __forceinline__ Row load(const float* p, int dim, int g) {
        Row q;
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            q.part[s] = v4f{0, 0, 0, 0};
            if (s * 16 + g * 4 < dim) q.part[s] = *reinterpret_cast<const v4f*>(p + s * 16 + g * 4);
        }
        return q;
    }
    static __device__ __forceinline__ v4f product(const v4f& k, const v4f& q, v4f acc) {
#pragma unroll
        for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(k[j], q[j], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ v4f scores(const float* k, const Row& q, int r, int g) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) acc = product(*reinterpret_cast<const v4f*>(k + r * kPitch + s * 16 + g * 4), q.part[s], acc);
        return acc;
    }
    static __device__ __forceinline__ v4f scores(const Row& k, const Row& q) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) acc = product(k.part[s], q.part[s], acc);
        return acc;
    }
    template <int H> struct Weights {
        v4f p[H];
        __device__ __forceinline__ Weights(const v4f (&z)[H]) {
#pragma unroll
            for (int t = 0; t < H; ++t) p[t] = z[t];
        }
    };
    typedef float Sum;
    template <int H> static __device__ __forceinline__ Sum add(Sum s, const Weights<H>& w) {
        float x = 0.f;
#pragma unroll
        for (int t = 0; t < H; ++t) x += (w.p[t][0] + w.p[t][1]) + (w.p[t][2] + w.p[t][3]);
        return s + x;
    }
    static __device__ __forceinline__ float sum(const Sum& s) { return sum_of_query(s); }
    template <int H> static __device__ __forceinline__ v4f values(const float* v, const Weights<H>& w, v4f acc, int b, int r, int g) {
#pragma unroll
        for (int t = 0; t < H; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc = __builtin_amdgcn_mfma_f32_16x16x4f32(v[(16 * t + 4 * g + e) * kPitch + 16 * b + r], w.p[t][e], acc, 0, 0, 0);
        return acc;
    }
    static __device__ __forceinline__ void store(float* p, v4f x) { *reinterpret_cast<v4f*>(p) = x; }
};

// HG heads of a workgroup, KVG key and value heads that they read at most, KB keys of a block
template <typename T, int DP, int HG_, int KVG_, int KB_>
struct AttentionShape {
    using Type = T;
    using Op = Operand<T, DP>;
    static constexpr int kDim = DP, HG = HG_, KVG = KVG_, KB = KB_;
    // 16 keys each, that a wave takes at once (two heads of 64 values: 6.4 ms at 30 000 keys with 4, 6.2 with 2, whose sums leave registers,
    // both with two waves a SIMD)
    static constexpr int H = KB == 64 && HG * DP < 128 ? 4 : 2;
    static constexpr int kHalf = KVG * KB * Op::kPitch;                                  // keys, or values, in LDS
    static constexpr int kTiny = kAttentionBlock / 64 * kTinyRows * Op::kPitch;          // the values of a tiny window for each wave
    static constexpr int kWordsHead = DP / Op::kPer;                                     // 16-byte words of a head's row
    static constexpr int kLoads = (2 * KVG * kWordsHead * KB + kAttentionBlock - 1) / kAttentionBlock;  // of a thread
    // Where the waves of a workgroup share the keys out: keys of a wave's block (eight words of a lane, sixteen in FP32 with heads
    // of 128 values), its keys and values in LDS
    static constexpr int KW = 256 / kWordsHead > 64 ? 64 : 256 / kWordsHead < 16 ? 16 : 256 / kWordsHead;
    static constexpr int kWave = 2 * KW * Op::kPitch;
    // Waves of a SIMD that the registers leave room for.  A third one is worth a few registers in memory: 30 000 keys, 8 heads of 64 values on 4 of keys
    // 6.2 -> 5.3 ms, few rows 3 800 and 16 heads of 64 values in FP32 948 -> 831 us, 3 800 and 8 of 64 in FP16 202 -> 177.  Kernels that keep to 168
    // by themselves are scheduled worse under the bound (53 000 rows, 8 heads of 32: 106 -> 110), those beyond 180 lose too many.
    static constexpr int kWavesListed = DP == 64 && HG == 2 && KVG == 1 ? 3 : 2, kWavesFew = DP <= 64 ? 3 : 2;
};

enum { kCapNone, kCapExponential, kCapSeries };

constexpr int kEnoughGroups = 1024;  // workgroups: four waves on every SIMD of 256 compute units

// 16 H keys and 16 queries of a head: from z = q.k on to the weights, running maximum and sum, products with the values at `v`
template <typename S, int CAP, bool BIAS, int H, bool TAIL>
__device__ __forceinline__ void attend(const AttentionArgs& a, v4f (&z)[H], const typename S::Type* v, const float (&far)[H][4], float slope,
                                       int left, float& most, typename S::Op::Sum& total, v4f (&acc)[S::kDim / 16], int r, int g) {
    using Op = typename S::Op;
#pragma unroll
    for (int t = 0; t < H; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = z[t][e];
            if constexpr (CAP != kCapNone) {
                // tanh(u) = 1 - 2 / (1 + e^2u), of which the exponential form's z is the half that depends on u; near 0, where that has lost
                // the last bits relative to u, the first terms of the series (the next one is below 2^-24 of the sum for |u| < 0.2)
                const float y = x * a.in_cap, f = __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(y));
                if constexpr (CAP == kCapSeries) {
                    const float u = y * (0.5f / kLog2e), u2 = u * u;
                    const float near = u * (1.f + u2 * (-1.f / 3.f + u2 * (2.f / 15.f + u2 * (-17.f / 315.f))));
                    x = fabsf(u) < 0.2f ? near : fmaf(-2.f, f, 1.f);
                } else {
                    x = -f;
                }
            }
            if constexpr (BIAS) x = fmaf(-slope, far[t][e], x);
            z[t][e] = x;
        }
    if constexpr (TAIL) {  // (keys that there are not)
#pragma unroll
        for (int t = 0; t < H; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) z[t][e] = 16 * t + 4 * g + e < left ? z[t][e] : -INFINITY;
    }
    float block_most = -INFINITY;
#pragma unroll
    for (int t = 0; t < H; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) block_most = fmaxf(block_most, z[t][e]);
    if (__any(block_most > most)) {
        const float new_most = fmaxf(most, most_of_query(block_most));
        const float shrink = most == new_most ? 1.f : __builtin_amdgcn_exp2f((most - new_most) * a.by);
        most = new_most;
        total *= shrink;
#pragma unroll
        for (int b = 0; b < S::kDim / 16; ++b) acc[b] *= shrink;
    }
    // (scores of -infinity alone leave nothing to subtract: they weigh 0, and 0 / 0 at the end)
    // The maximum leaves before the factor comes: fma(z, by, -(max by)), an instruction less, has what max by was rounded by in its exponent, 57 for scores
    // of 2^29, which no FP16 weight holds.  (30 000 keys, 8 heads of 64: 5.28 -> 5.35 ms; asking whether scores are that large, 5.48)
    const float top = most == -INFINITY ? 0.f : most;
#pragma unroll
    for (int t = 0; t < H; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) z[t][e] = __builtin_amdgcn_exp2f(fmaf(z[t][e] - top, a.by, Op::kLargest));
    const typename Op::template Weights<H> p(z);
    total = Op::template add<H>(total, p);
#pragma unroll
    for (int b = 0; b < S::kDim / 16; ++b) acc[b] = Op::template values<H>(v, p, acc[b], b, r, g);
}

// Of two voxels, in the unit of the slopes.  Cells are subtracted as they are, integers below 2^24: places in that unit would be rounded, and two of
// them far from the window's first cell differ by little more than that.  (Three products a distance more than with such places: 53 000 rows in windows,
// 8 heads of 32, 101 -> 104 us, 30 000 keys, 8 heads of 64, 5.09 -> 5.22 ms, 16 000 rows in FP32 60 -> 61 us.)
__device__ __forceinline__ float distance(const AttentionArgs& a, const float4& c, const float4& d) {
    const float dx = (c.x - d.x) * a.cell_x, dy = (c.y - d.y) * a.cell_y, dz = (c.z - d.z) * a.cell_z;
    return __builtin_amdgcn_sqrtf(fmaf(dx, dx, fmaf(dy, dy, dz * dz)));
}

template <typename S>
__device__ __forceinline__ void store_row(const AttentionArgs& a, int row, int head, const typename S::Op::Sum& total, const v4f (&acc)[S::kDim / 16],
                                          bool there, int g) {
    using Op = typename S::Op;
    const float by = 1.f / Op::sum(total);
    typename S::Type* dst = static_cast<typename S::Type*>(a.out) + ((size_t)(unsigned)row * a.heads + head) * a.dim;
#pragma unroll
    for (int b = 0; b < S::kDim / 16; ++b)
        if (there && 16 * b + 4 * g < a.dim) Op::store(dst + 16 * b + 4 * g, acc[b] * by);
}

template <typename S>
__device__ __forceinline__ typename S::Op::Row load_query(const AttentionArgs& a, const typename S::Type* row, int head, int g) {
    typename S::Op::Row q = S::Op::load(row + head * a.dim, a.dim, g);
    if (a.negate)
#pragma unroll
        for (int s = 0; s < S::Op::kParts; ++s) q.part[s] = -q.part[s];
    return q;
}

// A window of up to 16 H rows and a head, by one wave
template <typename S, int CAP, bool BIAS, int H>
__device__ __forceinline__ void tiny_window(const AttentionArgs& a, int start, int len, int head, typename S::Type* s_v) {
    using T = typename S::Type;
    using Op = typename S::Op;
    constexpr int kWords = 16 * H * S::kWordsHead, kLoads = (kWords + 63) / 64;  // words of the values, of a lane
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int kv = head / (a.heads / a.kv_heads);
    const size_t stride = (size_t)(a.heads + 2 * a.kv_heads) * a.dim;
    const T* const qkv = static_cast<const T*>(a.qkv);
    const auto place = [&](int i) { return start + (i < len ? i : len - 1); };
    int row[H];
    v4u word[kLoads];
    typename Op::Row q[H], k[H];
    float4 me[H], them[H][4];
#pragma unroll
    for (int t = 0; t < H; ++t) {
        row[t] = a.w.order[place(16 * t + r)];
        if constexpr (BIAS) {
            me[t] = a.w.cell[place(16 * t + r)];
#pragma unroll
            for (int e = 0; e < 4; ++e) them[t][e] = a.w.cell[place(16 * t + 4 * g + e)];
        }
    }
    int value_row[kLoads];
#pragma unroll
    for (int j = 0; j < kLoads; ++j) value_row[j] = a.w.order[place((64 * j + lane) / S::kWordsHead)];
#pragma unroll
    for (int t = 0; t < H; ++t) {
        q[t] = load_query<S>(a, qkv + (size_t)(unsigned)row[t] * stride, head, g);
        k[t] = Op::load(qkv + (size_t)(unsigned)row[t] * stride + (size_t)(a.heads + kv) * a.dim, a.dim, g);
    }
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int key = (64 * j + lane) / S::kWordsHead, d = (64 * j + lane) % S::kWordsHead * Op::kPer;
        word[j] = v4u{0, 0, 0, 0};
        if (key < len && d < a.dim)
            word[j] = *reinterpret_cast<const v4u*>(qkv + (size_t)(unsigned)value_row[j] * stride + (size_t)(a.heads + a.kv_heads + kv) * a.dim + d);
    }
    const float slope = BIAS ? a.slopes[head] * a.to_slope : 0.f;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
        const int key = (64 * j + lane) / S::kWordsHead, d = (64 * j + lane) % S::kWordsHead * Op::kPer;
        if (key < 16 * H) *reinterpret_cast<v4u*>(s_v + key * Op::kPitch + d) = word[j];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int u = 0; u < H; ++u) {  // 16 queries
        float far[H][4];
        v4f z[H];
#pragma unroll
        for (int t = 0; t < H; ++t) {
            z[t] = Op::scores(k[t], q[u]);
            if constexpr (BIAS) {
#pragma unroll
                for (int e = 0; e < 4; ++e) far[t][e] = distance(a, them[t][e], me[u]);
            }
        }
        float most = -INFINITY;
        typename Op::Sum total = {};
        v4f acc[S::kDim / 16] = {};
        attend<S, CAP, BIAS, H, true>(a, z, s_v, far, slope, len, most, total, acc, r, g);
        store_row<S>(a, row[u], head, total, acc, 16 * u + r < len, g);
    }
    __builtin_amdgcn_wave_barrier();
}

// Up to 64 queries of a window from q0 on and heads h_first .. h_first + hc - 1, by the workgroup
template <typename S, int CAP, bool BIAS>
__device__ __forceinline__ void window_rows(const AttentionArgs& a, int start, int len, int q0, int h_first, int hc, typename S::Type* s_kv, float4* s_cell,
                                            int32_t* s_row) {
    using T = typename S::Type;
    using Op = typename S::Op;
    constexpr int HG = S::HG, KB = S::KB, kLoads = S::kLoads;
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const T* const qkv = static_cast<const T*>(a.qkv);
    const int ratio = a.heads / a.kv_heads;
    const int kv_first = h_first / ratio, kvs = (h_first + hc - 1) / ratio - kv_first + 1;
    const unsigned stride = (unsigned)(a.heads + 2 * a.kv_heads) * (unsigned)a.dim;

    const int32_t* const order = a.w.order + start;
    const float4* const cells = a.w.cell + start;

    // Words of a block: key by key, of each the key's heads and then the value's, rounded up to a power of two.  A thread has words tid,
    // tid + 256, ...: the same ones of every step-th key.
    const int kv_words = (kvs > 2 ? 4 : kvs) * S::kWordsHead, step = kAttentionBlock / (2 * kv_words);
    const int word_at = tid & (2 * kv_words - 1), word_half = word_at >= kv_words ? 1 : 0, word_head = (word_at & (kv_words - 1)) / S::kWordsHead;
    const int word_d = word_at % S::kWordsHead * Op::kPer;
    const bool word_there = word_head < kvs && tid / (2 * kv_words) < KB;
    const int first_key = word_there && word_d < a.dim ? tid / (2 * kv_words) : 0x40000000;  // (beyond every key: no word)
    const T* const source = qkv + (size_t)(a.heads + kv_first + word_half * a.kv_heads + word_head) * a.dim + word_d;
    T* const target = s_kv + word_half * S::kHalf + (word_head * KB + tid / (2 * kv_words)) * Op::kPitch + word_d;

    const int tiles = len - q0 >= kItemRows ? 4 : (len - q0 + 15) / 16;
    // waves of a tile of 16 queries, and this wave's heads
    const int share = tiles == 1 ? 4 : tiles == 2 ? 2 : 1;
    const int per = (hc + share - 1) / share;
    const int tile = wave / share, h0 = wave % share * per;
    const int mine = tile >= tiles || h0 >= hc ? 0 : hc - h0 < per ? hc - h0 : per;

    v4u word[kLoads];  // (a thread's words of the next block: those of keys that there are)
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
        if (i * step < KB && first_key + i * step < len) word[i] = *reinterpret_cast<const v4u*>(source + (size_t)(unsigned)order[first_key + i * step] * stride);
    float4 cell = make_float4(0, 0, 0, 0);
    int32_t row = 0;
    if (tid < KB) {
        if (BIAS) cell = cells[tid < len ? tid : 0];
        row = order[KB + tid < len ? KB + tid : 0];
    }
    const int q_at = q0 + tile * 16 + r;
    const bool q_there = q_at < len && mine > 0;
    const int q_row = order[q_there ? q_at : 0];
    float4 me = make_float4(0, 0, 0, 0);
    if (BIAS) me = cells[q_there ? q_at : 0];
    typename Op::Row q[HG];
    float slope[HG], most[HG];
    typename Op::Sum total[HG];
    v4f acc[HG][S::kDim / 16];
#pragma unroll
    for (int i = 0; i < HG; ++i) {
        const int head = h_first + (i < mine ? h0 + i : 0);
        q[i] = load_query<S>(a, qkv + (size_t)(unsigned)q_row * stride, head, g);
        slope[i] = BIAS ? a.slopes[head] * a.to_slope : 0.f;
        most[i] = -INFINITY;
        total[i] = typename Op::Sum{};
#pragma unroll
        for (int b = 0; b < S::kDim / 16; ++b) acc[i][b] = v4f{0, 0, 0, 0};
    }
    for (int k0 = 0; k0 < len; k0 += KB) {
        const int left = len - k0;
        __syncthreads();  // (the block before, or the item before, is worked on)
        if (k0 == 0 && word_there && word_d >= a.dim)  // values behind a head's last one are zeros
            for (int key = 0; tid / (2 * kv_words) + key < KB; key += step) *reinterpret_cast<v4u*>(target + key * Op::kPitch) = v4u{0, 0, 0, 0};
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            if (first_key + i * step < KB) *reinterpret_cast<v4u*>(target + i * step * Op::kPitch) = first_key + i * step < left ? word[i] : v4u{0, 0, 0, 0};
        if (tid < KB) {
            if (BIAS) s_cell[tid] = cell;
            s_row[tid] = row;
        }
        __syncthreads();
        if (left > KB) {  // the next block, and the rows of the one behind it
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (i * step < KB && first_key + i * step < left - KB)
                    word[i] = *reinterpret_cast<const v4u*>(source + (size_t)(unsigned)s_row[first_key + i * step] * stride);
            if (tid < KB) {
                if (BIAS) cell = cells[KB + tid < left ? k0 + KB + tid : 0];
                row = order[2 * KB + tid < left ? k0 + 2 * KB + tid : 0];
            }
        }
        if (mine > 0) {
            const auto keys = [&](auto sixteens, auto tail, int k1) {  // 16 H keys from k1 on
                constexpr int H = decltype(sixteens)::value;
                constexpr bool TAIL = decltype(tail)::value;
                float far[H][4];
                if constexpr (BIAS) {
#pragma unroll
                    for (int t = 0; t < H; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) far[t][e] = distance(a, s_cell[k1 + 16 * t + 4 * g + e], me);
                }
#pragma unroll
                for (int i = 0; i < HG; ++i) {
                    if (i >= mine) continue;
                    const T* k = s_kv + (((h_first + h0 + i) / ratio - kv_first) * KB + k1) * Op::kPitch;
                    v4f z[H];
#pragma unroll
                    for (int t = 0; t < H; ++t) z[t] = Op::scores(k + 16 * t * Op::kPitch, q[i], r, g);
                    attend<S, CAP, BIAS, H, TAIL>(a, z, k + S::kHalf, far, slope[i], left - k1, most[i], total[i], acc[i], r, g);
                }
            };
            int k1 = 0;
#pragma unroll 1
            for (; k1 < KB && k1 + 16 * S::H <= left; k1 += 16 * S::H) keys(std::integral_constant<int, S::H>{}, std::false_type{}, k1);
#pragma unroll 1
            for (; k1 < KB && k1 < left; k1 += 32) keys(std::integral_constant<int, 2>{}, std::true_type{}, k1);
        }
    }
#pragma unroll
    for (int i = 0; i < HG; ++i)
        if (i < mine) store_row<S>(a, q_row, h_first + h0 + i, total[i], acc[i], q_there, g);
}

// Up to 16 queries of a window from q0 on and a head, by the workgroup: its waves have every fourth block of KW keys each, wait for nobody, and join
// their sums at the end.  s_part: kWave elements of a wave, s_cell: KW of a wave.
template <typename S, int CAP, bool BIAS>
__device__ __forceinline__ void shared_rows(const AttentionArgs& a, int start, int len, int q0, int head, typename S::Type* s_part, float4* s_cell) {
    using T = typename S::Type;
    using Op = typename S::Op;
    constexpr int KW = S::KW, DP = S::kDim, kWaves = kAttentionBlock / 64, kStep = 32 / S::kWordsHead, kLoads = KW / kStep;
    constexpr int kJoin = DP + 4;  // floats of a query: sums, maximum, sum of the weights
    static_assert(16 * kJoin * sizeof(float) <= S::kWave * sizeof(T), "a wave's sums lie where its keys were");
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const T* const qkv = static_cast<const T*>(a.qkv);
    const int kv = head / (a.heads / a.kv_heads);
    const size_t stride = (size_t)(a.heads + 2 * a.kv_heads) * a.dim;
    const int32_t* const order = a.w.order + start;
    const float4* const cells = a.w.cell + start;
    T* const s_k = s_part + wave * S::kWave;
    float4* const s_far = s_cell + wave * KW;

    // words of a block: key by key, the key's and then the value's.  A lane has the same ones of every kStep-th key
    const int first_key = lane / (2 * S::kWordsHead), half = lane / S::kWordsHead & 1, d = lane % S::kWordsHead * Op::kPer;
    const T* const source = qkv + (size_t)(a.heads + kv + half * a.kv_heads) * a.dim + (d < a.dim ? d : 0);
    T* const target = s_k + half * KW * Op::kPitch + first_key * Op::kPitch + d;
    const auto row_of = [&](int k0) { return order[k0 + lane < len ? k0 + lane : len - 1]; };  // of the key lane of a block
    v4u word[kLoads];
    const auto gather = [&](int row, int left) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const unsigned at = (unsigned)__shfl(row, first_key + i * kStep);
            word[i] = *reinterpret_cast<const v4u*>(source + (size_t)at * stride);
            if (d >= a.dim || first_key + i * kStep >= left) word[i] = v4u{0, 0, 0, 0};
        }
    };
    int k0 = wave * KW;
    int row = row_of(k0);
    const bool q_there = q0 + r < len;
    const int q_row = order[q_there ? q0 + r : len - 1];
    float4 cell = make_float4(0, 0, 0, 0), me = cell;
    if (BIAS) {
        cell = cells[k0 + lane < len ? k0 + lane : len - 1];
        me = cells[q_there ? q0 + r : len - 1];
    }
    gather(row, len - k0);
    row = row_of(k0 + kWaves * KW);
    const typename Op::Row q = load_query<S>(a, qkv + (size_t)(unsigned)q_row * stride, head, g);
    const float slope = BIAS ? a.slopes[head] * a.to_slope : 0.f;
    float most = -INFINITY;
    typename Op::Sum total = {};
    v4f acc[DP / 16] = {};
    __syncthreads();  // (the item before is worked on)
#pragma unroll 1
    for (; k0 < len; k0 += kWaves * KW) {
        const int left = len - k0;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) *reinterpret_cast<v4u*>(target + i * kStep * Op::kPitch) = word[i];
        if (BIAS && lane < KW) s_far[lane] = cell;
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        if (left > kWaves * KW) {  // the next block, and the rows of the one behind it
            gather(row, left - kWaves * KW);
            if (BIAS) cell = cells[kWaves * KW + lane < left ? k0 + kWaves * KW + lane : len - 1];
            row = row_of(k0 + 2 * kWaves * KW);
        }
        const auto keys = [&](auto tail) {
            constexpr int H = KW / 16;
            float far[H][4];
            v4f z[H];
#pragma unroll
            for (int t = 0; t < H; ++t) {
                if constexpr (BIAS) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) far[t][e] = distance(a, s_far[16 * t + 4 * g + e], me);
                }
                z[t] = Op::scores(s_k + 16 * t * Op::kPitch, q, r, g);
            }
            attend<S, CAP, BIAS, H, decltype(tail)::value>(a, z, s_k + KW * Op::kPitch, far, slope, left, most, total, acc, r, g);
        };
        if (left >= KW) keys(std::false_type{});
        else keys(std::true_type{});
        __builtin_amdgcn_wave_barrier();
    }
    float* const s_join = reinterpret_cast<float*>(s_k) + r * kJoin;
    const float sum = Op::sum(total);
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) *reinterpret_cast<v4f*>(s_join + 16 * b + 4 * g) = acc[b];
    if (g == 0) {
        s_join[DP] = most;
        s_join[DP + 1] = sum;
    }
    __syncthreads();
    const auto of_wave = [&](int w) { return reinterpret_cast<const float*>(s_part + w * S::kWave) + r * kJoin; };
    float all_most = -INFINITY, all = 0.f, by[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all_most = fmaxf(all_most, of_wave(w)[DP]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        by[w] = of_wave(w)[DP] == all_most ? 1.f : __builtin_amdgcn_exp2f((of_wave(w)[DP] - all_most) * a.by);
        all = fmaf(of_wave(w)[DP + 1], by[w], all);
    }
    const float over = 1.f / all;
    T* const dst = static_cast<T*>(a.out) + ((size_t)(unsigned)q_row * a.heads + head) * a.dim;
#pragma unroll
    for (int b = 0; b < DP / 16; ++b) {
        if (b % kWaves != wave) continue;
        v4f x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) x += *reinterpret_cast<const v4f*>(of_wave(w) + 16 * b + 4 * g) * by[w];
        if (q_there && 16 * b + 4 * g < a.dim) Op::store(dst + 16 * b + 4 * g, x * over);
    }
}

template <typename S, int CAP, bool BIAS>
__global__ void __launch_bounds__(kAttentionBlock, S::kWavesListed)
voxel_attention(AttentionArgs a) {
    using T = typename S::Type;
    using Op = typename S::Op;
    __shared__ __align__(16) T s_kv[2 * S::kHalf > S::kTiny ? 2 * S::kHalf : S::kTiny];  // [keys, values][kv head][key][kPitch]; tiny windows: [wave][key][kPitch]
    __shared__ float4 s_cell[S::KB];
    __shared__ int32_t s_row[S::KB];                // rows of the block to come
    T* const out = static_cast<T*>(a.out);
    const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int longs = a.w.head[kHeadLong], shorts = a.w.head[kHeadShort], tinies = a.w.head[kHeadTiny];
    // Heads of a workgroup: all that it can take where that leaves workgroups enough, else one.  (Groups of heads of an item side by side: long
    // items come first, and share what L2 has of the rows.)
    const int all = (a.heads + S::HG - 1) / S::HG;
    const int per_long = longs * all >= kEnoughGroups ? S::HG : 1, per_short = (longs + shorts) * all >= kEnoughGroups ? S::HG : 1;
    const int groups_long = (a.heads + per_long - 1) / per_long, groups_short = (a.heads + per_short - 1) / per_short;
    const int end_long = longs * groups_long, end_short = end_long + shorts * groups_short, end = end_short + (tinies + 3) / 4 * a.heads;
    for (int v = blockIdx.x; v < end; v += gridDim.x) {
        if (v < end_short) {
            const bool is_long = v < end_long;
            const int u = is_long ? v : v - end_long, gs = is_long ? groups_long : groups_short, per = is_long ? per_long : per_short;
            const int4 it = is_long ? long_item(a.w, u / gs) : short_item(a.w, u / gs);
            const int h = u % gs * per;
            const int start = __builtin_amdgcn_readfirstlane(it.x);
            window_rows<S, CAP, BIAS>(a, start, __builtin_amdgcn_readfirstlane(it.y), __builtin_amdgcn_readfirstlane(it.z), h,
                                      a.heads - h < per ? a.heads - h : per, s_kv, s_cell, s_row);
        } else {
            // (the heads of a window side by side)
            const int u = v - end_short, at = u / a.heads * 4 + wave, h = u % a.heads;
            __syncthreads();  // (an item of the other kind is worked on)
            if (at < tinies) {
                const int2 it = a.w.tiny[at];
                const int start = __builtin_amdgcn_readfirstlane(it.x), len = __builtin_amdgcn_readfirstlane(it.y);
                T* const s_v = s_kv + wave * kTinyRows * Op::kPitch;
                if (len <= 16) tiny_window<S, CAP, BIAS, 1>(a, start, len, h, s_v);
                else tiny_window<S, CAP, BIAS, 2>(a, start, len, h, s_v);
            }
        }
    }
    // rows that attend to nothing: outside the grid, and behind the last one
    const int n = a.w.head[kHeadRows], places = a.w.head[kHeadPlaces];
    const size_t row_words = (size_t)a.heads * a.dim / Op::kPer;
    const size_t thread = (size_t)blockIdx.x * kAttentionBlock + tid, threads = (size_t)gridDim.x * kAttentionBlock;
    for (size_t i = thread; i < (size_t)(n - places) * row_words; i += threads)
        reinterpret_cast<v4u*>(out)[(size_t)a.w.order[places + i / row_words] * row_words + i % row_words] = v4u{0, 0, 0, 0};
    if (a.write_pad)
        for (size_t i = (size_t)n * row_words + thread; i < (size_t)a.w.max_voxels * row_words; i += threads) reinterpret_cast<v4u*>(out)[i] = v4u{0, 0, 0, 0};
}

// The same where the list has spans (few rows): kFewPlaces places and a head are a workgroup's, which takes the tiny windows that begin
// among them and the blocks of 64 queries (16, SHARED) that do.
constexpr int kFewPlaces = 16;
// Waves that share a query's keys reach four times as much of the card with few queries, but read each key for 16 queries instead of 64 and have more
// registers.  FP16, 64 and 16 queries a workgroup: 1 866 rows of one window and 2 heads of 16 values 47 and 21 us, 3 800 and 8 of 64 431 and 177, but 24 of
// 64 439 and 468, and windows of 6 x 6 at 3 800 rows and 16 heads 30 and 37.  FP32, whose products take longer: 3 800 rows and 16 heads of 64 1 480 and 831.
constexpr int kSharedRows = 32768;  // rows times heads, FP16
template <typename S, int CAP, bool BIAS, bool SHARED>
__global__ void __launch_bounds__(kAttentionBlock, S::kWavesFew)
voxel_attention_few(AttentionArgs a) {
    using T = typename S::Type;
    using Op = typename S::Op;
    constexpr int kWaves = kAttentionBlock / 64, kKeys = SHARED ? kWaves * S::kWave : 2 * S::kHalf, kQueries = SHARED ? 16 : kItemRows;
    __shared__ __align__(16) T s_kv[kKeys > S::kTiny ? kKeys : S::kTiny];
    __shared__ float4 s_cell[SHARED ? kWaves * S::KW : S::KB];
    __shared__ int32_t s_row[SHARED ? 1 : S::KB];
    T* const out = static_cast<T*>(a.out);
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int first = (int)(blockIdx.x / (unsigned)a.heads) * kFewPlaces, head = (int)(blockIdx.x % (unsigned)a.heads);
    const int n = a.w.head[kHeadRows], places = a.w.head[kHeadPlaces];
    const int place = first + lane;
    const bool there = lane < kFewPlaces && place < places;
    const int2 span = there ? a.w.span[place] : make_int2(0, 0);  // (every wave has all of them)
    const int before = place - span.x;
    for (uint64_t m = __ballot(there && span.y > kTinyRows && before % kQueries == 0); m; m &= m - 1) {
        const int who = __builtin_ctzll(m), start = __builtin_amdgcn_readlane(span.x, who), len = __builtin_amdgcn_readlane(span.y, who);
        const int q0 = __builtin_amdgcn_readlane(before, who);
        if constexpr (SHARED) shared_rows<S, CAP, BIAS>(a, start, len, q0, head, s_kv, s_cell);
        else window_rows<S, CAP, BIAS>(a, start, len, q0, head, 1, s_kv, s_cell, s_row);
    }
    __syncthreads();  // (the last item is worked on)
    int turn = 0;
    for (uint64_t m = __ballot(there && span.y <= kTinyRows && before == 0); m; m &= m - 1, ++turn) {
        if ((turn & 3) != wave) continue;
        const int who = __builtin_ctzll(m), start = __builtin_amdgcn_readlane(span.x, who), len = __builtin_amdgcn_readlane(span.y, who);
        T* const s_v = s_kv + wave * kTinyRows * Op::kPitch;
        if (len <= 16) tiny_window<S, CAP, BIAS, 1>(a, start, len, head, s_v);
        else tiny_window<S, CAP, BIAS, 2>(a, start, len, head, s_v);
    }
    // rows that attend to nothing: outside the grid, and behind the last one
    const int words = a.dim / Op::kPer;
    for (int i = tid; i < kFewPlaces * words; i += kAttentionBlock) {
        const int p = first + i / words;
        if (p < places || p >= a.w.max_voxels || (p >= n && !a.write_pad)) continue;
        *reinterpret_cast<v4u*>(out + ((size_t)(p < n ? a.w.order[p] : p) * a.heads + head) * a.dim + i % words * Op::kPer) = v4u{0, 0, 0, 0};
    }
}

template <typename S, int CAP, bool BIAS>
void launch_attention_as(const AttentionArgs& a, hipStream_t stream) {
    if (a.w.max_voxels <= kFewRows) {
        using F = AttentionShape<typename S::Type, S::kDim, 1, 1, S::KB>;
        const dim3 grid((unsigned)(ceil_div(a.w.max_voxels, kFewPlaces) * a.heads));
        if (sizeof(typename S::Type) == 4 || a.w.max_voxels * a.heads <= kSharedRows) {
            hipLaunchKernelGGL((voxel_attention_few<F, CAP, BIAS, true>), grid, dim3(kAttentionBlock), 0, stream, a);
        } else if constexpr (sizeof(typename S::Type) == 2) {
            hipLaunchKernelGGL((voxel_attention_few<F, CAP, BIAS, false>), grid, dim3(kAttentionBlock), 0, stream, a);
        }
        return;
    }
    // (a tiny window's share of a workgroup is a quarter; what is beyond the grid is taken in turns)
    const int64_t most = ((int64_t)a.w.items_cap + ceil_div(a.w.max_voxels, 4)) * a.heads;
    const unsigned grid = (unsigned)(most < 4096 ? most : 4096);
    hipLaunchKernelGGL((voxel_attention<S, CAP, BIAS>), dim3(grid), dim3(kAttentionBlock), 0, stream, a);
}
template <typename S>
void launch_attention_shape(const AttentionArgs& a, hipStream_t stream) {
    constexpr bool kHalf = sizeof(typename S::Type) == 2;
    if (!a.capped) {
        if (a.slopes) launch_attention_as<S, kCapNone, true>(a, stream);
        else launch_attention_as<S, kCapNone, false>(a, stream);
    } else if (a.series) {
        if (a.slopes) launch_attention_as<S, kCapSeries, true>(a, stream);
        else launch_attention_as<S, kCapSeries, false>(a, stream);
    } else if constexpr (kHalf) {
        if (a.slopes) launch_attention_as<S, kCapExponential, true>(a, stream);
        else launch_attention_as<S, kCapExponential, false>(a, stream);
    }
}
// key and value heads that a group of `group` neighbouring heads reads, at most
inline int kv_heads_of(const AttentionArgs& a, int group) {
    const int ratio = a.heads / a.kv_heads;
    int most = 1;
    for (int h = 0; h < a.heads; h += group) {
        const int last = h + group < a.heads ? h + group - 1 : a.heads - 1, n = last / ratio - h / ratio + 1;
        most = n > most ? n : most;
    }
    return most;
}
// What a thread keeps of the next block are eight words at most.
template <typename T, int DP, int KB>
void launch_attention_dim(const AttentionArgs& a, hipStream_t stream) {
    // A second head uses the distances of the first; a wave's registers leave the card fewer waves.  FP16, HG 1 and 2: 7 200 voxels of one window times
    // 16 heads of 32 values 622 and 760 us, 16 000 in windows times 8 of 16 42.5 and 49, 12 000 times 16 of 16 44.5 and 49.7, 10 300 times 16 of 32 82
    // and 84, 53 000 times 8 of 32 142 and 106, 30 000 times 8 of 64 in one window 7.1 and 5.3 ms (with cap).  FP32 waits for the matrix cores:
    // 16 000 times 8 of 24 62 and 80 us.
    if constexpr (sizeof(T) == 2) {
        if ((int64_t)a.w.max_voxels * a.heads >= 200000) {
            if (kv_heads_of(a, 2) == 1) return launch_attention_shape<AttentionShape<T, DP, 2, 1, KB>>(a, stream);
            if constexpr (DP <= 64) return launch_attention_shape<AttentionShape<T, DP, 2, 2, KB>>(a, stream);
        }
    }
    launch_attention_shape<AttentionShape<T, DP, 1, 1, KB>>(a, stream);
}

#endif

}  // namespace sessd

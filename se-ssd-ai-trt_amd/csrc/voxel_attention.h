// voxel_attention.h -- attention among the rows of a window (voxel_windows.h): the kernel, for FP16 and FP32 tensors.
//
// A workgroup of four waves takes up to 64 queries of one window and a few heads, and walks over the window's keys in blocks of 64 (32
// where a head's values are many).  Keys, values and voxels of a block lie in LDS; those of the next one are gathered into registers in
// the meantime.  A wave has 16 queries; where the window has fewer than 64, waves share queries and deal the heads out.
//
// Scores are taken transposed, S^T = K Q^T: a lane of the result has one query (its column) and four keys, so that maximum and sum over the
// keys are mostly the lane's own, and the weights are where the second product, O^T = V^T P^T, wants them.  Maximum and sum run along
// with the blocks; sums that are there already are rescaled only where a block raises a maximum.
#pragma once

#include "voxel_windows.h"

namespace sessd {

struct AttentionArgs {
    const void* qkv;
    void* out;
    const int32_t* voxel_num;
    const float* slopes;  // or null
    WindowIndex w;
    int heads, kv_heads, dim;
    float scale;          // of the scores, to the base 2 where they are not capped; 2 / cap of it, to the base 2, where they are
    float cap;            // to the base 2; 0 = none
    bool series;          // small capped scores by the first terms of the series: the exponential form is not exact enough
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
    struct Row {
        v8h part[kParts];
    };
    static __device__ __forceinline__ Row query(const _Float16* p, int dim, int g) {
        Row q;
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            v8h x = {};
            if constexpr (DP >= 32) {
                if (s * 32 + g * 8 < dim) x = *reinterpret_cast<const v8h*>(p + s * 32 + g * 8);
            } else {
                v4h y = {};
                if (g * 4 < dim) y = *reinterpret_cast<const v4h*>(p + g * 4);
                x = v8h{y[0], y[1], y[2], y[3], 0, 0, 0, 0};
            }
            q.part[s] = x;
        }
        return q;
    }
    // 16 keys from `k` on times 16 queries
    static __device__ __forceinline__ v4f scores(const _Float16* k, const Row& q, int r, int g) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            if constexpr (DP >= 32)
                acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(*reinterpret_cast<const v8h*>(k + r * kPitch + s * 32 + g * 8), q.part[s], acc, 0, 0, 0);
            else
                acc = __builtin_amdgcn_mfma_f32_16x16x16f16(*reinterpret_cast<const v4h*>(k + r * kPitch + g * 4),
                                                            v4h{q.part[s][0], q.part[s][1], q.part[s][2], q.part[s][3]}, acc, 0, 0, 0);
        }
        return acc;
    }
    // 32 weights of a query, rounded to 11 bits: the product's own operands are FP16
    struct Weights {
        v8h p;
    };
    static __device__ __forceinline__ Weights weights(const v4f& s, const v4f& t) {
        Weights w;
#pragma unroll
        for (int e = 0; e < 4; ++e) w.p[e] = (_Float16)s[e], w.p[4 + e] = (_Float16)t[e];
        return w;
    }
    // sums of 16 values from 16 b on over 32 keys: LDS transposes four keys' values as it reads them, a lane gets value lane % 16 of keys
    // 4 (lane / 16) .. + 3 of either half, which is where its weights are
    static __device__ __forceinline__ v4f values(const _Float16* v, const Weights& w, v4f acc, int b, int r, int g) {
        typedef __attribute__((address_space(3))) v4s* lds;
        const _Float16* p = v + (4 * g + (r >> 2)) * kPitch + 16 * b + (r & 3) * 4;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)p);
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds)(p + 16 * kPitch));
        const v4h x = __builtin_bit_cast(v4h, lo), y = __builtin_bit_cast(v4h, hi);
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(v8h{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]}, w.p, acc, 0, 0, 0);
    }
    static __device__ __forceinline__ void store(_Float16* p, v4f x) { *reinterpret_cast<v4h*>(p) = v4h{(_Float16)x[0], (_Float16)x[1], (_Float16)x[2], (_Float16)x[3]}; }
};

template <int DP> struct Operand<float, DP> {
    static constexpr int kPer = 4, kPitch = DP + 4, kParts = DP / 16;
    // 16x16x4: the j-th instruction of a part takes value 16 s + 4 (lane / 16) + j
    struct Row {
        v4f part[kParts];
    };
    static __device__ __forceinline__ Row query(const float* p, int dim, int g) {
        Row q;
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            v4f x = {};
            if (s * 16 + g * 4 < dim) x = *reinterpret_cast<const v4f*>(p + s * 16 + g * 4);
            q.part[s] = x;
        }
        return q;
    }
    static __device__ __forceinline__ v4f scores(const float* k, const Row& q, int r, int g) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            const v4f x = *reinterpret_cast<const v4f*>(k + r * kPitch + s * 16 + g * 4);
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(x[j], q.part[s][j], acc, 0, 0, 0);
        }
        return acc;
    }
    struct Weights {
        v4f p[2];
    };
    static __device__ __forceinline__ Weights weights(const v4f& s, const v4f& t) { return Weights{{s, t}}; }
    static __device__ __forceinline__ v4f values(const float* v, const Weights& w, v4f acc, int b, int r, int g) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
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
    static constexpr int kHalf = KVG * KB * Op::kPitch;                                  // keys, or values, in LDS
    static constexpr int kWordsHead = DP / Op::kPer;                                     // 16-byte words of a head's row
    static constexpr int kLoads = (2 * KVG * kWordsHead * KB + kAttentionBlock - 1) / kAttentionBlock;  // of a thread
};

enum { kCapNone, kCapExponential, kCapSeries };

// 16 H keys times 16 queries of a head: scores, running maximum and sum, weights, products with the values
template <typename S, int CAP, bool BIAS, int H>
__device__ __forceinline__ void attend_block(const AttentionArgs& a, const typename S::Type* k, const typename S::Type* v, const typename S::Op::Row& q,
                                             const float (&far)[S::KB / 16][4], float slope, int left, float& most, float& total,
                                             v4f (&acc)[S::kDim / 16], int r, int g) {
    using Op = typename S::Op;
    v4f s[H];
#pragma unroll
    for (int t = 0; t < H; ++t) {
        s[t] = Op::scores(k + 16 * t * Op::kPitch, q, r, g);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float x = s[t][e] * a.scale;
            if constexpr (CAP != kCapNone) {
                // cap * tanh(u) = cap - 2 cap / (1 + e^2u); near 0, where that has lost the last bits relative to u, the first terms of the
                // series (the next one is below 2^-24 of the sum for |u| < 0.2)
                const float y = fmaf(-2.f * a.cap, __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x)), a.cap);
                if constexpr (CAP == kCapSeries) {
                    const float u = x * (0.5f / kLog2e), u2 = u * u;
                    const float near = a.cap * u * (1.f + u2 * (-1.f / 3.f + u2 * (2.f / 15.f + u2 * (-17.f / 315.f))));
                    x = fabsf(u) < 0.2f ? near : y;
                } else {
                    x = y;
                }
            }
            if constexpr (BIAS) x = fmaf(-slope, far[t][e], x);
            s[t][e] = x;
        }
    }
    if (left < 16 * H) {
#pragma unroll
        for (int t = 0; t < H; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s[t][e] = 16 * t + 4 * g + e < left ? s[t][e] : -INFINITY;
    }
    float block_most = -INFINITY;
#pragma unroll
    for (int t = 0; t < H; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) block_most = fmaxf(block_most, s[t][e]);
    if (__any(block_most > most)) {
        const float new_most = fmaxf(most, most_of_query(block_most));
        const float shrink = most == new_most ? 1.f : __builtin_amdgcn_exp2f(most - new_most);
        most = new_most;
        total *= shrink;
#pragma unroll
        for (int b = 0; b < S::kDim / 16; ++b) acc[b] *= shrink;
    }
    // (scores of -infinity alone leave nothing to subtract: they weigh 0, and 0 / 0 at the end)
    const float less = most == -INFINITY ? 0.f : most;
    float sum[H];
#pragma unroll
    for (int t = 0; t < H; ++t) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[t][e] = __builtin_amdgcn_exp2f(s[t][e] - less);
        sum[t] = (s[t][0] + s[t][1]) + (s[t][2] + s[t][3]);
    }
#pragma unroll
    for (int t = 0; t < H; t += 2) total += sum[t] + sum[t + 1];
#pragma unroll
    for (int t = 0; t < H; t += 2) {
        const typename Op::Weights p = Op::weights(s[t], s[t + 1]);
#pragma unroll
        for (int b = 0; b < S::kDim / 16; ++b) acc[b] = Op::values(v + 16 * t * Op::kPitch, p, acc[b], b, r, g);
    }
}

template <typename S, int CAP, bool BIAS>
__global__ void __launch_bounds__(kAttentionBlock, 2)
voxel_attention(AttentionArgs a) {
    using T = typename S::Type;
    using Op = typename S::Op;
    constexpr int HG = S::HG, KB = S::KB, kBlocks = S::kDim / 16, kLoads = S::kLoads;
    __shared__ __align__(16) T s_kv[2 * S::kHalf];  // [keys, values][kv head][key][kPitch]
    __shared__ float4 s_cell[KB];
    __shared__ int32_t s_row[KB];                   // rows of the block to come
    const int tid = threadIdx.x, lane = tid & 63, r = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const T* const qkv = static_cast<const T*>(a.qkv);
    T* const out = static_cast<T*>(a.out);
    const int h_first = blockIdx.y * HG;
    const int hc = a.heads - h_first < HG ? a.heads - h_first : HG;  // heads of this workgroup
    const int ratio = a.heads / a.kv_heads;
    const int kv_first = h_first / ratio, kvs = (h_first + hc - 1) / ratio - kv_first + 1;
    const unsigned stride = (unsigned)(a.heads + 2 * a.kv_heads) * (unsigned)a.dim;
    const T* const keys = qkv + (size_t)(a.heads + kv_first) * a.dim;

    // Words of a block: key by key, of each the key's heads and then the value's.  A thread has words tid, tid + 256, ...
    const int words_key = 2 * kvs * S::kWordsHead;
    int key_of[kLoads], from[kLoads], to[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
        const int c = i * kAttentionBlock + tid;
        const int key = c / words_key, rest = c - key * words_key;
        const int half = rest >= words_key / 2 ? 1 : 0, at = rest - half * (words_key / 2);
        const int head = at / S::kWordsHead, d = at % S::kWordsHead * Op::kPer;
        key_of[i] = key < KB && d < a.dim ? key : 0x40000000;
        from[i] = half * a.kv_heads * a.dim + head * a.dim + d;
        to[i] = half * S::kHalf + (head * KB + key) * Op::kPitch + d;
        // (values behind a head's last one are zeros, here and for good)
        if (key < KB && d >= a.dim) *reinterpret_cast<v4u*>(s_kv + to[i]) = v4u{0, 0, 0, 0};
    }

    const int longs = a.w.head[kHeadLong], items = longs + a.w.head[kHeadShort];
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int4 it = window_item(a.w, item, longs);
        const int start = __builtin_amdgcn_readfirstlane(it.x), len = __builtin_amdgcn_readfirstlane(it.y), q0 = __builtin_amdgcn_readfirstlane(it.z);
        const int32_t* const order = a.w.order + start;
        const float4* const cells = a.w.cell + start;
        const int tiles = len - q0 >= kItemRows ? 4 : (len - q0 + 15) / 16;
        // waves of a tile of 16 queries, and this wave's heads
        const int share = tiles == 1 ? 4 : tiles == 2 ? 2 : 1;
        const int per = (HG + share - 1) / share;
        const int tile = wave / share, h0 = wave % share * per;
        const int mine = tile >= tiles || h0 >= hc ? 0 : hc - h0 < per ? hc - h0 : per;

        v4u word[kLoads];  // (a thread's words of the next block: those of keys that there are)
#pragma unroll
        for (int i = 0; i < kLoads; ++i)
            if (key_of[i] < len) word[i] = *reinterpret_cast<const v4u*>(keys + (size_t)(unsigned)order[key_of[i]] * stride + from[i]);
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
        float slope[HG], most[HG], total[HG];
        v4f acc[HG][kBlocks];
#pragma unroll
        for (int i = 0; i < HG; ++i) {
            const int head = h_first + (i < mine ? h0 + i : 0);
            q[i] = Op::query(qkv + (size_t)(unsigned)q_row * stride + head * a.dim, a.dim, g);
            slope[i] = BIAS ? a.slopes[head] * kLog2e : 0.f;
            most[i] = -INFINITY;
            total[i] = 0.f;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b) acc[i][b] = v4f{0, 0, 0, 0};
        }
        for (int k0 = 0; k0 < len; k0 += KB) {
            const int left = len - k0;
            __syncthreads();  // (the block before, or the item before, is worked on)
#pragma unroll
            for (int i = 0; i < kLoads; ++i)
                if (key_of[i] < KB) *reinterpret_cast<v4u*>(s_kv + to[i]) = key_of[i] < left ? word[i] : v4u{0, 0, 0, 0};
            if (tid < KB) {
                if (BIAS) s_cell[tid] = cell;
                s_row[tid] = row;
            }
            __syncthreads();
            if (left > KB) {  // the next block, and the rows of the one behind it
#pragma unroll
                for (int i = 0; i < kLoads; ++i)
                    if (key_of[i] < left - KB) word[i] = *reinterpret_cast<const v4u*>(keys + (size_t)(unsigned)s_row[key_of[i]] * stride + from[i]);
                if (tid < KB) {
                    if (BIAS) cell = cells[KB + tid < left ? k0 + KB + tid : 0];
                    row = order[2 * KB + tid < left ? k0 + 2 * KB + tid : 0];
                }
            }
            if (mine > 0) {
                float far[KB / 16][4];
                if constexpr (BIAS) {
#pragma unroll
                    for (int t = 0; t < KB / 16; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float4 c = s_cell[16 * t + 4 * g + e];
                            const float dx = (c.x - me.x) * a.cell_x, dy = (c.y - me.y) * a.cell_y, dz = (c.z - me.z) * a.cell_z;
                            far[t][e] = __builtin_amdgcn_sqrtf(dx * dx + dy * dy + dz * dz);
                        }
                }
#pragma unroll
                for (int i = 0; i < HG; ++i) {
                    if (i >= mine) continue;
                    const T* k = s_kv + ((h_first + h0 + i) / ratio - kv_first) * KB * Op::kPitch;
                    const T* v = k + S::kHalf;
                    if (KB == 32 || left <= 32) attend_block<S, CAP, BIAS, 2>(a, k, v, q[i], far, slope[i], left, most[i], total[i], acc[i], r, g);
                    else attend_block<S, CAP, BIAS, KB / 16>(a, k, v, q[i], far, slope[i], left, most[i], total[i], acc[i], r, g);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < HG; ++i) {
            if (i >= mine) continue;
            const float by = 1.f / sum_of_query(total[i]);
            T* dst = out + ((size_t)(unsigned)q_row * a.heads + h_first + h0 + i) * a.dim;
#pragma unroll
            for (int b = 0; b < kBlocks; ++b)
                if (q_there && 16 * b + 4 * g < a.dim) Op::store(dst + 16 * b + 4 * g, acc[i][b] * by);
        }
    }
    // rows that attend to nothing: outside the grid, and behind the last one
    const int n = clamp_rows(a.voxel_num, a.w.max_voxels), places = a.w.head[kHeadPlaces];
    const size_t row_words = (size_t)a.heads * a.dim / Op::kPer;
    const size_t thread = ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * kAttentionBlock + tid, threads = (size_t)gridDim.x * gridDim.y * kAttentionBlock;
    for (size_t i = thread; i < (size_t)(n - places) * row_words; i += threads)
        reinterpret_cast<v4u*>(out)[(size_t)a.w.order[places + i / row_words] * row_words + i % row_words] = v4u{0, 0, 0, 0};
    if (a.write_pad)
        for (size_t i = (size_t)n * row_words + thread; i < (size_t)a.w.max_voxels * row_words; i += threads) reinterpret_cast<v4u*>(out)[i] = v4u{0, 0, 0, 0};
}

template <typename S, int CAP, bool BIAS>
void launch_attention_as(const AttentionArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)(a.w.items_cap < 4096 ? a.w.items_cap : 4096), (unsigned)ceil_div(a.heads, S::HG));
    hipLaunchKernelGGL((voxel_attention<S, CAP, BIAS>), grid, dim3(kAttentionBlock), 0, stream, a);
}
template <typename S>
void launch_attention_shape(const AttentionArgs& a, hipStream_t stream) {
    constexpr bool kHalf = sizeof(typename S::Type) == 2;
    if (a.cap == 0.f) {
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
// What a thread keeps of the next block are eight words at most: wide heads share a workgroup where they share keys.
template <typename T, int DP, int KVG, int KB>
void launch_attention_dim(const AttentionArgs& a, hipStream_t stream) {
    if constexpr (KVG == 4) launch_attention_shape<AttentionShape<T, DP, 4, 4, KB>>(a, stream);
    else if (kv_heads_of(a, 2 * KVG) <= KVG) launch_attention_shape<AttentionShape<T, DP, 2 * KVG, KVG, KB>>(a, stream);
    else launch_attention_shape<AttentionShape<T, DP, KVG, KVG, KB>>(a, stream);
}

#endif

}  // namespace sessd

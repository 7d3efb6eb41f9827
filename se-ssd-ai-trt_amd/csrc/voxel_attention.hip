// voxel_attention.hip -- VoxelAttentionPlugin: attention among the voxels of a window of the grid.
//
// The rows of a sparse tensor come in the order in which their voxels were met.  They are brought into an order by windows first:
//
//   window_count    a row's window and its ticket among the window's rows
//   window_base     the windows' places in the list, one behind the other
//   window_scatter  the list, a window's rows in the order of their tickets
//   window_rank     the same with a window's rows ascending: which ticket a row got is chance, the order of its sums is not
//
// and then
//
//   voxel_attention one wave for 16 places of the list and one head, over the keys of the windows that these places lie in
//
// A wave takes the scores transposed, S^T = K Q^T: the result's lane has one query (its column) and four keys, so that maximum and
// sum over the keys are mostly the lane's own, and the weights are where the second product, O^T = V^T P^T, wants them.
#include <cmath>

#include "plugins.h"

namespace sessd {

namespace {

constexpr int kBlock = 256;
constexpr int kQueries = 16;
constexpr int kKeys = 32;
constexpr int kMostWindows = 1 << 22;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v4h __attribute__((ext_vector_type(4)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

struct Grid {
    int shape[3];   // z,y,x
    int window[3];
    int shift[3];
    int count[3];   // windows
};

// What a plugin's workspace holds.  The first part, whose places follow from max_voxels alone, is what shared calls read.
struct Windows {
    int32_t* head;   // status word, places in the list
    int32_t* key;    // of a row: its window, -1 = outside the grid
    int32_t* order;  // the list: rows
    int2* span;      // of a place: first place of its window, first place behind it
    float4* cell;    // of a place: its voxel, x,y,z
    int32_t* slot;
    int32_t* list;
    int32_t* count;
    int32_t* base;
    size_t bytes;
};

Windows carve(void* workspace, int max_voxels, size_t windows) {
    WorkspaceCarver c(workspace);
    Windows w;
    w.head = c.take<int32_t>(64);
    w.key = c.take<int32_t>(max_voxels);
    w.order = c.take<int32_t>(max_voxels);
    w.span = c.take<int2>(max_voxels);
    w.cell = c.take<float4>(max_voxels);
    w.slot = c.take<int32_t>(max_voxels);
    w.list = c.take<int32_t>(max_voxels);
    w.count = c.take<int32_t>(windows);
    w.base = c.take<int32_t>(windows);
    w.bytes = c.total();
    return w;
}

__global__ void __launch_bounds__(kBlock)
window_count(const int32_t* __restrict__ coors, const int32_t* __restrict__ voxel_num, int max_voxels, Grid g, Windows w) {
    const int row = blockIdx.x * kBlock + threadIdx.x;
    const int n = clamp_rows(voxel_num, max_voxels);
    if (row >= n) return;
    const int4 c = reinterpret_cast<const int4*>(coors)[row];  // (b,z,y,x)
    if (c.x != 0 || c.y < 0 || c.y >= g.shape[0] || c.z < 0 || c.z >= g.shape[1] || c.w < 0 || c.w >= g.shape[2]) {
        atomicOr(&w.head[0], SESSD_STATUS_BAD_COORD);
        w.key[row] = -1;
        return;
    }
    const int key = ((c.y + g.shift[0]) / g.window[0] * g.count[1] + (c.z + g.shift[1]) / g.window[1]) * g.count[2] +
                    (c.w + g.shift[2]) / g.window[2];
    w.key[row] = key;
    // (a wave whose rows are all of one window asks once)
    const int first = __builtin_amdgcn_readfirstlane(key);
    const uint64_t here = __ballot(1);
    if (__ballot(key == first) == here) {
        int at = 0;
        const uint32_t rank = rank_in_wave(here);
        if (rank == 0) at = atomicAdd(&w.count[key], (int)__popcll(here));
        w.slot[row] = __builtin_amdgcn_readfirstlane(at) + (int)rank;
    } else {
        w.slot[row] = atomicAdd(&w.count[key], 1);
    }
}

__global__ void __launch_bounds__(kBlock)
window_base(int windows, Windows w) {
    const int i = blockIdx.x * kBlock + threadIdx.x;
    const uint32_t mine = i < windows ? (uint32_t)w.count[i] : 0u;
    const uint32_t upto = wave_scan(mine);
    int at = 0;
    if ((threadIdx.x & 63) == 63 && upto) at = atomicAdd(&w.head[1], (int)upto);
    at = __shfl(at, 63);
    if (mine) w.base[i] = at + (int)(upto - mine);
}

__global__ void __launch_bounds__(kBlock)
window_scatter(const int32_t* __restrict__ voxel_num, int max_voxels, Windows w) {
    const int row = blockIdx.x * kBlock + threadIdx.x;
    if (row >= clamp_rows(voxel_num, max_voxels)) return;
    const int key = w.key[row];
    if (key >= 0) w.list[w.base[key] + w.slot[row]] = row;
}

__global__ void __launch_bounds__(kBlock)
window_rank(const int32_t* __restrict__ coors, Windows w) {
    const int p = blockIdx.x * kBlock + threadIdx.x;
    if (p >= w.head[1]) return;
    const int row = w.list[p], key = w.key[row];
    const int start = w.base[key], len = w.count[key];
    int rank = 0;
    for (int i = 0; i < len; ++i) rank += w.list[start + i] < row ? 1 : 0;
    const int4 c = reinterpret_cast<const int4*>(coors)[row];
    w.order[start + rank] = row;
    w.span[start + rank] = make_int2(start, start + len);
    w.cell[start + rank] = make_float4((float)c.w, (float)c.z, (float)c.y, 0.f);
}

struct AttentionArgs {
    const void* qkv;
    void* out;
    const int32_t* voxel_num;
    const float* slopes;  // or null
    Windows w;
    int max_voxels, heads, kv_heads, dim;
    float scale, cap;     // of the scores
    float cell_x, cell_y, cell_z;
    int write_pad;
};

constexpr float kLog2e = 1.44269504088896340736f;

// c * tanh(x / c), all of it relative to c: near 0, where 1 - 2 / (1 + e^2u) has lost the last bits, by the first terms of the series
// (the next one is below 2^-24 of the sum for |u| < 0.2)
__device__ __forceinline__ float capped(float x, float cap, float inv) {
    const float u = x * inv, u2 = u * u;
    const float e = __builtin_amdgcn_exp2f(u * (2.f * kLog2e));
    const float far = 1.f - 2.f * __builtin_amdgcn_rcpf(1.f + e);
    const float near = u * (1.f + u2 * (-1.f / 3.f + u2 * (2.f / 15.f + u2 * (-17.f / 315.f))));
    return cap * (fabsf(u) < 0.2f ? near : far);
}

// Operand fragments of 16 rows (keys or queries) x DP values of a head: what a lane has of row lane % 16.
template <typename T, int DP> struct Frag;
template <int DP> struct Frag<__half, DP> {  // 16x16x32: eight neighbouring values of each 32; 16x16x16: four of 16
    static constexpr int kParts = DP >= 32 ? DP / 32 : 1, kPer = DP >= 32 ? 8 : 4;
    v8h part[kParts];
    __device__ __forceinline__ void load(const __half* p, int dim, int g, bool there) {
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            const int d = s * 4 * kPer + g * kPer;
            v8h x = {};
            if (there && d < dim) {
                if constexpr (kPer == 8) x = *reinterpret_cast<const v8h*>(p + d);
                else {
                    const v4h y = *reinterpret_cast<const v4h*>(p + d);
                    x = v8h{y[0], y[1], y[2], y[3], 0, 0, 0, 0};
                }
            }
            part[s] = x;
        }
    }
    static __device__ __forceinline__ v4f product(const Frag& a, const Frag& b) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            if constexpr (kPer == 8) acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.part[s], b.part[s], acc, 0, 0, 0);
            else
                acc = __builtin_amdgcn_mfma_f32_16x16x16f16(v4h{a.part[s][0], a.part[s][1], a.part[s][2], a.part[s][3]},
                                                            v4h{b.part[s][0], b.part[s][1], b.part[s][2], b.part[s][3]}, acc, 0, 0, 0);
        }
        return acc;
    }
};
template <int DP> struct Frag<float, DP> {  // 16x16x4: the j-th of four neighbouring values of each 16
    static constexpr int kParts = DP / 16;
    v4f part[kParts];
    __device__ __forceinline__ void load(const float* p, int dim, int g, bool there) {
#pragma unroll
        for (int s = 0; s < kParts; ++s) {
            const int d = s * 16 + g * 4;
            v4f x = {};
            if (there && d < dim) x = *reinterpret_cast<const v4f*>(p + d);
            part[s] = x;
        }
    }
    static __device__ __forceinline__ v4f product(const Frag& a, const Frag& b) {
        v4f acc = {};
#pragma unroll
        for (int s = 0; s < kParts; ++s)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(a.part[s][j], b.part[s][j], acc, 0, 0, 0);
        return acc;
    }
};

template <typename T, int DP>
__global__ void __launch_bounds__(kBlock)
voxel_attention(AttentionArgs a) {
    constexpr int kBlocks = DP / 16;            // of the head's values
    constexpr int kPitch = DP + 8;              // of a value row in LDS, halves
    __shared__ __half s_v[sizeof(T) == 2 ? kBlock / 64 : 1][sizeof(T) == 2 ? kKeys * kPitch : 1];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    const int head = blockIdx.y * (kBlock / 64) + wave;
    const int tile = blockIdx.x * kQueries;
    const T* qkv = static_cast<const T*>(a.qkv);
    T* out = static_cast<T*>(a.out);
    if (head >= a.heads) return;
    // the rows that attend to nothing: beyond the active ones, outside the grid
    const int n = clamp_rows(a.voxel_num, a.max_voxels);
    for (int i = 0; i < kQueries; ++i) {
        const int row = tile + i;
        if (row >= a.max_voxels || (row >= n && !a.write_pad)) break;
        if (row < n && a.w.key[row] >= 0) continue;
        for (int d = lane; d < a.dim; d += 64) out[((size_t)row * a.heads + head) * a.dim + d] = (T)0.f;
    }
    const int places = a.w.head[1];
    if (tile >= places) return;
    const int last = tile + kQueries < places ? tile + kQueries : places;
    const size_t stride = (size_t)(a.heads + 2 * a.kv_heads) * a.dim;
    const int kv = head * a.kv_heads / a.heads;
    const T* keys = qkv + (size_t)(a.heads + kv) * a.dim;
    const T* values = qkv + (size_t)(a.heads + a.kv_heads + kv) * a.dim;

    const int place = tile + r < last ? tile + r : last - 1;  // (queries beyond the end repeat the last one)
    const int row = a.w.order[place];
    const int my_start = a.w.span[place].x;
    const float4 me = a.w.cell[place];
    const float slope = a.slopes ? a.slopes[head] * kLog2e : 0.f;
    const float scale = a.cap > 0.f ? a.scale : a.scale * kLog2e, inv = a.cap > 0.f ? 1.f / a.cap : 0.f;
    Frag<T, DP> q;
    q.load(qkv + (size_t)row * stride + (size_t)head * a.dim, a.dim, g, true);

    float most = -INFINITY, total = 0.f;  // of the query: largest score, sum of the weights of this lane's keys
    v4f acc[kBlocks] = {};
    for (int at = tile; at < last;) {
        const int2 span = a.w.span[at];
        const bool mine = my_start == span.x;
        for (int k0 = span.x; k0 < span.y; k0 += kKeys) {
            v4f s[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const int k = k0 + 16 * t + r;
                const bool there = k < span.y;
                Frag<T, DP> f;
                f.load(keys + (size_t)(there ? a.w.order[k] : 0) * stride, a.dim, g, there);
                s[t] = Frag<T, DP>::product(f, q);
            }
            float block_most = -INFINITY;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int k = k0 + 16 * t + 4 * g + e;
                    float x = s[t][e] * scale;
                    if (a.cap > 0.f) x = capped(x, a.cap, inv) * kLog2e;
                    if (k < span.y) {
                        if (a.slopes) {
                            const float4 c = a.w.cell[k];
                            const float dx = (c.x - me.x) * a.cell_x, dy = (c.y - me.y) * a.cell_y, dz = (c.z - me.z) * a.cell_z;
                            x -= slope * sqrtf(dx * dx + dy * dy + dz * dz);
                        }
                    } else {
                        x = -INFINITY;
                    }
                    s[t][e] = x;
                    block_most = fmaxf(block_most, x);
                }
            block_most = fmaxf(block_most, __shfl_xor(block_most, 16));
            block_most = fmaxf(block_most, __shfl_xor(block_most, 32));
            const float new_most = mine ? fmaxf(most, block_most) : most;
            // (scores of -infinity alone leave nothing to subtract; they weigh 0, and 0 / 0 at the end)
            const float from = new_most == -INFINITY ? 0.f : new_most;
            const float shrink = mine ? __builtin_amdgcn_exp2f(most - from) : 1.f;
            most = new_most;
            float sum = 0.f;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[t][e] = __builtin_amdgcn_exp2f(s[t][e] - from);
                    sum += s[t][e];
                }
            total = mine ? total * shrink + sum : total;
            if constexpr (sizeof(T) == 2) {
                __half* v = s_v[wave];
                constexpr int kChunks = DP / 8;
#pragma unroll
                for (int i = lane; i < kKeys * kChunks; i += 64) {
                    const int k = k0 + i / kChunks, d = i % kChunks * 8;
                    v8h x = {};
                    if (k < span.y && d < a.dim) x = *reinterpret_cast<const v8h*>(values + (size_t)a.w.order[k] * stride + d);
                    *reinterpret_cast<v8h*>(v + i / kChunks * kPitch + d) = x;
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                v8h p;
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = (_Float16)s[0][e], p[4 + e] = (_Float16)s[1][e];
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    v8h x;
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        x[e] = reinterpret_cast<const _Float16*>(v)[(e / 4 * 16 + 4 * g + e % 4) * kPitch + 16 * b + r];
                    const v4f sums = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, p, acc[b] * shrink, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[b][e] = mine ? sums[e] : acc[b][e];  // (0 x what is not finite)
                }
                __builtin_amdgcn_wave_barrier();
            } else {
#pragma unroll
                for (int b = 0; b < kBlocks; ++b) {
                    v4f sums = acc[b] * shrink;
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int k = k0 + 16 * t + 4 * g + e, d = 16 * b + r;
                            float x = 0.f;
                            if (k < span.y && d < a.dim) x = values[(size_t)a.w.order[k] * stride + d];
                            sums = __builtin_amdgcn_mfma_f32_16x16x4f32(x, s[t][e], sums, 0, 0, 0);
                        }
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[b][e] = mine ? sums[e] : acc[b][e];
                }
            }
        }
        at = span.y;
    }
    total += __shfl_xor(total, 16);
    total += __shfl_xor(total, 32);
    if (tile + r >= last) return;
    T* dst = out + (size_t)row * a.heads * a.dim + (size_t)head * a.dim;
#pragma unroll
    for (int b = 0; b < kBlocks; ++b) {
        const int d = 16 * b + 4 * g;
        if (d >= a.dim) continue;
        if constexpr (sizeof(T) == 2) {
            v4h x;
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = (_Float16)(acc[b][e] / total);
            *reinterpret_cast<v4h*>(dst + d) = x;
        } else {
            *reinterpret_cast<v4f*>(dst + d) = acc[b] / total;
        }
    }
}

template <typename T>
void launch_attention(const AttentionArgs& a, hipStream_t stream) {
    const dim3 grid((unsigned)ceil_div(a.max_voxels, kQueries), (unsigned)ceil_div(a.heads, kBlock / 64));
    if (a.dim <= 16) hipLaunchKernelGGL((voxel_attention<T, 16>), grid, dim3(kBlock), 0, stream, a);
    else if (a.dim <= 32) hipLaunchKernelGGL((voxel_attention<T, 32>), grid, dim3(kBlock), 0, stream, a);
    else if (a.dim <= 64) hipLaunchKernelGGL((voxel_attention<T, 64>), grid, dim3(kBlock), 0, stream, a);
    else hipLaunchKernelGGL((voxel_attention<T, 128>), grid, dim3(kBlock), 0, stream, a);
}

Grid grid_of(const sessd_voxelattn_desc& d) {
    Grid g;
    for (int a = 0; a < 3; ++a) {  // x,y,z -> z,y,x
        g.shape[2 - a] = d.spatial_shape[a];
        g.window[2 - a] = d.window_shape[a];
        g.shift[2 - a] = d.window_shift[a];
        g.count[2 - a] = (int)(((int64_t)d.spatial_shape[a] - 1 + d.window_shift[a]) / d.window_shape[a]) + 1;
    }
    return g;
}
size_t windows_of(const Grid& g) { return (size_t)g.count[0] * g.count[1] * g.count[2]; }

}  // namespace

VoxelAttentionPlugin::~VoxelAttentionPlugin() {
    if (slopes_dev_) (void)hipFree(slopes_dev_);
}

int VoxelAttentionPlugin::create(const sessd_voxelattn_desc& d, const float* slopes, VoxelAttentionPlugin** out) {
    if (d.num_heads < 1 || d.num_kv_heads < 1 || d.head_dim < 1 || d.max_voxels < 1)
        return fail(SESSD_E_INVALID, "voxelattn: heads, head_dim and max_voxels must be positive");
    if (d.num_heads % d.num_kv_heads) return fail(SESSD_E_INVALID, "voxelattn: num_heads must be a multiple of num_kv_heads");
    if (d.head_dim % 8 || d.head_dim > 128 || d.num_heads > 1024)
        return fail(SESSD_E_UNSUPPORTED, "voxelattn: head_dim must be a multiple of 8 up to 128, num_heads at most 1024 (%d, %d)", d.head_dim,
                    d.num_heads);
    for (int a = 0; a < 3; ++a) {
        if (d.spatial_shape[a] < 1 || d.window_shape[a] < 1 || d.window_shift[a] < 0 || d.window_shift[a] >= d.window_shape[a])
            return fail(SESSD_E_INVALID, "voxelattn: shapes must be positive, shifts 0 .. window_shape - 1");
        if (d.spatial_shape[a] > 1 << 24 || d.window_shape[a] > 1 << 24)  // (a cell's place is exact in FP32)
            return fail(SESSD_E_UNSUPPORTED, "voxelattn: shapes beyond 2^24 cells");
        if (!std::isfinite(d.cell_size[a])) return fail(SESSD_E_INVALID, "voxelattn: cell_size must be finite");
    }
    const Grid g = grid_of(d);
    if ((double)g.count[0] * g.count[1] * g.count[2] > kMostWindows)
        return fail(SESSD_E_UNSUPPORTED, "voxelattn: %d x %d x %d windows, at most %d are supported", g.count[2], g.count[1], g.count[0], kMostWindows);
    if (!std::isfinite(d.softmax_scale) || !std::isfinite(d.score_cap) || d.score_cap < 0.f)
        return fail(SESSD_E_INVALID, "voxelattn: softmax_scale and score_cap must be finite, score_cap not negative");
    std::unique_ptr<VoxelAttentionPlugin> p(new VoxelAttentionPlugin());
    p->desc_ = d;
    if (slopes) {
        for (int h = 0; h < d.num_heads; ++h)
            if (!std::isfinite(slopes[h])) return fail(SESSD_E_INVALID, "voxelattn: the slopes must be finite");
        p->slopes_.assign(slopes, slopes + d.num_heads);
        SESSD_HIP_TRY(hipMalloc(reinterpret_cast<void**>(&p->slopes_dev_), d.num_heads * sizeof(float)));
        SESSD_HIP_TRY(hipMemcpy(p->slopes_dev_, slopes, d.num_heads * sizeof(float), hipMemcpyHostToDevice));
    }
    *out = p.release();
    return SESSD_OK;
}

// the desc's fields in their order, whether slopes follow, the slopes
size_t VoxelAttentionPlugin::getSerializationSize() const { return sizeof(sessd_voxelattn_desc) + sizeof(int) + slopes_.size() * sizeof(float); }

void VoxelAttentionPlugin::serialize(void* buffer) const {
    char* d = static_cast<char*>(buffer);
    writeToBuffer<sessd_voxelattn_desc>(d, desc_);
    writeToBuffer<int>(d, slopes_.empty() ? 0 : 1);
    for (float v : slopes_) writeToBuffer<float>(d, v);
}

int VoxelAttentionPlugin::deserialize(const void* data, size_t length, VoxelAttentionPlugin** out) {
    if (!data || length < sizeof(sessd_voxelattn_desc) + sizeof(int)) return fail(SESSD_E_INVALID, "voxelattn: blob too short");
    const char* d = static_cast<const char*>(data);
    const sessd_voxelattn_desc desc = readFromBuffer<sessd_voxelattn_desc>(d);
    std::vector<float> slopes;
    if (readFromBuffer<int>(d)) {
        const size_t left = (length - sizeof(sessd_voxelattn_desc) - sizeof(int)) / sizeof(float);
        if (desc.num_heads < 1 || left < (size_t)desc.num_heads) return fail(SESSD_E_INVALID, "voxelattn: blob too short for its slopes");
        slopes.resize((size_t)desc.num_heads);
        std::memcpy(slopes.data(), d, slopes.size() * sizeof(float));
    }
    return create(desc, slopes.empty() ? nullptr : slopes.data(), out);
}

int VoxelAttentionPlugin::check(const sessd_tensor_desc* in, const sessd_tensor_desc* out) const {
    const char* who = "voxelattn";
    if (in[0].type != SESSD_FLOAT && in[0].type != SESSD_HALF) return fail(SESSD_E_UNSUPPORTED, "voxelattn: features must be FP32 or FP16");
    if (out[0].type != in[0].type) return fail(SESSD_E_UNSUPPORTED, "voxelattn: the output must have the input's type");
    SESSD_TRY(check_rows(in[0], desc_.max_voxels, (desc_.num_heads + 2 * desc_.num_kv_heads) * desc_.head_dim, who, "qkv"));
    SESSD_TRY(check_rows(in[1], desc_.max_voxels, 4, who, "coors"));
    SESSD_TRY(check_rows(out[0], desc_.max_voxels, desc_.num_heads * desc_.head_dim, who, "the output"));
    if (in[1].type != SESSD_INT32 || !is_scalar_int(in[2])) return fail(SESSD_E_INVALID, "voxelattn: coors and voxel_num must be INT32, voxel_num one value");
    return SESSD_OK;
}

int VoxelAttentionPlugin::configurePlugin(const sessd_tensor_desc* in, int nbInputs, const sessd_tensor_desc* out, int nbOutputs) {
    if (!in || !out || nbInputs != 3 || nbOutputs != 1) return fail(SESSD_E_INVALID, "voxelattn.configure: expected 3 inputs and 1 output");
    SESSD_TRY(check(in, out));
    type_ = in[0].type;
    return SESSD_OK;
}

size_t VoxelAttentionPlugin::getWorkspaceSize(const sessd_tensor_desc*, int, const sessd_tensor_desc*, int) const {
    return carve(nullptr, desc_.max_voxels, windows_of(grid_of(desc_))).bytes;
}

int VoxelAttentionPlugin::checkCall(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                                    void* const* outputs, const void* workspace, const char* who) const {
    if (!inputDesc || !outputDesc || !inputs || !outputs || !workspace) return fail(SESSD_E_INVALID, "%s: null argument", who);
    if (!inputs[0] || !inputs[1] || !inputs[2] || !outputs[0]) return fail(SESSD_E_INVALID, "%s: null tensor pointer", who);
    if (inputDesc[0].type != type_) return fail(SESSD_E_INVALID, "%s: tensor dtypes differ from the configured ones", who);
    SESSD_TRY(check(inputDesc, outputDesc));
    if ((reinterpret_cast<uintptr_t>(inputs[0]) | reinterpret_cast<uintptr_t>(inputs[1]) | reinterpret_cast<uintptr_t>(outputs[0]) |
         reinterpret_cast<uintptr_t>(workspace)) & 15)
        return fail(SESSD_E_INVALID, "%s: tensors and workspace must be 16-byte aligned", who);
    return SESSD_OK;
}

int VoxelAttentionPlugin::attend(const void* const* inputs, void* const* outputs, const void* workspace, hipStream_t stream) const {
    AttentionArgs a;
    a.qkv = inputs[0];
    a.out = outputs[0];
    a.voxel_num = static_cast<const int32_t*>(inputs[2]);
    a.slopes = slopes_dev_;
    a.w = carve(const_cast<void*>(workspace), desc_.max_voxels, 0);
    a.max_voxels = desc_.max_voxels;
    a.heads = desc_.num_heads;
    a.kv_heads = desc_.num_kv_heads;
    a.dim = desc_.head_dim;
    a.scale = desc_.softmax_scale != 0.f ? desc_.softmax_scale : (float)(1.0 / std::sqrt((double)desc_.head_dim));
    a.cap = desc_.score_cap;
    a.cell_x = desc_.cell_size[0];
    a.cell_y = desc_.cell_size[1];
    a.cell_z = desc_.cell_size[2];
    a.write_pad = (flags_ & SESSD_FLAG_SKIP_PAD_ROWS) ? 0 : 1;
    if (type_ == SESSD_HALF) launch_attention<__half>(a, stream);
    else launch_attention<float>(a, stream);
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

int VoxelAttentionPlugin::enqueue(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                                  void* const* outputs, void* workspace, hipStream_t stream) {
    SESSD_TRY(checkCall(inputDesc, outputDesc, inputs, outputs, workspace, "voxelattn.enqueue"));
    const Grid g = grid_of(desc_);
    const size_t windows = windows_of(g);
    const Windows w = carve(workspace, desc_.max_voxels, windows);
    const int32_t* coors = static_cast<const int32_t*>(inputs[1]);
    const int32_t* num = static_cast<const int32_t*>(inputs[2]);
    FillArgs f;
    f.add(w.head, 64, 0);
    f.add(w.count, windows, 0);
    SESSD_TRY(launch_fill(f, stream));
    const dim3 rows((unsigned)ceil_div(desc_.max_voxels, kBlock));
    hipLaunchKernelGGL(window_count, rows, dim3(kBlock), 0, stream, coors, num, desc_.max_voxels, g, w);
    hipLaunchKernelGGL(window_base, dim3((unsigned)ceil_div((int64_t)windows, kBlock)), dim3(kBlock), 0, stream, (int)windows, w);
    hipLaunchKernelGGL(window_scatter, rows, dim3(kBlock), 0, stream, num, desc_.max_voxels, w);
    hipLaunchKernelGGL(window_rank, rows, dim3(kBlock), 0, stream, coors, w);
    SESSD_HIP_TRY(hipGetLastError());
    return attend(inputs, outputs, workspace, stream);
}

int VoxelAttentionPlugin::enqueueShared(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                                        void* const* outputs, const void* window_workspace, hipStream_t stream) {
    SESSD_TRY(checkCall(inputDesc, outputDesc, inputs, outputs, window_workspace, "voxelattn.enqueue_shared"));
    return attend(inputs, outputs, window_workspace, stream);
}

}  // namespace sessd

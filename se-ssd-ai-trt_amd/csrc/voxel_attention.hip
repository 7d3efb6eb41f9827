// voxel_attention.hip -- VoxelAttentionPlugin: attention among the voxels of a window of the grid, and the kernel of
// voxel_attention.h for FP16 tensors.
//
//   voxel_windows.hip   rows by windows, a list that layers on the same coordinates can share
//   voxel_attention.h   the attention itself, one launch
#include <cmath>

#include "plugins.h"
#include "voxel_attention.h"

namespace sessd {

int launch_attention_half(const AttentionArgs& a, hipStream_t stream) {
    if (a.dim <= 16) launch_attention_dim<_Float16, 16, 64>(a, stream);
    else if (a.dim <= 32) launch_attention_dim<_Float16, 32, 64>(a, stream);
    else if (a.dim <= 64) launch_attention_dim<_Float16, 64, 64>(a, stream);
    else launch_attention_dim<_Float16, 128, 64>(a, stream);
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

namespace {

WindowGrid grid_of(const sessd_voxelattn_desc& d) {
    WindowGrid g;
    for (int a = 0; a < 3; ++a) {  // x,y,z -> z,y,x
        g.shape[2 - a] = d.spatial_shape[a];
        g.window[2 - a] = d.window_shape[a];
        g.shift[2 - a] = d.window_shift[a];
        g.over[2 - a] = d.window_shape[a] == 1 ? 0 : ~(uint64_t)0 / (uint64_t)d.window_shape[a] + 1;
        g.count[2 - a] = (int)(((int64_t)d.spatial_shape[a] - 1 + d.window_shift[a]) / d.window_shape[a]) + 1;
    }
    return g;
}

}  // namespace

VoxelAttentionPlugin::~VoxelAttentionPlugin() {
    if (slopes_dev_) (void)hipFree(slopes_dev_);
}

int VoxelAttentionPlugin::create(const sessd_voxelattn_desc& d, const float* slopes, VoxelAttentionPlugin** out) {
    if (d.num_heads < 1 || d.num_kv_heads < 1 || d.head_dim < 1 || d.max_voxels < 1)
        return fail(SESSD_E_INVALID, "voxelattn: heads, head_dim and max_voxels must be positive");
    if (d.num_heads % d.num_kv_heads) return fail(SESSD_E_INVALID, "voxelattn: num_heads must be a multiple of num_kv_heads");
    if (d.head_dim % 8 || d.head_dim > 128 || d.num_heads > 1024 || d.max_voxels > kMostRows)
        return fail(SESSD_E_UNSUPPORTED, "voxelattn: head_dim must be a multiple of 8 up to 128, num_heads at most 1024, max_voxels at most %d (%d, %d, %d)", kMostRows,
                    d.head_dim, d.num_heads, d.max_voxels);
    for (int a = 0; a < 3; ++a) {
        if (d.spatial_shape[a] < 1 || d.window_shape[a] < 1 || d.window_shift[a] < 0 || d.window_shift[a] >= d.window_shape[a])
            return fail(SESSD_E_INVALID, "voxelattn: shapes must be positive, shifts 0 .. window_shape - 1");
        if (d.spatial_shape[a] > 1 << 24 || d.window_shape[a] > 1 << 24)  // (a cell, and the difference of two, is exact in FP32)
            return fail(SESSD_E_UNSUPPORTED, "voxelattn: shapes beyond 2^24 cells");
        if (!std::isfinite(d.cell_size[a])) return fail(SESSD_E_INVALID, "voxelattn: cell_size must be finite");
    }
    const WindowGrid g = grid_of(d);
    if ((double)g.count[0] * g.count[1] * g.count[2] > (double)kMostWindows)
        return fail(SESSD_E_UNSUPPORTED, "voxelattn: %d x %d x %d windows, at most %d are supported", g.count[2], g.count[1], g.count[0], (int)kMostWindows);
    if (!std::isfinite(d.softmax_scale) || !std::isfinite(d.score_cap) || d.score_cap < 0.f)
        return fail(SESSD_E_INVALID, "voxelattn: softmax_scale and score_cap must be finite, score_cap not negative");
    // (what a score is divided by and what a distance is times stays finite in FP32)
    const float scale = std::fabs(d.softmax_scale), cells = std::fmax(std::fabs(d.cell_size[0]), std::fmax(std::fabs(d.cell_size[1]), std::fabs(d.cell_size[2])));
    if ((scale != 0.f && (scale < 0x1p-40f || scale > 0x1p40f)) || (d.score_cap != 0.f && (d.score_cap < 0x1p-40f || d.score_cap > 0x1p40f)) || cells > 0x1p20f)
        return fail(SESSD_E_UNSUPPORTED, "voxelattn: softmax_scale and score_cap must be 0 or 2^-40 .. 2^40, cell_size at most 2^20");
    std::unique_ptr<VoxelAttentionPlugin> p(new VoxelAttentionPlugin());
    p->desc_ = d;
    SESSD_HIP_TRY(hipGetDevice(&p->device_));
    if (slopes) {
        for (int h = 0; h < d.num_heads; ++h) {
            if (!std::isfinite(slopes[h])) return fail(SESSD_E_INVALID, "voxelattn: the slopes must be finite");
            if (std::fabs(slopes[h]) > 0x1p20f) return fail(SESSD_E_UNSUPPORTED, "voxelattn: slopes beyond 2^20");
        }
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
    return carve_windows(nullptr, desc_.max_voxels, grid_of(desc_).windows()).bytes;
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
    return check_device(device_, who);
}

int VoxelAttentionPlugin::attend(const void* const* inputs, void* const* outputs, const void* workspace, hipStream_t stream) const {
    const bool half = type_ == SESSD_HALF;
    AttentionArgs a;
    a.qkv = inputs[0];
    a.out = outputs[0];
    a.slopes = slopes_dev_;
    a.w = carve_windows(const_cast<void*>(workspace), desc_.max_voxels, grid_of(desc_).windows());
    a.heads = desc_.num_heads;
    a.kv_heads = desc_.num_kv_heads;
    a.dim = desc_.head_dim;
    const double scale = desc_.softmax_scale != 0.f ? std::fabs((double)desc_.softmax_scale) : 1.0 / std::sqrt((double)desc_.head_dim);
    const double log2e = 1.4426950408889634, cap = desc_.score_cap;
    a.negate = desc_.softmax_scale < 0.f;
    a.capped = cap > 0.0;
    // The exponential form is within 2^-23 of the cap: of a score's own size in FP32 from caps of some hundreds on, below FP16's rounding of
    // the weights up to 512.
    a.series = !half || cap > 512.0;
    const double by = !a.capped ? scale * log2e : a.series ? cap * log2e : 2.0 * cap * log2e;
    a.by = (float)by;
    a.to_slope = (float)(log2e / by);
    a.in_cap = a.capped ? (float)(scale / cap * 2.0 * log2e) : 0.f;
    a.cell_x = desc_.cell_size[0];
    a.cell_y = desc_.cell_size[1];
    a.cell_z = desc_.cell_size[2];
    a.write_pad = (flags_ & SESSD_FLAG_SKIP_PAD_ROWS) ? 0 : 1;
    return half ? launch_attention_half(a, stream) : launch_attention_float(a, stream);
}

int VoxelAttentionPlugin::enqueue(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                                  void* const* outputs, void* workspace, hipStream_t stream) {
    SESSD_TRY(checkCall(inputDesc, outputDesc, inputs, outputs, workspace, "voxelattn.enqueue"));
    const WindowGrid g = grid_of(desc_);
    SESSD_TRY(launch_windows(static_cast<const int32_t*>(inputs[1]), static_cast<const int32_t*>(inputs[2]), g,
                             carve_windows(workspace, desc_.max_voxels, g.windows()), stream));
    return attend(inputs, outputs, workspace, stream);
}

int VoxelAttentionPlugin::enqueueShared(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                                        void* const* outputs, const void* window_workspace, hipStream_t stream) {
    SESSD_TRY(checkCall(inputDesc, outputDesc, inputs, outputs, window_workspace, "voxelattn.enqueue_shared"));
    return attend(inputs, outputs, window_workspace, stream);
}

}  // namespace sessd

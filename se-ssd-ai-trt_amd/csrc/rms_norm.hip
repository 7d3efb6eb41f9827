// rms_norm.hip -- RmsNormPlugin: the residual's addition, root-mean-square norm and rounding to e4m3 in one pass.
//
//   h = x + r,   y = gamma * h / sqrt(mean(h^2) + eps),   s = max(max|y| / 448, 2^-100),   q = e4m3(y / s)
//
// In q the root drops out: y / s = 448 * gamma h / max|gamma h|.  That quotient is taken in 64 bits and rounded to FP32 once, so that q is the e4m3
// nearest to what the formula says (or its neighbour, within 2^-24 of the middle of two), whatever the last bits of mean, root and scale are: with all
// of it in FP32 one value in 10^5 fell to the other side of a border between two e4m3, which is a difference of 6 %.  The kernel waits for memory
// either way.
//
// A row stays in the registers of the lanes that read it: its sum of squares and its largest magnitude are two reductions over
// those lanes, and each tensor is read or written once.  What bounds it is memory: 157 301 of 160 000 rows of 256 FP32 with residual 91 us, 5.8 TB/s
// (a large copy 4.8); 16 825 of 20 000 of 128 FP16 6 us.  Stores past the caches gain nothing here.
#include <cfloat>
#include <cmath>

#include "plugins.h"

namespace sessd {

namespace {

constexpr int kBlock = 256;
constexpr float kMost = 448.f;               // of e4m3
constexpr float kSmallestScale = 0x1p-100f;  // of a row of zeros: y / s stays finite, s a normal number

typedef float v4f __attribute__((ext_vector_type(4)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <int VEC>
__device__ __forceinline__ void load_row(const float* p, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        const v4f a = reinterpret_cast<const v4f*>(p)[0], b = reinterpret_cast<const v4f*>(p)[1];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = a[e], v[4 + e] = b[e];
    } else {
        v[0] = *p;
    }
}
template <int VEC>
__device__ __forceinline__ void load_row(const __half* p, float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        const v8h a = *reinterpret_cast<const v8h*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (float)a[e];
    } else {
        v[0] = __half2float(*p);
    }
}
template <int VEC>
__device__ __forceinline__ void store_row(float* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        v4f a, b;
#pragma unroll
        for (int e = 0; e < 4; ++e) a[e] = v[e], b[e] = v[4 + e];
        reinterpret_cast<v4f*>(p)[0] = a;
        reinterpret_cast<v4f*>(p)[1] = b;
    } else {
        *p = v[0];
    }
}
template <int VEC>
__device__ __forceinline__ void store_row(__half* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        v8h a;
#pragma unroll
        for (int e = 0; e < 8; ++e) a[e] = (_Float16)v[e];
        *reinterpret_cast<v8h*>(p) = a;
    } else {
        *p = __float2half_rn(v[0]);
    }
}
// to the nearest e4m3, ties to even; |v| <= 448 up to a rounding of the quotient, which falls to 448
template <int VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&v)[VEC]) {
    if constexpr (VEC == 8) {
        v2u w;
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            int t = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * e], v[4 * e + 1], 0, false);
            w[e] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * e + 2], v[4 * e + 3], t, true);
        }
        *reinterpret_cast<v2u*>(p) = w;
    } else {
        *p = (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[0], 0, false) & 0xff);
    }
}

// LANES lanes have a row, VEC neighbouring elements of it each, NV times.  `residual` and `sum` are null together.
// (sum may be feat or residual: a lane has read its elements before it writes them, and nobody else reads them)
template <typename T, int VEC, int LANES, int NV>
__global__ void __launch_bounds__(kBlock)
rms_norm(const T* feat, const T* residual, const float* __restrict__ gamma, const int32_t* __restrict__ voxel_num, int max_voxels,
         int channel, float eps, uint8_t* __restrict__ q, float* __restrict__ scale, T* sum, int write_pad) {
    const int row = blockIdx.x * (kBlock / LANES) + threadIdx.x / LANES, lane = threadIdx.x % LANES;
    if (row >= max_voxels) return;
    const int n = clamp_rows(voxel_num, max_voxels);
    const size_t base = (size_t)row * channel;
    if (row >= n) {
        if (!write_pad) return;
        float zero[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) zero[e] = 0.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = (j * LANES + lane) * VEC;
            if (c >= channel) continue;
            store_e4m3<VEC>(q + base + c, zero);
            if (sum) store_row<VEC>(sum + base + c, zero);
        }
        if (lane == 0) scale[row] = 0.f;
        return;
    }
    float h[NV][VEC];
    float squares = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LANES + lane) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[j][e] = 0.f;
        if (c >= channel) continue;
        load_row<VEC>(feat + base + c, h[j]);
        if (residual) {
            float r[VEC];
            load_row<VEC>(residual + base + c, r);
#pragma unroll
            for (int e = 0; e < VEC; ++e) h[j][e] += r[e];
            store_row<VEC>(sum + base + c, h[j]);
        }
#pragma unroll
        for (int e = 0; e < VEC; ++e) squares = fmaf(h[j][e], h[j][e], squares);
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) squares += __shfl_xor(squares, d);
    const float mean = squares / (float)channel + eps;
    double rms = 1.f / sqrtf(mean);
    if (mean < 0x1p-100f) {  // (eps is as small: the squares are at the end of FP32, or beyond it)
        double sum64 = 0.;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int e = 0; e < VEC; ++e) sum64 = fma((double)h[j][e], (double)h[j][e], sum64);
#pragma unroll
        for (int d = LANES / 2; d > 0; d /= 2) sum64 += __shfl_xor(sum64, d);
        rms = 1. / sqrt(sum64 / channel + (double)eps);
    }
    float g[NV][VEC];
    double most = 0.;  // of |gamma h|, exact
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LANES + lane) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) g[j][e] = 0.f;
        if (c >= channel) continue;
        load_row<VEC>(gamma + c, g[j]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) most = fmax(most, fabs((double)h[j][e] * (double)g[j][e]));
    }
#pragma unroll
    for (int d = LANES / 2; d > 0; d /= 2) most = fmax(most, __shfl_xor(most, d));
    float s = (float)(most * rms / (double)kMost);
    double by = (double)kMost / most;
    if (!(s > kSmallestScale)) {
        s = kSmallestScale;
        by = rms / (double)kSmallestScale;
    }
    // fmax() drops NaN: whether the row had something that is not finite shows in its sum of squares
    if (!(mean <= FLT_MAX && rms <= DBL_MAX && s <= FLT_MAX)) {
        s = __int_as_float(0x7fc00000);
        by = (double)s;
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        const int c = (j * LANES + lane) * VEC;
        if (c >= channel) continue;
        float v[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = (float)((double)h[j][e] * (double)g[j][e] * by);
        store_e4m3<VEC>(q + base + c, v);
    }
    if (lane == 0) scale[row] = s;
}

struct NormArgs {
    const void *feat, *residual;
    const float* gamma;
    const int32_t* num;
    int max_voxels, channel;
    float eps;
    uint8_t* q;
    float* scale;
    void* sum;
    int write_pad;
};

template <typename T, int VEC, int LANES, int NV>
void launch_norm(const NormArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((rms_norm<T, VEC, LANES, NV>), dim3((unsigned)ceil_div(a.max_voxels, kBlock / LANES)), dim3(kBlock), 0, stream,
                       static_cast<const T*>(a.feat), static_cast<const T*>(a.residual), a.gamma, a.num, a.max_voxels, a.channel,
                       a.eps, a.q, a.scale, static_cast<T*>(a.sum), a.write_pad);
}

// Widths that are multiples of 8: 16 bytes of a row of halves to a lane and as many lanes as the row asks for, up to a wave; others an
// element to a lane.
template <typename T>
void launch_norm_width(const NormArgs& a, hipStream_t stream) {
    const int groups = a.channel % 8 == 0 ? a.channel / 8 : 0;
    if (groups == 1) launch_norm<T, 8, 1, 1>(a, stream);
    else if (groups == 2) launch_norm<T, 8, 2, 1>(a, stream);
    else if (groups && groups <= 4) launch_norm<T, 8, 4, 1>(a, stream);
    else if (groups && groups <= 8) launch_norm<T, 8, 8, 1>(a, stream);
    else if (groups && groups <= 16) launch_norm<T, 8, 16, 1>(a, stream);
    else if (groups && groups <= 32) launch_norm<T, 8, 32, 1>(a, stream);
    else if (groups && groups <= 64) launch_norm<T, 8, 64, 1>(a, stream);
    else if (groups && groups <= 128) launch_norm<T, 8, 64, 2>(a, stream);
    else if (groups && groups <= 256) launch_norm<T, 8, 64, 4>(a, stream);
    else if (groups) launch_norm<T, 8, 64, 8>(a, stream);
    else if (a.channel <= 64) launch_norm<T, 1, 64, 1>(a, stream);
    else if (a.channel <= 256) launch_norm<T, 1, 64, 4>(a, stream);
    else if (a.channel <= 1024) launch_norm<T, 1, 64, 16>(a, stream);
    else launch_norm<T, 1, 64, 64>(a, stream);
}

}  // namespace

int check_rows(const sessd_tensor_desc& d, int max_voxels, int channels, const char* who, const char* what) {
    if (d.nbDims != 3 || d.d[0] != 1 || d.d[1] != max_voxels || d.d[2] != channels)
        return fail(SESSD_E_INVALID, "%s: %s must be [1,%d,%d]", who, what, max_voxels, channels);
    return SESSD_OK;
}

bool is_scalar_int(const sessd_tensor_desc& d) {
    for (int i = 0; i < d.nbDims && i < 8; ++i)
        if (d.d[i] != 1) return false;
    return d.type == SESSD_INT32;
}

int check_device(int device, const char* who) {
    int current = 0;
    SESSD_HIP_TRY(hipGetDevice(&current));
    if (current != device) return fail(SESSD_E_INVALID, "%s: the layer was made on device %d, the current one is %d", who, device, current);
    return SESSD_OK;
}

RmsNormPlugin::~RmsNormPlugin() {
    if (gamma_dev_) (void)hipFree(gamma_dev_);
}

int RmsNormPlugin::create(const sessd_rmsnorm_desc& d, const float* gamma, RmsNormPlugin** out) {
    if (d.channel < 1 || d.max_voxels < 1) return fail(SESSD_E_INVALID, "rmsnorm: channel and max_voxels must be positive");
    if (d.channel > 4096 || d.max_voxels > kMostRows)
        return fail(SESSD_E_UNSUPPORTED, "rmsnorm: at most 4096 channels and %d rows (%d, %d)", kMostRows, d.channel, d.max_voxels);
    if (!(d.eps >= 0.f) || !std::isfinite(d.eps)) return fail(SESSD_E_INVALID, "rmsnorm: eps must be finite and not negative");
    for (int i = 0; i < d.channel; ++i)
        if (!std::isfinite(gamma[i])) return fail(SESSD_E_INVALID, "rmsnorm: gamma must be finite");
    std::unique_ptr<RmsNormPlugin> p(new RmsNormPlugin());
    p->channel_ = d.channel;
    p->max_voxels_ = d.max_voxels;
    p->eps_ = d.eps;
    p->gamma_.assign(gamma, gamma + d.channel);
    SESSD_HIP_TRY(hipGetDevice(&p->device_));
    SESSD_HIP_TRY(hipMalloc(reinterpret_cast<void**>(&p->gamma_dev_), d.channel * sizeof(float)));
    SESSD_HIP_TRY(hipMemcpy(p->gamma_dev_, gamma, d.channel * sizeof(float), hipMemcpyHostToDevice));
    *out = p.release();
    return SESSD_OK;
}

// channel, max_voxels, eps, gamma
size_t RmsNormPlugin::getSerializationSize() const { return 2 * sizeof(int) + (1 + gamma_.size()) * sizeof(float); }

void RmsNormPlugin::serialize(void* buffer) const {
    char* d = static_cast<char*>(buffer);
    writeToBuffer<int>(d, channel_);
    writeToBuffer<int>(d, max_voxels_);
    writeToBuffer<float>(d, eps_);
    for (float v : gamma_) writeToBuffer<float>(d, v);
}

int RmsNormPlugin::deserialize(const void* data, size_t length, RmsNormPlugin** out) {
    if (!data || length < 3 * sizeof(int)) return fail(SESSD_E_INVALID, "rmsnorm: blob too short");
    const char* d = static_cast<const char*>(data);
    sessd_rmsnorm_desc desc;
    desc.channel = readFromBuffer<int>(d);
    desc.max_voxels = readFromBuffer<int>(d);
    desc.eps = readFromBuffer<float>(d);
    if (desc.channel < 1 || (length - 3 * sizeof(int)) / sizeof(float) < (size_t)desc.channel)
        return fail(SESSD_E_INVALID, "rmsnorm: blob too short for %d channels", desc.channel);
    std::vector<float> gamma((size_t)desc.channel);
    std::memcpy(gamma.data(), d, gamma.size() * sizeof(float));
    return create(desc, gamma.data(), out);
}

int RmsNormPlugin::check(const sessd_tensor_desc* in, const sessd_tensor_desc* out, bool residual) const {
    const char* who = "rmsnorm";
    if (in[0].type != SESSD_FLOAT && in[0].type != SESSD_HALF) return fail(SESSD_E_UNSUPPORTED, "rmsnorm: features must be FP32 or FP16");
    SESSD_TRY(check_rows(in[0], max_voxels_, channel_, who, "feat"));
    SESSD_TRY(check_rows(out[0], max_voxels_, channel_, who, "q"));
    SESSD_TRY(check_rows(out[1], max_voxels_, 1, who, "scale"));
    if (!is_scalar_int(in[1])) return fail(SESSD_E_INVALID, "rmsnorm: voxel_num must be one INT32");
    if (out[0].type != SESSD_FP8 || out[1].type != SESSD_FLOAT) return fail(SESSD_E_UNSUPPORTED, "rmsnorm: q must be FP8 and scale FP32");
    if (residual) {
        SESSD_TRY(check_rows(in[2], max_voxels_, channel_, who, "residual"));
        SESSD_TRY(check_rows(out[2], max_voxels_, channel_, who, "sum"));
        if (in[2].type != in[0].type || out[2].type != in[0].type)
            return fail(SESSD_E_UNSUPPORTED, "rmsnorm: residual and sum must have the features' type");
    }
    return SESSD_OK;
}

int RmsNormPlugin::configurePlugin(const sessd_tensor_desc* in, int nbInputs, const sessd_tensor_desc* out, int nbOutputs) {
    if (!in || !out || !((nbInputs == 2 && nbOutputs == 2) || (nbInputs == 3 && nbOutputs == 3)))
        return fail(SESSD_E_INVALID, "rmsnorm.configure: expected 2 inputs and 2 outputs, or 3 and 3 with a residual");
    SESSD_TRY(check(in, out, nbInputs == 3));
    residual_ = nbInputs == 3;
    type_ = in[0].type;
    return SESSD_OK;
}

int RmsNormPlugin::enqueue(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                           void* const* outputs, void*, hipStream_t stream) {
    if (!inputDesc || !outputDesc || !inputs || !outputs) return fail(SESSD_E_INVALID, "rmsnorm.enqueue: null argument");
    const int tensors = residual_ ? 3 : 2;
    for (int i = 0; i < tensors; ++i) {
        if (!inputs[i] || !outputs[i]) return fail(SESSD_E_INVALID, "rmsnorm.enqueue: null tensor pointer");
        if ((i != 1 && reinterpret_cast<uintptr_t>(inputs[i]) & 15) || reinterpret_cast<uintptr_t>(outputs[i]) & 15)
            return fail(SESSD_E_INVALID, "rmsnorm.enqueue: tensors must be 16-byte aligned");
    }
    if (inputDesc[0].type != type_) return fail(SESSD_E_INVALID, "rmsnorm.enqueue: tensor dtypes differ from the configured ones");
    SESSD_TRY(check(inputDesc, outputDesc, residual_));
    SESSD_TRY(check_device(device_, "rmsnorm.enqueue"));
    NormArgs a;
    a.feat = inputs[0];
    a.residual = residual_ ? inputs[2] : nullptr;
    a.gamma = gamma_dev_;
    a.num = static_cast<const int32_t*>(inputs[1]);
    a.max_voxels = max_voxels_;
    a.channel = channel_;
    a.eps = eps_;
    a.q = static_cast<uint8_t*>(outputs[0]);
    a.scale = static_cast<float*>(outputs[1]);
    a.sum = residual_ ? outputs[2] : nullptr;
    a.write_pad = (flags_ & SESSD_FLAG_SKIP_PAD_ROWS) ? 0 : 1;
    if (type_ == SESSD_HALF) launch_norm_width<__half>(a, stream);
    else launch_norm_width<float>(a, stream);
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

}  // namespace sessd

// linear8.hip -- Linear8Plugin: rows in e4m3 with a scale each times weights in e4m3 with a scale for each column.
//
//   out[i][c] = epilogue_c( (sum_k q[i][k] * wq[k][c]) * scale[i] * wscale[c] )
//
// An e4m3 value is a half, so the rows are widened in registers (the weights at create) and multiplied by the FP16 matrix
// instructions: products are exact, sums FP32, and one rounding to the output's type follows the epilogue.  The 8-bit matrix
// instructions add with fewer bits: 512 -> 128 channels were 1.4e-5 of the result's norm from the 64-bit sums, 5e-8 these.
// The product is taken transposed, D = Wq^T Q^T: a lane of the result has one row and, with the weights'
// columns dealt to the instructions as they are, 16 neighbouring columns of it, which it stores as whole 16-byte words.
// What bounds the layer at this library's widths is the output it writes.
#include <cmath>

#include "plugins.h"

namespace sessd {

namespace {

constexpr int kBlock = 256;
constexpr int kColumns = 64;  // of a wave: four instructions, 16 each
constexpr int kRows = 16;     // of a wave
constexpr int kStep = 32;     // values of k to an instruction

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef unsigned int v2u __attribute__((ext_vector_type(2)));

__device__ __forceinline__ v8h widen(v2u x) {
    const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[0], 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[0], 1.f, true);
    const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[1], 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x[1], 1.f, true);
    return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

// column of the 64 that row `i` of instruction `t` stands for: lane group g (rows 4g .. 4g + 3) gets 16g .. 16g + 15 over the four
__host__ __device__ constexpr int column_of(int t, int i) { return 16 * (i / 4) + 4 * t + i % 4; }

template <typename T>
__device__ __forceinline__ void store_columns(T* dst, const float (&v)[16], int left, bool wide) {
    if (wide && left >= 16) {
        if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                v8h x;
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (_Float16)v[8 * h + e];
                reinterpret_cast<v8h*>(dst)[h] = x;
            }
        } else {
#pragma unroll
            for (int h = 0; h < 4; ++h) {
                v4f x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = v[4 * h + e];
                reinterpret_cast<v4f*>(dst)[h] = x;
            }
        }
        return;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e)
        if (e < left) {
            if constexpr (sizeof(T) == 2) dst[e] = __float2half_rn(v[e]);
            else dst[e] = v[e];
        }
}

template <typename T>
__global__ void __launch_bounds__(kBlock)
linear8(const uint8_t* __restrict__ q, const float* __restrict__ scale, const int32_t* __restrict__ voxel_num, int max_voxels,
        int cin, int cout, const __half* __restrict__ w, const float* __restrict__ columns, int cout_pad, int relu,
        T* __restrict__ out, int write_pad) {
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int row = (blockIdx.x * (kBlock / 64) + (threadIdx.x >> 6)) * kRows + r;
    const int n = clamp_rows(voxel_num, max_voxels);
    const int cb = blockIdx.y;
    const int steps = (cin + kStep - 1) / kStep;
    const bool active = row < n;
    v4f acc[4] = {};
    const __half* wp = w + ((size_t)cb * steps * 4 * 64 + lane) * 8;
    const uint8_t* qp = q + (size_t)row * cin + g * 8;
    for (int ks = 0; ks < steps; ++ks) {
        v2u x = {};
        if (active && ks * kStep + g * 8 < cin) x = *reinterpret_cast<const v2u*>(qp + ks * kStep);
        const v8h b = widen(x);
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const v8h a = *reinterpret_cast<const v8h*>(wp + (size_t)(ks * 4 + t) * 64 * 8);
            acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, acc[t], 0, 0, 0);
        }
    }
    if (row >= max_voxels || (!active && !write_pad)) return;
    const float s = active ? scale[row] : 0.f;
    const int c0 = cb * kColumns + 16 * g;
    if (c0 >= cout) return;
    const v4f* col = reinterpret_cast<const v4f*>(columns + c0);
    float v[16];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const v4f ws = col[t], sc = col[cout_pad / 4 + t], sh = col[cout_pad / 2 + t];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            float y = acc[t][e] * s * ws[e] * sc[e] + sh[e];
            if (relu) y = y < 0.f ? 0.f : y;
            v[4 * t + e] = y;
        }
    }
    store_columns(out + (size_t)row * cout + c0, v, cout - c0, cout % (16 / (int)sizeof(T)) == 0);
}

// |v| <= 448 up to a rounding of the quotient: the nearest e4m3, ties to even, as a half
uint16_t nearest_e4m3(float v) {
    const float a = std::fabs(v);
    const int e = a < 0x1p-6f ? -6 : std::ilogb(a);  // -6: the exponent of the subnormal values as well
    const float r = std::ldexp(std::nearbyintf(std::ldexp(a, 3 - e)), e - 3), most = r > 448.f ? 448.f : r;
    float value;
    return nearest_half(std::copysign(most, v), &value);
}

int padded_columns(int cout) { return ceil_div(cout, kColumns) * kColumns; }

}  // namespace

Linear8Plugin::~Linear8Plugin() {
    if (weights_packed_dev_) (void)hipFree(weights_packed_dev_);
    if (columns_dev_) (void)hipFree(columns_dev_);
}

int Linear8Plugin::create(const sessd_linear8_desc& d, const float* weights, Linear8Plugin** out) {
    if (d.in_channel < 1 || d.out_channel < 1 || d.max_voxels < 1)
        return fail(SESSD_E_INVALID, "linear8: in_channel, out_channel and max_voxels must be positive");
    if (d.in_channel % 16 || d.in_channel > 4096 || d.out_channel > 4096)
        return fail(SESSD_E_UNSUPPORTED, "linear8: in_channel must be a multiple of 16 up to 4096, out_channel at most 4096 (%d, %d)",
                    d.in_channel, d.out_channel);
    const int cin = d.in_channel, cout = d.out_channel;
    for (size_t i = 0; i < (size_t)cin * cout; ++i)
        if (!std::isfinite(weights[i])) return fail(SESSD_E_INVALID, "linear8: the weights must be finite");
    std::unique_ptr<Linear8Plugin> p(new Linear8Plugin());
    p->in_channel_ = cin;
    p->out_channel_ = cout;
    p->max_voxels_ = d.max_voxels;
    p->weights_.assign(weights, weights + (size_t)cin * cout);
    p->wscale_.assign((size_t)cout, 0.f);
    for (int k = 0; k < cin; ++k)
        for (int c = 0; c < cout; ++c) p->wscale_[c] = std::fmax(p->wscale_[c], std::fabs(weights[(size_t)k * cout + c]));
    for (float& s : p->wscale_) s = std::fmax(s / 448.f, 0x1p-100f);
    const int steps = ceil_div(cin, kStep), blocks = ceil_div(cout, kColumns);
    std::vector<uint16_t> packed((size_t)blocks * steps * 4 * 64 * 8, 0);
    for (int cb = 0; cb < blocks; ++cb)
        for (int ks = 0; ks < steps; ++ks)
            for (int t = 0; t < 4; ++t)
                for (int lane = 0; lane < 64; ++lane) {
                    const int c = cb * kColumns + column_of(t, lane & 15);
                    uint16_t* dst = packed.data() + ((((size_t)cb * steps + ks) * 4 + t) * 64 + lane) * 8;
                    for (int e = 0; e < 8; ++e) {
                        const int k = ks * kStep + (lane >> 4) * 8 + e;
                        if (c < cout && k < cin) dst[e] = nearest_e4m3(weights[(size_t)k * cout + c] / p->wscale_[c]);
                    }
                }
    SESSD_HIP_TRY(hipMalloc(reinterpret_cast<void**>(&p->weights_packed_dev_), packed.size() * sizeof(uint16_t)));
    SESSD_HIP_TRY(hipMemcpy(p->weights_packed_dev_, packed.data(), packed.size() * sizeof(uint16_t), hipMemcpyHostToDevice));
    SESSD_TRY(p->uploadColumns());
    *out = p.release();
    return SESSD_OK;
}

// wscale, scale, shift for whole blocks of columns
int Linear8Plugin::uploadColumns() {
    const size_t pad = (size_t)padded_columns(out_channel_);
    std::vector<float> host(3 * pad, 0.f);
    for (int c = 0; c < out_channel_; ++c) {
        host[c] = wscale_[c];
        host[pad + c] = epi_.scale_host.empty() ? 1.f : epi_.scale_host[c];
        host[2 * pad + c] = epi_.shift_host.empty() ? 0.f : epi_.shift_host[c];
    }
    if (!columns_dev_) SESSD_HIP_TRY(hipMalloc(reinterpret_cast<void**>(&columns_dev_), host.size() * sizeof(float)));
    SESSD_HIP_TRY(hipMemcpy(columns_dev_, host.data(), host.size() * sizeof(float), hipMemcpyHostToDevice));
    return SESSD_OK;
}

int Linear8Plugin::setEpilogue(const float* scale, const float* shift, int relu) {
    Epilogue e;
    e.relu = relu ? 1 : 0;
    if (scale) e.scale_host.assign(scale, scale + out_channel_);
    if (shift) e.shift_host.assign(shift, shift + out_channel_);
    epi_ = e;
    return uploadColumns();
}

// in_channel, out_channel, max_voxels, weights, the epilogue as the convolutions write it
size_t Linear8Plugin::getSerializationSize() const {
    return 3 * sizeof(int) + weights_.size() * sizeof(float) + conv_epilogue_trailer_size(epi_);
}

void Linear8Plugin::serialize(void* buffer) const {
    char* d = static_cast<char*>(buffer);
    writeToBuffer<int>(d, in_channel_);
    writeToBuffer<int>(d, out_channel_);
    writeToBuffer<int>(d, max_voxels_);
    for (float v : weights_) writeToBuffer<float>(d, v);
    conv_write_epilogue_trailer(d, epi_);
}

int Linear8Plugin::deserialize(const void* data, size_t length, Linear8Plugin** out) {
    if (!data || length < 3 * sizeof(int)) return fail(SESSD_E_INVALID, "linear8: blob too short");
    const char* d = static_cast<const char*>(data);
    sessd_linear8_desc desc;
    desc.in_channel = readFromBuffer<int>(d);
    desc.out_channel = readFromBuffer<int>(d);
    desc.max_voxels = readFromBuffer<int>(d);
    if (desc.in_channel < 1 || desc.out_channel < 1 || desc.in_channel > 4096 || desc.out_channel > 4096)
        return fail(SESSD_E_INVALID, "linear8: blob with %d x %d channels", desc.in_channel, desc.out_channel);
    const size_t count = (size_t)desc.in_channel * desc.out_channel;
    size_t left = length - 3 * sizeof(int);
    if (left / sizeof(float) < count) return fail(SESSD_E_INVALID, "linear8: blob too short for its weights");
    std::vector<float> w(count);
    std::memcpy(w.data(), d, count * sizeof(float));
    d += count * sizeof(float);
    left -= count * sizeof(float);
    Linear8Plugin* p = nullptr;
    SESSD_TRY(create(desc, w.data(), &p));
    std::unique_ptr<Linear8Plugin> own(p);
    Epilogue e;
    SESSD_TRY(read_epilogue(d, left, desc.out_channel, &e));
    if (!e.scale_host.empty() || !e.shift_host.empty() || e.relu)
        SESSD_TRY(p->setEpilogue(e.scale_host.empty() ? nullptr : e.scale_host.data(), e.shift_host.empty() ? nullptr : e.shift_host.data(), e.relu));
    *out = own.release();
    return SESSD_OK;
}

int Linear8Plugin::check(const sessd_tensor_desc* in, const sessd_tensor_desc* out) const {
    const char* who = "linear8";
    if (in[0].type != SESSD_FP8 || in[1].type != SESSD_FLOAT) return fail(SESSD_E_UNSUPPORTED, "linear8: q must be FP8 and scale FP32");
    if (out[0].type != SESSD_FLOAT && out[0].type != SESSD_HALF) return fail(SESSD_E_UNSUPPORTED, "linear8: the output must be FP32 or FP16");
    SESSD_TRY(check_rows(in[0], max_voxels_, in_channel_, who, "q"));
    SESSD_TRY(check_rows(in[1], max_voxels_, 1, who, "scale"));
    SESSD_TRY(check_rows(out[0], max_voxels_, out_channel_, who, "the output"));
    if (!is_scalar_int(in[2])) return fail(SESSD_E_INVALID, "linear8: voxel_num must be one INT32");
    return SESSD_OK;
}

int Linear8Plugin::configurePlugin(const sessd_tensor_desc* in, int nbInputs, const sessd_tensor_desc* out, int nbOutputs) {
    if (!in || !out || nbInputs != 3 || nbOutputs != 1) return fail(SESSD_E_INVALID, "linear8.configure: expected 3 inputs and 1 output");
    SESSD_TRY(check(in, out));
    out_type_ = out[0].type;
    return SESSD_OK;
}

int Linear8Plugin::enqueue(const sessd_tensor_desc* inputDesc, const sessd_tensor_desc* outputDesc, const void* const* inputs,
                           void* const* outputs, void*, hipStream_t stream) {
    if (!inputDesc || !outputDesc || !inputs || !outputs) return fail(SESSD_E_INVALID, "linear8.enqueue: null argument");
    if (!inputs[0] || !inputs[1] || !inputs[2] || !outputs[0]) return fail(SESSD_E_INVALID, "linear8.enqueue: null tensor pointer");
    if (outputDesc[0].type != out_type_) return fail(SESSD_E_INVALID, "linear8.enqueue: tensor dtypes differ from the configured ones");
    SESSD_TRY(check(inputDesc, outputDesc));
    if ((reinterpret_cast<uintptr_t>(inputs[0]) | reinterpret_cast<uintptr_t>(inputs[1]) | reinterpret_cast<uintptr_t>(outputs[0])) & 15)
        return fail(SESSD_E_INVALID, "linear8.enqueue: tensors must be 16-byte aligned");
    const dim3 grid((unsigned)ceil_div(max_voxels_, kRows * (kBlock / 64)), (unsigned)ceil_div(out_channel_, kColumns));
    const int pad = padded_columns(out_channel_), write_pad = (flags_ & SESSD_FLAG_SKIP_PAD_ROWS) ? 0 : 1;
#define SESSD_LINEAR8(T)                                                                                                              \
    hipLaunchKernelGGL(linear8<T>, grid, dim3(kBlock), 0, stream, static_cast<const uint8_t*>(inputs[0]),                             \
                       static_cast<const float*>(inputs[1]), static_cast<const int32_t*>(inputs[2]), max_voxels_, in_channel_,        \
                       out_channel_, weights_packed_dev_, columns_dev_, pad, epi_.relu, static_cast<T*>(outputs[0]), write_pad)
    if (out_type_ == SESSD_HALF) SESSD_LINEAR8(__half);
    else SESSD_LINEAR8(float);
#undef SESSD_LINEAR8
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

}  // namespace sessd

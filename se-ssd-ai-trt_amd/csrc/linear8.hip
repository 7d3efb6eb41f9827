// linear8.hip -- Linear8Plugin: rows in e4m3 with a scale each times weights in e4m3 with a scale for each column.
//
//   out[i][c] = epilogue_c( (sum_k q[i][k] * wq[k][c]) * scale[i] * wscale[c] )
//
// An e4m3 value is a half, so the rows are widened in registers (the weights at create) and multiplied by the FP16 matrix
// instructions: products are exact, sums FP32, and one rounding to the output's type follows the epilogue.  The 8-bit matrix
// instructions add with fewer bits: 512 -> 128 channels were 1.4e-5 of the result's norm from the 64-bit sums, 5e-8 these.
// The product is taken transposed, D = Wq^T Q^T: a lane of the result has one row and, with the weights' columns dealt to the
// instructions as they are, 8 or 16 neighbouring columns of it, which it stores as whole 16-byte words.
//
// Up to kMostHeld input channels a wave keeps the weights of its columns (64, or 32 where the channels are many) in registers, 128 of
// them at most, and takes one block of 16 rows after the other, the next one's values requested while it multiplies: nothing of the
// weights is read twice, nothing goes through LDS but the epilogue's constants, and no wave waits for another.  The waves of a
// workgroup have neighbouring columns of the same rows.  What bounds it then is the output it writes: 150 000 rows 256 -> 1024 FP16 102 us, 3.6 TB/s and
// 770 TFLOP/s; 60 000 rows 512 -> 128 FP32, 7.3 blocks for each wave, 21 us; weights read anew for every 16 rows 266 and 30 us.  Inputs beyond
// kMostHeld, whose weights no wave's registers hold, do read them anew: 150 000 rows 1024 -> 256 FP16 248 us, 60 000 rows 2048 -> 512 FP32 368.
#include <cmath>
#include <utility>

#include "plugins.h"

namespace sessd {

namespace {

constexpr int kBlock = 256;
constexpr int kRows = 16;      // of a wave at a time
constexpr int kMostHeld = 512;
constexpr int kGroups = 512;   // workgroups of the kernel that holds its weights: two for each compute unit

// instructions, 16 columns each, of a wave: as many as leave the held weights 128 registers
constexpr int tiles_of(int cin) { return cin > 256 && cin <= kMostHeld ? 2 : 4; }
// Rows and weights meet in 64 input channels at a time, two instructions: lane group g has 16 neighbouring channels of each row, 8 to either
constexpr int pairs_of(int cin) { return (cin + 63) / 64; }
constexpr int channel_of(int step, int g, int e) { return step / 2 * 64 + g * 16 + step % 2 * 8 + e; }
// Column that row `i` of instruction `t` stands for: a lane (its group g has rows 4 g .. 4 g + 3) gets 16 bytes of neighbouring columns from each
// instruction in FP32 and from each two in FP16, and the four groups of a store 64 bytes of a row
constexpr int column_of(bool half, int t, int i) { return half ? 32 * (t / 2) + 8 * (i / 4) + 4 * (t % 2) + i % 4 : 16 * t + i; }

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef unsigned int v4u __attribute__((ext_vector_type(4)));

__device__ __forceinline__ v8h widen(unsigned x, unsigned y) {
    const v2h a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(x, 1.f, true);
    const v2h c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(y, 1.f, true);
    return v8h{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

struct LinearArgs {
    const uint8_t* q;
    const float* scale;
    const int32_t* voxel_num;
    int max_voxels, cin, cout, write_pad;
    const __half* w;       // [block of columns][step][instruction][lane][8]
    const float* columns;  // of the result: factor, addend, two rows of whole blocks; behind them 1 for a ReLU
    void* out;
};

// (past the caches: 150 000 x 256 -> 1024 150 us through them, 102 like this)
template <typename V>
__device__ __forceinline__ void put(V* to, const V& x) {
    __builtin_nontemporal_store(x, to);
}

// A lane's 4 NT columns of a row, of the block of columns from `c0` on
template <typename T, int NT>
__device__ __forceinline__ void store_columns(const LinearArgs& a, int row, int c0, const v4f (&acc)[NT], float s, const float* factor, const float* addend, bool relu, int g) {
    constexpr bool kHalf = sizeof(T) == 2;
    T* const dst = static_cast<T*>(a.out) + (size_t)row * a.cout + c0;
    const bool whole = a.cout % (16 / (int)sizeof(T)) == 0 && c0 + 16 * NT <= a.cout;
    float y[NT][4];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
        const int c = column_of(kHalf, t, 4 * g);
        const v4f f = *reinterpret_cast<const v4f*>(factor + c), b = *reinterpret_cast<const v4f*>(addend + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) y[t][e] = fmaf(acc[t][e] * s, f[e], b[e]);
    }
    if (relu) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[t][e] = y[t][e] < 0.f ? 0.f : y[t][e];
    }
    if (!whole) {
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = column_of(kHalf, t, 4 * g) + e;
                if (c0 + c >= a.cout) continue;
                if constexpr (kHalf) dst[c] = __float2half_rn(y[t][e]);
                else dst[c] = y[t][e];
            }
    } else if constexpr (kHalf) {
#pragma unroll
        for (int t = 0; t < NT; t += 2) {
            v8h x;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = (_Float16)y[t + e / 4][e % 4];
            put(reinterpret_cast<v8h*>(dst + column_of(true, t, 4 * g)), x);
        }
    } else {
#pragma unroll
        for (int t = 0; t < NT; ++t) put(reinterpret_cast<v4f*>(dst + column_of(false, t, 4 * g)), v4f{y[t][0], y[t][1], y[t][2], y[t][3]});
    }
}

// PAIRS: of 64 input channels
template <typename T, int PAIRS, int NT>
__global__ void __launch_bounds__(kBlock, 2)
linear8_held(LinearArgs a) {
    constexpr int kWide = 16 * NT;
    __shared__ __align__(16) float s_columns[kBlock / 64][2][kWide];
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4, wave = threadIdx.x >> 6;
    // (workgroups go to the eight dies in turn: neighbours in rows and columns on one of them)
    const int group = gridDim.x % 8 ? (int)blockIdx.x : (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8);
    const int blocks = (a.cout + kWide - 1) / kWide, id = group * (kBlock / 64) + wave;
    const int cb = id % blocks, stream = id / blocks, streams = (int)gridDim.x * (kBlock / 64) / blocks;
    if (stream >= streams) return;  // (what is left over; no wave waits for another)
    v8h w[2 * PAIRS][NT];
    const v8h* from = reinterpret_cast<const v8h*>(a.w) + (size_t)cb * 2 * PAIRS * NT * 64 + lane;
#pragma unroll
    for (int s = 0; s < 2 * PAIRS; ++s)
#pragma unroll
        for (int t = 0; t < NT; ++t) w[s][t] = from[(s * NT + t) * 64];
    if (lane < kWide)
#pragma unroll
        for (int i = 0; i < 2; ++i) s_columns[wave][i][lane] = a.columns[i * blocks * kWide + cb * kWide + lane];
    const bool relu = a.columns[2 * blocks * kWide] != 0.f;
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    const int n = clamp_rows(a.voxel_num, a.max_voxels), rows = a.write_pad ? a.max_voxels : n;
    v4u x[PAIRS];
    float scale;
    const bool whole = a.cin % 64 == 0;
    // 16 rows' values, zeros behind the last one (for most blocks without a branch, which each load would wait in front of)
    const auto request = [&](int first) {
        const uint8_t* const at = a.q + (size_t)(first + r) * a.cin + g * 16;
        if (whole && first + kRows <= n) {
            scale = a.scale[first + r];
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) x[p] = *reinterpret_cast<const v4u*>(at + p * 64);
        } else {
            scale = 0.f;
            if (first + r < n) scale = a.scale[first + r];
#pragma unroll
            for (int p = 0; p < PAIRS; ++p) {
                x[p] = v4u{0, 0, 0, 0};
                if (first + r < n && p * 64 + g * 16 < a.cin) x[p] = *reinterpret_cast<const v4u*>(at + p * 64);
            }
        }
    };
    const int turn = streams * kRows;
    request(stream * kRows);
    for (int first = stream * kRows; first < rows; first += turn) {
        v8h b[2 * PAIRS];
#pragma unroll
        for (int p = 0; p < PAIRS; ++p) {
            b[2 * p] = widen(x[p][0], x[p][1]);
            b[2 * p + 1] = widen(x[p][2], x[p][3]);
        }
        const float s = scale;
        request(first + turn);
        v4f acc[NT] = {};
#pragma unroll
        for (int k = 0; k < 2 * PAIRS; ++k)
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[k][t], b[k], acc[t], 0, 0, 0);
        if (first + r < rows) store_columns<T, NT>(a, first + r, cb * kWide, acc, s, s_columns[wave][0], s_columns[wave][1], relu, g);
    }
}

template <typename T>
__global__ void __launch_bounds__(kBlock)
linear8_wide(LinearArgs a) {
    constexpr int NT = 4, kWide = 16 * NT;
    const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
    const int row = ((int)blockIdx.x * (kBlock / 64) + (int)(threadIdx.x >> 6)) * kRows + r;
    const int n = clamp_rows(a.voxel_num, a.max_voxels), cb = blockIdx.y, blocks = gridDim.y, pairs = (a.cin + 63) / 64;
    v4f acc[NT] = {};
    const v8h* w = reinterpret_cast<const v8h*>(a.w) + (size_t)cb * 2 * pairs * NT * 64 + lane;
    for (int p = 0; p < pairs; ++p) {
        v4u x = {0, 0, 0, 0};
        if (row < n && p * 64 + g * 16 < a.cin) x = *reinterpret_cast<const v4u*>(a.q + (size_t)row * a.cin + p * 64 + g * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const v8h b = widen(x[2 * h], x[2 * h + 1]);
#pragma unroll
            for (int t = 0; t < NT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(w[((2 * p + h) * NT + t) * 64], b, acc[t], 0, 0, 0);
        }
    }
    if (row >= a.max_voxels || (row >= n && !a.write_pad)) return;
    store_columns<T, NT>(a, row, cb * kWide, acc, row < n ? a.scale[row] : 0.f, a.columns + cb * kWide, a.columns + (blocks + cb) * kWide, a.columns[2 * blocks * kWide] != 0.f, g);
}

template <typename T>
void launch_linear8(const LinearArgs& a, hipStream_t stream) {
    const int rows16 = ceil_div(a.max_voxels, kRows), blocks = ceil_div(a.cout, 16 * tiles_of(a.cin));
    if (a.cin > kMostHeld) {
        hipLaunchKernelGGL(linear8_wide<T>, dim3((unsigned)ceil_div(rows16, kBlock / 64), (unsigned)blocks), dim3(kBlock), 0, stream, a);
        return;
    }
    // (at least a wave for each block of columns)
    const int64_t most = ceil_div((int64_t)rows16 * blocks, kBlock / 64);
    const int groups = most < kGroups ? (int)most : kGroups > ceil_div(blocks, kBlock / 64) ? kGroups : ceil_div(blocks, kBlock / 64);
#define SESSD_HELD(P, NT) hipLaunchKernelGGL((linear8_held<T, P, NT>), dim3((unsigned)groups), dim3(kBlock), 0, stream, a)
    switch (pairs_of(a.cin)) {
        case 1: SESSD_HELD(1, 4); break;
        case 2: SESSD_HELD(2, 4); break;
        case 3: SESSD_HELD(3, 4); break;
        case 4: SESSD_HELD(4, 4); break;
        case 5: SESSD_HELD(5, 2); break;
        case 6: SESSD_HELD(6, 2); break;
        case 7: SESSD_HELD(7, 2); break;
        default: SESSD_HELD(8, 2); break;
    }
#undef SESSD_HELD
}

// |v| <= 448 up to a rounding of the quotient: the nearest e4m3, ties to even, as a half
uint16_t nearest_e4m3(float v) {
    const float a = std::fabs(v);
    const int e = a < 0x1p-6f ? -6 : std::ilogb(a);  // -6: the exponent of the subnormal values as well
    const float r = std::ldexp(std::nearbyintf(std::ldexp(a, 3 - e)), e - 3), most = r > 448.f ? 448.f : r;
    float value;
    return nearest_half(std::copysign(most, v), &value);
}

int padded_columns(int cin, int cout) { return ceil_div(cout, 16 * tiles_of(cin)) * 16 * tiles_of(cin); }

}  // namespace

Linear8Plugin::~Linear8Plugin() {
    if (weights_packed_dev_) (void)hipFree(weights_packed_dev_);
    if (columns_dev_) (void)hipFree(columns_dev_);
}

int Linear8Plugin::create(const sessd_linear8_desc& d, const float* weights, Linear8Plugin** out) {
    if (d.in_channel < 1 || d.out_channel < 1 || d.max_voxels < 1)
        return fail(SESSD_E_INVALID, "linear8: in_channel, out_channel and max_voxels must be positive");
    if (d.in_channel % 16 || d.in_channel > 4096 || d.out_channel > 4096 || d.max_voxels > kMostRows)
        return fail(SESSD_E_UNSUPPORTED, "linear8: in_channel must be a multiple of 16 up to 4096, out_channel at most 4096, max_voxels at most %d (%d, %d, %d)",
                    kMostRows, d.in_channel, d.out_channel, d.max_voxels);
    const int cin = d.in_channel, cout = d.out_channel;
    for (size_t i = 0; i < (size_t)cin * cout; ++i)
        if (!std::isfinite(weights[i])) return fail(SESSD_E_INVALID, "linear8: the weights must be finite");
    std::unique_ptr<Linear8Plugin> p(new Linear8Plugin());
    p->in_channel_ = cin;
    p->out_channel_ = cout;
    p->max_voxels_ = d.max_voxels;
    SESSD_HIP_TRY(hipGetDevice(&p->device_));
    p->weights_.assign(weights, weights + (size_t)cin * cout);
    p->wscale_.assign((size_t)cout, 0.f);
    for (int k = 0; k < cin; ++k)
        for (int c = 0; c < cout; ++c) p->wscale_[c] = std::fmax(p->wscale_[c], std::fabs(weights[(size_t)k * cout + c]));
    for (float& s : p->wscale_) s = std::fmax(s / 448.f, 0x1p-100f);
    const int tiles = tiles_of(cin), steps = 2 * pairs_of(cin), blocks = padded_columns(cin, cout) / (16 * tiles);
    const size_t count = (size_t)blocks * steps * tiles * 64 * 8;
    std::vector<uint16_t> packed(count);
    SESSD_HIP_TRY(hipMalloc(reinterpret_cast<void**>(&p->weights_packed_dev_), 2 * count * sizeof(uint16_t)));
    for (const bool half : {false, true}) {  // (the order of the columns is the output's)
        for (int cb = 0; cb < blocks; ++cb)
            for (int s = 0; s < steps; ++s)
                for (int t = 0; t < tiles; ++t)
                    for (int lane = 0; lane < 64; ++lane) {
                        const int c = cb * 16 * tiles + column_of(half, t, lane & 15);
                        uint16_t* dst = packed.data() + ((((size_t)cb * steps + s) * tiles + t) * 64 + lane) * 8;
                        for (int e = 0; e < 8; ++e) {
                            const int k = channel_of(s, lane >> 4, e);
                            dst[e] = c < cout && k < cin ? nearest_e4m3(weights[(size_t)k * cout + c] / p->wscale_[c]) : 0;
                        }
                    }
        SESSD_HIP_TRY(hipMemcpy(p->weights_packed_dev_ + (half ? count : 0), packed.data(), count * sizeof(uint16_t), hipMemcpyHostToDevice));
    }
    p->packed_count_ = count;
    SESSD_TRY(p->uploadColumns(p->epi_));
    *out = p.release();
    return SESSD_OK;
}

// Factor and addend of a column, for whole blocks of columns, and whether there is a ReLU.  All of it is in device memory, at an address that stays:
// calls in a captured graph have the new epilogue as a whole from their next replay on.  Queued calls on any stream may still read the old one.
// hipMemcpy waits for the default stream alone, hipFree for all that the device has.
int Linear8Plugin::uploadColumns(const Epilogue& e) {
    const size_t pad = (size_t)padded_columns(in_channel_, out_channel_);
    std::vector<float> host(2 * pad + 1, 0.f);
    for (int c = 0; c < out_channel_; ++c) {
        host[c] = e.scale_host.empty() ? wscale_[c] : wscale_[c] * e.scale_host[c];
        host[pad + c] = e.shift_host.empty() ? 0.f : e.shift_host[c];
    }
    host[2 * pad] = e.relu ? 1.f : 0.f;
    if (columns_dev_) {
        void* wait = nullptr;
        SESSD_HIP_TRY(hipMalloc(&wait, 256));
        SESSD_HIP_TRY(hipFree(wait));
    } else {
        SESSD_HIP_TRY(hipMalloc(reinterpret_cast<void**>(&columns_dev_), host.size() * sizeof(float)));
    }
    SESSD_HIP_TRY(hipMemcpy(columns_dev_, host.data(), host.size() * sizeof(float), hipMemcpyHostToDevice));
    return SESSD_OK;
}

int Linear8Plugin::setEpilogue(const float* scale, const float* shift, int relu) {
    SESSD_TRY(check_device(device_, "linear8.set_epilogue"));
    Epilogue e;
    e.relu = relu ? 1 : 0;
    if (scale) e.scale_host.assign(scale, scale + out_channel_);
    if (shift) e.shift_host.assign(shift, shift + out_channel_);
    SESSD_TRY(uploadColumns(e));
    epi_ = std::move(e);
    return SESSD_OK;
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
    SESSD_TRY(check_device(device_, "linear8.enqueue"));
    LinearArgs a;
    a.q = static_cast<const uint8_t*>(inputs[0]);
    a.scale = static_cast<const float*>(inputs[1]);
    a.voxel_num = static_cast<const int32_t*>(inputs[2]);
    a.max_voxels = max_voxels_;
    a.cin = in_channel_;
    a.cout = out_channel_;
    a.write_pad = (flags_ & SESSD_FLAG_SKIP_PAD_ROWS) ? 0 : 1;
    a.w = weights_packed_dev_ + (out_type_ == SESSD_HALF ? packed_count_ : 0);
    a.columns = columns_dev_;
    a.out = outputs[0];
    if (out_type_ == SESSD_HALF) launch_linear8<__half>(a, stream);
    else launch_linear8<float>(a, stream);
    SESSD_HIP_TRY(hipGetLastError());
    return SESSD_OK;
}

}  // namespace sessd

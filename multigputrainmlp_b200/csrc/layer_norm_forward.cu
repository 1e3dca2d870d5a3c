// Layer normalisation, forward: y = gamma * (x - mean) * rstd + beta over the columns of every row.
#include "layer_norm.cuh"

namespace mgt {
namespace ln {
namespace {

// Mean and spread of a row that lies in registers, in two reductions: the sum, then the sums of d = x - m and of d * d. The second sum
// of d corrects the rounding of the first mean (a row of large, nearly equal values), so that x - mean = d - shift is exact to an ulp.
struct Moments {
    float mean, shift, rstd;
};
__device__ __forceinline__ Moments Finish(float first, float2 sums, float cols, float eps) {
    const float shift = sums.x / cols;
    const float var = sums.y / cols - shift * shift;
    return {first + shift, shift, 1.0f / sqrtf((var < 0.0f ? 0.0f : var) + eps)};  // (a NaN stays one)
}

// kTower: x is a layer's output before its normalisation, the normalised row is added to the fp32 residual stream, and what a ReLU leaves
// goes to the stream and, as the next product's operand, to y.
template <class Tx, class Ty, int V, int NV, int kThreads, bool kTower>
__global__ void __launch_bounds__(kThreads)
ForwardKernel(const Forward a) {
    __shared__ float2 buffer[2 * (kThreads / 32)];
    Group g = MakeGroup(a.lanes, buffer);
    const uint32_t stride = gridDim.x * g.count;
    const float cols = static_cast<float>(a.cols);
    dependent_begin();
    float gamma[NV][V], beta[NV][V];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = PackColumn<V>(g, i);
#pragma unroll
        for (int j = 0; j < V; ++j) {
            gamma[i][j] = c + j < a.cols ? (a.gamma != nullptr ? a.gamma[c + j] : 1.0f) : 0.0f;
            beta[i][j] = c + j < a.cols && a.beta != nullptr ? a.beta[c + j] : 0.0f;
        }
    }
    const Tx* x = static_cast<const Tx*>(a.x);
    Ty* y = static_cast<Ty*>(a.y);
    Pack<Tx, V> next[NV];
    auto load = [&](uint64_t row) {
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i);
            LoadPack<Tx, V>(next[i], x + row * a.x_pitch + c, row < a.rows ? PackValid(c, a.cols) : 0U);
        }
    };
    uint64_t row = static_cast<uint64_t>(blockIdx.x) * g.count + g.index;
    const uint64_t warp_first = g.lanes < 32U ? row - (g.index & (32U / g.lanes - 1U)) : row;  // the loop's bound is a warp's
    const uint64_t ahead = row - warp_first;
    load(row);
    for (uint64_t first = warp_first; first < a.rows; first += stride) {
        row = first + ahead;
        float v[NV][V];
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = ToFloat(next[i].v[j]);  // (zero beyond the row's end)
                sum += v[i][j];
            }
        load(row + stride);  // the next row is on its way while this one is reduced
        const float m = Reduce(g, sum, 0.0f).x / cols;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                v[i][j] = c + j < a.cols ? v[i][j] - m : 0.0f;
                s1 += v[i][j];
                s2 += v[i][j] * v[i][j];
            }
        }
        const Moments mo = Finish(m, Reduce(g, s1, s2), cols, a.eps);
        if (row >= a.rows) continue;
        if (g.lane == 0U) {
            if (a.mean != nullptr) a.mean[row] = mo.mean;
            if (a.rstd != nullptr) a.rstd[row] = mo.rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i), valid = PackValid(c, a.cols);
            float out[V];
#pragma unroll
            for (int j = 0; j < V; ++j) out[j] = (v[i][j] - mo.shift) * mo.rstd * gamma[i][j] + beta[i][j];
            if (kTower) {
                float* state = a.state + row * a.x_pitch + c;
                Pack<float, V> old;
                LoadPack<float, V>(old, state, a.add ? valid : 0U);
#pragma unroll
                for (int j = 0; j < V; ++j) out[j] = fmaxf(old.v[j] + out[j], 0.0f);
                StorePack<float, V>(state, out, valid);
            }
            StorePack<Ty, V>(y + row * a.y_pitch + c, out, valid);
        }
    }
}

// Rows wider than the registers of a CTA: a CTA a row, which it reads three times (from its L1 and L2 after the first).
template <class Tx, class Ty, int V>
__global__ void __launch_bounds__(1024)
StreamForwardKernel(const Forward a) {
    __shared__ float2 buffer[2 * 32];
    Group g = MakeGroup(blockDim.x, buffer);
    const float cols = static_cast<float>(a.cols);
    const uint32_t step = blockDim.x * V;
    dependent_begin();
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_pitch;
        Ty* y = static_cast<Ty*>(a.y) + row * a.y_pitch;
        float sum = 0.0f;
#pragma unroll 4
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            Pack<Tx, V> p;
            LoadPack<Tx, V>(p, x + c, a.cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) sum += ToFloat(p.v[j]);
        }
        const float m = Reduce(g, sum, 0.0f).x / cols;
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 4
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            Pack<Tx, V> p;
            LoadPack<Tx, V>(p, x + c, a.cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = c + j < a.cols ? ToFloat(p.v[j]) - m : 0.0f;
                s1 += d;
                s2 += d * d;
            }
        }
        const Moments mo = Finish(m, Reduce(g, s1, s2), cols, a.eps);
        if (threadIdx.x == 0U) {
            if (a.mean != nullptr) a.mean[row] = mo.mean;
            if (a.rstd != nullptr) a.rstd[row] = mo.rstd;
        }
#pragma unroll 2
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            Pack<Tx, V> p;
            LoadPack<Tx, V>(p, x + c, a.cols - c);
            float out[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const uint32_t k = min(c + j, a.cols - 1U);
                out[j] = ((ToFloat(p.v[j]) - m) - mo.shift) * mo.rstd * (a.gamma != nullptr ? a.gamma[k] : 1.0f) + (a.beta != nullptr ? a.beta[k] : 0.0f);
            }
            StorePack<Ty, V>(y + c, out, a.cols - c);
        }
    }
}

constexpr uint32_t kCtasPerSm = 3;

template <class Tx, class Ty, int V, int NV, int kThreads, bool kTower>
void Run(Forward a, const Cut& cut, LaunchOn on) {
    const uint32_t rows = cut.threads / cut.lanes;
    const uint64_t want = (static_cast<uint64_t>(a.rows) + rows - 1U) / rows;
    a.lanes = cut.lanes;
    Launch(ForwardKernel<Tx, Ty, V, NV, kThreads, kTower>, static_cast<uint32_t>(want < 148U * kCtasPerSm ? want : 148U * kCtasPerSm), cut.threads, 0, on, a);
}
template <class Tx, class Ty, int V>
void RunByWidth(const Forward& a, LaunchOn on) {
    const Cut cut = CutRow(a.cols, V, 16);
    if (cut.stream) {
        Launch(StreamForwardKernel<Tx, Ty, V>, a.rows < 296U ? a.rows : 296U, 1024, 0, on, a);
        return;
    }
    constexpr int kMost = 16 / V, kFew = V == 1 ? 4 : 2;  // packs a thread that there are kernels for, besides one
    if (cut.threads > 256U) Run<Tx, Ty, V, kMost, 512, false>(a, cut, on);
    else if (cut.nv == 1) Run<Tx, Ty, V, 1, 256, false>(a, cut, on);
    else if (cut.nv <= kFew) Run<Tx, Ty, V, kFew, 256, false>(a, cut, on);
    else Run<Tx, Ty, V, kMost, 256, false>(a, cut, on);
}
template <class Tx, class Ty>
void RunTyped(const Forward& a, int32_t x_type, int32_t y_type, LaunchOn on) {
    constexpr int kV = sizeof(Tx) == 2 && sizeof(Ty) == 2 ? 8 : 4;
    if (RowsAligned(a.x, a.x_pitch, a.rows, x_type, kV) && RowsAligned(a.y, a.y_pitch, a.rows, y_type, kV)) RunByWidth<Tx, Ty, kV>(a, on);
    else RunByWidth<Tx, Ty, 1>(a, on);
}

}  // namespace

mgt_status_t LaunchForward(Forward a, int32_t x_type, int32_t y_type, LaunchOn on) {
    if (x_type == MGT_F32 && y_type == MGT_F32) RunTyped<float, float>(a, x_type, y_type, on);
    else if (x_type == MGT_F32 && y_type == MGT_F16) RunTyped<float, __half>(a, x_type, y_type, on);
    else if (x_type == MGT_F32 && y_type == MGT_BF16) RunTyped<float, __nv_bfloat16>(a, x_type, y_type, on);
    else if (x_type == MGT_F16 && y_type == MGT_F16) RunTyped<__half, __half>(a, x_type, y_type, on);
    else if (x_type == MGT_F16 && y_type == MGT_F32) RunTyped<__half, float>(a, x_type, y_type, on);
    else if (x_type == MGT_BF16 && y_type == MGT_BF16) RunTyped<__nv_bfloat16, __nv_bfloat16>(a, x_type, y_type, on);
    else if (x_type == MGT_BF16 && y_type == MGT_F32) RunTyped<__nv_bfloat16, float>(a, x_type, y_type, on);
    else return MGT_INVALID_CONFIG;
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}

mgt_status_t LaunchTowerForward(Forward a, bool bf16, LaunchOn on) {
    const Cut cut = CutRow(a.cols, 4, 16);  // widths of a tower: a warp a row at most
    if (cut.lanes > 32U || cut.stream) return MGT_INVALID_CONFIG;
    auto run = [&](auto type) {
        using T = decltype(type);
        if (cut.nv == 1) Run<float, T, 4, 1, 256, true>(a, cut, on);
        else if (cut.nv == 2) Run<float, T, 4, 2, 256, true>(a, cut, on);
        else Run<float, T, 4, 4, 256, true>(a, cut, on);
    };
    if (bf16) run(__nv_bfloat16{}); else run(__half{});
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}

}  // namespace ln
}  // namespace mgt

extern "C" {

mgt_status_t mgt_validate_layer_norm_config(const mgt_layer_norm_config_t* c) {
    if (c == nullptr || c->cols == 0 || c->cols > MGT_LAYER_NORM_MAX_COLS || !(c->eps > 0.0f) || !(c->eps <= 3.0e38f)) return MGT_INVALID_CONFIG;
    auto known = [](int32_t t) { return t == MGT_F32 || t == MGT_F16 || t == MGT_BF16; };
    if (!known(c->x_type) || !known(c->y_type) || !known(c->dx_type)) return MGT_INVALID_CONFIG;
    if (c->x_type != MGT_F32 && c->y_type != MGT_F32 && c->y_type != c->x_type) return MGT_INVALID_CONFIG;
    if (c->dx_type != c->x_type && !(c->x_type == MGT_F32 && c->y_type == MGT_F32)) return MGT_INVALID_CONFIG;
    if ((c->x_pitch != 0 && c->x_pitch < c->cols) || (c->y_pitch != 0 && c->y_pitch < c->cols) || (c->dx_pitch != 0 && c->dx_pitch < c->cols)) return MGT_INVALID_CONFIG;
    return MGT_OK;
}

mgt_status_t mgt_launch_layer_norm(const mgt_layer_norm_config_t* c, const void* x, const float* gamma, const float* beta, void* y, float* mean, float* rstd,
                                   void* stream) {
    if (mgt_validate_layer_norm_config(c) != MGT_OK) return MGT_INVALID_CONFIG;
    if (c->rows == 0) return MGT_OK;
    auto aligned = [](const void* p, uint32_t bytes) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (bytes - 1U)) == 0; };
    if (!aligned(x, mgt::ln::TypeBytes(c->x_type)) || !aligned(y, mgt::ln::TypeBytes(c->y_type))) return MGT_INVALID_CONFIG;
    for (const float* p : {gamma, beta, static_cast<const float*>(mean), static_cast<const float*>(rstd)})
        if (p != nullptr && !aligned(p, 4)) return MGT_INVALID_CONFIG;
    mgt::ln::Forward a{};
    a.x = x; a.y = y; a.gamma = gamma; a.beta = beta; a.mean = mean; a.rstd = rstd;
    a.x_pitch = c->x_pitch != 0 ? c->x_pitch : c->cols;
    a.y_pitch = c->y_pitch != 0 ? c->y_pitch : c->cols;
    a.rows = c->rows; a.cols = c->cols; a.eps = c->eps;
    return mgt::ln::LaunchForward(a, c->x_type, c->y_type, {static_cast<cudaStream_t>(stream), true});
}

}  // extern "C"

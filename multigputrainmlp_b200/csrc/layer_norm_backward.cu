// Layer normalisation, backward. With xhat = (x - mean) * rstd and g = dy * gamma:
//   dx = rstd * (g - mean_c(g) - xhat * mean_c(g * xhat)),  dgamma = sum_r dy * xhat,  dbeta = sum_r dy,  dbias = sum_r dx
// One pass over dy and x: a thread keeps the columns that it owns for all rows of its CTA, so the column sums stay in its registers and
// leave once a CTA, as a row of partial sums that a second, small kernel adds up in a fixed order.
#include "layer_norm.cuh"

namespace mgt {
namespace ln {
namespace {

constexpr uint32_t kSums = 3;
constexpr uint32_t kMostCtas = 296;     // partial rows at most: two CTAs on each of 148 SMs
constexpr uint32_t kColumnSlices = 37;  // widest rows: slices of the batch that the column sums are taken over

template <class Tdy, class Tx, class Tdx, int V, int NV, int kThreads>
__global__ void __launch_bounds__(kThreads)
BackwardKernel(const Backward a) {
    extern __shared__ float lanes_sums[];  // [groups][cols], more than one group
    __shared__ float2 buffer[2 * (kThreads / 32)];
    Group g = MakeGroup(a.lanes, buffer);
    const uint32_t stride = gridDim.x * g.count;
    const float cols = static_cast<float>(a.cols);
    dependent_begin();
    float gamma[NV][V], sums[kSums][NV][V] = {};
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = PackColumn<V>(g, i);
#pragma unroll
        for (int j = 0; j < V; ++j) gamma[i][j] = c + j < a.cols ? (a.gamma != nullptr ? a.gamma[c + j] : 1.0f) : 0.0f;
    }
    const Tdy* dy = static_cast<const Tdy*>(a.dy);
    const Tx* x = static_cast<const Tx*>(a.x);
    Tdx* dx = static_cast<Tdx*>(a.dx);
    Pack<Tdy, V> next_dy[NV];
    Pack<Tx, V> next_x[NV];
    float next_mean = 0.0f, next_rstd = 0.0f;
    auto load = [&](uint64_t row) {
        const bool in = row < a.rows;
        if (in) {
            next_mean = a.mean[row];
            next_rstd = a.rstd[row];
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i), valid = in ? PackValid(c, a.cols) : 0U;
            LoadPack<Tdy, V>(next_dy[i], dy + row * a.dy_pitch + c, valid);
            LoadPack<Tx, V>(next_x[i], x + row * a.x_pitch + c, valid);
        }
    };
    uint64_t row = static_cast<uint64_t>(blockIdx.x) * g.count + g.index;
    const uint64_t warp_first = g.lanes < 32U ? row - (g.index & (32U / g.lanes - 1U)) : row;  // the loop's bound is a warp's
    const uint64_t ahead = row - warp_first;
    load(row);
    for (uint64_t first = warp_first; first < a.rows; first += stride) {
        row = first + ahead;
        const float mean = next_mean, rstd = next_rstd;
        float xhat[NV][V], d[NV][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                d[i][j] = ToFloat(next_dy[i].v[j]);
                xhat[i][j] = c + j < a.cols ? (ToFloat(next_x[i].v[j]) - mean) * rstd : 0.0f;
                const float t = d[i][j] * gamma[i][j];
                s1 += t;
                s2 += t * xhat[i][j];
            }
        }
        load(row + stride);  // the next row is on its way while this one is reduced
        const float2 total = Reduce(g, s1, s2);
        if (row >= a.rows) continue;
        const float c1 = total.x / cols, c2 = total.y / cols;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i), valid = PackValid(c, a.cols);
            float out[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                out[j] = rstd * (d[i][j] * gamma[i][j] - c1 - xhat[i][j] * c2);
                sums[0][i][j] += d[i][j] * xhat[i][j];
                sums[1][i][j] += d[i][j];
                sums[2][i][j] += out[j];  // (before it is rounded to dx's type)
            }
            StorePack<Tdx, V>(dx + row * a.dx_pitch + c, out, valid);
        }
    }
    // this CTA's column sums: the groups in order
    float* partial = a.partial + static_cast<uint64_t>(blockIdx.x) * kSums * a.cols;
#pragma unroll
    for (uint32_t k = 0; k < kSums; ++k) {
        if (a.sums[k] == nullptr) continue;
        float* to = gridDim.x > 1U ? partial + k * a.cols : a.sums[k];
        float* mine = g.count > 1U ? lanes_sums + g.index * a.cols : to;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const uint32_t c = PackColumn<V>(g, i);
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < a.cols) mine[c + j] = sums[k][i][j];
        }
        if (g.count > 1U) {
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
                float s = 0.0f;
                for (uint32_t l = 0; l < g.count; ++l) s += lanes_sums[l * a.cols + c];
                to[c] = s;
            }
            __syncthreads();
        }
    }
}

// sums[k][c] = the partial rows' values added up: 64 threads share a column, each adds every 64th row in order, then a binary tree.
constexpr uint32_t kSumCols = 16, kSumParts = 64;
__global__ void __launch_bounds__(kSumCols * kSumParts)
SumPartialRowsKernel(const Backward a, uint32_t rows) {
    __shared__ float part_sums[kSumParts][kSumCols];
    const uint32_t c = threadIdx.x % kSumCols, part = threadIdx.x / kSumCols, col = blockIdx.x * kSumCols + c;
    dependent_begin();
    float* to = a.sums[blockIdx.y];
    if (to == nullptr) return;
    float s = 0.0f;
    if (col < a.cols) {
        const float* from = a.partial + static_cast<uint64_t>(blockIdx.y) * a.cols + col;
#pragma unroll 5
        for (uint32_t r = part; r < rows; r += kSumParts) s += from[static_cast<uint64_t>(r) * kSums * a.cols];
    }
    part_sums[part][c] = s;
    __syncthreads();
#pragma unroll
    for (uint32_t half = kSumParts / 2U; half > 0U; half >>= 1) {
        if (part < half) part_sums[part][c] += part_sums[part + half][c];
        __syncthreads();
    }
    if (part == 0U && col < a.cols) to[col] = part_sums[0][c];
}

// Rows wider than the registers of a CTA. First the two means of every row, left in `means` ...
template <class Tdy, class Tx, int V>
__global__ void __launch_bounds__(1024)
StreamMeansKernel(const Backward a, float2* means) {
    __shared__ float2 buffer[2 * 32];
    Group g = MakeGroup(blockDim.x, buffer);
    const float cols = static_cast<float>(a.cols);
    const uint32_t step = blockDim.x * V;
    dependent_begin();
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Tdy* dy = static_cast<const Tdy*>(a.dy) + row * a.dy_pitch;
        const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_pitch;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s1 = 0.0f, s2 = 0.0f;
#pragma unroll 2
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            Pack<Tdy, V> pd;
            Pack<Tx, V> px;
            LoadPack<Tdy, V>(pd, dy + c, a.cols - c);
            LoadPack<Tx, V>(px, x + c, a.cols - c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float t = c + j < a.cols ? ToFloat(pd.v[j]) * (a.gamma != nullptr ? a.gamma[c + j] : 1.0f) : 0.0f;
                s1 += t;
                s2 += t * ((ToFloat(px.v[j]) - mean) * rstd);
            }
        }
        const float2 total = Reduce(g, s1, s2);
        if (threadIdx.x == 0U) means[row] = make_float2(total.x / cols, total.y / cols);
    }
}
// ... then, a tile of columns and a slice of the rows at a time, dx and the column sums.
template <class Tdy, class Tx, class Tdx, int V>
__global__ void __launch_bounds__(256)
StreamColumnsKernel(const Backward a, const float2* means, uint32_t rows_each) {
    const uint32_t c = (blockIdx.x * 256U + threadIdx.x) * V;
    dependent_begin();
    if (c >= a.cols) return;
    const uint32_t valid = a.cols - c;
    const uint64_t r0 = static_cast<uint64_t>(blockIdx.y) * rows_each, r1 = min(static_cast<uint64_t>(a.rows), r0 + rows_each);
    float gamma[V], sums[kSums][V] = {};
#pragma unroll
    for (int j = 0; j < V; ++j) gamma[j] = j < valid ? (a.gamma != nullptr ? a.gamma[c + j] : 1.0f) : 0.0f;
#pragma unroll 4
    for (uint64_t row = r0; row < r1; ++row) {
        Pack<Tdy, V> pd;
        Pack<Tx, V> px;
        LoadPack<Tdy, V>(pd, static_cast<const Tdy*>(a.dy) + row * a.dy_pitch + c, valid);
        LoadPack<Tx, V>(px, static_cast<const Tx*>(a.x) + row * a.x_pitch + c, valid);
        const float mean = a.mean[row], rstd = a.rstd[row];
        const float2 m = means[row];
        float out[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const float d = ToFloat(pd.v[j]), xhat = (ToFloat(px.v[j]) - mean) * rstd;
            out[j] = rstd * (d * gamma[j] - m.x - xhat * m.y);
            sums[0][j] += d * xhat;
            sums[1][j] += d;
            sums[2][j] += out[j];
        }
        StorePack<Tdx, V>(static_cast<Tdx*>(a.dx) + row * a.dx_pitch + c, out, valid);
    }
    float* partial = a.partial + static_cast<uint64_t>(blockIdx.y) * kSums * a.cols;
#pragma unroll
    for (uint32_t k = 0; k < kSums; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j)
            if (j < valid) partial[k * a.cols + c + j] = sums[k][j];
}

void SumPartialRows(const Backward& a, uint32_t rows, LaunchOn on, uint32_t* launches) {
    Launch(SumPartialRowsKernel, dim3((a.cols + kSumCols - 1U) / kSumCols, kSums), kSumCols * kSumParts, 0, LaunchOn(on.stream, true), a, rows);
    ++*launches;
}

// Elements that a thread holds of a row: with an fp32 operand 8, else 16. Beside them are the next row's, gamma and three sums a column.
template <class Tdy, class Tx>
constexpr int kElements = sizeof(Tdy) == 4 || sizeof(Tx) == 4 ? 8 : 16;

template <class Tdy, class Tx, class Tdx, int V, int NV, int kThreads>
void Run(Backward a, const Cut& cut, LaunchOn on, uint32_t* launches) {
    const uint32_t groups = cut.threads / cut.lanes;
    const uint64_t want = (static_cast<uint64_t>(a.rows) + groups - 1U) / groups;
    const uint32_t ctas = static_cast<uint32_t>(want < kMostCtas ? want : kMostCtas);
    a.lanes = cut.lanes;
    const size_t smem = groups > 1U ? static_cast<size_t>(groups) * a.cols * sizeof(float) : 0;
    Launch(BackwardKernel<Tdy, Tx, Tdx, V, NV, kThreads>, ctas, cut.threads, smem, on, a);
    ++*launches;
    if (ctas > 1U && (a.sums[0] != nullptr || a.sums[1] != nullptr || a.sums[2] != nullptr)) SumPartialRows(a, ctas, on, launches);
}
template <class Tdy, class Tx, class Tdx, int V>
void RunByWidth(const Backward& a, LaunchOn on, uint32_t* launches) {
    constexpr int kE = kElements<Tdy, Tx>;
    const Cut cut = CutRow(a.cols, V, kE);
    if (cut.stream) {
        float2* means = reinterpret_cast<float2*>(a.partial + static_cast<uint64_t>(kMostCtas) * kSums * a.cols);
        Launch(StreamMeansKernel<Tdy, Tx, V>, a.rows < 296U ? a.rows : 296U, 1024, 0, on, a, means);
        const uint32_t slices = a.rows < kColumnSlices ? a.rows : kColumnSlices, rows_each = (a.rows - 1U) / slices + 1U;
        const uint32_t used = (a.rows - 1U) / rows_each + 1U;
        Launch(StreamColumnsKernel<Tdy, Tx, Tdx, V>, dim3((a.cols - 1U) / (256U * V) + 1U, used), 256, 0, LaunchOn(on.stream, true), a, static_cast<const float2*>(means), rows_each);
        *launches += 2;
        SumPartialRows(a, used, on, launches);
        return;
    }
    constexpr int kMost = kE / V, kFew = V == 1 ? 4 : 2;
    if (cut.threads > 256U) Run<Tdy, Tx, Tdx, V, kMost, 512>(a, cut, on, launches);
    else if (cut.nv == 1) Run<Tdy, Tx, Tdx, V, 1, 256>(a, cut, on, launches);
    else if (cut.nv <= kFew) Run<Tdy, Tx, Tdx, V, kFew, 256>(a, cut, on, launches);
    else Run<Tdy, Tx, Tdx, V, kMost, 256>(a, cut, on, launches);
}
template <class Tdy, class Tx, class Tdx>
void RunTyped(const Backward& a, int32_t dy_type, int32_t x_type, int32_t dx_type, LaunchOn on, uint32_t* launches) {
    constexpr int kV = sizeof(Tdy) == 2 && sizeof(Tx) == 2 && sizeof(Tdx) == 2 ? 8 : 4;
    if (RowsAligned(a.dy, a.dy_pitch, a.rows, dy_type, kV) && RowsAligned(a.x, a.x_pitch, a.rows, x_type, kV) && RowsAligned(a.dx, a.dx_pitch, a.rows, dx_type, kV))
        RunByWidth<Tdy, Tx, Tdx, kV>(a, on, launches);
    else RunByWidth<Tdy, Tx, Tdx, 1>(a, on, launches);
}

}  // namespace

uint64_t BackwardFloats(uint32_t rows, uint32_t cols) {
    return static_cast<uint64_t>(kMostCtas) * kSums * cols + (cols > 8U * kMostLanes ? 2ULL * rows : 0ULL) + 2ULL;
}

mgt_status_t LaunchBackward(Backward a, int32_t dy_type, int32_t x_type, int32_t dx_type, LaunchOn on, uint32_t* launches) {
    auto is = [&](int32_t dy, int32_t x, int32_t dx) { return dy_type == dy && x_type == x && dx_type == dx; };
    using H = __half;
    using B = __nv_bfloat16;
    if (is(MGT_F32, MGT_F32, MGT_F32)) RunTyped<float, float, float>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_F32, MGT_F32, MGT_F16)) RunTyped<float, float, H>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_F32, MGT_F32, MGT_BF16)) RunTyped<float, float, B>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_F16, MGT_F32, MGT_F32)) RunTyped<H, float, float>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_BF16, MGT_F32, MGT_F32)) RunTyped<B, float, float>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_F16, MGT_F16, MGT_F16)) RunTyped<H, H, H>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_F32, MGT_F16, MGT_F16)) RunTyped<float, H, H>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_BF16, MGT_BF16, MGT_BF16)) RunTyped<B, B, B>(a, dy_type, x_type, dx_type, on, launches);
    else if (is(MGT_F32, MGT_BF16, MGT_BF16)) RunTyped<float, B, B>(a, dy_type, x_type, dx_type, on, launches);
    else return MGT_INVALID_CONFIG;
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}

}  // namespace ln
}  // namespace mgt

extern "C" {

uint64_t mgt_layer_norm_backward_workspace_floats(const mgt_layer_norm_config_t* c) {
    return mgt_validate_layer_norm_config(c) == MGT_OK ? mgt::ln::BackwardFloats(c->rows, c->cols) : 0;
}

mgt_status_t mgt_launch_layer_norm_backward(const mgt_layer_norm_config_t* c, const void* dy, const void* x, const float* gamma, const float* mean, const float* rstd,
                                            void* dx, float* dgamma, float* dbeta, float* dbias, float* workspace, uint64_t workspace_floats, void* stream) {
    if (mgt_validate_layer_norm_config(c) != MGT_OK) return MGT_INVALID_CONFIG;
    auto aligned = [](const void* p, uint32_t bytes) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (bytes - 1U)) == 0; };
    float* sums[3] = {dgamma, dbeta, dbias};
    for (const float* p : {gamma, static_cast<const float*>(dgamma), static_cast<const float*>(dbeta), static_cast<const float*>(dbias)})
        if (p != nullptr && !aligned(p, 4)) return MGT_INVALID_CONFIG;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (c->rows == 0) {  // no rows: the sums over them are zero
        for (float* p : sums)
            if (p != nullptr && cudaMemsetAsync(p, 0, static_cast<size_t>(c->cols) * sizeof(float), s) != cudaSuccess) return MGT_CUDA_FAILURE;
        return MGT_OK;
    }
    if (!aligned(dy, mgt::ln::TypeBytes(c->y_type)) || !aligned(x, mgt::ln::TypeBytes(c->x_type)) || !aligned(dx, mgt::ln::TypeBytes(c->dx_type)) ||
        !aligned(mean, 4) || !aligned(rstd, 4) || !aligned(workspace, 8)) return MGT_INVALID_CONFIG;
    if (workspace_floats < mgt::ln::BackwardFloats(c->rows, c->cols)) return MGT_CAPACITY_EXCEEDED;
    mgt::ln::Backward a{};
    a.dy = dy; a.x = x; a.dx = dx; a.gamma = gamma; a.mean = mean; a.rstd = rstd;
    for (int k = 0; k < 3; ++k) a.sums[k] = sums[k];
    a.partial = workspace;
    a.dy_pitch = c->y_pitch != 0 ? c->y_pitch : c->cols;
    a.x_pitch = c->x_pitch != 0 ? c->x_pitch : c->cols;
    a.dx_pitch = c->dx_pitch != 0 ? c->dx_pitch : c->cols;
    a.rows = c->rows; a.cols = c->cols;
    uint32_t launches = 0;
    return mgt::ln::LaunchBackward(a, c->y_type, c->x_type, c->dx_type, {s, true}, &launches);
}

}  // extern "C"

// Layer normalisation, forward: y = gamma * (x - mean) * rstd + beta over the columns of every row.
#include "layer_norm.cuh"

namespace mgt {
namespace ln {
namespace {

// Mean and spread of a row that lies in registers, in two reductions: the sum, then the sums of d = x - m and of d * d. The second sum
// of d corrects the rounding of the first mean (a row of large, nearly equal values), so that x - mean = d - shift is exact to an ulp.
// The mean that a caller gets takes the correction only where it is larger than the spread. Below, what corrects is worse than what it
// corrects: x - m drops the same bits of m for all x of one binade, an error of up to 2^-25 of the spread that no averaging makes smaller,
// where the first sum is off by its own rounding alone (16-bit rows are often added up exactly): 1 346 rows of 5 304 fp16 values were off by
// 6.5e-6 of their means with the correction, and without it the means of none of 600 shapes are off by more than 2e-7.
struct Moments {
    float mean, shift, rstd;
};
// Squares of deviations of 1e18 are 1e36, and 340 of them more than a float holds. A thread has few enough of them (32); what it adds to
// the row's sum is divided by 2^12, so that those of 2^20 columns are a sum that a float holds (a product by a power of two, which rounds nothing).
// (131 072 x 512 bf16 47.2 -> 47.9 us, 53 248 x 224 to 16 bits 13.0 -> 13.2, 16 384 x 4 096 54.6 -> 54.8; a second pass over the registers for
// rows that overflow, behind a branch, 49.3, 13.3, 55.6.)
constexpr float kSquares = 0x1p-12f;
__device__ __forceinline__ Moments Finish(float first, const float (&sums)[2], float per_col, float eps) {
    const float shift = sums[0] * per_col;
    const float var = sums[1] * per_col * (1.0f / kSquares) - shift * shift, v = (var < 0.0f ? 0.0f : var) + eps;  // (a NaN stays one)
    const float r = rsqrtf(v);
    return {first * first <= v ? first : first + shift, shift, r * fmaf(-0.5f * r, v * r, 1.5f)};  // one Newton step: to an ulp, at a tenth of a root's and a division's price
}

// Rows on their way: no more than it takes, since more are slower (us, with 3, 4 and 5 of 32 bytes a thread: 131 072 x 512 bf16 46.7, 47.2, 47.7; with 4,
// 6 and 8 of 16: 300 000 x 128 26.8, 27.4, 27.9).
template <class Tx, class Lay, int kThreads>
constexpr int kDepth = kThreads * Lay::E > 8192 ? (sizeof(Tx) == 2 ? 2 : 1) : Lay::V == 1 ? (sizeof(Tx) == 2 ? 4 : 3) : Lay::E > 16 ? 2 : Lay::E * sizeof(Tx) >= 32 ? 3 : 4;
template <class Tx, class Lay, int kThreads>
constexpr uint32_t kCtas = kThreads > 256 ? 1 : (Lay::V == 1 && Lay::E > 8) || Lay::E * sizeof(Tx) >= 128 ? 2 : 3;  // an SM (single columns take more registers, 32 fp32 values more shared memory)
// Whether scale and shift lie in shared memory, for want of registers: rows of more than a warp's 512 columns, of which a thread holds 32, so
// that fewer warps have to meet for a row.
template <class Lay, int kThreads>
constexpr bool kFarColumns = Lay::E > 16 || kThreads > 512;

// kTower: x is a layer's output before its normalisation, the normalised row is added to the fp32 residual stream, and what a ReLU leaves
// goes to the stream and, as the next product's operand, to y.
template <class Tx, class Ty, class Lay, int kThreads, bool kTower>
__global__ void __launch_bounds__(kThreads, kCtas<Tx, Lay, kThreads>)
ForwardKernel(const Forward a) {
    extern __shared__ __align__(16) char memory[];  // the ring, then gamma and beta where registers have no room for them
    __shared__ float buffer[2 * 2 * (kThreads / 32)];
    constexpr bool kFar = kFarColumns<Lay, kThreads>;
    constexpr int V = Lay::V, E = Lay::E, D = kDepth<Tx, Lay, kThreads>, kPairs = Held<E>::kPairs;
    Group g = MakeGroup(a.lanes, buffer);
    const Share share = MakeShare(g, a.rows, blockIdx.x, gridDim.x);
    const Lay lay(g, a.cols);
    Ring<Tx, Lay, kThreads, D> ring(static_cast<const Tx*>(a.x), a.x_pitch, a.rows, memory, share, lay);
    const float per_col = 1.0f / static_cast<float>(a.cols);
    Ty* y = static_cast<Ty*>(a.y) + share.first * a.y_pitch + lay.base;
    float* state = kTower ? a.state + share.first * a.x_pitch + lay.base : nullptr;
    const uint64_t y_step = share.stride * a.y_pitch, state_step = share.stride * a.x_pitch;
    ring.Clear(lay);
    dependent_begin();
#pragma unroll
    for (int d = 0; d < D; ++d) {
        ring.Fetch(lay, d, d < share.mine);
        CopiesEnd();
    }
    Held<E> gamma, beta, v;
    float4* far = reinterpret_cast<float4*>(memory + Ring<Tx, Lay, kThreads, D>::kBytes) + g.lane;  // {two of gamma, two of beta} of a lane, for all groups
    if constexpr (kFar) {
        LoadColumns(gamma, lay, a.gamma, 1.0f);
        LoadColumns(beta, lay, a.beta, 0.0f);
#pragma unroll
        for (int k = 0; k < kPairs; ++k)
            if (g.index == 0U) far[k * g.lanes] = make_float4(gamma.pair[k].x, gamma.pair[k].y, beta.pair[k].x, beta.pair[k].y);
        __syncthreads();
    } else {
        LoadColumns(gamma, lay, a.gamma, 1.0f);
        LoadColumns(beta, lay, a.beta, 0.0f);
    }
    uint32_t slot = 0, row = share.first;
    for (uint32_t t = 0; t < share.turns; ++t) {
        const bool in = t < share.mine;
        CopiesWait<D - 1>();
        if (V == 1) __syncwarp();  // (what the other lanes copied is here, too)
        ring.Read(v, lay, slot, in);
        float sum[1] = {SumOf(v)};
        Reduce(g, sum);
        if (V == 1) __syncwarp();  // (everybody has what it read of the slot: the sum needed it)
        ring.Fetch(lay, slot, t + D < share.mine);
        CopiesEnd();
        slot = slot + 1U == D ? 0U : slot + 1U;
        const float first = sum[0] * per_col;
        if constexpr (V > 1) {
            lay.Each([&](int i, bool has) {
                const float2 m = Both(has ? -first : 0.0f);
#pragma unroll
                for (int k = 0; k < V / 2; ++k) v.pair[i * (V / 2) + k] = Add2(v.pair[i * (V / 2) + k], m);
            });
        } else {
            lay.Each([&](int i, bool has) { v.Set(i, has ? v.Get(i) - first : 0.0f); });
        }
        float2 s1 = Both(0.0f), s2 = Both(0.0f);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
            s1 = Add2(s1, v.pair[k]);
            s2 = Fma2(v.pair[k], v.pair[k], s2);
        }
        float s[2] = {s1.x + s1.y, (s2.x + s2.y) * kSquares};
        Reduce(g, s);
        const Moments mo = Finish(first, s, per_col, a.eps);
        if (in) {
            if (g.lane == 0U) {
                if (a.mean != nullptr) a.mean[row] = mo.mean;
                if (a.rstd != nullptr) a.rstd[row] = mo.rstd;
            }
            const float2 rstd = Both(mo.rstd), off = Both(-mo.shift * mo.rstd);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const float4 q = kFar ? far[k * g.lanes] : make_float4(gamma.pair[k].x, gamma.pair[k].y, beta.pair[k].x, beta.pair[k].y);
                v.pair[k] = Fma2(Fma2(v.pair[k], rstd, off), make_float2(q.x, q.y), make_float2(q.z, q.w));
            }
            lay.Each([&](int i, bool has) {
                if (!has) return;
                const uint32_t at = lay.Offset(i);
                if (kTower) {
                    const Pack<float, V> old = a.add ? LoadPack<float, V>(state + at) : Pack<float, V>{};
#pragma unroll
                    for (int j = 0; j < V; ++j) v.Set(i * V + j, fmaxf(old.v[j] + v.Get(i * V + j), 0.0f));
                    StorePack<float, V>(state + at, PackOf<float, V>(v, i));
                }
                StorePack<Ty, V>(y + at, PackOf<Ty, V>(v, i));
            });
        }
        y += y_step;
        if (kTower) state += state_step;
        row += share.stride;
    }
}

// Rows wider than the registers of a CTA: a CTA a row, which it reads three times (from its L1 and L2 after the first), four packs at once
// (the compiler keeps a load behind the store before it: y may be x).
template <class Tx, class Ty, int V>
__global__ void __launch_bounds__(1024)
StreamForwardKernel(const Forward a) {
    __shared__ float buffer[2 * 2 * 32];
    Group g = MakeGroup(blockDim.x, buffer);
    const float per_col = 1.0f / static_cast<float>(a.cols);
    const uint32_t step = blockDim.x * V;
    dependent_begin();
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_pitch;
        Ty* y = static_cast<Ty*>(a.y) + row * a.y_pitch;
        float sum[1] = {0.0f};
#pragma unroll 4
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            const Pack<Tx, V> p = LoadPack<Tx, V>(x + c);
#pragma unroll
            for (int j = 0; j < V; ++j) sum[0] += ToFloat(p.v[j]);
        }
        Reduce(g, sum);
        const float m = sum[0] * per_col;
        float s[2] = {0.0f, 0.0f};
#pragma unroll 4
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            const Pack<Tx, V> p = LoadPack<Tx, V>(x + c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = ToFloat(p.v[j]) - m;
                s[0] += d;
                s[1] += d * kSquares * d;
            }
        }
        Reduce(g, s);
        const Moments mo = Finish(m, s, per_col, a.eps);
        if (threadIdx.x == 0U) {
            if (a.mean != nullptr) a.mean[row] = mo.mean;
            if (a.rstd != nullptr) a.rstd[row] = mo.rstd;
        }
        for (uint32_t c0 = threadIdx.x * V; c0 < a.cols; c0 += 4U * step) {
            Pack<Tx, V> p[4];
#pragma unroll
            for (uint32_t i = 0; i < 4U; ++i)
                if (c0 + i * step < a.cols) p[i] = LoadPack<Tx, V>(x + c0 + i * step);
#pragma unroll
            for (uint32_t i = 0; i < 4U; ++i) {
                const uint32_t c = c0 + i * step;
                if (c >= a.cols) continue;
                Pack<Ty, V> out;
#pragma unroll
                for (int j = 0; j < V; ++j)
                    out.v[j] = FromFloat<Ty>(((ToFloat(p[i].v[j]) - m) - mo.shift) * mo.rstd * (a.gamma != nullptr ? a.gamma[c + j] : 1.0f) + (a.beta != nullptr ? a.beta[c + j] : 0.0f));
                StorePack<Ty, V>(y + c, out);
            }
        }
    }
}


template <class Tx, class Ty, class Lay, int kThreads, bool kTower>
mgt_status_t Run(Forward a, const Cut& cut, LaunchOn on) {
    const uint32_t rows = cut.threads / cut.lanes;
    const uint64_t want = (static_cast<uint64_t>(a.rows) + rows - 1U) / rows;
    a.lanes = cut.lanes;
    static std::atomic<uint64_t> allowed{0};
    constexpr uint32_t ring = Ring<Tx, Lay, kThreads, kDepth<Tx, Lay, kThreads>>::kBytes, far = kFarColumns<Lay, kThreads> ? Lay::E * 8U : 0U;
    if (!AllowShared(ForwardKernel<Tx, Ty, Lay, kThreads, kTower>, allowed, ring + far * kThreads)) return MGT_CUDA_FAILURE;
    const uint32_t smem = ring + far * cut.lanes, most = 148U * kCtas<Tx, Lay, kThreads>;
    Launch(ForwardKernel<Tx, Ty, Lay, kThreads, kTower>, static_cast<uint32_t>(want < most ? want : most), cut.threads, smem, on, a);
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}
// (packs that a kernel has room for and the row does not have lie beyond its end)
template <class Tx, class Ty, int V, bool kTower>
mgt_status_t RunByWidth(const Forward& a, LaunchOn on) {
    // 32 elements a thread for 16-bit rows beyond a warp's 512 columns (us, with 16 and with 32: 40 000 x 600 bf16 39.8, 26.2; x 1 024 41.4, 29.4;
    // 16 384 x 4 096 67.6, 54.2), for fp32 ones where 512 threads of 16 are too few (20 000 x 1 024 28.4, 29.0; 7 000 x 8 192 79.5, 92.3)
    const bool wide = V > 1 && !kTower && a.cols > (sizeof(Tx) == 2 ? 32U : 512U) * kElements;
    const Cut cut = wide ? CutRow(a.rows, a.cols, V, 512, 2U * kElements) : CutRow(a.rows, a.cols, V, 1024);
    constexpr int kMost = kElements / V;
    // three packs a thread where a row then leaves fewer places empty (us, without and with: 131 072 x 304 bf16 46.7, 31.2; 50 000 x 768 32.3, 26.4;
    // 30 000 x 1 280 45.1, 37.6; packs of four columns, fp32 to fp16: 131 072 x 304 51.3, 41.6)
    if constexpr (V == 8) {
        const Cut three = CutRow(a.rows, a.cols, V, 512, 24);
        if (!three.stream && three.nv == 3 && three.lanes * 3U < cut.lanes * (cut.nv > 2 ? 4U : cut.nv)) {
            if (three.threads > 256U) return Run<Tx, Ty, Layout<V, 3, 32, 0>, 512, false>(a, three, on);
            return Run<Tx, Ty, Layout<V, 3, 32, 0>, 256, false>(a, three, on);
        }
    }
    if (cut.stream || (kTower && cut.threads > 256U)) {
        if constexpr (kTower) return MGT_INVALID_CONFIG;  // (no tower is that wide)
        Launch(StreamForwardKernel<Tx, Ty, V>, a.rows < 296U ? a.rows : 296U, 1024, 0, on, a);
        return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
    }
    if constexpr (V == 1 && !kTower) {
        using Less = Layout<1, 12, 32, 4>;  // (nine columns a thread at least; us, with 16 and with 12: 4 000 x 10 001 bf16 88.6, 81.7)
        using Most = Layout<1, 16, 32, 4>;
        if (cut.threads > 512U) return cut.nv <= 12U ? Run<Tx, Ty, Less, 1024, false>(a, cut, on) : Run<Tx, Ty, Most, 1024, false>(a, cut, on);
        if (cut.threads > 256U) return cut.nv <= 12U ? Run<Tx, Ty, Less, 512, false>(a, cut, on) : Run<Tx, Ty, Most, 512, false>(a, cut, on);
    }
    if constexpr (V > 1 && !kTower) {
        using Lay = Layout<V, 2 * kMost, 32, 0>;
        if constexpr (sizeof(Tx) == 4)
            if (cut.threads > 256U && !wide)
                return cut.nv == 3 ? Run<Tx, Ty, Layout<V, 3, 32, 0>, 512, false>(a, cut, on) : Run<Tx, Ty, Layout<V, kMost, 32, 0>, 512, false>(a, cut, on);
        if (cut.threads > 256U) return Run<Tx, Ty, Lay, 512, false>(a, cut, on);
        if constexpr (sizeof(Tx) == 2)
            if (cut.nv > kMost) return Run<Tx, Ty, Lay, 256, false>(a, cut, on);
    }
    if constexpr (V == 1) {
        return SingleColumns(cut, [&](auto tag) { return Run<Tx, Ty, typename decltype(tag)::type, 256, kTower>(a, cut, on); });
    } else {
        if (cut.nv == 1) return Run<Tx, Ty, Layout<V, 1, 32, 0>, 256, kTower>(a, cut, on);
        if (cut.nv == 2) return Run<Tx, Ty, Layout<V, 2, 32, 0>, 256, kTower>(a, cut, on);
        if constexpr (V == 4)
            if (cut.nv == 3) return Run<Tx, Ty, Layout<V, 3, 32, 0>, 256, kTower>(a, cut, on);
        return Run<Tx, Ty, Layout<V, kMost, 32, 0>, 256, kTower>(a, cut, on);
    }
}
template <class Tx, class Ty>
mgt_status_t RunTyped(const Forward& a, int32_t x_type, int32_t y_type, LaunchOn on) {
    auto whole = [&](int v) { return a.cols % v == 0 && RowsAligned(a.x, a.x_pitch, a.rows, x_type, v) && RowsAligned(a.y, a.y_pitch, a.rows, y_type, v); };
    if constexpr (sizeof(Tx) == 2 && sizeof(Ty) == 2)
        if (whole(8)) return RunByWidth<Tx, Ty, 8, false>(a, on);
    if (whole(4)) return RunByWidth<Tx, Ty, 4, false>(a, on);
    return RunByWidth<Tx, Ty, 1, false>(a, on);
}

}  // namespace

mgt_status_t LaunchForward(Forward a, int32_t x_type, int32_t y_type, LaunchOn on) {
    if (x_type == MGT_F32 && y_type == MGT_F32) return RunTyped<float, float>(a, x_type, y_type, on);
    if (x_type == MGT_F32 && y_type == MGT_F16) return RunTyped<float, __half>(a, x_type, y_type, on);
    if (x_type == MGT_F32 && y_type == MGT_BF16) return RunTyped<float, __nv_bfloat16>(a, x_type, y_type, on);
    if (x_type == MGT_F16 && y_type == MGT_F16) return RunTyped<__half, __half>(a, x_type, y_type, on);
    if (x_type == MGT_F16 && y_type == MGT_F32) return RunTyped<__half, float>(a, x_type, y_type, on);
    if (x_type == MGT_BF16 && y_type == MGT_BF16) return RunTyped<__nv_bfloat16, __nv_bfloat16>(a, x_type, y_type, on);
    if (x_type == MGT_BF16 && y_type == MGT_F32) return RunTyped<__nv_bfloat16, float>(a, x_type, y_type, on);
    return MGT_INVALID_CONFIG;
}

mgt_status_t LaunchTowerForward(Forward a, bool bf16, LaunchOn on) {
    const bool whole = a.cols % 4U == 0 && a.x_pitch % 4U == 0 && a.y_pitch % 4U == 0;
    if (bf16) return whole ? RunByWidth<float, __nv_bfloat16, 4, true>(a, on) : RunByWidth<float, __nv_bfloat16, 1, true>(a, on);
    return whole ? RunByWidth<float, __half, 4, true>(a, on) : RunByWidth<float, __half, 1, true>(a, on);
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

// The norm of a gradient over all tensors of a model, and clipping by it. Replaces nothing in the reference, which does not clip.
//
// Squares and sums are 64-bit: the square of any fp32 number is exact there up to its last bits and neither overflows nor vanishes, and
// adding millions of them loses nothing that a float could show. The tensors are cut into chunks of equal length; a CTA leaves the sum of a
// chunk in the workspace and one CTA of a second kernel adds the chunks of every tensor, then the tensors, all in an order that the sizes
// alone fix. The list of tensors travels in the launch's parameters: nothing is copied or allocated, and a captured launch keeps its own.
#include "../../include/mgt_b200.h"
#include "launch.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>

namespace {

constexpr uint32_t kThreads = 256, kFinishThreads = 1024;
constexpr uint32_t kUnroll = 4;  // 16-byte loads of a thread in flight
constexpr uint32_t kLeastChunkBytes = 16384;  // four such loads a thread: more chunks than the chip holds CTAs, so that none waits long for a last one
constexpr uint32_t kMostChunks = 4000;  // of whole length: longer chunks beyond, so that their sums fit into the shared memory of a CTA

// Tensors of a call as the kernels get them: where a tensor begins in the line of chunks, and its type in the top bits of its count.
template <uint32_t kMost>
struct Table {
    const void* data[kMost];
    uint64_t count[kMost];
    uint32_t first_chunk[kMost + 1];
    uint32_t tensors;
    uint64_t chunk;
};
template <uint32_t kMost>
struct Outputs {
    void* data[kMost];
};
constexpr uint32_t kTypeShift = 62;
constexpr uint64_t kCountMask = (1ULL << kTypeShift) - 1ULL;

template <class T> struct Vec;
template <> struct Vec<float> {
    static constexpr uint32_t kCount = 4;
    static __device__ float Get(const uint4& w, uint32_t i) { return __uint_as_float((&w.x)[i]); }
    static __device__ float One(float v) { return v; }
    static __device__ float To(float v) { return v; }
    static __device__ void Put(uint4& w, uint32_t i, float v) { (&w.x)[i] = __float_as_uint(v); }
};
template <> struct Vec<__half> {
    static constexpr uint32_t kCount = 8;
    static __device__ float Get(const uint4& w, uint32_t i) { return __half2float(reinterpret_cast<const __half*>(&w)[i]); }
    static __device__ float One(__half v) { return __half2float(v); }
    static __device__ __half To(float v) { return __float2half_rn(v); }
    static __device__ void Put(uint4& w, uint32_t i, float v) { reinterpret_cast<__half*>(&w)[i] = __float2half_rn(v); }
};
template <> struct Vec<__nv_bfloat16> {
    static constexpr uint32_t kCount = 8;
    static __device__ float Get(const uint4& w, uint32_t i) { return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(&w)[i]); }
    static __device__ float One(__nv_bfloat16 v) { return __bfloat162float(v); }
    static __device__ __nv_bfloat16 To(float v) { return __float2bfloat16_rn(v); }
    static __device__ void Put(uint4& w, uint32_t i, float v) { reinterpret_cast<__nv_bfloat16*>(&w)[i] = __float2bfloat16_rn(v); }
};

// Elements before the first 16-byte boundary, at most n.
template <class T>
__device__ __forceinline__ uint64_t HeadCount(const T* p, uint64_t n) {
    const uint64_t head = ((16U - (reinterpret_cast<uintptr_t>(p) & 15U)) & 15U) / sizeof(T);
    return head < n ? head : n;
}

template <class T>
__device__ double SumOfSquares(const T* p, uint64_t n) {
    const uint64_t head = HeadCount(p, n);
    double s[2] = {0.0, 0.0};  // (four would not leave room for eight CTAs an SM)
    auto add = [&](float f, uint32_t j) {
        const double d = static_cast<double>(f);
        s[j & 1U] = fma(d, d, s[j & 1U]);
    };
    if (threadIdx.x < head) add(Vec<T>::One(p[threadIdx.x]), 0);
    const uint4* body = reinterpret_cast<const uint4*>(p + head);
    const uint32_t vectors = static_cast<uint32_t>((n - head) / Vec<T>::kCount);
    for (uint32_t first = threadIdx.x; first < vectors; first += kUnroll * kThreads) {
        uint4 w[kUnroll];
#pragma unroll
        for (uint32_t k = 0; k < kUnroll; ++k) w[k] = first + k * kThreads < vectors ? body[first + k * kThreads] : make_uint4(0U, 0U, 0U, 0U);
#pragma unroll
        for (uint32_t k = 0; k < kUnroll; ++k)
#pragma unroll
            for (uint32_t j = 0; j < Vec<T>::kCount; ++j) add(Vec<T>::Get(w[k], j), j);
    }
    const uint64_t at = head + vectors * Vec<T>::kCount + threadIdx.x;
    if (at < n) add(Vec<T>::One(p[at]), 0);
    return s[0] + s[1];
}

template <class T>
__device__ void Scale(const T* p, T* out, uint64_t n, float scale, bool zero) {
    const uint64_t head = HeadCount(p, n);
    auto scaled = [&](float f) { return zero ? 0.0f : f * scale; };  // (a gradient that is not finite becomes zero, not NaN)
    if (HeadCount(out, n) != head) {  // the two lie differently to a 16-byte boundary
        for (uint64_t i = threadIdx.x; i < n; i += kThreads) out[i] = Vec<T>::To(scaled(Vec<T>::One(p[i])));
        return;
    }
    if (threadIdx.x < head) out[threadIdx.x] = Vec<T>::To(scaled(Vec<T>::One(p[threadIdx.x])));
    const uint4* body = reinterpret_cast<const uint4*>(p + head);
    uint4* to = reinterpret_cast<uint4*>(out + head);
    const uint32_t vectors = static_cast<uint32_t>((n - head) / Vec<T>::kCount);
    for (uint32_t first = threadIdx.x; first < vectors; first += kUnroll * kThreads) {
        uint4 w[kUnroll];
#pragma unroll
        for (uint32_t k = 0; k < kUnroll; ++k)
            if (first + k * kThreads < vectors) w[k] = body[first + k * kThreads];
#pragma unroll
        for (uint32_t k = 0; k < kUnroll; ++k) {
            if (first + k * kThreads >= vectors) continue;
#pragma unroll
            for (uint32_t j = 0; j < Vec<T>::kCount; ++j) Vec<T>::Put(w[k], j, scaled(Vec<T>::Get(w[k], j)));
            __stcs(to + first + k * kThreads, w[k]);
        }
    }
    const uint64_t at = head + vectors * Vec<T>::kCount + threadIdx.x;
    if (at < n) out[at] = Vec<T>::To(scaled(Vec<T>::One(p[at])));
}

// The tensor that a chunk belongs to: the last one that begins at or before it.
template <uint32_t kMost>
__device__ __forceinline__ uint32_t TensorOf(const Table<kMost>& t, uint32_t chunk) {
    uint32_t lo = 0, hi = t.tensors;
    while (hi - lo > 1U) {
        const uint32_t mid = (lo + hi) / 2U;
        if (t.first_chunk[mid] <= chunk) lo = mid; else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ double WarpSum(double s) {
#pragma unroll
    for (uint32_t o = 16; o > 0U; o >>= 1) s += __shfl_xor_sync(0xffffffffU, s, o);
    return s;
}

template <uint32_t kMost>
__global__ void __launch_bounds__(kThreads, 8)
ChunkSquaresKernel(const __grid_constant__ Table<kMost> t, double* __restrict__ partial) {
    __shared__ double warps[kThreads / 32U];
    const uint32_t tensor = TensorOf(t, blockIdx.x);
    const uint64_t begin = static_cast<uint64_t>(blockIdx.x - t.first_chunk[tensor]) * t.chunk, all = t.count[tensor] & kCountMask;
    const uint64_t n = all - begin < t.chunk ? all - begin : t.chunk;
    const int32_t type = static_cast<int32_t>(t.count[tensor] >> kTypeShift);
    mgt::dependent_begin();
    double s = type == MGT_F32    ? SumOfSquares(static_cast<const float*>(t.data[tensor]) + begin, n)
               : type == MGT_F16 ? SumOfSquares(static_cast<const __half*>(t.data[tensor]) + begin, n)
                                 : SumOfSquares(static_cast<const __nv_bfloat16*>(t.data[tensor]) + begin, n);
    s = WarpSum(s);
    if ((threadIdx.x & 31U) == 0U) warps[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0U) {
        for (uint32_t w = 1; w < kThreads / 32U; ++w) s += warps[w];
        partial[blockIdx.x] = s;
    }
}

// result = {norm, scale}; norms: of every tensor, if wanted. The chunks' sums come to shared memory at once, all loads in flight together; a
// tensor's are then added by the lanes of a warp, and the tensors by the CTA.
template <uint32_t kMost>
__global__ void __launch_bounds__(kFinishThreads)
FinishNormKernel(const __grid_constant__ Table<kMost> t, const double* __restrict__ partial, float max_norm, float* __restrict__ result, float* __restrict__ norms) {
    __shared__ double chunks[kMostChunks + kMost], squares[kMost], warps[kFinishThreads / 32U];
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31U, all = t.first_chunk[t.tensors];
    mgt::dependent_begin();
    const double* sums = mgt::after_begin(partial);
#pragma unroll
    for (uint32_t c = threadIdx.x; c < kMostChunks + kMost; c += kFinishThreads)
        if (c < all) chunks[c] = sums[c];
    __syncthreads();
    for (uint32_t k = warp; k < t.tensors; k += kFinishThreads / 32U) {
        const uint32_t end = t.first_chunk[k + 1U];
        double s = 0.0;
#pragma unroll 4
        for (uint32_t c = t.first_chunk[k] + lane; c < end; c += 32U) s += chunks[c];
        s = WarpSum(s);
        if (lane == 0U) {
            squares[k] = s;
            if (norms != nullptr) norms[k] = static_cast<float>(sqrt(s));
        }
    }
    __syncthreads();
    double s = threadIdx.x < t.tensors ? squares[threadIdx.x] : 0.0;  // (no list is longer than the CTA)
    s = WarpSum(s);
    if (lane == 0U) warps[warp] = s;
    __syncthreads();
    if (warp == 0U) {
        s = WarpSum(warps[lane]);
        if (lane == 0U) {
            const double norm = sqrt(s);
            const float shown = static_cast<float>(norm);
            result[0] = shown;
            // a norm that no float holds, or none at all, keeps nothing of the gradient
            result[1] = !(shown <= 3.402823466e38f) ? 0.0f : norm > static_cast<double>(max_norm) ? static_cast<float>(static_cast<double>(max_norm) / norm) : 1.0f;
        }
    }
}

template <uint32_t kMost>
__global__ void __launch_bounds__(kThreads)
ScaleKernel(const __grid_constant__ Table<kMost> t, const __grid_constant__ Outputs<kMost> out, const float* __restrict__ result, bool in_place) {
    const uint32_t chunk = gridDim.x - 1U - blockIdx.x;  // from the end, which the pass for the norm has left in L2
    const uint32_t tensor = TensorOf(t, chunk);
    const uint64_t begin = static_cast<uint64_t>(chunk - t.first_chunk[tensor]) * t.chunk, all = t.count[tensor] & kCountMask;
    const uint64_t n = all - begin < t.chunk ? all - begin : t.chunk;
    const int32_t type = static_cast<int32_t>(t.count[tensor] >> kTypeShift);
    mgt::dependent_begin();
    const float* found = mgt::after_begin(result);
    const float norm = found[0], scale = found[1];
    const bool zero = !(norm <= 3.402823466e38f);
    if (in_place && !zero && scale == 1.0f) return;  // every product is the value that is there
    if (type == MGT_F32) Scale(static_cast<const float*>(t.data[tensor]) + begin, static_cast<float*>(out.data[tensor]) + begin, n, scale, zero);
    else if (type == MGT_F16) Scale(static_cast<const __half*>(t.data[tensor]) + begin, static_cast<__half*>(out.data[tensor]) + begin, n, scale, zero);
    else Scale(static_cast<const __nv_bfloat16*>(t.data[tensor]) + begin, static_cast<__nv_bfloat16*>(out.data[tensor]) + begin, n, scale, zero);
}

bool Aligned(const void* p, uintptr_t bytes) { return p != nullptr && (reinterpret_cast<uintptr_t>(p) & (bytes - 1U)) == 0; }

bool ValidTensors(const mgt_tensor_t* tensors, uint32_t count) {
    if (tensors == nullptr || count == 0 || count > MGT_MAX_TENSORS) return false;
    uint64_t total = 0;
    for (uint32_t i = 0; i < count; ++i) {
        const mgt_tensor_t& t = tensors[i];
        if (t.type != MGT_F32 && t.type != MGT_F16 && t.type != MGT_BF16) return false;
        if (t.count > MGT_MAX_TENSOR_ELEMENTS || (t.count != 0 && !Aligned(t.data, t.type == MGT_F32 ? 4U : 2U))) return false;
        total += t.count;
    }
    return total <= MGT_MAX_TENSOR_ELEMENTS;
}
// Whether what a call writes overlaps itself, what it reads of other tensors, or the factor: CTAs would race for it, and a factor might be
// applied twice. One pass where the tensors lie in order of their addresses, as the views of one buffer do.
bool Clashing(const mgt_tensor_t* tensors, uint32_t count, const float* result, const mgt_tensor_t* out) {
    struct Span {
        uintptr_t begin, end;
        uint32_t index;
    };
    Span written[MGT_MAX_TENSORS];
    auto span = [](const mgt_tensor_t& t, uint32_t i) {
        const uintptr_t at = reinterpret_cast<uintptr_t>(t.data);
        return Span{at, at + t.count * (t.type == MGT_F32 ? 4U : 2U), i};
    };
    uint32_t n = 0;
    bool sorted = true;
    for (uint32_t i = 0; i < count; ++i) {
        if (tensors[i].count == 0) continue;
        written[n] = span(out != nullptr ? out[i] : tensors[i], i);
        if (n != 0 && written[n].begin < written[n - 1U].begin) sorted = false;
        ++n;
    }
    if (!sorted) std::sort(written, written + n, [](const Span& a, const Span& b) { return a.begin < b.begin; });
    for (uint32_t k = 1; k < n; ++k)
        if (written[k].begin < written[k - 1U].end) return true;
    auto first_behind = [&](uintptr_t at) { return std::lower_bound(written, written + n, at, [](const Span& a, uintptr_t p) { return a.end <= p; }); };
    const uintptr_t factor = reinterpret_cast<uintptr_t>(result);
    const Span* over = first_behind(factor);
    if (over != written + n && over->begin < factor + 2U * sizeof(float)) return true;
    if (out == nullptr) return false;
    for (uint32_t i = 0; i < count; ++i) {
        if (tensors[i].count == 0) continue;
        const Span read = span(tensors[i], i);
        const Span* w = first_behind(read.begin);
        if (w != written + n && w->begin < read.end && !(w->index == i && w->begin == read.begin)) return true;
    }
    return false;
}
uint64_t ChunkOf(const mgt_tensor_t* tensors, uint32_t count) {
    uint64_t total = 0;
    uint32_t bytes = 2;  // of the widest type
    for (uint32_t i = 0; i < count; ++i) {
        total += tensors[i].count;
        if (tensors[i].type == MGT_F32) bytes = 4;
    }
    const uint64_t chunk = (total / kMostChunks + 1024ULL) / 1024ULL * 1024ULL;
    return chunk < kLeastChunkBytes / bytes ? kLeastChunkBytes / bytes : chunk;
}
uint32_t Chunks(const mgt_tensor_t* tensors, uint32_t count, uint64_t chunk) {
    uint64_t n = 0;
    for (uint32_t i = 0; i < count; ++i) n += (tensors[i].count + chunk - 1ULL) / chunk;
    return static_cast<uint32_t>(n);
}
template <uint32_t kMost>
void Fill(Table<kMost>* t, const mgt_tensor_t* tensors, uint32_t count) {
    t->tensors = count;
    t->chunk = ChunkOf(tensors, count);
    t->first_chunk[0] = 0;
    for (uint32_t i = 0; i < count; ++i) {
        t->data[i] = tensors[i].data;
        t->count[i] = tensors[i].count | static_cast<uint64_t>(tensors[i].type) << kTypeShift;
        t->first_chunk[i + 1U] = t->first_chunk[i] + static_cast<uint32_t>((tensors[i].count + t->chunk - 1ULL) / t->chunk);
    }
}

template <uint32_t kMost>
void RunNorm(const mgt_tensor_t* tensors, uint32_t count, float max_norm, float* result, float* norms, double* partial, cudaStream_t s) {
    Table<kMost> t;
    Fill(&t, tensors, count);
    const uint32_t chunks = t.first_chunk[count];
    if (chunks != 0) mgt::Launch(ChunkSquaresKernel<kMost>, chunks, kThreads, 0, {s, true}, t, partial);
    mgt::Launch(FinishNormKernel<kMost>, 1, kFinishThreads, 0, {s, true}, t, static_cast<const double*>(partial), max_norm, result, norms);
}
template <uint32_t kMost>
void RunScale(const mgt_tensor_t* tensors, uint32_t count, const mgt_tensor_t* out, const float* result, cudaStream_t s) {
    Table<kMost> t;
    Outputs<kMost> o;
    Fill(&t, tensors, count);
    for (uint32_t i = 0; i < count; ++i) o.data[i] = const_cast<void*>(out != nullptr ? out[i].data : tensors[i].data);
    if (t.first_chunk[count] != 0) mgt::Launch(ScaleKernel<kMost>, t.first_chunk[count], kThreads, 0, {s, true}, t, o, result, out == nullptr);
}

}  // namespace

extern "C" {

uint64_t mgt_gradient_norm_workspace_floats(const mgt_tensor_t* tensors, uint32_t tensor_count) {
    if (!ValidTensors(tensors, tensor_count)) return 0;
    return 2ULL * Chunks(tensors, tensor_count, ChunkOf(tensors, tensor_count)) + 2ULL;
}

mgt_status_t mgt_launch_gradient_norm(const mgt_tensor_t* tensors, uint32_t tensor_count, float max_norm, float* device_result, float* device_tensor_norms,
                                      float* workspace, uint64_t workspace_floats, void* stream) {
    if (!ValidTensors(tensors, tensor_count) || !(max_norm > 0.0f) || !Aligned(device_result, 4) || !Aligned(workspace, 8) ||
        (device_tensor_norms != nullptr && !Aligned(device_tensor_norms, 4))) {
        return MGT_INVALID_CONFIG;
    }
    if (workspace_floats < mgt_gradient_norm_workspace_floats(tensors, tensor_count)) return MGT_CAPACITY_EXCEEDED;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    double* partial = reinterpret_cast<double*>(workspace);
    if (tensor_count <= 96U) RunNorm<96>(tensors, tensor_count, max_norm, device_result, device_tensor_norms, partial, s);
    else RunNorm<MGT_MAX_TENSORS>(tensors, tensor_count, max_norm, device_result, device_tensor_norms, partial, s);
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}

mgt_status_t mgt_launch_clip_gradients(const mgt_tensor_t* tensors, uint32_t tensor_count, const float* device_result, const mgt_tensor_t* out_tensors, void* stream) {
    if (!ValidTensors(tensors, tensor_count) || !Aligned(device_result, 4)) return MGT_INVALID_CONFIG;
    if (out_tensors != nullptr) {
        if (!ValidTensors(out_tensors, tensor_count)) return MGT_INVALID_CONFIG;
        for (uint32_t i = 0; i < tensor_count; ++i)
            if (out_tensors[i].count != tensors[i].count || out_tensors[i].type != tensors[i].type) return MGT_INVALID_CONFIG;
    }
    if (Clashing(tensors, tensor_count, device_result, out_tensors)) return MGT_INVALID_CONFIG;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tensor_count <= 96U) RunScale<96>(tensors, tensor_count, out_tensors, device_result, s);
    else RunScale<MGT_MAX_TENSORS>(tensors, tensor_count, out_tensors, device_result, s);
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}

}  // extern "C"

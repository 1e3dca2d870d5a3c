// Layer normalisation: how a row is held. A row of C columns is shared by `lanes` threads (a power of two, at most a CTA); thread t has
// the packs t, t + lanes, ... of V neighbouring elements, NV of them at most, all in registers, so that a row is read once. Several rows
// lie side by side in a CTA. Groups of up to 32 lanes reduce by shuffles, wider ones through shared memory and a barrier of their own.
#pragma once

#include "layer_norm.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace mgt {
namespace ln {

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V neighbouring elements as they lie in memory, moved in accesses of up to 16 bytes.
template <class T, int V>
struct alignas(sizeof(T) * V > 16 ? 16 : sizeof(T) * V) Pack {
    T v[V];
};
template <int kBytes> struct Word { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };

template <class T, int V>
__device__ __forceinline__ void LoadPack(Pack<T, V>& out, const T* p, uint32_t valid) {
    using W = typename Word<(sizeof(T) * V > 16 ? 16 : sizeof(T) * V)>::type;
    constexpr int kWords = sizeof(T) * V / sizeof(W);
    if (valid >= V) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<W*>(&out)[i] = reinterpret_cast<const W*>(p)[i];
    } else {  // the last pack of a row, or none of it
#pragma unroll
        for (int i = 0; i < V; ++i) out.v[i] = i < valid ? p[i] : FromFloat<T>(0.0f);
    }
}
template <class T, int V>
__device__ __forceinline__ void StorePack(T* p, const float (&v)[V], uint32_t valid) {
    using W = typename Word<(sizeof(T) * V > 16 ? 16 : sizeof(T) * V)>::type;
    constexpr int kWords = sizeof(T) * V / sizeof(W);
    Pack<T, V> out;
#pragma unroll
    for (int i = 0; i < V; ++i) out.v[i] = FromFloat<T>(v[i]);
    if (valid >= V) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) reinterpret_cast<W*>(p)[i] = reinterpret_cast<const W*>(&out)[i];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < valid) p[i] = out.v[i];
    }
}

// The threads that share a row. Reductions alternate between two buffers: who writes one again has passed the barrier of the other, and
// with it everybody's reads of this one.
struct Group {
    uint32_t lanes, lane, index, count;  // threads of a group, place in it, group of the CTA, groups of the CTA
    float2* buffer;                      // [2][warps of the CTA]
    uint32_t turn;
};
__device__ __forceinline__ Group MakeGroup(uint32_t lanes, float2* buffer) {
    return {lanes, threadIdx.x & (lanes - 1U), threadIdx.x / lanes, blockDim.x / lanes, buffer, 0U};
}
// Sums of a and b over the group, in every one of its threads. All threads of a warp come here together.
__device__ __forceinline__ float2 Reduce(Group& g, float a, float b) {
    for (uint32_t o = min(g.lanes, 32U) >> 1; o > 0U; o >>= 1) {
        a += __shfl_xor_sync(0xffffffffU, a, o);
        b += __shfl_xor_sync(0xffffffffU, b, o);
    }
    if (g.lanes > 32U) {
        const uint32_t warps = g.lanes >> 5, warp = threadIdx.x >> 5, lane = threadIdx.x & 31U;
        float2* at = g.buffer + (g.turn & 1U) * (blockDim.x >> 5);
        g.turn ^= 1U;
        if (lane == 0U) at[warp] = make_float2(a, b);
        asm volatile("bar.sync %0, %1;" ::"r"(1U + g.index), "r"(g.lanes) : "memory");
        const float2 part = lane < warps ? at[g.index * warps + lane] : make_float2(0.0f, 0.0f);
        a = part.x;
        b = part.y;
        for (uint32_t o = warps >> 1; o > 0U; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffU, a, o);
            b += __shfl_xor_sync(0xffffffffU, b, o);
        }
        a = __shfl_sync(0xffffffffU, a, 0);
        b = __shfl_sync(0xffffffffU, b, 0);
    }
    return make_float2(a, b);
}

// Column of this thread's pack i, and how many of its elements the row has.
template <int V>
__device__ __forceinline__ uint32_t PackColumn(const Group& g, int i) { return (static_cast<uint32_t>(i) * g.lanes + g.lane) * V; }
__device__ __forceinline__ uint32_t PackValid(uint32_t column, uint32_t cols) { return column < cols ? cols - column : 0U; }

// ---- host side: how a row is cut
constexpr uint32_t kMostLanes = 512;
struct Cut {
    int v, nv;           // elements of a pack, packs a thread
    uint32_t lanes, threads;
    bool stream;         // wider than the registers of a CTA hold
};
inline uint32_t PowerOfTwo(uint32_t n) {
    uint32_t p = 1;
    while (p < n) p <<= 1;
    return p;
}
// elements: what a thread can hold. Packs a thread are 1, 2, 4, 8 or 16.
inline Cut CutRow(uint32_t cols, int v, int elements) {
    const uint32_t packs = (cols - 1U) / static_cast<uint32_t>(v) + 1U, most = static_cast<uint32_t>(elements / v);
    Cut c{v, 1, 1, 256, false};
    if (packs <= 32U) {
        c.lanes = PowerOfTwo(packs);
    } else if (packs <= 32U * most) {
        c.lanes = 32;
        c.nv = static_cast<int>(PowerOfTwo((packs + 31U) / 32U));
    } else {
        c.nv = static_cast<int>(most);
        if (packs > most * kMostLanes) {
            c.stream = true;
            return c;
        }
        c.lanes = PowerOfTwo((packs - 1U) / most + 1U);
        if (c.lanes > c.threads) c.threads = c.lanes;
    }
    return c;
}
inline uint32_t TypeBytes(int32_t type) { return type == MGT_F32 ? 4U : 2U; }
inline bool RowsAligned(const void* p, uint64_t pitch, uint32_t rows, int32_t type, int v) {
    const uint64_t bytes = TypeBytes(type) * static_cast<uint64_t>(v), unit = bytes > 16U ? 16U : bytes;
    return (reinterpret_cast<uintptr_t>(p) % unit) == 0 && (rows <= 1U || (pitch * TypeBytes(type)) % unit == 0);
}

}  // namespace ln
}  // namespace mgt

// Layer normalisation: how rows are held and fetched. A row of C columns is shared by `lanes` threads (a power of two, at most a CTA); thread
// t has the packs t, t + lanes, ... of V neighbouring elements, 16 elements at most. Several rows lie side by side in a CTA. Groups
// of up to 32 lanes reduce by shuffles, wider ones through shared memory and a barrier of their own.
//
// The kernels are bound by HBM, and what that takes is bytes in flight: some 45 KB an SM at 6.5 TB/s and a loaded latency of 1 us. One
// row ahead in registers leaves 24 KB in flight (131 072 x 512 bf16 forward 107 us); so a thread copies what it will need of its next rows to
// shared memory asynchronously, several rows deep.
#pragma once

#include "layer_norm.hpp"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace mgt {
namespace ln {

__device__ __forceinline__ float ToFloat(float v) { return v; }
__device__ __forceinline__ float ToFloat(__half v) { return __half2float(v); }
__device__ __forceinline__ float ToFloat(__nv_bfloat16 v) { return __bfloat162float(v); }
template <class T> __device__ __forceinline__ T FromFloat(float v);
template <> __device__ __forceinline__ float FromFloat<float>(float v) { return v; }
template <> __device__ __forceinline__ __half FromFloat<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 FromFloat<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V neighbouring elements as they lie in memory, moved in one access.
template <class T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};
template <int kBytes> struct Word { using type = uint4; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<2> { using type = uint16_t; };
template <class T, int V>
__device__ __forceinline__ Pack<T, V> LoadPack(const T* p) {
    Pack<T, V> out;
    using W = typename Word<sizeof(T) * V>::type;
    *reinterpret_cast<W*>(&out) = *reinterpret_cast<const W*>(p);
    return out;
}
template <class T, int V>
__device__ __forceinline__ void StorePack(T* p, const Pack<T, V>& v) {
    using W = typename Word<sizeof(T) * V>::type;
    *reinterpret_cast<W*>(p) = *reinterpret_cast<const W*>(&v);
}

// The elements that a thread holds of a row, as fp32 pairs (one element alone has a zero beside it): half as many instructions as by
// single values, and instructions are what bounds these kernels once their loads are far enough ahead.
__device__ __forceinline__ uint64_t& Bits(float2& v) { return reinterpret_cast<uint64_t&>(v); }
__device__ __forceinline__ float2 Add2(float2 a, float2 b) {
    float2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(Bits(r)) : "l"(Bits(a)), "l"(Bits(b)));
    return r;
}
__device__ __forceinline__ float2 Mul2(float2 a, float2 b) {
    float2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(Bits(r)) : "l"(Bits(a)), "l"(Bits(b)));
    return r;
}
__device__ __forceinline__ float2 Fma2(float2 a, float2 b, float2 c) {
    float2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(Bits(r)) : "l"(Bits(a)), "l"(Bits(b)), "l"(Bits(c)));
    return r;
}
__device__ __forceinline__ float2 Both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 Up(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 Up(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ float2 Up(float2 v) { return v; }
template <class T> struct Two;
template <> struct Two<float> { using type = float2; static __device__ __forceinline__ float2 Down(float2 v) { return v; } };
template <> struct Two<__half> { using type = __half2; static __device__ __forceinline__ __half2 Down(float2 v) { return __floats2half2_rn(v.x, v.y); } };
template <> struct Two<__nv_bfloat16> { using type = __nv_bfloat162; static __device__ __forceinline__ __nv_bfloat162 Down(float2 v) { return __floats2bfloat162_rn(v.x, v.y); } };
template <int E>
struct Held {
    static constexpr int kPairs = (E + 1) / 2;
    float2 pair[kPairs];
    __device__ __forceinline__ void Set(int k, float v) {
        if (k & 1) pair[k / 2].y = v; else pair[k / 2].x = v;
        if (E == 1) pair[0].y = 0.0f;
    }
    __device__ __forceinline__ float Get(int k) const { return k & 1 ? pair[k / 2].y : pair[k / 2].x; }
};

// The threads that share a row. Reductions alternate between two buffers: who writes one again has passed the barrier of the other, and
// with it everybody's reads of this one.
struct Group {
    uint32_t lanes, lane, index, count;  // threads of a group, place in it, group of the CTA, groups of the CTA
    float* buffer;                       // [2][warps of the CTA][values of a reduction]
    uint32_t turn;
};
__device__ __forceinline__ Group MakeGroup(uint32_t lanes, float* buffer) {
    return {lanes, threadIdx.x & (lanes - 1U), threadIdx.x / lanes, blockDim.x / lanes, buffer, 0U};
}
// Sums of N values (a power of two) over the group, in every one of its threads. All threads of a warp come here together. Groups of N lanes
// and more halve the values that a lane still adds up with every step, N - 1 shuffles for the first log2(N) of them instead of N log2(N).
constexpr __host__ __device__ int ReverseBits(int i, int n) { return n <= 1 ? 0 : (i & 1) * (n / 2) + ReverseBits(i / 2, n / 2); }
template <int N>
__device__ __forceinline__ void Reduce(Group& g, float (&v)[N]) {
    const uint32_t lane = threadIdx.x & 31U;
    if (g.lanes < N) {
#pragma unroll
        for (uint32_t o = N / 2U; o > 0U; o >>= 1) {
            if (o >= g.lanes) continue;  // (the same for the whole CTA)
#pragma unroll
            for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffU, v[n], o);
        }
        return;
    }
#pragma unroll
    for (int half = N / 2; half > 0; half /= 2) {  // lanes with the step's bit keep the upper half
        const int o = N / 2 / half;
        const bool up = (lane & o) != 0U;
#pragma unroll
        for (int n = 0; n < half; ++n) {
            const float give = up ? v[n] : v[n + half], keep = up ? v[n + half] : v[n];
            v[n] = keep + __shfl_xor_sync(0xffffffffU, give, o);
        }
    }
    float mine = v[0];  // of value ReverseBits(lane % N)
#pragma unroll
    for (uint32_t o = N; o < 32U; o <<= 1)
        if (o < g.lanes) mine += __shfl_xor_sync(0xffffffffU, mine, o);
    if (g.lanes > 32U) {
        const uint32_t warps = g.lanes >> 5, warp = threadIdx.x >> 5;
        float* at = g.buffer + (g.turn & 1U) * (blockDim.x >> 5) * N;
        g.turn ^= 1U;
        if (lane < N) at[warp * N + lane] = mine;
        asm volatile("bar.sync %0, %1;" ::"r"(1U + g.index), "r"(g.lanes) : "memory");
        mine = 0.0f;
#pragma unroll
        for (uint32_t w = 0; w < 32U; w += 32U / N)
            if (w + lane / N < warps) mine += at[(g.index * warps + w) * N + lane];
#pragma unroll
        for (uint32_t o = N; o < 32U; o <<= 1) mine += __shfl_xor_sync(0xffffffffU, mine, o);
    }
    const uint32_t base = g.lanes < 32U ? lane & ~(g.lanes - 1U) : 0U;
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = N == 1 ? mine : __shfl_sync(0xffffffffU, mine, base + ReverseBits(n, N));
}

// Which rows a group has: the first one, every stride-th from there, `mine` in all; `turns` of the warp's group that has most.
struct Share {
    uint32_t first, stride, mine, turns;
};
__device__ __forceinline__ Share MakeShare(const Group& g, uint32_t rows) {
    Share s;
    s.first = blockIdx.x * g.count + g.index;
    s.stride = gridDim.x * g.count;
    const uint32_t least = g.lanes < 32U ? s.first - (g.index & (32U / g.lanes - 1U)) : s.first;
    s.mine = s.first < rows ? (rows - 1U - s.first) / s.stride + 1U : 0U;
    s.turns = least < rows ? (rows - 1U - least) / s.stride + 1U : 0U;
    return s;
}

// Column of this thread's pack i. Packs are whole: the row has all of one or nothing.
template <int V>
__device__ __forceinline__ uint32_t PackColumn(const Group& g, int i) { return (static_cast<uint32_t>(i) * g.lanes + g.lane) * V; }

template <int kBytes>
__device__ __forceinline__ void CopyAsync(uint32_t to, const void* from) {
    if constexpr (kBytes == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
    else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(kBytes) : "memory");
}
__device__ __forceinline__ void CopiesEnd() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kLeft>
__device__ __forceinline__ void CopiesWait() { asm volatile("cp.async.wait_group %0;" ::"n"(kLeft) : "memory"); }

// What a thread has of its next kDepth rows of one operand, in shared memory.
//   V > 1   packs of 16 (or 8) bytes. A thread reads only what it copied itself: nothing is shared, and nothing waits.
//   V = 1   rows that begin anywhere: the group copies the 16-byte lines that its row lies in, and a thread reads its elements from them
//           behind a barrier of the group. Lines that reach beyond the matrix are copied by elements.
template <class T, int V, int NV, int kThreads, int kDepth>
struct Ring {
    static constexpr uint32_t kPackBytes = sizeof(T) * V;
    const T* next;       // the row to be fetched next
    const T* now;        // the row to be read next
    uint64_t step;       // elements from a row of the group to its next
    uint32_t cols, line_bytes;  // line_bytes: of a group's row (V = 1)
    char* slots;         // of this thread (V > 1) or group
    uintptr_t least, most;      // the matrix (V = 1)

    static __host__ __device__ uint32_t LineBytes(uint32_t cols) { return (cols * static_cast<uint32_t>(sizeof(T)) + 15U) / 16U * 16U + 16U; }
    static __host__ __device__ uint32_t Bytes(uint32_t cols, uint32_t groups) {
        return kDepth * (V > 1 ? NV * kThreads * kPackBytes : groups * LineBytes(cols));
    }
    __device__ __forceinline__ Ring(const void* base, uint64_t pitch, uint32_t rows, uint32_t cols_, char* memory, const Group& g, const Share& share) {
        next = now = static_cast<const T*>(base) + share.first * pitch + (V > 1 ? g.lane * V : 0U);
        step = share.stride * pitch;
        cols = cols_;
        line_bytes = LineBytes(cols_);
        slots = memory + (V > 1 ? threadIdx.x * kPackBytes : g.index * line_bytes);
        least = reinterpret_cast<uintptr_t>(base);
        most = reinterpret_cast<uintptr_t>(static_cast<const T*>(base) + (rows - 1ULL) * pitch + cols_);
    }
    __device__ __forceinline__ char* Slot(const Group& g, uint32_t turn, int i) const {
        if constexpr (V > 1) return slots + (turn * NV + i) * (kThreads * kPackBytes);
        else return slots + turn * g.count * line_bytes;
    }
    // The group's next row, zeros where there is none left.
    __device__ __forceinline__ void Fetch(const Group& g, uint32_t turn, bool in) {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (PackColumn<V>(g, i) >= cols) continue;
                if (in) CopyAsync<kPackBytes>(static_cast<uint32_t>(__cvta_generic_to_shared(Slot(g, turn, i))), next + i * g.lanes * V);
                else *reinterpret_cast<typename Word<kPackBytes>::type*>(Slot(g, turn, i)) = {};
            }
        } else if (in) {
            const uintptr_t begin = reinterpret_cast<uintptr_t>(next), end = begin + static_cast<uintptr_t>(cols) * sizeof(T);
            char* to = Slot(g, turn, 0) + 16U * g.lane;
            for (uintptr_t line = (begin & ~static_cast<uintptr_t>(15)) + 16U * g.lane; line < end; line += 16U * g.lanes, to += 16U * g.lanes) {
                if (line >= least && line + 16U <= most) {
                    CopyAsync<16>(static_cast<uint32_t>(__cvta_generic_to_shared(to)), reinterpret_cast<const void*>(line));
                } else {
                    for (uintptr_t e = line < begin ? begin : line; e < end && e < line + 16U; e += sizeof(T))
                        *reinterpret_cast<T*>(to + (e - line)) = *reinterpret_cast<const T*>(e);
                }
            }
        }
        next += step;
    }
    // Before the first fetch: what lies beyond the row's end is zero in every slot and stays so (V > 1).
    __device__ __forceinline__ void Clear(const Group& g) {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i)
                if (PackColumn<V>(g, i) >= cols)
                    for (uint32_t turn = 0; turn < kDepth; ++turn) *reinterpret_cast<typename Word<kPackBytes>::type*>(Slot(g, turn, i)) = {};
        }
    }
    // This thread's elements of a row that has arrived; zeros beyond the row's end, and where there is no row.
    __device__ __forceinline__ void Read(Held<NV * V>& out, const Group& g, uint32_t turn, bool in) {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const Pack<T, V> p = LoadPack<T, V>(reinterpret_cast<const T*>(Slot(g, turn, i)));
#pragma unroll
                for (int j = 0; j < V / 2; ++j) out.pair[i * (V / 2) + j] = Up(reinterpret_cast<const typename Two<T>::type*>(&p)[j]);
            }
        } else {
            const T* line = reinterpret_cast<const T*>(Slot(g, turn, 0) + (reinterpret_cast<uintptr_t>(now) & 15U));
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const uint32_t c = PackColumn<V>(g, i);
                out.Set(i, in && c < cols ? ToFloat(line[c]) : 0.0f);
            }
            now += step;
        }
    }
};
template <class T, int V, int E>
__device__ __forceinline__ Pack<T, V> PackOf(const Held<E>& v, int i) {
    Pack<T, V> p;
    if constexpr (V == 1) {
        p.v[0] = FromFloat<T>(v.Get(i));
    } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) reinterpret_cast<typename Two<T>::type*>(&p)[j] = Two<T>::Down(v.pair[i * (V / 2) + j]);
    }
    return p;
}
// `value` where the thread's elements are in the row, zero where they are not.
template <int V, int NV>
__device__ __forceinline__ void InRow(Held<NV * V>& out, const Group& g, uint32_t cols, float value) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const float v = PackColumn<V>(g, i) < cols ? value : 0.0f;
#pragma unroll
        for (int j = 0; j < V; ++j) out.Set(i * V + j, v);
    }
}
// A vector of columns that may begin anywhere; `none` for no vector, zero beyond the row's end.
template <int V, int NV>
__device__ __forceinline__ void LoadColumns(Held<NV * V>& out, const Group& g, uint32_t cols, const float* p, float none) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const uint32_t c = PackColumn<V>(g, i);
#pragma unroll
        for (int j = 0; j < V; ++j) out.Set(i * V + j, c < cols ? (p != nullptr ? p[c + j] : none) : 0.0f);
    }
}
template <int E>
__device__ __forceinline__ float SumOf(const Held<E>& v) {
    float2 s = v.pair[0];
#pragma unroll
    for (int k = 1; k < Held<E>::kPairs; ++k) s = Add2(s, v.pair[k]);
    return s.x + s.y;
}
// Everybody of the group sees what the group copied, or has read what it will overwrite.
__device__ __forceinline__ void GroupBarrier(const Group& g) {
    if (g.lanes <= 32U) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1U + g.index), "r"(g.lanes) : "memory");
}

// ---- host side: how a row is cut
constexpr uint32_t kMostLanes = 512, kElements = 16;
struct Cut {
    int nv;              // packs a thread: 1, 2, 4, 8 or 16
    uint32_t lanes, threads;
    bool stream;         // wider than a CTA holds
};
inline uint32_t PowerOfTwo(uint32_t n) {
    uint32_t p = 1;
    while (p < n) p <<= 1;
    return p;
}
// As few lanes a row as can hold it, which makes the reductions short, or more where the rows are too few to fill the chip's threads.
inline Cut CutRow(uint32_t rows, uint32_t cols, uint32_t v) {
    const uint32_t packs = (cols - 1U) / v + 1U, most = kElements / v;
    Cut c{1, 1, 256, false};
    if (packs > most * kMostLanes) {
        c.stream = true;
        return c;
    }
    c.lanes = PowerOfTwo((packs - 1U) / most + 1U);
    if (v == 1U && c.lanes < 4U) c.lanes = 4;  // (a line of 16 bytes and more a row: not too many rows a CTA)
    while (c.lanes < 256U && c.lanes < packs && static_cast<uint64_t>(rows) * c.lanes < 148ULL * 512ULL) c.lanes <<= 1;
    c.nv = static_cast<int>(PowerOfTwo((packs - 1U) / c.lanes + 1U));
    if (c.lanes > c.threads) c.threads = c.lanes;
    return c;
}
// Dynamic shared memory beyond 48 KB is an attribute of a kernel on a device: set on the first launch there.
template <class Kernel>
inline bool AllowShared(Kernel kernel, std::atomic<uint64_t>& done, int bytes) {
    int device = 0;
    if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return false;
    const uint64_t bit = 1ULL << device;
    if ((done.load(std::memory_order_relaxed) & bit) != 0) return true;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done.fetch_or(bit, std::memory_order_relaxed);
    return true;
}
inline uint32_t TypeBytes(int32_t type) { return type == MGT_F32 ? 4U : 2U; }
inline bool RowsAligned(const void* p, uint64_t pitch, uint32_t rows, int32_t type, int v) {
    const uint64_t bytes = TypeBytes(type) * static_cast<uint64_t>(v);
    return (reinterpret_cast<uintptr_t>(p) % bytes) == 0 && (rows <= 1U || (pitch * TypeBytes(type)) % bytes == 0);
}

}  // namespace ln
}  // namespace mgt

// Layer normalisation: how rows are held and fetched. A row of C columns is shared by `lanes` threads (a power of two, at most a CTA), which
// hold 16 or 32 of its elements each. Several rows lie side by side in a CTA. Groups of up to 32 lanes reduce by shuffles, wider ones
// through shared memory and a barrier of their own.
//
// The kernels are bound by HBM, and what that takes is bytes in flight: some 45 KB an SM at 6.5 TB/s and a loaded latency of 1 us. One
// row ahead in registers leaves 24 KB in flight (131 072 x 512 bf16 forward 107 us); so a thread copies what it will need of its next rows to
// shared memory asynchronously, two to four rows deep (one, where a row of 32 KB and more fills a CTA).
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
// cta of ctas: CTAs that share a row count as one.
__device__ __forceinline__ Share MakeShare(const Group& g, uint32_t rows, uint32_t cta, uint32_t ctas) {
    Share s;
    s.first = cta * g.count + g.index;
    s.stride = ctas * g.count;
    const uint32_t least = g.lanes < 32U ? s.first - (g.index & (32U / g.lanes - 1U)) : s.first;
    s.mine = s.first < rows ? (rows - 1U - s.first) / s.stride + 1U : 0U;
    s.turns = least < rows ? (rows - 1U - least) / s.stride + 1U : 0U;
    return s;
}

// Which columns a thread has.
//   V > 1   packs t, t + lanes, ... of V columns; a pack is whole: the row has all of it or nothing.
//   V = 1   L (8 or 32) neighbouring lanes share a stretch of the row, one column to each in turn; stretches differ by a column at most. So
//           places are constants, and only the last kMasked turns have to look at the stretch's end. (131 072 rows of 301 fp16, forward: 54 us,
//           82 where every turn asks.)
template <int V_, int NV_, int L_, int kMasked_>
struct Layout {
    static constexpr int V = V_, NV = NV_, L = L_, E = V * NV, kMasked = kMasked_;
    uint32_t cols, lanes, base;
    uint32_t begin, end, mask;  // V = 1: the stretch, and which of the lane's last turns lie in it
    __device__ __forceinline__ Layout(const Group& g, uint32_t cols_) : cols(cols_), lanes(g.lanes), base(g.lane * V), begin(0), end(0), mask(0) {
        if constexpr (V == 1) {
            const uint32_t stretch = g.lane / L, stretches = lanes / L;
            begin = stretch * cols / stretches;
            end = (stretch + 1U) * cols / stretches;
            base = begin + g.lane % L;
#pragma unroll
            for (int i = NV - kMasked; i < NV; ++i)
                if (base + i * L < end) mask |= 1U << i;
        }
    }
    __device__ __forceinline__ uint32_t Offset(int i) const { return V > 1 ? i * lanes * V : i * L; }  // of pack i from `base`
    __device__ __forceinline__ bool Has(int i) const {
        if constexpr (V > 1) return base + Offset(i) < cols;
        else return i < NV - kMasked || (mask >> i & 1U) != 0U;
    }
    // The values for the pair k of a thread's elements, zeros beyond the row's end.
    __device__ __forceinline__ float2 HasPair(int k, float2 v) const {
        if constexpr (V > 1) return Has(k / (V / 2)) ? v : make_float2(0.0f, 0.0f);
        else return make_float2(Has(2 * k) ? v.x : 0.0f, Has(2 * k + 1) ? v.y : 0.0f);
    }
    template <class F>
    __device__ __forceinline__ void Each(F f) const {  // f(i, whether the row has pack i)
#pragma unroll
        for (int i = 0; i < NV; ++i) f(i, Has(i));
    }
};

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
//   V = 1   rows that begin anywhere: the lanes of a stretch copy the 16-byte lines that it lies in, and read their elements from them
//           once the warp has met. Lines that reach beyond the matrix are copied by elements.
template <class T, class Lay, int kThreads, int kDepth>
struct Ring {
    static constexpr int V = Lay::V, NV = Lay::NV;
    static constexpr uint32_t kPackBytes = sizeof(T) * V;
    static constexpr uint32_t kLineBytes = (Lay::L * NV * sizeof(T) + 15U) / 16U * 16U + 16U;  // of a stretch (V = 1)
    static constexpr uint32_t kBytes = kDepth * (V > 1 ? NV * kThreads * kPackBytes : kThreads / Lay::L * kLineBytes);
    const T* next;              // this thread's (V > 1) or the stretch's columns in the row to be fetched next
    uint64_t step;              // elements from a row of the group to its next
    uint32_t now, now_step;     // where the row to be read next begins, from a 16-byte boundary (V = 1)
    char* slots;                // of this thread (V > 1) or stretch
    uintptr_t least, most;      // the matrix (V = 1)

    __device__ __forceinline__ Ring(const T* base, uint64_t pitch, uint32_t rows, char* memory, const Share& share, const Lay& lay) {
        next = base + share.first * pitch + (V > 1 ? lay.base : lay.begin);
        step = share.stride * pitch;
        slots = memory + (V > 1 ? threadIdx.x * kPackBytes : threadIdx.x / Lay::L * kLineBytes);
        now = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(next));
        now_step = static_cast<uint32_t>(step * sizeof(T));
        least = reinterpret_cast<uintptr_t>(base);
        most = reinterpret_cast<uintptr_t>(base + (rows - 1ULL) * pitch + lay.cols);
    }
    __device__ __forceinline__ char* Slot(uint32_t turn, int i) const {
        if constexpr (V > 1) return slots + (turn * NV + i) * (kThreads * kPackBytes);
        else return slots + turn * (kThreads / Lay::L * kLineBytes);
    }
    // The group's next row, zeros (V > 1) where there is none left.
    __device__ __forceinline__ void Fetch(const Lay& lay, uint32_t turn, bool in) {
        if constexpr (V > 1) {
            lay.Each([&](int i, bool has) {
                if (!has) return;
                if (in) CopyAsync<kPackBytes>(static_cast<uint32_t>(__cvta_generic_to_shared(Slot(turn, i))), next + lay.Offset(i));
                else *reinterpret_cast<typename Word<kPackBytes>::type*>(Slot(turn, i)) = {};
            });
        } else if (in) {
            const uint32_t shift = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(next)) & 15U, lane = threadIdx.x % Lay::L;
            const uint32_t bytes = (lay.end - lay.begin) * static_cast<uint32_t>(sizeof(T)) + shift, lines = (bytes + 15U) / 16U;
            const uintptr_t first = reinterpret_cast<uintptr_t>(next) - shift;
            char* to = Slot(turn, 0);
            if (first >= least && first + lines * 16U <= most) {
                const uint32_t at = static_cast<uint32_t>(__cvta_generic_to_shared(to)) + 16U * lane;
                const char* from = reinterpret_cast<const char*>(first) + 16U * lane;
#pragma unroll
                for (uint32_t k = 0; k < (kLineBytes / 16U + Lay::L - 1U) / Lay::L; ++k)
                    if (k * Lay::L + lane < lines) CopyAsync<16>(at + k * Lay::L * 16U, from + k * Lay::L * 16U);
            } else {
                for (uint32_t e = shift + lane * static_cast<uint32_t>(sizeof(T)); e < bytes; e += Lay::L * static_cast<uint32_t>(sizeof(T)))
                    *reinterpret_cast<T*>(to + e) = *reinterpret_cast<const T*>(first + e);
            }
        }
        next += step;
    }
    // Before the first fetch: what lies beyond the row's end is zero in every slot and stays so (V > 1).
    __device__ __forceinline__ void Clear(const Lay& lay) {
        if constexpr (V > 1) {
            lay.Each([&](int i, bool has) {
                if (has) return;
                for (uint32_t turn = 0; turn < kDepth; ++turn) *reinterpret_cast<typename Word<kPackBytes>::type*>(Slot(turn, i)) = {};
            });
        }
    }
    // This thread's elements of a row that has arrived; zeros beyond the row's end, and where there is no row (what a line holds that nothing was
    // copied to is read there and left aside).
    __device__ __forceinline__ void Read(Held<V * NV>& out, const Lay& lay, uint32_t turn, bool in) {
        if constexpr (V > 1) {
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const Pack<T, V> p = LoadPack<T, V>(reinterpret_cast<const T*>(Slot(turn, i)));
#pragma unroll
                for (int j = 0; j < V / 2; ++j) out.pair[i * (V / 2) + j] = Up(reinterpret_cast<const typename Two<T>::type*>(&p)[j]);
            }
        } else {
            const T* line = reinterpret_cast<const T*>(Slot(turn, 0) + (now & 15U)) + threadIdx.x % Lay::L;
            lay.Each([&](int i, bool has) { out.Set(i, has ? ToFloat(line[i * Lay::L]) : 0.0f); });
            if (!in) {
#pragma unroll
                for (int k = 0; k < Held<V * NV>::kPairs; ++k) out.pair[k] = Both(0.0f);
            }
            now += now_step;
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
// A vector of columns that may begin anywhere; `none` for no vector, zero beyond the row's end.
template <class Lay>
__device__ __forceinline__ void LoadColumns(Held<Lay::E>& out, const Lay& lay, const float* p, float none) {
    if (Lay::V > 1 && p != nullptr && (reinterpret_cast<uintptr_t>(p) & 15U) == 0U) {  // (single loads of packs touch a sector a lane)
#pragma unroll
        for (int i = 0; i < Lay::NV; ++i)
#pragma unroll
            for (int j = 0; j < Lay::V; j += 4) {
                const float4 v = lay.Has(i) ? *reinterpret_cast<const float4*>(p + lay.base + lay.Offset(i) + j) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                out.pair[(i * Lay::V + j) / 2] = make_float2(v.x, v.y);
                out.pair[(i * Lay::V + j) / 2 + 1] = make_float2(v.z, v.w);
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < Lay::NV; ++i)
#pragma unroll
        for (int j = 0; j < Lay::V; ++j) out.Set(i * Lay::V + j, lay.Has(i) ? (p != nullptr ? p[lay.base + lay.Offset(i) + j] : none) : 0.0f);
}
template <class Lay>
__device__ __forceinline__ void StoreColumns(float* p, const Held<Lay::E>& v, const Lay& lay) {
    if (Lay::V > 1 && (reinterpret_cast<uintptr_t>(p) & 15U) == 0U) {
#pragma unroll
        for (int i = 0; i < Lay::NV; ++i)
#pragma unroll
            for (int j = 0; j < Lay::V; j += 4) {
                const float2 a = v.pair[(i * Lay::V + j) / 2], b = v.pair[(i * Lay::V + j) / 2 + 1];
                if (lay.Has(i)) *reinterpret_cast<float4*>(p + lay.base + lay.Offset(i) + j) = make_float4(a.x, a.y, b.x, b.y);
            }
        return;
    }
#pragma unroll
    for (int i = 0; i < Lay::NV; ++i)
#pragma unroll
        for (int j = 0; j < Lay::V; ++j)
            if (lay.Has(i)) p[lay.base + lay.Offset(i) + j] = v.Get(i * Lay::V + j);
}
template <int E>
__device__ __forceinline__ float SumOf(const Held<E>& v) {
    float2 s = v.pair[0];
#pragma unroll
    for (int k = 1; k < Held<E>::kPairs; ++k) s = Add2(s, v.pair[k]);
    return s.x + s.y;
}
// ---- host side: how a row is cut
constexpr uint32_t kElements = 16;  // that a thread holds of a row
struct Cut {
    uint32_t nv;         // packs a thread
    uint32_t lanes, threads;
    bool stream;         // wider than a CTA holds
};
inline uint32_t PowerOfTwo(uint32_t n) {
    uint32_t p = 1;
    while (p < n) p <<= 1;
    return p;
}
// As few lanes a row as can hold it, which makes the reductions short, or more where the rows are too few to fill the chip's threads - far too
// few for more than a warp, whose lanes need no barrier (us, as few and more: forward 1 000 x 64 fp32 2.4, 1.8, 64 x 4 096 bf16 4.0, 2.6, but
// 2 000 x 224 fp32 to fp16 2.4, with two warps a row 3.7).
inline Cut CutRow(uint32_t rows, uint32_t cols, uint32_t v, uint32_t most_lanes, uint32_t elements = kElements) {
    const uint32_t packs = (cols - 1U) / v + 1U, most = elements / v;
    Cut c{1, 1, 256, false};
    if (packs > most * most_lanes) {
        c.stream = true;
        return c;
    }
    c.lanes = PowerOfTwo((packs - 1U) / most + 1U);
    if (v == 1U && c.lanes != 8U) c.lanes = c.lanes < 8U ? 8U : c.lanes < 32U ? 32U : c.lanes;  // stretches of 8 or 32 lanes
    while (c.lanes < 256U && c.lanes < packs && static_cast<uint64_t>(rows) * c.lanes < 148ULL * (c.lanes < 32U ? 512ULL : 128ULL)) c.lanes <<= 1;
    c.nv = (packs - 1U) / c.lanes + 1U;
    if (c.lanes > c.threads) c.threads = c.lanes;
    return c;
}
// Single columns: the layout with the fewest turns that hold a stretch, and with turns to mask for all numbers of columns that come to it.
template <class T>
struct Tag {
    using type = T;
};
template <class F>
inline mgt_status_t SingleColumns(const Cut& cut, F run) {
    if (cut.lanes < 32U) {
        if (cut.nv <= 2U) return run(Tag<Layout<1, 2, 8, 2>>{});
        if (cut.nv <= 4U) return run(Tag<Layout<1, 4, 8, 2>>{});
        if (cut.nv <= 8U) return run(Tag<Layout<1, 8, 8, 4>>{});
        return run(Tag<Layout<1, 16, 8, 8>>{});
    }
    if (cut.nv <= 2U) return run(Tag<Layout<1, 2, 32, 2>>{});
    if (cut.nv <= 4U) return run(Tag<Layout<1, 4, 32, 2>>{});
    if (cut.nv <= 6U) return run(Tag<Layout<1, 6, 32, 2>>{});
    if (cut.nv <= 8U) return run(Tag<Layout<1, 8, 32, 2>>{});
    if (cut.nv <= 10U) return run(Tag<Layout<1, 10, 32, 2>>{});
    if (cut.nv <= 12U) return run(Tag<Layout<1, 12, 32, 2>>{});
    return run(Tag<Layout<1, 16, 32, 4>>{});
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

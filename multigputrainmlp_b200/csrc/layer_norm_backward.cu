// Layer normalisation, backward. With xhat = (x - mean) * rstd and g = dy * gamma:
//   dx = rstd * (g - mean_c(g) - xhat * mean_c(g * xhat)),  dgamma = sum_r dy * xhat,  dbeta = sum_r dy,  dbias = sum_r dx
// One pass over dy and x: a thread keeps the columns that it owns for all rows of its CTA, so the column sums stay in its registers and
// leave once a CTA, as a row of partial sums that a second, small kernel adds up in a fixed order.
#include "layer_norm.cuh"

namespace mgt {
namespace ln {
namespace {

constexpr uint32_t kSums = 3, kMostLanes = 512;
constexpr uint32_t kSms = 148, kMostCtas = 2 * kSms;  // partial rows at most: two CTAs an SM
constexpr uint32_t kColumnSlices = 37;  // widest rows: slices of the batch that the column sums are taken over

inline __host__ __device__ uint32_t PartialPitch(uint32_t cols) { return (cols + 3U) / 4U * 4U; }

// What a kernel is made of: packs of a thread, threads, rows on their way, CTAs an SM. kPair: a cluster of two CTAs has a row, half of
// its columns each, and adds up the two sums of it through each other's shared memory.
template <class Tdy, class Tx, class Lay_, int kThreads_, bool kPair_ = false>
struct Form {
    using Lay = Lay_;
    static constexpr bool kPair = kPair_;
    static constexpr int V = Lay::V, kThreads = kThreads_, E = Lay::E;
    static constexpr int kBytes = E * (sizeof(Tdy) + sizeof(Tx)) * kThreads;  // of a row of every group
    // no more than it takes (us, with 2 and 3 of 16 KB and more: 53 248 x 224 fp32 29.7, 30.1; 20 000 x 1 024 46.5, 48.3; with 2, 3 and 6 of 12 KB: 100 000 x 384
    // bf16 49.1, 49.2, 50.9)
    static constexpr int kDepth = V == 1 || kBytes >= (12 << 10) ? 2 : 3;
    static constexpr int kCtas = kThreads > 256 ? 1 : 2;
    using RingDy = Ring<Tdy, Lay, kThreads, kDepth>;
    using RingX = Ring<Tx, Lay, kThreads, kDepth>;
    static constexpr uint32_t kGammaBytes = E * kThreads * 4U;
};

// Adds the other CTA's sums of the row that the cluster is at, in the order of the CTAs. Two places take turns: who writes one again has
// passed the barrier behind the other, and with it this CTA's reading of the first. (A CTA leaves after the barrier of its last row,
// behind which nothing is written to it.)
__device__ __forceinline__ void AddOther(float2& place, float (&s)[2]) {
    const uint32_t rank = blockIdx.x & 1U;
    if (threadIdx.x == 0U) {
        uint32_t there;
        asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(&place))), "r"(rank ^ 1U));
        asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(there), "f"(s[0]), "f"(s[1]) : "memory");
    }
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    const volatile float2& got = place;
    const float2 other = make_float2(got.x, got.y);
    s[0] = rank == 0U ? s[0] + other.x : other.x + s[0];
    s[1] = rank == 0U ? s[1] + other.y : other.y + s[1];
}

template <class Tdy, class Tx, class Tdx, class F>
__global__ void __launch_bounds__(F::kThreads, F::kCtas)
BackwardKernel(const Backward a) {
    extern __shared__ __align__(16) char memory[];  // gamma, the rings; at the end [groups][cols] sums, where there is more than one group
    using Lay = typename F::Lay;
    constexpr int V = F::V, E = F::E, D = F::kDepth, kThreads = F::kThreads, kPairs = Held<E>::kPairs;
    __shared__ float buffer[2 * 2 * (kThreads / 32)];
    Group g = MakeGroup(a.lanes, buffer);
    const uint32_t cta = F::kPair ? blockIdx.x / 2U : blockIdx.x, ctas = F::kPair ? gridDim.x / 2U : gridDim.x;
    const uint32_t half = ((a.cols - 1U) / V + 2U) / 2U * V, begin = F::kPair && (blockIdx.x & 1U) != 0U ? half : 0U;  // the first column, and how many
    const Lay lay(g, !F::kPair ? a.cols : begin != 0U ? a.cols - half : half);
    const Share share = MakeShare(g, a.rows, cta, ctas);
    typename F::RingDy ring_dy(static_cast<const Tdy*>(a.dy) + begin, a.dy_pitch, a.rows, memory + F::kGammaBytes, share, lay);
    typename F::RingX ring_x(static_cast<const Tx*>(a.x) + begin, a.x_pitch, a.rows, memory + F::kGammaBytes + F::RingDy::kBytes, share, lay);
    const float per_col = 1.0f / static_cast<float>(a.cols);
    Tdx* dx = static_cast<Tdx*>(a.dx) + share.first * a.dx_pitch + begin + lay.base;
    const uint64_t dx_step = share.stride * a.dx_pitch;
    ring_dy.Clear(lay);
    ring_x.Clear(lay);
    if constexpr (F::kPair) {  // (both are there to be written to)
        __syncwarp();
        asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
    }
    dependent_begin();
#pragma unroll
    for (int d = 0; d < D; ++d) {
        ring_dy.Fetch(lay, d, d < share.mine);
        ring_x.Fetch(lay, d, d < share.mine);
        CopiesEnd();
    }
    float next_mean, next_rstd;
    auto load_statistics = [&](uint32_t t) {  // (a row that is not there adds nothing to the sums)
        const uint32_t row = share.first + t * share.stride;
        next_mean = t < share.mine ? a.mean[row] : 0.0f;
        next_rstd = t < share.mine ? a.rstd[row] : 0.0f;
    };
    load_statistics(0);
    float2* gamma_at = reinterpret_cast<float2*>(memory) + threadIdx.x;  // this thread's columns: in registers they would spill beside the sums
    Held<E> gy, xhat, sums[kSums];
    LoadColumns(xhat, lay, a.gamma != nullptr ? a.gamma + begin : nullptr, 1.0f);
#pragma unroll
    for (int k = 0; k < kPairs; ++k) gamma_at[k * kThreads] = xhat.pair[k];
#pragma unroll
    for (uint32_t n = 0; n < kSums; ++n)
#pragma unroll
        for (int k = 0; k < kPairs; ++k) sums[n].pair[k] = Both(0.0f);
    __shared__ float2 pair_sums[2];
    uint32_t slot = 0;
    for (uint32_t t = 0; t < share.turns; ++t) {
        const bool in = t < share.mine;
        const float2 less = Both(-next_mean), rstd = Both(next_rstd);
        load_statistics(t + 1U);
        CopiesWait<D - 1>();
        if (V == 1) __syncwarp();  // (what the other lanes copied is here, too)
        ring_dy.Read(gy, lay, slot, in);
        ring_x.Read(xhat, lay, slot, in);
        float2 s1 = Both(0.0f), s2 = Both(0.0f);
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {  // (beyond the row's end dy is zero, and with it all that xhat enters: so that has to be a number)
            xhat.pair[k] = Mul2(Add2(xhat.pair[k], lay.HasPair(k, less)), rstd);
            sums[0].pair[k] = Fma2(gy.pair[k], xhat.pair[k], sums[0].pair[k]);
            sums[1].pair[k] = Add2(gy.pair[k], sums[1].pair[k]);
            gy.pair[k] = Mul2(gy.pair[k], gamma_at[k * kThreads]);
            s1 = Add2(s1, gy.pair[k]);
            s2 = Fma2(gy.pair[k], xhat.pair[k], s2);
        }
        float s[2] = {s1.x + s1.y, s2.x + s2.y};
        Reduce(g, s);
        if constexpr (F::kPair) AddOther(pair_sums[t & 1U], s);
        if (V == 1) __syncwarp();  // (everybody has what it read of the slot: the sums needed it)
        ring_dy.Fetch(lay, slot, t + D < share.mine);
        ring_x.Fetch(lay, slot, t + D < share.mine);
        CopiesEnd();
        slot = slot + 1U == D ? 0U : slot + 1U;
        if (in) {
            const float2 c1 = Both(-s[0] * per_col), c2 = Both(-s[1] * per_col);
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                gy.pair[k] = Mul2(rstd, Fma2(xhat.pair[k], c2, Add2(gy.pair[k], c1)));  // (rstd last: it is large where the differences are small)
                sums[2].pair[k] = Add2(gy.pair[k], sums[2].pair[k]);  // (before it is rounded to dx's type; beyond the row's end nobody looks)
            }
            lay.Each([&](int i, bool has) {
                if (has) StorePack<Tdx, V>(dx + lay.Offset(i), PackOf<Tdx, V>(gy, i));
            });
        }
        dx += dx_step;
    }
    CopiesWait<0>();
    float* lanes_sums = reinterpret_cast<float*>(memory);
    __syncthreads();  // (the rings are no longer read)
    // this CTA's column sums: the groups of a warp by shuffles, then the warps (or the groups of several) in order
    for (uint32_t o = g.lanes; o < 32U; o <<= 1)
#pragma unroll
        for (uint32_t n = 0; n < kSums; ++n)
#pragma unroll
            for (int k = 0; k < kPairs; ++k) {
                const float2 v = sums[n].pair[k];
                sums[n].pair[k] = Add2(v, make_float2(__shfl_xor_sync(0xffffffffU, v.x, o), __shfl_xor_sync(0xffffffffU, v.y, o)));
            }
    const uint32_t pitch = PartialPitch(a.cols), teams = kThreads / max(g.lanes, 32U), team = threadIdx.x / max(g.lanes, 32U);
    const bool speaks = g.lanes >= 32U || (threadIdx.x & 31U) < g.lanes;
    float* partial = a.partial + static_cast<uint64_t>(cta) * kSums * pitch;
#pragma unroll
    for (uint32_t k = 0; k < kSums; ++k) {
        if (a.sums[k] == nullptr) continue;
        float* to = (ctas > 1U ? partial + k * pitch : a.sums[k]) + begin;
        if (speaks) StoreColumns(teams > 1U ? lanes_sums + team * pitch : to, sums[k], lay);
        if (teams > 1U) {
            __syncthreads();
            for (uint32_t c = threadIdx.x; c < a.cols; c += kThreads) {
                float s = 0.0f;
                for (uint32_t l = 0; l < teams; ++l) s += lanes_sums[l * pitch + c];
                to[c] = s;
            }
            __syncthreads();
        }
    }
}

// sums[k][c] = the partial rows' values added up: 32 threads share four neighbouring columns, each adds every 32nd row in order (ten at
// most, all on their way at once), and the 32 then in order. Rows of partial sums are whole quads apart; what lies behind the last column is read and not used.
constexpr uint32_t kSumQuads = 8, kSumParts = 32;
__global__ void __launch_bounds__(kSumQuads * kSumParts)
SumPartialRowsKernel(const Backward a, uint32_t rows, uint32_t pitch) {
    __shared__ float4 part_sums[kSumParts][kSumQuads];
    const uint32_t q = threadIdx.x % kSumQuads, part = threadIdx.x / kSumQuads, quad = blockIdx.x * kSumQuads + q;
    dependent_begin();
    float* to = a.sums[blockIdx.y];
    if (to == nullptr) return;
    float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (quad * 4U < a.cols) {
        const float4* from = reinterpret_cast<const float4*>(a.partial + blockIdx.y * pitch) + quad;
        const uint64_t step = kSums * (pitch / 4U);
        float4 v[(kMostCtas + kSumParts - 1U) / kSumParts];
#pragma unroll
        for (uint32_t i = 0; i < sizeof(v) / sizeof(v[0]); ++i) {
            const uint32_t r = part + i * kSumParts;
            v[i] = r < rows ? from[r * step] : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
#pragma unroll
        for (uint32_t i = 0; i < sizeof(v) / sizeof(v[0]); ++i) {
            s.x += v[i].x; s.y += v[i].y; s.z += v[i].z; s.w += v[i].w;
        }
    }
    part_sums[part][q] = s;
    __syncthreads();
    const uint32_t col = blockIdx.x * kSumQuads * 4U + threadIdx.x;
    if (threadIdx.x < kSumQuads * 4U && col < a.cols) {
        float total = 0.0f;
#pragma unroll
        for (uint32_t p = 0; p < kSumParts; ++p) total += reinterpret_cast<const float*>(part_sums[p])[threadIdx.x];
        to[col] = total;
    }
}
// Rows wider than the registers of a CTA. First the two means of every row, left in `means` ...
template <class Tdy, class Tx, int V>
__global__ void __launch_bounds__(1024)
StreamMeansKernel(const Backward a, float2* means) {
    __shared__ float buffer[2 * 2 * 32];
    Group g = MakeGroup(blockDim.x, buffer);
    const float cols = static_cast<float>(a.cols);
    const uint32_t step = blockDim.x * V;
    dependent_begin();
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const Tdy* dy = static_cast<const Tdy*>(a.dy) + row * a.dy_pitch;
        const Tx* x = static_cast<const Tx*>(a.x) + row * a.x_pitch;
        const float mean = a.mean[row], rstd = a.rstd[row];
        float s[2] = {0.0f, 0.0f};
#pragma unroll 2
        for (uint32_t c = threadIdx.x * V; c < a.cols; c += step) {
            const Pack<Tdy, V> pd = LoadPack<Tdy, V>(dy + c);
            const Pack<Tx, V> px = LoadPack<Tx, V>(x + c);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float t = ToFloat(pd.v[j]) * (a.gamma != nullptr ? a.gamma[c + j] : 1.0f);
                s[0] += t;
                s[1] += t * ((ToFloat(px.v[j]) - mean) * rstd);
            }
        }
        Reduce(g, s);
        if (threadIdx.x == 0U) means[row] = make_float2(s[0] / cols, s[1] / cols);
    }
}
// ... then, a tile of columns and a slice of the rows at a time, dx and the column sums.
template <class Tdy, class Tx, class Tdx, int V>
__global__ void __launch_bounds__(256)
StreamColumnsKernel(const Backward a, const float2* means, uint32_t rows_each) {
    const uint32_t c = (blockIdx.x * 256U + threadIdx.x) * V;
    dependent_begin();
    if (c >= a.cols) return;
    const uint64_t r0 = static_cast<uint64_t>(blockIdx.y) * rows_each, r1 = min(static_cast<uint64_t>(a.rows), r0 + rows_each);
    float gamma[V], sums[kSums][V] = {};
#pragma unroll
    for (int j = 0; j < V; ++j) gamma[j] = a.gamma != nullptr ? a.gamma[c + j] : 1.0f;
    // four rows at once: the compiler keeps a load behind the store before it (dx may be dy or x)
    for (uint64_t first = r0; first < r1; first += 4U) {
        Pack<Tdy, V> pd[4];
        Pack<Tx, V> px[4];
        float mean[4], rstd[4];
        float2 m[4];
#pragma unroll
        for (uint32_t i = 0; i < 4U; ++i) {
            const uint64_t row = first + i;
            if (row >= r1) continue;
            pd[i] = LoadPack<Tdy, V>(static_cast<const Tdy*>(a.dy) + row * a.dy_pitch + c);
            px[i] = LoadPack<Tx, V>(static_cast<const Tx*>(a.x) + row * a.x_pitch + c);
            mean[i] = a.mean[row];
            rstd[i] = a.rstd[row];
            m[i] = means[row];
        }
#pragma unroll
        for (uint32_t i = 0; i < 4U; ++i) {
            const uint64_t row = first + i;
            if (row >= r1) continue;
            Pack<Tdx, V> out;
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = ToFloat(pd[i].v[j]), xhat = (ToFloat(px[i].v[j]) - mean[i]) * rstd[i], o = rstd[i] * (d * gamma[j] - m[i].x - xhat * m[i].y);
                sums[0][j] += d * xhat;
                sums[1][j] += d;
                sums[2][j] += o;
                out.v[j] = FromFloat<Tdx>(o);
            }
            StorePack<Tdx, V>(static_cast<Tdx*>(a.dx) + row * a.dx_pitch + c, out);
        }
    }
    const uint32_t pitch = PartialPitch(a.cols);
    float* partial = a.partial + static_cast<uint64_t>(blockIdx.y) * kSums * pitch;
#pragma unroll
    for (uint32_t k = 0; k < kSums; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) partial[k * pitch + c + j] = sums[k][j];
}

void SumPartialRows(const Backward& a, uint32_t rows, LaunchOn on, uint32_t* launches) {
    Launch(SumPartialRowsKernel, dim3((a.cols + 4U * kSumQuads - 1U) / (4U * kSumQuads), kSums), kSumQuads * kSumParts, 0, LaunchOn(on.stream, true), a, rows, PartialPitch(a.cols));
    ++*launches;
}

template <class Tdy, class Tx, class Tdx, class F>
mgt_status_t Run(Backward a, const Cut& cut, LaunchOn on, uint32_t* launches) {
    const uint32_t groups = cut.threads / cut.lanes;
    const uint64_t want = (static_cast<uint64_t>(a.rows) + groups - 1U) / groups;
    // One CTA an SM where two would not have four rows each for every group: half as many partial rows (us, with two and one: 20 000 x 64 bf16
    // 9.1, 7.9; 5 000 x 512 bf16 11.0, 9.3; 1 000 x 2 048 bf16 13.8, 10.7)
    const uint32_t full = kSms * F::kCtas / (F::kPair ? 2U : 1U), most = want < 4ULL * full && full > kSms ? kSms : full;
    const uint32_t ctas = static_cast<uint32_t>(want < most ? want : most);
    a.lanes = cut.lanes;
    constexpr uint32_t smem = F::kGammaBytes + F::RingDy::kBytes + F::RingX::kBytes;
    static_assert(smem >= F::E * F::kThreads * 4U + F::kThreads / 8U * 4U, "the sums of all warps or groups, a float a column of each");
    static std::atomic<uint64_t> allowed{0};
    if (!AllowShared(BackwardKernel<Tdy, Tx, Tdx, F>, allowed, smem)) return MGT_CUDA_FAILURE;
    if constexpr (F::kPair) LaunchClusters(2U, BackwardKernel<Tdy, Tx, Tdx, F>, 2U * ctas, cut.threads, smem, on, a);
    else Launch(BackwardKernel<Tdy, Tx, Tdx, F>, ctas, cut.threads, smem, on, a);
    ++*launches;
    if (ctas > 1U && (a.sums[0] != nullptr || a.sums[1] != nullptr || a.sums[2] != nullptr)) SumPartialRows(a, ctas, on, launches);
    return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
}
template <class Tdy, class Tx, class Tdx, int V>
mgt_status_t RunByWidth(const Backward& a, LaunchOn on, uint32_t* launches) {
    Cut cut = CutRow(a.rows, a.cols, V, 2U * kMostLanes);
    if (cut.stream) {
        float2* means = reinterpret_cast<float2*>(a.partial + static_cast<uint64_t>(kColumnSlices) * kSums * PartialPitch(a.cols));
        Launch(StreamMeansKernel<Tdy, Tx, V>, a.rows < 2U * kSms ? a.rows : 2U * kSms, 1024, 0, on, a, means);
        const uint32_t slices = a.rows < kColumnSlices ? a.rows : kColumnSlices, rows_each = (a.rows - 1U) / slices + 1U;
        const uint32_t used = (a.rows - 1U) / rows_each + 1U;
        Launch(StreamColumnsKernel<Tdy, Tx, Tdx, V>, dim3((a.cols - 1U) / (256U * V) + 1U, used), 256, 0, LaunchOn(on.stream, true), a, static_cast<const float2*>(means), rows_each);
        *launches += 2;
        SumPartialRows(a, used, on, launches);
        return cudaGetLastError() == cudaSuccess ? MGT_OK : MGT_CUDA_FAILURE;
    }
    // (packs that a kernel has room for and the row does not have lie beyond its end)
    constexpr int kMost = kElements / V;
    // twelve columns a thread where they do (us, with sixteen and with twelve: 8 000 x 5 001 fp32 157, 98; 4 000 x 10 001 bf16 148, 124; 4 000 x 9 000 bf16
    // 109, 100); rows of a 512-thread CTA by two CTAs of half as many columns a thread are slower (7 000 x 8 192 bf16 77.5, 147)
    if (cut.threads > kMostLanes) {
        cut.threads = cut.lanes = kMostLanes;  // of each of two CTAs
        if constexpr (V == 4)
            if (cut.nv == 3) return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, 3, 32, 0>, 512, true>>(a, cut, on, launches);
        if constexpr (V == 1)
            if (cut.nv <= 12U) return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<1, 12, 32, 4>, 512, true>>(a, cut, on, launches);
        return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, kMost, 32, V == 1 ? 4 : 0>, 512, true>>(a, cut, on, launches);
    }
    if (cut.threads > 256U) {
        if constexpr (V == 4)
            if (cut.nv == 3) return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, 3, 32, 0>, 512>>(a, cut, on, launches);
        if constexpr (V == 1)
            if (cut.nv <= 12U) return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<1, 12, 32, 4>, 512>>(a, cut, on, launches);
        return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, kMost, 32, V == 1 ? 4 : 0>, 512>>(a, cut, on, launches);
    }
    if constexpr (V == 1) {
        return SingleColumns(cut, [&](auto tag) { return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, typename decltype(tag)::type, 256>>(a, cut, on, launches); });
    } else {
        constexpr int kFew = V == 4 ? 2 : 1;
        if (cut.nv <= kFew) return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, kFew, 32, 0>, 256>>(a, cut, on, launches);
        if constexpr (V == 4)
            if (cut.nv == 3) return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, 3, 32, 0>, 256>>(a, cut, on, launches);
        return Run<Tdy, Tx, Tdx, Form<Tdy, Tx, Layout<V, kMost, 32, 0>, 256>>(a, cut, on, launches);
    }
}
template <class Tdy, class Tx, class Tdx>
mgt_status_t RunTyped(const Backward& a, int32_t dy_type, int32_t x_type, int32_t dx_type, LaunchOn on, uint32_t* launches) {
    auto whole = [&](int v) {
        return a.cols % v == 0 && RowsAligned(a.dy, a.dy_pitch, a.rows, dy_type, v) && RowsAligned(a.x, a.x_pitch, a.rows, x_type, v) &&
               RowsAligned(a.dx, a.dx_pitch, a.rows, dx_type, v);
    };
    if constexpr (sizeof(Tdy) == 2 && sizeof(Tx) == 2 && sizeof(Tdx) == 2)
        if (whole(8)) {  // three packs of four columns where two of eight leave more places empty (us, as eights and as fours: 20 001 x 2 056 bf16 84.8, 79.8)
            const Cut fours = CutRow(a.rows, a.cols, 4, 2U * kMostLanes);
            if (fours.stream || fours.nv != 3) return RunByWidth<Tdy, Tx, Tdx, 8>(a, on, launches);
        }
    if (whole(4)) return RunByWidth<Tdy, Tx, Tdx, 4>(a, on, launches);
    return RunByWidth<Tdy, Tx, Tdx, 1>(a, on, launches);
}

}  // namespace

uint64_t BackwardFloats(uint32_t rows, uint32_t cols) {
    const bool stream = cols > 2U * kElements * kMostLanes;  // (from there on whatever the packs are)
    return static_cast<uint64_t>(stream ? kColumnSlices : kMostCtas) * kSums * PartialPitch(cols) + (stream ? 2ULL * rows : 0ULL) + 4ULL;
}

mgt_status_t LaunchBackward(Backward a, int32_t dy_type, int32_t x_type, int32_t dx_type, LaunchOn on, uint32_t* launches) {
    auto is = [&](int32_t dy, int32_t x, int32_t dx) { return dy_type == dy && x_type == x && dx_type == dx; };
    using H = __half;
    using B = __nv_bfloat16;
    if (is(MGT_F32, MGT_F32, MGT_F32)) return RunTyped<float, float, float>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_F32, MGT_F32, MGT_F16)) return RunTyped<float, float, H>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_F32, MGT_F32, MGT_BF16)) return RunTyped<float, float, B>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_F16, MGT_F32, MGT_F32)) return RunTyped<H, float, float>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_BF16, MGT_F32, MGT_F32)) return RunTyped<B, float, float>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_F16, MGT_F16, MGT_F16)) return RunTyped<H, H, H>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_F32, MGT_F16, MGT_F16)) return RunTyped<float, H, H>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_BF16, MGT_BF16, MGT_BF16)) return RunTyped<B, B, B>(a, dy_type, x_type, dx_type, on, launches);
    if (is(MGT_F32, MGT_BF16, MGT_BF16)) return RunTyped<float, B, B>(a, dy_type, x_type, dx_type, on, launches);
    return MGT_INVALID_CONFIG;
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
    a.partial = reinterpret_cast<float*>((reinterpret_cast<uintptr_t>(workspace) + 15U) & ~static_cast<uintptr_t>(15));
    a.dy_pitch = c->y_pitch != 0 ? c->y_pitch : c->cols;
    a.x_pitch = c->x_pitch != 0 ? c->x_pitch : c->cols;
    a.dx_pitch = c->dx_pitch != 0 ? c->dx_pitch : c->cols;
    a.rows = c->rows; a.cols = c->cols;
    uint32_t launches = 0;
    return mgt::ln::LaunchBackward(a, c->y_type, c->x_type, c->dx_type, {s, true}, &launches);
}

}  // extern "C"

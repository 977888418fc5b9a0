// Balance of the experts: how often each was chosen, and the load-balance loss
//   loss = E sum_e f_e s_e,  f_e = count_e / (n H k),  s_e = (sum of the gates on e) / (n H),
// over n tokens, H heads and k choices.  The sum over experts is a sum over the chosen pairs,
//   loss = E / (n H k n H) sum_p count[id_p] gate_p,
// so no per-expert gate sum is formed (its additions would need an order), and the gradient of a
// gate is count[id_p] times the same factor (the counts themselves have none).
//
// The counts are sums of ones, so the order of their atomics does not show.  They are taken in LDS:
// a workgroup counts the ids of one range of kRange experts in one slice of the pairs, and a second
// kernel adds the slices (none for up to kOneSlice pairs).  Each id is read once per range, from L2.
// Counting in memory takes a zero fill and an atomic per pair: 524,288 pairs over 262,144 experts
// 40 us against 20 here, 16,000 skewed pairs over 4,096 (2,000 on one expert, whose atomics wait for one
// another) 24 against 5; it is kept for more than kMaxRanges ranges, where reading the ids that often would
// cost more.
#include "ethos_common.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr int kRange = 16384;      // experts whose counters a workgroup holds in LDS (64 KB)
constexpr int kMaxRanges = 32;
constexpr int kMaxSlices = 16;
constexpr int64_t kOneSlice = 16384;
constexpr int kSumBlocks = 512;    // partial sums of the loss

template <typename I>
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t p) {
    return (int64_t)((const I*)ids)[p];
}

// Workgroup (range, slice): counts of the range's ids in the slice, to out[slice][n_experts].
template <typename I>
__global__ __launch_bounds__(1024) void count_range_kernel(const void* __restrict__ ids, int64_t pairs, int64_t n_experts, int slices,
                                                           int32_t* __restrict__ out, int32_t* __restrict__ ticket) {
    __shared__ int32_t count[kRange];
    const int range = blockIdx.x / slices, slice = blockIdx.x % slices;
    const int64_t e0 = (int64_t)range * kRange;
    const int size = (int)(n_experts - e0 < kRange ? n_experts - e0 : kRange);
    if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
    for (int i = threadIdx.x; i < size; i += 1024) count[i] = 0;
    __syncthreads();
    const int64_t per = (pairs + slices - 1) / slices, p1 = per * (slice + 1) < pairs ? per * (slice + 1) : pairs;
    int64_t p = per * slice + threadIdx.x;
    for (; p + 3 * 1024 < p1; p += 4 * 1024) {
        int64_t e[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) e[j] = id_at<I>(ids, p + j * 1024) - e0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (e[j] >= 0 && e[j] < size) atomicAdd(count + e[j], 1);
    }
    for (; p < p1; p += 1024) {
        const int64_t e = id_at<I>(ids, p) - e0;
        if (e >= 0 && e < size) atomicAdd(count + e, 1);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < size; i += 1024) out[slice * n_experts + e0 + i] = count[i];
}

__global__ __launch_bounds__(256) void count_slices_kernel(const int32_t* __restrict__ part, int slices, int64_t n,
                                                           int32_t* __restrict__ counts) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        int32_t v[kMaxSlices], s = 0;
#pragma unroll
        for (int j = 0; j < kMaxSlices; ++j) v[j] = part[(j < slices ? j : 0) * n + i];
#pragma unroll
        for (int j = 0; j < kMaxSlices; ++j) s += j < slices ? v[j] : 0;
        counts[i] = s;
    }
}

__global__ __launch_bounds__(256) void count_zero_kernel(int32_t* __restrict__ counts, int64_t n, int32_t* __restrict__ ticket) {
    if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) counts[i] = 0;
}

template <typename I>
__global__ __launch_bounds__(256) void count_kernel(const void* __restrict__ ids, int64_t pairs, int64_t n_experts,
                                                    int32_t* __restrict__ counts) {
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < pairs; p += (int64_t)gridDim.x * 256) {
        const int64_t e = id_at<I>(ids, p);
        if (e >= 0 && e < n_experts) atomicAdd(counts + e, 1);
    }
}

__device__ __forceinline__ double block_sum(double v, double* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if (lane == 0) lds[wave] = v;
    __syncthreads();
    double s = 0.0;
    for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += lds[i];
    return s;
}

// The loss: each workgroup's part of the sum, then, in the one that finishes last, all of them in
// their order (`ticket` counts the finished ones and is zero on entry).
template <typename I, typename T>
__global__ __launch_bounds__(256) void balance_sum_kernel(const T* __restrict__ gates, const void* __restrict__ ids, int64_t pairs,
                                                          int64_t n_experts, const int32_t* __restrict__ counts, double scale,
                                                          double* part, int32_t* ticket, float* __restrict__ loss) {
    __shared__ double lds[4];
    __shared__ bool last;
    double s = 0.0;
    const int64_t step = (int64_t)gridDim.x * 256;
    int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
    for (; p + 3 * step < pairs; p += 4 * step) {
        int64_t e[4];
        int32_t c[4];
        float g[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            e[j] = id_at<I>(ids, p + j * step);
            g[j] = Elem<T>::to_f32(gates[p + j * step]);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) c[j] = counts[e[j] >= 0 && e[j] < n_experts ? e[j] : 0];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (e[j] >= 0 && e[j] < n_experts) s = __builtin_fma((double)c[j], (double)g[j], s);
    }
    for (; p < pairs; p += step) {
        const int64_t e = id_at<I>(ids, p);
        if (e >= 0 && e < n_experts) s = __builtin_fma((double)counts[e], (double)Elem<T>::to_f32(gates[p]), s);
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) {
        __hip_atomic_store(part + blockIdx.x, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)gridDim.x - 1;
    }
    __syncthreads();
    if (!last) return;
    s = 0.0;
    for (int i = threadIdx.x; i < (int)gridDim.x; i += 256) s += __hip_atomic_load(part + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    s = block_sum(s, lds);
    if (threadIdx.x == 0) *loss = (float)(s * scale);
}

template <typename I, typename T>
__global__ __launch_bounds__(256) void balance_grad_kernel(const void* __restrict__ ids, const int32_t* __restrict__ counts,
                                                           const float* __restrict__ dloss, int64_t pairs, int64_t n_experts,
                                                           double scale, T* __restrict__ dgates) {
    const double k = scale * (double)*dloss;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < pairs; p += (int64_t)gridDim.x * 256) {
        const int64_t e = id_at<I>(ids, p);
        const int32_t c = e >= 0 && e < n_experts ? counts[e] : 0;
        dgates[p] = Elem<T>::from_f32((float)(k * (double)c));
    }
}

int blocks_for(int64_t items, int64_t most) {
    const int64_t b = (items + 255) / 256;
    return (int)(b < 1 ? 1 : b > most ? most : b);
}

struct BalanceWs {
    int32_t* ticket;
    double* part;
    int32_t* slices;
    int ranges, n_slices;  // ranges 0: counting in memory
    size_t bytes;
};
BalanceWs balance_ws(char* p, int64_t pairs, int64_t n_experts) {
    BalanceWs w;
    w.ticket = (int32_t*)p;
    w.part = (double*)(p + 256);
    w.bytes = 256 + kSumBlocks * sizeof(double);
    w.slices = (int32_t*)(p + w.bytes);
    const int64_t ranges = (n_experts + kRange - 1) / kRange;
    w.ranges = ranges <= kMaxRanges ? (int)ranges : 0;
    w.n_slices = 1;
    if (w.ranges > 0 && pairs > kOneSlice) {
        // about one workgroup per CU, of at least 2,048 pairs
        int64_t s = 256 / ranges;
        s = s < pairs / 2048 ? s : pairs / 2048;
        w.n_slices = (int)(s < 2 ? 2 : s > kMaxSlices ? kMaxSlices : s);
        w.bytes += (size_t)w.n_slices * n_experts * 4;
    }
    return w;
}

}  // namespace

size_t balance_workspace_bytes(int64_t pairs, int64_t n_experts) { return balance_ws(nullptr, pairs, n_experts).bytes; }

int launch_balance(const void* gates, const void* ids, int ids_64, int64_t pairs, int64_t n_experts, double scale, int dtype,
                   void* ws, int32_t* counts, float* loss, int num_cus, hipStream_t stream) {
    const BalanceWs w = balance_ws((char*)ws, pairs, n_experts);
    if (w.ranges > 0) {
        int32_t* out = w.n_slices > 1 ? w.slices : counts;
        const dim3 grid((unsigned)(w.ranges * w.n_slices));
        if (ids_64)
            hipLaunchKernelGGL((count_range_kernel<int64_t>), grid, dim3(1024), 0, stream, ids, pairs, n_experts, w.n_slices, out, w.ticket);
        else
            hipLaunchKernelGGL((count_range_kernel<int32_t>), grid, dim3(1024), 0, stream, ids, pairs, n_experts, w.n_slices, out, w.ticket);
        if (w.n_slices > 1)
            hipLaunchKernelGGL(count_slices_kernel, dim3(blocks_for(n_experts, num_cus * 8)), dim3(256), 0, stream, w.slices, w.n_slices,
                               n_experts, counts);
    } else {
        hipLaunchKernelGGL(count_zero_kernel, dim3(blocks_for(n_experts, num_cus * 8)), dim3(256), 0, stream, counts, n_experts, w.ticket);
        const dim3 grid(blocks_for(pairs, num_cus * 8));
        if (ids_64) hipLaunchKernelGGL((count_kernel<int64_t>), grid, dim3(256), 0, stream, ids, pairs, n_experts, counts);
        else hipLaunchKernelGGL((count_kernel<int32_t>), grid, dim3(256), 0, stream, ids, pairs, n_experts, counts);
    }
    const dim3 grid(blocks_for(pairs, kSumBlocks));
#define ETHOS_SUM(I, T)                                                                                                            \
    hipLaunchKernelGGL((balance_sum_kernel<I, T>), grid, dim3(256), 0, stream, (const T*)gates, ids, pairs, n_experts, counts, scale, \
                       w.part, w.ticket, loss)
    if (dtype == kBF16) {
        if (ids_64) ETHOS_SUM(int64_t, uint16_t);
        else ETHOS_SUM(int32_t, uint16_t);
    } else {
        if (ids_64) ETHOS_SUM(int64_t, float);
        else ETHOS_SUM(int32_t, float);
    }
#undef ETHOS_SUM
    return (int)hipGetLastError();
}

int launch_balance_grad(const void* ids, int ids_64, const int32_t* counts, const float* dloss, int64_t pairs, int64_t n_experts,
                        double scale, int dtype, void* dgates, int num_cus, hipStream_t stream) {
    const dim3 grid(blocks_for(pairs, num_cus * 8));
#define ETHOS_GRAD(I, T)                                                                                                        \
    hipLaunchKernelGGL((balance_grad_kernel<I, T>), grid, dim3(256), 0, stream, ids, counts, dloss, pairs, n_experts, scale, (T*)dgates)
    if (dtype == kBF16) {
        if (ids_64) ETHOS_GRAD(int64_t, uint16_t);
        else ETHOS_GRAD(int32_t, uint16_t);
    } else {
        if (ids_64) ETHOS_GRAD(int64_t, float);
        else ETHOS_GRAD(int32_t, float);
    }
#undef ETHOS_GRAD
    return (int)hipGetLastError();
}

}  // namespace ethos

// Balance of the experts: how often each was chosen, and the load-balance loss
//   loss = E sum_e f_e s_e,  f_e = count_e / (n H k),  s_e = (sum of the gates on e) / (n H),
// over n tokens, H heads and k choices.  The sum over experts is a sum over the chosen pairs,
//   loss = E / (n H k n H) sum_p count[id_p] gate_p,
// so no per-expert gate sum is formed (its additions would need an order), and the gradient of a
// gate is count[id_p] times the same factor (the counts themselves have none).  The counts are sums
// of ones: whole-number atomics, whose order does not show.
#include "ethos_common.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr int kSumBlocks = 1024;  // partial sums of the loss

template <typename I>
__device__ __forceinline__ int64_t id_at(const void* ids, int64_t p) {
    return (int64_t)((const I*)ids)[p];
}

__global__ __launch_bounds__(256) void count_zero_kernel(int32_t* __restrict__ counts, int64_t n) {
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

template <typename I, typename T>
__global__ __launch_bounds__(256) void balance_sum_kernel(const T* __restrict__ gates, const void* __restrict__ ids, int64_t pairs,
                                                          int64_t n_experts, const int32_t* __restrict__ counts,
                                                          double* __restrict__ part) {
    __shared__ double lds[4];
    double s = 0.0;
    for (int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x; p < pairs; p += (int64_t)gridDim.x * 256) {
        const int64_t e = id_at<I>(ids, p);
        if (e >= 0 && e < n_experts) s += (double)counts[e] * (double)Elem<T>::to_f32(gates[p]);
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) part[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void balance_total_kernel(const double* __restrict__ part, int n, double scale,
                                                            float* __restrict__ loss) {
    __shared__ double lds[4];
    double s = 0.0;
    for (int i = threadIdx.x; i < n; i += 256) s += part[i];
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

}  // namespace

size_t balance_workspace_bytes(int64_t) { return kSumBlocks * sizeof(double); }

int launch_balance(const void* gates, const void* ids, int ids_64, int64_t pairs, int64_t n_experts, double scale, int dtype,
                   void* ws, int32_t* counts, float* loss, int num_cus, hipStream_t stream) {
    hipLaunchKernelGGL(count_zero_kernel, dim3(blocks_for(n_experts, num_cus * 8)), dim3(256), 0, stream, counts, n_experts);
    const dim3 grid(blocks_for(pairs, num_cus * 8));
    if (ids_64) hipLaunchKernelGGL((count_kernel<int64_t>), grid, dim3(256), 0, stream, ids, pairs, n_experts, counts);
    else hipLaunchKernelGGL((count_kernel<int32_t>), grid, dim3(256), 0, stream, ids, pairs, n_experts, counts);
    const int nb = blocks_for(pairs, kSumBlocks);
    double* part = (double*)ws;
#define ETHOS_SUM(I, T)                                                                                                 \
    hipLaunchKernelGGL((balance_sum_kernel<I, T>), dim3(nb), dim3(256), 0, stream, (const T*)gates, ids, pairs, n_experts, counts, part)
    if (dtype == kBF16) {
        if (ids_64) ETHOS_SUM(int64_t, uint16_t);
        else ETHOS_SUM(int32_t, uint16_t);
    } else {
        if (ids_64) ETHOS_SUM(int64_t, float);
        else ETHOS_SUM(int32_t, float);
    }
#undef ETHOS_SUM
    hipLaunchKernelGGL(balance_total_kernel, dim3(1), dim3(256), 0, stream, part, nb, scale, loss);
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

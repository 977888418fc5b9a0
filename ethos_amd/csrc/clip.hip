// Global gradient norm over many tensors, and clipping:
//   total = (sum over every tensor's values of g^2)^(1/2), or max |g|;
//   out = RN_T(g min(1, max_norm / (total + 1e-6))).
// Two passes over the gradients with one workgroup per piece of kPiece values: the squares' sums
// (float64: no gradient's square overflows or vanishes there) in a fixed order, one small kernel
// for the norm and the factor, then the scaled copy, last pieces first (what the norm read last may still be
// in the caches).  Bound by memory: the gradients are read twice, as the norm comes before the first scaled value.
// 535 MB in 186 tensors take 267 us (norm 92, copy 175), 6.0 TB/s of 1.6 GB.  What was measured there: pieces of 8192,
// 16384, 24576 and 32768 values 325, 267, 279 and 289 us; with the last, copies that go into the caches 318 us (they push
// out what the next norm reads, and leave it their own writing back), and one load on its way in the copy 331.  The
// tensors' addresses travel as kernel arguments, as many as fit their 4 KiB: a launch and pass for up to 180 tensors.
#include "ethos_common.hpp"
#include "ethos_rows.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr int kPiece = 16384;
constexpr int kPerLaunch = 180;
constexpr uint16_t kFloatBit = 0x8000;

// A launch's tensors; `out` is what the scaled copies go to.
struct ClipList {
    const void* in[kPerLaunch];
    void* out[kPerLaunch];
    int32_t first[kPerLaunch];  // first piece of the tensor in this launch
    uint16_t tail[kPerLaunch];  // values of its last piece, less one; kFloatBit: float32
    int32_t count;
    int32_t pieces;  // of this launch
    int32_t base;    // pieces before this launch
};
static_assert(sizeof(ClipList) + 32 <= 4096, "kernel arguments");
static_assert(kPiece <= kFloatBit, "a tail's bits");

// The tensor that holds piece b: the last one whose first piece is not past it.
__device__ __forceinline__ int clip_find(const ClipList& l, int b) {
    int lo = 0, hi = l.count - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (l.first[mid] <= b) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}
// Values of piece b of tensor t.
__device__ __forceinline__ int clip_size(const ClipList& l, int t, int b) {
    const int end = t + 1 < l.count ? l.first[t + 1] : l.pieces;
    return b + 1 < end ? kPiece : (l.tail[t] & (kFloatBit - 1)) + 1;
}

template <typename T, typename F>
__device__ __forceinline__ void clip_values(const T* p, int n, F f) {
    constexpr int N = Vec16<T>::kN;
    if (((uintptr_t)p & 15u) == 0) {
        typedef typename Vec16<T>::raw Raw;
        const int whole = n / N;
        int i = threadIdx.x;
        for (; i + 7 * 256 < whole; i += 8 * 256) {  // eight loads on their way
            Raw r[8];
#pragma unroll
            for (int c = 0; c < 8; ++c) r[c] = reinterpret_cast<const Raw*>(p)[i + c * 256];
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                float v[N];
                Vec16<T>::unpack(r[c], v);
#pragma unroll
                for (int j = 0; j < N; ++j) f(v[j]);
            }
        }
        for (; i < whole; i += 256) {
            float v[N];
            Vec16<T>::unpack(reinterpret_cast<const Raw*>(p)[i], v);
#pragma unroll
            for (int j = 0; j < N; ++j) f(v[j]);
        }
        for (i = whole * N + threadIdx.x; i < n; i += 256) f(Elem<T>::to_f32(p[i]));
    } else {
        for (int i = threadIdx.x; i < n; i += 256) f(Elem<T>::to_f32(p[i]));
    }
}

// Larger of two magnitudes, NaN if one is.
__device__ __forceinline__ double nan_max(double a, double b) { return a != a ? a : b != b ? b : a > b ? a : b; }

template <bool INF>
__device__ __forceinline__ double clip_join(double a, double b) {
    return INF ? nan_max(a, b) : a + b;
}

template <bool INF>
__device__ __forceinline__ double clip_reduce(double v, double* lds) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = clip_join<INF>(v, __shfl_xor(v, o));
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    double s = lds[0];
    for (int i = 1; i < (int)(blockDim.x >> 6); ++i) s = clip_join<INF>(s, lds[i]);
    return s;
}

template <bool INF>
__global__ __launch_bounds__(256) void clip_norm_kernel(ClipList l, double* __restrict__ part) {
    __shared__ double lds[4];
    const int t = clip_find(l, blockIdx.x);
    const int64_t at = (int64_t)((int)blockIdx.x - l.first[t]) * kPiece;
    const bool f32 = (l.tail[t] & kFloatBit) != 0;
    const int n = clip_size(l, t, blockIdx.x);
    double s = 0.0;
    auto add = [&](float v) { s = INF ? nan_max(s, fabs((double)v)) : __builtin_fma((double)v, (double)v, s); };
    if (f32) clip_values((const float*)l.in[t] + at, n, add);
    else clip_values((const uint16_t*)l.in[t] + at, n, add);
    s = clip_reduce<INF>(s, lds);
    if (threadIdx.x == 0) part[l.base + blockIdx.x] = s;
}

template <bool INF>
__global__ __launch_bounds__(1024) void clip_total_kernel(const double* __restrict__ part, int64_t n, double max_norm,
                                                          float* __restrict__ total, float* __restrict__ factor) {
    __shared__ double lds[16];
    double s = 0.0;
    int64_t i = threadIdx.x;
    for (; i + 7 * 1024 < n; i += 8 * 1024) {  // eight loads on their way
        double v[8];
#pragma unroll
        for (int c = 0; c < 8; ++c) v[c] = part[i + c * 1024];
#pragma unroll
        for (int c = 0; c < 8; ++c) s = clip_join<INF>(s, v[c]);
    }
    for (; i < n; i += 1024) s = clip_join<INF>(s, part[i]);
    s = clip_reduce<INF>(s, lds);
    if (threadIdx.x == 0) {
        const double norm = INF ? s : sqrt(s);
        *total = (float)norm;
        const double k = max_norm / (norm + 1e-6);
        *factor = k < 1.0 ? (float)k : k != k ? (float)k : 1.0f;
    }
}

// Values in words W, past the caches.
template <typename T, typename W>
__device__ __forceinline__ void clip_scale(const T* in, T* out, int n, float k) {
    constexpr int N = sizeof(W) / sizeof(T);
    union Word {
        W w;
        T t[N];
    };
    const int whole = n / N;
    auto load = [&](int i) {
        Word v;
        v.w = __builtin_nontemporal_load(reinterpret_cast<const W*>(in) + i);
        return v;
    };
    auto store = [&](int i, Word v) {
#pragma unroll
        for (int j = 0; j < N; ++j) v.t[j] = Elem<T>::from_f32(Elem<T>::to_f32(v.t[j]) * k);
        __builtin_nontemporal_store(v.w, reinterpret_cast<W*>(out) + i);
    };
    int i = threadIdx.x;
    for (; i + 3 * 256 < whole; i += 4 * 256) {  // four loads on their way
        Word v[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) v[c] = load(i + c * 256);
#pragma unroll
        for (int c = 0; c < 4; ++c) store(i + c * 256, v[c]);
    }
    for (; i < whole; i += 256) store(i, load(i));
    for (i = whole * N + threadIdx.x; i < n; i += 256) out[i] = Elem<T>::from_f32(Elem<T>::to_f32(in[i]) * k);
}

template <typename T>
__device__ __forceinline__ void clip_piece(const T* in, T* out, int n, float k) {
    const uintptr_t a = (uintptr_t)in | (uintptr_t)out;
    if ((a & 15u) == 0) clip_scale<T, u32x4_t>(in, out, n, k);
    else if ((a & 3u) == 0) clip_scale<T, uint32_t>(in, out, n, k);
    else clip_scale<T, T>(in, out, n, k);
}

__global__ __launch_bounds__(256) void clip_scale_kernel(ClipList l, const float* __restrict__ factor) {
    const int b = l.pieces - 1 - (int)blockIdx.x;
    const int t = clip_find(l, b);
    const float k = *factor;
    if (k == 1.0f && l.in[t] == l.out[t]) return;
    const int64_t at = (int64_t)(b - l.first[t]) * kPiece;
    const bool f32 = (l.tail[t] & kFloatBit) != 0;
    const int n = clip_size(l, t, b);
    if (f32) clip_piece((const float*)l.in[t] + at, (float*)l.out[t] + at, n, k);
    else clip_piece((const uint16_t*)l.in[t] + at, (uint16_t*)l.out[t] + at, n, k);
}

int64_t clip_pieces(int64_t size) { return (size + kPiece - 1) / kPiece; }

}  // namespace

size_t clip_workspace_bytes(const int64_t* sizes, int n_tensors) {
    int64_t p = 0;
    for (int i = 0; i < n_tensors; ++i) p += clip_pieces(sizes[i]);
    return (size_t)p * sizeof(double) + 256;
}

int launch_clip(const void* const* in, void* const* out, const int64_t* sizes, const int32_t* dtypes, int n_tensors, int inf_norm,
                double max_norm, void* ws, float* total, hipStream_t stream) {
    float* factor = (float*)ws;
    double* part = (double*)((char*)ws + 256);
    int64_t base = 0;
    for (int pass = 0; pass < 2; ++pass) {
        base = 0;
        ClipList l;
        l.count = 0;
        l.pieces = 0;
        l.base = 0;
        for (int i = 0; i <= n_tensors; ++i) {
            if (l.count == kPerLaunch || (i == n_tensors && l.count > 0)) {
                if (pass == 1) hipLaunchKernelGGL(clip_scale_kernel, dim3(l.pieces), dim3(256), 0, stream, l, factor);
                else if (inf_norm) hipLaunchKernelGGL((clip_norm_kernel<true>), dim3(l.pieces), dim3(256), 0, stream, l, part);
                else hipLaunchKernelGGL((clip_norm_kernel<false>), dim3(l.pieces), dim3(256), 0, stream, l, part);
                base += l.pieces;
                l.count = 0;
                l.pieces = 0;
                l.base = (int32_t)base;
            }
            if (i == n_tensors || sizes[i] == 0) continue;
            l.in[l.count] = in[i];
            l.out[l.count] = out[i];
            l.tail[l.count] = (uint16_t)((sizes[i] - 1) % kPiece | (dtypes[i] == kF32 ? kFloatBit : 0));
            l.first[l.count] = l.pieces;
            l.pieces += (int32_t)clip_pieces(sizes[i]);
            ++l.count;
        }
        if (pass == 0) {
            if (inf_norm)
                hipLaunchKernelGGL((clip_total_kernel<true>), dim3(1), dim3(1024), 0, stream, part, base, max_norm, total, factor);
            else
                hipLaunchKernelGGL((clip_total_kernel<false>), dim3(1), dim3(1024), 0, stream, part, base, max_norm, total, factor);
        }
    }
    return (int)hipGetLastError();
}

}  // namespace ethos

// Embedding rows and their table's gradient.
//   out[i] = RN_T(scale w[id_i]);   dw[v] = RN_T(scale sum over {i: id_i = v} dy[i]),
// the sums float32 in a fixed order, so the gradient is the same on every run.
//
// The lookup also writes each position's key (its id, or `vocab` where it has no part in the
// gradient).  The gradient sorts the positions by key (sort.hip's stable sort, with the zeros of
// the whole table written beside it by the CUs that the single sorting workgroup leaves idle) and cuts the
// sorted list into runs of kRun for a wave each, which loads its rows at once and adds up equal keys.  A
// segment within a run is the table's row; one that a run's border cuts is left as float32 partial
// rows, at most two a run, which a second kernel adds in order, four waves to a segment: a frequent
// token's sum is spread over many workgroups.
#include "ethos_common.hpp"
#include "ethos_launch.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr int kRun = 8;
// Runs of a launch (a multiple of 4), a workgroup of 256 threads each at most, whose threads have to stay below 2^32.  More
// runs take more launches: a loop in the kernels instead made their one turn of the usual sizes slower (8,192 positions of
// 1,024: joins 8.7 -> 11.4 us).
constexpr int64_t kLaunchRuns = (int64_t)1 << 23;

// Words of sizeof(W) bytes as floats.
template <typename T, typename W> struct Words {
    static constexpr int kN = sizeof(W) / sizeof(T);
    union {
        W w;
        T t[kN];
    };
    __device__ __forceinline__ float get(int j) const { return Elem<T>::to_f32(t[j]); }
    __device__ __forceinline__ void put(int j, float v) { t[j] = Elem<T>::from_f32(v); }
};

template <typename I, typename T, typename W>
__global__ __launch_bounds__(256) void embedding_kernel(const I* __restrict__ ids, const T* __restrict__ w, int64_t n, int d,
                                                        int64_t vocab, float scale, int64_t padding, T* __restrict__ out,
                                                        int32_t* __restrict__ keys) {
    constexpr int N = Words<T, W>::kN;
    const int words = d / N;
    const int64_t total = n * words;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / words;
        const int c = (int)(i - r * words);
        const int64_t id = (int64_t)ids[r];
        const bool in = id >= 0 && id < vocab;
        if (keys && c == 0) keys[r] = in && id != padding ? (int32_t)id : (int32_t)vocab;
        Words<T, W> v;
        v.w = reinterpret_cast<const W*>(w + (in ? id : 0) * d)[c];
        if (scale != 1.0f || !in)
#pragma unroll
            for (int j = 0; j < N; ++j) v.put(j, in ? v.get(j) * scale : __builtin_nanf(""));
        reinterpret_cast<W*>(out + r * d)[c] = v.w;
    }
}

// Run b's sums, one wave.  part: [runs][2][d]: the sum of the segment that began in an earlier run, and of
// the one that goes on in a later run (a segment that does both counts as the first).
template <typename T, typename W>
__global__ __launch_bounds__(256) void embedding_run_kernel(const T* __restrict__ dy, const int32_t* __restrict__ perm,
                                                            const int32_t* __restrict__ slot, const int32_t* __restrict__ uniq,
                                                            const int32_t* __restrict__ seg_off, int64_t n, int d, int64_t vocab,
                                                            float scale, float* __restrict__ part, T* __restrict__ dw, int64_t run0) {
    constexpr int N = Words<T, W>::kN;
    const int lane = threadIdx.x & 63;
    const int64_t run = run0 + (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t p0 = run * kRun;
    if (p0 >= n) return;
    const int len = n - p0 < kRun ? (int)(n - p0) : kRun;
    int32_t s[kRun], at[kRun];
#pragma unroll
    for (int q = 0; q < kRun; ++q) {
        s[q] = slot[p0 + (q < len ? q : 0)];
        at[q] = perm[p0 + (q < len ? q : 0)];
    }
    int64_t id[kRun];
#pragma unroll
    for (int q = 0; q < kRun; ++q) id[q] = uniq[s[q]];
    const bool from_before = seg_off[s[0]] < p0, goes_on = seg_off[s[len - 1] + 1] > p0 + len;
    for (int c = lane; c < d / N; c += 64) {
        Words<T, W> v[kRun];
#pragma unroll
        for (int q = 0; q < kRun; ++q) v[q].w = reinterpret_cast<const W*>(dy + (int64_t)at[q] * d)[c];
        float sum[N];
#pragma unroll
        for (int j = 0; j < N; ++j) sum[j] = 0.0f;
#pragma unroll
        for (int q = 0; q < kRun; ++q) {
            if (q >= len) break;
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] += v[q].get(j);
            const bool end = q == len - 1 || s[q + 1 < kRun ? q + 1 : q] != s[q];
            if (!end) continue;
            if (id[q] < vocab) {
                if (from_before && s[q] == s[0]) {
#pragma unroll
                    for (int j = 0; j < N; ++j) part[run * 2 * d + c * N + j] = sum[j];
                } else if (goes_on && q == len - 1) {
#pragma unroll
                    for (int j = 0; j < N; ++j) part[(run * 2 + 1) * d + c * N + j] = sum[j];
                } else {
                    Words<T, W> o;
#pragma unroll
                    for (int j = 0; j < N; ++j) o.put(j, sum[j] * scale);
                    reinterpret_cast<W*>(dw + id[q] * d)[c] = o.w;
                }
            }
#pragma unroll
            for (int j = 0; j < N; ++j) sum[j] = 0.0f;
        }
    }
}

// One workgroup per run: the segment that begins in it and goes on past it.  Each wave adds a quarter of the
// partial rows, eight loads at a time.
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(const int32_t* __restrict__ slot, const int32_t* __restrict__ uniq,
                                                             const int32_t* __restrict__ seg_off, int64_t n, int d, int64_t vocab,
                                                             float scale, const float* __restrict__ part, T* __restrict__ dw,
                                                             int64_t run0) {
    __shared__ float lds[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t run = run0 + blockIdx.x, p0 = run * kRun;
    const int64_t p1 = p0 + kRun < n ? p0 + kRun : n;
    const int s = slot[p1 - 1];
    const int64_t b = seg_off[s], e = seg_off[s + 1], id = uniq[s];
    if (b < p0 || e <= p1 || id >= vocab) return;
    // partial rows: run's second, then the first of each later run
    const int64_t later = (e - 1) / kRun - run, per = (later + 3) / 4;
    const int64_t k0 = run + 1 + per * wave, last = run + 1 + later, k1 = k0 + per < last ? k0 + per : last;
    for (int c0 = blockIdx.y * 64; c0 < d; c0 += gridDim.y * 64) {
        const int c = c0 + lane < d ? c0 + lane : d - 1;
        float v = wave == 0 ? part[(run * 2 + 1) * d + c] : 0.0f;
        for (int64_t k = k0; k < k1; k += 8) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = part[(k + j < k1 ? k + j : k) * 2 * d + c];
#pragma unroll
            for (int j = 0; j < 8; ++j) v += k + j < k1 ? x[j] : 0.0f;
        }
        lds[wave][lane] = v;
        __syncthreads();
        if (wave == 0 && c0 + lane < d)
            dw[id * d + c] = Elem<T>::from_f32(((lds[0][lane] + lds[1][lane]) + (lds[2][lane] + lds[3][lane])) * scale);
        __syncthreads();
    }
}

struct EmbedWs {
    int32_t *perm, *uniq, *seg_off, *pair_slot, *sorted_slot, *n_unique;
    void* sort;
    float* part;
    size_t bytes;
};
EmbedWs embed_ws(char* p, int64_t n, int d, int64_t vocab) {
    EmbedWs w;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* r = p + at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    w.perm = (int32_t*)take(n * 4);
    w.uniq = (int32_t*)take(n * 4);
    w.seg_off = (int32_t*)take((n + 1) * 4);
    w.pair_slot = (int32_t*)take(n * 4);
    w.sorted_slot = (int32_t*)take(n * 4);
    w.n_unique = (int32_t*)take(4);
    w.sort = take(sort_workspace_bytes(n, vocab + 1));
    w.part = (float*)take((size_t)((n + kRun - 1) / kRun) * 2 * d * 4);
    w.bytes = at;
    return w;
}

// The widest words that every row's address allows.
template <typename T, typename F>
void with_word(const void* a, const void* b, int d, F f) {
    const uintptr_t m = (uintptr_t)a | (uintptr_t)b | (uintptr_t)((int64_t)d * (int64_t)sizeof(T));
    if ((m & 15u) == 0) f(uint4{});
    else if ((m & 3u) == 0) f(uint32_t{});
    else f(T{});
}

template <typename I, typename T>
int embedding_t(const I* ids, const T* w, int64_t n, int d, int64_t vocab, float scale, int64_t padding, T* out, int32_t* keys,
                int num_cus, hipStream_t stream) {
    with_word<T>(w, out, d, [&](auto word) {
        typedef decltype(word) W;
        const int64_t items = n * (d * (int64_t)sizeof(T) / (int64_t)sizeof(W)), b = (items + 255) / 256;
        hipLaunchKernelGGL((embedding_kernel<I, T, W>), dim3((unsigned)(b < num_cus * 16 ? b : num_cus * 16)), dim3(256), 0, stream, ids,
                           w, n, d, vocab, scale, padding, out, keys);
    });
    return (int)hipGetLastError();
}

template <typename T>
int embedding_grad_t(const int32_t* keys, const T* dy, int64_t n, int d, int64_t vocab, float scale, void* ws, T* dw, int num_cus,
                     hipStream_t stream) {
    const int64_t bytes = vocab * d * (int64_t)sizeof(T);
    if (n == 0) return launch_zero(dw, bytes, num_cus, stream);
    const EmbedWs w = embed_ws((char*)ws, n, d, vocab);
    const int rc = launch_sort_segment_zero(keys, n, vocab + 1, w.sort, w.perm, w.uniq, w.seg_off, w.pair_slot, w.sorted_slot,
                                            w.n_unique, dw, bytes, num_cus, stream);
    if (rc != 0) return rc;
    const int64_t runs = (n + kRun - 1) / kRun;
    auto in_launch = [&](int64_t r) { return runs - r < kLaunchRuns ? runs - r : kLaunchRuns; };
    with_word<T>(dy, dw, d, [&](auto word) {
        typedef decltype(word) W;
        for (int64_t r = 0; r < runs; r += kLaunchRuns)
            hipLaunchKernelGGL((embedding_run_kernel<T, W>), dim3((unsigned)((in_launch(r) + 3) / 4)), dim3(256), 0, stream, dy, w.perm,
                               w.sorted_slot, w.uniq, w.seg_off, n, d, vocab, scale, w.part, dw, r);
    });
    // columns of a long segment over as many workgroups as there are blocks of 64, up to 16
    const int cols = (d + 63) / 64;
    for (int64_t r = 0; r < runs; r += kLaunchRuns)
        hipLaunchKernelGGL((embedding_join_kernel<T>), dim3((unsigned)in_launch(r), (unsigned)(cols < 16 ? cols : 16)), dim3(256), 0, stream,
                           w.sorted_slot, w.uniq, w.seg_off, n, d, vocab, scale, w.part, dw, r);
    return (int)hipGetLastError();
}

}  // namespace

int launch_embedding(const void* ids, int ids_64, const void* w, int64_t n, int d, int64_t vocab, float scale, int64_t padding,
                     int dtype, void* out, int32_t* keys, int num_cus, hipStream_t stream) {
#define ETHOS_EMBED(I, T) embedding_t((const I*)ids, (const T*)w, n, d, vocab, scale, padding, (T*)out, keys, num_cus, stream)
    if (dtype == kBF16) return ids_64 ? ETHOS_EMBED(int64_t, uint16_t) : ETHOS_EMBED(int32_t, uint16_t);
    return ids_64 ? ETHOS_EMBED(int64_t, float) : ETHOS_EMBED(int32_t, float);
#undef ETHOS_EMBED
}

size_t embedding_grad_workspace_bytes(int64_t n, int d, int64_t vocab) { return n > 0 ? embed_ws(nullptr, n, d, vocab).bytes : 256; }

int launch_embedding_grad(const int32_t* keys, const void* dy, int64_t n, int d, int64_t vocab, float scale, int dtype, void* ws,
                          void* dw, int num_cus, hipStream_t stream) {
    return dtype == kBF16 ? embedding_grad_t(keys, (const uint16_t*)dy, n, d, vocab, scale, ws, (uint16_t*)dw, num_cus, stream)
                          : embedding_grad_t(keys, (const float*)dy, n, d, vocab, scale, ws, (float*)dw, num_cus, stream);
}

}  // namespace ethos

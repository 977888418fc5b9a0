// The cache of latents in pages (the reference keeps none): the rows of new tokens, and copies of
// pages.  A token's row is its normalised latent c, rank values, then its rotated key, rope values
// (what model.py:104-125 forms of a token before its heads' keys and values): 640 bytes in bf16 for
// rank 256 and rope 64, where a cache of 16 heads' keys and values would hold 6,144.
#include "ethos_launch.hpp"
#include "ethos_rows.hpp"
#include "ethos_serve.hpp"

namespace ethos {
namespace {

// One wave a row, from row0 of the batch on: the latent times 1 / sqrt(mean of its squares + eps) and the gain, the key's halves
// [a, b] -> [a cos - b sin, b cos + a sin]; both in float32, rounded once.  One pass: a piece of
// 16 bytes of the latent a lane in registers, and half a wave's lanes a pair of the key each.  8,192 rows of 640 bytes: 7.4 to 7.9
// us, 1.4 TB/s; 64 rows 4.3: bound by the search for a row's sequence, its page and the angle, one after the other, not by memory.
template <typename T, int CH>
__global__ __launch_bounds__(256) void append_kernel(const T* __restrict__ rows, int64_t ld, const T* __restrict__ gain,
                                                     const float* __restrict__ rates, Batch b, int64_t row0, int rank, int rope,
                                                     float eps, T* __restrict__ pool) {
    constexpr int N = Vec16<T>::kN;
    typedef typename Vec16<T>::raw Raw;
    const int lane = threadIdx.x & 63;
    const int64_t r = row0 + (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (r >= b.n_rows) return;
    const T* x = rows + r * ld;
    Raw xr[CH], gr[CH];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * 64 + lane) * N;
        xr[c] = *reinterpret_cast<const Raw*>(x + (e < rank ? e : 0));
        gr[c] = *reinterpret_cast<const Raw*>(gain + (e < rank ? e : 0));
    }
    const int i = batch_seq_wave(b, r, lane);
    if (i < 0) return;
    const int64_t pos = (int64_t)b.lens[i] - b.starts[i + 1] + r;
    const int32_t page = batch_page(b, i, pos);
    if (page < 0) return;
    const int64_t page_rows = (int64_t)1 << b.page_log;
    T* y = pool + ((int64_t)page * page_rows + (pos & (page_rows - 1))) * (rank + rope);
    float f[CH][N], s = 0.0f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        Vec16<T>::unpack(xr[c], f[c]);
        const bool in = (c * 64 + lane) * N < rank;
#pragma unroll
        for (int v = 0; v < N; ++v) s = __builtin_fmaf(in ? f[c][v] : 0.0f, f[c][v], s);
    }
    const float k = 1.0f / sqrtf(wave_sum(s) / (float)rank + eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = (c * 64 + lane) * N;
        float g[N];
        Vec16<T>::unpack(gr[c], g);
#pragma unroll
        for (int v = 0; v < N; ++v) g[v] *= f[c][v] * k;
        if (e < rank) *reinterpret_cast<Raw*>(y + e) = Vec16<T>::pack(g);
    }
    for (int p = lane; p < rope / 2; p += 64) {
        float c, sn;
        rotary_angle(pos, rates[p], c, sn);
        const float u = Elem<T>::to_f32(x[rank + p]), v = Elem<T>::to_f32(x[rank + rope / 2 + p]);
        y[rank + p] = Elem<T>::from_f32(u * c - v * sn);
        y[rank + rope / 2 + p] = Elem<T>::from_f32(v * c + u * sn);
    }
}

// Pages to copy, in a launch's arguments: the host knows them (it gives pages out), and no array has
// to reach the device first.
constexpr int kPairsMax = 448;  // 3.5 KB of the 4 KB that arguments may take
struct PagePairs {
    int32_t src[kPairsMax], dst[kPairsMax];
};

// Block y of the grid copies block y of the pool; the pieces of its pages go round the workgroups.  64 pages of 40 KB in 12
// blocks: 63 MB read and written in 10.6 us, 5.9 TB/s; 300 in 6: 147 MB in 24.1, 6.1 TB/s (from caches that hold a part).
template <typename V>
__global__ __launch_bounds__(256) void copy_pages_kernel(unsigned char* pool, int64_t block_bytes, int64_t page_bytes, int n_pairs,
                                                         int parts, PagePairs pairs) {
    const int pair = blockIdx.x / parts, part = blockIdx.x % parts;
    unsigned char* base = pool + (int64_t)blockIdx.y * block_bytes;
    const V* s = reinterpret_cast<const V*>(base + pairs.src[pair] * page_bytes);
    V* d = reinterpret_cast<V*>(base + pairs.dst[pair] * page_bytes);
    const int64_t n = page_bytes / (int64_t)sizeof(V);
    for (int64_t i = (int64_t)part * 256 + threadIdx.x; i < n; i += (int64_t)parts * 256) d[i] = s[i];
}

}  // namespace

int launch_latent_append(const void* rows, int64_t ld, const void* gain, const float* rates, const Batch& b, int rank, int rope, float eps,
                         int dtype, void* pool, hipStream_t stream) {
    constexpr int64_t kLaunchRows = (int64_t)1 << 25;  // (a launch's threads have to stay below 2^32)
    for (int64_t row0 = 0; row0 < b.n_rows; row0 += kLaunchRows) {
        const int64_t n = b.n_rows - row0 < kLaunchRows ? b.n_rows - row0 : kLaunchRows;
        const dim3 grid((unsigned)((n + 3) / 4));
        if (dtype == kBF16)
            hipLaunchKernelGGL((append_kernel<uint16_t, 1>), grid, dim3(256), 0, stream, (const uint16_t*)rows, ld, (const uint16_t*)gain,
                               rates, b, row0, rank, rope, eps, (uint16_t*)pool);
        else
            hipLaunchKernelGGL((append_kernel<float, 2>), grid, dim3(256), 0, stream, (const float*)rows, ld, (const float*)gain, rates, b,
                               row0, rank, rope, eps, (float*)pool);
    }
    return (int)hipGetLastError();
}

int launch_copy_pages(void* pool, int64_t n_blocks, int64_t block_bytes, int64_t page_bytes, const int32_t* src, const int32_t* dst,
                      int n_pairs, int num_cus, hipStream_t stream) {
    const bool wide = page_bytes % 16 == 0 && block_bytes % 16 == 0 && ((uintptr_t)pool & 15u) == 0;
    const int64_t each = wide ? 16 : 2;
    for (int at = 0; at < n_pairs; at += kPairsMax) {
        PagePairs p;
        const int n = n_pairs - at < kPairsMax ? n_pairs - at : kPairsMax;
        for (int i = 0; i < n; ++i) p.src[i] = src[at + i], p.dst[i] = dst[at + i];
        for (int i = n; i < kPairsMax; ++i) p.src[i] = p.dst[i] = 0;
        // workgroups enough for four on every CU, each with at least one piece a thread
        int64_t parts = (4 * num_cus + n * n_blocks - 1) / (n * n_blocks), most = (page_bytes / each + 255) / 256;
        if (parts > most) parts = most;
        if (parts < 1) parts = 1;
        const dim3 grid((unsigned)(n * parts), (unsigned)n_blocks);
        if (wide)
            hipLaunchKernelGGL(copy_pages_kernel<uint4>, grid, dim3(256), 0, stream, (unsigned char*)pool, block_bytes, page_bytes, n,
                               (int)parts, p);
        else
            hipLaunchKernelGGL(copy_pages_kernel<uint16_t>, grid, dim3(256), 0, stream, (unsigned char*)pool, block_bytes, page_bytes, n,
                               (int)parts, p);
        const int rc = (int)hipGetLastError();
        if (rc != 0) return rc;
    }
    return 0;
}

}  // namespace ethos

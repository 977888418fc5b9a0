// Embedding rows and their table's gradient.
//   out[i] = RN_T(scale w[id_i]);   dw[v] = RN_T(scale sum over {i: id_i = v} dy[i]),
// the sums float32 in the order of the positions, so the gradient is the same on every run.
//
// The gradient sorts the positions by id (sort.hip's stable sort; positions of the padding id and
// ids outside the table get an id past it) and cuts the sorted list into chunks of kChunk: a
// workgroup adds up its chunk's runs of equal ids.  A run that is a whole segment is the table's
// row; a run cut by the chunk's border is left as a float32 partial row, at most two a chunk, and
// a second kernel adds a segment's partials in order.  So a frequent id's sum is spread over many
// workgroups.
#include "ethos_common.hpp"
#include "ethos_launch.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr int kChunk = 32;

// Rows of `row_bytes` / sizeof(W) words; an id outside the table gives NaN.
template <typename I, typename T, typename W>
__global__ __launch_bounds__(256) void embedding_kernel(const I* __restrict__ ids, const T* __restrict__ w, int64_t n, int d,
                                                        int64_t vocab, float scale, T* __restrict__ out) {
    constexpr int N = sizeof(W) / sizeof(T);
    const int words = d / N;
    const int64_t total = n * words;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / words;
        const int c = (int)(i - r * words);
        const int64_t id = (int64_t)ids[r];
        const bool in = id >= 0 && id < vocab;
        union {
            W w;
            T t[N];
        } v;
        v.w = reinterpret_cast<const W*>(w + (in ? id : 0) * d)[c];
        if (scale != 1.0f || !in)
#pragma unroll
            for (int j = 0; j < N; ++j) v.t[j] = Elem<T>::from_f32(in ? Elem<T>::to_f32(v.t[j]) * scale : __builtin_nanf(""));
        reinterpret_cast<W*>(out + r * d)[c] = v.w;
    }
}

// Sort keys: the id, or `vocab` where a position has no part in the gradient.
template <typename I>
__global__ __launch_bounds__(256) void embedding_keys_kernel(const I* __restrict__ ids, int64_t n, int64_t vocab, int64_t padding,
                                                             int32_t* __restrict__ keys) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int64_t id = (int64_t)ids[i];
    keys[i] = id >= 0 && id < vocab && id != padding ? (int32_t)id : (int32_t)vocab;
}

__global__ __launch_bounds__(256) void embedding_zero_kernel(uint4* __restrict__ p, int64_t n16, uint32_t* __restrict__ rest,
                                                             int64_t n_rest, int odd) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n16; i += (int64_t)gridDim.x * 256) p[i] = make_uint4(0, 0, 0, 0);
    if (blockIdx.x == 0) {
        for (int64_t i = threadIdx.x; i < n_rest; i += 256) rest[i] = 0;
        if (odd && threadIdx.x == 0) *reinterpret_cast<uint16_t*>(rest + n_rest) = 0;
    }
}

// Chunk b's runs.  part: [chunks][2][d]: the sum of the run that began in an earlier chunk, and of
// the run that goes on in a later one (a run that does both counts as the first).
template <typename T>
__global__ __launch_bounds__(256) void embedding_chunk_kernel(const T* __restrict__ dy, const int32_t* __restrict__ perm,
                                                              const int32_t* __restrict__ slot, const int32_t* __restrict__ uniq,
                                                              const int32_t* __restrict__ seg_off, int64_t n, int d, int64_t vocab,
                                                              float scale, float* __restrict__ part, T* __restrict__ dw) {
    const int64_t p0 = (int64_t)blockIdx.x * kChunk;
    const int64_t p1 = p0 + kChunk < n ? p0 + kChunk : n;
    for (int64_t p = p0; p < p1;) {
        const int s = slot[p];
        const int64_t b = seg_off[s], e = seg_off[s + 1];
        const int64_t end = e < p1 ? e : p1;
        const int64_t id = uniq[s];
        if (id < vocab) {
            for (int c = threadIdx.x; c < d; c += 256) {
                float v = 0.0f;
                for (int64_t q = p; q < end; ++q) v += Elem<T>::to_f32(dy[(int64_t)perm[q] * d + c]);
                if (b < p0) part[((int64_t)blockIdx.x * 2) * d + c] = v;
                else if (e > p1) part[((int64_t)blockIdx.x * 2 + 1) * d + c] = v;
                else dw[id * d + c] = Elem<T>::from_f32(v * scale);
            }
        }
        p = end;
    }
}

// One workgroup per chunk: the segment that begins in it and goes on past it.
template <typename T>
__global__ __launch_bounds__(256) void embedding_join_kernel(const int32_t* __restrict__ slot, const int32_t* __restrict__ uniq,
                                                             const int32_t* __restrict__ seg_off, int64_t n, int d, int64_t vocab,
                                                             float scale, const float* __restrict__ part, T* __restrict__ dw) {
    const int64_t p0 = (int64_t)blockIdx.x * kChunk;
    const int64_t p1 = p0 + kChunk < n ? p0 + kChunk : n;
    const int s = slot[p1 - 1];
    const int64_t b = seg_off[s], e = seg_off[s + 1], id = uniq[s];
    if (b < p0 || e <= p1 || id >= vocab) return;
    const int64_t last = (e - 1) / kChunk;
    for (int c = threadIdx.x; c < d; c += 256) {
        float v = part[((int64_t)blockIdx.x * 2 + 1) * d + c];
        for (int64_t k = blockIdx.x + 1; k <= last; ++k) v += part[k * 2 * d + c];
        dw[id * d + c] = Elem<T>::from_f32(v * scale);
    }
}

struct EmbedWs {
    int32_t *keys, *perm, *uniq, *seg_off, *pair_slot, *sorted_slot, *n_unique;
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
    w.keys = (int32_t*)take(n * 4);
    w.perm = (int32_t*)take(n * 4);
    w.uniq = (int32_t*)take(n * 4);
    w.seg_off = (int32_t*)take((n + 1) * 4);
    w.pair_slot = (int32_t*)take(n * 4);
    w.sorted_slot = (int32_t*)take(n * 4);
    w.n_unique = (int32_t*)take(4);
    w.sort = take(sort_workspace_bytes(n, vocab + 1));
    w.part = (float*)take((size_t)((n + kChunk - 1) / kChunk) * 2 * d * 4);
    w.bytes = at;
    return w;
}

template <typename I, typename T>
int embedding_t(const I* ids, const T* w, int64_t n, int d, int64_t vocab, float scale, T* out, int num_cus, hipStream_t stream) {
    // the widest loads that every row's address allows
    const uintptr_t a = (uintptr_t)w | (uintptr_t)out | (uintptr_t)((int64_t)d * (int64_t)sizeof(T));
    const int width = (a & 15u) == 0 ? 16 : (a & 3u) == 0 ? 4 : 2;
    const int64_t items = n * (d * (int64_t)sizeof(T) / width);
    int64_t b = (items + 255) / 256;
    b = b < (int64_t)num_cus * 16 ? b : (int64_t)num_cus * 16;
    const dim3 grid((unsigned)b);
    if (width == 16) hipLaunchKernelGGL((embedding_kernel<I, T, uint4>), grid, dim3(256), 0, stream, ids, w, n, d, vocab, scale, out);
    else if (width == 4) hipLaunchKernelGGL((embedding_kernel<I, T, uint32_t>), grid, dim3(256), 0, stream, ids, w, n, d, vocab, scale, out);
    else hipLaunchKernelGGL((embedding_kernel<I, T, T>), grid, dim3(256), 0, stream, ids, w, n, d, vocab, scale, out);
    return (int)hipGetLastError();
}

template <typename T>
int embedding_grad_t(const void* ids, int ids_64, const T* dy, int64_t n, int d, int64_t vocab, float scale, int64_t padding,
                     void* ws, T* dw, int num_cus, hipStream_t stream) {
    const int64_t bytes = vocab * d * (int64_t)sizeof(T), n16 = bytes / 16;
    hipLaunchKernelGGL(embedding_zero_kernel, dim3((unsigned)(num_cus * 16)), dim3(256), 0, stream, (uint4*)dw, n16,
                       (uint32_t*)dw + n16 * 4, bytes % 16 / 4, (int)(bytes % 4 / 2));
    if (n > 0) {
        const EmbedWs w = embed_ws((char*)ws, n, d, vocab);
        const dim3 kg((unsigned)((n + 255) / 256)), cg((unsigned)((n + kChunk - 1) / kChunk));
        if (ids_64)
            hipLaunchKernelGGL((embedding_keys_kernel<int64_t>), kg, dim3(256), 0, stream, (const int64_t*)ids, n, vocab, padding, w.keys);
        else
            hipLaunchKernelGGL((embedding_keys_kernel<int32_t>), kg, dim3(256), 0, stream, (const int32_t*)ids, n, vocab, padding, w.keys);
        const int rc = launch_sort_segment(w.keys, n, vocab + 1, w.sort, w.perm, w.uniq, w.seg_off, w.pair_slot, w.sorted_slot,
                                           w.n_unique, stream);
        if (rc != 0) return rc;
        hipLaunchKernelGGL((embedding_chunk_kernel<T>), cg, dim3(256), 0, stream, dy, w.perm, w.sorted_slot, w.uniq, w.seg_off, n, d,
                           vocab, scale, w.part, dw);
        hipLaunchKernelGGL((embedding_join_kernel<T>), cg, dim3(256), 0, stream, w.sorted_slot, w.uniq, w.seg_off, n, d, vocab, scale,
                           w.part, dw);
    }
    return (int)hipGetLastError();
}

}  // namespace

int launch_embedding(const void* ids, int ids_64, const void* w, int64_t n, int d, int64_t vocab, float scale, int dtype, void* out,
                     int num_cus, hipStream_t stream) {
    if (dtype == kBF16)
        return ids_64 ? embedding_t((const int64_t*)ids, (const uint16_t*)w, n, d, vocab, scale, (uint16_t*)out, num_cus, stream)
                      : embedding_t((const int32_t*)ids, (const uint16_t*)w, n, d, vocab, scale, (uint16_t*)out, num_cus, stream);
    return ids_64 ? embedding_t((const int64_t*)ids, (const float*)w, n, d, vocab, scale, (float*)out, num_cus, stream)
                  : embedding_t((const int32_t*)ids, (const float*)w, n, d, vocab, scale, (float*)out, num_cus, stream);
}

size_t embedding_grad_workspace_bytes(int64_t n, int d, int64_t vocab) { return n > 0 ? embed_ws(nullptr, n, d, vocab).bytes : 256; }

int launch_embedding_grad(const void* ids, int ids_64, const void* dy, int64_t n, int d, int64_t vocab, float scale, int64_t padding,
                          int dtype, void* ws, void* dw, int num_cus, hipStream_t stream) {
    return dtype == kBF16
               ? embedding_grad_t(ids, ids_64, (const uint16_t*)dy, n, d, vocab, scale, padding, ws, (uint16_t*)dw, num_cus, stream)
               : embedding_grad_t(ids, ids_64, (const float*)dy, n, d, vocab, scale, padding, ws, (float*)dw, num_cus, stream);
}

}  // namespace ethos

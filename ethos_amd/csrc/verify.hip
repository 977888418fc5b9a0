// Verification of drafted tokens against the model's probabilities, from given random numbers (the reference
// decodes nothing).  p_j = softmax(logits_j / temperature); draft j is accepted while u q_j(x_j) < p_j(x_j),
// q_j the probabilities it was drawn from (1 at x_j where there are none); behind the last accepted one a token is
// drawn from max(p - q, 0), or, where all were accepted, from p: the lowest index whose sum of weights up to it
// exceeds u times their sum.  Tokens so found are distributed as p's own.
//
// Exponentials and sums are float64: a row has 100,000 borders between its words, and a float32 sum's error, some
// 1e-6, would put every tenth random number on the wrong side of one.  The logits are read once, and once more in
// the one row of a sequence that a token is drawn from.
#include "ethos_launch.hpp"
#include "ethos_rows.hpp"
#include "ethos_serve.hpp"

namespace ethos {
namespace {

constexpr int kPiece = 8;               // values of a thread that follow each other
constexpr int kSpan = 256 * kPiece;     // of a workgroup
constexpr int kDraftsMax = 255;
constexpr int kChunksMax = 2048;

// Of a chunk of a row: its maximum, where that is first, and the sum of exp2((l - max) rate); NaN if any value is
// NaN, or +inf (unless greedy).
struct Chunk {
    double sum;
    float max;
    int32_t arg;
};

// 2^x for x <= 0 (and NaN), float64: 2^k e^(f ln 2), f in [-1/2, 1/2], the series to f^11, whose rest is 7e-15.
__device__ __forceinline__ double exp2_f64(double x) {
    x = x < -1100.0 ? -1100.0 : x;
    const double k = rint(x), y = (x - k) * 0.6931471805599453;
    double e = 1.0 / 39916800.0;
    e = __builtin_fma(e, y, 1.0 / 3628800.0);
    e = __builtin_fma(e, y, 1.0 / 362880.0);
    e = __builtin_fma(e, y, 1.0 / 40320.0);
    e = __builtin_fma(e, y, 1.0 / 5040.0);
    e = __builtin_fma(e, y, 1.0 / 720.0);
    e = __builtin_fma(e, y, 1.0 / 120.0);
    e = __builtin_fma(e, y, 1.0 / 24.0);
    e = __builtin_fma(e, y, 1.0 / 6.0);
    e = __builtin_fma(e, y, 0.5);
    e = __builtin_fma(e, y, 1.0);
    e = __builtin_fma(e, y, 1.0);
    return ldexp(e, (int)k);
}

// Values at e .. e + 7 of a row of n (any address a T may have); `fill` behind its end.
template <typename T>
__device__ __forceinline__ void load_piece(const T* row, int64_t e, int64_t n, float fill, float* f) {
    if (e + kPiece <= n) {
        T v[kPiece];
        __builtin_memcpy(v, row + e, sizeof(v));
#pragma unroll
        for (int i = 0; i < kPiece; ++i) f[i] = Elem<T>::to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < kPiece; ++i) f[i] = e + i < n ? Elem<T>::to_f32(row[e + i]) : fill;
    }
}

__device__ __forceinline__ double wave_sum_f64(double v) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) v += __shfl_xor(v, d, 64);
    return v;
}

__device__ __forceinline__ void take_first(float& m, int32_t& at, float om, int32_t oat) {
    if (om > m || (om == m && oat < at)) m = om, at = oat;
}

struct Args {
    const void* logits;
    const int64_t* drafts;
    const void* probs;  // nullptr: every draft had probability 1
    const int32_t* counts;
    const float *u_accept, *u_sample;
    int m;  // drafts of a sequence, at most
    int64_t vocab;
    double rate;  // log2 e / temperature; 0: greedy
    int chunks;
    Chunk* stats;    // [rows][chunks]
    double* weights; // [n_seq][chunks]
    int32_t* done;   // [n_seq]
    int32_t* accepted;
    int64_t* tokens;
};

__device__ __forceinline__ int draft_count(const Args& a, int64_t i) {
    const int n = a.counts ? a.counts[i] : a.m;
    return n < 0 ? 0 : n > a.m ? a.m : n;
}

// Chunk blockIdx.x % chunks of row blockIdx.x / chunks.
template <typename T, int PC>
__global__ __launch_bounds__(256) void chunk_kernel(Args a) {
    __shared__ float ms[4];
    __shared__ int32_t ats[4];
    __shared__ double ss[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = blockIdx.x / a.chunks;
    const int s = blockIdx.x % a.chunks;
    const int64_t i = row / (a.m + 1);
    const int j = (int)(row - i * (a.m + 1));
    if (j == 0 && s == 0 && tid == 0) a.done[i] = 0;
    if (j > draft_count(a, i)) return;
    const T* l = (const T*)a.logits + row * a.vocab;
    float f[PC][kPiece], m = -INFINITY;
    int32_t at = INT32_MAX;
#pragma unroll
    for (int c = 0; c < PC; ++c) load_piece(l, ((int64_t)s * PC + c) * kSpan + tid * kPiece, a.vocab, -INFINITY, f[c]);
#pragma unroll
    for (int c = 0; c < PC; ++c)
#pragma unroll
        for (int v = 0; v < kPiece; ++v)
            if (f[c][v] > m) m = f[c][v], at = (int32_t)(((int64_t)s * PC + c) * kSpan + tid * kPiece + v);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) take_first(m, at, __shfl_xor(m, d, 64), __shfl_xor(at, d, 64));
    if (lane == 0) ms[wave] = m, ats[wave] = at;
    __syncthreads();
    m = ms[0], at = ats[0];
    for (int w = 1; w < 4; ++w) take_first(m, at, ms[w], ats[w]);
    // (a chunk of -inf alone: every exponential 0)
    const float base = m == -INFINITY ? 0.0f : m;
    double sum = 0.0;
    if (a.rate != 0.0) {
#pragma unroll
        for (int c = 0; c < PC; ++c)
#pragma unroll
            for (int v = 0; v < kPiece; ++v) sum += exp2_f64(((double)f[c][v] - (double)base) * a.rate);
    } else {
#pragma unroll
        for (int c = 0; c < PC; ++c)
#pragma unroll
            for (int v = 0; v < kPiece; ++v) sum += f[c][v] != f[c][v] ? NAN : 0.0;
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        Chunk k;
        k.sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
        k.max = m;
        k.arg = at;
        a.stats[row * a.chunks + s] = k;
    }
}

// A row's maximum, sum and arg from its chunks, by a wave; NaN where the row has no distribution.
__device__ __forceinline__ Chunk join_chunks(const Args& a, int64_t row, int lane) {
    float m = -INFINITY;
    int32_t at = INT32_MAX;
    for (int s = lane; s < a.chunks; s += 64) {
        const Chunk k = a.stats[row * a.chunks + s];
        take_first(m, at, k.max, k.arg);
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) take_first(m, at, __shfl_xor(m, d, 64), __shfl_xor(at, d, 64));
    double sum = 0.0;
    for (int s = lane; s < a.chunks; s += 64) {
        const Chunk k = a.stats[row * a.chunks + s];
        sum += a.rate != 0.0 ? k.sum * (k.max == -INFINITY ? (k.sum == k.sum ? 0.0 : 1.0) : exp2_f64(((double)k.max - (double)m) * a.rate)) : k.sum;
    }
    Chunk r;
    r.sum = m == -INFINITY ? NAN : wave_sum_f64(sum);
    r.max = m;
    r.arg = at;
    return r;
}

// The weights that the token is drawn by, at 8 places of the row; p alone where there is no q.
template <typename T, typename Q>
__device__ __forceinline__ void weights8(const Args& a, const T* l, const Q* q, int64_t one, float max, double inv, int64_t e, double* w) {
    float f[kPiece], g[kPiece] = {};
    load_piece(l, e, a.vocab, -INFINITY, f);
    if (q) load_piece(q, e, a.vocab, 0.0f, g);
#pragma unroll
    for (int v = 0; v < kPiece; ++v) {
        const double p = exp2_f64(((double)f[v] - (double)max) * a.rate) * inv;
        w[v] = fmax(e + v == one ? p - 1.0 : p - (double)g[v], 0.0);
    }
}

// Chunk blockIdx.x % chunks of sequence blockIdx.x / chunks: which drafts are accepted, then the chunk's sum of
// weights; the sequence's last workgroup to come here finds the token.  Greedy: one workgroup a sequence.
template <typename T, typename Q, int PC>
__global__ __launch_bounds__(256) void draw_kernel(Args a) {
    __shared__ Chunk rows[kDraftsMax + 1];
    __shared__ unsigned char ok[kDraftsMax + 1];
    __shared__ double ss[kChunksMax > 256 ? kChunksMax : 256];
    __shared__ int turn, low, high;
    __shared__ double rest;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int parts = a.rate != 0.0 ? a.chunks : 1;
    const int64_t i = blockIdx.x / parts;
    const int s = blockIdx.x % parts, n = draft_count(a, i);
    const int64_t row0 = i * (a.m + 1);
    for (int j = wave; j <= n; j += 4) {
        const Chunk k = join_chunks(a, row0 + j, lane);
        if (lane == 0) {
            bool good = false;
            if (j < n && k.sum == k.sum) {
                const int64_t x = a.drafts[i * a.m + j];
                if (x >= 0 && x < a.vocab) {
                    const double u = (double)a.u_accept[i * a.m + j];
                    const double q = a.probs ? (double)Elem<Q>::to_f32(((const Q*)a.probs)[(i * a.m + j) * a.vocab + x]) : 1.0;
                    const double l = (double)Elem<T>::to_f32(((const T*)a.logits)[(row0 + j) * a.vocab + x]);
                    const double p = a.rate != 0.0 ? exp2_f64((l - (double)k.max) * a.rate) / k.sum : x == k.arg ? 1.0 : 0.0;
                    good = u * q < p;
                }
            }
            rows[j] = k;
            ok[j] = good;
        }
    }
    __syncthreads();
    int took = 0;
    while (took < n && ok[took]) ++took;
    const Chunk k = rows[took];
    if (k.sum != k.sum || a.rate == 0.0) {
        if (s == 0 && tid == 0) {
            a.accepted[i] = took;
            a.tokens[i] = k.sum != k.sum ? -1 : k.arg;
        }
        return;
    }
    const T* l = (const T*)a.logits + (row0 + took) * a.vocab;
    const Q* q = a.probs && took < n ? (const Q*)a.probs + (i * a.m + took) * a.vocab : nullptr;
    const int64_t one = !a.probs && took < n ? a.drafts[i * a.m + took] : -1;
    const double inv = 1.0 / k.sum;
    double w[PC][kPiece], part[PC], sum = 0.0;
#pragma unroll
    for (int c = 0; c < PC; ++c) {
        weights8(a, l, q, one, k.max, inv, ((int64_t)s * PC + c) * kSpan + tid * kPiece, w[c]);
        part[c] = 0.0;
#pragma unroll
        for (int v = 0; v < kPiece; ++v) part[c] += w[c][v];
        sum += part[c];
    }
    sum = wave_sum_f64(sum);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        __hip_atomic_store(&a.weights[i * parts + s], (ss[0] + ss[1]) + (ss[2] + ss[3]), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        turn = __hip_atomic_fetch_add(&a.done[i], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
        low = INT32_MAX;
        high = -1;
    }
    __syncthreads();
    if (turn != parts - 1) return;
    for (int c = tid; c < parts; c += 256) ss[c] = __hip_atomic_load(&a.weights[i * parts + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (tid == 0) {
        double all = 0.0;
        for (int c = 0; c < parts; ++c) all += ss[c];
        rest = all;
    }
    __syncthreads();
    const bool none = rest == 0.0;  // q covers p: drawn from p itself
    if (none) {
        __syncthreads();
        for (int c = tid; c < parts; c += 256) {
            const Chunk o = a.stats[(row0 + took) * a.chunks + c];
            ss[c] = o.max == -INFINITY ? 0.0 : o.sum * exp2_f64(((double)o.max - (double)k.max) * a.rate) * inv;
        }
        __syncthreads();
        if (tid == 0) {
            double all = 0.0;
            for (int c = 0; c < parts; ++c) all += ss[c];
            rest = all;
        }
        __syncthreads();
    }
    const double want = (double)a.u_sample[i] * rest;
    // the chunk, then the place in it
    double before = 0.0;
    int at = 0, some = 0;
    for (int c = 0; c < parts; ++c) {
        if (ss[c] > 0.0) some = c;
        if (before + ss[c] > want) break;
        before += ss[c];
        ++at;
    }
    if (at == parts) {  // rounding: the last place of any weight
        at = some;
        before = -INFINITY;
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < PC; ++c) {
        weights8(a, l, none ? nullptr : q, none ? -1 : one, k.max, inv, ((int64_t)at * PC + c) * kSpan + tid * kPiece, w[c]);
        part[c] = 0.0;
#pragma unroll
        for (int v = 0; v < kPiece; ++v) part[c] += w[c][v];
        double up = part[c];
        for (int d = 1; d < 64; d <<= 1) {
            const double o = __shfl_up(up, d, 64);
            if (lane >= d) up += o;
        }
        if (lane == 63) ss[c * 4 + wave] = up;
        part[c] = up - part[c];
    }
    __syncthreads();
    int first = INT32_MAX, last = -1;
#pragma unroll
    for (int c = 0; c < PC; ++c) {
        double sum_to = before + part[c];
        for (int z = 0; z < c * 4 + wave; ++z) sum_to += ss[z];
#pragma unroll
        for (int v = 0; v < kPiece; ++v) {
            sum_to += w[c][v];
            const int e = (c * 256 + tid) * kPiece + v;
            if (w[c][v] > 0.0) {
                if (sum_to > want && e < first) first = e;
                last = e;
            }
        }
    }
    if (first != INT32_MAX) atomicMin(&low, first);
    __syncthreads();
    if (low == INT32_MAX && last >= 0) atomicMax(&high, last);
    __syncthreads();
    if (tid == 0) {
        a.accepted[i] = took;
        a.tokens[i] = (int64_t)at * PC * kSpan + (low != INT32_MAX ? low : high);
    }
}

template <typename T, int PC>
void launch_all(const Args& a, int64_t n_seq, int probs_dtype, hipStream_t stream) {
    hipLaunchKernelGGL((chunk_kernel<T, PC>), dim3((unsigned)(n_seq * (a.m + 1) * a.chunks)), dim3(256), 0, stream, a);
    const dim3 grid((unsigned)(n_seq * (a.rate != 0.0 ? a.chunks : 1)));
    if (probs_dtype == kBF16) hipLaunchKernelGGL((draw_kernel<T, uint16_t, PC>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((draw_kernel<T, float, PC>), grid, dim3(256), 0, stream, a);
}

constexpr int kPieces = 4;
int chunks_of(int64_t vocab) { return (int)((vocab + kPieces * kSpan - 1) / (kPieces * kSpan)); }
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

size_t verify_workspace_bytes(int64_t n_seq, int n_drafts, int64_t vocab) {
    const size_t c = (size_t)chunks_of(vocab);
    return round256((size_t)n_seq * (n_drafts + 1) * c * sizeof(Chunk)) + round256((size_t)n_seq * c * 8) + round256((size_t)n_seq * 4);
}

int launch_verify(const void* logits, const int64_t* drafts, const void* probs, int probs_dtype, const int32_t* counts,
                  const float* u_accept, const float* u_sample, int64_t n_seq, int n_drafts, int64_t vocab, double temperature, int dtype,
                  void* ws, int32_t* accepted, int64_t* tokens, hipStream_t stream) {
    Args a;
    a.logits = logits;
    a.drafts = drafts;
    a.probs = n_drafts > 0 ? probs : nullptr;
    a.counts = counts;
    a.u_accept = u_accept;
    a.u_sample = u_sample;
    a.m = n_drafts;
    a.vocab = vocab;
    a.rate = temperature > 0.0 ? 1.4426950408889634 / temperature : 0.0;
    a.chunks = chunks_of(vocab);
    unsigned char* w = (unsigned char*)ws;
    a.stats = (Chunk*)w;
    w += round256((size_t)n_seq * (n_drafts + 1) * a.chunks * sizeof(Chunk));
    a.weights = (double*)w;
    w += round256((size_t)n_seq * a.chunks * 8);
    a.done = (int32_t*)w;
    a.accepted = accepted;
    a.tokens = tokens;
    if (dtype == kBF16) launch_all<uint16_t, kPieces>(a, n_seq, probs_dtype, stream);
    else launch_all<float, kPieces>(a, n_seq, probs_dtype, stream);
    return (int)hipGetLastError();
}

}  // namespace ethos

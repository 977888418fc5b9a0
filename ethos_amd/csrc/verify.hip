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
constexpr int kPartsMax = 1024;
constexpr int64_t kLaunchGroups = (int64_t)1 << 23;  // workgroups of a launch, whose threads have to stay below 2^32

// Of a chunk of a row: its maximum, where that is first, and the sum of exp2((l - max) rate); NaN if any value is
// NaN, or +inf (unless greedy).
struct Chunk {
    double sum;
    float max;
    int32_t arg;
};

// exp2((l - max) rate) for l <= max, in float64: 2^(k / 32 + r), |r| <= 1/64, as a table's 2^(k % 32 / 32), an
// exponent and the series of 2^r to r^4, whose rest is 1.2e-12.  (The table of 32 doubles is LDS's 64 banks once: lanes
// read it without conflicts.  With the series alone, to r^11 and over a range of 1, the rows' sums took 36 us where
// the table took 28, and 30 with the difference first: the kernel is bound by its vector instructions, a dozen of float64 a value.)
// Below 2^-1020: zero.  NaN stays.
// The difference comes before the scale: it is 0 at the maximum, however far from zero that is, where
// l rate - RN(max rate) would be the rounding of max rate, an exponent of any size for maxima of 1e16 and more.
struct Exp {
    double rate32, base;
};
__device__ __forceinline__ Exp exp_from(float base, double rate) {
    // (a maximum of -inf: no value has a weight)
    return Exp{rate * 32.0, base == -INFINITY ? 0.0 : (double)base};
}
__device__ __forceinline__ void exp_table(double* table, int tid) {
    if (tid < 32) table[tid] = exp2((double)tid / 32.0);
}
__device__ __forceinline__ double exp_of(const Exp& x, const double* table, float l) {
    constexpr double kLn = 0.6931471805599453 / 32.0, kMagic = 6755399441055744.0;  // 1.5 2^52: its sum's low word is a rounded k
    const double t = ((double)l - x.base) * x.rate32, s = t + kMagic, r = t - (s - kMagic);
    const int k = __double2loint(s);
    double e = __builtin_fma(r, kLn * kLn * kLn * kLn / 24.0, kLn * kLn * kLn / 6.0);
    e = __builtin_fma(e, r, kLn * kLn / 2.0);
    e = __builtin_fma(e, r, kLn);
    e = __builtin_fma(e, r, 1.0) * table[k & 31];
    e = __hiloint2double(__double2hiint(e) + ((k >> 5) << 20), __double2loint(e));
    return t < -32640.0 ? 0.0 : e;
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
    int64_t first;  // the row or sequence that a launch begins with
    double rate;    // log2 e / temperature; 0: greedy
    int chunks;   // of a row, for its sums
    int parts;    // of the row that a token is drawn from
    int part_pieces;
    int own_parts;  // up to so many parts of all sequences each workgroup decides for itself, which saves a launch
    Chunk* stats;    // [rows][chunks]
    Chunk* rows;     // [n_seq]: the row that a token is drawn from
    double* weights; // [n_seq][parts]
    int32_t* done;   // [n_seq]
    int32_t* accepted;
    int64_t* tokens;
};

__device__ __forceinline__ int draft_count(const Args& a, int64_t i) {
    const int n = a.counts ? a.counts[i] : a.m;
    return n < 0 ? 0 : n > a.m ? a.m : n;
}

// Chunk blockIdx.x % chunks of a launch's row blockIdx.x / chunks.  320 rows of 100,277 bf16 words: 64 MB in 34 us, 1.9 TB/s (269 of
// them, the others behind their sequences' drafts: 30), bound by the exponentials' instructions; the largest logits of those 269
// (temperature 0) 16.5.
template <typename T, int PC, bool GREEDY>
__global__ __launch_bounds__(256) void chunk_kernel(Args a) {
    __shared__ double table[32];
    __shared__ float ms[4];
    __shared__ int32_t ats[4];
    __shared__ double ss[4];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row = a.first + blockIdx.x / a.chunks;
    const int s = blockIdx.x % a.chunks;
    const int64_t i = row / (a.m + 1);
    const int j = (int)(row - i * (a.m + 1));
    const T* l = (const T*)a.logits + row * a.vocab;
    float f[PC][kPiece], m = -INFINITY;
    int32_t at = INT32_MAX;
    if (j == 0 && s == 0 && tid == 0) a.done[i] = 0;
    if (j > draft_count(a, i)) return;
#pragma unroll
    for (int c = 0; c < PC; ++c) load_piece(l, ((int64_t)s * PC + c) * kSpan + tid * kPiece, a.vocab, -INFINITY, f[c]);
    exp_table(table, tid);
#pragma unroll
    for (int c = 0; c < PC; ++c)
#pragma unroll
        for (int v = 0; v < kPiece; ++v) {
            if (GREEDY && f[c][v] > m) at = (int32_t)(((int64_t)s * PC + c) * kSpan + tid * kPiece + v);
            m = fmaxf(m, f[c][v]);
        }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        if (GREEDY) take_first(m, at, __shfl_xor(m, d, 64), __shfl_xor(at, d, 64));
        else m = fmaxf(m, __shfl_xor(m, d, 64));
    }
    if (lane == 0) ms[wave] = m, ats[wave] = at;
    __syncthreads();
    m = ms[0], at = ats[0];
    for (int w = 1; w < 4; ++w) take_first(m, at, ms[w], ats[w]);
    double sum = 0.0;
    const Exp x = exp_from(m, a.rate);
#pragma unroll
    for (int c = 0; c < PC; ++c)
#pragma unroll
        for (int v = 0; v < kPiece; ++v) {
            if (GREEDY) sum += f[c][v] != f[c][v] ? NAN : 0.0;
            else sum += exp_of(x, table, f[c][v]);
        }
    sum = wave_sum_f64(sum);
    if (lane == 0) ss[wave] = sum;
    __syncthreads();
    if (tid == 0) {
        Chunk k;
        k.sum = m == INFINITY && !GREEDY ? NAN : (ss[0] + ss[1]) + (ss[2] + ss[3]);
        k.max = m;
        k.arg = at;
        a.stats[row * a.chunks + s] = k;
    }
}

// A row's maximum, sum and arg from its chunks, by W neighbouring lanes (lane: its place among them); NaN where the row has no
// distribution.
template <int W>
__device__ __forceinline__ Chunk join_chunks(const Args& a, const double* table, int64_t row, int lane) {
    float m = -INFINITY;
    int32_t at = INT32_MAX;
    const Chunk* stats = a.stats + row * a.chunks;
    for (int s = lane; s < a.chunks; s += W) take_first(m, at, stats[s].max, stats[s].arg);
#pragma unroll
    for (int d = 1; d < W; d <<= 1) take_first(m, at, __shfl_xor(m, d, 64), __shfl_xor(at, d, 64));
    const Exp x = exp_from(m, a.rate);
    double sum = 0.0;
    for (int s = lane; s < a.chunks; s += W) {
        const Chunk k = stats[s];
        // (a chunk without a finite value: its sum is 0, or NaN)
        sum += k.max == -INFINITY || a.rate == 0.0 ? k.sum : k.sum * exp_of(x, table, k.max);
    }
#pragma unroll
    for (int d = 1; d < W; d <<= 1) sum += __shfl_xor(sum, d, 64);
    return Chunk{m == -INFINITY ? NAN : sum, m, at};
}

// A workgroup's sum, in a fixed order; ss: 4 values, free before and after.
__device__ __forceinline__ double block_sum_f64(double v, double* ss, int tid) {
    v = wave_sum_f64(v);
    __syncthreads();
    if ((tid & 63) == 0) ss[tid >> 6] = v;
    __syncthreads();
    v = (ss[0] + ss[1]) + (ss[2] + ss[3]);
    __syncthreads();
    return v;
}

// How many drafts of sequence i are accepted, and the row that its token is drawn from, by a workgroup (with the table
// of exponentials to be filled).
template <typename T, typename Q>
__device__ __forceinline__ int decide(const Args& a, int64_t i, int n, double* table, Chunk& row) {
    __shared__ Chunk rows[kDraftsMax + 1];
    __shared__ int first_bad;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int64_t row0 = i * (a.m + 1);
    // a thread a draft: what its test needs, on its way while the rows' sums are joined
    int64_t x = -1;
    float u = 0.0f, q_x = 1.0f, l_x = 0.0f;
    if (tid < n) {
        x = a.drafts[i * a.m + tid];
        u = a.u_accept[i * a.m + tid];
        if (x >= 0 && x < a.vocab) {
            l_x = Elem<T>::to_f32(((const T*)a.logits)[(row0 + tid) * a.vocab + x]);
            if (a.probs) q_x = Elem<Q>::to_f32(((const Q*)a.probs)[(i * a.m + tid) * a.vocab + x]);
        }
    }
    exp_table(table, tid);
    if (tid == 0) first_bad = n;
    __syncthreads();
    // rows of few chunks four a wave (16 sequences of 9 rows of 4 chunks, the kernel's time: 13.1 us with one a wave, 11.0 with four)
    if (a.chunks <= 16) {
        for (int j = tid >> 4; j <= n; j += 16) {
            const Chunk k = join_chunks<16>(a, table, row0 + j, lane & 15);
            if ((lane & 15) == 0) rows[j] = k;
        }
    } else {
        for (int j = wave; j <= n; j += 4) {
            const Chunk k = join_chunks<64>(a, table, row0 + j, lane);
            if (lane == 0) rows[j] = k;
        }
    }
    __syncthreads();
    if (tid < n) {
        const Chunk k = rows[tid];
        bool good = k.sum == k.sum && x >= 0 && x < a.vocab;
        if (good) {
            const double p = a.rate != 0.0 ? exp_of(exp_from(k.max, a.rate), table, l_x) / k.sum : x == k.arg ? 1.0 : 0.0;
            good = (double)u * (double)q_x < p;
        }
        if (!good) atomicMin(&first_bad, tid);
    }
    __syncthreads();
    row = rows[first_bad];
    return first_bad;
}

// The same for all sequences, and the tokens that are known then.
template <typename T, typename Q>
__global__ __launch_bounds__(256) void decide_kernel(Args a) {
    __shared__ double table[32];
    const int64_t i = a.first + blockIdx.x;
    Chunk k;
    const int took = decide<T, Q>(a, i, draft_count(a, i), table, k);
    if (threadIdx.x == 0) {
        a.accepted[i] = took;
        if (a.rate == 0.0 || k.sum != k.sum) a.tokens[i] = k.sum != k.sum ? -1 : k.arg;
        a.rows[i] = k;
    }
}

// What a token of a sequence is drawn from: row `took` of its logits, less q where a draft was refused there.
template <typename T, typename Q>
struct Draw {
    const T* l;
    const Q* q;
    int64_t one;  // the refused draft, where its probability was 1
    Exp x;
    double inv;
};
template <typename T, typename Q>
__device__ __forceinline__ Draw<T, Q> draw_of(const Args& a, int64_t i, int n, int took, const Chunk& k) {
    return Draw<T, Q>{(const T*)a.logits + (i * (a.m + 1) + took) * a.vocab,
                      a.probs && took < n ? (const Q*)a.probs + (i * a.m + took) * a.vocab : nullptr,
                      !a.probs && took < n ? a.drafts[i * a.m + took] : -1, exp_from(k.max, a.rate), 1.0 / k.sum};
}

// The weights at 8 places of the row; p alone where there is no q, NaN among them where q has one.
template <typename T, typename Q>
__device__ __forceinline__ void weights8(const Args& a, const double* table, const Draw<T, Q>& d, int64_t e, double* w) {
    float f[kPiece], g[kPiece] = {};
    load_piece(d.l, e, a.vocab, -INFINITY, f);
    if (d.q) load_piece(d.q, e, a.vocab, 0.0f, g);
#pragma unroll
    for (int v = 0; v < kPiece; ++v) {
        const double p = exp_of(d.x, table, f[v]) * d.inv;
        w[v] = fmax(e + v == d.one ? p - 1.0 : p - (double)g[v], 0.0);  // (0 of a NaN)
    }
    bool none = false;
#pragma unroll
    for (int v = 0; v < kPiece; ++v) none |= g[v] != g[v];
    if (none) w[0] = NAN;
}

// A part's sum of weights, by a workgroup; ss: 4 values.
template <int PC, typename T, typename Q>
__device__ __forceinline__ double part_sum(const Args& a, const double* table, const Draw<T, Q>& d, int part, double* ss, int tid) {
    double sum = 0.0, w[kPiece];
#pragma unroll 1
    for (int c = 0; c < PC; ++c) {
        weights8(a, table, d, ((int64_t)part * PC + c) * kSpan + tid * kPiece, w);
#pragma unroll
        for (int v = 0; v < kPiece; ++v) sum += w[v];
    }
    return block_sum_f64(sum, ss, tid);
}

// The token, from the parts' sums in LDS, by a workgroup; -1 without a distribution.
template <int PC, typename T, typename Q>
__device__ __forceinline__ int64_t find_token(const Args& a, const double* table, Draw<T, Q> d, float u, double* sums, double* ss, int tid) {
    __shared__ int low, high, chosen;
    __shared__ double rest, ahead;
    const int lane = tid & 63, wave = tid >> 6, parts = a.parts;
    if (tid == 0) low = INT32_MAX, high = -1;
    // The part that the random number falls into, the sum ahead of it, and all weights' (by the first wave).
    auto find_part = [&]() {
        __syncthreads();
        if (wave == 0) {
            double all = 0.0;
            for (int c = lane; c < parts; c += 64) all += sums[c];
            all = wave_sum_f64(all);
            const double want = (double)u * all;
            double before = 0.0;
            int at = parts, some = 0;
            for (int c0 = 0; c0 < parts && at == parts; c0 += 64) {
                const double v = c0 + lane < parts ? sums[c0 + lane] : 0.0;
                double up = v;
                for (int d = 1; d < 64; d <<= 1) {
                    const double o = __shfl_up(up, d, 64);
                    if (lane >= d) up += o;
                }
                const uint64_t hit = ballot(v > 0.0 && before + up > want), any = ballot(v > 0.0);
                if (any) some = c0 + 63 - __builtin_clzll(any);
                if (hit) {
                    const int first = __builtin_ctzll(hit);
                    at = c0 + first;
                    before += __shfl(up - v, first, 64);
                } else {
                    before += __shfl(up, 63, 64);
                }
            }
            if (lane == 0) {
                rest = all;
                chosen = at < parts ? at : some;
                ahead = at < parts ? before : -INFINITY;  // (rounding: the last place of any weight)
            }
        }
        __syncthreads();
    };
    find_part();
    if (rest != rest) return -1;
    if (rest == 0.0) {  // q covers p: drawn from p itself
        d.q = nullptr;
        d.one = -1;
        for (int p = 0; p < parts; ++p) {
            const double sum = part_sum<PC>(a, table, d, p, ss, tid);
            if (tid == 0) sums[p] = sum;
        }
        find_part();
    }
    const double want = (double)u * rest;
    int first = INT32_MAX, last = -1;
    double before = ahead;
#pragma unroll 1
    for (int c = 0; c < PC; ++c) {  // 2,048 places at a time
        double w[kPiece], own = 0.0;
        weights8(a, table, d, ((int64_t)chosen * PC + c) * kSpan + tid * kPiece, w);
#pragma unroll
        for (int v = 0; v < kPiece; ++v) own += w[v];
        double up = own;
        for (int d = 1; d < 64; d <<= 1) {
            const double o = __shfl_up(up, d, 64);
            if (lane >= d) up += o;
        }
        if (lane == 63) ss[wave] = up;
        __syncthreads();
        double sum_to = before + (up - own);
        for (int z = 0; z < wave; ++z) sum_to += ss[z];
        before += (ss[0] + ss[1]) + (ss[2] + ss[3]);
#pragma unroll
        for (int v = 0; v < kPiece; ++v) {
            sum_to += w[v];
            const int e = (c * 256 + tid) * kPiece + v;
            if (w[v] > 0.0) {
                if (sum_to > want && e < first) first = e;
                last = e;
            }
        }
        __syncthreads();
    }
    if (first != INT32_MAX) atomicMin(&low, first);
    __syncthreads();
    if (low == INT32_MAX && last >= 0) atomicMax(&high, last);
    __syncthreads();
    return (int64_t)chosen * PC * kSpan + (low != INT32_MAX ? low : high);
}

// Part blockIdx.x % parts of a launch's sequence blockIdx.x / parts: the part's sum of weights.  64 rows of 100,277 words, bf16 logits and
// float32 probabilities: 38 MB in 12 us, 3.2 TB/s, by loads and exponentials in turn.
template <typename T, typename Q, int PC>
__global__ __launch_bounds__(256) void part_kernel(Args a) {
    __shared__ double table[32], ss[4];
    const int tid = threadIdx.x;
    const int64_t i = a.first + blockIdx.x / a.parts;
    const int s = blockIdx.x % a.parts;
    const Chunk k = a.rows[i];
    if (k.sum != k.sum) return;
    exp_table(table, tid);
    __syncthreads();
    const double sum = part_sum<PC>(a, table, draw_of<T, Q>(a, i, draft_count(a, i), a.accepted[i], k), s, ss, tid);
    if (tid == 0) a.weights[i * a.parts + s] = sum;
}

// The token of a launch's sequence blockIdx.x from its parts' sums.
template <typename T, typename Q, int PC>
__global__ __launch_bounds__(256) void token_kernel(Args a) {
    __shared__ double table[32], sums[kPartsMax], ss[4];
    const int tid = threadIdx.x;
    const int64_t i = a.first + blockIdx.x;
    const Chunk k = a.rows[i];
    if (k.sum != k.sum) return;
    for (int c = tid; c < a.parts; c += 256) sums[c] = a.weights[i * a.parts + c];
    exp_table(table, tid);
    const int64_t token = find_token<PC>(a, table, draw_of<T, Q>(a, i, draft_count(a, i), a.accepted[i], k), a.u_sample[i], sums, ss, tid);
    if (tid == 0) a.tokens[i] = token;
}

// All three in one launch for few sequences: each workgroup decides by itself which row its part is of, and the
// sequence's last one to come here finds the token.  (For many, a launch each: a workgroup that says that it is done waits
// for the caches, some 0.2 us one after the other on an XCD.  64 sequences of 100,277 words: 85 us in one launch, and in three 4.7,
// 12 and 7.3.)
template <typename T, typename Q>
__global__ __launch_bounds__(256) void draw_kernel(Args a) {
    __shared__ double table[32], sums[kPartsMax], ss[4];
    __shared__ int turn;
    const int tid = threadIdx.x, parts = a.parts;
    const int64_t i = blockIdx.x / parts;
    const int s = blockIdx.x % parts, n = draft_count(a, i);
    Chunk k;
    const int took = decide<T, Q>(a, i, n, table, k);
    if (s == 0 && tid == 0) {
        a.accepted[i] = took;
        if (k.sum != k.sum) a.tokens[i] = -1;
    }
    if (k.sum != k.sum) return;
    const Draw<T, Q> d = draw_of<T, Q>(a, i, n, took, k);
    const double sum = part_sum<1>(a, table, d, s, ss, tid);
    if (tid == 0) {
        __hip_atomic_store(&a.weights[i * parts + s], sum, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        turn = __hip_atomic_fetch_add(&a.done[i], 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (turn != parts - 1) return;
    for (int c = tid; c < parts; c += 256) sums[c] = __hip_atomic_load(&a.weights[i * parts + c], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    const int64_t token = find_token<1>(a, table, d, a.u_sample[i], sums, ss, tid);
    if (tid == 0) a.tokens[i] = token;
}

// Chunks of 8,192 values, which spare sums and maxima of a workgroup and joins of chunks; of 2,048 where there are fewer than
// CUs.  us with 8,192 | 2,048, rows of 100,277, a call: 320 rows 55.7 | 62.3, 160 37.0 | 39.1, 80 27.4 | 28.5; its kernels' sum:
// 40 rows 26.2 | 26.5, 20 20.7 | 20.8, 5 17.4 | 17.0, one 15.9 | 13.9.
int chunk_pieces(int64_t rows, int64_t vocab, int num_cus) { return rows * ((vocab + 4 * kSpan - 1) / (4 * kSpan)) >= num_cus ? 4 : 1; }
// Parts of 2,048 values, of 32,768 where they would be too many to list.
int part_pieces(int64_t vocab) { return vocab <= (int64_t)kPartsMax * kSpan ? 1 : 16; }
int pieces_in(int64_t vocab, int pieces) { return (int)((vocab + (int64_t)pieces * kSpan - 1) / ((int64_t)pieces * kSpan)); }
size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

// `each` workgroups for each of n rows or sequences, in as many launches as that takes.
template <typename K>
void launch(K kernel, Args a, int64_t n, int each, hipStream_t stream) {
    const int64_t most = kLaunchGroups / each;
    for (a.first = 0; a.first < n; a.first += most) {
        const int64_t here = n - a.first < most ? n - a.first : most;
        hipLaunchKernelGGL(kernel, dim3((unsigned)(here * each)), dim3(256), 0, stream, a);
    }
}

template <typename T, typename Q>
void launch_draw(const Args& a, int64_t n_seq, hipStream_t stream) {
    if (a.rate != 0.0 && a.part_pieces == 1 && n_seq * a.parts <= a.own_parts) return launch(draw_kernel<T, Q>, a, n_seq, a.parts, stream);
    launch(decide_kernel<T, Q>, a, n_seq, 1, stream);
    if (a.rate == 0.0) return;
    if (a.part_pieces == 1) {
        launch(part_kernel<T, Q, 1>, a, n_seq, a.parts, stream);
        launch(token_kernel<T, Q, 1>, a, n_seq, 1, stream);
    } else {
        launch(part_kernel<T, Q, 16>, a, n_seq, a.parts, stream);
        launch(token_kernel<T, Q, 16>, a, n_seq, 1, stream);
    }
}

template <typename T>
void launch_all(const Args& a, int64_t n_seq, int probs_dtype, int pieces, hipStream_t stream) {
    const int64_t rows = n_seq * (a.m + 1);
    if (a.rate == 0.0) launch(chunk_kernel<T, 4, true>, a, rows, a.chunks, stream);
    else if (pieces == 4) launch(chunk_kernel<T, 4, false>, a, rows, a.chunks, stream);
    else launch(chunk_kernel<T, 1, false>, a, rows, a.chunks, stream);
    if (probs_dtype == kBF16) launch_draw<T, uint16_t>(a, n_seq, stream);
    else launch_draw<T, float>(a, n_seq, stream);
}

}  // namespace

size_t verify_workspace_bytes(int64_t n_seq, int n_drafts, int64_t vocab, int num_cus) {
    const int64_t rows = n_seq * (n_drafts + 1);
    // (chunks: of any temperature)
    return round256((size_t)rows * pieces_in(vocab, chunk_pieces(rows, vocab, num_cus)) * sizeof(Chunk)) + round256((size_t)n_seq * sizeof(Chunk)) +
           round256((size_t)n_seq * pieces_in(vocab, part_pieces(vocab)) * 8) + round256((size_t)n_seq * 4);
}

int launch_verify(const void* logits, const int64_t* drafts, const void* probs, int probs_dtype, const int32_t* counts,
                  const float* u_accept, const float* u_sample, int64_t n_seq, int n_drafts, int64_t vocab, double temperature, int dtype,
                  void* ws, int32_t* accepted, int64_t* tokens, int num_cus, hipStream_t stream) {
    const int64_t rows = n_seq * (n_drafts + 1);
    const int pieces = temperature > 0.0 ? chunk_pieces(rows, vocab, num_cus) : 4;
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
    a.chunks = pieces_in(vocab, pieces);
    a.part_pieces = part_pieces(vocab);
    a.parts = pieces_in(vocab, a.part_pieces);
    // us with the decision by itself | in every part's workgroup, four drafts of rows of 100,277: 1 sequence (49 parts) 24.8 | 20.8,
    // 4 24.3 | 20.5, 8 24.4 | 25.0, 16 28.5 | 37.8, 64 54 | 125.
    a.own_parts = 2 * num_cus;
    unsigned char* w = (unsigned char*)ws;
    a.stats = (Chunk*)w;
    w += round256((size_t)rows * a.chunks * sizeof(Chunk));
    a.rows = (Chunk*)w;
    w += round256((size_t)n_seq * sizeof(Chunk));
    a.weights = (double*)w;
    w += round256((size_t)n_seq * a.parts * 8);
    a.done = (int32_t*)w;
    a.accepted = accepted;
    a.tokens = tokens;
    if (dtype == kBF16) launch_all<uint16_t>(a, n_seq, probs_dtype, pieces, stream);
    else launch_all<float>(a, n_seq, probs_dtype, pieces, stream);
    return (int)hipGetLastError();
}

}  // namespace ethos

// Softmax cross entropy of rows h against a head matrix W [vocab, d], and its gradients, without
// the logits in memory:
//   l_iv = h_i . W_v,  lse_i = log sum_v exp(l_iv),  loss_i = lse_i - l_i,label,
//   dl_iv = g_i (exp(l_iv - lse_i) - [v = label_i]),  dh = dl W,  dW = dl^T h.
//
// Rows without a label (ignore_index) are left out before anything else: the rows with one are
// copied into a dense block (zero-padded to whole tiles), which every product reads; their count
// stays on the device.  The forward product keeps a maximum and a sum of exponentials per row and tile
// of vocabulary.  The backward forms the logits of a piece of the vocabulary again, turns them into dl
// (bf16) in its epilogue, and multiplies the piece by h and by W.
//
// bf16, where dl of the whole vocabulary is at most what a piece may take: the forward under gradients leaves the
// exponentials behind, in the memory that dl would take in the backward anyway (here held from the forward on), and the
// backward turns them into dl in place instead of forming the logits again (4,096 rows of 1,024 over 100,277 words: 270 to
// 298 us against 878 on the average).  They are fp16 values relative to the maximum of their row's B / 2 words, so at most
// 1 but for kScaled's factor: off by 2^-11 of their size, or by 2^-25 of the maximum's, against the 2^-8 of dl's own
// rounding to bf16.
//
// float32 operands go through the same kernels as three bf16 planes each, x = hi + mid + lo
// (ethos_split.hpp): a product is six bf16 products, each exact in float32, the lower five in a sum of their own or (in
// tiles of 256) the smallest first.
#include <type_traits>

#include "ethos_common.hpp"
#include "ethos_mfma.hpp"
#include "ethos_rows.hpp"
#include "ethos_split.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
// exp(l - x) is taken as exp2(l log2(e) - RN(x log2(e))) where |x| is below this: at l = x that is not 1 but 2^r, with r
// the rounding of x log2(e), here within 2^-14 (a factor of 4e-5 and less, as much as float32 rounds a logit of that size
// by; at 1e10 r is in the hundreds).  Beyond it x is subtracted first, which is exact near l = x and below it never positive.
constexpr float kScaled = 1024.0f;
constexpr int kPadRows = 256;  // labelled rows are padded with zero rows to a multiple of this

__host__ __device__ constexpr int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

constexpr int planes_of(int dtype) { return dtype == kBF16 ? 1 : 3; }

// What the forward leaves for the backward.
struct CeState {
    int32_t* count;  // labelled rows
    int32_t* idx;    // labelled row -> row of h
    int32_t* inv;    // row of h -> labelled row or -1
    int32_t* lab;    // label of a labelled row (-1: outside the vocabulary)
    float* lse;      // log of the sum of exponentials
    float* ll;       // logit of the label
    uint16_t* h;     // the labelled rows [planes][padded n][ldh]
    int32_t* ticket; // of the workgroups that finish the loss
    int64_t np;      // n padded
    int ldh;
    size_t bytes;
};
CeState ce_state(char* p, int64_t n, int d, int dtype) {
    CeState s;
    s.np = round_up(n, kPadRows);
    s.ldh = (int)round_up(d, 64);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char* r = p + at;
        at += (bytes + 255) / 256 * 256;
        return r;
    };
    s.count = (int32_t*)take(8);
    s.idx = (int32_t*)take(s.np * 4);
    s.inv = (int32_t*)take(s.np * 4);
    s.lab = (int32_t*)take(s.np * 4);
    s.lse = (float*)take(s.np * 4);
    s.ll = (float*)take(s.np * 4);
    s.h = (uint16_t*)take((size_t)s.np * s.ldh * 2 * planes_of(dtype));
    s.ticket = s.count + 1;
    s.bytes = at;
    return s;
}

// ------------------------------------------------------------------------ labelled rows
// One workgroup: the rows with a label, in order; loss (when a row's loss is asked for) is zero
// for the others.
__global__ __launch_bounds__(1024) void ce_rows_kernel(const int64_t* __restrict__ labels, int64_t n, int64_t vocab, int64_t ignore,
                                                       int32_t* __restrict__ count, int32_t* __restrict__ idx,
                                                       int32_t* __restrict__ inv, int32_t* __restrict__ lab,
                                                       float* __restrict__ loss_rows, int32_t* __restrict__ ticket) {
    __shared__ int32_t sums[2][16];
    const int tid = threadIdx.x, wave = tid >> 6;
    constexpr int C = 8;  // labels a thread asks for at once
    int32_t base = 0;
    for (int64_t i0 = 0; i0 < n; i0 += C * 1024) {
        int64_t l[C];
#pragma unroll
        for (int c = 0; c < C; ++c) l[c] = i0 + c * 1024 + tid < n ? labels[i0 + c * 1024 + tid] : ignore;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            const int64_t i = i0 + c * 1024 + tid;
            if (i0 + c * 1024 >= n) break;
            const bool use = l[c] != ignore;
            const uint64_t m = ballot(use);
            if ((tid & 63) == 0) sums[c & 1][wave] = __popcll(m);
            __syncthreads();
            int32_t before = base, all = 0;
            for (int w = 0; w < 16; ++w) {
                if (w < wave) before += sums[c & 1][w];
                all += sums[c & 1][w];
            }
            if (i < n) {
                const int32_t at = before + count_below(m);
                inv[i] = use ? at : -1;
                if (use) {
                    idx[at] = (int32_t)i;
                    lab[at] = l[c] >= 0 && l[c] < vocab ? (int32_t)l[c] : -1;
                } else if (loss_rows) {
                    loss_rows[i] = 0.0f;
                }
            }
            base += all;
        }
        __syncthreads();
    }
    if (tid == 0) {
        *count = base;
        *ticket = 0;
    }
}

// Eight values of T as bf16 planes, `stride` values apart.
__device__ __forceinline__ void put_planes(const uint16_t* src, uint16_t* out, int64_t) {
    *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(src);
}
__device__ __forceinline__ void put_planes(const float* src, uint16_t* out, int64_t stride) {
    const float4 a = reinterpret_cast<const float4*>(src)[0], b = reinterpret_cast<const float4*>(src)[1];
    uint4 p[3];
    split3(a.x, a.y, p[0].x, p[1].x, p[2].x);
    split3(a.z, a.w, p[0].y, p[1].y, p[2].y);
    split3(b.x, b.y, p[0].z, p[1].z, p[2].z);
    split3(b.z, b.w, p[0].w, p[1].w, p[2].w);
#pragma unroll
    for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(out + i * stride) = p[i];
}
__device__ __forceinline__ float dot8(const uint16_t* a, const uint16_t* b, float s) {
    float x[8], y[8];
    Vec16<uint16_t>::unpack(*reinterpret_cast<const uint4*>(a), x);
    Vec16<uint16_t>::unpack(*reinterpret_cast<const uint4*>(b), y);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(x[j], y[j], s);
    return s;
}
__device__ __forceinline__ float dot8(const float* a, const float* b, float s) {
#pragma unroll
    for (int j = 0; j < 8; ++j) s = __builtin_fmaf(a[j], b[j], s);
    return s;
}

// Row r of the dense block: row `row` of h (negative: zeros), and its label's logit.
template <typename T>
__device__ __forceinline__ void ce_gather_row(const T* h, int64_t ld, const T* w, int64_t row, int label, int64_t r, int d, int ldh,
                                              int64_t plane, uint16_t* out, float* ll, int lane) {
    const T* src = h + (row < 0 ? 0 : row) * ld;
    const T* word = w + (int64_t)(label < 0 ? 0 : label) * d;
    float s = 0.0f;
    for (int c = lane * 8; c < ldh; c += 64 * 8) {
        uint16_t* o = out + r * ldh + c;
        if (row >= 0 && c < d) {
            put_planes(src + c, o, plane);
            if (label >= 0) s = dot8(src + c, word + c, s);
        } else {
#pragma unroll
            for (int i = 0; i < (sizeof(T) == 2 ? 1 : 3); ++i) *reinterpret_cast<uint4*>(o + i * plane) = make_uint4(0, 0, 0, 0);
        }
    }
    s = wave_sum(s);
    if (lane == 0) ll[r] = label >= 0 ? s : __builtin_nanf("");
}

// A wave per row of the dense block.
template <typename T>
__global__ __launch_bounds__(256) void ce_gather_kernel(const T* __restrict__ h, int64_t ld, const T* __restrict__ w,
                                                        const int32_t* __restrict__ count, const int32_t* __restrict__ idx,
                                                        const int32_t* __restrict__ lab, int d, int ldh, int64_t plane,
                                                        uint16_t* __restrict__ out, float* __restrict__ ll) {
    const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t m = *count;
    if (r >= round_up(m, kPadRows)) return;
    ce_gather_row(h, ld, w, r < m ? (int64_t)idx[r] : -1, r < m ? lab[r] : -1, r, d, ldh, plane, out, ll, threadIdx.x & 63);
}

// Both steps for up to kFewRows rows, in one launch: every workgroup finds the labelled rows itself.
constexpr int kFewRows = 1024;
template <typename T>
__global__ __launch_bounds__(256) void ce_few_rows_kernel(const int64_t* __restrict__ labels, int n, int64_t vocab, int64_t ignore,
                                                          const T* __restrict__ h, int64_t ld, const T* __restrict__ w,
                                                          int32_t* __restrict__ count, int32_t* __restrict__ idx,
                                                          int32_t* __restrict__ inv, int32_t* __restrict__ lab,
                                                          float* __restrict__ loss_rows, int32_t* __restrict__ ticket, int d, int ldh,
                                                          int64_t plane, uint16_t* __restrict__ out, float* __restrict__ ll) {
    __shared__ int32_t sums[4];
    __shared__ int32_t rows[kFewRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const bool first = blockIdx.x == 0;
    int64_t l[kFewRows / 256];
#pragma unroll
    for (int c = 0; c < kFewRows / 256; ++c) l[c] = c * 256 + tid < n ? labels[c * 256 + tid] : ignore;
    int32_t m = 0;
#pragma unroll
    for (int c = 0; c < kFewRows / 256; ++c) {
        if (c * 256 >= n) break;
        const int i = c * 256 + tid;
        const bool use = l[c] != ignore;
        const uint64_t mask = ballot(use);
        if (lane == 0) sums[wave] = __popcll(mask);
        __syncthreads();
        int32_t at = m + count_below(mask);
        for (int v = 0; v < 4; ++v) {
            if (v < wave) at += sums[v];
            m += sums[v];
        }
        if (use) rows[at] = i;
        if (first && i < n) {
            inv[i] = use ? at : -1;
            if (use) {
                idx[at] = i;
                lab[at] = l[c] >= 0 && l[c] < vocab ? (int32_t)l[c] : -1;
            } else if (loss_rows) {
                loss_rows[i] = 0.0f;
            }
        }
        __syncthreads();
    }
    if (first && tid == 0) {
        *count = m;
        *ticket = 0;
    }
    const int r = blockIdx.x * 4 + wave;
    if (r >= round_up(m, kPadRows)) return;
    const int row = r < m ? rows[r] : -1;
    const int64_t label = row >= 0 ? labels[row] : -1;
    ce_gather_row(h, ld, w, row, label >= 0 && label < vocab ? (int32_t)label : -1, r, d, ldh, plane, out, ll, lane);
}

// W's planes, eight values a thread.
__global__ __launch_bounds__(256) void ce_split_kernel(const float* __restrict__ w, int64_t n8, uint16_t* __restrict__ out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n8; i += (int64_t)gridDim.x * 256)
        put_planes(w + i * 8, out + i * 8, n8 * 8);
}

// ------------------------------------------------------------------------ sums over the vocabulary
struct MaxSum {
    float m, s;  // maximum and the sum of exp(x - m); an empty set has m = -inf, s = 0
};
__device__ __forceinline__ MaxSum join(MaxSum a, MaxSum b) {
    const float m = fmaxf(a.m, b.m);
    const float z = m == -__builtin_inff() ? 0.0f : m;  // (-inf) - (-inf)
    return {m, a.s * __builtin_amdgcn_exp2f((a.m - z) * kLog2e) + b.s * __builtin_amdgcn_exp2f((b.m - z) * kLog2e)};
}

// lse and loss of each labelled row from its partial (maximum, sum) pairs part[e][np], e < n_part; 16 rows
// a workgroup, whose 64 groups of 16 lanes take every 64th pair.  A sum or mean over the rows: the workgroup
// that finishes last adds up the row losses in their order.
__global__ __launch_bounds__(1024) void ce_lse_kernel(const float2* __restrict__ part, int n_part, int64_t np,
                                                      const int32_t* __restrict__ count, const int32_t* __restrict__ idx,
                                                      const float* __restrict__ ll, int reduction, float* __restrict__ lse,
                                                      float* row_loss, int32_t* ticket, float* __restrict__ loss) {
    __shared__ MaxSum lds[16][16];
    __shared__ double sums[16];
    __shared__ bool last;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave * 4 + (lane >> 4);
    const int64_t r = (int64_t)blockIdx.x * 16 + (lane & 15);
    constexpr int C = 8;  // pairs asked for at once, before the count is known (rows past it are memory of the same array)
    float2 p[C];
    auto ask = [&](int e) {
#pragma unroll
        for (int j = 0; j < C; ++j) p[j] = part[(int64_t)(e + j * 64 < n_part ? e + j * 64 : n_part - 1) * np + r];
    };
    ask(first);
    const float x = ll[r];
    const int64_t m = *count;
    const int64_t row = reduction == kLossNone && r < m ? idx[r] : 0;
    MaxSum a = {-__builtin_inff(), 0.0f};
    for (int e = first; e < n_part; e += 64 * C) {
        if (e != first) ask(e);
        MaxSum b = {p[0].x, 0.0f};
#pragma unroll
        for (int j = 1; j < C; ++j) b.m = fmaxf(b.m, p[j].x);
        const float z = b.m == -__builtin_inff() ? 0.0f : b.m;
#pragma unroll
        for (int j = 0; j < C; ++j)
            if (e + j * 64 < n_part) b.s += p[j].y * __builtin_amdgcn_exp2f((p[j].x - z) * kLog2e);
        a = join(a, b);
    }
    a = join(a, {__shfl_xor(a.m, 16), __shfl_xor(a.s, 16)});
    a = join(a, {__shfl_xor(a.m, 32), __shfl_xor(a.s, 32)});
    if (lane < 16) lds[wave][lane] = a;
    __syncthreads();
    float out = 0.0f;
    if (wave == 0) {
        // the 16 waves' pairs of a row over four lanes each, then over those
        a = lds[lane >> 4][lane & 15];
        for (int w = 4; w < 16; w += 4) a = join(a, lds[w + (lane >> 4)][lane & 15]);
        a = join(a, {__shfl_xor(a.m, 16), __shfl_xor(a.s, 16)});
        a = join(a, {__shfl_xor(a.m, 32), __shfl_xor(a.s, 32)});
        const float sum = a.m + __builtin_amdgcn_logf(a.s) * 0.69314718055994530942f;
        // The label's logit x is summed in another order than the products: where it is all of the sum, it may come out
        // above it, which it never is.  (A NaN of either stays.)
        const float l = x != x || sum < x ? x : sum;
        out = l - x;
        if (lane < 16 && r < m) {
            lse[r] = l;
            if (reduction == kLossNone) loss[row] = out;
            else if (gridDim.x > 1) __hip_atomic_store(row_loss + r, out, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
    }
    if (reduction == kLossNone) return;
    double s = 0.0;
    if (gridDim.x == 1) {
        if (wave != 0) return;
        s = lane < 16 && r < m ? (double)out : 0.0;
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o);
        if (lane == 0) *loss = (float)(reduction == kLossMean ? s / (double)m : s);
        return;
    }
    __syncthreads();
    if (threadIdx.x == 0)
        last = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_ACQ_REL, __HIP_MEMORY_SCOPE_AGENT) == (int32_t)gridDim.x - 1;
    __syncthreads();
    if (!last) return;
    for (int64_t i = threadIdx.x; i < m; i += 1024) s += (double)__hip_atomic_load(row_loss + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += sums[i];
        *loss = (float)(reduction == kLossMean ? t / (double)m : t);
    }
}

// g of a labelled row: the loss's gradient, per row of h or of the whole.
__device__ __forceinline__ float row_gradient(const float* dloss, const int32_t* idx, int64_t r, int64_t m, int reduction) {
    return reduction == kLossNone ? dloss[idx[r]] : reduction == kLossMean ? *dloss / (float)m : *dloss;
}

// The first labelled row's g without its power of two.  dl is held in units of it, and the gradients are multiplied by it
// last, in float32: where all rows have one g (a mean, or equal weights), a label's dl of nearly -g would otherwise be
// rounded alike in every row, and whole gradients be off by up to the half step of bf16 (2^-8; error against float64
// 3.0e-3 for a mean over a third of 1,777 rows, with it 1.8e-3).  What is left of the kind is the rounding of 1 - p: where
// labels have one probability p below 2^-8, it is rounded alike too, by less than p and at most 2^-9, no more than the
// results' own rounding.
__device__ __forceinline__ float gradient_unit(const float* dloss, const int32_t* idx, int64_t m, int reduction) {
    if (m == 0) return 1.0f;
    const uint32_t b = __float_as_uint(row_gradient(dloss, idx, 0, m, reduction)), e = b & 0x7f800000u;
    return e == 0 || e == 0x7f800000u ? 1.0f : __uint_as_float((b & 0x007fffffu) | 0x3f800000u);
}

// ------------------------------------------------------------------------ products
// C[m][n] = sum_k A(m, k) B(k, n) in tiles of B x B (256: eight waves, two along m and four along n, 128 x 64 each;
// 128: four waves of 64 x 64, or eight of 64 x 32), k in steps of kK.  float32 operands are
// PL = 3 bf16 planes each: a step of tiles of 128 has all of them (P = 3) and takes every pair's products from it; tiles of
// 256, for which LDS has no room, go over the operands once for each pair (500 x 256 x 8,009: gradients 29 us against 38 with
// passes, logits 17.5 and 20).  Operands go from memory
// straight into LDS, which holds S steps: the one that is multiplied and those on their way.  An operand is stored with k
// contiguous ("K": rows of m or n) or with k as the row ("R"); R tiles are read with the transposing LDS
// loads.  LDS rows of a K tile are 64 k (8 pieces of 16 bytes, their places by k_piece); of an R
// tile B columns (B / 8 pieces), piece c at c ^ 4 (k % 4): 16 lanes' reads touch all banks.
constexpr int kTileMax = 256;
// dl is stored in panels of 256 words, [panel][np][256], so that a tile of it is one stretch of memory (with the rows of
// the whole piece, 200 KB apart, a tile is spread over as many pages: 920 us for 4,096 rows against 905)
constexpr int kPanel = 256;
constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer's end: reads zeros

// float32: the pairs of planes, (0, 0) into one sum and (0, 1), (1, 0), (1, 1), (0, 2), (2, 0), whose products are 2^-8 of
// that and less, into another.  The three left out, mid x lo, lo x mid and lo x lo, are at most 2^-22 of a product and
// 2^-26 on the root mean square, below the rounding of a float32 sum of 16 such products; a third of the products' time.
constexpr int kPairs = 6;
constexpr uint32_t kPairsA = 0x201100, kPairsB = 0x021010;

template <int TB, int TS, int TP> struct Tile {
    static constexpr int B = TB, S = TS, P = TP;
    static constexpr int kWaves = B == 256 || S == 4 || P > 1 ? 8 : 4, kThreads = kWaves * 64;
    static constexpr int kWN = kWaves / 2;                           // waves along n (two along m)
    static constexpr int kMI = B / 64, kNI = B / kWN / 32;           // MFMA tiles of a wave
    static constexpr int kK = P == 1 ? 64 : 32;                      // step of the reduction
    static constexpr int kPlane = B * kK * 2;                        // a plane of one operand's step
    static constexpr int kBytes = P * kPlane;                        // one operand's step
    static constexpr int kCopies = kBytes / 1024 / kWaves;           // copies of a wave per operand and step
    static constexpr int kLds = S * 2 * kBytes;
    static constexpr int kRowsLds = kWaves * 4096;                   // the logits' epilogue: 4 KB a wave
};

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(3))) bf16x8_t* lds_frag_ptr;
typedef __attribute__((address_space(3))) s16x4_t* lds_tr_ptr;

// One operand: where its tiles are in memory.
struct Feed {
    uint64_t base;  // address of the next step
    int64_t left;   // bytes from there to the operand's end
    int64_t step;   // bytes from a step to the next
    int k_left;     // K: k from the next step's first to the end
    uint32_t off[4];  // this lane's offsets in a plane (kCopies / P of them)
    int64_t plane;  // bytes from a plane to the next
    int64_t jump;   // dl by rows: bytes to the next panel, taken after the panel's last step
    int at;         // steps taken in the panel
    uint64_t base0;  // passes over the planes: the first plane's first step
    int64_t left0;
    int k0, at0;
};

// The piece of a K tile's row (of K k) at place c, and the other way round.
template <int K = 64>
__device__ __forceinline__ int k_piece(int row, int c) {
    return K == 64 ? c ^ ((row >> 1) & 7) : c ^ ((row >> 2) & 3);
}

template <typename Ti, bool KC>
__device__ __forceinline__ void feed_init(Feed& f, const uint16_t* p, int64_t bytes, int64_t ld, int k, int cols, int64_t plane,
                                          int wave, int lane) {
    f.base = f.base0 = (uint64_t)p;
    f.left = f.left0 = bytes;
    f.step = KC ? Ti::kK * 2 : Ti::kK * ld * 2;
    f.k_left = f.k0 = k;
    f.plane = plane * 2;
    f.jump = 0;
    f.at = f.at0 = 0;
#pragma unroll
    for (int j = 0; j < Ti::kCopies / Ti::P; ++j) {
        const int slot = (j * Ti::kWaves + wave) * 64 + lane;
        if (KC) {
            const int row = slot / (Ti::kK / 8), c = k_piece<Ti::kK>(row, slot % (Ti::kK / 8));
            f.off[j] = (uint32_t)(row * ld * 2 + c * 16);
        } else {
            const int kk = slot / (Ti::B / 8), c = (slot % (Ti::B / 8)) ^ ((kk & 3) << 2);
            f.off[j] = c * 8 < cols ? (uint32_t)(kk * ld * 2 + c * 16) : kOutside;
        }
    }
}

// Back to the first step, of plane p.
__device__ __forceinline__ void feed_plane(Feed& f, int p) {
    f.base = f.base0 + (uint64_t)(p * f.plane);
    f.left = f.left0;
    f.k_left = f.k0;
    f.at = f.at0;
}

// The next step's tile into LDS at `lds`: one of the wave's copies, or all of them and on to the step after.
template <typename Ti, bool KC>
__device__ __forceinline__ void feed_copy(const Feed& f, int j, uint32_t lds, int wave, int lane) {
    constexpr int kEach = Ti::kCopies / Ti::P;  // copies of a plane
    const int64_t left = f.left < 0 ? 0 : f.left > 0x7fffffff ? 0x7fffffff : f.left;
    uint32_t off = f.off[j % kEach];
    if (KC && f.k_left < Ti::kK) {
        const int slot = (j % kEach * Ti::kWaves + wave) * 64 + lane;
        off = k_piece<Ti::kK>(slot / (Ti::kK / 8), slot % (Ti::kK / 8)) * 8 < f.k_left ? off : kOutside;
    }
    lds_dma16(buffer_rsrc((const void*)(f.base + j / kEach * f.plane), (uint32_t)left), (int)off, 0,
              __builtin_amdgcn_readfirstlane(lds + (j * Ti::kWaves + wave) * 1024));
}
template <typename Ti>
__device__ __forceinline__ void feed_advance(Feed& f) {
    f.base += f.step;
    f.left -= f.step;
    f.k_left -= Ti::kK;
    if (++f.at == kPanel / Ti::kK) {
        f.at = 0;
        f.base += f.jump;
        f.left -= f.jump;
    }
}

// Fragments of 32 rows (or columns) i at row0 + 32 i, reduction step s of 16.
template <typename Ti, bool KC, int N> struct Reader {
    static constexpr int K = Ti::kK, B = Ti::B;
    uint32_t at[KC ? K / 16 : N];
    __device__ __forceinline__ void init(int row0, int lane) {
        if constexpr (KC) {
            const int row = row0 + (lane & 31);
#pragma unroll
            for (int s = 0; s < K / 16; ++s) at[s] = row * (K * 2) + (k_piece<K>(row, 2 * s + (lane >> 5)) << 4);
        } else {
            const int k = 8 * (lane >> 5) + ((lane & 15) >> 2);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (row0 + 32 * i) / 8 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
                at[i] = k * (B * 2) + ((c ^ ((k & 3) << 2)) << 4) + (lane & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ bf16x8_t get(uint32_t lds, int i, int s) const {
        if constexpr (KC) {
            return *(lds_frag_ptr)(size_t)(lds + at[s] + i * (K * 64));
        } else {
            union {
                s16x4_t h[2];
                bf16x8_t f;
            } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(lds + at[i] + s * (B * 32)));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(lds + at[i] + s * (B * 32) + B * 8));
            return u.f;
        }
    }
};

// This wave's copies but the last N have landed and its LDS reads are done, and so with every wave.
template <int N = 0>
__device__ __forceinline__ void step_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }

// The same of LDS accesses alone.
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// A tile's operands, and with passes over their planes the present one.
struct Pair {
    Feed a, b;
    int64_t steps, in;  // steps of a pass; taken of the present one
    int pass;
};

template <typename Ti, bool AK, bool BK>
__device__ __forceinline__ void tile_copy(const Pair& p, uint32_t to, int c, int wave, int lane) {
    constexpr int C = Ti::kCopies;
    if (c < C) feed_copy<Ti, AK>(p.a, c, to, wave, lane);
    else feed_copy<Ti, BK>(p.b, c - C, to + Ti::kBytes, wave, lane);
}

// Pass i: the pairs from the lowest up.
__device__ __forceinline__ void tile_pass(Pair& p, int i) {
    p.in = 0;
    p.pass = i;
    feed_plane(p.a, (int)(kPairsA >> (4 * (kPairs - 1 - i))) & 3);
    feed_plane(p.b, (int)(kPairsB >> (4 * (kPairs - 1 - i))) & 3);
}

template <typename Ti, int PL>
__device__ __forceinline__ void tile_advance(Pair& p) {
    feed_advance<Ti>(p.a);
    feed_advance<Ti>(p.b);
    if (PL > Ti::P && ++p.in == p.steps && p.pass + 1 < kPairs) tile_pass(p, p.pass + 1);
}

// The copies of a tile's first S steps (or those it has).
template <typename Ti, int PL, bool AK, bool BK>
__device__ __forceinline__ void tile_begin(Pair& p, int64_t steps, uint32_t lds, int wave, int lane) {
    p.steps = steps;
    if (PL > Ti::P) tile_pass(p, 0);
    const int64_t total = PL > Ti::P ? steps * kPairs : steps;
    const int n = total < Ti::S ? (int)total : Ti::S;
    for (int t = 0; t < n; ++t) {
#pragma unroll
        for (int c = 0; c < 2 * Ti::kCopies; ++c) tile_copy<Ti, AK, BK>(p, lds + t * 2 * Ti::kBytes, c, wave, lane);
        tile_advance<Ti, PL>(p);
    }
}

// The tile's products, after tile_begin, whose copies every wave has waited for.  Between the products of 16 k stand
// the LDS reads of the next 16, one at a time; the step's barrier stands before its last products, which cover the first
// reads of the next step and the copies into the step just freed.  (Reads and copies in a row before the products: 54% of
// the matrix pipes' cycles used at 2.0 GHz; so: 72% at 1.78 GHz, which the power allows; with no copies at all 81% at
// 1.82 GHz.)
template <typename Ti, int PL, bool AK, bool BK>
__device__ __forceinline__ void tile_run(Pair& p, uint32_t lds, f32x16_t (&acc)[Ti::kMI][Ti::kNI], int wave, int lane) {
    constexpr int B = Ti::B, S = Ti::S, P = Ti::P, MI = Ti::kMI, NI = Ti::kNI, C = Ti::kCopies, Q = (P == 1 ? 1 : kPairs) * MI * NI;
    constexpr int kReads = P * (MI + NI), kLast = Ti::kK / 16 - 1;
    Reader<Ti, AK, MI> ra;
    Reader<Ti, BK, NI> rb;
    ra.init(wave / Ti::kWN * (B / 2), lane);
    rb.init(wave % Ti::kWN * (32 * NI), lane);
    f32x16_t low[MI][NI];  // float32: the sum of the lower pairs
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = low[i][j] = f32x16_zero();
    if (p.steps <= 0) return;
    bf16x8_t a[2][P][MI], b[2][P][NI];
    // read r of 16 k: in the order in which the products take them
    auto read = [&](uint32_t from, int s, int r) {
        if (r >= kReads) return;
        const int l = r / (MI + NI), w = r % (MI + NI);
        if (w == 0) a[s & 1][l][0] = ra.get(from + l * Ti::kPlane, 0, s);
        else if (w <= NI) b[s & 1][l][w - 1] = rb.get(from + Ti::kBytes + l * Ti::kPlane, w - 1, s);
        else a[s & 1][l][w - NI] = ra.get(from + l * Ti::kPlane, w - NI, s);
    };
    // the products of 16 k, after each of which `between(q)` is issued
    auto multiply = [&](int s, auto between) {
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const int pair = q / (MI * NI), i = q / NI % MI, j = q % NI;
            const int la = kPairsA >> (4 * pair) & 3, lb = kPairsB >> (4 * pair) & 3;
            f32x16_t& c = pair == 0 ? acc[i][j] : low[i][j];
            c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[s & 1][la][i], b[s & 1][lb][j], c, 0, 0, 0);
            between(q);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr int R = (kReads + Q - 1) / Q;  // reads after a product
    const int64_t total = PL > Ti::P ? p.steps * kPairs : p.steps;
#pragma unroll
    for (int r = 0; r < kReads; ++r) read(lds, 0, r);
    uint32_t cur = 0, from = lds, next = lds + 2 * Ti::kBytes;
    auto flip = [&]() {
        cur = (cur + 1) % S;
        from = lds + cur * 2 * Ti::kBytes;
        next = lds + (cur + 1) % S * 2 * Ti::kBytes;
    };
    auto head = [&]() {  // all but the step's last products
#pragma unroll
        for (int s = 0; s < kLast; ++s)
            multiply(s, [&](int q) {
#pragma unroll
                for (int r = 0; r < R; ++r) read(from, s + 1, q * R + r);
            });
    };
    for (int64_t t = S; t < total; ++t) {
        head();
        if (t < 2 * S - 1) lds_barrier();  // (the first S steps are there; stores before them may still be on their way)
        else step_barrier<2 * C * (S - 2)>();
        multiply(kLast, [&](int q) {
            constexpr int N = (2 * C + Q - 1) / Q;  // copies after a product
#pragma unroll
            for (int r = 0; r < R; ++r) read(next, 0, q * R + r);
#pragma unroll
            for (int c = 0; c < N; ++c)
                if (q * N + c < 2 * C) tile_copy<Ti, AK, BK>(p, from, q * N + c, wave, lane);
        });
        tile_advance<Ti, PL>(p);
        flip();
    }
    // the steps that are in LDS or on their way (the last one's reads of a next step go unused)
    for (int t = total < Ti::S ? (int)total : S; t > 0; --t) {
        head();
        if (S == 4 && t == 4) step_barrier<4 * C>();
        else if (S == 4 && t == 3) step_barrier<2 * C>();
        else step_barrier();
        multiply(kLast, [&](int q) {
#pragma unroll
            for (int r = 0; r < R; ++r) read(next, 0, q * R + r);
        });
        flip();
    }
    if constexpr (P > 1) {
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                acc[i][j] += low[i][j];
                asm volatile("" : "+v"(acc[i][j]));  // (one value from here on: the compiler would keep both sums for the epilogue)
            }
    }
    lds_barrier();
}

// A tile of C transposed through LDS: rows n of B bf16 values m, the pieces of 16 bytes at
// c ^ (n % (B / 8)), then whole rows to memory.
template <int B>
__device__ __forceinline__ uint32_t row_slot(int n, int m) {
    return n * (B * 2) + (((m >> 3) ^ (n & (B / 8 - 1))) << 4) + (m & 7) * 2;
}
template <int B>
__device__ __forceinline__ void put4(uint32_t lds, int n, int m, uint32_t lo, uint32_t hi) {
    typedef __attribute__((address_space(3))) u32x2_t* ptr;
    *(ptr)(size_t)(lds + row_slot<B>(n, m)) = u32x2_t{lo, hi};
}
template <typename Ti>
__device__ __forceinline__ void tile_to_rows(uint32_t lds, uint16_t* out, int64_t ld, int rows, int cols, int tid) {
    constexpr int B = Ti::B;
    typedef const __attribute__((address_space(3))) u32x4_t* ptr;
#pragma unroll 4
    for (int q = tid; q < B * (B / 8); q += Ti::kThreads) {
        const int n = q / (B / 8), c = q % (B / 8);
        if (n < rows && c * 8 < cols) *reinterpret_cast<u32x4_t*>(out + (int64_t)n * ld + c * 8) = *(ptr)(size_t)(lds + row_slot<B>(n, c * 8));
    }
}

// Workgroup b runs on XCD b % 8: groups of `each` tiles that share an operand stay on one XCD.
struct Place {
    int64_t group;
    int within;
};
__device__ __forceinline__ Place tile_place(int64_t block, int each) {
    const int64_t i = block / 8;
    return {i / each * 8 + block % 8, (int)(i % each)};
}

// Logits of a piece of the vocabulary, transposed (a lane holds values of two rows of h): GRAD 0: the
// maximum and sum of exponentials over each wave's B / 2 words; 1: dl [planes][ldp / 256][np][256]; 2: as 0, and the
// exponentials (fp16, relative to that maximum) in dl's place.
struct LogitArgs {
    const uint16_t* w;   // the piece's first row, [planes][vocab][d]
    const float* w32;    // float32: the piece's first row itself
    const uint16_t* h;
    const int32_t *count, *idx, *lab;
    const float *lse, *ll, *dloss;
    int64_t v0, v1, np, ldp, w_plane;  // the piece [v0, v1)
    float2* part;
    uint16_t* p;
    int d, ldh, reduction;
};

__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f32x2_t f = {a, b};
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2_t));
}
__device__ __forceinline__ void unpack_f16x2(uint32_t v, float& a, float& b) {
    typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
    const f16x2_t h = __builtin_bit_cast(f16x2_t, v);
    a = (float)h[0];
    b = (float)h[1];
}

// A logit as a float32 chain: what an infinity needs, which against the other operand's lower planes gives
// NaN (times zero).
__device__ __forceinline__ float logit_chain(const LogitArgs& g, int64_t v, int64_t r) {
    float s = 0.0f;
    const uint16_t* h = g.h + r * g.ldh;
    const int64_t plane = g.np * g.ldh;
    for (int k = 0; k < g.d && s == s; ++k) {
        const float x = bf16_bits_to_f32(h[k]) + (bf16_bits_to_f32(h[k + plane]) + bf16_bits_to_f32(h[k + 2 * plane]));
        s = __builtin_fmaf(x, g.w32[v * g.d + k], s);
    }
    return s;
}

template <typename Ti, int PL, int GRAD>
__global__ __launch_bounds__(Ti::kThreads, 2) void ce_logits_kernel(LogitArgs g) {
    constexpr int B = Ti::B, MI = Ti::kMI, NI = Ti::kNI;
    __shared__ __align__(16) char smem[Ti::kLds + (GRAD ? Ti::kRowsLds : 0)];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lds = lds_addr(smem), mine = lds + Ti::kLds + wave * 4096;
    const int wm = wave / Ti::kWN * (B / 2), wn = wave % Ti::kWN * (32 * NI);
    const int64_t words = g.v1 - g.v0, m = *g.count;
    // this workgroup's tiles: those of the vocabulary tiles of its XCD, one after the other, every gridDim / 8th
    const int n_tiles = (int)((m + B - 1) / B), xcd = blockIdx.x % 8;
    const int64_t m_tiles = (words + B - 1) / B, tiles = (m_tiles - xcd + 7) / 8 * n_tiles;
    int64_t tile = blockIdx.x / 8;
    if (tile >= tiles) return;
    Pair p;
    int64_t m0, n0;
    auto begin = [&]() {
        m0 = (tile / n_tiles * 8 + xcd) * B;
        n0 = tile % n_tiles * B;
        feed_init<Ti, true>(p.a, g.w + m0 * g.d, (words - m0) * g.d * 2, g.d, g.d, 0, g.w_plane, wave, lane);
        feed_init<Ti, true>(p.b, g.h + n0 * g.ldh, (g.np - n0) * g.ldh * 2, g.ldh, g.d, 0, g.np * g.ldh, wave, lane);
        tile_begin<Ti, PL, true, true>(p, (g.d + Ti::kK - 1) / Ti::kK, lds, wave, lane);
    };
    begin();
    step_barrier();
    for (;;) {
        const int64_t tm0 = m0, tn0 = n0;
        // what the epilogue needs of this lane's rows
        float lse[NI], k[NI], label_value[NI];
        int label_at[NI];  // the label's word in the wave's B / 2 words
        if constexpr (GRAD == 1) {
            const float unit = gradient_unit(g.dloss, g.idx, m, g.reduction);
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int64_t r = tn0 + wn + j * 32 + (lane & 31), rc = r < m ? r : m - 1;
                lse[j] = g.lse[rc];
                k[j] = row_gradient(g.dloss, g.idx, rc, m, g.reduction) / unit;
                const int64_t v = (int64_t)g.lab[rc] - g.v0 - tm0 - wm;
                label_at[j] = v >= 0 && v < B / 2 && r < m && lane < 32 ? (int)v : -1;
                label_value[j] = expm1f(g.ll[rc] - lse[j]) * k[j];  // exp(l - lse) - 1 without the cancellation
            }
        }
        f32x16_t acc[MI][NI];
        tile_run<Ti, PL, true, true>(p, lds, acc, wave, lane);
        // the next tile's first steps are on their way during the epilogue
        tile += gridDim.x / 8;
        const bool more = tile < tiles;
        if (more) begin();
        // (hidden from the compiler, which would keep the epilogue's addresses in registers through the products)
        int el = lane;
        asm volatile("" : "+v"(el));
        if constexpr (PL > 1) {
            uint64_t again[NI] = {};
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (acc[i][j][e] != acc[i][j][e]) again[j] |= 1ull << (i * 16 + e);
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                if (ballot(again[j] != 0) == 0) continue;
                const int64_t r = tn0 + wn + j * 32 + (el & 31);
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int64_t v = tm0 + wm + i * 32 + mfma32_row(e, el);
                        if ((again[j] >> (i * 16 + e) & 1) && v < words && r < m) acc[i][j][e] = logit_chain(g, v, r);
                    }
            }
        }
        // words past the vocabulary
        if (tm0 + wm + B / 2 > words) {
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    if (tm0 + wm + i * 32 + mfma32_row(e, el) >= words)
#pragma unroll
                        for (int j = 0; j < NI; ++j) acc[i][j][e] = -__builtin_inff();
        }
        if constexpr (GRAD != 1) {
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int64_t r = tn0 + wn + j * 32 + (el & 31);
                float x = -__builtin_inff();
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x = fmaxf(x, acc[i][j][e]);
                x = fmaxf(x, __shfl_xor(x, 32));
                float s = 0.0f;
                if (ballot(!(fabsf(x) < kScaled)) == 0) {
                    const float z = x * kLog2e;
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -z));
                            s += v;
                            if (GRAD == 2) acc[i][j][e] = v;
                        }
                } else {
                    const float z = x == -__builtin_inff() ? 0.0f : x;
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float v = __builtin_amdgcn_exp2f((acc[i][j][e] - z) * kLog2e);
                            s += v;
                            if (GRAD == 2) acc[i][j][e] = v;
                        }
                }
                s += __shfl_xor(s, 32);
                if (el < 32) g.part[((g.v0 + tm0) / (B / 2) + wave / Ti::kWN) * g.np + r] = make_float2(x, s);
            }
        } else {
            // dl, in place
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const bool in = tn0 + wn + j * 32 + (el & 31) < m;
                const bool far = ballot(!(fabsf(lse[j]) < kScaled)) != 0;  // beyond scaling: relative to lse first
                const float z = far ? 0.0f : lse[j] * kLog2e;
                if (far) {
#pragma unroll
                    for (int i = 0; i < MI; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e) acc[i][j][e] -= lse[j];
                }
#pragma unroll
                for (int i = 0; i < MI; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const float v = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -z)) * k[j];
                        acc[i][j][e] = in ? v : 0.0f;
                    }
            }
        }
        if constexpr (GRAD == 0) {
            if (!more) break;
            step_barrier();
        } else {
            // the next tile's copies, before the stores, which no one waits for
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            // 32 rows by 64 words at a time through the wave's own LDS; what a plane leaves stays in acc
#pragma unroll
            for (int j = 0; j < NI; ++j)
#pragma unroll
                for (int c = 0; c < MI / 2; ++c)
#pragma unroll
                    for (int pl = 0; pl < PL; ++pl) {
                        const int n = el & 31;
#pragma unroll
                        for (int i = 0; i < 2; ++i)
#pragma unroll
                            for (int e = 0; e < 16; e += 4) {
                                f32x16_t& v = acc[2 * c + i][j];
                                uint32_t q[2];
#pragma unroll
                                for (int u = 0; u < 2; ++u) {
                                    q[u] = GRAD == 2 ? pack_f16x2(v[e + 2 * u], v[e + 2 * u + 1]) : pack_bf16x2(v[e + 2 * u], v[e + 2 * u + 1]);
                                    if (pl + 1 < PL) {
                                        v[e + 2 * u] -= __uint_as_float(q[u] << 16);
                                        v[e + 2 * u + 1] -= __uint_as_float(q[u] & 0xffff0000u);
                                    }
                                }
                                typedef __attribute__((address_space(3))) u32x2_t* ptr;
                                *(ptr)(size_t)(mine + n * 128 + (k_piece(n, i * 4 + (e >> 2)) << 4) + 8 * (el >> 5)) = u32x2_t{q[0], q[1]};
                            }
                        asm volatile("" ::: "memory");
                        if (GRAD == 1 && label_at[j] >= 0 && label_at[j] / 64 == c) {
                            typedef __attribute__((address_space(3))) uint16_t* ptr;
                            const int w = label_at[j] % 64;
                            const uint16_t x = f32_to_bf16_bits(label_value[j]);
                            label_value[j] -= bf16_bits_to_f32(x);
                            *(ptr)(size_t)(mine + n * 128 + (k_piece(n, w >> 3) << 4) + (w & 7) * 2) = x;
                        }
                        asm volatile("" ::: "memory");
                        uint16_t* out = g.p + pl * g.np * g.ldp + (tm0 / kPanel * g.np + tn0 + wn + j * 32) * kPanel + tm0 % kPanel + wm + c * 64;
#pragma unroll
                        for (int t = 0; t < 4; ++t) {
                            typedef const __attribute__((address_space(3))) u32x4_t* ptr;
                            const int r = t * 8 + (el >> 3);
                            __builtin_nontemporal_store(*(ptr)(size_t)(mine + r * 128 + (k_piece(r, el & 7) << 4)),
                                                        reinterpret_cast<u32x4_t*>(out + r * kPanel + (el & 7) * 8));
                        }
                        asm volatile("" ::: "memory");
                    }
            if (!more) break;
            lds_barrier();
        }
    }
}

// Parts of dh's reduction over a piece of ldp words, given the labelled rows: none longer than a CU's share of the
// launch's steps, of at least kPartWords words (a part writes and reads a float32 tile: 128 parts of 64 words for a
// 500 x 256 dh took 38 us to add up, longer than the products).
constexpr int kPartWords = 256;
__host__ __device__ inline int dh_parts(int64_t m, int tile, int cols, int64_t ldp, int num_cus, int with_dw) {
    const int64_t rows = (m + tile - 1) / tile * cols, steps = ldp / 64;
    const int64_t all = rows * steps + (with_dw ? (ldp + tile - 1) / tile * cols * ((m + 63) / 64) : 0);
    const int64_t share = all > num_cus ? (all + num_cus - 1) / num_cus : 1, slots = rows > 0 ? num_cus / rows : 1, most = ldp / kPartWords;
    int64_t s = (steps + share - 1) / share;
    s = s < slots ? s : slots;
    s = s < most ? s : most;
    return (int)(s < 1 ? 1 : s);
}

// The gradients of a piece: first the workgroups of dh, float32 partial sums [part][m][d] (added to when `add`), then
// those of dW, the tiles [v][d] of dl^T h as C[m = d][n = v].  In one launch, the short tiles of dW fill the CUs
// that the long parts of dh leave, and the other way round.
struct GradArgs {
    const uint16_t *p, *h, *w;
    const int32_t *count, *idx;
    const float* dloss;
    int64_t words, np, ldp, w_plane;
    float* part;
    void* dw;  // the piece's first row
    int d, ldh, cols, num_cus, add, with_dw, reduction;
    int64_t row_blocks;
};

template <typename Ti, int PL>
__device__ __forceinline__ void ce_row_grad(const GradArgs& g, int64_t block, uint32_t lds, int tid) {
    constexpr int B = Ti::B, MI = Ti::kMI, NI = Ti::kNI;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t m = *g.count;
    const int parts = dh_parts(m, B, g.cols, g.ldp, g.num_cus, g.with_dw);
    const Place at = tile_place(block, g.cols);
    const int part = (int)(at.group % parts);
    const int64_t m0 = at.group / parts * B;
    const int n0 = at.within * B;
    if (m0 >= m) return;
    const int64_t rows = round_up(m, kPadRows);
    const int64_t steps = (g.words + Ti::kK - 1) / Ti::kK, per = (steps + parts - 1) / parts;
    const int64_t s0 = per * part < steps ? per * part : steps, s1 = s0 + per < steps ? s0 + per : steps;
    f32x16_t acc[MI][NI];
    {
        Pair p;
        constexpr int64_t kSteps = kPanel / Ti::kK;
        const int64_t first = (s0 / kSteps * g.np + m0) * kPanel + s0 % kSteps * Ti::kK;
        feed_init<Ti, true>(p.a, g.p + first, (g.np * g.ldp - first) * 2, kPanel, INT32_MAX, 0, g.np * g.ldp, wave, lane);
        p.a.jump = (g.np - 1) * kPanel * 2;
        p.a.at = p.a.at0 = (int)(s0 % kSteps);
        feed_init<Ti, false>(p.b, g.w + s0 * Ti::kK * g.d + n0, ((g.words - s0 * Ti::kK) * g.d - n0) * 2, g.d, 0, g.d - n0, g.w_plane, wave,
                            lane);
        tile_begin<Ti, PL, true, false>(p, s1 - s0, lds, wave, lane);
        step_barrier();
        tile_run<Ti, PL, true, false>(p, lds, acc, wave, lane);
    }
    const int wm = wave / Ti::kWN * (B / 2), wn = wave % Ti::kWN * (32 * NI);
    float* out = g.part + (int64_t)part * rows * g.d;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
        const int n = n0 + wn + j * 32 + (lane & 31);
        if (n >= g.d) continue;
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float* o = out + (m0 + wm + i * 32 + mfma32_row(e, lane)) * g.d + n;
                *o = g.add ? *o + acc[i][j][e] : acc[i][j][e];
            }
    }
}

template <typename Ti, int PL>
__device__ __forceinline__ void ce_head_grad(const GradArgs& g, int64_t block, uint32_t lds, int tid) {
    constexpr int B = Ti::B, MI = Ti::kMI, NI = Ti::kNI;
    const int lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at = tile_place(block, g.cols);
    const int64_t n0 = at.group * B;
    const int m0 = at.within * B;
    if (n0 >= g.words) return;
    f32x16_t acc[MI][NI];
    {
        const int64_t rows = round_up(*g.count, kPadRows), steps = (*g.count + Ti::kK - 1) / Ti::kK;
        Pair p;
        feed_init<Ti, false>(p.a, g.h + m0, (rows * g.ldh - m0) * 2, g.ldh, 0, g.d - m0, g.np * g.ldh, wave, lane);
        feed_init<Ti, false>(p.b, g.p + n0 / kPanel * g.np * kPanel + n0 % kPanel, (rows * kPanel - n0 % kPanel) * 2, kPanel, 0, B,
                            g.np * g.ldp, wave, lane);
        tile_begin<Ti, PL, false, false>(p, steps, lds, wave, lane);
        step_barrier();
        tile_run<Ti, PL, false, false>(p, lds, acc, wave, lane);
    }
    const int wm = wave / Ti::kWN * (B / 2), wn = wave % Ti::kWN * (32 * NI);
    const int rows = g.words - n0 < B ? (int)(g.words - n0) : B;
    const float unit = gradient_unit(g.dloss, g.idx, *g.count, g.reduction);
#pragma unroll
    for (int j = 0; j < NI; ++j)
#pragma unroll
        for (int i = 0; i < MI; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int n = wn + j * 32 + (lane & 31), mm = wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5);
                const f32x16_t a = acc[i][j] * unit;
                if constexpr (PL == 1)
                    put4<B>(lds, n, mm, pack_bf16x2(a[e], a[e + 1]), pack_bf16x2(a[e + 2], a[e + 3]));
                else if (n < rows && m0 + mm < g.d)
                    *reinterpret_cast<float4*>((float*)g.dw + (n0 + n) * g.d + m0 + mm) = make_float4(a[e], a[e + 1], a[e + 2], a[e + 3]);
            }
    if constexpr (PL == 1) {
        lds_barrier();
        tile_to_rows<Ti>(lds, (uint16_t*)g.dw + n0 * g.d + m0, g.d, rows, g.d - m0, tid);
    }
}

template <typename Ti, int PL>
__global__ __launch_bounds__(Ti::kThreads, 2) void ce_grads_kernel(GradArgs g) {
    __shared__ __align__(16) char smem[Ti::kLds];
    if (blockIdx.x < g.row_blocks) ce_row_grad<Ti, PL>(g, blockIdx.x, lds_addr(smem), threadIdx.x);
    else ce_head_grad<Ti, PL>(g, blockIdx.x - g.row_blocks, lds_addr(smem), threadIdx.x);
}

// dh in h's rows and type: the sum of the parts, zeros for rows without a label; 4 columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void ce_row_grad_out_kernel(const float* __restrict__ part, const int32_t* __restrict__ count,
                                                              const int32_t* __restrict__ inv, const int32_t* __restrict__ idx,
                                                              const float* __restrict__ dloss, int reduction, int64_t n, int d, int tile,
                                                              int cols, int64_t ldp, int num_cus, int with_dw, T* __restrict__ dh) {
    const int64_t m = *count, size = round_up(m, kPadRows) * d;
    const int parts = dh_parts(m, tile, cols, ldp, num_cus, with_dw);
    const float unit = gradient_unit(dloss, idx, m, reduction);
    const int64_t total = n * (d / 4);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / (d / 4);
        const int c = (int)(i - r * (d / 4)) * 4;
        const int64_t at = inv[r];
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (at >= 0)
            for (int p0 = 0; p0 < parts; p0 += 4) {
                float4 v[4];
#pragma unroll
                for (int p = 0; p < 4; ++p) v[p] = *reinterpret_cast<const float4*>(part + (p0 + p < parts ? p0 + p : p0) * size + at * d + c);
#pragma unroll
                for (int p = 0; p < 4; ++p) {
                    if (p0 + p >= parts) break;
                    s.x += v[p].x;
                    s.y += v[p].y;
                    s.z += v[p].z;
                    s.w += v[p].w;
                }
            }
        s = make_float4(s.x * unit, s.y * unit, s.z * unit, s.w * unit);
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dh + r * d + c) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
        else *reinterpret_cast<float4*>(dh + r * d + c) = s;
    }
}

// Kept exponentials into dl, in place: times the row's gradient and exp(their maximum - lse), and the label's value.  A
// workgroup takes 64 rows of a panel (32 KB), 8 words a thread at a time; zeros for the padding's rows.
struct KeptArgs {
    const int32_t *count, *idx, *lab;
    const float *lse, *ll, *dloss;
    const float2* part;  // [ldp / words of a maximum][np]
    uint16_t* p;
    int64_t np;
    int each, reduction;  // words of a maximum
};
__global__ __launch_bounds__(256) void ce_kept_kernel(KeptArgs g) {
    const int64_t m = *g.count, r0 = (int64_t)blockIdx.y * 64;
    if (r0 >= round_up(m, kPadRows)) return;
    const int64_t panel = blockIdx.x;
    const int word = (threadIdx.x & 31) * 8;
    const float unit = gradient_unit(g.dloss, g.idx, m, g.reduction);
    uint16_t* p = g.p + (panel * g.np + r0 + (threadIdx.x >> 5)) * kPanel + word;
    const float2* part = g.part + (panel * kPanel + word) / g.each * g.np;
#pragma unroll
    for (int t = 0; t < 8; t += 4) {
        u32x4_t v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(p + (t + u) * 8 * kPanel));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int64_t r = r0 + (threadIdx.x >> 5) + (t + u) * 8, rc = r < m ? r : m > 0 ? m - 1 : 0;
            const float lse = g.lse[rc], x = part[rc].x, k = m > 0 ? row_gradient(g.dloss, g.idx, rc, m, g.reduction) / unit : 0.0f;
            // (no word of the row's there: zeros, or NaN; no word of it at all, a log-sum of -inf: NaN)
            const float f = x == -__builtin_inff() && lse > x ? k * 0.0f : k * expf(x - lse);
            const int64_t label = (int64_t)g.lab[rc] - panel * kPanel - word;
            float y[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) unpack_f16x2(v[u][j], y[2 * j], y[2 * j + 1]);
#pragma unroll
            for (int j = 0; j < 8; ++j) y[j] *= f;
            if (label >= 0 && label < 8) {
                const float one = expm1f(g.ll[rc] - lse) * k;  // exp(l - lse) - 1 without the cancellation
#pragma unroll
                for (int j = 0; j < 8; ++j) y[j] = j == label ? one : y[j];
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) v[u][j] = r < m ? pack_bf16x2(y[2 * j], y[2 * j + 1]) : 0u;
            __builtin_nontemporal_store(v[u], reinterpret_cast<u32x4_t*>(p + (t + u) * 8 * kPanel));
        }
    }
}

// ------------------------------------------------------------------------ sizes
constexpr size_t kPieceBytes = (size_t)1 << 30;  // of dl at a time

// The logits' tiles: of 256 where they give every CU one, or three in float32, where tiles of 128 take all planes at
// once (1,000 x 512 x 20,000, 316 tiles of 256: 139 us with tiles of 128, 171 with 256; 2,048 x 512 x 32,000, 1,000
// tiles: 400 and 361 us), else of 128.
int tile_for(int64_t rows, int64_t cols, int dtype, int num_cus) {
    return cols > 128 && (rows + 255) / 256 * ((cols + 255) / 256) >= num_cus * (dtype == kBF16 ? 1 : 3) ? 256 : 128;
}

// Words of the vocabulary in a piece: whole tiles, at most kPieceBytes for all rows.
int64_t piece_words(int64_t np, int64_t vocab, int planes) {
    int64_t v = (int64_t)(kPieceBytes / ((size_t)np * 2 * planes)) / kTileMax * kTileMax;
    v = v < kTileMax ? kTileMax : v;
    const int64_t all = round_up(vocab, kTileMax);
    const int64_t pieces = (all + v - 1) / v;
    return round_up((all + pieces - 1) / pieces, kTileMax);
}

struct Take {
    char* p;
    size_t at = 0;
    void* operator()(size_t bytes) {
        char* r = p + at;
        at += (bytes + 255) / 256 * 256;
        return r;
    }
};

struct FwdWs {
    float2* part;
    float* row_loss;
    uint16_t* w;  // float32: W's planes
    int tile, n_part;
    size_t bytes;
};
FwdWs fwd_ws(char* p, int64_t n, int d, int64_t vocab, int dtype, int num_cus) {
    FwdWs w;
    Take take{p};
    const int64_t np = round_up(n, kPadRows);
    w.tile = tile_for(vocab, n, dtype, num_cus);
    w.n_part = (int)(round_up(vocab, w.tile) / (w.tile / 2));
    w.part = (float2*)take((size_t)w.n_part * np * 8);
    w.row_loss = (float*)take((size_t)np * 4);
    w.w = dtype == kBF16 ? nullptr : (uint16_t*)take((size_t)vocab * d * 6);
    w.bytes = take.at;
    return w;
}

struct GradWs {
    uint16_t* p;  // dl of a piece (not kept exponentials, which have their own memory)
    float* part;  // dh's parts
    uint16_t* w;  // float32: W's planes
    int64_t piece, part_tiles;
    int logit_tile, grad_tile;
    size_t bytes;
};
GradWs grad_ws(char* p, int64_t n, int d, int64_t vocab, int dtype, int num_cus, bool kept) {
    GradWs w;
    Take take{p};
    const int64_t np = round_up(n, kPadRows);
    const int planes = planes_of(dtype);
    w.piece = kept ? round_up(vocab, kTileMax) : piece_words(np, vocab, planes);
    const int64_t words = vocab < w.piece ? vocab : w.piece;
    w.logit_tile = tile_for(words, n, dtype, num_cus);
    // tiles of 256 for bf16 gradients where dW's and dh's parts give every CU one (a float32 pass of 4,096 x 1,024 x 50,000: 9.4 ms
    // with 256, 8.9 with 128)
    const int64_t cols256 = (d + 255) / 256, m256 = (n + 255) / 256 * cols256;
    const int64_t row256 = m256 * (num_cus / m256 < 1 ? 1 : num_cus / m256 < w.piece / kPartWords ? num_cus / m256 : w.piece / kPartWords);
    w.grad_tile = dtype == kBF16 && d > 128 && (words + 255) / 256 * cols256 + row256 >= num_cus ? 256 : 128;
    w.p = kept ? nullptr : (uint16_t*)take((size_t)np * w.piece * 2 * planes);
    // parts x tiles of rows for any count of labelled rows: as many as fill the chip, or one part
    const int64_t cols = (d + w.grad_tile - 1) / w.grad_tile, slots = num_cus / cols;
    w.part_tiles = slots > np / w.grad_tile ? slots : np / w.grad_tile;
    // a part has the padded rows, up to two tiles of 128 for one
    w.part = (float*)take((size_t)w.part_tiles * kTileMax * d * 4);
    w.w = dtype == kBF16 ? nullptr : (uint16_t*)take((size_t)vocab * d * 6);
    w.bytes = take.at;
    return w;
}

unsigned xcd_grid(int64_t groups, int each) { return (unsigned)((groups + 7) / 8 * 8 * each); }

// f(tile, planes) as constants.  bf16 tiles of 128 that have a CU each (`alone`) get four steps in LDS and eight waves,
// otherwise two of four waves, with two steps each, share a CU.  100 rows of 4,096 against 16,000 words (125 tiles): 48 us with four
// steps, 62 with two.
template <int V> struct Int {
    static constexpr int v = V;
};
template <typename F>
void with_tile(int tile, bool alone, int dtype, F f) {
    if (dtype == kBF16) {
        if (tile == 256) f(Tile<256, 2, 1>{}, Int<1>{});
        else if (alone) f(Tile<128, 4, 1>{}, Int<1>{});
        else f(Tile<128, 2, 1>{}, Int<1>{});
    } else {
        if (tile == 256) f(Tile<256, 2, 1>{}, Int<3>{});
        else f(Tile<128, 2, 3>{}, Int<3>{});
    }
}

LogitArgs logit_args(const CeState& s, const void* w, const uint16_t* planes, int64_t v0, int64_t v1, int64_t vocab, int d, int dtype) {
    LogitArgs g{};
    g.w = (dtype == kBF16 ? (const uint16_t*)w : planes) + v0 * d;
    g.w32 = dtype == kBF16 ? nullptr : (const float*)w + v0 * d;
    g.w_plane = vocab * d;
    g.h = s.h;
    g.count = s.count;
    g.idx = s.idx;
    g.lab = s.lab;
    g.lse = s.lse;
    g.ll = s.ll;
    g.v0 = v0;
    g.v1 = v1;
    g.np = s.np;
    g.d = d;
    g.ldh = s.ldh;
    return g;
}

template <int GRAD>
void run_logits(const LogitArgs& g, int tile, int dtype, int64_t n, int num_cus, hipStream_t stream) {
    // as many workgroups as run at once (one to a CU, or two of bf16 tiles of 128)
    const int64_t m_tiles = (g.v1 - g.v0 + tile - 1) / tile, n_tiles = (n + tile - 1) / tile;
    const int64_t tiles = (m_tiles + 7) / 8 * 8 * n_tiles;
    const int64_t most = round_up(num_cus, 8) * (tile == 256 || dtype != kBF16 ? 1 : 2);
    const dim3 grid((unsigned)(tiles < most ? tiles : most));
    with_tile(tile, m_tiles * n_tiles <= num_cus, dtype, [&](auto t, auto pl) {
        typedef decltype(t) Ti;
        constexpr int PL = decltype(pl)::v;
        if constexpr (GRAD != 2 || PL == 1)  // (float32 exponentials are not kept)
            hipLaunchKernelGGL((ce_logits_kernel<Ti, PL, GRAD>), grid, dim3(Ti::kThreads), 0, stream, g);
    });
}

void split_weights(const void* w, int64_t vocab, int d, uint16_t* out, int num_cus, hipStream_t stream) {
    const int64_t n8 = vocab * d / 8, b = (n8 + 255) / 256;
    hipLaunchKernelGGL(ce_split_kernel, dim3((unsigned)(b < num_cus * 16 ? b : num_cus * 16)), dim3(256), 0, stream, (const float*)w, n8, out);
}

}  // namespace

size_t linear_ce_state_bytes(int64_t n, int d, int dtype) { return ce_state(nullptr, n, d, dtype).bytes; }
size_t linear_ce_workspace_bytes(int64_t n, int d, int64_t vocab, int dtype, int num_cus) {
    return fwd_ws(nullptr, n, d, vocab, dtype, num_cus).bytes;
}
// The kept exponentials, and behind them the maxima that they are relative to (with the sums).
size_t exps_values(int64_t n, int64_t vocab) { return (size_t)round_up(n, kPadRows) * round_up(vocab, kTileMax) * 2; }
size_t linear_ce_exps_bytes(int64_t n, int64_t vocab, int dtype, int num_cus) {
    if (dtype != kBF16) return 0;
    const int64_t maxima = round_up(vocab, kTileMax) / (tile_for(vocab, n, dtype, num_cus) / 2);
    return exps_values(n, vocab) + (size_t)round_up(n, kPadRows) * maxima * 8;
}
size_t linear_ce_grad_workspace_bytes(int64_t n, int d, int64_t vocab, int dtype, int num_cus, bool kept) {
    return grad_ws(nullptr, n, d, vocab, dtype, num_cus, kept).bytes;
}

int launch_linear_ce(const void* h, int64_t ldh, const void* w, const int64_t* labels, int64_t n, int d, int64_t vocab,
                     int64_t ignore, int reduction, int dtype, void* state, void* exps, void* ws, float* loss, int num_cus,
                     hipStream_t stream) {
    const CeState s = ce_state((char*)state, n, d, dtype);
    const FwdWs f = fwd_ws((char*)ws, n, d, vocab, dtype, num_cus);
    float* loss_rows = reduction == kLossNone ? loss : nullptr;
    const dim3 gg((unsigned)(s.np / 4));
    auto gather = [&](const auto* hh, const auto* ww) {
        typedef typename std::decay<decltype(*hh)>::type T;
        if (n <= kFewRows) {
            hipLaunchKernelGGL((ce_few_rows_kernel<T>), gg, dim3(256), 0, stream, labels, (int)n, vocab, ignore, hh, ldh, ww, s.count, s.idx,
                               s.inv, s.lab, loss_rows, s.ticket, d, s.ldh, s.np * s.ldh, s.h, s.ll);
            return;
        }
        hipLaunchKernelGGL(ce_rows_kernel, dim3(1), dim3(1024), 0, stream, labels, n, vocab, ignore, s.count, s.idx, s.inv, s.lab, loss_rows,
                           s.ticket);
        hipLaunchKernelGGL((ce_gather_kernel<T>), gg, dim3(256), 0, stream, hh, ldh, ww, s.count, s.idx, s.lab, d, s.ldh, s.np * s.ldh, s.h,
                           s.ll);
    };
    if (dtype == kBF16) {
        gather((const uint16_t*)h, (const uint16_t*)w);
    } else {
        gather((const float*)h, (const float*)w);
        split_weights(w, vocab, d, f.w, num_cus, stream);
    }
    LogitArgs g = logit_args(s, w, f.w, 0, vocab, vocab, d, dtype);
    g.part = f.part;
    if (exps) {
        g.p = (uint16_t*)exps;
        g.ldp = round_up(vocab, kTileMax);
        g.part = (float2*)((char*)exps + exps_values(n, vocab));
        run_logits<2>(g, f.tile, dtype, n, num_cus, stream);
    } else {
        run_logits<0>(g, f.tile, dtype, n, num_cus, stream);
    }
    hipLaunchKernelGGL(ce_lse_kernel, dim3((unsigned)((n + 15) / 16)), dim3(1024), 0, stream, g.part, f.n_part, s.np, s.count, s.idx, s.ll,
                       reduction, s.lse, f.row_loss, s.ticket, loss);
    return (int)hipGetLastError();
}

int launch_linear_ce_grad(const void* state, void* exps, const void* w, const float* dloss, int64_t n, int d, int64_t vocab, int reduction,
                          int dtype, void* ws, void* dh, void* dw, int num_cus, hipStream_t stream) {
    const CeState s = ce_state((char*)state, n, d, dtype);
    const GradWs b = grad_ws((char*)ws, n, d, vocab, dtype, num_cus, exps != nullptr);
    const int cols = (d + b.grad_tile - 1) / b.grad_tile;
    if (dtype != kBF16) split_weights(w, vocab, d, b.w, num_cus, stream);
    for (int64_t v0 = 0; v0 < vocab; v0 += b.piece) {
        const int64_t words = vocab - v0 < b.piece ? vocab - v0 : b.piece;
        LogitArgs g = logit_args(s, w, b.w, v0, v0 + words, vocab, d, dtype);
        g.p = exps ? (uint16_t*)exps : b.p;
        g.ldp = b.piece;
        g.dloss = dloss;
        g.reduction = reduction;
        if (exps) {
            const KeptArgs a{s.count, s.idx, s.lab, s.lse, s.ll, dloss, (const float2*)((char*)exps + exps_values(n, vocab)), g.p, s.np,
                             tile_for(vocab, n, dtype, num_cus) / 2, reduction};
            hipLaunchKernelGGL(ce_kept_kernel, dim3((unsigned)(b.piece / kPanel), (unsigned)(s.np / 64)), dim3(256), 0, stream, a);
        } else {
            run_logits<1>(g, b.logit_tile, dtype, n, num_cus, stream);
        }
        const int64_t row_blocks = dh ? xcd_grid(b.part_tiles, cols) : 0;
        const int64_t head_blocks = dw ? xcd_grid((words + b.grad_tile - 1) / b.grad_tile, cols) : 0;
        void* const dw_piece = dw ? (char*)dw + v0 * d * (dtype == kBF16 ? 2 : 4) : nullptr;
        const GradArgs a{g.p, s.h, g.w, s.count, s.idx, dloss, words, s.np, b.piece, g.w_plane, b.part, dw_piece, d, s.ldh, cols, num_cus,
                         v0 > 0 ? 1 : 0, dw ? 1 : 0, reduction, row_blocks};
        const int64_t head = dw ? (words + b.grad_tile - 1) / b.grad_tile * cols : 0;
        const int64_t row = dh ? (n + b.grad_tile - 1) / b.grad_tile * cols * dh_parts(n, b.grad_tile, cols, b.piece, num_cus, dw ? 1 : 0) : 0;
        with_tile(b.grad_tile, head + row <= num_cus, dtype, [&](auto t, auto pl) {
            typedef decltype(t) Ti;
            constexpr int PL = decltype(pl)::v;
            if constexpr (PL == 1 || Ti::P == PL)  // (float32 gradients: tiles of 128 alone)
                hipLaunchKernelGGL((ce_grads_kernel<Ti, PL>), dim3((unsigned)(row_blocks + head_blocks)), dim3(Ti::kThreads), 0, stream, a);
        });
    }
    if (dh) {
        int64_t blocks = (n * (d / 4) + 255) / 256;
        blocks = blocks < num_cus * 16 ? blocks : num_cus * 16;
        if (dtype == kBF16)
            hipLaunchKernelGGL((ce_row_grad_out_kernel<uint16_t>), dim3((unsigned)blocks), dim3(256), 0, stream, b.part, s.count, s.inv,
                               s.idx, dloss, reduction, n, d, b.grad_tile, cols, b.piece, num_cus, dw ? 1 : 0, (uint16_t*)dh);
        else
            hipLaunchKernelGGL((ce_row_grad_out_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, stream, b.part, s.count, s.inv, s.idx,
                               dloss, reduction, n, d, b.grad_tile, cols, b.piece, num_cus, dw ? 1 : 0, (float*)dh);
    }
    return (int)hipGetLastError();
}

}  // namespace ethos

// Softmax cross entropy of rows h against a head matrix W [vocab, d], and its gradients, without
// the logits in memory:
//   l_iv = h_i . W_v,  lse_i = log sum_v exp(l_iv),  loss_i = lse_i - l_i,label,
//   dl_iv = g_i (exp(l_iv - lse_i) - [v = label_i]),  dh = dl W,  dW = dl^T h.
//
// Rows without a label (ignore_index) are left out before anything else: the rows with one are
// copied into a dense block (zero-padded to whole tiles), which every product reads; their count
// stays on the device.  bf16: the forward product keeps a maximum and a sum of exponentials per row
// and tile of vocabulary.  The backward forms the logits of a piece of the vocabulary again,
// turns them into dl (bf16) in its epilogue, and multiplies the piece by h and by W.
// float32: the products of gemm.hip on a piece of float32 logits.
#include "ethos_common.hpp"
#include "ethos_gemm.hpp"
#include "ethos_mfma.hpp"
#include "ethos_rows.hpp"
#include "ethos_train.hpp"

namespace ethos {
namespace {

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kScaled = 1e38f;  // logits below this in size can be scaled by log2(e)
constexpr int kPadRows = 256;  // labelled rows are padded with zero rows to a multiple of this

__host__ __device__ constexpr int64_t round_up(int64_t a, int64_t b) { return (a + b - 1) / b * b; }

// What the forward leaves for the backward.
struct CeState {
    int32_t* count;  // labelled rows
    int32_t* idx;    // labelled row -> row of h
    int32_t* inv;    // row of h -> labelled row or -1
    int32_t* lab;    // label of a labelled row (-1: outside the vocabulary)
    float* lse;      // log of the sum of exponentials
    float* ll;       // logit of the label
    void* h;         // the labelled rows [padded n][ldh]
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
    s.count = (int32_t*)take(4);
    s.idx = (int32_t*)take(s.np * 4);
    s.inv = (int32_t*)take(s.np * 4);
    s.lab = (int32_t*)take(s.np * 4);
    s.lse = (float*)take(s.np * 4);
    s.ll = (float*)take(s.np * 4);
    s.h = take((size_t)s.np * s.ldh * (dtype == kBF16 ? 2 : 4));
    s.bytes = at;
    return s;
}

// ------------------------------------------------------------------------ labelled rows
// One workgroup: the rows with a label, in order; loss (when a row's loss is asked for) is zero
// for the others.
__global__ __launch_bounds__(1024) void ce_rows_kernel(const int64_t* __restrict__ labels, int64_t n, int64_t vocab, int64_t ignore,
                                                       int32_t* __restrict__ count, int32_t* __restrict__ idx,
                                                       int32_t* __restrict__ inv, int32_t* __restrict__ lab,
                                                       float* __restrict__ loss_rows) {
    __shared__ int32_t sums[16];
    const int tid = threadIdx.x, wave = tid >> 6;
    int32_t base = 0;
    for (int64_t i0 = 0; i0 < n; i0 += 1024) {
        const int64_t i = i0 + tid;
        const int64_t l = i < n ? labels[i] : ignore;
        const bool use = i < n && l != ignore;
        const uint64_t m = ballot(use);
        if ((tid & 63) == 0) sums[wave] = __popcll(m);
        __syncthreads();
        int32_t before = base, all = 0;
        for (int w = 0; w < 16; ++w) {
            if (w < wave) before += sums[w];
            all += sums[w];
        }
        if (i < n) {
            const int32_t at = before + count_below(m);
            inv[i] = use ? at : -1;
            if (use) {
                idx[at] = (int32_t)i;
                lab[at] = l >= 0 && l < vocab ? (int32_t)l : -1;
            } else if (loss_rows) {
                loss_rows[i] = 0.0f;
            }
        }
        base += all;
        __syncthreads();
    }
    if (tid == 0) *count = base;
}

// A wave per row of the dense block: the row of h (zeros in the padding) and its label's logit.
template <typename T>
__global__ __launch_bounds__(256) void ce_gather_kernel(const T* __restrict__ h, int64_t ld, const T* __restrict__ w,
                                                        const int32_t* __restrict__ count, const int32_t* __restrict__ idx,
                                                        const int32_t* __restrict__ lab, int d, int ldh, T* __restrict__ out,
                                                        float* __restrict__ ll) {
    constexpr int N = Vec16<T>::kN;
    typedef typename Vec16<T>::raw Raw;
    const int lane = threadIdx.x & 63;
    const int64_t r = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t m = *count;
    if (r >= round_up(m, kPadRows)) return;
    const bool in = r < m;
    const T* src = h + (in ? (int64_t)idx[r] : 0) * ld;
    const int label = in ? lab[r] : -1;
    const T* row = w + (int64_t)(label < 0 ? 0 : label) * d;
    float s = 0.0f;
    for (int c = lane * N; c < ldh; c += 64 * N) {
        Raw v = {};
        if (in && c < d) {
            v = *reinterpret_cast<const Raw*>(src + c);
            if (label >= 0) {
                float a[N], b[N];
                Vec16<T>::unpack(v, a);
                Vec16<T>::unpack(*reinterpret_cast<const Raw*>(row + c), b);
#pragma unroll
                for (int j = 0; j < N; ++j) s = __builtin_fmaf(a[j], b[j], s);
            }
        }
        *reinterpret_cast<Raw*>(out + r * ldh + c) = v;
    }
    s = wave_sum(s);
    if (lane == 0) ll[r] = label >= 0 ? s : __builtin_nanf("");
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

// lse and loss of each labelled row from its partial (maximum, sum) pairs part[e][np], e < n_part.
__global__ __launch_bounds__(256) void ce_lse_kernel(const float2* __restrict__ part, int n_part, int64_t np,
                                                     const int32_t* __restrict__ count, const int32_t* __restrict__ idx,
                                                     const float* __restrict__ ll, float* __restrict__ lse,
                                                     float* __restrict__ loss_rows, float* __restrict__ row_loss) {
    __shared__ MaxSum lds[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = (int64_t)blockIdx.x * 64 + lane, m = *count;
    if ((int64_t)blockIdx.x * 64 >= m) return;
    MaxSum a = {-__builtin_inff(), 0.0f};
    for (int e = wave; e < n_part; e += 4) {
        const float2 p = part[(int64_t)e * np + r];
        a = join(a, {p.x, p.y});
    }
    lds[wave][lane] = a;
    __syncthreads();
    if (wave != 0 || r >= m) return;
    for (int w = 1; w < 4; ++w) a = join(a, lds[w][lane]);
    const float x = ll[r];
    const float l = x == x ? a.m + __builtin_amdgcn_logf(a.s) * 0.69314718055994530942f : x;
    lse[r] = l;
    if (loss_rows) loss_rows[idx[r]] = l - x;
    else row_loss[r] = l - x;
}

__global__ __launch_bounds__(1024) void ce_total_kernel(const float* __restrict__ row_loss, const int32_t* __restrict__ count,
                                                        int mean, float* __restrict__ loss) {
    __shared__ double lds[16];
    const int64_t m = *count;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < m; i += 1024) s += (double)row_loss[i];
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        double t = 0.0;
        for (int i = 0; i < 16; ++i) t += lds[i];
        *loss = (float)(mean ? t / (double)m : t);
    }
}

// g of a labelled row: the loss's gradient, per row of h or of the whole.
__device__ __forceinline__ float row_gradient(const float* dloss, const int32_t* idx, int64_t r, int64_t m, int reduction) {
    return reduction == kLossNone ? dloss[idx[r]] : reduction == kLossMean ? *dloss / (float)m : *dloss;
}

// ------------------------------------------------------------------------ bf16 products
// C[m][n] = sum_k A(m, k) B(k, n) in tiles of 256 x 256, k in steps of 64, eight waves (two along m, four
// along n: 128 x 64 each, 128 accumulators a lane).  Operands go from memory straight into LDS, the
// next step's while the current one is multiplied.  An operand is stored with k contiguous ("K": rows
// of m or n) or with k as the row ("R"); R tiles are read with the transposing LDS loads.
// LDS rows of a K tile are 64 k (8 pieces of 16 bytes), piece c at c ^ (row / 2 % 8); of an R tile
// 256 columns (32 pieces), piece c at c ^ 4 (k % 4).
constexpr int kTile = 256, kStep = 64, kTileThreads = 512;
constexpr int kOperandBytes = kTile * kStep * 2;
constexpr uint32_t kOutside = 0x80000000u;  // an offset past every buffer's end: reads zeros

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(3))) bf16x8_t* lds_frag_ptr;
typedef __attribute__((address_space(3))) s16x4_t* lds_tr_ptr;

// One operand: where its tiles are in memory.
struct Feed {
    uint64_t base;   // address of the tile's first step
    int64_t left;    // bytes from there to the operand's end
    int64_t step;    // bytes from a step to the next
    int k_left;      // K: k from this step's first to the end
    uint32_t off[4];  // this lane's offsets
};

template <bool KC>
__device__ __forceinline__ void feed_init(Feed& f, const uint16_t* p, int64_t bytes, int64_t ld, int k, int cols, int wave, int lane) {
    f.base = (uint64_t)p;
    f.left = bytes;
    f.step = KC ? kStep * 2 : kStep * ld * 2;
    f.k_left = k;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int slot = (j * 8 + wave) * 64 + lane;
        if (KC) {
            const int row = slot >> 3, c = (slot & 7) ^ ((row >> 1) & 7);
            f.off[j] = (uint32_t)(row * ld * 2 + c * 16);
        } else {
            const int kk = slot >> 5, c = (slot & 31) ^ ((kk & 3) << 2);
            f.off[j] = c * 8 < cols ? (uint32_t)(kk * ld * 2 + c * 16) : kOutside;
        }
    }
}

// This step's tile into LDS at `lds`, and on to the next step.
template <bool KC>
__device__ __forceinline__ void feed_issue(Feed& f, uint32_t lds, int wave, int lane) {
    const int64_t left = f.left < 0 ? 0 : f.left > 0x7fffffff ? 0x7fffffff : f.left;
    const i32x4_t rs = buffer_rsrc((const void*)f.base, (uint32_t)left);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        uint32_t off = f.off[j];
        if (KC && f.k_left < kStep) {
            const int slot = (j * 8 + wave) * 64 + lane, c = (slot & 7) ^ ((slot >> 4) & 7);
            off = c * 8 < f.k_left ? off : kOutside;
        }
        lds_dma16(rs, (int)off, 0, lds + (j * 8 + wave) * 1024);
    }
    f.base += f.step;
    f.left -= f.step;
    f.k_left -= kStep;
}

// Fragments of 32 rows (or columns) i at row0 + 32 i, reduction step s of 16.
template <bool KC, int N> struct Reader {
    uint32_t at[KC ? 4 : N];
    __device__ __forceinline__ void init(int row0, int lane) {
        if constexpr (KC) {
            const int row = row0 + (lane & 31);
#pragma unroll
            for (int s = 0; s < 4; ++s) at[s] = row * 128 + (((2 * s + (lane >> 5)) ^ ((row >> 1) & 7)) << 4);
        } else {
            const int k = 8 * (lane >> 5) + ((lane & 15) >> 2);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int c = (row0 + 32 * i) / 8 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
                at[i] = k * 512 + ((c ^ ((k & 3) << 2)) << 4) + (lane & 1) * 8;
            }
        }
    }
    __device__ __forceinline__ bf16x8_t get(uint32_t lds, int i, int s) const {
        if constexpr (KC) {
            return *(lds_frag_ptr)(size_t)(lds + at[s] + i * 4096);
        } else {
            union {
                s16x4_t h[2];
                bf16x8_t f;
            } u;
            u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(lds + at[i] + s * 8192));
            u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(lds + at[i] + s * 8192 + 2048));
            return u.f;
        }
    }
};

__device__ __forceinline__ void step_barrier() {
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// The tile's products over `steps` steps; this wave's 128 x 64 part in acc[4][2].
template <bool AK, bool BK>
__device__ __forceinline__ void tile_product(Feed& fa, Feed& fb, int64_t steps, uint32_t lds, f32x16_t (&acc)[4][2], int wave, int lane) {
    Reader<AK, 4> ra;
    Reader<BK, 2> rb;
    ra.init((wave >> 2) * 128, lane);
    rb.init((wave & 3) * 64, lane);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = f32x16_zero();
    if (steps <= 0) return;
    feed_issue<AK>(fa, lds, wave, lane);
    feed_issue<BK>(fb, lds + kOperandBytes, wave, lane);
    step_barrier();
    for (int64_t t = 0; t < steps; ++t) {
        const uint32_t cur = lds + (uint32_t)(t & 1) * 2 * kOperandBytes;
        if (t + 1 < steps) {
            const uint32_t nxt = lds + (uint32_t)((t + 1) & 1) * 2 * kOperandBytes;
            feed_issue<AK>(fa, nxt, wave, lane);
            feed_issue<BK>(fb, nxt + kOperandBytes, wave, lane);
        }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            bf16x8_t a[4], b[2];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = ra.get(cur, i, s);
#pragma unroll
            for (int j = 0; j < 2; ++j) b[j] = rb.get(cur + kOperandBytes, j, s);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[i], b[j], acc[i][j], 0, 0, 0);
        }
        step_barrier();
    }
}

// A tile of C transposed through LDS: rows n of 256 bf16 values m, the pieces of 16 bytes at
// c ^ (n % 32), then whole rows to memory.
__device__ __forceinline__ void put4(uint32_t lds, int n, int m, float a, float b, float c, float d) {
    typedef __attribute__((address_space(3))) u32x2_t* ptr;
    *(ptr)(size_t)(lds + n * 512 + (((m >> 3) ^ (n & 31)) << 4) + (m & 4) * 2) = u32x2_t{pack_bf16x2(a, b), pack_bf16x2(c, d)};
}
__device__ __forceinline__ void tile_to_rows(uint32_t lds, uint16_t* out, int64_t ld, int rows, int cols, int tid) {
    typedef const __attribute__((address_space(3))) u32x4_t* ptr;
#pragma unroll 4
    for (int q = tid; q < kTile * 32; q += kTileThreads) {
        const int n = q >> 5, c = q & 31;
        if (n < rows && c * 8 < cols)
            *reinterpret_cast<u32x4_t*>(out + (int64_t)n * ld + c * 8) = *(ptr)(size_t)(lds + n * 512 + ((c ^ (n & 31)) << 4));
    }
}

// Workgroup b runs on XCD b % 8: groups of `each` tiles that share an operand stay on one XCD.
struct Place {
    int64_t group;
    int within;
};
__device__ __forceinline__ Place tile_place(int each) {
    const int64_t i = blockIdx.x / 8;
    return {i / each * 8 + blockIdx.x % 8, (int)(i % each)};
}

// Logits of a piece of the vocabulary, transposed (a lane holds values of two rows of h): GRAD 0: the
// maximum and sum of exponentials over each wave's 128 words; 1: dl rows [np][ldp].
struct LogitArgs {
    const uint16_t* w;  // the piece's first row
    const uint16_t* h;
    const int32_t *count, *idx, *lab;
    const float *lse, *ll, *dloss;
    int64_t v0, v1, np, ldp;  // the piece
    float2* part;
    uint16_t* p;
    int d, ldh, n_tiles, reduction;
};

template <int GRAD>
__global__ __launch_bounds__(kTileThreads, 2) void ce_logits_kernel(LogitArgs g) {
    __shared__ __align__(16) char smem[4 * kOperandBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at = tile_place(g.n_tiles);
    const int64_t m0 = at.group * kTile, words = g.v1 - g.v0, m = *g.count;
    const int64_t n0 = (int64_t)at.within * kTile;
    if (m0 >= words || n0 >= m) return;
    const uint32_t lds = lds_addr(smem);
    f32x16_t acc[4][2];
    {
        Feed fa, fb;
        feed_init<true>(fa, g.w + m0 * g.d, (words - m0) * g.d * 2, g.d, g.d, 0, wave, lane);
        feed_init<true>(fb, g.h + n0 * g.ldh, (g.np - n0) * g.ldh * 2, g.ldh, g.d, 0, wave, lane);
        tile_product<true, true>(fa, fb, (g.d + kStep - 1) / kStep, lds, acc, wave, lane);
    }
    const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
    // words past the vocabulary
    if (m0 + wm + 128 > words) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e)
                if (m0 + wm + i * 32 + mfma32_row(e, lane) >= words) acc[i][0][e] = acc[i][1][e] = -__builtin_inff();
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int nl = wn + j * 32 + (lane & 31);
        const int64_t r = n0 + nl;
        if constexpr (GRAD == 0) {
            float x = -__builtin_inff();
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) x = fmaxf(x, acc[i][j][e]);
            x = fmaxf(x, __shfl_xor(x, 32));
            float s = 0.0f;
            if (ballot(!(fabsf(x) < kScaled)) == 0) {
                const float z = x * kLog2e;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e], kLog2e, -z));
            } else {
                const float z = x == -__builtin_inff() ? 0.0f : x;
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) s += __builtin_amdgcn_exp2f((acc[i][j][e] - z) * kLog2e);
            }
            s += __shfl_xor(s, 32);
            if (lane < 32) g.part[((g.v0 + m0) / 128 + (wave >> 2)) * g.np + r] = make_float2(x, s);
        } else {
            const bool in = r < m;
            const float y = in ? g.lse[r] : 0.0f;
            if (ballot(!(fabsf(y) < kScaled)) != 0) {  // beyond scaling: from here on relative to lse
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) acc[i][j][e] -= y;
            }
            const float z = ballot(!(fabsf(y) < kScaled)) != 0 ? 0.0f : y * kLog2e;
            const float k = in ? row_gradient(g.dloss, g.idx, r, m, g.reduction) : 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 16; e += 4) {
                    float v[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) v[q] = __builtin_amdgcn_exp2f(__builtin_fmaf(acc[i][j][e + q], kLog2e, -z)) * k;
                    put4(lds, nl, wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5), in ? v[0] : 0.0f, in ? v[1] : 0.0f, in ? v[2] : 0.0f,
                         in ? v[3] : 0.0f);
                }
        }
    }
    if constexpr (GRAD == 1) {
        __syncthreads();
        // the label's value: exp(l - lse) - 1 without the cancellation
        if (tid < kTile && n0 + tid < m) {
            const int64_t r = n0 + tid, v = (int64_t)g.lab[r] - g.v0 - m0;
            if (v >= 0 && v < kTile) {
                const float x = expm1f(g.ll[r] - g.lse[r]) * row_gradient(g.dloss, g.idx, r, m, g.reduction);
                typedef __attribute__((address_space(3))) uint16_t* ptr;
                *(ptr)(size_t)(lds + tid * 512 + ((((int)v >> 3) ^ (tid & 31)) << 4) + ((int)v & 7) * 2) = f32_to_bf16_bits(x);
            }
        }
        __syncthreads();
        tile_to_rows(lds, g.p + n0 * g.ldp + m0, g.ldp, kTile, kTile, tid);
    }
}

// dW of a piece: the tiles [v][d] of dl^T h, as C[m = d][n = v].
struct HeadGradArgs {
    const uint16_t *h, *p;
    const int32_t* count;
    int64_t words, np, ldp;
    uint16_t* dw;  // the piece's first row
    int d, ldh, m_tiles;
};
__global__ __launch_bounds__(kTileThreads, 2) void ce_head_grad_kernel(HeadGradArgs g) {
    __shared__ __align__(16) char smem[4 * kOperandBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at = tile_place(g.m_tiles);
    const int64_t n0 = at.group * kTile;
    const int m0 = at.within * kTile;
    if (n0 >= g.words) return;
    const uint32_t lds = lds_addr(smem);
    f32x16_t acc[4][2];
    {
        const int64_t rows = round_up(*g.count, kPadRows);  // of h and dl
        Feed fa, fb;
        feed_init<false>(fa, g.h + m0, rows * g.ldh * 2 - m0 * 2, g.ldh, 0, g.d - m0, wave, lane);
        feed_init<false>(fb, g.p + n0, rows * g.ldp * 2 - n0 * 2, g.ldp, 0, kTile, wave, lane);
        tile_product<false, false>(fa, fb, (*g.count + kStep - 1) / kStep, lds, acc, wave, lane);
    }
    const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4)
                put4(lds, wn + j * 32 + (lane & 31), wm + i * 32 + 8 * (e >> 2) + 4 * (lane >> 5), acc[i][j][e], acc[i][j][e + 1],
                     acc[i][j][e + 2], acc[i][j][e + 3]);
    __syncthreads();
    const int64_t rows = g.words - n0;
    tile_to_rows(lds, g.dw + n0 * g.d + m0, g.d, rows < kTile ? (int)rows : kTile, g.d - m0, tid);
}

// Parts of dh's reduction over a piece: as many as fill the chip, given the labelled rows' tiles.
__host__ __device__ inline int dh_parts(int64_t m, int n_tiles, int num_cus) {
    const int64_t tiles = (m + kTile - 1) / kTile * n_tiles;
    const int64_t s = tiles > 0 ? num_cus / tiles : 1;
    return (int)(s < 1 ? 1 : s);
}

// dh of a piece as float32 partial sums [part][m][d], added to when `add`.
struct RowGradArgs {
    const uint16_t *p, *w;
    const int32_t* count;
    int64_t words, ldp;
    float* part;
    int d, n_tiles, num_cus, add;
};
__global__ __launch_bounds__(kTileThreads, 2) void ce_row_grad_kernel(RowGradArgs g) {
    __shared__ __align__(16) char smem[4 * kOperandBytes];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int64_t m = *g.count;
    const int parts = dh_parts(m, g.n_tiles, g.num_cus);
    const Place at = tile_place(g.n_tiles);
    const int part = (int)(at.group % parts);
    const int64_t m0 = at.group / parts * kTile;
    const int n0 = at.within * kTile;
    if (m0 >= m) return;
    const int64_t rows = round_up(m, kPadRows);
    const int64_t steps = (g.words + kStep - 1) / kStep, per = (steps + parts - 1) / parts;
    const int64_t s0 = per * part, s1 = s0 + per < steps ? s0 + per : steps;
    f32x16_t acc[4][2];
    {
        Feed fa, fb;
        feed_init<true>(fa, g.p + m0 * g.ldp + s0 * kStep, ((rows - m0) * g.ldp - s0 * kStep) * 2, g.ldp, INT32_MAX, 0, wave, lane);
        feed_init<false>(fb, g.w + s0 * kStep * g.d + n0, ((g.words - s0 * kStep) * g.d - n0) * 2, g.d, 0, g.d - n0, wave, lane);
        tile_product<true, false>(fa, fb, s1 - s0, lds_addr(smem), acc, wave, lane);
    }
    const int wm = (wave >> 2) * 128, wn = (wave & 3) * 64;
    float* out = g.part + (int64_t)part * rows * g.d;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const int n = n0 + wn + j * 32 + (lane & 31);
        if (n >= g.d) continue;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                float* o = out + (m0 + wm + i * 32 + mfma32_row(e, lane)) * g.d + n;
                *o = g.add ? *o + acc[i][j][e] : acc[i][j][e];
            }
    }
}

// dh in h's rows and type: the sum of the parts, zeros for rows without a label.  A row of `part` has
// d values; 4 columns a thread.
template <typename T>
__global__ __launch_bounds__(256) void ce_row_grad_out_kernel(const float* __restrict__ part, const int32_t* __restrict__ count,
                                                              const int32_t* __restrict__ inv, int64_t n, int d, int n_tiles,
                                                              int num_cus, int pad, T* __restrict__ dh) {
    const int64_t m = *count, size = (pad ? round_up(m, kPadRows) : m) * d;
    const int parts = n_tiles > 0 ? dh_parts(m, n_tiles, num_cus) : 1;
    const int64_t total = n * (d / 4);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t r = i / (d / 4);
        const int c = (int)(i - r * (d / 4)) * 4;
        const int64_t at = inv[r];
        float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (at >= 0)
            for (int p = 0; p < parts; ++p) {
                const float4 v = *reinterpret_cast<const float4*>(part + p * size + at * d + c);
                s.x += v.x;
                s.y += v.y;
                s.z += v.z;
                s.w += v.w;
            }
        if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(dh + r * d + c) = make_uint2(pack_bf16x2(s.x, s.y), pack_bf16x2(s.z, s.w));
        else *reinterpret_cast<float4*>(dh + r * d + c) = s;
    }
}

// ------------------------------------------------------------------------ float32: pieces of logits
// Maximum and sum of a row of a piece's logits [m][ld]; one workgroup per row.
__global__ __launch_bounds__(256) void ce_piece_stats_kernel(const float* __restrict__ logits, int64_t ld, int64_t words,
                                                             const int32_t* __restrict__ count, float2* __restrict__ part) {
    __shared__ MaxSum lds[4];
    const int64_t r = blockIdx.x;
    if (r >= *count) return;
    float x = -__builtin_inff();
    for (int64_t c = threadIdx.x; c < words; c += 256) x = fmaxf(x, logits[r * ld + c]);
    const float z = x == -__builtin_inff() ? 0.0f : x;
    MaxSum a = {x, 0.0f};
    for (int64_t c = threadIdx.x; c < words; c += 256) a.s += expf(logits[r * ld + c] - z);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) a = join(a, {__shfl_xor(a.m, o), __shfl_xor(a.s, o)});
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = a;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; ++w) a = join(a, lds[w]);
        part[r] = make_float2(a.m, a.s);
    }
}

// A piece's logits into dl, in place; the columns up to ld get zeros.
__global__ __launch_bounds__(256) void ce_piece_grad_kernel(float* __restrict__ logits, int64_t ld, int64_t v0, int64_t words,
                                                            const int32_t* __restrict__ count, const int32_t* __restrict__ idx,
                                                            const int32_t* __restrict__ lab, const float* __restrict__ lse,
                                                            const float* __restrict__ ll, const float* __restrict__ dloss, int reduction) {
    const int64_t r = blockIdx.x, m = *count;
    if (r >= m) return;
    const float g = row_gradient(dloss, idx, r, m, reduction), z = lse[r];
    const int64_t label = lab[r] - v0;
    for (int64_t c = threadIdx.x; c < ld; c += 256) {
        float* p = logits + r * ld + c;
        *p = c >= words ? 0.0f : g * (c == label ? expm1f(ll[r] - z) : expf(*p - z));
    }
}

__global__ __launch_bounds__(256) void ce_add_kernel(float* __restrict__ a, const float* __restrict__ b, const int32_t* __restrict__ count,
                                                     int d) {
    const int64_t n = (int64_t)*count * d;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) a[i] += b[i];
}

// ------------------------------------------------------------------------ sizes
constexpr size_t kPieceBytes = (size_t)1 << 30;  // of dl or of float32 logits at a time

// Words of the vocabulary in a piece: whole tiles, at most kPieceBytes for all rows.
int64_t piece_words(int64_t np, int64_t vocab, int elem) {
    int64_t v = (int64_t)(kPieceBytes / ((size_t)np * elem)) / kTile * kTile;
    v = v < kTile ? kTile : v;
    const int64_t all = round_up(vocab, kTile);
    const int64_t pieces = (all + v - 1) / v;
    return round_up((all + pieces - 1) / pieces, kTile);
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
    float* logits;
    int n_part;
    int64_t piece;
    size_t bytes;
};
FwdWs fwd_ws(char* p, int64_t n, int64_t vocab, int dtype) {
    FwdWs w;
    Take take{p};
    const int64_t np = round_up(n, kPadRows);
    w.piece = dtype == kBF16 ? 0 : piece_words(np, vocab, 4);
    w.n_part = dtype == kBF16 ? (int)(round_up(vocab, kTile) / 128) : (int)((vocab + w.piece - 1) / w.piece);
    w.part = (float2*)take((size_t)w.n_part * np * 8);
    w.row_loss = (float*)take((size_t)np * 4);
    w.logits = dtype == kBF16 ? nullptr : (float*)take((size_t)np * w.piece * 4);
    w.bytes = take.at;
    return w;
}

struct GradWs {
    void* p;      // dl of a piece
    float* part;  // dh: parts, or (float32) the sum and a piece's product
    float* split;
    int64_t piece, part_rows;
    int splits;
    size_t bytes;
};
GradWs grad_ws(char* p, int64_t n, int d, int64_t vocab, int dtype, int num_cus) {
    GradWs w;
    Take take{p};
    const int64_t np = round_up(n, kPadRows);
    const int elem = dtype == kBF16 ? 2 : 4;
    w.piece = piece_words(np, vocab, elem);
    w.p = take((size_t)np * w.piece * elem);
    w.split = nullptr;
    w.splits = 1;
    if (dtype == kBF16) {
        // parts x rows for any count of labelled rows: at most a tile per CU, or one part
        const int64_t cols = round_up(d, kTile) / kTile;
        const int64_t most = num_cus / cols > np / kTile ? num_cus / cols : np / kTile;
        w.part_rows = most * kTile;
        w.part = (float*)take((size_t)w.part_rows * d * 4);
    } else {
        w.part_rows = np;
        w.part = (float*)take((size_t)np * d * 4 * 2);
        w.splits = gemm_split(np, d, w.piece, num_cus);
        w.split = (float*)take((size_t)w.splits * np * d * 4);
    }
    w.bytes = take.at;
    return w;
}

unsigned xcd_grid(int64_t groups, int each) { return (unsigned)((groups + 7) / 8 * 8 * each); }

LogitArgs logit_args(const CeState& s, const void* w, int64_t v0, int64_t v1, int d, int64_t n) {
    LogitArgs g{};
    g.w = (const uint16_t*)w + v0 * d;
    g.h = (const uint16_t*)s.h;
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
    g.n_tiles = (int)((n + kTile - 1) / kTile);
    return g;
}

Gemm logits_gemm(const CeState& s, const float* w, int64_t n, int d, int64_t words, float* out, int64_t ld) {
    Gemm g;
    g.a = s.h;
    g.lda = s.ldh;
    g.b = w;
    g.ldb = d;
    g.c = out;
    g.ldc = ld;
    g.m = n;
    g.n = (int)words;
    g.k = d;
    g.dyn = s.count;
    return g;
}

}  // namespace

size_t linear_ce_state_bytes(int64_t n, int d, int dtype) { return ce_state(nullptr, n, d, dtype).bytes; }
size_t linear_ce_workspace_bytes(int64_t n, int, int64_t vocab, int dtype) { return fwd_ws(nullptr, n, vocab, dtype).bytes; }
size_t linear_ce_grad_workspace_bytes(int64_t n, int d, int64_t vocab, int dtype, int num_cus) {
    return grad_ws(nullptr, n, d, vocab, dtype, num_cus).bytes;
}

int launch_linear_ce(const void* h, int64_t ldh, const void* w, const int64_t* labels, int64_t n, int d, int64_t vocab,
                     int64_t ignore, int reduction, int dtype, void* state, void* ws, float* loss, int num_cus, hipStream_t stream) {
    const CeState s = ce_state((char*)state, n, d, dtype);
    const FwdWs f = fwd_ws((char*)ws, n, vocab, dtype);
    float* rows = reduction == kLossNone ? loss : nullptr;
    hipLaunchKernelGGL(ce_rows_kernel, dim3(1), dim3(1024), 0, stream, labels, n, vocab, ignore, s.count, s.idx, s.inv, s.lab, rows);
    const dim3 gg((unsigned)(s.np / 4));
    if (dtype == kBF16) {
        hipLaunchKernelGGL((ce_gather_kernel<uint16_t>), gg, dim3(256), 0, stream, (const uint16_t*)h, ldh, (const uint16_t*)w, s.count,
                           s.idx, s.lab, d, s.ldh, (uint16_t*)s.h, s.ll);
        LogitArgs g = logit_args(s, w, 0, vocab, d, n);
        g.part = f.part;
        hipLaunchKernelGGL((ce_logits_kernel<0>), dim3(xcd_grid((vocab + kTile - 1) / kTile, g.n_tiles)), dim3(kTileThreads), 0, stream,
                           g);
    } else {
        hipLaunchKernelGGL((ce_gather_kernel<float>), gg, dim3(256), 0, stream, (const float*)h, ldh, (const float*)w, s.count, s.idx,
                           s.lab, d, s.ldh, (float*)s.h, s.ll);
        for (int e = 0; e < f.n_part; ++e) {
            const int64_t v0 = e * f.piece, words = vocab - v0 < f.piece ? vocab - v0 : f.piece;
            const int rc = launch_gemm(kGemmFK_FK, logits_gemm(s, (const float*)w + v0 * d, n, d, words, f.logits, f.piece), num_cus, stream);
            if (rc != 0) return rc;
            hipLaunchKernelGGL(ce_piece_stats_kernel, dim3((unsigned)n), dim3(256), 0, stream, f.logits, f.piece, words, s.count,
                               f.part + e * s.np);
        }
    }
    hipLaunchKernelGGL(ce_lse_kernel, dim3((unsigned)(s.np / 64)), dim3(256), 0, stream, f.part, f.n_part, s.np, s.count, s.idx, s.ll,
                       s.lse, rows, f.row_loss);
    if (!rows)
        hipLaunchKernelGGL(ce_total_kernel, dim3(1), dim3(1024), 0, stream, f.row_loss, s.count, reduction == kLossMean ? 1 : 0, loss);
    return (int)hipGetLastError();
}

int launch_linear_ce_grad(const void* state, const void* w, const float* dloss, int64_t n, int d, int64_t vocab, int reduction,
                          int dtype, void* ws, void* dh, void* dw, int num_cus, hipStream_t stream) {
    const CeState s = ce_state((char*)state, n, d, dtype);
    const GradWs b = grad_ws((char*)ws, n, d, vocab, dtype, num_cus);
    const int cols = (d + kTile - 1) / kTile;
    const int64_t m_tiles = (n + kTile - 1) / kTile;
    for (int64_t v0 = 0; v0 < vocab; v0 += b.piece) {
        const int64_t words = vocab - v0 < b.piece ? vocab - v0 : b.piece;
        if (dtype == kBF16) {
            LogitArgs g = logit_args(s, w, v0, v0 + words, d, n);
            g.p = (uint16_t*)b.p;
            g.ldp = b.piece;
            g.dloss = dloss;
            g.reduction = reduction;
            hipLaunchKernelGGL((ce_logits_kernel<1>), dim3(xcd_grid((words + kTile - 1) / kTile, g.n_tiles)), dim3(kTileThreads), 0, stream,
                               g);
            if (dw) {
                const HeadGradArgs a{(const uint16_t*)s.h, (const uint16_t*)b.p, s.count, words, s.np, b.piece, (uint16_t*)dw + v0 * d,
                                     d, s.ldh, cols};
                hipLaunchKernelGGL(ce_head_grad_kernel, dim3(xcd_grid((words + kTile - 1) / kTile, cols)), dim3(kTileThreads), 0, stream, a);
            }
            if (dh) {
                const RowGradArgs a{(const uint16_t*)b.p, (const uint16_t*)w + v0 * d, s.count, words, b.piece, b.part, d, cols, num_cus,
                                    v0 > 0 ? 1 : 0};
                hipLaunchKernelGGL(ce_row_grad_kernel, dim3(xcd_grid(b.part_rows / kTile, cols)), dim3(kTileThreads), 0, stream, a);
            }
        } else {
            const float* wp = (const float*)w + v0 * d;
            float* p = (float*)b.p;
            int rc = launch_gemm(kGemmFK_FK, logits_gemm(s, wp, n, d, words, p, b.piece), num_cus, stream);
            if (rc != 0) return rc;
            hipLaunchKernelGGL(ce_piece_grad_kernel, dim3((unsigned)n), dim3(256), 0, stream, p, b.piece, v0, words, s.count, s.idx, s.lab,
                               s.lse, s.ll, dloss, reduction);
            if (dw) {
                Gemm g;
                g.a = p;
                g.lda = b.piece;
                g.b = s.h;
                g.ldb = s.ldh;
                g.c = (float*)dw + v0 * d;
                g.ldc = d;
                g.m = words;
                g.n = d;
                g.k = n;
                g.dyn = s.count;
                g.dyn_k = true;
                rc = launch_gemm(kGemmFR_FR, g, num_cus, stream);
                if (rc != 0) return rc;
            }
            if (dh) {
                Gemm g;
                g.a = p;
                g.lda = b.piece;
                g.b = wp;
                g.ldb = d;
                g.c = b.part + (v0 > 0 ? s.np * d : 0);
                g.ldc = d;
                g.m = n;
                g.n = d;
                g.k = words;
                g.split = b.splits;
                g.part = b.split;
                g.dyn = s.count;
                rc = launch_gemm(kGemmFK_FR, g, num_cus, stream);
                if (rc != 0) return rc;
                if (v0 > 0)
                    hipLaunchKernelGGL(ce_add_kernel, dim3((unsigned)(num_cus * 8)), dim3(256), 0, stream, b.part, b.part + s.np * d, s.count, d);
            }
        }
    }
    if (dh) {
        int64_t blocks = (n * (d / 4) + 255) / 256;
        blocks = blocks < num_cus * 16 ? blocks : num_cus * 16;
        if (dtype == kBF16)
            hipLaunchKernelGGL((ce_row_grad_out_kernel<uint16_t>), dim3((unsigned)blocks), dim3(256), 0, stream, b.part, s.count, s.inv, n,
                               d, cols, num_cus, 1, (uint16_t*)dh);
        else
            hipLaunchKernelGGL((ce_row_grad_out_kernel<float>), dim3((unsigned)blocks), dim3(256), 0, stream, b.part, s.count, s.inv, n, d,
                               0, num_cus, 0, (float*)dh);
    }
    return (int)hipGetLastError();
}

}  // namespace ethos

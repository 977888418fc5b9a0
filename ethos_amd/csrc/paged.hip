// Attention of new tokens over a cache of latents in pages: softmax(scale q k) v over the keys up to each
// token, with k of head h = [W_k,h c | key] and v = W_v,h c of a cached row [c | key] (model.py:104-160
// forms every head's keys and values; here they stay what they are made of).
//
// The weight goes to the queries instead: q . W_k,h c = (W_k,h^T q) . c, and W_v,h goes behind the sum over
// the keys, which all heads then take over the same rows: one read of the cache serves every head.  A
// sequence's rows are its (token, head) pairs, token by token, so that a tile of rows sees nearly the same keys.
//
// Three launches.  The first: queries [W_k,h^T q | rotated rest] per row, and the plan: tiles of rows,
// each with its tiles of kKeys keys, as one line of work that is cut into even shares, whatever the lengths
// of the sequences are.  The second goes over the keys with a running maximum and sum; where a share ends
// inside a tile of rows, each side leaves its sums.  The third joins them, in order, and multiplies with W_v,h.
//
// Three forms: any widths in float32 arithmetic (any_*), bf16 of the model's widths, and the same with many new tokens a
// sequence, where keys and values are formed first (expand and chunk_*).
//
// Without bounds of the host on lengths, tables or starts: what they hold is checked where it is used.  A page
// outside the cache reads as a row of NaN, a length beyond the table makes its sequence's outputs NaN.
#include <type_traits>

#include "ethos_launch.hpp"
#include "ethos_mfma.hpp"
#include "ethos_rows.hpp"
#include "ethos_serve.hpp"

namespace ethos {
namespace {

constexpr int kKeys = 64;          // keys of a tile of work
constexpr float kLog2E = 1.44269504f;
constexpr float kLowest = -0x1p126f;  // a running maximum's start: finite, so that masked scores weigh nothing
// Running maxima are of scores as they are, which a weight's exponent takes off before the scale: s scale2 - RN(max scale2) is
// the rounding of max scale2 at the maximum, 2^6 for scores of 2^29 and more than any exponent soon after.
constexpr int32_t kLongest = 1 << 30;  // a sequence's length, at most

// A tile of rows: `rows` of sequence seq from its row `row0` (token row0 / H, head row0 % H) on; the first new
// token of the sequence is row tok0 of the batch, at position pos0.
struct Item {
    int32_t seq, row0, rows, tok0, pos0;
    int32_t keys;  // tile of the sequence's first key, if all sequences' keys are laid out one after the other
    int64_t end;   // tiles of work up to this one's last, all before it included
};

// A token's sequence, kNoSeq without one, kBadSeq with one that has no result (its length does not fit its table, or its
// rows are not in the batch); and its place among the sequence's new tokens.
constexpr int kNoSeq = -1, kBadSeq = -2;
struct Token {
    int32_t seq, index;
};

struct Plan {
    int64_t tiles, quota;  // in all; of a workgroup
    int32_t n_items, pad[3];
};

// Where the workspace's parts are.
struct Layout {
    size_t plan, items, seq_item, tokens, specials, queries, sums, stats, bytes;
    int64_t max_items;
};

struct Shape {
    int H, rank, rope, nope, v_dim;
    int rows;    // of a tile
    int groups;  // workgroups that share the work
    int planes;  // how often the work is there: once for all heads, or once for each
    float scale2;
};

constexpr size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

Layout layout(int64_t n_rows, int n_seq, int H, int width, int tile_rows, int groups, size_t query_bytes, int rank) {
    Layout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += round256(bytes);
        return p;
    };
    l.max_items = (n_rows * H) / tile_rows + n_seq;
    l.plan = take(sizeof(Plan));
    l.items = take((size_t)l.max_items * sizeof(Item));
    l.seq_item = take((size_t)n_seq * 4);
    l.tokens = take((size_t)n_rows * sizeof(Token));
    l.specials = take((size_t)16 * width * 2);
    l.queries = take((size_t)n_rows * H * width * query_bytes);
    const size_t slots = (size_t)(l.max_items + groups);
    l.sums = take(slots * tile_rows * rank * 4);
    l.stats = take(slots * tile_rows * 8);
    l.bytes = at;
    return l;
}

// ------------------------------------------------------------------------- the plan
template <int NT>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* lds, int tid, int64_t& total) {  // inclusive, NT threads
    const int lane = tid & 63, wave = tid >> 6;
    for (int d = 1; d < 64; d <<= 1) {
        const int64_t o = __shfl_up(v, d, 64);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = v;
    __syncthreads();
    int64_t before = 0;
    total = 0;
    for (int w = 0; w < NT / 64; ++w) {
        if (w < wave) before += lds[w];
        total += lds[w];
    }
    return v + before;
}

// New tokens of sequence i that the batch really holds, and whether its length fits the table.
__device__ __forceinline__ int64_t new_tokens(const Batch& b, int i) {
    const int64_t first = b.starts[i], last = b.starts[i + 1];
    return first < 0 || last > b.n_rows || last < first ? 0 : last - first;
}
__device__ __forceinline__ bool fits(const Batch& b, int i) {
    return b.lens[i] >= 0 && b.lens[i] <= kLongest && (int64_t)b.lens[i] <= (int64_t)b.width << b.page_log;
}

__device__ __forceinline__ Token token_of(const Batch& b, int64_t t, int i) {
    if (i < 0) return Token{kNoSeq, 0};
    return new_tokens(b, i) > 0 && fits(b, i) ? Token{i, (int32_t)(t - b.starts[i])} : Token{kBadSeq, 0};
}

// One workgroup of NT threads: NT sequences at a time, then their items, NT at a time.
template <int NT>
__device__ void make_plan(const Batch& b, const Shape& s, int64_t max_items, Plan* plan, Item* items, int32_t* seq_item, int32_t* seq_keys,
                          int tid) {
    __shared__ int64_t lds[NT / 64];
    __shared__ int32_t ends[NT], counts[NT], tok0[NT], lens[NT], keys[NT];
    int64_t base = 0, tiles = 0, key_tiles = 0, total;
    for (int at = 0; at < b.n_seq; at += NT) {
        const int i = at + tid;
        if (seq_keys) {  // where each sequence's keys begin, if all are laid out one after the other
            const int64_t n = i < b.n_seq && new_tokens(b, i) > 0 && fits(b, i) ? (b.lens[i] + kKeys - 1) / kKeys : 0;
            const int64_t end = key_tiles + block_scan<NT>(n, lds, tid, total);
            if (i < b.n_seq) seq_keys[i] = keys[tid] = (int32_t)(end - n);
            key_tiles += total;
        }
        const int64_t count = i < b.n_seq ? new_tokens(b, i) : 0, n = (count * s.H + s.rows - 1) / s.rows;
        const int64_t end = block_scan<NT>(n, lds, tid, total);
        // (starts that overlap could ask for more than there is room for: those sequences get none)
        if (i < b.n_seq) seq_item[i] = base + end <= max_items ? (int32_t)(base + end - n) : -1;
        const int64_t here = total < max_items - base ? total : max_items - base;
        ends[tid] = (int32_t)(end < here ? end : here);
        counts[tid] = (int32_t)count;
        if (i < b.n_seq) tok0[tid] = b.starts[i], lens[tid] = fits(b, i) ? b.lens[i] : -1;
        __syncthreads();
        for (int64_t k0 = 0; k0 < here; k0 += NT) {
            const int k = (int)k0 + tid;
            Item it = {};
            int64_t work = 0;
            if (k < here) {
                int lo = 0;  // the first sequence whose items end behind k
                for (int step = NT / 2; step > 0; step >>= 1)
                    if (ends[lo + step - 1] <= k) lo += step;
                it.seq = at + lo;
                it.row0 = (k - (lo > 0 ? ends[lo - 1] : 0)) * s.rows;
                const int left = counts[lo] * s.H - it.row0;
                it.rows = left < s.rows ? left : s.rows;
                it.tok0 = tok0[lo];
                it.pos0 = lens[lo] - counts[lo];
                it.keys = seq_keys ? keys[lo] : 0;
                // keys up to the last row's own
                const int64_t keys = (int64_t)it.pos0 + (it.row0 + it.rows - 1) / s.H + 1;
                work = lens[lo] >= 0 && keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
            }
            it.end = tiles + block_scan<NT>(work, lds, tid, total);
            if (k < here) items[base + k] = it;
            tiles += total;
        }
        base += here;
        __syncthreads();
    }
    if (tid == 0) {
        if (seq_keys) seq_keys[b.n_seq] = (int32_t)key_tiles;
        // Few tiles a workgroup, two workgroups a CU: one on each, whose parts are then half as many to join.  us with two | one,
        // up to four tiles a workgroup of two: one sequence of 65,536 keys 35.2 | 28.2, 8 of 8,192 27.1 | 24.8, 16 of 8,192
        // 32.8 | 30.5; beyond: 8 of 20,000 35.7 | 36.1.
        tiles *= s.planes;
        const int64_t groups = s.rows <= 32 && tiles <= 4 * (int64_t)s.groups ? (s.groups + 1) / 2 : s.groups;
        plan->tiles = tiles;
        plan->quota = tiles > groups ? (tiles + groups - 1) / groups : 1;
        plan->n_items = (int32_t)base;
    }
}

// The first item whose work ends behind tile t (one exists), by all lanes of a wave.
__device__ __forceinline__ int find_item(const Item* items, int n_items, int64_t t, int lane) {
    int lo = 0, n = n_items;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 63) / 64;
        const int at = lo + (lane + 1) * step - 1;
        const bool before = at < lo + n && items[at].end <= t;
        const int k = __builtin_popcountll(ballot(before));
        lo += k * step;
        n = n - k * step < step ? n - k * step : step;
    }
    return lo;
}

// ------------------------------------------------------------------------- any widths, both types
// In float32 throughout, on 16 x 16 x 4 matrix products: tiles of 16 rows, a wave 16 keys of a step's 64.  A product's
// columns and keys may come in any order, so each lane takes four neighbouring columns at a time: of one of 16 keys for
// the scores, of 64 columns of one of four keys for the sums.  S^T = K Q^T leaves keys 4 g + e of a row in lane (row, g),
// which is where O^T = C^T P^T takes them with key 4 g + e in place g of its product e: nothing goes through LDS but the
// queries, and the waves run by themselves up to the end of a share, where their sums are joined.
//
// 512 float32 tokens over 2,048 keys, rank 256, rope 64, 16 heads: 301 us in all, 55 TFLOP/s of 132 that a large float32
// product reaches; what holds it there has not been measured apart (vector instructions over keys in LDS took 5,158).  16 sequences of
// one token and up to 4,096 keys: 65 us (758).  Five sequences of 33 tokens, rank 32: 19 us, the three kernels' times 5, 8 and 6:
// launches and dependent loads.
constexpr int kAnyRows = 16, kAnyKeys = 16, kAnyRank = 512, kAnyRope = 128, kAnyWidth = kAnyRank + kAnyRope;
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ f32x4_t load4(const float* p) { return *reinterpret_cast<const f32x4_t*>(p); }
__device__ __forceinline__ f32x4_t load4(const uint16_t* p) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    return f32x4_t{__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u)};
}

// Block 0 the plan and a row of zeros; each other block 16 tokens of a head, [c][token] = W_k,h^T q^T, a wave every
// fourth 64 columns.
template <typename T>
__global__ __launch_bounds__(256) void any_prepare_kernel(const T* __restrict__ q, const T* __restrict__ w, const float* __restrict__ rates,
                                                          Batch b, Shape s, int64_t max_items, Plan* plan, Item* items, int32_t* seq_item,
                                                          Token* tokens, T* __restrict__ zeros, float* __restrict__ queries) {
    __shared__ float qs[16][64 + 4];
    __shared__ int64_t pos[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, width = s.rank + s.rope;
    if (blockIdx.x == 0) {
        for (int e = tid; e < width; e += 256) zeros[e] = 0;
        make_plan<256>(b, s, max_items, plan, items, seq_item, nullptr, tid);
        return;
    }
    const int h = (blockIdx.x - 1) % s.H, qw = s.nope + s.rope;
    const int64_t t0 = (int64_t)((blockIdx.x - 1) / s.H) * 16;
    if (tid < 16 && t0 + tid < b.n_rows) {
        const int64_t t = t0 + tid;
        const int i = batch_seq(b, t);
        if (h == 0) tokens[t] = token_of(b, t, i);
        pos[tid] = i >= 0 ? (int64_t)b.lens[i] - b.starts[i + 1] + t : 0;
    }
    constexpr int NB = kAnyRank / 64 / 4;
    f32x4_t acc[NB][4] = {};
    const T* wh = w + (int64_t)h * (s.nope + s.v_dim) * s.rank;
    for (int j0 = 0; j0 < s.nope; j0 += 64) {
        __syncthreads();
        for (int e = tid; e < 16 * 64; e += 256) {
            const int64_t t = t0 + (e >> 6);
            const int j = j0 + (e & 63);
            qs[e >> 6][e & 63] = t < b.n_rows && j < s.nope ? Elem<T>::to_f32(q[(t * s.H + h) * qw + j]) : 0.0f;
        }
        __syncthreads();
        const int n = s.nope - j0 < 64 ? s.nope - j0 : 64;
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const int c = 64 * (wave + 4 * i), at = c + 4 * (lane & 15);
            if (c >= s.rank) break;
            for (int j = 0; j < n; j += 16) {
                f32x4_t a[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int r = j + 4 * k + g;
                    a[k] = load4(wh + (int64_t)(j0 + (r < n ? r : 0)) * s.rank + (at < s.rank ? at : 0));
                    if (r >= n) a[k] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        acc[i][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[k][d], qs[lane & 15][j + 4 * k + g], acc[i][d], 0, 0, 0);
            }
        }
    }
    if (s.nope == 0) __syncthreads();
    const int64_t my_t = t0 + (lane & 15);
    if (my_t < b.n_rows)
#pragma unroll
        for (int i = 0; i < NB; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int c = 64 * (wave + 4 * i) + 16 * g + 4 * e;
                if (c < s.rank)
                    *reinterpret_cast<f32x4_t*>(queries + (my_t * s.H + h) * width + c) = f32x4_t{acc[i][0][e], acc[i][1][e], acc[i][2][e], acc[i][3][e]};
            }
    const int half = s.rope / 2;
    for (int e = tid; e < 16 * half; e += 256) {
        const int64_t t = t0 + e / half;
        const int p = e % half;
        if (t >= b.n_rows) break;
        float c, sn;
        rotary_angle(pos[e / half], rates[p], c, sn);
        const T* r = q + (t * s.H + h) * qw + s.nope;
        const float u = Elem<T>::to_f32(r[p]), v = Elem<T>::to_f32(r[half + p]);
        float* to = queries + (t * s.H + h) * width + s.rank;
        to[p] = u * c - v * sn;
        to[half + p] = v * c + u * sn;
    }
}

// RB: the rank in blocks of 64 columns, rounded up.
template <typename T, int RB>
__global__ __launch_bounds__(256, RB > 4 ? 1 : 2) void any_attend_kernel(const T* __restrict__ pool, Batch b, Shape s, const Plan* plan,
                                                                         const Item* __restrict__ items, const T* __restrict__ zeros,
                                                                         const float* __restrict__ queries, float* __restrict__ sums,
                                                                         float2* __restrict__ stats) {
    __shared__ __align__(16) float qs[kAnyRows * (kAnyWidth + 4)];
    __shared__ __align__(16) float part[4][kAnyRows][64 + 4];
    __shared__ float tops[4][kAnyRows], ls[4][kAnyRows];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, g = lane >> 4, m = lane & 15;
    const int width = s.rank + s.rope, blocks = (width + 63) / 64 * 4, pitch = blocks * 16 + 4;
    const int64_t quota = plan->quota, last = plan->tiles;
    int64_t t = blockIdx.x * quota;
    const int64_t stop = t + quota < last ? t + quota : last;
    if (t >= stop) return;
    int item = find_item(items, plan->n_items, t, lane);
    for (; t < stop; ++item) {
        const Item it = items[item];
        const int64_t begin = item > 0 ? items[item - 1].end : 0;
        const int64_t to = it.end < stop ? it.end : stop;
        if (to <= t) continue;
        for (int e = tid; e < kAnyRows * blocks * 16; e += 256) {
            const int r = e / (blocks * 16), c = e - r * (blocks * 16);
            qs[r * pitch + c] = r < it.rows && c < width ? queries[((int64_t)it.tok0 * s.H + it.row0 + r) * width + c] : 0.0f;
        }
        const int first_pos = it.pos0 + it.row0 / s.H, my_pos = it.pos0 + (it.row0 + (m < it.rows ? m : it.rows - 1)) / s.H;
        const int end = it.pos0 + (it.row0 + it.rows - 1) / s.H + 1;  // keys that some row sees
        const float* my_q = qs + m * pitch + 4 * g;
        __syncthreads();
        f32x4_t o[RB][4] = {};
        float shift = kLowest, l = 0.0f;
        int32_t page = 0;  // of the lane's key, looked up a step before
        auto look_up = [&](int64_t k) {
            const int64_t key = k * kKeys + wave * kAnyKeys + m;
            page = key < end ? batch_page(b, it.seq, key) : -1;
        };
        look_up(t - begin);
        for (int64_t k = t - begin; k < to - begin; ++k) {
            const int key0 = (int)(k * kKeys) + wave * kAnyKeys;  // the wave's first key
            const bool lost = page < 0 && key0 + m < end;          // a key without a page
            const T* row = page < 0 ? zeros : pool + (((int64_t)page << b.page_log) + ((key0 + m) & ((1 << b.page_log) - 1))) * width;
            look_up(k + 1);
            if (key0 >= end) continue;
            f32x4_t x = {0.0f, 0.0f, 0.0f, 0.0f}, y = x;
            for (int j = 0; j < blocks; j += 4) {  // 64 columns at a time
                f32x4_t a[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int c = 16 * (j + i) + 4 * g;
                    a[i] = load4(c < width ? row + c : zeros);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const f32x4_t u = *reinterpret_cast<const f32x4_t*>(my_q + 16 * (j + i));
                    x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][0], u[0], x, 0, 0, 0);
                    y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][1], u[1], y, 0, 0, 0);
                    x = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][2], u[2], x, 0, 0, 0);
                    y = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][3], u[3], y, 0, 0, 0);
                }
            }
            x += y;
            // keys without a page, and rows that only some of the tile see and whose latents are not finite: no result for a
            // row that sees one of them, zeros for the others
            bool bad = lost;
            if (key0 + kAnyKeys - 1 > first_pos)
                for (int c = 4 * g; c < s.rank; c += 16) {
                    const f32x4_t v = load4(row + c);
                    bad |= !(isfinite(v[0]) && isfinite(v[1]) && isfinite(v[2]) && isfinite(v[3]));
                }
            uint64_t odd = ballot(bad);
            odd = (odd | odd >> 16 | odd >> 32 | odd >> 48) & 0xffff;
            float top = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int key = 4 * g + e;
                if ((odd >> key & 1) && key0 + key <= my_pos) l = NAN;
                x[e] = key0 + key > my_pos ? -INFINITY : x[e];
                top = fmaxf(top, x[e]);
            }
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (ballot(top > shift) != 0) {  // some row has a new maximum
                const float before = shift;
                shift = fmaxf(shift, top);
                const float r = exp2f((before - shift) * s.scale2);
                l *= r;
#pragma unroll
                for (int i = 0; i < RB; ++i)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[i][c] *= r;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = exp2f((x[e] - shift) * s.scale2);
                l += p;
                const uint64_t at = (uint64_t)(uintptr_t)row;
                const uint32_t lo = __shfl((int)(uint32_t)at, 4 * g + e, 64), hi = __shfl((int)(uint32_t)(at >> 32), 4 * g + e, 64);
                const T* from = odd >> (4 * g + e) & 1 ? zeros : (const T*)(uintptr_t)((uint64_t)hi << 32 | lo);
#pragma unroll
                for (int i = 0; i < RB; ++i) {
                    const int c = 64 * i + 4 * m;
                    const f32x4_t a = load4(from + (c < s.rank ? c : 0));  // (what lies beyond is not stored)
#pragma unroll
                    for (int d = 0; d < 4; ++d) o[i][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[d], p, o[i][d], 0, 0, 0);
                }
            }
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (g == 0) tops[wave][m] = shift, ls[wave][m] = l;
        __syncthreads();
        float all = tops[0][m], sum = 0.0f;
#pragma unroll
        for (int i = 1; i < 4; ++i) all = fmaxf(all, tops[i][m]);
#pragma unroll
        for (int i = 0; i < 4; ++i) sum += ls[i][m] * exp2f((tops[i][m] - all) * s.scale2);
        const float f = exp2f((shift - all) * s.scale2);
        const int64_t slot = ((int64_t)blockIdx.x + item) * kAnyRows;
        if (wave == 0 && g == 0 && m < it.rows) stats[slot + m] = make_float2(all, sum);
        const int r = tid >> 4, c = (tid & 15) * 4;
#pragma unroll
        for (int i = 0; i < RB; ++i) {
#pragma unroll
            for (int e = 0; e < 4; ++e)
                *reinterpret_cast<f32x4_t*>(&part[wave][m][16 * g + 4 * e]) = f32x4_t{o[i][0][e], o[i][1][e], o[i][2][e], o[i][3][e]} * f;
            __syncthreads();
            if (r < it.rows && 64 * i + c < s.rank) {
                f32x4_t v = *reinterpret_cast<const f32x4_t*>(&part[0][r][c]);
#pragma unroll
                for (int k = 1; k < 4; ++k) v += *reinterpret_cast<const f32x4_t*>(&part[k][r][c]);
                *reinterpret_cast<f32x4_t*>(sums + (slot + r) * s.rank + 64 * i + c) = v;
            }
            __syncthreads();
        }
        t = to;
    }
}

// The parts of a row's sums: n of them, in slots one apart.  `row`: of the token's sequence in a plane; in: its place in a part.
struct Parts {
    int64_t slot;
    int n;
    bool blind;  // its token sees no position: the result is zeros
};
__device__ __forceinline__ Parts row_parts(const Shape& s, const Plan* plan, const Item* items, const int32_t* seq_item, const Token& token,
                                           int64_t row, int plane, int& in) {
    Parts p = {0, 0, false};
    in = 0;
    if (token.seq < 0) return p;
    const int32_t first = seq_item[token.seq];
    if (first < 0) return p;  // there was no room for it
    const int64_t item = first + row / s.rows;
    in = (int)(row % s.rows);
    p.blind = items[item].pos0 + token.index < 0;
    int64_t begin = item > 0 ? items[item - 1].end : 0, end = items[item].end;
    if (end > begin) {
        const int64_t before = plane * (plan->tiles / s.planes);  // the work of the planes before
        begin += before, end += before;
        const int64_t a = begin / plan->quota, z = (end - 1) / plan->quota;
        p.slot = a + (int64_t)plane * plan->n_items + item;
        p.n = (int)(z - a + 1);
    }
    return p;
}
// What a row's sums are multiplied with.  No weight at all (nothing to join, or every score -inf) is no result, NaN, unless the
// token sees nothing.
__device__ __forceinline__ float inverse(float l, bool blind) { return l != 0.0f ? 1.0f / l : blind ? 0.0f : NAN; }

// A workgroup a (token, head), from row t0 of the batch on: joins its row's parts, four columns a thread and as many parts side by side as there are
// threads for, and multiplies with W_v,h, 16 threads a column.
template <typename T>
__global__ __launch_bounds__(256) void any_finish_kernel(const T* __restrict__ w, int64_t t0, Shape s, const Plan* plan,
                                                         const Item* __restrict__ items, const int32_t* __restrict__ seq_item,
                                                         const Token* __restrict__ tokens, const float* __restrict__ sums,
                                                         const float2* __restrict__ stats, T* __restrict__ out) {
    __shared__ __align__(16) float part[1024], o[kAnyRank];
    __shared__ float tops[256], ls[256];
    const int64_t t = t0 + blockIdx.x / s.H;
    const int h = blockIdx.x % s.H, tid = threadIdx.x;
    const Token token = tokens[t];
    if (token.seq == kNoSeq) return;  // behind the last sequence
    const int cols = s.rank / 4, groups = 256 / cols, grp = tid / cols, col = (tid - grp * cols) * 4;
    int in = 0;
    const Parts p = row_parts(s, plan, items, seq_item, token, (int64_t)token.index * s.H + h, 0, in);
    if (grp < groups) {
        float top = kLowest, l = 0.0f;
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = grp; k < p.n; k += 4 * groups) {  // four parts' loads on their way at a time
            float2 ml[4];
            f32x4_t x[4];
            float next = top;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int64_t at = (p.slot + (k + j * groups < p.n ? k + j * groups : k)) * s.rows + in;
                ml[j] = stats[at];
                x[j] = load4(sums + at * s.rank + col);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) next = fmaxf(next, ml[j].x);
            const float r = exp2f((top - next) * s.scale2);
            top = next;
            l *= r;
            v *= r;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (k + j * groups >= p.n) break;
                const float f = exp2f((ml[j].x - top) * s.scale2);
                l = __builtin_fmaf(ml[j].y, f, l);
                v += x[j] * f;
            }
        }
        *reinterpret_cast<f32x4_t*>(part + grp * s.rank + col) = v;
        if (col == 0) tops[grp] = top, ls[grp] = l;
    }
    __syncthreads();
    if (tid < cols) {
        float all = tops[0], l = 0.0f;
        for (int k = 1; k < groups; ++k) all = fmaxf(all, tops[k]);
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < groups; ++k) {
            const float f = exp2f((tops[k] - all) * s.scale2);
            l += ls[k] * f;
            v += *reinterpret_cast<const f32x4_t*>(part + k * s.rank + tid * 4) * f;
        }
        const float inv = inverse(l, p.blind);
        *reinterpret_cast<f32x4_t*>(o + tid * 4) = v * inv;
    }
    __syncthreads();
    for (int j = tid >> 4; j < s.v_dim; j += 16) {
        const T* wr = w + ((int64_t)h * (s.nope + s.v_dim) + s.nope + j) * s.rank;
        float v = 0.0f;
        for (int c = (tid & 15) * 4; c < s.rank; c += 64) {
            const f32x4_t a = load4(wr + c), x = *reinterpret_cast<const f32x4_t*>(o + c);
#pragma unroll
            for (int i = 0; i < 4; ++i) v = __builtin_fmaf(a[i], x[i], v);
        }
#pragma unroll
        for (int k = 1; k < 16; k <<= 1) v += __shfl_xor(v, k, 64);
        if ((tid & 15) == 0) out[(t * s.H + h) * s.v_dim + j] = Elem<T>::from_f32(v);
    }
}

constexpr int any_groups(int num_cus) { return 2 * num_cus; }

template <typename T>
int launch_any(const T* q, const T* w, const T* pool, const Batch& b, const float* rates, Shape s, unsigned char* ws, T* out, int num_cus,
               hipStream_t stream) {
    s.rows = kAnyRows;
    s.groups = any_groups(num_cus);
    const Layout l = layout(b.n_rows, b.n_seq, s.H, s.rank + s.rope, s.rows, s.groups, 4, s.rank);
    Plan* plan = (Plan*)(ws + l.plan);
    Item* items = (Item*)(ws + l.items);
    int32_t* seq_item = (int32_t*)(ws + l.seq_item);
    Token* tokens = (Token*)(ws + l.tokens);
    T* zeros = (T*)(ws + l.specials);
    float *queries = (float*)(ws + l.queries), *sums = (float*)(ws + l.sums);
    float2* stats = (float2*)(ws + l.stats);
    hipLaunchKernelGGL((any_prepare_kernel<T>), dim3((unsigned)((b.n_rows + 15) / 16 * s.H + 1)), dim3(256), 0, stream, q, w, rates, b, s,
                       l.max_items, plan, items, seq_item, tokens, zeros, queries);
    auto attend = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)s.groups), dim3(256), 0, stream, pool, b, s, plan, items, zeros, queries, sums, stats);
    };
    if (s.rank <= 64) attend(any_attend_kernel<T, 1>);
    else if (s.rank <= 128) attend(any_attend_kernel<T, 2>);
    else if (s.rank <= 256) attend(any_attend_kernel<T, 4>);
    else attend(any_attend_kernel<T, 8>);
    // (a launch's threads have to stay below 2^32; the other kernels' do with as many rows as a call may have)
    const int64_t most = ((int64_t)1 << 23) / s.H;
    for (int64_t t0 = 0; t0 < b.n_rows; t0 += most)
        hipLaunchKernelGGL((any_finish_kernel<T>), dim3((unsigned)((b.n_rows - t0 < most ? b.n_rows - t0 : most) * s.H)), dim3(256), 0, stream, w,
                           t0, s, plan, items, seq_item, tokens, sums, stats, out);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------- bf16, rank 256 and rope 64
// Tiles of rows are multiples of 16, the columns of S^T = K Q^T: a lane holds scores of one row, so that its
// maximum, sum and rescaling stay in the lane (and the three others of the row), and the exponentials
// lie as the B operand of O^T = C^T P^T takes them.  C is the latent part of the same rows of K, read from LDS once
// more with the transposing loads, keys in the order in which the scores lie.
//
// A tile of 64 cached rows is 40 KB of LDS in five planes of 64 columns: a copy of 1 KB is then 8 rows of a plane, and a
// lane's rows are the same ones in every plane.  In a plane's row of 128 bytes piece c lies at c ^ swizzle(row): 16
// rows' reads of one piece, and the transposing reads' 4 rows by 4 pieces, touch every bank once.  Rows go from
// memory straight into LDS, eight rows of a page (which has at least eight) and a plane at a time; rows behind the last key
// come from rows of zeros, rows without a page from rows of NaN, so that the loop has no bounds to check.
//
// The products' operands are bf16.  A value that is rounded for one goes in as two, its bf16 value and the bf16 value of
// what that leaves (2^-16 of it): the exponentials, the joined sums before W_v, and 128 of a query's 320 columns (columns weigh
// alike, so any would do: it is the last 64 of the latent's, which one wave forms, and the rotated 64).  With all rounded once the
// outputs' error against 64 bits is 1.9 times that of their own rounding, so it is 1.35 times (0.0022 of their norm; of this the
// queries' other columns are two thirds).  64 sequences of one token: 48.5 -> 49.8 us; 16 of five: 40.5 -> 44.4; all columns of a
// query in two: 54.0 and 48.7, for 1.1 times.
constexpr int kRank = 256, kRope = 64, kWidth = kRank + kRope;
constexpr int kRest = 128, kQuery = kWidth + kRest;  // a row's query, and what bf16 leaves of its last kRest columns
constexpr int kBlockLog = 3, kBlock = 1 << kBlockLog;  // rows of a copy
constexpr int kPlane = kKeys * 128, kStage = kWidth / 64 * kPlane;

typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(3))) bf16x8_t* lds_frag_ptr;
typedef __attribute__((address_space(3))) s16x4_t* lds_tr_ptr;
typedef __attribute__((address_space(3))) u32x4_t* lds_u4_ptr;
typedef __attribute__((address_space(3))) u32x2_t* lds_u2_ptr;
typedef __attribute__((address_space(3))) float* lds_f_ptr;

union Frag {
    u32x4_t u;
    uint32_t w[4];
    bf16x8_t f;
    _Float16 x __attribute__((ext_vector_type(8)));
    s16x4_t h[2];
};

// Two values as bf16, and what that leaves of them, as bf16 too: 16 bits of precision in two products.
__device__ __forceinline__ void split_bf16x2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_bf16x2(a, b);
    lo = pack_bf16x2(a - __uint_as_float(hi << 16), b - __uint_as_float(hi & 0xffff0000u));
}

__device__ __forceinline__ int swizzle(int row) { return ((row >> 1) & 1) << 2 | ((row >> 2) & 1) << 1 | ((row >> 3) & 1); }

// 16 bytes a lane into LDS at lds + 16 times the lane (lds: wave-uniform), from an address or from base + off.
// The caller waits (vmcnt).
__device__ __forceinline__ void copy16(const void* p, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(p) : "memory");
}
__device__ __forceinline__ void copy16(const void* base, uint32_t off, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(off), "s"(base) : "memory");
}
// This wave's copies but the last N have landed and its LDS accesses are done, and so with every wave.
template <int N>
__device__ __forceinline__ void copies_barrier() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory"); }
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The order of a stretch of code between branches: N LDS reads, then M times a matrix product and R reads, then the
// last products (left to itself the compiler reads one fragment ahead, and every product waits for LDS).  P products at a time.
template <int N, int M, int R, int L, int P = 1>
__device__ __forceinline__ void reads_ahead() {
    __builtin_amdgcn_sched_group_barrier(0x100, N, 0);
#pragma unroll
    for (int i = 0; i < M; ++i) {
        __builtin_amdgcn_sched_group_barrier(0x8, P, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x8, L, 0);
}

constexpr int kSeqsNear = 1024;

// Block 0: the plan and the two special rows.  The others: 32 tokens of a head; [c][token] = W_k,h^T q^T, the weight
// (k as the row) through LDS in the layout of the loss's R tiles.  64 sequences of a token, 16 heads: 7 to 8 us for 1.3 MB,
// which is the launch and three loads that wait for each other; the plan takes as long beside it.
__global__ __launch_bounds__(256) void prepare_kernel(const uint16_t* __restrict__ q, const uint16_t* __restrict__ w,
                                                      const float* __restrict__ rates, Batch b, Shape s, int64_t max_items, Plan* plan,
                                                      Item* items, int32_t* seq_item, Token* tokens, uint16_t* __restrict__ specials,
                                                      uint16_t* __restrict__ queries) {
    __shared__ __align__(16) uint16_t ws[64 * kRank];
    __shared__ int64_t pos[32];
    __shared__ int32_t starts[kSeqsNear], lens[kSeqsNear];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (blockIdx.x == 0) {
        for (int e = tid; e < 2 * kBlock * kWidth; e += 256) specials[e] = e < kBlock * kWidth ? 0 : 0x7fc0;
        make_plan<256>(b, s, max_items, plan, items, seq_item, nullptr, tid);
        return;
    }
    const int h = (blockIdx.x - 1) % s.H, qw = s.nope + kRope;
    const int64_t t0 = (int64_t)((blockIdx.x - 1) / s.H) * 32;
    const int64_t my_t = t0 + (lane & 31) < b.n_rows ? t0 + (lane & 31) : b.n_rows - 1;
    const uint16_t* qp = q + (my_t * s.H + h) * qw;
    f32x16_t acc[2] = {f32x16_zero(), f32x16_zero()};
    // the tokens' positions, by a search in LDS where there is room for the sequences
    auto find_positions = [&]() {
        const bool near = b.n_seq < kSeqsNear;
        if (near) {
            for (int i = tid; i <= b.n_seq; i += 256) starts[i] = b.starts[i];
            for (int i = tid; i < b.n_seq; i += 256) lens[i] = b.lens[i];
            __syncthreads();
        }
        if (tid < 32 && t0 + tid < b.n_rows) {
            const int64_t t = t0 + tid;
            Batch c = b;
            if (near) c.starts = starts, c.lens = lens;
            const int i = batch_seq(c, t);
            if (h == 0) tokens[t] = token_of(c, t, i);
            pos[tid] = i >= 0 ? (int64_t)c.lens[i] - c.starts[i + 1] + t : 0;
        }
    };
    // the queries' last parts: four of the 32 tokens by 32 angles a thread, read first and turned while the weight is on
    // its way
    float2 ends[4];
    const int p = tid & 31;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t t = t0 + (tid >> 5) + 8 * i;
        const uint16_t* r = q + ((t < b.n_rows ? t : b.n_rows - 1) * s.H + h) * qw + s.nope;
        ends[i] = make_float2(bf16_bits_to_f32(r[p]), bf16_bits_to_f32(r[32 + p]));
    }
    const float rate = rates[p];
    auto turn_ends = [&]() {
        find_positions();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = (tid >> 5) + 8 * i;
            if (t0 + at >= b.n_rows) break;
            float c, sn;
            rotary_angle(pos[at], rate, c, sn);
            uint16_t* to = queries + ((t0 + at) * s.H + h) * kQuery + kRank;
            uint32_t hi, lo;
            split_bf16x2(ends[i].x * c - ends[i].y * sn, ends[i].y * c + ends[i].x * sn, hi, lo);
            to[p] = (uint16_t)hi;
            to[32 + p] = (uint16_t)(hi >> 16);
            to[kRest + p] = (uint16_t)lo;
            to[kRest + 32 + p] = (uint16_t)(lo >> 16);
        }
    };
    if (s.nope == 0) turn_ends();
    for (int j0 = 0; j0 < s.nope; j0 += 64) {
        const int rows = s.nope - j0 < 64 ? s.nope - j0 : 64;
        const uint16_t* wh = w + ((int64_t)h * (s.nope + s.v_dim) + j0) * kRank;
        u32x4_t part[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = (tid >> 5) + 8 * i;
            part[i] = *reinterpret_cast<const u32x4_t*>(wh + (int64_t)(r < rows ? r : rows - 1) * kRank + (tid & 31) * 8);
        }
        if (j0 == 0) turn_ends();
        else __syncthreads();
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int r = (tid >> 5) + 8 * i;
            *reinterpret_cast<u32x4_t*>(ws + r * kRank + (((tid & 31) ^ ((r & 3) << 2)) * 8)) = part[i];
        }
        __syncthreads();
        const uint32_t lds = lds_addr(ws);
        const int k = 8 * half + ((lane & 15) >> 2);
        for (int st = 0; st < rows / 16; ++st) {
            Frag x;
            x.u = *reinterpret_cast<const u32x4_t*>(qp + j0 + 16 * st + 8 * half);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int c = wave * 8 + i * 4 + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
                const uint32_t at = lds + (16 * st + k) * (kRank * 2) + ((c ^ ((k & 3) << 2)) << 4) + (lane & 1) * 8;
                Frag a;
                a.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)at);
                a.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(at + 4 * kRank * 2));
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.f, x.f, acc[i], 0, 0, 0);
            }
        }
    }
    if (t0 + (lane & 31) < b.n_rows) {
        uint16_t* to = queries + (my_t * s.H + h) * kQuery + wave * 64 + 4 * half;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                uint2 hi, lo;
                split_bf16x2(acc[i][e], acc[i][e + 1], hi.x, lo.x);
                split_bf16x2(acc[i][e + 2], acc[i][e + 3], hi.y, lo.y);
                *reinterpret_cast<uint2*>(to + 32 * i + 2 * e) = hi;
                if (wave * 64 >= kWidth - kRest) *reinterpret_cast<uint2*>(to + kRest + 32 * i + 2 * e) = lo;
            }
    }
}

// WR KW waves: WR share a tile of 16 WR rows, 16 each, KW the 64 keys of a step.  S stages of LDS.  64 sequences of one token and up
// to 8,192 keys: 186 MB in 36.3 us, 5.1 TB/s (256 of 2,048: 335 MB in 62, 5.4), where plain streaming reads reach 5.6, with eight
// loads of a thread in flight 6.3, and a large copy moves 4.95: near memory's rate.  16 of five tokens and up to 4,096: 23 MB of
// cache in 24.9 us, three steps a workgroup.  LDS reads (a fragment serves 16 rows) account for some 4 us of that and the products
// for 5 at most; reading the queries and writing 16 MB of sums lie around the steps; the rest has not been told apart.
template <int WR, int KW, int S>
__global__ __launch_bounds__(WR * KW * 64, 2) void attend_kernel(const uint16_t* __restrict__ pool, Batch b, Shape s, const Plan* plan,
                                                                 const Item* __restrict__ items, const uint16_t* __restrict__ queries,
                                                                 const uint16_t* __restrict__ specials, float* __restrict__ sums,
                                                                 float2* __restrict__ stats) {
    constexpr int W = WR * KW, KB = 4 / KW, NB = 8 / W, NC = NB * (kWidth / 64), RT = 16 * WR;
    __shared__ __align__(16) unsigned char ring[S * kStage];
    const int tid = threadIdx.x, lane = tid & 63, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6), wr = wave / KW, wk = wave % KW;
    const uint32_t lds = lds_addr(ring);
    const int64_t quota = plan->quota, last = plan->tiles;
    int64_t t = blockIdx.x * quota;
    const int64_t stop = t + quota < last ? t + quota : last;
    if (t >= stop) return;

    // LDS places of the fragments: K's two steps of a plane, and C's four blocks of 16 columns of one
    uint32_t k_at[2], c_at[4];
    const int wave_key = 16 * KB * wk;
    {
        const int key = wave_key + (lane & 15), row = wave_key + 4 * g + ((lane & 15) >> 2);
#pragma unroll
        for (int i = 0; i < 2; ++i) k_at[i] = key * 128 + (((4 * i + g) ^ swizzle(key)) << 4);
#pragma unroll
        for (int d = 0; d < 4; ++d) c_at[d] = row * 128 + (((2 * d + ((lane & 3) >> 1)) ^ swizzle(row)) << 4) + (lane & 1) * 8;
    }

    int item = find_item(items, plan->n_items, t, lane);
    for (; t < stop; ++item) {
        const Item it = items[item];
        const int64_t begin = item > 0 ? items[item - 1].end : 0;
        const int64_t to = it.end < stop ? it.end : stop;
        if (to <= t) continue;
        const int k_begin = (int)(t - begin), k_end = (int)(to - begin);
        const int row_last = it.rows - 1;
        const int end = it.pos0 + (it.row0 + row_last) / s.H + 1;  // keys that some row sees
        const int first_pos = it.pos0 + it.row0 / s.H;
        const int my = wr * 16 + (lane & 15), my_row = my < row_last ? my : row_last;
        const int my_pos = it.pos0 + (it.row0 + my_row) / s.H;
        const int wave_row = wr * 16 < row_last ? wr * 16 : row_last;
        const int wave_pos = it.pos0 + (it.row0 + wave_row) / s.H;  // its first row's
        // (as constant memory: loads by the scalar unit, which do not queue behind the copies)
        const auto table = (const __attribute__((address_space(4))) int32_t*)(uintptr_t)(b.table + it.seq * b.table_ld);

        // page numbers of the rows that this wave copies of a step, and the copies
        int32_t pages[NB];
        auto load_pages = [&](int k) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int at = (int)((uint32_t)(k * kKeys + (wave * NB + i) * kBlock) >> b.page_log);
                pages[i] = table[at < b.width ? at : b.width - 1];
            }
        };
        auto copy_rows = [&](int k, int stage) {
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int blk = wave * NB + i, p0 = k * kKeys + blk * kBlock;
                const int32_t page = pages[i];
                const uint16_t* from = page >= 0 && page < b.n_pages
                                           ? pool + (((int64_t)page << b.page_log) + (p0 & ((1 << b.page_log) - 1))) * kWidth
                                           : specials + kBlock * kWidth;
                if (p0 >= end) from = specials;
                const int row = lane >> 3;
                const uint32_t off = row * (kWidth * 2) + (((lane & 7) ^ swizzle(blk * kBlock + row)) << 4);
                const uint32_t to_lds = lds + stage * kStage + blk * 1024;
                if (p0 < end && p0 + kBlock > end) {  // the sequence ends in this block
                    const unsigned char* mine = (const unsigned char*)(p0 + row < end ? from : specials) + off;
#pragma unroll
                    for (int pl = 0; pl < kWidth / 64; ++pl) copy16(mine + pl * 128, __builtin_amdgcn_readfirstlane(to_lds + pl * kPlane));
                } else {
#pragma unroll
                    for (int pl = 0; pl < kWidth / 64; ++pl) copy16(from + pl * 64, off, __builtin_amdgcn_readfirstlane(to_lds + pl * kPlane));
                }
            }
        };

        // zeros for the latents of these rows, by all waves, once every wave has its scores
        auto clear_odd = [&](uint64_t odd, uint32_t at) {
            lds_barrier();
            for (int e = tid; e < kKeys * 32; e += W * 64) {
                const int r = e & 63, c = e >> 6;
                if (odd >> r & 1) *(lds_u4_ptr)(size_t)(at + (c >> 3) * kPlane + r * 128 + (c & 7) * 16) = u32x4_t{0, 0, 0, 0};
            }
            lds_barrier();
        };
        const bool active = wr * 16 < it.rows;  // (a wave without rows of its own copies only)
        load_pages(k_begin);
        Frag fq[kQuery / 32];
        {
            const uint16_t* qp = queries + ((int64_t)it.tok0 * s.H + it.row0 + my_row) * kQuery + 8 * g;
#pragma unroll
            for (int i = 0; i < kQuery / 32; ++i) fq[i].u = *reinterpret_cast<const u32x4_t*>(qp + 32 * i);
            // (here, not in the loop, is where they are waited for)
#pragma unroll
            for (int i = 0; i < kQuery / 32; ++i) asm volatile("" : "+v"(fq[i].u));
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
        for (int i = 0; i < S - 1; ++i)
            if (k_begin + i < k_end) {
                copy_rows(k_begin + i, i);
                load_pages(k_begin + i + 1);
            }

        f32x4_t o[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        float shift = kLowest, l = 0.0f;  // the running maximum of the scores, and the lane's part of the sum
        int stage = 0;
        for (int k = k_begin; k < k_end; ++k) {
            if (S == 3 && k + 1 < k_end) copies_barrier<(S - 2) * NC>();
            else copies_barrier<0>();
            if (k + S - 1 < k_end) {
                copy_rows(k + S - 1, stage == 0 ? S - 1 : stage - 1);
                load_pages(k + S);
            }
            const uint32_t at = lds + stage * kStage;
            const int key0 = k * kKeys + wave_key;  // the wave's first key
            stage = stage == S - 1 ? 0 : stage + 1;
            // rows that some of the tile's rows do not see may hold anything: those whose latents are not finite
            uint64_t odd = 0;
            if (first_pos < end - 1 && k * kKeys + kKeys - 1 > first_pos) {
                // (each wave by itself, four of those rows at a time, 16 lanes a row)
                const int seen = first_pos + 1 - k * kKeys, stop_row = end - k * kKeys < kKeys ? end - k * kKeys : kKeys;
                for (int r0 = seen > 0 ? seen : 0; r0 < stop_row; r0 += 4) {
                    const int r = r0 + g;
                    bool bad = false;
                    if (r < stop_row)
#pragma unroll
                        for (int c = 0; c < kRank / 64; c += 2) {
                            const u32x4_t v = *(lds_u4_ptr)(size_t)(at + (c + ((lane >> 3) & 1)) * kPlane + r * 128 + ((lane & 7) << 4));
#pragma unroll
                            for (int i = 0; i < 4; ++i) bad |= (v[i] & 0x7f80u) == 0x7f80u || (v[i] & 0x7f800000u) == 0x7f800000u;
                        }
                    const uint64_t some = ballot(bad);
#pragma unroll
                    for (int i = 0; i < 4; ++i) odd |= (uint64_t)((some >> (16 * i) & 0xffff) != 0) << ((r0 + i) & 63);
                }
            }
            f32x4_t x[KB];
            if (odd != 0 && !active) clear_odd(odd, at);
            if (!active) continue;
#pragma unroll
            for (int i = 0; i < KB; ++i) x[i] = f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int st = 0; st < kWidth / 32; ++st)
#pragma unroll
                for (int i = 0; i < KB; ++i) {
                    const bf16x8_t a = *(lds_frag_ptr)(size_t)(at + k_at[st & 1] + (st >> 1) * kPlane + i * 16 * 128);
                    x[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, fq[st].f, x[i], 0, 0, 0);
                    if (st >= (kWidth - kRest) / 32) x[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, fq[st + kRest / 32].f, x[i], 0, 0, 0);
                }
            reads_ahead<8, KB * kWidth / 32 - 8, 1, 8 + KB * kRest / 32>();
            if (key0 + 16 * KB - 1 > wave_pos) {
#pragma unroll
                for (int i = 0; i < KB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[i][e] = key0 + 16 * i + 4 * g + e > my_pos ? -INFINITY : x[i][e];
            }
            if (odd != 0) {
                // a row that sees one of them has no result; for the others they are zeros
#pragma unroll
                for (int i = 0; i < KB; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = 16 * i + 4 * g + e;
                        if ((odd >> (wave_key + key) & 1) && key0 + key <= my_pos) l = NAN;
                    }
                clear_odd(odd, at);
            }
            float top = x[0][0];
#pragma unroll
            for (int i = 0; i < KB; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) top = fmaxf(top, x[i][e]);
            top = fmaxf(top, __shfl_xor(top, 16, 64));
            top = fmaxf(top, __shfl_xor(top, 32, 64));
            if (ballot(top > shift) != 0) {  // some row has a new maximum
                const float before = shift;
                shift = fmaxf(shift, top);
                const float r = __builtin_amdgcn_exp2f((before - shift) * s.scale2);
                l *= r;
#pragma unroll
                for (int i = 0; i < 16; ++i) o[i] *= r;
            }
            Frag p[KB / 2], rest[KB / 2];
#pragma unroll
            for (int i = 0; i < KB; ++i) {
                float e[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) e[j] = __builtin_amdgcn_exp2f((x[i][j] - shift) * s.scale2);
                l += (e[0] + e[1]) + (e[2] + e[3]);
#pragma unroll
                for (int j = 0; j < 2; ++j) split_bf16x2(e[2 * j], e[2 * j + 1], p[i / 2].w[(i & 1) * 2 + j], rest[i / 2].w[(i & 1) * 2 + j]);
            }
#pragma unroll
            for (int i = 0; i < KB / 2; ++i)
#pragma unroll
                for (int d = 0; d < 16; d += 2) {
                    Frag a[2];
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t c = at + (d >> 2) * kPlane + i * 32 * 128 + c_at[(d + j) & 3];
                        a[j].h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)c);
                        a[j].h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(c + 16 * 128));
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) o[d + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j].f, p[i].f, o[d + j], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 2; ++j) o[d + j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[j].f, rest[i].f, o[d + j], 0, 0, 0);
                }
            reads_ahead<12, 8 * KB / 2 - 3, 4, 12, 4>();
        }
        l += __shfl_xor(l, 16, 64);
        l += __shfl_xor(l, 32, 64);
        lds_barrier();
        if constexpr (KW == 2) {
            // the second wave's sums join the first's through LDS
            static_assert(WR * 66 * 256 <= S * kStage, "both waves' sums fit the ring");
            const uint32_t mine = lds + wr * 66 * 256 + lane * 4;
            if (wk == 1) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) *(lds_f_ptr)(size_t)(mine + (i * 4 + e) * 256) = o[i][e];
                *(lds_f_ptr)(size_t)(mine + 64 * 256) = shift;
                *(lds_f_ptr)(size_t)(mine + 65 * 256) = l;
            }
            lds_barrier();
            if (wk == 0) {
                const float other = *(lds_f_ptr)(size_t)(mine + 64 * 256), l2 = *(lds_f_ptr)(size_t)(mine + 65 * 256);
                const float both = fmaxf(shift, other);
                const float f = __builtin_amdgcn_exp2f((shift - both) * s.scale2), f2 = __builtin_amdgcn_exp2f((other - both) * s.scale2);
                shift = both;
                l = l * f + l2 * f2;
#pragma unroll
                for (int i = 0; i < 16; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[i][e] = o[i][e] * f + *(lds_f_ptr)(size_t)(mine + (i * 4 + e) * 256) * f2;
            }
            lds_barrier();
        }
        if (wk == 0 && my < it.rows) {
            const int64_t slot = ((int64_t)blockIdx.x + item) * RT + my;
            float* y = sums + slot * kRank + 4 * g;
#pragma unroll
            for (int i = 0; i < 16; ++i) *reinterpret_cast<f32x4_t*>(y + 16 * i) = o[i];
            if (g == 0) stats[slot] = make_float2(shift, l);
        }
        t = to;
    }
}

// TOK tokens of a head: 256 / TOK threads a token join its parts, 16 columns a thread and 16 / TOK parts side by side,
// then [v][token] = W_v,h o^T by 16 x 16 x 32 MFMAs, a wave for every 16 of v_dim.  64 tokens of 16 heads and up to 16 parts: 7 us
// for 20 MB of sums; one token's 256 parts: 10 us.  Bound by the chain token, tile, parts, sums: each read waits for the last.
template <int TOK>
__global__ __launch_bounds__(256) void finish_kernel(const uint16_t* __restrict__ w, int64_t n_rows, Shape s, const Plan* plan,
                                                     const Item* __restrict__ items, const int32_t* __restrict__ seq_item,
                                                     const Token* __restrict__ tokens, const float* __restrict__ sums,
                                                     const float2* __restrict__ stats, uint16_t* __restrict__ out) {
    constexpr int G = 16 / TOK;  // groups of 16 threads that share a token
    __shared__ __align__(16) uint16_t os[2][TOK][kRank + 8];
    __shared__ __align__(16) float part[G > 1 ? 16 : 1][kRank];
    __shared__ float tops[16], ls[16];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int h = blockIdx.x % s.H;
    const int64_t t0 = (int64_t)(blockIdx.x / s.H) * TOK;
    const int grp = tid >> 4, tok = grp / G, sub = grp % G, col = (tid & 15) * 4;
    const int64_t t = t0 + tok;
    // (the weight's first fragments, on their way meanwhile)
    bf16x8_t first[kRank / 32];
    const uint16_t* wv = w + ((int64_t)h * (s.nope + s.v_dim) + s.nope + (lane & 15)) * kRank + 8 * (lane >> 4);
#pragma unroll
    for (int st = 0; st < kRank / 32; ++st)
        first[st] = *reinterpret_cast<const bf16x8_t*>(wv + (int64_t)(wave * 16 < s.v_dim ? wave * 16 : 0) * kRank + 32 * st);
    const Token token = t < n_rows ? tokens[t] : Token{kNoSeq, 0};
    int in;
    const Parts p = row_parts(s, plan, items, seq_item, token, (int64_t)token.index * s.H + h, 0, in);
    float top = kLowest, l = 0.0f, v[16] = {};
    for (int k = sub; k < p.n; k += 4 * G) {  // four parts' loads on their way at a time
        float2 ml[4];
        f32x4_t x[4][4];
        float next = top;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t at = (p.slot + (k + j * G < p.n ? k + j * G : k)) * s.rows + in;
            ml[j] = stats[at];
#pragma unroll
            for (int c = 0; c < 4; ++c) x[j][c] = *reinterpret_cast<const f32x4_t*>(sums + at * kRank + c * 64 + col);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) next = fmaxf(next, ml[j].x);
        const float r = __builtin_amdgcn_exp2f((top - next) * s.scale2);
        top = next;
        l *= r;
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] *= r;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (k + j * G >= p.n) break;
            const float f = __builtin_amdgcn_exp2f((ml[j].x - top) * s.scale2);
            l = __builtin_fmaf(ml[j].y, f, l);
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = __builtin_fmaf(x[j][e >> 2][e & 3], f, v[e]);
        }
    }
    if constexpr (G > 1) {
#pragma unroll
        for (int c = 0; c < 4; ++c) *reinterpret_cast<f32x4_t*>(&part[grp][c * 64 + col]) = f32x4_t{v[4 * c], v[4 * c + 1], v[4 * c + 2], v[4 * c + 3]};
        if ((tid & 15) == 0) tops[grp] = top, ls[grp] = l;
        __syncthreads();
        // thread by thread again: token tid / (256 / TOK), columns of 16 G threads
        const int mine = tok * G;
        float all = tops[mine], sum = 0.0f, f[G];
#pragma unroll
        for (int g = 1; g < G; ++g) all = fmaxf(all, tops[mine + g]);
#pragma unroll
        for (int g = 0; g < G; ++g) {
            f[g] = __builtin_amdgcn_exp2f((tops[mine + g] - all) * s.scale2);
            sum += ls[mine + g] * f[g];
        }
        const float inv = inverse(sum, p.blind);
#pragma unroll
        for (int c = 0; c < TOK; ++c) {
            const int at = c * 16 * G + (sub * 16 + (tid & 15));
            float x = 0.0f;
#pragma unroll
            for (int g = 0; g < G; ++g) x += part[mine + g][at] * f[g];
            const uint16_t hi = f32_to_bf16_bits(x * inv);
            os[0][tok][at] = hi;
            os[1][tok][at] = f32_to_bf16_bits(x * inv - bf16_bits_to_f32(hi));
        }
    } else {
        const float inv = inverse(l, p.blind);
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            uint2 hi, lo;
            split_bf16x2(v[4 * c] * inv, v[4 * c + 1] * inv, hi.x, lo.x);
            split_bf16x2(v[4 * c + 2] * inv, v[4 * c + 3] * inv, hi.y, lo.y);
            *reinterpret_cast<uint2*>(&os[0][tok][c * 64 + col]) = hi;
            *reinterpret_cast<uint2*>(&os[1][tok][c * 64 + col]) = lo;
        }
    }
    __syncthreads();
    const int tc = (lane & 15) < TOK ? lane & 15 : TOK - 1;
    const int64_t to = t0 + (lane & 15);
    const bool live = (lane & 15) < TOK && to < n_rows && tokens[to].seq != kNoSeq;
    for (int vb = wave; vb < s.v_dim / 16; vb += 4) {
        f32x4_t acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int st = 0; st < kRank / 32; ++st) {
            const bf16x8_t a = vb == wave ? first[st] : *reinterpret_cast<const bf16x8_t*>(wv + (int64_t)vb * 16 * kRank + 32 * st);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const bf16x8_t x = *reinterpret_cast<const bf16x8_t*>(&os[half][tc][32 * st + 8 * (lane >> 4)]);
                acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, x, acc, 0, 0, 0);
            }
        }
        if (live)
            *reinterpret_cast<uint2*>(out + (to * s.H + h) * s.v_dim + vb * 16 + 4 * (lane >> 4)) =
                make_uint2(pack_bf16x2(acc[0], acc[1]), pack_bf16x2(acc[2], acc[3]));
    }
}

bool is_fast(int rank, int rope, int nope, int v_dim, int page_log, int dtype) {
    return dtype == kBF16 && rank == kRank && rope == kRope && nope % 16 == 0 && v_dim % 16 == 0 && page_log >= kBlockLog;
}

// Rows of a tile: as many as a sequence's new tokens have on the average, 32 to 128.  us, 64 sequences of up to 8,192 keys and 16
// heads: two tokens 59.1 (tiles of 16: 75.1), four 74.4 in tiles of 64, 81.9 of 128, 83.3 of 32; 16 sequences, two tokens 37.5
// in tiles of 32, 40.7 of 64.  (One token in tiles of 16: 50.0 and 30.2, of 32: 50.6 and 29.1; there are none of 16.)
int fast_rows(int64_t n_rows, int n_seq, int H) {
    const int64_t each = n_rows * H / n_seq;
    return each <= 32 ? 32 : each <= 64 ? 64 : 128;
}
// Workgroups of 32 rows leave room for a second one on their CU (64 sequences of one token: 55.4 us with one, 50.0 with two).
int fast_groups(int rows, int num_cus) { return rows <= 32 ? 2 * num_cus : num_cus; }

int launch_fast(const uint16_t* q, const uint16_t* w, const uint16_t* pool, const Batch& b, const float* rates, Shape s, unsigned char* ws,
                uint16_t* out, int num_cus, hipStream_t stream) {
    s.rows = fast_rows(b.n_rows, b.n_seq, s.H);
    s.groups = fast_groups(s.rows, num_cus);
    const Layout l = layout(b.n_rows, b.n_seq, s.H, kQuery, s.rows, s.groups, 2, kRank);
    Plan* plan = (Plan*)(ws + l.plan);
    Item* items = (Item*)(ws + l.items);
    int32_t* seq_item = (int32_t*)(ws + l.seq_item);
    Token* tokens = (Token*)(ws + l.tokens);
    uint16_t *specials = (uint16_t*)(ws + l.specials), *queries = (uint16_t*)(ws + l.queries);
    float* sums = (float*)(ws + l.sums);
    float2* stats = (float2*)(ws + l.stats);
    const unsigned tiles = (unsigned)((b.n_rows + 31) / 32);
    hipLaunchKernelGGL(prepare_kernel, dim3(tiles * s.H + 1), dim3(256), 0, stream, q, w, rates, b, s, l.max_items, plan, items, seq_item,
                       tokens, specials, queries);
    auto attend = [&](auto kernel, int threads) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)s.groups), dim3(threads), 0, stream, pool, b, s, plan, items, queries, specials, sums, stats);
    };
    if (s.rows == 32) attend(attend_kernel<2, 2, 2>, 256);
    else if (s.rows == 64) attend(attend_kernel<4, 2, 3>, 512);
    else attend(attend_kernel<8, 1, 3>, 512);
    // The more parts a row may have, the more threads join them.  us, with a token in 256 | 64 | 16 threads: one token of 65,536
    // keys (256 parts) 29.4 | 44.6 | -, 16 sequences of 8,192 (32) 32.4 | 34.6 | 43.0, 16 of 4,096 and 5 tokens (16) - | 43.6 | 48.2,
    // 64 of 4,096 (8) 47.6 | 45.3 | 46.8, 128 of 2,048 (4) 46.1 | 46.2 | 45.4, 256 of 2,048 (2) 79.7 | 80.0 | 76.8.
    const int64_t tiles_of_rows = b.n_rows * s.H / s.rows, parts = s.groups / (tiles_of_rows > b.n_seq ? tiles_of_rows : b.n_seq);
    auto finish = [&](auto kernel, int tokens_each) {
        hipLaunchKernelGGL(kernel, dim3((unsigned)((b.n_rows + tokens_each - 1) / tokens_each * s.H)), dim3(256), 0, stream, w, b.n_rows, s, plan,
                           items, seq_item, tokens, sums, stats, out);
    };
    if (parts >= 32) finish(finish_kernel<1>, 1);
    else if (parts >= 8) finish(finish_kernel<4>, 4);
    else finish(finish_kernel<16>, 16);
    return (int)hipGetLastError();
}

// ------------------------------------------------------------------------- many new tokens a sequence
// The same weight may go to the keys and values instead, once for each cached row and head: 65 K operations a
// row and head, after which a (token, head, key) takes 384 instead of 1,152.  That is the shorter way from some
// kChunkRows new tokens a sequence on.  Keys and values of a head lie one sequence behind the other, 64 | 64 columns a row,
// each sequence's rows filled up with zeros to a multiple of 64; the keys' rotated parts, which the heads share, likewise.
// The attention is then that of any causal head: 128 tokens of a head a workgroup, 32 a wave, keys in steps of 64,
// and heads as the outer dimension of the even shares, so that an XCD's workgroups read the same two heads' keys from its L2.
//
// Queries, keys, values and exponentials are fp16 there, of 11 bits instead of bf16's 8: the outputs' error against 64 bits
// is that of their own rounding (with bf16 up to twice that; 120.9 -> 124.6 us for 2,048 tokens, 7,001 keys, 16 heads).  For
// their range queries and keys are 2^-4 of themselves, values 2^-2, and a row's exponentials 2^6 at its maximum: a query or
// key of 2^20 or a value of 2^18 and more counts as infinite; fp16's steps near zero are 2^-20 of a key, 2^-22 of a value
// and 2^-30 of a weight, as fine as bf16's where a key is 2^-13 or more and a value 2^-15.
constexpr float kKeyScale = 0x1p-4f, kValueScale = 0x1p-2f, kQueryScale = 0x1p-4f, kTop = 6.0f;
constexpr int kHead = 64;         // columns of a head's keys (before the rotated ones) and of its values
constexpr int kChunkTok = 128;    // tokens of a tile
// New tokens a sequence, on the average, from which this is the shorter way.  It is measured on sequences that are alike; a batch
// of others takes one form all the same, and is right in either, but slower than two calls: a chunk of 2,048 tokens over 7,001 keys
// (129 us by itself) beside 63 single tokens of up to 8,192 keys (53) 489, beside four of 50,000 (41), whose keys are all formed
// for one token each, 802.  us, the weight with the queries | with the keys and
// values: 8 sequences of 4,096 keys, 64 tokens 92.5 | 115.0, 96 128.2 | 113.0, 128 158.0 | 115.6; one of 4,096, 64 tokens
// 43.5 | 48.5, 128 57.4 | 53.5, 256 73.4 | 50.2; one of 16,384, 128 tokens 96.4 | 81.8.
constexpr int kChunkRows = 96;
// Keys and values that a call may form, by what its table could hold: a limit on the workspace, not where the other form would be
// shorter.  Four sequences of 512 tokens over 65,000 keys: 1,549 us; over 66,000, beyond it: 3,562.
constexpr size_t kChunkBytes = (size_t)1 << 30;

struct ChunkLayout {
    size_t plan, items, seq_item, tokens, seq_keys, specials, turns, keys, shared, sums, stats, bytes;
    int64_t max_items, key_rows;
};

ChunkLayout chunk_layout(int64_t n_rows, int n_seq, int H, int64_t capacity, int groups) {
    ChunkLayout l;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t p = at;
        at += round256(bytes);
        return p;
    };
    l.max_items = n_rows / kChunkTok + n_seq;
    l.key_rows = n_seq * ((capacity + kKeys - 1) / kKeys * kKeys);
    l.plan = take(sizeof(Plan));
    l.items = take((size_t)l.max_items * sizeof(Item));
    l.seq_item = take((size_t)n_seq * 4);
    l.tokens = take((size_t)n_rows * sizeof(Token));
    l.seq_keys = take((size_t)(n_seq + 1) * 4);
    l.specials = take((size_t)16 * kWidth * 2);
    l.turns = take((size_t)n_rows * kRope / 2 * 8);
    l.keys = take((size_t)l.key_rows * H * 2 * kHead * 2);
    l.shared = take((size_t)l.key_rows * kRope * 2);
    const size_t slots = (size_t)(l.max_items * H + groups);
    l.sums = take(slots * kChunkTok * kHead * 4);
    l.stats = take(slots * kChunkTok * 8);
    l.bytes = at;
    return l;
}

// Block 0: the plan.  The others: eight tokens' sequences, cosines and sines.
__global__ __launch_bounds__(256) void chunk_prepare_kernel(const float* __restrict__ rates, Batch b, Shape s, int64_t max_items, Plan* plan,
                                                            Item* items, int32_t* seq_item, int32_t* seq_keys, Token* tokens,
                                                            uint16_t* __restrict__ specials, float2* __restrict__ turns) {
    if (blockIdx.x == 0) {
        for (int e = threadIdx.x; e < 2 * kBlock * kWidth; e += 256) specials[e] = e < kBlock * kWidth ? 0 : 0x7fc0;
        Shape one = s;
        one.H = 1;
        make_plan<256>(b, one, max_items, plan, items, seq_item, seq_keys, threadIdx.x);
        return;
    }
    const int64_t t = (int64_t)(blockIdx.x - 1) * 8 + (threadIdx.x >> 5);
    const int p = threadIdx.x & 31;
    const int64_t wave_t = t - ((threadIdx.x >> 5) & 1);  // the wave's two tokens
    int seq[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) seq[i] = wave_t + i < b.n_rows ? batch_seq_wave(b, wave_t + i, threadIdx.x & 63) : kNoSeq;
    if (t >= b.n_rows) return;
    const int i = (threadIdx.x & 32) ? seq[1] : seq[0];
    if (p == 0) tokens[t] = token_of(b, t, i);
    if (i < 0) return;
    float2 c;
    rotary_angle((int64_t)b.lens[i] - b.starts[i + 1] + t, rates[p], c.x, c.y);
    turns[t * 32 + p] = c;
}

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(3))) f16x8_t* lds_half_ptr;
__device__ __forceinline__ uint32_t pack_f16x2(float a, float b) { return __builtin_bit_cast(uint32_t, f16x2_t{(_Float16)a, (_Float16)b}); }
// Two bf16 values, times a scale, as fp16.
__device__ __forceinline__ uint32_t f16_of_bf16x2(uint32_t v, float scale) {
    return pack_f16x2(__uint_as_float(v << 16) * scale, __uint_as_float(v & 0xffff0000u) * scale);
}

constexpr int kRowStage = kRank / 64 * kPlane;  // the latents of 64 rows

// Keys and values of a head for some tiles of 64 cached rows: [column][row] = W_h c^T, a wave 32 of the
// head's 128 columns, the weight's fragments in registers, the rows from LDS in the planes of above, the next tile's on
// their way.  The result goes through LDS, so that its rows are stored 16 bytes a lane, one after the other (8 bytes a lane
// at 32 rows take 2.5 us more).  The rotated keys are copied by one head's workgroup of each tile.  7,001 rows and 16 heads:
// 20 us for 29 MB written and 7.3 GFLOP; bound by a chain of lookups, first copies and the weight, then four tiles a workgroup one
// after the other (copies two tiles ahead change nothing).
__global__ __launch_bounds__(256, 2) void expand_kernel(const uint16_t* __restrict__ w, const uint16_t* __restrict__ pool, Batch b, Shape s,
                                                        const int32_t* __restrict__ seq_keys, const uint16_t* __restrict__ specials,
                                                        int64_t key_rows, uint16_t* __restrict__ keys, uint16_t* __restrict__ shared) {
    __shared__ __align__(16) unsigned char ring[2 * kRowStage + kKeys * 4 * kHead];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lds = lds_addr(ring);
    // workgroups go round the eight XCDs: those of one take every eighth tile, each for all heads
    const int round = blockIdx.x / 8, h = round % s.H, step = gridDim.x / s.H;
    typedef const __attribute__((address_space(4))) int32_t* const_ptr;
    const const_ptr first = (const_ptr)(uintptr_t)seq_keys;
    const int total = first[b.n_seq];
    int tile = round / s.H * 8 + blockIdx.x % 8;
    if (tile >= total) return;

    // Where a tile's rows are: looked up a tile before they are copied, so that no copy waits for it.
    struct Place {
        int seq, key0, end;
        int32_t pages[2];
    };
    int seq = 0, seq_first = 0, seq_end = 0, seq_len = 0;  // the last tile's sequence; seq_end: its tiles' end
    auto look_up = [&](int u) {
        if (u >= seq_end) {
            int hi = b.n_seq;  // the last sequence whose tiles begin at or before this one
            while (hi - seq > 1) {
                const int mid = (seq + hi) >> 1;
                if (first[mid] <= u) seq = mid;
                else hi = mid;
            }
            seq_first = first[seq];
            seq_end = first[seq + 1];
            seq_len = ((const_ptr)(uintptr_t)b.lens)[seq];
        }
        Place p = {seq, (u - seq_first) * kKeys, seq_len, {}};
        const const_ptr table = (const_ptr)(uintptr_t)(b.table + seq * b.table_ld);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int at = (p.key0 + (2 * wave + i) * kBlock) >> b.page_log;
            p.pages[i] = table[at < b.width ? at : b.width - 1];
        }
        return p;
    };
    auto copy_tile = [&](const Place& p, int stage) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int blk = 2 * wave + i, p0 = p.key0 + blk * kBlock, row = lane >> 3;
            const uint16_t* from = p.pages[i] >= 0 && p.pages[i] < b.n_pages
                                       ? pool + (((int64_t)p.pages[i] << b.page_log) + (p0 & ((1 << b.page_log) - 1))) * kWidth
                                       : specials + kBlock * kWidth;
            const uint32_t off = row * (kWidth * 2) + (((lane & 7) ^ swizzle(blk * kBlock + row)) << 4);
            const unsigned char* mine = (const unsigned char*)(p0 + row < p.end ? from : specials) + off;
            const uint32_t to_lds = lds + stage * kRowStage + blk * 1024;
#pragma unroll
            for (int pl = 0; pl < kRank / 64; ++pl) copy16(mine + pl * 128, __builtin_amdgcn_readfirstlane(to_lds + pl * kPlane));
        }
    };
    Place now = look_up(tile), next = now;
    copy_tile(now, 0);
    if (tile + step < total) next = look_up(tile + step);
    bf16x8_t a[kRank / 16];
    {
        const uint16_t* wh = w + ((int64_t)h * 2 * kHead + wave * 32 + (lane & 31)) * kRank + 8 * half;
#pragma unroll
        for (int st = 0; st < kRank / 16; ++st) a[st] = *reinterpret_cast<const bf16x8_t*>(wh + 16 * st);
#pragma unroll
        for (int st = 0; st < kRank / 16; ++st) asm volatile("" : "+v"(a[st]));
    }
    int stage = 0;
    for (bool started = false; tile < total; tile += step, stage ^= 1, started = true) {
        // (behind this tile's copies are only the last tile's stores, four or more)
        if (started) copies_barrier<4>();
        else copies_barrier<0>();
        const Place here = now;
        now = next;
        if (tile + step < total) copy_tile(now, stage ^ 1);
        if (tile + 2 * step < total) next = look_up(tile + 2 * step);
        const uint32_t at = lds + stage * kRowStage, result = lds + 2 * kRowStage;
        f32x16_t acc[2] = {f32x16_zero(), f32x16_zero()};
#pragma unroll
        for (int st = 0; st < kRank / 16; ++st)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 32 * i + (lane & 31);
                const bf16x8_t x = *(lds_frag_ptr)(size_t)(at + (st >> 2) * kPlane + r * 128 + (((2 * (st & 3) + half) ^ swizzle(r)) << 4));
                acc[i] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a[st], x, acc[i], 0, 0, 0);
            }
        reads_ahead<8, 2 * kRank / 16 - 8, 1, 8>();
        // row r's piece c of 16 bytes lies at c ^ r % 16
        const float scale = wave < 2 ? kKeyScale : kValueScale;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int e = 0; e < 16; e += 4) {
                const int r = 32 * i + (lane & 31), c = 4 * wave + (e >> 2);
                *(lds_u2_ptr)(size_t)(result + r * (4 * kHead) + ((c ^ (r & 15)) << 4) + 8 * half) =
                    u32x2_t{pack_f16x2(acc[i][e] * scale, acc[i][e + 1] * scale), pack_f16x2(acc[i][e + 2] * scale, acc[i][e + 3] * scale)};
            }
        lds_barrier();
        uint16_t* to = keys + ((int64_t)h * key_rows + (int64_t)tile * kKeys) * (2 * kHead);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = 16 * i + (tid >> 4), c = tid & 15;
            *reinterpret_cast<u32x4_t*>(to + r * (2 * kHead) + c * 8) = *(lds_u4_ptr)(size_t)(result + r * (4 * kHead) + ((c ^ (r & 15)) << 4));
        }
        if (tile % s.H == h) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = 32 * i + (tid >> 3), c = tid & 7, p = here.key0 + r;
                u32x4_t v = {0, 0, 0, 0};
                if (p < here.end) {
                    const int32_t page = batch_page(b, here.seq, p);
                    v = page < 0 ? u32x4_t{0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u, 0x7fc07fc0u}
                                 : *reinterpret_cast<const u32x4_t*>(pool + (((int64_t)page << b.page_log) + (p & ((1 << b.page_log) - 1))) * kWidth +
                                                                     kRank + c * 8);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) v[j] = f16_of_bf16x2(v[j], kKeyScale);
                *reinterpret_cast<u32x4_t*>(shared + ((int64_t)tile * kKeys + r) * kRope + c * 8) = v;
            }
        }
    }
}

// A step's LDS: two planes of 64 rows for the keys and their rotated parts, one for the values.  A step takes the next
// one's keys and its own values, so each have a ring of three steps of their own: both are copied two steps ahead.
constexpr int kKeyStage = 2 * kPlane, kValueStage = kPlane, kValues = 3 * kKeyStage;  // (the values' ring behind the keys')
// How far a row's maximum may grow before its sums are rescaled: exponentials stay below 2^14.
constexpr float kSlack = 8.0f;

constexpr int kAhead = 2;  // steps of a product that the keys' fragments are read ahead

// The maximum of a lane and the one 32 from it, without a way through LDS.
__device__ __forceinline__ float halves_max(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}

// 16 bytes a lane from base + off into LDS at ring + at + 16 times the lane.
template <int AT>
__device__ __forceinline__ void copy16_at(const void* base, uint32_t off, uint32_t ring) {
    asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(ring), "v"(off), "s"(base), "n"(AT) : "memory", "scc");
}

// A tile's steps for a share of its keys, two workgroups a CU; a wave 32 tokens of its own, S^T = K Q^T and O^T = V^T P^T in
// 32 x 32 x 16 products, as in attend_kernel.  2,048 tokens over 7,001 keys, 16 heads: 75 GFLOP in 99 to 104 us by the
// card (97 at the least), 720 to 760 TFLOP/s, where large bf16 products reach 1,127 to 1,405.  Bound by a step's matrix and vector instructions, which overlap in part: 32 exponentials,
// their sum, rounding and maximum a lane beside 24 products.
__global__ __launch_bounds__(256, 2) void chunk_attend_kernel(const uint16_t* __restrict__ q, const float2* __restrict__ turns,
                                                              const uint16_t* __restrict__ keys, const uint16_t* __restrict__ shared, Shape s,
                                                              const Plan* plan, const Item* __restrict__ items, int64_t key_rows,
                                                              float* __restrict__ sums, float2* __restrict__ stats,
                                                              uint16_t* __restrict__ out) {
    __shared__ __align__(16) unsigned char ring[3 * (kKeyStage + kValueStage)];
    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t lds = lds_addr(ring);
    // neighbours in the work on one XCD (workgroups go round the eight)
    const int group = gridDim.x % 8 == 0 ? (int)(blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8) : (int)blockIdx.x;
    const int64_t quota = plan->quota, all = plan->tiles, each = all / s.planes;
    const int n_items = plan->n_items;
    int64_t t = group * quota;
    const int64_t stop = t + quota < all ? t + quota : all;
    if (t >= stop) return;
    uint32_t k_at[4], v_at[2][2];
    {
        const int key = lane & 31, row = 4 * half + ((lane & 15) >> 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) k_at[i] = key * 128 + (((2 * i + half) ^ swizzle(key)) << 4);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const int r = row + 8 * i, c = 4 * d + ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
                v_at[i][d] = r * 128 + ((c ^ swizzle(r)) << 4) + (lane & 1) * 8;
            }
    }
    // a lane's places in the copies of the wave's two blocks of 8 rows
    uint32_t key_off[2], value_off[2], shared_off[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int row = 16 * wave + 8 * i + (lane >> 3), piece = (lane & 7) ^ swizzle(row);
        key_off[i] = row * (4 * kHead) + piece * 16;
        value_off[i] = key_off[i] + 2 * kHead;
        shared_off[i] = row * (2 * kRope) + piece * 16;
    }
    const uint32_t to_keys = lds + wave * 2048, to_values = lds + kValues + wave * 2048;

    int h = (int)(t / each);
    int item = find_item(items, n_items, t - h * each, lane);
    for (; t < stop; ++item) {
        if (item == n_items) item = 0, ++h;
        const Item it = items[item];
        const int64_t before = h * each, begin = before + (item > 0 ? items[item - 1].end : 0), finish = before + it.end;
        const int64_t to = finish < stop ? finish : stop;
        if (to <= t) continue;
        const int k_begin = (int)(t - begin), n = (int)(to - t);  // the first step's number, and the steps
        const int my = wave * 32 + (lane & 31), my_row = my < it.rows ? my : it.rows - 1;
        const int first_pos = it.pos0 + it.row0, my_pos = first_pos + my_row;
        const int64_t row = (int64_t)it.tok0 + it.row0 + my_row;
        const int64_t key_row = ((int64_t)it.keys + k_begin) * kKeys;
        const unsigned char* kv = (const unsigned char*)(keys + ((int64_t)h * key_rows + key_row) * (2 * kHead));
        const unsigned char* kr = (const unsigned char*)(shared + key_row * kRope);

        auto copy_keys = [&](int j, int stage) {
            const unsigned char *from = kv + (int64_t)j * (kKeys * 4 * kHead), *rot = kr + (int64_t)j * (kKeys * 2 * kRope);
            const uint32_t at = to_keys + stage * kKeyStage;
            copy16_at<0>(from, key_off[0], at);
            copy16_at<1024>(from, key_off[1], at);
            copy16_at<kPlane>(rot, shared_off[0], at);
            copy16_at<kPlane + 1024>(rot, shared_off[1], at);
        };
        auto copy_values = [&](int j, int stage) {
            const unsigned char* from = kv + (int64_t)j * (kKeys * 4 * kHead);
            const uint32_t at = to_values + stage * kValueStage;
            copy16_at<0>(from, value_off[0], at);
            copy16_at<1024>(from, value_off[1], at);
        };
        copy_keys(0, 0);
        copy_values(0, 0);
        if (n > 1) copy_keys(1, 1), copy_values(1, 1);
        if (n > 2) copy_keys(2, 2);
        Frag fq[8];
        {
            const uint16_t* qp = q + (row * s.H + h) * (kHead + kRope) + 8 * half;
#pragma unroll
            for (int i = 0; i < 8; ++i) fq[i].u = *reinterpret_cast<const u32x4_t*>(qp + 16 * i);
            const float4* cs = reinterpret_cast<const float4*>(turns + row * 32 + 8 * half);
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float4 c = cs[8 * i + j];  // cos, sin of two angles
                    const uint32_t u = fq[4 + i].w[j], v = fq[6 + i].w[j];
                    const float u0 = __uint_as_float(u << 16), u1 = __uint_as_float(u & 0xffff0000u);
                    const float v0 = __uint_as_float(v << 16), v1 = __uint_as_float(v & 0xffff0000u);
                    fq[4 + i].w[j] = pack_f16x2((u0 * c.x - v0 * c.y) * kQueryScale, (u1 * c.z - v1 * c.w) * kQueryScale);
                    fq[6 + i].w[j] = pack_f16x2((v0 * c.x + u0 * c.y) * kQueryScale, (v1 * c.z + u1 * c.w) * kQueryScale);
                }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) fq[i].w[j] = f16_of_bf16x2(fq[i].w[j], kQueryScale);
#pragma unroll
            for (int i = 0; i < 8; ++i) asm volatile("" : "+v"(fq[i].u));
        }
        f32x16_t o[2] = {f32x16_zero(), f32x16_zero()}, x[2], y[2];
        float shift = kLowest, l = 0.0f;
        // the keys' fragments of a step of the product, from where its stage begins
        auto key_bases = [&](uint32_t at, uint32_t (&base)[4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                base[i] = at + k_at[i];
                asm volatile("" : "+v"(base[i]));  // (one sum each; the rest is the reads' constant offsets)
            }
        };
        auto read_keys = [&](const uint32_t (&base)[4], int st, int i) {
            return *(lds_half_ptr)(size_t)(base[st & 3] + (st >> 2) * kPlane + i * 32 * 128);
        };
        // What the wave's tokens do not see of step j.
        auto mask = [&](f32x16_t (&z)[2], int j) {
            const int sees = my_pos - (k_begin + j) * kKeys - 4 * half;  // (a lane's keys are 4 half and a constant each)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) z[i][e] = 32 * i + 8 * (e >> 2) + (e & 3) > sees ? -INFINITY : z[i][e];
        };
        // Rows of step j, which not all tokens see, whose values are not finite: no result for a token that sees one of them,
        // zeros for the others.
        auto clean = [&](int j, uint32_t at) {
            bool bad = false;
#pragma unroll 1
            for (int c = 0; c < 8; ++c) {
                const u32x4_t v = *(lds_u4_ptr)(size_t)(at + lane * 128 + (((c + (lane >> 1)) & 7) << 4));
#pragma unroll
                for (int i = 0; i < 4; ++i) bad |= (v[i] & 0x7c00u) == 0x7c00u || (v[i] & 0x7c000000u) == 0x7c000000u;
            }
            const uint64_t odd = ballot(bad);
            if (odd == 0) return;
            if ((k_begin + j) * kKeys + (int)__builtin_ctzll(odd) <= my_pos) l = NAN;  // (the first of them)
            lds_barrier();
            for (int e = tid; e < kKeys * 8; e += 256)
                if (odd >> (e >> 3) & 1) *(lds_u4_ptr)(size_t)(at + e * 16) = u32x4_t{0, 0, 0, 0};
            lds_barrier();
        };
        auto new_top = [&](float top) {
            top = halves_max(top);
            if (ballot((top - shift) * s.scale2 > kSlack) != 0) {  // some token's maximum has grown
                const float was = shift;
                shift = fmaxf(shift, top);
                const float r = __builtin_amdgcn_exp2f((was - shift) * s.scale2);
                l *= r;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; ++e) o[i][e] *= r;
            }
        };
        // Step j on its scores x, whose maximum is known; with `more`, the scores y of step j + 1 beside it.  In this
        // order: two products of y beside the exponentials of four of x, eight times; then the products with the values
        // beside the maximum of y.  (The fences keep it: by itself the compiler puts the exponentials first.)
        auto run_step = [&](auto more, f32x16_t (&x)[2], f32x16_t (&y)[2], int j, int stage) {
            const int next = stage == 2 ? 0 : stage + 1;
            // behind the keys of step j + 1 and the values of step j, six copies: the keys of j + 2 and the values of j + 1
            if (j + 2 < n) copies_barrier<6>();
            else copies_barrier<0>();
            if (j + 3 < n) copy_keys(j + 3, stage);
            if (j + 2 < n) copy_values(j + 2, next == 2 ? 0 : next + 1);
            uint32_t kb[4], vb[2][2];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    vb[i][d] = lds + kValues + stage * kValueStage + v_at[i][d];
                    asm volatile("" : "+v"(vb[i][d]));
                }
            if ((k_begin + j) * kKeys + kKeys - 1 > first_pos) clean(j, lds + kValues + stage * kValueStage);
            Frag p[4], fv[4][2];
            f16x8_t fk[8][2];
            if constexpr (more) {
                key_bases(lds + next * kKeyStage, kb);
#pragma unroll
                for (int st = 0; st < kAhead; ++st)
#pragma unroll
                    for (int i = 0; i < 2; ++i) fk[st][i] = read_keys(kb, st, i);
                y[0] = f32x16_zero();
                y[1] = f32x16_zero();
            }
#pragma unroll
            for (int st = 0; st < 8; ++st) {
                if constexpr (more) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (st + kAhead < 8) fk[st + kAhead][i] = read_keys(kb, st + kAhead, i);
                        y[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fk[st][i], fq[st].x, y[i], 0, 0, 0);
                    }
                }
                if (st >= 4) {
#pragma unroll
                    for (int d = 0; d < 2; ++d)
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            fv[st - 4][d].h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_tr_ptr)(size_t)(vb[i][d] + (st - 4) * 16 * 128));
                }
                if (st == 0) __builtin_amdgcn_s_setprio(1);  // (before a wave that is at its second part: 93.6 us against 96.5)
                float e[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) e[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[st >> 2][4 * (st & 3) + i] - shift, s.scale2, kTop));
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const uint32_t w = pack_f16x2(e[2 * i], e[2 * i + 1]);
                    p[st >> 1].w[2 * (st & 1) + i] = w;
                    // the sum of what the values are weighted with, rounded as they are
                    l = __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, w), f16x2_t{1, 1}, l, false);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            if constexpr (more)
                if ((k_begin + j + 1) * kKeys + kKeys - 1 > first_pos) mask(y, j + 1);
            __builtin_amdgcn_s_setprio(0);
            float top = -INFINITY;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int d = 0; d < 2; ++d) {
                    o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fv[i][d].x, p[i].x, o[d], 0, 0, 0);
                    if constexpr (more) {
#pragma unroll
                        for (int e = 0; e < 4; ++e) top = fmaxf(top, y[i >> 1][8 * (i & 1) + 4 * d + e]);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if constexpr (more) new_top(top);
        };
        // the first scores: behind their keys are up to 12 copies
        if (n > 2) copies_barrier<12>();
        else copies_barrier<0>();
        {
            uint32_t kb[4];
            key_bases(lds, kb);
            x[0] = f32x16_zero();
            x[1] = f32x16_zero();
#pragma unroll
            for (int st = 0; st < 8; ++st)
#pragma unroll
                for (int i = 0; i < 2; ++i) x[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(read_keys(kb, st, i), fq[st].x, x[i], 0, 0, 0);
            if (k_begin * kKeys + kKeys - 1 > first_pos) mask(x, 0);
            float top = x[0][0];
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) top = fmaxf(top, x[i][e]);
            new_top(top);
        }
        int j = 0, stage = 0;
        constexpr std::integral_constant<bool, true> more{};
        constexpr std::integral_constant<bool, false> none{};
        for (; j + 2 < n; j += 2) {
            run_step(more, x, y, j, stage);
            stage = stage == 2 ? 0 : stage + 1;
            run_step(more, y, x, j + 1, stage);
            stage = stage == 2 ? 0 : stage + 1;
        }
        if (j + 1 < n) {
            run_step(more, x, y, j, stage);
            run_step(none, y, x, j + 1, stage == 2 ? 0 : stage + 1);
        } else {
            run_step(none, x, y, j, stage);
        }
        l += __shfl_xor(l, 32, 64);
        lds_barrier();
        if (my < it.rows) {
            if (t == begin && to == finish) {  // the tile's whole work
                const float inv = inverse(l * kValueScale, my_pos < 0);
                uint16_t* z = out + (row * s.H + h) * kHead + 4 * half;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<uint2*>(z + 32 * i + 2 * e) = make_uint2(pack_bf16x2(o[i][e] * inv, o[i][e + 1] * inv),
                                                                                   pack_bf16x2(o[i][e + 2] * inv, o[i][e + 3] * inv));
            } else {
                const int64_t slot = ((int64_t)group + (int64_t)h * n_items + item) * kChunkTok + my;
                float* z = sums + slot * kHead + 4 * half;
#pragma unroll
                for (int i = 0; i < 2; ++i)
#pragma unroll
                    for (int e = 0; e < 16; e += 4)
                        *reinterpret_cast<f32x4_t*>(z + 32 * i + 2 * e) = f32x4_t{o[i][e], o[i][e + 1], o[i][e + 2], o[i][e + 3]};
                if (half == 0) stats[slot] = make_float2(shift, l);
            }
        }
        t = to;
    }
}

// 16 (token, head) rows a workgroup, 16 threads each: joins the parts of those that have several (9 us for 32,768 rows: 34 MB
// of sums).
__global__ __launch_bounds__(256) void chunk_finish_kernel(int64_t n_rows, Shape s, const Plan* plan, const Item* __restrict__ items,
                                                           const int32_t* __restrict__ seq_item, const Token* __restrict__ tokens,
                                                           const float* __restrict__ sums, const float2* __restrict__ stats,
                                                           uint16_t* __restrict__ out) {
    const int64_t r = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4), t = r / s.H;
    const int h = (int)(r - t * s.H), col = (threadIdx.x & 15) * 4;
    if (t >= n_rows) return;
    const Token token = tokens[t];
    if (token.seq == kNoSeq) return;
    int in;
    const Parts p = row_parts(s, plan, items, seq_item, token, token.index, h, in);
    if (p.n == 1) return;  // written as a whole
    float top = kLowest, l = 0.0f;
    f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int k = 0; k < p.n; ++k) {
        const int64_t at = (p.slot + k) * kChunkTok + in;
        const float2 ml = stats[at];
        const f32x4_t x = *reinterpret_cast<const f32x4_t*>(sums + at * kHead + col);
        const float next = fmaxf(top, ml.x);
        const float f = __builtin_amdgcn_exp2f((top - next) * s.scale2), f2 = __builtin_amdgcn_exp2f((ml.x - next) * s.scale2);
        top = next;
        l = l * f + ml.y * f2;
        v = v * f + x * f2;
    }
    const float inv = inverse(l * kValueScale, p.blind);
    *reinterpret_cast<uint2*>(out + r * kHead + col) = make_uint2(pack_bf16x2(v[0] * inv, v[1] * inv), pack_bf16x2(v[2] * inv, v[3] * inv));
}

bool is_chunk(int64_t n_rows, int n_seq, int H, int nope, int v_dim, int64_t capacity) {
    return nope == kHead && v_dim == kHead && n_rows >= (int64_t)kChunkRows * n_seq &&
           (size_t)n_seq * (size_t)(capacity + kKeys) <= kChunkBytes / (size_t)(H * 4 * kHead);
}
int chunk_groups(int num_cus) { return 2 * num_cus; }  // two workgroups a CU

int launch_chunk(const uint16_t* q, const uint16_t* w, const uint16_t* pool, const Batch& b, const float* rates, Shape s, unsigned char* ws,
                 uint16_t* out, int num_cus, hipStream_t stream) {
    s.rows = kChunkTok;
    s.groups = chunk_groups(num_cus);
    s.planes = s.H;
    s.scale2 /= kKeyScale * kQueryScale;
    const ChunkLayout l = chunk_layout(b.n_rows, b.n_seq, s.H, (int64_t)b.width << b.page_log, s.groups);
    Plan* plan = (Plan*)(ws + l.plan);
    Item* items = (Item*)(ws + l.items);
    int32_t *seq_item = (int32_t*)(ws + l.seq_item), *seq_keys = (int32_t*)(ws + l.seq_keys);
    Token* tokens = (Token*)(ws + l.tokens);
    float2 *turns = (float2*)(ws + l.turns), *stats = (float2*)(ws + l.stats);
    uint16_t *specials = (uint16_t*)(ws + l.specials), *keys = (uint16_t*)(ws + l.keys), *shared = (uint16_t*)(ws + l.shared);
    float* sums = (float*)(ws + l.sums);
    hipLaunchKernelGGL(chunk_prepare_kernel, dim3((unsigned)((b.n_rows + 7) / 8 + 1)), dim3(256), 0, stream, rates, b, s, l.max_items, plan, items,
                       seq_item, seq_keys, tokens, specials, turns);
    const unsigned expand_groups = (unsigned)(8 * s.H * ((2 * num_cus + 8 * s.H - 1) / (8 * s.H)));  // eight tiles for all heads, times
    hipLaunchKernelGGL(expand_kernel, dim3(expand_groups), dim3(256), 0, stream, w, pool, b, s, seq_keys, specials, l.key_rows, keys, shared);
    hipLaunchKernelGGL(chunk_attend_kernel, dim3((unsigned)s.groups), dim3(256), 0, stream, q, turns, keys, shared, s, plan, items,
                       l.key_rows, sums, stats, out);
    hipLaunchKernelGGL(chunk_finish_kernel, dim3((unsigned)((b.n_rows * s.H + 15) / 16)), dim3(256), 0, stream, b.n_rows, s, plan, items,
                       seq_item, tokens, sums, stats, out);
    return (int)hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace_bytes(int64_t n_rows, int n_seq, int H, int rank, int rope, int nope, int v_dim, int width,
                                       int page_log, int dtype, int num_cus) {
    const int rows = fast_rows(n_rows, n_seq, H);
    const int64_t capacity = (int64_t)width << page_log;
    if (is_fast(rank, rope, nope, v_dim, page_log, dtype) && is_chunk(n_rows, n_seq, H, nope, v_dim, capacity))
        return chunk_layout(n_rows, n_seq, H, capacity, chunk_groups(num_cus)).bytes;
    if (is_fast(rank, rope, nope, v_dim, page_log, dtype))
        return layout(n_rows, n_seq, H, kQuery, rows, fast_groups(rows, num_cus), 2, kRank).bytes;
    return layout(n_rows, n_seq, H, rank + rope, kAnyRows, any_groups(num_cus), 4, rank).bytes;
}

int launch_paged_attention(const void* q, const void* w, const void* pool, const Batch& b, const float* rates, int H, int rank, int rope,
                           int nope, int v_dim, int dtype, float scale, void* ws, void* out, int num_cus, hipStream_t stream) {
    const Shape s = {H, rank, rope, nope, v_dim, 0, 0, 1, scale * kLog2E};
    if (is_fast(rank, rope, nope, v_dim, b.page_log, dtype) &&
        is_chunk(b.n_rows, b.n_seq, H, nope, v_dim, (int64_t)b.width << b.page_log))
        return launch_chunk((const uint16_t*)q, (const uint16_t*)w, (const uint16_t*)pool, b, rates, s, (unsigned char*)ws, (uint16_t*)out,
                            num_cus, stream);
    if (is_fast(rank, rope, nope, v_dim, b.page_log, dtype))
        return launch_fast((const uint16_t*)q, (const uint16_t*)w, (const uint16_t*)pool, b, rates, s, (unsigned char*)ws, (uint16_t*)out,
                           num_cus, stream);
    if (dtype == kBF16)
        return launch_any((const uint16_t*)q, (const uint16_t*)w, (const uint16_t*)pool, b, rates, s, (unsigned char*)ws, (uint16_t*)out,
                          num_cus, stream);
    return launch_any((const float*)q, (const float*)w, (const float*)pool, b, rates, s, (unsigned char*)ws, (float*)out, num_cus, stream);
}

}  // namespace ethos

// Attention of new tokens over a cache of latents in pages: softmax(scale q k) v over the keys up to each
// token, with k of head h = [W_k,h c | key] and v = W_v,h c of a cached row [c | key] (model.py:104-160
// forms every head's keys and values; here they stay what they are made of).
//
// The weight goes to the queries instead: q . W_k,h c = (W_k,h^T q) . c, and W_v,h goes behind the sum over
// the keys, which all heads then take over the same rows: one read of the cache serves every head.  A
// sequence's rows are its (token, head) pairs, token by token, so that a tile of rows sees nearly the same keys.
//
// Three launches.  paged_prepare: queries [W_k,h^T q | rotated rest] per row, and the plan: tiles of rows,
// each with its tiles of kKeys keys, as one line of work that is cut into even shares, whatever the lengths
// of the sequences are.  The second goes over the keys with a running maximum and sum; where a share ends
// inside a tile of rows, each side leaves its sums.  The third joins them and multiplies with W_v,h.
//
// Without bounds of the host on lengths, tables or starts: what they hold is checked where it is used.  A page
// outside the cache reads as a row of NaN, a length beyond the table makes its sequence's outputs NaN.
#include "ethos_launch.hpp"
#include "ethos_mfma.hpp"
#include "ethos_rows.hpp"
#include "ethos_serve.hpp"

namespace ethos {
namespace {

constexpr int kKeys = 64;          // keys of a tile of work
constexpr float kLog2E = 1.44269504f;
constexpr float kLowest = -0x1p126f;  // a running maximum's start: finite, so that masked scores weigh nothing

// A tile of rows: `rows` of sequence seq from its row `row0` (token row0 / H, head row0 % H) on; the first new
// token of the sequence is row tok0 of the batch, at position pos0.
struct Item {
    int32_t seq, row0, rows, tok0, pos0, pad;
    int64_t end;  // tiles of work up to this one's last, all before it included
};

struct Plan {
    int64_t tiles, quota;  // in all; of a workgroup
    int32_t n_items, pad[3];
};

// Where the workspace's parts are.
struct Layout {
    size_t plan, items, seq_item, tok_seq, specials, queries, sums, stats, bytes;
    int64_t max_items;
};

struct Shape {
    int H, rank, rope, nope, v_dim;
    int rows;    // of a tile
    int groups;  // workgroups that share the work
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
    l.tok_seq = take((size_t)n_rows * 4);
    l.specials = take((size_t)2 * width * 4);
    l.queries = take((size_t)n_rows * H * width * query_bytes);
    const size_t slots = (size_t)(l.max_items + groups);
    l.sums = take(slots * tile_rows * rank * 4);
    l.stats = take(slots * tile_rows * 8);
    l.bytes = at;
    return l;
}

// ------------------------------------------------------------------------- the plan
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t* lds, int tid, int64_t& total) {  // inclusive, 1,024 threads
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
    for (int w = 0; w < 16; ++w) {
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
    return b.lens[i] >= 0 && (int64_t)b.lens[i] <= (int64_t)b.width << b.page_log;
}

// One workgroup of 1,024 threads.
__device__ void make_plan(const Batch& b, const Shape& s, int64_t max_items, Plan* plan, Item* items, int32_t* seq_item, int tid) {
    __shared__ int64_t lds[16];
    int64_t base = 0, total;
    for (int at = 0; at < b.n_seq; at += 1024) {
        const int i = at + tid;
        const int64_t n = i < b.n_seq ? (new_tokens(b, i) * s.H + s.rows - 1) / s.rows : 0;
        const int64_t end = base + block_scan(n, lds, tid, total);
        // (starts that overlap could ask for more than there is room for: those sequences get none)
        const int64_t first = end - n;
        if (i < b.n_seq) seq_item[i] = end <= max_items ? (int32_t)first : -1;
        for (int64_t k = first; k < end && end <= max_items; ++k) {
            Item it;
            it.seq = i;
            it.row0 = (int32_t)((k - first) * s.rows);
            const int64_t left = new_tokens(b, i) * s.H - it.row0;
            it.rows = (int32_t)(left < s.rows ? left : s.rows);
            it.tok0 = b.starts[i];
            it.pos0 = (int32_t)(b.lens[i] - new_tokens(b, i));
            it.pad = 0;
            it.end = 0;
            items[k] = it;
        }
        base += total;
    }
    const int64_t n_items = base < max_items ? base : max_items;
    __syncthreads();
    int64_t tiles = 0;
    for (int64_t at = 0; at < n_items; at += 1024) {
        const int64_t k = at + tid;
        int64_t n = 0;
        if (k < n_items) {
            const Item it = items[k];
            // keys up to the last row's own
            const int64_t keys = (int64_t)it.pos0 + (it.row0 + it.rows - 1) / s.H + 1;
            n = fits(b, it.seq) && keys > 0 ? (keys + kKeys - 1) / kKeys : 0;
        }
        const int64_t end = tiles + block_scan(n, lds, tid, total);
        if (k < n_items) items[k].end = end;
        tiles += total;
    }
    if (tid == 0) {
        plan->tiles = tiles;
        plan->quota = tiles > s.groups ? (tiles + s.groups - 1) / s.groups : 1;
        plan->n_items = (int32_t)n_items;
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
constexpr int kAnyRows = 8, kAnyKeys = 16, kAnyRank = 512, kAnyRope = 128, kAnyWidth = kAnyRank + kAnyRope;

// Block 0 the plan; each other block a token's rows.
template <typename T>
__global__ __launch_bounds__(1024) void any_prepare_kernel(const T* __restrict__ q, const T* __restrict__ w, const float* __restrict__ rates,
                                                           Batch b, Shape s, int64_t max_items, Plan* plan, Item* items, int32_t* seq_item,
                                                           int32_t* tok_seq, float* __restrict__ queries) {
    if (blockIdx.x == 0) {
        make_plan(b, s, max_items, plan, items, seq_item, threadIdx.x);
        return;
    }
    const int64_t t = blockIdx.x - 1;
    const int i = batch_seq(b, t), width = s.rank + s.rope, qw = s.nope + s.rope;
    if (threadIdx.x == 0) tok_seq[t] = i;
    if (i < 0) return;
    const int64_t pos = (int64_t)b.lens[i] - b.starts[i + 1] + t;
    const T* qt = q + t * s.H * qw;
    float* out = queries + t * s.H * width;
    for (int e = threadIdx.x; e < s.H * width; e += 1024) {
        const int h = e / width, c = e - h * width;
        const T* qh = qt + h * qw;
        float v = 0.0f;
        if (c < s.rank) {
            const T* wh = w + (int64_t)h * (s.nope + s.v_dim) * s.rank + c;
            for (int j = 0; j < s.nope; ++j) v = __builtin_fmaf(Elem<T>::to_f32(qh[j]), Elem<T>::to_f32(wh[(int64_t)j * s.rank]), v);
        } else {
            const int half = s.rope / 2, p = (c - s.rank) % half;
            float cs, sn;
            rotary_angle(pos, rates[p], cs, sn);
            const float u = Elem<T>::to_f32(qh[s.nope + p]), x = Elem<T>::to_f32(qh[s.nope + half + p]);
            v = c - s.rank < half ? u * cs - x * sn : x * cs + u * sn;
        }
        out[e] = v;
    }
}

// Tiles of 8 rows, 16 keys at a time in LDS; 32 threads score a row's 16 keys, two a key; then a thread sums two
// columns of the latent for all rows.  Keys that a row does not see are left out of its sums, whatever they hold.
template <typename T>
__global__ __launch_bounds__(256) void any_attend_kernel(const T* __restrict__ pool, Batch b, Shape s, const Plan* plan,
                                                         const Item* __restrict__ items, const float* __restrict__ queries,
                                                         float* __restrict__ sums, float2* __restrict__ stats) {
    __shared__ __align__(16) float qs[kAnyRows][kAnyWidth];
    __shared__ __align__(16) float ks[kAnyKeys][kAnyWidth + 4];
    __shared__ float ps[kAnyRows][kAnyKeys], turn[kAnyRows];
    const int tid = threadIdx.x, width = s.rank + s.rope;
    const int row = tid >> 5, key = (tid >> 1) & 15, part = tid & 1;
    const int64_t quota = plan->quota, last = plan->tiles;
    int64_t t = blockIdx.x * quota;
    const int64_t stop = t + quota < last ? t + quota : last;
    if (t >= stop) return;
    int item = find_item(items, plan->n_items, t, tid & 63);
    for (; t < stop; ++item) {
        const Item it = items[item];
        const int64_t begin = item > 0 ? items[item - 1].end : 0;
        const int64_t to = it.end < stop ? it.end : stop;
        if (to <= t) continue;
        for (int e = tid; e < kAnyRows * width; e += 256) {
            const int r = e / width, c = e - r * width;
            qs[r][c] = r < it.rows ? queries[((int64_t)it.tok0 * s.H + it.row0 + r) * width + c] : 0.0f;
        }
        const int64_t my_pos = (int64_t)it.pos0 + (it.row0 + (row < it.rows ? row : it.rows - 1)) / s.H;
        const int64_t end = (int64_t)it.pos0 + (it.row0 + it.rows - 1) / s.H + 1;  // keys that some row sees
        float acc[kAnyRows][2] = {}, m = kLowest, l = 0.0f;
        for (int64_t k0 = (t - begin) * kKeys; k0 < (to - begin) * kKeys; k0 += kAnyKeys) {
            if (k0 >= end) break;
            __syncthreads();
            for (int e = tid; e < kAnyKeys * width; e += 256) {
                const int r = e / width, c = e - r * width;
                float v = 0.0f;
                if (k0 + r < end) {
                    const int32_t page = batch_page(b, it.seq, k0 + r);
                    const int64_t in = (k0 + r) & (((int64_t)1 << b.page_log) - 1);
                    v = page < 0 ? NAN : Elem<T>::to_f32(pool[(((int64_t)page << b.page_log) + in) * width + c]);
                }
                ks[r][c] = v;
            }
            __syncthreads();
            float x = 0.0f;
            for (int c = part * 4; c < width; c += 8) {
                const float4 u = *reinterpret_cast<const float4*>(&qs[row][c]), v = *reinterpret_cast<const float4*>(&ks[key][c]);
                x = __builtin_fmaf(u.x, v.x, x);
                x = __builtin_fmaf(u.y, v.y, x);
                x = __builtin_fmaf(u.z, v.z, x);
                x = __builtin_fmaf(u.w, v.w, x);
            }
            x += __shfl_xor(x, 1, 64);
            x = k0 + key > my_pos ? -INFINITY : x * s.scale2;
            float top = x;
            for (int d = 2; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor(top, d, 64));
            const float next = fmaxf(m, top), r = exp2f(m - next), p = exp2f(x - next);
            float sum = p;
            for (int d = 2; d < 32; d <<= 1) sum += __shfl_xor(sum, d, 64);
            l = l * r + sum;
            m = next;
            if (part == 0) ps[row][key] = p;
            if (key == 0 && part == 0) turn[row] = r;
            __syncthreads();
#pragma unroll
            for (int r8 = 0; r8 < kAnyRows; ++r8) {
                const int64_t seen = (int64_t)it.pos0 + (it.row0 + (r8 < it.rows ? r8 : it.rows - 1)) / s.H - k0;
                const float f = turn[r8];
#pragma unroll
                for (int d = 0; d < 2; ++d) acc[r8][d] *= f;
                for (int k = 0; k < kAnyKeys && k <= seen; ++k) {
                    const float pk = ps[r8][k];
#pragma unroll
                    for (int d = 0; d < 2; ++d)
                        if (tid + 256 * d < s.rank) acc[r8][d] = __builtin_fmaf(pk, ks[k][tid + 256 * d], acc[r8][d]);
                }
            }
        }
        const int64_t slot = (int64_t)blockIdx.x + item;
        for (int r = 0; r < it.rows; ++r)
            for (int d = 0; d < 2; ++d)
                if (tid + 256 * d < s.rank) sums[(slot * kAnyRows + r) * s.rank + tid + 256 * d] = acc[r][d];
        if (key == 0 && part == 0 && row < it.rows) stats[slot * kAnyRows + row] = make_float2(m, l);
        t = to;
        __syncthreads();
    }
}

// The parts of a row's sums: workgroups first .. first + n - 1 left them, in slots one apart.
struct Parts {
    int64_t slot;
    int n;
    bool bad;  // the sequence's length does not fit its table, or there was no room for it
};
__device__ __forceinline__ Parts row_parts(const Batch& b, const Shape& s, const Plan* plan, const Item* items, const int32_t* seq_item, int i,
                                           int64_t row, int& in) {
    Parts p = {0, 0, true};
    const int32_t first = seq_item[i];
    if (first < 0 || new_tokens(b, i) == 0 || !fits(b, i)) return p;
    p.bad = false;
    const int64_t item = first + row / s.rows;
    in = (int)(row % s.rows);
    const int64_t begin = item > 0 ? items[item - 1].end : 0, end = items[item].end;
    if (end > begin) {
        const int64_t a = begin / plan->quota, z = (end - 1) / plan->quota;
        p.slot = a + item;
        p.n = (int)(z - a + 1);
    }
    return p;
}

// One workgroup a token: joins each row's parts, in order, and multiplies with W_v,h.
template <typename T>
__global__ __launch_bounds__(256) void any_finish_kernel(const T* __restrict__ w, Batch b, Shape s, const Plan* plan,
                                                         const Item* __restrict__ items, const int32_t* __restrict__ seq_item,
                                                         const int32_t* __restrict__ tok_seq, const float* __restrict__ sums,
                                                         const float2* __restrict__ stats, T* __restrict__ out) {
    __shared__ float o[kAnyRank];
    const int64_t t = blockIdx.x;
    const int i = tok_seq[t], tid = threadIdx.x;
    if (i < 0) return;  // behind the last sequence
    for (int h = 0; h < s.H; ++h) {
        int in = 0;
        const Parts p = row_parts(b, s, plan, items, seq_item, i, (t - b.starts[i]) * s.H + h, in);
        float top = kLowest, l = 0.0f;
        for (int k = 0; k < p.n; ++k) top = fmaxf(top, stats[(p.slot + k) * s.rows + in].x);
        for (int k = 0; k < p.n; ++k) {
            const float2 ml = stats[(p.slot + k) * s.rows + in];
            l += ml.y * exp2f(ml.x - top);
        }
        const float inv = p.bad ? NAN : l == 0.0f ? 0.0f : 1.0f / l;
        __syncthreads();
        for (int c = tid; c < s.rank; c += 256) {
            float v = 0.0f;
            for (int k = 0; k < p.n; ++k)
                v += sums[((p.slot + k) * s.rows + in) * s.rank + c] * exp2f(stats[(p.slot + k) * s.rows + in].x - top);
            o[c] = v * inv;
        }
        __syncthreads();
        for (int j = tid >> 2; j < s.v_dim; j += 64) {
            const T* wr = w + ((int64_t)h * (s.nope + s.v_dim) + s.nope + j) * s.rank;
            float v = 0.0f;
            for (int c = tid & 3; c < s.rank; c += 4) v = __builtin_fmaf(o[c], Elem<T>::to_f32(wr[c]), v);
            v += __shfl_xor(v, 1, 64);
            v += __shfl_xor(v, 2, 64);
            if ((tid & 3) == 0) out[(t * s.H + h) * s.v_dim + j] = Elem<T>::from_f32(v);
        }
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
    int32_t *seq_item = (int32_t*)(ws + l.seq_item), *tok_seq = (int32_t*)(ws + l.tok_seq);
    float *queries = (float*)(ws + l.queries), *sums = (float*)(ws + l.sums);
    float2* stats = (float2*)(ws + l.stats);
    hipLaunchKernelGGL((any_prepare_kernel<T>), dim3((unsigned)(b.n_rows + 1)), dim3(1024), 0, stream, q, w, rates, b, s, l.max_items, plan,
                       items, seq_item, tok_seq, queries);
    hipLaunchKernelGGL((any_attend_kernel<T>), dim3((unsigned)s.groups), dim3(256), 0, stream, pool, b, s, plan, items, queries, sums, stats);
    hipLaunchKernelGGL((any_finish_kernel<T>), dim3((unsigned)b.n_rows), dim3(256), 0, stream, w, b, s, plan, items, seq_item, tok_seq, sums,
                       stats, out);
    return (int)hipGetLastError();
}

}  // namespace

size_t paged_attention_workspace_bytes(int64_t n_rows, int n_seq, int H, int rank, int rope, int nope, int v_dim, int dtype,
                                       int num_cus) {
    return layout(n_rows, n_seq, H, rank + rope, kAnyRows, any_groups(num_cus), 4, rank).bytes;
}

int launch_paged_attention(const void* q, const void* w, const void* pool, const Batch& b, const float* rates, int H, int rank, int rope,
                           int nope, int v_dim, int dtype, float scale, void* ws, void* out, int num_cus, hipStream_t stream) {
    const Shape s = {H, rank, rope, nope, v_dim, 0, 0, scale * kLog2E};
    if (dtype == kBF16)
        return launch_any((const uint16_t*)q, (const uint16_t*)w, (const uint16_t*)pool, b, rates, s, (unsigned char*)ws, (uint16_t*)out,
                          num_cus, stream);
    return launch_any((const float*)q, (const float*)w, (const float*)pool, b, rates, s, (unsigned char*)ws, (float*)out, num_cus, stream);
}

}  // namespace ethos

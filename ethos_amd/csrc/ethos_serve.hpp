// Operators of serving from a cache: the cache's rows and pages (cache.hip), attention over it
// (paged.hip) and the verification of drafted tokens (verify.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "ethos_common.hpp"

namespace ethos {

// A batch of new tokens over a cache of pages.  Rows starts[i] .. starts[i + 1] - 1 are the new
// tokens of sequence i, the last ones of its lens[i]; position p of sequence i is row p % page of
// page table[i][p / page].  All of it is device data that no host check has seen: the kernels
// take every row, position and page through the functions below, which keep them in bounds.
struct Batch {
    const int32_t* table;
    int64_t table_ld;
    int32_t width;  // pages a row of the table holds
    const int32_t* lens;
    const int32_t* starts;
    int32_t n_seq;
    int64_t n_rows;
    int64_t n_pages;
    int32_t page_log;
};

// The sequence that row r belongs to, -1 without one.
__device__ __forceinline__ int batch_seq(const Batch& b, int64_t r) {
    int lo = 0, hi = b.n_seq;  // the last i with starts[i] <= r
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (b.starts[mid] <= r) lo = mid;
        else hi = mid;
    }
    return b.starts[lo] <= r && r < b.starts[lo + 1] ? lo : -1;
}

// The same by all lanes of a wave for one row of theirs: two rounds of loads for 4,096 sequences.
__device__ __forceinline__ int batch_seq_wave(const Batch& b, int64_t r, int lane) {
    int lo = 0, n = b.n_seq;  // the answer is in [lo, lo + n)
    while (n > 1) {
        const int step = (n + 63) / 64, at = lane * step;
        const int k = __builtin_popcountll(__builtin_amdgcn_ballot_w64(at < n && b.starts[lo + (at < n ? at : 0)] <= r));
        const int skip = k > 0 ? (k - 1) * step : 0;
        lo += skip;
        n = n - skip < step ? n - skip : step;
    }
    return b.starts[lo] <= r && r < b.starts[lo + 1] ? lo : -1;
}

// The page of position p of sequence i, -1 where there is none.
__device__ __forceinline__ int32_t batch_page(const Batch& b, int i, int64_t p) {
    const int64_t at = p >> b.page_log;
    if (p < 0 || at >= b.width) return -1;
    const int32_t page = b.table[i * b.table_ld + at];
    return page >= 0 && page < b.n_pages ? page : -1;
}

// cos and sin of position p times a rate: the angle in float64 and less its whole turns, so that far positions
// lose nothing (in float32 an angle of 65,536 would be off by 2^-8).
__device__ __forceinline__ void rotary_angle(int64_t p, float rate, float& c, float& s) {
    const double t = (double)p * (double)rate;
    const double turns = rint(t * 0.15915494309189535);
    const float a = (float)__builtin_fma(turns, -6.283185307179586, t);
    c = cosf(a);
    s = sinf(a);
}

int launch_latent_append(const void* rows, int64_t ld, const void* gain, const float* rates, const Batch& b, int rank, int rope, float eps,
                         int dtype, void* pool, hipStream_t stream);
int launch_copy_pages(void* pool, int64_t n_blocks, int64_t block_bytes, int64_t page_bytes, const int32_t* src, const int32_t* dst,
                      int n_pairs, int num_cus, hipStream_t stream);

size_t paged_attention_workspace_bytes(int64_t n_rows, int n_seq, int H, int rank, int rope, int nope, int v_dim, int width,
                                       int page_log, int dtype, int num_cus);
int launch_paged_attention(const void* q, const void* w, const void* pool, const Batch& b, const float* rates, int H, int rank, int rope,
                           int nope, int v_dim, int dtype, float scale, void* ws, void* out, int num_cus, hipStream_t stream);

size_t verify_workspace_bytes(int64_t n_seq, int n_drafts, int64_t vocab, int num_cus);
int launch_verify(const void* logits, const int64_t* drafts, const void* probs, int probs_dtype, const int32_t* counts,
                  const float* u_accept, const float* u_sample, int64_t n_seq, int n_drafts, int64_t vocab, double temperature, int dtype,
                  void* ws, int32_t* accepted, int64_t* tokens, int num_cus, hipStream_t stream);

}  // namespace ethos

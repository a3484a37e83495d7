// What the kernels of links.cu and links_bias.cu share: the mask of a vertex's successors and the learned
// relative position bias.
#pragma once

#include "dat_common.cuh"

namespace dat {

struct LinksMask {
    const int64_t *bound_end;      // [B, L]: successors j <= bound_end[b,i] (decoding), or null
    const unsigned char *nonpad;   // [B, L]: successor j allowed iff nonpad[b,j] != 0 (training), or null
};

// Learned relative position bias: content[b,i,j,h] + table[bucket[j-i-1], h] takes the place of the score.
// A bucket outside the table forbids the transition (score -inf, whatever the content is) and sets a bit of the status word.
struct LinksBias {
    const float *table;      // [n, H]
    const int64_t *bucket;   // [K]: bucket[d] belongs to the distance d + 1
    int n;
    int32_t *status;         // may be null
};

// first / last successor of vertex i inside the band and the graph: j in [i+1, jhi]
__device__ __forceinline__ int links_jhi(int i, int L, int K, const LinksMask &mk, int64_t row) {
    int jhi = i + K < L - 1 ? i + K : L - 1;
    if (mk.bound_end) {
        const int64_t be = mk.bound_end[row];
        jhi = be < jhi ? (be < 0 ? -1 : (int)be) : jhi;
    }
    return jhi;
}

__device__ __forceinline__ bool links_bucket_ok(const LinksBias &lb, int d) {
    const int64_t k = __ldg(lb.bucket + d);
    return k >= 0 && k < lb.n;
}
__device__ __forceinline__ float links_bias1(const LinksBias &lb, int d, int h, int H, bool &bad) {
    const int64_t k = __ldg(lb.bucket + d);
    if (k >= 0 && k < lb.n) return __ldg(lb.table + k * H + h);
    bad = true;
    return -INFINITY;
}

template <bool kBias>
int links_fwd_rows(const float *content, const float *log_gates, const LinksMask &mk, const LinksBias &lb, float *links,
                   float *head_lse, int bsz, int prelen, int heads, int translen, cudaStream_t st, const DeviceInfo &di,
                   const char *who);
template <bool kBias>
int links_bwd_rows(const float *grad_links, const float *content, const float *log_gates, const float *links,
                   const float *head_lse, const LinksMask &mk, const LinksBias &lb, float *grad_content,
                   float *grad_log_gates, int bsz, int prelen, int heads, int translen, cudaStream_t st,
                   const DeviceInfo &di, const char *who);

}  // namespace dat

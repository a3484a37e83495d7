// Band links from per-head scores with a learned relative position bias, forward and backward, for sm_100a.
//
// The scores of links.cu with table[bucket[j-i-1], h] added to content[b,i,j,h]: the bias belongs to the
// distance between two vertices, distances share a row of the table by buckets, and the table is learned.
// With z = content + bias and the other names of links.cu, the gradient of a score is
//     dc[b,i,j,h] = G p - exp(z - lse_h) S_h
// as there, and the table's is the sum of dc over all transitions of a bucket:
//     dT[k,h] = sum over (b,i,d) with bucket[d] = k of dc[b,i,i+1+d,h].
// The sum runs over the distances first (one column of partial sums per distance and head, rows in a fixed
// order, no atomics, so that results repeat bit for bit) and over the distances of a bucket at the end.
#include "links_common.cuh"

namespace dat {

constexpr int kLbThreads = 128;
constexpr int kLbSplits = 64;   // partial sums per distance and head

// part[split][d * H + h] = sum of dc[b,i,i+1+d,h] over the split's vertices (b,i)
__global__ void __launch_bounds__(kLbThreads)
links_bias_diag_kernel(const float *__restrict__ grad_content, double *__restrict__ part, int B, int L, int H, int K) {
    const int x = blockIdx.x * kLbThreads + threadIdx.x;
    if (x >= K * H) return;
    const int d = x / H;
    const int64_t rows = (int64_t)B * L;
    double acc = 0.0;
    for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
        const int i = (int)(row % L);
        if (i + 1 + d < L) acc += (double)grad_content[(row * L + i + 1) * H + x];
    }
    part[(size_t)blockIdx.y * K * H + x] = acc;
}

// grad_table[k, h] from the partial sums: one CTA per bucket, the distances dealt to P = 128 / H lanes of a head
__global__ void __launch_bounds__(kLbThreads)
links_bias_join_kernel(const double *__restrict__ part, const int64_t *__restrict__ bucket, float *__restrict__ grad_table,
                       int H, int K, int splits) {
    __shared__ double lane_s[kLbThreads];
    const int k = blockIdx.x, P = kLbThreads / H, h = threadIdx.x % H, p = threadIdx.x / H;
    double acc = 0.0;
    if (p < P)
        for (int d = p; d < K; d += P)
            if (__ldg(bucket + d) == k)
                for (int s = 0; s < splits; s++) acc += part[((size_t)s * K + d) * H + h];
    lane_s[threadIdx.x] = acc;
    __syncthreads();
    if (p == 0) {
        for (int q = 1; q < P; q++) acc += lane_s[q * H + h];
        grad_table[(size_t)k * H + h] = (float)acc;
    }
}

static int links_bias_check(const char *who, const float *table, const int64_t *bucket, int buckets, int bsz, int prelen,
                            int heads, int translen) {
    DAT_REQUIRE(bsz >= 0 && prelen >= 1 && heads >= 1 && translen >= 1 && buckets >= 1, DAT_ERR_BAD_ARG,
                "%s: bad sizes bsz=%d prelen=%d heads=%d translen=%d num_buckets=%d", who, bsz, prelen, heads, translen,
                buckets);
    DAT_REQUIRE(table && bucket, DAT_ERR_BAD_ARG, "%s: null pointer", who);
    return DAT_OK;
}

}  // namespace dat

extern "C" {

size_t dat_links_bias_workspace_bytes(int bsz, int prelen, int heads, int translen) {
    (void)bsz;
    (void)prelen;
    return (size_t)dat::kLbSplits * translen * heads * sizeof(double);
}

int dat_links_from_heads_biased(const float *content, const float *log_gates, const float *bias_table,
                                const int64_t *buckets, int num_buckets, const int64_t *bound_end,
                                const unsigned char *nonpad, float *links, float *head_lse, int32_t *status, int bsz,
                                int prelen, int heads, int translen, void *stream) {
    using namespace dat;
    const char *who = "dat_links_from_heads_biased";
    if (int rc = links_bias_check(who, bias_table, buckets, num_buckets, bsz, prelen, heads, translen)) return rc;
    if (bsz == 0) return DAT_OK;
    DAT_REQUIRE(content && log_gates && links, DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    return links_fwd_rows<true>(content, log_gates, LinksMask{bound_end, nonpad},
                                LinksBias{bias_table, buckets, num_buckets, status}, links, head_lse, bsz, prelen, heads,
                                translen, static_cast<cudaStream_t>(stream), di, who);
}

int dat_links_from_heads_biased_backward(const float *grad_links, const float *content, const float *log_gates,
                                         const float *bias_table, const int64_t *buckets, int num_buckets,
                                         const float *links, const float *head_lse, const int64_t *bound_end,
                                         const unsigned char *nonpad, float *grad_content, float *grad_log_gates,
                                         float *grad_bias_table, void *workspace, int bsz, int prelen, int heads,
                                         int translen, void *stream) {
    using namespace dat;
    const char *who = "dat_links_from_heads_biased_backward";
    if (int rc = links_bias_check(who, bias_table, buckets, num_buckets, bsz, prelen, heads, translen)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bsz == 0) {
        if (grad_bias_table) cudaMemsetAsync(grad_bias_table, 0, (size_t)num_buckets * heads * sizeof(float), st);
        return check_launch(who);
    }
    DAT_REQUIRE(grad_links && content && log_gates && links && head_lse && grad_content && grad_log_gates &&
                    (workspace || !grad_bias_table),
                DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    if (int rc = links_bwd_rows<true>(grad_links, content, log_gates, links, head_lse, LinksMask{bound_end, nonpad},
                                      LinksBias{bias_table, buckets, num_buckets, nullptr}, grad_content, grad_log_gates,
                                      bsz, prelen, heads, translen, st, di, who))
        return rc;
    if (!grad_bias_table) return DAT_OK;
    double *part = static_cast<double *>(workspace);
    const dim3 grid((unsigned)((translen * heads + kLbThreads - 1) / kLbThreads), kLbSplits);
    links_bias_diag_kernel<<<grid, kLbThreads, 0, st>>>(grad_content, part, bsz, prelen, heads, translen);
    if (int rc = check_launch(who)) return rc;
    links_bias_join_kernel<<<(unsigned)num_buckets, kLbThreads, 0, st>>>(part, buckets, grad_bias_table, heads, translen,
                                                                         kLbSplits);
    return check_launch(who);
}

}  // extern "C"

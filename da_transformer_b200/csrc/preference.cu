// Loss of paired log ratios (preference loss) of sentence log-likelihoods, for sm_100a.
//
// A pair holds the log-likelihoods that dag_loss gives a preferred and a rejected sentence, under the model
// that learns and, optionally, under a reference model.  With the rewards
//     r = beta * (log p - log p_ref) / length      (length = 1 unless lengths are given)
// and the margin h = r_chosen - r_rejected, smoothing e:
//     sigmoid  l = -(1-e) log sigma(h) - e log sigma(-h)      dl/dh = sigma(h) - (1-e)
//     hinge    l = (1-e) max(0, 1-h) + e max(0, 1+h)          dl/dh = e [h > -1] - (1-e) [h < 1]
//     squared  l = (1-e) (h - 1/2)^2 + e (h + 1/2)^2          dl/dh = 2 (h - 1/2) + 2e
// The loss is the mean over all pairs; a pair with a log-likelihood that is not finite (a sentence without a
// path through its graph) or a length below one adds nothing and gets no gradient, as dag_loss_mean treats it.
//
// A few KB in and out: bound by the latency of one launch and of the 64-bit exponential and logarithm, which
// the differences of values near -700 are taken in (as 32-bit numbers they keep 6e-5).  One thread-block
// cluster of eight CTAs spreads the pairs over eight SMs and joins the sums through distributed shared
// memory in the order of the ranks: no workspace, no atomics.
#include <cooperative_groups.h>

#include "dat_common.cuh"

namespace dat {

constexpr int kPrThreads = 512;
constexpr int kPrCtas = 8;
constexpr int kPrSums = 5;   // losses, chosen rewards, rejected rewards, correct pairs, invalid pairs

struct PreferenceArgs {
    const float *chosen, *rejected, *ref_chosen, *ref_rejected;   // [n]; the references may be null (both)
    const int64_t *chosen_length, *rejected_length;               // [n] or null (both)
    double beta, smoothing;
    int kind;
    float *loss;      // [1]
    float *rewards;   // [2, n]
    double *stats;    // [6]
    float *grad;      // [2, n] d loss / d (chosen, rejected), or null
    int32_t *status;
    int n;
};

__device__ __forceinline__ void preference_pair(const PreferenceArgs &a, double h, double &loss, double &slope) {
    const double e = a.smoothing;
    if (a.kind == DAT_PREFERENCE_SIGMOID) {
        const double small = exp(-fabs(h));        // in (0, 1]: no overflow for any margin
        const double soft = log1p(small);
        loss = (1.0 - e) * (soft + fmax(-h, 0.0)) + e * (soft + fmax(h, 0.0));
        // e sigma(h) - (1-e) sigma(-h): no difference of numbers near 1 for a pair that is far apart
        slope = (e * (h >= 0.0 ? 1.0 : small) - (1.0 - e) * (h >= 0.0 ? small : 1.0)) / (1.0 + small);
    } else if (a.kind == DAT_PREFERENCE_HINGE) {
        loss = (1.0 - e) * fmax(1.0 - h, 0.0) + e * fmax(1.0 + h, 0.0);
        slope = (h > -1.0 ? e : 0.0) - (h < 1.0 ? 1.0 - e : 0.0);
    } else {
        loss = (1.0 - e) * (h - 0.5) * (h - 0.5) + e * (h + 0.5) * (h + 0.5);
        slope = 2.0 * (h - 0.5) + 2.0 * e;
    }
}

__global__ void __cluster_dims__(kPrCtas, 1, 1) __launch_bounds__(kPrThreads)
preference_kernel(PreferenceArgs a) {
    namespace cg = cooperative_groups;
    cg::cluster_group cluster = cg::this_cluster();
    __shared__ double part[kPrSums][kPrThreads / 32];
    __shared__ double mine[kPrSums];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, rank = (int)cluster.block_rank();
    double s[kPrSums] = {};
    bool bad_length = false;
    for (int64_t p = rank * kPrThreads + tid; p < a.n; p += kPrCtas * kPrThreads) {
        double c = a.chosen[p], r = a.rejected[p], kc = a.beta, kr = a.beta;
        if (a.ref_chosen) {
            c -= a.ref_chosen[p];
            r -= a.ref_rejected[p];
        }
        bool good = isfinite(c) && isfinite(r);
        if (a.chosen_length) {
            const int64_t lc = a.chosen_length[p], lr = a.rejected_length[p];
            const bool ok = lc >= 1 && lr >= 1;
            bad_length |= !ok;
            good &= ok;
            kc /= (double)(ok ? lc : 1);
            kr /= (double)(ok ? lr : 1);
        }
        double loss = 0.0, slope = 0.0;
        c = good ? c * kc : 0.0;
        r = good ? r * kr : 0.0;
        const double h = c - r;
        if (good) preference_pair(a, h, loss, slope);
        a.rewards[p] = (float)c;
        a.rewards[(int64_t)a.n + p] = (float)r;
        if (a.grad) {
            a.grad[p] = (float)(slope * kc / a.n);
            a.grad[(int64_t)a.n + p] = (float)(-slope * kr / a.n);
        }
        s[0] += loss;
        s[1] += c;
        s[2] += r;
        s[3] += good && h > 0.0 ? 1.0 : 0.0;
        s[4] += good ? 0.0 : 1.0;
    }
    if (bad_length && a.status) atomicOr(a.status, DAT_STATUS_BAD_LENGTH);
#pragma unroll
    for (int k = 0; k < kPrSums; k++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
        if (lane == 0) part[k][warp] = s[k];
    }
    __syncthreads();
    if (tid < kPrSums) {
        double t = 0.0;
        for (int w = 0; w < kPrThreads / 32; w++) t += part[tid][w];
        mine[tid] = t;
    }
    cluster.sync();
    if (rank == 0 && tid < kPrSums) {
        double t = 0.0;
        for (int q = 0; q < kPrCtas; q++) t += *cluster.map_shared_rank(&mine[tid], q);
        a.stats[tid < 4 ? tid : 5] = t;
        if (tid == 0) *a.loss = a.n > 0 ? (float)(t / a.n) : 0.f;
        if (tid == 4) a.stats[4] = (double)a.n;
    }
    cluster.sync();   // the other CTAs' sums are read before they leave
}

}  // namespace dat

extern "C" int dat_preference_loss(const float *chosen, const float *rejected, const float *ref_chosen,
                                   const float *ref_rejected, const int64_t *chosen_length,
                                   const int64_t *rejected_length, double beta, double smoothing, int kind, float *loss,
                                   float *rewards, double *stats, float *grad, int32_t *status, int pairs, void *stream) {
    using namespace dat;
    const char *who = "dat_preference_loss";
    DAT_REQUIRE(pairs >= 0 && loss && stats && (pairs == 0 || (chosen && rejected && rewards)), DAT_ERR_BAD_ARG,
                "%s: bad argument", who);
    DAT_REQUIRE(!ref_chosen == !ref_rejected && !chosen_length == !rejected_length, DAT_ERR_BAD_ARG,
                "%s: references and lengths are given for both sentences of a pair or for neither", who);
    DAT_REQUIRE(kind >= DAT_PREFERENCE_SIGMOID && kind <= DAT_PREFERENCE_SQUARED, DAT_ERR_BAD_ARG, "%s: bad kind %d", who,
                kind);
    DAT_REQUIRE(smoothing >= 0.0 && smoothing <= 1.0, DAT_ERR_BAD_ARG, "%s: smoothing outside [0, 1]", who);
    const PreferenceArgs a{chosen, rejected, ref_chosen, ref_rejected, chosen_length, rejected_length, beta, smoothing,
                           kind, loss, rewards, stats, grad, status, pairs};
    preference_kernel<<<kPrCtas, kPrThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    return check_launch(who);
}

// Clipped policy loss with a KL term over the vertices' logits, forward and backward, for sm_100a.
//
// A step of a sampled path takes a token at a vertex and a transition to the next vertex, so that
//     lp[b,l] = log softmax(x[b,l,:])[token] (+ link_logp[b,l])
// and with r = exp(lp - old), advantage A and the active vertices N,
//     term = -min(r A, clip(r, 1-low, 1+high) A),     loss = 1/N sum_active (term + beta KL).
// KL, one of
//     full      sum_v p_v (log p_v - log q_v) over the vocabulary, q = softmax(y) of the reference model,
//     estimate  e^u - u - 1, u = ref_logp - lp.
// Gradient of the loss with respect to x_v of an active vertex, with delta the one-hot of the token:
//     1/N [ c (delta_v - p_v) + beta p_v (d_v - E_p d) ],   d = x - y (full KL only),
//     c = -A r where the clip does not hold the term, 0 where it does, + beta (1 - e^u) with the estimate.
//
// HBM-bound: the logits of the active vertices are read once and the dense gradient is written once.  To read
// them once the gradient is written by the forward, scaled by the gradient that the caller expects the loss to
// receive (1, or a loss scale).  The backward compares that with what arrives, on the device, and computes the
// gradient again from the logits where they differ.  Two forms: long rows pass through the shared memory
// (policy_ring_kernel), rows of a few KB take a CTA each that reads them a second time from the L1 or L2 cache
// (policy_fwd_kernel).
//
// Numerics: sums in fp32 with exact differences to a reference (the running maximum; in the ring kernel the
// token's logit, so that lp = -log S needs no further difference): a rounding of 2^-24 in each of a thread's additions,
// below 1e-6 of the sum together with the exponentials' own.  The log-probability and the KL of a row are
// put together in 64 bits (a maximum and a log-sum near 10 carry 5e-7, which would show in the ratio); the ring kernel takes
// the ratio, its term and the gradient's factors from there in 32 bits (1e-7 of each), because the gradient of a row waits
// for them: with all of it in 64 bits 32768 rows of 32000 took 3 % longer.  Sums over rows in 64 bits in a fixed order.  d is
// taken relative to its value at one place of the row, so that a constant between the two models' logits does not cancel.
//
// The KL over the vocabulary is E_p d + log(S_y / S), whose parts cancel where the models are close: the rounding of the
// sums leaves some 1e-7 of them, more than a KL near 0 has.  A row whose KL comes out below kPoNear is gone over
// again.  With u = d - o, o the mean of d from the first time, and phi(u) = e^-u - 1 + u,
//     KL = m + log(1 + f - m),   m = E_p u (near 0),   f = E_p phi(u),
// for any o, since E_p e^-u = e^o S_y / S.  phi is not negative and near u^2 / 2, by its power series for small u: nothing
// cancels but m with itself.  policy_fwd_kernel does it from the cache; after policy_ring_kernel a kernel of its own
// (policy_near_kernel) reads such rows again from memory.  32768 rows of 32000 bf16 logits, none and all of them close:
// 1.13 and 2.0 ms; with the second time inside the ring 1.25 and 1.73, since the code for it slowed the loops of all rows.
#include "cluster_util.cuh"
#include "dat_common.cuh"
#include "umma.cuh"

namespace dat {

constexpr int kPoThreads = 256;
constexpr int kPoWarps = kPoThreads / 32;
constexpr int kPoChunk = 256;   // rows whose results are summed together
constexpr int kPoSums = 5;      // terms, KL, ratios, clipped, active
constexpr float kPoNear = 0.0625f;   // KL below which a row is gone over again: above, 5e-7 is 1e-5 of it

// start of the caller's workspace
struct PolicyHead {
    double inv_n;      // 1 / active rows (1 / max(1, n))
    float scale;       // gradient that the forward assumed for the loss
    int chunks_done;
};

struct PolicyArgs {
    const void *x, *y;            // logits [rows, V]; y null without the full KL
    const int64_t *tokens;        // [rows]
    const float *old_logp;        // [rows]
    const float *advantage;
    int64_t adv_b, adv_l;         // strides of the advantage
    const float *link_logp;       // [rows] or null
    const float *ref_logp;        // [rows] or null
    const unsigned char *mask;    // [rows] or null
    float beta, clip_low, clip_high;
    float *loss;                  // [1]
    double *stats;                // [kPoSums]
    float *logp, *kl;             // [rows]
    float4 *row_state;            // [rows][2]: r, 1 / S, c / N, E_p d; ry (for the backward), or null
    void *grad;                   // [rows, V] or null
    PolicyHead *head;
    int *done;                    // [chunks]
    float4 *row_sums;             // [rows]: term, KL, ratio, clipped; of the ring kernel with y: see PolicyNear
    double *chunk_sums;           // [chunks, kPoSums]
    int32_t *status;
    int64_t rows;
    int L, V;
    bool vec;                     // x, y and grad start on 16-byte boundaries
};

// counts the active rows and clears the counters
__global__ void __launch_bounds__(1024)
policy_prep_kernel(const unsigned char *__restrict__ mask, int64_t rows, PolicyHead *head, int *done, int chunks,
                   const float *scale_ptr, float scale) {
    __shared__ long long part[32];
    const int tid = threadIdx.x;
    long long n = 0;
    pdl_trigger();
    if (mask)
        for (int64_t r = tid; r < rows; r += 1024) n += mask[r] != 0;
    for (int c = tid; c < chunks; c += 1024) done[c] = 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
    if ((tid & 31) == 0) part[tid >> 5] = n;
    __syncthreads();
    if (tid == 0) {
        long long t = 0;
        for (int w = 0; w < 32; w++) t += part[w];
        if (!mask) t = rows;
        head->inv_n = 1.0 / (double)(t > 0 ? t : 1);
        head->scale = scale_ptr ? *scale_ptr : scale;
        head->chunks_done = 0;
    }
}

template <typename T>
__device__ __forceinline__ void policy_split(bool vec, const T *p, int V, int &head, int &nvec) {
    constexpr int kVec = Elem<T>::kVec;
    if (!vec) {
        head = V;
        nvec = 0;
        return;
    }
    const int mis = (int)((reinterpret_cast<uintptr_t>(p) & 15u) / sizeof(T));
    head = mis ? kVec - mis : 0;
    if (head > V) head = V;
    nvec = (V - head) / kVec;
}

// Running state of a thread over its share of a row.
template <bool kRef>
struct PolicyState {
    float m = kNegBig, s = 0.f, t = 0.f;   // maximum, sum e^(x-m), sum e^(x-m) d
    float my = kNegBig, sy = 0.f;          // the same of the reference
    template <int N>
    __device__ __forceinline__ void update(const float (&x)[N], const float (&y)[N], float off) {
        float v = x[0];
#pragma unroll
        for (int i = 1; i < N; i++) v = fmaxf(v, x[i]);
        if (v > m) {
            const float f = ex2((m - v) * kLog2e);
            s *= f;
            if (kRef) t *= f;
            m = v;
        }
#pragma unroll
        for (int i = 0; i < N; i++) {
            const float e = ex2((x[i] - m) * kLog2e);
            s += e;
            // where p = 0 (a score of -inf) d may be -inf or NaN: fmaxf makes it a number, the product 0
            if (kRef) t = fmaf(e, fmaxf((x[i] - off) - y[i], kNegBig), t);
        }
        if (kRef) {
            v = y[0];
#pragma unroll
            for (int i = 1; i < N; i++) v = fmaxf(v, y[i]);
            if (v > my) {
                sy *= ex2((my - v) * kLog2e);
                my = v;
            }
#pragma unroll
            for (int i = 0; i < N; i++) sy += ex2((y[i] - my) * kLog2e);
        }
    }
};

// A pair of fp32 numbers in one 64-bit register, so that the two-lane instructions need no moves between them.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2(float a, float b) {
    F2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void f2_get(F2 v, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ F2 f2_add(F2 a, F2 b) {
    F2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
    F2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
    F2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ F2 f2_ex2(F2 v) {
    float a, b;
    f2_get(v, a, b);
    return f2(ex2(a), ex2(b));
}
__device__ __forceinline__ F2 f2_floor(F2 v) {   // what is below -1e30, or NaN, becomes -1e30
    float a, b;
    f2_get(v, a, b);
    return f2(fmaxf(a, kNegBig), fmaxf(b, kNegBig));
}

// 16 bytes of logits less a reference, as pairs (sm_100 subtracts an fp32 number from a 16-bit one in one instruction,
// rounded once)
__device__ __forceinline__ void policy_pairs(const uint4 &u, F2 (&p)[2], float r, const float *) {
    p[0] = f2_add(f2(__uint_as_float(u.x), __uint_as_float(u.y)), f2(-r, -r));
    p[1] = f2_add(f2(__uint_as_float(u.z), __uint_as_float(u.w)), f2(-r, -r));
}
__device__ __forceinline__ void policy_pairs(const uint4 &u, F2 (&p)[4], float r, const __nv_bfloat16 *) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a, b;
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.bf16 %0, l, %3;\n\tsub.rn.f32.bf16 %1, h, %3;\n\t}" : "=f"(a), "=f"(b) : "r"(w[i]), "f"(r));
        p[i] = f2(a, b);
    }
}
__device__ __forceinline__ void policy_pairs(const uint4 &u, F2 (&p)[4], float r, const __half *) {
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int i = 0; i < 4; i++) {
        float a, b;
        asm("{\n\t.reg .b16 l, h;\n\tmov.b32 {l, h}, %2;\n\tsub.rn.f32.f16 %0, l, %3;\n\tsub.rn.f32.f16 %1, h, %3;\n\t}" : "=f"(a), "=f"(b) : "r"(w[i]), "f"(r));
        p[i] = f2(a, b);
    }
}

// (e^-u - 1 + u) / u^2 for |u| < 1: the power series, whose first term left out is below 2^-23 of it
constexpr float kPoSmall = 1.f;
__device__ __forceinline__ F2 policy_phi(F2 u) {
    constexpr float c[8] = {-1.f / 362880.f, 1.f / 40320.f, -1.f / 5040.f, 1.f / 720.f, -1.f / 120.f, 1.f / 24.f, -1.f / 6.f, 0.5f};
    F2 p = f2(1.f / 3628800.f, 1.f / 3628800.f);
#pragma unroll
    for (int k = 0; k < 8; k++) p = f2_fma(u, p, f2(c[k], c[k]));
    return p;
}
// A thread's sums of e = e^(x - r), e u and e phi(u) with u = x - y - o
struct PolicyNearAcc {
    F2 s = 0, u_sum = 0, f_sum = 0;   // (0, 0)
    template <int N>
    __device__ __forceinline__ void add(const F2 (&x)[N], const F2 (&y)[N], float r, float o) {
        const auto both = [](float v) { return f2(v, v); };
        F2 e[N], u[N];
        float most = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) {
            e[i] = f2_ex2(f2_fma(x[i], both(kLog2e), both(-r * kLog2e)));   // (what r log2e is rounded by divides out)
            u[i] = f2_add(f2_fma(y[i], both(-1.f), x[i]), both(-o));
            float u0, u1;
            f2_get(u[i], u0, u1);
            asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(most) : "f"(most), "f"(u0), "f"(u1));
            s = f2_add(s, e[i]);
        }
        if (most < kPoSmall) {
#pragma unroll
            for (int i = 0; i < N; i++) {
                const F2 eu = f2_mul(e[i], u[i]);
                u_sum = f2_add(u_sum, eu);
                f_sum = f2_fma(f2_mul(eu, u[i]), policy_phi(u[i]), f_sum);
            }
        } else {
#pragma unroll
            for (int i = 0; i < N; i++) {
                float e0, e1, u0, u1, y0, y1, p0, p1;
                // (x = -inf: u is made a number, e is 0, and what is left of the term is what the reference has there)
                u[i] = f2_floor(u[i]);
                u_sum = f2_fma(e[i], u[i], u_sum);
                f2_get(e[i], e0, e1);
                f2_get(u[i], u0, u1);
                f2_get(y[i], y0, y1);
                f2_get(policy_phi(u[i]), p0, p1);
                f_sum = f2_add(f_sum, f2(term(e0, u0, y0 - r + o, p0), term(e1, u1, y1 - r + o, p1)));
            }
        }
    }
    __device__ __forceinline__ void add1(float x, float y, float r, float o) {   // (a place without weight beside it)
        const F2 px[1] = {f2(x, -INFINITY)}, py[1] = {f2(y, -INFINITY)};
        add(px, py, r, o);
    }
    // e e^-u = e^(y - r + o), which holds where e^-u alone would not
    static __device__ __forceinline__ float term(float e, float u, float yr, float phi) {
        return fabsf(u) < kPoSmall ? e * (u * u) * phi : ex2(yr * kLog2e) - e + e * u;
    }
    static __device__ __forceinline__ float both(F2 v) {
        float a, b;
        f2_get(v, a, b);
        return a + b;
    }
};
// the KL from the sums (what the 64-bit roundings may leave below 0 is 0; NaN stays)
__device__ __forceinline__ double policy_near_kl(double S, double U, double F) {
    const double kl = U / S + log1p((F - U) / S);
    return kl < 0.0 ? 0.0 : kl;
}

// d at v = 0, or 0 where that is no number
template <typename T>
__device__ __forceinline__ float policy_offset(const T *x, const T *y) {
    const float o = Elem<T>::to_float(x[0]) - Elem<T>::to_float(y[0]);
    return fabsf(o) < 1e30f ? o : 0.f;
}

// What the gradient of a row is made of: e (w (d - mean) + a) with e = exp(x - r), d = (x - r) - (y - ry),
// a = -c / (N S), w = beta / (N S), each times the loss's gradient, and tok_c = c / N times it at the token.
struct PolicyRow {
    float r, ry, a, w, mean, tok_c;
};
template <bool kRef>
__device__ __forceinline__ float policy_grad_one(const PolicyRow &p, float x, float y) {
    const float dx = x - p.r, e = ex2(dx * kLog2e);
    return e * (kRef ? fmaf(p.w, fmaxf(dx - (y - p.ry), kNegBig) - p.mean, p.a) : p.a);
}

// The gradient of one active row.
template <typename T, bool kRef>
__device__ __forceinline__ void policy_grad_row(const T *x, const T *y, T *g, bool vec, int V, const PolicyRow &p, int64_t tok) {
    constexpr int kVec = Elem<T>::kVec;
    const int tid = threadIdx.x;
    int head, nvec;
    policy_split(vec, x, V, head, nvec);
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head), *yv = reinterpret_cast<const uint4 *>(kRef ? y + head : x);
    uint4 *gv = reinterpret_cast<uint4 *>(g + head);
    auto one = [&](float xe, float ye) { return policy_grad_one<kRef>(p, xe, ye); };
    constexpr int U = 2;
    for (int v = tid; v < nvec; v += U * kPoThreads) {
        uint4 ux[U], uy[U];
#pragma unroll
        for (int q = 0; q < U; q++)
            if (v + q * kPoThreads < nvec) {
                ux[q] = xv[v + q * kPoThreads];
                if (kRef) uy[q] = yv[v + q * kPoThreads];
            }
#pragma unroll
        for (int q = 0; q < U; q++)
            if (v + q * kPoThreads < nvec) {
                float fx[kVec], fy[kVec];
                Elem<T>::unpack(ux[q], fx);
                if (kRef) Elem<T>::unpack(uy[q], fy);
#pragma unroll
                for (int i = 0; i < kVec; i++) fx[i] = one(fx[i], kRef ? fy[i] : 0.f);
                gv[v + q * kPoThreads] = Elem<T>::pack(fx);
            }
    }
    for (int e = tid; e < head; e += kPoThreads)
        g[e] = Elem<T>::from_float(one(Elem<T>::to_float(x[e]), kRef ? Elem<T>::to_float(y[e]) : 0.f));
    for (int e = head + nvec * kVec + tid; e < V; e += kPoThreads)
        g[e] = Elem<T>::from_float(one(Elem<T>::to_float(x[e]), kRef ? Elem<T>::to_float(y[e]) : 0.f));
    __syncthreads();
    if (tid == 0 && tok >= 0 && tok < V)
        g[tok] = Elem<T>::from_float(p.tok_c + one(Elem<T>::to_float(x[tok]), kRef ? Elem<T>::to_float(y[tok]) : 0.f));
}

template <typename T>
__device__ __forceinline__ void policy_zero_row(T *g, bool vec, int V) {
    constexpr int kVec = Elem<T>::kVec;
    int head, nvec;
    policy_split(vec, g, V, head, nvec);
    uint4 *gv = reinterpret_cast<uint4 *>(g + head);
    for (int v = threadIdx.x; v < nvec; v += kPoThreads) gv[v] = make_uint4(0, 0, 0, 0);
    for (int e = threadIdx.x; e < head; e += kPoThreads) g[e] = Elem<T>::from_float(0.f);
    for (int e = head + nvec * kVec + threadIdx.x; e < V; e += kPoThreads) g[e] = Elem<T>::from_float(0.f);
}

// Sums the rows' results: the CTA that finishes the last row of a chunk adds the chunk's, the one that finishes
// the last chunk adds the chunks', each in a fixed order.
__device__ __forceinline__ void policy_sums(const PolicyArgs &a, int64_t row) {
    __shared__ int last_s;
    __shared__ double part[kPoSums][kPoWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int chunk = (int)(row / kPoChunk);
    const int chunks = (int)((a.rows + kPoChunk - 1) / kPoChunk);
    const int64_t first = (int64_t)chunk * kPoChunk;
    const int n = a.rows - first < kPoChunk ? (int)(a.rows - first) : kPoChunk;
    if (tid == 0) {
        __threadfence();
        last_s = atomicAdd(a.done + chunk, 1) == n - 1;
    }
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    double s[kPoSums] = {};
    if (tid < n && (!a.mask || a.mask[first + tid])) {
        const float4 r = __ldcg(a.row_sums + first + tid);
        s[0] = r.x;
        s[1] = r.y;
        s[2] = r.z;
        s[3] = r.w;
        s[4] = 1.0;
    }
#pragma unroll
    for (int k = 0; k < kPoSums; k++) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s[k] += __shfl_xor_sync(0xffffffffu, s[k], o);
        if (lane == 0) part[k][warp] = s[k];
    }
    __syncthreads();
    if (tid == 0) {
        for (int k = 0; k < kPoSums; k++) {
            double t = 0.0;
            for (int w = 0; w < kPoWarps; w++) t += part[k][w];
            a.chunk_sums[(int64_t)chunk * kPoSums + k] = t;
        }
        __threadfence();
        last_s = atomicAdd(&a.head->chunks_done, 1) == chunks - 1;
    }
    __syncthreads();
    if (!last_s) return;
    __threadfence();
    if (warp < kPoSums) {
        double t = 0.0;
        for (int c = lane; c < chunks; c += 32) t += __ldcg(a.chunk_sums + (int64_t)c * kPoSums + warp);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (lane == 0) {
            a.stats[warp] = t;
            part[warp][0] = t;
        }
    }
    __syncthreads();
    if (tid == 0) *a.loss = (float)((part[0][0] + (double)a.beta * part[1][0]) * a.head->inv_n);
}

template <typename T, bool kRef>
__global__ void __launch_bounds__(kPoThreads)
policy_fwd_kernel(PolicyArgs a) {
    constexpr int kVec = Elem<T>::kVec;
    __shared__ float red[5][kPoWarps], red_near[3][kPoWarps];
    __shared__ PolicyRow row_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x;
    const int V = a.V;
    T *g = a.grad ? static_cast<T *>(a.grad) + row * V : nullptr;
    if (a.mask && !a.mask[row]) {
        if (g) policy_zero_row(g, a.vec, V);
        if (tid == 0) {
            a.logp[row] = 0.f;
            a.kl[row] = 0.f;
            if (a.row_state) a.row_state[2 * row] = a.row_state[2 * row + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        policy_sums(a, row);
        return;
    }
    const T *x = static_cast<const T *>(a.x) + row * V;
    const T *y = kRef ? static_cast<const T *>(a.y) + row * V : nullptr;
    const float off = kRef ? policy_offset(x, y) : 0.f;
    int head, nvec;
    policy_split(a.vec, x, V, head, nvec);
    const uint4 *xv = reinterpret_cast<const uint4 *>(x + head), *yv = reinterpret_cast<const uint4 *>(kRef ? y + head : x);
    PolicyState<kRef> st;
    constexpr int U = 2;
    int v = tid;
    for (; v + (U - 1) * kPoThreads < nvec; v += U * kPoThreads) {
        uint4 ux[U], uy[U];
#pragma unroll
        for (int q = 0; q < U; q++) {
            ux[q] = xv[v + q * kPoThreads];
            if (kRef) uy[q] = yv[v + q * kPoThreads];
        }
        float fx[U * kVec], fy[U * kVec];
#pragma unroll
        for (int q = 0; q < U; q++) {
            Elem<T>::unpack(ux[q], fx + q * kVec);
            if (kRef) Elem<T>::unpack(uy[q], fy + q * kVec);
        }
        st.update(fx, fy, off);
    }
    for (; v < nvec; v += kPoThreads) {
        float fx[kVec], fy[kVec];
        Elem<T>::unpack(xv[v], fx);
        if (kRef) Elem<T>::unpack(yv[v], fy);
        st.update(fx, fy, off);
    }
    for (int part = 0; part < 2; part++) {
        const int e0 = part ? head + nvec * kVec : 0, e1 = part ? V : head;
        for (int e = e0 + tid; e < e1; e += kPoThreads) {
            const float fx[1] = {Elem<T>::to_float(x[e])}, fy[1] = {kRef ? Elem<T>::to_float(y[e]) : 0.f};
            st.update(fx, fy, off);
        }
    }
    // the row's maxima, then its sums
    const float wm = warp_max(st.m), wmy = kRef ? warp_max(st.my) : 0.f;
    if (lane == 0) {
        red[0][warp] = wm;
        red[1][warp] = wmy;
    }
    __syncthreads();
    float M = red[0][0], My = red[1][0];
#pragma unroll
    for (int w = 1; w < kPoWarps; w++) {
        M = fmaxf(M, red[0][w]);
        My = fmaxf(My, red[1][w]);
    }
    const float f = ex2((st.m - M) * kLog2e);
    const float ws = warp_sum(st.s * f);
    const float wt = kRef ? warp_sum(st.t * f) : 0.f, wsy = kRef ? warp_sum(st.sy * ex2((st.my - My) * kLog2e)) : 0.f;
    if (lane == 0) {
        red[2][warp] = ws;
        red[3][warp] = wt;
        red[4][warp] = wsy;
    }
    __syncthreads();
    bool near = false;
    float shift = 0.f;   // o
    if (kRef) {
        float S = 0.f, Tt = 0.f, Sy = 0.f;
        for (int w = 0; w < kPoWarps; w++) {
            S += red[2][w];
            Tt += red[3][w];
            Sy += red[4][w];
        }
        const float mean = Tt / S;
        shift = off + mean;
        near = mean - ((M - off - My) + logf(S / Sy)) < kPoNear;   // the same in all threads
        if (near) {
            PolicyNearAcc acc;
            for (int q = tid; q < nvec; q += kPoThreads) {
                F2 px[kVec / 2], py[kVec / 2];
                policy_pairs(xv[q], px, 0.f, x);
                policy_pairs(yv[q], py, 0.f, x);
                acc.add(px, py, M, shift);
            }
            for (int part = 0; part < 2; part++) {
                const int e0 = part ? head + nvec * kVec : 0, e1 = part ? V : head;
                for (int e = e0 + tid; e < e1; e += kPoThreads)
                    acc.add1(Elem<T>::to_float(x[e]), Elem<T>::to_float(y[e]), M, shift);
            }
            const float we = warp_sum(acc.both(acc.s)), wu = warp_sum(acc.both(acc.u_sum)), wf = warp_sum(acc.both(acc.f_sum));
            if (lane == 0) {
                red_near[0][warp] = we;
                red_near[1][warp] = wu;
                red_near[2][warp] = wf;
            }
            __syncthreads();
        }
    }
    const int64_t tok = a.tokens[row];
    if (tid == 0) {
        double S = 0.0, Tt = 0.0, Sy = 0.0;
        for (int w = 0; w < kPoWarps; w++) {
            S += red[2][w];
            Tt += red[3][w];
            Sy += red[4][w];
        }
        const bool ok = tok >= 0 && tok < V;
        if (!ok && a.status) atomicOr(a.status, DAT_STATUS_BAD_INDEX);
        const int64_t b = row / a.L, l = row - b * a.L;
        const double A = a.advantage[b * a.adv_b + l * a.adv_l];
        const double log_s = log(S);
        double lp = ok ? (double)(Elem<T>::to_float(x[tok])) - (double)M - log_s : __longlong_as_double(0x7ff8000000000000ll);
        if (a.link_logp) lp += a.link_logp[row];
        const double r = exp(lp - (double)a.old_logp[row]);
        const double lo = 1.0 - (double)a.clip_low, hi = 1.0 + (double)a.clip_high;
        const double ra = r * A, rc = (r < lo ? lo : r > hi ? hi : r) * A;
        const double term = -(ra < rc ? ra : rc);
        const bool clipped = (A > 0.0 && r > hi) || (A < 0.0 && r < lo);
        double c = clipped ? 0.0 : -ra, kl = 0.0, mean_d = 0.0;
        if (kRef) {
            mean_d = Tt / S;
            kl = mean_d - (((double)M - (double)off - (double)My) + log_s - log(Sy));
            if (near) {
                double t[3] = {};
                for (int k = 0; k < 3; k++)
                    for (int w = 0; w < kPoWarps; w++) t[k] += red_near[k][w];
                kl = policy_near_kl(t[0], t[1], t[2]);
                mean_d = t[1] / t[0] + ((double)shift - (double)off);
            }
        } else if (a.ref_logp) {
            const double u = (double)a.ref_logp[row] - lp, eu = expm1(u);
            kl = eu - u;
            c -= (double)a.beta * eu;
        }
        a.logp[row] = (float)lp;
        a.kl[row] = (float)kl;
        a.row_sums[row] = make_float4((float)term, (float)kl, (float)r, clipped ? 1.f : 0.f);
        const double inv_n = a.head->inv_n, up = inv_n * (double)a.head->scale;
        const float ry = M - off;
        if (a.row_state) {
            a.row_state[2 * row] = make_float4(M, (float)(1.0 / S), (float)(c * inv_n), (float)mean_d);
            a.row_state[2 * row + 1] = make_float4(ry, 0.f, 0.f, 0.f);
        }
        row_s.r = M;
        row_s.ry = ry;
        row_s.a = (float)(-c * up / S);
        row_s.w = (float)((double)a.beta * up / S);
        row_s.mean = (float)mean_d;
        row_s.tok_c = (float)(c * up);
    }
    __syncthreads();
    if (g) policy_grad_row<T, kRef>(x, y, g, a.vec, V, row_s, tok);
    policy_sums(a, row);
}

// ---------------------------------------------------------------------------------------------------
// Rows of some KB and up that fit the shared memory: a persistent CTA keeps a row (and the reference's) in shared
// memory between the sum and the gradient, so that HBM sees every logit once.  Its warps share the work as a
// pipeline over rows: a producer brings chunks of rows by bulk asynchronous copies into a ring of slots, one half of
// the others sums row n + 1 while the other half writes the gradient of row n and frees its slots, and one warp
// writes the zeros of the inactive vertices' rows from a block of zeros by bulk copies.  (With all warps on one row
// the SM waits for the row's last sum, its numbers and the first chunk of the next: 32768 rows of 32000 bf16 logits
// and as many of the reference took 1.42 ms.)  Measured there: 1.12 to 1.16 ms, 5.3 to 5.5 TB/s of the bytes that it
// cannot do without; 32768 rows of 42000 fp16 logits, one in eight active: 0.63 ms for the whole call, 5.4 TB/s.
// The sums are taken relative to the token's logits r = x[token], ry = y[token] in place of the maxima: they are at
// least 1, and a row where one passes kPpHuge (a token less likely than e^-41, or no number) takes the maxima after all.  One
// barrier per row; every thread puts the row's numbers together for itself.
// Next to HBM the special-function unit bounds it: three exponentials per logit pair with the full KL, 24 of its
// cycles per 32 pairs and scheduler against 33 that HBM takes for the 6 bytes of each at 16 bits.
// ---------------------------------------------------------------------------------------------------
constexpr int kPpPolls = 1 << 20;      // bound of a wait (never reached)
constexpr int kPpZeros = 4096;         // bytes of zeros
// sums up to here keep the gradient's factors, c / (N S), normal numbers for any c / N above 2^-66
constexpr float kPpHuge = 0x1p60f;

constexpr int kPpDepth = 4;            // rows under way in a CTA
constexpr int kPpRanks = 8;            // CTAs that share a row at most

struct PolicyRing {
    int ranks;                    // CTAs (of a cluster) that share a row, its chunks dealt to them in turn
    int chunks, slots;            // chunks of a row that a CTA has, slots of the ring: chunks <= slots <= kPpDepth * chunks
    int zeros, bars, red, x, y;   // places in the shared memory
};
// a CTA's sums of a row, relative to (r, ry)
struct PolicyPart {
    float r, ry, S, T, Sy;
    uint32_t careful;   // the row has logits of -inf
};
// what the writing half needs of a row
struct PolicyHand {
    PolicyRow row;
    float xt, yt;   // the token's logits
    int tok;        // -1: outside the vocabulary
    uint32_t careful;
};
template <bool B>
struct PolicyBool {
    static constexpr bool value = B;
};
// position of a row's chunk in the ring: slot and the parity of the phase in which it is full
struct PolicyTurn {
    int slot = 0;
    uint32_t phase = 0;
    __device__ __forceinline__ void next(int slots) {
        if (++slot == slots) {
            slot = 0;
            phase ^= 1;
        }
    }
};

// Waits for a phase of a barrier.  false: gave up.
__device__ __forceinline__ bool policy_wait(uint64_t *mbar, uint32_t parity, int polls) {
    return umma::mbar_wait(mbar, parity, polls);
}

// The rows of a cluster, its number + k * clusters, 32 at a time through the mask; next() gives those whose bit is set.
struct PolicyWalk {
    const unsigned char *mask;
    int64_t rows;
    int step;            // clusters of the grid
    int64_t base;        // row of the block's lane 0
    unsigned bits, ahead;
    bool inactive;       // walk the rows that take no part
    __device__ __forceinline__ unsigned look(int64_t from) const {
        const int64_t r = from + (int64_t)(threadIdx.x & 31) * step;
        return r < rows ? ((!mask || mask[r] != 0) != inactive ? 1u : 0u) : 0u;
    }
    __device__ __forceinline__ PolicyWalk(const unsigned char *m, int64_t n, int ranks, bool skip)
        : mask(m), rows(n), step(gridDim.x / ranks), inactive(skip) {
        base = blockIdx.x / ranks;
        bits = __ballot_sync(0xffffffffu, look(base));
        ahead = look(base + 32 * (int64_t)step);
    }
    __device__ __forceinline__ int64_t next() {
        while (!bits) {
            base += 32 * (int64_t)step;
            if (base >= rows) return -1;
            bits = __ballot_sync(0xffffffffu, ahead);
            ahead = look(base + 32 * (int64_t)step);
        }
        const int j = __ffs(bits) - 1;
        bits &= bits - 1;
        return base + (int64_t)j * step;
    }
};

// A row in the ring: the 16-byte pieces that lie wholly inside it; the elements before and behind them are `head`
// and `tail` (each fewer than a piece has).
template <typename T>
struct PolicySpan {
    int head, vecs, tail;
    __device__ __forceinline__ PolicySpan(int64_t row, int V) {
        constexpr int kVec = Elem<T>::kVec;
        head = (int)(-(row * V) & (kVec - 1));
        if (head > V) head = V;
        vecs = (V - head) / kVec;
        tail = V - head - vecs * kVec;
    }
};

__device__ __forceinline__ void policy_bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t mbar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(mbar)
                 : "memory");
}
__device__ __forceinline__ void policy_arrive(uint64_t *mbar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(umma::smem_u32(mbar)) : "memory");
}

// Sums of a thread's logits relative to (r, ry).  kCareful: a logit of -inf in x makes d = (x-r) - (y-ry) -inf or NaN
// where p is 0; it is made a number there.  Without, such a row shows as a sum that is NaN.
template <bool kRef>
struct PolicyAcc {
    F2 s = 0, t = 0, sy = 0;   // (0, 0)
    template <bool kCareful, int N>
    __device__ __forceinline__ void add(const F2 (&x)[N], const F2 (&y)[N]) {
        const F2 l2e = f2(kLog2e, kLog2e), neg = f2(-1.f, -1.f);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const F2 a = x[i], e = f2_ex2(f2_mul(a, l2e));
            s = f2_add(s, e);
            if (kRef) {
                const F2 b = y[i];
                F2 d = f2_fma(b, neg, a);
                if (kCareful) d = f2_floor(d);
                t = f2_fma(e, d, t);
                sy = f2_add(sy, f2_ex2(f2_mul(b, l2e)));
            }
        }
    }
    __device__ __forceinline__ void add1(float x, float y, float r, float ry) {
        const float a = x - r, e = ex2(a * kLog2e);
        s = f2_add(s, f2(e, 0.f));
        if (kRef) {
            const float b = y - ry;
            t = f2_add(t, f2(e * fmaxf(a - b, kNegBig), 0.f));
            sy = f2_add(sy, f2(ex2(b * kLog2e), 0.f));
        }
    }
    static __device__ __forceinline__ float both(F2 v) {
        float a, b;
        f2_get(v, a, b);
        return a + b;
    }
};

// the gradient of pairs of logits
template <bool kRef, bool kCareful, int N>
__device__ __forceinline__ void policy_grad_pairs(const PolicyRow &p, const F2 (&x)[N], const F2 (&y)[N], float (&out)[2 * N]) {
    const float base = kRef ? fmaf(-p.w, p.mean, p.a) : p.a;
    const F2 l2e = f2(kLog2e, kLog2e), neg = f2(-1.f, -1.f), w = f2(p.w, p.w),
             bb = f2(base, base);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const F2 a = x[i], e = f2_ex2(f2_mul(a, l2e));
        F2 k = bb;
        if (kRef) {
            F2 d = f2_fma(y[i], neg, a);
            if (kCareful) d = f2_floor(d);
            k = f2_fma(d, w, bb);
        }
        f2_get(f2_mul(e, k), out[2 * i], out[2 * i + 1]);
    }
}

// the loss's numbers of a row from its sums
struct PolicyNumbers {
    float lp, u, term, kl, mean, cf, inv_s;
    bool clipped;
};
// log s in 64 bits: the exponent apart, so that the logarithm's rounding is one of a number below log 2 (a log-probability
// near -10 in 32 bits is off by up to 5e-7, and an estimated KL of a small step by as much over that step)
__device__ __forceinline__ double policy_log(float s) {
    if (!(s > 0.f && s < INFINITY)) return (double)logf(s);
    int k;
    const float m = frexpf(s, &k);
    return fma((double)k, 0.69314718055994530942, (double)logf(m));
}
// e^z - 1 - z without the cancellation of small z (its power series; the first term left out is below 2^-32 of the sum)
__device__ __forceinline__ float policy_excess(float z, float em) {
    if (fabsf(z) > 0.5f) return em - z;
    float t = 1.f;
#pragma unroll
    for (int k = 10; k >= 3; k--) t = fmaf(t * z, 1.f / k, 1.f);   // 1 + z/3 (1 + z/4 (1 + ..))
    return 0.5f * z * z * t;
}
template <bool kRef>
__device__ __forceinline__ PolicyNumbers policy_numbers(const PolicyArgs &a, const PolicyPart &p, bool ok, float xt, float A,
                                                        float old, float link, float ref) {
    PolicyNumbers n;
    const double lp = ok ? ((double)(xt - p.r) - policy_log(p.S)) + (double)link : __longlong_as_double(0x7ff8000000000000ll);
    n.lp = (float)lp;
    n.u = expf((float)(lp - (double)old));
    const float lo = 1.f - a.clip_low, hi = 1.f + a.clip_high;
    const float ra = n.u * A, rc = (n.u < lo ? lo : n.u > hi ? hi : n.u) * A;
    n.term = -(ra < rc ? ra : rc);
    n.clipped = (A > 0.f && n.u > hi) || (A < 0.f && n.u < lo);
    n.cf = n.clipped ? 0.f : -ra;
    n.kl = n.mean = 0.f;
    n.inv_s = 1.f / p.S;
    if (kRef) {
        n.mean = p.T / p.S;   // the KL apart: the gradient does not wait for it
    } else if (a.ref_logp) {
        const float z = (float)((double)ref - lp), em = expm1f(z);
        n.kl = policy_excess(z, em);
        n.cf = fmaf(-a.beta, em, n.cf);
    }
    return n;
}

// A row for policy_near_kernel: r and o (NaN: the row is not close), and the KL that the sums have got
struct PolicyNear {
    float r, o;
    double kl;
};
static_assert(sizeof(PolicyNear) == sizeof(float4), "a PolicyNear for each of row_sums");

// NT threads in each half, kPpVecs pieces of a chunk to each, three warps beside them
template <typename T, bool kRef, int NT, int kPpVecs>
__global__ void __launch_bounds__(2 * NT + 96, NT == 256 ? 1 : 3)
policy_ring_kernel(PolicyArgs a, PolicyRing ring) {
    constexpr int kVec = Elem<T>::kVec, kWarps = NT / 32, kChunk = NT * kPpVecs, kAll = 2 * NT + 96;
    extern __shared__ __align__(128) unsigned char posm[];
    __shared__ PolicyPart part_s[kPpDepth];               // a row's sums on their way to its numbers
    __shared__ PolicyHand hand_s[kPpDepth];               // and those on their way to the gradient
    __shared__ PolicyPart cluster_s[2][kPpRanks];         // the sums of all CTAs that share a row
    __shared__ __align__(8) uint64_t part_bar[kPpDepth], hand_bar[kPpDepth], cluster_bar[2];
    uint64_t *const full = reinterpret_cast<uint64_t *>(posm + ring.bars), *const empty = full + ring.slots;
    float4 *const red = reinterpret_cast<float4 *>(posm + ring.red);   // [2][kWarps]: S, T, Sy
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int V = a.V, ranks = ring.ranks, rank = blockIdx.x % ranks;
    for (int x = tid; x < kPpZeros / 16; x += kAll) reinterpret_cast<uint4 *>(posm + ring.zeros)[x] = make_uint4(0, 0, 0, 0);
    for (int x = tid; x < ring.slots; x += kAll) {
        umma::mbar_init(full + x, 1);
        umma::mbar_init(empty + x, kWarps);
    }
    if (tid < kPpDepth) {
        umma::mbar_init(part_bar + tid, 1);
        umma::mbar_init(hand_bar + tid, 1);
    }
    if (tid < 2) umma::mbar_init(cluster_bar + tid, 1);
    pdl_trigger();   // (policy_near_kernel, which waits for all of this)
    umma::fence_smem_to_async();
    __syncthreads();
    if (ranks > 1) cluster_barrier();   // every CTA's barriers stand before a neighbour's sums arrive on them
    bool stalled = false;
    const uint4 *const xs = reinterpret_cast<const uint4 *>(posm + ring.x), *const ys = reinterpret_cast<const uint4 *>(posm + ring.y);
    // x - r and y - ry of a piece of the ring
    const auto load = [&](int v, float r, float ry, F2 (&px)[kVec / 2], F2 (&py)[kVec / 2]) {
        policy_pairs(xs[v], px, r, static_cast<const T *>(nullptr));
        if (kRef) policy_pairs(ys[v], py, ry, static_cast<const T *>(nullptr));
    };
    const auto polls = [&] { return stalled ? 1 : kPpPolls; };
    PolicyTurn turn;

    if (warp == 2 * kWarps) {   // ---- producer
        PolicyWalk walk(a.mask, a.rows, ranks, false);
        for (int64_t row = walk.next(); row >= 0 && !stalled; row = walk.next()) {
            const PolicySpan<T> sp(row, V);
            const int64_t from = row * V + sp.head;
            for (int j = 0; j < ring.chunks && !stalled; j++, turn.next(ring.slots)) {
                const int c = j * ranks + rank, bytes = min(kChunk, sp.vecs - c * kChunk) * 16;
                if (lane == 0) {
                    stalled |= !policy_wait(empty + turn.slot, turn.phase ^ 1, kPpPolls);   // the ring begins empty
                    if (!stalled) {
                        const uint32_t mb = umma::smem_u32(full + turn.slot);
                        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mb),
                                     "r"(bytes > 0 ? bytes * (kRef ? 2 : 1) : 0)
                                     : "memory");
                        if (bytes > 0) {
                            const int64_t at = from + (int64_t)c * kChunk * kVec;
                            const uint32_t to = turn.slot * (kChunk * 16);
                            policy_bulk_load(umma::smem_u32(posm + ring.x) + to, static_cast<const T *>(a.x) + at, bytes, mb);
                            if (kRef) policy_bulk_load(umma::smem_u32(posm + ring.y) + to, static_cast<const T *>(a.y) + at, bytes, mb);
                        }
                    }
                }
                stalled = __any_sync(0xffffffffu, stalled);
            }
        }
    } else if (warp == 2 * kWarps + 1) {   // ---- zeros
        PolicyWalk walk(a.mask, a.rows, ranks, true);
        const uint32_t zeros = umma::smem_u32(posm + ring.zeros);
        for (int64_t row = a.mask ? walk.next() : -1; row >= 0; row = walk.next()) {
            if (lane == 0 && rank == 0) {
                a.logp[row] = 0.f;
                a.kl[row] = 0.f;
                if (a.row_state) a.row_state[2 * row] = a.row_state[2 * row + 1] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            if (!a.grad) continue;
            T *const g = static_cast<T *>(a.grad) + row * V;
            const PolicySpan<T> sp(row, V);
            const int bytes = sp.vecs * 16;
            if (rank == 0 && lane < sp.head) g[lane] = Elem<T>::from_float(0.f);
            if (rank == 0 && lane < sp.tail) g[V - sp.tail + lane] = Elem<T>::from_float(0.f);
            unsigned char *const mid = reinterpret_cast<unsigned char *>(g + sp.head);
            for (int at = (lane * ranks + rank) * kPpZeros; at < bytes; at += 32 * ranks * kPpZeros)
                asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(mid + at), "r"(zeros),
                             "r"(min(kPpZeros, bytes - at))
                             : "memory");
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
            asm volatile("cp.async.bulk.wait_group.read 4;" ::: "memory");   // a few rows at a time, beside the active ones
        }
        asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
    } else if (warp == 2 * kWarps + 2) {   // ---- numbers
        pdl_wait();   // the count of the active rows
        const double inv_n = a.head->inv_n;
        const float n1 = (float)inv_n, up = a.head->scale;
        PolicyWalk walk(a.mask, a.rows, ranks, false);
        double sums[kPoSums] = {};   // of this cluster's rows, in their order
        uint32_t n = 0;
        for (int64_t row = walk.next(); row >= 0; row = walk.next(), n++) {
            const int64_t b = row / a.L, l = row - b * a.L, tok = a.tokens[row];
            const bool ok = tok >= 0 && tok < V;
            const int64_t at = row * V + (ok ? tok : 0);
            const float xt = Elem<T>::to_float(static_cast<const T *>(a.x)[at]), yt = kRef ? Elem<T>::to_float(static_cast<const T *>(a.y)[at]) : 0.f;
            const float A = a.advantage[b * a.adv_b + l * a.adv_l], old = a.old_logp[row];
            const float link = a.link_logp ? a.link_logp[row] : 0.f, ref = a.ref_logp ? a.ref_logp[row] : 0.f;
            stalled |= !policy_wait(part_bar + n % kPpDepth, n / kPpDepth & 1, polls());
            PolicyPart p = part_s[n % kPpDepth];
            if (ranks > 1) {
                // to the neighbours, and theirs.  Two buffers do: a neighbour sends row n + 2 only after it has this
                // CTA's row n + 1, which is sent below once row n has been read.
                PolicyPart *const all = cluster_s[n & 1];
                uint64_t *const bar = cluster_bar + (n & 1);
                if (lane == 0) {
                    all[rank] = p;
                    cluster_mbar_expect(bar, (ranks - 1) * (uint32_t)sizeof(PolicyPart));
                }
                if (lane < ranks && lane != rank) {
                    const uint32_t to = cluster_map(all + rank, lane), rbar = cluster_map(bar, lane);
                    const uint32_t w[6] = {__float_as_uint(p.r), __float_as_uint(p.ry), __float_as_uint(p.S), __float_as_uint(p.T),
                                           __float_as_uint(p.Sy), p.careful};
#pragma unroll
                    for (int k = 0; k < 6; k++) cluster_st_async_b32(to + 4 * k, w[k], rbar);
                }
                __syncwarp();
                stalled |= !policy_wait(bar, n / 2 & 1, polls());
                // in the order of the ranks, relative to the largest reference (they differ only where a CTA took its
                // maximum)
                float r = -INFINITY, ry = -INFINITY;
                for (int q = 0; q < ranks; q++) {
                    if (all[q].S != 0.f) r = fmaxf(r, all[q].r);
                    if (all[q].Sy != 0.f) ry = fmaxf(ry, all[q].ry);
                }
                float S = 0.f, Tt = 0.f, Sy = 0.f;
                uint32_t careful = 0;
                for (int q = 0; q < ranks; q++) {
                    const PolicyPart o = all[q];
                    careful |= o.careful;
                    if (o.S != 0.f) {
                        const float f = o.r == r ? 1.f : ex2((o.r - r) * kLog2e), move = (o.r - r) - (o.ry - ry);
                        S = fmaf(o.S, f, S);
                        if (kRef) Tt = fmaf(move == 0.f ? o.T : fmaf(move, o.S, o.T), f, Tt);
                    }
                    if (kRef && o.Sy != 0.f) Sy = fmaf(o.Sy, o.ry == ry ? 1.f : ex2((o.ry - ry) * kLog2e), Sy);
                }
                p.r = r;
                p.ry = kRef ? ry : 0.f;
                p.S = S;
                p.T = Tt;
                p.Sy = kRef ? Sy : 1.f;
                p.careful = careful;
                __syncwarp();   // everybody has read the buffer
            }
            if (lane == 0) {
                const PolicyNumbers m = policy_numbers<kRef>(a, p, ok, xt, A, old, link, ref);
                PolicyHand &h = hand_s[n % kPpDepth];
                h.row.r = p.r;
                h.row.ry = p.ry;
                h.row.tok_c = m.cf * n1 * up;
                h.row.a = -h.row.tok_c * m.inv_s;
                h.row.w = a.beta * n1 * up * m.inv_s;
                h.row.mean = m.mean;
                h.xt = xt;
                h.yt = yt;
                h.tok = ok ? (int)tok : -1;
                h.careful = p.careful;
                policy_arrive(hand_bar + n % kPpDepth);
                if (rank == 0) {
                    if (!ok && a.status) atomicOr(a.status, DAT_STATUS_BAD_INDEX);
                    double kl = m.kl;
                    if (kRef) {
                        kl = (double)p.T / p.S - log((double)p.S / p.Sy);
                        const float o = kl < (double)kPoNear ? (p.r - p.ry) + m.mean : __int_as_float(0x7fc00000);
                        reinterpret_cast<PolicyNear *>(a.row_sums)[row] = PolicyNear{p.r, o, kl};
                    }
                    a.logp[row] = m.lp;
                    a.kl[row] = (float)kl;
                    sums[0] += (double)m.term;
                    sums[1] += kl;
                    sums[2] += (double)m.u;
                    sums[3] += m.clipped ? 1.0 : 0.0;
                    sums[4] += 1.0;
                    if (a.row_state) {
                        a.row_state[2 * row] = make_float4(p.r, m.inv_s, m.cf * n1, m.mean);
                        a.row_state[2 * row + 1] = make_float4(p.ry, 0.f, 0.f, 0.f);
                    }
                }
            }
        }
        if (lane == 0 && rank == 0)
            for (int k = 0; k < kPoSums; k++) a.chunk_sums[(int64_t)(blockIdx.x / ranks) * kPoSums + k] = sums[k];
    } else if (warp < kWarps) {   // ---- the summing half
        const auto sync = [] { asm volatile("bar.sync 1, %0;" ::"n"(NT) : "memory"); };
        PolicyWalk walk(a.mask, a.rows, ranks, false);
        // the next row's token and its logits are on their way while this row is worked on
        int64_t row = walk.next(), row1 = row >= 0 ? walk.next() : -1;
        const auto token = [&](int64_t r) { return r >= 0 ? a.tokens[r] : 0; };
        // as it lies in memory: a conversion here would wait for the load
        const auto logit = [&](const void *p, int64_t r, int64_t t) {
            return static_cast<const T *>(p)[r >= 0 ? r * V + (t >= 0 && t < V ? t : 0) : 0];
        };
        int64_t tok1 = token(row1);
        T xt = logit(a.x, row, token(row)), yt = kRef ? logit(a.y, row, token(row)) : xt;
        uint32_t n = 0;
        bool careful = false;
        for (; row >= 0; n++) {
            const T xt1 = logit(a.x, row1, tok1), yt1 = kRef ? logit(a.y, row1, tok1) : xt1;
            const int64_t row2 = row1 >= 0 ? walk.next() : -1, tok2 = token(row2);
            const PolicySpan<T> sp(row, V);
            const T *const x = static_cast<const T *>(a.x) + row * V, *const y = kRef ? static_cast<const T *>(a.y) + row * V : nullptr;
            // an element before or behind the pieces for the threads 0 .. head-1 and 8 .. 8+tail-1 of the first CTA
            const bool extra = rank == 0 && (tid < sp.head || (tid >= 8 && tid < 8 + sp.tail));
            const int te = tid < 8 ? tid : V - sp.tail + tid - 8;
            const T tx_raw = x[extra ? te : 0], ty_raw = kRef ? y[extra ? te : 0] : tx_raw;
            const int first = turn.slot;
            float r = Elem<T>::to_float(xt), ry = kRef ? Elem<T>::to_float(yt) : 0.f;
            PolicyAcc<kRef> acc;
            const auto sum = [&](auto care) {
                for (int j = 0; j < ring.chunks; j++, turn.next(ring.slots)) {
                    stalled |= !policy_wait(full + turn.slot, turn.phase, polls());
                    const int v = turn.slot * kChunk + tid, left = sp.vecs - (j * ranks + rank) * kChunk;
                    if (left >= kChunk) {
#pragma unroll
                        for (int q = 0; q < kPpVecs; q++) {
                            F2 px[kVec / 2], py[kVec / 2];
                            load(v + q * NT, r, ry, px, py);
                            acc.template add<decltype(care)::value>(px, py);
                        }
                    } else {
                        for (int q = 0; q < kPpVecs; q++)
                            if (tid + q * NT < left) {
                                F2 px[kVec / 2], py[kVec / 2];
                                load(v + q * NT, r, ry, px, py);
                                acc.template add<decltype(care)::value>(px, py);
                            }
                    }
                }
            };
            if (careful) sum(PolicyBool<true>());
            else sum(PolicyBool<false>());
            const float tx = Elem<T>::to_float(tx_raw), ty = Elem<T>::to_float(ty_raw);
            if (extra) acc.add1(tx, ty, r, ry);
            float S, Tt, Sy;
            const auto reduce = [&](float4 *slot) {
                const float ws = warp_sum(acc.both(acc.s));
                const float wt = kRef ? warp_sum(acc.both(acc.t)) : 0.f, wy = kRef ? warp_sum(acc.both(acc.sy)) : 0.f;
                if (lane == 0) slot[warp] = make_float4(ws, wt, wy, 0.f);
                sync();
                float4 q = slot[lane & (kWarps - 1)];
                if (lane >= kWarps) q = make_float4(0.f, 0.f, 0.f, 0.f);
                S = warp_sum(q.x);
                if (kRef) {
                    Tt = warp_sum(q.y);
                    Sy = warp_sum(q.z);
                } else {
                    Tt = 0.f;
                    Sy = 1.f;
                }
            };
            float4 *const slot = red + (n & 1 ? kWarps : 0);
            reduce(slot);
            if (!(S < kPpHuge && fabsf(Tt) < kPpHuge && Sy < kPpHuge)) {   // the same in all threads
                // the maxima in place of the token's logits; the row's slots are not freed before its gradient
                careful = kRef;   // and from here on: rows of one batch share their forbidden tokens
                const auto again = [&](auto f) {
                    int at = first;
                    for (int j = 0; j < ring.chunks; j++) {
                        for (int q = 0; q < kPpVecs; q++)
                            if ((j * ranks + rank) * kChunk + tid + q * NT < sp.vecs) {
                                F2 px[kVec / 2], py[kVec / 2];
                                load(at * kChunk + tid + q * NT, r, ry, px, py);
                                f(px, py);
                            }
                        if (++at == ring.slots) at = 0;
                    }
                };
                r = ry = 0.f;   // the logits themselves
                float m = -INFINITY, my = -INFINITY;
                again([&](const F2 (&px)[kVec / 2], const F2 (&py)[kVec / 2]) {
#pragma unroll
                    for (int i = 0; i < kVec / 2; i++) {
                        float u, w;
                        f2_get(px[i], u, w);
                        m = fmaxf(m, fmaxf(u, w));
                        if (kRef) {
                            f2_get(py[i], u, w);
                            my = fmaxf(my, fmaxf(u, w));
                        }
                    }
                });
                if (extra) {
                    m = fmaxf(m, tx);
                    my = fmaxf(my, ty);
                }
                m = warp_max(m);
                my = warp_max(my);
                sync();   // the sums have been read
                if (lane == 0) slot[warp] = make_float4(m, my, 0.f, 0.f);
                sync();
                const float4 q = slot[lane & (kWarps - 1)];
                r = warp_max(q.x);
                ry = kRef ? warp_max(q.y) : 0.f;
                // nothing but -inf in this CTA's share: any reference gives the sum 0
                r = r > -INFINITY ? r : 0.f;
                ry = ry > -INFINITY ? ry : 0.f;
                acc = PolicyAcc<kRef>();
                again([&](const F2 (&px)[kVec / 2], const F2 (&py)[kVec / 2]) { acc.template add<kRef>(px, py); });
                if (extra) acc.add1(tx, ty, r, ry);
                sync();
                reduce(slot);
            }
            if (tid == 0) {
                part_s[n % kPpDepth] = PolicyPart{r, ry, S, Tt, Sy, careful ? 1u : 0u};
                policy_arrive(part_bar + n % kPpDepth);
            }
            row = row1;
            row1 = row2;
            tok1 = tok2;
            xt = xt1;
            yt = yt1;
        }
        if (stalled)   // copies that may still be on their way, within a bound again
            for (int c = 0; c < ring.slots; c++) policy_wait(full + c, turn.phase, kPpPolls);
    } else {   // ---- the writing half
        const int wt = tid - NT;
        PolicyWalk walk(a.mask, a.rows, ranks, false);
        uint32_t n = 0;
        for (int64_t row = walk.next(); row >= 0; row = walk.next(), n++) {
            stalled |= !policy_wait(hand_bar + n % kPpDepth, n / kPpDepth & 1, polls());
            const PolicyHand h = hand_s[n % kPpDepth];
            const PolicyRow p = h.row;
            const PolicySpan<T> sp(row, V);
            T *const g = a.grad ? static_cast<T *>(a.grad) + row * V : nullptr;
            uint4 *const gv = reinterpret_cast<uint4 *>(g + sp.head);
            for (int j = 0; j < ring.chunks; j++, turn.next(ring.slots)) {
                // (full since the row was summed, which the hand-over above makes known here)
                const int v = turn.slot * kChunk + wt, to = (j * ranks + rank) * kChunk + wt;
                const auto store = [&](auto care, int q) {
                    F2 px[kVec / 2], py[kVec / 2];
                    float out[kVec];
                    load(v + q * NT, p.r, p.ry, px, py);
                    policy_grad_pairs<kRef, decltype(care)::value>(p, px, py, out);
                    gv[to + q * NT] = Elem<T>::pack(out);
                };
                if (g) {
                    if (to - wt + kChunk <= sp.vecs && !h.careful) {
#pragma unroll
                        for (int q = 0; q < kPpVecs; q++) store(PolicyBool<false>(), q);
                    } else {
                        for (int q = 0; q < kPpVecs; q++)
                            if (to + q * NT < sp.vecs) store(PolicyBool<kRef>(), q);
                    }
                }
                __syncwarp();
                if (lane == 0) policy_arrive(empty + turn.slot);
            }
            if (g) {
                if (rank == 0 && (wt < sp.head || (wt >= 8 && wt < 8 + sp.tail))) {
                    const int te = wt < 8 ? wt : V - sp.tail + wt - 8;
                    const float ty = kRef ? Elem<T>::to_float(static_cast<const T *>(a.y)[row * V + te]) : 0.f;
                    g[te] = Elem<T>::from_float(policy_grad_one<kRef>(p, Elem<T>::to_float(static_cast<const T *>(a.x)[row * V + te]), ty));
                }
                // the token's place once more, by the thread that wrote it
                const int at = h.tok - sp.head, piece = at / kVec;
                const bool inside = at >= 0 && piece < sp.vecs;
                const int mine = inside ? piece % NT : at < 0 ? h.tok : h.tok - (V - sp.tail) + 8;
                const int owner = inside ? piece / kChunk % ranks : 0;
                if (h.tok >= 0 && rank == owner && wt == mine)
                    g[h.tok] = Elem<T>::from_float(policy_grad_one<kRef>(p, h.xt, h.yt) + p.tok_c);
            }
        }
    }
    if (ranks > 1) {   // nobody leaves while a neighbour may still send to it
        __syncwarp();
        cluster_barrier();
    }
    if (stalled && lane == 0 && a.status) atomicOr(a.status, DAT_STATUS_STALLED);
    // the last CTA adds the CTAs' sums in their order
    __shared__ int last_s;
    pdl_wait();
    __syncthreads();
    if (tid == 0) {
        __threadfence();
        last_s = atomicAdd(&a.head->chunks_done, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last_s || warp > 0) return;
    __threadfence();
    double total[2] = {};
    for (int k = 0; k < kPoSums; k++) {
        double t = 0.0;
        for (int c = lane; c < (int)gridDim.x / ranks; c += 32) t += __ldcg(a.chunk_sums + (int64_t)c * kPoSums + k);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
        if (k < 2) total[k] = t;
        if (lane == 0) a.stats[k] = t;
    }
    if (lane == 0) *a.loss = (float)((total[0] + (double)a.beta * total[1]) * a.head->inv_n);
}

// The KL of the rows whose models are close, after policy_ring_kernel: a CTA a row, from memory (see the top).  The KL
// takes the place of what the ring kernel has put down, and the differences are added to the sums in the order of the CTAs.
// HBM (4.2 GB that the ring kernel has read before) and the fp32 units: 32768 rows of 32000 bf16 logits, all close, 0.88 ms; a
// handful of them 30 us (a row is 128 KB for one CTA).
constexpr int kPnThreads = 256, kPnWarps = kPnThreads / 32, kPnPerSm = 5;   // (3 and 4 per SM, with more loads ahead: 3 to 13 % slower)
template <typename T>
__global__ void __launch_bounds__(kPnThreads, kPnPerSm)
policy_near_kernel(PolicyArgs a) {
    constexpr int kVec = Elem<T>::kVec;
    __shared__ float red[2][3][kPnWarps];
    __shared__ unsigned close_s[kPnWarps];
    __shared__ int last_s;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    double more = 0.0;   // (thread 0)
    int par = 0;
    const auto gone_over = [&](int64_t row) {
        const float4 raw = __ldcg(a.row_sums + row);
        const float r = raw.x, o = raw.y;
        const T *x = static_cast<const T *>(a.x) + row * a.V, *y = static_cast<const T *>(a.y) + row * a.V;
        int head, nvec;
        policy_split(true, x, a.V, head, nvec);
        const uint4 *xv = reinterpret_cast<const uint4 *>(x + head), *yv = reinterpret_cast<const uint4 *>(y + head);
        PolicyNearAcc acc;
        for (int v = tid; v < nvec; v += kPnThreads) {
            F2 px[kVec / 2], py[kVec / 2];
            const uint4 ux = ld_stream16(xv + v), uy = ld_stream16(yv + v);
            policy_pairs(ux, px, 0.f, x);
            policy_pairs(uy, py, 0.f, x);
            acc.add(px, py, r, o);
        }
        for (int part = 0; part < 2; part++) {
            const int e0 = part ? head + nvec * kVec : 0, e1 = part ? a.V : head;
            for (int e = e0 + tid; e < e1; e += kPnThreads) acc.add1(Elem<T>::to_float(x[e]), Elem<T>::to_float(y[e]), r, o);
        }
        const float sums[3] = {warp_sum(acc.both(acc.s)), warp_sum(acc.both(acc.u_sum)), warp_sum(acc.both(acc.f_sum))};
        if (lane == 0) {
#pragma unroll
            for (int k = 0; k < 3; k++) red[par][k][warp] = sums[k];
        }
        __syncthreads();
        if (tid == 0) {
            double t[3] = {};
            for (int k = 0; k < 3; k++)
                for (int w = 0; w < kPnWarps; w++) t[k] += red[par][k][w];
            const double kl = policy_near_kl(t[0], t[1], t[2]);
            a.kl[row] = (float)kl;
            more += kl - __hiloint2double(__float_as_int(raw.w), __float_as_int(raw.z));
        }
        par ^= 1;   // (the next row's barrier stands between this row's reads and the writes of the row after it)
    };
    pdl_wait();
    // 256 rows at a time: which of them are close
    for (int64_t first = blockIdx.x; first < a.rows; first += (int64_t)kPnThreads * gridDim.x) {
        const int64_t mine = first + (int64_t)tid * gridDim.x;
        bool is_close = mine < a.rows && !(a.mask && !a.mask[mine]);
        if (is_close) {
            const float o = __ldcg(&a.row_sums[mine].y);
            is_close = o == o;
        }
        const unsigned b = __ballot_sync(0xffffffffu, is_close);
        __syncthreads();   // the bits of the rows before have been read
        if (lane == 0) close_s[warp] = b;
        __syncthreads();
        for (int w = 0; w < kPnWarps; w++)
            for (unsigned bits = close_s[w]; bits; bits &= bits - 1)
                gone_over(first + (int64_t)(32 * w + __ffs(bits) - 1) * gridDim.x);
    }
    if (tid == 0) {
        a.chunk_sums[blockIdx.x] = more;   // whose first use is over
        __threadfence();
        last_s = atomicAdd(a.done, 1) == (int)gridDim.x - 1;
    }
    __syncthreads();
    if (!last_s || warp > 0) return;
    __threadfence();
    double t = 0.0;
    for (int c = lane; c < (int)gridDim.x; c += 32) t += __ldcg(a.chunk_sums + c);
#pragma unroll
    for (int q = 16; q > 0; q >>= 1) t += __shfl_xor_sync(0xffffffffu, t, q);
    if (lane == 0 && t != 0.0) {
        const double kl = __ldcg(a.stats + 1) + t;
        a.stats[1] = kl;
        *a.loss = (float)((__ldcg(a.stats) + (double)a.beta * kl) * a.head->inv_n);
    }
}

struct PolicyBackwardArgs {
    const void *x, *y;
    const int64_t *tokens;
    const unsigned char *mask;
    const float4 *row_state;
    const PolicyHead *head;
    const float *grad_loss;     // [1]
    void *grad;                 // [rows, V]
    float *grad_link;           // [rows] or null
    float beta;
    int64_t rows;
    int V;
    bool vec, written;          // written: grad holds the gradient for head->scale
};

template <typename T, bool kRef>
__global__ void __launch_bounds__(kPoThreads)
policy_bwd_kernel(PolicyBackwardArgs a) {
    const float up = *a.grad_loss;
    if (a.grad_link)
        for (int64_t r = (int64_t)blockIdx.x * kPoThreads + threadIdx.x; r < a.rows; r += (int64_t)gridDim.x * kPoThreads)
            a.grad_link[r] = a.mask && !a.mask[r] ? 0.f : a.row_state[2 * r].z * up;
    if (!a.grad || (a.written && up == a.head->scale)) return;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        T *g = static_cast<T *>(a.grad) + row * a.V;
        if (a.mask && !a.mask[row]) {
            policy_zero_row(g, a.vec, a.V);
            continue;
        }
        const T *x = static_cast<const T *>(a.x) + row * a.V, *y = kRef ? static_cast<const T *>(a.y) + row * a.V : nullptr;
        const float4 st = a.row_state[2 * row];
        const float c = st.z * up;
        const PolicyRow p{st.x, a.row_state[2 * row + 1].x, -c * st.y, (float)((double)a.beta * a.head->inv_n * up * st.y),
                          st.w, c};
        policy_grad_row<T, kRef>(x, y, g, a.vec, a.V, p, a.tokens[row]);
    }
}

constexpr int kPoMaxCtas = 1024;   // persistent CTAs of a launch
static int64_t policy_chunks(int64_t rows) { return (rows + kPoChunk - 1) / kPoChunk; }

struct PolicyWorkspace {
    size_t done, sums, chunk, total;
    explicit PolicyWorkspace(int64_t rows) {
        const auto up = [](size_t n) { return (n + 15) / 16 * 16; };
        done = up(sizeof(PolicyHead));
        sums = up(done + (size_t)policy_chunks(rows) * sizeof(int));
        chunk = up(sums + (size_t)rows * sizeof(float4));
        // one line of sums per chunk of rows, or per persistent CTA (at most one per row)
        const int64_t lines = rows < kPoMaxCtas ? rows : kPoMaxCtas;
        total = up(chunk + (size_t)(policy_chunks(rows) > lines ? policy_chunks(rows) : lines) * kPoSums * sizeof(double));
    }
};

static bool aligned16(const void *a, const void *b, const void *c) {
    return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c)) & 15) == 0;
}

// The ring of a CTA with nt threads in each half and chunks of nt * vecs pieces, `per_sm` of them on an SM and `ranks`
// to a row; false: a row does not fit.
static bool policy_ring(int nt, int vecs, int per_sm, int ranks, int V, int size, bool ref, const DeviceInfo &di, PolicyRing &ring,
                        int &smem) {
    const auto up = [](int n) { return (n + 127) / 128 * 128; };
    const int64_t pieces = (int64_t)V * size / 16;   // 16-byte pieces inside a row
    const int chunk = nt * vecs, slot = chunk * 16 * (ref ? 2 : 1);
    if (pieces < 1 || pieces > (1 << 20)) return false;
    ring.ranks = ranks;
    ring.chunks = (int)((pieces + (int64_t)chunk * ranks - 1) / (chunk * ranks));
    const int avail = (di.max_smem_optin + 1024) / per_sm - 1024 - 1024;   // what the kernel declares itself is below 1024
    const int fixed = up(kPpZeros + 2 * kPpDepth * ring.chunks * 8) + up(2 * (nt / 32) * 16);
    ring.slots = (avail - fixed) / slot;
    if (ring.slots > kPpDepth * ring.chunks) ring.slots = kPpDepth * ring.chunks;
    if (ring.slots < ring.chunks) return false;
    ring.zeros = 0;
    ring.bars = kPpZeros;
    ring.red = up(ring.bars + 2 * ring.slots * 8);
    ring.x = up(ring.red + 2 * (nt / 32) * 16);
    ring.y = ring.x + ring.slots * chunk * 16;
    smem = ref ? ring.y + ring.slots * chunk * 16 : ring.y;
    return true;
}

template <typename T, bool kRef, int NT, int kPpVecs>
static int policy_ring_launch(const PolicyArgs &a, const PolicyRing &ring, int smem, int per_sm, const DeviceInfo &di,
                              cudaStream_t st, const char *who) {
    int64_t n = (int64_t)di.sm_count * per_sm / ring.ranks;   // clusters
    if (n > a.rows) n = a.rows;
    if (n > kPoMaxCtas) n = kPoMaxCtas;
    if (cudaFuncSetAttribute(policy_ring_kernel<T, kRef, NT, kPpVecs>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
        return check_launch(who);
    launch_after(policy_ring_kernel<T, kRef, NT, kPpVecs>, (unsigned)n * ring.ranks, 2 * NT + 96, smem, st, ring.ranks, a, ring);
    if (kRef) {
        int64_t grid = (int64_t)di.sm_count * kPnPerSm;
        if (grid > a.rows) grid = a.rows;
        if (grid > kPoMaxCtas) grid = kPoMaxCtas;
        if (int rc = check_launch(who)) return rc;
        launch_after(policy_near_kernel<T>, (unsigned)grid, kPnThreads, 0, st, 1, a);
    }
    return check_launch(who);
}

template <typename T>
static int policy_fwd_t(const PolicyArgs &a, const DeviceInfo &di, cudaStream_t st, const char *who) {
    // Rows of 8 KB and up: the ring.  On both sides of that, in a graph, bf16, 2000 / 4000 / 5000 / 8000 logits: 32768 rows
    // 133 / 174 / 199 / 254 us with the ring against 203 / 240 / 264 / 311 with a CTA per row, with the reference's logits
    // 209 / 270 / 319 / 399 against 305 / 377 / 414 / 496; 1280 rows 25 / 27 / 29 / 31 against 25 / 27 / 27 / 29, with the
    // reference's 37 / 39 / 41 / 47 against 29 / 31 / 33 / 39.  (The number of rows would be the better rule.)
    // With 128 threads in each half where three CTAs with two rows each fit an SM, else
    // with 256 and as few CTAs to a row as it takes for more than one row in a ring.  Chunks are as large as that allows:
    // a chunk of four pieces a thread keeps more arithmetic in flight than one of two (32x1024x32000 with the full KL
    // 1308 against 1390 us, 1623 with one), a ring without a spare chunk lets the halves wait for each other.
    // Fewer rows than SMs: more CTAs to a row, as long as each has a chunk of it.
    if (a.vec && (int64_t)a.V * sizeof(T) >= 8192) {
        PolicyRing ring{}, more{};
        int smem = 0, smem2 = 0;
        const bool ref = a.y != nullptr;
        const auto spread = [&](int nt, int vecs, int per_sm) {
            while (ring.ranks < kPpRanks && a.rows * ring.ranks * 2 <= di.sm_count && ring.chunks > 1 &&
                   policy_ring(nt, vecs, per_sm, ring.ranks * 2, a.V, sizeof(T), ref, di, more, smem2)) {
                ring = more;
                smem = smem2;
            }
        };
        if (policy_ring(128, 2, 3, 1, a.V, sizeof(T), ref, di, ring, smem) && ring.slots >= 2 * ring.chunks) {
            spread(128, 2, 3);
            return ref ? policy_ring_launch<T, true, 128, 2>(a, ring, smem, 3, di, st, who)
                       : policy_ring_launch<T, false, 128, 2>(a, ring, smem, 3, di, st, who);
        }
        for (int ranks = 1; ranks <= kPpRanks; ranks *= 2) {
            if (policy_ring(256, 4, 1, ranks, a.V, sizeof(T), ref, di, ring, smem) && ring.slots > ring.chunks) {
                spread(256, 4, 1);
                return ref ? policy_ring_launch<T, true, 256, 4>(a, ring, smem, 1, di, st, who)
                           : policy_ring_launch<T, false, 256, 4>(a, ring, smem, 1, di, st, who);
            }
            if (policy_ring(256, 2, 1, ranks, a.V, sizeof(T), ref, di, ring, smem) && ring.slots > ring.chunks) {
                spread(256, 2, 1);
                return ref ? policy_ring_launch<T, true, 256, 2>(a, ring, smem, 1, di, st, who)
                           : policy_ring_launch<T, false, 256, 2>(a, ring, smem, 1, di, st, who);
            }
        }
    }
    if (a.y)
        policy_fwd_kernel<T, true><<<(unsigned)a.rows, kPoThreads, 0, st>>>(a);
    else
        policy_fwd_kernel<T, false><<<(unsigned)a.rows, kPoThreads, 0, st>>>(a);
    return check_launch(who);
}

template <typename T>
static int policy_bwd_t(const PolicyBackwardArgs &a, const DeviceInfo &di, cudaStream_t st, const char *who) {
    int64_t grid = (int64_t)di.sm_count * 6;
    if (grid > a.rows) grid = a.rows;
    if (a.y)
        policy_bwd_kernel<T, true><<<(unsigned)grid, kPoThreads, 0, st>>>(a);
    else
        policy_bwd_kernel<T, false><<<(unsigned)grid, kPoThreads, 0, st>>>(a);
    return check_launch(who);
}

}  // namespace dat

extern "C" {

size_t dat_policy_loss_workspace_bytes(int bsz, int prelen) {
    if (bsz < 0 || prelen < 0) return 0;
    return dat::PolicyWorkspace((int64_t)bsz * prelen).total;
}

int dat_policy_loss(const void *word_ins_out, const void *ref_logits, int dtype, const int64_t *tokens,
                    const float *old_logp, const float *advantage, int64_t adv_stride_b, int64_t adv_stride_l,
                    const float *link_logp, const float *ref_logp, const unsigned char *mask, float kl_coef,
                    float clip_low, float clip_high, const float *grad_scale_ptr, float grad_scale, float *loss,
                    double *stats, float *logp, float *kl, float *row_state, void *grad_logits, void *workspace,
                    int32_t *status, int bsz, int prelen, int vocab, void *stream) {
    using namespace dat;
    const char *who = "dat_policy_loss";
    DAT_REQUIRE(bsz >= 0 && prelen >= 0 && vocab >= 1, DAT_ERR_BAD_ARG, "%s: bad sizes bsz=%d prelen=%d vocab=%d", who, bsz,
                prelen, vocab);
    DAT_REQUIRE(loss && stats && workspace, DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DAT_REQUIRE(!(ref_logits && ref_logp), DAT_ERR_BAD_ARG, "%s: ref_logits and ref_logp exclude each other", who);
    DAT_REQUIRE(clip_low >= 0.f && clip_high >= 0.f, DAT_ERR_BAD_ARG, "%s: negative clip range", who);
    DAT_REQUIRE(vocab <= 0x3fffffff, DAT_ERR_UNSUPPORTED, "%s: vocab = %d exceeds 2^30-1", who, vocab);
    const int64_t rows = (int64_t)bsz * prelen;
    DAT_REQUIRE(rows <= 0x7fffffff, DAT_ERR_UNSUPPORTED, "%s: bsz*prelen = %lld exceeds 2^31-1", who, (long long)rows);
    DAT_REQUIRE(dtype == DAT_F32 || dtype == DAT_F16 || dtype == DAT_BF16, DAT_ERR_UNSUPPORTED,
                "%s: unsupported dtype %d (fp32, fp16, bf16 only)", who, dtype);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (rows == 0) {
        cudaMemsetAsync(loss, 0, sizeof(float), st);
        cudaMemsetAsync(stats, 0, kPoSums * sizeof(double), st);
        return check_launch(who);
    }
    DAT_REQUIRE(word_ins_out && tokens && old_logp && advantage && logp && kl, DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    const PolicyWorkspace lay(rows);
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    PolicyArgs a{};
    a.x = word_ins_out;
    a.y = ref_logits;
    a.tokens = tokens;
    a.old_logp = old_logp;
    a.advantage = advantage;
    a.adv_b = adv_stride_b;
    a.adv_l = adv_stride_l;
    a.link_logp = link_logp;
    a.ref_logp = ref_logp;
    a.mask = mask;
    a.beta = kl_coef;
    a.clip_low = clip_low;
    a.clip_high = clip_high;
    a.loss = loss;
    a.stats = stats;
    a.logp = logp;
    a.kl = kl;
    a.row_state = reinterpret_cast<float4 *>(row_state);
    a.grad = grad_logits;
    a.head = reinterpret_cast<PolicyHead *>(ws);
    a.done = reinterpret_cast<int *>(ws + lay.done);
    a.row_sums = reinterpret_cast<float4 *>(ws + lay.sums);
    a.chunk_sums = reinterpret_cast<double *>(ws + lay.chunk);
    a.status = status;
    a.rows = rows;
    a.L = prelen;
    a.V = vocab;
    a.vec = aligned16(word_ins_out, ref_logits, grad_logits);
    policy_prep_kernel<<<1, 1024, 0, st>>>(mask, rows, a.head, a.done, (int)policy_chunks(rows), grad_scale_ptr, grad_scale);
    if (int rc = check_launch(who)) return rc;
    switch (dtype) {
        case DAT_F32: return policy_fwd_t<float>(a, di, st, who);
        case DAT_F16: return policy_fwd_t<__half>(a, di, st, who);
        default: return policy_fwd_t<__nv_bfloat16>(a, di, st, who);
    }
}

unsigned long long dat_stream_capture_id(void *stream) {
    cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (cudaStreamGetCaptureInfo(static_cast<cudaStream_t>(stream), &status, &id) != cudaSuccess) {
        cudaGetLastError();
        return 0;
    }
    return status == cudaStreamCaptureStatusActive ? id : 0;
}

int dat_policy_loss_backward(const void *word_ins_out, const void *ref_logits, int dtype, const int64_t *tokens,
                             const unsigned char *mask, float kl_coef, const float *row_state, const void *workspace,
                             const float *grad_loss, int grad_written, void *grad_logits, float *grad_link, int bsz,
                             int prelen, int vocab, void *stream) {
    using namespace dat;
    const char *who = "dat_policy_loss_backward";
    DAT_REQUIRE(bsz >= 0 && prelen >= 0 && vocab >= 1, DAT_ERR_BAD_ARG, "%s: bad sizes bsz=%d prelen=%d vocab=%d", who, bsz,
                prelen, vocab);
    const int64_t rows = (int64_t)bsz * prelen;
    if (rows == 0 || !(grad_logits || grad_link)) return DAT_OK;
    DAT_REQUIRE(word_ins_out && tokens && row_state && workspace && grad_loss, DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DAT_REQUIRE(dtype == DAT_F32 || dtype == DAT_F16 || dtype == DAT_BF16, DAT_ERR_UNSUPPORTED,
                "%s: unsupported dtype %d (fp32, fp16, bf16 only)", who, dtype);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    const PolicyBackwardArgs a{word_ins_out, ref_logits, tokens, mask, reinterpret_cast<const float4 *>(row_state),
                               static_cast<const PolicyHead *>(workspace), grad_loss, grad_logits, grad_link, kl_coef, rows,
                               vocab, aligned16(word_ins_out, ref_logits, grad_logits), grad_written != 0};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (dtype) {
        case DAT_F32: return policy_bwd_t<float>(a, di, st, who);
        case DAT_F16: return policy_bwd_t<__half>(a, di, st, who);
        default: return policy_bwd_t<__nv_bfloat16>(a, di, st, who);
    }
}

}  // extern "C"

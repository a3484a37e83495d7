// Band links from per-head scores with a learned relative position bias, forward and backward, for sm_100a.
//
// The scores of links.cu with table[bucket[j-i-1], h] added to content[b,i,j,h]: the bias belongs to the
// distance between two vertices, distances share a row of the table by buckets, and the table is learned.
// With z = content + bias and the other names of links.cu, the gradient of a score is
//     dc[b,i,j,h] = G p - exp(z - lse_h) S_h
// as there, and the table's is the sum of dc over all transitions of a bucket:
//     dT[k,h] = sum over (b,i,d) with bucket[d] = k of dc[b,i,i+1+d,h].
//
// HBM-bound: the scores of the valid transitions are read once forward and once backward, the band is written
// forward, the dense gradient backward.  A CTA owns a vertex at a time and keeps its scores in registers, a
// thread the same distances and heads (16 bytes: four heads of one distance) for every vertex it meets, so that
// the bias is expanded by distance once per CTA (shared memory, log2 units) and the table's gradient gathers in
// places of its own; the partial sums of the CTAs are added in a fixed order (no atomics: results repeat bit for
// bit).  One exponential per score and direction:
//   forward   e = exp(z - r_h), r_h the score of the nearest successor in place of the maximum over all of them:
//             the sum is at least 1, and a vertex where it overflows (a score 60 above r_h) or whose nearest
//             successor is masked takes the maximum after all.  links = log sum_h e_h exp(g_h) / S_h.
//   backward  soft = exp(z - lse_h), q_h = soft exp(g_h), p_h = q_h / sum q.
// Where sum q is below 2^-80 (a link below -55) it is taken again relative to its largest term, so that what
// the 32-bit exponent flushes stays below 2^-40 of what it is added to.
// Head counts of 4, 8, 16, 32 and up to 4096 score vectors per vertex; others take the kernels of links.cu (one
// CTA per vertex, scores in shared memory) and a pass over the gradient's diagonals.
#include "links_common.cuh"

namespace dat {

constexpr int kLbThreads = 128;
constexpr int kLbSplits = 16;           // partial sums per distance and head that the last kernel adds
constexpr float kLbTiny = 0x1p-80f;
constexpr float kLbHuge = 0x1p+86f;
constexpr int kLbMaxVec = 4096;         // score vectors per vertex: 512 threads with eight each

__device__ __forceinline__ int lb_row_of_slot(int q, int L) { return (q & 1) ? L - 1 - (q >> 1) : (q >> 1); }

// bias by distance in log2 units into shared memory; -inf for a bucket outside the table
template <int NT>
__device__ __forceinline__ void lb_expand(const LinksBias &lb, float *bl, int H, int K) {
    bool bad = false;
    for (int x = threadIdx.x; x < K * H; x += NT) bl[x] = links_bias1(lb, x / H, x % H, H, bad) * kLog2e;
    if (bad && lb.status) atomicOr(lb.status, DAT_STATUS_BAD_INDEX);
}

__device__ __forceinline__ float4 lb_ninf4() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }

// sum (or maximum) of v over the CTA's threads of the same head group, in every thread
template <int G, int NT, bool kMax>
__device__ __forceinline__ void lb_reduce(float (&v)[4], float *red, bool synced_before) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & (G - 1);
#pragma unroll
    for (int o = G; o < 32; o <<= 1) {
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const float w = __shfl_xor_sync(0xffffffffu, v[k], o);
            v[k] = kMax ? fmaxf(v[k], w) : v[k] + w;
        }
    }
    float4 *r4 = reinterpret_cast<float4 *>(red);
    if (!synced_before) __syncthreads();
    if (lane < G) r4[warp * G + g] = make_float4(v[0], v[1], v[2], v[3]);
}
template <int G, int NT, bool kMax>
__device__ __forceinline__ void lb_collect(float (&v)[4], const float *red) {
    const int g = threadIdx.x & (G - 1);
    const float4 *r4 = reinterpret_cast<const float4 *>(red);
    float4 a = r4[g];
#pragma unroll
    for (int w = 1; w < NT / 32; w++) {
        const float4 b = r4[w * G + g];
        a = kMax ? make_float4(fmaxf(a.x, b.x), fmaxf(a.y, b.y), fmaxf(a.z, b.z), fmaxf(a.w, b.w))
                 : make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
    }
    v[0] = a.x;
    v[1] = a.y;
    v[2] = a.z;
    v[3] = a.w;
}

template <int G>
__device__ __forceinline__ float lb_over_heads(float v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
template <int G>
__device__ __forceinline__ float lb_max_over_heads(float v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}

// G = H / 4 vectors per distance; thread t holds the vectors t, t + NT, ... of a vertex's row (U of them)
template <int G, int NT, int U>
__global__ void __launch_bounds__(NT)
lb_fwd_kernel(const float *__restrict__ content, const float *__restrict__ log_gates, LinksMask mk, LinksBias lb,
              float *__restrict__ links, float *__restrict__ head_lse, int B, int L, int K) {
    constexpr int H = 4 * G;
    extern __shared__ __align__(16) float lbsm[];
    float *bl = lbsm;                                  // [K * H]
    float *red = lbsm + (size_t)K * H;                 // [2][NT / 32][H]
    const int tid = threadIdx.x, lane = tid & 31, g = lane & (G - 1);
    lb_expand<NT>(lb, bl, H, K);
    __syncthreads();
    const float4 *bl4 = reinterpret_cast<const float4 *>(bl);
    const int64_t rows = (int64_t)B * L;
    int par = 0;
    for (int64_t slot = blockIdx.x; slot < rows; slot += gridDim.x, par ^= 1) {
        const int64_t b = slot / L;
        const int i = lb_row_of_slot((int)(slot - b * L), L);
        const int64_t row = b * L + i;
        const int jhi = links_jhi(i, L, K, mk, row);
        const int nj = jhi - i > 0 ? jhi - i : 0, nvec = nj * G;
        const unsigned char *np = mk.nonpad ? mk.nonpad + b * L + i + 1 : nullptr;
        const float4 *src = reinterpret_cast<const float4 *>(content + (row * L + i + 1) * (int64_t)H);
        if (nj == 0) {   // the whole CTA: no barrier, so the next vertex takes the same half of red
            for (int d = tid; d < K; d += NT) links[row * (int64_t)K + d] = -INFINITY;
            if (head_lse && tid < H) head_lse[row * H + tid] = -INFINITY;
            par ^= 1;
            continue;
        }
        float4 e4[U];
        unsigned live = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT;
            const bool ok = v < nvec && !(np && !np[v / G]);
            live |= ok ? 1u << u : 0u;
            e4[u] = ok ? __ldg(src + v) : lb_ninf4();
        }
        // r_h in log2 units
        float r[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        if (!(np && !np[0])) {
            const float4 c0 = __ldg(src + g), b0 = bl4[g];
            r[0] = fmaf(c0.x, kLog2e, b0.x);
            r[1] = fmaf(c0.y, kLog2e, b0.y);
            r[2] = fmaf(c0.z, kLog2e, b0.z);
            r[3] = fmaf(c0.w, kLog2e, b0.w);
        }
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        const bool no_r = !(fabsf(r[0]) < INFINITY && fabsf(r[1]) < INFINITY && fabsf(r[2]) < INFINITY && fabsf(r[3]) < INFINITY);
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (u * NT + (tid & ~31) >= nvec) {     // nothing of this warp
                e4[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                continue;
            }
            float4 t = bl4[min(tid + u * NT, K * G - 1)];
            fadd2_rn(t.x, t.y, t.x, t.y, -r[0], -r[1]);
            fadd2_rn(t.z, t.w, t.z, t.w, -r[2], -r[3]);
            ffma2_rn(t.x, t.y, e4[u].x, e4[u].y, kLog2e, kLog2e);
            ffma2_rn(t.z, t.w, e4[u].z, e4[u].w, kLog2e, kLog2e);
            const bool ok = live >> u & 1;
            e4[u] = ok ? make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w)) : make_float4(0.f, 0.f, 0.f, 0.f);
            fadd2_rn(sum[0], sum[1], sum[0], sum[1], e4[u].x, e4[u].y);
            fadd2_rn(sum[2], sum[3], sum[2], sum[3], e4[u].z, e4[u].w);
        }
        const bool bad = no_r || !(fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3])) < kLbHuge) ||
                         !(sum[0] + sum[1] + sum[2] + sum[3] < INFINITY);
        float *rd = red + par * (NT / 32) * H;
        lb_reduce<G, NT, false>(sum, rd, true);
        if (__syncthreads_or(bad)) {
            // the exact maximum of each head takes the place of r_h
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = tid + u * NT;
                if (live >> u & 1) {
                    const float4 c = __ldg(src + v), t = bl4[v];
                    m[0] = fmaxf(m[0], fmaf(c.x, kLog2e, t.x));
                    m[1] = fmaxf(m[1], fmaf(c.y, kLog2e, t.y));
                    m[2] = fmaxf(m[2], fmaf(c.z, kLog2e, t.z));
                    m[3] = fmaxf(m[3], fmaf(c.w, kLog2e, t.w));
                }
            }
            lb_reduce<G, NT, true>(m, rd, true);   // the sums that the slot held are not wanted
            __syncthreads();
            lb_collect<G, NT, true>(m, rd);
            sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) r[k] = m[k] > -INFINITY ? m[k] : 0.f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = tid + u * NT;
                e4[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live >> u & 1) {
                    const float4 c = __ldg(src + v), t = bl4[v];
                    e4[u] = make_float4(ex2(fmaf(c.x, kLog2e, t.x - r[0])), ex2(fmaf(c.y, kLog2e, t.y - r[1])),
                                        ex2(fmaf(c.z, kLog2e, t.z - r[2])), ex2(fmaf(c.w, kLog2e, t.w - r[3])));
                    sum[0] += e4[u].x;
                    sum[1] += e4[u].y;
                    sum[2] += e4[u].z;
                    sum[3] += e4[u].w;
                }
            }
            lb_reduce<G, NT, false>(sum, rd, false);
            __syncthreads();
        }
        lb_collect<G, NT, false>(sum, rd);
        // f_h = exp(g_h) / S_h; a head without a finite score takes no part
        float f[4];
        const float4 gate = __ldg(reinterpret_cast<const float4 *>(log_gates + row * H) + g);
        const float gt[4] = {gate.x, gate.y, gate.z, gate.w};
#pragma unroll
        for (int k = 0; k < 4; k++) {
            const bool some = sum[k] > 0.f && sum[k] < INFINITY;
            f[k] = some ? ex2(gt[k] * kLog2e) / sum[k] : 0.f;
            if (head_lse && tid < G) head_lse[row * H + 4 * g + k] = some ? (r[k] + lg2(sum[k])) * kLn2 : -INFINITY;
        }
        float *out = links + row * (int64_t)K;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT, d = v / G;
            if (u * NT + (tid & ~31) >= K * G) break;
            const bool ok = live >> u & 1;
            float q = lb_over_heads<G>(fmaf(e4[u].x, f[0], e4[u].y * f[1]) + fmaf(e4[u].z, f[2], e4[u].w * f[3]));
            float link = lg2(q) * kLn2;
            if (__any_sync(0xffffffffu, ok && q < kLbTiny)) {
                float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                if (ok) {
                    const float4 c = __ldg(src + v), bb = bl4[v];
                    const float cc[4] = {c.x, c.y, c.z, c.w}, bk[4] = {bb.x, bb.y, bb.z, bb.w};
#pragma unroll
                    for (int k = 0; k < 4; k++)   // log2 of e f without the exponential's flush
                        if (gt[k] > -INFINITY && sum[k] > 0.f && sum[k] < INFINITY)
                            t[k] = fmaf(cc[k], kLog2e, bk[k] - r[k]) + (gt[k] * kLog2e - lg2(sum[k]));
                }
                const float m = lb_max_over_heads<G>(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
                const float mm = m > -INFINITY ? m : 0.f;
                q = lb_over_heads<G>(ex2(t[0] - mm) + ex2(t[1] - mm) + ex2(t[2] - mm) + ex2(t[3] - mm));
                link = m > -INFINITY ? (m + lg2(q)) * kLn2 : -INFINITY;
            }
            if (g == 0 && d < K) out[d] = ok ? link : -INFINITY;
        }
    }
}

template <int G, int NT, int U>
__global__ void __launch_bounds__(NT)
lb_bwd_kernel(const float *__restrict__ grad_links, const float *__restrict__ content,
              const float *__restrict__ log_gates, const float *__restrict__ head_lse, LinksMask mk, LinksBias lb,
              float *__restrict__ grad_content, float *__restrict__ grad_log_gates, float *__restrict__ part, int B, int L,
              int K) {
    constexpr int H = 4 * G;
    extern __shared__ __align__(16) float lbsm[];
    float *bl = lbsm;                                       // [K * H]
    float *acc = lbsm + (size_t)K * H;                      // [K * H]: this CTA's share of the gradient by distance
    float *red = acc + (part ? (size_t)K * H : 0);          // [2][NT / 32][H]
    const int tid = threadIdx.x, lane = tid & 31, g = lane & (G - 1);
    lb_expand<NT>(lb, bl, H, K);
    if (part)
        for (int x = tid; x < K * H; x += NT) acc[x] = 0.f;
    __syncthreads();
    const float4 *bl4 = reinterpret_cast<const float4 *>(bl);
    float4 *acc4 = reinterpret_cast<float4 *>(acc);
    const int64_t rows = (int64_t)B * L;
    int par = 0;
    for (int64_t slot = blockIdx.x; slot < rows; slot += gridDim.x, par ^= 1) {
        const int64_t b = slot / L;
        const int i = lb_row_of_slot((int)(slot - b * L), L);
        const int64_t row = b * L + i;
        const int jhi = links_jhi(i, L, K, mk, row);
        const int nj = jhi - i > 0 ? jhi - i : 0, nvec = nj * G;
        const unsigned char *np = mk.nonpad ? mk.nonpad + b * L + i + 1 : nullptr;
        const float4 *src = reinterpret_cast<const float4 *>(content + (row * L + i + 1) * (int64_t)H);
        const float *gl = grad_links + row * (int64_t)K;
        float4 s4[U], p4[U];
        float gd[U];
        unsigned live = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT;
            const bool ok = v < nvec && !(np && !np[v / G]);
            live |= ok ? 1u << u : 0u;
            s4[u] = ok ? __ldg(src + v) : lb_ninf4();
            gd[u] = ok ? __ldg(gl + v / G) : 0.f;
        }
        const float4 lse = __ldg(reinterpret_cast<const float4 *>(head_lse + row * H) + g);
        const float4 gate = __ldg(reinterpret_cast<const float4 *>(log_gates + row * H) + g);
        // a head that takes no part (lse = -inf): soft = exp(-inf) = 0
        const float ls[4] = {lse.x > -INFINITY ? lse.x * kLog2e : INFINITY, lse.y > -INFINITY ? lse.y * kLog2e : INFINITY,
                             lse.z > -INFINITY ? lse.z * kLog2e : INFINITY, lse.w > -INFINITY ? lse.w * kLog2e : INFINITY};
        const float g2[4] = {gate.x * kLog2e, gate.y * kLog2e, gate.z * kLog2e, gate.w * kLog2e};
        const float eg[4] = {ex2(g2[0]), ex2(g2[1]), ex2(g2[2]), ex2(g2[3])};
        float S[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; u++) {
            if (u * NT + (tid & ~31) >= nvec) continue;   // nothing of this warp
            float4 t = bl4[min(tid + u * NT, K * G - 1)];
            fadd2_rn(t.x, t.y, t.x, t.y, -ls[0], -ls[1]);
            fadd2_rn(t.z, t.w, t.z, t.w, -ls[2], -ls[3]);
            ffma2_rn(t.x, t.y, s4[u].x, s4[u].y, kLog2e, kLog2e);
            ffma2_rn(t.z, t.w, s4[u].z, s4[u].w, kLog2e, kLog2e);
            if (!(live >> u & 1)) t = lb_ninf4();   // whatever the table holds
            s4[u] = make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w));
            float4 q = make_float4(s4[u].x * eg[0], s4[u].y * eg[1], s4[u].z * eg[2], s4[u].w * eg[3]);
            const float tot = lb_over_heads<G>((q.x + q.y) + (q.z + q.w));
            float w = tot >= kLbTiny ? __fdividef(gd[u], tot) : 0.f;
            if (__any_sync(0xffffffffu, gd[u] != 0.f && tot < kLbTiny)) {
                const float a[4] = {t.x + g2[0], t.y + g2[1], t.z + g2[2], t.w + g2[3]};
                const float m = lb_max_over_heads<G>(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
                if (tot < kLbTiny) {   // the same lanes of a distance
                    const float mm = m > -INFINITY ? m : 0.f;
                    q = make_float4(ex2(a[0] - mm), ex2(a[1] - mm), ex2(a[2] - mm), ex2(a[3] - mm));
                }
                const float tot2 = lb_over_heads<G>((q.x + q.y) + (q.z + q.w));
                w = tot2 > 0.f ? gd[u] / tot2 : 0.f;
            }
            p4[u] = make_float4(q.x * w, q.y * w, q.z * w, q.w * w);
            fadd2_rn(S[0], S[1], S[0], S[1], p4[u].x, p4[u].y);
            fadd2_rn(S[2], S[3], S[2], S[3], p4[u].z, p4[u].w);
        }
        float *rd = red + par * (NT / 32) * H;
        lb_reduce<G, NT, false>(S, rd, true);
        // the places of the dense row that no valid successor has
        float4 *rowv = reinterpret_cast<float4 *>(grad_content + row * (int64_t)L * H);
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int v = tid; v < (i + 1) * G; v += NT) rowv[v] = zero;
        for (int v = (i + 1) * G + nvec + tid; v < L * G; v += NT) rowv[v] = zero;
        __syncthreads();
        lb_collect<G, NT, false>(S, rd);
        if (tid < G)
            reinterpret_cast<float4 *>(grad_log_gates + row * H)[g] = make_float4(S[0], S[1], S[2], S[3]);
        float4 *dst = rowv + (i + 1) * G;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT;
            if (v >= nvec) break;
            float4 o = p4[u];
            ffma2_rn(o.x, o.y, s4[u].x, s4[u].y, -S[0], -S[1]);
            ffma2_rn(o.z, o.w, s4[u].z, s4[u].w, -S[2], -S[3]);
            dst[v] = o;
            if (part) {
                float4 a = acc4[v];
                fadd2_rn(a.x, a.y, a.x, a.y, o.x, o.y);
                fadd2_rn(a.z, a.w, a.z, a.w, o.z, o.w);
                acc4[v] = a;
            }
        }
    }
    if (part) {
        // a thread's own places: written by the thread that reads them
        float4 *p = reinterpret_cast<float4 *>(part + (size_t)blockIdx.x * K * H);
        for (int v = tid; v < K * G; v += NT) p[v] = acc4[v];
    }
}

// sums[split][x] = sum of part[n][x] over the split's n, x = d * H + h
__global__ void __launch_bounds__(kLbThreads)
lb_sum_kernel(const float *__restrict__ part, double *__restrict__ sums, int n, int KH) {
    const int x = blockIdx.x * kLbThreads + threadIdx.x;
    if (x >= KH) return;
    double acc = 0.0;
#pragma unroll 8
    for (int k = blockIdx.y; k < n; k += kLbSplits) acc += (double)part[(size_t)k * KH + x];
    sums[(size_t)blockIdx.y * KH + x] = acc;
}

// sums[split][d * H + h] = sum of dc[b,i,i+1+d,h] over the split's vertices (b,i)
__global__ void __launch_bounds__(kLbThreads)
lb_diag_kernel(const float *__restrict__ grad_content, double *__restrict__ sums, int B, int L, int H, int K) {
    const int x = blockIdx.x * kLbThreads + threadIdx.x;
    if (x >= K * H) return;
    const int d = x / H;
    const int64_t rows = (int64_t)B * L;
    double acc = 0.0;
    for (int64_t row = blockIdx.y; row < rows; row += kLbSplits) {
        const int i = (int)(row % L);
        if (i + 1 + d < L) acc += (double)grad_content[(row * L + i + 1) * H + x];
    }
    sums[(size_t)blockIdx.y * K * H + x] = acc;
}

// grad_table[k, h] from the partial sums: one CTA per bucket, the distances dealt to P = 128 / H lanes of a head
__global__ void __launch_bounds__(kLbThreads)
lb_join_kernel(const double *__restrict__ sums, const int64_t *__restrict__ bucket, float *__restrict__ grad_table, int H,
               int K) {
    __shared__ double lane_s[kLbThreads];
    const int k = blockIdx.x, P = kLbThreads / H, h = threadIdx.x % H, p = threadIdx.x / H;
    double acc = 0.0;
    if (p < P)
        for (int d = p; d < K; d += P)
            if (__ldg(bucket + d) == k) {
#pragma unroll
                for (int s = 0; s < kLbSplits; s++) acc += sums[((size_t)s * K + d) * H + h];
            }
    lane_s[threadIdx.x] = acc;
    __syncthreads();
    if (p == 0) {
        for (int q = 1; q < P; q++) acc += lane_s[q * H + h];
        grad_table[(size_t)k * H + h] = (float)acc;
    }
}

static bool lb_vector_form(int heads, int translen, const void *a, const void *b, const void *c, const void *d) {
    const int G = heads / 4;
    return heads % 4 == 0 && (G == 1 || G == 2 || G == 4 || G == 8) && (int64_t)translen * G <= kLbMaxVec &&
           ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b) | reinterpret_cast<uintptr_t>(c) |
             reinterpret_cast<uintptr_t>(d)) & 15) == 0;
}

// CTAs of a launch: as many as fit the device at once, at most one per vertex
template <typename F>
static int lb_grid(F kernel, int threads, size_t smem, int64_t rows, const DeviceInfo &di, int &grid, const char *who) {
    if (smem > 48 * 1024 &&
        cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
        return check_launch(who);
    int per_sm = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, smem);
    if (per_sm < 1) per_sm = 1;
    const int64_t n = (int64_t)di.sm_count * per_sm;
    grid = (int)(n < rows ? n : rows);
    return DAT_OK;
}

constexpr int kLbMaxPerSm = 16;   // CTAs per SM that the workspace has room for

struct LbArgs {
    const float *grad_links, *content, *log_gates, *head_lse_in;
    LinksMask mk;
    LinksBias lb;
    float *links, *head_lse, *grad_content, *grad_log_gates, *part;
    int B, L, K;
};

template <int G, int NT, int U>
static int lb_launch(const LbArgs &a, bool backward, int &grid, cudaStream_t st, const DeviceInfo &di, const char *who) {
    const int H = 4 * G;
    const int64_t rows = (int64_t)a.B * a.L;
    const size_t red = 2 * (NT / 32) * H * sizeof(float), table = (size_t)a.K * H * sizeof(float);
    if (!backward) {
        const size_t smem = table + red;
        if (int rc = lb_grid(lb_fwd_kernel<G, NT, U>, NT, smem, rows, di, grid, who)) return rc;
        lb_fwd_kernel<G, NT, U><<<grid, NT, smem, st>>>(a.content, a.log_gates, a.mk, a.lb, a.links, a.head_lse, a.B, a.L, a.K);
    } else {
        const size_t smem = table * (a.part ? 2 : 1) + red;
        if (int rc = lb_grid(lb_bwd_kernel<G, NT, U>, NT, smem, rows, di, grid, who)) return rc;
        if (grid > di.sm_count * kLbMaxPerSm) grid = di.sm_count * kLbMaxPerSm;
        lb_bwd_kernel<G, NT, U><<<grid, NT, smem, st>>>(a.grad_links, a.content, a.log_gates, a.head_lse_in, a.mk, a.lb,
                                                        a.grad_content, a.grad_log_gates, a.part, a.B, a.L, a.K);
    }
    return check_launch(who);
}

template <int G>
static int lb_dispatch(const LbArgs &a, bool backward, int &grid, cudaStream_t st, const DeviceInfo &di, const char *who) {
    const int nvec = a.K * G;
    if (nvec <= 2 * 128) return lb_launch<G, 128, 2>(a, backward, grid, st, di, who);
    if (nvec <= 4 * 128) return lb_launch<G, 128, 4>(a, backward, grid, st, di, who);
    if (nvec <= 8 * 128) return lb_launch<G, 128, 8>(a, backward, grid, st, di, who);
    if (nvec <= 8 * 256) return lb_launch<G, 256, 8>(a, backward, grid, st, di, who);
    return lb_launch<G, 512, 8>(a, backward, grid, st, di, who);
}

static int lb_run(const LbArgs &a, int heads, bool backward, int &grid, cudaStream_t st, const DeviceInfo &di,
                  const char *who) {
    switch (heads / 4) {
        case 1: return lb_dispatch<1>(a, backward, grid, st, di, who);
        case 2: return lb_dispatch<2>(a, backward, grid, st, di, who);
        case 4: return lb_dispatch<4>(a, backward, grid, st, di, who);
        default: return lb_dispatch<8>(a, backward, grid, st, di, who);
    }
}

static int lb_check(const char *who, const float *table, const int64_t *bucket, int buckets, int bsz, int prelen,
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
    using namespace dat;
    if (bsz < 0 || prelen < 1 || heads < 1 || translen < 1) return 0;
    DeviceInfo di;
    if (!device_info(&di)) return 0;
    int64_t n = (int64_t)di.sm_count * kLbMaxPerSm;
    if (n > (int64_t)bsz * prelen) n = (int64_t)bsz * prelen;
    return (size_t)translen * heads * (kLbSplits * sizeof(double) + (size_t)n * sizeof(float));
}

int dat_links_from_heads_biased(const float *content, const float *log_gates, const float *bias_table,
                                const int64_t *buckets, int num_buckets, const int64_t *bound_end,
                                const unsigned char *nonpad, float *links, float *head_lse, int32_t *status, int bsz,
                                int prelen, int heads, int translen, void *stream) {
    using namespace dat;
    const char *who = "dat_links_from_heads_biased";
    if (int rc = lb_check(who, bias_table, buckets, num_buckets, bsz, prelen, heads, translen)) return rc;
    if (bsz == 0) return DAT_OK;
    DAT_REQUIRE(content && log_gates && links, DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const LinksMask mk{bound_end, nonpad};
    const LinksBias lb{bias_table, buckets, num_buckets, status};
    if (lb_vector_form(heads, translen, content, log_gates, head_lse, nullptr)) {
        LbArgs a{};
        a.content = content;
        a.log_gates = log_gates;
        a.mk = mk;
        a.lb = lb;
        a.links = links;
        a.head_lse = head_lse;
        a.B = bsz;
        a.L = prelen;
        a.K = translen;
        int grid;
        return lb_run(a, heads, false, grid, st, di, who);
    }
    return links_fwd_rows<true>(content, log_gates, mk, lb, links, head_lse, bsz, prelen, heads, translen, st, di, who);
}

int dat_links_from_heads_biased_backward(const float *grad_links, const float *content, const float *log_gates,
                                         const float *bias_table, const int64_t *buckets, int num_buckets,
                                         const float *links, const float *head_lse, const int64_t *bound_end,
                                         const unsigned char *nonpad, float *grad_content, float *grad_log_gates,
                                         float *grad_bias_table, void *workspace, int bsz, int prelen, int heads,
                                         int translen, void *stream) {
    using namespace dat;
    const char *who = "dat_links_from_heads_biased_backward";
    if (int rc = lb_check(who, bias_table, buckets, num_buckets, bsz, prelen, heads, translen)) return rc;
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
    const LinksMask mk{bound_end, nonpad};
    const LinksBias lb{bias_table, buckets, num_buckets, nullptr};
    const int KH = translen * heads;
    double *sums = static_cast<double *>(workspace);
    const dim3 sgrid((unsigned)((KH + kLbThreads - 1) / kLbThreads), kLbSplits);
    if (lb_vector_form(heads, translen, content, log_gates, head_lse, grad_content) &&
        (reinterpret_cast<uintptr_t>(grad_log_gates) & 15) == 0) {
        LbArgs a{};
        a.grad_links = grad_links;
        a.content = content;
        a.log_gates = log_gates;
        a.head_lse_in = head_lse;
        a.mk = mk;
        a.lb = lb;
        a.grad_content = grad_content;
        a.grad_log_gates = grad_log_gates;
        a.part = grad_bias_table ? reinterpret_cast<float *>(sums + (size_t)kLbSplits * KH) : nullptr;
        a.B = bsz;
        a.L = prelen;
        a.K = translen;
        int grid;
        if (int rc = lb_run(a, heads, true, grid, st, di, who)) return rc;
        if (!grad_bias_table) return DAT_OK;
        lb_sum_kernel<<<sgrid, kLbThreads, 0, st>>>(a.part, sums, grid, KH);
    } else {
        if (int rc = links_bwd_rows<true>(grad_links, content, log_gates, links, head_lse, mk, lb, grad_content,
                                          grad_log_gates, bsz, prelen, heads, translen, st, di, who))
            return rc;
        if (!grad_bias_table) return DAT_OK;
        lb_diag_kernel<<<sgrid, kLbThreads, 0, st>>>(grad_content, sums, bsz, prelen, heads, translen);
    }
    if (int rc = check_launch(who)) return rc;
    lb_join_kernel<<<(unsigned)num_buckets, kLbThreads, 0, st>>>(sums, buckets, grad_bias_table, heads, translen);
    return check_launch(who);
}

}  // extern "C"

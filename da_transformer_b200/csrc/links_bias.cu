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
// forward, the dense gradient backward.  A vertex's scores lie in shared memory while it is worked on, and the exponentials
// and then the gradient take their place (a warp per vertex), or in registers (a CTA per vertex).  The bias is added in log2
// units; the table's gradient is gathered by distance over the vertices that a thread meets, and the partial sums of the CTAs
// are added in a fixed order in 64 bits (no atomics: results repeat bit for bit).  A thread's own sums are fp32, over some
// hundred vertices: 2^-24 of the sum in each addition, less than what the scores' gradients are rounded by.  One
// exponential per score and direction:
//   forward   e = exp(z - r_h), r_h the score of the nearest successor in place of the maximum over all of them:
//             the sum is at least 1, and a vertex where it overflows (a score 60 above r_h) or whose nearest
//             successor is masked takes the maximum after all.  links = log sum_h e_h exp(g_h) / S_h,
//             the gates relative to the vertex's largest.
//   backward  soft = exp(z - lse_h), q_h = soft exp(g_h), p_h = q_h / sum q.
// Where sum q is below 2^-80 (a link below -55) it is taken again relative to its largest term, so that what
// the 32-bit exponent flushes stays below 2^-40 of what it is added to: below 2^-126 in the backward, where soft and exp(g)
// are at most 1, and in the forward as long as exp(g_h) / S_h is a normal number (S_h may reach 2^86).  A vertex with a
// head whose factor is below 2^-100 takes all its links that way.  A valid score of NaN or +inf makes the sum of its head
// NaN, and with it every link and gradient of the vertex, as it does by definition.
// Two forms, a warp or a CTA per vertex (below): the first up to 32 heads and rows of 2048 vectors that fit its rings,
// the second 4, 8, 16 and 32 heads up to 4096 vectors.  What neither takes goes to the kernels of links.cu (one CTA per
// vertex, scores in shared memory) and a pass over the gradient's diagonals.
#include <functional>

#include "links_common.cuh"
#include "umma.cuh"

namespace dat {

constexpr float kLbTiny = 0x1p-80f;
constexpr float kLbHuge = 0x1p+86f;
constexpr float kLbRare = 0x1p-100f;
constexpr int kLbMaxVec = 4096;         // score vectors per vertex: 512 threads with eight each

// bias by distance in log2 units into shared memory; -inf for a bucket outside the table
template <int NT>
__device__ __forceinline__ void lb_expand(const LinksBias &lb, float *bl, int H, int K) {
    bool bad = false;
    for (int x = threadIdx.x; x < K * H; x += NT) bl[x] = links_bias1(lb, x / H, x % H, H, bad) * kLog2e;
    if (bad && lb.status) atomicOr(lb.status, DAT_STATUS_BAD_INDEX);
}

__device__ __forceinline__ float4 lb_ninf4() { return make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY); }

// One vertex of the walk: rows are dealt so that a CTA meets long and short rows in turn.
struct LbRow {
    int64_t row;   // b * L + i
    int i, nj;     // vertex, successors inside the band (before the padding mask); nj < 0: no such row
};
__device__ __forceinline__ LbRow lb_row(int slot, int rows, int L, int K, const LinksMask &mk) {
    LbRow r{0, 0, -1};
    if (slot < rows) {
        const int b = slot / L, q = slot - b * L;
        r.i = (q & 1) ? L - 1 - (q >> 1) : (q >> 1);
        r.row = (int64_t)b * L + r.i;
        const int jhi = links_jhi(r.i, L, K, mk, r.row);
        r.nj = jhi - r.i > 0 ? jhi - r.i : 0;
    }
    return r;
}
// bit u: the thread's vector tid + u * NT belongs to a valid successor; bit 31: so does the nearest successor
template <int G, int NT, int U>
__device__ __forceinline__ unsigned lb_live(const LbRow &r, int L, const LinksMask &mk) {
    const int tid = threadIdx.x;
    unsigned live = 0;
    if (r.nj <= 0) return 0;
    if (!mk.nonpad) {
#pragma unroll
        for (int u = 0; u < U; u++) live |= tid + u * NT < r.nj * G ? 1u << u : 0u;
        return live | 0x80000000u;
    }
    const unsigned char *np = mk.nonpad + (r.row - r.i) + r.i + 1;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int v = tid + u * NT;
        if (v < r.nj * G && np[v / G]) live |= 1u << u;
    }
    return np[0] ? live | 0x80000000u : live;
}
// the bits of lb_live whose distance has a bucket; the scores of the others are not looked at
template <int G, int NT, int U>
__device__ __forceinline__ unsigned lb_in_table(const LinksBias &lb, int K) {
    unsigned in = links_bucket_ok(lb, 0) ? 0x80000000u : 0;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int v = threadIdx.x + u * NT;
        if (v < K * G && links_bucket_ok(lb, v / G)) in |= 1u << u;
    }
    return in;
}
__device__ __forceinline__ void lb_copy16(float4 *dst, const float4 *src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void lb_copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void lb_copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// the thread's vectors of a row on their way into the stage (each thread reads only what it copied itself)
template <int G, int NT, int U>
__device__ __forceinline__ void lb_fetch(const LbRow &r, unsigned live, const float *content, int L, float4 *stage) {
    if (r.nj > 0) {
        const float4 *src = reinterpret_cast<const float4 *>(content + (r.row * L + r.i + 1) * (int64_t)(4 * G));
#pragma unroll
        for (int u = 0; u < U; u++)
            if (live >> u & 1) lb_copy16(stage + threadIdx.x + u * NT, src + threadIdx.x + u * NT);
    }
    lb_copy_commit();
}

// Sum (or maximum) of v over the warp's lanes of the same head group, left in red[warp][4g + k].  Halving exchange:
// two steps in which a lane hands over half of its values, then butterflies on what it keeps.
template <int G, int NT, bool kMax>
__device__ __forceinline__ void lb_reduce(const float (&v)[4], float *red) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & (G - 1);
    const auto op = [](float a, float b) { return kMax ? fmaxf(a, b) : a + b; };
    const bool up = lane & 16, up2 = lane & 8;
    float a = up ? v[0] : v[2], b = up ? v[1] : v[3];                   // given away
    a = op(up ? v[2] : v[0], __shfl_xor_sync(0xffffffffu, a, 16));      // kept: heads 0,1 below, 2,3 above
    b = op(up ? v[3] : v[1], __shfl_xor_sync(0xffffffffu, b, 16));
    float c = op(up2 ? b : a, __shfl_xor_sync(0xffffffffu, up2 ? a : b, 8));
    if (G < 8) c = op(c, __shfl_xor_sync(0xffffffffu, c, 4));
    if (G < 4) c = op(c, __shfl_xor_sync(0xffffffffu, c, 2));
    if (G < 2) c = op(c, __shfl_xor_sync(0xffffffffu, c, 1));
    if ((lane & 7) < G) red[warp * (4 * G) + 4 * g + (up ? 2 : 0) + (up2 ? 1 : 0)] = c;
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
// The gates of a vertex less its largest, in log2 units, so that their exponentials are at most 1 whatever the gates are;
// returns what was taken away (it is added to the link; the shares of the heads do not change with it)
template <int G>
__device__ __forceinline__ float lb_gates(float4 gate, float (&g2)[4]) {
    const float top = lb_max_over_heads<G>(fmaxf(fmaxf(gate.x, gate.y), fmaxf(gate.z, gate.w))), m = top > -INFINITY ? top : 0.f;
    g2[0] = (gate.x - m) * kLog2e;
    g2[1] = (gate.y - m) * kLog2e;
    g2[2] = (gate.z - m) * kLog2e;
    g2[3] = (gate.w - m) * kLog2e;
    return m;
}
// A head's factor f = exp(g) / S may lose terms that count, or is NaN: the links are taken from the logarithms (which also
// keep NaN from the masked places).  A gate of -inf leaves nothing to lose.
__device__ __forceinline__ bool lb_rare(float f, float g2) { return !(f >= kLbRare || (f == 0.f && g2 == -INFINITY)); }
// A head's log-sum in the backward; that of one without a finite score is +inf: soft = exp(-inf) = 0
__device__ __forceinline__ float lb_lse(float lse) { return lse == -INFINITY ? INFINITY : lse; }
// t = z - r with z = c log2e + b rounded as the reference r was, so that t is 0 where z is the reference
__device__ __forceinline__ float4 lb_shifted(float4 c, float4 b, const float (&r)[4]) {
    ffma2_rn(b.x, b.y, c.x, c.y, kLog2e, kLog2e);
    ffma2_rn(b.z, b.w, c.z, c.w, kLog2e, kLog2e);
    fadd2_rn(b.x, b.y, b.x, b.y, -r[0], -r[1]);
    fadd2_rn(b.z, b.w, b.z, b.w, -r[2], -r[3]);
    return b;
}
// Gradient of four scores, q w - soft S: the product is rounded as its sum S was, so that a vertex with one successor
// (soft = 1, S that product) has the gradient 0 that it has by definition
__device__ __forceinline__ float4 lb_grad(float4 soft, float4 q, float w, const float (&S)[4]) {
    fmul2_rn(q.x, q.y, q.x, q.y, w, w);
    fmul2_rn(q.z, q.w, q.z, q.w, w, w);
    ffma2_rn(q.x, q.y, soft.x, soft.y, -S[0], -S[1]);
    ffma2_rn(q.z, q.w, soft.z, soft.w, -S[2], -S[3]);
    return q;
}

// A CTA per vertex.  A thread holds the same distances and heads (16 bytes: four heads of one distance) of every vertex, the
// scores in registers; the bias is expanded by distance once per CTA.
// Shared memory of both kernels: the bias by distance [K * H], two rows of scores [K * H], red [2][NT / 32][H].
// A row's scores are copied while the row before is worked on, its mask is read one row earlier still.
// G = H / 4 vectors per distance; thread t holds the vectors t, t + NT, ... of a vertex's row (U of them).
template <int G, int NT, int U>
__global__ void __launch_bounds__(NT)
lb_fwd_kernel(const float *__restrict__ content, const float *__restrict__ log_gates, LinksMask mk, LinksBias lb,
              float *__restrict__ links, float *__restrict__ head_lse, int B, int L, int K) {
    constexpr int H = 4 * G;
    extern __shared__ __align__(16) float lbsm[];
    float *bl = lbsm, *red = lbsm + (size_t)3 * K * H;
    float4 *const bl4 = reinterpret_cast<float4 *>(bl);
    const int tid = threadIdx.x, lane = tid & 31, g = lane & (G - 1);
    const int rows = B * L, step = gridDim.x;
    int slot = blockIdx.x;
    LbRow r0 = lb_row(slot, rows, L, K, mk), r1 = lb_row(slot + step, rows, L, K, mk);
    const unsigned in_table = lb_in_table<G, NT, U>(lb, K);
    unsigned live0 = lb_live<G, NT, U>(r0, L, mk) & in_table, live1 = lb_live<G, NT, U>(r1, L, mk) & in_table;
    const auto nearest = [&](const LbRow &r) {
        return r.nj > 0 ? __ldg(reinterpret_cast<const float4 *>(content + (r.row * L + r.i + 1) * (int64_t)H) + g) : lb_ninf4();
    };
    const auto gates_of = [&](const LbRow &r) {
        return r.nj >= 0 ? __ldg(reinterpret_cast<const float4 *>(log_gates + r.row * H) + g) : lb_ninf4();
    };
    float4 near0 = nearest(r0), gate0 = gates_of(r0);
    lb_fetch<G, NT, U>(r0, live0, content, L, bl4 + (size_t)K * G);
    lb_expand<NT>(lb, bl, H, K);
    __syncthreads();
    int par = 0;
    for (; r0.nj >= 0; slot += step, par ^= 1) {
        float4 *const stage = bl4 + (size_t)(1 + par) * K * G;
        lb_fetch<G, NT, U>(r1, live1, content, L, bl4 + (size_t)(2 - par) * K * G);
        const float4 near1 = nearest(r1), gate1 = gates_of(r1);
        const LbRow r2 = lb_row(slot + 2 * step, rows, L, K, mk);
        const unsigned live2 = lb_live<G, NT, U>(r2, L, mk) & in_table;
        lb_copy_wait<1>();
        // r_h in log2 units
        const float4 b0 = bl4[g];
        float r[4] = {fmaf(near0.x, kLog2e, b0.x), fmaf(near0.y, kLog2e, b0.y), fmaf(near0.z, kLog2e, b0.z),
                      fmaf(near0.w, kLog2e, b0.w)};
        const bool no_r = !(live0 >> 31) || !(fabsf(r[0]) < INFINITY && fabsf(r[1]) < INFINITY && fabsf(r[2]) < INFINITY &&
                                              fabsf(r[3]) < INFINITY);
        float4 e4[U];
        float sum[4] = {0.f, 0.f, 0.f, 0.f};
        const int nvec = r0.nj * G;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT;
            e4[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (live0 >> u & 1) {
                const float4 t = lb_shifted(stage[v], bl4[v], r);
                e4[u] = make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w));
                fadd2_rn(sum[0], sum[1], sum[0], sum[1], e4[u].x, e4[u].y);
                fadd2_rn(sum[2], sum[3], sum[2], sum[3], e4[u].z, e4[u].w);
            }
        }
        const bool bad = (live0 & 0x7fffffffu) &&
                         (no_r || !(fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3])) < kLbHuge) ||
                          !(sum[0] + sum[1] + sum[2] + sum[3] < INFINITY));
        float *rd = red + par * (NT / 32) * H;
        lb_reduce<G, NT, false>(sum, rd);
        if (__syncthreads_or(bad)) {
            // the exact maximum of each head takes the place of r_h
            float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = tid + u * NT;
                if (live0 >> u & 1) {
                    const float4 c = stage[v], t = bl4[v];
                    m[0] = fmaxf(m[0], fmaf(c.x, kLog2e, t.x));
                    m[1] = fmaxf(m[1], fmaf(c.y, kLog2e, t.y));
                    m[2] = fmaxf(m[2], fmaf(c.z, kLog2e, t.z));
                    m[3] = fmaxf(m[3], fmaf(c.w, kLog2e, t.w));
                }
            }
            lb_reduce<G, NT, true>(m, rd);   // the sums that the place held are not wanted
            __syncthreads();
            lb_collect<G, NT, true>(m, rd);
            sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll
            for (int k = 0; k < 4; k++) r[k] = m[k] > -INFINITY ? m[k] : 0.f;
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int v = tid + u * NT;
                e4[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (live0 >> u & 1) {
                    const float4 t = lb_shifted(stage[v], bl4[v], r);
                    e4[u] = make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w));
                    fadd2_rn(sum[0], sum[1], sum[0], sum[1], e4[u].x, e4[u].y);
                    fadd2_rn(sum[2], sum[3], sum[2], sum[3], e4[u].z, e4[u].w);
                }
            }
            __syncthreads();
            lb_reduce<G, NT, false>(sum, rd);
            __syncthreads();
        }
        lb_collect<G, NT, false>(sum, rd);
        // f_h = exp(g_h) / S_h; a head without a finite score takes no part
        float g2[4], f[4];
        const float top = lb_gates<G>(gate0, g2);
        bool some[4], rare = false;
#pragma unroll
        for (int k = 0; k < 4; k++) {
            some[k] = sum[k] != 0.f;
            f[k] = some[k] ? __fdividef(ex2(g2[k]), sum[k]) : 0.f;
            rare |= some[k] && lb_rare(f[k], g2[k]);
        }
        rare = __any_sync(0xffffffffu, rare);
        if (head_lse && tid < G) {
#pragma unroll
            for (int k = 0; k < 4; k++)
                head_lse[r0.row * H + 4 * g + k] = some[k] ? r[k] + lg2(sum[k]) : -INFINITY;
        }
        float *out = links + r0.row * (int64_t)K;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT, d = v / G;
            if (u * NT + (tid & ~31) >= K * G) break;
            const bool ok = live0 >> u & 1;
            float link = -INFINITY;
            if (u * NT + (tid & ~31) < nvec) {
                float q = lb_over_heads<G>(fmaf(e4[u].x, f[0], e4[u].y * f[1]) + fmaf(e4[u].z, f[2], e4[u].w * f[3]));
                link = ok ? fmaf(lg2(q), kLn2, top) : -INFINITY;
                if (rare || __any_sync(0xffffffffu, ok && !(q >= kLbTiny))) {
                    float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                    if (ok) {   // log2 of e f without the exponential's flush
                        const float4 z = lb_shifted(stage[v], bl4[v], r);
                        if (some[0]) t[0] = z.x + (g2[0] - lg2(sum[0]));
                        if (some[1]) t[1] = z.y + (g2[1] - lg2(sum[1]));
                        if (some[2]) t[2] = z.z + (g2[2] - lg2(sum[2]));
                        if (some[3]) t[3] = z.w + (g2[3] - lg2(sum[3]));
                    }
                    const float m = lb_max_over_heads<G>(fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3])));
                    const float mm = m > -INFINITY ? m : 0.f;
                    q = lb_over_heads<G>(ex2(t[0] - mm) + ex2(t[1] - mm) + ex2(t[2] - mm) + ex2(t[3] - mm));
                    link = ok ? fmaf(mm + lg2(q), kLn2, top) : -INFINITY;
                }
            }
            if (g == 0 && d < K) out[d] = link;
        }
        r0 = r1;
        r1 = r2;
        live0 = live1;
        live1 = live2;
        near0 = near1;
        gate0 = gate1;
    }
    lb_copy_wait<0>();
}

template <int G, int NT, int U>
__global__ void __launch_bounds__(NT)
lb_bwd_kernel(const float *__restrict__ grad_links, const float *__restrict__ content,
              const float *__restrict__ log_gates, const float *__restrict__ head_lse, LinksMask mk, LinksBias lb,
              float *__restrict__ grad_content, float *__restrict__ grad_log_gates, float *__restrict__ part, int B, int L,
              int K) {
    constexpr int H = 4 * G;
    extern __shared__ __align__(16) float lbsm[];
    float *bl = lbsm, *red = lbsm + (size_t)3 * K * H;
    float4 *const bl4 = reinterpret_cast<float4 *>(bl);
    const int tid = threadIdx.x, lane = tid & 31, g = lane & (G - 1);
    const int rows = B * L, step = gridDim.x;
    int slot = blockIdx.x;
    LbRow r0 = lb_row(slot, rows, L, K, mk), r1 = lb_row(slot + step, rows, L, K, mk);
    const unsigned in_table = lb_in_table<G, NT, U>(lb, K);
    unsigned live0 = lb_live<G, NT, U>(r0, L, mk) & in_table, live1 = lb_live<G, NT, U>(r1, L, mk) & in_table;
    const auto of_row = [&](const float *p, const LbRow &r) {
        return r.nj >= 0 ? __ldg(reinterpret_cast<const float4 *>(p + r.row * H) + g) : lb_ninf4();
    };
    float gd[U];   // the incoming gradient, a row ahead like the scores
    const auto fetch_grad = [&](const LbRow &r, unsigned live, float (&to)[U]) {
#pragma unroll
        for (int u = 0; u < U; u++)
            to[u] = live >> u & 1 ? __ldg(grad_links + r.row * (int64_t)K + (tid + u * NT) / G) : 0.f;
    };
    float4 lse0 = of_row(head_lse, r0), gate0 = of_row(log_gates, r0);
    fetch_grad(r0, live0, gd);
    lb_fetch<G, NT, U>(r0, live0, content, L, bl4 + (size_t)K * G);
    lb_expand<NT>(lb, bl, H, K);
    __syncthreads();
    float4 acc[U];   // the gradient by distance of this CTA's rows
#pragma unroll
    for (int u = 0; u < U; u++) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    int par = 0;
    for (; r0.nj >= 0; slot += step, par ^= 1) {
        float4 *const stage = bl4 + (size_t)(1 + par) * K * G;
        lb_fetch<G, NT, U>(r1, live1, content, L, bl4 + (size_t)(2 - par) * K * G);
        const float4 lse1 = of_row(head_lse, r1), gate1 = of_row(log_gates, r1);
        const LbRow r2 = lb_row(slot + 2 * step, rows, L, K, mk);
        const unsigned live2 = lb_live<G, NT, U>(r2, L, mk) & in_table;
        const float ls[4] = {lb_lse(lse0.x), lb_lse(lse0.y), lb_lse(lse0.z), lb_lse(lse0.w)};
        float g2[4];
        lb_gates<G>(gate0, g2);
        const float eg[4] = {ex2(g2[0]), ex2(g2[1]), ex2(g2[2]), ex2(g2[3])};
        lb_copy_wait<1>();
        float4 p4[U];
        float S[4] = {0.f, 0.f, 0.f, 0.f};
        const int nvec = r0.nj * G;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT;
            p4[u] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (u * NT + (tid & ~31) >= nvec) continue;   // nothing of this warp
            const bool ok = live0 >> u & 1;
            const float4 t = ok ? lb_shifted(stage[v], bl4[v], ls) : lb_ninf4();
            const float4 soft = make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w));
            if (v < K * G) stage[v] = soft;
            float4 q = make_float4(soft.x * eg[0], soft.y * eg[1], soft.z * eg[2], soft.w * eg[3]);
            const float tot = lb_over_heads<G>((q.x + q.y) + (q.z + q.w));
            float w = tot >= kLbTiny ? __fdividef(gd[u], tot) : 0.f;
            if (__any_sync(0xffffffffu, ok && !(tot >= kLbTiny))) {
                const float a[4] = {t.x + g2[0], t.y + g2[1], t.z + g2[2], t.w + g2[3]};
                const float m = lb_max_over_heads<G>(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3])));
                if (!(tot >= kLbTiny)) {   // the same in all lanes of a distance
                    const float mm = m > -INFINITY ? m : 0.f;
                    q = make_float4(ex2(a[0] - mm), ex2(a[1] - mm), ex2(a[2] - mm), ex2(a[3] - mm));
                }
                const float tot2 = lb_over_heads<G>((q.x + q.y) + (q.z + q.w));
                w = ok && tot2 != 0.f ? gd[u] / tot2 : 0.f;
            }
            // a link of -inf has w = 0 times a gradient that may be anything
            p4[u] = w != 0.f ? make_float4(q.x * w, q.y * w, q.z * w, q.w * w) : p4[u];
            fadd2_rn(S[0], S[1], S[0], S[1], p4[u].x, p4[u].y);
            fadd2_rn(S[2], S[3], S[2], S[3], p4[u].z, p4[u].w);
        }
        float *rd = red + par * (NT / 32) * H;
        lb_reduce<G, NT, false>(S, rd);
        fetch_grad(r1, live1, gd);
        // the places of the dense row that no valid successor has
        float4 *rowv = reinterpret_cast<float4 *>(grad_content + r0.row * (int64_t)L * H);
        const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int v = tid; v < (r0.i + 1) * G; v += NT) rowv[v] = zero;
        for (int v = (r0.i + 1) * G + nvec + tid; v < L * G; v += NT) rowv[v] = zero;
        __syncthreads();
        lb_collect<G, NT, false>(S, rd);
        if (tid < G)
            reinterpret_cast<float4 *>(grad_log_gates + r0.row * H)[g] = make_float4(S[0], S[1], S[2], S[3]);
        float4 *dst = rowv + (r0.i + 1) * G;
        const bool odd = !(fabsf(S[0] + S[1] + S[2] + S[3]) < INFINITY);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int v = tid + u * NT;
            if (v >= nvec) break;
            const float4 soft = stage[v];
            float4 o = p4[u];
            ffma2_rn(o.x, o.y, soft.x, soft.y, -S[0], -S[1]);
            ffma2_rn(o.z, o.w, soft.z, soft.w, -S[2], -S[3]);
            if (odd && !(live0 >> u & 1)) o = make_float4(0.f, 0.f, 0.f, 0.f);   // a masked place beside NaN
            dst[v] = o;
            fadd2_rn(acc[u].x, acc[u].y, acc[u].x, acc[u].y, o.x, o.y);
            fadd2_rn(acc[u].z, acc[u].w, acc[u].z, acc[u].w, o.z, o.w);
        }
        r0 = r1;
        r1 = r2;
        live0 = live1;
        live1 = live2;
        lse0 = lse1;
        gate0 = gate1;
    }
    lb_copy_wait<0>();
    if (part) {
        float4 *p = reinterpret_cast<float4 *>(part + (size_t)blockIdx.x * K * H);
#pragma unroll
        for (int u = 0; u < U; u++)
            if (tid + u * NT < K * G) p[tid + u * NT] = acc[u];
    }
}

// ---------------------------------------------------------------------------------------------------
// One warp per vertex, four neighbouring vertices at a time: what a vertex costs beside its scores (its place, the
// reduction over the lanes, the gates) is paid by one warp and not by the four of a CTA per vertex.  A vertex's valid
// scores are one piece of memory: one bulk asynchronous copy brings it into the warp's ring in shared memory while
// the warp works on the vertex before, the exponentials and then the gradient take the scores' place, and a bulk
// copy writes the gradient back (the zeros around it come from a block of zeros).  Rows are triangular, so a ring
// little larger than the longest row holds two ordinary ones.
// A lane holds four heads of a distance, G lanes (a power of two) a distance.  kExact: H = 4 G, so that a row is an array
// of 16-byte vectors; other head counts up to 32 leave places empty (-inf, no part in anything) and read and write the
// row's numbers one by one, and where H is no multiple of four a row begins at any address: the copy takes the 16-byte
// pieces up to its end, the up to three numbers behind them are loaded singly, and the gradient is stored by the lanes.
// Used where a row has at most kLwMaxVec vectors, fits a ring, and the bias table takes a few KB.
// Forward and backward, called from Python, against the kernels of links.cu with the pass over the diagonals: 16 graphs of
// 512 vertices and 12 heads 76 + 147 us against 140 + 515, 32 and 6 heads 79 + 146 against 135 + 740, 64 and 3 heads
// 77 + 185 against 185 + 1265, 64 and one head 64 + 165 against 166 + 927.
// ---------------------------------------------------------------------------------------------------
constexpr int kLwRows = 4;          // vertices of a group, a warp each
constexpr int kLwMaxVec = 2048;     // score vectors per vertex (places of empty heads included)
constexpr int kLwMaxTable = 2048;   // floats of the bias table
constexpr int kLwZeros = 2048;      // bytes of zeros
constexpr int kLwU = 4;             // vectors of a lane taken together: loads first, then the arithmetic, then the stores
template <int N>
struct LwInt {
    static constexpr int value = N;
};
constexpr int kLwPolls = 1 << 20;   // bound of a wait for a copy (never reached)
constexpr uint32_t kLwFull = 0x7fc00d1eu;   // weight of a distance whose shares are taken in full (no result of arithmetic)

// span[b] = (last vertex that the mask allows, whether one between the first and it is not allowed); vertex 0 is
// nobody's successor
__global__ void __launch_bounds__(128)
lw_span_kernel(const unsigned char *__restrict__ nonpad, int2 *__restrict__ span, int L) {
    __shared__ int last_s[4], n_s[4];
    pdl_trigger();
    const unsigned char *np = nonpad + (int64_t)blockIdx.x * L;
    int last = -1, n = 0;
    for (int j = 1 + threadIdx.x; j < L; j += 128)
        if (np[j]) {
            last = j;
            n++;
        }
    last = __reduce_max_sync(0xffffffffu, last);
    n = __reduce_add_sync(0xffffffffu, n);
    if ((threadIdx.x & 31) == 0) {
        last_s[threadIdx.x >> 5] = last;
        n_s[threadIdx.x >> 5] = n;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 4; w++) {
            last = max(last, last_s[w]);
            n += n_s[w];
        }
        span[blockIdx.x] = make_int2(last, last >= 1 && n != last);
    }
}

// The walk: groups of four neighbouring vertices, dealt to the `step` sets of warps in turn.
// Forward (LwPairs): groups from the front of all sentences and from their backs in turn, front and back in opposite order,
// which gives every set pairs of one length.  Backward (LwEnds): sentence by sentence, groups from its two ends in turn
// (which end comes first changes from sentence to sentence: the stride may be even); a row's copy then seldom waits for
// the store of the long row before it.  64 graphs of 512 (500) vertices, 8 heads, forward 88 (86) us with LwPairs against
// 94 (106) with LwEnds, backward 187 (181) against 169 (173), called from Python.
struct LwRow {
    int64_t row;   // b * L + i
    int i, nj;     // vertex, successors up to the last one that the masks allow (after lw_resolve)
    bool exists, holes;
    // as they lie in memory: looked at a row later, when they have arrived
    int2 sp;
    int64_t bound;
};
struct LwPairs {
    int at, step, groups, near, B;   // number of the group in the walk, and of those that come from the front
    bool back;
    __device__ __forceinline__ LwPairs(int first, int step_, int B_, int L)
        : at(first), step(step_), groups(B_ * ((L + kLwRows - 1) / kLwRows)), near(first), B(B_), back(false) {}
    __device__ __forceinline__ bool next(int &b, int &q) {
        if (at >= groups) return false;
        const int t = back ? groups - 1 - near : near;
        if (back) near += step;
        back = !back;
        at += step;
        q = t / B;
        b = t - q * B;
        return true;
    }
};
struct LwEnds {
    int per, step_b, step_q, b, q, B;
    __device__ __forceinline__ LwEnds(int first, int step, int B_, int L) : B(B_) {
        per = (L + kLwRows - 1) / kLwRows;
        step_b = step / per;
        step_q = step - step_b * per;
        b = first / per;
        q = first - b * per;
    }
    __device__ __forceinline__ bool next(int &b_, int &q_) {
        if (b >= B) return false;
        b_ = b;
        q_ = ((q ^ b) & 1) ? per - 1 - (q >> 1) : (q >> 1);
        b += step_b;
        q += step_q;
        if (q >= per) {
            q -= per;
            b++;
        }
        return true;
    }
};
template <typename Walk>
__device__ __forceinline__ LwRow lw_row(Walk &walk, int L, const LinksMask &mk, const int2 *span) {
    LwRow r{0, 0, 0, false, false, {0, 0}, 0};
    int b, q;
    if (!walk.next(b, q)) return r;
    r.i = q * kLwRows + (threadIdx.x >> 5) % kLwRows;
    if (r.i >= L) return r;
    r.exists = true;
    r.row = (int64_t)b * L + r.i;
    if (mk.nonpad) r.sp = __ldcg(span + b);   // (a coherent load: the kernel that writes it may have run beside this one)
    if (mk.bound_end) r.bound = __ldg(mk.bound_end + r.row);
    return r;
}
__device__ __forceinline__ void lw_resolve(LwRow &r, int L, int K, const LinksMask &mk) {
    if (!r.exists) return;
    int jhi = min(r.i + K, L - 1);
    if (mk.nonpad) {
        jhi = min(jhi, r.sp.x);
        r.holes = r.sp.y != 0;
    }
    if (mk.bound_end && r.bound < jhi) jhi = r.bound < 0 ? -1 : (int)r.bound;
    r.nj = jhi - r.i > 0 ? jhi - r.i : 0;
}

// Vector v of a row (distance v / G, heads 4 (v % G) ..) from and to memory; `fill` stands for heads that are not there.
template <int G, bool kExact>
__device__ __forceinline__ float4 lw_get(const float *row, int v, int H, float fill) {
    if (kExact) return reinterpret_cast<const float4 *>(row)[v];
    const int h = (v & (G - 1)) * 4;
    const float *p = row + (v / G) * H + h;
    float4 r = make_float4(fill, fill, fill, fill);
    if ((H & 3) == 0) {
        if (h < H) r = *reinterpret_cast<const float4 *>(p);
    } else {
        if (h < H) r.x = p[0];
        if (h + 1 < H) r.y = p[1];
        if (h + 2 < H) r.z = p[2];
        if (h + 3 < H) r.w = p[3];
    }
    return r;
}
template <int G, bool kExact>
__device__ __forceinline__ void lw_put(float *row, int v, int H, float4 x) {
    if (kExact) {
        reinterpret_cast<float4 *>(row)[v] = x;
        return;
    }
    const int h = (v & (G - 1)) * 4;
    float *p = row + (v / G) * H + h;
    if ((H & 3) == 0) {
        if (h < H) *reinterpret_cast<float4 *>(p) = x;
    } else {
        if (h < H) p[0] = x.x;
        if (h + 1 < H) p[1] = x.y;
        if (h + 2 < H) p[2] = x.z;
        if (h + 3 < H) p[3] = x.w;
    }
}

// bias of vector v in log2 units, from the table in shared memory (rows of 4 G; its last row: -inf, for buckets outside)
template <int G>
__device__ __forceinline__ float4 lw_bias(const float4 *table, const unsigned short *bucket, int v) {
    return table[bucket[v / G] * G + (v & (G - 1))];
}
template <int G, int NT>
__device__ __forceinline__ bool lw_load_table(const LinksBias &lb, float *table, unsigned short *bucket, int H, int K) {
    bool bad = false;
    for (int x = threadIdx.x; x < lb.n * (4 * G); x += NT) {
        const int k = x / (4 * G), h = x - k * (4 * G);
        table[x] = h < H ? __ldg(lb.table + k * H + h) * kLog2e : 0.f;
    }
    for (int x = threadIdx.x; x < 4 * G; x += NT) table[lb.n * (4 * G) + x] = -INFINITY;
    for (int d = threadIdx.x; d < K; d += NT) {
        const int64_t k = __ldg(lb.bucket + d);
        const bool ok = k >= 0 && k < lb.n;
        bad |= !ok;
        bucket[d] = (unsigned short)(ok ? k : lb.n);
    }
    if (bad && lb.status) atomicOr(lb.status, DAT_STATUS_BAD_INDEX);
    return bad;
}

// The distances of a row whose transitions are not allowed although they lie inside its span: a hole in the mask, or a
// bucket outside the table.  Their scores may be anything.
struct LwDead {
    const unsigned char *np;       // mask of the row's successors, or null: no holes
    const unsigned short *bucket;
    int none;                      // bucket of the distances that have none; -1: all have one
    __device__ __forceinline__ bool any() const { return np || none >= 0; }
    __device__ __forceinline__ bool operator()(int d) const { return (np && !np[d]) || bucket[d] == none; }
};

// Shared memory, in bytes: table, buckets, zeros, barriers of the copies, then the rings.
struct LwSmem {
    int bucket, zeros, mbar, rings, ring;   // ring: bytes of one warp's
};
// dynamic shared memory of one CTA per SM (a little is left for what the kernels declare themselves) and of two
static int lw_one(const DeviceInfo &di) { return di.max_smem_optin - 256; }
static int lw_two(const DeviceInfo &di) { return (di.max_smem_optin + 1024) / 2 - 1024 - 256; }
// lanes of a distance
static int lw_lanes(int H) { return H <= 4 ? 1 : H <= 8 ? 2 : H <= 16 ? 4 : 8; }
// scores and the band's gradient, each with room for a beginning inside a 16-byte piece
static int lw_row_bytes(int K, int H) { return (K * H + 8) * 4 / 16 * 16 + (K + 8) * 4 / 16 * 16; }
static LwSmem lw_smem(int K, int H, int n, int warps, int avail) {
    LwSmem m;
    m.bucket = (n + 1) * (4 * lw_lanes(H)) * 4;
    m.zeros = (m.bucket + K * 2 + 15) / 16 * 16;
    m.mbar = m.zeros + kLwZeros;
    m.rings = m.mbar + (warps * 8 + 15) / 16 * 16;
    m.ring = (avail - m.rings) / warps / 16 * 16;
    return m;
}

__device__ __forceinline__ void lw_bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t mbar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
                 "l"(src), "r"(bytes), "r"(mbar)
                 : "memory");
}
__device__ __forceinline__ void lw_bulk_store(void *dst, uint32_t src, uint32_t bytes) {
    asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void lw_bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
// n zeros from p on: whole 16-byte pieces by the lanes' copies of the block of zeros, those around them (kEdges) singly
template <bool kEdges>
__device__ __forceinline__ void lw_zero(float *p, int n, uint32_t zeros) {
    const int lane = threadIdx.x & 31;
    if (kEdges) {
        const int head = min((int)(-(reinterpret_cast<uintptr_t>(p) >> 2) & 3), n), tail = (n - head) & 3;
        if (lane < head) p[lane] = 0.f;
        if (lane < tail) p[n - tail + lane] = 0.f;
        p += head;
        n -= head + tail;
    }
    for (int at = lane * (kLwZeros / 4); at < n; at += 32 * (kLwZeros / 4))
        lw_bulk_store(p + at, zeros, min(kLwZeros / 4, n - at) * 4);
}
// all bulk stores of this thread have read their shared memory
__device__ __forceinline__ void lw_bulk_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// A row in the ring: [window of the band's gradient (backward)][scores].  A window is the 16-byte pieces of an array
// that reach up to the row's end; the up to three numbers behind them are loaded singly (all of them where the array
// does not start on a 16-byte boundary: wide = false).
__device__ __forceinline__ int lw_skip(int64_t first) { return (int)(first & 3); }   // numbers of the first piece before the row
__device__ __forceinline__ int lw_whole(int skip, int n, bool wide) {                // numbers of the row that the pieces hold
    const int to = (skip + n) & ~3;
    return wide && to > 0 ? to - skip : 0;
}
struct LwSlot {
    int at, bytes;       // place in the ring
    int window, skip;    // of the band's gradient: bytes, numbers before the row
    int front;           // numbers before the row's scores
};
template <int G, bool kExact, bool kBackward>
__device__ __forceinline__ LwSlot lw_slot(const LwRow &r, int L, int H, int K) {
    LwSlot s{0, 0, 0, 0, 0};
    if (r.nj > 0) {
        if (kBackward) {
            s.skip = lw_skip(r.row * (int64_t)K);
            s.window = (s.skip + r.nj + 3) / 4 * 16;
        }
        if (!kExact) s.front = lw_skip((r.row * L + r.i + 1) * (int64_t)H);
        s.bytes = s.window + (kExact ? r.nj * (16 * G) : (s.front + r.nj * H + 3) / 4 * 16);
    }
    return s;
}
// the place after `at + bytes` in the ring that keeps clear of [at, at + bytes), or -1
__device__ __forceinline__ int lw_place(const LwSlot &cur, int need, int ring) {
    if (cur.at + cur.bytes + need <= ring) return cur.at + cur.bytes;
    return need <= cur.at ? 0 : -1;
}

// Lane 0: starts the copies of a row into its slot; all lanes fetch the single numbers behind the windows.
template <int G, bool kExact, bool kBackward>
__device__ __forceinline__ void lw_issue(const LwRow &r, const LwSlot &s, unsigned char *ring, uint64_t *mbar,
                                         const float *content, const float *grad_links, int L, int H, int K, bool wide) {
    if (r.nj <= 0) return;
    const int lane = threadIdx.x & 31;
    const float *const scores = content + (r.row * L + r.i + 1) * (int64_t)H;
    const float *const grad = kBackward ? grad_links + r.row * (int64_t)K : nullptr;
    const int n = r.nj * H, sc_whole = kExact ? n : lw_whole(s.front, n, true);
    const int grad_whole = kBackward ? lw_whole(s.skip, r.nj, wide) : 0;
    if (lane == 0) {
        const uint32_t mb = umma::smem_u32(mbar), base = umma::smem_u32(ring) + s.at;
        const uint32_t sc = sc_whole > 0 ? (s.front + sc_whole) * 4 : 0;
        const uint32_t win = kBackward && grad_whole > 0 ? (s.skip + grad_whole) * 4 : 0;
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(mb), "r"(sc + win) : "memory");
        if (sc) lw_bulk_load(base + s.window, scores - s.front, sc, mb);
        if (win) lw_bulk_load(base, grad - s.skip, win, mb);
    }
    if (kBackward) {
        float *w = reinterpret_cast<float *>(ring + s.at) + s.skip;
        for (int d = grad_whole + lane; d < r.nj; d += 32) w[d] = __ldg(grad + d);
    }
    if (!kExact) {
        float *w = reinterpret_cast<float *>(ring + s.at + s.window) + s.front;
        for (int x = sc_whole + lane; x < n; x += 32) w[x] = __ldg(scores + x);
    }
}

// sum or maximum over the lanes of a head group, in every lane: halving exchange, then each lane fetches its four
template <int G, bool kMax>
__device__ __forceinline__ void lw_reduce(float (&v)[4]) {
    const int lane = threadIdx.x & 31, g = lane & (G - 1);
    const auto op = [](float a, float b) { return kMax ? fmaxf(a, b) : a + b; };
    const bool up = lane & 16, up2 = lane & 8;
    float a = up ? v[0] : v[2], b = up ? v[1] : v[3];
    a = op(up ? v[2] : v[0], __shfl_xor_sync(0xffffffffu, a, 16));
    b = op(up ? v[3] : v[1], __shfl_xor_sync(0xffffffffu, b, 16));
    float c = op(up2 ? b : a, __shfl_xor_sync(0xffffffffu, up2 ? a : b, 8));
    if (G < 8) c = op(c, __shfl_xor_sync(0xffffffffu, c, 4));
    if (G < 4) c = op(c, __shfl_xor_sync(0xffffffffu, c, 2));
    if (G < 2) c = op(c, __shfl_xor_sync(0xffffffffu, c, 1));
#pragma unroll
    for (int k = 0; k < 4; k++) v[k] = __shfl_sync(0xffffffffu, c, (k >> 1) * 16 + (k & 1) * 8 + g);
}

// scores of places that are not allowed inside the span to -inf (each lane its own places)
template <int G, bool kExact>
__device__ __forceinline__ void lw_punch(const LwRow &r, float *buf, int H, const LwDead &dead) {
    for (int v = threadIdx.x & 31; v < r.nj * G; v += 32)
        if (dead(v / G)) lw_put<G, kExact>(buf, v, H, lb_ninf4());
}

// the four heads of lane group g of a row of [.., H], -inf for those that are not there
template <int G, bool kExact>
__device__ __forceinline__ float4 lw_heads(const float *p, int64_t row, int H, int g) {
    return lw_get<G, kExact>(p + row * H, g, H, -INFINITY);
}

// Runs f(N, partial, v) over a row's vectors: batches of kLwU * 32 without a condition inside, then the rest as one
// smaller batch in which lanes may lie behind the row's end.  v: the lane's first vector, the others 32 apart.
template <typename F>
__device__ __forceinline__ void lw_batches(int nvec, F f) {
    int v = threadIdx.x & 31;
    for (; v < (nvec & ~(32 * kLwU - 1)); v += 32 * kLwU) f(LwInt<kLwU>(), LwInt<0>(), v);
    const int left = nvec & (32 * kLwU - 1);
    if (left > 96) f(LwInt<4>(), LwInt<1>(), v);
    else if (left > 64) f(LwInt<3>(), LwInt<1>(), v);
    else if (left > 32) f(LwInt<2>(), LwInt<1>(), v);
    else if (left > 0) f(LwInt<1>(), LwInt<1>(), v);
}

// t = score + bias - r of N vectors, in log2 units (behind the row's end: the last vector's)
template <int G, bool kExact, int N, bool kPart>
__device__ __forceinline__ void lw_terms(float4 (&t)[N], const float *buf, int H, const float4 *table,
                                         const unsigned short *bucket, const float (&r)[4], int v, int nvec) {
    float4 c[N], b[N];
#pragma unroll
    for (int u = 0; u < N; u++) {
        const int x = kPart ? min(v + 32 * u, nvec - 1) : v + 32 * u;
        c[u] = lw_get<G, kExact>(buf, x, H, -INFINITY);
        // the head group of the clamped vector is the last one's and may be another: nothing of it is used
        b[u] = lw_bias<G>(table, bucket, x);
    }
    if (kPart) __syncwarp();   // the last vector is read by lanes that do not own it
#pragma unroll
    for (int u = 0; u < N; u++) t[u] = lb_shifted(c[u], b[u], r);
}
__device__ __forceinline__ float4 lw_exp2(float4 t) { return make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w)); }

// q_h = soft_h exp(g_h)
__device__ __forceinline__ float4 lw_gated(float4 soft, const float (&eg)[4]) {
    fmul2_rn(soft.x, soft.y, soft.x, soft.y, eg[0], eg[1]);
    fmul2_rn(soft.z, soft.w, soft.z, soft.w, eg[2], eg[3]);
    return soft;
}

// A link that the flush of the exponentials could have touched, from the terms' logarithms (g + z - lse, log2 units); top:
// what was taken from the gates
template <int G>
__device__ __noinline__ float lw_tiny_link(float a0, float a1, float a2, float a3, float top) {
    const float m = lb_max_over_heads<G>(fmaxf(fmaxf(a0, a1), fmaxf(a2, a3))), mm = m > -INFINITY ? m : 0.f;
    const float q = lb_over_heads<G>(ex2(a0 - mm) + ex2(a1 - mm) + ex2(a2 - mm) + ex2(a3 - mm));
    return fmaf(mm + lg2(q), kLn2, top);
}

// The link to an only successor: the log-sum-exp of the gates of the heads that have a sum, near 0 where the gates are
// log-probabilities, so that the 2^-22 of lg2 would be all of it.  Heads on lanes.
template <int G>
__device__ __noinline__ float lw_only_link(float4 gate, const float (&sum)[4], int H) {
    const int lane = threadIdx.x & 31;
    const float gates[4] = {gate.x, gate.y, gate.z, gate.w};
    float g = -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float o = __shfl_sync(0xffffffffu, sum[k] == 0.f ? -INFINITY : sum[k] > 0.f ? gates[k] : sum[k], lane / 4);
        if ((lane & 3) == k && lane < H) g = o;
    }
    const float m = warp_max(g), mm = m > -INFINITY ? m : 0.f;
    return mm + logf(warp_sum(expf(g - mm)));
}

// G_d p_h of a distance whose sum over the heads the 32-bit exponent has flushed: relative to its largest term (t, g2 in
// log2 units).  A link of -inf has no share, whatever its gradient is.
template <int G>
__device__ __noinline__ float4 lw_full_share(float4 t, const float (&g2)[4], float gd) {
    const float a[4] = {t.x + g2[0], t.y + g2[1], t.z + g2[2], t.w + g2[3]};
    const float m = lb_max_over_heads<G>(fmaxf(fmaxf(a[0], a[1]), fmaxf(a[2], a[3]))), mm = m > -INFINITY ? m : 0.f;
    const float4 p = make_float4(ex2(a[0] - mm), ex2(a[1] - mm), ex2(a[2] - mm), ex2(a[3] - mm));
    const float tot = lb_over_heads<G>((p.x + p.y) + (p.z + p.w)), k = gd / tot;
    return tot != 0.f ? make_float4(p.x * k, p.y * k, p.z * k, p.w * k) : make_float4(0.f, 0.f, 0.f, 0.f);
}

// What both kernels begin with: table, barriers, zeros.  Returns the bucket of distances that have none, -1 if all have.
template <int G, int NT>
__device__ __forceinline__ int lw_begin(const LwSmem &lay, unsigned char *sm, const LinksBias &lb, int H, int K) {
    const bool bad = lw_load_table<G, NT>(lb, reinterpret_cast<float *>(sm), reinterpret_cast<unsigned short *>(sm + lay.bucket), H, K);
    for (int x = threadIdx.x; x < kLwZeros / 16; x += NT)
        reinterpret_cast<float4 *>(sm + lay.zeros)[x] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (threadIdx.x < NT / 32) umma::mbar_init(reinterpret_cast<uint64_t *>(sm + lay.mbar) + threadIdx.x, 1);
    umma::fence_smem_to_async();
    return __syncthreads_or(bad) ? lb.n : -1;
}

// NG groups of four vertices at work in a CTA
template <int G, bool kExact, int NG>
__global__ void __launch_bounds__(NG * kLwRows * 32, NG == 2 ? 2 : 1)
lw_fwd_kernel(const float *__restrict__ content, const float *__restrict__ log_gates, LinksMask mk,
              const int2 *span, LinksBias lb, LwSmem lay, float *__restrict__ links,
              float *__restrict__ head_lse, int B, int L, int heads, int K) {
    const int H = kExact ? 4 * G : heads;
    extern __shared__ __align__(16) unsigned char lwsm[];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane & (G - 1);
    const float4 *const table = reinterpret_cast<const float4 *>(lwsm);
    const unsigned short *const bucket = reinterpret_cast<const unsigned short *>(lwsm + lay.bucket);
    unsigned char *const ring = lwsm + lay.rings + warp * lay.ring;
    uint64_t *const mbar = reinterpret_cast<uint64_t *>(lwsm + lay.mbar) + warp;
    const int none = lw_begin<G, NG * kLwRows * 32>(lay, lwsm, lb, H, K);
    pdl_wait();   // the spans
    const int groups = B * ((L + kLwRows - 1) / kLwRows), step = gridDim.x * NG;
    int group = warp / kLwRows * gridDim.x + blockIdx.x;
    LwPairs walk(group, step, B, L);
    LwRow r0 = lw_row(walk, L, mk, span), r1 = lw_row(walk, L, mk, span);
    lw_resolve(r0, L, K, mk);
    LwSlot s0 = lw_slot<G, kExact, false>(r0, L, H, K);
    lw_issue<G, kExact, false>(r0, s0, ring, mbar, content, nullptr, L, H, K, false);
    const auto gates_of = [&](const LwRow &r) {
        return r.exists ? lw_heads<G, kExact>(log_gates, r.row, H, g) : lb_ninf4();
    };
    float4 gate = gates_of(r0);
    uint32_t phase = 0;
    bool stalled = false;
    for (; group < groups; group += step) {
        if (r0.nj > 0) {
            stalled |= !umma::mbar_wait(mbar, phase, stalled ? 1 : kLwPolls);
            phase ^= 1;
        }
        if (!kExact) __syncwarp();   // the numbers that came singly
        // the next row on its way, where the ring has room for it beside this one
        lw_resolve(r1, L, K, mk);
        LwSlot s1 = lw_slot<G, kExact, false>(r1, L, H, K);
        s1.at = lw_place(s0, s1.bytes, lay.ring);
        const bool later = s1.at < 0;
        if (!later) lw_issue<G, kExact, false>(r1, s1, ring, mbar, content, nullptr, L, H, K, false);
        const float4 gate1 = gates_of(r1);
        const LwRow r2 = lw_row(walk, L, mk, span);
        if (r0.exists) {
            const int nvec = r0.nj * G;
            float *const buf = reinterpret_cast<float *>(ring + s0.at) + s0.front;
            const float *const src = content + (r0.row * L + r0.i + 1) * (int64_t)H;
            const LwDead dead{r0.holes ? mk.nonpad + r0.row + 1 : nullptr, bucket, none};   // b * L + i + 1
            if (dead.any()) {
                lw_punch<G, kExact>(r0, buf, H, dead);
                __syncwarp();
            }
            // r_h in log2 units
            float r[4] = {0.f, 0.f, 0.f, 0.f}, sum[4] = {0.f, 0.f, 0.f, 0.f};
            bool bad = false;
            if (nvec > 0) {
                const float4 c = lw_get<G, kExact>(buf, g, H, 0.f), b0 = lw_bias<G>(table, bucket, g);
                r[0] = fmaf(c.x, kLog2e, b0.x);
                r[1] = fmaf(c.y, kLog2e, b0.y);
                r[2] = fmaf(c.z, kLog2e, b0.z);
                r[3] = fmaf(c.w, kLog2e, b0.w);
                bad = !(fabsf(r[0]) < INFINITY && fabsf(r[1]) < INFINITY && fabsf(r[2]) < INFINITY && fabsf(r[3]) < INFINITY);
                __syncwarp();   // before the nearest successor's place is written over
            }
            lw_batches(nvec, [&](auto n, auto part, int v) {
                constexpr int N = decltype(n)::value;
                constexpr bool kPart = decltype(part)::value;
                float4 t[N];
                lw_terms<G, kExact, N, kPart>(t, buf, H, table, bucket, r, v, nvec);
#pragma unroll
                for (int u = 0; u < N; u++) {
                    const float4 e = lw_exp2(t[u]);
                    if (!kPart || v + 32 * u < nvec) {
                        lw_put<G, kExact>(buf, v + 32 * u, H, e);
                        fadd2_rn(sum[0], sum[1], sum[0], sum[1], e.x, e.y);
                        fadd2_rn(sum[2], sum[3], sum[2], sum[3], e.z, e.w);
                    }
                }
            });
            bad |= !(fmaxf(fmaxf(sum[0], sum[1]), fmaxf(sum[2], sum[3])) < kLbHuge) ||
                   !(sum[0] + sum[1] + sum[2] + sum[3] < INFINITY);
            if (__any_sync(0xffffffffu, bad)) {   // the exact maximum of each head takes the place of r_h
                float m[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                for (int v = lane; v < nvec; v += 32)
                    if (!dead(v / G)) {
                        const float4 c = lw_get<G, kExact>(src, v, H, -INFINITY), t = lw_bias<G>(table, bucket, v);
                        m[0] = fmaxf(m[0], fmaf(c.x, kLog2e, t.x));
                        m[1] = fmaxf(m[1], fmaf(c.y, kLog2e, t.y));
                        m[2] = fmaxf(m[2], fmaf(c.z, kLog2e, t.z));
                        m[3] = fmaxf(m[3], fmaf(c.w, kLog2e, t.w));
                    }
                __syncwarp();
                lw_reduce<G, true>(m);
                sum[0] = sum[1] = sum[2] = sum[3] = 0.f;
#pragma unroll
                for (int k = 0; k < 4; k++) r[k] = m[k] > -INFINITY ? m[k] : 0.f;
                for (int v = lane; v < nvec; v += 32) {
                    float4 e = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (!dead(v / G)) {
                        const float4 t = lb_shifted(lw_get<G, kExact>(src, v, H, -INFINITY), lw_bias<G>(table, bucket, v), r);
                        e = make_float4(ex2(t.x), ex2(t.y), ex2(t.z), ex2(t.w));
                        fadd2_rn(sum[0], sum[1], sum[0], sum[1], e.x, e.y);
                        fadd2_rn(sum[2], sum[3], sum[2], sum[3], e.z, e.w);
                    }
                    lw_put<G, kExact>(buf, v, H, e);
                }
                __syncwarp();
            }
            lw_reduce<G, false>(sum);
            // f_h = exp(g_h) / S_h; a head without a finite score takes no part
            float g2[4], f[4], ls[4];
            const float top = lb_gates<G>(gate, g2);
            bool rare = false;
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const bool some = sum[k] != 0.f;
                ls[k] = some ? lg2(sum[k]) : INFINITY;
                f[k] = some ? __fdividef(ex2(g2[k]), sum[k]) : 0.f;
                rare |= some && lb_rare(f[k], g2[k]);
            }
            const float enough = __any_sync(0xffffffffu, rare) ? INFINITY : kLbTiny;   // of the links' sums
            if (head_lse && lane < G) {
                float4 o;
                o.x = ls[0] == INFINITY ? -INFINITY : r[0] + ls[0];
                o.y = ls[1] == INFINITY ? -INFINITY : r[1] + ls[1];
                o.z = ls[2] == INFINITY ? -INFINITY : r[2] + ls[2];
                o.w = ls[3] == INFINITY ? -INFINITY : r[3] + ls[3];
                lw_put<G, kExact>(head_lse + r0.row * H, g, H, o);
            }
            float *const out = links + r0.row * (int64_t)K;
            if (r0.nj == 1) {
                const float link = lw_only_link<G>(gate, sum, H);
                if (lane == 0) out[0] = link;
            }
            lw_batches(r0.nj == 1 ? 0 : nvec, [&](auto n, auto part, int v) {
                constexpr int N = decltype(n)::value;
                constexpr bool kPart = decltype(part)::value;
                float q[N];
                float least = 1.f;
#pragma unroll
                for (int u = 0; u < N; u++) {
                    const float4 e = lw_get<G, kExact>(buf, kPart ? min(v + 32 * u, nvec - 1) : v + 32 * u, H, 0.f);
                    q[u] = lb_over_heads<G>(fmaf(e.x, f[0], e.y * f[1]) + fmaf(e.z, f[2], e.w * f[3]));
                    if (kPart && v + 32 * u >= nvec) q[u] = 1.f;
                    least = fminf(least, q[u]);
                }
                const bool tiny = __any_sync(0xffffffffu, least < enough);
#pragma unroll
                for (int u = 0; u < N; u++) q[u] = fmaf(lg2(q[u]), kLn2, top);
                if (tiny) {
                    for (int u = 0; u < N; u++) {
                        const int x = v + 32 * u;
                        float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                        if (x < nvec && !dead(x / G)) {   // log2 of e f without the exponential's flush
                            const float4 z = lb_shifted(lw_get<G, kExact>(src, x, H, -INFINITY), lw_bias<G>(table, bucket, x), r);
                            if (ls[0] != INFINITY) t[0] = z.x + (g2[0] - ls[0]);
                            if (ls[1] != INFINITY) t[1] = z.y + (g2[1] - ls[1]);
                            if (ls[2] != INFINITY) t[2] = z.z + (g2[2] - ls[2]);
                            if (ls[3] != INFINITY) t[3] = z.w + (g2[3] - ls[3]);
                        }
                        const float link = lw_tiny_link<G>(t[0], t[1], t[2], t[3], top);
                        if (g == 0 && x < nvec) out[x / G] = link;
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < N; u++)
                        if (g == 0 && (!kPart || v + 32 * u < nvec)) out[(v + 32 * u) / G] = q[u];
                }
            });
            for (int d = r0.nj + lane; d < K; d += 32) out[d] = -INFINITY;
        }
        // this row's place may be copied over from here on
        umma::fence_smem_to_async();
        __syncwarp();
        if (later) {
            s1.at = 0;
            lw_issue<G, kExact, false>(r1, s1, ring, mbar, content, nullptr, L, H, K, false);
        }
        r0 = r1;
        s0 = s1;
        r1 = r2;
        gate = gate1;
    }
    if (stalled && lb.status) atomicOr(lb.status, DAT_STATUS_STALLED);
}

// Backward.  With q_h = soft_h exp(g_h) and w_d = G_d / sum_h q_h the gradient of a score is q_h w_d - soft_h S_h: the
// scores' place holds soft and then the gradient itself, which the four rows' warps add to their sums by distance (registers of the 128
// threads, UA vectors each).
template <int G, bool kExact, int UA, int NG>
__global__ void __launch_bounds__(NG * kLwRows * 32, UA <= 4 ? 2 : 1)
lw_bwd_kernel(const float *__restrict__ grad_links, const float *__restrict__ content,
              const float *__restrict__ log_gates, const float *__restrict__ head_lse, LinksMask mk,
              const int2 *span, LinksBias lb, LwSmem lay, float *__restrict__ grad_content,
              float *__restrict__ grad_log_gates, float *__restrict__ part, int B, int L, int heads, int K) {
    const int H = kExact ? 4 * G : heads;
    const bool whole = kExact || (H & 3) == 0;   // rows of 16-byte pieces
    extern __shared__ __align__(16) unsigned char lwsm[];
    __shared__ int2 row_at[NG * kLwRows];   // where a row's gradient lies (bytes from lwsm), its vectors
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane & (G - 1);
    const float4 *const table = reinterpret_cast<const float4 *>(lwsm);
    const unsigned short *const bucket = reinterpret_cast<const unsigned short *>(lwsm + lay.bucket);
    unsigned char *const ring = lwsm + lay.rings + warp * lay.ring;
    uint64_t *const mbar = reinterpret_cast<uint64_t *>(lwsm + lay.mbar) + warp;
    const uint32_t zeros = umma::smem_u32(lwsm + lay.zeros);
    const bool wide = (reinterpret_cast<uintptr_t>(grad_links) & 15) == 0;
    const int set = warp / kLwRows, set_tid = tid - set * (kLwRows * 32);
    const auto set_sync = [&] { asm volatile("bar.sync %0, %1;" ::"r"(set + 1), "n"(kLwRows * 32) : "memory"); };
    const int none = lw_begin<G, NG * kLwRows * 32>(lay, lwsm, lb, H, K);
    pdl_trigger();
    const int groups = B * ((L + kLwRows - 1) / kLwRows), step = gridDim.x * NG;
    int group = blockIdx.x * NG + set;
    LwEnds walk(group, step, B, L);
    LwRow r0 = lw_row(walk, L, mk, span), r1 = lw_row(walk, L, mk, span);
    lw_resolve(r0, L, K, mk);
    LwSlot s0 = lw_slot<G, kExact, true>(r0, L, H, K);
    lw_issue<G, kExact, true>(r0, s0, ring, mbar, content, grad_links, L, H, K, wide);
    const auto of_row = [&](const float *p, const LwRow &r) {
        return r.exists ? lw_heads<G, kExact>(p, r.row, H, g) : lb_ninf4();
    };
    float4 lse = of_row(head_lse, r0), gate = of_row(log_gates, r0);
    float4 acc[UA];
#pragma unroll
    for (int u = 0; u < UA; u++) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    uint32_t phase = 0;
    bool stalled = false;
    for (; group < groups; group += step) {
        if (r0.nj > 0) {
            stalled |= !umma::mbar_wait(mbar, phase, stalled ? 1 : kLwPolls);
            phase ^= 1;
        }
        __syncwarp();
        const float4 lse1 = of_row(head_lse, r1), gate1 = of_row(log_gates, r1);
        const LwRow r2 = lw_row(walk, L, mk, span);
        const int nvec = r0.nj * G;
        float *const buf = reinterpret_cast<float *>(ring + s0.at + s0.window) + s0.front;
        const float *const src = content + (r0.row * L + r0.i + 1) * (int64_t)H;
        const LwDead dead{r0.holes ? mk.nonpad + r0.row + 1 : nullptr, bucket, none};
        float *const weight = reinterpret_cast<float *>(ring + s0.at) + s0.skip;   // G_d, then w_d
        if (dead.any()) {
            lw_punch<G, kExact>(r0, buf, H, dead);
            __syncwarp();
        }
        const float ls[4] = {lb_lse(lse.x), lb_lse(lse.y), lb_lse(lse.z), lb_lse(lse.w)};
        float g2[4];
        lb_gates<G>(gate, g2);
        const float eg[4] = {ex2(g2[0]), ex2(g2[1]), ex2(g2[2]), ex2(g2[3])};
        float S[4] = {0.f, 0.f, 0.f, 0.f};
        lw_batches(nvec, [&](auto n, auto part, int v) {
            constexpr int N = decltype(n)::value;
            constexpr bool kPart = decltype(part)::value;
            float4 t[N], q[N];
            float w[N];
            lw_terms<G, kExact, N, kPart>(t, buf, H, table, bucket, ls, v, nvec);
            bool tiny = false;
#pragma unroll
            for (int u = 0; u < N; u++) {
                const bool in = !kPart || v + 32 * u < nvec;
                if (kPart && !in) t[u] = lb_ninf4();
                w[u] = in ? weight[(v + 32 * u) / G] : 0.f;
            }
#pragma unroll
            for (int u = 0; u < N; u++) {
                const bool in = !kPart || v + 32 * u < nvec;
                const float4 soft = lw_exp2(t[u]);
                q[u] = lw_gated(soft, eg);
                const float tot = lb_over_heads<G>((q[u].x + q[u].y) + (q[u].z + q[u].w));
                if (in) {
                    lw_put<G, kExact>(buf, v + 32 * u, H, soft);
                    tiny |= !(tot >= kLbTiny);
                }
                if (tot >= kLbTiny) w[u] = __fdividef(w[u], tot);
            }
            if (__any_sync(0xffffffffu, tiny)) {
#pragma unroll
                for (int u = 0; u < N; u++) {
                    const float tot = lb_over_heads<G>((q[u].x + q[u].y) + (q[u].z + q[u].w));
                    const float4 p = lw_full_share<G>(t[u], g2, w[u]);
                    if (!(tot >= kLbTiny)) {   // the same in all lanes of a distance
                        S[0] += p.x;
                        S[1] += p.y;
                        S[2] += p.z;
                        S[3] += p.w;
                        q[u] = make_float4(0.f, 0.f, 0.f, 0.f);
                        w[u] = __uint_as_float(kLwFull);   // the second pass takes the share in full again
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < N; u++) {
                if (g == 0 && (!kPart || v + 32 * u < nvec)) weight[(v + 32 * u) / G] = w[u];
                const float k = __float_as_uint(w[u]) == kLwFull ? 0.f : w[u];
                ffma2_rn(S[0], S[1], q[u].x, q[u].y, k, k);
                ffma2_rn(S[2], S[3], q[u].z, q[u].w, k, k);
            }
        });
        __syncwarp();
        // the next row on its way: the gradient of the row before this one has left its place
        lw_resolve(r1, L, K, mk);
        LwSlot s1 = lw_slot<G, kExact, true>(r1, L, H, K);
        s1.at = lw_place(s0, s1.bytes, lay.ring);
        const bool later = s1.at < 0;
        if (!later) {
            lw_bulk_read();
            __syncwarp();
            lw_issue<G, kExact, true>(r1, s1, ring, mbar, content, grad_links, L, H, K, wide);
        }
        if (r0.exists) {
            lw_reduce<G, false>(S);
            if (lane < G)
                lw_put<G, kExact>(grad_log_gates + r0.row * H, g, H, make_float4(S[0], S[1], S[2], S[3]));
            lw_batches(nvec, [&](auto n, auto part, int v) {
                constexpr int N = decltype(n)::value;
                constexpr bool kPart = decltype(part)::value;
                float4 o[N];
                float w[N];
#pragma unroll
                for (int u = 0; u < N; u++) {
                    const int x = kPart ? min(v + 32 * u, nvec - 1) : v + 32 * u;
                    o[u] = lw_get<G, kExact>(buf, x, H, 0.f);
                    w[u] = weight[x / G];
                }
                if (kPart) __syncwarp();   // the last vector is read by lanes that do not own it
                bool full = false;
#pragma unroll
                for (int u = 0; u < N; u++) full |= __float_as_uint(w[u]) == kLwFull;
                if (__any_sync(0xffffffffu, full)) {   // see the first pass
                    for (int u = 0; u < N; u++) {
                        const int x = min(v + 32 * u, nvec - 1);
                        const bool out = dead(x / G);
                        const float4 t = out ? lb_ninf4() : lb_shifted(lw_get<G, kExact>(src, x, H, -INFINITY), lw_bias<G>(table, bucket, x), ls);
                        const float4 p = lw_full_share<G>(t, g2, __ldg(grad_links + r0.row * (int64_t)K + x / G));
                        float4 k = lb_grad(o[u], lw_gated(o[u], eg), w[u], S);
                        if (__float_as_uint(w[u]) == kLwFull)
                            k = make_float4(fmaf(-S[0], o[u].x, p.x), fmaf(-S[1], o[u].y, p.y), fmaf(-S[2], o[u].z, p.z),
                                            fmaf(-S[3], o[u].w, p.w));
                        if (out) k = make_float4(0.f, 0.f, 0.f, 0.f);   // also beside NaN
                        if (v + 32 * u < nvec) lw_put<G, kExact>(buf, v + 32 * u, H, k);
                    }
                } else {
#pragma unroll
                    for (int u = 0; u < N; u++) {
                        o[u] = lb_grad(o[u], lw_gated(o[u], eg), w[u], S);
                        if (!kPart || v + 32 * u < nvec) lw_put<G, kExact>(buf, v + 32 * u, H, o[u]);
                    }
                }
            });
            umma::fence_smem_to_async();
            __syncwarp();
            float *const dense = grad_content + r0.row * (int64_t)L * H;
            const int before = (r0.i + 1) * H, total = L * H, behind = before + r0.nj * H;
            if (whole) {
                if (lane == 0 && nvec > 0) lw_bulk_store(dense + before, umma::smem_u32(buf), (behind - before) * 4);
            } else {
                for (int x = lane; x < behind - before; x += 32) dense[before + x] = buf[x];
            }
            // the places of the dense row that no valid successor has
            lw_zero<!kExact>(dense, before, zeros);
            lw_zero<!kExact>(dense + behind, total - behind, zeros);
            lw_bulk_commit();
        }
        if (part) {
            if (lane == 0) row_at[warp] = make_int2((int)(reinterpret_cast<unsigned char *>(buf) - lwsm), nvec);
            set_sync();
#pragma unroll
            for (int w = 0; w < kLwRows; w++) {
                const int2 at = row_at[set * kLwRows + w];
                const float *const dc = reinterpret_cast<const float *>(lwsm + at.x);
#pragma unroll
                for (int u = 0; u < UA; u++) {
                    if (u * (kLwRows * 32) >= at.y) break;
                    const int v = set_tid + u * (kLwRows * 32);
                    if (v < at.y) {
                        const float4 o = lw_get<G, kExact>(dc, v, H, 0.f);
                        fadd2_rn(acc[u].x, acc[u].y, acc[u].x, acc[u].y, o.x, o.y);
                        fadd2_rn(acc[u].z, acc[u].w, acc[u].z, acc[u].w, o.z, o.w);
                    }
                }
            }
            set_sync();
        }
        if (later) {
            lw_bulk_read();
            umma::fence_smem_to_async();
            __syncwarp();
            s1.at = 0;
            lw_issue<G, kExact, true>(r1, s1, ring, mbar, content, grad_links, L, H, K, wide);
        }
        r0 = r1;
        s0 = s1;
        r1 = r2;
        lse = lse1;
        gate = gate1;
    }
    lw_bulk_read();
    if (stalled && lb.status) atomicOr(lb.status, DAT_STATUS_STALLED);
    if (part) {
        // the groups' sums together, through the rings, whose copies have all come and gone
        float4 *const sums = reinterpret_cast<float4 *>(lwsm + lay.rings);
        __syncthreads();
#pragma unroll
        for (int u = 0; u < UA; u++) {
            const int v = set_tid + u * (kLwRows * 32);
            if (set > 0 && v < K * G) sums[(set - 1) * K * G + v] = acc[u];
        }
        __syncthreads();
        if (set == 0) {
            float *const p = part + (size_t)blockIdx.x * K * H;
#pragma unroll
            for (int u = 0; u < UA; u++) {
                const int v = set_tid + u * (kLwRows * 32);
                if (v < K * G) {
#pragma unroll
                    for (int q = 0; q < NG - 1; q++) {
                        const float4 o = sums[q * K * G + v];
                        acc[u].x += o.x;
                        acc[u].y += o.y;
                        acc[u].z += o.z;
                        acc[u].w += o.w;
                    }
                    lw_put<G, kExact>(p, v, H, acc[u]);
                }
            }
        }
    }
}

// What the kernel before has written is read by coherent loads (__ldcg) in the following three, which may have begun beside
// it: the read-only path is for what nobody writes while a kernel runs.
// by_distance[x] = sum of part[n][x] over the n CTAs, x = d * H + h: 32 columns per CTA, 16 lanes of rows each
constexpr int kLbSumCols = 32, kLbSumLanes = 16;
__global__ void __launch_bounds__(kLbSumCols * kLbSumLanes)
lb_sum_kernel(const float *part, double *by_distance, int n, int KH) {
    __shared__ double lane_s[kLbSumLanes][kLbSumCols];
    const int c = threadIdx.x % kLbSumCols, q = threadIdx.x / kLbSumCols, x = blockIdx.x * kLbSumCols + c;
    double acc = 0.0;
    pdl_trigger();
    pdl_wait();
    if (x < KH) {
#pragma unroll 8
        for (int k = q; k < n; k += kLbSumLanes) acc += (double)__ldcg(part + (size_t)k * KH + x);
    }
    lane_s[q][c] = acc;
    __syncthreads();
    if (q == 0 && x < KH) {
#pragma unroll
        for (int k = 1; k < kLbSumLanes; k++) acc += lane_s[k][c];
        by_distance[x] = acc;
    }
}

// The same sums from the dense gradient: by_distance[d * H + h] = sum of dc[b,i,i+1+d,h] over the vertices (b,i)
__global__ void __launch_bounds__(kLbSumCols * kLbSumLanes)
lb_diag_kernel(const float *grad_content, double *by_distance, int B, int L, int H, int K) {
    __shared__ double lane_s[kLbSumLanes][kLbSumCols];
    const int c = threadIdx.x % kLbSumCols, q = threadIdx.x / kLbSumCols, x = blockIdx.x * kLbSumCols + c;
    double acc = 0.0;
    pdl_trigger();
    pdl_wait();
    if (x < K * H) {
        const int n = L - 1 - x / H;   // vertices that have a successor at this distance
        for (int b = 0; b < B; b++) {
            const float *p = grad_content + ((int64_t)b * L * L + 1) * H + x;
#pragma unroll 8
            for (int i = q; i < n; i += kLbSumLanes) acc += (double)__ldcg(p + (int64_t)i * (L + 1) * H);
        }
    }
    lane_s[q][c] = acc;
    __syncthreads();
    if (q == 0 && x < K * H) {
#pragma unroll
        for (int k = 1; k < kLbSumLanes; k++) acc += lane_s[k][c];
        by_distance[x] = acc;
    }
}

// grad_table[k, h]: one CTA per bucket, the distances dealt to P lanes of a head
constexpr int kLbJoinThreads = 256;
__global__ void __launch_bounds__(kLbJoinThreads)
lb_join_kernel(const double *by_distance, const int64_t *__restrict__ bucket, float *__restrict__ grad_table, int H, int K) {
    __shared__ double lane_s[kLbJoinThreads];
    const int k = blockIdx.x, P = kLbJoinThreads / H, h = threadIdx.x % H, p = threadIdx.x / H;
    double acc = 0.0;
    pdl_wait();
    if (p < P) {
#pragma unroll 8
        for (int d = p; d < K; d += P) {
            const double v = __ldcg(by_distance + (size_t)d * H + h);
            acc += __ldg(bucket + d) == k ? v : 0.0;
        }
    }
    lane_s[threadIdx.x] = acc;
    __syncthreads();
    if (p == 0) {
        for (int q = 1; q < P; q++) acc += lane_s[q * H + h];
        grad_table[(size_t)k * H + h] = (float)acc;
    }
}

// shared memory of a CTA per vertex with NT threads, and the partial bands of the backward's CTAs by size alone: at most two
// CTAs per SM with a warp per vertex, as many as their shared memory lets run (and 16) with a CTA per vertex, where the head
// count has that form; the kernels of links.cu leave none
static size_t lb_smem(int K, int H, int NT) { return ((size_t)3 * K * H + 2 * (NT / 32) * H) * sizeof(float); }
constexpr int kLbMaxPerSm = 16;
static bool lb_vectors(int K, int H) {
    const int G = H / 4;
    return H % 4 == 0 && (G == 1 || G == 2 || G == 4 || G == 8) && (int64_t)K * G <= kLbMaxVec;
}
static int lb_bands_per_sm(int K, int H, const DeviceInfo &di) {
    const int warp = H <= 32 && (int64_t)K * lw_lanes(H) <= kLwMaxVec ? 2 : 0;
    if (!lb_vectors(K, H)) return warp;
    const int64_t fit = di.max_smem_optin / (int64_t)lb_smem(K, H, 128);
    return fit > kLbMaxPerSm ? kLbMaxPerSm : fit > 2 ? (int)fit : 2;
}

// a warp per vertex: by size alone, so that a forward and its backward agree on who fills the spans
static bool lw_fits(int K, int H, int n, const DeviceInfo &di) {
    return H <= 32 && (int64_t)K * lw_lanes(H) <= kLwMaxVec && (int64_t)n * 4 * lw_lanes(H) <= kLwMaxTable &&
           lw_smem(K, H, n, 2 * kLwRows, lw_one(di)).ring >= lw_row_bytes(K, H);
}

// the kernels of this file: a warp or a CTA per vertex, by size, on 16-byte boundaries
static bool lb_own_form(int heads, int translen, int n, const DeviceInfo &di, const void *a, const void *b, const void *c,
                        const void *d) {
    return (lw_fits(translen, heads, n, di) || lb_vectors(translen, heads)) &&
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

struct LbArgs {
    const float *grad_links, *content, *log_gates, *head_lse_in;
    LinksMask mk;
    LinksBias lb;
    int2 *span;
    bool after;   // the kernel that fills the spans has just been launched
    float *links, *head_lse, *grad_content, *grad_log_gates, *part;
    int B, L, H, K;
};

template <int G, int NT, int U>
static int lb_launch(const LbArgs &a, bool backward, int &grid, cudaStream_t st, const DeviceInfo &di, const char *who) {
    const int H = 4 * G;
    const int64_t rows = (int64_t)a.B * a.L;
    const size_t smem = lb_smem(a.K, H, NT);
    if (!backward) {
        if (int rc = lb_grid(lb_fwd_kernel<G, NT, U>, NT, smem, rows, di, grid, who)) return rc;
        lb_fwd_kernel<G, NT, U><<<grid, NT, smem, st>>>(a.content, a.log_gates, a.mk, a.lb, a.links, a.head_lse, a.B, a.L, a.K);
    } else {
        if (int rc = lb_grid(lb_bwd_kernel<G, NT, U>, NT, smem, rows, di, grid, who)) return rc;
        const int most = di.sm_count * lb_bands_per_sm(a.K, a.H, di);
        if (grid > most) grid = most;
        lb_bwd_kernel<G, NT, U><<<grid, NT, smem, st>>>(a.grad_links, a.content, a.log_gates, a.head_lse_in, a.mk, a.lb,
                                                        a.grad_content, a.grad_log_gates, a.part, a.B, a.L, a.K);
    }
    return check_launch(who);
}

// CTAs of NG groups, `per_sm` of them to an SM
template <int NG, typename F, typename... Args>
static int lw_start(F kernel, int per_sm, const LbArgs &a, int &parts, cudaStream_t st, const DeviceInfo &di,
                    const char *who, LwSmem &lay, Args... args) {
    const int64_t groups = (int64_t)a.B * ((a.L + kLwRows - 1) / kLwRows);
    const int smem = per_sm > 1 ? lw_two(di) : lw_one(di);
    lay = lw_smem(a.K, a.H, a.lb.n, NG * kLwRows, smem);
    int64_t n = (int64_t)di.sm_count * per_sm;
    if (n > (groups + NG - 1) / NG) n = (groups + NG - 1) / NG;
    parts = (int)n;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) == cudaSuccess) {
        if (a.after) launch_after(kernel, (unsigned)n, NG * kLwRows * 32, smem, st, 1, args...);
        else kernel<<<(unsigned)n, NG * kLwRows * 32, smem, st>>>(args...);
    }
    return check_launch(who);
}
template <int G, bool kExact>
static int lw_launch(const LbArgs &a, bool backward, int &parts, cudaStream_t st, const DeviceInfo &di, const char *who) {
    const int row = lw_row_bytes(a.K, a.H), nvec = a.K * G;
    const int two = lw_smem(a.K, a.H, a.lb.n, 2 * kLwRows, lw_two(di)).ring;     // rings of eight warps, two CTAs per SM
    const int one = lw_smem(a.K, a.H, a.lb.n, 3 * kLwRows, lw_one(di)).ring;     // of twelve, one CTA
    LwSmem lay;
    const auto fwd = [&](auto kernel, auto ng, int per_sm) {
        return lw_start<decltype(ng)::value>(kernel, per_sm, a, parts, st, di, who, lay, a.content, a.log_gates, a.mk, a.span,
                                             a.lb, std::ref(lay), a.links, a.head_lse, a.B, a.L, a.H, a.K);
    };
    const auto bwd = [&](auto kernel, auto ng, int per_sm) {
        return lw_start<decltype(ng)::value>(kernel, per_sm, a, parts, st, di, who, lay, a.grad_links, a.content, a.log_gates,
                                             a.head_lse_in, a.mk, a.span, a.lb, std::ref(lay), a.grad_content,
                                             a.grad_log_gates, a.part, a.B, a.L, a.H, a.K);
    };
    // Two CTAs per SM, of eight warps, where their rings hold the longest row; else one of twelve; longer rows leave room
    // for eight.  Forward alone in a graph, 16 against 12 warps per SM: 16 graphs of 1024 vertices and 8 heads, bands of 256,
    // 300, 340 and 380 (the largest that fits) 39 / 43 / 47 / 49 against 43 / 47 / 49 / 53 us; 64 of 512 and 4 heads 49
    // against 55; 32 of 512, 12 heads and a band of 200 64 against 66, 16 heads and bands of 150 and 190 45 / 51 against 47 / 53.
    if (!backward) {
        if (two >= row) return fwd(lw_fwd_kernel<G, kExact, 2>, LwInt<2>(), 2);
        if (one >= row) return fwd(lw_fwd_kernel<G, kExact, 3>, LwInt<3>(), 1);
        return fwd(lw_fwd_kernel<G, kExact, 2>, LwInt<2>(), 1);
    }
    if (nvec <= 4 * kLwRows * 32 && two >= row) return bwd(lw_bwd_kernel<G, kExact, 4, 2>, LwInt<2>(), 2);
    if (nvec <= 8 * kLwRows * 32 && one >= row) return bwd(lw_bwd_kernel<G, kExact, 8, 3>, LwInt<3>(), 1);
    return bwd(lw_bwd_kernel<G, kExact, 16, 2>, LwInt<2>(), 1);
}
static int lw_run(const LbArgs &a, bool backward, int &parts, cudaStream_t st, const DeviceInfo &di, const char *who) {
    switch (lw_lanes(a.H)) {
        case 1: return a.H == 4 ? lw_launch<1, true>(a, backward, parts, st, di, who) : lw_launch<1, false>(a, backward, parts, st, di, who);
        case 2: return a.H == 8 ? lw_launch<2, true>(a, backward, parts, st, di, who) : lw_launch<2, false>(a, backward, parts, st, di, who);
        case 4: return a.H == 16 ? lw_launch<4, true>(a, backward, parts, st, di, who) : lw_launch<4, false>(a, backward, parts, st, di, who);
        default: return a.H == 32 ? lw_launch<8, true>(a, backward, parts, st, di, who) : lw_launch<8, false>(a, backward, parts, st, di, who);
    }
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

static int lb_run(const LbArgs &a, bool backward, int &grid, cudaStream_t st, const DeviceInfo &di, const char *who) {
    if (lw_fits(a.K, a.H, a.lb.n, di)) return lw_run(a, backward, grid, st, di, who);
    switch (a.H / 4) {
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
    DAT_REQUIRE((int64_t)bsz * prelen <= 0x3fffffff, DAT_ERR_UNSUPPORTED, "%s: bsz*prelen = %lld exceeds 2^30-1", who,
                (long long)bsz * prelen);
    return DAT_OK;
}

}  // namespace dat

extern "C" {

size_t dat_links_bias_workspace_bytes(int bsz, int prelen, int heads, int translen) {
    using namespace dat;
    if (bsz < 0 || prelen < 1 || heads < 1 || translen < 1) return 0;
    DeviceInfo di;
    if (!device_info(&di)) return 0;
    int64_t n = (int64_t)di.sm_count * lb_bands_per_sm(translen, heads, di);
    const int64_t rows = (int64_t)bsz * prelen + 3;   // a CTA per vertex, or groups of up to four in CTAs of three
    if (n > rows) n = rows;
    return (size_t)translen * heads * (sizeof(double) + (size_t)n * sizeof(float)) + 16;
}

int dat_links_from_heads_biased(const float *content, const float *log_gates, const float *bias_table,
                                const int64_t *buckets, int num_buckets, const int64_t *bound_end,
                                const unsigned char *nonpad, float *links, float *head_lse, int32_t *spans,
                                int32_t *status, int bsz, int prelen, int heads, int translen, void *stream) {
    using namespace dat;
    const char *who = "dat_links_from_heads_biased";
    if (int rc = lb_check(who, bias_table, buckets, num_buckets, bsz, prelen, heads, translen)) return rc;
    if (bsz == 0) return DAT_OK;
    DAT_REQUIRE(content && log_gates && links && (spans || !nonpad), DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const LinksMask mk{bound_end, nonpad};
    const LinksBias lb{bias_table, buckets, num_buckets, status};
    const bool after = nonpad && lw_fits(translen, heads, num_buckets, di);
    if (after) {
        lw_span_kernel<<<(unsigned)bsz, 128, 0, st>>>(nonpad, reinterpret_cast<int2 *>(spans), prelen);
        if (int rc = check_launch(who)) return rc;
    }
    if (lb_own_form(heads, translen, num_buckets, di, content, log_gates, head_lse, nullptr)) {
        LbArgs a{};
        a.content = content;
        a.log_gates = log_gates;
        a.mk = mk;
        a.lb = lb;
        a.span = const_cast<int2 *>(reinterpret_cast<const int2 *>(spans));
        a.links = links;
        a.head_lse = head_lse;
        a.after = after;
        a.B = bsz;
        a.L = prelen;
        a.H = heads;
        a.K = translen;
        int grid;
        return lb_run(a, false, grid, st, di, who);
    }
    return links_fwd_rows<true>(content, log_gates, mk, lb, links, head_lse, bsz, prelen, heads, translen, st, di, who);
}

int dat_links_from_heads_biased_backward(const float *grad_links, const float *content, const float *log_gates,
                                         const float *bias_table, const int64_t *buckets, int num_buckets,
                                         const float *links, const float *head_lse, const int64_t *bound_end,
                                         const unsigned char *nonpad, const int32_t *spans, float *grad_content,
                                         float *grad_log_gates, float *grad_bias_table, void *workspace, int32_t *status,
                                         int bsz, int prelen, int heads, int translen, void *stream) {
    using namespace dat;
    const char *who = "dat_links_from_heads_biased_backward";
    if (int rc = lb_check(who, bias_table, buckets, num_buckets, bsz, prelen, heads, translen)) return rc;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bsz == 0) {
        if (grad_bias_table) cudaMemsetAsync(grad_bias_table, 0, (size_t)num_buckets * heads * sizeof(float), st);
        return check_launch(who);
    }
    DAT_REQUIRE(grad_links && content && log_gates && links && head_lse && grad_content && grad_log_gates &&
                    (workspace || !grad_bias_table) && (spans || !nonpad),
                DAT_ERR_BAD_ARG, "%s: null pointer", who);
    DeviceInfo di;
    if (!device_info(&di)) return DAT_ERR_NO_DEVICE;
    const LinksMask mk{bound_end, nonpad};
    const LinksBias lb{bias_table, buckets, num_buckets, status};
    const int KH = translen * heads;
    double *sums = static_cast<double *>(workspace);
    const unsigned sgrid = (unsigned)((KH + kLbSumCols - 1) / kLbSumCols);
    constexpr int kSum = kLbSumCols * kLbSumLanes;
    if (lb_own_form(heads, translen, num_buckets, di, content, log_gates, head_lse, grad_content) &&
        (reinterpret_cast<uintptr_t>(grad_log_gates) & 15) == 0) {
        LbArgs a{};
        a.grad_links = grad_links;
        a.content = content;
        a.log_gates = log_gates;
        a.head_lse_in = head_lse;
        a.mk = mk;
        a.lb = lb;
        a.span = const_cast<int2 *>(reinterpret_cast<const int2 *>(spans));
        a.grad_content = grad_content;
        a.grad_log_gates = grad_log_gates;
        a.part = grad_bias_table ? reinterpret_cast<float *>(sums + (KH + 1) / 2 * 2) : nullptr;
        a.B = bsz;
        a.L = prelen;
        a.H = heads;
        a.K = translen;
        int grid;
        if (int rc = lb_run(a, true, grid, st, di, who)) return rc;
        if (!grad_bias_table) return DAT_OK;
        launch_after(lb_sum_kernel, sgrid, kSum, 0, st, 1, a.part, sums, grid, KH);
    } else {
        if (int rc = links_bwd_rows<true>(grad_links, content, log_gates, links, head_lse, mk, lb, grad_content,
                                          grad_log_gates, bsz, prelen, heads, translen, st, di, who))
            return rc;
        if (!grad_bias_table) return DAT_OK;
        launch_after(lb_diag_kernel, sgrid, kSum, 0, st, 1, grad_content, sums, bsz, prelen, heads, translen);
    }
    if (int rc = check_launch(who)) return rc;
    launch_after(lb_join_kernel, (unsigned)num_buckets, kLbJoinThreads, 0, st, 1, sums, buckets, grad_bias_table, heads, translen);
    return check_launch(who);
}

}  // extern "C"

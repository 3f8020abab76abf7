// Group norm with an activation on channels-last maps, and its gradient: x [N, P, C], the C / G channels of a group share the
// statistics of their P C / G values,
//
//   xh = (x - mean) rstd,   y = act(w xh + b);      dz = dy act'(w xh + b),  db = sum dz,  dw = sum dz xh,
//   dx = rstd (w dz - mean(w dz) - xh mean(w dz xh))        (means over a group)
//
// Bound by memory: a thread owns V neighbouring channels (16 bytes of bf16) of every few rows, so a wave reads and writes whole
// lines, and keeps the channels' parameters in registers.  A map is cut into chunks of rows; the chunks' statistics
// (count, mean, sum of squares about the mean - no difference of large sums) are joined in a small launch, always in the same order.
// 16 maps of 128 x 128 x 256 bf16: 22 us statistics, 5 join, 47 result.  Where a workgroup can hold a group, and its piece of a row is 64 bytes or more, one
// launch does it all (1369 x 1024, 32 groups: 10 us against 17 in three; pieces of 16 bytes: 99 against 77).
#include <initializer_list>
#include "common.h"
#include "../../include/mars_hip.h"

namespace {

constexpr int TH = 256;             // threads a workgroup
constexpr int KR = 4;               // rows a thread holds at a time

struct Norm {
    const void* x;
    int64_t x_n, x_p;
    const float *w, *b;
    int N, P, C, G, Cg, V, act;
    int vpr;                        // vectors a row: C / V
    int ncb;                        // column blocks of up to TH vectors
    int chunks, rows;               // chunks of `rows` rows
    int stream;                     // results too large to find again in a cache: stored past them
};

template <typename T, int V> __device__ __forceinline__ void load_vec(const T* p, float (&v)[V]) {
    if constexpr (sizeof(T) == 2) {
        if constexpr (V == 8) { const bf16x8 r = *(const bf16x8*)p;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = (float)r[e];
        } else if constexpr (V == 4) { const bf16x4 r = *(const bf16x4*)p;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (float)r[e];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (float)p[e];
        }
    } else {
        if constexpr (V >= 4) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) { const f32x4 r = *(const f32x4*)(p + 4 * i);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = r[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = (float)p[e];
        }
    }
}
template <typename T, int V, bool STREAM = false> __device__ __forceinline__ void store_vec(T* p, const float (&v)[V]) {
    if constexpr (sizeof(T) == 2) {
        if constexpr (V == 8) { bf16x8 r;
#pragma unroll
            for (int e = 0; e < 8; ++e) r[e] = (__bf16)v[e];
            if constexpr (STREAM) __builtin_nontemporal_store(r, (bf16x8*)p);
            else *(bf16x8*)p = r;
        } else if constexpr (V == 4) { *(bf16x4*)p = (bf16x4){(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = (T)v[e];
        }
    } else {
        if constexpr (V >= 4) {
#pragma unroll
            for (int i = 0; i < V / 4; ++i) {
                const f32x4 r = {v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
                if constexpr (STREAM) __builtin_nontemporal_store(r, (f32x4*)(p + 4 * i));
                else *(f32x4*)(p + 4 * i) = r;
            }
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = (T)v[e];
        }
    }
}

// Phi(z) = (1 + erf(z / sqrt 2)) / 2 and, for the slope, exp(-z^2 / 2), on v_exp_f32 and v_rcp_f32 (erff and IEEE divisions made these kernels bound by
// arithmetic).  Phi(-|z|) = exp(-z^2 / 2) t p(t) with t = 1 / (1 + 0.43 |z| / sqrt 2): p is fitted to erfcx(x) / 2t over 0 <= x <= 9.6 (the exponential is zero
// in f32 from there) with the smallest largest RELATIVE error, 8.5e-8, by reweighted least squares in 64 bits.  So the tail keeps its digits, but for the
// 1.5 z^2 roundings that f32 leaves of the exponential of -z^2 / 2; a fit of the absolute error (1.5e-7 for the usual five terms) is as large as Phi itself from
// z = -5 on.
__device__ __forceinline__ float normal_cdf(float z, float& e) {
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.43f * 0.70710678118654752f, 1.f));
    e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170368f);
    float p = 0.03683450073f;
    p = fmaf(p, t, -0.15510785580f);
    p = fmaf(p, t, 0.19172063470f);
    p = fmaf(p, t, -0.04274427518f);
    p = fmaf(p, t, 0.12336096168f);
    p = fmaf(p, t, 0.10249371082f);
    p = fmaf(p, t, 0.12218486518f);
    p = fmaf(p, t, 0.12125748396f);
    const float h = p * t * e;                                      // (1 - erf(|z| / sqrt 2)) / 2
    return z < 0.f ? h : 1.f - h;
}
__device__ __forceinline__ float sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(z * -1.44269504088896340736f)); }

// 0 none, 1 erf GELU, 2 z sigmoid(1.702 z), 3 ReLU, 4 z sigmoid(z)
__device__ __forceinline__ float act_of(float z, int act) {
    float e;
    switch (act) {
        case 1: return z * normal_cdf(z, e);
        case 2: return z * sigmoid(1.702f * z);
        case 3: return z > 0.f || z != z ? z : 0.f;
        case 4: return z * sigmoid(z);
        default: return z;
    }
}
__device__ __forceinline__ float slope_of(float z, int act) {
    switch (act) {
        case 1: { float e; const float c = normal_cdf(z, e); return fmaf(z * e, 0.39894228040143268f, c); }
        case 2: { const float s = sigmoid(1.702f * z); return fmaf(1.702f * z * s, 1.f - s, s); }
        case 3: return z > 0.f ? 1.f : 0.f;
        case 4: { const float s = sigmoid(z); return fmaf(z * s, 1.f - s, s); }
        default: return 1.f;
    }
}

// statistics of two sets of values joined: counts, means, sums of squares about the mean
struct Stat { float n, mean, m2; };
__device__ __forceinline__ Stat join(const Stat& a, const Stat& b) {
    const float n = a.n + b.n;
    if (n == 0.f) return a;
    const float f = b.n / n, d = b.mean - a.mean;
    return Stat{n, fmaf(d, f, a.mean), a.m2 + b.m2 + d * d * a.n * f};
}

// grid (chunks, column blocks, N): part[n][chunk][column block][group] for the groups with a channel in the block
template <typename T, int V>
__global__ __launch_bounds__(TH) void norm_stat_kernel(const Norm a, Stat* __restrict__ part) {
    __shared__ Stat sh[TH];
    const int tid = threadIdx.x, n = blockIdx.z, cb = blockIdx.y, chunk = blockIdx.x;
    const int v0 = cb * TH, nv = min(TH, a.vpr - v0);               // this block's vectors
    const int rl = tid / nv, cv = tid - rl * nv, nrl = TH / nv;     // row lanes
    const bool on = rl < nrl;
    Stat st{0.f, 0.f, 0.f};
    if (on) {
        const T* base = (const T*)a.x + (int64_t)n * a.x_n + (int64_t)(v0 + cv) * V;
        const int r1 = min((chunk + 1) * a.rows, a.P);
        for (int r = chunk * a.rows + rl; r < r1; r += nrl * KR) {
            float x[KR][V];
            int cnt = 0;
#pragma unroll
            for (int k = 0; k < KR; ++k) {
                if (r + k * nrl < r1) { load_vec<T, V>(base + (int64_t)(r + k * nrl) * a.x_p, x[k]); ++cnt; }
            }
            float s = 0.f, q = 0.f;
#pragma unroll
            for (int k = 0; k < KR; ++k)
                if (k < cnt) {
#pragma unroll
                    for (int e = 0; e < V; ++e) s += x[k][e];
                }
            const float nn = (float)(cnt * V), mean = s / nn;
#pragma unroll
            for (int k = 0; k < KR; ++k)
                if (k < cnt) {
#pragma unroll
                    for (int e = 0; e < V; ++e) q = fmaf(x[k][e] - mean, x[k][e] - mean, q);
                }
            st = join(st, Stat{nn, mean, q});
        }
    }
    sh[tid] = st;
    __syncthreads();
    // row lanes, pairwise
    for (int s = 1; s < nrl; s *= 2) {
        if (on && rl % (2 * s) == 0 && rl + s < nrl) sh[tid] = join(sh[tid], sh[tid + s * nv]);
        __syncthreads();
    }
    // the vectors of a group, pairwise (a group may begin or end outside the block)
    const int cgv = a.Cg / V, g = (v0 + cv) / cgv, first = max(g * cgv - v0, 0), last = min((g + 1) * cgv - v0, nv), i = cv - first;
    for (int s = 1; s < cgv && s < nv; s *= 2) {
        if (rl == 0 && i % (2 * s) == 0 && cv + s < last) sh[cv] = join(sh[cv], sh[cv + s]);
        __syncthreads();
    }
    if (rl == 0 && i == 0) part[(((int64_t)n * a.chunks + chunk) * a.ncb + cb) * a.G + g] = sh[cv];
}

// one wave a (n, group): mean and rstd from the chunks
__global__ __launch_bounds__(64) void norm_join_kernel(const Norm a, const Stat* __restrict__ part, float eps, float* __restrict__ stat) {
    const int g = blockIdx.x, n = blockIdx.y, lane = threadIdx.x;
    const int per = TH * a.V, cb0 = g * a.Cg / per, cb1 = ((g + 1) * a.Cg - 1) / per;
    Stat st{0.f, 0.f, 0.f};
    for (int c = lane; c < a.chunks; c += 64)
        for (int cb = cb0; cb <= cb1; ++cb) st = join(st, part[(((int64_t)n * a.chunks + c) * a.ncb + cb) * a.G + g]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        const Stat other{__shfl_xor(st.n, o, 64), __shfl_xor(st.mean, o, 64), __shfl_xor(st.m2, o, 64)};
        st = (lane & o) ? join(other, st) : join(st, other);
    }
    if (lane == 0) {
        float* s = stat + ((int64_t)n * a.G + g) * 2;
        s[0] = st.mean;
        s[1] = 1.0f / sqrtf(st.m2 / st.n + eps);
    }
}

template <typename TI, typename TO, int V, bool STREAM>
__global__ __launch_bounds__(TH) void norm_apply_kernel(const Norm a, const float* __restrict__ stat, TO* __restrict__ out, int64_t o_n, int64_t o_p) {
    const int tid = threadIdx.x, n = blockIdx.z, cb = blockIdx.y, chunk = blockIdx.x;
    const int v0 = cb * TH, nv = min(TH, a.vpr - v0), rl = tid / nv, cv = tid - rl * nv, nrl = TH / nv;
    if (rl >= nrl) return;
    const int c = (v0 + cv) * V, g = c / a.Cg;
    const float mean = stat[((int64_t)n * a.G + g) * 2], rstd = stat[((int64_t)n * a.G + g) * 2 + 1];
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { w[e] = a.w[c + e] * rstd; b[e] = a.b[c + e]; }
    const TI* xp = (const TI*)a.x + (int64_t)n * a.x_n + c;
    TO* op = out + (int64_t)n * o_n + c;
    const int r1 = min((chunk + 1) * a.rows, a.P);
    for (int r = chunk * a.rows + rl; r < r1; r += nrl * KR) {
        float x[KR][V];
#pragma unroll
        for (int k = 0; k < KR; ++k)
            if (r + k * nrl < r1) load_vec<TI, V>(xp + (int64_t)(r + k * nrl) * a.x_p, x[k]);
#pragma unroll
        for (int k = 0; k < KR; ++k)
            if (r + k * nrl < r1) {
                float y[V];
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = act_of(fmaf(x[k][e] - mean, w[e], b[e]), a.act);
                store_vec<TO, V, STREAM>(op + (int64_t)(r + k * nrl) * o_p, y);
            }
    }
}

struct NormBwd {
    const void* dy;
    int64_t dy_n, dy_p;
    void* dx;
    int64_t dx_n, dx_p;
    const float* stat;
    float *part, *sums;             // [N][chunks][C][2], [N][C][2]: sums of dz and dz xh
    float *dw, *db;
};

// grid (chunks, column blocks, N): sums of dz and dz xh per channel of a chunk
template <typename TX, typename TY, int V>
__global__ __launch_bounds__(TH) void norm_bwd_sum_kernel(const Norm a, const NormBwd d) {
    __shared__ float sh[TH][2 * V + 1];
    const int tid = threadIdx.x, n = blockIdx.z, cb = blockIdx.y, chunk = blockIdx.x;
    const int v0 = cb * TH, nv = min(TH, a.vpr - v0), rl = tid / nv, cv = tid - rl * nv, nrl = TH / nv;
    float s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) s1[e] = s2[e] = 0.f;
    const int c = (v0 + cv) * V;
    if (rl < nrl) {
        const int g = c / a.Cg;
        const float mean = d.stat[((int64_t)n * a.G + g) * 2], rstd = d.stat[((int64_t)n * a.G + g) * 2 + 1];
        float w[V], b[V];
#pragma unroll
        for (int e = 0; e < V; ++e) { w[e] = a.w[c + e]; b[e] = a.b[c + e]; }
        const TX* xp = (const TX*)a.x + (int64_t)n * a.x_n + c;
        const TY* yp = (const TY*)d.dy + (int64_t)n * d.dy_n + c;
        const int r1 = min((chunk + 1) * a.rows, a.P);
        for (int r = chunk * a.rows + rl; r < r1; r += nrl * KR) {
            float x[KR][V], y[KR][V];
#pragma unroll
            for (int k = 0; k < KR; ++k)
                if (r + k * nrl < r1) {
                    load_vec<TX, V>(xp + (int64_t)(r + k * nrl) * a.x_p, x[k]);
                    load_vec<TY, V>(yp + (int64_t)(r + k * nrl) * d.dy_p, y[k]);
                }
#pragma unroll
            for (int k = 0; k < KR; ++k)
                if (r + k * nrl < r1) {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float xh = (x[k][e] - mean) * rstd, dz = y[k][e] * slope_of(fmaf(xh, w[e], b[e]), a.act);
                        s1[e] += dz;
                        s2[e] = fmaf(dz, xh, s2[e]);
                    }
                }
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) { sh[tid][2 * e] = s1[e]; sh[tid][2 * e + 1] = s2[e]; }
    __syncthreads();
    for (int i = tid; i < nv * 2 * V; i += TH) {
        const int v = i / (2 * V), k = i - v * 2 * V;
        float s = 0.f;
        for (int r = 0; r < nrl; ++r) s += sh[r * nv + v][k];
        d.part[(((int64_t)n * a.chunks + chunk) * a.C + (v0 + v) * V) * 2 + k] = s;
    }
}

// grid (ceil(2 C / 64), N): the chunks' sums; four waves take the chunks in turn
__global__ __launch_bounds__(256) void norm_bwd_join_kernel(const Norm a, const NormBwd d) {
    __shared__ float sh[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = blockIdx.y, i = blockIdx.x * 64 + lane;
    float s = 0.f;
    if (i < 2 * a.C) {
        const float* p = d.part + (int64_t)n * a.chunks * a.C * 2 + i;
        constexpr int U = 8;                                        // loads in flight
        for (int c = wave; c < a.chunks; c += 4 * U) {
            float v[U];
#pragma unroll
            for (int u = 0; u < U; ++u) v[u] = c + 4 * u < a.chunks ? p[(int64_t)(c + 4 * u) * a.C * 2] : 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u) s += v[u];
        }
    }
    sh[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < 2 * a.C) d.sums[(int64_t)n * a.C * 2 + i] = (sh[0][lane] + sh[1][lane]) + (sh[2][lane] + sh[3][lane]);
}

// grid (chunks + 1, column blocks, N): dx of a chunk; the workgroups behind the last chunk add dw and db up over the batch
template <typename TX, typename TY, int V, bool STREAM>
__global__ __launch_bounds__(TH) void norm_bwd_apply_kernel(const Norm a, const NormBwd d) {
    __shared__ float sh[2][TH];
    const int tid = threadIdx.x, n = blockIdx.z, cb = blockIdx.y, chunk = blockIdx.x;
    if (chunk == a.chunks) {
        if (cb != 0) return;
        const int per = (a.C + a.N - 1) / a.N;
        for (int c = n * per + tid; c < min((n + 1) * per, a.C); c += TH) {
            float s1 = 0.f, s2 = 0.f;
            for (int i = 0; i < a.N; ++i) { s1 += d.sums[((int64_t)i * a.C + c) * 2]; s2 += d.sums[((int64_t)i * a.C + c) * 2 + 1]; }
            d.db[c] = s1;
            d.dw[c] = s2;
        }
        return;
    }
    const int v0 = cb * TH, nv = min(TH, a.vpr - v0), rl = tid / nv, cv = tid - rl * nv, nrl = TH / nv;
    // means over the groups that have a channel in this block
    const int g_first = v0 * V / a.Cg, g_last = ((v0 + nv) * V - 1) / a.Cg;
    const float inv = 1.0f / ((float)a.P * (float)a.Cg);
    const int g = (rl < nrl) ? (v0 + cv) * V / a.Cg : g_first;
    float m1 = 0.f, m2 = 0.f;
    if (a.ncb == 1 && a.Cg <= 64) {                                 // a thread adds its group's few channels up by itself, from LDS
        __shared__ float ch[2][TH * V];
        for (int c = tid; c < a.C; c += TH) {
            ch[0][c] = a.w[c] * d.sums[((int64_t)n * a.C + c) * 2];
            ch[1][c] = a.w[c] * d.sums[((int64_t)n * a.C + c) * 2 + 1];
        }
        __syncthreads();
        for (int i = 0; i < a.Cg; ++i) { m1 += ch[0][g * a.Cg + i]; m2 += ch[1][g * a.Cg + i]; }
        m1 *= inv;
        m2 *= inv;
    } else for (int g0 = g_first; g0 <= g_last; g0 += TH) {         // a wave a group, up to TH groups a step
        const int ng = min(TH, g_last - g0 + 1);
        __syncthreads();
        for (int q = tid >> 6; q < ng; q += TH / 64) {
            float t1 = 0.f, t2 = 0.f;
            for (int c = tid & 63; c < a.Cg; c += 64) {
                const int ch = (g0 + q) * a.Cg + c;
                const float w = a.w[ch];
                t1 = fmaf(w, d.sums[((int64_t)n * a.C + ch) * 2], t1);
                t2 = fmaf(w, d.sums[((int64_t)n * a.C + ch) * 2 + 1], t2);
            }
            t1 = wave_sum(t1);
            t2 = wave_sum(t2);
            if ((tid & 63) == 0) { sh[0][q] = t1 * inv; sh[1][q] = t2 * inv; }
        }
        __syncthreads();
        if (g >= g0 && g < g0 + ng) { m1 = sh[0][g - g0]; m2 = sh[1][g - g0]; }
    }
    if (rl >= nrl) return;
    const int c = (v0 + cv) * V;
    const float mean = d.stat[((int64_t)n * a.G + g) * 2], rstd = d.stat[((int64_t)n * a.G + g) * 2 + 1];
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { w[e] = a.w[c + e]; b[e] = a.b[c + e]; }
    const TX* xp = (const TX*)a.x + (int64_t)n * a.x_n + c;
    const TY* yp = (const TY*)d.dy + (int64_t)n * d.dy_n + c;
    TX* op = (TX*)d.dx + (int64_t)n * d.dx_n + c;
    const bool one = a.P == 1 && a.Cg == 1;                         // a group of one value is its own mean: no gradient
    const int r1 = min((chunk + 1) * a.rows, a.P);
    for (int r = chunk * a.rows + rl; r < r1; r += nrl * KR) {
        float x[KR][V], y[KR][V];
#pragma unroll
        for (int k = 0; k < KR; ++k)
            if (r + k * nrl < r1) {
                load_vec<TX, V>(xp + (int64_t)(r + k * nrl) * a.x_p, x[k]);
                load_vec<TY, V>(yp + (int64_t)(r + k * nrl) * d.dy_p, y[k]);
            }
#pragma unroll
        for (int k = 0; k < KR; ++k)
            if (r + k * nrl < r1) {
                float o[V];
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float xh = (x[k][e] - mean) * rstd, dz = y[k][e] * slope_of(fmaf(xh, w[e], b[e]), a.act);
                    o[e] = one ? 0.f : rstd * (dz * w[e] - m1 - xh * m2);
                }
                store_vec<TX, V, STREAM>(op + (int64_t)(r + k * nrl) * d.dx_p, o);
            }
    }
}

// ---- maps whose group fits the registers of one workgroup: everything in one launch, x (and dy) read once.  A workgroup of 1024 owns one
// (n, group); a thread holds K vectors of V channels, row lanes TF / (Cg / V) apart.  Groups of one image run on one XCD: a group's
// piece of a row is shorter than a cache line, and the neighbours' pieces are found in the same L2.
constexpr int TF = 1024;

template <typename T, int V> struct Raw { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct Raw<T, 1> { typedef T type; };
template <typename T, int V> __device__ __forceinline__ void widen(const typename Raw<T, V>::type& r, float (&v)[V]) {
    if constexpr (V == 1) v[0] = (float)r;
    else {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (float)r[e];
    }
}

__device__ __forceinline__ void group_of_block(const Norm& a, int& n, int& g) {
    const int id = blockIdx.x, full = (a.N >> 3) * 8 * a.G;
    if (id < full) { const int j = id >> 3; n = (j / a.G) * 8 + (id & 7); g = j % a.G; }
    else { n = id / a.G; g = id % a.G; }
}

// sum over the workgroup, the same for every thread and every call
__device__ __forceinline__ float sum_all(float v, float* sh) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < TF / 64; ++i) s += sh[i];
    return s;
}

template <typename TI, typename TO, int V, int K>
__global__ __launch_bounds__(TF) void norm_group_kernel(const Norm a, float eps, float* __restrict__ stat, TO* __restrict__ out, int64_t o_n, int64_t o_p) {
    __shared__ float sh[TF / 64];
    int n, g;
    group_of_block(a, n, g);
    const int cgv = a.Cg / V, step = TF / cgv, rl = threadIdx.x / cgv, c = g * a.Cg + (threadIdx.x - rl * cgv) * V;
    const bool on = rl < step;
    typename Raw<TI, V>::type x[K];
    const TI* xp = (const TI*)a.x + (int64_t)n * a.x_n + c;
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = rl + k * step;
        if (on && r < a.P) x[k] = *(const typename Raw<TI, V>::type*)(xp + (int64_t)r * a.x_p);
    }
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && rl + k * step < a.P) {
            float v[V];
            widen<TI, V>(x[k], v);
#pragma unroll
            for (int e = 0; e < V; ++e) s += v[e];
        }
    const float cnt = (float)a.P * (float)a.Cg, mean = sum_all(s, sh) / cnt;
    float q = 0.f;
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && rl + k * step < a.P) {
            float v[V];
            widen<TI, V>(x[k], v);
#pragma unroll
            for (int e = 0; e < V; ++e) q = fmaf(v[e] - mean, v[e] - mean, q);
        }
    const float rstd = 1.0f / sqrtf(sum_all(q, sh) / cnt + eps);
    if (stat != nullptr && threadIdx.x == 0) { stat[((int64_t)n * a.G + g) * 2] = mean; stat[((int64_t)n * a.G + g) * 2 + 1] = rstd; }
    if (!on) return;
    float w[V], b[V];
#pragma unroll
    for (int e = 0; e < V; ++e) { w[e] = a.w[c + e] * rstd; b[e] = a.b[c + e]; }
    TO* op = out + (int64_t)n * o_n + c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = rl + k * step;
        if (r < a.P) {
            float v[V];
            widen<TI, V>(x[k], v);
#pragma unroll
            for (int e = 0; e < V; ++e) v[e] = act_of(fmaf(v[e] - mean, w[e], b[e]), a.act);
            store_vec<TO, V>(op + (int64_t)r * o_p, v);
        }
    }
}

template <typename TX, typename TY, int V, int K>
__global__ __launch_bounds__(TF) void norm_group_bwd_kernel(const Norm a, const NormBwd d) {
    __shared__ float sh[TF][2 * V + 1];
    int n, g;
    group_of_block(a, n, g);
    const int cgv = a.Cg / V, step = TF / cgv, rl = threadIdx.x / cgv, cv = threadIdx.x - rl * cgv, c = g * a.Cg + cv * V;
    const bool on = rl < step;
    typename Raw<TX, V>::type x[K];
    typename Raw<TY, V>::type y[K];
    const TX* xp = (const TX*)a.x + (int64_t)n * a.x_n + c;
    const TY* yp = (const TY*)d.dy + (int64_t)n * d.dy_n + c;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = rl + k * step;
        if (on && r < a.P) {
            x[k] = *(const typename Raw<TX, V>::type*)(xp + (int64_t)r * a.x_p);
            y[k] = *(const typename Raw<TY, V>::type*)(yp + (int64_t)r * d.dy_p);
        }
    }
    const float mean = d.stat[((int64_t)n * a.G + g) * 2], rstd = d.stat[((int64_t)n * a.G + g) * 2 + 1];
    float w[V], b[V], s1[V], s2[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        w[e] = on ? a.w[c + e] : 0.f;
        b[e] = on ? a.b[c + e] : 0.f;
        s1[e] = s2[e] = 0.f;
    }
    // (the slope is worked out again for dx below: cheaper than a register for each dz)
#pragma unroll
    for (int k = 0; k < K; ++k)
        if (on && rl + k * step < a.P) {
            float xv[V], yv[V];
            widen<TX, V>(x[k], xv);
            widen<TY, V>(y[k], yv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (xv[e] - mean) * rstd, dz = yv[e] * slope_of(fmaf(xh, w[e], b[e]), a.act);
                s1[e] += dz;
                s2[e] = fmaf(dz, xh, s2[e]);
            }
        }
#pragma unroll
    for (int e = 0; e < V; ++e) { sh[threadIdx.x][2 * e] = s1[e]; sh[threadIdx.x][2 * e + 1] = s2[e]; }
    __syncthreads();
    // row lanes, halves onto halves: row 0 of sh ends up with the group's channel sums
    for (int m = step; m > 1;) {
        const int h = (m + 1) / 2;
        if (rl < m - h) {
#pragma unroll
            for (int e = 0; e < 2 * V; ++e) sh[threadIdx.x][e] += sh[threadIdx.x + h * cgv][e];
        }
        __syncthreads();
        m = h;
    }
    // the two means of the group: a wave (every wave its own copy), then the channel sums for dw and db
    float t1 = 0.f, t2 = 0.f;
    for (int i = threadIdx.x & 63; i < a.Cg; i += 64) {
        const float wc = a.w[g * a.Cg + i];
        t1 = fmaf(wc, sh[i / V][2 * (i % V)], t1);
        t2 = fmaf(wc, sh[i / V][2 * (i % V) + 1], t2);
    }
    const float inv = 1.0f / ((float)a.P * (float)a.Cg);
    const float m1 = wave_sum(t1) * inv, m2 = wave_sum(t2) * inv;
    for (int i = threadIdx.x; i < a.Cg; i += TF) {
        const int ch = g * a.Cg + i;
        const float u1 = sh[i / V][2 * (i % V)], u2 = sh[i / V][2 * (i % V) + 1];
        if (a.N == 1) { d.db[ch] = u1; d.dw[ch] = u2; }
        else { d.sums[((int64_t)n * a.C + ch) * 2] = u1; d.sums[((int64_t)n * a.C + ch) * 2 + 1] = u2; }
    }
    if (!on) return;
    TX* op = (TX*)d.dx + (int64_t)n * d.dx_n + c;
    const bool one = a.P == 1 && a.Cg == 1;                         // a group of one value is its own mean: no gradient
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int r = rl + k * step;
        if (r < a.P) {
            float xv[V], yv[V];
            widen<TX, V>(x[k], xv);
            widen<TY, V>(y[k], yv);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const float xh = (xv[e] - mean) * rstd, dz = yv[e] * slope_of(fmaf(xh, w[e], b[e]), a.act);
                xv[e] = one ? 0.f : rstd * (dz * w[e] - m1 - xh * m2);
            }
            store_vec<TX, V>(op + (int64_t)r * d.dx_p, xv);
        }
    }
}

// dw, db: the batch entries' sums in order
__global__ __launch_bounds__(256) void norm_bwd_batch_kernel(const Norm a, const NormBwd d) {
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= a.C) return;
    float s1 = 0.f, s2 = 0.f;
    for (int i = 0; i < a.N; ++i) { s1 += d.sums[((int64_t)i * a.C + c) * 2]; s2 += d.sums[((int64_t)i * a.C + c) * 2 + 1]; }
    d.db[c] = s1;
    d.dw[c] = s2;
}

// rows a thread has to hold for a workgroup to own a group: 0 where that is more than `most`, or where a group's piece of a row is narrower than 64 bytes
int held_rows(const Norm& a, int V, int most, int es) {
    if (a.Cg / V > TF || a.Cg * es < 64) return 0;
    const int64_t step = TF / (a.Cg / V), k = (a.P + step - 1) / step;
    return k <= most ? (int)k : 0;
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

// widest vector that divides a group and keeps every row aligned: 8, 4, 2 or 1 channels
int vec_width(int Cg, std::initializer_list<uint64_t> addresses, int es) {
    int V = 8;
    while (V > 1) {
        bool ok = Cg % V == 0;
        const uint64_t al = (uint64_t)(V * es < 16 ? V * es : 16);
        for (const uint64_t x : addresses) ok = ok && x % al == 0;
        if (ok) break;
        V /= 2;
    }
    return V;
}

// the group kernels hold raw vectors: 16 bytes of the wider type (f32: 4 channels)
int vec_for_group(const Norm& a, int dt_a, int dt_b) { return a.V == 8 && (dt_a == 0 || dt_b == 0) ? 4 : a.V; }

// The map is read twice, so stores that would push it out of the last-level cache go past it.  With n maps of 64 x 64 x 256, forward / step, us:
//   results in bf16   n = 8: 20.0 / 44 past the cache, 19.8 / 48 through it   n = 16: 24.5 / 70, 27.3 / 76   n = 64: 72 / 221, 75 / 235   n = 96: 109 / 378, 126 / 427
//   results in f32    n = 16: 45 / 111, 39 / 104   n = 32: 80 / 205, 69 / 206   n = 48: 121 / 327, 126 / 368   n = 64: 152 / 437, 170 / 461
// (an f32 vector of eight channels is two stores of half a line each: they want the cache for as long as it holds them)
bool past_cache(const Norm& a, int es) { return (int64_t)a.N * a.P * a.C >= (es == 2 ? 1ll << 24 : 3ll << 24); }

// chunks of rows: about 1024 workgroups, at least KR rows a thread
void cut(Norm& a) {
    a.vpr = a.C / a.V;
    a.ncb = (a.vpr + TH - 1) / TH;
    const int nrl = TH / (a.vpr < TH ? a.vpr : TH), least = nrl * KR;
    const int64_t want = 1024 / ((int64_t)a.N * a.ncb) + 1;
    int64_t rows = (a.P + want - 1) / want;
    rows = (rows + least - 1) / least * least;
    a.rows = (int)rows;
    a.chunks = (int)((a.P + rows - 1) / rows);
}

int norm_check(const char* what, int N, int P, int C, int G, int act, int dt_a, int dt_b) {
    MARS_CHECK(N > 0 && P > 0 && C > 0 && G > 0 && N <= 65535 && C < (1 << 24) && P < (1 << 30), "%s: bad shape N=%d P=%d C=%d", what, N, P, C);
    MARS_CHECK(C % G == 0, "%s: %d channels do not divide into %d groups", what, C, G);
    MARS_CHECK(act >= 0 && act <= 4, "%s: activation %d", what, act);
    MARS_CHECK((dt_a == 0 || dt_a == 1) && (dt_b == 0 || dt_b == 1), "%s: dtype", what);
    return 0;
}

#define MARS_NORM_V(F, TA, TB)           \
    switch (a.V) {                       \
        case 8: F(TA, TB, 8); break;     \
        case 4: F(TA, TB, 4); break;     \
        case 2: F(TA, TB, 2); break;     \
        default: F(TA, TB, 1); break;    \
    }
#define MARS_NORM_T(F)                                                                  \
    if (dx_t == 1) { if (dy_t == 1) { MARS_NORM_V(F, __bf16, __bf16) } else { MARS_NORM_V(F, __bf16, float) } } \
    else { if (dy_t == 1) { MARS_NORM_V(F, float, __bf16) } else { MARS_NORM_V(F, float, float) } }

// workspace of the forward call, whatever vector width its addresses allow
int64_t fwd_ws(int N, int P, int C, int G) {
    int64_t most = 0;
    for (int V = 1; V <= 8; V *= 2) {
        if ((C / G) % V) continue;
        Norm a{};
        a.N = N; a.P = P; a.C = C; a.V = V;
        cut(a);
        const int64_t b = (int64_t)N * a.chunks * a.ncb * G * (int64_t)sizeof(Stat);
        if (b > most) most = b;
    }
    return align256(most) + align256((int64_t)N * G * 8);
}
int64_t bwd_ws(int N, int P, int C, int G) {
    int64_t most = 0;
    for (int V = 1; V <= 8; V *= 2) {
        if ((C / G) % V) continue;
        Norm a{};
        a.N = N; a.P = P; a.C = C; a.V = V;
        cut(a);
        const int64_t b = (int64_t)N * a.chunks * C * 8;
        if (b > most) most = b;
    }
    return align256(most) + align256((int64_t)N * C * 8);
}

}  // namespace

extern "C" int64_t marship_group_norm_act_ws(int N, int P, int C, int G, int backward) {
    if (N <= 0 || P <= 0 || C <= 0 || G <= 0 || C % G) return 0;
    return backward ? bwd_ws(N, P, C, G) : fwd_ws(N, P, C, G);
}

extern "C" int marship_group_norm_act(const void* x, int64_t x_n, int64_t x_p, const float* w, const float* b, void* out, int64_t o_n, int64_t o_p, int N, int P,
                                      int C, int G, float eps, int act, int x_dtype, int out_dtype, float* stat, void* ws, int64_t ws_bytes, void* stream) {
    MARS_CHECK(x && w && b && out, "group_norm_act: null pointer");
    if (const int rc = norm_check("group_norm_act", N, P, C, G, act, x_dtype, out_dtype)) return rc;
    MARS_CHECK(eps >= 0.f, "group_norm_act: eps");
    const int64_t need = fwd_ws(N, P, C, G);
    MARS_CHECK(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "group_norm_act: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
    const int xe = x_dtype == 1 ? 2 : 4, oe = out_dtype == 1 ? 2 : 4;
    Norm a{};
    a.x = x; a.x_n = x_n; a.x_p = x_p; a.w = w; a.b = b;
    a.N = N; a.P = P; a.C = C; a.G = G; a.Cg = C / G; a.act = act;
    const int vx = vec_width(a.Cg, {(uint64_t)x, (uint64_t)(x_n * xe), (uint64_t)(x_p * xe)}, xe);
    const int vo = vec_width(a.Cg, {(uint64_t)out, (uint64_t)(o_n * oe), (uint64_t)(o_p * oe)}, oe);
    const int vw = vx < vo ? vx : vo;
    a.V = vw;
    cut(a);
    a.stream = past_cache(a, oe);
    MARS_CHECK((int64_t)a.chunks < (1 << 23) && a.ncb <= 65535 && (int64_t)N * G < (1 << 22), "group_norm_act: more workgroups than a launch takes");
    hipStream_t s = (hipStream_t)stream;
    a.V = vec_for_group(a, x_dtype, out_dtype);
    const int dx_t = x_dtype, dy_t = out_dtype;
    if (const int k = held_rows(a, a.V, 16, xe)) {
        const dim3 gb((unsigned)(N * G));
#define MARS_GROUP(TA, TB, VV)                                                                                                                       \
    do {                                                                                                                                             \
        if (k <= 4) hipLaunchKernelGGL((norm_group_kernel<TA, TB, VV, 4>), gb, dim3(TF), 0, s, a, eps, stat, (TB*)out, o_n, o_p);                     \
        else if (k <= 8) hipLaunchKernelGGL((norm_group_kernel<TA, TB, VV, 8>), gb, dim3(TF), 0, s, a, eps, stat, (TB*)out, o_n, o_p);                \
        else hipLaunchKernelGGL((norm_group_kernel<TA, TB, VV, 16>), gb, dim3(TF), 0, s, a, eps, stat, (TB*)out, o_n, o_p);                           \
    } while (0)
        MARS_NORM_T(MARS_GROUP)
        MARS_LAUNCH_CHECK();
        return 0;
    }
    a.V = vw;
    Stat* part = (Stat*)ws;
    float* st = stat != nullptr ? stat : (float*)((char*)ws + (need - align256((int64_t)N * G * 8)));
    const dim3 grid((unsigned)a.chunks, (unsigned)a.ncb, (unsigned)N);
#define MARS_STAT(TA, TB, VV) hipLaunchKernelGGL((norm_stat_kernel<TA, VV>), grid, dim3(TH), 0, s, a, part)
    if (dx_t == 1) { MARS_NORM_V(MARS_STAT, __bf16, __bf16) } else { MARS_NORM_V(MARS_STAT, float, float) }
    MARS_LAUNCH_CHECK();
    hipLaunchKernelGGL(norm_join_kernel, dim3((unsigned)G, (unsigned)N), dim3(64), 0, s, a, part, eps, st);
    MARS_LAUNCH_CHECK();
#define MARS_APPLY(TA, TB, VV)                                                                                                               \
    do {                                                                                                                                     \
        if (a.stream) hipLaunchKernelGGL((norm_apply_kernel<TA, TB, VV, true>), grid, dim3(TH), 0, s, a, st, (TB*)out, o_n, o_p);             \
        else hipLaunchKernelGGL((norm_apply_kernel<TA, TB, VV, false>), grid, dim3(TH), 0, s, a, st, (TB*)out, o_n, o_p);                     \
    } while (0)
    MARS_NORM_T(MARS_APPLY)
    MARS_LAUNCH_CHECK();
    return 0;
}

extern "C" int marship_group_norm_act_bwd(const void* x, int64_t x_n, int64_t x_p, const float* w, const float* b, const float* stat, const void* dy, int64_t dy_n,
                                          int64_t dy_p, void* dx, int64_t dx_n, int64_t dx_p, float* dw, float* db, int N, int P, int C, int G, int act,
                                          int x_dtype, int dy_dtype, void* ws, int64_t ws_bytes, void* stream) {
    MARS_CHECK(x && w && b && stat && dy && dx && dw && db, "group_norm_act_bwd: null pointer");
    if (const int rc = norm_check("group_norm_act_bwd", N, P, C, G, act, x_dtype, dy_dtype)) return rc;
    const int64_t need = bwd_ws(N, P, C, G);
    MARS_CHECK(ws && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "group_norm_act_bwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes, (long long)need);
    const int xe = x_dtype == 1 ? 2 : 4, ye = dy_dtype == 1 ? 2 : 4;
    Norm a{};
    a.x = x; a.x_n = x_n; a.x_p = x_p; a.w = w; a.b = b;
    a.N = N; a.P = P; a.C = C; a.G = G; a.Cg = C / G; a.act = act;
    const int vx = vec_width(a.Cg, {(uint64_t)x, (uint64_t)(x_n * xe), (uint64_t)(x_p * xe), (uint64_t)dx, (uint64_t)(dx_n * xe), (uint64_t)(dx_p * xe)}, xe);
    const int vy = vec_width(a.Cg, {(uint64_t)dy, (uint64_t)(dy_n * ye), (uint64_t)(dy_p * ye)}, ye);
    const int vw = vx < vy ? vx : vy;
    a.V = vw;
    cut(a);
    a.stream = past_cache(a, xe);
    MARS_CHECK((int64_t)a.chunks < (1 << 23) && a.ncb <= 65535 && (int64_t)N * G < (1 << 22), "group_norm_act_bwd: more workgroups than a launch takes");
    NormBwd d{};
    d.dy = dy; d.dy_n = dy_n; d.dy_p = dy_p; d.dx = dx; d.dx_n = dx_n; d.dx_p = dx_p; d.stat = stat; d.dw = dw; d.db = db;
    d.part = (float*)ws;
    d.sums = (float*)((char*)ws + (need - align256((int64_t)N * C * 8)));
    hipStream_t s = (hipStream_t)stream;
    const int dx_t = x_dtype, dy_t = dy_dtype;
    a.V = vec_for_group(a, x_dtype, dy_dtype);
    if (const int k = held_rows(a, a.V, 8, xe)) {
        const dim3 gb((unsigned)(N * G));
#define MARS_BGROUP(TA, TB, VV)                                                                                  \
    do {                                                                                                         \
        if (k <= 2) hipLaunchKernelGGL((norm_group_bwd_kernel<TA, TB, VV, 2>), gb, dim3(TF), 0, s, a, d);         \
        else if (k <= 4) hipLaunchKernelGGL((norm_group_bwd_kernel<TA, TB, VV, 4>), gb, dim3(TF), 0, s, a, d);    \
        else hipLaunchKernelGGL((norm_group_bwd_kernel<TA, TB, VV, 8>), gb, dim3(TF), 0, s, a, d);                \
    } while (0)
        MARS_NORM_T(MARS_BGROUP)
        MARS_LAUNCH_CHECK();
        if (N > 1) {
            hipLaunchKernelGGL(norm_bwd_batch_kernel, dim3((unsigned)((C + 255) / 256)), dim3(256), 0, s, a, d);
            MARS_LAUNCH_CHECK();
        }
        return 0;
    }
    a.V = vw;
    const dim3 grid((unsigned)a.chunks, (unsigned)a.ncb, (unsigned)N), grid1((unsigned)a.chunks + 1, (unsigned)a.ncb, (unsigned)N);
#define MARS_BSUM(TA, TB, VV) hipLaunchKernelGGL((norm_bwd_sum_kernel<TA, TB, VV>), grid, dim3(TH), 0, s, a, d)
    MARS_NORM_T(MARS_BSUM)
    MARS_LAUNCH_CHECK();
    hipLaunchKernelGGL(norm_bwd_join_kernel, dim3((unsigned)((2 * C + 63) / 64), (unsigned)N), dim3(256), 0, s, a, d);
    MARS_LAUNCH_CHECK();
#define MARS_BAPPLY(TA, TB, VV)                                                                                                              \
    do {                                                                                                                                     \
        if (a.stream) hipLaunchKernelGGL((norm_bwd_apply_kernel<TA, TB, VV, true>), grid1, dim3(TH), 0, s, a, d);                             \
        else hipLaunchKernelGGL((norm_bwd_apply_kernel<TA, TB, VV, false>), grid1, dim3(TH), 0, s, a, d);                                     \
    } while (0)
    MARS_NORM_T(MARS_BAPPLY)
    MARS_LAUNCH_CHECK();
    return 0;
}

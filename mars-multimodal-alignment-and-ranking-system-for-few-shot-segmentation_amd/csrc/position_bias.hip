// Learned relative-position bias by buckets, and its gradient: for tokens on grids (a line is a grid of one row)
//
//   bias[h, (qy, qx), (ky, kx)] = table[by[ky - qy + qh - 1], bx[kx - qx + qw - 1], h]
//
// Both directions move the H Lq Lk floats of the bias once and compute next to nothing.  Forward: for one query row of the grid the bias
// depends on (ky, kx - qx) only, so a workgroup looks the few thousand distinct values up once into LDS and every
// output is one LDS read (consecutive lanes, consecutive words) and one coalesced store.  Backward: a thread owns one
// offset kx - qx of one grid-row offset ky - qy and adds up its diagonal, reading whole row pieces with its neighbours; the offsets
// of a bucket are joined in LDS, pieces in a second launch.  No atomics: the sums have one order.
#include "common.h"
#include "../../include/mars_hip.h"

namespace {

struct BiasArgs {
    const int32_t *by, *bx;
    int H, qh, qw, kh, kw, ny, nx;
    int64_t sh, sl;                 // strides of the bias (or its gradient): head, query row
};

// bucket (iy, ix) -> row of the table, or -1: an entry of a map outside the table stands for "no bias" and has no gradient
__device__ __forceinline__ int table_row(int y, int x, int ny, int nx) {
    return (unsigned)y < (unsigned)ny && (unsigned)x < (unsigned)nx ? y * nx + x : -1;
}

constexpr int FWD_LDS = 12288;      // floats: three workgroups a CU
constexpr int KXC = 4096;           // key columns a workgroup takes at most

// grid: x = key tiles (kyt * ncx + cx), y = qy * ncq + cq, z = head
__global__ __launch_bounds__(256) void bucket_bias_kernel(const float* __restrict__ table, const BiasArgs a, float* __restrict__ out, int qxn,
                                                          int ncq, int kyn, int ncx) {
    __shared__ float e[FWD_LDS];
    const int tid = threadIdx.x, h = blockIdx.z;
    const int qy = blockIdx.y / ncq, qx0 = (blockIdx.y - qy * ncq) * qxn, nq = min(qxn, a.qw - qx0);
    const int kyt = blockIdx.x / ncx, ky0 = kyt * kyn, nky = min(kyn, a.kh - ky0);
    const int kx0 = (blockIdx.x - kyt * ncx) * KXC, nkx = min(KXC, a.kw - kx0);
    // e[y][x]: offset (ky0 + y - qy, kx0 + x - (qx0 + nq - 1))
    const int ew = nq + nkx - 1;
    for (int i = tid; i < nky * ew; i += 256) {
        const int y = i / ew, x = i - y * ew;
        const int row = table_row(a.by[ky0 + y - qy + a.qh - 1], a.bx[kx0 + x - (qx0 + nq - 1) + a.qw - 1], a.ny, a.nx);
        e[i] = row < 0 ? 0.f : table[(int64_t)row * a.H + h];
    }
    __syncthreads();
    float* o = out + h * a.sh + ((int64_t)qy * a.qw + qx0) * a.sl + (int64_t)ky0 * a.kw + kx0;
    for (int i = tid; i < nky * nkx; i += 256) {
        const int y = i / nkx, x = i - y * nkx;
        const float* er = e + y * ew + x + nq - 1;
        float* oi = o + (int64_t)y * a.kw + x;
        for (int q = 0; q < nq; ++q) oi[q * a.sl] = er[-q];
    }
}

constexpr int DXC = 512;            // offsets a workgroup takes
constexpr int ROWC = 1024;          // query rows a workgroup takes

// grid: x = row chunk * ndx + offset chunk, y = grid-row offset dy, z = head.  part[h][dy][x][nx]
__global__ __launch_bounds__(512) void bucket_bias_grad_kernel(const float* __restrict__ g, const BiasArgs a, float* __restrict__ part, int ndx) {
    __shared__ float acc[512 + DXC + 512];      // [row subset][offset], sums an offset, [wave][bucket]
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, h = blockIdx.z, dy = blockIdx.y;
    const int chunk = blockIdx.x / ndx, dx0 = (blockIdx.x - chunk * ndx) * DXC;
    const int nd_all = a.qw + a.kw - 1, nd = min(DXC, nd_all - dx0);
    const int nblk = (nd + 63) / 64;                                // waves that the offsets take: 1 .. 8
    const int subs = 8 / nblk;                                      // row subsets
    const int sub = wave / nblk, dxb = wave - sub * nblk;
    const int oy = dy - (a.qh - 1);                                 // ky - qy
    const int Lq = a.qh * a.qw;
    // query rows of this chunk whose ky exists
    const int qlo = max(0, -oy), qhi = min(a.qh, a.kh - oy);
    const int r0 = max(chunk * ROWC, qlo * a.qw), r1 = min(min((chunk + 1) * ROWC, Lq), qhi * a.qw);
    if (sub < subs) {
        float s = 0.f;
        const int dx = dx0 + dxb * 64 + lane, ox = dx - (a.qw - 1);
        if (r0 < r1) {
            const float* gh = g + h * a.sh;
            int r = r0 + sub;
            int qy = r / a.qw, qx = r - qy * a.qw;
            constexpr int U = 8;
            while (r < r1) {
                float v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int kx = qx + ox;
                    const bool on = r < r1 && dx < nd_all && (unsigned)kx < (unsigned)a.kw;
                    v[u] = on ? gh[(int64_t)r * a.sl + (int64_t)(qy + oy) * a.kw + kx] : 0.f;
                    r += subs;
                    qx += subs;
                    while (qx >= a.qw) { qx -= a.qw; ++qy; }
                }
#pragma unroll
                for (int u = 0; u < U; ++u) s += v[u];
            }
        }
        acc[sub * nblk * 64 + dxb * 64 + lane] = s;
    }
    __syncthreads();
    // sums of an offset over the row subsets, then of a bucket over its offsets: 512 / nxp slices of the offsets a bucket
    float* tot = acc + 512;
    for (int i = tid; i < nd; i += 512) {
        float s = 0.f;
        for (int w = 0; w < subs; ++w) s += acc[w * nblk * 64 + i];
        tot[i] = s;
    }
    __syncthreads();
    float* res = tot + DXC;
    float* dst = part + (((int64_t)h * gridDim.y + dy) * gridDim.x + blockIdx.x) * a.nx;
    const int32_t* bx = a.bx + dx0;
    for (int b0 = 0; b0 < a.nx; b0 += 64) {
        const int bucket = b0 + lane;
        float s = 0.f;
        const int per = (nd + 7) / 8;
        if (bucket < a.nx)
            for (int i = wave * per; i < min(nd, (wave + 1) * per); ++i) s += bx[i] == bucket ? tot[i] : 0.f;
        __syncthreads();
        res[wave * 64 + lane] = s;
        __syncthreads();
        if (wave == 0 && bucket < a.nx) {
            float t = 0.f;
            for (int w = 0; w < 8; ++w) t += res[w * 64 + lane];
            dst[bucket] = t;
        }
    }
}

// dtable[iy][ix][h]: grid (ceil(nx / 64), ny, H); the four waves take the grid-row offsets in turn
__global__ __launch_bounds__(256) void bucket_bias_grad_join_kernel(const float* __restrict__ part, const BiasArgs a, float* __restrict__ dtable,
                                                                    int nparts) {
    __shared__ float acc[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ix = blockIdx.x * 64 + lane, iy = blockIdx.y, h = blockIdx.z;
    const int ndy = a.qh + a.kh - 1;
    float s = 0.f;
    if (ix < a.nx)
        for (int dy = 0; dy < ndy; ++dy) {
            if (a.by[dy] != iy) continue;
            const float* p = part + ((int64_t)h * ndy + dy) * nparts * a.nx + ix;
            for (int c = wave; c < nparts; c += 4) s += p[(int64_t)c * a.nx];
        }
    acc[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && ix < a.nx) dtable[((int64_t)iy * a.nx + ix) * a.H + h] = (acc[0][lane] + acc[1][lane]) + (acc[2][lane] + acc[3][lane]);
}

int bias_check(const char* what, const void* p, const int32_t* by, const int32_t* bx, const void* t, int H, int qh, int qw, int kh, int kw, int ny, int nx,
               int64_t sh, int64_t sl) {
    MARS_CHECK(p && by && bx && t, "%s: null pointer", what);
    MARS_CHECK(H > 0 && qh > 0 && qw > 0 && kh > 0 && kw > 0 && ny > 0 && nx > 0, "%s: empty shape", what);
    MARS_CHECK((int64_t)qh * qw < (1ll << 30) && (int64_t)kh * kw < (1ll << 30) && (int64_t)ny * nx < (1ll << 30), "%s: too many tokens or buckets", what);
    MARS_CHECK(H <= 65535, "%s: %d heads", what, H);
    MARS_CHECK(sl >= (int64_t)kh * kw && (H == 1 || sh >= (int64_t)(qh * qw - 1) * sl + (int64_t)kh * kw), "%s: rows overlap", what);
    return 0;
}

int grad_parts(int qh, int qw, int kw, int& ndx) {
    ndx = (qw + kw - 1 + DXC - 1) / DXC;
    return (int)(((int64_t)qh * qw + ROWC - 1) / ROWC) * ndx;
}

}  // namespace

extern "C" int marship_bucket_bias(const float* table, const int32_t* by, const int32_t* bx, float* out, int64_t s_head, int64_t s_row, int H, int qh,
                                   int qw, int kh, int kw, int ny, int nx, void* stream) {
    if (const int rc = bias_check("bucket_bias", table, by, bx, out, H, qh, qw, kh, kw, ny, nx, s_head, s_row)) return rc;
    const BiasArgs a{by, bx, H, qh, qw, kh, kw, ny, nx, s_head, s_row};
    const int ncq = (qw + 31) / 32, qxn = (qw + ncq - 1) / ncq;               // query columns a workgroup: up to 32, evenly
    const int ncx = (kw + KXC - 1) / KXC, ew = qxn + (kw < KXC ? kw : KXC) - 1;
    int kyn = FWD_LDS / ew;                                                    // (ew <= 4127: at least two key rows)
    if (kyn > kh) kyn = kh;
    const int64_t gx = (int64_t)((kh + kyn - 1) / kyn) * ncx, gy = (int64_t)qh * ncq;
    MARS_CHECK(gx * 256 < (1ll << 32) && gy <= 65535, "bucket_bias: more workgroups than a launch takes");
    hipLaunchKernelGGL(bucket_bias_kernel, dim3((unsigned)gx, (unsigned)gy, (unsigned)H), dim3(256), 0, (hipStream_t)stream, table, a, out, qxn, ncq, kyn,
                       ncx);
    MARS_LAUNCH_CHECK();
    return 0;
}

extern "C" int64_t marship_bucket_bias_bwd_ws(int H, int qh, int qw, int kh, int kw, int nx) {
    if (H <= 0 || qh <= 0 || qw <= 0 || kh <= 0 || kw <= 0 || nx <= 0) return 0;
    int ndx;
    return (int64_t)H * (qh + kh - 1) * grad_parts(qh, qw, kw, ndx) * nx * 4;
}

extern "C" int marship_bucket_bias_bwd(const float* dbias, int64_t s_head, int64_t s_row, const int32_t* by, const int32_t* bx, float* dtable, int H, int qh,
                                       int qw, int kh, int kw, int ny, int nx, void* ws, int64_t ws_bytes, void* stream) {
    if (const int rc = bias_check("bucket_bias_bwd", dbias, by, bx, dtable, H, qh, qw, kh, kw, ny, nx, s_head, s_row)) return rc;
    const int64_t need = marship_bucket_bias_bwd_ws(H, qh, qw, kh, kw, nx);
    MARS_CHECK(ws != nullptr && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "bucket_bias_bwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
               (long long)need);
    const BiasArgs a{by, bx, H, qh, qw, kh, kw, ny, nx, s_head, s_row};
    int ndx;
    const int nparts = grad_parts(qh, qw, kw, ndx);
    MARS_CHECK(qh + kh - 1 <= 65535 && ny <= 65535 && (int64_t)nparts * 512 < (1ll << 32), "bucket_bias_bwd: more workgroups than a launch takes");
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(bucket_bias_grad_kernel, dim3((unsigned)nparts, (unsigned)(qh + kh - 1), (unsigned)H), dim3(512), 0, s, dbias, a, (float*)ws, ndx);
    MARS_LAUNCH_CHECK();
    hipLaunchKernelGGL(bucket_bias_grad_join_kernel, dim3((unsigned)((nx + 63) / 64), (unsigned)ny, (unsigned)H), dim3(256), 0, s, (const float*)ws, a, dtable,
                       nparts);
    MARS_LAUNCH_CHECK();
    return 0;
}

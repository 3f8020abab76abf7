// Learned relative-position bias by buckets, and its gradient: for tokens on grids (a line is a grid of one row)
//
//   bias[h, (qy, qx), (ky, kx)] = table[by[ky - qy + qh - 1], bx[kx - qx + qw - 1], h]
//
// Both directions move the H Lq Lk floats of the bias once and compute next to nothing.  Forward: for one query row of the grid the bias
// depends on (ky, kx - qx) only, so a workgroup looks the few thousand distinct values up once into LDS and every
// output is one LDS read (consecutive lanes, consecutive words) and one coalesced store.  Backward: a thread owns offsets
// kx - qx and adds up their diagonals; the offsets of a bucket are joined in LDS, the workgroups' tables in a second launch.  No
// atomics: the sums have one order.  Two forms of the first launch: on grids with eight key rows or more a workgroup takes one query row of the
// grid with a wave for every eighth key row, so that it reads whole rows of the gradient; on lines its waves share the query rows.
// 16 heads, 37 x 37 grid, forward: 26 us (4.6 TB/s; 8 and 16 heads, 64 x 64 grid: 116 and 233 us, with stores past the caches 123 and 242); 8 heads, 64 x 64 grid, backward: 101 us (5.3 TB/s; the form for lines took 166 there).
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
constexpr int ROWC = 1024;          // query rows a workgroup takes: whole grid rows, or a piece of one

// grid: x = (grid-row chunk * ncq + column chunk) * ndx + offset chunk, y = grid-row offset dy, z = head.  part[h][dy][x][nx]
__global__ __launch_bounds__(512) void bucket_bias_grad_kernel(const float* __restrict__ g, const BiasArgs a, float* __restrict__ part, int ndx, int ncq,
                                                               int qyn) {
    __shared__ float acc[512];                  // [row subset][offset]
    __shared__ int mx[DXC];                     // buckets of this workgroup's offsets
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.z, dy = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rc = blockIdx.x / ndx, dx0 = (blockIdx.x - rc * ndx) * DXC;
    const int cy = rc / ncq, qx0 = (rc - cy * ncq) * ROWC, qx1 = min(qx0 + ROWC, a.qw);
    const int nd_all = a.qw + a.kw - 1, nd = min(DXC, nd_all - dx0);
    const int nblk = (nd + 63) / 64;                                // waves that the offsets take: 1 .. 8
    const int subs = 8 / nblk;                                      // row subsets
    const int sub = wave / nblk, dxb = wave - sub * nblk;
    const int oy = dy - (a.qh - 1);                                 // ky - qy
    // grid rows of this chunk whose ky exists
    const int qy0 = max(cy * qyn, -oy), qy1 = min(min((cy + 1) * qyn, a.qh), a.kh - oy);
    if (tid < nd) mx[tid] = a.bx[dx0 + tid];
    if (sub < subs) {
        float s = 0.f;
        const int dx = dx0 + dxb * 64 + lane, ox = dx < nd_all ? dx - (a.qw - 1) : a.kw;        // (an offset that does not exist: kx is never on the grid)
        // columns for which some lane of the wave has a key: qx + ox in [0, kw)
        const int o_lo = dx0 + dxb * 64 - (a.qw - 1), o_hi = min(dx0 + dxb * 64 + 63, nd_all - 1) - (a.qw - 1);
        const int lo = max(qx0, -o_hi), hi = min(qx1, a.kw - o_lo);
        const int64_t step = (a.sl + 1) * subs;                     // to the same offset in the row `subs` further
        for (int qy = qy0; qy < qy1; ++qy) {
            const float* p = g + h * a.sh + ((int64_t)qy * a.qw + lo + sub) * a.sl + (int64_t)(qy + oy) * a.kw + (lo + sub + ox);
            constexpr int U = 16;                                   // loads in flight
            for (int qx = lo + sub; qx < hi; qx += U * subs) {
                float v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) {
                    const int q = qx + u * subs;
                    v[u] = q < hi && (unsigned)(q + ox) < (unsigned)a.kw ? p[u * step] : 0.f;
                }
#pragma unroll
                for (int u = 0; u < U; ++u) s += v[u];
                p += U * step;
            }
        }
        acc[sub * nblk * 64 + dxb * 64 + lane] = s;
    }
    __syncthreads();
    // an offset's sum over the row subsets: lane l of every wave holds offsets l, l + 64, ...; then each wave takes buckets in turn
    float tot[DXC / 64];
    int bucket[DXC / 64];
#pragma unroll
    for (int j = 0; j < DXC / 64; ++j) {
        const int i = lane + 64 * j;
        tot[j] = 0.f;
        bucket[j] = i < nd ? mx[i] : -1;
        if (i < nd)
            for (int w = 0; w < subs; ++w) tot[j] += acc[w * nblk * 64 + i];
    }
    float* dst = part + (((int64_t)h * gridDim.y + dy) * gridDim.x + blockIdx.x) * a.nx;
    for (int b = wave; b < a.nx; b += 8) {
        float s = 0.f;
#pragma unroll
        for (int j = 0; j < DXC / 64; ++j) s += bucket[j] == b ? tot[j] : 0.f;
        s = wave_sum(s);
        if (lane == 0) dst[b] = s;
    }
}

constexpr int GKY = 64, GDX = 128;  // key rows and offsets a workgroup of the grid form takes

// grid: x = ((qy * ncq + cq) * nky + cky) * ndx + cdx, y = head.  part[h][x][ny][nx]
template <int KJ>
__global__ __launch_bounds__(512) void bucket_bias_grad_rows_kernel(const float* __restrict__ g, const BiasArgs a, float* __restrict__ part, int ncq, int qxn,
                                                                    int nky, int ndx) {
    __shared__ float e[GKY][GDX + 1];           // sums a (key row, offset)
    __shared__ float t[GKY][64 + 1];            // sums a (key row, bucket of the row axis), 64 buckets at a time
    __shared__ int mx[GDX], my[GKY];            // buckets of this workgroup's offsets and key rows
    const int tid = threadIdx.x, lane = tid & 63, h = blockIdx.y;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int id = blockIdx.x;
    const int dx0 = (id % ndx) * GDX; id /= ndx;
    const int ky0 = (id % nky) * GKY; id /= nky;
    const int qx0 = (id % ncq) * qxn, qx1 = min(qx0 + qxn, a.qw), qy = id / ncq;
    const int nd_all = a.qw + a.kw - 1, nd = min(GDX, nd_all - dx0), nk = min(GKY, a.kh - ky0);
    // this wave's key rows: ky0 + wave, + 8, ...; a lane's offsets: dx0 + lane, + 64
    if (tid < nd) mx[tid] = a.bx[dx0 + tid];
    if (tid < nk) my[tid] = a.by[ky0 + tid - qy + a.qh - 1];
    float s[KJ][2];
#pragma unroll
    for (int j = 0; j < KJ; ++j) s[j][0] = s[j][1] = 0.f;
    const int ox0 = dx0 + lane < nd_all ? dx0 + lane - (a.qw - 1) : a.kw, ox1 = dx0 + lane + 64 < nd_all ? dx0 + lane + 64 - (a.qw - 1) : a.kw;   // (kw: never on the grid)
    int at[KJ];                                                     // bytes to a key row (one that does not exist: the last one, not used below)
#pragma unroll
    for (int j = 0; j < KJ; ++j) at[j] = min(ky0 + wave + 8 * j, a.kh - 1) * a.kw * 4;
    const float* row = g + h * a.sh + ((int64_t)qy * a.qw + qx0) * a.sl;
    // Lanes without a key read behind the end of a buffer resource over the row, which gives 0 and no traffic: with a branch around every load the
    // loop was bound by them (189 us for a 64 x 64 grid and eight heads)
    constexpr int U = 32 / KJ < 4 ? 4 : 32 / KJ, NOWHERE = (int)0x80000000;      // query columns whose loads are in flight together
    for (int qx = qx0; qx < qx1; qx += U) {
        float v[U][KJ][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int q = min(qx + u, qx1 - 1), past = qx + u < qx1 ? 0 : NOWHERE;   // (columns behind the last: the sign bit takes any offset off the grid)
            const auto rsrc = __builtin_amdgcn_make_buffer_rsrc((void*)(row + (int64_t)(q - qx0) * a.sl), 0, a.kh * a.kw * 4, 0x00027000);
            const int o0 = (unsigned)((q + ox0) | past) < (unsigned)a.kw ? (q + ox0) * 4 : NOWHERE;
            const int o1 = (unsigned)((q + ox1) | past) < (unsigned)a.kw ? (q + ox1) * 4 : NOWHERE;
#pragma unroll
            for (int j = 0; j < KJ; ++j) {
                v[u][j][0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, o0, at[j], 0));
                v[u][j][1] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rsrc, o1, at[j], 0));
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < KJ; ++j) { s[j][0] += v[u][j][0]; s[j][1] += v[u][j][1]; }
    }
#pragma unroll
    for (int j = 0; j < KJ; ++j) { e[wave + 8 * j][lane] = s[j][0]; e[wave + 8 * j][lane + 64] = s[j][1]; }
    __syncthreads();
    float* dst = part + ((int64_t)h * gridDim.x + blockIdx.x) * a.ny * a.nx;
    // Buckets of the row axis, then of the grid rows.  Which offsets (key rows) a bucket has is one bit mask for the whole wave, so each sum is
    // read once and by the lanes side by side; a compare an output and offset would take longer than reading the gradient.
    const int m0 = lane < nd ? mx[lane] : -1, m1 = lane + 64 < nd ? mx[lane + 64] : -1, mk = lane < nk ? my[lane] : -1;
    for (int b0 = 0; b0 < a.nx; b0 += 64) {
        const int nb = min(64, a.nx - b0);
        for (int b = wave; b < nb; b += 8) {
            float u = 0.f;                                          // lane: key row
            for (unsigned long long hit = __ballot(m0 == b0 + b); hit != 0; hit &= hit - 1) u += e[lane][__builtin_ctzll(hit)];
            for (unsigned long long hit = __ballot(m1 == b0 + b); hit != 0; hit &= hit - 1) u += e[lane][64 + __builtin_ctzll(hit)];
            t[lane][b] = u;
        }
        __syncthreads();
        for (int y = wave; y < a.ny; y += 8) {
            float u = 0.f;                                          // lane: bucket of the row axis
            for (unsigned long long hit = __ballot(mk == y); hit != 0; hit &= hit - 1) u += t[__builtin_ctzll(hit)][lane];
            if (lane < nb) dst[(int64_t)y * a.nx + b0 + lane] = u;
        }
        __syncthreads();
    }
}

// dtable[iy][ix][h] of the grid form's tables: grid (ceil(ny nx / 64), H), four waves take the tables in turn
__global__ __launch_bounds__(256) void bucket_bias_grad_rows_join_kernel(const float* __restrict__ part, const BiasArgs a, float* __restrict__ dtable, int nparts) {
    __shared__ float acc[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.y, n = a.ny * a.nx, i = blockIdx.x * 64 + lane;
    const float* p = part + (int64_t)h * nparts * n + min(i, n - 1);
    float s = 0.f;
    constexpr int U = 8;
    for (int c = wave; c < nparts; c += 4 * U) {
        float v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) v[u] = c + 4 * u < nparts ? p[(int64_t)(c + 4 * u) * n] : 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u) s += v[u];
    }
    acc[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && i < n) dtable[(int64_t)i * a.H + h] = (acc[0][lane] + acc[1][lane]) + (acc[2][lane] + acc[3][lane]);
}

// dtable[iy][ix][h]: grid (ceil(nx / 64), ny, H); the four waves take the grid-row offsets in turn, 64 of them looked at in one load
__global__ __launch_bounds__(256) void bucket_bias_grad_join_kernel(const float* __restrict__ part, const BiasArgs a, float* __restrict__ dtable,
                                                                    int nparts) {
    __shared__ float acc[4][64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, ix = blockIdx.x * 64 + lane, iy = blockIdx.y, h = blockIdx.z;
    const int ndy = a.qh + a.kh - 1;
    float s = 0.f;
    for (int d0 = 0; d0 < ndy; d0 += 64) {
        unsigned long long hit = __ballot(d0 + lane < ndy && a.by[min(d0 + lane, ndy - 1)] == iy);
        while (hit != 0) {
            const int dy = d0 + __builtin_ctzll(hit);
            hit &= hit - 1;
            const float* p = part + ((int64_t)h * ndy + dy) * nparts * a.nx + min(ix, a.nx - 1);
            constexpr int U = 8;
            for (int c = wave; c < nparts; c += 4 * U) {
                float v[U];
#pragma unroll
                for (int u = 0; u < U; ++u) v[u] = c + 4 * u < nparts ? p[(int64_t)(c + 4 * u) * a.nx] : 0.f;
#pragma unroll
                for (int u = 0; u < U; ++u) s += v[u];
            }
        }
    }
    acc[wave][lane] = s;
    __syncthreads();
    if (wave == 0 && ix < a.nx) dtable[((int64_t)iy * a.nx + ix) * a.H + h] = (acc[0][lane] + acc[1][lane]) + (acc[2][lane] + acc[3][lane]);
}

// what the workspace query asks too: beyond these the counts of workgroups leave their types; it answers 0 for a shape that the call refuses
int shape_check(const char* what, int H, int qh, int qw, int kh, int kw, int ny, int nx) {
    MARS_CHECK(H > 0 && qh > 0 && qw > 0 && kh > 0 && kw > 0 && ny > 0 && nx > 0, "%s: empty shape", what);
    MARS_CHECK((int64_t)qh * qw < (1ll << 29) && (int64_t)kh * kw < (1ll << 29) && (int64_t)ny * nx < (1ll << 30), "%s: too many tokens or buckets", what);
    MARS_CHECK(H <= 65535, "%s: %d heads", what, H);
    return 0;
}

int bias_check(const char* what, const void* p, const int32_t* by, const int32_t* bx, const void* t, int H, int qh, int qw, int kh, int kw, int ny, int nx,
               int64_t sh, int64_t sl) {
    MARS_CHECK(p && by && bx && t, "%s: null pointer", what);
    if (const int rc = shape_check(what, H, qh, qw, kh, kw, ny, nx)) return rc;
    MARS_CHECK(sl >= (int64_t)kh * kw && (H == 1 || sh >= (int64_t)(qh * qw - 1) * sl + (int64_t)kh * kw), "%s: rows overlap", what);
    return 0;
}

// the gradient's first launch cut into workgroups: `parts` of them for one head (grid form), or for one head and grid-row offset
struct GradCut { bool rows; int ndx, ncq, qyn, qxn, nky; int64_t parts; };
GradCut grad_cut(int H, int qh, int qw, int kh, int kw) {
    GradCut c{};
    c.rows = kh >= 8;
    if (c.rows) {
        c.ndx = (qw + kw - 1 + GDX - 1) / GDX;
        c.nky = (kh + GKY - 1) / GKY;
        const int64_t wgs = (int64_t)H * qh * c.ndx * c.nky;
        c.ncq = wgs >= 512 ? 1 : (int)((512 + wgs - 1) / wgs);      // few grid rows: pieces of them
        if (c.ncq > (qw + 7) / 8) c.ncq = (qw + 7) / 8;
        c.qxn = (qw + c.ncq - 1) / c.ncq;
        c.ncq = (qw + c.qxn - 1) / c.qxn;
        c.parts = (int64_t)qh * c.ncq * c.nky * c.ndx;
        return c;
    }
    c.ndx = (qw + kw - 1 + DXC - 1) / DXC;
    c.ncq = (qw + ROWC - 1) / ROWC;
    c.qyn = qw >= ROWC ? 1 : ROWC / qw;
    c.parts = (int64_t)((qh + c.qyn - 1) / c.qyn) * c.ncq * c.ndx;
    return c;
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
    hipLaunchKernelGGL(bucket_bias_kernel, dim3((unsigned)gx, (unsigned)gy, (unsigned)H), dim3(256), 0, (hipStream_t)stream, table, a, out, qxn, ncq, kyn, ncx);
    MARS_LAUNCH_CHECK();
    return 0;
}

extern "C" int64_t marship_bucket_bias_bwd_ws(int H, int qh, int qw, int kh, int kw, int ny, int nx) {
    if (shape_check("bucket_bias_bwd_ws", H, qh, qw, kh, kw, ny, nx) != 0) return 0;
    const GradCut c = grad_cut(H, qh, qw, kh, kw);
    return (int64_t)H * c.parts * (c.rows ? (int64_t)ny * nx : (int64_t)(qh + kh - 1) * nx) * 4;
}

extern "C" int marship_bucket_bias_bwd(const float* dbias, int64_t s_head, int64_t s_row, const int32_t* by, const int32_t* bx, float* dtable, int H, int qh,
                                       int qw, int kh, int kw, int ny, int nx, void* ws, int64_t ws_bytes, void* stream) {
    if (const int rc = bias_check("bucket_bias_bwd", dbias, by, bx, dtable, H, qh, qw, kh, kw, ny, nx, s_head, s_row)) return rc;
    const int64_t need = marship_bucket_bias_bwd_ws(H, qh, qw, kh, kw, ny, nx);
    MARS_CHECK(ws != nullptr && (uintptr_t)ws % 16 == 0 && ws_bytes >= need, "bucket_bias_bwd: workspace of %lld bytes, %lld needed", (long long)ws_bytes,
               (long long)need);
    const BiasArgs a{by, bx, H, qh, qw, kh, kw, ny, nx, s_head, s_row};
    const GradCut c = grad_cut(H, qh, qw, kh, kw);
    if (c.rows) {
        MARS_CHECK(c.parts * 512 < (1ll << 32), "bucket_bias_bwd: more workgroups than a launch takes");
        const dim3 grid((unsigned)c.parts, (unsigned)H);
#define MARS_GRAD_ROWS(KJ)                                                                                                                                  \
    case KJ: hipLaunchKernelGGL((bucket_bias_grad_rows_kernel<KJ>), grid, dim3(512), 0, (hipStream_t)stream, dbias, a, (float*)ws, c.ncq, c.qxn, c.nky, c.ndx); break
        switch (((kh < GKY ? kh : GKY) + 7) / 8) {                  // key rows a wave
            MARS_GRAD_ROWS(1); MARS_GRAD_ROWS(2); MARS_GRAD_ROWS(3); MARS_GRAD_ROWS(4);
            MARS_GRAD_ROWS(5); MARS_GRAD_ROWS(6); MARS_GRAD_ROWS(7);
            default: hipLaunchKernelGGL((bucket_bias_grad_rows_kernel<8>), grid, dim3(512), 0, (hipStream_t)stream, dbias, a, (float*)ws, c.ncq, c.qxn, c.nky, c.ndx);
        }
#undef MARS_GRAD_ROWS
        MARS_LAUNCH_CHECK();
        hipLaunchKernelGGL(bucket_bias_grad_rows_join_kernel, dim3((unsigned)((ny * nx + 63) / 64), (unsigned)H), dim3(256), 0, (hipStream_t)stream,
                           (const float*)ws, a, dtable, (int)c.parts);
        MARS_LAUNCH_CHECK();
        return 0;
    }
    MARS_CHECK(qh + kh - 1 <= 65535 && ny <= 65535 && c.parts * 512 < (1ll << 32), "bucket_bias_bwd: more workgroups than a launch takes");
    hipStream_t s = (hipStream_t)stream;
    hipLaunchKernelGGL(bucket_bias_grad_kernel, dim3((unsigned)c.parts, (unsigned)(qh + kh - 1), (unsigned)H), dim3(512), 0, s, dbias, a, (float*)ws, c.ndx, c.ncq,
                       c.qyn);
    MARS_LAUNCH_CHECK();
    hipLaunchKernelGGL(bucket_bias_grad_join_kernel, dim3((unsigned)((nx + 63) / 64), (unsigned)ny, (unsigned)H), dim3(256), 0, s, (const float*)ws, a, dtable,
                       (int)c.parts);
    MARS_LAUNCH_CHECK();
    return 0;
}

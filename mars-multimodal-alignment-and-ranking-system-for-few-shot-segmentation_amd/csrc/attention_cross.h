// Device pieces shared by the forward and backward kernels of the attention between two token sets
// (attention_cross.hip, attention_cross_bwd.hip).
//
// Everything runs on the 32x32 matrix instructions with one fragment shape for both types: a fragment is eight
// consecutive elements of row (lane & 31), elements 8 (lane >> 5) .. + 7 of a contraction step of 16.  For bf16 that is
// one v_mfma_f32_32x32x16_bf16; for f32 the eight elements go through eight v_mfma_f32_32x32x2_f32, of which number e
// contracts elements e and 8 + e (any order of the contraction will do as long as both operands agree).  A product
// leaves column (lane & 31) and rows 8 (i >> 2) + 4 (lane >> 5) + (i & 3) in accumulator register i, and registers
// 8u .. 8u + 7 are, as they stand, the B operand of contraction step u of a following product whose A operand is read
// transposed (read_cols): no value crosses lanes between the two products of an attention.
#pragma once
#include "common.h"
#include "../../include/mars_hip.h"

namespace xattn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void* lds_ptr_t;
typedef __attribute__((address_space(3))) unsigned char* lds_t;          // a tile in LDS
typedef const __attribute__((address_space(1))) void* gbl_ptr_t;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;
typedef const __attribute__((address_space(3))) bf16x8* lds_bf16x8_t;
typedef const __attribute__((address_space(3))) f32x4* lds_f32x4_t;
typedef const __attribute__((address_space(3))) float* lds_f32_t;

static __device__ uint4 zero_chunk;          // 16 bytes of zeros: what a fill reads behind the end of a row

constexpr float LOG2E = 1.4426950408889634f;

template <typename T> struct FragOf;
template <> struct FragOf<__bf16> { typedef bf16x8 type; };
template <> struct FragOf<float> { typedef f32x8 type; };
template <typename T> using frag_t = typename FragOf<T>::type;

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

__device__ __forceinline__ f32x16 zero16() {
    f32x16 z;
#pragma unroll
    for (int i = 0; i < 16; ++i) z[i] = 0.f;
    return z;
}

// accumulator registers 8u .. 8u + 7 as the B operand of contraction step u
template <typename T> __device__ __forceinline__ frag_t<T> pack_step(const f32x16& s, int u) {
    frag_t<T> r;
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = (T)s[8 * u + e];
    return r;
}

// row of accumulator register i in a 32-row block
__device__ __forceinline__ int acc_row(int i, int hh) { return 8 * (i >> 2) + 4 * hh + (i & 3); }

// the larger of two values, NaN if one is (v_maximum3_f32; fmaxf would first quieten each operand with an instruction of its own)
__device__ __forceinline__ float vmax(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// x of this lane combined with x of the same column in the other half-wave
__device__ __forceinline__ float halves_sum(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
__device__ __forceinline__ float halves_max(float x) {
    const unsigned u = __builtin_bit_cast(unsigned, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return vmax(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}

// The kernels are built for head dims HD of 16, 32, 64, 80, 96 and 128; a head is zero-padded to the next of them for the products that contract
// over it, and to a multiple of 32 (HDP) where its elements are the rows of a product.
constexpr int padded(int HD) { return (HD + 31) / 32 * 32; }
inline int built_for(int hd) { return hd <= 16 ? 16 : hd <= 32 ? 32 : hd <= 64 ? 64 : hd <= 80 ? 80 : hd <= 96 ? 96 : 128; }

// ---- LDS tiles: rows of HDP elements in 16-byte chunks, filled by LDS-DMA.  Chunk c of row r sits at slot
// c ^ swizzle(r): of the rows that a fragment read touches with one chunk number, those whose row starts fall on the same
// banks (64 banks of 4 bytes) use different slots.
template <typename T, int HDP> struct Tile {
    static constexpr int ROWB = HDP * (int)sizeof(T), LPR = ROWB / 16;
    static __device__ __forceinline__ int swizzle(int r) {
        if constexpr (LPR % 16 == 0) return r & 15;
        else if constexpr (LPR % 8 == 0) return (r >> 1) & 7;
        else return (r >> 2) & 3;
    }
    // rows [0, NR) by NW waves of which this is number w: fill number i of a lane is 16 bytes of row row_of_fill(i) (FILLS of them)
    template <int NR, int NW> struct Fill {
        static constexpr int PIECES = NR * LPR / 64, FILLS = (PIECES + NW - 1) / NW;
        static_assert(NR * LPR % 64 == 0, "a tile is a whole number of 1-KiB pieces");
        static __device__ __forceinline__ int row_of_fill(int i, int w, int lane) { return ((w + i * NW) * 64 + lane) / LPR; }
        // at(i): the first byte of fill i's row; hdb: bytes of a row that exist (the rest is zeros).  Straight-line code: a branch or a wait
        // between two fills would hold up the later ones by a trip to memory
        template <typename F> static __device__ __forceinline__ void run(lds_t dst, int w, int lane, int hdb, F at) {
            const unsigned char* zeros = (const unsigned char*)&zero_chunk;
#pragma unroll
            for (int i = 0; i < FILLS; ++i) {
                const int p = w + i * NW;
                if (PIECES % NW == 0 || p < PIECES) {
                    const int c = p * 64 + lane, row = c / LPR, slot = c - row * LPR, byte = (slot ^ swizzle(row)) * 16;
                    const unsigned char* s = at(i) + byte;
                    s = byte < hdb ? s : zeros;
                    __builtin_amdgcn_global_load_lds((gbl_ptr_t)s, (lds_ptr_t)(dst + p * 1024), 16, 0, 0);
                }
            }
        }
    };
    // fragment of rows r0 + (lane & 31), contraction step ks over the row's elements
    static __device__ __forceinline__ frag_t<T> rows(lds_t t, int r0, int ks, int lane) {
        const int row = r0 + (lane & 31), hh = lane >> 5, sw = swizzle(row);
        if constexpr (sizeof(T) == 2) {
            return *(lds_bf16x8_t)(t + row * ROWB + (((2 * ks + hh) ^ sw) << 4));
        } else {
            const f32x4 a = *(lds_f32x4_t)(t + row * ROWB + (((4 * ks + 2 * hh) ^ sw) << 4));
            const f32x4 b = *(lds_f32x4_t)(t + row * ROWB + (((4 * ks + 2 * hh + 1) ^ sw) << 4));
            return (f32x8){a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    // fragment of columns 32 m + (lane & 31): its elements are rows r0 + 8 (e >> 2) + 4 (lane >> 5) + (e & 3), the rows that pack_step's
    // registers belong to
    static __device__ __forceinline__ frag_t<T> cols(lds_t t, int r0, int m, int lane) {
        const int hh = lane >> 5;
        if constexpr (sizeof(T) == 2) {
            // ds_read_b64_tr_b16: sixteen lanes read four rows of sixteen 16-bit columns and each gets one column
            const int i = lane & 15, chunk = 4 * m + 2 * ((lane >> 4) & 1) + ((i & 3) >> 1);
            const int ra = r0 + 4 * hh + (i >> 2), rb = ra + 8;
            const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(t + ra * ROWB + ((chunk ^ swizzle(ra)) << 4) + 8 * (i & 1)));
            const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(t + rb * ROWB + ((chunk ^ swizzle(rb)) << 4) + 8 * (i & 1)));
            return __builtin_bit_cast(bf16x8, (s16x8){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
        } else {
            const int d = 32 * m + (lane & 31), chunk = d >> 2;
            f32x8 r;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int row = r0 + 8 * (e >> 2) + 4 * hh + (e & 3);
                r[e] = *(lds_f32_t)(t + row * ROWB + ((chunk ^ swizzle(row)) << 4) + 4 * (d & 3));
            }
            return r;
        }
    }
};

// sixteen bias values of a query row for 32 keys from j0, in the order of an accumulator: keys j0 + acc_row(i).  WHOLE: all 32 keys exist and
// stand in order, four of them a load (rows of any alignment); otherwise by the list of attended keys, the last one again behind its end
typedef float f32x4_any __attribute__((ext_vector_type(4), aligned(4)));
template <bool WHOLE> __device__ __forceinline__ void load_bias(float (&v)[16], const float* row, const int32_t* idx, int j0, int n, int hh) {
    if (row == nullptr) {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = 0.f;
        return;
    }
    if (WHOLE && idx == nullptr) {
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const f32x4_any x = *(const f32x4_any*)(row + j0 + 8 * a + 4 * hh);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * a + e] = x[e];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int j = min(j0 + 8 * (i >> 2) + 4 * hh + (i & 3), n - 1);
        v[i] = row[idx == nullptr ? j : idx[j]];
    }
}

// The barrier between a tile's fills and its reads.  A wave's own LDS reads wait for the wave's own fills, but nothing waits for the other
// waves': each wave drains its fills (vmcnt 0) before it arrives.
__device__ __forceinline__ void tile_barrier() {
    __builtin_amdgcn_s_waitcnt(0x0f70);
    __syncthreads();
}

// fragment ks of a row in memory (nullptr: zeros); hd: elements of the row that exist, a multiple of 16 bytes
template <typename T> __device__ __forceinline__ frag_t<T> load_frag(const T* row, int ks, int hh, int hd) {
    frag_t<T> f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (T)0.f;
    const int c = 16 * ks + 8 * hh;
    if (row == nullptr) return f;
    if constexpr (sizeof(T) == 2) {
        if (c < hd) f = *(const bf16x8*)(row + c);
    } else {
        if (c < hd) { const f32x4 a = *(const f32x4*)(row + c); f[0] = a[0]; f[1] = a[1]; f[2] = a[2]; f[3] = a[3]; }
        if (c + 4 < hd) { const f32x4 a = *(const f32x4*)(row + c + 4); f[4] = a[0]; f[5] = a[1]; f[6] = a[2]; f[7] = a[3]; }
    }
    return f;
}

template <typename T> __device__ __forceinline__ void store4(T* p, float a, float b, float c, float d) {
    if constexpr (sizeof(T) == 2) *(bf16x4*)p = (bf16x4){(__bf16)a, (__bf16)b, (__bf16)c, (__bf16)d};
    else *(f32x4*)p = (f32x4){a, b, c, d};
}

// ---- problem description as the kernels take it.  The query rows of the heads that share a key head are one list of
// R = grp Lq rows: row r is token r % Lq of head hk grp + r / Lq, so that a key head's K and V are read once for all of them
// (one new token a sequence: the rows of a block ARE the heads of a group) and the gradients of K and V sum over them.
struct Strides { int64_t b, l, h; };
struct Prob {
    const void *q, *k, *v, *out, *dout;
    Strides sq, sk, sv, so, sdo;
    const float* bias;
    int64_t bias_h, bias_l;
    const float* stat;              // backward
    const int32_t* idx;             // [B, Lk]: attended keys of a batch entry in order, the others behind them (nullptr: key j is row j)
    const int32_t* cnt;             // [B]: attended keys (nullptr: Lk)
    int B, Lq, Lk, H, Hkv, grp, R, hd;
    float scale;
};

__device__ __forceinline__ int key_count(const Prob& p, int b) {
    return p.cnt == nullptr ? p.Lk : min(max(p.cnt[b], 0), p.Lk);
}
__device__ __forceinline__ int key_row(const int32_t* idx, int j) { return idx == nullptr ? j : idx[j]; }
// token and head of row r
__device__ __forceinline__ void row_of(const Prob& p, int hk, int r, int& l, int& h) {
    if (p.grp == 1) { l = r; h = hk; }
    else { const int a = r / p.Lq; l = r - a * p.Lq; h = hk * p.grp + a; }
}
template <typename T> __device__ __forceinline__ const T* row_ptr(const void* base, const Strides& s, int b, int l, int h) {
    return (const T*)base + b * s.b + l * s.l + h * s.h;
}

// Workgroup id -> (batch entry and key head, block).  The blocks of one (entry, head) read the same rows of the other operand; ids that are
// equal mod 8 share an XCD and its L2, so they walk the blocks of one (entry, head) after the other.  Entries beyond the last
// full group of eight keep the launch order.  (A matter of speed only.)
__device__ __forceinline__ void place_block(int id, int nbh, int nblk, int& bh, int& blk) {
    const int full = (nbh >> 3) * 8 * nblk;
    if (id < full) {
        const int x = id & 7, j = id >> 3;
        bh = (j / nblk) * 8 + x;
        blk = j % nblk;
    } else {
        bh = id / nblk;
        blk = id % nblk;
    }
}

// key tiles [t0, t1) of split s of ns
__device__ __forceinline__ void split_range(int tiles, int s, int ns, int& t0, int& t1) {
    const int per = (tiles + ns - 1) / ns;
    t0 = min(s * per, tiles);
    t1 = min(t0 + per, tiles);
}

// host side (attention_cross.hip)
int check(const MarsCrossAttn* a, bool backward);
void describe(const MarsCrossAttn* a, Prob& p);
int prepare_keys(const MarsCrossAttn* a, Prob& p, int32_t* ws, hipStream_t s);
int64_t key_ws_bytes(const MarsCrossAttn* a);

}  // namespace xattn

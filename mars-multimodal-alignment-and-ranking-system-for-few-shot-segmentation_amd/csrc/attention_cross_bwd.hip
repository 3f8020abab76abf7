// Gradients of the attention between two token sets (attention_cross.hip).  With P the softmax, recomputed tile by tile from
// the row statistics of the forward pass:
//
//   D_i = dO_i . O_i     dP = dO V^T     dS = P (dP - D)     dV = P^T dO     dQ = scale dS K     dK = scale dS^T Q     dbias = sum_b dS
//
// Three passes, none with atomics, so that every sum has one order:
//   queries  a wave owns 32 query rows and walks the keys: S^T = K Q^T and dP^T = V dO^T with the query as lane column, dS^T is the
//            operand of dQ^T += K^T dS^T.  It also makes D and leaves the row values for the other passes, 32 rows a block.
//            bf16: the stored O is rounded, and D' = dO . O with it (half a step of each O_d, against a D that is a small difference of
//            large terms) put 3e-3 into dbias and took dQ from 1.7e-3 to 2.6e-3.  But sum_j P (dP - D') = D - D' exactly: the pass works
//            with D', adds up e = sum_j dS' in f32 and R = sum_j P_j K_j, and ends with dQ = scale (sum dS' K - e R) and D = D' + e.
//            One product more in this pass, and no second copy of O in memory.
//   keys     a wave owns 32 keys and walks the query rows of every head that shares them: S = Q K^T, dP = dO V^T with the key as
//            lane column; P and dS are the operands of dV^T += dO^T P and dK^T += Q^T dS.
//   bias     (only where its gradient is asked for) a wave owns a 32 x 64 piece of one head's scores and walks the batch.
// With one attended key P is 1 whatever the score and dS is 0: dQ, dK and dbias are set to it, because dP - D is the difference of two roundings of one number.
// Recomputing S and dP in each pass costs 2 of 7 products more than one pass over all would, but that one would add into dQ from
// every key block: atomics, in an order that changes.
// 8 x 16 heads of 64, 1369 queries over 684 keys on average: queries 87 us, keys 107 (705 and 575 TFLOP/s of their own products); 2 x 16 heads of 80,
// 4096 x 4096: 376 and 430 us in a kernel trace, 741 as a call without one.
#include <type_traits>
#include "attention_cross.h"

namespace xattn {

int64_t bwd_ws_bytes(const MarsCrossAttn* a);

namespace {

// Row values of 32 query rows: 128 floats - [0, 32) offset of the exponent, [32, 64) factor of the exponential (bias only), [64, 96) D.
// Without a bias P = 2^(c2 s - offset) with offset = log2(e) maximum + log2(sum).  With one, P = 2^((s - offset) log2 e) factor with offset = maximum
// and factor = 1 / sum: where the mask is the type's lowest value the sum's logarithm would be lost in the maximum.
// Rows that do not exist or have no key: offset +inf and factor 0, so that the exponential itself is 0 whatever the score.  (The key pass holds the last row
// again in their place: with an offset of 0 a score above 88.7 of it would be inf * 0.)
constexpr int RSB = 128;
constexpr int FEW_KEYS = 256;           // see cross_bwd_q_kernel
// waves a SIMD that the two passes are built for (three of the key pass's would spill: 109 -> 142 us on eight 1369 x 684 x 16 heads of 64; the query
// pass with three, walking tiles of 32 keys: 98 -> 89)
template <typename T, int HDP, bool BIAS> constexpr int q_waves() { return sizeof(T) == 4 || HDP > 96 ? 1 : HDP > 64 || BIAS ? 2 : 3; }
template <typename T, int HDP> constexpr int kv_waves() { return sizeof(T) == 4 || HDP > 96 ? 1 : 2; }

struct Bwd {
    Prob p;
    void *dq, *dk, *dv;
    Strides sdq, sdk, sdv;
    float* dbias;
    int64_t dbias_h, dbias_l;
    const uint8_t* mask;
    const int32_t* kv_len;
    float* rows;                     // [B Hkv][nrb * 4][RSB]
    float *part_q, *part_k, *part_v; // [ns][..][HDP] partial sums, where a pass is split (part_q bf16: dS' K, then P K, of a row)
    float* part_e;                   // [nsq][B Hkv][R]: partial sums of dS'
    int nrb, nsq;                    // query pass: blocks of 128 rows, splits of the keys
    int by_count;                    // query pass: two launches, for entries of up to FEW_KEYS attended keys and for the others
    int nkb, nsk;                    // key pass: blocks of 128 keys, splits of the query rows
};

template <bool BIAS> __device__ __forceinline__ float prob(float s, float c2, float off, float fac) {
    return BIAS ? __builtin_amdgcn_exp2f((s - off) * LOG2E) * fac : __builtin_amdgcn_exp2f(fmaf(s, c2, -off));
}

// FINE (bf16, up to FEW_KEYS attended keys): what the rounding of dS leaves over goes through the matrix instruction too, and dQ is off by its own rounding alone
// (1.7e-3 in norm; 2.4e-3 with a rounded dS, up to 2.6e-3 where the keys are few).  A fifth product: nothing where the launch is the time, a fifth
// of this pass on long axes, where it is left out as it is for dK and dV.  How many keys of a long axis an entry attends to is known on the device alone:
// there both forms are launched and each takes its own entries (one kernel with both loops would need the registers of both).
template <typename T, int HD, bool BIAS, bool FINE>
__global__ __launch_bounds__(256, (q_waves<T, padded(HD), BIAS || FINE>())) void cross_bwd_q_kernel(const Bwd f) {
    constexpr int HDP = padded(HD);
    using TL = Tile<T, HDP>;
    constexpr int KT = (HDP > 64 && sizeof(T) == 4) || q_waves<T, HDP, BIAS || FINE>() == 3 ? 32 : 64, TB = KT * TL::ROWB, KB = KT / 32, KS = HD / 16, DM = HDP / 32;
    __shared__ __attribute__((aligned(16))) unsigned char buf0[2][TB];
    __shared__ __attribute__((aligned(16))) unsigned char buf1[2][TB];
    const Prob& p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bh, blk;
    place_block(blockIdx.x, p.B * p.Hkv, f.nrb * f.nsq, bh, blk);
    const int rb = blk % f.nrb, split = blk / f.nrb;
    const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
    const int r = rb * 128 + wave * 32 + (lane & 31);
    const bool row_ok = r < p.R;
    int l = 0, h = 0;
    if (row_ok) row_of(p, hk, r, l, h);
    const int n = key_count(p, b);
    if (f.by_count && (n <= FEW_KEYS) != FINE) return;              // (the whole workgroup)
    const int32_t* idx = p.idx == nullptr ? nullptr : p.idx + (int64_t)b * p.Lk;
    const int hdb = p.hd * (int)sizeof(T);
    const unsigned char* kbase = (const unsigned char*)row_ptr<T>(p.k, p.sk, b, 0, hk);
    const unsigned char* vbase = (const unsigned char*)row_ptr<T>(p.v, p.sv, b, 0, hk);
    const int64_t kl = p.sk.l * (int)sizeof(T), vl = p.sv.l * (int)sizeof(T);
    // rows of a tile's fills: looked up a tile ahead, as in the forward pass
    using FL = typename TL::template Fill<KT, 4>;
    int rows[FL::FILLS];
    auto look_up = [&](int t) {
#pragma unroll
        for (int i = 0; i < FL::FILLS; ++i) rows[i] = max(min(t * KT + FL::row_of_fill(i, wave, lane), n - 1), 0);
        if (idx != nullptr && n > 0) {
#pragma unroll
            for (int i = 0; i < FL::FILLS; ++i) rows[i] = idx[rows[i]];
        }
    };
    auto issue = [&](int t, lds_t dst) {
        FL::run(dst, wave, lane, hdb, [&](int i) { return kbase + rows[i] * kl; });
        FL::run(dst + TB, wave, lane, hdb, [&](int i) { return vbase + rows[i] * vl; });
        look_up(t + 1);
    };
    int t0, t1;
    split_range((n + KT - 1) / KT, split, f.nsq, t0, t1);
    look_up(t0);
    const lds_t b0 = (lds_t)buf0[0], b1 = (lds_t)buf1[0];
    if (t0 < t1) issue(t0, b0);

    frag_t<T> qf[KS], dof[KS];
    const T* qrow = row_ok ? row_ptr<T>(p.q, p.sq, b, l, h) : nullptr;
    const T* dorow = row_ok ? row_ptr<T>(p.dout, p.sdo, b, l, h) : nullptr;
    const T* orow = row_ok ? row_ptr<T>(p.out, p.so, b, l, h) : nullptr;
    const float c2 = p.scale * LOG2E;
    float D = 0.f, off = INFINITY, fac = 0.f;
    if (row_ok) {
        const float* st = p.stat + (((int64_t)b * p.H + h) * p.Lq + l) * 2;
        const float m = st[0], sum = st[1];
        if (sum != 0.f) {
            off = BIAS ? m : fmaf(m, LOG2E, __builtin_amdgcn_logf(sum));
            fac = 1.0f / sum;
        }
    }
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = load_frag<T>(qrow, ks, hh, p.hd);
        dof[ks] = load_frag<T>(dorow, ks, hh, p.hd);
        const frag_t<T> of = load_frag<T>(orow, ks, hh, p.hd);
#pragma unroll
        for (int e = 0; e < 8; ++e) D = fmaf((float)dof[ks][e], (float)of[e], D);
    }
    D = halves_sum(D);
    const float* brow = BIAS && row_ok ? p.bias + h * p.bias_h + l * p.bias_l : nullptr;

    constexpr bool MEND = sizeof(T) == 2;                           // D from a rounded O
    f32x16 dq[DM], pk[MEND ? DM : 1];
    float e = 0.f;
#pragma unroll
    for (int m = 0; m < DM; ++m) dq[m] = zero16();
#pragma unroll
    for (int m = 0; m < (MEND ? DM : 1); ++m) pk[m] = zero16();
    auto tile_of = [&](auto whole_tag, int t, lds_t kt, lds_t vt, auto next) {
        constexpr bool WHOLE = decltype(whole_tag)::value;
        float bias[BIAS ? KB : 1][16];
        if constexpr (BIAS) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) load_bias<WHOLE>(bias[kb], brow, idx, t * KT + 32 * kb, n, hh);
        }
        next();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = mma(TL::rows(kt, 32 * kb, ks, lane), qf[ks], s);
                dp = mma(TL::rows(vt, 32 * kb, ks, lane), dof[ks], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if constexpr (BIAS) s[i] = fmaf(s[i], p.scale, bias[kb][i]);
                float pr = prob<BIAS>(s[i], c2, off, fac);
                if (!WHOLE && t * KT + 32 * kb + acc_row(i, hh) >= n) pr = 0.f;
                s[i] = pr;
                dp[i] = pr * (dp[i] - D);
                if constexpr (MEND) e += dp[i];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // (dS of bf16 heads is rounded to bf16 for the matrix instruction, as P is in the forward pass)
                const frag_t<T> df = pack_step<T>(dp, u);
                frag_t<T> pf = df, rest = df;
                if constexpr (MEND) pf = pack_step<T>(s, u);
                if constexpr (FINE) {
#pragma unroll
                    for (int x = 0; x < 8; ++x) rest[x] = (T)(dp[8 * u + x] - (float)df[x]);
                }
#pragma unroll
                for (int m = 0; m < DM; ++m) {
                    const frag_t<T> kc = TL::cols(kt, 32 * kb + 16 * u, m, lane);
                    dq[m] = mma(kc, df, dq[m]);
                    if constexpr (FINE) dq[m] = mma(kc, rest, dq[m]);
                    if constexpr (MEND) pk[m] = mma(kc, pf, pk[m]);
                }
            }
            if constexpr (HDP > 64) __builtin_amdgcn_sched_barrier(0);  // (two blocks in flight would not fit the registers)
        }
    };
    // (whole tiles in the loop, the ragged one behind it: as in the forward pass)
    const int tw = min(t1, n / KT);
    int t = t0;
    bool odd = false;
    while (t < tw) {
        tile_barrier();
        tile_of(std::true_type{}, t, b0, b0 + TB, [&] { if (t + 1 < t1) issue(t + 1, b1); });
        odd = true;
        if (++t >= tw) break;
        tile_barrier();
        tile_of(std::true_type{}, t, b1, b1 + TB, [&] { if (t + 1 < t1) issue(t + 1, b0); });
        odd = false;
        ++t;
    }
    if (t < t1) {
        tile_barrier();
        const lds_t at = odd ? b1 : b0;
        tile_of(std::false_type{}, t, at, at + TB, [] {});
    }
    if constexpr (MEND) e = halves_sum(e);
    if (split == 0 && hh == 0) {
        // (split: the launch that joins the sums adds the others' share to D; rows behind the last one have no share in anything)
        float* rs = f.rows + ((int64_t)bh * f.nrb * 4 + rb * 4 + wave) * RSB + lane;
        rs[0] = off;
        rs[32] = fac;
        rs[64] = f.nsq > 1 ? D : D + e;
    }
    if (!row_ok) return;
    const bool one = n <= 1;
    if (f.nsq > 1) {
        const int64_t row = ((int64_t)split * p.B * p.Hkv + bh) * p.R + r;
        float* po = f.part_q + row * HDP * (MEND ? 2 : 1);
#pragma unroll
        for (int m = 0; m < DM; ++m)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int d = 32 * m + 8 * a + 4 * hh;
                *(f32x4*)(po + d) = (f32x4){one ? 0.f : dq[m][4 * a], one ? 0.f : dq[m][4 * a + 1], one ? 0.f : dq[m][4 * a + 2], one ? 0.f : dq[m][4 * a + 3]};
                if constexpr (MEND) *(f32x4*)(po + HDP + d) = (f32x4){pk[m][4 * a], pk[m][4 * a + 1], pk[m][4 * a + 2], pk[m][4 * a + 3]};
            }
        if (MEND && hh == 0) f.part_e[row] = one ? 0.f : e;
        return;
    }
    T* out = (T*)f.dq + b * f.sdq.b + l * f.sdq.l + h * f.sdq.h;
#pragma unroll
    for (int m = 0; m < DM; ++m)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int d = 32 * m + 8 * a + 4 * hh;
            float v[4];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                v[c] = dq[m][4 * a + c];
                if constexpr (MEND) v[c] = fmaf(-e, pk[m][4 * a + c], v[c]);
                v[c] = one ? 0.f : v[c] * p.scale;
            }
            if (d < p.hd) store4(out + d, v[0], v[1], v[2], v[3]);
        }
}

template <typename T, int HDP> struct KeyCfg {
    static constexpr int QT = HDP <= 64 ? 64 : 32;                  // query rows a tile
    static constexpr int TB = QT * Tile<T, HDP>::ROWB, RB = QT / 32 * RSB * 4;
};

template <typename T, int HD, bool BIAS>
__global__ __launch_bounds__(256, (kv_waves<T, padded(HD)>())) void cross_bwd_kv_kernel(const Bwd f) {
    constexpr int HDP = padded(HD);
    using TL = Tile<T, HDP>;
    using Cfg = KeyCfg<T, HDP>;
    constexpr int QT = Cfg::QT, TB = Cfg::TB, KS = HD / 16, DM = HDP / 32;
    __shared__ __attribute__((aligned(16))) unsigned char buf0[2 * TB + Cfg::RB];
    __shared__ __attribute__((aligned(16))) unsigned char buf1[2 * TB + Cfg::RB];
    const Prob& p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    int bh, blk;
    place_block(blockIdx.x, p.B * p.Hkv, f.nkb * f.nsk, bh, blk);
    const int kblk = blk % f.nkb, split = blk / f.nkb;
    const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
    const int n = key_count(p, b);
    const int32_t* idx = p.idx == nullptr ? nullptr : p.idx + (int64_t)b * p.Lk;
    const int pos = kblk * 128 + wave * 32 + (lane & 31);
    const bool exists = pos < p.Lk, attended = pos < n;
    const int key = exists ? key_row(idx, pos) : 0;                 // (the list has all Lk keys, those not attended at its end)
    const int hdb = p.hd * (int)sizeof(T);

    f32x16 dk[DM], dv[DM];
#pragma unroll
    for (int m = 0; m < DM; ++m) { dk[m] = zero16(); dv[m] = zero16(); }

    if (kblk * 128 < n) {
        frag_t<T> kf[KS], vf[KS];
        const T* krow = attended ? row_ptr<T>(p.k, p.sk, b, key, hk) : nullptr;
        const T* vrow = attended ? row_ptr<T>(p.v, p.sv, b, key, hk) : nullptr;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { kf[ks] = load_frag<T>(krow, ks, hh, p.hd); vf[ks] = load_frag<T>(vrow, ks, hh, p.hd); }
        int t0, t1;
        split_range((p.R + QT - 1) / QT, split, f.nsk, t0, t1);
        const float* rows = f.rows + (int64_t)bh * f.nrb * 4 * RSB;
        const unsigned char* qbase = (const unsigned char*)row_ptr<T>(p.q, p.sq, b, 0, 0);
        const unsigned char* dobase = (const unsigned char*)row_ptr<T>(p.dout, p.sdo, b, 0, 0);
        using FL = typename TL::template Fill<QT, 4>;
        // (rows behind the last one: that one again - their P is 0)
        auto issue = [&](int t, lds_t dst) {
            int64_t oq[FL::FILLS], od[FL::FILLS];
#pragma unroll
            for (int i = 0; i < FL::FILLS; ++i) {
                int l, h;
                row_of(p, hk, min(t * QT + FL::row_of_fill(i, wave, lane), p.R - 1), l, h);
                oq[i] = (l * p.sq.l + h * p.sq.h) * (int)sizeof(T);
                od[i] = (l * p.sdo.l + h * p.sdo.h) * (int)sizeof(T);
            }
            FL::run(dst, wave, lane, hdb, [&](int i) { return qbase + oq[i]; });
            FL::run(dst + TB, wave, lane, hdb, [&](int i) { return dobase + od[i]; });
            // the row values: 512 bytes a block of 32 rows (they exist up to the next multiple of 128 rows)
            if (wave == 0 && lane < QT)
                __builtin_amdgcn_global_load_lds((gbl_ptr_t)(rows + (int64_t)t * (QT / 32) * RSB + 4 * lane), (lds_ptr_t)(dst + 2 * TB), 16, 0, 0);
        };
        const float c2 = p.scale * LOG2E;
        const unsigned blane = BIAS ? (unsigned)(4 * hh * p.bias_l) + key : 0;      // (a lane whose key is not attended reads its bias too: its column is not used)
        auto tile = [&](int t, lds_t base, auto next) {
            const lds_t qt = base, dot = base + TB;
#pragma unroll
            for (int qb = 0; qb < QT / 32; ++qb) {
                const lds_f32_t rs = (lds_f32_t)(base + 2 * TB) + qb * RSB;
                float bias[16];
                if constexpr (BIAS) {
                    const int r0 = t * QT + 32 * qb;
                    int l0, h0;
                    row_of(p, hk, min(r0, p.R - 1), l0, h0);
                    if (l0 + 32 <= p.Lq) {                          // 32 rows of one head: whole-wave row addresses, the lanes' part in 32 bits
                        const float* base = p.bias + h0 * p.bias_h + l0 * p.bias_l;
#pragma unroll
                        for (int i = 0; i < 16; ++i) bias[i] = (base + (8 * (i >> 2) + (i & 3)) * p.bias_l)[blane];
                    } else {
#pragma unroll
                        for (int i = 0; i < 16; ++i) {
                            const int r = r0 + acc_row(i, hh);
                            int l, h;
                            row_of(p, hk, min(r, p.R - 1), l, h);
                            bias[i] = r < p.R ? p.bias[h * p.bias_h + l * p.bias_l + key] : 0.f;
                        }
                    }
                }
                if (qb == 0) next();
                f32x16 s = zero16(), dp = zero16();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    s = mma(TL::rows(qt, 32 * qb, ks, lane), kf[ks], s);
                    dp = mma(TL::rows(dot, 32 * qb, ks, lane), vf[ks], dp);
                }
#pragma unroll
                for (int a = 0; a < 4; ++a) {
                    const f32x4 off = *(lds_f32x4_t)(rs + 8 * a + 4 * hh), D = *(lds_f32x4_t)(rs + 64 + 8 * a + 4 * hh);
                    f32x4 fac = {1.f, 1.f, 1.f, 1.f};
                    if constexpr (BIAS) fac = *(lds_f32x4_t)(rs + 32 + 8 * a + 4 * hh);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int i = 4 * a + e;
                        if constexpr (BIAS) s[i] = fmaf(s[i], p.scale, bias[i]);
                        const float pr = prob<BIAS>(s[i], c2, off[e], fac[e]);
                        s[i] = pr;
                        dp[i] = pr * (dp[i] - D[e]);
                    }
                }
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const frag_t<T> pf = pack_step<T>(s, u), df = pack_step<T>(dp, u);
#pragma unroll
                    for (int m = 0; m < DM; ++m) {
                        dv[m] = mma(TL::cols(dot, 32 * qb + 16 * u, m, lane), pf, dv[m]);
                        dk[m] = mma(TL::cols(qt, 32 * qb + 16 * u, m, lane), df, dk[m]);
                    }
                }
            }
        };
        const lds_t b0 = (lds_t)buf0, b1 = (lds_t)buf1;
        if (t0 < t1) issue(t0, b0);
        for (int t = t0; t < t1; t += 2) {
            tile_barrier();
            tile(t, b0, [&] { if (t + 1 < t1) issue(t + 1, b1); });
            if (t + 1 < t1) {
                tile_barrier();
                tile(t + 1, b1, [&] { if (t + 2 < t1) issue(t + 2, b0); });
            }
        }
    }
    if (!exists) return;
    if (n <= 1) {
#pragma unroll
        for (int m = 0; m < DM; ++m) dk[m] = zero16();
    }
    if (f.nsk > 1) {
        const int64_t o = (((int64_t)split * p.B * p.Hkv + bh) * p.Lk + pos) * HDP;
#pragma unroll
        for (int m = 0; m < DM; ++m)
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const int d = 32 * m + 8 * a + 4 * hh;
                *(f32x4*)(f.part_k + o + d) = (f32x4){dk[m][4 * a], dk[m][4 * a + 1], dk[m][4 * a + 2], dk[m][4 * a + 3]};
                *(f32x4*)(f.part_v + o + d) = (f32x4){dv[m][4 * a], dv[m][4 * a + 1], dv[m][4 * a + 2], dv[m][4 * a + 3]};
            }
        return;
    }
    // (a key that is not attended still has its zeros)
    T* ok = (T*)f.dk + b * f.sdk.b + key * f.sdk.l + hk * f.sdk.h;
    T* ov = (T*)f.dv + b * f.sdv.b + key * f.sdv.l + hk * f.sdv.h;
#pragma unroll
    for (int m = 0; m < DM; ++m)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int d = 32 * m + 8 * a + 4 * hh;
            if (d < p.hd) {
                if (attended) {
                    store4(ok + d, dk[m][4 * a] * p.scale, dk[m][4 * a + 1] * p.scale, dk[m][4 * a + 2] * p.scale, dk[m][4 * a + 3] * p.scale);
                    store4(ov + d, dv[m][4 * a], dv[m][4 * a + 1], dv[m][4 * a + 2], dv[m][4 * a + 3]);
                } else {
                    store4(ok + d, 0.f, 0.f, 0.f, 0.f);
                    store4(ov + d, 0.f, 0.f, 0.f, 0.f);
                }
            }
        }
}

// sums of the splits.  KEYS: rows of dk (y 0) and dv (y 1); otherwise rows of dq
template <typename T, int HDP, bool KEYS>
__global__ __launch_bounds__(256) void cross_bwd_sum_kernel(const Bwd f) {
    constexpr int LR = HDP / 4;
    const Prob& p = f.p;
    const int per = KEYS ? p.Lk : p.R, ns = KEYS ? f.nsk : f.nsq;
    const int64_t rows = (int64_t)p.B * p.Hkv * per;
    const int64_t g = (int64_t)blockIdx.x * (256 / LR) + threadIdx.x / LR;
    const int d = 4 * (threadIdx.x % LR);
    if (threadIdx.x >= 256 / LR * LR || g >= rows || d >= p.hd) return;
    const int bh = (int)(g / per), r = (int)(g - (int64_t)bh * per), b = bh / p.Hkv, hk = bh - b * p.Hkv;
    const bool second = KEYS && blockIdx.y == 1;
    const float* part = KEYS ? (second ? f.part_v : f.part_k) : f.part_q;
    float a0 = 0.f, a1 = 0.f, a2 = 0.f, a3 = 0.f;
    if constexpr (!KEYS && sizeof(T) == 2) {
        float e = 0.f, k0 = 0.f, k1 = 0.f, k2 = 0.f, k3 = 0.f;
        for (int s = 0; s < ns; ++s) {
            const float* po = part + (s * rows + g) * 2 * HDP + d;
            const f32x4 v = *(const f32x4*)po, k = *(const f32x4*)(po + HDP);
            a0 += v[0]; a1 += v[1]; a2 += v[2]; a3 += v[3];
            k0 += k[0]; k1 += k[1]; k2 += k[2]; k3 += k[3];
            e += f.part_e[s * rows + g];
        }
        a0 = fmaf(-e, k0, a0) * p.scale;
        a1 = fmaf(-e, k1, a1) * p.scale;
        a2 = fmaf(-e, k2, a2) * p.scale;
        a3 = fmaf(-e, k3, a3) * p.scale;
        if (d == 0) f.rows[((int64_t)bh * f.nrb * 4 + (r >> 5)) * RSB + 64 + (r & 31)] += e;
    } else if (!KEYS || r < key_count(p, b)) {
        for (int s = 0; s < ns; ++s) {
            const f32x4 v = *(const f32x4*)(part + (s * rows + g) * HDP + d);
            a0 += v[0]; a1 += v[1]; a2 += v[2]; a3 += v[3];
        }
        if (!second) { a0 *= p.scale; a1 *= p.scale; a2 *= p.scale; a3 *= p.scale; }
    }
    T* o;
    if constexpr (KEYS) {
        const int key = key_row(p.idx == nullptr ? nullptr : p.idx + (int64_t)b * p.Lk, r);
        const Strides& s = second ? f.sdv : f.sdk;
        o = (T*)(second ? f.dv : f.dk) + b * s.b + key * s.l + hk * s.h;
    } else {
        int l, h;
        row_of(p, hk, r, l, h);
        o = (T*)f.dq + b * f.sdq.b + l * f.sdq.l + h * f.sdq.h;
    }
    store4(o + d, a0, a1, a2, a3);
}

// dbias[h, i, j] = sum_b dS: grid (key tiles of 64, query blocks of 128, heads); keys are taken where they stand (the lists of attended keys
// differ from entry to entry), with the key as lane column so that rows of bias and dbias are read and written in whole lines.  While one
// batch entry is worked on, the next one's K and V tiles, query rows and row values are on their way.
// (A masked key below kv_len is loaded with the others of its tile.  Keys are lane columns: what it holds stays in its own, which is not used.)
template <typename T, int HD>
__global__ __launch_bounds__(256, (HD <= 64 && sizeof(T) == 2) ? 2 : 1) void cross_bwd_bias_kernel(const Bwd f) {
    constexpr int HDP = padded(HD);
    using TL = Tile<T, HDP>;
    constexpr int KT = 64, TB = KT * TL::ROWB, KS = HD / 16;
    __shared__ __attribute__((aligned(16))) unsigned char buf0[2][TB];
    __shared__ __attribute__((aligned(16))) unsigned char buf1[2][TB];
    __shared__ __attribute__((aligned(16))) float rowv[4][3][32];
    const Prob& p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int j0 = blockIdx.x * KT, h = blockIdx.z, hk = h / p.grp, r0 = (h - hk * p.grp) * p.Lq;
    const int i0 = blockIdx.y * 128 + wave * 32;                    // this wave's query tokens
    const int hdb = p.hd * (int)sizeof(T);
    const int l = min(i0 + (lane & 31), p.Lq - 1), r = r0 + l;
    f32x16 acc[2] = {zero16(), zero16()};
    float bias[2][16];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int li = min(i0 + acc_row(i, hh), p.Lq - 1), j = min(j0 + 32 * kb + (lane & 31), p.Lk - 1);
            bias[kb][i] = p.bias[h * p.bias_h + li * p.bias_l + j];
        }
    auto length = [&](int b) { return f.kv_len == nullptr ? p.Lk : min(max(f.kv_len[b], 0), p.Lk); };
    // the next batch entry from b with keys in this tile, and more than one in all (the same for the whole workgroup)
    auto entry = [&](int b) {
        while (b < p.B && (j0 >= length(b) || key_count(p, b) <= 1)) ++b;
        return b;
    };
    frag_t<T> qf[KS], dof[KS];
    float off = 0.f, fac = 0.f, D = 0.f;
    bool on[2];
    auto fetch = [&](int b, lds_t dst) {
        const int len = length(b);
        const T* qrow = row_ptr<T>(p.q, p.sq, b, l, h);
        const T* dorow = row_ptr<T>(p.dout, p.sdo, b, l, h);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { qf[ks] = load_frag<T>(qrow, ks, hh, p.hd); dof[ks] = load_frag<T>(dorow, ks, hh, p.hd); }
        const float* rs = f.rows + (((int64_t)b * p.Hkv + hk) * f.nrb * 4 + (r >> 5)) * RSB + (r & 31);
        off = rs[0];
        fac = rs[32];
        D = rs[64];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            const int j = j0 + 32 * kb + (lane & 31);
            on[kb] = j < len && (f.mask == nullptr || f.mask[(int64_t)b * p.Lk + j] != 0);
        }
        const unsigned char* kbase = (const unsigned char*)row_ptr<T>(p.k, p.sk, b, 0, hk);
        const unsigned char* vbase = (const unsigned char*)row_ptr<T>(p.v, p.sv, b, 0, hk);
        using FL = typename TL::template Fill<KT, 4>;
        FL::run(dst, wave, lane, hdb, [&](int i) { return kbase + min(j0 + FL::row_of_fill(i, wave, lane), len - 1) * p.sk.l * (int)sizeof(T); });
        FL::run(dst + TB, wave, lane, hdb, [&](int i) { return vbase + min(j0 + FL::row_of_fill(i, wave, lane), len - 1) * p.sv.l * (int)sizeof(T); });
    };
    // one entry: its tiles are in cur; returns the entry whose fetch into the other buffer it started
    auto work = [&](int b, lds_t cur, lds_t other) {
        rowv[wave][0][lane & 31] = off;                             // (both half-waves hold the same rows)
        rowv[wave][1][lane & 31] = fac;
        rowv[wave][2][lane & 31] = D;
        frag_t<T> q[KS], d[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) { q[ks] = qf[ks]; d[ks] = dof[ks]; }
        const bool on0 = on[0], on1 = on[1];
        tile_barrier();
        const int nb = entry(b + 1);
        if (nb < p.B) fetch(nb, other);
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            f32x16 s = zero16(), dp = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                s = mma(q[ks], TL::rows(cur, 32 * kb, ks, lane), s);
                dp = mma(d[ks], TL::rows(cur + TB, 32 * kb, ks, lane), dp);
            }
#pragma unroll
            for (int a = 0; a < 4; ++a) {
                const f32x4 o4 = *(const f32x4*)&rowv[wave][0][8 * a + 4 * hh], f4 = *(const f32x4*)&rowv[wave][1][8 * a + 4 * hh],
                            d4 = *(const f32x4*)&rowv[wave][2][8 * a + 4 * hh];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int i = 4 * a + e;
                    // (a row that is not attended may hold anything: its values stay in this lane's column and are not used)
                    const float ds = prob<true>(fmaf(s[i], p.scale, bias[kb][i]), 0.f, o4[e], f4[e]) * (dp[i] - d4[e]);
                    acc[kb][i] += (kb == 0 ? on0 : on1) ? ds : 0.f;
                }
            }
        }
        return nb;
    };
    const lds_t b0 = (lds_t)buf0[0], b1 = (lds_t)buf1[0];
    int b = entry(0);
    if (b < p.B) fetch(b, b0);
    while (b < p.B) {
        b = work(b, b0, b1);
        if (b < p.B) b = work(b, b1, b0);
    }
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int li = i0 + acc_row(i, hh), j = j0 + 32 * kb + (lane & 31);
            if (li < p.Lq && j < p.Lk) f.dbias[h * f.dbias_h + li * f.dbias_l + j] = acc[kb][i];
        }
}

struct BwdPlan { int hd, hdp, nrb, nsq, nkb, nsk; int64_t rows_bytes, q_bytes, e_bytes, k_bytes; };
int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

int splits(int64_t blocks, int64_t most) {
    if (blocks >= 256) return 1;
    int64_t ns = (512 + blocks - 1) / blocks;
    if (ns > most) ns = most;
    return ns < 1 ? 1 : (int)ns;
}

BwdPlan plan_bwd(const MarsCrossAttn* a) {
    BwdPlan pl;
    const int64_t R = (int64_t)(a->H / a->Hkv) * a->Lq, nbh = (int64_t)a->B * a->Hkv;
    pl.hd = built_for(a->hd);
    pl.hdp = padded(pl.hd);
    pl.nrb = (int)((R + 127) / 128);
    pl.nkb = (a->Lk + 127) / 128;
    pl.nsq = splits(nbh * pl.nrb, ((int64_t)a->Lk + 127) / 128);
    pl.nsk = splits(nbh * pl.nkb, (R + 127) / 128);
    pl.rows_bytes = align256(nbh * pl.nrb * 4 * RSB * 4);
    pl.q_bytes = pl.nsq > 1 ? align256((int64_t)pl.nsq * nbh * R * pl.hdp * 4 * (a->dtype == 1 ? 2 : 1)) : 0;
    pl.e_bytes = pl.nsq > 1 && a->dtype == 1 ? align256((int64_t)pl.nsq * nbh * R * 4) : 0;
    pl.k_bytes = pl.nsk > 1 ? align256((int64_t)pl.nsk * nbh * a->Lk * pl.hdp * 4) : 0;
    return pl;
}

template <typename T, int HD> int launch_bwd(const Bwd& f, hipStream_t s) {
    constexpr int HDP = padded(HD);
    const Prob& p = f.p;
    const int64_t nbh = (int64_t)p.B * p.Hkv, qb = nbh * f.nrb * f.nsq, kb = nbh * f.nkb * f.nsk, per = 256 / (HDP / 4);
    const dim3 block(256);
    constexpr bool F = sizeof(T) == 2;
    const bool few = F && p.Lk <= FEW_KEYS, both = F && !few && p.cnt != nullptr;
    Bwd fq = f;
    fq.by_count = both;
    if (few || both) {
        if (p.bias != nullptr) hipLaunchKernelGGL((cross_bwd_q_kernel<T, HD, true, F>), dim3((unsigned)qb), block, 0, s, fq);
        else hipLaunchKernelGGL((cross_bwd_q_kernel<T, HD, false, F>), dim3((unsigned)qb), block, 0, s, fq);
        MARS_LAUNCH_CHECK();
    }
    if (!few) {
        if (p.bias != nullptr) hipLaunchKernelGGL((cross_bwd_q_kernel<T, HD, true, false>), dim3((unsigned)qb), block, 0, s, fq);
        else hipLaunchKernelGGL((cross_bwd_q_kernel<T, HD, false, false>), dim3((unsigned)qb), block, 0, s, fq);
        MARS_LAUNCH_CHECK();
    }
    if (f.nsq > 1) {
        hipLaunchKernelGGL((cross_bwd_sum_kernel<T, HDP, false>), dim3((unsigned)((nbh * p.R + per - 1) / per)), block, 0, s, f);
        MARS_LAUNCH_CHECK();
    }
    if (p.bias != nullptr) hipLaunchKernelGGL((cross_bwd_kv_kernel<T, HD, true>), dim3((unsigned)kb), block, 0, s, f);
    else hipLaunchKernelGGL((cross_bwd_kv_kernel<T, HD, false>), dim3((unsigned)kb), block, 0, s, f);
    MARS_LAUNCH_CHECK();
    if (f.nsk > 1) {
        hipLaunchKernelGGL((cross_bwd_sum_kernel<T, HDP, true>), dim3((unsigned)((nbh * p.Lk + per - 1) / per), 2), block, 0, s, f);
        MARS_LAUNCH_CHECK();
    }
    if (f.dbias != nullptr) {
        const unsigned gy = (unsigned)((p.Lq + 127) / 128);
        hipLaunchKernelGGL((cross_bwd_bias_kernel<T, HD>), dim3((unsigned)((p.Lk + 63) / 64), gy, (unsigned)p.H), block, 0, s, f);
        MARS_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T> int launch_bwd_hd(const Bwd& f, int hd, hipStream_t s) {
    switch (hd) {
        case 16: return launch_bwd<T, 16>(f, s);
        case 32: return launch_bwd<T, 32>(f, s);
        case 64: return launch_bwd<T, 64>(f, s);
        case 80: return launch_bwd<T, 80>(f, s);
        case 96: return launch_bwd<T, 96>(f, s);
        default: return launch_bwd<T, 128>(f, s);
    }
}

}  // namespace

int64_t bwd_ws_bytes(const MarsCrossAttn* a) {
    const BwdPlan pl = plan_bwd(a);
    return pl.rows_bytes + pl.q_bytes + pl.e_bytes + 2 * pl.k_bytes;
}

}  // namespace xattn

extern "C" int marship_cross_attn_bwd(const MarsCrossAttn* a, void* stream) {
    using namespace xattn;
    if (const int rc = check(a, true)) return rc;
    const int64_t need = marship_cross_attn_ws(a, 1);
    MARS_CHECK(a->ws != nullptr && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= need, "cross_attn_bwd: workspace of %lld bytes, %lld needed",
               (long long)a->ws_bytes, (long long)need);
    hipStream_t s = (hipStream_t)stream;
    Bwd f{};
    describe(a, f.p);
    if (const int rc = prepare_keys(a, f.p, (int32_t*)a->ws, s)) return rc;
    const BwdPlan pl = plan_bwd(a);
    char* w = (char*)a->ws + key_ws_bytes(a);
    f.rows = (float*)w;
    f.part_q = (float*)(w + pl.rows_bytes);
    f.part_e = (float*)(w + pl.rows_bytes + pl.q_bytes);
    f.part_k = (float*)(w + pl.rows_bytes + pl.q_bytes + pl.e_bytes);
    f.part_v = (float*)(w + pl.rows_bytes + pl.q_bytes + pl.e_bytes + pl.k_bytes);
    f.dq = a->dq; f.dk = a->dk; f.dv = a->dv;
    f.sdq = Strides{a->dq_s[0], a->dq_s[1], a->dq_s[2]};
    f.sdk = Strides{a->dk_s[0], a->dk_s[1], a->dk_s[2]};
    f.sdv = Strides{a->dv_s[0], a->dv_s[1], a->dv_s[2]};
    f.dbias = a->dbias; f.dbias_h = a->dbias_s[0]; f.dbias_l = a->dbias_s[1];
    f.mask = a->mask;
    f.kv_len = a->kv_len;
    f.nrb = pl.nrb; f.nsq = pl.nsq; f.nkb = pl.nkb; f.nsk = pl.nsk;
    return a->dtype == 1 ? launch_bwd_hd<__bf16>(f, pl.hd, s) : launch_bwd_hd<float>(f, pl.hd, s);
}

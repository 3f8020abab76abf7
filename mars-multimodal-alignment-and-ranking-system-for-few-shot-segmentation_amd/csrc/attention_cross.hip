// Attention of one set of tokens over another of another length (query patches over support patches; prompt tokens over
// an image; a new token over an encoder's states), forward:
//
//   s_ij = scale q_i . k_j + bias[h, i, j] over the attended keys,   o_i = sum_j softmax_j(s_ij) v_j
//
// One pass over the keys with a running maximum and sum.  A wave owns 32 query rows and computes S^T = K Q^T on the
// 32x32 matrix instructions, so that a query is a lane column: row statistics are per-lane values that meet in one
// half-wave swap, and the exponentials are, as they stand, the operand of O^T += V^T P^T.
//
// Masked keys are not computed and then thrown away: where the caller gives a mask, a first launch lists the attended keys of each
// batch entry, and the fills gather K and V rows through that list.  A support image's foreground is a tenth to
// a half of its patches, a row costs the same gathered or not (it is at least one 32-byte sector, mostly one or two cache lines),
// and whatever stands in a masked row - infinities, NaN - is never read.
//
// Few rows (one new token a sequence) are bound by memory: the four waves of a workgroup take key tiles in turn through buffers of their own, the keys
// are cut over the chip and joined (16 sequences over up to 8192 keys, 16 / 4 heads of 128: 40 us for 206 MB).  Many rows are bound by
// vector ALU and matrix pipe one after the other: a wave's 64 scores cost 16 cycles of exponential and 14 of other vector work, and 16 (64-wide heads) in the
// two products; 1369 over 6845, 32 heads of 64: 115 us with the join of two cuts, 668 TFLOP/s.
#include <type_traits>
#include "attention_cross.h"

namespace xattn {
namespace {

// ------------------------------------------------------------------------------------------------ lists of attended keys
// idx[b] = attended keys in order, then the others in order; cnt[b] = how many.  A workgroup of 1024 per batch entry: ballots
// within a wave, a scan over its sixteen waves, 1024 keys a step.
__global__ __launch_bounds__(1024) void list_keys_kernel(const uint8_t* __restrict__ mask, const int32_t* __restrict__ kv_len, int Lk,
                                                         int32_t* __restrict__ idx, int32_t* __restrict__ cnt) {
    __shared__ int wsum[16];
    const int b = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const uint8_t* m = mask + (int64_t)b * Lk;
    const int len = kv_len == nullptr ? Lk : min(max(kv_len[b], 0), Lk);
    int32_t* out = idx + (int64_t)b * Lk;
    auto scan = [&](int total0, auto emit) {
        int total = total0;
        for (int j0 = 0; j0 < Lk; j0 += 1024) {
            const int j = j0 + tid;
            const bool on = j < len && m[j] != 0;
            const unsigned long long bal = __ballot(on);
            const int before = __popcll(bal & ((1ull << lane) - 1));
            __syncthreads();
            if (lane == 0) wsum[wave] = __popcll(bal);
            __syncthreads();
            int base = total;
            for (int w = 0; w < wave; ++w) base += wsum[w];
            for (int w = 0; w < 16; ++w) total += wsum[w];
            if (j < Lk) emit(j, on, base + before);
        }
        return total;
    };
    const int n = scan(0, [&](int j, bool on, int pos) { if (on) out[pos] = j; });
    // an unattended key stands behind the n attended ones, after the unattended keys before it
    scan(0, [&](int j, bool on, int pos) { if (!on) out[n + j - pos] = j; });
    if (tid == 0) cnt[b] = n;
}

// ------------------------------------------------------------------------------------------------ forward
struct Fwd {
    Prob p;
    void* out;                      // [B, Lq, H, hd] by p.so, or nullptr where there are partial results to join
    float* stat;                    // [B, H, Lq, 2]: row maximum and sum of exp(s - maximum); may be nullptr
    float *part_o, *part_s;         // partial results: [ns][B Hkv][R][HDP] un-normalised, [ns][B Hkv][R][2]
    int nrb, ns;                    // row blocks, splits of the keys
};

// FEW: at most 32 rows: the four waves share them and take key tiles in turn, each through LDS buffers of its own (no barrier),
// and join their results at the end.  Otherwise each wave has 32 rows of a 128-row block and the workgroup shares the tiles.
template <typename T, int HD, bool FEW> struct FwdCfg {
    static constexpr int HDP = padded(HD);
    static constexpr int KT = FEW ? 32 : 64;                                             // keys per tile
    static constexpr int TB = KT * HDP * (int)sizeof(T);
    static constexpr int COPIES = FEW ? 4 : 1;
    static constexpr int BUFS = COPIES * 4 * TB <= 128 * 1024 ? 2 : 1;
    static constexpr int WPE = COPIES * BUFS * 2 * TB <= 80 * 1024 ? 2 : 1;              // waves a SIMD that the LDS leaves room for
};

template <typename T, int HD, bool BIAS, bool FEW>
__global__ __launch_bounds__(256, (FwdCfg<T, HD, FEW>::WPE)) void cross_fwd_kernel(const Fwd f) {
    using Cfg = FwdCfg<T, HD, FEW>;
    constexpr int HDP = Cfg::HDP;
    using TL = Tile<T, HDP>;
    constexpr int KT = Cfg::KT, TB = Cfg::TB, KB = KT / 32, KS = HD / 16, DM = HDP / 32;
    __shared__ __attribute__((aligned(16))) unsigned char buf0[Cfg::COPIES][2][TB];
    __shared__ __attribute__((aligned(16))) unsigned char buf1[Cfg::BUFS == 2 ? Cfg::COPIES : 1][Cfg::BUFS == 2 ? 2 : 1][Cfg::BUFS == 2 ? TB : 16];
    const Prob& p = f.p;
    const int tid = threadIdx.x, lane = tid & 63, hh = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int cw = FEW ? wave : 0;                              // which copy of the buffers
    int bh, blk;
    place_block(blockIdx.x, p.B * p.Hkv, f.nrb * f.ns, bh, blk);
    const int rb = blk % f.nrb, split = blk / f.nrb;
    const int b = bh / p.Hkv, hk = bh - b * p.Hkv;
    const int r = FEW ? rb * 32 + (lane & 31) : rb * 128 + wave * 32 + (lane & 31);
    const bool row_ok = r < p.R;
    int l = 0, h = 0;
    if (row_ok) row_of(p, hk, r, l, h);
    frag_t<T> qf[KS];
    const T* qrow = row_ok ? row_ptr<T>(p.q, p.sq, b, l, h) : nullptr;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = load_frag<T>(qrow, ks, hh, p.hd);
    const float* brow = BIAS && row_ok ? p.bias + h * p.bias_h + l * p.bias_l : nullptr;

    const int n = key_count(p, b);
    const int32_t* idx = p.idx == nullptr ? nullptr : p.idx + (int64_t)b * p.Lk;
    int t0, t1;
    split_range((n + KT - 1) / KT, split, f.ns, t0, t1);
    const int hdb = p.hd * (int)sizeof(T);
    const unsigned char* kbase = (const unsigned char*)row_ptr<T>(p.k, p.sk, b, 0, hk);
    const unsigned char* vbase = (const unsigned char*)row_ptr<T>(p.v, p.sv, b, 0, hk);
    const int64_t kl = p.sk.l * (int)sizeof(T), vl = p.sv.l * (int)sizeof(T);

    // The rows that this thread's fills of a tile take; with a list of attended keys they are looked up a tile ahead, so that no fill
    // waits for its index.  (Keys behind the last attended one: that one again - their scores are set to -inf and
    // their values to 0, so that an infinity among the last key's is not multiplied by a probability of 0.)
    constexpr int NW = FEW ? 1 : 4, STEP = FEW ? 4 : 1;
    using FL = typename TL::template Fill<KT, NW>;
    const int fw = FEW ? 0 : wave;
    int rows[FL::FILLS];
    auto look_up = [&](int t) {
#pragma unroll
        for (int i = 0; i < FL::FILLS; ++i) rows[i] = max(min(t * KT + FL::row_of_fill(i, fw, lane), n - 1), 0);
        if (idx != nullptr && n > 0) {
#pragma unroll
            for (int i = 0; i < FL::FILLS; ++i) rows[i] = idx[rows[i]];
        }
    };
    // fills of tile t, whose rows are looked up; then the rows of the next one
    auto issue = [&](int t, lds_t dst) {
        FL::run(dst, fw, lane, hdb, [&](int i) { return kbase + rows[i] * kl; });
        FL::run(dst + TB, fw, lane, hdb, [&](int i) { return vbase + rows[i] * vl; });
        look_up(t + STEP);
    };

    f32x16 o[DM];
#pragma unroll
    for (int m = 0; m < DM; ++m) o[m] = zero16();
    float mrun = -INFINITY, lsum = 0.f;
    const float c2 = p.scale * LOG2E;

    // one tile: scores, running maximum, exponentials, products with V.  Without a bias the maximum is of the raw products
    // (scale > 0) and scale and log2 e come with the exponent; with one the scores are kept in natural units, because
    // a mask made of the type's lowest value would overflow in units of log 2.
    // next(): the fills of a later tile, issued behind this tile's bias loads (loads come back in order: the other way round the first use of
    // the bias would wait for the fills)
    auto tile_of = [&](auto whole_tag, int t, lds_t kt, lds_t vt, auto next) {
        constexpr bool WHOLE = decltype(whole_tag)::value;
        f32x16 s[KB];
        float bias[BIAS ? KB : 1][16];
        if constexpr (BIAS) {
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) load_bias<WHOLE>(bias[kb], brow, idx, t * KT + 32 * kb, n, hh);
        }
        next();
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            s[kb] = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) s[kb] = mma(TL::rows(kt, 32 * kb, ks, lane), qf[ks], s[kb]);
            if constexpr (BIAS) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] = fmaf(s[kb][i], p.scale, bias[kb][i]);
            }
            if constexpr (!WHOLE) {
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (t * KT + 32 * kb + acc_row(i, hh) >= n) s[kb][i] = -INFINITY;
            }
        }
        float mx = s[0][0];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = vmax(mx, s[kb][i]);
        const float mnew = vmax(mrun, halves_max(mx));
        // (a bias of -inf on every key so far: nothing to scale, and the exponentials must come out as zeros)
        const float mref = BIAS && mnew == -INFINITY ? 0.f : mnew;
        const float unit = BIAS ? LOG2E : c2;
        const float alpha = __builtin_amdgcn_exp2f((mrun - mref) * unit);
        mrun = mnew;
        lsum *= alpha;
        const float sub = mref * unit;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(BIAS ? (s[kb][i] - mref) * unit : fmaf(s[kb][i], unit, -sub));
                lsum += s[kb][i];
            }
        if (!__all(alpha == 1.f)) {
#pragma unroll
            for (int m = 0; m < DM; ++m)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[m][i] *= alpha;
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                // probabilities of bf16 heads are rounded to bf16 for the matrix instruction (at most half a step, 2^-8 of each, with signs
                // that do not agree: below the rounding of the result); their sum is taken before the rounding
                const frag_t<T> pf = pack_step<T>(s[kb], u);
#pragma unroll
                for (int m = 0; m < DM; ++m) {
                    frag_t<T> vc = TL::cols(vt, 32 * kb + 16 * u, m, lane);
                    if constexpr (!WHOLE) {
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (t * KT + 32 * kb + 16 * u + 8 * (e >> 2) + 4 * hh + (e & 3) >= n) vc[e] = (T)0.f;
                    }
                    o[m] = mma(vc, pf, o[m]);
                }
            }
    };
    // whole tiles in the loops, the ragged one behind them: both forms inside one loop would make the compiler carry the accumulators
    // through the join in a second set of registers
    const int tw = min(t1, n / KT);
    constexpr std::true_type whole{};
    constexpr std::false_type ragged{};
    auto nothing = [] {};

    const lds_t my0 = (lds_t)buf0[cw][0], my1 = Cfg::BUFS == 2 ? (lds_t)buf1[Cfg::BUFS == 2 ? cw : 0][0] : my0;
    if constexpr (!FEW) {
        look_up(t0);
        if (t0 < t1) issue(t0, my0);
        int t = t0;
        if constexpr (Cfg::BUFS == 2) {
            bool odd = false;
            while (t < tw) {
                tile_barrier();
                tile_of(whole, t, my0, my0 + TB, [&] { if (t + 1 < t1) issue(t + 1, my1); });
                odd = true;
                if (++t >= tw) break;
                tile_barrier();
                tile_of(whole, t, my1, my1 + TB, [&] { if (t + 1 < t1) issue(t + 1, my0); });
                odd = false;
                ++t;
            }
            if (t < t1) {
                tile_barrier();
                const lds_t at = odd ? my1 : my0;
                tile_of(ragged, t, at, at + TB, nothing);
            }
        } else {
            for (; t < tw; ++t) {
                tile_barrier();
                tile_of(whole, t, my0, my0 + TB, nothing);
                tile_barrier();
                if (t + 1 < t1) issue(t + 1, my0);
            }
            if (t < t1) {
                tile_barrier();
                tile_of(ragged, t, my0, my0 + TB, nothing);
            }
        }
    } else {
        // a wave's own buffers need its own waits only
        int t = t0 + wave;
        look_up(t);
        if (t < t1) issue(t, my0);
        if constexpr (Cfg::BUFS == 2) {
            bool odd = false;
            while (t < tw) {
                __builtin_amdgcn_s_waitcnt(0);
                tile_of(whole, t, my0, my0 + TB, [&] { if (t + 4 < t1) issue(t + 4, my1); });
                odd = true;
                t += 4;
                if (t >= tw) break;
                __builtin_amdgcn_s_waitcnt(0);
                tile_of(whole, t, my1, my1 + TB, [&] { if (t + 4 < t1) issue(t + 4, my0); });
                odd = false;
                t += 4;
            }
            if (t < t1) {
                __builtin_amdgcn_s_waitcnt(0);
                const lds_t at = odd ? my1 : my0;
                tile_of(ragged, t, at, at + TB, nothing);
            }
        } else {
            for (; t < tw; t += 4) {
                __builtin_amdgcn_s_waitcnt(0);
                tile_of(whole, t, my0, my0 + TB, nothing);
                __builtin_amdgcn_s_waitcnt(0);
                if (t + 4 < t1) issue(t + 4, my0);
            }
            if (t < t1) {
                __builtin_amdgcn_s_waitcnt(0);
                tile_of(ragged, t, my0, my0 + TB, nothing);
            }
        }
    }
    lsum = halves_sum(lsum);

    if constexpr (FEW) {
        // join the waves: maxima and sums, then the rescaled accumulators, wave by wave through LDS
        float* xs = (float*)buf0[0][0];                         // [4][32][2]
        float* xo = xs + 4 * 32 * 2;                            // [32][HDP + 4]
        static_assert((4 * 32 * 2 + 32 * (HDP + 4)) * 4 <= Cfg::COPIES * 2 * TB, "the exchange fits the tile buffers");
        __syncthreads();
        if (hh == 0) { xs[(wave * 32 + lane) * 2] = mrun; xs[(wave * 32 + lane) * 2 + 1] = lsum; }
        __syncthreads();
        float mall = -INFINITY, lall = 0.f;
        for (int w = 0; w < 4; ++w) mall = vmax(mall, xs[(w * 32 + (lane & 31)) * 2]);
        const float mref = mall == -INFINITY ? 0.f : mall;
        const float unit = BIAS ? LOG2E : c2;
        for (int w = 0; w < 4; ++w) {
            const float mw = xs[(w * 32 + (lane & 31)) * 2];
            lall += xs[(w * 32 + (lane & 31)) * 2 + 1] * __builtin_amdgcn_exp2f((mw - mref) * unit);
        }
        const float mine = __builtin_amdgcn_exp2f((mrun - mref) * unit);
        for (int w = 3; w >= 0; --w) {
            if (wave == w) {
#pragma unroll
                for (int m = 0; m < DM; ++m)
#pragma unroll
                    for (int a = 0; a < 4; ++a) {
                        float* x = xo + (lane & 31) * (HDP + 4) + 32 * m + 8 * a + 4 * hh;
                        f32x4 v = {o[m][4 * a] * mine, o[m][4 * a + 1] * mine, o[m][4 * a + 2] * mine, o[m][4 * a + 3] * mine};
                        if (w < 3) { const f32x4 c = *(const f32x4*)x; v[0] += c[0]; v[1] += c[1]; v[2] += c[2]; v[3] += c[3]; }
                        if (w > 0) *(f32x4*)x = v;
                        else { o[m][4 * a] = v[0]; o[m][4 * a + 1] = v[1]; o[m][4 * a + 2] = v[2]; o[m][4 * a + 3] = v[3]; }
                    }
            }
            __syncthreads();
        }
        if (wave != 0) return;
        mrun = mall;
        lsum = lall;
    }

    if (!row_ok) return;
    const float mnat = BIAS ? mrun : mrun * p.scale;
    if (f.ns > 1) {
        const int64_t row = ((int64_t)split * p.B * p.Hkv + bh) * p.R + r;
        float* po = f.part_o + row * HDP;
#pragma unroll
        for (int m = 0; m < DM; ++m)
#pragma unroll
            for (int a = 0; a < 4; ++a) *(f32x4*)(po + 32 * m + 8 * a + 4 * hh) = (f32x4){o[m][4 * a], o[m][4 * a + 1], o[m][4 * a + 2], o[m][4 * a + 3]};
        if (hh == 0) { f.part_s[row * 2] = mnat; f.part_s[row * 2 + 1] = lsum; }
        return;
    }
    const float inv = lsum == 0.f ? 0.f : 1.0f / lsum;          // a row without keys: zeros
    T* orow = (T*)f.out + b * p.so.b + l * p.so.l + h * p.so.h;
#pragma unroll
    for (int m = 0; m < DM; ++m)
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            const int d = 32 * m + 8 * a + 4 * hh;
            if (d < p.hd) store4(orow + d, o[m][4 * a] * inv, o[m][4 * a + 1] * inv, o[m][4 * a + 2] * inv, o[m][4 * a + 3] * inv);
        }
    if (f.stat != nullptr && hh == 0) {
        float* st = f.stat + (((int64_t)b * p.H + h) * p.Lq + l) * 2;
        st[0] = mnat;
        st[1] = lsum;
    }
}

// Joins the splits.  A lane owns four elements of a row, HDP / 4 lanes a row.  DEEP: the lane groups of a wave take the splits of one row in turn (each with
// its own running maximum) and meet in shuffles, so that the loads of a row are few trips to memory deep; otherwise (few splits, many rows)
// each group has a row of its own.
template <typename T, int HDP, bool DEEP>
__global__ __launch_bounds__(256) void cross_join_kernel(const Fwd f) {
    constexpr int LR = HDP / 4 == 24 ? 32 : HDP / 4, NG = 64 / LR;          // lanes a row (96: eight of 32 stay idle), groups a wave
    const Prob& p = f.p;
    const int64_t rows = (int64_t)p.B * p.Hkv * p.R;
    const int lane = threadIdx.x & 63, grp = lane / LR, d = 4 * (lane % LR), first = DEEP ? grp : 0, step = DEEP ? NG : 1;
    const int64_t wave = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), g = DEEP ? wave : wave * NG + grp;
    if (g >= rows) return;                                                  // (DEEP: the whole wave)
    const bool on = d < HDP;
    float m = -INFINITY, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    auto add = [&](float mo, float lo, const f32x4& v) {
        const float mn = vmax(m, mo), ref = mn == -INFINITY ? 0.f : mn;
        const float wa = __builtin_amdgcn_exp2f((m - ref) * LOG2E), wb = __builtin_amdgcn_exp2f((mo - ref) * LOG2E);
        l = l * wa + lo * wb;
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] = acc[e] * wa + v[e] * wb;
        m = mn;
    };
    constexpr int U = 4;
    for (int s0 = first; s0 < f.ns; s0 += step * U) {
        float ms[U], ls[U];
        f32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int s = s0 + u * step;
            ms[u] = -INFINITY;
            ls[u] = 0.f;
            v[u] = (f32x4){0.f, 0.f, 0.f, 0.f};
            if (s < f.ns) {
                ms[u] = f.part_s[(s * rows + g) * 2];
                ls[u] = f.part_s[(s * rows + g) * 2 + 1];
                if (on) v[u] = *(const f32x4*)(f.part_o + (s * rows + g) * HDP + d);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) add(ms[u], ls[u], v[u]);
    }
#pragma unroll
    for (int o = DEEP ? LR : 64; o < 64; o <<= 1) {
        const float mo = __shfl_xor(m, o, 64), lo = __shfl_xor(l, o, 64);
        const f32x4 v = {__shfl_xor(acc[0], o, 64), __shfl_xor(acc[1], o, 64), __shfl_xor(acc[2], o, 64), __shfl_xor(acc[3], o, 64)};
        add(mo, lo, v);
    }
    if (DEEP && grp != 0) return;
    const int bh = (int)(g / p.R), r = (int)(g - (int64_t)bh * p.R), b = bh / p.Hkv, hk = bh - b * p.Hkv;
    int tok, h;
    row_of(p, hk, r, tok, h);
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    if (on && d < p.hd) store4((T*)f.out + b * p.so.b + tok * p.so.l + h * p.so.h + d, acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
    if (f.stat != nullptr && d == 0) {
        float* st = f.stat + (((int64_t)b * p.H + h) * p.Lq + tok) * 2;
        st[0] = m;
        st[1] = l;
    }
}

// How a launch is cut: row blocks, and splits of the keys where the row blocks alone leave CUs idle.
struct FwdPlan { bool few; int hd, hdp, nrb, ns; int64_t part_bytes; };
FwdPlan plan_fwd(const MarsCrossAttn* a) {
    FwdPlan pl;
    const int64_t R = (int64_t)(a->H / a->Hkv) * a->Lq;
    pl.hd = built_for(a->hd);
    pl.hdp = padded(pl.hd);
    pl.few = R <= 32;
    pl.nrb = (int)(pl.few ? 1 : (R + 127) / 128);
    const int64_t blocks = (int64_t)a->B * a->Hkv * pl.nrb;
    const int tiles = (a->Lk + 63) / 64;
    pl.ns = 1;
    if (blocks < 256) {
        const int64_t want = (512 + blocks - 1) / blocks;
        const int most = pl.few ? (tiles + 3) / 4 : (tiles + 1) / 2;             // at least two tiles a wave
        pl.ns = (int)(want < most ? want : most);
        if (pl.ns < 1) pl.ns = 1;
    } else if (!pl.few && blocks < 1024) {
        // Little more than a round of workgroups: some CUs work on one more than the others.  Cutting the keys evens that out where it gains more than
        // the partial results cost (written and read once at memory speed, and a launch) - 1369 queries over 6845 keys, 32 heads of 64: 352 workgroups on
        // 256 CUs, two cuts, 138 -> 118 us in bf16; over 1369 keys in f32 205 -> 174 us (48 heads over 2000:
        // 407 -> 352).  The rates are about what full rounds reach in each type.
        const double t1 = 4.0 * a->B * a->H * (double)a->Lq * a->Lk * pl.hd / (a->dtype == 1 ? 5e14 : 1e14), round1 = (double)((blocks + 255) / 256);
        double best = t1;
        for (int ns = 2; ns <= 4 && ns <= (tiles + 7) / 8; ++ns) {
            const double t = t1 * (double)((blocks * ns + 255) / 256) / ns / round1 + 8.0 * ns * a->B * a->Hkv * R * pl.hdp / 4e12 + 5e-6;
            if (t < 0.95 * best) { best = t; pl.ns = ns; }
        }
    }
    pl.part_bytes = pl.ns > 1 ? (int64_t)pl.ns * a->B * a->Hkv * R * (pl.hdp + 2) * 4 : 0;
    return pl;
}

template <typename T, int HD> int launch_fwd(const Fwd& f, bool few, hipStream_t s) {
    constexpr int HDP = padded(HD);
    const int64_t blocks = (int64_t)f.p.B * f.p.Hkv * f.nrb * f.ns;
    const dim3 grid((unsigned)blocks), block(256);
    if (f.p.bias != nullptr) {
        if (few) hipLaunchKernelGGL((cross_fwd_kernel<T, HD, true, true>), grid, block, 0, s, f);
        else hipLaunchKernelGGL((cross_fwd_kernel<T, HD, true, false>), grid, block, 0, s, f);
    } else {
        if (few) hipLaunchKernelGGL((cross_fwd_kernel<T, HD, false, true>), grid, block, 0, s, f);
        else hipLaunchKernelGGL((cross_fwd_kernel<T, HD, false, false>), grid, block, 0, s, f);
    }
    MARS_LAUNCH_CHECK();
    if (f.ns > 1) {
        const int64_t rows = (int64_t)f.p.B * f.p.Hkv * f.p.R;
        const bool deep = f.ns > 4;
        const int64_t per = deep ? 4 : 4 * (64 / (HDP / 4 == 24 ? 32 : HDP / 4)), groups = (rows + per - 1) / per;
        if (deep) hipLaunchKernelGGL((cross_join_kernel<T, HDP, true>), dim3((unsigned)groups), block, 0, s, f);
        else hipLaunchKernelGGL((cross_join_kernel<T, HDP, false>), dim3((unsigned)groups), block, 0, s, f);
        MARS_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T> int launch_fwd_hd(const Fwd& f, const FwdPlan& pl, hipStream_t s) {
    switch (pl.hd) {
        case 16: return launch_fwd<T, 16>(f, pl.few, s);
        case 32: return launch_fwd<T, 32>(f, pl.few, s);
        case 64: return launch_fwd<T, 64>(f, pl.few, s);
        case 80: return launch_fwd<T, 80>(f, pl.few, s);
        case 96: return launch_fwd<T, 96>(f, pl.few, s);
        default: return launch_fwd<T, 128>(f, pl.few, s);
    }
}

int64_t align256(int64_t x) { return (x + 255) / 256 * 256; }

}  // namespace

// ------------------------------------------------------------------------------------------------ host side, shared with the backward
static bool rows_ok(const void* ptr, const int64_t* st, int es) {
    return ((uintptr_t)ptr % 16 == 0) && (st[0] * es) % 16 == 0 && (st[1] * es) % 16 == 0 && (st[2] * es) % 16 == 0;
}

// what the workspace queries ask too: they divide by the counts of what a shape is cut into, and answer 0 for a shape that the call refuses
static int check_shape(const MarsCrossAttn* a, const char* what) {
    MARS_CHECK(a->B > 0 && a->Lq > 0 && a->Lk > 0 && a->H > 0 && a->Hkv > 0, "%s: bad shape B=%d Lq=%d Lk=%d H=%d Hkv=%d", what, a->B, a->Lq, a->Lk,
               a->H, a->Hkv);
    MARS_CHECK(a->H % a->Hkv == 0, "%s: %d query heads are no multiple of %d key heads", what, a->H, a->Hkv);
    MARS_CHECK(a->hd > 0 && a->hd <= 128, "%s: head dim %d (up to 128, a multiple of 16 bytes)", what, a->hd);
    MARS_CHECK((int64_t)(a->H / a->Hkv) * a->Lq < (1ll << 30) && a->Lk < (1 << 30), "%s: too many rows", what);
    MARS_CHECK((int64_t)a->B * a->H < (1ll << 30), "%s: too many heads", what);
    return 0;
}

int check(const MarsCrossAttn* a, bool backward) {
    const char* what = backward ? "cross_attn_bwd" : "cross_attn";
    MARS_CHECK(a && a->q && a->k && a->v && a->out, "%s: null pointer", what);
    MARS_CHECK(a->dtype == 0 || a->dtype == 1, "%s: dtype %d", what, a->dtype);
    const int es = a->dtype == 1 ? 2 : 4;
    if (const int rc = check_shape(a, what)) return rc;
    MARS_CHECK((a->hd * es) % 16 == 0, "%s: head dim %d (up to 128, a multiple of 16 bytes)", what, a->hd);
    MARS_CHECK(a->bias == nullptr || (a->bias_s[1] >= 0 && a->bias_s[1] < (1 << 28)), "%s: bias rows too far apart", what);
    MARS_CHECK(a->scale > 0.f && a->scale < INFINITY, "%s: scale must be positive and finite", what);
    MARS_CHECK(rows_ok(a->q, a->q_s, es) && rows_ok(a->k, a->k_s, es) && rows_ok(a->v, a->v_s, es) && rows_ok(a->out, a->out_s, es),
               "%s: rows must be 16-byte aligned", what);
    if (backward) {
        MARS_CHECK(a->stat && a->dout && a->dq && a->dk && a->dv, "%s: null pointer", what);
        MARS_CHECK(rows_ok(a->dout, a->dout_s, es) && rows_ok(a->dq, a->dq_s, es) && rows_ok(a->dk, a->dk_s, es) && rows_ok(a->dv, a->dv_s, es),
                   "%s: rows must be 16-byte aligned", what);
        MARS_CHECK(a->dbias == nullptr || a->bias != nullptr, "%s: a gradient of a bias that is not there", what);
    }
    // What the launches take, all of it before the first one: a refused call has written nothing.  (Only launches of fewer than 1024 blocks are cut further.)
    const int64_t nbh = (int64_t)a->B * a->Hkv, R = (int64_t)(a->H / a->Hkv) * a->Lq, most = 1ll << 24;
    MARS_CHECK(nbh * ((R + 127) / 128) < most && (!backward || nbh * (((int64_t)a->Lk + 127) / 128) < most), "%s: more workgroups than a launch takes", what);
    MARS_CHECK(a->mask == nullptr || (int64_t)a->B * 1024 < (1ll << 32), "%s: %d batch entries are more than a launch takes", what, a->B);
    MARS_CHECK(!backward || a->dbias == nullptr || (((int64_t)a->Lq + 127) / 128 <= 65535 && a->H <= 65535 && ((int64_t)a->Lk + 63) / 64 < most),
               "%s: more workgroups than a launch takes", what);
    return 0;
}

static Strides st3(const int64_t* s) { return Strides{s[0], s[1], s[2]}; }

void describe(const MarsCrossAttn* a, Prob& p) {
    p = Prob{};
    p.q = a->q; p.k = a->k; p.v = a->v; p.out = a->out; p.dout = a->dout;
    p.sq = st3(a->q_s); p.sk = st3(a->k_s); p.sv = st3(a->v_s); p.so = st3(a->out_s); p.sdo = st3(a->dout_s);
    p.bias = a->bias; p.bias_h = a->bias_s[0]; p.bias_l = a->bias_s[1];
    p.stat = a->stat;
    p.B = a->B; p.Lq = a->Lq; p.Lk = a->Lk; p.H = a->H; p.Hkv = a->Hkv; p.hd = a->hd;
    p.grp = a->H / a->Hkv;
    p.R = p.grp * a->Lq;
    p.scale = a->scale;
    p.cnt = a->kv_len;
}

int64_t key_ws_bytes(const MarsCrossAttn* a) { return a->mask ? align256((int64_t)a->B * a->Lk * 4) + align256((int64_t)a->B * 4) : 0; }

int prepare_keys(const MarsCrossAttn* a, Prob& p, int32_t* ws, hipStream_t s) {
    if (a->mask == nullptr) return 0;
    int32_t* cnt = (int32_t*)((char*)ws + align256((int64_t)a->B * a->Lk * 4));
    hipLaunchKernelGGL(list_keys_kernel, dim3((unsigned)a->B), dim3(1024), 0, s, a->mask, a->kv_len, a->Lk, ws, cnt);
    MARS_LAUNCH_CHECK();
    p.idx = ws;
    p.cnt = cnt;
    return 0;
}

int64_t bwd_ws_bytes(const MarsCrossAttn* a);

}  // namespace xattn

extern "C" int64_t marship_cross_attn_ws(const MarsCrossAttn* a, int backward) {
    if (a == nullptr || xattn::check_shape(a, "cross_attn_ws") != 0) return 0;
    const int64_t keys = xattn::key_ws_bytes(a);
    if (backward) return keys + xattn::bwd_ws_bytes(a);
    return keys + xattn::align256(xattn::plan_fwd(a).part_bytes);
}

extern "C" int marship_cross_attn(const MarsCrossAttn* a, void* stream) {
    using namespace xattn;
    if (const int rc = check(a, false)) return rc;
    const int64_t need = marship_cross_attn_ws(a, 0);
    MARS_CHECK(need == 0 || (a->ws != nullptr && (uintptr_t)a->ws % 16 == 0 && a->ws_bytes >= need), "cross_attn: workspace of %lld bytes, %lld needed",
               (long long)a->ws_bytes, (long long)need);
    hipStream_t s = (hipStream_t)stream;
    Fwd f{};
    describe(a, f.p);
    if (const int rc = prepare_keys(a, f.p, (int32_t*)a->ws, s)) return rc;
    const FwdPlan pl = plan_fwd(a);
    f.out = a->out;
    f.stat = a->stat;
    f.nrb = pl.nrb;
    f.ns = pl.ns;
    if (pl.ns > 1) {
        const int64_t rows = (int64_t)a->B * a->Hkv * f.p.R;
        f.part_o = (float*)((char*)a->ws + key_ws_bytes(a));
        f.part_s = f.part_o + pl.ns * rows * pl.hdp;
    }
    return a->dtype == 1 ? launch_fwd_hd<__bf16>(f, pl, s) : launch_fwd_hd<float>(f, pl, s);
}

// Softmax attention of any length: backward, from the inputs, the output and the saved row statistics; the probabilities are
// formed again, never stored.  With P = exp(x - m) / l, dP_ij = dO_i . v_j and delta_i = sum_d dO_id O_id:
//
//   dV_j = sum_i P_ij dO_i,   dS_ij = P_ij (dP_ij - delta_i),   dQ_i = scale * sum_j dS_ij k_j,   dK_j = scale * sum_i dS_ij q_i
//
// Two passes, so that every sum has one owner and a fixed order (no atomics; the same bits every time):
//   dK / dV: a wave owns 32 keys (their K and V rows stay in registers as fragments) and walks the rows of all query heads that
//     share the key head; S = Q K^T has the key in the lane, so P^T and dS^T are register by register the A operands of
//     dV += P^T dO and dK += dS^T Q.
//   dQ: a wave owns 32 rows and walks the keys, as in the forward; dS^T is the B operand of dQ^T += K^T dS^T.
// The two recompute S and dP: 14 products of 2 * pairs * dh operations where one pass with atomics needs 10.
// delta comes from a small kernel before both.
#include "attention_long_dev.h"
#include <algorithm>

namespace nr {
namespace al {

// delta[row] = sum_d dout * out, 16 lanes per row
template <class T>
__global__ __launch_bounds__(256) void attn_delta_kernel(const Args a) {
    const int64_t idx = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 4;          // (n, i, head)
    const int lane = threadIdx.x & 15;
    const int64_t rows = a.N * a.Sq * a.H;
    float s = 0.f;
    int64_t n = 0;
    int i = 0, head = 0;
    if (idx < rows) {
        const int64_t ni = idx / a.H;
        head = (int)(idx - ni * a.H);
        n = ni / a.Sq;
        i = (int)(ni - n * a.Sq);
        const T* o = static_cast<const T*>(a.out) + n * a.so.n + i * a.so.s + head * a.so.h;
        const T* g = static_cast<const T*>(a.dout) + n * a.sdo.n + i * a.sdo.s + head * a.sdo.h;
        for (int d = lane; d < a.dh; d += 16) s = fmaf((float)o[d], (float)g[d], s);
    }
#pragma unroll
    for (int x = 8; x > 0; x >>= 1) s += __shfl_xor(s, x, 64);
    if (idx < rows && lane == 0) a.delta[n * a.sd.n + i * a.sd.s + head * a.sd.h] = s;
}

// ---------------------------------------------------------------- dK, dV
template <class T, int DHP> struct DkvCfg {
    static constexpr int QSUB = sizeof(T) == 2 ? 2 : 1, QT = 32 * QSUB, PITCH = DHP + Ty<T>::PAD;
    static constexpr size_t TILES = (size_t)2 * 2 * QT * PITCH * sizeof(T);
    static constexpr size_t BYTES = TILES + (size_t)2 * 4 * QT * 4;              // + two stages of m, 1/l, delta, last key
};

template <class T, int DHP, bool VEC>
__global__ __launch_bounds__(256) void attn_dkv_kernel(const Args a) {
    typedef DkvCfg<T, DHP> C;
    constexpr int QSUB = C::QSUB, QT = C::QT, PITCH = C::PITCH, KS = DHP / 16, DT = DHP / 32;
    constexpr bool NAT = sizeof(T) == 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* Qs = reinterpret_cast<T*>(smem);
    T* Gs = Qs + 2 * QT * PITCH;
    float* St = reinterpret_cast<float*>(smem + C::TILES);                       // [2][4][QT]
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    uint32_t b = xcd_order(blockIdx.x, gridDim.x);
    const int sp = b % a.splits; b /= a.splits;
    int kb = b % a.nblk_r; b /= a.nblk_r;
    const int g = b % a.G;
    const int64_t n = b / a.G;
    if (a.causal) kb = heavy_light(kb, a.nblk_r);
    const int key = kb * 128 + 32 * w + l31;
    bool there = key < a.Sk;
    const bool masked = there && a.mask && a.mask[n * a.Sk + key] == 0;
    const float sink = masked ? a.fill : 0.f;                                    // additive mode
    if (!a.additive && masked) there = false;
    typename Ty<T>::Frag kf[KS], vf[KS];
    {   // an absent key's rows read as zero
        const T* kp = static_cast<const T*>(a.k) + n * a.sk.n + (int64_t)key * a.sk.s + g * a.sk.h;
        const T* vp = static_cast<const T*>(a.v) + n * a.sv.n + (int64_t)key * a.sv.s + g * a.sv.h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kf[ks] = load_frag<VEC>(kp + 16 * ks + 8 * h, there ? a.dh - 16 * ks - 8 * h : 0);
            vf[ks] = load_frag<VEC>(vp + 16 * ks + 8 * h, there ? a.dh - 16 * ks - 8 * h : 0);
        }
    }
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) { dk[t] = zero16(); dv[t] = zero16(); }
    const float scale2 = a.scale * LOG2E;
    const int off = a.Sk - a.Sq;
    const T* qb = static_cast<const T*>(a.q) + n * a.sq.n;
    const T* gb = static_cast<const T*>(a.dout) + n * a.sdo.n;

    const int rbeg = sp * a.per_split, rend = min(a.R, rbeg + a.per_split);
    const bool dead = !__syncthreads_or(there);                                  // no key of this block is there
    // causal: a tile of rows of one head whose last row does not reach the block's first key has nothing to add
    auto skip = [&](int r0) {
        if (!a.causal) return false;
        const int last = min(r0 + QT, rend) - 1;
        const int h0 = r0 / a.Sq;
        return h0 == last / a.Sq && last - h0 * a.Sq + off < kb * 128;
    };
    auto next = [&](int r0) {
        while (r0 < rend && skip(r0)) {
            // the first row of this head that reaches the block, or the next head
            const int h0 = r0 / a.Sq, want = h0 * a.Sq + min(a.Sq, max(0, kb * 128 - off));
            r0 += max(QT, (want - r0) / QT * QT);
        }
        return r0;
    };
    Stage<T, DHP, QT, VEC> sq, sg;
    float st[3];
    int st_lim = 0;
    auto fetch = [&](int r0) {
        auto at = [&](const T* base, const AttnStrides& s, int r) -> const T* {
            const int row = r0 + r;
            if (row >= rend) return nullptr;
            const int hh = row / a.Sq, i = row - hh * a.Sq;
            return base + i * s.s + (g * a.rep + hh) * s.h;
        };
        sq.load(tid, a.dh, [&](int r) { return at(qb, a.sq, r); });
        sg.load(tid, a.dh, [&](int r) { return at(gb, a.sdo, r); });
        if (tid < QT) {
            const int row = r0 + tid;
            st[0] = 0.f; st[1] = 0.f; st[2] = 0.f; st_lim = -1;
            if (row < rend) {
                const int hh = row / a.Sq, i = row - hh * a.Sq, head = g * a.rep + hh;
                const int64_t x = (n * a.H + head) * a.Sq + i;
                st[0] = a.row_max[x];
                st[1] = a.row_sum[x];
                st[2] = a.delta[n * a.sd.n + i * a.sd.s + head * a.sd.h];
                st_lim = a.causal ? i + off : 0x7fffffff;
            }
        }
    };
    auto put = [&](int buf) {
        sq.store(tid, Qs + buf * QT * PITCH, [](int) { return true; });
        sg.store(tid, Gs + buf * QT * PITCH, [](int) { return true; });
        if (tid < QT) {
            float* s = St + buf * 4 * QT + tid;
            s[0] = NAT ? st[0] : st[0] * LOG2E;
            s[QT] = st[1] != 0.f ? 1.f / st[1] : 0.f;
            s[2 * QT] = st[2];
            reinterpret_cast<int*>(s)[3 * QT] = st_lim;
        }
    };
    int r0 = dead ? rend : next(rbeg), buf = 0;
    if (r0 < rend) { fetch(r0); put(0); }
    __syncthreads();
    while (r0 < rend) {
        const int r1 = next(r0 + QT);
        if (r1 < rend) fetch(r1);
        const T* Qt = Qs + buf * QT * PITCH;
        const T* Gt = Gs + buf * QT * PITCH;
        const float* S0 = St + buf * 4 * QT;
#pragma unroll
        for (int s = 0; s < QSUB; ++s) {
            f32x16 x = zero16(), dp = zero16();
            const T* qr = Qt + (32 * s + l31) * PITCH + 8 * h;
            const T* gr = Gt + (32 * s + l31) * PITCH + 8 * h;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                x = mul(near_frag(qr + 16 * ks), kf[ks], x);
                dp = mul(near_frag(gr + 16 * ks), vf[ks], dp);
            }
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int rr = 32 * s + 8 * q + 4 * h;
                const f32x4 mx = *reinterpret_cast<const f32x4*>(S0 + rr), rl = *reinterpret_cast<const f32x4*>(S0 + QT + rr);
                const f32x4 de = *reinterpret_cast<const f32x4*>(S0 + 2 * QT + rr);
                const int* lm = reinterpret_cast<const int*>(S0) + 3 * QT + rr;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * q + e;
                    float p;
                    if (NAT) {
                        float y = x[r] * a.scale;
                        if (a.additive) y += sink;
                        p = __builtin_amdgcn_exp2f((y - mx[e]) * LOG2E) * rl[e];
                    } else p = __builtin_amdgcn_exp2f(fmaf(x[r], scale2, -mx[e])) * rl[e];
                    if (!there || key > lm[e]) p = 0.f;
                    float pd = p, dpd = dp[r];
                    if (a.drop) {
                        const int row = r0 + rr + e, hh = row / a.Sq, i = row - hh * a.Sq;
                        const uint64_t idx = ((uint64_t)(n * a.H + g * a.rep + hh) * a.Sq + i) * a.Sk + key;
                        const float f = philox_pick(philox4x32_10(a.seed, idx >> 2, a.site), (int)(idx & 3)) >= a.thr ? a.keep : 0.f;
                        pd *= f; dpd *= f;
                    }
                    x[r] = pd;
                    dp[r] = p * (dpd - de[e]);
                }
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const typename Ty<T>::Frag pf = tile_frag<T>(x, k2), sf = tile_frag<T>(dp, k2);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    dv[d] = mul(pf, col_frag<PITCH>(Gt, 32 * s + 16 * k2, 32 * d, lane), dv[d]);
                    dk[d] = mul(sf, col_frag<PITCH>(Qt, 32 * s + 16 * k2, 32 * d, lane), dk[d]);
                }
            }
        }
        if (r1 < rend) put(buf ^ 1);
        __syncthreads();
        buf ^= 1;
        r0 = r1;
    }
    const int64_t rows = a.N * a.G * a.Sk;
    T* dkp = static_cast<T*>(a.dk) + n * a.sdk.n + g * a.sdk.h;
    T* dvp = static_cast<T*>(a.dv) + n * a.sdv.n + g * a.sdv.h;
    float* pk = a.part + (2 * sp * rows + (n * a.G + g) * a.Sk) * a.dhs;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int kk = kb * 128 + 32 * w + tile_row(r, h);
        if (kk >= a.Sk) continue;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int c = 32 * d + l31;
            if (c >= a.dh) continue;
            if (a.splits > 1) {
                pk[(int64_t)kk * a.dhs + c] = dk[d][r] * a.scale;
                pk[(rows + kk) * a.dhs + c] = dv[d][r];
            } else {
                dkp[kk * a.sdk.s + c] = (T)(dk[d][r] * a.scale);
                dvp[kk * a.sdv.s + c] = (T)dv[d][r];
            }
        }
    }
}

// ---------------------------------------------------------------- dQ
template <class T, int DHP, int WK> struct DqCfg {
    static constexpr int KSUB = (sizeof(T) == 2 && WK == 1) ? 2 : 1, KT = 32 * KSUB * WK, PITCH = DHP + Ty<T>::PAD;
    static constexpr int NBUF = (sizeof(T) == 4 && DHP == 128 && WK == 4) ? 1 : 2;
    static constexpr size_t LDS = (size_t)NBUF * 2 * KT * PITCH * sizeof(T);
    static constexpr size_t JOIN = WK > 1 ? (size_t)WK * DHP * 32 * 4 : 0;
    static constexpr size_t BYTES = LDS > JOIN ? LDS : JOIN;
};

template <class T, int DHP, bool VEC, int WK>
__global__ __launch_bounds__(256) void attn_dq_kernel(const Args a) {
    typedef DqCfg<T, DHP, WK> C;
    constexpr int WQ = 4 / WK, KSUB = C::KSUB, KT = C::KT, PITCH = C::PITCH, KS = DHP / 16, DT = DHP / 32, WORDS = (KT + 63) / 64;
    constexpr bool NAT = sizeof(T) == 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* Ks = reinterpret_cast<T*>(smem);
    T* Vs = Ks + C::NBUF * KT * PITCH;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wq = w / WK, wk = w % WK;

    uint32_t b = xcd_order(blockIdx.x, gridDim.x);
    const int sp = b % a.splits; b /= a.splits;
    int rb = b % a.nblk_r; b /= a.nblk_r;
    const int g = b % a.G;
    const int64_t n = b / a.G;
    if (a.causal) rb = heavy_light(rb, a.nblk_r);
    const int r0 = rb * 32 * WQ;
    const int row = r0 + 32 * wq + l31;
    const bool live = row < a.R;
    const int hh = live ? row / a.Sq : 0, i = live ? row - hh * a.Sq : 0, head = g * a.rep + hh;
    const int lim = a.causal ? i + a.Sk - a.Sq : 0x7fffffff;
    int lim_min = live ? lim : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lim_min = min(lim_min, __shfl_xor(lim_min, o, 64));
    lim_min = __builtin_amdgcn_readfirstlane(lim_min);
    typename Ty<T>::Frag qf[KS], gf[KS];
    const T* qp = static_cast<const T*>(a.q) + n * a.sq.n + i * a.sq.s + head * a.sq.h;
    const T* gp = static_cast<const T*>(a.dout) + n * a.sdo.n + i * a.sdo.s + head * a.sdo.h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        qf[ks] = load_frag<VEC>(qp + 16 * ks + 8 * h, live ? a.dh - 16 * ks - 8 * h : 0);
        gf[ks] = load_frag<VEC>(gp + 16 * ks + 8 * h, live ? a.dh - 16 * ks - 8 * h : 0);
    }
    float m = 0.f, rl = 0.f, de = 0.f;
    if (live) {
        const int64_t x = (n * a.H + head) * a.Sq + i;
        m = a.row_max[x];
        if (!NAT) m *= LOG2E;
        rl = a.row_sum[x];
        rl = rl != 0.f ? 1.f / rl : 0.f;
        de = a.delta[n * a.sd.n + i * a.sd.s + head * a.sd.h];
    }
    const int begin = sp * a.per_split;
    int end = min(a.Sk, begin + a.per_split);
    if (a.causal) {
        const int last = min(r0 + 32 * WQ, a.R) - 1;
        const int imax = r0 / a.Sq == last / a.Sq ? last % a.Sq : a.Sq - 1;
        end = min(end, imax + a.Sk - a.Sq + 1);
    }
    const int64_t* mask = a.mask ? a.mask + n * a.Sk : nullptr;
    if (mask && !a.additive) end = present_end(mask, begin, end, tid);
    const T* kp = static_cast<const T*>(a.k) + n * a.sk.n + g * a.sk.h;
    const T* vp = static_cast<const T*>(a.v) + n * a.sv.n + g * a.sv.h;
    const float scale2 = a.scale * LOG2E;
    f32x16 dq[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = zero16();

    Stage<T, DHP, KT, VEC> sk, sv;
    KeyBits<WORDS> kb;
    uint64_t bits[WORDS];
    const int tiles = end > begin ? (end - begin + KT - 1) / KT : 0;
    auto fetch = [&](int j) {
        kb.load(mask, j, end, lane);
        sk.load(tid, a.dh, [&](int r) { return j + r < end ? kp + (int64_t)(j + r) * a.sk.s : nullptr; });
        sv.load(tid, a.dh, [&](int r) { return j + r < end ? vp + (int64_t)(j + r) * a.sv.s : nullptr; });
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int x = 0; x < WORDS; ++x) bits[x] = kb.bits(x);
        auto keep = [&](int r) { return a.additive || ((bits[r >> 6] >> (r & 63)) & 1); };
        sk.store(tid, Ks + buf * KT * PITCH, keep);
        sv.store(tid, Vs + buf * KT * PITCH, keep);
    };
    if (tiles) { fetch(begin); put(0); }
    __syncthreads();
    for (int t = 0; t < tiles; ++t) {
        const int j0 = begin + t * KT, buf = C::NBUF == 2 ? (t & 1) : 0;
        uint64_t now[WORDS];
#pragma unroll
        for (int x = 0; x < WORDS; ++x) now[x] = bits[x];
        if (t + 1 < tiles) fetch(j0 + KT);
        const T* Kt = Ks + buf * KT * PITCH;
        const T* Vt = Vs + buf * KT * PITCH;
#pragma unroll
        for (int s = 0; s < KSUB; ++s) {
            const int ko = 32 * (wk * KSUB + s), kw = j0 + ko;
            uint32_t sub = (uint32_t)(now[ko >> 6] >> (ko & 63));
            if (!sub && !(a.additive && kw < end)) continue;
            f32x16 x = zero16(), dp = zero16();
            const T* kr = Kt + (ko + l31) * PITCH + 8 * h;
            const T* vr = Vt + (ko + l31) * PITCH + 8 * h;
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                x = mul(near_frag(kr + 16 * ks), qf[ks], x);
                dp = mul(near_frag(vr + 16 * ks), gf[ks], dp);
            }
            if (NAT) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= a.scale;
                if (a.additive) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) if (!((sub >> tile_row(r, h)) & 1)) x[r] += a.fill;
                    const int left = end - kw;
                    sub = left >= 32 ? ~0u : (left > 0 ? (1u << left) - 1 : 0u);
                }
            }
            if (sub != ~0u || kw + 31 > lim_min) hide(x, sub, kw, lim, h);
            const uint64_t rlin = ((uint64_t)(n * a.H + head) * a.Sq + i) * a.Sk;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                uint32_t kp4 = 0;
                if (a.drop) kp4 = keep4(a, rlin + kw + 8 * q + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int r = 4 * q + e;
                    const float p = __builtin_amdgcn_exp2f(NAT ? (x[r] - m) * LOG2E : fmaf(x[r], scale2, -m)) * rl;
                    const float g1 = a.drop ? (((kp4 >> e) & 1) ? dp[r] * a.keep : 0.f) : dp[r];
                    dp[r] = p * (g1 - de);
                }
            }
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                const typename Ty<T>::Frag sf = tile_frag<T>(dp, k2);
#pragma unroll
                for (int d = 0; d < DT; ++d) dq[d] = mul(col_frag<PITCH>(Kt, ko + 16 * k2, 32 * d, lane), sf, dq[d]);
            }
        }
        if (C::NBUF == 1) __syncthreads();
        if (t + 1 < tiles) put(C::NBUF == 2 ? 1 - buf : 0);
        __syncthreads();
    }
    if (WK > 1) {
        float* slab = reinterpret_cast<float*>(smem);                            // [WK][DHP][32]
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) slab[(wk * DHP + 32 * d + tile_row(r, h)) * 32 + l31] = dq[d][r];
        __syncthreads();
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q == wk) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float t = 0.f;
#pragma unroll
                        for (int x = 0; x < WK; ++x) t += slab[(x * DHP + 32 * d + tile_row(4 * q + e, h)) * 32 + l31];
                        dq[d][4 * q + e] = t;
                    }
                }
    }
    if (!live) return;
    const int64_t rt = (n * a.G + g) * a.R + row, rows = a.N * a.G * a.R;
    T* dp = static_cast<T*>(a.dq) + n * a.sdq.n + i * a.sdq.s + head * a.sdq.h;
    float* pr = a.part + (sp * rows + rt) * a.dhs;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            if (WK > 1 && q != wk) continue;
            const int c = 32 * d + 8 * q + 4 * h;
            const f32x4 v = {dq[d][4 * q] * a.scale, dq[d][4 * q + 1] * a.scale, dq[d][4 * q + 2] * a.scale, dq[d][4 * q + 3] * a.scale};
            if (a.splits > 1) store4<true>(pr + c, v, a.dhs - c);
            else store4<VEC>(dp + c, v, a.dh - c);
        }
}

// sums the splits of dQ (which = 0), or of dK and dV (which = 1): four columns per thread, splits in order
template <class T>
__global__ __launch_bounds__(256) void attn_sum_kernel(const Args a, int which) {
    const int quads = a.dhs / 4;
    const int64_t L = which ? a.Sk : a.R, rows = a.N * a.G * L, total = rows * quads * (which ? 2 : 1);
    int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= total) return;
    const int second = idx >= rows * quads;      // dV
    if (second) idx -= rows * quads;
    const int64_t rt = idx / quads;
    const int c = (int)(idx - rt * quads) * 4;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.splits; ++s) {
        const float* p = a.part + ((which ? (2 * s + second) * rows : s * rows) + rt) * a.dhs + c;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += c + e < a.dh ? p[e] : 0.f;
    }
    const int64_t ng = rt / L;
    const int r = (int)(rt - ng * L);
    const int64_t n = ng / a.G, g = ng - n * a.G;
    T* dst;
    if (!which) {
        const int hh = r / a.Sq, i = r - hh * a.Sq;
        dst = static_cast<T*>(a.dq) + n * a.sdq.n + i * a.sdq.s + (g * a.rep + hh) * a.sdq.h;
    } else {
        const AttnStrides& st = second ? a.sdv : a.sdk;
        dst = static_cast<T*>(second ? a.dv : a.dk) + n * st.n + r * st.s + g * st.h;
    }
    store4<false>(dst + c, o, a.dh - c);
}

// ---------------------------------------------------------------- host
struct BwdPlan { int wk, nblk_q, nblk_k; Split q, kv; size_t ws; };
static BwdPlan plan_bwd(const AttnProblem& p) {
    BwdPlan f;
    const int64_t R = (int64_t)(p.H / p.G) * p.Sq;
    f.wk = R <= 32 ? 4 : 1;
    f.nblk_q = cdiv(R, 32 * (4 / f.wk));
    f.nblk_k = cdiv(p.Sk, 128);
    f.q = split_axis(p.N * p.G * f.nblk_q, p.Sk, 128);
    f.kv = split_axis(p.N * p.G * f.nblk_k, (int)R, 64);
    const size_t row = (size_t)((p.dh + 3) / 4 * 4) * 4;
    const size_t wq = f.q.splits > 1 ? f.q.splits * (size_t)(p.N * p.G * R) * row : 0;
    const size_t wk = f.kv.splits > 1 ? 2 * f.kv.splits * (size_t)(p.N * p.G * p.Sk) * row : 0;
    f.ws = std::max(wq, wk);                     // the two passes run one after the other
    return f;
}

template <class T, int DHP, bool VEC>
static int launch_dkv(const Args& a, unsigned grid, hipStream_t s) {
    constexpr size_t bytes = DkvCfg<T, DHP>::BYTES;
    if (bytes > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_dkv_kernel<T, DHP, VEC>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DHP, VEC>), dim3(grid), dim3(256), bytes, s, a);
    return check_launch("attention_bwd dk/dv");
}
template <class T, int DHP, bool VEC, int WK>
static int launch_dq(const Args& a, unsigned grid, hipStream_t s) {
    constexpr size_t bytes = DqCfg<T, DHP, WK>::BYTES;
    if (bytes > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_dq_kernel<T, DHP, VEC, WK>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    hipLaunchKernelGGL((attn_dq_kernel<T, DHP, VEC, WK>), dim3(grid), dim3(256), bytes, s, a);
    return check_launch("attention_bwd dq");
}
template <class T, bool VEC> static int pick_dkv(const Args& a, unsigned grid, hipStream_t s) {
    if (a.dh <= 32) return launch_dkv<T, 32, VEC>(a, grid, s);
    if (a.dh <= 64) return launch_dkv<T, 64, VEC>(a, grid, s);
    return launch_dkv<T, 128, VEC>(a, grid, s);
}
template <class T, bool VEC, int WK> static int pick_dq(const Args& a, unsigned grid, hipStream_t s) {
    if (a.dh <= 32) return launch_dq<T, 32, VEC, WK>(a, grid, s);
    if (a.dh <= 64) return launch_dq<T, 64, VEC, WK>(a, grid, s);
    return launch_dq<T, 128, VEC, WK>(a, grid, s);
}
template <class T> static int run_sum(const Args& a, int which, hipStream_t s) {
    if (a.splits == 1) return NR_OK;
    const int64_t threads = a.N * a.G * (int64_t)(which ? 2 * (int64_t)a.Sk : a.R) * (a.dhs / 4);
    hipLaunchKernelGGL((attn_sum_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a, which);
    return check_launch("attention_bwd sum");
}

template <class T>
static int run_bwd(Args a, const BwdPlan& f, bool vec, bool room, hipStream_t s) {
    const int64_t rows = a.N * a.Sq * a.H;
    hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((rows * 16 + 255) / 256)), dim3(256), 0, s, a);
    if (int rc = check_launch("attention_bwd delta")) return rc;
    a.nblk_r = f.nblk_k; a.splits = room ? f.kv.splits : 1; a.per_split = room ? f.kv.per : a.R;
    unsigned grid = (unsigned)(a.N * a.G * (int64_t)a.nblk_r * a.splits);
    if (int rc = vec ? pick_dkv<T, true>(a, grid, s) : pick_dkv<T, false>(a, grid, s)) return rc;
    if (int rc = run_sum<T>(a, 1, s)) return rc;
    a.nblk_r = f.nblk_q; a.splits = room ? f.q.splits : 1; a.per_split = room ? f.q.per : a.Sk;
    grid = (unsigned)(a.N * a.G * (int64_t)a.nblk_r * a.splits);
    int rc = f.wk == 4 ? (vec ? pick_dq<T, true, 4>(a, grid, s) : pick_dq<T, false, 4>(a, grid, s))
                       : (vec ? pick_dq<T, true, 1>(a, grid, s) : pick_dq<T, false, 1>(a, grid, s));
    return rc != NR_OK ? rc : run_sum<T>(a, 0, s);
}

}  // namespace al

size_t attn_long_bwd_ws_bytes(const AttnProblem& p) { return al::plan_bwd(p).ws; }

int attn_long_bwd(const AttnProblem& p, const AttnGrad& g, void* ws, size_t ws_bytes, hipStream_t s) {
    if (p.N == 0 || p.Sq == 0 || p.Sk == 0) return NR_OK;
    const al::BwdPlan f = al::plan_bwd(p);
    const int64_t grid = p.N * p.G * std::max<int64_t>((int64_t)f.nblk_k * f.kv.splits, (int64_t)f.nblk_q * f.q.splits);
    const int64_t rows = p.N * p.Sq * p.H;
    NR_UNSUPPORTED(grid > 0x7fffffff || rows > ((int64_t)1 << 34), "attention_bwd: %lld workgroups", (long long)grid);
    al::Args a = al::make_args(p);
    a.out = const_cast<void*>(g.out); a.so = g.so; a.dout = g.dout; a.sdo = g.sdo;
    a.row_max = const_cast<float*>(g.row_max); a.row_sum = const_cast<float*>(g.row_sum);
    a.delta = g.delta; a.sd = g.sd;
    a.dq = g.dq; a.dk = g.dk; a.dv = g.dv; a.sdq = g.sdq; a.sdk = g.sdk; a.sdv = g.sdv;
    a.part = static_cast<float*>(ws);
    const size_t e = p.bf16 ? 2 : 4;
    const bool vec = al::all_aligned(p) && al::aligned16(g.dout, g.sdo, p.dh, e) && al::aligned16(g.dq, g.sdq, p.dh, e);
    const bool room = !f.ws || (ws && ws_bytes >= f.ws);      // without room for the partial sums nothing is split
    return p.bf16 ? al::run_bwd<__bf16>(a, f, vec, room, s) : al::run_bwd<float>(a, f, vec, room, s);
}

}  // namespace nr

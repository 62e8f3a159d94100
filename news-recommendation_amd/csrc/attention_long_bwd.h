// Softmax attention of any length: backward kernels (instantiated by attention_long_bwd_{f32,bf16}.hip), from the inputs, the output
// and the saved row statistics; the probabilities are formed again, never stored.  With P = exp(x - m) / l, dP_ij = dO_i . v_j and delta_i = sum_d dO_id O_id:
//
//   dV_j = sum_i P_ij dO_i,   dS_ij = P_ij (dP_ij - delta_i),   dQ_i = scale * sum_j dS_ij k_j,   dK_j = scale * sum_i dS_ij q_i
//
// Two passes, so that every sum has one owner and a fixed order (no atomics; the same bits every time):
//   dK / dV: a wave owns 32 keys (their K and V rows stay in registers as fragments) and walks the rows of all query heads that
//     share the key head; S = Q K^T has the key in the lane, so P^T and dS^T are register by register the A operands of
//     dV += P^T dO and dK += dS^T Q.
//   dQ: a wave owns 32 rows and walks the keys, as in the forward; dS^T is the B operand of dQ^T += K^T dS^T.
// The two recompute S and dP: 14 products of 2 * pairs * dh operations where one pass with atomics needs 10.
// delta: the dQ pass forms it from the rows it holds anyway and, running first, leaves it for the other; where it has no place of
// its own but lies in dQ's rows (attention_long.h), a small kernel writes it there, the dK / dV pass reads it and dQ goes last.
//
// Measured (MI355X).  4001 x 4001 causal, 16 heads (4 of them with keys) of 128, bf16: dQ 160 us (600 TFLOP/s of its three products),
// dK / dV 222 us (580 of its four), 19 us to join the splits.  dK / dV holds K and V fragments and both sums, 256 registers at 128
// columns: one wave per SIMD, so a tile's LDS reads and exponentials are hidden only by its own products.  16 x 512 ragged, 12 heads
// of 64, bf16: dQ 34 us, dK / dV 41 us (three waves per SIMD; 52 on average in one run of two); fp32 histories of 200, 12 heads of 25: 42
// and 52 us, bound by the latency of a block's few tiles.  Dropout of 0.1: the same texts dQ 78 us, dK / dV 209 (a call of the generator
// per element, of whose four numbers one is used: a lane's elements are rows of one key); the histories 63 and 94; 16 x 512, 12 heads of
// 64 in fp32: 143 and 293.
//
// Registers that do not fit and go to scratch memory, per lane (in brackets where addresses are unaligned): dK / dV, bf16, 64 columns 9
// (22), fp32, 64 columns 10 (20), 128 columns 61 (78); dQ, fp32, 128 columns and few rows 0 (285), 64 columns 0 (28), bf16, 128 columns 0
// (36), its one-tile form 34 (116).  With dropout: dK / dV, bf16, 32 columns 29 (60), 64 columns 128 (265), fp32, 64 columns 74 (86), 128
// columns 98 (115); dQ, fp32, 64 columns 27 (40), 128 columns and few rows 18 (300), bf16, 128 columns 18 (61), one-tile form 62 (187).
#pragma once
#include "attention_long_dev.h"

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
// a tile holds QT positions of one query head; the tiles of all query heads of the key head follow one another
template <class T, int DHP> struct DkvCfg {
    static constexpr int QSUB = sizeof(T) == 2 ? 2 : 1, QT = 32 * QSUB;
    typedef typename MulType<T, 1>::M M;
    typedef Lds<M, QT, DHP> L;
    static constexpr size_t TILES = 2 * 2 * L::BYTES;
    static constexpr size_t BYTES = TILES + (size_t)2 * 3 * QT * 4;              // + two stages of the rows' statistics
    static constexpr int WAVES = DHP <= 64 ? (sizeof(T) == 2 ? 3 : 2) : 1;
};

template <class T, int DHP, bool VEC, bool DROP>
__global__ __launch_bounds__(256, (DkvCfg<T, DHP>::WAVES)) void attn_dkv_kernel(const Args a) {
    typedef DkvCfg<T, DHP> C;
    constexpr int QSUB = C::QSUB, QT = C::QT, KS = DHP / 16, DT = DHP / 32;
    constexpr bool NAT = sizeof(T) == 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef typename C::M M;
    typedef typename C::L L;
    char* Qs = smem;
    char* Gs = smem + 2 * L::BYTES;
    float* St = reinterpret_cast<float*>(smem + C::TILES);                       // [2][3][QT]: fp32 m, 1 / l, delta; bf16 m + log2 l, -, delta
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);

    const Slot slot = deal(blockIdx.x, (uint32_t)(a.N * a.G), a.nblk * a.splits);
    const int64_t n = slot.head / a.G;
    const int g = slot.head - (int)n * a.G, kb = slot.w / a.splits, sp = slot.w - kb * a.splits;
    const int key0 = kb * 128 + 32 * w, key = key0 + l31;
    bool there = key < a.Sk;
    const bool masked = there && a.mask && a.mask[n * a.Sk + key] == 0;
    const float sink = masked ? a.fill : 0.f;                                    // additive mode
    if (!a.additive && masked) there = false;
    typename Ty<M>::Frag kf[KS], vf[KS];
    {   // an absent key's rows read as zero.  (What its scores then give stays in its own rows of dK and dV, which are written as zero.)
        const T* kp = static_cast<const T*>(a.k) + n * a.sk.n + (int64_t)key * a.sk.s + g * a.sk.h;
        const T* vp = static_cast<const T*>(a.v) + n * a.sv.n + (int64_t)key * a.sv.s + g * a.sv.h;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kf[ks] = As<M>::frag(load_frag<VEC>(kp + 16 * ks + 8 * h, there ? a.dh - 16 * ks - 8 * h : 0));
            vf[ks] = As<M>::frag(load_frag<VEC>(vp + 16 * ks + 8 * h, there ? a.dh - 16 * ks - 8 * h : 0));
        }
    }
    f32x16 dk[DT], dv[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) { dk[t] = zero16(); dv[t] = zero16(); }
    const float scale2 = a.scale * LOG2E;
    const int off = a.Sk - a.Sq;
    const uint64_t alive = __ballot(there);

    // the tiles of this block: per query head those from the first position that reaches the block's keys on, cut evenly over the splits
    const int tq = (a.Sq + QT - 1) / QT, t0 = a.causal ? min(tq, max(0, kb * 128 - off) / QT) : 0, per = tq - t0;
    const int64_t all = (int64_t)a.rep * per;
    const int ubeg = (int)(all * sp / a.splits);
    const int left = __syncthreads_or(there) ? (int)(all * (sp + 1) / a.splits) - ubeg : 0;      // no key of this block is there: nothing to add
    int hh = per ? ubeg / per : 0, i0 = (t0 + ubeg - hh * per) * QT;             // query head (of the key head's) and first position of the tile

    Stage<T, DHP, QT, VEC> sq, sg;
    sq.setup(tid, a.sq.s, a.dh);
    sg.setup(tid, a.sdo.s, a.dh);
    float st[3];
    auto fetch = [&](int hh, int i0, bool any) {
        const int head = g * a.rep + hh, rows = any ? a.Sq - i0 : 0;
        sq.load(static_cast<const T*>(a.q) + n * a.sq.n + i0 * a.sq.s + head * a.sq.h, rows);
        sg.load(static_cast<const T*>(a.dout) + n * a.sdo.n + i0 * a.sdo.s + head * a.sdo.h, rows);
        if (tid < QT) {
            // no row: exp(-INFINITY) whatever its scores are.  (They are not always 0: where rows share memory a tile holds more of it
            // behind the last one, and exp(score - 0) * (1 / INFINITY) was inf * 0 for fp32 scores past 88.)
            st[0] = st[1] = INFINITY; st[2] = 0.f;
            if (tid < rows) {
                const int64_t x = (n * a.H + head) * a.Sq + i0 + tid;
                st[0] = a.row_max[x];
                st[1] = a.row_sum[x];
                st[2] = a.delta[n * a.sd.n + (i0 + tid) * a.sd.s + head * a.sd.h];
            }
        }
    };
    auto put = [&](int buf) {
        sq.template store<L>(Qs + buf * L::BYTES);
        sg.template store<L>(Gs + buf * L::BYTES);
        if (tid < QT) {
            float* s = St + buf * 3 * QT + tid;
            if (NAT) { s[0] = st[0]; s[QT] = 1.f / st[1]; }
            else s[0] = st[0] + __builtin_amdgcn_logf(st[1]);
            s[2 * QT] = st[2];
        }
    };
    int buf = 0;
    if (left > 0) { fetch(hh, i0, true); put(0); }
    __syncthreads();
    for (int u = 0; u < left; ++u) {
        int hh1 = hh, i1 = i0 + QT;
        if (i1 >= a.Sq) { ++hh1; i1 = t0 * QT; }
        fetch(hh1, i1, u + 1 < left);
        const char* Qt = Qs + buf * L::BYTES;
        const char* Gt = Gs + buf * L::BYTES;
        const float* S0 = St + buf * 3 * QT;
        if (alive && !(a.causal && i0 + QT - 1 + off < key0)) {
            // not unrolled: with both halves' reads in flight the kernel ran out of registers (4001 x 128 causal: 261 us against 225)
#pragma unroll 1
            for (int s = 0; s < QSUB; ++s) {
                f32x16 x = zero16(), dp = zero16();
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    x = mul(L::near(Qt, 32 * s + l31, 16 * ks + 8 * h), kf[ks], x);
                    dp = mul(L::near(Gt, 32 * s + l31, 16 * ks + 8 * h), vf[ks], dp);
                }
                if (a.causal && i0 + 32 * s + off < key0 + 31) {                 // the diagonal: row i sees the key if i + off >= key
                    const int first = key - off - (i0 + 32 * s) - 4 * h;
#pragma unroll
                    for (int r = 0; r < 16; ++r) if (tile_row(r, 0) < first) x[r] = -INFINITY;
                }
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int rr = 32 * s + 8 * q + 4 * h;
                    const f32x4 mx = *reinterpret_cast<const f32x4*>(S0 + rr), de = *reinterpret_cast<const f32x4*>(S0 + 2 * QT + rr);
                    f32x4 rl;
                    if (NAT) rl = *reinterpret_cast<const f32x4*>(S0 + QT + rr);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * q + e;
                        float p;
                        if (NAT) {
                            float y = x[r] * a.scale;
                            if (a.additive) y += sink;
                            p = __builtin_amdgcn_exp2f((y - mx[e]) * LOG2E) * rl[e];
                        } else p = __builtin_amdgcn_exp2f(fmaf(x[r], scale2, -mx[e]));
                        float pd = p, dpd = dp[r];
                        if (DROP) {
                            const uint64_t idx = ((uint64_t)(n * a.H + g * a.rep + hh) * a.Sq + i0 + rr + e) * a.Sk + key;
                            const float f = philox_pick(philox4x32_10(a.seed, idx >> 2, a.site), (int)(idx & 3)) >= a.thr ? a.keep : 0.f;
                            pd *= f; dpd *= f;
                        }
                        x[r] = pd;
                        dp[r] = p * (dpd - de[e]);
                    }
                }
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                    const typename Ty<M>::Frag pf = tile_frag<M>(x, k2), sf = tile_frag<M>(dp, k2);
#pragma unroll
                    for (int d = 0; d < DT; ++d) {
                        dv[d] = mul(pf, L::col(Gt, 32 * s + 16 * k2, 32 * d, lane), dv[d]);
                        dk[d] = mul(sf, L::col(Qt, 32 * s + 16 * k2, 32 * d, lane), dk[d]);
                    }
                }
            }
        }
        put(buf ^ 1);
        __syncthreads();
        buf ^= 1;
        hh = hh1; i0 = i1;
    }
    const int64_t total = a.N * a.G * a.Sk;
    T* dkp = static_cast<T*>(a.dk) + n * a.sdk.n + g * a.sdk.h;
    T* dvp = static_cast<T*>(a.dv) + n * a.sdv.n + g * a.sdv.h;
    float* pk = a.part + (2 * sp * total + (n * a.G + g) * a.Sk) * a.dhs;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int row = tile_row(r, h), kk = key0 + row;
        if (kk >= a.Sk) continue;
        const bool on = (alive >> row) & 1;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int c = 32 * d + l31;
            if (c >= a.dh) continue;
            const float gk = on ? dk[d][r] * a.scale : 0.f, gv = on ? dv[d][r] : 0.f;
            if (a.splits > 1) {
                pk[(int64_t)kk * a.dhs + c] = gk;
                pk[(total + kk) * a.dhs + c] = gv;
            } else {
                dkp[kk * a.sdk.s + c] = (T)gk;
                dvp[kk * a.sdv.s + c] = (T)gv;
            }
        }
    }
}

// ---------------------------------------------------------------- dQ
template <class T, int DHP, int WK> struct DqCfg {
    static constexpr int KSUB = (sizeof(T) == 2 && WK == 1) ? 2 : 1, KT = 32 * KSUB * WK;
    typedef typename MulType<T, WK>::M M;
    typedef Lds<M, KT, DHP> L;
    static constexpr int NBUF = (sizeof(T) == 4 && DHP == 128 && WK == 4) ? 1 : 2;
    static constexpr size_t TILES = NBUF * 2 * L::BYTES;
    static constexpr size_t JOIN = WK > 1 ? (size_t)WK * DHP * 32 * 4 : 0;
    static constexpr size_t BITS = TILES > JOIN ? TILES : JOIN, RED = BITS + SPAN / 8, BYTES = RED + (WK > 1 ? WK * 32 * 4 : 0);
    static constexpr int WAVES = BYTES <= 80 * 1024 && DHP <= (sizeof(T) == 2 ? 128 : 64) ? 2 : 1;
};

// WHOLE: all keys fit one tile (kernels of their own: in the same ones the few lines cost the long case its registers, 150 -> 241 us
// for 4001 x 128 causal)
template <class T, int DHP, bool VEC, int WK, bool DROP, bool WHOLE>
__global__ __launch_bounds__(256, (DqCfg<T, DHP, WK>::WAVES)) void attn_dq_kernel(const Args a) {
    typedef DqCfg<T, DHP, WK> C;
    constexpr int WQ = 4 / WK, KSUB = C::KSUB, KT = C::KT, KS = DHP / 16, DT = DHP / 32, WORDS = (KT + 63) / 64;
    constexpr bool NAT = sizeof(T) == 4;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    typedef typename C::M M;
    typedef typename C::L L;
    char* Ks = smem;
    char* Vs = smem + C::NBUF * L::BYTES;
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6), wq = w / WK, wk = w % WK;

    const Slot slot = deal(blockIdx.x, (uint32_t)(a.N * a.G), a.nblk * a.splits);
    const int64_t n = slot.head / a.G;
    const int g = slot.head - (int)n * a.G, rb = slot.w / a.splits, sp = slot.w - rb * a.splits;
    const Rows rows = row_block(a, rb, 32 * WQ);
    const int row = rows.r0 + 32 * wq + l31;
    const bool live = row < rows.rend;
    const int hh = live ? row / a.Sq : 0, i = live ? row - hh * a.Sq : 0, head = g * a.rep + hh;
    const int lim = a.causal ? i + a.Sk - a.Sq : 0x7fffffff;
    int lim_min = live ? lim : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lim_min = min(lim_min, __shfl_xor(lim_min, o, 64));
    lim_min = __builtin_amdgcn_readfirstlane(lim_min);
    typename Ty<M>::Frag qf[KS], gf[KS];
    float de = 0.f;                              // delta of the row, from its output and gradient
    const T* op = static_cast<const T*>(a.out) + n * a.so.n + i * a.so.s + head * a.so.h;
    const T* qp = static_cast<const T*>(a.q) + n * a.sq.n + i * a.sq.s + head * a.sq.h;
    const T* gp = static_cast<const T*>(a.dout) + n * a.sdo.n + i * a.sdo.s + head * a.sdo.h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const int left = live ? a.dh - 16 * ks - 8 * h : 0;
        const auto gr = load_frag<VEC>(gp + 16 * ks + 8 * h, left), orow = load_frag<VEC>(op + 16 * ks + 8 * h, left);
        qf[ks] = As<M>::frag(load_frag<VEC>(qp + 16 * ks + 8 * h, left));
        gf[ks] = As<M>::frag(gr);
#pragma unroll
        for (int e = 0; e < 8; ++e) de = fmaf((float)orow[e], (float)gr[e], de);
    }
    de += __shfl_xor(de, 32, 64);
    // kept for the dK / dV pass if that one follows
    if (a.keep_delta && live && h == 0 && wk == 0 && sp == 0) a.delta[n * a.sd.n + i * a.sd.s + head * a.sd.h] = de;
    float m = NAT ? 0.f : INFINITY, rl = 0.f;                          // bf16: m + log2 l, no separate 1 / l
    if (live) {
        const int64_t x = (n * a.H + head) * a.Sq + i;
        m = a.row_max[x];
        rl = a.row_sum[x];
        if (NAT) rl = 1.f / rl;
        else m += __builtin_amdgcn_logf(rl);
    }
    int begin = sp * a.per_split, stop = min(a.Sk, begin + a.per_split);
    if (a.causal) {
        const int last = min(rows.r0 + 32 * WQ, rows.rend) - 1;
        const int imax = rows.r0 / a.Sq == last / a.Sq ? last % a.Sq : a.Sq - 1;
        stop = min(stop, imax + a.Sk - a.Sq + 1);
    }
    const int64_t* mask = a.mask ? a.mask + n * a.Sk : nullptr;
    const bool cut = mask && !a.additive;
    const T* kp = static_cast<const T*>(a.k) + n * a.sk.n + g * a.sk.h;
    const T* vp = static_cast<const T*>(a.v) + n * a.sv.n + g * a.sv.h;
    const float scale2 = a.scale * LOG2E;
    f32x16 dq[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) dq[t] = zero16();

    Stage<T, DHP, KT, VEC> sk, sv;
    sk.setup(tid, a.sk.s, a.dh);
    sv.setup(tid, a.sv.s, a.dh);
    KeyBits kb;
    kb.words = reinterpret_cast<uint64_t*>(smem + C::BITS);
    kb.masked = mask != nullptr;
    int end = stop;
    const T *kn = nullptr, *vn = nullptr;        // the next tile
    const int64_t kstep = KT * a.sk.s, vstep = KT * a.sv.s;
    auto fetch = [&](int left) {                 // (none left: zeros, no memory is read)
        sk.load(kn, left);
        sv.load(vn, left);
        kn += kstep;
        vn += vstep;
    };
    for (; begin < stop; begin += SPAN) {        // (one turn without a mask)
        end = stop;
        kn = kp + begin * a.sk.s;
        vn = vp + begin * a.sv.s;
        fetch(end - begin);                      // on its way while the key bits are read
        kb.from = begin;
        kb.end = stop;
        if (mask) {
            kb.end = end = min(stop, begin + SPAN);
            const int there = kb.fill(mask, lane, w);
            if (cut) kb.end = end = there;
        }
        auto put = [&](int buf, int j) {
            uint64_t bits[WORDS];
            bool all = true;
#pragma unroll
            for (int x = 0; x < WORDS; ++x) {
                bits[x] = cut ? kb.at(j + 64 * x) : ~0ull;
                all = all && (KT < 64 ? (uint32_t)bits[x] == ~0u : bits[x] == ~0ull);
            }
            if (all) {
                sk.template store<L>(Ks + buf * L::BYTES);
                sv.template store<L>(Vs + buf * L::BYTES);
            } else {
                auto keep = [&](int r) { return (bits[WORDS > 1 ? r >> 6 : 0] >> (r & 63)) & 1; };
                sk.template store_if<L>(Ks + buf * L::BYTES, keep);
                sv.template store_if<L>(Vs + buf * L::BYTES, keep);
            }
        };
        const int tiles = (end - begin + KT - 1) / KT;
        if (tiles > 0) put(0, begin);
        __syncthreads();
        // the scores and dP of 32 keys; false if none of them is there
        auto scores = [&](const char* Kt, const char* Vt, int j0, uint64_t mine, int s, f32x16& x, f32x16& dp) {
            const int ko = 32 * (wk * KSUB + s), kw = j0 + ko;
            uint32_t sub = (uint32_t)(mine >> (32 * s));
            if (!sub && !(a.additive && kw < end)) return false;
            x = zero16(); dp = zero16();
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                x = mul(L::near(Kt, ko + l31, 16 * ks + 8 * h), qf[ks], x);
                dp = mul(L::near(Vt, ko + l31, 16 * ks + 8 * h), gf[ks], dp);
            }
            if (NAT) {
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= a.scale;
                if (a.additive) {
#pragma unroll
                    for (int r = 0; r < 16; ++r) if (!((sub >> tile_row(r, h)) & 1)) x[r] += a.fill;
                    sub = (uint32_t)kb.range(kw);
                }
            }
            if (sub != ~0u || kw + 31 > lim_min) hide(x, sub, kw, lim, lim_min, h);
            return true;
        };
        if (WHOLE && tiles > 0) {
            // all of the row's keys are in this tile: delta = sum_j P dP, without the stored output's rounding.  (Among few keys dP and
            // delta are near each other: with 2 keys the bf16 output's rounding alone put dQ off by 4.4e-3 of its norm, 1.9e-3 so.)
            float sum = 0.f;
#pragma unroll 1
            for (int s = 0; s < KSUB; ++s) {
                f32x16 x, dp;
                if (!scores(Ks, Vs, begin, kb.at(begin + 32 * wk * KSUB), s, x, dp)) continue;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t kp4 = 0xf;
                    if (DROP) kp4 = keep4(a, ((uint64_t)(n * a.H + head) * a.Sq + i) * a.Sk + begin + 32 * (wk * KSUB + s) + 8 * q + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (!DROP || ((kp4 >> e) & 1)) sum = fmaf(__builtin_amdgcn_exp2f(fmaf(x[4 * q + e], scale2, -m)), DROP ? dp[4 * q + e] * a.keep : dp[4 * q + e], sum);
                }
            }
            sum += __shfl_xor(sum, 32, 64);
            if (WK > 1) {
                float* red = reinterpret_cast<float*>(smem + C::RED);
                if (h == 0) red[wk * 32 + l31] = sum;
                __syncthreads();
                sum = 0.f;
#pragma unroll
                for (int y = 0; y < WK; ++y) sum += red[y * 32 + l31];
            }
            de = sum;
            if (a.keep_delta && live && h == 0 && wk == 0) a.delta[n * a.sd.n + i * a.sd.s + head * a.sd.h] = de;
        }
        for (int t = 0; t < tiles; ++t) {
            const int j0 = begin + t * KT, buf = C::NBUF == 2 ? (t & 1) : 0;
            fetch(end - j0 - KT);
            const char* Kt = Ks + buf * L::BYTES;
            const char* Vt = Vs + buf * L::BYTES;
            const uint64_t mine = kb.at(j0 + 32 * wk * KSUB);
#pragma unroll
            for (int s = 0; s < KSUB; ++s) {
                const int ko = 32 * (wk * KSUB + s), kw = j0 + ko;
                f32x16 x, dp;
                if (!scores(Kt, Vt, j0, mine, s, x, dp)) continue;
                const uint64_t rlin = ((uint64_t)(n * a.H + head) * a.Sq + i) * a.Sk;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint32_t kp4 = 0;
                    if (DROP) kp4 = keep4(a, rlin + kw + 8 * q + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int r = 4 * q + e;
                        const float p = NAT ? __builtin_amdgcn_exp2f((x[r] - m) * LOG2E) * rl : __builtin_amdgcn_exp2f(fmaf(x[r], scale2, -m));
                        const float g1 = DROP ? (((kp4 >> e) & 1) ? dp[r] * a.keep : 0.f) : dp[r];
                        dp[r] = p * (g1 - de);
                    }
                }
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) {
                    const typename Ty<M>::Frag sf = tile_frag<M>(dp, k2);
#pragma unroll
                    for (int d = 0; d < DT; ++d) dq[d] = mul(L::col(Kt, ko + 16 * k2, 32 * d, lane), sf, dq[d]);
                }
            }
            if (C::NBUF == 1) __syncthreads();
            put(C::NBUF == 2 ? 1 - buf : 0, j0 + KT);
            __syncthreads();
        }
        if (!mask) break;
    }
    if (WK > 1) {
        float* slab = reinterpret_cast<float*>(smem);                            // [WK][DHP][32]
        __syncthreads();
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
    const int64_t rt = (n * a.G + g) * a.R + row, total = a.N * a.G * a.R;
    T* dp = static_cast<T*>(a.dq) + n * a.sdq.n + i * a.sdq.s + head * a.sdq.h;
    float* pr = a.part + (sp * total + rt) * a.dhs;
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

// ---------------------------------------------------------------- launches
template <class T, int DHP, bool VEC, bool DROP>
static int launch_dkv(const Args& a, unsigned grid, hipStream_t s) {
    constexpr size_t bytes = DkvCfg<T, DHP>::BYTES;
    if (bytes > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_dkv_kernel<T, DHP, VEC, DROP>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    hipLaunchKernelGGL((attn_dkv_kernel<T, DHP, VEC, DROP>), dim3(grid), dim3(256), bytes, s, a);
    return check_launch("attention_bwd dk/dv");
}
template <class T, int DHP, bool VEC, int WK, bool DROP>
static int launch_dq(const Args& a, unsigned grid, hipStream_t s) {
    typedef DqCfg<T, DHP, WK> C;
    auto go = [&](auto kernel) {
        if (C::BYTES > 64 * 1024) (void)hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)C::BYTES);
        hipLaunchKernelGGL(kernel, dim3(grid), dim3(256), C::BYTES, s, a);
        return check_launch("attention_bwd dq");
    };
    if constexpr (sizeof(T) == 2)                // (fp32: the output's rounding does not matter)
        if (a.splits == 1 && a.Sk <= C::KT) return go(&attn_dq_kernel<T, DHP, VEC, WK, DROP, true>);
    return go(&attn_dq_kernel<T, DHP, VEC, WK, DROP, false>);
}
template <class T, bool VEC, bool DROP> static int pick_dkv(const Args& a, unsigned grid, hipStream_t s) {
    if (a.dh <= 32) return launch_dkv<T, 32, VEC, DROP>(a, grid, s);
    if (a.dh <= 64) return launch_dkv<T, 64, VEC, DROP>(a, grid, s);
    return launch_dkv<T, 128, VEC, DROP>(a, grid, s);
}
template <class T, bool VEC, int WK, bool DROP> static int pick_dq(const Args& a, unsigned grid, hipStream_t s) {
    if (a.dh <= 32) return launch_dq<T, 32, VEC, WK, DROP>(a, grid, s);
    if (a.dh <= 64) return launch_dq<T, 64, VEC, WK, DROP>(a, grid, s);
    return launch_dq<T, 128, VEC, WK, DROP>(a, grid, s);
}
template <class T> static int run_sum(const Args& a, int which, hipStream_t s) {
    if (a.splits == 1) return NR_OK;
    const int64_t threads = a.N * a.G * (int64_t)(which ? 2 * (int64_t)a.Sk : a.R) * (a.dhs / 4);
    hipLaunchKernelGGL((attn_sum_kernel<T>), dim3((unsigned)((threads + 255) / 256)), dim3(256), 0, s, a, which);
    return check_launch("attention_bwd sum");
}
template <class T, bool DROP>
static int passes(Args a, const BwdPlan& f, bool vec, bool room, hipStream_t s) {
    auto keys = [&]() {
        Args b = a;
        b.nblk = f.nblk_k; b.splits = room ? f.kv.splits : 1;
        const unsigned grid = (unsigned)(b.N * b.G * (int64_t)b.nblk * b.splits);
        if (int rc = vec ? pick_dkv<T, true, DROP>(b, grid, s) : pick_dkv<T, false, DROP>(b, grid, s)) return rc;
        return run_sum<T>(b, 1, s);
    };
    auto rows = [&]() {
        Args b = a;
        b.nblk = f.nblk_q; b.head_blocks = f.head_blocks; b.splits = room ? f.q.splits : 1; b.per_split = room ? f.q.per : a.Sk;
        const unsigned grid = (unsigned)(b.N * b.G * (int64_t)b.nblk * b.splits);
        const int rc = f.wk == 4 ? (vec ? pick_dq<T, true, 4, DROP>(b, grid, s) : pick_dq<T, false, 4, DROP>(b, grid, s))
                                 : (vec ? pick_dq<T, true, 1, DROP>(b, grid, s) : pick_dq<T, false, 1, DROP>(b, grid, s));
        return rc != NR_OK ? rc : run_sum<T>(b, 0, s);
    };
    if (a.keep_delta) {
        const int rc = rows();
        return rc != NR_OK ? rc : keys();
    }
    const int rc = keys();
    return rc != NR_OK ? rc : rows();
}
template <class T>
int run_bwd(Args a, const BwdPlan& f, bool vec, bool drop, bool room, hipStream_t s) {
    if (!a.keep_delta) {
        const int64_t rows = a.N * a.Sq * a.H;
        hipLaunchKernelGGL((attn_delta_kernel<T>), dim3((unsigned)((rows * 16 + 255) / 256)), dim3(256), 0, s, a);
        if (int rc = check_launch("attention_bwd delta")) return rc;
    }
    return drop ? passes<T, true>(a, f, vec, room, s) : passes<T, false>(a, f, vec, room, s);
}

}  // namespace al
}  // namespace nr

// Softmax attention of any length: forward kernels (instantiated by attention_long_fwd_{f32,bf16}.hip).
//
//   o_i = sum_j p_ij v_j,   p_ij = exp(x_ij - max_j x_ij) / sum_j exp(..),   x_ij = scale * q_i . k_j
//
// over the keys j that are there (key mask) and, causal, not behind the query (j <= i + Sk - Sq).  One pass over the keys with
// the running maximum m and sum l of every row: a new tile's maximum m' rescales what was summed so far by exp(m - m').
//
// Tiling.  A workgroup of four waves takes 128 rows of one key head and walks the keys in tiles staged through LDS; a wave owns
// 32 rows.  The query heads that share a key head are laid one below the other (row r = query head r / Sq, position r % Sq), so
// K and V are read once for all of them.  A wave forms S^T = K Q^T (row = key, column = query): a lane then holds 16 scores of
// ONE row per 32 keys, the softmax needs one exchange (the other lane half), and the probabilities are, register by register, the
// B operand of O^T += V^T P^T (mma.h, "tile" order) - they never pass through LDS.
// With at most 32 rows (a few candidates over a long history) the four waves take a quarter of every tile's keys each instead
// (WK = 4) and meet at the end through LDS; when the workgroups do not fill the chip the keys are also split over workgroups
// and joined by attn_join_kernel.
//
// Rounding: scores, maximum, sum and output are fp32; bf16 inputs round the probabilities to bf16 (the matrix instruction's
// operand), half a step each, against a sum taken in fp32 from the unrounded ones.
//
// Measured (MI355X).  Long rows are bound by issue: per 64 keys and 32 rows a wave has 2 * 64 * 32 * 2 * dh operations for the matrix
// pipe beside 2048 exponentials with their maximum and sum on the vector pipe.  8192 x 8192 causal, 16 heads (4 of them with keys) of
// 128, bf16: 309 - 323 us a pass by card, 850 - 890 TFLOP/s, where a large matrix product of the library reaches 1363 (a launch on its
// own under the profiler, at a lower clock: 352 - 372); heads of 64 without causal order: 700 TFLOP/s (the exponentials weigh twice as
// much); fp32, 4096 x 64: 185 TFLOP/s (105 on the fp32 matrix instruction).  Short ones are bound by the latency of a block's few tiles
// and the last round of workgroups: 32 x 512 ragged, 12 heads of 64, bf16: 36 - 37 us a pass (39.5 - 42 on its own), 2.8 TB/s and 430
// TFLOP/s; 32 fp32 histories of 200, 12 heads of 25: 24 us (25.5 - 27).  5 rows over 20011 keys in splits: 19 us + 4 for the join, 4.3
// TB/s of keys.  Dropout of 0.1: 16 x 512 ragged, 12 heads of 64, bf16: 24 -> 67 us, 85 where Sk is no multiple of 4 (keep4 then calls
// the generator twice); the fp32 histories 27 -> 53: the generator takes the difference.
//
// Registers that do not fit and go to scratch memory: 128 columns in fp32 with few rows and unaligned addresses 158 per lane; 128 columns
// in bf16, unaligned, 7 (45 with dropout).  The others hold all of theirs.
#pragma once
#include "attention_long_dev.h"

namespace nr {
namespace al {

template <class T, int DHP, int WK> struct FwdCfg {
    static constexpr int KSUB = (sizeof(T) == 2 && WK == 1) ? 2 : 1;     // 32-key pieces of a tile per wave
    static constexpr int KT = 32 * KSUB * WK;
    typedef typename MulType<T, WK>::M M;
    typedef Lds<M, KT, DHP> L;
    static constexpr int NBUF = (sizeof(T) == 4 && DHP == 128 && WK == 4) ? 1 : 2;       // two stages where 160 KB hold them
    static constexpr size_t TILES = NBUF * 2 * L::BYTES;
    static constexpr size_t JOIN = WK > 1 ? (size_t)(WK * DHP * 32 + 2 * WK * 32) * 4 : 0;
    static constexpr size_t BITS = TILES > JOIN ? TILES : JOIN;          // offset of the key bits
    static constexpr size_t BYTES = BITS + SPAN / 8;
    static constexpr int WAVES = BYTES <= 80 * 1024 ? 2 : 1;             // per SIMD: registers for two where the LDS holds two
};

template <class T, int DHP, bool VEC, int WK, bool DROP>
__global__ __launch_bounds__(256, (FwdCfg<T, DHP, WK>::WAVES)) void attn_fwd_kernel(const Args a) {
    typedef FwdCfg<T, DHP, WK> C;
    constexpr int WQ = 4 / WK, KSUB = C::KSUB, KT = C::KT, KS = DHP / 16, DT = DHP / 32, WORDS = (KT + 63) / 64;
    constexpr bool NAT = sizeof(T) == 4;         // fp32: exp(x - m) with the difference formed first (the mask's -1e5 would cost
                                                 // a product's rounding); bf16: one fma per score in units of log 2
    // the maximum may lag behind by this much before the sums are rescaled (bf16: probabilities up to 2^8, no precision is lost
    // in a floating format; the rescaling of every row's sums becomes rare)
    constexpr float SLACK = NAT ? 0.f : 8.f;
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

    // this lane's row
    const int row = rows.r0 + 32 * wq + l31;
    const bool live = row < rows.rend;
    const int hh = live ? row / a.Sq : 0, i = live ? row - hh * a.Sq : 0, head = g * a.rep + hh;
    const int lim = a.causal ? i + a.Sk - a.Sq : 0x7fffffff;             // last key of the row
    int lim_min = live ? lim : 0x7fffffff;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) lim_min = min(lim_min, __shfl_xor(lim_min, o, 64));
    lim_min = __builtin_amdgcn_readfirstlane(lim_min);
    typename Ty<M>::Frag qf[KS];
    const T* qp = static_cast<const T*>(a.q) + n * a.sq.n + i * a.sq.s + head * a.sq.h;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) qf[ks] = As<M>::frag(load_frag<VEC>(qp + 16 * ks + 8 * h, live ? a.dh - 16 * ks - 8 * h : 0));

    // keys of this block
    int begin = sp * a.per_split, stop = min(a.Sk, begin + a.per_split);
    if (a.causal) {
        const int last = min(rows.r0 + 32 * WQ, rows.rend) - 1;
        const int imax = rows.r0 / a.Sq == last / a.Sq ? last % a.Sq : a.Sq - 1;
        stop = min(stop, imax + a.Sk - a.Sq + 1);
    }
    const int64_t* mask = a.mask ? a.mask + n * a.Sk : nullptr;
    const bool cut = mask && !a.additive;        // keys that are not there need not be read
    const T* kp = static_cast<const T*>(a.k) + n * a.sk.n + g * a.sk.h;
    const T* vp = static_cast<const T*>(a.v) + n * a.sv.n + g * a.sv.h;

    const float scale2 = a.scale * LOG2E;
    float m = NEVER, l = 0.f;
    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t) o[t] = zero16();

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
            // an absent key's row reads as zero: whatever its memory holds (a NaN as well) must not reach 0 * v
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
        for (int t = 0; t < tiles; ++t) {
            const int j0 = begin + t * KT, buf = C::NBUF == 2 ? (t & 1) : 0;
            fetch(end - j0 - KT);
            const char* Kt = Ks + buf * L::BYTES;
            const char* Vt = Vs + buf * L::BYTES;
            const int kw = j0 + 32 * wk * KSUB;                          // first key of this wave's piece
            const uint64_t mine = kb.at(kw);
            uint32_t sub[KSUB], any = 0, all = ~0u;
#pragma unroll
            for (int s = 0; s < KSUB; ++s) {
                sub[s] = (uint32_t)(mine >> (32 * s));
                any |= sub[s]; all &= sub[s];
            }
            if (any || (a.additive && kw < end)) {
                f32x16 x[KSUB];
#pragma unroll
                for (int s = 0; s < KSUB; ++s) {
                    x[s] = zero16();
#pragma unroll
                    for (int ks = 0; ks < KS; ++ks) x[s] = mul(L::near(Kt, 32 * (wk * KSUB + s) + l31, 16 * ks + 8 * h), qf[ks], x[s]);
                }
                if (NAT) {
#pragma unroll
                    for (int s = 0; s < KSUB; ++s) {
#pragma unroll
                        for (int r = 0; r < 16; ++r) x[s][r] *= a.scale;
                        if (a.additive) {                                // absent keys sink by `fill`; past the end there is no key
#pragma unroll
                            for (int r = 0; r < 16; ++r) if (!((sub[s] >> tile_row(r, h)) & 1)) x[s][r] += a.fill;
                            sub[s] = (uint32_t)kb.range(kw + 32 * s);
                            all = s ? all & sub[s] : sub[s];
                        }
                    }
                }
                if (all != ~0u || kw + 32 * KSUB - 1 > lim_min)
#pragma unroll
                    for (int s = 0; s < KSUB; ++s) hide(x[s], sub[s], kw + 32 * s, lim, lim_min, h);
                float top = x[0][0];
#pragma unroll
                for (int s = 0; s < KSUB; ++s)
#pragma unroll
                    for (int r = 0; r < 16; ++r) top = fmaxf(top, x[s][r]);
                top = fmaxf(top, __shfl_xor(top, 32, 64));
                const float mn = NAT ? top : top * scale2;
                if (__any(mn > m + SLACK)) {
                    const float to = fmaxf(m, mn), f = __builtin_amdgcn_exp2f(NAT ? (m - to) * LOG2E : m - to);
                    l *= f;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int r = 0; r < 16; ++r) o[d][r] *= f;
                    m = to;
                }
                float sum = 0.f;
#pragma unroll
                for (int s = 0; s < KSUB; ++s)
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        x[s][r] = __builtin_amdgcn_exp2f(NAT ? (x[s][r] - m) * LOG2E : fmaf(x[s][r], scale2, -m));
                        sum += x[s][r];
                    }
                l += sum;
                if (DROP) {
                    const uint64_t rl = ((uint64_t)(n * a.H + head) * a.Sq + i) * a.Sk;
#pragma unroll
                    for (int s = 0; s < KSUB; ++s)
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t kp4 = keep4(a, rl + kw + 32 * s + 8 * q + 4 * h);
#pragma unroll
                            for (int e = 0; e < 4; ++e) x[s][4 * q + e] *= ((kp4 >> e) & 1) ? a.keep : 0.f;
                        }
                }
#pragma unroll
                for (int s = 0; s < KSUB; ++s)
#pragma unroll
                    for (int k2 = 0; k2 < 2; ++k2) {
                        const typename Ty<M>::Frag pf = tile_frag<M>(x[s], k2);
#pragma unroll
                        for (int d = 0; d < DT; ++d)
                            o[d] = mul(L::col(Vt, 32 * (wk * KSUB + s) + 16 * k2, 32 * d, lane), pf, o[d]);
                    }
            }
            if (C::NBUF == 1) __syncthreads();
            put(C::NBUF == 2 ? 1 - buf : 0, j0 + KT);
            __syncthreads();
        }
        if (!mask) break;
    }
    l += __shfl_xor(l, 32, 64);

    if (WK > 1) {                                // the waves' quarters of the keys meet (in wave order: the same result every time)
        float* slab = reinterpret_cast<float*>(smem);                    // [WK][DHP][32]
        float* ml = slab + WK * DHP * 32;                                // [2][WK][32]
        __syncthreads();
        if (h == 0) { ml[wk * 32 + l31] = m; ml[(WK + wk) * 32 + l31] = l; }
        __syncthreads();
        float M = NEVER;
#pragma unroll
        for (int x = 0; x < WK; ++x) M = fmaxf(M, ml[x * 32 + l31]);
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < WK; ++x)
            sum += ml[(WK + x) * 32 + l31] * __builtin_amdgcn_exp2f(NAT ? (ml[x * 32 + l31] - M) * LOG2E : ml[x * 32 + l31] - M);
        const float f = __builtin_amdgcn_exp2f(NAT ? (m - M) * LOG2E : m - M);
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) slab[(wk * DHP + 32 * d + tile_row(r, h)) * 32 + l31] = o[d][r] * f;
        __syncthreads();
        m = M; l = sum;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q)
                if (q == wk % 4) {               // wave wk finishes registers 4 wk .. 4 wk + 3 of every tile
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float t = 0.f;
#pragma unroll
                        for (int x = 0; x < WK; ++x) t += slab[(x * DHP + 32 * d + tile_row(4 * q + e, h)) * 32 + l31];
                        o[d][4 * q + e] = t;
                    }
                }
    }
    if (!live) return;
    auto mine = [&](int q) { return WK == 1 || q == wk; };
    if (a.splits > 1) {
        const int64_t rt = (n * a.G + g) * a.R + row, total = a.N * a.G * a.R;
        float* pr = a.part + (sp * total + rt) * a.dhs;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int c = 32 * d + 8 * q + 4 * h;
                if (mine(q)) store4<true>(pr + c, f32x4{o[d][4 * q], o[d][4 * q + 1], o[d][4 * q + 2], o[d][4 * q + 3]}, a.dhs - c);
            }
        if (h == 0 && wk == 0) { a.part_ml[2 * (sp * total + rt)] = m; a.part_ml[2 * (sp * total + rt) + 1] = l; }
        return;
    }
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);          // no key: a zero row (and a NaN stays one)
    T* op = static_cast<T*>(a.out) + n * a.so.n + i * a.so.s + head * a.so.h;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int c = 32 * d + 8 * q + 4 * h;
            if (mine(q)) store4<VEC>(op + c, f32x4{o[d][4 * q] * inv, o[d][4 * q + 1] * inv, o[d][4 * q + 2] * inv, o[d][4 * q + 3] * inv}, a.dh - c);
        }
    if (a.row_max && h == 0 && wk == 0) {
        const int64_t x = (n * a.H + head) * a.Sq + i;
        a.row_max[x] = l == 0.f ? 0.f : m;
        a.row_sum[x] = l == 0.f ? 1.f : l;
    }
}

// joins the splits of a row: four output columns per item.  With few items (few rows, so many splits) GROUPS threads share one, each
// with every GROUPS-th split, and meet through LDS in a fixed order: 240 rows of 64 in 32 splits took 12 us with one thread each.
template <class T, int GROUPS>
__global__ __launch_bounds__(256) void attn_join_kernel(const Args a) {
    constexpr bool NAT = sizeof(T) == 4;
    constexpr int ITEMS = 256 / GROUPS;
    __shared__ float sm[GROUPS][ITEMS], sl[GROUPS][ITEMS];
    __shared__ f32x4 so[GROUPS][ITEMS];
    const int quads = a.dhs / 4, item = threadIdx.x % ITEMS, grp = threadIdx.x / ITEMS;
    const int64_t idx = (int64_t)blockIdx.x * ITEMS + item, rows = a.N * a.G * a.R;
    const bool live = idx < rows * quads;
    const int64_t rt = live ? idx / quads : 0;
    const int c = (int)(idx - rt * quads) * 4, splits = live ? a.splits : 0;
    auto pw = [](float x) { return __builtin_amdgcn_exp2f(NAT ? x * LOG2E : x); };
    float M = NEVER;
#pragma unroll 4
    for (int s = grp; s < splits; s += GROUPS) M = fmaxf(M, a.part_ml[2 * (s * rows + rt)]);
    float l = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = grp; s < splits; s += GROUPS) {
        const float f = pw(a.part_ml[2 * (s * rows + rt)] - M);
        l = fmaf(a.part_ml[2 * (s * rows + rt) + 1], f, l);
        const f32x4 x = *reinterpret_cast<const f32x4*>(a.part + (s * rows + rt) * a.dhs + c);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = fmaf(x[e], f, o[e]);
    }
    if (GROUPS > 1) {
        sm[grp][item] = M; sl[grp][item] = l; so[grp][item] = o;
        __syncthreads();
        if (grp) return;
        for (int g = 1; g < GROUPS; ++g) M = fmaxf(M, sm[g][item]);
        l = 0.f; o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int g = 0; g < GROUPS; ++g) {
            const float f = pw(sm[g][item] - M);
            l = fmaf(sl[g][item], f, l);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[e] = fmaf(so[g][item][e], f, o[e]);
        }
    }
    if (!live) return;
    const int64_t ng = rt / a.R;
    const int row = (int)(rt - ng * a.R), hh = row / a.Sq, i = row - hh * a.Sq;
    const int64_t n = ng / a.G, head = (ng - n * a.G) * a.rep + hh;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] *= inv;
    store4<false>(static_cast<T*>(a.out) + n * a.so.n + i * a.so.s + head * a.so.h + c, o, a.dh - c);
    if (a.row_max && c == 0) {
        const int64_t x = (n * a.H + head) * a.Sq + i;
        a.row_max[x] = l == 0.f ? 0.f : M;
        a.row_sum[x] = l == 0.f ? 1.f : l;
    }
}

// ---------------------------------------------------------------- launches
template <class T, int DHP, bool VEC, int WK, bool DROP>
static int launch_fwd(const Args& a, unsigned grid, hipStream_t s) {
    constexpr size_t bytes = FwdCfg<T, DHP, WK>::BYTES;
    if (bytes > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&attn_fwd_kernel<T, DHP, VEC, WK, DROP>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    hipLaunchKernelGGL((attn_fwd_kernel<T, DHP, VEC, WK, DROP>), dim3(grid), dim3(256), bytes, s, a);
    return check_launch("attention_fwd");
}
template <class T, bool VEC, int WK, bool DROP>
static int pick_fwd(const Args& a, unsigned grid, hipStream_t s) {
    if (a.dh <= 32) return launch_fwd<T, 32, VEC, WK, DROP>(a, grid, s);
    if (a.dh <= 64) return launch_fwd<T, 64, VEC, WK, DROP>(a, grid, s);
    return launch_fwd<T, 128, VEC, WK, DROP>(a, grid, s);
}
template <class T, bool DROP>
static int pick_fwd(const Args& a, bool vec, int wk, unsigned grid, hipStream_t s) {
    return wk == 4 ? (vec ? pick_fwd<T, true, 4, DROP>(a, grid, s) : pick_fwd<T, false, 4, DROP>(a, grid, s))
                   : (vec ? pick_fwd<T, true, 1, DROP>(a, grid, s) : pick_fwd<T, false, 1, DROP>(a, grid, s));
}
template <class T>
int run_fwd(const Args& a, bool vec, bool drop, int wk, unsigned grid, hipStream_t s) {
    int rc = drop ? pick_fwd<T, true>(a, vec, wk, grid, s) : pick_fwd<T, false>(a, vec, wk, grid, s);
    if (rc != NR_OK || a.splits == 1) return rc;
    const int64_t items = a.N * a.G * a.R * (a.dhs / 4);
    if (items <= 16384) hipLaunchKernelGGL((attn_join_kernel<T, 16>), dim3((unsigned)((items + 15) / 16)), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((attn_join_kernel<T, 1>), dim3((unsigned)((items + 255) / 256)), dim3(256), 0, s, a);
    return check_launch("attention_fwd join");
}

}  // namespace al
}  // namespace nr

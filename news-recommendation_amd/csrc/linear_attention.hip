// Linear attention with a decay for each head, chunked.
//
//   S_t = w S_{t-1} + k_t v_t^T,  o_t = scale * q_t S_t   (w = e^{log_decay[h]}, S_t [dk,dv])
//
// A chunk of 64 tokens that starts from state S gives, with i, j positions in the chunk and m its token count,
//   o_i = scale * ( sum_{j <= i} w^{i-j} (q_i . k_j) v_j  +  w^{i+1} q_i S ),     S' = w^m S + sum_i w^{m-1-i} k_i v_i^T
// so everything is a matrix product; the powers are of exponents >= 0 (no overflow however fast a head forgets).
//
// The backward is the same form three times over: with g = dO,
//   dq_t = scale * sum_{s <= t} w^{t-s} (g_t . v_s) k_s           = the forward of (g, v, k), starting from S_0^T
//   dk_s = sum_{t >= s} w^{t-s} scale (v_s . g_t) q_t             = from the other end, (v, g, q), starting from dS_last^T
//   dv_s = sum_{t >= s} w^{t-s} scale (k_s . q_t) g_t             = from the other end, (k, q, g), starting from dS_last; it ends in dS_0
// From the other end (rev) the carried state R already holds the step to the next token: o_i = sum_{j >= i} w^{j-i} (..) + w^{m-1-i} x_i R,
// R' = w^m R + sum_i w^{i+1} y_i z_i^T.  One kernel computes o = form(x, y, z) for all of them; the three of a backward are one launch,
// neighbours on one XCD, so that what they read twice comes from its L2.
//
// Work split.  A wave owns 32 columns of z / o and of the state, which stays in its registers in fp32 (rows a, column b: a D tile,
// mma.h) for the whole walk; a workgroup has one wave per 32 columns.  Registers feed both products of the state: as D tiles they
// are the A operand of o^T += S^T x^T without a transpose, and the z fragments are the A operand of o^T += z^T A^T and the B
// operand of S += y^T z.  When heads * sequences do not fill the chip the tokens are also cut into segments: every segment's own
// sum first (lin_state), a scan over them (lin_scan), then the walk with the right starting states.
//
// Rounding (bf16): the decayed scores, and the state where a query meets it, are rounded to bf16 as operands of a product (half a
// step each, against an output of the same type); what goes INTO the state is not (Weighed), and every sum, and the state from chunk
// to chunk, is fp32.
#include "linear_attention.h"
#include "attention_long_dev.h"
#include <algorithm>

namespace nr {
namespace lin {

using namespace mma;

constexpr int C = 64;                            // tokens per chunk

struct Job {
    const void *x, *y, *z;
    AttnStrides sx, sy, sz, so;
    void* o;
    const float* init; int init_t;               // starting state [da,db] (init_t: stored [db,da]), NULL: zero
    float* last;                                 // final state [da,db], NULL: not wanted
    float* seg;                                  // [N*H][G][da*db]: segment sums, then starting states
    int da, db, rev;
    float amul, imul, umul;                      // factors of the scores, of the state's product, of what is added to the state
};
struct Args {
    Job job[3];
    int jobs, G, per;                            // segments of `per` tokens (a multiple of C)
    int64_t N;
    int S, H;
    const float* log_decay;
    const int64_t* lens;
};

__device__ __forceinline__ float power(float a2, int n) { return n == 0 ? 1.f : __builtin_amdgcn_exp2f(a2 * (float)n); }
__device__ __forceinline__ int length_of(const Args& a, int64_t n) {
    if (!a.lens) return a.S;
    const int64_t l = a.lens[n];
    return (int)(l < 0 ? 0 : (l > a.S ? a.S : l));
}
// 8 elements of a row in "tile" order: p points at column 16 * kstep + 4 * h
__device__ __forceinline__ bf16x8 spread_frag(const __bf16* p) {
    const bf16x4 a = *reinterpret_cast<const bf16x4*>(p), b = *reinterpret_cast<const bf16x4*>(p + 8);
    return bf16x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
__device__ __forceinline__ f32x8 spread_frag(const float* p) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 8);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}
// what a chunk adds to the state: S += y^T (w z), k-step kb of it.  bf16: w z goes in as the sum of three bf16 numbers, its fp32
// value to the last bit but one: the state is an fp32 result and carries on for the whole sequence (with two of them the state of
// 1000 tokens was off by 2.5e-6 of its norm, with one by 2.8e-3, against 4e-7 in fp32 throughout)
template <class T> struct Weighed;
template <> struct Weighed<float> {
    f32x8 v;
    __device__ __forceinline__ Weighed(const f32x8& z, const float* w, int h) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(w + 4 * h), b = *reinterpret_cast<const f32x4*>(w + 8 + 4 * h);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = z[e] * a[e]; v[4 + e] = z[4 + e] * b[e]; }
    }
    __device__ __forceinline__ f32x16 add(const f32x8& y, const f32x16& s) const { return mul(y, v, s); }
};
template <> struct Weighed<__bf16> {
    bf16x8 hi, mid, lo;
    __device__ __forceinline__ Weighed(const bf16x8& z, const float* w, int h) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(w + 4 * h), b = *reinterpret_cast<const f32x4*>(w + 8 + 4 * h);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = (float)z[e] * (e < 4 ? a[e & 3] : b[e & 3]);
            hi[e] = (__bf16)x;
            const float y = x - (float)hi[e];
            mid[e] = (__bf16)y;
            lo[e] = (__bf16)(y - (float)mid[e]);
        }
    }
    __device__ __forceinline__ f32x16 add(const bf16x8& y, const f32x16& s) const { return mul(y, hi, mul(y, mid, mul(y, lo, s))); }
};

// where a workgroup stands: job, head, segment
struct Place {
    int job, seg, h, s0, s1, send, nc;
    int64_t n, nh;
    float a2;
    __device__ __forceinline__ Place(const Args& a) {
        const al::Slot slot = al::deal(blockIdx.x, (uint32_t)(a.N * a.H), a.G * a.jobs);
        nh = slot.head;
        seg = slot.w / a.jobs;
        job = slot.w - seg * a.jobs;
        n = nh / a.H;
        h = (int)(nh - n * a.H);
        a2 = a.log_decay[h] * al::LOG2E;
        s0 = seg * a.per;
        send = min(a.S, s0 + a.per);
        s1 = max(s0, min(length_of(a, n), send));
        nc = (s1 - s0 + C - 1) / C;
    }
};

// the weights of what a chunk of m tokens adds to the state, times umul: w^{m-1-i}, from the other end w^{i+1}; zero behind m
__device__ __forceinline__ float add_weight(float a2, int i, int m, int rev, float umul) {
    return i < m ? umul * power(a2, rev ? i + 1 : m - 1 - i) : 0.f;
}

template <class T, int DA, int DB, bool VEC>
__global__ __launch_bounds__(2 * DB) void lin_state_kernel(const Args a) {
    constexpr int NT = 2 * DB, PA = DA + Ty<T>::PAD, PB = DB + Ty<T>::PAD, AT = DA / 32;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* Ys = reinterpret_cast<T*>(smem);
    T* Zs = Ys + C * PA;
    float* wu = reinterpret_cast<float*>(Zs + C * PB);
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at(a);
    const Job& J = a.job[at.job];
    const T* yp = static_cast<const T*>(J.y) + at.n * J.sy.n + at.h * J.sy.h;
    const T* zp = static_cast<const T*>(J.z) + at.n * J.sz.n + at.h * J.sz.h;
    f32x16 S[AT];
#pragma unroll
    for (int t = 0; t < AT; ++t) S[t] = zero16();
    al::Stage<T, DA, C, VEC, NT> ty;
    al::Stage<T, DB, C, VEC, NT> tz;
    ty.setup(tid, J.sy.s, J.da);
    tz.setup(tid, J.sz.s, J.db);
    auto fetch = [&](int c) {
        const int t0 = at.s0 + C * c;
        ty.load(yp + t0 * J.sy.s, J.sy.s, at.s1 - t0, J.da);
        tz.load(zp + t0 * J.sz.s, J.sz.s, at.s1 - t0, J.db);
    };
    if (at.nc) fetch(J.rev ? at.nc - 1 : 0);
    int had = -1;
    for (int t = 0; t < at.nc; ++t) {
        const int c = J.rev ? at.nc - 1 - t : t, m = min(C, at.s1 - at.s0 - C * c);
        __syncthreads();
        ty.store(Ys);
        tz.store(Zs);
        if (m != had && tid < C) wu[tid] = add_weight(at.a2, tid, m, J.rev, J.umul);
        had = m;
        __syncthreads();
        if (t + 1 < at.nc) fetch(J.rev ? c - 1 : c + 1);
        const float all = power(at.a2, m);
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[x][r] *= all;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const Weighed<T> zw(col_frag<PB>(Zs, 16 * kb, 32 * w, lane), wu + 16 * kb, h);
#pragma unroll
            for (int x = 0; x < AT; ++x) S[x] = zw.add(col_frag<PA>(Ys, 16 * kb, 32 * x, lane), S[x]);
        }
    }
    float* dst = J.seg + (at.nh * a.G + at.seg) * (int64_t)(J.da * J.db);
    const int b = 32 * w + l31;
    if (b < J.db)
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                if (row < J.da) dst[row * J.db + b] = S[x][r];
            }
}

// segment sums -> the states that the segments start from (in place), and the final state
__global__ __launch_bounds__(256) void lin_scan_kernel(const Args a) {
    const Job& J = a.job[blockIdx.y];
    const int64_t E = (int64_t)J.da * J.db, idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= a.N * a.H * E) return;
    const int64_t nh = idx / E, e = idx - nh * E, n = nh / a.H;
    const float a2 = a.log_decay[nh - n * a.H] * al::LOG2E;
    const int len = length_of(a, n);
    float s = 0.f;
    if (J.init) {
        const int64_t row = e / J.db, col = e - row * J.db;
        s = J.init[nh * E + (J.init_t ? col * J.da + row : e)];
    }
    float* p = J.seg + nh * a.G * E + e;
    for (int t = 0; t < a.G; ++t) {
        const int g = J.rev ? a.G - 1 - t : t;
        const int m = min(max(len - g * a.per, 0), a.per);
        const float add = p[g * E];
        p[g * E] = s;
        s = fmaf(power(a2, m), s, add);
    }
    if (J.last) J.last[nh * E + e] = s;
}

template <class T, int DA, int DB, bool VEC>
__global__ __launch_bounds__(2 * DB) void lin_out_kernel(const Args a) {
    constexpr int NT = 2 * DB, PA = DA + Ty<T>::PAD, PB = DB + Ty<T>::PAD, AT = DA / 32, KA = DA / 16;
    extern __shared__ __attribute__((aligned(16))) char smem[];
    T* Xs = reinterpret_cast<T*>(smem);
    T* Ys = Xs + C * PA;
    T* Zs = Ys + C * PA;
    float* wu = reinterpret_cast<float*>(Zs + C * PB);
    const int tid = threadIdx.x, lane = tid & 63, l31 = lane & 31, h = lane >> 5, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Place at(a);
    const Job& J = a.job[at.job];
    const T* xp = static_cast<const T*>(J.x) + at.n * J.sx.n + at.h * J.sx.h;
    const T* yp = static_cast<const T*>(J.y) + at.n * J.sy.n + at.h * J.sy.h;
    const T* zp = static_cast<const T*>(J.z) + at.n * J.sz.n + at.h * J.sz.h;
    T* op = static_cast<T*>(J.o) + at.n * J.so.n + at.h * J.so.h;
    const int b = 32 * w + l31, rev = J.rev;
    const int64_t E = (int64_t)J.da * J.db;

    f32x16 S[AT];
    {
        const float* src = a.G > 1 ? J.seg + (at.nh * a.G + at.seg) * E : (J.init ? J.init + at.nh * E : nullptr);
        const bool turned = a.G == 1 && J.init_t;
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                S[x][r] = src && row < J.da && b < J.db ? src[turned ? b * J.da + row : row * J.db + b] : 0.f;
            }
    }
    // decays between the tokens of a 32 x 32 tile of scores (row j, column i = l31): on the diagonal and one tile off it
    f32x16 near, far;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        const int d = rev ? tile_row(r, h) - l31 : l31 - tile_row(r, h);
        near[r] = d >= 0 ? J.amul * power(at.a2, d) : 0.f;
        far[r] = J.amul * power(at.a2, d + 32);
    }
    al::Stage<T, DA, C, VEC, NT> tx, ty;
    al::Stage<T, DB, C, VEC, NT> tz;
    tx.setup(tid, J.sx.s, J.da);
    ty.setup(tid, J.sy.s, J.da);
    tz.setup(tid, J.sz.s, J.db);
    auto fetch = [&](int c) {
        const int t0 = at.s0 + C * c;
        tx.load(xp + t0 * J.sx.s, J.sx.s, at.s1 - t0, J.da);
        ty.load(yp + t0 * J.sy.s, J.sy.s, at.s1 - t0, J.da);
        tz.load(zp + t0 * J.sz.s, J.sz.s, at.s1 - t0, J.db);
    };
    if (at.nc) fetch(rev ? at.nc - 1 : 0);
    int had = -1;
    for (int t = 0; t < at.nc; ++t) {
        const int c = rev ? at.nc - 1 - t : t, t0 = at.s0 + C * c, m = min(C, at.s1 - t0);
        __syncthreads();
        tx.store(Xs);
        ty.store(Ys);
        tz.store(Zs);
        if (m != had && tid < C) wu[tid] = add_weight(at.a2, tid, m, rev, J.umul);
        had = m;
        __syncthreads();
        if (t + 1 < at.nc) fetch(rev ? c - 1 : c + 1);
        typename Ty<T>::Frag zf[4];
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) zf[kb] = col_frag<PB>(Zs, 16 * kb, 32 * w, lane);
#pragma unroll
        for (int it = 0; it < 2; ++it) {
            if (32 * it >= m) break;
            const T* xr = Xs + (32 * it + l31) * PA;
            f32x16 o = zero16(), os = zero16();
#pragma unroll
            for (int jt = 0; jt < 2; ++jt) {
                if (rev ? jt < it : jt > it) continue;
                f32x16 x = zero16();
                const T* yr = Ys + (32 * jt + l31) * PA;
#pragma unroll
                for (int k = 0; k < KA; ++k) x = mul(near_frag(yr + 16 * k + 8 * h), near_frag(xr + 16 * k + 8 * h), x);
#pragma unroll
                for (int r = 0; r < 16; ++r) x[r] *= jt == it ? near[r] : far[r];
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) o = mul(zf[2 * jt + k2], tile_frag<T>(x, k2), o);
            }
#pragma unroll
            for (int x = 0; x < AT; ++x)
#pragma unroll
                for (int k2 = 0; k2 < 2; ++k2) os = mul(tile_frag<T>(S[x], k2), spread_frag(xr + 32 * x + 16 * k2 + 4 * h), os);
            const int i = 32 * it + l31;
            const float wi = J.imul * power(at.a2, rev ? max(m - 1 - i, 0) : i + 1);
            if (i < m) {
                T* row = op + (int64_t)(t0 + i) * J.so.s;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    f32x4 v;
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = fmaf(wi, os[4 * q + e], o[4 * q + e]);
                    const int col = 32 * w + 8 * q + 4 * h;
                    store4<VEC>(row + col, v, J.db - col);
                }
            }
        }
        const float all = power(at.a2, m);
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) S[x][r] *= all;
#pragma unroll
        for (int kb = 0; kb < 4; ++kb) {
            const Weighed<T> zw(zf[kb], wu + 16 * kb, h);
#pragma unroll
            for (int x = 0; x < AT; ++x) S[x] = zw.add(col_frag<PA>(Ys, 16 * kb, 32 * x, lane), S[x]);
        }
    }
    if (J.last && a.G == 1 && b < J.db)
#pragma unroll
        for (int x = 0; x < AT; ++x)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = 32 * x + tile_row(r, h);
                if (row < J.da) J.last[at.nh * E + row * J.db + b] = S[x][r];
            }
    // rows behind the sequence's length
    for (int x = tid; x < (at.send - at.s1) * J.db; x += NT) {
        const int row = x / J.db;
        op[(int64_t)(at.s1 + row) * J.so.s + (x - row * J.db)] = (T)0.f;
    }
}

// ---------------------------------------------------------------- one token
// a workgroup per head: 16-byte pieces of the state's rows over the threads, the row sums meet through LDS in row-group order
template <class T, bool VEC>
__global__ __launch_bounds__(256) void lin_step_kernel(const T* __restrict__ q, const T* __restrict__ k, const T* __restrict__ v,
                                                       const float* __restrict__ log_decay, const float* state, int H, int dk, int dv, int lanes,
                                                       float scale, T* __restrict__ out, float* out_state) {
    constexpr int E = VEC ? 4 : 1;
    __shared__ float part[256 * E];
    const int64_t nh = blockIdx.x;
    const int h = (int)(nh % H), groups = 256 / lanes, col = (threadIdx.x % lanes) * E, grp = threadIdx.x / lanes;
    const float w = __builtin_amdgcn_exp2f(log_decay[h] * al::LOG2E);
    const float* src = state + nh * dk * dv;
    float* dst = out_state + nh * dk * dv;
    const int c0 = col;
    if (c0 < dv) {                                           // lanes * E >= dv
        float vv[E], o[E];
#pragma unroll
        for (int e = 0; e < E; ++e) { vv[e] = (float)v[nh * dv + c0 + e]; o[e] = 0.f; }
#pragma unroll 4
        for (int r = grp; r < dk; r += groups) {
            const float kr = (float)k[nh * dk + r], qr = (float)q[nh * dk + r];
            float s[E];
            if (VEC) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(src + r * dv + c0);
#pragma unroll
                for (int e = 0; e < E; ++e) s[e] = x[e];
            } else s[0] = src[r * dv + c0];
#pragma unroll
            for (int e = 0; e < E; ++e) { s[e] = fmaf(w, s[e], kr * vv[e]); o[e] = fmaf(qr, s[e], o[e]); }
            if (VEC) *reinterpret_cast<f32x4*>(dst + r * dv + c0) = f32x4{s[0], s[E > 1 ? 1 : 0], s[E > 2 ? 2 : 0], s[E > 3 ? 3 : 0]};
            else dst[r * dv + c0] = s[0];
        }
#pragma unroll
        for (int e = 0; e < E; ++e) part[threadIdx.x * E + e] = o[e];
    }
    __syncthreads();
    for (int c = threadIdx.x; c < dv; c += 256) {
        const int lane = c / E, e = c % E;
        float o = 0.f;
        for (int g = 0; g < groups; ++g) o += part[(g * lanes + lane) * E + e];
        out[nh * dv + c] = (T)(o * scale);
    }
}

// ---------------------------------------------------------------- host
// heads * sequences that leave the chip part empty are cut into segments, down to 256 tokens each
static void cut(Args& a) {
    const int64_t blocks = a.jobs * a.N * a.H;
    a.G = 1; a.per = (a.S + C - 1) / C * C;
    if (blocks <= 0 || blocks >= 1024 || a.S <= 512) return;
    const int64_t want = std::min<int64_t>((1024 + blocks - 1) / blocks, a.S / 256);
    a.per = (int)((((int64_t)a.S + want - 1) / want + C - 1) / C * C);
    a.G = (a.S + a.per - 1) / a.per;
}
static int pad32(int d) { return d <= 32 ? 32 : (d <= 64 ? 64 : 128); }

template <class T, int DA, int DB, bool VEC> static int launch(const Args& a, hipStream_t s) {
    constexpr size_t pa = DA + Ty<T>::PAD, pb = DB + Ty<T>::PAD;
    constexpr size_t out_lds = (2 * pa + pb) * C * sizeof(T) + C * 4, state_lds = (pa + pb) * C * sizeof(T) + C * 4;
    const int64_t grid = a.jobs * a.N * a.H * a.G;
    NR_UNSUPPORTED(grid > 0x7fffffff, "linear_attention: %lld workgroups", (long long)grid);
    if (a.G > 1) {
        if (state_lds > 64 * 1024)
            (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&lin_state_kernel<T, DA, DB, VEC>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)state_lds);
        hipLaunchKernelGGL((lin_state_kernel<T, DA, DB, VEC>), dim3((unsigned)grid), dim3(2 * DB), state_lds, s, a);
        if (int rc = check_launch("linear_attention states")) return rc;
        int64_t most = 0;
        for (int j = 0; j < a.jobs; ++j) most = std::max<int64_t>(most, a.N * a.H * (int64_t)(a.job[j].da * a.job[j].db));
        hipLaunchKernelGGL(lin_scan_kernel, dim3((unsigned)((most + 255) / 256), a.jobs), dim3(256), 0, s, a);
        if (int rc = check_launch("linear_attention scan")) return rc;
    }
    if (out_lds > 64 * 1024)
        (void)hipFuncSetAttribute(reinterpret_cast<const void*>(&lin_out_kernel<T, DA, DB, VEC>), hipFuncAttributeMaxDynamicSharedMemorySize, (int)out_lds);
    hipLaunchKernelGGL((lin_out_kernel<T, DA, DB, VEC>), dim3((unsigned)grid), dim3(2 * DB), out_lds, s, a);
    return check_launch("linear_attention");
}
template <class T, int DA, bool VEC> static int pick_b(const Args& a, hipStream_t s) {
    const int b = pad32(a.job[0].db);
    return b == 32 ? launch<T, DA, 32, VEC>(a, s) : (b == 64 ? launch<T, DA, 64, VEC>(a, s) : launch<T, DA, 128, VEC>(a, s));
}
template <class T, bool VEC> static int pick_a(const Args& a, hipStream_t s) {
    const int d = pad32(a.job[0].da);
    return d == 32 ? pick_b<T, 32, VEC>(a, s) : (d == 64 ? pick_b<T, 64, VEC>(a, s) : pick_b<T, 128, VEC>(a, s));
}
static int run(const Args& a, bool bf16, hipStream_t s) {
    const size_t e = bf16 ? 2 : 4;
    bool vec = true;
    for (int j = 0; j < a.jobs; ++j) {
        const Job& J = a.job[j];
        vec = vec && al::aligned16(J.x, J.sx, J.da, e, C) && al::aligned16(J.y, J.sy, J.da, e, C) && al::aligned16(J.z, J.sz, J.db, e, C) && al::aligned16(J.o, J.so, J.db, e, C);
    }
    return bf16 ? (vec ? pick_a<__bf16, true>(a, s) : pick_a<__bf16, false>(a, s)) : (vec ? pick_a<float, true>(a, s) : pick_a<float, false>(a, s));
}
static Args base(const LinProblem& p) {
    Args a{};
    a.N = p.N; a.S = p.S; a.H = p.H; a.log_decay = p.log_decay; a.lens = p.lens;
    return a;
}
static size_t seg_floats(const Args& a) {
    size_t f = 0;
    if (a.G > 1)
        for (int j = 0; j < a.jobs; ++j) f += (size_t)(a.N * a.H) * a.G * a.job[j].da * a.job[j].db;
    return f;
}
static void place_segs(Args& a, float*& ws) {
    if (a.G > 1)
        for (int j = 0; j < a.jobs; ++j) { a.job[j].seg = ws; ws += (size_t)(a.N * a.H) * a.G * a.job[j].da * a.job[j].db; }
}
static AttnStrides dense(int S, int H, int d) { return {(int64_t)S * H * d, (int64_t)H * d, d}; }

static Args fwd_args(const LinProblem& p, void* out, float* last) {
    Args a = base(p);
    a.jobs = 1;
    a.job[0] = Job{p.q, p.k, p.v, p.sq, p.sk, p.sv, dense(p.S, p.H, p.dv), out, p.state, 0, last, nullptr, p.dk, p.dv, 0, p.scale, p.scale, 1.f};
    cut(a);
    return a;
}
// the three products of the backward: one launch, or two where dk and dv are padded to different widths
static int bwd_args(const LinProblem& p, const void* g, const float* dlast, void* dq, void* dk, void* dv, float* dstate, Args (&a)[2]) {
    const AttnStrides sg = dense(p.S, p.H, p.dv), sk = dense(p.S, p.H, p.dk);
    const Job jq{g, p.v, p.k, sg, p.sv, p.sk, sk, dq, p.state, 1, nullptr, nullptr, p.dv, p.dk, 0, p.scale, p.scale, 1.f};
    const Job jk{p.v, g, p.q, p.sv, sg, p.sq, sk, dk, dlast, 1, nullptr, nullptr, p.dv, p.dk, 1, p.scale, 1.f, p.scale};
    const Job jv{p.k, p.q, g, p.sk, p.sq, sg, sg, dv, dlast, 0, dstate, nullptr, p.dk, p.dv, 1, p.scale, 1.f, p.scale};
    a[0] = a[1] = base(p);
    a[0].job[0] = jq; a[0].job[1] = jk; a[0].jobs = 2;
    if (pad32(p.dk) == pad32(p.dv)) {
        a[0].job[2] = jv; a[0].jobs = 3;
        cut(a[0]);
        return 1;
    }
    a[1].job[0] = jv; a[1].jobs = 1;
    cut(a[0]);
    cut(a[1]);
    return 2;
}

}  // namespace lin

size_t lin_fwd_ws_bytes(const LinProblem& p) { return lin::seg_floats(lin::fwd_args(p, nullptr, nullptr)) * 4; }
int lin_fwd(const LinProblem& p, void* out, float* last, void* ws, size_t ws_bytes, hipStream_t s) {
    lin::Args a = lin::fwd_args(p, out, last);
    if (ws_bytes < lin::seg_floats(a) * 4 || (!ws && lin::seg_floats(a))) { set_error("linear_attention_fwd: workspace too small"); return NR_ERR_WORKSPACE; }
    float* w = static_cast<float*>(ws);
    lin::place_segs(a, w);
    return lin::run(a, p.bf16, s);
}
size_t lin_bwd_ws_bytes(const LinProblem& p) {
    lin::Args a[2];
    const int n = lin::bwd_args(p, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, a);
    return (lin::seg_floats(a[0]) + (n == 2 ? lin::seg_floats(a[1]) : 0)) * 4;
}
int lin_bwd(const LinProblem& p, const void* dout, const float* dlast, void* dq, void* dk, void* dv, float* dstate, void* ws, size_t ws_bytes,
            hipStream_t s) {
    lin::Args a[2];
    const int n = lin::bwd_args(p, dout, dlast, dq, dk, dv, dstate, a);
    const size_t need = lin_bwd_ws_bytes(p);
    if (ws_bytes < need || (!ws && need)) { set_error("linear_attention_bwd: workspace too small"); return NR_ERR_WORKSPACE; }
    float* w = static_cast<float*>(ws);
    for (int i = 0; i < n; ++i) {
        lin::place_segs(a[i], w);
        if (int rc = lin::run(a[i], p.bf16, s)) return rc;
    }
    return NR_OK;
}

int lin_step(const void* q, const void* k, const void* v, const float* log_decay, const float* state, int64_t N, int H, int dk, int dv, bool bf16,
             float scale, void* out, float* out_state, hipStream_t s) {
    const int64_t grid = N * H;
    NR_UNSUPPORTED(grid > 0x7fffffff, "linear_attention_step: %lld heads", (long long)grid);
    const bool vec = dv % 4 == 0 && ((reinterpret_cast<uintptr_t>(state) | reinterpret_cast<uintptr_t>(out_state)) & 15) == 0;
    int lanes = 8;                                           // threads along a row of the state
    while (lanes * (vec ? 4 : 1) < dv) lanes *= 2;
#define NR_STEP(T, VEC) hipLaunchKernelGGL((lin::lin_step_kernel<T, VEC>), dim3((unsigned)grid), dim3(256), 0, s, static_cast<const T*>(q), \
        static_cast<const T*>(k), static_cast<const T*>(v), log_decay, state, H, dk, dv, lanes, scale, static_cast<T*>(out), out_state)
    if (bf16) { if (vec) NR_STEP(__bf16, true); else NR_STEP(__bf16, false); }
    else      { if (vec) NR_STEP(float, true); else NR_STEP(float, false); }
#undef NR_STEP
    return check_launch("linear_attention_step");
}

}  // namespace nr
